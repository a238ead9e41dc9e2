"""The native module where the library of its C++ PyTorch operators is missing or
does not load: the ops over ctypes stay, the operators say why they cannot run."""

import os
import shutil
import subprocess
import sys
from pathlib import Path

import pytest

PACKAGE = Path(__file__).resolve().parents[1] / "jakal-net_amd"

CHECK = """
import torch
import jakal_net as J
import jakal_net_native as jn

assert jn.__file__.startswith({where!r})
assert jn.ABI_VERSION >= 19 and jn._LIB.jn_layer_norm_backward_workspace_bytes(4, 8) > 0
assert "propagation_topk" in jn.supported_ops()
x = torch.randn(3, 4)
for call in (lambda: jn.layer_norm(x), lambda: jn.stabilize(x[:, 0], x), lambda: jn.grad_norm([x]),
             lambda: jn.cross_entropy(x, torch.zeros(3, dtype=torch.int64)), lambda: jn.clip_grads([x], 1.0)):
    try:
        call()
    except NotImplementedError as exc:
        assert "libjakal_net_torch.so" in str(exc) and "did not load" in str(exc)
    else:
        raise AssertionError("no error")
assert J.native_status().available
assert torch.equal(J.layer_norm(x), torch.nn.functional.layer_norm(x, (4,)))  # CPU tensors take the PyTorch form
print("checked")
"""


@pytest.mark.parametrize("kind", ["missing", "broken"])
def test_the_module_loads_without_its_torch_operators(tmp_path, kind):
    shutil.copy(PACKAGE / "jakal_net_native.py", tmp_path)
    (tmp_path / "lib").mkdir()
    if kind == "broken":
        (tmp_path / "lib" / "libjakal_net_torch.so").write_bytes(b"no library")
    env = dict(os.environ, JAKAL_NET_HIP_LIB=str(PACKAGE / "lib" / "libjakal_net_hip.so"),
               PYTHONPATH=os.pathsep.join([str(tmp_path), str(PACKAGE)]))
    done = subprocess.run([sys.executable, "-c", CHECK.format(where=str(tmp_path))], env=env, cwd=tmp_path,
                          capture_output=True, text=True, timeout=120)
    assert done.returncode == 0 and "checked" in done.stdout, done.stderr
