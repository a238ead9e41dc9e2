"""The training-step operators that are timed beside the propagation ops.

Between its propagations a Progressive-B step normalises every layer update
(``stabilize``: tanh of the states, layer norm of the values, both times the
path's scale), normalises rows (``layer_norm``), takes the vocabulary cross
entropy and limits the gradients' global norm.  Each case is one call of one of
them as a program makes it: the forward alone, or forward and backward.

``run`` computes them in plain torch operations in 32 bits, or, where ``own`` is
true, through ``jakal_net``.  Inputs are what the operators meet in the model:
values a little off zero mean and unit variance, norm weights near 1, logits a
few units wide, gradients of the parameter list at the scale a mean loss leaves.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch
from torch.nn import functional as F

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _norm(rows, dim, dtype="fp32", params=None, affine="both", train=True):
    """Layer norm of rows x dim elements; params: the type of weight and bias; affine: both, weight or none."""
    return dict(op="norm", rows=rows, dim=dim, dtype=dtype, params=params or dtype, affine=affine, train=train)


def _stabilize(batch, nodes, dim, scale, dtype="fp32", params=None, train=True):
    """The end of a layer update over [batch, nodes] states and [batch, nodes, dim] values."""
    return dict(op="stabilize", batch=batch, nodes=nodes, dim=dim, scale=scale, dtype=dtype, params=params or dtype,
                train=train)


def _loss(rows, vocab, dtype="fp32", reduction="mean", ignored=0.0, train=True):
    """Cross entropy of rows x vocab logits; ignored: the share of padded positions."""
    return dict(op="loss", rows=rows, vocab=vocab, dtype=dtype, reduction=reduction, ignored=ignored, train=train)


def _clip(vocab, dim, rank, blocks, dtype="fp32", out="fp32", norm="2", clips=True, only_norm=False):
    """The gradients of a Progressive-B model (blocks = 0: of one family's score modules); clips: whether the limit
    is below their norm; only_norm: the norm is read and nothing scaled."""
    return dict(op="clip", vocab=vocab, dim=dim, rank=rank, blocks=blocks, dtype=dtype, out=out, norm=norm,
                clips=clips, only_norm=only_norm)


def listed():
    return [
        # the head's norm over the 64 query slots of one answered sequence
        dict(name="norm_query_infer", **_norm(64, 512, train=False)),
        # a norm over 16 graphs of 4096 nodes in bf16, training step
        dict(name="norm_graph_bf16_train", **_norm(16 * 4096, 512, dtype="bf16")),
        # odd rows and an odd width: no row but the first starts on 16 bytes
        dict(name="norm_ragged_train", **_norm(3 * 1531, 383)),
        # the update of the query slots of a decoding round, forward only
        dict(name="stabilize_query_infer", **_stabilize(16, 64, 512, 0.25, train=False)),
        # the update of the sequence layer in a training step: the model makes about twenty such calls
        dict(name="stabilize_sequence_train", **_stabilize(16, 512, 512, 0.25)),
        # scoring the 64 query tokens of one sequence: one loss a token, forward only
        dict(name="loss_query_score", **_loss(64, 16384, reduction="none", train=False)),
        # the model's own loss under bf16 autocast: 16 sequences of 64 query slots
        dict(name="loss_query_train", **_loss(16 * 64, 16384, dtype="bf16")),
        # a loss over every prefix position, a fifth of them padding: the largest
        dict(name="loss_prefix_train", **_loss(16 * 512, 16384, dtype="bf16", ignored=0.2)),
        # an odd vocabulary and odd rows in fp32, summed
        dict(name="loss_ragged_train", **_loss(1531, 4099, reduction="sum", ignored=0.1)),
        # the norm of one layer family's score gradients, as a monitor reads it: latency only
        dict(name="norm_of_scores", **_clip(0, 512, 64, 0, only_norm=True)),
        # the whole model's fp32 gradients, clipped into the optimizer's buffers
        dict(name="clip_model", **_clip(16384, 512, 64, 4)),
        # the same list in bf16, clipped into fp32 buffers beside master weights
        dict(name="clip_model_bf16", **_clip(16384, 512, 64, 4, dtype="bf16")),
    ]


NORM_ELEMENTS = 16 * 4096 * 512
LOSS_ELEMENTS = 16 * 512 * 16384


def _spread(rng, low, high):
    """A whole number between low and high, even over the logarithm."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _width(rng, low, high):
    """A row length: mostly a multiple of 8, else any."""
    d = _spread(rng, low, high)
    return max(low, d // 8 * 8) if rng.random() < 0.6 else d


def draw(rng):
    op = rng.choice(["norm", "norm", "stabilize", "stabilize", "loss", "loss", "loss", "clip", "clip"])
    dtype = rng.choice(["fp32", "fp32", "bf16", "bf16", "fp16"])
    params = rng.choice(["fp32", dtype])
    train = rng.random() < 0.7
    if op == "norm":
        dim = _width(rng, 8, 8192)
        rows = _spread(rng, 1, min(65536, NORM_ELEMENTS // dim))
        return _norm(rows, dim, dtype, params, rng.choice(["both", "both", "weight", "none"]), train)
    if op == "stabilize":
        dim = _width(rng, 16, 1024)
        batch = _spread(rng, 1, 16)
        nodes = _spread(rng, 1, min(4096, NORM_ELEMENTS // (dim * batch)))
        return _stabilize(batch, nodes, dim, round(rng.uniform(0.02, 1.0), 3), dtype, params, train)
    if op == "loss":
        vocab = _width(rng, 32, 65536)
        rows = _spread(rng, 2, min(8192, LOSS_ELEMENTS // vocab))
        return _loss(rows, vocab, dtype, rng.choice(["mean", "mean", "sum", "none"]),
                     rng.choice([0.0, 0.1, 0.3]) if rows > 16 else 0.0, train)
    blocks = rng.choice([0, 1, 2, 4])
    out = rng.choice(["fp32", dtype])
    return _clip(_spread(rng, 97, 16384), _width(rng, 16, 512), _spread(rng, 4, 64), blocks, dtype, out,
                 rng.choice(["2", "2", "2", "inf"]), rng.random() < 0.75, rng.random() < 0.25)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, *shape, scale=1.0, mean=0.0, dtype=torch.float32):
    return (torch.randn(shape, generator=g, device="cuda") * scale + mean).to(dtype)


def _shapes(case):
    """Parameter shapes of the model (of one score family where blocks is 0)."""
    d, r, v = case["dim"], case["rank"], case["vocab"]
    score = [(r, d), (r, d), (r,), ()]
    if not case["blocks"]:
        return score * 4
    norm, linear = [(d,), (d,)], [(d, d), (d,)]
    block = norm * 3 + [(256,), (256, d), (64,), (64, d)] + score * 4
    return ([(v, d), (d, 1), (d,)] + linear + [(1, d), (1,)] + norm * 4 + score * 5 + block * case["blocks"] + linear
            + [(4 * d, d), (4 * d,), (v, 4 * d), (v,)])


def _offsets(tensors):
    ends = [0]
    for t in tensors:
        ends.append(ends[-1] + (t.numel() + 63) // 64 * 64)
    return ends


def _views(buffer, tensors):
    return [buffer[at:at + t.numel()].view(t.shape) for at, t in zip(_offsets(tensors), tensors)]


def _affine(case, g, dim):
    kind = DTYPES[case["params"]]
    given = {"both": 2, "weight": 1, "none": 0}[case.get("affine", "both")]
    weight = _normal(g, dim, scale=0.1, mean=1.0, dtype=kind) if given else None
    bias = _normal(g, dim, scale=0.1, dtype=kind) if given > 1 else None
    return weight, bias


def prepare(case, seed):
    g = _generator(seed)
    state = dict(case=case)
    op = case["op"]
    if op == "clip":
        grads = [_normal(g, *s, scale=1e-3, dtype=DTYPES[case["dtype"]]) for s in _shapes(case)]
        size = sum(t.numel() for t in grads)
        norm = 1e-3 * math.sqrt(size) if case["norm"] == "2" else 3e-3
        state.update(grads=grads, limit=norm * (0.3 if case["clips"] else 10.0))
        if not case["only_norm"]:
            # the optimizer's gradients: views of one buffer, each on its own 64 elements
            buffer = torch.zeros(_offsets(grads)[-1], device="cuda", dtype=DTYPES[case["out"]])
            state.update(buffer=buffer, out=_views(buffer, grads))
        return state
    dtype = DTYPES[case["dtype"]]
    if op == "loss":
        rows, vocab = case["rows"], case["vocab"]
        logits = _normal(g, rows, vocab, scale=2.5, dtype=dtype)
        target = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
        if case["ignored"]:
            target[torch.rand(rows - 1, generator=g, device="cuda").lt(case["ignored"]).nonzero().squeeze(-1)] = -100
        state.update(logits=logits.requires_grad_(case["train"]), target=target)
        if case["reduction"] == "none" and case["train"]:
            state["grad"] = _normal(g, rows, scale=0.1, mean=1.0)
        return state
    lead = (case["rows"],) if op == "norm" else (case["batch"], case["nodes"])
    dim = case["dim"]
    state["val"] = _normal(g, *lead, dim, scale=1.3, mean=0.2, dtype=dtype).requires_grad_(case["train"])
    weight, bias = _affine(case, g, dim)
    if case["train"]:
        for p in (weight, bias):
            if p is not None:
                p.requires_grad_()
        state["grad"] = _normal(g, *lead, dim, scale=0.1, dtype=dtype)
    state.update(weight=weight, bias=bias)
    if op == "stabilize":
        state["state"] = _normal(g, *lead, scale=2.0, dtype=dtype).requires_grad_(case["train"])
        if case["train"]:
            state["grad_state"] = _normal(g, *lead, scale=0.1, dtype=dtype)
    return state


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
EPS = 1e-5


def run(state):
    case = state["case"]
    kind = case["op"]
    if own:
        return {"norm": _own_norm, "stabilize": _own_stabilize, "loss": _own_loss, "clip": _own_clip}[kind](state, case)
    with torch.no_grad():
        return {"norm": _plain_norm, "stabilize": _plain_stabilize, "loss": _plain_loss,
                "clip": _plain_clip}[kind](state, case)


def _jakal():
    if "jakal_net" not in sys.modules:
        sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "jakal-net_amd"))
    import jakal_net

    return jakal_net


def _own_norm(state, case):
    J = _jakal()
    y = J.layer_norm(state["val"], state["weight"], state["bias"], eps=EPS, implementation="native")
    out = {"y": y.detach()}
    if case["train"]:
        names = [n for n in ("val", "weight", "bias") if state[n] is not None]
        grads = torch.autograd.grad(y, [state[n] for n in names], state["grad"])
        out.update({"grad_" + n: t for n, t in zip(names, grads)})
    return out


def _own_stabilize(state, case):
    J = _jakal()
    t, y = J.stabilize(state["state"], state["val"], state["weight"], state["bias"], eps=EPS, scale=case["scale"],
                       implementation="native")
    out = {"state": t.detach(), "y": y.detach()}
    if case["train"]:
        names = ("state", "val", "weight", "bias")
        grads = torch.autograd.grad([t, y], [state[n] for n in names], [state["grad_state"], state["grad"]])
        out.update({"grad_" + n: t for n, t in zip(names, grads)})
    return out


def _own_loss(state, case):
    J = _jakal()
    loss = J.cross_entropy(state["logits"], state["target"], reduction=case["reduction"], implementation="native")
    out = {"loss": loss.detach()}
    if case["train"]:
        out["grad_logits"] = torch.autograd.grad(loss, state["logits"], state.get("grad"))[0]
    return out


def _own_clip(state, case):
    J = _jakal()
    kind = float(case["norm"])
    if case["only_norm"]:
        return {"norm": J.grad_norm(state["grads"], kind, implementation="native")}
    norm = J.clip_grads(state["grads"], state["limit"], kind, out=state["out"], implementation="native")
    return {"norm": norm, "grads": state["buffer"]}


def _plain_rows(state, case, scale):
    """Layer norm of scale * val with its gradients."""
    val, weight, bias = state["val"], state["weight"], state["bias"]
    x = val.float() * scale
    x = x - x.mean(-1, keepdim=True)
    r = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
    h = x * r
    y = h if weight is None else h * weight.float()
    out = {"y": (y if bias is None else y + bias.float()).to(val.dtype)}
    if case["train"]:
        g = state["grad"].float()
        gw = g if weight is None else g * weight.float()
        dx = scale * r * (gw - gw.mean(-1, keepdim=True) - h * (gw * h).mean(-1, keepdim=True))
        out["grad_val"] = dx.to(val.dtype)
        rows = tuple(range(g.dim() - 1))
        if weight is not None:
            out["grad_weight"] = (g * h).sum(rows).to(weight.dtype)
        if bias is not None:
            out["grad_bias"] = g.sum(rows).to(bias.dtype)
    return out


def _plain_norm(state, case):
    return _plain_rows(state, case, 1.0)


def _plain_stabilize(state, case):
    s = state["state"]
    t = torch.tanh(s.float() * case["scale"])
    out = {"state": t.to(s.dtype), "y": None}
    if case["train"]:
        out["grad_state"] = (case["scale"] * (1.0 - t * t) * state["grad_state"].float()).to(s.dtype)
    out.update(_plain_rows(state, case, case["scale"]))
    return out


def _plain_loss(state, case):
    z, target = state["logits"].float(), state["target"]
    valid = target != -100
    at = torch.where(valid, target, 0).unsqueeze(-1)
    z = z - z.max(-1, keepdim=True).values
    e = torch.exp(z)
    total = e.sum(-1, keepdim=True)
    loss = torch.where(valid, (torch.log(total) - z.gather(-1, at)).squeeze(-1), 0.0)
    count = valid.sum()
    reduced = {"none": loss, "sum": loss.sum(), "mean": loss.sum() / count}[case["reduction"]]
    out = {"loss": reduced}
    if case["train"]:
        scale = torch.ones_like(loss) if case["reduction"] == "sum" else state.get("grad", 1.0 / count)
        p = e / total
        p.scatter_add_(-1, at, torch.full_like(at, -1.0, dtype=p.dtype))
        p = p * torch.where(valid, scale, 0.0).unsqueeze(-1)
        out["grad_logits"] = p.to(state["logits"].dtype)
    return out


def _plain_clip(state, case):
    grads = state["grads"]
    if case["norm"] == "2":
        norm = torch.sqrt(torch.stack([(t.float() * t.float()).sum() for t in grads]).sum())
    else:
        norm = torch.stack([t.float().abs().max() for t in grads]).max()
    if case["only_norm"]:
        return {"norm": norm}
    scale = torch.clamp(state["limit"] / (norm + 1e-6), max=1.0)
    for t, o in zip(grads, state["out"]):
        o.copy_(t.float() * scale)
    return {"norm": norm, "grads": state["buffer"]}


# ---------------------------------------------------------------------------
# what a pass cannot do without, and its definition in 64 bits
# ---------------------------------------------------------------------------
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}


def work(case):
    e = SIZE[case["dtype"]]
    if case["op"] == "clip":
        n = sum(math.prod(s) for s in _shapes(case))
        written = 0 if case["only_norm"] else SIZE[case["out"]]
        return {"bytes": n * (e + written), "flops": n * (3 if written else 2)}
    if case["op"] == "loss":
        rows, vocab = case["rows"], case["vocab"]
        n = rows * vocab
        # a padded row's logits need not be read
        read = int(round(rows * (1.0 - case["ignored"]))) * vocab
        out = rows * 4 if case["reduction"] == "none" else 4
        return {"bytes": read * e + rows * 8 + out + (n * e if case["train"] else 0),
                "flops": read * (7 if case["train"] else 4)}
    dim, p = case["dim"], SIZE[case["params"]]
    rows = case["rows"] if case["op"] == "norm" else case["batch"] * case["nodes"]
    given = {"both": 2, "weight": 1, "none": 0}[case.get("affine", "both")]
    width = dim + (1 if case["op"] == "stabilize" else 0)
    times = 2 if case["train"] else 1
    return {"bytes": times * (2 * rows * width * e + given * dim * p),
            "flops": rows * dim * (22 if case["train"] else 8)}


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "clip":
        flat = [t.double().reshape(-1) for t in state["grads"]]
        norm = torch.linalg.vector_norm(torch.cat(flat), float(case["norm"]))
        if case["only_norm"]:
            return {"norm": norm}
        factor = min(1.0, state["limit"] / (float(norm) + 1e-6))
        buffer = state["buffer"].double()
        for t, o in zip(state["grads"], _views(buffer, state["grads"])):
            o.copy_(factor * t.double())
        return {"norm": norm, "grads": buffer}
    if case["op"] == "loss":
        z = state["logits"].detach().double().requires_grad_(case["train"])
        loss = F.cross_entropy(z, state["target"], ignore_index=-100, reduction=case["reduction"])
        out = {"loss": loss.detach()}
        if case["train"]:
            grad = state["grad"].double() if "grad" in state else None
            out["grad_logits"] = torch.autograd.grad(loss, z, grad)[0]
        return out
    leaves = {n: state[n].detach().double().requires_grad_(case["train"])
              for n in ("state", "val", "weight", "bias") if state.get(n) is not None}
    scale = case.get("scale", 1.0)
    y = F.layer_norm(leaves["val"] * scale, (case["dim"],), leaves.get("weight"), leaves.get("bias"), EPS)
    out, ends, seeds = {}, [y], [state.get("grad")]
    if case["op"] == "stabilize":
        t = torch.tanh(leaves["state"] * scale)
        out["state"] = t.detach()
        ends.append(t)
        seeds.append(state.get("grad_state"))
    out["y"] = y.detach()
    if case["train"]:
        grads = torch.autograd.grad(ends, list(leaves.values()), [g.double() for g in seeds])
        out.update({"grad_" + n: t for n, t in zip(leaves, grads)})
    return out
