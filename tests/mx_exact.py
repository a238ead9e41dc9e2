"""Operands of products whose sums are the same in any order: small whole numbers times
powers of two, whose partial sums stay below 2^24, and single elements with as many bits
as their type has.  fp32 sums of them are exact, so that a product is its float64 value
rounded once, and a lost term, slice or split shows, however long the sum is."""

from __future__ import annotations

import torch

from mx_oracle import RUN

# whole magnitudes of a run, the largest last: of the format's bits each
MAGNITUDES = {"e2m1": [0.0, 1.0, 2.0, 3.0, 4.0, 6.0], "e4m3": [float(i) for i in range(16)]}
BITS = {torch.float32: 24, torch.float16: 11, torch.bfloat16: 8}


def _generator(seed: int, dev) -> torch.Generator:
    return torch.Generator(device=dev).manual_seed(seed)


def whole(seed: int, *shape: int, dev="cpu", top: int = 3) -> torch.Tensor:
    """Whole numbers from -top to top, in fp32."""
    return torch.randint(-top, top + 1, shape, generator=_generator(seed, dev), device=dev).float()


def kept(seed: int, rows: int, dim: int, form: str, dev="cpu") -> torch.Tensor:
    """[rows, dim] whole numbers that the format holds as they are, runs times 1, 2 or 4."""
    g = _generator(seed, dev)
    runs = -(-dim // RUN)
    grid = torch.tensor(MAGNITUDES[form], device=dev)
    v = grid[torch.randint(0, len(grid), (rows, runs, RUN), generator=g, device=dev)]
    v[..., 0] = grid[-1]
    v = v * (1 - 2 * torch.randint(0, 2, (rows, runs, RUN), generator=g, device=dev))
    v = v * torch.exp2(torch.randint(0, 3, (rows, runs, 1), generator=g, device=dev).float())
    return v.flatten(-2)[:, :dim].contiguous()


def places(count: int, size: int) -> torch.Tensor:
    """`count` places in an axis of `size`: its ends, both sides of multiples of the slices and tiles, and others."""
    at = [0, size - 1, size - 2, size - 8, size - 9]
    for step in (32, 64, 128, 256):
        for k in (1, 2, 3, size // step // 2, size // step - 1, size // step):
            at += [k * step - 1, k * step]
    at = sorted({p for p in at if 0 <= p < size})
    return torch.tensor([at[i % len(at)] if i < len(at) else (i * 7919) % size for i in range(count)])


def lonely(seed: int, rows: int, dim: int, dtype: torch.dtype, bits: int, dev="cpu") -> torch.Tensor:
    """[rows, dim] of zeros but for one number in [1, 2) a row, with `bits` bits (those of its type at most)."""
    bits = min(bits, BITS[dtype])
    v = torch.randint(2 ** (bits - 1), 2 ** bits, (rows,), generator=torch.Generator().manual_seed(seed)) | 1
    x = torch.zeros(rows, dim, dtype=dtype)
    x[torch.arange(rows), places(rows, dim)] = (v.double() / 2 ** (bits - 1)).to(dtype)
    return x.to(dev)


def product(a: torch.Tensor, b: torch.Tensor, bias=None) -> torch.Tensor:
    """a @ b + bias in float64, of sums that fp32 holds whatever their order."""
    a, b = a.double(), b.double()
    assert float((a.abs() @ b.abs()).max()) < 2.0 ** 24
    return a @ b if bias is None else a @ b + bias.double()


def same(what: str, got: torch.Tensor, want: torch.Tensor) -> None:
    """got is want rounded once to its type."""
    want = want.to(got.dtype)
    assert got.shape == want.shape, f"{what}: shape {tuple(got.shape)} for {tuple(want.shape)}"
    wrong = got != want
    assert not bool(wrong.any()), f"{what}: {int(wrong.sum())} of {wrong.numel()} differ, the first at {wrong.nonzero()[0].tolist()}"
