"""Oracles of the 8-bit path in 64 bits, written from the definitions (no code of the package)."""

import torch

F64 = torch.float64
BLOCK = 128


def e4m3_grid() -> torch.Tensor:
    """The finite non-negative e4m3 values in order: 0, subnormals of 2^-9, then 8 values per power of two up to 448."""
    values = [k * 2.0**-9 for k in range(8)]
    for e in range(-6, 9):
        values += [(1 + m / 8) * 2.0**e for m in range(8)]
    values = [v for v in values if v <= 448.0]
    assert len(values) == 127
    return torch.tensor(values, dtype=F64)


def round_e4m3(v: torch.Tensor) -> torch.Tensor:
    """Nearest grid value; of two equally near, the one with an even code (its place in the grid)."""
    grid = e4m3_grid().to(v.device)
    mag = v.abs()
    hi = torch.searchsorted(grid, mag).clamp(max=len(grid) - 1)
    lo = (hi - 1).clamp(min=0)
    dlo, dhi = mag - grid[lo], grid[hi] - mag
    pick = torch.where((dlo < dhi) | ((dlo == dhi) & (lo % 2 == 0)), lo, hi)
    return torch.where(v < 0, -grid[pick], grid[pick])


def quantize(x: torch.Tensor, square: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes as 64-bit values with NaN for what is not finite, scales) of a matrix; blocks of 1 x 128 or 128 x 128."""
    x = x.double()
    R, C = x.shape
    br = BLOCK if square else 1
    nr, nc = -(-R // br), -(-C // BLOCK)
    scales = torch.ones(nr, nc, dtype=F64, device=x.device)
    codes = torch.empty_like(x)
    powers = torch.exp2(torch.arange(-116, 128, dtype=F64, device=x.device))
    for j in range(nc):
        cols = slice(j * BLOCK, (j + 1) * BLOCK)
        part = x[:, cols]
        fin = part.isfinite()
        top = torch.where(fin, part.abs(), 0.0).amax(dim=1)
        top = torch.stack([top[i * br:(i + 1) * br].max() for i in range(nr)]) if square else top
        # smallest power of two s with top <= 448 s
        s = powers[torch.searchsorted(448.0 * powers, top).clamp(max=len(powers) - 1)]
        scales[:, j] = torch.where(top > 0, s, 1.0)
        rows = scales[:, j].repeat_interleave(br)[:R, None]
        codes[:, cols] = torch.where(fin, round_e4m3(torch.where(fin, part, 0.0) / rows), float("nan"))
    return codes, scales


def values(x: torch.Tensor, square: bool = False) -> torch.Tensor:
    """What the codes and scales of ``x`` stand for."""
    c, s = quantize(x, square)
    br = BLOCK if square else 1
    return c * s.repeat_interleave(br, 0)[: c.shape[0]].repeat_interleave(BLOCK, 1)[:, : c.shape[1]]


def values_along_rows(x: torch.Tensor) -> torch.Tensor:
    """``x`` quantised in blocks of 128 x 1."""
    return values(x.t()).t()


def half_step(dtype: torch.dtype) -> float:
    """Largest relative error of one rounding to ``dtype``."""
    return torch.finfo(dtype).eps / 2


def product_bound(a: torch.Tensor, b: torch.Tensor, y: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """Elementwise error that ``a @ b.T`` with exact products may have: an fp32 sum of K terms in any order, each addition
    rounded or truncated (2^-23 of a partial sum, which is at most the sum of magnitudes), then one rounding to ``dtype``
    (below the smallest normal number, half a subnormal step)."""
    K = a.shape[1]
    fi = torch.finfo(dtype)
    return (K + 64) * 2.0**-23 * (a.abs() @ b.abs().t()) * (1 + half_step(dtype)) + half_step(dtype) * y.abs() + fi.smallest_normal * fi.eps / 2


def assert_within(got: torch.Tensor, want: torch.Tensor, bound: torch.Tensor, what: str) -> None:
    off = (got.double() - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} values out of bounds, worst {float((off / bound.clamp_min(1e-300)).max()):.3g} times the bound"


def norm(x: torch.Tensor, residual: torch.Tensor | None, gain: torch.Tensor | None, eps: float) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(y, stored sum, r) in 64 bits; the sum as the type of the inputs holds it."""
    t = x if residual is None else (x.double() + residual.double()).to(x.dtype)
    t = t.double()
    r = (t.square().mean(dim=-1, keepdim=True) + eps).rsqrt()
    return t * r * (1.0 if gain is None else gain.double()), t, r


def norm_backward(g: torch.Tensor, gsum: torch.Tensor | None, t: torch.Tensor, r: torch.Tensor, gain: torch.Tensor | None) -> tuple[torch.Tensor, torch.Tensor]:
    """(gradient of the sum, gradient of the gain) for y = t r gain."""
    g = g.double()
    wg = g if gain is None else g * gain.double()
    dt = r * (wg - t * r * r * (wg * t).mean(dim=-1, keepdim=True))
    return dt if gsum is None else dt + gsum.double(), (g * t * r).reshape(-1, t.shape[-1]).sum(0)
