"""Matrices and rows in 8-bit floating point with a scale for each block of 128, and what is computed with them, in 64 bits, elementary torch."""

import torch

F64 = torch.float64


def block_power(largest: torch.Tensor) -> torch.Tensor:
    """Exponents s of the least powers of two, from 2^-126 on, with largest <= 448 * 2^s."""
    mantissa, exponent = torch.frexp(largest.to(F64))          # largest = mantissa * 2^exponent, mantissa in [0.5, 1); 448 = 0.875 * 2^9
    s = torch.where(mantissa > 0.875, exponent - 8, exponent - 9)
    return torch.where(largest > 0, s, -126).clamp(min=-126)


def e4m3(x: torch.Tensor) -> torch.Tensor:
    """x (64 bits, at most 448) to the nearest e4m3 number, ties to even; not finite: NaN."""
    _, exponent = torch.frexp(x)
    step = torch.exp2((exponent - 1).clamp(min=-6).to(F64) - 3)
    return torch.where(x.isfinite(), torch.round(x / step) * step, torch.nan)


def code_blocks(x: torch.Tensor, rows: int) -> tuple[torch.Tensor, torch.Tensor]:
    """What the codes of x [R, C] in blocks of rows x 128 stand for, and the blocks' exponents s."""
    R, C = x.shape
    nr, nc = -(-R // rows), -(-C // 128)
    padded = torch.zeros((nr * rows, nc * 128), dtype=F64, device=x.device)
    padded[:R, :C] = x.to(F64)
    grid = padded.view(nr, rows, nc, 128)
    s = block_power(torch.where(grid.isfinite(), grid.abs(), 0.0).amax(dim=(1, 3)))
    unit = torch.exp2(s.to(F64))[:, None, :, None]
    return (e4m3(grid / unit) * unit).reshape(nr * rows, nc * 128)[:R, :C], s


def rows(x: torch.Tensor) -> torch.Tensor:
    return code_blocks(x, 1)[0]


def product(x: torch.Tensor, w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x~ w~^T for rows x and the values w (64 bits) of a matrix, and the sums of the terms' magnitudes."""
    coded = rows(x)
    return coded @ w.t(), coded.abs() @ w.abs().t()


def sum_error(k: int) -> float:
    """How far a sum of k products, exact ones, may be off, in terms of the sum of their magnitudes: tensor cores add at least 16 products at once,
    each such step off by at most the last of float32's 24 bits of the largest partial sum (2^-23, whichever way it is cut); and a few
    roundings to nearest where blocks' sums are scaled and slices of K meet."""
    return (k / 16 + 24) * 2.0 ** -23


def gated(sums: torch.Tensor, act: str, limits=None, bias=None) -> torch.Tensor:
    """act(gate) * up of sums whose columns are blocks of 8 gates and their 8 ups."""
    if bias is not None:
        sums = sums + bias.to(F64)
    parts = sums.view(sums.shape[0], -1, 2, 8)
    g, u = parts[:, :, 0].flatten(1), parts[:, :, 1].flatten(1)
    if act == "relu":
        return g.clamp(min=0) * u
    if act == "silu":
        return g * torch.sigmoid(g) * u
    limit, alpha, shift = limits
    g, u = g.clamp(max=limit), u.clamp(-limit, limit)
    return g * torch.sigmoid(alpha * g) * (u + shift)


def gated_error(sums: torch.Tensor, error: torch.Tensor, act: str, limits=None, bias=None) -> torch.Tensor:
    """A bound on the error of ``gated`` for sums that are off by at most ``error``, evaluated in float32: |d/dg silu| <= 1.1, the
    activations themselves to 2^-19 of their value."""
    if bias is not None:
        sums = sums + bias.to(F64)
    parts, errors = sums.abs().view(sums.shape[0], -1, 2, 8), error.view(sums.shape[0], -1, 2, 8)
    g, u = parts[:, :, 0].flatten(1), parts[:, :, 1].flatten(1)
    dg, du = errors[:, :, 0].flatten(1), errors[:, :, 1].flatten(1)
    if act == "bounded":
        limit, alpha, shift = limits
        u = u.clamp(max=limit) + abs(shift)
    value = g * u
    return 1.2 * dg * (u + du) + g * du + 2.0 ** -18 * value + 2.0 ** -120


def code_spread(x: torch.Tensor, error: torch.Tensor) -> torch.Tensor:
    """By how much the coded value of x [M, K] may differ where x is off by up to ``error``: codes are monotone, so the ends bound it; where the
    block's scale may be another one, half a step of either."""
    def ends(s):
        unit = torch.exp2(s.to(F64))[..., None]
        low, high = e4m3((grid - err) / unit) * unit, e4m3(((grid + err) / unit).clamp(-448, 448)) * unit
        return low, high
    M, K = x.shape
    nb = -(-K // 128)
    grid, err = torch.zeros((M, nb * 128), dtype=F64, device=x.device), torch.zeros((M, nb * 128), dtype=F64, device=x.device)
    grid[:, :K], err[:, :K] = x, error
    grid, err = grid.view(M, nb, 128), err.view(M, nb, 128)
    s_low, s_high = block_power((grid.abs() - err).clamp(min=0).amax(-1)), block_power((grid.abs() + err).amax(-1))
    l0, h0 = ends(s_low)
    l1, h1 = ends(s_high)
    here = e4m3(grid / torch.exp2(block_power(grid.abs().amax(-1)).to(F64))[..., None]) * torch.exp2(block_power(grid.abs().amax(-1)).to(F64))[..., None]
    spread = torch.maximum(torch.maximum(h0, h1) - here, here - torch.minimum(l0, l1))
    return spread.clamp(min=0).reshape(M, nb * 128)[:, :K]
