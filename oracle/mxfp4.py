"""MXFP4 and the routed layers over it in 64 bits, with bounds on what another correct implementation may differ by.

Written from the format: 32 columns share a scale 2^(floor(log2 max) - 2), at least 2^-127; an element is the nearest of
0, 0.5, 1, 1.5, 2, 3, 4, 6 (and its negative) times the scale, ties to the even code, larger ones to 6; a block that holds an
infinity or a NaN is NaN."""
from __future__ import annotations

import torch

GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
BF16, FP32 = 2.0 ** -8, 2.0 ** -24  # half a step, relative to the value


def _blocks(t):
    rows, columns = t.shape
    nb = -(-columns // 32)
    return torch.nn.functional.pad(t.double(), (0, 32 * nb - columns)).reshape(rows, nb, 32)


def exponents(t):
    """[rows, blocks]: log2 of the blocks' scales; 128 where a block is NaN."""
    top = _blocks(t).abs().amax(-1)
    e = torch.frexp(torch.where(torch.isfinite(top) & (top > 0), top, 1.0)).exponent - 3
    e = torch.where(top > 0, e.clamp(min=-127), torch.full_like(e, -127))
    return torch.where(torch.isfinite(top), e, torch.full_like(e, 128))


def _numbers(size):
    """Code 0 ... 7 of non-negative sizes in units of the scale."""
    grid = torch.tensor(GRID, dtype=torch.float64, device=size.device)
    below = torch.bucketize(size.contiguous(), grid, right=True).sub(1).clamp(0, 7)
    above = (below + 1).clamp(max=7)
    middle = (grid[below] + grid[above]) / 2
    up = (size > middle) | ((size == middle) & (below % 2 == 1))
    return torch.where(up, above, below)


def codes(t):
    """[rows, blocks, 32] codes 0 ... 15 of finite blocks (0 in NaN blocks), and the exponents."""
    e = exponents(t)
    b = torch.where((e < 128).unsqueeze(-1), _blocks(t), 0.0)
    c = _numbers(b.abs() * torch.exp2(-e.clamp(max=127).double()).unsqueeze(-1))
    return c + 8 * (b < 0), e


def values(t):
    """What `t` stands for once it is quantised, in fp64."""
    c, e = codes(t)
    grid = torch.tensor(GRID, dtype=torch.float64, device=t.device)
    v = grid[c % 8] * torch.where(c >= 8, -1.0, 1.0) * torch.exp2(e.clamp(max=127).double()).unsqueeze(-1)
    v = torch.where((e < 128).unsqueeze(-1), v, float("nan"))
    return v.flatten(1)[:, :t.shape[1]]


def pack(t):
    """codes uint8 [rows, 16 blocks] and scales uint8 [rows, blocks] as the format stores them."""
    c, e = codes(t)
    pair = c.reshape(t.shape[0], -1, 2)
    return (pair[..., 0] + 16 * pair[..., 1]).to(torch.uint8), (e + 127).to(torch.uint8)


def product(a, w):
    """a w^T in fp64, and a bound on the error of fp32 sums of the same exact products: each of the K / 64 instructions rounds the
    running sum and at most six levels of its own, by less than a step (twice FP32) of the magnitudes summed."""
    bound = (a.shape[1] / 64 + 8) * 2 * FP32 * (a.abs() @ w.abs().T)
    return a @ w.T, bound


def stored(value, bound):
    """The bound once the result is rounded to bf16."""
    return bound + BF16 * (value.abs() + bound)


def linear(a, wv, wt, mask):
    """(c, bound) over values a, wv, wt."""
    (v, bv), (t, bt) = product(a, wv), product(a, wt)
    m = mask.unsqueeze(-1)
    c, b = torch.where(m, v, t), torch.where(m, bv, bt)
    return c, stored(c, b)


def _swiglu(a, w1, w3):
    (g, bg), (u, bu) = product(a, w1), product(a, w3)
    s = torch.sigmoid(g)
    h = g * s * u
    # |silu'| < 1.1; the kernels' exp2 and reciprocal are good to a step each, and the exponent's own rounding grows with the gate
    bound = 1.1 * bg * (u.abs() + bu) + (g * s).abs() * bu + (g.abs() + 4) * 2 * FP32 * h.abs()
    return g, u, h, bound


def doubtful(h, bound):
    """How far each element's MXFP4 value may move where h is known to `bound` only: the distance between the values that the two ends
    of its interval take, over all scales that the block may get."""
    lo, hi = _blocks(h.abs() - bound).clamp(min=0), _blocks(h.abs() + bound)
    grid = torch.tensor(GRID, dtype=torch.float64, device=h.device)
    e_lo, e_hi = exponents(lo.amax(-1)[..., None].expand_as(lo).reshape(h.shape[0], -1)), exponents(hi.reshape(h.shape[0], -1))
    ends = []
    for e in (e_lo, e_hi):
        scale = torch.exp2(e.double()).unsqueeze(-1)
        ends += [grid[_numbers(x / scale)] * scale for x in (lo, hi)]
    ends = torch.stack(ends)
    crosses = (_blocks(h).abs() < _blocks(bound)) * ends.amax(0)  # (the sign is in doubt as well)
    return (ends.amax(0) - ends.amin(0) + crosses).reshape(h.shape[0], -1)[:, :h.shape[1]]


def _ffn_rows(a, w1, w2, w3):
    _, _, h, bound = _swiglu(a, w1, w3)
    y, b = product(values(h), w2)
    return y, stored(y, b + doubtful(h, bound) @ w2.abs().T)


def ffn(a, w, mask):
    """(y, bound) over values: a, and w of w1 ... u3."""
    v, t = _ffn_rows(a, w["w1"], w["w2"], w["w3"]), _ffn_rows(a, w["u1"], w["u2"], w["u3"])
    m = mask.unsqueeze(-1)
    return tuple(torch.where(m, x, y) for x, y in zip(v, t))


def linear_grad(g, wv, wt, mask):
    """(da, bound): the rows' gradient over constant weights."""
    return linear(g.double(), wv.T, wt.T, mask)


def _ffn_grad_rows(g, a, w1, w2, w3):
    (gate, bg), (up, bu) = product(a, w1), product(a, w3)
    dh, bdh = product(g.double(), w2.T)
    s = torch.sigmoid(gate)
    d1 = s + gate * s * (1 - s)
    d2 = (s * (1 - s) * (2 + gate * (1 - 2 * s))).abs()  # |silu''|
    dt1, dt3 = dh * up * d1, dh * gate * s
    # dh, gate and up are fp32 sums, dt1 and dt3 are rounded to bf16; to first order, with a tenth more for the products of errors.  The
    # sigmoid's exponential is good to a step, its exponent's rounding grows with the gate, and six operations follow.
    steps = (gate.abs() + 8) * 2 * FP32
    b1 = 1.1 * (bdh * (up * d1).abs() + dh.abs() * (d1.abs() * bu + up.abs() * (d2 * bg + steps * (s + (gate * s * (1 - s)).abs()))) + BF16 * dt1.abs())
    b3 = 1.1 * (bdh * (gate * s).abs() + dh.abs() * (d1.abs() * bg + steps * (gate * s).abs()) + BF16 * dt3.abs())
    (x, bx), (y, by) = product(dt1, w1.T), product(dt3, w3.T)
    da = x + y
    return da, stored(da, bx + by + b1 @ w1.abs() + b3 @ w3.abs())


def ffn_grad(g, a, w, mask):
    v, t = _ffn_grad_rows(g, a, w["w1"], w["w2"], w["w3"]), _ffn_grad_rows(g, a, w["u1"], w["u2"], w["u3"])
    m = mask.unsqueeze(-1)
    return tuple(torch.where(m, x, y) for x, y in zip(v, t))
