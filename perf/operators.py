"""The routed layers over weights held in 4 bits, as a list of cases that can be timed.

A number of an MXFP4 tensor is one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign, times a power of two that 32 neighbours of a
row share.  A service keeps the two weight sets of a mask-routed block in that form, quantises the rows that arrive, and has
matrix cores multiply the 4-bit numbers; fine-tuning with adapters runs the same layers over frozen weights and needs the
gradient of the rows.

    quantise   rows -> MXFP4 -> the values it stands for
    linear     y[m] = Q(x[m]) (W_v if mask[m] else W_t)^T
    ffn        y[m] = Q(silu(Q(x[m]) W1^T) * (Q(x[m]) W3^T)) W2^T, with u1, u2, u3 for the rows of the other modality

with Q the rounding to MXFP4 of runs of 32 columns.  `train` cases add the gradient of x, with both roundings passed over
(straight-through) and the weights constant.

    listed()          the fixed cases
    draw(rng)         one more case from the ranges that the fixed ones stand for
    prepare(case, s)  inputs and weights on the GPU, made from the seed s
    run(state)        one pass: in elementary torch operations, or (own) through the package's entry points
    exact(case, s)    the same in 64 bits
    work(case)        bytes and operations that one pass cannot do without
"""
from __future__ import annotations

import random

import torch

own = False

# op, train: as above.  k, n: input and output features of the linear layer, or model width and intermediate size of the
# feed-forward layer; k columns of the quantised rows.  mask: "spans" (runs of image tokens between runs of text), "mixed" (each
# row on its own, as in a decode batch of unrelated sequences), "visual" / "text" (one modality only).
_LISTED = (
    # The rows of a small decode batch: nothing but latency.
    dict(name="quantise_8", op="quantise", dtype="bfloat16", m=8, k=4096),
    # The rows of a batch of long prompts, or a weight: bandwidth.
    dict(name="quantise_32768", op="quantise", dtype="bfloat16", m=32768, k=4096),
    # One token through a projection.
    dict(name="linear_decode_1", op="linear", train=False, m=1, k=1024, n=1024, mask="text"),
    # A prompt of one sequence through a projection.
    dict(name="linear_fwd_2048", op="linear", train=False, m=2048, k=1024, n=1024, mask="spans"),
    # Extents that are no multiples of a tile, nor of 32 along the quantised axis; odd row count.
    dict(name="linear_fwd_ragged", op="linear", train=False, m=3001, k=2056, n=1544, mask="spans"),
    # Adapter training over a frozen projection, rows of both modalities fully interleaved.
    dict(name="linear_train_8192", op="linear", train=True, m=8192, k=1024, n=1024, mask="mixed"),
    # Single-stream decode of a large layer: one modality's weights are read from memory once.
    dict(name="ffn_decode_1", op="ffn", train=False, m=1, k=4096, n=14336, mask="text"),
    # A decode batch of sequences in both modalities, odd size.
    dict(name="ffn_decode_27", op="ffn", train=False, m=27, k=4096, n=14336, mask="mixed"),
    # A short prompt: too many rows to be bound by the weights' bytes alone, too few to fill the chip with large tiles.
    dict(name="ffn_prefill_300", op="ffn", train=False, m=300, k=4096, n=14336, mask="spans"),
    # An ordinary prompt with an image in it, odd size.
    dict(name="ffn_prefill_1411", op="ffn", train=False, m=1411, k=4096, n=14336, mask="spans"),
    # A batch of long prompts through a large layer.
    dict(name="ffn_prefill_32768", op="ffn", train=False, m=32768, k=4096, n=14336, mask="spans"),
    # Adapter training over a frozen large layer.
    dict(name="ffn_train_4096", op="ffn", train=True, m=4096, k=4096, n=14336, mask="spans"),
)

_MAX_FLOPS = 2 * 32768 * 4096 * 14336 * 3
_MAX_VALUES = 32768 * 4096
_IMAGE_TOKENS = 576


def listed():
    return [dict(c) for c in _LISTED]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(lo * (hi / lo) ** rng.random())))


def _extent(rng, lo, hi):
    """A layer's extent: mostly a multiple of 64, as models have them, else a multiple of 8."""
    unit = 64 if rng.random() < 0.75 else 8
    return max(lo, _log_int(rng, lo, hi) // unit * unit)


def draw(rng: random.Random):
    kind = rng.choice(("quantise", "linear_fwd", "linear_train", "ffn_decode", "ffn_prefill", "ffn_train"))
    while True:
        if kind == "quantise":
            case = dict(op="quantise", dtype=rng.choice(("bfloat16", "bfloat16", "float16", "float32")),
                        m=_log_int(rng, 1, 32768), k=_log_int(rng, 512, 16384) if rng.random() < 0.25 else _extent(rng, 512, 16384))
            if case["m"] * case["k"] * (2 if case["dtype"] == "float32" else 1) <= _MAX_VALUES:
                return case
            continue
        if kind.startswith("linear"):
            m = _log_int(rng, 65, 16384) if kind == "linear_train" else _log_int(rng, 1, 32768)
            k, n = _extent(rng, 512, 8192), _extent(rng, 512, 8192)
        else:
            k = _extent(rng, 1024, 8192)
            n = int(k * rng.uniform(2.0, 3.5)) // 64 * 64 if k % 64 == 0 else int(k * rng.uniform(2.0, 3.5)) // 8 * 8
            m = _log_int(rng, *{"ffn_decode": (1, 64), "ffn_prefill": (65, 32768), "ffn_train": (65, 8192)}[kind])
        mask = rng.choice(("mixed", "mixed", "visual", "text") if m <= 64 else ("spans", "spans", "mixed", "visual", "text"))
        case = dict(op=kind.split("_")[0], train=kind.endswith("train"), m=m, k=k, n=n,
                    mask=mask if m > 1 else rng.choice(("visual", "text")))
        if work(case)["flops"] <= _MAX_FLOPS:
            return case


def _mask(case, seed):
    m, kind = case["m"], case["mask"]
    rng = random.Random(seed)
    if kind in ("visual", "text"):
        return torch.full((m,), kind == "visual")
    if kind == "mixed":
        return torch.rand(m, generator=torch.Generator().manual_seed(seed)) < 0.5
    span = min(_IMAGE_TOKENS, max(1, m // 4))  # a short prompt holds a smaller image
    mask = torch.zeros(m, dtype=torch.bool)
    at = rng.randrange(span)
    while at < m:
        mask[at:at + span] = True
        at += span + rng.randrange(span // 2, span + span // 2 + 1)
    return mask


def _names(case):
    """The weights and their shapes, as nn.Linear holds them: [out features, in features]."""
    k, n = case["k"], case["n"]
    if case["op"] == "linear":
        return (("v", (n, k)), ("t", (n, k)))
    return tuple((s + i, (k, n) if i == "2" else (n, k)) for s in "wu" for i in "123")


def _normal(gen, rows, cols, std):
    return torch.randn((rows, cols), generator=gen, device="cuda", dtype=torch.float32).mul_(std).bfloat16()


def _inputs(case, seed):
    """x, the upstream gradient and the weights before they are quantised: all in bf16, the quantised rows in the case's type."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    m, k = case["m"], case["k"]
    x = _normal(gen, m, k, 1.0)                       # behind a normalisation layer
    x *= 1 + 15 * (torch.rand(k, generator=gen, device="cuda") < 0.01).to(x.dtype)  # ... some of whose channels are large
    if case["op"] == "quantise":
        return x.to(getattr(torch, case["dtype"])), None, {}
    weights = {name: _normal(gen, *shape, 0.02) for name, shape in _names(case)}
    out = case["n"] if case["op"] == "linear" else k
    return x, _normal(gen, m, out, 1.0) if case["train"] else None, weights


# ---- the plain form: elementary operations in 32 bits -------------------------------------------------------------------------

def _parts(t):
    """[rows, columns] in fp32 -> the numbers -6 ... 6 of its MXFP4 form [rows, blocks, 32] and the blocks' exponents [rows, blocks]."""
    rows, columns = t.shape
    blocks = -(-columns // 32)
    t = torch.nn.functional.pad(t, (0, blocks * 32 - columns)).view(rows, blocks, 32)
    top = t.abs().amax(-1)
    # the largest power of two not above the block's largest magnitude, over the largest of the format, 4
    exponent = torch.where(top > 0, torch.frexp(top).exponent - 3, -127).clamp_(-127, 127)
    t = torch.ldexp(t, -exponent.unsqueeze(-1))
    size = t.abs()
    step = torch.where(size < 2, 0.5, torch.where(size < 4, 1.0, 2.0))
    return torch.copysign((torch.round(size / step) * step).clamp_(max=6.0), t), exponent  # (round: ties to even)


def _values(numbers, exponent, columns):
    return torch.ldexp(numbers, exponent.unsqueeze(-1)).view(numbers.shape[0], -1)[:, :columns]


def _rounded(t):
    return _values(*_parts(t), t.shape[1])


def _pack(numbers, exponent):
    """As they are kept: two numbers to a byte, the even column in the low half, and a byte of exponent + 127 for 32 columns."""
    size = numbers.abs()
    code = torch.where(size < 2, size * 2, torch.where(size < 4, size + 2, size / 2 + 4)).to(torch.uint8)
    code = (code | (torch.signbit(numbers).to(torch.uint8) << 3)).view(numbers.shape[0], -1, 2)
    return code[..., 0] | (code[..., 1] << 4), (exponent + 127).to(torch.uint8)


def _unpack(codes, scales, columns):
    code = torch.stack((codes & 15, codes >> 4), -1).view(codes.shape[0], -1, 32)
    sizes = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float32, device=codes.device)
    numbers = sizes[(code & 7).long()]
    return _values(torch.where(code > 7, -numbers, numbers), scales.int() - 127, columns)


def _by_modality(state, first, second):
    """Rows of both modalities through their own function."""
    parts = [(rows, f(rows)) for rows, f in ((state["rows_v"], first), (state["rows_t"], second)) if rows.numel()]
    outs = []
    for at in zip(*(p for _, p in parts)):
        out = at[0].new_empty(state["x"].shape[0], at[0].shape[1])
        for (rows, _), part in zip(parts, at):
            out[rows] = part
        outs.append(out.bfloat16())
    return tuple(outs) if len(outs) > 1 else outs[0]


def _plain(state):
    x = state["x"].float()
    if state["op"] == "quantise":
        return _rounded(x).to(state["x"].dtype)
    weight = {name: _unpack(*parts, columns) for name, (*parts, columns) in state["kept"].items()}
    x, train = _rounded(x), state["train"]

    def linear(w):
        def rows_of(rows):
            return (x[rows] @ w.T, *((state["grad"][rows].float() @ w,) if train else ()))
        return rows_of

    def ffn(w1, w2, w3):
        def rows_of(rows):
            gate, up = x[rows] @ w1.T, x[rows] @ w3.T
            s = torch.sigmoid(gate)
            y = _rounded(gate * s * up) @ w2.T
            if not train:
                return (y,)
            dh = state["grad"][rows].float() @ w2
            return y, (dh * up * (s + gate * s * (1 - s))) @ w1 + (dh * gate * s) @ w3
        return rows_of

    if state["op"] == "linear":
        return _by_modality(state, linear(weight["v"]), linear(weight["t"]))
    return _by_modality(state, ffn(weight["w1"], weight["w2"], weight["w3"]), ffn(weight["u1"], weight["u2"], weight["u3"]))


# ---- the package's operators ---------------------------------------------------------------------------------------------------

def _own(state):
    import ffn_kernel_amd as F

    if state["op"] == "quantise":
        return F.mxfp4_dequantise(F.mxfp4_quantise(state["x"]), state["x"].dtype)
    op = F.MaskedLinearMXFP4 if state["op"] == "linear" else F.MaskedFFNMXFP4
    if not state["train"]:
        with torch.no_grad():
            return op.apply(state["x"], *state["held"], state["mask"])
    y = op.apply(state["x"], *state["held"], state["mask"])
    return y.detach(), torch.autograd.grad(y, state["x"], state["grad"])[0]


def prepare(case, seed):
    x, grad, weights = _inputs(case, seed)
    state = dict(op=case["op"], x=x)
    if case["op"] == "quantise":
        return state
    state.update(train=case["train"], x=x.requires_grad_(case["train"]), grad=grad, mask=_mask(case, seed).cuda())
    state["rows_v"], state["rows_t"] = state["mask"].nonzero().view(-1), (~state["mask"]).nonzero().view(-1)
    # A checkpoint of 4-bit weights: codes, scales, columns.
    state["kept"] = {name: (*_pack(*_parts(w.float())), w.shape[1]) for name, w in weights.items()}
    if own:  # the handles that a program makes of them once
        import ffn_kernel_amd as F
        state["held"] = [F.MXFP4.from_parts(*parts) for parts in state["kept"].values()]
    return state


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return _plain(state)


# ---- the definition in 64 bits -------------------------------------------------------------------------------------------------

_GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _nearest(t):
    """[rows, columns] in fp64 -> the MXFP4 value of each: the nearest point of the block's grid, halfway ones to the even code."""
    rows, columns = t.shape
    out = torch.empty_like(t)
    grid = torch.tensor(_GRID, dtype=torch.float64, device=t.device)
    middle = (grid[1:] + grid[:-1]) / 2
    whole = columns // 32 * 32
    for part, at in ((t[:, :whole].reshape(-1, 32), slice(0, whole)), (t[:, whole:], slice(whole, columns))):
        if part.numel() == 0:
            continue
        top = part.abs().amax(-1, keepdim=True)
        scale = torch.exp2(torch.floor(torch.log2(torch.where(top > 0, top, 1.0))) - 2)
        scale = torch.where(scale * 8 <= top, scale * 2, torch.where(scale * 4 > top, scale / 2, scale))  # (log2 next to a power of two)
        scale = torch.where(top > 0, scale.clamp(min=2.0 ** -127), 2.0 ** -127)
        size = part.abs() / scale
        code = torch.bucketize(size, middle)           # points whose upper middle is below the size: ties stay below
        tie = (code < 7) & (size == middle[code.clamp(max=6)]) & (code % 2 == 1)
        out[:, at] = (torch.sign(part) * grid[code + tie] * scale).view(rows, -1)
    return out


def exact(case, seed):
    x, grad, weights = _inputs(case, seed)
    if case["op"] == "quantise":
        return _nearest(x.double())
    mask, train = _mask(case, seed).cuda(), case["train"]
    x = _nearest(x.double())
    results = [torch.empty(case["m"], case["n"] if case["op"] == "linear" else case["k"], dtype=torch.float64, device="cuda")]
    if train:
        results.append(torch.empty_like(x))
    for rows, first in ((mask, 0), (~mask, 1)):
        if not bool(rows.any()):
            continue
        mine = list(weights.values())
        mine = [_nearest(w.double()) for w in (mine[first:first + 1] if case["op"] == "linear" else mine[3 * first:3 * first + 3])]
        g = grad[rows].double() if train else None
        if case["op"] == "linear":
            results[0][rows] = x[rows] @ mine[0].T
            if train:
                results[1][rows] = g @ mine[0]
            continue
        a, b = x[rows] @ mine[0].T, x[rows] @ mine[2].T
        silu = a / (1 + torch.exp(-a))
        results[0][rows] = _nearest(silu * b) @ mine[1].T
        if train:
            dh, s = g @ mine[1], 1 / (1 + torch.exp(-a))
            results[1][rows] = (dh * b * s * (1 + a * (1 - s))) @ mine[0] + (dh * silu) @ mine[2]
    return tuple(results) if train else results[0]


def work(case):
    m, k = case["m"], case["k"]

    def held(values):
        return values * 17 / 32                        # a byte for two numbers, and one for 32

    if case["op"] == "quantise":                       # rows in, the 4-bit tensor and its values out
        size = 4 if case["dtype"] == "float32" else 2
        return {"bytes": 2 * size * m * k + held(m * k), "flops": 0}
    n, linear = case["n"], case["op"] == "linear"
    present = 1 if case["mask"] in ("visual", "text") else 2
    per_set = k * n if linear else 3 * k * n
    out = n if linear else k
    flops = 2 * m * per_set
    nbytes = held(present * per_set) + 2 * (m * k + m * out) + m
    if case["train"]:
        flops *= 2                                     # the gradient of x
        nbytes += 2 * (m * out + m * k)                # upstream in, dx out
    return {"bytes": nbytes, "flops": flops}
