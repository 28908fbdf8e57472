"""MXFP4 operators on the GPU against the 64-bit oracle, element by element within its error bounds: tail blocks, odd extents, row
counts either side of every path, one modality alone, strides, infinities and NaN, both forms of the rows, gradients, graphs, modules."""
import copy

import pytest
import torch

import ffn_kernel_amd as F
from ffn_kernel_amd import _lib
from oracle import mxfp4 as ref
from tests.helpers import note

pytestmark = pytest.mark.gpu
FFN = ("w1", "w2", "w3", "u1", "u2", "u3")


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rows(m, k, seed, dtype=torch.bfloat16):
    """Rows with some large channels and some whole blocks of zeros."""
    g = gen(seed)
    t = torch.randn(m, k, generator=g, device="cuda")
    t *= 1 + 15 * (torch.rand(k, generator=g, device="cuda") < 0.02)
    if k > 64:
        t[::3, 32:64] = 0
    return t.to(dtype)


def weight(n, k, seed, std=0.05):
    return (torch.randn(n, k, generator=gen(seed), device="cuda") * std).bfloat16()


def a_mask(m, kind, seed=0):
    if kind in ("visual", "text"):
        return torch.full((m,), kind == "visual", device="cuda")
    return torch.rand(m, generator=gen(seed + 77), device="cuda") < 0.4


def within(got, value, bound, what):
    got = got.double()
    assert got.shape == value.shape, what
    assert torch.equal(got.isnan(), value.isnan()), f"{what}: NaN elsewhere"
    excess = ((got - value).abs() / (bound + 1e-300)).nan_to_num(0.0)
    at = excess.argmax().item() if excess.numel() else 0
    assert excess.numel() == 0 or excess.max().item() <= 1.0, f"{what}: {excess.max().item():.3f} of the bound at {at}: {got.flatten()[at].item()} for {value.flatten()[at].item()}"


# ---- quantisation: codes, scales and values are exact -----------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("m,k", [(1, 1), (1, 32), (2, 31), (3, 33), (5, 100), (8, 4096), (7, 1544), (65, 2056), (1, 40000), (300, 8), (2500, 4104), (1030, 8192)])
def test_quantise_is_exact(m, k, dtype):
    note(f"quantise {m}x{k} {dtype}")
    t = rows(m, k, m + k, dtype)
    if k > 8:  # values on the borders of the grid, both zeros, tiny ones
        t[0, :8] = torch.tensor([6.0, 0.25, -0.75, 2.5, -5.0, 1.25, -0.0, 2.0 ** -20], dtype=dtype)
    q = F.mxfp4_quantise(t)
    codes, scales = ref.pack(t)
    nb = scales.shape[1]
    held = q.scales.transpose(0, 1).reshape(m, -1)
    assert torch.equal(held[:, :nb], scales) and not held[:, nb:].any() and torch.equal(q.parts()[1], scales)
    sign = lambda c: torch.where((c & 7) == 0, c & 7, c)  # (a zero's sign is free)
    assert torch.equal(sign(q.codes & 15), sign(codes & 15)) and torch.equal(sign(q.codes >> 4), sign(codes >> 4))
    for out in (torch.bfloat16, torch.float16, torch.float32):
        assert torch.equal(F.mxfp4_dequantise(q, out), ref.values(t).to(out))
    again = F.MXFP4.from_parts(codes[:, :(k + 1) // 2], scales, k)
    assert torch.equal(again.dequantise(torch.float32), q.dequantise(torch.float32)) and again.shape == (m, k)


def test_quantise_extremes():
    note("quantise extremes")
    t = torch.zeros(6, 96, device="cuda")
    t[0, 5], t[1, 40], t[2, 70] = float("inf"), float("nan"), -float("inf")
    t[3, :3] = torch.tensor([2.0 ** 127, -(2.0 ** 127) * 1.99, 2.0 ** 125])
    t[4, :3] = torch.tensor([2.0 ** -126, -(2.0 ** -127), 2.0 ** -149])
    t[5, 32:35] = torch.tensor([2.0 ** -124, 1.5 * 2.0 ** -126, -(2.0 ** -125)])
    q = F.mxfp4_quantise(t)
    assert torch.equal(q.parts()[1], ref.pack(t)[1])
    v, w = F.mxfp4_dequantise(q, torch.float32), ref.values(t).float()
    assert torch.equal(v.isnan(), w.isnan()) and torch.equal(v.nan_to_num(0.0), w.nan_to_num(0.0))
    assert v[0, :32].isnan().all() and not v[0, 32:].isnan().any()


def test_quantise_reads_rows_as_they_lie():
    note("quantise strides")
    big = rows(40, 300, 5)
    for view in (big[:, :200], big[::2], big[3:, 7:207], big.T, big[:1].expand(9, 300), big[:, ::3], big[:, :0], big[:0]):
        q = F.mxfp4_quantise(view)
        assert q.shape == tuple(view.shape) and torch.equal(q.dequantise(torch.float32), ref.values(view).float())
    p = torch.nn.Parameter(big.clone())
    assert not F.mxfp4_quantise(p).dequantise().requires_grad


# ---- the linear layer -----------------------------------------------------------------------------------------------------------

def linear_case(m, k, n, kind, seed=1):
    x, wv, wt, mask = rows(m, k, seed), weight(n, k, seed + 1), weight(n, k, seed + 2), a_mask(m, kind, seed)
    return x, F.mxfp4_quantise(wv), F.mxfp4_quantise(wt), mask, (ref.values(x), ref.values(wv), ref.values(wt))


@pytest.mark.parametrize("kind", ["mixed", "visual", "text"])
@pytest.mark.parametrize("m,k,n", [(1, 1, 1), (1, 32, 16), (2, 33, 7), (3, 4096, 130), (8, 1024, 1024), (15, 520, 33), (16, 512, 64), (17, 544, 31), (27, 2056, 200),
                                   (33, 100, 48), (48, 1000, 96), (49, 7168, 65), (64, 1544, 257), (64, 256, 512), (65, 40, 24), (65, 1, 3), (66, 256, 31),
                                   (100, 264, 129), (127, 512, 128), (130, 1544, 260), (257, 768, 384), (300, 96, 1030), (300, 8192, 256), (513, 1032, 520)])
def test_linear_forward(m, k, n, kind):
    note(f"linear {m}x{k}->{n} {kind}")
    x, qv, qt, mask, (a, wv, wt) = linear_case(m, k, n, kind)
    value, bound = ref.linear(a, wv, wt, mask)
    y = F.MaskedLinearMXFP4.apply(x, qv, qt, mask)
    within(y, value, bound, "rows in bf16")
    within(F.masked_linear_mxfp4_forward(F.mxfp4_quantise(x), qv, qt, mask), value, bound, "rows in MXFP4")
    assert torch.equal(y, F.MaskedLinearMXFP4.apply(x, qv, qt, mask)), "the same call twice"


@pytest.mark.parametrize("m,k,n,kind", [(2100, 1024, 4160, "mixed"), (4097, 296, 4100, "mixed"), (3000, 520, 8200, "visual"), (2048, 768, 6144, "text"), (70000, 64, 72, "mixed")])
def test_linear_forward_on_large_tiles(m, k, n, kind):
    note(f"linear large {m}x{k}->{n} {kind}")
    x, qv, qt, mask, (a, wv, wt) = linear_case(m, k, n, kind)
    value, bound = ref.linear(a, wv, wt, mask)
    within(F.masked_linear_mxfp4_forward(x, qv, qt, mask), value, bound, "rows in bf16")
    within(F.masked_linear_mxfp4_forward(F.mxfp4_quantise(x), qv, qt, mask), value, bound, "rows in MXFP4")


@pytest.mark.parametrize("m,k,n,kind", [(2048, 64, 4096, "mixed"), (2048, 100, 4098, "mixed"), (1030, 64, 2060, "text"), (65, 14336, 64, "mixed"), (49, 5120, 68, "visual"),
                                        (66, 8190, 130, "mixed"), (66, 4100, 66, "mixed"), (150, 8200, 1284, "mixed"), (3000, 7200, 64, "mixed"), (300, 14330, 36, "text"),
                                        (8192, 4096, 60, "mixed"), (128, 14336, 704, "mixed")])
def test_linear_forward_on_every_tile_and_number_of_k_ranges(m, k, n, kind):
    note(f"linear plan {m}x{k}->{n} {kind}")
    x, qv, qt, mask, (a, wv, wt) = linear_case(m, k, n, kind)
    value, bound = ref.linear(a, wv, wt, mask)
    within(F.masked_linear_mxfp4_forward(x, qv, qt, mask), value, bound, "rows in bf16")


def test_linear_rows_that_32_bits_do_not_reach():
    """Codes of more than 4 GiB: the rows are quantised in routed order; rows in MXFP4 are refused."""
    note("linear 17 GB of rows")
    k, n, times = 8192, 40, 257
    x, qv, qt, _, (a, wv, wt) = linear_case(4096, k, n, "mixed")
    many = x.repeat(times, 1)
    m = many.shape[0]
    assert m * k // 2 > 1 << 32
    mask = torch.rand(m, generator=gen(5), device="cuda") < 0.5
    y = F.masked_linear_mxfp4_forward(many, qv, qt, mask).view(times, 4096, n)
    visual = ref.linear(a, wv, wt, torch.ones(4096, dtype=torch.bool, device="cuda"))
    text = ref.linear(a, wv, wt, torch.zeros(4096, dtype=torch.bool, device="cuda"))
    for i in (*range(0, times, 32), times - 1):
        value, bound = (torch.where(mask.view(times, 4096, 1)[i], v, t) for v, t in zip(visual, text))
        within(y[i], value, bound, f"rows from {4096 * i}")
    held = F.mxfp4_quantise(many)
    assert torch.equal(held.codes[-4096:], F.mxfp4_quantise(x).codes)
    with pytest.raises(ValueError, match="32-bit offsets"):
        F.masked_linear_mxfp4_forward(held, qv, qt, mask)


@pytest.mark.parametrize("m", [5, 64, 65, 300])
def test_linear_infinities_stay_in_their_rows(m):
    note(f"linear inf / nan {m}")
    x, qv, qt, mask, (_, wv, wt) = linear_case(m, 512, 96, "mixed")
    x[1, 300], x[m - 1, 2] = float("inf"), float("nan")
    value, bound = ref.linear(ref.values(x).nan_to_num(0.0), wv, wt, mask)
    value[1], value[m - 1] = float("nan"), float("nan")
    within(F.masked_linear_mxfp4_forward(x, qv, qt, mask), value, bound, "rows with an infinity or a NaN are NaN, the others not")


def test_linear_infinite_weights_reach_their_modality_only():
    note("linear inf weights")
    for m in (20, 200):
        x, _, qt, mask, (a, wv, wt) = linear_case(m, 256, 64, "mixed")
        bad = weight(64, 256, 2)
        bad[5, 7] = float("inf")
        value, bound = ref.linear(a, ref.values(bad).nan_to_num(0.0), wt, mask)
        value[mask, 5] = float("nan")
        within(F.masked_linear_mxfp4_forward(x, F.mxfp4_quantise(bad), qt, mask), value, bound, "column 5 of the visual rows")


@pytest.mark.parametrize("m", [9, 100])
def test_linear_views_routing_and_empty_calls(m):
    note(f"linear views {m}")
    wide, qv, qt, mask, (a, wv, wt) = linear_case(m, 300, 72, "mixed")
    x = wide[:, 4:260]
    qv, qt = F.mxfp4_quantise(weight(72, 256, 8)), F.mxfp4_quantise(weight(72, 256, 9))
    value, bound = ref.linear(ref.values(x), qv.dequantise(torch.float32).double(), qt.dequantise(torch.float32).double(), mask)
    strided = torch.zeros(m, 3, dtype=torch.bool, device="cuda")
    strided[:, 1] = mask
    within(F.masked_linear_mxfp4_forward(x, qv, qt, strided[:, 1]), value, bound, "views")
    within(F.masked_linear_mxfp4_forward(x, qv, qt, mask, routing=F.route(mask)), value, bound, "a partition made earlier")
    within(F.masked_linear_mxfp4_forward(x[:1].expand(m, 256), qv, qt, mask), *ref.linear(ref.values(x[:1].expand(m, 256)), qv.dequantise(torch.float32).double(), qt.dequantise(torch.float32).double(), mask), "one row repeated")
    assert F.masked_linear_mxfp4_forward(x[:0], qv, qt, mask[:0]).shape == (0, 72)
    with pytest.raises(ValueError, match="routing"):
        F.masked_linear_mxfp4_forward(x, qv, qt, mask, routing=F.route(mask[:-1]))


def test_refusals_on_the_gpu():
    note("refusals")
    x, qv, qt, mask, _ = linear_case(8, 64, 32, "mixed")
    other, up = F.mxfp4_quantise(weight(32, 96, 4)), F.mxfp4_quantise(weight(96, 64, 4))
    for call in (lambda: F.MaskedLinearMXFP4.apply(x, qv, other, mask), lambda: F.MaskedLinearMXFP4.apply(x, other, other, mask),
                 lambda: F.MaskedLinearMXFP4.apply(x.float(), qv, qt, mask), lambda: F.MaskedLinearMXFP4.apply(x[0], qv, qt, mask),
                 lambda: F.MaskedLinearMXFP4.apply(x, qv, qt, mask[:-1]), lambda: F.MaskedLinearMXFP4.apply(x, qv, qt, mask.int()),
                 lambda: F.MaskedLinearMXFP4.apply(x, qv, qt, mask.cpu()), lambda: F.MaskedLinearMXFP4.apply(x.cpu(), qv, qt, mask),
                 lambda: F.MaskedFFNMXFP4.apply(x, up, up, up, up, up, up, mask), lambda: F.mxfp4_dequantise(qv, torch.float64),
                 lambda: F.MXFP4(qv.codes[:, :16], qv.scales, 32), lambda: F.MXFP4(qv.codes, qv.scales, 65), lambda: F.MXFP4(qv.codes[1:], qv.scales, 64),
                 lambda: F.masked_linear_mxfp4_backward(x, qv, qt, mask),
                 lambda: F.MaskedLinearMXFP4.apply(x.clone().requires_grad_(), qv, qt, mask)):  # 32 output features: no backward for them
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        F.MaskedLinearMXFP4.apply(x, qv, weight(32, 64, 1), mask)


# ---- the feed-forward layer -----------------------------------------------------------------------------------------------------

def ffn_case(m, d, h, kind, seed=11):
    w = {n: weight(d, h, seed + i, 1.2 / h ** 0.5) if n[1] == "2" else weight(h, d, seed + i, 1.2 / d ** 0.5) for i, n in enumerate(FFN)}
    x = rows(m, d, seed + 9)
    return x, [F.mxfp4_quantise(w[n]) for n in FFN], a_mask(m, kind, seed), ref.values(x), {n: ref.values(w[n]) for n in FFN}


@pytest.mark.parametrize("kind", ["mixed", "visual", "text"])
@pytest.mark.parametrize("m,d,h", [(1, 32, 32), (1, 1024, 2048), (2, 40, 33), (5, 512, 520), (16, 256, 1000), (17, 1000, 1056), (31, 1032, 2000), (48, 544, 96), (64, 768, 1544),
                                   (64, 31, 65), (65, 64, 40), (66, 33, 31), (100, 512, 1032), (129, 520, 776), (300, 1024, 2816), (515, 264, 520)])
def test_ffn_forward(m, d, h, kind):
    note(f"ffn {m} {d} {h} {kind}")
    x, q, mask, a, w = ffn_case(m, d, h, kind)
    value, bound = ref.ffn(a, w, mask)
    y = F.MaskedFFNMXFP4.apply(x, *q, mask)
    within(y, value, bound, "rows in bf16")
    within(F.masked_ffn_mxfp4_forward(F.mxfp4_quantise(x), *q, mask), value, bound, "rows in MXFP4")
    assert torch.equal(y, F.MaskedFFNMXFP4.apply(x, *q, mask)), "the same call twice"


@pytest.mark.parametrize("m,d,h,kind", [(2100, 512, 4160, "mixed"), (3000, 264, 4104, "visual"), (4500, 1024, 2080, "mixed")])
def test_ffn_forward_on_large_tiles(m, d, h, kind):
    note(f"ffn large {m} {d} {h} {kind}")
    x, q, mask, a, w = ffn_case(m, d, h, kind)
    value, bound = ref.ffn(a, w, mask)
    within(F.masked_ffn_mxfp4_forward(x, *q, mask), value, bound, "rows in bf16")
    y, pre = F.masked_ffn_mxfp4_forward(x, *q, mask, save_pre=True)
    within(y, value, bound, "with the projections kept")


@pytest.mark.parametrize("m", [7, 64, 65, 200])
def test_ffn_keeps_its_projections_in_routed_order(m):
    note(f"ffn pre {m}")
    d, h = 96, 136
    x, q, mask, a, w = ffn_case(m, d, h, "mixed")
    y, pre = F.masked_ffn_mxfp4_forward(x, *q, mask, save_pre=True)
    order = torch.cat((mask.nonzero().view(-1), (~mask).nonzero().view(-1)))
    for half, names in ((0, ("w1", "u1")), (h, ("w3", "u3"))):
        (v, bv), (t, bt) = (ref.product(a, w[n]) for n in names)
        value, bound = torch.where(mask[:, None], v, t), torch.where(mask[:, None], bv, bt)
        within(pre[:, half:half + h], value[order], bound[order], f"projection at {half}")
    within(y, *ref.ffn(a, w, mask), "result")


def test_ffn_infinities_stay_in_their_rows():
    note("ffn inf")
    for m in (6, 90):
        x, q, mask, _, w = ffn_case(m, 256, 320, "mixed")
        x[2, 17] = float("inf")
        value, bound = ref.ffn(ref.values(x).nan_to_num(0.0), w, mask)
        value[2] = float("nan")
        within(F.masked_ffn_mxfp4_forward(x, *q, mask), value, bound, "row 2 is NaN, the others not")


@pytest.mark.parametrize("m,d,h,kind", [(256, 64, 14336, "mixed"), (300, 72, 14340, "mixed"), (100, 64, 11008, "mixed"), (130, 136, 8200, "visual"), (65, 264, 1000, "mixed"),
                                        (48, 1024, 1032, "mixed"), (49, 1024, 1032, "mixed"), (56, 256, 8192, "text")])
def test_ffn_forward_on_every_tile(m, d, h, kind):
    note(f"ffn plan {m} {d} {h} {kind}")
    x, q, mask, a, w = ffn_case(m, d, h, kind)
    within(F.masked_ffn_mxfp4_forward(x, *q, mask), *ref.ffn(a, w, mask), "rows in bf16")


# ---- gradients ----------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("kind", ["mixed", "visual", "text"])
@pytest.mark.parametrize("m,k,n", [(1, 8, 64), (5, 264, 128), (64, 512, 136), (65, 32, 64), (100, 1032, 200), (300, 256, 520), (2050, 1024, 1024)])
def test_linear_gradient(m, k, n, kind):
    note(f"linear grad {m}x{k}->{n} {kind}")
    x, qv, qt, mask, (a, wv, wt) = linear_case(m, k, n, kind)
    g = rows(m, n, 3)
    x.requires_grad_()
    y = F.MaskedLinearMXFP4.apply(x, qv, qt, mask)
    within(y.detach(), *ref.linear(a, wv, wt, mask), "forward")
    da, = torch.autograd.grad(y, x, g)
    value, bound = ref.linear_grad(g.double(), wv, wt, mask)
    within(da, value, bound, "gradient")
    wide = torch.empty(m, n + 3, device="cuda", dtype=torch.bfloat16)
    wide[:, 1:n + 1] = g
    within(F.masked_linear_mxfp4_backward(wide[:, 1:n + 1], qv, qt, mask), value, bound, "an upstream gradient off 16 bytes")


@pytest.mark.parametrize("kind", ["mixed", "visual", "text"])
@pytest.mark.parametrize("m,d,h", [(1, 64, 64), (7, 136, 72), (64, 256, 520), (65, 128, 200), (130, 264, 512), (300, 512, 1032), (1100, 1024, 2056)])
def test_ffn_gradient(m, d, h, kind):
    note(f"ffn grad {m} {d} {h} {kind}")
    x, q, mask, a, w = ffn_case(m, d, h, kind)
    g = rows(m, d, 3)
    x.requires_grad_()
    y = F.MaskedFFNMXFP4.apply(x, *q, mask)
    within(y.detach(), *ref.ffn(a, w, mask), "forward")
    da, = torch.autograd.grad(y, x, g)
    within(da, *ref.ffn_grad(g, a, w, mask), "gradient")
    with torch.no_grad():
        assert not F.MaskedFFNMXFP4.apply(x, *q, mask).requires_grad


def test_rows_in_mxfp4_carry_no_gradient():
    note("no gradient")
    x, q, mask, _, _ = ffn_case(70, 64, 64, "mixed")
    y = F.MaskedFFNMXFP4.apply(F.mxfp4_quantise(x.requires_grad_()), *q, mask)
    assert not y.requires_grad


@pytest.mark.parametrize("m", [1, 20, 64, 65, 200, 700])
def test_calls_from_c_and_from_python_answer_alike(m, monkeypatch):
    note(f"call.cpp {m}")
    from ffn_kernel_amd import mxfp4

    class Nothing:
        def __getattr__(self, name):
            return lambda *a: NotImplemented

    d, h = 264, 520
    x, q, mask, _, _ = ffn_case(m, d, h, "mixed")
    g = rows(m, d, 3)

    def everything():
        held = F.mxfp4_quantise(x)
        out = [*held.parts(), F.mxfp4_dequantise(held, torch.float16)]
        out.append(F.masked_linear_mxfp4_forward(x, q[0], q[3], mask))
        out.append(F.masked_linear_mxfp4_forward(held, q[0], q[3], mask))
        out.append(F.masked_linear_mxfp4_backward(out[-1], q[0], q[3], mask))
        out += F.masked_ffn_mxfp4_forward(x, *q, mask, save_pre=True)
        out += [F.masked_ffn_mxfp4_forward(x, *q, mask), F.masked_ffn_mxfp4_forward(held, *q, mask)]
        out.append(F.masked_ffn_mxfp4_backward(g, *q, mask, out[7]))
        return out

    usual = everything()
    monkeypatch.setattr(mxfp4, "_native", lambda: Nothing())
    for i, (a, b) in enumerate(zip(usual, everything(), strict=True)):
        assert torch.equal(a, b), i


def test_gradients_against_differences():
    """The layers are constant in pieces (rows are rounded to four bits), so the gradient is that of the layer without the rounding:
    differences of the 64-bit layer over the same weights, along directions.  The rounding of the rows moves it: the rows lie on the
    grid here, where there is none, and the intermediate's rounding does not enter."""
    note("differences")
    m, d, h = 40, 64, 128
    x, q, mask, _, w = ffn_case(m, d, h, "mixed")
    x = ref.values(x).bfloat16()
    g = rows(m, d, 3)

    def layer(t):
        def side(w1, w2, w3):
            a = t @ w1.T
            return (a / (1 + torch.exp(-a)) * (t @ w3.T)) @ w2.T
        return torch.where(mask[:, None], side(*(w[n] for n in FFN[:3])), side(*(w[n] for n in FFN[3:])))

    leaf = x.clone().requires_grad_()
    F.MaskedFFNMXFP4.apply(leaf, *q, mask).backward(g)
    _, bound = ref.ffn_grad(g, ref.values(x), w, mask)
    for seed in range(4):
        v = torch.randn(m, d, generator=gen(seed), device="cuda", dtype=torch.float64)
        e = 1e-5
        slope = ((layer(x.double() + e * v) - layer(x.double() - e * v)) / (2 * e) * g.double()).sum(1)
        # the central difference's own error is e^2 times a third derivative: 1e-10 of values of the slope's size, far inside 1e-6
        assert (((leaf.grad.double() * v).sum(1) - slope).abs() <= (bound * v.abs()).sum(1) + 1e-6 * slope.abs().max()).all()


# ---- a run of them together, as a block uses them --------------------------------------------------------------------------------

@pytest.mark.parametrize("batch,seq", [(1, 1), (3, 9), (2, 150)])
def test_modules_of_a_block(batch, seq):
    note(f"modules {batch}x{seq}")
    torch.manual_seed(4)
    d, h = 256, 520
    proj, ffn = F.MaskedLinearModule(d, d, device="cuda"), F.MaskedFFNModule(d, h, device="cuda")
    proj4, ffn4 = F.MaskedLinearMXFP4Module.from_module(proj), F.MaskedFFNMXFP4Module.from_module(ffn)
    x = rows(batch * seq, d, 6).view(batch, seq, d).requires_grad_()
    mask = a_mask(batch * seq, "mixed").view(batch, seq)
    y = ffn4(proj4(x, mask), mask)
    y.backward(torch.ones_like(y))
    m, a = mask.view(-1), ref.values(x.detach().view(-1, d))
    mid = proj4(x, mask).detach().view(-1, d)
    within(mid, *ref.linear(a, ref.values(proj.linear_v.weight.detach()), ref.values(proj.linear_t.weight.detach()), m), "projection")
    w = {n: ref.values(getattr(ffn, n).weight.detach()) for n in FFN}
    within(y.detach().view(-1, d), *ref.ffn(ref.values(mid), w, m), "feed-forward")
    assert x.grad.isfinite().all() and x.grad.abs().max() > 0
    # a state that is saved and loaded, copied and moved answers alike
    fresh = F.MaskedFFNMXFP4Module(d, h, device="cuda")
    fresh.load_state_dict(ffn4.state_dict())
    moved = copy.deepcopy(ffn4).cpu().cuda()
    with torch.no_grad():
        for other in (fresh, moved, copy.deepcopy(ffn4)):
            assert torch.equal(other(proj4(x, mask), mask), y)


def test_rows_quantised_once_serve_several_projections():
    note("shared rows")
    x, qv, qt, mask, _ = linear_case(200, 512, 96, "mixed")
    q = F.mxfp4_quantise(x)
    routing = F.route(mask)
    for seed in (3, 5):
        a, b = F.mxfp4_quantise(weight(96, 512, seed)), F.mxfp4_quantise(weight(96, 512, seed + 1))
        assert torch.equal(F.masked_linear_mxfp4_forward(q, a, b, mask, routing=routing), F.masked_linear_mxfp4_forward(x, a, b, mask))


@pytest.mark.parametrize("m", [4, 64, 150, 2100])
def test_graphs_and_streams(m):
    note(f"graph {m}")
    d, h = 256, 4160 if m > 1000 else 544
    x, q, mask, _, _ = ffn_case(m, d, h, "mixed")
    p = F.mxfp4_quantise(weight(d, d, 2)), F.mxfp4_quantise(weight(d, d, 3))

    def block(t):
        with torch.no_grad():
            return F.MaskedFFNMXFP4.apply(F.MaskedLinearMXFP4.apply(t, *p, mask), *q, mask)

    want = block(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(block(x), want)
    torch.cuda.current_stream().wait_stream(side)
    held = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = block(held)
    for seed in (21, 22, 23):
        held.copy_(rows(m, d, seed))
        graph.replay()
        replayed = out.clone()
        eager = block(held)
        torch.cuda.synchronize()
        assert torch.equal(replayed, eager)


@pytest.mark.parametrize("m", [30, 150])
def test_backward_on_another_stream_and_in_a_graph(m):
    note(f"backward graph {m}")
    d, h = 256, 520
    x, q, mask, _, _ = ffn_case(m, d, h, "mixed")
    p = F.mxfp4_quantise(weight(d, d, 2)), F.mxfp4_quantise(weight(d, d, 3))
    g = rows(m, d, 9)

    def gradient(t):
        leaf = t.detach().requires_grad_()
        return torch.autograd.grad(F.MaskedFFNMXFP4.apply(F.MaskedLinearMXFP4.apply(leaf, *p, mask), *q, mask), leaf, g)[0]

    want = gradient(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(gradient(x), want)
        held = x.clone()
        gradient(held)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = gradient(held)
    for seed in (31, 32, 33):
        held.copy_(rows(m, d, seed))
        graph.replay()
        replayed = out.clone()
        eager = gradient(held)
        torch.cuda.synchronize()
        assert torch.equal(replayed, eager)


def test_two_graphs_and_a_mask_that_changes():
    """Each graph has room of its own; a replay routes by what the mask holds by then."""
    note("two graphs")
    m, d, h = 150, 256, 544
    x, q, mask, _, _ = ffn_case(m, d, h, "mixed")
    other = rows(m, d, 5)
    mask = mask.clone()
    with torch.no_grad():
        F.MaskedFFNMXFP4.apply(x, *q, mask)
        torch.cuda.synchronize()
        graphs = []
        for t in (x, other):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = F.MaskedFFNMXFP4.apply(t, *q, mask)
            graphs.append((graph, out, t))
        for seed in (1, 2, 3):
            mask.copy_(a_mask(m, "mixed", seed))
            for graph, _, _ in graphs:
                graph.replay()
            for _, out, t in graphs:
                assert torch.equal(out, F.masked_ffn_mxfp4_forward(t, *q, mask.clone()))


def test_two_threads_on_streams_of_their_own():
    """Each thread's calls, of other sizes and masks, are in flight with the other's."""
    note("two threads")
    import threading
    jobs, failed = [], []
    for m, d, h in ((150, 256, 544), (40, 520, 264)):
        x, q, mask, _, _ = ffn_case(m, d, h, "mixed")
        jobs.append((x, q, mask, F.masked_ffn_mxfp4_forward(x, *q, mask)))
    torch.cuda.synchronize()

    def work(job):
        x, q, mask, want = job
        try:
            with torch.cuda.stream(torch.cuda.Stream()), torch.no_grad():
                outs = [F.MaskedFFNMXFP4.apply(x, *q, mask) for _ in range(30)]
                torch.cuda.current_stream().synchronize()
                assert all(torch.equal(out, want) for out in outs)
                torch.cuda.current_stream().synchronize()
        except BaseException as e:  # noqa: BLE001 (shown by the test)
            failed.append(e)

    threads = [threading.Thread(target=work, args=(job,)) for job in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed


def test_empty_batches_train():
    note("empty training")
    x, q, mask, _, _ = ffn_case(8, 64, 128, "mixed")
    leaf = x[:0].clone().requires_grad_()
    y = F.MaskedFFNMXFP4.apply(leaf, *q, mask[:0])
    y = y + F.MaskedLinearMXFP4.apply(leaf, F.mxfp4_quantise(weight(64, 64, 1)), F.mxfp4_quantise(weight(64, 64, 2)), mask[:0])
    y.sum().backward()
    assert y.shape == (0, 64) and leaf.grad.shape == (0, 64)
    proj = F.MaskedLinearMXFP4Module.from_module(F.MaskedLinearModule(64, 40, device="cuda"))
    with pytest.raises(ValueError, match="multiple of 64"):  # 40 output features have no backward: said at the forward
        proj(x.requires_grad_(), mask)
    with torch.no_grad():
        assert proj(x, mask).shape == (8, 40)


# ---- what a short call skips when there is nothing to record ------------------------------------------------------------------------

@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
def test_traces_replay_the_layers():
    note("traces")
    x, q, mask, _, _ = ffn_case(100, 64, 128, "mixed")
    p = F.mxfp4_quantise(weight(64, 64, 2)), F.mxfp4_quantise(weight(64, 64, 3))

    def block(t, m):
        return F.MaskedFFNMXFP4.apply(F.MaskedLinearMXFP4.apply(t, *p, m), *q, m)

    traced = torch.jit.trace(block, (x, mask), check_trace=False)
    for seed in (4, 5):
        other = rows(100, 64, seed)
        assert torch.equal(traced(other, ~mask), block(other, ~mask))


def test_forward_mode_is_refused():
    note("forward mode")
    x, q, mask, _, _ = ffn_case(100, 64, 128, "mixed")
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda t: F.MaskedFFNMXFP4.apply(t, *q, mask), lambda t: F.MaskedLinearMXFP4.apply(t, q[0], q[3], mask)):
            with pytest.raises(NotImplementedError):
                call(dual)
            call(x)


# ---- weight streams whose wavefronts take several 512-column groups, as many, or none -------------------------------------------------

@pytest.mark.parametrize("m,k,n", [(16, 5120, 70), (9, 2600, 100), (1, 14336, 130), (16, 14330, 33), (2, 9000, 49), (27, 14336, 130), (32, 2600, 24), (20, 1544, 16),
                                   (40, 14336, 72), (48, 7000, 31), (64, 8200, 40)])
@pytest.mark.parametrize("kind", ["mixed", "text"])
def test_linear_streams_of_long_rows(m, k, n, kind):
    note(f"linear stream {m}x{k}->{n} {kind}")
    x, qv, qt, mask, (a, wv, wt) = linear_case(m, k, n, kind)
    value, bound = ref.linear(a, wv, wt, mask)
    y = F.masked_linear_mxfp4_forward(x, qv, qt, mask)
    within(y, value, bound, "rows in bf16")
    within(F.masked_linear_mxfp4_forward(F.mxfp4_quantise(x), qv, qt, mask), value, bound, "rows in MXFP4")
    assert torch.equal(y, F.masked_linear_mxfp4_forward(x, qv, qt, mask)), "the same call twice"


@pytest.mark.parametrize("m,d,h", [(16, 4096, 264), (9, 2600, 520), (16, 5000, 40), (27, 4096, 264), (27, 2600, 136), (32, 5000, 31), (48, 4096, 136), (33, 2600, 72),
                                   (16, 72, 9000), (27, 64, 14330), (40, 64, 8200)])
@pytest.mark.parametrize("kind", ["mixed", "visual"])
def test_ffn_streams_of_long_rows(m, d, h, kind):
    note(f"ffn stream {m} {d} {h} {kind}")
    x, q, mask, a, w = ffn_case(m, d, h, kind)
    value, bound = ref.ffn(a, w, mask)
    y = F.masked_ffn_mxfp4_forward(x, *q, mask)
    within(y, value, bound, "rows in bf16")
    within(F.masked_ffn_mxfp4_forward(F.mxfp4_quantise(x), *q, mask), value, bound, "rows in MXFP4")
    assert torch.equal(y, F.masked_ffn_mxfp4_forward(x, *q, mask)), "the same call twice"


# The rows that a stream quantises itself: wavefronts with several groups, one, and none in one workgroup, up to the longest rows.
@pytest.mark.parametrize("m,k,n", [(1, 8192, 130), (2, 8192, 70), (4, 4096, 40), (2, 6176, 33), (3, 2592, 31), (8, 2048, 24), (16, 1024, 72), (1, 544, 16)])
@pytest.mark.parametrize("kind", ["mixed", "text"])
def test_linear_streams_that_quantise_their_rows(m, k, n, kind):
    note(f"linear fused stream {m}x{k}->{n} {kind}")
    x, qv, qt, mask, (a, wv, wt) = linear_case(m, k, n, kind)
    value, bound = ref.linear(a, wv, wt, mask)
    y = F.masked_linear_mxfp4_forward(x, qv, qt, mask)
    within(y, value, bound, "rows in bf16")
    assert torch.equal(y, F.masked_linear_mxfp4_forward(F.mxfp4_quantise(x), qv, qt, mask)), "rows in MXFP4"


@pytest.mark.parametrize("m,d,h", [(1, 4096, 1000), (4, 4096, 264), (1, 8192, 72), (2, 8192, 40), (2, 6176, 200), (1, 2592, 520), (3, 2560, 136), (5, 1568, 33),
                                   (16, 1024, 264), (9, 1760, 96)])
@pytest.mark.parametrize("kind", ["mixed", "visual"])
def test_ffn_streams_that_quantise_their_rows(m, d, h, kind):
    note(f"ffn fused stream {m} {d} {h} {kind}")
    x, q, mask, a, w = ffn_case(m, d, h, kind)
    value, bound = ref.ffn(a, w, mask)
    y = F.masked_ffn_mxfp4_forward(x, *q, mask)
    within(y, value, bound, "rows in bf16")
    assert torch.equal(y, F.masked_ffn_mxfp4_forward(F.mxfp4_quantise(x), *q, mask)), "rows in MXFP4"


def test_training_keeps_the_weights_it_ran_with():
    note("saved weights")
    d, h, m = 64, 128, 100
    x, q, mask, _, _ = ffn_case(m, d, h, "mixed")
    ffn = F.MaskedFFNMXFP4Module(d, h, device="cuda")
    for name, w in zip(FFN, q):
        getattr(ffn, f"{name}_codes").copy_(w.codes), getattr(ffn, f"{name}_scales").copy_(w.scales)
    g = rows(m, d, 3)
    leaf = x.clone().requires_grad_()
    want, = torch.autograd.grad(ffn(leaf, mask), leaf, g)
    with torch.autograd.graph.save_on_cpu():
        y = ffn(leaf, mask)
    assert torch.equal(torch.autograd.grad(y, leaf, g)[0], want)
    y = torch.utils.checkpoint.checkpoint(ffn, leaf, mask, use_reentrant=False)
    assert torch.equal(torch.autograd.grad(y, leaf, g)[0], want)
    y = ffn(leaf, mask)
    ffn.load_state_dict({k: torch.zeros_like(v) for k, v in ffn.state_dict().items()})
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(g)


def test_weights_quantised_in_inference_mode_train():
    note("inference mode")
    x, _, _, mask, (_, wv, wt) = linear_case(70, 128, 64, "mixed")
    with torch.inference_mode():
        v, t = F.mxfp4_quantise(wv.bfloat16()), F.mxfp4_quantise(wt.bfloat16())
        t = F.MXFP4.from_parts(*t.parts(), 128)
        narrow = F.mxfp4_quantise(torch.zeros(64, 1, device="cuda", dtype=torch.bfloat16))  # (the call that Python takes)
    assert not any(p.is_inference() for q in (v, t, narrow) for p in (q.codes, q.scales))
    g = rows(70, 64, 3)
    x.requires_grad_()
    da, = torch.autograd.grad(F.MaskedLinearMXFP4.apply(x, v, t, mask), x, g)
    within(da, *ref.linear_grad(g.double(), wv, wt, mask), "gradient")


def test_a_module_that_moves_away_frees_its_weights():
    note("offload")
    import io
    import weakref

    x, q, mask, _, _ = ffn_case(70, 64, 128, "mixed")
    ffn = F.MaskedFFNMXFP4Module.from_module(F.MaskedFFNModule(64, 128, device="cuda"))
    with torch.no_grad():
        want = ffn(x, mask)
        gone = [weakref.ref(b) for b in ffn.buffers()]
        ffn.cpu()
        assert not any(ref() is not None for ref in gone)
        assert torch.equal(ffn.cuda()(x, mask), want)
        gone = [weakref.ref(b) for b in ffn.buffers()]
        ffn.load_state_dict({k: v.clone() for k, v in ffn.state_dict().items()}, assign=True)
        assert not any(ref() is not None for ref in gone)
        assert torch.equal(ffn(x, mask), want)
        file = io.BytesIO()
        torch.save(ffn, file)
        for device in ("cpu", "cuda"):
            file.seek(0)
            other = torch.load(file, map_location=device, weights_only=False)  # (this test's own file)
            assert torch.equal(other.cuda()(x, mask), want)


def test_upstream_gradients_whose_rows_lie_far_apart():
    note("upstream gradient over 4.6 GB")
    m, d, h = 1100, 64, 128
    x, q, mask, a, w = ffn_case(m, d, h, "mixed")
    g = rows(m, d, 3)
    far = torch.empty(m, 1 << 21, device="cuda", dtype=torch.bfloat16)[:, 64:64 + d]
    far.copy_(g)
    x.requires_grad_()
    da, = torch.autograd.grad(F.MaskedFFNMXFP4.apply(x, *q, mask), x, far)
    within(da, *ref.ffn_grad(g, a, w, mask), "feed-forward")
    v, t = F.mxfp4_quantise(weight(d, d, 1)), F.mxfp4_quantise(weight(d, d, 2))
    assert torch.equal(F.masked_linear_mxfp4_backward(far, v, t, mask), F.masked_linear_mxfp4_backward(g, v, t, mask))


@pytest.mark.parametrize("m", [5, 40, 100])
def test_bytes_behind_the_last_block_do_not_count(m):
    note(f"last bytes {m}")
    d, h = 264, 1001
    x, q, mask, a, w = ffn_case(m, d, h, "mixed")
    value, bound = ref.ffn(a, w, mask)

    def spoilt(t):
        codes, scales = t.codes.clone(), t.scales.clone()
        if t.columns % 32:
            codes[:, -(-t.columns // 2):] = 0x77
        if t.columns % 2:
            codes[:, t.columns // 2] |= 0x70
        blocks = -(-t.columns // 32)
        scales[-1, :, (blocks - 1) % 16 + 1:] = 200
        return codes, scales

    bad = [F.MXFP4(*spoilt(t), t.columns) for t in q]
    within(F.masked_ffn_mxfp4_forward(F.MXFP4(*spoilt(F.mxfp4_quantise(x)), d), *bad, mask), value, bound, "handed over")
    ffn = F.MaskedFFNMXFP4Module(d, h, device="cuda")
    with torch.no_grad():
        ffn(x, mask)
        ffn.load_state_dict({f"{n}_{part}": s for n, t in zip(FFN, q) for part, s in zip(("codes", "scales"), spoilt(t))})
        within(ffn(x, mask), value, bound, "loaded")
        assert torch.equal(ffn.w2_scales, q[1].scales) and torch.equal(ffn.w2_codes, q[1].codes)


@pytest.mark.parametrize("m,d,h,kind", [(2100, 256, 6664, "mixed"), (700, 136, 264, "visual")])
def test_gradients_on_every_tile(m, d, h, kind):
    """The dh GEMM over fp32 projections on each tile, the big ones with a launch for what is past whole rounds, and both dx GEMMs."""
    x, q, mask, a, w = ffn_case(m, d, h, kind)
    g, lib = rows(m, d, 3), _lib.load()
    _, pre = F.masked_ffn_mxfp4_forward(x, *q, mask, save_pre=True)
    ffn, linear = ref.ffn_grad(g, a, w, mask), ref.linear_grad(g.double(), w["w2"], w["u2"], mask)
    try:
        for tile in (0, 1, 2, 3, 4, 6, 7):
            note(f"gradient on tile {tile}: {m} {d} {h} {kind}")
            lib.ffnk_debug_force_tile(tile)
            within(F.masked_ffn_mxfp4_backward(g, *q, mask, pre), *ffn, f"feed-forward, tile {tile}")
            within(F.masked_linear_mxfp4_backward(g, q[1], q[4], mask), *linear, f"linear, tile {tile}")
    finally:
        lib.ffnk_debug_force_tile(-1)
