"""MXFP4 without a GPU: the oracle's rounding against the format's own definition, its gradients against differences, what the
operators refuse, and the C ABI's answers to bad arguments."""
import ctypes

import pytest
import torch

import ffn_kernel_amd as F
from ffn_kernel_amd import _lib
from oracle import mxfp4 as ref


def test_oracle_rounds_to_the_nearest_with_ties_to_even_codes():
    # block maximum 4: scale 1
    t = torch.zeros(1, 32)
    given = [4.0, 0.25, 0.26, 0.75, 0.74, 1.25, 1.75, 2.5, 3.5, 3.49, -0.25, -0.75, -2.5, -3.5, -1.3]
    wanted = [4.0, 0.0, 0.5, 1.0, 0.5, 1.0, 2.0, 2.0, 4.0, 3.0, 0.0, -1.0, -2.0, -4.0, -1.5]
    t[0, :len(given)] = torch.tensor(given)
    assert ref.values(t)[0, :len(given)].tolist() == wanted
    assert ref.exponents(t).item() == 0
    t[0, 0] = 5.0   # a tie between 4 and 6: 4 has the even code
    assert ref.values(t)[0, 0].item() == 4.0
    t[0, 0] = 7.99  # the largest of a block saturates
    assert ref.values(t)[0, 0].item() == 6.0
    t[0, 0] = 8.0
    assert ref.exponents(t).item() == 1 and ref.values(t)[0, 0].item() == 8.0


def test_oracle_blocks_and_extremes():
    t = torch.zeros(3, 70)
    t[0, 40], t[0, 69] = 3.0, -1.0
    t[1, 3], t[1, 35] = float("inf"), float("nan")
    t[2, 0] = 2.0 ** -140
    v = ref.values(t)
    assert v.shape == (3, 70) and v[0, 40].item() == 3.0 and v[0, 69].item() == -1.0
    assert ref.exponents(t)[0].tolist() == [-127, -1, -2]
    assert v[1, :64].isnan().all() and not v[1, 64:].isnan().any()
    assert v[2].abs().max().item() == 0.0  # far under the smallest scale
    codes, scales = ref.pack(t)
    assert codes.shape == (3, 48) and scales.tolist()[0] == [0, 126, 125] and scales[1, 0].item() == 255
    assert codes[0, 20].item() == 7 and codes[0, 34].item() == 14 << 4  # column 40 in a low half, 69 in a high one


def test_doubtful_covers_both_sides_of_a_border():
    h = torch.zeros(1, 32, dtype=torch.float64)
    h[0, 0], h[0, 1], h[0, 2] = 4.0 + 1e-3, 2.5, 1.3
    bound = torch.full_like(h, 1e-6)
    d = ref.doubtful(h, bound)
    assert d[0, 1].item() == 1.0 and d[0, 2].item() == 0.0 and d[0, 0].item() == 0.0
    h[0, 0] = 8.0  # the scale itself is in doubt: 1 or 2
    assert ref.doubtful(h, bound)[0, 0].item() >= 2.0


# The rows' gradient is that of the function with both quantisations passed over, at the quantised rows.
def test_oracle_gradients_against_differences():
    gen = torch.Generator().manual_seed(3)
    M, d, h = 5, 64, 96
    draw = lambda *s: ref.values(torch.randn(*s, generator=gen))
    a, mask = draw(M, d), torch.tensor([True, False, True, True, False])
    w = {n: draw(d, h) if n[1] == "2" else draw(h, d) for n in ("w1", "w2", "w3", "u1", "u2", "u3")}
    g = torch.randn(M, d, generator=gen, dtype=torch.float64)

    def loss(x):
        rows = []
        for s, on in (("w", mask), ("u", ~mask)):
            y = torch.nn.functional.silu(x @ w[s + "1"].T) * (x @ w[s + "3"].T) @ w[s + "2"].T
            rows.append((y * g * on.unsqueeze(-1)).sum())
        return sum(rows)

    da, _ = ref.ffn_grad(g, a, w, mask)
    for _ in range(6):
        v = torch.randn(M, d, generator=gen, dtype=torch.float64)
        eps = 1e-6
        slope = (loss(a + eps * v) - loss(a - eps * v)) / (2 * eps)
        assert abs(slope - (da * v).sum()) <= 1e-6 * (da.abs() * v.abs()).sum()
    gl = torch.randn(M, h, generator=gen, dtype=torch.float64)
    dl, _ = ref.linear_grad(gl, w["w1"], w["u1"], mask)
    v = torch.randn(M, d, generator=gen, dtype=torch.float64)
    c = torch.where(mask.unsqueeze(-1), v @ w["w1"].T, v @ w["u1"].T)
    assert abs((c * gl).sum() - (dl * v).sum()) <= 1e-9 * (dl.abs() * v.abs()).sum()


@pytest.mark.parametrize("call", [
    lambda: F.mxfp4_quantise([1.0]),
    lambda: F.mxfp4_dequantise(torch.zeros(2, 2)),
    lambda: F.masked_linear_mxfp4_forward(F, None, None, None),
])
def test_wrong_kinds_are_type_errors(call):
    with pytest.raises(TypeError):
        call()


@pytest.mark.parametrize("t", [torch.zeros(4), torch.zeros(2, 2, dtype=torch.float64), torch.zeros(2, 2, dtype=torch.int8), torch.zeros(2, 32)])
def test_quantise_refuses(t):
    with pytest.raises(ValueError):
        F.mxfp4_quantise(t)


def test_from_parts_refuses():
    codes, scales = torch.zeros(4, 16, dtype=torch.uint8), torch.zeros(4, 1, dtype=torch.uint8)
    for c, s, k in ((codes, scales, 64), (codes, scales[:3], 32), (codes.float(), scales, 32), (codes[0], scales, 32), (codes, scales, -1),
                    (codes, scales[:, :0], 32)):
        with pytest.raises((ValueError, RuntimeError)):
            F.MXFP4.from_parts(c, s, k)
    with pytest.raises(ValueError, match="GPU"):
        F.MXFP4.from_parts(codes, scales, 32)  # all there, but in host memory


def test_short_linear_calls_need_no_workspace():
    need = _lib.load().ffnk_mxfp4_workspace_bytes_linear_fwd
    whole = _lib.load().ffnk_mxfp4_workspace_bytes
    op = _lib.OP_LINEAR_FWD
    assert need(1 << 20, 1024, 1, 1024, 64) == 0                             # quantised in the stream
    assert need(None, 0, 64, 1024, 64) == 0                                  # rows in MXFP4
    assert need((1 << 20) + 2, 1024, 1, 1024, 64) == whole(op, 1, 1024, 64)  # off 16 bytes
    assert need(1 << 20, 1024, 64, 1024, 64) == whole(op, 64, 1024, 64)
    assert need(None, 0, 65, 1024, 64) == whole(op, 65, 1024, 64)
    assert need(None, 0, -1, 1024, 64) == ctypes.c_size_t(-1).value


def test_workspace_and_refusals_of_the_c_abi():
    lib = _lib.load()
    bad = ctypes.c_size_t(-1).value
    size = lib.ffnk_mxfp4_workspace_bytes
    assert size(_lib.OP_LINEAR_FWD, 8, 4096, 4096) >= 8 * 4096 * 17 // 32
    assert size(_lib.OP_FFN_FWD, 300, 4096, 14336) >= 300 * (4096 + 14336) * 17 // 32 + 300 * 4
    assert size(_lib.OP_FFN_BWD, 300, 4096, 14336) >= 6 * 4096 * 14336 * 2
    assert size(_lib.OP_LINEAR_BWD, 300, 512, 256) >= 2 * 512 * 256 * 2
    assert size(_lib.OP_FFN_UP, 300, 512, 256) == bad and size(_lib.OP_LINEAR_FWD, -1, 8, 8) == bad and size(_lib.OP_LINEAR_FWD, 8, 0, 8) == bad
    t = _lib.Mxfp4Struct(0x1000, 0x2000)
    q, half, off = ctypes.addressof(t), _lib.Mxfp4Struct(0x1000, None), _lib.Mxfp4Struct(0x1008, 0x2000)
    E = dict(NULL=-1, SHAPE=-2, STRIDE=-3, ALIGN=-4, WORKSPACE=-5, OP=-6)
    quantise, dequantise, linear, ffn = lib.ffnk_mxfp4_quantise, lib.ffnk_mxfp4_dequantise, lib.ffnk_mxfp4_linear_fwd, lib.ffnk_mxfp4_ffn_fwd
    assert quantise(0x100, 0, 32, q, -1, 32, None) == E["SHAPE"]
    assert quantise(0x100, 7, 32, q, 1, 32, None) == E["OP"]
    assert quantise(None, 0, 32, q, 1, 32, None) == E["NULL"]
    assert quantise(0x100, 0, 31, q, 1, 32, None) == E["STRIDE"]
    assert quantise(0x101, 0, 32, q, 1, 32, None) == E["ALIGN"] and quantise(0x102, 2, 32, q, 1, 32, None) == E["ALIGN"]
    assert quantise(0x100, 0, 32, ctypes.addressof(half), 1, 32, None) == E["NULL"]
    assert quantise(0x100, 0, 32, ctypes.addressof(off), 1, 32, None) == E["ALIGN"]
    assert quantise(None, 0, 0, None, 0, 32, None) == 0
    assert dequantise(q, None, 0, 32, 1, 32, None) == E["NULL"] and dequantise(q, 0x100, 0, 8, 1, 32, None) == E["STRIDE"]
    ws = (0x4000, 1 << 30)
    assert linear(0x100, 64, None, q, q, 0x10, 0x100, 64, 65, 64, 64, None, 0, None, None, 0) == E["WORKSPACE"]
    assert linear(0x102, 64, None, q, q, 0x10, 0x100, 64, 4, 64, 64, None, 0, None, None, 0) == E["WORKSPACE"]
    assert linear(0x100, 64, q, q, q, 0x10, 0x100, 64, 4, 64, 64, *ws, None, None, 0) == E["NULL"]      # x and xq
    assert linear(None, 64, None, q, q, 0x10, 0x100, 64, 4, 64, 64, *ws, None, None, 0) == E["NULL"]
    assert linear(0x100, 64, None, q, None, 0x10, 0x100, 64, 4, 64, 64, *ws, None, None, 0) == E["NULL"]
    assert linear(0x100, 64, None, q, q, None, 0x100, 64, 4, 64, 64, *ws, None, None, 0) == E["NULL"]
    assert linear(0x100, 63, None, q, q, 0x10, 0x100, 64, 4, 64, 64, *ws, None, None, 0) == E["STRIDE"]
    assert linear(0x100, 64, None, q, q, 0x10, 0x100, 63, 4, 64, 64, *ws, None, None, 0) == E["STRIDE"]
    assert linear(0x100, 64, None, q, q, 0x10, 0x100, 64, 4, 0, 64, *ws, None, None, 0) == E["SHAPE"]
    assert linear(None, 0, q, q, q, 0x10, 0x100, 64, 1 << 24, 1 << 10, 64, 0x4000, 1 << 62, None, None, 0) == E["SHAPE"]  # past 32-bit offsets
    assert ffn(0x100, 64, None, q, q, q, q, q, None, 0x10, 0x100, 64, None, 4, 64, 64, *ws, None, None, 0) == E["NULL"]
    assert b"U3" in lib.ffnk_last_error()
    lb, fb = lib.ffnk_mxfp4_linear_bwd, lib.ffnk_mxfp4_ffn_bwd
    assert lb(0x100, 64, q, q, 0x10, 0x100, 63, 4, 63, 64, *ws, None, None) == E["STRIDE"]
    assert lb(0x100, 72, q, q, 0x10, 0x100, 64, 4, 64, 72, *ws, None, None) == E["STRIDE"]
    assert lb(0x100, 64, q, q, 0x10, 0x100, 64, 4, 64, 64, 0x4000, 64, None, None) == E["WORKSPACE"]
    assert fb(0x100, 64, q, q, q, q, q, q, 0x10, None, 0x100, 64, 4, 64, 64, *ws, None, None) == E["NULL"]
    assert fb(0x100, 64, q, q, q, q, q, q, 0x10, 0x108, 0x100, 64, 4, 64, 64, *ws, None, None) == E["STRIDE"]
    assert linear(None, 0, None, None, None, None, None, 64, 0, 64, 64, None, 0, None, None, 0) == 0  # no rows


# ---- the layers under a tracer and in forward mode: a stand-in for the foreign call, which torch cannot see into either -----------

@pytest.fixture
def unseen_layers(monkeypatch):
    """Both forwards as functions of host memory alone: 2 a, whatever the weights."""
    from ffn_kernel_amd import mxfp4

    def twice(a, *rest, save_pre=False, **_):
        y, held = torch.empty_like(a), 2 * a.detach()
        ctypes.memmove(y.data_ptr(), held.data_ptr(), 4 * a.numel())
        return (y, torch.zeros(a.shape[0], 2)) if save_pre else y

    monkeypatch.setattr(mxfp4, "masked_linear_mxfp4_forward", twice)
    monkeypatch.setattr(mxfp4, "masked_ffn_mxfp4_forward", twice)
    return [lambda a, mask, n=n, f=f: f.apply(a, *[object()] * n, mask) for n, f in ((2, F.MaskedLinearMXFP4), (6, F.MaskedFFNMXFP4))]


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
@pytest.mark.parametrize("requires_grad", [False, True])
@pytest.mark.parametrize("layer", [0, 1])
def test_a_trace_holds_the_call(unseen_layers, layer, requires_grad):
    call, mask = unseen_layers[layer], torch.ones(3, dtype=torch.bool)
    with torch.no_grad():
        traced = torch.jit.trace(call, (torch.randn(3, 4).requires_grad_(requires_grad), mask), check_trace=False)
        for seed in (1, 2):
            a = torch.randn(3, 4, generator=torch.Generator().manual_seed(seed))
            held = [torch.full((3, 4), 7.0) for _ in range(64)]  # so that memory handed out anew holds something else
            del held
            assert torch.equal(traced(a, mask), 2 * a)


@pytest.mark.parametrize("layer", [0, 1])
def test_forward_mode_is_refused(unseen_layers, layer):
    call, mask = unseen_layers[layer], torch.ones(3, dtype=torch.bool)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(torch.randn(3, 4), torch.ones(3, 4))
        with pytest.raises(NotImplementedError):
            call(dual, mask)
        plain = torch.randn(3, 4)
        assert torch.equal(call(plain, mask), 2 * plain)  # no derivative on its way
    with pytest.raises((NotImplementedError, RuntimeError)):
        torch.func.jvp(lambda a: call(a, mask), (torch.randn(3, 4),), (torch.ones(3, 4),))
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda a: call(a, mask))(torch.randn(2, 3, 4))


def test_conversions_refuse_a_tracer():
    weight = torch.zeros(2, 32)
    for convert in (F.mxfp4_quantise, lambda t: F.mxfp4_dequantise(t)):
        with pytest.raises(RuntimeError, match="cannot be traced"):
            torch.jit.trace(lambda t: convert(t) or t, (torch.zeros(2, 32),), check_trace=False)
    with pytest.raises(ValueError, match="GPU"):  # a constant of the trace: refused for where it lies alone
        torch.jit.trace(lambda t: F.mxfp4_quantise(weight) and t, (torch.zeros(2, 32),), check_trace=False)


@pytest.mark.parametrize("layer,count", [(F.MaskedLinearMXFP4, 2), (F.MaskedFFNMXFP4, 6)])
@pytest.mark.parametrize("part", ["codes", "scales"])
def test_a_backward_over_changed_weights_is_refused(monkeypatch, layer, count, part):
    from ffn_kernel_amd import mxfp4

    def held():  # (an MXFP4 tensor in host memory, which its constructor refuses)
        q = F.MXFP4.__new__(F.MXFP4)
        q._codes, q._scales, q._columns, q._struct = torch.zeros(64, 32, dtype=torch.uint8), torch.zeros(1, 64, 16, dtype=torch.uint8), 64, None
        return q

    seen = []
    for name in ("masked_linear_mxfp4", "masked_ffn_mxfp4"):
        monkeypatch.setattr(mxfp4, f"{name}_forward", lambda a, *_, save_pre=False: (2 * a, torch.zeros(3, 128)) if save_pre else 2 * a)
        monkeypatch.setattr(mxfp4, f"{name}_backward", lambda grad, *weights, **_: seen.append(weights) or 2 * grad)
    a, mask, weights = torch.randn(3, 64, requires_grad=True), torch.ones(3, dtype=torch.bool), [held() for _ in range(count)]
    layer.apply(a, *weights, mask).sum().backward()
    assert torch.equal(a.grad, torch.full((3, 64), 2.0)) and all(w is q for w, q in zip(seen[0], weights))
    for w in weights:
        y = layer.apply(a, *weights, mask)
        getattr(w, part).copy_(torch.ones_like(getattr(w, part)))  # what load_state_dict does
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()


def test_a_module_keeps_no_weights_of_an_earlier_state():
    import copy
    import pickle

    module = F.MaskedLinearMXFP4Module(64, 64)

    def held():
        module._held["linear_v"] = object()  # (what a forward leaves)
        return module._held

    for change in (lambda: module.cpu(), lambda: module.to(torch.device("cpu")), lambda: module.load_state_dict(module.state_dict()),
                   lambda: module.load_state_dict({k: torch.ones_like(v) for k, v in module.state_dict().items()}, assign=True),
                   lambda: torch.nn.Sequential(module).float()):
        held()
        change()
        assert not module._held
    held()
    for other in (pickle.loads(pickle.dumps(module)), copy.deepcopy(module), copy.copy(module)):
        assert not other._held and other.state_dict().keys() == module.state_dict().keys() and other._columns == module._columns
        assert other._held is not module._held
    assert module._held
    block = torch.nn.ModuleList([module])
    block.load_state_dict(block.state_dict())
    assert not module._held


def test_addresses_are_those_of_the_tensors_by_then():
    q = F.MXFP4.__new__(F.MXFP4)
    q._codes, q._scales, q._columns, q._struct = torch.zeros(2, 16, dtype=torch.uint8), torch.zeros(1, 2, 16, dtype=torch.uint8), 32, None
    for _ in range(2):
        t = _lib.Mxfp4Struct.from_address(q._address)
        assert (t.codes, t.scales) == (q.codes.data_ptr(), q.scales.data_ptr())
        kept = q.codes.data  # (so that the new memory is other memory)
        q.codes.data, q.scales.data = torch.ones(2, 16, dtype=torch.uint8), torch.ones(1, 2, 16, dtype=torch.uint8)


def unheld(rows, columns):
    """An MXFP4 tensor of these extents without memory."""
    q = F.MXFP4.__new__(F.MXFP4)
    q._codes, q._scales, q._columns, q._struct = torch.empty(rows, 0, dtype=torch.uint8), torch.empty(0, rows, 16, dtype=torch.uint8), columns, None
    return q


# A forward that keeps its rows' gradient refuses what its backward would; both go by the rule of the C ABI.
@pytest.mark.parametrize("m,k,n", [(100, 64, 64), (524287, 512, 4096), (524288, 512, 4096), (1 << 24, 64, 64), (1 << 24, 64, 128), ((1 << 24) - 1, 64, 128),
                                   (16777215 // 2, 8, 200), (300, 8, 1 << 23), (300, 8, (1 << 23) - 64), (256, 72, 8 * 1048575), (5, 64, 72), (5, 63, 64), (5, 72, 136)])
def test_what_has_no_backward_is_refused_at_the_forward(m, k, n):
    from ffn_kernel_amd import mxfp4

    t = _lib.Mxfp4Struct(0x1000, 0x2000)
    q, lib = ctypes.addressof(t), _lib.load()
    linear = lib.ffnk_mxfp4_linear_bwd(0x100, n, q, q, 0x10, 0x100, k, m, k, n, None, 0, None, None)
    ffn = lib.ffnk_mxfp4_ffn_bwd(0x100, n, q, q, q, q, q, q, 0x10, 0x100, 0x100, n, m, n, k, None, 0, None, None)
    assert {linear, ffn} <= {-3, -5}  # a stride or extent that it does not take; no workspace given
    a, mask = torch.zeros(1, requires_grad=True).bfloat16(), torch.ones(1, dtype=torch.bool)
    up, down = unheld(k, n), unheld(n, k)
    for code, check, call in ((linear, lambda: mxfp4._check_differentiable(m, n, k), lambda: F.MaskedLinearMXFP4.apply(a.expand(m, k), down, down, mask)),
                              (ffn, lambda: mxfp4._check_differentiable(m, n, doubled=k),
                               lambda: F.MaskedFFNMXFP4.apply(a.expand(m, n), up, down, up, up, down, up, mask))):
        if code == -5:
            check()
            continue
        with pytest.raises(ValueError):
            check()
        with pytest.raises(ValueError, match="MXFP4 backward"):
            call()


def test_rows_far_apart_are_copied_for_the_backward():
    from ffn_kernel_amd import mxfp4

    assert mxfp4._reach(1 << 20, 2040, 128) and not mxfp4._reach(1 << 20, 2048, 128) and not mxfp4._reach(2, 1 << 23, 8)


@pytest.mark.parametrize("columns", [0, 1, 31, 32, 33, 511, 512, 513, 1000])
@pytest.mark.parametrize("inference", [False, True])
def test_bytes_past_the_last_column_and_block_are_cleared(columns, inference):
    from ffn_kernel_amd import mxfp4

    with torch.inference_mode(inference):
        codes = torch.full((3, mxfp4._code_bytes(columns)), 255, dtype=torch.uint8)
        scales = torch.full(mxfp4._scale_shape(3, columns), 255, dtype=torch.uint8)
    versions = None if inference else (codes._version, scales._version)
    mxfp4._clear_tails(codes, scales, columns)
    assert inference or (codes._version, scales._version) == versions
    blocks = -(-columns // 32)
    by_row, numbers = scales.transpose(0, 1).reshape(3, -1), torch.stack((codes & 15, codes >> 4), -1).view(3, -1)
    assert (by_row[:, :blocks] == 255).all() and not by_row[:, blocks:].any()
    assert (numbers[:, :columns] == 15).all() and not numbers[:, columns:].any()


def test_tensors_of_a_partition_can_be_assigned():
    for r in (F.Routing(torch.zeros(5, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)), F.Routing._unmade(5, torch.device("cpu"))):
        perm, counts = torch.arange(5, dtype=torch.int32), torch.tensor([2, 3], dtype=torch.int32)
        r.perm = perm
        assert r.perm is perm and r.counts.shape == (2,) and r.M == 5
        r.counts = counts
        held = _lib.RoutingStruct.from_address(r.address)
        assert r.counts is counts and (held.perm, held.counts) == (perm.data_ptr(), counts.data_ptr())


def test_parts_of_a_traced_value_are_refused():
    codes, scales = torch.zeros(4, 16, dtype=torch.uint8), torch.zeros(4, 1, dtype=torch.uint8)
    for build in (lambda t: F.MXFP4.from_parts(t, scales, 32), lambda t: F.MXFP4.from_parts(codes, t[:, :1], 32)):
        with pytest.raises(RuntimeError, match="cannot be traced"):
            torch.jit.trace(lambda t: build(t) and t, (codes,), check_trace=False)


def test_a_trace_of_a_module_holds_no_preparation_of_its_weights(monkeypatch):
    """Columns that end inside a group of 512: the constructor clears what lies past them, outside the trace."""
    from ffn_kernel_amd import mxfp4

    monkeypatch.setattr(F.MXFP4, "_hold", lambda self, codes, scales, columns: [setattr(self, n, v) for n, v in (
        ("_codes", codes), ("_scales", scales), ("_columns", columns), ("_struct", None))])
    monkeypatch.setattr(mxfp4, "masked_linear_mxfp4_forward", lambda a, *_: a.new_empty(a.shape))
    module = F.MaskedLinearMXFP4Module(40, 40)
    module.linear_t_scales.fill_(3)
    traced = torch.jit.trace(module, (torch.zeros(3, 40), torch.ones(3, dtype=torch.bool)), check_trace=False)
    assert "aten::fill_" not in str(traced.graph) and "MaskedLinearMXFP4" in str(traced.graph)
    assert module.linear_t_scales[0, :, 2:].sum() == 0 and (module.linear_t_scales[0, :, :2] == 3).all()


@pytest.mark.parametrize("layer", [0, 1])
def test_transforms_of_something_else_let_the_layers_run(unseen_layers, layer):
    call, mask, a = unseen_layers[layer], torch.ones(3, dtype=torch.bool), torch.randn(3, 4)
    beside = lambda t: (call(a, mask) * t).sum()
    t = torch.randn(3, 4)
    assert torch.equal(torch.func.vmap(beside)(torch.stack((t, t)))[1], (2 * a * t).sum())
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(t, torch.ones(3, 4))
        assert torch.equal(torch.autograd.forward_ad.unpack_dual(beside(dual)).tangent, (2 * a).sum())
    for transform in (torch.func.grad(beside), lambda t: torch.func.jvp(beside, (t,), (torch.ones(3, 4),))):
        with pytest.raises(RuntimeError):  # what they allocate in there has no memory
            transform(t)


def test_tensors_that_do_not_fit_a_partition_are_refused():
    r = F.Routing._unmade(5, torch.device("cpu"))
    for name, t in (("perm", torch.zeros(4, dtype=torch.int32)), ("perm", torch.zeros(5, dtype=torch.int64)), ("perm", torch.zeros(10, dtype=torch.int32)[::2]),
                    ("counts", torch.zeros(1, dtype=torch.int32)), ("counts", [2, 3]), ("counts", torch.zeros(2, dtype=torch.int32, device="meta"))):
        with pytest.raises(ValueError, match=name):
            setattr(r, name, t)
