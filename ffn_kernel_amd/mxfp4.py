"""The routed layers over weights held in 4 bits (MXFP4, OCP Microscaling): quantisation, MaskedLinear and MaskedFFN.

    q = mxfp4_quantise(weight)                          # nn.Linear.weight [out, in], blocks of 32 along `in`
    MaskedLinearMXFP4.apply(a, b1, b2, mask) -> c       # MaskedLinear with b1, b2 the quantised weights (not transposed views)
    MaskedFFNMXFP4.apply(a, w1, w2, w3, u1, u2, u3, mask)

A block of 32 columns shares a power of two; its elements are 0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign.  The rows `a` (bf16) are
quantised the same way in the call, and so is the SwiGLU intermediate, so that the matrix cores multiply 4-bit operands; sums are
held in fp32.  `a` may also be an MXFP4 tensor: rows that several projections share are quantised once.

The weights are constants.  The gradient of `a` passes the quantisations over (straight-through), which is what training adapters
over a frozen model asks for.  No counterpart in the reference.
"""
from __future__ import annotations

import ctypes

import torch
from torch.autograd import Function, forward_ad
from torch.autograd.function import once_differentiable

from . import _lib, ops
from .ops import (Routing, _grad_mode, _on_device, _require_cuda_bf16, _require_mask, _route_cache, _routing_arg, _same_device,
                  _stream_ptr, _workspace)

_BLOCK = 32
_DTYPES = {torch.bfloat16: _lib.DT_BF16, torch.float16: _lib.DT_FP16, torch.float32: _lib.DT_FP32}


def _code_bytes(columns: int) -> int:
    return -(-columns // _BLOCK) * 16


def _scale_shape(rows: int, columns: int) -> tuple:
    return (-(-columns // (_BLOCK * 16)), rows, 16)


_tracing, _transforms_active = torch._C._is_tracing, torch._C._are_functorch_transforms_active


def _refuse_tracer(name: str, t=None) -> None:
    """torch.jit.trace sees neither the launch nor, in an MXFP4 object, the tensors: the replays would find the traced call's codes, or
    memory that nobody wrote.  A constant of the trace (`t`) may be quantised in it."""
    if not (isinstance(t, torch.Tensor) and torch._C._get_value_trace(t).node().kind() == "prim::Constant"):
        raise RuntimeError(f"{name} cannot be traced: call it ahead of torch.jit.trace (the layers' apply quantises bf16 rows and is traced whole)")


def _clear_tails(codes: torch.Tensor, scales: torch.Tensor, columns: int) -> None:
    """0 to what lies past the last column and the last block.  Nothing that a caller holds changes its meaning by it, so the tensors'
    versions stay."""
    held, blocks = -(-columns // 2), -(-columns // _BLOCK)
    for t, any_past in ((codes, columns % _BLOCK), (scales, blocks % 16)):
        if not any_past or t.numel() == 0:
            continue
        with torch.inference_mode() if t.is_inference() else torch.autograd._unsafe_preserve_version_counter(t), torch.no_grad():
            if t is scales:
                t[-1, :, blocks % 16:] = 0
                continue
            t[:, held:] = 0
            if columns % 2:
                t[:, held - 1] &= 15


class MXFP4:
    """A [rows, columns] tensor in MXFP4 on a GPU: `codes` uint8 [rows, 16 ceil(columns / 32)], two elements to a byte with the even
    column in the low half, and `scales` uint8 [ceil(columns / 512), rows, 16], one exponent byte (bias 127) for 32 columns: those of
    512 columns together, and of all rows behind one another, as the products load them (parts() has them row by row).  Bytes past
    the last column and the last block are 0, and the products count on it: the constructor sets them in the tensors that it is given."""
    __slots__ = ("_codes", "_scales", "_columns", "_struct")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, columns: int):
        tracer = torch._C._get_tracing_state()
        torch._C._set_tracing_state(None)  # (a trace keeps the object; its replays need not clear anything)
        try:
            self._hold(codes, scales, columns)
            _clear_tails(codes, scales, self._columns)
        finally:
            torch._C._set_tracing_state(tracer)

    @classmethod
    def _whole(cls, codes: torch.Tensor, scales: torch.Tensor, columns: int) -> "MXFP4":
        """Of tensors whose last bytes are known to be 0, or still to be written."""
        q = cls.__new__(cls)
        q._hold(codes, scales, columns)
        return q

    def _hold(self, codes: torch.Tensor, scales: torch.Tensor, columns: int) -> None:
        rows = codes.shape[0] if isinstance(codes, torch.Tensor) and codes.dim() == 2 else 0
        for name, t, shape in (("codes", codes, (rows, _code_bytes(columns))), ("scales", scales, _scale_shape(rows, columns))):
            if not isinstance(t, torch.Tensor) or t.dtype != torch.uint8 or t.shape != shape:
                raise ValueError(f"{name} must be a torch.uint8 tensor {list(shape)} for {rows} rows of {columns} columns")
            if not t.is_cuda:
                raise ValueError(f"{name} must live on a GPU (got {t.device}); libffnk has no CPU path")
            if not t.is_contiguous() or t.data_ptr() % 16:
                raise ValueError(f"{name} must be contiguous and 16-byte aligned")
        if codes.device != scales.device:
            raise ValueError(f"codes are on {codes.device}, scales on {scales.device}")
        self._codes, self._scales, self._columns, self._struct = codes, scales, int(columns), None

    @classmethod
    def from_parts(cls, codes: torch.Tensor, scales: torch.Tensor, columns: int | None = None) -> "MXFP4":
        """From codes [rows, at least ceil(columns / 2)] and scales [rows, at least ceil(columns / 32)] (uint8 or float8_e8m0fnu) as
        checkpoints hold them; columns: two for each byte of codes where it is not given.  Copies both."""
        if _tracing():
            _refuse_tracer("MXFP4.from_parts", codes)
            _refuse_tracer("MXFP4.from_parts", scales)
        scales = scales.view(torch.uint8)
        if codes.dim() != 2 or scales.dim() != 2 or codes.dtype != torch.uint8 or codes.shape[0] != scales.shape[0]:
            raise ValueError(f"codes and scales must be 8-bit [rows, ...] tensors, got {tuple(codes.shape)} and {tuple(scales.shape)}")
        rows, columns = codes.shape[0], 2 * codes.shape[1] if columns is None else int(columns)
        held, blocks = -(-columns // 2), -(-columns // _BLOCK)
        if columns < 0 or codes.shape[1] < held or scales.shape[1] < blocks:
            raise ValueError(f"{columns} columns need {held} bytes of codes and {blocks} scales a row, got {codes.shape[1]} and {scales.shape[1]}")
        with torch.inference_mode(False):
            new_codes = torch.zeros((rows, _code_bytes(columns)), dtype=torch.uint8, device=codes.device)
            new_scales = torch.zeros((rows, -(-blocks // 16) * 16), dtype=torch.uint8, device=codes.device)
            new_codes[:, :held] = codes[:, :held]
            if columns % 2:
                new_codes[:, held - 1] &= 15
            new_scales[:, :blocks] = scales[:, :blocks]
            return cls._whole(new_codes, new_scales.view(rows, -1, 16).transpose(0, 1).contiguous(), columns)

    def parts(self) -> tuple:
        """(codes [rows, 16 ceil(columns / 32)], scales [rows, ceil(columns / 32)]): what from_parts takes, the scales as a copy."""
        rows, columns = self.shape
        return self._codes, self._scales.transpose(0, 1).reshape(rows, -1)[:, :-(-columns // _BLOCK)]

    def __reduce__(self):
        return MXFP4, (self._codes, self._scales, self._columns)

    @property
    def _address(self) -> int:
        """Of its ffnk_mxfp4_t, with the addresses that its tensors have by now (an assignment to .data gives them others)."""
        if self._struct is None:
            self._struct = _lib.Mxfp4Struct()
        self._struct.codes, self._struct.scales = self._codes.data_ptr(), self._scales.data_ptr()
        return ctypes.addressof(self._struct)

    codes = property(lambda self: self._codes)
    scales = property(lambda self: self._scales)
    columns = property(lambda self: self._columns)
    rows = property(lambda self: self._codes.shape[0])
    shape = property(lambda self: (self._codes.shape[0], self._columns))
    device = property(lambda self: self._codes.device)

    def dequantise(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        return mxfp4_dequantise(self, dtype)

    def __repr__(self):
        return f"MXFP4(shape={self.shape}, device='{self.device}')"


_native_call = None


def _native():
    """_call.so with the MXFP4 functions bound (ops._native): they take the usual call and return NotImplemented for any other."""
    global _native_call
    if _native_call is None:
        module, lib = ops._native(), _lib.load()
        names = ("quantise", "dequantise", "workspace_bytes", "workspace_bytes_linear_fwd", "linear_fwd", "linear_bwd", "ffn_fwd", "ffn_bwd")
        module.bind_mxfp4(tuple(ctypes.cast(getattr(lib, f"ffnk_mxfp4_{n}"), ctypes.c_void_p).value for n in names), MXFP4)
        _native_call = module
    return _native_call


def _require_mxfp4(name: str, q) -> None:
    if not isinstance(q, MXFP4):
        raise TypeError(f"{name} must be an MXFP4 tensor (mxfp4_quantise), got {type(q).__name__}")


def _dense_rows(t: torch.Tensor) -> torch.Tensor:
    """[M, K] rows with unit column stride that do not overlap; anything else is copied once."""
    M, K = t.shape
    return t if (K <= 1 or t.stride(1) == 1) and (M <= 1 or t.stride(0) >= K) else t.contiguous()


def _row_stride(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else max(t.shape[1], 1)


def mxfp4_quantise(t: torch.Tensor) -> MXFP4:
    """The rows of `t` ([rows, columns], bf16, fp16 or fp32) in MXFP4, in blocks of 32 columns (ffnk_mxfp4_quantise): the scale is the
    largest power of two not above the block's largest magnitude, over 4; elements go to the nearest number, ties to the even code,
    and saturate at 6.  A block with an infinity or a NaN is NaN.  The result carries no gradient."""
    if _tracing():
        _refuse_tracer("mxfp4_quantise", t)
    result = _native().mx_quantise(t)
    if result is not NotImplemented:
        return result
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"t must be a torch.Tensor, got {type(t).__name__}")
    if t.dim() != 2 or t.dtype not in _DTYPES:
        raise ValueError(f"t must be a 2-D bf16, fp16 or fp32 tensor, got {t.dtype} {tuple(t.shape)}")
    if not t.is_cuda:
        raise ValueError(f"t must live on a GPU (got {t.device}); libffnk has no CPU path")
    t = _dense_rows(t.detach())
    rows, columns = t.shape
    with _on_device(t.device):
        with torch.inference_mode(False):  # (a backward can keep what was quantised ahead of it in any mode)
            codes = torch.empty((rows, _code_bytes(columns)), dtype=torch.uint8, device=t.device)
            scales = torch.empty(_scale_shape(rows, columns), dtype=torch.uint8, device=t.device)
        q = MXFP4._whole(codes, scales, columns)
        _lib.check(_lib.load().ffnk_mxfp4_quantise(t.data_ptr(), _DTYPES[t.dtype], _row_stride(t), q._address, rows, columns,
                                                   _stream_ptr(t.device)), "ffnk_mxfp4_quantise")
    return q


def mxfp4_dequantise(q: MXFP4, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values that `q` stands for, as a [rows, columns] tensor of bf16 (exact for normal numbers), fp16 or fp32."""
    if _tracing():
        _refuse_tracer("mxfp4_dequantise")
    result = _native().mx_dequantise(q, dtype)
    if result is not NotImplemented:
        return result
    _require_mxfp4("q", q)
    if dtype not in _DTYPES:
        raise ValueError(f"dtype must be bf16, fp16 or fp32, got {dtype}")
    rows, columns = q.shape
    with _on_device(q.device):
        t = torch.empty((rows, columns), dtype=dtype, device=q.device)
        _lib.check(_lib.load().ffnk_mxfp4_dequantise(q._address, t.data_ptr(), _DTYPES[dtype], max(columns, 1), rows, columns,
                                                     _stream_ptr(q.device)), "ffnk_mxfp4_dequantise")
    return t


def _mx_workspace(op: int, M: int, K: int, N: int, dev: torch.device) -> torch.Tensor:
    n = _lib.load().ffnk_mxfp4_workspace_bytes(op, M, K, N)
    if n == ctypes.c_size_t(-1).value:
        raise ValueError(f"ffnk_mxfp4_workspace_bytes: invalid op/extents op={op} M={M} K={K} N={N}")
    return _workspace(n, dev)


def _rows_of_call(a):
    """(a as the kernels take it, address of its bf16 rows, their stride, address of its MXFP4 struct): one of the two is there."""
    if isinstance(a, MXFP4):
        return a, None, 0, a._address
    _require_cuda_bf16("a", a, 2)
    a = _dense_rows(a)
    return a, a.data_ptr(), _row_stride(a), None


def _check_weights(K: int, dev, shape, **weights) -> None:
    for name, w in weights.items():
        _require_mxfp4(name, w)
        if w.shape != shape:
            raise ValueError(f"{name} shape {w.shape} != {shape}")
    _same_device(dev, **weights)


def _reach(rows: int, stride: int, columns: int) -> bool:
    """Whether the 32-bit offsets of the backward GEMMs span `rows` of the upstream gradient, the last one filled up to 64 columns."""
    return 2 * (max(rows, 256) * stride + -columns % 64) < 1 << 32


def _check_differentiable(rows: int, contraction: int, *extents: int, doubled: int = 0) -> None:
    """What the backward GEMMs over dequantised weights take; `contraction`: the layer's output features; doubled: the intermediate's."""
    if any(e % 8 for e in (contraction, *extents, doubled)) or (contraction % 64 and contraction < 128):
        raise ValueError(f"the MXFP4 backward needs extents that are multiples of 8 and output features that are a multiple of 64 or at "
                         f"least 128, got {(contraction, *extents, *([doubled] if doubled else []))}")
    if not _reach(0, contraction, contraction) or not _reach(0, 2 * (doubled + -doubled % 64), 0):
        raise ValueError(f"the MXFP4 backward has no extents as large as {max(contraction, doubled)}")
    if not _reach(rows, contraction, contraction):
        raise ValueError(f"the MXFP4 backward reaches 4 GiB of upstream gradient, {rows} rows of {contraction} columns pass it: split the rows")


def masked_linear_mxfp4_forward(a, b1: MXFP4, b2: MXFP4, mask: torch.Tensor, routing: Routing | None = None) -> torch.Tensor:
    """c[m] = Q(a[m]) @ (b1 if mask[m] else b2)^T.  a: bf16 [M, K] or MXFP4; b1, b2: MXFP4 [N, K]; routing: as in
    masked_linear_forward."""
    result = _native().mx_linear_fwd(a, b1, b2, mask, routing)
    if result is not NotImplemented:
        return result
    a, x, ld, xq = _rows_of_call(a)
    M, K = a.shape
    dev = a.device
    _require_mxfp4("b1", b1)
    N = b1.rows
    _check_weights(K, dev, (N, K), b1=b1, b2=b2)
    mask = _require_mask(mask, M, dev)
    with _on_device(dev):
        c = torch.empty((M, N), device=dev, dtype=torch.bfloat16)
        if M == 0 or N == 0 or K == 0:
            return c.zero_()
        stream = _stream_ptr(dev)
        routing, rt = _routing_arg(routing, mask, M, stream)
        ws = _mx_workspace(_lib.OP_LINEAR_FWD, M, K, N, dev)
        rc = _lib.load().ffnk_mxfp4_linear_fwd(x, ld, xq, b1._address, b2._address, mask.data_ptr(), c.data_ptr(), N, M, K, N, ws.data_ptr(),
                                               ws.numel(), stream, rt, 1)
    _lib.check(rc, "ffnk_mxfp4_linear_fwd")
    return c


def masked_linear_mxfp4_backward(grad: torch.Tensor, b1: MXFP4, b2: MXFP4, mask: torch.Tensor, routing: Routing | None = None) -> torch.Tensor:
    """da[m] = grad[m] @ (b1 if mask[m] else b2): the gradient of the rows over constant weights."""
    result = _native().mx_linear_bwd(grad, b1, b2, mask, routing)
    if result is not NotImplemented:
        return result
    _require_cuda_bf16("grad", grad, 2)
    _require_mxfp4("b1", b1)
    M, dev = grad.shape[0], grad.device
    N, K = b1.shape
    if grad.shape != (M, N):
        raise ValueError(f"grad shape {tuple(grad.shape)} != {(M, N)}")
    _check_weights(K, dev, (N, K), b1=b1, b2=b2)
    _check_differentiable(M, N, K)
    mask = _require_mask(mask, M, dev)
    grad = _aligned_rows(grad)
    with _on_device(dev):
        da = torch.empty((M, K), device=dev, dtype=torch.bfloat16)
        if M == 0 or K == 0 or N == 0:
            return da.zero_()
        stream = _stream_ptr(dev)
        routing, rt = _routing_arg(routing, mask, M, stream)
        ws = _mx_workspace(_lib.OP_LINEAR_BWD, M, K, N, dev)
        rc = _lib.load().ffnk_mxfp4_linear_bwd(grad.data_ptr(), _row_stride(grad), b1._address, b2._address, mask.data_ptr(), da.data_ptr(), K,
                                               M, K, N, ws.data_ptr(), ws.numel(), stream, rt)
    _lib.check(rc, "ffnk_mxfp4_linear_bwd")
    return da


def _aligned_rows(t: torch.Tensor) -> torch.Tensor:
    """Rows of a multiple of 8 columns that the direct kernels load as they are; others are copied, also those too far apart for them."""
    t = _dense_rows(t)
    if _row_stride(t) % 8 == 0 and t.data_ptr() % 16 == 0 and _reach(t.shape[0], _row_stride(t), t.shape[1]):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _check_ffn(a_shape, dev, w1, w2, w3, u1, u2, u3):
    d = a_shape[1]
    _require_mxfp4("w1", w1)
    h = w1.rows
    _check_weights(d, dev, (h, d), w1=w1, w3=w3, u1=u1, u3=u3)
    _check_weights(h, dev, (d, h), w2=w2, u2=u2)
    return d, h


def masked_ffn_mxfp4_forward(a, w1: MXFP4, w2: MXFP4, w3: MXFP4, u1: MXFP4, u2: MXFP4, u3: MXFP4, mask: torch.Tensor, save_pre: bool = False,
                             routing: Routing | None = None):
    """Q(silu(Q(a) @ w1^T) * (Q(a) @ w3^T)) @ w2^T for rows with mask, u1, u2, u3 for the others.  a: bf16 [M, d] or MXFP4;
    w1, w3, u1, u3: MXFP4 [h, d]; w2, u2: MXFP4 [d, h].

    save_pre: also return both projections, fp32 [M, 2h] in routed order (gate | up), for masked_ffn_mxfp4_backward."""
    result = _native().mx_ffn_fwd(a, w1, w2, w3, u1, u2, u3, mask, bool(save_pre), routing)
    if result is not NotImplemented:
        return result
    a, x, ld, xq = _rows_of_call(a)
    M, dev = a.shape[0], a.device
    d, h = _check_ffn(a.shape, dev, w1, w2, w3, u1, u2, u3)
    mask = _require_mask(mask, M, dev)
    with _on_device(dev):
        out = torch.empty((M, d), device=dev, dtype=torch.bfloat16)
        pre = torch.empty((M, 2 * h), device=dev, dtype=torch.float32) if save_pre else None
        if M == 0 or d == 0 or h == 0:
            return (out.zero_(), pre) if save_pre else out.zero_()
        stream = _stream_ptr(dev)
        routing, rt = _routing_arg(routing, mask, M, stream)
        ws = _mx_workspace(_lib.OP_FFN_FWD, M, d, h, dev)
        rc = _lib.load().ffnk_mxfp4_ffn_fwd(x, ld, xq, w1._address, w2._address, w3._address, u1._address, u2._address, u3._address, mask.data_ptr(),
                                            out.data_ptr(), d, pre.data_ptr() if save_pre else None, M, d, h, ws.data_ptr(), ws.numel(), stream, rt,
                                            1)
    _lib.check(rc, "ffnk_mxfp4_ffn_fwd")
    return (out, pre) if save_pre else out


def masked_ffn_mxfp4_backward(grad: torch.Tensor, w1: MXFP4, w2: MXFP4, w3: MXFP4, u1: MXFP4, u2: MXFP4, u3: MXFP4, mask: torch.Tensor,
                              pre: torch.Tensor, routing: Routing | None = None) -> torch.Tensor:
    """Gradient of the rows over constant weights: dh = grad @ w2, da = (dh * up * silu'(gate)) @ w1 + (dh * silu(gate)) @ w3, with the
    projections that masked_ffn_mxfp4_forward(..., save_pre=True) returned for the same mask."""
    result = _native().mx_ffn_bwd(grad, w1, w2, w3, u1, u2, u3, mask, pre, routing)
    if result is not NotImplemented:
        return result
    _require_cuda_bf16("grad", grad, 2)
    M, dev = grad.shape[0], grad.device
    d, h = _check_ffn(grad.shape, dev, w1, w2, w3, u1, u2, u3)
    _check_differentiable(M, d, doubled=h)
    mask = _require_mask(mask, M, dev)
    if not isinstance(pre, torch.Tensor):
        raise TypeError(f"pre must be a torch.Tensor, got {type(pre).__name__}")
    if pre.dtype != torch.float32 or pre.shape != (M, 2 * h) or pre.device != dev or not pre.is_contiguous() or pre.data_ptr() % 16:
        raise ValueError(f"pre must be a contiguous, 16-byte aligned fp32 [{M}, {2 * h}] tensor on {dev}")
    grad = _aligned_rows(grad)
    with _on_device(dev):
        da = torch.empty((M, d), device=dev, dtype=torch.bfloat16)
        if M == 0 or d == 0 or h == 0:
            return da.zero_()
        stream = _stream_ptr(dev)
        routing, rt = _routing_arg(routing, mask, M, stream)
        ws = _mx_workspace(_lib.OP_FFN_BWD, M, d, h, dev)
        rc = _lib.load().ffnk_mxfp4_ffn_bwd(grad.data_ptr(), _row_stride(grad), w1._address, w2._address, w3._address, u1._address, u2._address,
                                            u3._address, mask.data_ptr(), pre.data_ptr(), da.data_ptr(), d, M, d, h, ws.data_ptr(), ws.numel(),
                                            stream, rt)
    _lib.check(rc, "ffnk_mxfp4_ffn_bwd")
    return da


def _nothing_to_record(a) -> bool:
    """Whether a forward can do without Function.apply, a third of a short call's host time.  Not where a gradient of `a` is wanted, nor where
    a tracer takes the call down (it would keep the result's allocation alone), `a` carries a forward-mode derivative or belongs to a
    function transform (which Function.apply refuses)."""
    if torch.is_grad_enabled() and isinstance(a, torch.Tensor) and a.requires_grad or _tracing():
        return False
    if forward_ad._current_level < 0 and not _transforms_active() or not isinstance(a, torch.Tensor):
        return True
    return not torch._C._functorch.is_functorch_wrapped_tensor(a) and (forward_ad._current_level < 0 or forward_ad.unpack_dual(a).tangent is None)


def _save(ctx, weights, *tensors) -> None:
    """For the backward: the weights' memory too, so that autograd refuses one over weights that were changed in place since."""
    ctx.save_for_backward(*(t for w in weights for t in (w.codes, w.scales)), *tensors)
    ctx.weights = weights


def _saved(ctx) -> tuple:
    """(weights, tensors) as _save got them; hooks on saved tensors may have put others in the weights' place."""
    held, weights = ctx.saved_tensors, ctx.weights
    pairs = [(w, held[2 * i], held[2 * i + 1]) for i, w in enumerate(weights)]
    if any(codes is not w._codes or scales is not w._scales for w, codes, scales in pairs):
        weights = tuple(MXFP4._whole(codes, scales, w.columns) for w, codes, scales in pairs)
    return weights, held[2 * len(weights):]


def _gradient_of_rows(ctx) -> bool:
    """Of a forward under Function.apply, which runs with gradients switched off (ops._grad_mode)."""
    return _grad_mode.enabled and ctx.needs_input_grad[0]


class MaskedLinearMXFP4(Function):
    """c = Q(a) @ (b1 where mask else b2)^T over MXFP4 weights [N, K]; differentiable in a bf16 `a`."""

    @classmethod
    def apply(cls, a, b1, b2, mask):
        if _nothing_to_record(a):
            return masked_linear_mxfp4_forward(a, b1, b2, mask)
        _grad_mode.enabled = torch.is_grad_enabled()
        return super().apply(a, b1, b2, mask)

    @staticmethod
    def forward(ctx, a, b1, b2, mask):
        if not _gradient_of_rows(ctx):
            return masked_linear_mxfp4_forward(a, b1, b2, mask)
        if isinstance(b1, MXFP4):
            _check_differentiable(a.shape[:1].numel(), *b1.shape)
        _route_cache.last = None
        out = masked_linear_mxfp4_forward(a, b1, b2, mask)
        _save(ctx, (b1, b2), mask)
        ctx.routing = _route_cache.last
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        weights, (mask,) = _saved(ctx)
        return masked_linear_mxfp4_backward(grad, *weights, mask, routing=ctx.routing), None, None, None


class MaskedFFNMXFP4(Function):
    """Routed SwiGLU FFN over MXFP4 weights (w1, w3, u1, u3: [h, d]; w2, u2: [d, h]); differentiable in a bf16 `a`, for which the
    forward keeps both projections in fp32: the gradient is rounded at dt1, dt3 and itself only (against 64 bits at d = 4096, h = 14336 off by
    0.0023 of its norm, 0.0017 of it the last rounding; with them and dh in bf16 0.0034)."""

    @classmethod
    def apply(cls, a, w1, w2, w3, u1, u2, u3, mask):
        if _nothing_to_record(a):
            return masked_ffn_mxfp4_forward(a, w1, w2, w3, u1, u2, u3, mask)
        _grad_mode.enabled = torch.is_grad_enabled()
        return super().apply(a, w1, w2, w3, u1, u2, u3, mask)

    @staticmethod
    def forward(ctx, a, w1, w2, w3, u1, u2, u3, mask):
        weights = (w1, w2, w3, u1, u2, u3)
        if not _gradient_of_rows(ctx):
            return masked_ffn_mxfp4_forward(a, *weights, mask)
        if isinstance(w2, MXFP4):
            _check_differentiable(a.shape[:1].numel(), w2.rows, doubled=w2.columns)
        _route_cache.last = None
        out, pre = masked_ffn_mxfp4_forward(a, *weights, mask, save_pre=True)
        _save(ctx, weights, mask, pre)
        ctx.routing = _route_cache.last
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        weights, (mask, pre) = _saved(ctx)
        return (masked_ffn_mxfp4_backward(grad, *weights, mask, pre, routing=ctx.routing), *([None] * 7))
