"""nn.Module wrappers around MaskedLinear / MaskedFFN with the parameter names of the reference's
README modules (`TritonLinear`, README.md:60-74 / test_linear.py:52-65; `Triton` FFN, README.md:101-124 /
test_ffn.py:50-72), so that their state_dicts are interchangeable with the reference's PyTorch
`Torch` modules (`linear_v`, `linear_t`; `w1..w3`, `u1..u3`).

Inputs may be 2-D `[M, D]` with mask `[M]` or 3-D `[B, S, D]` with mask `[B, S]`; the modules
flatten and unflatten as the reference's wrappers do.
"""
from __future__ import annotations

import torch
import torch.nn as nn

from .mxfp4 import MXFP4, MaskedFFNMXFP4, MaskedLinearMXFP4, mxfp4_quantise
from .ops import MaskedFFN, MaskedLinear


def _flatten(x: torch.Tensor, mask: torch.Tensor):
    if x.dim() == 3:
        if mask.shape != x.shape[:2]:
            raise ValueError(f"mask shape {tuple(mask.shape)} does not match x {tuple(x.shape)}")
        return x.flatten(0, 1), mask.flatten(0, 1), x.shape[0]
    if x.dim() == 2:
        return x, mask.reshape(-1), None
    raise ValueError(f"x must be [M, D] or [B, S, D], got {tuple(x.shape)}")


def _unflatten(y: torch.Tensor, batch):
    return y if batch is None else y.unflatten(0, (batch, -1))


class MaskedLinearModule(nn.Module):
    """Two bias-free Linear layers, one per modality; rows are routed by `visual_mask`.
    Differentiable (forward + backward), like the reference's `Triton` module of test_linear.py."""

    def __init__(self, in_dim: int, out_dim: int, device=None, dtype=torch.bfloat16):
        super().__init__()
        self.linear_v = nn.Linear(in_dim, out_dim, bias=False, device=device, dtype=dtype)
        self.linear_t = nn.Linear(in_dim, out_dim, bias=False, device=device, dtype=dtype)

    def forward(self, x: torch.Tensor, visual_mask: torch.Tensor) -> torch.Tensor:
        x2, m, batch = _flatten(x, visual_mask)
        y = MaskedLinear.apply(x2, self.linear_v.weight.T, self.linear_t.weight.T, m)
        return _unflatten(y, batch)


class MaskedFFNModule(nn.Module):
    """SwiGLU FFN with visual weights (w1, w2, w3) and text weights (u1, u2, u3).  The reference's
    `Triton` module of test_ffn.py / README.md:101-124 runs under no_grad on `.weight.data` because
    its op has no backward; this one passes the parameters themselves, so it trains as well (wrap the
    call in torch.no_grad() for inference, as with any module)."""

    def __init__(self, hidden_size: int, intermediate_size: int, device=None, dtype=torch.bfloat16):
        super().__init__()
        mk = lambda i, o: nn.Linear(i, o, bias=False, device=device, dtype=dtype)
        self.w1, self.w2, self.w3 = mk(hidden_size, intermediate_size), mk(intermediate_size, hidden_size), mk(hidden_size, intermediate_size)
        self.u1, self.u2, self.u3 = mk(hidden_size, intermediate_size), mk(intermediate_size, hidden_size), mk(hidden_size, intermediate_size)

    def forward(self, x: torch.Tensor, mask: torch.Tensor) -> torch.Tensor:
        x2, m, batch = _flatten(x, mask)
        y = MaskedFFN.apply(x2, self.w1.weight.T, self.w2.weight.T, self.w3.weight.T,
                            self.u1.weight.T, self.u2.weight.T, self.u3.weight.T, m)
        return _unflatten(y, batch)


class _MXFP4Weights(nn.Module):
    """Weights held in MXFP4 as buffers (`<name>_codes`, `<name>_scales`): constants that follow the module to a device and into its
    state_dict.  Made from a bf16 module with from_module, or empty (zeros) for load_state_dict."""

    def __init__(self, shapes: dict, device=None):
        super().__init__()
        self._columns = {name: columns for name, (_, columns) in shapes.items()}
        self._held = {}
        for name, (rows, columns) in shapes.items():
            blocks = -(-columns // 32)
            self.register_buffer(f"{name}_codes", torch.zeros((rows, 16 * blocks), dtype=torch.uint8, device=device))
            self.register_buffer(f"{name}_scales", torch.zeros((-(-blocks // 16), rows, 16), dtype=torch.uint8, device=device))

    def _quantise(self, weights: dict) -> None:
        for name, w in weights.items():
            q = mxfp4_quantise(w)
            setattr(self, f"{name}_codes", q.codes)
            setattr(self, f"{name}_scales", q.scales)

    # The MXFP4 objects of a state live as long as it does: they hold its memory.
    def _apply(self, fn, recurse=True):
        self._held = {}
        return super()._apply(fn, recurse)

    def _load_from_state_dict(self, *args, **kwargs):
        self._held = {}
        super()._load_from_state_dict(*args, **kwargs)

    def __getstate__(self):
        return {**super().__getstate__(), "_held": {}}

    def weight(self, name: str) -> MXFP4:
        codes, scales = self._buffers[f"{name}_codes"], self._buffers[f"{name}_scales"]
        held = self._held.get(name)
        if held is None or held.codes is not codes or held.scales is not scales:
            held = self._held[name] = MXFP4(codes, scales, self._columns[name])
        return held


class MaskedLinearMXFP4Module(_MXFP4Weights):
    """MaskedLinearModule over weights in MXFP4; its rows are differentiable, its weights constants."""

    def __init__(self, in_dim: int, out_dim: int, device=None):
        super().__init__({"linear_v": (out_dim, in_dim), "linear_t": (out_dim, in_dim)}, device)

    @classmethod
    def from_module(cls, m: MaskedLinearModule) -> "MaskedLinearMXFP4Module":
        new = cls(m.linear_v.in_features, m.linear_v.out_features, device="meta")
        new._quantise({"linear_v": m.linear_v.weight, "linear_t": m.linear_t.weight})
        return new

    def forward(self, x: torch.Tensor, visual_mask: torch.Tensor) -> torch.Tensor:
        x2, m, batch = _flatten(x, visual_mask)
        return _unflatten(MaskedLinearMXFP4.apply(x2, self.weight("linear_v"), self.weight("linear_t"), m), batch)


class MaskedFFNMXFP4Module(_MXFP4Weights):
    """MaskedFFNModule over weights in MXFP4; its rows are differentiable, its weights constants."""
    _NAMES = ("w1", "w2", "w3", "u1", "u2", "u3")

    def __init__(self, hidden_size: int, intermediate_size: int, device=None):
        up, down = (intermediate_size, hidden_size), (hidden_size, intermediate_size)
        super().__init__({name: down if name[1] == "2" else up for name in self._NAMES}, device)

    @classmethod
    def from_module(cls, m: MaskedFFNModule) -> "MaskedFFNMXFP4Module":
        new = cls(m.w1.in_features, m.w1.out_features, device="meta")
        new._quantise({name: getattr(m, name).weight for name in cls._NAMES})
        return new

    def forward(self, x: torch.Tensor, mask: torch.Tensor) -> torch.Tensor:
        x2, m, batch = _flatten(x, mask)
        return _unflatten(MaskedFFNMXFP4.apply(x2, *(self.weight(name) for name in self._NAMES), m), batch)
