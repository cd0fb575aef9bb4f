"""A linear layer in 8-bit integers: int8 weight with one scale per output channel, activations quantised per token on the fly.

    y[m, n] = act(sa[m] sw[n] sum_k a8[m, k] w8[n, k] + bias[n]) + residual[m, n]

The counterpart of the `nn.Linear` projections of audiocraft/modules/transformer.py:362-399, 454-574 for serving: a quarter of
the f32 weight's bytes and the int8 rate of the matrix cores.  No gradients.
"""
import typing as tp

import torch
from torch import nn

from .. import _C

_DTYPES = (torch.float32, torch.bfloat16)


class Int8Linear:
    """Built once from a weight [N, K] (nn.Linear layout, f32 or bf16, on the GPU) and an optional bias [N]; the int8 weight is laid
    out for the matrix cores (include/acmi.h, "int8 fragments").  activation: 'none' or 'gelu' (by erf).

    A token (channel) that holds a NaN or an infinity gives NaN in its whole output row (column)."""

    ACTIVATIONS = {'none': 0, 'gelu': 1}

    def __init__(self, weight: torch.Tensor, bias: tp.Optional[torch.Tensor] = None, activation: str = 'none'):
        if weight.dim() != 2 or weight.dtype not in _DTYPES or not weight.is_cuda or 0 in weight.shape:
            raise ValueError(f"Int8Linear: weight {tuple(weight.shape)} {weight.dtype} on {weight.device}: [N, K] float32 or bfloat16 on the GPU")
        if weight.shape[1] > 131072:
            raise ValueError(f"Int8Linear: K {weight.shape[1]} (at most 131072: the 32-bit integer sums)")
        if weight.shape[0] > 1 << 25:
            raise ValueError(f"Int8Linear: N {weight.shape[0]} (at most 2^25)")
        if activation not in self.ACTIVATIONS:
            raise ValueError(f"Int8Linear: activation {activation!r} ({', '.join(self.ACTIVATIONS)})")
        self.out_features, self.in_features = weight.shape
        self.activation, self._act = activation, self.ACTIVATIONS[activation]
        w = weight.detach()
        with _C.device_lock:
            self.codes, self.scale = _C.quantize_rows_i8(w if w.stride(1) == 1 and w.stride(0) >= w.shape[1] else w.contiguous())
        self._index = self.codes.get_device()
        self.bias = None
        if bias is not None:
            if bias.shape != (self.out_features,) or bias.device != weight.device:
                raise ValueError(f"Int8Linear: bias {tuple(bias.shape)} on {bias.device}, expected [{self.out_features}] on {weight.device}")
            self.bias = bias.detach().to(torch.float32, copy=True).contiguous()   # (its own: the weight's codes do not follow the caller's tensors either)

    @classmethod
    def from_linear(cls, linear: nn.Linear, activation: str = 'none') -> 'Int8Linear':
        return cls(linear.weight, linear.bias, activation)

    def __call__(self, x: torch.Tensor, residual: tp.Optional[torch.Tensor] = None) -> torch.Tensor:
        """x [..., K] f32 or bf16 -> [..., N] in x's dtype; residual [..., N] f32 is added last."""
        dt = x.dtype
        if x.dim() == 0 or x.shape[-1] != self.in_features or (dt is not torch.float32 and dt is not torch.bfloat16) or x.get_device() != self._index:
            raise ValueError(f"Int8Linear: x {tuple(x.shape)} {x.dtype} on {x.device}: [..., {self.in_features}] float32 or bfloat16 on {self.codes.device}")
        rows = x if x.dim() == 2 else x.reshape(-1, self.in_features)
        M = rows.shape[0]
        if M > 1 << 30:
            raise ValueError(f"Int8Linear: {M} tokens in one call (at most 2^30)")
        if rows.stride(1) != 1 or (M > 1 and rows.stride(0) < self.in_features):
            rows = rows.contiguous()
        if residual is not None:
            if residual.shape != x.shape[:-1] + (self.out_features,) or residual.dtype != torch.float32 or residual.device != x.device:
                raise ValueError(f"Int8Linear: residual {tuple(residual.shape)} {residual.dtype}, expected float32 {tuple(x.shape[:-1]) + (self.out_features,)}")
            residual = residual.contiguous()
        with _C.device_lock:
            out = torch.empty(M, self.out_features, device=x.device, dtype=dt)
            if M:
                _C.linear_i8(rows, self.codes, self.scale, out, self.bias, residual, self._act)
        return out if x.dim() == 2 else out.view(x.shape[:-1] + (self.out_features,))
