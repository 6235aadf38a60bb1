"""Linear layers in 8-bit integers for inference: a frozen model that scores or writes summaries.

Weights are quantised once, one scale per output channel; activations in every call, one scale per token; the integer sum is exact.
"""
import torch
import torch.nn as nn

from . import kernels as kn


class Int8Linear(nn.Module):
    """y = x W^T (+ bias) (then GELU, erf form) with W [N, K] (f32 or bf16) held as int8 [N, Kp] + one f32 scale per row.  x [..., K] f32 or bf16,
    y [..., N] in out_dtype (default: x's).  A token whose values are not all finite gives NaN.
    Casts of a module around it (.bfloat16(), .to(dtype)) leave its scales and bias f32.  A state dict is loaded by a layer of the same sizes (made from
    zeros, say).  No gradient: inputs that require one, or carry a forward-mode tangent, are refused."""

    def __init__(self, weight, bias=None, gelu=False, out_dtype=None):
        super().__init__()
        if weight.dim() != 2 or 0 in weight.shape:
            raise ValueError("weight: [N, K] expected, got %s" % (tuple(weight.shape),))
        if bias is not None and tuple(bias.shape) != (weight.shape[0],):
            raise ValueError("bias: [%d] expected, got %s" % (weight.shape[0], tuple(bias.shape)))
        if out_dtype not in (None, torch.float32, torch.bfloat16):
            raise TypeError("unsupported dtype %s" % out_dtype)
        self.out_features, self.in_features = weight.shape
        self.gelu, self.out_dtype = bool(gelu), out_dtype
        q, scale = kn.quantize_rows(weight.detach())
        self.register_buffer("qweight", q)
        self.register_buffer("scale", scale)
        self.register_buffer("bias", None if bias is None else bias.detach().to(torch.float32).clone())

    def _apply(self, fn, recurse=True):
        """The weights are 8-bit, scales and bias f32, whatever type the model around them is cast to: only the device follows."""
        kept = {n: t for n, t in self._buffers.items() if t is not None}
        super()._apply(fn, recurse)
        for name, t in kept.items():
            moved = self._buffers[name]
            if moved.dtype != t.dtype:
                self._buffers[name] = t.to(moved.device)
        return self

    @classmethod
    def from_linear(cls, linear, **kw):
        return cls(linear.weight, linear.bias, **kw)

    def forward(self, x):
        if x.requires_grad and torch.is_grad_enabled():
            raise RuntimeError("Int8Linear is for inference: no gradient (use torch.no_grad() or detach the input)")
        kn.no_tangent(x, "Int8Linear")
        K = self.in_features
        if x.dim() < 1 or x.shape[-1] != K:
            raise ValueError("x: [..., %d] expected, got %s" % (K, tuple(x.shape)))
        rows = x if x.dim() == 2 else x.reshape(-1, K)
        if (K > 1 and rows.stride(1) != 1) or (rows.shape[0] > 1 and rows.stride(0) < K):
            rows = rows.contiguous()
        y = kn.linear_i8(rows, self.qweight, self.scale, None, self.bias, self.gelu, self.out_dtype)
        return y if x.dim() == 2 else y.reshape(*x.shape[:-1], self.out_features)
