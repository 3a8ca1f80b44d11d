"""Matrix products in 8-bit integers, with a scale per token and per output channel.

``quantize_rows`` turns rows into int8 codes and one fp32 scale each (weights once,
activations at every call); ``matmul_w8a8`` multiplies activations with such a weight:
the sum over K is exact in int32 and the result is rounded once. ``Int8Linear`` is the
module. The reference only simulates this (its ``quantize_inputs`` path rounds the
activations and multiplies in floating point, pare/layers/linear.py:120-138).
"""

from __future__ import annotations

import torch
import torch.nn as nn

from . import _lib
from .kernels import _DeviceGuard, _raw_stream

_VALUES = {torch.float16: _lib.PMI_F16, torch.bfloat16: _lib.PMI_BF16, torch.float32: _lib.PMI_F32}


def _code_width(K: int) -> int:
    return -(-K // 16) * 16


def _rows(x: torch.Tensor, fn: str) -> torch.Tensor:
    """x after its checks, with contiguous rows."""
    if not x.is_cuda:
        raise RuntimeError(f"{fn} requires HIP (cuda) tensors.")
    assert x.dim() == 2 and x.dtype in _VALUES, (
        f"x must be a float16, bfloat16 or float32 [M, K] tensor, got {x.dtype} {tuple(x.shape)}")
    if x.stride(1) != 1 and x.shape[1] > 1 or (x.shape[0] > 1 and x.stride(0) < x.shape[1]):
        x = x.contiguous()
    return x


def quantize_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes int8 [M, K rounded up to 16], scales fp32 [M]) of x [M, K] (fp16, bf16 or
    fp32): code = round(x * (127 / amax)), scale = amax / 127, amax the row's largest
    |x|; zeros in the codes' last columns past K. A row of zeros has scale 0, one with
    an infinity or NaN such a scale. K <= 131072."""
    x = _rows(x, "quantize_rows")
    M, K = x.shape
    codes = torch.empty(M, _code_width(K), dtype=torch.int8, device=x.device)
    scales = torch.empty(M, dtype=torch.float32, device=x.device)
    with _DeviceGuard(x.device):
        _lib.check(_lib.lib().pmi_quantize_rows(x.data_ptr(), _VALUES[x.dtype], max(x.stride(0), K), codes.data_ptr(),
                                                scales.data_ptr(), M, K, _raw_stream(x.device)),
                   "pmi_quantize_rows")
    return codes, scales


def _check_weight(x: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor, bias: torch.Tensor | None, K: int) -> int:
    dev = x.device
    assert w.dim() == 2 and w.dtype == torch.int8 and w.is_contiguous() and w.shape[1] == _code_width(K), \
        f"w must be a contiguous int8 [N, {_code_width(K)}] tensor (quantize_rows), got {w.dtype} {tuple(w.shape)}"
    N = w.shape[0]
    assert w_scales.dtype == torch.float32 and tuple(w_scales.shape) == (N,) and w_scales.is_contiguous(), \
        f"w_scales must be a contiguous float32 [{N}] tensor"
    if bias is not None:
        assert tuple(bias.shape) == (N,) and bias.dtype in _VALUES, f"bias must be a float [{N}] tensor"
    for name, t in (("w", w), ("w_scales", w_scales), ("bias", bias)):
        if t is not None and t.device != dev:
            raise RuntimeError(f"{name} is on {t.device}, x is on {dev}")
    return N


def _bias_and_out(bias: torch.Tensor | None, out: torch.Tensor | None, M: int, N: int, dtype: torch.dtype,
                  dev: torch.device) -> tuple[torch.Tensor | None, torch.Tensor]:
    if bias is not None:
        bias = bias.to(dtype).contiguous()
    if out is None:
        return bias, torch.empty(M, N, dtype=dtype, device=dev)
    assert out.dtype == dtype and tuple(out.shape) == (M, N) and out.is_contiguous() and out.device == dev, \
        f"out must be a contiguous [{M}, {N}] {dtype} tensor on {dev}"
    return bias, out


def matmul_int8(codes: torch.Tensor, scales: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor, K: int,
                dtype: torch.dtype, *, bias: torch.Tensor | None = None,
                out: torch.Tensor | None = None) -> torch.Tensor:
    """y [M, N] of ``dtype`` (fp16, bf16 or fp32) = (codes . w^T) * scales[:, None] * w_scales
    (+ bias) of rows that ``quantize_rows`` made from K columns: for one input of several
    products. ``matmul_w8a8`` quantises and multiplies."""
    if not codes.is_cuda:
        raise RuntimeError("matmul_int8 requires HIP (cuda) tensors.")
    assert dtype in _VALUES, "dtype must be float16, bfloat16 or float32"
    assert codes.dim() == 2 and codes.dtype == torch.int8 and codes.is_contiguous() and \
        codes.shape[1] == _code_width(K), f"codes must be a contiguous int8 [M, {_code_width(K)}] tensor"
    M = codes.shape[0]
    assert scales.dtype == torch.float32 and tuple(scales.shape) == (M,) and scales.is_contiguous() and \
        scales.device == codes.device, f"scales must be a contiguous float32 [{M}] tensor on {codes.device}"
    N = _check_weight(codes, w, w_scales, bias, K)
    dev = codes.device
    bias, out = _bias_and_out(bias, out, M, N, dtype, dev)
    with _DeviceGuard(dev):
        _lib.check(_lib.lib().pmi_matmul_w8a8(
            codes.data_ptr(), scales.data_ptr(), w.data_ptr(), w_scales.data_ptr(),
            bias.data_ptr() if bias is not None else None, out.data_ptr(), _VALUES[dtype], M, N, K,
            _raw_stream(dev)), "pmi_matmul_w8a8")
    return out


def matmul_w8a8(x: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor, *, bias: torch.Tensor | None = None,
                out: torch.Tensor | None = None) -> torch.Tensor:
    """y [M, N] = x [M, K] @ W^T (+ bias) in 8-bit integers, of x's type (fp16, bf16 or
    fp32): x is quantised row by row, ``w`` and ``w_scales`` are ``quantize_rows`` of the
    weight [N, K]. RuntimeError when x is not on a HIP device, AssertionError on layout
    violations."""
    x = _rows(x, "matmul_w8a8")
    M, K = x.shape
    dev = x.device
    N = _check_weight(x, w, w_scales, bias, K)
    bias, out = _bias_and_out(bias, out, M, N, x.dtype, dev)
    scratch = torch.empty(M * (_code_width(K) + 4), dtype=torch.int8, device=dev)
    with _DeviceGuard(dev):
        _lib.check(_lib.lib().pmi_matmul_w8a8_rows(
            x.data_ptr(), _VALUES[x.dtype], max(x.stride(0), K), w.data_ptr(), w_scales.data_ptr(),
            bias.data_ptr() if bias is not None else None, out.data_ptr(), M, N, K, scratch.data_ptr(),
            scratch.numel(), _raw_stream(dev)), "pmi_matmul_w8a8_rows")
    return out


class Int8Linear(nn.Module):
    """A linear layer in 8-bit integers: weights quantised once per output channel,
    activations per token at every call. Buffers ``weight`` int8 [out, in rounded up to
    16], ``scale`` fp32 [out], which both keep their types when the module is converted
    (``half()``, ``to(dtype)``); ``bias`` optional. Runs on the HIP device only, and forward only: the
    bias takes no gradient, and an input that needs one is refused."""

    def __init__(self, weight: torch.Tensor, scale: torch.Tensor, in_features: int,
                 bias: torch.Tensor | None = None) -> None:
        super().__init__()
        if weight.dtype != torch.int8 or weight.dim() != 2 or weight.shape[1] != _code_width(in_features):
            raise ValueError(f"weight must be int8 [out, {_code_width(in_features)}]")
        if tuple(scale.shape) != (weight.shape[0],):
            raise ValueError(f"scale must be [{weight.shape[0]}]")
        self.in_features = in_features
        self.out_features = weight.shape[0]
        self.register_buffer("weight", weight.contiguous())
        self.register_buffer("scale", scale.float())
        self.bias = nn.Parameter(bias.detach().clone(), requires_grad=False) if bias is not None else None

    def _apply(self, fn, recurse=True):
        # conversions of a model's floating-point tensors reach the scale as well: fp16 would round it,
        # and lose what lies under 2^-24
        scale = self.scale
        super()._apply(fn, recurse)
        if self.scale.dtype != torch.float32:
            self.scale = scale.to(self.scale.device)
        return self

    @classmethod
    def from_weight(cls, weight: torch.Tensor, bias: torch.Tensor | None = None) -> "Int8Linear":
        """Quantises a weight [out, in]; one on the CPU on the current HIP device, and the
        buffers are returned on the weight's device."""
        w = weight.detach()
        home = w.device
        codes, scale = quantize_rows(w if w.is_cuda else w.to("cuda"))
        return cls(codes.to(home), scale.to(home), w.shape[1], bias)

    @classmethod
    def from_linear(cls, linear: nn.Linear) -> "Int8Linear":
        return cls.from_weight(linear.weight, linear.bias)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if not x.is_cuda:
            raise RuntimeError("pare_amd.Int8Linear runs on the HIP device only (no CPU fallback); move the module "
                               "and input to cuda")
        if x.requires_grad and torch.is_grad_enabled():
            raise RuntimeError("pare_amd.Int8Linear has no backward pass: detach the input or call it under no_grad, "
                               "its gradient would be left out")
        y = matmul_w8a8(x.reshape(-1, self.in_features), self.weight, self.scale, bias=self.bias)
        return y.reshape(*x.shape[:-1], self.out_features)

    def extra_repr(self) -> str:
        return f"in={self.in_features}, out={self.out_features}, dtype=INT8, bias={self.bias is not None}"
