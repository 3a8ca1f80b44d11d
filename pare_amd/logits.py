"""What a serving loop does to the logits before it chooses a token: penalties for repeated
tokens, biases, and masks of the tokens that a grammar allows.

``process_logits`` gives the processed logits, ``greedy_tokens`` only the token with the
largest of each row, in half the bytes. Each row has its own history, penalties, biases and
mask; nothing waits for the device, and both can be captured into a graph. The reference has
no counterpart: its decode is HuggingFace's greedy generate (pare/eval/throughput.py:84-126).
"""

from __future__ import annotations

from typing import NamedTuple

import torch
from torch.autograd import forward_ad

from . import _lib
from .kernels import _DeviceGuard, _raw_stream, _workspace

_VALUES = {torch.float16: _lib.PMI_F16, torch.bfloat16: _lib.PMI_BF16, torch.float32: _lib.PMI_F32}


class LogitRules(NamedTuple):
    """What the rows of a batch have beside their histories, as ``process_logits`` takes it."""

    repetition: torch.Tensor | None = None    # fp32 [R] each
    presence: torch.Tensor | None = None
    frequency: torch.Tensor | None = None
    bias_ids: torch.Tensor | None = None      # int32 and fp32 [R, n]
    bias: torch.Tensor | None = None
    allowed: torch.Tensor | None = None       # int32 [masks, ceil(V / 32)]
    allowed_rows: torch.Tensor | None = None  # int32 [R]


def _tensor(name: str, t: torch.Tensor, dev: torch.device, dtype: torch.dtype, shape: tuple) -> None:
    if t.device != dev:
        raise RuntimeError(f"{name} is on {t.device}, expected {dev}")
    assert t.dtype == dtype and tuple(t.shape) == shape and t.is_contiguous(), (
        f"{name} must be a contiguous {dtype} {list(shape)} tensor, got {t.dtype} {list(t.shape)}")


def _rows(name: str, t: torch.Tensor) -> int:
    """The row stride of a tensor with contiguous rows that do not overlap."""
    assert t.shape[1] <= 1 or t.stride(1) == 1, f"{name} must have contiguous rows"
    assert t.shape[0] <= 1 or t.stride(0) >= t.shape[1], f"the rows of {name} may not overlap"
    return max(t.stride(0), t.shape[1])


def _arguments(fn, logits, history, history_lens, prompt_lens, repetition, presence, frequency, bias_ids, bias,
               allowed, allowed_rows):
    """The arguments of the entry points up to the rows' masks, after their checks."""
    if not logits.is_cuda:
        raise RuntimeError(f"{fn} requires HIP (cuda) tensors.")
    dev = logits.device
    assert logits.dim() == 2 and logits.dtype in _VALUES, (
        f"logits must be a float16, bfloat16 or float32 [R, V] tensor, got {logits.dtype} {list(logits.shape)}")
    R, V = logits.shape
    L = history_stride = n_bias = masks = words = 0
    if history is not None:
        if history.device != dev:
            raise RuntimeError(f"history is on {history.device}, expected {dev}")
        assert history.dtype == torch.int32 and history.dim() == 2 and history.shape[0] == R, (
            f"history must be an int32 [{R}, L] tensor")
        L, history_stride = history.shape[1], _rows("history", history)
    for name, t in (("history_lens", history_lens), ("prompt_lens", prompt_lens)):
        if t is not None:
            assert history is not None, f"{name} needs a history"
            _tensor(name, t, dev, torch.int32, (R,))
    for name, t in (("repetition", repetition), ("presence", presence), ("frequency", frequency)):
        if t is not None:
            assert history is not None, f"{name} needs a history"
            _tensor(name, t, dev, torch.float32, (R,))
    assert (bias_ids is None) == (bias is None), "bias_ids and bias come together"
    if bias_ids is not None:
        assert bias_ids.dim() == 2, f"bias_ids must be an int32 [{R}, n] tensor"
        n_bias = bias_ids.shape[1]
        _tensor("bias_ids", bias_ids, dev, torch.int32, (R, n_bias))
        _tensor("bias", bias, dev, torch.float32, (R, n_bias))
    if allowed is not None:
        words = -(-V // 32)
        assert allowed.dim() == 2 and (allowed_rows is not None or allowed.shape[0] == R), (
            f"allowed must be an int32 [masks, {words}] tensor, one mask a row without allowed_rows")
        masks = allowed.shape[0]
        _tensor("allowed", allowed, dev, torch.int32, (masks, words))
    if allowed_rows is not None:
        assert allowed is not None, "allowed_rows needs allowed"
        _tensor("allowed_rows", allowed_rows, dev, torch.int32, (R,))

    def at(t):
        return t.data_ptr() if t is not None else None

    return [logits.data_ptr(), _VALUES[logits.dtype], _rows("logits", logits), at(history), history_stride, L,
            at(history_lens), at(prompt_lens), at(repetition), at(presence), at(frequency), at(bias_ids), at(bias),
            n_bias, at(allowed), masks, words, at(allowed_rows)]


def _host(greedy, logits, *rest):
    """The call through the host extension, or None where it is not a plain one: the general path then
    takes it."""
    if not logits.is_cuda:
        return None
    dev = torch._C._cuda_getDevice()
    stream = torch._C._cuda_getCurrentRawStream(dev)
    return _lib.host().logits(greedy, logits, *rest, dev, stream,
                              lambda nbytes: _workspace(logits.device, stream, nbytes))


def _no_gradient(**tensors: torch.Tensor | None) -> None:
    """Refuses tensors whose gradient or tangent would be left out."""
    for name, t in tensors.items():
        if t is None:
            continue
        if t.requires_grad and torch.is_grad_enabled():
            raise RuntimeError(f"process_logits has no backward pass: detach {name} or call it under no_grad, the "
                               "gradient would be left out")
        if forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError(f"process_logits has no forward-mode derivative: the tangent of {name} would be left out")


def process_logits(logits: torch.Tensor, *, history: torch.Tensor | None = None,
                   history_lens: torch.Tensor | None = None, prompt_lens: torch.Tensor | None = None,
                   repetition: torch.Tensor | None = None, presence: torch.Tensor | None = None,
                   frequency: torch.Tensor | None = None, bias_ids: torch.Tensor | None = None,
                   bias: torch.Tensor | None = None, allowed: torch.Tensor | None = None,
                   allowed_rows: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Logits [R, V] (fp16, bf16 or fp32, contiguous rows) with, in this order and in fp32:

    - x / ``repetition[r]`` where x > 0, else x * ``repetition[r]``, for the tokens of the row's
      history: the first ``history_lens[r]`` (int32 [R], default all) of ``history`` int32 [R, L]
      (L < 2^30; a count past 2^24 is rounded to fp32);
    - x - ``frequency[r]`` * c - ``presence[r]`` for tokens that are c > 0 times in it behind the
      first ``prompt_lens[r]`` (int32 [R], default 0);
    - x + ``bias[r, i]`` for token ``bias_ids[r, i]`` (int32 and fp32 [R, n]; a token's biases
      are added up first);
    - -inf for tokens that the row's mask does not allow: bit t % 32 of word t / 32 of
      ``allowed[allowed_rows[r]]`` (int32 [masks, ceil(V / 32)]; default: mask r), whatever the logit
      is; a row without such a mask (-1) allows all.

    The penalties are fp32 [R], each optional. Tokens outside 0 .. V - 1 are skipped (-1: none).
    Rounded once. ``out`` may be ``logits``, or a tensor that shares no value with them. Logits, penalties,
    biases and an ``out`` that need a gradient are refused, and so are forward-mode tangents."""
    y = _host(False, logits, history, history_lens, prompt_lens, repetition, presence, frequency, bias_ids, bias,
              allowed, allowed_rows, out)
    if y is not None:
        return y if out is None else out
    _no_gradient(logits=logits, repetition=repetition, presence=presence, frequency=frequency, bias=bias, out=out)
    args = _arguments("process_logits", logits, history, history_lens, prompt_lens, repetition, presence, frequency,
                      bias_ids, bias, allowed, allowed_rows)
    R, V = logits.shape
    dev = logits.device
    if out is None:
        out = torch.empty(R, V, dtype=logits.dtype, device=dev)
    else:
        if out.device != dev:
            raise RuntimeError(f"out is on {out.device}, expected {dev}")
        assert out.dtype == logits.dtype and tuple(out.shape) == (R, V), (
            f"out must be a {logits.dtype} [{R}, {V}] tensor")
    with _DeviceGuard(dev):
        _lib.check(_lib.lib().pmi_process_logits(*args, out.data_ptr(), _rows("out", out), R, V, _raw_stream(dev)),
                   "pmi_process_logits")
    return out


def greedy_tokens(logits: torch.Tensor, *, history: torch.Tensor | None = None,
                  history_lens: torch.Tensor | None = None, prompt_lens: torch.Tensor | None = None,
                  repetition: torch.Tensor | None = None, presence: torch.Tensor | None = None,
                  frequency: torch.Tensor | None = None, bias_ids: torch.Tensor | None = None,
                  bias: torch.Tensor | None = None, allowed: torch.Tensor | None = None,
                  allowed_rows: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """The token (int64 [R]) with the largest of each row of ``process_logits``, of the same
    arguments, without writing those: the lowest token of equal ones, NaN above all numbers, token 0
    where the mask allows nothing. ``out``: int64 with R elements at a constant stride (such as a [R, 1]
    buffer of tokens). At most 16384 rows."""
    y = _host(True, logits, history, history_lens, prompt_lens, repetition, presence, frequency, bias_ids, bias,
              allowed, allowed_rows, out)
    if y is not None:
        return y if out is None else out
    args = _arguments("greedy_tokens", logits, history, history_lens, prompt_lens, repetition, presence, frequency,
                      bias_ids, bias, allowed, allowed_rows)
    R, V = logits.shape
    dev = logits.device
    if out is None:
        out = torch.empty(R, dtype=torch.int64, device=dev)
    else:
        if out.device != dev:
            raise RuntimeError(f"out is on {out.device}, expected {dev}")
        assert out.dtype == torch.int64 and out.numel() == R and out.dim() >= 1 and out.shape[0] == R, (
            f"out must be an int64 tensor of {R} rows with one element each")
    stride = out.stride(0) if R > 1 else 1
    assert stride >= 1, "the elements of out may not overlap"
    L = _lib.lib()
    with _DeviceGuard(dev):
        stream = _raw_stream(dev)
        ws = _workspace(dev, stream, L.pmi_greedy_tokens_workspace_bytes(R, V, _VALUES[logits.dtype]))
        _lib.check(L.pmi_greedy_tokens(*args, out.data_ptr(), stride, R, V, ws.data_ptr() if ws is not None else None,
                                       ws.numel() if ws is not None else 0, stream), "pmi_greedy_tokens")
    return out
