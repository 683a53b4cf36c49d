"""Choice of a token from logits with given random numbers, on libb200norm.so: the step after the softmax
of a language model's head (its probabilities never reach memory).

A row's tokens are ordered by logit, equal ones by index.  Of them are kept: the first `top_k`; of those the
shortest prefix that holds `top_p` of their weight, exp((logit - max) / temperature); of those the ones with
at least `min_p` of the likeliest token's weight.  The token drawn is the lowest index at which the running
sum of the kept weights, in index order, exceeds uniform * total.  The likeliest token always stays.

The drawn token depends on the row and its settings alone, not on the batch around it: weights are summed as
integers.
"""
from __future__ import annotations

from operator import index

import torch

from . import _lib
from .functional import _code, _flat, _on_device, _ptr, _raw_stream, _require_cuda


def _setting(value, name, shape, device, dtype, low, high):
    """-> (tensor of one value a row or None, scalar)."""
    if isinstance(value, torch.Tensor):
        if value.shape != shape or value.device != device:
            raise RuntimeError(f"b200norm: {name} is a number or one value a row, of shape {tuple(shape)} on {device}; got "
                               f"{tuple(value.shape)} on {value.device}")
        if value.dtype == torch.bool or value.is_floating_point() != (dtype == torch.float32):
            raise RuntimeError(f"b200norm: {name} of dtype {value.dtype}")
        if value.dtype in (torch.int64, torch.uint64):  # a larger number means the same as the largest of 32 bits, or as -1
            value = value.view(torch.int64).clamp(-1, 2 ** 31 - 1)
        return value.to(dtype).contiguous(), 0
    if not low <= value <= high:
        raise RuntimeError(f"b200norm: {name} must lie in [{low}, {high}], got {value}")
    return None, float(value) if dtype == torch.float32 else index(value)


def sample(logits, uniform, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Tokens (int64, logits.shape[:-1]) drawn from `logits` (..., V), V up to 262144, float32, float16 or bfloat16.

    uniform: one number in [0, 1) a row.  temperature (0: the likeliest token, the lowest index among equals), top_k
    (0: all), top_p (1: all) and min_p (0: all) are numbers, or tensors of one value a row, whose values are not
    checked: a temperature that is not positive means 0, a top_k outside [1, V) all, a min_p above 1 means 1.
    Logits of -inf are never drawn; those of +inf share the draw among themselves.  A row that holds a NaN, or nothing
    above -inf, gives -1."""
    _require_cuda(logits)
    if logits.dtype == torch.float64:
        raise RuntimeError("b200norm: logits dtype torch.float64 is not supported (float32, float16, bfloat16)")
    shape, device = logits.shape[:-1], logits.device
    code = _code(logits, "logits")
    if uniform.shape != shape or uniform.device != device or not uniform.is_floating_point():
        raise RuntimeError(f"b200norm: uniform holds one number a row, of shape {tuple(shape)} on {device}; got "
                           f"{tuple(uniform.shape)} of {uniform.dtype} on {uniform.device}")
    inf = float("inf")
    t_v, t = _setting(temperature, "temperature", shape, device, torch.float32, 0.0, inf)
    k_v, k = _setting(top_k, "top_k", shape, device, torch.int32, 0, 2 ** 31 - 1)
    p_v, p = _setting(top_p, "top_p", shape, device, torch.float32, 0.0, 1.0)
    m_v, m = _setting(min_p, "min_p", shape, device, torch.float32, 0.0, 1.0)
    tokens = torch.empty(*shape, dtype=torch.int64, device=device) if shape else uniform.new_empty((), dtype=torch.int64)
    u = uniform if uniform.dtype == torch.float32 and uniform.is_contiguous() else uniform.to(torch.float32).contiguous()
    x, M, V, xs = _flat(logits)
    lib = _lib.load()
    with _on_device(device.index):
        _lib.check(lib.b200norm_sample(x.data_ptr(), xs, u.data_ptr(), _ptr(t_v), t, _ptr(k_v), k, _ptr(p_v), p,
                                       _ptr(m_v), m, tokens.data_ptr(), M, V, code, _raw_stream(device.index)))
    return tokens


class Sampler:
    """Callable with fixed settings: Sampler(temperature, top_k, top_p, min_p)(logits, uniform) -> tokens."""

    def __init__(self, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
        self.temperature, self.top_k, self.top_p, self.min_p = temperature, top_k, top_p, min_p

    def __call__(self, logits, uniform):
        return sample(logits, uniform, temperature=self.temperature, top_k=self.top_k, top_p=self.top_p, min_p=self.min_p)
