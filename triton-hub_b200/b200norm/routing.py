"""Choice of experts from router logits on libb200norm.so: softmax, the k likeliest experts of each token,
how many tokens chose each expert, and the balance loss, with gradients.

    p = softmax(logits);  gates: p of the chosen, or (normalize) their share of the chosen p
    f_e = counts_e / (n k),  P_e = mean p_e over the n live tokens,  loss = E * sum_e f_e P_e   (1 when balanced)

The gradient reaches the logits through the gates and through P; f is a count.  Ties go to the lower index.
"""
from __future__ import annotations

from functools import lru_cache
from operator import index as as_int

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .functional import _code, _flat, _on_device, _ptr, _raw_stream, _require_cuda, _unrecorded


@lru_cache(maxsize=4096)  # the answer never changes; of as many sizes as a program meets in turn, not of all it ever met
def _workspace_bytes(index, T, E, k, code):
    """Bytes of the forward's workspace, 1 for none; `index` is the current device."""
    n = _lib.load().b200norm_route_workspace_bytes(T, E, k, code)
    if n == 0:
        _lib.check(_lib.ERR_ARG)
    return n


def _route_fwd(logits, k, normalize=True, mask=None, *, need_lse=True, keep=False):
    """Returns (gates fp32 (..., k), experts int32 (..., k), counts int32 (E + 1,) whose last is the number of live
    tokens, loss fp32 scalar, lse fp32 (T,) or None).  `keep`: lse is int32 (T + E + 1,), the bits of its values and behind
    them the counts once more, for a backward whose caller gives `counts` away."""
    _require_cuda(logits)
    if logits.dtype == torch.float64:
        raise RuntimeError("b200norm: router logits of dtype torch.float64 are not supported (float32, float16, bfloat16)")
    shape, device = logits.shape[:-1], logits.device
    code = _code(logits, "router logits")
    if mask is not None:
        if mask.shape != shape or mask.device != device or mask.dtype not in (torch.bool, torch.uint8):
            raise RuntimeError(f"b200norm: mask is bool, one value a token, of shape {tuple(shape)} on {device}; got "
                               f"{tuple(mask.shape)} of {mask.dtype} on {mask.device}")
        mask = mask.contiguous()
    x, T, E, xs = _flat(logits)
    k = as_int(k)
    gates = torch.empty(*shape, k, dtype=torch.float32, device=device)
    experts = torch.empty(*shape, k, dtype=torch.int32, device=device)
    counts = torch.empty(E + 1, dtype=torch.int32, device=device)
    loss = gates.new_empty(())
    lse = None
    if keep:  # whole numbers, lest a hook on saved tensors should round them
        lse = torch.empty(T + E + 1, dtype=torch.int32, device=device)
    elif need_lse:
        lse = torch.empty(T, dtype=torch.float32, device=device)
    lib = _lib.load()
    index = device.index
    with _on_device(index):
        ws_bytes = _workspace_bytes(index, T, E, k, code)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=device) if ws_bytes > 1 else None
        _lib.check(lib.b200norm_route_fwd_kept(
            x.data_ptr(), xs, _ptr(mask), gates.data_ptr(), experts.data_ptr(), _ptr(lse), counts.data_ptr(),
            lse.data_ptr() + 4 * T if keep else None, loss.data_ptr(), _ptr(ws), ws_bytes, T, E, k, int(bool(normalize)), code,
            _raw_stream(index)))
    return gates, experts, counts, loss, lse


def _route_bwd(logits, gates, experts, counts, lse, dgates, dloss, normalize=True):
    """Gradients of (gates, loss), either of which may be None, with respect to the logits.  counts None: those that
    _route_fwd kept behind lse."""
    _require_cuda(logits)
    k = experts.shape[-1]
    x, T, E, xs = _flat(logits)
    dgs = k
    for t in (dgates, dloss):
        if t is not None and t.device != logits.device:
            raise RuntimeError(f"b200norm: gradient on {t.device}, router logits on {logits.device}")
    if dgates is not None:
        assert dgates.shape == experts.shape, 'expect input and output shape to be the same'
        dgates, _, _, dgs = _flat(dgates if dgates.dtype == torch.float32 else dgates.to(torch.float32))
    if dloss is not None and dloss.dtype != torch.float32:
        dloss = dloss.to(torch.float32)
    dlogits = torch.empty_like(logits) if x is logits else torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    lib = _lib.load()
    index = logits.device.index
    with _on_device(index):
        _lib.check(lib.b200norm_route_bwd(
            x.data_ptr(), xs, gates.data_ptr(), experts.data_ptr(), lse.data_ptr(),
            lse.data_ptr() + 4 * T if counts is None else counts.data_ptr(), _ptr(dgates), dgs, _ptr(dloss), dlogits.data_ptr(),
            T, E, k, int(bool(normalize)), _code(x, "router logits"), _raw_stream(index)))
    return dlogits


class route(torch.autograd.Function):
    """(logits (..., E), k, normalize, mask or None) -> (gates (..., k) fp32, experts (..., k) int32, counts (E,) int32,
    loss fp32 scalar).  E up to 1024, k up to 32.  mask: bool, one value a token; tokens whose mask is False, and
    tokens all of whose logits are -inf, choose nothing: experts -1, gates 0, no count, no gradient.  So do the slots
    left over when fewer than k logits of a token are above -inf.  A NaN among a live token's logits makes its gates
    and the loss NaN.  A gate is good to (60 + 1.2 d) 2^-23 of itself, d being its logit's distance from the largest."""

    @classmethod
    def apply(cls, logits, k, normalize=True, mask=None):
        if _unrecorded():  # a decode step's call is spared autograd's bookkeeping
            gates, experts, counts, loss, _ = _route_fwd(logits, k, normalize, mask, need_lse=False)
            return gates, experts, counts[:-1], loss
        return super().apply(logits, k, normalize, mask)

    @staticmethod
    def forward(ctx, logits, k, normalize=True, mask=None):
        # The backward's counts are its own: those that are returned may be summed over ranks, which no version counter tells.
        wanted = ctx.needs_input_grad[0]
        gates, experts, counts, loss, lse = _route_fwd(logits, k, normalize, mask, need_lse=wanted, keep=wanted)
        chosen = counts[:-1]
        ctx.mark_non_differentiable(experts, chosen)
        ctx.set_materialize_grads(False)
        if wanted:
            ctx.save_for_backward(logits, gates, experts, lse)
            ctx.normalize = normalize
        return gates, experts, chosen, loss

    @staticmethod
    @once_differentiable
    def backward(ctx, dgates, _dexperts, _dcounts, dloss):
        if dgates is None and dloss is None:
            return None, None, None, None
        logits, gates, experts, lse = ctx.saved_tensors
        return _route_bwd(logits, gates, experts, None, lse, dgates, dloss, ctx.normalize), None, None, None


class Router:
    """Callable with fixed settings: Router(top_k, normalize)(logits, mask=None) -> (gates, experts, counts, loss),
    see `route`."""

    def __init__(self, top_k, normalize=True):
        self.top_k, self.normalize = top_k, normalize
        self.route_fn = route.apply

    def __call__(self, logits, mask=None):
        return self.route_fn(logits, self.top_k, self.normalize, mask)
