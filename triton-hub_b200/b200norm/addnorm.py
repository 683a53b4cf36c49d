"""RMSNorm with the residual addition in front of it, and with an 8-bit output behind it, on libb200norm.so.

    add_rmsnorm   h = x + residual;  y = rmsnorm(h) * weight;  returns (y, h)          forward and backward
    rmsnorm_fp8   the same norm (residual optional), y as float8_e4m3fn with scales    forward only

The residual stream (residual, h and their gradients) has x's type or float32.  h is rounded to its type
before the norm, so y is what RMSNorm makes of the h that comes back, and the backward, which reads h, sees
the forward's values.  The reference has neither form; the modules keep RMSNorm's constructor arguments.
"""
from __future__ import annotations

from functools import lru_cache

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from . import functional as Fn
from .functional import _code, _dual_level, _flat, _on_device, _params, _ptr, _raw_stream, _require_cuda, _unrecorded


@lru_cache(maxsize=4096)  # the answer never changes; of as many sizes as a program meets in turn, not of all it ever met
def _workspace_bytes(index, M, N, io, res):
    """Bytes of the backward's workspace; `index` is the current device."""
    n = _lib.load().b200norm_add_rms_bwd_workspace_bytes(M, N, io, res)
    if n == 0:
        _lib.check(_lib.ERR_ARG)
    return n


def _check_residual(x, residual):
    """`residual` goes with x: the same shape and device, a type that is taken."""
    if residual.shape != x.shape:
        raise RuntimeError(f"b200norm: residual of shape {tuple(residual.shape)}, input of shape {tuple(x.shape)}")
    if residual.device != x.device:
        raise RuntimeError(f"b200norm: residual on {residual.device}, input on {x.device}")
    if x.dtype == torch.float64 or residual.dtype not in (x.dtype, torch.float32):
        raise RuntimeError(f"b200norm: input of dtype {x.dtype} with a residual of dtype {residual.dtype}; it takes float32, "
                           "float16 and bfloat16 with a residual of the same dtype or float32")


def _like(t, rows):
    """An uninitialised contiguous tensor shaped like t; `rows` is what _flat made of t."""
    return torch.empty_like(t) if rows is t else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _add_rmsnorm_fwd(x, residual, weight, eps, *, need_rstd=True):
    """Returns (y shaped and typed like x, h typed like residual, rstd (M,) fp32 or None)."""
    _require_cuda(x)
    _check_residual(x, residual)
    device = x.device
    xr, M, N, xs = _flat(x)
    r, _, _, rs = _flat(residual)
    Fn._check_dim(x, N)
    weight, _, wcode = _params(weight, None, N, device)
    y, h = _like(x, xr), _like(residual, r)
    rstd = torch.empty(M, dtype=torch.float32, device=device) if need_rstd else None
    lib = _lib.load()
    index = device.index
    with _on_device(index):
        _lib.check(lib.b200norm_add_rms_fwd(
            xr.data_ptr(), xs, r.data_ptr(), rs, _ptr(weight), y.data_ptr(), N, h.data_ptr(), N, _ptr(rstd), M, N, eps,
            _code(x, "input"), _code(r, "residual"), wcode, _raw_stream(index)))
    return y, h, rstd


def _add_rmsnorm_bwd(h, dy, dh, weight, rstd, *, need_dw=True):
    """Gradients of (y, h) -> (x, residual, weight).  `dy` decides x's type; `dh` may be None.  When the two
    types are one, dx and dresidual are the same tensor."""
    _require_cuda(h)
    device, shape = h.device, h.shape
    assert dy.shape == shape and (dh is None or dh.shape == shape), 'expect input and output shape to be the same'
    for t in (dy, dh, rstd):
        if t is not None and t.device != device:
            raise RuntimeError(f"b200norm: gradient on {t.device}, input on {device}")
    if dh is not None and dh.dtype != h.dtype:
        dh = dh.to(h.dtype)
    hr, M, N, hs = _flat(h)
    dyr, _, _, dys = _flat(dy)
    dhr, _, _, dhs = _flat(dh) if dh is not None else (None, M, N, N)
    Fn._check_dim(dy, N)
    weight, _, wcode = _params(weight, None, N, device)
    dx = _like(dy, dyr)
    dres = _like(h, hr) if h.dtype != dy.dtype else None
    dw = torch.empty_like(weight) if (weight is not None and need_dw) else None
    io, res = _code(dyr, "input"), _code(hr, "residual")
    lib = _lib.load()
    index = device.index
    with _on_device(index):
        ws, ws_bytes = None, 0
        if dw is not None:
            ws_bytes = _workspace_bytes(index, M, N, io, res)
            ws = torch.empty(ws_bytes, dtype=torch.uint8, device=device)
        _lib.check(lib.b200norm_add_rms_bwd(
            hr.data_ptr(), hs, dyr.data_ptr(), dys, _ptr(dhr), dhs, _ptr(weight), rstd.data_ptr(), dx.data_ptr(), N, _ptr(dres),
            N, _ptr(dw), _ptr(ws), ws_bytes, M, N, io, res, wcode, _raw_stream(index)))
    return dx, (dx if dres is None else dres), dw


class add_rmsnorm(torch.autograd.Function):
    """(x, residual, weight or None, eps) -> (y, h).  Saves (h, weight, rstd)."""

    @classmethod
    def apply(cls, x, residual, weight, eps):
        if _unrecorded():  # a decode step's call is spared autograd's bookkeeping
            return _add_rmsnorm_fwd(x, residual, weight, eps, need_rstd=False)[:2]
        return super().apply(x, residual, weight, eps)

    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        y, h, rstd = _add_rmsnorm_fwd(x, residual, weight, eps)
        ctx.save_for_backward(h, weight, rstd)
        ctx.x_dtype = x.dtype
        ctx.set_materialize_grads(False)
        return y, h

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh):
        h, weight, rstd = ctx.saved_tensors
        if dy is None:  # only h was used: the addition alone
            return (None, None, None, None) if dh is None else (dh.to(ctx.x_dtype), dh, None, None)
        dx, dres, dw = _add_rmsnorm_bwd(h, dy, dh, weight, rstd, need_dw=ctx.needs_input_grad[2])
        return dx, dres, dw, None


def rmsnorm_fp8(x, weight=None, eps=1e-5, *, residual=None, group=0, scale_dtype=torch.float32):
    """RMSNorm with an 8-bit output: returns (q, scale), or (q, scale, h) with a residual, where
    q.float() * scale (each scale over its columns) is the norm of h = x + residual (of x without one).

    q: float8_e4m3fn, shaped like x, the nearest value to the norm / scale in fp32.  group: columns that share a scale: 32,
    64 or 128 (the last group of a row may be shorter), or 0 for the whole row.  scale: x.shape[:-1] + (ceil(N / group),),
    the group's largest magnitude / 448, as float32 (good to two roundings of its own), or as float8_e8m0fnu rounded up to
    a power of two.
    A group of zeros has the scale 2^-64 / 448; one that holds a NaN has the scale NaN.

    For inference: it has no gradient, and refuses inputs that ask for one."""
    _require_cuda(x)
    given = [t for t in (x, weight, residual) if t is not None]
    if torch.is_grad_enabled() and any(t.requires_grad for t in given):
        raise RuntimeError("b200norm: rmsnorm_fp8 has no gradient; call it under torch.no_grad()")
    if _dual_level() >= 0 and any(torch.autograd.forward_ad.unpack_dual(t).tangent is not None for t in given):
        raise RuntimeError("b200norm: rmsnorm_fp8 has no gradient, nor a forward-mode derivative")
    if group not in (0, 32, 64, 128):
        raise RuntimeError(f"b200norm: a scale covers 32, 64 or 128 columns, or (0) a row; got {group}")
    if scale_dtype not in (torch.float32, torch.float8_e8m0fnu):
        raise RuntimeError(f"b200norm: scales are float32 or float8_e8m0fnu, not {scale_dtype}")
    if x.dtype == torch.float64:
        raise RuntimeError("b200norm: input dtype torch.float64 is not supported (float32, float16, bfloat16)")
    shape, device = x.shape, x.device
    if residual is not None:
        _check_residual(x, residual)
    x, M, N, xs = _flat(x)
    Fn._check_dim(x, N)
    code = rcode = _code(x, "input")
    r, rs, h = None, N, None
    if residual is not None:
        r, _, _, rs = _flat(residual)
        h, rcode = _like(residual, r), _code(r, "residual")
    weight, _, wcode = _params(weight, None, N, device)
    q = torch.empty(*shape, dtype=torch.float8_e4m3fn, device=device)
    scale = torch.empty(*shape[:-1], -(-N // group) if group else 1, dtype=scale_dtype, device=device)
    lib = _lib.load()
    index = device.index
    with _on_device(index):
        _lib.check(lib.b200norm_rms_fp8(
            x.data_ptr(), xs, _ptr(r), rs, _ptr(weight), q.data_ptr(), N, scale.data_ptr(), _ptr(h), N, M, N, eps, int(group),
            0 if scale_dtype == torch.float32 else 1, code, rcode, wcode, _raw_stream(index)))
    return (q, scale) if h is None else (q, scale, h)


from .modules import RMSNorm  # noqa: E402  (the modules below reuse its parameter and init)


class AddRMSNorm(RMSNorm):
    """RMSNorm of x + residual: forward(x, residual) -> (y, h), h being the sum.  Same constructor, parameter
    and state_dict as RMSNorm."""

    def forward(self, x, residual):
        return add_rmsnorm.apply(x, residual, self.weight, self.eps)


class RMSNormFP8(RMSNorm):
    """RMSNorm with an 8-bit output: forward(x[, residual]) -> (q, scale[, h]), see rmsnorm_fp8.  RMSNorm's
    constructor plus `group` and `scale_dtype`; same parameter and state_dict."""

    def __init__(self, dimension, eps=1e-5, elementwise_affine=True, group=0, scale_dtype=torch.float32, device=None,
                 dtype=None):
        super().__init__(dimension, eps, elementwise_affine, device, dtype)
        self.group = group
        self.scale_dtype = scale_dtype

    def forward(self, x, residual=None):
        return rmsnorm_fp8(x, self.weight, self.eps, residual=residual, group=self.group, scale_dtype=self.scale_dtype)
