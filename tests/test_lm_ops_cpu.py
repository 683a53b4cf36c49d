"""The residual norms, the expert choice and the token choice without a GPU: the argument checks of their C entry points
(which run before any CUDA call), their modules' parameters, and the refusal of CPU tensors."""
import inspect

import pytest
import torch

import b200norm
from b200norm import AddRMSNorm, RMSNorm, RMSNormFP8, Router, Sampler, _lib

ERR, UNSUPPORTED, OK = _lib.ERR_ARG, _lib.ERR_UNSUPPORTED, _lib.OK
P = 4096  # stands for a device pointer: every call here is refused, or has nothing to do, before it is used


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def said(lib, text):
    return text in lib.b200norm_last_error()


def add_fwd(lib, M=4, N=8, io=_lib.F32, res=_lib.F32, w=_lib.F32, x=P, r=P, y=P, h=P, xs=8, rs=8, ys=8, hs=8):
    return lib.b200norm_add_rms_fwd(x, xs, r, rs, None, y, ys, h, hs, P, M, N, 1e-6, io, res, w, None)


def test_add_rms_fwd_checks(lib):
    assert add_fwd(lib, io=_lib.F64, res=_lib.F64) == ERR and said(lib, b"fp32, fp16 and bf16")
    assert add_fwd(lib, io=_lib.F16, res=_lib.BF16) == ERR
    assert add_fwd(lib, io=_lib.F32, res=_lib.BF16) == ERR
    assert add_fwd(lib, io=9, res=9) == ERR
    assert add_fwd(lib, w=7) == ERR and said(lib, b"weight dtype")
    assert add_fwd(lib, M=-1) == ERR and add_fwd(lib, N=0) == ERR
    assert add_fwd(lib, N=16385, xs=16385, rs=16385, ys=16385, hs=16385) == UNSUPPORTED and said(lib, b"64KB")
    for name in ("x", "r", "y", "h"):
        assert add_fwd(lib, **{name: None}) == ERR and said(lib, b"null")
    for name in ("xs", "rs", "ys", "hs"):
        assert add_fwd(lib, **{name: 7}) == ERR and said(lib, b"stride")
    assert add_fwd(lib, M=0, x=None, r=None, y=None, h=None) == OK  # nothing to do


def add_bwd(lib, M=4, N=8, io=_lib.F32, res=_lib.F32, h=P, dy=P, rstd=P, dx=P, dres=None, dw=None, hs=8, dys=8, dhs=8, dxs=8,
            drs=8):
    return lib.b200norm_add_rms_bwd(h, hs, dy, dys, P, dhs, None, rstd, dx, dxs, dres, drs, dw, None, 0, M, N, io, res, _lib.F32,
                                    None)


def test_add_rms_bwd_checks(lib):
    assert add_bwd(lib, io=_lib.F16, res=_lib.BF16) == ERR
    for name in ("h", "dy", "rstd", "dx"):
        assert add_bwd(lib, **{name: None}) == ERR and said(lib, b"null")
    assert add_bwd(lib, io=_lib.BF16) == ERR and said(lib, b"null")        # two types need a second gradient buffer
    assert add_bwd(lib, dres=P) == ERR and said(lib, b"equals dx")         # one type has one gradient
    for name in ("hs", "dys", "dhs", "dxs"):
        assert add_bwd(lib, **{name: 7}) == ERR and said(lib, b"stride")
    assert add_bwd(lib, io=_lib.BF16, dres=P, drs=7) == ERR and said(lib, b"stride")
    assert add_bwd(lib, M=0, h=None, dy=None, rstd=None, dx=None) == OK
    assert lib.b200norm_add_rms_bwd_workspace_bytes(4, 8, _lib.F64, _lib.F64) == 0
    assert lib.b200norm_add_rms_bwd_workspace_bytes(4, 0, _lib.F32, _lib.F32) == 0


def fp8(lib, M=4, N=8, io=_lib.F32, res=_lib.F32, x=P, r=None, q=P, scale=P, h=None, group=0, xs=8, rs=8, qs=8, hs=8):
    return lib.b200norm_rms_fp8(x, xs, r, rs, None, q, qs, scale, h, hs, M, N, 1e-6, group, 0, io, res, _lib.F32, None)


def test_rms_fp8_checks(lib):
    assert fp8(lib, io=_lib.F64, res=_lib.F64) == ERR
    for group in (-1, 1, 16, 48, 256):
        assert fp8(lib, group=group) == ERR and said(lib, b"columns")
    for name in ("x", "q", "scale"):
        assert fp8(lib, **{name: None}) == ERR and said(lib, b"null")
    assert fp8(lib, h=P) == ERR and said(lib, b"there is none")
    assert fp8(lib, xs=7) == ERR and fp8(lib, qs=7) == ERR and fp8(lib, r=P, rs=7) == ERR and fp8(lib, r=P, h=P, hs=7) == ERR
    assert fp8(lib, M=0, x=None, q=None, scale=None) == OK


def route_fwd(lib, T=4, E=16, k=2, dtype=_lib.F32, logits=P, stride=16, gates=P, experts=P, counts=P, loss=P):
    return lib.b200norm_route_fwd(logits, stride, None, gates, experts, None, counts, loss, None, 0, T, E, k, 1, dtype, None)


def route_bwd(lib, T=4, E=16, k=2, dtype=_lib.F32, logits=P, stride=16, gates=P, experts=P, lse=P, counts=P, dgs=2, dlogits=P):
    return lib.b200norm_route_bwd(logits, stride, gates, experts, lse, counts, P, dgs, None, dlogits, T, E, k, 1, dtype, None)


def test_route_checks(lib):
    for call in (route_fwd, route_bwd):
        assert call(lib, dtype=_lib.F64) == ERR and said(lib, b"fp32, fp16 or bf16")
        assert call(lib, E=0) == ERR and call(lib, E=1025, stride=1025) == ERR and said(lib, b"experts")
        assert call(lib, T=-1) == ERR
        for k in (0, -3, 17):
            assert call(lib, k=k) == ERR and said(lib, b"top_k")
        assert call(lib, E=64, k=33, stride=64) == ERR and said(lib, b"top_k")
        assert call(lib, T=2 ** 31, k=2) == ERR and said(lib, b"32-bit")
        assert call(lib, stride=15) == ERR and said(lib, b"stride")
    for name in ("logits", "gates", "experts", "counts", "loss"):
        assert route_fwd(lib, **{name: None}) == ERR and said(lib, b"null")
    for name in ("logits", "gates", "experts", "lse", "counts", "dlogits"):
        assert route_bwd(lib, **{name: None}) == ERR and said(lib, b"null")
    assert route_bwd(lib, dgs=1) == ERR and said(lib, b"stride")
    assert route_bwd(lib, T=0, logits=None, dlogits=None) == OK
    assert lib.b200norm_route_workspace_bytes(4, 16, 17, _lib.F32) == 0
    assert lib.b200norm_route_workspace_bytes(4, 16, 2, _lib.F64) == 0


def sample(lib, M=4, V=16, dtype=_lib.F32, logits=P, stride=16, uniform=P, tokens=P):
    return lib.b200norm_sample(logits, stride, uniform, None, 1.0, None, 0, None, 1.0, None, 0.0, tokens, M, V, dtype, None)


def test_sample_checks(lib):
    assert sample(lib, dtype=_lib.F64) == ERR and said(lib, b"fp32, fp16 or bf16")
    assert sample(lib, M=-1) == ERR and sample(lib, V=0) == ERR
    assert sample(lib, V=262145, stride=262145) == UNSUPPORTED and said(lib, b"262144")
    assert sample(lib, M=2 ** 31) == ERR and said(lib, b"too many rows")
    for name in ("logits", "uniform", "tokens"):
        assert sample(lib, **{name: None}) == ERR and said(lib, b"null")
    assert sample(lib, stride=15) == ERR and said(lib, b"stride")
    assert sample(lib, M=0, logits=None, uniform=None, tokens=None) == OK


def test_modules_are_rmsnorms():
    plain = RMSNorm(64, eps=1e-6, dtype=torch.bfloat16)
    torch.nn.init.normal_(plain.weight)
    for m in (AddRMSNorm(64, eps=1e-6, dtype=torch.bfloat16), RMSNormFP8(64, eps=1e-6, group=32, dtype=torch.bfloat16)):
        assert torch.all(m.weight == 1) and m.weight.dtype == torch.bfloat16 and m.eps == 1e-6
        m.load_state_dict(plain.state_dict())
        assert torch.equal(m.weight, plain.weight)
        assert list(m.state_dict()) == list(plain.state_dict())
    assert AddRMSNorm(8, elementwise_affine=False).weight is None
    m = RMSNormFP8(8, group=128, scale_dtype=torch.float8_e8m0fnu)
    assert (m.group, m.scale_dtype) == (128, torch.float8_e8m0fnu)
    own = list(inspect.signature(AddRMSNorm.__init__).parameters)
    assert own == list(inspect.signature(RMSNorm.__init__).parameters)


def test_cpu_tensors_are_refused():
    x = torch.randn(4, 64)
    for call in (lambda: AddRMSNorm(64)(x, x), lambda: b200norm.add_rmsnorm.apply(x, x, None, 1e-6), lambda: RMSNormFP8(64)(x),
                 lambda: b200norm.rmsnorm_fp8(x), lambda: Router(2)(x), lambda: b200norm.route.apply(x, 2),
                 lambda: Sampler()(x, torch.rand(4)), lambda: b200norm.sample(x, torch.rand(4))):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            call()
        with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA tensors only"):
            call()


@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_raises_with_and_without_gradients(grad, monkeypatch):
    # stand-ins for the kernels' calls: what matters is which way a call takes.  no_grad leaves forward mode on
    def route_fwd(x, k, *args, **kwargs):
        return x[..., :k] * 1, x[..., :k].int(), torch.zeros(x.shape[-1] + 1, dtype=torch.int32), x.sum() * 0, None

    monkeypatch.setattr(b200norm.addnorm, "_add_rmsnorm_fwd", lambda x, r, w, eps, **kwargs: (x * 1, x + r, None))
    monkeypatch.setattr(b200norm.routing, "_route_fwd", route_fwd)
    x = torch.randn(4, 64)
    with torch.set_grad_enabled(grad):
        y, h = b200norm.add_rmsnorm.apply(x, x, None, 1e-6)
        gates, experts, counts, loss = b200norm.route.apply(x, 2)
        assert torch.equal(h, x + x) and gates.shape == (4, 2) and counts.shape == (64,)
        with torch.autograd.forward_ad.dual_level():
            d = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
            for call in (lambda: b200norm.add_rmsnorm.apply(d, x, None, 1e-6), lambda: b200norm.route.apply(d, 2)):
                with pytest.raises(NotImplementedError, match="jvp"):
                    call()


def test_rmsnorm_fp8_refuses_a_tangent(monkeypatch):
    monkeypatch.setattr(b200norm.addnorm, "_require_cuda", lambda x: None)  # refused before any CUDA call
    x = torch.randn(4, 64)
    with torch.no_grad(), torch.autograd.forward_ad.dual_level():
        d = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        for kw in (dict(x=d), dict(x=x, residual=d), dict(x=x, weight=d[0])):
            with pytest.raises(RuntimeError, match="forward-mode"):
                b200norm.rmsnorm_fp8(**kw)


def test_addresses_inside_an_element_are_refused(lib):
    B, F = _lib.BF16, _lib.F32

    def refused(rc):
        return rc == ERR and said(lib, b"inside an element")

    for name in ("x", "r", "y", "h"):
        assert refused(add_fwd(lib, **{name: P + 2})) and refused(add_fwd(lib, io=B, res=B, **{name: P + 1}))
    for name in ("h", "dy", "rstd", "dx"):
        assert refused(add_bwd(lib, **{name: P + 2}))
        assert refused(add_bwd(lib, io=B, dres=P, **{name: P + 1}))
    assert refused(add_bwd(lib, io=B, dres=P + 2)) and refused(add_bwd(lib, dw=P + 2))
    assert refused(fp8(lib, x=P + 2)) and refused(fp8(lib, scale=P + 1)) and refused(fp8(lib, r=P + 2)) and refused(fp8(lib, r=P, h=P + 3))
    for dtype, step in ((F, 2), (B, 1)):
        assert refused(route_fwd(lib, dtype=dtype, logits=P + step)) and refused(route_bwd(lib, dtype=dtype, logits=P + step))
        assert refused(route_bwd(lib, dtype=dtype, dlogits=P + step)) and refused(sample(lib, dtype=dtype, logits=P + step))
    for name in ("gates", "experts", "counts"):
        assert refused(route_fwd(lib, **{name: P + 2})) and refused(route_bwd(lib, **{name: P + 2}))
    assert refused(route_fwd(lib, loss=P + 1)) and refused(route_bwd(lib, lse=P + 2))
    assert refused(sample(lib, uniform=P + 2)) and refused(sample(lib, tokens=P + 4))
    # a weight's and a weight gradient's elements are those of its own type
    for w, step in ((_lib.F64, 4), (F, 2), (B, 1)):
        rc = lib.b200norm_add_rms_fwd(P, 8, P, 8, P + step, P, 8, P, 8, P, 4, 8, 1e-6, F, F, w, None)
        assert refused(rc)
