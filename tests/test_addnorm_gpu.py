"""Residual + RMSNorm (forward, backward) and RMSNorm with an 8-bit output on the GPU, against the formulas in
64 bits.

Bounds.  u = 2^-24 is half a step of fp32.  A row's sum of N non-negative products runs through at most 64 serial
additions in a thread, 5 in the warp and 32 across warps, each rounded (u), with 3 roundings in a product:
|error| <= 104 u * sum of magnitudes.  rstd takes half of that and 3 roundings of its own, an output element at most 4
more: relative error of y before its store <= 60 u; a store to type t adds eps(t) / 2, or half the smallest subnormal.
dx: every term of d = w dy rstd - h rstd^2 c1 + dh carries at most 120 u of its own magnitude besides c1's 104 u and rstd's
2 * 55 u: 240 u of the sum of the terms' magnitudes (with sum |xhat w dy| in c1) covers all.
dweight: M products added in some order, each with at most 60 u: (M + 64) u of the sum of magnitudes, and a store.
"""
import pytest
import torch

import b200norm
from b200norm import addnorm as A

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [(F32, F32), (F16, F16), (BF16, BF16), (F16, F32), (BF16, F32)]
SHAPES = [(1, 1), (3, 5), (7, 64), (5, 100), (33, 256), (2, 1000), (4, 1001), (9, 1024), (11, 2048), (5, 4096), (21, 4104),
          (3, 5120), (2, 8193), (2, 12288), (3, 16384)]


def store_error(ref, dtype):
    return ref.abs() * (torch.finfo(dtype).eps / 2) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def make(M, N, t, r, w=None, seed=0, layout="contiguous"):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def rows(dtype, scale=1.0):
        def draw(m, n):
            return (torch.randn(m, n, generator=g, device=DEV) * scale).to(dtype)
        if layout == "contiguous":
            return draw(M, N)
        if layout == "padded":  # row stride larger than the row, still whole packets
            return draw(M, N + 32)[:, :N]
        if layout == "offset":  # every row starts three elements behind a packet boundary, in every buffer alike
            return draw(M, N + 32)[:, 3:N + 3]
        raise ValueError(layout)

    x, res = rows(t), rows(r, 2.0)
    weight = None if w is None else (1 + 0.1 * torch.randn(N, generator=g, device=DEV)).to(w)
    return x, res, weight, torch.randn(M, N, generator=g, device=DEV).to(t), torch.randn(M, N, generator=g, device=DEV).to(r)


def check_forward(x, res, w, eps, y, h):
    t, r = x.dtype, res.dtype
    assert y.dtype == t and h.dtype == r and y.shape == h.shape == x.shape
    assert torch.equal(h, (x.float() + res.float()).to(r))
    h64 = h.double()
    ref = h64 / torch.sqrt(h64.square().mean(-1, keepdim=True) + eps) * (1 if w is None else w.double())
    assert ((y.double() - ref).abs() <= store_error(ref, t) * (1 + 1e-6) + 60 * U * ref.abs()).all()


def check_backward(h, dy, dh, w, eps, dx, dres, dw):
    N = h.shape[-1]
    h64, g64, d64 = h.double().reshape(-1, N), dy.double().reshape(-1, N), 0 if dh is None else dh.double().reshape(-1, N)
    w64 = torch.ones(N, dtype=torch.float64, device=h.device) if w is None else w.double()
    rs = 1 / torch.sqrt(h64.square().mean(-1, keepdim=True) + eps)
    xhat, wdy = h64 * rs, w64 * g64
    ref = (wdy - xhat * (xhat * wdy).mean(-1, keepdim=True)) * rs + d64
    size = wdy.abs() * rs + xhat.abs() * rs * (xhat * wdy).abs().mean(-1, keepdim=True) + (0 if dh is None else d64.abs())
    for got, t in ((dx, dy.dtype), (dres, h.dtype)):
        assert got.dtype == t and got.shape == h.shape
        assert ((got.double().reshape(-1, N) - ref).abs() <= store_error(ref, t) * (1 + 1e-6) + 240 * U * size).all()
    if w is not None:
        terms = g64 * xhat
        ref = terms.sum(0)
        bound = store_error(ref, w.dtype) * (1 + 1e-6) + (h64.shape[0] + 64) * U * terms.abs().sum(0)
        assert dw.dtype == w.dtype and ((dw.double() - ref).abs() <= bound).all()


def check(M, N, t, r, w, layout="contiguous", eps=1e-6, with_dh=True):
    x, res, weight, dy, dh = make(M, N, t, r, w, seed=M * 131 + N, layout=layout)
    y, h, rstd = A._add_rmsnorm_fwd(x, res, weight, eps)
    check_forward(x, res, weight, eps, y, h)
    if layout == "offset":  # the gradients' buffers alike
        h = torch.empty(M, N + 32, dtype=r, device=DEV)[:, 3:N + 3].copy_(h)
        dy = torch.empty(M, N + 32, dtype=t, device=DEV)[:, 3:N + 3].copy_(dy)
    dx, dres, dw = A._add_rmsnorm_bwd(h, dy, dh if with_dh else None, weight, rstd)
    check_backward(h, dy, dh if with_dh else None, weight, eps, dx, dres, dw)


@pytest.mark.parametrize("t,r", TYPES)
def test_shapes(t, r):
    for M, N in SHAPES + ([(2, 24576), (2, 32768)] if t != F32 else []):
        check(M, N, t, r, t)


@pytest.mark.parametrize("t,r", TYPES)
@pytest.mark.parametrize("layout", ["padded", "offset"])
def test_layouts(t, r, layout):
    for M, N in [(1, 1), (6, 40), (9, 1001), (5, 2048), (3, 8192)]:
        check(M, N, t, r, F32, layout=layout)


@pytest.mark.parametrize("t,r", TYPES)
def test_more_rows_than_resident_groups(t, r):
    # the row loops run more than once, at row lengths of every kind of row group
    for M, N in [(60001, 64), (20011, 129), (9001, 1001), (4097, 1536), (3001, 4100)]:
        check(M, N, t, r, BF16)


@pytest.mark.parametrize("w", [None, F32, F16, BF16, torch.float64])
@pytest.mark.parametrize("t", [F32, BF16])
def test_weight_types(t, w):
    check(17, 512, t, t, w)
    check(5, 333, t, t, w)


def test_no_gradient_of_h():
    check(33, 1000, BF16, BF16, BF16, with_dh=False)
    check(33, 1000, F16, F32, F32, with_dh=False)


def test_unlike_alignments_and_orders():
    g = torch.Generator(device=DEV).manual_seed(5)
    base = torch.randn(40, 999, generator=g, device=DEV).to(BF16)
    cases = [
        (base[:, 1:900], base[:, 40:939]),                                   # two different offsets
        (base.t()[:900].t(), base[:, :900].contiguous()),                    # strided alike
        (torch.randn(900, 40, generator=g, device=DEV).to(BF16).t(), base[:, :900]),   # columns contiguous
        (base[:1, :900].expand(40, 900), base[:, :900]),                     # one row for all
    ]
    w = torch.ones(901, device=DEV, dtype=BF16)[1:]  # a weight off its packet boundary
    for x, res in cases:
        n = x.shape[1]
        y, h, rstd = A._add_rmsnorm_fwd(x, res, w[:n], 1e-6)
        check_forward(x, res, w[:n], 1e-6, y, h)
        dy = torch.randn(x.shape, generator=g, device=DEV).to(BF16)
        dyv = torch.empty(40, 1000, dtype=BF16, device=DEV)[:, 5:5 + n].copy_(dy)
        check_backward(h, dyv, None, w[:n], 1e-6, *A._add_rmsnorm_bwd(h, dyv, None, w[:n], rstd))


def test_zeros_and_infinities():
    x = torch.zeros(4, 256, device=DEV, dtype=BF16)
    x[1] = 3.0e38
    x[2, 7] = float("inf")
    x[3, 9] = float("nan")
    y, h, _ = A._add_rmsnorm_fwd(x, torch.zeros_like(x), None, 1e-6)
    assert torch.equal(y[0], torch.zeros_like(y[0])) and torch.equal(h.isnan(), x.isnan())
    assert (y[1] == 0).all()           # the sum of squares overflows fp32, as RMSNorm's does
    assert y[2, 7].isnan() and (y[2, :7] == 0).all()
    assert y[3].isnan().all()


def test_module_gradients_against_autograd_in_64_bits():
    torch.manual_seed(0)
    m = b200norm.AddRMSNorm(96, eps=1e-5, device=DEV, dtype=F32)
    with torch.no_grad():
        m.weight.normal_(1, 0.1)
    x, r = torch.randn(2, 5, 96, device=DEV, requires_grad=True), torch.randn(2, 5, 96, device=DEV, requires_grad=True)
    y, h = m(x, r)
    (y.sin().sum() + (h * h).sum()).backward()
    x64, r64, w64 = (t.detach().double().requires_grad_(True) for t in (x, r, m.weight))
    h64 = x64 + r64
    y64 = h64 / torch.sqrt(h64.square().mean(-1, keepdim=True) + 1e-5) * w64
    (y64.sin().sum() + (h64 * h64).sum()).backward()
    for a, b in ((x, x64), (r, r64), (m.weight, w64)):
        torch.testing.assert_close(a.grad.double(), b.grad, rtol=1e-4, atol=1e-5)  # sums of up to 96 terms of size 1
    assert x.grad.data_ptr() != r.grad.data_ptr()


def test_gradient_against_differences():
    # central differences of the operator itself: error of the difference h^2 |f'''| / 6 + 2 u |f| / h = 1e-6 + 1e-3 at h = 1e-3
    torch.manual_seed(1)
    x, r, w = torch.randn(3, 24, device=DEV), torch.randn(3, 24, device=DEV), torch.rand(24, device=DEV) + 0.5
    a, b = torch.randn(3, 24, device=DEV), torch.randn(3, 24, device=DEV)

    def f(x, w):
        y, h = b200norm.add_rmsnorm.apply(x, r, w, 1e-5)
        return (y.double() * a).sum() + (h.double() * b).sum()

    xg, wg = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    gx, gw = torch.autograd.grad(f(xg, wg), (xg, wg))
    for t, grad, call in ((x, gx, lambda v: f(v, w)), (w, gw, lambda v: f(x, v))):
        d = torch.randn_like(t)
        step = 1e-2
        num = (call(t + step * d) - call(t - step * d)) / (2 * step)
        assert abs(float(num) - float((grad * d).sum())) <= 5e-3 * float((grad.abs() * d.abs()).sum())


def test_only_one_output_used_and_shared_leaves():
    x = torch.randn(4, 64, device=DEV, requires_grad=True)
    w = torch.ones(64, device=DEV, requires_grad=True)
    y, h = b200norm.add_rmsnorm.apply(x, x, w, 1e-6)  # the same leaf twice
    h.sum().backward()
    assert torch.equal(x.grad, torch.full_like(x, 2.0)) and w.grad is None
    x.grad = None
    y, h = b200norm.add_rmsnorm.apply(x, x, w, 1e-6)
    (y * y).sum().backward()
    ref = x.detach().double().requires_grad_(True)
    h64 = 2 * ref
    (h64.square() / (h64.square().mean(-1, keepdim=True) + 1e-6)).sum().backward()
    torch.testing.assert_close(x.grad.double(), ref.grad, rtol=1e-4, atol=1e-5)
    with pytest.raises(RuntimeError, match="once_differentiable|differentiat"):
        y, h = b200norm.add_rmsnorm.apply(x, x, w, 1e-6)
        g, = torch.autograd.grad((y * y).sum(), x, create_graph=True)
        g.sum().backward()


def test_same_as_addition_then_rmsnorm():
    x, r, w, dy, dh = make(64, 4096, BF16, BF16, BF16)
    y, h = b200norm.add_rmsnorm.apply(x, r, w, 1e-6)
    y2 = b200norm.rmsnorm.apply(x + r, w, 1e-6)
    assert torch.equal(h, x + r)
    # both within their bound of the exact value: at most one step of bf16 apart
    assert ((y.double() - y2.double()).abs() <= 2.0 ** -7 * y2.double().abs() + 1e-30).all()


def test_empty_batch():
    x = torch.empty(0, 64, device=DEV, dtype=BF16, requires_grad=True)
    w = torch.ones(64, device=DEV, dtype=BF16, requires_grad=True)
    y, h = b200norm.add_rmsnorm.apply(x, torch.empty_like(x), w, 1e-6)
    assert y.shape == h.shape == (0, 64)
    y.sum().backward()
    assert torch.equal(w.grad, torch.zeros_like(w)) and x.grad.shape == (0, 64)
    q, s = b200norm.rmsnorm_fp8(x.detach(), w.detach(), group=32)
    assert q.shape == (0, 64) and s.shape == (0, 2)


# ---------------------------------------------------------------------------------------------
# 8 bits
# ---------------------------------------------------------------------------------------------
def check_fp8(x, res, w, eps, group, e8m0):
    out = b200norm.rmsnorm_fp8(x, w, eps, residual=res, group=group,
                               scale_dtype=torch.float8_e8m0fnu if e8m0 else F32)
    N = x.shape[-1]
    q, scale = out[0], out[1]
    h = x
    if res is not None:
        assert len(out) == 3 and torch.equal(out[2], (x.float() + res.float()).to(res.dtype))
        h = out[2]
    G = -(-N // group) if group else 1
    assert q.dtype == torch.float8_e4m3fn and q.shape == x.shape and scale.shape == (*x.shape[:-1], G)
    h64 = h.double()
    y = h64 / torch.sqrt(h64.square().mean(-1, keepdim=True) + eps) * (1 if w is None else w.double())
    size = group or N
    pad = torch.nn.functional.pad(y, (0, G * size - N)).reshape(*x.shape[:-1], G, size)
    want = pad.abs().amax(-1).clamp(min=2.0 ** -64) / 448
    s = scale.float().double()
    if e8m0:
        # a power of two, the lowest that is not below the scale (which fp32 knows to 60 u)
        assert (torch.frexp(scale.float())[0] == 0.5).all()
        assert (s >= want * (1 - 64 * U)).all() and (s < 2 * want * (1 + 64 * U)).all()
    else:
        assert ((s - want).abs() <= 64 * U * want).all()
    exact = (pad / s[..., None]).reshape(*x.shape[:-1], G * size)[..., :N]
    # The nearest e4m3 value: half a step is 2^-4 of the power of two below the value (2^-10 among the subnormals), and the
    # unrounded quotient is good to 64 u.  The largest value may sit a rounding above 448 and is cut there.
    step = torch.exp2(torch.floor(torch.log2(exact.abs().clamp(min=2.0 ** -6)))) * 2.0 ** -4
    err = (q.float().double() - exact.clamp(-448, 448)).abs()
    assert (err <= step + 64 * U * exact.abs()).all()


@pytest.mark.parametrize("group,e8m0", [(0, False), (0, True), (32, False), (32, True), (64, False), (128, False), (128, True)])
@pytest.mark.parametrize("t,r", [(F32, None), (F32, F32), (F16, F16), (BF16, None), (BF16, BF16), (BF16, F32), (F16, F32)])
def test_fp8(t, r, group, e8m0):
    for M, N in [(3, 8), (5, 32), (2, 48), (7, 200), (4, 128), (3, 1001), (9, 1024), (2, 4104), (3, 8192), (2, 16384)]:
        x, res, w, _, _ = make(M, N, t, r or t, BF16 if N % 3 else None, seed=N)
        check_fp8(x, res if r else None, w, 1e-6, group, e8m0)


@pytest.mark.parametrize("group", [0, 64])
def test_fp8_rows_loop_and_layouts(group):
    x, res, w, _, _ = make(30011, 72, BF16, BF16, F32, seed=2)
    check_fp8(x, res, w, 1e-6, group, False)
    for layout in ("padded", "offset"):
        x, res, w, _, _ = make(300, 1000, F16, F32, F16, seed=3, layout=layout)
        check_fp8(x, res, w, 1e-6, group, group != 0)
    x, res, w, _, _ = make(2, 32768, BF16, BF16, BF16, seed=4)
    check_fp8(x, res, w, 1e-6, group, False)
    x = torch.randn(2, 3, 130, device=DEV)
    check_fp8(x, None, None, 1e-6, group, False)


def test_fp8_unlike_alignments():
    g = torch.Generator(device=DEV).manual_seed(6)
    for t in (F32, BF16):
        base = torch.randn(40, 3000, generator=g, device=DEV).to(t)
        for n in (33, 900, 2500):
            for group, e8m0 in ((0, False), (32, True), (128, False)):
                check_fp8(base[:, 1:1 + n], base[:, 40:40 + n], torch.ones(n + 1, device=DEV, dtype=t)[1:], 1e-6, group, e8m0)
                check_fp8(base.t()[:n].t(), None, None, 1e-6, group, e8m0)


@pytest.mark.parametrize("t,r", [(F32, None), (BF16, BF16), (F16, F32)])
def test_fp8_many_rows_off_the_packets(t, r):
    # scales whose columns begin and end inside packets, at every kind of row group
    for M, N in [(70001, 33), (9001, 131), (4001, 777), (700, 4099), (301, 8191)]:
        x, res, w, _, _ = make(M, N, t, r or t, F32, seed=N)
        check_fp8(x, res if r else None, w, 1e-6, [0, 32, 64, 128][N % 4], N % 3 == 0)


def test_fp8_overflowing_squares():
    # the sum of squares is infinite and the norm 0, as RMSNorm's, though h * w overflows on the way
    x = torch.full((3, 512), 3e38, device=DEV)
    x[1, 5] = float("inf")
    w = torch.full((512,), 2.0, device=DEV)
    for xs in (x, x[:, :509]):
        for group in (0, 64):
            q, s = b200norm.rmsnorm_fp8(xs, w[:xs.shape[1]], 1e-6, group=group)
            assert (q[[0, 2]].float() == 0).all() and s[[0, 2]].isfinite().all()
            assert q[1, 5].float().isnan() and s[1, 0].isnan()


def test_fp8_zero_rows_and_poison():
    x = torch.zeros(3, 256, device=DEV)
    x[1] = 1.0
    x[2, 40] = float("nan")
    for e8m0 in (torch.float32, torch.float8_e8m0fnu):
        q, s = b200norm.rmsnorm_fp8(x, None, 1e-6, group=64, scale_dtype=e8m0)
        assert (q[0].float() == 0).all() and (s[0].float() > 0).all() and s[0].float().isfinite().all()
        assert q[2].float().isnan().all() and s[2].float().isnan().all()
    # one huge column: only its group is scaled for it
    w = torch.ones(256, device=DEV)
    w[200] = 1e4
    q, s = b200norm.rmsnorm_fp8(torch.ones(1, 256, device=DEV), w, 0.0, group=64)
    torch.testing.assert_close(s, torch.tensor([[1, 1, 1, 1e4]], device=DEV) / 448)
    assert q[0, 200].float() == 448 and q[0, 199].float() == 0.04296875  # 448e-4 = 0.0448 to e4m3


def test_refusals():
    x = torch.randn(4, 64, device=DEV)
    with pytest.raises(RuntimeError, match="residual of shape"):
        b200norm.add_rmsnorm.apply(x, x[:1], None, 1e-6)
    with pytest.raises(RuntimeError, match="dtype"):
        b200norm.add_rmsnorm.apply(x, x.half(), None, 1e-6)
    with pytest.raises(RuntimeError, match="dtype"):
        b200norm.add_rmsnorm.apply(x.double(), x.double(), None, 1e-6)
    with pytest.raises(RuntimeError, match="on cpu"):
        b200norm.add_rmsnorm.apply(x, x.cpu(), None, 1e-6)
    with pytest.raises(RuntimeError, match="64KB"):
        b200norm.add_rmsnorm.apply(torch.zeros(1, 16385, device=DEV), torch.zeros(1, 16385, device=DEV), None, 1e-6)
    with pytest.raises(RuntimeError, match="no gradient"):
        b200norm.rmsnorm_fp8(x.requires_grad_(True))
    x = x.detach()
    with pytest.raises(RuntimeError, match="columns"):
        b200norm.rmsnorm_fp8(x, group=16)
    with pytest.raises(RuntimeError, match="scales"):
        b200norm.rmsnorm_fp8(x, scale_dtype=torch.float16)
    with pytest.raises(RuntimeError, match="float64"):
        b200norm.rmsnorm_fp8(x.double())
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        b200norm.rmsnorm_fp8(x.cpu())


def test_graph_capture_and_replay():
    x, r, w, dy, dh = make(40, 1024, BF16, BF16, BF16)
    A._add_rmsnorm_bwd(*[A._add_rmsnorm_fwd(x, r, w, 1e-6)[1], dy, dh, w, A._add_rmsnorm_fwd(x, r, w, 1e-6)[2]])
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y, h, rstd = A._add_rmsnorm_fwd(x, r, w, 1e-6)
        dx, dres, dw = A._add_rmsnorm_bwd(h, dy, dh, w, rstd)
        q, s, h8 = b200norm.rmsnorm_fp8(x, w, 1e-6, residual=r, group=128)
    for seed in (1, 2):
        nx, nr, _, _, _ = make(40, 1024, BF16, BF16, BF16, seed=seed)
        x.copy_(nx)
        r.copy_(nr)
        g.replay()
        torch.cuda.synchronize()
        check_forward(nx, nr, w, 1e-6, y, h)
        check_backward(h, dy, dh, w, 1e-6, dx, dres, dw)
        assert torch.equal(h8, h)


def test_two_runs_agree_bit_for_bit():
    x, r, w, dy, dh = make(5000, 1001, BF16, F32, BF16)
    a = A._add_rmsnorm_fwd(x, r, w, 1e-6)
    b = A._add_rmsnorm_fwd(x, r, w, 1e-6)
    for u, v in zip(a, b):
        assert torch.equal(u, v)
    c, d = (A._add_rmsnorm_bwd(a[1], dy, dh, w, a[2]) for _ in range(2))
    for u, v in zip(c, d):
        assert torch.equal(u, v)


def test_other_stream():
    x, r, w, dy, dh = make(512, 2048, BF16, BF16, BF16)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        x2 = x * 1
        y, h, rstd = A._add_rmsnorm_fwd(x2, r, w, 1e-6)
        out = A._add_rmsnorm_bwd(h, dy, dh, w, rstd)
    torch.cuda.current_stream().wait_stream(s)
    check_forward(x, r, w, 1e-6, y, h)
    check_backward(h, dy, dh, w, 1e-6, *out)


@pytest.mark.parametrize("t,r", TYPES)
def test_short_rows_of_every_length(t, r):
    # heads and tails of every size around few or no whole packets, several rows to a warp
    for N in list(range(1, 41)) + [119, 127, 135, 255, 257, 263]:
        check(37, N, t, r, F32 if N % 2 else None, with_dh=N % 3 != 0)
        check(6, N, t, r, t, layout="offset")
        x, res, w, _, _ = make(37, N, t, r, t, seed=N)
        check_fp8(x, res if N % 2 else None, w, 1e-6, [0, 32, 64, 128][N % 4], N % 5 == 0)


@pytest.mark.parametrize("t,r", TYPES)
def test_wide_rows_more_than_a_ring_holds(t, r):
    for M, N in [(1301, 4101), (1301, 8199), (901, 10001), (901, 10240), (650, 12296), (650, 16377)]:
        check(M, N, t, r, F32 if N % 2 else t, with_dh=N != 16377)
        x, res, w, _, _ = make(M, N, t, r, t, seed=N)
        check_fp8(x, res if N % 2 else None, w, 1e-6, [0, 32, 64, 128][M % 4], N % 3 == 0)
        check_fp8(x, res, None, 1e-6, 0, False)


@pytest.mark.parametrize("group,e8m0", [(32, True), (64, False), (128, False)])
@pytest.mark.parametrize("t", [F32, F16, BF16])
def test_fp8_scales_over_several_packets_of_a_thread(t, group, e8m0):
    # short rows, where a scale's columns are more than the lanes of a row hold at once
    for N in (8, 24, 40, 64, 72, 96, 104, 120, 128, 136, 192, 200, 256, 264, 512):
        x, res, w, _, _ = make(3001, N, t, t, F32, seed=N)
        check_fp8(x, None, w, 1e-6, group, e8m0)
        check_fp8(x[:5], res[:5], None, 1e-6, group, e8m0)


def exact_rows(M, N, dtype, seed):
    """Rows of +-1, whose root mean square is exactly 1, so that y is the weight with a sign."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randint(0, 2, (M, N), generator=g, device=DEV) * 2 - 1).to(dtype)


@pytest.mark.parametrize("group", [0, 32, 64, 128])
@pytest.mark.parametrize("t,r", [(F32, None), (BF16, None), (BF16, BF16), (F16, F32)])
def test_fp8_quotients_on_a_border_between_two_values(t, r, group):
    # 1 / N and N products of it with 1 add up to 1 in fp32 at these lengths: y is known without an error, and so are
    # its scale, max |y| times 1 / 448, and its quotients, all of them rounded to fp32.  The weights are odd multiples of half
    # a step of e4m3 and of the scale, so the quotients are borders between two values: an ulp either way shows.
    for N in (32, 100, 256, 1000, 1001, 2048, 4104, 8192, 16384):
        g = torch.Generator(device=DEV).manual_seed(N)
        amax = 1.75 * (1 + torch.randint(0, 32, (), generator=g, device=DEV).float() / 32)
        scale = (amax / 448).item()
        half = (1 + (2 * torch.randint(0, 8, (N,), generator=g, device=DEV) + 1).float() / 16)
        w = half * torch.exp2(torch.randint(0, 8, (N,), generator=g, device=DEV).float()) * scale
        w[::32] = amax
        for off in (0, 1):
            n = N - off
            x = exact_rows(5, N + 32, t, N)[:, off:n + off]
            res = torch.zeros(5, N + 32, dtype=r, device=DEV)[:, off:n + off] if r else None
            if float(torch.tensor(1.0) / n * n) != 1.0:
                continue
            q, s, *_ = b200norm.rmsnorm_fp8(x, w[:n], 0.0, residual=res, group=group)
            y = x.float() * w[:n]
            size = group or n
            G = -(-n // size)
            pad = torch.nn.functional.pad(y, (0, G * size - n)).reshape(5, G, size)
            want = pad.abs().amax(-1) * (torch.ones((), device=DEV) / 448)
            assert torch.equal(s, want), (N, off)
            quot = (pad / want[..., None]).reshape(5, G * size)[:, :n].to(torch.float8_e4m3fn)
            assert torch.equal(q.float(), quot.float()), (N, off)


@pytest.mark.parametrize("t", [F32, BF16])
def test_fp8_row_scale_is_finite_where_the_norm_is(t):
    # h w passes the largest number, h w / |h| does not
    for N in (64, 200, 1000, 1001, 4096, 16384):
        x = torch.full((4, N), 1e17, device=DEV).to(t)
        x[1, ::2] *= -1
        x[2] = 1.0
        w = torch.ones(N, device=DEV)
        w[3::5] = 1e22
        w[4::7] = -1e22
        check_fp8(x, None, w, 1e-6, 0, False)
        check_fp8(x, torch.zeros_like(x), w, 1e-6, 0, True)
        check_fp8(x, None, w, 1e-6, 128, False)


def kernels_of(call):
    """Names of the operators' kernels that a call launches."""
    call()
    torch.cuda.synchronize()
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as p:
        call()
        torch.cuda.synchronize()
    names = [e.name for e in p.events() if "addnorm" in e.name]
    return names or pytest.skip("the profiler shows no kernels here")


@pytest.mark.parametrize("t,r,lengths", [(F32, F32, (6340, 6344, 6356, 6368, 6372)), (BF16, BF16, (13568, 13576, 13632, 13648, 13656)),
                                         (F16, F32, (7608, 7616, 7640, 7648, 11416, 11424, 11464, 11472))])
def test_lengths_where_a_ring_just_fits(t, r, lengths):
    # a slot more than the row's kernel has room for sent these to the kernel for unlike alignments
    for N in lengths:
        x, res, w, dy, dh = make(300, N, t, r, t, seed=N)
        y, h, rstd = A._add_rmsnorm_fwd(x, res, w, 1e-6)
        check_backward(h, dy, dh, w, 1e-6, *A._add_rmsnorm_bwd(h, dy, dh, w, rstd))
        check_backward(h, dy, None, w, 1e-6, *A._add_rmsnorm_bwd(h, dy, None, w, rstd))
        names = kernels_of(lambda: A._add_rmsnorm_bwd(h, dy, dh, w, rstd))
        assert any("addnorm_bwd_kernel" in n for n in names), (N, names)  # not the one that works element by element
