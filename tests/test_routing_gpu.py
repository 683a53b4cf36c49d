"""Choice of experts, counts and balance loss on the GPU, against the formulas in 64 bits.

Bounds.  u = 2^-24.  expf is good to 2 u relative and its argument x - max, rounded once, adds |x - max| u; with logits of
a spread below 40 every exponential is good to 44 u, a sum of them to 44 u plus at most 32 + 5 additions, a quotient to one
more: gates to 2 * 90 u relative.  The loss is a sum of positive terms each good to that, with at most T / 16 additions in a
warp and 16 + grid beyond: (200 + T) u.  A gradient is a sum of terms good to 200 u of their magnitudes plus, for the balance
part, the factor's own few roundings: 400 u of the sum of the magnitudes, and its store."""
import pytest
import torch

import b200norm
from b200norm import routing as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24


def reference(x, k, normalize, mask):
    """gates, experts, counts, live, loss in 64 bits; x (T, E)."""
    x = x.double()
    T, E = x.shape
    live = (x > -float("inf")).any(-1)
    if mask is not None:
        live = live & mask.bool()
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :k]
    p = torch.softmax(torch.where(live[:, None], x, torch.zeros_like(x)), -1)
    chosen = live[:, None] & (x.gather(1, order) > -float("inf"))
    gates = p.gather(1, order) * chosen
    if normalize:
        gates = gates / gates.sum(-1, keepdim=True).clamp(min=1e-300)
    counts = torch.zeros(E + 1, dtype=torch.int64, device=x.device)
    counts.scatter_add_(0, torch.where(chosen, order, E).reshape(-1), torch.ones(T * k, dtype=torch.int64, device=x.device))
    n = int(live.sum())
    p = p * live[:, None]
    loss = E * (counts[:E].double() / max(1, n * k) * p.sum(0) / max(1, n)).sum()
    return gates, torch.where(chosen, order, -1), counts[:E], n, loss, p


def reference_grad(p, gates, experts, counts, n, k, normalize, dgates, dloss, live):
    E = p.shape[1]
    c = dloss * E * counts.double() / max(1, n * n * k)
    dg = dgates * (experts >= 0)
    at = experts.clamp(min=0)
    if normalize:
        part = gates * (dg - (gates * dg).sum(-1, keepdim=True))
        d = p * (c - (p * c).sum(-1, keepdim=True))
        size = p * (c.abs() + (p * c.abs()).sum(-1, keepdim=True))
        psize = gates * (dg.abs() + (gates * dg.abs()).sum(-1, keepdim=True))
    else:
        part = gates * dg
        d = p * (c - (p * c).sum(-1, keepdim=True) - part.sum(-1, keepdim=True))
        size = p * (c.abs() + (p * c.abs()).sum(-1, keepdim=True) + part.abs().sum(-1, keepdim=True))
        psize = part.abs()
    d = d.scatter_add(1, at, part * (experts >= 0))
    size = size.scatter_add(1, at, psize * (experts >= 0))
    return d * live[:, None], size * live[:, None]


def check(x, k, normalize, mask=None, dgates=True, dloss=0.3):
    T, E = x.shape
    g, e, buf, loss, lse = R._route_fwd(x, k, normalize, mask)
    rg, re, rc, n, rl, p = reference(x, k, normalize, mask)
    assert torch.equal(e.long(), re)
    assert torch.equal(buf[:E].long(), rc) and int(buf[E]) == n
    assert ((g.double() - rg).abs() <= 180 * U * rg + 1e-37).all()
    assert abs(float(loss) - float(rl)) <= (200 + T) * U * float(rl)
    gen = torch.Generator(device=DEV).manual_seed(T + E)
    dg = torch.randn(T, k, generator=gen, device=DEV) if dgates else None
    dl = torch.full((), dloss, device=DEV) if dloss is not None else None
    got = R._route_bwd(x, g, e, buf, lse, dg, dl, normalize)
    live = (lse > -float("inf")).double()
    ref, size = reference_grad(p, rg, re, rc, n, k, normalize, dg.double() if dgates else torch.zeros_like(rg),
                               dloss or 0.0, live)
    assert got.dtype == x.dtype and got.shape == x.shape
    info = torch.finfo(x.dtype)
    bound = ref.abs() * info.eps / 2 * (1 + 1e-6) + info.smallest_normal * info.eps / 2 + 400 * U * size + 1e-37
    assert ((got.double() - ref).abs() <= bound).all()


def logits(T, E, dtype, seed=0, spread=1.5):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(T, E, generator=g, device=DEV) * spread).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("normalize", [False, True])
def test_sizes(dtype, normalize):
    for T, E, k in [(1, 1, 1), (5, 2, 2), (3, 7, 3), (64, 8, 2), (65, 33, 4), (200, 64, 6), (130, 100, 8), (1000, 128, 8),
                    (77, 160, 6), (300, 256, 8), (40, 511, 5), (64, 512, 32), (50, 1000, 10), (33, 1024, 1)]:
        check(logits(T, E, dtype, seed=E), k, normalize)


@pytest.mark.parametrize("normalize", [False, True])
def test_many_tokens(normalize):
    check(logits(70001, 64, torch.float32), 4, normalize)
    check(logits(30000, 130, torch.bfloat16), 3, normalize, torch.arange(30000, device=DEV) % 3 != 0)


@pytest.mark.parametrize("normalize", [False, True])
def test_masks(normalize):
    x = logits(300, 64, torch.float32)
    mask = torch.rand(300, device=DEV) < 0.5
    check(x, 4, normalize, mask)
    check(x, 4, normalize, mask.to(torch.uint8))
    check(x, 4, normalize, torch.zeros(300, dtype=torch.bool, device=DEV))   # nothing is left
    check(x, 4, normalize, mask, dgates=False)
    check(x, 4, normalize, mask, dloss=None)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("normalize", [False, True])
def test_forbidden_experts_and_empty_rows(dtype, normalize):
    x = logits(200, 40, dtype)
    x[:, ::3] = -float("inf")
    x[5] = -float("inf")          # nothing to choose: not live
    x[6, 2:] = -float("inf")      # one expert for four slots (x[6, 0] is -inf)
    check(x, 4, normalize)
    lowest = logits(20, 8, dtype)
    lowest[:, 4:] = torch.finfo(dtype).min   # masks of the type's lowest value: allowed, weight zero
    check(lowest, 6, normalize)


def test_ties_go_to_the_lower_index():
    x = torch.zeros(4, 70, device=DEV)
    x[1, ::2] = -0.0              # -0 and +0 are one value
    x[2, 30:] = 1.0
    x[3] = torch.arange(70, device=DEV) // 7
    _, e, _, _, _ = R._route_fwd(x, 5)
    assert e.tolist() == [[0, 1, 2, 3, 4], [0, 1, 2, 3, 4], [30, 31, 32, 33, 34], [63, 64, 65, 66, 67]]
    check(x, 5, True)
    check(logits(100, 64, torch.bfloat16, spread=0.02), 8, False)


def test_balanced_loss_is_one_and_collapse_is_not():
    E = 16
    x = torch.full((E * 4, E), -20.0, device=DEV)
    x[torch.arange(E * 4, device=DEV), torch.arange(E * 4, device=DEV) % E] = 20.0
    _, _, counts, loss = b200norm.Router(1)(x)
    assert counts.tolist() == [4] * E
    torch.testing.assert_close(loss, torch.ones((), device=DEV))
    x = torch.full((64, E), -20.0, device=DEV)
    x[:, 3] = 20.0
    torch.testing.assert_close(b200norm.Router(1)(x)[3], torch.full((), float(E), device=DEV))


def test_nan_and_infinity_are_seen():
    x = logits(10, 16, torch.float32)
    x[4, 3] = float("nan")
    g, e, _, loss = b200norm.route.apply(x, 3)
    assert g[4].isnan().all() and loss.isnan() and not g[:4].isnan().any()
    assert ((e >= -1) & (e < 16)).all()
    x[4, 3] = -float("nan")
    assert ((b200norm.route.apply(x, 3)[1] >= -1)).all()
    mask = torch.ones(10, dtype=torch.bool, device=DEV)
    mask[4] = False
    g, e, _, loss = b200norm.route.apply(x, 3, True, mask)
    assert loss.isfinite() and (g[4] == 0).all() and (e[4] == -1).all()


@pytest.mark.parametrize("normalize", [False, True])
def test_module_gradient_against_autograd_in_64_bits(normalize):
    x = logits(24, 12, torch.float32, seed=3).reshape(2, 12, 12).requires_grad_(True)
    router = b200norm.Router(3, normalize)
    gates, experts, counts, loss = router(x)
    assert gates.shape == experts.shape == (2, 12, 3) and counts.shape == (12,) and loss.shape == ()
    a = torch.randn_like(gates)
    (gates * a).sum().add(loss, alpha=2.0).backward()
    y = x.detach().double().requires_grad_(True)
    p = torch.softmax(y, -1)
    g = p.gather(-1, experts.long())
    if normalize:
        g = g / g.sum(-1, keepdim=True)
    bal = 12 * (counts.double() / (24 * 3) * p.reshape(24, 12).mean(0)).sum()
    (g * a.double()).sum().add(bal, alpha=2.0).backward()
    torch.testing.assert_close(x.grad.double(), y.grad, rtol=1e-5, atol=1e-6)


def test_gradient_against_differences():
    # where the choice does not change; error of the difference h^2 |f'''| / 6 + u |f| / h ~ 2e-5 + 1e-4 at h = 1e-2
    x = (torch.arange(60, device=DEV).reshape(5, 12) * 7 % 12).float() * 0.3
    a = torch.randn(5, 3, device=DEV, generator=torch.Generator(device=DEV).manual_seed(0))
    d = torch.randn(5, 12, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1))
    for normalize in (False, True):
        def f(v):
            gates, _, _, loss = b200norm.route.apply(v, 3, normalize)
            return (gates.double() * a).sum() + 5 * loss.double()
        v = x.clone().requires_grad_(True)
        grad, = torch.autograd.grad(f(v), v)
        num = (f(x + 1e-2 * d) - f(x - 1e-2 * d)) / 2e-2
        assert abs(float(num) - float((grad * d).sum())) <= 2e-3 * float((grad.abs() * d.abs()).sum())


def test_strides_and_orders():
    base = logits(90, 200, torch.bfloat16)
    check(base[:, 3:67], 4, True)
    check(base[::2, :128], 4, False)
    check(base.t()[:64], 4, True)
    check(base[:1, :64].expand(50, 64), 4, True)


def test_empty_batch():
    x = torch.empty(0, 16, device=DEV, requires_grad=True)
    gates, experts, counts, loss = b200norm.route.apply(x, 2)
    assert gates.shape == (0, 2) and counts.tolist() == [0] * 16 and float(loss.detach()) == 0
    (gates.sum() + loss).backward()
    assert x.grad.shape == (0, 16)


def test_two_runs_agree_and_graphs_replay():
    x = logits(20000, 96, torch.float32)
    a, b = R._route_fwd(x, 6), R._route_fwd(x, 6)
    assert all(torch.equal(u, v) for u, v in zip(a, b))
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = []
    for g in graphs:  # each keeps its own workspace
        with torch.cuda.graph(g):
            o = R._route_fwd(x, 6)
            outs.append(o + (R._route_bwd(x, o[0], o[1], o[2], o[4], None, o[3]),))
    want = R._route_bwd(x, a[0], a[1], a[2], a[4], None, a[3])
    for _ in range(2):
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for o in outs:
            assert all(torch.equal(u, v) for u, v in zip(o, a)) and torch.equal(o[5], want)


def test_refusals():
    x = logits(4, 16, torch.float32)
    for k in (0, 17, 33):
        with pytest.raises(RuntimeError, match="top_k"):
            b200norm.route.apply(x, k)
    with pytest.raises(RuntimeError, match="experts"):
        b200norm.route.apply(logits(2, 1025, torch.float32), 2)
    with pytest.raises(RuntimeError, match="mask"):
        b200norm.route.apply(x, 2, True, torch.ones(5, dtype=torch.bool, device=DEV))
    with pytest.raises(RuntimeError, match="mask"):
        b200norm.route.apply(x, 2, True, torch.ones(4, device=DEV))
    with pytest.raises(RuntimeError, match="float64"):
        b200norm.route.apply(x.double(), 2)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        b200norm.route.apply(x.cpu(), 2)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_returned_counts_are_the_callers(dtype):
    for T in (100, 3000):
        x = logits(T, 64, dtype, seed=1)
        grads = []
        # as it is; behind the version counter's back, as a collective changes it; in the open
        for change in (lambda c: None, lambda c: c.data.mul_(8), lambda c: c.mul_(8)):
            v = x.clone().requires_grad_(True)
            gates, experts, counts, loss = b200norm.route.apply(v, 4)
            change(counts)
            (loss + gates.square().sum()).backward()
            grads.append(v.grad)
        assert torch.equal(grads[0], grads[1]) and torch.equal(grads[0], grads[2])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("normalize", [False, True])
def test_logits_far_from_zero(dtype, normalize):
    # The kernels' exponentials are good to 2 u and, beyond what check() derives, to |d| 1.3 u more for the product d log2 e
    # (half an ulp of it, and log2 e's own): below 32 u for the differences d of up to 13 here, of 44 u.
    for E, k in ((64, 4), (7, 2), (33, 3), (160, 6), (512, 8)):
        x = logits(90, E, torch.float32, seed=E)
        for offset in (1e4, -1e4, 1e6, -1e6, 1e30, -1e30):
            check((x + offset).to(dtype), k, normalize)
        y = x.to(dtype)
        y[::2] = torch.finfo(dtype).min
        y[1] = torch.finfo(dtype).max
        check(y, k, normalize)


def test_masked_tokens_get_no_gradient_whatever_the_loss():
    x = logits(40, 32, torch.float32)
    x[::3, 5] = float("nan")
    mask = torch.arange(40, device=DEV) % 3 != 0
    for dl in (float("inf"), float("nan")):
        v = x.clone().requires_grad_(True)
        gates, _, _, loss = b200norm.route.apply(v, 4, True, mask)
        torch.autograd.backward([gates, loss], [torch.full_like(gates, float("inf")), torch.full((), dl, device=DEV)])
        assert (v.grad[~mask] == 0).all()


def test_negative_nan_shows():
    for normalize in (False, True):
        for E in (8, 16, 64, 300, 1000):
            x = logits(10, E, torch.float32)
            x.view(torch.int32)[4, 3] = -1  # a NaN with its sign set
            g, e, _, loss = b200norm.route.apply(x, 3, normalize)
            assert g[4].isnan().all() and loss.isnan() and g[[0, 1, 2, 3, 5, 6, 7, 8, 9]].isfinite().all()
            assert ((e >= 0) & (e < E)).all()


def test_hooks_that_round_saved_numbers():
    # saved tensors in 16 bits: logits that have no more, gates and log-sums off by 2^-9; the counts are whole numbers
    x = logits(700, 64, torch.bfloat16).float()

    def grad(loss_weight):
        v = x.clone().requires_grad_(True)
        gates, _, _, loss = b200norm.route.apply(v, 4)
        return torch.autograd.grad(loss_weight * loss + (gates * gates).sum() * 1e-3, v)[0]

    want = grad(100.0)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.bfloat16().float() if t.is_floating_point() else t, lambda t: t):
        got = grad(100.0)
    assert (got - want).norm() <= 2.0 ** -6 * want.norm()


def test_experts_that_are_none_get_no_gradient():
    # the saved choices, changed where no version counter sees it, to others that do not exist
    x = logits(50, 40, torch.float32)
    for normalize in (False, True):
        v = x.clone().requires_grad_(True)
        gates, experts, _, _ = b200norm.route.apply(v, 4, normalize)
        o = R._route_fwd(x, 4, normalize)
        dg = torch.randn(50, 4, device=DEV)
        none = o[1].clone()
        none[::2, 1] = -1
        experts.data[::2, 1] = torch.tensor([40, 64, 2 ** 31 - 1, -2, -2 ** 31], device=DEV, dtype=torch.int32).repeat(5)
        got, = torch.autograd.grad(gates, v, dg)
        assert torch.equal(got, R._route_bwd(x, o[0], none, o[2], o[4], dg, None, normalize))
