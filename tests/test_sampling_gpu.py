"""Choice of a token on the GPU, against the definition in 64 bits.  Tokens have to be equal: the operator's weights are
good to 2^-44 of the likeliest token's, so a token may differ only when u * total falls within V * 2^-44 of a border between
two tokens, which for the tests' sizes happens once in some 10^7 draws."""
import pytest
import torch

import b200norm

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
INF = float("inf")


def reference(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    x = logits.float()
    M, V = x.shape

    def col(v, dtype=torch.float32):
        return torch.as_tensor(v, dtype=dtype, device=x.device).double().expand(M).reshape(M, 1)

    T, k, p, mp = col(temperature), col(top_k, torch.int32), col(top_p), col(min_p)
    top = x.amax(-1, keepdim=True)
    d = torch.where(x == top, torch.zeros_like(x, dtype=torch.float64), x.double() - top.double())
    w = torch.exp(d / torch.where(T > 0, T, torch.ones_like(T)))
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices
    ranked = w.gather(1, order)
    rank = torch.arange(V, device=x.device)
    keep = (k < 1) | (k >= V) | (rank < k)
    total = (ranked * keep).sum(-1, keepdim=True)
    before = (ranked * keep).cumsum(-1) - ranked * keep
    keep = keep & ((p >= 1) | (before < p * total) | (rank == 0))
    keep = keep & (ranked >= mp.clamp(max=1))
    keep = torch.where(T > 0, keep, rank == 0)
    kept = torch.zeros_like(w).scatter_(1, order, ranked * keep)
    cum = kept.cumsum(-1)
    token = (cum > u.double().reshape(M, 1) * cum[:, -1:]).to(torch.int8).argmax(-1)
    return torch.where(x.isnan().any(-1) | (top[:, 0] == -INF), -1, token)


def make(M, V, dtype, seed=0, scale=2.5):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(M, V, generator=g, device=DEV) * scale
    at = torch.randint(V, (M, 6), generator=g, device=DEV)
    x.scatter_add_(1, at, 4 + 4 * torch.rand(M, 6, generator=g, device=DEV))
    return x.to(dtype), torch.rand(M, generator=g, device=DEV)


def check(x, u, **kw):
    got = b200norm.sample(x, u, **kw)
    assert got.dtype == torch.int64 and got.shape == u.shape
    want = reference(x.reshape(-1, x.shape[-1]), u.reshape(-1), **{k: v.reshape(-1) if isinstance(v, torch.Tensor) else v
                                                                    for k, v in kw.items()})
    assert torch.equal(got.reshape(-1), want), (kw, got.tolist()[:16], want.tolist()[:16])


SETTINGS = [dict(), dict(temperature=0.6), dict(temperature=0.0), dict(top_k=1), dict(top_k=5), dict(top_k=50, temperature=1.7),
            dict(top_p=0.9), dict(top_p=0.3, temperature=0.5), dict(top_p=0.0), dict(min_p=0.05), dict(min_p=1.0),
            dict(top_k=40, top_p=0.8, min_p=0.02, temperature=0.9), dict(top_k=1000, top_p=0.99, temperature=3.0)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("kw", SETTINGS, ids=str)
def test_settings(dtype, kw):
    for M, V in [(1, 1), (4, 2), (3, 17), (64, 1000), (33, 4099), (5, 32768), (7, 50001), (3, 131072), (2, 262144)]:
        x, u = make(M, V, dtype, seed=V)
        check(x, u, **kw)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_many_rows(dtype):
    x, u = make(700, 9001, dtype)
    check(x, u, temperature=0.8, top_p=0.9)
    x, u = make(300, 33000, dtype)
    check(x, u, top_k=20)
    check(x, u)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_settings_per_row(dtype):
    M, V = 48, 20011
    x, u = make(M, V, dtype, seed=9)
    g = torch.Generator(device=DEV).manual_seed(4)
    t = torch.rand(M, generator=g, device=DEV) * 2
    t[::7] = 0
    k = torch.randint(0, 200, (M,), generator=g, device=DEV)
    k[::5] = 0
    k[3] = -4
    k[4] = V + 10
    p = torch.rand(M, generator=g, device=DEV) * 1.2
    mp = torch.rand(M, generator=g, device=DEV) * 0.3
    mp[1] = 7.0
    check(x, u, temperature=t, top_k=k, top_p=p, min_p=mp)
    check(x, u, temperature=t.double(), top_k=k.to(torch.int32), top_p=0.7)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_equal_logits(dtype):
    # ties: first by index, at every border
    u = torch.tensor([0.0, 0.25, 0.5, 0.999], device=DEV)
    x = torch.full((4, 8192), 1.5, dtype=dtype, device=DEV)
    assert b200norm.sample(x, u).tolist() == [0, 2048, 4096, int(0.999 * 8192)]
    assert b200norm.sample(x, u, top_k=100).tolist() == [0, 25, 50, 99]
    assert b200norm.sample(x, u, top_p=0.5).tolist() == [0, 1024, 2048, int(0.999 * 4096)]
    assert b200norm.sample(x, u, temperature=0).tolist() == [0] * 4
    for kw in SETTINGS:
        check(x, u, **kw)
    x[:, 1000:] = -3.0
    x[:, 5::3] = 2.25
    for kw in SETTINGS:
        check(x, u, **kw)
    coarse = (torch.randn(16, 40000, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)) * 2).round().to(dtype)
    u = torch.rand(16, device=DEV)
    for kw in SETTINGS:
        check(coarse, u, **kw)
    signs = torch.zeros(2, 5000, dtype=dtype, device=DEV)
    signs[:, ::2] = -0.0          # -0 and +0 are one value
    check(signs, u[:2], top_k=7)
    assert b200norm.sample(signs, u[:2], temperature=0).tolist() == [0, 0]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_masked_and_extreme_logits(dtype):
    x, u = make(12, 6007, dtype, seed=2)
    x[0, 1:] = -INF                         # one token left
    x[1] = -INF                             # none
    x[2, 100] = float("nan")
    x[3, :6000] = -INF
    x[4] = torch.finfo(dtype).min           # masks of the type's lowest value
    x[4, 17] = 0.0
    x[5] = torch.finfo(dtype).min           # ... and nothing else
    x[6, 50] = INF
    x[6, 70] = INF
    x[7] = x[7] * 1000 if dtype != torch.float16 else x[7] * 100
    x[8] = x[8] * 1e-3
    x[9] = -x[9].abs() - 1
    x[10, 8] = -float("nan")
    x[11] = -INF                            # the lowest number is the maximum, beside -inf
    x[11, 40:50] = torch.finfo(dtype).min
    for kw in SETTINGS:
        check(x, u, **kw)
    assert b200norm.sample(x, u)[[0, 1, 2, 10]].tolist() == [0, -1, -1, -1]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_large_offsets_and_extreme_temperatures(dtype):
    # logits far from zero, where a step of fp32 is larger than the temperature, and temperatures at both ends
    x, u = make(6, 5000, dtype, seed=8)
    for offset in (1e4, -1e4, 1e10, -1e10, 3e38, -3e38):
        y = (x.float() + offset).to(dtype)
        for kw in (dict(), dict(top_p=0.7), dict(top_k=30, min_p=0.1), dict(temperature=0.01), dict(top_p=0.5, temperature=20.0)):
            check(y, u, **kw)
    x[:, ::9] = -INF
    for t in (1e-30, 1e-3, 1e3, 1e35):
        check(x, u, temperature=t)
        check(x, u, temperature=t, top_k=700, top_p=0.6)
        check(x, u, temperature=t, min_p=0.5, top_p=0.9)


def test_wide_prefixes():
    # neither list nor bin holds few tokens: flat rows, many equal logits, top-k beyond the list
    g = torch.Generator(device=DEV).manual_seed(3)
    u = torch.rand(8, generator=g, device=DEV)
    flat = torch.rand(8, 100000, generator=g, device=DEV) * 0.01
    for x in (flat, flat.bfloat16(), flat * 1e-4 - 7, (flat * 300).round()):
        for kw in (dict(top_p=0.9), dict(top_k=3000), dict(top_k=99999, top_p=0.999), dict(top_k=600, top_p=0.4, min_p=0.5),
                   dict(top_k=257), dict(top_k=255), dict(top_p=1e-3), dict(top_k=513, top_p=0.999999)):
            check(x, u, **kw)


def test_uniform_at_its_ends():
    x, _ = make(3, 3000, torch.float32)
    u = torch.tensor([0.0, 1 - 2.0 ** -24, 0.5], device=DEV)
    check(x, u)
    check(x, u, top_p=0.5)
    # out of range: cut to it
    assert torch.equal(b200norm.sample(x, torch.tensor([-1.0, 1.0, 0.5], device=DEV))[::2], b200norm.sample(x, u)[::2])
    assert (b200norm.sample(x, torch.tensor([float("nan"), 2.0, 1.0], device=DEV)) >= 0).all()


def test_frequencies_follow_the_distribution():
    # 200000 draws of 5 tokens: five standard deviations of a share are below 5 * sqrt(0.25 / 2e5) = 0.0056
    logits = torch.tensor([0.0, 1.0, 2.0, -1.0, 0.5], device=DEV)
    n = 200000
    u = torch.rand(n, device=DEV, generator=torch.Generator(device=DEV).manual_seed(0))
    t = b200norm.sample(logits.expand(n, 5), u, temperature=0.7)
    share = torch.bincount(t, minlength=5) / n
    assert ((share - torch.softmax(logits / 0.7, 0)).abs() < 0.0056).all()


def test_batch_and_split_do_not_matter():
    # the same row alone (spread over eight CTAs) and in a batch (over two): the same token
    x, u = make(200, 30000, torch.bfloat16, seed=6)
    all_rows = b200norm.sample(x, u, top_p=0.95)
    for i in (0, 17, 199):
        assert torch.equal(b200norm.sample(x[i:i + 1], u[i:i + 1], top_p=0.95), all_rows[i:i + 1])


def test_strides_orders_and_shapes():
    base, _ = make(20, 5000, torch.bfloat16)
    u = torch.rand(20, device=DEV)
    check(base[:, 3:4000], u, top_p=0.9)
    check(base[:, ::2], u, top_k=9)
    check(base.t()[:20, :20].contiguous().t(), u, top_k=9)
    check(base[:1].expand(20, 5000), u)
    check(base.reshape(4, 5, 5000), u.reshape(4, 5), temperature=torch.full((4, 5), 0.5, device=DEV))
    one = b200norm.Sampler(top_k=3)(base[0], u[0])
    assert one.shape == () and torch.equal(one, b200norm.sample(base[:1], u[:1], top_k=3)[0])
    assert b200norm.sample(base[:0], u[:0]).shape == (0,)


def test_graph_replay_and_other_stream():
    x, u = make(16, 40000, torch.bfloat16)
    b200norm.sample(x, u, top_k=40, top_p=0.9)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        t = b200norm.sample(x, u, top_k=40, top_p=0.9)
    for seed in (1, 2, 3):
        nx, nu = make(16, 40000, torch.bfloat16, seed=seed)
        x.copy_(nx)
        u.copy_(nu)
        g.replay()
        assert torch.equal(t, reference(nx, nu, top_k=40, top_p=0.9))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        t = b200norm.sample(x, u)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(t, reference(x, u))


def test_refusals():
    x, u = make(4, 100, torch.float32)
    for kw, what in ((dict(temperature=-1.0), "temperature"), (dict(top_p=1.5), "top_p"), (dict(min_p=-0.1), "min_p"),
                     (dict(top_k=-1), "top_k"), (dict(temperature=float("nan")), "temperature"),
                     (dict(top_k=torch.ones(4, device=DEV)), "top_k"), (dict(top_p=torch.ones(4, device=DEV, dtype=torch.int32)), "top_p"),
                     (dict(top_p=torch.ones(3, device=DEV)), "top_p"), (dict(min_p=torch.ones(4)), "min_p")):
        with pytest.raises(RuntimeError, match=what):
            b200norm.sample(x, u, **kw)
    for bad in (u[:3], u.cpu(), u.long()):
        with pytest.raises(RuntimeError, match="uniform"):
            b200norm.sample(x, bad)
    with pytest.raises(RuntimeError, match="262144"):
        b200norm.sample(torch.zeros(1, 262145, device=DEV), u[:1])
    with pytest.raises(RuntimeError, match="float64"):
        b200norm.sample(x.double(), u)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        b200norm.sample(x.cpu(), u.cpu())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_prefixes_that_end_above_and_below_min_p(dtype):
    x, u = make(40, 30011, dtype, seed=8)
    flat = (torch.randn(40, 30011, generator=torch.Generator(device=DEV).manual_seed(3), device=DEV) * 0.7).to(dtype)
    for rows in (x, flat):
        for p in (0.05, 0.5, 0.9, 0.999):
            for mp in (1e-9, 1e-4, 0.02, 0.4, 0.999, 1.0):
                check(rows, u, top_p=p, min_p=mp)
                check(rows, u, top_p=p, min_p=mp, top_k=3000, temperature=1.4)
    spread = torch.linspace(0, 1, 40, device=DEV)
    check(x, u, top_p=0.3 + 0.7 * spread.flip(0), min_p=0.1 * spread ** 3, temperature=0.8)


def test_top_k_of_64_bits_without_a_sign():
    x, u = make(6, 1000, torch.float32)
    for many in (2 ** 32 + 5, 2 ** 63 + 5):
        k = torch.full((6,), many, dtype=torch.uint64, device=DEV)
        assert torch.equal(b200norm.sample(x, u, top_k=k), b200norm.sample(x, u))
    k = torch.full((6,), 5, dtype=torch.uint64, device=DEV)
    assert torch.equal(b200norm.sample(x, u, top_k=k), b200norm.sample(x, u, top_k=5))


def test_a_row_alone_over_eight_ctas_and_in_a_batch_over_two():
    # 40000 fp32: parts of 20 KB when alone, of 80 KB when 200 rows fill the SMs
    x, u = make(200, 40000, torch.float32, seed=6)
    for kw in (dict(), dict(top_k=50), dict(top_k=2000), dict(top_p=0.95), dict(min_p=0.01), dict(top_k=3000, top_p=0.9, min_p=1e-3)):
        whole = b200norm.sample(x, u, **kw)
        assert torch.equal(whole, reference(x, u, **kw))
        for i in range(200):
            assert torch.equal(b200norm.sample(x[i:i + 1], u[i:i + 1], **kw), whole[i:i + 1])
