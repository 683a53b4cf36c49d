"""The residual norms, the expert choice and the token choice as they are used together: a training step, a serving step in
one CUDA graph, several streams and threads, outputs inside larger buffers, rows more than 2^31 elements apart."""
import subprocess
import sys
import threading
from pathlib import Path

import pytest
import torch

import b200norm
from b200norm import _lib
from b200norm import addnorm as A
from b200norm import routing as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def randn(*shape, seed=0, dtype=F32, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)


def rand(*shape, seed=0):
    return torch.rand(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV)


# ---- training: two blocks of residual norm, router, and a product that stands for the experts -------------------------------

class Block(torch.nn.Module):
    def __init__(self, n, experts, k, dtype, seed):
        super().__init__()
        self.norm = b200norm.AddRMSNorm(n, eps=1e-6, device=DEV, dtype=dtype)
        self.router = torch.nn.Parameter(randn(n, experts, seed=seed, dtype=dtype, scale=n ** -0.5))
        self.bank = torch.nn.Parameter(randn(experts, n, seed=seed + 1, dtype=dtype))
        self.route = b200norm.Router(k)

    def forward(self, x, residual, mask):
        y, h = self.norm(x, residual)
        gates, experts, counts, loss = self.route(y @ self.router, mask)
        chosen = self.bank[experts.clamp(min=0).long()]
        return (gates.to(y.dtype).unsqueeze(-1) * chosen).sum(-2) * y, h, loss, experts, counts


def plain_block(x, residual, norm_w, router, bank, experts, counts, k, mask):
    """The block in 64 bits, with the choice that the operator made."""
    h = x + residual
    y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-6) * norm_w
    p = torch.softmax(y @ router, -1)
    on = (experts >= 0)
    at = experts.clamp(min=0).long()
    g = p.gather(-1, at) * on
    g = g / g.sum(-1, keepdim=True).clamp(min=1e-300)
    n = int(mask.sum())
    loss = p.shape[-1] * (counts.double() / (n * k) * (p * mask.unsqueeze(-1)).reshape(-1, p.shape[-1]).sum(0) / n).sum()
    return (g.unsqueeze(-1) * bank[at]).sum(-2) * y, h, loss


def test_a_training_step_against_autograd_in_64_bits():
    # Every stage (norm, product, softmax, gates, gather, product) errs by at most 400 * 2^-24 of the sum of the magnitudes
    # of its terms, forward and backward; a sum of 48 terms has magnitudes up to sqrt(48) < 8 times its norm; two blocks of
    # five stages, both ways: 20 * 400 * 8 * 2^-24 < 2^-8 of a gradient's norm.
    n, E, k = 48, 12, 3
    blocks = [Block(n, E, k, F32, seed) for seed in (1, 11)]
    for i, b in enumerate(blocks):
        b.norm.weight.data.copy_(1 + 0.1 * randn(n, seed=30 + i))
    x, res = randn(2, 33, n, seed=3).requires_grad_(True), randn(2, 33, n, seed=4).requires_grad_(True)
    mask = torch.ones(2, 33, dtype=torch.bool, device=DEV)
    mask[1, 20:] = False  # a padded batch
    seen = []
    a, h, total = x, res, 0.
    for b in blocks:
        a, h, loss, experts, counts = b(a, h, mask)
        seen.append((experts, counts))
        total = total + 0.5 * loss
        assert (experts[~mask] == -1).all() and int(counts.sum()) == int(mask.sum()) * k
    weight = randn(2, 33, n, seed=5)
    ((a * weight).sum() + (h * weight.flip(0)).sum() + total).backward()
    leaves = [x, res] + [p for b in blocks for p in (b.norm.weight, b.router, b.bank)]

    wide = [t.detach().double().requires_grad_(True) for t in leaves]
    a, h, total = wide[0], wide[1], 0.
    for i, (experts, counts) in enumerate(seen):
        a, h, loss = plain_block(a, h, *wide[2 + 3 * i:5 + 3 * i], experts, counts, k, mask)
        total = total + 0.5 * loss
    ((a * weight.double()).sum() + (h * weight.flip(0).double()).sum() + total).backward()
    for got, want in zip(leaves, wide):
        assert (got.grad.double() - want.grad).norm() <= 2.0 ** -8 * want.grad.norm()


def test_a_bf16_step_is_its_operators_one_by_one():
    n, E, k = 256, 16, 2
    x, res, w = randn(70, n, dtype=BF16), randn(70, n, seed=1), (1 + 0.1 * randn(n, seed=2)).to(BF16)
    m = randn(n, E, seed=3, dtype=BF16, scale=n ** -0.5)
    leaves = [t.detach().requires_grad_(True) for t in (x, res, w, m)]
    y, h = b200norm.add_rmsnorm.apply(*leaves[:3], 1e-6)
    logits = y @ leaves[3]
    gates, experts, counts, loss = b200norm.route.apply(logits, k, False, None)
    dg, dh = randn(70, k, seed=4), randn(70, n, seed=5)
    torch.autograd.backward([gates, loss, h], [dg, torch.full((), 0.25, device=DEV), dh])

    y2, h2, rstd = A._add_rmsnorm_fwd(x, res, w, 1e-6)
    out = R._route_fwd(y2 @ m, k, False)
    assert torch.equal(y, y2) and torch.equal(h, h2) and torch.equal(gates, out[0]) and torch.equal(experts, out[1])
    assert torch.equal(counts, out[2][:-1]) and torch.equal(loss, out[3])
    dl = R._route_bwd(y2 @ m, out[0], out[1], out[2], out[4], dg, torch.full((), 0.25, device=DEV), False)
    dx, dres, dw = A._add_rmsnorm_bwd(h2, dl @ m.t(), dh, w, rstd)
    for leaf, want in zip(leaves, (dx, dres, dw)):
        assert leaf.grad.dtype == leaf.dtype and torch.equal(leaf.grad, want)
    torch.testing.assert_close(leaves[3].grad, y2.t() @ dl, rtol=2 ** -7, atol=2 ** -12)  # the library's product


def test_gradients_that_are_broadcast():
    # the gradient of a sum is one number, expanded: stride 0 in every direction
    x, r = randn(9, 100, dtype=BF16).requires_grad_(True), randn(9, 100, seed=1, dtype=BF16).requires_grad_(True)
    y, h = b200norm.add_rmsnorm.apply(x, r, None, 1e-6)
    (y.sum() + h.sum()).backward()
    want = A._add_rmsnorm_bwd(h.detach(), torch.ones_like(x), torch.ones_like(x), None, A._add_rmsnorm_fwd(x, r, None, 1e-6)[2])
    assert torch.equal(x.grad, want[0]) and torch.equal(r.grad, want[1])
    l = randn(9, 16).requires_grad_(True)
    gates, experts, counts, loss = b200norm.route.apply(l, 3, False)
    gates.sum().backward()
    o = R._route_fwd(l.detach(), 3, False)
    assert torch.equal(l.grad, R._route_bwd(l.detach(), o[0], o[1], o[2], o[4], torch.ones(9, 3, device=DEV), None, False))


def test_a_training_step_captured_in_a_graph():
    n, E, k = 128, 8, 2
    x, res = randn(40, n, dtype=BF16).requires_grad_(True), randn(40, n, seed=1, dtype=BF16).requires_grad_(True)
    w, m = torch.ones(n, device=DEV, dtype=BF16, requires_grad=True), randn(n, E, seed=2, dtype=BF16).requires_grad_(True)
    mask = torch.ones(40, dtype=torch.bool, device=DEV)

    def step():
        y, h = b200norm.add_rmsnorm.apply(x, res, w, 1e-6)
        gates, experts, counts, loss = b200norm.route.apply(y @ m, k, True, mask)
        grads = torch.autograd.grad((gates * gates).sum() + loss + h.float().square().mean(), [x, res, w, m])
        return [t.detach() for t in (y, h, gates, experts, counts, loss)] + list(grads)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (5, 6):
        with torch.no_grad():
            x.copy_(randn(40, n, seed=seed, dtype=BF16))
            mask.copy_(torch.arange(40, device=DEV) % seed != 0)
        for t in out:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(out, step()):
            # the products in between are the library's, which may take another algorithm when captured
            torch.testing.assert_close(got, want, rtol=2 ** -6, atol=2 ** -7)


# ---- serving ----------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("M", [1, 5, 64])
def test_a_serving_step_in_one_graph(M):
    n, V = 512, 4099
    first = b200norm.RMSNormFP8(n, eps=1e-6, group=128, device=DEV, dtype=BF16)
    last = b200norm.AddRMSNorm(n, eps=1e-6, device=DEV, dtype=BF16)
    mix, head = randn(n, n, seed=1, dtype=BF16, scale=n ** -0.5), randn(n, V, seed=2, dtype=BF16, scale=3 * n ** -0.5)
    pick, router = b200norm.Sampler(temperature=0.8, top_k=40, top_p=0.95), b200norm.Router(2)
    x, res, u = randn(M, n, seed=3, dtype=BF16), randn(M, n, seed=4), rand(M, seed=5)

    @torch.no_grad()
    def step():
        q, scale, h = first(x, res)
        z = (q.float() * scale.repeat_interleave(128, -1)).to(BF16) @ mix
        y, h2 = last(z, h)
        logits = y @ head
        routed = router(y[:, :64])
        return dict(q=q, scale=scale, h=h, z=z, y=y, h2=h2, logits=logits, routed=routed, token=pick(logits, u))

    for _ in range(2):
        step()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):  # two graphs of the same step share nothing
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step())
        graphs.append(g)
    for seed in (11, 12, 13):
        x.copy_(randn(M, n, seed=seed, dtype=BF16))
        u.copy_(rand(M, seed=seed))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        with torch.no_grad():
            for o in outs:  # each operator's output is what it makes of the graph's own intermediate results
                q, scale, h = first(x, res)
                assert torch.equal(o["q"].view(torch.uint8), q.view(torch.uint8)) and torch.equal(o["scale"], scale)
                assert torch.equal(o["h"], h) and torch.equal(h, x.float() + res)
                y, h2 = last(o["z"], o["h"])
                assert torch.equal(o["y"], y) and torch.equal(o["h2"], h2)
                assert torch.equal(o["token"], pick(o["logits"], u)) and ((o["token"] >= 0) & (o["token"] < V)).all()
                assert all(torch.equal(a, b) for a, b in zip(o["routed"], router(o["y"][:, :64])))


def all_operators(seed, M=300, n=1000, V=20011):
    """One call of each, with its inputs drawn from the seed; every output in one list."""
    x, r, w = randn(M, n, seed=seed, dtype=BF16), randn(M, n, seed=seed + 1, dtype=BF16), randn(n, seed=seed + 2, dtype=BF16)
    logits, u = randn(64, V, seed=seed + 3, dtype=BF16, scale=3.0), rand(64, seed=seed + 4)

    def run():
        y, h, rstd = A._add_rmsnorm_fwd(x, r, w, 1e-6)
        out = [y, h, rstd, *A._add_rmsnorm_bwd(h, y, r, w, rstd)]
        with torch.no_grad():
            q, s, h8 = b200norm.rmsnorm_fp8(x, w, 1e-6, residual=r, group=64)
        out += [q.view(torch.uint8), s, h8]
        routed = R._route_fwd(x[:, :96], 4)
        out += [*routed, R._route_bwd(x[:, :96], routed[0], routed[1], routed[2], routed[4], routed[0], routed[3])]
        return out + [b200norm.sample(logits, u, top_p=0.9), b200norm.sample(logits, u, top_k=30)]

    return run


def test_streams_at_once():
    runs = [all_operators(100 * i) for i in range(3)]
    want = [run() for run in runs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in runs]
    got = [[] for _ in runs]
    for _ in range(4):
        for i, (run, s) in enumerate(zip(runs, streams)):
            with torch.cuda.stream(s):
                got[i].append(run())
    torch.cuda.synchronize()
    for a, g in zip(want, got):
        for b in g:
            assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_threads_at_once():
    runs = [all_operators(100 * i, M=70) for i in range(4)]
    want = [run() for run in runs]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(5):
                    out = runs[i]()
                    torch.cuda.current_stream().synchronize()
                    if not all(torch.equal(u, v) for u, v in zip(want[i], out)):
                        wrong.append(i)
        except Exception as exc:  # noqa: BLE001 -- shown by the assertion below
            wrong.append(exc)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert wrong == []


# ---- outputs inside larger buffers: what lies around them stays as it was -----------------------------------------------------

CODE = {F32: _lib.F32, F16: _lib.F16, BF16: _lib.BF16}


class Frame:
    """Rows inside a buffer of a fixed byte: M rows of n from element `lead`, `stride` apart."""

    def __init__(self, M, n, dtype, lead, gap, source=None):
        size = torch.empty((), dtype=dtype).element_size()
        self.buf = torch.full((lead * size + (M + 2) * (n + gap) * size,), 0x5A, dtype=torch.uint8, device=DEV)
        self.rows = self.buf.view(dtype).as_strided((M, n), (n + gap, 1), lead)
        if source is not None:
            self.rows.copy_(source)
        self.inside = torch.zeros(self.buf.numel() // size, dtype=torch.bool, device=DEV)
        self.inside.as_strided((M, n), (n + gap, 1), lead).fill_(True)
        self.size = size

    def check(self):
        outside = ~self.inside.repeat_interleave(self.size)
        assert (self.buf[outside] == 0x5A).all()

    @property
    def at(self):
        return self.rows.data_ptr(), self.rows.stride(0)


@pytest.mark.parametrize("t,r", [(BF16, BF16), (F16, F32), (F32, F32)])
@pytest.mark.parametrize("n,leads,gap", [(512, (0,) * 5, 64), (501, (3,) * 5, 11), (100, (8, 0, 1, 5, 2), 7), (4099, (5,) * 5, 5)])
def test_nothing_around_the_rows_is_written(t, r, n, leads, gap):
    lib, M = _lib.load(), 37
    s = torch.cuda.current_stream().cuda_stream
    x, res, dy, dh = (randn(M, n, seed=i, dtype=d) for i, d in enumerate((t, r, t, r)))
    w = randn(n, seed=9)
    fx, fr, fy = Frame(M, n, t, leads[0], gap, x), Frame(M, n, r, leads[1], gap, res), Frame(M, n, t, leads[2], gap)
    fh, fq = Frame(M, n, r, leads[3], gap), Frame(M, n, torch.uint8, leads[2], gap)
    rstd = torch.zeros(M + 8, device=DEV)
    _lib.check(lib.b200norm_add_rms_fwd(*fx.at, *fr.at, w.data_ptr(), *fy.at, *fh.at, rstd.data_ptr(), M, n, 1e-6, CODE[t],
                                        CODE[r], _lib.F32, s))
    y, h, rs = A._add_rmsnorm_fwd(x, res, w, 1e-6)
    # the layouts differ, and with them the order of a sum: 104 halves of 2^-23 on it, a step on the store
    close = dict(rtol=max(2 * torch.finfo(t).eps, 2.0 ** -16), atol=2.0 ** -24)
    assert torch.equal(fh.rows, h) and (rstd[M:] == 0).all()
    torch.testing.assert_close(fy.rows, y, **close)
    torch.testing.assert_close(rstd[:M], rs, rtol=2.0 ** -17, atol=0)

    fdy, fdh, fdx = Frame(M, n, t, leads[0], gap, dy), Frame(M, n, r, leads[1], gap, dh), Frame(M, n, t, leads[2], gap)
    fdr = Frame(M, n, r, leads[4], gap) if t != r else None
    dw = torch.full((n + 8,), 7.0, device=DEV)
    need = lib.b200norm_add_rms_bwd_workspace_bytes(M, n, CODE[t], CODE[r])
    ws = torch.full((need + 256,), 0x33, dtype=torch.uint8, device=DEV)
    _lib.check(lib.b200norm_add_rms_bwd(*fh.at, *fdy.at, *fdh.at, w.data_ptr(), rstd.data_ptr(), *fdx.at,
                                        *(fdr.at if fdr else (None, n)), dw.data_ptr(), ws.data_ptr(), need, M, n, CODE[t], CODE[r],
                                        _lib.F32, s))
    dx, dr, dwant = A._add_rmsnorm_bwd(h, dy, dh, w, rs)
    assert (dw[n:] == 7).all() and (ws[need:] == 0x33).all()
    # entries are sums that may cancel: relative to the largest
    for got, want, dtype in ((fdx.rows, dx, t), (fdr.rows if fdr else fdx.rows, dr, r), (dw[:n], dwant, F32)):
        assert (got.float() - want.float()).abs().max() <= (torch.finfo(dtype).eps + 2.0 ** -14) * want.float().abs().max()

    for group in (0, 32, 128):
        groups = -(-n // group) if group else 1
        scale = torch.full((M * groups + 8,), 3.0, device=DEV)
        _lib.check(lib.b200norm_rms_fp8(*fx.at, *fr.at, w.data_ptr(), *fq.at, scale.data_ptr(), *fh.at, M, n, 1e-6, group, 0,
                                        CODE[t], CODE[r], _lib.F32, s))
        q, sc, _ = b200norm.rmsnorm_fp8(x, w, 1e-6, residual=res, group=group)
        torch.testing.assert_close(scale[:M * groups].view(M, groups), sc, rtol=2.0 ** -16, atol=0)
        assert (scale[M * groups:] == 3).all() and torch.equal(fh.rows, h)
        # a step of e4m3 where the two norms lie on either side of a border
        assert ((fq.rows.view(torch.float8_e4m3fn).float() - q.float()).abs() <= q.float().abs() * 0.125 + 2.0 ** -9).all()
    for f in (fx, fr, fy, fh, fq, fdy, fdh, fdx, fdr):
        if f is not None:
            f.check()


def test_choices_stay_inside_their_outputs():
    x = randn(50, 40, dtype=BF16)
    k, lib, s = 5, _lib.load(), torch.cuda.current_stream().cuda_stream
    gates, experts = torch.full((60, k), 9.0, device=DEV), torch.full((60, k), 9, dtype=torch.int32, device=DEV)
    counts, lse = torch.full((50,), 9, dtype=torch.int32, device=DEV), torch.full((60,), 9.0, device=DEV)
    loss, dl = torch.full((4,), 9.0, device=DEV), torch.full((60, 40), 9.0, dtype=BF16, device=DEV)
    _lib.check(lib.b200norm_route_fwd(x.data_ptr(), 40, None, gates.data_ptr(), experts.data_ptr(), lse.data_ptr(), counts.data_ptr(),
                                      loss.data_ptr(), None, 0, 50, 40, k, 1, _lib.BF16, s))
    _lib.check(lib.b200norm_route_bwd(x.data_ptr(), 40, gates.data_ptr(), experts.data_ptr(), lse.data_ptr(), counts.data_ptr(), None,
                                      k, loss.data_ptr(), dl.data_ptr(), 50, 40, k, 1, _lib.BF16, s))
    want = R._route_fwd(x, k)
    assert torch.equal(gates[:50], want[0]) and torch.equal(experts[:50], want[1]) and torch.equal(counts[:41], want[2])
    assert torch.equal(loss[0], want[3]) and torch.equal(lse[:50], want[4])
    for rest in (gates[50:], experts[50:], counts[41:], loss[1:], lse[50:], dl[50:]):
        assert (rest == 9).all()
    u, tokens = rand(50), torch.full((60,), 9, dtype=torch.int64, device=DEV)
    _lib.check(lib.b200norm_sample(x.data_ptr(), 40, u.data_ptr(), None, 1.0, None, 0, None, 1.0, None, 0.0, tokens.data_ptr(), 50,
                                   40, _lib.BF16, s))
    assert torch.equal(tokens[:50], b200norm.sample(x, u)) and (tokens[50:] == 9).all()


def test_a_workspace_that_is_too_small_is_refused():
    lib, s = _lib.load(), torch.cuda.current_stream().cuda_stream
    x = randn(3000, 128)
    o = R._route_fwd(x, 4)
    need = lib.b200norm_route_workspace_bytes(3000, 128, 4, _lib.F32)
    assert need > 1
    ws = torch.empty(need, dtype=torch.uint8, device=DEV)
    for ptr, size in ((ws.data_ptr(), need - 1), (None, need)):
        assert lib.b200norm_route_fwd(x.data_ptr(), 128, None, o[0].data_ptr(), o[1].data_ptr(), None, o[2].data_ptr(),
                                      o[3].data_ptr(), ptr, size, 3000, 128, 4, 1, _lib.F32, s) == _lib.ERR_ARG
        assert b"workspace" in lib.b200norm_last_error()
    y, h, rstd = A._add_rmsnorm_fwd(x, x, None, 1e-6)
    dw = torch.empty(128, device=DEV)
    for ptr, size in ((ws.data_ptr(), 8), (None, 1 << 30)):
        assert lib.b200norm_add_rms_bwd(h.data_ptr(), 128, x.data_ptr(), 128, None, 128, dw.data_ptr(), rstd.data_ptr(), y.data_ptr(),
                                        128, None, 128, dw.data_ptr(), ptr, size, 3000, 128, _lib.F32, _lib.F32, _lib.F32,
                                        s) == _lib.ERR_ARG
        assert b"workspace" in lib.b200norm_last_error()


def test_rows_beyond_32_bit_offsets():
    n, far = 64, 2 ** 30 + 24  # the last of three rows starts beyond 2^31 elements
    buf = torch.empty(2 * far + n, dtype=BF16, device=DEV)
    x = buf.as_strided((3, n), (far, 1))
    x.copy_(randn(3, n, seed=1, dtype=BF16))
    c, r = x.contiguous(), randn(3, n, seed=2, dtype=BF16)
    y, h, rstd = A._add_rmsnorm_fwd(x, r, None, 1e-6)
    assert all(torch.equal(a, b) for a, b in zip((y, h, rstd), A._add_rmsnorm_fwd(c, r, None, 1e-6)))
    for a, b in ((A._add_rmsnorm_bwd(h, x, r, None, rstd), A._add_rmsnorm_bwd(h, c, r, None, rstd)),
                 (A._add_rmsnorm_bwd(x, y, x, None, rstd), A._add_rmsnorm_bwd(c, y, c, None, rstd))):
        assert torch.equal(a[0], b[0])
    for group in (0, 32):
        a, b = b200norm.rmsnorm_fp8(x, None, 1e-6, group=group), b200norm.rmsnorm_fp8(c, None, 1e-6, group=group)
        assert torch.equal(a[0].view(torch.uint8), b[0].view(torch.uint8)) and torch.equal(a[1], b[1])
    a, b = R._route_fwd(x, 4), R._route_fwd(c, 4)
    assert all(torch.equal(u, v) for u, v in zip(a, b))
    assert torch.equal(R._route_bwd(x, *a[:3], a[4], a[0], a[3]), R._route_bwd(c, *b[:3], b[4], b[0], b[3]))
    u = rand(3)
    assert torch.equal(b200norm.sample(x, u, top_p=0.9), b200norm.sample(c, u, top_p=0.9))


def test_a_single_row_without_a_leading_dimension():
    x, r = randn(1, 512, dtype=BF16), randn(1, 512, seed=1, dtype=BF16)
    for a, b in zip(b200norm.add_rmsnorm.apply(x[0], r[0], None, 1e-6), b200norm.add_rmsnorm.apply(x, r, None, 1e-6)):
        assert a.shape == (512,) and torch.equal(a, b[0])
    for a, b in zip(b200norm.rmsnorm_fp8(x[0], group=64), b200norm.rmsnorm_fp8(x, group=64)):
        assert torch.equal(a.view(torch.uint8), b[0].view(torch.uint8))
    a, b = b200norm.route.apply(x[0, :64], 4), b200norm.route.apply(x[:, :64], 4)
    assert a[0].shape == a[1].shape == (4,) and torch.equal(a[0], b[0][0]) and torch.equal(a[1], b[1][0]) and torch.equal(a[2], b[2])
    u = rand(1)
    token = b200norm.sample(x[0], u[0])
    assert token.shape == () and int(token) == int(b200norm.sample(x, u)[0])


def test_settings_of_other_integer_types():
    import numpy as np
    x, u = randn(6, 1000, scale=3.0), rand(6)
    want = b200norm.sample(x, u, top_k=7, temperature=0.5)
    assert torch.equal(b200norm.sample(x, u, top_k=np.int64(7), temperature=np.float64(0.5)), want)
    k = torch.full((6,), 7, dtype=torch.int64, device=DEV)
    assert torch.equal(b200norm.sample(x, u, top_k=k, temperature=0.5), want)
    assert torch.equal(b200norm.sample(x, u, top_k=k + 2 ** 32), b200norm.sample(x, u))  # more than there are: all
    with pytest.raises(TypeError):
        b200norm.sample(x, u, top_k=7.5)
    a, b = b200norm.route.apply(x[:, :64], np.int32(4)), b200norm.route.apply(x[:, :64], 4)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    for p, q in zip(b200norm.rmsnorm_fp8(x, group=np.int64(32)), b200norm.rmsnorm_fp8(x, group=32)):
        assert torch.equal(p.view(torch.uint8), q.view(torch.uint8))


FIRST_CALL = """
import sys, torch
sys.path.insert(0, %r)
import b200norm
from b200norm import addnorm as A, routing as R
x = torch.randn(3000, 4096, device="cuda:0")
u = torch.rand(3000, device="cuda:0")
calls = {"fp8": lambda: b200norm.rmsnorm_fp8(x, group=128), "add": lambda: A._add_rmsnorm_bwd(x, x, None, u.new_ones(4096), u),
         "route": lambda: R._route_fwd(x[:, :64], 4), "sample": lambda: (b200norm.sample(x, u, top_p=0.9),)}
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = calls[sys.argv[1]]()
graph.replay()
for a, b in zip(got, calls[sys.argv[1]]()):
    assert torch.equal(a.reshape(-1).view(torch.uint8), b.reshape(-1).view(torch.uint8))
print("same")
"""


@pytest.mark.parametrize("name", ["fp8", "add", "route", "sample"])
def test_the_first_call_of_a_process_may_be_a_captured_one(name):
    root = str(Path(b200norm.__file__).resolve().parent.parent)
    done = subprocess.run([sys.executable, "-c", FIRST_CALL % root, name], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "same" in done.stdout, done.stderr[-2000:]


def test_tables_of_sizes_stay_bounded():
    # a server meets a new number of tokens at almost every step
    x, w = randn(6000, 16), torch.ones(16, device=DEV)
    rstd = torch.ones(6000, device=DEV)
    for T in range(1, 6000):
        R._route_fwd(x[:T], 2, need_lse=False)
        A._add_rmsnorm_bwd(x[:T], x[:T], None, w, rstd[:T])
    for table in (R._workspace_bytes, A._workspace_bytes):
        assert 0 < table.cache_info().currsize < 5000
