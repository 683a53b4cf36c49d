"""Cases for the operators that stand beside RMSNorm and Softmax in a language model: the residual
addition fused into RMSNorm (forward, and forward + backward), RMSNorm with an 8-bit output and scales,
the choice of experts from router logits with its balance loss, and the choice of a token from logits.

`run` computes them in elementary torch operations, or (`own`) through the framework's entry points."""
import functools
import math
import os
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6
E4M3_MAX = 448.0
AMAX_FLOOR = 2.0 ** -64  # a group of zeros still gets a finite scale


@functools.lru_cache(None)
def _framework():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "triton-hub_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import b200norm
    return b200norm


# ---------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------
def listed():
    return [
        # a decode step of eight sequences: the block's residual addition and norm, launch-bound
        {"name": "add_norm_decode_bf16", "op": "add_norm", "rows": 8, "dim": 4096, "dtype": "bf16", "res": "bf16", "w": "bf16",
         "train": False},
        # a training step's residual + norm, forward and backward, at the benchmark's row length
        {"name": "add_norm_train_bf16", "op": "add_norm", "rows": 16384, "dim": 4096, "dtype": "bf16", "res": "bf16",
         "w": "bf16", "train": True},
        # training with the residual stream and the parameters held in fp32
        {"name": "add_norm_train_res32", "op": "add_norm", "rows": 6001, "dim": 5120, "dtype": "bf16", "res": "f32", "w": "f32",
         "train": True},
        # rows of an odd length: no 16-byte packet is aligned from row to row
        {"name": "add_norm_train_odd_f16", "op": "add_norm", "rows": 3001, "dim": 1001, "dtype": "f16", "res": "f16", "w": "f32",
         "train": True},
        # a decode step's norm in front of 8-bit products, scales per 128 columns
        {"name": "norm_fp8_decode", "op": "norm_fp8", "rows": 16, "dim": 4096, "dtype": "bf16", "res": "bf16", "w": "bf16",
         "group": 128, "e8m0": False},
        # prefill of long prompts, one scale a row
        {"name": "norm_fp8_prefill_rows", "op": "norm_fp8", "rows": 16384, "dim": 5120, "dtype": "bf16", "res": "bf16",
         "w": "bf16", "group": 0, "e8m0": False},
        # power-of-two scales per 32 columns (the tensor cores' block-scaled form), a ragged last group, no residual
        {"name": "norm_fp8_mx_ragged", "op": "norm_fp8", "rows": 8191, "dim": 4104, "dtype": "f16", "res": "", "w": "f32",
         "group": 32, "e8m0": True},
        # one sequence's next token, the usual truncations, launch-bound
        {"name": "sample_one_f32", "op": "sample", "rows": 1, "vocab": 32768, "dtype": "f32", "per_row": False,
         "temperature": 0.8, "top_k": 50, "top_p": 0.9, "min_p": 0.0, "banned": False},
        # a serving batch whose requests each bring their own settings
        {"name": "sample_batch_bf16", "op": "sample", "rows": 64, "vocab": 131072, "dtype": "bf16", "per_row": True,
         "temperature": 0.7, "top_k": 0, "top_p": 0.95, "min_p": 0.02, "banned": True},
        # rollouts from the whole distribution, an odd vocabulary
        {"name": "sample_full_odd_f32", "op": "sample", "rows": 128, "vocab": 100003, "dtype": "f32", "per_row": False,
         "temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0, "banned": False},
        # a decode step's routing: few tokens, few experts
        {"name": "route_decode_bf16", "op": "route", "tokens": 64, "experts": 64, "dtype": "bf16", "k": 6, "normalize": True,
         "mask": False, "train": False},
        # a training step's routing with its balance loss, forward and backward, padded positions masked
        {"name": "route_train_f32", "op": "route", "tokens": 65536, "experts": 128, "dtype": "f32", "k": 8, "normalize": True,
         "mask": True, "train": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["add_norm", "norm_fp8", "sample", "route"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op in ("add_norm", "norm_fp8"):
        dim = _log(rng, 64, 16384)
        step = rng.choice([1, 2, 8, 64])
        dim = max(step, dim // step * step)
        size = 4 if dtype == "f32" else 2
        rows = _log(rng, 1, max(2, min(32768, (128 << 20) // (dim * size))))
        res = rng.choice([dtype, dtype, "f32"])
        if op == "add_norm":
            if res != dtype:
                rows = max(1, rows // 2)
            return {"op": op, "rows": rows, "dim": dim, "dtype": dtype, "res": res, "w": rng.choice([dtype, "f32"]),
                    "train": rng.random() < 0.7}
        e8m0 = rng.random() < 0.4
        return {"op": op, "rows": rows, "dim": dim, "dtype": dtype, "res": rng.choice(["", dtype]),
                "w": rng.choice([dtype, "f32"]), "group": rng.choice([32, 64, 128]) if e8m0 else rng.choice([0, 32, 64, 128]),
                "e8m0": e8m0}
    if op == "sample":
        vocab = _log(rng, 1000, 262144)
        rows = _log(rng, 1, max(2, min(256, 12_000_000 // vocab)))
        return {"op": op, "rows": rows, "vocab": vocab, "dtype": dtype, "per_row": rng.random() < 0.5,
                "temperature": round(rng.uniform(0.3, 1.5), 3), "top_k": rng.choice([0, 0, _log(rng, 1, 1000)]),
                "top_p": rng.choice([1.0, round(rng.uniform(0.3, 0.99), 3)]),
                "min_p": rng.choice([0.0, 0.0, round(rng.uniform(0.005, 0.2), 4)]), "banned": rng.random() < 0.3}
    experts = rng.choice([_log(rng, 4, 512), 8, 64, 128, 256])
    tokens = _log(rng, 1, min(65536, 8_000_000 // experts))
    return {"op": op, "tokens": tokens, "experts": experts, "dtype": dtype, "k": rng.randint(1, min(8, experts)),
            "normalize": rng.random() < 0.6, "mask": rng.random() < 0.5, "train": rng.random() < 0.7}


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def prepare(case, seed):
    dev = torch.device("cuda" if torch.cuda.is_available() else "cpu")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)

    def normal(*shape, dtype="f32", scale=1.0, shift=0.0):
        return (torch.randn(*shape, generator=g, device=dev) * scale + shift).to(DTYPES[dtype])

    s = {"case": case}
    if case["op"] in ("add_norm", "norm_fp8"):
        M, N, t = case["rows"], case["dim"], case["dtype"]
        s["x"] = normal(M, N, dtype=t)
        s["res"] = normal(M, N, dtype=case["res"], scale=2.0) if case["res"] else None
        s["w"] = normal(N, dtype=case["w"], scale=0.1, shift=1.0)
        if case["op"] == "add_norm" and case["train"]:
            s["dy"], s["dh"] = normal(M, N, dtype=t), normal(M, N, dtype=case["res"])
            s["leaves"] = [s[k].requires_grad_(True) for k in ("x", "res", "w")]
    elif case["op"] == "sample":
        M, V = case["rows"], case["vocab"]
        logits = normal(M, V, scale=2.5)
        # a few likely tokens above the bulk, as a trained model's logits have them
        at = torch.randint(V, (M, 12), generator=g, device=dev)
        logits.scatter_add_(1, at, 5.0 + 5.0 * torch.rand(M, 12, generator=g, device=dev))
        if case["banned"]:
            logits.masked_fill_(torch.rand(M, V, generator=g, device=dev) < 0.05, -math.inf)
        s["logits"] = logits.to(DTYPES[case["dtype"]])
        s["u"] = torch.rand(M, generator=g, device=dev)
        for name in ("temperature", "top_k", "top_p", "min_p"):
            s[name] = case[name]
        if case["per_row"]:  # every request's own settings, spread around the case's
            spread = torch.rand(3, M, generator=g, device=dev)
            s["temperature"] = case["temperature"] * (0.75 + 0.5 * spread[0])
            s["top_p"] = case["top_p"] - 0.2 * spread[1] if case["top_p"] < 1 else torch.ones(M, device=dev)
            s["min_p"] = case["min_p"] * spread[2]
            s["top_k"] = torch.full((M,), case["top_k"], dtype=torch.int32, device=dev)
    else:
        T, E = case["tokens"], case["experts"]
        bias = normal(E, scale=0.5)  # some experts are liked more than others
        s["logits"] = (normal(T, E, scale=1.5) + bias).to(DTYPES[case["dtype"]])
        s["mask"] = torch.rand(T, generator=g, device=dev) < 0.9 if case["mask"] else None
        if case["train"]:
            s["logits"].requires_grad_(True)
            s["dgates"] = normal(T, case["k"])
            s["dloss"] = torch.full((), 0.01, device=dev)
    return s


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def run(s):
    op = s["case"]["op"]
    if own:
        return {"add_norm": _own_add_norm, "norm_fp8": _own_norm_fp8, "sample": _own_sample, "route": _own_route}[op](s)
    with torch.no_grad():
        return {"add_norm": _add_norm, "norm_fp8": _norm_fp8, "sample": _sample, "route": _route}[op](s)


def _own_add_norm(s):
    b = _framework()
    if not s["case"]["train"]:
        with torch.no_grad():
            y, h = b.add_rmsnorm.apply(s["x"], s["res"], s["w"], EPS)
        return {"y": y, "h": h}
    y, h = b.add_rmsnorm.apply(s["x"], s["res"], s["w"], EPS)
    dx, dr, dw = torch.autograd.grad((y, h), s["leaves"], (s["dy"], s["dh"]))
    return {"y": y, "h": h, "dx": dx, "dres": dr, "dw": dw}


def _add_norm(s):
    x, r, w = s["x"].float(), s["res"].float(), s["w"].float()
    h = (x + r).to(s["res"].dtype)
    hf = h.float()
    rstd = torch.rsqrt((hf * hf).mean(-1, keepdim=True) + EPS)
    xhat = hf * rstd
    out = {"y": (xhat * w).to(s["x"].dtype), "h": h}
    if s["case"]["train"]:
        dy = s["dy"].float()
        g = w * dy
        d = (g - xhat * (xhat * g).mean(-1, keepdim=True)) * rstd + s["dh"].float()
        out["dx"], out["dres"] = d.to(s["x"].dtype), d.to(s["res"].dtype)
        out["dw"] = (dy * xhat).sum(0).to(s["w"].dtype)
    return out


def _own_norm_fp8(s):
    c = s["case"]
    scales = torch.float8_e8m0fnu if c["e8m0"] else torch.float32
    got = _framework().rmsnorm_fp8(s["x"], s["w"], EPS, residual=s["res"], group=c["group"], scale_dtype=scales)
    return dict(zip(("q", "scale", "h"), got))


def _norm_fp8(s):
    c = s["case"]
    M, N, group = c["rows"], c["dim"], c["group"] or c["dim"]
    out = {}
    h = s["x"].float()
    if s["res"] is not None:
        out["h"] = (h + s["res"].float()).to(s["res"].dtype)
        h = out["h"].float()
    y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS) * s["w"].float()
    G = -(-N // group)
    y = torch.nn.functional.pad(y, (0, G * group - N)).reshape(M, G, group)
    scale = y.abs().amax(-1, keepdim=True).clamp(min=AMAX_FLOOR) / E4M3_MAX
    if c["e8m0"]:  # the next power of two: the exponent, one more where the fraction is not zero
        scale = ((scale.view(torch.int32) + 0x7FFFFF) & 0x7F800000).view(torch.float32)
    q = (y / scale).clamp(-E4M3_MAX, E4M3_MAX).reshape(M, G * group)[:, :N]
    out["q"] = q.to(torch.float8_e4m3fn)
    scale = scale.reshape(M, G)
    out["scale"] = scale.to(torch.float8_e8m0fnu) if c["e8m0"] else scale
    return out


def _own_sample(s):
    return _framework().sample(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                               min_p=s["min_p"])


def _sample(s):
    x = s["logits"].float()
    V = x.shape[1]

    def column(v):  # a setting as (rows, 1) or (1, 1), rounded to 32 bits
        return torch.as_tensor(v, dtype=torch.float32, device=x.device).double().reshape(-1, 1)

    top = x.amax(-1, keepdim=True)
    # sums over a vocabulary and values next to a border: 64 bits
    weight = torch.exp((x.double() - top.double()) / column(s["temperature"]))
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices
    ranked = weight.gather(1, order)
    rank = torch.arange(V, device=x.device)
    k = torch.as_tensor(s["top_k"], device=x.device).reshape(-1, 1)
    keep = (k <= 0) | (rank < k)
    in_k = ranked * keep
    sums = in_k.cumsum(-1)
    keep = keep & ((sums - in_k < column(s["top_p"]) * sums[:, -1:]) | (rank == 0))
    keep = keep & (ranked >= column(s["min_p"]))
    kept = torch.zeros_like(weight).scatter_(1, order, ranked * keep)
    sums = kept.cumsum(-1)
    # the first token whose sum passes u * total
    return (sums > s["u"].double().reshape(-1, 1) * sums[:, -1:]).to(torch.int8).argmax(-1)


def _own_route(s):
    b, c = _framework(), s["case"]
    if not c["train"]:
        with torch.no_grad():
            gates, experts, counts, loss = b.route.apply(s["logits"], c["k"], c["normalize"], s["mask"])
        return {"gates": gates, "experts": experts, "counts": counts, "loss": loss}
    gates, experts, counts, loss = b.route.apply(s["logits"], c["k"], c["normalize"], s["mask"])
    dlogits, = torch.autograd.grad((gates, loss), s["logits"], (s["dgates"], s["dloss"]))
    return {"gates": gates, "experts": experts, "counts": counts, "loss": loss, "dlogits": dlogits}


def _route(s):
    c = s["case"]
    T, E, k = c["tokens"], c["experts"], c["k"]
    x = s["logits"].float()
    e = torch.exp(x - x.amax(-1, keepdim=True))
    p = e / e.sum(-1, keepdim=True)
    experts = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :k]
    gates = p.gather(1, experts)
    live = torch.ones(T, 1, device=x.device) if s["mask"] is None else s["mask"].float().reshape(T, 1)
    total = gates.sum(-1, keepdim=True)
    if c["normalize"]:
        gates = gates / total
    hot = torch.zeros(T, E, device=x.device).scatter_(1, experts, live.expand(T, k))
    counts = hot.sum(0)
    n = live.sum().clamp(min=1)
    share, mean = counts / (n * k), (p * live).sum(0) / n
    out = {"gates": gates * live, "experts": torch.where(live > 0, experts, -1).int(), "counts": counts.int(),
           "loss": E * (share * mean).sum()}
    if c["train"]:
        to_p = s["dloss"] * E / n * share
        d = p * (to_p - (p * to_p).sum(-1, keepdim=True))
        dg = s["dgates"]
        if c["normalize"]:
            part = gates * (dg - (gates * dg).sum(-1, keepdim=True))
        else:
            part = gates * dg
            d = d - p * part.sum(-1, keepdim=True)
        d = d.scatter_add_(1, experts, part)
        out["dlogits"] = (d * live).to(s["logits"].dtype)
    return out


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------
def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2, "": 0}
    if case["op"] in ("add_norm", "norm_fp8"):
        n, t, r, w = case["rows"] * case["dim"], size[case["dtype"]], size[case["res"]], size[case["w"]]
        params = case["dim"] * w
        if case["op"] == "norm_fp8":
            groups = -(-case["dim"] // case["group"]) if case["group"] else 1
            return {"bytes": n * (t + 2 * r + 1) + case["rows"] * groups * (1 if case["e8m0"] else 4) + params, "flops": 8 * n}
        nbytes = n * (2 * t + 2 * r) + params  # x, residual -> y, h
        if case["train"]:  # h, dy, dh -> dx, dres (one tensor where their types are one), dweight
            nbytes += n * (2 * r + t + (t if case["res"] != case["dtype"] else 0)) + 2 * params
        return {"bytes": nbytes, "flops": n * (6 + (14 if case["train"] else 0))}
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size[case["dtype"]] + case["rows"] * 12, "flops": 20 * n}
    n, pairs = case["tokens"] * case["experts"], case["tokens"] * case["k"]
    nbytes = n * size[case["dtype"]] + pairs * 8 + case["tokens"] * (1 if case["mask"] else 0) + case["experts"] * 4
    if case["train"]:
        nbytes += 2 * n * size[case["dtype"]] + pairs * 8
    return {"bytes": nbytes, "flops": n * (8 + (8 if case["train"] else 0))}


# ---------------------------------------------------------------------------------------------
# from the definitions, in 64 bits
# ---------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "sample":
        return None
    return {"add_norm": _exact_add_norm, "norm_fp8": _exact_norm_fp8, "route": _exact_route}[case["op"]](s)


def _rms64(h, w):
    return h / torch.sqrt(h.square().mean(-1, keepdim=True) + EPS) * w


def _exact_add_norm(s):
    h = (s["x"].detach().double() + s["res"].detach().double()).to(s["res"].dtype)
    h64, w = h.double().requires_grad_(True), s["w"].detach().double().requires_grad_(True)
    y = _rms64(h64, w)
    out = {"y": y.detach(), "h": h64.detach()}
    if s["case"]["train"]:
        d, dw = torch.autograd.grad((y * s["dy"].double()).sum() + (h64 * s["dh"].double()).sum(), (h64, w))
        out.update(dx=d, dres=d, dw=dw)
    return out


def _exact_norm_fp8(s):
    c = s["case"]
    h = s["x"].double()
    out = {}
    if s["res"] is not None:
        out["h"] = (h + s["res"].double()).to(s["res"].dtype).double()
        h = out["h"]
    y = _rms64(h, s["w"].double())
    blocks = y.split(c["group"] or c["dim"], dim=-1)
    scales = [b.abs().amax(-1, keepdim=True).clamp(min=AMAX_FLOOR) / E4M3_MAX for b in blocks]
    if c["e8m0"]:
        scales = [torch.exp2(torch.ceil(torch.log2(v.float().double()))) for v in scales]
    out["q"] = torch.cat([b / v for b, v in zip(blocks, scales)], -1)
    out["scale"] = torch.cat(scales, -1)
    return out


def _exact_route(s):
    c = s["case"]
    x = s["logits"].detach().double().requires_grad_(True)
    live = torch.ones(c["tokens"], dtype=torch.bool, device=x.device) if s["mask"] is None else s["mask"]
    p = torch.softmax(x, -1)
    experts = torch.argsort(x.detach(), dim=-1, descending=True, stable=True)[:, :c["k"]]
    gates = torch.gather(torch.log_softmax(x, -1), 1, experts)
    gates = torch.softmax(gates, -1) if c["normalize"] else gates.exp()
    counts = torch.bincount(experts[live].reshape(-1), minlength=c["experts"]).double()
    n = max(1, int(live.sum()))
    loss = c["experts"] * torch.dot(counts / (n * c["k"]), p[live].sum(0) / n)
    gates = gates * live.double()[:, None]
    out = {"gates": gates.detach(), "experts": None, "counts": None, "loss": loss.detach()}
    if c["train"]:
        out["dlogits"], = torch.autograd.grad((gates * s["dgates"].double()).sum() + loss * s["dloss"].double(), x)
    return out
