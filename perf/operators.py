"""Workloads of the text-decoder operators that run beside the detector: attention with capped scores, distance bias
and document / prefix masks; the per-head norm and rotation of queries and keys that feeds it; token sampling.

`listed()` gives the cases, `draw(rng)` one more of the same ranges, `prepare` the inputs, `run` one pass (in plain
torch operations, or through the library where `own` is true), `exact` the result in 64 bits, `work` the bytes and
operations of a pass.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
GOLDEN = 0.6180339887498949


def _ops():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "yolo-baremetal_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import yb_ops

    return yb_ops


# ------------------------------------------------------------------ the cases

def _attention(name, **kw):
    case = {"name": name, "op": "attention", "batch": 1, "rows": 1, "keys": 1, "heads": 1, "kv_heads": 1, "dim": 64,
            "type": "bf16", "cap": 0.0, "slopes": False, "causal": True, "ragged": False, "prefix": 0, "docs": 0}
    case.update(kw)
    return case


def _rotate(name, **kw):
    case = {"name": name, "op": "rotate", "batch": 1, "rows": 1, "cache": 64, "heads": 1, "kv_heads": 1, "dim": 64,
            "rotary": 64, "type": "bf16", "interleaved": False, "far": 0, "ragged": False}
    case.update(kw)
    return case


def _sample(name, **kw):
    case = {"name": name, "op": "sample", "batch": 1, "vocab": 1000, "type": "f32", "temperature": 1.0, "top_k": 0,
            "top_p": 1.0, "min_p": 0.0, "mixed": False}
    case.update(kw)
    return case


def listed():
    return [
        # One token of one short conversation: what counts is the latency of the call.
        _attention("attention-step-short", rows=1, keys=401, heads=8, kv_heads=2, dim=64, type="f16"),
        # One token each of a batch of conversations of very different lengths over a long cache, capped scores.
        _attention("attention-step-ragged", batch=24, rows=1, keys=16384, heads=32, kv_heads=8, dim=128, cap=30.0,
                   ragged=True),
        # Two whole prompts, capped scores, four heads to a key head.
        _attention("attention-prompt-capped", batch=2, rows=4096, keys=4096, heads=16, kv_heads=4, dim=128, cap=50.0),
        # Documents packed into one long row, each seeing only itself, with a linear distance bias.
        _attention("attention-documents", rows=8191, keys=8191, heads=12, kv_heads=12, dim=80, type="f16", slopes=True,
                   docs=9),
        # The rest of a few prompts behind a cached part, whose first tokens (an image's, say) see one another.
        _attention("attention-prefix-chunk", batch=3, rows=700, keys=1337, heads=14, kv_heads=2, dim=64, ragged=True,
                   prefix=256),
        # One token each of a batch, queries and keys from one packed projection, written into the cache.
        _rotate("rotate-step", batch=16, rows=1, cache=1024, heads=32, kv_heads=8, dim=128, rotary=128, ragged=True),
        # A long prompt.
        _rotate("rotate-prompt", rows=8191, cache=8192, heads=32, kv_heads=8, dim=128, rotary=128),
        # Ragged prompts in 32 bits, neighbouring pairs rotated, far positions, part of the head rotated.
        _rotate("rotate-prompt-far", batch=3, rows=1001, cache=1024, heads=8, kv_heads=8, dim=96, rotary=64,
                type="f32", interleaved=True, far=1000000, ragged=True),
        # One conversation's next token with the usual filters.
        _sample("sample-one", vocab=32000, temperature=0.8, top_k=50, top_p=0.95),
        # A batch with each request's own settings.
        _sample("sample-batch-mixed", batch=64, vocab=128000, type="bf16", temperature=0.9, top_k=200, top_p=0.9,
                min_p=0.02, mixed=True),
        # A wide batch without filters, as a sampler for training data runs.
        _sample("sample-wide", batch=256, vocab=131072),
        # An odd vocabulary, nucleus only.
        _sample("sample-nucleus-odd", batch=17, vocab=50001, type="f16", temperature=1.2, top_p=0.8),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "rotate", "sample"])
    if op == "attention":
        while True:
            kind = rng.choice(["step", "prompt", "documents", "prefix"])
            kv = rng.choice([1, 2, 3, 4, 8])
            heads = kv * rng.choice([1, 2, 3, 4, 7, 8])
            case = {"op": op, "batch": _log(rng, 1, 32) if kind == "step" else _log(rng, 1, 6),
                    "rows": rng.choice([1, 1, 2, 5]) if kind == "step" else _log(rng, 16, 8191),
                    "heads": heads, "kv_heads": kv, "dim": rng.choice([32, 40, 64, 64, 80, 96, 128, 128]),
                    "type": rng.choice(["f16", "bf16"]), "cap": rng.choice([0.0, 20.0, 30.0, 50.0]),
                    "slopes": rng.random() < 0.3, "causal": kind != "documents" or rng.random() < 0.5,
                    "ragged": rng.random() < 0.6, "prefix": 0, "docs": 0}
            if kind == "step":
                case["keys"] = max(case["rows"], _log(rng, 1, 16384))
            elif kind == "documents":
                case.update(batch=1, keys=case["rows"], docs=rng.randint(2, 12), ragged=False)
            else:
                case["keys"] = case["rows"] + (_log(rng, 1, 2000) if rng.random() < 0.5 else 0)
                if kind == "prefix":
                    case["prefix"] = rng.randint(1, max(1, case["keys"] // 2))
            pairs = case["batch"] * heads * case["rows"] * case["keys"]
            cache = case["batch"] * case["keys"] * kv * case["dim"]
            if pairs <= 4.0e8 and cache <= 3.0e8:
                return case
    if op == "rotate":
        while True:
            dim = rng.choice([32, 64, 64, 96, 128, 128])
            kv = rng.choice([1, 2, 4, 8])
            batch, rows = _log(rng, 1, 32), 1 if rng.random() < 0.3 else _log(rng, 1, 8191)
            case = {"op": op, "batch": batch, "rows": rows, "cache": rows + rng.randint(0, 200),
                    "heads": kv * rng.choice([1, 2, 4, 5]), "kv_heads": kv, "dim": dim,
                    "rotary": rng.choice([dim, dim, dim // 2]), "type": rng.choice(["f16", "bf16", "f32"]),
                    "interleaved": rng.random() < 0.4, "far": rng.choice([0, 0, 5000, 1000000]),
                    "ragged": rng.random() < 0.5}
            if batch * case["cache"] * (case["heads"] + 2 * kv) * dim * SIZE[case["type"]] <= 8.0e7:
                return case
    while True:
        case = {"op": op, "batch": _log(rng, 1, 256), "vocab": _log(rng, 500, 200000),
                "type": rng.choice(["f16", "bf16", "f32"]), "temperature": round(rng.uniform(0.5, 1.5), 2),
                "top_k": rng.choice([0, 0, 1, 40, 1000]), "top_p": rng.choice([1.0, 0.95, 0.9, 0.5]),
                "min_p": rng.choice([0.0, 0.0, 0.05]), "mixed": rng.random() < 0.5}
        if case["batch"] * case["vocab"] <= 2.5e7:
            return case


# ------------------------------------------------- lengths that follow from a case

def _lengths(n, most, least=1):
    """n lengths in [least, most], spread evenly; the first is the longest."""
    return np.array([most - int((most - least + 1) * ((i * GOLDEN) % 1.0)) for i in range(n)], dtype=np.int32)


def _attention_lengths(case):
    b, rows, keys = case["batch"], case["rows"], case["keys"]
    if not case["ragged"]:
        return np.full(b, rows, np.int32), np.full(b, keys, np.int32)
    k_len = _lengths(b, keys)
    q_len = np.minimum(_lengths(b, rows), k_len).astype(np.int32)
    return q_len, k_len


def _documents(case):
    """Begin and end of each row's document, [rows, 2]."""
    n, rows = case["docs"], case["rows"]
    cuts = sorted({int(rows * ((i * GOLDEN) % 1.0)) for i in range(1, n)} | {0, rows})
    out = np.zeros((rows, 2), np.int32)
    for a, e in zip(cuts[:-1], cuts[1:]):
        out[a:e] = (a, e)
    return out


def _prefixes(case):
    return _lengths(case["batch"], case["prefix"])


def _visible(case):
    """(first key, end of keys) of every row of every sequence: two lists of arrays."""
    q_len, k_len = _attention_lengths(case)
    lo, hi = [], []
    for b in range(case["batch"]):
        n, m = int(q_len[b]), int(k_len[b])
        begin, end = np.zeros(n, np.int64), np.full(n, m, np.int64)
        if case["docs"]:
            d = _documents(case)[:n]
            begin, end = d[:, 0].astype(np.int64), np.minimum(d[:, 1], m).astype(np.int64)
        if case["causal"]:
            last = m - n + np.arange(n) + 1
            if case["prefix"]:
                last = np.maximum(last, int(_prefixes(case)[b]))
            end = np.minimum(end, last)
        lo.append(begin)
        hi.append(np.maximum(begin, end))
    return lo, hi


def work(case):
    size = SIZE[case["type"]]
    if case["op"] == "attention":
        lo, hi = _visible(case)
        pairs = sum(int((h - l).sum()) for l, h in zip(lo, hi))
        rows = sum(len(l) for l in lo)
        keys = 0
        for l, h in zip(lo, hi):
            seen = np.zeros(case["keys"] + 1, np.int64)
            some = h > l
            np.add.at(seen, l[some], 1)
            np.add.at(seen, h[some], -1)
            keys += int((np.cumsum(seen) > 0).sum())
        return {"bytes": size * case["dim"] * (2 * rows * case["heads"] + 2 * keys * case["kv_heads"]),
                "flops": 4 * case["dim"] * case["heads"] * pairs}
    if case["op"] == "rotate":
        tokens = int(_rotate_lengths(case).sum())
        width = (case["heads"] + 2 * case["kv_heads"]) * case["dim"]
        return {"bytes": 2 * size * tokens * width, "flops": 8 * tokens * width}
    n = case["batch"] * case["vocab"]
    return {"bytes": n * size + 8 * case["batch"], "flops": 4 * n}


def _rotate_lengths(case):
    if not case["ragged"]:
        return np.full(case["batch"], case["rows"], np.int32)
    return _lengths(case["batch"], case["rows"])


# ------------------------------------------------------------------ the inputs

def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    return {"attention": _prepare_attention, "rotate": _prepare_rotate, "sample": _prepare_sample}[case["op"]](case, gen)


def _normal(gen, *shape, dtype, gain=1.0):
    return (torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32) * gain).to(dtype)


def _prepare_attention(case, gen):
    dt, b, d = DTYPES[case["type"]], case["batch"], case["dim"]
    q_len, k_len = _attention_lengths(case)
    st = {"case": case, "scale": d ** -0.5, "q_len": None, "k_len": None, "prefix": None, "key_range": None,
          "slopes": None}
    # Queries and keys of unit size with learned gains give scores of a few units.
    st["q"] = _normal(gen, b, case["rows"], case["heads"], d, dtype=dt, gain=1.5)
    st["k"] = _normal(gen, b, case["keys"], case["kv_heads"], d, dtype=dt)
    st["v"] = _normal(gen, b, case["keys"], case["kv_heads"], d, dtype=dt)
    st["out"] = _normal(gen, b, case["rows"], case["heads"], d, dtype=dt)
    if case["ragged"]:
        st["q_len"] = torch.from_numpy(q_len).cuda()
        st["k_len"] = torch.from_numpy(k_len).cuda()
    if case["prefix"]:
        st["prefix"] = torch.from_numpy(_prefixes(case)).cuda()
    if case["docs"]:
        st["key_range"] = torch.from_numpy(_documents(case)).cuda()[None].contiguous()
    if case["slopes"]:
        st["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / case["heads"]) for h in range(case["heads"])],
                                    dtype=torch.float32, device="cuda")
    if own:
        st["attention"] = _ops().Attention(case["heads"], case["kv_heads"], d, dt, scale=st["scale"], cap=case["cap"],
                                           causal=case["causal"])
    return st


def _prepare_rotate(case, gen):
    dt, b, s, d = DTYPES[case["type"]], case["batch"], case["rows"], case["dim"]
    hq, hk = case["heads"], case["kv_heads"]
    qkv = _normal(gen, b, s, (hq + 2 * hk) * d, dtype=dt, gain=2.0)  # one packed projection
    st = {"case": case, "eps": 1e-6}
    st["q"] = qkv[..., : hq * d].unflatten(-1, (hq, d))
    st["k"] = qkv[..., hq * d: (hq + hk) * d].unflatten(-1, (hk, d))
    st["v"] = qkv[..., (hq + hk) * d:].unflatten(-1, (hk, d))
    st["q_weight"] = 1.0 + _normal(gen, d, dtype=torch.float32, gain=0.2)
    st["k_weight"] = 1.0 + _normal(gen, d, dtype=torch.float32, gain=0.2)
    r = case["rotary"]
    st["inv_freq"] = 10000.0 ** (-torch.arange(0, r, 2, dtype=torch.float64, device="cuda") / r)
    st["q_out"] = _normal(gen, b, s, hq, d, dtype=dt)
    st["k_cache"] = _normal(gen, b, case["cache"], hk, d, dtype=dt)
    st["v_cache"] = _normal(gen, b, case["cache"], hk, d, dtype=dt)
    start = np.array([int((case["cache"] - s) * (((i + 1) * GOLDEN) % 1.0)) for i in range(b)], dtype=np.int32)
    st["start"] = torch.from_numpy(start).cuda()
    st["length"] = torch.from_numpy(_rotate_lengths(case)).cuda() if case["ragged"] else None
    st["positions"] = None
    if case["far"]:  # the cache holds a window of a longer text
        pos = start[:, None].astype(np.int64) + np.arange(s)[None] + case["far"]
        st["positions"] = torch.from_numpy(pos.astype(np.int32)).cuda()
    return st


def _prepare_sample(case, gen):
    b, n = case["batch"], case["vocab"]
    logits = torch.randn(b, n, generator=gen, device="cuda") * 2.5
    # A few tokens stand out, as they do behind a trained model's last layer.
    few = torch.randint(0, n, (b, 8), generator=gen, device="cuda")
    logits.scatter_add_(1, few, torch.rand(b, 8, generator=gen, device="cuda") * 8.0)
    st = {"case": case, "logits": logits.to(DTYPES[case["type"]])}
    st["u"] = torch.rand(b, generator=gen, device="cuda")
    i = torch.arange(b, device="cuda")
    off = (i % 4 == 3) if case["mixed"] else torch.zeros(b, dtype=torch.bool, device="cuda")
    st["temperature"] = torch.full((b,), float(case["temperature"]), device="cuda")
    st["top_k"] = st["top_p"] = st["min_p"] = None
    if case["mixed"]:  # every fourth request has no filters, every seventh takes the best token
        st["temperature"] = torch.where(i % 7 == 6, 0.0, st["temperature"] + 0.01 * (i % 5))
    if case["top_k"]:
        st["top_k"] = torch.where(off, 0, case["top_k"]).to(torch.int32)
    if case["top_p"] < 1.0:
        st["top_p"] = torch.where(off, 1.0, case["top_p"]).to(torch.float32)
    if case["min_p"] > 0.0:
        st["min_p"] = torch.where(off, 0.0, case["min_p"]).to(torch.float32)
    return st


# -------------------------------------------------------------------- one pass

def run(st):
    op = st["case"]["op"]
    if own:
        return _RUN_OWN[op](st)
    return _RUN_PLAIN[op](st)


def _own_attention(st):
    return st["attention"](st["q"], st["k"], st["v"], out=st["out"], q_len=st["q_len"], k_len=st["k_len"],
                           prefix=st["prefix"], key_range=st["key_range"], slopes=st["slopes"])


def _own_rotate(st):
    _ops().qk_norm_rope(st["q"], st["k"], st["q_weight"], st["k_weight"], st["inv_freq"], q_out=st["q_out"],
                        k_out=st["k_cache"], v=st["v"], v_out=st["v_cache"], start=st["start"], length=st["length"],
                        positions=st["positions"], eps=st["eps"], interleaved=st["case"]["interleaved"])
    return st["q_out"], st["k_cache"], st["v_cache"]


def _own_sample(st):
    return _ops().sample(st["logits"], st["u"], temperature=st["temperature"], top_k=st["top_k"], top_p=st["top_p"],
                         min_p=st["min_p"])


def _plain_attention(st):
    case, q, k, v, out = st["case"], st["q"], st["k"], st["v"], st["out"]
    b, rows, heads, d = q.shape
    keys, kv = k.shape[1], k.shape[2]
    dev = q.device
    q_len = st["q_len"] if st["q_len"] is not None else torch.full((b,), rows, device=dev)
    k_len = st["k_len"] if st["k_len"] is not None else torch.full((b,), keys, device=dev)
    i = torch.arange(rows, device=dev)
    j = torch.arange(keys, device=dev)
    pos = (k_len - q_len)[:, None] + i[None]  # [b, rows]
    see = (j[None, None] < k_len[:, None, None]).expand(b, rows, keys)
    if case["causal"]:
        c = j[None, None] <= pos[..., None]
        if st["prefix"] is not None:
            c = c | (j[None, None] < st["prefix"][:, None, None])
        see = see & c
    if st["key_range"] is not None:
        r = st["key_range"]
        see = see & (j >= r[..., 0:1]) & (j < r[..., 1:2])
    used = (j[None] < k_len[:, None])[..., None, None]
    qf = q.float().view(b, rows, kv, heads // kv, d).permute(0, 2, 3, 1, 4).reshape(b, kv, -1, d)
    kf = torch.where(used, k.float(), 0.0).permute(0, 2, 3, 1)
    vf = torch.where(used, v.float(), 0.0).permute(0, 2, 1, 3)
    s = torch.matmul(qf, kf) * st["scale"]
    if case["cap"] > 0.0:
        s = torch.tanh(s / case["cap"]) * case["cap"]
    s = s.view(b, heads, rows, keys)
    if st["slopes"] is not None:
        s = s - st["slopes"][None, :, None, None] * (pos[..., None] - j).abs().float()[:, None]
    s = torch.where(see[:, None], s, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    l = p.sum(-1, keepdim=True)
    p = p / torch.where(l == 0.0, 1.0, l)
    o = torch.matmul(p.view(b, kv, -1, keys), vf).view(b, heads, rows, d).permute(0, 2, 1, 3)
    out.copy_(torch.where((i[None] < q_len[:, None])[..., None, None], o.to(q.dtype), out))
    return out


def _plain_rotate(st):
    case = st["case"]
    b, s = case["batch"], case["rows"]
    dev, half = st["q"].device, case["rotary"] // 2
    t = torch.arange(s, device=dev)
    row = st["start"][:, None].long() + t[None]
    pos = st["positions"].long() if st["positions"] is not None else row
    angle = pos[..., None].double() * st["inv_freq"]
    cos, sin = torch.cos(angle).float()[:, :, None], torch.sin(angle).float()[:, :, None]
    live = torch.ones(b, s, dtype=torch.bool, device=dev)
    if st["length"] is not None:
        live = t[None] < st["length"][:, None]

    def norm_rotate(x, w):
        y = x.float()
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + st["eps"]) * w
        if case["interleaved"]:
            a, c = y[..., 0: 2 * half: 2], y[..., 1: 2 * half: 2]
            turned = torch.stack((a * cos - c * sin, c * cos + a * sin), -1).flatten(-2)
        else:
            a, c = y[..., :half], y[..., half: 2 * half]
            turned = torch.cat((a * cos - c * sin, c * cos + a * sin), -1)
        return torch.cat((turned, y[..., 2 * half:]), -1).to(x.dtype)

    q = norm_rotate(st["q"], st["q_weight"])
    st["q_out"].copy_(torch.where(live[..., None, None], q, st["q_out"]))
    at = (torch.arange(b, device=dev)[:, None].expand(b, s), row)
    keep = live[..., None, None]
    st["k_cache"][at] = torch.where(keep, norm_rotate(st["k"], st["k_weight"]), st["k_cache"][at])
    st["v_cache"][at] = torch.where(keep, st["v"], st["v_cache"][at])
    return st["q_out"], st["k_cache"], st["v_cache"]


def _plain_sample(st):
    # Weights and running sums in 64 bits: the borders between 100,000 tokens lie closer than 32 bits resolve.
    x = st["logits"].double()
    b, n = x.shape
    t = st["temperature"].double()[:, None]
    greedy = t <= 0.0
    best = x.amax(1, keepdim=True)
    w = torch.exp((x - best) / torch.where(greedy, 1.0, t))
    if st["top_k"] is not None or st["top_p"] is not None:
        order = torch.sort(st["logits"].float(), dim=1, descending=True, stable=True).indices
        ws = w.gather(1, order)
        if st["top_k"] is not None:
            k = st["top_k"].long()[:, None]
            rank = torch.arange(n, device=x.device)[None]
            ws = torch.where((k <= 0) | (rank < k), ws, 0.0)
        if st["top_p"] is not None:
            p = st["top_p"].double()[:, None]
            run_ = torch.cumsum(ws, 1)
            before = run_ - ws
            ws = torch.where((p >= 1.0) | (before < p * run_[:, -1:]), ws, 0.0)
        w = torch.zeros_like(w).scatter(1, order, ws)
    if st["min_p"] is not None:
        w = torch.where(w >= st["min_p"].double()[:, None], w, 0.0)
    run_ = torch.cumsum(w, 1)
    goal = st["u"].double()[:, None] * run_[:, -1:]
    token = (run_ > goal).int().argmax(1)
    logprob = torch.log(w.gather(1, token[:, None]) / run_[:, -1:])[:, 0]
    first = (x == best).int().argmax(1)
    token = torch.where(greedy[:, 0], first, token).to(torch.int32)
    return token, torch.where(greedy[:, 0], 0.0, logprob).float()


_RUN_OWN = {"attention": _own_attention, "rotate": _own_rotate, "sample": _own_sample}
_RUN_PLAIN = {"attention": _plain_attention, "rotate": _plain_rotate, "sample": _plain_sample}


# ---------------------------------------------------- the definition, in 64 bits

def exact(case, seed):
    global own
    kept, own = own, False  # inputs only, no handle
    try:
        st = prepare(case, seed)
    finally:
        own = kept
    return {"attention": _exact_attention, "rotate": _exact_rotate, "sample": _exact_sample}[case["op"]](case, st)


def _exact_attention(case, st):
    lo, hi = _visible(case)
    _, k_len = _attention_lengths(case)
    out = st["out"].double()
    group = case["heads"] // case["kv_heads"]
    for b in range(case["batch"]):
        n, m = len(lo[b]), int(k_len[b])
        first = torch.from_numpy(lo[b]).cuda()[:, None]
        end = torch.from_numpy(hi[b]).cuda()[:, None]
        key = torch.arange(m, device="cuda")[None]
        hidden = (key < first) | (key >= end)
        for h in range(case["heads"]):
            x = st["q"][b, :n, h].double() @ st["k"][b, :m, h // group].double().T
            x *= st["scale"]
            if case["cap"] > 0.0:
                x = case["cap"] * torch.tanh(x / case["cap"])
            if case["slopes"]:
                row = torch.arange(n, device="cuda")[:, None] + (m - n)
                x -= float(st["slopes"][h]) * (row - key).abs().double()
            x.masked_fill_(hidden, -math.inf)
            x -= x.amax(1, keepdim=True).clamp_min(-1e300)
            x.exp_()
            total = x.sum(1, keepdim=True)
            o = x @ st["v"][b, :m, h // group].double()
            out[b, :n, h] = torch.where(total > 0.0, o / total.clamp_min(1e-300), 0.0)
    return out


def _exact_rotate(case, st):
    n = _rotate_lengths(case)
    q_out, k_cache, v_cache = st["q_out"].double(), st["k_cache"].double(), st["v_cache"].double()
    r = case["rotary"]
    if case["interleaved"]:
        left, right = torch.arange(0, r, 2), torch.arange(1, r, 2)
    else:
        left, right = torch.arange(0, r // 2), torch.arange(r // 2, r)

    def apply(x, w, turn):
        x = x.double()
        y = x * w.double() / torch.sqrt((x ** 2).sum(-1, keepdim=True) / x.shape[-1] + st["eps"])
        z = torch.complex(y[..., left], y[..., right]) * turn
        y[..., left], y[..., right] = z.real, z.imag
        return y

    for b in range(case["batch"]):
        m, a = int(n[b]), int(st["start"][b])
        pos = (st["positions"][b, :m] if st["positions"] is not None else a + torch.arange(m, device="cuda")).double()
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                           torch.outer(pos, st["inv_freq"]))[:, None]
        q_out[b, :m] = apply(st["q"][b, :m], st["q_weight"], turn)
        k_cache[b, a: a + m] = apply(st["k"][b, :m], st["k_weight"], turn)
        v_cache[b, a: a + m] = st["v"][b, :m].double()
    return q_out, k_cache, v_cache


def _exact_sample(case, st):
    logits = st["logits"].double().cpu().numpy()
    u = st["u"].cpu().numpy().astype(np.float64)

    def setting(name, b, default):
        return default if st[name] is None else st[name][b].item()

    tokens, logprobs = [], []
    for b in range(case["batch"]):
        x = logits[b]
        t = setting("temperature", b, 1.0)
        if t <= 0.0:
            tokens.append(int(np.argmax(x)))
            logprobs.append(0.0)
            continue
        w = np.exp((x - x.max()) / t)
        k, p = setting("top_k", b, 0), setting("top_p", b, 1.0)
        kept = np.ones(x.size, dtype=bool)
        if k > 0 or p < 1.0:
            order = np.argsort(-x, kind="stable")
            count = min(k, x.size) if k > 0 else x.size
            mass = np.cumsum(w[order[:count]])
            if p < 1.0:
                count = 1 + int(np.searchsorted(mass[:-1], p * mass[-1], side="left"))
            kept[:] = False
            kept[order[:count]] = True
        kept &= w >= setting("min_p", b, 0.0)
        at = np.flatnonzero(kept)
        mass = np.cumsum(w[at])
        tokens.append(int(at[min(int(np.searchsorted(mass, u[b] * mass[-1], side="right")), at.size - 1)]))
        logprobs.append(float(np.log(w[tokens[-1]] / mass[-1])))
    return torch.tensor(tokens, dtype=torch.int32), torch.tensor(logprobs, dtype=torch.float64)
