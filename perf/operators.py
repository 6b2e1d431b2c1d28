"""Token-by-token decoding over a paged key / value cache, measured: appending rotated keys and values to the cache,
attention of new tokens over it, and drawing the next token from the logits.

Each operator has its plain form here (elementary torch operations) and the call a user makes of the library.

  append   a = pos * inv_freq;  (x1, x2) -> (x1 cos a - x2 sin a, x2 cos a + x1 sin a) for the pairs of q and k;
           the cache row of token i of sequence b is position kv_len[b] - n_b + i, in page block_table[b, position // P]
  attend   o_i = sum_j softmax_j(scale q_i . k_j) v_j over the keys j < kv_len[b] that query i sees: j <= position of i
           where causal, j > position of i - window where a window is given; a query that sees no key gives zeros
  sample   p = softmax(logits / T); tokens sorted by logit, ties by index; kept: the first top_k of them, of these the
           ones before which less than top_p of the kept mass lies, of these the ones with p >= min_p max(p);
           answer: the first kept index, in the vocabulary's order, whose running sum of p exceeds u times the kept
           mass; T = 0: the largest logit. Also the answer's probability among the kept ones.
"""
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # one stream's next token: 4 heads of 128, everything is latency
        {"name": "append_one", "op": "append", "dtype": "bf16", "batch": 1, "new": 1, "ragged": False, "ctx": 37,
         "q_heads": 4, "kv_heads": 4, "dim": 128, "rot": 128, "interleaved": False, "page": 16, "lens": 1},
        # a batch of decoding requests, half of each head rotated in neighbouring pairs, pages of an odd size
        {"name": "append_batch", "op": "append", "dtype": "f16", "batch": 64, "new": 1, "ragged": False, "ctx": 4000,
         "q_heads": 16, "kv_heads": 4, "dim": 96, "rot": 48, "interleaved": True, "page": 24, "lens": 2},
        # prompts of different lengths entering at once, far into long contexts
        {"name": "append_chunks", "op": "append", "dtype": "bf16", "batch": 12, "new": 2600, "ragged": True,
         "ctx": 120000, "q_heads": 32, "kv_heads": 8, "dim": 128, "rot": 128, "interleaved": False, "page": 64,
         "lens": 3},
        # one stream's next token over a short cache
        {"name": "attend_one", "op": "attend", "dtype": "bf16", "batch": 1, "new": 1, "ragged": False, "ctx": 200,
         "q_heads": 4, "kv_heads": 4, "dim": 128, "page": 16, "causal": True, "window": 0, "lens": 4},
        # a batch of decoding requests of every length
        {"name": "attend_batch", "op": "attend", "dtype": "bf16", "batch": 64, "new": 1, "ragged": False, "ctx": 8192,
         "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "causal": True, "window": 0, "lens": 5},
        # two requests with very long caches
        {"name": "attend_long", "op": "attend", "dtype": "f16", "batch": 2, "new": 1, "ragged": False, "ctx": 131072,
         "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 128, "causal": True, "window": 0, "lens": 6},
        # chunks of prompts, ragged, beside what is cached already
        {"name": "attend_chunks", "op": "attend", "dtype": "bf16", "batch": 8, "new": 700, "ragged": True,
         "ctx": 6000, "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "causal": True, "window": 0, "lens": 7},
        # two long prompts in large chunks: the matrix products bound it
        {"name": "attend_prompt", "op": "attend", "dtype": "bf16", "batch": 2, "new": 4096, "ragged": False,
         "ctx": 4096, "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "causal": True, "window": 0, "lens": 8},
        # 64 speech streams' chunks of 15 rows that see themselves whole and 40 rows back, in 32 bits
        {"name": "attend_streams", "op": "attend", "dtype": "f32", "batch": 64, "new": 15, "ragged": False,
         "ctx": 600, "q_heads": 4, "kv_heads": 4, "dim": 128, "page": 10, "causal": False, "window": 55, "lens": 9},
        # one stream's next token from a speech vocabulary
        {"name": "sample_one", "op": "sample", "dtype": "f32", "batch": 1, "vocab": 8404, "mode": "topk_topp",
         "banned": 0.0},
        # a batch of requests with settings of their own, some tokens banned, logits in 16 bits (many ties)
        {"name": "sample_batch", "op": "sample", "dtype": "bf16", "batch": 64, "vocab": 128000, "mode": "mixed",
         "banned": 0.02},
        # a large batch that samples from nearly the whole distribution
        {"name": "sample_full", "op": "sample", "dtype": "f32", "batch": 256, "vocab": 131071, "mode": "topp",
         "banned": 0.0},
    ]


def draw(rng):
    def log(a, b):
        return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))

    case = {"op": rng.choice(["append", "attend", "attend", "sample"]), "dtype": rng.choice(["bf16", "bf16", "f16", "f32"])}
    if case["op"] == "sample":
        case |= {"batch": log(1, 256), "vocab": log(1000, 131072), "mode": rng.choice(["mixed", "topk_topp", "topp", "plain", "minp"]),
                 "banned": rng.choice([0.0, 0.02, 0.5])}
        return case
    kv = rng.choice([1, 2, 4, 8])
    case |= {"lens": rng.randrange(1 << 30), "q_heads": kv * rng.choice([1, 2, 3, 4, 7, 8]), "kv_heads": kv, "dim": rng.choice([32, 64, 64, 80, 96, 128, 128, 128, 256]),
             "page": rng.choice([1, 8, 16, 16, 17, 32, 64, 64, 100, 128, 256])}
    one = rng.random() < 0.5
    if case["op"] == "append":
        batch = log(1, 128) if one else log(1, 16)
        new = 1 if one else log(2, 2000)
        rot = rng.choice([r for r in (16, 32, 48, 64, 80, 96, 128, 256) if r <= case["dim"]] + [case["dim"] // 16 * 16])
        case |= {"batch": batch, "new": new, "ragged": not one and rng.random() < 0.7, "ctx": log(1, 120000), "rot": rot,
                 "interleaved": rng.random() < 0.4}
        return case
    batch = log(1, 96) if one else log(1, 12)
    new = 1 if one else log(2, 2000)
    ctx = log(1, 60000) if one else log(1, 8000)
    case |= {"batch": batch, "new": new, "ragged": not one and rng.random() < 0.7, "ctx": ctx,
             "causal": rng.random() < 0.75, "window": rng.choice([0, 0, 0, log(1, 4000)])}

    def large():   # no more than the largest listed one, the plain form's score matrix included
        w = work(case)
        return (w["flops"] > 3e11 or w["bytes"] > 8e8 or
                batch * case["new"] * case["q_heads"] * (case["ctx"] + case["new"]) > 2e9)

    while large():
        case[max(("ctx", "new"), key=case.get)] //= 2
    return case


def lengths(case):
    """(new tokens, keys in the cache with them) of each sequence."""
    r = random.Random(case["lens"])
    new = [r.randint(max(1, case["new"] // 8), case["new"]) if case["ragged"] else case["new"] for _ in range(case["batch"])]
    if case["ragged"] and case["batch"] > 2:
        new[1] = 0   # a request that waits this step out
    if case["ragged"]:
        new[-1] = case["new"]
    old = [r.randint(case["ctx"] // 8, case["ctx"]) for _ in range(case["batch"])]
    old[0] = case["ctx"]
    return new, [n + o for n, o in zip(new, old)]


def seen(case):
    """(visible query-key pairs, distinct visible keys) of one head over all sequences."""
    pairs = keys = 0
    for n, m in zip(*lengths(case)):
        if not n:
            continue
        p = np.arange(m - n, m, dtype=np.int64)
        hi = p + 1 if case["causal"] else np.full(n, m, np.int64)
        lo = np.maximum(p - case["window"] + 1, 0) if case["window"] else np.zeros(n, np.int64)
        pairs += int((hi - lo).sum())
        keys += int(hi[-1] - lo[0])
    return pairs, keys


def work(case):
    s = BYTES[case["dtype"]]
    if case["op"] == "sample":
        n = case["batch"] * case["vocab"]
        return {"bytes": n * s + case["batch"] * 28, "flops": 4 * n}
    new, _ = lengths(case)
    n, d = sum(new), case["dim"]
    if case["op"] == "append":
        return {"bytes": 2 * s * n * d * (case["q_heads"] + 2 * case["kv_heads"]) + 12 * case["batch"],
                "flops": 3 * n * case["rot"] * (case["q_heads"] + case["kv_heads"])}
    pairs, keys = seen(case)
    return {"bytes": s * d * (2 * n * case["q_heads"] + 2 * keys * case["kv_heads"]) + 4 * (keys // case["page"]) + 12 * case["batch"],
            "flops": 4 * pairs * d * case["q_heads"]}


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dt)

    if case["op"] == "sample":
        return _prepare_sample(case, seed, g, dt)
    new, kv = lengths(case)
    batch, page, n = case["batch"], case["page"], sum(new)
    hq, hk, d = case["q_heads"], case["kv_heads"], case["dim"]
    state = {"case": case, "most_new": max(new), "most_kv": max(kv),
             "kv_len": torch.tensor(kv, dtype=torch.int32, device="cuda"),
             "cu_q": None if max(new) == min(new) == 1 else
             torch.tensor([0] + np.cumsum(new).tolist(), dtype=torch.int32, device="cuda")}
    # the projection's output: q, k and v side by side in one row per token
    qkv = normal(n, hq + 2 * hk, d)
    state |= {"q": qkv[:, :hq], "k": qkv[:, hq:hq + hk], "v": qkv[:, hq + hk:]}
    r = random.Random(seed)
    width = -(-max(kv) // page)
    table = np.full((batch, width), -1, np.int32)
    if case["op"] == "append":   # the pages before the new tokens are not touched: one shared page stands for them
        first = [(m - c) // page for c, m in zip(new, kv)]
        last = [-(-m // page) for m in kv]
        pool = 1 + sum(b - a for a, b in zip(first, last))
    else:
        first, last = [0] * batch, [-(-m // page) for m in kv]
        pool = sum(last)
    ids = list(range(1 if case["op"] == "append" else 0, pool))
    r.shuffle(ids)
    at = 0
    for b, (f, e) in enumerate(zip(first, last)):
        table[b, :f] = 0
        table[b, f:e] = ids[at:at + e - f]
        at += e - f
    state["table"] = torch.from_numpy(table).cuda()
    state["k_pages"], state["v_pages"] = normal(pool, page, hk, d), normal(pool, page, hk, d)
    if case["op"] == "append":
        half = case["rot"] // 2
        state["inv_freq"] = (10000.0 ** (-torch.arange(half, dtype=torch.float64) / half)).float().cuda()
    return state


def _prepare_sample(case, seed, g, dt):
    batch, vocab, r = case["batch"], case["vocab"], random.Random(seed)
    x = torch.randn((batch, vocab), generator=g, device="cuda") * 2.5
    best = torch.randint(0, vocab, (batch, 24), generator=g, device="cuda")   # the few tokens that fit
    x.scatter_(1, best, 8 + 4 * torch.randn((batch, 24), generator=g, device="cuda"))
    if case["banned"]:
        x.masked_fill_(torch.rand((batch, vocab), generator=g, device="cuda") < case["banned"], -math.inf)
    x[:, vocab // 2] = 6.0   # some token is always allowed
    mode = case["mode"]

    def rows(make):
        return torch.tensor([make() for _ in range(batch)], device="cuda")

    def some(make, off):
        return lambda: make() if mode != "mixed" or r.random() < 0.6 else off

    temperature = rows(lambda: 0.0 if mode == "mixed" and r.random() < 0.15 else r.uniform(0.3, 1.4)).float()
    top_k = rows(some(lambda: r.randint(1, 200), 0)).int() if mode in ("mixed", "topk_topp") else None
    top_p = rows(some(lambda: r.uniform(0.5, 0.99), 1.0)).float() if mode in ("mixed", "topk_topp", "topp") else None
    min_p = rows(some(lambda: r.uniform(0.005, 0.2), 0.0)).float() if mode in ("mixed", "minp") else None
    return {"case": case, "logits": x.to(dt), "u": torch.rand(batch, generator=g, device="cuda"),
            "temperature": temperature, "top_k": top_k, "top_p": top_p, "min_p": min_p}


def run(state):
    case = state["case"]
    if own:
        return _own(state, case)
    return {"append": _append, "attend": _attend, "sample": _sample}[case["op"]](state, case)


def _own(s, case):
    from funasr_amd import runtime as rt
    if case["op"] == "append":
        q = rt.op_kv_append(s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["kv_len"], s["cu_q"], q=s["q"],
                            inv_freq=s["inv_freq"], interleaved=case["interleaved"])
        return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    if case["op"] == "attend":
        return rt.op_paged_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["kv_len"], s["cu_q"],
                                     causal=case["causal"], window=case["window"])
    token, prob = rt.op_sample(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                               min_p=s["min_p"])
    return {"token": token, "prob": prob}


def _positions(s, case):
    """(sequence, place among its new tokens, position) of every new token."""
    n = s["q"].shape[0]
    cu = s["cu_q"].long() if s["cu_q"] is not None else torch.arange(case["batch"] + 1, device="cuda")
    i = torch.arange(n, device="cuda")
    seq = torch.searchsorted(cu[1:].contiguous(), i, right=True)
    place = i - cu[seq]
    return seq, place, s["kv_len"].long()[seq] - (cu[seq + 1] - cu[seq]) + place


def _rotated(x, pos, inv_freq, interleaved):
    angle = pos.double()[:, None] * inv_freq.double()     # far positions: 32 bits would lose the angle
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    x, half = x.float(), inv_freq.numel()
    a, b = (x[..., 0:2 * half:2], x[..., 1:2 * half:2]) if interleaved else (x[..., :half], x[..., half:2 * half])
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((turned, x[..., 2 * half:]), -1)


def _append(s, case):
    seq, _, pos = _positions(s, case)
    page, slot = s["table"].long()[seq, pos // case["page"]], pos % case["page"]
    dt = s["q"].dtype
    q = _rotated(s["q"], pos, s["inv_freq"], case["interleaved"]).to(dt)
    s["k_pages"][page, slot] = _rotated(s["k"], pos, s["inv_freq"], case["interleaved"]).to(dt)
    s["v_pages"][page, slot] = s["v"]
    return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _attend(s, case):
    batch, hq, hk, d = case["batch"], case["q_heads"], case["kv_heads"], case["dim"]
    seq, place, pos = _positions(s, case)
    j = torch.arange(s["most_kv"], device="cuda")
    pages, slots = s["table"].long().clamp_min(0)[:, j // case["page"]], j % case["page"]
    k = s["k_pages"][pages, slots].float().permute(0, 2, 3, 1).contiguous()          # [batch, hk, d, keys]
    v = s["v_pages"][pages, slots].float().permute(0, 2, 1, 3).contiguous()          # [batch, hk, keys, d]
    q = torch.zeros((batch, s["most_new"], hq, d), device="cuda")
    q[seq, place] = s["q"].float()
    at = torch.full((batch, s["most_new"]), -1, device="cuda")
    at[seq, place] = pos
    q = q.view(batch, s["most_new"], hk, hq // hk, d).permute(0, 2, 1, 3, 4).reshape(batch, hk, -1, d)
    visible = j < s["kv_len"].long()[:, None, None]
    if case["causal"]:
        visible = visible & (j <= at[..., None])
    if case["window"]:
        visible = visible & (j > at[..., None] - case["window"])
    hidden = ~visible.expand(batch, s["most_new"], -1).repeat_interleave(hq // hk, 1)[:, None]
    x = torch.matmul(q, k).mul_(d ** -0.5).masked_fill_(hidden, -math.inf)
    top = x.amax(-1, keepdim=True)
    x = x.sub_(top.masked_fill(top == -math.inf, 0.0)).exp_()
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x, v) / total.masked_fill(total == 0, 1.0)
    o = o.view(batch, hk, s["most_new"], hq // hk, d).permute(0, 2, 1, 3, 4).reshape(batch, s["most_new"], hq, d)
    return o[seq, place].to(s["q"].dtype)


def _sample(s, case):
    # in 64 bits: the running sums are compared with borders
    batch, vocab = case["batch"], case["vocab"]
    x = s["logits"].double()
    t = s["temperature"].double()[:, None]
    greedy = t <= 0
    order = torch.sort(x, dim=-1, descending=True, stable=True)
    rank = torch.arange(vocab, device="cuda")
    p = ((order.values - order.values[:, :1]) / torch.where(greedy, 1.0, t)).exp()
    keep = (rank == 0) | (p > 0)
    if s["top_k"] is not None:
        k = s["top_k"].long()[:, None]
        keep = keep & ((k <= 0) | (rank < k))
    if s["top_p"] is not None:
        among = torch.where(keep, p, 0.0)
        before = among.cumsum(-1) - among
        limit = s["top_p"].double()[:, None]
        keep = keep & ((limit >= 1) | (rank == 0) | (before < limit * among.sum(-1, keepdim=True)))
    if s["min_p"] is not None:
        keep = keep & (p >= s["min_p"].double()[:, None])
    keep = torch.where(greedy, rank == 0, keep)
    w = torch.zeros_like(p).scatter_(1, order.indices, torch.where(keep, p, 0.0))
    run_sum = w.cumsum(-1)
    total = run_sum[:, -1:]
    token = (run_sum <= s["u"].double()[:, None] * total).sum(-1, keepdim=True)
    return {"token": token[:, 0].int(), "prob": (w.gather(1, token) / total)[:, 0].float()}


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "sample": _exact_sample}[case["op"]](s, case)


def _exact_append(s, case):
    new, kv = lengths(case)
    k_pages, v_pages, q = s["k_pages"].double(), s["v_pages"].double(), s["q"].double().clone()
    table, half, done = s["table"].tolist(), case["rot"] // 2, 0
    freq = s["inv_freq"].double()
    for b, (n, m) in enumerate(zip(new, kv)):
        if not n:
            continue
        pos = torch.arange(m - n, m, device="cuda")
        turn = torch.polar(torch.ones(1, dtype=torch.float64, device="cuda"), pos[:, None] * freq)[:, None]

        def turned(x):
            x = x.double().clone()
            even, odd = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if case["interleaved"] else (slice(0, half), slice(half, 2 * half))
            z = torch.complex(x[..., even].contiguous(), x[..., odd].contiguous()) * turn
            x[..., even], x[..., odd] = z.real, z.imag
            return x

        q[done:done + n] = turned(s["q"][done:done + n])
        page = torch.tensor([table[b][p // case["page"]] for p in range(m - n, m)], device="cuda")
        k_pages[page, pos % case["page"]] = turned(s["k"][done:done + n])
        v_pages[page, pos % case["page"]] = s["v"][done:done + n].double()
        done += n
    return {"q": q, "k_pages": k_pages, "v_pages": v_pages}


def _exact_attend(s, case):
    new, kv = lengths(case)
    out, done = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), 0
    group = case["q_heads"] // case["kv_heads"]
    for b, (n, m) in enumerate(zip(new, kv)):
        if not n:
            continue
        pages = s["table"][b, :-(-m // case["page"])].long()
        k = s["k_pages"][pages].flatten(0, 1)[:m].double()
        v = s["v_pages"][pages].flatten(0, 1)[:m].double()
        far = torch.arange(m - n, m, device="cuda")[:, None] - torch.arange(m, device="cuda")[None]   # query - key
        off = torch.zeros_like(far, dtype=torch.bool)
        if case["causal"]:
            off |= far < 0
        if case["window"]:
            off |= far >= case["window"]
        for h in range(case["q_heads"]):
            x = s["q"][done:done + n, h].double() @ k[:, h // group].t().contiguous() / math.sqrt(case["dim"])
            x[off] = -math.inf
            out[done:done + n, h] = torch.exp(x - torch.logsumexp(x, 1, keepdim=True)).nan_to_num(0.0) @ v[:, h // group].contiguous()
        done += n
    return out


def _exact_sample(s, case):
    x, u, t = s["logits"].double().cpu().numpy(), s["u"].double().cpu().numpy(), s["temperature"].double().cpu().numpy()
    setting = {n: None if s[n] is None else s[n].double().cpu().numpy() for n in ("top_k", "top_p", "min_p")}
    token, prob = np.zeros(case["batch"], np.int32), np.ones(case["batch"])
    for b in range(case["batch"]):
        row = x[b]
        if t[b] <= 0:
            token[b] = int(np.argmax(row))
            continue
        p = np.exp((row - row.max()) / t[b])
        order = np.argsort(-row, kind="stable")
        order = order[:max(1, int(np.count_nonzero(p)))]
        if setting["top_k"] is not None and setting["top_k"][b] > 0:
            order = order[:int(setting["top_k"][b])]
        if setting["top_p"] is not None and setting["top_p"][b] < 1:
            sums = np.cumsum(p[order])
            order = order[:1 + int(np.searchsorted(sums[:-1], setting["top_p"][b] * sums[-1], side="left"))]
        if setting["min_p"] is not None:
            order = order[p[order] >= setting["min_p"][b]]
        kept = np.sort(order)
        sums = np.cumsum(p[kept])
        at = min(int(np.searchsorted(sums, u[b] * sums[-1], side="right")), len(kept) - 1)
        token[b], prob[b] = kept[at], p[kept[at]] / sums[-1]
    return {"token": token, "prob": prob}
