"""Timed cases of the operators of a decode step over a paged KV cache.

Four operators, as a serving program calls them, one after the other:

* ``pages``: block tables, slots and lengths from the requests' lengths;
* ``append``: per-head norm of q and k, rotation, append of k and v to pages;
* ``attention``: one new token per request over its pages;
* ``logprobs``: log-probabilities of given tokens, entropy, top alternatives.

With ``own`` false, :func:`run` computes them in their plain form; with
``own`` true it calls this package.
"""

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-5


# ------------------------------------------------------------------ cases --
def listed():
    return [
        # eight requests decode one token each with the 1024-token context of the decode benchmark
        {"name": "pages decode b8", "op": "pages", "batch": 8, "cached": 1024, "new": 1, "page": 64, "pad": 0,
         "mix": 1},
        # prompts of very different lengths are admitted together, on top of cached prefixes; rows of padding behind
        {"name": "pages prefill b96", "op": "pages", "batch": 96, "cached": 4097, "new": 1300, "page": 16, "pad": 37,
         "mix": 2},
        # one token, one rank of a 64 / 8 head model over 8 GPUs: latency
        {"name": "append t1 tp8", "op": "append", "tokens": 1, "q_heads": 8, "kv_heads": 1, "dim": 128,
         "rotary": 128, "interleaved": False, "norm": False, "page": 64, "dtype": "bf16", "max_pos": 4096},
        # a decode batch with normed heads, interleaved pairs on half of each head
        {"name": "append t61 interleaved", "op": "append", "tokens": 61, "q_heads": 32, "kv_heads": 8, "dim": 128,
         "rotary": 64, "interleaved": True, "norm": True, "page": 16, "dtype": "fp16", "max_pos": 8192},
        # a chunk of prompts of a 32 / 8 head model
        {"name": "append t8191 normed", "op": "append", "tokens": 8191, "q_heads": 32, "kv_heads": 8, "dim": 128,
         "rotary": 128, "interleaved": False, "norm": True, "page": 64, "dtype": "bf16", "max_pos": 32768},
        # one request of the decode benchmark on one of 8 ranks: latency
        {"name": "attention b1 c1025 tp8", "op": "attention", "batch": 1, "context": 1025, "ragged": False,
         "empty": False, "q_heads": 8, "kv_heads": 1, "dim": 128, "page": 64, "dtype": "bf16", "mix": 3},
        # the decode benchmark's batch, requests of all lengths, one slot of the batch empty
        {"name": "attention b32 ragged", "op": "attention", "batch": 32, "context": 2500, "ragged": True,
         "empty": True, "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "dtype": "bf16", "mix": 4},
        # one very long request, half-width heads: all the GPU on one cache
        {"name": "attention b1 c131071 d64", "op": "attention", "batch": 1, "context": 131071, "ragged": False,
         "empty": False, "q_heads": 32, "kv_heads": 8, "dim": 64, "page": 128, "dtype": "fp16", "mix": 5},
        # a full batch of long requests: the bandwidth case
        {"name": "attention b64 c8192", "op": "attention", "batch": 64, "context": 8192, "ragged": True,
         "empty": False, "q_heads": 64, "kv_heads": 8, "dim": 128, "page": 64, "dtype": "bf16", "mix": 6},
        # one decoded token of the whole vocabulary: latency
        {"name": "logprobs t1", "op": "logprobs", "rows": 1, "vocab": 128256, "top": 5, "dtype": "bf16", "shard": 0},
        # a decode batch on one of 8 vocabulary shards
        {"name": "logprobs t32 shard fp32", "op": "logprobs", "rows": 32, "vocab": 16128, "top": 8, "dtype": "fp32",
         "shard": 3},
        # log-probabilities of a prompt chunk
        {"name": "logprobs t1023", "op": "logprobs", "rows": 1023, "vocab": 128256, "top": 20, "dtype": "bf16",
         "shard": 0},
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["pages", "append", "attention", "logprobs"])
    page = rng.choice([16, 32, 64, 128])
    if op == "pages":
        return {"op": op, "batch": _spread(rng, 1, 400), "cached": _spread(rng, 1, 20000),
                "new": rng.choice([1, 1, _spread(rng, 2, 300)]), "page": page, "pad": rng.randrange(64),
                "mix": rng.randrange(1 << 20)}
    if op == "append":
        kv, dim = rng.choice([1, 2, 4, 8]), rng.choice([64, 128])
        return {"op": op, "tokens": _spread(rng, 1, 8000), "q_heads": kv * rng.choice([1, 2, 3, 4, 5, 8]) if kv < 8
                else kv * rng.choice([1, 2, 3, 4]), "kv_heads": kv, "dim": dim,
                "rotary": rng.choice([dim, dim, dim // 2, dim // 4]), "interleaved": rng.random() < 0.4,
                "norm": rng.random() < 0.5, "page": page, "dtype": rng.choice(["bf16", "fp16"]),
                "max_pos": _spread(rng, 256, 32768)}
    if op == "attention":
        kv, dim = rng.choice([1, 2, 4, 8]), rng.choice([64, 128])
        batch, context = _spread(rng, 1, 200), _spread(rng, 1, 30000)
        while batch * context * kv * dim > 64 * 8192 * 8 * 128 // 2:
            batch, context = max(1, batch * 2 // 3), max(1, context * 3 // 4)
        return {"op": op, "batch": batch, "context": context, "ragged": rng.random() < 0.7,
                "empty": rng.random() < 0.3, "q_heads": kv * rng.choice([1, 2, 3, 4, 5, 7, 8, 12, 16]),
                "kv_heads": kv, "dim": dim, "page": page, "dtype": rng.choice(["bf16", "fp16"]),
                "mix": rng.randrange(1 << 20)}
    vocab = rng.choice([128256, 16128, 16032, _spread(rng, 100, 260000)])
    rows = min(_spread(rng, 1, 1000), 1023 * 128256 * 2 // (vocab * 4))
    return {"op": op, "rows": rows, "vocab": vocab, "top": rng.choice([0, 1, 5, 20, 32]),
            "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "shard": rng.choice([0, 0, 1, 7])}


def _lengths(case):
    """Cached lengths (attention: lengths) and new tokens of each request: part of the case, not of the seed."""
    r = random.Random(case["mix"])
    if case["op"] == "pages":
        cached = [r.randint(0, case["cached"]) for _ in range(case["batch"])]
        new = [1 if case["new"] == 1 else r.randint(0, case["new"]) for _ in range(case["batch"])]
        new[0] = max(1, new[0])
        return cached, new
    n = [r.randint(1, case["context"]) if case["ragged"] else case["context"] for _ in range(case["batch"])]
    n[0] = case["context"]
    if case["empty"] and case["batch"] > 1:
        n[1] = 0
    return n


def _ceil(a, b):
    return -(-a // b)


def work(case):
    if case["op"] == "pages":
        cached, new = _lengths(case)
        p = case["page"]
        fresh = sum(_ceil(c + n, p) - _ceil(c, p) for c, n in zip(cached, new))
        seen = sum(_ceil(c + n, p) - c // p for c, n in zip(cached, new) if n)  # pages that new tokens lie in
        rows = sum(new) + case["pad"]
        return {"bytes": rows * 12 + len(new) * 12 + 4 * seen + 4 * fresh, "flops": 0}
    if case["op"] == "append":
        e, width = DTYPES[case["dtype"]].itemsize, (case["q_heads"] + 2 * case["kv_heads"]) * case["dim"]
        rotated = (case["q_heads"] + case["kv_heads"]) * case["rotary"]
        # every token's row of the two tables (a row used twice is read once)
        table = min(case["tokens"], case["max_pos"]) * case["rotary"] * 4
        return {"bytes": case["tokens"] * (2 * width * e + 12) + table, "flops": case["tokens"] * 3 * rotated}
    if case["op"] == "attention":
        e, total = DTYPES[case["dtype"]].itemsize, sum(_lengths(case))
        return {"bytes": (2 * total * case["kv_heads"] + 2 * case["batch"] * case["q_heads"]) * case["dim"] * e
                + 4 * case["batch"], "flops": 4 * total * case["q_heads"] * case["dim"]}
    e = DTYPES[case["dtype"]].itemsize
    return {"bytes": case["rows"] * (case["vocab"] * e + 8 + 12 + 12 * case["top"]),
            "flops": 6 * case["rows"] * case["vocab"]}


# ----------------------------------------------------------------- inputs --
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dev = "cuda"
    s = {"case": case}

    def randn(*shape, dtype=torch.float32, scale=1.0):
        return (torch.randn(*shape, generator=g, device=dev) * scale).to(dtype)

    if case["op"] == "pages":
        cached, new = _lengths(case)
        p = case["page"]
        held = [_ceil(c, p) for c in cached]
        width = max(_ceil(c + n, p) for c, n in zip(cached, new)) + 3
        total = sum(_ceil(c + n, p) for c, n in zip(cached, new)) + 11
        perm = torch.randperm(total, generator=g, device=dev).int()
        at = torch.arange(width, device=dev)[None] < torch.tensor(held, device=dev)[:, None]
        tables = torch.full((len(cached), width), -1, dtype=torch.int32, device=dev)
        tables[at] = perm[:sum(held)]
        starts = torch.tensor([0] + new, device=dev).cumsum(0).int()
        # the free list, of which the first three were taken by earlier steps
        s.update(cached=torch.tensor(cached, dtype=torch.int32, device=dev), starts=starts, tables=tables,
                 free=torch.cat([perm[:3], perm[sum(held):]]).contiguous(),
                 taken=torch.full((1,), 3, dtype=torch.int32, device=dev), rows=sum(new) + case["pad"])
    elif case["op"] == "append":
        t, d, dt, p = case["tokens"], case["dim"], DTYPES[case["dtype"]], case["page"]
        hq, hkv = case["q_heads"], case["kv_heads"]
        pages = _ceil(t, p) + 5
        inv = 500000.0 ** (-torch.arange(0, case["rotary"], 2, device=dev, dtype=torch.float64) / case["rotary"])
        ang = torch.arange(case["max_pos"], device=dev, dtype=torch.float64)[:, None] * inv
        s.update(qkv=randn(t, (hq + 2 * hkv) * d, dtype=dt), cos=ang.cos().float(), sin=ang.sin().float(),
                 positions=torch.randint(case["max_pos"], (t,), generator=g, device=dev).int(),
                 slots=torch.randperm(pages * p, generator=g, device=dev)[:t],
                 k_pages=randn(pages, hkv, p, d, dtype=dt), v_pages=randn(pages, hkv, p, d, dtype=dt),
                 q_norm=1 + randn(d, scale=0.2).to(dt) if case["norm"] else None,
                 k_norm=1 + randn(d, scale=0.2).to(dt) if case["norm"] else None)
    elif case["op"] == "attention":
        n, d, dt, p = _lengths(case), case["dim"], DTYPES[case["dtype"]], case["page"]
        held = [_ceil(c, p) for c in n]
        pages, width = sum(held) + 2, max(held)
        tables = torch.zeros(len(n), width, dtype=torch.int32, device=dev)
        at = torch.arange(width, device=dev)[None] < torch.tensor(held, device=dev)[:, None]
        tables[at] = torch.randperm(pages, generator=g, device=dev)[:sum(held)].int()
        s.update(q=randn(len(n), case["q_heads"], d, dtype=dt), tables=tables,
                 lengths=torch.tensor(n, dtype=torch.int32, device=dev),
                 k_pages=torch.randn(pages, case["kv_heads"], p, d, generator=g, device=dev, dtype=dt),
                 v_pages=torch.randn(pages, case["kv_heads"], p, d, generator=g, device=dev, dtype=dt))
    else:
        t, v = case["rows"], case["vocab"]
        logits = torch.randn(t, v, generator=g, device=dev, dtype=DTYPES[case["dtype"]])
        logits *= 2.5
        # a few likely tokens in each row, as a model gives
        hot = torch.randint(v, (t, 12), generator=g, device=dev)
        logits.scatter_add_(1, hot, (torch.rand(t, 12, generator=g, device=dev) * 9).to(logits.dtype))
        start = case["shard"] * v
        own_tokens = torch.randint(v, (t,), generator=g, device=dev) + start
        if start:  # a shard of the vocabulary: some tokens lie in another one
            far = torch.randint(8 * v, (t,), generator=g, device=dev)
            own_tokens = torch.where(torch.rand(t, generator=g, device=dev) < 0.3, far, own_tokens)
        s.update(logits=logits, tokens=own_tokens, start=start)
    return s


# --------------------------------------------------------- the plain form --
def _pages(s):
    c, starts, p = s["cached"].long(), s["starts"].long(), s["case"]["page"]
    width, n_free = s["tables"].shape[1], s["free"].numel()
    end = c + starts[1:] - starts[:-1]
    old = ((c + p - 1) // p).clamp(max=width)
    need = ((end + p - 1) // p).clamp(max=width) - old
    ahead = need.cumsum(0) - need
    j = torch.arange(width, device=c.device)[None] - old[:, None]
    at = s["taken"].long() + ahead[:, None] + j
    page = torch.where(at < n_free, s["free"][at.clamp(0, n_free - 1)], -1)
    tables = torch.where((j >= 0) & (j < need[:, None]), page, s["tables"])
    got = torch.minimum((n_free - s["taken"].long() - ahead).clamp(min=0), need)
    lengths = torch.minimum(end, (old + got) * p).int()
    taken = (s["taken"] + need.sum()).clamp(max=n_free).int()
    t = torch.arange(s["rows"], device=c.device)
    live = t < starts[-1]
    b = (torch.searchsorted(starts, t, right=True) - 1).clamp(max=c.numel() - 1)
    pos = torch.where(live, c[b] + t - starts[b], 0)
    held = tables[b, (pos // p).clamp(max=width - 1)].long()
    slots = torch.where(live & (pos // p < width) & (held >= 0), held * p + pos % p, -1)
    return pos.int(), slots, lengths, taken, tables


def _rms(x, w):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()


def _rotate(x, cos, sin, rotary, interleaved):
    r, rest = x[..., :rotary], x[..., rotary:]
    cos, sin = cos[:, None], sin[:, None]
    if interleaved:
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = r[..., :rotary // 2], r[..., rotary // 2:]
        r = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([r, rest], -1)


def _append(s):
    c = s["case"]
    hq, hkv, p = c["q_heads"], c["kv_heads"], c["page"]
    x = s["qkv"].float().view(c["tokens"], hq + 2 * hkv, c["dim"])
    q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
    if c["norm"]:
        q, k = _rms(q, s["q_norm"]), _rms(k, s["k_norm"])
    pos = s["positions"].long()
    cos, sin = s["cos"][pos], s["sin"][pos]
    q = _rotate(q, cos, sin, c["rotary"], c["interleaved"])
    k = _rotate(k, cos, sin, c["rotary"], c["interleaved"])
    s["k_pages"][s["slots"] // p, :, s["slots"] % p] = k.to(s["qkv"].dtype)
    s["v_pages"][s["slots"] // p, :, s["slots"] % p] = v.to(s["qkv"].dtype)
    return q.to(s["qkv"].dtype), s["k_pages"], s["v_pages"]


def _attention(s):
    c = s["case"]
    b, hkv, d = c["batch"], c["kv_heads"], c["dim"]
    used = s["tables"].long()
    # [batch, kv head, position, dim] of every table entry, in 32 bits
    k = s["k_pages"][used].float().transpose(1, 2).reshape(b, hkv, -1, d)
    live = torch.arange(k.shape[2], device=k.device)[None] < s["lengths"][:, None]
    q = s["q"].float().view(b, hkv, -1, d)
    x = torch.matmul(q, k.transpose(2, 3)) / math.sqrt(d)
    del k
    x = x.masked_fill(~live[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    e = torch.exp(x - top)
    total = e.sum(-1, keepdim=True)
    w = e / torch.where(total > 0, total, 1)
    v = s["v_pages"][used].float().transpose(1, 2).reshape(b, hkv, -1, d)
    v = v.masked_fill(~live[:, None, :, None], 0)
    return torch.matmul(w, v).view(b, c["q_heads"], d).to(s["q"].dtype)


def _logprobs(s):
    x, k = s["logits"].float(), s["case"]["top"]
    v = x.shape[1]
    top = x.amax(-1, keepdim=True)
    y = x - top
    e = torch.exp(y)
    total = e.sum(-1)
    log_total = torch.log(total)
    lse = top[:, 0] + log_total
    entropy = log_total - (e * y).sum(-1) / total
    at = s["tokens"] - s["start"]
    here = (at >= 0) & (at < v)
    picked = y.gather(1, at.clamp(0, v - 1)[:, None])[:, 0] - log_total
    picked = torch.where(here, picked, -math.inf)
    # order by value, then by the lowest index: one whole number for both
    bits = x.view(torch.int32)
    key = torch.where(bits < 0, bits ^ 0x7fffffff, bits).long() * (1 << 32) + (v - 1 - torch.arange(v, device=x.device))
    best = v - 1 - (key.topk(k, dim=-1).values & 0xffffffff)
    return picked, entropy, lse, y.gather(1, best) - log_total[:, None], best + s["start"]


PLAIN = {"pages": _pages, "append": _append, "attention": _attention, "logprobs": _logprobs}


# ------------------------------------------------------- this package's calls --
def _own_pages(s):
    import numa_allreduce_b200 as nab

    r = nab.assign_pages(s["cached"], s["tables"], s["free"], s["taken"], s["case"]["page"], query_start=s["starts"],
                         num_tokens=s["rows"])
    return r.positions, r.slots, r.lengths, r.taken, s["tables"]


def _own_append(s):
    import numa_allreduce_b200 as nab

    q = nab.rope_append_paged(s["qkv"], s["cos"], s["sin"], s["positions"], s["slots"], s["k_pages"], s["v_pages"],
                              s["case"]["q_heads"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS,
                              interleaved=s["case"]["interleaved"])
    return q, s["k_pages"], s["v_pages"]


def _own_attention(s):
    import numa_allreduce_b200 as nab

    return nab.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["tables"], s["lengths"])


def _own_logprobs(s):
    import numa_allreduce_b200 as nab

    r = nab.token_logprobs(s["logits"], s["tokens"], top_k=s["case"]["top"], vocab_start=s["start"])
    return r.logprob, r.entropy, r.lse, r.top_logprobs, r.top_tokens


OWN = {"pages": _own_pages, "append": _own_append, "attention": _own_attention, "logprobs": _own_logprobs}


def run(state):
    return (OWN if own else PLAIN)[state["case"]["op"]](state)


# ------------------------------------------------------------- in 64 bits --
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "pages":
        return None  # whole numbers: compared as they are
    if case["op"] == "append":
        hq, hkv, r = case["q_heads"], case["kv_heads"], case["rotary"]
        x = s["qkv"].double().reshape(case["tokens"], hq + 2 * hkv, case["dim"])
        heads = []
        for part, w in ((x[:, :hq], s["q_norm"]), (x[:, hq:hq + hkv], s["k_norm"])):
            if w is not None:
                part = part / part.square().mean(-1, keepdim=True).add(EPS).sqrt() * w.double()
            # the pairs as complex numbers, turned by the table's angle
            turn = torch.complex(s["cos"].double(), s["sin"].double())[s["positions"].long()][:, None]
            if case["interleaved"]:
                z = torch.complex(part[..., 0:r:2].contiguous(), part[..., 1:r:2].contiguous()) * turn
                rotated = torch.view_as_real(z).reshape(*part.shape[:2], r)
            else:
                z = torch.complex(part[..., :r // 2].contiguous(), part[..., r // 2:r].contiguous()) * turn
                rotated = torch.cat([z.real, z.imag], -1)
            heads.append(torch.cat([rotated, part[..., r:]], -1))
        page, row = s["slots"] // case["page"], s["slots"] % case["page"]
        k_pages, v_pages = s["k_pages"].double(), s["v_pages"].double()
        k_pages[page, :, row] = heads[1]
        v_pages[page, :, row] = x[:, hq + hkv:]
        return heads[0], k_pages, v_pages
    if case["op"] == "attention":
        g = case["q_heads"] // case["kv_heads"]
        out = torch.zeros_like(s["q"], dtype=torch.float64)
        for b, n in enumerate(_lengths(case)):
            if n == 0:
                continue
            ids = s["tables"][b, :_ceil(n, case["page"])].long()
            k, v = (t[ids].permute(1, 0, 2, 3).reshape(case["kv_heads"], -1, case["dim"])[:, :n].double()
                    for t in (s["k_pages"], s["v_pages"]))
            q = s["q"][b].double().reshape(case["kv_heads"], g, case["dim"])
            w = torch.einsum("hgd,hnd->hgn", q, k).div(math.sqrt(case["dim"])).softmax(-1)
            out[b] = torch.einsum("hgn,hnd->hgd", w, v).reshape(case["q_heads"], case["dim"])
        return out
    picked, entropy, lse, tops, ids = [], [], [], [], []
    for t in range(0, case["rows"], 64):
        x = s["logits"][t:t + 64].double()
        total = x.logsumexp(-1, keepdim=True)
        lp = x - total
        at = s["tokens"][t:t + 64] - s["start"]
        inside = (at >= 0) & (at < case["vocab"])
        chosen = lp.gather(1, torch.where(inside, at, 0)[:, None])[:, 0]
        chosen[~inside] = -math.inf
        picked.append(chosen)
        entropy.append(-(lp.exp() * lp).sum(-1))
        lse.append(total[:, 0])
        value, index = lp.sort(dim=-1, descending=True, stable=True)
        tops.append(value[:, :case["top"]])
        ids.append(index[:, :case["top"]] + s["start"])
    return torch.cat(picked), torch.cat(entropy), torch.cat(lse), torch.cat(tops), torch.cat(ids)
