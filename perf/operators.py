"""The attention, cache and sampling operators: cases, plain forms in elementary torch operations, and the framework's calls.

Four operators of a serving step over several sequences, each a "do" of a case:

* ``append``  rows of new keys and values into the pages of a cache
* ``prompt``  causal attention over packed prompts (``"pages": 0``) or over a cache's pages for a chunk of a prompt (a page size)
* ``decode``  attention of one new token for each sequence over a cache's pages
* ``sample``  a token for each row of logits, from given random numbers

``run`` computes them in their plain form where ``own`` is false and calls ``fastllama_amd.ops`` where it is true.
"""
import math
import random

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _ints(text):
    return [int(x) for x in text.split(",")]


def _text(values):
    return ",".join(str(v) for v in values)


def _spread(rng, n, lo, hi):
    """n whole numbers of lo..hi, spread over their logarithm."""
    return [min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))) for _ in range(n)]


def listed():
    ragged = _spread(random.Random(64), 62, 1, 4096) + [4096, 1]
    return [
        # a short prompt at the width of the tests' smallest model, in the framework's own activations' type: all latency
        {"name": "prompt-37-f32", "do": "prompt", "type": "f32", "heads": 4, "kv_heads": 4, "dim": 32, "q": "37", "kv": "37", "pages": 0},
        # one n_batch of a 7B prompt behind 1536 cached positions, n_ctx 2048, read from the cache's pages
        {"name": "prompt-chunk-512-at-1536", "do": "prompt", "type": "f16", "heads": 32, "kv_heads": 32, "dim": 128, "q": "512", "kv": "2048", "pages": 32},
        # prompts of several users in one call, lengths as they come, grouped heads
        {"name": "prompt-packed-8", "do": "prompt", "type": "bf16", "heads": 32, "kv_heads": 8, "dim": 128, "q": "1,700,33,1500,2,817,260,783",
         "kv": "1,700,33,1500,2,817,260,783", "pages": 0},
        # a long document: the matrix units' rate
        {"name": "prompt-8192", "do": "prompt", "type": "bf16", "heads": 32, "kv_heads": 8, "dim": 128, "q": "8192", "kv": "8192", "pages": 0},
        # one user early in a 7B chat, a cache in the framework's own type: latency
        {"name": "decode-1x300-f32", "do": "decode", "type": "f32", "heads": 32, "kv_heads": 32, "dim": 128, "kv": "300", "pages": 16},
        # one user behind a long document: few rows, a long axis
        {"name": "decode-1x32768", "do": "decode", "type": "bf16", "heads": 32, "kv_heads": 8, "dim": 128, "kv": "32768", "pages": 64},
        # a full batch of a 7B model at the end of its n_ctx, a head of keys for each head of queries
        {"name": "decode-16x2048", "do": "decode", "type": "f16", "heads": 32, "kv_heads": 32, "dim": 128, "kv": _text([2048 - 3 * i for i in range(16)]), "pages": 32},
        # a busy server: 64 users at lengths from 1 to 4096, grouped heads
        {"name": "decode-64-ragged", "do": "decode", "type": "f16", "heads": 32, "kv_heads": 8, "dim": 128, "kv": _text(ragged), "pages": 16},
        # the new rows of 64 users' tokens, f32 activations into an f16 cache
        {"name": "append-64x1", "do": "append", "type": "f16", "from": "f32", "kv_heads": 8, "dim": 128, "q": _text([1] * 64), "past": _text([n - 1 for n in ragged]), "pages": 16},
        # the rows of packed prompts of a 7B model
        {"name": "append-4000", "do": "append", "type": "bf16", "from": "bf16", "kv_heads": 32, "dim": 128, "q": "1800,77,1,2000,122", "past": "0,0,5,48,1029", "pages": 64},
        # one user's next token, LLaMA's vocabulary and usual settings: latency
        {"name": "sample-1x32000", "do": "sample", "type": "f32", "rows": 1, "vocab": 32000, "mode": "usual"},
        # a busy server with a large vocabulary and each user's own settings
        {"name": "sample-128x128256", "do": "sample", "type": "f32", "rows": 128, "vocab": 128256, "mode": "mixed"},
    ]


def draw(rng):
    do = rng.choice(["prompt", "prompt", "decode", "decode", "append", "sample"])
    kind = rng.choice(["f32", "f16", "bf16"])
    dim = rng.choice([32, 64, 80, 128, 128, 128])
    kv_heads = rng.choice([1, 2, 4, 8, 8, 32])
    heads = kv_heads * (1 if kv_heads == 32 else rng.choice([1, 2, 4, 5, 8]))
    pages = rng.choice([16, 32, 64, 256])
    if do == "prompt":
        total = _spread(rng, 1, 16, 1500 if kind == "f32" else 5000)[0]
        q = []
        while sum(q) < total:
            q += _spread(rng, 1, 1, total - sum(q))
        q = q[:48]
        past = [0] * len(q)
        if rng.random() < 0.4:  # chunks behind what is cached
            past = [rng.choice([0, rng.randrange(1, 2000)]) if i < 4 else 0 for i in range(len(q))]
        return {"do": do, "type": kind, "heads": min(heads, 40), "kv_heads": kv_heads if heads <= 40 else min(40, heads), "dim": dim, "q": _text(q),
                "kv": _text([a + b for a, b in zip(q, past)]), "pages": rng.choice([0, 0, pages])}
    if do == "decode":
        n = _spread(rng, 1, 1, 64)[0]
        return {"do": do, "type": kind, "heads": heads, "kv_heads": kv_heads, "dim": dim, "kv": _text(_spread(rng, n, 1, 32768 // (1 + n // 2))), "pages": pages}
    if do == "append":
        n = _spread(rng, 1, 1, 64)[0]
        return {"do": do, "type": kind, "from": rng.choice([kind, "f32"]), "kv_heads": kv_heads, "dim": dim, "q": _text(_spread(rng, n, 1, 1 + 3000 // n)),
                "past": _text([rng.randrange(0, 1000) for _ in range(n)]), "pages": pages}
    return {"do": do, "type": kind, "rows": _spread(rng, 1, 1, 128)[0], "vocab": _spread(rng, 1, 300, 131072)[0], "mode": rng.choice(["usual", "mixed", "plain"])}


def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)


def _starts(lengths):
    return [0] + np.cumsum(lengths).tolist()


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _tables(gen, lengths, page):
    """Pages in no order: (table [sequences, most pages], pages in the cache). Places behind a sequence's last page hold -1."""
    need = [(n + page - 1) // page for n in lengths]
    total = sum(need) + 3
    order = torch.randperm(total, generator=gen, device="cuda").tolist()
    most, at, rows = max(1, max(need)), 0, []
    for n in need:
        rows.append(order[at:at + n] + [-1] * (most - n))
        at += n
    return _i32(rows), total


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    s = dict(case)
    kind = TYPES[case["type"]]
    if case["do"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        # probabilities fall with the rank about as in a language model; a few tokens are banned
        rank = torch.argsort(torch.rand((rows, vocab), generator=gen, device="cuda"), dim=1).float()
        x = 12.0 - 1.15 * torch.log1p(rank) + 0.5 * _randn(gen, rows, vocab)
        x[torch.rand((rows, vocab), generator=gen, device="cuda") < 0.01] = float("-inf")
        s["logits"] = x.to(kind)
        s["u"] = torch.rand(rows, generator=gen, device="cuda")
        s["temperature"], s["top_k"], s["top_p"], s["min_p"] = 0.8, 40, 0.95, 0.0
        if case["mode"] == "plain":
            s["temperature"], s["top_k"], s["top_p"], s["min_p"] = 1.0, 0, 1.0, 0.0
        if case["mode"] == "mixed":  # each row's own settings: some greedy, some with one of the cuts, some with all
            pick = lambda *v: torch.tensor(v, device="cuda")[torch.randint(0, len(v), (rows,), generator=gen, device="cuda")]  # noqa: E731
            s["temperature"] = pick(0.0, 0.7, 0.8, 1.0, 1.0, 1.3)
            s["top_k"] = pick(0, 0, 1, 40, 200, 5000).int()
            s["top_p"] = pick(1.0, 1.0, 0.95, 0.9, 0.5)
            s["min_p"] = pick(0.0, 0.0, 0.02, 0.1)
        return s
    dim, kv_heads = case["dim"], case["kv_heads"]
    offset = 0.4 * _randn(gen, 1, kv_heads, dim)  # keys and values stand off zero by channel, as in trained models
    if case["do"] == "append":
        q, past = _ints(case["q"]), _ints(case["past"])
        s["table"], pages = _tables(gen, [a + b for a, b in zip(q, past)], case["pages"])
        s["k"], s["v"] = ((_randn(gen, sum(q), kv_heads, dim) + offset).to(TYPES[case["from"]]) for _ in range(2))
        s["n_past"], s["cu"] = _i32(past), _i32(_starts(q))
        s["k_pages"], s["v_pages"] = (_randn(gen, pages, kv_heads, case["pages"], dim).to(kind) for _ in range(2))
        return s
    kv = _ints(case["kv"])
    q = _ints(case["q"]) if case["do"] == "prompt" else [1] * len(kv)
    s["q"] = (1.5 * _randn(gen, sum(q), case["heads"], dim)).to(kind)
    s["cu_q"], s["cu_kv"], s["kv_len"] = _i32(_starts(q)), _i32(_starts(kv)), _i32(kv)
    if case["pages"]:
        s["table"], pages = _tables(gen, kv, case["pages"])
        s["k_pages"], s["v_pages"] = ((_randn(gen, pages, kv_heads, case["pages"], dim) + offset.view(1, kv_heads, 1, dim)).to(kind) for _ in range(2))
    else:
        s["k"], s["v"] = ((_randn(gen, sum(kv), kv_heads, dim) + offset).to(kind) for _ in range(2))
    return s


def _rows_of_pages(pages, table, kv_len):
    """The keys or values of all sequences, packed [sum of kv_len, kv heads, dim], from the pages [pages, kv heads, page, dim]."""
    n, _, page, _ = pages.shape
    at = torch.arange(table.shape[1] * page, device=pages.device)
    inside = at[None, :] < kv_len[:, None]
    seq, pos = inside.nonzero(as_tuple=True)
    return pages[table[seq, pos // page].long(), :, pos % page]


def _plain_attention(q, k, v, cu_q, cu_kv, scale):
    """Softmax over each query's visible keys of its own sequence; packed rows, 32 bits."""
    heads, kv_heads = q.shape[1], k.shape[1]
    q, k, v = (x.float().transpose(0, 1).contiguous() for x in (q, k, v))
    rows, keys = torch.arange(q.shape[1], device=q.device), torch.arange(k.shape[1], device=q.device)
    seq_q, seq_k = torch.searchsorted(cu_q[1:], rows, right=True), torch.searchsorted(cu_kv[1:], keys, right=True)
    last = cu_kv[1:][seq_q] - cu_q[1:][seq_q] + rows  # the last key that a row sees: the ends of queries and keys stand together
    seen = (seq_q[:, None] == seq_k[None, :]) & (keys[None, :] <= last[:, None])
    s = (q.view(kv_heads, heads // kv_heads * q.shape[1], -1) @ k.transpose(1, 2).contiguous()).view(heads, q.shape[1], -1) * scale
    s = s.masked_fill_(~seen, float("-inf"))
    p = torch.exp(s.sub_(s.amax(-1, keepdim=True)))
    p /= p.sum(-1, keepdim=True)
    out = p.view(kv_heads, heads // kv_heads * q.shape[1], -1) @ v
    return out.view(heads, q.shape[1], -1).transpose(0, 1)


def _plain_decode(q, k_pages, v_pages, table, kv_len, scale):
    """As above for one query of each sequence: padded to the longest, 32 bits."""
    n, page = table.shape[0], k_pages.shape[2]
    seen = torch.arange(table.shape[1] * page, device=q.device)[None, :] < kv_len[:, None]
    at = table.clamp_min(0).long()
    k, v = (x[at].float().permute(0, 2, 1, 3, 4).reshape(n, x.shape[1], -1, x.shape[3]) for x in (k_pages, v_pages))
    q = q.float().view(n, k.shape[1], -1, q.shape[2])
    s = (q @ k.transpose(2, 3).contiguous()) * scale
    s = s.masked_fill_(~seen[:, None, None, :], float("-inf"))
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    return (p @ v).reshape(n, -1, q.shape[3])


def _column(x, like):
    return x.double()[:, None] if torch.is_tensor(x) else torch.full((like.shape[0], 1), float(np.float32(x)), dtype=torch.float64, device=like.device)


def _plain_sample(logits, u, temperature, top_k, top_p, min_p):
    """64 bits: a token near a border of the sums would go the other way in 32."""
    x, at = torch.sort(logits.double(), dim=1, descending=True, stable=True)
    t, k, p, m = (_column(v, x) for v in (temperature, top_k, top_p, min_p))
    place = torch.arange(x.shape[1], device=x.device)[None, :]
    w = torch.exp((x - x[:, :1]) / torch.where(t > 0, t, 1.0))
    w = torch.where((place < torch.where((k > 0) & (t > 0), k, torch.where(t > 0, float(x.shape[1]), 1.0))), w, 0.0)
    before = torch.cumsum(w, 1) - w
    keep = ((before < p * w.sum(1, keepdim=True)) | (p >= 1)) & (w >= m) & (w > 0)
    keep[:, 0] = True
    kept = torch.zeros_like(w).scatter_(1, at, torch.where(keep, w, 0.0))  # back in the order of the tokens
    total = torch.cumsum(kept, 1)
    return (total <= u.double()[:, None] * total[:, -1:]).sum(1).int()


def _plain(s):
    if s["do"] == "sample":
        return _plain_sample(s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])
    if s["do"] == "append":
        rows = torch.arange(s["k"].shape[0], device="cuda")
        seq = torch.searchsorted(s["cu"][1:], rows, right=True)
        pos = s["n_past"][seq] + rows - s["cu"][seq]
        page = s["k_pages"].shape[2]
        at = s["table"][seq, pos // page].long()
        s["k_pages"][at, :, pos % page] = s["k"].to(s["k_pages"].dtype)
        s["v_pages"][at, :, pos % page] = s["v"].to(s["v_pages"].dtype)
        return s["k_pages"], s["v_pages"]
    scale = 1 / math.sqrt(s["dim"])
    if s["do"] == "decode":
        return _plain_decode(s["q"], s["k_pages"], s["v_pages"], s["table"], s["kv_len"], scale).to(s["q"].dtype)
    k, v = (_rows_of_pages(s[x], s["table"], s["kv_len"]) for x in ("k_pages", "v_pages")) if s["pages"] else (s["k"], s["v"])
    return _plain_attention(s["q"], k, v, s["cu_q"], s["cu_kv"], scale).to(s["q"].dtype)


def _own(s):
    from fastllama_amd import ops
    if s["do"] == "sample":
        return ops.sample(s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])
    if s["do"] == "prompt" and not s["pages"]:
        return ops.attn_prompt(s["q"], s["k"], s["v"], s["cu_q"], s["cu_kv"])
    if "cache" not in s:  # a view that a program keeps with its tensors
        s["cache"] = ops.KVPages(s["k_pages"], s["v_pages"])
    if s["do"] == "append":
        ops.kv_append(s["cache"], s["k"], s["v"], s["table"], s["n_past"], s["cu"])
        return s["k_pages"], s["v_pages"]
    if s["do"] == "prompt":
        return ops.attn_pages(s["q"], s["cache"], s["table"], s["kv_len"], s["cu_q"])
    return ops.attn_pages(s["q"], s["cache"], s["table"], s["kv_len"])


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    if case["do"] == "sample":  # a subtraction, a scaling, an exponential of about ten steps and a sum for each logit
        size = 4 if case["type"] == "f32" else 2
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size + 28 * case["rows"], "flops": 13 * n}
    size = 4 if case["type"] == "f32" else 2
    if case["do"] == "append":
        n = 2 * sum(_ints(case["q"])) * case["kv_heads"] * case["dim"]
        return {"bytes": n * (size + (4 if case["from"] == "f32" else 2)), "flops": n}
    kv = _ints(case["kv"])
    q = _ints(case["q"]) if case["do"] == "prompt" else [1] * len(kv)
    pairs = sum(a * b - a * (a - 1) // 2 for a, b in zip(q, kv))
    return {"bytes": size * case["dim"] * 2 * (sum(q) * case["heads"] + sum(kv) * case["kv_heads"]), "flops": 4 * pairs * case["heads"] * case["dim"]}


def exact(case, seed):
    s = prepare(case, seed)
    if case["do"] == "append":  # copies: what a row becomes by one rounding, position by position
        q, past, page = _ints(case["q"]), _ints(case["past"]), case["pages"]
        table, k_pages, v_pages, first = s["table"].tolist(), s["k_pages"].clone(), s["v_pages"].clone(), 0
        for b, n in enumerate(q):
            for j in range(0, n):
                p, slot = divmod(past[b] + j, page)
                k_pages[table[b][p], :, slot].copy_(s["k"][first + j])
                v_pages[table[b][p], :, slot].copy_(s["v"][first + j])
            first += n
        return k_pages.double(), v_pages.double()
    if case["do"] == "sample":
        x, u = s["logits"].double().cpu().numpy(), s["u"].double().cpu().numpy()
        get = lambda v, r: float(v[r]) if torch.is_tensor(v) else float(np.float32(v))  # noqa: E731
        tokens = []
        for r, l in enumerate(x):
            t, k, p, m = (get(s[n], r) for n in ("temperature", "top_k", "top_p", "min_p"))
            order = np.lexsort((np.arange(l.size), -l))
            if t <= 0:
                tokens.append(int(order[0]))
                continue
            w = np.exp((l[order] - l[order[0]]) / t)
            n = int(k) if 0 < k < l.size else l.size
            total = math.fsum(w[:n])
            if p < 1:
                n = min(n, int(np.searchsorted(np.cumsum(w[:n]), p * total)) + 1)
            n = max(1, min(n, int((w >= max(m, 1e-300)).sum())))
            kept = np.sort(order[:n])
            c = np.cumsum(np.exp((l[kept] - l[order[0]]) / t))
            tokens.append(int(kept[min(n - 1, int(np.searchsorted(c, u[r] * c[-1], side="right")))]))
        return torch.tensor(tokens, dtype=torch.int32)
    kv, group, dim = _ints(case["kv"]), case["heads"] // case["kv_heads"], case["dim"]
    q = _ints(case["q"]) if case["do"] == "prompt" else [1] * len(kv)
    out = torch.empty((sum(q), case["heads"], dim), dtype=torch.float64, device="cuda")
    at_q = at_k = 0
    for b, (lq, lk) in enumerate(zip(q, kv)):
        if case["pages"]:
            take = s["table"][b, :(lk + case["pages"] - 1) // case["pages"]].long()
            k, v = (s[x][take].permute(1, 0, 2, 3).reshape(case["kv_heads"], -1, dim)[:, :lk].double() for x in ("k_pages", "v_pages"))
        else:
            k, v = (s[x][at_k:at_k + lk].permute(1, 0, 2).double() for x in ("k", "v"))
        hidden = torch.ones((lq, lk), dtype=torch.bool, device="cuda").triu(lk - lq + 1)
        for h in range(case["heads"]):
            score = torch.mm(s["q"][at_q:at_q + lq, h].double(), k[h // group].t().contiguous()) / math.sqrt(dim)
            out[at_q:at_q + lq, h] = torch.mm(torch.softmax(score.masked_fill(hidden, -math.inf), dim=1), v[h // group].contiguous())
        at_q, at_k = at_q + lq, at_k + lk
    return out
