"""GPU: forms of the operators over several sequences that are chosen for large problems only: 16-bit prompts of many rows (workgroups of 128 and 256 rows),
sampling with parts of several rounds and with candidate lists that overflow.  Oracles and bounds: test_serve_ops_gpu.py."""
import math

import numpy as np
import pytest
import torch

from test_serve_ops_gpu import BF16, F16, F32, TYPES, attention64, check_prompt, i32, logits_like, near, ops, randn, sample64, scatter, starts  # noqa: F401

pytestmark = pytest.mark.gpu

LENS = [1, 255, 0, 257, 31, 33, 128, 129]
# Heads and keys heads such that a key head's rows make (rows / 128 + sequences) * key heads >= 512: one wave has 32 rows, a workgroup 128.
HEADS = [(64, 64), (192, 64), (320, 64)]


@pytest.mark.parametrize("T", [F16, BF16])
@pytest.mark.parametrize("D", [32, 64, 80, 128])
@pytest.mark.parametrize("H,Hkv", HEADS)
@pytest.mark.parametrize("pages", [0, 16, 64])
def test_prompt_many_rows(ops, T, D, H, Hkv, pages):
    assert (sum(LENS) * (H // Hkv) // 128 + len(LENS)) * Hkv >= 512
    check_prompt(ops, T, H, Hkv, D, LENS, LENS if D != 64 else [n + 70 if n % 2 else n for n in LENS], seed=D + H, pages=pages)


@pytest.mark.parametrize("T", [F16, BF16])
@pytest.mark.parametrize("D", [72, 128])
@pytest.mark.parametrize("H,Hkv,lens", [(256, 256, [1, 255, 257, 0, 40]), (512, 128, [1, 64, 65, 130]), (520, 104, [300, 1, 3])])
def test_prompt_many_rows_of_many_heads(ops, T, D, H, Hkv, lens):
    check_prompt(ops, T, H, Hkv, D, lens, lens, seed=D)
    check_prompt(ops, T, H, Hkv, D, lens, [n + 77 for n in lens], seed=D + 1)


LONG = [(256, 256, [300, 1, 257], [2200, 2500, 2100]), (2048, 128, [64], [2048]), (320, 64, [450, 0, 30], [4000, 100, 2300])]


@pytest.mark.parametrize("T", [F16, BF16])
@pytest.mark.parametrize("D", [72, 128])
@pytest.mark.parametrize("H,Hkv,lq,lk", LONG)
def test_prompt_workgroups_of_256_rows(ops, T, D, H, Hkv, lq, lk):
    """Many rows, 2048 keys a sequence and more."""
    assert sum(lq) * (H // Hkv) // 256 * Hkv >= 512 and sum(lk) // 2048 >= len(lq)
    check_prompt(ops, T, H, Hkv, D, lq, lk, seed=D)


@pytest.mark.parametrize("T", [F16, BF16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("at", [0, 5, 63, 64, 200, 299])
def test_prompt_workgroups_of_256_rows_not_finite(ops, T, bad, at):
    """A value that is not finite at the at-th new position of the first sequence: its rows from there on have it, nothing else does."""
    H, Hkv, lq, lk = LONG[0]
    q, k, v = randn(1, sum(lq), H, 128, dtype=T), randn(2, sum(lk), Hkv, 128, dtype=T), randn(3, sum(lk), Hkv, 128, dtype=T)
    want = [attention64(q[a:a + m], k[b:b + n], v[b:b + n], 128 ** -0.5) for a, b, m, n in zip(np.cumsum([0] + lq), np.cumsum([0] + lk), lq, lk)]
    v[lk[0] - lq[0] + at] = bad
    got = ops.attn_prompt(q, k, v, starts(lq), starts(lk)).split(lq)
    near(got[0][:at], want[0][0][:at], want[0][1][:at])
    seen = got[0][at:].double()
    assert (seen.isnan().all() if math.isnan(bad) else (seen == bad).all())
    for g, (w, b) in zip(got[1:], want[1:]):
        near(g, w, b)


@pytest.mark.parametrize("T", [F16, BF16])
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("Hkv,pages", [(64, 0), (64, 16), (256, 0)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_prompt_many_rows_not_finite(ops, T, D, Hkv, pages, bad):
    """A key (of head 0) and a value (of all heads) that are not finite, in one place of a sequence among others: the rows before it are as without it, those
    that see it have it, the other sequences do not."""
    lens = LENS if Hkv == 64 else [1, 255, 257, 0, 40]
    q, k, v = (randn(50 + i, sum(lens), Hkv, D, dtype=T) for i in range(3))
    for at in (0, 63, 64, 200):
        a = lens[0]                                            # the second sequence: 255 rows
        k2, v2 = k.clone(), v.clone()
        k2[a + at, 0], v2[a + at] = bad, bad
        if pages:
            cache, table = scatter(ops, k2, v2, lens, pages, 7)
            got = ops.attn_pages(q, cache, table, i32(lens), starts(lens))
        else:
            got = ops.attn_prompt(q, k2, v2, starts(lens))
        b = 0
        for i, n in enumerate(lens):
            want, bound = attention64(q[b:b + n], k[b:b + n], v[b:b + n], D ** -0.5)
            upto = at if i == 1 else n
            near(got[b:b + upto], want[:upto], bound[:upto], (i, at))
            b += n
        seen = got[a + at:a + 255, 1:].double()
        assert (seen.isnan().all() if math.isnan(bad) else (seen == bad).all())


# ------------------------------------------------------------------------------------------------ sampling
SETTINGS = [(1.0, 0, 1.0, 0.0), (0.8, 40, 0.95, 0.0), (0.7, 0, 0.9, 0.0), (1.3, 0, 1.0, 0.05), (0.0, 40, 0.5, 0.5), (1.0, 300, 0.5, 0.01), (2.0, 5000, 0.97, 0.0),
            (1.0, 9000, 1.0, 0.001), (3.0, 20000, 0.6, 0.0), (50.0, 0, 0.999, 0.0)]


def check_rows(ops, rows, V, T, settings, step):
    """Rows with the settings in turn; every step-th is checked against sorting."""
    l, u = logits_like(rows + V, rows, V, T), torch.rand(rows, generator=torch.Generator().manual_seed(V))
    f = lambda i: torch.tensor([settings[r % len(settings)][i] for r in range(rows)], dtype=F32, device="cuda")
    got = ops.sample(l, u.cuda(), f(0), f(1).int(), f(2), f(3)).tolist()
    for r in range(0, rows, step):
        assert got[r] == sample64(l[r].float().cpu().numpy(), u[r].item(), *settings[r % len(settings)]), (r, settings[r % len(settings)])


@pytest.mark.parametrize("T", TYPES)
@pytest.mark.parametrize("rows,V", [(200, 50257), (300, 40000), (350, 50257), (70, 262144)])
def test_sample_parts_of_several_rounds(ops, T, rows, V):
    check_rows(ops, rows, V, T, SETTINGS, 7)


@pytest.mark.parametrize("T", TYPES)
@pytest.mark.parametrize("rows,V", [(10, 32000), (260, 128256), (20, 9000)])
def test_sample_more_candidates_than_the_lists_hold(ops, T, rows, V):
    check_rows(ops, rows, V, T, [(1.0, 5000, 1.0, 0.0), (0.8, 5000, 0.95, 0.0), (2.0, 8500, 0.9, 0.001), (0.9, 4097, 1.0, 0.0), (1.0, 8999, 0.3, 0.0)], 13 if rows > 100 else 1)


def test_sample_all_rows_one_large_top_k(ops):
    l, u = logits_like(4, 4, 32000, F32), torch.rand(4, generator=torch.Generator().manual_seed(4))
    for k in (129, 4096, 4097, 5000, 31999, 32000):
        want = [sample64(l[r].cpu().numpy(), u[r].item(), 0.9, k, 0.95, 0.0) for r in range(4)]
        assert ops.sample(l, u.cuda(), 0.9, k, 0.95).tolist() == want, k


@pytest.mark.parametrize("T", [F32, BF16])
@pytest.mark.parametrize("V", [5, 5000])
def test_sample_temperatures_of_the_largest_size(ops, T, V):
    """Logits over all of the type's range, at temperatures beside which even their distances are small: each weighs something."""
    settings = [(t, k, p, m) for t in (math.inf, 3e38, 1e37, 1e33, 1e31) for k, p, m in ((0, 1.0, 0.0), (2, 1.0, 0.0), (0, 0.5, 0.0), (300, 0.9, 0.0), (0, 1.0, 0.3))]
    rows, rng = len(settings), np.random.default_rng(V)
    l = torch.from_numpy(rng.uniform(-3.3e38, 3.3e38, (rows, V)).astype(np.float32)).cuda().to(T)
    l[:, 1], l[:, 3] = -math.inf, torch.finfo(T).min
    u = torch.from_numpy(rng.random(rows).astype(np.float32))
    f = lambda i: torch.tensor([s[i] for s in settings], dtype=F32, device="cuda")
    got = ops.sample(l, u.cuda(), f(0), f(1).int(), f(2), f(3)).tolist()
    ln = l.double().cpu().numpy()

    def want(x, u, t, *cuts):                                # (-infinity / infinity is no number; distances of 1e-21 weigh 1 in 64 bits as well)
        return sample64(x * 1e-60, u, 1.0, *cuts) if t == math.inf else sample64(x, u, t, *cuts)
    assert got == [want(ln[r], u[r].item(), *settings[r]) for r in range(rows)]


# ------------------------------------------------------------------------------------------------ pages
@pytest.mark.parametrize("T", TYPES)
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("page", [16, 128])
def test_absent_pages_on_both_sides_of_the_range(ops, T, D, page):
    """Places behind a sequence's pages and holes among them hold -1, n_pages and 2^30 in turn, the lengths reach into them: those keys are absent."""
    lens, H, Hkv = [300, 40, 257], 4, 2
    k, v = (randn(i, sum(lens), Hkv, D, dtype=T) for i in (1, 2))
    cache, table = scatter(ops, k, v, lens, page, 3)
    n_pages, wide = cache.k.shape[0], max(lens) // page + 4
    absent = [-1, n_pages, 1 << 30]
    full = i32([[absent[(b + j) % 3] for j in range(wide)] for b in range(3)])
    for b, n in enumerate(lens):
        need = -(-n // page)
        full[b, :need] = table[b, :need]
    full[0, 1] = n_pages                                       # a hole
    there = [torch.tensor([i for i in range(n) if b or i // page != 1], device="cuda") for b, n in enumerate(lens)]
    # (the rest of a last page holds what is not finite: the lengths end with the page)
    long = [-(-n // page) * page + 3 * page for n in lens]
    for b, n in enumerate(lens):
        last = table[b, -(-n // page) - 1].item()
        if n % page:
            cache.k[last, :, n % page:], cache.v[last, :, n % page:] = 0.25, 0.5
    q = randn(5, 3, H, D, dtype=T)
    for cu in (None, i32([0, 1, 2, 3])):
        got, a = ops.attn_pages(q, cache, full, i32(long), cu), 0
        for b, n in enumerate(lens):
            rest = (-n) % page
            kb, vb = (torch.cat([x[a:a + n][there[b]], torch.full((rest, Hkv, D), y, dtype=T, device="cuda")]) for x, y in ((k, 0.25), (v, 0.5)))
            near(got[b:b + 1], *attention64(q[b:b + 1], kb, vb, D ** -0.5), (b, cu is None))
            a += n


# ------------------------------------------------------------------------------------------------ weights that f16 can hardly hold
def sinks(seed, rows, keys, H, Hkv, gap):
    """Every 32nd key outweighs the others by e^gap and has the value 0: what comes out is the others' share."""
    q, k, v = (torch.zeros(n, h, 64, device="cuda") for n, h in ((rows, H), (keys, Hkv), (keys, Hkv)))
    q[:, :, 0] = 1
    k[:, :, 0] = 0.05 * randn(seed, keys, Hkv)
    v += 256 + 16 * randn(seed + 1, keys, Hkv, 64)
    k[::32, :, 0], v[::32] = gap, 0
    return q.half(), k.half(), v.half()


@pytest.mark.parametrize("gap", [14.0, 18.0])
@pytest.mark.parametrize("rows,keys,H,Hkv,pages", [(1, 200, 2, 2, 16), (1, 5000, 4, 2, 64), (3, 5000, 2, 1, 0), (40, 300, 2, 2, 16), (300, 400, 128, 128, 0), (300, 400, 128, 128, 64)])
def test_small_weights_beside_large_ones_in_f16(ops, rows, keys, H, Hkv, pages, gap):
    """As attention64's bound, but for its term for p below f16's range: p is held as 2^7 p, its smallest step 2^-24, so half a step of it is 2^-32 (of a sum
    of 1 or more)."""
    q, k, v = sinks(1, rows, keys, H, Hkv, gap)
    want, bound = attention64(q, k, v, 1.0)
    s = torch.matmul(q.double().transpose(0, 1), k.double().repeat_interleave(H // Hkv, 1).permute(1, 2, 0).contiguous())
    seen = torch.arange(keys, device="cuda")[None, :] <= torch.arange(rows, device="cuda")[:, None] + (keys - rows)
    l = torch.where(seen, torch.exp(s - s.amax(-1, keepdim=True)), 0.0).sum(-1, keepdim=True)
    total = (seen.double() @ v.double().abs().repeat_interleave(H // Hkv, 1).transpose(0, 1).contiguous() / l).transpose(0, 1)
    bound = bound + (2.0 ** -32 - 2.0 ** -25) * total
    assert (bound < 0.1 * want).all()
    if pages:
        cache, table = scatter(ops, k, v, [keys], pages, 1)
        for cu in ([None] if rows == 1 else []) + [i32([0, rows])]:
            near(ops.attn_pages(q, cache, table, i32([keys]), cu, 1.0), want, bound)
    else:
        near(ops.attn_prompt(q, k, v, i32([0, rows]), i32([0, keys]), 1.0), want, bound)


# ------------------------------------------------------------------------------------------------ parts of a row that are joined
@pytest.mark.parametrize("T", TYPES)
@pytest.mark.parametrize("first,end", [(0, 4990), (1024, 2048), (0, 40), (2500, 2501)])
@pytest.mark.parametrize("form", ["decode", "pages", "prompt", "short"])
def test_keys_that_are_no_numbers_reach_the_rows_that_see_them(ops, T, first, end, form):
    """NaN in the keys of one key head, also in all keys that one wave, chunk or part has: its query heads become NaN, the others are as without."""
    keys, rows, H, Hkv, D = 5000 if form != "short" else 60, 1 if form == "decode" else 3, 4, 2, 64
    q, k, v = randn(1, rows, H, D, dtype=T), randn(2, keys, Hkv, D, dtype=T), randn(3, keys, Hkv, D, dtype=T)
    want, bound = attention64(q, k, v, D ** -0.5)
    first, end = (first, end) if form != "short" else (min(first, 31), min(end, 58))
    k[first:end, 0] = float("nan")
    if form in ("decode", "pages"):
        cache, table = scatter(ops, k, v, [keys], 64, 1)
        got = ops.attn_pages(q, cache, table, i32([keys]), None if form == "decode" else i32([0, rows]))
    else:
        got = ops.attn_prompt(q, k, v, i32([0, rows]), i32([0, keys]))
    assert got[:, :2].isnan().all()
    near(got[:, 2:], want[:, 2:], bound[:, 2:])


@pytest.mark.parametrize("T", TYPES)
@pytest.mark.parametrize("form", ["decode", "pages", "prompt"])
def test_an_infinite_value_of_no_weight_reaches_the_rows_that_see_it(ops, T, form):
    """A stretch of keys far below all others, one of their values infinite: its feature is not finite, the others are as without."""
    keys, rows, D = 5000, 1 if form == "decode" else 3, 64
    q, k, v = torch.ones((rows, 2, D), dtype=T, device="cuda"), randn(2, keys, 1, D, dtype=T, scale=0.1), randn(3, keys, 1, D, dtype=T)
    k[1024:2048] -= 25                                        # 64 * 25 / 8 = 200 below
    want, bound = attention64(q, k, v, D ** -0.5)
    v[1500, 0, 5] = float("inf")
    if form == "prompt":
        got = ops.attn_prompt(q, k, v, i32([0, rows]), i32([0, keys]))
    else:
        cache, table = scatter(ops, k, v, [keys], 64, 1)
        got = ops.attn_pages(q, cache, table, i32([keys]), None if form == "decode" else i32([0, rows]))
    assert not got[:, :, 5].isfinite().any()
    rest = [d for d in range(D) if d != 5]
    near(got[:, :, rest], want[:, :, rest], bound[:, :, rest])
