"""GPU: the operators over several sequences (paged cache, attention over prompts and pages, sampling) against plain 64-bit computations of their
formulas.  Tolerances are bounds of the arithmetic: attention64()."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [F32, F16, BF16]


@pytest.fixture(scope="module")
def ops():
    from fastllama_amd import hip, ops
    hip.require_device(0)
    return ops


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def starts(lens):
    return i32([0] + np.cumsum(lens).tolist())


def randn(seed, *shape, dtype=F32, scale=1.0):
    g = torch.Generator("cuda").manual_seed(seed)
    return (scale * torch.randn(shape, generator=g, device="cuda")).to(dtype)


def attention64(q, k, v, scale):
    """One sequence: q [lq, H, D], k, v [lk, Hkv, D] -> (out, bound) [lq, H, D] in 64 bits.  The bound of a kernel's error, for h = half a step of
    the type and u = 2^-24 (half a step of f32), with A = sum p |v| / sum p:
      rounding of the output            h |out| + its smallest step
      rounding of p before the product  h A in the 16-bit types, 2^-25 sum |v| / sum p where f16's p leave its range (p <= 2^-24; sum p >= 1)
      the score                         a chain of D products and two scalings: (D + 3) u S, S = the largest sum |q k| scale; p moves by e^that, up and
                                        down the fraction: 2 A of it
      the exponential and the sums      4 u (its argument's and its own step) (1 + S), and a chain of lk additions in both sums: 2 lk u, times A"""
    T, (lq, H, D), (lk, G) = q.dtype, q.shape, (k.shape[0], q.shape[1] // k.shape[1])
    q, k, v = (x.double().transpose(0, 1) for x in (q, k, v))
    k, v = k.repeat_interleave(G, 0), v.repeat_interleave(G, 0)
    seen = (torch.arange(lk, device="cuda")[None, :] <= torch.arange(lq, device="cuda")[:, None] + (lk - lq))[None]
    k, v0 = torch.nan_to_num(k, 0, 0, 0), torch.nan_to_num(v, 0, 0, 0)        # what is not finite stands in places that no row sees
    if lk == 0:
        z = torch.zeros((lq, H, D), dtype=torch.float64, device="cuda")
        return z, z
    s = (q @ k.transpose(1, 2).contiguous() * scale).masked_fill(~seen, -math.inf)
    p = torch.where(seen, torch.exp(s - s.amax(-1, keepdim=True).clamp_min(-1e300)), 0.0)
    l = p.sum(-1, keepdim=True).clamp_min(1e-300)
    out, A = p @ v0 / l, p @ v0.abs() / l
    S = ((q.abs() @ k.abs().transpose(1, 2).contiguous() * scale) * seen).amax(-1, keepdim=True)
    h, u = torch.finfo(T).eps / 2, 2.0 ** -24
    bound = h * out.abs() + torch.finfo(T).smallest_normal * (2.0 ** -10 if T == F16 else 1)
    bound = bound + A * (2 * (D + 3) * u * S + 4 * u * (1 + S) + 2 * lk * u + (0 if T == F32 else h))
    if T == F16:
        bound = bound + 2.0 ** -25 * (seen.double() @ v0.abs()) / l
    return out.transpose(0, 1), bound.transpose(0, 1)


def near(got, want, bound, what=""):
    off = (got.double() - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} outside; worst {float((off / bound.clamp_min(1e-30)).nan_to_num(9e9).max()):.3g} of the bound"


def check_prompt(ops, T, H, Hkv, D, lq, lk, seed=0, scale=None, pages=0):
    q, k, v = (randn(seed + i, n, h, D, dtype=T, scale=x) for i, (n, h, x) in enumerate(((sum(lq), H, 1.5), (sum(lk), Hkv, 1.0), (sum(lk), Hkv, 1.0))))
    if pages:
        cache, table = scatter(ops, k, v, lk, pages, seed)
        got = ops.attn_pages(q, cache, table, i32(lk), starts(lq), scale)
    else:
        got = ops.attn_prompt(q, k, v, starts(lq), starts(lk), scale)
    a = b = 0
    for m, n in zip(lq, lk):
        want, bound = attention64(q[a:a + m], k[b:b + n], v[b:b + n], D ** -0.5 if scale is None else scale)
        near(got[a:a + m], want, bound, (T, H, Hkv, D, m, n))
        a, b = a + m, b + n


def scatter(ops, k, v, lens, page, seed, spare=2, poison=float("nan"), order="phsd"):
    """A cache whose pages hold the packed k, v in shuffled places, `poison` everywhere else; places behind a sequence's pages name no page."""
    need = [-(-n // page) for n in lens]
    total, (Hkv, D) = sum(need) + spare, k.shape[1:]
    shape = dict(p=total, h=Hkv, s=page, d=D)
    base = [torch.full([shape[c] for c in order], poison, dtype=k.dtype, device="cuda") for _ in range(2)]
    kc, vc = (x.permute([order.index(c) for c in "phsd"]) for x in base)
    perm, at, row, tables = np.random.default_rng(seed).permutation(total).tolist(), 0, 0, []
    for n, m in zip(lens, need):
        mine = perm[at:at + m]
        at += m
        for i, pg in enumerate(mine):
            c = min(page, n - i * page)
            kc[pg, :, :c] = k[row + i * page:row + i * page + c].transpose(0, 1)
            vc[pg, :, :c] = v[row + i * page:row + i * page + c].transpose(0, 1)
        row += n
        tables.append(mine + [-1, 1 << 30][:1] * (max(1, max(need)) - m))
    return ops.KVPages(kc, vc), i32(tables)


# ------------------------------------------------------------------------------------------------ attention over prompts
@pytest.mark.parametrize("T", TYPES)
@pytest.mark.parametrize("H,Hkv,D", [(4, 4, 32), (8, 2, 128), (5, 1, 64), (6, 2, 8), (3, 3, 80), (2, 1, 120)])
def test_prompt_lengths_and_heads(ops, T, H, Hkv, D):
    lens = [1, 0, 37, 64, 65, 2, 130, 31, 33, 200]
    check_prompt(ops, T, H, Hkv, D, lens, lens, seed=H * D)


@pytest.mark.parametrize("T", TYPES)
@pytest.mark.parametrize("lq,lk", [([5, 64, 1, 3], [300, 64, 129, 1]), ([7, 0, 40], [0, 9, 17]), ([1], [1]), ([130], [257])])
@pytest.mark.parametrize("pages", [0, 16, 64, 128])
def test_prompt_rows_behind_a_past_and_rows_without_keys(ops, T, lq, lk, pages):
    check_prompt(ops, T, 4, 2, 64, lq, lk, seed=3, pages=pages)


@pytest.mark.parametrize("T", TYPES)
@pytest.mark.parametrize("n", [1000, 2050])
def test_prompt_long(ops, T, n):
    check_prompt(ops, T, 2, 1, 128, [n], [n], seed=n)
    check_prompt(ops, T, 2, 2, 128, [300], [n], seed=n, pages=32)


@pytest.mark.parametrize("T", TYPES)
@pytest.mark.parametrize("H,Hkv,lq,lk", [(2, 1, [3], [5000]), (8, 2, [16, 1, 0, 70], [9000, 3000, 700, 70]), (5, 5, [1, 1], [4096, 513]), (1, 1, [129], [2600])])
@pytest.mark.parametrize("pages", [0, 64])
def test_prompt_few_rows_behind_many_keys(ops, T, H, Hkv, lq, lk, pages):
    check_prompt(ops, T, H, Hkv, 64 if pages else 128, lq, lk, seed=H, pages=pages)


@pytest.mark.parametrize("T", TYPES)
@pytest.mark.parametrize("lk", [1100, 4300])
def test_prompt_a_workgroup_for_each_cu_behind_many_keys(ops, T, lk):
    check_prompt(ops, T, 28, 28, 64, [460 if T != F32 else 900], [lk], seed=lk, pages=64)


@pytest.mark.parametrize("T", TYPES)
def test_prompt_not_finite_behind_many_keys(ops, T):
    """As above for keys cut into parts: the last row's last key holds a value that is not finite, the rows before it do not see it."""
    q, k, v = randn(1, 4, 2, 64, dtype=T), randn(2, 4000, 1, 64, dtype=T), randn(3, 4000, 1, 64, dtype=T)
    want, bound = attention64(q, k, v, 0.125)
    v[-1] = float("nan")
    got = ops.attn_prompt(q, k, v, i32([0, 4]), i32([0, 4000]))
    near(got[:3], want[:3], bound[:3])
    assert got[3].isnan().all()


@pytest.mark.parametrize("T", TYPES)
@pytest.mark.parametrize("scale", [0.01, 2.0])
def test_prompt_flat_and_sharp_scores(ops, T, scale):
    check_prompt(ops, T, 2, 2, 128, [150, 70], [150, 200], seed=9, scale=scale)


@pytest.mark.parametrize("T", TYPES)
def test_prompt_rising_scores(ops, T):
    """Every key outweighs all before it: the running maximum moves on at every step, by far more than one rounding can hide."""
    n, D = 300, 64
    k = torch.arange(n, device="cuda", dtype=F32).view(n, 1, 1).expand(n, 1, D).to(T).contiguous()
    q = torch.full((n, 1, D), 0.25, device="cuda").to(T)
    v = randn(4, n, 1, D, dtype=T)
    got = ops.attn_prompt(q, k, v, starts([n]), scale=0.125)
    want, bound = attention64(q, k, v, 0.125)
    near(got, want, bound)
    near(ops.attn_prompt(q, -k, v, starts([n]), scale=0.125), *attention64(q, -k, v, 0.125))


def test_prompt_strides_of_one_fused_projection_and_heads_first(ops):
    """q, k, v as slices of one [rows, (H + 2 Hkv) D] product, the output heads-first; rows behind the last sequence stay."""
    H, Hkv, D, lens = 4, 2, 64, [19, 70]
    n = sum(lens)
    x = randn(5, n + 6, (H + 2 * Hkv) * D, dtype=BF16)
    q, k, v = (t.unflatten(1, (-1, D)) for t in x.split([H * D, Hkv * D, Hkv * D], 1))
    out = torch.full((H, n + 6, D), 7.0, dtype=BF16, device="cuda").transpose(0, 1)
    ops.attn_prompt(q, k, v, starts(lens), out=out)
    assert (out[n:] == 7).all()
    a = 0
    for m in lens:
        near(out[a:a + m], *attention64(q[a:a + m], k[a:a + m], v[a:a + m], D ** -0.5))
        a += m


@pytest.mark.parametrize("T", TYPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_prompt_what_a_row_may_not_see_cannot_touch_it(ops, T, bad):
    """Not-finite keys and values of later positions, of other sequences and between them."""
    H, D, n = 2, 64, 100
    q, k, v = (randn(20 + i, 3 * n, H, D, dtype=T) for i in range(3))
    for at in (40, 41, 77):
        k2, v2 = k.clone(), v.clone()
        k2[:n], v2[:n], k2[2 * n:], v2[2 * n:] = bad, bad, bad, bad
        k2[n + at, 0], v2[n + at] = bad, bad
        cu_q, cu_kv = i32([0, 0, n, n]), i32([0, n, 2 * n, 3 * n])
        got = ops.attn_prompt(q, k2, v2, cu_q, cu_kv)
        want, bound = attention64(q[:n], k[n:2 * n], v[n:2 * n], D ** -0.5)
        near(got[:at], want[:at], bound[:at], at)
        seen = got[at:n, 1].double()                      # head 1: finite scores, a value that is not
        assert (seen.isnan().all() if math.isnan(bad) else (seen == bad).all())


def test_prompt_row_starts_outside_the_rows_are_cut(ops):
    q, k, v = (randn(30 + i, 50, 2, 32, dtype=F16) for i in range(3))
    got = ops.attn_prompt(q, k, v, i32([-5, 20, 1 << 30]), i32([-9, 20, 1 << 30]))
    for a, b in ((0, 20), (20, 50)):
        near(got[a:b], *attention64(q[a:b], k[a:b], v[a:b], 32 ** -0.5))


def test_prompt_no_rows_no_keys_no_sequences(ops):
    q, none = randn(1, 5, 2, 32, dtype=F16), randn(1, 0, 2, 32, dtype=F16)
    assert (ops.attn_prompt(q, none, none, i32([0, 5]), i32([0, 0])) == 0).all()
    assert ops.attn_prompt(none, none, none, i32([0, 0])).shape == (0, 2, 32)
    out = torch.full_like(q, 3.0)
    ops.attn_prompt(q, q, q, i32([0]), out=out)
    assert (out == 3).all()


@pytest.mark.parametrize("T", [F16, F32])
def test_prompt_many_short_sequences(ops, T):
    lens = [(i * 7) % 5 for i in range(400)]
    check_prompt(ops, T, 2, 1, 32, lens, lens, seed=11)


# ------------------------------------------------------------------------------------------------ one new token over pages
def check_decode(ops, T, H, Hkv, D, lens, page, seed=0, order="phsd", scale=None):
    q = randn(seed, len(lens), H, D, dtype=T, scale=1.5)
    k, v = (randn(seed + i, sum(lens), Hkv, D, dtype=T) for i in (1, 2))
    cache, table = scatter(ops, k, v, lens, page, seed, order=order)
    got = ops.attn_pages(q, cache, table, i32(lens), scale=scale)
    a = 0
    for i, n in enumerate(lens):
        near(got[i:i + 1], *attention64(q[i:i + 1], k[a:a + n], v[a:a + n], D ** -0.5 if scale is None else scale), (T, H, Hkv, D, n, page))
        a += n


@pytest.mark.parametrize("T", TYPES)
@pytest.mark.parametrize("H,Hkv,D", [(4, 4, 32), (8, 1, 128), (15, 3, 64), (6, 2, 8), (3, 3, 80), (20, 1, 128), (40, 1, 64), (32, 2, 128)])
def test_decode_lengths_and_heads(ops, T, H, Hkv, D):
    check_decode(ops, T, H, Hkv, D, [1, 0, 15, 16, 17, 33, 300, 64, 2], 16, seed=H + D)


@pytest.mark.parametrize("T", TYPES)
@pytest.mark.parametrize("page", [16, 32, 64, 256, 1024])
@pytest.mark.parametrize("order", ["phsd", "pshd", "hpsd"])
def test_decode_page_sizes_and_layouts(ops, T, page, order):
    check_decode(ops, T, 8, 4, 128, [700, 3, 1025, 512], page, seed=page, order=order)


@pytest.mark.parametrize("T", TYPES)
@pytest.mark.parametrize("lens", [[5000], [9000, 1, 4096], [2048] * 3])
def test_decode_long(ops, T, lens):
    check_decode(ops, T, 4, 2, 128, lens, 64, seed=7)


@pytest.mark.parametrize("T", TYPES)
@pytest.mark.parametrize("scale", [0.01, 2.0])
def test_decode_flat_and_sharp_scores(ops, T, scale):
    check_decode(ops, T, 4, 4, 64, [3000, 40], 32, seed=8, scale=scale)


@pytest.mark.parametrize("cu", [False, True])
def test_pages_outside_the_cache_are_keys_that_are_not_there(ops, cu):
    """A page number below 0 or past the cache inside a sequence: its keys count as absent.  Lengths past the table are cut to it."""
    H, D, page, n = 4, 64, 16, 100
    q, k, v = randn(1, 3, H, D, dtype=F16), randn(2, 3 * n, H, D, dtype=F16), randn(3, 3 * n, H, D, dtype=F16)
    cache, table = scatter(ops, k, v, [n, n, n], page, 5)
    table[0, 2], table[0, 4], table[1, :] = -7, cache.k.shape[0], -1
    lens = i32([n, n, 112])
    cache.k[table[2, -1].item(), :, 4:] = 1.0              # the slots of the last page that n = 100 leaves unused
    cache.v[table[2, -1].item(), :, 4:] = 1.0
    huge = i32([n, -3, 1 << 30])
    for length in (lens, huge):
        got = ops.attn_pages(q, cache, table, length, i32([0, 1, 2, 3]) if cu else None)
        keep = torch.tensor([i for i in range(n) if i // page not in (2, 4)], device="cuda")
        near(got[0:1], *attention64(q[0:1], k[:n][keep], v[:n][keep], D ** -0.5))
        assert (got[1] == 0).all()
        one = torch.ones((12, H, D), dtype=F16, device="cuda")
        near(got[2:3], *attention64(q[2:3], torch.cat([k[2 * n:], one]), torch.cat([v[2 * n:], one]), D ** -0.5))


def test_decode_offsets_past_32_bits(ops):
    """A cache of more than 2^31 elements, the sequence in its last pages."""
    n_pages, page, Hkv, D = 40000, 64, 8, 128
    kc = torch.empty((n_pages, Hkv, page, D), dtype=F16, device="cuda")
    vc = torch.empty_like(kc)
    k, v = (randn(i, 200, Hkv, D, dtype=F16) for i in (1, 2))
    q = randn(3, 1, 16, D, dtype=F16)
    assert kc.numel() > 1 << 31
    cache, table = ops.KVPages(kc, vc), i32([[n_pages - 1, n_pages - 3, 17, n_pages - 2]])
    ops.kv_append(cache, k, v, table, i32([0]), i32([0, 200]))
    want = attention64(q, k, v, D ** -0.5)
    near(ops.attn_pages(q, cache, table, i32([200])), *want)
    near(ops.attn_pages(q, cache, table, i32([200]), i32([0, 1])), *want)


def test_decode_strided_queries_and_table(ops):
    H, D, lens = 4, 64, [40, 90]
    k, v = (randn(i, sum(lens), H, D, dtype=BF16) for i in (1, 2))
    cache, table = scatter(ops, k, v, lens, 16, 1)
    wide = torch.full((2, 50), -1, dtype=torch.int32, device="cuda")
    wide[:, 3:3 + table.shape[1]] = table
    q = randn(4, 2, 3 * H * D, dtype=BF16)[:, H * D:2 * H * D].unflatten(1, (H, D))
    got = ops.attn_pages(q, cache, wide[:, 3:3 + table.shape[1]], i32(lens))
    a = 0
    for i, n in enumerate(lens):
        near(got[i:i + 1], *attention64(q[i:i + 1], k[a:a + n], v[a:a + n], D ** -0.5))
        a += n


# ------------------------------------------------------------------------------------------------ append
@pytest.mark.parametrize("S,T", [(F32, F32), (F32, F16), (F32, BF16), (F16, F16), (BF16, BF16)])
@pytest.mark.parametrize("order", ["phsd", "pshd"])
def test_append(ops, S, T, order):
    lens, past, page, H, D = [1, 0, 37, 130, 16], [15, 4, 0, 100, 16], 16, 3, 40
    need = [-(-(a + b) // page) for a, b in zip(lens, past)]
    perm, rows, at = torch.randperm(sum(need) + 2).tolist(), [], 0
    for n in need:
        rows.append(perm[at:at + n] + [-1] * (max(need) - n))
        at += n
    shape = dict(p=sum(need) + 2, h=H, s=page, d=D)
    base = [randn(i, *[shape[c] for c in order], dtype=T) for i in (1, 2)]
    kc, vc = (x.permute([order.index(c) for c in "phsd"]) for x in base)
    wk, wv = kc.clone(), vc.clone()
    k, v = (randn(i, sum(lens) + 3, H, D, dtype=S) for i in (3, 4))
    r = 0
    for b, n in enumerate(lens):
        for j in range(n):
            p = past[b] + j
            wk[rows[b][p // page], :, p % page], wv[rows[b][p // page], :, p % page] = k[r].to(T), v[r].to(T)
            r += 1
    ops.kv_append(ops.KVPages(kc, vc), k, v, i32(rows), i32(past), starts(lens))   # (three rows behind the last sequence go nowhere)
    assert torch.equal(kc, wk) and torch.equal(vc, wv)


def test_append_one_row_each_and_places_that_are_not_there(ops):
    H, D, page = 2, 64, 16
    kc, vc = randn(1, 6, H, page, D, dtype=F16), randn(2, 6, H, page, D, dtype=F16)
    wk, wv = kc.clone(), vc.clone()
    k, v = randn(3, 6, H, D), randn(4, 6, H, D)
    table = i32([[0, 1], [2, -1], [6, 3], [4, 5], [4, 5], [-2147483648, 2147483647]])
    past = [17, 16, 3, 32, -1, 20]                        # only row 0 has a place: no page, no such page, past the table, before 0, no such page
    ops.kv_append(ops.KVPages(kc, vc), k, v, table, i32(past))
    wk[1, :, 1], wv[1, :, 1] = k[0].to(F16), v[0].to(F16)
    assert torch.equal(kc, wk) and torch.equal(vc, wv)


@pytest.mark.parametrize("T", [F16, BF16])
def test_append_rounds_to_nearest_even_and_keeps_what_is_not_finite(ops, T):
    h = torch.finfo(T).eps / 2
    x = torch.tensor([1 + h, 1 + 3 * h, 1 + h * 1.0001, float("inf"), -float("inf"), float("nan"), -0.0, 1e-8], device="cuda").view(1, 1, 8)
    cache = ops.KVPages.empty(1, 16, 1, 8, T)
    ops.kv_append(cache, x, -x, i32([[0]]), i32([5]))
    for got, want in ((cache.k[0, 0, 5], x[0, 0].to(T)), (cache.v[0, 0, 5], (-x[0, 0]).to(T))):
        fine = ~torch.isnan(want)
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(got.view(torch.int16)[fine], want.view(torch.int16)[fine])


# ------------------------------------------------------------------------------------------------ sampling
def sample64(l, u, T, k, p, m):
    """The formula for one row, in 64 bits, by sorting."""
    l = np.where(np.isnan(l), -np.inf, l.astype(np.float64))
    if not (l > -np.inf).any():
        return -1
    order = np.lexsort((np.arange(l.size), -l))
    if not T > 0:
        return int(order[0])
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(l == l.max(), 1.0, np.exp(np.where(l == l.max(), 0.0, l - l.max()) / np.float64(np.float32(T))))
    ws = w[order]
    n = min(int(k), l.size) if k > 0 else l.size
    if p < 1:
        n = min(n, int(np.searchsorted(np.cumsum(ws[:n]), np.float64(np.float32(p)) * math.fsum(ws[:n]))) + 1)
    if m > 0:
        n = min(n, int((ws >= min(1.0, float(np.float32(m)))).sum()))
    kept = np.sort(order[:max(1, n)])
    c = np.cumsum(w[kept])
    return int(kept[min(len(kept) - 1, int(np.searchsorted(c, np.float64(np.float32(u)) * c[-1], side="right")))])


def logits_like(seed, rows, V, T):
    rng = np.random.default_rng(seed)
    x = 12 - 1.15 * np.log1p(np.argsort(rng.random((rows, V)), 1)) + 0.5 * rng.standard_normal((rows, V))
    x[rng.random((rows, V)) < 0.02] = -np.inf
    return torch.from_numpy(x.astype(np.float32)).cuda().to(T)


SETTINGS = [(1.0, 0, 1.0, 0.0), (0.8, 40, 0.95, 0.0), (0.7, 0, 0.9, 0.0), (1.3, 0, 1.0, 0.05), (0.0, 40, 0.5, 0.5), (1.0, 1, 1.0, 0.0), (1.0, 300, 0.5, 0.01),
            (2.0, 0, 0.0, 0.0), (1.0, 1 << 30, 1.0, 1.0), (0.05, 5, 0.99, 0.3), (50.0, 0, 0.999, 0.0)]


@pytest.mark.parametrize("T", TYPES)
@pytest.mark.parametrize("V", [1, 2, 63, 512, 1000, 32000, 50257, 131071, 262144])
def test_sample_against_sorting(ops, T, V):
    """Equal tokens: a border of the 64-bit sums would have to be nearer than 2^-30 to a number of 24 bits for them to differ by rounding."""
    rows = len(SETTINGS)
    l = logits_like(V, rows, V, T)
    u = torch.rand(rows, generator=torch.Generator().manual_seed(V))
    ln = l.float().cpu().numpy()
    t, k, p, m = (list(c) for c in zip(*SETTINGS))
    f = lambda c: torch.tensor(c, dtype=F32, device="cuda")
    got = ops.sample(l, u.cuda(), f(t), i32(k), f(p), f(m)).tolist()
    want = [sample64(ln[r], u[r].item(), *SETTINGS[r]) for r in range(rows)]
    assert got == want
    for r, s in enumerate(SETTINGS[:4]):                  # the same as plain numbers, one row
        assert ops.sample(l[r:r + 1], u[r:r + 1].cuda(), *s).tolist() == [want[r]]


def test_sample_ties_and_borders(ops):
    inf, nan = float("inf"), float("nan")
    rows = [
        ([1.0, 1.0, 1.0, 1.0], 0.0, (1.0, 2, 1.0, 0.0), 0),          # of equals the lowest indexes are kept
        ([1.0, 1.0, 1.0, 1.0], 0.99, (1.0, 2, 1.0, 0.0), 1),
        ([1.0, 1.0, 1.0, 1.0], 0.5, (1.0, 0, 1.0, 0.0), 2),          # the running sum has to exceed u times the whole
        ([1.0, 1.0, 1.0, 1.0], 0.9, (1.0, 0, 0.5, 0.0), 1),          # a prefix whose sum equals top_p's share is long enough
        ([1.0, 1.0, 1.0, 1.0], 0.99, (1.0, 0, 0.51, 0.0), 2),
        ([-inf, -inf, -inf, -inf], 0.3, (1.0, 0, 1.0, 0.0), -1),
        ([nan, nan, -inf, nan], 0.3, (0.0, 0, 1.0, 0.0), -1),
        ([nan, 2.0, -inf, 1.0], 0.0, (0.0, 0, 1.0, 0.0), 1),
        ([nan, -inf, -3e38, -inf], 0.999, (1.0, 0, 1.0, 0.0), 2),
        ([inf, 5.0, inf, 1.0], 0.6, (1.0, 0, 1.0, 0.0), 2),          # infinities share the weight
        ([inf, 5.0, inf, 1.0], 0.6, (1.0, 1, 1.0, 0.0), 0),
        ([0.0, -0.0, 0.0, -1.0], 0.0, (0.0, 0, 1.0, 0.0), 0),        # -0 is 0
        ([-0.0, 0.0, -0.0, -1.0], 0.99, (1.0, 2, 1.0, 0.0), 1),
        ([3e38, -3e38, 0.0, 3e38], 0.75, (1e-30, 0, 1.0, 0.0), 3),
        ([0.0, 1.0, 2.0, 3.0], 1.0, (1.0, 0, 1.0, 0.0), 3),          # u outside [0, 1) goes to its end
        ([0.0, 1.0, 2.0, 3.0], nan, (1.0, 0, 1.0, 0.0), 0),
        ([0.0, 1.0, 2.0, 3.0], 0.0, (1.0, 0, 1.0, 2.0), 3),          # min_p past 1 keeps the largest
        ([3.0, 1.0, 3.0, 3.0], 0.4, (nan, 0, nan, nan), 0),          # no temperature: greedy
        ([3.0, 1.0, 3.0, 3.0], 0.4, (inf, 0, 1.0, 0.0), 1),          # all alike
    ]
    f = lambda c: torch.tensor(c, dtype=F32, device="cuda")
    t, k, p, m = zip(*(r[2] for r in rows))
    got = ops.sample(f([r[0] for r in rows]), f([r[1] for r in rows]), f(t), i32(k), f(p), f(m)).tolist()
    assert got == [r[3] for r in rows]


@pytest.mark.parametrize("V", [64, 40000])
def test_sample_all_logits_alike(ops, V):
    u = torch.linspace(0, 0.9999, 50, device="cuda")
    l = torch.full((50, V), 2.5, device="cuda")
    want = (u.double() * V).floor().int()
    assert torch.equal(ops.sample(l, u), want)
    assert torch.equal(ops.sample(l, u, top_k=10), (u.double() * 10).floor().int())
    assert torch.equal(ops.sample(l, u, top_p=0.25), (u.double() * (V // 4)).floor().int())


def test_sample_strided_rows_and_unaligned(ops):
    l = logits_like(5, 7, 1003, F16)
    u = torch.rand(7, device="cuda")
    want = ops.sample(l, u, 0.8, 40, 0.95)
    wide = torch.full((7, 1200), 99.0, dtype=F16, device="cuda")
    wide[:, 5:1008] = l
    assert torch.equal(ops.sample(wide[:, 5:1008], u, 0.8, 40, 0.95), want)


def test_sample_more_rows_than_one_launch_takes(ops):
    l = logits_like(9, 4500, 300, F32)
    u, t = torch.rand(4500, device="cuda"), torch.rand(4500, device="cuda") + 0.2
    k, p = torch.randint(0, 300, (4500,), device="cuda").int(), torch.rand(4500, device="cuda") + 0.3
    got = ops.sample(l, u, t, k, p, 0.01)
    for a in range(0, 4500, 900):
        b = slice(a, a + 900)
        assert torch.equal(got[b], ops.sample(l[b], u[b], t[b], k[b], p[b], 0.01))


def test_sample_follows_the_distribution(ops):
    """65536 evenly spaced u: each token comes up in its share of them, within the two ends of its stretch."""
    V, n = 50, 1 << 16
    l = logits_like(6, 1, V, F32)
    u = (torch.arange(n, device="cuda") + 0.5) / n
    got = torch.bincount(ops.sample(l.expand(n, V).contiguous(), u.float(), 0.9, 20, 0.9).long(), minlength=V).double()
    w = torch.softmax(l[0].double() / float(np.float32(0.9)), 0)
    order = torch.argsort(w, descending=True)[:20]
    c = torch.cumsum(w[order], 0)
    kept = order[:int((c < float(np.float32(0.9)) * c[-1]).sum()) + 1]
    share = torch.zeros(V, dtype=torch.float64, device="cuda")
    share[kept] = w[kept] / w[kept].sum() * n
    assert ((got - share).abs() <= 1.0).all()


def test_model_logits_sample(ops):
    """fl_model_logits_sample on a model's own logits = fl_sample on those logits."""
    import ctypes as C
    import oracle
    from fastllama_amd import hip
    from harness import ggjt
    from harness.flmodel import FlModel
    cfg = ggjt.TINY
    m = FlModel(cfg, oracle.Q4_0, ggjt.synth_tensors(cfg, oracle.Q4_0, oracle.Port().quantize_q4, seed=3), n_ctx=64, max_batch=32)
    logits = m.eval(ggjt.text_tokens("draw a token for each row")[:20], all_logits=True)
    n = len(logits)
    u = np.random.default_rng(1).random(n).astype(np.float32)
    L, got = hip.load(), np.full(n, -9, np.int32)
    p = hip.SampleParams(temperature=0.8, top_k=40, top_p=0.95, min_p=0.0)
    call = lambda row0, rows: L.fl_model_logits_sample(m.h, row0, rows, u[row0:].ctypes.data_as(C.c_void_p), C.byref(p), got[row0:].ctypes.data_as(C.c_void_p))
    hip.check(call(0, n))
    want = ops.sample(torch.from_numpy(logits).cuda(), torch.from_numpy(u).cuda(), 0.8, 40, 0.95).cpu().numpy()
    assert np.array_equal(got, want)
    got[:] = -9
    hip.check(call(5, 3))
    assert np.array_equal(got[5:8], want[5:8]) and (got[8:] == -9).all()
    assert call(0, 1 << 20) == hip.FL_EINVAL and call(n - 1, (1 << 31) - 1) == hip.FL_EINVAL


def test_python_entry_points_refuse(ops):
    """What the wrappers see on device tensors: shapes, types, strides and places that do not fit."""
    from fastllama_amd import hip
    d, host = torch.zeros(2, 2, 8, device="cuda"), torch.zeros(2, 2, 8)
    cu, table, lens = i32([0, 2]), i32([[0], [1]]), i32([3, 4])
    c = ops.KVPages.empty(4, 16, 2, 8, F32)
    l, u = torch.zeros(2, 50, device="cuda"), torch.zeros(2, device="cuda")
    ops.attn_prompt(d, d, d, cu), ops.attn_pages(d, c, table, lens), ops.kv_append(c, d, d, table, lens), ops.sample(l, u)
    for bad in (lambda: ops.attn_prompt(host, d, d, cu), lambda: ops.attn_prompt(d, d.half(), d.half(), cu), lambda: ops.attn_prompt(d[0], d, d, cu),
                lambda: ops.attn_prompt(d, d, d, cu.long()), lambda: ops.attn_prompt(d.double(), d.double(), d.double(), cu), lambda: ops.attn_prompt(d, d, d, cu.cpu()),
                lambda: ops.attn_prompt(d, d, d, cu, out=d.half()), lambda: ops.attn_prompt(d.transpose(1, 2), d, d, cu), lambda: ops.attn_prompt(d, d[:1], d[:1], cu),
                lambda: ops.attn_prompt(d, d, d, cu, i32([0, 1, 2])), lambda: ops.attn_prompt(d, d, d, cu, scale=-1.0), lambda: ops.attn_prompt(d, d, d, cu, scale=3e38),
                lambda: ops.attn_prompt(d[:, :, :4].contiguous(), d[:, :, :4].contiguous(), d[:, :, :4].contiguous(), cu),
                lambda: ops.attn_prompt(torch.zeros(40, device="cuda")[1:33].view(2, 2, 8), d, d, cu),              # not at 16 bytes
                lambda: ops.attn_prompt(torch.zeros(2, 3, 8, device="cuda"), d, d, cu),                               # 3 heads over 2
                lambda: ops.attn_prompt(d, d, d, cu, out=torch.zeros(1, 2, 8, device="cuda").expand(2, 2, 8)),
                lambda: ops.attn_pages(d.half(), c, table, lens), lambda: ops.attn_pages(d, c, table[:1], lens), lambda: ops.attn_pages(d, c, table, lens[:1]),
                lambda: ops.attn_pages(d, c, table.long(), lens), lambda: ops.attn_pages(d, c, i32([[0, 1], [2, 3]]).t(), lens), lambda: ops.attn_pages(d, c, table, lens, cu),
                lambda: ops.kv_append(c, d, d[:1], table, lens), lambda: ops.kv_append(c, d.half(), d.half(), table, lens), lambda: ops.kv_append(c, d, d, table[:1], lens),
                lambda: ops.KVPages(c.k, c.v[:2]), lambda: ops.KVPages(c.k, c.v.half()), lambda: ops.KVPages(c.k.cpu(), c.v), lambda: ops.KVPages(c.k[0], c.v[0]),
                lambda: ops.attn_pages(d, ops.KVPages(c.k[:, :, :12], c.v[:, :, :12]), table, lens),                  # pages of 12
                lambda: ops.sample(l.cpu(), u), lambda: ops.sample(l, u[:1]), lambda: ops.sample(l, u.double()), lambda: ops.sample(l.t(), u), lambda: ops.sample(l[0], u),
                lambda: ops.sample(l, u, top_k=u), lambda: ops.sample(l, u, temperature=lens), lambda: ops.sample(l.int(), u), lambda: ops.sample(l[:, :0], u),
                lambda: ops.sample(l, u, out=u)):
        with pytest.raises(hip.FastLlamaHipError):
            bad()


# ------------------------------------------------------------------------------------------------ streams, graphs, together
def test_calls_on_two_streams_at_once(ops):
    """Two caches attended and two batches sampled on streams of their own, many calls in flight: each as if alone."""
    jobs = []
    for j in range(2):
        lens = [1500 + 700 * j, 3, 900]
        k, v = (randn(10 * j + i, sum(lens), 2, 128, dtype=F16) for i in (1, 2))
        cache, table = scatter(ops, k, v, lens, 32, j)
        jobs.append((randn(10 * j, 3, 8, 128, dtype=F16), cache, table, i32(lens), logits_like(j, 5, 20000, F32), torch.rand(5, device="cuda")))
    want = [(ops.attn_pages(*j[:4]), ops.sample(*j[4:], 0.8, 0, 0.9)) for j in jobs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in jobs], [[], []]
    for _ in range(20):
        for i, (s, j) in enumerate(zip(streams, jobs)):
            with torch.cuda.stream(s):
                got[i].append((ops.attn_pages(*j[:4]), ops.sample(*j[4:], 0.8, 0, 0.9)))
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        for a, t in g:
            assert torch.equal(a, w[0]) and torch.equal(t, w[1])


class Layers:
    """A small decoder of the framework's own products and these operators, for several sequences: 2 layers, 8 query and 2 key heads."""
    E, H, Hkv, D, L, V = 256, 8, 2, 32, 2, 512

    def __init__(self, ops, cache_type):
        import oracle
        port, rng = oracle.Port(), np.random.default_rng(0)
        self.ops = ops
        w = lambda M, K: ops.QTensor(2, port.quantize_q4(2, (rng.standard_normal((M, K)) * K ** -0.5).astype(np.float32)), M, K)
        self.qkv = [w((self.H + 2 * self.Hkv) * self.D, self.E) for _ in range(self.L)]
        self.wo = [w(self.E, self.H * self.D) for _ in range(self.L)]
        self.head = w(self.V, self.E)
        self.emb = torch.from_numpy(rng.standard_normal((self.V, self.E)).astype(np.float32)).cuda()
        self.pages = [ops.KVPages.empty(40, 16, self.Hkv, self.D, cache_type) for _ in range(self.L)]
        self.T = cache_type

    def project(self, i, x):
        y = self.ops.mul_mat(self.qkv[i], x)
        return [t.unflatten(1, (-1, self.D)) for t in y.split([self.H * self.D, self.Hkv * self.D, self.Hkv * self.D], 1)]

    def step(self, tokens, table, n_past, kv_len, cu=None):
        """hidden rows of new tokens (cu: several for each sequence) through cache and attention"""
        x = self.emb[tokens.long()]
        for i in range(self.L):
            q, k, v = self.project(i, x)
            self.ops.kv_append(self.pages[i], k, v, table, n_past, cu)
            a = self.ops.attn_pages(q.to(self.T), self.pages[i], table, kv_len, cu)
            x = x + self.ops.mul_mat(self.wo[i], a.float().flatten(1).contiguous())
        return x

    def prompt(self, tokens, cu):
        """the same without a cache"""
        x = self.emb[tokens.long()]
        for i in range(self.L):
            q, k, v = self.project(i, x)
            a = self.ops.attn_prompt(q.to(self.T), k.to(self.T), v.to(self.T), cu)
            x = x + self.ops.mul_mat(self.wo[i], a.float().flatten(1).contiguous())
        return x


@pytest.mark.parametrize("T", [F32, F16])
def test_serving_together(ops, T):
    """Prompts of three users through the cache in chunks, then tokens one at a time; every row's hidden state against a pass over the whole packed
    text without a cache.  Q8_0 may round a value the other way where the attention's last bits differ: half a step of 1/127 of a block's largest
    value, in each of two products; 0.05 of the largest hidden value is far above that and far below what a wrong key or position does (~1)."""
    m, lens = Layers(ops, T), [37, 5, 64]
    table = i32([[3, 9, 11, 30, 2, 17], [0, 1, 4, 5, 6, 7], [39, 38, 12, 13, 33, 20]])
    rng = np.random.default_rng(1)
    text = [rng.integers(0, m.V, n).tolist() for n in lens]
    rows = [[] for _ in lens]
    for chunk in ([20, 5, 16], [17, 0, 48]):              # prompts, in two chunks
        at = [len(r) for r in rows]
        take = [t[a:a + c] for t, a, c in zip(text, at, chunk)]
        x = m.step(i32(sum(take, [])), table, i32(at), i32([a + c for a, c in zip(at, chunk)]), starts(chunk))
        for r, part in zip(rows, x.split(chunk)):
            r += list(part)
    u = torch.rand((6, 3), generator=torch.Generator().manual_seed(2)).cuda()
    for s in range(6):                                    # tokens
        last = torch.stack([r[-1] for r in rows])
        token = ops.sample(ops.mul_mat(m.head, last), u[s], 0.9, 50, 0.95)
        for t, new in zip(text, token.tolist()):
            assert 0 <= new < m.V
            t.append(new)
        n = [len(t) for t in text]
        for r, part in zip(rows, m.step(token, table, i32([a - 1 for a in n]), i32(n))):
            r.append(part)
    want = m.prompt(i32(sum(text, [])), starts([len(t) for t in text]))
    got = torch.stack(sum(rows, []))
    assert float((got - want).abs().max()) <= 0.05 * float(want.abs().max())


def test_serving_step_replayed_in_a_graph(ops):
    """One step (append, attention, sampling) captured once and replayed as the sequences grow, with eager work in between; every replay is compared
    with the eager result on a second cache."""
    H, Hkv, D, V = 8, 2, 64, 2000
    table, lens = i32([[3, 9, 11, 30], [0, 1, 4, 5]]), [14, 30]
    caches = [ops.KVPages.empty(40, 16, Hkv, D, F16) for _ in range(2)]
    k, v = randn(1, sum(lens), Hkv, D), randn(2, sum(lens), Hkv, D)
    for c in caches:
        ops.kv_append(c, k, v, table, i32([0, 0]), starts(lens))
    q, kn, vn, n_past, kv_len = randn(3, 2, H, D, dtype=F16), randn(4, 2, Hkv, D), randn(5, 2, Hkv, D), i32(lens), i32([n + 1 for n in lens])
    logits, u = logits_like(3, 2, V, F32), torch.rand(2, device="cuda")

    def step(c):
        ops.kv_append(c, kn, vn, table, n_past)
        return ops.attn_pages(q, c, table, kv_len), ops.sample(logits, u, 0.8, 40, 0.95), ops.attn_pages(q, c, table, kv_len, i32_cu)

    i32_cu = i32([0, 1, 2])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(caches[0])
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):                                    # two graphs, each with its own memory
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(caches[0])
        graphs.append((g, out))
    for i in range(20):
        for t, s in ((q, 10 + i), (kn, 40 + i), (vn, 70 + i)):
            t.copy_(randn(s, *t.shape))
        logits.copy_(logits_like(i, 2, V, F32))
        u.copy_(torch.rand(2, device="cuda"))
        want = [x.clone() for x in step(caches[1])]
        g, out = graphs[i % 2]
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b), i
        n_past += 1
        kv_len += 1


@pytest.mark.parametrize("what", ["prompt", "pages", "decode", "sample"])
def test_the_same_call_twice_gives_the_same_bits(ops, what):
    q, k, v = randn(1, 500, 8, 128, dtype=BF16), randn(2, 500, 2, 128, dtype=BF16), randn(3, 500, 2, 128, dtype=BF16)
    cache, table = scatter(ops, k, v, [500], 16, 1)
    l, u = logits_like(1, 64, 32000, F32), torch.rand(64, device="cuda")
    call = {"prompt": lambda: ops.attn_prompt(q, k, v, i32([0, 500])), "pages": lambda: ops.attn_pages(q, cache, table, i32([500]), i32([0, 500])),
            "decode": lambda: ops.attn_pages(q[:1], cache, table, i32([500])), "sample": lambda: ops.sample(l, u, 0.9, 0, 0.9)}[what]
    want = call()
    for _ in range(10):
        assert torch.equal(call(), want)
