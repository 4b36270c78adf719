"""CPU: what the entry points of the operators over several sequences refuse.  Arguments are checked before the device is touched, so a call that
is fine up to there ends with FL_ENODEV here."""
import ctypes as C

import pytest

from fastllama_amd import hip


@pytest.fixture(scope="module")
def L():
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is present: the addresses here are made up")
    return hip.load()


P = 1 << 20      # an address that nothing reads


def cache(**kw):
    a = dict(k_dev=P, v_dev=P, type=hip.F16, n_pages=4, page_size=16, n_head_kv=2, head_dim=64, page_stride=2048, head_stride=1024, slot_stride=64)
    a.update(kw)
    return C.byref(hip.KVPagesDesc(**a))


def heads(p=P, ts=128, hs=64):
    return C.byref(hip.Heads(p, ts, hs))


GOOD = hip.FL_ENODEV
BAD_CACHES = [dict(k_dev=None), dict(v_dev=P + 8), dict(type=2), dict(type=7), dict(n_pages=0), dict(page_size=8), dict(page_size=24), dict(page_size=1 << 17),
              dict(n_head_kv=0), dict(head_dim=0), dict(head_dim=12), dict(head_dim=136), dict(page_stride=2044), dict(head_stride=-8), dict(slot_stride=3)]


def append(L, c=None, src=hip.F32, k=None, v=None, n=3, cu=P, past=P, table=P, ld=5, nt=5, ns=2):
    return L.fl_kv_append(c or cache(), src, k or heads(), v or heads(), n, cu, past, table, ld, nt, ns, None)


def test_append_refuses(L):
    assert append(L) == GOOD and append(L, src=hip.F16) == GOOD and append(L, n=2, cu=None) == GOOD
    for kw in BAD_CACHES:
        assert append(L, cache(**kw)) == hip.FL_EINVAL, kw
    for kw in (dict(src=hip.BF16), dict(src=2), dict(n=-1), dict(cu=None), dict(past=None), dict(table=None), dict(ns=0), dict(nt=0), dict(ld=4), dict(ld=-1),
               dict(nt=1 << 28, ld=1 << 28), dict(k=heads(None)), dict(v=heads(P + 4)), dict(k=heads(ts=130)), dict(v=heads(hs=-64)),
               dict(c=cache(slot_stride=0)), dict(c=cache(page_stride=0)), dict(c=cache(head_stride=0))):
        assert append(L, **kw) == hip.FL_EINVAL, kw
        assert b"fl_kv_append" in L.fl_last_error()
    assert L.fl_kv_append(None, 0, heads(), heads(), 1, None, P, P, 1, 1, 1, None) == hip.FL_EINVAL
    assert append(L, n=0, k=heads(None), v=heads(None)) == hip.FL_OK            # nothing to do


def prompt(L, type=hip.F16, D=64, H=4, Hkv=2, scale=0.1, q=None, nq=9, k=None, v=None, nk=9, cq=P, ck=P, ns=2, out=None, ws=P, size=1 << 40):
    return L.fl_attn_prompt(type, D, H, Hkv, scale, q or heads(ts=256), nq, k or heads(), v or heads(), nk, cq, ck, ns, out or heads(ts=256), ws, size, None)


def test_prompt_refuses(L):
    assert prompt(L) == GOOD and prompt(L, type=hip.F32) == GOOD and prompt(L, nk=0, k=heads(None), v=heads(None)) == GOOD
    for kw in (dict(type=3), dict(D=4), dict(D=132), dict(D=256), dict(H=3), dict(H=0), dict(Hkv=0), dict(H=65538), dict(scale=0.0), dict(scale=-1.0),
               dict(scale=float("nan")), dict(scale=float("inf")), dict(q=heads(None)), dict(q=heads(P + 2)), dict(k=heads(ts=100)), dict(v=heads(hs=4)),
               dict(nq=-1), dict(nk=-1), dict(ns=-1), dict(cq=None), dict(ck=None), dict(out=heads(None)), dict(out=heads(ts=0)), dict(out=heads(ts=256, hs=0))):
        assert prompt(L, **kw) == hip.FL_EINVAL, kw
        assert b"fl_attn_prompt" in L.fl_last_error()
    assert prompt(L, nq=0, q=heads(None), out=heads(None)) == hip.FL_OK and prompt(L, ns=0) == hip.FL_OK


def pages(L, c=None, H=4, scale=0.1, q=None, nq=2, cu=None, lens=P, table=P, ld=5, nt=5, ns=2, out=None, ws=P, size=1 << 30):
    return L.fl_attn_pages(c or cache(), H, scale, q or heads(ts=256), nq, cu, lens, table, ld, nt, ns, out or heads(ts=256), ws, size, None)


def test_pages_refuses(L):
    assert pages(L) == GOOD and pages(L, nq=9, cu=P) == GOOD
    for kw in BAD_CACHES:
        assert pages(L, cache(**kw)) == hip.FL_EINVAL, kw
    for kw in (dict(H=3), dict(H=0), dict(scale=0.0), dict(q=heads(None)), dict(nq=3), dict(nq=-1), dict(lens=None), dict(table=None), dict(nt=0), dict(ld=4),
               dict(nt=1 << 27, ld=1 << 27), dict(ns=-1), dict(out=heads(ts=0))):
        assert pages(L, **kw) == hip.FL_EINVAL, kw
        assert b"fl_attn_pages" in L.fl_last_error()
    assert pages(L, nq=0, ns=0, q=heads(None), out=heads(None)) == hip.FL_OK


def test_pages_workspace(L):
    """What the query names is enough, anything less is refused, also where it is not aligned."""
    for H, nt, ns in ((4, 5, 2), (4, 4096, 1), (64, 256, 64), (2, 100000, 3)):
        size = L.fl_attn_pages_workspace(cache(), H, ns, nt, ns, 1)
        assert pages(L, H=H, nq=ns, ld=nt, nt=nt, ns=ns, size=size, ws=P if size else None) == GOOD
        if size:
            for kw in (dict(size=size - 1), dict(ws=None), dict(ws=P + 4)):
                assert pages(L, **{**dict(H=H, nq=ns, ld=nt, nt=nt, ns=ns, size=size), **kw}) == hip.FL_EINVAL
    assert L.fl_attn_pages_workspace(None, 4, 2, 5, 2, 1) == 0 and L.fl_attn_pages_workspace(cache(), 0, 2, 5, 2, 1) == 0
    seen = 0
    for H, nq, n in ((4, 9, 40), (2, 16, 30000), (4, 100, 5000), (64, 5000, 5000)):     # several rows a sequence; prompts
        size = L.fl_attn_pages_workspace(cache(), H, nq, n // 16, 3, 0)
        kw = dict(H=H, nq=nq, cu=P, ld=n, nt=n // 16, ns=3)
        assert pages(L, **kw, size=size, ws=P if size else None) == GOOD
        also = L.fl_attn_prompt_workspace(hip.F16, 64, H, 2, nq, n, 3)
        kp = dict(H=H, nq=nq, nk=n, ns=3)
        assert prompt(L, **kp, size=also, ws=P if also else None) == GOOD
        for f, need, k in ((pages, size, kw), (prompt, also, kp)):
            if need:
                seen += 1
                for bad in (dict(size=need - 1), dict(ws=None), dict(ws=P + 4)):
                    assert f(L, **{**k, "size": need, **bad}) == hip.FL_EINVAL
    assert seen >= 2 and L.fl_attn_prompt_workspace(2, 64, 4, 2, 9, 9, 1) == 0


def sample(L, type=hip.F32, l=P, ld=100, rows=2, V=100, u=P, p=C.byref(hip.SampleParams()), out=P, ws=P, size=1 << 40):
    return L.fl_sample(type, l, ld, rows, V, u, p, out, ws, size, None)


def test_sample_refuses(L):
    assert sample(L) == GOOD and sample(L, V=hip.SAMPLE_MAX_VOCAB, ld=hip.SAMPLE_MAX_VOCAB) == GOOD and sample(L, rows=1, ld=0) == GOOD
    for kw in (dict(type=2), dict(l=None), dict(l=P + 2), dict(ld=99), dict(ld=-1), dict(rows=-1), dict(V=0), dict(V=hip.SAMPLE_MAX_VOCAB + 1, ld=1 << 20), dict(u=None),
               dict(p=None), dict(out=None), dict(ws=None), dict(ws=P + 8), dict(size=L.fl_sample_workspace(2, 100) - 1)):
        assert sample(L, **kw) == hip.FL_EINVAL, kw
        assert b"fl_sample" in L.fl_last_error()
    assert sample(L, rows=0, l=None) == hip.FL_OK
    for rows, V in ((1, 1), (3, 4097), (200, 32000), (5000, 262144)):
        size = L.fl_sample_workspace(rows, V)
        assert size > 0 and sample(L, rows=rows, V=V, ld=V, size=size) == GOOD and sample(L, rows=rows, V=V, ld=V, size=size - 1) == hip.FL_EINVAL
    assert L.fl_sample_workspace(0, 5) == 0 and L.fl_sample_workspace(5, 0) == 0 and L.fl_sample_workspace(5, 1 << 30) == 0
    assert L.fl_model_logits_sample(None, 0, 1, P, C.byref(hip.SampleParams()), P) == hip.FL_EINVAL


def test_python_entry_points_refuse_host_tensors():
    """ops: no CPU path, as for the other operators; shapes and types that do not fit are named."""
    import torch
    from fastllama_amd import ops
    x, one = torch.zeros(2, 2, 8), torch.zeros(3, dtype=torch.int32)
    E = hip.FastLlamaHipError
    with pytest.raises(E, match="no CPU path"):
        ops.KVPages(torch.zeros(1, 1, 16, 8), torch.zeros(1, 1, 16, 8))
    if torch.cuda.is_available():
        d, one = x.cuda(), one.cuda()
        for bad in (lambda: ops.attn_prompt(x, x, x, one), lambda: ops.attn_prompt(d, d, d.half(), one), lambda: ops.attn_prompt(d[0], d, d, one),
                    lambda: ops.attn_prompt(d, d, d, one.long()), lambda: ops.attn_prompt(d.double(), d.double(), d.double(), one),
                    lambda: ops.attn_prompt(d, d, d, one, out=d.half()), lambda: ops.attn_prompt(d.transpose(1, 2), d, d, one),
                    lambda: ops.attn_prompt(d, d[:1], d[:1], one), lambda: ops.sample(d[0].cpu(), d[0, :, 0]), lambda: ops.sample(d[0], d[0, 0]),
                    lambda: ops.sample(d[0], d[0, :, 0].contiguous(), top_k=d[0, :, 0].contiguous())):
            with pytest.raises(E):
                bad()
