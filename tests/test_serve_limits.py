"""CPU: sizes at the end of 32 bits, refused before the device is touched (nothing that fits is)."""
import ctypes as C

from test_serve_ops import GOOD, L, P, append, cache, heads, prompt  # noqa: F401

from fastllama_amd import hip

MOST = (1 << 31) - 512


def test_rows_and_keys_end_below_32_bits(L):
    """The last row's workgroup and the last key's tile are counted to their ends."""
    for H in (1, 2):
        assert prompt(L, H=H, Hkv=1, nq=MOST // H, out=heads(ts=256), size=1 << 50) == GOOD
        assert prompt(L, H=H, Hkv=1, nq=MOST // H + 1, size=1 << 50) == hip.FL_EINVAL
    assert prompt(L, nq=(1 << 31) - 1, H=1, Hkv=1, size=1 << 50) == hip.FL_EINVAL
    assert prompt(L, nk=MOST, size=1 << 50) == GOOD
    for n in (MOST + 1, (1 << 31) - 1):
        assert prompt(L, nk=n, size=1 << 50) == hip.FL_EINVAL
        assert b"fl_attn_prompt" in L.fl_last_error()


def test_an_append_is_one_launch(L):
    big = dict(c=cache(n_head_kv=128, head_dim=128, head_stride=2048, page_stride=1 << 18, slot_stride=128), k=heads(ts=16384, hs=128), v=heads(ts=16384, hs=128))
    n = ((1 << 32) - 256) // (128 * 16)
    assert append(L, n=n, **big) == GOOD
    assert append(L, n=n + 1, **big) == hip.FL_EINVAL and b"fl_kv_append" in L.fl_last_error()
