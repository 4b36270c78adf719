"""Host-side mirror of the reference's operator interface for the Q4 hot path, over the C-ABI.

Names and argument meaning follow the reference (``quantize_fns_t`` include/ggml.h:850-862 and
``ggml_mul_mat`` lib/ggml.c:4925-4948):

* ``QTensor``              a Q4_0/Q4_1 weight ``ne = [K, M]`` resident in HBM (QW16 layout)
* ``quantize_row_q8_0``    quantize_fns[type].quantize_row_q_dot
* ``dequantize_row_q``     quantize_fns[type].dequantize_row_q
* ``vec_dot_q``            quantize_fns[type].vec_dot_q
* ``mul_mat``              ggml_mul_mat(W, x) for quantized W  ->  ggml_compute_forward_mul_mat_q_f32

and the operators of a serving step over several sequences, which the reference does not have:

* ``KVPages``              a paged K/V cache over tensors of the caller's; ``kv_append`` writes rows into it
* ``attn_prompt``          causal attention with grouped heads over packed prompts
* ``attn_pages``           the same over a paged cache: one new token for each sequence, or chunks of prompts
* ``sample``               temperature / top-k / top-p / min-p from given uniform numbers

Inference only: no operator here records a gradient, also for tensors that require one.

torch is used only to own device memory and to pick the stream; every computation happens inside
libfastllama_hip.so.  Nothing here computes on the CPU.
"""
from __future__ import annotations

import ctypes as C

import numpy as np
import torch

from . import hip
from .hip import Q4_0, Q4_1, BLOCK_BYTES, Q8_BLOCK_BYTES, QK, check


def _stream() -> C.c_void_p:
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def _dev(t: torch.Tensor) -> C.c_void_p:
    if not t.is_cuda:
        raise hip.FastLlamaHipError("expected a device tensor: fastllama_amd has no CPU path")
    return C.c_void_p(t.data_ptr())


class QTensor:
    """Quantized weight matrix W[M rows][K], uploaded from the reference's AoS block bytes."""

    def __init__(self, qtype: int, blocks, M: int, K: int):
        lib = hip.load()
        hip.require_device(torch.cuda.current_device())
        self.qtype, self.M, self.K = qtype, M, K
        if qtype not in BLOCK_BYTES:
            raise hip.FastLlamaHipError(f"type {qtype} is not Q4_0 (2) / Q4_1 (3)")
        nbytes = M * (K // QK) * BLOCK_BYTES[qtype]
        if isinstance(blocks, torch.Tensor) and blocks.is_cuda:
            assert blocks.numel() * blocks.element_size() == nbytes
            h = lib.fl_qtensor_from_device(qtype, _dev(blocks), M, K, _stream())
        else:
            arr = np.ascontiguousarray(blocks, dtype=np.uint8)
            assert arr.size == nbytes, (arr.size, nbytes)
            h = lib.fl_qtensor_upload(qtype, arr.ctypes.data_as(C.c_void_p), M, K, _stream())
        if not h:
            raise hip.FastLlamaHipError("fl_qtensor_upload: " + lib.fl_last_error().decode())
        self.handle = C.c_void_p(h)

    def download(self) -> np.ndarray:
        out = np.empty((self.M, self.K // QK * BLOCK_BYTES[self.qtype]), dtype=np.uint8)
        check(hip.load().fl_qtensor_download(self.handle, out.ctypes.data_as(C.c_void_p), _stream()),
              "fl_qtensor_download")
        return out

    @property
    def device_bytes(self) -> int:
        return hip.load().fl_qtensor_device_bytes(self.handle)

    def free(self):
        if getattr(self, "handle", None):
            hip.load().fl_qtensor_free(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


class QAct:
    """The Q8_0 activation scratch of mul_mat_q_f32 (params->wdata, lib/ggml.c:8105-8119)."""

    def __init__(self, max_N: int, K: int):
        lib = hip.load()
        hip.require_device(torch.cuda.current_device())
        h = lib.fl_qact_create(max_N, K)
        if not h:
            raise hip.FastLlamaHipError("fl_qact_create: " + lib.fl_last_error().decode())
        self.handle = C.c_void_p(h)
        self.max_N, self.K, self.N = max_N, K, 0

    def quantize(self, x: torch.Tensor, layout: int | None = None) -> "QAct":
        assert x.dtype == torch.float32 and x.dim() == 2 and x.stride(1) == 1
        N, K = x.shape
        lib = hip.load()
        if layout is None:
            check(lib.fl_quantize_q8(self.handle, _dev(x), x.stride(0), N, K, _stream()), "fl_quantize_q8")
        else:
            check(lib.fl_quantize_q8_layout(self.handle, _dev(x), x.stride(0), N, K, layout, _stream()),
                  "fl_quantize_q8_layout")
        self.N, self.K = N, K
        return self

    def export(self) -> torch.Tensor:
        """-> uint8 [N, K/32*40] device tensor in the reference's block_q8_0 layout."""
        out = torch.empty((self.N, self.K // QK * Q8_BLOCK_BYTES), dtype=torch.uint8, device="cuda")
        check(hip.load().fl_qact_export(self.handle, _dev(out), _stream()), "fl_qact_export")
        return out

    def free(self):
        if getattr(self, "handle", None):
            hip.load().fl_qact_free(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


def quantize_row_q8_0(x: torch.Tensor) -> torch.Tensor:
    """quantize_row_q_dot(x, y, k): f32 [k] -> block_q8_0 bytes (uint8 [k/32*40]) on the device."""
    assert x.dtype == torch.float32 and x.dim() == 1 and x.is_contiguous()
    k = x.numel()
    y = torch.empty(k // QK * Q8_BLOCK_BYTES, dtype=torch.uint8, device=x.device)
    check(hip.load().fl_quantize_row_q8_0(_dev(x), _dev(y), k, _stream()), "fl_quantize_row_q8_0")
    return y


def quantize_row_q(qtype: int, x: torch.Tensor, reference: bool = False) -> torch.Tensor:
    """quantize_row_q(x, y, k) / quantize_row_q_reference: f32 [k] -> block_q4_0 / block_q4_1 bytes on the device."""
    assert x.dtype == torch.float32 and x.is_contiguous()
    k = x.numel()
    y = torch.empty(k // QK * BLOCK_BYTES[qtype], dtype=torch.uint8, device=x.device)
    name = "fl_quantize_row_q4_%d%s" % (0 if qtype == Q4_0 else 1, "_reference" if reference else "")
    check(getattr(hip.load(), name)(_dev(x), _dev(y), k, _stream()), name)
    return y


def dequantize_row_q(qtype: int, blocks: torch.Tensor, k: int) -> torch.Tensor:
    """dequantize_row_q(x, y, k): AoS Q4 block bytes -> f32 [k]."""
    y = torch.empty(k, dtype=torch.float32, device=blocks.device)
    fn = hip.load().fl_dequantize_row_q4_0 if qtype == Q4_0 else hip.load().fl_dequantize_row_q4_1
    check(fn(_dev(blocks), _dev(y), k, _stream()), "fl_dequantize_row_q4")
    return y


def vec_dot_q(qtype: int, n: int, wrow: torch.Tensor, xq: torch.Tensor) -> torch.Tensor:
    """vec_dot_q(n, s, x, y): one Q4 row times one Q8_0 row (both AoS bytes) -> f32 [1]."""
    s = torch.empty(1, dtype=torch.float32, device=wrow.device)
    fn = hip.load().fl_vec_dot_q4_0_q8_0 if qtype == Q4_0 else hip.load().fl_vec_dot_q4_1_q8_0
    check(fn(n, _dev(s), _dev(wrow), _dev(xq), _stream()), "fl_vec_dot_q4")
    return s


def mul_mat(W: QTensor, x: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """ggml_mul_mat(W[K,M], x[K,N]) -> y[M,N]; tensors are row-major so x is [N, K], y is [N, M]."""
    assert x.dtype == torch.float32 and x.dim() == 2 and x.stride(1) == 1 and x.shape[1] == W.K
    N = x.shape[0]
    if out is None:
        ld = (W.M + 3) // 4 * 4
        buf = torch.empty((N, ld), dtype=torch.float32, device=x.device)
        out = buf[:, :W.M]
    check(hip.load().fl_mul_mat_q_f32(W.handle, _dev(x), x.stride(0), _dev(out), out.stride(0), N, _stream()),
          "fl_mul_mat_q_f32")
    return out


def mul_mat_q(W: QTensor, a: QAct, which: int | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """COMPUTE phase only, on an already quantized activation workspace."""
    if out is None:
        ld = (W.M + 3) // 4 * 4
        out = torch.empty((a.N, ld), dtype=torch.float32, device="cuda")[:, :W.M]
    lib = hip.load()
    if which is None:
        check(lib.fl_mul_mat_q(W.handle, a.handle, _dev(out), out.stride(0), _stream()), "fl_mul_mat_q")
    else:
        check(lib.fl_debug_mul_mat_q(W.handle, a.handle, _dev(out), out.stride(0), which, _stream()),
              "fl_debug_mul_mat_q")
    return out


# ---- several sequences (fastllama_hip.h "several sequences": the formulas, limits and what is done with places outside the buffers) ----
_Error = hip.FastLlamaHipError
_TYPES = {torch.float32: hip.F32, torch.float16: hip.F16, torch.bfloat16: hip.BF16}


def _type(t: torch.Tensor, what: str) -> int:
    n = _TYPES.get(t.dtype)
    if n is None:
        raise _Error(f"{what}: {t.dtype} is not float32, float16 or bfloat16")
    return n


def _elsewhere(t, device: int, what: str) -> Exception:
    """The kernels run on the current device's current stream: why a tensor that is not there is refused."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        return _Error(f"{what}: expected a device tensor: fastllama_amd has no CPU path")
    return _Error(f"{what} is on {t.device}, the current device is cuda:{device}")


def _heads(t: torch.Tensor, device: int, what: str) -> hip.Heads:
    """[rows, heads, head_dim] of any strides, the last axis dense"""
    if not isinstance(t, torch.Tensor) or t.get_device() != device:
        raise _elsewhere(t, device, what)
    shape, stride = t.shape, t.stride()
    if len(shape) != 3 or (stride[2] != 1 and shape[2] != 1):
        raise _Error(f"{what}: want [rows, heads, head_dim] with a dense last axis, got {tuple(shape)} strides {stride}")
    return hip.Heads(t.data_ptr(), stride[0] if shape[0] > 1 else 0, stride[1] if shape[1] > 1 else 0)


def _row(t: torch.Tensor, device: int, what: str, n: int, dtype: torch.dtype = torch.int32) -> int:
    """The address of n dense values."""
    if not isinstance(t, torch.Tensor) or t.get_device() != device:
        raise _elsewhere(t, device, what)
    shape = t.shape
    if t.dtype != dtype or len(shape) != 1 or shape[0] != n or (n > 1 and t.stride(0) != 1):
        raise _Error(f"{what}: want {n} dense {dtype}, got {tuple(shape)} {t.dtype}")
    return t.data_ptr()


def _table(t: torch.Tensor, device: int) -> tuple[int, int, int, int]:
    """(address, row stride, sequences, pages) of [sequences, pages]"""
    if not isinstance(t, torch.Tensor) or t.get_device() != device:
        raise _elsewhere(t, device, "table")
    shape, stride = t.shape, t.stride()
    if t.dtype != torch.int32 or len(shape) != 2 or (shape[1] > 1 and stride[1] != 1):
        raise _Error(f"table: want int32 [sequences, pages] with a dense last axis, got {tuple(shape)} {t.dtype}")
    return t.data_ptr(), stride[0] if shape[0] > 1 else shape[1], shape[0], shape[1]


def _raw_stream(device: int) -> int:
    return torch._C._cuda_getCurrentRawStream(device)


class KVPages:
    """A paged K/V cache: ``k`` and ``v`` are [n_pages, n_head_kv, page_size, head_dim] views (any strides, the last axis dense, both alike) of
    float32, float16 or bfloat16.  Position p of a sequence is slot p % page_size of page table[sequence][p // page_size]."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor):
        for t, what in ((k, "k"), (v, "v")):
            if not (isinstance(t, torch.Tensor) and t.is_cuda):
                raise _Error(f"{what}: expected a device tensor: fastllama_amd has no CPU path")
            if not (t.dim() == 4 and (t.stride(3) == 1 or t.shape[3] == 1)):
                raise _Error(f"{what}: want [n_pages, n_head_kv, page_size, head_dim] with a dense last axis, got {tuple(t.shape)}")
        if not (k.shape == v.shape and k.dtype == v.dtype and k.device == v.device):
            raise _Error("k and v are not alike")
        strides = [tuple(t.stride(i) if t.shape[i] > 1 else 0 for i in range(3)) for t in (k, v)]
        if not (strides[0] == strides[1]):
            raise _Error("k and v have other strides")
        self.k, self.v, self.device = k, v, k.get_device()
        (n, h, p, d), (sp, sh, ss) = k.shape, strides[0]
        self.desc = hip.KVPagesDesc(k.data_ptr(), v.data_ptr(), _type(k, "k"), n, p, h, d, sp, sh, ss)
        self.ref = C.byref(self.desc)

    @classmethod
    def empty(cls, n_pages: int, page_size: int, n_head_kv: int, head_dim: int, dtype: torch.dtype = torch.float16) -> "KVPages":
        shape = (n_pages, n_head_kv, page_size, head_dim)
        return cls(torch.empty(shape, dtype=dtype, device="cuda"), torch.empty(shape, dtype=dtype, device="cuda"))

    def check(self, device: int) -> None:
        if self.device != device:
            raise _Error(f"the cache is on cuda:{self.device}, the current device is cuda:{device}")


def kv_append(pages: KVPages, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, n_past: torch.Tensor, cu: torch.Tensor | None = None) -> None:
    """Rows ``k``, ``v`` [rows, n_head_kv, head_dim] (the cache's type, or float32: rounded once) become the positions behind n_past[b] of their
    sequences: rows cu[b]..cu[b+1]-1, or one row for each sequence where cu is None.  No two rows of a call may go to one slot."""
    device, d = torch.cuda.current_device(), pages.desc
    pages.check(device)
    kh, vh, (tab, ld, n, width) = _heads(k, device, "k"), _heads(v, device, "v"), _table(table, device)
    shape = k.shape
    if shape != v.shape or k.dtype != v.dtype or shape[1] != d.n_head_kv or shape[2] != d.head_dim:
        raise _Error(f"k, v: want [rows, {d.n_head_kv}, {d.head_dim}] alike, got {tuple(shape)} and {tuple(v.shape)}")
    if cu is None and n != shape[0]:
        raise _Error(f"{shape[0]} rows for {n} sequences and no row starts")
    check(hip.load().fl_kv_append(pages.ref, _type(k, "k"), kh, vh, shape[0], None if cu is None else _row(cu, device, "cu", n + 1),
                                  _row(n_past, device, "n_past", n), tab, ld, width, n, _raw_stream(device)), "fl_kv_append")


def _out(q: torch.Tensor, out: torch.Tensor | None) -> torch.Tensor:
    if out is None:
        return torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if out.shape != q.shape or out.dtype != q.dtype:
        raise _Error(f"out: want {tuple(q.shape)} {q.dtype}, got {tuple(out.shape)} {out.dtype}")
    return out


def attn_prompt(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_q: torch.Tensor, cu_kv: torch.Tensor | None = None, scale: float | None = None,
                out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of packed rows ``q`` [rows, n_head, head_dim] over ``k``, ``v`` [keys, n_head_kv, head_dim]; sequence b owns the rows
    cu_q[b]..cu_q[b+1]-1 and the keys cu_kv[b]..cu_kv[b+1]-1 (None: as the rows).  The last row sees every key of its sequence, each row before it
    one less; one that sees none becomes 0.  Rows outside every sequence are not written.  scale: 1 / sqrt(head_dim) unless given."""
    device = torch.cuda.current_device()
    qh, kh, vh = _heads(q, device, "q"), _heads(k, device, "k"), _heads(v, device, "v")
    qs, ks = q.shape, k.shape
    if ks != v.shape or ks[2] != qs[2] or not q.dtype == k.dtype == v.dtype:
        raise _Error(f"q, k, v: {tuple(qs)} {q.dtype}, {tuple(ks)} {k.dtype}, {tuple(v.shape)} {v.dtype} do not fit together")
    n = cu_q.numel() - 1
    if n < 0 or (cu_kv is None and qs[0] != ks[0]):
        raise _Error("cu_q is empty, or other numbers of rows and keys and no cu_kv")
    cu = _row(cu_q, device, "cu_q", n + 1)
    out = _out(q, out)
    lib, kind = hip.load(), _type(q, "q")
    size = lib.fl_attn_prompt_workspace(kind, qs[2], qs[1], ks[1], qs[0], ks[0], n)
    ws = torch.empty(size, dtype=torch.uint8, device=q.device) if size else None
    check(lib.fl_attn_prompt(kind, qs[2], qs[1], ks[1], qs[2] ** -0.5 if scale is None else scale, qh, qs[0], kh, vh, ks[0], cu,
                             cu if cu_kv is None else _row(cu_kv, device, "cu_kv", n + 1), n, _heads(out, device, "out"), ws.data_ptr() if size else None, size,
                             _raw_stream(device)), "fl_attn_prompt")
    return out


def attn_pages(q: torch.Tensor, pages: KVPages, table: torch.Tensor, kv_len: torch.Tensor, cu_q: torch.Tensor | None = None, scale: float | None = None,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of ``q`` [rows, n_head, head_dim] over the first kv_len[b] positions of each sequence in the cache: one row for each
    sequence (its newest token), or with ``cu_q`` the rows cu_q[b]..cu_q[b+1]-1 of each (its newest tokens, already in the cache)."""
    device, d = torch.cuda.current_device(), pages.desc
    pages.check(device)
    qh, (tab, ld, n, width) = _heads(q, device, "q"), _table(table, device)
    rows, heads, dim = q.shape
    if q.dtype != pages.k.dtype or dim != d.head_dim:
        raise _Error(f"q: {tuple(q.shape)} {q.dtype} does not fit a cache of head_dim {d.head_dim}, {pages.k.dtype}")
    if cu_q is None and n != rows:
        raise _Error(f"{rows} rows for {n} sequences and no row starts")
    lens, cu = _row(kv_len, device, "kv_len", n), None if cu_q is None else _row(cu_q, device, "cu_q", n + 1)
    out = _out(q, out)
    lib = hip.load()
    size = lib.fl_attn_pages_workspace(pages.ref, heads, rows, width, n, cu_q is None)
    ws = torch.empty(size, dtype=torch.uint8, device=q.device) if size else None
    check(lib.fl_attn_pages(pages.ref, heads, dim ** -0.5 if scale is None else scale, qh, rows, cu, lens, tab, ld, width, n, _heads(out, device, "out"),
                            ws.data_ptr() if size else None, size, _raw_stream(device)), "fl_attn_pages")
    return out


def sample(logits: torch.Tensor, u: torch.Tensor, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, out: torch.Tensor | None = None) -> torch.Tensor:
    """A token (int32 [rows]) for each row of ``logits`` [rows, n_vocab] from the uniform numbers ``u`` [rows] in [0, 1).  Each setting is a number
    for all rows or a device tensor of one for each (float32; top_k int32).  Off: top_k <= 0, top_p >= 1, min_p <= 0; temperature <= 0 is greedy."""
    device = torch.cuda.current_device()
    if not isinstance(logits, torch.Tensor) or logits.get_device() != device:
        raise _elsewhere(logits, device, "logits")
    shape, stride = logits.shape, logits.stride()
    if len(shape) != 2 or (stride[1] != 1 and shape[1] != 1):
        raise _Error(f"logits: want [rows, n_vocab] with a dense last axis, got {tuple(shape)} strides {stride}")
    rows, vocab = shape
    p = hip.SampleParams()
    for what, x in (("temperature", temperature), ("top_p", top_p), ("min_p", min_p)):
        if isinstance(x, torch.Tensor):
            setattr(p, what + "_dev", _row(x, device, what, rows, torch.float32))
        else:
            setattr(p, what, x)
    if isinstance(top_k, torch.Tensor):
        p.top_k_dev = _row(top_k, device, "top_k", rows)
    else:
        p.top_k = max(0, min(int(top_k), vocab))
    if out is None:
        out = torch.empty(rows, dtype=torch.int32, device=logits.device)
    lib = hip.load()
    size = lib.fl_sample_workspace(rows, vocab)
    ws = torch.empty(size, dtype=torch.uint8, device=logits.device)
    check(lib.fl_sample(_type(logits, "logits"), logits.data_ptr(), stride[0] if rows > 1 else vocab, rows, vocab, _row(u, device, "u", rows, torch.float32), p,
                        _row(out, device, "out", rows), ws.data_ptr(), size, _raw_stream(device)), "fl_sample")
    return out
