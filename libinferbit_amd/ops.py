"""Host-side mirror of the reference's matvec operator entry points.

Names and argument meaning follow the reference (src/threading.c,
src/kernels/scalar.c, src/inferbit_internal.h:199-277): ``out`` first, then
weights, scales, activations, then sizes.  Operands are torch tensors
resident on the current GPU; work is enqueued on torch's current stream so
torch.cuda events time it.  Calls that name another GPU for themselves (the
4-bit cache's, and those around a batch's projections) run on their operands'
and its current stream.  Errors raise IbhError (the library's negative
INFERBIT_ERROR_* code plus its message).
"""
from __future__ import annotations

import torch

import ctypes

import numpy as np

from ._lib import Int4gTensor, Kv4Desc, LoraDesc, PqPolicy, PqTensor, check, lib

SCALE_F16, SCALE_F32 = 0, 1


def _ptr(t: torch.Tensor):
    """The address of t, a contiguous tensor of the current GPU: a launch there reaches no other GPU's memory."""
    if not t.is_cuda:
        raise ValueError("libinferbit_amd ops take GPU tensors")
    if t.get_device() != torch._C._cuda_getDevice():
        raise ValueError(f"operand on {t.device}, the current GPU is cuda:{torch._C._cuda_getDevice()}")
    if not t.is_contiguous():
        raise ValueError("operand must be contiguous")
    return t.data_ptr()


def _gpu(t) -> int:
    """The GPU that t is on."""
    index = t.get_device()
    if index < 0:
        raise ValueError("libinferbit_amd ops take GPU tensors")
    return index


def _on(t, index: int, dtype, shape):
    """The address of t, a contiguous tensor of GPU `index` with the given type and shape."""
    if t.get_device() == index and t.dtype is dtype and t.shape == shape and t.is_contiguous():
        return t.data_ptr()
    if t.get_device() != index:
        raise ValueError(f"operand on {t.device}, another is on cuda:{index}")
    if t.dtype is not dtype:
        raise TypeError(f"operand must be {dtype}, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"operand must be {list(shape)}, got {list(t.shape)}")
    raise ValueError("operand must be contiguous")


def _spaced(t, index: int, shape):
    """(address, floats between rows) of t, fp32 rows [B, n] of contiguous elements on GPU `index`."""
    if t.get_device() == index and t.dtype is torch.float32 and t.shape == shape and t.is_contiguous():
        return t.data_ptr(), shape[1]
    if t.get_device() != index:
        raise ValueError(f"operand on {t.device}, another is on cuda:{index}")
    if t.dtype is not torch.float32:
        raise TypeError(f"operand must be torch.float32, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"operand must be {list(shape)}, got {list(t.shape)}")
    s0, s1 = t.stride()
    if shape[0] <= 1:
        s0 = shape[1]
    if (s1 != 1 and shape[1] > 1) or s0 < shape[1] or s0 > 0x7fffffff:
        raise ValueError("rows must not overlap and their elements must be contiguous")
    return t.data_ptr(), s0


def _call_on(index: int, name: str, *args) -> None:
    """A call on GPU `index`, on its current stream."""
    # the stream's handle without the Python object around it: that takes 1.8 us of a call's 8
    stream = torch._C._cuda_getCurrentRawStream(index)
    if torch._C._cuda_getDevice() == index:
        rc = getattr(lib(), name)(*args, stream)
    else:
        with torch.cuda.device(index):
            rc = getattr(lib(), name)(*args, stream)
    if rc:
        check(rc, name)


def _scratch(ws, need: int, index: int):
    """(address, bytes, the tensor to keep) of the given workspace, or of `need` bytes on GPU `index`."""
    if ws is not None:
        return _on(ws, index, torch.uint8, ws.shape), ws.numel(), ws
    if not need:
        return None, 0, None
    ws = torch.empty(need, dtype=torch.uint8, device=index)
    return ws.data_ptr(), need, ws


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _scale_kind(s: torch.Tensor) -> int:
    if s.dtype in (torch.float16, torch.int16, torch.uint16):
        return SCALE_F16
    if s.dtype == torch.float32:
        return SCALE_F32
    raise TypeError(f"scales must be fp16 bits or fp32, got {s.dtype}")


def init(device: int = 0) -> None:
    check(lib().ibh_init(device), "ibh_init")


def parallel_matmul(out, w, scales, x, M: int, N: int, bits: int) -> None:
    """ib_parallel_matmul (src/threading.c:244-258): out[M] = W[M,N] x[N] * scales."""
    check(lib().ibh_matmul(_ptr(out), _ptr(w), _ptr(scales), _scale_kind(scales), _ptr(x), M, N, bits,
                           _stream()), "ibh_matmul")


def quantize_input_int8_g128(x, q, s, N: int) -> int:
    """ib_quantize_input_int8_g128 (src/threading.c:401-432); returns the group count."""
    check(lib().ibh_quantize_act_g128(_ptr(x), _ptr(q), _ptr(s), N, _stream()), "ibh_quantize_act_g128")
    return (N + 127) // 128


def parallel_matmul_w4a8(out, w, scales_w, qx, scales_a, M: int, N: int) -> None:
    """ib_parallel_matmul_w4a8 (src/threading.c:283-294), x86 AVX2 kernel semantics."""
    check(lib().ibh_matmul_w4a8(_ptr(out), _ptr(w), _ptr(scales_w), _scale_kind(scales_w), _ptr(qx),
                                _ptr(scales_a), M, N, _stream()), "ibh_matmul_w4a8")


def matmul_w4a8_x(out, w, scales_w, x, M: int, N: int, qx_ws, sa_ws) -> None:
    """tensor_matmul's INT4 branch (src/forward.c:158-172): quantize x, then W4A8."""
    check(lib().ibh_matmul_w4a8_x(_ptr(out), _ptr(w), _ptr(scales_w), _scale_kind(scales_w), _ptr(x), M, N,
                                  _ptr(qx_ws), _ptr(sa_ws), _stream()), "ibh_matmul_w4a8_x")


def matmul_w4a8_batch(out, w, scales_w, qx, scales_a, M: int, N: int, B: int, M_stride: int) -> None:
    """ib_kern.matmul_w4a8_batch (src/kernels/scalar.c:86-124)."""
    check(lib().ibh_matmul_w4a8_batch(_ptr(out), _ptr(w), _ptr(scales_w), _scale_kind(scales_w), _ptr(qx),
                                      _ptr(scales_a), M, N, B, M_stride, _stream()), "ibh_matmul_w4a8_batch")


def matmul_int8_batch(out, w, scales_w, x, M: int, N: int, B: int, M_stride: int) -> None:
    """ib_kern.matmul_int8_batch (src/kernels/scalar.c:70-84)."""
    check(lib().ibh_matmul_int8_batch(_ptr(out), _ptr(w), _ptr(scales_w), _scale_kind(scales_w), _ptr(x), M,
                                      N, B, M_stride, _stream()), "ibh_matmul_int8_batch")


def gemm_int8(out, w, scales, x, M: int, N: int, B: int, M_stride: int, ws=None) -> None:
    """Prefill INT8 GEMM, matmul_int8_batch semantics at any B (src/kernels/scalar.c:70-84)."""
    if ws is None:
        ws = torch.empty(lib().ibh_gemm_int8_workspace_bytes(N, B), dtype=torch.uint8, device=out.device)
    check(lib().ibh_gemm_int8(_ptr(out), _ptr(w), _ptr(scales), _scale_kind(scales), _ptr(x), M, N, B, M_stride,
                              _ptr(ws), ws.numel(), _stream()), "ibh_gemm_int8")


def _optptr(t):
    return None if t is None else _ptr(t)


def kv_cache_write(kdata, vdata, kscales, vscales, pos: int, k, v, n_kv: int, head_dim: int, kv_bits: int) -> None:
    """kv_cache_write (src/forward.c:352-413) into device cache tensors."""
    check(lib().ibh_kv_write(_ptr(kdata), _ptr(vdata), _optptr(kscales), _optptr(vscales), pos, _ptr(k), _ptr(v),
                             n_kv, head_dim, kv_bits, _stream()), "ibh_kv_write")


def attn_decode(out, q, kdata, vdata, kscales, vscales, pos: int, n_heads: int, n_kv: int, head_dim: int,
                kv_bits: int) -> None:
    """ib_attn_head_task for all heads of a layer (src/forward.c:449-504)."""
    check(lib().ibh_attn_decode(_ptr(out), _ptr(q), _ptr(kdata), _ptr(vdata), _optptr(kscales), _optptr(vscales),
                                pos, n_heads, n_kv, head_dim, kv_bits, None, 0, _stream()), "ibh_attn_decode")


KV4_PAGE = 64


class Kv4Cache:
    """A paged 4-bit KV cache (ibh_kv4_cache): `pool` uint8 [n_pages,
    kv4_page_bytes], `table` int32 [n_seq, max_pages], `lens` int32 [n_seq],
    all contiguous on one GPU and kept by reference.  Calls on it run on that
    GPU, on its current stream."""

    def __init__(self, pool, table, lens, n_kv: int, head_dim: int):
        if table.dim() != 2 or lens.dim() != 1 or table.shape[0] != lens.shape[0]:
            raise ValueError("table must be [n_seq, max_pages] and lens [n_seq]")
        if table.dtype != torch.int32 or lens.dtype != torch.int32 or pool.dtype != torch.uint8:
            raise TypeError("a cache is a uint8 pool with an int32 table and int32 lens")
        self.device, self.index = pool.device, pool.get_device()
        self.pool, self.table, self.lens = pool, table, lens
        self.n_seq, self.max_pages = table.shape
        self.n_kv, self.head_dim = n_kv, head_dim
        size = lib().ibh_kv4_page_bytes(n_kv, head_dim)
        if not size or pool.numel() % size:
            raise ValueError(f"the pool is not whole pages of {n_kv} heads of {head_dim}")
        _gpu(pool)
        self.desc = Kv4Desc(self._on(pool, torch.uint8, pool.numel()), self._on(table, torch.int32, table.numel()),
                            self._on(lens, torch.int32, self.n_seq), pool.numel() // size, self.n_seq, self.max_pages,
                            n_kv, head_dim)
        self.ref = ctypes.byref(self.desc)

    def _on(self, t, dtype, numel):
        """The address of t, a contiguous tensor of this cache's GPU with the given type and size."""
        if t.get_device() != self.index:
            raise ValueError(f"operand on {t.device}, the cache is on {self.device}")
        if t.dtype != dtype:
            raise TypeError(f"operand must be {dtype}, got {t.dtype}")
        if t.numel() != numel:
            raise ValueError(f"operand must have {numel} elements, got {t.numel()}")
        if not t.is_contiguous():
            raise ValueError("operand must be contiguous")
        return t.data_ptr()

    def _rows(self, t, width: int):
        """(address, rows per sequence, floats between rows) of [n_seq, n, width] fp32 rows with unit inner stride."""
        if t.get_device() != self.index:
            raise ValueError(f"operand on {t.device}, the cache is on {self.device}")
        if t.dtype != torch.float32:
            raise TypeError(f"operand must be torch.float32, got {t.dtype}")
        shape = t.shape
        if len(shape) != 3 or shape[0] != self.n_seq or shape[2] != width:
            raise ValueError(f"operand must be [{self.n_seq}, n, {width}], got {list(shape)}")
        n = shape[1]
        s0, s1, s2 = t.stride()
        if n == 1:
            s1 = s0 if self.n_seq > 1 else width
        if s2 != 1 or s1 < width or s1 > 0x7fffffff or (self.n_seq > 1 and s0 != n * s1):
            raise ValueError("rows must be evenly spaced with contiguous elements")
        return t.data_ptr(), n, s1

    def _call(self, name: str, *args) -> None:
        _call_on(self.index, name, *args)


def kv4_append(cache: Kv4Cache, k, v) -> None:
    """Stores k, v [n_seq, n_new, n_kv * head_dim] as the last n_new positions of every sequence (lens counts them)."""
    width = cache.n_kv * cache.head_dim
    (pk, n, sk), (pv, nv, sv) = cache._rows(k, width), cache._rows(v, width)
    if n != nv or sk != sv:
        raise ValueError("k and v must have the same rows")
    cache._call("ibh_kv4_append", cache.ref, pk, pv, n, sk)


def kv4_read(cache: Kv4Cache, k, v) -> None:
    """The values of the last k.shape[1] positions of every sequence into k, v [n_seq, n, n_kv * head_dim]."""
    width = cache.n_kv * cache.head_dim
    (pk, n, sk), (pv, nv, sv) = cache._rows(k, width), cache._rows(v, width)
    if n != nv or sk != sv:
        raise ValueError("k and v must have the same rows")
    cache._call("ibh_kv4_read", cache.ref, pk, pv, n, sk)


def kv4_attn(out, q, cache: Kv4Cache, n_heads: int, weights_in=None, weights_out=None, ws=None) -> None:
    """Attention of the last q.shape[1] positions of every sequence: q [n_seq, n_q, n_heads * head_dim] (rows may be
    spaced), out the same, contiguous; weights fp32 [n_seq, n_kv, 64 * max_pages], accumulated from in to out."""
    pq, n_q, sq = cache._rows(q, n_heads * cache.head_dim)
    po = cache._on(out, torch.float32, cache.n_seq * n_q * n_heads * cache.head_dim)
    if (weights_in is None) != (weights_out is None):
        raise ValueError("weights_in and weights_out go together")
    wi = wo = None
    if weights_in is not None:
        size = cache.n_seq * cache.n_kv * cache.max_pages * KV4_PAGE
        wi, wo = (cache._on(w, torch.float32, size) for w in (weights_in, weights_out))
    need = 0 if ws is not None else lib().ibh_kv4_attn_workspace_bytes(cache.ref, n_heads, n_q, wi is not None)
    pw, nw, ws = _scratch(ws, need, cache.index)
    cache._call("ibh_kv4_attn", cache.ref, po, pq, n_heads, n_q, sq, wi, wo, pw, nw)


def kv4_evict(src: Kv4Cache, dst: Kv4Cache, weights_src, weights_dst, budget: int, sink: int, recent: int,
              kept, ws=None) -> None:
    """Cuts every sequence to `budget` positions by accumulated weight: rows, weights and lengths into dst (src itself
    for in place, where no page is shared), the kept positions into kept int32 [n_seq, n_kv, budget]."""
    if dst.index != src.index:
        raise ValueError(f"the caches are on {src.device} and {dst.device}")
    n = src.n_seq * src.n_kv
    pw, nw, ws = _scratch(ws, 0 if ws is not None else lib().ibh_kv4_evict_workspace_bytes(src.ref), src.index)
    src._call("ibh_kv4_evict", src.ref, dst.ref,
              src._on(weights_src, torch.float32, n * src.max_pages * KV4_PAGE),
              src._on(weights_dst, torch.float32, n * dst.max_pages * KV4_PAGE), budget, sink, recent,
              src._on(kept, torch.int32, n * budget), pw, nw)


def add_rmsnorm(y, x, weight, eps: float, delta=None, h=None, q=None, s=None) -> None:
    """The RMS norm of x + delta, rows [B, N] (which may be spaced): y fp32 [B, N] and / or the codes q int8 [B, N] with
    their scales s [B, ceil(N / 128)] for matmul_w4a8_batch; the sum itself into h.  y or h may be x or delta."""
    shape, index, f32 = x.shape, _gpu(x), torch.float32
    if len(shape) != 2 or not shape[1]:
        raise ValueError("x must be [B, N] with N at least 1")
    if (y is None and q is None) or (q is None) != (s is None):
        raise ValueError("y, or q with s, or all three are wanted")
    B, N = shape
    px, sx = _spaced(x, index, shape)
    pd, sd = (None, 0) if delta is None else _spaced(delta, index, shape)
    _call_on(index, "ibh_add_rmsnorm", None if y is None else _on(y, index, f32, shape),
             None if q is None else _on(q, index, torch.int8, shape),
             None if s is None else _on(s, index, f32, (B, (N + 127) // 128)),
             None if h is None else _on(h, index, f32, shape), px, pd, _on(weight, index, f32, (N,)), eps, N, B, sx, sd)


_LORA_KINDS = {torch.float16: 0, torch.bfloat16: 1}


def lora(out, x, a, b, ids, base=None, scales=None, ranks=None, ws=None) -> None:
    """Adds to each row of base [B, M] (None: zeros; may be out) what its adapter makes of its row of x [B, N]:
    out[r] = base[r] + scales[i] * b[i] @ (a[i] @ x[r]), i = ids[r] (int32 [B]; negative: no adapter).  a [n, rank, N]
    and b [n, M, rank] in fp16 or bf16, scales fp32 [n], ranks int32 [n].  Rows of out, base and x may be spaced."""
    dtype, sa, sb = a.dtype, a.shape, b.shape
    if len(sa) != 3 or len(sb) != 3 or x.dim() != 2:
        raise ValueError("a must be [n, rank, N], b [n, M, rank] and x [B, N]")
    (n, R, N), B, M = sa, x.shape[0], sb[1]
    kind = _LORA_KINDS.get(dtype)
    if kind is None:
        raise TypeError(f"adapters must be fp16 or bf16, got {dtype}")
    index = _gpu(x)
    ref = ctypes.byref(LoraDesc(_on(a, index, dtype, sa), _on(b, index, dtype, (n, M, R)),
                                None if scales is None else _on(scales, index, torch.float32, (n,)),
                                None if ranks is None else _on(ranks, index, torch.int32, (n,)), n, R, N, M, kind))
    po, so = _spaced(out, index, (B, M))
    pb, sb = (None, 0) if base is None else _spaced(base, index, (B, M))
    px, sx = _spaced(x, index, (B, N))
    pi = _on(ids, index, torch.int32, (B,))
    pw, nw, ws = _scratch(ws, 0 if ws is not None else lib().ibh_lora_workspace_bytes(ref, B), index)
    _call_on(index, "ibh_lora", ref, po, pb, px, pi, B, so, sb, sx, pw, nw)


def logprobs(out, logits, tokens, entropy=None, top_ids=None, top_logprobs=None, ws=None) -> None:
    """From logits [B, V] (rows may be spaced): the log-probabilities of tokens (int32 [B] or [B, n]; None with out) into
    out of the same shape, the entropy into entropy [B], the k best into top_ids (int32) and top_logprobs [B, k]."""
    index, shape = _gpu(logits), logits.shape
    if len(shape) != 2 or not shape[1]:
        raise ValueError("logits must be [B, V] with V at least 1")
    B, V = shape
    pz, sz = _spaced(logits, index, shape)
    if (out is None) != (tokens is None) or (top_ids is None) != (top_logprobs is None):
        raise ValueError("out and tokens go together, and top_ids and top_logprobs")
    n = k = 0
    po = pt = pi = pl = None
    if tokens is not None:
        st = tokens.shape
        if len(st) not in (1, 2) or st[0] != B:
            raise ValueError(f"tokens must be [{B}] or [{B}, n], got {list(st)}")
        n = 1 if len(st) == 1 else st[1]
        po, pt = _on(out, index, torch.float32, st), _on(tokens, index, torch.int32, st)
    if top_ids is not None:
        sk = top_ids.shape
        if len(sk) != 2 or sk[0] != B:
            raise ValueError("top_ids and top_logprobs must be [B, k]")
        k = sk[1]
        pi, pl = _on(top_ids, index, torch.int32, sk), _on(top_logprobs, index, torch.float32, sk)
    pw, nw, ws = _scratch(ws, 0 if ws is not None else lib().ibh_logprobs_workspace_bytes(V, B, k), index)
    _call_on(index, "ibh_logprobs", po, None if entropy is None else _on(entropy, index, torch.float32, (B,)), pi, pl, pz,
             pt, V, B, sz, n, k, pw, nw)


class PqDeviceTensor:
    """A PQ tensor (ib_pq_tensor layout, src/pq_decode.h:39-87) uploaded to the
    GPU once.  `t` maps the reference field names used by the oracle
    (cb1l, cb1r, cb2l, cb2r, i1l, i1r, i2l, i2r, row_scale, ocols, oside,
    oscale) and sizes (M, N, G, K, K_l2, n_levels, n_outlier, C,
    l2_idx_bytes) to numpy arrays / ints."""

    _MAP = {"cb1l": "codebook_l1_l", "cb1r": "codebook_l1_r", "cb2l": "codebook_l2_l", "cb2r": "codebook_l2_r",
            "i1l": "indices_l1_l", "i1r": "indices_l1_r", "i2l": "indices_l2_l", "i2r": "indices_l2_r",
            "row_scale": "row_scale", "ocols": "outlier_cols", "oside": "outlier_sidecar",
            "oscale": "outlier_scale"}

    def __init__(self, t: dict):
        import torch
        self.keep = []
        s = PqTensor()
        for n in ("M", "N", "G", "K", "n_levels", "n_outlier", "C"):
            setattr(s, n, int(t[n]))
        s.K_l2 = int(t.get("K_l2", 0))
        s.l2_idx_bytes = int(t.get("l2_idx_bytes", 1))
        s.format = int(t.get("format", 0))
        for k, f in self._MAP.items():
            a = t.get(k)
            if a is not None:
                d = torch.from_numpy(np.ascontiguousarray(a).view(np.uint8).reshape(-1).copy()).cuda()
                self.keep.append(d)
                setattr(s, f, d.data_ptr())
        if s.n_outlier > 0:
            mask = np.ones(s.N, bool)
            mask[np.asarray(t["ocols"])] = False
            inner = np.nonzero(mask)[0].astype(np.int32)
            d = torch.from_numpy(inner.view(np.uint8).copy()).cuda()
            self.keep.append(d)
            s.inner_cols = d.data_ptr()
        self.s = s
        self.M = s.M
        # a workspace of its own (tables, slab partials), allocated once
        self.ws = torch.empty(max(1, lib().ibh_pq_workspace_bytes(ctypes.byref(s))), dtype=torch.uint8,
                              device="cuda")
        check(lib().ibh_pq_workspace_init(_ptr(self.ws), self.ws.numel(), _stream()), "ibh_pq_workspace_init")
        self._topk_ws = {}

    def matmul(self, x, out) -> None:
        """ib_pq_matmul_fp32 (src/pq_decode.c:1684)."""
        check(lib().ibh_pq_matmul(ctypes.byref(self.s), _ptr(x), _ptr(out), _ptr(self.ws), self.ws.numel(),
                                  _stream()), "ibh_pq_matmul")

    def matmul_policy(self, x, out, variant: int, skip_threshold: float = 0.0, act_threshold: float = 0.0) -> None:
        """ib_pq_session_matmul with an ib_pq_policy (src/pq_decode.c:4464-4491)."""
        p = PqPolicy(variant, skip_threshold, act_threshold)
        check(lib().ibh_pq_matmul_policy(ctypes.byref(self.s), _ptr(x), _ptr(out), ctypes.byref(p), _ptr(self.ws),
                                         self.ws.numel(), _stream()), "ibh_pq_matmul_policy")

    def matmul_q8lut(self, x, out) -> None:
        """ib_pq_matmul_fp32_q8lut (src/pq_decode.c:2451-2561)."""
        check(lib().ibh_pq_matmul_q8lut(ctypes.byref(self.s), _ptr(x), _ptr(out), _ptr(self.ws), self.ws.numel(),
                                        _stream()), "ibh_pq_matmul_q8lut")

    def lm_head_topk(self, x, k_top: int):
        """ib_pq_lm_head_topk (src/pq_decode.c:2259-2346): (logits [k], ids [k]) on the GPU."""
        need = lib().ibh_pq_topk_workspace_bytes(ctypes.byref(self.s), k_top)
        ws = self._topk_ws.get(k_top)
        if ws is None:
            # prepared once, kept for later calls with the same K_top
            ws = torch.empty(max(1, need), dtype=torch.uint8, device="cuda")
            check(lib().ibh_pq_workspace_init(_ptr(ws), ws.numel(), _stream()), "ibh_pq_workspace_init")
            self._topk_ws[k_top] = ws
        lg = torch.empty(k_top, device="cuda")
        ids = torch.empty(k_top, dtype=torch.int32, device="cuda")
        check(lib().ibh_pq_lm_head_topk(ctypes.byref(self.s), _ptr(x), k_top, _ptr(lg), _ptr(ids), _ptr(ws), need,
                                        _stream()), "ibh_pq_lm_head_topk")
        return lg, ids

    def matmul_streaming(self, x, out) -> None:
        """ib_pq_matmul_fp32_streaming_cached (src/pq_decode.c:2987): every chunk."""
        check(lib().ibh_pq_matmul_streaming(ctypes.byref(self.s), _ptr(x), _ptr(out), _ptr(self.ws),
                                            self.ws.numel(), _stream()), "ibh_pq_matmul_streaming")


class Int4gDeviceTensor:
    """An IBF v5 INT4 group-scale tensor (struct ib_int4_tensor,
    src/pq_decode.c:3474-3482) uploaded to the GPU once.  `t` maps q
    (uint8 [M, N/2]), s (fp16 bits [M, N/G]) and the optional inv_act
    (fp32 [N]), outl_idx / outl_val (uint16 / fp16 bits [M, K_out]) to numpy
    arrays (None or absent = not present)."""

    def __init__(self, t: dict):
        self.keep = []
        s = Int4gTensor()
        q = np.ascontiguousarray(t["q"], np.uint8)
        sc = np.ascontiguousarray(t["s"], np.uint16)
        s.M, s.N = q.shape[0], q.shape[1] * 2
        s.G = s.N // sc.shape[1]
        for f in ("q", "s", "inv_act", "outl_idx", "outl_val"):
            a = t.get(f)
            if a is not None:
                d = torch.from_numpy(np.ascontiguousarray(a).view(np.uint8).reshape(-1).copy()).cuda()
                self.keep.append(d)
                setattr(s, f, d.data_ptr())
        s.K_out = 0 if t.get("outl_idx") is None else int(np.asarray(t["outl_idx"]).shape[1])
        self.s = s
        self.M, self.N = s.M, s.N

    def _here(self) -> None:
        _ptr(self.keep[0])                               # on the current GPU still

    def matmul(self, x, out, act_sparse_rel: float = 0.0) -> None:
        """ib_pq_session_matmul on this tensor (src/pq_decode.c:4442-4452)."""
        self._here()
        check(lib().ibh_int4g_matmul(ctypes.byref(self.s), _ptr(x), _ptr(out), act_sparse_rel, None, 0, _stream()),
              "ibh_int4g_matmul")

    def matmul_batched(self, x, out, act_sparse_rel: float = 0.0) -> None:
        """ib_pq_session_matmul_batched (src/pq_decode.c:4501-4539): x [B, N], out [B, M]."""
        self._here()
        B = x.shape[0]
        check(lib().ibh_int4g_matmul_batched(ctypes.byref(self.s), B, _ptr(x), _ptr(out), act_sparse_rel, None, 0,
                                             _stream()), "ibh_int4g_matmul_batched")
