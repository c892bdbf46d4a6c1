"""Operators on a layer's KV cache (include/hoard_cache.h): attention of a tree of drafted tokens, attention that
accumulates its weights, eviction by those weights, attention over blocks of the cache that a score selects.

`CacheOps` holds the head layout, the workspace and the C descriptor for caches of one shape; its methods keep the C
names and take torch CUDA tensors. Caches are [max_rows][n_head_kv][head_dim] tensors of f16 or bf16, of any row and
head strides that are multiples of 8 elements (a [n_head_kv][max_rows][head_dim] buffer passes as its transpose).
Wrong tensors raise ValueError, refused arguments HoardError; nothing is launched then. One CacheOps is driven by one
host thread at a time, and its calls share one workspace: calls on streams that may overlap, captured graphs among
them, need a CacheOps each. A CacheOps may be dropped while calls on any stream run (its workspace is given back when they have
completed), but not before a graph that captured its calls, and a stream that is not torch's own has to outlive it.
A result that a call allocates belongs to the stream of the call; `out` may be `q` itself.
"""
from __future__ import annotations

import ctypes
import math
import struct

import torch

from hoard_b200.moe import HoardError, _ptr, lib

MAX_TOKENS = 64         # query tokens of one call (HOARD_KV_MAX_TOKENS)
KV_TYPES = {torch.float16: 1, torch.bfloat16: 30}


class Desc(ctypes.Structure):
    """hoard_kv_desc"""
    _fields_ = [("n_head", ctypes.c_int), ("n_head_kv", ctypes.c_int), ("head_dim", ctypes.c_int),
                ("kv_type", ctypes.c_int), ("max_rows", ctypes.c_int), ("max_tokens", ctypes.c_int),
                ("max_acc_tokens", ctypes.c_int), ("block", ctypes.c_int), ("row_stride", ctypes.c_int64),
                ("head_stride", ctypes.c_int64), ("scale", ctypes.c_float)]


# hoard_kv_query: q and its token and head strides, k_cache, v_cache, visible, gate and its strides, out, m, n_past,
# n_past_dev
_QUERY = struct.Struct("@PqqPPPPqqPiiP")
_raw_stream, _current_device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice
_F32, _NO_STRIDE = torch.float32, (0, 0)
_bound = False


def _kv():
    global _bound
    L = lib()
    if not _bound:
        vp, i32, i64, f32 = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float
        L.hoard_kv_ws_bytes.argtypes = [vp]
        L.hoard_kv_ws_bytes.restype = i64
        L.hoard_kv_attention.argtypes = [vp, vp, vp, vp, vp]
        L.hoard_kv_evict.argtypes = [vp, vp, vp, vp, vp, i32, i32, i32, i32, vp, vp, vp, vp]
        L.hoard_kv_block_bounds.argtypes = [vp, vp, vp, i32, i32, vp, vp]
        L.hoard_kv_block_attention.argtypes = [vp, vp, vp, i32, i32, i32, vp, vp, vp]
        L.hoard_kv_take.argtypes = [vp, vp, vp, i32, vp, i32, vp]
        L.hoard_kv_store.argtypes = [vp, vp, i64, i64, vp, vp, vp, vp, i32, f32, i32, f32, vp, i32, i32, vp, vp, vp, vp,
                                     vp, vp, vp]
        _bound = True
    return L


def tree_visibility(parents):
    """parents[i]: the drafted token that token i follows (an earlier index), or -1 for the last token of the past.
    Returns (words, depths): words[i] has bit j set where token j is i itself or one of its ancestors -- as Python
    integers in the signed 64-bit range that torch.int64 holds -- and depths[i] = 0 for a token that follows the past."""
    if not 1 <= len(parents) <= MAX_TOKENS:
        raise ValueError(f"a tree has 1..{MAX_TOKENS} tokens")
    words, depths = [], []
    for i, p in enumerate(parents):
        if not -1 <= p < i:
            raise ValueError(f"parents[{i}] = {p}: a parent is an earlier token or -1")
        words.append((words[p] if p >= 0 else 0) | 1 << i)
        depths.append(depths[p] + 1 if p >= 0 else 0)
    return [w - (1 << 64) if w >> 63 else w for w in words], depths


def _ints(*values):
    """Refuses what C's int does not hold (ctypes would cut it off)."""
    if min(values) < -2**31 or max(values) >= 2**31:
        raise ValueError(f"{values} are not all ints of 32 bits")


class CacheOps:
    """The cache operators for one head layout and cache shape on one device.

    max_tokens: most query tokens of a call (1..64). max_acc_tokens: most query tokens of a call that accumulates
    weights. block: rows of a block for block_bounds / block_attention (16, 32, 64, 128; 0: not used). scale: of the
    scores, 1 / sqrt(head_dim) by default."""

    def __init__(self, *, n_head: int, n_head_kv: int, head_dim: int, kv_dtype: torch.dtype, max_rows: int,
                 max_tokens: int = 1, max_acc_tokens: int = 1, block: int = 0, scale: float | None = None,
                 device: int | None = None):
        if kv_dtype not in KV_TYPES:
            raise ValueError("kv_dtype must be torch.float16 or torch.bfloat16")
        if head_dim < 1:
            raise ValueError("head_dim must be positive")
        self.n_head, self.n_head_kv, self.head_dim, self.kv_dtype = n_head, n_head_kv, head_dim, kv_dtype
        self.max_rows, self.max_tokens, self.block = max_rows, max_tokens, block
        self._d = Desc(n_head, n_head_kv, head_dim, KV_TYPES[kv_dtype], max_rows, max_tokens, max_acc_tokens, block, 0, 0,
                       1.0 / math.sqrt(head_dim) if scale is None else scale)
        self._q = ctypes.create_string_buffer(_QUERY.size)
        # pointers that stay, as ctypes takes them fastest
        self._dp, self._qp = (ctypes.c_void_p(ctypes.addressof(x)) for x in (self._d, self._q))
        self._cache_shape, self._cache_stride = (max_rows, n_head_kv, head_dim), None
        n = _kv().hoard_kv_ws_bytes(self._dp)
        if n < 0:
            raise HoardError(-1, "hoard_kv_ws_bytes: descriptor refused")
        self.device = torch.cuda.current_device() if device is None else device
        self._ws = torch.empty(n, dtype=torch.uint8, device=torch.device("cuda", self.device))
        self._wsp = ctypes.c_void_p(self._ws.data_ptr())
        # the workspace belongs to the stream that is current now; the others that calls ran on
        self._home, self._streams = _raw_stream(self.device), set()

    # ---- plumbing ----
    # The checks read each attribute of a tensor once: at the sizes of a decode step they are a good part of a call.
    def _run(self, fn, stream, *args):
        """fn(*args, stream) on this object's device."""
        if _current_device() != self.device:
            with torch.cuda.device(self.device):
                return self._run(fn, stream, *args)
        raw = _raw_stream(self.device) if stream is None else getattr(stream, "cuda_stream", stream)
        if raw != self._home and raw not in self._streams:
            self._ws.record_stream(torch.cuda.ExternalStream(raw if raw != 1 else 0, device=self._ws.device))      # 1: cudaStreamLegacy
            self._streams.add(raw)
        rc = fn(*args, raw)
        if rc != 0:
            raise HoardError(rc, f"{fn.__name__} failed ({lib().hoard_strerror(rc).decode()})")

    def _new(self, shape, stream):
        """A float32 tensor of the call's stream."""
        if stream is None:
            return torch.empty(shape, dtype=_F32, device=self._ws.device)
        if not hasattr(stream, "cuda_stream"):
            stream = torch.cuda.ExternalStream(stream, device=self._ws.device)
        with torch.cuda.stream(stream):
            return torch.empty(shape, dtype=_F32, device=self._ws.device)

    def _caches(self, k_cache, v_cache=None):
        """Checks the caches and sets the descriptor's strides to theirs."""
        s, dev = k_cache.stride(), self.device
        if (k_cache.shape != self._cache_shape or k_cache.dtype is not self.kv_dtype or k_cache.get_device() != dev
                or s[2] != 1):
            raise ValueError(f"caches are {list(self._cache_shape)} {self.kv_dtype} tensors on device {dev} with "
                             "contiguous heads")
        if v_cache is not None and (v_cache.shape != self._cache_shape or v_cache.dtype is not self.kv_dtype
                                    or v_cache.get_device() != dev or v_cache.stride() != s):
            raise ValueError("the V cache has the K cache's shape, type, device and strides")
        if s != self._cache_stride:
            if not s[0] or not s[1]:               # expanded: its rows or heads are the same memory
                raise ValueError("caches have a row and a head of memory for each of theirs")
            self._d.row_stride, self._d.head_stride = s[0], s[1]
            self._cache_stride = s

    def _heads(self, x, shape, what):
        """Strides of a float32 [m][n_head][head_dim] tensor with contiguous heads."""
        s = x.stride()
        if x.shape != shape or x.dtype is not torch.float32 or x.get_device() != self.device or s[2] != 1:
            raise ValueError(f"{what} is a {list(shape)} float32 tensor on device {self.device} with contiguous heads")
        return s

    def _contiguous(self, x, shape, dtype, what):
        if x.shape != shape or x.dtype is not dtype or x.get_device() != self.device or not x.is_contiguous():
            raise ValueError(f"{what} is a contiguous {list(shape)} {dtype} tensor on device {self.device}")
        return x.data_ptr()

    def _query(self, q, k_cache, v_cache, n_past, vis, gate, out, n_past_dev, stream):
        dev, shape, qs, ks = self.device, q.shape, q.stride(), k_cache.stride()
        if (len(qs) != 3 or shape[1] != self.n_head or shape[2] != self.head_dim or q.dtype is not _F32
                or q.get_device() != dev or qs[2] != 1):
            raise ValueError(f"q is a [m, {self.n_head}, {self.head_dim}] float32 tensor on device {dev} with contiguous heads")
        if ks != self._cache_stride or k_cache.shape != self._cache_shape or k_cache.dtype is not self.kv_dtype or \
                k_cache.get_device() != dev or v_cache.stride() != ks or v_cache.shape != self._cache_shape or \
                v_cache.dtype is not self.kv_dtype or v_cache.get_device() != dev:
            self._caches(k_cache, v_cache)
        m = shape[0]
        if gate is None:
            gp, gs = 0, _NO_STRIDE
        else:
            gs = self._heads(gate, shape, "gate")
            gp = gate.data_ptr()
        if out is None:
            out = self._new(shape, stream)
        elif out.shape != shape or out.dtype is not _F32 or out.get_device() != dev or not out.is_contiguous():
            raise ValueError(f"out is a contiguous {list(shape)} float32 tensor on device {dev}")
        try:
            _QUERY.pack_into(self._q, 0, q.data_ptr(), qs[0], qs[1], k_cache.data_ptr(), v_cache.data_ptr(),
                             0 if vis is None else self._contiguous(vis, (m,), torch.int64, "vis"), gp, gs[0], gs[1],
                             out.data_ptr(), m, n_past,
                             0 if n_past_dev is None else self._contiguous(n_past_dev, (1,), torch.int32, "n_past_dev"))
        except struct.error:
            raise ValueError(f"n_past {n_past} is not an int of 32 bits") from None
        return out

    # ---- attention ----
    def tree_attention(self, q, k_cache, v_cache, n_past: int = 0, *, vis=None, gate=None, acc=None, out=None,
                       n_past_dev=None, stream=None):
        """hoard_kv_attention: q [m][n_head][head_dim] over the past rows and the tokens' own rows n_past..n_past+m-1.
        vis (int64 [m], see tree_visibility): which own rows a token sees; None: those of tokens up to itself. gate: the
        output times sigmoid(gate). acc (float32 [n_head_kv][max_rows]) gets the weights added. n_past_dev (int32 [1]):
        n_past in device memory. Returns out [m][n_head][head_dim]."""
        out = self._query(q, k_cache, v_cache, n_past, vis, gate, out, n_past_dev, stream)
        accp = None if acc is None else self._contiguous(acc, (self.n_head_kv, self.max_rows), torch.float32, "acc")
        self._run(_kv().hoard_kv_attention, stream, self._dp, self._qp, accp, self._wsp)
        return out

    def block_bounds(self, k_cache, bounds, row0: int = 0, row1: int = 0, *, row1_dev=None, stream=None):
        """hoard_kv_block_bounds: minimum and maximum of the keys of the complete blocks that end in (row0, row1], into
        bounds [n_head_kv][max_rows // block][2][head_dim]; row1_dev (int32 [1]): those of row *row1_dev alone."""
        self._caches(k_cache)
        p = self._bounds(bounds)
        _ints(row0, row1)
        d = None if row1_dev is None else self._contiguous(row1_dev, (1,), torch.int32, "row1_dev")
        self._run(_kv().hoard_kv_block_bounds, stream, self._dp, k_cache.data_ptr(), p, row0, row1, d)
        return bounds

    def _bounds(self, bounds):
        if not self.block:
            raise ValueError("this CacheOps was created without blocks (block=16, 32, 64 or 128)")
        return self._contiguous(bounds, (self.n_head_kv, self.max_rows // self.block, 2, self.head_dim), self.kv_dtype,
                                "bounds")

    def block_attention(self, q, k_cache, v_cache, bounds, n_past: int = 0, *, n_sink: int, n_local: int, n_sel: int,
                        vis=None, gate=None, out=None, sel_out=None, n_past_dev=None, stream=None):
        """hoard_kv_block_attention: tree_attention over the first n_sink and last n_local blocks of the past and the
        n_sel others with the largest score, chosen for each token and KV head. sel_out (int32 [m][n_head_kv][n_sel]),
        if given, receives the chosen blocks, ascending, then -1."""
        bp = self._bounds(bounds)
        out = self._query(q, k_cache, v_cache, n_past, vis, gate, out, n_past_dev, stream)
        _ints(n_sink, n_local, n_sel)
        sp = None if sel_out is None else self._contiguous(sel_out, (q.shape[0], self.n_head_kv, n_sel), torch.int32,
                                                           "sel_out")
        self._run(_kv().hoard_kv_block_attention, stream, self._dp, self._qp, bp, n_sink, n_local, n_sel, sp, self._wsp)
        return out

    # ---- rows ----
    def evict(self, k_cache, v_cache, acc, row_pos, n_rows: int, n_keep: int, *, n_sink: int = 0,
              recent_from: int = 2**31 - 1, acc_out=None, pos_out=None, stream=None):
        """hoard_kv_evict: keeps n_keep of the n_rows rows of each KV head in rows 0..n_keep-1: those at positions below
        n_sink or from recent_from on, then those of the largest acc. acc, row_pos: [n_head_kv][max_rows]; updated in
        place, or written to acc_out / pos_out."""
        self._caches(k_cache, v_cache)
        _ints(n_rows, n_keep, n_sink, recent_from)
        shape = (self.n_head_kv, self.max_rows)
        ap = self._contiguous(acc, shape, torch.float32, "acc")
        pp = self._contiguous(row_pos, shape, torch.int32, "row_pos")
        ao = ap if acc_out is None else self._contiguous(acc_out, shape, torch.float32, "acc_out")
        po = pp if pos_out is None else self._contiguous(pos_out, shape, torch.int32, "pos_out")
        self._run(_kv().hoard_kv_evict, stream, self._dp, k_cache.data_ptr(), v_cache.data_ptr(), ap, pp, n_rows, n_keep,
                  n_sink, recent_from, ao, po, self._wsp)

    def take(self, k_cache, v_cache, row0: int, path, stream=None):
        """hoard_kv_take: rows row0 + path[i] to rows row0 + i (path ascending): the accepted path of a drafted tree."""
        self._caches(k_cache, v_cache)
        n = len(path)
        _ints(row0, *path)
        self._run(_kv().hoard_kv_take, stream, self._dp, k_cache.data_ptr(), v_cache.data_ptr(), row0,
                  (ctypes.c_int32 * max(1, n))(*path), n)

    def store(self, q, k, v, k_cache, v_cache, pos, row0: int = 0, *, q_norm=None, k_norm=None, mode: int = 0,
              eps: float = 1e-6, rope_dim: int | None = None, freq_base: float = 1e4, q_out=None, row0_dev=None, acc=None,
              row_pos=None, stream=None):
        """hoard_kv_store: QK norm and RoPE of m tokens' q [m][n_head][head_dim] and k, at positions pos (int32 [m]), and
        their k, v [m][n_head_kv][head_dim] into cache rows row0.. (row0_dev: in device memory). Returns the rotated q."""
        m = q.shape[0]
        _ints(row0, mode)
        shape, kshape = (m, self.n_head, self.head_dim), (m, self.n_head_kv, self.head_dim)
        qs = self._heads(q, shape, "q")
        self._caches(k_cache, v_cache)
        kp, vp = (self._contiguous(x, kshape, torch.float32, w) for x, w in ((k, "k"), (v, "v")))
        if q_out is None:
            q_out = self._new(shape, stream)
        qo = self._contiguous(q_out, shape, torch.float32, "q_out")
        if mode in (1, 2):
            full = mode == 1
            for x, heads, what in ((q_norm, self.n_head, "q_norm"), (k_norm, self.n_head_kv, "k_norm")):
                if x is None:
                    raise ValueError(f"mode {mode} needs {what}")
                self._contiguous(x, ((heads if full else 1) * self.head_dim,), torch.float32, what)
        pp = self._contiguous(pos, (m,), torch.int32, "pos")
        rd = None if row0_dev is None else self._contiguous(row0_dev, (1,), torch.int32, "row0_dev")
        side = (self.n_head_kv, self.max_rows)
        ap = None if acc is None else self._contiguous(acc, side, torch.float32, "acc")
        rp = None if row_pos is None else self._contiguous(row_pos, side, torch.int32, "row_pos")
        self._run(_kv().hoard_kv_store, stream, self._dp, q.data_ptr(), qs[0], qs[1], kp, vp, _ptr(q_norm),
                  _ptr(k_norm), mode, eps, self.head_dim if rope_dim is None else rope_dim, freq_base, pp, m, row0, rd, qo,
                  k_cache.data_ptr(), v_cache.data_ptr(), ap, rp)
        return q_out
