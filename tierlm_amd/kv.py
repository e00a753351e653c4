"""Attention for a batch of sequences over a paged key-value cache (tlm_hip_kv_*): with fp8.add_rmsnorm,
fp8.matmul and fp8.MoeBlock, a layer of a served batch.

    cache = kv.Cache(n_pages, kv_heads, head_dim, page=64, dtype=torch.bfloat16)     # one a layer
    q = kv.append(cache, qkv, heads, tables, lens, inv_freq=kv.rope_frequencies(head_dim, 1e6))
    y = kv.decode(q, cache, tables, lens)              # one new token a sequence: [B, heads, head_dim]
    y = kv.prompt(q, cache, tables, lens, cu)          # packed rows, causal: [T, heads, head_dim]

Sequence b's position p lies in page tables[b, p // page] (int32 [B, pages]); lens[b] (int32) is its length after
the call's own rows, which are rows cu[b] .. cu[b + 1] - 1 (int32 [B + 1]; without cu, row b).  A length of 0 is a
padded slot: nothing is written, attention gives zeros.  Page numbers outside the cache name no page, and what
lies there is neither written nor seen.  Lengths, bounds and tables are read on the device: a captured
graph follows them.  A result given as `out` lies apart from the rows that the call reads.

Device memory is torch tensors on the current HIP device; work goes on torch's current stream.  Arguments that
do not fit raise ValueError, sizes past a call's limits HipError, before anything is launched.
"""
import ctypes as C
import math

import torch

from ._lib import KvBatch, KvCache, check, lib
from .fp8 import _current_device, _here, _raw_stream, _rows_ok

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_CACHE = {torch.float16: 1, torch.bfloat16: 2}
_I32, _F32, _F64 = torch.int32, torch.float32, torch.float64
_decode_bytes, _prompt_bytes = lib.tlm_hip_kv_decode_workspace_bytes, lib.tlm_hip_kv_prompt_workspace_bytes
_append, _decode, _prompt = lib.tlm_hip_kv_append, lib.tlm_hip_kv_decode, lib.tlm_hip_kv_prompt


class Cache:
    """Keys and values of one layer: n_pages pages of `page` positions (a power of two from 16 to 4096) for
    kv_heads heads of head_dim values (a multiple of 32 up to 256), float16 or bfloat16.

    .k [n_pages, kv_heads, page / 16, head_dim / 16, 16, 16] holds value 16 i + j of the block's position p at
    [..., i, p, j], .v [n_pages, kv_heads, page / 16, head_dim, 16] value d at [..., d, p].  Pages may be copied
    (cache.k[dst] = cache.k[src]); the two tensors themselves stay the cache's.  keys() and values() give pages as
    [kv_heads, positions, head_dim].  The memory is not cleared: a position is read once its sequence's length
    covers it."""

    def __init__(self, n_pages, kv_heads, head_dim, page=64, dtype=torch.bfloat16, device=None):
        if dtype not in _CACHE:
            raise ValueError("dtype must be float16 or bfloat16")
        if n_pages < 1 or kv_heads < 1:
            raise ValueError("a cache has at least one page and one head")
        if head_dim < 32 or head_dim > 256 or head_dim % 32:
            raise ValueError("head_dim must be a multiple of 32 up to 256")
        if page < 16 or page > 4096 or page & (page - 1):
            raise ValueError("page must be a power of two from 16 to 4096")
        if device is None:
            device = torch.device("cuda", torch.cuda.current_device())
        self.n_pages, self.kv_heads, self.head_dim, self.page, self.dtype = n_pages, kv_heads, head_dim, page, dtype
        self._k = torch.empty(n_pages, kv_heads, page // 16, head_dim // 16, 16, 16, dtype=dtype, device=device)
        self._v = torch.empty(n_pages, kv_heads, page // 16, head_dim, 16, dtype=dtype, device=device)
        self._dev = self._k.get_device()
        self._c = KvCache(_CACHE[dtype], kv_heads, head_dim, page, n_pages, self._k.data_ptr(), self._v.data_ptr())
        self._ref = C.byref(self._c)
        self._sizes = {}            # bytes of a workspace by the call's sizes

    @property
    def k(self):
        return self._k

    @property
    def v(self):
        return self._v

    def keys(self, pages):
        """The keys of these pages (a list, or an int tensor), end to end: [kv_heads, positions, head_dim]."""
        k = self.k[torch.as_tensor(pages, device=self.k.device).long()]
        return k.permute(1, 0, 2, 4, 3, 5).reshape(self.kv_heads, -1, self.head_dim)

    def values(self, pages):
        v = self.v[torch.as_tensor(pages, device=self.v.device).long()]
        return v.permute(1, 0, 2, 4, 3).reshape(self.kv_heads, -1, self.head_dim)


def rope_frequencies(head_dim, theta, device=None):
    """theta^(-2 j / head_dim), j < head_dim / 2: the inv_freq (float64) of plain rotary positions."""
    j = torch.arange(head_dim // 2, dtype=_F64)
    return (float(theta) ** (j * (-2.0 / head_dim))).to(torch.device("cuda") if device is None else device)


def _batch(cache, rows, tables, lens, cu, others):
    """The C batch, once its tensors fit."""
    shape, pages = lens.shape, tables.shape
    if len(shape) != 1 or lens.dtype is not _I32 or not lens.is_contiguous():
        raise ValueError("lens must be contiguous int32 [B]")
    B = shape[0]
    if len(pages) != 2 or pages[0] != B or pages[1] < 1 or tables.dtype is not _I32 or not _rows_ok(tables):
        raise ValueError(f"tables must be int32 [{B}, pages] with contiguous rows")
    pages = pages[1]
    pcu = None
    dev = cache._dev
    if cu is None:
        if rows != B:
            raise ValueError(f"{rows} rows for {B} sequences need cu")
    else:
        if cu.shape != (B + 1,) or cu.dtype is not _I32 or not cu.is_contiguous():
            raise ValueError(f"cu must be contiguous int32 [{B + 1}]")
        if cu.get_device() != dev:
            _here(cache.k, cu)
        pcu = cu.data_ptr()
    if dev < 0 or not dev == lens.get_device() == tables.get_device() == _current_device():
        _here(cache.k, lens, tables)
    for t in others:
        if t.get_device() != dev:
            _here(cache.k, t)
    return KvBatch(B, rows, pcu, lens.data_ptr(), tables.data_ptr(), max(tables.stride(0), pages), pages)


def _vector(t, n, dtype, what, dev):
    """The address of a contiguous vector (None: null)."""
    if t is None:
        return None
    if t.shape != (n,) or t.dtype is not dtype or not t.is_contiguous():
        raise ValueError(f"{what} must be contiguous {dtype} [{n}]")
    if t.get_device() != dev:
        raise ValueError(f"{what} is on {t.device}, not on the cache's device")
    return t.data_ptr()


def _apart(out, x, rows, stride, width):
    """Refuses a result that begins or ends among the rows read: other groups may not have read theirs yet."""
    a, b = x.data_ptr(), out.data_ptr()
    if rows and a < b + out.numel() * out.element_size() and b < a + ((rows - 1) * stride + width) * x.element_size():
        raise ValueError("out must not overlap the rows that the call reads")


def append(cache, qkv, heads, tables, lens, cu=None, *, q_norm=None, k_norm=None, eps=1e-6, inv_freq=None,
           rope_scale=1.0, out=None):
    """Rows of q | k | v (float32, float16 or bfloat16 [T, (heads + 2 kv_heads) head_dim], any row stride): norms of
    the query and key heads (q_norm, k_norm: float32 [head_dim]), rotary positions (inv_freq: float64 [head_dim / 2],
    pairs j and j + head_dim / 2), keys and values to their pages.  Returns the queries, [T, heads,
    head_dim] of the cache's dtype."""
    hd, dev, shape = cache.head_dim, cache._dev, qkv.shape
    dt = _TYPES.get(qkv.dtype)
    if heads < 1 or heads % cache.kv_heads:
        raise ValueError(f"heads must be a multiple of the cache's {cache.kv_heads}")
    width = (heads + 2 * cache.kv_heads) * hd
    if dt is None or len(shape) != 2 or shape[1] != width or not _rows_ok(qkv):
        raise ValueError(f"qkv must be float32, float16 or bfloat16 [T, {width}] with contiguous rows")
    T = shape[0]
    pq, pk = _vector(q_norm, hd, _F32, "q_norm", dev), _vector(k_norm, hd, _F32, "k_norm", dev)
    pf = _vector(inv_freq, hd // 2, _F64, "inv_freq", dev)
    if out is None:
        out = cache._k.new_empty((T, heads, hd))
    elif out.shape != (T, heads, hd) or out.dtype is not cache.dtype or not out.is_contiguous() or \
            out.data_ptr() % 16:
        raise ValueError(f"out must be contiguous {cache.dtype} [{T}, {heads}, {hd}], 16-byte aligned")
    else:
        _apart(out, qkv, T, qkv.stride(0), width)
    b = _batch(cache, T, tables, lens, cu, (qkv, out))
    rc = _append(cache._ref, C.byref(b), dt, qkv.data_ptr(), max(qkv.stride(0), width), heads, pq, pk, eps, pf,
                 rope_scale, out.data_ptr(), _raw_stream(dev))
    if rc:
        check(rc)
    return out


def _queries(q, cache, scale, out, dtype):
    """Row stride and heads of q, the scale and the result."""
    shape = q.shape
    if q.dtype is not cache.dtype or len(shape) != 3 or shape[2] != cache.head_dim:
        raise ValueError(f"q must be {cache.dtype} [T, heads, {cache.head_dim}]")
    T, heads, hd = shape
    if heads < 1 or heads % cache.kv_heads:
        raise ValueError(f"q's heads must be a multiple of the cache's {cache.kv_heads}")
    stride = heads * hd
    if not q.is_contiguous():
        s0, s1, s2 = q.stride()
        if s2 != 1 or (s1 != hd and heads > 1) or (s0 < stride and T > 1):
            raise ValueError("q's heads must lie side by side in rows that do not overlap")
        stride = max(s0, stride)
    if scale is None:
        scale = 1.0 / math.sqrt(hd)
    elif not 0.0 < scale < math.inf:
        raise ValueError("scale must be finite and positive")
    if out is None:
        if dtype is None:
            out = q.new_empty(shape)
        elif dtype in _TYPES:
            out = q.new_empty(shape, dtype=dtype)
        else:
            raise ValueError("dtype must be float32, float16 or bfloat16")
    elif out.shape != shape or out.dtype not in _TYPES or not out.is_contiguous():
        raise ValueError(f"out must be contiguous float32, float16 or bfloat16 {tuple(shape)}")
    else:
        _apart(out, q, T, stride, heads * hd)
    return T, stride, heads, scale, out


def _workspace(cache, q, call, ref, key):
    """A call's own workspace (None: it needs none) from torch's allocator, which orders its reuse on the stream."""
    nbytes = cache._sizes.get(key)
    if nbytes is None:
        if len(cache._sizes) >= 4096:
            cache._sizes.clear()
        nbytes = cache._sizes[key] = call(cache._ref, ref, key[1])
    return q.new_empty(nbytes, dtype=torch.uint8) if nbytes else None


def decode(q, cache, tables, lens, *, scale=None, out=None, dtype=None):
    """Attention of one new token a sequence: q [B, heads, head_dim] of the cache's dtype (rows of any stride) over
    the lens[b] positions of sequence b -> [B, heads, head_dim] of `dtype` (q's without it).  scale: 1 /
    sqrt(head_dim) without it."""
    T, stride, heads, scale, out = _queries(q, cache, scale, out, dtype)
    b = _batch(cache, T, tables, lens, None, (q, out))
    ref = C.byref(b)
    ws = _workspace(cache, q, _decode_bytes, ref, (T, heads, b.table_pages))
    rc = _decode(cache._ref, ref, q.data_ptr(), stride, heads, scale, _TYPES[out.dtype], out.data_ptr(),
                 None if ws is None else ws.data_ptr(), _raw_stream(cache._dev))
    if rc:
        check(rc)
    return out


def prompt(q, cache, tables, lens, cu, *, scale=None, out=None, dtype=None):
    """Causal attention of packed rows: row i of sequence b's n sees its positions up to lens[b] - n + i, cached
    ones included.  q [T, heads, head_dim] -> [T, heads, head_dim]; rows outside cu's are left as they are."""
    T, stride, heads, scale, out = _queries(q, cache, scale, out, dtype)
    b = _batch(cache, T, tables, lens, cu, (q, out))
    ref = C.byref(b)
    ws = _workspace(cache, q, _prompt_bytes, ref, (T, heads, b.table_pages, b.B))
    rc = _prompt(cache._ref, ref, q.data_ptr(), stride, heads, scale, _TYPES[out.dtype], out.data_ptr(),
                 None if ws is None else ws.data_ptr(), _raw_stream(cache._dev))
    if rc:
        check(rc)
    return out
