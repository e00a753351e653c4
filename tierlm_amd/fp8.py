"""8-bit floating point on device tensors: E4M3 matrices with a scale per 128 x
128 block (the reference's FP8 weights, src/lib/tlm_quant.c:761-776), the
activation quantiser, their product, and a routed MoE block for a few tokens
(tlm_hip_fp8_*).

    Wp = fp8.pack(W, scale)                  # once: W [rows, n] float8_e4m3fn, scale [rows/128, n/128]
    codes, s = fp8.quantize(x)               # x [T, n] float32, float16 or bfloat16
    Y = fp8.matmul(Wp, rows, n, codes, s)    # [T, rows]

Device memory is torch tensors on the current HIP device; work goes on torch's
current stream.  Arguments that do not fit raise ValueError before anything
is launched.
"""
import ctypes as C

import torch

from ._lib import MoeDesc, check, lib
from .quant import _ptr, stream

FP8 = 100                       # TLM_HIP_DT_FP8
BLOCK = 128
MOE_MAX_TOKENS = 64             # TLM_HIP_FP8_MOE_MAX_TOKENS
E4M3 = torch.float8_e4m3fn
_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def _blocks(n):
    return -(-n // BLOCK)


def _want(ok, what):
    if not ok:
        raise ValueError(what)


def _on_device(*tensors):
    for t in tensors:
        _want(t.is_cuda and t.device.index == torch.cuda.current_device(),
              f"a tensor is on {t.device}, not on the current HIP device")


def _out(t, shape, dtype, like, what):
    if t is None:
        return torch.empty(shape, dtype=dtype, device=like.device)
    _want(tuple(t.shape) == tuple(shape) and t.dtype == dtype and t.is_contiguous(),
          f"{what} must be a contiguous {dtype} tensor of shape {tuple(shape)}")
    return t


def packed_bytes(rows, n):
    return int(lib.tlm_hip_fp8_packed_bytes(rows, n))


def pack(W, scale, out=None):
    """E4M3 rows W [rows, n] (float8_e4m3fn or uint8 codes, any row stride) and
    f32 scales [rows / 128, n / 128] (rounded up) -> the packed matrix (uint8)."""
    _want(W.dim() == 2 and W.dtype in (E4M3, torch.uint8) and W.numel() > 0 and (W.shape[1] == 1 or W.stride(1) == 1),
          "W must be a 2-D float8_e4m3fn or uint8 tensor with contiguous rows")
    rows, n = W.shape
    _want(tuple(scale.shape) == (_blocks(rows), _blocks(n)) and scale.dtype == torch.float32 and
          (scale.shape[1] == 1 or scale.stride(1) == 1),
          f"scale must be float32 [{_blocks(rows)}, {_blocks(n)}] with contiguous rows")
    rb, ss = (W.stride(0) if rows > 1 else n), (scale.stride(0) if scale.shape[0] > 1 else _blocks(n))
    _want(rb >= n and ss >= _blocks(n), "rows of W or scale overlap")
    out = _out(out, (packed_bytes(rows, n),), torch.uint8, W, "out")
    _on_device(W, scale, out)
    check(lib.tlm_hip_fp8_pack(_ptr(W), rb, _ptr(scale), ss, rows, n, _ptr(out), stream()))
    return out


def quantize(x, codes=None, scale=None):
    """x [T, n] (or [n]) -> E4M3 codes [T, np] and f32 scales [T, np / 128], np
    = n rounded up to 128; rows of x may have any stride."""
    x = x[None] if x.dim() == 1 else x
    _want(x.dim() == 2 and x.dtype in _TYPES and x.shape[1] > 0 and (x.shape[1] == 1 or x.stride(1) == 1),
          "x must be float32, float16 or bfloat16 [T, n] with contiguous rows")
    T, n = x.shape
    xs = x.stride(0) if T > 1 else n
    _want(xs >= n, "rows of x overlap")
    codes = _out(codes, (T, _blocks(n) * BLOCK), E4M3, x, "codes")
    scale = _out(scale, (T, _blocks(n)), torch.float32, x, "scale")
    _on_device(x, codes, scale)
    check(lib.tlm_hip_fp8_quantize(_TYPES[x.dtype], _ptr(x), xs, n, T, _ptr(codes), _ptr(scale), stream()))
    return codes, scale


def matmul(Wp, rows, n, codes, scale, out=None, dtype=torch.float32):
    """Y[t, r] = packed row r . token t: codes [T, np] and scale [T, np / 128] as
    quantize() gives them; Y [T, rows] of `dtype`, or `out` (rows of any stride)."""
    _want(rows > 0 and n > 0 and Wp.dtype == torch.uint8 and Wp.is_contiguous() and Wp.numel() >= packed_bytes(rows, n),
          f"Wp is not a packed matrix of {rows} x {n}")
    _want(codes.dim() == 2 and codes.dtype in (E4M3, torch.uint8) and codes.is_contiguous() and
          codes.shape[1] == _blocks(n) * BLOCK, f"codes must be contiguous E4M3 [T, {_blocks(n) * BLOCK}]")
    T = codes.shape[0]
    _want(tuple(scale.shape) == (T, _blocks(n)) and scale.dtype == torch.float32 and scale.is_contiguous(),
          f"scale must be contiguous float32 [{T}, {_blocks(n)}]")
    if out is None:
        _want(dtype in _TYPES, "dtype must be float32, float16 or bfloat16")
        out = torch.empty((T, rows), dtype=dtype, device=Wp.device)
    _want(tuple(out.shape) == (T, rows) and out.dtype in _TYPES and (rows == 1 or out.stride(1) == 1),
          f"out must be float32, float16 or bfloat16 [{T}, {rows}] with contiguous rows")
    ys = out.stride(0) if T > 1 else rows
    _want(ys >= rows, "rows of out overlap")
    _on_device(Wp, codes, scale, out)
    check(lib.tlm_hip_fp8_matmul(_ptr(Wp), rows, n, _ptr(codes), _ptr(scale), T, _TYPES[out.dtype], _ptr(out), ys,
                                 stream()))
    return out


class MoeBlock:
    """One routed MoE block of E4M3 matrices for up to 64 tokens a call.  Expert
    e's packed gate / up / down pointers are expert_ptrs[3e .. 3e + 2]; packed
    matrices are the caller's to keep alive, as are the tensors a call is given.
    The workspace grows to the largest T seen and is one per block, so calls of
    one block must not overlap (other streams); a block captured into a graph has to
    run once with its largest T before."""

    def __init__(self, *, D, de, E, k, ffn_norm, router_w, expert_ptrs, router=0, routed_scale=1.0, eps=1e-6,
                 router_bias=None, mask=None, ds=0, shared=None, shared_gate_inp=None):
        _want(len(expert_ptrs) == 3 * E and all(expert_ptrs), "expert_ptrs must hold 3 E packed matrices")
        _want((ds > 0) == (shared is not None), "ds and shared go together")
        for t, shape, dt, what in ((ffn_norm, (D,), torch.float32, "ffn_norm"),
                                   (router_w, (E, D), torch.float32, "router_w"),
                                   (router_bias, (E,), torch.float32, "router_bias"), (mask, (E,), torch.uint8, "mask"),
                                   (shared_gate_inp, (D,), torch.float32, "shared_gate_inp")):
            _want(t is None or (tuple(t.shape) == shape and t.dtype == dt and t.is_contiguous()),
                  f"{what} must be a contiguous {dt} tensor of shape {shape}")
            if t is not None:
                _on_device(t)
        if shared is not None:
            _want(len(shared) == 3 and all(m.numel() >= packed_bytes(*rn) for m, rn in
                                           zip(shared, ((ds, D), (ds, D), (D, ds)))), "shared must be 3 packed matrices")
            _on_device(*shared)
        self.keep = [ffn_norm, router_w, router_bias, mask, shared, shared_gate_inp]
        self.device = ffn_norm.device
        self.table = torch.tensor(list(expert_ptrs), dtype=torch.int64, device=self.device)

        def p(t):
            return t.data_ptr() if t is not None else None

        sg, su, sd = shared if shared is not None else (None, None, None)
        self.desc = MoeDesc(D, de, ds, E, k, router, routed_scale, eps, FP8, FP8, p(ffn_norm), p(router_w),
                            p(router_bias), p(mask), self.table.data_ptr(), p(sg), p(su), p(sd), p(shared_gate_inp))
        check(lib.tlm_hip_fp8_moe(C.byref(self.desc), None, None, 0, None, None, None, None))   # the sizes fit
        self.workspace, self._room = None, 0

    def reserve(self, T):
        """Make the workspace large enough for T tokens."""
        if T > self._room:
            nbytes = int(lib.tlm_hip_fp8_moe_workspace_bytes(C.byref(self.desc), T))
            if not nbytes:
                check(lib.tlm_hip_fp8_moe(C.byref(self.desc), None, None, T, None, None, None, None))
            self.workspace = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
            self._room = T

    def __call__(self, h, out=None, ids=None, w=None):
        """out = h + MoE(h) for h (f32 [T, D] or [D]), T <= 64; without `out` h itself
        is updated.  ids (int32) / w (f32), [T, k], receive the routing.  Returns
        out."""
        D, k = self.desc.D, self.desc.k
        T = h.numel() // D
        _want(h.dtype == torch.float32 and h.is_contiguous() and h.dim() in (1, 2) and h.shape[-1] == D,
              f"h must be contiguous float32 [T, {D}]")
        out = h if out is None else _out(out, h.shape, torch.float32, h, "out")
        _on_device(h, out)
        for t, dt, what in ((ids, torch.int32, "ids"), (w, torch.float32, "w")):
            if t is not None:
                _out(t, (T, k), dt, h, what)
                _on_device(t)
        self.reserve(T)
        check(lib.tlm_hip_fp8_moe(C.byref(self.desc), _ptr(h), _ptr(out), T, _ptr(ids), _ptr(w),
                                  _ptr(self.workspace), stream()))
        return out
