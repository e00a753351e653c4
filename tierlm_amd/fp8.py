"""8-bit floating point on device tensors: E4M3 matrices with a scale per 128 x
128 block (the reference's FP8 weights, src/lib/tlm_quant.c:761-776), the
activation quantiser, their product, and a routed MoE block for a few tokens
(tlm_hip_fp8_*).

    Wp = fp8.pack(W, scale)                  # once: W [rows, n] float8_e4m3fn, scale [rows/128, n/128]
    codes, s = fp8.quantize(x)               # x [T, n] float32, float16 or bfloat16
    Y = fp8.matmul(Wp, rows, n, codes, s)    # [T, rows]

Device memory is torch tensors on the current HIP device; work goes on torch's
current stream.  Arguments that do not fit raise ValueError, sizes past a
call's limits and misaligned memory HipError, before anything is launched.
"""
import ctypes as C

import torch

from ._lib import MoeDesc, check, lib

FP8 = 100                       # TLM_HIP_DT_FP8
BLOCK = 128
MOE_MAX_TOKENS = 64             # TLM_HIP_FP8_MOE_MAX_TOKENS
E4M3 = torch.float8_e4m3fn
_CODES = (E4M3, torch.uint8)
_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_U8, _I32, _F32 = torch.uint8, torch.int32, torch.float32
_pack, _quantize, _matmul, _moe = (lib.tlm_hip_fp8_pack, lib.tlm_hip_fp8_quantize, lib.tlm_hip_fp8_matmul,
                                   lib.tlm_hip_fp8_moe)
_packed_bytes = lib.tlm_hip_fp8_packed_bytes
_raw_stream, _current_device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice


def _blocks(n):
    return -(-n // BLOCK)


def _here(*tensors):
    """The current device's index, on which all the tensors must be."""
    dev = tensors[0].get_device()
    if dev < 0 or dev != _current_device():
        raise ValueError(f"a tensor is on {tensors[0].device}, not on the current HIP device")
    for t in tensors:
        if t.get_device() != dev:
            raise ValueError(f"a tensor is on {t.device}, not on the current HIP device")
    return dev


def _rows_ok(t):
    """2-D with contiguous rows that do not overlap (any row stride)."""
    if t.dim() != 2:
        return False
    if t.is_contiguous():
        return True
    s0, s1 = t.stride()
    rows, n = t.shape
    return (s1 == 1 or n == 1) and (s0 >= n or rows <= 1)


def _out(t, shape, dtype, like, what):
    if t is None:
        return like.new_empty(shape, dtype=dtype)
    if t.shape != shape or t.dtype != dtype or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous {dtype} tensor of shape {tuple(shape)}")
    return t


def packed_bytes(rows, n):
    return int(_packed_bytes(rows, n))


def pack(W, scale, out=None):
    """E4M3 rows W [rows, n] (float8_e4m3fn or uint8 codes, any row stride) and
    f32 scales [rows / 128, n / 128] (rounded up) -> the packed matrix (uint8)."""
    if W.dtype not in _CODES or not _rows_ok(W) or W.numel() == 0:
        raise ValueError("W must be a 2-D float8_e4m3fn or uint8 tensor with contiguous rows")
    rows, n = W.shape
    nr, nb = -(-rows // BLOCK), -(-n // BLOCK)
    if scale.shape != (nr, nb) or scale.dtype is not _F32 or not _rows_ok(scale):
        raise ValueError(f"scale must be float32 [{nr}, {nb}] with contiguous rows")
    dev = W.get_device()
    if dev < 0 or not dev == scale.get_device() == _current_device():
        _here(W, scale)
    if out is None:
        out = W.new_empty(_packed_bytes(rows, n), dtype=_U8)
    elif _out(out, (_packed_bytes(rows, n),), _U8, W, "out").get_device() != dev or out.data_ptr() % 16:
        raise ValueError("out must be on the current HIP device, 16-byte aligned")
    rc = _pack(W.data_ptr(), max(W.stride(0), n), scale.data_ptr(), max(scale.stride(0), nb), rows, n, out.data_ptr(),
               _raw_stream(dev))
    if rc:
        check(rc)
    return out


def quantize(x, codes=None, scale=None):
    """x [T, n] (or [n]) -> E4M3 codes [T, np] and f32 scales [T, np / 128], np
    = n rounded up to 128; rows of x may have any stride.  At most 2^26 blocks of
    128 a call."""
    if x.dim() == 1:
        x = x[None]
    dt = _TYPES.get(x.dtype)
    if dt is None or not _rows_ok(x):
        raise ValueError("x must be float32, float16 or bfloat16 [T, n] with contiguous rows")
    T, n = x.shape
    if n == 0:
        raise ValueError("x must have at least one value a row")
    nb = -(-n // BLOCK)
    dev = x.get_device()
    if dev < 0 or dev != _current_device():
        _here(x)
    if codes is None:
        codes = x.new_empty(T, nb * BLOCK, dtype=E4M3)
    elif _out(codes, (T, nb * BLOCK), E4M3, x, "codes").get_device() != dev:
        _here(x, codes)
    if scale is None:
        scale = x.new_empty(T, nb) if dt == 0 else x.new_empty(T, nb, dtype=_F32)
    elif _out(scale, (T, nb), torch.float32, x, "scale").get_device() != dev:
        _here(x, scale)
    rc = _quantize(dt, x.data_ptr(), x.stride(0), n, T, codes.data_ptr(), scale.data_ptr(), _raw_stream(dev))
    if rc:
        check(rc)
    return codes, scale


def matmul(Wp, rows, n, codes, scale, out=None, dtype=torch.float32):
    """Y[t, r] = packed row r . token t: codes [T, np] and scale [T, np / 128] as
    quantize() gives them; Y [T, rows] of `dtype`, or `out` (rows of any stride)."""
    nb = -(-n // BLOCK)
    if rows <= 0 or n <= 0 or Wp.dtype is not _U8 or not Wp.is_contiguous() or Wp.numel() < _packed_bytes(rows, n):
        raise ValueError(f"Wp is not a packed matrix of {rows} x {n}")
    shape = codes.shape
    if codes.dtype not in _CODES or len(shape) != 2 or shape[1] != nb * BLOCK or not codes.is_contiguous():
        raise ValueError(f"codes must be contiguous E4M3 [T, {nb * BLOCK}]")
    T = shape[0]
    if scale.shape != (T, nb) or scale.dtype is not _F32 or not scale.is_contiguous():
        raise ValueError(f"scale must be contiguous float32 [{T}, {nb}]")
    if out is None:
        dt = _TYPES.get(dtype)
        if dt is None:
            raise ValueError("dtype must be float32, float16 or bfloat16")
        out = scale.new_empty(T, rows) if dt == 0 else scale.new_empty(T, rows, dtype=dtype)
    else:
        dt = _TYPES.get(out.dtype)
        if out.shape != (T, rows) or dt is None or not _rows_ok(out):
            raise ValueError(f"out must be float32, float16 or bfloat16 [{T}, {rows}] with contiguous rows")
    dev = Wp.get_device()
    if dev < 0 or not dev == codes.get_device() == scale.get_device() == out.get_device() == _current_device():
        _here(Wp, codes, scale, out)
    rc = _matmul(Wp.data_ptr(), rows, n, codes.data_ptr(), scale.data_ptr(), T, dt, out.data_ptr(), out.stride(0),
                 _raw_stream(dev))
    if rc:
        check(rc)
    return out


def matmul_kernel(rows, n, T):
    """The name of the kernel that matmul() launches for T tokens (None where there is no launch)."""
    name = lib.tlm_hip_fp8_matmul_kernel(rows, n, T)
    return name.decode() if name else None


class MoeBlock:
    """One routed MoE block of E4M3 matrices for up to 64 tokens a call.  Expert
    e's packed gate / up / down pointers are expert_ptrs[3e .. 3e + 2], 0 for
    experts that the mask prunes (they stay pruned where the mask is changed later); packed
    matrices are the caller's to keep alive, as are the tensors a call is given.
    The workspace is one per block and grows with the largest T seen (reserve()
    sizes it ahead), so calls of one block must not overlap (other streams, two
    graphs at once), and the block is kept until its calls are done and as long
    as a graph that holds one is replayed."""

    def __init__(self, *, D, de, E, k, ffn_norm, router_w, expert_ptrs, router=0, routed_scale=1.0, eps=1e-6,
                 router_bias=None, mask=None, ds=0, shared=None, shared_gate_inp=None):
        if len(expert_ptrs) != 3 * E or any(p % 16 for p in expert_ptrs):
            raise ValueError("expert_ptrs must hold 3 E packed matrices, 16-byte aligned")
        if (ds > 0) != (shared is not None):
            raise ValueError("ds and shared go together")
        given = [(t, shape, dt, what) for t, shape, dt, what in (
            (ffn_norm, (D,), _F32, "ffn_norm"), (router_w, (E, D), _F32, "router_w"), (router_bias, (E,), _F32, "router_bias"),
            (mask, (E,), _U8, "mask"), (shared_gate_inp, (D,), _F32, "shared_gate_inp")) if t is not None]
        for t, shape, dt, what in given:
            _out(t, shape, dt, t, what)
        if not all(expert_ptrs):
            pruned = [False] * E if mask is None else mask.tolist()
            if not all(pruned[i // 3] or p for i, p in enumerate(expert_ptrs)):
                raise ValueError("expert_ptrs may be 0 only for experts that the mask prunes")
        if shared is not None:
            if len(shared) != 3 or any(m.dtype is not _U8 or not m.is_contiguous() or m.data_ptr() % 16 or
                                       m.numel() < packed_bytes(*rn)
                                       for m, rn in zip(shared, ((ds, D), (ds, D), (D, ds)))):
                raise ValueError("shared must be 3 packed matrices, 16-byte aligned")
        _here(*(t for t, *_ in given), *(shared or ()))
        self.keep = [ffn_norm, router_w, router_bias, mask, shared, shared_gate_inp]
        self.device = ffn_norm.device
        self.table = torch.tensor(list(expert_ptrs), dtype=torch.int64, device=self.device)

        def p(t):
            return t.data_ptr() if t is not None else None

        sg, su, sd = shared if shared is not None else (None, None, None)
        self.desc = MoeDesc(D, de, ds, E, k, router, routed_scale, eps, FP8, FP8, p(ffn_norm), p(router_w),
                            p(router_bias), p(mask), self.table.data_ptr(), p(sg), p(su), p(sd), p(shared_gate_inp))
        self._desc = C.byref(self.desc)
        self.D, self.k = D, k
        check(_moe(self._desc, None, None, 0, None, None, None, None))   # the sizes fit
        self._dev = ffn_norm.get_device()
        self.workspace, self._pws, self._room, self._earlier = None, None, 0, []

    def reserve(self, T):
        """Make the workspace large enough for T tokens (it at least doubles; a smaller one that a
        captured graph may hold stays allocated)."""
        if T > self._room:
            room = min(max(T, 2 * self._room), max(T, MOE_MAX_TOKENS))
            nbytes = int(lib.tlm_hip_fp8_moe_workspace_bytes(self._desc, room))
            if not nbytes:
                check(_moe(self._desc, None, None, T, None, None, None, None))
            if self.workspace is not None:
                self._earlier.append(self.workspace)
            self.workspace = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
            self._pws = self.workspace.data_ptr()
            self._room = room

    def __call__(self, h, out=None, ids=None, w=None):
        """out = h + MoE(h) for h (f32 [T, D] or [D]), T <= 64; without `out` h itself
        is updated.  ids (int32) / w (f32), [T, k], receive the routing.  Returns
        out."""
        shape = h.shape
        if h.dtype is not _F32 or not h.is_contiguous() or len(shape) not in (1, 2) or shape[-1] != self.D:
            raise ValueError(f"h must be contiguous float32 [T, {self.D}]")
        T = shape[0] if len(shape) == 2 else 1
        dev, ph = h.get_device(), h.data_ptr()
        if dev != self._dev or dev != _current_device():
            _here(h, self.table)
        po = pi = pw = None
        if out is None:
            out, po = h, ph
        else:
            if out.shape != shape or out.dtype is not _F32 or not out.is_contiguous() or out.get_device() != dev:
                _here(h, _out(out, shape, _F32, h, "out"))
            po = out.data_ptr()
            if po != ph and abs(po - ph) < 4 * T * self.D:
                raise ValueError("out must be h itself or not overlap it")
        if ids is not None:
            if ids.shape != (T, self.k) or ids.dtype is not _I32 or not ids.is_contiguous() or ids.get_device() != dev:
                _here(h, _out(ids, (T, self.k), _I32, h, "ids"))
            pi = ids.data_ptr()
        if w is not None:
            if w.shape != (T, self.k) or w.dtype is not _F32 or not w.is_contiguous() or w.get_device() != dev:
                _here(h, _out(w, (T, self.k), _F32, h, "w"))
            pw = w.data_ptr()
        if T > self._room:
            self.reserve(T)
        if T:
            rc = _moe(self._desc, ph, po, T, pi, pw, self._pws, _raw_stream(dev))
            if rc:
                check(rc)
        return out
