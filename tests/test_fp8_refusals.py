"""The 8-bit floating-point entry points refuse what they cannot do before any
launch (no GPU here): sizes, types, strides, alignment, missing pointers."""
import ctypes as C

import pytest

from tierlm_amd import fp8, lib
from tierlm_amd._lib import MoeDesc

EINVAL, ERANGE, EUNSUP = -3, -5, -7
P = C.c_void_p(1 << 20)          # an aligned address that no refused call follows
ODD = C.c_void_p((1 << 20) + 1)
HALF = C.c_void_p((1 << 20) + 2)


def test_packed_bytes():
    assert fp8.packed_bytes(1, 1) == 2048 + 16
    assert fp8.packed_bytes(16, 128) == 2048 + 16
    assert fp8.packed_bytes(17, 129) == 2 * 2 * 2048 + 16
    assert fp8.packed_bytes(257, 640) == 17 * 5 * 2048 + 64          # 3 x 5 scales of 4 bytes, padded to 16
    assert fp8.packed_bytes(151936, 2048) == 151936 * 2048 + 1187 * 16 * 4
    for rows, n in ((0, 128), (128, 0), (-1, 5), ((1 << 25) + 1, 128), (16, (1 << 22) + 1)):
        assert fp8.packed_bytes(rows, n) == 0


@pytest.mark.parametrize("want,args", [
    (EINVAL, (None, 128, P, 1, 16, 128, P)), (EINVAL, (P, 128, None, 1, 16, 128, P)),
    (EINVAL, (P, 128, P, 1, 16, 128, None)), (EINVAL, (P, 127, P, 1, 16, 128, P)),
    (EINVAL, (P, 256, P, 1, 16, 129, P)), (EINVAL, (P, 128, P, 1, 0, 128, P)), (EINVAL, (P, 128, P, 1, 16, 0, P)),
    (EINVAL, (P, 128, P, 1, 16, 128, HALF)), (EINVAL, (P, 128, ODD, 1, 16, 128, P)),
    (ERANGE, (P, 1 << 22, P, 1 << 15, 1 << 25, 1 << 22, P))])
def test_pack_refuses(want, args):
    assert lib.tlm_hip_fp8_pack(*args, None) == want
    assert b"fp8_pack" in lib.tlm_hip_errmsg()


@pytest.mark.parametrize("want,args", [
    (EUNSUP, (8, P, 128, 128, 1, P, P)), (EUNSUP, (-1, P, 128, 128, 1, P, P)), (EINVAL, (0, P, 128, 0, 1, P, P)),
    (EINVAL, (0, P, 128, 128, -1, P, P)), (EINVAL, (0, None, 128, 128, 1, P, P)),
    (EINVAL, (0, P, 128, 128, 1, None, P)), (EINVAL, (0, P, 128, 128, 1, P, None)),
    (EINVAL, (0, P, 127, 128, 2, P, P)), (EINVAL, (0, HALF, 128, 128, 1, P, P)), (EINVAL, (1, ODD, 128, 128, 1, P, P)),
    (EINVAL, (0, P, 128, 128, 1, HALF, P)), (EINVAL, (0, P, 128, 128, 1, P, HALF)),
    (ERANGE, (0, P, 128, 128, (1 << 26) + 1, P, P)), (0, (0, None, 128, 128, 0, None, None))])
def test_quantize_refuses(want, args):
    assert lib.tlm_hip_fp8_quantize(*args, None) == want


@pytest.mark.parametrize("want,args", [
    (EUNSUP, (P, 16, 128, P, P, 1, 8, P, 16)), (EINVAL, (P, 0, 128, P, P, 1, 0, P, 16)),
    (EINVAL, (P, 16, 0, P, P, 1, 0, P, 16)), (EINVAL, (P, 16, 128, P, P, -1, 0, P, 16)),
    (EINVAL, (None, 16, 128, P, P, 1, 0, P, 16)), (EINVAL, (P, 16, 128, None, P, 1, 0, P, 16)),
    (EINVAL, (P, 16, 128, P, None, 1, 0, P, 16)), (EINVAL, (P, 16, 128, P, P, 1, 0, None, 16)),
    (EINVAL, (P, 16, 128, P, P, 2, 0, P, 15)), (EINVAL, (HALF, 16, 128, P, P, 1, 0, P, 16)),
    (EINVAL, (P, 16, 128, HALF, P, 1, 0, P, 16)), (EINVAL, (P, 16, 128, P, HALF, 1, 0, P, 16)),
    (EINVAL, (P, 16, 128, P, P, 1, 0, HALF, 16)), (EINVAL, (P, 16, 128, P, P, 1, 2, ODD, 16)),
    (ERANGE, (P, 16, 128, P, P, (1 << 20) + 1, 0, P, 16)),
    (ERANGE, (P, 1 << 20, 128, P, P, (1 << 15) + 1, 0, P, 1 << 20)), (0, (None, 16, 128, None, None, 0, 0, None, 16))])
def test_matmul_refuses(want, args):
    assert lib.tlm_hip_fp8_matmul(*args, None) == want


def desc(**kw):
    d = MoeDesc()
    d.D, d.de, d.ds, d.E, d.k, d.router = 512, 256, 0, 32, 4, 0
    d.routed_scale, d.eps, d.expert_dt, d.shared_dt = 1.0, 1e-6, fp8.FP8, fp8.FP8
    d.ffn_norm = d.router_w = d.experts = 1 << 20
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def moe(d, h=P, out=P, T=1, ids=None, w=None, ws=P):
    return lib.tlm_hip_fp8_moe(C.byref(d), h, out, T, ids, w, ws, None)


@pytest.mark.parametrize("want,kw", [
    (EINVAL, dict(E=0)), (EINVAL, dict(E=257)), (EINVAL, dict(k=0)), (EINVAL, dict(k=33)), (EINVAL, dict(E=3)),
    (EINVAL, dict(router=3)), (EINVAL, dict(router=-1)), (EUNSUP, dict(expert_dt=14)),
    (EUNSUP, dict(ds=64, shared_dt=8)), (EINVAL, dict(D=0)), (EINVAL, dict(D=16385)), (EINVAL, dict(de=0)),
    (EINVAL, dict(de=65537)), (EINVAL, dict(ds=-1)), (EINVAL, dict(ds=65537)), (EINVAL, dict(ds=64)),
    (EINVAL, dict(ffn_norm=None)), (EINVAL, dict(router_w=None)), (EINVAL, dict(experts=None)),
    (EINVAL, dict(router_w=(1 << 20) + 2))])
def test_moe_refuses_descriptors(want, kw):
    assert moe(desc(**kw)) == want
    assert b"fp8_moe" in lib.tlm_hip_errmsg()


def test_moe_refuses_calls():
    d = desc()
    assert moe(d, h=None) == EINVAL and moe(d, out=None) == EINVAL and moe(d, ws=None) == EINVAL
    assert moe(d, ws=C.c_void_p((1 << 20) + 128)) == EINVAL and moe(d, h=HALF) == EINVAL and moe(d, out=HALF) == EINVAL
    assert moe(d, ids=HALF) == EINVAL and moe(d, w=HALF) == EINVAL
    assert moe(desc(router_bias=HALF)) == EINVAL and moe(desc(shared_gate_inp=HALF)) == EINVAL
    for off in (4, 4 * 512 - 4):                                       # out begins inside h, or h inside out
        assert moe(d, out=C.c_void_p((1 << 20) + off)) == EINVAL and moe(d, h=C.c_void_p((1 << 20) + off)) == EINVAL
    assert moe(d, T=65) == ERANGE and moe(d, T=-1) == ERANGE
    assert moe(d, T=0, h=None, out=None, ws=None) == 0
    assert lib.tlm_hip_fp8_moe(None, P, P, 1, None, None, P, None) == EINVAL
    size = lib.tlm_hip_fp8_moe_workspace_bytes
    assert size(C.byref(d), 0) == 0 and size(C.byref(d), 65) == 0 and size(C.byref(desc(E=0)), 1) == 0
    assert 0 < size(C.byref(d), 1) < size(C.byref(d), 64)


def test_python_checks_raise():
    import torch
    w, s = torch.zeros(16, 128, dtype=torch.uint8), torch.zeros(1, 1)
    with pytest.raises(ValueError):
        fp8.pack(w, s)                                   # not on the device
    with pytest.raises(ValueError):
        fp8.pack(w.float(), s)                           # not codes
    with pytest.raises(ValueError):
        fp8.pack(w, torch.zeros(2, 1))                   # scales of another shape
    with pytest.raises(ValueError):
        fp8.pack(w.t(), s)                               # columns contiguous, not rows
    with pytest.raises(ValueError):
        fp8.quantize(torch.zeros(2, 128, dtype=torch.float64))
    with pytest.raises(ValueError):
        fp8.quantize(torch.zeros(1, 128).expand(2, 128))     # overlapping rows
    with pytest.raises(ValueError):
        fp8.quantize(torch.zeros(2, 128))
    wp, c = torch.zeros(4096, dtype=torch.uint8), torch.zeros(2, 128, dtype=torch.uint8)
    for args in ((wp[:100], 16, 128, c, torch.zeros(2, 1)), (wp, 16, 129, c, torch.zeros(2, 1)),
                 (wp, 16, 128, c, torch.zeros(2, 2)), (wp, 16, 128, c.float(), torch.zeros(2, 1)),
                 (wp, 16, 128, c, torch.zeros(2, 1))):
        with pytest.raises(ValueError):
            fp8.matmul(*args)
