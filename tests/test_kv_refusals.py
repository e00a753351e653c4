"""The paged cache's entry points refuse what they cannot do before any launch (no GPU here), and the functions that
turn lengths and page numbers into addresses hold over all small cases."""
import ctypes as C
import os
import subprocess

import pytest
import torch

from tierlm_amd import fp8, kv, lib
from tierlm_amd._lib import KvBatch, KvCache

EINVAL, ERANGE, EUNSUP = -3, -5, -7
P = 1 << 20                      # an aligned address that no refused call follows
HERE = os.path.dirname(os.path.abspath(__file__))


def cache(**kw):
    a = dict(dt=2, kv_heads=2, head_dim=64, page=16, n_pages=9, k=P, v=P)
    a.update(kw)
    return KvCache(*(a[f] for f, _ in KvCache._fields_))


def batch(**kw):
    a = dict(B=3, rows=3, cu=None, lens=P, tables=P, table_stride=4, table_pages=4)
    a.update(kw)
    return KvBatch(*(a[f] for f, _ in KvBatch._fields_))


BAD = [
    (EUNSUP, dict(dt=0), {}, {}), (EUNSUP, dict(dt=8), {}, {}), (EUNSUP, dict(head_dim=0), {}, {}),
    (EUNSUP, dict(head_dim=16), {}, {}), (EUNSUP, dict(head_dim=80), {}, {}), (EUNSUP, dict(head_dim=288), {}, {}),
    (EINVAL, dict(page=0), {}, {}), (EINVAL, dict(page=8), {}, {}), (EINVAL, dict(page=48), {}, {}),
    (EINVAL, dict(page=8192), {}, {}), (EINVAL, dict(kv_heads=0), {}, {}), (EINVAL, dict(kv_heads=3), {}, {}),
    (EINVAL, dict(n_pages=0), {}, {}), (EINVAL, dict(n_pages=1 << 31), {}, {}), (EINVAL, dict(k=None), {}, {}),
    (EINVAL, dict(v=None), {}, {}), (EINVAL, dict(k=P + 8), {}, {}), (EINVAL, dict(v=P + 2), {}, {}),
    (EINVAL, {}, dict(B=-1), {}), (EINVAL, {}, dict(rows=-1), {}), (EINVAL, {}, dict(rows=4), {}),
    (ERANGE, {}, dict(B=(1 << 20) + 1, rows=(1 << 20) + 1), {}), (ERANGE, {}, dict(rows=1 << 28, cu=P), {}), (ERANGE, {}, dict(rows=1 << 62, cu=P), {}),
    (EINVAL, {}, dict(table_pages=0), {}), (EINVAL, {}, dict(table_pages=(1 << 26) + 1, table_stride=1 << 27), {}),
    (EINVAL, {}, dict(table_stride=3), {}), (EINVAL, {}, dict(lens=None), {}), (EINVAL, {}, dict(tables=None), {}),
    (EINVAL, {}, dict(lens=P + 2), {}), (EINVAL, {}, dict(tables=P + 1), {}),
    (EINVAL, {}, {}, dict(heads=0)), (EINVAL, {}, {}, dict(heads=-2)), (EINVAL, {}, {}, dict(heads=7)),
    (EINVAL, {}, {}, dict(x=None)), (EINVAL, {}, {}, dict(x=P + 1)), (EINVAL, {}, {}, dict(out=None)),
    (EINVAL, {}, {}, dict(out=P + 1)), (EINVAL, {}, {}, dict(stride=8 * 64 - 1)), (EUNSUP, {}, {}, dict(dt=8))]


@pytest.mark.parametrize("call", ["append", "decode", "prompt"])
@pytest.mark.parametrize("want,ck,bk,ak", BAD)
def test_refuses(call, want, ck, bk, ak):
    a = dict(heads=8, x=P, out=P, stride=12 * 64, dt=2)
    a.update(ak)
    c, b = cache(**ck), batch(**bk)
    c, b = C.byref(c), C.byref(b)
    if call == "append":
        rc = lib.tlm_hip_kv_append(c, b, a["dt"], a["x"], a["stride"], a["heads"], None, None, 1e-6, None, 1.0, a["out"], None)
    elif call == "decode":
        rc = lib.tlm_hip_kv_decode(c, b, a["x"], a["stride"], a["heads"], 0.1, a["dt"], a["out"], P, None)
    else:
        rc = lib.tlm_hip_kv_prompt(c, b, a["x"], a["stride"], a["heads"], 0.1, a["dt"], a["out"], P, None)
    if call == "decode" and "cu" in bk:
        want = EINVAL if "rows" not in bk else want
    assert rc == want, lib.tlm_hip_errmsg()
    assert ("kv_" + call).encode() in lib.tlm_hip_errmsg()


def test_refuses_more():
    c, b = C.byref(cache()), C.byref(batch())
    assert lib.tlm_hip_kv_append(None, b, 0, P, 768, 8, None, None, 1e-6, None, 1.0, P, None) == EINVAL
    assert lib.tlm_hip_kv_append(c, None, 0, P, 768, 8, None, None, 1e-6, None, 1.0, P, None) == EINVAL
    for eps in (-1e-6, float("nan"), float("inf")):
        assert lib.tlm_hip_kv_append(c, b, 0, P, 768, 8, None, None, eps, None, 1.0, P, None) == EINVAL
    assert lib.tlm_hip_kv_append(c, b, 0, P, 768, 8, P + 2, None, 0.0, None, 1.0, P, None) == EINVAL
    assert lib.tlm_hip_kv_append(c, b, 0, P, 768, 8, None, P + 1, 0.0, None, 1.0, P, None) == EINVAL
    assert lib.tlm_hip_kv_append(c, b, 0, P, 768, 8, None, None, 0.0, P + 4, 1.0, P, None) == EINVAL
    assert lib.tlm_hip_kv_append(c, b, 0, P, 767, 8, None, None, 0.0, None, 1.0, P, None) == EINVAL
    assert lib.tlm_hip_kv_append(c, b, 0, P, 768, 8, None, None, 0.0, None, 1.0, P + 8, None) == EINVAL
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        assert lib.tlm_hip_kv_decode(c, b, P, 512, 8, scale, 2, P, P, None) == EINVAL
        assert lib.tlm_hip_kv_prompt(c, b, P, 512, 8, scale, 2, P, P, None) == EINVAL
    assert lib.tlm_hip_kv_decode(c, C.byref(batch(cu=P)), P, 512, 8, 0.1, 2, P, P, None) == EINVAL


def test_workspace():
    """None up to 512 positions of table; beyond, it must be there and aligned."""
    c = C.byref(cache())
    small, wide = batch(table_pages=32, table_stride=32), batch(table_pages=33, table_stride=33)
    ws = lib.tlm_hip_kv_decode_workspace_bytes
    assert ws(c, C.byref(small), 8) == 0
    assert ws(c, C.byref(wide), 8) > 0 and ws(c, C.byref(wide), 7) == 0
    for p in (None, P + 16):
        assert lib.tlm_hip_kv_decode(c, C.byref(wide), P, 512, 8, 0.1, 2, P, p, None) == EINVAL
        assert b"workspace" in lib.tlm_hip_errmsg()
    ws = lib.tlm_hip_kv_prompt_workspace_bytes
    small, wide = batch(cu=P, table_pages=127, table_stride=127), batch(cu=P, table_pages=128, table_stride=128)
    assert ws(c, C.byref(small), 8) == 0 and ws(c, C.byref(wide), 8) > 0 and ws(c, C.byref(wide), 7) == 0
    assert ws(c, C.byref(batch(cu=P, rows=1 << 20, table_pages=128, table_stride=128)), 8) == 0      # rows enough
    assert ws(c, C.byref(batch(cu=P, rows=0, table_pages=128, table_stride=128)), 8) == 0
    for p in (None, P + 16):
        assert lib.tlm_hip_kv_prompt(c, C.byref(wide), P, 512, 8, 0.1, 2, P, p, None) == EINVAL
        assert b"workspace" in lib.tlm_hip_errmsg()


def test_nothing_to_do():
    c = C.byref(cache())
    for b in (batch(B=0, rows=0, lens=None, tables=None), batch(B=2, rows=0, cu=P, lens=None, tables=None)):
        assert lib.tlm_hip_kv_append(c, C.byref(b), 0, None, 768, 8, None, None, 1e-6, None, 1.0, None, None) == 0
        assert lib.tlm_hip_kv_prompt(c, C.byref(b), None, 512, 8, 0.1, 2, None, None, None) == 0
    b = batch(B=0, rows=0, lens=None, tables=None)
    assert lib.tlm_hip_kv_decode(c, C.byref(b), None, 512, 8, 0.1, 2, None, None, None) == 0


def test_norm_refuses():
    f = lib.tlm_hip_fp8_add_rmsnorm

    def call(want, **kw):
        a = dict(hdt=0, h=P, hs=128, xdt=2, x=P, xs=128, w=P, eps=1e-6, n=128, T=2, out=P, os=128, codes=P, scale=P, stream=None)
        a.update(kw)
        assert f(*a.values()) == want, kw
        if want:
            assert b"fp8_add_rmsnorm" in lib.tlm_hip_errmsg()

    for kw in (dict(n=0), dict(n=(1 << 22) + 1), dict(T=-1), dict(h=None), dict(w=None), dict(codes=None), dict(scale=None),
               dict(hs=127), dict(xs=127), dict(os=127), dict(h=P + 2), dict(x=P + 1), dict(w=P + 2), dict(out=P + 2),
               dict(codes=P + 8), dict(scale=P + 2), dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf"))):
        call(EINVAL, **kw)
    for kw in (dict(hdt=8), dict(xdt=8), dict(hdt=-1)):
        call(EUNSUP, **kw)
    call(ERANGE, T=(1 << 22) + 1)
    call(ERANGE, n=1 << 22, T=(1 << 11) + 1, hs=1 << 22, xs=1 << 22, os=1 << 22)
    call(0, T=0, h=None, x=None, w=None, out=None, codes=None, scale=None)


def test_python_refuses():
    """What the binding refuses needs no GPU to be refused: shapes, types and strides come before the device."""
    for kw in (dict(dtype=torch.float32), dict(page=24), dict(page=8), dict(page=8192), dict(head_dim=48), dict(head_dim=512),
               dict(n_pages=0), dict(kv_heads=0)):
        a = dict(n_pages=2, kv_heads=2, head_dim=64, device="cpu")
        a.update(kw)
        with pytest.raises(ValueError):
            kv.Cache(**a)
    c = kv.Cache(4, 2, 64, page=16, dtype=torch.float16, device="cpu")
    lens, tables = torch.zeros(3, dtype=torch.int32), torch.zeros(3, 2, dtype=torch.int32)
    q = torch.zeros(3, 8, 64, dtype=torch.float16)
    cu = torch.zeros(4, dtype=torch.int32)
    good = dict(q=q, cache=c, tables=tables, lens=lens)
    for kw in (dict(q=q.float()), dict(q=q[:, :7]), dict(q=q[..., :32]), dict(q=q[0]), dict(q=q[:, ::2]),
               dict(lens=lens.long()), dict(lens=lens[:2]), dict(lens=torch.zeros(6, dtype=torch.int32)[::2]),
               dict(tables=tables.long()), dict(tables=tables[:2]), dict(tables=tables[:, :0]), dict(tables=tables.T),
               dict(scale=0.0), dict(scale=float("nan")), dict(out=q[:2]), dict(out=q.double()), {}):
        with pytest.raises(ValueError):
            kv.decode(**{**good, **kw})
        with pytest.raises(ValueError):
            kv.prompt(**{**good, **kw}, cu=cu)
    for bad in (cu[:3], cu.long(), torch.zeros(8, dtype=torch.int32)[::2]):
        with pytest.raises(ValueError):
            kv.prompt(**good, cu=bad)
    x = torch.zeros(3, 12 * 64)
    good = dict(cache=c, qkv=x, heads=8, tables=tables, lens=lens)
    for kw in (dict(qkv=x.double()), dict(qkv=x[:, 1:]), dict(heads=7), dict(heads=0), dict(qkv=x[0]),
               dict(q_norm=torch.ones(32)), dict(k_norm=torch.ones(64, dtype=torch.float64)), dict(inv_freq=torch.ones(32)),
               dict(out=q.float()), dict(out=q[:2]), {}):
        with pytest.raises(ValueError):
            kv.append(**{**good, **kw})
    h, w = torch.zeros(2, 64), torch.zeros(64)
    for a in ((h.double(), h, w), (h, h[:1], w), (h, h.int(), w), (h, h, w[:5]), (h, h, w.double()), (h[0], h, w), (h, h, w)):
        with pytest.raises(ValueError):
            fp8.add_rmsnorm(*a)


def test_python_refuses_results_among_the_inputs():
    """A result that overlaps the rows read, by a value at either end; one right behind or before passes this check (and
    ends at the device's)."""
    c = kv.Cache(4, 2, 64, page=16, dtype=torch.float16, device="cpu")
    lens, tables, cu = torch.zeros(3, dtype=torch.int32), torch.zeros(3, 2, dtype=torch.int32), torch.zeros(4, dtype=torch.int32)
    m, n = 3 * 8 * 64, 3 * 12 * 64
    flat = torch.zeros(2 * n + 64, dtype=torch.float16)
    for at, match in ((0, "overlap"), (m - 1, "overlap"), (m, "device"), (m + 9, "device")):
        for q, out in ((flat[:m], flat[at:at + m]), (flat[at:at + m], flat[:m])):
            for call, more in ((kv.decode, ()), (kv.prompt, (cu,))):
                with pytest.raises(ValueError, match=match):
                    call(q.view(3, 8, 64), c, tables, lens, *more, out=out.view(3, 8, 64))
    # rows further apart: their span counts, up to the last row's end
    q = flat.as_strided((3, 8, 64), (600, 64, 1))
    with pytest.raises(ValueError, match="overlap"):
        kv.decode(q, c, tables, lens, out=flat[2 * 600 + 504:][:m].view(3, 8, 64))
    with pytest.raises(ValueError, match="device"):
        kv.decode(q, c, tables, lens, out=flat[2 * 600 + 512:][:m].view(3, 8, 64))
    skip = -(flat.data_ptr() // 2) % 8                                   # append's result is 16-byte aligned
    for at, match in ((0, "overlap"), (n - 8, "overlap"), (n, "device")):
        with pytest.raises(ValueError, match=match):
            kv.append(c, flat[skip:skip + n].view(3, 12 * 64), 8, tables, lens,
                      out=flat[skip + at:skip + at + m].view(3, 8, 64))


def test_places(tmp_path):
    exe = str(tmp_path / "places")
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-fsanitize=undefined", "-fno-sanitize-recover=all",
                    os.path.join(HERE, "kv_places.cpp"), "-o", exe], check=True)
    assert subprocess.run([exe], check=True, capture_output=True, text=True).stdout == "ok\n"


@pytest.fixture
def failed():
    if torch.cuda.is_available():
        pytest.skip("addresses that a launch would follow")
    note = getattr(lib, "_Z15tlmh_set_failedi")           # tlmh_set_failed(int), of the library's own start
    note.argtypes, note.restype = [C.c_int], None
    yield note
    note(0)


def test_a_failed_self_test_refuses_the_calls(failed):
    c, b = C.byref(cache()), C.byref(batch())
    calls = {"kv_append": lambda: lib.tlm_hip_kv_append(c, b, 0, P, 768, 8, None, None, 1e-6, None, 1.0, P, None),
             "kv_decode": lambda: lib.tlm_hip_kv_decode(c, b, P, 512, 8, 0.1, 2, P, P, None),
             "kv_prompt": lambda: lib.tlm_hip_kv_prompt(c, b, P, 512, 8, 0.1, 2, P, P, None)}
    norm = lambda: lib.tlm_hip_fp8_add_rmsnorm(0, P, 128, 2, P, 128, P, 1e-6, 128, 2, P, 128, P, P, None)   # noqa: E731
    failed(1 << 27)
    for name, call in calls.items():
        assert call() == -1 and name.encode() in lib.tlm_hip_errmsg() and b"self-test" in lib.tlm_hip_errmsg()
    norm()
    assert b"self-test" not in lib.tlm_hip_errmsg()
    failed(1 << 28)
    assert norm() == -1 and b"self-test" in lib.tlm_hip_errmsg()
    calls["kv_decode"]()                                   # no device: another error
    assert b"self-test" not in lib.tlm_hip_errmsg()


def test_struct_layout(tmp_path):
    """The C structs as the compiler lays them out."""
    src = tmp_path / "s.c"
    src.write_text('''#include <stdio.h>
#include "tlm_hip.h"
int main(void) { printf("%zu %zu %zu %zu %zu\\n", sizeof(tlm_hip_kv_cache), offsetof(tlm_hip_kv_cache, v),
                        sizeof(tlm_hip_kv_batch), offsetof(tlm_hip_kv_batch, tables), offsetof(tlm_hip_kv_batch, table_pages));
                 return 0; }''')
    exe = str(tmp_path / "s")
    subprocess.run(["gcc", "-I", os.path.join(os.path.dirname(HERE), "include"), str(src), "-o", exe], check=True)
    got = [int(v) for v in subprocess.run([exe], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [C.sizeof(KvCache), KvCache.v.offset, C.sizeof(KvBatch), KvBatch.tables.offset, KvBatch.table_pages.offset]
