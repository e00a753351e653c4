"""Rows of q | k | v into the paged cache, against the definition in 64 bits.

Tolerance, counted from the roundings: a norm's sum of hd squares (hd + 1 roundings, half of them in the root),
its root, quotient and two products; an angle's sine and cosine to 2^-22 of 1 (the double angle's own error
is below 2^-30 for positions under 2^22), two products and a sum; then one rounding to the cache's type."""
import math

import pytest
import torch

from tests.kv_ref import HALF_STEP, Batch, gen
from tierlm_amd import kv

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def reference(x, heads, kv_heads, hd, pos, q_norm, k_norm, eps, freq, rope_scale):
    """q [T, H, hd], k, v [T, KV, hd] and the bound on q's and k's error before their last rounding, 64 bits."""
    T = x.shape[0]
    x = x.double().view(T, heads + 2 * kv_heads, hd)
    y, v = x[:, :heads + kv_heads], x[:, heads + kv_heads:]
    n = 0.0
    for w, sl in ((q_norm, slice(0, heads)), (k_norm, slice(heads, heads + kv_heads))):
        if w is not None:
            y = y.clone()
            y[:, sl] = y[:, sl] * torch.rsqrt(y[:, sl].square().mean(-1, keepdim=True) + eps) * w.double()
            n = hd / 2 + 8
    mag = torch.cat([y[..., :hd // 2].abs() + y[..., hd // 2:].abs()] * 2, -1) if freq is not None else y.abs()
    if freq is not None:
        a = pos.double()[:, None, None] * freq
        c, s = torch.cos(a) * rope_scale, torch.sin(a) * rope_scale
        lo, hi = y[..., :hd // 2], y[..., hd // 2:]
        y = torch.cat([lo * c - hi * s, hi * c + lo * s], -1)
        n, mag = n + 4 + 8, mag * abs(rope_scale)
    return y[:, :heads], y[:, heads:], v, mag * (n * 2.0 ** -24)


def check(dtype, xdtype, heads, kv_heads, hd, page, new, lens, *, norms=True, rope=True, rope_scale=1.0, seed=0, cu=True,
          stride=0, offset=0):
    b = Batch(dtype, heads, kv_heads, hd, page, new, lens, seed=seed)
    g = gen(seed + 100)
    T, width = b.cu_list[-1], (heads + 2 * kv_heads) * hd
    x = torch.randn(T, width, generator=g, device="cuda").to(xdtype)
    if stride:
        wide = torch.zeros(T * (width + stride) + offset, dtype=xdtype, device="cuda")
        xs = wide.as_strided((T, width), (width + stride, 1), offset)
        xs.copy_(x)
        x = xs
    q_norm = 1 + 0.1 * torch.randn(hd, generator=g, device="cuda") if norms else None
    k_norm = 1 + 0.1 * torch.randn(hd, generator=g, device="cuda") if norms else None
    freq = kv.rope_frequencies(hd, 1e6) if rope else None
    k0, v0 = b.cache.k.clone(), b.cache.v.clone()
    q = kv.append(b.cache, x, heads, b.tables, b.lens, b.cu if cu else None, q_norm=q_norm, k_norm=k_norm, eps=1e-6,
                  inv_freq=freq, rope_scale=rope_scale)
    pos = torch.cat([torch.arange(m - n, m) for n, m in zip(new, lens)]).cuda()
    wq, wk, wv, tol = reference(x, heads, kv_heads, hd, pos, q_norm, k_norm, 1e-6, freq, rope_scale)
    half, tiny = HALF_STEP[dtype], 2.0 ** -25 if dtype is F16 else 0.0

    def near(got, want, tol):
        err, bound = (got.double() - want).abs(), tol + (want.abs() + tol) * half + tiny
        assert (err <= bound).all(), float((err / bound).max())

    near(q, wq, tol[:, :heads])
    # what the call wrote, value by value; nothing else has changed
    k1, v1 = b.cache.k.clone(), b.cache.v.clone()
    for i, (n, m) in enumerate(zip(new, lens)):
        sl = slice(b.cu_list[i], b.cu_list[i + 1])
        ids = b.tables_list[i]
        if n == 0:
            continue
        near(b.cache.keys(ids)[:, m - n:m].transpose(0, 1), wk[sl], tol[sl, heads:])
        assert torch.equal(b.cache.values(ids)[:, m - n:m].transpose(0, 1), wv[sl].to(xdtype).to(dtype))
        b.cache.k.copy_(k0)
        b.cache.v.copy_(v0)
        b.put(i, torch.zeros(n, kv_heads, hd, dtype=dtype, device="cuda"),
              torch.zeros(n, kv_heads, hd, dtype=dtype, device="cuda"), m - n)
        k0, v0 = b.cache.k.clone(), b.cache.v.clone()
        b.cache.k.copy_(k1)
        b.cache.v.copy_(v1)
        b.put(i, torch.zeros(n, kv_heads, hd, dtype=dtype, device="cuda"),
              torch.zeros(n, kv_heads, hd, dtype=dtype, device="cuda"), m - n)
        k1, v1 = b.cache.k.clone(), b.cache.v.clone()
        b.cache.k.copy_(k1)
        b.cache.v.copy_(v1)
    assert torch.equal(k0.view(torch.int16), k1.view(torch.int16))
    assert torch.equal(v0.view(torch.int16), v1.view(torch.int16))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("xdtype", [F32, F16, BF16])
def test_types(hip, dtype, xdtype):
    check(dtype, xdtype, 8, 2, 64, 16, [5, 40, 1], [5, 57, 33])


@pytest.mark.parametrize("hd", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (9, 3), (40, 1)])
def test_heads(hip, hd, heads, kv_heads):
    check(BF16, F32, heads, kv_heads, hd, 32, [3, 21], [20, 21], seed=hd)


@pytest.mark.parametrize("new,lens", [
    ([1], [1]), ([15], [15]), ([16], [16]), ([17], [17]), ([7], [23]), ([8], [24]), ([8], [16]), ([9], [25]), ([16], [33]),
    ([100], [131]), ([0, 5, 0, 12, 0], [3, 5, 0, 28, 16])])
@pytest.mark.parametrize("page", [16, 64])
def test_places(hip, new, lens, page):
    """Rows that begin and end inside blocks and half blocks; what lies around them stays."""
    check(F16, F32, 4, 2, 32, page, new, lens, seed=sum(new))


@pytest.mark.parametrize("norms", [False, True])
@pytest.mark.parametrize("rope", [False, True])
def test_parts(hip, norms, rope):
    check(BF16, BF16, 8, 2, 128, 64, [33, 2], [40, 2], norms=norms, rope=rope, rope_scale=1.0 if not rope else 1.3)


@pytest.mark.parametrize("which", ["q", "k"])
def test_one_norm(hip, which):
    """The other heads pass as they are."""
    b = Batch(F16, 4, 2, 64, 16, [20], [30], seed=11)
    g = gen(12)
    x, w = torch.randn(20, 8 * 64, generator=g, device="cuda"), 1 + 0.1 * torch.randn(64, generator=g, device="cuda")
    qn, kn = (w, None) if which == "q" else (None, w)
    q = kv.append(b.cache, x, 4, b.tables, b.lens, b.cu, q_norm=qn, k_norm=kn)
    wq, wk, _, tol = reference(x, 4, 2, 64, torch.arange(10, 30, device="cuda"), qn, kn, 1e-6, None, 1.0)
    k = b.cache.keys(b.tables_list[0])[:, 10:30].transpose(0, 1)
    for got, want, t in ((q, wq, tol[:, :4]), (k, wk, tol[:, 4:])):
        assert ((got.double() - want).abs() <= t + (want.abs() + t) * 2.0 ** -11 + 2.0 ** -25).all()
    plain = k if which == "q" else q
    assert torch.equal(plain, (x[:, 256:384] if which == "q" else x[:, :256]).reshape(20, -1, 64).to(F16))


@pytest.mark.parametrize("B", [3, 64, 65, 300])
def test_many_sequences(hip, B):
    check(F16, F32, 4, 2, 32, 16, [(5 * i) % 7 for i in range(B)], [(5 * i) % 7 + (i * 3) % 20 for i in range(B)], seed=B)


def test_a_row_a_sequence(hip):
    check(BF16, F32, 32, 4, 128, 64, [1] * 70, [1 + 13 * i for i in range(70)], cu=False)


def test_stride(hip):
    check(F16, BF16, 8, 2, 96, 16, [11, 30], [20, 30], stride=7, offset=3)


@pytest.mark.parametrize("heads,kv_heads,hd,new,lens,cu", [
    (17, 17, 32, [4003], [4010], True), (1, 1, 32, [70001], [70001], True), (16, 16, 64, [3, 3000, 0, 1200], [3, 3005, 0, 1300], True),
    (15, 15, 32, [1] * 288, list(range(1, 289)), False), (57, 19, 96, [3600], [3600], True)])
def test_two_heads_a_group(hip, heads, kv_heads, hd, new, lens, cu):
    """Batches that fill the card, where a group takes two key heads: an odd number of them, and a single one."""
    check(BF16, F32, heads, kv_heads, hd, 64, new, lens, seed=heads, cu=cu)


def test_far_positions(hip):
    """A page late in a long context: the angles of position 2^20 are the definition's."""
    hd, heads, n = 64, 4, 20
    first = (1 << 20) - 7
    cache = kv.Cache(4, 2, hd, page=4096, dtype=F16)
    pages = (first + n) // 4096 + 1
    tables = torch.full((1, pages), -1, dtype=torch.int32, device="cuda")
    tables[0, first // 4096], tables[0, (first + n) // 4096] = 2, 1
    x = torch.randn(n, (heads + 4) * hd, generator=gen(3), device="cuda")
    freq = kv.rope_frequencies(hd, 1e4)
    lens = torch.tensor([first + n], dtype=torch.int32, device="cuda")
    q = kv.append(cache, x, heads, tables, lens, torch.tensor([0, n], dtype=torch.int32, device="cuda"), inv_freq=freq)
    wq, wk, _, tol = reference(x, heads, 2, hd, torch.arange(first, first + n, device="cuda"), None, None, 0.0, freq, 1.0)
    for got, want, t in ((q, wq, tol[:, :heads]),
                         (torch.cat([cache.keys([2])[:, first % 4096:], cache.keys([1])[:, :n - 7]], 1).transpose(0, 1), wk,
                          tol[:, heads:])):
        assert ((got.double() - want).abs() <= t + (want.abs() + t) * 2.0 ** -11 + 2.0 ** -25).all()


def test_places_that_are_none(hip):
    """Padded slots, pages that name none, positions past the table, rows before position 0: nothing is written,
    and the queries of rows with a position are computed."""
    hd, heads = 64, 4
    b = Batch(BF16, heads, 2, hd, 16, [1] * 4, [20, 20, 20, 20], seed=4, spare=5)
    x = torch.randn(4, (heads + 4) * hd, generator=gen(5), device="cuda")
    freq = kv.rope_frequencies(hd, 1e4)
    want = kv.append(b.cache, x, heads, b.tables, b.lens, inv_freq=freq)
    k0, v0 = b.cache.k.clone(), b.cache.v.clone()
    b.tables[1, 1], b.tables[2, 1] = -1, b.cache.n_pages
    lens = torch.tensor([0, 20, 20, 33], dtype=torch.int32, device="cuda")
    q = kv.append(b.cache, 2 * x, heads, b.tables, lens, inv_freq=freq)
    assert torch.equal(b.cache.k.view(torch.int16), k0.view(torch.int16))
    assert torch.equal(b.cache.v.view(torch.int16), v0.view(torch.int16))
    assert (q[0] == 0).all() and torch.equal(q[1:3], 2 * want[1:3])
    # a prompt of more rows than positions: its last rows are the first positions
    c = Batch(F16, heads, 2, hd, 16, [40], [40], seed=6)
    x = torch.randn(40, (heads + 4) * hd, generator=gen(6), device="cuda")
    lens = torch.tensor([25], dtype=torch.int32, device="cuda")
    k0 = c.cache.keys(c.tables_list[0]).clone()
    q = kv.append(c.cache, x, heads, c.tables, lens, c.cu)
    assert (q[:15] == 0).all() and torch.equal(q[15:], x[15:, :heads * hd].view(25, heads, hd).to(F16))
    k1 = c.cache.keys(c.tables_list[0])
    assert torch.equal(k1[:, :25], x[15:, heads * hd:(heads + 2) * hd].view(25, 2, hd).to(F16).transpose(0, 1))
    assert torch.equal(k1[:, 25:].contiguous().view(torch.int16), k0[:, 25:].contiguous().view(torch.int16))


def test_rows_behind_the_last_sequence_stay(hip):
    b = Batch(BF16, 4, 2, 64, 16, [5, 9], [5, 20], seed=7)
    x = torch.randn(20, 8 * 64, generator=gen(7), device="cuda")
    out = torch.full((20, 4, 64), 7.0, dtype=BF16, device="cuda")
    kv.append(b.cache, x, 4, b.tables, b.lens, b.cu, out=out)
    assert (out[14:] == 7).all() and not (out[:14] == 7).any()


def test_poisoned_row(hip):
    """An infinity or NaN stays in its row's head."""
    b = Batch(BF16, 4, 2, 64, 16, [20], [20], seed=8)
    x = torch.randn(20, 8 * 64, generator=gen(8), device="cuda")
    w = torch.ones(64, device="cuda")
    want = kv.append(b.cache, x, 4, b.tables, b.lens, b.cu, q_norm=w, k_norm=w)
    k = b.cache.keys(b.tables_list[0])[:, :20].clone()
    x[3, 70], x[9, 4 * 64 + 1] = math.inf, math.nan
    q = kv.append(b.cache, x, 4, b.tables, b.lens, b.cu, q_norm=w, k_norm=w)
    keep = torch.ones(20, 4, dtype=torch.bool, device="cuda")
    keep[3, 1] = False
    assert torch.equal(q[keep], want[keep]) and torch.isnan(q[3, 1, 6])
    k2 = b.cache.keys(b.tables_list[0])[:, :20]
    keep = torch.ones(2, 20, dtype=torch.bool, device="cuda")
    keep[0, 9] = False
    assert torch.equal(k2[keep], k[keep]) and torch.isnan(k2[0, 9]).all()


def test_graph(hip):
    """A captured append follows the lengths and tables on the device."""
    b = Batch(BF16, 8, 2, 64, 16, [1, 1], [30, 9], seed=9, spare=4)
    x = torch.randn(2, 12 * 64, generator=gen(9), device="cuda")
    freq = kv.rope_frequencies(64, 1e4)
    out = torch.empty(2, 8, 64, dtype=BF16, device="cuda")
    kv.append(b.cache, x, 8, b.tables, b.lens, inv_freq=freq, out=out)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        kv.append(b.cache, x, 8, b.tables, b.lens, inv_freq=freq, out=out)
    for i in range(4):
        b.lens.copy_(torch.tensor([28 + i, 3 * i + 1], dtype=torch.int32))
        b.cache.k.zero_()
        b.cache.v.zero_()
        g.replay()
        torch.cuda.synchronize()
        k, v, q = b.cache.k.clone(), b.cache.v.clone(), out.clone()
        b.cache.k.zero_()
        b.cache.v.zero_()
        kv.append(b.cache, x, 8, b.tables, b.lens, inv_freq=freq, out=out)
        assert torch.equal(q, out) and torch.equal(k, b.cache.k) and torch.equal(v, b.cache.v)
        assert int((k != 0).any(-1).any(-2).sum()) > 0
