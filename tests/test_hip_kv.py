"""Attention over the paged cache on the device against its definition in 64 bits (kv_ref: tolerances are counted
there): decode and prompt at the lengths, layouts and masks where they can go wrong."""
import math

import pytest
import torch

from tests.kv_ref import Batch, close, gen, reference
from tierlm_amd import kv

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def check_decode(b, scale=None, dtype=None):
    sc = 1.0 / math.sqrt(b.cache.head_dim) if scale is None else scale
    got = kv.decode(b.q, b.cache, b.tables, b.lens, scale=scale, dtype=dtype)
    for i, n in enumerate(b.lens_list):
        want, tol = reference(b.q[i:i + 1], b.k[i], b.v[i], sc, n - 1)
        close(got[i:i + 1], want, tol, f"sequence {i} of {n}")
    return got


def check_prompt(b, scale=None, dtype=None):
    sc = 1.0 / math.sqrt(b.cache.head_dim) if scale is None else scale
    got = kv.prompt(b.q, b.cache, b.tables, b.lens, b.cu, scale=scale, dtype=dtype)
    for i, (n, m) in enumerate(zip(b.new, b.lens_list)):
        lo, hi = b.cu_list[i], b.cu_list[i + 1]
        want, tol = reference(b.q[lo:hi], b.k[i], b.v[i], sc, m - n)
        close(got[lo:hi], want, tol, f"sequence {i}: {n} of {m}")
    return got


# lengths at the ends of blocks, tiles and groups of waves; an empty sequence among them
LENS = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 127, 128, 129, 255, 256, 257, 300]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("page", [16, 64, 256])
def test_decode_lengths(hip, dtype, page):
    check_decode(Batch(dtype, 8, 2, 64, page, [1] * len(LENS), LENS, seed=page))


@pytest.mark.parametrize("hd", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("heads,kv_heads", [(3, 3), (8, 1), (16, 1), (34, 2), (40, 1), (130, 2)])
def test_decode_heads(hip, hd, heads, kv_heads):
    check_decode(Batch(BF16 if hd % 64 else F16, heads, kv_heads, hd, 32, [1] * 3, [1, 77, 200], seed=hd + heads))


@pytest.mark.parametrize("hd,heads,kv_heads", [(64, 8, 2), (128, 32, 4), (256, 34, 2), (96, 5, 5), (128, 40, 1)])
@pytest.mark.parametrize("lens", [[5000], [0, 4000, 1, 129, 128, 2500], [3000] * 3, [1] * 70 + [4001]])
def test_decode_split(hip, hd, heads, kv_heads, lens):
    """A wide table: sequences are split over their length, by the lengths that the device sees."""
    b = Batch(BF16, heads, kv_heads, hd, 64, [1] * len(lens), lens, seed=hd, width=200)
    check_decode(b)


def test_decode_many_sequences(hip):
    """More sequences than a wave scans at once, split and not."""
    lens = [(37 * i) % 191 for i in range(300)]
    for width in (12, 40, 64, 65, 200):
        check_decode(Batch(F16, 4, 2, 32, 16, [1] * 300, lens, seed=3, width=width))


@pytest.mark.parametrize("B,heads,kv_heads,hd", [(70, 36, 2, 96), (300, 64, 4, 64), (64, 40, 8, 128), (40, 60, 3, 224)])
def test_decode_split_many_heads(hip, B, heads, kv_heads, hd):
    """Sequences of several shares, their heads joined several a group."""
    lens = [(997 * i) % 1400 if i % 9 else 1 + i for i in range(B)]
    check_decode(Batch(BF16, heads, kv_heads, hd, 32, [1] * B, lens, seed=B, width=50))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("scale", [1e-6, 0.25, 3.0])
def test_decode_scale_and_type(hip, dtype, scale):
    """Nearly equal weights, ordinary ones, and nearly all weight on one position."""
    for cache in (F16, BF16):
        check_decode(Batch(cache, 8, 2, 128, 64, [1] * 3, [700, 1, 90], seed=4), scale=scale, dtype=dtype)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("new,lens", [
    ([1], [1]), ([5], [5]), ([64], [64]), ([65], [65]), ([200], [200]), ([1], [500]), ([33], [1000]),
    ([3, 1, 0, 70, 16, 1], [3, 90, 40, 70, 47, 1]), ([100, 0, 0, 100], [100, 0, 5, 130])])
def test_prompt_lengths(hip, dtype, new, lens):
    check_prompt(Batch(dtype, 8, 2, 64, 16, new, lens, seed=len(new)))


@pytest.mark.parametrize("hd", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (8, 1), (9, 3), (40, 2), (130, 1)])
def test_prompt_heads(hip, hd, heads, kv_heads):
    check_prompt(Batch(F16 if hd % 64 else BF16, heads, kv_heads, hd, 32, [90, 7], [150, 7], seed=hd + heads))


@pytest.mark.parametrize("hd", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_prompt_many_groups(hip, hd, dtype):
    """Enough rows to fill the chip: 128 of them a group, their positions in one piece."""
    check_prompt(Batch(dtype, 208, 16, hd, 64, [200, 0, 151, 1], [200, 3, 300, 70], seed=hd))


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_prompt_few_groups(hip, hd):
    """As many groups as take 64 rows, and as few as take 32."""
    for heads, kv_heads, n in ((64, 4, 200), (16, 2, 40)):
        check_prompt(Batch(BF16, heads, kv_heads, hd, 16, [n], [n + 333], seed=hd))


@pytest.mark.parametrize("hd", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("new,lens,width", [
    ([16], [4000], 63), ([1], [2100], 63), ([5, 0, 40, 1], [3000, 4, 40, 0], 60), ([100], [1500], 64), ([3] * 9, [2047] * 9, 200),
    ([2, 30], [130, 300], 400)])
def test_prompt_parts(hip, hd, new, lens, width):
    """Few rows over far-reaching tables: positions split over groups and joined; short sequences among them."""
    check_prompt(Batch(BF16 if hd % 64 else F16, 16, 2, hd, 64, new, lens, seed=hd, width=width))


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_prompt_parts_of_more_rows(hip, hd):
    """64 rows a group, two parts or more."""
    check_prompt(Batch(BF16, 32, 2, hd, 64, [290 if hd < 256 else 150], [3000], seed=hd))


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256, 1024])
def test_prompt_pages(hip, page):
    check_prompt(Batch(BF16, 8, 2, 128, page, [300, 77], [1300, 77], seed=page))


@pytest.mark.parametrize("B", [64, 65, 200, 257, 700])
def test_prompt_many_sequences(hip, B):
    new = [(7 * i) % 13 for i in range(B)]
    check_prompt(Batch(F16, 4, 2, 32, 16, new, [n + i % 40 for i, n in enumerate(new)], seed=5))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("scale", [1e-6, 0.25, 3.0])
def test_prompt_scale_and_type(hip, dtype, scale):
    for cache in (F16, BF16):
        check_prompt(Batch(cache, 8, 2, 128, 64, [150, 1], [400, 90], seed=6), scale=scale, dtype=dtype)


def test_prompt_rising_scores(hip):
    """Scores that rise along the context: the running maximum moves in every tile."""
    for dtype in (F16, BF16):
        b = Batch(dtype, 4, 2, 64, 16, [130], [900], seed=7)
        up = torch.linspace(0.1, 3.0, 900, device="cuda")[:, None, None]
        k = (b.k[0].abs() * up).to(dtype)
        b.q = b.q.abs()
        b.k[0] = k
        b.put(0, k, b.v[0])
        check_prompt(b)
        one = Batch(dtype, 4, 2, 64, 16, [1], [900], seed=7)
        one.q, one.k[0] = b.q[-1:].contiguous(), k
        one.put(0, k, one.v[0])
        check_decode(one)


def test_decode_and_prompt_agree(hip):
    """A prompt's last rows, and the same queries one at a time."""
    b = Batch(BF16, 16, 2, 128, 64, [200], [1000], seed=8)
    y = kv.prompt(b.q, b.cache, b.tables, b.lens, b.cu, dtype=F32)
    for i in (0, 57, 199):
        lens = torch.tensor([801 + i], dtype=torch.int32, device="cuda")
        z = kv.decode(b.q[i:i + 1], b.cache, b.tables, lens, dtype=F32)
        want, tol = reference(b.q[i:i + 1], b.k[0][:801 + i], b.v[0][:801 + i], 1 / math.sqrt(128), 800 + i)
        close(z, want, tol)
        close(y[i:i + 1], want, tol)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_masked_places_may_hold_anything(hip, dtype):
    """Infinities and NaN behind a row's position leave its bits alone; rows that see them get them."""
    # 32 rows a group, 64 and 128, and parts
    for first, n, H, KV in ((0, 150, 8, 2), (70, 40, 8, 2), (0, 300, 64, 2), (90, 200, 416, 16), (2300, 40, 8, 2)):
        b = Batch(dtype, H, KV, 64, 16, [n], [first + n], seed=9)
        want = kv.prompt(b.q, b.cache, b.tables, b.lens, b.cu, dtype=F32)
        for where, value in ((first + 20, math.inf), (first + n - 1, math.nan), (first + n // 2, -math.inf)):
            for which in "kv":
                c = Batch(dtype, H, KV, 64, 16, [n], [first + n], seed=9)
                k, v = c.k[0].clone(), c.v[0].clone()
                (k if which == "k" else v)[where, :, 5] = value
                c.put(0, k, v)
                got = kv.prompt(c.q, c.cache, c.tables, c.lens, c.cu, dtype=F32)
                row = where - first
                assert torch.equal(got[:row], want[:row]), (where, value, which)
                if which == "v":
                    seen = got[row:, :, 5]
                    assert torch.isnan(seen).all() if math.isnan(value) else (seen == value).all()
                    keep = torch.arange(64, device="cuda") != 5
                    assert torch.equal(got[row:, :, keep], want[row:, :, keep])
                elif math.isnan(value):
                    assert torch.isnan(got[row:]).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("width", [16, 300])
def test_decode_values_that_are_not_finite(hip, dtype, width):
    """A seen infinity comes through with its sign, whatever its weight's bits (equal keys: weights of exactly 1 too); a NaN as
    one; other values and other sequences as without them."""
    for equal in (False, True):
        b = Batch(dtype, 8, 2, 64, 16, [1] * 3, [200, 90, 70], seed=25, width=width)
        if equal:
            for i, n in enumerate(b.lens_list):
                b.k[i] = torch.ones_like(b.k[i])
                b.put(i, b.k[i], b.v[i])
        want = kv.decode(b.q, b.cache, b.tables, b.lens, dtype=F32)
        for where, value in ((0, math.inf), (63, -math.inf), (199, math.nan)):
            v = b.v[0].clone()
            v[where, :, 5] = value
            b.put(0, b.k[0], v)
            got = kv.decode(b.q, b.cache, b.tables, b.lens, dtype=F32)
            seen = got[0, :, 5]
            assert torch.isnan(seen).all() if math.isnan(value) else (seen == value).all(), (where, value, equal)
            keep = torch.arange(64, device="cuda") != 5
            assert torch.equal(got[0][:, keep], want[0][:, keep]) and torch.equal(got[1:], want[1:])


@pytest.mark.parametrize("width", [16, 300])
def test_decode_unseen_places(hip, width):
    """Positions past the length hold NaN in every test here; beside it, infinities in the pages of others."""
    b = Batch(F16, 8, 2, 64, 16, [1] * 4, [1, 17, 40, 200], seed=10, spare=20, width=width)
    got = check_decode(b)
    b.cache.k[torch.isnan(b.cache.k)] = math.inf
    b.cache.v[torch.isnan(b.cache.v)] = -math.inf
    assert torch.equal(kv.decode(b.q, b.cache, b.tables, b.lens), got)


def test_pages_that_are_none(hip):
    """Numbers outside the cache name no page: their positions are not seen.  Lengths past the tables end with them."""
    for width in (None, 300):
        b = Batch(BF16, 8, 2, 64, 16, [1] * 3, [200, 90, 64], seed=11, width=width)
        for i, (row, gone) in enumerate(((0, 3), (1, 0), (2, 3))):
            b.tables[row, gone] = (-1, b.cache.n_pages, 2 ** 31 - 1)[i]
        got = kv.decode(b.q, b.cache, b.tables, b.lens, dtype=F32)
        for i, (row, gone) in enumerate(((0, 3), (1, 0), (2, 3))):
            keep = torch.arange(b.lens_list[row], device="cuda") // 16 != gone
            want, tol = reference(b.q[row:row + 1], b.k[row][keep], b.v[row][keep], 1 / 8, 10 ** 6)
            close(got[row:row + 1], want, tol)
        c = Batch(BF16, 8, 2, 64, 16, [60, 30, 64], [200, 90, 64], seed=11, width=width)
        c.tables[0, 3] = -7
        c.tables[2] = -1
        got = kv.prompt(c.q, c.cache, c.tables, c.lens, c.cu, dtype=F32)
        keep = torch.arange(200, device="cuda") // 16 != 3
        want, tol = reference(c.q[:60], c.k[0][keep], c.v[0][keep], 1 / 8, 140 - 16)
        close(got[:60], want, tol)
        assert (got[90:] == 0).all()
        if width is None:
            lens = torch.tensor([2 ** 31 - 1, -5, 0], dtype=torch.int32, device="cuda")
            full = torch.full_like(c.lens, c.tables.shape[1] * 16)
            tables = c.tables.clone()
            tables[:] = tables[0].clamp(min=0)
            q = c.q[:3].contiguous()
            a, e = kv.decode(q, c.cache, tables, lens), kv.decode(q, c.cache, tables, full)
            assert torch.equal(a[0].isnan(), e[0].isnan()) and torch.equal(a[0].nan_to_num(), e[0].nan_to_num())
            assert (a[1:] == 0).all()


def test_rows_before_the_first_position(hip):
    """More rows than positions: those before position 0 see nothing."""
    b = Batch(F16, 8, 2, 64, 16, [40, 3], [40, 3], seed=12)
    lens = torch.tensor([25, 0], dtype=torch.int32, device="cuda")
    got = kv.prompt(b.q, b.cache, b.tables, lens, b.cu, dtype=F32)
    assert (got[:15] == 0).all() and (got[40:] == 0).all()
    want, tol = reference(b.q[15:40], b.k[0][:25], b.v[0][:25], 1 / 8, 0)
    close(got[15:40], want, tol)


def test_rows_behind_the_last_sequence_stay(hip):
    b = Batch(BF16, 8, 2, 64, 16, [20, 9], [20, 50], seed=13)
    q = torch.cat([b.q, b.q[:7]])
    out = torch.full((36, 8, 64), 7.0, dtype=BF16, device="cuda")
    kv.prompt(q, b.cache, b.tables, b.lens, b.cu, out=out)
    assert (out[29:] == 7).all()
    assert torch.equal(out[:29], kv.prompt(b.q, b.cache, b.tables, b.lens, b.cu))


@pytest.mark.parametrize("cu", [[0, 20, 9], [-5, 20, 1000], [29, 0, 29], [7, 3, 1]])
def test_row_bounds_that_are_wrong(hip, cu):
    """Bounds out of order or of range: nothing outside the rows is read or written, rows of sound sequences
    are theirs."""
    b = Batch(BF16, 8, 2, 64, 16, [20, 9], [20, 50], seed=13)
    bad = torch.tensor(cu, dtype=torch.int32, device="cuda")
    store = torch.full((29 + 128, 8, 64), 7.0, dtype=BF16, device="cuda")
    kv.prompt(b.q, b.cache, b.tables, b.lens, bad, out=store[64:93])
    torch.cuda.synchronize()
    assert (store[:64] == 7).all() and (store[93:] == 7).all()


def test_strides(hip):
    """Queries as a part of wider rows at an odd offset, tables as a part of wider ones."""
    b = Batch(BF16, 8, 2, 64, 16, [1] * 5, [9, 30, 100, 0, 55], seed=14, width=9)
    wide = torch.zeros(5, 8 * 64 + 33, dtype=BF16, device="cuda")
    q = wide.as_strided((5, 8, 64), (8 * 64 + 33, 64, 1), 11)
    q.copy_(b.q)
    tables = torch.full((5, 23), 2 ** 30, dtype=torch.int32, device="cuda")
    tables[:, 3:12] = b.tables
    want = kv.decode(b.q, b.cache, b.tables, b.lens)
    assert torch.equal(kv.decode(q, b.cache, tables[:, 3:12], b.lens), want)
    cu = torch.arange(6, dtype=torch.int32, device="cuda")
    p = kv.prompt(b.q, b.cache, b.tables, b.lens, cu)
    assert torch.equal(kv.prompt(q, b.cache, tables[:, 3:12], b.lens, cu), p)
    for i, n in enumerate(b.lens_list):
        w, tol = reference(b.q[i:i + 1], b.k[i], b.v[i], 1 / 8, n - 1)
        close(p[i:i + 1], w, tol)


def test_same_bits(hip):
    b = Batch(BF16, 32, 4, 128, 64, [1] * 6, [4000, 1, 700, 90, 3000, 2], seed=15, width=100)
    want = kv.decode(b.q, b.cache, b.tables, b.lens)
    for _ in range(5):
        assert torch.equal(kv.decode(b.q, b.cache, b.tables, b.lens), want)
    # a place of its own in the batch does not matter to a sequence that is not split
    c = Batch(F16, 8, 2, 64, 16, [70, 30], [200, 60], seed=16)
    y = kv.prompt(c.q, c.cache, c.tables, c.lens, c.cu)
    alone = kv.prompt(c.q[70:], c.cache, c.tables[1:], c.lens[1:], torch.tensor([0, 30], dtype=torch.int32, device="cuda"))
    assert torch.equal(y[70:], alone)


def test_empty_calls(hip):
    b = Batch(BF16, 8, 2, 64, 16, [0, 0], [5, 0], seed=17)
    assert kv.prompt(b.q, b.cache, b.tables, b.lens, b.cu).shape == (0, 8, 64)
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    q = torch.empty(0, 8, 64, dtype=BF16, device="cuda")
    assert kv.decode(q, b.cache, torch.empty(0, 3, dtype=torch.int32, device="cuda"), none).shape == (0, 8, 64)


def test_streams_and_graphs(hip):
    """Two graphs of a decode, one of a prompt, replayed in turn with eager work between, lengths changing under
    them; another stream."""
    b = Batch(BF16, 32, 4, 128, 64, [1] * 5, [3000, 40, 700, 2, 1500], seed=18, width=60)
    p = Batch(F16, 8, 2, 64, 16, [90, 31], [200, 31], seed=19)
    outs = [torch.empty(5, 32, 128, dtype=BF16, device="cuda") for _ in range(2)]
    lens = [b.lens.clone(), b.lens.clone()]
    y = torch.empty(121, 8, 64, dtype=F16, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        for o, n in zip(outs, lens):
            kv.decode(b.q, b.cache, b.tables, n, out=o)
        kv.prompt(p.q, p.cache, p.tables, p.lens, p.cu, out=y)
        side.synchronize()
        for o, n in zip(outs, lens):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                kv.decode(b.q, b.cache, b.tables, n, out=o)
            graphs.append(g)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            kv.prompt(p.q, p.cache, p.tables, p.lens, p.cu, out=y)
    torch.cuda.synchronize()
    want_p = kv.prompt(p.q, p.cache, p.tables, p.lens, p.cu)
    for i in range(4):
        for j, n in enumerate(lens):
            n.copy_(torch.clamp(b.lens - 300 * i * (j + 1), min=0))
        y.zero_()
        for gr in (*graphs, g):
            gr.replay()
        torch.cuda.synchronize()
        for o, n in zip(outs, lens):
            assert torch.equal(o, kv.decode(b.q, b.cache, b.tables, n)), i
        assert torch.equal(y, want_p)


def test_far_pages(hip):
    """Pages past 2^31 elements and 2^32 bytes of a cache; decode whole and in shares, prompt."""
    lens = [300, 70]
    for width in (None, 40):
        b = Batch(BF16, 16, 8, 256, 64, [1, 1], lens, seed=20, spare=20000, width=width, last=True)
        assert min(b.tables_list[0]) * b.cache.k[0].numel() > 2 ** 31
        check_decode(b)
        del b
    b = Batch(BF16, 16, 8, 256, 64, [50, 70], lens, seed=21, spare=20000, last=True)
    check_prompt(b)
    # and appended there: what a second cache of few pages gets
    x = torch.randn(120, 32 * 256, generator=gen(22), device="cuda")
    q = kv.append(b.cache, x, 16, b.tables, b.lens, b.cu)
    c = Batch(BF16, 16, 8, 256, 64, [50, 70], lens, seed=21)
    assert torch.equal(q, kv.append(c.cache, x, 16, c.tables, c.lens, c.cu))
    for i, n in enumerate(lens):
        for a in ("keys", "values"):
            assert torch.equal(getattr(b.cache, a)(b.tables_list[i])[:, :n], getattr(c.cache, a)(c.tables_list[i])[:, :n])


def test_rows_past_32_bits(hip):
    """A batch whose queries, rows and results pass 2^31 elements: 1400 sequences of 100 rows of 64 heads of 256."""
    B, n, H, hd = 1400, 100, 64, 256
    cache = kv.Cache(B * 7, 1, hd, page=16, dtype=BF16)
    tables = torch.arange(B * 7, dtype=torch.int32, device="cuda").view(B, 7)
    lens = torch.full((B,), n, dtype=torch.int32, device="cuda")
    cu = (torch.arange(B + 1, device="cuda") * n).to(torch.int32)
    x = torch.randn(B * n, (H + 2) * hd, generator=gen(23), device="cuda", dtype=BF16)
    q = kv.append(cache, x, H, tables, lens, cu)
    assert torch.equal(q.view(B * n, -1), x[:, :H * hd])
    y = kv.prompt(q, cache, tables, lens, cu)
    last = torch.empty(B, H, hd, dtype=BF16, device="cuda")
    kv.decode(q[n - 1::n], cache, tables, lens, out=last)
    for b in (0, 700, B - 1):
        k, v = cache.keys(tables[b].tolist())[:, :n].transpose(0, 1), cache.values(tables[b].tolist())[:, :n].transpose(0, 1)
        assert torch.equal(k.reshape(n, hd), x[b * n:(b + 1) * n, H * hd:(H + 1) * hd])
        want, tol = reference(q[b * n:(b + 1) * n], k, v, 1 / 16, 0)
        close(y[b * n:(b + 1) * n], want, tol)
        close(last[b:b + 1], want[-1:], tol[-1:])


def test_two_streams_at_once(hip):
    """Decodes of one cache on two streams at a time, each with a workspace of its own."""
    b = Batch(BF16, 32, 4, 128, 64, [1] * 5, [3000, 40, 700, 2, 1500], seed=24, width=60)
    c = Batch(BF16, 32, 4, 128, 64, [1] * 5, [3000, 40, 700, 2, 1500], seed=24, width=60)
    lens2 = torch.tensor([100, 40, 699, 0, 1499], dtype=torch.int32, device="cuda")
    want = [kv.decode(c.q, c.cache, c.tables, n) for n in (c.lens, lens2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(20):
        for s, n, o in zip(streams, (b.lens, lens2), outs):
            with torch.cuda.stream(s):
                o.append(kv.decode(b.q, b.cache, b.tables, n))
    torch.cuda.synchronize()
    for w, o in zip(want, outs):
        assert all(torch.equal(w, y) for y in o)
