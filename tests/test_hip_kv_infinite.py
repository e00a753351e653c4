"""Attention over keys and values that are not finite, where a weight is 0: scores of minus infinity, and infinite values whose
weight rounds to 0.  Whole sequences and shares, every number of rows a group, positions split over groups."""
import math

import pytest
import torch

from tests.kv_ref import Batch, close, reference
from tierlm_amd import kv

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32

# new rows, positions, heads, key heads, head_dim, width of the tables: 32 rows a group, 64, 128 (narrow and wide heads), parts
PROMPTS = [([150, 7], [150, 400], 8, 2, 64, None), ([290], [700], 16, 2, 128, None), ([200, 0, 151], [200, 3, 300], 208, 16, 64, None),
           ([300], [340], 416, 16, 256, None), ([40, 3], [2900, 2000], 8, 2, 64, 200), ([60], [2300], 16, 2, 256, 200)]


def below(b, upto):
    """Scores of minus infinity at the positions before upto[i] of sequence i: queries are positive there."""
    b.q[..., 3] = b.q[..., 3].abs() + 1
    for i, n in enumerate(upto):
        b.k[i] = b.k[i].clone()
        b.k[i][:n, :, 3] = -math.inf
        b.put(i, b.k[i], b.v[i])


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("width", [None, 300])
def test_decode_scores_of_minus_infinity(hip, dtype, width):
    """All of them: NaN.  Some: weights of 0.  No position: zeros."""
    lens = [200, 1, 0, 90, 400, 33] if width is None else [3000, 1, 0, 90, 2500, 33]
    b = Batch(dtype, 8, 2, 64, 16, [1] * 6, lens, seed=41, width=width)
    below(b, [lens[0], 1, 0, 50, lens[4] - 1, 0])
    b.tables[3, 5] = -1                                   # positions 80 .. 89
    got = kv.decode(b.q, b.cache, b.tables, b.lens, dtype=F32)
    assert torch.isnan(got[:2]).all() and (got[2] == 0).all()
    for i, lo, hi in ((3, 50, 80), (4, lens[4] - 1, lens[4]), (5, 0, 33)):
        want, tol = reference(b.q[i:i + 1], b.k[i][lo:hi], b.v[i][lo:hi], 1 / 8, 10 ** 6)
        close(got[i:i + 1], want, tol, f"sequence {i}")
    # only the pages that are none are left beside scores of minus infinity, or they are all there is
    b.tables[3, 3:] = -1
    b.tables[4] = -1
    got = kv.decode(b.q, b.cache, b.tables, b.lens, dtype=F32)
    assert torch.isnan(got[3]).all() and (got[4] == 0).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("new,lens,heads,kv_heads,hd,width", PROMPTS)
def test_prompt_scores_of_minus_infinity(hip, dtype, new, lens, heads, kv_heads, hd, width):
    """Rows that see nothing else are NaN, those behind them as if these positions were not there."""
    for cut in (None, 1):                                 # up to the middle of the new rows, or all but the last row's own
        b = Batch(dtype, heads, kv_heads, hd, 16, new, lens, seed=42, width=width)
        upto = [m - (n + 1) // 2 if cut is None else m - cut for n, m in zip(new, lens)]
        below(b, upto)
        got = kv.prompt(b.q, b.cache, b.tables, b.lens, b.cu, dtype=F32)
        for i, (n, m) in enumerate(zip(new, lens)):
            if n == 0:
                continue
            rows = got[b.cu_list[i]:b.cu_list[i + 1]]
            first = upto[i] - (m - n)                     # the first row that sees a finite score
            assert torch.isnan(rows[:first]).all()
            want, tol = reference(b.q[b.cu_list[i] + first:b.cu_list[i + 1]], b.k[i][upto[i]:], b.v[i][upto[i]:],
                                  1 / math.sqrt(hd), 0)
            close(rows[first:], want, tol, f"sequence {i}")


def test_prompt_pages_that_are_none_beside_them(hip):
    """Rows whose positions are on no page get zeros, those that see a score of minus infinity beside them NaN."""
    for width in (None, 200):
        b = Batch(F16, 8, 2, 64, 16, [60], [60 if width is None else 2560], seed=43, width=width)
        m = b.lens_list[0]
        below(b, [m])
        b.tables[0, :-(-m // 16) - 2] = -1                # all but the last two pages
        got = kv.prompt(b.q, b.cache, b.tables, b.lens, b.cu, dtype=F32)
        named = (b.tables[0].repeat_interleave(16)[:m] >= 0).nonzero()[0].item()
        sees = torch.arange(m - 60, m, device="cuda") >= named
        assert (got[~sees] == 0).all() and torch.isnan(got[sees]).all() and sees.any() and not sees.all()


def lowered(b, first, last, by):
    """Scores of the positions first .. last of every sequence lowered by `by` powers of two of weight or more (queries of at
    least 1, keys of 0 elsewhere)."""
    hd = b.cache.head_dim
    b.q[..., 3] = b.q[..., 3].abs() + 1
    for i, k in enumerate(b.k):
        k = k.clone()
        k[..., 3] = 0
        k[first:last + 1, :, 3] = -by * math.sqrt(hd)
        b.k[i] = k
        b.put(i, k, b.v[i])


def planted(b, i, at, value):
    v = b.v[i].clone()
    for p, x in zip(at, value):
        v[p, :, 5] = x
    b.put(i, b.k[i], v)


def arrives(rows, value):
    total = sum(value)
    return torch.isnan(rows).all() if math.isnan(total) else (rows == total).all()


INF = math.inf
# where (a share of the sequence's positions), and what
PLACES = [((0.0,), (INF,)), ((0.45,), (-INF,)), ((0.1, 0.3), (INF, INF)), ((0.05, 0.8), (INF, -INF)), ((0.2,), (math.nan,)),
          ((0.99,), (-INF,))]


@pytest.mark.parametrize("dtype,by", [(F16, 45.0), (F16, 300.0), (BF16, 300.0)])
@pytest.mark.parametrize("width", [None, 300])
@pytest.mark.parametrize("heads,kv_heads,hd", [(8, 2, 64), (40, 1, 64), (16, 2, 256)])
def test_decode_infinite_values_of_no_weight(hip, dtype, by, width, heads, kv_heads, hd):
    """The first half's weights round to 0, its infinities come through all the same; the others' bits stay."""
    lens = [300, 100, 40] if width is None else [4000, 100, 1500]
    for half in (True, False):                            # the first half, or the first planted position alone
        for where, value in PLACES:
            at = [int(x * lens[0]) for x in where]
            b = Batch(dtype, heads, kv_heads, hd, 16, [1] * 3, lens, seed=44, width=width)
            lowered(b, 0 if half else at[0], lens[0] // 2 if half else at[0], by)
            want = kv.decode(b.q, b.cache, b.tables, b.lens, dtype=F32)
            planted(b, 0, at, value)
            got = kv.decode(b.q, b.cache, b.tables, b.lens, dtype=F32)
            assert arrives(got[0, :, 5], value), (where, value)
            keep = torch.arange(hd, device="cuda") != 5
            assert torch.equal(got[0][:, keep], want[0][:, keep]) and torch.equal(got[1:], want[1:])


@pytest.mark.parametrize("dtype,by", [(F16, 45.0), (F16, 300.0), (BF16, 300.0)])
@pytest.mark.parametrize("new,lens,heads,kv_heads,hd,width", PROMPTS)
def test_prompt_infinite_values_of_no_weight(hip, dtype, by, new, lens, heads, kv_heads, hd, width):
    """As in decode, for the rows that see them; inside the positions that all rows see and at the border."""
    n, m = new[0], lens[0]
    for half in (True, False):
        for where, value in PLACES:
            at = [int(x * m) for x in where]
            b = Batch(dtype, heads, kv_heads, hd, 16, new, lens, seed=45, width=width)
            lowered(b, 0 if half else at[0], m // 2 if half else at[0], by)
            want = kv.prompt(b.q, b.cache, b.tables, b.lens, b.cu, dtype=F32)
            planted(b, 0, at, value)
            got = kv.prompt(b.q, b.cache, b.tables, b.lens, b.cu, dtype=F32)
            keep = torch.arange(hd, device="cuda") != 5
            assert torch.equal(got[:, :, keep], want[:, :, keep]) and torch.equal(got[n:], want[n:])
            edges = [max(0, p - (m - n)) for p in at] + [n]      # the first rows that see each
            assert torch.equal(got[:edges[0]], want[:edges[0]])
            for j in range(len(at)):
                assert arrives(got[edges[j]:edges[j + 1], :, 5], value[:j + 1]), (where, value, j)


def test_rows_that_are_nan_stay(hip):
    """A NaN query beside an infinite value: its row is NaN, the others have the infinity."""
    for width in (None, 300):
        b = Batch(BF16, 8, 2, 64, 16, [1] * 2, [300, 300], seed=46, width=width)
        b.q[1, 2, 0] = math.nan
        for i in range(2):
            planted(b, i, [7], [INF])
        got = kv.decode(b.q, b.cache, b.tables, b.lens, dtype=F32)
        keep = torch.arange(8, device="cuda") != 2
        assert torch.isnan(got[1, 2]).all() and (got[1, keep, 5] == INF).all() and (got[0, :, 5] == INF).all()
        assert not torch.isnan(got[0]).any() and not torch.isnan(got[1, keep]).any()
        b = Batch(F16, 8, 2, 64, 16, [90], [400], seed=47, width=width)
        b.q[33, 2, 0] = math.nan
        planted(b, 0, [20], [-INF])
        got = kv.prompt(b.q, b.cache, b.tables, b.lens, b.cu, dtype=F32)
        rows = torch.ones(90, 8, dtype=torch.bool, device="cuda")
        rows[33, 2] = False
        assert torch.isnan(got[33, 2]).all() and (got[rows][:, 5] == -INF).all() and not torch.isnan(got[rows]).any()
