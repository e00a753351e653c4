"""The paged cache where a batch is not all sound: steps with slots that have run empty, row bounds out of order or of range.
What is there is checked slot by slot, what is not stays as it was."""
import math

import pytest
import torch

from tests.kv_ref import Batch, close, gen, reference
from tests.test_hip_kv_layer import Layer, check, ints, tables_of
from tierlm_amd import fp8, kv

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def test_steps_with_slots_that_run_empty(hip):
    """Three sequences that end one after the other, the first slot first, and a slot that is never used: every live row
    against the definition, zeros for the others."""
    ends, page = [11, 39, 24], 16
    tables, pages = tables_of(ends + [16], page, 2)
    g, layer = gen(3), Layer(pages)
    for p in range(max(ends)):
        lens = [p + 1 if p < n else 0 for n in ends] + [0]
        h = torch.randn(4, Layer.D, generator=g, device="cuda")
        out, q, y = layer.attention(h, None, tables, ints(*lens))
        for i, n in enumerate(lens):
            if n:
                check(layer, q[i:i + 1], y[i:i + 1], tables[i:i + 1], [n], [1])
                assert (q[i] != 0).any() and (out[i] != 0).any()
            else:
                assert (q[i] == 0).all() and (y[i] == 0).all() and (out[i] == 0).all()


def test_a_layer_of_long_prompts(hip):
    """A whole layer for more rows than the MoE block takes at once: the block in pieces of 64."""
    new, page = [70, 9, 66], 16
    tables, pages = tables_of(new, page, 5)
    layer = Layer(pages)
    h = torch.randn(sum(new), Layer.D, generator=gen(6), device="cuda")
    with pytest.raises(Exception):
        layer.moe(h.clone())
    x, q, y = layer.attention(h, None, tables, ints(*new), ints(0, 70, 79, 145))
    check(layer, q, y, tables, new, new)
    h.add_(x)
    want = [layer.moe(piece.clone()) for piece in h.split(64)]
    for piece in h.split(fp8.MOE_MAX_TOKENS):
        layer.moe(piece)
    assert torch.equal(h, torch.cat(want)) and torch.isfinite(h).all()


# bounds, and what they are inside the rows: each sequence's first row and number of rows
BOUNDS = [([0, 20, 9], [(0, 20), (20, 0)]), ([-5, 20, 1000], [(0, 20), (20, 9)]), ([29, 0, 29], [(29, 0), (0, 29)]),
          ([7, 3, 1], [(7, 0), (3, 0)]), ([-9, -3, -1], [(0, 0), (0, 0)]), ([40, 50, 60], [(29, 0), (29, 0)]),
          ([2 ** 31 - 1, -2 ** 31, 5], [(29, 0), (0, 5)]), ([3, 3, 2 ** 31 - 1], [(3, 0), (3, 26)])]


@pytest.mark.parametrize("cu,have", BOUNDS)
@pytest.mark.parametrize("width", [None, 200])
def test_prompt_row_bounds_that_are_wrong(hip, cu, have, width):
    b = Batch(BF16, 8, 2, 64, 16, [20, 9], [20, 50], seed=13, width=width)
    store = torch.full((29 + 128, 8, 64), 7.0, dtype=BF16, device="cuda")
    kv.prompt(b.q, b.cache, b.tables, b.lens, ints(*cu), out=store[64:93])
    assert (store[:64] == 7).all() and (store[93:] == 7).all()
    out, left = store[64:93], torch.ones(29, dtype=torch.bool, device="cuda")
    for i, (lo, n) in enumerate(have):
        m = b.lens_list[i]
        none = max(0, n - m)                              # rows before the first position
        want, tol = reference(b.q[lo + none:lo + n], b.k[i], b.v[i], 1 / 8, m - n + none)
        close(out[lo + none:lo + n], want, tol, f"sequence {i}")
        assert (out[lo:lo + none] == 0).all()
        left[lo:lo + n] = False
    assert (out[left] == 7).all()


@pytest.mark.parametrize("cu,have", BOUNDS)
@pytest.mark.parametrize("page", [16, 64])
def test_append_row_bounds_that_are_wrong(hip, cu, have, page):
    """The rows that a sequence has are written at its last positions, bit for bit; nothing else of the cache changes."""
    heads, kv_heads, hd = 8, 2, 64
    b = Batch(F16, heads, kv_heads, hd, page, [20, 9], [20, 50], seed=13, spare=3)
    x = torch.randn(29 + 64, (heads + 2 * kv_heads) * hd, generator=gen(14), device="cuda")
    x[:32], x[61:] = math.nan, math.nan                   # rows that are not the call's
    x = x[32:61]
    store = torch.full((29 + 128, heads, hd), 7.0, dtype=F16, device="cuda")
    expect = Batch(F16, heads, kv_heads, hd, page, [20, 9], [20, 50], seed=13, spare=3)
    kv.append(b.cache, x, heads, b.tables, b.lens, ints(*cu), out=store[64:93])
    assert (store[:64] == 7).all() and (store[93:] == 7).all()
    q, left = store[64:93], torch.ones(29, dtype=torch.bool, device="cuda")
    rows = x.view(29, heads + 2 * kv_heads, hd).to(F16)
    for i, (lo, n) in enumerate(have):
        m = b.lens_list[i]
        none = max(0, n - m)
        expect.put(i, rows[lo + none:lo + n, heads:heads + kv_heads], rows[lo + none:lo + n, heads + kv_heads:], m - n + none)
        assert torch.equal(q[lo + none:lo + n], rows[lo + none:lo + n, :heads]) and (q[lo:lo + none] == 0).all()
        left[lo:lo + n] = False
    assert (q[left] == 7).all()
    for a, e in ((b.cache.k, expect.cache.k), (b.cache.v, expect.cache.v)):
        assert torch.equal(a.view(torch.int16), e.view(torch.int16))
