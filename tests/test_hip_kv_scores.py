"""Attention where one position's score, or two equal ones', is far above every other: the weights are 1 or 1/2 and 0, so the
result is that position's value, or the two's mean, however large the scores are.

Scores are whole numbers times a power of two and exact in f32, different ones at least 2^10 powers of two of weight apart.
Tolerance: a weight is rounded once to the cache's type and stands over a sum of unrounded ones (f32, an exponential to 2^-22
beside it), the result once to its own."""
import math

import pytest
import torch

from tests.kv_ref import HALF_STEP, Batch
from tierlm_amd import kv

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
UNIT = 2.0 ** 6


def peaked(b, sign, seed):
    """Queries and keys whose scores are sign UNIT n, n whole numbers from 2^13 to 2^14 in random order, each twice.  Returns
    the numbers of each sequence."""
    g = torch.Generator().manual_seed(seed)
    b.q.zero_()
    b.q[..., :2] = sign * UNIT
    numbers = []
    for i, m in enumerate(b.lens_list):
        n = 2 ** 13 + torch.randperm(2 ** 13, generator=g)[:m // 2 + 1].repeat(2)[torch.randperm(m // 2 * 2 + 2, generator=g)][:m]
        n = n.cuda()
        k = torch.zeros_like(b.k[i])
        k[..., 0] = (n // 128 * 128)[:, None].to(k.dtype)
        k[..., 1] = (n % 128)[:, None].to(k.dtype)
        assert torch.equal(k.double().sum(-1), n.double()[:, None].expand(-1, k.shape[1]))
        b.k[i] = k
        b.put(i, k, b.v[i])
        numbers.append(n * sign)
    return numbers


def check(got, numbers, v, first, heads, dtype):
    """Rows of one sequence: row i sees the positions 0 .. first + i."""
    n, m = got.shape[0], v.shape[0]
    group = heads // v.shape[1]
    sees = torch.arange(m, device="cuda")[None] <= (first + torch.arange(n, device="cuda"))[:, None]
    s = numbers.double()[None].expand(n, m).masked_fill(~sees, -math.inf)
    p = (s == s.amax(1, keepdim=True)).double()
    p = p / p.sum(1, keepdim=True)
    vv = v.double().repeat_interleave(group, 1).permute(1, 0, 2).contiguous()         # [heads, m, hd]
    want = torch.stack([p @ x for x in vv], 1)
    mag = torch.stack([p @ x.abs() for x in vv], 1)
    err = (got.double() - want).abs()
    bound = mag * (HALF_STEP[dtype] + 2.0 ** -20) + want.abs() * HALF_STEP[got.dtype]
    assert (err <= bound).all(), (int((~(err <= bound)).sum()), err.numel(), float((err / bound.clamp(min=1e-300)).max()))


POWERS = [24, 26, 27, 28, 29, 30, 31, 32, 33, 34, 60, 120, 140]       # scores as powers of two of weight: 2^24 .. 2^140


def scale_of(power, i):
    """A scale that is no power of two itself and brings the largest score near 2^power powers of two."""
    return 2.0 ** (power - 20) * (1.0, 1.234567, 1.41421, 1.87)[i % 4] * math.log(2.0)


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("width", [None, 200])
def test_decode(hip, dtype, width, sign):
    """A sequence a group, and in shares (a wide table)."""
    lens = [1, 2, 17, 130, 300, 400] if width is None else [1, 300, 2900, 40, 1200]
    b = Batch(dtype, 8, 2, 64, 16, [1] * len(lens), lens, seed=31, width=width)
    numbers = peaked(b, sign, 32)
    for i, power in enumerate(POWERS):
        got = kv.decode(b.q, b.cache, b.tables, b.lens, scale=scale_of(power, i), dtype=F32)
        for j, m in enumerate(lens):
            check(got[j:j + 1], numbers[j], b.v[j], m - 1, 8, dtype)


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("new,lens,heads,kv_heads,hd,width", [
    ([150, 7], [150, 400], 8, 2, 64, None),           # 32 rows a group
    ([290], [700], 16, 2, 128, None),                 # 64
    ([200, 0, 151], [200, 3, 300], 208, 16, 64, None),    # 128
    ([60], [90], 8, 2, 256, None),
    ([40, 3], [2900, 2000], 8, 2, 64, 200)])          # positions split over groups
def test_prompt(hip, dtype, new, lens, heads, kv_heads, hd, width, sign):
    b = Batch(dtype, heads, kv_heads, hd, 16, new, lens, seed=33, width=width)
    numbers = peaked(b, sign, 34)
    for i, power in enumerate(POWERS):
        got = kv.prompt(b.q, b.cache, b.tables, b.lens, b.cu, scale=scale_of(power, i), dtype=F32)
        for j, (n, m) in enumerate(zip(new, lens)):
            check(got[b.cu_list[j]:b.cu_list[j + 1]], numbers[j], b.v[j], m - n, heads, dtype)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_neighbours_keep_their_bits(hip, dtype):
    """A row of far scores among ordinary ones changes nothing for them."""
    for new, lens, H, KV, hd in (([150], [400], 8, 2, 64), ([290], [700], 16, 2, 128), ([300], [300], 208, 16, 64), ([60], [2900], 8, 2, 64)):
        b = Batch(dtype, H, KV, hd, 16, new, lens, seed=35, width=200)
        want = kv.prompt(b.q, b.cache, b.tables, b.lens, b.cu, dtype=F32)
        q = b.q.clone()
        q[5] *= 1000.0
        got = kv.prompt(q, b.cache, b.tables, b.lens, b.cu, dtype=F32)
        keep = torch.arange(new[0], device="cuda") != 5
        assert torch.equal(got[keep], want[keep]) and not torch.equal(got[5], want[5])


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("scale", [1e-30, 1e-38, 2e-44])
def test_tiny_scales(hip, dtype, scale):
    """Scales down to floats without a leading one: every weight is the same."""
    from tests.kv_ref import close, reference
    for lens, width in (([1, 33, 300], None), ([2900, 40], 200)):
        b = Batch(dtype, 8, 2, 64, 16, [1] * len(lens), lens, seed=36, width=width)
        got = kv.decode(b.q, b.cache, b.tables, b.lens, scale=scale, dtype=F32)
        for i, n in enumerate(lens):
            want, tol = reference(b.q[i:i + 1], b.k[i], b.v[i], scale, n - 1)
            close(got[i:i + 1], want, tol)
        p = Batch(dtype, 8, 2, 64, 16, [40], [lens[0] + 40], seed=37, width=width)
        got = kv.prompt(p.q, p.cache, p.tables, p.lens, p.cu, scale=scale, dtype=F32)
        want, tol = reference(p.q, p.k[0], p.v[0], scale, lens[0])
        close(got, want, tol)
