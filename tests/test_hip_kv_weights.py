"""Decode attention's weights enter the second product as two numbers of the cache's type, so a float result is off by the square of
that type's half step, the scores' own error and a sum's roundings, not by a half step of each weight."""
import math

import pytest
import torch

from tests.kv_ref import HALF_STEP, Batch
from tierlm_amd import kv

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def definition(q, k, v, scale):
    """One row's attention in 64 bits, and the bound on a float result's error (see kv_ref.reference for the scores' part)."""
    H, hd = q.shape
    m, KV, _ = k.shape
    out, tol = torch.zeros(H, hd, dtype=torch.float64, device=q.device), torch.zeros(H, hd, dtype=torch.float64, device=q.device)
    half = HALF_STEP[q.dtype]
    for h in range(H):
        kk, vv, qq = k[:, h // (H // KV)].double(), v[:, h // (H // KV)].double(), q[h].double()
        p = torch.softmax(kk @ qq * scale, 0)
        mag = float((kk.abs() @ qq.abs()).max() * scale)
        e = (hd + 6) * 2.0 ** -24 * mag + 2.0 ** -21
        out[h] = p @ vv
        # two numbers a weight: the second's half step is the square of one; in f16 it is no finer than 2^-25 beside weights
        # of 2^8; sums of m + 64 terms of either number
        tol[h] = (p @ vv.abs()) * (half * half + 2 * e + 4 * (m + 64) * 2.0 ** -24) + 2.0 ** -33 * vv.abs().sum(0)
    return out, tol


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("heads,kv_heads,hd", [(8, 2, 64), (40, 1, 64), (4, 4, 128), (17, 1, 256), (6, 2, 96), (4, 2, 32)])
@pytest.mark.parametrize("lens,width", [([1, 2, 33, 300], None), ([3000, 5, 1200], 200)])
def test_float_results(hip, dtype, heads, kv_heads, hd, lens, width):
    for scale in (0.02, 1 / math.sqrt(hd), 0.7):
        b = Batch(dtype, heads, kv_heads, hd, 16, [1] * len(lens), lens, seed=71, width=width)
        got = kv.decode(b.q, b.cache, b.tables, b.lens, scale=scale, dtype=F32)
        for i, n in enumerate(lens):
            want, tol = definition(b.q[i], b.k[i], b.v[i], scale)
            err = (got[i].double() - want).abs()
            bound = tol + want.abs() * HALF_STEP[F32]
            assert (err <= bound).all(), (n, scale, float((err / bound).max()))
