"""Query and key heads whose squares a float does not hold: their norms are the definition's, as the residual's norm is.
Tolerances as for ordinary sizes, counted in the append tests."""
import math

import pytest
import torch

from tests.kv_ref import HALF_STEP, Batch, gen
from tests.test_hip_kv_append import reference
from tierlm_amd import kv

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("xdtype,size,eps", [
    (F32, 1e20, 1e-6), (F32, 1e30, 0.0), (F32, 2e37, 1e-6), (BF16, 1e25, 1e-6), (BF16, 3e36, 0.0), (F32, 1e-22, 0.0), (F32, 1e-37, 0.0),
    (BF16, 1e-30, 0.0), (F32, 1e-30, 1e-6), (F32, 1e-20, 1e-38), (F32, 1e18, 1e-6)])
@pytest.mark.parametrize("hd", [32, 96, 128, 256])
def test_sizes(hip, dtype, xdtype, size, eps, hd):
    heads, kv_heads, n, m = 5, 1, 20, 50
    b = Batch(dtype, heads, kv_heads, hd, 16, [n], [m], seed=61)
    g = gen(62)
    x = torch.randn(n, (heads + 2) * hd, generator=g, device="cuda")
    x[:, :(heads + 1) * hd] *= size
    # every third row as it comes: ordinary sizes beside the others
    x[::3, :(heads + 1) * hd] /= size
    x = x.to(xdtype)
    qn, kn = (1 + 0.1 * torch.randn(hd, generator=g, device="cuda") for _ in range(2))
    freq = kv.rope_frequencies(hd, 1e6)
    q = kv.append(b.cache, x, heads, b.tables, b.lens, b.cu, q_norm=qn, k_norm=kn, eps=eps, inv_freq=freq)
    eps = float(torch.tensor(eps, dtype=F32))
    wq, wk, _, tol = reference(x, heads, kv_heads, hd, torch.arange(m - n, m, device="cuda"), qn, kn, eps, freq, 1.0)
    k = b.cache.keys(b.tables_list[0])[:, m - n:m].transpose(0, 1)
    tiny = 2.0 ** -25 if dtype is F16 else 2.0 ** -134
    for got, want, t in ((q, wq, tol[:, :heads]), (k, wk, tol[:, heads:])):
        err, bound = (got.double() - want).abs(), t + (want.abs() + t) * HALF_STEP[dtype] + tiny
        assert (err <= bound).all(), float((err / bound).max())


def test_ordinary_rows_keep_their_bits(hip):
    """Beside rows of every size, and with an infinity or NaN in another row."""
    b = Batch(BF16, 8, 2, 64, 16, [40], [40], seed=63)
    x = torch.randn(40, 12 * 64, generator=gen(64), device="cuda")
    w = torch.ones(64, device="cuda")
    want = kv.append(b.cache, x, 8, b.tables, b.lens, b.cu, q_norm=w, k_norm=w)
    keys = b.cache.keys(b.tables_list[0])[:, :40].clone()
    for value in (1e25, 0.0, 1e-30, math.inf, math.nan):
        y = x.clone()
        y[7], y[8, :300] = value, value
        q = kv.append(b.cache, y, 8, b.tables, b.lens, b.cu, q_norm=w, k_norm=w)
        keep = torch.ones(40, dtype=torch.bool, device="cuda")
        keep[7:9] = False
        assert torch.equal(q[keep], want[keep]) and torch.equal(b.cache.keys(b.tables_list[0])[:, :40][:, keep], keys[:, keep])
