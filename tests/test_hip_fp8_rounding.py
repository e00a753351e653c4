"""The sums of the 8-bit product are float sums whatever the result's type: a 16-bit result is the
float result rounded once, so it is off the definition by half a step of its type and by the sum's own
roundings, (127 + nb + 2) 2^-24 of the sum of magnitudes, and by nothing else."""
import pytest
import torch

from tests.test_hip_fp8 import HALF_STEP, gen, matrix, randn, values
from tierlm_amd import fp8

pytestmark = pytest.mark.gpu

# (T, rows, n): few tokens, row groups, tiles of each size, part tiles and part blocks
SIZES = [(1, 40, 300), (16, 512, 2048), (33, 300, 1500), (40, 4096, 1024), (100, 5000, 256), (130, 4100, 700),
         (250, 16300, 300), (250, 65300, 200), (300, 5000, 2000), (66, 16901, 1590), (1024, 2100, 512)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,rows,n", SIZES)
def test_16_bit_results_are_the_float_results_rounded(hip, T, rows, n, dtype):
    """Activations whose channels spread over decades, where a sum of fewer bits shows most."""
    g = gen(T + rows + n)
    w, s = matrix(g, rows, n)
    P = fp8.pack(w, s)
    codes, scale = fp8.quantize(randn(g, T, n) * torch.exp(1.5 * randn(g, n)))
    Y = fp8.matmul(P, rows, n, codes, scale, dtype=dtype)
    assert torch.equal(Y, fp8.matmul(P, rows, n, codes, scale).to(dtype))
    X = (codes.double() * scale.double().repeat_interleave(128, 1))[:, :n]
    W = values(w, s)
    want, size = X @ W.T, X.abs() @ W.abs().T
    sums = (127 + -(-n // 128) + 2) * 2.0 ** -24 * size
    tol = sums + HALF_STEP[dtype] * (want.abs() + sums) + 2.0 ** -25 * (dtype == torch.float16)
    assert ((Y.double() - want).abs() <= tol).all()
