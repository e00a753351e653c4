"""Block scales at the ends of the float range: a product of two scales that is no float itself does not
spoil a result that is one.  Weight scales are between 2^-96 and 2^96, activation scales between 2^-126 and 2^126.

Tolerance: (127 + nb + 2) 2^-24 of the sum of magnitudes, and half a subnormal step, 2^-150, for each of the nb
sums where results end that low."""
import pytest
import torch

from tests.test_fp8_kernel_choice import SIZES
from tests.test_hip_fp8 import E4M3, gen, matrix, randn, values
from tierlm_amd import fp8

pytestmark = pytest.mark.gpu
every_kernel = pytest.mark.parametrize("name", SIZES)


def check(Y, w, s, codes, scale, n):
    X = (codes.double() * scale.double().repeat_interleave(128, 1))[:, :n]
    W = values(w, s)
    nb = -(-n // 128)
    want, mags = X @ W.T, X.abs() @ W.abs().T
    assert want.abs().max().item() < 2.0 ** 127
    tol = (127 + nb + 2) * 2.0 ** -24 * mags + nb * 2.0 ** -150
    assert torch.isfinite(Y).all()
    assert ((Y.double() - want).abs() <= tol).all(), ((Y.double() - want).abs() / tol).max().item()


@every_kernel
def test_the_smallest_activations(hip, name):
    """The quantiser's least scale, 2^-126, with weight scales below 1: the product of the two is subnormal."""
    T, rows, n = SIZES[name]
    g = gen(T + rows + 10)
    w, s = matrix(g, rows, n)
    s *= 0.02
    x = randn(g, T, n) * 2.0 ** -121
    x[T // 2] *= 2.0 ** -10                                # codes of small tokens go down to the subnormal ones
    codes, scale = fp8.quantize(x)
    assert scale.min().item() == 2.0 ** -126
    check(fp8.matmul(fp8.pack(w, s), rows, n, codes, scale), w, s, codes, scale, n)


@every_kernel
def test_the_largest_activations(hip, name):
    """Scales whose product is past the floats, codes that bring the result back; rows and tokens of zeros
    give zeros."""
    T, rows, n = SIZES[name]
    g = gen(T + rows + 11)
    nb = -(-n // 128)
    w = torch.randint(0, 8, (rows, n), generator=g, device="cuda", dtype=torch.uint8).view(E4M3)     # up to 7 * 2^-9
    x = torch.zeros(T, nb * 128, device="cuda", dtype=torch.uint8)
    x[:, :n:16] = torch.randint(0, 8, (T, -(-n // 16)), generator=g, device="cuda", dtype=torch.uint8)
    x, s = x.view(E4M3), torch.full((-(-rows // 128), nb), 2.0 ** 20, device="cuda")
    scale = torch.full((T, nb), 2.0 ** 108, device="cuda")
    w.view(torch.uint8)[5] = 0
    if T > 1:
        x.view(torch.uint8)[T // 2] = 0
    Y = fp8.matmul(fp8.pack(w, s), rows, n, x, scale)
    check(Y, w, s, x, scale, n)
    assert (Y[:, 5] == 0).all() and (T == 1 or (Y[T // 2] == 0).all())


@every_kernel
def test_scales_far_apart(hip, name):
    """Every power of two that a token's blocks can have, against weight scales that bring them together."""
    T, rows, n = SIZES[name]
    g = gen(T + rows + 12)
    w, s = matrix(g, rows, n)
    codes, scale = fp8.quantize(randn(g, T, n))
    nb = scale.shape[1]
    up = torch.randint(-85, 86, (nb,), generator=g, device="cuda").float()
    scale *= torch.exp2(up)
    s *= torch.exp2(-up)
    check(fp8.matmul(fp8.pack(w, s), rows, n, codes, scale), w, s, codes, scale, n)
