"""The residual's addition, RMS norm and E4M3 codes in one call: the sum bit for bit, the codes and scales bit for bit
those of the quantiser on the same f32 values (the mean in double, its root's reciprocal rounded once, two f32
products), and the definition in 64 bits within the code's half step."""
import math

import numpy as np
import pytest
import torch

from tierlm_amd import fp8

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
EPS = 2.0 ** -20


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def inputs(T, n, hdt, xdt, seed=0):
    g = gen(seed)
    big = torch.exp(0.5 * torch.randn(n, generator=g, device="cuda"))
    h = (torch.randn(T, n, generator=g, device="cuda") * big).to(hdt)
    x = (torch.randn(T, n, generator=g, device="cuda") * big).to(xdt)
    return h, x, 1 + 0.1 * torch.randn(n, generator=g, device="cuda")


def steps(h, x, w, eps=EPS):
    """The definition's roundings, one by one."""
    s = (h.float() + x.float()).to(h.dtype) if x is not None else h
    f = s.float().cpu().numpy()
    mean = (f.astype(np.float64) ** 2).sum(1, keepdims=True) / f.shape[1]
    with np.errstate(all="ignore"):
        r = (1.0 / np.sqrt(mean + np.float64(np.float32(eps)))).astype(np.float32)
        y = (f * r) * w.cpu().numpy()
    return s, torch.from_numpy(y).to(h.device)


def same(a, b):
    return torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("hdt", [F32, F16, BF16])
@pytest.mark.parametrize("xdt", [F32, F16, BF16])
@pytest.mark.parametrize("T,n", [(1, 1), (3, 127), (2, 512), (5, 513), (7, 1111), (1, 2048), (3, 1024), (3, 1025), (3, 2049), (2, 4096), (2, 4097), (2, 5000), (2, 6144), (3, 6145),
                                 (2, 8192), (2, 8193),
                                 (3, 9001), (1, 16384), (2, 16385), (1, 40000)])
def test_against_the_quantiser(hip, hdt, xdt, T, n):
    h, x, w = inputs(T, n, hdt, xdt, seed=n)
    s, y = steps(h, x, w)
    want = fp8.quantize(y)
    codes, scale = fp8.add_rmsnorm(h, x, w, EPS)
    assert same(h, s)
    assert same(codes, want[0]) and same(scale, want[1])
    # another place for the sum, and none added
    h2, x2, _ = inputs(T, n, hdt, xdt, seed=n)
    out = torch.empty_like(h2)
    codes, scale = fp8.add_rmsnorm(h2, x2, w, EPS, out=out)
    assert same(out, s) and same(h2, inputs(T, n, hdt, xdt, seed=n)[0]) and same(codes, want[0]) and same(scale, want[1])
    codes, scale = fp8.add_rmsnorm(s, None, w, EPS)
    assert same(codes, want[0]) and same(scale, want[1])


@pytest.mark.parametrize("n", [700, 20000])
def test_sum_not_stored(hip, n):
    """The C call without a place for the sum: h stays, the codes are those of the sum."""
    from tierlm_amd import lib
    h, x, w = inputs(3, n, F16, BF16, seed=n)
    s, y = steps(h, x, w)
    want, keep = fp8.quantize(y), h.clone()
    codes, scale = torch.empty_like(want[0]), torch.empty_like(want[1])
    rc = lib.tlm_hip_fp8_add_rmsnorm(1, h.data_ptr(), n, 2, x.data_ptr(), n, w.data_ptr(), EPS, n, 3, None, 0,
                                     codes.data_ptr(), scale.data_ptr(), torch.cuda.current_stream().cuda_stream)
    assert rc == 0 and same(h, keep) and same(codes, want[0]) and same(scale, want[1])


@pytest.mark.parametrize("n", [100, 2048, 20000])
def test_definition(hip, n):
    """64 bits: r, s r and y are off by at most 2^-24 each of themselves (three roundings), the code by half its step."""
    h, x, w = inputs(4, n, F32, F32, seed=n)
    s = (h + x).double()
    y = s * torch.rsqrt(s.square().mean(1, keepdim=True) + EPS) * w.double()
    codes, scale = fp8.add_rmsnorm(h, x, w, EPS)
    nb = scale.shape[1]
    got = codes.float().double().view(4, nb, 128) * scale.double()[..., None]
    got = got.view(4, -1)[:, :n]
    step = scale.double().repeat_interleave(128, 1)[:, :n] * 2.0 ** -9
    assert ((got - y).abs() <= y.abs() * (2.0 ** -4 + 4 * 2.0 ** -24) + step / 2 * 1.001).all()


def test_strides(hip):
    T, n = 9, 333
    h, x, w = inputs(T, n, F16, BF16, seed=3)
    want_h = h.clone()
    want = fp8.add_rmsnorm(want_h, x, w, EPS)
    store = torch.zeros(T * 500, dtype=F16, device="cuda")
    hs = store.as_strided((T, n), (400, 1), 7)
    hs.copy_(h)
    before = store.clone()
    xs = torch.zeros(T, n + 5, dtype=BF16, device="cuda")[:, 3:3 + n]
    xs.copy_(x)
    codes, scale = fp8.add_rmsnorm(hs, xs, w, EPS)
    assert same(codes, want[0]) and same(scale, want[1]) and torch.equal(hs, want_h)
    before.as_strided((T, n), (400, 1), 7).copy_(want_h)
    assert torch.equal(store, before)


def test_poison_and_zeros(hip):
    """A row of zeros gives zeros; infinities and NaN stay in their row."""
    h, x, w = inputs(6, 700, F32, F32, seed=4)
    want = fp8.add_rmsnorm(h.clone(), x, w, EPS)
    h2, x2 = h.clone(), x.clone()
    h2[1], x2[1] = 0, 0
    h2[2, 5], x2[4, 699] = math.inf, math.nan
    codes, scale = fp8.add_rmsnorm(h2, x2, w, EPS)
    for t in (0, 3, 5):
        assert same(codes[t], want[0][t]) and same(scale[t], want[1][t])
    assert (codes[1].float() == 0).all() and (scale[1] == 0).all()
    assert torch.isnan(scale[2, 0]) and torch.isnan(scale[4]).all()
    # all zeros without eps: 0 times infinity
    codes, scale = fp8.add_rmsnorm(torch.zeros(1, 130, device="cuda"), None, w[:130].contiguous(), 0.0)
    assert torch.isnan(scale).all()


@pytest.mark.parametrize("size", [1e-30, 1e-18, 1e18])
def test_sizes(hip, size):
    """Squares that a float does not hold."""
    h, x, w = inputs(3, 1000, F32, F32, seed=5)
    h, x = h * size, x * size
    s, y = steps(h, x, w, 0.0)
    codes, scale = fp8.add_rmsnorm(h, x, w, 0.0)
    want = fp8.quantize(y)
    assert same(codes, want[0]) and same(scale, want[1])


def test_graph_and_stream(hip):
    h, x, w = inputs(4, 2048, F32, BF16, seed=6)
    out = torch.empty_like(h)
    codes, scale = fp8.add_rmsnorm(h, x, w, EPS, out=out)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        fp8.add_rmsnorm(h, x, w, EPS, out=out, codes=codes, scale=scale)
    for i in range(3):
        h.copy_(inputs(4, 2048, F32, BF16, seed=7 + i)[0])
        g.replay()
        torch.cuda.synchronize()
        got = codes.clone(), scale.clone(), out.clone()
        want = fp8.add_rmsnorm(h, x, w, EPS, out=out)
        assert same(got[0], want[0]) and same(got[1], want[1]) and same(got[2], out)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = fp8.add_rmsnorm(h, x, w, EPS, out=out)
    side.synchronize()
    assert same(again[0], want[0])


def test_empty(hip):
    codes, scale = fp8.add_rmsnorm(torch.empty(0, 256, device="cuda"), torch.empty(0, 256, device="cuda"),
                                   torch.ones(256, device="cuda"))
    assert codes.shape == (0, 256) and scale.shape == (0, 2)
