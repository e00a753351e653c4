"""Every kernel of the 8-bit product on the inputs that are hard for it, all result types: whole code tables,
NaN and infinite codes and scales, results inside larger buffers, graphs and streams.

Tolerance: sums are float sums for results of every type, (127 + nb + 2) 2^-24 of the sum of magnitudes; a
16-bit result is rounded once more, half a step of its type (binary16's subnormal ones: 2^-25)."""
import pytest
import torch

from tests.test_fp8_kernel_choice import SIZES
from tests.test_hip_fp8 import E4M3, HALF_STEP, gen, matrix, randn, values
from tierlm_amd import fp8

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]
every_kernel = pytest.mark.parametrize("name", SIZES)
every_type = pytest.mark.parametrize("dtype", TYPES)


def size(name):
    T, rows, n = SIZES[name]
    assert fp8.matmul_kernel(rows, n, T) == name
    return T, rows, n


def check(Y, w, s, codes, scale, n, keep_t=slice(None), keep_r=slice(None)):
    W = values(w, s)[keep_r]
    X = (codes.double() * scale.double().repeat_interleave(128, 1))[keep_t, :n]
    Y = Y[keep_t][:, keep_r]
    want, mags = X @ W.T, X.abs() @ W.abs().T
    tol = (127 + -(-n // 128) + 2) * 2.0 ** -24 * mags
    if Y.dtype != torch.float32:
        tol += HALF_STEP[Y.dtype] * (want.abs() + tol) + 2.0 ** -25 * (Y.dtype == torch.float16)
    if Y.dtype == torch.float16:                       # past its largest number the result is an infinity
        big = want.abs() + tol >= 65520
        assert torch.equal(torch.isinf(Y)[~big], torch.zeros_like(big)[~big])
        Y, want = Y.masked_fill(big, 0), want.masked_fill(big, 0)
    off = (Y.double() - want).abs() - tol
    assert (off <= 0).all(), off.max().item()


@every_type
@every_kernel
def test_every_code(hip, name, dtype):
    """Every finite code on both sides; subnormal codes alone; scales of either sign."""
    T, rows, n = size(name)
    g = gen(T + rows)
    nb, np_ = -(-n // 128), -(-n // 128) * 128
    fin = torch.tensor([c for c in range(256) if c & 0x7F != 0x7F], dtype=torch.uint8, device="cuda")
    w = fin[torch.randint(0, fin.numel(), (rows, n), generator=g, device="cuda")].view(E4M3)
    ws = torch.exp(randn(g, -(-rows // 128), nb)) * 2.0 ** -8
    ws *= torch.sign(randn(g, *ws.shape))
    P = fp8.pack(w, ws)
    for lim in (fin.numel(), 8):
        x = torch.zeros(T, np_, dtype=torch.uint8, device="cuda")
        x[:, :n] = fin[torch.randint(0, lim, (T, n), generator=g, device="cuda")]
        x = x.view(E4M3)
        xs = torch.exp(randn(g, T, nb)) * torch.sign(randn(g, T, nb)) * 2.0 ** -8
        check(fp8.matmul(P, rows, n, x, xs, dtype=dtype), w, ws, x, xs, n)


@every_type
@every_kernel
def test_poisoned(hip, name, dtype):
    """A NaN code, an infinite and a NaN weight scale, a token with a NaN, one with an infinity and one of zeros
    reach their own rows and tokens and no others."""
    T, rows, n = size(name)
    g = gen(T + rows + 1)
    w, s = matrix(g, rows, n)
    w.view(torch.uint8)[7, n - 1] = 0xFF
    w.view(torch.uint8)[130, 0] = 0x7F
    s[2, 1] = float("inf")
    if rows > 600:
        s[4, 0] = float("nan")
    x = randn(g, T, n)
    bad = []
    if T > 2:
        bad = [T // 2, T - 1]
        x[T // 2, 3], x[T - 1, n - 1] = float("nan"), float("-inf")
        x[0] = 0
    codes, scale = fp8.quantize(x)
    Y = fp8.matmul(fp8.pack(w, s), rows, n, codes, scale, dtype=dtype)
    want = torch.ones(T, rows, dtype=torch.bool, device="cuda")
    want[bad] = False
    want[:, 7] = want[:, 130] = False
    want[:, 256:384] = False
    if rows > 600:
        want[:, 512:640] = False
    assert torch.equal(torch.isfinite(Y), want)
    keep_t, keep_r = want.any(1), want.any(0)
    if T > 2:
        assert (Y[0][keep_r] == 0).all()
    check(Y, w, s, codes, scale, n, keep_t, keep_r)


@every_type
@every_kernel
def test_the_rest_of_the_buffer(hip, name, dtype):
    """Rows of the result at odd strides and addresses: what lies between, before and behind them stays."""
    T, rows, n = size(name)
    g = gen(T + rows + 2)
    w, s = matrix(g, rows, n)
    P = fp8.pack(w, s)
    codes, scale = fp8.quantize(randn(g, T, n))
    for offset, more in ((0, 0), (1, 1), (3, 6)):
        ys = rows + more
        buf = torch.full((offset + (T + 2) * ys,), 7.0, dtype=dtype, device="cuda")
        out = buf[offset:offset + T * ys].view(T, ys)[:, :rows]
        assert fp8.matmul(P, rows, n, codes, scale, out=out) is out
        check(out, w, s, codes, scale, n)
        assert (buf[offset:offset + T * ys].view(T, ys)[:, rows:] == 7).all()
        assert (buf[:offset] == 7).all() and (buf[offset + T * ys:] == 7).all()


@every_type
@every_kernel
def test_graph_on_a_side_stream(hip, name, dtype):
    """Captured with the quantiser and replayed on another stream between eager calls on other inputs."""
    T, rows, n = size(name)
    g = gen(T + rows + 3)
    w, s = matrix(g, rows, n)
    P = fp8.pack(w, s)
    x = randn(g, T, n)
    codes, scale = fp8.quantize(x)
    Y = fp8.matmul(P, rows, n, codes, scale, dtype=dtype)
    check(Y, w, s, codes, scale, n)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fp8.quantize(x, codes=codes, scale=scale)
        fp8.matmul(P, rows, n, codes, scale, out=Y)
    side = torch.cuda.Stream()
    for i in range(3):
        x.copy_(randn(g, T, n) * 10.0 ** (i - 1))
        Y.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        want = fp8.matmul(P, rows, n, *fp8.quantize(x), dtype=dtype)
        torch.cuda.synchronize()
        assert torch.equal(Y, want), i


@every_type
def test_all_kernels_at_once(hip, dtype):
    """Each kernel on a stream of its own, several times over, with tensors of its own."""
    g, cases = gen(5), []
    for name in SIZES:
        T, rows, n = size(name)
        w, s = matrix(g, rows, n)
        args = (fp8.pack(w, s), rows, n, *fp8.quantize(randn(g, T, n)))
        cases.append((args, fp8.matmul(*args, dtype=dtype), torch.cuda.Stream()))
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for args, want, stream in cases:
            with torch.cuda.stream(stream):
                got.append((fp8.matmul(*args, dtype=dtype), want))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in got)


def test_offsets_past_32_bits_in_tiles(hip):
    """A matrix and a result of more than 4 GB each through the tiles, 16-bit results among them."""
    g = gen(6)
    rows, n, T = 70001, 65500, 300
    assert fp8.matmul_kernel(rows, n, T).startswith("tile")
    w = torch.randint(0, 120, (rows, n), generator=g, device="cuda", dtype=torch.uint8).view(E4M3)
    s = torch.exp(0.5 * randn(g, -(-rows // 128), -(-n // 128))) * 2.0 ** -20
    P = fp8.pack(w, s)
    assert P.numel() > 1 << 32
    codes, scale = fp8.quantize(randn(g, T, n))
    Y = fp8.matmul(P, rows, n, codes, scale, dtype=torch.bfloat16)
    for r in (0, 34944, 69888):                       # a block of 128 rows from each on
        e = min(r + 128, rows)
        check(Y[:, r:e], w[r:e], s[r // 128:r // 128 + 1], codes, scale, n)
    del w, P, Y
    T, rows, n = 80003, 30003, 128
    assert fp8.matmul_kernel(rows, n, T).startswith("tile")
    w, s = matrix(g, rows, n)
    codes, scale = fp8.quantize(randn(g, T, n))
    Y = fp8.matmul(fp8.pack(w, s), rows, n, codes, scale, dtype=torch.float16)
    assert Y.numel() * 2 > 1 << 32
    for t in (0, 40000, T - 100):
        check(Y[t:t + 100], w, s, codes[t:t + 100], scale[t:t + 100], n)
