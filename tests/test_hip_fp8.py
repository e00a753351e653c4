"""8-bit floating point on the device against the definitions in 64 bits: packing,
the activation quantiser (bit for bit) and the product.

Tolerance of a product, counted from its roundings: a block's 128 products are
exact, their sum takes 127 additions, the chain one fma per block and one
product of the two scales, so an f32 result is off by at most
(127 + nb + 2) 2^-24 S with S the sum of the magnitudes.  A 16-bit output adds half a
step of its type, and its sums may come from the 8-bit matrix instructions, which align
every 8 products to the largest of them and cut what lies below 2^-13 of that one's
power of two: at most 7 products lose less than 2^-13 max each, 7 * 2^-13 S in all."""
import numpy as np
import pytest
import torch

from tierlm_amd import fp8

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def matrix(g, rows, n, spread=0.5):
    w = (randn(g, rows, n) * 100).clamp(-448, 448).to(E4M3)
    s = torch.exp(spread * randn(g, -(-rows // 128), -(-n // 128))) * 0.01
    return w, s


def values(w, s):
    rows, n = w.shape
    return w.double() * s.double().repeat_interleave(128, 0)[:rows].repeat_interleave(128, 1)[:, :n]


def ref_quantize(x):
    """numpy, 64 bits: (code values [T, np], scales [T, nb])"""
    x = x.detach().cpu().to(torch.float64).numpy()
    T, n = x.shape
    nb = -(-n // 128)
    v = np.zeros((T, nb * 128))
    v[:, :n] = x
    v = v.reshape(T, nb, 128)
    bad = ~np.isfinite(v).all(-1)
    amax = np.where(bad, 1.0, np.abs(np.where(np.isfinite(v), v, 0)).max(-1))
    m, e = np.frexp(amax)
    e = np.maximum(np.where(m > 0.875, e - 8, e - 9), -126)
    y = np.where(bad[..., None], 0.0, v / np.ldexp(1.0, e)[..., None])
    step = np.ldexp(1.0, np.maximum(np.frexp(np.abs(y))[1] - 1, -6) - 3)
    codes = np.rint(y / step) * step
    scale = np.where(bad, np.nan, np.where(amax > 0, np.ldexp(1.0, e), 0.0))
    return codes.reshape(T, nb * 128), scale


def check_product(Y, w, s, codes, scale, n):
    W = values(w, s)
    X = (codes.double() * scale.double().repeat_interleave(128, 1))[:, :n]
    want, size = X @ W.T, X.abs() @ W.abs().T
    nb = -(-n // 128)
    tol = (127 + nb + 2) * 2.0 ** -24 * size + HALF_STEP[Y.dtype] * want.abs() * (Y.dtype != torch.float32)
    tol += 7 * 2.0 ** -13 * size * (Y.dtype != torch.float32)
    tol += 2.0 ** -25 * (Y.dtype == torch.float16)       # half a step of a subnormal binary16
    off = ((Y.double() - want).abs() - tol).max().item()
    assert off <= 0, (off, ((Y.double() - want).abs() / tol).max().item())


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,n", [(1, 1), (1, 2048), (3, 127), (5, 128), (7, 129), (33, 1111), (130, 640), (2, 16384)])
def test_quantize(hip, dtype, T, n):
    g = gen(T * 1000 + n)
    x = (randn(g, T, n) * torch.exp(3 * randn(g, T, 1))).clamp(-6e4, 6e4).to(dtype)
    codes, scale = fp8.quantize(x)
    torch.cuda.synchronize()
    want_c, want_s = ref_quantize(x)
    assert np.array_equal(codes.float().cpu().numpy(), want_c.astype(np.float32))
    assert np.array_equal(scale.cpu().numpy(), want_s.astype(np.float32))


def test_quantize_edges(hip):
    """Largest magnitudes around 448 times a power of two, ties between codes, subnormal codes, zero blocks,
    the smallest scale, infinities and NaN, signed zeros."""
    x = torch.zeros(12, 256)
    x[0, :4] = torch.tensor([448.0, 447.99997, 1.0625, -1.0625])          # 1.0625: between codes 1 and 1.125
    x[1, :3] = torch.tensor([448.00003, 9.0, -3.1875])                     # the next power
    x[2, :4] = torch.tensor([256.0, 2.0 ** -9, 2.0 ** -10, 3 * 2.0 ** -10])   # subnormal codes and their ties
    x[3, 0], x[3, 130] = 1e-38, 3.4e38                                      # both ends of the scales
    x[4, 5], x[5, 200] = float("nan"), float("inf")
    x[6, 0], x[6, 1] = -0.0, -float("inf")
    x[7, 0] = 1e-45                                                        # a subnormal float
    x[8] = torch.linspace(-448, 448, 256)
    x[9] = torch.arange(256) * 2.0 ** -10
    x[10, :2] = torch.tensor([3.4028235e38, -3.4028235e38])
    x[11, :128] = -1.75
    codes, scale = fp8.quantize(x.cuda())
    torch.cuda.synchronize()
    want_c, want_s = ref_quantize(x)
    assert np.array_equal(codes.float().cpu().numpy(), want_c.astype(np.float32))
    assert np.array_equal(scale.cpu().numpy(), want_s.astype(np.float32), equal_nan=True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("offset,stride", [(0, 300), (1, 301), (3, 1000), (8, 304)])
def test_quantize_strides(hip, dtype, offset, stride):
    g = gen(offset * 7 + stride)
    buf = randn(g, 9 * stride + 16).to(dtype)
    x = buf[offset:offset + 9 * stride].view(9, stride)[:, :300]
    guard = torch.full((9 * 384 + 64,), 77, dtype=torch.uint8, device="cuda")
    codes, scale = fp8.quantize(x, codes=guard[:9 * 384].view(E4M3).view(9, 384))
    torch.cuda.synchronize()
    want_c, want_s = ref_quantize(x)
    assert np.array_equal(codes.float().cpu().numpy(), want_c.astype(np.float32))
    assert np.array_equal(scale.cpu().numpy(), want_s.astype(np.float32))
    assert (guard[9 * 384:] == 77).all()


@pytest.mark.parametrize("rows,n,stride,offset", [(16, 128, 128, 0), (1, 1, 1, 0), (37, 300, 300, 0), (37, 300, 304, 0),
                                                  (130, 257, 259, 3), (16, 16, 32, 16)])
def test_pack_keeps_every_code(hip, rows, n, stride, offset):
    """The packed bytes by the layout's definition, odd strides and addresses of the rows, zeros in the padding."""
    g = gen(rows + n)
    buf = torch.randint(0, 256, (rows * stride + offset + 16,), generator=g, device="cuda", dtype=torch.uint8)
    W = buf[offset:offset + rows * stride].view(rows, stride)[:, :n]
    nb, rb, nt = -(-n // 128), -(-rows // 128), -(-rows // 16)
    s = randn(g, rb, nb + 3)[:, :nb]
    P = fp8.pack(W, s).cpu().numpy()
    full = np.zeros((nt * 16, nb * 128), np.uint8)
    full[:rows, :n] = W.cpu().numpy()
    # row tile, block, half, 16-value group, row of the tile, value
    u = full.reshape(nt, 16, nb, 2, 4, 16).transpose(0, 2, 3, 4, 1, 5)
    assert np.array_equal(P[:u.size], np.ascontiguousarray(u).reshape(-1))
    assert np.array_equal(P[u.size:u.size + rb * nb * 4].view(np.float32).reshape(rb, nb), s.cpu().numpy())


SHAPES = [(1, 1, 1), (1, 16, 128), (1, 512, 512), (1, 4096, 2048), (1, 1000, 1111), (2, 130, 257), (5, 257, 640),
          (15, 33, 1024), (16, 512, 2048), (17, 128, 384), (31, 1000, 100), (33, 300, 1500), (64, 768, 2048),
          (65, 520, 129), (77, 1000, 1111), (127, 129, 256), (128, 256, 512), (129, 257, 640), (255, 400, 1000),
          (300, 1024, 2048), (513, 272, 768), (1000, 777, 333), (2048, 512, 256)]


@pytest.mark.parametrize("T,rows,n", SHAPES)
def test_matmul(hip, T, rows, n):
    g = gen(T * 31 + rows + n)
    w, s = matrix(g, rows, n)
    codes, scale = fp8.quantize(randn(g, T, n) * torch.exp(randn(g, T, 1)))
    for dtype in (torch.float32, torch.bfloat16):
        check_product(fp8.matmul(fp8.pack(w, s), rows, n, codes, scale, dtype=dtype), w, s, codes, scale, n)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,rows,n,ys", [(3, 40, 200, 41), (20, 100, 256, 104), (70, 250, 384, 251),
                                         (300, 250, 384, 252), (300, 256, 128, 300)])
def test_matmul_leaves_the_rest_of_y(hip, dtype, T, rows, n, ys):
    """Row strides of Y, aligned for wide stores or not: what lies between and behind the rows stays."""
    g = gen(T + rows + ys)
    w, s = matrix(g, rows, n)
    codes, scale = fp8.quantize(randn(g, T, n))
    for offset in (0, 1):
        buf = torch.full((offset + (T + 3) * ys,), 7.0, dtype=dtype, device="cuda")
        out = buf[offset:offset + T * ys].view(T, ys)[:, :rows]
        fp8.matmul(fp8.pack(w, s), rows, n, codes, scale, out=out)
        check_product(out, w, s, codes, scale, n)
        assert (buf[offset:offset + T * ys].view(T, ys)[:, rows:] == 7).all()
        assert (buf[:offset] == 7).all() and (buf[offset + T * ys:] == 7).all()


@pytest.mark.parametrize("T", [1, 16, 70, 300])
def test_matmul_every_code(hip, T):
    """Every finite code as weight and activation, subnormal ones among them, against exact sums."""
    g = gen(T)
    rows, n = 300, 512
    fin = torch.tensor([c for c in range(256) if c & 0x7F != 0x7F], dtype=torch.uint8, device="cuda")
    w = fin[torch.randint(0, fin.numel(), (rows, n), generator=g, device="cuda")].view(E4M3)
    x = fin[torch.randint(0, fin.numel(), (T, n), generator=g, device="cuda")].view(E4M3)
    small = torch.randint(0, 8, (T, n), generator=g, device="cuda", dtype=torch.uint8).view(E4M3)   # subnormal alone
    ws = torch.exp(randn(g, 3, 4))
    for c in (x, small):
        xs = torch.exp(randn(g, T, 4)) * torch.sign(randn(g, T, 4))
        check_product(fp8.matmul(fp8.pack(w, ws), rows, n, c, xs), w, ws, c, xs, n)


@pytest.mark.parametrize("T", [1, 16, 70, 300])
def test_matmul_poisoned(hip, T):
    """NaN codes and scales reach their rows and tokens and no others."""
    g = gen(T + 5)
    rows, n = 300, 400
    w, s = matrix(g, rows, n)
    w.view(torch.uint8)[7, 399] = 0x7F
    s[2, 1] = float("inf")
    x = randn(g, T, n)
    x[T - 1, 3] = float("inf")
    codes, scale = fp8.quantize(x)
    assert torch.isnan(scale[T - 1, 0])
    Y = fp8.matmul(fp8.pack(w, s), rows, n, codes, scale)
    ok = torch.isfinite(Y)
    want = torch.ones(T, rows, dtype=torch.bool, device="cuda")
    want[T - 1], want[:, 7], want[:, 256:] = False, False, False
    assert torch.equal(ok, want)
    keep = [r for r in range(256) if r != 7]
    if T > 1:
        W = values(w, s)[keep]
        X = (codes[:T - 1].double() * scale[:T - 1].double().repeat_interleave(128, 1))[:, :n]
        tol = (127 + 4 + 2) * 2.0 ** -24 * (X.abs() @ W.abs().T)
        assert ((Y[:T - 1][:, keep].double() - X @ W.T).abs() <= tol).all()


def test_empty_calls(hip):
    x = torch.empty(0, 200, device="cuda")
    codes, scale = fp8.quantize(x)
    assert codes.shape == (0, 256) and scale.shape == (0, 2)
    g = gen(1)
    w, s = matrix(g, 20, 200)
    assert fp8.matmul(fp8.pack(w, s), 20, 200, codes, scale).shape == (0, 20)


@pytest.mark.parametrize("T", [1, 40, 300])
def test_linear_streams_and_graph(hip, T):
    """Quantise and product together on a side stream, and captured: every replay gives the eager bits
    for the inputs then in place."""
    g = gen(T + 9)
    rows, n = 500, 700
    w, s = matrix(g, rows, n)
    P = fp8.pack(w, s)
    x = randn(g, T, n)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        Y = fp8.matmul(P, rows, n, *fp8.quantize(x))
    side.synchronize()
    want = fp8.matmul(P, rows, n, *fp8.quantize(x))
    assert torch.equal(Y, want)
    codes, scale = fp8.quantize(x)
    check_product(want, w, s, codes, scale, n)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fp8.quantize(x, codes=codes, scale=scale)
        fp8.matmul(P, rows, n, codes, scale, out=Y)
    for i in range(4):
        x.copy_(randn(g, T, n) * 10.0 ** (i - 2))
        graph.replay()
        got = Y.clone()
        assert torch.equal(got, fp8.matmul(P, rows, n, *fp8.quantize(x))), i
        torch.cuda.synchronize()


# (T, rows) of large products, whose tiles stream through LDS
TILES = [(100, 5000), (100, 8100), (100, 16300), (250, 16300), (250, 32700), (250, 65300), (33, 66000)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n", [100, 256, 300, 512, 900])
@pytest.mark.parametrize("T,rows", TILES)
def test_matmul_tiles(hip, T, rows, n, dtype):
    """Part tiles of rows and tokens and one to eight blocks of values (the stages' whole and part rounds), the
    tokens' scales spread over powers of two."""
    g = gen(T + rows + n)
    w, s = matrix(g, rows, n)
    codes, scale = fp8.quantize(randn(g, T, n) * torch.exp2(torch.randint(-6, 7, (T, 1), generator=g, device="cuda")))
    scale *= 1 + torch.rand(scale.shape, generator=g, device="cuda")      # not powers of two alone
    check_product(fp8.matmul(fp8.pack(w, s), rows, n, codes, scale, dtype=dtype), w, s, codes, scale, n)


# (T, rows, n), one at least for each kernel that the product chooses from (the float results' and the 16-bit
# ones' differ): few groups and many, short rows and long; then few rows of very many tokens
GROUPS = [(17, 21, 302), (18, 2101, 308), (17, 4336, 356), (17, 4232, 582), (17, 25365, 303), (18, 8960, 533),
          (36, 14529, 1677), (34, 12974, 322), (17, 52136, 541), (34, 16717, 2094), (67, 49172, 338), (33, 8290, 626),
          (33, 18207, 570), (66, 23694, 324), (66, 16901, 1590), (131, 35900, 565), (16, 9000, 2100),
          (100, 8200, 4196), (100, 4100, 1100), (30, 16500, 1100), (100, 6500, 1100), (100, 4100, 700),
          (30, 25000, 300), (100, 2100, 1100), (25, 9000, 1100), (100, 3200, 1100), (30, 4200, 700),
          (30, 4200, 1100), (16, 16500, 1100), (5, 32800, 1100), (9, 8200, 130), (5, 100, 9000), (16, 40, 700),
          (5000, 10, 300), (40000, 64, 256), (70000, 16, 130), (70000, 70, 130)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,rows,n", GROUPS)
def test_matmul_row_groups(hip, T, rows, n, dtype):
    g = gen(T + rows + n)
    w, s = matrix(g, rows, n)
    codes, scale = fp8.quantize(randn(g, T, n) * torch.exp2(torch.randint(-6, 7, (T, 1), generator=g, device="cuda")))
    scale *= 1 + torch.rand(scale.shape, generator=g, device="cuda")
    check_product(fp8.matmul(fp8.pack(w, s), rows, n, codes, scale, dtype=dtype), w, s, codes, scale, n)


@pytest.mark.parametrize("T,rows,n", [(1, 64, 20000), (16, 100, 9000), (20, 64, 8192), (40, 64, 16384), (300, 5000, 2000)])
def test_matmul_long_rows(hip, T, rows, n):
    g = gen(T + n)
    w, s = matrix(g, rows, n)
    codes, scale = fp8.quantize(randn(g, T, n))
    for dtype in (torch.float32, torch.bfloat16):
        check_product(fp8.matmul(fp8.pack(w, s), rows, n, codes, scale, dtype=dtype), w, s, codes, scale, n)


def test_repeats_its_bits(hip):
    g = gen(77)
    w, s = matrix(g, 3000, 1000)
    P = fp8.pack(w, s)
    for T in (1, 20, 64, 200, 1000):
        codes, scale = fp8.quantize(randn(g, T, 1000))
        for dtype in (torch.float32, torch.float16):
            a = fp8.matmul(P, 3000, 1000, codes, scale, dtype=dtype)
            for _ in range(3):
                assert torch.equal(a, fp8.matmul(P, 3000, 1000, codes, scale, dtype=dtype))


def test_two_calls_at_once(hip):
    """Products on two streams at a time, each with tensors of its own."""
    g = gen(78)
    w, s = matrix(g, 4096, 2048)
    P = fp8.pack(w, s)
    xs = [fp8.quantize(randn(g, T, 2048)) for T in (5, 300)]
    want = [fp8.matmul(P, 4096, 2048, *x) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = [[], []]
    for _ in range(5):
        for i, (x, st) in enumerate(zip(xs, streams)):
            with torch.cuda.stream(st):
                got[i].append(fp8.matmul(P, 4096, 2048, *x))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(v, want[i]) for v in got[i])


def test_offsets_past_32_bits(hip):
    """A matrix, a result and activations of more than 4 GB each: their first, middle and last parts."""
    g = gen(80)
    rows, n = 70001, 65500
    w = torch.randint(0, 120, (rows, n), generator=g, device="cuda", dtype=torch.uint8).view(E4M3)
    s = torch.exp(0.5 * randn(g, -(-rows // 128), -(-n // 128))) * 0.01
    P = fp8.pack(w, s)
    assert P.numel() > 1 << 32
    for T in (1, 20, 300):
        codes, scale = fp8.quantize(randn(g, T, n))
        Y = fp8.matmul(P, rows, n, codes, scale)
        for r in (0, 34944, 69888):                       # a block of 128 rows from each on
            e = min(r + 128, rows)
            check_product(Y[:, r:e], w[r:e], s[r // 128:r // 128 + 1], codes, scale, n)
    del w, P, Y
    T, rows, n = 40001, 30003, 128
    w, s = matrix(g, rows, n)
    codes, scale = fp8.quantize(randn(g, T, n))
    Y = fp8.matmul(fp8.pack(w, s), rows, n, codes, scale)
    assert Y.numel() * 4 > 1 << 32
    for t in (0, 20000, T - 100):
        check_product(Y[t:t + 100], w, s, codes[t:t + 100], scale[t:t + 100], n)
    del Y
    T, n = 33001, 65536
    x = torch.randn(T, n, generator=g, device="cuda", dtype=torch.bfloat16)
    codes, scale = fp8.quantize(x)
    for t in (0, 16500, T - 3):
        want, ws = ref_quantize(x[t:t + 3].float())
        assert np.array_equal(codes[t:t + 3].double().cpu().numpy(), want)
        assert np.array_equal(scale[t:t + 3].cpu().numpy(), ws.astype(np.float32))


def test_most_tokens(hip):
    """2^20 tokens of a few rows: the second axis of a launch has to hold them."""
    g = gen(81)
    T, n = 1 << 20, 130
    codes, scale = fp8.quantize(randn(g, T, n))
    for rows in (16, 1):
        w, s = matrix(g, rows, n)
        Y = fp8.matmul(fp8.pack(w, s), rows, n, codes, scale)
        check_product(Y, w, s, codes, scale, n)
