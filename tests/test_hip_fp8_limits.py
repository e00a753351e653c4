"""The 8-bit calls at the ends of their sizes, with nothing to do, side by side and in graphs that share a block."""
import pytest
import torch

from tests.test_hip_fp8 import E4M3, check_product, gen, matrix, randn
from tests.test_hip_fp8_moe import build, check
from tierlm_amd import fp8

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [1, 20, 64])
def test_most_rows(hip, T):
    """2^25 rows: the first, middle and last of them."""
    g = gen(T)
    rows, n = 1 << 25, 5
    w = torch.randint(0, 120, (rows, n), generator=g, device="cuda", dtype=torch.uint8).view(E4M3)
    s = torch.exp(0.5 * randn(g, rows // 128, 1)) * 0.01
    codes, scale = fp8.quantize(randn(g, T, n))
    Y = fp8.matmul(fp8.pack(w, s), rows, n, codes, scale)
    for r in (0, 1 << 24, rows - 256):
        check_product(Y[:, r:r + 256], w[r:r + 256], s[r // 128:r // 128 + 2], codes, scale, n)
    del Y


@pytest.mark.parametrize("T", [1, 3, 40, 300])
def test_longest_rows(hip, T):
    """2^22 values a row, quantised and multiplied."""
    g = gen(T + 1)
    rows, n = 20, 1 << 22
    w, s = matrix(g, rows, n)
    codes, scale = fp8.quantize(randn(g, T, n).to(torch.bfloat16))
    Y = fp8.matmul(fp8.pack(w, s), rows, n, codes, scale)
    for t in range(0, T, 50):
        check_product(Y[t:t + 50], w, s, codes[t:t + 50], scale[t:t + 50], n)


@pytest.mark.parametrize("T", [1, 3, 64])
def test_widest_block(hip, T):
    """16384 x 65536 of one expert."""
    c, g = build(T, 16384, 65536, 1, 1)
    h = randn(g, T, 16384)
    ids, w = torch.empty(T, 1, dtype=torch.int32, device="cuda"), torch.empty(T, 1, device="cuda")
    out = c.block(h, out=torch.empty_like(h), ids=ids, w=w)
    check(c, h, out, ids, w)


def test_no_tokens(hip):
    c, g = build(2, 256, 128, 16, 4)
    h = torch.empty(0, 256, device="cuda")
    ids, w = torch.empty(0, 4, dtype=torch.int32, device="cuda"), torch.empty(0, 4, device="cuda")
    assert c.block(h) is h and c.block(h, out=torch.empty_like(h), ids=ids, w=w).shape == (0, 256)
    assert c.block(randn(g, 1, 256)).shape == (1, 256)
    P = fp8.pack(*matrix(g, 20, 300))
    assert fp8.matmul(P, 20, 300, *fp8.quantize(torch.empty(0, 300, device="cuda")), dtype=torch.float16).shape == (0, 20)


def test_two_blocks_of_the_same_matrices_at_once(hip):
    """Blocks own their workspaces: the same experts on two streams."""
    c, g = build(3, 512, 256, 32, 4, 256)
    other = fp8.MoeBlock(D=512, de=256, E=32, k=4, ffn_norm=c.norm, router_w=c.router_w,
                         expert_ptrs=[m.data_ptr() for ex in c.packed for m in ex], ds=256, shared=c.spacked)
    hs = [randn(g, T, 512) for T in (1, 5, 23, 64)]
    want = [c.block(h, out=torch.empty_like(h)) for h in hs]
    other.reserve(64)
    outs = [[torch.empty_like(h) for h in hs] for _ in range(10)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for i, row in enumerate(outs):
        for h, out in zip(hs, row):
            with torch.cuda.stream(streams[i % 2]):
                (c.block, other)[i % 2](h, out=out)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for row in outs for a, b in zip(row, want))


def test_two_graphs_of_one_block_in_turn(hip):
    """Captured without a call before (the workspace is made during the capture), with different numbers of tokens,
    replayed one after the other between eager calls."""
    c, g = build(4, 512, 256, 32, 4, 256)
    ref = build(4, 512, 256, 32, 4, 256)[0]
    hs = [randn(g, T, 512) for T in (2, 40)]
    outs, graphs = [torch.empty_like(h) for h in hs], []
    ref.block(hs[0], out=outs[0]), ref.block(hs[1], out=outs[1])
    torch.cuda.synchronize()
    for h, out in zip(hs, outs):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            c.block(h, out=out)
    for i in range(4):
        for h, out, graph in zip(hs, outs, graphs):
            h.copy_(randn(g, *h.shape))
            graph.replay()
            many = randn(g, 64, 512)
            got = c.block(many, out=torch.empty_like(many))
            assert torch.equal(got, ref.block(many, out=torch.empty_like(many)))
            assert torch.equal(out, ref.block(h, out=torch.empty_like(h))), i
            torch.cuda.synchronize()
