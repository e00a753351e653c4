"""A routed MoE block with 8-bit floating-point weights for up to 64 tokens
against its definition in 64 bits.

The tolerance of every element follows the roundings through the block in 64 bits
(u = 2^-24, |.| sums of magnitudes): x within 5 u (mean, eps and square root,
reciprocal, two products); a product of length n within (n + 8 + 5) u of its sum of
magnitudes (n + 2 additions over the three planes and the waves, the scale's fma); silu within
6 u of its value (expf, sum, quotient) and 1.1 times its argument's error; a routing
weight within the scores' error plus 8 u.  A float below 2^-126 may be lost whole (no
relative bound holds there), so every value also carries that much.  Expert ids must be the largest k but
for scores closer than the scores' own error."""
import types

import pytest
import torch

from tests.test_hip_fp8 import gen, matrix, randn, values
from tierlm_amd import fp8

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TINY = 2.0 ** -126


def build(seed, D, de, E, k, ds=0, router=0, scale=1.0, gate=False, mask=None, bias=True, skew=0.0):
    g, c = gen(seed), types.SimpleNamespace(D=D, de=de, E=E, k=k, ds=ds, router=router, scale=scale, mask=mask)
    c.norm = 1 + 0.1 * randn(g, D)
    c.router_w = randn(g, E, D) / D ** 0.5
    if skew:   # every token near one direction that a few experts like
        c.router_w[:4] += skew / D ** 0.5
    c.bias = 0.1 * randn(g, E) if router == 2 and bias else None

    def mat(rows, n):
        w, s = matrix(g, rows, n)
        return w, s / n ** 0.5

    c.experts = [(mat(de, D), mat(de, D), mat(D, de)) for _ in range(E)]
    c.shared = (mat(ds, D), mat(ds, D), mat(D, ds)) if ds else None
    c.gate_inp = randn(g, D) / D ** 0.5 if gate else None
    c.packed = [[fp8.pack(*m) for m in ex] for ex in c.experts]
    c.spacked = [fp8.pack(*m) for m in c.shared] if ds else None
    c.block = fp8.MoeBlock(D=D, de=de, E=E, k=k, ffn_norm=c.norm, router_w=c.router_w,
                           expert_ptrs=[m.data_ptr() for ex in c.packed for m in ex], router=router, routed_scale=scale,
                           eps=1e-6, router_bias=c.bias, ds=ds, shared=c.spacked, shared_gate_inp=c.gate_inp,
                           mask=None if mask is None else mask.to("cuda", torch.uint8))
    return c, g


def ffn(mats, x, dx):
    """(value, error bound) of down (silu(gate x) * up x) for rows x with errors dx."""
    G, Up, Dn = (values(*m) for m in mats)
    n, m = G.shape[1], G.shape[0]

    def product(W, v, dv):
        return v @ W.T, dv @ W.abs().T + (n if W is not Dn else m) * U * (v.abs() @ W.abs().T) + \
            13 * U * (v.abs() @ W.abs().T) + TINY * (1 + W.abs().sum(1))

    g, dg = product(G, x, dx)
    u, du = product(Up, x, dx)
    sg = g * torch.sigmoid(g)
    dsg = 1.1 * dg + 6 * U * sg.abs()
    h = sg * u
    dh = dsg * u.abs() + sg.abs() * du + dsg * du + U * h.abs()
    return product(Dn, h, dh)


def check(c, h, out, ids, w):
    T = h.shape[0]
    h, E, k = h.double(), c.E, c.k
    x = h * torch.rsqrt((h * h).mean(1, keepdim=True) + 1e-6) * c.norm.double()
    dx = 5 * U * x.abs()
    R = c.router_w.double()
    l, dl = x @ R.T, dx @ R.abs().T + U * (x @ R.T).abs()
    dl = dl.max().item()
    off = torch.zeros(E, dtype=torch.bool, device="cuda") if c.mask is None else c.mask.cuda()
    p = torch.sigmoid(l) if c.router == 2 else torch.softmax(l.masked_fill(off, -torch.inf), 1)
    sel = (p + (c.bias.double() if c.bias is not None else 0)) if c.router == 2 else l
    dsel = dl + 8 * U if c.router == 2 else dl
    sel = sel.masked_fill(off, -torch.inf)
    kk = min(k, int((~off).sum()))
    assert (ids[:, kk:] == -1).all() and (w[:, kk:] == 0).all()
    i = ids[:, :kk].long()
    assert ((i >= 0) & (i < E)).all() and not off[i].any()
    best = sel.sort(1, descending=True)[0][:, :kk]
    got = sel.gather(1, i)
    assert ((got - best).abs() <= 2 * dsel).all()
    assert all(len(set(r.tolist())) == kk for r in i)
    wt = p.gather(1, i)
    if c.router != 1:
        wt = wt / (wt.sum(1, keepdim=True) + (1e-20 if c.router == 2 else 0))
    wt = wt * c.scale
    dw = wt * (4 * dl + 8 * U)
    assert ((w[:, :kk].double() - wt).abs() <= dw).all(), ((w[:, :kk].double() - wt).abs() / dw).max()
    want, tol = h.clone(), torch.zeros_like(h)
    size = torch.zeros_like(h)
    for e in i.unique().tolist():
        t, r = torch.where(i == e)
        y, dy = ffn(c.experts[e], x[t], dx[t])
        want.index_add_(0, t, y * wt[t, r, None])
        size.index_add_(0, t, (y * wt[t, r, None]).abs())
        tol.index_add_(0, t, dy * wt[t, r, None] + y.abs() * dw[t, r, None])
    if c.ds:
        s, dsh = ffn(c.shared, x, dx)
        gate = 1.0
        if c.gate_inp is not None:
            a = x @ c.gate_inp.double()
            gate = torch.sigmoid(a)[:, None]
            tol += s.abs() * (gate * 6 * U + (dx @ c.gate_inp.double().abs() + U * a.abs())[:, None])
        want, tol, size = want + gate * s, tol + dsh, size + (gate * s).abs()
    tol += (kk + 3) * U * size + U * want.abs()
    diff = (out.double() - want).abs()
    assert (diff <= tol).all(), (diff / tol).nan_to_num(0).max().item()


def go(c, g, T, spread=0.3):
    h = randn(g, T, c.D) * torch.exp(spread * randn(g, T, 1))
    keep = h.clone()
    out = torch.full_like(h, 7.0)
    ids = torch.full((T, c.k), 99, dtype=torch.int32, device="cuda")
    w = torch.full((T, c.k), 99.0, device="cuda")
    assert c.block(h, out=out, ids=ids, w=w) is out
    assert torch.equal(h, keep)
    check(c, h, out, ids, w)
    return h, out, ids, w


@pytest.mark.parametrize("T", [1, 2, 3, 5, 8, 9, 16, 17, 33, 64])
@pytest.mark.parametrize("shape", [(512, 256, 32, 4, 256), (256, 384, 20, 3, 0)])
def test_block(hip, T, shape):
    c, g = build(T + shape[0], *shape)
    go(c, g, T)


@pytest.mark.parametrize("D,de,E,k,ds,T", [(1, 1, 1, 1, 0, 1), (16, 16, 2, 2, 16, 3), (100, 37, 5, 2, 9, 7),
                                           (1000, 333, 10, 3, 200, 61), (129, 257, 256, 32, 0, 5),
                                           (2048, 768, 16, 8, 0, 1), (2048, 768, 16, 8, 0, 6), (4096, 100, 9, 9, 513, 11),
                                           (640, 1536, 7, 1, 0, 64), (300, 128, 130, 6, 0, 40)])
@pytest.mark.parametrize("router", [0, 1, 2])
def test_block_sizes(hip, D, de, E, k, ds, T, router):
    c, g = build(D + T, D, de, E, k, ds, router=router, scale=2.5 if router == 2 else 1.0, gate=T % 2 == 1 and ds > 0)
    go(c, g, T)


@pytest.mark.parametrize("D,de,E,k,T", [(129, 257, 256, 32, 64), (512, 128, 128, 2, 24), (1024, 256, 128, 4, 10),
                                        (4096, 512, 16, 4, 14), (1000, 300, 8, 4, 4), (2048, 130, 40, 3, 16),
                                        (300, 2000, 64, 8, 12), (7, 3, 1, 1, 64)])
def test_block_launches(hip, D, de, E, k, T):
    """Each way through the launches: routed in gate/up or before it, down per token or per expert, experts with
    as many tokens as there are."""
    c, g = build(D + de + T, D, de, E, k)
    go(c, g, T)


@pytest.mark.parametrize("T", [1, 4, 21, 64])
def test_crowded_experts(hip, T):
    """Every token near one direction: the same few experts for all of them."""
    c, g = build(T, 512, 256, 64, 4, 0, skew=3.0)
    h = 1.0 + 0.2 * randn(g, T, 512)
    out, ids, w = torch.empty_like(h), torch.empty(T, 4, dtype=torch.int32, device="cuda"), torch.empty(T, 4, device="cuda")
    c.block(h, out=out, ids=ids, w=w)
    assert ids.unique().numel() <= 8
    check(c, h, out, ids, w)


@pytest.mark.parametrize("router", [0, 1, 2])
@pytest.mark.parametrize("left", [12, 4, 3, 1, 0])
@pytest.mark.parametrize("T", [1, 9])
def test_masked_experts(hip, router, left, T):
    """Pruned experts are never chosen; with fewer than k left the ranks behind them are empty, with none
    only the shared expert is added."""
    mask = torch.ones(12, dtype=torch.bool)
    mask[torch.randperm(12, generator=torch.Generator().manual_seed(left + 1))[:left]] = False
    c, g = build(left + 50, 256, 128, 12, 4, 128, router=router, mask=mask)
    go(c, g, T)


@pytest.mark.parametrize("router", [0, 1, 2])
def test_equal_scores_take_the_lowest(hip, router):
    c, g = build(3, 256, 64, 40, 5, router=router, bias=False)
    c.router_w[:] = c.router_w[0]
    h, out, ids, w = go(c, g, 6)
    assert (ids.cpu() == torch.arange(5, dtype=torch.int32)).all()


def test_in_place_and_repeats(hip):
    """out == h; a call repeats its bits; a token's result does not change with the tokens beside it in the
    routing it gets."""
    c, g = build(8, 512, 256, 32, 4, 256)
    h, out, ids, w = go(c, g, 23)
    for _ in range(3):
        x = h.clone()
        assert c.block(x) is x and torch.equal(x, out)
    one = c.block(h[5].clone())
    check(c, h[5:6], one[None], ids[5:6], w[5:6])


@pytest.mark.parametrize("T", [1, 7])
def test_poisoned_tokens(hip, T):
    """A token with a NaN gives NaN; the others keep their bits."""
    c, g = build(9, 256, 128, 16, 4, 128)
    h, out, ids, w = go(c, g, T)
    h[T - 1, 3] = float("nan")
    got = c.block(h, out=torch.empty_like(h))
    assert torch.isnan(got[T - 1]).all()
    assert torch.isfinite(got[:T - 1]).all()


def test_small_and_large_tokens(hip):
    """Zero, tiny and huge residuals."""
    c, g = build(10, 256, 128, 16, 4, 128)
    h = randn(g, 5, 256)
    h[0] = 0
    h[1] *= 1e-30
    h[2] *= 1e15
    out, ids, w = torch.empty_like(h), torch.empty(5, 4, dtype=torch.int32, device="cuda"), torch.empty(5, 4, device="cuda")
    c.block(h, out=out, ids=ids, w=w)
    check(c, h, out, ids, w)


def test_graph_and_streams(hip):
    """Captured with quantise and product beside it, replayed between eager calls of another workspace, on
    a side stream."""
    c, g = build(11, 512, 256, 32, 4, 256)
    other = build(11, 512, 256, 32, 4, 256)[0]
    wm, sm = matrix(g, 300, 512)
    P = fp8.pack(wm, sm)
    h = randn(g, 12, 512)
    out, Y = torch.empty_like(h), torch.empty(12, 300, device="cuda")
    codes, scale = fp8.quantize(h)
    c.block(h, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.block(h, out=out)
        fp8.quantize(out, codes=codes, scale=scale)
        fp8.matmul(P, 300, 512, codes, scale, out=Y)
    side = torch.cuda.Stream()
    for i in range(4):
        h.copy_(randn(g, 12, 512))
        want = other.block(h, out=torch.empty_like(h))
        want_y = fp8.matmul(P, 300, 512, *fp8.quantize(want))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        side.synchronize()
        assert torch.equal(out, want) and torch.equal(Y, want_y), i


def test_block_refuses(hip):
    c, g = build(12, 256, 128, 16, 4)
    for bad in (torch.zeros(2, 255, device="cuda"), torch.zeros(2, 256, device="cuda", dtype=torch.float16),
                torch.zeros(2, 256), torch.zeros(2, 512, device="cuda")[:, :256]):
        with pytest.raises(ValueError):
            c.block(bad)
    h = torch.zeros(2, 256, device="cuda")
    with pytest.raises(ValueError):
        c.block(h, out=torch.zeros(3, 256, device="cuda"))
    with pytest.raises(ValueError):
        c.block(h, ids=torch.zeros(2, 4, device="cuda"))
    from tierlm_amd._lib import HipError
    with pytest.raises(HipError):
        c.block(torch.zeros(65, 256, device="cuda"))
    with pytest.raises(ValueError):
        fp8.MoeBlock(D=256, de=128, E=2, k=1, ffn_norm=c.norm, router_w=c.router_w[:2].contiguous(), expert_ptrs=[1, 2, 3])
    with pytest.raises(HipError):
        fp8.MoeBlock(D=256, de=128, E=2, k=3, ffn_norm=c.norm, router_w=c.router_w[:2].contiguous(),
                     expert_ptrs=[m.data_ptr() for ex in c.packed[:2] for m in ex])


def test_workspace_grows_under_a_graph(hip):
    """A graph captured with few tokens still replays after the block has grown for more."""
    c, g = build(13, 256, 128, 16, 4)
    h = randn(g, 3, 256)
    out = torch.empty_like(h)
    c.block(h, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.block(h, out=out)
    many = randn(g, 64, 256)
    c.block(many, out=torch.empty_like(many))
    for i in range(3):
        h.copy_(randn(g, 3, 256))
        graph.replay()
        got = out.clone()
        assert torch.equal(got, c.block(h, out=torch.empty_like(h))), i
        torch.cuda.synchronize()


def test_overlapping_out_is_refused(hip):
    c, g = build(14, 256, 128, 16, 4)
    buf = randn(g, 3, 256)
    with pytest.raises(ValueError):
        c.block(buf[:2], out=buf[1:])


def test_one_matrix_for_two_experts(hip):
    """Expert pointers may repeat."""
    c, g = build(15, 256, 128, 8, 3)
    c.experts[5], c.packed[5] = c.experts[2], c.packed[2]
    c.block = fp8.MoeBlock(D=256, de=128, E=8, k=3, ffn_norm=c.norm, router_w=c.router_w,
                           expert_ptrs=[m.data_ptr() for ex in c.packed for m in ex])
    for T in (1, 30):
        go(c, g, T)


def test_pruned_experts_need_no_matrices(hip):
    mask = torch.zeros(16, dtype=torch.bool)
    mask[[0, 3, 7, 15]] = True
    c, g = build(16, 256, 128, 16, 4, mask=mask)
    ptrs = [0 if mask[e] else m.data_ptr() for e, ex in enumerate(c.packed) for m in ex]
    c.block = fp8.MoeBlock(D=256, de=128, E=16, k=4, ffn_norm=c.norm, router_w=c.router_w, expert_ptrs=ptrs,
                           mask=mask.to("cuda", torch.uint8))
    for T in (1, 3, 40):
        go(c, g, T)


def test_wide_model(hip):
    """The longest residual: rows past what the router keeps in registers."""
    for D, T in ((5000, 3), (16384, 2)):
        c, g = build(D, D, 64, 6, 2, 48, gate=True)
        go(c, g, T)
