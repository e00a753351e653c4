"""A layer's attention half as a served batch runs it, operator after operator: residual norm to codes, the q | k | v
product, append, attention, quantise, the output product, the next norm; then the MoE block.  Prompts in one call and the same
tokens one at a time must agree, and each step with the definition in 64 bits on the operands that it was given."""
import math

import pytest
import torch

from tests.kv_ref import HALF_STEP, close, reference
from tierlm_amd import fp8, kv

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def matrix(g, rows, n):
    w = (torch.randn(rows, n, generator=g, device="cuda") * 100).clamp(-448, 448).to(E4M3)
    s = torch.full((-(-rows // 128), -(-n // 128)), 0.01 / math.sqrt(n), device="cuda")
    return fp8.pack(w, s)


class Layer:
    """Hidden 256, 8 query heads on 2 of 64, 8 experts of width 128."""
    D, H, KV, hd, E, de, k = 256, 8, 2, 64, 8, 128, 2

    def __init__(self, pages, page=16):
        g = gen(1)
        self.norm, self.norm2 = (1 + 0.1 * torch.randn(self.D, generator=g, device="cuda") for _ in range(2))
        self.qn, self.kn = (1 + 0.1 * torch.randn(self.hd, generator=g, device="cuda") for _ in range(2))
        self.rows = (self.H + 2 * self.KV) * self.hd
        self.wqkv, self.wo = matrix(g, self.rows, self.D), matrix(g, self.D, self.H * self.hd)
        self.freq = kv.rope_frequencies(self.hd, 1e6)
        self.cache = kv.Cache(pages, self.KV, self.hd, page=page, dtype=torch.bfloat16)
        self.mats = [matrix(g, *rn) for _ in range(self.E) for rn in ((self.de, self.D), (self.de, self.D), (self.D, self.de))]
        self.moe = fp8.MoeBlock(D=self.D, de=self.de, E=self.E, k=self.k, ffn_norm=self.norm2,
                                router_w=torch.randn(self.E, self.D, generator=g, device="cuda") / 16,
                                expert_ptrs=[m.data_ptr() for m in self.mats])

    def attention(self, h, x, tables, lens, cu=None):
        """h += x, then the attention's output (f32 [T, D]) on h; q and the attention in between."""
        T = h.shape[0]
        qkv = fp8.matmul(self.wqkv, self.rows, self.D, *fp8.add_rmsnorm(h, x, self.norm))
        q = kv.append(self.cache, qkv, self.H, tables, lens, cu, q_norm=self.qn, k_norm=self.kn, inv_freq=self.freq)
        y = (kv.decode(q, self.cache, tables, lens) if cu is None else kv.prompt(q, self.cache, tables, lens, cu))
        return fp8.matmul(self.wo, self.D, self.H * self.hd, *fp8.quantize(y.view(T, -1))), q, y


def tables_of(lens, page, seed):
    need = [-(-n // page) for n in lens]
    perm = torch.randperm(sum(need), generator=torch.Generator().manual_seed(seed)).tolist()
    t = torch.full((len(lens), max(need)), -1, dtype=torch.int32)
    for b, m in enumerate(need):
        for j in range(m):
            t[b, j] = perm.pop()
    return t.cuda(), sum(need)


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def check(layer, q, y, tables, lens, new, first_row=0):
    """The attention of these rows against the cache's present content."""
    at = first_row
    for b, (n, m) in enumerate(zip(new, lens)):
        ids = tables[b, :-(-m // layer.cache.page)].tolist() if m else []
        k, v = layer.cache.keys(ids)[:, :m].transpose(0, 1), layer.cache.values(ids)[:, :m].transpose(0, 1)
        want, tol = reference(q[at:at + n], k, v, 1 / math.sqrt(layer.hd), m - n)
        close(y[at:at + n], want, tol)
        at += n


def test_prompts_and_steps(hip):
    """Three prompts packed, then six steps of all three with a padded slot; against the same tokens step by step from
    the start in another cache."""
    new, steps, page = [5, 33, 18], 6, 16
    tables, pages = tables_of([n + steps for n in new] + [16], page, 2)
    g = gen(3)
    tokens = [torch.randn(n + steps, Layer.D, generator=g, device="cuda") for n in new]
    a, b = Layer(pages), Layer(pages)
    # packed prompts
    h = torch.cat([t[:n] for t, n in zip(tokens, new)])
    x = torch.zeros_like(h)
    cu, lens = ints(0, 5, 38, 56), ints(*new)
    out, q, y = a.attention(h, x, tables[:3], lens, cu)
    check(a, q, y, tables, new, new)
    prompt_out = [out[i:j] for i, j in ((0, 5), (5, 38), (38, 56))]
    # one token of each a step, the fourth slot empty
    zero = torch.zeros(1, Layer.D, device="cuda")
    for p in range(max(new) + steps):
        lens_list = [p + 1 if p < n + steps else 0 for n in new] + [0]
        h = torch.cat([t[p:p + 1] if p < t.shape[0] else zero for t in tokens] + [zero])
        out, q, y = b.attention(h, None, tables, ints(*lens_list))
        assert (y[3] == 0).all() and (out[3] == 0).all()
        check(b, q, y, tables, lens_list, [1 if m else 0 for m in lens_list]) if all(lens_list[:3]) else None
        for i, n in enumerate(new):
            if p < n:
                # the same inputs but for the order of sums: the product's results to f32 rounding, q and k to their type's half
                # step, which the output product's quantiser may turn into a code's half step (2^-4) of a value
                want, got = prompt_out[i][p].double(), out[i].double()
                assert (got - want).norm() <= 2.0 ** -4 * want.norm(), (p, i)
    # the packed cache goes on from where the prompts ended
    for s in range(steps):
        lens_list = [n + s + 1 for n in new] + [0]
        h = torch.cat([t[n + s:n + s + 1] for t, n in zip(tokens, new)] + [zero])
        out, q, y = a.attention(h, None, tables, ints(*lens_list))
        check(a, q[:3], y[:3], tables[:3], lens_list[:3], [1, 1, 1])
        for i, n in enumerate(new):
            ids = tables[i, :-(-(n + steps) // page)].tolist()
            ka, kb = a.cache.keys(ids)[:, :n + s + 1].double(), b.cache.keys(ids)[:, :n + s + 1].double()
            assert ((ka - kb).abs() <= 2.0 ** -7 * kb.abs() + 2.0 ** -7).all()


def test_whole_layer_in_a_graph(hip):
    """A step of the whole layer for four slots, captured once: lengths advance on the device, every replay equals the
    eager step."""
    page, lens0 = 16, [7, 30, 0, 16]
    tables, pages = tables_of([n + 8 for n in lens0], page, 4)
    layer, twin = Layer(pages), Layer(pages)
    for c in (layer, twin):
        c.cache.k.zero_()
        c.cache.v.zero_()
    h, x = torch.zeros(4, Layer.D, device="cuda"), torch.zeros(4, Layer.D, device="cuda")
    lens, on = ints(*lens0), ints(1, 1, 0, 1)

    def step(layer, h, x, lens):
        lens.add_(on)
        out, _, _ = layer.attention(h, x, tables, lens)
        return layer.moe(h + out)

    h2, x2, lens2 = h.clone(), x.clone(), lens.clone()
    step(layer, h, x, lens)
    lens.copy_(lens2)
    layer.cache.k.zero_()
    layer.cache.v.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        result = step(layer, h, x, lens)
    g = gen(5)
    for i in range(5):
        hs, xs = (torch.randn(4, Layer.D, generator=g, device="cuda") for _ in range(2))
        for dst in (h, h2):
            dst.copy_(hs)
        for dst in (x, x2):
            dst.copy_(xs)
        graph.replay()
        want = step(twin, h2, x2, lens2)
        torch.cuda.synchronize()
        assert torch.equal(lens, lens2) and lens.tolist() == [n + (i + 1) * o for n, o in zip(lens0, (1, 1, 0, 1))]
        assert torch.equal(result, want) and torch.equal(h, h2)
        assert torch.equal(layer.cache.k, twin.cache.k) and torch.equal(layer.cache.v, twin.cache.v)
