"""Attention over a paged cache by its definition in 64 bits, and batches to try it on (helpers of the kv tests)."""
import math

import torch

from tierlm_amd import kv

HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


class Batch:
    """Sequences of new[b] rows and lens[b] positions with pages dealt at random; the cache's content random
    everywhere, NaN where no sequence has a position."""

    def __init__(self, dtype, heads, kv_heads, hd, page, new, lens, seed=0, spare=1, width=None, last=False):
        g = gen(seed)
        self.heads, self.new, self.lens_list = heads, list(new), list(lens)
        B = len(lens)
        need = [max(0, -(-n // page)) for n in lens]
        n_pages = sum(need) + spare
        self.cache = kv.Cache(n_pages, kv_heads, hd, page=page, dtype=dtype)
        perm = torch.randperm(n_pages, generator=torch.Generator().manual_seed(seed + 1)).tolist()
        if last:                     # the cache's last pages
            perm = list(range(n_pages))
        self.tables_list = [[perm.pop() for _ in range(m)] for m in need]
        width = width or max(max(need), 1)
        t = torch.full((B, width), -1, dtype=torch.int32)
        for b, row in enumerate(self.tables_list):
            t[b, :len(row)] = torch.tensor(row, dtype=torch.int32)
        self.tables = t.cuda()
        self.lens = torch.tensor(self.lens_list, dtype=torch.int32).cuda()
        self.cu_list = [0]
        for n in new:
            self.cu_list.append(self.cu_list[-1] + n)
        self.cu = torch.tensor(self.cu_list, dtype=torch.int32).cuda()
        self.cache.k.fill_(math.nan)
        self.cache.v.fill_(math.nan)
        self.k, self.v = [], []      # [len, kv_heads, hd] of each sequence
        for b, n in enumerate(lens):
            k = torch.randn(n, kv_heads, hd, generator=g, device="cuda").to(dtype)
            v = torch.randn(n, kv_heads, hd, generator=g, device="cuda").to(dtype)
            self.k.append(k)
            self.v.append(v)
            self.put(b, k, v)
        self.q = (1.5 * torch.randn(self.cu_list[-1], heads, hd, generator=g, device="cuda")).to(dtype)

    def put(self, b, k, v, first=0):
        """Positions first.. of sequence b, written value by value by the layout's definition."""
        n = k.shape[0]
        if n == 0:
            return
        page, hd = self.cache.page, self.cache.head_dim
        p = torch.arange(first, first + n, device="cuda")
        ids = torch.tensor(self.tables_list[b], device="cuda")[p // page]
        h = torch.arange(self.cache.kv_heads, device="cuda")
        e = torch.arange(hd, device="cuda")
        i, hh, ee = ids[:, None, None], h[None, :, None], e[None, None, :]
        blk, at = (p % page // 16)[:, None, None], (p % 16)[:, None, None]
        self.cache.k[i, hh, blk, ee // 16, at, ee % 16] = k
        self.cache.v[i, hh, blk, ee, at] = v


def reference(q, k, v, scale, first):
    """q [n, H, hd], k and v [m, KV, hd], row i sees positions 0 .. first + i: (out, error's weight, |v| sum) in 64
    bits.  Zeros for rows that see nothing."""
    n, H, hd = q.shape
    m, KV, _ = k.shape
    out = torch.zeros(n, H, hd, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    half = HALF_STEP[q.dtype]
    if m == 0 or n == 0:
        return out, tol
    sees = torch.arange(m, device=q.device)[None] <= (first + torch.arange(n, device=q.device))[:, None]
    for h in range(H):
        kk, vv = k[:, h // (H // KV)].double(), v[:, h // (H // KV)].double()
        qq = q[:, h].double()
        s = (qq @ kk.T.contiguous()) * scale
        mag = ((qq.abs() @ kk.abs().T.contiguous()) * scale).masked_fill(~sees, 0.0).amax(1, keepdim=True)
        s = s.masked_fill(~sees, -math.inf)
        p = torch.exp(s - s.amax(1, keepdim=True).clamp(min=-1e300))
        total = p.sum(1, keepdim=True)
        p = torch.where(total > 0, p / total, torch.zeros_like(p))
        out[:, h] = p @ vv
        # A score is off by hd additions and four products, exponential and all by 2^-21 more; weights are rounded
        # to the cache's type and summed over m positions in f32 (both products), their sum too; an f16 weight below
        # 2^-14 of its range by 2^-33 of the largest.
        e = (hd + 6) * 2.0 ** -24 * mag + 2.0 ** -21
        tol[:, h] = (p @ vv.abs()) * (half + 2 * e + 2 * (m + 64) * 2.0 ** -24) + 2.0 ** -33 * vv.abs().sum(0)
    return out, tol


def close(got, want, tol, what=""):
    """Within tol and the result's own half step (a subnormal's: 2^-25 in f16)."""
    bound = tol * 1.0001 + (want.abs() + tol) * HALF_STEP[got.dtype] + (2.0 ** -25 if got.dtype is torch.float16 else 0.0)
    err = (got.double() - want).abs()
    bad = ~(err <= bound)
    assert not bad.any(), (what, int(bad.sum()), float((err / bound.clamp(min=1e-300))[bad].max()),
                           [int(i) for i in bad.nonzero()[0]])
