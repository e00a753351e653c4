"""The attention half of a layer for a batch of sequences, as cases that can be timed and compared.

Kinds (a case's "kind"):

  norm     what a sublayer hands on: the residual's addition, the RMS norm, E4M3 codes with a scale per 128 values
           (the next product's input)
  append   rows of q | k | v behind a projection: norms of the query and key heads, rotary positions, keys
           and values into a paged cache; the queries come back
  decode   attention of one new token a sequence over the paged cache
  prompt   causal attention of prompts packed end to end (some behind a cached prefix), over the paged cache

`own` false computes the plain form in elementary torch operations; true makes the package's calls.
The cache's layout is the operators' format: a page holds blocks of 16 positions, a key block as
[head_dim / 16][16 positions][16 values], a value block as [head_dim][16 positions].
Head layouts are those of Qwen3-30B-A3B (32 query heads on 4 of 128), of Qwen3-235B-A22B (64 on 4 of
128) and of the synthetic four-layer model (8 on 2 of 64), and odd ones."""
import math
import random

import torch

own = False

E4M3 = torch.float8_e4m3fn
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 2.0 ** -20                           # a float whatever the width it is held in
THETA = 1e6
MOST_NORM = 8192 * 4096                    # values of a norm
MOST_APPEND = 8192 * 72 * 128              # values of an append
MOST_CACHE = 61 * 2000 * 4 * 128           # keys of the cache behind one
MOST_DECODE = 64 * 4097 * 4 * 2 * 128      # cached values that a decode reads
MOST_PROMPT = 2 * 16384 * 16384 * 32 * 128   # operations of a prompt


def listed():
    return [
        # a decode step's residual before a projection: latency alone
        {"name": "norm_1x2048", "kind": "norm", "T": 1, "n": 2048, "x": "bf16", "h": "f32"},
        # 61 sequences of a model of odd width, all in 16 bits
        {"name": "norm_61x1111_f16", "kind": "norm", "T": 61, "n": 1111, "x": "f16", "h": "f16"},
        # a long prompt's residuals (235B)
        {"name": "norm_8192x4096", "kind": "norm", "T": 8192, "n": 4096, "x": "bf16", "h": "f32"},
        # a decode step of 61 sequences (30B): one row each
        {"name": "append_61_30b", "kind": "append", "B": 61, "T": 61, "past": 4000, "H": 32, "KV": 4, "hd": 128,
         "page": 64, "x": "f32", "dt": "bf16"},
        # prompts of five sequences packed end to end (235B), some behind a cached prefix
        {"name": "append_8192_235b", "kind": "append", "B": 5, "T": 8192, "past": 700, "H": 64, "KV": 4, "hd": 128,
         "page": 64, "x": "bf16", "dt": "bf16"},
        # one sequence of the small model, not far into its context: latency alone
        {"name": "decode_1_small", "kind": "decode", "B": 1, "len": 300, "H": 8, "KV": 2, "hd": 64, "page": 16,
         "dt": "f16"},
        # one sequence of 30B at the end of a long context: the cache's length has to be split
        {"name": "decode_1_131071", "kind": "decode", "B": 1, "len": 131071, "H": 32, "KV": 4, "hd": 128, "page": 64,
         "dt": "bf16"},
        # 64 sequences of 235B, each somewhere in its first 8192 positions
        {"name": "decode_64_235b", "kind": "decode", "B": 64, "len": 8192, "H": 64, "KV": 4, "hd": 128, "page": 64,
         "dt": "bf16"},
        # an odd head layout, small pages, f16
        {"name": "decode_7_odd", "kind": "decode", "B": 7, "len": 5001, "H": 15, "KV": 5, "hd": 96, "page": 16,
         "dt": "f16"},
        # a short prompt of 30B
        {"name": "prompt_77_30b", "kind": "prompt", "B": 1, "T": 77, "past": 0, "H": 32, "KV": 4, "hd": 128, "page": 64,
         "dt": "bf16"},
        # nine prompts of the small model's heads packed end to end, most behind a cached prefix
        {"name": "prompt_3001_small", "kind": "prompt", "B": 9, "T": 3001, "past": 1500, "H": 8, "KV": 2, "hd": 64,
         "page": 16, "dt": "f16"},
        # one long prompt of 30B: the largest product
        {"name": "prompt_16384_30b", "kind": "prompt", "B": 1, "T": 16384, "past": 0, "H": 32, "KV": 4, "hd": 128,
         "page": 64, "dt": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def _heads(rng):
    KV = rng.choice([1, 2, 3, 4, 4, 4, 8])
    return {"H": KV * rng.choice([1, 2, 3, 4, 5, 8, 8, 16]), "KV": KV, "hd": rng.choice([32, 64, 96, 128, 128, 128, 192, 256]),
            "page": rng.choice([16, 32, 64, 128]), "dt": rng.choice(["f16", "bf16"])}


def draw(rng):
    kind = rng.choice(["norm", "append", "decode", "decode", "decode", "prompt", "prompt", "prompt"])
    types = ["f32", "f16", "bf16"]
    if kind == "norm":
        n = _log(rng, 32, 16384)
        return {"kind": kind, "T": _log(rng, 1, MOST_NORM // n if n > 4096 else 8192), "n": n, "x": rng.choice(types),
                "h": rng.choice(types)}
    heads = _heads(rng)
    H, KV, hd = heads["H"], heads["KV"], heads["hd"]
    if kind == "append":
        T = _log(rng, 1, min(8192, MOST_APPEND // ((H + 2 * KV) * hd) * 2 // 3))
        B = rng.choice([T if T <= 128 else 1, 1, _log(rng, 1, min(T, 64))])
        past = _log(rng, 1, min(4000, MOST_CACHE // (B * KV * hd))) - 1
        return {"kind": kind, "B": B, "T": T, "past": past, "x": rng.choice(types), **heads}
    if kind == "decode":
        B = _log(rng, 1, 128)
        return {"kind": kind, "B": B, "len": _log(rng, 1, min(131072, MOST_DECODE // (B * KV * hd * 2))), **heads}
    T = _log(rng, 1, 8192)
    B = _log(rng, 1, min(T, 16))
    past = rng.choice([0, _log(rng, 1, 4000)])
    while T > 1 and 4 * T * (past + T // 2 + 1) * H * hd > MOST_PROMPT:
        T = T // 2
    return {"kind": kind, "B": min(B, T), "T": T, "past": past, **heads}


# ---- inputs ------------------------------------------------------------------------------------

class _State:
    pass


class _Rand:
    """Tensors on the GPU from one seed."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(seed * 7919 + 47)

    def normal(self, *shape):
        return torch.randn(*shape, generator=self.g, device="cuda", dtype=torch.float32)

    def typed(self, dt, *shape):
        return torch.randn(*shape, generator=self.g, device="cuda", dtype=TYPES[dt])

    def acts(self, T, n):
        """Activations as a layer sees them: most channels about 1, a few much larger, tokens of different size."""
        return self.normal(T, n) * torch.exp(0.5 * self.normal(n)) * torch.exp(0.5 * self.normal(T, 1))


def _lengths(case):
    """New rows and positions (cached ones and new ones) of each sequence, the same for every seed."""
    B = case["B"]
    rng = random.Random(B * 1000003 + case.get("T", 0) * 101 + case.get("past", 0) * 7 + case.get("len", 0))
    if case["kind"] == "decode":
        lens = [rng.randint(1, case["len"]) for _ in range(B)]
        lens[rng.randrange(B)] = case["len"]
        return [1] * B, lens
    cuts = [0] + sorted(rng.sample(range(1, case["T"]), B - 1)) + [case["T"]]
    new = [b - a for a, b in zip(cuts, cuts[1:])]
    return new, [n + rng.randint(0, case["past"]) for n in new]


def prepare(case, seed):
    r, s = _Rand(seed), _State()
    s.case, kind = case, case["kind"]
    if kind == "norm":
        T, n = case["T"], case["n"]
        s.x, s.h = r.acts(T, n).to(TYPES[case["x"]]), r.acts(T, n).to(TYPES[case["h"]])
        s.w = 1.0 + 0.1 * r.normal(n)
        if own:
            from tierlm_amd import quant
            quant.init(0)
            s.h0, s.h = s.h, torch.empty_like(s.h)
        return s
    H, KV, hd, page = (case[k] for k in ("H", "KV", "hd", "page"))
    s.new, s.lens_list = _lengths(case)
    T, B = sum(s.new), case["B"]
    need = [-(-n // page) for n in s.lens_list]
    n_pages = sum(need) + 1
    free = torch.randperm(n_pages, generator=torch.Generator().manual_seed(seed * 31 + 5), dtype=torch.int32)
    s.tables = torch.full((B, max(need)), -1, dtype=torch.int32)
    at = 0
    for b, m in enumerate(need):
        s.tables[b, :m] = free[at:at + m]
        at += m
    s.tables = s.tables.cuda()
    s.lens = torch.tensor(s.lens_list, dtype=torch.int32, device="cuda")
    s.cu_list = [0]
    for n in s.new:
        s.cu_list.append(s.cu_list[-1] + n)
    s.cu = torch.tensor(s.cu_list, dtype=torch.int32, device="cuda")
    s.k = r.typed(case["dt"], n_pages, KV, page // 16, hd // 16, 16, 16)
    s.v = r.typed(case["dt"], n_pages, KV, page // 16, hd, 16)
    if kind == "append":
        s.x = (r.normal(T, (H + 2 * KV) * hd) * torch.exp(0.3 * r.normal(T, 1))).to(TYPES[case["x"]])
        s.q_norm, s.k_norm = 1.0 + 0.1 * r.normal(hd), 1.0 + 0.1 * r.normal(hd)
        s.inv_freq = THETA ** (torch.arange(hd // 2, dtype=torch.float64, device="cuda") * (-2.0 / hd))
    else:
        s.q = (r.normal(T, H, hd) * 1.5).to(TYPES[case["dt"]])
    if own:
        from tierlm_amd import kv, quant
        quant.init(0)
        s.cache = kv.Cache(n_pages, KV, hd, page=page, dtype=TYPES[case["dt"]])
        s.cache.k.copy_(s.k)
        s.cache.v.copy_(s.v)
        s.k, s.v = s.cache.k, s.cache.v
    return s


# ---- the plain forms ---------------------------------------------------------------------------

def _norm(s):
    """The sum of squares in 64 bits: a value next to the border of two codes keeps its side."""
    T, n = s.x.shape
    h = (s.h.float() + s.x.float()).to(s.h.dtype)
    f = h.float()
    r = (1.0 / torch.sqrt(f.double().square().mean(-1, keepdim=True) + EPS)).float()
    nb = -(-n // 128)
    b = torch.nn.functional.pad(f * r * s.w, (0, 128 * nb - n)).reshape(T, nb, 128)
    m, e = torch.frexp(b.abs().amax(-1))                  # amax = m 2^e, 0.5 <= m < 1
    e = torch.where(m > 0.875, e - 8, e - 9).clamp(min=-126)
    one = torch.ones_like(m)
    codes = (b * torch.ldexp(one, -e)[..., None]).to(E4M3)
    return h, codes.reshape(T, 128 * nb), torch.where(m > 0, torch.ldexp(one, e), 0.0)


def _places(s):
    """Page, block and position in the block of every new row, and its position."""
    page, pos, seq = s.case["page"], [], []
    for b, (n, m) in enumerate(zip(s.new, s.lens_list)):
        pos.append(torch.arange(m - n, m))
        seq.append(torch.full((n,), b))
    pos, seq = torch.cat(pos).cuda(), torch.cat(seq).cuda()
    return s.tables[seq, pos // page].long(), pos % page // 16, pos % 16, pos


def _append(s):
    H, KV, hd = (s.case[k] for k in ("H", "KV", "hd"))
    p, blk, at, pos = _places(s)
    T = s.x.shape[0]
    x = s.x.float().reshape(T, H + 2 * KV, hd)
    w = torch.cat([s.q_norm.expand(H, hd), s.k_norm.expand(KV, hd)])
    y = x[:, :H + KV]
    y = y * (1.0 / torch.sqrt(y.square().mean(-1, keepdim=True) + EPS)) * w
    a = pos.double()[:, None] * s.inv_freq                # far positions: the angle in 64 bits
    c, sn = torch.cos(a).float()[:, None], torch.sin(a).float()[:, None]
    lo, hi = y[..., :hd // 2], y[..., hd // 2:]
    y = torch.cat([lo * c - hi * sn, hi * c + lo * sn], -1).to(s.k.dtype)
    s.k[p, :, blk, :, at] = y[:, H:].reshape(T, KV, hd // 16, 16)
    s.v[p, :, blk, :, at] = x[:, H + KV:].to(s.v.dtype)
    return y[:, :H].contiguous(), s.k, s.v


def _context(s, b):
    """Keys [KV, hd, len] and values [KV, len, hd] of sequence b, in 32 bits."""
    page, n = s.case["page"], s.lens_list[b]
    ids = s.tables[b, :-(-n // page)].long()
    k = s.k[ids].permute(1, 3, 5, 0, 2, 4).reshape(s.case["KV"], s.case["hd"], -1)[:, :, :n]
    v = s.v[ids].permute(1, 0, 2, 4, 3).reshape(s.case["KV"], -1, s.case["hd"])[:, :n]
    return k.float().contiguous(), v.float().contiguous()


def _softmax(x):
    x = torch.exp(x - x.amax(-1, keepdim=True))
    return x / x.sum(-1, keepdim=True)


def _attend(s):
    """Row by row in chunks whose scores fit; row i of a sequence sees what is not behind its own position."""
    H, KV, hd = (s.case[k] for k in ("H", "KV", "hd"))
    G, out = H // KV, torch.empty_like(s.q)
    for b, (n, m) in enumerate(zip(s.new, s.lens_list)):
        k, v = _context(s, b)
        step = max(1, 2 ** 28 // (H * m))
        for i in range(0, n, step):
            j = min(n, i + step)
            q = s.q[s.cu_list[b] + i:s.cu_list[b] + j].float() * (1.0 / math.sqrt(hd))
            x = q.reshape(j - i, KV, G, hd).permute(1, 2, 0, 3).reshape(KV, -1, hd) @ k
            if m - n + i + 1 < m:
                rows, cols = torch.arange(i, j, device="cuda") + (m - n), torch.arange(m, device="cuda")
                x.view(KV, G, j - i, m).masked_fill_(cols[None] > rows[:, None], -math.inf)
            y = (_softmax(x) @ v).reshape(KV, G, j - i, hd).permute(2, 0, 1, 3).reshape(j - i, H, hd)
            out[s.cu_list[b] + i:s.cu_list[b] + j] = y.to(out.dtype)
    return out


def run(s):
    kind = s.case["kind"]
    if not own:
        return _norm(s) if kind == "norm" else _append(s) if kind == "append" else _attend(s)
    from tierlm_amd import fp8, kv
    if kind == "norm":      # the residual before the sum is the state's; a program's own would be updated in place
        codes, scale = fp8.add_rmsnorm(s.h0, s.x, s.w, EPS, out=s.h)
        return s.h, codes, scale
    if kind == "append":
        q = kv.append(s.cache, s.x, s.case["H"], s.tables, s.lens, cu=None if s.case["B"] == s.case["T"] else s.cu,
                      q_norm=s.q_norm, k_norm=s.k_norm, eps=EPS, inv_freq=s.inv_freq)
        return q, s.k, s.v
    if kind == "decode":
        return kv.decode(s.q, s.cache, s.tables, s.lens)
    return kv.prompt(s.q, s.cache, s.tables, s.lens, s.cu)


# ---- what a pass cannot do without -------------------------------------------------------------

def work(case):
    if case["kind"] == "norm":
        T, n = case["T"], case["n"]
        return {"bytes": T * n * (SIZE[case["x"]] + 2 * SIZE[case["h"]] + 1) + T * -(-n // 128) * 4 + n * 4,
                "flops": 7 * T * n}
    H, KV, hd = (case[k] for k in ("H", "KV", "hd"))
    new, lens = _lengths(case)
    if case["kind"] == "append":
        values = sum(new) * (H + 2 * KV) * hd
        return {"bytes": values * (SIZE[case["x"]] + 2), "flops": 6 * values}
    seen = sum(sum(range(m - n + 1, m + 1)) for n, m in zip(new, lens))
    return {"bytes": 4 * sum(lens) * KV * hd + 4 * sum(new) * H * hd, "flops": 4 * seen * H * hd}


# ---- the definitions in 64 bits ----------------------------------------------------------------

def _exact_norm(s):
    x, h = s.x.double(), s.h.double()
    T, n = x.shape
    h = (x + h).to(s.h.dtype).double()     # held in its own type between layers
    y = h * torch.rsqrt((h * h).sum(1, keepdim=True) / n + EPS) * s.w.double()
    nb = -(-n // 128)
    v = torch.zeros(T, nb * 128, dtype=torch.float64, device=x.device)
    v[:, :n] = y
    v = v.view(T, nb, 128)
    amax = v.abs().max(-1).values
    e = torch.ceil(torch.log2(torch.clamp(amax, min=1e-300) / 448.0)).clamp(min=-126.0)
    e = torch.where(448.0 * torch.exp2(e - 1.0) >= amax, e - 1.0, e).clamp(min=-126.0)   # log2 rounds
    e = torch.where(448.0 * torch.exp2(e) < amax, e + 1.0, e)
    u = v / torch.exp2(e)[..., None]
    step = torch.exp2(torch.floor(torch.log2(torch.clamp(u.abs(), min=2.0 ** -6))).clamp(min=-6.0) - 3.0)
    return h, (torch.round(u / step) * step).view(T, nb * 128), torch.where(amax > 0, torch.exp2(e), 0.0)


def _exact_append(s):
    H, KV, hd, page = (s.case[k] for k in ("H", "KV", "hd", "page"))
    k, v, out = s.k.double(), s.v.double(), torch.empty(s.x.shape[0], H, hd, dtype=torch.float64, device="cuda")
    freq = torch.tensor([THETA ** (-2.0 * j / hd) for j in range(hd // 2)], dtype=torch.float64, device="cuda")
    for b, (n, m) in enumerate(zip(s.new, s.lens_list)):
        rows = s.x[s.cu_list[b]:s.cu_list[b + 1]].double().view(n, H + 2 * KV, hd)
        pos = torch.arange(m - n, m, device="cuda")
        turn = torch.polar(torch.ones(n, hd // 2, dtype=torch.float64, device="cuda"), pos[:, None] * freq)[:, None]

        def rotated(x, w):
            x = x * torch.rsqrt((x * x).sum(-1, keepdim=True) / hd + EPS) * w.double()
            z = torch.complex(x[..., :hd // 2].contiguous(), x[..., hd // 2:].contiguous()) * turn
            return torch.cat([z.real, z.imag], -1)

        out[s.cu_list[b]:s.cu_list[b + 1]] = rotated(rows[:, :H], s.q_norm)
        keys, values = rotated(rows[:, H:H + KV], s.k_norm), rows[:, H + KV:]
        for first in range((m - n) // page * page, m, page):     # a page at a time
            lo, hi = max(first, m - n), min(first + page, m)
            at, sel = torch.arange(lo - first, hi - first, device="cuda"), slice(lo - (m - n), hi - (m - n))
            pid = int(s.tables[b, first // page])
            k[pid].permute(1, 3, 0, 2, 4)[at // 16, at % 16] = keys[sel].view(hi - lo, KV, hd // 16, 16)
            v[pid].permute(1, 3, 0, 2)[at // 16, at % 16] = values[sel]
    return out, k, v


def _exact_attend(s):
    H, KV, hd, page = (s.case[k] for k in ("H", "KV", "hd", "page"))
    out = torch.empty(s.q.shape, dtype=torch.float64, device="cuda")
    for b, (n, m) in enumerate(zip(s.new, s.lens_list)):
        j = torch.arange(m, device="cuda")
        pid = s.tables[b][j // page].long()
        for h in range(H):
            g = h // (H // KV)
            k = s.k[pid, g, j % page // 16, :, j % 16].reshape(m, hd).double()
            v = s.v[pid, g, j % page // 16, :, j % 16].double()
            for i in range(0, n, 2048):
                q = s.q[s.cu_list[b] + i:s.cu_list[b] + min(n, i + 2048), h].double()
                x = torch.matmul(k, q.T.contiguous()).T / math.sqrt(hd)
                x = x + torch.triu(torch.full_like(x, -math.inf), diagonal=m - n + i + 1)
                out[s.cu_list[b] + i:s.cu_list[b] + i + q.shape[0], h] = torch.softmax(x, 1) @ v
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if own and case["kind"] == "norm":
        s.h = s.h0
    return {"norm": _exact_norm, "append": _exact_append}.get(case["kind"], _exact_attend)(s)
