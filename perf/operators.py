"""The library's 8-bit floating-point operators, as cases that can be timed and compared.

Kinds (a case's "kind"):

  quantize   T activation vectors of n values to E4M3 codes with a scale per 128 values
  matmul     T vectors already in codes, times a matrix of E4M3 codes with a scale per 128 x 128
  linear     both, as a program calls them for one projection: quantise, then multiply
  moe        a whole mixture-of-experts layer (norm, router, experts, shared expert, residual) for
             a few tokens, its matrices E4M3 with a scale per 128 x 128

`own` false computes the plain form in elementary torch operations; true makes the package's calls.
Sizes are those of the synthetic four-layer model (hidden 512, 32 experts of width 256 and a
shared one), of Qwen3-30B-A3B (hidden 2048, 128 experts of width 768) and of Qwen3-235B-A22B
(hidden 4096, width 1536), and odd ones."""
import math

import torch

own = False

E4M3 = torch.float8_e4m3fn
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
MOST_MACS = 4096 * 8192 * 4096          # of a matmul
MOST_WEIGHTS = 151936 * 2048            # of a matmul's matrix
MOST_EXPERTS = 128 * 3 * 1536 * 4096    # of a layer's experts


def listed():
    return [
        # a decode step's activation vector before a projection: latency alone
        {"name": "quantize_1x2048", "kind": "quantize", "T": 1, "n": 2048, "x": "f32"},
        # a prompt's activations before a down projection, in 16 bits
        {"name": "quantize_4096x8192_bf16", "kind": "quantize", "T": 4096, "n": 8192, "x": "bf16"},
        # the smallest projection of the small model, one token: two launches and nothing to hide them behind
        {"name": "linear_1_512x512", "kind": "linear", "T": 1, "rows": 512, "n": 512, "x": "f32", "y": "f32"},
        # the head of a 151936-word model for one token: the largest matrix that a decode step reads
        {"name": "matmul_1_head", "kind": "matmul", "T": 1, "rows": 151936, "n": 2048, "y": "f32"},
        # a batch of 16 sequences at decode through an output projection (235B)
        {"name": "matmul_16_4096x8192", "kind": "matmul", "T": 16, "rows": 4096, "n": 8192, "y": "f32"},
        # a short prompt through a matrix of odd sizes, quantised on the way
        {"name": "linear_77_1000x1111", "kind": "linear", "T": 77, "rows": 1000, "n": 1111, "x": "bf16", "y": "bf16"},
        # a long prompt's query projection (235B): the largest product
        {"name": "matmul_4096_8192x4096", "kind": "matmul", "T": 4096, "rows": 8192, "n": 4096, "y": "bf16"},
        # the small model's layer, one token, with its shared expert: latency alone
        {"name": "moe_1_small", "kind": "moe", "T": 1, "D": 512, "de": 256, "E": 32, "k": 4, "ds": 256, "router": 0},
        # a decode step of 30B
        {"name": "moe_1_30b", "kind": "moe", "T": 1, "D": 2048, "de": 768, "E": 128, "k": 8, "ds": 0, "router": 0},
        # eight sequences at decode, 30B: half as many distinct experts as tokens ask for
        {"name": "moe_8_30b", "kind": "moe", "T": 8, "D": 2048, "de": 768, "E": 128, "k": 8, "ds": 0, "router": 0},
        # as many sequences as the layer takes at once, 235B: nearly every expert, few tokens each
        {"name": "moe_64_235b", "kind": "moe", "T": 64, "D": 4096, "de": 1536, "E": 128, "k": 8, "ds": 0, "router": 0},
        # odd widths, few experts with many tokens each, sigmoid scores with a bias, a shared expert
        {"name": "moe_61_odd", "kind": "moe", "T": 61, "D": 1000, "de": 333, "E": 10, "k": 3, "ds": 200, "router": 2},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["quantize", "matmul", "matmul", "linear", "moe", "moe", "moe"])
    types = ["f32", "f32", "f16", "bf16"]
    if kind == "quantize":
        n = _log(rng, 32, 16384)
        return {"kind": kind, "T": _log(rng, 1, min(8192, 4096 * 8192 // n)), "n": n, "x": rng.choice(types)}
    if kind != "moe":
        while True:
            rows, n = _log(rng, 64, 151936), _log(rng, 32, 16384)
            if rows * n <= MOST_WEIGHTS:
                break
        T = _log(rng, 1, max(1, min(4096, MOST_MACS // (rows * n), 2 * 10**8 // rows)))
        return {"kind": kind, "T": T, "rows": rows, "n": n, **({"x": rng.choice(types)} if kind == "linear" else {}),
                "y": rng.choice(types)}
    while True:
        D, de, E, ds = _log(rng, 256, 4096), _log(rng, 64, 1536), _log(rng, 8, 128), rng.choice([0, 0, _log(rng, 64, 1024)])
        if 3 * D * (E * de + ds) <= MOST_EXPERTS:
            break
    return {"kind": kind, "T": _log(rng, 1, 64), "D": D, "de": de, "E": E, "k": min(E, rng.randint(1, 8)),
            "ds": ds, "router": rng.choice([0, 0, 1, 2])}


# ---- inputs ------------------------------------------------------------------------------------

class _State:
    pass


class _Rand:
    """Tensors on the GPU from one seed."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(seed * 7919 + 31)

    def normal(self, *shape):
        return torch.randn(*shape, generator=self.g, device="cuda", dtype=torch.float32)

    def acts(self, T, n):
        """Activations as a layer sees them: most channels about 1, a few much larger, tokens of different size."""
        return self.normal(T, n) * torch.exp(0.5 * self.normal(n)) * torch.exp(self.normal(T, 1))

    def matrix(self, *shape):
        """E4M3 codes [..., rows, n] and scales [..., rows / 128, n / 128] (rounded up) of normal weights, as a
        checkpoint holds them: each block's largest weight near 448."""
        *lead, rows, n = shape
        w = self.normal(*lead, rows, n) * 100.0
        w = w.clamp_(-448.0, 448.0).to(E4M3)
        s = torch.exp(0.3 * self.normal(*lead, -(-rows // 128), -(-n // 128))) * (0.01 / math.sqrt(n))
        return w, s


def _library():
    from tierlm_amd import fp8, quant
    quant.init(0)
    return fp8


def prepare(case, seed):
    r, s = _Rand(seed), _State()
    s.case, kind = case, case["kind"]
    if kind == "moe":
        T, D, de, E, ds = (case[k] for k in ("T", "D", "de", "E", "ds"))
        s.h = r.normal(T, D) * torch.exp(0.3 * r.normal(T, 1))
        s.norm = 1.0 + 0.1 * r.normal(D)
        s.router_w = r.normal(E, D) / math.sqrt(D)
        s.bias = 0.1 * r.normal(E) if case["router"] == 2 else None
        s.routed_scale, s.eps = (2.5 if case["router"] == 2 else 1.0), 1e-6
        s.gate, s.up, s.down = r.matrix(E, de, D), r.matrix(E, de, D), r.matrix(E, D, de)
        s.shared = [r.matrix(ds, D), r.matrix(ds, D), r.matrix(D, ds)] if ds else None
        if own:   # the weights laid out once, as a program keeps them from its start on
            fp8 = _library()
            s.mats = [fp8.pack(m[0][e], m[1][e]) for e in range(E) for m in (s.gate, s.up, s.down)]
            s.smats = [fp8.pack(w, sc) for w, sc in s.shared] if ds else None
            s.block = fp8.MoeBlock(D=D, de=de, E=E, k=case["k"], ffn_norm=s.norm, router_w=s.router_w,
                                   expert_ptrs=[m.data_ptr() for m in s.mats], router=case["router"],
                                   routed_scale=s.routed_scale, eps=s.eps, router_bias=s.bias, ds=ds, shared=s.smats)
            s.out, s.w = torch.empty_like(s.h), torch.empty(T, case["k"], device="cuda")
            s.ids = torch.empty(T, case["k"], dtype=torch.int32, device="cuda")
        return s
    T, n = case["T"], case["n"]
    x = r.acts(T, n)
    if kind == "matmul":   # codes in hand: an earlier layer quantised them
        s.codes, s.scale = _quantize(x)
    else:
        s.x = x.to(TYPES[case["x"]])
    if kind != "quantize":
        s.w, s.ws = r.matrix(case["rows"], n)
        if own:
            fp8 = _library()
            s.wp = fp8.pack(s.w, s.ws)
    elif own:
        _library()
    return s


# ---- the plain forms ---------------------------------------------------------------------------

def _pad(x, n):
    return torch.nn.functional.pad(x, (0, n - x.shape[-1]))


def _quantize(x):
    """codes [T, np] and scales [T, np / 128], np the length rounded up to 128: the least power of two that
    brings the block's largest magnitude to 448 or below."""
    T, n = x.shape
    nb = -(-n // 128)
    b = _pad(x.float(), 128 * nb).reshape(T, nb, 128)
    m, e = torch.frexp(b.abs().amax(-1))                  # amax = m 2^e, 0.5 <= m < 1
    e = torch.where(m > 0.875, e - 8, e - 9).clamp(min=-126)
    one = torch.ones_like(m)
    codes = (b * torch.ldexp(one, -e)[..., None]).to(E4M3)
    return codes.reshape(T, 128 * nb), torch.where(m > 0, torch.ldexp(one, e), 0.0)


def _values(codes, scale):
    T, np_ = codes.shape
    return (codes.float().reshape(T, np_ // 128, 128) * scale[..., None]).reshape(T, np_)


def _weights(w, s):
    """The values of a matrix (or of a stack of them): code times its 128 x 128 block's scale."""
    rows, n = w.shape[-2:]
    full = s.repeat_interleave(128, -2)[..., :rows, :].repeat_interleave(128, -1)[..., :n]
    return w.float() * full


def _silu(x):
    return x / (1.0 + torch.exp(-x))


def _route(s, xb):
    """ids and weights in rank order; the scores in 64 bits, so that two close ones keep their order."""
    case = s.case
    logits = xb.double() @ s.router_w.double().T
    p = torch.exp(logits - logits.amax(-1, keepdim=True))
    p = 1.0 / (1.0 + torch.exp(-logits)) if case["router"] == 2 else p / p.sum(-1, keepdim=True)
    sel = p + s.bias.double() if s.bias is not None else p
    ids = torch.sort(sel, dim=-1, descending=True, stable=True)[1][:, :case["k"]]
    w = torch.gather(p, 1, ids)
    if case["router"] != 1:
        w = w / (w.sum(-1, keepdim=True) + (1e-20 if case["router"] == 2 else 0.0))
    return ids, (w * s.routed_scale).float()


def _moe(s):
    T, D = s.h.shape
    E, k = s.case["E"], s.case["k"]
    ms = s.h.double().square().mean(-1, keepdim=True).float()
    xb = s.h / torch.sqrt(ms + s.eps) * s.norm
    ids, w = _route(s, xb)
    if T * k <= E:      # the chosen experts, one for each token and rank
        at = ids.reshape(-1)
        xs = xb.repeat_interleave(k, 0)[..., None]
        h = _silu(_weights(s.gate[0][at], s.gate[1][at]) @ xs) * (_weights(s.up[0][at], s.up[1][at]) @ xs)
        y = (_weights(s.down[0][at], s.down[1][at]) @ h).reshape(T, k, D)
    else:               # every expert for every token, and the chosen ones' results
        xs = xb.T.contiguous()
        h = _silu(_weights(*s.gate) @ xs) * (_weights(*s.up) @ xs)
        y = (_weights(*s.down) @ h).permute(2, 0, 1)[torch.arange(T, device=ids.device)[:, None], ids]
    out = (y * w[..., None]).sum(1)
    if s.shared:
        g, u, d = (_weights(*m) for m in s.shared)
        out = out + (_silu(xb @ g.T) * (xb @ u.T)) @ d.T
    return s.h + out, ids.int(), w


def run(s):
    kind = s.case["kind"]
    if own:
        from tierlm_amd import fp8
        if kind == "moe":
            return s.block(s.h, out=s.out, ids=s.ids, w=s.w), s.ids, s.w
        if kind == "matmul":
            return fp8.matmul(s.wp, s.case["rows"], s.case["n"], s.codes, s.scale, dtype=TYPES[s.case["y"]])
        codes, scale = fp8.quantize(s.x)
        if kind == "quantize":
            return codes, scale
        return fp8.matmul(s.wp, s.case["rows"], s.case["n"], codes, scale, dtype=TYPES[s.case["y"]])
    if kind == "moe":
        return _moe(s)
    if kind == "matmul":
        codes, scale = s.codes, s.scale
    else:
        codes, scale = _quantize(s.x)
    if kind == "quantize":   # E4M3 numbers and the scales that they are multiplied with
        return codes, scale
    x, n = _values(codes, scale), s.case["n"]
    return (x[:, :n] @ _weights(s.w, s.ws).T).to(TYPES[s.case["y"]])


# ---- what a pass cannot do without -------------------------------------------------------------

def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}
    kind, T = case["kind"], case["T"]
    if kind == "moe":
        D, de, E, k, ds = (case[x] for x in ("D", "de", "E", "k", "ds"))
        used = E * (1.0 - (1.0 - k / E) ** T)     # the experts that T tokens of k choices reach, on average
        mats = used * 3 * D * de + 3 * D * ds
        return {"bytes": int(mats * (1 + 4 / 16384) + E * D * 4 + D * 4 + 2 * T * D * 4 + T * k * 8),
                "flops": 2 * T * (3 * D * (k * de + ds) + E * D)}
    n = case["n"]
    codes = T * n + T * (-(-n // 128)) * 4
    if kind == "quantize":
        return {"bytes": T * n * size[case["x"]] + codes, "flops": 3 * T * n}
    rows = case["rows"]
    moved = rows * n + (-(-rows // 128)) * (-(-n // 128)) * 4 + T * rows * size[case["y"]]
    moved += codes if kind == "matmul" else T * n * size[case["x"]]
    return {"bytes": moved, "flops": 2 * T * rows * n}


# ---- the definitions in 64 bits ----------------------------------------------------------------

def _exact_codes(x):
    """x [T, n] in 64 bits -> the codes' values [T, np] and the scales [T, np / 128], by arithmetic alone."""
    T, n = x.shape
    nb = -(-n // 128)
    v = torch.zeros(T, nb * 128, dtype=torch.float64, device=x.device)
    v[:, :n] = x.double()
    v = v.view(T, nb, 128)
    amax = v.abs().max(-1).values
    e = torch.ceil(torch.log2(torch.clamp(amax, min=1e-300) / 448.0)).clamp(min=-126.0)
    e = torch.where(448.0 * torch.exp2(e - 1.0) >= amax, e - 1.0, e).clamp(min=-126.0)   # log2 rounds
    e = torch.where(448.0 * torch.exp2(e) < amax, e + 1.0, e)
    y = v / torch.exp2(e)[..., None]
    step = torch.exp2(torch.floor(torch.log2(torch.clamp(y.abs(), min=2.0 ** -6))).clamp(min=-6.0) - 3.0)
    return (torch.round(y / step) * step).view(T, nb * 128), torch.where(amax > 0, torch.exp2(e), 0.0)


def _exact_matrix(w, s):
    rows, n = w.shape
    out = w.to(torch.float64)
    i = torch.arange(rows, device=w.device) // 128
    j = torch.arange(n, device=w.device) // 128
    return out * s.to(torch.float64)[i][:, j]


def _exact_moe(s):
    case = s.case
    h = s.h.double()
    xb = h * torch.rsqrt((h * h).mean(1, keepdim=True) + s.eps) * s.norm.double()
    score = xb @ s.router_w.double().T
    if case["router"] == 2:
        p = torch.sigmoid(score)
        pick = p + s.bias.double()
    else:
        p = pick = torch.softmax(score, 1)
    ids = torch.argsort(-pick, dim=1, stable=True)[:, :case["k"]]
    w = p.gather(1, ids)
    if case["router"] == 0:
        w = w / w.sum(1, keepdim=True)
    elif case["router"] == 2:
        w = w / (w.sum(1, keepdim=True) + 1e-20)
    w = w * s.routed_scale

    def ffn(x, g, u, d):
        a = x @ g.T
        return (a * torch.sigmoid(a) * (x @ u.T)) @ d.T

    out = h.clone()
    for e in torch.unique(ids).tolist():
        t, r = torch.where(ids == e)
        mats = [_exact_matrix(m[0][e], m[1][e]) for m in (s.gate, s.up, s.down)]
        out.index_add_(0, t, ffn(xb[t], *mats) * w[t, r, None])
    if s.shared:
        out = out + ffn(xb, *[_exact_matrix(*m) for m in s.shared])
    return out, None, w


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "moe":
        return _exact_moe(s)
    codes, scale = (s.codes.double(), s.scale.double()) if case["kind"] == "matmul" else _exact_codes(s.x)
    if case["kind"] == "quantize":
        return codes, scale
    x = codes * scale.repeat_interleave(128, 1)
    n, rows = case["n"], case["rows"]
    return torch.cat([x[:, :n] @ _exact_matrix(s.w[i:i + 16384], s.ws[i // 128:(i + 16384) // 128]).T
                      for i in range(0, rows, 16384)], 1)
