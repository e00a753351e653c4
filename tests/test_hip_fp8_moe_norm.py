"""The norm of a token in the 8-bit MoE block: its factor belongs to the token's whole vector, so a rounding of
it does not average out as the elements' own roundings do.

What a token's result has in common with the definition's, <y, want> / <want, want> - 1, is therefore to be far
below a float's rounding: x's two roundings, the sums', silu's and the product's are each element's own, at most 16
u = 16 * 2^-24 together, and average to 16 u / sqrt(1024) = u / 2 over the 1024 hidden values; a factor with
the roundings of a mean, a root and a reciprocal is off by 1.5 u on its own and goes into gate and up."""
import pytest
import torch

from tests.test_hip_fp8 import randn, values
from tests.test_hip_fp8_moe import build
from tierlm_amd import fp8

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def definition(c, h):
    h = h.double()
    x = h * torch.rsqrt((h * h).mean(1, keepdim=True) + torch.tensor(1e-6).double().item()) * c.norm.double()
    G, Up, Dn = (values(*m) for m in c.experts[0])
    g = x @ G.T
    return (g * torch.sigmoid(g) * (x @ Up.T)) @ Dn.T


@pytest.mark.parametrize("T", [64, 1])
def test_a_tokens_factor_is_not_rounded(hip, T):
    c, g = build(40, 2048, 1024, 1, 1)
    off = []
    for _ in range(64 // T):
        h = randn(g, T, 2048) * torch.exp(randn(g, T, 1))
        y = c.block(h, out=torch.empty_like(h)).double() - h.double()
        want = definition(c, h)
        off.append((y * want).sum(1) / (want * want).sum(1) - 1)
    rms = torch.cat(off).square().mean().sqrt().item()
    assert rms <= U / 2, rms / U


@pytest.mark.parametrize("size", [1e-30, 1e-12, 1e12, 1e25, 1e30])
def test_sizes_whose_squares_are_no_floats(hip, size):
    """x is of size 1 for a residual of any size (and small where eps is the larger): the router sees it."""
    c, g = build(41, 256, 128, 16, 4)
    h = randn(g, 3, 256) * size
    ids, w = torch.empty(3, 4, dtype=torch.int32, device="cuda"), torch.empty(3, 4, device="cuda")
    out = c.block(h, out=torch.empty_like(h), ids=ids, w=w)
    assert torch.isfinite(out).all()
    x = h.double() * torch.rsqrt(h.double().square().mean(1, keepdim=True) + 1e-6) * c.norm.double()
    l = x @ c.router_w.double().T
    dl = 8 * U * (x.abs() @ c.router_w.double().abs().T).max().item() + 2.0 ** -120
    best = l.sort(1, descending=True)[0][:, :4]
    assert ((l.gather(1, ids.long()) - best).abs() <= 2 * dl).all()
    p = torch.softmax(l, 1).gather(1, ids.long())
    want = p / p.sum(1, keepdim=True)
    assert ((w.double() - want).abs() <= want * (4 * dl + 8 * U)).all()
