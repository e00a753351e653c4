"""Experts without matrices in the 8-bit MoE block: they are never chosen, whatever the mask says by the time
of the call, on each way through the launches."""
import pytest
import torch

from tests.test_hip_fp8 import randn
from tests.test_hip_fp8_moe import build
from tierlm_amd import fp8

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("router", [0, 1, 2])
@pytest.mark.parametrize("T", [1, 3, 40])       # one token; routed in gate/up; routed before it, every expert
def test_experts_without_matrices_stay_pruned(hip, T, router):
    mask = torch.zeros(16, dtype=torch.bool)
    mask[[0, 3, 7, 15]] = True
    c, g = build(20 + T, 256, 128, 16, 4, router=router, mask=mask)
    m = mask.to("cuda", torch.uint8)
    ptrs = [0 if mask[e] else p.data_ptr() for e, ex in enumerate(c.packed) for p in ex]
    block = fp8.MoeBlock(D=256, de=128, E=16, k=4, ffn_norm=c.norm, router_w=c.router_w, expert_ptrs=ptrs, mask=m,
                         router=router, router_bias=c.bias)
    h = randn(g, T, 256)
    want, ids, w = c.block(h, out=torch.empty_like(h)), *(torch.empty(T, 4, dtype=t, device="cuda")
                                                          for t in (torch.int32, torch.float32))
    for change in (lambda: None, lambda: m.zero_(), lambda: setattr(block.desc, "mask", None)):
        change()
        out = block(h, out=torch.empty_like(h), ids=ids, w=w)
        assert not torch.isin(ids.cpu(), torch.tensor([0, 3, 7, 15], dtype=torch.int32)).any()
        assert torch.equal(out, want)


@pytest.mark.parametrize("which", [0, 1, 2])
def test_one_matrix_missing_is_enough(hip, which):
    """The table is the caller's in C: any of the three pointers null prunes the expert, all experts' leaves h."""
    c, g = build(30 + which, 256, 128, 8, 2)
    for T in (1, 5, 30):
        h = randn(g, T, 256)
        ids = torch.empty(T, 2, dtype=torch.int32, device="cuda")
        keep = c.block.table.clone()
        c.block.table[3 * 4 + which] = 0
        out = c.block(h, out=torch.empty_like(h), ids=ids)
        assert not (ids == 4).any() and torch.isfinite(out).all()
        c.block.table[which::3] = 0
        out = c.block(h, out=torch.empty_like(h), ids=ids)
        assert (ids == -1).all() and torch.equal(out, h)
        c.block.table.copy_(keep)
