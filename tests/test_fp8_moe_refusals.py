"""The 8-bit MoE block refuses matrices that are not there, misaligned or of another kind, before it
looks at a device (no GPU here)."""
import ctypes as C

import pytest
import torch

from tests.test_fp8_refusals import EINVAL, desc, moe
from tierlm_amd import fp8, lib

E, D, DE, DS = 4, 128, 64, 16


def block(mask=None, ptrs=None, **kw):
    ptrs = [1 << 20] * (3 * E) if ptrs is None else ptrs
    return fp8.MoeBlock(D=D, de=DE, E=E, k=2, ffn_norm=torch.ones(D), router_w=torch.zeros(E, D), expert_ptrs=ptrs,
                        mask=None if mask is None else torch.tensor(mask, dtype=torch.uint8), **kw)


@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("mask", [None, [0, 0, 0, 0], [1, 1, 0, 1]])
def test_a_missing_matrix_of_an_expert_that_may_be_chosen(which, mask):
    ptrs = [1 << 20] * (3 * E)
    ptrs[3 * 2 + which] = 0
    with pytest.raises(ValueError, match="only for experts that the mask prunes"):
        block(mask, ptrs)


def test_a_missing_matrix_of_a_pruned_expert_is_let_through():
    with pytest.raises(ValueError, match="not on the current HIP device"):      # the next check
        block([0, 0, 1, 0], [0 if i // 3 == 2 else 1 << 20 for i in range(3 * E)])


def test_misaligned_experts():
    with pytest.raises(ValueError, match="16-byte aligned"):
        block(ptrs=[1 << 20] * (3 * E - 1) + [(1 << 20) + 8])


def test_shared_matrices():
    good = [torch.zeros(fp8.packed_bytes(r, n), dtype=torch.uint8) for r, n in ((DS, D), (DS, D), (D, DS))]
    odd = torch.zeros(good[0].numel() + 16, dtype=torch.uint8)
    for bad in (good[0][:-1], good[0].view(torch.int8), torch.zeros(2 * good[0].numel(), dtype=torch.uint8)[::2],
                odd[odd.data_ptr() % 16 + 8:][:good[0].numel()]):
        with pytest.raises(ValueError, match="3 packed matrices"):
            block(ds=DS, shared=[bad, good[1], good[2]])
    with pytest.raises(ValueError, match="3 packed matrices"):
        block(ds=DS, shared=good[:2])
    with pytest.raises(ValueError, match="not on the current HIP device"):
        block(ds=DS, shared=good)


def test_c_entry():
    P = 1 << 20
    assert moe(desc(experts=P + 4)) == EINVAL
    for m in ("sg", "su", "sd"):
        assert moe(desc(**{**dict(ds=64, sg=P, su=P, sd=P), m: P + 8})) == EINVAL
    assert b"16-byte" in lib.tlm_hip_errmsg()
    assert lib.tlm_hip_fp8_moe_workspace_bytes(C.byref(desc(ds=64)), 1) > 0
