"""A token with a NaN or an infinity in the 8-bit MoE block gives NaN; every other token keeps its bits, before and
behind it in the experts' lists, on each way through the launches."""
import pytest
import torch

from tests.test_hip_fp8 import randn
from tests.test_hip_fp8_moe import build

pytestmark = pytest.mark.gpu

# (D, de, E, k, ds, T)
WAYS = {"routed in gate/up, down per token": (256, 128, 16, 4, 128, 7),
        "routed in gate/up, down per expert": (4096, 512, 16, 4, 0, 14),
        "routed before, down per token": (256, 128, 16, 4, 128, 20),
        "routed before, down per expert": (256, 128, 16, 4, 128, 40),
        "fewer choices than experts": (512, 256, 64, 2, 0, 9)}


@pytest.mark.parametrize("router", [0, 1, 2])
@pytest.mark.parametrize("bad", ["nan", "inf"])
@pytest.mark.parametrize("way", WAYS)
def test_the_others_keep_their_bits(hip, way, bad, router):
    D, de, E, k, ds, T = WAYS[way]
    c, g = build(60 + T, D, de, E, k, ds, router=router, gate=ds > 0)
    h = randn(g, T, D)
    h[T // 3] = h[0]                                       # two tokens with the same lists
    want_ids, want_w = torch.empty(T, k, dtype=torch.int32, device="cuda"), torch.empty(T, k, device="cuda")
    want = c.block(h, out=torch.empty_like(h), ids=want_ids, w=want_w)
    assert torch.isfinite(want).all() and torch.equal(want[0], want[T // 3])
    for t in (0, T // 2, T - 1):
        x = h.clone()
        x[t, 5] = float(bad)
        ids, w = torch.empty_like(want_ids), torch.empty_like(want_w)
        out = c.block(x, out=torch.empty_like(h), ids=ids, w=w)
        others = torch.arange(T, device="cuda") != t
        assert torch.isnan(out[t]).all()
        assert torch.equal(out[others], want[others])
        assert torch.equal(ids[others], want_ids[others]) and torch.equal(w[others], want_w[others])


def test_one_token(hip):
    c, g = build(61, 256, 128, 16, 4, 128)
    h = randn(g, 256)
    keep = c.block(h, out=torch.empty_like(h))
    for bad in ("nan", "inf", "-inf"):
        x = h.clone()
        x[255] = float(bad)
        assert torch.isnan(c.block(x, out=torch.empty_like(h))).all()
    assert torch.equal(c.block(h, out=torch.empty_like(h)), keep)      # nothing of it stays in the workspace
