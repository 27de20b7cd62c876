"""The block operators (norms, int8, moe and their layers) at the edges of what their documentation allows."""
import pytest
import torch

from test_gpu_moe import Stack, U

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


# ---- the router

@pytest.mark.parametrize("experts", [9, 40])                    # one launch, and two
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("wide", [False, True])
def test_one_score_that_is_no_number(pkg, experts, renormalize, wide):
    """softmax over scores of which one is NaN or +inf has no number in it: all of the token's weights are NaN, also where that expert is not among the chosen."""
    g = torch.Generator(device=DEV)
    g.manual_seed(91)
    x = torch.randn(3, 64, device=DEV, generator=g).bfloat16()
    w = torch.randn(experts, 64, device=DEV, generator=g).to(torch.float32 if wide else torch.bfloat16)
    x[1, 5], x[2, 5] = 0.0, 0.0
    x[1, 6] = x[1, 7] = 1.0
    bad = w.clone()
    bad[2, 5] = float("nan")                                    # NaN times 0 is NaN too
    ids, weights = pkg.moe.route(x, bad, 6, renormalize=renormalize)
    assert bool(weights.isnan().all())
    assert not bool((ids == 2).any())                           # it comes last
    bad = w.clone()
    bad[2, 6], bad[2, 7] = float("inf"), float("-inf")          # inf - inf: one token's score only, where both meet the same sign
    ids, weights = pkg.moe.route(x[1:2], bad, 6, renormalize=renormalize)
    assert bool(weights.isnan().all()) and not bool((ids == 2).any())
    bad[2, 7] = w[2, 7]
    ids, weights = pkg.moe.route(x[1:2], bad, 6, renormalize=renormalize)          # +inf
    assert int(ids[0, 0]) == 2 and bool(weights.isnan().all())
    bad[2, 6] = float("-inf")                                   # -inf: probability 0, the others as without it
    ids, weights = pkg.moe.route(x[1:2], bad, 6, renormalize=renormalize)
    rest = torch.cat((w[:2], w[3:]))
    same, share = pkg.moe.route(x[1:2], rest, 6, renormalize=renormalize)
    assert torch.equal(ids, same + (same >= 2).int()) and bool((weights - share).abs().max() <= 2 * U)


def test_a_layer_whose_router_holds_a_nan(pkg):
    """NaN through the kernels and through the experts one by one alike."""
    g = torch.Generator(device=DEV)
    g.manual_seed(92)
    gate, up, down = (Stack(pkg, "Q8_0", s, "bf16", 3 + i, shrink=0.25).tensor for i, s in enumerate(((6, 64, 64), (6, 64, 64), (6, 64, 64))))
    router = torch.randn(6, 64, device=DEV, generator=g)
    router[4, 3] = float("nan")
    x = torch.randn(65, 64, device=DEV, generator=g).bfloat16()
    layer = pkg.ops.GGMLMoE(router, gate, up, down, top_k=2)
    assert bool(layer(x[:64]).isnan().all()) and bool(layer(x).isnan().all())
