"""The block operators at the edges of what their documentation allows, as far as that is decided without a GPU."""
import pytest
import torch


def _stacks(experts=3, ff=8, dim=4):
    return torch.ones(experts, ff, dim), torch.ones(experts, ff, dim), torch.ones(experts, dim, ff)


@pytest.mark.parametrize("bad", [dict(activation="relu"), dict(activation="gelu"), dict(activation=None), dict(top_k=0), dict(top_k=4), dict(top_k=-1)])
def test_a_mixture_that_is_not_one_is_refused_when_it_is_made(pkg, bad):
    """Not when it runs: the experts one by one would take any activation for gelu, and any number of places for as many as there are experts."""
    with pytest.raises(ValueError):
        pkg.ops.GGMLMoE(torch.zeros(3, 4), *_stacks(), **{"top_k": 2, **bad})
    layer = pkg.ops.GGMLMoE(torch.zeros(3, 4), *_stacks(), top_k=3, activation="gelu_tanh")
    x = torch.full((2, 4), 0.25)
    torch.testing.assert_close(layer(x), torch.full((2, 4), 8 * float(torch.nn.functional.gelu(torch.tensor(1.0), approximate="tanh"))))
