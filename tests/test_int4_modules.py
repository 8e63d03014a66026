"""CPU checks of the linear modules on 4-bit weights: refusals that come before a launch."""
import pytest
import torch
from torch.autograd import forward_ad

from pdscope_amd import ops
from pdscope_amd.hf import Int4Linear, install_int4_linears


def module(N=16, K=128, G=64):
    return Int4Linear(ops.Int4Weight(torch.zeros(ops.int4_bytes(N, K, G), dtype=torch.uint8), N, K, G, False))


def test_no_gradient_of_either_mode():
    q, x = module(), torch.zeros((2, 128), dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="no gradient"):
        q(x.clone().requires_grad_())
    for grad in (True, False):  # no_grad() does not leave tangents out
        with torch.set_grad_enabled(grad), forward_ad.dual_level():
            with pytest.raises(RuntimeError, match="no gradient"):
                q(forward_ad.make_dual(x, torch.ones_like(x)))
            with pytest.raises(ValueError, match="on the GPU"):  # as without a level: its own refusal
                q(x)


def test_a_model_that_is_a_linear_module_itself_is_refused():
    """No parent holds it, so nothing could be replaced."""
    with pytest.raises(ValueError, match="itself"):
        install_int4_linears(torch.nn.Linear(128, 48), 64)


@pytest.mark.parametrize("group", [0, -64, 16, 48, 256])
def test_groups_that_a_matrix_cannot_have(group):
    """Before any module is looked at: a model without linear modules has its answer too."""
    for model in (torch.nn.Sequential(torch.nn.Linear(768, 48)), torch.nn.Sequential()):
        with pytest.raises(ValueError, match="32, 64 or 128"):
            install_int4_linears(model, group)
