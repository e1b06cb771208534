"""Forward over reverse through kronfluence_amd/functional.py (see tests/test_model_ops_transforms_cpu.py)."""

import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu


def test_a_tangent_of_the_incoming_gradient_is_refused():
    """The backward kernels would drop it."""
    from kronfluence_amd import functional

    x = torch.randn(3, 64, device="cuda", requires_grad=True)
    for y in (functional.layer_norm(x), functional.rms_norm(x), functional.attention(*[x.view(1, 3, 1, 64)] * 3)):
        with forward_ad.dual_level():
            g = forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y))
            with pytest.raises(Exception, match="forward-mode"):
                torch.autograd.grad(y, x, g)
