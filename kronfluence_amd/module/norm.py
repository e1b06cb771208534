"""``nn.LayerNorm`` / ``nn.RMSNorm`` on the HIP kernels (``kronfluence_amd.functional``): the same parameters, names and state dict.

Norms are not tracked (the reference tracks ``nn.Linear`` and ``nn.Conv2d`` only); these modules make the MODEL's own passes
between the tracked layers cheaper.  ``kronfluence_amd.utils.model.apply_fused_norms`` installs them.
"""

from __future__ import annotations

from torch import nn

from kronfluence_amd import functional


class FusedLayerNorm(nn.LayerNorm):
    """``nn.LayerNorm`` over one axis."""

    def forward(self, x):
        return functional.layer_norm(x, self.weight, self.bias, eps=self.eps)


class FusedRMSNorm(nn.RMSNorm):
    """``nn.RMSNorm`` over one axis."""

    def forward(self, x):
        return functional.rms_norm(x, self.weight, eps=self.eps)


def fused(module: nn.Module):
    """The fused counterpart of ``module``, sharing its parameters; ``None`` if it has none (another class, a subclass with a forward
    of its own, several axes) or if the module carries hooks, which would be lost."""
    kinds = {nn.LayerNorm: FusedLayerNorm, nn.RMSNorm: FusedRMSNorm}
    kind = kinds.get(type(module))
    if kind is None or len(module.normalized_shape) != 1:
        return None
    if module._forward_hooks or module._forward_pre_hooks or module._backward_hooks or module._backward_pre_hooks:
        return None
    other = kind(module.normalized_shape, eps=module.eps, elementwise_affine=False)
    other.elementwise_affine = module.elementwise_affine
    for name, parameter in module._parameters.items():
        other.register_parameter(name, parameter)
    other.train(module.training)
    return other
