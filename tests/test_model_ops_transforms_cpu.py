"""What kronfluence_amd/functional.py cannot carry through a call is refused: tangents of forward-mode differentiation, traces, and the
wrappers of torch.func and of tensor subclasses.  The kernels write into fresh tensors, so a tangent or a node of a trace would be lost
without a word.  Refused before it matters where the tensors live."""

import pytest
import torch
from torch.autograd import forward_ad

from kronfluence_amd import _native as nat
from kronfluence_amd import functional

X, W = torch.randn(3, 8), torch.ones(8)
Q = torch.randn(1, 4, 2, 8)
CALLS = {
    "layer_norm": lambda x: functional.layer_norm(x, W, W), "rms_norm": lambda x: functional.rms_norm(x, W),
    "layer_norm weight": lambda x: functional.layer_norm(X, x[0]), "layer_norm bias": lambda x: functional.layer_norm(X, W, x[0]),
    "attention q": lambda x: functional.attention(x.reshape(1, 3, 1, 8), Q[:, :3, :1], Q[:, :3, :1]),
    "attention k": lambda x: functional.attention(Q[:, :3, :1], x.reshape(1, 3, 1, 8), Q[:, :3, :1]),
    "attention v": lambda x: functional.attention(Q[:, :3, :1], Q[:, :3, :1], x.reshape(1, 3, 1, 8)),
}


@pytest.mark.parametrize("requires_grad", [False, True])
@pytest.mark.parametrize("call", sorted(CALLS))
def test_forward_mode_tangents_are_refused(call, requires_grad):
    with forward_ad.dual_level():
        x = forward_ad.make_dual(X.clone().requires_grad_(requires_grad), torch.ones_like(X))
        with pytest.raises(nat.KfError, match="forward-mode"):
            CALLS[call](x)
    with pytest.raises(nat.KfError, match="lives on cpu"):   # (the same call without a tangent gets further)
        CALLS[call](X)


@pytest.mark.parametrize("call", ["layer_norm", "rms_norm", "attention q"])
def test_traces_are_refused(call):
    from torch.fx.experimental.proxy_tensor import make_fx

    with pytest.raises(nat.KfError, match="trace"):
        torch.jit.trace(CALLS[call], X, check_trace=False)
    with pytest.raises(nat.KfError, match="trace"):
        make_fx(CALLS[call])(X)


@pytest.mark.parametrize("call", ["layer_norm", "rms_norm", "attention q"])
def test_wrapped_tensors_are_refused(call):
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.testing._internal.two_tensor import TwoTensor

    with pytest.raises(nat.KfError, match="plain tensors"):
        torch.func.vmap(CALLS[call])(X[None])
    with pytest.raises(nat.KfError, match="plain tensors"):
        torch.func.grad(lambda x: CALLS[call](x).sum())(X)
    with pytest.raises(nat.KfError, match="plain tensors|forward-mode"):
        torch.func.jvp(CALLS[call], (X,), (X,))
    with pytest.raises(nat.KfError, match="plain tensors"):
        CALLS[call](TwoTensor(X, X))
    with FakeTensorMode(allow_non_fake_inputs=True) as mode, pytest.raises(nat.KfError, match="plain tensors"):
        CALLS[call](mode.from_tensor(X))


def test_subclasses_without_a_dispatch_of_their_own_are_plain():
    class Named(torch.Tensor):
        pass

    with pytest.raises(nat.KfError, match="lives on cpu"):
        functional.layer_norm(X.as_subclass(Named), torch.nn.Parameter(W))
