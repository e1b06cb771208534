"""Refusals of kronfluence_amd/functional.py and of the C entries behind it: no GPU is needed to refuse a call (what a call asks for
is checked before where its tensors live)."""

import ctypes

import pytest
import torch

from kronfluence_amd import _native as nat
from kronfluence_amd import functional

BF16 = torch.bfloat16


def test_tensors_off_the_gpu_are_refused():
    q = torch.zeros(1, 4, 2, 64, dtype=BF16)
    with pytest.raises(nat.KfError, match="lives on cpu"):
        functional.attention(q, q, q)
    with pytest.raises(nat.KfError, match="lives on cpu"):
        functional.layer_norm(torch.zeros(2, 8))
    with pytest.raises(nat.KfError, match="lives on cpu"):
        functional.rms_norm(torch.zeros(2, 8), torch.ones(8))


def heads(*shape, dtype=BF16):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("change,message", [
    (dict(q=heads(1, 4, 2, 64, dtype=torch.float16), k=heads(1, 4, 2, 64, dtype=torch.float16), v=heads(1, 4, 2, 64, dtype=torch.float16)), "bfloat16 or float32"),
    (dict(k=heads(1, 4, 2, 64, dtype=torch.float32)), "one dtype"),
    (dict(k=heads(1, 5, 2, 64)), "shape of q"),
    (dict(v=heads(1, 4, 1, 64)), "shape of q"),
    (dict(v=heads(1, 4, 2, 32)), "shape of q"),
    (dict(k=heads(1, 4, 3, 64), v=heads(1, 4, 3, 64)), "multiple"),
    (dict(k=heads(1, 4, 0, 64), v=heads(1, 4, 0, 64)), "multiple"),
    (dict(q=heads(1, 4, 2, 136), k=heads(1, 4, 2, 136), v=heads(1, 4, 2, 136)), "widths up to 128"),
    (dict(q=heads(1, 4, 2, 0), k=heads(1, 4, 2, 0), v=heads(1, 4, 2, 0)), "widths up to 128"),
    (dict(q=heads(4, 2, 64), k=heads(4, 2, 64), v=heads(4, 2, 64)), r"\[batch, length, heads, width\]"),
    (dict(cu_seqlens=torch.tensor([0, 4], dtype=torch.int32)), r"\[tokens, heads, width\]"),
    (dict(cu_seqlens=torch.tensor([0, 4], dtype=torch.int32), lengths=torch.tensor([4], dtype=torch.int32)), "exclude"),
    (dict(lengths=torch.tensor([4, 4], dtype=torch.int32)), "one entry per row"),
    (dict(lengths=torch.tensor([4.0])), "int32 or int64"),
    (dict(lengths=torch.tensor([[4]])), "vector"),
    (dict(scale=0.0), "positive"), (dict(scale=-1.0), "positive"), (dict(scale=float("inf")), "positive"), (dict(scale=float("nan")), "positive"),
])
def test_attention_refuses(change, message):
    call = dict(q=heads(1, 4, 2, 64), k=heads(1, 4, 2, 64), v=heads(1, 4, 2, 64))
    call.update(change)
    with pytest.raises(nat.KfError, match=message):
        functional.attention(**call)


def test_attention_packed_refuses_an_empty_offset_vector():
    q = heads(4, 2, 64)
    with pytest.raises(nat.KfError, match="cu_seqlens"):
        functional.attention(q, q, q, cu_seqlens=torch.zeros(0, dtype=torch.int32))


@pytest.mark.parametrize("change,message", [
    (dict(x=torch.zeros(2, 8, dtype=torch.float64)), "float32, bfloat16 or float16"),
    (dict(x=torch.zeros(2, 8, dtype=torch.int64)), "float32, bfloat16 or float16"),
    (dict(x=torch.zeros(())), "last axis"),
    (dict(x=torch.zeros(2, 0)), "last axis"),
    (dict(weight=torch.ones(7)), "vector of x's width"),
    (dict(weight=torch.ones(1, 8)), "vector of x's width"),
    (dict(weight=torch.ones(8), bias=torch.ones(8, dtype=BF16)), "one of the dtypes"),
    (dict(weight=torch.ones(8, dtype=torch.float64)), "one of the dtypes"),
    (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
    (dict(out_dtype=torch.float64), "return float32"),
])
def test_norms_refuse(change, message):
    call = dict(x=torch.zeros(2, 8))
    call.update(change)
    with pytest.raises(nat.KfError, match=message):
        functional.layer_norm(**call)
    if "bias" not in call:
        with pytest.raises(nat.KfError, match=message):
            functional.rms_norm(**call)


def view(width=64, heads=2, pointer=1 << 20):
    return nat.kf_heads_view(pointer, 4 * heads * width, heads * width, width)


def test_c_entries_refuse_without_touching_memory():
    """Bad sizes, types, alignments and workspaces come back as status codes; no pointer is read and nothing is launched."""
    lib, ok = nat.lib(), view()
    INVALID, DTYPE, WORKSPACE = -1, -2, -4

    def forward(out=ok, q=ok, k=ok, v=ok, dtype=nat.KF_BF16, sequences=1, length=4, rows=4, heads=2, kv_heads=2, width=64, lengths=None,
                offsets=None, order=None, scale=1.0):
        return lib.kf_attention_forward(out, None, q, k, v, dtype, sequences, length, rows, heads, kv_heads, width, lengths, offsets, order, 1, scale, None)

    assert forward(dtype=nat.KF_F16) == DTYPE
    for bad in (dict(width=136), dict(width=0), dict(width=60), dict(heads=3), dict(kv_heads=0), dict(rows=5), dict(length=0), dict(sequences=0),
                dict(scale=0.0), dict(scale=float("nan")), dict(lengths=16, offsets=16), dict(order=16), dict(rows=1 << 31, length=1 << 31),
                dict(sequences=1 << 40, length=1, rows=1 << 40), dict(q=view(pointer=(1 << 20) + 8)), dict(k=view(width=63)), dict(out=view(pointer=0)),
                dict(heads=1 << 40, kv_heads=1)):
        assert forward(**bad) == INVALID, bad

    def backward(bytes_=4 * 2 * 4, workspace=1 << 20, lse=1 << 20, **kw):
        views = [kw.pop("dq", ok)] + [ok] * 4
        return lib.kf_attention_backward(*views, lse, ok, ok, ok, nat.KF_BF16, 1, 4, kw.get("rows", 4), 2, 2, 64, None, None, None, 1, 1.0, workspace, bytes_, None)

    assert lib.kf_attention_backward_workspace_bytes(1, 4, 4, 2, 2, 64, 0, 1) == 4 * 2 * 4
    assert backward(bytes_=31) == WORKSPACE and backward(workspace=None) == WORKSPACE
    assert backward(lse=None) == INVALID and backward(dq=view(pointer=4)) == INVALID and backward(rows=3) == INVALID

    assert lib.kf_attention_order_bytes(3, 100, 4) == 0            # everything fits the card at once
    assert lib.kf_attention_order_bytes(24, 12011, 16) == 4 * (12011 // 128 + 25)
    assert lib.kf_attention_order_bytes(1 << 20, 1 << 28, 8) == 0    # too many to order, and enough to even out
    for bad in ((None, 16, 2, 8), (16, None, 2, 8), (16, 16, 0, 8), (16, 16, 2, 0), (16, 16, 1 << 20, 1 << 28)):
        assert lib.kf_attention_order(*bad, 1, None) == INVALID, bad

    def norm(y=1 << 20, y_dtype=0, x=1 << 20, x_dtype=0, rows=2, width=8, stride=8, weight=None, w_dtype=0, eps=1e-5):
        return lib.kf_norm_forward(y, y_dtype, None, x, x_dtype, rows, width, stride, weight, None, w_dtype, 1, eps, None)

    assert norm(y_dtype=nat.KF_F64) == DTYPE and norm(x_dtype=nat.KF_I32) == DTYPE and norm(weight=16, w_dtype=nat.KF_F64) == DTYPE
    for bad in (dict(y=None), dict(x=None), dict(rows=0), dict(width=0), dict(stride=-1), dict(eps=-1.0), dict(eps=float("inf"))):
        assert norm(**bad) == INVALID, bad

    def norm_backward(dx=None, dw=None, db=None, grad=1 << 20, stats=1 << 20, workspace=None, bytes_=0, w_dtype=0):
        return lib.kf_norm_backward(dx, dw, db, grad, 0, 1 << 20, 0, stats, 2, 8, 8, None, w_dtype, 1, workspace, bytes_, None)

    assert norm_backward() == 0   # nothing is asked for
    assert norm_backward(dw=16) == WORKSPACE and norm_backward(db=16, workspace=16, bytes_=8) == WORKSPACE
    assert norm_backward(dx=16, grad=None) == INVALID and norm_backward(dx=16, stats=None) == INVALID and norm_backward(dw=16, w_dtype=3) == DTYPE
    assert lib.kf_norm_backward_workspace_bytes(2, 8) >= 2 * 8 * 4
    assert ctypes.sizeof(nat.kf_heads_view) == 32


def test_apply_fused_norms_shares_parameters_and_names():
    from torch import nn

    from kronfluence_amd.module.norm import FusedLayerNorm, FusedRMSNorm
    from kronfluence_amd.utils.model import apply_fused_norms

    class Own(nn.LayerNorm):
        def forward(self, x):
            return super().forward(x) + 1

    class Model(nn.Module):
        def __init__(self):
            super().__init__()
            self.a, self.b, self.c = nn.LayerNorm(8, eps=1e-3), nn.RMSNorm(8), nn.LayerNorm(8, bias=False)
            self.d, self.e, self.f = nn.LayerNorm(8, elementwise_affine=False), nn.LayerNorm((2, 8)), Own(8)
            self.again, self.hooked = self.a, nn.LayerNorm(8)
            self.nest = nn.Sequential(nn.Linear(8, 8), nn.RMSNorm(8, eps=1e-4))

    model = Model()
    model.hooked.register_forward_hook(lambda *_: None)
    model.b.weight.requires_grad_(False)
    before, kept = dict(model.named_parameters()), list(model.state_dict())
    model.eval()
    assert apply_fused_norms(model) is model
    after = dict(model.named_parameters())
    assert set(after) == set(before) and all(after[name] is before[name] for name in before) and list(model.state_dict()) == kept
    assert type(model.a) is type(model.again) is type(model.c) is type(model.d) is FusedLayerNorm and model.a.eps == 1e-3
    assert type(model.b) is type(model.nest[1]) is FusedRMSNorm and model.b.eps is None and model.nest[1].eps == 1e-4
    assert type(model.e) is type(model.hooked) is nn.LayerNorm and type(model.f) is Own and not model.a.training
    assert model.c.bias is None and model.d.weight is None
    assert type(apply_fused_norms(nn.LayerNorm(4))) is FusedLayerNorm
    apply_fused_norms(model)
    assert type(model.a) is FusedLayerNorm and list(model.state_dict()) == kept
    with pytest.raises(nat.KfError, match="lives on cpu"):   # no CPU path, as everywhere in the package
        model.a(torch.zeros(2, 8))
