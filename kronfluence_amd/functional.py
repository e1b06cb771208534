"""Differentiable operators for the MODEL's own forward and backward passes.

Every stage runs the user's model over the data between the tracked layers; these are the parts of a transformer that sit there --
attention and the norms -- on the HIP kernels of ``libkronfluence_hip.so``, forward and backward.  They take what the torch calls
they stand in for take, except that heads are an axis (``[batch, length, heads, width]``: a reshape of the projection's output, no
transposed copy) and that grouped key / value heads, padded and packed batches need neither repeated heads nor a mask tensor:

>>> from kronfluence_amd import functional
>>> q, k, v = self.c_attn(h).view(b, t, 3, heads, width).unbind(2)        # slices: read in place
>>> y = functional.attention(q, k, v, causal=True).flatten(2)              # out, [b, t, heads * width]
>>> h = functional.layer_norm(x, self.ln.weight, self.ln.bias, eps=self.ln.eps)

Like the rest of the package they raise ``KfError`` for tensors that are not on an MI355X and for arguments the kernels do not take.
First derivatives only.  Under ``torch.autocast`` they cast as the torch operators do: attention runs in the autocast dtype, a norm
returns float32 (reading its input as it is, with no cast in between).
"""

from __future__ import annotations

import math
from typing import Optional

import torch
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from kronfluence_amd import ops

__all__ = ["attention", "layer_norm", "rms_norm"]


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lengths, cu_seqlens, causal, scale):
        out, lse = ops.attention_forward(q, k, v, causal, scale, lengths, cu_seqlens)
        ctx.save_for_backward(q, k, v, out, lse, lengths, cu_seqlens)
        ctx.causal, ctx.scale = causal, scale
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        q, k, v, out, lse, lengths, cu_seqlens = ctx.saved_tensors
        dq, dk, dv = ops.attention_backward(grad, out, lse, q, k, v, ctx.causal, ctx.scale, lengths, cu_seqlens)
        return dq, dk, dv, None, None, None, None


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, causal: bool = True, scale: Optional[float] = None,
              lengths: Optional[torch.Tensor] = None, cu_seqlens: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``softmax(scale * q k^T + mask) v`` over whole prompts, for every sequence and head.

    ``q``: ``[batch, length, heads, width]``, ``k`` / ``v``: ``[batch, length, kv_heads, width]`` (``heads`` a multiple of
    ``kv_heads``: grouped heads), or -- with ``cu_seqlens`` -- packed rows ``[tokens, heads, width]``.  bfloat16 or float32;
    ``width <= 128``; any strides (a contiguous last axis and 16-byte aligned rows are read in place, others are copied).

    ``lengths`` (``[batch]``, int32 / int64 on the device) counts the real tokens of each row, the first ones; ``cu_seqlens``
    (``[sequences + 1]``, the first row of every sequence, ascending from 0) cuts a packed batch.  Entries are clamped to the rows
    that exist; neither is read by the host.  A token sees the tokens of its own sequence, with ``causal`` those up to itself.

    Rows of no sequence (padding; packed rows behind the last offset) are 0 in the output and in every gradient, whatever the inputs
    hold there.  An infinity or NaN at a REAL token may reach every row of its sequence, as it does in the plain formula (0 * inf).
    ``scale`` is positive and ``1 / sqrt(width)`` by default.
    """
    if torch.is_autocast_enabled("cuda") and q.is_cuda:
        dtype = torch.get_autocast_dtype("cuda")
        q, k, v = q.to(dtype), k.to(dtype), v.to(dtype)
    width = q.shape[-1] if q.dim() else 0
    scale = 1.0 / math.sqrt(max(width, 1)) if scale is None else float(scale)
    whole = 16 // q.element_size()
    pad = -width % whole if 0 < width <= ops.ATTENTION_MAX_WIDTH else 0
    if pad and k.dim() == v.dim() == q.dim() and k.shape[-1] == v.shape[-1] == width:   # zero columns change no product
        q, k, v = (F.pad(t, (0, pad)) for t in (q, k, v))
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        out = _Attention.apply(q, k, v, lengths, cu_seqlens, bool(causal), scale)
    else:
        out = ops.attention_forward(q, k, v, bool(causal), scale, lengths, cu_seqlens, with_lse=False)[0]
    return out[..., :width] if pad else out


class _Norm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, centred, out_dtype):
        out, stats = ops.norm_forward(x, weight, bias, eps, centred, out_dtype)
        ctx.save_for_backward(x, weight, stats)
        ctx.centred, ctx.bias_dtype = centred, None if bias is None else bias.dtype
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, weight, stats = ctx.saved_tensors
        with_x, with_weight, with_bias = ctx.needs_input_grad[:3]
        dx, dweight, dbias = ops.norm_backward(grad, x, stats, weight, ctx.centred, with_input=with_x,
                                               weight_dtype=weight.dtype if with_weight else None,
                                               bias_dtype=ctx.bias_dtype if with_bias else None)
        return dx, dweight, dbias, None, None, None


def _norm(x: torch.Tensor, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor], eps: float, centred: bool,
          out_dtype: Optional[torch.dtype]) -> torch.Tensor:
    if out_dtype is None:
        out_dtype = torch.float32 if torch.is_autocast_enabled("cuda") and x.is_cuda else x.dtype
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias)):
        return _Norm.apply(x, weight, bias, float(eps), centred, out_dtype)
    return ops.norm_forward(x, weight, bias, float(eps), centred, out_dtype, with_stats=False)[0]


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, *, eps: float = 1e-5,
               out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last axis, of any width.

    ``x``: float32, bfloat16 or float16, rows at any stride; ``weight`` / ``bias``: vectors of one dtype of the three (not necessarily
    ``x``'s), or ``None``.  ``out_dtype`` defaults to ``x.dtype`` (float32 under autocast).  Statistics, sums and the gradients of
    ``weight`` and ``bias`` are accumulated in float32 in a fixed order; frozen vectors cost nothing in the backward pass.
    """
    return _norm(x, weight, bias, eps, True, out_dtype)


def rms_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, *, eps: Optional[float] = None,
             out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``x / sqrt(mean(x^2) + eps) * weight`` over the last axis: :func:`layer_norm` without the mean.  ``eps`` defaults to the machine
    epsilon of ``x.dtype``, as in ``torch.nn.RMSNorm``."""
    return _norm(x, weight, None, torch.finfo(x.dtype).eps if eps is None else eps, False, out_dtype)
