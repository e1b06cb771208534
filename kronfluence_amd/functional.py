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
First derivatives in reverse mode only: ``create_graph=True``, forward-mode tangents, ``torch.func`` transforms, traces and tensor subclasses
with a dispatch of their own are refused.  Under ``torch.autocast`` they cast as the torch operators do: attention runs
in the autocast dtype, a layer norm returns float32 (reading its input as it is, with no cast in between), an RMS norm its input's dtype.
"""

from __future__ import annotations

from typing import Optional

import torch

from kronfluence_amd import _native as nat

__all__ = ["attention", "layer_norm", "rms_norm"]

_AUTOCAST = (torch.float32, torch.bfloat16, torch.float16)   # what autocast casts: float64 and integers stay, and are refused as outside of it


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, causal: bool = True, scale: Optional[float] = None,
              lengths: Optional[torch.Tensor] = None, cu_seqlens: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``softmax(scale * q k^T + mask) v`` over whole prompts, for every sequence and head.

    ``q``: ``[batch, length, heads, width]``, ``k`` / ``v``: ``[batch, length, kv_heads, width]`` (``heads`` a multiple of
    ``kv_heads``: grouped heads), or -- with ``cu_seqlens`` -- packed rows ``[tokens, heads, width]``.  bfloat16 or float32;
    ``width <= 128``; any strides (a contiguous last axis and 16-byte aligned rows are read in place, others are copied).

    ``lengths`` (``[batch]``, int32 / int64 on the device) counts the real tokens of each row, the first ones; ``cu_seqlens``
    (``[sequences + 1]``, the first row of every sequence and the last one's end, ascending) cuts a packed batch.  Entries are clamped to
    the rows that exist, and an offset below one before it counts as that one (its sequence is empty); neither is read by the host.  A
    token sees the tokens of its own sequence, with ``causal`` those up to itself.

    Rows of no sequence (padding; packed rows in front of the first offset or behind the last) are 0 in the output and in every gradient,
    whatever the inputs hold there.  An infinity or NaN at a REAL token may reach every row of its sequence, as it does in the plain formula (0 * inf); float32
    infinities and values from 3.39e38 on give NaN there, and below 1e-33 the last bits may be lost.
    ``scale`` is positive and ``1 / sqrt(width)`` by default.  A bfloat16 call with a graph keeps, beside q, k, v and the output, 8 bits per
    output element for its backward pass.
    """
    if torch.is_autocast_enabled("cuda") and q.is_cuda:
        dtype = torch.get_autocast_dtype("cuda")
        q, k, v = (t.to(dtype) if t.dtype in _AUTOCAST else t for t in (q, k, v))
    return nat.autograd().attention(q, k, v, bool(causal), scale, lengths, cu_seqlens)


def _norm(x: torch.Tensor, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor], eps: float, centred: bool,
          out_dtype: Optional[torch.dtype]) -> torch.Tensor:
    if out_dtype is None:
        out_dtype = torch.float32 if centred and torch.is_autocast_enabled("cuda") and x.is_cuda else x.dtype
    return nat.autograd().norm(x, weight, bias, eps, centred, out_dtype)


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
    """``x / sqrt(mean(x^2) + eps) * weight`` over the last axis: :func:`layer_norm` without the mean.  ``eps`` defaults to float32's machine
    epsilon for inputs of every dtype, as ``torch.nn.RMSNorm`` takes it on the GPU; ``out_dtype`` to ``x.dtype``."""
    if eps is None:
        eps = torch.finfo(torch.float32).eps
    return _norm(x, weight, None, eps, False, out_dtype)
