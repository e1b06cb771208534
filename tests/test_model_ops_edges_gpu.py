"""Attention (kronfluence_amd/functional.py) where it is most easily wrong: rows of no sequence, rows whose softmax is peaked, batches that
take the split or the dealt-out paths.  Bounds are those of tests/test_model_ops_gpu.py with a tighter one for D in bf16:

D is the product of do with an output that carries the next eight bits (a unit of them is 2^-8 of a bf16 step, 2^-15 |out| at most; rounded
to half a unit, or to a whole one beside the tie that the signed byte does not reach: 2 U^2 |out|) and that the ROUNDED p sum to one in:
out = sum_j p_j (1 + e_j) v_j / (1 + sum_k p_k e_k), |e_j| <= U, so that to first order
    D - D_exact = sum_j p_j (e_j - sum_k p_k e_k) dp_j = sum_j e_j p_j (dp_j - D_exact) = sum_j e_j ds_j
-- at most U sum |ds_j| (and ep sum |ds_j| from p's own fp32 errors), however far do . out is above the gradients.  Beside it stand the fp32
sums: (n + 16) E sum |do| (p |v|) and (2 width + 4) E sum |do| |out|."""

import math

import pytest
import torch
from test_model_ops_gpu import BF16, E, F32, HALF, close, make

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def functional():
    from kronfluence_amd import functional

    return functional


def expected(q, k, v, g, causal, exact_rows=0):
    """Values and bounds of one sequence and one kv head (``q``, ``g`` [n, group, width]; ``k``, ``v`` [n, width]): out, dq, dk, dv.  The first
    ``exact_rows`` rows take D from p and dp in fp32."""
    dtype = q.dtype
    U, Up = HALF[dtype], HALF[dtype] if dtype == BF16 else 0.0
    q, k, v, g = (t.double().transpose(0, 1) if t.dim() == 3 else t.double()[None] for t in (q, k, v, g))
    group, n, width = q.shape
    scale = 1.0 / math.sqrt(width)
    s = scale * q @ k.transpose(1, 2)
    if causal:
        s = s.masked_fill(~torch.ones(n, n, dtype=torch.bool, device=s.device).tril(), -math.inf)
    p = torch.softmax(s, dim=-1)
    ep = (width + 8) * E * float((scale * q.abs() @ k.abs().transpose(1, 2)).max()) + (n + 16) * E
    out, dp = p @ v, g @ v.transpose(1, 2)
    delta = (p * dp).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    gv = g.abs() @ v.abs().transpose(1, 2)
    if dtype == BF16:    # p_j (e_j - mean e) v_j = e_j p_j (v_j - out)
        err_out = (ep + Up) * ((p @ v.abs()) + out.abs()) + n * E * (p @ v.abs()) + U * out.abs()
        err_delta = ((ep + U) * (1 + 2 * U) * ds.abs().sum(-1, keepdim=True) + (n + 16) * E * (p * gv).sum(-1, keepdim=True)
                     + (2 * U * U + (2 * width + 4) * E) * (g.abs() * out.abs()).sum(-1, keepdim=True))
    else:
        err_out = (ep + n * E) * (p @ v.abs()) + U * out.abs()
        err_delta = (g.abs() * err_out).sum(-1, keepdim=True) + (width + 2) * E * (g.abs() * out.abs()).sum(-1, keepdim=True)
    if exact_rows:
        few = (p * ((ep + (n + 4) * E) * dp.abs() + (width + 2) * E * gv)).sum(-1, keepdim=True)
        err_delta = torch.where(torch.arange(n, device=s.device)[:, None] < exact_rows, few, err_delta)
    err_ds = (ep + 2 * E + Up + (n + 2) * E) * ds.abs() + p * (err_delta + (width + 2) * E * gv) + E * p * (dp.abs() + delta.abs())
    dq, dk, dv = scale * ds @ k, (scale * ds.transpose(1, 2) @ q).sum(0), (p.transpose(1, 2) @ g).sum(0)
    err_dq = scale * err_ds @ k.abs() + U * dq.abs()
    err_dk = (scale * err_ds.transpose(1, 2) @ q.abs()).sum(0) + group * n * E * (scale * ds.abs().transpose(1, 2) @ q.abs()).sum(0) + U * dk.abs()
    err_dv = ((ep + Up + (group * n + 2) * E) * (p.transpose(1, 2) @ g.abs())).sum(0) + U * dv.abs()
    last = lambda t: t.transpose(0, 1)
    return (last(out), last(err_out)), (last(dq), last(err_dq)), (dk, err_dk), (dv, err_dv)


def passes(functional, q, k, v, g, causal, **batch):
    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    out = functional.attention(q, k, v, causal=causal, **batch)
    return (out.detach(),) + torch.autograd.grad(out, (q, k, v), g)


def check(functional, q, k, v, g, causal, spans, exact_rows=0, **batch):
    """Every sequence against 64 bits; rows outside all of ``spans`` are 0."""
    got = passes(functional, q, k, v, g, causal, **batch)
    group = q.shape[-2] // k.shape[-2]
    want = [torch.zeros(t.shape, dtype=torch.float64, device=t.device) for t in (q, q, k, v)]
    bound = [torch.zeros_like(w) for w in want]
    for span in spans:
        for h in range(k.shape[-2]):
            of = slice(h * group, (h + 1) * group)
            for i, (value, error) in enumerate(expected(q[span][:, of], k[span][:, h], v[span][:, h], g[span][:, of], causal, exact_rows)):
                want[i][span][:, of if i < 2 else h] = value
                bound[i][span][:, of if i < 2 else h] = error
    for name, a, w, b in zip(("out", "dq", "dk", "dv"), got, want, bound):
        close(a, w, b, name)
    return got


def poison(*shapes):
    """Blocks of the sizes that the call will allocate, filled with NaN and given back to the allocator."""
    blocks = [torch.full(shape, math.nan, dtype=dtype, device="cuda") for shape, dtype in shapes for _ in range(8)]
    torch.cuda.synchronize()
    del blocks


def offsets_of(lengths, kind=torch.int32):
    return torch.tensor([sum(lengths[:i]) for i in range(len(lengths) + 1)], dtype=kind, device="cuda")


# ------------------------------------------------------------------------------------------------
# rows of no sequence
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("width", [64, 128])
def test_padding_beside_an_infinite_value(functional, dtype, causal, width):
    """Padding rows that share a block of 32 with real ones stay 0 although a real token's v is infinite (its own rows may be anything)."""
    lengths = [3, 33, 64, 100, 1]
    q, k, v, g = (make((len(lengths), 150, 2, width), dtype, i, 1.0 if i < 4 else 0.1) for i in (1, 2, 3, 4))
    v[:, 0, :, 5], v[:, 0, :, 6] = math.inf, math.nan
    got = passes(functional, q, k, v, g, causal, lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    packed = [torch.cat([t[i, :n] for i, n in enumerate(lengths)] + [t[0, :20]]) for t in (q, k, v, g)]
    rows = passes(functional, *packed, causal, cu_seqlens=offsets_of(lengths))
    for name, a, b in zip(("out", "dq", "dk", "dv"), got, rows):
        assert all(not a[i, n:].any() for i, n in enumerate(lengths)), name
        assert not b[sum(lengths):].any(), name


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
@pytest.mark.parametrize("front,lengths,tail", [(1, [5], 0), (127, [1, 130], 3), (128, [64], 0), (300, [0, 129, 7], 200), (129, [], 5), (257, [0], 0),
                                                (140, [30] * 40, 1)])
def test_packed_rows_in_front_of_the_first_sequence(functional, dtype, causal, kind, front, lengths, tail):
    """cu_seqlens that starts above 0: the rows in front belong to no sequence, whatever they and the allocator's memory hold."""
    total = front + sum(lengths) + tail
    q, g = make((total, 4, 64), dtype, 1), make((total, 4, 64), dtype, 4, 0.1)
    k, v = make((total, 2, 64), dtype, 2), make((total, 2, 64), dtype, 3)
    for t in (q, k, v, g):
        t[:front], t[total - tail:] = math.nan, math.nan
    offsets = offsets_of(lengths, kind) + front
    spans = [(slice(a, b),) for a, b in zip(offsets.tolist(), offsets.tolist()[1:]) if b > a]
    poison((q.shape, dtype), (k.shape, dtype))
    check(functional, q, k, v, g, causal, spans, cu_seqlens=offsets)


@pytest.mark.parametrize("front,lengths,heads,kv_heads,dtype", [(200, [900, 3, 0, 500], 32, 1, BF16), (77, [1100], 32, 1, F32), (1, [1200, 40], 64, 2, BF16)])
def test_packed_rows_in_front_where_tiles_are_ordered_and_split(functional, front, lengths, heads, kv_heads, dtype):
    from kronfluence_amd import _native

    total = front + sum(lengths) + 9
    call = (len(lengths), 0, total, heads, kv_heads, 32, 1, 1)
    assert _native.lib().kf_attention_backward_workspace_bytes(*call) > 8 * total * heads     # dk and dv in parts
    q, g = make((total, heads, 32), dtype, 1), make((total, heads, 32), dtype, 4, 0.1)
    k, v = make((total, kv_heads, 32), dtype, 2), make((total, kv_heads, 32), dtype, 3)
    for t in (q, k, v, g):
        t[:front], t[total - 9:] = math.nan, math.nan
    offsets = offsets_of(lengths) + front
    spans = [(slice(a, b),) for a, b in zip(offsets.tolist(), offsets.tolist()[1:]) if b > a]
    poison((q.shape, dtype), (k.shape, dtype), ((total * heads * 40,), F32))
    check(functional, q, k, v, g, True, spans, cu_seqlens=offsets)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
@pytest.mark.parametrize("offsets,total", [([0, 100, 60, 200], 210), ([50, 20, 180, 170, 260], 300), ([0, 500, 100], 300), ([-7, 40, 1 << 30], 130),
                                           ([90, 0], 140), ([200] + list(range(0, 1400)) + [1300], 1500)])
def test_offsets_that_do_not_ascend(functional, dtype, kind, offsets, total):
    """Offsets outside the rows are clamped, and one below the one before it counts as that one: every row is written once."""
    if kind == torch.int64:
        offsets = [n if n < 1 << 30 else 1 << 40 for n in offsets]
    q, g = make((total, 2, 64), dtype, 1), make((total, 2, 64), dtype, 4, 0.1)
    k, v = make((total, 1, 64), dtype, 2), make((total, 1, 64), dtype, 3)
    ascending, most = [], 0
    for n in offsets:
        most = max(most, min(max(n, 0), total))
        ascending.append(most)
    poison((q.shape, dtype), (k.shape, dtype))
    got = passes(functional, q, k, v, g, True, cu_seqlens=torch.tensor(offsets, dtype=kind, device="cuda"))
    want = passes(functional, q, k, v, g, True, cu_seqlens=torch.tensor(ascending, dtype=kind, device="cuda"))
    for name, a, b in zip(("out", "dq", "dk", "dv"), got, want):
        assert torch.equal(a, b), name
        assert not a[:ascending[0]].any() and not a[ascending[-1]:].any(), name
    spans = [(slice(a, b),) for a, b in zip(ascending, ascending[1:]) if b > a]
    check(functional, q, k, v, g, True, spans, cu_seqlens=torch.tensor(offsets, dtype=kind, device="cuda"))


# ------------------------------------------------------------------------------------------------
# peaked rows: gradients far below do . out
# ------------------------------------------------------------------------------------------------
def peaked(shape, kv_shape, kind):
    """bf16 q, k, v, g.  "sharp": random scores ten times the usual; "sink": the first key outweighs all the others together."""
    q, k, v, g = make(shape, BF16, 1), make(kv_shape, BF16, 2), make(kv_shape, BF16, 3), make(shape, BF16, 4, 0.05)
    if kind == "sharp":
        return q * 10, k, v, g
    q = (q.float() + 1.0).to(BF16)
    k[..., 0, :, :] = {"sink": 1.25, "strong sink": 2.5}[kind]      # scores of 10 and 20 above the others
    return q, k, v, g


@pytest.mark.parametrize("kind", ["sharp", "sink", "strong sink"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("batch,length,heads,kv_heads,width", [
    (2, 33, 2, 1, 64), (2, 64, 4, 2, 32), (2, 100, 2, 2, 64), (1, 128, 4, 1, 64),       # rows of the one-kernel backward
    (2, 64, 2, 1, 128), (1, 129, 2, 1, 64), (1, 130, 2, 2, 96), (1, 513, 4, 1, 64), (1, 700, 2, 1, 128)])
def test_gradients_of_peaked_rows(functional, kind, causal, batch, length, heads, kv_heads, width):
    q, k, v, g = peaked((batch, length, heads, width), (batch, length, kv_heads, width), kind)
    check(functional, q, k, v, g, causal, [(i, slice(0, length)) for i in range(batch)], exact_rows=32 if causal else 0)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,kv_heads,width,length", [(4, 1, 32, 33), (2, 2, 64, 40), (4, 2, 64, 128), (3, 3, 32, 100), (2, 1, 96, 64)])
def test_few_keys_in_padded_rows(functional, causal, heads, kv_heads, width, length):
    """Sequences of 2 to 32 tokens in longer rows (33 to 128 and width <= 64: the one-kernel backward): D to fp32's accuracy."""
    lengths = [2, 2, 3, 5, 8, 17, 31, 32]
    q, k, v, g = (make((len(lengths), length, n, width), BF16, seed, scale)
                  for n, seed, scale in ((heads, 1, 3.0), (kv_heads, 2, 1.0), (kv_heads, 3, 1.0), (heads, 4, 0.05)))
    for i, n in enumerate(lengths):
        q[i, n:], k[i, n:], v[i, n:], g[i, n:] = math.nan, math.inf, math.nan, -math.inf
    check(functional, q, k, v, g, causal, [(i, slice(0, n)) for i, n in enumerate(lengths)], exact_rows=32,
          lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"))


# ------------------------------------------------------------------------------------------------
# dk and dv in parts; whole (sequence, head) pairs dealt to the XCDs
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("causal,lengths,heads,kv_heads,width", [
    (True, [1030], 32, 1, 72), (False, [1030], 32, 1, 96), (True, [1030], 64, 2, 128), (False, [1030, 1, 517], 32, 1, 128),
    (True, [1030, 0, 129, 1029], 32, 1, 64), (False, [0, 700], 32, 1, 32)])
def test_dk_dv_in_parts(functional, dtype, causal, lengths, heads, kv_heads, width):
    """Dense and padded batches whose dk and dv are summed from parts, NaN behind the tokens."""
    from kronfluence_amd import _native

    batch, length = len(lengths), 1030
    call = (batch, length, batch * length, heads, kv_heads, width, 0, int(causal))
    delta = (batch * length * heads * 4 + 15) // 16 * 16
    whole = 2 * kv_heads * batch * length * width * 4
    parts, rest = divmod(_native.lib().kf_attention_backward_workspace_bytes(*call) - delta, whole)
    assert rest == 0 and parts >= 2
    q, k, v, g = (make((batch, length, n, width), dtype, seed, scale)
                  for n, seed, scale in ((heads, 1, 1.5), (kv_heads, 2, 1.0), (kv_heads, 3, 1.0), (heads, 4, 0.1)))
    for i, n in enumerate(lengths):
        q[i, n:], k[i, n:], v[i, n:], g[i, n:] = math.nan, math.inf, math.nan, -math.inf
    padded = {} if lengths == [length] else {"lengths": torch.tensor(lengths, dtype=torch.int32, device="cuda")}
    check(functional, q, k, v, g, causal, [(i, slice(0, n)) for i, n in enumerate(lengths) if n], **padded)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("causal,batch,length,heads,kv_heads,width", [(True, 33, 300, 4, 2, 64), (False, 16, 129, 4, 4, 128), (True, 70, 200, 2, 1, 32),
                                                                      (False, 66, 257, 1, 1, 72), (True, 9, 520, 16, 8, 64)])
def test_pairs_dealt_to_the_xcds(functional, dtype, causal, batch, length, heads, kv_heads, width):
    """At least 64 (sequence, key / value head) pairs: blocks of pairs of one XCD, more and fewer than a multiple of eight."""
    lengths = [max(0, length - 37 * (i % 8)) if i % 5 else length for i in range(batch)]
    q, k, v, g = (make((batch, length, n, width), dtype, seed, scale)
                  for n, seed, scale in ((heads, 1, 1.5), (kv_heads, 2, 1.0), (kv_heads, 3, 1.0), (heads, 4, 0.1)))
    for i, n in enumerate(lengths):
        q[i, n:], k[i, n:], v[i, n:], g[i, n:] = math.nan, math.inf, math.nan, -math.inf
    check(functional, q, k, v, g, causal, [(i, slice(0, n)) for i, n in enumerate(lengths) if n],
          lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"))


# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float64, torch.int64])
def test_autocast_casts_no_other_types(functional, dtype):
    """As torch's operators under autocast: float64 is not rounded to bf16 on the way in, an integer is no head."""
    from kronfluence_amd._native import KfError

    q = torch.ones(1, 5, 1, 8, dtype=dtype, device="cuda")
    with torch.autocast("cuda", torch.bfloat16), pytest.raises(KfError, match="bfloat16 or float32"):
        functional.attention(q, q, q)
