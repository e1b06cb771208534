"""Attention and norms of the model passes (kronfluence_amd/functional.py) against the formulas in 64 bits.

Tolerances are elementwise bounds on the rounding errors the kernels may make, evaluated in 64 bits next to the expected values
(first order; U = half a step of the output type, E = 2^-24 half a step of fp32):

attention   p carries the fp32 errors of a width-long product, of exp2 and of the sum over n keys -- relative
            ep = (width + 8) E max(scale |q| |k|) + (n + 16) E -- and, with bf16 inputs, one rounding U to its operand type.
            out:  (ep + Up) (p |v|) + U |out|
            D:    sum |do| err(out) + (width + 2) E |do| |out|;   (ep + (n + 4) E) sum p |dp| + (width + 2) E sum p |do| |v| for rows that see
                  32 keys at most
            ds:   (ep + Up) |ds| + p (err(D) + (width + 2) E |do| |v|) + E p (|dp| + |D|);    rounded once more (U) for dq, dk
            dq:   scale err(ds) |k| + (n + 2) E scale |ds| |k| + U |dq|;   dk, dv likewise
            (Up = U for bf16, 0 for fp32: fp32 operands are not rounded)
norms       mu and the mean square are sums of `width` values in a tree of at most K = width / 64 + 16 additions per path:
            err(mu) = K E mean |x|,  rel(r) = K E + err(mu) r (|mean xhat| <= 1),  err(xhat) as below,  y: |w| err(xhat) + U |y|.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
# fp16 values below 2^-14 are subnormal, 2^-24 apart: there half a step is 2^-25 whatever the value (bf16 and fp32 have fp32's exponents:
# their subnormals begin at 2^-126)
FLOOR = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def functional():
    from kronfluence_amd import functional

    return functional


def close(got, want, bound, what):
    got = got.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    worst = ((got - want).abs() / (bound + 1e-300)).max().item() if want.numel() else 0.0
    off = (got - want).abs() > bound
    assert not bool(off.any()) and bool(torch.isfinite(got).all()), (what, worst, int(off.sum()), got.numel())


# ------------------------------------------------------------------------------------------------
# attention
# ------------------------------------------------------------------------------------------------
def expected_sequence(q, k, v, g, causal, scale, few=False):
    """Values and error bounds for one sequence and one kv head: ``q``, ``g`` [n, group, width], ``k``, ``v`` [n, width]."""
    dtype = q.dtype
    U, Up = HALF[dtype], HALF[dtype] if dtype == BF16 else 0.0
    q, k, v, g = (t.double().transpose(0, 1) if t.dim() == 3 else t.double()[None] for t in (q, k, v, g))
    n, width = q.shape[1], q.shape[2]
    s = scale * q @ k.transpose(1, 2)
    if causal:
        s = s.masked_fill(~torch.ones(n, n, dtype=torch.bool, device=s.device).tril(), -math.inf)
    p = torch.softmax(s, dim=-1)
    ep = (width + 8) * E * float((scale * q.abs() @ k.abs().transpose(1, 2)).max()) + (n + 16) * E
    out = p @ v
    err_out = (ep + Up + n * E) * (p @ v.abs()) + U * out.abs()
    dp = g @ v.transpose(1, 2)
    delta = (g * out).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    dq, dk, dv = scale * ds @ k, scale * ds.transpose(1, 2) @ q, p.transpose(1, 2) @ g
    err_delta = (g.abs() * err_out).sum(-1, keepdim=True) + (width + 2) * E * (g.abs() * out.abs()).sum(-1, keepdim=True)
    if few:
        err_delta = (p * ((ep + (n + 4) * E) * dp.abs() + (width + 2) * E * (g.abs() @ v.abs().transpose(1, 2)))).sum(-1, keepdim=True)
    err_ds = ((ep + 2 * E) * ds.abs() + p * (err_delta + (width + 2) * E * (g.abs() @ v.abs().transpose(1, 2)))
              + E * p * (dp.abs() + delta.abs()) + Up * ds.abs() + (n + 2) * E * ds.abs())
    err_dq = scale * err_ds @ k.abs() + U * dq.abs()
    # the group's heads sum into one dk, dv
    dk_sum, dv_sum = dk.sum(0), dv.sum(0)
    err_dk = (scale * err_ds.transpose(1, 2) @ q.abs()).sum(0) + q.shape[0] * n * E * (scale * ds.abs().transpose(1, 2) @ q.abs()).sum(0) + U * dk_sum.abs()
    err_dv = ((ep + Up + (q.shape[0] * n + 2) * E) * (p.transpose(1, 2) @ g.abs())).sum(0) + U * dv_sum.abs()
    heads_last = lambda t: t.transpose(0, 1)
    return ((heads_last(out), heads_last(err_out)), (heads_last(dq), heads_last(err_dq)), (dk_sum, err_dk), (dv_sum, err_dv))


def check_attention(functional, q, k, v, g, causal, spans, scale=None, lengths=None, cu_seqlens=None, few=False):
    """``spans``: (index of the sequence's rows) for every sequence that has tokens; rows outside every span must come back 0."""
    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    out = functional.attention(q, k, v, causal=causal, scale=scale, lengths=lengths, cu_seqlens=cu_seqlens)
    grads = torch.autograd.grad(out, (q, k, v), g)
    with torch.no_grad():
        again = functional.attention(q, k, v, causal=causal, scale=scale, lengths=lengths, cu_seqlens=cu_seqlens)
    assert torch.equal(again, out), "the call without a graph gives the same output"
    assert out.dtype == q.dtype and all(d.dtype == q.dtype and d.shape == t.shape for d, t in zip(grads, (q, k, v)))
    heads, kv_heads, width = q.shape[-2], k.shape[-2], q.shape[-1]
    group = heads // kv_heads
    want = [torch.zeros(t.shape, dtype=torch.float64, device=t.device) for t in (q, q, k, v)]
    bound = [torch.zeros_like(w) for w in want]
    for span in spans:
        for h in range(kv_heads):
            of = slice(h * group, (h + 1) * group)
            parts = expected_sequence(q.detach()[span][:, of], k.detach()[span][:, h], v.detach()[span][:, h], g[span][:, of], causal,
                                      1.0 / math.sqrt(width) if scale is None else scale, few)
            for i, (value, error) in enumerate(parts):
                place = of if i < 2 else h
                want[i][span][:, place] = value
                bound[i][span][:, place] = error
    for name, got, w, b in zip(("out", "dq", "dk", "dv"), (out.detach(),) + grads, want, bound):
        close(got, w, b, name)
    return (out.detach(),) + grads


def make(shape, dtype, seed, scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("batch,length,heads,kv_heads,width", [
    (1, 1, 1, 1, 8), (2, 2, 2, 1, 16), (1, 17, 4, 2, 32), (3, 31, 3, 3, 64), (2, 33, 4, 1, 128), (2, 64, 2, 2, 40), (1, 65, 8, 2, 72),
    (2, 127, 2, 1, 96), (1, 128, 4, 4, 80), (1, 129, 6, 2, 128), (1, 300, 2, 1, 64), (1, 513, 4, 2, 128), (2, 100, 2, 2, 100), (1, 70, 2, 1, 33),
])
def test_attention_dense(functional, dtype, causal, batch, length, heads, kv_heads, width):
    q = make((batch, length, heads, width), dtype, 1, 1.5)
    k, v = make((batch, length, kv_heads, width), dtype, 2), make((batch, length, kv_heads, width), dtype, 3)
    g = make(q.shape, dtype, 4, 0.1)
    check_attention(functional, q, k, v, g, causal, [(i, slice(0, length)) for i in range(batch)])


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("width", [32, 64, 128])
def test_attention_padded_rows_hold_anything(functional, dtype, causal, width):
    """Lengths of zero, one, odd ones and the whole row; NaN and infinities behind them, in the gradient too."""
    lengths = [0, 1, 2, 63, 64, 65, 128, 129, 150]
    shape = (len(lengths), 150, 2, width)
    q, k, v, g = make(shape, dtype, 1), make(shape, dtype, 2), make(shape, dtype, 3), make(shape, dtype, 4, 0.1)
    for i, n in enumerate(lengths):
        q[i, n:], k[i, n:], v[i, n:], g[i, n:] = math.nan, math.inf, math.nan, -math.inf
    spans = [(i, slice(0, n)) for i, n in enumerate(lengths) if n]
    for kind in (torch.int32, torch.int64):
        check_attention(functional, q, k, v, g, causal, spans, lengths=torch.tensor(lengths, dtype=kind, device="cuda"))


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("length,heads,kv_heads,width", [(128, 4, 2, 64), (128, 3, 3, 32), (100, 4, 1, 48), (33, 2, 2, 64), (32, 2, 1, 8), (31, 6, 2, 40),
                                                         (1, 2, 1, 64)])
def test_attention_short_padded_batches(functional, causal, length, heads, kv_heads, width):
    """Batches of at most 128 tokens a row (with more than 32 the backward pass is one kernel): every length around its blocks of 32, NaN behind the tokens."""
    lengths = sorted({n for n in (0, 1, 2, 31, 32, 33, 63, 64, 65, 95, 96, 97, 127, 128, length) if n <= length})
    q, k, v, g = (make((len(lengths), length, n, width), BF16, seed, scale)
                  for n, seed, scale in ((heads, 1, 2.0), (kv_heads, 2, 1.0), (kv_heads, 3, 1.0), (heads, 4, 0.1)))
    for i, n in enumerate(lengths):
        q[i, n:], k[i, n:], v[i, n:], g[i, n:] = math.nan, math.inf, math.nan, -math.inf
    spans = [(i, slice(0, n)) for i, n in enumerate(lengths) if n]
    check_attention(functional, q, k, v, g, causal, spans, lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,kv_heads,width", [(4, 1, 32), (2, 2, 64), (2, 1, 128)])
def test_attention_gradients_of_rows_with_few_keys(functional, dtype, causal, heads, kv_heads, width):
    """Peaked rows with 2 to 32 keys: do . out there is far greater than the gradients it is taken off, so a rounded out must not enter."""
    lengths = [2, 2, 2, 2, 3, 5, 8, 17, 31, 32]
    q, k, v, g = (make((sum(lengths), n, width), dtype, seed, scale)
                  for n, seed, scale in ((heads, 1, 3.0), (kv_heads, 2, 1.0), (kv_heads, 3, 1.0), (heads, 4, 0.05)))
    offsets = [0]
    for n in lengths:
        offsets.append(offsets[-1] + n)
    spans = [slice(a, b) for a, b in zip(offsets, offsets[1:])]
    check_attention(functional, q, k, v, g, causal, spans, cu_seqlens=torch.tensor(offsets, dtype=torch.int32, device="cuda"), few=True)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lengths,tail", [([5], 0), ([0, 0, 7, 1, 1, 0, 130, 128, 3, 0], 9), ([127, 1, 129, 64, 0], 200), ([1] * 40, 0), ([], 6), ([0], 3)])
def test_attention_packed(functional, dtype, causal, lengths, tail):
    total = sum(lengths) + tail
    shape, kv_shape = (total, 4, 64), (total, 2, 64)
    q, k, v, g = make(shape, dtype, 1), make(kv_shape, dtype, 2), make(kv_shape, dtype, 3), make(shape, dtype, 4, 0.1)
    bounds = [0]
    for n in lengths:
        bounds.append(bounds[-1] + n)
    for t in (q, k, v, g):
        t[bounds[-1]:] = math.nan
    spans = [(slice(a, b),) for a, b in zip(bounds, bounds[1:]) if b > a]
    check_attention(functional, q, k, v, g, causal, spans, cu_seqlens=torch.tensor(bounds, dtype=torch.int32, device="cuda"))


@pytest.mark.parametrize("causal", [True, False])
def test_attention_packed_in_order_of_cost(functional, causal):
    """Enough work that the tiles are ordered: short documents in front of a long one, empty ones between, a tail; heads of a group."""
    from kronfluence_amd import _native

    lengths, tail = [3, 40, 0, 700, 129, 1, 0, 1500, 64], 20
    total = sum(lengths) + tail
    assert _native.lib().kf_attention_order_bytes(len(lengths), total, 32) > 0
    q, g = make((total, 32, 32), BF16, 1), make((total, 32, 32), BF16, 4, 0.1)
    k, v = make((total, 2, 32), BF16, 2), make((total, 2, 32), BF16, 3)
    bounds = [0]
    for n in lengths:
        bounds.append(bounds[-1] + n)
    spans = [(slice(a, b),) for a, b in zip(bounds, bounds[1:]) if b > a]
    first = check_attention(functional, q, k, v, g, causal, spans, cu_seqlens=torch.tensor(bounds, dtype=torch.int32, device="cuda"))
    again = check_attention(functional, q, k, v, g, causal, spans, cu_seqlens=torch.tensor(bounds, dtype=torch.int32, device="cuda"))
    assert all(torch.equal(x, y) for x, y in zip(first, again))


def test_attention_packed_is_the_padded_batch(functional):
    """The same sequences packed and padded: the same bits."""
    lengths = [130, 1, 64, 200]
    q, k, v = (make((4, 200, h, 64), BF16, i) for i, h in ((1, 4), (2, 2), (3, 2)))
    padded = functional.attention(q, k, v, lengths=torch.tensor(lengths, device="cuda"))
    packed = [torch.cat([t[i, :n] for i, n in enumerate(lengths)]) for t in (q, k, v)]
    cu = torch.tensor([0] + lengths, device="cuda").cumsum(0)
    out = functional.attention(*packed, cu_seqlens=cu)
    assert torch.equal(out, torch.cat([padded[i, :n] for i, n in enumerate(lengths)]))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_attention_strides(functional, dtype):
    """Slices of a fused projection, heads in front of tokens, every second token, an offset that is not 16-byte aligned, a last axis
    that is not contiguous, heads expanded from one."""
    b, t, h, d = 2, 70, 2, 64
    g = make((b, t, h, d), dtype, 9, 0.1)
    spans = [(i, slice(0, t)) for i in range(b)]
    dense = [make((b, t, h, d), dtype, i) for i in (1, 2, 3)]
    plain = check_attention(functional, *dense, g, True, spans)
    fused = torch.stack(dense, dim=2)
    head_first = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in dense]
    doubled = [x.repeat_interleave(2, dim=1)[:, ::2] for x in dense]
    base = [torch.empty(x.numel() + 1, dtype=dtype, device="cuda") for x in dense]
    shifted = [y[1:].view(x.shape).copy_(x) for x, y in zip(dense, base)]
    turned = [x.transpose(2, 3).contiguous().transpose(2, 3) for x in dense]
    for kind, operands in (("fused", fused.unbind(2)), ("heads first", head_first), ("every second token", doubled), ("unaligned", shifted),
                           ("turned", turned)):
        for x, y in zip(plain, check_attention(functional, *operands, g, True, spans)):
            assert torch.equal(x, y), kind
    one = make((b, t, 1, d), dtype, 5)
    check_attention(functional, dense[0], one.expand(b, t, h, d), one.expand(b, t, h, d), g, False, spans)
    turned_g = g.transpose(1, 2).contiguous().transpose(1, 2)
    for x, y in zip(plain, check_attention(functional, *dense, turned_g, True, spans)):
        assert torch.equal(x, y)


def test_attention_gradient_of_a_sum(functional):
    """The gradient a reduction sends back is an expanded scalar (all strides 0)."""
    q, k, v = (make((1, 40, 2, 32), BF16, i).requires_grad_() for i in (1, 2, 3))
    functional.attention(q, k, v).sum().backward()
    ones = torch.ones(1, 40, 2, 32, dtype=BF16, device="cuda")
    want = check_attention(functional, q, k, v, ones, True, [(0, slice(0, 40))])
    for t, w in zip((q, k, v), want[1:]):
        assert torch.equal(t.grad, w)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_attention_large_and_equal_scores(functional, dtype):
    """Scores of +-300 (a softmax that is one-hot), equal scores, and a scale given by the caller."""
    b, t, h, d = 1, 140, 2, 64
    k, v, g = make((b, t, h, d), dtype, 2), make((b, t, h, d), dtype, 3), make((b, t, h, d), dtype, 4, 0.1)
    spans = [(0, slice(0, t))]
    check_attention(functional, torch.zeros_like(k), k, v, g, True, spans)
    check_attention(functional, 4.0 * k, k, v, g, False, spans, scale=1.0)
    check_attention(functional, make((b, t, h, d), dtype, 5), k, v, g, True, spans, scale=0.01)


@pytest.mark.parametrize("causal", [True, False])
def test_attention_gradient_against_differences(functional, causal):
    """<dL/dx, e> against central differences of the fp32 operator itself along random directions.  Tolerance: the truncation of
    the fourth-order difference, bounded by its distance from the second-order one, plus 2^-24 (width + n) sum |out g| / h."""
    b, t, h, d = 1, 37, 2, 32
    inputs = [make((b, t, h, d), F32, i) for i in (1, 2, 3)]
    g = make((b, t, h, d), F32, 4)
    leaves = [x.clone().requires_grad_() for x in inputs]
    out = functional.attention(*leaves, causal=causal)
    grads = torch.autograd.grad(out, leaves, g)
    noise = E * (d + t) * float((out.detach().abs().double() * g.abs().double()).sum())

    def loss(i, e, step):
        moved = [x + step * e if n == i else x for n, x in enumerate(inputs)]
        return float((functional.attention(*moved, causal=causal).double() * g.double()).sum())

    for i, grad in enumerate(grads):
        e = make((b, t, h, d), F32, 20 + i)
        step = 2.0 ** -6
        one = (loss(i, e, step) - loss(i, e, -step)) / (2 * step)
        two = (loss(i, e, 2 * step) - loss(i, e, -2 * step)) / (4 * step)
        best = one + (one - two) / 3
        assert abs(best - float((grad.double() * e.double()).sum())) <= abs(one - two) / 3 + 2 * noise / step, (i, one, two)


def test_attention_on_another_stream_and_twice(functional):
    """Bit for bit the same on a second stream, twice, and with two calls in flight at once."""
    q, k, v = (make((2, 300, h, 64), BF16, i).requires_grad_() for i, h in ((1, 8), (2, 2), (3, 2)))
    g = make((2, 300, 8, 64), BF16, 4, 0.1)

    def step():
        out = functional.attention(q, k, v)
        return (out.detach(),) + torch.autograd.grad(out, (q, k, v), g)

    first = step()
    side = [torch.cuda.Stream() for _ in range(2)]
    results = []
    for s in side:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            results.append(step())
    torch.cuda.synchronize()
    for other in results + [step()]:
        for x, y in zip(first, other):
            assert torch.equal(x, y)


def capture(step):
    """``step`` warmed up and captured on a side stream: (graph, its outputs)."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outputs = step()
    return graph, outputs


def test_attention_and_norm_in_two_captured_graphs(functional):
    """Forward and backward captured twice (two graphs with workspaces of their own), replayed in turn with eager work between, on
    new inputs; every replay against the eager result."""
    shape = (2, 200, 4, 64)
    x = make((2, 200, 256), BF16, 1).requires_grad_()
    w, b = make((256,), F32, 2).requires_grad_(), make((256,), F32, 3).requires_grad_()
    lengths = torch.tensor([200, 77], device="cuda", dtype=torch.int32)
    g = make(shape, BF16, 4, 0.1)

    def step(causal):
        h = functional.layer_norm(x, w, b, out_dtype=BF16).view(shape)
        out = functional.attention(h, h, h, causal=causal, lengths=lengths)
        return (out.detach(),) + torch.autograd.grad(out, (x, w, b), g)

    graphs = [capture(lambda causal=causal: step(causal)) for causal in (True, False)]
    for turn in range(3):
        with torch.no_grad():
            x.copy_(make((2, 200, 256), BF16, 50 + turn))
            lengths.copy_(torch.tensor([200 - turn, 77 * turn], device="cuda", dtype=torch.int32))
        eager = [step(causal) for causal in (True, False)]
        torch.cuda.synchronize()
        for graph, _ in graphs:
            graph.replay()
        for (_, got), want in zip(graphs, eager):
            for a, e in zip(got, want):
                assert torch.equal(a, e), turn


@pytest.mark.parametrize("dtype,lengths,packed", [(BF16, [100, 64, 1, 0], False), (F32, [100, 64, 1, 0], False), (BF16, [300] * 30 + [0, 1, 77], True),
                                                  (F32, [300] * 30 + [0, 1, 77], True)])
def test_every_form_of_attention_captured(functional, dtype, lengths, packed):
    """As above: short rows in one backward kernel, fp32, packed documents in order of cost with new offsets at every replay."""
    heads, width, most = 4, 64, max(lengths)
    shape = (sum(lengths) + 5, heads, width) if packed else (len(lengths), most, heads, width)
    q, k, v = (make(shape, dtype, i + 1).requires_grad_() for i in range(3))
    g = make(shape, dtype, 4, 0.1)

    def rows(turn):
        if not packed:
            return torch.tensor([max(0, n - turn) for n in lengths], dtype=torch.int32, device="cuda")
        turned = lengths[turn:] + lengths[:turn]
        return torch.tensor([sum(turned[:i]) for i in range(len(turned) + 1)], dtype=torch.int32, device="cuda")

    counts = rows(0)

    def step():
        out = functional.attention(q, k, v, **({"cu_seqlens": counts} if packed else {"lengths": counts}))
        return (out.detach(),) + torch.autograd.grad(out, (q, k, v), g)

    graph, got = capture(step)
    for turn in range(3):
        with torch.no_grad():
            counts.copy_(rows(32 * turn if packed else turn))
            q.copy_(make(shape, dtype, 60 + turn))
        eager = step()
        torch.cuda.synchronize()
        graph.replay()
        for a, e in zip(got, eager):
            assert torch.equal(a, e), turn


def test_second_derivatives_are_refused(functional):
    """A graph of the gradients would silently lack these operators."""
    from kronfluence_amd._native import KfError

    x = make((3, 64), F32, 1).requires_grad_()
    for y in (functional.layer_norm(x), functional.rms_norm(x), functional.attention(x.view(1, 3, 1, 64), *[x.view(1, 3, 1, 64)] * 2)):
        with pytest.raises((KfError, RuntimeError), match="first derivatives"):
            torch.autograd.grad(y.sum(), x, create_graph=True)


def test_saved_tensors_are_guarded(functional):
    """Writing in place to a tensor the backward pass reads is an error, as with torch's own operators."""
    x, w = make((3, 64), F32, 1).requires_grad_(), make((64,), F32, 2)
    y = functional.layer_norm(x, w)
    w.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_attention_empty_batches(functional):
    for shape in ((0, 5, 2, 64), (3, 0, 2, 64)):
        q = torch.zeros(shape, dtype=BF16, device="cuda", requires_grad=True)
        out = functional.attention(q, q, q)
        out.sum().backward()
        assert out.shape == shape and q.grad.shape == shape
    q = torch.zeros((0, 2, 64), dtype=BF16, device="cuda", requires_grad=True)
    functional.attention(q, q, q, cu_seqlens=torch.zeros(3, dtype=torch.int32, device="cuda")).sum().backward()
    q = make((4, 2, 64), BF16, 1).requires_grad_()
    out = functional.attention(q, q, q, cu_seqlens=torch.zeros(1, dtype=torch.int32, device="cuda"))   # no sequence at all
    out.sum().backward()
    assert not out.any() and not q.grad.any()


def test_attention_under_autocast(functional):
    q, k, v = (make((1, 50, 2, 64), F32, i).requires_grad_() for i in (1, 2, 3))
    with torch.autocast("cuda", dtype=BF16):
        out = functional.attention(q, k, v)
    assert out.dtype == BF16
    assert torch.equal(out, functional.attention(q.to(BF16), k.to(BF16), v.to(BF16)))
    out.float().sum().backward()
    assert q.grad.dtype == F32


# ------------------------------------------------------------------------------------------------
# norms
# ------------------------------------------------------------------------------------------------
def check_norm(functional, x, w, b, g, centred, eps=1e-5, out_dtype=None):
    leaves = [t for t in (x, w, b) if t is not None]
    for t in leaves:
        t.requires_grad_()
    call = (lambda: functional.layer_norm(x, w, b, eps=eps, out_dtype=out_dtype)) if centred else (lambda: functional.rms_norm(x, w, eps=eps, out_dtype=out_dtype))
    y = call()
    grads = dict(zip([n for n, t in (("dx", x), ("dw", w), ("db", b)) if t is not None], torch.autograd.grad(y, leaves, g)))
    with torch.no_grad():
        assert torch.equal(call(), y)
    assert y.dtype == (out_dtype or x.dtype)
    x64, g64 = x.detach().double().reshape(-1, x.shape[-1]), g.double().reshape(-1, x.shape[-1])
    w64 = torch.ones(x.shape[-1], dtype=torch.float64, device=x.device) if w is None else w.detach().double()
    b64 = torch.zeros_like(w64) if b is None else b.detach().double()
    rows, width = x64.shape
    K = width / 64 + 16
    mu = x64.mean(-1, keepdim=True) if centred else torch.zeros(rows, 1, dtype=torch.float64, device=x.device)
    err_mu = K * E * x64.abs().mean(-1, keepdim=True) if centred else 0.0
    var = (x64 - mu).square().mean(-1, keepdim=True) + eps
    r = 1 / var.sqrt()
    h = (x64 - mu) * r
    err_c = err_mu + E * (x64 - mu).abs()                                      # of x - mu
    rel_r = (K + 4) * E + ((x64 - mu).abs() * err_c).mean(-1, keepdim=True) * r * r
    err_h = r * err_c + h.abs() * (rel_r + 2 * E)
    want = h * w64 + b64
    close(y.detach().reshape(rows, width), want, w64.abs() * err_h + 2 * E * (want.abs() + (h * w64).abs()) + HALF[y.dtype] * want.abs() + FLOOR[y.dtype], "y")
    u = g64 * w64
    m_u = u.mean(-1, keepdim=True) if centred else torch.zeros_like(r)
    m_uh = (u * h).mean(-1, keepdim=True)
    inner = u - m_u - h * m_uh
    err_m = (K + 3) * E * u.abs().mean(-1, keepdim=True) if centred else 0.0
    err_muh = ((K + 3) * E * u.abs() * h.abs() + u.abs() * err_h).mean(-1, keepdim=True)
    err_in = 3 * E * (u.abs() + m_u.abs() + (h * m_uh).abs()) + err_m + h.abs() * err_muh + err_h * m_uh.abs()
    dx = r * inner
    close(grads["dx"].reshape(rows, width), dx, r * err_in + dx.abs() * (rel_r + HALF[x.dtype] + 2 * E) + FLOOR[x.dtype], "dx")
    R = rows / 64 + 40     # additions a row's term passes through
    if w is not None:
        dw = (g64 * h).sum(0)
        close(grads["dw"], dw, (g64.abs() * (err_h + R * E * h.abs())).sum(0) + HALF[w.dtype] * dw.abs() + FLOOR[w.dtype], "dw")
    if b is not None:
        db = g64.sum(0)
        close(grads["db"], db, R * E * g64.abs().sum(0) + HALF[b.dtype] * db.abs() + FLOOR[b.dtype], "db")
    return y.detach(), grads


@pytest.mark.parametrize("centred", [True, False])
@pytest.mark.parametrize("rows,width", [(1, 1), (5, 2), (3, 7), (130, 8), (9, 9), (257, 64), (33, 511), (4, 512), (70, 513), (41, 769), (6, 1000),
                                        (5, 1025), (9, 2048), (7, 2049), (5, 4096), (600, 4097), (3, 8193), (2, 16384), (5, 16385), (520, 16400),
                                        (5000, 40)])
def test_norm_sizes(functional, centred, rows, width):
    x = make((rows, width), F32, 1) * 2 + 0.3
    w, b = make((width,), F32, 2, 0.3) + 1, make((width,), F32, 3) if centred else None
    check_norm(functional, x, w, b, make((rows, width), F32, 4), centred)


@pytest.mark.parametrize("x_dtype", [F32, BF16, F16])
@pytest.mark.parametrize("y_dtype", [F32, BF16, F16])
@pytest.mark.parametrize("w_dtype", [F32, BF16, F16, None])
@pytest.mark.parametrize("centred", [True, False])
def test_norm_types(functional, x_dtype, y_dtype, w_dtype, centred):
    for rows, width in ((37, 200), (6, 2056)):
        x = make((rows, width), x_dtype, 1)
        w = None if w_dtype is None else make((width,), w_dtype, 2)
        b = None if w_dtype is None or not centred else make((width,), w_dtype, 3)
        check_norm(functional, x, w, b, make((rows, width), y_dtype, 4), centred, out_dtype=y_dtype)


def test_norm_strides_and_shapes(functional):
    """Row strides, transposed and expanded inputs, three and one dimensions, an odd element offset, an expanded gradient."""
    w, b = make((65,), F32, 2), make((65,), F32, 3)
    base = make((12, 3, 130), BF16, 1)
    views = [base[:, :, :65], base[::2, 1, 3:68], base[:1, 1, :65].expand(7, 65), make((65, 9), BF16, 5).t(), base[0, 0, :65], base.flatten()[1:66 * 65 - 64].view(65, 65)]
    for x in views:
        x = x.detach()
        y, grads = check_norm(functional, x, w, b, make(x.shape, F32, 7), True, out_dtype=F32)
        dense, dense_grads = check_norm(functional, x.detach().contiguous(), w, b, make(x.shape, F32, 7), True, out_dtype=F32)
        assert torch.equal(y, dense) and all(torch.equal(grads[n], dense_grads[n]) for n in grads)
    x = make((4, 65), F32, 8).requires_grad_()
    functional.layer_norm(x, w.detach(), b.detach()).sum().backward()
    assert torch.equal(x.grad, check_norm(functional, x.detach().clone(), w, b, torch.ones(4, 65, device="cuda"), True)[1]["dx"])


def test_norm_frozen_vectors_and_inputs(functional):
    """Each gradient alone is the one of the full call."""
    x, w, b, g = make((50, 300), F32, 1), make((300,), F32, 2), make((300,), F32, 3), make((50, 300), F32, 4)
    _, full = check_norm(functional, x.clone(), w.clone(), b.clone(), g, True)
    for names in (("dx",), ("dw",), ("db",), ("dw", "db"), ("dx", "db")):
        leaves = {n: t.clone().requires_grad_(n in names) for n, t in (("dx", x), ("dw", w), ("db", b))}
        y = functional.layer_norm(*leaves.values())
        for n, got in zip(names, torch.autograd.grad(y, [leaves[n] for n in names], g)):
            assert torch.equal(got, full[n]), (names, n)
    check_norm(functional, x.clone(), None, b.clone(), g, True)     # a bias without a weight


def test_norm_constant_rows_offsets_and_eps(functional):
    """A row of equal values (variance 0), a large common offset, eps = 0 and large eps, a row of NaN beside good rows."""
    x = make((6, 520), F32, 1)
    x[1] = 3.0
    x[2] += 1000.0
    w, b, g = make((520,), F32, 2), make((520,), F32, 3), make((6, 520), F32, 4)
    check_norm(functional, x.clone(), w, b, g, True)
    check_norm(functional, x.clone(), w, None, g, False, eps=0.5)
    check_norm(functional, x[3:].clone(), w, b, g[3:], True, eps=0.0)
    x[4, 7] = math.nan
    y = functional.layer_norm(x, w.detach(), b.detach())
    assert bool(y[4].isnan().all()) and not bool(y[[0, 1, 2, 3, 5]].isnan().any())


def test_norm_gradient_against_differences(functional):
    """As for attention: fp32 central differences along random directions, fourth order."""
    x, w, b, g = make((5, 70), F32, 1), make((70,), F32, 2) + 1, make((70,), F32, 3), make((5, 70), F32, 4)
    for centred in (True, False):
        inputs = [x, w, b] if centred else [x, w]
        call = functional.layer_norm if centred else lambda x, w: functional.rms_norm(x, w, eps=1e-5)
        leaves = [t.clone().requires_grad_() for t in inputs]
        y = call(*leaves)
        grads = torch.autograd.grad(y, leaves, g)
        noise = 32 * E * float((y.detach().double().abs() * g.double().abs()).sum())
        for i, grad in enumerate(grads):
            e, step = make(inputs[i].shape, F32, 30 + i), 2.0 ** -6
            at = lambda s: float((call(*[t + s * e if n == i else t for n, t in enumerate(inputs)]).double() * g.double()).sum())
            one, two = (at(step) - at(-step)) / (2 * step), (at(2 * step) - at(-2 * step)) / (4 * step)
            want = float((grad.double() * e.double()).sum())
            assert abs(one + (one - two) / 3 - want) <= abs(one - two) / 3 + 2 * noise / step, (centred, i, one, two, want)


def test_norm_under_autocast_and_on_empty_rows(functional):
    x = make((4, 96), BF16, 1)
    w = make((96,), F32, 2)
    with torch.autocast("cuda", dtype=BF16):
        y = functional.layer_norm(x, w)
    assert y.dtype == F32 and torch.equal(y, functional.layer_norm(x, w, out_dtype=F32))
    empty = torch.zeros(0, 96, device="cuda", requires_grad=True)
    weight = w.clone().requires_grad_()
    functional.layer_norm(empty, weight).sum().backward()
    assert empty.grad.shape == (0, 96) and not weight.grad.any()


# ------------------------------------------------------------------------------------------------
# tensors of more than 2^32 elements
# ------------------------------------------------------------------------------------------------
@pytest.fixture
def room():
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 120 << 30:
        pytest.skip("needs 120 GB of free device memory")
    yield
    torch.cuda.empty_cache()


def test_attention_offsets_past_32_bits(functional, room):
    """The last sequences of a packed batch of 2^32 elements and more are those of a small batch, bit for bit."""
    heads, width, each, n = 8, 16, 64, (1 << 25) // 64 + 1
    q, k, v, g = (torch.empty(n * each + 5, heads, width, dtype=BF16, device="cuda") for _ in range(4))
    last = slice((n - 3) * each, n * each)
    for i, t in enumerate((q, k, v, g)):
        t.zero_()
        t[last] = make((3 * each, heads, width), BF16, i + 1)
    assert q.numel() > 1 << 32
    offsets = torch.arange(0, (n + 1) * each, each, dtype=torch.int32, device="cuda")

    def both(q, k, v, g, offsets):
        q, k, v = (t.requires_grad_() for t in (q, k, v))
        out = functional.attention(q, k, v, cu_seqlens=offsets)
        return (out.detach(),) + torch.autograd.grad(out, (q, k, v), g)

    want = both(*(t[last].clone() for t in (q, k, v, g)), offsets[:4].clone())
    got = both(q, k, v, g, offsets)
    for name, a, b in zip(("out", "dq", "dk", "dv"), got, want):
        assert torch.equal(a[last], b) and not bool(a[n * each:].any()) and not bool(a[:each].any()), name


@pytest.mark.parametrize("width", [4096, 20000])
def test_norm_offsets_past_32_bits(functional, room, width):
    rows = (1 << 32) // width + 7
    x, g = (torch.zeros(rows, width, dtype=BF16, device="cuda") for _ in range(2))
    x[-3:], g[-3:] = make((3, width), BF16, 1), make((3, width), BF16, 2)
    w = make((width,), F32, 3)

    def both(x, g):
        x = x.requires_grad_()
        y = functional.layer_norm(x, w)
        return y.detach(), torch.autograd.grad(y, x, g)[0]

    want = both(x[-3:].clone(), g[-3:].clone())
    for a, b in zip(both(x, g), want):
        assert torch.equal(a[-3:], b) and not bool(a[:-3].any())
