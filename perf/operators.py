"""The operators a transformer model's own forward and backward passes are made of, as measured cases.

Every stage of the influence path runs the user's model forward and backward over the data (covariance, Lambda, query and train
passes); between the tracked Linear layers a transformer spends that time in attention and in its norms.  The cases below are those
passes at the shapes of ``bench.py``'s encoder and decoder workloads (T = 128 with padding, T = 512 causal, grouped heads at head
width 128), a packed batch and a long prompt, and the ends of the ranges: single tokens, odd widths, wide rows.

``own`` selects between the plain formulas (elementary torch operations in 32 bits, rounded once at the end) and
``kronfluence_amd.functional``.
"""

import math
import random

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------
def _attention_case(name=None, layout="dense", batch=1, length=1, tokens=0, heads=1, kv_heads=1, width=64, causal=True, dtype="bf16",
                    train=True, fused=False):
    case = {"op": "attention", "layout": layout, "batch": batch, "length": length, "tokens": tokens, "heads": heads,
            "kv_heads": kv_heads, "width": width, "causal": causal, "dtype": dtype, "train": train, "fused": fused}
    return case if name is None else dict(case, name=name)


def _norm_case(name=None, op="layer_norm", rows=1, width=1, dtype="fp32", out="fp32", weights="fp32", train=True, affine=True):
    case = {"op": op, "rows": rows, "width": width, "dtype": dtype, "out": out, "weights": weights, "train": train, "affine": affine}
    return case if name is None else dict(case, name=name)


def listed():
    return [
        # one short sentence through a small model: launch latency is all there is
        _attention_case("attention_one_sentence", batch=1, length=17, heads=4, kv_heads=2, width=32, train=False),
        # the encoder workload: 256 sentences of up to 128 tokens, right-padded, every token sees every real token
        _attention_case("attention_encoder_padded", layout="padded", batch=256, length=128, heads=12, kv_heads=12, width=64, causal=False),
        # the decoder workload at T = 512, read as slices of the fused projection's output
        _attention_case("attention_decoder_fused", batch=64, length=512, heads=12, kv_heads=12, width=64, fused=True),
        # one block of the grouped-query decoder workload
        _attention_case("attention_grouped", batch=16, length=512, heads=32, kv_heads=8, width=128),
        # documents of different lengths packed into one row of tokens (empty and one-token documents among them)
        _attention_case("attention_packed", layout="packed", batch=24, tokens=12011, heads=16, kv_heads=4, width=128),
        # one long document
        _attention_case("attention_long", batch=1, length=8192, heads=32, kv_heads=8, width=128),
        # a model in the framework's default precision, odd length and padding
        _attention_case("attention_fp32_padded", layout="padded", batch=24, length=233, heads=12, kv_heads=12, width=64, dtype="fp32"),
        # the decoder's residual stream under autocast: fp32 in, fp32 out, 32 sequences of 512 tokens
        _norm_case("layer_norm_residual", rows=32 * 512, width=768),
        # the encoder at the largest batch: bf16 in, fp32 out (what autocast asks of a norm), 1 024 sequences of 128
        _norm_case("layer_norm_autocast", rows=1024 * 128, width=768, dtype="bf16", out="fp32"),
        # a few rows of an odd width, forward only
        _norm_case("layer_norm_few_rows", rows=7, width=769, train=False),
        # the grouped-query decoder's norm: 16 sequences of 512 at width 4 096, bf16 throughout
        _norm_case("rms_norm_wide", op="rms_norm", rows=16 * 512, width=4096, dtype="bf16", out="bf16", weights="bf16"),
        # an odd width in fp16 with fp32 weights
        _norm_case("rms_norm_odd", op="rms_norm", rows=3001, width=1001, dtype="fp16", out="fp16"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng: random.Random):
    if rng.random() < 0.6:
        kv_heads = rng.choice([1, 2, 3, 4, 8, 12])
        heads = min(32, kv_heads * rng.choice([1, 1, 2, 4, 8])) // kv_heads * kv_heads
        width = rng.choice([16, 32, 40, 64, 64, 64, 72, 80, 96, 100, 128, 128, 128])
        dtype = "fp32" if rng.random() < 0.25 else "bf16"
        layout = rng.choice(["dense", "padded", "packed"])
        length = _log_int(rng, 1, 4096)
        budget = (2 ** 28 if dtype == "fp32" else 2 ** 30) // (heads * length * length)     # scores of one pass
        budget //= 8 if layout == "packed" else 1       # the longest document of a packed row is several times the mean
        batch = _log_int(rng, 1, max(1, min(256, budget)))
        return _attention_case(layout=layout, batch=batch, length=length, tokens=max(1, batch * length * 2 // 3 - rng.randrange(7)),
                               heads=heads, kv_heads=kv_heads, width=width, causal=rng.random() < 0.7, dtype=dtype,
                               train=rng.random() < 0.75, fused=layout != "packed" and heads == kv_heads and rng.random() < 0.5)
    width = _log_int(rng, 8, 16384)
    rows = _log_int(rng, 1, max(1, min(131072, 2 ** 26 // width)))
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    return _norm_case(op=rng.choice(["layer_norm", "rms_norm"]), rows=rows, width=width, dtype=dtype,
                      out=rng.choice([dtype, "fp32"]), weights=rng.choice([dtype, "fp32"]), train=rng.random() < 0.75,
                      affine=rng.random() < 0.85)


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------
def _lengths(case, seed):
    """The lengths of the case's sequences: plain integers made from the seed."""
    rng = random.Random(seed * 1000003 + 17)
    batch, length = case["batch"], case["length"]
    if case["layout"] == "dense":
        return [length] * batch
    if case["layout"] == "padded":
        # mostly between an eighth and the whole length, now and then a full row
        return [length if rng.random() < 0.15 else rng.randint(max(1, length // 8), length) for _ in range(batch)]
    # packed: cut the tokens at random places; close cuts make one-token documents, equal ones empty documents
    total = case["tokens"] - case["tokens"] // 50       # the last tokens of the row belong to no document
    cuts = sorted(rng.randint(0, total) for _ in range(batch - 1))
    if batch > 4:
        cuts[1] = cuts[0]
        cuts[2] = min(total, cuts[1] + 1)
        cuts.sort()
    bounds = [0] + cuts + [total]
    return [b - a for a, b in zip(bounds, bounds[1:])]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _TYPES[case["dtype"]]

    def normal(*shape, scale=1.0, to=dtype):
        return (torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32) * scale).to(to)

    if case["op"] == "attention":
        heads, kv_heads, width = case["heads"], case["kv_heads"], case["width"]
        lead = (case["tokens"],) if case["layout"] == "packed" else (case["batch"], case["length"])
        if case["fused"]:
            joint = normal(*lead, heads + 2 * kv_heads, width)
            q, k, v = (x.detach() for x in joint.split([heads, kv_heads, kv_heads], dim=-2))
        else:
            q, k, v = normal(*lead, heads, width, scale=1.5), normal(*lead, kv_heads, width), normal(*lead, kv_heads, width)
        lengths = _lengths(case, seed)
        state = {"case": case, "q": q, "k": k, "v": v, "lengths": None, "cu_seqlens": None}
        if case["layout"] == "padded":
            state["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        if case["layout"] == "packed":
            offsets = [0]
            for n in lengths:
                offsets.append(offsets[-1] + n)
            state["cu_seqlens"] = torch.tensor(offsets, dtype=torch.int32, device="cuda")
            state["longest"] = max(lengths)     # the program that packed the documents knows it
        if case["train"]:
            for x in (q, k, v):
                x.requires_grad_(True)
            state["grad"] = normal(*lead, heads, width, scale=0.05)
        return state

    rows, width, weights = case["rows"], case["width"], _TYPES[case["weights"]]
    # a residual stream: rows of different sizes, a few channels far larger than the others, a small common offset
    x = torch.randn(rows, width, generator=gen, device="cuda") * (0.5 + 2.0 * torch.rand(rows, 1, generator=gen, device="cuda"))
    x = x * (1.0 + 4.0 * (torch.rand(width, generator=gen, device="cuda") > 0.99)) + 0.25
    state = {"case": case, "x": x.to(dtype), "weight": None, "bias": None, "eps": 1e-5, "out": _TYPES[case["out"]]}
    if case["affine"]:
        state["weight"] = 1.0 + normal(width, scale=0.2, to=torch.float32)
        state["weight"] = state["weight"].to(weights)
        if case["op"] == "layer_norm":
            state["bias"] = normal(width, scale=0.1, to=weights)
    if case["train"]:
        for name in ("x", "weight", "bias"):
            if state[name] is not None:
                state[name].requires_grad_(True)
        state["grad"] = normal(rows, width, scale=0.05, to=state["out"])
    return state


# ------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if own:
        return _own_attention(state) if op == "attention" else _own_norm(state)
    return _plain_attention(state) if op == "attention" else _plain_norm(state)


def _own_attention(state):
    from kronfluence_amd import functional

    q, k, v, causal = state["q"], state["k"], state["v"], state["case"]["causal"]
    if not state["case"]["train"]:
        with torch.no_grad():
            return {"out": functional.attention(q, k, v, causal=causal, lengths=state["lengths"], cu_seqlens=state["cu_seqlens"])}
    out = functional.attention(q, k, v, causal=causal, lengths=state["lengths"], cu_seqlens=state["cu_seqlens"])
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), state["grad"])
    return {"out": out.detach(), "dq": dq, "dk": dk, "dv": dv}


def _own_norm(state):
    from kronfluence_amd import functional

    x, weight, bias, eps = state["x"], state["weight"], state["bias"], state["eps"]

    def forward():
        if state["case"]["op"] == "layer_norm":
            return functional.layer_norm(x, weight, bias, eps=eps, out_dtype=state["out"])
        return functional.rms_norm(x, weight, eps=eps, out_dtype=state["out"])

    if not state["case"]["train"]:
        with torch.no_grad():
            return {"out": forward()}
    out = forward()
    leaves = {n: t for n, t in (("dx", x), ("dweight", weight), ("dbias", bias)) if t is not None}
    grads = torch.autograd.grad(out, tuple(leaves.values()), state["grad"])
    return {"out": out.detach(), **dict(zip(leaves, grads))}


@torch.no_grad()
def _plain_attention(state):
    case = state["case"]
    q, k, v, grad = state["q"], state["k"], state["v"], state.get("grad")
    dtype, (heads, width), kv_heads = q.dtype, q.shape[-2:], k.shape[-2]
    group, scale = heads // kv_heads, 1.0 / math.sqrt(width)

    if case["layout"] == "packed":      # the documents as rows of a padded batch
        cu = state["cu_seqlens"].long()
        at = cu[:-1, None] + torch.arange(max(1, state["longest"]), device=q.device)
        real = at < cu[1:, None]
        rows = at.clamp(max=q.shape[0] - 1)
        token = torch.arange(q.shape[0], device=q.device)
        document = torch.searchsorted(cu[1:], token, right=True).clamp(max=len(cu) - 2)
        place = (token - cu[document]).clamp(max=at.shape[1] - 1)
        spread = lambda x: x[rows]
    else:
        length = q.shape[1]
        real = torch.ones(q.shape[:2], dtype=torch.bool, device=q.device)
        if state["lengths"] is not None:
            real = torch.arange(length, device=q.device) < state["lengths"][:, None]
        spread = lambda x: x

    def by_head(x):     # [batch, length, h, width] -> [batch, kv_heads, h / kv_heads, length, width] in 32 bits
        x = spread(x).float()
        x = torch.where(real[:, :, None, None], x, torch.zeros((), device=x.device))
        return x.unflatten(2, (kv_heads, -1)).permute(0, 2, 3, 1, 4).contiguous()

    def back(x):        # the reverse, in the inputs' type; rows of no sequence are zero
        x = x.permute(0, 3, 1, 2, 4).flatten(2, 3)
        x = torch.where(real[:, :, None, None], x, torch.zeros((), device=x.device)).to(dtype)
        if case["layout"] != "packed":
            return x
        return torch.where((token < cu[-1])[:, None, None], x[document, place], torch.zeros((), dtype=dtype, device=x.device))

    qh, kh, vh = by_head(q), by_head(k), by_head(v)
    n = real.shape[1]
    seen = real[:, None, None, None, :]
    if case["causal"]:
        seen = seen & torch.ones(n, n, dtype=torch.bool, device=q.device).tril()
    # the group's heads share their keys: one product over the group's rows
    s = torch.matmul(qh.flatten(2, 3), kh.squeeze(2).transpose(-1, -2)).unflatten(2, (group, n)).mul_(scale)
    s.masked_fill_(~seen, float("-inf"))
    top = s.amax(dim=-1, keepdim=True)
    top = torch.where(torch.isfinite(top), top, torch.zeros((), device=q.device))
    p = s.sub_(top).exp_()
    total = p.sum(dim=-1, keepdim=True)
    p.div_(torch.where(total > 0, total, torch.ones((), device=q.device)))
    result = {"out": back(torch.matmul(p.flatten(2, 3), vh.squeeze(2)).unflatten(2, (group, n)))}
    if grad is None:
        return result
    gh = by_head(grad)
    dv = torch.matmul(p.flatten(2, 3).transpose(-1, -2), gh.flatten(2, 3)).unsqueeze(2)
    dp = torch.matmul(gh.flatten(2, 3), vh.squeeze(2).transpose(-1, -2)).unflatten(2, (group, n))
    ds = dp.sub_((p * dp).sum(dim=-1, keepdim=True)).mul_(p).mul_(scale)
    dq = torch.matmul(ds.flatten(2, 3), kh.squeeze(2)).unflatten(2, (group, n))
    dk = torch.matmul(ds.flatten(2, 3).transpose(-1, -2), qh.flatten(2, 3)).unsqueeze(2)
    return dict(result, dq=back(dq), dk=back(dk), dv=back(dv))


@torch.no_grad()
def _plain_norm(state):
    x, weight, bias, eps = state["x"], state["weight"], state["bias"], state["eps"]
    centred = state["case"]["op"] == "layer_norm"
    xf = x.float()
    if centred:
        xf = xf - xf.mean(dim=-1, keepdim=True)
    rstd = torch.rsqrt((xf * xf).mean(dim=-1, keepdim=True) + eps)
    xhat = xf * rstd
    y = xhat if weight is None else xhat * weight.float()
    if bias is not None:
        y = y + bias.float()
    result = {"out": y.to(state["out"])}
    if not state["case"]["train"]:
        return result
    g = state["grad"].float()
    u = g if weight is None else g * weight.float()
    dx = u - xhat * (u * xhat).mean(dim=-1, keepdim=True)
    if centred:
        dx = dx - u.mean(dim=-1, keepdim=True)
    result["dx"] = (dx * rstd).to(x.dtype)
    if weight is not None:
        result["dweight"] = (g * xhat).sum(dim=0).to(weight.dtype)
    if bias is not None:
        result["dbias"] = g.sum(dim=0).to(bias.dtype)
    return result


# ------------------------------------------------------------------------------------------------
# what a pass cannot do without, and its results in 64 bits
# ------------------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "attention":
        size = _TYPES[case["dtype"]].itemsize
        lengths = _lengths(case, 1)
        tokens = sum(lengths)
        pairs = sum(n * (n + 1) // 2 if case["causal"] else n * n for n in lengths)
        row_q, row_k = case["heads"] * case["width"] * size, case["kv_heads"] * case["width"] * size
        read = tokens * (row_q + 2 * row_k)
        if not case["train"]:
            return {"bytes": read + tokens * row_q, "flops": 4 * pairs * case["heads"] * case["width"]}
        # out, its gradient, dq, dk, dv; products: q k', p v and the backward's q k', do v', p' do, ds k, ds' q
        return {"bytes": read + 2 * tokens * row_q + tokens * (row_q + 2 * row_k), "flops": 14 * pairs * case["heads"] * case["width"]}
    size, out = _TYPES[case["dtype"]].itemsize, _TYPES[case["out"]].itemsize
    n, w = case["rows"] * case["width"], case["width"] * _TYPES[case["weights"]].itemsize * (2 if case["op"] == "layer_norm" else 1)
    w = w if case["affine"] else 0
    if not case["train"]:
        return {"bytes": n * (size + out) + w, "flops": 8 * n}
    return {"bytes": n * (size + out) + n * (size + out) + 2 * w, "flops": 20 * n}


def _exact_sequence(q, k, v, grad, causal):
    """One sequence, every head of one group, in 64 bits by the chain rule of autograd."""
    q, k, v = (x.detach().double().requires_grad_(grad is not None) for x in (q, k, v))
    scores = torch.einsum("thd,sd->hts", q, k) / math.sqrt(q.shape[-1])
    if causal:
        n = q.shape[0]
        scores = scores + torch.triu(torch.full((n, n), float("-inf"), dtype=torch.float64, device=q.device), diagonal=1)
    probabilities = torch.softmax(scores, dim=-1)
    out = torch.einsum("hts,sd->thd", probabilities, v)
    if grad is None:
        return (out,)
    return (out.detach(),) + torch.autograd.grad(out, (q, k, v), grad.double())


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "attention":
        lengths = _lengths(case, seed)
        if sum(n > 0 for n in lengths) * case["kv_heads"] > 4096:
            return None
        q, k, v, grad = state["q"], state["k"], state["v"], state.get("grad")
        names = ["out", "dq", "dk", "dv"] if case["train"] else ["out"]
        result = {n: torch.zeros(t.shape, dtype=torch.float64, device="cuda") for n, t in zip(names, (q, q, k, v))}
        group, start = case["heads"] // case["kv_heads"], 0
        for i, n in enumerate(lengths):
            where = slice(start, start + n) if case["layout"] == "packed" else (i, slice(0, n))
            start += n
            if n == 0:
                continue
            for h in range(case["kv_heads"]):
                of = slice(h * group, (h + 1) * group)
                parts = _exact_sequence(q[where][:, of], k[where][:, h], v[where][:, h], None if grad is None else grad[where][:, of],
                                        case["causal"])
                for name, part in zip(names, parts):
                    result[name][where][:, of if name in ("out", "dq") else h] = part.detach()
        return result
    x, weight, bias = state["x"], state["weight"], state["bias"]
    x64, w64, b64 = (None if t is None else t.detach().double().requires_grad_(case["train"]) for t in (x, weight, bias))
    if case["op"] == "layer_norm":
        y = (x64 - x64.mean(-1, keepdim=True)) / torch.sqrt(x64.var(-1, unbiased=False, keepdim=True) + state["eps"])
    else:
        y = x64 / torch.sqrt(x64.pow(2).mean(-1, keepdim=True) + state["eps"])
    y = y if w64 is None else y * w64
    y = y if b64 is None else y + b64
    if not case["train"]:
        return {"out": y}
    leaves = {n: t for n, t in (("dx", x64), ("dweight", w64), ("dbias", b64)) if t is not None}
    return {"out": y.detach(), **dict(zip(leaves, torch.autograd.grad(y, tuple(leaves.values()), state["grad"].double())))}
