"""bench.py's transformers on the package's own attention and norms (``MODEL_KERNELS``): the operators together, as a model uses them.

Tolerances, normwise.  Every operation of the model returns its result within K E of its norm (E = 2^-24, K <= 256: the longest sums run
over 256 products, one rounding each at worst); a gradient passes at most 60 operations on the way forward and 60 on the way back:
120 * 256 * E = 1.9e-3.  Under bf16 autocast operands are rounded by at most U = 2^-8 each, independently of each other: of 240 such
roundings the root sum of squares is 0.06, allowed 0.1.
"""

import copy

import pytest
import torch

pytestmark = pytest.mark.gpu

MODELS = {
    "gpt2": lambda bench: bench.GPT2(layers=2, width=64, heads=2, vocab=50, positions=70),
    "llama": lambda bench: bench.LlamaSlice(blocks=2, width=128, vocab=50, heads=4, kv_heads=2, inter=256),
    "bert": lambda bench: bench.Bert(layers=2, width=64, heads=4, inter=128, vocab=50, positions=70),
}


def rel(got, want):
    return float((got.double().cpu() - want.double().cpu()).norm() / want.double().cpu().norm())


def parts(bench, kind):
    if kind == "bert":
        return bench.synth_glue(dict(vocab=50, tokens=67), 9, 3, "cpu"), bench.glue_loss
    return bench.synth_tokens(dict(vocab=50, tokens=67), 5, 3, "cpu"), bench.lm_loss


def passes(model, batch, loss):
    value = loss(model, batch)
    names, leaves = zip(*[(n, p) for n, p in model.named_parameters() if p.requires_grad])
    return value.detach(), dict(zip(names, torch.autograd.grad(value, leaves, allow_unused=True)))


@pytest.mark.parametrize("amp", [False, True])
@pytest.mark.parametrize("kind", sorted(MODELS))
def test_loss_and_every_gradient_against_64_bits(kind, amp, monkeypatch):
    import bench
    from kronfluence_amd.module.norm import FusedLayerNorm, FusedRMSNorm
    from kronfluence_amd.utils.model import apply_fused_norms

    torch.manual_seed(0)
    plain = MODELS[kind](bench)
    for name, p in plain.named_parameters():   # norms with weights of their own
        if "ln" in name or "norm" in name:
            p.data += 0.2 * torch.randn_like(p)
    batch, loss = parts(bench, kind)
    want, want_grads = passes(copy.deepcopy(plain).double(), batch, loss)
    monkeypatch.setattr(bench, "MODEL_KERNELS", True)
    model = apply_fused_norms(plain.cuda())
    assert not any(type(m) in (torch.nn.LayerNorm, torch.nn.RMSNorm) for m in model.modules())
    assert any(isinstance(m, (FusedLayerNorm, FusedRMSNorm)) for m in model.modules())
    batch = tuple(t.cuda() for t in batch)
    with torch.autocast("cuda", torch.bfloat16, enabled=amp):
        got, grads = passes(model, batch, loss)
    bound = 0.1 if amp else 1.9e-3
    assert rel(got, want) <= bound
    top = max(float(g.norm()) for g in want_grads.values() if g is not None)
    for name, g in want_grads.items():
        if g is None:
            assert grads[name] is None, name
        else:   # (a key bias moves no score, its gradient is rounding alone: measured against the largest gradient)
            assert float((grads[name].double().cpu() - g).norm()) <= bound * max(float(g.norm()), 1e-2 * top), name


@pytest.mark.parametrize("kind", ["gpt2", "bert"])
def test_scores_through_every_stage_and_the_captured_train_pass(kind, tmp_path, monkeypatch):
    """Covariances and pairwise scores with the package's kernels against torch's in the same model (fp32: the bound above, doubled for
    the two sides, times 2 or 4 for the products of two activations or gradients a covariance, of four gradients a score is made of); the
    scores on one set of factors, the train pass eager and replayed from a graph."""
    import bench
    from kronfluence_amd import Analyzer, FactorArguments, ScoreArguments, prepare_model
    from kronfluence_amd.score import dot_product
    from kronfluence_amd.utils.model import apply_fused_norms
    from torch.utils import data

    spec = dict(vocab=50, tokens=67)
    make = bench.synth_glue if kind == "bert" else bench.synth_tokens
    train, query = (data.TensorDataset(*make(spec, n, seed, "cpu")) for n, seed in ((67, 1), (5, 2)))

    def analyzer(own):
        monkeypatch.setattr(bench, "MODEL_KERNELS", own)
        torch.manual_seed(0)
        raw = MODELS[kind](bench)
        task = bench.make_glue_task() if kind == "bert" else bench.make_lm_task(raw.tracked_names())
        model = prepare_model(raw, task)
        return Analyzer("m", apply_fused_norms(model) if own else model, task, output_dir=str(tmp_path), disable_tqdm=True)

    def scores(own, mode):
        monkeypatch.setenv("KF_TRAIN_GRAPH", mode)
        for key in ("captures", "replays", "fallbacks"):
            dot_product.GRAPH_LOG[key] = 0
        out = analyzer(own).compute_pairwise_scores(
            f"s{own}{mode}", "torch", query, train, per_device_query_batch_size=3, per_device_train_batch_size=8,
            score_args=ScoreArguments(damping_factor=None, query_gradient_accumulation_steps=64))
        return out["all_modules"], dict(dot_product.GRAPH_LOG)

    fargs = FactorArguments(use_empirical_fisher=True)
    analyzer(False).fit_all_factors("torch", train, per_device_batch_size=8, factor_args=fargs)
    mine = analyzer(True)
    mine.fit_covariance_matrices("own", train, per_device_batch_size=8, factor_args=fargs)
    theirs, ours = mine.load_covariance_matrices("torch"), mine.load_covariance_matrices("own")
    for key in ("activation_covariance", "gradient_covariance"):
        top = max(float(c.norm()) for c in theirs[key].values())
        for name, c in theirs[key].items():
            assert float((ours[key][name] - c).norm()) <= 2 * 2 * 1.9e-3 * max(float(c.norm()), 1e-4 * top), (key, name)

    want, _ = scores(False, "0")
    eager, _ = scores(True, "0")
    replayed, log = scores(True, "1")
    assert log["captures"] == 1 and log["replays"] == 7 and log["fallbacks"] == 0, log   # 8 whole batches, the ragged ninth eager
    assert rel(eager, want) <= 2 * 4 * 1.9e-3, rel(eager, want)
    assert rel(replayed, eager) <= 2e-6, rel(replayed, eager)   # the same kernels on the same inputs; only the score sums' order may differ


@pytest.mark.parametrize("amp", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_fused_norms_return_what_the_torch_modules_return(dtype, amp):
    """Types and default epsilon (rows so small that it is most of the denominator); values to the output type's rounding, one step apart
    at most where both sides round once, plus the fp32 errors of 8 terms."""
    from torch import nn

    from kronfluence_amd.module.norm import fused

    x = 3e-4 * torch.randn(5, 8, generator=torch.Generator().manual_seed(2)).cuda().to(dtype)
    for module in (nn.LayerNorm(8), nn.RMSNorm(8), nn.RMSNorm(8, elementwise_affine=False), nn.LayerNorm(8, bias=False)):
        module = module.cuda().to(dtype)
        with torch.autocast("cuda", torch.bfloat16, enabled=amp):
            want, got = module(x).detach(), fused(module)(x).detach()
        assert got.dtype == want.dtype, (module, got.dtype, want.dtype)
        step = 2 * 2.0 ** -8 if want.dtype == torch.bfloat16 else 32 * 2.0 ** -24
        assert float((got.float() - want.float()).abs().max()) <= step * float(want.float().abs().max()), module
