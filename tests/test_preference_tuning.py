"""Preference tuning as a whole: the steps and the wrapper of ``train.finetune`` on a small model (CPU and GPU), and the operators of one step in a
row (embedding with sorted gradients, kept feed-forward block, kept linear layer, losses) against the same in 64 bits."""
import copy
import math

import pytest
import torch

from nmtgminor_b200 import ops
from nmtgminor_b200.data.synthetic import synthetic_dict, token_budget_batches
from nmtgminor_b200.models.factory import build_model
from nmtgminor_b200.ops import kept, preference as pref
from nmtgminor_b200.options import default_options
from nmtgminor_b200.parallel.flat import FlatParameterStore
from nmtgminor_b200.train import finetune as FT
from nmtgminor_b200.train.engine import TrainEngine


def _options(extra=()):
    return default_options(["-model_size", "64", "-layers", "2", "-n_heads", "2", "-inner_size", "256", "-tie_weights", "-join_embedding", "-dropout", "0.0",
                            "-attn_dropout", "0.0", "-emb_dropout", "0.0", "-optim", "adam", "-learning_rate", "0.002", "-update_method",
                            "regular"] + list(extra))


def _model(seed=0, words=300, extra=()):
    torch.manual_seed(seed)
    d = synthetic_dict(words)
    return build_model(_options(extra), {"src": d, "tgt": d})


def _batch(words=300, tokens=400):
    for seed in range(1, 50):
        b = token_budget_batches(words, 4, 20, tokens, 1, seed=seed, padded=False)[0]
        if (b.packed_target_input().cu.numel() - 1) % 2 == 0:
            return b
    raise AssertionError("no batch of pairs")


def test_a_model_against_itself():
    """With the frozen model's weights: h = 0 but for rounding, so log 2 a pair; ratios 1, so minus the advantages of the words, no KL, nothing clipped."""
    model, batch = _model(), _batch()
    wrapper = FT.PreferenceWrapper(model, copy.deepcopy(model), beta=0.3).train()
    assert len(list(wrapper.parameters())) == len(list(model.parameters()))
    out = wrapper(batch)
    pairs = out["scores"].shape[0] // 2
    # the wrapper's two sums of a sentence's words are taken in 32 and in 64 bits: apart by 2^-24 of the sum for each of 20 words at most, which the
    # loss has half beta of for each sentence (and the order of a pair is then open)
    off = 20 * 2 ** -24 * out["scores"].abs()
    assert ((out["scores"] - out["reference_scores"]).abs() <= off).all()
    assert abs(out["loss"].item() - pairs * math.log(2.0)) <= 0.5 * 0.3 * off.sum() + 2 ** -20 * pairs
    lp, cu = FT.word_scores(model, batch)
    advantages = torch.randn(cu.numel() - 1, generator=torch.Generator().manual_seed(1))
    loss, clipped, kl, _ = FT.policy_step(model, batch, lp, advantages, lp, kl_coef=0.1)
    words = (batch.packed_target_output() != 0).float()
    each = torch.cat([a.expand(n) for a, n in zip(advantages, (cu[1:] - cu[:-1]).tolist())])
    want = -(each * words[:each.shape[0]]).sum()
    assert abs(loss.item() - want.item()) <= 2 ** -20 * each.abs().sum() and clipped.item() == 0 and kl.item() == 0
    assert "loss" in wrapper.eval()(batch)


def test_gradients_of_the_steps():
    """A step's gradient of the parameters is that of the loss written over the logits of the model."""
    model, batch = _model(extra=["-ffn_keep8"]), _batch()
    frozen = _model(1).eval()
    params = list(model.parameters())
    ref = FT.sentence_scores(frozen, batch)
    got = torch.autograd.grad(FT.preference_step(model, batch, ref, beta=0.2, kind="hinge")[0], params, allow_unused=True)
    logits, labels, cu = FT.packed_logits(model, batch)
    want = torch.autograd.grad(pref.preference_loss_reference(logits, labels, cu, ref, beta=0.2, kind="hinge")[0], params, allow_unused=True)
    assert any(g is not None and g.abs().sum() > 0 for g in got)
    for g, w in zip(got, want):
        assert (g is None) == (w is None) and (g is None or torch.equal(g, w))


def test_wrapper_trains_through_the_engine():
    model = _model(extra=["-ffn_keep8"])
    engine = TrainEngine(FT.PreferenceWrapper(model, _model(1), beta=0.5), _options(), device="cpu")
    for _ in range(3):
        loss, ranked = engine.train_step(_batch())
        assert torch.isfinite(loss).all() and ranked.item() >= 0
    assert all(torch.isfinite(p).all() for p in model.parameters())


def test_what_is_refused():
    model, batch = _model(), _batch()
    for seed in range(1, 50):
        odd = token_budget_batches(300, 4, 20, 400, 1, seed=seed, padded=False)[0]
        if (odd.packed_target_input().cu.numel() - 1) % 2:
            break
    with pytest.raises(ValueError):
        FT.preference_step(model, odd)
    lp, cu = FT.word_scores(model, batch)
    with pytest.raises(ValueError):
        FT.policy_step(model, batch, lp, torch.ones(cu.numel()))
    for extra in (["-ffn_glu"], ["-weight_drop", "0.1"]):
        with pytest.raises(NotImplementedError):
            _model(extra=["-ffn_keep8"] + extra)


# ---------------------------------------------------------------------------------------------------------------------
# GPU
# ---------------------------------------------------------------------------------------------------------------------
class _Rounded(torch.autograd.Function):
    """To bf16 and back, values and gradients."""

    @staticmethod
    def forward(ctx, x):
        return x.bfloat16().to(x.dtype)

    @staticmethod
    def backward(ctx, g):
        return g.bfloat16().to(g.dtype)


def _norm_close(got, want, share, name):
    error = (got.double() - want).norm()
    assert error <= share * want.norm(), (name, (error / want.norm()).item())


def _flat(value):
    p = torch.nn.Parameter(value.float().cuda())
    p.work, p.main_grad = value.bfloat16().cuda(), torch.zeros(value.shape, device="cuda")
    return p


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["preference", "policy"])
@pytest.mark.parametrize("rows,words,width,inner", [(47, 301, 64, 160), (900, 9001, 256, 1024)])
def test_the_operators_of_a_step_in_a_row(which, rows, words, width, inner):
    """Table, block, layer and loss in the flat store's manner, two steps into the same buffers.  Each operator's results, forward and backward, are held
    against 64 bits from the bf16 matrices that the operators before and behind it left, so that a code or a sign turned over by an earlier
    rounding does not count.  Matrices in bf16 are then off by their rounding (rms 2^-9.8 of the norm) and, inside the block, by one more of the hidden
    gradient; a code that turns over because 32 bits and 64 round to two bf16 neighbours is one of 2^10, by 2^-3.5, 2^-8.5 of the norm: 2^-8 + 2^-9 in
    all.  The table's gradient has 32-bit sums of what it gets."""
    g = torch.Generator().manual_seed(rows)
    bf = lambda *shape: torch.randn(*shape, generator=g).bfloat16()
    values = {"table": bf(words, width) / width ** 0.5, "w1": bf(inner, width) / width ** 0.5, "b1": bf(inner) * 0.1, "w2": bf(width, inner) / inner ** 0.5,
              "b2": bf(width) * 0.1, "w3": bf(width, width) / width ** 0.5, "b3": bf(width) * 0.1, "out": bf(words, width) * (1.5 / width ** 0.5)}
    values = {k: v.bfloat16() for k, v in values.items()}
    tokens = torch.randint(1, words, (rows,), generator=g)
    tokens[::7] = 5
    tokens[3] = 0
    labels = torch.randint(1, words, (rows,), generator=g)
    labels[2:6] = 0
    cu = torch.tensor([0, rows // 5, rows // 3, rows // 3, rows - 4]).int()
    other = torch.randn(4, generator=g) * 5 - 8.0 * rows / 4
    old, adv = torch.randn(rows, generator=g) * 0.1 - math.log(words), torch.randn(rows, generator=g)

    def lost(logits, labels, cu, other, old, adv, **kw):
        if which == "preference":
            return pref.preference_loss(logits, labels, cu, other, beta=0.01, average=True, **kw)[0]
        return pref.policy_loss(logits, labels, old, adv, old, clip=0.9, clip_high=50.0, kl_coef=0.01, **kw)[0]

    def block(x, p):                           # in 64 bits, with the matrices that the kernels leave in bf16 rounded
        z = _Rounded.apply(kept.linear_reference(x, p["w1"], p["b1"]))
        y = torch.nn.functional.linear(_Rounded.apply(kept.act_reference(z, 2)), p["w2"].detach(), p["b2"]) + x
        again = kept.act_reference(kept.restore_reference(kept.quantise_reference(z.detach())).to(z.dtype), 2)
        term = torch.nn.functional.linear(_Rounded.apply(again), p["w2"])
        return y + (term - term.detach())

    flat = {k: _flat(v) for k, v in values.items()}
    there = [t.cuda() for t in (tokens, labels, cu, other, old, adv)]
    share = 2 ** -8 + 2 ** -9
    for n in (1, 2):
        x0 = ops.embedding(there[0], flat["table"], scale=width ** 0.5, pad_idx=0, sorted_grad=True)
        x1 = ops.mlp(x0, flat["w1"], flat["b1"], flat["w2"], flat["b2"], "gelu", 0.0, 0.0, x0, True, keep8=True)
        x2 = ops.linear(x1, flat["w3"], flat["b3"], "relu", 0.0, x1, True, keep8=True)
        logits = ops.linear(x2, flat["out"], None, "none", 0.0, None, True, keep8=True)
        kept_logits = logits.detach().clone()
        for t in (x0, x1, x2, logits):
            t.retain_grad()
        loss = lost(logits, *there[1:], inplace=True)
        loss.backward()
        wide = {k: v.double().cuda().requires_grad_(True) for k, v in values.items()}
        given = {k: t.detach().double().requires_grad_(True) for k, t in (("x0", x0), ("x1", x1), ("x2", x2), ("logits", kept_logits))}
        want = {"x0": ops.embedding(there[0], wide["table"], scale=width ** 0.5, pad_idx=0), "x1": block(given["x0"], wide),
                "x2": ops.linear(given["x1"], wide["w3"], wide["b3"], "relu", 0.0, given["x1"], True, keep8=True),
                "logits": ops.linear(given["x2"], wide["out"], None, "none", 0.0, None, True, keep8=True)}
        want_loss = lost(given["logits"], *there[1:4], *(t.double() for t in there[4:]))
        want_loss.backward()
        for name, got in (("logits", logits), ("x2", x2), ("x1", x1), ("x0", x0)):
            _norm_close(kept_logits if name == "logits" else got.detach(), want[name].detach(), share, name)
            grad = got.grad.double()
            if name == "x0":
                grad[there[0] == 0] = 0.0                                        # padding has no gradient
            want[name].backward(grad)
        # a log-probability is off by 2^-19 and its rounding, the loss by what it makes of that
        assert abs(loss.item() - want_loss.item()) <= 2 ** -14 * max(abs(want_loss.item()), rows ** 0.5)
        for name, got in (("logits", logits), ("x2", x2), ("x1", x1), ("x0", x0)):
            _norm_close(got.grad, given[name].grad, share, "gradient of " + name)
        for name, p in flat.items():
            _norm_close(p.main_grad, n * wide[name].grad, 2 ** -20 if name == "table" else share, "gradient of " + name)
    assert (flat["table"].main_grad[0] == 0).all() and ops.check_status() == 0


@pytest.mark.gpu
def test_wrapper_trains_through_a_captured_step():
    """The engine's captured step and its steps kernel by kernel: the first loss is log 2 a pair for a model and
    its copy, and the same in both."""
    batch = token_budget_batches(300, 4, 20, 400, 1, seed=3, static=True, padded=False)[0].pin_memory()
    if (batch.packed_target_input().cu.numel() - 1) % 2:
        batch = _batch().pin_memory()
    losses = []
    torch.use_deterministic_algorithms(True, warn_only=True)
    try:
        for graph in (False, True):
            model = _model(extra=["-ffn_keep8"])
            frozen = copy.deepcopy(model)
            assert not FT.PreferenceWrapper(model, frozen).graph_capturable and FT.PreferenceWrapper(model).graph_capturable
            FlatParameterStore(frozen, "cuda")
            for b in frozen.buffers():
                b.data = b.data.cuda()
            engine = TrainEngine(FT.PreferenceWrapper(model, frozen, beta=0.5), _options(), device="cuda", cuda_graph=graph)
            losses.append([engine.train_step(batch)[0].item() for _ in range(6)])
            assert bool(engine._graphs) == graph
            torch.cuda.synchronize()
    finally:
        torch.use_deterministic_algorithms(False)
    pairs = (batch.packed_target_input().cu.numel() - 1) // 2
    for run in losses:
        assert all(math.isfinite(v) for v in run)
        # both models' logits are the same numbers, and so are the words' scores; a sentence's sum is rounded once for the frozen one (2^-24 of at most 20
        # words of 2^4 each), times beta and the slope of 1 / 2
        assert abs(run[0] - pairs * math.log(2.0)) <= 2 ** -16 * pairs
    assert ops.check_status() == 0


@pytest.mark.gpu
def test_a_captured_pass_beside_a_living_eager_graph():
    """The flat store's chain has no leaf in common with other calls: its backward pass is captured while an eager graph of the same parameters lives."""
    g = torch.Generator().manual_seed(4)
    table, w, out = (_flat(torch.randn(*shape, generator=g).bfloat16() * 0.1) for shape in ((300, 64), (128, 64), (300, 128)))
    tokens, labels = (torch.randint(1, 300, (90,), generator=g).cuda() for _ in range(2))
    cu = torch.tensor([0, 30, 50, 70, 90]).int().cuda()

    def forward():
        x = ops.embedding(tokens, table, sorted_grad=True)
        return pref.preference_loss(ops.linear(ops.linear(x, w, None, "relu", keep8=True), out, keep8=True), labels, cu, inplace=True)[0]

    def step():
        for p in (table, w, out):
            p.main_grad.zero_()
        loss = forward()
        loss.backward()
        return loss.detach()

    alive = forward()
    want, grads = step().clone(), [p.main_grad.clone() for p in (table, w, out)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = step()
    for p in (table, w, out):
        p.main_grad.fill_(7.0)
    graph.replay()
    assert torch.equal(loss, want)
    for p, grad in zip((table, w, out), grads):
        assert (p.main_grad - grad).norm() <= 2 ** -16 * grad.norm()        # split sums are added in any order
    alive.backward()
    assert ops.check_status() == 0
