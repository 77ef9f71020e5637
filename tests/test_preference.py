"""Losses of preference tuning: the plain restatements against formulas written out and against differences (CPU), the kernels against the
restatements in 64 bits (GPU)."""
import math

import pytest
import torch

from nmtgminor_b200 import ops
from nmtgminor_b200.ops import preference as pref

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---------------------------------------------------------------------------------------------------------------------
# CPU
# ---------------------------------------------------------------------------------------------------------------------
def _small(seed=0, rows=11, vocab=7):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, vocab, generator=g, dtype=torch.float64) * 2
    y = torch.randint(1, vocab, (rows,), generator=g)
    y[3] = 0
    return g, x, y


def test_logprobs_of_words_and_sequences():
    _, x, y = _small()
    lp = pref.token_logprobs(x, y, temperature=0.7)
    for r in range(len(y)):
        want = 0.0 if y[r] == 0 else float(torch.log(torch.softmax(x[r] / 0.7, 0)[y[r]]))
        assert abs(float(lp[r]) - want) < 1e-12
    cu = torch.tensor([0, 4, 4, 9])
    s = pref.sequence_logprobs(lp, cu)
    assert torch.allclose(s, torch.stack([lp[0:4].sum(), lp.new_zeros(()), lp[4:9].sum()]), atol=1e-12)


@pytest.mark.parametrize("kind,smoothing,margin,nll,average", [("sigmoid", 0.0, 0.0, 0.0, False), ("sigmoid", 0.1, 0.3, 0.2, True),
                                                               ("hinge", 0.0, 0.2, 0.0, False), ("ipo", 0.0, 0.0, 0.5, True)])
def test_preference_loss_written_out(kind, smoothing, margin, nll, average):
    g, x, y = _small(1, rows=12)
    cu = torch.tensor([0, 3, 5, 5, 9], dtype=torch.int32)        # pair 1 has an empty preferred sequence; rows 9.. are outside
    r = torch.randn(4, generator=g, dtype=torch.float64)
    beta = 0.4
    loss, ranked, scores = pref.preference_loss(x, y, cu, r, beta, kind, smoothing, margin, nll, average)
    lp = [0.0 if y[i] == 0 else float(torch.log_softmax(x[i], 0)[y[i]]) for i in range(12)]
    want, n_ranked = 0.0, 0
    for p in range(2):
        s, c = [], []
        for q in (2 * p, 2 * p + 1):
            a, b = int(cu[q]), int(cu[q + 1])
            s.append(sum(lp[a:b]))
            c.append(max(1, sum(int(y[i] != 0) for i in range(a, b))) if average else 1)
            assert abs(float(scores[q]) - s[-1]) < 1e-12
        h = (s[0] - float(r[2 * p])) / c[0] - (s[1] - float(r[2 * p + 1])) / c[1]
        z = beta * h - margin
        sig = 1 / (1 + math.exp(-z))
        want += {"sigmoid": -(1 - smoothing) * math.log(sig) - smoothing * math.log(1 - sig), "hinge": max(0.0, 1 - z),
                 "ipo": (h - 0.5 / beta) ** 2}[kind] - nll * s[0] / c[0]
        n_ranked += h > 0
    assert abs(float(loss) - want) < 1e-10 and int(ranked) == n_ranked


def test_policy_loss_written_out():
    g, x, y = _small(2)
    old, adv, r = (torch.randn(11, generator=g, dtype=torch.float64) for _ in range(3))
    old, r = old - 2, r * 0.3 - 2
    loss, clipped, kl, lp = pref.policy_loss(x, y, old, adv, r, clip=0.1, clip_high=0.3, kl_coef=0.2)
    want, n, k = 0.0, 0, 0.0
    for i in range(11):
        if y[i] == 0:
            continue
        l = float(torch.log_softmax(x[i], 0)[y[i]])
        ratio, a, d = math.exp(l - float(old[i])), float(adv[i]), float(r[i]) - l
        held = min(max(ratio, 0.9), 1.3)
        want += -min(ratio * a, held * a) + 0.2 * (math.exp(d) - d - 1)
        n += ratio * a > held * a
        k += math.exp(d) - d - 1
    assert abs(float(loss) - want) < 1e-9 and int(clipped) == n and abs(float(kl) - k) < 1e-9 and float(lp[3]) == 0.0


def test_gradients_of_the_restatements_against_differences():
    g, x, y = _small(3, rows=6, vocab=4)
    x.requires_grad_(True)
    cu = torch.tensor([0, 2, 3, 5, 6])
    v = torch.randn(6, generator=g, dtype=torch.float64) * 0.3
    assert torch.autograd.gradcheck(lambda t: pref.token_logprobs(t, y, temperature=1.3), (x,))
    for kind in pref.KINDS:
        assert torch.autograd.gradcheck(lambda t: pref.preference_loss(t, y, cu, v[:4], 0.7, kind, nll_weight=0.1, average=True)[0], (x,))
    assert torch.autograd.gradcheck(lambda t: pref.policy_loss(t, y, v - 1.5, v, v - 1.4, kl_coef=0.3)[0], (x,))


def test_grad_scale_on_the_cpu():
    g, x, y = _small(4)
    cu = torch.tensor([0, 5, 10])
    for scale in (0.25, torch.tensor([0.25])):
        a, b = x.float().requires_grad_(True), x.float().requires_grad_(True)
        pref.preference_loss(a, y, cu)[0].backward()
        pref.preference_loss(b, y, cu, grad_scale=scale)[0].backward()
        assert torch.allclose(b.grad, 0.25 * a.grad)


def _refusals(device):
    x, y = torch.randn(6, 5, device=device), torch.ones(6, dtype=torch.int64, device=device)
    cu, v = torch.tensor([0, 3, 6], device=device), torch.zeros(6, device=device)
    bad = [
        lambda: pref.token_logprobs(x[0], y), lambda: pref.token_logprobs(x, y[:5]), lambda: pref.token_logprobs(x[:, :0], y),
        lambda: pref.token_logprobs(x, y, temperature=0.0), lambda: pref.token_logprobs(x, y, temperature=float("inf")),
        lambda: pref.token_logprobs(x, y, temperature=float("nan")), lambda: pref.token_logprobs(x, y.float()),
        lambda: pref.token_logprobs(x.long(), y),
        lambda: pref.preference_loss(x, y, cu[:2]), lambda: pref.preference_loss(x, y, cu.float()),
        lambda: pref.preference_loss(x, y, cu, v[:3]), lambda: pref.preference_loss(x, y, cu, beta=0.0),
        lambda: pref.preference_loss(x, y, cu, kind="square"), lambda: pref.preference_loss(x, y, cu, smoothing=1.0),
        lambda: pref.preference_loss(x, y, cu, kind="hinge", smoothing=0.1), lambda: pref.preference_loss(x, y, cu, kind="ipo", margin=1.0),
        lambda: pref.preference_loss(x, y, cu, v[:2].clone().requires_grad_(True)),
        lambda: pref.policy_loss(x, y, v[:5], v), lambda: pref.policy_loss(x, y, v, v[:, None]), lambda: pref.policy_loss(x, y, v, v, clip=1.5),
        lambda: pref.policy_loss(x, y, v, v, clip_high=-0.1), lambda: pref.policy_loss(x, y, v, v, kl_coef=0.1),
        lambda: pref.policy_loss(x, y, v.clone().requires_grad_(True), v), lambda: pref.policy_loss(x, y, v, v, v[:2]),
        lambda: pref.policy_loss(x, y, v, v, grad_scale=torch.ones(2, device=device)),
    ]
    for f in bad:
        with pytest.raises((ValueError, TypeError)):
            f()
    if device != "cpu":
        for f in (lambda: pref.token_logprobs(x, y.cpu()), lambda: pref.preference_loss(x, y, cu.cpu()),
                  lambda: pref.policy_loss(x, y, v.cpu(), v), lambda: pref.policy_loss(x, y, v, v, grad_scale=torch.ones(1))):
            with pytest.raises(ValueError):
                f()


def test_refusals_on_the_cpu():
    _refusals("cpu")


# ---------------------------------------------------------------------------------------------------------------------
# GPU
# ---------------------------------------------------------------------------------------------------------------------
# words: every block size, clusters of 2, 4 and 8, rows that no cluster holds; odd ones, and fewer than a vector
VOCABS = [1, 3, 8, 37, 1000, 1024, 1025, 4093, 8000, 9001, 16390, 32000, 32768, 51865, 70001, 131073, 250054, 262144, 270005]


def _logits(rows, vocab, kind, layout, seed=0, spread=2.5):
    """dense: rows one after another; padded: rows 16-byte aligned; odd: rows and start off every alignment but the element's."""
    g = torch.Generator().manual_seed(seed + rows + vocab)
    dtype = TYPES[kind]
    width = {"dense": vocab, "padded": (vocab + 7) // 8 * 8, "odd": vocab + 3}[layout]
    skip = 5 if layout == "odd" else 0
    flat = torch.empty(rows * width + skip, dtype=dtype, device=DEV)
    x = flat[skip:].view(rows, width)[:, :vocab]
    x.copy_((torch.randn(rows, vocab, generator=g) * spread).to(DEV))
    y = torch.randint(0, vocab, (rows,), generator=g).to(DEV)
    if rows > 3:
        y[1], y[2], y[3] = 0, -5, vocab + 2          # padding, and two that are no words
    if rows > 4:
        y[4] = vocab - 1
    favour = (torch.rand(rows, generator=g) * 10).to(DEV)
    inside = (y >= 0) & (y < vocab)
    x[inside, y[inside]] += favour[inside].to(dtype)
    return x, y


def _logprobs_close(got, want):
    """exp2 is off by 2^-22, its argument by 2^-24 of itself (below 64 where it counts), the sum of a row by a few roundings more: 2^-19 of
    the sum in all, which is so much of the log-probability; then one rounding of the result."""
    assert ((got.double() - want).abs() <= 2 ** -19 + 2 ** -23 * want.abs()).all(), (got.double() - want).abs().max()


def _grads_close(got, want, coef, kind):
    """The rounding of the result (half a step of the type; of fp16 also half its smallest number), and in 32 bits before it 2^-16 of the
    exponential (argument as above, sum, coefficient); at the label coef (1 - p) is off by that share of coef."""
    half = {"bf16": 2 ** -8, "fp16": 2 ** -11, "fp32": 2 ** -24}[kind]
    bound = (half + 2 ** -16) * want.abs() + (2 ** -25 if kind == "fp16" else 0.0)
    err = (got.double() - want).abs()
    bad = err > bound
    if bad.any():       # labels only
        rows = bad.any(1)
        assert (bad.sum(1) <= 1).all()
        assert (err.amax(1)[rows] <= half * want.abs().amax(1)[rows] + 2 ** -16 * coef.double().abs()[rows]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["dense", "padded", "odd"])
@pytest.mark.parametrize("kind", ["bf16", "fp16", "fp32"])
def test_token_logprobs(kind, layout):
    for vocab in VOCABS:
        for rows in (1, 7) if vocab > 9001 else (1, 7, 300):
            x, y = _logits(rows, vocab, kind, layout)
            xd = x.double().requires_grad_(True)
            want = pref.token_logprobs(xd, y, temperature=1.25)
            leaf = x.detach().requires_grad_(True)
            got = pref.token_logprobs(leaf, y, temperature=1.25)
            weight = torch.randn(rows, generator=torch.Generator().manual_seed(vocab)).to(DEV)
            _logprobs_close(got.detach(), want.detach())
            with torch.no_grad():
                assert torch.equal(pref.token_logprobs(x, y, temperature=1.25), got)
            grad = torch.autograd.grad(got, leaf, weight)[0]
            _grads_close(grad, torch.autograd.grad(want, xd, weight.double())[0], weight, kind)
            assert grad.stride() == x.stride() or rows == 1
    assert ops.check_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "fp32"])
def test_masked_logits(kind):
    """-inf and the type's lowest value in most places, in all but the label's, in the label's own, everywhere; NaN and +inf."""
    dtype = TYPES[kind]
    low = torch.finfo(dtype).min
    for vocab in (40, 5000, 70001):
        x, _ = _logits(12, vocab, kind, "padded")
        y = torch.full((12,), 2, device=DEV)
        x[0, 10:] = -math.inf
        x[1, 10:] = low
        x[2] = -math.inf
        x[2, 2] = 1.0
        x[3] = low
        x[3, 2] = 1.0
        x[4, 2] = -math.inf
        x[5, 2] = low
        x[6] = low                      # nothing left, by the lowest value: every word alike
        x[7] = -math.inf                # nothing left: NaN
        x[8, 7] = math.nan
        x[9, 7] = math.inf
        leaf = x.detach().requires_grad_(True)
        got = pref.token_logprobs(leaf, y)
        grad = torch.autograd.grad(got.sum(), leaf)[0]
        xd = x.double().requires_grad_(True)
        want = torch.log_softmax(xd, 1)[:, 2]
        wgrad = torch.autograd.grad(want[:7].sum(), xd)[0]
        rows = [0, 1, 2, 3, 6, 10, 11]
        _logprobs_close(got.detach()[rows], want.detach()[rows])
        assert got[4] == -math.inf and got[5] < -1e38
        _grads_close(grad[:7], wgrad[:7], torch.ones(7, device=DEV), kind)
        assert torch.isnan(got[7:10]).all()
        assert torch.isnan(grad[7]).all() and torch.isnan(grad[8]).all()


def _pairs(lengths, vocab, kind, layout, extra=0, seed=0):
    cu = torch.tensor([0] + lengths).cumsum(0).int().to(DEV)
    x, y = _logits(sum(lengths) + extra, vocab, kind, layout, seed)
    g = torch.Generator().manual_seed(seed + 1)
    lp = pref.token_logprobs(x.double(), y)
    r = (pref.sequence_logprobs(lp, cu) + 5 * torch.randn(len(lengths), generator=g).to(DEV).double()).float()
    return x, y, cu, r


def _coefs(x, y, f):
    """d loss / d log-probability of the rows, in 64 bits: f is a loss of logits, whose gradient is coef * (onehot - p) with some p < 1."""
    xd = x.double().requires_grad_(True)
    loss = f(xd)
    return loss, torch.autograd.grad(loss[0], xd)[0]


LENGTHS = {"one": [5, 9], "few": [3, 1, 0, 6, 40, 17, 0, 0, 8, 0], "many": [1 + (7 * i) % 29 for i in range(120)], "long": [700, 3, 2, 900]}


@pytest.mark.gpu
@pytest.mark.parametrize("kind,layout", [("bf16", "padded"), ("bf16", "odd"), ("fp16", "dense"), ("fp32", "dense")])
@pytest.mark.parametrize("lengths", list(LENGTHS))
def test_preference_loss(kind, layout, lengths):
    for vocab in (37, 3000, 9001, 40001) if lengths != "many" else (37, 3000):
        x, y, cu, r = _pairs(LENGTHS[lengths], vocab, kind, layout, extra=4)
        for cfg in ({}, {"kind": "hinge", "margin": 0.5, "beta": 0.3}, {"kind": "ipo", "average": True, "beta": 0.5, "nll_weight": 0.1},
                    {"smoothing": 0.1, "average": True, "nll_weight": 0.3, "temperature": 0.8}):
            (loss, ranked, scores), grad = _coefs(x, y, lambda t: pref.preference_loss(t, y, cu, r, **cfg))
            leaf = x.detach().requires_grad_(True)
            got = pref.preference_loss(leaf, y, cu, r, **cfg)
            mine = torch.autograd.grad(got[0], leaf)[0]
            n = x.shape[0]
            assert ((got[2].double() - scores).abs() <= n * 2 ** -19 + 2 ** -22 * scores.abs()).all()
            assert got[1].item() == ranked.item()
            slope = 2 * (scores.abs().max() + 40) if cfg.get("kind") == "ipo" else 1.0
            assert abs(got[0].item() - loss.item()) <= 1e-6 * abs(loss.item()) + slope * n * 2 ** -18
            # a coefficient follows the scores: its own error is below 1e-4 of itself, or of the largest where it is a difference
            top = grad.abs().amax(1)
            half = {"bf16": 2 ** -8, "fp16": 2 ** -11, "fp32": 2 ** -24}[kind]
            err = (mine.double() - grad).abs()
            scale = max(1.0, float(slope))
            assert (err <= (half + 1e-4) * grad.abs() + 2 ** -24 + 2e-5 * scale * (1 if cfg.get("kind") == "ipo" else cfg.get("beta", 0.1) + 1)).all()
            assert (mine[sum(LENGTHS[lengths]):] == 0).all() and (top >= 0).all()
            with torch.no_grad():
                again = pref.preference_loss(x, y, cu, r, **cfg)
            assert all(torch.equal(a, b) for a, b in zip(again, got))
            # the same rows at the same addresses modulo 16 give the same bits (a row's elements are dealt out by its alignment)
            assert torch.equal(torch.autograd.grad(pref.preference_loss(leaf, y, cu, r, **cfg)[0], leaf)[0], mine)
    assert ops.check_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("kind,layout", [("bf16", "padded"), ("bf16", "odd"), ("fp16", "dense"), ("fp32", "padded")])
@pytest.mark.parametrize("vocab", [1, 37, 1025, 4093, 9001, 32000, 51865, 250054, 270005])
def test_policy_loss(kind, layout, vocab):
    for rows in (1, 9, 500) if vocab < 10000 else (1, 9):
        x, y = _logits(rows, vocab, kind, layout)
        g = torch.Generator().manual_seed(rows)
        lp = pref.token_logprobs(x.double(), y)
        old = (lp + 0.15 * torch.randn(rows, generator=g).to(DEV).double()).float()
        r = (lp + 0.3 * torch.randn(rows, generator=g).to(DEV).double()).float()
        adv = torch.randn(rows, generator=g).to(DEV)
        for cfg in (dict(ref_logprobs=r, kl_coef=0.05), dict(clip=0.1, clip_high=0.3, temperature=1.0)):
            (loss, clipped, kl, want), grad = _coefs(x, y, lambda t: pref.policy_loss(t, y, old, adv, **cfg))
            leaf = x.detach().requires_grad_(True)
            got = pref.policy_loss(leaf, y, old, adv, **cfg)
            mine = torch.autograd.grad(got[0], leaf)[0]
            _logprobs_close(got[3], want)
            assert got[1].item() == clipped.item()
            assert abs(got[0].item() - loss.item()) <= rows * 1e-5 and abs(got[2].item() - kl.item()) <= rows * 1e-5
            half = {"bf16": 2 ** -8, "fp16": 2 ** -11, "fp32": 2 ** -24}[kind]
            # the ratio follows the log-probability: 2^-18 of it; the coefficient, a difference of two such terms, 2^-15 of 4 (|A| < 4)
            assert ((mine.double() - grad).abs() <= (half + 2 ** -15) * grad.abs() + 2 ** -13).all()
            with torch.no_grad():
                assert all(torch.equal(a, b) for a, b in zip(pref.policy_loss(x, y, old, adv, **cfg), got))
    assert ops.check_status() == 0


@pytest.mark.gpu
def test_gradient_against_differences_of_the_loss():
    x, y, cu, r = _pairs([4, 6, 3, 5], 50, "fp32", "dense")
    leaf = x.detach().requires_grad_(True)
    grad = torch.autograd.grad(pref.preference_loss(leaf, y, cu, r, beta=0.5)[0], leaf)[0]
    g = torch.Generator().manual_seed(3)
    d = torch.randn(x.shape, generator=g).to(DEV)
    d /= d.norm()
    h = 0.05
    at = lambda s: pref.preference_loss((x.double() + s * h * d.double()).float(), y, cu, r, beta=0.5)[0].item()
    diff = (at(1) - at(-1)) / (2 * h)
    # third derivative of the loss along a unit vector is below 1: h^2 / 6; the losses' own roundings 1e-6 / h
    assert abs(diff - float((grad.double() * d.double()).sum())) <= h * h + 1e-4


@pytest.mark.gpu
def test_upstream_gradient_scale_and_consumed_logits():
    x, y, cu, r = _pairs([9, 6, 30, 25], 3001, "bf16", "odd")
    leaf = x.detach().requires_grad_(True)
    base = torch.autograd.grad(pref.preference_loss(leaf, y, cu, r)[0], leaf)[0]
    third = torch.autograd.grad(pref.preference_loss(leaf, y, cu, r)[0] * 0.25, leaf)[0]
    assert torch.equal(third, base * 0.25)                       # a power of two: no rounding
    for scale in (0.25, torch.tensor(0.25, device=DEV)):
        loss = pref.preference_loss(leaf, y, cu, r, grad_scale=scale)[0]
        assert torch.equal(torch.autograd.grad(loss, leaf)[0], base * 0.25)
    flat = torch.empty(x.shape[0] * (x.stride(0)) + 5, dtype=x.dtype, device=DEV)
    spare = flat[5:].view(x.shape[0], x.stride(0))
    spare.fill_(7.0)
    view = spare[:, :x.shape[1]]
    view.copy_(x)
    consumed = view.detach().requires_grad_(True)
    version = consumed._version
    grad = torch.autograd.grad(pref.preference_loss(consumed, y, cu, r, inplace=True)[0], consumed)[0]
    assert torch.equal(grad, base) and grad.data_ptr() == view.data_ptr() and torch.equal(view, base) and consumed._version > version
    assert (spare[:, x.shape[1]:] == 7.0).all() and (flat[:5] == flat[:5]).all()
    view.copy_(x)
    consumed = view.detach().requires_grad_(True)
    old, adv = torch.full((x.shape[0],), -4.0, device=DEV), torch.ones(x.shape[0], device=DEV)
    leaf = x.detach().requires_grad_(True)
    want = torch.autograd.grad(pref.policy_loss(leaf, y, old, adv)[0], leaf)[0]
    assert torch.equal(torch.autograd.grad(pref.policy_loss(consumed, y, old, adv, inplace=True)[0], consumed)[0], want)


@pytest.mark.gpu
def test_a_second_backward_pass_is_refused():
    x, y, cu, r = _pairs([3, 4], 100, "bf16", "dense")
    leaf = x.detach().requires_grad_(True)
    loss = pref.preference_loss(leaf, y, cu, r)[0]
    loss.backward(retain_graph=True)
    with pytest.raises(RuntimeError, match="second backward"):
        loss.backward()


@pytest.mark.gpu
def test_offsets_out_of_order_and_nothing_to_do():
    """Offsets that fall or leave the rows are put in order (running maximum, clamped); no rows, no pairs, only empty pairs."""
    x, y = _logits(20, 300, "bf16", "dense")
    bad = torch.tensor([-3, 5, 2, 90, 11], dtype=torch.int32, device=DEV)
    good = torch.tensor([0, 5, 5, 20, 20], dtype=torch.int32, device=DEV)
    a, b = x.detach().requires_grad_(True), x.detach().requires_grad_(True)
    la, lb = pref.preference_loss(a, y, bad), pref.preference_loss(b, y, good)
    assert torch.equal(la[0], lb[0]) and torch.equal(la[2], lb[2])
    assert torch.equal(torch.autograd.grad(la[0], a)[0], torch.autograd.grad(lb[0], b)[0])
    for n, cu in ((20, [0]), (0, [0]), (0, [0, 0, 0]), (20, [7, 7, 7, 7, 7])):
        leaf = x[:n].detach().requires_grad_(True)
        c = torch.tensor(cu, dtype=torch.int32, device=DEV)
        loss, ranked, scores = pref.preference_loss(leaf, y[:n], c)
        assert abs(loss.item() - math.log(2.0) * (len(cu) // 2)) < 1e-6 and ranked.item() == 0 and (scores == 0).all()
        assert (torch.autograd.grad(loss, leaf)[0] == 0).all()
    leaf = x[:0].detach().requires_grad_(True)
    none = torch.zeros(0, device=DEV)
    loss, clipped, kl, lp = pref.policy_loss(leaf, y[:0], none, none)
    assert loss.item() == 0 and clipped.item() == 0 and kl.item() == 0 and lp.numel() == 0
    assert pref.token_logprobs(x[:0], y[:0]).numel() == 0
    assert ops.check_status() == 0


@pytest.mark.gpu
def test_layouts_that_are_copied():
    """A transposed matrix, rows that overlap (expanded), every other column, 32-bit labels."""
    x, y = _logits(8, 600, "fp32", "dense")
    want = pref.token_logprobs(x, y)
    assert torch.equal(pref.token_logprobs(x.t().contiguous().t(), y), want)
    wide = torch.zeros(8, 1200, device=DEV)
    wide[:, ::2] = x
    assert torch.equal(pref.token_logprobs(wide[:, ::2], y.int()), want)
    same = pref.token_logprobs(x[:1].expand(8, 600), y)
    assert torch.equal(same, pref.token_logprobs(x[:1].repeat(8, 1), y))
    leaf = x.t().contiguous().requires_grad_(True)
    grad = torch.autograd.grad(pref.token_logprobs(leaf.t(), y).sum(), leaf)[0]
    assert grad.shape == leaf.shape


@pytest.mark.gpu
def test_streams_and_captured_graphs():
    """Two calls at once on two streams, and two captured graphs replayed in turn and at once, give the bits of calls by themselves."""
    one, two = _pairs([30, 20, 50, 44], 8000, "bf16", "padded"), _pairs([10, 25, 31, 31, 5, 6], 9001, "bf16", "odd", seed=5)

    def step(c):
        x, y, cu, r = c
        leaf = x.detach().requires_grad_(True)
        loss, ranked, scores = pref.preference_loss(leaf, y, cu, r)
        lp = pref.token_logprobs(x, y)
        return [loss.detach(), ranked, scores, torch.autograd.grad(loss, leaf)[0], lp]

    want = [step(one), step(two)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, c in enumerate((one, two)):
            with torch.cuda.stream(streams[i]):
                got[i].append(step(c))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for out in got[i] for a, b in zip(out, want[i]))
    graphs, outs = [], []
    for c in (one, two):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(c))
        graphs.append(g)
    for _ in range(3):
        for i, g in enumerate(graphs):
            with torch.cuda.stream(streams[i]):
                g.replay()
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for a, b in zip(outs[i], want[i]))
    assert ops.check_status() == 0


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    _refusals(DEV)
    x, y = _logits(4, 10, "fp32", "dense")
    with pytest.raises(RuntimeError):
        ops.ext().row_scores(x, y[:3], 0, 1.0, False)
    with pytest.raises(RuntimeError):
        ops.ext().row_scores(x[:1].expand(4, 10), y, 0, 1.0, False)
    with pytest.raises(RuntimeError):
        ops.ext().row_scores(x.double(), y, 0, 1.0, False)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab,kind,layout", [(8400, 8001, "bf16", "odd"), (8300, 8104, "fp16", "dense"), (2070, 32500, "bf16", "dense"),
                                                    (270, 250054, "bf16", "padded"), (15000, 4700, "bf16", "padded"), (40, 1700011, "fp16", "odd"), (4500, 9001, "fp32", "odd")])
def test_large_batches(rows, vocab, kind, layout):
    """As many rows as keep every SM busy for long: rows handed out as they come, runs of padding among them, a captured graph replayed; the same
    bits each time."""
    x, y = _logits(5, vocab, kind, layout)
    g = torch.Generator(device=DEV).manual_seed(rows)
    width, skip = x.stride(0), x.storage_offset()
    x = (torch.randn(rows * width + skip, generator=g, device=DEV, dtype=x.dtype) * 2)[skip:].view(rows, width)[:, :vocab]
    y = torch.randint(1, vocab, (rows,), generator=g, device=DEV)
    y[rows // 3:rows // 2] = 0
    y[-3:] = vocab
    weight = torch.randn(rows, generator=g, device=DEV)
    leaf = x.detach().requires_grad_(True)
    got = pref.token_logprobs(leaf, y, temperature=0.9)
    grad = torch.autograd.grad(got, leaf, weight)[0]
    for r in range(0, rows, 500):
        xd = x[r:r + 500].double().requires_grad_(True)
        want = pref.token_logprobs(xd, y[r:r + 500], temperature=0.9)
        _logprobs_close(got.detach()[r:r + 500], want.detach())
        _grads_close(grad[r:r + 500], torch.autograd.grad(want, xd, weight[r:r + 500].double())[0], weight[r:r + 500] / 0.9, kind)
    with torch.no_grad():
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = pref.token_logprobs(x, y, temperature=0.9)
        for _ in range(3):
            out.zero_()
            graph.replay()
            assert torch.equal(out, got)
    cu = torch.linspace(0, rows, 21, device=DEV).int()
    loss, ranked, scores = pref.preference_loss(leaf, y, cu, temperature=0.9)
    sums = pref.sequence_logprobs(got.detach(), cu)
    assert ((scores - sums).abs() <= 2 ** -22 * (pref.sequence_logprobs(-got.detach(), cu) + 1)).all()     # one rounding of each word's, one of the sum
    assert ranked == (sums[0::2] > sums[1::2]).sum()
    assert torch.isfinite(torch.autograd.grad(loss, leaf)[0]).all() and ops.check_status() == 0


@pytest.mark.gpu
def test_no_second_derivative():
    x, y = _logits(9, 40, "fp32", "dense")
    leaf = x.requires_grad_(True)
    zero = torch.zeros(9, device=DEV)
    for f in (lambda: pref.token_logprobs(leaf, y).sum(), lambda: pref.policy_loss(leaf, y, zero, zero)[0],
              lambda: pref.preference_loss(leaf, y, torch.tensor([0, 4, 9], device=DEV))[0]):
        with pytest.raises(RuntimeError):
            torch.autograd.grad(f(), leaf, create_graph=True)


def test_temperatures_out_of_range():
    x, y = torch.zeros(2, 3), torch.ones(2, dtype=torch.long)
    for t in (0.0, -1.0, math.nan, math.inf, 1e-39):
        with pytest.raises(ValueError):
            pref.token_logprobs(x, y, temperature=t)


@pytest.mark.gpu
def test_more_than_2_31_logits():
    """Offsets beyond 32 bits: the last rows of a matrix of 2.2e9 logits against the same rows by themselves."""
    rows, vocab = 8800, 250054
    x = torch.empty(rows, 250056, dtype=torch.bfloat16, device=DEV).normal_(generator=torch.Generator(device=DEV).manual_seed(3))[:, :vocab]
    y = torch.randint(1, vocab, (rows,), generator=torch.Generator().manual_seed(3)).to(DEV)
    weight = torch.ones(rows, device=DEV)
    last = x[-7:].clone().double().requires_grad_(True)
    want = pref.token_logprobs(last, y[-7:])
    leaf = x.requires_grad_(True)
    got = pref.token_logprobs(leaf, y)
    grad = torch.autograd.grad(got, leaf, weight)[0]
    _logprobs_close(got.detach()[-7:], want.detach())
    _grads_close(grad[-7:], torch.autograd.grad(want, last, weight[-7:].double())[0], weight[-7:], "bf16")
    cu = torch.tensor([0, rows - 7, rows], device=DEV)
    for f in (lambda: pref.preference_loss(leaf, y, cu, inplace=False), lambda: pref.policy_loss(leaf, y, got.detach(), weight)):
        grad = None
        grad = torch.autograd.grad(f()[0], leaf)[0]
        ratio = grad[-7:].float() / torch.autograd.grad(pref.token_logprobs(leaf[-7:], y[-7:]), leaf, weight[-7:])[0][-7:].float()
        assert (ratio.nan_to_num(ratio[0, 0].item()) / ratio[0, 0] - 1).abs().max() <= 2 ** -6          # one coefficient; four roundings of bf16
    assert ops.check_status() == 0


def test_a_word_of_probability_0_stays_in_its_sequence():
    lp = torch.tensor([-1.0, -2.0, -math.inf, -0.5, -1.5, math.nan, -0.25, -math.inf, -3.0])
    got = pref.sequence_logprobs(lp, torch.tensor([0, 2, 4, 5, 7, 7, 9]))
    assert got[:3].tolist() == [-3.0, -math.inf, -1.5] and torch.isnan(got[3]) and got[4] == 0.0 and got[5] == -math.inf
    leaf = lp[:2].clone().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(pref.sequence_logprobs(leaf, torch.tensor([0, 1, 2])).sum(), leaf)[0], torch.ones(2))


@pytest.mark.gpu
@pytest.mark.parametrize("kind,vocab,layout", [("fp32", 5500, "dense"), ("bf16", 12001, "odd"), ("fp16", 13000, "padded"), ("bf16", 20001, "padded"),
                                               ("bf16", 45000, "odd"), ("bf16", 114688, "dense"), ("bf16", 114689, "odd"), ("fp32", 57344, "dense"),
                                               ("fp32", 57350, "odd"), ("fp16", 4096, "dense"), ("bf16", 4097, "odd"), ("fp32", 2048, "padded"), ("fp32", 2049, "odd"),
                                               ("fp16", 57344, "dense"), ("bf16", 57345, "odd"), ("bf16", 200003, "odd"), ("bf16", 229376, "padded"), ("fp16", 229380, "odd"),
                                               ("fp32", 120001, "odd"), ("bf16", 458752, "dense"), ("fp16", 458753, "padded")])
def test_policy_loss_at_the_sizes_where_its_kernels_change(kind, vocab, layout):
    """Rows of every number of threads and blocks, of all the shared memory that these have and of a word more; masked logits, padding, an inplace
    gradient."""
    rows = 40
    x, y = _logits(rows, vocab, kind, layout)
    x[7, 5:] = -math.inf
    y[7] = 2
    x[8] = torch.finfo(TYPES[kind]).min
    g = torch.Generator().manual_seed(vocab)
    lp = pref.token_logprobs(x.double(), y)
    old, r = (lp + 0.2 * torch.randn(rows, generator=g).to(DEV).double()).float(), (lp + 0.3 * torch.randn(rows, generator=g).to(DEV).double()).float()
    adv = torch.randn(rows, generator=g).to(DEV)
    (loss, clipped, kl, want), grad = _coefs(x, y, lambda t: pref.policy_loss(t, y, old, adv, r, kl_coef=0.1))
    leaf = x.detach().requires_grad_(True)
    got = pref.policy_loss(leaf, y, old, adv, r, kl_coef=0.1)
    mine = torch.autograd.grad(got[0], leaf)[0]
    _logprobs_close(got[3], want)
    assert got[1].item() == clipped.item() and abs(got[0].item() - loss.item()) <= rows * 1e-5 and abs(got[2].item() - kl.item()) <= rows * 1e-5
    half = {"bf16": 2 ** -8, "fp16": 2 ** -11, "fp32": 2 ** -24}[kind]
    # as in test_policy_loss: the coefficient off by 2^-15 of 4
    assert ((mine.double() - grad).abs() <= (half + 2 ** -15) * grad.abs() + 2 ** -13).all()
    assert (mine[1:4] == 0).all()
    consumed = x.detach().clone(memory_format=torch.contiguous_format).requires_grad_(True)
    plain = x.detach().clone(memory_format=torch.contiguous_format).requires_grad_(True)
    over = pref.policy_loss(consumed, y, old, adv, r, kl_coef=0.1, inplace=True)
    first = torch.autograd.grad(over[0], consumed)[0]
    assert first.data_ptr() == consumed.data_ptr()
    assert torch.equal(first, torch.autograd.grad(pref.policy_loss(plain, y, old, adv, r, kl_coef=0.1)[0], plain)[0])
    assert ops.check_status() == 0


def test_logprobs_of_very_large_logits():
    """Rows of the type's lowest value have every word alike, rows with +inf or nothing but -inf NaN, on the CPU as on a GPU."""
    for dtype in (torch.float64, torch.float32, torch.bfloat16):
        x = torch.zeros(4, 50, dtype=dtype)
        x[0], x[1], x[2], x[3, 7] = torch.finfo(torch.float32 if dtype == torch.float64 else dtype).min, 1e30, -math.inf, math.inf
        got = pref.token_logprobs(x, torch.full((4,), 3))
        assert ((got[:2] + math.log(50)).abs() <= 2 ** -19).all() and torch.isnan(got[2:]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab,kind", [(900, 2500, "bf16"), (700, 1500, "fp32"), (700, 9001, "fp16"), (200, 131073, "bf16"), (2100, 32500, "bf16"), (300, 60000, "fp32")])
def test_captured_losses_beside_other_work(rows, vocab, kind):
    """All three operators captured in one graph and replayed while the same operators run on another stream: the bits of eager calls, each time.  Their
    kernels are scheduled while the ones before them end, in graphs, too."""
    x, y = _logits(rows, vocab, kind, "padded")
    g = torch.Generator().manual_seed(rows)
    cu = torch.linspace(0, rows - 3, 15).int().to(DEV)
    adv, old = torch.randn(rows, generator=g).to(DEV), pref.token_logprobs(x, y) + 0.1
    other = x.flip(0).contiguous()

    def step(t):
        leaf = t.detach().requires_grad_(True)
        pairs = pref.preference_loss(leaf, y, cu, beta=0.05)
        policy = pref.policy_loss(leaf, y, old, adv)
        lp = pref.token_logprobs(leaf, y)
        return [o.detach() for o in (*pairs, *policy, lp)] + [torch.autograd.grad(f, leaf)[0] for f in (pairs[0], policy[0])] + [torch.autograd.grad(lp, leaf, adv)[0]]

    want, beside = step(x), step(other)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(x)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(4):
        for o in out:
            o.fill_(7.0)
        torch.cuda.synchronize()
        with torch.cuda.stream(streams[0]):
            graph.replay()
        with torch.cuda.stream(streams[1]):
            got = step(other)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
        assert all(torch.equal(a, b) for a, b in zip(got, beside))
    assert ops.check_status() == 0
