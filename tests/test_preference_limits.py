"""Losses of preference tuning where their terms leave the numbers: words of probability 0 and ratios beyond 32 bits.  Expected values are written
out in 64 bits, apart from the restatements, which are tested like the kernels."""
import math

import pytest
import torch

from nmtgminor_b200 import ops
from nmtgminor_b200.ops import preference as pref

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
HALF = {torch.bfloat16: 2 ** -8, torch.float16: 2 ** -11, torch.float32: 2 ** -24, torch.float64: 0.0}
# rows that a warp holds, a block, a cluster of blocks, and none of them
SIZES = [("cpu", 40, torch.float32), ("cpu", 40, torch.float64), *(pytest.param("cuda", v, d, marks=pytest.mark.gpu) for v, d in (
    (40, torch.float32), (40, torch.float16), (9001, torch.bfloat16), (60001, torch.float32), (270005, torch.float32)))]


def _rows(device, rows, vocab, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + vocab)
    x = (torch.randn(rows, vocab, generator=g) * 2).to(dtype).to(device)
    return x, torch.randint(1, vocab, (rows,), generator=g).to(device)


def _close(got, coef, x, y, slack=0.0):
    """Gradient rows coef * (onehot - softmax).  Against 64 bits: half a step of the type, 2^-15 of an exponential (its argument's roundings, the sum, the
    coefficient), at the label of coef p; half of fp16's smallest number.  ``slack``: error of the coefficients themselves."""
    p = torch.softmax(x.double(), 1)
    hot = torch.nn.functional.one_hot(y, x.shape[1]).double()
    c = torch.as_tensor(coef, dtype=torch.float64, device=x.device)[:, None]
    want = c * (hot - p)
    low = 2 ** -25 if x.dtype == torch.float16 else 1e-36
    bound = (HALF[x.dtype] + 2 ** -15) * want.abs() + 2 ** -15 * c.abs() * p * hot + slack * (hot - p).abs() + low
    assert ((got.double() - want).abs() <= bound).all(), ((got.double() - want).abs() - bound).max()


@pytest.mark.parametrize("device,vocab,dtype", SIZES)
@pytest.mark.parametrize("where", ["preferred", "rejected"])
@pytest.mark.parametrize("kind,smoothing", [("sigmoid", 0.0), ("sigmoid", 0.1), ("hinge", 0.0), ("ipo", 0.0)])
def test_a_word_of_probability_0_in_a_pair(device, vocab, dtype, where, kind, smoothing):
    """z = inf costs a pair nothing and gives it no gradient, unless the smoothed term or the square is infinite; z = -inf costs inf, its gradient is
    that of a loss linear in z."""
    x, y = _rows(device, 11, vocab, dtype)
    x[2 if where == "preferred" else 7, y[2 if where == "preferred" else 7]] = -math.inf
    cu = torch.tensor([0, 5, 11], device=device)
    beta, won = 0.3, int(where == "rejected")
    leaf = x.detach().requires_grad_(True)
    loss, ranked, scores = pref.preference_loss(leaf, y, cu, None, beta, kind, smoothing, pad_idx=-1)
    assert loss.item() == (0.0 if won and kind != "ipo" and not smoothing else math.inf) and ranked.item() == won
    assert scores[won] == -math.inf and torch.isfinite(scores[1 - won])
    grad = torch.autograd.grad(loss, leaf)[0]
    if kind == "ipo":
        assert not torch.isfinite(grad).all()
        return
    slope = (beta * smoothing if won else -beta * (1 - smoothing)) if kind == "sigmoid" else (0.0 if won else -beta)
    _close(grad, [slope] * 5 + [-slope] * 6, x, y)


@pytest.mark.parametrize("device,vocab,dtype", SIZES)
def test_a_pair_at_infinity_leaves_the_others_alone(device, vocab, dtype):
    x, y = _rows(device, 20, vocab, dtype, 1)
    x[13, y[13]] = -math.inf
    cu = torch.tensor([0, 4, 9, 12, 20], device=device)
    with torch.no_grad():
        loss, ranked, scores = pref.preference_loss(x, y, cu, pad_idx=-1)
        alone = pref.preference_loss(x[:9], y[:9], cu[:3], pad_idx=-1)
    assert loss.item() == pytest.approx(alone[0].item(), rel=1e-5) and ranked.item() == alone[1].item() + 1      # the same rows, dealt out to other threads


@pytest.mark.parametrize("device", DEVICES)
def test_a_word_of_probability_0_on_both_sides_is_not_hidden(device):
    x, y = _rows(device, 8, 50, torch.float32)
    x[1, y[1]] = x[6, y[6]] = -math.inf
    cu = torch.tensor([0, 3, 8], device=device)
    for kind in pref.KINDS:
        assert math.isnan(pref.preference_loss(x, y, cu, kind=kind, pad_idx=-1)[0].item())
    if device == "cuda":
        assert ops.check_status() == 0


@pytest.mark.parametrize("device,vocab,dtype", SIZES)
def test_infinite_kl_terms(device, vocab, dtype):
    """Words that the frozen model finds e^100 times as probable, and one of probability 0: the reported KL is infinite, the loss and its gradient are
    without it those of the ratios; with it the loss is infinite.  NaN only where both models give a word probability 0."""
    x, y = _rows(device, 8, vocab, dtype, 2)
    x[3, y[3]] = -math.inf
    lp = torch.log_softmax(x.double(), 1).gather(1, y[:, None]).squeeze(1)
    adv = torch.linspace(-1, 1, 8, device=device)
    old = (lp + 0.05).float()
    old[3] = -3.0
    ref = (lp + 0.3).float()
    ref[1] = lp[1].float() + 800.0                              # e^800: beyond 64 bits, too
    ref[3] = -4.0
    ratio = torch.exp(lp - old.double())
    assert ((ratio - 0.8).abs() > 0.01).all() and ((ratio - 1.2).abs() > 0.01).all()
    held = ratio.clamp(0.8, 1.2)
    clipped = ratio * adv > held * adv
    leaf = x.detach().requires_grad_(True)
    loss, n, kl, got = pref.policy_loss(leaf, y, old, adv, ref, pad_idx=-1)
    want = -torch.minimum(ratio * adv, held * adv).sum()
    # 8 ratios, each off by 2^-18 of at most 1.2 (of its log-probability 2^-19 and their difference's rounding), |A| <= 1
    assert abs(loss.item() - want.item()) <= 8 * 1.2 * 2 ** -18 and n.item() == clipped.sum().item()
    assert kl.item() == math.inf and got[3] == -math.inf
    grad = torch.autograd.grad(loss, leaf)[0]
    _close(grad, torch.where(clipped, 0.0, -ratio * adv), x, y, slack=1.2 * 2 ** -18)
    with torch.no_grad():
        loss, _, kl, _ = pref.policy_loss(x, y, old, adv, ref, kl_coef=0.1, pad_idx=-1)
        assert loss.item() == math.inf and kl.item() == math.inf
        ref[3] = -math.inf
        assert math.isnan(pref.policy_loss(x, y, old, adv, ref, pad_idx=-1)[2].item())


@pytest.mark.parametrize("device", DEVICES)
def test_offsets_of_sequence_scores(device):
    """Offsets that fall or leave the rows, as ``preference_loss`` takes them: an index out of range otherwise.  No sequences, no rows."""
    lp = -torch.arange(1.0, 21.0, device=device)
    bad, good = (torch.tensor(c, device=device) for c in ([-3, 5, 2, 90, 11], [0, 5, 5, 20, 20]))
    want = torch.tensor([-15.0, 0.0, -195.0, 0.0], device=device)
    assert torch.equal(pref.sequence_logprobs(lp, bad), want) and torch.equal(pref.sequence_logprobs(lp, good.int()), want)
    assert pref.sequence_logprobs(lp, bad[:1]).shape == (0,)
    assert torch.equal(pref.sequence_logprobs(lp[:0], good), torch.zeros(4, device=device))
    x, y = _rows(device, 20, 40, torch.float32)
    scores = pref.preference_loss(x, y, bad, pad_idx=-1)[2]
    assert ((pref.sequence_logprobs(pref.token_logprobs(x, y, -1), bad) - scores).abs() <= 20 * 2 ** -23 * (scores.abs() + 1)).all()
    far = torch.tensor([0, 5, 2, 2 ** 32 + 3, 11], device=device)
    assert torch.equal(pref.preference_loss(x, y, far, pad_idx=-1)[2], scores)
    assert torch.equal(pref.sequence_logprobs(lp, good.cpu()), want)
    for words, cu in ((lp[None], good), (lp, good[:0]), (lp, good[None])):
        with pytest.raises(ValueError):
            pref.sequence_logprobs(words, cu)


@pytest.mark.parametrize("device,vocab,dtype", SIZES)
def test_what_is_left_out_has_a_gradient_of_zero(device, vocab, dtype):
    """NaN and infinities in rows of padding and outside every sequence, in their scores and advantages, too; a ratio beyond the type's range where it is clipped."""
    x, y = _rows(device, 9, vocab, dtype, 3)
    lp = torch.log_softmax(x.double(), 1).gather(1, y[:, None]).squeeze(1)
    old, adv = lp.float(), torch.ones(9, device=device)
    y[2], y[3], y[4] = 0, -1, vocab + 4
    for r, v in ((2, math.nan), (3, math.inf), (4, -math.inf)):
        x[r] = v
        old[r] = adv[r] = v
    old[7] = lp[7].float() - 2000.0                             # ratio e^2000, held at 1.2
    out = torch.tensor([2, 3, 4], device=device)
    keep = torch.tensor([0, 1, 5, 6, 8], device=device)
    leaf = x.detach().requires_grad_(True)
    grad = torch.autograd.grad(pref.token_logprobs(leaf, y).sum(), leaf)[0]
    assert (grad[out] == 0).all()
    _close(grad[keep], [1.0] * 5, x[keep], y[keep])
    loss, n, _, _ = pref.policy_loss(leaf, y, old, adv)
    # five ratios of 1, off by their log-probabilities' 2^-19 and the rounding of ``old``, below 2^-20 for 16; the held one
    assert abs(loss.item() + 5 + 1.2) <= 5 * 2 ** -18 and n.item() == 1
    grad = torch.autograd.grad(loss, leaf)[0]
    assert (grad[out] == 0).all() and (grad[7] == 0).all()
    _close(grad[keep], [-1.0] * 5, x[keep], y[keep], slack=2 ** -18)
    y[2:5] = 1                                                  # words, but outside the sequences
    x[4], x[2] = x[2].clone(), 0.0
    for cu in ([5, 7, 9], [0, 1, 2]):
        c = torch.tensor(cu, device=device)
        z = x if cu[0] else x.flip(0)
        labels = y if cu[0] else y.flip(0)
        leaf = z.detach().requires_grad_(True)
        grad = torch.autograd.grad(pref.preference_loss(leaf, labels, c, pad_idx=-1)[0], leaf)[0]
        inside = torch.zeros(9, dtype=torch.bool, device=device)
        inside[cu[0]:cu[-1]] = True
        assert (grad[~inside] == 0).all() and torch.isfinite(grad[inside]).all() and (grad[inside] != 0).any()


@pytest.mark.parametrize("device,vocab,dtype", SIZES)
def test_no_pair_at_all(device, vocab, dtype):
    """One offset: a loss of 0, and a gradient of 0 for every row."""
    x, y = _rows(device, 4, vocab, dtype)
    leaf = x.detach().requires_grad_(True)
    loss, ranked, scores = pref.preference_loss(leaf, y, torch.tensor([2], device=device), pad_idx=-1)
    assert loss.item() == 0 and ranked.item() == 0 and scores.shape == (0,)
    assert (torch.autograd.grad(loss, leaf)[0] == 0).all()


@pytest.mark.parametrize("device,dtype", [("cpu", torch.float64), *(pytest.param("cuda", d, marks=pytest.mark.gpu) for d in (torch.float32, torch.bfloat16))])
@pytest.mark.parametrize("size", [1e-1, 1e-3, 1e-5])
def test_kl_terms_near_0(device, dtype, size):
    """A single word: its log-probability is 0 exactly, and e^d - d - 1 as good as its rounding."""
    x = torch.zeros(700, 1, dtype=dtype, device=device)
    y = torch.zeros(700, dtype=torch.int64, device=device)
    ref = ((torch.rand(700, generator=torch.Generator().manual_seed(5)) - 0.5) * size).to(device)
    d = ref.double()
    want = (d ** 2 / 2 + d ** 3 / 6 + d ** 4 / 24 + d ** 5 / 120 + d ** 6 / 720 + d ** 7 / 5040).sum().item()       # the next term: below 2^-36 of it
    kl = pref.policy_loss(x, y, ref, ref, ref, kl_coef=0.1, pad_idx=-1)[2].item()
    # the result is rounded to 32 bits; a double's expm1(d) - d is off by some 2^-52 d, of d^2 / 2
    assert abs(kl - want) <= (2 ** -23 + 2 ** -49 / size) * want


@pytest.mark.parametrize("device,vocab,dtype", SIZES)
@pytest.mark.parametrize("kind", list(pref.KINDS))
def test_a_pair_without_a_value_shows_in_its_gradient(device, vocab, dtype, kind):
    """inf - inf, or NaN in one of its rows: NaN in the gradient of every row of the pair, under each kind; the next pair is not touched."""
    x, y = _rows(device, 12, vocab, dtype, 4)
    cu = torch.tensor([0, 3, 8, 10, 12], device=device)
    for damage in (lambda z: z[1].index_fill_(0, y[1], -math.inf) + z[6].index_fill_(0, y[6], -math.inf), lambda z: z[2].fill_(math.nan)):
        leaf = x.clone()
        damage(leaf)
        leaf.requires_grad_(True)
        loss = pref.preference_loss(leaf, y, cu, kind=kind, pad_idx=-1)[0]
        grad = torch.autograd.grad(loss, leaf)[0]
        assert math.isnan(loss.item()) and torch.isnan(grad[:8]).all() and torch.isfinite(grad[8:]).all()
