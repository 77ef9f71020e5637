"""The losses of preference tuning element by element: gradients written out in 64 bits, coef * (onehot - softmax) / T, each element held to its own size.

What an element may be off by.  Half a step of its type.  Its exponential: an argument of at most 126 log 2 = 88 with four roundings of 2^-24, the
exponential itself 2^-22, the row's sum 2^-19, and a few roundings of the coefficient: 2^-15 of it in all; exponentials below 2^-126 are 0.  At the label
the element is coef (1 - p), off by 2^-15 of coef p.  Its coefficient: what the log-probabilities it is made of are off by, 2^-19 each, times the slope's
own slope.  fp16 rounds to multiples of 2^-24."""
import math

import pytest
import torch

from nmtgminor_b200 import ops
from nmtgminor_b200.ops import preference as pref

DEV = "cuda"
TYPES = {"bf16": (torch.bfloat16, 2 ** -8), "fp16": (torch.float16, 2 ** -11), "fp32": (torch.float32, 2 ** -24)}
WORD = 2 ** -19


def _rows(rows, vocab, kind, layout, seed):
    """Logits whose first and last words, which unaligned rows take one by one, have probability; padding, and labels among these words."""
    g = torch.Generator().manual_seed(seed + rows + vocab)
    width, skip = {"dense": (vocab, 0), "padded": ((vocab + 7) // 8 * 8, 0), "odd": (vocab + 3, 5)}[layout]
    x = torch.empty(rows * width + skip, dtype=TYPES[kind][0], device=DEV)[skip:].view(rows, width)[:, :vocab]
    x.copy_((torch.randn(rows, vocab, generator=g) * 2).to(DEV))
    x[:, :9] += 5
    x[:, -9:] += 5
    y = torch.randint(0, vocab, (rows,), generator=g).to(DEV)
    for r in range(0, rows, 3):
        y[r] = (r * 5 + 1) % min(9, vocab) if r % 2 else vocab - 1 - r % min(9, vocab)
    y[rows // 2], y[-1] = -1, vocab
    real = (y >= 0) & (y < vocab)
    lp = torch.log_softmax(x.double() , 1).gather(1, y.where(real, 0)[:, None]).squeeze(1) * real
    return x, y, real, lp, g


def _check(got, coef, off, x, y, real, kind, scale=1.0):
    half = TYPES[kind][1]
    coef, off = coef * real, off * real
    for r in range(0, x.shape[0], 64):
        s = slice(r, r + 64)
        p = torch.softmax(x[s].double(), 1)
        label = y[s].where(real[s], 0)[:, None]
        part = -p
        part.scatter_add_(1, label, real[s].double()[:, None])
        want = scale * coef[s, None] * part
        bound = (half + 2 ** -15) * want.abs() + abs(scale) * (off[s, None] * part.abs() + 2 ** -125 * coef[s, None].abs()) + {"fp16": 2 ** -25, "bf16": 2 ** -133, "fp32": 2 ** -149}[kind]
        at = 2 ** -15 * abs(scale) * coef[s, None].abs() * p.gather(1, label) * real[s, None]
        bound.scatter_add_(1, label, at)
        err = (got[s].double() - want).abs()
        assert (err <= bound).all(), (kind, tuple(x.shape), (err - bound).max().item())
    assert (got[~real] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["padded", "odd"])
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("vocab", [11, 2045, 4099, 9001, 33001, 51865, 120005, 250054, 458761])
def test_policy_gradient_element_by_element(kind, layout, vocab):
    rows = 70 if vocab < 60000 else 24
    x, y, real, lp, g = _rows(rows, vocab, kind, layout, 1)
    adv = torch.randn(rows, generator=g).to(DEV)
    old = (lp + 0.3 * torch.randn(rows, generator=g).to(DEV)).float()
    ref = (lp + 0.3 * torch.randn(rows, generator=g).to(DEV)).float()
    ratio = torch.exp(lp - old.double())
    for border in (0.8, 1.3):                                   # no ratio where its error decides
        old = torch.where((ratio - border).abs() < 1e-3, old + 0.01, old)
    ratio = torch.exp(lp - old.double())
    held = ratio.clamp(0.8, 1.3)
    free = ~(ratio * adv > held * adv)
    d = ref.double() - lp
    for kl, scale in ((0.0, 1.0), (0.2, 1.0), (0.2, 0.7)):
        coef = torch.where(free, -ratio * adv, 0.0) - kl * torch.expm1(d)
        # a log-probability's error, and the roundings of expf and expm1f (2 units in the last place each)
        off = (ratio * adv.abs() * free + kl * torch.exp(d)) * (WORD + 2 ** -21)
        leaf = x.detach().requires_grad_(True)
        loss, clipped, kl_sum, got = pref.policy_loss(leaf, y, old, adv, ref, 0.2, 0.3, kl, pad_idx=-1, **({} if scale == 1.0 else {"grad_scale": scale}))
        _check(torch.autograd.grad(loss, leaf)[0], coef, off, x, y, real, kind, scale)
        kls = (torch.expm1(d) - d)[real]
        want = (-torch.minimum(ratio * adv, held * adv)[real] + kl * kls).sum()
        slack = (off[real] + WORD * kl * d[real].abs()).sum().item() + 1.3 * WORD * adv[real].abs().sum().item()
        assert abs(loss.item() - want.item()) <= slack + 2 ** -23 * abs(want.item())
        assert abs(kl_sum.item() - kls.sum().item()) <= WORD * torch.expm1(d)[real].abs().sum().item() + 2 ** -23 * kls.sum().item() + rows * WORD ** 2
        assert clipped.item() == (~free & real).sum().item()
        assert ((got.double() - lp)[real].abs() <= WORD + 2 ** -23 * lp[real].abs()).all()
    assert ops.check_status() == 0


CONFIGS = [dict(), dict(kind="hinge", margin=0.5, beta=0.3), dict(kind="ipo", average=True, beta=0.5, nll_weight=0.1), dict(kind="ipo", beta=0.05),
           dict(smoothing=0.1, average=True, nll_weight=0.3, beta=0.7, margin=0.2)]


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["padded", "odd"])
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("vocab,lengths", [(11, [3, 1, 0, 6, 40, 17]), (2045, [9, 4, 30, 31]), (4099, [1, 1, 12, 50]), (9001, [300, 3, 2, 200]), (33001, [40, 33]),
                                           (51865, [20, 31, 9, 8]), (250054, [7, 12])])
def test_paired_gradient_element_by_element(kind, layout, vocab, lengths):
    rows, n = sum(lengths) + 2, len(lengths)
    x, y, real, lp, g = _rows(rows, vocab, kind, layout, 2)
    cu = torch.tensor([0] + lengths).cumsum(0).to(DEV)
    real = real & (torch.arange(rows, device=DEV) < cu[-1])
    lp = lp * real
    seq = torch.repeat_interleave(torch.arange(n, device=DEV), torch.tensor(lengths, device=DEV), output_size=rows - 2)
    zero = torch.zeros(n, dtype=torch.float64, device=DEV)
    scores, count, size = zero.index_add(0, seq, lp[:-2]), zero.index_add(0, seq, real[:-2].double()), zero.index_add(0, seq, lp[:-2].abs())
    ref = (scores + 3 * torch.randn(n, generator=g).to(DEV)).float()
    for cfg in CONFIGS:
        beta, margin, eps, nll = cfg.get("beta", 0.1), cfg.get("margin", 0.0), cfg.get("smoothing", 0.0), cfg.get("nll_weight", 0.0)
        each = 1.0 / count.clamp(min=1.0) if cfg.get("average") else torch.ones_like(scores)
        h = ((scores - ref.double()) * each)[0::2] - ((scores - ref.double()) * each)[1::2]
        # a word's log-probability is off by WORD, and its sums are in 64 bits
        dh = (count * each * WORD)[0::2] + (count * each * WORD)[1::2] + 2 ** -50 * ((size + ref.abs()) * each).sum()
        z = beta * h - margin
        if cfg.get("kind") == "ipo":
            loss, slope, off = (h - 0.5 / beta) ** 2, 2 * (h - 0.5 / beta), 2 * dh + 2 ** -23 / beta
            loss_off = slope.abs() * (dh + 2 ** -24 / beta) + (dh + 2 ** -24 / beta) ** 2
        elif cfg.get("kind") == "hinge":
            assert ((z - 1).abs() > 1e-2).all()
            loss, slope, off = torch.relu(1 - z), torch.where(z < 1, -beta, 0.0), torch.zeros_like(z)
            loss_off = beta * dh + 2 ** -24 * (beta * h.abs() + margin)
        else:
            loss = -(1 - eps) * torch.nn.functional.logsigmoid(z) - eps * torch.nn.functional.logsigmoid(-z)
            slope = beta * (eps * torch.sigmoid(z) - (1 - eps) * torch.sigmoid(-z))
            dz = beta * dh + 2 ** -24 * (beta * h.abs() + abs(margin))
            off, loss_off = beta / 4 * dz, dz
        off = off + 2 ** -23 * (slope.abs() + nll + beta * eps)            # beta, smoothing and the weight are held in 32 bits
        coef = torch.stack([(slope - nll) * each[0::2], -slope * each[1::2]], 1).flatten()
        coef_off = torch.stack([off * each[0::2], off * each[1::2]], 1).flatten()
        of = torch.cat([seq, seq.new_zeros(2)])
        leaf = x.detach().requires_grad_(True)
        got, ranked, sums = pref.preference_loss(leaf, y, cu, ref, pad_idx=-1, **cfg)
        _check(torch.autograd.grad(got, leaf)[0], coef[of], coef_off[of], x, y, real, kind)
        want = (loss - nll * (scores * each)[0::2]).sum().item()
        slack = loss_off.sum() + nll * ((count * each * WORD)[0::2] + 2 ** -23 * (scores * each)[0::2].abs()).sum() + 2 ** -23 * beta * eps * h.abs().sum()
        assert abs(got.item() - want) <= slack.item() + 2 ** -23 * abs(want)
        assert (h.abs() > dh).all() and ranked.item() == (h > 0).sum().item()
        assert ((sums.double() - scores).abs() <= count * WORD + 2 ** -24 * scores.abs()).all()
    assert ops.check_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("vocab", [11, 4099, 51865, 250054])
def test_weighted_log_probabilities_element_by_element(kind, vocab):
    """The gradient of a weighted sum of log-probabilities, with a temperature, unaligned rows."""
    x, y, real, _, g = _rows(30, vocab, kind, "odd", 3)
    weight = torch.randn(30, generator=g).to(DEV)
    for temperature in (1.0, 1.7):
        leaf = x.detach().requires_grad_(True)
        grad = torch.autograd.grad(pref.token_logprobs(leaf, y, -1, temperature), leaf, weight)[0]
        _check(grad, weight.double() / temperature, 2 ** -23 * weight.double().abs(), x.double() / temperature, y, real, kind)
    assert ops.check_status() == 0 and math.isfinite(grad.float().abs().max().item())
