"""Losses of preference tuning over rows of logits: log-probabilities of target words with their gradient, the paired preference
loss and the clipped policy loss with a KL term.

They stand beside ``ops.cross_entropy``: logits ``[rows, vocab]`` of packed sequences (bf16, fp16 or fp32; elements of a row adjacent, any
row stride), labels ``[rows]``, rows whose label is ``pad_idx`` or no word left out, sums over the others returned.  On a GPU each is one
pass of ``csrc/preference.cu`` over the logits, which computes the gradient together with the loss; on the CPU, and for fp64, it is the
plain PyTorch restatement below, which is also the tests' oracle.

A row whose target has probability 0 (a logit of -inf) has log-probability -inf; rows with NaN, with a logit of +inf, or with nothing
but -inf have NaN, as ``torch.log_softmax`` has.

The gradient tensor of the two losses belongs to the backward pass, so a second pass through the same loss (``retain_graph``) is refused.
``grad_scale`` (a float, or one fp32 element on the logits' device that is read when the kernel runs) multiplies the gradient where it is
computed; the upstream gradient of the loss is then taken to be 1, as in ``ops.generator_cross_entropy``.  Without it an upstream gradient
other than 1 costs another pass over the gradient of fp32 and bf16 logits, and a second rounding where it is no power of two; the gradient of fp16 logits is then
made in the backward pass, so that a scaled loss keeps what fp16 would lose.  A backward pass can be captured in a CUDA graph where, as PyTorch asks of every operator, no graph
of the same leaves made outside the capture is alive.  ``inplace`` writes the gradient over the logits, which are consumed (as ``ops.cross_entropy``
consumes its own): nothing else may read or change them behind the call.
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn.functional as F

from . import LAUNCHES, ext, reference as ref

KINDS = {"sigmoid": 0, "hinge": 1, "ipo": 2}
_TYPES = (torch.bfloat16, torch.float16, torch.float32)


# ---------------------------------------------------------------------------------------------------
# plain restatements
# ---------------------------------------------------------------------------------------------------
def _valid(labels, vocab, pad_idx):
    return (labels != pad_idx) & (labels >= 0) & (labels < vocab)


def _bounds(cu, rows):
    """Offsets within the rows and in order, as the kernels take them."""
    return cu.long().clamp(0, rows).cummax(0).values


def token_logprobs_reference(logits, labels, pad_idx=0, temperature=1.0):
    lf = (logits if logits.dtype == torch.float64 else logits.float()) * (1.0 / temperature)
    valid = _valid(labels, logits.shape[1], pad_idx)
    lf = lf.masked_fill(~valid[:, None], 0.0)                   # NaN in rows of padding would reach their gradient
    lp = torch.log_softmax(lf, -1).gather(1, labels.masked_fill(~valid, 0)[:, None]).squeeze(1)
    return torch.where(valid, lp, torch.zeros_like(lp))


def preference_loss_reference(logits, labels, cu, ref_logprobs=None, beta=0.1, kind="sigmoid", smoothing=0.0, margin=0.0, nll_weight=0.0,
                              average=False, pad_idx=0, temperature=1.0):
    rows = torch.arange(logits.shape[0], device=cu.device)
    ends = _bounds(cu, logits.shape[0])
    labels = labels.masked_fill((rows < ends[0]) | (rows >= ends[-1]), pad_idx)
    lp = token_logprobs_reference(logits, labels, pad_idx, temperature)
    valid = _valid(labels, logits.shape[1], pad_idx)
    cu_l = ends.tolist()
    bounds = list(zip(cu_l[:-1], cu_l[1:]))
    scores = torch.stack([lp[a:b].sum() for a, b in bounds]) if bounds else lp[:0]          # no pair: a loss of 0 with a gradient of 0
    count = torch.tensor([max(int(valid[a:b].sum()), 1) for a, b in bounds], dtype=lp.dtype, device=lp.device)
    each = 1.0 / count if average else torch.ones_like(scores)
    ratio = (scores if ref_logprobs is None else scores - ref_logprobs.to(lp.dtype)) * each
    h = ratio[0::2] - ratio[1::2]
    if kind == "ipo":
        loss = (h - 0.5 / beta) ** 2
    else:
        z = beta * h - margin
        if kind == "hinge":
            loss = torch.relu(1.0 - z) * torch.where(torch.isnan(z), z, torch.ones_like(z)).detach()      # NaN shows in the gradient, too
        else:
            loss = -(1.0 - smoothing) * F.logsigmoid(z)
        if smoothing:                                           # 0 * inf at z = inf otherwise
            loss = loss - smoothing * F.logsigmoid(-z)
    if nll_weight:
        loss = loss - nll_weight * (scores * each)[0::2]
    return loss.sum().reshape(1), (h > 0).sum().to(lp.dtype).reshape(1), scores.detach()


def policy_loss_reference(logits, labels, old_logprobs, advantages, ref_logprobs=None, clip=0.2, clip_high=None, kl_coef=0.0, pad_idx=0,
                          temperature=1.0):
    lp = token_logprobs_reference(logits, labels, pad_idx, temperature)
    valid = _valid(labels, logits.shape[1], pad_idx)
    zero = torch.zeros_like(lp)
    adv = advantages.to(lp.dtype)
    delta = torch.where(valid, lp - old_logprobs.to(lp.dtype), zero)
    ratio = torch.exp(delta.detach())
    held = ratio.clamp(1.0 - clip, 1.0 + (clip if clip_high is None else clip_high))
    clipped = valid & (ratio * adv > held * adv)
    # where a ratio is clipped, the exponential has no part in the gradient: 0 * inf otherwise
    loss = torch.where(valid, -torch.where(clipped, held, torch.exp(torch.where(clipped, zero, delta))) * adv, zero)
    kl = zero
    if ref_logprobs is not None:
        d = torch.where(valid, ref_logprobs.to(lp.dtype) - (lp if kl_coef else lp.detach()), zero)
        kl = torch.where(d == float("inf"), torch.exp(d), torch.expm1(d) - d)      # inf, not inf - inf, for a word of probability 0
        if kl_coef:                                             # a KL term that is only reported may be infinite
            loss = loss + kl_coef * kl
    return loss.sum().reshape(1), clipped.sum().to(lp.dtype).reshape(1), kl.detach().sum().reshape(1), lp.detach()


# ---------------------------------------------------------------------------------------------------
# arguments
# ---------------------------------------------------------------------------------------------------
def _check_rows(logits, labels, temperature):
    if logits.dim() != 2 or labels.dim() != 1 or labels.shape[0] != logits.shape[0]:
        raise ValueError("logits must be [rows, vocab] and labels [rows], got %s and %s" % (tuple(logits.shape), tuple(labels.shape)))
    if logits.shape[1] < 1:
        raise ValueError("the vocabulary is empty")
    if labels.dtype not in (torch.int64, torch.int32):
        raise TypeError("labels must be int64 or int32")
    if not logits.is_floating_point():
        raise TypeError("logits must be floating-point")
    if labels.device != logits.device:
        raise ValueError("labels are on %s, logits on %s" % (labels.device, logits.device))
    if not 1e-30 <= temperature <= 1e30:
        raise ValueError("temperature must be positive (from 1e-30 to 1e30)")


def _check_vector(t, n, logits, name):
    if t.dim() != 1 or t.shape[0] != n:
        raise ValueError("%s must hold %d numbers, got %s" % (name, n, tuple(t.shape)))
    if t.device != logits.device:
        raise ValueError("%s is on %s, logits on %s" % (name, t.device, logits.device))
    if t.requires_grad:
        raise ValueError("%s has no gradient here: detach it" % name)


def _kernel_takes(logits):
    return logits.is_cuda and logits.dtype in _TYPES


def _as_rows(logits):
    """Rows of adjacent elements that do not overlap (a transposed or expanded matrix is copied)."""
    return logits if logits.stride(1) == 1 and (logits.shape[0] <= 1 or logits.stride(0) >= logits.shape[1]) else logits.contiguous()


def _scale_args(grad_scale, logits):
    if grad_scale is None:
        return None, 1.0
    if isinstance(grad_scale, torch.Tensor):
        if grad_scale.numel() != 1 or grad_scale.device != logits.device:
            raise ValueError("grad_scale must be one element on the logits' device")
        return grad_scale.detach().float().reshape(1), 1.0
    return None, float(grad_scale)


# ---------------------------------------------------------------------------------------------------
# log-probabilities
# ---------------------------------------------------------------------------------------------------
def token_logprobs(logits, labels, pad_idx: int = 0, temperature: float = 1.0):
    """Log-probability of every label under ``softmax(logits / temperature)``: fp32 ``[rows]``, 0 in rows of padding.  Differentiable with
    respect to the logits (any objective over the log-probabilities of words: minimum risk, sequence-level rewards); without gradients one
    pass that reads the logits once (scores of a frozen model)."""
    _check_rows(logits, labels, temperature)
    if not _kernel_takes(logits):
        return token_logprobs_reference(logits, labels.long(), pad_idx, temperature)
    x, y = _as_rows(logits), labels.long().contiguous()
    LAUNCHES[0] += 2
    if torch.is_grad_enabled() and logits.requires_grad:
        return ext().row_scores_node(x, y, int(pad_idx), float(temperature))
    return ext().row_scores(x, y, int(pad_idx), float(temperature), False)[0]


def sequence_logprobs(logprobs, cu):
    """Sums of the words' log-probabilities over the sequences of ``cu``: what ``preference_loss`` takes from the frozen model.  fp32, summed in
    64 bits.  A sequence with a word of probability 0, or with NaN, is that and no other one.  Offsets are put in order as there."""
    if logprobs.dim() != 1 or cu.dim() != 1 or cu.shape[0] < 1:
        raise ValueError("sequence_logprobs: log-probabilities [rows] and offsets [sequences + 1], got %s and %s" % (tuple(logprobs.shape), tuple(cu.shape)))
    bounds = _bounds(cu, logprobs.shape[0])
    sums = lambda t: torch.diff(torch.cat([t.new_zeros(1), t.cumsum(0)])[bounds])
    lp = logprobs.double()
    finite = torch.isfinite(lp)
    total = sums(lp.masked_fill(~finite, 0.0))
    total = total.masked_fill(sums((lp == -float("inf")).double()) > 0, -float("inf"))
    return total.masked_fill(sums((~finite & (lp != -float("inf"))).double()) > 0, float("nan")).to(logprobs.dtype)


# ---------------------------------------------------------------------------------------------------
# losses
# ---------------------------------------------------------------------------------------------------
def _run_reference(out, grad_scale, logits):
    if grad_scale is None or not torch.is_grad_enabled():
        return out
    s = grad_scale if isinstance(grad_scale, torch.Tensor) else torch.tensor(float(grad_scale))
    return (ref.scale_gradient(out[0], s.to(logits.device)),) + out[1:]


def preference_loss(logits, labels, cu, ref_logprobs: Optional[torch.Tensor] = None, beta: float = 0.1, kind: str = "sigmoid",
                    smoothing: float = 0.0, margin: float = 0.0, nll_weight: float = 0.0, average: bool = False, pad_idx: int = 0,
                    temperature: float = 1.0, grad_scale=None, inplace: bool = False):
    """Paired preference loss.  The rows are packed sequences with offsets ``cu [2 * pairs + 1]``: sequence ``2i`` is the preferred
    translation of pair ``i``, sequence ``2i + 1`` the rejected one; rows outside every sequence count as padding, and
    offsets that fall or leave the rows are put in order (running maximum, clamped).  With ``lp`` a sequence's
    summed log-probability and ``ref_logprobs [2 * pairs]`` the frozen model's (None: no reference),

        ``h = (lp_w - ref_w) - (lp_l - ref_l)``,  ``z = beta * h - margin``

    and ``kind`` "sigmoid" ``-(1 - smoothing) log sigmoid(z) - smoothing log sigmoid(-z)``, "hinge" ``max(0, 1 - z)``, "ipo"
    ``(h - 1 / (2 beta))^2``, plus ``- nll_weight * lp_w``.  ``average`` divides ``lp`` and ``ref`` by the sequence's number of words.

    Returns ``(loss_sum [1], n_ranked [1], lp [2 * pairs])``: the sum over pairs, the number of pairs with ``h > 0``, the sequences'
    log-probabilities (no gradient)."""
    _check_rows(logits, labels, temperature)
    if cu.dim() != 1 or cu.shape[0] % 2 != 1 or cu.dtype not in (torch.int32, torch.int64) or cu.device != logits.device:
        raise ValueError("cu must be 2 * pairs + 1 integer offsets on the logits' device")
    if kind not in KINDS:
        raise ValueError("kind must be one of %s, not %r" % (sorted(KINDS), kind))
    if not beta > 0.0:
        raise ValueError("beta must be positive")
    if not 0.0 <= smoothing < 1.0 or (smoothing and kind != "sigmoid"):
        raise ValueError("smoothing must be in [0, 1), and 0 with kind %r" % kind)
    if margin and kind == "ipo":
        raise ValueError("kind 'ipo' has no margin")
    if ref_logprobs is not None:
        _check_vector(ref_logprobs, cu.shape[0] - 1, logits, "ref_logprobs")
    scale_at, scale = _scale_args(grad_scale, logits)
    if not _kernel_takes(logits):
        return _run_reference(preference_loss_reference(logits, labels.long(), cu, ref_logprobs, beta, kind, smoothing, margin, nll_weight,
                                                        average, pad_idx, temperature), grad_scale, logits)
    x, y = _as_rows(logits), labels.long().contiguous()
    c = (cu if cu.dtype == torch.int32 else cu.clamp(0, logits.shape[0]).int()).contiguous()
    r = None if ref_logprobs is None else ref_logprobs.float().contiguous()
    cfg = (x, y, c, r, KINDS[kind], float(beta), float(smoothing), float(margin), float(nll_weight), bool(average), int(pad_idx), float(temperature))
    LAUNCHES[0] += 4
    if torch.is_grad_enabled() and logits.requires_grad:
        return ext().preference_loss_node(*cfg, bool(inplace), scale_at, scale, grad_scale is not None)
    return ext().preference_loss(*cfg, 0, scale_at, scale)[:-1]


def policy_loss(logits, labels, old_logprobs, advantages, ref_logprobs: Optional[torch.Tensor] = None, clip: float = 0.2,
                clip_high: Optional[float] = None, kl_coef: float = 0.0, pad_idx: int = 0, temperature: float = 1.0, grad_scale=None,
                inplace: bool = False):
    """Clipped policy loss with a KL term, word by word.  With ``lp`` the log-probability of a row's label, ``r = exp(lp - old_logprobs)`` and
    ``A`` the row's advantage (a sentence's, repeated over its rows),

        ``loss = sum -min(r A, clip(r, 1 - clip, 1 + clip_high) A) + kl_coef * (exp(d) - d - 1)``,  ``d = ref_logprobs - lp``

    over the rows that are not padding (``clip_high`` None: as ``clip``; ``ref_logprobs`` None: no KL term).  Returns ``(loss_sum [1], n_clipped
    [1], kl_sum [1], lp [rows])``; only the loss has a gradient."""
    _check_rows(logits, labels, temperature)
    _check_vector(old_logprobs, logits.shape[0], logits, "old_logprobs")
    _check_vector(advantages, logits.shape[0], logits, "advantages")
    if ref_logprobs is not None:
        _check_vector(ref_logprobs, logits.shape[0], logits, "ref_logprobs")
    elif kl_coef:
        raise ValueError("kl_coef without ref_logprobs")
    high = clip if clip_high is None else clip_high
    if not 0.0 <= clip <= 1.0 or not high >= 0.0:
        raise ValueError("clip must be in [0, 1] and clip_high at least 0")
    scale_at, scale = _scale_args(grad_scale, logits)
    if not _kernel_takes(logits):
        return _run_reference(policy_loss_reference(logits, labels.long(), old_logprobs, advantages, ref_logprobs, clip, high, kl_coef,
                                                    pad_idx, temperature), grad_scale, logits)
    x, y = _as_rows(logits), labels.long().contiguous()
    old, adv = old_logprobs.float().contiguous(), advantages.float().contiguous()
    r = None if ref_logprobs is None else ref_logprobs.float().contiguous()
    cfg = (x, y, old, adv, r, float(clip), float(high), float(kl_coef), int(pad_idx), float(temperature))
    LAUNCHES[0] += 2
    if torch.is_grad_enabled() and logits.requires_grad:
        return ext().policy_loss_node(*cfg, bool(inplace), scale_at, scale, grad_scale is not None)
    return ext().policy_loss(*cfg, 0, scale_at, scale)[:-1]
