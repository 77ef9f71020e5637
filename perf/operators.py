"""Timed operators of preference tuning: what a step of it does beyond the products, norms and attention of ordinary training.

Five operators, each in its plain form (elementary torch operations in 32 bits, rounded once) and as the framework's own call:

* ``logprobs``    log-probability of every target word from a matrix of logits: the scoring pass of the frozen model, and with
  ``grad`` the gradient of a weighted sum of them;
* ``preference``  the paired loss ``-log sigmoid(beta * ((w - ref_w) - (l - ref_l)))`` over summed log-probabilities of a preferred
  translation w and a rejected one l (sequences 2i and 2i + 1), and its gradient with respect to the logits;
* ``policy``      the clipped policy loss with a KL term, ``-min(r A, clip(r) A) + k (e^d - d - 1)`` with ``r = exp(lp - old)`` and
  ``d = ref - lp``, word by word, and its gradient with respect to the logits;
* ``embedding``   lookup with scaling, and its gradient, every row's sum taken in the order of the tokens;
* ``kept``        activations that wait for the backward pass in 8 bits (blocks of 32 elements of a row share a power of two, the
  elements are 4-bit-exponent, 3-bit-mantissa numbers): an activation function that keeps its input so, and a linear layer that
  keeps its input so for the gradient of its weights.

Vocabularies are those of ``bench.py`` and ``bench_speech.py`` (8000, 32000, Whisper's 51865, mBART-50's 250054), widths those of
the same models, lengths 10 to 120 words, as there.  Logits of an odd vocabulary lie in rows padded to 16 bytes, as the framework's
own output layer leaves them; drawn cases have dense rows, too.
"""
import math

import numpy as np
import torch

own = False

PAD = 0
BLOCK = 32                       # elements that share a power of two
BETA, CLIP, KL = 0.1, 0.2, 0.05
MOST_LOGITS = 390_000_000        # elements of the largest drawn matrix of logits
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # the frozen model's score of one translation: latency
        {"name": "score one sentence", "op": "logprobs", "rows": 37, "vocab": 32000, "type": "bf16", "padded": True, "grad": False},
        # scores of a batch of transcripts with gradients (minimum-risk training, any objective a user writes himself)
        {"name": "score transcripts, with gradient", "op": "logprobs", "rows": 3584, "vocab": 51865, "type": "bf16", "padded": True,
         "grad": True},
        # a few pairs on a small model: what the loss costs beyond its bytes
        {"name": "preference small", "op": "preference", "pairs": 4, "lo": 10, "hi": 50, "vocab": 8000, "type": "bf16", "padded": True},
        # 68 pairs of Transformer-big, about 8200 target words: the ordinary step
        {"name": "preference big", "op": "preference", "pairs": 68, "lo": 20, "hi": 100, "vocab": 32000, "type": "bf16", "padded": True},
        # mBART-50's vocabulary: rows of half a megabyte
        {"name": "preference large vocabulary", "op": "preference", "pairs": 12, "lo": 20, "hi": 110, "vocab": 250054, "type": "bf16",
         "padded": True},
        # sampled translations of a small model with 32-bit logits
        {"name": "policy small", "op": "policy", "rows": 300, "vocab": 8000, "type": "fp32", "padded": False},
        # 64 sentences with 4 samples each: the ordinary step
        {"name": "policy big", "op": "policy", "rows": 15360, "vocab": 32000, "type": "bf16", "padded": True},
        # the default widths of a development run
        {"name": "embedding tiny", "op": "embedding", "rows": 960, "vocab": 8000, "width": 256, "type": "bf16", "into": "dense"},
        # Transformer-big through the flat gradient buffer that the trainer clears and accumulates into
        {"name": "embedding big", "op": "embedding", "rows": 8200, "vocab": 32000, "width": 1024, "type": "bf16", "into": "flat"},
        # a long batch on mBART-50's table, 32-bit weights
        {"name": "embedding large vocabulary", "op": "embedding", "rows": 65536, "vocab": 250054, "width": 1024, "type": "fp32",
         "into": "dense"},
        # the feed-forward block of Transformer-big: its GELU
        {"name": "activation kept", "op": "kept", "part": "activation", "rows": 8200, "width": 4096, "act": "gelu"},
        # and its second linear layer
        {"name": "linear kept", "op": "kept", "part": "linear", "rows": 8200, "width": 4096, "out": 1024},
    ]


def _between(rng, lo, hi):
    """Whole number from ``lo`` to ``hi``, even over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["logprobs", "preference", "preference", "policy", "policy", "embedding", "embedding", "kept"])
    kind = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "embedding":
        vocab = _between(rng, 500, 250054)
        width = rng.choice([64, 200, 256, 300, 512, 768, 1000, 1024, 1280])
        into = rng.choice(["dense", "flat"])
        if into == "flat":                    # the flat store's working copies are bf16, its embedding kernels 16 elements wide
            kind, width = "bf16", width // 16 * 16
        return {"op": op, "rows": _between(rng, 1, 65536), "vocab": vocab, "width": width, "type": kind, "into": into}
    if op == "kept":
        if rng.random() < 0.5:
            return {"op": op, "part": "activation", "rows": _between(rng, 1, 8200), "width": _between(rng, 8, 4096),
                    "act": rng.choice(["relu", "gelu", "silu"])}
        return {"op": op, "part": "linear", "rows": _between(rng, 1, 8200), "width": _between(rng, 8, 512) * 8,
                "out": _between(rng, 8, 128) * 8}
    vocab = _between(rng, 300, 250054)
    case = {"vocab": vocab, "type": kind, "padded": rng.random() < 0.6}
    most = max(1, min(20000, (MOST_LOGITS if kind != "fp32" else MOST_LOGITS // 2) // vocab))
    if op == "preference":
        hi = _between(rng, 4, max(4, min(400, most // 2)))
        return dict(case, op=op, pairs=_between(rng, 1, max(1, min(200, most // (2 * hi + 2)))), lo=rng.randint(1, hi), hi=hi)
    case = dict(case, op=op, rows=_between(rng, 1, most))
    return dict(case, grad=rng.random() < 0.7) if op == "logprobs" else case


# ---------------------------------------------------------------------------------------------------------------------
# inputs, from the seed alone
# ---------------------------------------------------------------------------------------------------------------------
def _offsets(case):
    """Offsets of the 2 * pairs sequences: the same for every seed, so that every batch of a case is the same amount of work."""
    r = np.random.RandomState(17 + case["pairs"])
    return np.concatenate([[0], np.cumsum(r.randint(case["lo"], case["hi"] + 1, size=2 * case["pairs"]))]).astype(np.int32)


def _rows(case):
    return int(_offsets(case)[-1]) if case["op"] == "preference" else case["rows"]


def _zipf(g, n, vocab):
    """Word ids as a text has them: the k-th word with a share of about 1 / k; three in a hundred are padding."""
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    ids = torch.exp(u * math.log(vocab)).long().clamp(1, vocab - 1)
    return torch.where(torch.rand(n, generator=g, device="cuda") < 0.03, torch.full_like(ids, PAD), ids)


def _row_scores(logits, labels):
    """Log-probabilities of the labels in 64 bits, a few rows at a time."""
    out = []
    for r in range(0, logits.shape[0], 512):
        x = logits[r:r + 512].double()
        out.append(x.gather(1, labels[r:r + 512, None]).squeeze(1) - torch.logsumexp(x, 1))
    return torch.cat(out)


def _logits(case, g, n):
    """Logits with the spread of a trained model's, the target word favoured in most rows."""
    vocab, kind = case["vocab"], TYPES[case["type"]]
    each = 16 // torch.empty((), dtype=kind).element_size()
    width = (vocab + each - 1) // each * each if case["padded"] else vocab
    x = torch.randn(n, width, generator=g, device="cuda", dtype=kind)[:, :vocab]
    x *= 2.5
    labels = _zipf(g, n, vocab)
    favour = 12.0 * torch.rand(n, generator=g, device="cuda")
    x[torch.arange(n, device="cuda"), labels] += favour.to(kind)
    return x, labels


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case}
    n = _rows(case)
    normal = lambda *shape: torch.randn(*shape, generator=g, device="cuda")
    if case["op"] in ("logprobs", "preference", "policy"):
        s["logits"], s["labels"] = _logits(case, g, n)
        if case["op"] == "logprobs":
            if case["grad"]:
                s["weights"] = normal(n)
        else:
            lp = torch.where(s["labels"] == PAD, 0.0, _row_scores(s["logits"], s["labels"]))
            if case["op"] == "preference":
                cu = torch.from_numpy(_offsets(case)).cuda()
                ends = torch.cat([lp.new_zeros(1), lp.cumsum(0)])[cu.long()]
                s["cu"], s["ref"] = cu, (ends[1:] - ends[:-1] + 8.0 * normal(2 * case["pairs"])).float()
            else:
                s["old"], s["ref"] = (lp + 0.15 * normal(n)).float(), (lp + 0.3 * normal(n)).float()
                s["advantages"] = normal(n)
        if case["op"] != "logprobs" or case["grad"]:
            s["logits"].requires_grad_(True)
    elif case["op"] == "embedding":
        kind, vocab, width = TYPES[case["type"]], case["vocab"], case["width"]
        s["tokens"] = _zipf(g, n, vocab)
        table = (normal(vocab, width) / math.sqrt(width)).to(kind)
        s["table"] = torch.nn.Parameter(table)
        if case["into"] == "flat":           # what parallel.flat.FlatParameterStore attaches to a parameter
            s["table"].work, s["table"].main_grad = table, torch.zeros(vocab, width, device="cuda")
        s["dy"] = (0.01 * normal(n, width)).to(kind)
    else:
        x = normal(n, case["width"]) * 1.5
        x[:, normal(case["width"]) > 2.5] *= 20.0                      # the few large channels that trained models have
        s["x"] = x.bfloat16().requires_grad_(True)
        if case["part"] == "activation":
            s["dy"] = (0.01 * normal(n, case["width"])).bfloat16()
        else:
            weight = (normal(case["out"], case["width"]) / math.sqrt(case["width"])).bfloat16()
            bias = (0.1 * normal(case["out"])).bfloat16()
            s["weight"], s["bias"] = torch.nn.Parameter(weight.float()), torch.nn.Parameter(bias.float())
            for p, work in ((s["weight"], weight), (s["bias"], bias)):
                p.work, p.main_grad = work, torch.zeros(work.shape, device="cuda")
            s["dy"] = (0.01 * normal(n, case["out"])).bfloat16()
    return s


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def run(s):
    return (_own if own else _plain)(s)


def _own(s):
    from nmtgminor_b200 import ops
    from nmtgminor_b200.ops import kept, preference
    case = s["case"]
    if case["op"] == "logprobs":
        if not case["grad"]:
            return {"logprobs": preference.token_logprobs(s["logits"], s["labels"], pad_idx=PAD)}
        lp = preference.token_logprobs(s["logits"], s["labels"], pad_idx=PAD)
        return {"logprobs": lp.detach(), "grad": torch.autograd.grad(lp, s["logits"], s["weights"])[0]}
    if case["op"] == "preference":
        loss, correct, scores = preference.preference_loss(s["logits"], s["labels"], s["cu"], s["ref"], beta=BETA, pad_idx=PAD)
        grad = torch.autograd.grad(loss, s["logits"])[0]
        return {"loss": loss.detach(), "correct": correct, "scores": scores, "grad": grad}
    if case["op"] == "policy":
        loss, clipped, kl, lp = preference.policy_loss(s["logits"], s["labels"], s["old"], s["advantages"], s["ref"], clip=CLIP,
                                                       kl_coef=KL, pad_idx=PAD)
        grad = torch.autograd.grad(loss, s["logits"])[0]
        return {"loss": loss.detach(), "clipped": clipped, "kl": kl, "logprobs": lp, "grad": grad}
    if case["op"] == "embedding":
        table, scale = s["table"], math.sqrt(case["width"])
        if case["into"] == "flat":
            table.main_grad.zero_()
            out = ops.embedding(s["tokens"], table, scale=scale, pad_idx=PAD, sorted_grad=True)
            out.backward(s["dy"])
            return {"out": out.detach(), "grad": table.main_grad}
        out = ops.embedding(s["tokens"], table, scale=scale, pad_idx=PAD, sorted_grad=True)
        return {"out": out.detach(), "grad": torch.autograd.grad(out, table, s["dy"])[0]}
    if case["part"] == "activation":
        y = kept.activation(s["x"], case["act"])
        return {"y": y.detach(), "dx": torch.autograd.grad(y, s["x"], s["dy"])[0]}
    s["weight"].main_grad.zero_()
    s["bias"].main_grad.zero_()
    y = ops.linear(s["x"], s["weight"], s["bias"], keep8=True)
    dx = torch.autograd.grad(y, s["x"], s["dy"])[0]
    return {"y": y.detach(), "dx": dx, "dw": s["weight"].main_grad, "db": s["bias"].main_grad}


def _softmax_parts(x, labels):
    """(exp(x - max), its sums, log-probabilities of the labels) of a matrix of logits; the log-probabilities in 64 bits."""
    x = x.float()
    top = x.amax(1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(1)
    at = x.gather(1, labels[:, None]).squeeze(1)
    lp = at.double() - top.squeeze(1).double() - torch.log(total.double())
    return e, total, torch.where(labels == PAD, 0.0, lp)


def _logits_grad(e, total, labels, coef, kind):
    """coef * (onehot - softmax), rows of padding zero."""
    coef = torch.where(labels == PAD, 0.0, coef.float())
    g = e * (-coef / total)[:, None]
    g[torch.arange(g.shape[0], device=g.device), labels] += coef
    return g.to(kind)


def _round_e4m3(v):
    """Nearest number of 4 exponent and 3 mantissa bits, ties to even, for magnitudes up to 448."""
    return v.to(torch.float8_e4m3fn).to(v.dtype)


def _kept_values(x):
    """x as blocks of 32 elements of a row with a shared power of two hold it: the smallest power that brings the block's largest
    magnitude to 448 or less."""
    rows, width = x.shape
    full = torch.nn.functional.pad(x.float(), (0, -width % BLOCK)).view(rows, -1, BLOCK)
    fraction, exponent = torch.frexp(full.abs().amax(-1, keepdim=True))
    exponent = torch.where(fraction > 0.875, exponent - 8, exponent - 9).clamp(-127, 127)
    exponent = torch.where(fraction == 0, torch.full_like(exponent, -127), exponent)
    return torch.ldexp(_round_e4m3(torch.ldexp(full, -exponent)), exponent).view(rows, -1)[:, :width]


def _plain(s):
    case = s["case"]
    with torch.no_grad():
        if case["op"] in ("logprobs", "preference", "policy"):
            x, labels, kind = s["logits"].detach(), s["labels"], TYPES[case["type"]]
            e, total, lp = _softmax_parts(x, labels)
            real = labels != PAD
            if case["op"] == "logprobs":
                out = {"logprobs": lp.float()}
                if case["grad"]:
                    out["grad"] = _logits_grad(e, total, labels, s["weights"], kind)
                return out
            if case["op"] == "preference":
                cu = s["cu"].long()
                ends = torch.cat([lp.new_zeros(1), lp.cumsum(0)])[cu]
                scores = ends[1:] - ends[:-1]
                ratio = scores - s["ref"].double()
                z = BETA * (ratio[0::2] - ratio[1::2])
                loss = torch.log1p(torch.exp(-z.abs())) + torch.clamp(-z, min=0.0)
                slope = -BETA / (1.0 + torch.exp(z))
                coef = torch.stack([slope, -slope], 1).reshape(-1)
                coef = coef[torch.bucketize(torch.arange(x.shape[0], device=x.device), cu[1:], right=True)]
                return {"loss": loss.sum().reshape(1).float(), "correct": (z > 0).sum().reshape(1).float(), "scores": scores.float(),
                        "grad": _logits_grad(e, total, labels, coef, kind)}
            ratio, adv = torch.exp(lp - s["old"].double()), s["advantages"].double()
            ahead = s["ref"].double() - lp
            plain, held = ratio * adv, ratio.clamp(1.0 - CLIP, 1.0 + CLIP) * adv
            free = plain <= held
            kl = torch.where(real, torch.exp(ahead) - ahead - 1.0, 0.0)
            loss = torch.where(real, -torch.minimum(plain, held), 0.0) + KL * kl
            coef = torch.where(free, -plain, 0.0) + KL * (1.0 - torch.exp(ahead))
            return {"loss": loss.sum().reshape(1).float(), "clipped": (real & ~free).sum().reshape(1).float(),
                    "kl": kl.sum().reshape(1).float(), "logprobs": lp.float(), "grad": _logits_grad(e, total, labels, coef, kind)}
        if case["op"] == "embedding":
            table, scale, tokens = s["table"].detach(), math.sqrt(case["width"]), s["tokens"]
            out = (table[tokens].float() * scale).to(table.dtype)
            real = (tokens != PAD).float()[:, None]
            grad = torch.zeros(table.shape, device=table.device).index_add_(0, tokens, s["dy"].float() * (scale * real))
            return {"out": out, "grad": grad if case["into"] == "flat" else grad.to(table.dtype)}
        x, dy = s["x"].detach(), s["dy"]
        held = _kept_values(x)
        if case["part"] == "activation":
            return {"y": _act(x.float(), case["act"])[0].bfloat16(), "dx": (dy.float() * _act(held, case["act"])[1]).bfloat16()}
        w, b = s["weight"].work.float(), s["bias"].work.float()
        return {"y": (x.float() @ w.t() + b).bfloat16(), "dx": (dy.float() @ w).bfloat16(), "dw": dy.float().t() @ held,
                "db": dy.float().sum(0)}


def _act(z, name):
    """The activation function and its slope."""
    if name == "relu":
        return z.clamp(min=0.0), (z > 0).to(z.dtype)
    if name == "gelu":
        area = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
        return z * area, area + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    gate = 1.0 / (1.0 + torch.exp(-z))
    return z * gate, gate * (1.0 + z * (1.0 - gate))


# ---------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "embedding":
        if case["rows"] * case["width"] + case["vocab"] * case["width"] > 600_000_000:
            return None
        tokens, scale = s["tokens"], case["width"] ** 0.5
        table, dy = s["table"].detach().double(), s["dy"].double()
        dy[tokens == PAD] = 0.0
        order = torch.argsort(tokens, stable=True)
        grad = torch.zeros_like(table)
        grad.index_put_((tokens[order],), scale * dy[order], accumulate=True)
        return {"out": scale * table[tokens], "grad": grad}
    if case["op"] == "kept":
        x, dy = s["x"].detach().double(), s["dy"].double()
        held = _exact_kept(x)
        if case["part"] == "linear":
            w, b = s["weight"].work.double(), s["bias"].work.double()
            return {"y": torch.addmm(b, x, w.t()), "dx": dy @ w, "dw": dy.t() @ held, "db": dy.sum(0)}
        probe = held.clone().requires_grad_(True)
        fn = {"relu": torch.relu, "gelu": torch.nn.functional.gelu, "silu": torch.nn.functional.silu}[case["act"]]
        with torch.enable_grad():
            slope = torch.autograd.grad(fn(probe).sum(), probe)[0]
        return {"y": fn(x), "dx": dy * slope}
    logits, labels = s["logits"].detach(), s["labels"]
    lp = _row_scores(logits, labels).masked_fill(labels == PAD, 0.0)
    out = {}
    if case["op"] == "logprobs":
        out["logprobs"] = lp
        weight = s.get("weights")
    else:
        free = lp.clone().requires_grad_(True)            # the losses as functions of the log-probabilities
        with torch.enable_grad():
            if case["op"] == "preference":
                lengths = np.diff(s["cu"].cpu().numpy()).tolist()
                scores = torch.stack([part.sum() for part in free.split(lengths)])
                ratio = (scores - s["ref"].double()).view(-1, 2)
                z = BETA * (ratio[:, 0] - ratio[:, 1])
                loss = -torch.nn.functional.logsigmoid(z).sum()
                out["loss"], out["correct"], out["scores"] = loss.detach().view(1), (z > 0).sum().double().view(1), scores.detach()
            else:
                real = labels != PAD
                r, a = (free - s["old"].double()).exp(), s["advantages"].double()
                d = s["ref"].double() - free
                kl = ((d.exp() - d - 1.0) * real).sum()
                low, high = r * a, r.clip(1.0 - CLIP, 1.0 + CLIP) * a
                loss = KL * kl - (torch.where(low <= high, low, high) * real).sum()
                out.update(loss=loss.detach().view(1), clipped=((low > high) & real).sum().double().view(1), kl=kl.detach().view(1),
                           logprobs=lp)
        weight = torch.autograd.grad(loss, free)[0]
    if weight is not None:
        weight = weight.double().masked_fill(labels == PAD, 0.0)
        grad = torch.empty(logits.shape, dtype=torch.float64, device=logits.device)
        for r in range(0, logits.shape[0], 512):
            p = torch.softmax(logits[r:r + 512].double(), 1).neg_()
            p.scatter_add_(1, labels[r:r + 512, None], torch.ones_like(p[:, :1]))
            torch.mul(p, weight[r:r + 512, None], out=grad[r:r + 512])
        out["grad"] = grad
    return out


def _exact_kept(x):
    rows, width = x.shape
    blocks = torch.nn.functional.pad(x, (0, -width % BLOCK)).view(rows, -1, BLOCK)
    most = blocks.abs().amax(2, keepdim=True)
    power = torch.ceil(torch.log2(most / 448.0)).clamp(-127, 127)              # -inf of a block of zeros: -127
    unit = torch.exp2(power)
    v = blocks / unit
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3.0)
    return (torch.round(v / step) * step * unit).view(rows, -1)[:, :width]


# ---------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------
def work(case):
    n = _rows(case)
    if case["op"] in ("logprobs", "preference", "policy"):
        size = TYPES[case["type"]].itemsize
        grad = case["op"] != "logprobs" or case["grad"]
        return {"bytes": n * case["vocab"] * size * (2 if grad else 1) + 24 * n, "flops": n * case["vocab"] * (7 if grad else 4)}
    if case["op"] == "embedding":
        size, width, vocab = TYPES[case["type"]].itemsize, case["width"], case["vocab"]
        used = vocab * (1.0 - (1.0 - 1.0 / vocab) ** n) if n < vocab else vocab       # rows looked up, at most
        grads = vocab * width * (4 if case["into"] == "flat" else size)
        return {"bytes": int(min(n, used) * width * size + 2 * n * width * size + grads + 8 * n), "flops": 3 * n * width}
    if case["part"] == "activation":
        return {"bytes": n * case["width"] * 10, "flops": 30 * n * case["width"]}
    width, out = case["width"], case["out"]
    return {"bytes": 2 * n * (2 * width + 2 * out) + 2 * 2 * width * out + 4 * width * out, "flops": 6 * n * width * out}
