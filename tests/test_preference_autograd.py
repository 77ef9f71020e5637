"""Gradients of the preference-tuning losses as autograd passes them on: upstream factors, a second pass, captured passes, logits that are
consumed.  Expected gradients are written out in 64 bits: coef * (onehot - softmax)."""

import pytest
import torch

from nmtgminor_b200 import ops
from nmtgminor_b200.ops import preference as pref

DEV = "cuda"
# rows that a warp holds, a block, a cluster of blocks, and none of them
VOCABS = [(3, 700), (40, 3000), (25, 51865), (9, 250054), (5, 458760)]


def _case(rows, vocab, dtype, which, seed=0):
    """Logits, a loss of them, the rows' coefficients in 64 bits and a bound on the kernels' error of these."""
    g = torch.Generator().manual_seed(seed + vocab)
    x = (torch.randn(rows, (vocab + 7) // 8 * 8, generator=g) * 2.5).to(dtype).to(DEV)[:, :vocab]
    y = torch.randint(1, vocab, (rows,), generator=g).to(DEV)
    y[0] = 0
    real = (y != 0).double()
    lp = torch.log_softmax(x.double(), 1).gather(1, y[:, None]).squeeze(1) * real
    word = 2 ** -19                                             # error of a log-probability: see tests/test_preference.py
    if which == "policy":
        adv = torch.randn(rows, generator=g).to(DEV)
        old = (lp + 0.02).float()                               # nothing is clipped
        ratio = torch.exp(lp - old.double())
        return x, y, lambda t, **kw: pref.policy_loss(t, y, old, adv, **kw)[0], -ratio * adv * real, 2 * word * adv.double().abs()
    cu = torch.tensor([0, rows // 3, rows], device=DEV)
    ref = torch.tensor([lp[:rows // 3].sum().item() - 3.0, lp[rows // 3:].sum().item() + 2.0], device=DEV)
    beta = 0.3
    h = lp[:rows // 3].sum() - ref[0].double() - lp[rows // 3:].sum() + ref[1].double()
    slope = -beta * torch.sigmoid(-beta * h)
    coef = torch.where(torch.arange(rows, device=DEV) < rows // 3, slope, -slope) * real
    off = (beta ** 2 / 4 * rows * word + 2 ** -22) * torch.ones(rows, dtype=torch.float64, device=DEV)
    return x, y, lambda t, **kw: pref.preference_loss(t, y, cu, ref, beta, **kw)[0], coef, off


def _close(got, coef, off, x, y, factor):
    """Half a step of fp16 (and of its smallest number), 2^-15 of an exponential, at the label of coef p, and the coefficients' error."""
    p = torch.softmax(x.double(), 1)
    hot = torch.nn.functional.one_hot(y, x.shape[1]).double()
    want = factor * coef[:, None] * (hot - p)
    bound = (2 ** -11 + 2 ** -15) * want.abs() + abs(factor) * (2 ** -15 * coef.abs()[:, None] * p * hot + off[:, None] * (hot - p).abs()) + 2 ** -25
    assert ((got.double() - want).abs() <= bound).all(), ((got.double() - want).abs() - bound).max()


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["preference", "policy"])
@pytest.mark.parametrize("rows,vocab", VOCABS)
def test_a_scaled_loss_keeps_small_gradients_in_fp16(which, rows, vocab):
    """One rounding, with the factor in: factors as loss scaling has them, and one that is no power of two; the logits' place taken or not; captured."""
    x, y, loss, coef, off = _case(rows, vocab, torch.float16, which)
    for factor in (2.0 ** 12, 1000.0 / 3.0, 1.0, -2.0 ** -4):
        leaf = x.detach().requires_grad_(True)
        grad = torch.autograd.grad(loss(leaf) * factor, leaf)[0]
        _close(grad, coef, off, x, y, factor)
        assert (grad[0] == 0).all() and grad.stride() == x.stride()
        scaled = torch.autograd.grad(loss(leaf, grad_scale=factor), leaf)[0]
        assert torch.equal(scaled, grad)
        wide = torch.zeros(x.shape[0], x.stride(0), dtype=x.dtype, device=DEV)
        wide[:, x.shape[1]:] = 7.0
        consumed = wide[:, :x.shape[1]].copy_(x).detach().requires_grad_(True)
        version = consumed._version
        over = torch.autograd.grad(loss(consumed, inplace=True) * factor, consumed)[0]
        assert torch.equal(over, grad) and over.data_ptr() == consumed.data_ptr() and consumed._version > version
        assert (wide[:, x.shape[1]:] == 7.0).all()
    leaf = x.detach().requires_grad_(True)
    grad = torch.autograd.grad(loss(leaf) * 3.0, leaf)[0]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = torch.autograd.grad(loss(leaf) * 3.0, leaf)[0]
    for _ in range(2):
        captured.fill_(7.0)
        graph.replay()
        assert torch.equal(captured, grad)
    assert ops.check_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["preference", "policy"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_one_backward_pass_of_a_loss(which, dtype):
    """A second pass is refused in every type; logits overwritten before an fp16 gradient is made of them, too, and create_graph."""
    x, y, loss, coef, off = _case(12, 3000, dtype, which)
    leaf = x.detach().requires_grad_(True)
    value = loss(leaf)
    value.backward(retain_graph=True)
    with pytest.raises(RuntimeError, match="second backward"):
        value.backward()
    with pytest.raises(RuntimeError):
        torch.autograd.grad(loss(leaf), leaf, create_graph=True)
    if dtype == torch.float16:
        logits = leaf * 1.0
        value = loss(logits)
        with torch.no_grad():
            logits.zero_()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            value.backward()
    none = x[:0].detach().requires_grad_(True)
    zero = torch.zeros(0, device=DEV)
    empty = pref.policy_loss(none, y[:0], zero, zero)[0] if which == "policy" else pref.preference_loss(none, y[:0], torch.zeros(3, dtype=torch.int32, device=DEV))[0]
    assert torch.autograd.grad(empty * 3.0, none)[0].shape == none.shape
    outside = x.detach().requires_grad_(True)                   # no pair at all: a gradient of zeros
    assert (torch.autograd.grad(pref.preference_loss(outside, y, torch.zeros(1, dtype=torch.int32, device=DEV))[0] * 3.0, outside)[0] == 0).all()
    assert ops.check_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["preference", "policy"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("scale", [None, 0.5])
def test_what_a_loss_keeps_is_a_saved_tensor(which, dtype, scale):
    """The gradient (or what it is made of) can be moved off the GPU by hooks, and is freed with the pass; logits consumed in place and changed behind
    the call are refused."""
    x, y, loss, coef, off = _case(20, 9001, dtype, which)
    kw = {} if scale is None else {"grad_scale": scale}
    leaf = x.detach().requires_grad_(True)
    want = torch.autograd.grad(loss(leaf, **kw) * 2.0, leaf)[0]
    moved = []

    def pack(t):
        moved.append(t.numel())
        return t.cpu()

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t.to(DEV)):
        value = loss(leaf, **kw)
    assert max(moved) == x.numel()
    assert torch.equal(torch.autograd.grad(value * 2.0, leaf)[0], want)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    value = loss(leaf, **kw)
    grad = torch.autograd.grad(value * 2.0, leaf)[0]
    assert torch.equal(grad, want)
    del grad
    assert torch.cuda.memory_allocated() - before <= 1024       # the loss itself
    with pytest.raises(RuntimeError, match="second"):
        torch.autograd.grad(value, leaf)
    logits = x.detach().clone().requires_grad_(True) * 1.0
    value = loss(logits, inplace=True, **kw)
    with torch.no_grad():
        logits.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        value.backward()
    assert ops.check_status() == 0


@pytest.mark.gpu
def test_losses_from_several_threads():
    """Threads with a stream each, first calls among them, of rows of every length: the results of calls one after another."""
    from concurrent.futures import ThreadPoolExecutor
    cases = [_case(11, vocab, dtype, which, 7) for vocab in (2600, 5300, 12000, 17000, 33000, 66000) for dtype in (torch.bfloat16, torch.float32)
             for which in ("preference", "policy")]
    streams = [torch.cuda.Stream() for _ in range(6)]
    torch.cuda.synchronize()

    def run(i):
        x, y, loss = cases[i % len(cases)][:3]
        with torch.cuda.stream(streams[i % 6]):
            leaf = x.detach().requires_grad_(True)
            out = loss(leaf), pref.token_logprobs(leaf, y)
            grads = [torch.autograd.grad(o.sum(), leaf)[0] for o in out]
            streams[i % 6].synchronize()
        return [o.detach() for o in out] + grads

    with ThreadPoolExecutor(6) as pool:
        together = list(pool.map(run, range(2 * len(cases))))
    alone = [run(i) for i in range(len(cases))]
    for i, got in enumerate(together):
        assert all(torch.equal(a, b) for a, b in zip(got, alone[i % len(cases)]))
    assert ops.check_status() == 0
