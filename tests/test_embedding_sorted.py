"""The embedding gradient by sorted tokens: against sums in 64 bits, its order, its types and widths, and the flat store's path with positions and
dropout."""
import math

import pytest
import torch

from nmtgminor_b200 import ops

DEV = "cuda"
HALF = {torch.bfloat16: 2 ** -8, torch.float16: 2 ** -11, torch.float32: 2 ** -24}


def test_on_the_cpu():
    g = torch.Generator().manual_seed(0)
    table = torch.randn(20, 6, generator=g, dtype=torch.float64).requires_grad_(True)
    pos = torch.randn(5, 6, generator=g, dtype=torch.float64).requires_grad_(True)
    tokens, at = torch.randint(0, 20, (40,), generator=g), torch.arange(40) % 9
    out = ops.embedding(tokens, table, at, pos, scale=2.0, pad_idx=3, sorted_grad=True)
    assert torch.allclose(out, 2.0 * table[tokens] + pos[at.clamp(max=4)])
    dy = torch.randn(40, 6, generator=g, dtype=torch.float64)
    gt, gp = torch.autograd.grad(out, (table, pos), dy)
    want = torch.zeros(20, 6, dtype=torch.float64).index_add_(0, tokens, 2.0 * dy * (tokens != 3)[:, None])
    assert torch.allclose(gt, want) and torch.allclose(gp, torch.zeros(5, 6, dtype=torch.float64).index_add_(0, at.clamp(max=4), dy))


def _refusals(device):
    t, tok = torch.zeros(5, 4, device=device), torch.zeros(3, dtype=torch.int64, device=device)
    for f in (lambda: ops.embedding(tok.int(), t, sorted_grad=True), lambda: ops.embedding(tok[None], t, sorted_grad=True),
              lambda: ops.embedding(tok, t[0], sorted_grad=True), lambda: ops.embedding(tok, t[:0], sorted_grad=True)):
        with pytest.raises(ValueError):
            f()


def test_refusals_on_the_cpu():
    _refusals("cpu")


# rows: one tile up to 2048, merged tiles up to 16384 (keys of up to 18 bits), radix passes beyond; vocabularies of 1 to 3 digits.  Where exactly the
# kernels change: test_embedding_sorted_edges.py
CASES = [(1, 1, 8), (7, 5, 1), (64, 3, 40), (65, 1000, 256), (1000, 7, 200), (4095, 32000, 64), (8192, 700, 16), (8193, 700, 16), (9000, 32000, 136),
         (20000, 250054, 24), (40000, 2, 8), (5000, 600000, 8), (12345, 1100000, 4)]


def _tokens(rows, vocab, spread, seed=0):
    g = torch.Generator().manual_seed(seed + rows + vocab)
    if spread == "zipf":
        t = torch.exp(torch.rand(rows, generator=g, dtype=torch.float64) * math.log(vocab)).long().clamp(0, vocab - 1)
    elif spread == "one":
        t = torch.full((rows,), vocab - 1)
    else:
        t = torch.randint(-2, vocab + 3, (rows,), generator=g)            # some are no words
    return t.to(DEV)


def _close(got, want, size, count, dtype):
    """One rounding to the type, and a 32-bit addition a term: 2^-24 of what the terms add up to without their signs, each."""
    low = 2 ** -25 if dtype == torch.float16 else 0.0
    assert ((got.double() - want).abs() <= HALF[dtype] * want.abs() + 2 ** -24 * (count + 4)[:, None] * size + low).all()


def _sums(tokens, vocab, dy, pad):
    ok = (tokens >= 0) & (tokens < vocab) & (tokens != pad)
    idx = torch.where(ok, tokens, 0)
    d = dy.double() * ok[:, None]
    zero = torch.zeros(vocab, dy.shape[1], dtype=torch.float64, device=DEV)
    return (zero.index_add(0, idx, d), zero.index_add(0, idx, d.abs()),
            torch.zeros(vocab, dtype=torch.float64, device=DEV).index_add(0, idx, ok.double()))


@pytest.mark.gpu
@pytest.mark.parametrize("spread", ["zipf", "one", "uniform"])
@pytest.mark.parametrize("dtype", list(HALF))
def test_gradient_of_a_table(dtype, spread):
    for rows, vocab, width in CASES:
        g = torch.Generator().manual_seed(width)
        tokens = _tokens(rows, vocab, spread)
        table = torch.randn(vocab, width, generator=g).to(dtype).to(DEV).requires_grad_(True)
        dy = torch.randn(rows, width, generator=g).to(dtype).to(DEV)
        pad = 2 if spread != "one" else -1
        out = ops.embedding(tokens, table, scale=1.5, pad_idx=pad, sorted_grad=True)
        inside = torch.where((tokens >= 0) & (tokens < vocab), tokens, 0)
        assert torch.equal(out, (table.detach()[inside].float() * 1.5).to(dtype))
        grad = torch.autograd.grad(out, table, dy)[0]
        want, size, count = _sums(tokens, vocab, dy, pad)
        _close(grad, 1.5 * want, 1.5 * size, count, dtype)
        assert (grad[count == 0] == 0).all()
        again = torch.autograd.grad(ops.embedding(tokens, table, scale=1.5, pad_idx=pad, sorted_grad=True), table, dy)[0]
        assert torch.equal(grad, again)


@pytest.mark.gpu
def test_sums_are_taken_in_the_order_of_the_tokens():
    """Terms whose sum in 32 bits depends on the order: every chunk of 8 sorted rows is added up from the first to the last."""
    tokens = torch.tensor([3, 1] * 4 + [1, 1, 1, 1], device=DEV)
    v = torch.tensor([0, 2.0 ** 24, 0, 1.0, 0, 1.0, 0, 1.0, -2.0 ** 24, 1.0, 1.0, 0.0], device=DEV)
    table = torch.zeros(4, 4, device=DEV).requires_grad_(True)
    grad = torch.autograd.grad(ops.embedding(tokens, table, sorted_grad=True), table, v[:, None].expand(12, 4).contiguous())[0]
    acc = torch.zeros((), dtype=torch.float32)
    for x, t in zip(v.cpu(), tokens.cpu()):
        if t == 1:
            acc = acc + x
    assert (grad[1] == acc.item()).all() and (grad[3] == 0).all() and acc.item() != 5.0


class _Flat:
    def __init__(self, shape, seed):
        g = torch.Generator().manual_seed(seed)
        work = torch.randn(*shape, generator=g).bfloat16().to(DEV)
        self.p = torch.nn.Parameter(work.float())
        self.p.work, self.p.main_grad = work, torch.randn(*shape, generator=g).to(DEV)
        self.before = self.p.main_grad.clone()

    def added(self):
        return self.p.main_grad.double() - self.before.double()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab,width", [(5, 9, 16), (777, 1000, 256), (9001, 32000, 512)])
@pytest.mark.parametrize("p", [0.0, 0.25])
def test_flat_store_with_positions_and_dropout(rows, vocab, width, p):
    """The same forward pass, mask and gradients as the path with atomic additions, up to the rounding of 32-bit sums."""
    tokens = _tokens(rows, vocab, "zipf")
    tokens[0] = 0
    pos = torch.arange(rows, device=DEV) % 50                             # beyond the table of 40: its last row
    dy = torch.randn(rows, width, generator=torch.Generator().manual_seed(1)).bfloat16().to(DEV)
    outs = []
    for sort in (False, True, True):
        ops.manual_seed(11)
        table, ptab = _Flat((vocab, width), 1), _Flat((40, width), 2)
        out = ops.embedding(tokens, table.p, pos, ptab.p, 3.0, p, True, 0, pos_trainable=True, sorted_grad=sort)
        out.backward(dy)
        outs.append((out.detach(), table, ptab))
    assert torch.equal(outs[0][0], outs[1][0])
    for a, b in ((outs[1][1], outs[2][1]), (outs[1][2], outs[2][2])):
        assert torch.equal(a.p.main_grad, b.p.main_grad)
    mask = torch.ones_like(dy, dtype=torch.float64)
    if p > 0:
        ops.manual_seed(11)
        sid = 1
        mask = ops.ext().dropout_add(torch.ones_like(dy), None, p, ops._Rng.seed, sid).double()
        mask = (mask != 0) * (256.0 / (256 - int(256 * p + 0.5)))
    d = dy.double() * mask
    for store, idx, scale in ((outs[1][1], tokens, 3.0), (outs[1][2], pos.clamp(max=39), 1.0)):
        ok = (tokens != 0).double()[:, None]
        zero = torch.zeros_like(store.before, dtype=torch.float64)
        want, size = zero.index_add(0, idx, scale * d * ok), zero.index_add(0, idx, (scale * d * ok).abs())
        count = torch.zeros(zero.shape[0], dtype=torch.float64, device=DEV).index_add(0, idx, torch.ones(rows, dtype=torch.float64, device=DEV))
        assert ((store.added() - want).abs() <= 2 ** -24 * (count + 6)[:, None] * size + 2 ** -23 * (store.before.double().abs() + want.abs())).all()


@pytest.mark.gpu
def test_deterministic_algorithms_ask_for_it():
    tokens = _tokens(3000, 50, "zipf")
    dy = torch.randn(3000, 64, generator=torch.Generator().manual_seed(1)).bfloat16().to(DEV)
    grads = []
    before = torch.are_deterministic_algorithms_enabled()
    try:
        torch.use_deterministic_algorithms(True, warn_only=True)
        for _ in range(3):
            table = _Flat((50, 64), 1)
            ops.embedding(tokens, table.p).backward(dy)
            grads.append(table.p.main_grad)
    finally:
        torch.use_deterministic_algorithms(before)
    assert torch.equal(grads[0], grads[1]) and torch.equal(grads[0], grads[2])


@pytest.mark.gpu
def test_streams_graphs_and_no_rows():
    tables = [torch.randn(3000, 96, device=DEV).requires_grad_(True) for _ in range(2)]
    toks = [_tokens(n, 3000, "zipf", n) for n in (700, 10000)]
    dys = [torch.randn(n, 96, device=DEV) for n in (700, 10000)]
    step = lambda i: torch.autograd.grad(ops.embedding(toks[i], tables[i], sorted_grad=True), tables[i], dys[i])[0]
    want = [step(0), step(1)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(i))
        graphs.append(g)
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
    out = ops.embedding(toks[0][:0], tables[0], sorted_grad=True)
    assert out.shape == (0, 96) and (torch.autograd.grad(out, tables[0], dys[0][:0])[0] == 0).all()


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    _refusals(DEV)
    t, tok, dy = torch.zeros(5, 4, device=DEV), torch.zeros(3, dtype=torch.int64, device=DEV), torch.zeros(3, 4, device=DEV)
    with pytest.raises(ValueError):
        ops.embedding(tok.cpu(), t, sorted_grad=True)
    for f in (lambda: ops.ext().embed_grad(tok, None, dy[:2], None, 5, 5, 1.0, 0.0, 0, 0, 0), lambda: ops.ext().embed_grad(tok, None, dy, t[:4], 5, 5, 1.0, 0.0, 0, 0, 0),
              lambda: ops.ext().embed_grad(tok, tok[:1], dy, None, 5, 5, 1.0, 0.0, 0, 0, 0), lambda: ops.ext().embed_grad(tok, None, dy.double(), None, 5, 5, 1.0, 0.0, 0, 0, 0),
              lambda: ops.ext().embed_grad(tok, None, dy, None, 5, 5, 1.0, 1.0, 0, 0, 0)):
        with pytest.raises(RuntimeError):
            f()


@pytest.mark.gpu
def test_tables_of_more_than_2_31_elements():
    """Offsets beyond 32 bits in the table, its gradient and dy: the words at the end against their rows by themselves."""
    vocab, width, rows = 270000, 8192, 265000
    table = torch.nn.Parameter(torch.empty(vocab, width, dtype=torch.bfloat16, device="cuda").normal_(generator=torch.Generator(device="cuda").manual_seed(1)))
    tokens = torch.arange(rows, device="cuda") + (vocab - rows)
    tokens[-3:] = vocab - 1
    out = ops.embedding(tokens, table, scale=2.0, pad_idx=0, sorted_grad=True)
    assert torch.equal(out.detach()[-9:], table.detach()[tokens[-9:]] * 2)
    dy = torch.empty_like(out).normal_(generator=torch.Generator(device="cuda").manual_seed(2))
    grad = torch.autograd.grad(out, table, dy)[0]
    assert torch.equal(grad[-9:-3], dy[-9:-3] * 2) and (grad[:vocab - rows] == 0).all() and (grad[-3:-1] == 0).all()
    want = 2 * dy[-3:].double().sum(0)
    assert ((grad[-1].double() - want).abs() <= 2 ** -8 * want.abs() + 2 ** -22 * dy[-3:].double().abs().sum(0)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize("rows,vocab,width", [(300, 50, 12), (9000, 700, 300), (20000, 5000, 20), (40, 9, 2), (600, 30, 6)])
def test_widths_between_vectors(dtype, rows, vocab, width):
    g = torch.Generator().manual_seed(width)
    tokens = _tokens(rows, vocab, "zipf")
    table = torch.randn(vocab, width, generator=g).to(dtype).to(DEV).requires_grad_(True)
    dy = torch.randn(rows, width, generator=g).to(dtype).to(DEV)
    out = ops.embedding(tokens, table, scale=1.5, pad_idx=2, sorted_grad=True)
    exact = 1.5 * table.detach().double()[tokens]
    assert ((out.detach().double() - exact).abs() <= HALF[dtype] * exact.abs() + (2 ** -25 if dtype == torch.float16 else 0)).all()
    grad = torch.autograd.grad(out, table, dy)[0]
    held = dy.double() * (tokens != 2)[:, None]
    want, size = (torch.zeros(vocab, width, dtype=torch.float64, device=DEV).index_add_(0, tokens, t) for t in (held, held.abs()))
    _close(grad, 1.5 * want, 1.5 * size, torch.bincount(tokens, minlength=vocab), dtype)
    assert torch.equal(grad, torch.autograd.grad(ops.embedding(tokens, table, scale=1.5, pad_idx=2, sorted_grad=True), table, dy)[0])


def test_plain_tables_keep_their_own_gradient_unless_asked():
    """Deterministic algorithms change the flat store's gradients alone: an ordinary table's are PyTorch's, padding included, as ever."""
    table = torch.randn(6, 3, requires_grad=True)
    tokens = torch.tensor([[1, 0], [2, 1]], dtype=torch.int32)
    want = torch.autograd.grad(ops.embedding(tokens, table, pad_idx=0).sum(), table)[0]
    before = torch.are_deterministic_algorithms_enabled()
    try:
        torch.use_deterministic_algorithms(True)
        assert torch.equal(torch.autograd.grad(ops.embedding(tokens, table, pad_idx=0).sum(), table)[0], want)
    finally:
        torch.use_deterministic_algorithms(before)
    assert want[0].sum() != 0
