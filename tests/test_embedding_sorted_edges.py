"""The sorted embedding gradient on both sides of every change of its kernels: rows of one tile, of merged tiles and of radix passes, chunks of 8 and 16,
keys that leave room for a row's number beside them and keys that do not, vectors and single columns."""
import pytest
import torch

from nmtgminor_b200 import ops

DEV = "cuda"
HALF = {torch.bfloat16: 2 ** -8, torch.float16: 2 ** -11, torch.float32: 2 ** -24}
ROWS = [31, 32, 33, 2047, 2048, 2049, 4095, 4096, 4097, 16383, 16384, 16385]


def _check(tokens, vocab, width, dtype, pad=0, seed=0):
    g = torch.Generator().manual_seed(seed + len(tokens) + width)
    table = torch.randn(vocab, width, generator=g).to(dtype).to(DEV).requires_grad_(True)
    dy = torch.randn(len(tokens), width, generator=g).to(dtype).to(DEV)
    runs = [torch.autograd.grad(ops.embedding(tokens, table, scale=1.5, pad_idx=pad, sorted_grad=True), table, dy)[0] for _ in range(2)]
    ok = (tokens >= 0) & (tokens < vocab) & (tokens != pad)
    at, d = torch.where(ok, tokens, 0), 1.5 * dy.double() * ok[:, None]
    zero = torch.zeros(vocab, width, dtype=torch.float64, device=DEV)
    want, size = zero.index_add(0, at, d), zero.index_add(0, at, d.abs())
    terms = torch.zeros(vocab, dtype=torch.float64, device=DEV).index_add(0, at, ok.double())
    # one rounding to the type, and one of 32 bits for every term, of what the terms add up to without their signs
    bound = HALF[dtype] * want.abs() + 2 ** -24 * (terms + 4)[:, None] * size + (2 ** -25 if dtype == torch.float16 else 0.0)
    assert ((runs[0].double() - want).abs() <= bound).all() and (runs[0][terms == 0] == 0).all()
    assert torch.equal(*runs)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("spread", ["even", "few", "one"])
def test_rows_where_the_kernels_change(rows, spread):
    g = torch.Generator().manual_seed(rows)
    vocab = {"even": 5000, "few": 3, "one": 9}[spread]
    tokens = torch.randint(-1, vocab + 1, (rows,), generator=g).to(DEV) if spread != "one" else torch.full((rows,), 7, device=DEV)
    for dtype, width in ((torch.bfloat16, 16), (torch.float32, 9), (torch.float16, 12)):
        _check(tokens, vocab, width, dtype)
    assert ops.check_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [1023, 1024, 131071, 131072, 262142, 262143, 262144, 262145])
@pytest.mark.parametrize("rows", [2048, 2049, 16384, 16385])
def test_keys_where_the_kernels_change(rows, vocab):
    """Rows without a key among those of the last words, the last row among them: its key and number together are the number that fills a tile up."""
    g = torch.Generator().manual_seed(vocab)
    tokens = (vocab - 1 - torch.randint(0, 40, (rows,), generator=g)).to(DEV)
    tokens[-1], tokens[::5], tokens[3] = vocab, vocab + 5, 0
    _check(tokens, vocab, 8, torch.bfloat16, pad=0)
    _check(tokens.flip(0), vocab, 4, torch.float32, pad=vocab - 1)
    assert ops.check_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [2048, 2049, 16384, 16385])
def test_positions_where_the_kernels_change(rows):
    """Keys that are positions, brought into a table shorter than they are."""
    g = torch.Generator().manual_seed(rows)
    flat = []
    for n, seed in ((700, 1), (50, 2)):
        p = torch.nn.Parameter(torch.randn(n, 32, generator=g).to(DEV))
        p.work, p.main_grad = p.detach().bfloat16(), torch.zeros(n, 32, device=DEV)
        flat.append(p)
    tokens, pos = torch.randint(0, 700, (rows,), generator=g).to(DEV), torch.randint(-3, 60, (rows,), generator=g).to(DEV)
    dy = torch.randn(rows, 32, generator=g).bfloat16().to(DEV)
    ops.embedding(tokens, flat[0], pos, flat[1], 1.0, 0.0, True, 0, pos_trainable=True, sorted_grad=True).backward(dy)
    d = dy.double() * (tokens != 0)[:, None]
    for p, at in ((flat[0], tokens), (flat[1], pos.clamp(0, 49))):
        zero = torch.zeros(p.shape, dtype=torch.float64, device=DEV)
        count = torch.bincount(at, minlength=p.shape[0])[:, None] + 4
        assert ((p.main_grad.double() - zero.index_add(0, at, d)).abs() <= 2 ** -24 * count * zero.index_add(0, at, d.abs())).all()
    assert ops.check_status() == 0
