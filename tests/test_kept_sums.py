"""Weight gradients of layers that keep their input in 8 bits: long sums over rows, against the sums of the same bf16 and kept numbers in 64 bits."""
import pytest
import torch

from nmtgminor_b200 import ops
from nmtgminor_b200.ops import kept

DEV = "cuda"


def _flat(value):
    p = torch.nn.Parameter(value.to(DEV))
    p.work, p.main_grad = p.detach().bfloat16(), torch.zeros(value.shape, device=DEV)
    return p


def _close(got, want, rows):
    """The sum is cut into parts of about 2048 rows; in a part every 16 rows are one addition, off by at most 2^-23 of what is summed so far; the
    parts meet in 32 bits."""
    parts = round(rows / 2048)
    off = (rows / parts / 16) * 2 ** -23 + parts * 2 ** -24
    error = ((got.double() - want).norm() / want.norm()).item()
    assert error <= off, (error, off)


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["relu", "gelu", "silu"])
def test_long_sums_of_a_block(act):
    rows, width, inner = 24000, 1024, 4096
    g = torch.Generator().manual_seed(9)
    x = torch.randn(rows, width, generator=g).bfloat16().to(DEV).requires_grad_(True)
    w1, w2 = _flat(torch.randn(inner, width, generator=g) / width ** 0.5), _flat(torch.randn(width, inner, generator=g) / inner ** 0.5)
    b1, b2 = _flat(torch.zeros(inner)), _flat(torch.zeros(width))
    dy = torch.randn(rows, width, generator=g).bfloat16().to(DEV)
    ops.mlp(x, w1, b1, w2, b2, act, 0.0, 0.0, None, True, keep8=True).backward(dy)
    with torch.no_grad():
        act_id = ops.ACT_IDS[act]
        if act == "relu":
            h = kept.restore(kept.quantise(ops.linear(x, w1, b1, act)))
        else:
            z, h = kept.restore_activated(kept.quantise(ops.linear(x, w1, b1)), act_id, 0.0, 0, 0, True)
            dz = torch.empty_like(h)
            ops.gemm(dy, w2.work, dz, b_mn_major=True, aux=z, act=ops._ACT_BWD[act_id])
            _close(w1.main_grad, dz.double().t() @ kept.restore(kept.quantise(x.detach())).double(), rows)
        _close(w2.main_grad, dy.double().t() @ h.double(), rows)
    assert ops.check_status() == 0


@pytest.mark.gpu
def test_long_sums_of_a_layer():
    rows, width, out = 24000, 4096, 1024
    g = torch.Generator().manual_seed(10)
    x = torch.randn(rows, width, generator=g).bfloat16().to(DEV).requires_grad_(True)
    w = _flat(torch.randn(out, width, generator=g) / width ** 0.5)
    dy = torch.randn(rows, out, generator=g).bfloat16().to(DEV)
    ops.linear(x, w, keep8=True).backward(dy)
    _close(w.main_grad, dy.double().t() @ kept.restore(kept.quantise(x.detach())).double(), rows)
    assert ops.check_status() == 0
