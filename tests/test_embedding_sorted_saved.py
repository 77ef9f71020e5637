"""What the sorted embedding gradient of the flat store keeps for the backward pass: tokens and positions as saved tensors."""
import pytest
import torch

from nmtgminor_b200 import ops

DEV = "cuda"


def _flat(rows, width, seed):
    p = torch.nn.Parameter(torch.randn(rows, width, generator=torch.Generator().manual_seed(seed)).to(DEV))
    p.work, p.main_grad = p.detach().bfloat16(), torch.zeros(rows, width, device=DEV)
    return p


@pytest.mark.gpu
@pytest.mark.parametrize("positions", [False, True])
def test_tokens_and_positions_are_saved_tensors(positions):
    """Overwritten between the passes they are refused, as are second passes through a freed graph; hooks see them; a kept graph adds again."""
    table, ptab = _flat(60, 32, 1), _flat(20, 32, 2)
    tokens, pos = torch.arange(1, 13, device=DEV), torch.arange(12, device=DEV) if positions else None

    def forward():
        return ops.embedding(tokens, table, pos, ptab if positions else None, 2.0, 0.0, True, 0, pos_trainable=positions, sorted_grad=True)

    for changed in (tokens, pos):
        if changed is None:
            continue
        out = forward()
        changed += 1
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            out.sum().backward()
        assert (table.main_grad == 0).all() and (ptab.main_grad == 0).all()
        changed -= 1
    out = forward()
    out.sum().backward(retain_graph=True)
    once = table.main_grad.clone()
    assert (once[1:13] == 2.0).all() and once.sum() == 2.0 * 12 * 32
    out.sum().backward()
    assert torch.equal(table.main_grad, 2 * once) and (not positions or (ptab.main_grad[:12] == 2.0).all())
    with pytest.raises(RuntimeError, match="second time"):
        out.sum().backward()
    assert torch.equal(table.main_grad, 2 * once)
    seen = []

    def pack(t):
        seen.append(t)
        return t.cpu()

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t.to(DEV)):
        out = forward()
    assert [t.data_ptr() for t in seen] == [t.data_ptr() for t in (tokens, pos) if t is not None]
    table.main_grad.zero_()
    out.sum().backward()
    assert torch.equal(table.main_grad, once) and ops.check_status() == 0
