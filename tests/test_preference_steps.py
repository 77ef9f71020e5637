"""Steps of preference tuning over rows that no sentence has."""
import torch

from nmtgminor_b200.train import finetune as FT


class _Model:
    pad_idx = 0


def test_advantages_of_sentences(monkeypatch):
    """Rows behind the last sentence, empty sentences, and no sentence at all, whose advantage would be looked up in front of an empty list."""
    x = torch.randn(9, 20, generator=torch.Generator().manual_seed(0))
    y = torch.arange(1, 10)
    old = torch.log_softmax(x, 1).gather(1, y[:, None]).squeeze(1)
    for cu, adv, want in (([0, 4, 4, 7], [2.0, 5.0, -1.0], [2.0] * 4 + [-1.0] * 3), ([0], [], [])):
        labels = y.clone()
        labels[len(want):] = 0                                  # padding
        monkeypatch.setattr(FT, "packed_logits", lambda model, batch: (x, labels, torch.tensor(cu)))
        loss, clipped, _, _ = FT.policy_step(_Model(), None, old, torch.tensor(adv))
        assert abs(loss.item() + sum(want)) <= 2 ** -18 * 9 and clipped.item() == 0
