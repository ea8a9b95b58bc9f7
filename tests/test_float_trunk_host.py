"""What the small float trunk (uor_fbs.float_trunk) does by itself, on the CPU: stand-ins take the place of the operators, of
which a trunk without layers needs only the ends and a norm."""

from types import SimpleNamespace

import pytest
import torch
import torch.nn.functional as F

ft = pytest.importorskip("uor_fbs.float_trunk")


def stand_ins(**other):
    """uor_fbs.trunk's functions that a trunk without layers calls: the norm leaves its rows as they are."""
    return SimpleNamespace(**{**dict(embed=lambda tokens, table, dtype: table[tokens].to(dtype), norms=lambda rows, pre: (rows, rows),
                                     norms_backward=lambda d_rows, d_n, rows, pre: SimpleNamespace(dpre=None, dresidual=d_n),
                                     embed_backward=lambda dy, tokens, table: torch.zeros_like(table).index_add_(0, tokens, dy.float())), **other})


def config(**other):
    return ft.Config(**{**dict(vocab=6, width=5, layers=0, dtype=torch.float32), **other})


@pytest.mark.parametrize("none", [-1, -7, 6, 7, 1 << 40], ids=str)
def test_a_target_outside_the_vocabulary_is_none(none, monkeypatch):
    """With whole logits: what F.cross_entropy gives that leaves the row out."""
    monkeypatch.setattr(ft, "trunk", stand_ins())
    cfg = config()
    p = ft.make_params(cfg, 3, device="cpu")
    tokens, targets = torch.tensor([3, 0, 5, 1]), torch.tensor([2, none, 5, none])
    loss, grads = ft.gradients(cfg, p, tokens, targets, None)
    wide = {k: v.double().requires_grad_() for k, v in p.items()}
    want = F.cross_entropy(wide["embed"][tokens] @ wide["head"], torch.tensor([2, -1, 5, -1]), ignore_index=-1)
    want.backward()
    # Sums of 6 terms, each of them some 8 roundings of 2^-24 off.
    assert abs(loss - want) <= 50 * 2.0 ** -24 * (1 + abs(want))
    for k in ("head", "embed"):
        assert torch.allclose(grads[k].double(), wide[k].grad, rtol=0, atol=50 * 2.0 ** -24 * (1 + float(wide[k].grad.abs().max()))), k
