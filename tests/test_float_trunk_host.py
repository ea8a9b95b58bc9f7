"""What the small float trunk (uor_fbs.float_trunk) does by itself, on the CPU: stand-ins take the place of the operators, of
which a trunk without layers needs only the ends and a norm."""

from types import SimpleNamespace

import pytest
import torch
import torch.nn.functional as F

ft = pytest.importorskip("uor_fbs.float_trunk")
DTYPES = ft.trunk.DTYPES


def stand_ins(**other):
    """uor_fbs.trunk's functions that a trunk without layers calls: the norm leaves its rows as they are."""
    return SimpleNamespace(**{**dict(MAX_ROWS=100, MAX_VOCAB=100, DTYPES=DTYPES, embed=lambda tokens, table, dtype: table[tokens].to(dtype),
                                     norms=lambda rows, pre: (rows, rows),
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


def limited(rows=3, words=4):
    """Stand-ins whose lookup and its gradient take so much at most, of the trunk's types, and tokens outside their table."""
    def check(tokens, table):
        assert tokens.numel() <= rows and len(table) <= words and table.dtype in (torch.bfloat16, torch.float32)
        return (tokens >= 0) & (tokens < len(table))

    def embed(tokens, table, dtype):
        there = check(tokens, table)
        return (table[torch.where(there, tokens, 0)] * there[:, None]).to(dtype)

    def embed_backward(dy, tokens, table):
        there = check(tokens, table)
        return torch.zeros_like(table).index_add_(0, torch.where(there, tokens, 0), dy.float() * there[:, None])

    return stand_ins(embed=embed, embed_backward=embed_backward, MAX_ROWS=rows, MAX_VOCAB=words, DTYPES=DTYPES)


TOKENS = [[2], [3, 0, 8], [3, 0, 8, 1], [8, 8, 4, 3, 3, 8, 7, 0, 1, 2]]


@pytest.mark.parametrize("tokens", [[], *TOKENS], ids=len)
@pytest.mark.parametrize("places", [torch.int32, torch.int64], ids=str)
def test_more_rows_and_words_than_a_lookup_takes(tokens, places, monkeypatch):
    monkeypatch.setattr(ft, "trunk", limited())
    cfg = config(vocab=9)
    p = ft.make_params(cfg, 3, device="cpu")
    tokens = torch.tensor(tokens, dtype=places)
    assert torch.equal(ft.prompts(cfg, p, tokens, None), p["embed"][tokens] @ p["head"])
    assert torch.equal(ft.step(cfg, p, tokens, None, None), p["embed"][tokens] @ p["head"])


@pytest.mark.parametrize("tokens", TOKENS, ids=len)
@pytest.mark.parametrize("places", [torch.int32, torch.int64], ids=str)
def test_the_gradient_of_more_rows_and_words_than_a_call_takes(tokens, places, monkeypatch):
    cfg = config(vocab=9)
    p = ft.make_params(cfg, 3, device="cpu")
    tokens, targets = torch.tensor(tokens, dtype=places), torch.arange(len(tokens)) % 9
    monkeypatch.setattr(ft, "trunk", limited(100, 100))
    want = ft.gradients(cfg, p, tokens, targets, None)[1]["embed"]
    monkeypatch.setattr(ft, "trunk", limited())
    got = ft.gradients(cfg, p, tokens, targets, None)[1]["embed"]
    # The same sums of up to ten values of at most 1, in another order.
    assert torch.allclose(got, want, rtol=0, atol=10 * 2.0 ** -24 * 10)


@pytest.mark.parametrize("kind", [torch.float16, torch.float64], ids=str)
def test_tables_of_other_types(kind, monkeypatch):
    monkeypatch.setattr(ft, "trunk", limited(100, 100))
    cfg = config()
    p = ft.make_params(cfg, 3, device="cpu")
    p["embed"] = p["embed"].to(kind)
    tokens = torch.tensor([3, 0, 5])
    assert torch.equal(ft.prompts(cfg, p, tokens, None), p["embed"].float()[tokens] @ p["head"])
