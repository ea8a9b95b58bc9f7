"""GPU tests of the small float trunk (uor_fbs.float_trunk), which runs the operators together.

Tolerance of the f32 comparisons. A logit or a gradient goes through at most 2 layers x 8 sums each
way, of at most 128 terms; an f32 sum is off by 2^-24 a term of its terms' absolute sum, which is about
sqrt(128) of the sum itself where signs are random: 32 x 128 x 12 x 2^-24 = 3e-3 of the whole's norm.
"""

import pytest
import torch
import torch.nn.functional as F

import trunk_cases as oracle

pytestmark = pytest.mark.gpu
ft = pytest.importorskip("uor_fbs.float_trunk")

BOUND = 32 * 128 * 12 * 2.0 ** -24


def close(a, b, name=""):
    a, b = a.detach().cpu().double(), b.detach().cpu().double()
    assert a.shape == b.shape, name
    assert (a - b).norm() <= BOUND * b.norm() + 1e-12, (name, float((a - b).norm() / b.norm()))


def config(**other):
    return ft.Config(**{**dict(vocab=24, width=40, layers=2, heads=4, groups=2, dim=24, state=20, dtype=torch.float32), **other})


def ragged(lengths, vocab, seed=5):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(0, vocab, (sum(lengths),), generator=g).cuda(), oracle.offsets_of(lengths).cuda()


def plain(cfg, p, tokens, offsets):
    """The logits in 64 bits on the CPU, row after row."""
    def rms(v, w):
        return v / torch.sqrt((v * v).mean(-1, keepdim=True) + 1e-6) * w

    out = []
    for a, b in oracle.bounds(offsets.cpu(), tokens.numel()):
        residual = p["embed"][tokens[a:b].cpu()]
        n = rms(residual, p["first"])
        for i in range(cfg.layers):
            w = {k: p[f"{i}.{k}"] for k in ft.LAYER}
            rows = n @ w["w_in"]
            past = torch.cat([rows.new_zeros(cfg.taps - 1, cfg.channels), rows[:, :cfg.channels]])
            mixed = F.silu(sum(past[k:k + b - a] * w["conv"][:, k] for k in range(cfg.taps)) + w["conv_bias"])
            x, B, C = ft._parts(cfg, mixed)
            share = cfg.heads // cfg.groups
            B, C = B.repeat_interleave(share, 1), C.repeat_interleave(share, 1)
            dt = F.softplus(rows[:, cfg.channels:] + w["dt_bias"])
            h, ys = rows.new_zeros(cfg.heads, cfg.dim, cfg.state), []
            for t in range(b - a):
                h = h * torch.exp(-dt[t] * torch.exp(w["A_log"]))[:, None, None] + (dt[t][:, None] * x[t])[..., None] * B[t][:, None]
                ys.append((h * C[t][:, None]).sum(-1) + w["D"][:, None] * x[t])
            y = torch.stack(ys) if ys else x
            residual = residual + w["scale"] * rms(y.flatten(1) @ w["w_out"] * F.silu(n @ w["w_gate"]), w["post"])
            n = rms(residual, w["pre"])
        out.append(n @ p["head"])
    return torch.cat(out)


def test_gradients_against_64_bits():
    cfg = config()
    p = ft.make_params(cfg, 3)
    tokens, offsets = ragged([5, 0, 70, 1], cfg.vocab)
    targets = torch.randint(-1, cfg.vocab, (76,), generator=torch.Generator().manual_seed(1)).cuda()
    loss, grads = ft.gradients(cfg, p, tokens, targets, offsets)
    wide = {k: v.detach().cpu().double().requires_grad_() for k, v in p.items()}
    logits = plain(cfg, wide, tokens, offsets)
    want = F.cross_entropy(logits, targets.cpu(), ignore_index=-1)
    want.backward()
    close(ft.prompts(cfg, p, tokens, offsets), logits, "logits")
    close(loss.reshape(1), want.reshape(1), "loss")
    assert set(grads) == set(p)
    for k, v in wide.items():
        close(grads[k], v.grad, k)


@pytest.mark.parametrize("taps", [1, 4])
def test_sessions_go_on_where_their_prompts_end(taps):
    cfg = config(taps=taps)
    p = ft.make_params(cfg, 4)
    tokens, offsets = ragged([9, 30, 2], cfg.vocab)
    more, _ = ragged([5, 5, 5], cfg.vocab, 6)
    state, slots = ft.make_state(cfg, 7), torch.tensor([6, 0, 3], dtype=torch.int32).cuda()
    ft.prompts(cfg, p, tokens, offsets, state, slots.long())
    got = torch.stack([ft.step(cfg, p, more.view(3, 5)[:, t], state, slots) for t in range(5)], 1)
    for i, (a, b) in enumerate(oracle.bounds(offsets.cpu(), tokens.numel())):
        whole = torch.cat([tokens[a:b], more.view(3, 5)[i]])
        close(got[i], ft.prompts(cfg, p, whole, oracle.offsets_of([whole.numel()]).cuda())[-5:], f"session {i}")


def test_the_step_as_a_graph():
    cfg = config(dtype=torch.bfloat16, dim=32, state=32, width=64)
    p = ft.make_params(cfg, 4)
    slots = torch.tensor([2, 0], dtype=torch.int32).cuda()
    tokens = torch.tensor([3, 4]).cuda()
    state, other = ft.make_state(cfg, 3), ft.make_state(cfg, 3)
    ft.step(cfg, p, tokens, other, slots)  # libraries are loaded before the capture
    for t in (*other.conv, *other.scan):
        t.zero_()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ft.step(cfg, p, tokens, state, slots)
    for now in ([1, 2], [7, 9], [5, 5], [0, 11]):
        tokens.copy_(torch.tensor(now))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ft.step(cfg, p, tokens, other, slots))
        assert all(torch.equal(a, b) for a, b in zip((*state.conv, *state.scan), (*other.conv, *other.scan)))


def test_a_trunk_learns_to_repeat():
    cfg = ft.Config(vocab=16, width=64, layers=2)
    p = ft.make_params(cfg)
    losses = ft.train(cfg, p, 300, count=64, length=6)
    assert losses[0] > 2.0 and sum(losses[-10:]) / 10 < 0.5
