"""GPU tests of a trunk's ends over its vocabulary (uor_fbs.trunk: embed, loss, choose) against their
definitions in 64 bits.

Tolerances. An output's own rounding is half a step of its type, `eps / 2` of its value (2^-8 for bf16). Before it
stand sums in 32 bits, each off by 2^-24 of the sum of absolute terms, once a term.

A logit z is a sum of `width` products: off by width 2^-24 |x| . |W|, call it dz. A row's sum of exponentials
is taken in chains of 16 values a tile, some 40 and one for each 256 words long, of exponentials good to 2^-22 of
themselves whose exponents (z - most) log2 e are rounded to 2^-24 of up to |z| + |most|. So lse is off by
dlse = max dz + 2^-22 + (40 + vocab / 256 + 4 max |z|) 2^-24 + 2^-23 |lse|, and the loss by dlse + dz + 2^-23 |loss|.

A gradient's G is its softmax times its weight: off by dG = (dz + dlse + 2^-22 + 4 max |z| 2^-24) |weight p|, and in
bf16, but for the target's, by its rounding 2^-8 |G|. dx is off by dG . |W| and (vocab + 8) 2^-24 |G| . |W|, dW the same
over rows.
"""

import pytest
import torch

import ends_cases as oracle

pytestmark = pytest.mark.gpu
trunk = pytest.importorskip("uor_fbs.trunk")

TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
STEP = 2.0 ** -24


@pytest.fixture(params=list(TYPES))
def dtype(request):
    return TYPES[request.param]


class Make:
    def __init__(self, dtype, seed):
        self.dtype, self.gen = dtype, torch.Generator().manual_seed(seed)

    def __call__(self, *shape, scale=1.0, dtype=None):
        return (torch.randn(shape, generator=self.gen) * scale).to(dtype or self.dtype).cuda()

    def ints(self, lo, hi, n, dtype=torch.int64):
        return torch.randint(lo, hi, (n,), generator=self.gen).to(dtype).cuda()


def within(name, got, want, allowed):
    got = got.detach().double()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    off = (got - want).abs()
    bad = ~(off <= allowed + 1e-30)
    assert not bad.any(), (name, int(bad.sum()), float(off[bad].max()), float((off / (allowed + 1e-30))[bad].max()))


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


# ---------------------------------------------------------------------------------------------
# The embedding.

EMBEDS = [(1, 1, 1), (5, 7, 3), (1, 300, 8), (300, 40, 64), (257, 1000, 100), (33, 50, 513), (1500, 20, 7), (70, 9, 1030), (4097, 130, 40),
          (9, 17, 8192)]


@pytest.mark.parametrize("rows,vocab,width", EMBEDS)
@pytest.mark.parametrize("out", list(TYPES))
def test_embed(dtype, out, rows, vocab, width):
    m = Make(dtype, rows + vocab)
    table, tokens = m(vocab, width), m.ints(-1, vocab + 1, rows, torch.int32 if rows % 2 else torch.int64)
    for scale in (1.0, 11.3125):  # a number of 32 bits
        y = trunk.embed(tokens, table, scale=scale, dtype=TYPES[out])
        want = oracle.embed(tokens, table, scale)
        assert y.dtype == TYPES[out]
        within("y", y, want, (half_step(TYPES[out]) + STEP) * want.abs())


def counted(name, got, want, size, count, dtype):
    assert got.dtype == dtype, name
    within(name, got, want, half_step(dtype) * (want.abs() + (count + 2) * STEP * size) + (count + 2) * STEP * size)


@pytest.mark.parametrize("rows,vocab,width", EMBEDS + [(4096, 5, 24), (20000, 1 << 20, 16), (70000, 3000, 12)])
@pytest.mark.parametrize("table", list(TYPES))
def test_embed_backward(dtype, table, rows, vocab, width):
    m = Make(dtype, rows + vocab)
    tokens, dy = m.ints(-1, vocab + 1, rows, torch.int32 if rows % 2 else torch.int64), m(rows, width)
    got = trunk.embed_backward(dy, tokens, torch.empty(vocab, width, dtype=TYPES[table], device="cuda"), scale=3.25)
    counted("dE", got, *oracle.embed_backward(dy, tokens, vocab, 3.25), TYPES[table])


@pytest.mark.parametrize("rows", [1, 16, 17, 128, 1000, 4096, 5000, 40000])
@pytest.mark.parametrize("kind", ["one word", "two words", "padding", "ascending", "descending", "the last word", "far outside"])
def test_embed_backward_of_words_that_many_rows_have(rows, kind):
    m = Make(torch.bfloat16, rows)
    vocab, width = 700, 72
    i = torch.arange(rows)
    tokens = {"one word": torch.full((rows,), 3), "two words": 3 + 400 * (i % 7 == 0).long(), "padding": torch.full((rows,), -1),
              "ascending": i * vocab // rows, "descending": vocab - 1 - i * vocab // rows, "the last word": torch.full((rows,), vocab - 1),
              "far outside": torch.where(i % 2 == 0, (1 << 32) + 3, -(1 << 40) + i)}[kind].cuda()
    dy = m(rows, width)
    got = trunk.embed_backward(dy, tokens, torch.empty(vocab, width, device="cuda"))
    counted("dE", got, *oracle.embed_backward(dy, tokens, vocab, 1.0), torch.float32)
    assert torch.equal(got, trunk.embed_backward(dy, tokens, torch.empty(vocab, width, device="cuda")))


def test_embed_of_strided_and_unaligned_rows():
    m = Make(torch.bfloat16, 3)
    wide, dys = m(60, 101), m(90, 101)
    tokens = m.ints(0, 60, 180)[::2]
    for cut in (slice(0, 96), slice(1, 98), slice(3, 100)):
        table, dy = wide[:, cut], dys[:, cut]
        within("y", trunk.embed(tokens, table), oracle.embed(tokens, table, 1.0), 0.0)
        counted("dE", trunk.embed_backward(dy, tokens, table), *oracle.embed_backward(dy, tokens, 60, 1.0), torch.bfloat16)
    row = m(1, 64).expand(90, 64)
    counted("dE", trunk.embed_backward(row, tokens, wide[:, :64]), *oracle.embed_backward(row, tokens, 60, 1.0), torch.bfloat16)


def test_what_is_not_finite_stays_with_its_word():
    m = Make(torch.float32, 5)
    table, tokens, dy = m(9, 20), torch.tensor([1, 4, -1, 4, 8, 9]).cuda(), m(6, 20)
    table[2], table[4, 7] = float("nan"), float("inf")
    y = trunk.embed(tokens, table)
    assert torch.equal(torch.isfinite(y), torch.isfinite(oracle.embed(tokens, table, 1.0)))
    dy[2], dy[5], dy[3, 2] = float("nan"), float("inf"), float("nan")
    got = trunk.embed_backward(dy, tokens, table)
    want = torch.ones(9, 20, dtype=torch.bool).cuda()
    want[4, 2] = False
    assert torch.equal(torch.isfinite(got), want)


def test_embed_of_no_rows():
    table = Make(torch.float32, 5)(9, 20)
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    assert trunk.embed(none, table).shape == (0, 20)
    assert torch.equal(trunk.embed_backward(torch.empty(0, 20, device="cuda"), none, table), torch.zeros_like(table))


def test_embed_in_autograd():
    m = Make(torch.float32, 8)
    table, tokens = m(50, 24).requires_grad_(), m.ints(-1, 50, 200)
    y = trunk.embed(tokens, table, scale=2.0, dtype=torch.bfloat16)
    y.sum().backward()  # a broadcast gradient
    counted("dE", table.grad, *oracle.embed_backward(torch.ones(200, 24).cuda(), tokens, 50, 2.0), torch.float32)


# ---------------------------------------------------------------------------------------------
# The loss.


def loss_case(dtype, rows, vocab, width, seed=1, masked=0.2, places=torch.int64):
    m = Make(dtype, seed + rows + vocab)
    weight, targets = m(vocab, width, scale=width ** -0.5), m.ints(0, vocab, rows, places)
    x = (m(rows, width, dtype=torch.float32) + m(rows, 1, dtype=torch.float32).abs() * 4 * weight[targets.long()].float()).to(dtype)
    off = torch.rand(rows, generator=m.gen) < masked
    targets[off.cuda()] = m.ints(-3, 0, 1, places)[0]
    return x, weight, targets, m


class Bounds:
    """How far a call's results may be off, from its operands."""

    def __init__(self, x, weight, targets):
        width, vocab = x.shape[1], weight.shape[0]
        self.there = (targets >= 0) & (targets < vocab)
        self.z = oracle.logits(x, weight)
        self.dz = (width + 1) * STEP * (x.double().abs() @ weight.double().abs().t())
        most = self.z.abs().amax(1)
        self.exp = 2.0 ** -22 + 4 * most * STEP
        lse = torch.logsumexp(self.z, 1)
        self.lse = self.dz.amax(1) + self.exp + (40 + vocab / 256) * STEP + 2.0 ** -23 * lse.abs()
        at = targets.long().clamp(0, vocab - 1)[:, None]
        self.loss = self.lse + self.dz.gather(1, at)[:, 0] + 2.0 ** -23 * (lse.abs() + self.z.gather(1, at)[:, 0].abs())

    def gradient(self, x, weight, targets, dlosses, dlse):
        """Of dx and dweight, without their own rounding."""
        g, others = oracle.logit_gradient(x, weight, targets, dlosses, dlse)
        a = torch.zeros(len(x), dtype=torch.float64, device=x.device) if dlosses is None else dlosses.double()
        b = torch.zeros_like(a) if dlse is None else dlse.double()
        p = torch.softmax(self.z, 1) * ((a.abs() + b.abs()) * self.there)[:, None]
        dg = (self.dz + self.lse[:, None] + self.exp[:, None] + 4 * STEP) * p
        if x.dtype == torch.bfloat16:
            dg = dg + half_step(x.dtype) * (others.abs() + dg)
        w, rows = weight.double().abs(), x.double().abs() * self.there[:, None]
        return ((dg + (len(weight) + 8) * STEP * (g.abs() + dg)) @ w, (dg + (len(x) + 8) * STEP * (g.abs() + dg)).t() @ rows)


LOSSES = [(1, 1, 1), (1, 2, 8), (5, 7, 3), (64, 256, 32), (129, 257, 33), (128, 512, 64), (300, 1000, 65), (7, 5003, 100), (200, 130, 520),
          (4500, 300, 16), (2, 40000, 24), (33, 700, 1030), (30, 500, 700), (64, 300, 448), (65, 300, 448), (16, 20000, 72), (257, 3000, 200)]


def check_loss(x, weight, targets):
    losses, lse = trunk.loss(x, weight, targets)
    want, want_lse = oracle.loss(x, weight, targets)
    b = Bounds(x, weight, targets)
    within("lse", lse, want_lse, b.lse * b.there)
    within("losses", losses, want, b.loss * b.there)
    again = trunk.loss(x, weight, targets)
    assert torch.equal(losses, again[0]) and torch.equal(lse, again[1])
    return lse


def check_gradients(x, weight, targets, lse, da, db, out=None):
    dx, dw = trunk.loss_backward(da, x, weight, targets, lse, dlse=db, dtype=out)
    want_x, want_w = oracle.loss_backward(da, x, weight, targets, db)
    off_x, off_w = Bounds(x, weight, targets).gradient(x, weight, targets, da, db)
    assert dx.dtype == x.dtype and dw.dtype == (out or weight.dtype)
    within("dx", dx, want_x, half_step(dx.dtype) * (want_x.abs() + off_x) + off_x)
    within("dweight", dw, want_w, half_step(dw.dtype) * (want_w.abs() + off_w) + off_w)
    again = trunk.loss_backward(da, x, weight, targets, lse, dlse=db, dtype=out)
    assert torch.equal(dx, again.dx) and torch.equal(dw, again.dweight)


@pytest.mark.parametrize("rows,vocab,width", LOSSES)
def test_loss_and_gradients(dtype, rows, vocab, width):
    x, weight, targets, m = loss_case(dtype, rows, vocab, width, places=torch.int32 if rows % 2 else torch.int64)
    lse = check_loss(x, weight, targets)
    da, db = m(rows, dtype=torch.float32), m(rows, dtype=torch.float32)
    check_gradients(x, weight, targets, lse, da, db)


@pytest.mark.parametrize("which", ["losses", "lse"])
def test_gradients_of_one_output(dtype, which):
    x, weight, targets, m = loss_case(dtype, 150, 600, 48)
    d = m(150, dtype=torch.float32)
    lse = trunk.loss(x, weight, targets)[1]
    check_gradients(x, weight, targets, lse, d if which == "losses" else None, d if which == "lse" else None, out=torch.float32)


@pytest.mark.parametrize("out", list(TYPES))
@pytest.mark.parametrize("rows,vocab,width", [(40, 300, 33), (300, 2000, 64), (5000, 70000, 8)])
def test_gradients_of_one_input_and_of_another_type(dtype, out, rows, vocab, width):
    x, weight, targets, m = loss_case(dtype, rows, vocab, width)
    da, lse = m(rows, dtype=torch.float32), trunk.loss(x, weight, targets)[1]
    check_gradients(x, weight, targets, lse, da, None, out=TYPES[out])
    both = trunk.loss_backward(da, x, weight, targets, lse, dtype=TYPES[out])
    dx, none = trunk.loss_backward(da, x, weight, targets, lse, dweight=False)
    assert none is None and torch.equal(dx, both.dx)
    none, dw = trunk.loss_backward(da, x, weight, targets, lse, dx=False, dtype=TYPES[out])
    assert none is None and torch.equal(dw, both.dweight)


@pytest.mark.parametrize("masked", [0.0, 0.5, 0.99, 1.0])
@pytest.mark.parametrize("rows", [20, 130, 4500])
def test_rows_without_a_target_take_no_part(dtype, rows, masked):
    x, weight, targets, m = loss_case(dtype, rows, 300, 40, masked=masked)
    da = m(rows, dtype=torch.float32)
    lse = check_loss(x, weight, targets)
    check_gradients(x, weight, targets, lse, da, None)
    # Whatever they hold.
    none = targets < 0
    worse, wrong = x.clone(), da.clone()
    worse[none], wrong[none] = float("nan"), float("inf")
    got, other = trunk.loss(worse, weight, targets), trunk.loss(x, weight, targets)
    assert torch.equal(got[0], other[0]) and torch.equal(got[1], other[1])
    got, other = trunk.loss_backward(wrong, worse, weight, targets, lse), trunk.loss_backward(da, x, weight, targets, lse)
    assert torch.equal(got.dx, other.dx) and torch.equal(got.dweight, other.dweight)
    assert not got.dx[none].any()


@pytest.mark.parametrize("rows,vocab", [(24000, 24000), (600, 1000000), (200000, 3000), (40000, 14500), (14500, 40000)])
def test_gradients_in_several_pieces(dtype, rows, vocab):
    """More logits than a piece holds, along both axes and along one."""
    x, weight, targets, m = loss_case(dtype, rows, vocab, 24)
    da = m(rows, dtype=torch.float32)
    lse = trunk.loss(x, weight, targets)[1]
    check_gradients(x, weight, targets, lse, da, None)


def test_a_word_that_most_rows_have(dtype):
    x, weight, targets, m = loss_case(dtype, 5000, 400, 40)
    targets[: 4000] = 7
    lse = check_loss(x, weight, targets)
    check_gradients(x, weight, targets, lse, m(5000, dtype=torch.float32), None)


def test_large_logits_and_a_sure_target(dtype):
    m = Make(dtype, 4)
    weight = m(300, 32)
    targets = torch.arange(100).cuda() % 300
    x = (weight[targets].float() * torch.linspace(-30, 30, 100).cuda()[:, None]).to(dtype)  # logits up to some 1,000
    lse = check_loss(x, weight, targets)
    check_gradients(x, weight, targets, lse, m(100, dtype=torch.float32), None)


def test_matrices_as_they_lie(dtype):
    """Strided rows, unaligned ones, a transposed matrix, a broadcast row and weight."""
    m = Make(dtype, 9)
    xs, ws, targets = m(90, 101), m(210, 101, scale=0.1), m.ints(0, 210, 180)[::2]
    for cut in (slice(0, 96), slice(1, 97), slice(5, 100)):
        x, weight = xs[:, cut], ws[:, cut]
        lse = check_loss(x, weight, targets)
        check_gradients(x, weight, targets, lse, torch.ones(1).cuda().expand(90), None)
    check_loss(xs[:, :64], m(64, 210, scale=0.1).t(), targets)
    check_loss(m(1, 64).expand(90, 64), ws[:, :64], targets)
    tokens, _ = trunk.choose(xs[:, 1:97], ws[:, 1:97])
    assert torch.equal(tokens, oracle.logits(xs[:, 1:97], ws[:, 1:97]).argmax(1))


def test_what_is_not_finite_stays_with_its_row(dtype):
    x, weight, targets, m = loss_case(dtype, 200, 300, 40, masked=0.0)
    x[5, 3], x[70, 0] = float("nan"), float("inf")
    losses, lse = trunk.loss(x, weight, targets)
    want = torch.ones(200, dtype=torch.bool).cuda()
    want[[5, 70]] = False
    assert torch.equal(torch.isfinite(losses), want) and torch.equal(torch.isfinite(lse), want)
    dx, dw = trunk.loss_backward(m(200, dtype=torch.float32), x, weight, targets, lse)
    assert torch.equal(torch.isfinite(dx).all(1), want) and not torch.isfinite(dw).any()


def test_loss_of_no_rows():
    x, weight, targets, _ = loss_case(torch.bfloat16, 3, 20, 16)
    losses, lse = trunk.loss(x[:0], weight, targets[:0])
    assert losses.shape == lse.shape == (0,)
    dx, dw = trunk.loss_backward(losses, x[:0], weight, targets[:0], lse)
    assert dx.shape == (0, 16) and torch.equal(dw, torch.zeros_like(weight))
    assert trunk.choose(x[:0], weight)[0].shape == (0,)


def test_loss_in_autograd(dtype):
    x, weight, targets, _ = loss_case(dtype, 200, 300, 40)
    x.requires_grad_(), weight.requires_grad_()
    losses, lse = trunk.loss(x, weight, targets)
    losses.retain_grad(), lse.retain_grad()  # as autograd forms them: the order of their products is its own
    count = (targets >= 0).sum()
    (losses.sum() / count + 1e-2 * (lse * lse).sum() / count).backward()
    got = trunk.loss_backward(losses.grad, x, weight, targets, lse.detach(), dlse=lse.grad)
    assert torch.equal(x.grad, got.dx) and torch.equal(weight.grad, got.dweight)
    weight.grad = None
    trunk.loss(x.detach(), weight, targets)[0].sum().backward()  # of one input alone
    assert torch.equal(weight.grad, trunk.loss_backward(torch.ones(200).cuda(), x, weight, targets, lse.detach()).dweight)


# ---------------------------------------------------------------------------------------------
# The choice.


@pytest.mark.parametrize("rows,vocab,width", LOSSES + [(1, 131072, 64), (16, 3000, 256), (17, 3000, 256), (1024, 1000, 96)])
def test_choose(dtype, rows, vocab, width):
    x, weight, _, _ = loss_case(dtype, rows, vocab, width, masked=0.0)
    tokens, logprobs = trunk.choose(x, weight)
    b = Bounds(x, weight, torch.zeros(rows, dtype=torch.int64).cuda())
    assert tokens.dtype == torch.int64 and logprobs.dtype == torch.float32
    chosen = b.z.gather(1, tokens[:, None])[:, 0]
    assert (chosen >= b.z.amax(1) - 2 * b.dz.amax(1)).all()  # the largest, as far as sums in 32 bits tell
    clear = b.z.topk(min(2, vocab), 1).values
    sure = clear[:, 0] - clear[:, -1] > 2 * b.dz.amax(1) if vocab > 1 else torch.ones(rows, dtype=torch.bool).cuda()
    assert torch.equal(tokens[sure], b.z.argmax(1)[sure])
    lse = torch.logsumexp(b.z, 1)
    within("logprobs", logprobs, chosen - lse, b.lse + b.dz.amax(1) + 2.0 ** -23 * (lse.abs() + chosen.abs()))


@pytest.mark.parametrize("rows", [1, 16, 40, 130])
def test_the_lowest_of_equals(dtype, rows):
    """The same words at several places, with sums of whole numbers, which are exact."""
    m = Make(dtype, 2)
    weight = m.ints(-3, 4, 2000 * 32).view(2000, 32).to(dtype)
    x = m.ints(-3, 4, rows * 32).view(rows, 32).to(dtype)
    weight[1000:] = weight[:1000]
    z = oracle.logits(x, weight)
    tokens, _ = trunk.choose(x, weight)
    assert torch.equal(tokens, torch.where(z == z.amax(1, keepdim=True), torch.arange(2000).cuda(), 2000).amin(1))
    assert torch.equal(trunk.choose(torch.zeros_like(x), weight)[0], torch.zeros(rows, dtype=torch.int64).cuda())


@pytest.mark.parametrize("rows", [3, 140])
def test_logits_that_are_no_numbers_are_not_chosen(rows):
    m = Make(torch.float32, 2)
    weight, x = m(500, 16), m(rows, 16)
    weight[17] = float("nan")
    x[1] = float("nan")
    x[2] = 0.0
    tokens, logprobs = trunk.choose(x, weight)
    z = oracle.logits(x, weight)
    want = torch.where(torch.isnan(z), -float("inf"), z).argmax(1)
    want[1] = 0
    assert torch.equal(tokens, want) and not torch.isfinite(logprobs).any()
    weight[17] = -float("inf")
    x = x.abs() + 0.1
    tokens, logprobs = trunk.choose(x, weight)
    assert torch.equal(tokens, oracle.logits(x, weight).argmax(1))
    assert torch.equal(torch.isfinite(logprobs), torch.arange(rows).cuda() != 1)  # that row's are still no numbers


# ---------------------------------------------------------------------------------------------
# Streams, graphs and the trunk.


def step_of(tokens, table, weight, targets):
    """A training step of a trunk without layers."""
    x = trunk.embed(tokens, table, dtype=weight.dtype)
    losses, lse = trunk.loss(x, weight, targets)
    g = trunk.loss_backward(torch.full_like(losses, 0.25), x, weight, targets, lse)
    return losses, g.dweight, trunk.embed_backward(g.dx, tokens, table), *trunk.choose(x, weight)


@pytest.mark.parametrize("rows", [100, 5000])
def test_on_another_stream_and_as_a_graph(dtype, rows):
    m = Make(dtype, 6)
    table, weight = m(400, 40, dtype=torch.float32), m(400, 40, scale=0.2)
    tokens, targets = m.ints(-1, 400, rows), m.ints(-1, 400, rows)
    want = step_of(tokens, table, weight, targets)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step_of(tokens, table, weight, targets)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step_of(tokens, table, weight, targets)
    for _ in range(4):
        tokens.copy_(m.ints(-1, 400, rows)), targets.copy_(m.ints(-1, 400, rows))
        weight.copy_(m(400, 40, scale=0.2))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step_of(tokens, table, weight, targets)))


def test_two_graphs_side_by_side():
    m = Make(torch.bfloat16, 6)
    table, weight = m(400, 40, dtype=torch.float32), m(400, 40, scale=0.2)
    inputs = [(m.ints(-1, 400, 300), m.ints(-1, 400, 300)) for _ in range(2)]
    want = [step_of(a, table, weight, b) for a, b in inputs]
    torch.cuda.synchronize()
    graphs, outs = [torch.cuda.CUDAGraph() for _ in inputs], []
    for graph, (a, b) in zip(graphs, inputs):
        with torch.cuda.graph(graph):
            outs.append(step_of(a, table, weight, b))
    sides = [torch.cuda.Stream() for _ in graphs]
    for _ in range(5):
        for side, graph in zip(sides, graphs):
            with torch.cuda.stream(side):
                graph.replay()
        torch.cuda.synchronize()
        for out, one in zip(outs, want):
            assert all(torch.equal(a, b) for a, b in zip(out, one))
