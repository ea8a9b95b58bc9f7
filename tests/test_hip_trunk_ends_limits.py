"""GPU tests of a trunk's ends at the sizes where their offsets, their scratch memory or their shared memory end, and of
calls made at once. Tolerances are those of test_hip_trunk_ends, counted over the rows that have a part in a sum: zeros are
added exactly.
"""

import threading

import pytest
import torch

import ends_cases as oracle
from test_hip_trunk_ends import (Bounds, Make, check_gradients, check_loss, counted, dtype, half_step, loss_case, step_of, trunk,  # noqa: F401
                                 within)

pytestmark = pytest.mark.gpu


def check_choice(x, weight):
    tokens, logprobs = trunk.choose(x, weight)
    b = Bounds(x, weight, torch.zeros(len(x), dtype=torch.int64).cuda())
    chosen, lse = b.z.gather(1, tokens[:, None])[:, 0], torch.logsumexp(b.z, 1)
    assert (chosen >= b.z.amax(1) - 2 * b.dz.amax(1)).all()
    within("logprobs", logprobs, chosen - lse, b.lse + b.dz.amax(1) + 2.0 ** -23 * (lse.abs() + chosen.abs()))


@pytest.mark.parametrize("rows,vocab,width", [(59, 700, 512), (60, 700, 512), (3, 900, 8192), (7, 700, 8192), (64, 300, 463), (64, 300, 465), (70, 1, 40),
                                              (1, 1, 8192), (130, 300, 8192), (1100, 1, 3)])
def test_shared_memory_and_one_word(dtype, rows, vocab, width):  # noqa: F811
    """About as many rows as shared memory holds, the longest rows, and a vocabulary of one word."""
    x, weight, targets, m = loss_case(dtype, rows, vocab, width)
    lse = check_loss(x, weight, targets)
    check_gradients(x, weight, targets, lse, m(rows, dtype=torch.float32), m(rows, dtype=torch.float32))
    check_choice(x, weight)


@pytest.mark.parametrize("masked", [0.0, 0.45, 0.97])
@pytest.mark.parametrize("rows,vocab,width", [(3800, 3900, 330), (5000, 2500, 609), (1000, 9000, 100), (2100, 700, 1300)])
def test_uneven_shares(dtype, rows, vocab, width, masked):  # noqa: F811
    """Tiles that no whole number of turns of the card takes, and fewer rows with a target than there are."""
    x, weight, targets, m = loss_case(dtype, rows, vocab, width, masked=masked)
    lse = check_loss(x, weight, targets)
    check_gradients(x, weight, targets, lse, m(rows, dtype=torch.float32), None)
    check_choice(x, weight)


def on_gpu(seed, dtype, *shape):  # noqa: F811
    return torch.randn(shape, generator=torch.Generator("cuda").manual_seed(seed), device="cuda", dtype=dtype)


@pytest.mark.parametrize("rows", [5, 40, 1100])
def test_the_largest_vocabulary(dtype, rows):  # noqa: F811
    """2^23 words; the matrix is laid out anew for 1,100 rows, of which 40 have a target, and its panels' offsets near 2^31."""
    vocab, width = 1 << 23, 16 if rows < 1000 else 256 // dtype.itemsize
    weight, x = on_gpu(1, dtype, vocab, width) * 0.1, on_gpu(2, dtype, rows, width)
    m = Make(dtype, 3)
    targets, da = m.ints(0, vocab, rows), m(rows, dtype=torch.float32)
    targets[-1] = vocab - 1
    if rows > 1000:
        targets[torch.randperm(rows - 1, generator=m.gen)[:rows - 40].cuda()] = vocab
    some = targets < vocab
    losses, lse = trunk.loss(x, weight, targets)
    b = Bounds(x[some], weight, targets[some])
    want, want_lse = oracle.loss(x[some], weight, targets[some])
    within("lse", lse[some], want_lse, b.lse)
    within("losses", losses[some], want, b.loss)
    del b, want, want_lse
    dx, dw = trunk.loss_backward(da, x, weight, targets, lse)
    assert not dx[~some].any() and not losses[~some].any()
    want_x, want_w = oracle.loss_backward(da[some], x[some], weight, targets[some])
    off_x, off_w = Bounds(x[some], weight, targets[some]).gradient(x[some], weight, targets[some], da[some], None)
    within("dx", dx[some], want_x, half_step(dtype) * (want_x.abs() + off_x) + off_x)
    within("dweight", dw, want_w, half_step(dtype) * (want_w.abs() + off_w) + off_w)
    del want_w, off_w
    check_choice(x[some], weight)
    y = trunk.embed(targets, weight, scale=2.0)
    within("y", y, oracle.embed(targets, weight, 2.0), 0.0)  # a power of two
    counted("dtable", trunk.embed_backward(x, targets, weight), *oracle.embed_backward(x, targets, vocab, 1.0), dtype)
    torch.cuda.empty_cache()


def test_the_most_rows(dtype):  # noqa: F811
    """2^24 rows, of which 1,000 have a weight in the gradients; the last among them."""
    rows, vocab, width = 1 << 24, 9, 8
    weight, x = on_gpu(1, dtype, vocab, width), on_gpu(2, dtype, rows, width)
    targets = torch.randint(-1, vocab, (rows,), generator=torch.Generator("cuda").manual_seed(3), device="cuda")
    losses, lse = trunk.loss(x, weight, targets)
    some = torch.cat([torch.arange(0, rows, rows // 900)[:900], torch.arange(rows - 100, rows)]).cuda()
    for at in (slice(0, 1 << 20), slice(rows - (1 << 20), rows)):
        b = Bounds(x[at], weight, targets[at])
        want, want_lse = oracle.loss(x[at], weight, targets[at])
        within("lse", lse[at], want_lse, b.lse * b.there)
        within("losses", losses[at], want, b.loss * b.there)
    da = torch.zeros(rows, device="cuda")
    da[some] = on_gpu(4, torch.float32, 1000)
    dx, dw = trunk.loss_backward(da, x, weight, targets, lse)
    want_x, want_w = oracle.loss_backward(da[some], x[some], weight, targets[some])
    off_x, off_w = Bounds(x[some], weight, targets[some]).gradient(x[some], weight, targets[some], da[some], None)
    within("dx", dx[some], want_x, half_step(dtype) * (want_x.abs() + off_x) + off_x)
    within("dweight", dw, want_w, half_step(dtype) * (want_w.abs() + off_w) + off_w)
    dx[some] = 0
    assert not dx.any()
    at = some[-200:]
    check_choice(x[at], weight)
    tokens = trunk.choose(x, weight)[0]
    assert torch.equal(tokens[at], trunk.choose(x[at], weight)[0])
    y = trunk.embed(targets, weight)
    assert torch.equal(y[at], trunk.embed(targets[at], weight))
    dy = torch.zeros_like(x)
    dy[some] = x[some]
    counted("dtable", trunk.embed_backward(dy, targets, weight), *oracle.embed_backward(dy[some], targets[some], vocab, 1.0), dtype)
    torch.cuda.empty_cache()


def test_two_threads_at_once(dtype):  # noqa: F811
    m = Make(dtype, 6)
    table, weight = m(400, 40, dtype=torch.float32), m(400, 40, scale=0.2)
    inputs = [(m.ints(-1, 400, n), m.ints(-1, 400, n)) for n in (100, 5000)]
    want = [step_of(a, table, weight, b) for a, b in inputs]
    torch.cuda.synchronize()
    wrong = []

    def run(which):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = step_of(inputs[which][0], table, weight, inputs[which][1])
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want[which])):
                    wrong.append(which)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
