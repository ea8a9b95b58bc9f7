"""GPU tests of the embedding's gradient at words that do not occur: every value of their rows is written, and nothing beside them."""

import pytest
import torch

from test_hip_trunk_ends import TYPES, trunk

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("table", list(TYPES))
@pytest.mark.parametrize("width", [1, 2, 3, 4, 5, 7, 8, 9, 15, 31, 33, 36, 60, 100, 250, 256, 257, 333, 511, 513, 516, 600, 1001, 1028, 8191, 8192])
def test_rows_of_words_that_do_not_occur(table, width):
    vocab, kind = 131, TYPES[table]
    tokens = torch.tensor([0, 130, 64, 64, -1, 77, 131]).cuda()
    dy = torch.full((7, width), 2.0, device="cuda", dtype=torch.bfloat16)
    want = torch.zeros(vocab, width, device="cuda", dtype=kind)
    for word, count in ((0, 1), (130, 1), (64, 2), (77, 1)):
        want[word] = 2.0 * count
    # What memory held before is not there any more, and what lies around the gradient is as it was.
    size = vocab * width
    whole = torch.full((size + 256,), 7.0, device="cuda", dtype=kind)
    a = trunk.CEmbed(0, trunk.DTYPES[torch.bfloat16], trunk.DTYPES[kind], 7, vocab, width, 1, 1.0, width, width, tokens.data_ptr())
    a.dy, a.dtable = dy.data_ptr(), whole[128:].data_ptr()
    trunk._call("embed_backward", a, 0)
    assert torch.equal(whole[128:size + 128].view(vocab, width), want)
    assert (whole[:128] == 7.0).all() and (whole[size + 128:] == 7.0).all()
