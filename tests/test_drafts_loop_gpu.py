"""ops.step_arrays and ops.ngram_drafts at the ends of their ranges, beside their plain statements."""
import pytest
import torch

import plain_drafts as plain

pytestmark = pytest.mark.gpu


def dev():
    return torch.device("cuda:0")


@pytest.fixture(scope="module")
def ops():
    from tinyinfer_b200 import ops
    return ops


def ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=dev())


@pytest.mark.parametrize("s,rows", [(0, 0), (0, 5), (3, 0), (3, 1)])
def test_arrays_without_requests_or_rows(ops, s, rows):
    """Tokens are taken, too, where no request brings any or no row is there for them."""
    tokens = torch.arange(s * 4, dtype=torch.int32, device=dev()).view(s, 4)
    table = [[[3, 4], [5, 6], [7, 8]]]
    counts = [1] * s if rows else [0] * s
    got = ops.step_arrays(ints([0] * s), ints(counts), ints(table), rows=rows, max_count=3, page_size=8, tokens=tokens, pad_page=9)
    want = plain.step_arrays([0] * s, counts, table, rows=rows, max_count=3, page_size=8, tokens=tokens.tolist(), pad_page=9)
    for name, value in want.items():
        assert getattr(got, name).tolist() == value or (not value and getattr(got, name).numel() == 0), name


@pytest.mark.parametrize("starts,counts", [([0, 100], [9, 1]), ([100, 0], [1, 9]), ([100], [9])])
def test_the_status_word_keeps_what_was_left_out(ops, starts, counts):
    """A request that brings too many tokens beside a token without a page, in either order, many times: one code stays."""
    table = ints([[3, 4]] * len(starts))
    for _ in range(20):
        word = torch.zeros(1, dtype=torch.int32, device=dev())
        ops.step_arrays(ints(starts), ints(counts), table, rows=20, max_count=4, page_size=8, status=word)
        assert word.item() == 5
