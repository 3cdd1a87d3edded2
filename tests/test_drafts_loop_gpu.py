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


def test_the_loop_that_the_readme_shows(ops):
    """Its lines, run as they stand around a model whose logits are a function of a token and its position: the texts are those of
    decoding one by one."""
    import re
    from pathlib import Path
    readme = (Path(__file__).resolve().parent.parent / "README.md").read_text()
    lines = next(b for b in re.findall(r"```python\n(.*?)```", readme, re.S) if "ngram_drafts" in b)
    S, D, vocab, longest, steps = 4, 3, 29, 200, 25
    g = torch.Generator().manual_seed(2)
    table = (3.0 * torch.randn(vocab, 2, vocab, generator=g)).to(dev())
    prompts, sampling = ints([3, 9, 1, 6]), dict(
        temperature=torch.tensor([1.0, 0.8, 0.5, 1.2], device=dev()), topk=ints([0, 5, 0, 0]), greedy=ints([1, 0, 0, 0]),
        seed=ints([1, 2, 3, 4], torch.int64), stream_id=ints([5, 6, 7, 8]))
    history = torch.randint(0, vocab, (S, longest), generator=g, dtype=torch.int32).to(dev())
    first, n = history.clone(), prompts.tolist()
    names = dict(S=S, D=D, history=history, lengths=prompts.clone(), prompts=prompts, spare_page=99, **sampling,
                 block_tables=torch.arange(S * 4, dtype=torch.int32, device=dev()).view(S, 4),
                 model=lambda step: table[step.token_ids.long(), step.positions.long() % 2].contiguous(),
                 found=ops.VerifiedDrafts(torch.full((S, D + 1), -1, dtype=torch.int32, device=dev()), ints([0] * S), None))
    held = 0
    for _ in range(steps):
        exec(lines, names)
        held += int((names["found"].counts - 1).sum())
    assert held > 5
    for r in range(S):
        text, made = first[r, :n[r]].tolist(), int(names["lengths"][r]) - n[r]
        assert made >= steps - 1
        for i in range(made):
            row = table[text[-1], (len(text) - 1) % 2][None].contiguous()
            one = {k: t[r:r + 1].contiguous() for k, t in sampling.items()}
            text.append(int(ops.sample(row, one["temperature"], one["topk"], one["greedy"], one["seed"], one["stream_id"], ints([i]))))
        assert history[r, :len(text)].tolist() == text, r
