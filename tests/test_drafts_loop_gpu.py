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


@pytest.mark.parametrize("n", [70001, 9000])
@pytest.mark.parametrize("max_match,min_match", [(32, 1), (32, 32), (3, 2)])
def test_long_texts_of_one_token(ops, n, max_match, min_match):
    """Every place matches: the latest is taken. Behind one other token, which the longest matches do not pass, and repeated in pairs."""
    texts = torch.full((4, n + 3), 7, dtype=torch.int32)
    texts[1, n - 20] = 8
    texts[2, ::2] = 6
    texts[3, n - 1] = 8
    got = ops.ngram_drafts(texts.to(dev()), ints([n] * 4), max_drafts=5, max_match=max_match, min_match=min_match)
    for i in range(4):
        text = texts[i, :n].tolist()
        tail, best = text[-200:], (0, 0)
        # a match ends as far back as 200 tokens only if none of that length stands nearer: the texts repeat within 25 tokens, or never match
        for e in range(1, n) if i == 3 else list(range(n - 100, n)) + list(range(1, 100)):
            l = 0
            while l < min(max_match, e) and text[e - 1 - l] == text[n - 1 - l]:
                l += 1
            best = max(best, (l, e)) if l >= min_match else best
        want = list(text)
        for t in range(5 if best[0] else 0):
            want.append(want[best[1] + t])
        assert got.tokens[i].tolist() == text[-1:] + want[n:] + [-1] * (5 - len(want) + n), i


def test_two_threads_at_once(ops):
    """Each with its own stream and vocabulary, the larger of which needs more shared memory than any kernel has without asking."""
    import threading

    def job(vocab, out, barrier):
        g = torch.Generator().manual_seed(vocab)
        rows = (2.0 * torch.randn(8, vocab, generator=g)).to(dev())
        opts = dict(temperature=torch.full((4,), 0.8, device=dev()), topk=ints([100] * 4), greedy=ints([0] * 4), stream_id=ints([1, 2, 3, 4]),
                    seed=ints([5] * 4, torch.int64), step=ints([0] * 4))
        want = ops.sample(rows[::2].contiguous(), *(opts[n] for n in ("temperature", "topk", "greedy", "seed", "stream_id", "step")))
        fed = torch.stack((want, want), 1).flatten()
        torch.cuda.synchronize()
        stream = torch.cuda.Stream()
        try:
            with torch.cuda.stream(stream):
                barrier.wait(60)
                got = [ops.verify_drafts(rows, fed, ints([0, 2, 4, 6, 8]), max_drafts=1, **opts) for _ in range(20)]
            stream.synchronize()
            out.append(all(g.counts.tolist() == [2] * 4 and torch.equal(g.tokens[:, 0], want) for g in got))
        except Exception as e:                           # noqa: BLE001 (said by the test's own thread)
            out.append(e)

    out, barrier, lock = [], threading.Barrier(2), [40007, 400009]
    threads = [threading.Thread(target=job, args=(v, out, barrier)) for v in lock]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert out == [True, True]
