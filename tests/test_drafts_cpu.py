"""Decoding with drafts on the host: the plain statements beside each other and beside brute force, and the operators' checks of
their arguments, which run before anything is launched."""
import numpy as np
import pytest
import torch

import plain_drafts as plain
import plain_qwen3


def test_streams_are_those_of_the_sampler():
    """The noise of a row is the sampler's, block by block and as a whole."""
    rng = np.random.RandomState(0)
    for vocab, seed, stream, step in ((389, 11, 3, 0), (64, 2 ** 40 + 5, 7, 900)):
        row = rng.randn(vocab).astype(np.float32) * 2
        u = plain.uniforms(vocab, step, stream, 0, seed)
        assert all(plain.uniform(plain.philox(i // 4, step, stream, 0, seed)[i % 4]) == u[i] for i in (0, 1, 5, vocab - 1))
        for k in (0, 5):
            want = plain_qwen3.sample(row, greedy=False, temperature=0.8, topk=k, seed=seed, stream=stream, step=step)
            assert plain.draw(row, temperature=0.8, topk=k, greedy=False, seed=seed, stream=stream, step=step)[0] == want


def test_the_rule_for_drawn_drafts_gives_the_target_s_distribution():
    """min(p, q) summed with the rest drawn from what is left of p beyond q is p."""
    rng = np.random.RandomState(1)
    p, q = (plain.probabilities(plain.scaled((rng.randn(20) * 2).astype(np.float32), 0.9, 12)) for _ in range(2))
    left = np.maximum(p - q, 0)
    total = np.minimum(p, q) + (1 - np.minimum(p, q).sum()) * left / left.sum()
    assert np.abs(total - p).max() < 1e-15


def test_lookup_of_drafts():
    assert plain.ngram([1, 2, 3, 9, 1, 2, 3], max_drafts=3) == [9, 1, 2]
    assert plain.ngram([5, 5, 5], max_drafts=4) == [5, 5, 5, 5]
    assert plain.ngram([1, 2, 1, 2], max_drafts=5, max_match=2) == [1, 2, 1, 2, 1]
    assert plain.ngram([1, 2, 3], max_drafts=3) == [] and plain.ngram([], max_drafts=3) == [] and plain.ngram([4], max_drafts=3) == []
    assert plain.ngram([1, 7, 2, 7, 3, 7], max_drafts=1) == [3]                    # the latest
    assert plain.ngram([8, 7, 2, 7, 3, 8, 7], max_drafts=1) == [2]                 # the longest before the latest
    assert plain.ngram([7, 2, 7], max_drafts=1, min_match=2, max_match=2) == []


@pytest.fixture
def ops(monkeypatch):
    """The operators with host tensors let through to the launch, which is recorded instead of made."""
    from tinyinfer_b200 import ops
    real = ops._check

    def check(t, name, dtype=None, ndim=None):
        if isinstance(t, torch.Tensor) and not t.is_cuda:
            if dtype is not None and t.dtype != dtype:
                raise ops.KernelError(f"{name} must be {dtype}")
            if ndim is not None and t.dim() != ndim:
                raise ops.KernelError(f"{name} must have {ndim} dimensions")
            if not t.is_contiguous():
                raise ops.KernelError(f"{name} must be contiguous")
            return t
        return real(t, name, dtype, ndim)

    calls = []
    monkeypatch.setattr(ops, "_check", check)
    monkeypatch.setattr(ops, "_stream_of", lambda device: 0)
    monkeypatch.setattr(ops, "_verify_scratch_words", lambda *a: 16)
    monkeypatch.setattr(ops, "_run", lambda lib, name, *args: calls.append((name, args)))
    ops_calls = ops
    ops_calls.calls = calls
    yield ops_calls
    del ops.calls


def i32(*values):
    return torch.tensor(values, dtype=torch.int32)


def test_host_tensors_are_refused():
    from tinyinfer_b200 import ops
    with pytest.raises(ops.KernelError, match="CUDA tensor"):
        ops.verify_drafts(torch.zeros(2, 4), i32(0, 1), i32(0, 2), max_drafts=1)
    with pytest.raises(ops.KernelError, match="CUDA tensor"):
        ops.ngram_drafts(torch.zeros(2, 4, dtype=torch.int32), i32(0, 1), max_drafts=1)
    with pytest.raises(ops.KernelError, match="CUDA tensor"):
        ops.step_arrays(i32(0), i32(1), torch.zeros(1, 4, dtype=torch.int32), rows=1, max_count=1, page_size=16)


def sampling(s=2):
    return dict(temperature=torch.ones(s), topk=torch.zeros(s, dtype=torch.int32), greedy=torch.zeros(s, dtype=torch.int32),
                seed=torch.zeros(s, dtype=torch.int64), stream_id=torch.zeros(s, dtype=torch.int32), step=torch.zeros(s, dtype=torch.int32))


def test_arguments_of_the_verification(ops):
    x, fed, cu = torch.zeros(4, 9), i32(1, 2, 3, 4), i32(0, 2, 4)
    good = sampling()
    for kw, said in ((dict(max_drafts=-1), "max_drafts"), (dict(max_drafts=32), "max_drafts"),
                     (dict(max_drafts=1, temperature=good["temperature"]), "go together"),
                     (dict(max_drafts=1, draft_logits=torch.zeros(2, 1, 9)), "no use"),
                     (dict(max_drafts=1, draft_logits=torch.zeros(2, 2, 9), **good), "draft_logits must be"),
                     (dict(max_drafts=2, draft_logits=torch.zeros(2, 9, 2).transpose(1, 2), **good), "side by side"),
                     (dict(max_drafts=1, draft_logits=torch.zeros(2, 1, 9, dtype=torch.bfloat16), **good), "float32"),
                     (dict(max_drafts=1, **dict(good, topk=good["topk"].long())), "topk"),
                     (dict(max_drafts=1, **dict(good, step=good["step"][:1])), "one entry per request")):
        with pytest.raises(ops.KernelError, match=said):
            ops.verify_drafts(x, fed, cu, **kw)
    for args in ((x.t(), fed, cu), (x.double(), fed, cu), (x, fed[:3], cu), (x, fed.long(), cu), (x, fed, cu[:0]), (torch.zeros(4, 0), fed, cu)):
        with pytest.raises(ops.KernelError):
            ops.verify_drafts(*args, max_drafts=1)
    assert not ops.calls
    q = torch.zeros(3, 2, 9).transpose(0, 1)             # draft by draft
    out = ops.verify_drafts(x, fed, cu, max_drafts=3, draft_logits=q, **good)
    assert out.tokens.shape == (2, 4) and out.accept.shape == (2, 3) and out.counts.shape == (2,)
    name, args = ops.calls.pop()
    assert name == "ti_verify_drafts" and args[6:10] == (4, 9, 2, 3) and args[17:19] == (9, 18)
    ops.verify_drafts(x, fed, cu, max_drafts=0)
    assert ops.calls.pop()[1][10:17] == (None,) * 7


def test_arguments_of_the_lookup(ops):
    h, n = torch.zeros(2, 8, dtype=torch.int32), i32(3, 4)
    for kw in (dict(max_drafts=32), dict(max_drafts=2, max_match=33), dict(max_drafts=2, min_match=0), dict(max_drafts=2, max_match=2, min_match=3),
               dict(max_drafts=2, tokens=i32(1, 2).view(2, 1)), dict(max_drafts=2, tokens=i32(1).view(1, 1), counts=i32(1)),
               dict(max_drafts=2, tokens=torch.zeros(2, 513, dtype=torch.int32), counts=n), dict(max_drafts=2, limits=i32(1)),
               dict(max_drafts=2, state_slots=n.long())):
        with pytest.raises(ops.KernelError):
            ops.ngram_drafts(h, n, **kw)
    for args in ((h, i32(3, 4, 5)), (h.t(), n), (h.long(), n), (h[0], n)):
        with pytest.raises(ops.KernelError):
            ops.ngram_drafts(*args, max_drafts=2)
    assert not ops.calls
    out = ops.ngram_drafts(h, i32(3, 4, 5), max_drafts=2, state_slots=i32(0, 1, 1))
    assert out.tokens.shape == (3, 3) and out.starts.shape == (3,) and out.lengths.shape == (3,)


def test_arguments_of_a_step_s_arrays(ops):
    table = i32(1, 2, 3, 4).view(2, 2)
    fine = dict(rows=4, max_count=2, page_size=8)
    for kw in (dict(rows=-1), dict(max_count=0), dict(page_size=0), dict(tokens=i32(1, 2).view(2, 1)), dict(state_slots=i32(0))):
        with pytest.raises(ops.KernelError):
            ops.step_arrays(i32(0, 1), i32(1, 1), table, **dict(fine, **kw))
    for starts, counts in ((i32(0, 1, 2), i32(1, 1, 1)), (i32(0, 1), i32(1)), (i32(0, 1).long(), i32(1, 1))):
        with pytest.raises(ops.KernelError):
            ops.step_arrays(starts, counts, table, **fine)
    assert not ops.calls
    out = ops.step_arrays(i32(0, 1), i32(1, 1), torch.zeros(3, 2, 5, dtype=torch.int32), rows=7, max_count=300, page_size=8,
                          tokens=torch.zeros(2, 300, dtype=torch.int32))
    assert {n: tuple(getattr(out, n).shape) for n in out._fields} == dict(
        token_ids=(7,), positions=(7,), token_seq=(7,), cache_slots=(3, 7), cu_seqlens=(4,), q_starts=(3,), context_lens=(3,),
        tiles=(6, 4), block_tables=(3, 3, 5))
    spans = sorted((t.data_ptr(), t.data_ptr() + 4 * t.numel()) for t in out)
    assert all(a[1] <= b[0] and b[0] % 16 == spans[0][0] % 16 for a, b in zip(spans, spans[1:]))


def test_status_words():
    from tinyinfer_b200 import ops
    assert "more tokens than its arrays" in ops.status_message(0, 5) and "text has no row" in ops.status_message(0, 6)
    assert "without a page" in ops.status_message(0, 1) and ops.status_message(0, 0) is None


@pytest.mark.parametrize("kw", [dict(rows=1 << 30), dict(rows=1 << 32), dict(max_count=1 << 30), dict(max_count=(1 << 32) + 2),
                                dict(page_size=1 << 32), dict(page_size=(1 << 32) + 8), dict(pad_page=1 << 31)])
def test_sizes_that_pass_32_bits_are_refused(ops, kw):
    with pytest.raises(ops.KernelError, match="bad sizes"):
        ops.step_arrays(i32(0, 1), i32(1, 1), i32(1, 2, 3, 4).view(2, 2), **dict(dict(rows=4, max_count=2, page_size=8), **kw))
    assert not ops.calls


def test_a_status_without_a_word_or_of_another_device_is_refused(ops):
    table, h = i32(1, 2, 3, 4).view(2, 2), torch.zeros(2, 8, dtype=torch.int32)
    for status in (i32(), torch.zeros(1, dtype=torch.int32, device="meta")):
        with pytest.raises(ops.KernelError):
            ops.step_arrays(i32(0, 1), i32(1, 1), table, rows=4, max_count=2, page_size=8, status=status)
        with pytest.raises(ops.KernelError):
            ops.ngram_drafts(h, i32(3, 4), max_drafts=2, status=status)
    assert not ops.calls
