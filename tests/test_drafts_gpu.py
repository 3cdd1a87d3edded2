"""Decoding with drafts: ops.verify_drafts, ops.ngram_drafts and ops.step_arrays beside their plain statements, at the sizes and
masks where they can go wrong, and a run of the three together with a model."""
import math

import numpy as np
import pytest
import torch

import plain_drafts as plain

pytestmark = pytest.mark.gpu
NEG = float("-inf")


def dev():
    return torch.device("cuda:0")


@pytest.fixture(scope="module")
def ops():
    from tinyinfer_b200 import ops
    return ops


def ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=dev())


# ------------------------------------------------------------------------------------------------ verification
def rows_of(counts):
    cu = [0]
    for c in counts:
        cu.append(cu[-1] + c)
    return cu


def options(s, seed, temperature=None, topk=None, greedy=None):
    g = torch.Generator().manual_seed(seed)
    return dict(temperature=torch.tensor(temperature or [0.7] * s, dtype=torch.float32, device=dev()),
                topk=ints(topk or [0] * s), greedy=ints(greedy or [0] * s),
                seed=torch.randint(0, 1 << 60, (s,), generator=g).to(dev()),
                stream_id=torch.randint(0, 1 << 30, (s,), generator=g).to(torch.int32).to(dev()),
                step=torch.randint(0, 100000, (s,), generator=g).to(torch.int32).to(dev()))


def accept_tolerance(largest, vocab):
    """A probability's relative error: the scaled logit and the maximum carry half a step each (2^-24 of up to ``largest``), their
    difference another, the exponential two steps, the sum half a step per addition of a thread (at least 256 of them) and of the tree over
    them (12); p over q has that twice, and a division."""
    return 2 * 2.0 ** -24 * (4 * largest + 4 + vocab / 256 + 12) + 2.0 ** -23


def check(ops, logits, fed, counts, d, opts=None, draft_logits=None, cu=None, may_skip=0.1):
    """The operator beside the plain statement; requests with a decision closer than the arithmetic tells apart are left out of the
    comparison of tokens (their number is bounded)."""
    s = len(counts)
    cu_rows = rows_of(counts) if cu is None else cu
    got = ops.verify_drafts(logits, ints(fed), ints(cu_rows), max_drafts=d, draft_logits=draft_logits, **(opts or {}))
    tokens, n_out, accept = got.tokens.tolist(), got.counts.tolist(), got.accept.cpu().double().numpy()
    x = logits.cpu().numpy()
    host = {k: v.tolist() for k, v in (opts or {}).items()}
    sized = np.abs(x[np.isfinite(x) & (np.abs(x) < 1e30)])
    skipped = 0
    for r in range(s):
        kw = {}
        if opts:
            kw = dict(temperature=host["temperature"][r], topk=host["topk"][r], greedy=bool(host["greedy"][r]), seed=host["seed"][r],
                      stream=host["stream_id"][r], step=host["step"][r])
        largest = float(sized.max()) / kw.get("temperature", 1.0) if sized.size else 0.0
        rel = accept_tolerance(min(largest, 1e30), x.shape[1])          # (finite, so that 0 x it is 0)
        lo, hi = max(cu_rows[r], 0), min(cu_rows[r + 1], x.shape[0])
        dl = None if draft_logits is None else draft_logits[r].cpu().numpy()
        want, acc, margin = plain.verify(x[lo:max(hi, lo)], fed[lo:max(hi, lo)], max_drafts=d, draft_logits=dl, **kw)
        assert np.all(np.abs(accept[r] - acc) <= rel * acc + 1e-37), (r, accept[r], acc)
        if margin <= 2 * rel + 2e-6:
            skipped += 1
            continue
        assert n_out[r] == len(want) and tokens[r] == want + [-1] * (d + 1 - len(want)), (r, tokens[r], want, margin)
    assert skipped <= max(1, may_skip * s), skipped
    return got


def batch(counts, vocab, seed, std=2.0, hit=0.6):
    """Logits and fed tokens: a draft is the row's likely token or any."""
    g = torch.Generator().manual_seed(seed)
    n = sum(counts)
    logits = torch.randn(n, vocab, generator=g) * std
    likely = torch.randint(0, vocab, (n,), generator=g)
    logits[torch.arange(n), likely] += 6.0
    fed = torch.randint(0, vocab, (n,), generator=g)
    for i in range(n - 1):
        if torch.rand((), generator=g) < hit:
            fed[i + 1] = likely[i]
    return logits.to(dev()), fed.tolist()


def near(logits, counts, d, seed, std=0.7):
    """Draft logits near the target's, laid out draft by draft (a transposed view), NaN where there is no draft."""
    g = torch.Generator().manual_seed(seed + 1)
    s, v = len(counts), logits.shape[1]
    out = torch.full((max(d, 1), s, v), float("nan"))
    cu = rows_of(counts)
    for r in range(s):
        for j in range(min(counts[r] - 1, d)):
            out[j, r] = logits[cu[r] + j].cpu() + std * torch.randn(v, generator=g)
    return out.to(dev()).transpose(0, 1)[:, :d]


@pytest.mark.parametrize("vocab", [1, 2, 3, 5, 31, 515, 1003, 4097, 20480, 32003, 151936, 200001])
@pytest.mark.parametrize("with_q", [False, True])
def test_verification(ops, vocab, with_q):
    counts = [1, 4, 2, 3, 4, 4, 1, 3, 4, 2, 4, 4]
    d, s = 3, len(counts)
    logits, fed = batch(counts, vocab, seed=vocab)
    ks = [0, 0, 1, 2, 50, 100, 100, 256, 257, 1000, vocab, vocab + 5]
    opts = options(s, vocab, temperature=[0.5, 0.7, 1.0, 1.3] * 3, topk=ks, greedy=[0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 1])
    check(ops, logits, fed, counts, d, opts, near(logits, counts, d, vocab) if with_q else None)


def test_verification_of_greedy_requests(ops):
    counts = [1, 5, 3, 2, 5, 4]
    logits, fed = batch(counts, 1001, seed=1, hit=0.8)
    logits[2, 7] = logits[2, 900] = 40.0                 # a tie: the first index
    fed[3] = 900
    check(ops, logits, fed, counts, 4)
    mixed = options(6, 5, topk=[0, 3, 0, 50, 0, 0], greedy=[1, 0, 1, 0, 1, 1])
    check(ops, logits, fed, counts, 4, mixed)


@pytest.mark.parametrize("d", [0, 1, 7, 31])
def test_numbers_of_drafts(ops, d):
    """Up to 31 drafts; a request with more rows than max_drafts + 1 has the others passed over; requests without rows."""
    counts = [d + 1, 0, 1, d + 3, max(1, d), 0]
    logits, fed = batch(counts, 777, seed=d, hit=0.95)
    opts = options(6, d, topk=[0, 0, 10, 20, 0, 0])
    got = check(ops, logits, fed, counts, d, opts)
    assert got.counts.tolist()[1] == 0 and got.counts.tolist()[5] == 0
    clipped = [min(c, d + 1) for c in counts]
    check(ops, logits, fed, counts, d, opts, near(logits, clipped, d, d) if d else None)


def test_without_drafts_the_token_is_the_one_that_sample_draws(ops):
    for vocab, seed in ((515, 0), (32003, 1), (151936, 2)):
        s = 24
        logits, fed = batch([1] * s, vocab, seed, std=2.5)
        opts = options(s, seed, temperature=[0.6, 1.0, 1.7] * 8, topk=[0, 1, 40, 100, 256, 1000] * 4, greedy=[0, 0, 0, 0, 0, 1, 0, 0] * 3)
        got = ops.verify_drafts(logits, ints(fed), ints(range(s + 1)), max_drafts=4, **opts)
        want = ops.sample(logits, *(opts[n] for n in ("temperature", "topk", "greedy", "seed", "stream_id", "step")))
        assert got.tokens[:, 0].tolist() == want.tolist()
        assert got.counts.tolist() == [1] * s and bool((got.tokens[:, 1:] == -1).all()) and not got.accept.any()


def test_where_every_draft_holds_the_next_token_is_the_one_that_sample_draws(ops):
    """With the draft model's logits, too: no drafts, or drafts that are sure to hold (the two models' logits are the same)."""
    for vocab, k in ((515, 0), (32003, 0), (151936, 0), (32003, 40), (20000, 1000), (9000, 5000)):
        s, d = 12, 2
        logits, fed = batch([d + 1] * s, vocab, seed=vocab + k, std=2.5)
        x = logits.view(s, d + 1, vocab)
        opts = options(s, vocab, temperature=[0.6, 1.0, 1.7] * 4, topk=[k] * s)
        fed = ints(fed).view(s, d + 1)
        fed[:, 1:] = x[:, :d].argmax(2).to(torch.int32)
        for counts, rows, tokens in (([1] * s, x[:, d].contiguous(), fed[:, 0].contiguous()), ([d + 1] * s, logits, fed.flatten())):
            got = ops.verify_drafts(rows, tokens, ints(rows_of(counts)), max_drafts=d, draft_logits=x[:, :d], **opts)
            assert got.counts.tolist() == counts
            want = ops.sample(x[:, d].contiguous(), *(opts[n] for n in ("temperature", "topk", "greedy", "seed", "stream_id")),
                              opts["step"] + (counts[0] - 1))
            assert got.tokens[:, counts[0] - 1].tolist() == want.tolist(), (vocab, k, counts[0])


@pytest.mark.parametrize("vocab", [600, 40007])
def test_masks_and_values_that_are_no_numbers(ops, vocab):
    """Rows that a mask leaves empty, by -inf or by the type's lowest value; infinities; NaN; drafts outside the vocabulary; drafts
    that the mask forbids; equal logits at the threshold; a draft the draft model gives nothing."""
    counts = [3] * 10
    s, d = 10, 2
    logits, fed = batch(counts, vocab, seed=3, hit=1.0)
    x = logits.view(s, 3, vocab)
    x[0, 0] = NEG                                        # nothing: no draft holds, token 0
    x[1, 0] = float("nan")
    x[2, 0, 5:] = NEG
    fed[7] = 100                                         # forbidden by the mask
    x[3, 0] = torch.finfo(torch.float32).min             # all equal: every token alike
    x[4, 1, ::2] = float("nan")
    x[5, 0] = (x[5, 0] * 2).round() / 2                  # many equal logits at the threshold
    fed[3 * 6 + 1], fed[3 * 6 + 2] = vocab, -1           # outside the vocabulary
    x[7, 1, 17] = float("inf")
    fed[3 * 7 + 2] = 17
    x[8, 0] = torch.finfo(torch.float32).min
    x[8, 0, 11] = 3.0
    fed[3 * 8 + 1] = 11
    x[9, 0, 0], x[9, 0, 1:] = -0.0, 0.0                  # one value
    for topk in (0, 7, 100):
        opts = options(s, topk, topk=[topk] * s, temperature=[0.7] * 3 + [1.0] + [0.7] * 4 + [1.0, 0.7])
        got = check(ops, logits, fed, counts, d, opts)
        assert got.tokens[0].tolist() == [0, -1, -1] and got.tokens[1].tolist() == [0, -1, -1]
        q = near(torch.nan_to_num(logits, 0.0, 20.0, -20.0), counts, d, topk)
        q[5, 0, fed[16]] = NEG                           # q = 0 at the draft: it holds if p has anything there
        q[4, 0] = NEG                                    # a draft model's row with nothing
        q[3, 0, 3] = float("nan")
        check(ops, logits, fed, counts, d, opts, q)


@pytest.mark.parametrize("with_q", [False, True])
def test_thresholds_in_the_thousands(ops, with_q):
    """More tokens kept than a block has room for, by a large k or by equal logits: the row itself is gone over."""
    vocab, ks = 50021, [1023, 1025, 1500, 2047, 2100, 3500, 9000, 50000]
    counts = [3] * len(ks)
    logits, fed = batch(counts, vocab, seed=9, hit=0.7)
    opts = options(len(ks), 9, topk=ks, temperature=[0.8, 1.0] * 4)
    check(ops, logits, fed, counts, 2, opts, near(logits, counts, 2, 9) if with_q else None)
    x = logits.view(len(ks), 3, vocab)
    x[0, 0, ::7] = 9.0                                   # 7,146 equal logits above all but a few
    x[1, :, 100:2600] = 30.0                             # 2,500 above all
    x[2] = 1.0                                           # all of them
    x[3, 1, :] = NEG
    x[3, 1, :3000] = torch.linspace(-1, 1, 3000, device=dev())           # fewer than k are left
    opts = options(len(ks), 10, topk=[10, 100, 5, 4000, 40, 40, 40, 40], temperature=[0.8, 1.0] * 4)
    check(ops, logits, fed, counts, 2, opts, near(logits.nan_to_num(0.0, 20.0, -20.0), counts, 2, 10) if with_q else None,
          may_skip=0.3)


@pytest.mark.parametrize("vocab", [2500, 40007])
@pytest.mark.parametrize("with_q", [False, True])
def test_thresholds_in_the_hundreds(ops, vocab, with_q):
    ks = [255, 256, 383, 384, 385, 450, 511, 512, 513, 700, 1023, 1500]
    counts = [3] * len(ks)
    logits, fed = batch(counts, vocab, seed=vocab + 1)
    logits[4] = torch.round(logits[4])                       # many equal ones, at the threshold too
    check(ops, logits, fed, counts, 2, options(len(ks), vocab, topk=ks), near(logits, counts, 2, vocab) if with_q else None)


def test_many_requests_and_the_largest_vocabulary(ops):
    rng = np.random.RandomState(4)
    counts = rng.randint(0, 4, 400).tolist()
    logits, fed = batch(counts, 300, seed=13)
    opts = options(400, 13, topk=rng.choice([0, 1, 20, 299], 400).tolist(), greedy=rng.choice([0, 0, 1], 400).tolist(),
                   temperature=rng.choice([0.5, 1.0, 1.5], 400).tolist())
    check(ops, logits, fed, counts, 3, opts)
    check(ops, logits, fed, counts, 3, opts, near(logits, counts, 3, 13))
    for vocab in (1 << 19, (1 << 19) + 1):
        x = torch.randn(2, vocab, device=dev())
        x[0, vocab - 1] = 12.0
        one = options(1, 1, topk=[50])
        if vocab > 1 << 19:
            with pytest.raises(ops.KernelError, match="vocabulary"):
                ops.verify_drafts(x, ints([0, vocab - 1]), ints([0, 2]), max_drafts=1, **one)
            continue
        for opts in (None, one, options(1, 2)):
            check(ops, x, [0, vocab - 1], [2], 1, opts, may_skip=1)


def test_temperatures(ops):
    counts = [3] * 6
    logits, fed = batch(counts, 3001, seed=8, hit=0.5)
    opts = options(6, 1, temperature=[1e-3, 0.05, 100.0, 1e6, 1e-30, 3e-39], topk=[0, 5, 0, 9, 0, 5])
    check(ops, logits, fed, counts, 2, opts, may_skip=0.5)
    check(ops, logits, fed, counts, 2, opts, near(logits, counts, 2, 4), may_skip=0.5)


def test_rows_that_no_request_claims_are_not_looked_at(ops):
    counts = [3, 2, 4]
    logits, fed = batch(counts, 1500, seed=5)
    opts = options(3, 2, topk=[0, 10, 0])
    want = ops.verify_drafts(logits, ints(fed), ints([0, 3, 5, 9]), max_drafts=3, **opts)
    more = torch.full((16, 1500), float("nan"), device=dev())
    more[2:5], more[7:9], more[9:13] = logits[:3], logits[3:5], logits[5:9]
    fed2 = [9] * 2 + fed[:3] + [9] * 2 + fed[3:]+ [9] * 3
    # requests need not cover all rows: the first begins behind row 0, the last ends before the end
    a = ops.verify_drafts(more, ints(fed2), ints([2, 5, 5, 5]), max_drafts=3, **opts)
    assert a.tokens[0].tolist() == want.tokens[0].tolist() and a.counts.tolist() == [want.counts[0].item(), 0, 0]
    # bounds that are none: clipped to the rows there are, an end before its beginning is no row
    b = ops.verify_drafts(logits, ints(fed), ints([-7, 3, 1, 4]), max_drafts=3, **opts)
    assert b.tokens[0].tolist() == want.tokens[0].tolist() and b.counts[1].item() == 0
    c = ops.verify_drafts(logits, ints(fed), ints([5, 400, 2 ** 31 - 1, -2 ** 31]), max_drafts=3, **opts)
    assert c.counts[1].item() == 0 and c.counts[2].item() == 0
    none = ops.verify_drafts(logits[:0], ints([]), ints([0, 0, 0, 0]), max_drafts=3, **opts)
    assert none.counts.tolist() == [0, 0, 0] and bool((none.tokens == -1).all())
    assert ops.verify_drafts(logits, ints(fed), ints([0]), max_drafts=3).tokens.shape == (0, 4)


@pytest.mark.parametrize("shift", [1, 2, 3])
def test_rows_off_sixteen_byte_boundaries(ops, shift):
    counts = [4, 2, 3]
    for vocab in (1024, 1025, 32002):
        logits, fed = batch(counts, vocab, seed=vocab + shift)
        wide = torch.full((logits.numel() + 8,), float("nan"), device=dev())
        moved = wide[shift:shift + logits.numel()].view(logits.shape)
        moved.copy_(logits)
        q = near(logits, counts, 3, 6)
        wide_q = torch.full((3, 3, vocab + shift), float("nan"), device=dev())     # rows further apart than they are long
        wide_q[:, :, :vocab] = q
        opts = options(3, vocab, topk=[0, 20, 0])
        a = check(ops, moved, fed, counts, 3, opts, wide_q[:, :, :vocab])
        b = ops.verify_drafts(logits, ints(fed), ints(rows_of(counts)), max_drafts=3, draft_logits=q.contiguous(), **opts)
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_the_same_draft_logits_let_every_draft_hold(ops):
    counts = [5] * 8
    logits, fed = batch(counts, 2048, seed=4)
    x = logits.view(8, 5, 2048)
    for k in (0, 30):
        opts = options(8, k, topk=[k] * 8)
        # drafts drawn from the very distribution: the ratio is 1
        drawn = ops.sample(x[:, :4].reshape(32, 2048).contiguous(), *(opts[n].repeat_interleave(4) for n in (
            "temperature", "topk", "greedy", "seed", "stream_id", "step"))).view(8, 4)
        fed_t = ints(fed).view(8, 5).clone()
        fed_t[:, 1:] = drawn
        got = ops.verify_drafts(logits, fed_t.flatten(), ints(rows_of(counts)), max_drafts=4, draft_logits=x[:, :4], **opts)
        assert bool((got.accept == 1.0).all()) and got.counts.tolist() == [5] * 8
        assert torch.equal(got.tokens[:, :4], drawn)


@pytest.mark.parametrize("topk", [0, 6])
@pytest.mark.parametrize("drawn", [False, True])
def test_tokens_are_distributed_as_the_target_says(ops, topk, drawn):
    """40,000 requests with one draft and the same rows: the first token's frequencies are the target's softmax, whether the draft was
    drawn (with sample's noise of the same stream and step) or certain. A frequency is off by more than five standard deviations
    once in two million."""
    v, n, t = 12, 40000, 0.9
    g = torch.Generator().manual_seed(11)
    target, other = torch.randn(v, generator=g) * 1.5, torch.randn(v, generator=g) * 1.5
    opts = options(n, 6, temperature=[t] * n, topk=[topk] * n)
    opts["seed"] = torch.full((n,), 1234, dtype=torch.int64, device=dev())
    opts["stream_id"] = torch.arange(n, dtype=torch.int32, device=dev())
    q = other.to(dev()).expand(n, v).contiguous()
    if drawn:
        draft = ops.sample(q, *(opts[k] for k in ("temperature", "topk", "greedy", "seed", "stream_id", "step")))
    else:
        draft = torch.full((n,), 3, dtype=torch.int32, device=dev())
    fed = torch.stack((torch.zeros_like(draft), draft), 1).flatten().contiguous()
    logits = target.to(dev()).expand(2 * n, v).contiguous()
    got = ops.verify_drafts(logits, fed, torch.arange(0, 2 * n + 1, 2, dtype=torch.int32, device=dev()), max_drafts=1,
                            draft_logits=q.view(n, 1, v) if drawn else None, **opts)
    p = plain.probabilities(plain.scaled(target.numpy(), t, topk))
    for token in (got.tokens[:, 0], got.tokens[:, 1][got.counts == 2]):       # the bonus token too
        if not len(token):                               # the draft is below the threshold: it never holds
            continue
        freq = np.bincount(token.cpu().numpy(), minlength=v) / len(token)
        assert np.all(np.abs(freq - p) <= 5.0 * np.sqrt(p * (1 - p) / len(token)) + 1e-9), (freq, p)
    held = float((got.counts == 2).double().mean())
    pq = plain.probabilities(plain.scaled(other.numpy(), t, topk))
    likely = float(np.minimum(p, pq).sum()) if drawn else float(p[3])
    assert abs(held - likely) <= 5.0 * math.sqrt(likely * (1 - likely) / n) + 1e-9


def test_a_request_does_not_depend_on_its_batch(ops):
    counts = [3, 5, 1, 4, 5, 2]
    logits, fed = batch(counts, 5003, seed=12)
    opts = options(6, 3, topk=[0, 40, 0, 0, 100, 3])
    q = near(logits, counts, 4, 2)
    whole = ops.verify_drafts(logits, ints(fed), ints(rows_of(counts)), max_drafts=4, draft_logits=q, **opts)
    cu = rows_of(counts)
    for r in range(6):
        one = ops.verify_drafts(logits[cu[r]:cu[r + 1]].contiguous(), ints(fed[cu[r]:cu[r + 1]]), ints([0, counts[r]]), max_drafts=4,
                                draft_logits=q[r:r + 1], **{k: t[r:r + 1] for k, t in opts.items()})
        assert all(torch.equal(a[0], b[r]) for a, b in zip(one, whole))


def test_two_streams_and_two_graphs_do_not_meet(ops):
    """Calls of different sizes on two streams at once, and two captured graphs replayed side by side, give what they give alone."""
    cases = []
    for vocab, s, k in ((60001, 9, 0), (32000, 17, 50)):
        counts = [4] * s
        logits, fed = batch(counts, vocab, seed=vocab)
        cases.append(dict(args=(logits, ints(fed), ints(rows_of(counts))), kw=dict(max_drafts=3, draft_logits=near(logits, counts, 3, s),
                                                                                 **options(s, s, topk=[k] * s))))
    want = [ops.verify_drafts(*c["args"], **c["kw"]) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(20):
        for i, (c, st) in enumerate(zip(cases, streams)):
            with torch.cuda.stream(st):
                got[i].append(ops.verify_drafts(*c["args"], **c["kw"]))
    torch.cuda.synchronize()
    for w, outs in zip(want, got):
        assert all(torch.equal(a, b) for o in outs for a, b in zip(o, w))
    graphs, outs = [], []
    for c in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.verify_drafts(*c["args"], **c["kw"]))
        graphs.append(g)
    for _ in range(5):
        for o in outs:
            for t in o:
                t.zero_()
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for o, w in zip(outs, want) for a, b in zip(o, w))


# ------------------------------------------------------------------------------------------------ drafts from the text
def ngram_check(ops, texts, d, max_match=3, min_match=1, room=None, limits=None, new=None):
    room = room or max(len(t) for t in texts) + 8
    history = torch.full((len(texts), room), -9, dtype=torch.int32)
    for i, t in enumerate(texts):
        history[i, :len(t)] = torch.tensor(t, dtype=torch.int32)
    history = history.to(dev())
    kw = {}
    if new is not None:
        width = max(1, max(len(t) for t in new))
        kw = dict(tokens=ints([list(t) + [77] * (width - len(t)) for t in new]), counts=ints([len(t) for t in new]))
    status = torch.zeros(1, dtype=torch.int32, device=dev())
    got = ops.ngram_drafts(history, ints([len(t) for t in texts]), max_drafts=d, max_match=max_match, min_match=min_match,
                           limits=None if limits is None else ints(limits), status=status, **kw)
    for i, t in enumerate(texts):
        text = list(t) + (list(new[i]) if new is not None else [])
        want = plain.ngram(text, max_drafts=d, max_match=max_match, min_match=min_match)
        want = want[:d if limits is None else min(d, max(0, limits[i]))]
        first = [text[-1]] if text else []
        assert got.tokens[i].tolist() == first + want + [-1] * (d + 1 - len(first) - len(want)), (i, want)
        assert (got.counts[i].item(), got.starts[i].item(), got.lengths[i].item()) == (len(first) + len(want), max(0, len(text) - 1), len(text))
        assert history[i].tolist() == text + [-9] * (room - len(text))
    assert status.item() == 0
    return got


@pytest.mark.parametrize("words", [1, 2, 5, 40, 3000])
@pytest.mark.parametrize("max_match,min_match", [(1, 1), (3, 1), (4, 2), (32, 3)])
def test_drafts_from_the_text(ops, words, max_match, min_match):
    g = np.random.RandomState(words * 37 + max_match)
    texts = [g.randint(0, words, n).tolist() for n in (0, 1, 2, 3, 4, 7, 31, 33, 200, 511, 512, 513, 1500)]
    ngram_check(ops, texts, 5, max_match, min_match)
    new = [g.randint(0, words, n % 7).tolist() for n in range(len(texts))]
    ngram_check(ops, texts, 5, max_match, min_match, new=new)
    ngram_check(ops, texts, 5, max_match, min_match, limits=[i - 2 for i in range(len(texts))])


def test_drafts_from_long_texts(ops):
    """The only occurrence lies at the very beginning, in the middle of the text, right before its end; the latest of equals wins."""
    g = np.random.RandomState(5)
    n = 70001
    texts = []
    for at in (0, 1, 4099, 35000, n - 8, n - 4, None):
        t = (np.arange(n) % 50000 + 10).astype(int)
        t = g.permutation(t)
        t[t < 4] = 5
        t[-3:] = (1, 2, 3)
        if at is not None:
            t[at:at + 3] = (1, 2, 3)
        texts.append(t.tolist())
    texts[6][100:103] = texts[6][40000:40003] = [1, 2, 3]
    history = torch.tensor(texts, dtype=torch.int32, device=dev())
    got = ops.ngram_drafts(history, ints([n] * 7), max_drafts=4, max_match=3, min_match=3)
    for i, t in enumerate(np.array(texts)):
        same = (t[:-3] == t[-3]) & (t[1:-2] == t[-2]) & (t[2:-1] == t[-1])         # of the three tokens from there on
        found = np.flatnonzero(same)
        want = [-1] * 4
        if len(found):
            period = t[found[-1] + 3:]                   # behind the end the drafts go on as they began
            want = [int(period[j % len(period)]) for j in range(4)]
        assert got.tokens[i].tolist() == [int(t[-1])] + want, i
    assert got.counts.tolist() == [5, 5, 5, 5, 5, 1, 5]  # (the sixth overwrote its own end)


def test_texts_by_slot_and_texts_that_do_not_fit(ops):
    history = torch.full((5, 12), -9, dtype=torch.int32, device=dev())
    history[3, :6] = ints([1, 2, 3, 1, 2, 3])
    history[0, :12] = ints(list(range(12)))
    before = history.clone()
    status = torch.zeros(1, dtype=torch.int32, device=dev())
    tokens, counts = ints([[1, 2], [7, 7], [7, 7], [7, 7], [5, 6]]), ints([1, 1, 1, 1, 2])
    # row 3; a full row; no such rows; a length that is none
    got = ops.ngram_drafts(history, ints([6, 12, 4, 4, -1]), max_drafts=2, tokens=tokens, counts=counts,
                           state_slots=ints([3, 0, 5, -1, 2]), status=status)
    assert got.tokens.tolist() == [[1, 2, 3], [-1] * 3, [-1] * 3, [-1] * 3, [-1] * 3]
    assert got.counts.tolist() == [3, 0, 0, 0, 0] and got.starts.tolist() == [6, 0, 0, 0, 0] and got.lengths.tolist() == [7, 12, 0, 0, 0]
    assert status.item() == 6
    before[3, 6] = 1
    assert torch.equal(history, before)
    # counts beyond the tokens there are, and below none
    got = ops.ngram_drafts(history, ints([3, 3]), max_drafts=1, tokens=ints([[5], [6]]), counts=ints([9, -3]), state_slots=ints([1, 2]))
    assert got.lengths.tolist() == [4, 3] and history[1, 3].item() == 5 and history[2, 3].item() == -9


# ------------------------------------------------------------------------------------------------ a step's arrays
def arrays_check(ops, starts, counts, tables, *, rows, max_count, page_size, with_tokens=True, state_slots=None, pad_page=-1, status=0):
    g = np.random.RandomState(rows + page_size)
    tokens = g.randint(0, 1000, (len(starts), max_count + 2)).tolist() if with_tokens else None
    word = torch.zeros(1, dtype=torch.int32, device=dev())
    got = ops.step_arrays(ints(starts), ints(counts), ints(tables), rows=rows, max_count=max_count, page_size=page_size,
                          tokens=ints(tokens) if with_tokens and starts else None,
                          state_slots=None if state_slots is None else ints(state_slots), pad_page=pad_page, status=word)
    want = plain.step_arrays(starts, counts, tables, rows=rows, max_count=max_count, page_size=page_size,
                             tokens=tokens if starts else None, state_slots=state_slots, pad_page=pad_page)
    for name, value in want.items():
        mine = getattr(got, name)
        assert (mine is None) == (value is None), name
        if value is not None:
            assert mine.tolist() == value, name
            assert mine.data_ptr() % 16 == 0 and mine.is_contiguous()
    assert word.item() == status
    return got


@pytest.mark.parametrize("s", [1, 2, 7, 64, 300, 1100])
@pytest.mark.parametrize("page_size,max_count,groups", [(16, 5, 1), (64, 1, 3), (24, 300, 2)])
def test_arrays_of_a_step(ops, s, page_size, max_count, groups):
    if s * max_count > 60000:
        max_count = 60000 // s
    g = np.random.RandomState(s + page_size)
    counts = [0 if g.rand() < 0.2 else int(g.randint(1, max_count + 1)) for _ in range(s)]
    starts = [int(x) for x in g.randint(0, 900, s)]
    width = -(-(900 + max_count) // page_size) + (s % 3)
    slots = g.permutation(s + 4)[:s].tolist()
    tables = g.randint(0, 5000, (groups, s + 4, width)).tolist()
    arrays_check(ops, starts, counts, tables, rows=sum(counts) + s % 5, max_count=max_count, page_size=page_size, state_slots=slots, pad_page=5000)
    arrays_check(ops, starts, counts, tables, rows=sum(counts), max_count=max_count, page_size=page_size, with_tokens=False)


def test_arrays_that_do_not_fit(ops):
    table = [[[3, 4, 5, 6], [7, 8, -1, 9], [1, 2, 0, 10]]]
    # more tokens than rows: cut off, in the middle of a request
    arrays_check(ops, [0, 5, 2], [3, 4, 5], table, rows=9, max_count=5, page_size=8, status=5)
    arrays_check(ops, [0, 5, 2], [3, 4, 5], table, rows=2, max_count=5, page_size=8, status=5)
    # more than max_count of one request
    arrays_check(ops, [0, 5, 2], [3, 4, 9], table, rows=20, max_count=5, page_size=8, status=5)
    # no such row of the tables; a start that is none; counts below zero bring nothing
    arrays_check(ops, [0, 5, 2], [2, 2, 2], table, rows=8, max_count=5, page_size=8, state_slots=[0, 3, 1], status=5)
    arrays_check(ops, [0, -5, 2], [2, 2, 2], table, rows=8, max_count=5, page_size=8, status=5)
    arrays_check(ops, [0, 5, 2], [2, -2, 2], table, rows=8, max_count=5, page_size=8)
    # positions without a page: a hole in the table, the table's end
    arrays_check(ops, [0, 14, 2], [2, 5, 2], table, rows=9, max_count=5, page_size=8, status=1)
    arrays_check(ops, [30, 1, 2], [4, 1, 2], table, rows=7, max_count=5, page_size=8, status=1)
    # sums that pass 32 bits
    arrays_check(ops, [0, 0, 0], [2 ** 31 - 1] * 3, table, rows=7, max_count=5, page_size=8, status=5)
    with pytest.raises(ops.KernelError):
        ops.step_arrays(ints([0]), ints([1]), ints([[1]]), rows=2 ** 30 + 1, max_count=1, page_size=8)
    # a slot beyond 32 bits is no slot
    word = torch.zeros(1, dtype=torch.int32, device=dev())
    got = ops.step_arrays(ints([70]), ints([1]), ints([[1, 2 ** 30]]), rows=1, max_count=1, page_size=64, status=word)
    assert got.cache_slots.tolist() == [[-1]] and word.item() == 1
    none = ops.step_arrays(ints([]), ints([]), ints([[1, 2]]), rows=2, max_count=1, page_size=64, pad_page=9)
    assert none.token_seq.tolist() == [0, 0] and none.cu_seqlens.tolist() == [0, 2] and none.block_tables.tolist() == [[[9, -1]]]


# ------------------------------------------------------------------------------------------------ all three
def test_offsets_that_pass_32_bits(ops):
    """Logits, draft logits, texts and tables of more than 2^31 elements, of which only the last are looked at."""
    buf = torch.empty((1 << 31) + (1 << 22), dtype=torch.int32, device=dev())          # 8.6 GB
    counts, vocab = [4, 2, 4], 32003
    logits, fed = batch(counts, vocab, seed=71)
    q = near(logits, counts, 3, 71)
    opts = options(3, 71, topk=[0, 20, 0])
    want = check(ops, logits, fed, counts, 3, opts, q)
    rows = buf.numel() // vocab
    far = buf[:rows * vocab].view(rows, vocab).view(torch.float32)
    far[-10:] = logits
    far_fed = torch.zeros(rows, dtype=torch.int32, device=dev())
    far_fed[-10:] = ints(fed)
    cu = ints([rows - 10 + c for c in rows_of(counts)])
    got = ops.verify_drafts(far, far_fed, cu, max_drafts=3, draft_logits=q, **opts)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    # draft logits whose requests, then whose drafts, lie 2^29 and more elements apart
    for strides in ((1 << 30, 1 << 18, 1), (1 << 18, 1 << 30, 1)):
        far_q = buf.view(torch.float32).as_strided((3, 3, vocab), strides, 1 << 20)
        assert 2 * (1 << 30) + 2 * (1 << 18) + (1 << 20) + vocab <= buf.numel()
        far_q.copy_(q)
        got = ops.verify_drafts(logits, ints(fed), ints(rows_of(counts)), max_drafts=3, draft_logits=far_q, **opts)
        assert all(torch.equal(x, y) for x, y in zip(got, want))
    # texts
    room = 1 << 20
    rows = buf.numel() // room
    history = buf[:rows * room].view(rows, room)
    history[-1, :5] = ints([4, 8, 15, 4, 8])
    got = ops.ngram_drafts(history, ints([5]), max_drafts=2, state_slots=ints([rows - 1]), tokens=ints([[15, 4]]), counts=ints([2]))
    assert got.tokens.tolist() == [[4, 8, 15]] and history[-1, :7].tolist() == [4, 8, 15, 4, 8, 15, 4]
    # tables of two groups
    rows = buf.numel() // 2048
    tables = buf[:rows * 2048].view(2, rows // 2, 1024 * 2)
    tables[0, -1, :3], tables[1, -1, :3] = ints([5, 6, 7]), ints([8, 9, 10])
    got = ops.step_arrays(ints([30]), ints([3]), tables, rows=3, max_count=3, page_size=16, state_slots=ints([rows // 2 - 1]))
    assert got.cache_slots.tolist() == [[6 * 16 + 14, 6 * 16 + 15, 7 * 16], [9 * 16 + 14, 9 * 16 + 15, 10 * 16]]
    assert got.block_tables[:, 0, :4].tolist() == [[5, 6, 7, -1], [8, 9, 10, -1]]


def test_requests_that_share_what_they_read(ops):
    """Texts and tables by the same slot twice (nothing is brought, so nothing is written), draft logits of one row for all."""
    history = ints([[9] * 8, [1, 2, 3, 1, 2, 3, 1, 0]])
    got = ops.ngram_drafts(history, ints([7, 5, 7]), max_drafts=3, state_slots=ints([1, 1, 1]))
    assert got.tokens.tolist() == [[1, 2, 3, 1], [2, 3, 1, 2], [1, 2, 3, 1]]
    arrays_check(ops, [0, 9, 0], [3, 4, 3], [[[3, 4, 5], [7, 8, 9]]], rows=12, max_count=4, page_size=8, state_slots=[1, 1, 1], pad_page=2)
    counts = [3, 2, 4]
    logits, fed = batch(counts, 2500, seed=72)
    q = (2.0 * torch.randn(2500, generator=torch.Generator().manual_seed(73))).to(dev())
    opts = options(3, 72, topk=[0, 30, 0])
    a = check(ops, logits, fed, counts, 3, opts, q.expand(3, 3, 2500))
    b = ops.verify_drafts(logits, ints(fed), ints(rows_of(counts)), max_drafts=3, draft_logits=q.expand(3, 3, 2500).contiguous(), **opts)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


# ------------------------------------------------------------------------------------------------ refusals
def test_refusals(ops):
    logits, fed, cu = torch.zeros(4, 9, device=dev()), ints([1, 2, 3, 4]), ints([0, 2, 4])
    good = options(2, 0)
    for kw in (dict(max_drafts=-1), dict(max_drafts=32), dict(max_drafts=1, temperature=good["temperature"]),
               dict(max_drafts=1, draft_logits=torch.zeros(2, 1, 9, device=dev())),
               dict(max_drafts=1, draft_logits=torch.zeros(2, 2, 9, device=dev()), **good),
               dict(max_drafts=2, draft_logits=torch.zeros(2, 9, 2, device=dev()).transpose(1, 2), **good),
               dict(max_drafts=1, draft_logits=torch.zeros(2, 1, 9, device=dev(), dtype=torch.bfloat16), **good),
               dict(max_drafts=1, **dict(good, topk=good["topk"].long())), dict(max_drafts=1, **dict(good, step=good["step"][:1]))):
        with pytest.raises(ops.KernelError):
            ops.verify_drafts(logits, fed, cu, **kw)
    for bad in ((logits.t(), fed, cu), (logits.double(), fed, cu), (logits, fed[:3], cu), (logits, fed.long(), cu), (logits.cpu(), fed, cu),
                (logits, fed, cu.cpu()), (logits, fed, cu[:0]), (torch.zeros(4, 0, device=dev()), fed, cu)):
        with pytest.raises(ops.KernelError):
            ops.verify_drafts(*bad, max_drafts=1)
    h, n = torch.zeros(2, 8, dtype=torch.int32, device=dev()), ints([3, 4])
    for bad in (dict(max_drafts=32), dict(max_drafts=2, max_match=33), dict(max_drafts=2, min_match=0), dict(max_drafts=2, max_match=2, min_match=3),
                dict(max_drafts=2, tokens=ints([[1], [2]])), dict(max_drafts=2, tokens=ints([[1]]), counts=ints([1])),
                dict(max_drafts=2, limits=ints([1])), dict(max_drafts=2, state_slots=n.long())):
        with pytest.raises(ops.KernelError):
            ops.ngram_drafts(h, n, **bad)
    with pytest.raises(ops.KernelError):
        ops.ngram_drafts(h, ints([3, 4, 5]), max_drafts=2)
    with pytest.raises(ops.KernelError):
        ops.ngram_drafts(h.t(), n, max_drafts=2)
    table = ints([[1, 2], [3, 4]])
    for bad in (dict(rows=-1), dict(max_count=0), dict(page_size=0), dict(tokens=ints([[1], [2]])), dict(state_slots=ints([0]))):
        with pytest.raises(ops.KernelError):
            ops.step_arrays(ints([0, 1]), ints([1, 1]), table, **dict(dict(rows=4, max_count=2, page_size=8), **bad))
    with pytest.raises(ops.KernelError):
        ops.step_arrays(ints([0, 1, 2]), ints([1, 1, 1]), table, rows=4, max_count=2, page_size=8)
    with pytest.raises(ops.KernelError):
        ops.step_arrays(ints([0, 1]), ints([1]), table, rows=4, max_count=2, page_size=8)


def test_tensors_of_another_device_than_the_current_one_are_refused(ops, monkeypatch):
    calls = [lambda: ops.verify_drafts(torch.zeros(2, 9, device=dev()), ints([1, 2]), ints([0, 2]), max_drafts=1),
             lambda: ops.ngram_drafts(ints([[1, 2]]), ints([2]), max_drafts=1),
             lambda: ops.step_arrays(ints([0]), ints([1]), ints([[1]]), rows=1, max_count=1, page_size=8)]
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    for call in calls:
        with pytest.raises(ops.KernelError, match="current device is cuda:1"):
            call()


def test_what_the_status_word_says(ops):
    assert "more tokens than its arrays" in ops.status_message(0, 5) and "text has no row" in ops.status_message(0, 6)
    assert "without a page" in ops.status_message(0, 1) and ops.status_message(0, 0) is None


# ------------------------------------------------------------------------------------------------ the three together
def drafted_step(runner, arrays, max_context, logit_rows):
    """The StepContext of a step whose arrays were built on the device."""
    from tinyinfer_b200.engine.batch import CacheView, StepContext
    s = arrays.q_starts.shape[0] - 1
    rows = arrays.positions.shape[0]
    step = StepContext(
        num_tokens=rows, num_seqs=s + 1, num_logit_rows=rows, token_ids=arrays.token_ids, positions=arrays.positions,
        token_seq=arrays.token_seq, cu_seqlens=arrays.cu_seqlens, q_starts=arrays.q_starts, context_lens=arrays.context_lens,
        state_slots=torch.zeros(s + 1, dtype=torch.int32, device=dev()), logit_rows=logit_rows,
        block_tables=list(arrays.block_tables), status=runner.buffers.status, max_q_len=128, max_context=max_context,
        num_real_seqs=s, decode_rows=torch.zeros(4, dtype=torch.int32, device=dev()), num_decode=0, prefill_tiles=arrays.tiles,
        num_prefill_tiles=arrays.tiles.shape[0])
    for entry in range(runner.model.spec.num_cache_entries):
        g = runner.manager.group_of_entry[entry]
        step.views[entry] = CacheView(kv=runner.storage.kv[entry], block_table=step.block_tables[g], page_size=runner.manager.page_size,
                                      writes=True, state=None)
    return step


@pytest.mark.parametrize("name,dtype,captured", [("B", "float32", False), ("C", "float32", True), ("C", "bfloat16", True)])
def test_decoding_with_drafts_gives_the_tokens_of_decoding_without(ops, tmp_path, name, dtype, captured):
    """Texts -> ngram_drafts -> step_arrays -> the model -> verify_drafts -> texts, nothing read back between the steps (and, captured,
    nothing launched but a graph): the tokens are those that the engine decodes one by one, greedy and sampled requests alike. In
    bfloat16 the two runs' products differ in order, so the tokens may part at a near tie; there every greedy token has to be within
    rounding of its row's largest logit in the plain model, and the sampled requests are only run."""
    import helpers
    import plain_qwen3
    from tinyinfer_b200 import LLM, SamplingParams
    from tinyinfer_b200.engine.batch import StepEntry
    cfg = helpers.TINY[name]
    folder = helpers.make_model_folder(tmp_path / "m", cfg, seed=3, dtype=dtype, std=0.08)
    page, new, d, longest = 64, 40, 4, 256
    rng = np.random.RandomState(1)
    prompts = [rng.randint(0, cfg["vocab_size"], n).tolist() for n in (5, 70, 33, 1)]
    prompts[1] = (prompts[1][:9] * 8)[:70]               # a prompt that repeats itself
    params = [SamplingParams(greedy=True, max_tokens=new, ignore_eos=True), SamplingParams(greedy=True, max_tokens=new, ignore_eos=True),
              SamplingParams(temperature=0.5, topk=8, seed=77, max_tokens=new, ignore_eos=True),
              SamplingParams(temperature=0.9, topk=0, seed=78, max_tokens=new, ignore_eos=True)]
    make = dict(dtype=dtype, max_num_seqs=4, max_num_batched_tokens=256, kvcache_block_size=page, num_kvcache_blocks=24, max_model_len=longest)
    llm = LLM(folder, **make)
    runner, s = llm.runner, 4
    # prompts but for their last token through the runner; pages for as far as the texts can grow
    for i, p in enumerate(prompts):
        runner.admit(i)
        if len(p) > 1:
            runner.step([StepEntry(i, p[:-1], [])])
        runner.manager.extend(i, len(p) + new + d + 1)
    groups, width = runner.manager.groups, longest // page + 1
    tables = torch.full((len(groups), s, width), -1, dtype=torch.int32)
    for g in range(len(groups)):
        for i in range(s):
            held = runner.manager.get(i).tables[g]
            tables[g, i, :len(held)] = torch.tensor(held, dtype=torch.int32)
    tables = tables.to(dev())
    history = torch.zeros((s, longest), dtype=torch.int32, device=dev())
    for i, p in enumerate(prompts):
        history[i, :len(p)] = ints(p)
    lengths = ints([len(p) for p in prompts])
    first, goal = lengths.clone(), lengths + new
    found, counts = torch.zeros((s, d + 1), dtype=torch.int32, device=dev()), torch.zeros(s, dtype=torch.int32, device=dev())
    # seeds, streams and steps as the engine gives them to its sampler
    fixed = dict(temperature=torch.tensor([1.0, 1.0, 0.5, 0.9], device=dev()), topk=ints([0, 0, 8, 0]), greedy=ints([1, 1, 0, 0]),
                 seed=ints([0, 0, 77, 78], torch.int64), stream_id=ints(STREAMS))
    rows = s * (d + 1) + 3
    logit_rows = torch.arange(rows, dtype=torch.int32, device=dev())
    held_drafts = torch.zeros((), dtype=torch.int64, device=dev())

    def one_step():
        drafts = ops.ngram_drafts(history, lengths, max_drafts=d, max_match=3, tokens=found, counts=counts, status=runner.buffers.status)
        lengths.copy_(drafts.lengths)
        # a text that has reached its goal sits the steps out
        brings = torch.where(drafts.lengths >= goal, torch.zeros_like(drafts.counts), drafts.counts)
        arrays = ops.step_arrays(drafts.starts, brings, tables, rows=rows, max_count=d + 1, page_size=page, tokens=drafts.tokens,
                                 pad_page=runner.storage.dump_page(runner.manager, 0), status=runner.buffers.status)
        logits = runner.model.forward(drafted_step(runner, arrays, longest, logit_rows))
        out = ops.verify_drafts(logits, arrays.token_ids, arrays.cu_seqlens[:s + 1], max_drafts=d, step=drafts.lengths - first, **fixed)
        found.copy_(out.tokens)
        counts.copy_(out.counts)
        held_drafts.add_((out.counts - 1).clamp(min=0).sum())

    one_step()
    graph = None
    if captured:
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            one_step()
    for _ in range(new + 1):
        graph.replay() if captured else one_step()
    torch.cuda.synchronize()
    runner.check_status()
    assert int(held_drafts) > 10                         # the repeating prompt's drafts hold
    texts = [history[i, :first[i] + new].tolist() for i in range(s)]
    assert lengths.min().item() >= 0 and bool((lengths >= goal).all())
    for i in range(s):
        runner.release(i)
    del graph
    fresh = LLM(folder, **make)
    want = fresh.generate(prompts, params)
    if dtype == "float32":
        for i in range(s):
            assert texts[i][len(prompts[i]):] == want[i]["token_ids"], i
    else:
        pcfg, w = plain_qwen3.read_model_folder(folder, torch.float64)
        for i in range(2):
            logits = plain_qwen3.forward(pcfg, w, texts[i]).numpy()
            for k in range(len(prompts[i]), len(texts[i])):
                row = logits[k - 1]
                assert row.max() - row[texts[i][k]] <= 3e-2 * np.abs(logits).max(), (i, k)


STREAMS = [0, 1, 2, 3]
