"""Verification of drafts where the logits lie far from 0: masks of a large negative number, which float32 still divides by the
temperature, rows that lie there as a whole, and temperatures near 0."""
import math

import numpy as np
import pytest
import torch

import plain_drafts as plain

pytestmark = pytest.mark.gpu
NAMES = ("temperature", "topk", "greedy", "seed", "stream_id", "step")


def dev():
    return torch.device("cuda:0")


@pytest.fixture(scope="module")
def ops():
    from tinyinfer_b200 import ops
    return ops


def ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=dev())


def options(temperature, topk, seed):
    s = len(temperature)
    g = torch.Generator().manual_seed(seed)
    return dict(temperature=torch.tensor(temperature, dtype=torch.float32, device=dev()), topk=ints(topk), greedy=ints([0] * s),
                seed=torch.randint(0, 1 << 60, (s,), generator=g).to(dev()),
                stream_id=torch.randint(0, 1 << 30, (s,), generator=g).to(torch.int32).to(dev()),
                step=torch.randint(0, 100000, (s,), generator=g).to(torch.int32).to(dev()))


def sizes(row, temperature, topk):
    """How large the scaled logits are that have weight (they lie within 110 of the largest), and whether they differ."""
    s = plain.scaled(row, temperature, topk)
    near = s[s >= s.max() - 110.0] if s.max() > -math.inf else s[:0]
    near = near[np.isfinite(near)]
    return (float(np.abs(near).max()), bool((near != near[0]).any())) if near.size else (0.0, False)


def tolerances(rows, temperature, topk):
    """(of a probability's ratio, relative; of a draw's lead).
    A row without a threshold weighs its logits by their distance from the largest, up to 110 / ln 2 = 159 in powers of two: the
    difference, the factor (two roundings) and the product are half a step (2^-24) each, the exponential four steps of 2^-24, the sum a
    half step for each addition of a thread and of the tree (vocab / 256 + 16). With a threshold the scaled logits are subtracted, each
    a half step off at its own size, where they differ. A ratio has all that twice, and a division. A score s + G has the quotient's half
    step and the sum's at the size of s, and 2^-19 of G (at most 17, two logarithms of a few steps)."""
    size, extra = 0.0, 0.0
    for row in rows:
        largest, differ = sizes(row, temperature, topk)
        size = max(size, largest)
        if differ and 0 < topk < row.shape[0]:
            extra = max(extra, largest)
    vocab = rows[0].shape[0]
    rel = 2 * 2.0 ** -24 * (4 * 159 * math.log(2) + 4 * extra + 8 + vocab / 256 + 16) + 2.0 ** -23
    return rel, 2 * (2 * 2.0 ** -24 * size + 2.0 ** -19)


def leftover_is_decided(row, dl, rel, temperature, topk, seed, stream, step):
    """Whether float32 can tell which token the draw behind a failed draft gives. What is left of p beyond q is a difference: it is known
    to rel (p + q) and to 2^-126, below which a probability is nothing. (Where p and q are 1 but for 1e-66 the formula has tokens left
    of which float32 has none, and p itself is drawn from.)"""
    p, q = (plain.probabilities(plain.scaled(v, temperature, topk)) for v in (row, dl))
    left, off = np.maximum(p - q, 0.0), rel * (p + q) + 2.0 ** -126
    race = -np.log(-np.log(plain.uniforms(row.shape[0], step, stream, 2, seed)))
    with np.errstate(divide="ignore"):
        least, most = np.log(np.maximum(left - off, 0.0)) + race, np.log(left + off) + race
    winner = int(np.argmax(np.log(left + 1e-300) + race))
    return least[winner] > np.delete(most, winner).max(initial=-math.inf)


def check(ops, x, fed, opts, q=None, allowed=None):
    """x [S, 2, V]: a draft each. The operator beside the plain statement in 64 bits; returns how many requests' tokens were compared
    (where two scores lie closer than float32 tells apart, they are not)."""
    s, _, vocab = x.shape
    got = ops.verify_drafts(x.reshape(2 * s, vocab), ints(fed).flatten(), ints(range(0, 2 * s + 1, 2)), max_drafts=1, draft_logits=q, **opts)
    tokens, counts, accept = got.tokens.tolist(), got.counts.tolist(), got.accept.cpu().double().numpy()
    assert np.isfinite(accept).all() and (accept >= 0).all()
    host, compared = {n: t.tolist() for n, t in opts.items()}, 0
    for r in range(s):
        rows = x[r].cpu().numpy()
        dl = None if q is None else q[r].cpu().numpy()
        t, k = host["temperature"][r], host["topk"][r]
        want, acc, margin = plain.verify(rows, fed[r], max_drafts=1, draft_logits=dl, temperature=t, topk=k, greedy=False,
                                         seed=host["seed"][r], stream=host["stream_id"][r], step=host["step"][r])
        rel, lead = tolerances(list(rows) + ([] if dl is None else list(dl)), t, k)
        assert abs(accept[r, 0] - acc[0]) <= rel * acc[0] + 1e-37, (r, t, k, accept[r, 0], acc[0])
        assert 1 <= counts[r] <= 2 and all(0 <= i < vocab for i in tokens[r][:counts[r]]) and tokens[r][counts[r]:] == [-1] * (2 - counts[r])
        if allowed is not None and allowed[r] is not None:
            assert all(i in allowed[r] for i in tokens[r][:counts[r]]), (r, t, k, tokens[r])
        decided = margin > 2 * rel + lead
        if decided and dl is not None and len(want) == 1:
            decided = leftover_is_decided(rows[0], dl[0], rel, t, k, host["seed"][r], host["stream_id"][r], host["step"][r])
        if decided:
            compared += 1
            assert tokens[r][:counts[r]] == want, (r, t, k, tokens[r], want, margin)
    return compared


TEMPERATURES = [0.3, 0.45, 0.6, 0.7, 0.9, 1.0, 1.3, 1.5]


@pytest.mark.parametrize("mask", [-1e4, -1e9, -1e10, -1e15, -1e20, -1e30, -1e38])
@pytest.mark.parametrize("topk", [0, 20])
def test_rows_masked_by_a_large_negative_number(ops, mask, topk):
    """A few tokens allowed, side by side or far apart, half of the vocabulary, all but one; looked-up drafts and drawn ones, against draft
    logits under the same mask and without; drafts that the mask forbids never hold."""
    vocab = 20011
    g = torch.Generator().manual_seed(5)
    some = [[40, 41, 42], [3, 9000, 20010], list(range(10000)), [i for i in range(vocab) if i != 77]]
    temperature = TEMPERATURES * len(some)
    s = len(temperature)
    x, allowed, fed = torch.full((s, 2, vocab), mask), [], []
    for r in range(s):
        own = some[r // len(TEMPERATURES)]
        x[r][:, own] = 3.0 * torch.randn(2, len(own), generator=g)
        allowed.append(set(own))
        likely = own[int(x[r, 0, own].argmax())]
        fed.append([1, 77 if r % 3 == 0 else likely])    # (77 is forbidden by all masks but the third)
    x = x.to(dev())
    opts = options(temperature, [topk] * s, seed=int(-math.log10(-mask)) + 60)
    open_q = (2.0 * torch.randn(s, 1, vocab, generator=g)).to(dev())
    like_q = torch.where(x[:, :1] == mask, x[:, :1], x[:, :1] + 0.7 * torch.randn(s, 1, vocab, generator=g).to(dev()))
    for q in (None, open_q, like_q):
        assert check(ops, x, fed, opts, q, allowed) >= s // 2
    # every request's draft forbidden: none holds, and none is written
    forbidden = [[1, next(i for i in range(vocab) if i not in a)] for a in allowed]
    for q in (None, open_q):
        check(ops, x, forbidden, opts, q, allowed)


@pytest.mark.parametrize("mask", [-1e4, -1e9, -1e10, -1e15, -1e20, -1e30, -1e38])
@pytest.mark.parametrize("topk", [0, 20])
def test_rows_that_lie_at_the_mask_as_a_whole(ops, mask, topk):
    """Every token alike: a probability of 1 / V each; what is drawn is what sample draws."""
    vocab, s = 9001, len(TEMPERATURES)
    x = torch.full((s, 2, vocab), mask, device=dev())
    opts = options(TEMPERATURES, [topk] * s, seed=7)
    drawn = ops.sample(x[:, 0].contiguous(), *(opts[n] for n in NAMES)).tolist()
    fed = [[1, drawn[r] if r % 2 else (drawn[r] + 1) % vocab] for r in range(s)]
    check(ops, x, fed, opts)
    got = ops.verify_drafts(x.view(2 * s, vocab), ints(fed).flatten(), ints(range(0, 2 * s + 1, 2)), max_drafts=1, **opts)
    assert got.tokens[:, 0].tolist() == drawn and got.counts.tolist() == [1 + r % 2 for r in range(s)]
    check(ops, x, fed, opts, x[:, :1])                   # the same logits: every draft holds
    check(ops, x, fed, opts, torch.randn(s, 1, vocab, generator=torch.Generator().manual_seed(3)).to(dev()))


COLD = [1e-2, 1e-3, 1e-4, 1e-5, 1e-6, 1e-7, 1e-8, 1e-10, 1e-15, 1e-20, 1e-25, 1e-29, 1e-31]


@pytest.mark.parametrize("shift", [0.0, 30.0, -1000.0])
@pytest.mark.parametrize("topk", [0, 20])
def test_temperatures_near_0(ops, shift, topk):
    """The largest logit has all the weight, or shares it with its equals."""
    vocab, s = 20011, len(COLD)
    g = torch.Generator().manual_seed(9)
    x = shift + 3.0 * torch.randn(s, 2, vocab, generator=g)
    best = x[:, 0].argmax(1).tolist()
    fed = [[1, best[r] if r % 4 else (best[r] + 5) % vocab] for r in range(s)]
    x[2::3, 0, 19000:19003] = x[2::3, 0].amax(1)[:, None]           # of several equals each has its share
    x = x.to(dev())
    opts = options(COLD, [topk] * s, seed=11)
    # (a draw among equals whose noise is lost beside s is left to the comparison with sample)
    assert check(ops, x, fed, opts) >= s // 3
    for q in (x[:, :1], x[:, :1] + 0.5 * torch.randn(s, 1, vocab, generator=g).to(dev())):
        check(ops, x, fed, opts, q)


@pytest.mark.parametrize("vocab", [600, 40007])
@pytest.mark.parametrize("topk", [0, 7, 300])
def test_rows_whose_quotients_are_all_infinite(ops, vocab, topk):
    """The type's lowest value over a temperature below 1 is -inf: such a row has nothing, as one of -inf has. No draft holds, not the
    first finite logit's either, and the token is the one that sample gives. At a temperature of 1 or more all tokens are alike."""
    temperature = [0.3, 0.5, 0.7, 0.99, 1.0, 1.3]
    s = len(temperature)
    x = torch.full((s, 2, vocab), torch.finfo(torch.float32).min, device=dev())
    x[:, :, :5] = float("-inf")
    opts = options(temperature, [topk] * s, seed=21)
    other = torch.randn(s, 1, vocab, generator=torch.Generator().manual_seed(4)).to(dev())
    first = ops.sample(x[:, 0].contiguous(), *(opts[n] for n in NAMES)).tolist()
    for draft in (5, 6, 0, vocab - 1):
        fed = [[1, draft]] * s
        for q in (None, other, x[:, :1]):
            check(ops, x, fed, opts, q)
            got = ops.verify_drafts(x.reshape(2 * s, vocab), ints(fed).flatten(), ints(range(0, 2 * s + 1, 2)), max_drafts=1,
                                    draft_logits=q, **opts)
            assert got.tokens[:4].tolist() == [[0, -1]] * 4 and got.counts[:4].tolist() == [1] * 4 and not got.accept[:4].any()
            if q is None:
                assert got.tokens[:, 0].tolist() == first
    # the target has something, the draft model's row nothing: what p gives anything holds
    check(ops, other.expand(s, 2, vocab).contiguous(), [[1, int(other[r, 0].argmax())] for r in range(s)], opts, x[:, :1])


@pytest.mark.parametrize("scale", [1e-4, 1.0, 1e6])
@pytest.mark.parametrize("topk", [0, 50])
def test_quotients_that_rounding_makes_equal(ops, scale, topk):
    """Logits a step of float32 apart over temperatures near 0: their quotients differ by less than a rounding, so some are equal, the
    noise of others is lost beside them, and of equal scores the first wins. The token is the one that sample gives, drafts of it hold,
    also behind drafts that are sure to hold against the same draft logits."""
    vocab, temperature = 5003, [10.0 ** -e for e in range(3, 28)] * 2
    s = len(temperature)
    g = torch.Generator().manual_seed(31)
    top = (20.0 + 4.0 * torch.rand(s, 2, 1, generator=g)) * scale * torch.where(torch.rand(s, 2, 1, generator=g) < 0.3, -1.0, 1.0)
    steps = torch.randint(0, 9, (s, 2, vocab), generator=g, dtype=torch.int32)
    x = (top.view(torch.int32) - steps * torch.sign(top).int()).view(torch.float32)
    x[:, :, ::3] -= 5.0 * scale
    x = x.to(dev())
    opts = options(temperature, [topk] * s, seed=32)
    rows = [x[:, j].contiguous() for j in range(2)]
    first = ops.sample(rows[0], *(opts[n] for n in NAMES))
    second = ops.sample(rows[1], *(opts["step"] + 1 if n == "step" else opts[n] for n in NAMES))
    fed = torch.stack((first, first), 1).flatten()
    cu = ints(range(0, 2 * s + 1, 2))
    got = ops.verify_drafts(x.reshape(2 * s, vocab), fed, cu, max_drafts=1, **opts)
    assert got.tokens[:, 0].tolist() == first.tolist() and got.counts.tolist() == [2] * s
    assert got.tokens[:, 1].tolist() == second.tolist()
    sure = ops.argmax(rows[0])                           # p = q there: it holds
    got = ops.verify_drafts(x.reshape(2 * s, vocab), torch.stack((sure, sure), 1).flatten(), cu, max_drafts=1, draft_logits=x[:, :1], **opts)
    assert got.counts.tolist() == [2] * s and got.tokens[:, 1].tolist() == second.tolist()


@pytest.mark.parametrize("topk", [0, 20])
@pytest.mark.parametrize("temperature", [1e30, 3e38, math.inf])
def test_temperatures_that_make_all_tokens_alike(ops, temperature, topk):
    vocab, s = 9001, 6
    g = torch.Generator().manual_seed(41)
    x = torch.randn(s, 2, vocab, generator=g).to(dev())
    opts = options([temperature] * s, [topk] * s, seed=42)
    drawn = ops.sample(x[:, 0].contiguous(), *(opts[n] for n in NAMES)).tolist()
    fed = [[1, drawn[r] if r % 2 else (drawn[r] + 1) % vocab] for r in range(s)]
    for q in (None, x[:, 1:], 30.0 * x[:, 1:]):
        check(ops, x, fed, opts, q)
    if topk and temperature == math.inf:                 # quotients of 0 and -0: equal here, as s >= k-th largest has it, not in sample
        return
    got = ops.verify_drafts(x.view(2 * s, vocab), ints(fed).flatten(), ints(range(0, 2 * s + 1, 2)), max_drafts=1, **opts)
    assert got.tokens[:, 0].tolist() == drawn and got.counts.tolist() == [1 + r % 2 for r in range(s)]


@pytest.mark.parametrize("vocab", [700, 30011])
def test_zeros_of_either_sign_at_the_threshold(ops, vocab):
    """s >= the k-th largest keeps -0 where that is +0: the draws and the shares are those of all zeros, many more than k."""
    s, k = 8, 5
    x = torch.full((s, 2, vocab), -1.0)
    x[:, :, :200:2], x[:, :, 1:200:2] = 0.0, -0.0
    x[:, :, 300] = 1.0
    x = x.to(dev())
    opts = options([0.5, 1.0] * 4, [k] * s, seed=51)
    other = torch.randn(s, 1, vocab, generator=torch.Generator().manual_seed(52)).to(dev())
    for draft in (0, 1, 300, 500):
        for q in (None, other):
            assert check(ops, x, [[1, draft]] * s, opts, q) >= s // 2
        check(ops, x, [[1, draft]] * s, opts, x[:, 1:])  # (p = q: nothing is left beyond it, which float32 cannot tell from next to nothing)


@pytest.mark.parametrize("size", [1.04e6, 1.05e6, 5e7, 5.36e8, 5.38e8, 1.08e9, 3e12])
def test_where_the_noise_fades(ops, size):
    """Scaled logits from where a step of float32 is a sixteenth to where it is past all noise, of either sign, in two to nine neighbouring
    values of float32, some tiles nothing but the lower ones: the tokens are sample's."""
    vocab, s = 30011, 8
    g = torch.Generator().manual_seed(61)
    top = torch.tensor([-size, size] * (s // 2)).view(s, 1, 1).expand(s, 2, 1).contiguous()
    steps = torch.randint(0, 9, (s, 2, vocab), generator=g, dtype=torch.int32)
    steps[2:4] = steps[2:4].clamp(max=1)
    steps[:, :, :20000] += 3
    x = (top.view(torch.int32) - steps * torch.sign(top).int()).view(torch.float32).to(dev())
    opts = options([1.0, 1.0, 1.0, 1.0, 0.9, 0.9, 1.4, 1.4], [0] * s, seed=62)
    rows = [x[:, j].contiguous() for j in range(2)]
    first = ops.sample(rows[0], *(opts[n] for n in NAMES))
    second = ops.sample(rows[1], *(opts["step"] + 1 if n == "step" else opts[n] for n in NAMES))
    got = ops.verify_drafts(x.reshape(2 * s, vocab), torch.stack((first, first), 1).flatten(), ints(range(0, 2 * s + 1, 2)), max_drafts=1, **opts)
    assert got.tokens[:, 0].tolist() == first.tolist() and got.tokens[:, 1].tolist() == second.tolist() and got.counts.tolist() == [2] * s


@pytest.mark.parametrize("off", [0.0, 9e5, 3e6, -1.2e7])
@pytest.mark.parametrize("topk", [0, 8])
@pytest.mark.parametrize("which", [11, 17, 29])
def test_tokens_are_distributed_as_the_target_says_far_from_0(ops, off, topk, which):
    """40,000 requests with a draft each, drawn from q: the first tokens' frequencies are p's, whatever the roundings at the size of the
    logits, which is the draft model's, too. With a threshold p and q are the softmax of the float32 quotients, without one of x / T. A
    frequency is off by more than five standard deviations once in two million."""
    v, n, t = 12, 40000, np.float32(0.9)
    g = torch.Generator().manual_seed(which)
    target, other = torch.randn(v, generator=g) * 1.5 + off, torch.randn(v, generator=g) * 1.5 + off

    def softmax(x):
        s = (x.numpy() / t).astype(np.float64) if topk else x.double().numpy() / float(t)
        s[x.numpy() / t < np.sort(x.numpy() / t)[-(topk or v)]] = -math.inf
        w = np.exp(s - s.max())
        return w / w.sum()

    p, q = softmax(target), softmax(other)
    opts = options([float(t)] * n, [topk] * n, seed=6)
    opts["seed"] = torch.full((n,), 1234, dtype=torch.int64, device=dev())
    opts["stream_id"] = torch.arange(n, dtype=torch.int32, device=dev())
    draft = torch.multinomial(torch.tensor(q), n, True, generator=g).int().to(dev())
    fed = torch.stack((torch.zeros_like(draft), draft), 1).flatten().contiguous()
    got = ops.verify_drafts(target.to(dev()).expand(2 * n, v).contiguous(), fed, torch.arange(0, 2 * n + 1, 2, dtype=torch.int32, device=dev()),
                            max_drafts=1, draft_logits=other.to(dev()).expand(n, 1, v), **opts)
    freq = np.bincount(got.tokens[:, 0].cpu().numpy(), minlength=v) / n
    assert np.all(np.abs(freq - p) <= 5.0 * np.sqrt(p * (1 - p) / n) + 1e-9), (freq, p)
