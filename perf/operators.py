"""Timed cases of decoding with drafts: ``ops.verify_drafts``, ``ops.ngram_drafts`` and ``ops.step_arrays``, each beside its
plain form in elementary torch operations.

* ``verify``: ``requests`` requests bring up to ``drafts`` drafted tokens each and rows of logits over ``vocab`` tokens. Which
  drafts hold, and the token that follows them, by the request's temperature, top-k threshold and random stream. ``kind``:
  ``greedy``, ``sampled``, or ``mixed`` (of four requests one is greedy, one has no top-k threshold). ``draft_logits``: the drafts
  were drawn by a model whose logits are there too, and hold by the ratio of the probabilities; otherwise they come from a lookup,
  and hold where they are what the stream draws.
* ``ngram``: ``requests`` requests with texts of up to ``context`` tokens take up to ``drafts`` + 1 verified tokens in and get
  drafts that followed the latest longest match (at most ``match`` tokens) of their last tokens.
* ``arrays``: positions, owners, slots, attention tiles and block tables of a step to which ``requests`` requests bring up to
  ``count`` tokens each, behind up to ``context`` stored ones, in pages of ``page`` tokens and ``groups`` groups of cache entries.

``ragged`` spreads a case's numbers of drafts, lengths or tokens over their range; otherwise every request has the largest.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False
DEVICE = "cuda:0"
TILE = 128                # query rows of an attention tile
_MASK = 0xFFFFFFFF


def _verify(name, requests, drafts, vocab, kind, topk=0, temperature=1.0, draft_logits=False, ragged=False):
    return dict(name=name, op="verify", requests=requests, drafts=drafts, vocab=vocab, kind=kind, topk=topk,
                temperature=temperature, draft_logits=draft_logits, ragged=ragged)


def _ngram(name, requests, context, drafts, match, ragged=False):
    return dict(name=name, op="ngram", requests=requests, context=context, drafts=drafts, match=match, ragged=ragged)


def _arrays(name, requests, count, context, page, groups, ragged=False):
    return dict(name=name, op="arrays", requests=requests, count=count, context=context, page=page, groups=groups, ragged=ragged)


def listed():
    return [
        # one interactive request, four drafts, greedy: what it adds to a step is pure latency
        _verify("verify 1x4 greedy", 1, 4, 151936, "greedy"),
        # a small batch with looked-up drafts and the sampler's default threshold
        _verify("verify 8x5 lookup top-k 100", 8, 5, 151936, "sampled", 100, 0.8, ragged=True),
        # a vocabulary whose rows start off 16-byte boundaries
        _verify("verify 13x3 odd vocabulary", 13, 3, 32003, "mixed", 50, 0.7, draft_logits=True, ragged=True),
        # a serving batch with a draft model: greedy, thresholded and open requests side by side
        _verify("verify 32x4 mixed", 32, 4, 102400, "mixed", 100, 1.0, draft_logits=True),
        # the same where every request has the sampler's default threshold
        _verify("verify 64x4 top-k 100", 64, 4, 151936, "sampled", 100, 1.0, draft_logits=True),
        # the largest: every request samples from the whole vocabulary
        _verify("verify 64x7 open", 64, 7, 151936, "sampled", 0, 1.0, draft_logits=True),
        # lookups: a chat turn, a serving batch of documents, a large batch of long documents
        _ngram("ngram 1 x 2k", 1, 2048, 4, 3),
        _ngram("ngram 64 x 32k", 64, 32768, 5, 4, ragged=True),
        _ngram("ngram 256 x 128k", 256, 131071, 8, 3),
        # drafted steps: a small batch; a large one in small pages; portions of prompts in two groups of cache entries
        _arrays("arrays 8 x 5", 8, 5, 4096, 64, 1, ragged=True),
        _arrays("arrays 512 x 9 at 40k", 512, 9, 40960, 16, 1, ragged=True),
        _arrays("arrays 64 portions", 64, 1021, 32768, 64, 2, ragged=True),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _unnamed(case):
    del case["name"]
    return case


def draw(rng):
    op = rng.choice(("verify", "verify", "verify", "ngram", "arrays"))
    if op == "verify":
        kind = rng.choice(("greedy", "sampled", "sampled", "mixed"))
        topk = 0 if kind == "greedy" else rng.choice((0, _log_int(rng, 1, 256), _log_int(rng, 1, 256)))
        vocab, drafts = _log_int(rng, 500, 160000), rng.randint(1, 8)
        logits = kind != "greedy" and rng.random() < 0.6
        most = max(1, 64 * 15 * 151936 // (vocab * (2 * drafts + 1)))
        return _unnamed(_verify("", _log_int(rng, 1, min(256, most)), drafts, vocab, kind, topk, round(rng.uniform(0.3, 1.5), 2), logits,
                                rng.random() < 0.5))
    if op == "ngram":
        requests = _log_int(rng, 1, 256)
        return _unnamed(_ngram("", requests, _log_int(rng, 2, 131071), rng.randint(1, 8), rng.randint(1, 6), rng.random() < 0.7))
    count = rng.choice((rng.randint(1, 9), _log_int(rng, 1, 1021)))
    return _unnamed(_arrays("", _log_int(rng, 1, 512 if count < 10 else 64), count, _log_int(rng, 16, 40960), rng.choice((16, 32, 64, 256)),
                            rng.randint(1, 3), rng.random() < 0.7))


def _spread(case, least, most):
    """A number per request between ``least`` and ``most``, the same for every seed: a step's sizes are known to its caller."""
    n = case["requests"]
    if not case["ragged"]:
        return [most] * n
    return [least + (most - least) * ((i * 7 + 3) % 11) // 10 for i in range(n)]


def _kinds(case):
    """Per request: greedy, top-k threshold (0: none)."""
    kind, k = case["kind"], case["topk"]
    if kind == "mixed":
        return [int(i % 4 == 0) for i in range(case["requests"])], [0 if i % 4 == 1 else k for i in range(case["requests"])]
    return [int(kind == "greedy")] * case["requests"], [k] * case["requests"]


# ------------------------------------------------------------------------------------------------ inputs
def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=DEVICE)


def _prepare_verify(case, gen):
    s, d, v = case["requests"], case["drafts"], case["vocab"]
    drafts = _spread(case, 0, d)
    greedy, topk = _kinds(case)
    owner = [r for r in range(s) for _ in range(drafts[r] + 1)]
    place = [j for r in range(s) for j in range(drafts[r] + 1)]
    cu = [0]
    for n in drafts:
        cu.append(cu[-1] + n + 1)
    rows = cu[-1]
    # logits as trained models give them: a broad body and one token that stands out more or less
    logits = torch.empty((rows, v), device=DEVICE).normal_(0.0, 2.0, generator=gen)
    likely = torch.randint(0, v, (rows,), device=DEVICE, generator=gen)
    lift = torch.empty((rows,), device=DEVICE).uniform_(4.0, 16.0, generator=gen)
    logits[torch.arange(rows, device=DEVICE), likely] += lift
    temperature = torch.full((s,), float(case["temperature"]), device=DEVICE)
    owner_t, place_t = _ints(owner, torch.int64), _ints(place, torch.int64)
    behind = torch.nonzero(place_t > 0).flatten()                    # rows that were fed a drafted token
    before = behind - 1                                              # the rows whose next token it is
    token_ids = torch.randint(0, v, (rows,), device=DEVICE, generator=gen).to(torch.int32)
    state = dict(op="verify", logits=logits, drafts=d, vocab=v, kmax=case["topk"], all_greedy=all(greedy), owner=owner_t, place=place_t, before=before,
                 cu_rows=_ints(cu), temperature=temperature, topk=_ints(topk), greedy=_ints(greedy),
                 seed=torch.randint(0, 1 << 62, (s,), device=DEVICE, generator=gen),
                 stream_id=torch.arange(s, dtype=torch.int32, device=DEVICE) * 3 + 5,
                 step=torch.randint(0, 4096, (s,), device=DEVICE, generator=gen).to(torch.int32), draft_logits=None)
    if case["draft_logits"]:
        # a draft model near the target, and drafts drawn from it
        dl = torch.zeros((d, s, v), device=DEVICE).transpose(0, 1)   # laid out draft by draft, as a draft model's steps leave it
        noisy = logits[before] + torch.empty((len(before), v), device=DEVICE).normal_(0.0, 0.8, generator=gen)
        dl[owner_t[before], place_t[before]] = noisy
        scaled = noisy / temperature[owner_t[before]][:, None]
        if case["topk"]:
            limit = scaled.topk(min(v, case["topk"]), dim=1).values[:, -1:]
            limited = (_ints(topk)[owner_t[before]] > 0)[:, None]
            scaled = scaled.masked_fill(limited & (scaled < limit), -math.inf)
        noise = -torch.log(torch.empty_like(scaled).exponential_(1.0, generator=gen))
        token_ids[behind] = (scaled + noise).argmax(1).to(torch.int32)
        state["draft_logits"] = dl
    else:
        right = torch.empty((len(before),), device=DEVICE).uniform_(0.0, 1.0, generator=gen) < 0.75
        token_ids[behind] = torch.where(right, likely[before], token_ids[behind].long()).to(torch.int32)
    state["token_ids"] = token_ids
    return state


def _prepare_ngram(case, gen):
    s, d = case["requests"], case["drafts"]
    lengths = _spread(case, max(1, case["context"] // 4), case["context"])
    room = case["context"] + d + 1
    counts = [1 + (5 * i) % (d + 1) for i in range(s)]
    history = torch.randint(0, 4000, (s, room), device=DEVICE, generator=gen).to(torch.int32)
    tokens = torch.randint(0, 4000, (s, d + 1), device=DEVICE, generator=gen).to(torch.int32)
    # half of the texts have said their last tokens before, as code and quoting answers do
    for i in range(0, s, 2):
        tail = torch.cat((history[i, :lengths[i]], tokens[i, :counts[i]]))[-case["match"]:]
        at = int((lengths[i] - len(tail)) * (0.1 + 0.8 * ((i * 13) % 17) / 17))
        if at >= 0:
            history[i, at:at + len(tail)] = tail
    return dict(op="ngram", history=history, lengths=_ints(lengths), tokens=tokens, counts=_ints(counts), drafts=d,
                match=case["match"])


def _prepare_arrays(case, gen):
    s, c, page, g = case["requests"], case["count"], case["page"], case["groups"]
    counts = _spread(case, 0, c)
    starts = list(reversed(_spread(case, 0, case["context"])))
    width = -(-(case["context"] + c) // page)
    slots = s + 3
    order = torch.randperm(slots, device=DEVICE, generator=gen)[:s].to(torch.int32)
    tables = torch.randint(0, 1 << 20, (g, slots, width), device=DEVICE, generator=gen).to(torch.int32)
    tokens = torch.randint(0, 150000, (s, c), device=DEVICE, generator=gen).to(torch.int32)
    return dict(op="arrays", starts=_ints(starts), counts=_ints(counts), tokens=tokens, tables=tables, state_slots=order,
                rows=sum(counts) + 5, page=page, count=c, pad_page=1 << 20)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(int(seed))
    return {"verify": _prepare_verify, "ngram": _prepare_ngram, "arrays": _prepare_arrays}[case["op"]](case, gen)


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    if own:
        return _run_own(state)
    return {"verify": _plain_verify, "ngram": _plain_ngram, "arrays": _plain_arrays}[state["op"]](state)


def _run_own(st):
    from tinyinfer_b200 import ops
    if st["op"] == "verify":
        sampling = {} if st["all_greedy"] else {name: st[name] for name in ("temperature", "topk", "greedy", "seed", "stream_id", "step",
                                                                            "draft_logits")}
        out = ops.verify_drafts(st["logits"], st["token_ids"], st["cu_rows"], max_drafts=st["drafts"], **sampling)
        return dict(tokens=out.tokens, counts=out.counts, accept=out.accept)
    if st["op"] == "ngram":
        out = ops.ngram_drafts(st["history"], st["lengths"], max_drafts=st["drafts"], max_match=st["match"], tokens=st["tokens"],
                               counts=st["counts"])
        return dict(tokens=out.tokens, counts=out.counts, starts=out.starts, lengths=out.lengths, history=st["history"])
    out = ops.step_arrays(st["starts"], st["counts"], st["tables"], rows=st["rows"], max_count=st["count"], page_size=st["page"],
                          tokens=st["tokens"], state_slots=st["state_slots"], pad_page=st["pad_page"])
    return dict(token_ids=out.token_ids, positions=out.positions, token_seq=out.token_seq, cache_slots=out.cache_slots,
                cu_seqlens=out.cu_seqlens, q_starts=out.q_starts, context_lens=out.context_lens, tiles=out.tiles,
                block_tables=out.block_tables)


def _philox(c0, c1, c2, c3, key):
    """Philox-4x32-10 (Salmon et al., 2011) of int64 tensors that hold 32-bit words: the four words of each block. A product of
    two words wraps around in 64 bits, which leaves all its bits where they belong."""
    even, odd = torch.stack((c0, c2)), torch.stack((c1, c3))
    shape = (2,) + (1,) * c0.dim()
    factors = torch.tensor((0xD2511F53, 0xCD9E8D57), device=key.device).view(shape)
    bump = torch.tensor((0x9E3779B9, 0xBB67AE85), device=key.device).view(shape)
    keys = torch.stack((key & _MASK, (key >> 32) & _MASK))
    for r in range(10):
        product = even * factors
        even, odd = (((product >> 32) & _MASK).flip(0)) ^ odd ^ ((keys + r * bump) & _MASK), (product & _MASK).flip(0)
    return even[0], odd[0], even[1], odd[1]


def _uniform(word):                          # in (0, 1), exact in 32 bits
    return ((word >> 9).to(torch.float32) + 0.5) * (1.0 / 8388608.0)


def _noise_words(v, seed, step, stream, domain):
    """Row by row a word per token; seed, step, stream and domain are columns."""
    blocks = torch.arange((v + 3) // 4, device=seed.device)[None, :]
    words = _philox(*torch.broadcast_tensors(blocks, step, stream, domain), seed)
    return torch.stack(words, dim=2).reshape(seed.shape[0], -1)[:, :v]


def _noisy(s, seed, step, stream):
    """Scaled logits with the Gumbel noise of their row's stream."""
    words = _noise_words(s.shape[1], seed, step, stream, torch.zeros_like(step))
    return s - torch.log(-torch.log(_uniform(words)))


def _scaled(x, temperature, topk, kmax):
    """Rows over their temperature, what the threshold drops and what is no number at -inf."""
    s = x / temperature[:, None]
    s = torch.where(torch.isnan(s), -math.inf, s)
    v = s.shape[1]
    if 0 < kmax < v:
        limit = torch.topk(s, kmax, dim=1).values[:, -1:]
        limited = ((topk > 0) & (topk < v))[:, None]
        s = torch.where(limited & (s < limit), -math.inf, s)
    return s


def _weights(s):
    """exp(s - max) of every row and their sum in 64 bits."""
    m = s.amax(1, keepdim=True)
    w = torch.where(s == m, 1.0, torch.exp(s - m))
    w = torch.where(s == -math.inf, 0.0, w)
    return w, w.sum(1, dtype=torch.float64)


def _emitted(st, cu, held, drawn):
    """The drafts that held, then the token drawn behind them, then -1."""
    jj = torch.arange(st["drafts"] + 1, device=cu.device)[None, :]
    fed = st["token_ids"][(cu[:-1, None] + 1 + jj).clamp(max=st["token_ids"].shape[0] - 1)]
    return torch.where(jj < held[:, None], fed, torch.where(jj == held[:, None], drawn[:, None].int(), -1))


def _plain_greedy(st):
    cu, before = st["cu_rows"].long(), st["before"]
    best = st["logits"].argmax(1)
    accept = torch.zeros((cu.shape[0] - 1, st["drafts"]), device=cu.device)
    accept[st["owner"][before], st["place"][before]] = (st["token_ids"][before + 1] == best[before]).float()
    held = accept.int().cumprod(1).sum(1)
    return dict(tokens=_emitted(st, cu, held, best[cu[:-1] + held]), counts=(held + 1).int(), accept=accept)


def _plain_verify(st):
    if st["all_greedy"]:
        return _plain_greedy(st)
    logits, cu = st["logits"], st["cu_rows"].long()
    owner, place, before = st["owner"], st["place"], st["before"]
    d, v, n_req = st["drafts"], st["vocab"], cu.shape[0] - 1
    greedy, topk = st["greedy"] > 0, st["topk"]
    s = _scaled(logits, st["temperature"][owner], topk[owner], st["kmax"])
    w, z = _weights(s)
    best = logits.argmax(1)
    # how likely each draft is to hold
    drafted = st["token_ids"][before + 1].long()
    p = w[before, drafted].double() / z[before]
    q = torch.ones_like(p)
    if st["draft_logits"] is not None:
        dl = st["draft_logits"][owner[before], place[before]]
        dw, dz = _weights(_scaled(dl, st["temperature"][owner[before]], topk[owner[before]], st["kmax"]))
        q = dw.gather(1, drafted[:, None])[:, 0].double() / dz
    a = torch.where(q > 0, p / q, (p > 0).double()).clamp(max=1.0)
    a = torch.where(greedy[owner[before]], (drafted == best[before]).double(), a)
    accept = torch.zeros((n_req, d), dtype=torch.float64, device=logits.device)
    accept[owner[before], place[before]] = a
    if st["draft_logits"] is None:
        # what the stream draws for every row
        owner_ = owner[:, None]
        drawn = _noisy(s, st["seed"][owner_], st["step"].long()[owner_] + place[:, None], st["stream_id"].long()[owner_]).argmax(1)
        drawn = torch.where(greedy[owner], best, drawn)
        holds = torch.zeros((n_req, d), dtype=torch.int64, device=logits.device)
        holds[owner[before], place[before]] = (drawn[before] == drafted).long()
        held = holds.cumprod(1).sum(1)
        return dict(tokens=_emitted(st, cu, held, drawn[cu[:-1] + held]), counts=(held + 1).int(), accept=accept.float())
    seed, stream, step = st["seed"][:, None], st["stream_id"].long()[:, None], st["step"].long()[:, None]
    j = torch.arange(d, device=logits.device)[None, :]
    u = _uniform(_philox(torch.zeros_like(step + j), step + j, stream.expand(-1, d), torch.ones_like(step + j), seed.expand(-1, d))[0])
    held = (u < accept).int().cumprod(1).sum(1)
    at = cu[:-1] + held                                              # the row that the next token is drawn from
    rejected = (held < cu[1:] - cu[:-1] - 1)[:, None]
    row_of = torch.zeros((logits.shape[0],), dtype=torch.int64, device=logits.device)
    row_of[before] = torch.arange(len(before), device=logits.device)
    pr = (w[at] / z[at][:, None]).float()
    qr = (dw[row_of[at]] / dz[row_of[at]][:, None]).float() if len(before) else pr
    left = (pr - qr).clamp(min=0.0)
    left = torch.where((left > 0).any(1, keepdim=True), left, pr)
    e = -torch.log(_uniform(_noise_words(v, seed, step + held[:, None], stream, torch.where(rejected, 2, 0))))
    score = torch.where(rejected, torch.where(left > 0, left / e, -math.inf), s[at] - torch.log(e))
    drawn = torch.where(greedy, best[at], score.argmax(1))
    return dict(tokens=_emitted(st, cu, held, drawn), counts=(held + 1).int(), accept=accept.float())


def _plain_ngram(st):
    history, d, m = st["history"], st["drafts"], st["match"]
    s, room = history.shape
    dev = history.device
    at = torch.arange(d + 1, device=dev)[None, :]
    fresh = at < st["counts"][:, None]
    places = (st["lengths"][:, None] + at).long()
    history.scatter_(1, places, torch.where(fresh, st["tokens"], history.gather(1, places)))
    n = (st["lengths"] + st["counts"]).long()[:, None]
    # how many of the last m tokens stand in front of every place e, counted backwards
    padded = torch.nn.functional.pad(history, (m, 0), value=-1)
    last = padded.gather(1, n + torch.arange(m, device=dev)[None, :])
    same = (padded.unfold(1, m, 1) == last[:, None, :]).flip(2)
    length = torch.nn.functional.pad(~same, (0, 1), value=True).to(torch.uint8).argmax(2)      # the first that differs
    e = torch.arange(room + 1, device=dev)[None, :]
    key = torch.where((e >= 1) & (e < n) & (length >= 1), length * (1 << 32) + e, 0).amax(1, keepdim=True)
    found, e = key > 0, key & _MASK
    drafts = history.gather(1, e + (at[:, :d] % (n - e).clamp(min=1)))
    drafts = torch.where(found, drafts, -1)
    newest = history.gather(1, n - 1)
    counts = torch.where(found, d + 1, 1)[:, 0].int()
    return dict(tokens=torch.cat((newest, drafts), 1), counts=counts, starts=(n - 1)[:, 0].int(), lengths=n[:, 0].int(), history=history)


def _plain_arrays(st):
    starts, counts, tables = st["starts"].long(), st["counts"].long(), st["tables"]
    rows, page, s = st["rows"], st["page"], starts.shape[0]
    g, _, width = tables.shape
    dev = starts.device
    zero = torch.zeros(1, dtype=torch.int64, device=dev)
    cu = torch.cat((zero, counts.cumsum(0)))
    t = torch.arange(rows, device=dev)
    seq = torch.searchsorted(cu[1:], t, right=True)                  # s behind the last request
    real = seq < s
    of = seq.clamp(max=s - 1)
    offset = t - cu[of]
    positions = torch.where(real, starts[of] + offset, 0)
    token_ids = torch.where(real, st["tokens"][of, offset.clamp(0, st["count"] - 1)].long(), 0)
    context = starts + counts
    held = (context + page - 1) // page
    j = torch.arange(width, device=dev)
    mine = tables[:, st["state_slots"].long()]
    mine = torch.where(j[None, None, :] < held[None, :, None], mine, -1)
    pad = torch.full((g, 1, width), -1, dtype=torch.int32, device=dev)
    pad[:, :, 0] = st["pad_page"]
    block_tables = torch.cat((mine, pad), 1)
    pages = block_tables[:, of, (positions // page).clamp(max=width - 1)].long()
    slots = torch.where(real[None, :] & (pages >= 0), pages * page + positions % page, -1)
    per = -(-st["count"] // TILE)
    k = torch.arange(per, device=dev)[None, :] * TILE
    left = (counts[:, None] - k).clamp(0, TILE)
    tiles = torch.stack((torch.arange(s, device=dev)[:, None].expand(-1, per), cu[:-1, None] + torch.minimum(k, counts[:, None]), left,
                         starts[:, None] + torch.minimum(k, counts[:, None])), 2).reshape(-1, 4)
    end = torch.full((1,), rows, dtype=torch.int64, device=dev)
    return dict(token_ids=token_ids.int(), positions=positions.int(), token_seq=seq.int(), cache_slots=slots.int(),
                cu_seqlens=torch.cat((cu, end)).int(), q_starts=torch.cat((starts, zero)).int(),
                context_lens=torch.cat((context, zero + 1)).int(), tiles=tiles.int(), block_tables=block_tables)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    s = case["requests"]
    if case["op"] == "verify":
        drafts = _spread(case, 0, case["drafts"])
        greedy, _ = _kinds(case)
        rows = sum(drafts) + s
        drawn = sum(n for n, g in zip(drafts, greedy) if not g) if case["draft_logits"] else 0
        elements = (rows + drawn) * case["vocab"]
        return dict(bytes=4.0 * elements + 4 * rows + s * (32 + 4 * (2 * case["drafts"] + 2)), flops=4.0 * elements)
    if case["op"] == "ngram":
        tokens = sum(_spread(case, max(1, case["context"] // 4), case["context"])) + s
        return dict(bytes=4.0 * tokens + 4 * s * (3 * case["drafts"] + 8), flops=float(tokens))
    counts, starts = _spread(case, 0, case["count"]), list(reversed(_spread(case, 0, case["context"])))
    rows, page, g = sum(counts) + 5, case["page"], case["groups"]
    width = -(-(case["context"] + case["count"]) // page)
    held = sum(-(-(a + b) // page) for a, b in zip(starts, counts))
    words = g * (held + (s + 1) * width + rows) + 3 * rows + sum(counts) + 4 * s * -(-case["count"] // TILE) + 6 * s
    return dict(bytes=4.0 * words, flops=float(words))


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits
def _words64(blocks, c1, c2, c3, seed):
    """Philox-4x32-10 of one request's counters in unsigned 64-bit arithmetic: uniform numbers, four a block."""
    u64, low = np.uint64, np.uint64(_MASK)
    c = [np.asarray(blocks, dtype=u64)] + [np.full(len(blocks), x & _MASK, dtype=u64) for x in (c1, c2, c3)]
    k = [seed & _MASK, (seed >> 32) & _MASK]
    for _ in range(10):
        p0, p1 = c[0] * u64(0xD2511F53), c[2] * u64(0xCD9E8D57)
        c = [(p1 >> u64(32)) ^ c[1] ^ u64(k[0]), p1 & low, (p0 >> u64(32)) ^ c[3] ^ u64(k[1]), p0 & low]
        k = [(k[0] + 0x9E3779B9) & _MASK, (k[1] + 0xBB67AE85) & _MASK]
    return ((np.stack(c, 1).reshape(-1) >> u64(9)).astype(np.float64) + 0.5) / 8388608.0


def _distribution64(row, temperature, k):
    x = row.double()
    scaled = (row / temperature).double()                # the threshold is on what the 32-bit division gives
    drop = torch.isnan(x) | (x == -math.inf)
    if 0 < k < row.shape[0]:
        kth = torch.sort(torch.where(torch.isnan(x), -math.inf, scaled), descending=True).values[k - 1]
        drop |= scaled < kth
    return torch.softmax(torch.where(drop, -math.inf, x / float(temperature)), 0)


def _drawn64(st, r, row, place):
    """The token that request r's stream draws from a row of logits."""
    x = st["logits"][row]
    if int(st["greedy"][r]):
        return int(x.argmax())
    p = _distribution64(x, st["temperature"][r], int(st["topk"][r]))
    u = _words64(np.arange((len(x) + 3) // 4), int(st["step"][r]) + place, int(st["stream_id"][r]), 0, int(st["seed"][r]))[:len(x)]
    return int((p.log() - (-torch.from_numpy(u).to(p.device).log()).log()).argmax())


def _exact_verify(st):
    cu, fed = st["cu_rows"].tolist(), st["token_ids"].tolist()
    n_req, d, v = len(cu) - 1, st["drafts"], st["vocab"]
    tokens = torch.full((n_req, d + 1), -1, dtype=torch.int32)
    counts = torch.zeros(n_req, dtype=torch.int32)
    accept = torch.zeros((n_req, d), dtype=torch.float64)
    seeds, streams, steps = st["seed"].tolist(), st["stream_id"].tolist(), st["step"].tolist()
    greedy, topk, with_q = st["greedy"].tolist(), st["topk"].tolist(), st["draft_logits"] is not None
    for r in range(n_req):
        t, n, held = st["temperature"][r], cu[r + 1] - cu[r] - 1, None
        for j in range(n):
            row, draft = st["logits"][cu[r] + j], fed[cu[r] + j + 1]
            if greedy[r]:
                accept[r, j] = float(int(row.argmax()) == draft)
            else:
                p = float(_distribution64(row, t, topk[r])[draft])
                q = 1.0 if st["draft_logits"] is None else float(_distribution64(st["draft_logits"][r, j], t, topk[r])[draft])
                accept[r, j] = min(1.0, p / q) if q > 0 else float(p > 0)
            if held is None and with_q and not _words64([0], steps[r] + j, streams[r], 1, seeds[r])[0] < float(accept[r, j]):
                held = j
            if held is None and not with_q and _drawn64(st, r, cu[r] + j, j) != draft:
                held = j
        refused = held is not None
        held = n if held is None else held
        if refused and with_q and not greedy[r]:
            p = _distribution64(st["logits"][cu[r] + held], t, topk[r])
            q = _distribution64(st["draft_logits"][r, held], t, topk[r])
            p = torch.where(p > q, p - q, 0.0) if bool((p > q).any()) else p
            u = torch.from_numpy(_words64(np.arange((v + 3) // 4), steps[r] + held, streams[r], 2, seeds[r])[:v]).to(p.device)
            token = int((p.log() - (-u.log()).log()).argmax())
        else:
            token = _drawn64(st, r, cu[r] + held, held)
        tokens[r, :held] = torch.tensor(fed[cu[r] + 1:cu[r] + 1 + held], dtype=torch.int32)
        tokens[r, held] = token
        counts[r] = held + 1
    return dict(tokens=tokens, counts=counts, accept=accept)


def exact(case, seed):
    if case["op"] != "verify":               # the other operators' outputs are whole numbers
        return None
    return _exact_verify(prepare(case, seed))
