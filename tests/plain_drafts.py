"""Plain statements of decoding with drafts, one request at a time: verification in float64 (the top-k threshold on the float32
quotient it is defined on), the lookup of drafts and the arrays of a step on Python integers."""
from __future__ import annotations

import math

import numpy as np

MASK = 0xFFFFFFFF


def philox(c0, c1, c2, c3, seed):
    """The four words of the Philox-4x32-10 block with this counter under a 64-bit key."""
    c, k = [c0 & MASK, c1 & MASK, c2 & MASK, c3 & MASK], [seed & MASK, (seed >> 32) & MASK]
    for _ in range(10):
        p0, p1 = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(p1 >> 32) ^ c[1] ^ k[0], p1 & MASK, (p0 >> 32) ^ c[3] ^ k[1], p0 & MASK]
        k = [(k[0] + 0x9E3779B9) & MASK, (k[1] + 0xBB67AE85) & MASK]
    return c


def uniform(word):
    return ((word >> 9) + 0.5) / 8388608.0


def uniforms(v, step, stream, domain, seed):
    """A number per token, by the blocks of four that the stream hands out."""
    c = [np.arange((v + 3) // 4, dtype=np.uint64)] + [np.full((v + 3) // 4, x & MASK, dtype=np.uint64) for x in (step, stream, domain)]
    k = [seed & MASK, (seed >> 32) & MASK]
    s32, low = np.uint64(32), np.uint64(MASK)
    for _ in range(10):
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(p1 >> s32) ^ c[1] ^ np.uint64(k[0]), p1 & low, (p0 >> s32) ^ c[3] ^ np.uint64(k[1]), p0 & low]
        k = [(k[0] + 0x9E3779B9) & MASK, (k[1] + 0xBB67AE85) & MASK]
    return ((np.stack(c, 1).reshape(-1)[:v] >> np.uint64(9)).astype(np.float64) + 0.5) / 8388608.0


def scaled(row, temperature, k):
    """The row over its temperature in float64, -inf where it is NaN or below the k-th largest float32 quotient."""
    with np.errstate(over="ignore"):
        q32 = (row / np.float32(temperature)).astype(np.float32)
    s = row.astype(np.float64) / float(np.float32(temperature))
    s[np.isinf(q32)] = q32[np.isinf(q32)]                # what float32 division makes infinite is infinite
    s[np.isnan(row)] = -math.inf
    ok = ~np.isnan(row)
    if 0 < k < row.shape[0] and ok.any():
        order = np.sort(q32[ok])[::-1]
        if k <= order.shape[0]:
            s[ok & (q32 < order[k - 1])] = -math.inf
    return s


def probabilities(s):
    m = s.max()
    if m == -math.inf:
        return np.zeros_like(s)
    with np.errstate(invalid="ignore"):
        w = np.where(s == m, 1.0, np.exp(s - m))
    return w / w.sum()


def first_largest(row):
    ok = ~np.isnan(row)
    return -1 if not ok.any() else int(np.argmax(np.where(ok, row, -np.inf))) if (row[ok] > -np.inf).any() else int(np.argmax(ok))


def gap(score):
    """The first largest entry and by how much it leads."""
    i = int(np.argmax(score))
    rest = np.delete(score, i)
    if not rest.size or rest.max() == -math.inf or score[i] == math.inf:
        return i, math.inf                               # (among infinite ones the first wins, exactly)
    return i, float(score[i] - rest.max())


def draw(row, *, temperature, topk, greedy, seed, stream, step):
    """The token that a row draws (-1: it has none) and by how much it leads."""
    if greedy:
        return first_largest(row), math.inf
    s = scaled(row, temperature, topk)
    if s.max() == -math.inf:
        return -1, math.inf
    return gap(s - np.log(-np.log(uniforms(row.shape[0], step, stream, 0, seed))))


def verify(logits, fed, *, max_drafts, temperature=1.0, topk=0, greedy=True, seed=0, stream=0, step=0, draft_logits=None):
    """One request: its rows [n + 1, V] and the tokens it was fed. Returns (tokens, accept, margin): margin is how far the
    nearest decision was from going the other way, in relative terms."""
    rows = min(logits.shape[0], max_drafts + 1)
    accept = np.zeros(max_drafts)
    if rows == 0:
        return [], accept, math.inf
    vocab, held, margin = logits.shape[1], None, math.inf
    for j in range(rows - 1):
        d = fed[j + 1]
        if greedy:
            accept[j] = float(d >= 0 and d == first_largest(logits[j]))
        elif 0 <= d < vocab:
            p = probabilities(scaled(logits[j], temperature, topk))[d]
            q = 1.0 if draft_logits is None else probabilities(scaled(draft_logits[j], temperature, topk))[d]
            accept[j] = min(1.0, p / q) if q > 0 else float(p > 0)
        if held is None and draft_logits is not None and not greedy:
            u = uniform(philox(0, step + j, stream, 1, seed)[0])
            if 0.0 < accept[j] < 1.0:
                margin = min(margin, abs(u - accept[j]) / accept[j])
            if not u < accept[j]:
                held = j
        elif held is None:
            token, lead = draw(logits[j], temperature=temperature, topk=topk, greedy=greedy, seed=seed, stream=stream, step=step + j)
            margin = min(margin, lead)
            if token < 0 or token != d:
                held = j
    failed = held is not None
    held = rows - 1 if held is None else held
    if failed and draft_logits is not None and not greedy:
        p, q = (probabilities(scaled(x[held], temperature, topk)) for x in (logits, draft_logits))
        left = np.maximum(p - q, 0.0)
        left = left if (left > 0).any() else p
        with np.errstate(divide="ignore"):
            score = np.log(left) - np.log(-np.log(uniforms(vocab, step + held, stream, 2, seed)))
        token, lead = gap(score) if score.max() > -math.inf else (-1, math.inf)
    else:
        token, lead = draw(logits[held], temperature=temperature, topk=topk, greedy=greedy, seed=seed, stream=stream, step=step + held)
    token, margin = max(token, 0), min(margin, lead)
    return list(fed[1:held + 1]) + [token], accept, margin


def ngram(text, *, max_drafts, max_match=3, min_match=1):
    """The drafts that follow ``text``."""
    n, best = len(text), (0, 0)
    for e in range(1, n):
        l = 0
        while l < min(max_match, e) and text[e - 1 - l] == text[n - 1 - l]:
            l += 1
        if l >= min_match:
            best = max(best, (l, e))
    if best[0] == 0:
        return []
    out = list(text)
    for t in range(max_drafts):
        out.append(out[best[1] + t])
    return out[n:]


def step_arrays(starts, counts, tables, *, rows, max_count, page_size, tokens=None, state_slots=None, pad_page=-1, tile=128):
    """``tables[group][row]``: lists. Returns a dict of lists, named as the operator's result."""
    s, width = len(starts), len(tables[0][0])
    out = dict(token_ids=[], positions=[], token_seq=[], cache_slots=[[] for _ in tables], cu_seqlens=[0], q_starts=[], context_lens=[],
               tiles=[], block_tables=[[] for _ in tables])
    for r in range(s):
        slot = r if state_slots is None else state_slots[r]
        there = 0 <= slot < len(tables[0]) and starts[r] >= 0
        n = min(max(counts[r], 0), max_count, rows - len(out["positions"])) if there else 0
        start = starts[r] if there else 0
        first = len(out["positions"])
        for i in range(n):
            pos = start + i
            out["positions"].append(pos)
            out["token_seq"].append(r)
            if tokens is not None:
                out["token_ids"].append(tokens[r][i])
            for g, t in enumerate(tables):
                page = t[slot][pos // page_size] if pos // page_size < width else -1
                out["cache_slots"][g].append(page * page_size + pos % page_size if page >= 0 else -1)
        out["cu_seqlens"].append(first + n)
        out["q_starts"].append(start)
        out["context_lens"].append(start + n)
        for k in range(-(-max_count // tile)):
            off = min(k * tile, n)
            out["tiles"].append([r, first + off, min(n - off, tile), start + off])
        held = min(width, -(-(start + n) // page_size)) if there else 0
        for g, t in enumerate(tables):
            out["block_tables"][g].append((list(t[slot][:held]) if there else []) + [-1] * (width - held))
    left = rows - len(out["positions"])
    out["positions"] += [0] * left
    out["token_seq"] += [s] * left
    out["token_ids"] += [0] * left
    out["cu_seqlens"].append(rows)
    out["q_starts"].append(0)
    out["context_lens"].append(1)
    for g in range(len(tables)):
        out["cache_slots"][g] += [-1] * left
        out["block_tables"][g].append([pad_page] + [-1] * (width - 1))
    if tokens is None:
        out["token_ids"] = None
    return out
