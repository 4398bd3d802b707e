"""Plain restatements, in 64 bits, of the decoding operators (paged key-value cache, beam search) -- test infrastructure.  Pages, tables and counts as
include/mmamd.h describes them; everything is numpy and loops."""
from __future__ import annotations

import math

import numpy as np


def place(table, row, t, page, pages):
    """(page, place) of token t of a row, or None where it has none."""
    if t < 0 or t >= table.shape[1] * page:
        return None
    p = int(table[row, t // page])
    return (p, t % page) if 0 <= p < pages else None


def paged_attention(q, key_pages, value_pages, table, lengths, k=None, v=None, scale=None, weight_loss=0.0):
    """(out [rows, heads, dim] float64, key_pages, value_pages after the call, err): err bounds what 32-bit arithmetic may lose, see `fp32_loss`,
    and a loss of `weight_loss` of every weight."""
    kp, vp = key_pages.copy(), value_pages.copy()
    rows, heads, dim = q.shape
    pages, kv_heads, page, _ = kp.shape
    group = heads // kv_heads
    scale = 1.0 / math.sqrt(dim) if scale is None else scale
    cap = table.shape[1] * page
    out, err = np.zeros((rows, heads, dim)), np.zeros((rows, heads, dim))
    for r in range(rows):
        n = int(lengths[r])
        seen = min(max(n, 0), cap)
        if k is not None and 0 <= n < cap:
            at = place(table, r, n, page, pages)
            if at is not None:
                kp[at[0], :, at[1]], vp[at[0], :, at[1]] = k[r], v[r]
            seen = n + 1
        places = [a for a in (place(table, r, t, page, pages) for t in range(seen)) if a is not None]
        if not places:
            continue
        ids, offs = np.array([a[0] for a in places]), np.array([a[1] for a in places])
        for h in range(heads):
            kk, vv = kp[ids, h // group, offs].astype(np.float64), vp[ids, h // group, offs].astype(np.float64)
            qq = q[r, h].astype(np.float64)
            s = scale * (kk @ qq)
            w = np.exp(s - s.max())
            w /= w.sum()
            out[r, h] = w @ vv
            err[r, h] = (fp32_loss(scale * (np.abs(kk) @ np.abs(qq)).max(), dim, len(places)) + weight_loss) * (w @ np.abs(vv))
    return out, kp, vp, err


def fp32_loss(abs_score, dim, n):
    """Relative to sum w |v|: a score of `dim` products summed in 32 bits is off by at most (dim + 4) 2^-24 of the sum of their magnitudes, and a weight and
    the sum of the weights by as much each; exp2 and the rescaling by 2^-21; n weights and n products summed by (2 n + 64) 2^-24, n at most the serial length of one lane
    (n / 16 + 64)."""
    return 2 * (dim + 4) * 2.0 ** -24 * abs_score + 2.0 ** -20 + (2 * (n / 16 + 64)) * 2.0 ** -24


def paged_append(k, v, key_pages, value_pages, table, start, counts=None):
    kp, vp = key_pages.copy(), value_pages.copy()
    rows, tokens = k.shape[:2]
    for r in range(rows):
        for j in range(tokens if counts is None else min(int(counts[r]), tokens)):
            at = place(table, r, int(start[r]) + j, kp.shape[2], kp.shape[0])
            if at is not None:
                kp[at[0], :, at[1]], vp[at[0], :, at[1]] = k[r, j], v[r, j]
    return kp, vp


def paged_fork(pool, table, lengths, refcounts, parents, reserve):
    """(pool after, table, lengths, refcounts, shortage)."""
    pages, page = pool.shape[0], pool.shape[-2]
    slots, cap = table.shape[1], table.shape[1] * page
    after = pool.copy()
    free = [x for x in range(pages) if refcounts[x] <= 0]
    counts = refcounts.astype(np.int64).copy()
    for x in table.reshape(-1):
        if 0 <= x < pages:
            counts[x] -= 1
    new = np.full((len(parents), slots), -1, np.int32)
    lens = np.zeros(len(parents), np.int32)
    short, seen = 0, set()

    def take():
        nonlocal short
        if free:
            return free.pop(0)
        short += 1
        return -1

    for r, p in enumerate(int(x) for x in parents):
        there = 0 <= p < len(lengths)
        n = min(max(int(lengths[p]), 0), cap) if there else 0
        m = min(n + max(0, int(reserve if np.isscalar(reserve) else reserve[r])), cap)
        full, rest = n // page, n % page
        for j in range(full):
            x = int(table[p, j])
            new[r, j] = x if 0 <= x < pages else -1
        if rest:
            src = int(table[p, full])
            if 0 <= src < pages:
                if refcounts[src] == 1 and p not in seen:
                    new[r, full] = src
                else:
                    new[r, full] = dst = take()
                    if dst >= 0:
                        after[dst][..., :rest, :] = pool[src][..., :rest, :]
        if there:
            seen.add(p)
        for j in range(-(-n // page), -(-m // page)):
            new[r, j] = take()
        lens[r] = n
    for x in new.reshape(-1):
        if x >= 0:
            counts[x] += 1
    return after, new, lens, counts.astype(np.int32), short


def paged_compact(pool, table, refcounts):
    """(pool after, table, refcounts, live)."""
    after, pages = pool.copy(), pool.shape[0]
    live = int((refcounts > 0).sum())
    holes = [x for x in range(live) if refcounts[x] <= 0]
    to, counts = {}, np.zeros_like(refcounts)
    for x in range(pages):
        if refcounts[x] > 0:
            to[x] = x if x < live else holes.pop(0)
            if to[x] != x:
                after[to[x]] = pool[x]
            counts[to[x]] = refcounts[x]
    new = np.array([[to.get(int(x), -1) for x in row] for row in table], np.int32).reshape(table.shape)
    return after, new, counts, live


def beam_search_step(logits, scores, lengths, finished, sequences, eos, penalty=0.0):
    """(scores float64, lengths, finished, tokens, parents, sequences)."""
    groups, beams = scores.shape
    vocab = logits.shape[1]
    x = logits.astype(np.float64).reshape(groups, beams, vocab)
    out = [[], [], [], [], [], []]
    for g in range(groups):
        offers = []
        for b in range(beams):
            total = np.full(vocab, -np.inf)
            s = float(scores[g, b])
            if finished[g, b]:
                if s > -np.inf:
                    total[eos] = s
            elif s > -np.inf:
                with np.errstate(all="ignore"):
                    top = x[g, b].max()
                    lse = top + np.log(np.exp(x[g, b] - top).sum())
                if np.isfinite(lse):
                    total = s + (x[g, b] - lse)
            n = int(lengths[g, b]) + (0 if finished[g, b] else 1)
            rank = total / float(max(n, 1)) ** penalty
            offers += [(-rank[t], b * vocab + t, total[t]) for t in np.argsort(-rank, kind="stable")[:beams]]
        offers.sort()
        for _, flat, total in offers[:beams]:
            b, token = divmod(int(flat), vocab)
            row = None if sequences is None else sequences[g, b].copy()
            fin, n = bool(finished[g, b]), int(lengths[g, b])
            if row is not None and not fin and 0 <= n < row.size:
                row[n] = token
            for to, y in zip(out, (total, n if fin else n + 1, fin or token == eos, token, g * beams + b, row)):
                to.append(y)
    kinds = (np.float64, np.int32, bool, np.int64, np.int32)
    res = [np.array(y, t).reshape(groups, beams) for y, t in zip(out, kinds)]
    return (*res, None if sequences is None else np.array(out[5], np.int64).reshape(groups, beams, sequences.shape[2]))
