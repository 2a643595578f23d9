"""Plain 64-bit forms of the paged-cache operators (numpy), for the tests."""

from __future__ import annotations

import math

import numpy as np


def slots(lengths, counts, start, free, free_count, table, tokens, page):
    """offsets, lengths_out, positions, slots, table_out, free_left, from the operator's definition."""
    requests, columns = table.shape
    out = np.full_like(table, -1)
    offsets, after = [0], []
    positions, places = np.full(tokens, -1, np.int32), np.full(tokens, -1, np.int32)
    stack = [int(p) for p in free[:max(0, min(int(free_count), len(free)))]]
    left = len(stack)
    row = 0
    for b in range(requests):
        held, new = max(0, int(lengths[b])), max(0, int(counts[b]))
        have = min(columns, -(-held // page))
        want = min(columns, -(-(held + new) // page))
        out[b, :have] = table[b, :have]
        for column in range(have, want):
            out[b, column] = stack.pop() if stack else -1
            left -= 1
        for i in range(new):
            if row < tokens:
                place = held + i
                p = int(out[b, place // page]) if place // page < columns else -1
                positions[row] = start + place
                places[row] = p * page + place % page if p >= 0 else -1
            row += 1
        offsets.append(min(row, tokens))
        after.append(held + new)
    return (np.array(offsets, np.int32), np.array(after, np.int32), positions, places, out, np.array([left], np.int32))


def rotary(x, positions, angles, layout, inverse=False):
    """x [tokens, heads, dim] turned, in 64 bits; padding gives zeros, positions past the table NaN."""
    x = x.astype(np.float64)
    out = x.copy()
    rotated = angles.shape[1]
    for t, p in enumerate(positions):
        if p < 0 or p >= angles.shape[0]:
            out[t] = 0.0 if p < 0 else np.nan
            continue
        c, s = angles[p, :rotated // 2].astype(np.float64), angles[p, rotated // 2:].astype(np.float64)
        s = -s if inverse else s
        if layout == "half":
            i, j = np.arange(rotated // 2), np.arange(rotated // 2) + rotated // 2
        else:
            i, j = 2 * np.arange(rotated // 2), 2 * np.arange(rotated // 2) + 1
        out[t][:, i] = x[t][:, i] * c - x[t][:, j] * s
        out[t][:, j] = x[t][:, j] * c + x[t][:, i] * s
    return out


def keys_of(cache, pages, count, page):
    """[count, kv, dim] of the first keys behind a page list, and which of them are there."""
    at = np.arange(count)
    p = np.asarray(pages)[at // page]
    there = (p >= 0) & (p < cache.shape[0])
    rows = cache[np.where(there, p, 0), :, at % page]
    return rows.astype(np.float64), there


def attention(q, k_cache, v_cache, offsets, lengths, table, prefix_pages, prefix_length, scale=None):
    """(output, bound): the output in 64 bits, and what an fp16 result may differ from it by.

    The operator rounds its output to fp16 (2^-11 of it, 2^-25 below fp16's normal values) and the softmax
    weights entering the second product to fp16: 2^-11 of each, so of sum_j p_j |v_j|, and at most 2^-25
    of the largest for a subnormal one.  Scores are fp32 sums of dim products of scale |q||k|: dim 2^-24 of
    their sum changes a weight by that relative amount; so do the exponent's two roundings, 2^-23 of it.
    """
    tokens, heads, dim = q.shape
    kv, page = k_cache.shape[1], k_cache.shape[2]
    share = heads // kv
    scale = 1.0 / math.sqrt(dim) if scale is None else scale
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    pk, p_there = keys_of(k_cache, prefix_pages, prefix_length, page)
    pv, _ = keys_of(v_cache, prefix_pages, prefix_length, page)
    for b in range(len(lengths)):
        first, last, length = int(offsets[b]), int(offsets[b + 1]), int(lengths[b])
        k, there = keys_of(k_cache, table[b], length, page)
        v, _ = keys_of(v_cache, table[b], length, page)
        for i in range(first, last):
            sees = np.arange(length) <= length - (last - first) + i - first
            mask = np.concatenate([p_there, there & sees])
            if not mask.any():
                continue
            kk, vv = np.concatenate([pk, k])[mask], np.concatenate([pv, v])[mask]
            for h in range(heads):
                kh, vh, qh = kk[:, h // share], vv[:, h // share], q[i, h].astype(np.float64)
                s = scale * (kh @ qh)
                with np.errstate(invalid="ignore", over="ignore"):
                    w = np.exp(s - s.max())
                    w /= w.sum()
                    out[i, h] = w @ vh
                    size = w @ np.abs(vh)
                    worst = scale * np.max(np.abs(kh) @ np.abs(qh))
                    rest = len(w) * 2.0 ** -25 * w.max() * np.abs(vh).max(axis=0)
                    bound[i, h] = (2.0 ** -11 * np.abs(out[i, h]) + 2.0 ** -25 + rest
                                   + size * (2.0 ** -11 + 2 * (dim * 2.0 ** -24 * worst + 2.0 ** -22 * (1 + worst))))
    return out, bound


def paging(rng, lengths, page, prefix, spare=3):
    """(table, prefix pages, page count): pages of each request and of the prefix in a random order."""
    held = [-(-n // page) for n in lengths]
    shared = max(1, -(-prefix // page))
    pages = sum(held) + shared + spare
    order = rng.permutation(pages).astype(np.int32)
    table = np.full((len(lengths), max(1, *held)), -1, np.int32)
    at = 0
    for b, n in enumerate(held):
        table[b, :n] = order[at:at + n]
        at += n
    return table, order[at:at + shared].copy(), pages
