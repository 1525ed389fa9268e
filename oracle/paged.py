"""The paged cache's operators in plain form: the page tables request by
request, attention and the norm + RoPE rows in float64.  No reference
counterpart (its cache is one run of tokens per sequence, S:519-611); pinned by
closed forms in tests/test_oracle_paged.py."""
from __future__ import annotations

import numpy as np

POOL_EMPTY, TABLE_FULL, SLOTS_FULL, BAD_LENGTH, RING_FULL = 1, 2, 4, 8, 16


def advance(seq_lens, new_tokens, table, free_pages, state, page, cap, row=0):
    """One step of the page tables, one request after the other.  Arrays are
    not changed; returns (lens, table, free_pages, state, slots, positions,
    starts).  row > 0: the tokens of request i end at place (i + 1) * row."""
    lens, table, ring = seq_lens.astype(np.int64), table.copy(), free_pages.copy()
    head, count, status = int(state[0]), int(state[1]), int(state[2])
    pages, width = len(ring), table.shape[1]
    slots, positions = np.full(cap, -1, np.int64), np.full(cap, -1, np.int32)
    starts = np.zeros(len(lens) + 1, np.int64)
    wanted = taken = freed = 0
    for i, n in enumerate(int(x) for x in new_tokens):
        have = int(lens[i])
        at = int(starts[i])
        starts[i + 1] = min(at + max(n, 0), cap + 1)
        if have < 0 or have > width * page:
            status |= BAD_LENGTH
        elif n < 0:
            kept = max(have + n, 0)
            for j in range(-(-kept // page), -(-have // page)):
                if count + freed < pages:
                    ring[(head + count + freed) % pages] = table[i, j]
                freed += 1
            lens[i] = kept
        elif n > 0 and have + n > width * page:
            status |= TABLE_FULL
        elif n > 0 and (n > row if row else at + n > cap):
            status |= SLOTS_FULL
        elif n > 0:
            first, last = -(-have // page), -(-(have + n) // page)
            wanted += last - first                 # refused requests' pages count too
            if last > first and wanted > count:
                status |= POOL_EMPTY
                continue
            for j in range(first, last):
                table[i, j] = free_pages[(head + taken + j - first) % pages]
            taken += last - first
            at = (i + 1) * row - n if row else at
            for t in range(n):
                positions[at + t] = have + t
                slots[at + t] = int(table[i, (have + t) // page]) * page + (have + t) % page
            lens[i] = have + n
    if count + freed > pages:
        status |= RING_FULL
    out = np.array([(head + taken) % pages, min(count + freed, pages) - taken, status, 0], np.int32)
    return lens.astype(np.int32), table, ring, out, slots, positions, starts.astype(np.int32)


def attention(q, k, v, scale):
    """q [heads, d], k / v [n, d] (one KV head), float64: (out [heads, d], lse
    [heads], sum p |v| [heads, d]); zeros and -inf where n is 0."""
    if len(k) == 0:
        z = np.zeros(q.shape)
        return z, np.full(len(q), -np.inf), z
    s = q @ k.T * scale
    m = s.max(-1, keepdims=True)
    p = np.exp(s - m)
    z = p.sum(-1, keepdims=True)
    return p @ v / z, (m + np.log(z))[:, 0], p @ np.abs(v) / z


def norm_rope(x, w, eps, cos, sin):
    """x [..., d] float64: RMSNorm with weight w, then the rotate-half RoPE with
    cos / sin [..., d / 2]."""
    h = x.shape[-1] // 2
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w
    a, b = y[..., :h], y[..., h:]
    return np.concatenate([a * cos - b * sin, b * cos + a * sin], -1)
