"""Paged-cache and beam-search operators restated in NumPy, request by request, in 64 bits.

The definitions the device operators are checked against (no counterpart in the reference, whose
cache is one array per sequence and whose decoding keeps one hypothesis).
"""

from __future__ import annotations

import numpy as np


def extend(lens, new_lens, tables, free_pages, free_count, page_size, max_tokens, release=None):
    """State after the call and its outputs: (tables, free_pages, slots, seq, pos, offsets, lens, free_count)."""
    tables, stack = tables.copy(), free_pages.copy()
    B, cols = tables.shape
    blocks = lambda n: -(-n // page_size)  # noqa: E731
    count = int(np.clip(free_count, 0, len(stack)))
    base = [max(int(n), 0) for n in lens]
    if release is not None:
        for b in range(B):
            if release[b]:
                for page in tables[b, :min(blocks(base[b]), cols)].tolist():
                    if count < len(stack):
                        stack[count] = page
                        count += 1
                base[b] = 0
    slots, seq, pos = np.full(max_tokens, -1, np.int64), np.full(max_tokens, -1, np.int32), np.zeros(max_tokens, np.int32)
    offsets, out_lens, row, open_ = [0], list(base), 0, True
    for b in range(B):
        n = max(int(new_lens[b]), 0)
        need = blocks(base[b] + n) - blocks(base[b])
        open_ = open_ and need <= count and row + n <= max_tokens and base[b] + n <= cols * page_size
        if open_:
            for j in range(blocks(base[b]), blocks(base[b] + n)):
                count -= 1
                tables[b, j] = stack[count]
            for t in range(base[b], base[b] + n):
                slots[row] = int(tables[b, t // page_size]) * page_size + t % page_size
                seq[row], pos[row] = b, t
                row += 1
            out_lens[b] = base[b] + n
        offsets.append(row)
    return tables, stack, slots, seq, pos, np.array(offsets, np.int32), np.array(out_lens, np.int32), count


def give_back(tables, lens, page_size, free_pages, free_count, shares, release=None, parents=None):
    """(free_pages, free_count, shares, lens) after rows left their pages: released ones all of them, beams the full
    pages that their parent does not have in the same column (and takes instead)."""
    stack, shares, lens = free_pages.copy(), shares.copy(), np.maximum(lens, 0)
    count, P = int(np.clip(free_count, 0, len(stack))), len(shares)
    cols, left = tables.shape[1], []
    for b in range(len(tables)):
        if release is not None:
            if release[b]:
                left += tables[b, :min(-(-int(lens[b]) // page_size), cols)].tolist()
                lens[b] = 0
            continue
        K = parents.shape[1]
        p = int(parents.reshape(-1)[b])
        if 0 <= p < K and p != b % K:
            first = b // K * K
            for j in range(min(int(lens[first]) // page_size, cols)):
                old, new = int(tables[b, j]), int(tables[first + p, j])
                if old != new:
                    left.append(old)
                    if 0 <= new < P:
                        shares[new] += 1
    left = [p for p in left if 0 <= p < P]
    for p in left:
        shares[p] -= 1
    for p in left:
        if shares[p] < 0:
            if count < len(stack):
                stack[count] = p
                count += 1
            shares[p] = 0
    return stack, count, shares, lens


def rope_rows(x, cos, sin):
    """Half-split rotation of rows ``(rows, heads, dim)`` by tables rows ``(rows, dim)``, in float64."""
    x = x.astype(np.float64)
    h = x.shape[-1] // 2
    return x * cos[:, None].astype(np.float64) + np.concatenate([-x[..., h:], x[..., :h]], -1) * sin[:, None].astype(np.float64)


def attention(q, k_pages, v_pages, tables, lens, scale, window=0):
    """(out, lse) in float64; a page number outside the pool hides its tokens."""
    B, H, D = q.shape
    P, Hk, ps, _ = k_pages.shape
    out, lse = np.zeros((B, H, D)), np.full((B, H), -np.inf)
    for b in range(B):
        n = min(max(int(lens[b]), 0), tables.shape[1] * ps)
        t = np.arange(max(0, n - window) if window else 0, n)
        page = tables[b, t // ps] if len(t) else np.zeros(0, np.int64)
        t, page = t[(page >= 0) & (page < P)], page[(page >= 0) & (page < P)]
        if not len(t):
            continue
        for h in range(H):
            g = h // (H // Hk)
            k = k_pages[page, g, t % ps].astype(np.float64)
            v = v_pages[page, g, t % ps].astype(np.float64)
            s = scale * (k @ q[b, h].astype(np.float64))
            m = s.max()
            if m == -np.inf:
                continue
            e = np.exp(s - m)
            out[b, h] = e @ v / e.sum()
            lse[b, h] = m + np.log(e.sum())
    return out, lse


def beam(logits, scores, counts, done, stop=(0, 0), min_len=None, alpha=0.0):
    """(tokens, parents, scores, counts, done): the best K of each group's candidates, scores in float64."""
    G, K, V = logits.shape
    outs = ([], [], [], [], [])
    for g in range(G):
        cum, key = np.full((K, V), -np.inf), np.full((K, V), -np.inf)
        for k in range(K):
            s = float(scores[g, k])
            s = s if s > -np.inf else -np.inf
            if done[g, k]:
                cum[k, 0] = s
                key[k, 0] = s / max(int(counts[g, k]), 1) ** alpha
                continue
            x = logits[g, k].astype(np.float64)
            x = np.where(np.isnan(x), -np.inf, x)
            m = x.max()
            if m == -np.inf or s == -np.inf:
                continue
            with np.errstate(invalid="ignore"):
                d = np.where(x == m, 0.0, x - m)
            with np.errstate(divide="ignore"):
                lp = d - np.log(np.exp(d).sum())
            if min_len is not None and counts[g, k] < min_len[g]:
                lp[stop[0]:stop[1]] = -np.inf
            cum[k] = s + lp
            key[k] = cum[k] / (int(counts[g, k]) + 1) ** alpha
        # equal keys (a huge score leaves no room for the logits): the lower hypothesis, its larger logit, the lower token
        x = np.where((key > -np.inf) & (np.asarray(done[g])[:, None] == 0), np.nan_to_num(logits[g].astype(np.float64), nan=-np.inf,
                                                                                          posinf=np.inf, neginf=-np.inf), -np.inf)
        rows, toks = np.divmod(np.arange(K * V), V)
        best = np.lexsort((toks, -x.ravel(), rows, -key.ravel()))[:K]
        par, tok = best // V, best % V
        was = np.asarray(done[g])[par] != 0
        outs[0].append(np.where(was, 0, tok))
        outs[1].append(par)
        outs[2].append(cum.ravel()[best])
        outs[3].append(np.asarray(counts[g])[par] + ~was)
        outs[4].append(was | ((tok >= stop[0]) & (tok < stop[1])))
    return tuple(np.array(o) for o in outs)


def reorder(k_pages, v_pages, tables, parents, lens):
    """New (k_pages, v_pages, tables); pools ``(layers, pages, kv_heads, page_size, dim)``."""
    k_new, v_new, t_new = k_pages.copy(), v_pages.copy(), tables.copy()
    G, K = parents.shape
    P, ps = k_pages.shape[1], k_pages.shape[3]
    for g in range(G):
        n = min(max(int(lens[g * K]), 0), tables.shape[1] * ps)
        full, rest = n // ps, n % ps
        for k in range(K):
            p = int(parents[g, k]) if 0 <= parents[g, k] < K else k
            t_new[g * K + k, :full] = tables[g * K + p, :full]
            if rest and p != k:
                dst, src = int(tables[g * K + k, full]), int(tables[g * K + p, full])
                if 0 <= dst < P and 0 <= src < P:
                    k_new[:, dst, :, :rest] = k_pages[:, src, :, :rest]
                    v_new[:, dst, :, :rest] = v_pages[:, src, :, :rest]
    return k_new, v_new, t_new
