"""Paged-cache operators in fp64 numpy, sequence by sequence, head by head.

The definitions of ``include/fna2.h``: attention of a chunk of new tokens over
the rows that a block table names, the cached rows' attention weights, the
append of new rows (RMSNorm, rotation) and eviction by weight.  bf16 and fp16
inputs are taken as they are; nothing is rounded.
"""
from __future__ import annotations

import math

import numpy as np


def _np(t):
    return None if t is None else t.detach().double().cpu().numpy()


def rows_of(pages, table_row, head, n, page_size):
    """Rows 0 .. n - 1 of one head: ([n, F], [n] whether the row is there)."""
    P, F = pages.shape[0], pages.shape[3]
    out, there = np.zeros((n, F)), np.zeros(n, bool)
    for j in range(n):
        p = int(table_row[j // page_size])
        if 0 <= p < P:
            out[j], there[j] = pages[p, head, j % page_size], True
    return out, there


def attend(q, k_pages, v_pages, table, lens, cu, r_q=None, rk_pages=None, gs=None, scale=None,
           causal=True):
    """(out [T, H, D], lse [T, H], weights [N, H_KV, capacity], the same
    average of |V| as out is of V: what roundings of P scale with)."""
    q, kp, vp, rq, rkp, gs = map(_np, (q, k_pages, v_pages, r_q, rk_pages, gs))
    table, lens, cu = (np.asarray(x.cpu()) for x in (table, lens, cu))
    T, H, D = q.shape
    hkv, ps = kp.shape[1], kp.shape[2]
    g = H // hkv
    hg = 0 if rq is None else rq.shape[1]
    scale = D ** -0.5 if scale is None else scale
    cap = table.shape[1] * ps
    out, lse, mag = np.zeros((T, H, D)), np.full((T, H), -np.inf), np.zeros((T, H, D))
    w = np.zeros((len(lens), hkv, cap))
    for b in range(len(lens)):
        length = max(int(lens[b]), 0)
        n = min(length, cap)
        t0, m = int(cu[b]), int(cu[b + 1] - cu[b])
        for kv in range(hkv):
            K, there = rows_of(kp, table[b], kv, n, ps)
            V, _ = rows_of(vp, table[b], kv, n, ps)
            for h in range(kv * g, (kv + 1) * g):
                rk = rows_of(rkp, table[b], h, n, ps)[0] if h < hg else None
                for i in range(m):
                    see = there & ((np.arange(n) <= length - m + i) if causal else True)
                    if not see.any():
                        continue
                    s = scale * (K[see] @ q[t0 + i, h])
                    if h < hg:
                        s = s + gs[h] * (rk[see] @ rq[t0 + i, h])
                    top = s.max()
                    p = np.exp(s - top)
                    l = p.sum() + 1e-6
                    out[t0 + i, h] = (p[:, None] * V[see]).sum(0) / l
                    mag[t0 + i, h] = (p[:, None] * np.abs(V[see])).sum(0) / l
                    lse[t0 + i, h] = top + math.log(l)
                    w[b, kv, :n][see] += p / l
    return out, lse, w, mag


def norm_rope(x, weight, pos, inv_freq, eps):
    """[heads, D] rows of one token."""
    x = np.asarray(x, np.float64)
    D = x.shape[-1]
    if weight is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * weight
    if inv_freq is not None:
        a = float(pos) * inv_freq
        x1, x2 = x[..., : D // 2], x[..., D // 2:]
        x = np.concatenate([x1 * np.cos(a) - x2 * np.sin(a), x2 * np.cos(a) + x1 * np.sin(a)], -1)
    return x


def append(q, k, v, k_pages, v_pages, table, lens, cu, r_k=None, rk_pages=None, inv_freq=None,
           positions=None, norm_q=None, norm_k=None, eps=1e-6, position_shift=None):
    """(q_out, k_pages, v_pages, rk_pages) after the append."""
    q, k, v, rk = map(_np, (q, k, v, r_k))
    kp, vp, rkp = (None if t is None else _np(t).copy() for t in (k_pages, v_pages, rk_pages))
    inv, wq, wk = map(_np, (inv_freq, norm_q, norm_k))
    table, lens, cu = (np.asarray(x.cpu()) for x in (table, lens, cu))
    pos = None if positions is None else np.asarray(positions.cpu())
    P, _, ps, _ = kp.shape
    cap = table.shape[1] * ps
    out = q.copy()
    for b in range(len(lens)):
        n = max(int(lens[b]), 0)
        m = int(cu[b + 1] - cu[b])
        for i in range(m):
            t, row = int(cu[b]) + i, n - m + i
            at = row if pos is None else int(pos[t])
            at += 0 if position_shift is None else int(position_shift[b])
            out[t] = norm_rope(q[t], wq, at, inv, eps)
            if not 0 <= row < cap:
                continue
            p = int(table[b, row // ps])
            if not 0 <= p < P:
                continue
            kp[p, :, row % ps] = norm_rope(k[t], wk, at, inv, eps)
            vp[p, :, row % ps] = v[t]
            if rk is not None:
                rkp[p, :, row % ps] = rk[t]
    return out, kp, vp, rkp


def keep_rows(weights, n, budget, recent, first):
    """The rows of one (sequence, KV head) that are kept, ascending."""
    if n <= budget:
        return list(range(n))
    w = [float(weights[j]) if j < len(weights) else 0.0 for j in range(n)]
    rank = lambda j: (0 if math.isnan(w[j]) else 1, 0.0 if math.isnan(w[j]) else -w[j], j)
    mid = sorted(range(first, n - recent), key=rank)[: budget - first - recent]
    return sorted(list(range(first)) + mid + list(range(n - recent, n)))


def evict(k_pages, v_pages, table, lens, weights, budget, recent=0, first=0, rk_pages=None,
          heads=None):
    """(kept, new_lens, weights, k_pages, v_pages, rk_pages)."""
    kp, vp, rkp = (None if t is None else _np(t).copy() for t in (k_pages, v_pages, rk_pages))
    w = weights.detach().cpu().numpy()
    table, lens = (np.asarray(x.cpu()) for x in (table, lens))
    P, hkv, ps, _ = kp.shape
    N, cap = len(lens), w.shape[2]
    kept = np.full((N, hkv, budget), -1, np.int32)
    new = np.zeros(N, np.int32)
    wo = np.zeros_like(w)
    hg = 0 if rkp is None else rkp.shape[1]
    g = (heads or hkv) // hkv
    for b in range(N):
        n = min(max(int(lens[b]), 0), table.shape[1] * ps)
        new[b] = min(n, budget)
        at = lambda j: (int(table[b, j // ps]), j % ps)
        there = lambda j: 0 <= at(j)[0] < P
        for kv in range(hkv):
            rows = keep_rows(w[b, kv], n, budget, recent, first)
            kept[b, kv, : len(rows)] = rows
            for r, j in enumerate(rows):
                if r < cap:
                    wo[b, kv, r] = w[b, kv, j] if j < cap else 0.0
                if n > budget and j != r and there(j) and there(r):
                    (ps_, po), (pd, do) = at(j), at(r)
                    kp[pd, kv, do], vp[pd, kv, do] = kp[ps_, kv, po], vp[ps_, kv, po]
                    for h in range(kv * g, min((kv + 1) * g, hg)):
                        rkp[pd, h, do] = rkp[ps_, h, po]
    return kept, new, wo, kp, vp, rkp
