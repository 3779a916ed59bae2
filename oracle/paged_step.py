"""Oracle (CPU) of the operators around the paged cache — test infrastructure only; never
imported by the product.

assign_pages_np     pages, slots and positions of a step's new tokens, request by request, with
release_pages_np    a Python list as the free list's stack; and the pages' way back
norm_rope_np        RMSNorm of head rows and the position rotation, in float64: each pair of
                    dimensions turned as a complex number
token_logprobs_np   log probabilities, entropy and alternatives of logits rows, in float64

None has a counterpart in the reference: parity is with the definitions in
include/fdllm_hip.h.
"""
from __future__ import annotations

import numpy as np


def assign_pages_np(new_lens, lens, table, free, page_size, width=0, rows=0):
    """``lens`` (list), ``table`` (2-D array) and ``free`` (list of ids, the last one handed out
    first) are changed in place. Returns a dict of lists / arrays."""
    max_pages = table.shape[1]
    n_rows = len(lens) * width if width else rows
    out = {"slots": np.full(n_rows, -1, np.int64), "positions": np.zeros(n_rows, np.int64),
           "sequences": np.full(n_rows, -1, np.int64), "row_starts": [], "starts": [], "seqlens": [], "granted": []}
    at, short = 0, False
    for b, new in enumerate(new_lens):
        n, old = max(int(new), 0), max(int(lens[b]), 0)
        first = b * width if width else at
        out["row_starts"].append(min(at, 2 ** 31 - 1))
        at += n
        have, total = -(-old // page_size), -(-(old + n) // page_size)
        ok = n > 0 and old + n < 2 ** 31 and total <= max_pages and (n <= width if width else at <= rows)
        if ok and total > have:
            short = short or total - have > len(free)
            ok = not short
        if ok:
            for j in range(have, total):
                table[b, j] = free.pop()
            lens[b] = old + n
        elif lens[b] < 0:
            lens[b] = 0
        last = min(first + (min(n, width) if width else n), n_rows)
        for r in range(first, last):
            pos = old + r - first
            out["positions"][r], out["sequences"][r] = pos, b
            if ok:
                out["slots"][r] = int(table[b, pos // page_size]) * page_size + pos % page_size
        out["starts"].append(old)
        out["seqlens"].append(old + (n if ok else 0))
        out["granted"].append(n if ok else 0)
    out["row_starts"].append(min(at, 2 ** 31 - 1))
    return out


def release_pages_np(keep_lens, lens, table, free, page_size):
    gone = []
    for b, keep in enumerate(keep_lens):
        old = max(int(lens[b]), 0)
        new = min(max(int(keep), 0), old)
        gone += [int(table[b, j]) for j in range(-(-new // page_size), -(-old // page_size))]
        lens[b] = new
    free.extend(reversed(gone))


def norm_rope_np(x, positions, inv_freq, weight=None, eps=1e-6, interleaved=False, rope_scale=1.0):
    """x [B, S, H, D] -> float64 of the same shape."""
    y = np.array(x, np.float64)
    if weight is not None:
        y = y / np.sqrt(np.mean(y * y, -1, keepdims=True) + eps) * np.asarray(weight, np.float64)
    half = len(inv_freq)
    i = np.arange(half)
    first, second = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    angle = np.asarray(positions, np.float64)[..., None] * np.asarray(inv_freq, np.float64)
    z = (y[..., first] + 1j * y[..., second]) * (rope_scale * np.exp(1j * angle))[:, :, None, :]
    y[..., first], y[..., second] = z.real, z.imag
    return y


def token_logprobs_np(logits, tokens=None, top_k=0):
    """logits [N, V], tokens [N, M] -> (logprobs [N, M], entropy [N], top_logprobs, top_tokens)."""
    x = np.asarray(logits, np.float64)
    n, vocab = x.shape
    lp = np.full((n, 0 if tokens is None else tokens.shape[1]), np.nan)
    ent, top = np.full(n, np.nan), np.full((n, top_k), np.nan)
    ids = np.full((n, top_k), -1, np.int64)
    for r in range(n):
        row = x[r]
        m = row.max() if not np.isnan(row).any() else np.nan
        if not np.isfinite(m):
            continue
        p = np.exp(row - m)
        logp = row - m - np.log(p.sum())
        q = p / p.sum()
        ent[r] = -np.sum(q[q > 0] * logp[q > 0])
        for j in range(lp.shape[1]):
            t = int(tokens[r, j])
            lp[r, j] = logp[t] if 0 <= t < vocab else np.nan
        order = np.argsort(-row, kind="stable")[:top_k]
        ids[r], top[r] = order, logp[order]
    return lp, ent, top, ids
