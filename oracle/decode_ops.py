"""A decoding step's operators in 64 bits (test infrastructure only): rows entering a paged
key-value cache, attention over it, sampling. Each is the operator's definition in
``include/lh_b200.h`` written out in numpy; nothing here is on a product path."""

from __future__ import annotations

import numpy as np


def rotate(x, positions, theta: float):
    """Pairs (2i, 2i+1) of the last dimension turned by ``position * theta^(-2i/D)``; x (T, H, D)."""
    x = np.asarray(x, dtype=np.float64)
    d = x.shape[-1]
    angle = np.asarray(positions, dtype=np.float64)[:, None] * theta ** (-np.arange(0, d, 2) / d)
    turned = (x[..., 0::2] + 1j * x[..., 1::2]) * np.exp(1j * angle)[:, None, :]
    out = np.empty_like(x)
    out[..., 0::2], out[..., 1::2] = turned.real, turned.imag
    return out


def paged_append(q, k, v, k_pages, v_pages, slots, positions=None, theta: float = 10000.0):
    """(q, k_pages, v_pages) after the call, and whether a slot pointed outside the pool."""
    k, v = np.asarray(k, np.float64), np.asarray(v, np.float64)
    if theta:
        k = rotate(k, positions, theta)
        q = None if q is None else rotate(q, positions, theta)
    k_pages, v_pages = np.array(k_pages, np.float64), np.array(v_pages, np.float64)
    pages, page = k_pages.shape[:2]
    bad = False
    for t, s in enumerate(np.asarray(slots)):
        if s < 0:
            continue
        if s >= pages * page:
            bad = True
            continue
        k_pages[s // page, s % page], v_pages[s // page, s % page] = k[t], v[t]
    return q, k_pages, v_pages, bad


def sequence_rows(pages, table_row, length: int):
    """The first ``length`` rows that a sequence's pages hold, and which of them exist (rows of
    a page outside the pool do not)."""
    n_pages, page = pages.shape[:2]
    reach = len(table_row) * page
    j = np.arange(min(max(int(length), 0), reach))
    ids = np.asarray(table_row, dtype=np.int64)[j // page]
    there = (ids >= 0) & (ids < n_pages)
    return np.where(there[:, None, None], pages[np.where(there, ids, 0), j % page], 0.0), there


def paged_attention(q, k_pages, v_pages, page_table, lengths, scale: float):
    """(o, spread, bad): o (B, Hq, S, D); ``spread`` = sum of p |v|, what errors of p act on; bad:
    an index pointed outside its table."""
    q, k_pages, v_pages = (np.asarray(a, np.float64) for a in (q, k_pages, v_pages))
    b_, hq, s_, d = q.shape
    hkv, page = k_pages.shape[2], k_pages.shape[1]
    o, spread, bad = np.zeros_like(q), np.zeros_like(q), False
    for b in range(b_):
        n = int(lengths[b])
        bad |= n < 0 or n > page_table.shape[1] * page
        n = min(max(n, 0), page_table.shape[1] * page)
        k, there = sequence_rows(k_pages, page_table[b], n)
        v, _ = sequence_rows(v_pages, page_table[b], n)
        bad |= not there.all()
        for h in range(hq):
            for s in range(s_):
                m = n - s_ + s + 1
                if m <= 0 or not there[:m].any():
                    continue
                kk, vv = k[:m, h // (hq // hkv)][there[:m]], v[:m, h // (hq // hkv)][there[:m]]
                z = kk @ q[b, h, s] * scale
                p = np.exp(z - z.max())
                p /= p.sum()
                o[b, h, s], spread[b, h, s] = p @ vv, p @ np.abs(vv)
    return o, spread, bad


def sample_row(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, log-probability) of one row of logits."""
    x = np.asarray(x, np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    top = x.max()
    if top == -np.inf:
        return -1, -np.inf
    first = int(np.argmax(x))
    if not temperature > 0:
        return first, 0.0
    with np.errstate(invalid="ignore"):
        w = np.where(x == top, 1.0, np.where(x == -np.inf, 0.0, np.nan_to_num(np.exp((x - top) / float(temperature)), nan=0.0)))
    ids = np.lexsort((np.arange(x.size), -x))
    if 0 < top_k < x.size:
        ids = ids[:top_k]
    if top_p < 1:
        c = np.cumsum(w[ids])
        ids = ids[: max(1, int(np.searchsorted(c, float(top_p) * c[-1], side="left")) + 1)]
    if min_p > 0:
        ids = ids[(w[ids] >= float(min_p)) | (x[ids] == top)]
    ids = np.sort(ids)
    ids = ids[w[ids] > 0]
    c = np.cumsum(w[ids])
    if not u > 0:
        at = 0
    else:
        at = min(int(np.searchsorted(c, float(u) * c[-1], side="right")), ids.size - 1) if u < 1 else ids.size - 1
    return int(ids[at]), float(np.log(w[ids[at]] / c[-1]))


def sample(logits, uniform, temperature=None, top_k=None, top_p=None, min_p=None):
    n = len(logits)
    setting = lambda a, off: [off] * n if a is None else list(np.asarray(a))
    rows = [sample_row(*a) for a in zip(logits, uniform, setting(temperature, 1.0), setting(top_k, 0), setting(top_p, 1.0), setting(min_p, 0.0))]
    return np.array([t for t, _ in rows], np.int64), np.array([p for _, p in rows], np.float64)
