"""Float64 restatement of the paged key-value cache's operators, used as the
oracle on the CPU: plain loops over sequences, heads and tokens, following
include/cmpext3_paged.h word for word."""
from __future__ import annotations

import numpy as np
import torch


def f64(t: torch.Tensor) -> np.ndarray:
    return t.detach().cpu().to(torch.float64).numpy()


def new_count(b, S, lens, new_lens):
    n = S if new_lens is None else min(max(int(new_lens[b]), 0), S)
    return min(n, max(int(lens[b]), 0))


def page_of(table, b, col, num_pages):
    """The page in a column of a sequence's table row, None when there is none."""
    if col < 0 or col >= table.shape[1]:
        return None
    p = int(table[b, col])
    return p if 0 <= p < num_pages else None


def rotate(x, cos, sin, interleaved):
    """x [..., D] rotated in its first 2 * len(cos) channels; also the sum of the
    magnitudes that each result is made of."""
    R = 2 * len(cos)
    out, mag = x.copy(), np.abs(x)
    for j in range(R // 2):
        a, b = (2 * j, 2 * j + 1) if interleaved else (j, j + R // 2)
        out[..., a] = x[..., a] * cos[j] - x[..., b] * sin[j]
        out[..., b] = x[..., b] * cos[j] + x[..., a] * sin[j]
        mag[..., a] = np.abs(x[..., a] * cos[j]) + np.abs(x[..., b] * sin[j])
        mag[..., b] = np.abs(x[..., b] * cos[j]) + np.abs(x[..., a] * sin[j])
    return out, mag


def append(key, value, num_pages, page_size, table, lens, query=None, cos=None, sin=None, positions=None,
           new_lens=None, interleaved=False):
    """What the call writes: {(page, slot): (keys, their magnitudes, values)} with rows [Hkv, D], the rotated
    queries with their magnitudes (NaN rows for tokens not stored), and the set
    of (page, slot 0 written?) touched."""
    k, v = f64(key), f64(value)
    q = None if query is None else f64(query)
    B, _, S, _ = k.shape
    table, lens = table.cpu().numpy(), lens.cpu().numpy()
    c, s = (None, None) if cos is None else (f64(cos), f64(sin))
    out = None if q is None else np.zeros_like(q)
    mag = None if q is None else np.zeros_like(q)
    writes = {}
    for b in range(B):
        n = new_count(b, S, lens, new_lens)
        for i in range(n):
            pos = int(lens[b]) - n + i
            page = page_of(table, b, pos // page_size, num_pages)
            row = pos if positions is None else int(positions[b, i])
            ok = page is not None and (c is None or 0 <= row < c.shape[0])
            if not ok:
                if q is not None:
                    out[b, :, i] = np.nan
                continue
            kk, km = (k[b, :, i], 0 * k[b, :, i]) if c is None else rotate(k[b, :, i], c[row], s[row], interleaved)
            writes[(page, pos % page_size)] = (kk, km, v[b, :, i])
            if q is not None:
                out[b, :, i], mag[b, :, i] = rotate(q[b, :, i], c[row], s[row], interleaved)
    return writes, out, mag


def attention(query, key_pages, value_pages, table, lens, scale, new_lens=None, selected=None):
    """(out, weighted, top): the attention [B, H, S, D], the sum of p |v| behind
    each value, and each row's largest sum of |q k| (times |scale|)."""
    q, kp, vp = f64(query), f64(key_pages), f64(value_pages)
    B, H, S, D = q.shape
    P, Hkv, page_size, _ = kp.shape
    table, lens = table.cpu().numpy(), lens.cpu().numpy()
    out, wt = np.zeros_like(q), np.zeros_like(q)
    top = np.zeros((B, H, S))
    for b in range(B):
        n, length = new_count(b, S, lens, new_lens), max(int(lens[b]), 0)
        pages = -(-length // page_size)
        for hk in range(Hkv if n else 0):  # only padding: zeros
            cols = range(pages) if selected is None else [int(x) for x in selected[b, hk] if int(x) >= 0]
            at = [page_of(table, b, c, P) if c < pages else None for c in cols]
            heads = slice(hk * H // Hkv, (hk + 1) * H // Hkv)
            if length and (None in at or length > table.shape[1] * page_size):
                out[b, heads] = np.nan
                continue
            keys, vals, place = [], [], []
            for c, p in zip(cols, at):
                live = min(page_size, length - c * page_size)
                keys.append(kp[p, hk, :live]); vals.append(vp[p, hk, :live])
                place.append(c * page_size + np.arange(live))
            if not keys:
                continue
            keys, vals, place = np.concatenate(keys), np.concatenate(vals), np.concatenate(place)
            for i in range(n):
                seen = place <= length - n + i
                if not seen.any():
                    continue
                for h in range(heads.start, heads.stop):
                    x = keys[seen] @ q[b, h, i] * scale
                    e = np.exp(x - x.max())
                    p = e / e.sum()
                    out[b, h, i] = p @ vals[seen]
                    wt[b, h, i] = p @ np.abs(vals[seen])
                    top[b, h, i] = (np.abs(keys[seen]) @ np.abs(q[b, h, i])).max() * abs(scale)
    return out, wt, top


def select(query, key_bounds, table, lens, page_size, n_selected):
    q, e = f64(query), f64(key_bounds)
    B, H, _, _ = q.shape
    P, Hkv = e.shape[:2]
    table, lens = table.cpu().numpy(), lens.cpu().numpy()
    out = np.full((B, Hkv, n_selected), -1, dtype=np.int32)
    for b in range(B):
        pages = min(-(-max(int(lens[b]), 0) // page_size), table.shape[1])
        for hk in range(Hkv):
            scores = []
            for c in range(pages - 1):
                p = page_of(table, b, c, P)
                s = np.inf
                if p is not None:
                    g = q[b, hk * H // Hkv:(hk + 1) * H // Hkv, 0]
                    with np.errstate(invalid="ignore"):  # a channel without a part counts as 0, whatever its bound
                        up, down = np.maximum(g, 0).sum(0), np.minimum(g, 0).sum(0)
                        s = (np.where(up == 0, 0, up * e[p, hk, 1]) + np.where(down == 0, 0, down * e[p, hk, 0])).sum()
                    s = np.inf if np.isnan(s) else s
                scores.append((-s, c))
            got = sorted(c for _, c in sorted(scores)[:n_selected - 1]) + ([pages - 1] if pages else [])
            out[b, hk, :len(got)] = got
    return out
