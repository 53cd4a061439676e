"""Inputs and tolerances shared by the tests of the paged cache's operators."""
from __future__ import annotations

import numpy as np
import torch

from oracle import paged_oracle as po

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
U32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(DTYPES[dtype]).eps / 2


class Cache:
    """A pool whose slots hold NaN until a sequence owns them, and the tables of
    sequences of the given lengths over randomly ordered pages (columns behind a
    sequence's last page name no page)."""

    def __init__(self, dtype, lens, Hkv, D, page, seed=0, spare=3, layout="hps", width=None, device="cuda"):
        g = torch.Generator().manual_seed(seed)
        per = [-(-max(n, 0) // page) for n in lens]
        P = sum(per) + spare
        self.page, self.Hkv, self.D, self.dtype = page, Hkv, D, DTYPES[dtype]
        order = torch.randperm(P, generator=g)
        M = max(per + [0]) if width is None else width
        table = torch.full((len(lens), M), -7, dtype=torch.int32)
        at = 0
        for b, n in enumerate(per):
            table[b, :min(n, M)] = order[at:at + n][:M]
            at += n
        shape = (P, Hkv, page, D)
        self.kp, self.vp = (torch.full(shape, float("nan")) for _ in range(2))
        for b, n in enumerate(lens):
            for j in range(min(max(n, 0), M * page)):
                p = table[b, j // page]
                self.kp[p, :, j % page] = torch.randn(Hkv, D, generator=g)
                self.vp[p, :, j % page] = torch.randn(Hkv, D, generator=g)
        move = (lambda t: t.transpose(1, 2).contiguous().to(device).transpose(1, 2)) if layout == "psh" \
            else (lambda t: t.to(device))
        self.kp, self.vp = move(self.kp.to(self.dtype)), move(self.vp.to(self.dtype))
        self.table = table.to(device)
        self.lens = torch.tensor(lens, dtype=torch.int32, device=device)
        self.g = g

    def rows(self, heads, S, device="cuda", std=1.0):
        """[B, heads, S, D] as a projection leaves it."""
        x = torch.randn(len(self.lens), S, heads, self.D, generator=self.g) * std
        return x.to(self.dtype).to(device).transpose(1, 2)


def check_attention(dtype, got, q, cache, scale, new_lens=None, selected=None):
    """Against the float64 attention.  An output is off by its own rounding, by
    its weights' relative error times the sum of p |v| behind it, and by the fp32
    sums: a score of D products is off by at most (D + 8) half steps of its sum
    of magnitudes, which moves every weight by twice that; weights are rounded
    once to the tensors' type (numerator and the sum of the rounded ones: two
    half steps) and n products are summed."""
    want, wt, top = po.attention(q, cache.kp, cache.vp, cache.table, cache.lens, scale, new_lens, selected)
    u = half_step(dtype)
    n = max([int(x) for x in cache.lens.cpu()] + [1])
    D = q.shape[-1]
    rel = 2 * (D + 8) * U32 * top[..., None] + 2 * (n + 64) * U32 + (0 if dtype == "fp32" else 2 * u)
    tol = u * np.abs(want) + 1.01 * rel * wt + (2.0 ** -24 if dtype == "fp16" else 0)
    g = po.f64(got)
    assert got.dtype == q.dtype and got.shape == q.shape
    assert np.array_equal(np.isnan(g), np.isnan(want)), "NaN rows"
    err = np.abs(g - want)
    bad = np.nan_to_num(err - tol, nan=0.0) > 0
    assert not bad.any(), f"{bad.sum()} values off, worst by {np.nanmax(err):.3e} (tolerance {np.nanmin(tol):.1e}..)"
    assert (g[want == 0] == 0).all() or not (wt == 0).any()


def tables(rows, rot, device="cuda", theta=10000.0):
    inv = theta ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    a = torch.arange(rows, dtype=torch.float64)[:, None] * inv
    return a.cos().float().to(device), a.sin().float().to(device)
