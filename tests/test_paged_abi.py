"""Paged cache entry points without a GPU: what they refuse before any launch,
their workspace sizes, and the binding's and the wrappers' own refusals."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import cmpext3
from cmpext3 import abi
from oracle import paged_oracle as po

A = 1 << 32  # stands for every tensor: nothing on the host reads it
vp, ci = ctypes.c_void_p, ctypes.c_int


def s3(*s):
    return (ctypes.c_int64 * 3)(*s)


def attn(dt=1, B=2, H=4, Hkv=2, S=1, D=64, P=10, page=16, q=A, kp=A, v=A, o=A, qs=None, kps=None, vps=None, os=None,
         table=A, width=3, stride=3, lens=A, new=None, sel=None, nsel=0, scale=0.125, ws=None, wsb=0):
    pool = s3(Hkv * page * D, page * D, D)
    rows = s3(H * S * D, S * D, D)
    return abi.lib().cmpext3_paged_attn(vp(q), vp(kp), vp(v), vp(o), dt, B, H, Hkv, S, D, P, page, qs or rows,
                                        kps or pool, vps or pool, os or rows, vp(table), width, stride, vp(lens),
                                        vp(new), vp(sel), nsel, ctypes.c_float(scale), vp(ws), wsb, None)


def append(dt=1, B=2, H=4, Hkv=2, S=1, D=64, P=10, page=16, k=A, v=A, q=None, qo=None, kp=A, vpg=A, kb=None, ks=None,
           kps=None, kbs=None, table=A, width=3, stride=3, lens=A, new=None, pos=None, cos=None, sin=None, rows=0,
           rot=0, rs=0):
    pool, r, e = s3(Hkv * page * D, page * D, D), s3(Hkv * S * D, S * D, D), s3(Hkv * 2 * D, 2 * D, D)
    qr = s3(H * S * D, S * D, D)
    return abi.lib().cmpext3_paged_append(*map(vp, (k, v, q, qo, kp, vpg, kb)), dt, B, H, Hkv, S, D, P, page, ks or r, r,
                                          qr, qr, kps or pool, pool, kbs or e, vp(table), width, stride,
                                          *map(vp, (lens, new, pos, cos, sin)), rows, rot, rs, 0, None)


def select(dt=1, B=2, H=4, Hkv=2, D=64, P=10, page=16, q=A, kb=A, out=A, qs=None, kbs=None, table=A, width=3, stride=3,
           lens=A, n=2, ws=A, wsb=1 << 20):
    return abi.lib().cmpext3_paged_select(vp(q), vp(kb), vp(out), dt, B, H, Hkv, D, P, page, qs or s3(H * D, D, D),
                                          kbs or s3(Hkv * 2 * D, 2 * D, D), vp(table), width, stride, vp(lens), n,
                                          vp(ws), wsb, None)


INV, DT, HD, AL, BIG = abi.E_INVALID, abi.E_DTYPE, abi.E_HEAD_DIM, abi.E_ALIGN, abi.E_TOO_LARGE


@pytest.mark.parametrize("args,code", [
    (dict(dt=3), DT), (dict(dt=-1), DT), (dict(B=-1), INV), (dict(H=5), INV), (dict(Hkv=0), INV), (dict(P=0), INV),
    (dict(page=0), INV), (dict(width=-1), INV), (dict(D=60), HD), (dict(D=264), HD), (dict(D=0), HD),
    (dict(dt=2, D=6), HD), (dict(S=17), BIG), (dict(width=1 << 30), BIG), (dict(B=1 << 30), BIG),
    (dict(scale=float("inf")), INV), (dict(scale=float("nan")), INV), (dict(sel=A, nsel=0), INV),
    (dict(q=0), INV), (dict(o=0), INV), (dict(kp=0), INV), (dict(v=0), INV), (dict(lens=0), INV), (dict(table=0), INV),
    (dict(q=A + 2), AL), (dict(o=A + 8), AL), (dict(kp=A + 4), AL), (dict(lens=A + 2), AL), (dict(table=A + 1), AL),
    (dict(new=A + 1), AL), (dict(sel=A + 2, nsel=1), AL), (dict(ws=A + 8, wsb=99999), AL),
    (dict(qs=s3(256, 64, -64), S=2), INV), (dict(qs=s3(256, 68, 64)), AL), (dict(kps=s3(2048, 1024, 32)), INV),
    (dict(kps=s3(2048, 1024, 0)), INV), (dict(vps=s3(2048, 1024, 68)), AL), (dict(vps=s3(2048, 1024, 1 << 27)), BIG),
    (dict(kps=s3(-2048, 1024, 64)), INV), (dict(stride=-3), INV), (dict(sel=A, nsel=1 << 28), BIG),
])
def test_attention_refuses_before_launch(args, code):
    assert attn(**args) == code


@pytest.mark.parametrize("args,code", [
    (dict(dt=3), DT), (dict(Hkv=0), INV), (dict(D=20), HD), (dict(P=0), INV), (dict(k=0), INV), (dict(v=0), INV),
    (dict(kp=0), INV), (dict(vpg=0), INV), (dict(lens=0), INV), (dict(k=A + 2), AL), (dict(kb=A + 2), AL),
    (dict(kbs=s3(256, 132, 64), kb=A), AL), (dict(q=A), INV), (dict(qo=A), INV), (dict(q=A, qo=A + 4096), INV),
    (dict(cos=A), INV), (dict(sin=A), INV), (dict(cos=A, sin=A, rows=4, rot=63), INV),
    (dict(cos=A, sin=A, rows=4, rot=66), INV), (dict(cos=A, sin=A, rows=0, rot=64), INV),
    (dict(cos=A, sin=A, rows=4, rot=0), INV), (dict(cos=A + 2, sin=A, rows=4, rot=64, rs=32), AL),
    (dict(cos=A, sin=A, rows=4, rot=64, rs=-32), INV), (dict(cos=A, sin=A, rows=4, rot=64, rs=32, q=A, qo=A), INV),
    (dict(cos=A, sin=A, rows=4, rot=64, rs=32, q=A, qo=A + 4096, H=3), INV), (dict(pos=A + 1), AL),
    (dict(B=1 << 27), BIG), (dict(Hkv=1 << 28, B=1), BIG), (dict(S=1 << 20, page=1, B=16, kb=A), BIG), (dict(ks=s3(128, 64, -1), S=3), INV),
])
def test_append_refuses_before_launch(args, code):
    assert append(**args) == code


@pytest.mark.parametrize("args,code", [
    (dict(dt=3), DT), (dict(H=5), INV), (dict(D=20), HD), (dict(P=0), INV), (dict(page=0), INV), (dict(n=0), INV),
    (dict(q=0), INV), (dict(kb=0), INV), (dict(out=0), INV), (dict(lens=0), INV), (dict(ws=0), INV),
    (dict(wsb=8), INV), (dict(ws=A + 8), AL), (dict(out=A + 2), AL), (dict(q=A + 2), AL),
    (dict(kbs=s3(256, 128, 68)), AL), (dict(width=1 << 28), BIG), (dict(n=1 << 30), BIG),
])
def test_select_refuses_before_launch(args, code):
    assert select(**args) == code


def test_nothing_to_do_is_no_error_even_without_pointers():
    none = dict(q=0, lens=0, table=0, width=0)
    assert attn(B=0, kp=0, v=0, o=0, **none) == abi.OK
    assert attn(S=0, kp=0, v=0, o=0, **none) == abi.OK
    assert append(B=0, k=0, v=0, kp=0, vpg=0, lens=0, table=0) == abi.OK
    assert append(S=0, k=0, v=0, kp=0, vpg=0, lens=0, table=0) == abi.OK
    assert select(B=0, kb=0, out=0, **none) == abi.OK


def test_workspace_sizes():
    size = abi.lib().cmpext3_paged_attn_workspace_size
    assert size(7, 2, 4, 2, 1, 64, 16, 100, 0) == 0 and size(1, 2, 4, 2, 17, 64, 16, 100, 0) == 0
    assert size(1, 0, 4, 2, 1, 64, 16, 100, 0) == 0 and size(1, 2, 4, 2, 1, 64, 16, 0, 0) == 0
    assert abi.lib().cmpext3_paged_select_workspace_size(2, 3, 100) >= 2 * 3 * 100 * 8
    assert abi.lib().cmpext3_paged_select_workspace_size(2, 3, 0) == 0


def test_cpu_tensors_are_refused():
    q, kp = torch.zeros(2, 4, 1, 64), torch.zeros(5, 2, 16, 64)
    t, n = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    for call in (lambda: cmpext3.paged_attention(q, kp, kp, t, n),
                 lambda: cmpext3.paged_append(q[:, :2], q[:, :2], kp, kp.clone(), t, n),
                 lambda: cmpext3.paged_select(q, torch.zeros(5, 2, 2, 64), t, n, 16, 2)):
        with pytest.raises(RuntimeError, match="GPU"):
            call()


def test_the_float64_restatement_is_plain_attention():
    """The oracle itself: over an identity table it is softmax attention with a causal corner, and its page scores
    bound every key's product."""
    g = torch.Generator().manual_seed(0)
    q = torch.randn(1, 4, 3, 8, generator=g, dtype=torch.float64)
    kp, v = (torch.randn(4, 2, 5, 8, generator=g, dtype=torch.float64) for _ in range(2))
    table, lens = torch.arange(4, dtype=torch.int32)[None], torch.tensor([18], dtype=torch.int32)
    out, wt, _ = po.attention(q, kp, v, table, lens, 0.3)
    k1, v1 = (t.transpose(0, 1).reshape(2, 20, 8)[:, :18].repeat_interleave(2, 0)[None] for t in (kp, v))
    mask = torch.ones(3, 18, dtype=torch.bool).tril(15)
    want = torch.nn.functional.scaled_dot_product_attention(q, k1, v1, attn_mask=mask, scale=0.3)
    assert np.allclose(out, want.numpy(), atol=1e-12) and (wt >= abs(out) - 1e-12).all()
    bounds = torch.stack([kp.amin(2), kp.amax(2)], 2)
    picked = po.select(q[:, :, :1], bounds, table, lens, 5, 2)
    scores = [sum(np.maximum(po.f64(q)[0, h, 0] * po.f64(bounds)[p, 0, 0],
                             po.f64(q)[0, h, 0] * po.f64(bounds)[p, 0, 1]).sum() for h in range(2)) for p in range(3)]
    assert picked[0, 0].tolist() == sorted([int(np.argmax(scores)), 3])
    products = torch.einsum("hd,psd->phs", q[0, :2, 0], kp[:3, 0]).sum(1).amax(1)
    assert (np.array(scores) >= products.numpy() - 1e-12).all()
