"""GPU tests of the paged cache's operators against their float64 restatement."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import cmpext3
from cmpext3 import abi
from oracle import paged_oracle as po
from paged_cases import DTYPES, U32, Cache, check_attention, half_step, tables

pytestmark = pytest.mark.gpu

# dtype, lens, H, Hkv, D, page, S, layout
ATTENTION = [
    ("bf16", [300], 16, 8, 128, 16, 1, "hps"),
    ("bf16", [1, 15, 16, 17, 0, 33, 64, 1000], 16, 8, 128, 16, 1, "hps"),
    ("fp16", [5, 0, 129, 700, 31, 64], 8, 2, 64, 32, 1, "psh"),
    ("fp32", [5, 0, 129, 300, 31, 64], 8, 2, 64, 16, 1, "psh"),
    ("fp32", [1, 2, 77, 250], 6, 3, 40, 24, 3, "hps"),
    ("fp32", [513, 100], 4, 1, 256, 16, 1, "hps"),
    ("fp32", [513, 100], 4, 4, 4, 16, 1, "hps"),
    ("fp16", [65, 130, 7], 5, 5, 80, 24, 4, "psh"),
    ("bf16", [90, 33], 4, 2, 96, 8, 2, "hps"),
    ("bf16", [90, 33], 4, 2, 160, 1, 1, "hps"),
    ("fp16", [190, 33], 4, 2, 192, 40, 1, "hps"),
    ("bf16", [2100, 16], 4, 2, 256, 64, 1, "hps"),
    ("bf16", [2100, 16], 2, 1, 8, 128, 1, "hps"),
    ("bf16", [400, 17, 0], 64, 2, 128, 16, 1, "hps"),     # 32 query heads a key head
    ("fp16", [400, 17, 16], 20, 1, 64, 16, 16, "hps"),    # 320 rows of one key head
    ("bf16", [33, 70], 6, 2, 72, 16, 5, "psh"),
    ("bf16", [20011, 3], 8, 1, 64, 16, 1, "hps"),         # one long, one short
    ("fp16", [1] * 70, 2, 1, 64, 16, 1, "hps"),           # more sequences than lanes
    ("bf16", [(37 * b) % 200 for b in range(300)], 4, 2, 64, 16, 1, "hps"),
]


@pytest.mark.parametrize("case", ATTENTION, ids=lambda c: f"{c[0]}-{max(c[1])}x{len(c[1])}-h{c[2]}.{c[3]}-d{c[4]}-p{c[5]}-s{c[6]}-{c[7]}")
def test_attention(case):
    dtype, lens, H, Hkv, D, page, S, layout = case
    c = Cache(dtype, lens, Hkv, D, page, seed=len(lens), layout=layout)
    q = c.rows(H, S)
    out = cmpext3.paged_attention(q, c.kp, c.vp, c.table, c.lens)
    check_attention(dtype, out, q, c, D ** -0.5)
    again = cmpext3.paged_attention(q, c.kp, c.vp, c.table, c.lens)
    assert torch.equal(out, again)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0])
def test_attention_scales(dtype, scale):
    c = Cache(dtype, [100, 37], 2, 64, 16)
    q = c.rows(4, 1)
    check_attention(dtype, cmpext3.paged_attention(q, c.kp, c.vp, c.table, c.lens, scale), q, c, scale)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_attention_of_padded_blocks(dtype):
    """new_lens: later columns are padding; more new tokens than the sequence holds are the first ones it holds."""
    c = Cache(dtype, [40, 3, 0, 100, 7], 2, 64, 16)
    q = c.rows(4, 6)
    new = torch.tensor([2, 6, 4, 0, -1], dtype=torch.int32, device="cuda")
    out = cmpext3.paged_attention(q, c.kp, c.vp, c.table, c.lens, 0.125, new_lens=new)
    check_attention(dtype, out, q, c, 0.125, new.cpu())
    assert (out[0, :, 2:] == 0).all() and (out[2:] == 0).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("page,S", [(16, 1), (32, 1), (24, 3)])
def test_attention_over_selected_pages(dtype, page, S):
    lens = [500, 40, 0, 1, 333]
    c = Cache(dtype, lens, 3, 64, page)
    g = torch.Generator().manual_seed(3)
    sel = torch.full((len(lens), 3, 7), -1, dtype=torch.int32)
    for b, n in enumerate(lens):
        pages = -(-n // page)
        for h in range(3):
            pick = torch.randperm(max(pages, 1), generator=g)[:min(5, pages)].to(torch.int32)
            sel[b, h, 1:1 + len(pick)] = pick  # any order, -1 at both ends
    sel[0, 1] = -1  # a head that attends to nothing
    q = c.rows(6, S)
    out = cmpext3.paged_attention(q, c.kp, c.vp, c.table, c.lens, selected=sel.cuda())
    check_attention(dtype, out, q, c, 0.125, None, sel)
    assert (out[0, 2:4] == 0).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_bad_pages_make_nan_rows_of_their_sequence_alone(dtype):
    c = Cache(dtype, [100, 100, 100, 100, 60], 2, 64, 16, width=5)  # 100 tokens: 7 pages, past the row
    c.lens = torch.tensor([80, 100, 80, 80, 60], dtype=torch.int32, device="cuda")
    c.table[2, 1], c.table[3, 4] = -1, c.kp.shape[0]
    q = c.rows(4, 1)
    out = cmpext3.paged_attention(q, c.kp, c.vp, c.table, c.lens)
    check_attention(dtype, out, q, c, 0.125)
    assert out[1:4].isnan().all() and not out[0].isnan().any() and not out[4].isnan().any()
    sel = torch.tensor([[[0], [2]], [[0], [2]], [[0], [1]], [[4], [0]], [[4], [3]]], dtype=torch.int32, device="cuda")
    out = cmpext3.paged_attention(q, c.kp, c.vp, c.table, c.lens, selected=sel)  # page 4 is none of 60 tokens
    check_attention(dtype, out, q, c, 0.125, None, sel.cpu())
    assert out[4, :2].isnan().all() and not out[4, 2:].isnan().any()


def test_lengths_past_every_bound_are_refused_rows():
    c = Cache("bf16", [30, 30, 30], 1, 64, 16)
    c.lens = torch.tensor([2 ** 31 - 1, -2 ** 31, 30], dtype=torch.int32, device="cuda")
    q = c.rows(2, 1)
    out = cmpext3.paged_attention(q, c.kp, c.vp, c.table, c.lens)
    assert out[0].isnan().all() and (out[1] == 0).all() and out[2].isfinite().all()
    k = c.rows(1, 1)
    before = c.kp.clone()
    cos, sin = tables(64, 64)
    got = cmpext3.paged_append(k, k, c.kp, c.vp, c.table, c.lens, query=q, cos=cos, sin=sin)
    assert got[0].isnan().all() and (got[1] == 0).all() and got[2].isfinite().all()
    changed = ~((c.kp == before) | (c.kp.isnan() & before.isnan())).flatten(2).all(-1).flatten()
    assert changed.nonzero().flatten().tolist() == [int(c.table[2, 1])]


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_infinite_and_low_scores(dtype):
    """A key that outweighs all others, scores below any exponent, and the type's lowest values in V."""
    c = Cache(dtype, [70, 70], 1, 64, 16)
    p = int(c.table[0, 2])
    c.kp[p, 0, 3] = 50.0
    c.vp[p, 0, 3] = torch.finfo(c.dtype).min / 4
    q = c.rows(2, 1)
    q[0] = 3.0
    q[1] = -30.0
    out = cmpext3.paged_attention(q, c.kp, c.vp, c.table, c.lens, 1.0)
    check_attention(dtype, out, q, c, 1.0)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("D,H", [(64, 4), (128, 20), (256, 2)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_values_of_later_tokens_reach_no_earlier_one(dtype, D, H, bad):
    """A NaN or an infinity in a new token's V is its own row's and the later ones'; padding columns stay zero
    whatever V holds."""
    c = Cache(dtype, [37, 70, 100], 2, D, 16)
    q = c.rows(H, 6)
    c.vp[c.table[0, 34 // 16].long(), :, 34 % 16, 5] = bad   # token 34: column 3 of 6
    c.vp[c.table[1, 0].long(), 1, 2, D - 1] = bad            # an old token: every row of its head
    c.vp[c.table[2, 99 // 16].long(), 0, 99 % 16, 0] = bad   # the last of three
    new = torch.tensor([6, 4, 3], dtype=torch.int32, device="cuda")
    out = cmpext3.paged_attention(q, c.kp, c.vp, c.table, c.lens, 0.1, new_lens=new)
    got = po.f64(out)
    want, wt, top = po.attention(q, c.kp, c.vp, c.table, c.lens, 0.1, new.cpu())
    assert np.array_equal(np.isfinite(got), np.isfinite(want))
    assert np.array_equal(np.isnan(got), np.isnan(want)) and (got[np.isinf(want)] == want[np.isinf(want)]).all()
    assert (got[1, :, 4:] == 0).all() and (got[2, :, 3:] == 0).all()
    ok = np.isfinite(want)
    u = half_step(dtype)
    rel = 2 * (D + 8) * U32 * top[..., None] + 2 * (100 + 64) * U32 + (0 if dtype == "fp32" else 2 * u)
    tol = u * np.abs(want[ok]) + (1.01 * rel * wt)[ok] + 2.0 ** -24
    assert (np.abs(got[ok] - want[ok]) <= tol).all()


def test_attention_past_32_bit_offsets():
    """Pages beyond 4 GiB into the pool."""
    P, Hkv, page, D = 40000, 8, 32, 256  # 5.2 GB for K, the same memory for V
    pool = torch.zeros(P, Hkv, page, D, dtype=torch.bfloat16, device="cuda")
    c = Cache("bf16", [200, 77], Hkv, D, page)
    far = c.kp.shape[0]
    pool[P - far:] = c.kp
    table = torch.where(c.table >= 0, c.table + (P - far), c.table)
    q = c.rows(16, 1)
    want = cmpext3.paged_attention(q, c.kp, c.kp, c.table, c.lens)
    got = cmpext3.paged_attention(q, pool, pool, table, c.lens)
    assert torch.equal(got, want)
    k, v = c.rows(Hkv, 1), c.rows(Hkv, 1)
    small = c.kp.clone()
    cmpext3.paged_append(k, v, small, small.clone(), c.table, c.lens)
    cmpext3.paged_append(k, v, pool, pool.new_empty(0).new_zeros(pool.shape), table, c.lens)
    assert torch.equal(pool[P - far:].view(torch.int16), small.view(torch.int16))


# dtype, lens (with the new tokens), new_lens or None, S, H, Hkv, D, page, rot, pairs, bounds, layout
APPEND = [
    ("bf16", [40, 1, 0, 300, 16, 17], None, 1, 16, 8, 128, 16, 128, False, True, "hps"),
    ("bf16", [100, 130], None, 100, 4, 2, 128, 16, 128, False, True, "hps"),
    ("fp16", [70, 37, 1, 50], [33, 37, 1, 0], 37, 5, 5, 80, 24, 40, True, False, "psh"),
    ("fp16", [70, 37, 5, 50], [33, 20, 9, -3], 37, 4, 2, 72, 24, 72, False, True, "psh"),
    ("fp32", [64, 20], None, 20, 2, 2, 64, 16, 64, False, True, "hps"),
    ("fp32", [64, 20], [1, 3], 3, 4, 1, 40, 1, 20, True, True, "hps"),
    ("fp32", [64, 20], None, 7, 4, 1, 256, 128, 256, False, False, "hps"),
    ("bf16", [300, 270], None, 260, 2, 1, 256, 256, 256, False, True, "hps"),
    ("bf16", [90], None, 80, 3, 3, 8, 16, 6, True, True, "psh"),
    ("fp16", [90], None, 80, 3, 3, 24, 8, 12, False, True, "hps"),
    ("bf16", [600, 90], None, 90, 3, 3, 160, 512, 0, False, True, "hps"),
    ("fp16", [30, 31], None, 2, 3, 3, 128, 16, 2, False, False, "hps"),
]


@pytest.mark.parametrize("case", APPEND, ids=lambda c: f"{c[0]}-{max(c[1])}x{len(c[1])}-s{c[3]}-h{c[4]}.{c[5]}-d{c[6]}-p{c[7]}-r{c[8]}{'i' if c[9] else ''}{'b' if c[10] else ''}-{c[11]}")
@pytest.mark.parametrize("own_positions", [False, True])
def test_append(case, own_positions):
    dtype, lens, new, S, H, Hkv, D, page, rot, pairs, bounds, layout = case
    c = Cache(dtype, lens, Hkv, D, page, seed=S, layout=layout)
    k, v = c.rows(Hkv, S), c.rows(Hkv, S)
    q = c.rows(H, S) if rot else None
    cos, sin = tables(max(lens) + 5, rot) if rot else (None, None)
    nl = None if new is None else torch.tensor(new, dtype=torch.int32, device="cuda")
    positions = None
    if own_positions and rot:
        positions = torch.randint(0, max(lens) + 5, (len(lens), S), generator=c.g).to(torch.int32).cuda()
    kb = None
    if bounds:  # of what the pages hold (NaN slots hold nothing)
        lo = torch.where(c.kp.isnan(), torch.inf, c.kp.float()).amin(2, keepdim=True)
        hi = torch.where(c.kp.isnan(), -torch.inf, c.kp.float()).amax(2, keepdim=True)
        kb = torch.cat([lo, hi], 2).to(c.dtype)
    kp0, vp0, kb0 = c.kp.clone(), c.vp.clone(), None if kb is None else kb.clone()
    got = cmpext3.paged_append(k, v, c.kp, c.vp, c.table, c.lens, query=q, cos=cos, sin=sin, positions=positions,
                               new_lens=nl, interleaved=pairs, key_bounds=kb)
    writes, want_q, mag_q = po.append(k, v, kp0.shape[0], page, c.table, c.lens, q, cos, sin, positions, new, pairs)
    u = half_step(dtype)

    def close(a, want, mag, what):  # one rounding, after two products and a sum in fp32
        a = po.f64(a)
        assert np.array_equal(np.isnan(a), np.isnan(want)), what
        tiny = 2.0 ** -25 if dtype == "fp16" else 0.0  # half a subnormal step
        off = np.nan_to_num(np.abs(a - want) - (u * np.abs(want) + 3 * U32 * mag * (1 + u) + tiny))
        assert (off <= 0).all(), f"{what}: {np.nanmax(np.abs(a - want))}"

    if q is not None:
        assert got.shape == q.shape and got.dtype == q.dtype
        close(got, want_q, mag_q, "query")
    else:
        assert got is None
    written = torch.zeros(kp0.shape[0], page, dtype=torch.bool)
    for (p, s), (kk, km, vv) in writes.items():
        written[p, s] = True
        close(c.kp[p, :, s], kk, km, "key")
        assert np.array_equal(po.f64(c.vp[p, :, s]), vv), "value"
    keep = ~written.cuda()[:, None, :, None].expand_as(kp0)
    assert torch.equal(c.kp[keep].nan_to_num(9.0), kp0[keep].nan_to_num(9.0)), "another slot's key changed"
    assert torch.equal(c.vp[keep].nan_to_num(9.0), vp0[keep].nan_to_num(9.0)), "another slot's value changed"
    if kb is not None:
        touched = {p for p, _ in writes}
        for p in range(kp0.shape[0]):
            if p not in touched:
                assert torch.equal(kb[p], kb0[p])
                continue
            x = c.kp[p, :, written[p]].float()
            lo, hi = x.amin(1), x.amax(1)
            if not written[p, 0]:
                lo, hi = torch.minimum(lo, kb0[p, :, 0].float()), torch.maximum(hi, kb0[p, :, 1].float())
            assert torch.equal(kb[p, :, 0].float(), lo) and torch.equal(kb[p, :, 1].float(), hi)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("S,page", [(1, 16), (5, 16), (40, 128)])
def test_bounds_leave_out_nan_keys(dtype, S, page):
    c = Cache(dtype, [90, S], 2, 64, page)
    k = c.rows(2, S)
    k[:, 0, S // 2] = float("nan")
    k[1, 1, 0] = float("inf")
    kb = torch.zeros(c.kp.shape[0], 2, 2, 64, dtype=c.dtype, device="cuda")
    kb[:, :, 0], kb[:, :, 1] = -0.5, 0.5
    was = kb.clone()
    cmpext3.paged_append(k, k, c.kp, c.vp, c.table, c.lens, key_bounds=kb)
    for b, n in enumerate([90, S]):
        for p in range((n - S) // page, -(-n // page)):
            first, last = max(p * page, n - S), min((p + 1) * page, n)
            x = k[b, :, first - n + S:last - n + S].float().cpu().numpy()
            lo, hi = np.fmin.reduce(x, axis=1, initial=np.inf), np.fmax.reduce(x, axis=1, initial=-np.inf)
            page_no = int(c.table[b, p])
            if first > p * page:
                lo, hi = np.fmin(lo, po.f64(was[page_no, :, 0])), np.fmax(hi, po.f64(was[page_no, :, 1]))
            assert np.array_equal(po.f64(kb[page_no, :, 0]), lo) and np.array_equal(po.f64(kb[page_no, :, 1]), hi)


def test_append_leaves_out_tokens_without_a_page_or_a_rotation_row():
    c = Cache("bf16", [40, 40, 40], 2, 64, 16, width=2)
    c.table[1, 1] = c.kp.shape[0] + 5
    k, v, q = c.rows(2, 12), c.rows(2, 12), c.rows(4, 12)
    cos, sin = tables(100, 64)
    pos = torch.arange(12, dtype=torch.int32, device="cuda").repeat(3, 1)
    pos[2, 0], pos[2, 3] = -1, 100
    c.lens = torch.tensor([40, 32, 32], dtype=torch.int32, device="cuda")  # tokens 28..39; 20..31; 20..31
    kp0 = c.kp.clone()
    got = cmpext3.paged_append(k, v, c.kp, c.vp, c.table, c.lens, query=q, cos=cos, sin=sin, positions=pos)
    lost = got.isnan().all(3).all(1)
    assert lost[0].tolist() == [i >= 4 for i in range(12)]
    assert lost[1].all()
    assert lost[2].tolist() == [i in (0, 3) for i in range(12)]
    assert not got[0, :, :4].isnan().any() and not got[2][:, [1, 2, 4, 11]].isnan().any()
    writes, _, _ = po.append(k, v, c.kp.shape[0], 16, c.table, c.lens, q, cos, sin, pos)
    changed = ~((c.kp == kp0) | (c.kp.isnan() & kp0.isnan())).all(3).all(1)
    assert {tuple(x) for x in changed.nonzero().tolist()} == set(writes)


# dtype, lens, H, Hkv, D, page, picked
SELECT = [
    ("bf16", [300], 16, 8, 128, 16, 4),
    ("bf16", [1, 0, 16, 17, 1000, 64], 16, 8, 128, 16, 5),
    ("fp16", [4000, 900, 33], 8, 2, 64, 8, 64),
    ("fp32", [400, 900, 33], 4, 4, 40, 16, 1),
    ("fp32", [400, 900, 33], 4, 1, 256, 24, 200),
    ("bf16", [20000, 100], 4, 1, 72, 1, 300),
    ("fp16", [9000, 9001], 2, 1, 8, 2, 17),
    ("bf16", [5000, 100], 20, 1, 256, 4, 1000),
]


def _bounds(c, P, lo=-1.0, hi=1.0):
    a = torch.randn(P, c.Hkv, 1, c.D, generator=c.g)
    w = torch.rand(P, c.Hkv, 1, c.D, generator=c.g)
    return torch.cat([a + lo * w, a + hi * w], 2).to(c.dtype).cuda()


class Tables:
    def __init__(self, dtype, lens, Hkv, D, page, seed=0):
        self.g = torch.Generator().manual_seed(seed)
        self.dtype, self.Hkv, self.D = DTYPES[dtype], Hkv, D
        per = [-(-n // page) for n in lens]
        self.P = sum(per) + 2
        order, at = torch.randperm(self.P, generator=self.g), 0
        self.table = torch.full((len(lens), max(per)), -1, dtype=torch.int32)
        for b, n in enumerate(per):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.table = self.table.cuda()
        self.lens = torch.tensor(lens, dtype=torch.int32, device="cuda")

    def query(self, H):
        return torch.randn(len(self.lens), H, 1, self.D, generator=self.g).to(self.dtype).cuda()


@pytest.mark.parametrize("case", SELECT, ids=lambda c: f"{c[0]}-{max(c[1])}x{len(c[1])}-h{c[2]}.{c[3]}-d{c[4]}-p{c[5]}-k{c[6]}")
def test_select(case):
    dtype, lens, H, Hkv, D, page, K = case
    t = Tables(dtype, lens, Hkv, D, page)
    kb, q = _bounds(t, t.P), t.query(H)
    got = cmpext3.paged_select(q, kb, t.table, t.lens, page, K)
    assert got.dtype == torch.int32
    assert np.array_equal(got.cpu().numpy(), po.select(q, kb, t.table, t.lens, page, K))


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_select_ties_zeros_and_special_values(dtype):
    """Equal scores go to the lower page, -0 is 0, an infinite bound and a NaN count as they should."""
    t = Tables(dtype, [900, 900, 900, 640], 1, 64, 16)
    kb = torch.zeros(t.P, 1, 2, 64, dtype=t.dtype, device="cuda")
    kb[t.table[0, ::2].long()] = -0.0
    kb[t.table[1, 7::3].long()] = 1.0
    kb[t.table[2, 5].long(), :, 1, 3] = float("nan")
    kb[t.table[2, 9].long(), :, 1, 3] = float("inf")
    kb[t.table[2, 2].long(), :, :, 4] = float("-inf")
    t.table[3, 11] = -5
    q = t.query(3)
    q[2] = q[2].abs()
    for K in (1, 2, 3, 5, 40, 57, 58, 60):
        got = cmpext3.paged_select(q, kb, t.table, t.lens, 16, K)
        want = po.select(q, kb, t.table, t.lens, 16, K)
        if K > 1:
            assert 11 in want[3, 0]
        assert np.array_equal(got.cpu().numpy(), want), K


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_a_run_of_steps(dtype):
    """Prompts of different lengths, then tokens one by one: append, select, attend, against contiguous caches."""
    B, H, Hkv, D, page, K = 3, 4, 2, 64, 16, 3
    g = torch.Generator().manual_seed(1)
    dt = DTYPES[dtype]
    P, M = 24, 6
    kp, vp = (torch.full((P, Hkv, page, D), float("nan"), dtype=dt, device="cuda") for _ in range(2))
    kb = torch.full((P, Hkv, 2, D), float("nan"), dtype=dt, device="cuda")
    table = torch.randperm(P, generator=g)[:B * M].reshape(B, M).to(torch.int32).cuda()
    cos, sin = tables(M * page, D)
    new = torch.tensor([37, 15, 64], dtype=torch.int32, device="cuda")
    lens = new.clone()

    def rows(heads, S):
        return torch.randn(B, heads, S, D, generator=g).to(dt).cuda()

    cmpext3.paged_append(rows(Hkv, 64), rows(Hkv, 64), kp, vp, table, lens, query=rows(H, 64), cos=cos, sin=sin,
                         new_lens=new, key_bounds=kb)
    cache = type("C", (), {})()
    cache.kp, cache.vp, cache.table, cache.lens = kp, vp, table, lens
    for _ in range(20):
        lens += 1
        q = cmpext3.paged_append(rows(Hkv, 1), rows(Hkv, 1), kp, vp, table, lens, query=rows(H, 1), cos=cos, sin=sin,
                                 key_bounds=kb)
        for b in range(B):
            n = int(lens[b])
            for p in range(-(-n // page)):
                x = kp[table[b, p].long(), :, :min(page, n - p * page)].float()
                e = kb[table[b, p].long()].float()
                assert torch.equal(e[:, 0], x.amin(1)) and torch.equal(e[:, 1], x.amax(1))
        sel = cmpext3.paged_select(q, kb, table, lens, page, K)
        assert np.array_equal(sel.cpu().numpy(), po.select(q, kb, table, lens, page, K))
        check_attention(dtype, cmpext3.paged_attention(q, kp, vp, table, lens, selected=sel), q, cache, D ** -0.5,
                        None, sel.cpu())
        check_attention(dtype, cmpext3.paged_attention(q, kp, vp, table, lens), q, cache, D ** -0.5)


def _steps(state, H, Hkv, D, page):
    q = cmpext3.paged_append(state["k"], state["v"], state["kp"], state["vp"], state["table"], state["lens"],
                             query=state["q"], cos=state["cos"], sin=state["sin"], key_bounds=state["kb"])
    sel = cmpext3.paged_select(q, state["kb"], state["table"], state["lens"], page, 20)
    return q, sel, cmpext3.paged_attention(q, state["kp"], state["vp"], state["table"], state["lens"], selected=sel), \
        cmpext3.paged_attention(q, state["kp"], state["vp"], state["table"], state["lens"])


def _state(seed, lens=(3000, 77, 1500)):
    c = Cache("bf16", list(lens), 2, 128, 16, seed=seed)
    lo = torch.where(c.kp.isnan(), torch.inf, c.kp.float()).amin(2, keepdim=True)
    hi = torch.where(c.kp.isnan(), -torch.inf, c.kp.float()).amax(2, keepdim=True)
    cos, sin = tables(4000, 128)
    return dict(k=c.rows(2, 1), v=c.rows(2, 1), q=c.rows(8, 1), kp=c.kp, vp=c.vp, table=c.table, lens=c.lens,
                cos=cos, sin=sin, kb=torch.cat([lo, hi], 2).to(c.dtype))


def test_captured_steps_replay_beside_eager_ones():
    """Two graphs over their own states, replayed several times with eager work between: every replay gives the
    eager result of its inputs."""
    states = [_state(1), _state(2, (900, 2048, 4000))]
    args = (8, 2, 128, 16)
    graphs, outs = [], []
    for s in states:
        _steps(s, *args)
    torch.cuda.synchronize()
    for s in states:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_steps(s, *args))
        graphs.append(g)
    for r in range(4):
        for s, g, o in zip(states, graphs, outs):
            s["q"].copy_(torch.randn(s["q"].shape, generator=torch.Generator().manual_seed(r)).to(torch.bfloat16))
            g.replay()
            eager = _steps(s, *args)
            torch.cuda.synchronize()
            for a, b in zip(o, eager):
                assert torch.equal(a, b)
        for s, g, o in zip(states, graphs, outs):
            g.replay()
        torch.cuda.synchronize()
        for s, o in zip(states, outs):
            for a, b in zip(o, _steps(s, *args)):
                assert torch.equal(a, b)


def test_a_captured_step_follows_growing_sequences():
    """One graph of a decode step, replayed as sequences grow past pages and tiles, one ends and another begins: the
    work is dealt out on the device, so every replay is the eager step of its lengths."""
    c = Cache("bf16", [500, 15, 0, 300], 2, 128, 16, width=40)
    c.table.copy_(torch.randperm(200, generator=c.g)[:160].reshape(4, 40).to(torch.int32))
    P = 200
    pools = [[torch.zeros(P, 2, 16, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2)] for _ in range(2)]
    bounds = [torch.zeros(P, 2, 2, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    cos, sin = tables(640, 128)
    lens = c.lens.clone()
    k, v, q = (torch.zeros(4, h, 1, 128, dtype=torch.bfloat16, device="cuda") for h in (2, 2, 8))

    def step(pool, kb):
        r = cmpext3.paged_append(k, v, *pool, c.table, lens, query=q, cos=cos, sin=sin, key_bounds=kb)
        sel = cmpext3.paged_select(r, kb, c.table, lens, 16, 6)
        return (r, sel, cmpext3.paged_attention(r, *pool, c.table, lens),
                cmpext3.paged_attention(r, *pool, c.table, lens, selected=sel))

    step(pools[0], bounds[0])
    torch.cuda.synchronize()
    for pool in pools:  # the keys that are there at the start
        for t, seed in zip(pool, (1, 2)):
            t.copy_(torch.randn(t.shape, generator=torch.Generator().manual_seed(seed)))
    for kb in bounds:
        kb.copy_(torch.stack([pools[0][0].amin(2), pools[0][0].amax(2)], 2))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(pools[0], bounds[0])
    for i in range(24):
        if i == 7:
            lens[0], lens[2] = 0, 0  # one ends ...
        if i == 9:
            lens[2] = 63             # ... another begins
        lens.copy_(torch.where(lens > 0, lens + 1, lens))
        for t in (k, v, q):
            t.copy_(torch.randn(t.shape, generator=c.g))
        graph.replay()
        want = step(pools[1], bounds[1])
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b), i
        assert torch.equal(pools[0][0], pools[1][0]) and torch.equal(bounds[0], bounds[1])


def test_streams_of_their_own():
    """Calls on two streams at once, each with its own workspace."""
    states = [_state(1), _state(2, (900, 2048, 4000))]
    want = [[t.clone() for t in _steps(s, 8, 2, 128, 16)] for s in states]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in states]
    got = [[] for _ in states]
    for _ in range(5):
        for i, (s, st) in enumerate(zip(states, streams)):
            with torch.cuda.stream(st):
                got[i].append(_steps(s, 8, 2, 128, 16))
    torch.cuda.synchronize()
    for w, rounds in zip(want, got):
        for o in rounds:
            assert all(torch.equal(a, b) for a, b in zip(o, w))


def test_layouts_of_the_new_rows():
    """Rows off 16 bytes, expanded heads and transposed tables are taken as they are."""
    c = Cache("bf16", [50, 20], 2, 64, 16)
    wide = torch.randn(2, 4, 1, 67, generator=c.g).to(torch.bfloat16).cuda()
    q = wide[..., 1:65]
    check_attention("bf16", cmpext3.paged_attention(q, c.kp, c.vp, c.table, c.lens), q, c, 0.125)
    q1 = q[:, :1].expand(2, 4, 1, 64)
    check_attention("bf16", cmpext3.paged_attention(q1, c.kp, c.vp, c.table, c.lens), q1, c, 0.125)
    t = c.table.t().contiguous().t()
    assert torch.equal(cmpext3.paged_attention(q, c.kp, c.vp, t, c.lens),
                       cmpext3.paged_attention(q, c.kp, c.vp, c.table, c.lens))
    padded = torch.full((2, 9), 12345, dtype=torch.int32, device="cuda")
    padded[:, :c.table.shape[1]] = c.table
    assert torch.equal(cmpext3.paged_attention(q, c.kp, c.vp, padded[:, :c.table.shape[1]], c.lens),
                       cmpext3.paged_attention(q, c.kp, c.vp, c.table, c.lens))
    # a pool with room between its pages and heads
    room = torch.zeros(c.kp.shape[0], 3, 17, 72, dtype=torch.bfloat16, device="cuda")
    kp, vp = room[:, 1:, :16, :64], c.vp
    kp.copy_(c.kp)
    assert torch.equal(cmpext3.paged_attention(q, kp, vp, c.table, c.lens),
                       cmpext3.paged_attention(q, c.kp, vp, c.table, c.lens))
    k = torch.randn(2, 2, 1, 67, generator=c.g).to(torch.bfloat16).cuda()[..., 3:]
    a, b = c.kp.clone(), c.kp.clone()
    cmpext3.paged_append(k, k, a, c.vp.clone(), c.table, c.lens)
    cmpext3.paged_append(k.contiguous(), k.contiguous(), b, c.vp.clone(), c.table, c.lens)
    assert torch.equal(a.view(torch.int16), b.view(torch.int16)) and not torch.equal(a.view(torch.int16), c.kp.view(torch.int16))


def test_empty_calls():
    c = Cache("bf16", [50, 20], 2, 64, 16)
    q = c.rows(4, 1)
    assert cmpext3.paged_attention(q[:0], c.kp, c.vp, c.table[:0], c.lens[:0]).shape == (0, 4, 1, 64)
    assert cmpext3.paged_attention(q[:, :, :0], c.kp, c.vp, c.table, c.lens).shape == (2, 4, 0, 64)
    zero = torch.zeros_like(c.lens)
    assert (cmpext3.paged_attention(q, c.kp, c.vp, c.table[:, :0], zero) == 0).all()
    assert cmpext3.paged_attention(q, c.kp, c.vp, c.table[:, :0], c.lens).isnan().all()
    kb = torch.zeros(c.kp.shape[0], 2, 2, 64, dtype=torch.bfloat16, device="cuda")
    assert (cmpext3.paged_select(q, kb, c.table[:, :0], zero, 16, 4) == -1).all()
    assert (cmpext3.paged_select(q, kb, c.table, zero, 16, 4) == -1).all()
    k = c.rows(2, 1)
    before = c.kp.clone()
    assert cmpext3.paged_append(k[:, :, :0], k[:, :, :0], c.kp, c.vp, c.table, c.lens) is None
    cmpext3.paged_append(k, k, c.kp, c.vp, c.table, zero)
    assert torch.equal(before.view(torch.int16), c.kp.view(torch.int16))


def test_refusals():
    c = Cache("bf16", [50, 20], 2, 64, 16)
    q, k = c.rows(4, 1), c.rows(2, 1)
    kb = torch.zeros(c.kp.shape[0], 2, 2, 64, dtype=torch.bfloat16, device="cuda")
    cos, sin = tables(64, 64)
    att = lambda **o: cmpext3.paged_attention(*[o.pop(n, d) for n, d in (  # noqa: E731
        ("q", q), ("kp", c.kp), ("vp", c.vp), ("t", c.table), ("l", c.lens))], **o)
    app = lambda **o: cmpext3.paged_append(*[o.pop(n, d) for n, d in (  # noqa: E731
        ("k", k), ("v", k), ("kp", c.kp), ("vp", c.vp), ("t", c.table), ("l", c.lens))], **o)
    sel = lambda **o: cmpext3.paged_select(*[o.pop(n, d) for n, d in (  # noqa: E731
        ("q", q), ("kb", kb), ("t", c.table), ("l", c.lens), ("page", 16), ("n", 4))], **o)
    att(), app(), sel()
    bad = [
        lambda: att(q=q.cpu()), lambda: att(q=q.float()), lambda: att(q=q[:, :3]), lambda: att(q=q[0]),
        lambda: att(q=q.expand(2, 4, 17, 64)), lambda: att(kp=c.kp.half()), lambda: att(kp=c.kp.cpu()),
        lambda: att(kp=c.kp[..., :56]), lambda: att(vp=c.vp[1:]), lambda: att(vp=c.vp[:, :1]),
        lambda: att(t=c.table.long()), lambda: att(t=c.table[:1]), lambda: att(l=c.lens.long()),
        lambda: att(l=c.lens.cpu()), lambda: att(scale=float("nan")), lambda: att(new_lens=c.lens[:1]),
        lambda: att(selected=torch.zeros(2, 2, 0, dtype=torch.int32, device="cuda")),
        lambda: att(selected=torch.zeros(2, 4, 3, dtype=torch.int32, device="cuda")),
        lambda: att(q=q.clone().requires_grad_()),
        lambda: att(kp=torch.zeros(5, 2, 16, 65, dtype=torch.bfloat16, device="cuda")[..., :64],
                    vp=torch.zeros(5, 2, 16, 65, dtype=torch.bfloat16, device="cuda")[..., :64]),
        lambda: att(q=q[..., :60], kp=c.kp[..., :60], vp=c.vp[..., :60]),
        lambda: att(kp=c.kp[:, :, :1].expand_as(c.kp)),
        lambda: app(v=k[:, :1]), lambda: app(query=q), lambda: app(cos=cos), lambda: app(query=q, cos=cos),
        lambda: app(query=q, cos=cos.half(), sin=sin.half()), lambda: app(query=q[:, :3], cos=cos, sin=sin),
        lambda: app(query=q, cos=torch.cat([cos, cos], 1), sin=torch.cat([sin, sin], 1)),
        lambda: app(positions=torch.zeros(2, 1, dtype=torch.int32, device="cuda")),
        lambda: app(query=q, cos=cos, sin=sin, positions=torch.zeros(2, 2, dtype=torch.int32, device="cuda")),
        lambda: app(key_bounds=kb[1:]), lambda: app(key_bounds=kb[:, :, :1]), lambda: app(key_bounds=kb.float()),
        lambda: app(k=k.clone().requires_grad_()), lambda: app(kp=c.kp.cpu()),
        lambda: sel(q=c.rows(4, 2)), lambda: sel(n=0), lambda: sel(page=0), lambda: sel(kb=kb[:, :, :1]),
        lambda: sel(kb=kb.half()), lambda: sel(q=q[:, :3]), lambda: sel(l=c.lens[:1]),
    ]
    before = c.kp.clone()
    for i, f in enumerate(bad):
        with pytest.raises(RuntimeError):
            f()
            print("not refused:", i)
    assert torch.equal(before.view(torch.int16), c.kp.view(torch.int16))
    with torch.no_grad():
        att(q=q.clone().requires_grad_())


# how the tables lie in memory: half of doubled ones, a column in two, transposed, one row for all, unlike each other
TABLES = {
    "halves": lambda t: (torch.cat([t[0], t[0]], 1)[:, :t[0].shape[1]], torch.cat([t[1], t[1]], 1)[:, :t[0].shape[1]]),
    "one pair of tensors": lambda t: torch.cat(t, 1).chunk(2, 1),
    "from an odd word": lambda t: tuple(torch.cat([x[:, :1], x], 1)[:, 1:] for x in t),
    "spread": lambda t: tuple(x.repeat_interleave(2, 1)[:, ::2] for x in t),
    "transposed": lambda t: tuple(x.t().contiguous().t() for x in t),
    "mixed": lambda t: (torch.cat([t[0], t[0]], 1)[:, :t[0].shape[1]], t[1]),
    "one row": lambda t: tuple(x[7:8].expand_as(x) for x in t),
}


@pytest.mark.parametrize("lies", TABLES)
@pytest.mark.parametrize("dtype,rot,pairs", [("bf16", 64, False), ("fp16", 24, True), ("fp32", 12, False), ("fp32", 2, False)])
def test_rotation_tables_of_any_layout(dtype, rot, pairs, lies):
    c = Cache(dtype, [70, 33], 2, 64, 16)
    k, v, q = c.rows(2, 9), c.rows(2, 9), c.rows(4, 9)
    cos, sin = TABLES[lies](tables(80, rot))
    out = []
    for t in ((cos, sin), (cos.contiguous(), sin.contiguous())):
        kp, vp = torch.zeros_like(c.kp), torch.zeros_like(c.vp)
        out.append((cmpext3.paged_append(k, v, kp, vp, c.table, c.lens, query=q, cos=t[0], sin=t[1], interleaved=pairs), kp, vp))
    assert all(torch.equal(a, b) for a, b in zip(*out)) and not out[0][0].isnan().any()


def test_tables_that_are_learned_are_refused():
    c = Cache("bf16", [50, 20], 2, 64, 16)
    k = c.rows(2, 1)
    for i in range(2):
        t = list(tables(64, 64))
        t[i].requires_grad_()
        with pytest.raises(RuntimeError, match="no backward"):
            cmpext3.paged_append(k, k, c.kp, c.vp, c.table, c.lens, cos=t[0], sin=t[1])
        with torch.no_grad():
            cmpext3.paged_append(k, k, c.kp, c.vp, c.table, c.lens, cos=t[0], sin=t[1])


# dtype, lens, H, Hkv, D, page, S: shares that span units, units cut by themselves, whole units
SPLITS = [
    ("bf16", [5000, 70, 0, 2600], 8, 2, 128, 16, 1),
    ("fp16", [(97 * b) % 3000 for b in range(70)], 8, 4, 64, 16, 1),
    ("fp32", [3000, 40, 900], 6, 3, 64, 24, 2),
    ("bf16", [30000], 4, 1, 256, 64, 1),
    ("bf16", [70000], 2, 1, 8, 16, 1),
    ("fp16", [2000] * 70, 64, 8, 64, 32, 1),
    ("bf16", [9000, 9001], 64, 2, 128, 16, 1),
]


@pytest.mark.parametrize("case", SPLITS, ids=lambda c: f"{c[0]}-{max(c[1])}x{len(c[1])}-h{c[2]}.{c[3]}-d{c[4]}")
def test_whole_and_split_sequences_agree(case):
    """Without a workspace no sequence is split; a workspace that is too small counts as none; a split leaves its
    counters at zero and repeats bit for bit.  Both lie within the tolerance of the float64 attention."""
    dtype, lens, H, Hkv, D, page, S = case
    c = Cache(dtype, lens, Hkv, D, page)
    q = c.rows(H, S).contiguous()
    args = (q, c.kp, c.vp, c.table, c.lens)
    whole = abi.paged_attention(*args, workspace=None)
    n = abi.paged_workspace_size(abi.dtype_code(q.dtype), len(lens), H, Hkv, S, D, page, c.table.shape[1])
    assert n > abi.WORKSPACE_COUNTER_BYTES
    ws = torch.zeros(n, dtype=torch.uint8, device="cuda")
    split = abi.paged_attention(*args, workspace=ws)
    assert not ws[:abi.WORKSPACE_COUNTER_BYTES].any()
    assert torch.equal(split, abi.paged_attention(*args, workspace=ws))
    assert not ws[:abi.WORKSPACE_COUNTER_BYTES].any()
    assert torch.equal(split, cmpext3.paged_attention(*args))
    assert torch.equal(whole, abi.paged_attention(*args, workspace=ws[:n - 16]))
    some = [b for b in range(len(lens)) if b < 4]
    sub = Cache.__new__(Cache)
    sub.kp, sub.vp, sub.table, sub.lens = c.kp, c.vp, c.table[some], c.lens[some]
    check_attention(dtype, whole[some], q[some], sub, D ** -0.5)
    check_attention(dtype, split[some], q[some], sub, D ** -0.5)


def test_the_c_entry_points_are_what_the_binding_calls():
    s = _state(5)
    kp, vp, kb = s["kp"].clone(), s["vp"].clone(), s["kb"].clone()
    q = cmpext3.paged_append(s["k"], s["v"], s["kp"], s["vp"], s["table"], s["lens"], query=s["q"], cos=s["cos"],
                             sin=s["sin"], key_bounds=s["kb"])
    q2 = abi.paged_append(s["k"], s["v"], kp, vp, s["table"], s["lens"], s["q"], s["cos"], s["sin"], key_bounds=kb)
    assert torch.equal(q, q2) and torch.equal(kb, s["kb"])
    assert torch.equal(kp.view(torch.int16), s["kp"].view(torch.int16))
    sel = cmpext3.paged_select(q, kb, s["table"], s["lens"], 16, 9)
    assert torch.equal(sel, abi.paged_select(q, kb, s["table"], s["lens"], 16, 9))
    assert torch.equal(cmpext3.paged_attention(q, kp, vp, s["table"], s["lens"], selected=sel),
                       abi.paged_attention(q, kp, vp, s["table"], s["lens"], selected=sel))
    with pytest.raises(RuntimeError, match="code"):
        abi.paged_attention(q, kp, vp, s["table"], s["lens"], float("nan"))
