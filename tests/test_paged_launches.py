"""What reaches a stream when the paged cache's entry points are called (no GPU), as tests/test_launches.py does it."""
from __future__ import annotations

import pytest

from test_launches import _run, recorder  # noqa: F401

PAGED = """
attn = lib.cmpext3_paged_attn; app = lib.cmpext3_paged_append; sel = lib.cmpext3_paged_select
def attention(dt, B, H, Hkv, S, D, page, width, ws=None, nbytes=0, nsel=0):
    rows, pool = s3(H * S * D, S * D, D), s3(Hkv * page * D, page * D, D)
    return attn(vp(A), vp(A), vp(A), vp(A), dt, B, H, Hkv, S, D, 100, page, rows, pool, pool, rows, vp(A), width,
                i64(width), vp(A), None, vp(A) if nsel else None, nsel, ctypes.c_float(0.1), vp(ws), sz(nbytes), None)
def append(dt, B, H, Hkv, S, D, page, bounds=False, rot=0):
    rows, pool = s3(Hkv * S * D, S * D, D), s3(Hkv * page * D, page * D, D)
    return app(vp(A), vp(A), vp(A) if rot else None, vp(A + 65536) if rot else None, vp(A), vp(A), vp(A) if bounds else None,
               dt, B, H, Hkv, S, D, 100, page, rows, rows, s3(H * S * D, S * D, D), s3(H * S * D, S * D, D), pool, pool,
               s3(Hkv * 2 * D, 2 * D, D), vp(A), 10, i64(10), vp(A), None, None, vp(A) if rot else None,
               vp(A) if rot else None, 50, rot, i64(rot // 2), 0, None)
def select(dt, B, H, Hkv, D, width, n, ws=A, nbytes=1 << 40):
    return sel(vp(A), vp(A), vp(A), dt, B, H, Hkv, D, 100, 16, s3(H * D, D, D), s3(Hkv * 2 * D, 2 * D, D), vp(A), width,
               i64(width), vp(A), n, vp(ws), sz(nbytes), None)
"""


def test_one_launch_a_call(recorder):  # noqa: F811
    got = _run(recorder, PAGED + """
out = []
def one(f):
    rec.recorder_clear(); rc = f(); out.append([rc, [n[1] for n in launches()], [n[2] for n in launches()]])
one(lambda: attention(BF16, 16, 16, 8, 1, 128, 16, 256, A, 1 << 30))
one(lambda: attention(BF16, 1, 16, 8, 1, 128, 16, 19, A, 1 << 30))
one(lambda: attention(F32, 2, 4, 4, 16, 64, 24, 9))
one(lambda: attention(F16, 2, 64, 2, 2, 64, 24, 9, None, 0, 5))
one(lambda: append(BF16, 4, 16, 8, 2048, 128, 16, True, 128))
one(lambda: append(BF16, 4, 16, 8, 1, 128, 16))
one(lambda: select(BF16, 4, 16, 8, 128, 1024, 20))
one(lambda: select(F32, 4, 16, 8, 128, 1025, 20))
one(lambda: attention(BF16, 2, 4, 2, 17, 64, 16, 9))
one(lambda: append(BF16, 0, 4, 2, 1, 64, 16))
one(lambda: select(BF16, 2, 4, 2, 64, 2000, 5, A, 100))
print(json.dumps(out))
""")
    rcs, names, grids = zip(*got)
    assert rcs == (0,) * 8 + (7, 0, 1)
    assert [len(n) for n in names] == [1, 1, 1, 1, 1, 1, 1, 2, 0, 0, 0]
    for call, kernel in zip(names, ["paged_attn"] * 4 + ["paged_append"] * 2 + ["paged_short", "paged_scores"]):
        assert kernel in call[0]
    assert "paged_best" in names[7][1]
    assert grids[0][0] <= 2 * 256 and grids[1][0] < 40  # the chip's fill; a short cache's


def test_a_selections_launches_stay_together(recorder):  # noqa: F811
    seen = _run(recorder, PAGED + """
rec.recorder_slow(b"paged_scores", 2000)
def go(tag):
    rec.recorder_tag(tag)
    for _ in range(8):
        assert select(BF16, 2, 4, 2, 64, 5000, 9) == 0
ts = [threading.Thread(target=go, args=(t,)) for t in (1, 2)]
[t.start() for t in ts]; [t.join() for t in ts]
print(json.dumps(launches()))
""")
    assert len(seen) == 32 and {tag for tag, *_ in seen} == {1, 2}
    for a, b in zip(seen[::2], seen[1::2]):
        assert a[0] == b[0] and "paged_scores" in a[1] and "paged_best" in b[1]


def test_paged_attention_waits_for_a_call_that_uses_its_workspace(recorder):  # noqa: F811
    """A masked attention call hands its mask's bits from one launch to the next through the workspace that the
    paged calls of the stream use too."""
    seen = _run(recorder, PAGED + """
rec.recorder_slow(b"attn_mask_bits", 3000)
n, ws, done = 1 << 28, 1 << 34, []
def masked():
    rec.recorder_tag(1)
    for _ in range(8):
        assert fwd("ws", BF16, 1, 2, 700, 128, True, ws, n) == 0
    done.append(1)
def paged():
    rec.recorder_tag(2)
    while True:
        assert attention(BF16, 2, 8, 2, 1, 128, 16, 200, ws, n) == 0
        if done:
            break
ts = [threading.Thread(target=masked), threading.Thread(target=paged)]
[t.start() for t in ts]; [t.join() for t in ts]
print(json.dumps(launches()))
""")
    bits = [i for i, (_, name, *_) in enumerate(seen) if "attn_mask_bits" in name]
    assert len(bits) == 8 and {tag for tag, *_ in seen} == {1, 2}
    for i in bits:
        assert seen[i + 1][0] == 1 and "attn_fwd_pipe16" in seen[i + 1][1]


@pytest.mark.parametrize("S,page", [(1, 16), (4096, 8), (65536, 1), (2, 512)])
def test_append_grids_stay_launchable(recorder, S, page):  # noqa: F811
    """A grid is less than 2^32 threads, or the call is refused."""
    got = _run(recorder, PAGED + f"""
out = []
for B in (1, 64, 4096, 1 << 16, 1 << 20):
    rec.recorder_clear(); rc = append(BF16, B, 32, 8, {S}, 64, {page}, True, 64)
    out.append([rc, [n[3] for n in launches()]])
print(json.dumps(out))
""")
    assert got[0][0] == 0
    for rc, threads in got:
        assert (rc == 0 and len(threads) == 1 and 0 < threads[0] < 1 << 32) or (rc == 7 and not threads)
