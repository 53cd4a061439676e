"""The paged key-value cache's operators, as a serving program calls them.

append     new tokens' keys and values into their pages, rotated on the way, with the queries' rotation
attention  new tokens' attention over the pages of their sequences, or over some of those pages
select     the pages that each sequence's new token attends to, by the channel bounds of their keys

`own` false: the plain forms in elementary torch operations; true: cmpext3's calls.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
_THETA = 10000.0


# ---------------------------------------------------------------- cases
#
#   op, dtype, B, H, Hkv, D, page (slots of a page)
#   lo, hi      shortest and longest sequence, the new tokens among them; the rest lie between
#   idle        every fourth place of the batch has no sequence (length 0)
#   new         query or new-token columns; ragged: a sequence brings 0..new of them
#   layout      "hps" pool [pages, heads, slots, D], "psh" the same as a view of [pages, slots, heads, D]
#   append:     rot (rotated dims), pairs (2i, 2i + 1 instead of halves), bounds (of each page's keys kept)
#   attention:  picked (pages of each sequence attended to; 0: all)
#   select:     picked


def _case(name, op, dtype, B, H, Hkv, D, page, lo, hi, idle=False, new=1, ragged=False, layout="hps", rot=0,
          pairs=False, bounds=False, picked=0):
    c = dict(op=op, dtype=dtype, B=B, H=H, Hkv=Hkv, D=D, page=page, lo=lo, hi=hi, idle=idle, new=new, ragged=ragged,
             layout=layout, rot=rot, pairs=pairs, bounds=bounds, picked=picked)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one user's conversation, a short one: latency alone counts
        _case("attn_one_bf16", "attention", "bf16", 1, 16, 8, 128, 16, 300, 300),
        # a served batch, caches equally full
        _case("attn_batch_bf16", "attention", "bf16", 16, 16, 8, 128, 16, 4096, 4096),
        # a served batch of ragged conversations with idle places, odd lengths, four query heads a key head
        _case("attn_ragged_fp16", "attention", "fp16", 64, 32, 8, 64, 32, 1, 4001, idle=True, layout="psh"),
        # one long document at head dim 256: the largest
        _case("attn_long_d256_bf16", "attention", "bf16", 1, 16, 8, 256, 64, 131072, 131072),
        # full precision, short blocks of guessed tokens, an odd page size
        _case("attn_block_fp32", "attention", "fp32", 8, 12, 12, 64, 24, 77, 1531, new=4, ragged=True),
        # long caches of which a few hundred pages a head are attended to
        _case("attn_picked_bf16", "attention", "bf16", 8, 32, 8, 128, 32, 16384, 32768, picked=128),
        # a decode step's new tokens
        _case("append_step_bf16", "append", "bf16", 16, 16, 8, 128, 16, 40, 300, rot=128, bounds=True),
        # prompts of one length, as the projection leaves them, bounds kept
        _case("append_prompt_bf16", "append", "bf16", 4, 16, 8, 128, 16, 2048, 2048, new=2048, rot=128, bounds=True),
        # chunks of ragged prompts, half of each head rotated in pairs, an odd page size
        _case("append_chunk_fp16", "append", "fp16", 8, 10, 10, 80, 24, 600, 1531, new=513, ragged=True, layout="psh",
              rot=40, pairs=True),
        # full precision
        _case("append_prompt_fp32", "append", "fp32", 2, 8, 8, 64, 16, 1024, 1024, new=1024, rot=64),
        # pages of a batch of ordinary conversations
        _case("select_batch_bf16", "select", "bf16", 16, 16, 8, 128, 16, 2000, 4096, picked=64),
        # pages of one long document
        _case("select_long_fp16", "select", "fp16", 1, 32, 8, 128, 16, 131072, 131072, picked=256),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "append", "append", "select"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    es = 4 if dtype == "fp32" else 2
    Hkv = rng.choice([1, 2, 4, 5, 8, 10])
    H = Hkv * rng.choice([1, 1, 2, 4, 8])
    D = rng.choice([40, 64, 64, 72, 80, 96, 128, 128, 128, 160, 192, 256])
    page = rng.choice([8, 16, 16, 24, 32, 64, 128])
    layout = rng.choice(["hps", "hps", "psh"])
    B = _log_int(rng, 1, 64)
    budget = (1 << 28) // (B * Hkv * D * es)  # tokens of a sequence: 256 MiB of keys in all
    if op == "append":
        new = _log_int(rng, 1, max(1, min(2048, budget // 8)))
        rot = rng.choice([D, D, D // 2 // 2 * 2, 0])
        hi = new + _log_int(rng, 1, 600)
        return _case("", op, dtype, B, H, Hkv, D, page, rng.randint(new, hi), hi, rng.random() < 0.3, new,
                     rng.random() < 0.5, layout, rot, rng.random() < 0.4, rng.random() < 0.5)
    hi = _log_int(rng, 16, max(17, min(65536, budget)))
    lo = hi if rng.random() < 0.3 else rng.randint(1, hi)
    if op == "select":
        return _case("", op, dtype, B, H, Hkv, D, page, lo, hi, rng.random() < 0.3, layout="hps",
                     picked=_log_int(rng, 1, 256))
    new = rng.choice([1, 1, 1, 2, 3, 5, 8])
    picked = _log_int(rng, 2, 128) if new == 1 and rng.random() < 0.3 else 0
    return _case("", op, dtype, B, H, Hkv, D, page, max(lo, new), max(hi, new), rng.random() < 0.3, new,
                 new > 1 and rng.random() < 0.5, layout, picked=picked)


def _lens(c):
    """Tokens of each sequence, and how many of them are new."""
    lens, new = [], []
    for b in range(c["B"]):
        f = (b * 0.6180339887498949) % 1.0
        n = c["hi"] if b == 0 else c["lo"] + int(round((c["hi"] - c["lo"]) * f))
        if c["idle"] and b % 4 == 3:
            n = 0
        lens.append(n)
        k = c["new"] if not c["ragged"] or b % 3 == 0 else (c["new"] * (b % 3)) // 3
        new.append(min(k, n))
    return lens, new


def _pages(c):
    lens, _ = _lens(c)
    per = [-(-n // c["page"]) for n in lens]
    return per, max(1, max(per))


# ---------------------------------------------------------------- inputs


def _pool(c, P, gen, dt, heads_slots):
    if c["layout"] == "psh":
        return torch.randn(P, heads_slots[1], heads_slots[0], c["D"], generator=gen, device="cuda",
                           dtype=torch.float32).to(dt).transpose(1, 2)
    return torch.randn(P, heads_slots[0], heads_slots[1], c["D"], generator=gen, device="cuda",
                       dtype=torch.float32).to(dt)


def prepare(c, seed):
    dev = "cuda"
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt = _DTYPES[c["dtype"]]
    lens, new = _lens(c)
    per, M = _pages(c)
    B, H, Hkv, D, page, S = c["B"], c["H"], c["Hkv"], c["D"], c["page"], c["new"]
    P = sum(per) + 3
    order = torch.randperm(P, generator=gen, device=dev).to(torch.int32)
    table = torch.zeros(B, M, dtype=torch.int32, device=dev)
    at = 0
    for b in range(B):  # a sequence's pages lie anywhere in the pool
        table[b, :per[b]] = order[at:at + per[b]]
        at += per[b]
    s = dict(case=c, table=table, lens=torch.tensor(lens, dtype=torch.int32, device=dev),
             new=torch.tensor(new, dtype=torch.int32, device=dev) if c["ragged"] else None)

    def rows(heads):  # what a projection leaves: [B, S, heads, D] memory seen as [B, heads, S, D]
        return torch.randn(B, S, heads, D, generator=gen, device=dev).to(dt).transpose(1, 2)

    if c["op"] == "select":
        a = torch.randn(P, Hkv, 1, D, generator=gen, device=dev)
        w = torch.rand(P, Hkv, 1, D, generator=gen, device=dev) * 2
        s["bounds"] = torch.cat([a - w, a + w], dim=2).to(dt)
        s["q"] = rows(H)
        return s
    s["kp"] = _pool(c, P, gen, dt, (Hkv, page))
    s["vp"] = _pool(c, P, gen, dt, (Hkv, page))
    s["q"] = rows(H)
    if c["op"] == "attention":
        s["scale"] = 1.0 / math.sqrt(D)
        s["picked"] = None
        if c["picked"]:
            K = c["picked"]
            sel = torch.full((B, Hkv, K), -1, dtype=torch.int32, device=dev)
            for b in range(B):
                n = per[b]
                if n == 0:
                    continue
                r = torch.rand(Hkv, n, generator=gen, device=dev)
                r[:, n - 1] = 2.0  # the newest page is among them
                k = min(K, n)
                sel[b, :, :k] = r.topk(k, dim=1).indices.sort(dim=1).values.to(torch.int32)
            s["picked"] = sel
        return s
    s["k"], s["v"] = rows(Hkv), rows(Hkv)
    s["cos"] = s["sin"] = None
    if not c["rot"]:
        s["q"] = None  # nothing to do to the queries
    else:
        inv = _THETA ** (-torch.arange(0, c["rot"], 2, dtype=torch.float64, device=dev) / c["rot"])
        ang = torch.arange(max(c["hi"], 1), dtype=torch.float64, device=dev)[:, None] * inv
        s["cos"], s["sin"] = ang.cos().float(), ang.sin().float()
    s["bounds"] = None
    if c["bounds"]:
        a = torch.randn(P, Hkv, 1, D, generator=gen, device=dev)
        s["bounds"] = torch.cat([a - 1, a + 1], dim=2).to(dt)
    return s


# ---------------------------------------------------------------- plain forms


def _new_of(s, b, S):
    n = s["lens"][b].clamp(min=0)
    return torch.minimum(n, s["new"][b] if s["new"] is not None else n.new_tensor(S)), n


def _rotate(x, cos, sin, pairs):
    r = 2 * cos.shape[-1]
    out = x.clone()
    if pairs:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        out[..., 0:r:2], out[..., 1:r:2] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = x[..., :r // 2], x[..., r // 2:r]
        out[..., :r // 2], out[..., r // 2:r] = a * cos - b * sin, b * cos + a * sin
    return out


def _plain_append(s):
    c = s["case"]
    S, page, pairs = c["new"], c["page"], c["pairs"]
    dt = s["k"].dtype
    B = c["B"]
    i = torch.arange(S, device="cuda")
    new = s["new"] if s["new"] is not None else torch.full_like(s["lens"], S)
    new = torch.minimum(new, s["lens"]).long()
    pos = s["lens"].long()[:, None] - new[:, None] + i  # [B, S]
    live = i < new[:, None]
    k, q = s["k"].float(), None
    if s["cos"] is not None:
        at = pos.clamp(min=0, max=s["cos"].shape[0] - 1)
        cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]
        q, k = _rotate(s["q"].float(), cos, sin, pairs), _rotate(k, cos, sin, pairs)
        q = torch.where(live[:, None, :, None], q, torch.zeros_like(q)).to(dt)
    k = k.to(dt)
    b_at, i_at = live.nonzero(as_tuple=True)
    p_at = pos[b_at, i_at]
    rows = s["table"][b_at, p_at // page].long()
    slots = p_at % page
    s["kp"][rows, :, slots] = k[b_at, :, i_at]
    s["vp"][rows, :, slots] = s["v"][b_at, :, i_at]
    out = [s["kp"], s["vp"]] if q is None else [q, s["kp"], s["vp"]]
    if s["bounds"] is not None:
        # lowest and highest of each touched page: a page that begins with a new token starts anew
        first = rows[slots == 0]
        lo, hi = s["bounds"][:, :, 0].float(), s["bounds"][:, :, 1].float()
        lo[first], hi[first] = math.inf, -math.inf
        kk = k[b_at, :, i_at].float()
        at = rows[:, None, None].expand_as(kk)
        lo = lo.scatter_reduce(0, at, kk, "amin")
        hi = hi.scatter_reduce(0, at, kk, "amax")
        s["bounds"].copy_(torch.stack([lo, hi], dim=2))
        out.append(s["bounds"])
    return out


def _plain_attention(s):
    c = s["case"]
    B, H, Hkv, D, page, S = c["B"], c["H"], c["Hkv"], c["D"], c["page"], c["new"]
    G = H // Hkv
    out = torch.empty(B, H, S, D, dtype=s["q"].dtype, device="cuda")
    M = s["table"].shape[1]
    slot = torch.arange(page, device="cuda")
    heads = torch.arange(Hkv, device="cuda")[:, None]
    for b in range(B):
        new, n = _new_of(s, b, S)
        i = torch.arange(S, device="cuda")
        limit = torch.where(i < new, n - new + i + 1, torch.zeros_like(i))  # [S]
        if s["picked"] is None:
            rows = s["table"][b].long()
            k, v = s["kp"][rows].transpose(0, 1), s["vp"][rows].transpose(0, 1)  # [Hkv, M, page, D]
            pos = (torch.arange(M, device="cuda")[:, None] * page + slot).reshape(1, -1)
        else:
            sel = s["picked"][b].long()  # [Hkv, K]
            rows = s["table"][b].long()[sel.clamp(min=0)]
            k, v = s["kp"][rows, heads], s["vp"][rows, heads]
            pos = torch.where(sel[..., None] >= 0, sel[..., None] * page + slot, 1 << 30).reshape(Hkv, -1)
        k, v = k.reshape(Hkv, -1, D).float(), v.reshape(Hkv, -1, D).float()
        q = s["q"][b].float().reshape(Hkv, G * S, D) * s["scale"]
        x = torch.matmul(q, k.transpose(1, 2).contiguous()).reshape(Hkv, G, S, -1)
        keep = pos[:, None, None, :] < limit[None, None, :, None]
        x = torch.where(keep, x, torch.full_like(x, -math.inf))
        top = x.amax(dim=-1, keepdim=True)
        p = torch.exp(x - torch.where(top == -math.inf, torch.zeros_like(top), top))
        total = p.sum(dim=-1, keepdim=True)
        v = torch.where((pos < n)[..., None], v, torch.zeros_like(v))
        o = torch.matmul((p / torch.where(total == 0, torch.ones_like(total), total)).reshape(Hkv, G * S, -1), v)
        out[b] = o.reshape(H, S, D).to(out.dtype)
    return out


def _plain_select(s):
    c = s["case"]
    B, H, Hkv, D, page, K = c["B"], c["H"], c["Hkv"], c["D"], c["page"], c["picked"]
    M = s["table"].shape[1]
    out = torch.full((B, Hkv, K), -1, dtype=torch.int32, device="cuda")
    index = torch.arange(M, device="cuda")
    take = min(K, M)
    for b in range(B):
        n = (s["lens"][b] + page - 1) // page
        q = s["q"][b].double().reshape(Hkv, H // Hkv, D)
        up, down = q.clamp(min=0).sum(dim=1), q.clamp(max=0).sum(dim=1)
        e = s["bounds"][s["table"][b].long()].double()  # [M, Hkv, 2, D]
        score = ((up * e[:, :, 1]) + (down * e[:, :, 0])).sum(dim=-1).t()  # [Hkv, M]
        score = torch.where(index == n - 1, math.inf, score)
        score = torch.where(index < n, score, -math.inf)
        best = score.sort(dim=1, descending=True, stable=True).indices[:, :take]
        best = torch.where(best < n, best, M).sort(dim=1).values
        out[b, :, :take] = torch.where(best < M, best, -1).to(torch.int32)
    return out


# ---------------------------------------------------------------- the framework's calls

_own = None


def _package():
    global _own
    if _own is None:
        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        sys.path.insert(0, os.path.join(root, "torch-cmp-patch_amd"))
        os.environ.setdefault("CMPEXT3_AUTOPATCH", "0")
        import cmpext3
        _own = cmpext3
    return _own


def _own_run(s):
    c = s["case"]
    m = _package()
    if c["op"] == "append":
        q = m.paged_append(s["k"], s["v"], s["kp"], s["vp"], s["table"], s["lens"], query=s["q"], cos=s["cos"],
                           sin=s["sin"], new_lens=s["new"], interleaved=c["pairs"], key_bounds=s["bounds"])
        return ([] if q is None else [q]) + [s["kp"], s["vp"]] + ([] if s["bounds"] is None else [s["bounds"]])
    if c["op"] == "attention":
        return m.paged_attention(s["q"], s["kp"], s["vp"], s["table"], s["lens"], s["scale"], new_lens=s["new"],
                                 selected=s["picked"])
    return m.paged_select(s["q"], s["bounds"], s["table"], s["lens"], c["page"], c["picked"])


def run(state):
    if own:
        return _own_run(state)
    return {"append": _plain_append, "attention": _plain_attention, "select": _plain_select}[state["case"]["op"]](state)


# ---------------------------------------------------------------- work, definition


def work(c):
    es = 4 if c["dtype"] == "fp32" else 2
    lens, new = _lens(c)
    per, _ = _pages(c)
    D, H, Hkv, B = c["D"], c["H"], c["Hkv"], c["B"]
    if c["op"] == "append":
        n = sum(new)
        touched = sum(-(-a // c["page"]) - (a - k) // c["page"] for a, k in zip(lens, new) if k)
        opened = sum(-(-a // c["page"]) - -(-(a - k) // c["page"]) for a, k in zip(lens, new) if k)
        heads = 2 * Hkv + (H if c["rot"] else 0)
        rows = 2 * n * heads * D * es + ((B * c["new"] - n) * H * D * es if c["rot"] else 0)
        edges = (2 * touched - opened) * Hkv * 2 * D * es if c["bounds"] else 0
        return {"bytes": rows + edges + 4 * max(lens) * c["rot"] + 4 * (touched + B),
                "flops": 3 * n * (H + Hkv) * c["rot"] + (2 * n * Hkv * D if c["bounds"] else 0)}
    if c["op"] == "attention":
        if c["picked"]:
            K = c["picked"]
            keys = [a if p <= K else (K - 1) * c["page"] + a - (p - 1) * c["page"] for a, p in zip(lens, per)]
            index = 4 * B * Hkv * K + 4 * sum(min(K * Hkv, p) for p in per)
        else:
            keys, index = lens, 4 * sum(per)
        # a query row weighs the keys up to its own token
        pairs = sum(k * (a - k) + k * (k + 1) // 2 for a, k in zip(keys, new)) * H
        return {"bytes": 2 * es * D * Hkv * sum(keys) + 2 * es * B * H * c["new"] * D + index + 4 * B,
                "flops": 4 * D * pairs}
    return {"bytes": 2 * es * D * Hkv * sum(per) + es * B * H * D + 4 * sum(per) + 4 * B + 4 * B * Hkv * c["picked"],
            "flops": 4 * D * Hkv * sum(per) + 2 * B * H * D}


def exact(c, seed):
    s = prepare(c, seed)
    lens, new = _lens(c)
    D, H, Hkv, page, S = c["D"], c["H"], c["Hkv"], c["page"], c["new"]
    G = H // Hkv
    table = s["table"].tolist()
    if c["op"] == "select":
        found = torch.full((c["B"], Hkv, c["picked"]), -1, dtype=torch.int32, device="cuda")
        for b, n in enumerate(lens):
            pages = -(-n // page)
            if pages == 0:
                continue
            lo, hi = s["bounds"][table[b][:pages]].double().unbind(2)  # [pages, Hkv, D]
            bound = torch.zeros(pages, Hkv, dtype=torch.float64, device="cuda")
            for h in range(H):
                q = s["q"][b, h, 0].double()
                bound[:, h // G] += torch.maximum(q * lo[:, h // G], q * hi[:, h // G]).sum(dim=-1)
            for h in range(Hkv):
                got = sorted((-x, p) for p, x in enumerate(bound[:-1, h].tolist()))[:c["picked"] - 1]
                got = sorted(p for _, p in got) + [pages - 1]
                found[b, h, :len(got)] = torch.tensor(got, dtype=torch.int32, device="cuda")
        return found
    if c["op"] == "attention":
        out = torch.zeros(c["B"], H, S, D, dtype=torch.float64, device="cuda")
        for b, n in enumerate(lens):
            for h in range(Hkv):
                if s["picked"] is None:
                    pages = list(range(-(-n // page)))
                else:
                    pages = [p for p in s["picked"][b, h].tolist() if p >= 0]
                if not pages:
                    continue
                at = [table[b][p] for p in pages]
                k, v = s["kp"][at, h].double().flatten(0, 1), s["vp"][at, h].double().flatten(0, 1)
                place = (torch.tensor(pages, device="cuda")[:, None] * page + torch.arange(page, device="cuda")).flatten()
                for i in range(new[b]):
                    seen = place <= n - new[b] + i
                    q = s["q"][b, h * G:(h + 1) * G, i].double()
                    out[b, h * G:(h + 1) * G, i] = torch.softmax(q @ k[seen].t() * s["scale"], dim=-1) @ v[seen]
        return out
    q = s["q"].double() if c["rot"] else None
    kp, vp = s["kp"].double(), s["vp"].double()
    bounds = None if s["bounds"] is None else s["bounds"].double()
    for b, n in enumerate(lens):
        m = new[b]
        if q is not None:
            q[b, :, m:] = 0
        if m == 0:
            continue
        k = s["k"][b, :, :m].double()
        place = torch.arange(n - m, n, device="cuda")
        if c["rot"]:
            r = c["rot"]
            turn = torch.complex(s["cos"][place].double(), s["sin"][place].double())
            for x in (k, q[b, :, :m]):
                part = x[..., :r].unflatten(-1, (-1, 2)) if c["pairs"] else x[..., :r].unflatten(-1, (2, -1)).transpose(-1, -2)
                z = torch.view_as_real(torch.view_as_complex(part.contiguous()) * turn)
                x[..., :r] = (z if c["pairs"] else z.transpose(-1, -2)).flatten(-2)
        for p in range((n - m) // page, -(-n // page)):
            a, e = max(p * page, n - m), min((p + 1) * page, n)
            row = table[b][p]
            kk = k[:, a - n + m:e - n + m]
            kp[row, :, a - p * page:e - p * page] = kk
            vp[row, :, a - p * page:e - p * page] = s["v"][b, :, a - n + m:e - n + m].double()
            if bounds is not None:
                lo, hi = kk.amin(dim=1), kk.amax(dim=1)
                if a > p * page:
                    lo, hi = torch.minimum(lo, bounds[row, :, 0]), torch.maximum(hi, bounds[row, :, 1])
                bounds[row, :, 0], bounds[row, :, 1] = lo, hi
    return ([] if q is None else [q]) + [kp, vp] + ([] if bounds is None else [bounds])
