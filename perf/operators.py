"""Cases for the drafter's key/value cache: the page plan, the append, and the two attentions that read it.

Serving keeps every request's keys and values in pages of one pool.  A step of a batch of
requests plans its pages (``cache_plan``: pages taken and given back, block tables, slot
maps), writes the new rows' keys and values into them (``cache_append``), and attends from
the new rows to everything cached before them (``attn_paged``); requests that were forked
from one prompt attend to its pages together (``attn_paged_shared``).

Shapes: q ``[T, Hq * hd]`` holds the new rows of all requests one after another, request b
in rows ``cu[b] .. cu[b + 1]``; the caches are ``[pages, Hkv, page, hd]``; request b's key t
lies in page ``table[b, t // page]`` at ``t % page``; ``lens[b]`` counts its keys, the new
rows among them, so its row j sees the keys below ``lens[b] - n_b + j + 1``.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEV = "cuda"
_DT = {"bf16": torch.bfloat16, "fp32": torch.float32}
_GOLD = 0.6180339887498949


# ------------------------------------------------------------------- cases ----


def listed():
    heads_7b = dict(hq=28, hkv=4, hd=128)  # the 7B-class drafter
    heads_14b = dict(hq=40, hkv=8, hd=128)  # the 14B-class drafter
    heads_half_b = dict(hq=14, hkv=2, hd=64)  # heads of the smallest targets
    heads_tiny = dict(hq=4, hkv=2, hd=64)  # the fp32 configuration
    return [
        # a handful of interactive requests draft their next tokens
        dict(name="plan_draft_8", op="plan", batch=8, len_min=90, len_max=2000, grow_min=5,
             grow_max=9, page=64, fresh=0),
        # a serving batch takes in new prompts while others finish
        dict(name="plan_prompts_512", op="plan", batch=512, len_min=0, len_max=2048, grow_min=1,
             grow_max=4093, page=16, fresh=2),
        # the rows of that handful's draft step, fp32
        dict(name="append_draft_48", op="append", rows=48, hkv=2, hd=64, page=64, dtype="fp32"),
        # a batch of prompts' rows
        dict(name="append_prompts_16411", op="append", rows=16411, hkv=8, hd=128, page=64,
             dtype="bf16"),
        # one request, one token: only latency counts
        dict(name="paged_token_1x600", op="paged", batch=1, len_min=601, len_max=601, q_min=1,
             q_max=1, page=64, dtype="bf16", **heads_half_b),
        # a few requests verify and draft: accepted tokens plus prediction slots, ragged
        dict(name="paged_draft_8x8k", op="paged", batch=8, len_min=900, len_max=8200, q_min=5,
             q_max=9, page=64, dtype="bf16", **heads_7b),
        # a full serving batch, one token each, lengths far apart
        dict(name="paged_token_64x32k", op="paged", batch=64, len_min=1000, len_max=32700,
             q_min=1, q_max=1, page=64, dtype="bf16", **heads_7b),
        # prompts in chunks: many rows against a cache that holds what came before
        dict(name="paged_prompt_2x4k", op="paged", batch=2, len_min=3500, len_max=4500,
             q_min=900, q_max=1100, page=32, dtype="bf16", **heads_7b),
        # fp32 serving of the small configuration
        dict(name="paged_fp32_16x2k", op="paged", batch=16, len_min=100, len_max=2050, q_min=1,
             q_max=5, page=16, dtype="fp32", **heads_tiny),
        # a few samples of one short prompt
        dict(name="shared_4x512", op="shared", batch=4, shared=512, len_min=5, len_max=77,
             q_min=1, q_max=1, page=64, dtype="bf16", **heads_half_b),
        # drafts for samples of one prompt
        dict(name="shared_32x8k", op="shared", batch=32, shared=8192, len_min=9, len_max=300,
             q_min=5, q_max=5, page=64, dtype="bf16", **heads_7b),
        # many samples of one long document
        dict(name="shared_64x64k", op="shared", batch=64, shared=65536, len_min=20, len_max=1000,
             q_min=4, q_max=6, page=128, dtype="bf16", **heads_14b),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["plan", "append", "paged", "paged", "shared", "shared"])
    page = rng.choice([16, 32, 64, 128])
    if op == "plan":
        fresh = rng.choice([0, 2, 3])
        batch = _log_int(rng, 1, 512)
        grow = _log_int(rng, 1, max(1, min(4096, 1_000_000 // batch))) if fresh else \
            rng.randint(1, 17)
        return dict(op=op, batch=batch, len_min=rng.randint(0, 100),
                    len_max=_log_int(rng, 101, 8192), grow_min=rng.randint(1, grow),
                    grow_max=grow, page=page, fresh=fresh)
    if op == "append":
        hkv, hd = rng.choice([(4, 128), (2, 64), (8, 128), (5, 128), (1, 64)])
        return dict(op=op, rows=_log_int(rng, 1, 16400), hkv=hkv, hd=hd, page=page,
                    dtype=rng.choice(["bf16", "bf16", "fp32"]))
    hq, hkv, hd = rng.choice([(28, 4, 128), (40, 8, 128), (14, 2, 64), (4, 2, 64), (15, 5, 128),
                              (6, 6, 64)])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
    if op == "paged":
        if rng.random() < 0.25:  # a prompt in chunks
            dtype, batch = "bf16", rng.randint(1, 3)
            q_max = _log_int(rng, 17, 1100)
            len_max = q_max + _log_int(rng, 1, 3400)
            return dict(op=op, batch=batch, len_min=q_max, len_max=len_max,
                        q_min=max(1, q_max // 2), q_max=q_max, page=page, dtype=dtype, hq=hq,
                        hkv=hkv, hd=hd)
        batch = _log_int(rng, 1, 64)
        cap = 900_000 if dtype == "bf16" else 60_000  # keys of the whole batch
        len_max = _log_int(rng, 17, max(18, min(131_000, cap // batch)))
        q_max = rng.randint(1, 16)
        return dict(op=op, batch=batch, len_min=rng.randint(min(16, len_max), len_max),
                    len_max=len_max, q_min=rng.randint(1, q_max), q_max=q_max, page=page,
                    dtype=dtype, hq=hq, hkv=hkv, hd=hd)
    batch = _log_int(rng, 2, 64)
    q_max = rng.randint(1, 6)
    cap = 60_000 if dtype == "bf16" else 4_000
    shared = max(1, _log_int(rng, page, cap) // page) * page
    len_max = _log_int(rng, 17, 1000 if dtype == "bf16" else 300)
    return dict(op=op, batch=batch, shared=shared, len_min=rng.randint(6, len_max),
                len_max=len_max, q_min=rng.randint(1, q_max), q_max=q_max, page=page,
                dtype=dtype, hq=hq, hkv=hkv, hd=hd)


def _spread(n, lo, hi, phase):
    """n whole numbers over lo..hi, spread evenly and out of order (no seed: part of the case)."""
    return [lo + int((hi - lo + 1) * ((phase + (i + 1) * _GOLD) % 1.0)) for i in range(n)]


def _requests(case):
    """(own keys, new rows) of every request of an attention case; the shared keys come on top."""
    lens = _spread(case["batch"], case["len_min"], case["len_max"], 0.2)
    news = _spread(case["batch"], case["q_min"], case["q_max"], 0.7)
    return lens, [min(n, t) for n, t in zip(news, lens)]


def _plan_lens(case):
    """(cached, wanted) of every request of a plan case."""
    b = case["batch"]
    have = _spread(b, case["len_min"], case["len_max"], 0.2)
    grow = _spread(b, case["grow_min"], case["grow_max"], 0.7)
    want = []
    for i in range(b):
        if case["fresh"] and i % case["fresh"] == 0:
            have[i] = 0  # a new request: its whole prompt
        if i % 8 == 5:
            want.append(0)  # a finished request gives its pages back
        elif i % 8 == 6:
            want.append(max(0, have[i] - grow[i] % 8))  # rejected drafts are taken back
        else:
            want.append(have[i] + grow[i])
    return have, want


# ------------------------------------------------------------------- state ----


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=DEV)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    page = case["page"]
    if case["op"] == "plan":
        have, want = _plan_lens(case)
        b = case["batch"]
        used = [-(-t // page) for t in have]
        need = [-(-t // page) for t in want]
        grown = sum(max(0, n - u) for n, u in zip(need, used))
        total = sum(used) + grown + 7
        perm = torch.randperm(total, device=DEV, generator=g, dtype=torch.int32)
        width = max(max(used), max(need), 1) + 1
        table = torch.full((b, width), -1, dtype=torch.int32, device=DEV)
        at = torch.arange(width, device=DEV)[None]
        first = torch.cumsum(_ints([0] + used[:-1], torch.int64), 0)[:, None]
        held = at < _ints(used)[:, None]
        table = torch.where(held, perm[(first + at).clamp_(max=total - 1)], table)
        free = torch.full((total,), -1, dtype=torch.int32, device=DEV)
        n_free, head = total - sum(used), total // 3
        free[(head + torch.arange(n_free, device=DEV)) % total] = perm[sum(used):]
        return dict(case=case, lens=_ints(have), new_lens=_ints(want), table=table.contiguous(),
                    free=free, ring=_ints([head, head + n_free, 0], torch.int64),
                    ring_out=_ints([0, 0, 0], torch.int64), page=page,
                    rows=sum(max(0, w - h) for h, w in zip(have, want)))
    dt = _DT[case["dtype"]]
    hkv, hd = case["hkv"], case["hd"]
    if case["op"] == "append":
        rows = case["rows"]
        pages = -(-(rows + rows // 8) // page) + 1
        slots = torch.randperm(pages * page, device=DEV, generator=g)[:rows]
        slots[:: max(7, rows // 5)] = -1  # rows behind a batch's last sequence have no slot
        k, v = (torch.randn(rows, hkv * hd, device=DEV, generator=g).to(dt) for _ in range(2))
        kc, vc = (torch.randn(pages, hkv, page, hd, device=DEV, generator=g).to(dt)
                  for _ in range(2))
        return dict(case=case, k=k, v=v, slots=slots, k_cache=kc, v_cache=vc)
    lens, news = _requests(case)
    shared = case.get("shared", 0)
    sp = shared // page
    used = [-(-t // page) for t in lens]
    width = sp + max(used)
    pages = sp + sum(used) + 3
    perm = torch.randperm(pages, device=DEV, generator=g, dtype=torch.int32)
    at = torch.arange(width, device=DEV)[None]
    first = torch.cumsum(_ints([0] + used[:-1], torch.int64), 0)[:, None]
    mine = (at >= sp) & (at < sp + _ints(used)[:, None])
    table = torch.where(mine, perm[(sp + first + at - sp).clamp_(0, pages - 1)],
                        torch.zeros((), dtype=torch.int32, device=DEV))
    if sp:
        table[:, :sp] = perm[:sp]
    rows = sum(news)
    cu = [0]
    for n in news:
        cu.append(cu[-1] + n)
    kc, vc = (torch.empty(pages, hkv, page, hd, dtype=dt, device=DEV).normal_(generator=g)
              for _ in range(2))
    q = torch.randn(rows, case["hq"] * hd, device=DEV, generator=g).to(dt)
    return dict(case=case, q=q, k_cache=kc, v_cache=vc, table=table.contiguous(),
                lens=_ints([shared + t for t in lens]), cu=_ints(cu), shared=shared,
                max_len=max(lens), max_new=max(news))


# --------------------------------------------------------------- plain forms ----


def _plan_plain(s):
    lens, want, table, free = (s[k].long() for k in ("lens", "new_lens", "table", "free"))
    page, total, width = s["page"], free.shape[0], table.shape[1]
    head, tail = s["ring"][0], s["ring"][1]
    used, need = (lens + page - 1) // page, (want + page - 1) // page
    grow, drop = (need - used).clamp(min=0), (used - need).clamp(min=0)
    grown, dropped = torch.cumsum(grow, 0), torch.cumsum(drop, 0)
    ok = ((grow == 0) | (grown <= tail - head)) & \
        ((drop == 0) | (dropped <= total - (tail - head)))
    at = torch.arange(width, device=lens.device)[None]
    fresh = (at >= used[:, None]) & (at < need[:, None]) & ok[:, None]
    src = head + (grown - grow)[:, None] + at - used[:, None]
    filled = torch.where(fresh, free[src % total], table)
    gone = (at >= need[:, None]) & (at < used[:, None]) & ok[:, None]
    dst = (tail + (dropped - drop)[:, None] + at - need[:, None]) % total
    back = torch.cat([free, free[:1]])
    back.scatter_(0, torch.where(gone, dst, total).reshape(-1), table.reshape(-1))
    s["table"].copy_(filled)
    s["free"].copy_(back[:total])
    new = (want - lens).clamp(min=0)
    cu = torch.cat([new.new_zeros(1), torch.cumsum(new, 0)])
    row = torch.arange(s["rows"], device=lens.device)
    b = torch.searchsorted(cu[1:], row, right=True)
    pos = lens[b] + row - cu[b]
    slots = filled[b, pos // page] * page + pos % page
    slots = torch.where(ok[b], slots, -1)
    s["ring_out"].copy_(torch.stack([head + torch.where(ok, grow, 0).sum(),
                                     tail + torch.where(ok, drop, 0).sum(), (~ok).sum()]))
    return (torch.where(ok, want, lens).int(), cu.int(), slots, pos, s["ring_out"], s["table"],
            s["free"])


def _append_plain(s):
    hkv, page, hd = s["k_cache"].shape[1:]
    keep = s["slots"] >= 0
    at = s["slots"][keep]
    for x, cache in ((s["k"], s["k_cache"]), (s["v"], s["v_cache"])):
        cache[at // page, :, at % page] = x[keep].unflatten(1, (hkv, hd))
    return s["k_cache"], s["v_cache"]


def _attn_plain(s):
    q, lens, cu, table = s["q"].float(), s["lens"].long(), s["cu"].long(), s["table"].long()
    pages, hkv, page, hd = s["k_cache"].shape
    rows, hq = q.shape[0], q.shape[1] // hd
    rep, batch, new, shared = hq // hkv, lens.shape[0], s["max_new"], s["shared"]
    sp, width = shared // page, -(-s["max_len"] // page)
    dev = q.device
    n = cu[1:] - cu[:-1]
    j = torch.arange(new, device=dev)
    pick = (cu[:-1, None] + j).clamp(max=rows - 1)  # [B, new]
    qp = q[pick].unflatten(2, (hkv, rep, hd)).permute(0, 2, 3, 1, 4) / math.sqrt(hd)
    qp = qp.reshape(batch, hkv, rep * new, hd)

    def own_keys(cache):
        x = cache[table[:, sp:sp + width]].float()  # [B, P, hkv, page, hd]
        return x.permute(0, 2, 1, 3, 4).reshape(batch, hkv, width * page, hd)

    key = shared + torch.arange(width * page, device=dev)
    sees = (key[None, None] < (lens - n)[:, None, None] + j[None, :, None] + 1)  # [B, new, keys]
    sees = sees[:, None, None].expand(batch, 1, rep, new, width * page).reshape(
        batch, 1, rep * new, width * page)
    x = (qp @ own_keys(s["k_cache"]).transpose(2, 3)).masked_fill_(~sees, -math.inf)
    m = x.amax(-1, keepdim=True)
    if sp:
        flat = qp.permute(1, 0, 2, 3).reshape(hkv, batch * rep * new, hd)
        kp, vp = (c[table[0, :sp]].permute(1, 0, 2, 3).reshape(hkv, shared, hd).float()
                  for c in (s["k_cache"], s["v_cache"]))
        y = flat @ kp.transpose(1, 2)
        m = torch.maximum(m, y.amax(-1).view(hkv, batch, rep * new).transpose(0, 1)[..., None])
        y = torch.exp(y - m.transpose(0, 1).reshape(hkv, batch * rep * new, 1))
    m = m.masked_fill(m == -math.inf, 0.0)
    x = torch.exp(x - m)
    total = x.sum(-1, keepdim=True)
    o = x @ own_keys(s["v_cache"])
    if sp:
        total = total + y.sum(-1).view(hkv, batch, rep * new).transpose(0, 1)[..., None]
        o = o + (y @ vp).view(hkv, batch, rep * new, hd).transpose(0, 1)
    o, lse = o / total, (m + torch.log(total))[..., 0]
    o = o.view(batch, hq, new, hd).transpose(1, 2).reshape(batch, new, hq * hd)
    lse = lse.view(batch, hq, new).transpose(1, 2)
    row = torch.arange(rows, device=dev)
    b = torch.searchsorted(cu[1:], row, right=True)
    return o[b, row - cu[b]].to(s["q"].dtype), lse[b, row - cu[b]].t().contiguous()


def run(state):
    op = state["case"]["op"]
    if own:
        from parallel_eagle_b200 import ops

        if op == "plan":
            granted, cu, slots, pos, ring = ops.cache_plan(
                state["lens"], state["new_lens"], state["table"], state["free"], state["ring"],
                state["page"], state["rows"], ring_out=state["ring_out"])
            return granted, cu, slots, pos, ring, state["table"], state["free"]
        if op == "append":
            ops.cache_append(state["k"], state["v"], state["slots"], state["k_cache"],
                             state["v_cache"])
            return state["k_cache"], state["v_cache"]
        if op == "paged":
            return ops.attn_paged(state["q"], state["k_cache"], state["v_cache"], state["table"],
                                  state["lens"], state["cu"])
        return ops.attn_paged_shared(state["q"], state["k_cache"], state["v_cache"],
                                     state["table"], state["lens"], state["cu"], state["shared"])
    if op == "plan":
        return _plan_plain(state)
    if op == "append":
        return _append_plain(state)
    return _attn_plain(state)


# ---------------------------------------------------------------- work, exact ----


def work(case):
    page = case["page"]
    if case["op"] == "plan":
        have, want = _plan_lens(case)
        rows = sum(max(0, w - h) for h, w in zip(have, want))
        moved = sum(abs(-(-w // page) + (-h // page)) for h, w in zip(have, want))
        # per row a slot and a position, per page moved one entry read and one written
        return {"bytes": 16 * rows + 8 * moved + 16 * case["batch"], "flops": 0}
    es = _DT[case["dtype"]].itemsize
    if case["op"] == "append":
        kept = case["rows"] - len(range(0, case["rows"], max(7, case["rows"] // 5)))
        return {"bytes": 4 * kept * case["hkv"] * case["hd"] * es + 8 * case["rows"], "flops": 0}
    lens, news = _requests(case)
    shared, rows = case.get("shared", 0), sum(news)
    pairs = sum(n * (shared + t) - n * (n - 1) // 2 for t, n in zip(lens, news))
    keys = shared + sum(lens)
    return {"bytes": 2 * keys * case["hkv"] * case["hd"] * es
            + 2 * rows * case["hq"] * case["hd"] * es + 4 * rows * case["hq"],
            "flops": 4 * pairs * case["hq"] * case["hd"]}


def exact(case, seed):
    """Attention from its definition in 64 bits, one request and head at a time; the append's
    copies.  The plan gives whole numbers, which have no rounding to judge."""
    if case["op"] == "plan":
        return None
    s = prepare(case, seed)
    if case["op"] == "append":
        _, hkv, page, hd = s["k_cache"].shape
        row = torch.nonzero(s["slots"] >= 0)[:, 0]
        at, out = s["slots"][row], []
        for x, cache in ((s["k"], s["k_cache"]), (s["v"], s["v_cache"])):
            by_slot = cache.transpose(1, 2).reshape(-1, hkv * hd).double()
            by_slot[at] = x[row].double()
            out.append(by_slot.view(-1, page, hkv, hd).transpose(1, 2).contiguous())
        return tuple(out)
    lens, cu, table = s["lens"].tolist(), s["cu"].tolist(), np.asarray(s["table"].cpu())
    pages, hkv, page, hd = s["k_cache"].shape
    hq = case["hq"]
    o = torch.empty(cu[-1], hq, hd, dtype=torch.float64, device=DEV)
    lse = torch.empty(hq, cu[-1], dtype=torch.float64, device=DEV)
    for b, total in enumerate(lens):
        idx = torch.from_numpy(table[b, :-(-total // page)].astype(np.int64)).to(DEV)
        new = cu[b + 1] - cu[b]
        limit = torch.arange(total - new + 1, total + 1, device=DEV)[:, None]
        hidden = torch.arange(total, device=DEV)[None] >= limit
        for h in range(hkv):
            k, v = (c[idx, h].reshape(-1, hd)[:total].double() for c in (s["k_cache"],
                                                                        s["v_cache"]))
            for i in range(h * (hq // hkv), (h + 1) * (hq // hkv)):
                z = s["q"][cu[b]:cu[b + 1], i * hd:(i + 1) * hd].double() @ k.t() * hd ** -0.5
                z[hidden] = -math.inf
                top = torch.logsumexp(z, 1)
                lse[i, cu[b]:cu[b + 1]] = top
                o[cu[b]:cu[b + 1], i] = torch.exp(z - top[:, None]) @ v
    return o.reshape(cu[-1], hq * hd), lse
