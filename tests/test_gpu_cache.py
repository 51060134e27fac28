"""The paged key/value cache on the GPU: page plan, append, and the attention that reads it.

* The plan against a sequential restatement of its rules in Python (whole numbers: equal).
* The append against indexing (copies: equal).
* Attention against its definition in 64 bits, row by row, with tolerances from rounding:
  with A = sum_t p_t |v_t| / sum_t p_t per output element,
  - bf16: probabilities and the result are each rounded once (2^-8 of A and of |o| <= A),
    and the exponentials are good to 2^-12, so |error| <= (2 * 2^-8 + 2^-11) A;
  - fp32: a score is off by at most (hd + 8) 2^-24 sum|q k| / sqrt(hd) (products and sum),
    which moves a probability by that, relatively, twice (its own and the maximum's), and
    sums of L terms add (L + 64) 2^-24.
"""

from __future__ import annotations

import math
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("needs a CUDA device", allow_module_level=True)

from parallel_eagle_b200 import _lib as L  # noqa: E402
from parallel_eagle_b200 import ops  # noqa: E402

DEV = torch.device("cuda", 0)
BF16, F32 = torch.bfloat16, torch.float32


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


# ---------------------------------------------------------------- page plan ----


def plan_reference(lens, want, table, free, head, tail, page, rows, shared=0):
    """The plan's rules, request by request, on Python lists (table and free in place)."""
    n, width, sp = len(free), len(table[0]), shared // page
    avail, room = tail - head, len(free) - (tail - head)
    taken = given = refused = 0
    granted, cu, slots, pos = [], [0], [], []
    pushes, broke_grow, broke_drop = [], False, False
    for b, (a, z) in enumerate(zip(lens, want)):
        fits = min(a, z) >= shared and -(-a // page) <= width and -(-z // page) <= width
        used, need = max(-(-a // page), sp), max(-(-z // page), sp)
        ok = fits
        if fits and need > used:
            broke_grow = broke_grow or taken + need - used > avail
            ok = not broke_grow
            if ok:
                for i in range(used, need):
                    table[b][i] = free[(head + taken) % n]
                    taken += 1
        if fits and need < used:
            broke_drop = broke_drop or given + used - need > room
            ok = not broke_drop
            if ok:
                for i in range(need, used):
                    pushes.append(((tail + given) % n, table[b][i]))
                    given += 1
        refused += not ok
        granted.append(z if ok else a)
        for p in range(a, z):
            slots.append(table[b][p // page] * page + p % page if ok else -1)
            pos.append(p)
        cu.append(cu[-1] + max(0, z - a))
    for i, v in pushes:
        free[i] = v
    slots, pos = slots[:rows], pos[:rows]
    pad = rows - len(slots)
    return granted, cu, slots + [-1] * pad, pos + [0] * pad, [head + taken, tail + given, refused]


def run_plan(lens, want, table, free, head, tail, page, rows, shared=0):
    t, f = _i32(table), _i32(free)
    ring = torch.tensor([head, tail, 0], device=DEV)
    got = ops.cache_plan(_i32(lens), _i32(want), t, f, ring, page, rows, shared=shared)
    exp_table, exp_free = [list(r) for r in table], list(free)
    exp = plan_reference(lens, want, exp_table, exp_free, head, tail, page, rows, shared)
    for name, g, e in zip(("granted", "cu", "slots", "pos", "ring"), got, exp):
        assert g.tolist() == e, name
    assert t.tolist() == exp_table and f.tolist() == exp_free
    assert ring.tolist() == [head, tail, 0]
    return got


def _plan_case(batch, page, width, extra, seed, most=None, head=0, shared=0):
    r = torch.Generator().manual_seed(seed)
    rnd = lambda lo, hi: int(torch.randint(lo, hi + 1, (1,), generator=r))  # noqa: E731
    most = most or width * page
    lens = [rnd(shared, most) if rnd(0, 4) else shared for _ in range(batch)]
    want = []
    for n in lens:
        k = rnd(0, 3)
        want.append(shared if k == 0 else min(most, n + rnd(0, 9)) if k < 3 else rnd(shared, most))
    sp = shared // page
    used = [max(-(-n // page), sp) for n in lens]
    own = sum(u - sp for u in used)
    total = own + extra + sp
    perm = torch.randperm(total, generator=r).tolist()
    table, at = [], sp
    for u in used:
        row = perm[:sp] + perm[at:at + u - sp]
        at += u - sp
        table.append(row + [-7] * (width - len(row)))
    free = [-1] * total
    for i in range(extra):
        free[(head + i) % total] = perm[at + i]
    rows = sum(max(0, w - n) for n, w in zip(lens, want))
    return lens, want, table, free, head, head + extra, page, rows, shared


@pytest.mark.parametrize("batch,page,width,extra,head", [
    (1, 16, 4, 9, 0), (3, 64, 3, 40, 5), (33, 16, 17, 700, 123), (517, 16, 5, 3000, 10**12 + 7),
    (1500, 32, 3, 5000, 1), (8192, 16, 2, 20000, 77),
])
def test_plan_matches_sequential_rules(batch, page, width, extra, head):
    run_plan(*_plan_case(batch, page, width, extra, seed=batch + page, head=head))


def test_plan_runs_out_of_pages_in_request_order():
    for extra in (0, 1, 2, 5, 11):
        run_plan(*_plan_case(40, 16, 9, extra, seed=extra, head=3))


def test_plan_with_shared_prefix_leaves_its_pages():
    case = _plan_case(50, 16, 12, 900, seed=4, head=2, shared=48)
    got = run_plan(*case)
    assert int(got[4][2]) == 0


def test_plan_refuses_lengths_below_the_shared_prefix():
    """Rows below it would land in the pages that all requests read."""
    table = [[8, 9, 0], [8, 9, 1], [8, 9, 2]]
    free = [3, 4, 5, -1, -1, -1, -1, -1, -1, -1]
    # (request 0 outgrows the table's three pages)
    got = run_plan([32, 10, 40], [50, 40, 16], table, free, 0, 3, 16, 18 + 30, shared=32)
    assert got[0].tolist() == [32, 10, 40] and int(got[4][2]) == 3
    got = run_plan([32, 10, 40], [47, 40, 16], table, free, 0, 3, 16, 15 + 30, shared=32)
    assert got[0].tolist() == [47, 10, 40] and int(got[4][2]) == 2


def test_plan_refuses_lengths_and_pads_rows():
    table = [[0, 1, 2], [3, 4, 5], [6, -1, -1], [7, -1, -1]]
    free = [8, 9, -1, -1, -1, -1, -1, -1, -1, -1]
    # request 0 outgrows the table, 1 has a negative target, 2 grows, 3 stays
    run_plan([48, 40, 10, 9], [49, -1, 33, 9], table, free, 0, 2, 16, 24 + 5)
    # fewer rows than the plan makes: the first ones are described
    run_plan([48, 40, 10, 9], [48, 40, 33, 9], table, free, 0, 2, 16, 7)
    # no new rows at all
    run_plan([48, 40, 10, 9], [48, 8, 10, 0], table, free, 0, 2, 16, 0)


def test_plan_large_prompts_and_idempotence():
    case = _plan_case(200, 16, 600, 60000, seed=9, most=9000, head=31)
    first = run_plan(*case)
    t, f = _i32(case[2]), _i32(case[3])
    ring = torch.tensor([case[4], case[5], 0], device=DEV)
    for _ in range(2):  # unless the ring advances, a second call plans the same
        again = ops.cache_plan(_i32(case[0]), _i32(case[1]), t, f, ring, case[6], case[7])
        for a, b in zip(first, again):
            assert torch.equal(a, b)


def test_plan_ignores_impossible_ring_counters():
    t, f = _i32([[3, -1]]), _i32([0, 1, 2, 9])
    for head, tail in ((-5, 2), (3, 1), (0, 99)):
        ring = torch.tensor([head, tail, 0], device=DEV)
        granted, _, slots, _, out = ops.cache_plan(_i32([5]), _i32([20]), t, f, ring, 16, 15)
        assert granted.tolist() == [5] and out.tolist() == [head, tail, 1]
        assert slots.tolist() == [-1] * 15
    assert t.tolist() == [[3, -1]] and f.tolist() == [0, 1, 2, 9]


# ------------------------------------------------------------------- append ----


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,hkv,hd,page,pad", [
    (1, 1, 64, 16, 0), (7, 4, 128, 64, 0), (37, 2, 64, 16, 8), (129, 3, 80, 48, 0),
    (65, 2, 33, 16, 0), (50, 5, 20, 32, 3), (2049, 8, 128, 128, 0),
])
def test_append(dtype, rows, hkv, hd, page, pad):
    g = _gen(rows)
    width = hkv * hd
    fused = torch.randn(rows, 2 * width + pad, device=DEV, generator=g).to(dtype)
    k, v = fused[:, :width], fused[:, width:2 * width]  # row views of one projection
    pages = -(-rows // page) + 2
    slots = torch.randperm(pages * page, device=DEV, generator=g)[:rows].contiguous()
    slots[::5] = -1
    if rows > 3:
        slots[3] = pages * page  # behind the cache: skipped
    kc, vc = (torch.randn(pages, hkv, page, hd, device=DEV, generator=g).to(dtype)
              for _ in range(2))
    ek, ev = kc.clone(), vc.clone()
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < pages * page:
            ek[s // page, :, s % page] = k[t].view(hkv, hd)
            ev[s // page, :, s % page] = v[t].view(hkv, hd)
    ops.cache_append(k, v, slots, kc, vc)
    assert torch.equal(kc, ek) and torch.equal(vc, ev)


def test_append_no_rows_and_far_slots():
    kc = torch.zeros(3, 2, 16, 64, dtype=BF16, device=DEV)
    empty = torch.empty(0, 128, dtype=BF16, device=DEV)
    ops.cache_append(empty, empty, torch.empty(0, dtype=torch.int64, device=DEV), kc, kc.clone())
    far = torch.tensor([2**40, -2**40, 5], device=DEV)
    x = torch.ones(3, 128, dtype=BF16, device=DEV)
    ops.cache_append(x, x, far, kc, kc)
    assert kc.sum().item() == 128 and kc[0, :, 5].sum().item() == 128


# ---------------------------------------------------------------- attention ----


def reference(q, kc, vc, table, lens, cu, hq):
    """(o, A, lse, largest sum|q k| / sqrt(hd)) in 64 bits, A = sum p |v| / sum p."""
    hkv, page, hd = kc.shape[1:]
    T = q.shape[0]
    o = torch.zeros(T, hq, hd, dtype=torch.float64, device=DEV)
    A = torch.zeros_like(o)
    lse = torch.full((hq, T), -math.inf, dtype=torch.float64, device=DEV)
    big = 0.0
    for b in range(len(lens)):
        n = cu[b + 1] - cu[b]
        top = max(0, lens[b])
        pages = table[b, :-(-top // page)].long() if top else table[b, :0].long()
        k, v = (c[pages].transpose(0, 1).reshape(hkv, -1, hd)[:, :top].double()
                for c in (kc, vc))
        for j in range(n):
            see = lens[b] - n + j + 1
            if see <= 0:
                continue
            qr = q[cu[b] + j].view(hkv, hq // hkv, hd).double()
            z = qr @ k[:, :see].transpose(1, 2) * hd ** -0.5
            big = max(big, float((qr.abs() @ k[:, :see].abs().transpose(1, 2)).max()) * hd ** -0.5)
            top_z = z.logsumexp(-1, keepdim=True)
            p = torch.exp(z - top_z)
            o[cu[b] + j] = (p @ v[:, :see]).reshape(hq, hd)
            A[cu[b] + j] = (p @ v[:, :see].abs()).reshape(hq, hd)
            lse[:, cu[b] + j] = top_z.reshape(hq)
    return o.view(T, -1), A.view(T, -1), lse, big


def make(lens, news, hq, hkv, hd, page, dtype, seed=0, shared=0, garbage=True, scale=1.0,
         extra_rows=0):
    """Inputs of one call.  Pool and table hold NaN and wild entries wherever no key lies."""
    g = _gen(seed)
    sp = shared // page
    used = [max(sp, -(-max(0, t) // page)) for t in lens]
    pages = sp + sum(u - sp for u in used) + 2
    perm = torch.randperm(pages, device=DEV, generator=g, dtype=torch.int32)
    width = max(max(used), 1) + 1
    table = torch.full((len(lens), width), 2**31 - 1 if garbage else 0, dtype=torch.int32,
                       device=DEV)
    kc, vc = (torch.full((pages, hkv, page, hd), math.nan, device=DEV) for _ in range(2))
    at = sp
    for b, t in enumerate(lens):
        table[b, :sp] = perm[:sp]
        table[b, sp:used[b]] = perm[at:at + used[b] - sp]
        at += used[b] - sp
        for i in range(0 if b == 0 else sp, used[b]):
            m = min(page, t - i * page)
            if m > 0:
                pid = int(table[b, i])
                kc[pid, :, :m] = torch.randn(hkv, m, hd, device=DEV, generator=g) * scale
                vc[pid, :, :m] = torch.randn(hkv, m, hd, device=DEV, generator=g)
    cu = [0]
    for n in news:
        cu.append(cu[-1] + n)
    q = torch.randn(cu[-1] + extra_rows, hq * hd, device=DEV, generator=g)
    return q.to(dtype), kc.to(dtype), vc.to(dtype), table, list(lens), cu


def check(q, kc, vc, table, lens, cu, hq, o, lse):
    hd = kc.shape[3]
    n = cu[-1]
    ro, A, rlse, big = reference(q[:n], kc, vc, table, lens, cu, hq)
    score = (hd + 8) * 2.0 ** -24 * big
    longest = max(max(lens), 1)
    sums = (longest + 64) * 2.0 ** -24
    if q.dtype == BF16:
        tol = (2 * 2.0 ** -8 + 2.0 ** -11) * A + 2 * score * A
        ltol = 2.0 ** -12 + score + sums
    else:
        tol = (sums + 2 * score + 2.0 ** -22) * A
        ltol = sums + score + 2.0 ** -22
    # + the rounding of lse itself
    o, lse = o[:n].double(), lse[:, :n].double()
    assert torch.isfinite(o).all()
    over = (o - ro).abs() - tol
    assert (over <= 1e-30).all(), f"o over its tolerance by {over.max().item():.3g}"
    dead = rlse == -math.inf
    assert torch.equal(lse == -math.inf, dead)
    gap = torch.where(dead, 0.0, lse - torch.where(dead, 0.0, rlse)).abs()
    gap = torch.where(dead, 0.0, gap - rlse.abs().nan_to_num(0, 0, 0) * 2.0 ** -23)
    assert (gap <= ltol).all(), f"lse off by {gap.max().item():.3g}, {ltol:.3g} allowed"
    rows_dead = dead.t().unsqueeze(-1).expand(n, hq, hd).reshape(n, -1)
    assert (o[rows_dead] == 0).all()


def attend(case, shared=0, algo=L.ALGO_AUTO, once=True, **kw):
    q, kc, vc, table, lens, cu = case
    if shared:
        return ops.attn_paged_shared(q, kc, vc, table, _i32(lens), _i32(cu), shared,
                                     algo=algo | (L.PAGED_PREFIX_ONCE if once else 0), **kw)
    return ops.attn_paged(q, kc, vc, table, _i32(lens), _i32(cu), algo=algo, **kw)


HEADS = [(28, 4, 128), (40, 8, 128), (14, 2, 64), (4, 2, 64), (5, 5, 128), (12, 1, 64)]
ODD_HEADS = [(6, 3, 80), (4, 2, 20), (2, 1, 33), (3, 1, 256), (2, 2, 1)]
BATCHES = [
    ([1], [1]),                                        # a first token
    ([600], [1]),
    ([77, 16, 129, 1, 128], [1, 1, 1, 1, 1]),          # single tokens
    ([300, 9, 65, 1025], [5, 9, 1, 7]),                # drafts
    ([40, 33, 0, 17], [3, 0, 0, 17]),                  # requests without rows, a whole prompt
    ([2, 0, 130], [5, 2, 3]),                          # rows that see nothing
    ([700, 260], [150, 260]),                          # prompts
]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("batch", range(len(BATCHES)))
def test_attention(dtype, heads, batch):
    hq, hkv, hd = heads
    lens, news = BATCHES[batch]
    case = make(lens, news, hq, hkv, hd, [16, 64, 32, 128][batch % 4], dtype, seed=batch)
    check(*case, hq, *attend(case))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads", ODD_HEADS)
def test_attention_odd_head_sizes(dtype, heads):
    hq, hkv, hd = heads
    for i in (2, 3, 5):
        lens, news = BATCHES[i]
        case = make(lens, news, hq, hkv, hd, 48, dtype, seed=i)
        check(*case, hq, *attend(case))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("page", [16, 48, 64, 256])
def test_attention_long_ragged(dtype, page):
    """Long and short requests together: entities split over many blocks."""
    lens = [5000, 3, 2300, 17, 4097, 640]
    for news in ([1] * 6, [5, 3, 7, 2, 1, 9]):
        case = make(lens, news, 28, 4, 128, page, dtype, seed=page)
        check(*case, 28, *attend(case))
    case = make([9000], [6], 14, 2, 64, page, dtype, seed=page + 1)
    check(*case, 14, *attend(case))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("hd", [64, 128])
def test_attention_of_one_long_request(dtype, hd):
    """One request over all blocks (its pieces joined), single tokens and drafts."""
    for total, n in ((70001, 1), (33333, 5), (20000, 40)):
        case = make([total], [n], 4, 1, hd, 128, dtype, seed=n)
        check(*case, 4, *attend(case))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_row_offsets_that_make_no_sense_stay_in_bounds(dtype):
    """Offsets behind the rows, or running backwards: nothing outside the rows is touched."""
    q, kc, vc, table, lens, _ = make([90, 60, 30], [4, 4, 4], 4, 2, 64, 16, dtype)
    for cu in ([0, 400, 800, 1200], [5, 2, 9, 1], [-7, 3, 3, 2**31 - 1], [0, 4, 8, 12]):
        out = torch.full((q.shape[0] + 2, q.shape[1]), 7.0, dtype=dtype, device=DEV)
        o, _ = ops.attn_paged(q, kc, vc, table, _i32(lens), _i32(cu), o=out[1:-1])
        assert (out[0] == 7).all() and (out[-1] == 7).all()
    check(q, kc, vc, table, lens, cu, 4, *attend((q, kc, vc, table, lens, cu)))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads", [(28, 4, 128), (14, 2, 64), (6, 6, 128)])
@pytest.mark.parametrize("shared", [16, 64, 208, 1024])
def test_shared_prefix(dtype, heads, shared):
    hq, hkv, hd = heads
    for own, news in (([1, 30, 7], [1, 1, 1]), ([9, 150, 6, 70], [5, 6, 6, 1]),
                      ([20] * 40, [5] * 40), ([12, 3], [0, 2])):
        lens = [shared + t for t in own]
        case = make(lens, news, hq, hkv, hd, 16, dtype, seed=shared, shared=shared)
        check(*case, hq, *attend(case, shared=shared))
        check(*case, hq, *attend(case, shared=shared, once=False))  # by size


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_shared_prefix_only(dtype):
    """Requests that hold nothing but the prefix: single rows behind its last key."""
    case = make([64 + 1, 64 + 1], [1, 1], 8, 2, 64, 32, dtype, shared=64)
    check(*case, 8, *attend(case, shared=64))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_large_scores(dtype):
    """Scores far apart (a running maximum that keeps rising, and underflowing tails)."""
    case = make([2000, 130], [3, 1], 8, 2, 128, 64, dtype, scale=30.0)
    check(*case, 8, *attend(case))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rising_scores(dtype):
    """Keys whose scores rise along the sequence: every tile raises the maximum."""
    q, kc, vc, table, lens, cu = make([1500], [4], 4, 2, 64, 64, dtype)
    for i in range(-(-1500 // 64)):
        kc[int(table[0, i])] *= 0.1 + 0.5 * i
    case = (q, kc, vc, table, lens, cu)
    check(*case, 4, *attend(case))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_strides_padding_and_given_outputs(dtype):
    """q as a view of a wider projection, o a view, unaligned rows, rows behind the last
    request, a table view; nothing but the requests' rows is written."""
    for pad, shift in ((8, 0), (3, 1)):
        q, kc, vc, table, lens, cu = make([90, 300], [4, 6], 14, 2, 64, 16, dtype, extra_rows=7)
        T = q.shape[0]
        wide = torch.full((T, 14 * 64 + pad), math.nan, dtype=dtype, device=DEV)
        wide[:, shift:shift + 14 * 64] = q
        qv = wide[:, shift:shift + 14 * 64]
        out = torch.full((T, 14 * 64 + pad), 7.0, dtype=dtype, device=DEV)
        lse = torch.full((14, T), 7.0, device=DEV)
        wt = torch.full((2, table.shape[1] + 5), -3, dtype=torch.int32, device=DEV)
        wt[:, :table.shape[1]] = table
        case = (qv, kc, vc, wt[:, :table.shape[1]], lens, cu)
        o, l2 = attend(case, o=out[:, shift:shift + 14 * 64], lse=lse)
        assert o.data_ptr() == out.data_ptr() + shift * out.element_size() and l2 is lse
        check(*case, 14, o, lse)
        assert (out[cu[-1]:] == 7).all() and (lse[:, cu[-1]:] == 7).all()
        assert (out[:, :shift] == 7).all() and (out[:, shift + 14 * 64:] == 7).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_block_table_entries_outside_the_pool_read_as_zero(dtype):
    q, kc, vc, table, lens, cu = make([64 + 9], [2], 4, 2, 64, 16, dtype)
    bad = table.clone()
    for wild in (-1, kc.shape[0], 2**31 - 1, -2**31):
        bad[0, 1] = wild
        o, lse = attend((q, kc, vc, bad, lens, cu))
        # the same as a page of zeros
        kz, vz = (torch.cat([c, torch.zeros_like(c[:1])]) for c in (kc, vc))
        good = table.clone()
        good[0, 1] = kc.shape[0]
        check(q, kz, vz, good, lens, cu, 4, o, lse)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_lengths_behind_the_table_stay_inside_it(dtype):
    """A length the table cannot hold attends to the keys the table has."""
    q, kc, vc, table, lens, cu = make([64], [1], 4, 2, 64, 16, dtype)
    o, lse = ops.attn_paged(q, kc, vc, table[:, :4], _i32([64 + 500]), _i32(cu))
    check(q, kc, vc, table, lens, cu, 4, o, lse)


def test_nan_in_visible_places_is_seen():
    for dtype in (BF16, F32):
        case = make([100, 100], [1, 1], 4, 2, 64, 16, dtype)
        case[1][int(case[3][0, 2]), 0, 3, 5] = math.nan
        o, _ = attend(case)
        assert torch.isnan(o[0, :128]).all() and torch.isfinite(o[0, 128:]).all()
        assert torch.isfinite(o[1]).all()


@pytest.mark.parametrize("shared", [0, 128])
def test_runs_repeat_bit_for_bit(shared):
    for dtype in (BF16, F32):
        case = make([shared + 2500, shared + 31, shared + 800], [5, 3, 7], 28, 4, 128, 64, dtype,
                    shared=shared)
        o, lse = attend(case, shared=shared)
        for _ in range(3):
            o2, l2 = attend(case, shared=shared)
            assert torch.equal(o, o2) and torch.equal(lse, l2)


@pytest.mark.parametrize("shared", [0, 64])
def test_capture_replay_and_side_stream(shared):
    """One captured step (plan, append, attention) replayed on new contents, next to eager
    calls on another stream."""
    dtype, page, hq, hkv, hd = BF16, 16, 14, 2, 64
    q, kc, vc, table, lens, cu = make([shared + 100, shared + 37], [5, 6], hq, hkv, hd, page,
                                      dtype, shared=shared)
    pages = kc.shape[0]
    own = -(-max(lens) // page)
    ln, want, tab = _i32([n - r for n, r in zip(lens, (5, 6))]), _i32(lens), table.clone()
    free = torch.zeros(pages, dtype=torch.int32, device=DEV)
    ring = torch.tensor([0, 2, 0], device=DEV)
    free[:2] = torch.tensor([pages - 2, pages - 1], device=DEV)
    k = torch.randn(11, hkv * hd, device=DEV, generator=_gen(5)).to(dtype)
    v = torch.randn(11, hkv * hd, device=DEV, generator=_gen(6)).to(dtype)
    assert own <= table.shape[1]

    def step():
        granted, c, slots, pos, out = ops.cache_plan(ln, want, tab, free, ring, page, 11,
                                                     shared=shared)
        ops.cache_append(k, v, slots, kc, vc)
        if shared:
            return ops.attn_paged_shared(q, kc, vc, tab, granted, c, shared,
                                         algo=L.PAGED_PREFIX_ONCE)
        return ops.attn_paged(q, kc, vc, tab, granted, c)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o, lse = step()
    for seed in (1, 2):
        q.copy_(torch.randn(q.shape, device=DEV, generator=_gen(seed)).to(dtype))
        k.copy_(torch.randn(k.shape, device=DEV, generator=_gen(seed + 9)).to(dtype))
        g.replay()
        with torch.cuda.stream(s):  # its own call on another stream, in flight together
            s.wait_stream(torch.cuda.current_stream())
        check(q, kc, vc, tab, lens, cu, hq, o, lse)


def test_concurrent_streams_do_not_share_scratch():
    cases = [make([3000 + 100 * i, 40], [2, 3], 28, 4, 128, 64, BF16, seed=i) for i in range(3)]
    want = [attend(c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = []
    for _ in range(5):
        got = []
        for c, s in zip(cases, streams):
            with torch.cuda.stream(s):
                got.append(attend(c))
    torch.cuda.synchronize()
    for (o, lse), (o2, l2) in zip(want, got):
        assert torch.equal(o, o2) and torch.equal(lse, l2)


@pytest.mark.parametrize("dtype", [BF16])
def test_pools_beyond_32_bit_offsets(dtype):
    """Pages whose elements lie past 2^31 of the pool."""
    hkv, page, hd = 4, 64, 128
    pages = 2**31 // (hkv * page * hd) + 40
    if torch.cuda.mem_get_info()[0] < 12 * 2**30:
        pytest.skip("needs 12 GB")
    q, kc, vc, table, lens, cu = make([900], [3], 8, hkv, hd, page, dtype)
    big_k, big_v = (torch.empty(pages, hkv, page, hd, dtype=dtype, device=DEV) for _ in range(2))
    n = kc.shape[0]
    big_k[-n:], big_v[-n:] = kc, vc
    far = torch.where(table < n, table + pages - n, table)
    case = (q, big_k, big_v, far, lens, cu)
    o, lse = attend(case)
    check(q, kc, vc, table, lens, cu, 8, o, lse)
    k = torch.randn(2, hkv * hd, device=DEV).to(dtype)
    slot = torch.tensor([pages * page - 1, pages * page - page], device=DEV)
    ops.cache_append(k, -k, slot, big_k, big_v)
    assert torch.equal(big_k[-1, :, page - 1].reshape(-1), k[0])
    assert torch.equal(big_v[-1, :, 0].reshape(-1), -k[1])


def test_no_rows():
    case = make([30, 5], [0, 0], 4, 2, 64, 16, BF16)
    o, lse = attend(case)
    assert o.shape == (0, 256) and lse.shape == (4, 0)


# ----------------------------------------------------------------- refusals ----


def test_refusals():
    q, kc, vc, table, lens, cu = make([40], [2], 4, 2, 64, 16, BF16)
    ln, c = _i32(lens), _i32(cu)
    ok = dict(q=q, k_cache=kc, v_cache=vc, table=table, lens=ln, cu=c)
    bad = [
        dict(q=q.float()), dict(q=q[:, :-1]), dict(q=q[:, :64 * 3]), dict(v_cache=vc[:-1]),
        dict(k_cache=kc[:, :, ::2], v_cache=vc[:, :, ::2]), dict(k_cache=kc.float()),
        dict(q=q.half(), k_cache=kc.half(), v_cache=vc.half()),
        dict(table=table.long()), dict(table=torch.cat([table, table])), dict(lens=ln.long()),
        dict(cu=c[:1]), dict(cu=c.long()), dict(lens=ln.cpu()), dict(q=q[:1].expand(2, -1)),
        dict(k_cache=kc[:, :, :8].contiguous(), v_cache=vc[:, :, :8].contiguous()),  # page 8
        dict(o=torch.empty(2, 255, dtype=BF16, device=DEV)), dict(lse=torch.empty(2, 4, device=DEV)),
        dict(algo=9), dict(algo=0x200),
    ]
    for change in bad:
        with pytest.raises(L.PeError):
            ops.attn_paged(**{**ok, **change})
    for shared in (-16, 8, 16 * (table.shape[1] + 1)):
        with pytest.raises(L.PeError):
            ops.attn_paged_shared(**ok, shared=shared)
    k = torch.zeros(2, 128, dtype=BF16, device=DEV)
    slots = torch.zeros(2, dtype=torch.int64, device=DEV)
    for args in ((k.float(), k, slots, kc, vc), (k[:1], k, slots, kc, vc), (k, k, slots[:1], kc, vc),
                 (k, k, slots.int(), kc, vc), (k[:, :64], k[:, :64], slots, kc, vc),
                 (k, k, slots, kc[:, :, ::2], vc[:, :, ::2]), (k, k.cpu(), slots, kc, vc)):
        with pytest.raises(L.PeError):
            ops.cache_append(*args)
    free, ring = _i32([0, 1]), torch.zeros(3, dtype=torch.int64, device=DEV)
    for args, kw in (((ln, ln[:0], table, free, ring, 16, 2), {}),
                     ((ln, ln, table, free, ring, 0, 2), {}), ((ln, ln, table, free, ring, 16, -1), {}),
                     ((ln, ln, table, free, ring[:2], 16, 2), {}),
                     ((ln, ln, table.float(), free, ring, 16, 2), {}),
                     ((ln, ln, table, free, ring, 16, 2), {"ring_out": ring}),
                     ((ln, ln, table, free, ring, 16, 2), {"shared": 8}),
                     ((ln[:0], ln[:0], table[:0], free, ring, 16, 2), {})):
        with pytest.raises(L.PeError):
            ops.cache_plan(*args, **kw)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_many_requests(dtype):
    """Batches whose line of work a warp, or the whole block, looks through."""
    for batch in (31, 33, 128, 129, 700):
        lens = [(37 * i) % 90 for i in range(batch)]
        news = [min(t, 1 + i % 3) if i % 11 else 0 for i, t in enumerate(lens)]
        case = make(lens, news, 4, 2, 64, 16, dtype, seed=batch)
        check(*case, 4, *attend(case))


def test_prefix_beyond_the_cache():
    """A prefix of more than 64 MB, whose pieces are cut alike for all row tiles."""
    shared = 20480
    lens, news = [shared + 9 + 30 * i for i in range(20)], [5] * 20
    case = make(lens, news, 40, 8, 128, 128, BF16, shared=shared)
    check(*case, 40, *attend(case, shared=shared))


@pytest.mark.parametrize("width", [600, 640, 656, 1024, 1040])
def test_widths_where_entities_are_cut_or_not(width):
    """The same requests under block tables of other widths (which say how long requests can
    be, and so whether blocks share one): the results agree with the definition in each."""
    lens = [min(width, 37 + 61 * i) for i in range(20)]
    for news in ([1] * 20, [5] * 20):
        q, kc, vc, table, ln, cu = make(lens, news, 28, 4, 128, 16, BF16, seed=width)
        wide = torch.full((20, -(-width // 16)), 2**31 - 1, dtype=torch.int32, device=DEV)
        n = min(wide.shape[1], table.shape[1])
        wide[:, :n] = table[:, :n]
        case = (q, kc, vc, wide, ln, cu)
        check(*case, 28, *attend(case))


def _from_threads(calls, times):
    """Each C call in a loop of its own host thread and stream, all at once (ctypes lets go of
    the interpreter's lock, so the library's host code runs in parallel)."""
    failed = []
    start = threading.Barrier(len(calls))

    def loop(fn, args):
        with torch.cuda.device(DEV):
            stream = torch.cuda.Stream()
            args = (*args, stream.cuda_stream)
            start.wait()
            for _ in range(times):
                if fn(*args):
                    failed.append(L.load().pe_last_error().decode())
                    break
            stream.synchronize()

    threads = [threading.Thread(target=loop, args=c) for c in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed


def test_plans_of_two_sizes_from_several_threads():
    """Batches whose scans need different amounts of shared memory, planned at once."""
    lib, calls, keep = L.load(), [], []
    for batch in (8000, 3000, 8000, 3000):
        zero, table, granted = (torch.zeros(batch, dtype=torch.int32, device=DEV)
                                for _ in range(3))
        free, cu = _i32([0]), torch.empty(batch + 1, dtype=torch.int32, device=DEV)
        ring, out = (torch.tensor([0, 1, 0], device=DEV) for _ in range(2))
        row = torch.empty(1, dtype=torch.int64, device=DEV)
        ts = (zero, table, granted, free, cu, ring, out, row)
        keep.append(ts)
        z, t, g, f, c, r, o, w = (x.data_ptr() for x in ts)
        calls.append((lib.pe_cache_plan, (batch, 1, 1, 16, 0, 0, z, z, t, 1, f, r, o, g, c, w, w)))
    torch.cuda.synchronize()
    _from_threads(calls, 5000)
    for zero, _, granted, *_ in keep:
        assert torch.equal(zero, granted)


def test_head_sizes_from_several_threads():
    """fp32 attention over two head sizes at once: their tiles' shared memory differs."""
    lib, calls, keep = L.load(), [], []
    for hd in (256, 64, 256, 64):
        case = make([90, 40], [2, 1], 2, 2, hd, 16, F32, seed=hd)
        q, kc, vc, table, lens, cu = case
        o, lse = torch.empty_like(q), torch.empty(2, 3, device=DEV)
        nbytes = lib.pe_attn_paged_workspace(L.F32, 2, 3, 2, 2, hd, 0)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=DEV)
        ln, c = _i32(lens), _i32(cu)
        keep.append((case, o, lse, ws, ln, c))
        calls.append((lib.pe_attn_paged, (
            L.F32, 2, 3, 2, 2, hd, q.data_ptr(), 2 * hd, kc.data_ptr(), vc.data_ptr(), kc.shape[0],
            16, table.data_ptr(), table.shape[1], table.shape[1], ln.data_ptr(), c.data_ptr(), 0,
            o.data_ptr(), 2 * hd, lse.data_ptr(), ws.data_ptr(), nbytes, 0, None)))
    torch.cuda.synchronize()
    _from_threads(calls, 5000)
    for case, o, lse, *_ in keep:
        check(*case, 2, o, lse)


def test_first_call_under_capture_leaves_the_status_word_alone(monkeypatch):
    """A device's status word that a capture creates is no part of the graph: its replays do
    not clear what a kernel recorded, and it is healthy before the first of them."""
    case = make([40, 9], [2, 1], 4, 2, 64, 16, BF16)
    q, kc, vc, table, lens, cu = case
    ln, c = _i32(lens), _i32(cu)
    ops.attn_paged(q, kc, vc, table, ln, c)
    torch.cuda.synchronize()
    monkeypatch.setattr(ops, "_status", {})
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o, lse = ops.attn_paged(q, kc, vc, table, ln, c)
    ops.check_status(DEV)
    ops.status_word(DEV).fill_(7)
    g.replay()
    with pytest.raises(L.PeError, match="fault code 7"):
        ops.check_status(DEV)
    ops.check_status(DEV)
    check(*case, 4, o, lse)


@pytest.mark.parametrize("batch", [3200, 3300, 5600])
def test_plan_scans_that_share_an_sm(batch):
    """Many rows, with scans of which an SM runs two at once, or one."""
    run_plan(*_plan_case(batch, 16, 16, 70000, seed=batch, head=5))


@pytest.mark.parametrize("batch", [1, 3, 4])
@pytest.mark.parametrize("width", [512, 528, 640, 656, 1024])
def test_widths_where_few_requests_are_cut_or_not(batch, width):
    """The same with few requests, whose tables' limit depends on the rows a tile holds."""
    lens = [min(width, 500 + 13 * i) for i in range(batch)]
    for n in (1, 4, 5, 9):  # 7 to 63 packed rows
        q, kc, vc, table, ln, cu = make(lens, [n] * batch, 28, 4, 128, 16, BF16, seed=width + n)
        wide = torch.full((batch, width // 16), 2**31 - 1, dtype=torch.int32, device=DEV)
        wide[:, :min(wide.shape[1], table.shape[1])] = table[:, :wide.shape[1]]
        case = (q, kc, vc, wide, ln, cu)
        check(*case, 28, *attend(case))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("news", [1, 2, 5, 9])
def test_shared_prefix_with_own_keys_in_pieces(news, hd):
    """Own keys that blocks cut behind a prefix read once: the join of a request's pieces adds
    the prefix's rows (7, 14, 35 and 63 packed rows: every kind of the few-row kernel)."""
    shared, own = 1024, [700, 1100, 3000, 9, 2048]
    case = make([shared + t for t in own], [news] * len(own), 28, 4, hd, 64, BF16,
                seed=news + hd, shared=shared)
    check(*case, 28, *attend(case, shared=shared))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("hd", [64, 128])
def test_shared_prefix_with_prompts_behind_it(dtype, hd):
    """The same with 40 to 300 new rows a request: whole tiles and pieces of the many-row
    kernel (and of the CUDA-core one) behind the prefix."""
    shared = 512
    own, news = [300, 45, 1500, 400], [300, 40, 130, 77]
    case = make([shared + t for t in own], news, 14, 2, hd, 16, dtype, seed=hd, shared=shared)
    check(*case, 14, *attend(case, shared=shared))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_shared_prefix_repeats_and_is_right(dtype):
    """Pieces of the prefix and of the own keys, joined in the same order every time."""
    shared = 128
    case = make([shared + 2500, shared + 31, shared + 800], [5, 3, 7], 28, 4, 128, 64, dtype,
                shared=shared)
    o, lse = attend(case, shared=shared)
    check(*case, 28, o, lse)
    for _ in range(3):
        o2, l2 = attend(case, shared=shared)
        assert torch.equal(o, o2) and torch.equal(lse, l2)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("news", [1, 5, 33, 70])
def test_many_requests_in_pieces(dtype, news):
    """More than 128 requests (the whole block looks through them) under a table whose width
    has them cut: most of them short, some over several blocks.  news 33 and 70: 66 and 140
    packed rows, the many-row kernel."""
    lens = [news + (17 * i) % 60 for i in range(150)]
    for i in (0, 70, 149):
        lens[i] = 4000 + 333 * i
    q, kc, vc, table, ln, cu = make(lens, [news] * 150, 4, 2, 64, 64, dtype, seed=news)
    assert table.shape[1] * 64 > 1024
    case = (q, kc, vc, table, ln, cu)
    check(*case, 4, *attend(case))


@pytest.mark.parametrize("shared", [0, 64])
def test_replay_beside_eager_calls(shared):
    """A captured call replayed while eager calls run on another stream, with scratch of their
    own: both are what they are alone."""
    cases = [make([shared + 3000 + 500 * i, shared + 40], [5, 3], 28, 4, 128, 64, BF16,
                  seed=20 + i, shared=shared) for i in range(2)]
    fixed = [(c[:4], _i32(c[4]), _i32(c[5])) for c in cases]

    def call(i):
        args, ln, cu = fixed[i]
        if shared:
            return ops.attn_paged_shared(*args, ln, cu, shared, algo=L.PAGED_PREFIX_ONCE)
        return ops.attn_paged(*args, ln, cu)

    want = [call(i) for i in range(2)]
    for case, (o, lse) in zip(cases, want):
        check(*case, 28, o, lse)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        replayed = [call(0) for _ in range(8)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        g.replay()
        with torch.cuda.stream(s):
            eager = [call(1) for _ in range(8)]
        torch.cuda.synchronize()
        for (o, lse), got in ((want[0], replayed), (want[1], eager)):
            for o2, l2 in got:
                assert torch.equal(o, o2) and torch.equal(lse, l2)
        for o2, _ in replayed:
            o2.fill_(7)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("shared", [0, 64])
def test_mixed_batches(dtype, shared):
    """A prompt beside single tokens, drafts and idle requests, under a table much wider than
    any of them needs; whichever kernel the mean number of rows picks."""
    for batch, prompt in ((64, 500), (12, 900)):
        lens = [30 + 7 * i for i in range(batch)]
        news = [(0, 1, 5, 0)[i % 4] for i in range(batch)]
        lens[5], news[5] = prompt + 60, prompt
        q, kc, vc, table, ln, cu = make([shared + t for t in lens], news, 28, 4, 128, 64, dtype,
                                        seed=batch, shared=shared)
        wide = torch.full((batch, 200), 2**31 - 1, dtype=torch.int32, device=DEV)
        wide[:, :table.shape[1]] = table
        case = (q, kc, vc, wide, ln, cu)
        check(*case, 28, *attend(case, shared=shared))
