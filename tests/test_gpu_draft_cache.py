"""Drafting from the key/value cache on the GPU: the logits of
``ParallelDrafter.draft_logits_cached`` against ``draft_logits`` over the whole context, for
batches of requests over several rounds -- prompts, accepted tokens, rejected ones taken
back, finished requests, a shared prompt.

Both paths run the same kernels on the same values apart from attention, whose sums run in
another order: fp32 logits within 1e-4 and bf16 logits within 2e-2 relative Frobenius, the
bounds that the draft path meets against the reference.
"""

from __future__ import annotations

import pytest
import torch

from gpu_harness import build_drafter, make_case, recipe

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("needs a CUDA device", allow_module_level=True)

from parallel_eagle_b200 import _lib as L  # noqa: E402
from parallel_eagle_b200 import decode, ops  # noqa: E402
from parallel_eagle_b200.cache import DraftCache  # noqa: E402

DEV = torch.device("cuda", 0)
# (hidden, heads, kv heads, intermediate, vocab, layers), dtype, tolerance
MODELS = [
    ((256, 4, 2, 688, 1024, 2), torch.float32, 1e-4),
    ((512, 4, 2, 768, 2048, 2), torch.bfloat16, 2e-2),   # head_dim 128
    ((448, 7, 1, 512, 1000, 1), torch.bfloat16, 2e-2),   # head_dim 64, 7 heads a group
]


def _model(i, n, batch):
    (hidden, nh, nkv, inter, vocab, layers), dtype, tol = MODELS[i]
    case = make_case(hidden, nh, nkv, inter, vocab, layers, 5, n, dtype=dtype, seed=7 + i,
                     batch=batch)
    seqs = [(ids.to(DEV), feats.to(DEV)) for ids, feats in case["seqs"]]
    return build_drafter(case).eval(), seqs, tol


def _round(model, cache, seqs, have, news, k, tol):
    """One cached draft of every request with new tokens, held against the whole context."""
    ids = torch.cat([s[0][h:h + n] for s, h, n in zip(seqs, have, news)])
    feats = torch.cat([s[1][h:h + n] for s, h, n in zip(seqs, have, news)])
    got = model.draft_logits_cached(cache, ids, feats, news, k)
    at = 0
    for b, n in enumerate(news):
        have[b] += n
        if n:
            want = model.draft_logits(seqs[b][0][:have[b]], seqs[b][1][:have[b]], k)
            assert got[at].shape == want.shape and got.dtype == want.dtype
            assert recipe.rel_fro(got[at].float().cpu(), want.float().cpu()) < tol, (b, have[b])
            at += 1
    assert at == got.shape[0] and cache.lengths == have
    assert cache.lens.tolist() == have
    ops.check_status(DEV)


def _check_pages(cache):
    """Every page is free, shared or some request's, and exactly one of them."""
    head, tail, refused = cache._ring.tolist()
    free = [cache._free[i % cache.pages].item() for i in range(head, tail)]
    own = []
    sp = cache.shared // cache.page
    for b, n in enumerate(cache.lengths):
        own += cache.table[b, sp:max(sp, -(-n // cache.page))].tolist()
    own += cache.table[0, :sp].tolist()
    assert sorted(free + own) == list(range(cache.pages))
    assert refused == 0 and cache.free_pages == len(free)


@pytest.mark.parametrize("i", range(len(MODELS)))
@pytest.mark.parametrize("page", [16, 64])
def test_rounds_of_a_batch(i, page):
    model, seqs, tol = _model(i, 150, 4)
    cache = DraftCache(model, 4, pages=4 * (-(-160 // page)) + 3, page=page, max_len=160)
    have = [0] * 4
    _round(model, cache, seqs, have, [70, 1, 33, 16], 5, tol)   # prompts
    _check_pages(cache)
    _round(model, cache, seqs, have, [3, 5, 1, 2], 5, tol)      # accepted tokens
    _round(model, cache, seqs, have, [1, 0, 4, 0], 3, tol)      # some requests wait
    cache.truncate(2, 20)                                       # tokens taken back
    have[2] = 20
    cache.finish(0)                                             # a finished request ...
    have[0] = 0
    _check_pages(cache)
    seqs[0] = seqs[3]                                           # ... and a new one
    _round(model, cache, seqs, have, [90, 2, 7, 1], 5, tol)
    _round(model, cache, seqs, have, [1, 1, 1, 1], 1, tol)      # next tokens only
    _check_pages(cache)
    for b in range(4):
        cache.finish(b)
    assert cache.free_pages == cache.pages
    _check_pages(cache)


@pytest.mark.parametrize("i", range(len(MODELS)))
def test_shared_prompt(i):
    """Requests forked from one prompt: its whole pages are computed and read once."""
    model, seqs, tol = _model(i, 140, 3)
    prompt = 75
    for b in (1, 2):
        seqs[b] = tuple(torch.cat([seqs[0][j][:prompt], seqs[b][j][prompt:]]) for j in (0, 1))
    cache = DraftCache(model, 3, pages=40, page=16, max_len=160)
    n = cache.set_prefix(model, seqs[0][0][:prompt], seqs[0][1][:prompt])
    assert n == 64 and cache.shared == 64 and cache.free_pages == 40 - 4
    have = [n] * 3
    _round(model, cache, seqs, have, [prompt - n] * 3, 5, tol)
    _round(model, cache, seqs, have, [2, 5, 1], 5, tol)
    cache.finish(1)
    have[1] = n
    _check_pages(cache)
    _round(model, cache, seqs, have, [1, 40, 3], 4, tol)
    _check_pages(cache)
    with pytest.raises(ValueError):
        cache.set_prefix(model, *seqs[0])
    with pytest.raises(ValueError):
        cache.truncate(0, 10)


def test_proposals_match_the_uncached_ones():
    model, seqs, _ = _model(0, 120, 3)
    cache = DraftCache(model, 3, pages=60, page=16)
    have, news = [0, 0, 0], [60, 45, 100]
    trees = [decode.propose_trees, decode.propose_tree]
    ids = torch.cat([s[0][:n] for s, n in zip(seqs, news)])
    feats = torch.cat([s[1][:n] for s, n in zip(seqs, news)])
    got = trees[0](model, cache, ids, feats, news, 4, 3, 12)
    for b, n in enumerate(news):
        assert tuple(got[b]) == tuple(trees[1](model, seqs[b][0][:n], seqs[b][1][:n], 4, 3, 12))
        have[b] = n
    news = [4, 0, 2]
    ids = torch.cat([s[0][h:h + n] for s, h, n in zip(seqs, have, news)])
    feats = torch.cat([s[1][h:h + n] for s, h, n in zip(seqs, have, news)])
    got = decode.propose_chains(model, cache, ids, feats, news, 5)
    want = [decode.propose_chain(model, seqs[b][0][:h + n], seqs[b][1][:h + n], 5)
            for b, (h, n) in enumerate(zip(have, news)) if n]
    assert got == want


def test_refusals_leave_the_cache_as_it_was():
    model, seqs, tol = _model(1, 150, 2)
    cache = DraftCache(model, 2, pages=6, page=16, max_len=80)
    have = [0, 0]
    _round(model, cache, seqs, have, [30, 20], 4, tol)
    ids, feats = seqs[0]
    with pytest.raises(L.PeError, match="free pages"):
        model.draft_logits_cached(cache, ids[:60], feats[:60], [40, 20], 4)
    with pytest.raises(L.PeError, match="length"):
        model.draft_logits_cached(cache, ids[:60], feats[:60], [60, 0], 4)
    for news, k in (([1], 4), ([1, 1, 1], 4), ([2, 1], 4), ([-1, 3], 4), ([1, 1], 0)):
        with pytest.raises(ValueError):
            model.draft_logits_cached(cache, ids[:2], feats[:2], news, k)
    with pytest.raises(ValueError):
        model.draft_logits_cached(cache, ids[:0], feats[:0], [0, 0], 4)
    with pytest.raises(ValueError):
        decode.propose_chains(model, cache, ids[:2], feats[:2], [1, 1], 0)
    for args in ((0, 4, 16), (1, 0, 16), (1, 4, 8), (1, 4, 24)):
        with pytest.raises(ValueError):
            DraftCache(model, *args)
    assert cache.lengths == have
    _check_pages(cache)
    _round(model, cache, seqs, have, [1, 2], 4, tol)


def test_cache_moves_to_another_stream(monkeypatch):
    """Lengths and ring that a resize replaces are not given to the stream they came from while
    the stream that plans still reads them."""
    model, _, _ = _model(0, 20, 1)
    cache = DraftCache(model, 2, pages=8, page=16)
    plan = ops.cache_plan

    def late_plan(*args, **kw):
        torch.cuda._sleep(100_000_000)
        return plan(*args, **kw)

    monkeypatch.setattr(ops, "cache_plan", late_plan)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        cu, slots, pos = cache.resize([20, 5])
    junk = [torch.full((6,), 77, dtype=torch.int32, device=DEV) for _ in range(200)]
    torch.cuda.synchronize()
    assert cache.lens.tolist() == [20, 5] and cu.tolist() == [0, 20, 25]
    assert pos.tolist() == [*range(20), *range(5)] and slots.min() >= 0
    _check_pages(cache)
    assert all((j == 77).all() for j in junk)


def test_prefixes_one_after_another():
    """A prefix is given back when its requests are finished, and the next one takes its pages."""
    model, seqs, tol = _model(1, 140, 3)
    cache = DraftCache(model, 3, pages=14, page=16, max_len=112)
    free = cache.free_pages
    cache.drop_prefix()  # there is none
    for prompt, own in ((75, 9), (33, 30), (90, 2)):
        for b in range(3):
            seqs[b] = tuple(torch.cat([seqs[-1][j][:prompt], seqs[b][j][prompt:]]) for j in (0, 1))
        n = cache.set_prefix(model, seqs[0][0][:prompt], seqs[0][1][:prompt])
        assert n == prompt // 16 * 16 and cache.free_pages == free - n // 16
        have = [n] * 3
        _round(model, cache, seqs, have, [prompt - n + own, 0, prompt - n + 1], 5, tol)
        _check_pages(cache)
        with pytest.raises(ValueError, match="finished"):
            cache.drop_prefix()
        for b in range(3):
            cache.finish(b)
        _check_pages(cache)
        cache.drop_prefix()
        assert cache.shared == 0 and cache.lengths == [0] * 3 and cache.free_pages == free
        assert cache.lens.tolist() == [0] * 3
        _check_pages(cache)
    have = [0] * 3
    _round(model, cache, seqs, have, [40, 7, 20], 4, tol)  # and without one
    cache.drop_prefix()  # there is none
    assert cache.lengths == [40, 7, 20]
    _check_pages(cache)


def test_proposals_report_a_kernel_that_gave_up():
    """What a bounded wait records reaches the caller with the drafts of that call, once."""
    model, seqs, _ = _model(1, 60, 2)
    cache = DraftCache(model, 2, pages=20, page=16)
    ids, feats = (torch.cat([s[j][:9] for s in seqs]) for j in (0, 1))
    calls = [lambda: decode.propose_trees(model, cache, ids, feats, [9, 9], 4, 2, 8),
             lambda: decode.propose_chains(model, cache, ids, feats, [9, 9], 4)]
    for call in calls:
        want = call()
        cache.truncate(0, 0)
        cache.truncate(1, 0)
        ops.status_word(DEV).fill_(403)
        with pytest.raises(L.PeError, match="fault code 403"):
            call()
        cache.truncate(0, 0)
        cache.truncate(1, 0)
        assert call() == want
        cache.truncate(0, 0)
        cache.truncate(1, 0)
