"""Host-side checks of the paged cache entry points: argument validation happens before any
CUDA call, and the wrappers refuse host tensors (no GPU needed)."""

from __future__ import annotations

import pytest
import torch

from parallel_eagle_b200 import _lib, ops

BF16, F32, F16 = 1, 0, 2


def _plan(lib, B=1, width=4, pages=8, page=16, rows=3, shared=0, table_ld=4, p=1):
    p = p or None
    # distinct non-null addresses that are never dereferenced on the host
    return lib.pe_cache_plan(B, width, pages, page, rows, shared, p, p, p, table_ld, p, p,
                             p and p + 64, p and p + 128, p, p, p, None)


def test_plan_validates():
    lib = _lib.load()
    for kw in (dict(B=0), dict(B=8193), dict(page=0), dict(width=0), dict(table_ld=3),
               dict(pages=0), dict(rows=-1), dict(shared=-16), dict(shared=8), dict(shared=80),
               dict(width=1 << 28, table_ld=1 << 28), dict(p=0)):
        assert _plan(lib, **kw) == 1, kw
        assert b"cache_plan" in lib.pe_last_error()
    # outputs that alias the inputs they are computed from
    assert lib.pe_cache_plan(1, 4, 8, 16, 3, 0, 1, 1, 1, 4, 1, 1, 1, 129, 1, 1, 1, None) == 1
    assert b"alias" in lib.pe_last_error()


def _append(lib, dtype=BF16, rows=4, Hkv=2, hd=64, k_ld=128, v_ld=128, pages=4, page=16, p=16):
    p = p or None
    return lib.pe_cache_append(dtype, rows, Hkv, hd, p, k_ld, p, v_ld, p, pages, page, p, p, None)


def test_append_validates():
    lib = _lib.load()
    for kw in (dict(dtype=F16), dict(rows=-1), dict(Hkv=0), dict(hd=0), dict(k_ld=127),
               dict(v_ld=64), dict(pages=-1), dict(page=0), dict(p=0)):
        assert _append(lib, **kw) == 1, kw
        assert b"cache_append" in lib.pe_last_error()
    assert _append(lib, rows=0, p=0) == 0


def _attn(lib, dtype=BF16, B=2, T=4, Hq=4, Hkv=2, hd=64, q_ld=256, pages=8, page=16, table_ld=4,
          width=4, shared=0, o_ld=256, ws=256, nbytes=1 << 40, algo=0, p=16):
    p = p or None
    return lib.pe_attn_paged(dtype, B, T, Hq, Hkv, hd, p, q_ld, p, p, pages, page, p, table_ld,
                             width, p, p, shared, p, o_ld, p, ws, nbytes, algo, None, None)


def test_attention_validates():
    lib = _lib.load()
    for kw in (dict(dtype=F16), dict(Hq=3), dict(Hq=0), dict(Hkv=0), dict(Hq=514, Hkv=2),
               dict(hd=0), dict(hd=257), dict(B=0), dict(T=-1), dict(T=1 << 30), dict(page=8),
               dict(page=24), dict(pages=0), dict(width=0), dict(width=1 << 27, table_ld=1 << 27),
               dict(table_ld=3), dict(shared=-16), dict(shared=8), dict(shared=80), dict(q_ld=255),
               dict(o_ld=128), dict(algo=7), dict(algo=0x200), dict(p=0)):
        assert _attn(lib, **kw) == 1, kw
        assert b"attn_paged" in lib.pe_last_error()
    # a workspace that is missing, short or misaligned
    for kw in (dict(ws=None), dict(nbytes=16), dict(ws=264)):
        assert _attn(lib, **kw) == 4, kw
        assert b"workspace" in lib.pe_last_error()
    assert _attn(lib, T=0, p=0) == 0


def test_workspace_sizes():
    lib = _lib.load()
    own = lib.pe_attn_paged_workspace(BF16, 8, 40, 28, 4, 128, 0)
    assert own > 0
    # a shared prefix adds its rows' fp32 result
    assert lib.pe_attn_paged_workspace(BF16, 8, 40, 28, 4, 128, 64) >= own + 40 * 28 * 129 * 4
    assert lib.pe_attn_paged_workspace(BF16, 0, 40, 28, 4, 128, 0) == 0
    assert lib.pe_attn_paged_workspace(BF16, 8, 0, 28, 4, 128, 0) == 0


def test_wrappers_refuse_host_tensors():
    i = torch.zeros(2, dtype=torch.int32)
    table = torch.zeros(2, 3, dtype=torch.int32)
    cache = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    rows = torch.zeros(2, 128, dtype=torch.bfloat16)
    ring = torch.zeros(3, dtype=torch.int64)
    calls = [
        lambda: ops.cache_plan(i, i, table, i, ring, 16, 2),
        lambda: ops.cache_append(rows, rows, torch.zeros(2, dtype=torch.int64), cache, cache),
        lambda: ops.attn_paged(rows, cache, cache, table, i, torch.zeros(3, dtype=torch.int32)),
        lambda: ops.attn_paged_shared(rows, cache, cache, table, i,
                                      torch.zeros(3, dtype=torch.int32), 16),
    ]
    for call in calls:
        with pytest.raises(_lib.PeError, match="CUDA tensors only"):
            call()


def test_draft_cache_needs_a_gpu():
    import types

    from parallel_eagle_b200.cache import DraftCache

    d = types.SimpleNamespace(device=torch.device("cpu"), param_dtype=torch.float32)
    with pytest.raises(_lib.PeError, match="CUDA only"):
        DraftCache(d, 1, 4)
    with pytest.raises(ValueError, match="multiple of 16"):
        DraftCache(d, 1, 4, page=24)
    for max_len in (0, -5):
        with pytest.raises(ValueError, match="max_len"):
            DraftCache(d, 1, 4, max_len=max_len)


def test_sizes_whose_products_wrap_are_refused():
    """Sizes so large that a product of them passes 2^63 are refused like any other too large
    ones, before anything is launched."""
    lib = _lib.load()
    big = 1 << 62
    for kw in (dict(width=big, table_ld=big, page=16), dict(width=1 << 61, table_ld=1 << 61, B=8)):
        assert _plan(lib, **kw) == 1, kw
        assert b"cache_plan" in lib.pe_last_error()
    for kw in (dict(pages=big), dict(pages=1 << 60, page=1 << 20), dict(rows=big),
               dict(rows=1 << 57, Hkv=1)):
        assert _append(lib, **kw) == 1, kw
        assert b"cache_append" in lib.pe_last_error()
    for kw in (dict(T=big), dict(T=1 << 61, Hq=8, q_ld=512, o_ld=512),
               dict(pages=(1 << 31) - 1, Hq=1 << 14, Hkv=1 << 14, page=1 << 20, q_ld=1 << 20,
                    o_ld=1 << 20)):
        assert _attn(lib, **kw) == 1, kw
        assert b"attn_paged" in lib.pe_last_error()


def test_cuda_core_grid_is_one_wave():
    """The partial results of a call (two a block, 16 rows of head_dim + 2 floats) are those of
    the blocks that the GPU holds at once: registers allow three an SM for bf16, four for fp32
    (148 SMs)."""
    lib = _lib.load()
    for dtype, blocks, hd in ((BF16, 3, 80), (BF16, 3, 40), (F32, 4, 80)):
        per_block = 2 * 16 * (hd + 2) * 4
        most = 148 * blocks * (per_block + 64)
        assert lib.pe_attn_paged_workspace(dtype, 4, 4, 4, 2, hd, 0) <= most + 3 * 256
