"""The paged cache's host side on the CPU: handing pages out and back, the
page look-up the kernels share, and the refusals of the C entry points."""
import ctypes

import pytest
import torch


@pytest.fixture()
def cache(rb):
    """Host side and table of a cache of 6 pages of 16, three sequences."""
    from riallm_b200.paged import PagedKVCache
    c = object.__new__(PagedKVCache)
    c.page_size, c.num_pages, c.max_pages = 16, 6, 4
    c.table = torch.full((3, 4), -1, dtype=torch.int32)
    c._init_host(3)
    return c


def test_reserve_and_release(rb, cache):
    cache.reserve([17, 0, 16])
    assert cache.free_pages == 3
    held = cache.table[cache.table >= 0].tolist()
    assert len(held) == len(set(held)) == 3 and all(0 <= p < 6 for p in held)
    assert (cache.table >= 0).sum(1).tolist() == [2, 0, 1]
    before = cache.table.clone()
    cache.reserve([32, 0, 3])  # nothing new
    assert torch.equal(cache.table, before)
    with pytest.raises(rb.MemoryError_, match="4 pages wanted, 3 free"):
        cache.reserve([64, 32])
    assert torch.equal(cache.table, before) and cache.free_pages == 3
    with pytest.raises(rb.ConfigError, match="at most 4"):
        cache.reserve([65])
    with pytest.raises(rb.ConfigError, match="sequences"):
        cache.reserve([1, 1, 1, 1])
    cache.release(0)
    assert cache.free_pages == 5 and (cache.table[0] == -1).all()
    cache.release()
    assert cache.free_pages == 6 and (cache.table == -1).all()


def test_window_gives_pages_back_once(rb, cache):
    cache.reserve([64])
    cache.release_before([47], sinks=3)  # positions 3..46: page 1 alone lies in them wholly
    assert (cache.table[0] >= 0).tolist() == [True, False, True, True]
    assert cache.free_pages == 3
    cache.release_before([47], sinks=3)
    cache.reserve([64])  # what was given back stays away
    assert (cache.table[0] >= 0).tolist() == [True, False, True, True]
    cache.release_before([1000])  # no further than the pages held
    assert cache.free_pages == 5 and cache.table[0, 0] >= 0
    cache.release(0)
    assert cache.free_pages == 6 and sorted(cache._free) == list(range(6))
    cache.reserve([33])
    assert (cache.table[0] >= 0).tolist() == [True, True, True, False]


def test_page_lookup_bounds(rb):
    L = rb.lib()
    table = (ctypes.c_int32 * 8)(3, -1, 5, 99, 6, 0, -7, 2**31 - 1)  # num_pages 7; row stride 4, 3 pages used

    def row(b, kh, j, max_pages=3):
        return L.riallm_paged_row(table, 4, max_pages, 7, 2, 32, b, kh, j)
    assert row(0, 0, 0) == (3 * 2 + 0) * 32
    assert row(0, 1, 31) == (3 * 2 + 1) * 32 + 31
    assert row(0, 0, 32) == -1 and row(0, 0, 63) == -1      # entry -1
    assert row(0, 1, 64) == (5 * 2 + 1) * 32
    assert row(0, 0, 96) == -1                              # past max_pages: entry 3 is not read
    assert row(0, 0, 96, 4) == -1                           # entry 99 of 7 pages
    assert row(1, 1, 5) == (6 * 2 + 1) * 32 + 5
    assert row(1, 0, 64) == -1 and row(1, 0, 96, 4) == -1   # -7, 2^31 - 1
    assert row(0, 0, -1) == -1 and row(0, 0, 2**40) == -1 and row(0, 0, -2**40) == -1


def test_argument_structures_match_the_header(rb, tmp_path):
    """The packed layouts have the C structures' sizes and last offsets."""
    import subprocess
    from conftest import ROOT
    from riallm_b200.paged import _APPEND, _ATTEND
    from riallm_b200.sampling import _VERIFY
    src = tmp_path / "s.c"
    src.write_text('#include "riallm_cuda.h"\n#include <stdio.h>\nint main(void){printf("%zu %zu %zu %zu %zu %zu",'
                   "sizeof(riallm_rope_paged_append_args),offsetof(riallm_rope_paged_append_args,d),"
                   "sizeof(riallm_paged_attention_args),offsetof(riallm_paged_attention_args,sinks),"
                   "sizeof(riallm_verify_draft_args),offsetof(riallm_verify_draft_args,V));return 0;}")
    subprocess.run(["gcc", "-I", ROOT + "/include", str(src), "-o", str(tmp_path / "s")], check=True)
    got = list(map(int, subprocess.run([str(tmp_path / "s")], check=True, capture_output=True, text=True).stdout.split()))
    want = [v for s in (_APPEND, _ATTEND, _VERIFY) for v in (s.size, s.size - 4)]
    assert got == want


CONFIG, INVALID = 3, 7


def _append(L, B=1, T=1, nh=8, nkv=2, d=128, num_pages=4, ps=16, max_pages=2, stride=2):
    from riallm_b200.paged import _APPEND
    args = _APPEND.pack(0, 0, 0, 0, 0, 0, 0, stride, max_pages, num_pages, ps, B, T, nh, nkv, d)
    return L.riallm_cuda_rope_paged_append(None, args, None)


def _attend(L, B=1, T=1, nh=8, nkv=2, d=128, num_pages=4, ps=16, max_pages=2, stride=2, window=0, sinks=0):
    from riallm_b200.paged import _ATTEND
    args = _ATTEND.pack(0, 0, 0, 0, 0, 0, stride, max_pages, num_pages, ps, B, T, nh, nkv, d, window, sinks)
    return L.riallm_cuda_paged_attention(None, args, None, 0, None)


@pytest.mark.parametrize("call", [_append, _attend])
@pytest.mark.parametrize("bad", [dict(B=-1), dict(T=-1), dict(nh=0), dict(nh=7), dict(nh=258, nkv=2), dict(d=96),
                                 dict(d=0), dict(ps=8), dict(ps=48), dict(ps=256), dict(num_pages=0),
                                 dict(max_pages=0), dict(stride=1), dict(num_pages=2**26, nkv=2, nh=2),
                                 dict(max_pages=2**28, stride=2**28), dict(B=2**20, T=2**20),
                                 dict(nh=65536, nkv=65536, num_pages=1)])
def test_entry_points_refuse_bad_shapes(rb, call, bad):
    assert call(rb.lib(), **bad) == CONFIG


@pytest.mark.parametrize("call", [_append, _attend])
def test_positions_end_a_block_below_32_bits(rb, call):
    """The last position's block of 128 keys, and the page after it, are
    counted in int32; 2^31 - 257 positions leave room for both."""
    for ps in (16, 128):
        most = (2**31 - 257) // ps
        assert call(rb.lib(), ps=ps, max_pages=most, stride=most) == INVALID  # past the checks of sizes: NULL
        assert call(rb.lib(), ps=ps, max_pages=most + 1, stride=most + 1) == CONFIG


def test_entry_points_refuse_null(rb):
    L = rb.lib()
    assert _append(L) == INVALID and _attend(L) == INVALID
    assert L.riallm_cuda_rope_paged_append(None, None, None) == INVALID
    assert L.riallm_cuda_paged_attention(None, None, None, 0, None) == INVALID
    assert L.riallm_cuda_verify_draft(None, None, None, 0, None) == INVALID
    assert _attend(L, window=-1) == CONFIG and _attend(L, sinks=-1) == CONFIG


def _verify(L, dtype=0, B=1, n=2, V=10):
    from riallm_b200.sampling import _VERIFY
    return L.riallm_cuda_verify_draft(None, _VERIFY.pack(0, 0, 0, 0, 0, 0, 0, 0, dtype, B, n, V), None, 0, None)


def test_verify_refusals(rb):
    L = rb.lib()
    assert _verify(L) == INVALID
    for bad in (dict(dtype=2), dict(dtype=-1), dict(B=-1), dict(n=-1), dict(n=256), dict(V=0)):
        assert _verify(L, **bad) == CONFIG


def test_python_refusals(rb):
    from riallm_b200 import paged, sampling
    x = torch.zeros(2, 8 * 128, dtype=torch.bfloat16)
    pages = torch.zeros(4, 2, 16, 128, dtype=torch.bfloat16)
    pos, table = torch.zeros(1, dtype=torch.int32), torch.zeros(1, 2, dtype=torch.int32)
    with pytest.raises(rb.ConfigError, match="CUDA"):
        paged.paged_attention(x, pos, table, pages, pages)
    with pytest.raises(rb.ConfigError, match="CUDA"):
        paged.rope_paged_append(x, pos, table, pages, pages, torch.zeros(64))
    with pytest.raises(rb.ConfigError, match="CUDA"):
        sampling.verify_draft(torch.zeros(1, 3, 10), None, None, torch.zeros(1))
    for bad in (dict(page_size=8), dict(head_dim=96), dict(layers=0), dict(num_pages=0), dict(max_batch=0)):
        args = dict(layers=1, kv_heads=2, head_dim=128, num_pages=4, page_size=16, max_batch=1)
        args.update(bad)
        with pytest.raises(rb.ConfigError):
            paged.PagedKVCache(**args)


def test_lookup_drafts():
    from riallm_b200.sampling import lookup_drafts
    assert lookup_drafts([1, 2, 3, 4, 1, 2], 3) == [3, 4, 1]
    assert lookup_drafts([1, 2, 9, 1, 2, 3, 1, 2], 2) == [3, 1]   # the latest earlier place
    assert lookup_drafts([5, 6, 7, 6], 2) == [7, 6]               # one token where two are not found
    assert lookup_drafts([1, 2, 3], 4) == [] and lookup_drafts([1], 4) == [] and lookup_drafts([], 4) == []
    assert lookup_drafts([3, 3], 4) == [3]
    assert lookup_drafts([1, 2, 1, 2], 0) == []
