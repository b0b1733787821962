"""The long-context paged-cache entry points on the CPU: sizes, and every
argument error reported before anything is launched."""
import ctypes

import pytest

from hero_amd import _lib
from hero_amd._lib import AttnDecodeArgs, AttnPagedArgs, AttnSparseArgs, KvReadArgs

lib = _lib.lib
P = 4096  # a fake, well aligned device pointer: never followed, the calls below are all refused


def sparse_args(**change):
    """arguments that would pass every check, with some fields changed"""
    f = dict(proj=P, proj_stride=2 * 8 * 128 + 2 * 2 * 128, k_off=2048, v_off=2304, q_gamma=P, k_gamma=P, eps=1e-6, rope_cs=P, positions=P, q_rot=P,
             score_scale=0.1, window=0, act_out=P, out_f32=P, b=3, hq=8, hkv=2, dh=128, pages=P, page_table=P, page_size=64, max_pages=10, work=P,
             work_bytes=1 << 30, q8=0, pool_pages=30, rope_positions=640, row_seq=None, seqs=3, summaries=P, selected=P, top=8, sink=1, recent=2)
    assert set(change) <= set(f)
    f.update(change)
    a = AttnDecodeArgs(f["proj"], f["proj_stride"], f["k_off"], f["v_off"], f["q_gamma"], f["k_gamma"], f["eps"], f["rope_cs"], None, None, 0, f["positions"],
                       None, f["q_rot"], f["score_scale"], f["window"], f["act_out"], f["out_f32"], f["b"], f["hq"], f["hkv"], f["dh"])
    p = AttnPagedArgs(a, f["pages"], f["page_table"], f["page_size"], f["max_pages"], f["work"], f["work_bytes"], f["q8"])
    return AttnSparseArgs(p, f["pool_pages"], f["rope_positions"], f["row_seq"], f["seqs"], f["summaries"], f["selected"], f["top"], f["sink"], f["recent"])


ROWS = [  # refused by all three calls over rows
    (dict(dh=64), b"128"), (dict(dh=256, q8=1, proj_stride=1 << 20), b"256"), (dict(q8=2), b"q8"), (dict(page_size=24), b"page_size"),
    (dict(page_size=8), b"page_size"), (dict(page_size=512), b"page_size"), (dict(max_pages=0), b"geometry"), (dict(max_pages=(1 << 18) + 1), b"geometry"),
    (dict(pool_pages=0), b"pool_pages"), (dict(b=0), b"count"), (dict(b=4), b"row_seq"), (dict(seqs=0), b"count"), (dict(positions=None), b"null"),
    (dict(page_table=None), b"null"), (dict(positions=P + 2), b"aligned"), (dict(row_seq=P + 1), b"aligned"), (dict(hq=7), b"query heads"),
    (dict(hq=18, proj_stride=1 << 20), b"query heads"), (dict(window=5), b"window"), (dict(q_rot=None), b"q_rot"), (dict(q_rot=P + 4), b"q_rot"),
    (dict(b=1 << 21, seqs=1 << 21), b"rows"),
]
APPEND = [
    (dict(proj=None), b"null"), (dict(k_gamma=None), b"null"), (dict(rope_cs=None), b"null"), (dict(pages=None), b"null"), (dict(summaries=None), b"null"),
    (dict(pages=P + 2), b"aligned"), (dict(summaries=P + 8), b"aligned"), (dict(rope_positions=0), b"rope_positions"), (dict(k_off=-1), b"slices"),
    (dict(v_off=2305), b"slices"), (dict(proj_stride=2047, k_off=0, v_off=0), b"slices"), (dict(proj=P + 2), b"aligned"),
]
SELECT = [
    (dict(top=0), b"top"), (dict(top=4097), b"top"), (dict(selected=None), b"selected"), (dict(recent=0), b"recent"), (dict(sink=-1), b"sink"),
    (dict(sink=7), b"sink"), (dict(sink=0x7fffffff, recent=0x7fffffff), b"sink"), (dict(summaries=None), b"summaries"), (dict(work=None), b"work"), (dict(work_bytes=3 * 2 * 10 * 8 - 1), b"work_bytes"),
]
ATTEND = [
    (dict(top=0), b"top"), (dict(selected=None), b"selected"), (dict(proj=None), b"proj"), (dict(pages=None), b"pages"), (dict(pages=P + 8), b"pages"),
    (dict(proj_stride=2047), b"gates"), (dict(out_f32=None, act_out=None), b"no output"), (dict(out_f32=P + 4), b"aligned"), (dict(act_out=P + 1), b"aligned"),
]


@pytest.mark.parametrize("call,change,needle", [(c, *x) for c, more in (("hero_kv_append_paged", APPEND), ("hero_attn_select_pages", SELECT), ("hero_attn_sparse_paged", ATTEND))
                                                for x in ROWS + more])
def test_calls_over_rows_refuse_bad_arguments(call, change, needle):
    assert getattr(lib, call)(ctypes.byref(sparse_args(**change)), None) == _lib.HERO_EINVAL
    assert needle in lib.hero_last_error()


@pytest.mark.parametrize("call", ["hero_kv_append_paged", "hero_attn_select_pages", "hero_attn_sparse_paged", "hero_kv_read_paged"])
def test_null_args_are_refused(call):
    assert getattr(lib, call)(None, None) == _lib.HERO_EINVAL
    assert b"null args" in lib.hero_last_error()


@pytest.mark.parametrize("change,needle", [
    (dict(f16=2), b"f16"), (dict(k_out=None, v_out=None, k_max=None, k_min=None), b"no output"), (dict(pages=None), b"pages"), (dict(summaries=None), b"summaries"),
    (dict(k_min=P + 8), b"outputs"), (dict(rows=0), b"count"), (dict(rows=4), b"row_seq"), (dict(hkv=0), b"count"), (dict(dh=256, q8=1), b"256"), (dict(pages=P + 4), b"aligned"),
])
def test_read_refuses_bad_arguments(change, needle):
    f = dict(pages=P, page_table=P, page_size=64, max_pages=10, q8=0, pool_pages=30, summaries=P, positions=P, row_seq=None, rows=3, seqs=3, hkv=2, dh=128, f16=0,
             k_out=P, v_out=P, k_max=P, k_min=P)
    f.update(change)
    assert lib.hero_kv_read_paged(ctypes.byref(KvReadArgs(**f)), None) == _lib.HERO_EINVAL
    assert needle in lib.hero_last_error()


def test_size_helpers():
    assert lib.hero_kv_summary_bytes(10, 8, 128) == 10 * (8 * 256 + 32)
    assert lib.hero_kv_summary_bytes(1, 3, 256) == 3 * 512 + 16
    for bad in ((0, 8, 128), (1, 0, 128), (1, 8, 64)):
        assert lib.hero_kv_summary_bytes(*bad) == -1
    assert lib.hero_attn_select_work_bytes(3, 2, 10) >= 3 * 2 * 10 * 8
    for bad in ((0, 2, 10), (3, 0, 10), (3, 2, 0), (1 << 23, 2, 10)):
        assert lib.hero_attn_select_work_bytes(*bad) == -1
    assert lib.hero_attn_sparse_work_bytes(3, 8, 2, 128, 64, 8) >= 0
    for bad in ((0, 8, 2, 128, 64, 8), (3, 7, 2, 128, 64, 8), (3, 18, 2, 128, 64, 8), (3, 8, 2, 64, 64, 8), (3, 8, 2, 128, 24, 8), (3, 8, 2, 128, 64, 0)):
        assert lib.hero_attn_sparse_work_bytes(*bad) == -1


@pytest.mark.parametrize("hq,hkv,dh,ps,top", [(32, 8, 128, 64, 32), (8, 8, 128, 16, 5), (16, 2, 128, 256, 1), (16, 4, 256, 64, 4096), (8, 1, 128, 16, 2049)])
def test_workspaces_grow_with_the_rows(hq, hkv, dh, ps, top):
    """one workspace for the largest call serves every smaller one"""
    sizes = [lib.hero_attn_sparse_work_bytes(r, hq, hkv, dh, ps, top) for r in list(range(1, 300)) + [1000, 60000]]
    assert sizes == sorted(sizes) and sizes[0] >= 0
    sizes = [lib.hero_attn_select_work_bytes(r, hkv, 700) for r in range(1, 300)]
    assert sizes == sorted(sizes)


@pytest.mark.parametrize("change", [dict(b=3), dict(b=1, top=40), dict(b=70, seqs=70, hq=16, hkv=8, proj_stride=1 << 15, top=2049), dict(dh=256, hq=4, proj_stride=1 << 15)])
def test_attention_refuses_a_workspace_that_is_missing_or_small(change):
    a = sparse_args(**change)
    need = lib.hero_attn_sparse_work_bytes(a.p.a.b, a.p.a.hq, a.p.a.hkv, a.p.a.dh, a.p.page_size, a.top)
    assert need > 0
    for work in (dict(work=None), dict(work=P + 8), dict(work_bytes=need - 1), dict(work_bytes=0), dict(work_bytes=-1)):
        assert lib.hero_attn_sparse_paged(ctypes.byref(sparse_args(**change, **work)), None) == _lib.HERO_EINVAL
        assert b"work" in lib.hero_last_error()


def test_selection_refuses_a_misaligned_workspace():
    assert lib.hero_attn_select_pages(ctypes.byref(sparse_args(work=P + 8)), None) == _lib.HERO_EINVAL
    assert b"work" in lib.hero_last_error()
