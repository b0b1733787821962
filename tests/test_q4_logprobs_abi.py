"""The 4-bit cache and the log probability entry points on the CPU: sizes, and every
argument error reported before anything is launched."""
import ctypes

import pytest

from hero_amd import _lib
from hero_amd._lib import AttnDecodeArgs, AttnQ4Args, KvReadArgs

lib = _lib.lib
P = 4096  # a fake, well aligned device pointer: never followed, the calls below are all refused


def q4_args(**change):
    """arguments that would pass every check, with some fields changed"""
    f = dict(proj=P, proj_stride=2 * 8 * 128 + 2 * 2 * 128, k_off=2048, v_off=2304, q_gamma=P, k_gamma=P, eps=1e-6, rope_cs=P, positions=P, q_rot=P,
             score_scale=0.1, window=0, act_out=P, out_f32=P, b=3, hq=8, hkv=2, dh=128, pages=P, pool_pages=30, page_table=P, page_size=64, max_pages=10,
             row_seq=None, seqs=3, sinks=0, rope_positions=640, rope_pos=None, rope_axes=1, plane_axis=(), work=P, work_bytes=1 << 40)
    assert set(change) <= set(f)
    f.update(change)
    a = AttnDecodeArgs(f["proj"], f["proj_stride"], f["k_off"], f["v_off"], f["q_gamma"], f["k_gamma"], f["eps"], f["rope_cs"], None, None, 0, f["positions"],
                       None, f["q_rot"], f["score_scale"], f["window"], f["act_out"], f["out_f32"], f["b"], f["hq"], f["hkv"], f["dh"])
    return AttnQ4Args(a, f["pages"], f["pool_pages"], f["page_table"], f["page_size"], f["max_pages"], f["row_seq"], f["seqs"], f["sinks"], f["rope_positions"],
                      f["rope_pos"], f["rope_axes"], (ctypes.c_uint8 * 128)(*f["plane_axis"]), f["work"], f["work_bytes"])


ROWS = [  # refused by both calls over rows
    (dict(dh=64), b"128"), (dict(page_size=24), b"page_size"), (dict(page_size=8), b"page_size"), (dict(page_size=512), b"page_size"), (dict(max_pages=0), b"geometry"),
    (dict(max_pages=(1 << 18) + 1), b"geometry"), (dict(pool_pages=0), b"pool_pages"), (dict(b=0), b"count"), (dict(b=4), b"row_seq"), (dict(seqs=0), b"count"),
    (dict(positions=None), b"null"), (dict(page_table=None), b"null"), (dict(positions=P + 2), b"aligned"), (dict(row_seq=P + 1), b"aligned"), (dict(hq=7), b"query heads"),
    (dict(hq=18, proj_stride=1 << 20), b"query heads"), (dict(hkv=0), b"count"), (dict(q_rot=None), b"q_rot"), (dict(q_rot=P + 4), b"q_rot"),
    (dict(b=1 << 21, seqs=1 << 21), b"rows"), (dict(pages=None), b"pages"), (dict(pages=P + 8), b"pages"), (dict(proj=None), b"proj"), (dict(proj=P + 2), b"proj"),
]
APPEND = [
    (dict(k_gamma=None), b"null"), (dict(q_gamma=None), b"null"), (dict(rope_cs=None), b"null"), (dict(rope_cs=P + 4), b"misaligned"), (dict(rope_pos=P + 2), b"misaligned"),
    (dict(rope_positions=0), b"rope_positions"), (dict(k_off=-1), b"slices"), (dict(v_off=2305), b"slices"), (dict(k_off=(1 << 63) - 1), b"slices"),
    (dict(proj_stride=2047, k_off=0, v_off=0), b"slices"), (dict(rope_axes=0), b"rope_axes"), (dict(rope_axes=5, rope_pos=P), b"rope_axes"), (dict(rope_axes=3), b"rope_pos"),
    (dict(plane_axis=[0] * 63 + [1]), b"plane_axis"), (dict(rope_axes=3, rope_pos=P, plane_axis=[0, 1, 2, 3]), b"plane_axis"),
]
ATTEND = [
    (dict(proj_stride=2047), b"gates"), (dict(window=-1), b"window"), (dict(sinks=-1, window=5), b"sinks"), (dict(sinks=4), b"sinks"), (dict(out_f32=None, act_out=None), b"no output"),
    (dict(out_f32=P + 4), b"aligned"), (dict(act_out=P + 8), b"aligned"),
]


@pytest.mark.parametrize("call,change,needle", [(c, *x) for c, more in (("hero_kv_append_q4", APPEND), ("hero_attn_q4", ATTEND)) for x in ROWS + more])
def test_calls_over_rows_refuse_bad_arguments(call, change, needle):
    assert getattr(lib, call)(ctypes.byref(q4_args(**change)), None) == _lib.HERO_EINVAL
    assert needle in lib.hero_last_error()


@pytest.mark.parametrize("call", ["hero_kv_append_q4", "hero_attn_q4", "hero_kv_read_q4"])
def test_null_args_are_refused(call):
    assert getattr(lib, call)(None, None) == _lib.HERO_EINVAL
    assert b"null args" in lib.hero_last_error()


@pytest.mark.parametrize("change,needle", [
    (dict(f16=2), b"f16"), (dict(k_out=None, v_out=None), b"no output"), (dict(pages=None), b"pages"), (dict(pages=P + 4), b"pages"), (dict(k_max=P), b"k_max"), (dict(k_min=P), b"k_min"),
    (dict(v_out=P + 8), b"outputs"), (dict(rows=0), b"count"), (dict(rows=4), b"row_seq"), (dict(hkv=0), b"count"), (dict(dh=192), b"128"), (dict(page_size=40), b"page_size"),
])
def test_read_refuses_bad_arguments(change, needle):
    f = dict(pages=P, page_table=P, page_size=64, max_pages=10, q8=0, pool_pages=30, summaries=None, positions=P, row_seq=None, rows=3, seqs=3, hkv=2, dh=128, f16=0,
             k_out=P, v_out=P, k_max=None, k_min=None)
    f.update(change)
    assert lib.hero_kv_read_q4(ctypes.byref(KvReadArgs(**f)), None) == _lib.HERO_EINVAL
    assert needle in lib.hero_last_error()


def test_page_sizes():
    assert lib.hero_attn_q4_page_bytes(8, 128, 64) == 2 * 8 * 64 * 72
    assert lib.hero_attn_q4_page_bytes(3, 256, 16) == 2 * 3 * 16 * 144
    for bad in ((0, 128, 64), (8, 64, 64), (8, 128, 24), (8, 128, 8), (8, 128, 512)):
        assert lib.hero_attn_q4_page_bytes(*bad) == -1


@pytest.mark.parametrize("hq,hkv,dh,ctx,window,sinks", [(32, 8, 128, 32768, 0, 0), (16, 4, 256, 262144, 0, 0), (8, 8, 128, 4096, 1024, 4), (8, 1, 128, 1 << 24, 0, 0), (3, 3, 256, 64, 0, 0)])
def test_attention_workspaces_grow_with_the_rows(hq, hkv, dh, ctx, window, sinks):
    """one workspace for the largest call serves every smaller one"""
    sizes = [lib.hero_attn_q4_work_bytes(r, hq, hkv, dh, ctx, window, sinks) for r in list(range(1, 300)) + [1000, 60000]]
    assert sizes == sorted(sizes) and sizes[0] >= 0


def test_attention_workspace_refuses_shapes():
    good = (3, 8, 2, 128, 640, 0, 0)
    assert lib.hero_attn_q4_work_bytes(*good) >= 0
    for i, bad in ((0, 0), (0, 1 << 21), (1, 7), (1, 18), (2, 0), (3, 64), (4, 0), (4, (1 << 24) + 1), (5, -1), (6, -1)):
        assert lib.hero_attn_q4_work_bytes(*good[:i], bad, *good[i + 1:]) == -1


@pytest.mark.parametrize("change", [dict(max_pages=1000), dict(b=1, max_pages=4000), dict(row_seq=P, b=70, max_pages=1000), dict(window=5000, sinks=3, max_pages=1000)])
def test_attention_refuses_a_workspace_that_is_missing_or_small(change):
    a = q4_args(**change)
    need = lib.hero_attn_q4_work_bytes(a.a.b, a.a.hq, a.a.hkv, a.a.dh, a.page_size * a.max_pages, a.a.window, a.sinks)
    assert need > 0
    for work in (dict(work=None), dict(work=P + 8), dict(work_bytes=need - 1), dict(work_bytes=0), dict(work_bytes=-1)):
        assert lib.hero_attn_q4(ctypes.byref(q4_args(**change, **work)), None) == _lib.HERO_EINVAL
        assert b"work" in lib.hero_last_error()


# ---- log probabilities
def logprobs(**change):
    f = dict(logits=P, stride=1000, m=3, v=1000, targets=P, temp=1.0, top_n=5, logprob=P, entropy=P, top_ids=P, top_logprobs=P, work=P, work_bytes=1 << 40)
    assert set(change) <= set(f)
    f.update(change)
    return lib.hero_logprobs(*f.values(), None)


@pytest.mark.parametrize("change,needle", [
    (dict(m=0), b"m and v"), (dict(v=0), b"m and v"), (dict(m=(1 << 24) + 1), b"m and v"), (dict(top_n=-1), b"top_n"), (dict(top_n=65), b"top_n"), (dict(v=4, stride=4), b"top_n"),
    (dict(logits=None), b"logits"), (dict(logits=P + 2), b"logits"), (dict(stride=999), b"stride"), (dict(stride=1 << 60), b"stride"), (dict(temp=0.0), b"temp"),
    (dict(temp=-1.0), b"temp"), (dict(temp=float("nan")), b"temp"), (dict(temp=float("inf")), b"temp"), (dict(top_ids=None), b"top_ids"), (dict(top_logprobs=None), b"top_ids"),
    (dict(top_n=0), b"top_ids"), (dict(top_n=0, top_ids=None, top_logprobs=None, logprob=None, entropy=None), b"no output"), (dict(targets=None), b"targets"),
    (dict(targets=P + 2), b"misaligned"), (dict(entropy=P + 1), b"misaligned"), (dict(work=None), b"work"), (dict(work=P + 8), b"work"), (dict(work_bytes=0), b"work"), (dict(work_bytes=-1), b"work"),
])
def test_logprobs_refuses_bad_arguments(change, needle):
    assert logprobs(**change) == _lib.HERO_EINVAL
    assert needle in lib.hero_last_error()


def test_logprobs_workspace():
    need = lib.hero_logprobs_work_bytes(3, 1000, 5)
    assert logprobs(work_bytes=need - 1) == _lib.HERO_EINVAL
    for v, top in ((1000, 0), (151936, 20), (64, 64)):
        sizes = [lib.hero_logprobs_work_bytes(m, v, top) for m in list(range(1, 300)) + [5000, 1 << 20]]
        assert sizes == sorted(sizes) and sizes[0] >= 0
    for bad in ((0, 1000, 5), (3, 0, 0), (3, 1000, 65), (3, 4, 5), (3, 1000, -1), (1 << 25, 1000, 5)):
        assert lib.hero_logprobs_work_bytes(*bad) == -1
