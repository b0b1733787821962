"""The long-context paged-cache operators: append, read, page selection, sparse
attention. Stored bytes, page summaries and selected pages are compared for
equality (with the oracle, with hero_attn_decode_paged, and with integer and
64-bit forms of their definitions); the attention with a 64-bit softmax under a
bound computed from the data."""
import numpy as np
import pytest

import oracle
from gpu_util import act_to_blocks, bits, check, dev, empty, host, ptr, stream

pytestmark = pytest.mark.gpu

EPS = np.float32(1e-6)
HALF_ULP = 2.0 ** -24  # a rounding to fp32, relative


@pytest.fixture(scope="module")
def lib():
    from hero_amd._lib import lib as _lib

    import torch

    assert torch.cuda.is_available(), "GPU tests need a GPU"
    return _lib


class Cache:
    """A paged cache in host memory: random finite contents, a shuffled page table."""

    def __init__(self, rng, seqs, max_pages, hkv, dh=128, ps=64, q8=False, spare=3, poison=False):
        self.seqs, self.max_pages, self.hkv, self.dh, self.ps, self.q8 = seqs, max_pages, hkv, dh, ps, q8
        self.n = seqs * max_pages + spare
        self.table = rng.permutation(self.n)[: seqs * max_pages].astype(np.int32).reshape(seqs, max_pages)
        shape = (self.n, 2, hkv, ps, dh)
        if q8:
            self.codes = rng.integers(-127, 128, shape).astype(np.int8)
            self.d = (rng.random(shape[:-1] + (dh // 32,)) * 0.02 + 0.01).astype(np.float16)
            if poison:
                self.d[:] = np.nan
        else:
            self.kv = rng.standard_normal(shape).astype(np.float16)
            if poison:
                self.kv[:] = np.nan
        self.sum_bytes = hkv * 2 * dh + -(-hkv * 4 // 16) * 16

    def bytes(self):
        if not self.q8:
            return np.ascontiguousarray(self.kv).view(np.uint8).reshape(self.n, -1)
        return np.concatenate([self.codes.view(np.uint8).reshape(self.n, -1), np.ascontiguousarray(self.d).view(np.uint8).reshape(self.n, -1)], 1)

    def values(self):
        """[page][2][hkv][ps][dh] float32: what is stored"""
        if not self.q8:
            return self.kv.astype(np.float32)
        return (self.codes.reshape(self.d.shape + (32,)).astype(np.float32) * self.d.astype(np.float32)[..., None]).reshape(self.codes.shape)

    def load(self, raw):
        raw = raw.reshape(self.n, -1)
        if not self.q8:
            self.kv = raw.view(np.float16).reshape(self.kv.shape)
        else:
            m = 2 * self.hkv * self.ps * self.dh
            self.codes = np.ascontiguousarray(raw[:, :m]).view(np.int8).reshape(self.codes.shape)
            self.d = np.ascontiguousarray(raw[:, m:]).view(np.float16).reshape(self.d.shape)

    def store(self, page, kv, slot, row):
        """row [hkv][dh] fp32 as append stores it"""
        if not self.q8:
            self.kv[page, kv, :, slot] = row.astype(np.float16)
            return
        for g in range(self.hkv):
            b = oracle.quantize_row_q8_0(row[g])
            self.codes[page, kv, g, slot] = b["qs"].reshape(-1)
            self.d[page, kv, g, slot] = b["d"].view(np.float16)


def round11(x):
    return ((np.asarray(x, np.float32).view(np.uint32) + np.uint32(0x1000)) & np.uint32(0xFFFFE000)).view(np.float32)


def quantize(x):
    """codes and 11-bit step of the last axis, in the reference quantizer's fp32 steps"""
    d = (np.abs(x).max(-1, keepdims=True) / np.float32(127)).astype(np.float32)
    inv = np.where(d != 0, np.float32(1) / np.where(d != 0, d, np.float32(1)), np.float32(0)).astype(np.float32)
    v = (x * inv).astype(np.float64)
    return (np.sign(v) * np.floor(np.abs(v) + 0.5)).astype(np.int64), round11(d[..., 0])


def summary_of(keys):
    """keys [n][dh] as stored -> int8 [2][dh], step"""
    q, d = quantize(np.concatenate([keys.max(0), -keys.min(0)])[None])
    return q[0].astype(np.int8).reshape(2, -1), d[0]


def sparse_args(c, hq, rows, pos, seq=None, dev_seq=None, **f):
    from hero_amd._lib import AttnDecodeArgs, AttnPagedArgs, AttnSparseArgs

    dh, kw = c.dh, c.hkv * c.dh
    f = {"proj": None, "stride": 2 * hq * dh + 2 * kw, "k_off": 2 * hq * dh, "v_off": 2 * hq * dh + kw, "gq": None, "gk": None, "cs": None, "q_rot": None,
         "scale": 1.0, "act": None, "out": None, "pages": None, "table": None, "work": None, "work_bytes": 0, "rope": 0, "summaries": None, "selected": None,
         "top": 0, "sink": 0, "recent": 1, "pool_pages": c.n, **f}
    a = AttnDecodeArgs(f["proj"], f["stride"], f["k_off"], f["v_off"], f["gq"], f["gk"], EPS, f["cs"], None, None, 0, pos, None, f["q_rot"], f["scale"], 0,
                       f["act"], f["out"], rows, hq, c.hkv, dh)
    p = AttnPagedArgs(a, f["pages"], f["table"], c.ps, c.max_pages, f["work"], f["work_bytes"], 1 if c.q8 else 0)
    return AttnSparseArgs(p, f["pool_pages"], f["rope"], dev_seq, c.seqs, f["summaries"], f["selected"], f["top"], f["sink"], f["recent"])


# ---- append -----------------------------------------------------------------------------
def rotated(x, gamma, inv, pos):
    return oracle.rope_apply(oracle.rmsnorm(x, gamma, EPS), inv, int(pos))


def run_append(lib, rng, c, hq, seq, pos, table=None, row_seq=True, stride_more=0, rope=None):
    """appends random rows; returns (proj, gammas, inv, q_rot, summaries before, after) and leaves the pool in c"""
    rows, dh, kw = len(pos), c.dh, c.hkv * c.dh
    stride = 2 * hq * dh + 2 * kw + stride_more
    proj = rng.standard_normal((rows, stride)).astype(np.float32)
    gq, gk = ((1 + 0.1 * rng.standard_normal(dh)).astype(np.float32) for _ in range(2))
    inv, span = oracle.rope_inv_freq(dh, 1e6, 32), c.max_pages * c.ps
    rope = span if rope is None else rope
    sums = rng.integers(0, 256, (c.n, c.sum_bytes)).astype(np.uint8)
    d = {k: dev(v) for k, v in dict(proj=proj, gq=gq, gk=gk, cs=oracle.rope_table(dh, 1e6, 32, rope), pages=c.bytes(), table=c.table if table is None else table,
                                    pos=np.asarray(pos, np.int32), seq=np.asarray(seq, np.int32), sums=sums).items()}
    q0 = rng.standard_normal((rows, hq, dh)).astype(np.float32)
    d_q = dev(q0)
    args = sparse_args(c, hq, rows, ptr(d["pos"]), dev_seq=ptr(d["seq"]) if row_seq else None, proj=ptr(d["proj"]), stride=stride, gq=ptr(d["gq"]), gk=ptr(d["gk"]),
                       cs=ptr(d["cs"]), q_rot=ptr(d_q), pages=ptr(d["pages"]), table=ptr(d["table"]), rope=rope, summaries=ptr(d["sums"]))
    check(lib.hero_kv_append_paged(args, stream()))
    got_q = host(d_q, np.float32, (rows, hq, dh))
    c.load(host(d["pages"], np.uint8))
    return proj, gq, gk, inv, q0, got_q, sums, host(d["sums"], np.uint8, sums.shape)


def check_append(before, c, hq, seq, pos, table, ran, rope=None):
    proj, gq, gk, inv, q0, got_q, sums0, sums = ran
    dh, kw, span = c.dh, c.hkv * c.dh, c.max_pages * c.ps
    rope = span if rope is None else rope
    ends = {}
    for r in range(len(pos)):
        if not (0 <= pos[r] < min(span, rope) and 0 <= seq[r] < c.seqs):
            assert np.array_equal(got_q[r], q0[r]), f"row {r} is left out"
            continue
        q = proj[r, : 2 * hq * dh].reshape(hq, 2, dh)[:, 0]
        assert np.array_equal(bits(got_q[r]), bits(rotated(q, gq, inv, pos[r]).reshape(hq, dh))), f"row {r}: q"
        page = table[seq[r], pos[r] // c.ps]
        if not 0 <= page < c.n:
            continue
        before.store(page, 0, pos[r] % c.ps, rotated(proj[r, 2 * hq * dh:2 * hq * dh + kw].reshape(c.hkv, dh), gk, inv, pos[r]).reshape(c.hkv, dh))
        before.store(page, 1, pos[r] % c.ps, proj[r, 2 * hq * dh + kw:2 * hq * dh + 2 * kw].reshape(c.hkv, dh))
        ends[page] = max(ends.get(page, 0), pos[r] % c.ps + 1)
    assert np.array_equal(c.bytes(), before.bytes()), "the pool: appended rows as the oracle stores them, every other byte as it was"
    values = before.values()
    want = sums0.copy()
    for page, n in ends.items():
        for g in range(c.hkv):
            q, d = summary_of(values[page, 0, g, :n])
            want[page, g * 2 * dh:(g + 1) * 2 * dh] = q.view(np.uint8).reshape(-1)
            want[page, c.hkv * 2 * dh + 4 * g:][:4] = np.array([d], np.float32).view(np.uint8)
    assert np.array_equal(sums, want), "summaries of the touched pages, the others as they were"


def copy_of(c):
    import copy

    return copy.deepcopy(c)


@pytest.mark.parametrize("q8,dh,ps,hq,hkv", [(False, 128, 16, 8, 2), (True, 128, 16, 8, 2), (False, 128, 64, 6, 2), (True, 128, 64, 8, 8), (False, 256, 64, 8, 4),
                                             (False, 256, 16, 3, 3), (True, 128, 256, 8, 1), (False, 128, 48, 4, 2)])
def test_append_of_ragged_rows_equals_oracle(lib, q8, dh, ps, hq, hkv):
    """Chunks of several sequences in one call -- starting and ending inside
    pages, a single row, a sequence without rows, padding rows between and behind
    -- and the page summaries over the old and new keys."""
    rng = np.random.default_rng(ps + dh + hq)
    c = Cache(rng, 5, -(-330 // ps), hkv, dh, ps, q8)
    span = c.max_pages * ps
    seq, pos = [], []
    for s, (first, n) in enumerate([(0, ps + 3), (ps - 1, 2), (37, 1), (0, 0), (span - 5, 5)]):
        seq += [s] * n
        pos += list(range(first, first + n))
        if s == 1:
            seq, pos = seq + [2, 7, -1], pos + [-1, 3, 4]  # padding, sequences out of range
    seq, pos = seq + [4, 0, 0], pos + [span, -5, -1]
    before = copy_of(c)
    ran = run_append(lib, rng, c, hq, seq, pos, stride_more=3)
    check_append(before, c, hq, seq, pos, c.table, ran)


@pytest.mark.parametrize("q8", [False, True])
def test_append_ignores_bad_pages_and_positions_past_the_rope_table(lib, q8):
    rng = np.random.default_rng(5)
    c = Cache(rng, 3, 4, 2, 128, 32, q8)
    table = c.table.copy()
    table[0, 1], table[1, 0], table[2, 2] = -1, c.n, 1 << 30
    seq = [0] * 100 + [1] * 40 + [2] * 20
    pos = list(range(10, 110)) + list(range(0, 40)) + list(range(60, 80))
    before = copy_of(c)
    ran = run_append(lib, rng, c, 4, seq, pos, table=table, rope=75)
    check_append(before, c, 4, seq, pos, table, ran, rope=75)


def test_append_of_thousands_of_rows(lib):
    """More rows than one look of the workgroups that search for runs takes in:
    a long chunk, then rows of many sequences."""
    rng = np.random.default_rng(61)
    c = Cache(rng, 130, 66, 1, 128, 64)
    n = 4100
    seq, pos = [0] * n + list(range(1, 130)), list(range(63, 63 + n)) + [int(p) for p in rng.integers(0, 66 * 64, 129)]
    before = copy_of(c)
    ran = run_append(lib, rng, c, 1, seq, pos)
    check_append(before, c, 1, seq, pos, c.table, ran)


@pytest.mark.parametrize("q8,dh,ps", [(False, 128, 16), (False, 128, 64), (True, 128, 16), (True, 128, 64), (False, 256, 64)])
def test_append_stores_what_the_decode_attention_stores(lib, q8, dh, ps):
    """Token by token through hero_attn_decode_paged and in one chunk through
    hero_kv_append_paged: the same pool bytes and rotated queries."""
    from hero_amd._lib import AttnDecodeArgs, AttnPagedArgs

    rng = np.random.default_rng(11)
    hq, hkv, n = 8, 2, 70
    c = Cache(rng, 1, -(-n // ps), hkv, dh, ps, q8)
    start, pos = c.bytes().copy(), list(range(n))
    proj, gq, gk, _, _, got_q, _, _ = run_append(lib, rng, c, hq, [0] * n, pos)
    d_pages, d_table, d_gq, d_gk = dev(start), dev(c.table), dev(gq), dev(gk)
    d_cs = dev(oracle.rope_table(dh, 1e6, 32, c.max_pages * ps))
    wb = lib.hero_attn_paged_work_bytes(c.max_pages * ps, 0, 1, hq, hkv, dh)
    work, act, q_rot = empty(wb), empty(lib.hero_q8_0_act_bytes(1, hq * dh)), empty(hq * dh * 4)
    for t in range(n):
        d_p, d_pos = dev(proj[t]), dev(np.array([t], np.int32))
        a = AttnDecodeArgs(ptr(d_p), proj.shape[1], 2 * hq * dh, 2 * hq * dh + hkv * dh, ptr(d_gq), ptr(d_gk), EPS, ptr(d_cs), None, None, 0, ptr(d_pos), None,
                           ptr(q_rot), 0.1, 0, ptr(act), None, 1, hq, hkv, dh)
        check(lib.hero_attn_decode_paged(AttnPagedArgs(a, ptr(d_pages), ptr(d_table), ps, c.max_pages, ptr(work), wb, 1 if q8 else 0), stream()))
        assert np.array_equal(bits(host(q_rot, np.float32)), bits(got_q[t].reshape(-1))), t
    assert np.array_equal(host(d_pages, np.uint8), c.bytes().reshape(-1))


# ---- read -------------------------------------------------------------------------------
@pytest.mark.parametrize("f16", [0, 1])
@pytest.mark.parametrize("q8,dh,ps,hkv", [(False, 128, 64, 2), (True, 128, 64, 8), (False, 256, 16, 3), (True, 128, 16, 1)])
def test_read_returns_what_is_stored(lib, q8, dh, ps, hkv, f16):
    """Rows in any order, twice, left out and in bad pages; every combination of
    missing outputs; fp32 values are exact, fp16 ones rounded once."""
    from hero_amd._lib import KvReadArgs

    rng = np.random.default_rng(ps + hkv)
    c = Cache(rng, 3, 6, hkv, dh, ps, q8)
    c.table[1, 2] = c.n  # holds nothing
    rows = 77
    seq, pos = rng.integers(0, 3, rows).astype(np.int32), rng.integers(0, 6 * ps, rows).astype(np.int32)
    pos[5], seq[9], pos[11], seq[12], pos[12] = -1, 3, 6 * ps, 1, 2 * ps
    seq[20], pos[20] = seq[21], pos[21]
    sums = np.zeros((c.n, c.sum_bytes), np.uint8)
    codes, steps = rng.integers(-127, 128, (c.n, hkv, 2, dh)).astype(np.int8), round11(rng.random((c.n, hkv)) + 0.1)
    sums[:, : hkv * 2 * dh] = codes.reshape(c.n, -1).view(np.uint8)
    sums[:, hkv * 2 * dh: hkv * 2 * dh + 4 * hkv] = steps.view(np.uint8).reshape(c.n, -1)
    t = np.float16 if f16 else np.float32
    live = [r for r in range(rows) if 0 <= pos[r] < 6 * ps and 0 <= seq[r] < 3 and c.table[seq[r], pos[r] // ps] < c.n]
    assert len(live) < rows - 3
    page = np.array([c.table[seq[r], pos[r] // ps] for r in live])
    values = c.values()
    want = [values[page, 0, :, pos[live] % ps], values[page, 1, :, pos[live] % ps],
            codes[page, :, 0].astype(np.float32) * steps[page][..., None], -codes[page, :, 1].astype(np.float32) * steps[page][..., None]]
    d = [dev(x) for x in (c.bytes(), c.table, pos, seq, sums)]
    for outs in (15, 1, 2, 12, 6):
        fill = rng.standard_normal((4, rows, hkv * dh)).astype(t)
        d_out = [dev(x) for x in fill]
        at = [ptr(x) if outs >> i & 1 else None for i, x in enumerate(d_out)]
        check(lib.hero_kv_read_paged(KvReadArgs(ptr(d[0]), ptr(d[1]), ps, 6, int(q8), c.n, ptr(d[4]) if outs & 12 else None, ptr(d[2]), ptr(d[3]), rows, 3, hkv, dh, f16, *at),
                                     stream()))
        for i in range(4):
            expect = fill[i].copy()
            if outs >> i & 1:
                expect[live] = want[i].reshape(len(live), -1).astype(t)
            assert np.array_equal(host(d_out[i], t, (rows, hkv * dh)), expect), f"output {i} of {outs}"


# ---- selection --------------------------------------------------------------------------
def select_reference(q_rot, codes, steps, table, seq, pos, ps, n_pool, top, sink, recent):
    rows, hq, dh = q_rot.shape
    hkv = codes.shape[1]
    out = np.full((rows, hkv, top), -1, np.int32)
    q, dq = quantize(q_rot)
    split = np.concatenate([np.maximum(q, 0), np.maximum(-q, 0)], -1).reshape(rows, hkv, hq // hkv, 2 * dh)
    dq = dq.reshape(rows, hkv, -1)
    for r in range(rows):
        if not (0 <= pos[r] < table.shape[1] * ps and 0 <= seq[r] < table.shape[0]):
            continue
        vis = pos[r] // ps + 1
        page = table[seq[r], :vis].astype(np.int64)
        ok = (page >= 0) & (page < n_pool)
        b = codes[np.where(ok, page, 0)].reshape(vis, hkv, 2 * dh).astype(np.int64)
        for g in range(hkv):
            score = ((b[:, g] @ split[r, g].T).astype(np.float64) * dq[r, g].astype(np.float64)).max(1) * steps[np.where(ok, page, 0), g].astype(np.float64)
            score[~ok] = -np.inf
            score[:sink] = np.inf
            score[max(0, vis - recent):] = np.inf
            take = np.sort(np.argsort(-score, kind="stable")[:top])
            out[r, g, : len(take)] = take
    return out


def run_select(lib, q_rot, codes, steps, table, seq, pos, ps, n_pool, top, sink, recent, row_seq=True):
    rows, hq, dh = q_rot.shape
    n, hkv = codes.shape[:2]

    class C:  # the fields sparse_args reads
        pass

    c = C()
    c.dh, c.hkv, c.n, c.ps, c.max_pages, c.seqs, c.q8 = dh, hkv, n_pool, ps, table.shape[1], table.shape[0], False
    sums = np.zeros((n, hkv * 2 * dh + -(-hkv * 4 // 16) * 16), np.uint8)
    sums[:, : hkv * 2 * dh] = codes.reshape(n, -1).view(np.uint8)
    sums[:, hkv * 2 * dh: hkv * 2 * dh + 4 * hkv] = steps.view(np.uint8).reshape(n, -1)
    d = {k: dev(v) for k, v in dict(q=q_rot, sums=sums, table=table.astype(np.int32), pos=np.asarray(pos, np.int32), seq=np.asarray(seq, np.int32)).items()}
    wb = lib.hero_attn_select_work_bytes(rows, hkv, c.max_pages)
    work, sel = dev(np.full(wb, 0xFF, np.uint8)), dev(np.full((rows, hkv, top), 77, np.int32))
    args = sparse_args(c, hq, rows, ptr(d["pos"]), dev_seq=ptr(d["seq"]) if row_seq else None, q_rot=ptr(d["q"]), table=ptr(d["table"]), work=ptr(work), work_bytes=wb,
                       summaries=ptr(d["sums"]), selected=ptr(sel), top=top, sink=sink, recent=recent)
    check(lib.hero_attn_select_pages(args, stream()))
    return host(sel, np.int32, (rows, hkv, top))


def select_inputs(rng, n, hkv, hq, dh, rows):
    codes = rng.integers(-127, 128, (n, hkv, 2, dh)).astype(np.int8)
    steps = round11(rng.random((n, hkv)) * 0.05 + 0.005)
    return codes, steps, rng.standard_normal((rows, hq, dh)).astype(np.float32)


@pytest.mark.parametrize("hq,hkv,dh,ps,top,sink,recent", [(32, 8, 128, 64, 16, 1, 2), (8, 2, 128, 16, 5, 0, 1), (6, 2, 128, 64, 33, 2, 1), (8, 8, 256, 32, 7, 1, 1),
                                                          (16, 2, 128, 64, 64, 0, 3), (10, 2, 256, 64, 8, 3, 5), (7, 1, 128, 128, 4, 1, 2), (4, 2, 128, 64, 1, 0, 1)])
def test_select_equals_the_integer_definition(lib, hq, hkv, dh, ps, top, sink, recent):
    """Rows of ragged chunks and padding, lists longer and shorter than the pages
    seen, pages that hold nothing."""
    rng = np.random.default_rng(hq * ps + top)
    seqs, max_pages = 3, 150
    n = seqs * max_pages
    rows = 41
    codes, steps, q = select_inputs(rng, n, hkv, hq, dh, rows)
    table = rng.permutation(n).astype(np.int32).reshape(seqs, max_pages)
    table[0, 3], table[1, 5], table[2, 0] = -1, n, 1 << 30
    seq = [0] * 20 + [1] * 1 + [2] * 20
    pos = list(range(max_pages * ps - 20, max_pages * ps)) + [7 * ps] + list(range(top * ps - 10, top * ps + 10))
    pos[3], seq[4], pos[40], seq[30] = -1, -2, max_pages * ps, 3
    got = run_select(lib, q, codes, steps, table, seq, pos, ps, n, top, sink, recent)
    assert np.array_equal(got, select_reference(q, codes, steps, table, seq, pos, ps, n, top, sink, recent))


@pytest.mark.parametrize("pages,ps,top", [(63, 64, 8), (64, 64, 8), (65, 64, 8), (255, 16, 200), (1000, 64, 64), (1025, 64, 1024), (4097, 64, 64), (5000, 16, 4096), (17000, 16, 300)])
def test_select_of_single_tokens_over_short_and_long_contexts(lib, pages, ps, top):
    rng = np.random.default_rng(pages)
    hq, hkv, dh, B = 8, 2, 128, 2
    codes, steps, q = select_inputs(rng, 2048, hkv, hq, dh, B)
    table = rng.integers(0, 2048, (B, pages)).astype(np.int32)  # pages shared: equal scores
    pos = [pages * ps - 1, (pages - 1) * ps]
    got = run_select(lib, q, codes, steps, table, [0, 1], pos, ps, 2048, top, 1, 2, row_seq=False)
    assert np.array_equal(got, select_reference(q, codes, steps, table, [0, 1], pos, ps, 2048, top, 1, 2))


@pytest.mark.parametrize("hq,hkv,dh,pages,ps,top", [(8, 2, 128, 600, 64, 20), (8, 2, 128, 1030, 64, 40), (16, 2, 256, 1100, 16, 30), (4, 2, 128, 4200, 16, 64), (8, 1, 128, 16500, 16, 100),
                                                    (2, 2, 128, 1024, 16, 500)])
def test_select_of_chunks_over_long_contexts(lib, hq, hkv, dh, pages, ps, top):
    """Rows of two sequences in one tile, at the ends of long lists."""
    rng = np.random.default_rng(pages + top)
    codes, steps, q = select_inputs(rng, 3000, hkv, hq, dh, 9)
    table = rng.integers(0, 3000, (2, pages)).astype(np.int32)
    seq, pos = [0] * 6 + [1] * 3, [pages * ps - 6 + i for i in range(6)] + [pages * ps // 2 + i for i in range(3)]
    got = run_select(lib, q, codes, steps, table, seq, pos, ps, 3000, top, 1, 2)
    assert np.array_equal(got, select_reference(q, codes, steps, table, seq, pos, ps, 3000, top, 1, 2))


@pytest.mark.parametrize("pages", [100, 700, 5000])
@pytest.mark.parametrize("good", [0, 3])
def test_select_where_hardly_a_page_holds_anything(lib, pages, good):
    """Pages that hold nothing rank behind those that do, and among themselves by
    number; NaN steps and queries stay inside their rows."""
    rng = np.random.default_rng(pages)
    codes, steps, q = select_inputs(rng, 200, 2, 8, 128, 3)
    table = np.full((3, pages), -1, np.int32)
    for s in range(3):
        table[s, rng.permutation(pages)[:good]] = np.arange(good)
    pos = [pages * 16 - 1] * 3
    got = run_select(lib, q, codes, steps, table, range(3), pos, 16, 200, 12, 1, 2, row_seq=False)
    want = select_reference(q, codes, steps, table, range(3), pos, 16, 200, 12, 1, 2)
    assert np.array_equal(got, want)
    steps[7] = np.nan
    q[1, 2, 5], q[1, 6, 0] = np.nan, np.inf
    table[0, 5] = 7
    again = run_select(lib, q, codes, steps, table, range(3), pos, 16, 200, 12, 1, 2, row_seq=False)
    assert np.array_equal(again[2], want[2])
    for r in (0, 1):  # some choice, in range, ascending, with the pages that are always there
        assert np.all(np.diff(again[r], axis=1) > 0) and again[r].min() == 0 and again[r].max() == pages - 1


def test_select_breaks_ties_to_the_lowest_page(lib):
    """All pages alike, zero queries and zero steps: the first pages are taken;
    two values of the score: the larger first, then the first of the smaller."""
    rng = np.random.default_rng(3)
    hq, hkv, dh, pages, top = 4, 2, 128, 90, 12
    codes, steps, q = select_inputs(rng, pages, hkv, hq, dh, 1)
    codes[:], steps[:] = codes[:1], steps[:1]
    table = np.arange(pages, dtype=np.int32)[None]
    for kind in range(4):
        s, x = steps.copy(), q.copy()
        if kind == 1:
            x[:] = 0
        elif kind == 2:
            s[:] = 0
        elif kind == 3:
            s[::9] = round11(s[0] * np.float32(1.5))
            codes = np.abs(codes)
        got = run_select(lib, x, codes, s, table, [0], [pages * 64 - 1], 64, pages, top, 0, 1)
        assert np.array_equal(got, select_reference(x, codes, s, table, [0], [pages * 64 - 1], 64, pages, top, 0, 1)), kind
        if kind < 3:
            assert got[0, 0].tolist() == list(range(top - 1)) + [pages - 1]


# ---- attention --------------------------------------------------------------------------
def attend_reference(q, gate, k, v, scale):
    """q, gate [dh], k, v [n][dh] in float64 -> (out, bound on an fp32 evaluation's error).
    The bound: a score sums dh products in fp32, each with the query's own
    rounding: off by at most (dh + 4) u scale sum|q k| (u = 2^-24), and the scaling to the
    exponent's base, the subtraction of the maximum and the exponential add at most
    6 u (|s| + |max| + 1) more; the weights' relative error is twice that (numerator and total),
    the weighted sum and the total add n + 8 roundings each, and the gate 8."""
    u = HALF_ULP
    if len(k) == 0:
        return np.zeros_like(q), np.zeros_like(q)
    s = scale * (k @ q)
    err = (len(q) + 4) * u * scale * (np.abs(k) @ np.abs(q)) + 6 * u * (np.abs(s) + np.abs(s.max()) + 1)
    w = np.exp(s - s.max())
    w /= w.sum()
    sig = 1 / (1 + np.exp(-gate))
    return (w @ v) * sig, (2 * err.max() + (2 * len(k) + 24) * u) * (w @ np.abs(v)) * sig + 1e-37


def run_attend(lib, c, hq, q_rot, proj, seq, pos, sel, row_seq=True, act=True, out=True, pool=None, pool_pages=None, table=None, fill=0.0):
    rows, top = len(pos), sel.shape[2]
    d = {k: dev(v) for k, v in dict(q=q_rot, proj=proj, table=c.table if table is None else table, pos=np.asarray(pos, np.int32), seq=np.asarray(seq, np.int32),
                                    sel=sel.astype(np.int32)).items()}
    d_pages = dev(c.bytes()) if pool is None else pool
    wb = lib.hero_attn_sparse_work_bytes(rows, hq, c.hkv, c.dh, c.ps, top)
    work = dev(np.full(max(16, wb), 0xFF, np.uint8))
    d_out, d_act = dev(np.full((rows, hq * c.dh), fill, np.float32)), dev(np.full(lib.hero_q8_0_act_bytes(rows, hq * c.dh), 0x55, np.uint8))
    args = sparse_args(c, hq, rows, ptr(d["pos"]), dev_seq=ptr(d["seq"]) if row_seq else None, q_rot=ptr(d["q"]), proj=ptr(d["proj"]), stride=proj.shape[1],
                       scale=float(np.float32(1 / np.sqrt(c.dh))), pages=ptr(d_pages), table=ptr(d["table"]), work=ptr(work), work_bytes=wb, selected=ptr(d["sel"]), top=top,
                       act=ptr(d_act) if act else None, out=ptr(d_out) if out else None, pool_pages=c.n if pool_pages is None else pool_pages)
    check(lib.hero_attn_sparse_paged(args, stream()))
    return host(d_out, np.float32, (rows, hq * c.dh)), host(d_act, np.uint8)


def check_attend(c, hq, q_rot, proj, seq, pos, sel, got, act=None, table=None, rows=None, fill=0.0, dropped=0.0):
    """`dropped`: what a weight may lose, as a part of the largest weight, per key, where the value
    block's step is the largest of the row's keys."""
    values, dh, grp = c.values(), c.dh, hq // c.hkv
    table = c.table if table is None else table
    scale = float(np.float32(1 / np.sqrt(dh)))
    blocks = None
    for r in range(len(pos)) if rows is None else rows:
        if not (0 <= pos[r] < c.max_pages * c.ps and 0 <= seq[r] < c.seqs):
            assert np.all(got[r] == np.float32(fill)), f"row {r} is left out"
            continue
        for g in range(c.hkv):
            ks, vs = [np.zeros((0, dh))], [np.zeros((0, dh))]
            for lp in sel[r, g]:
                if 0 <= lp <= pos[r] // c.ps and 0 <= table[seq[r], lp] < c.n:
                    n, page = min(c.ps, pos[r] + 1 - lp * c.ps), table[seq[r], lp]
                    ks.append(values[page, 0, g, :n].astype(np.float64))
                    vs.append(values[page, 1, g, :n].astype(np.float64))
            k, v = np.concatenate(ks), np.concatenate(vs)
            for h in range(g * grp, (g + 1) * grp):
                want, bound = attend_reference(q_rot[r, h].astype(np.float64), proj[r, h * 2 * dh + dh:(h + 1) * 2 * dh].astype(np.float64), k, v, scale)
                if dropped:
                    largest = np.repeat(np.abs(v).reshape(len(v), dh // 32, 32).max((0, 2)), 32)
                    bound = bound + dropped * len(k) * largest
                d = np.abs(got[r, h * dh:(h + 1) * dh] - want)
                assert np.all(d <= bound), f"row {r} head {h}: {np.max(d / bound):.3g} of the bound"
        if act is not None:
            if blocks is None:
                m = got.shape[0]
                qs = act[: got.size].view(np.int8).reshape(m, -1)
                ds = act[got.size:].view(np.float32).reshape(m, -1)
            b = oracle.quantize_row_q8_0(got[r])
            assert np.array_equal(qs[r], b["qs"].reshape(-1)) and np.array_equal(ds[r], b["d"].view(np.float16).astype(np.float32)), f"row {r}: act"


def random_lists(rng, rows, hkv, top, seen):
    """ascending distinct pages among those seen, -1 behind; some lists short or empty"""
    sel = np.full((rows, hkv, top), -1, np.int32)
    for r in range(rows):
        for g in range(hkv):
            n = min(top, max(0, seen[r]))
            if n and rng.random() < 0.2:
                n = int(rng.integers(0, n + 1))
            sel[r, g, :n] = np.sort(rng.permutation(max(1, seen[r]))[:n])
    return sel


SHAPES = [(False, 128, 64, 32, 8, 8), (True, 128, 64, 32, 8, 8), (False, 128, 16, 8, 2, 7), (True, 128, 16, 8, 2, 7), (False, 256, 64, 16, 4, 6), (False, 256, 32, 5, 1, 9),
          (False, 128, 48, 6, 2, 5), (True, 128, 48, 6, 2, 5), (False, 128, 256, 8, 8, 3), (True, 128, 256, 16, 2, 3), (False, 128, 64, 7, 1, 40), (True, 128, 32, 5, 1, 33),
          (False, 256, 128, 16, 2, 2), (True, 128, 64, 2, 1, 1), (False, 128, 64, 8, 1, 1)]


@pytest.mark.parametrize("q8,dh,ps,hq,hkv,top", SHAPES)
def test_attend_equals_64_bit_softmax(lib, q8, dh, ps, hq, hkv, top):
    """Ragged rows of three sequences with padding, the first position of a page
    and the last, contexts of one key, empty and short lists."""
    rng = np.random.default_rng(ps * hq + top + dh)
    max_pages = max(6, top + 3)
    c = Cache(rng, 3, max_pages, hkv, dh, ps, q8)
    seq = [0, 0, 0, 0, 1, 1, 2, 2, 2, 0, 5]
    pos = [max_pages * ps - 2, max_pages * ps - 1, 0, 1, ps, ps - 1, 17, 15, 16, -1, 3]
    rows = len(pos)
    q = (rng.standard_normal((rows, hq, dh)) * 1.5).astype(np.float32)
    proj = rng.standard_normal((rows, 2 * hq * dh + 5)).astype(np.float32)
    sel = random_lists(rng, rows, hkv, top, [p // ps + 1 for p in pos])
    sel[0, 0] = -1
    got, act = run_attend(lib, c, hq, q, proj, seq, pos, sel, fill=7.0)
    check_attend(c, hq, q, proj, seq, pos, sel, got, act, fill=7.0)
    assert np.all(got[0, : hq // hkv * dh] == 0), "nothing selected: zeros"


@pytest.mark.parametrize("q8,dh,ps,hq,hkv,top", [(False, 128, 64, 32, 8, 32), (True, 128, 64, 32, 8, 32), (False, 256, 64, 16, 4, 48), (True, 128, 16, 8, 2, 100)])
@pytest.mark.parametrize("b", [1, 16])
def test_attend_of_single_tokens(lib, q8, dh, ps, hq, hkv, top, b):
    rng = np.random.default_rng(b + top)
    c = Cache(rng, b, top + 9, hkv, dh, ps, q8)
    pos = [c.max_pages * ps - 1 - int(i) for i in rng.integers(0, 5 * ps, b)]
    q = (rng.standard_normal((b, hq, dh)) * 1.5).astype(np.float32)
    proj = rng.standard_normal((b, 2 * hq * dh)).astype(np.float32)
    sel = random_lists(rng, b, hkv, top, [p // ps + 1 for p in pos])
    got, act = run_attend(lib, c, hq, q, proj, range(b), pos, sel, row_seq=False)
    check_attend(c, hq, q, proj, range(b), pos, sel, got, act, rows=[0, b // 2, b - 1])


@pytest.mark.parametrize("q8,dh,rows,top", [(False, 128, 70, 2100), (True, 128, 3, 4096), (False, 256, 66, 4096), (True, 128, 66, 2049)])
def test_attend_of_very_long_lists(lib, q8, dh, rows, top):
    """Lists longer than one workgroup takes in, of pages that are mostly not
    there: in front, behind, and one here and there."""
    rng = np.random.default_rng(top + rows)
    hq, hkv, ps = 16, 8, 16
    c = Cache(rng, 1, 40, hkv, dh, ps, q8)
    pos = [int(p) for p in rng.integers(300, 640, rows)]
    sel = np.full((rows, hkv, top), -1, np.int32)
    for r in range(rows):
        for g in range(hkv):
            n = int(rng.integers(1, 19))
            sel[r, g, rng.permutation(top)[:n]] = rng.permutation(19)[:n]
    sel[0, 0] = -1
    sel[1, 0, :] = np.where(np.arange(top) == top - 1, 3, -1)
    q, proj = rng.standard_normal((rows, hq, dh)).astype(np.float32), rng.standard_normal((rows, 2 * hq * dh)).astype(np.float32)
    got, act = run_attend(lib, c, hq, q, proj, [0] * rows, pos, sel)
    check_attend(c, hq, q, proj, [0] * rows, pos, sel, got, act, rows=[0, 1, 2, rows // 2, rows - 1])


@pytest.mark.parametrize("q8", [False, True])
def test_attend_outputs_may_be_asked_for_one_at_a_time(lib, q8):
    rng = np.random.default_rng(8)
    c = Cache(rng, 2, 5, 2, 128, 64, q8)
    q, proj, pos = rng.standard_normal((2, 8, 128)).astype(np.float32), rng.standard_normal((2, 2048)).astype(np.float32), [300, 10]
    sel = random_lists(rng, 2, 2, 4, [5, 1])
    out, act = run_attend(lib, c, 8, q, proj, [0, 1], pos, sel)
    o2, a2 = run_attend(lib, c, 8, q, proj, [0, 1], pos, sel, act=False)
    o3, a3 = run_attend(lib, c, 8, q, proj, [0, 1], pos, sel, out=False)
    assert np.array_equal(bits(out), bits(o2)) and np.all(a2 == 0x55)
    assert np.array_equal(act, a3) and np.all(o3 == 0)


@pytest.mark.parametrize("q8,dh,ps", [(False, 128, 64), (True, 128, 64), (False, 256, 32), (False, 128, 16), (True, 128, 16)])
def test_attend_is_blind_to_what_lies_behind_the_position(lib, q8, dh, ps):
    """NaNs in every slot past a row's position and in every page that is not
    selected, infinities among them: the row's output is the same."""
    rng = np.random.default_rng(6)
    hq, hkv, top = 8, 2, 4
    c = Cache(rng, 1, 8, hkv, dh, ps, q8)
    pos = [5 * ps + 9, 6 * ps + ps - 1, 3 * ps, 7 * ps + 17 % ps]
    sel = np.array([[[0, 2, 4, 5]] * hkv, [[1, 3, 5, 6]] * hkv, [[0, 1, 2, 3]] * hkv, [[4, 5, 6, 7]] * hkv], np.int32)
    q, proj = rng.standard_normal((4, hq, dh)).astype(np.float32), rng.standard_normal((4, 2 * hq * dh)).astype(np.float32)
    for r in range(4):
        one = (q[r:r + 1], proj[r:r + 1], [0], pos[r:r + 1], sel[r:r + 1])
        got, _ = run_attend(lib, c, hq, *one)
        check_attend(c, hq, *one, got)
        bad = copy_of(c)
        for lp in range(8):
            n = pos[r] + 1 - lp * ps if lp in sel[r, 0] else 0
            page = bad.table[0, lp]
            for t in range(max(0, n), ps):
                if q8:
                    bad.d[page, :, :, t], bad.codes[page, :, :, t] = (np.nan, np.inf)[t % 2], 127
                else:
                    bad.kv[page, :, :, t] = (np.nan, np.inf, -np.inf)[t % 3]
        again, _ = run_attend(lib, bad, hq, *one)
        assert np.array_equal(bits(got), bits(again)), r


def test_attend_takes_lists_in_any_order_twice_and_out_of_range(lib):
    rng = np.random.default_rng(12)
    c = Cache(rng, 2, 6, 2, 128, 64)
    c.table[0, 4], c.table[1, 1] = -3, c.n
    sel = np.array([[[5, 0, 3, 3, -1, 1], [99, 6, -7, 2, 1 << 30, 0]], [[1, 1, 1, 0, 2, 5], [4, 4, 4, 4, 4, 4]]], np.int32)
    pos, q, proj = [5 * 64 + 3, 3 * 64], rng.standard_normal((2, 8, 128)).astype(np.float32), rng.standard_normal((2, 2048)).astype(np.float32)
    got, act = run_attend(lib, c, 8, q, proj, [0, 1], pos, sel)
    check_attend(c, 8, q, proj, [0, 1], pos, sel, got, act)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("scale", [1e-30, 1e-4, 60.0, 3e4])
def test_attend_of_small_and_large_queries(lib, q8, scale):
    """Queries from far below fp16's range to near its end: weights from equal
    ones to a single one."""
    rng = np.random.default_rng(4)
    c = Cache(rng, 1, 4, 2, 128, 64, q8)
    q = (rng.standard_normal((1, 8, 128)) * scale).astype(np.float32)
    q[0, 3] = 0
    q[0, 5, 7] = np.float32(scale * 40)
    proj, sel = rng.standard_normal((1, 2048)).astype(np.float32), np.array([[[0, 1, 3]] * 2], np.int32)
    got, act = run_attend(lib, c, 8, q, proj, [0], [250], sel)
    check_attend(c, 8, q, proj, [0], [250], sel, got, act)


@pytest.mark.parametrize("q8", [False, True])
def test_attend_weights_keep_both_their_terms(lib, q8):
    """Nearly equal weights of 32 keys over many rows: the bound is then 7e-6 of
    the mean value, half of what one weight kept to fp16 only would be off by."""
    rng = np.random.default_rng(77)
    c = Cache(rng, 64, 1, 8, 128, 32, q8)
    q, proj = (rng.standard_normal((64, 32, 128)) * 0.02).astype(np.float32), np.full((64, 8192), 20, np.float32)
    sel = np.zeros((64, 8, 1), np.int32)
    got, act = run_attend(lib, c, 32, q, proj, range(64), [31] * 64, sel, row_seq=False)
    check_attend(c, 32, q, proj, range(64), [31] * 64, sel, got, act)


def test_attend_of_subnormal_values(lib):
    """Cached values below fp16's normal range are not flushed."""
    rng = np.random.default_rng(78)
    c = Cache(rng, 1, 2, 2, 128, 64)
    c.kv[:, 1] = (rng.integers(-1023, 1024, c.kv[:, 1].shape) * 2.0 ** -24).astype(np.float16)
    q, proj = rng.standard_normal((1, 8, 128)).astype(np.float32), rng.standard_normal((1, 2048)).astype(np.float32)
    sel = np.array([[[0, 1]] * 2], np.int32)
    got, act = run_attend(lib, c, 8, q, proj, [0], [100], sel)
    check_attend(c, 8, q, proj, [0], [100], sel, got, act)


def test_attend_of_values_of_every_size(lib):
    """Cached values from fp16's smallest to its largest, keys among them."""
    rng = np.random.default_rng(14)
    c = Cache(rng, 1, 3, 1, 128, 64)
    c.kv[:, 1] = (rng.standard_normal(c.kv[:, 1].shape) * 2.0 ** rng.integers(-24, 14, c.kv[:, 1].shape)).astype(np.float16)
    c.kv[:, 0] = (rng.standard_normal(c.kv[:, 0].shape) * 2.0 ** rng.integers(-20, 3, c.kv[:, 0].shape)).astype(np.float16)
    q, proj, sel = rng.standard_normal((1, 4, 128)).astype(np.float32), rng.standard_normal((1, 1024)).astype(np.float32), np.array([[[0, 1, 2]]], np.int32)
    got, act = run_attend(lib, c, 4, q, proj, [0], [180], sel)
    check_attend(c, 4, q, proj, [0], [180], sel, got, act)


@pytest.mark.parametrize("rows", [1, 2, 5])
@pytest.mark.parametrize("hq,hkv,ps", [(8, 2, 64), (8, 1, 16), (2, 1, 32)])
def test_attend_over_steps_of_every_size(lib, rows, hq, hkv, ps):
    """Q8_0 blocks whose steps run from fp16's smallest to 2^9, zeros among them. A
    weight of at most 2^15 (the largest at least 2^13), times its step over a power of
    two at most twice the largest step, is two fp16 terms, so off by at most 2^-25
    where it is small: by 2 2^-25 / 2^13 = 2^-37 of the largest weight in units of the
    largest step, or of codes up to 127 times it."""
    rng = np.random.default_rng(90 + rows + hq)
    c = Cache(rng, 1, 5, hkv, 128, ps, True)
    shape = c.d[:, 0].shape
    c.codes[..., ::32] = 127  # a block's largest value is 127 of its steps
    c.d[:, 0] = (2.0 ** rng.integers(-18, -5, shape)).astype(np.float16)
    c.d[:, 1] = (rng.integers(1, 4, shape) * 2.0 ** rng.integers(-24, 9, shape)).astype(np.float16)
    c.d[:, 1][rng.random(shape) < 0.1] = 0
    c.d[1::2, 1] *= np.float16(2.0 ** -6)
    pos = [5 * ps - 9 + i for i in range(rows)]
    q, proj = rng.standard_normal((rows, hq, 128)).astype(np.float32), rng.standard_normal((rows, 2 * hq * 128)).astype(np.float32)
    sel = np.array([[[0, 2, 4] if (r + g) % 2 else [1, 3, 4] for g in range(hkv)] for r in range(rows)], np.int32)
    got, act = run_attend(lib, c, hq, q, proj, [0] * rows, pos, sel)
    check_attend(c, hq, q, proj, [0] * rows, pos, sel, got, act, dropped=2.0 ** -37)


def test_rows_of_a_chunk_equal_single_tokens(lib):
    """A row's attention is the same in a chunk of 70 rows and alone, up to the
    order of fp32 sums; and over all pages it is the chunk's full attention."""
    rng = np.random.default_rng(9)
    c = Cache(rng, 1, 7, 8, 128, 64)
    n = 70
    pos = list(range(7 * 64 - n, 7 * 64))
    q, proj = rng.standard_normal((n, 32, 128)).astype(np.float32), rng.standard_normal((n, 8192)).astype(np.float32)
    sel = np.full((n, 8, 7), -1, np.int32)
    for r in range(n):
        sel[r, :, : pos[r] // 64 + 1] = np.arange(pos[r] // 64 + 1)
    got, act = run_attend(lib, c, 32, q, proj, [0] * n, pos, sel)
    check_attend(c, 32, q, proj, [0] * n, pos, sel, got, act, rows=[0, 1, 5, 6, 33, 69])


def chunk_lists(rng, seq, pos, ps, hkv, top):
    """lists of neighbouring rows that mostly agree, as a chunk's do"""
    shared = rng.standard_normal((max(seq) + 1, hkv, max(pos) // ps + 1))
    sel = np.full((len(pos), hkv, top), -1, np.int32)
    for r in range(len(pos)):
        if pos[r] < 0:
            continue
        seen = pos[r] // ps + 1
        score = shared[seq[r], :, :seen] + 0.5 * rng.standard_normal((hkv, seen))
        n = min(top, seen)
        sel[r, :, :n] = np.sort(np.argsort(-score, axis=1)[:, :n], axis=1)
    return sel


CHUNKS = [(False, 128, 64, 32, 8, 6), (False, 128, 16, 24, 8, 20), (False, 128, 32, 16, 8, 9), (False, 128, 64, 8, 8, 5), (False, 256, 64, 32, 8, 4), (False, 256, 16, 16, 8, 11),
          (False, 128, 48, 64, 8, 7), (True, 128, 64, 32, 8, 6), (True, 128, 16, 16, 8, 20), (True, 128, 64, 64, 8, 5), (False, 128, 64, 32, 8, 128), (False, 128, 64, 16, 8, 129),
          (False, 128, 16, 32, 8, 256), (False, 128, 16, 24, 8, 257)]


@pytest.mark.parametrize("q8,dh,ps,hq,hkv,top", CHUNKS)
def test_attend_of_large_chunks(lib, q8, dh, ps, hq, hkv, top):
    """Chunks of three sequences of many rows, which share page reads between
    rows: rows of two sequences in one tile, padding inside tiles, empty lists,
    lists in any order, pages twice, out of range and holding nothing."""
    rng = np.random.default_rng(ps + hq + top + dh)
    c = Cache(rng, 3, max(9, min(top, 40) + 2), hkv, dh, ps, q8)
    span = c.max_pages * ps
    seq = [0] * 71 + [1] * 33 + [2] * 40
    pos = list(range(span - 71, span)) + list(range(ps - 3, ps + 30)) + list(range(0, 40))
    pos[5] = pos[70] = -1
    seq[100] = 3
    sel = chunk_lists(rng, [0 if s > 2 else s for s in seq], pos, ps, hkv, top)
    sel[2], sel[20, 1] = -1, -1
    sel[8] = sel[8][:, ::-1]
    sel[9, :, 1] = sel[9, :, 0]
    sel[10, 0, :3], sel[11, 0, :2] = sel[10, 0, 0], sel[10, 0, 0]
    sel[12, 1, 0], sel[13, 2, 1] = 1 << 30, -9
    table = c.table.copy()
    table[0, 1], table[2, 0] = -1, c.n
    q = (rng.standard_normal((len(pos), hq, dh)) * 1.5).astype(np.float32)
    proj = rng.standard_normal((len(pos), 2 * hq * dh)).astype(np.float32)
    got, act = run_attend(lib, c, hq, q, proj, seq, pos, sel, fill=3.0, table=table)
    check_attend(c, hq, q, proj, seq, pos, sel, got, act, fill=3.0, table=table, rows=[0, 1, 2, 3, 4, 5, 8, 9, 10, 11, 12, 13, 20, 21, 69, 70, 71, 72, 99, 100, 101, 103, 104, 105, 143])


@pytest.mark.parametrize("q8,hq", [(False, 32), (False, 16), (True, 32)])
def test_rows_of_a_chunk_do_not_reach_each_other(lib, q8, hq):
    """A page that only some rows of a tile select, and keys behind some rows'
    positions, hold infinities and NaNs: they reach the rows that see them and
    no other."""
    rng = np.random.default_rng(50 + hq)
    hkv, dh, ps, n = 8, 128, 64, 140
    c = Cache(rng, 1, 6, hkv, dh, ps, q8)
    pos = list(range(6 * ps - n, 6 * ps))
    sel = np.zeros((n, hkv, 2), np.int32)
    sel[:, :, 1] = np.array(pos)[:, None] // ps
    sel[::3, :, 0] = 1
    bad = copy_of(c)
    for value, page, slots in ((np.nan, 1, slice(None)), (np.inf, 5, slice(40, 64)), (-np.inf, 4, slice(50, 52))):
        at = c.table[0, page]
        if q8:
            bad.d[at, :, :, slots] = value
        else:
            bad.kv[at, 1, :, slots] = value
    q, proj = rng.standard_normal((n, hq, dh)).astype(np.float32), rng.standard_normal((n, 2 * hq * dh)).astype(np.float32)
    got, act = run_attend(lib, bad, hq, q, proj, [0] * n, pos, sel)
    first_bad = {5: 5 * ps + 40, 4: 4 * ps + 50}
    clean = [r for r in range(n) if r % 3 and not any(pos[r] >= f and page == pos[r] // ps for page, f in first_bad.items())]
    assert len(clean) > 30
    assert np.all(np.isfinite(got[clean])) and not np.any(np.isfinite(got[::3]))
    hit = [r for r in range(n) if pos[r] // ps == 5 and pos[r] >= first_bad[5]]
    assert not np.any(np.isfinite(got[hit]))
    check_attend(c, hq, q, proj, [0] * n, pos, sel, got, rows=clean[:12] + clean[-12:])


@pytest.mark.parametrize("q8", [False, True])
def test_offsets_past_32_bits(lib, q8):
    """Pages whose byte offset in the pool passes 2^32: appended, read, selected
    and attended to."""
    import torch

    from hero_amd._lib import KvReadArgs

    rng = np.random.default_rng(2)
    hq, hkv, dh, ps = 8, 8, 128, 256
    page_bytes = lib.hero_attn_page_bytes(hkv, dh, ps, int(q8))
    n = (1 << 32) // page_bytes + 9
    few = Cache(rng, 1, 3, hkv, dh, ps, q8, spare=0)
    few.table = np.array([[0, 1, 2]], np.int32)
    far = np.array([[n - 2, n - 7, n - 1]], np.int32)
    assert (n - 7) * page_bytes > 1 << 32
    pool = torch.zeros((n, page_bytes), dtype=torch.uint8, device="cuda")
    sums = torch.zeros(lib.hero_kv_summary_bytes(n, hkv, dh), dtype=torch.uint8, device="cuda")
    rows, pos = 5, [510, 511, 512, 513, 514]
    proj = rng.standard_normal((rows, 2 * hq * dh + 2 * hkv * dh)).astype(np.float32)
    g = np.ones(dh, np.float32)
    pool[far[0].tolist()] = dev(few.bytes()).view(3, -1)
    near = {"pool": dev(few.bytes()), "sums": empty(lib.hero_kv_summary_bytes(3, hkv, dh)), "table": dev(few.table), "n": 3}
    d = {k: dev(v) for k, v in dict(proj=proj, g=g, cs=oracle.rope_table(dh, 1e6, 32, 600), pos=np.array(pos, np.int32), seq=np.zeros(rows, np.int32)).items()}
    res = []
    for where in ({"pool": pool, "sums": sums, "table": dev(far), "n": n}, near):
        q_rot, sel, out = empty(rows * hq * dh * 4), empty(rows * hkv * 2 * 4), empty(rows * hq * dh * 4)
        kv = [empty(rows * hkv * dh * 4) for _ in range(4)]
        wb = max(lib.hero_attn_select_work_bytes(rows, hkv, 3), lib.hero_attn_sparse_work_bytes(rows, hq, hkv, dh, ps, 2))
        work = empty(wb)
        args = sparse_args(few, hq, rows, ptr(d["pos"]), dev_seq=ptr(d["seq"]), proj=ptr(d["proj"]), gq=ptr(d["g"]), gk=ptr(d["g"]), cs=ptr(d["cs"]), q_rot=ptr(q_rot),
                           scale=0.1, out=ptr(out), pages=ptr(where["pool"]), table=ptr(where["table"]), work=ptr(work), work_bytes=wb, rope=600, summaries=ptr(where["sums"]),
                           selected=ptr(sel), top=2, sink=0, recent=1, pool_pages=where["n"])
        check(lib.hero_kv_append_paged(args, stream()))
        check(lib.hero_kv_read_paged(KvReadArgs(ptr(where["pool"]), ptr(where["table"]), ps, 3, int(q8), where["n"], ptr(where["sums"]), ptr(d["pos"]), ptr(d["seq"]), rows, 1,
                                                hkv, dh, 0, *[ptr(x) for x in kv]), stream()))
        check(lib.hero_attn_select_pages(args, stream()))
        check(lib.hero_attn_sparse_paged(args, stream()))
        res.append([host(x, np.uint8) for x in (q_rot, *kv, sel, out)])
    for a, b in zip(*res):
        assert np.array_equal(a, b)
    assert np.any(res[0][1]) and np.any(res[0][-1])


# ---- together ---------------------------------------------------------------------------
@pytest.mark.parametrize("q8,dh", [(False, 128), (True, 128), (False, 256)])
def test_a_decoded_run_with_every_page_selected_equals_the_paged_attention(lib, q8, dh):
    """A prompt in two chunks and then tokens one by one: append, select with room
    for every page, attend; against hero_attn_decode_paged fed the same tokens.
    Both are fp32 evaluations of one softmax over the same stored values."""
    from hero_amd._lib import AttnDecodeArgs, AttnPagedArgs

    rng = np.random.default_rng(21)
    hq, hkv, ps, n, prompt = 8, 2, 64, 150, 130
    c = Cache(rng, 1, 3, hkv, dh, ps, q8)
    proj = rng.standard_normal((n, 2 * hq * dh + 2 * hkv * dh)).astype(np.float32)
    g, cs = dev(np.ones(dh, np.float32)), dev(oracle.rope_table(dh, 1e6, 32, c.max_pages * ps))
    scale = float(np.float32(1 / np.sqrt(dh)))
    pool, table = dev(c.bytes()), dev(c.table)
    d_proj, d_pos = dev(proj), dev(np.arange(n, dtype=np.int32))
    d_seq, sums = empty(n * 4), empty(lib.hero_kv_summary_bytes(c.n, hkv, dh))
    q_rot, out, sel = empty(n * hq * dh * 4), empty(n * hq * dh * 4), empty(n * hkv * 4 * 4)
    wb = max(lib.hero_attn_select_work_bytes(n, hkv, 3), lib.hero_attn_sparse_work_bytes(n, hq, hkv, dh, ps, 4))
    work = empty(wb)
    for r0, r1 in [(0, 100), (100, prompt)] + [(t, t + 1) for t in range(prompt, n)]:
        args = sparse_args(c, hq, r1 - r0, ptr(d_pos) + 4 * r0, dev_seq=ptr(d_seq), proj=ptr(d_proj) + 4 * r0 * proj.shape[1], gq=ptr(g), gk=ptr(g), cs=ptr(cs),
                           q_rot=ptr(q_rot) + 4 * r0 * hq * dh, scale=scale, out=ptr(out) + 4 * r0 * hq * dh, pages=ptr(pool), table=ptr(table), work=ptr(work), work_bytes=wb,
                           rope=c.max_pages * ps, summaries=ptr(sums), selected=ptr(sel) + r0 * hkv * 16, top=4, sink=1, recent=2)
        for call in (lib.hero_kv_append_paged, lib.hero_attn_select_pages, lib.hero_attn_sparse_paged):
            check(call(args, stream()))
    got, lists = host(out, np.float32, (n, hq * dh)), host(sel, np.int32, (n, hkv, 4))
    for r in range(n):
        assert np.array_equal(lists[r], np.broadcast_to([i if i <= r // ps else -1 for i in range(4)], (hkv, 4)))
    c.load(host(pool, np.uint8))
    check_attend(c, hq, host(q_rot, np.float32, (n, hq, dh)), proj, [0] * n, list(range(n)), lists, got, rows=[0, 1, 63, 64, 99, 100, 129, 130, 149])
    # the same tokens through the one-token kernel
    pool2, w2 = dev(np.zeros_like(c.bytes())), lib.hero_attn_paged_work_bytes(c.max_pages * ps, 0, 1, hq, hkv, dh)
    work2, act, qr, o2 = empty(w2), empty(lib.hero_q8_0_act_bytes(1, hq * dh)), empty(hq * dh * 4), empty(hq * dh * 4)
    for t in range(n):
        a = AttnDecodeArgs(ptr(d_proj) + 4 * t * proj.shape[1], proj.shape[1], 2 * hq * dh, 2 * hq * dh + hkv * dh, ptr(g), ptr(g), EPS, ptr(cs), None, None, 0,
                           ptr(d_pos) + 4 * t, None, ptr(qr), scale, 0, ptr(act), ptr(o2), 1, hq, hkv, dh)
        check(lib.hero_attn_decode_paged(AttnPagedArgs(a, ptr(pool2), ptr(table), ps, c.max_pages, ptr(work2), w2, int(q8)), stream()))
        if t % 10 == 9 or t < 2:
            one = host(o2, np.float32)
            np.testing.assert_allclose(got[t], one, rtol=1e-4, atol=1e-4 * np.abs(one).max(), err_msg=str(t))  # as the split kernel is held to its oracle


@pytest.mark.parametrize("q8", [False, True])
def test_captured_steps_replay_like_eager_ones(lib, q8):
    """append, select and attend captured on a stream of their own, replayed on
    new rows and positions with eager calls on another workspace in between."""
    import torch

    rng = np.random.default_rng(31)
    hq, hkv, dh, ps, b, top = 8, 2, 128, 64, 3, 5
    c = Cache(rng, b, 12, hkv, dh, ps, q8)
    width = 2 * hq * dh + 2 * hkv * dh
    g, cs, table = dev(np.ones(dh, np.float32)), dev(oracle.rope_table(dh, 1e6, 32, c.max_pages * ps)), dev(c.table)
    sums0 = rng.integers(0, 256, (c.n, c.sum_bytes)).astype(np.uint8)
    sums0[:, hkv * 2 * dh:] = 0
    sums0[:, hkv * 2 * dh: hkv * 2 * dh + 4 * hkv] = round11(rng.random((c.n, hkv)) * 0.05 + 0.01).view(np.uint8).reshape(c.n, -1)
    wb = max(lib.hero_attn_select_work_bytes(b, hkv, 12), lib.hero_attn_sparse_work_bytes(b, hq, hkv, dh, ps, top))

    def state():
        s = dict(pool=dev(c.bytes()), sums=dev(sums0), proj=empty(b * width * 4), pos=empty(b * 4), q=empty(b * hq * dh * 4), out=empty(b * hq * dh * 4),
                 act=empty(lib.hero_q8_0_act_bytes(b, hq * dh)), sel=empty(b * hkv * top * 4), work=empty(wb))
        s["args"] = sparse_args(c, hq, b, ptr(s["pos"]), proj=ptr(s["proj"]), gq=ptr(g), gk=ptr(g), cs=ptr(cs), q_rot=ptr(s["q"]), scale=0.088, out=ptr(s["out"]),
                                act=ptr(s["act"]), pages=ptr(s["pool"]), table=ptr(table), work=ptr(s["work"]), work_bytes=wb, rope=c.max_pages * ps, summaries=ptr(s["sums"]),
                                selected=ptr(s["sel"]), top=top, sink=1, recent=2)
        return s

    def step(s, st):
        for call in (lib.hero_kv_append_paged, lib.hero_attn_select_pages, lib.hero_attn_sparse_paged):
            check(call(s["args"], st))

    eager, graphed = state(), state()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        step(graphed, side.cuda_stream)
    for i in range(4):
        proj = torch.from_numpy(rng.standard_normal((b, width)).astype(np.float32).view(np.uint8).reshape(-1))
        pos = torch.from_numpy(np.array([600 + i, 63 + i, 127 + 130 * i], np.int32).view(np.uint8))
        for s in (eager, graphed):
            s["proj"].copy_(proj)
            s["pos"].copy_(pos)
        graph.replay()
        step(eager, stream())
        torch.cuda.synchronize()
        for k in ("pool", "sums", "q", "sel", "out", "act"):
            assert torch.equal(eager[k], graphed[k]), (i, k)
    assert len(np.unique(host(eager["sel"], np.int32))) > 5


def test_two_streams_with_workspaces_of_their_own(lib):
    import torch

    rng = np.random.default_rng(41)
    hq, hkv, dh, ps, top = 32, 8, 128, 64, 16
    c = Cache(rng, 4, 20, hkv, dh, ps)
    q, proj = rng.standard_normal((4, hq, dh)).astype(np.float32), rng.standard_normal((4, 2 * hq * dh)).astype(np.float32)
    pos = [1279, 1000, 640, 20]
    sel = random_lists(rng, 4, hkv, top, [p // ps + 1 for p in pos])
    want, _ = run_attend(lib, c, hq, q, proj, range(4), pos, sel, row_seq=False)
    d = [dev(x) for x in (c.bytes(), c.table, q, proj, np.array(pos, np.int32), sel)]
    wb = max(16, lib.hero_attn_sparse_work_bytes(4, hq, hkv, dh, ps, top))
    runs = []
    torch.cuda.synchronize()
    for _ in range(2):
        s, work, out = torch.cuda.Stream(), empty(wb), empty(4 * hq * dh * 4)
        args = sparse_args(c, hq, 4, ptr(d[4]), proj=ptr(d[3]), stride=2 * hq * dh, q_rot=ptr(d[2]), scale=float(np.float32(1 / np.sqrt(dh))), out=ptr(out), pages=ptr(d[0]),
                           table=ptr(d[1]), work=ptr(work), work_bytes=wb, selected=ptr(d[5]), top=top)
        runs.append((s, work, out, args))
    torch.cuda.synchronize()
    for _ in range(20):
        for s, _, _, args in runs:
            check(lib.hero_attn_sparse_paged(args, s.cuda_stream))
    torch.cuda.synchronize()
    for _, _, out, _ in runs:
        assert np.array_equal(bits(host(out, np.float32, want.shape)), bits(want))
