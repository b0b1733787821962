"""The long-context paged-cache operators at the edges of their definitions:
infinities among the stored keys and values, queries near the end of fp32's
range, a few keys of nearly equal weight, forms of single tokens, workspaces."""
import numpy as np
import pytest

import oracle
from gpu_util import bits, check, dev, empty, host, ptr, stream
from test_gpu_paged_long import (Cache, check_append, check_attend, copy_of, lib, quantize, random_lists, round11, run_append, run_attend, run_select, select_inputs,  # noqa: F401
                                 select_reference, sparse_args)

pytestmark = pytest.mark.gpu

U = 2.0 ** -24  # half a step of fp32, relative


# ---- infinities among what a row sees -----------------------------------------------------
def attend_ieee(q, gate, k, v, scale):
    """The definition in float64 with IEEE infinities, and the bound on an fp32
    evaluation's error where the result is finite: that of attend_reference over the
    keys of a score that is finite (the others have weight 0, or there is no finite result)."""
    from test_gpu_paged_long import attend_reference

    with np.errstate(all="ignore"):
        s = scale * (k * q).sum(1)
        w = np.exp(s - s.max())
        out = (w[:, None] * v).sum(0) / w.sum() / (1 + np.exp(-gate))
        near = np.isfinite(s)
        bound = np.zeros_like(out)
        if near.any():
            _, bound = attend_reference(q, gate, k[near], np.where(np.isfinite(v[near]), v[near], 0), scale)
    return out, bound


def check_ieee(c, hq, q, proj, seq, pos, sel, got):
    """every result, kind by kind; returns how many of each there were: finite ones,
    infinities, NaNs"""
    with np.errstate(invalid="ignore"):
        values = c.values().astype(np.float64)
    dh, grp = c.dh, hq // c.hkv
    scale, count = float(np.float32(1 / np.sqrt(dh))), np.zeros(3, int)
    for r in range(len(pos)):
        for g in range(c.hkv):
            at = [(c.table[seq[r], lp], min(c.ps, pos[r] + 1 - lp * c.ps)) for lp in sel[r, g] if lp >= 0]
            k, v = (np.concatenate([values[page, what, g, :n] for page, n in at]) for what in (0, 1))
            for h in range(g * grp, (g + 1) * grp):
                want, bound = attend_ieee(q[r, h].astype(np.float64), proj[r, h * 2 * dh + dh:(h + 1) * 2 * dh].astype(np.float64), k, v, scale)
                x, fin = got[r, h * dh:(h + 1) * dh], np.isfinite(want)
                name = f"row {r} head {h}"
                assert np.array_equal(np.isnan(x), np.isnan(want)), f"{name}: NaNs {np.isnan(x).sum()}, wanted {np.isnan(want).sum()}"
                assert np.array_equal(x[np.isinf(want)], want[np.isinf(want)]), f"{name}: infinities"
                assert np.all(np.abs(x[fin] - want[fin]) <= bound[fin]), f"{name}: {np.max(np.abs(x[fin] - want[fin]) / bound[fin]):.3g} of the bound"
                count += [fin.sum(), np.isinf(want).sum(), np.isnan(want).sum()]
    return count


# (q8, dh, ps, hq, hkv, rows, top, row_seq): single tokens over split and whole lists, chunks
# whose rows share pages (two rows a workgroup, four) and chunks whose rows do not
SEES = [(False, 128, 64, 8, 2, 2, 12, False), (True, 128, 64, 8, 2, 2, 12, False), (False, 256, 16, 4, 2, 3, 9, False), (True, 128, 16, 8, 1, 2, 3, False),
        (False, 128, 64, 16, 8, 130, 3, True), (False, 128, 16, 32, 8, 129, 4, True), (False, 256, 16, 16, 8, 130, 3, True), (True, 128, 16, 32, 8, 66, 2, True)]


def chunk_of(rng, q8, dh, ps, hq, hkv, rows, top, row_seq):
    seqs = 1 if row_seq else rows
    c = Cache(rng, seqs, top + 2 + -(-rows // ps), hkv, dh, ps, q8)
    span = c.max_pages * ps
    seq = [0] * rows if row_seq else list(range(rows))
    pos = [span - rows + r if row_seq else span - 1 - 5 * r for r in range(rows)]
    q = rng.standard_normal((rows, hq, dh)).astype(np.float32)
    proj = rng.standard_normal((rows, 2 * hq * dh)).astype(np.float32)
    sel = np.empty((rows, hkv, top), np.int32)
    for r in range(rows):
        for g in range(hkv):
            sel[r, g] = np.sort(np.concatenate([rng.permutation(top)[: top - 1], [pos[r] // ps]]))  # pages 0 .. top - 1, and the row's own
    return c, seq, pos, q, proj, sel


@pytest.mark.parametrize("q8,dh,ps,hq,hkv,rows,top,row_seq", SEES)
def test_an_infinite_key_gives_what_the_definition_gives(lib, q8, dh, ps, hq, hkv, rows, top, row_seq):
    """A key whose score is -inf has weight 0, one of +inf makes the result NaN: in
    one page of each sequence an infinite channel (Q8_0: a block of an infinite
    step), of either sign to the heads of a group."""
    rng = np.random.default_rng(dh + ps + rows + hq)
    c, seq, pos, q, proj, sel = chunk_of(rng, q8, dh, ps, hq, hkv, rows, top, row_seq)
    for s in range(c.seqs):
        at = c.table[s, 1]
        if q8:
            c.d[at, 0, :, 3, 1] = np.inf
            c.codes[at, 0, :, 3, 32:64] = rng.integers(1, 128, (c.hkv, 32))
        else:
            c.kv[at, 0, :, 3, 5], c.kv[at, 0, 0, 7, 9] = np.inf, -np.inf
    if q8:  # of one sign, so that the block's products have one
        sign = rng.integers(0, 2, q.shape[:2]) * 2 - 1
        q[..., 32:64] = np.abs(q[..., 32:64]) * sign[..., None]
        q[0, 0, 40] *= -1  # of both
    got, _ = run_attend(lib, c, hq, q, proj, seq, pos, sel, row_seq=row_seq)
    fin, inf, nan = check_ieee(c, hq, q, proj, seq, pos, sel, got)
    assert fin and not inf and (nan or rows == 2)  # the lists of two rows may miss the page


@pytest.mark.parametrize("q8,dh,ps,hq,hkv,rows,top,row_seq", SEES)
def test_an_infinite_value_gives_what_the_definition_gives(lib, q8, dh, ps, hq, hkv, rows, top, row_seq):
    """Values of both infinities: the channels that hold one are infinite, those that
    hold both NaN (Q8_0: and where a code of 0 meets an infinite step), the others
    finite."""
    rng = np.random.default_rng(1 + dh + ps + rows + hq)
    c, seq, pos, q, proj, sel = chunk_of(rng, q8, dh, ps, hq, hkv, rows, top, row_seq)
    for s in range(c.seqs):
        at = c.table[s, 1]
        if q8:
            c.d[at, 1, :, 3, 1] = c.d[at, 1, :, 9, 3] = np.inf
            c.codes[at, 1, :, 3, 40] = 0
        else:
            c.kv[at, 1, :, 3, 5], c.kv[at, 1, :, 4, 100], c.kv[at, 1, :, 6, 77] = np.inf, -np.inf, np.inf
            c.kv[at, 1, :, 11, 77], c.kv[at, 1, 0, 12, dh - 1] = -np.inf, np.nan
    got, _ = run_attend(lib, c, hq, q, proj, seq, pos, sel, row_seq=row_seq)
    fin, inf, nan = check_ieee(c, hq, q, proj, seq, pos, sel, got)
    assert fin and (inf and nan or rows == 2)


@pytest.mark.parametrize("q8,dh,ps,hq,hkv,rows,top,row_seq", SEES)
def test_keys_of_weight_zero(lib, q8, dh, ps, hq, hkv, rows, top, row_seq):
    """A page whose keys all score -inf beside others: it takes no part, also where
    a range of a list or a wave of a workgroup holds nothing else. Alone it leaves a
    softmax over nothing but -inf: NaN, unlike a list without a page, which gives 0."""
    rng = np.random.default_rng(2 + dh + ps + rows + hq)
    c, seq, pos, q, proj, sel = chunk_of(rng, q8, dh, ps, hq, hkv, rows, top, row_seq)
    q[..., :32] = np.abs(q[..., :32]) + np.float32(0.01)
    for s in range(c.seqs):
        at = c.table[s, 1]
        if q8:
            c.d[at, 0, :, :, 0] = np.inf
            c.codes[at, 0, :, :, :32] = -rng.integers(1, 128, (hkv, ps, 32))
        else:
            c.kv[at, 0, :, :, 7] = -np.inf
    sel[rows // 2] = -1
    sel[rows // 2, :, 0] = 1
    none = rows // 2 + 1 if rows > 2 else None
    if none:
        sel[none] = -1
    got, _ = run_attend(lib, c, hq, q, proj, seq, pos, sel, row_seq=row_seq)
    assert np.all(np.isnan(got[rows // 2]))
    keep = [r for r in range(rows) if r != none]
    if none:
        assert np.all(got[none] == 0)
    pick = lambda x: [x[r] for r in keep]  # noqa: E731
    fin, inf, nan = check_ieee(c, hq, q[keep], proj[keep], pick(seq), pick(pos), sel[keep], got[keep])
    assert fin and not inf and nan == hq * dh


@pytest.mark.parametrize("q8,dh,hq,hkv,row_seq,rows", [(False, 128, 8, 2, False, 3), (True, 128, 8, 2, False, 3), (False, 256, 4, 2, False, 3), (False, 128, 32, 8, True, 130)])
def test_a_cache_of_nans_but_for_what_is_seen(lib, q8, dh, hq, hkv, row_seq, rows):
    """Every value and step of the pool is NaN but the keys that some row sees."""
    rng = np.random.default_rng(dh + rows)
    ps, top = 16, 4
    c = Cache(rng, 1 if row_seq else rows, 20, hkv, dh, ps, q8, poison=True)
    seq = [0] * rows if row_seq else list(range(rows))
    pos = [20 * ps - rows - 3 + r if row_seq else 150 - 37 * r for r in range(rows)]
    sel = np.empty((rows, hkv, top), np.int32)
    clean = Cache(rng, c.seqs, 20, hkv, dh, ps, q8)
    for r in range(rows):
        own = pos[r] // ps
        sel[r] = [0, 2, own - 1, own]
        for lp in sel[r, 0]:
            at, n = c.table[seq[r], lp], min(ps, max(p for p, s in zip(pos, seq) if s == seq[r]) + 1 - lp * ps) if lp == own else ps
            if q8:
                c.d[at, :, :, :n] = clean.d[at, :, :, :n]
            else:
                c.kv[at, :, :, :n] = clean.kv[at, :, :, :n]
    q, proj = rng.standard_normal((rows, hq, dh)).astype(np.float32), rng.standard_normal((rows, 2 * hq * dh)).astype(np.float32)
    got, act = run_attend(lib, c, hq, q, proj, seq, pos, sel, row_seq=row_seq)
    check_attend(c, hq, q, proj, seq, pos, sel, got, act, rows=list(range(rows))[:: max(1, rows // 12)])
    assert np.all(np.isfinite(got))


# ---- selection by queries near the end of fp32's range ------------------------------------
def tiny_reference(q, codes, steps, table, seq, pos, ps, n_pool, top, sink, recent):
    """the selection's definition with a step q / 127 of any size: heads are brought to fp32's
    normal range by a power of two first, which changes no code, and the step is taken back in 64 bits"""
    rows, hq, _ = q.shape
    hkv = codes.shape[1]
    small = np.abs(q).max(-1) < 2.0 ** -80
    x = np.where(small[..., None], q.astype(np.float64) * 2.0 ** 64, q).astype(np.float32)
    k, d = quantize(x)
    d = d.astype(np.float64) * np.where(small, 2.0 ** -64, 1)
    split = np.concatenate([np.maximum(k, 0), np.maximum(-k, 0)], -1).reshape(rows, hkv, hq // hkv, -1)
    d = d.reshape(rows, hkv, -1)
    out = np.full((rows, hkv, top), -1, np.int32)
    for r in range(rows):
        vis = pos[r] // ps + 1
        page = table[seq[r], :vis]
        for g in range(hkv):
            score = ((codes[page, g].reshape(vis, -1).astype(np.int64) @ split[r, g].T).astype(np.float64) * d[r, g]).max(1) * steps[page, g].astype(np.float64)
            score[:sink] = score[vis - recent:] = np.inf
            take = np.sort(np.argsort(-score, kind="stable")[:top])
            out[r, g, : len(take)] = take
    return out


@pytest.mark.parametrize("hq,hkv,dh", [(8, 2, 128), (4, 1, 256), (2, 2, 128), (8, 1, 128)])
@pytest.mark.parametrize("pages", [40, 700])
@pytest.mark.parametrize("row_seq", [False, True])
def test_select_by_tiny_queries(lib, hq, hkv, dh, pages, row_seq):
    """Heads whose step's reciprocal passes fp32's range, heads of subnormals, zeros and
    ordinary heads: the codes and the order of the pages are the definition's. Every score
    of a tiny head has a sign of its own: bounds of either sign, some pages negative."""
    rng = np.random.default_rng(pages + hq)
    rows = 6
    codes, steps, q = select_inputs(rng, pages, hkv, hq, dh, rows)
    size = np.array([1e-36, 3e-37, 1e-38, 2e-40, 3e-43, 1.0])
    q = (q * size[:, None, None]).astype(np.float32)
    q[5, ::2] = (q[5, ::2] * np.float32(1e-39))
    q[1, 0] = 0
    table = np.stack([rng.permutation(pages) for _ in range(rows)]).astype(np.int32)
    seq = [0, 0, 0, 1, 1, 2] if row_seq else list(range(rows))
    pos = [pages * 16 - 6 + r for r in range(rows)]
    got = run_select(lib, q, codes, steps, table, seq, pos, 16, pages, 12, 1, 2, row_seq=row_seq)
    assert np.array_equal(got, tiny_reference(q, codes, steps, table, seq, pos, 16, pages, 12, 1, 2))


# ---- a few keys of nearly equal weight ------------------------------------------------------
@pytest.mark.parametrize("q8,dh,hq,hkv,rows,row_seq", [(False, 128, 4, 1, 1, False), (True, 128, 4, 1, 1, False), (True, 128, 8, 1, 1, False), (False, 256, 2, 1, 1, False),
                                                       (False, 128, 32, 8, 130, True), (False, 256, 16, 8, 130, True)])
def test_weights_close_to_the_largest_are_kept_to_fp32(lib, q8, dh, hq, hkv, rows, row_seq):
    """Two keys, values 1 and -1 in every channel, scores 0 and -x: the result is
    -tanh(x / 2), which the error of one weight makes up. x = scale q k is exact up to
    three roundings of 2^-24 of itself; the hardware's exponential is good to 1 ulp
    (2^-24 just below 1); two fp16 terms of a value in [4096, 8192) (times a step of a
    half: [2048, 4096)) leave 2^-24 of the largest, 11 bits and then 11 of a rest of at
    most half a step of the first; both products and their difference are exact. The result is
    off by half of that, so by 2^-24; total, division and a gate of 1 each round a result
    below 2^-15."""
    scale = float(np.float32(1 / np.sqrt(dh)))
    rng = np.random.default_rng(dh + rows + hq)
    c = Cache(rng, 1, 2, hkv, dh, 16, q8)
    x = rng.random((rows, hq)) * 2.0 ** -18 + 2.0 ** -23  # at most a half of 2^-16
    q = np.zeros((rows, hq, dh), np.float32)
    q[..., 3] = (x / scale).astype(np.float32)
    if q8:
        c.codes[:, 0], c.codes[:, 1, :, 0], c.codes[:, 1, :, 1], c.d[:] = 0, 1, -1, 1
        c.codes[:, 0, :, 1, 3] = -1
    else:
        c.kv[:, 0], c.kv[:, 1, :, 0], c.kv[:, 1, :, 1] = 0, 1, -1
        c.kv[:, 0, :, 1, 3] = -1
    proj = np.full((rows, 2 * hq * dh), 40, np.float32)  # sigmoid(40) rounds to 1
    got, _ = run_attend(lib, c, hq, q, proj, [0] * rows, [1] * rows, np.zeros((rows, hkv, 1), np.int32), row_seq=row_seq)
    want = np.tanh(scale * q[..., 3].astype(np.float64) / 2)
    d = np.abs(got.reshape(rows, hq, dh) - want[..., None])
    assert d.max() <= U + 2.0 ** -38, f"{d.max() / U:.3g} of half an fp32 step"


# ---- forms of single tokens, wide heads, workspaces -----------------------------------------
@pytest.mark.parametrize("q8,dh,ps,hq,hkv", [(False, 128, 64, 32, 8), (True, 128, 64, 32, 8), (False, 256, 64, 16, 4), (True, 128, 16, 7, 1), (False, 128, 256, 8, 2), (False, 256, 16, 3, 3),
                                             (True, 128, 256, 16, 2)])
@pytest.mark.parametrize("b", [1, 17])
def test_append_of_single_tokens_equals_oracle(lib, q8, dh, ps, hq, hkv, b):
    """A row of each sequence: first and last slots of pages, padding and positions past
    the table, the stored bytes, the rotated queries and the summaries."""
    rng = np.random.default_rng(ps + dh + b)
    c = Cache(rng, b, 5, hkv, dh, ps, q8)
    pos = [int(p) for p in rng.integers(0, 5 * ps, b)]
    if b > 1:
        pos[1], pos[2], pos[3], pos[4], pos[5] = 0, ps - 1, -1, 5 * ps, 3 * ps
    table = c.table.copy()
    if b > 1:
        table[6, pos[6] // ps], table[7, pos[7] // ps] = -1, c.n
    before = copy_of(c)
    ran = run_append(lib, rng, c, hq, list(range(b)), pos, table=table, row_seq=False, stride_more=1)
    check_append(before, c, hq, list(range(b)), pos, table, ran)


@pytest.mark.parametrize("q8,dh", [(False, 128), (True, 128), (False, 256)])
def test_append_over_a_cache_of_nans(lib, q8, dh):
    """What lies in and behind a page's other slots is overwritten or left, and does not
    reach the rows that are stored: a prompt from position 0 on, then tokens."""
    rng = np.random.default_rng(3)
    c = Cache(rng, 2, 6, 2, dh, 16, q8, poison=True)
    with np.errstate(invalid="ignore"):
        for seq, pos, row_seq in (([0] * 37 + [1] * 5, list(range(37)) + list(range(5)), True), ([0, 1], [37, 5], False)):
            before = copy_of(c)
            ran = run_append(lib, rng, c, 4, seq, pos, row_seq=row_seq)
            check_append(before, c, 4, seq, pos, c.table, ran)


@pytest.mark.parametrize("hq,hkv,dh", [(2, 2, 128), (4, 2, 128), (3, 1, 128), (8, 2, 128), (16, 2, 128), (5, 1, 128), (2, 2, 256), (4, 2, 256), (8, 2, 256), (16, 2, 256), (7, 1, 256)])
@pytest.mark.parametrize("pages", [33, 512, 513, 2100, 4097])
def test_select_of_single_tokens_of_every_group(lib, hq, hkv, dh, pages):
    """Each count of query heads per K/V head at both widths, in one launch (up to 512
    pages) and in two, rows that see some or all of their pages, a page in twenty gone."""
    rng = np.random.default_rng(hq * dh + pages)
    codes, steps, q = select_inputs(rng, 900, hkv, hq, dh, 3)
    table = rng.integers(0, 900, (3, pages)).astype(np.int32)
    table[rng.random(table.shape) < 0.05] = -1
    pos = [pages * 16 - 1, pages * 16 // 2, (pages - 1) * 16]
    got = run_select(lib, q, codes, steps, table, range(3), pos, 16, 900, 10, 1, 2, row_seq=False)
    assert np.array_equal(got, select_reference(q, codes, steps, table, range(3), pos, 16, 900, 10, 1, 2))


@pytest.mark.parametrize("hq,hkv", [(2, 2), (4, 2), (8, 2), (16, 2), (6, 1)])
@pytest.mark.parametrize("pages", [300, 500, 767, 1024, 1025])
def test_select_of_chunks_of_wide_heads(lib, hq, hkv, pages):
    """256-wide heads up to the most pages whose scores stay in shared memory (over 64 KB
    of it), and one more; rows of two sequences in one tile."""
    rng = np.random.default_rng(hq + pages)
    codes, steps, q = select_inputs(rng, 900, hkv, hq, 256, 11)
    table = rng.integers(0, 900, (2, pages)).astype(np.int32)
    seq, pos = [0] * 7 + [1] * 4, [pages * 16 - 7 + i for i in range(7)] + [pages * 8 + i for i in range(4)]
    got = run_select(lib, q, codes, steps, table, seq, pos, 16, 900, 30, 2, 1)
    assert np.array_equal(got, select_reference(q, codes, steps, table, seq, pos, 16, 900, 30, 2, 1))


GUARD = 4096


@pytest.mark.parametrize("hq,hkv,dh,ps,rows,pages,top,row_seq", [(8, 2, 128, 64, 1, 700, 20, False), (16, 2, 256, 16, 5, 513, 9, False), (8, 1, 128, 16, 9, 1025, 40, True),
                                                                 (8, 2, 128, 16, 3, 5000, 64, False), (8, 8, 128, 16, 2, 17000, 30, False)])
def test_select_stays_inside_its_workspace(lib, hq, hkv, dh, ps, rows, pages, top, row_seq):
    rng = np.random.default_rng(pages)
    codes, steps, q = select_inputs(rng, 300, hkv, hq, dh, rows)
    table = rng.integers(0, 300, (rows, pages)).astype(np.int32)
    c = Cache(rng, rows, 1, hkv, dh, ps)
    c.max_pages, c.n = pages, 300
    sums = np.zeros((300, c.sum_bytes), np.uint8)
    sums[:, : hkv * 2 * dh] = codes.reshape(300, -1).view(np.uint8)
    sums[:, hkv * 2 * dh: hkv * 2 * dh + 4 * hkv] = steps.view(np.uint8).reshape(300, -1)
    pos = [pages * ps - 1 - r for r in range(rows)]
    wb, d = lib.hero_attn_select_work_bytes(rows, hkv, pages), [dev(x) for x in (q, sums, table, np.array(pos, np.int32), np.arange(rows, dtype=np.int32))]
    work, sel = dev(np.full(wb + GUARD, 0xA5, np.uint8)), empty(rows * hkv * top * 4)
    args = sparse_args(c, hq, rows, ptr(d[3]), dev_seq=ptr(d[4]) if row_seq else None, q_rot=ptr(d[0]), table=ptr(d[2]), work=ptr(work), work_bytes=wb, summaries=ptr(d[1]),
                       selected=ptr(sel), top=top, sink=1, recent=2)
    check(lib.hero_attn_select_pages(args, stream()))
    assert np.all(host(work, np.uint8)[wb:] == 0xA5)


@pytest.mark.parametrize("q8,hq,hkv,dh,ps,rows,top,row_seq", [(False, 32, 8, 128, 64, 1, 32, False), (True, 32, 8, 128, 64, 16, 32, False), (False, 16, 4, 256, 64, 8, 48, False),
                                                              (True, 8, 1, 128, 16, 3, 4096, False), (False, 16, 8, 128, 16, 70, 2100, True), (False, 7, 1, 128, 48, 100, 7, True)])
def test_attend_stays_inside_its_workspace(lib, q8, hq, hkv, dh, ps, rows, top, row_seq):
    rng = np.random.default_rng(top)
    c = Cache(rng, 1 if row_seq else rows, 60, hkv, dh, ps, q8)
    pos = [60 * ps - 1 - r for r in range(rows)]
    sel = random_lists(rng, rows, hkv, top, [min(60, top)] * rows)
    wb = lib.hero_attn_sparse_work_bytes(rows, hq, hkv, dh, ps, top)
    assert wb > 0
    d = [dev(x) for x in (rng.standard_normal((rows, hq, dh)).astype(np.float32), rng.standard_normal((rows, 2 * hq * dh)).astype(np.float32), c.bytes(), c.table,
                          np.array(pos, np.int32), np.zeros(rows, np.int32), sel)]
    work, out = dev(np.full(wb + GUARD, 0xA5, np.uint8)), empty(rows * hq * dh * 4 + GUARD)
    args = sparse_args(c, hq, rows, ptr(d[4]), dev_seq=ptr(d[5]) if row_seq else None, q_rot=ptr(d[0]), proj=ptr(d[1]), stride=2 * hq * dh, scale=0.1, pages=ptr(d[2]), table=ptr(d[3]),
                       work=ptr(work), work_bytes=wb, selected=ptr(d[6]), top=top, out=ptr(out))
    check(lib.hero_attn_sparse_paged(args, stream()))
    assert np.all(host(work, np.uint8)[wb:] == 0xA5) and np.all(host(out, np.uint8)[rows * hq * dh * 4:] == 0)


@pytest.mark.parametrize("q8", [False, True])
def test_decoded_rows_with_row_seq_equal_those_without(lib, q8):
    """Tokens of many sequences, their sequences named: the same stored bytes and lists,
    and the attention of rows that share nothing in the kernels for chunks."""
    rng = np.random.default_rng(15)
    b, hq, hkv, ps, top = 130, 32, 8, 16, 4
    c = Cache(rng, b, 9, hkv, 128, ps, q8)
    pos = [int(p) for p in rng.integers(0, 9 * ps, b)]
    pools, sums = [], []
    for row_seq in (False, True):
        one = copy_of(c)
        ran = run_append(lib, np.random.default_rng(1), one, hq, list(range(b)), pos, row_seq=row_seq)
        pools.append(one.bytes())
        sums.append((ran[5], ran[7]))
    assert np.array_equal(*pools) and all(np.array_equal(x, y) for x, y in zip(*sums))
    codes, steps, q = select_inputs(rng, c.n, hkv, hq, 128, b)
    lists = [run_select(lib, q, codes, steps, c.table, range(b), pos, ps, c.n, top, 1, 2, row_seq=r) for r in (False, True)]
    assert np.array_equal(*lists)
    proj = rng.standard_normal((b, 2 * hq * 128)).astype(np.float32)
    for r in (False, True):
        got, act = run_attend(lib, c, hq, q, proj, range(b), pos, lists[0], row_seq=r)
        check_attend(c, hq, q, proj, range(b), pos, lists[0], got, act, rows=[0, 1, 2, 3, 64, 65, 128, 129])


@pytest.mark.parametrize("q8,dh,row_seq", [(False, 128, True), (True, 128, False), (False, 256, True), (False, 256, False)])
def test_append_and_attend_at_the_alignments_the_header_allows(lib, q8, dh, row_seq):
    """A projection and norm weights at 4 bytes past an even address, a rotation table at 8,
    pools, queries and outputs at 16: the results of the aligned calls."""
    rng = np.random.default_rng(19)
    hq, hkv, ps, rows, top = 4, 2, 16, 5, 3
    c = Cache(rng, 1 if row_seq else rows, 4, hkv, dh, ps, q8)
    kw, rope = hkv * dh, 4 * ps
    stride = 2 * hq * dh + 2 * kw + 1
    proj, g = rng.standard_normal(rows * stride).astype(np.float32), (1 + 0.1 * rng.standard_normal((2, dh))).astype(np.float32)
    cs, seq = oracle.rope_table(dh, 1e6, 32, rope), np.array([0] * rows if row_seq else range(rows), np.int32)
    pos = np.array([14 + r if row_seq else 13 * r for r in range(rows)], np.int32)
    sel = np.full((rows, hkv, top), -1, np.int32)
    for r in range(rows):
        sel[r, :, : pos[r] // ps + 1] = np.arange(pos[r] // ps + 1)[:top]
    got = []
    for off in (0, 1):
        def put(x, at):
            raw = np.ascontiguousarray(x).view(np.uint8).reshape(-1)
            t = dev(np.concatenate([np.zeros(at, np.uint8), raw]))
            return t, ptr(t) + at

        d = {"proj": put(proj, 4 * off), "gq": put(g[0], 4 * off), "gk": put(g[1], 4 * off), "cs": put(cs, 8 * off), "pages": put(c.bytes(), 16 * off), "table": put(c.table, 4 * off),
             "pos": put(pos, 4 * off), "seq": put(seq, 4 * off), "sums": put(np.zeros((c.n, c.sum_bytes), np.uint8), 16 * off), "q": put(np.zeros((rows, hq, dh), np.float32), 16 * off),
             "sel": put(sel, 4 * off), "out": put(np.zeros((rows, hq * dh), np.float32), 16 * off)}
        p = {k: v[1] for k, v in d.items()}
        work = empty(max(16, lib.hero_attn_sparse_work_bytes(rows, hq, hkv, dh, ps, top)))
        args = sparse_args(c, hq, rows, p["pos"], dev_seq=p["seq"] if row_seq else None, proj=p["proj"], stride=stride, gq=p["gq"], gk=p["gk"], cs=p["cs"], q_rot=p["q"], scale=0.1,
                           pages=p["pages"], table=p["table"], rope=rope, summaries=p["sums"], selected=p["sel"], top=top, out=p["out"], work=ptr(work), work_bytes=work.numel())
        check(lib.hero_kv_append_paged(args, stream()))
        check(lib.hero_attn_sparse_paged(args, stream()))
        got.append([host(d[k][0], np.uint8)[{"pages": 16, "sums": 16, "q": 16, "out": 16}[k] * off:] for k in ("pages", "sums", "q", "out")])
    for a, b in zip(*got):
        assert np.array_equal(a, b) and a.any()


@pytest.mark.parametrize("q8,dh,hq,hkv,rows", [(False, 128, 8, 2, 2), (True, 128, 8, 2, 2), (True, 128, 8, 1, 2), (False, 256, 8, 2, 2), (False, 128, 32, 8, 130), (False, 256, 16, 8, 130)])
def test_a_query_that_is_not_finite_stays_in_its_head(lib, q8, dh, hq, hkv, rows):
    """NaN, infinity and both signs of it in some heads: those are NaN (an infinite channel meets
    keys of both signs or of zero), the others as without them."""
    rng = np.random.default_rng(23)
    c = Cache(rng, 1, 20, hkv, dh, 16, q8)
    pos = [200 + r % 100 for r in range(rows)]
    q, proj = rng.standard_normal((rows, hq, dh)).astype(np.float32), rng.standard_normal((rows, 2 * hq * dh)).astype(np.float32)
    sel = random_lists(rng, rows, hkv, 4, [12] * rows)
    sel[:, :, 0] = 0
    bad = np.zeros((rows, hq), bool)
    for i, (r, h) in enumerate([(0, 1), (1, 0), (1, hq - 1), (rows - 1, 2)]):
        q[r, h, 3 * i] = (np.nan, np.inf, -np.inf, np.inf)[i]
        bad[r, h] = True
    clean = np.where(np.isfinite(q), q, 0).astype(np.float32)
    got, _ = run_attend(lib, c, hq, q, proj, [0] * rows, pos, sel, row_seq=True)
    want, _ = run_attend(lib, c, hq, clean, proj, [0] * rows, pos, sel, row_seq=True)
    x, y = got.reshape(rows, hq, dh), want.reshape(rows, hq, dh)
    assert np.all(np.isnan(x[bad])) and np.array_equal(bits(x[~bad]), bits(y[~bad]))


def test_captured_attention_over_infinities_replays_like_eager_calls(lib):
    """The rows that are formed again in plain fp32, in a captured graph, with eager calls in between."""
    import torch

    rng = np.random.default_rng(29)
    hq, hkv, dh, ps, top, rows = 8, 2, 128, 64, 12, 2
    c, seq, pos, q, proj, sel = chunk_of(rng, False, dh, ps, hq, hkv, rows, top, False)
    c.kv[c.table[0, 1], 1, :, 3, 5], c.kv[c.table[1, 2], 0, :, 4, 9] = np.inf, -np.inf
    want, _ = run_attend(lib, c, hq, q, proj, seq, pos, sel, row_seq=False)
    wb = lib.hero_attn_sparse_work_bytes(rows, hq, hkv, dh, ps, top)
    d = [dev(x) for x in (q, proj, c.bytes(), c.table, np.array(pos, np.int32), sel)]
    work, out = empty(wb), empty(rows * hq * dh * 4)
    args = sparse_args(c, hq, rows, ptr(d[4]), q_rot=ptr(d[0]), proj=ptr(d[1]), stride=2 * hq * dh, scale=float(np.float32(1 / np.sqrt(dh))), pages=ptr(d[2]), table=ptr(d[3]),
                       work=ptr(work), work_bytes=wb, selected=ptr(d[5]), top=top, out=ptr(out))
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        check(lib.hero_attn_sparse_paged(args, side.cuda_stream))
    for _ in range(3):
        out.zero_()
        graph.replay()
        assert np.array_equal(bits(host(out, np.float32)), bits(want.reshape(-1)))
        again, _ = run_attend(lib, c, hq, q, proj, seq, pos, sel, row_seq=False)
        assert np.array_equal(bits(again), bits(want))
    assert np.isinf(want).any() or np.isnan(want).any()
