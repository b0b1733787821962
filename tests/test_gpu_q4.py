"""The 4-bit paged cache: append (norms, rotary positions of several axes, 4-bit
blocks), read and attention. Stored bytes are compared for equality with the
definition in 64 bits; the attention with a 64-bit softmax over the stored values,
under a bound computed from the data."""
import ctypes

import numpy as np
import pytest

import oracle
from gpu_util import act_to_blocks, bits, check, dev, empty, host, ptr, stream, ulp_diff

pytestmark = pytest.mark.gpu

EPS = np.float32(1e-6)


@pytest.fixture(scope="module")
def lib():
    from hero_amd._lib import lib as _lib

    import torch

    assert torch.cuda.is_available(), "GPU tests need a GPU"
    return _lib


# ---- the pages, on the host ---------------------------------------------------------------
def places(dh, what):
    """[16 positions][dh]: the byte of a code in its record, whether it is the upper half, its step's index"""
    i, ch = np.meshgrid(np.arange(16), np.arange(dh), indexing="ij")
    h, r = ch // 128, ch % 128
    if what == 0:
        a, b, j = r // 32, r // 8 % 4, r % 8
        field, word, step = j // 2 + 4 * (j % 2), ((h * 16 + i) * 4 + b) * 4 + a, i * (dh // 32) + ch // 32
    else:
        field, word, step = r // 16, ((h * 4 + i // 4) * 16 + r % 16) * 4 + i % 4, (i // 4 * (dh // 32) + ch // 32) * 4 + i % 4
    return 4 * word + field // 2, field % 2, step


def round8(m):
    """m / -8 as fp16, its magnitude rounded to 8 significant bits; 0 has no sign"""
    with np.errstate(over="ignore"):
        h = (m.astype(np.float32) * np.float32(-0.125)).astype(np.float16).view(np.uint16).astype(np.int32)
    size = ((h & 0x7FFF) + 4) & 0x7FF8
    return np.where(size > 0, size | (h & 0x8000), 0).astype(np.uint16).view(np.float16)


def blocks(x):
    """fp32 [..., dh] -> codes -8 .. 7 [..., dh], fp16 steps [..., dh / 32]"""
    x = np.clip(np.where(np.isnan(x), 0, x), -65280, 65280).reshape(x.shape[:-1] + (-1, 32))
    hi, lo = x.max(-1), x.min(-1)
    d = round8(np.where(hi >= -lo, hi, lo))
    step = d.astype(np.float64)[..., None]
    q = np.where(step != 0, np.round(x.astype(np.float64) / np.where(step != 0, step, 1)), 0)
    return np.clip(q, -8, 7).reshape(x.shape[:-2] + (-1,)).astype(np.int64), d


class Pool:
    """A 4-bit pool in host memory: random codes and steps, a shuffled page table."""

    def __init__(self, rng, seqs, max_pages, hkv, dh=128, ps=64, spare=3, poison=False):
        self.seqs, self.max_pages, self.hkv, self.dh, self.ps = seqs, max_pages, hkv, dh, ps
        self.n = seqs * max_pages + spare
        self.table = rng.permutation(self.n)[: seqs * max_pages].astype(np.int32).reshape(seqs, max_pages)
        self.rec = rng.integers(0, 256, (self.n, 2, hkv, ps // 16, 9 * dh)).astype(np.uint8)
        d = round8(rng.uniform(1.6, 2.6, self.rec.shape[:-1] + (dh // 2,)) * rng.choice([-1, 1], self.rec.shape[:-1] + (dh // 2,)))
        if poison:
            d[:] = np.nan
        self.rec[..., 8 * dh:] = d.view(np.uint8)
        self.at = [places(dh, w) for w in (0, 1)]

    def values(self, page, what):
        """[hkv][ps][dh] float64"""
        byte, up, step = self.at[what]
        r = self.rec[page, what]
        codes = (r[..., byte] >> (4 * up)) & 15
        d = np.ascontiguousarray(r[..., 8 * self.dh:]).view(np.float16)[..., step]
        return ((codes.astype(np.int64) - 8) * d.astype(np.float64)).reshape(self.hkv, self.ps, self.dh)

    def store(self, page, what, slot, codes, d):
        """codes [hkv][dh], d [hkv][dh / 32]"""
        byte, up, step = (t[slot % 16] for t in self.at[what])
        r = self.rec[page, what, :, slot // 16]
        for u in (0, 1):
            sel = np.flatnonzero(up == u)
            r[:, byte[sel]] = (r[:, byte[sel]] & (0xF0, 0x0F)[u]) | ((codes[:, sel] + 8) << (4 * u)).astype(np.uint8)
        first = step[::32]
        r[:, 8 * self.dh:].view(np.uint8)[:, 2 * first] = (d.view(np.uint16) & 255).astype(np.uint8)
        r[:, 8 * self.dh:].view(np.uint8)[:, 2 * first + 1] = (d.view(np.uint16) >> 8).astype(np.uint8)

    def sequence(self, seq, n, what):
        """the first n positions of a sequence [hkv][n][dh] float64; NaN where a page holds nothing"""
        out = np.full((self.hkv, -(-n // self.ps) * self.ps, self.dh), np.nan)
        for lp in range(-(-n // self.ps)):
            if 0 <= self.table[seq, lp] < self.n:
                out[:, lp * self.ps:(lp + 1) * self.ps] = self.values(self.table[seq, lp], what)
        return out[:, :n]


def q4_args(c, hq, rows, pos, dev_seq=None, **f):
    from hero_amd._lib import AttnDecodeArgs, AttnQ4Args

    dh, kw = c.dh, c.hkv * c.dh
    f = {"proj": None, "stride": 2 * hq * dh + 2 * kw, "k_off": 2 * hq * dh, "v_off": 2 * hq * dh + kw, "gq": None, "gk": None, "cs": None, "q_rot": None,
         "scale": 1.0, "window": 0, "act": None, "out": None, "pages": None, "table": None, "work": None, "work_bytes": 0, "rope": 1, "sinks": 0,
         "rope_pos": None, "axes": 1, "plane_axis": (), "pool_pages": c.n, **f}
    a = AttnDecodeArgs(f["proj"], f["stride"], f["k_off"], f["v_off"], f["gq"], f["gk"], EPS, f["cs"], None, None, 0, pos, None, f["q_rot"], f["scale"], f["window"],
                       f["act"], f["out"], rows, hq, c.hkv, dh)
    return AttnQ4Args(a, f["pages"], f["pool_pages"], f["table"], c.ps, c.max_pages, dev_seq, c.seqs, f["sinks"], f["rope"], f["rope_pos"], f["axes"],
                      (ctypes.c_uint8 * 128)(*f["plane_axis"]), f["work"], f["work_bytes"])


# ---- append -------------------------------------------------------------------------------
def rotated64(x, gamma, cs):
    """x [heads][dh] -> norm and rotation in 64 bits, rounded to fp32; cs [dh / 2][2]"""
    x = x.astype(np.float64)
    x = gamma.astype(np.float64) * x / np.sqrt((x * x).mean(-1, keepdims=True) + float(EPS))
    lo, hi = np.split(x, 2, -1)
    c, s = cs[:, 0].astype(np.float64), cs[:, 1].astype(np.float64)
    return np.concatenate([lo * c - hi * s, hi * c + lo * s], -1).astype(np.float32)


def run_append(lib, rng, c, hq, seq, pos, proj=None, row_seq=True, stride_more=0, rope=200, rope_pos=None, plane_axis=(), gamma=None):
    """appends rows to c on the device and on the host, and compares the whole pool and the queries"""
    rows, dh, kw = len(pos), c.dh, c.hkv * c.dh
    stride = 2 * hq * dh + 2 * kw + stride_more
    if proj is None:
        proj = rng.standard_normal((rows, stride)).astype(np.float32)
    gq, gk = ((1 + 0.1 * rng.standard_normal(dh)).astype(np.float32) for _ in range(2))
    gk = gk if gamma is None else gamma
    angle = np.arange(rope)[:, None] * 1e4 ** (-np.arange(dh // 2) / (dh // 2))
    cs = np.stack([np.cos(angle), np.sin(angle)], -1).astype(np.float32)
    pos, seq = np.asarray(pos, np.int32), np.asarray(seq, np.int32)
    d = {k: dev(v) for k, v in dict(proj=proj, gq=gq, gk=gk, cs=cs, pages=c.rec, table=c.table, pos=pos, seq=seq).items()}
    q0 = rng.standard_normal((rows, hq, dh)).astype(np.float32)
    d_q = dev(q0)
    axes = 1 if rope_pos is None else rope_pos.shape[0]
    d_rp = None if rope_pos is None else dev(rope_pos.astype(np.int32))
    args = q4_args(c, hq, rows, ptr(d["pos"]), ptr(d["seq"]) if row_seq else None, proj=ptr(d["proj"]), stride=stride, gq=ptr(d["gq"]), gk=ptr(d["gk"]), cs=ptr(d["cs"]),
                   q_rot=ptr(d_q), pages=ptr(d["pages"]), table=ptr(d["table"]), rope=rope, rope_pos=None if d_rp is None else ptr(d_rp), axes=axes, plane_axis=plane_axis)
    check(lib.hero_kv_append_q4(args, stream()))
    got_q, got = host(d_q, np.float32, q0.shape), host(d["pages"], np.uint8, c.rec.shape)
    axis = np.array(list(plane_axis) or [0] * (dh // 2))
    left_out = 0
    for r in range(rows):
        at = np.full(1, pos[r]) if rope_pos is None else rope_pos[:, r]
        if not (0 <= pos[r] < c.max_pages * c.ps and 0 <= seq[r] < c.seqs and np.all((at >= 0) & (at < rope))):
            assert np.array_equal(got_q[r], q0[r]), f"row {r} is left out"
            left_out += 1
            continue
        turn = cs[at[axis], np.arange(dh // 2)]
        want = rotated64(proj[r, : 2 * hq * dh].reshape(hq, 2, dh)[:, 0], gq, turn)
        fine = np.isfinite(want)
        # both round a 64-bit value once: they differ only where those lie on two sides of a tie
        assert ulp_diff(got_q[r][fine], want[fine]).max(initial=0) <= 1 and np.mean(bits(got_q[r]) != bits(want)) <= (0.01 if fine.all() else 1), f"row {r}: q"
        page = c.table[seq[r], pos[r] // c.ps]
        if 0 <= page < c.n:
            c.store(page, 0, pos[r] % c.ps, *blocks(rotated64(proj[r, 2 * hq * dh:2 * hq * dh + kw].reshape(c.hkv, dh), gk, turn)))
            c.store(page, 1, pos[r] % c.ps, *blocks(proj[r, 2 * hq * dh + kw:2 * hq * dh + 2 * kw].reshape(c.hkv, dh)))
    assert np.array_equal(got, c.rec), "the pool: appended rows as defined, every other byte as it was"
    return left_out


@pytest.mark.parametrize("dh,ps,hq,hkv,axes", [(128, 16, 8, 2, 1), (128, 64, 6, 2, 3), (128, 256, 8, 1, 2), (256, 64, 8, 4, 3), (256, 16, 3, 3, 1), (128, 48, 4, 4, 4), (256, 32, 7, 1, 4)])
def test_append_of_ragged_rows(lib, dh, ps, hq, hkv, axes):
    """Chunks of several sequences in one call, starting and ending inside pages, a
    single row, padding rows between and behind, sequences and positions out of range,
    rotary positions past the table, pages that hold nothing."""
    rng = np.random.default_rng(ps + dh + hq)
    c = Pool(rng, 5, -(-150 // ps) + 1, hkv, dh, ps)
    span = c.max_pages * ps
    c.table[0, 0] = -1
    seq, pos = [], []
    for s, (first, n) in enumerate([(0, ps + 3), (ps - 1, 2), (span // 3, 1), (0, 0), (span - 5, 5)]):
        seq += [s] * n
        pos += list(range(first, first + n))
        if s == 1:
            seq, pos = seq + [2, 7, -1], pos + [-1, 3, 4]
    seq, pos = seq + [4, 0, 0], pos + [span, -5, -1]
    c.table[4, 0] = c.n
    rope_pos = None if axes == 1 else rng.integers(0, 200, (axes, len(pos)))
    if axes > 1:
        rope_pos[axes - 1, 2], rope_pos[0, 4] = 200, -1
    left = run_append(lib, rng, c, hq, seq, pos, stride_more=3, rope=200 if axes > 1 else span, rope_pos=rope_pos,
                      plane_axis=() if axes == 1 else rng.integers(0, axes, dh // 2).tolist())
    assert left == (6 if axes == 1 else 8)


def test_append_without_row_seq_and_in_any_order(lib):
    rng = np.random.default_rng(3)
    run_append(lib, rng, Pool(rng, 9, 2, 2), 4, list(range(9)), [0, 127, 64, 5, 63, -1, 15, 16, 128], row_seq=False)
    order = rng.permutation(60)
    run_append(lib, rng, Pool(rng, 2, 1, 2), 4, (order % 2).tolist(), (order // 2).tolist())
    run_append(lib, rng, Pool(rng, 1, 1, 1), 1, [0], [0])


def test_append_of_thousands_of_rows(lib):
    rng = np.random.default_rng(61)
    c = Pool(rng, 2, 20, 1)
    run_append(lib, rng, c, 1, [0] * 1200 + [1] * 900, list(range(63, 1263)) + list(range(900)), rope=1300)


@pytest.mark.parametrize("hq,hkv,dh", [(9, 3, 128), (5, 5, 256), (48, 6, 128)])
def test_append_of_many_heads(lib, hq, hkv, dh):
    rng = np.random.default_rng(hq)
    rows = 25000 // (hq + 2 * hkv) + 5
    c = Pool(rng, 3, -(-rows // 64) + 1, hkv, dh)
    c.table[1, 0] = -1
    rows -= rows % 3  # (every row a place of its own)
    seq, pos = np.arange(rows) * 3 // rows, np.arange(rows) % (rows // 3) + 10
    pos[rng.integers(0, rows, 20)] = -1
    kw, stride = hkv * dh, 2 * hq * dh + 2 * hkv * dh + 5
    proj = rng.standard_normal((rows, stride)).astype(np.float32)
    proj[::7, -2 * kw:] = np.round(proj[::7, -2 * kw:] * 4)  # ties and blocks of equal magnitudes
    proj[3, -kw - 5 + 9], proj[5, -kw - 5 + 3], proj[6, 2 * hq * dh + 1] = np.nan, np.inf, 1e30
    run_append(lib, rng, c, hq, seq, pos, proj=proj, stride_more=5, rope_pos=rng.integers(0, 200, (2, rows)), plane_axis=rng.integers(0, 2, dh // 2).tolist())


def test_append_blocks_at_borders(lib):
    """Values: blocks of zeros, subnormal steps, exact ties, equal magnitudes of both signs, the
    largest that the format holds, infinities and NaN. Keys: a weight of 0, a row of zeros, non-finite rows."""
    rng = np.random.default_rng(8)
    hq = hkv = 2
    rows = 40
    c = Pool(rng, 1, 1, hkv)
    proj = rng.standard_normal((rows, 2 * hq * 128 + 2 * hkv * 128)).astype(np.float32)
    v = proj[:, 2 * hq * 128 + hkv * 128:].reshape(rows, -1, 32)
    v[0] = 0
    for r in range(1, 12):
        v[r] *= np.float32(2.0 ** (-26 + r))  # steps from 0 up through the multiples of 2^-21
    v[12, :, 0], v[12, :, 1] = 8, -8          # of equal magnitudes the positive one counts
    v[13] = np.round(v[13] * 4) / 2           # multiples of a half ...
    v[13, :, 5] = -8                          # ... of a step of 1: ties
    v[14] = np.round(v[14] * 4) / 2
    v[14, :, 5] = 8                           # ... of -1
    v[15, :, 3], v[16, :, 3], v[17, :, 3] = 65280, -70000, 3e38
    v[18, :, 4], v[19, :, 4], v[20, :, 4] = np.inf, -np.inf, np.nan
    v[21] = np.nan
    v[22] = np.float32(1e-45)
    for r in range(23, 30):  # steps of many mantissas, values next to the borders between codes
        d = round8(np.array([r * 1.37]))[0].astype(np.float32)
        k = rng.integers(-8, 7, v[r].shape) + np.float32(0.5)
        v[r] = np.nextafter((k * d).astype(np.float32), np.float32(rng.choice([-1e9, 1e9])))
        v[r, :, 7] = -8 * d
    k = proj[:, 2 * hq * 128: 2 * hq * 128 + hkv * 128]
    k[30], k[31, 5], k[32, 6], k[33] = 0, np.inf, np.nan, np.float32(1e-30)
    k[34] = np.float32(1e30)
    gamma = (1 + 0.1 * rng.standard_normal(128)).astype(np.float32)
    gamma[5], gamma[70] = 0, 1e5
    with np.errstate(invalid="ignore", over="ignore"):
        run_append(lib, rng, c, hq, [0] * rows, list(range(rows)), proj=proj, gamma=gamma)


# ---- read ---------------------------------------------------------------------------------
@pytest.mark.parametrize("f16", [0, 1])
@pytest.mark.parametrize("dh,ps,hkv", [(128, 64, 2), (256, 16, 3), (128, 48, 1)])
def test_read_returns_what_is_stored(lib, dh, ps, hkv, f16):
    from hero_amd._lib import KvReadArgs

    rng = np.random.default_rng(ps + hkv)
    c = Pool(rng, 3, 6, hkv, dh, ps)
    c.table[1, 2] = c.n
    rows = 77
    seq, pos = rng.integers(0, 3, rows).astype(np.int32), rng.integers(0, 6 * ps, rows).astype(np.int32)
    pos[5], seq[9], pos[11], seq[12], pos[12] = -1, 3, 6 * ps, 1, 2 * ps
    seq[20], pos[20] = seq[21], pos[21]
    t = np.float16 if f16 else np.float32
    d = [dev(x) for x in (c.rec, c.table, pos, seq)]
    for outs in (3, 1, 2):
        fill = rng.standard_normal((2, rows, hkv * dh)).astype(t)
        want, d_out = fill.copy(), [dev(x) for x in fill]
        for r in range(rows):
            if 0 <= pos[r] < 6 * ps and 0 <= seq[r] < 3 and c.table[seq[r], pos[r] // ps] < c.n:
                for w in (0, 1):
                    if outs >> w & 1:
                        want[w, r] = c.values(c.table[seq[r], pos[r] // ps], w)[:, pos[r] % ps].reshape(-1).astype(t)
        at = [ptr(x) if outs >> i & 1 else None for i, x in enumerate(d_out)]
        check(lib.hero_kv_read_q4(KvReadArgs(ptr(d[0]), ptr(d[1]), ps, 6, 0, c.n, None, ptr(d[2]), ptr(d[3]), rows, 3, hkv, dh, f16, *at, None, None), stream()))
        for w in (0, 1):
            assert np.array_equal(host(d_out[w], t, (rows, hkv * dh)), want[w]), f"output {w} of {outs}"


# ---- attention ----------------------------------------------------------------------------
def attend64(c, hq, q, gate, seq, pos, scale, window, sinks):
    """(outputs, bound, largest score) in 64 bits; rows that are left out: NaN.

    The bound: a score is a sum of dh products of a query kept to 2^-23 of its head's largest channel, formed in
    fp32: each product and addition is off by 2^-24 of the sum of magnitudes at most, (dh + 4) of them; a further 2^-22
    of the score for its scaling and the difference from the maximum. A weight is off by that (as exp' = exp)
    and 2^-22; the sums over n keys by (n / 32 + 40) 2^-24 (32 keys a product, 40 joins), the gate and
    division by 2^-21. Doubled: numerator and total both carry the weights' errors."""
    rows, dh, grp = len(pos), c.dh, hq // c.hkv
    out, bound = np.full((rows, hq, dh), np.nan), np.zeros((rows, hq, dh))
    cache, largest = {}, 0.0
    for r in range(rows):
        if not (0 <= pos[r] < c.max_pages * c.ps and 0 <= seq[r] < c.seqs):
            continue
        if seq[r] not in cache:
            n = max(int(p) for p, s in zip(pos, seq) if s == seq[r] and p < c.max_pages * c.ps) + 1
            cache[seq[r]] = [c.sequence(seq[r], n, w) for w in (0, 1)]
        k, v = (x[:, : pos[r] + 1] for x in cache[seq[r]])
        j = np.arange(pos[r] + 1)
        ok = ~np.isnan(k[0, :, 0])
        if window:
            ok &= (j > pos[r] - window) | (j < sinks)
        k, v = k[:, ok], v[:, ok]
        g = 1 / (1 + np.exp(-gate[r].astype(np.float64)))
        if not ok.any():
            out[r] = 0
            continue
        for h in range(hq):
            x = q[r, h].astype(np.float64)
            s = k[h // grp] @ x * scale
            mags = (np.abs(k[h // grp]) @ np.abs(x)) * scale
            largest = max(largest, np.abs(s).max())
            off = (dh + 4) * 2.0 ** -24 * mags + 2.0 ** -23 * np.abs(x).max() * np.abs(k[h // grp]).sum(1) * scale + 2.0 ** -22 * (np.abs(s) + np.abs(s).max())
            w = np.exp(s - s.max())
            w /= w.sum()
            o = w @ v[h // grp]
            rel = (w * off)[:, None] + w[:, None] * (2.0 ** -22 + (len(w) / 32 + 40) * 2.0 ** -24)
            out[r, h] = o * g[h]
            bound[r, h] = (2 * ((rel * np.abs(v[h // grp])).sum(0) + rel.sum() * np.abs(o)) + np.abs(o) * 2.0 ** -21 + 2.0 ** -38 * len(w) * np.abs(v[h // grp]).max()) * g[h]
    return out, bound, largest


def run_attend(lib, rng, c, hq, seq, pos, window=0, sinks=0, row_seq=True, q=None, scale=None, act=True, work_more=0, pool_offset=0):
    rows, dh = len(pos), c.dh
    scale = 1 / np.sqrt(dh) if scale is None else scale
    if q is None:
        q = rng.standard_normal((rows, hq, dh)).astype(np.float32)
    stride = 2 * hq * dh + 5
    proj = rng.standard_normal((rows, stride)).astype(np.float32)
    gate = proj[:, : 2 * hq * dh].reshape(rows, hq, 2, dh)[:, :, 1]
    pos, seq = np.asarray(pos, np.int32), np.asarray(seq, np.int32)
    d = {k: dev(v) for k, v in dict(q=q, proj=proj, pages=c.rec, table=c.table, pos=pos, seq=seq).items()}
    fill = rng.standard_normal((rows, hq * dh)).astype(np.float32)
    out, d_act = dev(fill), empty(lib.hero_q8_0_act_bytes(rows, hq * dh))
    wb = lib.hero_attn_q4_work_bytes(rows, hq, c.hkv, dh, c.max_pages * c.ps, window, sinks)
    work = dev(np.full(max(wb, 16) + work_more, 0xFF, np.uint8))
    args = q4_args(c, hq, rows, ptr(d["pos"]), ptr(d["seq"]) if row_seq else None, proj=ptr(d["proj"]), stride=stride, q_rot=ptr(d["q"]), scale=scale, window=window, sinks=sinks,
                   act=ptr(d_act) if act else None, out=ptr(out), pages=ptr(d["pages"]), table=ptr(d["table"]), work=ptr(work) if wb else None, work_bytes=wb)
    check(lib.hero_attn_q4(args, stream()))
    got = host(out, np.float32, (rows, hq, dh))
    live = np.array([0 <= p < c.max_pages * c.ps and 0 <= s < c.seqs for p, s in zip(pos, seq)])
    assert np.array_equal(got[~live], fill.reshape(got.shape)[~live]), "left-out rows stay as they were"
    if act and live.any() and np.isfinite(got[live]).all():
        a = act_to_blocks(host(d_act, np.uint8), rows, hq * dh)
        want = oracle.quantize_row_q8_0(got.reshape(rows, -1)[live].reshape(-1)).reshape(-1)
        assert np.array_equal(a[live].reshape(-1), want), "act_out is out_f32 quantized"
    want, bound, largest = attend64(c, hq, q, gate, seq, pos, scale, window, sinks)
    return got[live], want[live], bound[live], largest


def compare(got, want, bound, largest):
    assert np.all(np.abs(got - want) <= bound), f"off by {np.max(np.abs(got - want) / np.maximum(bound, 1e-300)):.3g} of the bound"
    # the bound adds every rounding up; they are independent. A score is rounded about four times, 2^-24 of its magnitude each: weights
    # are off by 2^-22 of the largest score (random rows: ~8, so 2^-19; scores that rise to 80 along the context: ten times that)
    assert np.linalg.norm(got - want) <= 2.0 ** -22 * max(8, largest) * np.linalg.norm(want)


GEOMETRY = [(32, 8, 128, 64), (8, 2, 128, 16), (16, 2, 128, 48), (6, 2, 128, 32), (5, 1, 128, 256), (3, 3, 128, 64), (14, 2, 128, 64), (12, 2, 128, 16), (16, 4, 256, 64), (6, 1, 256, 16),
            (2, 2, 256, 48), (4, 2, 256, 128)]


@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (40, 0), (100, 4), (33, 70), (64, 16)])
@pytest.mark.parametrize("hq,hkv,dh,ps", GEOMETRY)
def test_tokens_of_many_sequences(lib, hq, hkv, dh, ps, window, sinks):
    """A row per sequence: lengths of 1, around records and pages, some hundreds; one left out."""
    rng = np.random.default_rng(hq + dh + ps + window)
    lengths = [1, 2, 16, 17, 31, 32, 33, ps, ps + 1, 101, 300]
    c = Pool(rng, len(lengths) + 1, -(-300 // ps), hkv, dh, ps)
    compare(*run_attend(lib, rng, c, hq, range(len(lengths) + 1), [n - 1 for n in lengths] + [-1], window, sinks, row_seq=False))


@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 1), (50, 4), (20, 100)])
@pytest.mark.parametrize("hq,hkv,dh,ps", GEOMETRY)
def test_chunks_and_tokens_in_one_call(lib, hq, hkv, dh, ps, window, sinks):
    """Chunks that start at 0 and inside pages, single tokens between them, padding, rows out of order."""
    rng = np.random.default_rng(hq * dh + ps + window)
    c = Pool(rng, 6, -(-260 // ps), hkv, dh, ps)
    seq, pos = [], []
    for s, (first, n) in enumerate([(0, 37), (100, 1), (201, 50), (15, 2), (0, 1)]):
        seq += [s] * n
        pos += list(range(first, first + n))
        if s == 2:
            seq, pos = seq + [3, 9], pos + [-1, 4]
    seq, pos = seq + [5] * 5 + [0] * 3, pos + [90, 3, 57, 12, 200] + [-1] * 3
    compare(*run_attend(lib, rng, c, hq, seq, pos, window, sinks))


@pytest.mark.parametrize("hq,hkv,dh,rows,first,window,sinks,row_seq", [
    (32, 8, 128, 1, 5000, 0, 0, False), (8, 1, 128, 2, 9001, 0, 0, False), (16, 4, 256, 1, 3000, 0, 0, False), (8, 8, 128, 3, 4000, 2500, 5, False),
    (32, 8, 128, 70, 2000, 0, 0, True), (16, 2, 128, 33, 3000, 1000, 17, True), (8, 2, 256, 40, 1500, 0, 0, True), (4, 4, 128, 300, 700, 64, 4, True), (8, 2, 128, 1, 4500, 0, 0, True)])
def test_long_rows_split_over_workgroups(lib, hq, hkv, dh, rows, first, window, sinks, row_seq):
    rng = np.random.default_rng(rows + first)
    seqs = 1 if row_seq else rows
    c = Pool(rng, seqs, -(-(first + rows) // 64), hkv, dh)
    pos = list(range(first, first + rows)) if row_seq else [first - 900 * i for i in range(rows)]
    compare(*run_attend(lib, rng, c, hq, [0] * rows if row_seq else range(rows), pos, window, sinks, row_seq, work_more=64))


@pytest.mark.parametrize("window,sinks", [(0, 0), (70, 5)])
@pytest.mark.parametrize("hq,hkv,dh", [(32, 8, 128), (8, 1, 128), (4, 4, 128), (6, 2, 128), (16, 4, 256)])
def test_runs_of_every_length_in_one_call(lib, hq, hkv, dh, window, sinks):
    """Single tokens and runs of a few rows (drafts) of many sequences in any order, chunks that begin and end at any row
    of a group of columns, padding between some of them, the same sequence twice."""
    rng = np.random.default_rng(hq + window)
    few = 16 // (hq // hkv)
    c = Pool(rng, 30, 5, hkv, dh)
    seq, pos = [], []
    lengths = [1, 1, few, few + 1, 2, 40, 1, 37, few - 1, 1, 64, few + 2, 1, 1, 3, 61, few, few, 1]
    for i, n in enumerate(lengths):
        n = max(1, n)
        s = int(rng.permutation(30)[0]) if i in (4, 9) else i
        first = int(rng.integers(0, 320 - n))
        seq += [s] * n
        pos += list(range(first, first + n))
        if i in (2, 7, 8):
            seq, pos = seq + [s], pos + [-1]
    compare(*run_attend(lib, rng, c, hq, seq, pos, window, sinks, work_more=64))
    order = rng.permutation(30)[: 23]
    compare(*run_attend(lib, rng, c, hq, order.tolist(), rng.integers(0, 320, 23).tolist(), window, sinks))
    compare(*run_attend(lib, rng, c, hq, order[: few].tolist(), rng.integers(0, 320, few).tolist(), window, sinks))
    compare(*run_attend(lib, rng, c, hq, [order[0]] * few, (np.arange(few) + 250).tolist(), window, sinks))


@pytest.mark.parametrize("hq,hkv,dh,rows", [(8, 2, 128, 20), (4, 1, 256, 9), (8, 1, 128, 2), (4, 4, 128, 100)])
def test_long_runs_and_single_tokens_split_over_workgroups(lib, hq, hkv, dh, rows):
    """rows of several sequences with contexts of thousands: the ranges of both kinds of run are joined alike"""
    rng = np.random.default_rng(rows)
    c = Pool(rng, 3, 40, hkv, dh)
    half = rows // 2
    seq = [0] + [1] * (rows - half - 1) + [2] * half
    pos = [2500] + list(range(1800, 1800 + rows - half - 1)) + list(range(2000, 2000 + half))
    compare(*run_attend(lib, rng, c, hq, seq, pos, work_more=64))


@pytest.mark.parametrize("hkv,dh,rows,first,row_seq", [(256, 128, 17, 9000, True), (128, 256, 17, 9000, True), (768, 128, 1, 5000, False), (160, 128, 17, 2100, True)])
def test_long_ranges(lib, hkv, dh, rows, first, row_seq):
    """So many heads that thousands of keys are left to a workgroup: compared for some of the heads. Pages that a
    sequence has more than once."""
    rng = np.random.default_rng(hkv + dh)
    c = Pool(rng, 1, 20, hkv, dh)
    c.max_pages = -(-(first + rows) // 64)
    c.table = rng.integers(0, c.n, (1, c.max_pages)).astype(np.int32)
    pos, seq = np.arange(first, first + rows, dtype=np.int32), np.zeros(rows, np.int32)
    q = rng.standard_normal((rows, hkv, dh)).astype(np.float32)
    stride = 2 * hkv * dh
    proj = rng.standard_normal((rows, stride)).astype(np.float32)
    d = {k: dev(v) for k, v in dict(q=q, proj=proj, pages=c.rec, table=c.table, pos=pos, seq=seq).items()}
    wb = lib.hero_attn_q4_work_bytes(rows, hkv, hkv, dh, c.max_pages * 64, 0, 0)
    out, work = empty(rows * hkv * dh * 4), dev(np.full(max(wb, 16), 0xFF, np.uint8))
    args = q4_args(c, hkv, rows, ptr(d["pos"]), ptr(d["seq"]) if row_seq else None, proj=ptr(d["proj"]), stride=stride, q_rot=ptr(d["q"]), scale=dh ** -0.5, out=ptr(out),
                   pages=ptr(d["pages"]), table=ptr(d["table"]), work=ptr(work), work_bytes=wb)
    check(lib.hero_attn_q4(args, stream()))
    heads = [0, hkv // 3, hkv - 1]
    few = Pool(rng, 1, 1, len(heads), dh)
    few.rec, few.n, few.table, few.max_pages = c.rec[:, :, heads], c.n, c.table, c.max_pages
    gate = proj.reshape(rows, hkv, 2, dh)[:, heads, 1]
    compare(host(out, np.float32, (rows, hkv, dh))[:, heads], *attend64(few, len(heads), q[:, heads], gate, seq, pos, dh ** -0.5, 0, 0))


@pytest.mark.parametrize("hkv,rows,row_seq,keys_a_sum", [(264, 17, True, 32), (768, 1, False, 128)])
def test_totals_of_equal_weights(lib, hkv, rows, row_seq, keys_a_sum):
    """So many heads that the keys are not split, and all weights but the first key's equal: every addition to the
    total errs to the same side then. Values but the first key's are 0, so that the total alone decides. It is off by 2^-24 of itself for each
    sum that a lane adds to it (one for so many keys), for the 16 terms of such a sum and 40 joins at most; 2^-22
    for the weights' exponents and 2^-22 for the end's roundings."""
    rng = np.random.default_rng(hkv)
    n, dh = 60000, 128
    c = Pool(rng, 1, 2, hkv, spare=0)
    c.max_pages, c.table = -(-n // 64), np.ones((1, -(-n // 64)), np.int32)
    c.table[0, 0] = 0
    c.rec[..., : 8 * dh] = 0x88  # codes 0
    c.rec[..., 8 * dh:] = np.ones(dh // 2, np.float16).view(np.uint8)
    first, ones = np.zeros((hkv, dh), np.int64), np.ones((hkv, dh // 32), np.float16)
    first[:, 0] = 7
    c.store(0, 0, 0, first, ones)
    c.store(0, 1, 0, first, ones)
    q = np.zeros((rows, hkv, dh), np.float32)
    q[..., 0] = np.linspace(0.2, 0.8, hkv)
    pos = np.arange(n - rows, n, dtype=np.int32)
    d = {k: dev(v) for k, v in dict(q=q, proj=np.zeros((rows, 2 * hkv * dh), np.float32), pages=c.rec, table=c.table, pos=pos, seq=np.zeros(rows, np.int32)).items()}
    wb = lib.hero_attn_q4_work_bytes(rows, hkv, hkv, dh, c.max_pages * 64, 0, 0)
    out, work = empty(rows * hkv * dh * 4), empty(max(wb, 16))
    args = q4_args(c, hkv, rows, ptr(d["pos"]), ptr(d["seq"]) if row_seq else None, proj=ptr(d["proj"]), stride=2 * hkv * dh, q_rot=ptr(d["q"]), out=ptr(out), pages=ptr(d["pages"]),
                   table=ptr(d["table"]), work=ptr(work), work_bytes=wb)
    check(lib.hero_attn_q4(args, stream()))
    got = host(out, np.float32, (rows, hkv, dh))
    want = 0.5 * 7 / (1 + pos[:, None] * np.exp(-7 * q[..., 0].astype(np.float64)))
    assert not got[..., 1:].any()
    assert np.abs(got[..., 0] / want - 1).max() <= 2.0 ** -24 * (n / keys_a_sum + 16 + 40) + 2.0 ** -21


def test_calls_at_once_and_one_workspace_after_another(lib):
    """Calls of every form: on two streams at once with a workspace each, and on one stream with one for all, give what they
    give alone."""
    import torch

    rng = np.random.default_rng(5)
    hq, hkv, dh, seqs = 8, 2, 128, 3
    c = Pool(rng, seqs, 40, hkv, dh)
    calls = []
    for seq, pos, row_seq in [([0, 1, 2], [2500, 1700, 9], False), ([1] * 3, [2000, 2001, 2002], True), ([0] * 50 + [2] + [1] * 49, [*range(2000, 2050), 77, *range(1800, 1849)], True)]:
        rows = len(pos)
        d = {k: dev(v) for k, v in dict(q=rng.standard_normal((rows, hq, dh)).astype(np.float32), proj=rng.standard_normal((rows, 2 * hq * dh)).astype(np.float32), pages=c.rec,
                                        table=c.table, pos=np.array(pos, np.int32), seq=np.array(seq, np.int32)).items()}
        wb = lib.hero_attn_q4_work_bytes(rows, hq, hkv, dh, c.max_pages * 64, 0, 0)
        calls.append((rows, row_seq, d, wb))

    def run(call, work, on):
        rows, row_seq, d, wb = call
        out = torch.zeros(rows * hq * dh * 4, dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        args = q4_args(c, hq, rows, ptr(d["pos"]), ptr(d["seq"]) if row_seq else None, proj=ptr(d["proj"]), stride=2 * hq * dh, q_rot=ptr(d["q"]), scale=0.1, out=ptr(out),
                       pages=ptr(d["pages"]), table=ptr(d["table"]), work=ptr(work), work_bytes=wb)
        return out, lambda: check(lib.hero_attn_q4(args, on))

    alone = []
    for call in calls:
        out, go = run(call, empty(call[3]), stream())
        go()
        alone.append(out)
    torch.cuda.synchronize()
    shared = empty(max(call[3] for call in calls))
    sides = [torch.cuda.Stream(), torch.cuda.Stream()]
    own = [[empty(call[3]) for call in calls] for _ in sides]
    for on in (None, *sides):
        again = [run(call, shared, stream() if on is None else on.cuda_stream) for call in calls * 2]
        for _, go in again:
            go()
        torch.cuda.synchronize()
        for (out, _), want in zip(again, alone * 2):
            assert torch.equal(out, want)
    both = [[run(call, w, s.cuda_stream) for call, w in zip(calls, own[k])] for k, s in enumerate(sides)]
    for one, two in zip(both[0], both[1][::-1]):
        one[1]()
        two[1]()
    torch.cuda.synchronize()
    for k in (0, 1):
        for (out, _), want in zip(both[k], alone):
            assert torch.equal(out, want)


@pytest.mark.parametrize("row_seq", [False, True])
def test_what_no_row_sees_has_no_influence(lib, row_seq):
    """Slots past the rows, whole pages behind them, pages before a window: NaN steps there change nothing.
    Pages that hold nothing are not there; a row that sees nothing else gets zeros."""
    rng = np.random.default_rng(17)
    c, bad = Pool(rng, 3, 6, 2, 128, 32), Pool(rng, 3, 6, 2, 128, 32, poison=True)
    pos = [70, 33, 17]
    for s in range(3):  # the bad pool's pages with the good one's rows in them
        for lp in range(6):
            n = np.clip(pos[s] + 1 - 32 * lp, 0, 32)
            byte = [np.unique(c.at[w][0][: 16]) for w in (0, 1)]
            assert len(byte[0])
            for w in (0, 1):
                for slot in range(n):
                    i, rec = slot % 16, (c.table[s, lp], w, slice(None), slot // 16)
                    b, u, st = (t[i] for t in c.at[w])
                    codes = (c.rec[rec][:, b] >> (4 * u)) & 15
                    d = np.ascontiguousarray(c.rec[rec][:, 8 * 128:]).view(np.float16)[:, st[::32]]
                    bad.store(bad.table[s, lp], w, slot, codes.astype(np.int64) - 8, np.ascontiguousarray(d))
    got, want, bound, largest = run_attend(lib, rng, bad, 8, range(3), pos, row_seq=row_seq)
    assert np.isfinite(want).all()
    compare(got, want, bound, largest)
    bad.table[0, 0], bad.table[0, 2], bad.table[1, :] = -1, bad.n, 1 << 30
    got, want, bound, largest = run_attend(lib, rng, bad, 8, range(3), pos, row_seq=row_seq)
    assert not got[1].any() and np.isfinite(got).all()
    compare(got, want, bound, largest)
    # poison before the window
    c = Pool(rng, 1, 8, 2, 128, 32)
    c.rec[c.table[0, 1], ..., 8 * 128:] = 0xFF
    keep = c.rec.copy()
    got, want, bound, largest = run_attend(lib, rng, c, 8, [0], [200], window=100, sinks=20, row_seq=row_seq)
    assert np.isfinite(want).all() and np.array_equal(keep, c.rec)
    compare(got, want, bound, largest)


@pytest.mark.parametrize("row_seq", [False, True])
@pytest.mark.parametrize("what", ["peaked", "rising", "falling", "tiny_values", "subnormal_steps", "large_queries", "one_channel", "zero_query"])
def test_extreme_rows(lib, what, row_seq):
    """Scores that rise or fall by thousands along the context, weights that all but one vanish, values and
    queries at the ends of their ranges."""
    rng = np.random.default_rng(23)
    hq, n = 8, 700
    c = Pool(rng, 1, 11, 2)
    q = rng.standard_normal((1, hq, 128)).astype(np.float32)
    scale = 128 ** -0.5
    if what == "peaked":
        q *= 20
    elif what in ("rising", "falling"):
        q[:] = 1
        c.table[0] = np.arange(11)
        steps = c.rec[..., 0, :, :, 8 * 128:].view(np.float16)
        c.rec[:, 0, :, :, : 8 * 128] = 0x77  # codes -1
        ramp = (np.arange(c.n * 64) if what == "rising" else np.arange(c.n * 64)[::-1]).reshape(c.n, 1, 4, 16, 1)
        steps[:] = np.broadcast_to(round8(ramp * 0.01 * 8), (c.n, 2, 4, 16, 4)).reshape(steps.shape)
    elif what == "tiny_values":
        c.rec[:, 1, ..., 8 * 128:] = round8(rng.uniform(1, 2, c.rec[:, 1, ..., 8 * 128:].shape[:-1] + (64,)) * 2.0 ** -10).view(np.uint8)
    elif what == "subnormal_steps":
        c.rec[..., 8 * 128:] = round8(rng.uniform(1, 9, c.rec[..., 8 * 128:].shape[:-1] + (64,)) * 2.0 ** -18).view(np.uint8)
    elif what == "large_queries":
        q *= np.float32(1e20)
        scale = 1e-20
    elif what == "one_channel":
        q[..., 3] = 3e4
        scale = 1e-4
    else:
        q[:] = 0
    got, want, bound, largest = run_attend(lib, rng, c, hq, [0], [n - 1], row_seq=row_seq, q=q, scale=scale)
    compare(got, want, bound, largest)


@pytest.mark.parametrize("form", ["token", "few", "chunk"])
@pytest.mark.parametrize("dh,hkv", [(128, 2), (256, 1)])
@pytest.mark.parametrize("top", [118, 120, 125, 128])
def test_queries_up_to_the_largest_that_fp32_holds(lib, top, dh, hkv, form):
    """Queries just below 2^top in units of log2 over keys of steps about 2^-18. One key has all codes 7 where the others'
    are random: it takes all of the weight, so a row is its value times the gate, with one rounding for the
    division, one for the product and the gate's 4 ulp. Then keys of zeros: the mean of the values."""
    rng = np.random.default_rng(top + dh)
    hq, n, best = 4 * hkv, 150, 37
    c = Pool(rng, 1, 3, hkv, dh)
    c.rec[:, 0, ..., 8 * dh:] = round8(rng.uniform(1, 2, c.rec[:, 0, ..., 8 * dh:].shape[:-1] + (dh // 2,)) * -8 * 2.0 ** -18).view(np.uint8)
    c.store(c.table[0, 0], 0, best, np.full((hkv, dh), 7), np.full((hkv, dh // 32), 2.0 ** -18, np.float16))
    rows = {"token": 1, "few": 3, "chunk": 30}[form]
    q = (rng.uniform(0.5, 0.999, (rows, hq, dh)) * 2.0 ** top / np.log2(np.e)).astype(np.float32)
    got, want, _, _ = run_attend(lib, rng, c, hq, [0] * rows, list(range(n - rows, n)), row_seq=form != "token", q=q, scale=1.0)
    assert np.all(np.abs(got - want) <= 2.0 ** -20 * np.abs(want))
    c.rec[:, 0, ..., : 8 * dh] = 0x88
    compare(*run_attend(lib, rng, c, hq, [0] * rows, list(range(n - rows, n)), row_seq=form != "token", q=q, scale=1.0))


def test_queries_that_are_not_finite_give_rows_that_are_not(lib):
    rng = np.random.default_rng(5)
    c = Pool(rng, 2, 2, 2)
    q = rng.standard_normal((2, 8, 128)).astype(np.float32)
    q[0, 1, 7], q[0, 6, 9] = np.nan, np.inf
    with np.errstate(invalid="ignore"):
        got, want, _, _ = run_attend(lib, rng, c, 8, [0, 1], [100, 90], row_seq=False, q=q)
    assert np.isnan(got[0, 1]).all() and np.isnan(got[0, 6]).all()
    rest = [0, 2, 3, 4, 5, 7]
    assert np.allclose(got[0, rest], want[0, rest], rtol=0, atol=2.0 ** -19 * np.abs(want[0, rest]).max()) and np.isfinite(got[1]).all()


def test_pools_past_32_bit_offsets(lib):
    """pages at the end of a pool of 4.6 GB: appended, read back and attended to"""
    import torch

    from hero_amd._lib import KvReadArgs

    rng = np.random.default_rng(44)
    hq, hkv, dh, ps, n = 8, 8, 128, 256, 300
    c = Pool(rng, 1, 2, hkv, dh, ps, spare=0)
    pages = 15600
    big = torch.zeros(pages, lib.hero_attn_q4_page_bytes(hkv, dh, ps), dtype=torch.uint8, device="cuda")
    assert big.numel() > 1 << 32
    table = np.array([[pages - 1, pages - 2]], np.int32)
    big[pages - 2:] = torch.from_numpy(c.rec[c.table[0, ::-1]].reshape(2, -1)).cuda()
    proj = rng.standard_normal((1, 2 * (hq + hkv) * dh)).astype(np.float32)
    cs, one = np.tile(np.array([1, 0], np.float32), (n + 1, dh // 2, 1)), np.ones(dh, np.float32)
    d = {k: dev(v) for k, v in dict(proj=proj, cs=cs, one=one, table=table, pos=np.array([n], np.int32)).items()}
    d_q, out = empty(hq * dh * 4), empty(hq * dh * 4)
    wb = lib.hero_attn_q4_work_bytes(1, hq, hkv, dh, 2 * ps, 0, 0)
    work = empty(max(16, wb))
    c.n = pages
    args = q4_args(c, hq, 1, ptr(d["pos"]), proj=ptr(d["proj"]), gq=ptr(d["one"]), gk=ptr(d["one"]), cs=ptr(d["cs"]), q_rot=ptr(d_q), pages=big.data_ptr(), table=ptr(d["table"]),
                   rope=n + 1, out=ptr(out), scale=0.1, work=ptr(work), work_bytes=wb)
    check(lib.hero_kv_append_q4(args, stream()))
    check(lib.hero_attn_q4(args, stream()))
    k_out, v_out = empty(hkv * dh * 4), empty(hkv * dh * 4)
    check(lib.hero_kv_read_q4(KvReadArgs(big.data_ptr(), ptr(d["table"]), ps, 2, 0, pages, None, ptr(d["pos"]), None, 1, 1, hkv, dh, 0, ptr(k_out), ptr(v_out), None, None), stream()))
    k = blocks(rotated64(proj[0, 2 * hq * dh:2 * hq * dh + hkv * dh].reshape(hkv, dh), one, cs[0]))
    v = blocks(proj[0, 2 * hq * dh + hkv * dh:].reshape(hkv, dh))
    for got, (codes, step) in ((k_out, k), (v_out, v)):
        assert np.array_equal(host(got, np.float32).reshape(hkv, dh), codes * np.repeat(step.astype(np.float32), 32, -1))
    page = c.table[0, 1]
    c.store(page, 0, n % ps, *k), c.store(page, 1, n % ps, *v)
    gate = proj[:, : 2 * hq * dh].reshape(1, hq, 2, dh)[:, :, 1]
    c.n = 2
    compare(host(out, np.float32, (1, hq, dh)), *attend64(c, hq, host(d_q, np.float32, (1, hq, dh)), gate, [0], [n], 0.1, 0, 0))


@pytest.mark.parametrize("hq,hkv,dh,rows,past,window,sinks", [(32, 8, 128, 1, 4000, 0, 0), (16, 4, 256, 4, 900, 300, 4), (8, 2, 128, 40, 500, 0, 0)])
def test_captured_and_replayed(lib, hq, hkv, dh, rows, past, window, sinks):
    """append and attention in one graph, on a stream of its own: every replay, over inputs that change in
    between, equals the eager calls"""
    import torch

    rng = np.random.default_rng(rows)
    chunk = rows > 4
    seqs = 1 if chunk else rows
    c = Pool(rng, seqs, -(-(past + rows) // 64), hkv, dh)
    pos = (past + np.arange(rows) if chunk else past - np.arange(rows)).astype(np.int32)
    cs, one = np.tile(np.array([0.6, 0.8], np.float32), (past + rows, dh // 2, 1)), np.ones(dh, np.float32)
    stride = 2 * (hq + hkv) * dh
    d = {k: dev(v) for k, v in dict(cs=cs, one=one, table=c.table, pos=pos, seq=np.zeros(rows, np.int32)).items()}
    wb = lib.hero_attn_q4_work_bytes(rows, hq, hkv, dh, c.max_pages * 64, window, sinks)
    first = torch.from_numpy(c.rec.reshape(-1).copy()).cuda()
    sides = []
    for _ in range(2):
        sides.append(dict(pages=first.clone(), q=empty(rows * hq * dh * 4), out=empty(rows * hq * dh * 4), work=empty(max(16, wb)), proj=empty(rows * stride * 4)))

    def calls(s, on):
        args = q4_args(c, hq, rows, ptr(d["pos"]), ptr(d["seq"]) if chunk else None, proj=ptr(s["proj"]), stride=stride, gq=ptr(d["one"]), gk=ptr(d["one"]), cs=ptr(d["cs"]),
                       q_rot=ptr(s["q"]), pages=ptr(s["pages"]), table=ptr(d["table"]), rope=past + rows, out=ptr(s["out"]), scale=0.1, window=window, sinks=sinks,
                       work=ptr(s["work"]), work_bytes=wb)
        check(lib.hero_kv_append_q4(args, on))
        check(lib.hero_attn_q4(args, on))

    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        calls(sides[0], torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        new = torch.from_numpy(rng.standard_normal(rows * stride).astype(np.float32)).cuda().view(torch.uint8)
        for s in sides:
            s["proj"].copy_(new)
            s["pages"].copy_(first)
            s["out"].zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        calls(sides[1], stream())
        for k in ("pages", "q", "out"):
            assert torch.equal(sides[0][k], sides[1][k]), k
        assert bool(sides[0]["out"].any())


def test_a_token_at_a_time_equals_a_chunk(lib):
    """What a prompt's chunk and its tokens one by one store is the same; what they attend to agrees to rounding."""
    rng = np.random.default_rng(90)
    hq, hkv, dh, n = 8, 2, 128, 70
    c = Pool(rng, 1, 2, hkv, dh)
    stride = 2 * (hq + hkv) * dh
    proj = rng.standard_normal((n, stride)).astype(np.float32)
    angle = np.arange(n)[:, None] * 1e4 ** (-np.arange(dh // 2) / (dh // 2))
    d = {k: dev(v) for k, v in dict(cs=np.stack([np.cos(angle), np.sin(angle)], -1).astype(np.float32), one=np.ones(dh, np.float32), table=c.table, seq=np.zeros(n, np.int32)).items()}
    outs, pools = [], []
    for step in (1, n):
        pages, out, q = dev(c.rec), empty(n * hq * dh * 4), empty(n * hq * dh * 4)
        for r in range(0, n, step):
            d_p, d_pos = dev(proj[r:r + step]), dev(np.arange(r, r + step, dtype=np.int32))
            args = q4_args(c, hq, step, ptr(d_pos), ptr(d["seq"]), proj=ptr(d_p), stride=stride, gq=ptr(d["one"]), gk=ptr(d["one"]), cs=ptr(d["cs"]), q_rot=ptr(q) + r * hq * dh * 4,
                           pages=ptr(pages), table=ptr(d["table"]), rope=n, out=ptr(out) + r * hq * dh * 4, scale=dh ** -0.5)
            check(lib.hero_kv_append_q4(args, stream()))
            check(lib.hero_attn_q4(args, stream()))
            host(out, np.float32)
        outs.append(host(out, np.float32))
        pools.append(host(pages, np.uint8))
    assert np.array_equal(*pools)
    assert np.linalg.norm(outs[0] - outs[1]) <= 2.0 ** -18 * np.linalg.norm(outs[1])
