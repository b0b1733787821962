"""hero_logprobs against the formulas in 64 bits."""
import numpy as np
import pytest

from gpu_util import check, dev, empty, host, ptr, stream

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib():
    from hero_amd._lib import lib as _lib

    import torch

    assert torch.cuda.is_available(), "GPU tests need a GPU"
    return _lib


def run(lib, x, targets, temp=1.0, top=0, stride=None, outs=("logprob", "entropy"), shift=0):
    """x [m][v]; returns the outputs, rows prefilled with 7 (ids: -7)"""
    m, v = x.shape
    stride = stride or v
    flat = np.full(shift + m * stride, np.nan, np.float32)
    for r in range(m):
        flat[shift + r * stride: shift + r * stride + v] = x[r]
    d_x, d_t = dev(flat), None if targets is None else dev(np.asarray(targets, np.int32))
    res = {k: dev(np.full(m, 7, np.float32)) for k in outs}
    if top:
        res["top_ids"], res["top_logprobs"] = dev(np.full((m, top), -7, np.int32)), dev(np.full((m, top), 7, np.float32))
    wb = lib.hero_logprobs_work_bytes(m, v, top)
    work = dev(np.full(max(16, wb), 0xFF, np.uint8))
    at = [ptr(res[k]) if k in res else None for k in ("logprob", "entropy", "top_ids", "top_logprobs")]
    check(lib.hero_logprobs(ptr(d_x) + 4 * shift, stride, m, v, None if d_t is None else ptr(d_t), temp, top, *at, ptr(work), wb, stream()))
    return {k: host(t, np.int32 if k == "top_ids" else np.float32, (m, top) if k.startswith("top") else (m,)) for k, t in res.items()}


def formulas(x, targets, temp, top):
    z = x.astype(np.float64) / float(np.float32(temp))
    big = z.max(-1, keepdims=True)
    e = np.exp(z - big)
    log_sum = big[:, 0] + np.log(e.sum(-1))
    p = e / e.sum(-1, keepdims=True)
    ent = -np.where(p > 0, p * np.where(p > 0, z - log_sum[:, None], 0), 0).sum(-1)
    order = np.argsort(-(x + 0.0).astype(np.float64), axis=-1, kind="stable")[:, :top]
    lp = z - log_sum[:, None]
    return lp[np.arange(len(x)), targets], ent, order, np.take_along_axis(lp, order, -1), e.sum(-1), np.where(p > 0, p * np.where(p > 0, big - z, 0), 0).sum(-1)


def compare(got, x, targets, temp, top, rows=None):
    """A lane adds up to v / 64 terms one after another and 12 joins follow, each off by half an ulp of its
    result; a term's exponent is rounded twice, 2^-23 of its distance from the maximum; the sum's relative error is at most
    that of the terms weighted by their shares, the average distance D. z and the division by temp are off by 2^-23 of the
    target's distance, logarithms by 2 ulp."""
    rows = np.arange(len(x)) if rows is None else rows
    lp, ent, ids, top_lp, total, dist = formulas(x[rows], np.asarray(targets)[rows], temp, top)
    log_total = np.log(total)
    rel = 2.0 ** -24 * (x.shape[1] / 64 + 16 + 12 + 4) + 2.0 ** -23 * (dist + 1)
    base = rel * (1 - 1 / total) + 2.0 ** -22 * log_total  # what is left of the sum's error where one logit is all of it
    if "logprob" in got:
        zt = np.abs(lp + log_total)
        assert np.all(np.abs(got["logprob"][rows] - lp) <= base + 2.0 ** -22 * (zt + np.abs(lp)) + 1e-37)
    if "entropy" in got:  # the second sum carries its terms' errors once more, relative to itself
        assert np.all(np.abs(got["entropy"][rows] - ent) <= base + 2 * rel * dist + 2.0 ** -22 * np.abs(ent) + 1e-37)
    if top:
        assert np.array_equal(got["top_ids"][rows], ids)
        assert np.all(np.abs(got["top_logprobs"][rows] - top_lp) <= base[:, None] + 2.0 ** -22 * (np.abs(top_lp + log_total[:, None]) + np.abs(top_lp)) + 1e-37)


@pytest.mark.parametrize("m,v,top,temp", [(1, 1, 1, 1.0), (2, 2, 2, 0.5), (5, 63, 5, 1.0), (3, 64, 64, 1.0), (4, 1000, 20, 1.3), (2, 1023, 64, 1.0), (2, 1024, 1, 1.0), (2, 1025, 3, 1.0),
                                          (7, 4097, 40, 0.7), (1, 151936, 20, 1.0), (3, 262144, 5, 0.7), (16, 32000, 64, 1.0), (70, 20011, 2, 2.0), (4200, 1500, 1, 1.0)])
@pytest.mark.parametrize("ties", [False, True])
def test_rows_of_every_size(lib, m, v, top, temp, ties):
    rng = np.random.default_rng(m + v)
    x = (rng.standard_normal((m, v)) * 3).astype(np.float32)
    if ties:
        x = np.round(x * 4) / 4
    t = rng.integers(0, v, m)
    t[0] = x[0].argmax()
    compare(run(lib, x, t, temp, top), x, t, temp, top)


@pytest.mark.parametrize("shift,more", [(0, 0), (1, 3), (2, 1), (3, 64)])
def test_strides_and_alignment(lib, shift, more):
    rng = np.random.default_rng(shift)
    x = rng.standard_normal((6, 3001)).astype(np.float32)
    t = rng.integers(0, 3001, 6)
    compare(run(lib, x, t, 1.0, 10, stride=3001 + more, shift=shift), x, t, 1.0, 10)


@pytest.mark.parametrize("order", ["rising", "falling", "equal", "blocks"])
def test_orders_that_fill_the_lists_again_and_again(lib, order):
    v = 40000
    x = np.arange(v, dtype=np.float32)[None] * np.float32(1e-3)
    if order == "falling":
        x = x[:, ::-1].copy()
    elif order == "equal":
        x[:] = -2.5
    elif order == "blocks":
        x = np.floor(x)
    x = np.concatenate([x, x - 50, x + 80])
    t = [0, v - 1, v // 2]
    compare(run(lib, x, t, 1.0, 64), x, t, 1.0, 64)


@pytest.mark.parametrize("case", ["equal", "two values", "together", "together, ties", "every 16384", "NaN but ten"])
@pytest.mark.parametrize("v", [8192, 60000])
def test_many_logits_among_the_largest(lib, case, v):
    rng = np.random.default_rng(v)
    x = (rng.standard_normal((3, v)) * 2).astype(np.float32)
    if case == "equal":
        x[:] = 1.25
    elif case == "two values":
        x[:] = np.where(rng.random((3, v)) < 0.5, 3, -1)
    elif case.startswith("together"):  # a few thousand neighbours far above all others
        x[:, 1000:6500] += 100
        if case.endswith("ties"):
            x[:, 1000:6500] = np.round(x[:, 1000:6500] / 4) * 4
    elif case == "every 16384":
        x[:, np.arange(v) % 16384 < 2000] += 40
    else:
        x[:] = np.nan
        x[:, 7:7 + 64 * 90:64 * 9] = np.arange(10, dtype=np.float32)
    t = [5, 1001, 7]
    got = run(lib, x, t, 1.0, 64)
    if case == "NaN but ten":
        for r in range(3):
            assert got["top_ids"][r].tolist() == [7 + 576 * i for i in range(9, -1, -1)] + [i for i in range(55) if i != 7][:54]
    else:
        compare(got, x, t, 1.0, 64)


def test_ranges_of_many_batches(lib):
    rng = np.random.default_rng(1)
    x = (rng.standard_normal((2, 3000017)) * 3).astype(np.float32)
    compare(run(lib, x, [0, 3000016], 1.0, 20), x, [0, 3000016], 1.0, 20)


def test_zeros_of_both_signs_tie(lib):
    x = np.full((1, 5000), -1, np.float32)
    x[0, [4000, 17, 900, 3]] = [0.0, -0.0, 0.0, -0.0]
    assert run(lib, x, [0], 1.0, 4)["top_ids"].tolist() == [[3, 17, 900, 4000]]


def test_masked_tokens(lib):
    """-inf logits have probability 0, and rank by id behind every other"""
    rng = np.random.default_rng(2)
    x = rng.standard_normal((3, 9000)).astype(np.float32)
    x[:, rng.random(9000) < 0.7] = -np.inf
    x[1] = -np.inf
    x[1, 8000] = 1.5
    t = [int(np.flatnonzero(x[0] > -9)[5]), 8000, int(np.flatnonzero(x[2] == -np.inf)[3])]
    got = run(lib, x, t, 1.0, 8)
    compare(got, x, t, 1.0, 8, rows=np.array([0]))
    assert got["logprob"][1] == 0 and got["entropy"][1] == 0 and got["top_logprobs"][1].tolist() == [0] + [-np.inf] * 7
    assert got["top_ids"][1].tolist() == [8000, 0, 1, 2, 3, 4, 5, 6]
    assert got["logprob"][2] == -np.inf


def test_rows_that_are_not_finite(lib):
    rng = np.random.default_rng(3)
    x = rng.standard_normal((5, 4000)).astype(np.float32)
    x[0, 77], x[1, 5], x[2], x[3, 40:] = np.nan, np.inf, -np.inf, np.nan
    t = [3, 5, 0, 2, 9]
    got = run(lib, x, t, 1.0, 64)
    for k in ("logprob", "entropy"):
        assert np.isnan(got[k][:4]).all()
    assert np.isnan(got["top_logprobs"][:4]).all()
    order = np.argsort(-x[0], kind="stable")
    assert got["top_ids"][0].tolist() == [i for i in order if i != 77][:64]
    assert got["top_ids"][1, 0] == 5 and got["top_ids"][2].tolist() == list(range(64))
    assert got["top_ids"][3].tolist() == sorted(range(40), key=lambda i: (-x[3, i], i)) + list(range(40, 64))
    compare(got, x, t, 1.0, 64, rows=np.array([4]))


@pytest.mark.parametrize("temp", [1.0, 2.0, 1e38, 3.4e38])
@pytest.mark.parametrize("m,v", [(1, 200000), (3, 2000), (2100, 600)])
def test_logits_further_apart_than_fp32_reaches(lib, m, v, temp):
    """Logits over all of fp32's range, masks of its lowest value among them: differences pass it, quotients by temp do
    not (but for temp 1, where one that does is -inf)."""
    rng = np.random.default_rng(v)
    x = rng.uniform(-3.4e38, 3.4e38, (m, v)).astype(np.float32)
    x[rng.random((m, v)) < 0.2] = np.finfo(np.float32).min
    t = rng.integers(0, v, m)
    t[0] = x[0].argmin()
    got = run(lib, x, t, temp, 5)
    if temp > 1:
        return compare(got, x, t, temp, 5)
    lp, ent, ids, top_lp, *_ = formulas(x, t, temp, 5)
    with np.errstate(over="ignore"):  # one logit has it all, the others' log probabilities are differences
        assert np.allclose(got["logprob"], lp.astype(np.float32), rtol=2.0 ** -22, atol=0) and np.allclose(got["top_logprobs"], top_lp.astype(np.float32), rtol=2.0 ** -22, atol=0)
    assert np.array_equal(got["top_ids"], ids) and not got["entropy"].any() and not ent.any()


def test_alternatives_of_rows_that_one_wave_reads_alone(lib):
    """more batches than maxima are kept before they are stored"""
    rng = np.random.default_rng(9)
    m, v = 1100, 70001
    x = (rng.standard_normal((m, v), dtype=np.float32) * 3).astype(np.float32)
    t = rng.integers(0, v, m)
    compare(run(lib, x, t, 1.0, 20), x, t, 1.0, 20, rows=np.array([0, 1, 5, 500, 1098, 1099]))


def test_sums_of_thousands_of_equal_terms(lib):
    """Rows that one wave each sums alone, all logits but one equal: every addition to a sum errs to the same side then.
    A lane adds up 16 terms and then v / 1024 such sums, which bounds the sum's error by 2^-24 of it for each of these, for
    the 12 joins and 4 more; a term's exponent and the logarithms as in compare()."""
    import torch

    m, v = 1030, 262144
    gap = np.resize(np.array([2.5, 1.375, 5.875, 3.75, 5.625, 11.0]), m)
    x = (-torch.from_numpy(gap.astype(np.float32)).cuda())[:, None].expand(m, v).contiguous()
    x[:, 77] = 0
    t = dev(np.full(m, 77, np.int32))
    lp, ent, wb = empty(4 * m), empty(4 * m), lib.hero_logprobs_work_bytes(m, v, 0)
    work = empty(wb)
    check(lib.hero_logprobs(x.data_ptr(), v, m, v, ptr(t), 1.0, 0, ptr(lp), ptr(ent), None, None, ptr(work), wb, stream()))
    r = (v - 1) * np.exp(-gap)
    rel, dist, want = 2.0 ** -24 * (v / 1024 + 16 + 12 + 4) + 2.0 ** -23 * (gap + 1), gap * r / (1 + r), np.log1p(r)
    assert np.all(np.abs(host(lp, np.float32) + want) <= rel + 2.0 ** -21 * want)
    assert np.all(np.abs(host(ent, np.float32) - (want + dist)) <= rel + 2 * rel * dist + 2.0 ** -21 * (want + dist))


def test_nearly_certain_tokens_keep_their_precision(lib):
    """log probabilities and entropies of 1e-3 down to 1e-30, to a relative 2^-23 (v / 64 + 40 + 2 * distance)"""
    v = 2000
    for gap in (10, 20, 40, 75):
        x = np.zeros((1, v), np.float32)
        x[0, 1234] = gap
        got = run(lib, x, [1234], 1.0, 1)
        r = (v - 1) * np.exp(-float(gap))
        tol = 2.0 ** -23 * (v / 64 + 40 + 2 * gap)
        assert abs(got["logprob"][0] + np.log1p(r)) <= tol * r
        assert got["top_logprobs"][0, 0] == got["logprob"][0]
        ent = np.log1p(r) + r * gap / (1 + r)
        assert abs(got["entropy"][0] - ent) <= 2 * tol * ent


def test_left_out_rows_and_missing_outputs(lib):
    rng = np.random.default_rng(4)
    x = rng.standard_normal((6, 1500)).astype(np.float32)
    t = [3, -1, 1500, 1499, 0, -(1 << 31)]
    live = np.array([0, 3, 4])
    for outs in (("logprob", "entropy"), ("logprob",), ("entropy",), ()):
        for top in (0, 3):
            if not outs and not top:
                continue
            got = run(lib, x, t, 1.0, top, outs=outs)
            compare(got, x, np.clip(t, 0, 1499), 1.0, top, rows=live)
            for k in got:
                assert np.all(got[k][[1, 2, 5]] == (-7 if k == "top_ids" else 7)), k
    got = run(lib, x, None, 1.0, 3, outs=("entropy",))
    compare(got, x, np.zeros(6, int), 1.0, 3)


def test_rows_past_32_bit_offsets(lib):
    """the last row of 4.5 GB of logits"""
    import torch

    m, v = 8, 1000
    stride = 160_000_000
    x = torch.zeros((m - 1) * stride + v, device="cuda")
    assert x.numel() * 4 > 1 << 32
    row = np.random.default_rng(1).standard_normal((1, v)).astype(np.float32)
    x[(m - 1) * stride:] = torch.from_numpy(row[0]).cuda()
    t = dev(np.full(m, 5, np.int32))
    lp, wb = empty(4 * m), lib.hero_logprobs_work_bytes(m, v, 0)
    work = empty(wb)
    check(lib.hero_logprobs(x.data_ptr(), stride, m, v, ptr(t), 1.0, 0, ptr(lp), None, None, None, ptr(work), wb, stream()))
    got = host(lp, np.float32)
    assert np.all(np.abs(got[:-1] + np.log(v)) < 1e-5)
    compare({"logprob": got[-1:]}, row, [5], 1.0, 0)


@pytest.mark.parametrize("m,v,top", [(1, 151936, 20), (5, 3000, 3)])
def test_captured_and_replayed(lib, m, v, top):
    import torch

    rng = np.random.default_rng(v)
    wb = lib.hero_logprobs_work_bytes(m, v, top)
    x = torch.zeros(m, v, device="cuda")
    t = torch.from_numpy(rng.integers(0, v, m).astype(np.int32)).cuda()
    res = [dict(lp=torch.zeros(m, device="cuda"), ent=torch.zeros(m, device="cuda"), ids=torch.zeros(m, top, dtype=torch.int32, device="cuda"),
                tl=torch.zeros(m, top, device="cuda"), work=empty(wb)) for _ in range(2)]

    def call(r, on):
        check(lib.hero_logprobs(x.data_ptr(), v, m, v, t.data_ptr(), 0.8, top, *(r[k].data_ptr() for k in ("lp", "ent", "ids", "tl", "work")), wb, on))

    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        call(res[0], torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        x.copy_(torch.from_numpy(rng.standard_normal((m, v)).astype(np.float32)))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        call(res[1], stream())
        for k in ("lp", "ent", "ids", "tl"):
            assert torch.equal(res[0][k], res[1][k]), k
        assert bool(res[0]["lp"].all())


def test_millions_of_rows(lib):
    """more workgroups of the second launch than one dimension of a grid takes"""
    import torch

    m, v = (1 << 23) + 77, 3
    x = torch.randn(m, v, device="cuda")
    t = torch.randint(0, v, (m,), device="cuda", dtype=torch.int32)
    lp, ids, tlp, wb = empty(4 * m), empty(4 * m), empty(4 * m), lib.hero_logprobs_work_bytes(m, v, 1)
    work = empty(wb)
    check(lib.hero_logprobs(ptr(x), v, m, v, ptr(t), 1.0, 1, ptr(lp), None, ptr(ids), ptr(tlp), ptr(work), wb, stream()))
    torch.cuda.synchronize()
    want = torch.log_softmax(x.double(), -1)
    # three terms: a few roundings of values below 2^4
    assert (lp.view(torch.float32) - want.gather(1, t.long()[:, None])[:, 0]).abs().max().item() <= 2.0 ** -19
    assert torch.equal(ids.view(torch.int32).long(), x.argmax(-1))
    assert (tlp.view(torch.float32) - want.max(-1).values).abs().max().item() <= 2.0 ** -19


def test_calls_at_once(lib):
    """on two streams, a workspace each"""
    import torch

    rng = np.random.default_rng(6)
    m, v, top = 3, 50000, 20
    want, sides, xs = [], [torch.cuda.Stream(), torch.cuda.Stream()], []
    for _ in sides:
        x = (rng.standard_normal((m, v)) * 3).astype(np.float32)
        t = rng.integers(0, v, m)
        want.append(run(lib, x, t, 1.0, top))
        xs.append((dev(x), dev(t.astype(np.int32)), empty(4 * m), empty(4 * m), empty(4 * m * top), empty(4 * m * top), empty(lib.hero_logprobs_work_bytes(m, v, top))))
    torch.cuda.synchronize()
    for _ in range(3):
        for s, (x, t, lp, ent, ids, tlp, work) in zip(sides, xs):
            check(lib.hero_logprobs(ptr(x), v, m, v, ptr(t), 1.0, top, ptr(lp), ptr(ent), ptr(ids), ptr(tlp), ptr(work), lib.hero_logprobs_work_bytes(m, v, top), s.cuda_stream))
    torch.cuda.synchronize()
    for w, (_, _, lp, ent, ids, tlp, _) in zip(want, xs):
        for k, got in (("logprob", lp), ("entropy", ent), ("top_ids", ids), ("top_logprobs", tlp)):
            assert np.array_equal(host(got, w[k].dtype, w[k].shape), w[k]), k


def test_a_serving_step(lib):
    """Tokens enter a 4-bit cache, attend to it, pass an output projection of Q8_0 weights into logits, and the
    next tokens' log probabilities come out: four steps of three sequences against the formulas in 64 bits on
    what was stored."""
    import oracle
    from gpu_util import act_to_blocks, pack_weight
    from test_gpu_q4 import Pool, attend64, blocks, q4_args, rotated64

    rng = np.random.default_rng(12)
    hq, hkv, dh, seqs, vocab = 8, 2, 128, 3, 4096
    c = Pool(rng, seqs, 4, hkv, dh)
    stride, k_in = 2 * (hq + hkv) * dh, hq * dh
    w = oracle.quantize_row_q8_0((rng.standard_normal(vocab * k_in) * 0.2).astype(np.float32)).reshape(vocab, k_in // 32)
    packed = pack_weight(lib, w, vocab, k_in)
    w64 = (w["qs"].astype(np.float64) * w["d"].view(np.float16).astype(np.float64)[..., None]).reshape(vocab, k_in)
    angle = np.arange(256)[:, None] * 1e4 ** (-np.arange(dh // 2) / (dh // 2))
    cs, gamma = np.stack([np.cos(angle), np.sin(angle)], -1).astype(np.float32), (1 + 0.1 * rng.standard_normal(dh)).astype(np.float32)
    pages, d_t, d_cs, d_g = dev(c.rec), dev(c.table), dev(cs), dev(gamma)
    q, act = empty(seqs * k_in * 4), empty(lib.hero_q8_0_act_bytes(seqs, k_in))
    logits, lp, ent = empty(seqs * vocab * 4), empty(seqs * 4), empty(seqs * 4)
    ids, tl = empty(seqs * 5 * 4), empty(seqs * 5 * 4)
    wb = lib.hero_logprobs_work_bytes(seqs, vocab, 5)
    work = empty(wb)
    for step in range(4):
        pos = np.array([100 + step, 15 + step, step], np.int32)
        proj = rng.standard_normal((seqs, stride)).astype(np.float32)
        token = rng.integers(0, vocab, seqs).astype(np.int32)
        d_p, d_pos, d_tok = dev(proj), dev(pos), dev(token)
        args = q4_args(c, hq, seqs, ptr(d_pos), proj=ptr(d_p), stride=stride, gq=ptr(d_g), gk=ptr(d_g), cs=ptr(d_cs), q_rot=ptr(q), pages=ptr(pages), table=ptr(d_t), rope=256,
                       act=ptr(act), scale=dh ** -0.5, window=64, sinks=4)
        check(lib.hero_kv_append_q4(args, stream()))
        check(lib.hero_attn_q4(args, stream()))
        check(lib.hero_q8_0_gemm(ptr(packed), ptr(act), ptr(logits), None, seqs, vocab, k_in, stream()))
        check(lib.hero_logprobs(ptr(logits), vocab, seqs, vocab, ptr(d_tok), 1.0, 5, ptr(lp), ptr(ent), ptr(ids), ptr(tl), ptr(work), wb, stream()))
        for s in range(seqs):
            page, slot = c.table[s, pos[s] // 64], pos[s] % 64
            c.store(page, 0, slot, *blocks(rotated64(proj[s, 2 * hq * dh:2 * hq * dh + hkv * dh].reshape(hkv, dh), gamma, cs[pos[s]])))
            c.store(page, 1, slot, *blocks(proj[s, 2 * hq * dh + hkv * dh:].reshape(hkv, dh)))
        assert np.array_equal(host(pages, np.uint8), c.rec.reshape(-1))
        gate = proj[:, : 2 * hq * dh].reshape(seqs, hq, 2, dh)[:, :, 1]
        want, bound, _ = attend64(c, hq, host(q, np.float32, (seqs, hq, dh)), gate, range(seqs), pos, dh ** -0.5, 64, 4)
        a = act_to_blocks(host(act, np.uint8), seqs, k_in)
        d = a["d"].view(np.float16).astype(np.float64)[..., None]
        a64 = a["qs"] * d
        # a Q8_0 value is off by half a step (and 2^-11 of it for the step's own rounding) of what was quantized
        assert np.all(np.abs(a64 - want.reshape(a64.shape)) <= bound.reshape(a64.shape) + d * (0.5 + 127 * 2.0 ** -11))
        x = host(logits, np.float32, (seqs, vocab))
        x64 = a64.reshape(seqs, k_in) @ w64.T
        mags = np.abs(a64.reshape(seqs, k_in)) @ np.abs(w64.T)
        assert np.all(np.abs(x - x64) <= (k_in / 32 + 4) * 2.0 ** -24 * mags)
        compare({"logprob": host(lp, np.float32), "entropy": host(ent, np.float32), "top_ids": host(ids, np.int32, (seqs, 5)), "top_logprobs": host(tl, np.float32, (seqs, 5))},
                x, token, 1.0, 5)
