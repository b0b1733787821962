"""The long-context paged-cache operators, case by case: appending rows to a
paged fp16 or Q8_0 cache (query / key norms and rotation, quantization, page
summaries), reading rows back, selecting the pages a query attends to by a cheap
score, and the attention over the selected pages.

Sizes are those of the repository's configurations: an ~8B hybrid (32 query
heads over 8 K/V heads of 128), the 256-wide heads of the Qwen 3.5 9B one (16
over 4), pages of 64 positions, up to sixteen sequences decoded together, and
contexts up to half of the reference's 262144 positions.
"""
import functools
import math

import torch

own = False

EPS = 1e-6
ROPE_BASE = 1e6
ROPE_POSITIONS = 32768


def listed():
    return [
        # One new token of one chat enters its cache: the smallest call, latency and launches count.
        {"name": "append_token", "kind": "append", "cache": "fp16", "hq": 32, "hkv": 8, "dh": 128, "ps": 64, "seqs": 1, "rows": 1, "past": 5000, "decode": True},
        # One new token of each of sixteen sequences into a Q8_0 cache.
        {"name": "append_batch_q8", "kind": "append", "cache": "q8", "hq": 32, "hkv": 8, "dh": 128, "ps": 64, "seqs": 16, "rows": 16, "past": 9000, "decode": True},
        # A prompt's chunk after a first one, which ended inside a page.
        {"name": "append_prompt_q8", "kind": "append", "cache": "q8", "hq": 32, "hkv": 8, "dh": 128, "ps": 64, "seqs": 1, "rows": 1000, "past": 1000, "decode": False},
        # A cached prefix is read back whole, to be handed to an fp32 cache.
        {"name": "read_prefix_q8", "kind": "read", "cache": "q8", "hkv": 8, "dh": 128, "ps": 64, "seqs": 1, "rows": 8192, "past": 0, "f16": False},
        # A short prefix of 256-wide heads, as fp16.
        {"name": "read_short_wide", "kind": "read", "cache": "fp16", "hkv": 4, "dh": 256, "ps": 64, "seqs": 1, "rows": 257, "past": 0, "f16": True},
        # One token picks 32 of the pages of a 32k chat.
        {"name": "select_token", "kind": "select", "hq": 32, "hkv": 8, "dh": 128, "ps": 64, "seqs": 1, "rows": 1, "past": 32000, "top": 32, "decode": True},
        # Sixteen long documents at once, one token each.
        {"name": "select_batch_long", "kind": "select", "hq": 32, "hkv": 8, "dh": 128, "ps": 64, "seqs": 16, "rows": 16, "past": 131000, "top": 64, "decode": True},
        # A chunk of a long prompt: every row picks its own pages.
        {"name": "select_prompt", "kind": "select", "hq": 32, "hkv": 8, "dh": 128, "ps": 64, "seqs": 1, "rows": 500, "past": 16001, "top": 16, "decode": False},
        # One token's attention over 2048 of a 32k chat's keys.
        {"name": "attend_token", "kind": "attend", "cache": "fp16", "hq": 32, "hkv": 8, "dh": 128, "ps": 64, "seqs": 1, "rows": 1, "past": 32000, "top": 32, "decode": True},
        # Sixteen sequences over a Q8_0 cache.
        {"name": "attend_batch_q8", "kind": "attend", "cache": "q8", "hq": 32, "hkv": 8, "dh": 128, "ps": 64, "seqs": 16, "rows": 16, "past": 32000, "top": 32, "decode": True},
        # Eight sequences with the 256-wide heads.
        {"name": "attend_batch_wide", "kind": "attend", "cache": "fp16", "hq": 16, "hkv": 4, "dh": 256, "ps": 64, "seqs": 8, "rows": 8, "past": 16000, "top": 48, "decode": True},
        # A prompt's chunk, each row over its own 1024 keys: the largest.
        {"name": "attend_prompt", "kind": "attend", "cache": "fp16", "hq": 32, "hkv": 8, "dh": 128, "ps": 64, "seqs": 1, "rows": 500, "past": 16001, "top": 16, "decode": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the same ranges: single tokens of one to sixteen sequences, and
    chunks of prompts of one to three sequences (some rows are padding), every
    cache type, group size and page size, contexts from a few tokens to 131k."""
    kind = rng.choice(["append", "append", "read", "select", "select", "attend", "attend", "attend"])
    cache = rng.choice(["fp16", "q8"])
    dh = rng.choice([128, 128, 256]) if cache == "fp16" else 128
    hq, hkv = rng.choice([(32, 8), (32, 8), (16, 4), (8, 2), (16, 2), (24, 8), (8, 8)])
    c = {"kind": kind, "hkv": hkv, "dh": dh, "ps": rng.choice([64, 64, 64, 16, 32, 128])}
    if kind in ("append", "read", "attend"):
        c["cache"] = cache
    if kind == "read":
        c.update(seqs=rng.randint(1, 4), rows=_log(rng, 1, 8192), past=rng.randint(0, 8000), f16=rng.random() < 0.5)
        return c
    c["hq"] = hq
    c["decode"] = rng.random() < 0.6
    if c["decode"]:
        c["seqs"] = c["rows"] = rng.choice([1, 2, rng.randint(3, 16)])
        c["past"] = _log(rng, 1, 32000 if kind != "select" else 131000)
    else:
        c["seqs"] = rng.randint(1, 3)
        c["rows"] = _log(rng, 4, 1000 if kind == "append" else 400)
        c["past"] = _log(rng, 1, 16000)
    if kind in ("select", "attend"):
        c["top"] = rng.choice([4, 8, 16, rng.randint(4, 16)]) * (64 // min(c["ps"], 64)) * (2 if c["decode"] else 1)
    return c


# ---- inputs ------------------------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(1000003 * (seed + 1))
    return g


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, device="cuda", generator=g, dtype=dtype)


@functools.lru_cache(maxsize=4)
def _rope(dh):
    """cos / sin [positions][dh/2][2] of the first quarter of the planes, as a loader lays them out once"""
    inv = torch.zeros(dh // 2, dtype=torch.float64, device="cuda")
    inv[: dh // 8] = ROPE_BASE ** (-2.0 * torch.arange(dh // 8, dtype=torch.float64, device="cuda") / dh)
    angle = torch.arange(ROPE_POSITIONS, dtype=torch.float64, device="cuda")[:, None] * inv
    return torch.stack([torch.cos(angle), torch.sin(angle)], -1).float()


def _rows(c, g):
    """Each row's sequence and position. Decoded tokens: a row per sequence, lengths differing a little. A chunk: the
    sequences' rows one after another; past one sequence, the last few rows are padding (position -1)."""
    rows, seqs, past = c["rows"], c["seqs"], c["past"]
    if c.get("decode"):
        less = torch.randint(0, max(1, past // 8), (rows,), device="cuda", generator=g)
        less[0] = 0
        return torch.arange(rows, device="cuda"), past - less
    seq = torch.arange(rows, device="cuda") * seqs // rows
    first = torch.zeros(seqs, dtype=torch.long, device="cuda").scatter_reduce(0, seq, torch.arange(rows, device="cuda"), "amin", include_self=False)
    start = past - torch.arange(seqs, device="cuda") * (past // 4)
    pos = start[seq] + torch.arange(rows, device="cuda") - first[seq]
    if seqs > 1:
        pos[rows - rows // 10:] = -1
    return seq, pos


def _max_pages(c):
    return -(-(c["past"] + (1 if c.get("decode") else c["rows"])) // c["ps"])


def _pool(c, g):
    """The page pool: fp16 [page][2][hkv][ps][dh], or the bytes of Q8_0 pages (int8 rows, then fp16 scales per 32 values)."""
    n, hkv, ps, dh = c["seqs"] * _max_pages(c), c["hkv"], c["ps"], c["dh"]
    if c["cache"] == "fp16":
        return _randn(g, n, 2, hkv, ps, dh, dtype=torch.float16)
    values = 2 * hkv * ps * dh
    pool = torch.empty(n, values + values // 16, dtype=torch.uint8, device="cuda")
    q, d = _pool_parts(c, pool)
    q.copy_((torch.randn(n, 2, hkv, ps, dh, device="cuda", generator=g, dtype=torch.float16) * 45).clamp_(-127, 127))
    d.copy_(torch.rand(d.shape, device="cuda", generator=g) * 0.02 + 0.01)
    return pool


def _pool_parts(c, pool):
    """A Q8_0 pool's int8 values [page][2][hkv][ps][dh] and fp16 scales [page][2][hkv][ps][dh/32], as views."""
    hkv, ps, dh = c["hkv"], c["ps"], c["dh"]
    values = 2 * hkv * ps * dh
    return pool[:, :values].view(torch.int8).unflatten(1, (2, hkv, ps, dh)), pool[:, values:].view(torch.float16).unflatten(1, (2, hkv, ps, dh // 32))


def _summary_bytes(c):
    """Bytes of a page's summary: per K/V head the int8 max and -min of its channels, then a scale per head, to 16 bytes."""
    return c["hkv"] * 2 * c["dh"] + -(-c["hkv"] * 4 // 16) * 16


def _summary_parts(c, s):
    """The int8 bounds [page][hkv][2 = max, -min][dh] and fp32 scales [page][hkv], as views."""
    n = c["hkv"] * 2 * c["dh"]
    return s[:, :n].view(torch.int8).unflatten(1, (c["hkv"], 2, c["dh"])), s[:, n:n + 4 * c["hkv"]].view(torch.float32)


def _summaries(c, g):
    """Bounds as 64 keys of a page have them: around +-2.4 deviations, differing per channel."""
    n = c["seqs"] * _max_pages(c)
    s = torch.zeros(n, _summary_bytes(c), dtype=torch.uint8, device="cuda")
    q, d = _summary_parts(c, s)
    shape = (n, c["hkv"], c["dh"])
    mid, half = _randn(g, *shape) * 12, 60 + _randn(g, *shape) * 15
    q[:, :, 0] = (mid + half).clamp(-127, 127).to(torch.int8)
    q[:, :, 1] = (half - mid).clamp(-127, 127).to(torch.int8)
    d.copy_(_round11(torch.rand(n, c["hkv"], device="cuda", generator=g) * 0.01 + 0.025))
    return s


def _selected(c, g, seq, pos):
    """Lists as the selection gives them: rows of a chunk agree on many pages; page 0 and the last two are always there."""
    n, top, rows, hkv = _max_pages(c), c["top"], c["rows"], c["hkv"]
    visible = pos // c["ps"] + 1  # 0 for a padded row
    score = _randn(g, c["seqs"], hkv, n)[seq] + 0.5 * _randn(g, rows, hkv, n)
    page = torch.arange(n, device="cuda")
    score = torch.where((page < 1) | (page >= visible[:, None, None] - 2), math.inf, score)
    score = torch.where(page >= visible[:, None, None], -math.inf, score)
    idx = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :top]
    idx = torch.where(torch.arange(idx.shape[-1], device="cuda") < visible[:, None, None], idx, n)
    idx = torch.sort(idx, -1).values
    out = torch.full((rows, hkv, top), -1, dtype=torch.int32, device="cuda")
    out[..., : idx.shape[-1]] = torch.where(idx < n, idx, -1)
    return out


def prepare(case, seed):
    c, g = case, _gen(seed)
    kind, rows, hkv, dh = c["kind"], c["rows"], c["hkv"], c["dh"]
    seq, pos = _rows(c, g)
    s = {"case": c, "pos": pos.int(), "seq": seq.int()}
    if kind in ("append", "attend"):
        s["proj"] = _randn(g, rows, 2 * c["hq"] * dh + 2 * hkv * dh)  # [q | gate] pairs, k, v
    if kind == "append":
        s["gq"], s["gk"], s["rope"] = 1 + 0.1 * _randn(g, dh), 1 + 0.1 * _randn(g, dh), _rope(dh)
        s["q_rot"] = torch.zeros(rows, c["hq"], dh, device="cuda")
    elif kind != "read":  # select and attend take normalised, rotated queries; consecutive rows' are alike
        s["q_rot"] = 0.8 * _randn(g, c["seqs"], c["hq"], dh)[seq] + 0.6 * _randn(g, rows, c["hq"], dh)
    n = _max_pages(c)
    s["table"] = torch.randperm(c["seqs"] * n, device="cuda", generator=g).to(torch.int32).view(c["seqs"], n)
    if "cache" in c:
        s["pool"] = _pool(c, g)
    if kind == "select":
        s["summaries"] = _summaries(c, g)
        s["selected"] = torch.full((rows, hkv, c["top"]), -1, dtype=torch.int32, device="cuda")
    if kind == "append":
        s["summaries"] = torch.zeros(c["seqs"] * n, _summary_bytes(c), dtype=torch.uint8, device="cuda")
    if kind == "attend":
        s["selected"] = _selected(c, g, seq, pos)
        s["out"] = torch.zeros(rows, c["hq"] * dh, device="cuda")
    if kind in ("append", "read"):
        t = torch.float16 if kind == "append" or c["f16"] else torch.float32
        s["back"] = [torch.zeros(rows, hkv * dh, dtype=t, device="cuda") for _ in range(4 if kind == "append" else 2)]
    if own:
        _plan(s)
    return s


# ---- the framework's calls -----------------------------------------------------------------------------
def _plan(s):
    """The argument structs and workspace that a program keeps beside its cache."""
    from hero_amd._lib import AttnDecodeArgs, AttnPagedArgs, AttnSparseArgs, KvReadArgs, lib

    c = s["case"]
    p = lambda name: s[name].data_ptr() if name in s else None  # noqa: E731
    hkv, dh, n, rows = c["hkv"], c["dh"], _max_pages(c), c["rows"]
    q8 = 1 if c.get("cache") == "q8" else 0
    row_seq = None if c.get("decode") else s["seq"].data_ptr()
    if c["kind"] in ("append", "read"):
        out = [t.data_ptr() for t in s["back"]] + [None, None]  # keys, values, and the page's bounds where they are asked for
        s["read"] = KvReadArgs(p("pool"), p("table"), c["ps"], n, q8, s["pool"].shape[0], p("summaries"), p("pos"), row_seq, rows, c["seqs"], hkv, dh,
                               1 if s["back"][0].dtype == torch.float16 else 0, *out[:4])
    if c["kind"] == "read":
        return
    hq = c["hq"]
    a = AttnDecodeArgs(p("proj"), 2 * (hq + hkv) * dh, 2 * hq * dh, 2 * hq * dh + hkv * dh, p("gq"), p("gk"), EPS, p("rope"), None, None, 0, p("pos"), None, p("q_rot"),
                       1.0 / math.sqrt(dh), 0, None, p("out"), rows, hq, hkv, dh)
    if c["kind"] == "select":
        work = lib.hero_attn_select_work_bytes(rows, hkv, n)
    elif c["kind"] == "attend":
        work = lib.hero_attn_sparse_work_bytes(rows, hq, hkv, dh, c["ps"], c["top"])
    else:
        work = 0
    s["work"] = torch.empty(max(16, work), dtype=torch.uint8, device="cuda")
    paged = AttnPagedArgs(a, p("pool"), p("table"), c["ps"], n, p("work"), work, q8)
    s["args"] = AttnSparseArgs(paged, c["seqs"] * n, ROPE_POSITIONS, row_seq, c["seqs"], p("summaries"), p("selected"), c.get("top", 0), 1, 2)


def _run_own(s):
    from hero_amd._lib import check, lib

    stream = torch.cuda.current_stream().cuda_stream
    kind = s["case"]["kind"]
    if kind == "append":
        check(lib.hero_kv_append_paged(s["args"], stream))
        check(lib.hero_kv_read_paged(s["read"], stream))
        return [s["q_rot"], *s["back"]]
    if kind == "read":
        check(lib.hero_kv_read_paged(s["read"], stream))
        return s["back"]
    if kind == "select":
        check(lib.hero_attn_select_pages(s["args"], stream))
        return s["selected"]
    check(lib.hero_attn_sparse_paged(s["args"], stream))
    return s["out"]


# ---- the plain forms -----------------------------------------------------------------------------------
def _round11(x):
    """x >= 0 to 11 significant bits, halves away from zero."""
    return ((x.view(torch.int32) + 0x1000) & -0x2000).view(torch.float32)


def _quantize(x):
    """Symmetric 8-bit codes of the last axis, in fp32 steps, and the step before its own rounding."""
    d = x.abs().amax(-1, keepdim=True) / torch.full((), 127.0, device=x.device)  # a tensor: division by a number multiplies by its reciprocal
    v = x * torch.where(d > 0, torch.ones_like(d) / d, torch.zeros_like(d))
    return torch.sign(v) * torch.floor(v.abs() + 0.5), d.squeeze(-1)


def _norm_rotate(x, gamma, cs):
    """RMSNorm of each head and the rotation of its planes (i, i + dh/2); x [rows][heads][dh], cs [rows][dh/2][2]."""
    x = gamma * x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
    lo, hi = x.chunk(2, -1)
    cos, sin = cs[:, None, :, 0], cs[:, None, :, 1]
    return torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1)


def _place(s):
    """Rows that are no padding, their pool pages and their slots in them (padding: page 0, slot 0)."""
    c, pos, seq = s["case"], s["pos"].long(), s["seq"].long()
    live = pos >= 0
    at = torch.where(live, pos, torch.zeros_like(pos))
    return live, s["table"][seq, at // c["ps"]].long(), at % c["ps"]


def _stored(s, page, what, slot=None):
    """What the pool holds of pages (and slots) as fp32: [rows][hkv][ps][dh], or [rows][hkv][dh]."""
    c, heads = s["case"], torch.arange(s["case"]["hkv"], device="cuda")
    pick = (lambda t: t[page, what]) if slot is None else (lambda t: t[page[:, None], what, heads, slot[:, None]])
    if c["cache"] == "fp16":
        return pick(s["pool"]).float()
    q, d = (pick(t).float() for t in _pool_parts(c, s["pool"]))
    return (q.unflatten(-1, (-1, 32)) * d[..., None]).flatten(-2)


def _plain_append(s):
    c = s["case"]
    rows, hq, hkv, dh = c["rows"], c["hq"], c["hkv"], c["dh"]
    live, page, slot = _place(s)
    cs = s["rope"][torch.where(live, s["pos"], torch.zeros_like(s["pos"])).long()]
    proj, kw = s["proj"], hkv * dh
    q = _norm_rotate(proj[:, : 2 * hq * dh].view(rows, hq, 2, dh)[:, :, 0], s["gq"], cs)
    k = _norm_rotate(proj[:, 2 * hq * dh:2 * hq * dh + kw].view(rows, hkv, dh), s["gk"], cs)
    v = proj[:, 2 * hq * dh + kw:].view(rows, hkv, dh)
    heads, at, to = torch.arange(hkv, device="cuda"), slot[live][:, None], page[live][:, None]
    for what, x in ((0, k[live]), (1, v[live])):
        if c["cache"] == "fp16":
            s["pool"][to, what, heads, at] = x.half()
        else:
            codes, d = _quantize(x.unflatten(-1, (-1, 32)))
            qs, ds = _pool_parts(c, s["pool"])
            qs[to, what, heads, at] = codes.flatten(-2).to(torch.int8)
            ds[to, what, heads, at] = _round11(d).half()  # an 11-bit value: exact
    # the page's bounds over its slots up to the last one this call wrote
    last = torch.full((s["pool"].shape[0],), -1, device="cuda").scatter_reduce(0, page[live], slot[live], "amax")
    seen = (torch.arange(c["ps"], device="cuda") <= last[page][:, None])[:, None, :, None]
    keys = _stored(s, page, 0)
    hi, lo = torch.where(seen, keys, -math.inf).amax(2), torch.where(seen, keys, math.inf).amin(2)
    codes, d = _quantize(torch.cat([hi, -lo], -1))
    qs, ds = _summary_parts(c, s["summaries"])
    qs[page[live]] = codes[live].unflatten(-1, (2, dh)).to(torch.int8)
    ds[page[live]] = _round11(d)[live]
    s["q_rot"].copy_(torch.where(live[:, None, None], q, s["q_rot"]))
    bounds = (codes * _round11(d)[..., None]).unflatten(-1, (2, dh))
    back = [_stored(s, page, 0, slot), _stored(s, page, 1, slot), bounds[:, :, 0], -bounds[:, :, 1]]
    for to, x in zip(s["back"], back):
        to.copy_(torch.where(live[:, None], x.reshape(rows, kw), to.float()))
    return [s["q_rot"], *s["back"]]


def _plain_read(s):
    live, page, slot = _place(s)
    for what, to in enumerate(s["back"]):
        to.copy_(torch.where(live[:, None], _stored(s, page, what, slot).flatten(1), to.float()))
    return s["back"]


def _plain_select(s):
    """Sums of products of 8-bit codes stay under 2^24: exact in fp32, in any order; the scores have at most 44 bits."""
    c, seq, pos = s["case"], s["seq"].long(), s["pos"].long()
    rows, hkv, dh, n, top = c["rows"], c["hkv"], c["dh"], _max_pages(c), c["top"]
    codes, d = _quantize(s["q_rot"].view(rows, hkv, -1, dh))
    split = torch.cat([codes.clamp(min=0), (-codes).clamp(min=0)], -1)
    bounds, scale = _summary_parts(c, s["summaries"])
    at = s["table"].long()
    b = bounds[at].float().flatten(-2).permute(0, 2, 3, 1).contiguous()[seq]  # [rows][hkv][2 dh][pages]
    score = (torch.matmul(split, b).double() * _round11(d).double()[..., None]).amax(2) * scale[at].double().transpose(1, 2)[seq]
    visible = (pos // c["ps"] + 1)[:, None, None]
    page = torch.arange(n, device="cuda")
    score = torch.where((page < 1) | (page >= visible - 2), math.inf, score)
    score = torch.where(page >= visible, -math.inf, score)
    idx = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :top]
    idx = torch.sort(torch.where(idx < visible, idx, n), -1).values
    idx = torch.where(idx < n, idx, -1).int()
    s["selected"][..., : idx.shape[-1]] = idx
    return s["selected"]


def _plain_attend(s):
    c, seq, pos = s["case"], s["seq"].long(), s["pos"].long()
    rows, hq, hkv, dh, ps, top = c["rows"], c["hq"], c["hkv"], c["dh"], c["ps"], c["top"]
    idx = s["selected"].long()
    page = s["table"].long()[seq[:, None, None], idx.clamp(min=0)]
    heads = torch.arange(hkv, device="cuda")[None, :, None]

    def gathered(what):
        if c["cache"] == "fp16":
            return s["pool"][page, what, heads].float().view(rows, hkv, top * ps, dh)
        q, d = (t[page, what, heads].float() for t in _pool_parts(c, s["pool"]))
        return (q.unflatten(-1, (-1, 32)) * d[..., None]).view(rows, hkv, top * ps, dh)

    seen = (idx[..., None] >= 0) & (idx[..., None] * ps + torch.arange(ps, device="cuda") <= pos[:, None, None, None])
    seen = seen.view(rows, hkv, 1, top * ps)
    q = s["q_rot"].view(rows, hkv, hq // hkv, dh)
    w = torch.matmul(gathered(0), q.transpose(-1, -2).contiguous()).transpose(-1, -2) / math.sqrt(dh)
    w = torch.where(seen, w, -math.inf)
    w = torch.where(seen, torch.exp(w - w.amax(-1, keepdim=True)), torch.zeros_like(w))
    total = w.sum(-1, keepdim=True)
    w = w / torch.where(total > 0, total, torch.ones_like(total))
    o = torch.matmul(w.contiguous(), gathered(1)).view(rows, hq, dh)
    gate = s["proj"][:, : 2 * hq * dh].view(rows, hq, 2, dh)[:, :, 1]
    o = (o / (1 + torch.exp(-gate))).reshape(rows, hq * dh)
    s["out"].copy_(torch.where(pos[:, None] >= 0, o, s["out"]))
    return s["out"]


PLAIN = {"append": _plain_append, "read": _plain_read, "select": _plain_select, "attend": _plain_attend}


def run(state):
    return _run_own(state) if own else PLAIN[state["case"]["kind"]](state)


# ---- the definition in 64 bits ---------------------------------------------------------------------------
def _codes64(x):
    """Symmetric 8-bit codes of the last axis in 64 bits, their step rounded to 11 bits."""
    d = x.abs().amax(-1, keepdim=True) / 127
    m, e = torch.frexp(d)
    step = torch.floor(m * 2048 + 0.5) / 2048 * torch.exp2(e.double())
    v = torch.where(d > 0, x / torch.where(d > 0, d, 1.0), 0.0)
    return torch.sign(v) * torch.floor(v.abs() + 0.5), step


def _pool64(c, s):
    """[page][2][hkv][ps][dh] float64"""
    if c["cache"] == "fp16":
        return s["pool"].double()
    q, d = _pool_parts(c, s["pool"])
    return (q.double().unflatten(-1, (-1, 32)) * d.double()[..., None]).flatten(-2)


def _exact_append(c, s):
    rows, hq, hkv, dh, ps = c["rows"], c["hq"], c["hkv"], c["dh"], c["ps"]
    pool = _pool64(c, s)
    pos, seq, p = s["pos"].tolist(), s["seq"].tolist(), s["proj"].double()
    live = [r for r in range(rows) if pos[r] >= 0]
    at = torch.tensor([pos[r] for r in live], device="cuda")
    ang = s["rope"].double()[at]

    def turned(x, gamma):  # as complex numbers, plane i = channels i and i + dh/2
        x = x * gamma.double() * torch.rsqrt(x.square().sum(-1, keepdim=True) / dh + EPS)
        z = torch.complex(x[..., : dh // 2], x[..., dh // 2:]) * torch.complex(ang[..., 0], ang[..., 1])[:, None]
        return torch.cat([z.real, z.imag], -1)

    q = torch.zeros(rows, hq, dh, dtype=torch.float64, device="cuda")
    q[live] = turned(p[live, : 2 * hq * dh].reshape(-1, hq, 2 * dh)[..., :dh], s["gq"])
    kv = [turned(p[live, 2 * hq * dh:2 * hq * dh + hkv * dh].reshape(-1, hkv, dh), s["gk"]), p[live, 2 * hq * dh + hkv * dh:].reshape(-1, hkv, dh)]
    if c["cache"] == "fp16":
        kv = [x.half().double() for x in kv]
    else:
        kv = [(lambda qd: (qd[0] * qd[1]).flatten(-2))(_codes64(x.unflatten(-1, (-1, 32)))) for x in kv]
    back = [torch.zeros(rows, hkv * dh, dtype=torch.float64, device="cuda") for _ in range(4)]
    table, end = s["table"].tolist(), {}
    for i, r in enumerate(live):
        page = table[seq[r]][pos[r] // ps]
        pool[page, 0, :, pos[r] % ps], pool[page, 1, :, pos[r] % ps] = kv[0][i], kv[1][i]
        end[page] = max(end.get(page, 0), pos[r] % ps + 1)
        back[0][r], back[1][r] = kv[0][i].flatten(), kv[1][i].flatten()
    for page, n in end.items():
        keys = pool[page, 0, :, :n]
        codes, step = _codes64(torch.cat([keys.amax(1), -keys.amin(1)], -1))
        here = [r for r in live if table[seq[r]][pos[r] // ps] == page]
        back[2][here], back[3][here] = (codes * step)[:, :dh].flatten(), -(codes * step)[:, dh:].flatten()
    return [q, *back]


def _exact_read(c, s):
    pool, out = _pool64(c, s), []
    pos, seq = s["pos"].long(), s["seq"].long()
    live = pos >= 0
    for what in (0, 1):
        rows = torch.zeros(c["rows"], c["hkv"] * c["dh"], dtype=torch.float64, device="cuda")
        rows[live] = pool[s["table"][seq[live], pos[live] // c["ps"]].long(), what, :, pos[live] % c["ps"]].flatten(1)
        out.append(rows)
    return out


def _exact_attend(c, s):
    hq, hkv, dh, ps = c["hq"], c["hkv"], c["dh"], c["ps"]
    grp, pos, seq = hq // hkv, s["pos"].tolist(), s["seq"].tolist()
    table, q, gate = s["table"].long(), s["q_rot"].double(), s["proj"].double()
    out = torch.zeros(c["rows"], hq * dh, dtype=torch.float64, device="cuda")
    parts = None if c["cache"] == "fp16" else _pool_parts(c, s["pool"])
    for r in range(c["rows"]):
        if pos[r] < 0:
            continue
        idx = s["selected"][r].long()
        phys, head = table[seq[r]][idx.clamp(min=0)], torch.arange(hkv, device="cuda")[:, None]

        def of(what):
            if parts is None:
                return s["pool"][phys, what, head].double().flatten(1, 2)
            return (parts[0][phys, what, head].double().unflatten(-1, (-1, 32)) * parts[1][phys, what, head].double()[..., None]).flatten(-2).flatten(1, 2)

        k, v = of(0), of(1)
        hide = ((idx < 0)[..., None] | (idx[..., None] * ps + torch.arange(ps, device="cuda") > pos[r])).flatten(1)
        w = torch.bmm(q[r].view(hkv, grp, dh), k.transpose(1, 2).contiguous()) * dh ** -0.5
        w = torch.softmax(w.masked_fill(hide[:, None], -math.inf), -1).nan_to_num(0.0)
        g = gate[r, : 2 * hq * dh].view(hq, 2, dh)[:, 1]
        out[r] = (torch.bmm(w, v).view(hq, dh) * torch.sigmoid(g)).flatten()
    return out


def exact(case, seed):
    if case["kind"] == "select":
        return None  # page indexes: whole numbers, compared as they are
    return {"append": _exact_append, "read": _exact_read, "attend": _exact_attend}[case["kind"]](case, prepare(case, seed))


# ---- what a pass cannot do without -------------------------------------------------------------------------
def _sequences(c):
    """(first position, rows) of each sequence, as _rows lays them out (a batch's lengths at their longest)."""
    rows, seqs, past = c["rows"], c["seqs"], c["past"]
    if c.get("decode"):
        return [(past, 1)] * seqs
    count = [0] * seqs
    for r in range(rows - (rows // 10 if seqs > 1 else 0)):
        count[r * seqs // rows] += 1
    return [(past - i * (past // 4), n) for i, n in enumerate(count)]


def work(case):
    c = case
    hkv, dh, ps, rows, kind = c["hkv"], c["dh"], c["ps"], c["rows"], c["kind"]
    kw = hkv * dh
    per = 34 / 32 if c.get("cache") == "q8" else 2.0
    seqs = _sequences(c)
    live = sum(n for _, n in seqs)
    if kind == "read":
        return {"bytes": int(2 * live * kw * (per + (2 if c["f16"] else 4))), "flops": 2 * live * kw}
    hq = c["hq"]
    if kind == "append":  # projections in; queries, rows and touched pages' summaries out; then the rows and bounds read back
        touched = sum((f + n - 1) // ps - f // ps + 1 for f, n in seqs if n)
        old = sum(f % ps for f, n in seqs if n) * kw * per
        return {"bytes": int(live * (4 * (2 * hq * dh + 2 * kw) + 4 * kw * per + 8 * kw) + old + 2 * touched * _summary_bytes(c)), "flops": 12 * live * (hq + 2 * hkv) * dh}
    pages = [[(f + i) // ps + 1 for i in range(n)] for f, n in seqs]
    if kind == "select":
        seen = sum(max(p, default=0) for p in pages)
        return {"bytes": seen * _summary_bytes(c) + live * (4 * hq * dh + 4 * hkv * c["top"]), "flops": 4 * dh * hq * sum(map(sum, pages))}
    keys = sum(min(p, c["top"]) * ps for q in pages for p in q)  # selected positions, over all rows
    once = sum(min(f + n, min(c["top"], (f + n - 1) // ps + 1) * ps * n) for f, n in seqs if n)  # of them, distinct ones at most
    return {"bytes": int(2 * once * kw * per + live * (12 * hq * dh + 4 * hkv * c["top"])), "flops": 4 * keys * hq * dh}
