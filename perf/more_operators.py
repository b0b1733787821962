"""The 4-bit paged cache and the token log probabilities, case by case: rows appended
to 4-bit pages (query / key norms, rotary positions of one or three axes,
quantization), attention over those pages with and without a sliding window whose
first tokens stay visible, and log probabilities of given tokens with entropy and
the most likely alternatives.

Sizes are those of the repository's configurations: an ~8B hybrid (32 query heads
over 8 K/V heads of 128, a vocabulary of 151936), the 256-wide heads of the Qwen
3.5 9B one (16 over 4), the vocabulary of 262144 of the Gemma one, pages of 64
positions, up to sixteen sequences decoded together.

A block of 32 neighbouring channels of a stored row has a step d of 8 significant
bits, held as fp16, and codes c in -8 .. 7; it stands for c * d, which fp16 holds
exactly. Sixteen positions of one head are a record of 9 * dh bytes, codes first:
see _values.
"""
import functools
import math

import torch

own = False

EPS = 1e-6
ROPE_BASE = 1e6
ROPE_POSITIONS = 32768
TILE = 16  # positions of a record


def listed():
    return [
        # One new token of one chat enters its 4-bit cache: the smallest call, latency and launches count.
        {"name": "append_token", "kind": "append", "hq": 32, "hkv": 8, "dh": 128, "ps": 64, "seqs": 1, "rows": 1, "past": 5000, "axes": 1, "decode": True},
        # A prompt's chunk with an image in it, after a first chunk that ended inside a page: time, height and width rotate their own planes.
        {"name": "append_prompt_image", "kind": "append", "hq": 32, "hkv": 8, "dh": 128, "ps": 64, "seqs": 1, "rows": 1000, "past": 1000, "axes": 3, "decode": False},
        # One token of a chat that has just begun.
        {"name": "attend_token_short", "kind": "attend", "hq": 32, "hkv": 8, "dh": 128, "ps": 64, "seqs": 1, "rows": 1, "past": 300, "window": 0, "sinks": 0, "decode": True},
        # One token of a 32k chat, over all of it.
        {"name": "attend_token", "kind": "attend", "hq": 32, "hkv": 8, "dh": 128, "ps": 64, "seqs": 1, "rows": 1, "past": 32000, "window": 0, "sinks": 0, "decode": True},
        # Sixteen such chats decoded together: what the 4-bit cache is for.
        {"name": "attend_batch", "kind": "attend", "hq": 32, "hkv": 8, "dh": 128, "ps": 64, "seqs": 16, "rows": 16, "past": 32000, "window": 0, "sinks": 0, "decode": True},
        # The same chats in a layer with a sliding window and four tokens that stay.
        {"name": "attend_batch_window", "kind": "attend", "hq": 32, "hkv": 8, "dh": 128, "ps": 64, "seqs": 16, "rows": 16, "past": 32000, "window": 4096, "sinks": 4, "decode": True},
        # Eight sequences with the 256-wide heads.
        {"name": "attend_batch_wide", "kind": "attend", "hq": 16, "hkv": 4, "dh": 256, "ps": 64, "seqs": 8, "rows": 8, "past": 16000, "window": 0, "sinks": 0, "decode": True},
        # A chunk of a long prompt: the largest.
        {"name": "attend_prompt", "kind": "attend", "hq": 32, "hkv": 8, "dh": 128, "ps": 64, "seqs": 1, "rows": 500, "past": 16001, "window": 0, "sinks": 0, "decode": False},
        # Chunks of three prompts, and some padding, in a layer with a window.
        {"name": "attend_prompt_window", "kind": "attend", "hq": 32, "hkv": 8, "dh": 128, "ps": 64, "seqs": 3, "rows": 1000, "past": 8000, "window": 1024, "sinks": 16, "decode": False},
        # A decoded token's log probability with the twenty alternatives that serving interfaces offer.
        {"name": "logprobs_token", "kind": "logprobs", "rows": 1, "vocab": 151936, "top": 20, "temp": 1.0},
        # Sixteen decoded tokens of a large vocabulary at a sampling temperature.
        {"name": "logprobs_batch", "kind": "logprobs", "rows": 16, "vocab": 262144, "top": 5, "temp": 0.7},
        # A prompt is scored: every position's own token, and the best one.
        {"name": "logprobs_prompt", "kind": "logprobs", "rows": 1000, "vocab": 151936, "top": 1, "temp": 1.0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the same ranges: single tokens of one to sixteen sequences, chunks of one to three prompts (past one, the
    last rows are padding), every head width, group and page size, windows with and without tokens that stay, contexts
    from a few tokens to 32k; rows of logits from one to a thousand over small and large vocabularies."""
    kind = rng.choice(["append", "append", "attend", "attend", "attend", "attend", "logprobs", "logprobs"])
    if kind == "logprobs":
        vocab = rng.choice([151936, 248320, 262144, _log(rng, 100, 200000)])
        rows = _log(rng, 1, min(1000, 120_000_000 // vocab))
        return {"kind": kind, "rows": rows, "vocab": vocab, "top": rng.choice([0, 1, 5, 20, rng.randint(0, 64)]), "temp": rng.choice([1.0, 1.0, 0.7, 1.3])}
    dh = rng.choice([128, 128, 256])
    hq, hkv = rng.choice([(32, 8), (32, 8), (16, 4), (8, 2), (16, 2), (24, 8), (8, 8)])
    c = {"kind": kind, "hq": hq, "hkv": hkv, "dh": dh, "ps": rng.choice([64, 64, 64, 16, 32, 48, 128]), "decode": rng.random() < 0.6}
    if c["decode"]:
        c["seqs"] = c["rows"] = rng.choice([1, 2, rng.randint(3, 16)])
        c["past"] = _log(rng, 1, 32000)
    else:
        c["seqs"] = rng.randint(1, 3)
        c["rows"] = _log(rng, 4, 1000 if kind == "append" else 400)
        c["past"] = _log(rng, 1, 16000)
    if kind == "append":
        c["axes"] = rng.choice([1, 3])
        c["past"] = min(c["past"], 30000)
    else:
        c["window"] = rng.choice([0, 0, _log(rng, 1, 8192)])
        c["sinks"] = rng.choice([0, 4, rng.randint(1, 100)]) if c["window"] else 0
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


def _plane_axes(c):
    """The axis of each plane, taking turns (time, height, width, time, ...); one axis: all 0."""
    return [i % c["axes"] for i in range(c["dh"] // 2)]


def _sequences(c):
    """(first position, rows) of each sequence. Decoded tokens: a row each, lengths differing by up to an eighth."""
    rows, seqs, past = c["rows"], c["seqs"], c["past"]
    if c["decode"]:
        return [(past - i * 37 % max(1, past // 8), 1) for i in range(seqs)]
    live = rows - (rows // 10 if seqs > 1 else 0)
    count = [sum(r * seqs // rows == i for r in range(live)) for i in range(seqs)]
    return [(past - i * (past // 4), n) for i, n in enumerate(count)]


def _rows(c):
    """Each row's sequence and position; padding rows, at the end, have position -1."""
    seq, pos = [], []
    for i, (first, n) in enumerate(_sequences(c)):
        seq += [i] * n
        pos += range(first, first + n)
    left = c["rows"] - len(seq)
    return torch.tensor(seq + [c["seqs"] - 1] * left, device="cuda"), torch.tensor(pos + [-1] * left, device="cuda")


def _rope_positions(c, seq, pos):
    """Rotary positions [axes][rows]. A chunk holds an image of 32 columns in its second quarter: its tokens stand at one
    time, a height and a width each, and what follows goes on behind the largest of them. A decoded token's image lies behind it."""
    first = torch.tensor([f for f, _ in _sequences(c)], device="cuda")[seq]
    count = torch.tensor([n for _, n in _sequences(c)], device="cuda")[seq]
    live = pos >= 0
    if c["decode"]:
        at = pos - pos // 3
        p = torch.stack([at] * c["axes"])
    else:
        i, a = pos - first, count // 4  # the image: rows a .. 2 a of the sequence
        inside = (i >= a) & (i < 2 * a)
        behind = torch.maximum((a - 1).clamp(min=0) // 32, (a - 1).clamp(max=31)) + 1
        text = torch.where(i >= 2 * a, first + i - a + behind.clamp(max=a), first + i)
        offset = [torch.zeros_like(i), (i - a) // 32, (i - a) % 32]
        p = torch.stack([torch.where(inside, first + a + offset[k], text) for k in range(c["axes"])])
    return torch.where(live, p, torch.full_like(p, -1)).int()


def _max_pages(c):
    return -(-max(f + n for f, n in _sequences(c)) // c["ps"])


def _pool(c, g):
    """Records of 4-bit pages [page][2 = K, V][hkv][ps / 16][9 * dh bytes]: codes as quantized rows have them, steps of 8 bits."""
    n, hkv, ps, dh = c["seqs"] * _max_pages(c), c["hkv"], c["ps"], c["dh"]
    pool = torch.empty(n, 2, hkv, ps // TILE, 9 * dh, dtype=torch.uint8, device="cuda")
    nibble = lambda: (_randn(g, *pool.shape[:-1], 8 * dh, dtype=torch.float16) * 3.5 + 8).round_().clamp_(0, 15).to(torch.uint8)  # noqa: E731
    pool[..., : 8 * dh] = nibble()
    pool[..., : 8 * dh] |= nibble() << 4
    steps = (torch.rand(*pool.shape[:-1], dh // 2, device="cuda", generator=g) * 0.12 + 0.2).half().view(torch.int16)
    sign = torch.randint(0, 2, steps.shape, device="cuda", generator=g, dtype=torch.int16) * -32768
    pool[..., 8 * dh:] = ((steps & -8) | sign).view(torch.uint8)
    return pool


def prepare(case, seed):
    c, g = case, _gen(seed)
    kind, rows = c["kind"], c["rows"]
    if kind == "logprobs":
        # logits as an fp16 head gives them: ties are common; the tokens are sampled from them, with a few padded rows in batches
        x = (_randn(g, rows, c["vocab"]) * 2.5 + 6.0 * (_randn(g, rows, c["vocab"]) > 4.0)).half().float()
        noise = torch.rand(rows, c["vocab"], device="cuda", generator=g).clamp_(min=1e-20).log_().neg_().log_().neg_()
        token = noise.add_(x / c["temp"]).argmax(-1).int()
        token[rows - rows // 50:] = -1
        s = {"case": c, "logits": x, "token": token}
        s["logprob"], s["entropy"] = torch.zeros(rows, device="cuda"), torch.zeros(rows, device="cuda")
        s["top_ids"] = torch.full((rows, c["top"]), -1, dtype=torch.int32, device="cuda")
        s["top_logprobs"] = torch.zeros(rows, c["top"], device="cuda")
    else:
        hq, hkv, dh = c["hq"], c["hkv"], c["dh"]
        seq, pos = _rows(c)
        s = {"case": c, "pos": pos.int(), "seq": seq.int(), "proj": _randn(g, rows, 2 * (hq + hkv) * dh)}  # [q | gate] pairs, k, v
        n = _max_pages(c)
        s["table"] = torch.randperm(c["seqs"] * n, device="cuda", generator=g).to(torch.int32).view(c["seqs"], n)
        s["pool"] = _pool(c, g)
        if kind == "append":
            s["gq"], s["gk"], s["rope"] = 1 + 0.1 * _randn(g, dh), 1 + 0.1 * _randn(g, dh), _rope(dh)
            s["rope_pos"] = _rope_positions(c, seq, pos)
            s["q_rot"] = torch.zeros(rows, hq, dh, device="cuda")
            s["back"] = [torch.zeros(rows, hkv * dh, dtype=torch.float16, device="cuda") for _ in range(2)]
        else:  # attention takes normalised, rotated queries; consecutive rows' are alike
            s["q_rot"] = 0.8 * _randn(g, c["seqs"], hq, dh)[seq] + 0.6 * _randn(g, rows, hq, dh)
            s["out"] = torch.zeros(rows, hq * dh, device="cuda")
    if own:
        _plan(s)
    return s


# ---- the framework's calls -----------------------------------------------------------------------------
def _plan(s):
    """The argument structs and workspace that a program keeps beside its cache or its logits."""
    import ctypes

    from hero_amd._lib import AttnDecodeArgs, AttnQ4Args, KvReadArgs, lib

    c = s["case"]
    p = lambda name: s[name].data_ptr() if name in s else None  # noqa: E731
    if c["kind"] == "logprobs":
        work = lib.hero_logprobs_work_bytes(c["rows"], c["vocab"], c["top"])
        s["work"] = torch.empty(max(16, work), dtype=torch.uint8, device="cuda")
        return
    hq, hkv, dh, n, rows = c["hq"], c["hkv"], c["dh"], _max_pages(c), c["rows"]
    row_seq = None if c["decode"] else s["seq"].data_ptr()
    a = AttnDecodeArgs(p("proj"), 2 * (hq + hkv) * dh, 2 * hq * dh, 2 * hq * dh + hkv * dh, p("gq"), p("gk"), EPS, p("rope"), None, None, 0, p("pos"), None, p("q_rot"),
                       1.0 / math.sqrt(dh), c.get("window", 0), None, p("out"), rows, hq, hkv, dh)
    work = 0
    if c["kind"] == "attend":
        work = lib.hero_attn_q4_work_bytes(rows, hq, hkv, dh, n * c["ps"], c["window"], c["sinks"])
    s["work"] = torch.empty(max(16, work), dtype=torch.uint8, device="cuda")
    axes = (ctypes.c_uint8 * 128)(*(_plane_axes(c) if c["kind"] == "append" else []))
    s["args"] = AttnQ4Args(a, p("pool"), c["seqs"] * n, p("table"), c["ps"], n, row_seq, c["seqs"], c.get("sinks", 0), ROPE_POSITIONS, p("rope_pos"), c.get("axes", 1), axes,
                           p("work"), work)
    if c["kind"] == "append":
        s["read"] = KvReadArgs(p("pool"), p("table"), c["ps"], n, 0, c["seqs"] * n, None, p("pos"), row_seq, rows, c["seqs"], hkv, dh, 1,
                               s["back"][0].data_ptr(), s["back"][1].data_ptr(), None, None)


def _run_own(s):
    from hero_amd._lib import check, lib

    c, stream = s["case"], torch.cuda.current_stream().cuda_stream
    if c["kind"] == "append":
        check(lib.hero_kv_append_q4(s["args"], stream))
        check(lib.hero_kv_read_q4(s["read"], stream))
        return [s["q_rot"], *s["back"]]
    if c["kind"] == "attend":
        check(lib.hero_attn_q4(s["args"], stream))
        return s["out"]
    at = [s[k].data_ptr() if s[k].numel() else None for k in ("logprob", "entropy", "top_ids", "top_logprobs")]
    check(lib.hero_logprobs(s["logits"].data_ptr(), c["vocab"], c["rows"], c["vocab"], s["token"].data_ptr(), c["temp"], c["top"], *at, s["work"].data_ptr(),
                            s["work"].numel(), stream))
    return [s["logprob"], s["entropy"], s["top_ids"], s["top_logprobs"]]


# ---- the plain forms -----------------------------------------------------------------------------------
def _values(records, what, dh):
    """What records [...][9 * dh] of keys (0) or values (1) stand for, as fp32 [..., 16 positions, dh].

    Keys' codes are [dh / 128][16 positions][4 = b][4 = a][4 bytes]: channel 128 h + 32 a + 8 b + j; the eight four-bit
    fields of a word, lowest first, are j = 0, 2, 4, 6, 1, 3, 5, 7. Steps [16 positions][dh / 32].
    Values' codes are [dh / 128][4 = p][16 = b][4 = i][4 bytes]: position 4 p + i, channel 128 h + b + 16 m, m the field.
    Steps [4 = p][dh / 32][4 = i]. A field holds c + 8."""
    lead, h = records.shape[:-1], dh // 128
    b = records[..., : 8 * dh]
    fields = torch.stack([b & 15, b >> 4], -1).to(torch.float32) - 8
    d = records[..., 8 * dh:].contiguous().view(torch.float16).float()
    n = len(lead)
    if what == 0:
        # [h][position][b][a][2 = odd j][4 = j / 2] -> [position][h][a][b][j / 2][odd j]
        x = fields.view(*lead, h, 16, 4, 4, 2, 4).permute(*range(n), n + 1, n, n + 3, n + 2, n + 5, n + 4).reshape(*lead, 16, dh // 32, 32)
        return (x * d.view(*lead, 16, dh // 32, 1)).flatten(-2)
    # [h][p][b][i][m] -> [p][i][h][m][b]
    x = fields.view(*lead, h, 4, 16, 4, 8).permute(*range(n), n + 1, n + 3, n, n + 4, n + 2).reshape(*lead, 16, dh // 32, 32)
    d = d.view(*lead, 4, dh // 32, 4).transpose(-1, -2).reshape(*lead, 16, dh // 32, 1)
    return (x * d).flatten(-2)


def _quantized(x):
    """Rows [..., dh] in fp32 -> codes + 8 [..., dh / 32, 32] and steps as fp16 [..., dh / 32]."""
    x = torch.where(torch.isnan(x), torch.zeros_like(x), x).clamp(-65280, 65280).unflatten(-1, (-1, 32))
    hi, lo = x.amax(-1), x.amin(-1)
    bits = (torch.where(hi >= -lo, hi, lo) / -8).half().view(torch.int16).int()
    d = ((((bits & 0x7FFF) + 4) & -8) | (bits & 0x8000)).to(torch.int16).view(torch.float16)
    step = d.double()[..., None]  # 64 bits: values next to a border between two codes
    q = torch.where(step != 0, torch.round(x.double() / torch.where(step != 0, step, torch.ones_like(step))), torch.zeros_like(x, dtype=torch.float64))
    return (q.clamp(-8, 7) + 8).to(torch.uint8), d


def _norm_rotate(x, gamma, cs):
    """RMSNorm of each head and the rotation of its planes (i, i + dh/2), in 64 bits as codes are next to borders."""
    x = x.double()
    x = gamma.double() * x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
    lo, hi = x.chunk(2, -1)
    cos, sin = cs[:, None, :, 0].double(), cs[:, None, :, 1].double()
    return torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1).float()


def _plain_append(s):
    c = s["case"]
    rows, hq, hkv, dh, ps = c["rows"], c["hq"], c["hkv"], c["dh"], c["ps"]
    pos, live = s["pos"].long(), s["pos"] >= 0
    at = torch.where(live, pos, torch.zeros_like(pos))
    page, slot = s["table"][s["seq"].long(), at // ps].long(), at % ps
    plane = torch.arange(dh // 2, device="cuda")
    cs = s["rope"][torch.where(live, s["rope_pos"], torch.zeros_like(s["rope_pos"])).long().t()[:, plane % c["axes"]], plane]  # [rows][dh / 2][2]
    proj, kw, h = s["proj"], hkv * dh, dh // 128
    q = _norm_rotate(proj[:, : 2 * hq * dh].view(rows, hq, 2, dh)[:, :, 0], s["gq"], cs)
    k = _norm_rotate(proj[:, 2 * hq * dh:2 * hq * dh + kw].view(rows, hkv, dh), s["gk"], cs)
    v = proj[:, 2 * hq * dh + kw:].view(rows, hkv, dh)
    page, slot, heads = page[live][:, None], slot[live][:, None], torch.arange(hkv, device="cuda")
    tile, i = slot // TILE, slot % TILE
    codes, d = _quantized(k[live])
    f = codes.view(-1, hkv, h, 4, 4, 4, 2)  # [h][a][b][j / 2][odd j] -> [h][b][a][odd j][j / 2]
    f = f.permute(0, 1, 2, 4, 3, 6, 5).reshape(-1, hkv, h, 4, 4, 4, 2)
    s["pool"][:, 0, :, :, : 8 * dh].unflatten(-1, (h, 16, 64)).permute(0, 1, 2, 4, 3, 5)[page, heads, tile, i] = (f[..., 0] | f[..., 1] << 4).reshape(-1, hkv, h, 64)
    s["pool"][:, 0, :, :, 8 * dh:].unflatten(-1, (16, dh // 16))[page, heads, tile, i] = d.contiguous().view(torch.uint8)
    codes, d = _quantized(v[live])
    f = codes.view(-1, hkv, h, 4, 2, 16)  # [h][m / 2][odd m][b] -> [h][b][m / 2]
    f = (f[..., 0, :] | f[..., 1, :] << 4).transpose(-1, -2)
    s["pool"][:, 1, :, :, : 8 * dh].unflatten(-1, (h, 4, 16, 4, 4)).permute(0, 1, 2, 4, 6, 3, 5, 7)[page, heads, tile, i // 4, i % 4] = f
    s["pool"][:, 1, :, :, 8 * dh:].unflatten(-1, (4, dh // 32, 4, 2)).permute(0, 1, 2, 3, 5, 4, 6)[page, heads, tile, i // 4, i % 4] = d.view(torch.uint8).unflatten(-1, (-1, 2))
    s["q_rot"].copy_(torch.where(live[:, None, None], q, s["q_rot"]))
    for what, to in enumerate(s["back"]):
        x = _values(s["pool"][page, what, heads, tile], what, dh)  # [live][hkv][16][dh]
        to[live] = x[torch.arange(x.shape[0], device="cuda")[:, None], heads, i].flatten(1).half()
    return [s["q_rot"], *s["back"]]


def _seen_pages(c):
    """Per sequence the logical pages that its rows may see: those of the tokens that stay, and of the windows; equally
    many for each, padded with -1."""
    out = []
    for first, n in _sequences(c):
        last = (first + max(n, 1) - 1) // c["ps"]
        lo = max(0, first - c["window"] + 1) // c["ps"] if c["window"] else 0
        stay = -(-c["sinks"] // c["ps"]) if c["window"] else 0
        out.append([p for p in range(min(stay, lo))] + list(range(lo, last + 1)))
    most = max(map(len, out))
    return torch.tensor([p + [-1] * (most - len(p)) for p in out], device="cuda")


def _plain_attend(s):
    c, seq, pos = s["case"], s["seq"].long(), s["pos"].long()
    rows, hq, hkv, dh, ps, seqs = c["rows"], c["hq"], c["hkv"], c["dh"], c["ps"], c["seqs"]
    grp, counts = hq // hkv, [n for _, n in _sequences(c)]
    lead = torch.tensor([sum(counts[:i]) for i in range(seqs)], device="cuda")
    most = max(max(counts), 1)
    # the rows by sequences [seqs][most], past the last one of a sequence any other
    row = (lead[:, None] + torch.arange(most, device="cuda")).clamp(max=rows - 1)
    real = torch.arange(most, device="cuda") < torch.tensor(counts, device="cuda")[:, None]
    seen = _seen_pages(c)
    phys = s["table"][torch.arange(seqs, device="cuda")[:, None], seen.clamp(min=0)].long()
    k = _values(s["pool"][phys, 0], 0, dh).permute(0, 2, 1, 3, 4, 5).reshape(seqs * hkv, -1, dh)
    q = s["q_rot"][row].view(seqs, most, hkv, grp, dh).permute(0, 2, 1, 3, 4).reshape(seqs * hkv, most * grp, dh)
    w = torch.bmm(q, k.transpose(1, 2).contiguous()).view(seqs, hkv, most, grp, -1) / math.sqrt(dh)
    del k
    key = (seen[:, :, None] * ps + torch.arange(ps, device="cuda")).flatten(1)[:, None]  # [seqs][1][keys]
    at = pos[row][:, :, None]
    ok = (seen >= 0).repeat_interleave(ps, 1)[:, None] & (key <= at) & real[:, :, None]
    if c["window"]:
        ok = ok & ((key > at - c["window"]) | (key < c["sinks"]))
    ok = ok[:, None, :, None]
    w = torch.where(ok, w, -math.inf)
    w = torch.where(ok, torch.exp(w - w.amax(-1, keepdim=True)), torch.zeros_like(w))
    total = w.sum(-1, keepdim=True)
    w = (w / torch.where(total > 0, total, torch.ones_like(total))).view(seqs * hkv, most * grp, -1)
    v = _values(s["pool"][phys, 1], 1, dh).permute(0, 2, 1, 3, 4, 5).reshape(seqs * hkv, -1, dh)
    o = torch.bmm(w, v).view(seqs, hkv, most, grp, dh).permute(0, 2, 1, 3, 4).reshape(seqs, most, hq, dh)
    gate = s["proj"][:, : 2 * hq * dh].view(rows, hq, 2, dh)[:, :, 1][row]
    o = (o / (1 + torch.exp(-gate))).reshape(seqs, most, hq * dh)
    s["out"][row[real]] = o[real]
    return s["out"]


def _plain_logprobs(s):
    c, x, token = s["case"], s["logits"], s["token"].long()
    rows, vocab, top = c["rows"], c["vocab"], c["top"]
    live = (token >= 0) & (token < vocab)
    z = x / c["temp"]
    best = z.amax(-1, keepdim=True)
    z = z - best
    e = torch.exp(z)
    total = e.sum(-1, keepdim=True)
    log_total = torch.log(total)
    own_z = z.gather(1, torch.where(live, token, torch.zeros_like(token))[:, None])
    s["logprob"].copy_(torch.where(live, (own_z - log_total)[:, 0], s["logprob"]))
    s["entropy"].copy_(torch.where(live, (log_total - (e * z).sum(-1, keepdim=True) / total)[:, 0], s["entropy"]))
    if top:
        bits = (x + 0.0).view(torch.int32).long()  # -0 and 0 are one logit
        key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits) * (1 << 32) + (vocab - 1 - torch.arange(vocab, device="cuda"))
        ids = vocab - 1 - (torch.topk(key, top, dim=-1, sorted=True).values & 0xFFFFFFFF)
        s["top_ids"].copy_(torch.where(live[:, None], ids.int(), s["top_ids"]))
        s["top_logprobs"].copy_(torch.where(live[:, None], z.gather(1, ids) - log_total, s["top_logprobs"]))
    return [s["logprob"], s["entropy"], s["top_ids"], s["top_logprobs"]]


PLAIN = {"append": _plain_append, "attend": _plain_attend, "logprobs": _plain_logprobs}


def run(state):
    return _run_own(state) if own else PLAIN[state["case"]["kind"]](state)


# ---- the definition in 64 bits ---------------------------------------------------------------------------
def _block64(x):
    """What blocks [..., 32] in 64 bits stand for once stored."""
    top, low = x.max(-1).values, x.min(-1).values
    m = -torch.where(top + low >= 0, top, low) / 8
    d = m.half().double()
    f, e = torch.frexp(d)
    scale = torch.exp2((e.double() - 8).clamp(min=-21))  # 8 bits, or multiples of 2^-21
    d = torch.sign(d) * torch.floor(d.abs() / scale + 0.5) * scale
    q = torch.where(d[..., None] != 0, x / torch.where(d != 0, d, 1.0)[..., None], 0.0)
    return torch.round(q).clamp(-8, 7) * d[..., None]


def _exact_append(c, s):
    rows, hq, hkv, dh = c["rows"], c["hq"], c["hkv"], c["dh"]
    live = torch.nonzero(s["pos"] >= 0)[:, 0]
    p, kw = s["proj"].double()[live], hkv * dh
    ang = torch.stack([s["rope"][s["rope_pos"][a][live].long(), i] for i, a in enumerate(_plane_axes(c))], 1).double()
    turn = torch.complex(ang[..., 0], ang[..., 1])[:, None]

    def turned(x, gamma):  # as complex numbers, plane i = channels i and i + dh/2
        x = x * gamma.double() * torch.rsqrt(x.square().sum(-1, keepdim=True) / dh + EPS)
        z = torch.complex(x[..., : dh // 2], x[..., dh // 2:]) * turn
        return torch.cat([z.real, z.imag], -1)

    q = torch.zeros(rows, hq, dh, dtype=torch.float64, device="cuda")
    q[live] = turned(p[:, : 2 * hq * dh].reshape(-1, hq, 2 * dh)[..., :dh], s["gq"])
    out = [q]
    for x in (turned(p[:, 2 * hq * dh:2 * hq * dh + kw].reshape(-1, hkv, dh), s["gk"]).float().double(), p[:, 2 * hq * dh + kw:].reshape(-1, hkv, dh)):
        y = torch.zeros(rows, kw, dtype=torch.float64, device="cuda")
        y[live] = _block64(x.unflatten(-1, (-1, 32))).flatten(1)
        out.append(y)
    return out


def _places(dh, what):
    """For each (position of a record, channel): the byte of its code and whether it is the upper half, and its step's index."""
    byte, high, step = [], [], []
    for i in range(16):
        for ch in range(dh):
            h, r = divmod(ch, 128)
            if what == 0:
                a, b, j = r // 32, r // 8 % 4, r % 8
                field = j // 2 + 4 * (j % 2)
                word = ((h * 16 + i) * 4 + b) * 4 + a
                step.append(i * (dh // 32) + ch // 32)
            else:
                field, word = r // 16, ((h * 4 + i // 4) * 16 + r % 16) * 4 + i % 4
                step.append((i // 4 * (dh // 32) + ch // 32) * 4 + i % 4)
            byte.append(4 * word + field // 2)
            high.append(field % 2)
    t = lambda v: torch.tensor(v, device="cuda")  # noqa: E731
    return t(byte), t(high), t(step)


def _exact_attend(c, s):
    hq, hkv, dh, ps = c["hq"], c["hkv"], c["dh"], c["ps"]
    grp, out = hq // hkv, torch.zeros(c["rows"], hq * dh, dtype=torch.float64, device="cuda")
    places, r0 = [_places(dh, w) for w in (0, 1)], 0
    for i, (first, n) in enumerate(_sequences(c)):
        if not n:
            continue
        pages = s["pool"][s["table"][i].long()]  # [page][2][hkv][tiles][bytes]

        def of(w, g):
            byte, high, step = places[w]
            r = pages[:, w, g].reshape(-1, 9 * dh)
            codes = (r[:, byte].int() >> (4 * high).int()) & 15
            return ((codes - 8).double() * r[:, 8 * dh:].contiguous().view(torch.float16)[:, step].double()).view(-1, dh)[: first + n]

        at = torch.arange(first, first + n, device="cuda")[:, None]
        key = torch.arange(first + n, device="cuda")
        hide = key > at
        if c["window"]:
            hide = hide | ((key <= at - c["window"]) & (key >= c["sinks"]))
        for g in range(hkv):
            q = s["q_rot"][r0:r0 + n, g * grp:(g + 1) * grp].double().reshape(-1, dh)
            w = (q @ of(0, g).t().contiguous() * dh ** -0.5).view(n, grp, -1).masked_fill_(hide[:, None], -math.inf)
            o = (torch.softmax(w, -1).view(n * grp, -1) @ of(1, g)).view(n, grp, dh)
            gate = s["proj"][r0:r0 + n, : 2 * hq * dh].double().view(n, hq, 2, dh)[:, g * grp:(g + 1) * grp, 1]
            out[r0:r0 + n].view(n, hq, dh)[:, g * grp:(g + 1) * grp] = o * torch.sigmoid(gate)
        r0 += n
    return out


def _exact_logprobs(c, s):
    rows, top = c["rows"], c["top"]
    lp, ent = torch.zeros(rows, dtype=torch.float64, device="cuda"), torch.zeros(rows, dtype=torch.float64, device="cuda")
    best = torch.zeros(rows, top, dtype=torch.float64, device="cuda")
    for r, t in enumerate(s["token"].tolist()):
        if t < 0:
            continue
        z = torch.log_softmax(s["logits"][r].double() / c["temp"], 0)
        lp[r], ent[r] = z[t], -(z.exp() * z).sum()
        best[r] = torch.topk(z, top).values
    return [lp, ent, None, best]


def exact(case, seed):
    return {"append": _exact_append, "attend": _exact_attend, "logprobs": _exact_logprobs}[case["kind"]](case, prepare(case, seed))


# ---- what a pass cannot do without -------------------------------------------------------------------------
def work(case):
    c = case
    if c["kind"] == "logprobs":
        live = c["rows"] - c["rows"] // 50
        return {"bytes": 4 * live * (c["vocab"] + 3 + 2 * c["top"]), "flops": 6 * live * c["vocab"]}
    hq, hkv, dh, kw = c["hq"], c["hkv"], c["dh"], c["hkv"] * c["dh"]
    seqs = _sequences(c)
    live = sum(n for _, n in seqs)
    if c["kind"] == "append":  # queries, keys and values in; queries and 4-bit rows out; then the rows read back as fp16
        return {"bytes": int(live * (8 * hq * dh + 8 * kw + 2 * 2 * kw * 9 / 16 + 4 * kw)), "flops": 12 * live * (hq + 2 * hkv) * dh}

    def seen(pos):
        return pos + 1 if not c["window"] else min(pos + 1, c["window"] + min(c["sinks"], max(0, pos + 1 - c["window"])))

    keys = sum(seen(f + i) for f, n in seqs for i in range(n))
    once = sum(min(f + n, seen(f) + n - 1) for f, n in seqs if n)  # of them, distinct ones
    return {"bytes": int(2 * once * kw * 9 / 16 + live * 12 * hq * dh), "flops": 4 * keys * hq * dh}
