"""Cases of the rotary-position, 4-bit cache and attention operators
(include/hip_kv.h through llm.c_amd/hipkv.py): what they are timed on, their
plain forms in elementary torch operations, and their results in 64 bits.

Shapes are those of this repository's OLMoE (16 heads, 16 kv heads of 128)
and Mixtral (32 heads, 8 kv heads of 128) models, with heads of 64 and 256
besides.  Cached rows are made as codes and scales, with the spread that
quantized normal values have; slots that no row was stored in hold NaN
scales, as memory that was never written may.

The library's calls pass no stream: they run on the library's own stream, in
call order.
"""
import math
import os
import random
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TYPE_ID = {"f32": 0, "f16": 1, "bf16": 2}
TILE = 32  # cached rows of one tile


def _rope(type, rows, heads, D, rot, layout, scaling, far, name=None):
    return dict(({"name": name} if name else {}), kind="rope", type=type, rows=rows, heads=heads,
                D=D, rot=rot, layout=layout, scaling=scaling, far=far)


def _append(type, seqs, rows, context, H, KH, D, rot, layout, page, name=None):
    return dict(({"name": name} if name else {}), kind="append", type=type, seqs=seqs, rows=rows,
                context=context, H=H, KH=KH, D=D, rot=rot, layout=layout, page=page)


def _attn(type, seqs, rows, context, H, KH, D, page, window=0, ragged=False, name=None):
    return dict(({"name": name} if name else {}), kind="attn", type=type, seqs=seqs, rows=rows,
                context=context, H=H, KH=KH, D=D, page=page, window=window, ragged=ragged)


def listed():
    return [
        # the queries of one generated token of sixteen sequences
        _rope("f32", 16, 32, 128, 128, "pairs", "plain", 4096, name="rope_step16"),
        # the queries of an 8192-row chunk, deep in a context stretched 4 times
        _rope("bf16", 8192, 32, 128, 128, "halves", "yarn", 131072, name="rope_chunk8192"),
        # one generated token of sixteen sequences: keys, values and queries
        _append("f32", 16, 1, 1100, 32, 8, 128, 128, "pairs", 64, name="append_step16"),
        # five prompts of different lengths behind cached prefixes
        _append("bf16", 5, 1500, 700, 16, 16, 128, 64, "halves", 32, name="append_prompts5"),
        # one long prompt in the framework's own type
        _append("f32", 1, 8192, 0, 32, 8, 128, 128, "pairs", 256, name="append_prompt8192"),
        # a generated token of one short sequence, a kv head for every head
        _attn("f32", 1, 1, 1024, 16, 16, 128, 64, name="attn_step1"),
        # sixteen sequences in lockstep, grouped heads
        _attn("f32", 16, 1, 1100, 32, 8, 128, 64, name="attn_step16"),
        # one very long context
        _attn("bf16", 1, 1, 131072, 32, 8, 128, 256, name="attn_long1"),
        # a large batch of sequences of every length
        _attn("f32", 64, 1, 16384, 32, 8, 128, 64, ragged=True, name="attn_batch64"),
        # a prompt in the framework's own type
        _attn("f32", 1, 2048, 2048, 16, 16, 128, 64, name="attn_prompt2048"),
        # chunks of four prompts on cached rows, with a sliding window
        _attn("bf16", 4, 512, 8192, 32, 8, 128, 64, window=4096, name="attn_chunks4"),
        # a long prompt in 16 bits
        _attn("bf16", 1, 8192, 8192, 32, 8, 128, 128, name="attn_prompt8192"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49))))))


def draw(rng):
    """Another case of the listed ones' ranges."""
    kind = rng.choice(("rope", "append", "attn", "attn"))
    type = rng.choice(("f32", "f16", "bf16"))
    D = rng.choice((64, 128, 128, 256))
    layout = rng.choice(("pairs", "halves"))
    KH = rng.choice((1, 2, 4, 5, 8, 16))
    H = KH * rng.choice((1, 2, 3, 4, 7, 8))
    page = rng.choice((32, 64, 128, 256))
    rot = rng.choice((D, D, D // 2, D // 4))
    most = 8192 * 32 * 128  # values of the largest chunk
    if kind == "rope":
        heads = rng.choice((1, 5, 8, 16, 32))
        return _rope(type, _log_int(rng, 1, most // 2 // (heads * D)), heads, D, rot, layout,
                     rng.choice(("plain", "linear", "ntk", "yarn")), _log_int(rng, 64, 131072))
    if kind == "append":
        total = _log_int(rng, 1, min(16384, most // 2 // (H * D)))
        seqs = rng.randrange(1, min(total, 24) + 1)
        return _append(type, seqs, max(1, total // seqs), rng.choice((0, _log_int(rng, 1, 3000))),
                       H, KH, D, rot, layout, page)
    form = rng.choice(("step", "step", "few", "prompt"))
    if form == "prompt":
        n = _log_int(rng, 17, 2048)
        seqs = rng.randrange(1, max(1, min(4, 2048 // n)) + 1)
        context = n + rng.choice((0, _log_int(rng, 1, 2048)))
        H = KH * min(H // KH, 4)
    else:
        n = 1 if form == "step" else rng.randrange(2, 17)
        seqs = _log_int(rng, 1, 64)
        context = n + _log_int(rng, 1, min(131072 - n, (1 << 30) // (seqs * KH * D)))
    return _attn(type, seqs, n, context, H, KH, D, page,
                 window=rng.choice((0, 0, _log_int(rng, 1, 2 * context))), ragged=rng.random() < 0.6)


# --------------------------------------------------------------------------
# the shape of a case: lengths belong to the case, not to the seed
# --------------------------------------------------------------------------

def _lengths(case):
    """Rows of each sequence in this call, and cached rows after it."""
    rng = random.Random("%d %d %d" % (case["seqs"], case["rows"], case["context"]))
    if case["kind"] == "append":
        rows = [max(1, int(case["rows"] * rng.uniform(0.5, 1.5))) if case["rows"] > 1 else 1
                for _ in range(case["seqs"])]
        if case["seqs"] == 1:
            rows = [case["rows"]]
        before = [rng.randrange(case["context"] // 2, case["context"] + 1) for _ in rows]
        return rows, [n + b for n, b in zip(rows, before)]
    rows = [case["rows"]] * case["seqs"]
    lens = [case["context"]] * case["seqs"]
    if case["ragged"]:
        lens = [min(case["context"], max(1, int(case["context"] ** rng.uniform(0.6, 1.0))))
                for _ in lens]
        rows = [min(n, m) for n, m in zip(rows, lens)]
    return rows, lens


def _tile_bytes(D):
    return 34 * D + 64


def _visible(case):
    """(cached rows that some row sees, (row, cached row) pairs) of all sequences."""
    seen = pairs = 0
    w = case["window"] or (1 << 60)
    for n, m in zip(*_lengths(case)):
        seen += min(m, n - 1 + w)
        # rows at positions m - n .. m - 1 see min(p + 1, w) cached rows each
        full = max(0, min(n, m - w + 1)) if w < m else 0
        k = n - full
        pairs += full * w + k * (m - n) + k * (k + 1) // 2
    return seen, pairs


def work(case):
    b = 4 if case["type"] == "f32" else 2
    D = case["D"]
    if case["kind"] == "rope":
        n = case["rows"] * case["heads"] * D
        return {"bytes": 2 * n * b + 4 * case["rows"], "flops": 3 * n}
    if case["kind"] == "append":
        rows = sum(_lengths(case)[0])
        kv = rows * case["KH"] * D
        codes = rows * case["KH"] * _tile_bytes(D) / TILE
        return {"bytes": 2 * rows * case["H"] * D * b + 4 * kv * b + 2 * codes,
                "flops": 3 * rows * case["H"] * D + 20 * kv}
    rows = sum(_lengths(case)[0])
    seen, pairs = _visible(case)
    return {"bytes": seen * case["KH"] * _tile_bytes(D) / TILE + 2 * rows * case["H"] * D * b,
            "flops": 4 * D * case["H"] * pairs}


# --------------------------------------------------------------------------
# inputs, made on the GPU from the seed
# --------------------------------------------------------------------------

def _freqs(D, rot, scaling):
    """Radians a position for each pair, and what cos and sin are multiplied by."""
    i = torch.arange(0, rot, 2, dtype=torch.float64)
    theta, factor, context = 1e6, 4.0, 32768.0
    if scaling == "ntk":
        theta *= factor ** (rot / max(rot - 2, 1))
    f, mag = theta ** (-i / rot), 1.0
    if scaling == "linear":
        f = f / factor
    if scaling == "yarn":  # pairs that turn often keep their angle, slow ones are stretched
        at = [rot * math.log(context / (turns * 2 * math.pi)) / (2 * math.log(theta))
              for turns in (32.0, 1.0)]
        lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rot - 1)
        ramp = ((i / 2 - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        f = f / factor * ramp + f * (1 - ramp)
        mag = 0.1 * math.log(factor) + 1
    return f.cuda(), mag


def _pool(g, case, pages):
    """Pages of codes and scales: codes spread as those of normal values are."""
    KH, D, tiles = case["KH"], case["D"], case["page"] // TILE
    pool = torch.empty(pages, KH, tiles, _tile_bytes(D), dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 26) // (KH * tiles * 32 * D))
    for a in range(0, pages, step):
        part = pool[a:a + step]
        shape = (*part.shape[:3], 32 * D)

        def nibbles():
            return torch.randn(shape, generator=g, device="cuda", dtype=torch.float16).mul_(3).round_() \
                .clamp_(-8, 7).add_(8).to(torch.uint8)

        part[..., :32 * D] = nibbles() | (nibbles() << 4)
        d = torch.randn(*part.shape[:3], D + 32, generator=g, device="cuda")
        d = ((0.2 + 0.05 * d.abs()) * torch.where(d < 0, -1.0, 1.0)).half()
        part[..., 32 * D:] = d.view(torch.uint8)
    return pool


def _slots(table, lens, page):
    """(page, tile, row in the tile) of every cached row below max(lens), [seqs][.]."""
    t = torch.arange(max(lens), device="cuda")
    return table[:, t // page].long(), (t % page // TILE)[None], (t % TILE)[None]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt, D = TYPES[case["type"]], case["D"]

    def rand(*shape):
        return torch.randn(*shape, generator=g, device="cuda").to(dt)

    if case["kind"] == "rope":
        f, mag = _freqs(D, case["rot"], case["scaling"])
        x = rand(case["rows"], case["heads"], D)
        pos = torch.randint(max(0, case["far"] - case["rows"]), case["far"], (case["rows"],), generator=g,
                            device="cuda", dtype=torch.int32)
        return dict(case=case, x=x, pos=pos, freq=f, mag=mag, out=torch.empty_like(x))

    rows, lens = _lengths(case)
    H, KH, page = case["H"], case["KH"], case["page"]
    need = [-(-m // page) for m in lens]
    pages = sum(need) + 3
    ids = torch.randperm(pages, generator=g, device="cuda").int()
    host = torch.zeros(len(lens), max(need), dtype=torch.int64)
    at = 0
    for s, n in enumerate(need):
        host[s, :n] = torch.arange(at, at + n)
        at += n
    table = ids[host.cuda()].contiguous()
    start = [0]
    for n in rows:
        start.append(start[-1] + n)
    st = dict(case=case, pool=_pool(g, case, pages), table=table, pages=pages, rows=rows, lens=lens,
              row_start=torch.tensor(start, dtype=torch.int32, device="cuda"),
              len=torch.tensor(lens, dtype=torch.int32, device="cuda"))
    # slots without a row hold NaN scales
    gone = torch.full((pages, page), float("nan"), device="cuda")
    used = torch.arange(max(lens), device="cuda")[None] < st["len"][:, None]
    p, _, _ = _slots(table, lens, page)
    at = torch.arange(max(lens), device="cuda")[None].expand_as(used) % page
    gone[p[used], at[used]] = 0
    gone = gone.view(pages, 1, page // TILE, TILE, 1).half()
    view = st["pool"][..., 32 * D:].contiguous().view(torch.float16)
    ks, vs = view[..., :D].unflatten(-1, (TILE, D // 32)) + gone, view[..., D:] + gone[..., 0]
    st["pool"][..., 32 * D:] = torch.cat([ks.flatten(-2), vs], -1).view(torch.uint8)
    del view, ks, vs, gone

    T = start[-1]
    if case["kind"] == "attn":
        st.update(q=2 * rand(T, H, D), out=torch.empty(T, H, D, dtype=dt, device="cuda"))
        return st
    # q, k and v as a product leaves them: one row of all heads a token; some
    # channels of the keys are larger than the rest, as they are in models
    wide = 1 + 7 * (torch.rand(KH, D, generator=g, device="cuda") < 0.05)
    qkv = rand(T, H + 2 * KH, D)
    qkv[:, H:H + KH] *= wide.to(dt)
    f, mag = _freqs(D, case["rot"], "plain")
    st.update(qkv=qkv, freq=f, mag=mag, q_out=torch.empty(T, H, D, dtype=dt, device="cuda"),
              k_out=torch.empty(T, KH, D, dtype=dt, device="cuda"),
              v_out=torch.empty(T, KH, D, dtype=dt, device="cuda"))
    return st


# --------------------------------------------------------------------------
# plain forms
# --------------------------------------------------------------------------

def _rotate(x, pos, freq, mag, layout):
    """x [T][heads][D] in 64 bits, its first 2 * len(freq) channels rotated."""
    x, rot = x.double(), 2 * freq.numel()
    a = pos.double()[:, None] * freq[None]
    c, s = (torch.cos(a) * mag)[:, None], (torch.sin(a) * mag)[:, None]
    y = x.clone()
    if layout == "pairs":
        x1, x2 = x[..., 0:rot:2], x[..., 1:rot:2]
        y[..., 0:rot:2], y[..., 1:rot:2] = x1 * c - x2 * s, x2 * c + x1 * s
    else:
        x1, x2 = x[..., :rot // 2], x[..., rot // 2:rot]
        y[..., :rot // 2], y[..., rot // 2:rot] = x1 * c - x2 * s, x2 * c + x1 * s
    return y


def _codes(x):
    """Codes 0 .. 15 and f16 scales of the groups x [...][n] of fp32 values."""
    lo, hi = x.amin(-1), x.amax(-1)
    m = torch.where(hi > -lo, hi, lo)
    d = (m * -0.125).clamp(-65504, 65504).half()
    w = d.double()[..., None]
    q = torch.floor(x.double() / torch.where(w == 0, 1.0, w) + 8.5).clamp(0, 15)
    return torch.where(w == 0, 8.0, q).to(torch.int32), d


# bits of code j of a word (bits 30, 31, 0, 1 for j = 7)
_SHIFT = [(2 + 4 * (j >> 1) + 16 * (j & 1)) % 32 for j in range(8)]


def _word(codes):
    """int32 words of codes [...][8]."""
    sh = torch.tensor(_SHIFT, device=codes.device, dtype=torch.int64)
    c = codes.long()
    w = ((c << sh) & 0xffffffff | c * (sh == 30) >> 2).sum(-1)
    return torch.where(w >= 1 << 31, w - (1 << 32), w).to(torch.int32)


def _unword(w):
    """codes [...][8] of int32 words: the word turned right by 2 holds code j
    in its nibble j / 2 + 4 * (j % 2)."""
    u = ((w >> 2) & 0x3fffffff) | (w << 30)
    sh = torch.tensor([4 * (j >> 1) + 16 * (j & 1) for j in range(8)], device=w.device, dtype=torch.int32)
    return (u[..., None] >> sh) & 15


def _per(D):
    return min(4, D // 32)  # words of a lane that follow each other


def _tiles_of(tiles, D):
    """(k, v) [...][32][D] fp32 of tiles [...][bytes]."""
    lead, per = tiles.shape[:-1], _per(D)
    kw = tiles[..., :16 * D].contiguous().view(torch.int32)
    vw = tiles[..., 16 * D:32 * D].contiguous().view(torch.int32)
    d = tiles[..., 32 * D:].contiguous().view(torch.float16).float()
    # keys: [half of the tile][group / per][8-channel part][row][group % per] words of 8 channels
    k = _unword(kw.view(*lead, 2, D // 32 // per, 4, 16, per))
    n = len(lead)
    k = k.permute(*range(n), n, n + 3, n + 1, n + 4, n + 2, n + 5).reshape(*lead, 32, D // 32, 32)
    k = (k - 8).float() * d[..., :D].reshape(*lead, 32, D // 32, 1)
    # values: [channel / 64][4-row part][channel % 16][channel / 16 % 4] words of 8 rows
    v = _unword(vw.view(*lead, D // 64, 4, 16, 4)).unflatten(-1, (2, 4))
    v = v.permute(*range(n), n + 4, n + 1, n + 5, n, n + 3, n + 2).reshape(*lead, 32, D)
    return k.flatten(-2), (v - 8).float() * d[..., D:, None]


def _append_plain(s):
    case = s["case"]
    H, KH, D, page, dt = case["H"], case["KH"], case["D"], case["page"], TYPES[case["type"]]
    n = s["row_start"].diff()
    seq = torch.repeat_interleave(torch.arange(len(s["lens"]), device="cuda"), n, output_size=s["qkv"].shape[0])
    at = torch.arange(s["qkv"].shape[0], device="cuda") - s["row_start"][1:][seq] + s["len"][seq]
    q, k, v = s["qkv"][:, :H], s["qkv"][:, H:H + KH], s["qkv"][:, H + KH:]
    q = _rotate(q, at, s["freq"], s["mag"], case["layout"]).float().to(dt)
    k = _rotate(k, at, s["freq"], s["mag"], case["layout"]).float()
    kc, kd = _codes(k.unflatten(-1, (D // 32, 32)))
    vc, vd = _codes(v.float())
    # where each row goes
    pg, tile, r = s["table"][seq, at // page].long(), at % page // TILE, at % TILE
    pool, per = s["pool"], _per(D)
    kw = _word(kc.view(-1, KH, D // 32, 4, 8))  # [T][KH][group][part]
    gi, pi = torch.arange(D // 32, device="cuda"), torch.arange(4, device="cuda")
    word = (gi // per * 64 * per + gi % per)[:, None] + pi * 16 * per
    base = (r // 16 * (2 * D) + r % 16 * per)[:, None, None]
    head = torch.arange(KH, device="cuda")
    words = pool.view(torch.int32)  # [pages][KH][tiles][bytes / 4]
    words[pg[:, None, None, None], head[:, None, None], tile[:, None, None, None],
          (word[None] + base)[:, None]] = kw
    # a row's code is 4 bits of a word that seven other rows share: the words
    # are taken apart, the row's codes put in, and written again
    ch = torch.arange(D, device="cuda")
    j = r % 4 + 4 * (r // 16)
    part = r % 16 // 4
    vi = 4 * D + (ch // 64 * 256 + ch % 16 * 4 + ch // 16 % 4)[None] + (part * 64)[:, None]
    sh = torch.tensor(_SHIFT, device="cuda")[j]
    ones = 15 << sh
    clear = (ones & 0xffffffff | ones >> 32)[:, None, None].expand(-1, KH, D)
    c = vc.long() << sh[:, None, None]
    c = c & 0xffffffff | c >> 32
    flat = ((pg[:, None] * KH + head) * (page // TILE) + tile[:, None])[..., None] * (_tile_bytes(D) // 4) + vi[:, None]
    which, back = torch.unique(flat.flatten(), return_inverse=True)
    old = words.view(-1)[which].long() & 0xffffffff
    drop = torch.zeros_like(old).index_add_(0, back, clear.flatten())
    put = torch.zeros_like(old).index_add_(0, back, c.flatten())
    w = old & ~drop | put
    words.view(-1)[which] = torch.where(w >= 1 << 31, w - (1 << 32), w).to(torch.int32)
    halves = pool.view(torch.float16)
    halves[pg[:, None, None], head[:, None], tile[:, None, None],
           16 * D + (r * (D // 32))[:, None, None] + gi] = kd
    halves[pg[:, None], head, tile[:, None], 17 * D + r[:, None]] = vd
    # the values that the stored codes stand for
    k, v = _tiles_of(pool[pg, :, tile], D)  # [T][KH][32][D]
    pick = torch.arange(len(r), device="cuda")
    return {"q": q, "k": k[pick, :, r].to(dt), "v": v[pick, :, r].to(dt)}


def _attn_plain(s):
    case = s["case"]
    H, KH, D, page, dt = case["H"], case["KH"], case["D"], case["page"], TYPES[case["type"]]
    S, most, N = len(s["lens"]), max(s["lens"]), max(s["rows"])
    k, v = _tiles_of(s["pool"][s["table"].long()], D)  # [S][pages][KH][tiles][32][D]
    k = k.permute(0, 2, 1, 3, 4, 5).reshape(S, KH, -1, D)[:, :, :most]
    v = v.permute(0, 2, 1, 3, 4, 5).reshape(S, KH, -1, D)[:, :, :most]
    j = torch.arange(most, device="cuda")
    v = torch.where((j < s["len"][:, None])[:, None, :, None], v, 0.0)
    n = s["row_start"].diff()
    i = torch.arange(N, device="cuda")
    row = (s["row_start"][:-1, None] + i).clamp_max(s["q"].shape[0] - 1)  # [S][N]
    p = (s["len"] - n)[:, None] + i
    see = (j <= p[..., None]) & (j < s["len"][:, None, None])  # [S][N][most]
    if case["window"]:
        see &= j > p[..., None] - case["window"]
    q = s["q"].float()[row].view(S, N, KH, H // KH, D).permute(0, 2, 3, 1, 4)
    x = q.reshape(S, KH, -1, D) @ k.transpose(-1, -2).contiguous() * D ** -0.5
    x = x.view(S, KH, H // KH, N, most).masked_fill_(~see[:, None, None], -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True))
    o = (x.view(S, KH, -1, most) @ v) / x.sum(-1).view(S, KH, -1, 1)
    o = o.view(S, KH, H // KH, N, D).permute(0, 3, 1, 2, 4).reshape(S, N, H, D)
    return o[i[None] < n[:, None]].to(dt)


def run(s):
    case = s["case"]
    if own:
        return _run_own(s)
    if case["kind"] == "rope":
        return _rotate(s["x"], s["pos"], s["freq"], s["mag"], case["layout"]).float().to(s["x"].dtype)
    return _append_plain(s) if case["kind"] == "append" else _attn_plain(s)


def _run_own(s):
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "llm.c_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import hipkv
    case, ty = s["case"], TYPE_ID[s["case"]["type"]]
    D = case["D"]
    if case["kind"] != "attn":
        rope = hipkv.Rope(case["rot"], hipkv.PAIRS if case["layout"] == "pairs" else hipkv.HALVES,
                          s["freq"].data_ptr(), s["mag"])
    if case["kind"] == "rope":
        n = case["heads"] * D
        hipkv.rope(rope, ty, s["x"].data_ptr(), n, s["out"].data_ptr(), n, case["rows"], case["heads"],
                   D, s["pos"].data_ptr())
        return s["out"]
    H, KH = case["H"], case["KH"]
    cache = hipkv.Cache(s["pool"].data_ptr(), s["pages"], case["page"], KH, D)
    batch = hipkv.Batch(len(s["lens"]), sum(s["rows"]), max(s["rows"]), max(s["lens"]),
                        s["row_start"].data_ptr(), s["len"].data_ptr(), s["table"].data_ptr(),
                        s["table"].shape[1])
    if case["kind"] == "attn":
        if "ws" not in s:
            s["ws"] = torch.empty(hipkv.attn_ws(cache, batch, H), dtype=torch.uint8, device="cuda")
        hipkv.attn(cache, batch, ty, s["q"].data_ptr(), H * D, H, s["out"].data_ptr(), H * D, D ** -0.5,
                   case["window"], s["ws"].data_ptr(), s["ws"].numel())
        return s["out"]
    n, x = (H + 2 * KH) * D, s["qkv"].data_ptr()
    b = s["qkv"].element_size()
    hipkv.append(cache, batch, ty, x + H * D * b, x + (H + KH) * D * b, n, rope=rope, q=x, q_stride=n,
                 heads=H, q_out=s["q_out"].data_ptr(), q_out_stride=H * D)
    hipkv.read(cache, batch, ty, s["k_out"].data_ptr(), s["v_out"].data_ptr(), KH * D)
    return {"q": s["q_out"], "k": s["k_out"], "v": s["v_out"]}


# --------------------------------------------------------------------------
# results in 64 bits, from the definitions
# --------------------------------------------------------------------------

def _turn64(x, pos, freq, mag, layout):
    """Each pair as a complex number times mag * e^(i pos freq)."""
    x = x.double()
    rot, T, heads = 2 * freq.numel(), *x.shape[:2]
    head = x[..., :rot].reshape(T, heads, *((rot // 2, 2) if layout == "pairs" else (2, rot // 2)))
    if layout != "pairs":
        head = head.transpose(2, 3)
    z = torch.view_as_complex(head.contiguous())
    z = z * torch.polar(torch.full_like(freq, mag).expand(T, -1), pos.double()[:, None] * freq)[:, None]
    y = torch.view_as_real(z)
    y = (y if layout == "pairs" else y.transpose(2, 3)).reshape(T, heads, rot)
    return torch.cat([y, x[..., rot:]], -1)


def _round64(x, group):
    """Values of x's 4-bit form, groups of `group` channels with an f16 scale."""
    y = x.float().double().unflatten(-1, (-1, group))
    top, low = y.max(-1, keepdim=True).values, y.min(-1, keepdim=True).values
    big = torch.where(top > -low, top, low)
    d = (big / -8).clamp(-65504, 65504).float().half().double()
    n = torch.floor(y / torch.where(d == 0, torch.ones_like(d), d) + 0.5).clamp(-8, 7)
    return (n * d).flatten(-2)


def _row64(pool, table, page, D, length):
    """(k, v) [length][KH][D] of one sequence's cached rows, word by word of the layout."""
    t = torch.arange(length, device="cuda")
    tile = pool[table[t // page].long(), :, t % page // TILE]  # [length][KH][bytes]
    words = tile[..., :32 * D].contiguous().view(torch.int32).long() & 0xffffffff
    scales = tile[..., 32 * D:].contiguous().view(torch.float16).double()
    r, c, per = (t % TILE)[:, None], torch.arange(D, device="cuda")[None], _per(D)

    def take(index, j):
        w = words.gather(-1, index[:, None].expand(-1, words.shape[1], -1))
        b = (2 + 4 * (j // 2) + 16 * (j % 2)).expand_as(index)[:, None]
        return (((w | w << 32) >> b) & 15).double() - 8

    g, part = c // 32, c % 32 // 8
    k = take(((r // 16 * (D // 32 // per) + g // per) * 64 + part * 16 + r % 16) * per + g % per, c % 8)
    k *= scales.gather(-1, (r * (D // 32) + g)[:, None].expand(-1, words.shape[1], -1))
    lane = r % 16 // 4 * 16 + c % 16
    v = take(4 * D + (c // 64 * 64 + lane) * 4 + c // 16 % 4, r % 4 + 4 * (r // 16) + 0 * c)
    return k, v * scales.gather(-1, (D + r)[:, None].expand(-1, words.shape[1], -1))


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rope":
        return _turn64(s["x"], s["pos"], s["freq"], s["mag"], case["layout"])
    H, KH, D = case["H"], case["KH"], case["D"]
    if case["kind"] == "append":
        at = torch.cat([torch.arange(m - n, m, device="cuda") for n, m in zip(s["rows"], s["lens"])])
        q, k, v = s["qkv"].split([H, KH, KH], 1)
        return {"q": _turn64(q, at, s["freq"], s["mag"], case["layout"]),
                "k": _round64(_turn64(k, at, s["freq"], s["mag"], case["layout"]), 32),
                "v": _round64(v, D)}
    out, r0 = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda"), 0
    for n, m, table in zip(s["rows"], s["lens"], s["table"]):
        k, v = _row64(s["pool"], table, case["page"], D, m)
        j = torch.arange(m, device="cuda")
        step = max(1, (1 << 28) // m)
        for h in range(H):
            kh, vh = k[:, h // (H // KH)].t().contiguous(), v[:, h // (H // KH)].contiguous()
            for a in range(0, n, step):
                e = min(n, a + step)
                p = torch.arange(m - n + a, m - n + e, device="cuda")[:, None]
                x = s["q"][r0 + a:r0 + e, h].double() @ kh / math.sqrt(D)
                hide = (j > p) | (j <= p - case["window"]) if case["window"] else j > p
                out[r0 + a:r0 + e, h] = torch.softmax(x.masked_fill_(hide, -math.inf), -1) @ vh
        r0 += n
    return out
