"""Cases of the 8-bit floating-point products (include/hip_f8.h through
llm.c_amd/hipf8.py): rows quantized to e4m3 with a scale for each 128 channels,
the product with a matrix that has a scale for each 128 x 128 block, pairs of
tokens and experts sorted by expert, the product grouped by expert, and the
experts' outputs weighted and added per token.  What they are timed on, their
plain forms in elementary torch operations, and their results in 64 bits.

Shapes are those of this repository's OLMoE (width 2048, 64 experts of 1024, 8
a token) and Mixtral (width 4096, 8 experts of 14336, 2 a token) models.

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
BLOCK = 128
LEAST = 2.0 ** -96  # of a row block's scale


def _case(name, kind, **kw):
    return dict(({"name": name} if name else {}), kind=kind, **kw)


def _quantize(type, rows, K, pad=0, name=None):
    return _case(name, "quantize", type=type, rows=rows, K=K, pad=pad)


def _mul(type, rows, N, K, gated=False, add=False, name=None):
    return _case(name, "mul", type=type, rows=rows, N=N, K=K, gated=gated, add=add)


def _sort(tokens, topk, experts, skew=0.0, away=0.0, name=None):
    return _case(name, "sort", tokens=tokens, topk=topk, experts=experts, skew=skew, away=away)


def _group(type, tokens, topk, experts, N, K, gated, gather, skew=0.0, away=0.0, name=None):
    return _case(name, "group", type=type, tokens=tokens, topk=topk, experts=experts, N=N, K=K, gated=gated,
                 gather=gather, skew=skew, away=away)


def _combine(type, tokens, topk, experts, N, add, away=0.0, name=None):
    return _case(name, "combine", type=type, tokens=tokens, topk=topk, experts=experts, N=N, add=add, away=away)


def listed():
    return [
        # the inputs of one generated token of sixteen sequences, in the framework's own type
        _quantize("f32", 16, 4096, name="quantize_step16"),
        # a long prompt's rows, in 16 bits
        _quantize("bf16", 8192, 4096, name="quantize_prompt8192"),
        # the lm_head of one generated token
        _mul("f32", 1, 50304, 2048, name="mul_head1"),
        # the output product of a prompt of odd length, with its residual
        _mul("f16", 333, 4096, 4096, add=True, name="mul_chunk333"),
        # a long prompt through a dense layer's gate and up matrices
        _mul("bf16", 8192, 14336, 4096, gated=True, name="mul_prompt8192"),
        # which rows go to which expert, for one generated token of sixteen sequences
        _sort(16, 8, 64, name="sort_step16"),
        # the same for a long prompt with a skewed router, a quarter of the experts elsewhere
        _sort(8192, 8, 64, skew=1.0, away=0.25, name="sort_prompt8192"),
        # the experts' gate and up products of one generated token of sixteen sequences
        _group("bf16", 16, 2, 8, 14336, 4096, True, True, name="group_step16"),
        # the experts' down products of a prompt with a skewed router, in the framework's own type
        _group("f32", 512, 8, 64, 2048, 1024, False, False, skew=1.0, name="group_prompt512"),
        # the experts' gate and up products of a long prompt
        _group("bf16", 4096, 2, 8, 14336, 4096, True, True, name="group_prompt4096"),
        # the experts' outputs of one generated token of sixteen sequences
        _combine("f32", 16, 2, 8, 4096, True, name="combine_step16"),
        # the experts' outputs of a long prompt, a quarter of them elsewhere
        _combine("bf16", 8192, 8, 64, 2048, True, away=0.25, name="combine_prompt8192"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def _size(rng, lo, hi):
    """A count of channels: a multiple of 128 or 16 as models have them, or any."""
    n, by = _log_int(rng, lo, hi), rng.choice((128, 128, 16, 1))
    return max(lo, min(hi, -(-n // by) * by))


def draw(rng):
    """Another case of the listed ones' ranges."""
    kind = rng.choice(("quantize", "mul", "mul", "sort", "group", "group", "combine"))
    type = rng.choice(("f32", "f16", "bf16"))
    if kind == "quantize":
        K = _size(rng, 16, 14336)
        return _quantize(type, _log_int(rng, 1, 8192 * 4096 // K), K, pad=rng.choice((0, 0, 8, 128)))
    experts = rng.choice((4, 8, 12, 16, 32, 64, 128))
    topk = rng.randrange(1, min(8, experts) + 1)
    skew, away = rng.choice((0.0, 0.5, 1.0)), rng.choice((0.0, 0.0, 0.25, 0.5))
    if kind == "sort":
        return _sort(_log_int(rng, 1, 8192), topk, experts, skew, away)
    if kind == "combine":
        N = _size(rng, 64, 8192)
        return _combine(type, _log_int(rng, 1, min(8192, (1 << 27) // (topk * N))), topk, experts, N,
                        rng.random() < 0.5, away)
    gated = rng.random() < 0.5
    most = 8192 * 14336 * 4096  # products of the largest case, each for gate and up
    if kind == "mul":
        N, K = _size(rng, 16, 32768), _size(rng, 16, 14336)
        while N * K > 1 << 27:
            N //= 2
        rows = _log_int(rng, 1, 8192)
        return _mul(type, min(rows, most // (N * K)), N, K, gated, rng.random() < 0.3 and not gated)
    N, K = _size(rng, 64, 14336), _size(rng, 64, 14336)
    while N * K * experts > 1 << 28:
        N = max(64, N // 2)
        K = max(64, K - K // 3)
    tokens = _log_int(rng, 1, max(1, min(4096, (1 << 28) // (experts * max(N, K)))))
    return _group(type, tokens, topk, experts, N, K, gated, rng.random() < 0.5, skew, away)


# --------------------------------------------------------------------------
# the routing of a case: it belongs to the case, not to the seed, so that a
# case's work is known (the sort's own ids are drawn from the seed)
# --------------------------------------------------------------------------

def _routing(case, seed=None):
    """Expert ids [tokens][topk] on the host, distinct in a token; an id of `experts`
    and more is no expert of this process."""
    g = torch.Generator()
    g.manual_seed(case["tokens"] * 1000003 + case["topk"] * 1009 + case["experts"] if seed is None else seed)
    NE, T, k = case["experts"], case["tokens"], case["topk"]
    like = case.get("skew", 0.0) * torch.randn(NE, generator=g)
    noise = torch.rand(T, NE, generator=g).clamp_min(1e-30)
    ids = (like - torch.log((-torch.log(noise)).clamp_min(1e-30))).topk(k, dim=1).indices
    far = torch.randperm(NE, generator=g)[:int(case["away"] * NE)]
    gone = torch.zeros(NE, dtype=torch.bool)
    gone[far] = True
    return torch.where(gone[ids], ids + NE, ids).int()


def _sorted(ids, experts):
    """(start [experts + 1], from [rows], pos [tokens][topk]) of ids, on their device."""
    flat = ids.flatten().long()
    here = (flat >= 0) & (flat < experts)
    key = torch.where(here, flat, experts)
    order = torch.sort(key, stable=True).indices
    start = torch.searchsorted(key[order], torch.arange(experts + 1, device=ids.device))
    at = torch.empty_like(order).scatter_(0, order, torch.arange(order.numel(), device=ids.device))
    pos = torch.where(here, at, -1).view(ids.shape)
    return start.int(), (order // ids.shape[1]).int(), pos.int()


def _experts_rows(case):
    ids = _routing(case).flatten()
    return torch.bincount(ids[ids < case["experts"]].long(), minlength=case["experts"])


def work(case):
    kind = case["kind"]
    b = 4 if case.get("type") == "f32" else 2
    if kind == "quantize":
        n, K = case["rows"], case["K"]
        return {"bytes": n * K * (b + 1) + 4 * n * -(-K // BLOCK), "flops": 4 * n * K}
    if kind == "sort":
        P = case["tokens"] * case["topk"]
        return {"bytes": 12 * P + 4 * case["experts"], "flops": 4 * P}
    N = case["N"]
    if kind == "combine":
        ids = _routing(case)
        P = int((ids < case["experts"]).sum())
        T = case["tokens"]
        return {"bytes": P * N * b + T * N * b * (2 if case["add"] else 1) + 8 * T * case["topk"], "flops": 2 * P * N}
    K, mats = case["K"], 2 if case["gated"] else 1
    KB, NB = -(-K // BLOCK), -(-N // BLOCK)
    matrix = mats * (N * K + 4 * NB * KB)
    if kind == "mul":
        T = case["rows"]
        return {"bytes": matrix + T * (K + 4 * KB) + T * N * b * (2 if case["add"] else 1),
                "flops": 2 * T * N * K * mats}
    n = _experts_rows(case)
    rows = int(n.sum())
    read = case["tokens"] if case["gather"] else rows
    return {"bytes": 4 * case["experts"] + int((n > 0).sum()) * matrix + read * (K + 4 * KB) + rows * N * b,
            "flops": 2 * rows * N * K * mats}


# --------------------------------------------------------------------------
# inputs, made on the GPU from the seed
# --------------------------------------------------------------------------

def _weights(g, count, N, K):
    """Matrices of codes and a scale for each 128 x 128 block, as normal values of standard
    deviation 0.02 have them."""
    codes = torch.empty(count, N, K, dtype=torch.float8_e4m3fn, device="cuda")
    for i in range(count):
        codes[i] = (torch.randn(N, K, generator=g, device="cuda") * 112).clamp_(-448, 448).to(codes.dtype)
    scale = torch.rand(count, -(-N // BLOCK), -(-K // BLOCK), generator=g, device="cuda")
    return codes, (0.7 + 0.6 * scale) * (0.02 / 112)


def _padded(codes, to=16):
    """Rows of codes, a multiple of 16 bytes apart."""
    room = torch.zeros(*codes.shape[:-1], -(-codes.shape[-1] // to) * to, dtype=codes.dtype, device=codes.device)
    room.view(torch.uint8)[..., :codes.shape[-1]] = codes.view(torch.uint8)
    return room


def _rows(g, rows, K):
    """Quantized rows: channels of different sizes, as a norm's output has them."""
    x = torch.randn(rows, K, generator=g, device="cuda")
    x *= 1 + 7 * (torch.rand(K, generator=g, device="cuda") < 0.02)
    codes, scale = _quantized(x)
    return _padded(codes), scale


def _wide(width, type):
    """Values that rows of `width` are apart: a multiple of 16 bytes."""
    by = 4 if type == "f32" else 8
    return -(-width // by) * by


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    kind, s = case["kind"], dict(case=case)
    if kind == "sort":
        s["ids"] = _routing(case, seed).cuda()
        P = case["tokens"] * case["topk"]
        s.update(start=torch.zeros(case["experts"] + 1, dtype=torch.int32, device="cuda"),
                 frm=torch.zeros(P, dtype=torch.int32, device="cuda"),
                 pos=torch.zeros(case["tokens"], case["topk"], dtype=torch.int32, device="cuda"))
        return s
    dt = TYPES[case["type"]]
    if kind == "quantize":
        n, K = case["rows"], case["K"]
        x = torch.randn(n, _wide(K, case["type"]) + case["pad"], generator=g, device="cuda")
        x *= 1 + 7 * (torch.rand(x.shape[1], generator=g, device="cuda") < 0.02)
        s.update(x=x.to(dt), codes=torch.zeros(n, -(-K // 16) * 16, dtype=torch.float8_e4m3fn, device="cuda"),
                 scale=torch.zeros(-(-K // BLOCK), n, device="cuda"))
        return s
    N = case["N"]
    wide = _wide(N, case["type"])
    if kind == "mul":
        n, K = case["rows"], case["K"]
        s["x"], s["xs"] = _rows(g, n, K)
        s["w"], s["ws"] = _weights(g, 1, N, K)
        if case["gated"]:
            s["u"], s["us"] = _weights(g, 1, N, K)
        s.update(add=torch.randn(n, wide, generator=g, device="cuda").to(dt) if case["add"] else None,
                 out=torch.zeros(n, wide, dtype=dt, device="cuda"))
    else:
        ids = _routing(case).cuda()
        T, k = ids.shape
        s["start"], s["frm"], s["pos"] = _sorted(ids, case["experts"])
    if kind == "group":
        K = case["K"]
        s["most"] = int(_experts_rows(case).max())
        s["x"], s["xs"] = _rows(g, T if case["gather"] else T * k, K)
        s["w"], s["ws"] = _weights(g, case["experts"], N, K)
        if case["gated"]:
            s["u"], s["us"] = _weights(g, case["experts"], N, K)
        s["out"] = torch.zeros(T * k, wide, dtype=dt, device="cuda")
    if kind == "combine":
        s["w"] = torch.softmax(torch.randn(T, k, generator=g, device="cuda"), 1)
        s["y"] = torch.randn(T * k, wide, generator=g, device="cuda").to(dt)
        s.update(add=torch.randn(T, wide, generator=g, device="cuda").to(dt) if case["add"] else None,
                 out=torch.zeros(T, wide, dtype=dt, device="cuda"))
    for name in ("w", "u"):
        if name in s and kind != "combine" and s[name].shape[-1] % 16:
            s[name] = _padded(s[name])
    return s


# --------------------------------------------------------------------------
# plain forms
# --------------------------------------------------------------------------

def _blocks(x):
    """x [..][K] as [..][blocks][128], zeros behind the last."""
    K = x.shape[-1]
    return torch.nn.functional.pad(x, (0, -K % BLOCK)).unflatten(-1, (-1, BLOCK))


def _quantized(x):
    """(codes [rows][K], scales [blocks][rows]): a scale is the block's largest magnitude / 448,
    a code the nearest e4m3 value to x / scale (64 bits: values next to a border)."""
    K = x.shape[-1]
    b = _blocks(x.double())
    s = b.abs().amax(-1)
    s = (s / torch.full_like(s, 448.0)).clamp_min(LEAST).float()
    q = b / s.double()[..., None]
    # the values next to q are a step of 2^(e - 4) apart, q = m 2^e with m in [1/2, 1)
    near = q.abs().clamp_min(2.0 ** -6)
    step = near / torch.frexp(near).mantissa / 16
    q = (torch.round(q / step) * step).clamp(-448, 448)
    return q.flatten(-2)[..., :K].float().to(torch.float8_e4m3fn).contiguous(), s.t().contiguous()


def _rows32(codes, scale, K):
    """What quantized rows stand for."""
    return (_blocks(codes[..., :K].float()) * scale.t()[..., None]).flatten(-2)[..., :K]


def _mat32(codes, scale, K):
    """What matrices [count][N][K] stand for."""
    N = codes.shape[1]
    scale = scale.repeat_interleave(BLOCK, 1)[:, :N]
    return (_blocks(codes[..., :K].float()) * scale[..., None]).flatten(-2)[..., :K]


def _gate(y, z):
    return y / (1 + torch.exp(-y)) * z


def _group_plain(s):
    case = s["case"]
    NE, N, K, most = case["experts"], case["N"], case["K"], s["most"]
    # the experts' rows, padded to the most rows that one of them has
    at = s["start"][:-1, None].long() + torch.arange(most, device="cuda")
    here = at < s["start"][1:, None]
    at = at.clamp_max(s["frm"].numel() - 1)
    x = _rows32(s["x"], s["xs"], K)[s["frm"].long()[at] if case["gather"] else at]
    y = x @ _mat32(s["w"], s["ws"], K).transpose(1, 2)
    if case["gated"]:
        y = _gate(y, x @ _mat32(s["u"], s["us"], K).transpose(1, 2))
    out = s["out"].clone()
    out[at[here], :N] = y[here].to(out.dtype)
    return out[:, :N]


def run(s):
    case = s["case"]
    kind = case["kind"]
    if own:
        return _run_own(s)
    if kind == "quantize":
        codes, scale = _quantized(s["x"][:, :case["K"]])
        return {"codes": codes, "scale": scale}
    if kind == "sort":
        start, frm, pos = _sorted(s["ids"], case["experts"])
        # places behind the last expert's rows are left as they were
        used = torch.arange(frm.numel(), device="cuda") < start[-1]
        return {"start": start, "from": torch.where(used, frm, s["frm"]), "pos": pos}
    if kind == "group":
        return _group_plain(s)
    N = case["N"]
    if kind == "mul":
        x = _rows32(s["x"], s["xs"], case["K"])
        y = x @ _mat32(s["w"], s["ws"], case["K"])[0].t()
        if case["gated"]:
            y = _gate(y, x @ _mat32(s["u"], s["us"], case["K"])[0].t())
    else:
        here = s["pos"] >= 0
        y = s["y"][s["pos"].clamp_min(0).long(), :N].float()  # [tokens][topk][N]
        y = torch.where(here[..., None], y * s["w"][..., None], 0.0).sum(1)
    if case["add"]:
        y = y + s["add"][:, :N].float()
    return y.to(s["out"].dtype)


def _run_own(s):
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "llm.c_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import hipf8
    case = s["case"]
    kind = case["kind"]
    if kind == "sort":
        hipf8.sort(s["ids"].data_ptr(), case["tokens"], case["topk"], case["experts"], s["start"].data_ptr(),
                   s["frm"].data_ptr(), s["pos"].data_ptr())
        return {"start": s["start"], "from": s["frm"], "pos": s["pos"]}
    ty = TYPE_ID[case["type"]]
    if kind == "quantize":
        n, K = case["rows"], case["K"]
        if "rows" not in s:
            s["rows"] = hipf8.Rows(s["codes"].data_ptr(), s["codes"].shape[1], s["scale"].data_ptr(), n, n, K)
        hipf8.quantize(ty, s["x"].data_ptr(), s["x"].shape[1], s["rows"])
        return {"codes": s["codes"][:, :K], "scale": s["scale"]}
    N, out = case["N"], s["out"]
    if kind == "combine":
        add = s["add"]
        hipf8.combine(ty, s["y"].data_ptr(), s["y"].shape[1], s["y"].shape[0], s["pos"].data_ptr(),
                      s["w"].data_ptr(), case["tokens"], case["topk"], N, add.data_ptr() if case["add"] else None,
                      add.shape[1] if case["add"] else 0, out.data_ptr(), out.shape[1])
        return out[:, :N]
    if "rows" not in s:  # the descriptions of the weights and rows, which a program keeps
        x, KB, NB = s["x"], -(-case["K"] // BLOCK), -(-N // BLOCK)
        s["rows"] = hipf8.Rows(x.data_ptr(), x.shape[1], s["xs"].data_ptr(), x.shape[0], x.shape[0], case["K"])
        s["mats"] = [hipf8.Mat(s[w].data_ptr(), s[w].shape[2], s[w + "s"].data_ptr(), KB, N, case["K"],
                               s[w].shape[0], s[w].shape[1] * s[w].shape[2], NB * KB)
                     for w in ("w", "u") if w in s] + [None]
    W, U = s["mats"][:2]
    if kind == "mul":
        add = s["add"]
        hipf8.mul(s["rows"], W, U, ty, out.data_ptr(), out.shape[1], add.data_ptr() if case["add"] else None,
                  add.shape[1] if case["add"] else 0)
    else:
        hipf8.group_mul(s["rows"], s["frm"].data_ptr() if case["gather"] else None, s["start"].data_ptr(),
                        out.shape[0], W, U, ty, out.data_ptr(), out.shape[1])
    return out[:, :N]


# --------------------------------------------------------------------------
# results in 64 bits, from the definitions
# --------------------------------------------------------------------------

def _e4m3_64(q):
    """The nearest e4m3 value of magnitudes q, by a table of all of them; ties to the even code."""
    value = [(m if e == 0 else 8 + m) * 2.0 ** (max(e, 1) - 10) for e in range(16) for m in range(8)][:127]
    value = torch.tensor(value, dtype=torch.float64, device=q.device)
    middle = (value[1:] + value[:-1]) / 2
    low, high = torch.bucketize(q, middle), torch.bucketize(q, middle, right=True)
    return value[torch.where(low % 2 == 0, low, high)]


def _deq64(codes, row_scale, K):
    """codes [n][..] times row_scale [n][blocks]."""
    x = codes[:, :K].double()
    return x * row_scale.double()[:, torch.arange(K, device=x.device) // BLOCK]


def _mat64(codes, scale, K):
    return _deq64(codes, scale[torch.arange(codes.shape[0], device=codes.device) // BLOCK], K)


def _product64(s, x, e, K):
    y = x @ _mat64(s["w"][e], s["ws"][e], K).t()
    if "u" not in s:
        return y
    return y * torch.sigmoid(y) * (x @ _mat64(s["u"][e], s["us"][e], K).t())


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "sort":
        ids, NE = s["ids"].tolist(), case["experts"]
        if len(ids) > 1024:
            return None  # whole numbers
        of = [[(t, k) for t, row in enumerate(ids) for k, i in enumerate(row) if i == e] for e in range(NE)]
        start, frm, pos = [0], [], torch.full((case["tokens"], case["topk"]), -1, dtype=torch.int32)
        for pairs in of:
            for t, k in pairs:
                pos[t, k] = len(frm)
                frm.append(t)
            start.append(len(frm))
        frm += [0] * (case["tokens"] * case["topk"] - len(frm))
        return {"start": torch.tensor(start, dtype=torch.int32), "from": torch.tensor(frm, dtype=torch.int32), "pos": pos}
    if kind == "quantize":
        K = case["K"]
        x = s["x"][:, :K].double()
        KB = -(-K // BLOCK)
        room = torch.zeros(x.shape[0], KB * BLOCK, dtype=torch.float64, device="cuda")
        room[:, :K] = x
        top = room.view(-1, KB, BLOCK).abs().max(-1).values
        exactly = (top / torch.full_like(top, 448)).clamp_min(LEAST)
        q = x.abs() / exactly.float().double().repeat_interleave(BLOCK, 1)[:, :K]
        return {"codes": torch.copysign(_e4m3_64(q), x), "scale": exactly.t().contiguous()}
    if kind == "combine":
        N = case["N"]
        y = torch.zeros(case["tokens"], N, dtype=torch.float64, device="cuda")
        if case["add"]:
            y += s["add"][:, :N].double()
        for k in range(case["topk"]):
            here = (s["pos"][:, k] >= 0).nonzero().flatten()
            y[here] += s["w"][here, k, None].double() * s["y"][s["pos"][here, k].long(), :N].double()
        return y
    K, N = case["K"], case["N"]
    x = _deq64(s["x"], s["xs"].t(), K)
    if kind == "mul":
        y = _product64(s, x, 0, K)
        return y + s["add"][:, :N].double() if case["add"] else y
    out = torch.zeros(s["out"].shape[0], N, dtype=torch.float64, device="cuda")
    start = s["start"].tolist()
    for e in range(case["experts"]):
        a, b = start[e], start[e + 1]
        if b > a:
            out[a:b] = _product64(s, x[s["frm"][a:b].long()] if case["gather"] else x[a:b], e, K)
    return out
