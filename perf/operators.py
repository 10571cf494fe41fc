"""Workloads of the serving operators: normed and rotated queries and keys, the 4-bit key/value
cache, single-token attention over that cache, and windowed attention over packed prompts.

``run`` computes each operator in its plain form (elementary torch operations in 32 bits) while
``own`` is false, and calls ``shapeforge_b200.ops`` while it is true.  ``exact`` is the operator's
definition in 64 bits.

The 4-bit cache, [pages, heads, page_size / 16, 18 * D] bytes, holds for every 16 tokens of a head
one record: key codes (16 rows of D / 2 bytes), value codes (the same), then (scale, minimum) in
bf16 for every row and every group of 64 elements, of the keys and of the values.  A code q stands
for minimum + scale * q.  In a row, with G = d // 64 and N = D / 64:
  keys    d = 64 G + 16 t + 8 h + n   is in byte  t * 8 N + G * 8 + h * 4 + n // 2,
  values  d = 64 G + 8 c + n          is in byte  (c ^ 4 ((row >> 1) & 1)) * 4 N + G * 4 + n // 2,
the even n in the low four bits.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ---- cases --------------------------------------------------------------------------------------


def listed():
    return [
        # One decoding step of a batch: latency counts.
        {"name": "norm_rope_decode", "op": "norm_rope", "tokens": 64, "hq": 32, "hk": 8, "dim": 128, "rotary": 128, "dtype": "bf16", "far": 131072},
        # A prompt batch; q and k are views of the packed projection.
        {"name": "norm_rope_prompt", "op": "norm_rope", "tokens": 16384, "hq": 32, "hk": 8, "dim": 128, "rotary": 128, "dtype": "bf16", "far": 32768},
        # Odd token count, few heads, half of each head rotated.
        {"name": "norm_rope_partial", "op": "norm_rope", "tokens": 4099, "hq": 12, "hk": 4, "dim": 64, "rotary": 32, "dtype": "fp16", "far": 1048576},
        # The step's new tokens into their pages, and back.
        {"name": "kv4_step", "op": "kv4", "tokens": 64, "hk": 8, "dim": 128, "page": 64, "dtype": "bf16"},
        # A long prompt into the cache, and back for the next chunk of it.
        {"name": "kv4_prompt", "op": "kv4", "tokens": 32768, "hk": 8, "dim": 128, "page": 64, "dtype": "bf16"},
        # One request, moderate context: latency and the split over the keys.
        {"name": "decode_single", "op": "decode", "batch": 1, "longest": 4097, "hq": 32, "hk": 8, "dim": 128, "page": 64, "window": 0, "sinks": 0, "dtype": "bf16"},
        # A full batch of ragged contexts, a windowed layer with sinks.
        {"name": "decode_window", "op": "decode", "batch": 64, "longest": 8192, "hq": 32, "hk": 8, "dim": 128, "page": 64, "window": 1024, "sinks": 4, "dtype": "bf16"},
        # The same kind of batch, a layer that sees everything: bandwidth counts.
        {"name": "decode_full", "op": "decode", "batch": 32, "longest": 16384, "hq": 64, "hk": 8, "dim": 128, "page": 64, "window": 0, "sinks": 0, "dtype": "bf16"},
        # Few wide head groups, short pages, the other type and head size.
        {"name": "decode_wide_group", "op": "decode", "batch": 17, "longest": 5001, "hq": 24, "hk": 2, "dim": 64, "page": 16, "window": 0, "sinks": 0, "dtype": "fp16"},
        # A handful of short prompts, ragged.
        {"name": "prompt_short", "op": "window", "seqs": 9, "tokens": 1203, "context": 0, "hq": 32, "hk": 8, "dim": 128, "window": 128, "sinks": 4, "dtype": "bf16"},
        # A long prompt through a windowed layer.
        {"name": "prompt_window", "op": "window", "seqs": 1, "tokens": 16384, "context": 0, "hq": 16, "hk": 2, "dim": 128, "window": 4096, "sinks": 4, "dtype": "bf16"},
        # The next chunks of three prompts behind contexts that were read back from the cache.
        {"name": "prompt_chunk", "op": "window", "seqs": 3, "tokens": 1536, "context": 8200, "hq": 28, "hk": 4, "dim": 128, "window": 0, "sinks": 0, "dtype": "fp16"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm_rope", "kv4", "decode", "decode", "window", "window"])
    dim = rng.choice([64, 128, 128])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    group, hk = rng.choice([(1, 8), (2, 4), (3, 4), (4, 8), (5, 3), (7, 4), (8, 4), (8, 8), (12, 2), (16, 1)])
    hq = group * hk
    if op == "norm_rope":
        tokens = min(_log(rng, 1, 16384), 16384 * 40 // (hq + hk))
        return {"op": op, "tokens": tokens, "hq": hq, "hk": hk, "dim": dim, "rotary": rng.choice([dim, dim, dim // 2]), "dtype": dtype,
                "far": _log(rng, 4096, 1 << 20)}
    if op == "kv4":
        return {"op": op, "tokens": _log(rng, 1, 32768), "hk": hk, "dim": dim, "page": rng.choice([16, 32, 64, 128]), "dtype": dtype}
    window = rng.choice([0, 0, _log(rng, 16, 4096)])
    sinks = rng.choice([0, 1, 4, 16, 130]) if window else 0
    if op == "decode":
        batch = _log(rng, 1, 128)
        longest = min(_log(rng, 16, 65536), max(16, 32 * 16384 * 64 // (batch * max(64, hq))))
        return {"op": op, "batch": batch, "longest": longest, "hq": hq, "hk": hk, "dim": dim, "page": rng.choice([16, 32, 64, 128]),
                "window": window, "sinks": sinks, "dtype": dtype}
    tokens = min(_log(rng, 1, 10800), int(10800 * math.sqrt(16 / max(16, hq))))
    context = rng.choice([0, 0, _log(rng, 1, 8192)])
    seqs = min(_log(rng, 1, 32), tokens)
    if seqs * context > 24600 or hq * tokens * (tokens + seqs * context) > 16 * 10800 * 10800:
        context = 0
    return {"op": op, "seqs": seqs, "tokens": tokens, "context": context, "hq": hq, "hk": hk, "dim": dim, "window": window, "sinks": sinks,
            "dtype": dtype}


# ---- inputs -------------------------------------------------------------------------------------


def _randn(gen, *shape):
    return torch.randn(*shape, device="cuda", generator=gen)


def _split_lengths(total, parts, gen):
    """`parts` lengths of at least 1 that sum to `total` (host)."""
    if parts == 1:
        return [total]
    cuts = (torch.randperm(total - 1, generator=gen)[: parts - 1] + 1).sort().values.tolist()
    return [b - a for a, b in zip([0, *cuts], [*cuts, total])]


def _decode_lengths(case, seed):
    """Context lengths of a ragged batch: one of the longest, the others spread below it (host)."""
    gen = torch.Generator().manual_seed(seed * 2 + 1)
    n, b = case["longest"], case["batch"]
    lens = (torch.rand(b, generator=gen) * n).long() + 1
    lens[int(torch.randint(b, (1,), generator=gen))] = n
    return lens.clamp(max=n)


def _random_cache(gen, pages, heads, page, dim):
    """A filled cache: codes as quantised normal values have them, scales and minima to match."""
    tiles, groups = page // 16, dim // 64
    shape = (pages, heads, tiles)
    cache = torch.empty(*shape, 18 * dim, dtype=torch.uint8, device="cuda")
    flat = cache.view(-1, 18 * dim)
    step = 1 << 15
    for i in range(0, flat.shape[0], step):
        part = flat[i : i + step]
        codes = (_randn(gen, part.shape[0], 16 * dim, 2).mul_(2.9).add_(7.5)).round_().clamp_(0, 15).to(torch.uint8)
        part[:, : 16 * dim] = codes[..., 0] | (codes[..., 1] << 4)
        scale = torch.rand(part.shape[0], 32 * groups, device="cuda", generator=gen) * 0.2 + 0.25
        low = -scale * (7.0 + torch.rand(part.shape[0], 32 * groups, device="cuda", generator=gen))
        part[:, 16 * dim :] = torch.stack([scale, low], dim=-1).to(torch.bfloat16).view(part.shape[0], -1).view(torch.uint8)
    return cache


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    host = torch.Generator().manual_seed(seed * 2 + 1)
    dt, op, dim = DTYPES[case["dtype"]], case["op"], case["dim"]
    state = dict(case)
    if op == "norm_rope":
        t, hq, hk = case["tokens"], case["hq"], case["hk"]
        # The projection's output, [T, (hq + 2 hk) * D]: q and k are views of it.
        packed = _randn(gen, t, hq + 2 * hk, dim).to(dt)
        state["q"], state["k"] = packed[:, :hq], packed[:, hq : hq + hk]
        state["wq"], state["wk"] = ((1 + 0.2 * _randn(gen, dim)).to(dt) for _ in range(2))
        state["positions"] = torch.randint(case["far"], (t,), device="cuda", generator=gen, dtype=torch.int32)
    elif op == "kv4":
        t, hk, page = case["tokens"], case["hk"], case["page"]
        pages = -(-t // page) + 8
        state["cache"] = torch.zeros(pages, hk, page // 16, 18 * dim, dtype=torch.uint8, device="cuda")
        # Keys have channels of their own size, as they do after a norm with weights.
        state["k"] = (_randn(gen, t, hk, dim) * (0.5 + torch.rand(dim, device="cuda", generator=gen))).to(dt)
        state["v"] = _randn(gen, t, hk, dim).to(dt)
        # Consecutive tokens of a request share a page; the pages are in any order.
        order = torch.randperm(pages, device="cuda", generator=gen)
        at = torch.arange(t, device="cuda")
        state["slots"] = (order[at // page] * page + at % page).to(torch.int32)
    elif op == "decode":
        b, hq, hk, page = case["batch"], case["hq"], case["hk"], case["page"]
        lens = _decode_lengths(case, seed)
        need = -(-lens // page)
        width, pages = -(-case["longest"] // page), int(need.sum()) + 3
        order = torch.randperm(pages, generator=host)
        first = torch.cumsum(need, 0) - need
        table = order[(first[:, None] + torch.arange(width)[None]).clamp(max=pages - 1)]
        table[torch.arange(width)[None] >= need[:, None]] = 0
        state["cache"] = _random_cache(gen, pages, hk, page, dim)
        state["table"] = table.to(torch.int32).cuda()
        state["lens"] = lens.to(torch.int32).cuda()
        state["q"] = _randn(gen, b, hq, dim).to(dt)
    else:
        hq, hk = case["hq"], case["hk"]
        lq = _split_lengths(case["tokens"], case["seqs"], host)
        lk = [n + case["context"] for n in lq]
        state["cu_q"] = torch.tensor([0, *lq], dtype=torch.int32).cumsum(0).to(torch.int32).cuda()
        state["cu_k"] = torch.tensor([0, *lk], dtype=torch.int32).cumsum(0).to(torch.int32).cuda()
        state["q"] = _randn(gen, sum(lq), hq, dim).to(dt)
        state["k"] = _randn(gen, sum(lk), hk, dim).to(dt)
        state["v"] = _randn(gen, sum(lk), hk, dim).to(dt)
    return state


# ---- the operators as a user's program calls them -----------------------------------------------


def _own(s):
    from shapeforge_b200 import ops

    if s["op"] == "norm_rope":
        return ops.qk_norm_rope(s["q"], s["k"], s["wq"], s["wk"], s["positions"], base=1e6, eps=1e-6, rotary_dim=s["rotary"])
    if s["op"] == "kv4":
        ops.kv4_store(s["k"], s["v"], s["slots"], s["cache"])
        return ops.kv4_load(s["cache"], s["slots"], s["k"].dtype)
    if s["op"] == "decode":
        return ops.kv4_attention(s["q"], s["cache"], s["table"], s["lens"], s["dim"] ** -0.5, window=s["window"], sinks=s["sinks"])
    return ops.window_attention(s["q"], s["k"], s["v"], s["cu_q"], s["dim"] ** -0.5, window=s["window"], sinks=s["sinks"],
                                cu_seqlens_k=s["cu_k"])


def run(state):
    if own:
        return _own(state)
    if state["op"] == "norm_rope":
        return _plain_norm_rope(state)
    if state["op"] == "kv4":
        return _plain_kv4(state)
    if state["op"] == "decode":
        return _plain_decode(state)
    return _plain_window(state)


# ---- plain forms --------------------------------------------------------------------------------


def _plain_norm_rope(s):
    half = s["rotary"] // 2
    freq = 1e6 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
    angle = s["positions"].double()[:, None, None] * freq
    cos, sin = angle.cos().float(), angle.sin().float()

    def one(x, w):
        x = x.float()
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w.float()
        a, b, rest = x[..., :half], x[..., half : 2 * half], x[..., 2 * half :]
        return torch.cat([a * cos - b * sin, a * sin + b * cos, rest], dim=-1)

    return one(s["q"], s["wq"]).to(s["q"].dtype), one(s["k"], s["wk"]).to(s["k"].dtype)


def _quantise(x):
    """Codes (uint8), scales and minima (bf16 values in fp32) of groups of 64: [..., G, 64], [..., G]."""
    x = x.float().unflatten(-1, (-1, 64))
    low = x.amin(-1)
    # A quotient of tensors: torch multiplies by 1 / 15 where the divisor is a number.
    scale = ((x.amax(-1) - low) / torch.full_like(low, 15)).bfloat16().float()
    low = low.bfloat16().float()
    codes = ((x - low[..., None]) / scale[..., None]).round().nan_to_num(0).clamp(0, 15)
    return codes.to(torch.uint8), scale, low


def _swap(rows, codes):
    """Value chunks [tokens, heads, 8, ...]: the upper and lower four change places in rows 2, 3 of every 4."""
    odd = ((rows >> 1) & 1).bool()[:, None, None, None, None]
    return torch.where(odd, codes.roll(4, 2), codes)


def _tile_rows(s):
    """The records as [pages * tiles, heads, 18 * D], and each slot's record and row."""
    cache = s["cache"]
    per = cache.shape[2]
    slot = s["slots"].long()
    return cache, slot // (16 * per), (slot // 16) % per, slot % 16


def _plain_kv4(s):
    cache, page, tile, row = _tile_rows(s)
    t, hk, d = s["k"].shape
    g = d // 64
    rows = cache[..., : 16 * d].view(*cache.shape[:3], 2, 16, d // 2)
    params = cache[..., 16 * d :].view(torch.bfloat16).view(*cache.shape[:3], 2, 16, g, 2)
    heads = torch.arange(hk, device="cuda")[None]
    at = (page[:, None], heads, tile[:, None])
    for which, x in ((0, s["k"]), (1, s["v"])):
        codes, scale, low = _quantise(x)
        both = codes.unflatten(-1, (-1, 2))
        packed = both[..., 0] | (both[..., 1] << 4)  # [T, H, G, 32]
        if which == 0:
            packed = packed.unflatten(-1, (4, 8)).transpose(2, 3)  # t, G, (h, n/2)
        else:
            packed = _swap(row, packed.unflatten(-1, (8, 4)).transpose(2, 3))  # c, G, n/2
        rows[(*at, which, row[:, None])] = packed.reshape(t, hk, d // 2)
        params[(*at, which, row[:, None])] = torch.stack([scale, low], dim=-1).bfloat16()
    back = []
    for which in (0, 1):
        packed = rows[(*at, which, row[:, None])]
        if which == 0:
            packed = packed.view(t, hk, 4, g, 8).transpose(2, 3)
        else:
            packed = _swap(row, packed.view(t, hk, 8, g, 4)).transpose(2, 3)
        packed = packed.reshape(t, hk, g, 32)
        codes = torch.stack([packed & 15, packed >> 4], dim=-1).flatten(-2).float()
        p = params[(*at, which, row[:, None])].float()
        back.append((p[..., 1:] + p[..., :1] * codes).flatten(-2).to(s["k"].dtype))
    return tuple(back)


def _dequantise(tiles, dim):
    """Records [..., 18 * D] to keys and values [..., 16, D] in fp32."""
    g = dim // 64
    lead = tiles.shape[:-1]
    packed = tiles[..., : 16 * dim].unflatten(-1, (2, 16, dim // 2))
    params = tiles[..., 16 * dim :].contiguous().view(torch.bfloat16).view(*lead, 2, 16, g, 2).float()
    key = packed[..., 0, :, :].unflatten(-1, (4, g, 8)).transpose(-3, -2).reshape(*lead, 16, g, 32)
    val = packed[..., 1, :, :].unflatten(-1, (8, g, 4))
    odd = (torch.arange(16, device="cuda") >> 1 & 1).bool()[:, None, None, None]
    val = torch.where(odd, val.roll(4, -3), val).transpose(-3, -2).reshape(*lead, 16, g, 32)
    out = []
    for which, p in ((0, key), (1, val)):
        codes = torch.stack([p & 15, p >> 4], dim=-1).flatten(-2).float()
        out.append((params[..., which, :, :, 1:] + params[..., which, :, :, :1] * codes).flatten(-2))
    return out


def _plain_decode(s):
    b, hq, d = s["q"].shape
    hk = s["hk"]
    tiles = s["cache"][s["table"].long()].transpose(1, 2).flatten(2, 3)  # [B, H, tiles, 18 D]
    k, v = (x.flatten(2, 3) for x in _dequantise(tiles, d))  # [B, H, S, D]
    scores = s["q"].float().view(b, hk, hq // hk, d) @ k.transpose(-1, -2) * d**-0.5
    j, n = torch.arange(k.shape[2], device="cuda")[None], s["lens"].long()[:, None]
    seen = j < n
    if s["window"]:
        seen &= (j >= n - s["window"]) | (j < s["sinks"])
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    p = (scores - scores.amax(-1, keepdim=True)).exp()
    return ((p / p.sum(-1, keepdim=True)) @ v).view(b, hq, d).to(s["q"].dtype)


def _plain_window(s):
    t, hq, d = s["q"].shape
    tk, hk = s["k"].shape[:2]
    cu_q, cu_k = s["cu_q"].long(), s["cu_k"].long()
    i, j = torch.arange(t, device="cuda"), torch.arange(tk, device="cuda")
    sq, sk = (torch.searchsorted(cu[1:], x, right=True) for cu, x in ((cu_q, i), (cu_k, j)))
    pos = i - cu_q[sq] + (cu_k[sq + 1] - cu_k[sq]) - (cu_q[sq + 1] - cu_q[sq])
    key = (j - cu_k[sk])[None]
    seen = (sq[:, None] == sk[None]) & (key <= pos[:, None])
    if s["window"]:
        seen &= (key > pos[:, None] - s["window"]) | (key < s["sinks"])
    q = s["q"].float().view(t, hk, hq // hk, d).permute(1, 2, 0, 3)
    p = (q @ s["k"].float().permute(1, 2, 0)[:, None]).mul_(d**-0.5).masked_fill_(~seen, -math.inf)
    p = p.sub_(p.amax(-1, keepdim=True)).exp_()
    p = p.div_(p.sum(-1, keepdim=True))
    return (p @ s["v"].float().transpose(0, 1)[:, None]).permute(2, 0, 1, 3).reshape(t, hq, d).to(s["q"].dtype)


# ---- the work that cannot be left out -----------------------------------------------------------


def _seen(n, window, sinks):
    return n if not window else min(n, window + min(sinks, max(0, n - window)))


def work(case):
    op, d = case["op"], case["dim"]
    if op == "norm_rope":
        rows = case["tokens"] * (case["hq"] + case["hk"])
        return {"bytes": rows * d * 4 + case["tokens"] * 4 + 4 * d, "flops": rows * d * 8}
    if op == "kv4":
        # Values in and out in 16 bits, records written and read.
        rows = case["tokens"] * case["hk"]
        return {"bytes": rows * (8 * d + 2 * (18 * d) // 16) + 8 * case["tokens"], "flops": rows * d * 2 * 8}
    if op == "decode":
        # The lengths are those of seed 0: other seeds' differ a little.
        keys = sum(_seen(int(n), case["window"], case["sinks"]) for n in _decode_lengths(case, 0))
        rows = case["batch"] * case["hq"] * d
        return {"bytes": keys * case["hk"] * (18 * d) // 16 + 4 * rows + 4 * keys // case["page"], "flops": 4 * keys * case["hq"] * d}
    # Equal lengths stand for the ragged ones.
    per, rest = divmod(case["tokens"], case["seqs"])
    pairs = 0
    for n, many in ((per, case["seqs"] - rest), (per + 1, rest)):
        if many:
            c, w, k = case["context"], case["window"], case["sinks"]
            pairs += many * (n * c + n * (n + 1) // 2 if not w else sum(_seen(p + 1, w, k) for p in range(c, c + n)))
    tk = case["tokens"] + case["seqs"] * case["context"]
    return {"bytes": 4 * case["tokens"] * case["hq"] * d + 4 * tk * case["hk"] * d, "flops": 4 * pairs * case["hq"] * d}


# ---- the definitions in 64 bits -----------------------------------------------------------------


def _exact_norm_rope(s):
    m = s["rotary"] // 2
    outs = []
    for x, w in ((s["q"], s["wq"]), (s["k"], s["wk"])):
        x = x.to(torch.float64)
        y = x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + 1e-6) * w.to(torch.float64)
        turn = s["positions"].to(torch.float64).view(-1, 1, 1) * torch.exp(-math.log(1e6) * torch.arange(m, device="cuda", dtype=torch.float64) / m)
        z = torch.complex(y[..., :m], y[..., m : 2 * m]) * torch.polar(torch.ones_like(turn), turn)
        outs.append(torch.cat([z.real, z.imag, y[..., 2 * m :]], dim=-1))
    return tuple(outs)


def _exact_kv4(s):
    outs = []
    for x in (s["k"], s["v"]):
        t, h, d = x.shape
        x = x.to(torch.float64).reshape(t * h * d // 64, 64)
        low, high = x.min(1, keepdim=True).values, x.max(1, keepdim=True).values
        scale = ((high - low) / 15).to(torch.bfloat16).to(torch.float64)
        low = low.to(torch.bfloat16).to(torch.float64)
        code = torch.where(scale > 0, torch.round((x - low) / torch.where(scale > 0, scale, 1.0)), 0.0).clamp(0, 15)
        outs.append((low + scale * code).view(t, h, d))
    return tuple(outs)


def _byte_of(dim, which, row):
    """Byte and shift of every element of a row, from the layout's definition."""
    n_groups = dim // 64
    d = torch.arange(dim, device="cuda")
    big, n = d // 64, d % 8
    if which == 0:
        byte = (d % 64 // 16) * 8 * n_groups + big * 8 + (d % 16 // 8) * 4 + n // 2
    else:
        byte = ((d % 64 // 8) ^ (4 * (row >> 1 & 1))) * 4 * n_groups + big * 4 + n // 2
    return byte, 4 * (n % 2)


def _exact_decode(s):
    b, hq, d = s["q"].shape
    hk, page, groups = s["hk"], s["page"], d // 64
    outs = torch.zeros(b, hq, d, dtype=torch.float64, device="cuda")
    lens, maps = s["lens"].tolist(), [[_byte_of(d, w, r) for r in range(16)] for w in (0, 1)]
    byte = torch.stack([torch.stack([m[0] for m in maps[w]]) for w in (0, 1)])  # [2, 16, D]
    shift = torch.stack([torch.stack([m[1] for m in maps[w]]) for w in (0, 1)])
    start = (torch.arange(2, device="cuda")[:, None, None] * 16 + torch.arange(16, device="cuda")[None, :, None]) * (d // 2)
    for i in range(b):
        n = lens[i]
        keep = torch.arange(n, device="cuda")
        if s["window"]:
            keep = keep[(keep >= n - s["window"]) | (keep < s["sinks"])]
        tiles = torch.unique(keep // 16)
        rec = s["cache"][s["table"][i, (tiles * 16 // page)].long(), :, tiles % (page // 16)]  # [tiles, H, 18 D]
        codes = rec[..., (start + byte).flatten()].view(*rec.shape[:2], 2, 16, d)
        codes = ((codes >> shift.to(torch.uint8)) & 15).to(torch.float64)
        par = rec[..., 16 * d :].contiguous().view(torch.bfloat16).view(*rec.shape[:2], 2, 16, groups, 2).to(torch.float64)
        val = par[..., 1].repeat_interleave(64, -1) + par[..., 0].repeat_interleave(64, -1) * codes
        where = (tiles[:, None] * 16 + torch.arange(16, device="cuda")).flatten()
        good = torch.isin(where, keep)
        k, v = (val[:, :, w].transpose(0, 1).reshape(hk, -1, d)[:, good] for w in (0, 1))
        q = s["q"][i].to(torch.float64).view(hk, hq // hk, d)
        outs[i] = (torch.softmax(torch.bmm(q, k.transpose(1, 2)) / math.sqrt(d), dim=-1) @ v).view(hq, d)
    return outs


def _exact_window(s):
    t, hq, d = s["q"].shape
    hk = s["k"].shape[1]
    cu_q, cu_k = s["cu_q"].tolist(), s["cu_k"].tolist()
    out = torch.zeros(t, hq, d, dtype=torch.float64, device="cuda")
    for a, b, e, f in zip(cu_q, cu_q[1:], cu_k, cu_k[1:]):
        k, v = (x[e:f].to(torch.float64).transpose(0, 1).repeat_interleave(hq // hk, 0) for x in (s["k"], s["v"]))
        for r in range(a, b, 1024):
            q = s["q"][r : min(b, r + 1024)].to(torch.float64).transpose(0, 1)
            pos = (f - e) - (b - r) + torch.arange(q.shape[1], device="cuda")[:, None]
            key = torch.arange(f - e, device="cuda")[None]
            seen = key <= pos
            if s["window"]:
                seen = seen & ((pos - key < s["window"]) | (key < s["sinks"]))
            w = torch.where(seen, torch.bmm(q, k.transpose(1, 2)) / math.sqrt(d), -math.inf)
            out[r : r + q.shape[1]] = torch.bmm(torch.softmax(w, dim=-1), v).transpose(0, 1)
    return out


def exact(case, seed):
    state = prepare(case, seed)
    return {"norm_rope": _exact_norm_rope, "kv4": _exact_kv4, "decode": _exact_decode, "window": _exact_window}[case["op"]](state)
