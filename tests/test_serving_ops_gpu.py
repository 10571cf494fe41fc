"""The serving operators on the B200 against their 64-bit definitions (oracle/serving.py).

Tolerances.  Every output is rounded once to its type: half a step, u |value| with u = eps / 2 (bf16
2^-8, fp16 2^-11; the smallest subnormal step where that is larger).  On top of that
 * qk_norm_rope: fp32 arithmetic on both members of a pair (norm: a sum of D squares, relative 2^-18 at
   D <= 512 at worst; sine and cosine 2^-20 absolute), 2^-17 (|a| + |b|);
 * kv4_store / kv4_load: the codes are exact and the value is one fp32 fma, so the rounded value is
   reproduced bit for bit;
 * attention: each weight is rounded once before P.V, by at most half a step of the type it is rounded
   to (bf16 2^-8, fp16 2^-11 relative), which moves the result by at most that times sum p |v - centre|;
   an fp16 weight in its subnormal range is off by up to 2^-25 of the unit it is held in, n of them by
   n 2^-25 max |v|.  A score of D products in fp32 is off by at most (D + 16) 2^-23 max sum |q k| scale,
   which moves weights by twice that relative to sum p |v|; exponential and sums 2^-19 of it.
 * attention over the cache holds every weight times scale as fp16 (2^-11 whatever the tensors' type) in a
   unit of at most the head's largest weight times scale, and a value as a code within 8 of its centre:
   subnormal weights give n 2^-25 8 max p scale.  An element comes out of the difference of two fp32 sums of
   whole bytes, 17 times the code's size, over n / 128 steps a warp and 9 to join, each relative to a sum
   of at most n weights: (n / 128 + 9) 2^-23 17 n 8 max p scale.
"""

from __future__ import annotations

import math

import pytest
import torch

from oracle import serving
from shapeforge_b200 import _native, ops

pytestmark = pytest.mark.gpu

TD = {"bf16": torch.bfloat16, "fp16": torch.float16}
U = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
TINY = {torch.bfloat16: 2.0**-133, torch.float16: 2.0**-24}


@pytest.fixture(autouse=True)
def _status(cuda_device):
    ops.kernel_status()
    yield
    assert ops.kernel_status() == (0, 0)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, device="cuda", generator=g).to(dtype)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def close(got, want, slack):
    """|got - want| <= half a step of the type + slack, NaN and infinities alike."""
    g = got.double()
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(g), nan), f"NaN in {int(torch.isnan(g).sum())} places, expected {int(nan.sum())}"
    inf = torch.isinf(want)
    assert torch.equal(g[inf], want[inf])
    ok = ~nan & ~inf
    limit = U[got.dtype] * want.abs() * (1 + 2.0**-7) + TINY[got.dtype] + slack * (1 + U[got.dtype])
    over = ((g - want).abs() - limit)[ok]
    assert not over.numel() or over.max() <= 0, f"off by {over.max().item():.3g} more than the limit; worst error {(g - want).abs()[ok].max().item():.3g}"


def attention_slack(r, d, n, p_rounding, fp16_p=False):
    slack = p_rounding * r.mass + ((d + 16) * 2.0**-23 * r.score * 2 + 2.0**-19) * r.size
    return slack + (n * 2.0**-25 * r.peak if fp16_p else 0)


# ---- qk_norm_rope -------------------------------------------------------------------------------


def check_norm_rope(q, k, wq, wk, pos, outs, base=10000.0, eps=1e-6, rotary=None):
    rotary = q.shape[2] if rotary is None else rotary
    for x, w, got in ((q, wq, outs[0]), (k, wk, outs[1])):
        want, size = serving.qk_norm_rope(x, w, pos, base, eps, rotary)
        close(got, want, 2.0**-17 * size)


NORM_SHAPES = [(1, 1, 1, 64, 64), (1, 32, 8, 128, 128), (7, 5, 3, 64, 32), (33, 28, 4, 128, 64), (130, 16, 1, 128, 128), (3, 2, 2, 256, 256),
               (5, 3, 1, 96, 96), (4, 3, 2, 80, 48), (6, 2, 1, 512, 128), (9, 4, 2, 20, 6), (3, 1, 1, 7, 2), (11, 3, 0, 64, 64), (11, 0, 3, 64, 64),
               (5, 2, 1, 576, 64), (17, 4, 4, 64, 0), (400, 40, 8, 128, 128)]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("shape", NORM_SHAPES, ids=["x".join(map(str, s)) for s in NORM_SHAPES])
def test_qk_norm_rope(shape, dtype):
    t, hq, hk, d, rotary = shape
    g, dt = gen(1), TD[dtype]
    q, k = randn(g, t, hq, d, dtype=dt) * 3, randn(g, t, hk, d, dtype=dt)
    wq, wk = (1 + randn(g, d) / 4).to(dt), (1 + randn(g, d) / 4).to(dt)
    pos = torch.randint(1 << 20, (t,), device="cuda", generator=g, dtype=torch.int32)
    pos[0] = 0
    outs = ops.qk_norm_rope(q, k, wq, wk, pos, base=5e5, rotary_dim=rotary)
    check_norm_rope(q, k, wq, wk, pos, outs, base=5e5, rotary=rotary)


def test_qk_norm_rope_views_in_place_and_odd_alignment():
    g = gen(2)
    for offset in (0, 1):  # one element off 16-byte alignment: the general kernel
        buf = randn(g, 9 * 10 * 64 + 8, dtype=torch.bfloat16)
        packed = buf[offset : offset + 9 * 10 * 64].view(9, 10, 64)
        q, k, rest = packed[:, :6], packed[:, 6:8], packed[:, 8:].clone()
        w = (1 + randn(g, 64) / 4).bfloat16()
        pos = torch.arange(9, device="cuda", dtype=torch.int32) * 1000
        q0, k0 = q.clone(), k.clone()
        outs = ops.qk_norm_rope(q, k, w, w, pos)
        check_norm_rope(q0, k0, w, w, pos, outs)
        back = ops.qk_norm_rope(q, k, w, w, pos, q_out=q, k_out=k)
        assert back[0] is q and torch.equal(q, outs[0]) and torch.equal(k, outs[1]) and torch.equal(packed[:, 8:], rest)


def test_qk_norm_rope_head_major_and_negative_positions():
    """[H, T, D] storage seen as [T, H, D]; positions below zero turn the other way."""
    g = gen(3)
    q = randn(g, 6, 21, 128, dtype=torch.float16).transpose(0, 1)
    k = randn(g, 2, 21, 128, dtype=torch.float16).transpose(0, 1)
    w = torch.ones(128, device="cuda", dtype=torch.float16)
    pos = torch.arange(21, device="cuda", dtype=torch.int32) * 99991 - 1000000
    out = torch.empty(6, 21, 128, device="cuda", dtype=torch.float16).transpose(0, 1)
    outs = ops.qk_norm_rope(q, k, w, w, pos, q_out=out)
    assert outs[0] is out
    check_norm_rope(q, k, w, w, pos, outs)


def test_qk_norm_rope_specials():
    """Zero rows give zeros (eps > 0); a NaN or infinity stays in its own row."""
    q = torch.zeros(4, 2, 64, device="cuda", dtype=torch.bfloat16)
    k = randn(gen(4), 4, 1, 64, dtype=torch.bfloat16)
    q[1, 0, 3], q[2, 1, 40] = math.nan, math.inf
    w = torch.ones(64, device="cuda", dtype=torch.bfloat16)
    pos = torch.arange(4, device="cuda", dtype=torch.int32)
    a, b = ops.qk_norm_rope(q, k, w, w, pos)
    assert not a[0].any() and not a[3].any() and not a[1, 1].any() and not a[2, 0].any()
    assert torch.isnan(a[1, 0]).all() and torch.isnan(a[2, 1]).any()
    check_norm_rope(k, k, w, w, pos, (b, b))


# ---- the cache ----------------------------------------------------------------------------------


def stored(x):
    """What a stored tensor reads back as: the fp32 fma of its codes, rounded to the type."""
    return serving.kv4_values(*serving.kv4_quantise(x)).float().to(x.dtype)


def same(a, b):
    assert torch.equal(torch.nan_to_num(a, nan=1.25e4), torch.nan_to_num(b, nan=1.25e4))


CACHE_SHAPES = [(1, 1, 64, 16), (5, 3, 128, 32), (67, 8, 128, 64), (300, 2, 64, 48), (33, 40, 128, 16), (1000, 1, 64, 128)]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("shape", CACHE_SHAPES, ids=["x".join(map(str, s)) for s in CACHE_SHAPES])
def test_kv4_store_and_load(shape, dtype):
    t, h, d, page = shape
    g, dt = gen(5), TD[dtype]
    pages = -(-t // page) + 2
    cache = ops.kv4_cache(pages, page, h, d)
    slots = torch.randperm(pages * page, device="cuda", generator=g)[:t].to(torch.int32)
    # Groups of very different sizes and offsets, and ties by the thousand (small integers).
    k = randn(g, t, h, d) * torch.exp(4 * randn(g, t, h, 1)) + 3 * randn(g, t, h, 1)
    v = torch.randint(-20, 21, (t, h, d), device="cuda", generator=g).float()
    k, v = k.to(dt), v.to(dt)
    assert ops.kv4_store(k, v, slots, cache) is cache
    kb, vb = ops.kv4_load(cache, slots, dt)
    same(kb, stored(k))
    same(vb, stored(v))
    # The bytes are those of the documented layout, and nothing else was touched.
    host, filled = cache.cpu(), {}
    for i, s in enumerate(slots.tolist()):
        filled.setdefault((s // page, (s % page) // 16), []).append((s % 16, i))
    (kc, ks, km), (vc, vs, vm) = serving.kv4_quantise(k), serving.kv4_quantise(v)
    for (p, tile), rows in list(filled.items())[:6]:
        codes, scale, low = serving.kv4_unpack(host[p, h - 1, tile], d)
        for row in range(16):
            i = dict(rows).get(row)
            for which, (c, s, m) in enumerate(((kc, ks, km), (vc, vs, vm))):
                assert torch.equal(codes[which, row], (c[i, h - 1].flatten().cpu() if i is not None else torch.zeros(d, dtype=torch.long)))
                assert torch.equal(scale[which, row], s[i, h - 1].cpu() if i is not None else torch.zeros(d // 64, dtype=torch.double))
                same(low[which, row], m[i, h - 1].cpu() if i is not None else torch.zeros(d // 64, dtype=torch.double))


def test_kv4_quotient_rounds_as_division_does():
    """Codes at and next to every border, over the range of scales: IEEE division decides."""
    n = 4096
    exps = torch.arange(n, device="cuda") % 200 - 100
    step = torch.exp2(exps.double()) * (1 + (torch.arange(n, device="cuda") * 37 % 128).double() / 128)
    x = (torch.arange(64, device="cuda").double() / 4)[None] * step[:, None]     # multiples of a quarter of ~ the scale
    x[:, 63] = 15 * step
    k = x.to(torch.bfloat16).view(n, 1, 64)
    cache = ops.kv4_cache(n // 16, 16, 1, 64)
    slots = torch.arange(n, device="cuda", dtype=torch.int32)
    ops.kv4_store(k, -k, slots, cache)
    kb, vb = ops.kv4_load(cache, slots)
    same(kb, stored(k))
    same(vb, stored(-k))


def test_kv4_specials_padding_and_repeats():
    g = gen(6)
    k = randn(g, 8, 2, 64, dtype=torch.bfloat16)
    k[0, 0] = 0.75                                     # a constant group: scale 0, the value itself
    k[1, 1, 5], k[2, 0, 6], k[3, 0, 7] = math.nan, math.inf, -math.inf
    k[4, 0, 0], k[4, 0, 1] = 3e38, -3e38               # a range past fp32
    k[5, 0] = randn(g, 64).bfloat16() * 2.0**-126      # subnormal values, scale 0 or subnormal
    k[5, 1, :2] = torch.tensor([1e38, -1e38])
    cache = ops.kv4_cache(2, 16, 2, 64)
    before = cache.clone()
    slots = i32([3, -1, 5, 31, 17, 9, 0, -7])
    ops.kv4_store(k, k.flip(0).contiguous(), slots, cache)
    want_k, want_v = stored(k), stored(k.flip(0))
    skip = slots < 0
    want_k[skip], want_v[skip] = 0, 0
    kb, vb = ops.kv4_load(cache, slots)
    same(kb, want_k)
    same(vb, want_v)
    rows = i32([9, 9, 3, -2, 9, 1])
    kb, _ = ops.kv4_load(cache, rows)
    zero = torch.zeros_like(want_k[0])
    same(kb, torch.stack([want_k[5], want_k[5], want_k[0], zero, want_k[5], zero]))
    # Only padding: the cache stays as it is.
    cache.copy_(before)
    ops.kv4_store(k, k, torch.full((8,), -1, device="cuda", dtype=torch.int32), cache)
    assert torch.equal(cache, before)


def test_kv4_slots_past_the_cache_are_skipped_and_reported():
    cache = ops.kv4_cache(2, 16, 1, 64)
    k = randn(gen(7), 3, 1, 64, dtype=torch.bfloat16)
    ops.kv4_store(k, k, i32([0, 32, 2**31 - 1]), cache)
    assert ops.kernel_status() == (3, 110)
    kb, _ = ops.kv4_load(cache, i32([0, 1, 31]))
    same(kb, torch.cat([stored(k[:1]), torch.zeros_like(k[:2])]))
    kb, vb = ops.kv4_load(cache, i32([32, 0]))
    assert ops.kernel_status() == (3, 111)
    assert not kb[0].any() and not vb[0].any()
    same(kb[1:], stored(k[:1]))


def test_kv4_views():
    """k and v as views of a packed projection, read back into views."""
    packed = randn(gen(8), 50, 12, 128, dtype=torch.float16)
    k, v = packed[:, 4:8], packed[:, 8:]
    cache = ops.kv4_cache(1, 64, 4, 128)
    slots = torch.arange(50, device="cuda", dtype=torch.int32)
    ops.kv4_store(k, v, slots, cache)
    out = torch.zeros(50, 8, 128, device="cuda", dtype=torch.float16)
    ops.kv4_load(cache, slots, k_out=out[:, :4], v_out=out[:, 4:])
    same(out[:, :4], stored(k))
    same(out[:, 4:], stored(v))


# ---- attention over the cache -------------------------------------------------------------------


def filled_cache(g, pages, page, h, d, dt, scale=1.0):
    cache = ops.kv4_cache(pages, page, h, d)
    n = pages * page
    k, v = randn(g, n, h, d) * scale, randn(g, n, h, d) + randn(g, 1, h, d)
    ops.kv4_store(k.to(dt), v.to(dt), torch.arange(n, device="cuda", dtype=torch.int32), cache)
    return cache, serving.kv4_quantise(k.to(dt)), serving.kv4_quantise(v.to(dt))


def check_decode(out, q, kq, vq, page, table, lens, scale, window, sinks, hidden=()):
    b, hq, d = q.shape
    h = kq[0].shape[1]
    kv, vv = serving.kv4_values(*kq), serving.kv4_values(*vq)
    centre = (vq[2] + 8 * vq[1])[..., None].expand(*vq[2].shape, 64).flatten(-2)
    cap = table.shape[1] * page
    for i in range(b):
        n = max(0, min(int(lens[i]), cap))
        j = torch.arange(n, device="cuda")
        rows = table[i].long()[j // page] * page + j % page if n else j
        seen = j >= 0
        if window:
            seen = (j >= n - window) | (j < sinks)
        for bad in hidden:
            seen = seen & (table[i].long()[j // page] != bad if n else seen)
        rows = torch.where(seen, rows, torch.zeros_like(rows))
        for c in range(h):
            g = hq // h
            r = serving.attend(q[i, c * g : (c + 1) * g], kv[rows, c], vv[rows, c], scale, seen[None].expand(g, n), centre[rows, c],
                               vq[1][rows, c].amax(-1))
            # The score's own parts (scale * code against the minimum) are up to ~4 times its size.
            r.score *= 4
            slack = attention_slack(r, d, n, 2.0**-11) + n * (2.0**-25 + (n / 128 + 9) * 2.0**-23 * 17) * 8 * r.heaviest
            close(out[i, c * g : (c + 1) * g], r.value, slack)


DECODE = [
    # batch, lengths, Hq, Hk, D, page, window, sinks
    ([1], 1, 1, 64, 16, 0, 0),
    ([1, 0, 16, 17, 15], 8, 8, 128, 16, 0, 0),
    ([33, 400, 129], 12, 4, 64, 48, 0, 0),
    ([700], 32, 4, 128, 64, 0, 0),
    ([255, 256, 257, 5], 14, 2, 128, 32, 0, 0),
    ([1000, 3, 64], 24, 2, 64, 16, 0, 0),
    ([513, 77], 16, 1, 128, 64, 0, 0),
    ([300, 40], 40, 1, 64, 32, 0, 0),
    ([4500, 1, 900, 0], 8, 1, 128, 128, 0, 0),
    ([500, 100, 20, 131, 132], 8, 2, 128, 32, 128, 4),
    ([500, 100, 21], 6, 2, 64, 16, 16, 0),
    ([500, 90, 7], 6, 2, 64, 16, 1, 1),
    ([900, 300], 4, 4, 128, 64, 250, 130),
    ([900, 300], 4, 1, 128, 64, 600, 20),
    ([900, 300], 4, 1, 64, 64, 5000, 4),
    ([260, 300], 4, 1, 64, 64, 10, 1 << 20),
]


@pytest.mark.parametrize("variant", [0, 1, 3])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("case", DECODE, ids=[f"{len(c[0])}x{max(c[0])}-{'x'.join(map(str, c[1:]))}" for c in DECODE])
def test_kv4_attention(case, dtype, variant):
    lens, hq, h, d, page, window, sinks = case
    g, dt = gen(9), TD[dtype]
    b = len(lens)
    width = -(-max(lens) // page) + 1
    pages = b * width + 1
    cache, kq, vq = filled_cache(g, pages, page, h, d, dt)
    table = torch.randperm(pages, device="cuda", generator=g)[: b * width].view(b, width).to(torch.int32)
    q = randn(g, b, hq, d, dtype=dt)
    out = torch.full((b, hq, d), math.nan, device="cuda", dtype=dt)
    assert ops.kv4_attention(q, cache, table, i32(lens), d**-0.5, window=window, sinks=sinks, out=out, variant=variant) is out
    check_decode(out, q, kq, vq, page, table, lens, d**-0.5, window, sinks)


CLUSTERS = [
    # lengths, Hq, Hk, D, page, width, window, sinks: a few requests whose (request, head) pairs go to 16, 8, 4 and 2 CTAs each
    ([1500], 8, 1, 128, 32, 60, 0, 0),
    ([1, 17, 0, 640], 32, 8, 128, 16, 41, 0, 0),
    ([700, 3, 0, 500, 111, 690, 16, 15], 64, 8, 128, 64, 11, 0, 0),
    ([300, 0, 272, 299], 64, 32, 64, 16, 19, 0, 0),
    ([2000, 90], 24, 2, 64, 16, 130, 0, 0),
    ([900, 33], 40, 1, 128, 16, 60, 0, 0),
    ([1500, 300], 16, 4, 128, 32, 60, 700, 20),
    ([1024], 5, 1, 64, 1024, 1, 0, 0),
]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("case", CLUSTERS, ids=[f"{len(c[0])}x{max(c[0])}-{'x'.join(map(str, c[1:]))}" for c in CLUSTERS])
def test_kv4_attention_in_clusters(case, dtype):
    """Small batches need no workspace; tiles that a cluster's last CTAs do not get, and empty requests, count nothing."""
    lens, hq, h, d, page, width, window, sinks = case
    g, dt, b = gen(44), TD[dtype], len(lens)
    assert ops.kv4_attention_workspace_bytes(b, hq, h, d, page, width, window, sinks) == 0
    assert ops.kv4_attention_workspace_bytes(b, hq, h, d, page, width, window, sinks, variant=1) > 0
    cache, kq, vq = filled_cache(g, b * width, page, h, d, dt)
    table = torch.randperm(b * width, device="cuda", generator=g).view(b, width).to(torch.int32)
    q = randn(g, b, hq, d, dtype=dt)
    out = torch.full((b, hq, d), math.nan, device="cuda", dtype=dt)
    ops.kv4_attention(q, cache, table, i32(lens), d**-0.5, window=window, sinks=sinks, out=out)
    check_decode(out, q, kq, vq, page, table, lens, d**-0.5, window, sinks)
    for _ in range(3):
        assert torch.equal(ops.kv4_attention(q, cache, table, i32(lens), d**-0.5, window=window, sinks=sinks), out)


def test_kv4_attention_peaked_and_large_scores():
    """Scores far apart (one key takes nearly all), growing along the keys, and large queries."""
    g = gen(10)
    cache, kq, vq = filled_cache(g, 12, 64, 2, 128, torch.bfloat16)
    table = torch.arange(12, device="cuda", dtype=torch.int32).view(1, 12)
    for factor in (1e-6, 30.0, 1e4):
        q = randn(g, 1, 8, 128, dtype=torch.bfloat16) * factor
        q[0, 3] = 0
        out = ops.kv4_attention(q, cache, table, i32([760]), 128**-0.5)
        check_decode(out, q, kq, vq, 64, table, [760], 128**-0.5, 0, 0)


def test_kv4_attention_values_of_very_different_size():
    """Values a million times larger at keys that get no weight, and at keys that get all of it: the others keep
    their precision (the weights' unit follows the scales both ways)."""
    g = gen(30)
    n, page, d = 1200, 48, 64
    for big, first in ((1e6, True), (1e6, False), (1e-6, True), (1e30, False)):
        k, v = randn(g, n, 1, d), randn(g, n, 1, d)
        rows = torch.arange(5, 200) if first else torch.arange(800, 1100)
        v[rows] *= big
        q = randn(g, 1, 4, d, dtype=torch.bfloat16)
        k[rows] = -60 * q[0, 0].float() / q[0, 0].float().norm() + 0.1 * k[rows]     # head 0 gives them nothing
        cache = ops.kv4_cache(n // page, page, 1, d)
        kb, vb = k.bfloat16(), v.bfloat16()
        ops.kv4_store(kb, vb, torch.arange(n, device="cuda", dtype=torch.int32), cache)
        table = torch.arange(n // page, device="cuda", dtype=torch.int32).view(1, -1)
        out = ops.kv4_attention(q, cache, table, i32([n]), 1.0)
        kq, vq = serving.kv4_quantise(kb), serving.kv4_quantise(vb)
        kv, vv = serving.kv4_values(*kq), serving.kv4_values(*vq)
        want = torch.softmax((q[0].double() @ kv[:, 0].T), -1) @ vv[:, 0]
        size = torch.softmax((q[0].double() @ kv[:, 0].T), -1) @ vv[:, 0].abs()
        # Of each head's own result: half a step, the weights' 2^-11, and a score error of 80 products of
        # up to 60 * 8 in all, (80 * 2^-23 * 500) = 2^-7.7 of the weights, at most.
        assert ((out[0].double() - want).abs() <= 2.0**-8 * want.abs() + (2.0**-11 + 2.0**-7) * size + 1e-30).all()


def test_kv4_attention_ignores_what_it_does_not_see():
    """NaN minima in rows past the length, before the window, in other pages and in unused table entries."""
    g = gen(11)
    cache, kq, vq = filled_cache(g, 6, 32, 2, 64, torch.bfloat16)
    table = i32([[4, 1, 3, -5, 1000], [2, 0, -1, -1, 7777]])
    lens, window, sinks = [75, 40], 30, 3
    q = randn(g, 2, 4, 64, dtype=torch.bfloat16)
    clean = ops.kv4_attention(q, cache, table, i32(lens), 0.125, window=window, sinks=sinks)
    check_decode(clean, q, kq, vq, 32, table.clamp(0, 5), lens, 0.125, window, sinks)
    junk = cache.clone()
    tiles = junk.view(6, 2, 2, -1)
    nan = torch.tensor([float("nan")] * 2, dtype=torch.bfloat16).view(torch.uint8).to("cuda")
    def spoil(page, row):
        tile, r = divmod(row, 16)
        for which in (0, 1):
            at = 16 * 64 + which * 64 + r * 4
            tiles[page, :, tile, at : at + 4] = nan
    for i, (row_pages, n) in enumerate(zip(([4, 1, 3], [2, 0]), lens)):
        for j in range(len(row_pages) * 32):
            if j >= n or (j < n - window and j >= sinks):
                spoil(row_pages[j // 32], j % 32)
    for row in range(32):
        spoil(5, row)
    for variant in (0, 1):
        assert torch.equal(ops.kv4_attention(q, junk, table, i32(lens), 0.125, window=window, sinks=sinks, variant=variant),
                           ops.kv4_attention(q, cache, table, i32(lens), 0.125, window=window, sinks=sinks, variant=variant))
    # Seen NaN reaches exactly the heads that read it.
    tiles[3, 1, 0, 16 * 64 + 64 + 5 * 4 : 16 * 64 + 64 + 5 * 4 + 4] = nan
    out = ops.kv4_attention(q, junk, table, i32(lens), 0.125, window=window, sinks=sinks)
    assert torch.isnan(out[0, 2:]).all() and torch.equal(out[0, :2], clean[0, :2]) and torch.equal(out[1], clean[1])


def test_kv4_attention_bad_pages_and_lengths():
    g = gen(12)
    cache, kq, vq = filled_cache(g, 4, 16, 1, 64, torch.bfloat16)
    table = i32([[0, 9, 2], [1, 3, -1]])
    q = randn(g, 2, 2, 64, dtype=torch.bfloat16)
    for variant in (0, 1):
        out = ops.kv4_attention(q, cache, table, i32([48, 32]), 0.125, variant=variant)
        assert ops.kernel_status() == (3, 112)
        check_decode(out, q, kq, vq, 16, table, [48, 32], 0.125, 0, 0, hidden=(9,))
        out = ops.kv4_attention(q, cache, i32([[0, 1, 2], [1, 3, 0]]), i32([-3, 2**31 - 1]), 0.125, variant=variant)
        assert ops.kernel_status() == (3, 113)
        assert not out[0].any()
        check_decode(out[1:], q[1:], kq, vq, 16, i32([[1, 3, 0]]), [48], 0.125, 0, 0)
    empty = ops.kv4_attention(q, cache, torch.empty(2, 0, dtype=torch.int32, device="cuda"), i32([0, 0]), 0.125)
    assert not empty.any()


def test_kv4_attention_strides_workspace_and_same_bits():
    g = gen(13)
    cache, kq, vq = filled_cache(g, 40, 64, 2, 128, torch.bfloat16)
    wide = torch.randperm(40, device="cuda", generator=g).to(torch.int32).view(2, 20).repeat(1, 2)
    table = wide[:, :18]
    packed = randn(g, 2, 24, 128, dtype=torch.bfloat16)
    q = packed[:, 8:16]
    out = torch.zeros(8, 2, 128, device="cuda", dtype=torch.bfloat16).transpose(0, 1)
    lens = [1100, 640]
    need = ops.kv4_attention_workspace_bytes(2, 8, 2, 128, 64, 18, variant=1)
    ws = torch.full((need + 64,), 0xAB, dtype=torch.uint8, device="cuda")
    ops.kv4_attention(q, cache, table, i32(lens), 0.1, out=out, workspace=ws[:need], variant=1)
    check_decode(out, q, kq, vq, 64, table, lens, 0.1, 0, 0)
    assert (ws[need:] == 0xAB).all()
    with pytest.raises(_native.SfError):
        ops.kv4_attention(q, cache, table, i32(lens), 0.1, workspace=ws[: need - 16], variant=1)
    for _ in range(3):
        assert torch.equal(ops.kv4_attention(q, cache, table, i32(lens), 0.1, variant=1), out)


# ---- windowed attention of prompts --------------------------------------------------------------


def cu(lens):
    return torch.tensor([0, *lens], dtype=torch.int32).cumsum(0).to(torch.int32)


def check_window(out, q, k, v, cu_q, cu_k, scale, window, sinks, variant, before=None):
    inside, r = serving.window_attention(q, k, v, cu_q.tolist(), cu_k.tolist(), scale, window, sinks)
    d, half = q.shape[2], q.dtype == torch.float16
    n = int((cu_k[1:] - cu_k[:-1]).max()) if len(cu_k) > 1 else 0
    slack = attention_slack(r, d, n, 2.0**-11 if half else 2.0**-8, fp16_p=half)
    close(out[inside], r.value[inside], slack[inside])
    if before is not None:
        assert torch.equal(out[~inside], before[~inside])


WINDOW = [
    # query lengths, contexts in front, Hq, Hk, D, window, sinks
    ([1], [0], 1, 1, 64, 0, 0),
    ([1, 1, 1], [0, 5, 300], 8, 2, 128, 0, 0),
    ([5, 0, 17, 1, 40], [0, 0, 0, 0, 0], 4, 4, 64, 0, 0),
    ([130], [0], 2, 2, 128, 0, 0),
    ([300, 77], [0, 0], 6, 2, 128, 0, 0),
    ([129, 257, 3], [100, 0, 700], 7, 1, 128, 0, 0),
    ([200], [0], 16, 1, 64, 0, 0),
    ([500, 60], [0, 0], 8, 2, 128, 128, 4),
    ([500, 60], [33, 500], 5, 1, 64, 100, 0),
    ([400], [0], 3, 1, 128, 17, 1),
    ([400], [10], 2, 2, 64, 1, 0),
    ([400], [10], 2, 1, 64, 1, 3),
    ([700], [0], 4, 1, 128, 250, 130),
    ([300], [0], 4, 2, 128, 40, 1 << 20),
    ([300], [0], 4, 2, 128, 1 << 30, 4),
    ([70], [-30], 2, 1, 128, 0, 0),
    ([90, 40], [-20, 9], 4, 1, 64, 16, 2),
    ([33], [600], 128, 1, 64, 200, 5),
    ([20], [60], 40, 2, 128, 0, 0),
]


@pytest.mark.parametrize("variant", [0, 2])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("case", WINDOW, ids=[f"{'_'.join(map(str, c[0]))}+{'_'.join(map(str, c[1]))}-{'x'.join(map(str, c[2:]))}" for c in WINDOW])
def test_window_attention(case, dtype, variant):
    lq, ctx, hq, hk, d, window, sinks = case
    g, dt = gen(14), TD[dtype]
    lk = [max(0, a + b) for a, b in zip(lq, ctx)]
    cu_q, cu_k = cu(lq), cu(lk)
    pad = 3  # rows behind the last sequence
    q = randn(g, sum(lq) + pad, hq, d, dtype=dt)
    k, v = randn(g, sum(lk) + pad, hk, d, dtype=dt), randn(g, sum(lk) + pad, hk, d, dtype=dt)
    out = torch.full_like(q, 7.5)
    before = out.clone()
    args = (q, k, v, cu_q.cuda(), d**-0.5)
    assert ops.window_attention(*args, window=window, sinks=sinks, cu_seqlens_k=cu_k.cuda(), out=out, variant=variant) is out
    check_window(out, q, k, v, cu_q, cu_k, d**-0.5, window, sinks, variant, before)


SPLIT = [
    # query lengths, contexts in front, Hq, Hk, D, window, sinks: few queries, many keys
    ([1], [4000], 8, 2, 128, 0, 0),
    ([1, 3, 40], [3000, 100, 2000], 4, 4, 64, 0, 0),
    ([2, 0, 30], [1500, 700, -10], 14, 2, 128, 0, 0),
    ([5, 1], [2600, 2100], 16, 1, 64, 1500, 4),
    ([9], [3333], 3, 1, 128, 2000, 300),
    ([130], [1900], 12, 4, 128, 0, 0),
]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("case", SPLIT, ids=[f"{'_'.join(map(str, c[0]))}+{'_'.join(map(str, c[1]))}-{'x'.join(map(str, c[2:]))}" for c in SPLIT])
def test_window_attention_split_over_keys(case, dtype):
    lq, ctx, hq, hk, d, window, sinks = case
    g, dt = gen(31), TD[dtype]
    lk = [max(0, a + b) for a, b in zip(lq, ctx)]
    cu_q, cu_k = cu(lq), cu(lk)
    q = randn(g, sum(lq) + 2, hq, d, dtype=dt)
    k, v = randn(g, sum(lk), hk, d, dtype=dt), randn(g, sum(lk), hk, d, dtype=dt)
    need = ops.window_attention_workspace_bytes(q.shape[0], k.shape[0], len(lq), hq, hk, d, window, sinks)
    assert need > 0
    ws = torch.full((need + 64,), 0xFF, dtype=torch.uint8, device="cuda")   # NaN everywhere it is not written
    out = torch.full_like(q, 7.5)
    before = out.clone()
    ops.window_attention(q, k, v, cu_q.cuda(), d**-0.5, window=window, sinks=sinks, cu_seqlens_k=cu_k.cuda(), out=out, workspace=ws[:need])
    check_window(out, q, k, v, cu_q, cu_k, d**-0.5, window, sinks, 0, before)
    assert (ws[need:] == 0xFF).all()
    for _ in range(2):
        assert torch.equal(ops.window_attention(q, k, v, cu_q.cuda(), d**-0.5, window=window, sinks=sinks, cu_seqlens_k=cu_k.cuda(),
                                                out=before.clone()), out)
    # Without a workspace of that size, or asked to, the keys stay together.
    for kw in (dict(workspace=ws[: need - 16]), dict(variant=4)):
        whole = ops.window_attention(q, k, v, cu_q.cuda(), d**-0.5, window=window, sinks=sinks, cu_seqlens_k=cu_k.cuda(), out=before.clone(), **kw)
        check_window(whole, q, k, v, cu_q, cu_k, d**-0.5, window, sinks, 0, before)


LAST_ROUND = [
    # More pairs of row tiles than SMs by a few, many keys: only the last round's are split.
    ([640], [1500], 64, 1, 64, 0, 0),
    ([400, 300, 333], [900, 2000, 1500], 40, 2, 128, 900, 4),
    ([330, 300], [2900, 3010], 64, 1, 64, 1500, 200),
    ([560, 0, 760, 20], [1100, 50, 900, 3000], 28, 4, 128, 0, 0),
    ([650, 3], [1300, 1400], 64, 1, 128, 0, 0),
]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("case", LAST_ROUND, ids=[f"{'_'.join(map(str, c[0]))}-{'x'.join(map(str, c[2:]))}" for c in LAST_ROUND])
def test_window_attention_split_in_the_last_round(case, dtype):
    lq, ctx, hq, hk, d, window, sinks = case
    g, dt = gen(45), TD[dtype]
    lk = [max(0, a + b) for a, b in zip(lq, ctx)]
    cu_q, cu_k = cu(lq), cu(lk)
    q = randn(g, sum(lq) + 2, hq, d, dtype=dt)
    k, v = randn(g, sum(lk), hk, d, dtype=dt), randn(g, sum(lk), hk, d, dtype=dt)
    need = ops.window_attention_workspace_bytes(q.shape[0], k.shape[0], len(lq), hq, hk, d, window, sinks)
    assert need > 0 or window == 900  # whose pairs differ too much for it
    ws = torch.full((need + 64,), 0xFF, dtype=torch.uint8, device="cuda")   # NaN everywhere it is not written
    out = torch.full_like(q, 7.5)
    before = out.clone()
    ops.window_attention(q, k, v, cu_q.cuda(), d**-0.5, window=window, sinks=sinks, cu_seqlens_k=cu_k.cuda(), out=out, workspace=ws[:need])
    check_window(out, q, k, v, cu_q, cu_k, d**-0.5, window, sinks, 0, before)
    assert (ws[need:] == 0xFF).all()
    v[-1, 0] = math.nan  # seen by the last query of the last sequence alone
    again = ops.window_attention(q, k, v, cu_q.cuda(), d**-0.5, window=window, sinks=sinks, cu_seqlens_k=cu_k.cuda(), out=before.clone())
    last = sum(lq) - 1
    assert torch.isnan(again[last, : hq // hk]).all()
    # Its tile's other rows are computed again key by key: not the same bits, the same bounds.
    again[last], v[-1, 0] = out[last], 0
    whole, clean = serving.window_attention(q, k, v, cu_q.tolist(), cu_k.tolist(), d**-0.5, window, sinks)
    whole[last] = False
    close(again[whole], clean.value[whole], attention_slack(clean, d, max(lk), U[dt], fp16_p=dt == torch.float16)[whole])


def test_window_attention_split_masked_specials():
    """What a query does not see stays out of its result when its keys are split, and what it sees comes in."""
    g = gen(32)
    q, k, v = randn(g, 3, 4, 128, dtype=torch.bfloat16), randn(g, 2000, 2, 128, dtype=torch.bfloat16), randn(g, 2000, 2, 128, dtype=torch.bfloat16)
    c, ck = cu([3]), cu([2000])
    clean = ops.window_attention(q, k, v, c.cuda(), 0.09, cu_seqlens_k=ck.cuda())
    assert ops.window_attention_workspace_bytes(3, 2000, 1, 4, 2, 128) > 0
    v[1998], k[1999, 1] = math.nan, math.inf   # seen by the last two queries and the last one
    out = ops.window_attention(q, k, v, c.cuda(), 0.09, cu_seqlens_k=ck.cuda())
    assert torch.isfinite(out[0]).all() and torch.isnan(out[1:]).all()
    _, r = serving.window_attention(q, k.nan_to_num(0, 0, 0), v.nan_to_num(0, 0, 0), c.tolist(), ck.tolist(), 0.09, 0, 0)
    close(out[0], r.value[0], attention_slack(r, 128, 2000, 2.0**-8)[0])
    assert (clean[0] - out[0]).abs().max() < 1e-2


@pytest.mark.parametrize("d", [8, 20, 80, 96, 256])
def test_window_attention_other_head_sizes(d):
    g = gen(15)
    q, k, v = randn(g, 90, 4, d, dtype=torch.bfloat16), randn(g, 90, 2, d, dtype=torch.bfloat16), randn(g, 90, 2, d, dtype=torch.bfloat16)
    c = cu([50, 40])
    out = ops.window_attention(q, k, v, c.cuda(), d**-0.5, window=20, sinks=2)
    check_window(out, q, k, v, c, c, d**-0.5, 20, 2, 2)


@pytest.mark.parametrize("variant", [0, 2])
def test_window_attention_views(variant):
    """q, k, v as views of one packed projection, head-major output, a view one element off alignment."""
    g = gen(16)
    c = cu([100, 61])
    packed = randn(g, 161, 12, 128, dtype=torch.bfloat16)
    q, k, v = packed[:, :8], packed[:, 8:10], packed[:, 10:]
    out = torch.zeros(8, 161, 128, device="cuda", dtype=torch.bfloat16).transpose(0, 1)
    ops.window_attention(q, k, v, c.cuda(), 0.1, window=64, out=out, variant=variant)
    check_window(out, q, k, v, c, c, 0.1, 64, 0, variant)
    odd = randn(g, 161 * 12 * 128 + 1, dtype=torch.bfloat16)[1:].view(161, 12, 128)
    out = ops.window_attention(odd[:, :8], odd[:, 8:10], odd[:, 10:], c.cuda(), 0.1, window=64)
    check_window(out, odd[:, :8], odd[:, 8:10], odd[:, 10:], c, c, 0.1, 64, 0, 2)


@pytest.mark.parametrize("variant", [0, 2])
@pytest.mark.parametrize("d", [64, 128])
def test_window_attention_masked_specials(d, variant):
    """Infinities and NaN in keys and values reach the queries that see them, and no others: future keys,
    keys before the window, other sequences, rows behind the last sequence."""
    g = gen(17)
    lens = [150, 90]
    c = cu(lens)
    q, k, v = (randn(g, 243, h, d, dtype=torch.bfloat16) for h in (4, 2, 2))
    for row, val in ((70, math.nan), (71, math.inf), (149, -math.inf), (150, math.nan), (239, math.nan)):
        v[row] = val
    v[241:], k[240:] = math.nan, math.nan
    k[30, 1], k[200] = math.nan, math.inf
    out = ops.window_attention(q, k, v, c.cuda(), d**-0.5, window=40, sinks=2, variant=variant)[:240]
    i = torch.arange(240, device="cuda")
    def sees(j):
        lo, hi = (0, 150) if j < 150 else (150, 240)
        return (i >= j) & (i < hi) & ((i - j < 40) | (j - lo < 2))
    spoiled = torch.zeros(240, 4, dtype=torch.bool, device="cuda")
    for j in (70, 71, 149, 150, 239, 200):
        spoiled |= sees(j)[:, None]
    spoiled[:, 2:] |= sees(30)[:, None]
    assert torch.equal(~torch.isfinite(out).all(-1), spoiled)
    k2, v2 = torch.nan_to_num(k, 0, 0, 0), torch.nan_to_num(v, 0, 0, 0)
    _, r = serving.window_attention(q[:240], k2, v2, c.tolist(), c.tolist(), d**-0.5, 40, 2)
    slack = attention_slack(r, d, 150, 2.0**-8)
    close(out[~spoiled], r.value[~spoiled], slack[~spoiled])


@pytest.mark.parametrize("variant", [0, 2])
def test_window_attention_bad_tables_stay_inside(variant):
    """Offsets past the tensors or running backwards are cut to the tensors' rows."""
    g = gen(18)
    q, k, v = (randn(g, 50, h, 64, dtype=torch.bfloat16) for h in (2, 1, 1))
    for table in ([0, 20, 1000], [-5, 30, 50], [0, 40, 10, 50], [60, 70], [2**31 - 1, 0]):
        out = ops.window_attention(q, k, v, i32(table), 0.125, variant=variant)
        assert out.shape == q.shape
    torch.cuda.synchronize()


def test_window_attention_peaked_scores():
    g = gen(19)
    c = cu([400])
    for dt in (torch.bfloat16, torch.float16):
        q, k, v = (randn(g, 400, h, 128, dtype=dt) for h in (2, 1, 1))
        q *= 20
        k *= torch.linspace(0.1, 3, 400, device="cuda")[:, None, None].to(dt)
        out = ops.window_attention(q, k, v, c.cuda(), 128**-0.5)
        check_window(out, q, k, v, c, c, 128**-0.5, 0, 0, 0)


# ---- together -----------------------------------------------------------------------------------


def serve(g, dt=torch.bfloat16, hq=8, hk=2, d=128, page=32, window=100, sinks=4, lens=(150, 37, 1), steps=3):
    """Two layers' worth of a small serving run: prompts, their cache, decoding steps; returns every
    operator's inputs and outputs."""
    b = len(lens)
    total = sum(lens)
    w = [(1 + randn(g, d) / 8).to(dt) for _ in range(2)]
    qkv = randn(g, total, hq + 2 * hk, d, dtype=dt)
    pos = torch.cat([torch.arange(n) for n in lens]).to(torch.int32).cuda()
    c = cu(lens).cuda()
    width = -(-(max(lens) + steps) // page)
    table = torch.randperm(b * width, device="cuda", generator=g).view(b, width).to(torch.int32)
    seq = torch.cat([torch.full((n,), i) for i, n in enumerate(lens)]).cuda()
    slots = (table[seq, pos.long() // page] * page + pos % page).to(torch.int32)
    cache = ops.kv4_cache(b * width, page, hk, d)
    q, k = ops.qk_norm_rope(qkv[:, :hq], qkv[:, hq : hq + hk], *w, pos)
    v = qkv[:, hq + hk :]
    o = ops.window_attention(q, k, v, c, d**-0.5, window=window, sinks=sinks)
    ops.kv4_store(k, v, slots, cache)
    rec = {"prompt": (q, k, v, c, o), "cache": cache, "table": table, "steps": [], "kv": [(k[a:e], v[a:e]) for a, e in zip(c.tolist(), c.tolist()[1:])]}
    now = i32(list(lens))
    for _ in range(steps):
        one = randn(g, b, hq + 2 * hk, d, dtype=dt)
        q1, k1 = ops.qk_norm_rope(one[:, :hq], one[:, hq : hq + hk], *w, now)
        at = (table[torch.arange(b, device="cuda"), now.long() // page] * page + now % page).to(torch.int32)
        ops.kv4_store(k1, one[:, hq + hk :], at, cache)
        now = now + 1
        o1 = ops.kv4_attention(q1, cache, table, now, d**-0.5, window=window, sinks=sinks)
        rec["kv"] = [(torch.cat([a, k1[i : i + 1]]), torch.cat([e, one[i : i + 1, hq + hk :]])) for i, (a, e) in enumerate(rec["kv"])]
        rec["steps"].append((q1, now.tolist(), o1))
    return rec


def test_a_serving_run():
    """Prompt attention, the cache and the decoding steps agree with the definition over the whole history."""
    rec = serve(gen(20))
    q, k, v, c, o = rec["prompt"]
    check_window(o, q, k, v, c.cpu(), c.cpu(), 128**-0.5, 100, 4, 0)
    for q1, lens, o1 in rec["steps"]:
        for i, n in enumerate(lens):
            kq, vq = serving.kv4_quantise(rec["kv"][i][0]), serving.kv4_quantise(rec["kv"][i][1])
            # One request's tokens in order: a table of single-row pages.
            check_decode(o1[i : i + 1], q1[i : i + 1], kq, vq, 1, torch.arange(n, device="cuda")[None], [n], 128**-0.5, 100, 4)


def test_next_chunk_reads_its_context_from_the_cache():
    """A prompt's second chunk: its context read back with kv4_load, attention over context and chunk."""
    g, d = gen(21), 64
    first, second = 90, 50
    k, v = randn(g, first + second, 2, d, dtype=torch.float16), randn(g, first + second, 2, d, dtype=torch.float16)
    q = randn(g, second, 6, d, dtype=torch.float16)
    cache = ops.kv4_cache(5, 32, 2, d)
    slots = i32([3 * 32 + i if i < 32 else 32 + i - 32 if i < 64 else 4 * 32 + i - 64 for i in range(first)])
    ops.kv4_store(k[:first], v[:first], slots, cache)
    kc, vc = (torch.empty_like(x) for x in (k, v))
    ops.kv4_load(cache, slots, k_out=kc[:first], v_out=vc[:first])
    kc[first:], vc[first:] = k[first:], v[first:]
    out = ops.window_attention(q, kc, vc, cu([second]).cuda(), d**-0.5, window=64, sinks=4, cu_seqlens_k=cu([first + second]).cuda())
    same(kc[:first], stored(k[:first]))
    check_window(out, q, kc, vc, cu([second]), cu([first + second]), d**-0.5, 64, 4, 0)


def test_captured_replayed_and_on_other_streams():
    """One decoding step captured and replayed on new inputs, and the same on a side stream: the same bits."""
    g = gen(22)
    hq, hk, d, page = 8, 2, 128, 32
    cache, _, _ = filled_cache(g, 64, page, hk, d, torch.bfloat16)
    table = torch.arange(64, device="cuda", dtype=torch.int32).view(2, 32)
    w = torch.ones(d, device="cuda", dtype=torch.bfloat16)
    one = randn(g, 2, hq + 2 * hk, d, dtype=torch.bfloat16)
    pos = i32([700, 333])

    def step():
        q, k = ops.qk_norm_rope(one[:, :hq], one[:, hq : hq + hk], w, w, pos)
        at = (table[torch.arange(2, device="cuda"), pos.long() // page] * page + pos % page).to(torch.int32)
        ops.kv4_store(k, one[:, hq + hk :], at, cache)
        a = ops.kv4_attention(q, cache, table, pos + 1, d**-0.5)
        b = ops.kv4_attention(q, cache, table, pos + 1, d**-0.5, window=64, sinks=4)
        c = ops.window_attention(q, k, one[:, hq + hk :], cu_one, d**-0.5)
        kl, vl = ops.kv4_load(cache, every)
        e = ops.window_attention(q, kl, vl, cu_one, d**-0.5, cu_seqlens_k=cu_all)  # split over the keys
        return a, b, c, e

    cu_one, cu_all, every = i32([0, 1, 2]), i32([0, 900, 2048]), torch.arange(2048, device="cuda", dtype=torch.int32)
    assert ops.window_attention_workspace_bytes(2, 2048, 2, hq, hk, d) > 0
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):  # two graphs at once, each with its own workspace
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    for seed in range(3):
        one.copy_(randn(gen(100 + seed), 2, hq + 2 * hk, d))
        pos.copy_(i32([700 + seed, 1000 - seed]))
        start = cache.clone()
        want = [x.clone() for x in step()]
        after = cache.clone()
        for graph, out in graphs:
            cache.copy_(start)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(out, want)) and torch.equal(cache, after)
        cache.copy_(start)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            got = step()
        side.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_two_streams_at_once():
    """Overlapping calls, each with the workspace it allocated, give what they give alone."""
    g = gen(23)
    cache, _, _ = filled_cache(g, 128, 64, 2, 128, torch.bfloat16)
    table = torch.randperm(128, device="cuda", generator=g).to(torch.int32).view(2, 64)
    qs = [randn(g, 2, 8, 128, dtype=torch.bfloat16) for _ in range(2)]
    lens = i32([4000, 3333])
    want = [ops.kv4_attention(q, cache, table, lens, 0.09) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    outs = [[], []]
    for _ in range(8):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(ops.kv4_attention(qs[i], cache, table, lens, 0.09))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in outs[i])


def test_generic_dispatch_and_timed_batches():
    """The operators through sf_run_op and sf_run_batch (contiguous tensors), graph-timed batches included."""
    g = gen(24)
    q, k, v = (randn(g, 40, h, 64, dtype=torch.bfloat16) for h in (4, 2, 2))
    w, pos, c = torch.ones(64, device="cuda", dtype=torch.bfloat16), torch.arange(40, device="cuda", dtype=torch.int32), i32([0, 25, 40])
    stream = torch.cuda.current_stream().cuda_stream
    def run(op, dims, attrs, tensors, variant=0):
        desc = _native.op_desc(op, "bf16", dims=dims, attrs=attrs, variant=variant)
        ptrs = [t.data_ptr() for t in tensors]
        _native.run_op(desc, ptrs, stream)
        assert _native.run_batch(desc, [ptrs], 3, stream) > 0 and _native.run_batch(desc, [ptrs], 3, stream, use_graph=True) > 0
    qo, ko, o = torch.empty_like(q), torch.empty_like(k), torch.empty_like(q)
    run("qk_norm_rope", (40, 4, 2, 64, 64), (1e4, 1e-6), (q, k, w, w, pos, qo, ko))
    want = ops.qk_norm_rope(q, k, w, w, pos)
    assert torch.equal(qo, want[0]) and torch.equal(ko, want[1])
    run("window_attention", (40, 40, 2, 4, 2, 64, 16, 1), (0.125,), (qo, ko, v, c, c, o))
    assert torch.equal(o, ops.window_attention(qo, ko, v, c, 0.125, window=16, sinks=1))
    cache, kb, vb = ops.kv4_cache(3, 16, 2, 64), torch.empty_like(k), torch.empty_like(v)
    run("kv4_store", (40, 2, 64, 3, 16), (), (ko, v, pos, cache))
    run("kv4_load", (40, 2, 64, 3, 16), (), (cache, pos, kb, vb))
    assert torch.equal(kb, ops.kv4_load(cache, pos)[0]) and torch.equal(vb, stored(v))
    table, lens = i32([[0, 1, 2], [2, 0, 1]]), i32([40, 17])
    need = ops.kv4_attention_workspace_bytes(2, 4, 2, 64, 16, 3, variant=1)
    ws, one = torch.empty(need, dtype=torch.uint8, device="cuda"), torch.empty(2, 4, 64, device="cuda", dtype=torch.bfloat16)
    run("kv4_attention", (2, 4, 2, 64, 3, 16, 3, need), (0.125, 20, 1), (qo, cache, table, lens, one, ws), variant=1)
    assert torch.equal(one, ops.kv4_attention(qo[:2].contiguous(), cache, table, lens, 0.125, window=20, sinks=1, variant=1))


# ---- the ends of the range ----------------------------------------------------------------------


@pytest.mark.parametrize("variant", [0, 1, 3])
def test_kv4_attention_with_every_page_hidden(variant):
    """A request whose pages all lie outside the cache sees nothing, like one of length 0; its neighbour is as ever."""
    g = gen(40)
    cache, kq, vq = filled_cache(g, 4, 16, 2, 128, torch.bfloat16)
    q = randn(g, 3, 8, 128, dtype=torch.bfloat16)
    for n in (16, 400):
        table = torch.full((3, 25), -1, dtype=torch.int32, device="cuda")
        table[1] = torch.arange(25, device="cuda") % 4
        table[2] = 4
        out = ops.kv4_attention(q, cache, table, i32([n, n, n]), 0.1, variant=variant)
        assert ops.kernel_status() == (3, 112)
        assert not out[0].any() and not out[2].any()
        check_decode(out[1:2], q[1:2], kq, vq, 16, table[1:2], [n], 0.1, 0, 0)
    none = ops.kv4_cache(0, 16, 2, 128)
    out = ops.kv4_attention(q, none, table, i32([5, 400, 0]), 0.1, variant=variant)
    assert ops.kernel_status() == (3, 112) and not out.any()
    assert not ops.kv4_load(none, i32([-1, 0, 7]))[0].any()
    assert ops.kernel_status()[0] == 3


@pytest.mark.parametrize("variant", [0, 1, 3])
@pytest.mark.parametrize("batch", [70, 1023, 1030])
def test_kv4_attention_many_requests(batch, variant):
    """More requests than a warp scans at a time, and more than the keys are dealt evenly for; lengths 0 among them."""
    g = gen(41)
    h, d, page, width = 1, 64, 16, 40
    cache, kq, vq = filled_cache(g, 300, page, h, d, torch.float16)
    table = torch.randint(300, (batch, width), device="cuda", generator=g).to(torch.int32)
    lens = torch.randint(width * page + 1, (batch,), device="cuda", generator=g) * (torch.rand(batch, device="cuda", generator=g) > 0.3)
    q = randn(g, batch, 3, d, dtype=torch.float16)
    out = ops.kv4_attention(q, cache, table, lens.to(torch.int32), 0.1, variant=variant)
    some = [0, 1, 31, 32, 33, 64, batch // 2, batch - 2, batch - 1]
    check_decode(out[some], q[some], kq, vq, page, table[some], lens[some].tolist(), 0.1, 0, 0)
    assert not out[lens == 0].any()
    # The same request gives close to the same wherever it stands (the split's order of sums differs).
    alone = torch.cat([ops.kv4_attention(q[i : i + 1], cache, table[i : i + 1], lens[i : i + 1].to(torch.int32), 0.1) for i in range(0, batch, 9)])
    # Each is off by at most half a step, 2^-11 of the weights' mass and 14 2^-23 17 n 8 max p (n <= 640, max p < 0.02):
    # under 2^-8 of the largest value.
    assert (alone.float() - out[::9].float()).abs().max() <= 2.0**-7 * out.float().abs().max()


@pytest.mark.parametrize("variant", [0, 2])
@pytest.mark.parametrize("seqs", [33, 100, 1500, 40000])
def test_window_attention_many_sequences(seqs, variant):
    """More sequences than a warp looks at in one step of its search, most of them short or empty."""
    g = gen(42)
    lens = torch.randint(0, 4, (seqs,), device="cuda", generator=g) * (torch.rand(seqs, device="cuda", generator=g) > 0.5)
    lens[seqs // 2], lens[-1] = 70, 0
    more = torch.randint(0, 3, (seqs,), device="cuda", generator=g)
    cu_q = torch.cat([lens.new_zeros(1), lens.cumsum(0)]).to(torch.int32)
    cu_k = torch.cat([lens.new_zeros(1), (lens + more).cumsum(0)]).to(torch.int32)
    q = randn(g, int(cu_q[-1]), 4, 64, dtype=torch.bfloat16)
    k, v = randn(g, int(cu_k[-1]), 2, 64, dtype=torch.bfloat16), randn(g, int(cu_k[-1]), 2, 64, dtype=torch.bfloat16)
    out = ops.window_attention(q, k, v, cu_q, 0.125, window=20, sinks=1, cu_seqlens_k=cu_k, out=torch.full_like(q, math.nan), variant=variant)
    # Rounded outputs and one side's rounded weights: 3 2^-8 of the largest value.
    other = ops.window_attention(q, k, v, cu_q, 0.125, window=20, sinks=1, cu_seqlens_k=cu_k, variant=2 - variant)
    assert torch.isfinite(out).all() and (out.float() - other.float()).abs().max() <= 2.0**-6 * other.float().abs().max()
    # A stretch of sequences against the definition.
    for a in (0, seqs // 2 - 8, seqs - 16):
        cq, ck = cu_q[a : a + 17].cpu(), cu_k[a : a + 17].cpu()
        q0, q1, k0, k1 = int(cq[0]), int(cq[-1]), int(ck[0]), int(ck[-1])
        check_window(out[q0:q1], q[q0:q1], k[k0:k1], v[k0:k1], cq - cq[0], ck - ck[0], 0.125, 20, 1, variant)


def test_offsets_past_32_bits():
    """A cache, rows and strides that reach past 2^32 bytes and 2^31 elements."""
    g = gen(43)
    page, h, d = 64, 2, 128
    pages = 2**32 // (h * (page // 16) * 18 * d) + 9
    cache = ops.kv4_cache(pages, page, h, d)
    k, v = randn(g, 100, h, d, dtype=torch.bfloat16), randn(g, 100, h, d, dtype=torch.bfloat16)
    slots = (pages - 2) * page + torch.arange(100, device="cuda", dtype=torch.int32)
    ops.kv4_store(k, v, slots, cache)
    assert ops.kernel_status() == (0, 0) and not cache[: 2].any() and not cache[pages - 3].any()
    same(ops.kv4_load(cache, slots)[0], stored(k))
    table, q = i32([[pages - 2, pages - 1]]), randn(g, 1, 8, d, dtype=torch.bfloat16)
    out = ops.kv4_attention(q, cache, table, i32([100]), 0.1)
    check_decode(out, q, serving.kv4_quantise(k), serving.kv4_quantise(v), page, i32([[0, 1]]), [100], 0.1, 0, 0)
    del cache
    far = 2**30  # elements from one token to the next
    room = torch.empty(2 * far + 64 * 1024, device="cuda", dtype=torch.bfloat16)
    view = lambda at, heads: room[at:].as_strided((3, heads, d), (far, d, 1))
    fq, fk, fv, fo = view(0, 4), view(4096, 2), view(8192, 2), view(12288, 4)
    fq.copy_(randn(g, 3, 4, d)), fk.copy_(randn(g, 3, 2, d)), fv.copy_(randn(g, 3, 2, d))
    for variant in (0, 1, 2):
        ops.window_attention(fq, fk, fv, i32([0, 3]), 0.1, out=fo, variant=variant)
        check_window(fo, fq.contiguous(), fk.contiguous(), fv.contiguous(), cu([3]), cu([3]), 0.1, 0, 0, variant)
    w, pos = torch.ones(d, device="cuda", dtype=torch.bfloat16), i32([5, 6, 2**31 - 1])
    for variant in (1, 2):
        a, b = ops.qk_norm_rope(fq, fk, w, w, pos, q_out=fo, variant=variant)
        check_norm_rope(fq.contiguous(), fk.contiguous(), w, w, pos, (fo, b))
    small = ops.kv4_cache(1, 16, 2, d)
    ops.kv4_store(fk, fv, i32([0, 5, 9]), small)
    kb, vb = ops.kv4_load(small, i32([0, 5, 9]), k_out=view(20000, 2), v_out=view(24000, 2))
    same(kb, stored(fk.contiguous()))
    same(vb, stored(fv.contiguous()))
