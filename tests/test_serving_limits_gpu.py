"""The serving operators on the B200 at the edges of what a call may hold: heads whose queries differ by
orders of magnitude, infinite and zero queries (64-bit definitions: oracle/serving.py; tolerances: see
tests/test_serving_ops_gpu.py, whose helpers are used)."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import serving
from shapeforge_b200 import ops
from tests.test_serving_ops_gpu import (  # noqa: F401
    LAST_ROUND, SPLIT, TD, WINDOW, _status, attention_slack, check_decode, check_window, close, cu, filled_cache, gen, i32, randn)

pytestmark = pytest.mark.gpu


# ---- every query head of kv4_attention stands alone ------------------------------------------------


HEADS = [(8, 2, 64), (16, 2, 128), (12, 1, 128), (40, 1, 64)]  # 4 and 8 heads a block of 8, 12 and 40 in blocks of 16


def decode_case(g, hq, h, d, dt, n=500, page=32):
    width = -(-n // page)
    cache, kq, vq = filled_cache(g, width + 1, page, h, d, dt)
    table = torch.randperm(width + 1, device="cuda", generator=g)[:width].view(1, width).to(torch.int32)
    return cache, kq, vq, table, randn(g, 1, hq, d, dtype=dt)


@pytest.mark.parametrize("variant", [0, 1, 3])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("shape", HEADS, ids=["x".join(map(str, s)) for s in HEADS])
def test_an_infinite_query_spoils_its_own_head_alone(shape, dtype, variant):
    hq, h, d = shape
    cache, kq, vq, table, q = decode_case(gen(60), hq, h, d, TD[dtype])
    want = ops.kv4_attention(q, cache, table, i32([500]), d**-0.5, variant=variant)
    check_decode(want, q, kq, vq, 32, table, [500], d**-0.5, 0, 0)
    for value in (math.inf, -math.inf, math.nan):
        bad = q.clone()
        bad[0, 1, 5] = bad[0, hq - 1, d - 1] = value
        out = ops.kv4_attention(bad, cache, table, i32([500]), d**-0.5, variant=variant)
        assert torch.isnan(out[0, 1]).all() and torch.isnan(out[0, hq - 1]).all()
        out[0, [1, hq - 1]] = want[0, [1, hq - 1]]
        check_decode(out, q, kq, vq, 32, table, [500], d**-0.5, 0, 0)


@pytest.mark.parametrize("dtype, small", [("bf16", 2.0**-30), ("bf16", 2.0**-70), ("fp16", 2.0**-14)])
@pytest.mark.parametrize("shape", HEADS, ids=["x".join(map(str, s)) for s in HEADS])
def test_heads_of_very_different_size_keep_their_precision(shape, dtype, small):
    """Head 0 a multiple of the others (2^30, 2^70, or what fp16 has room for): each within its own bound."""
    hq, h, d = shape
    cache, kq, vq, table, q = decode_case(gen(61), hq, h, d, TD[dtype])
    scale = 1.0 / (math.sqrt(d) * small)
    lone = q * small
    want = ops.kv4_attention(lone, cache, table, i32([500]), scale)
    check_decode(want, lone, kq, vq, 32, table, [500], scale, 0, 0)
    both = lone.clone()
    both[0, 0] = q[0, 0] * 4
    out = ops.kv4_attention(both, cache, table, i32([500]), scale)
    first = out[0, 0].clone()
    out[0, 0] = want[0, 0]
    check_decode(out, lone, kq, vq, 32, table, [500], scale, 0, 0)
    # One key has nearly all of head 0's weight, where it leads by more than a score's error (four times its
    # D products' in fp32) and 2^30 in weight.
    kv, vv = serving.kv4_values(*kq), serving.kv4_values(*vq)
    at = torch.arange(500, device="cuda")
    rows = table[0].long()[at // 32] * 32 + at % 32
    scores = both[0, 0].double() @ kv[rows, 0].T * scale
    error = 4 * (d + 16) * 2.0**-23 * (both[0, 0].double().abs() @ kv[rows, 0].abs().T * scale).max()
    top = scores.topk(2)
    if top.values[0] - top.values[1] > 2 * error + 21:
        best = vv[rows[top.indices[0]], 0]
        # Half a step of the type and of the weight, at most 2^-8 of the value each.
        assert (first.double() - best).abs().max() <= 2.0**-7 * best.abs().max()


@pytest.mark.parametrize("shape", HEADS, ids=["x".join(map(str, s)) for s in HEADS])
def test_zero_tiny_and_huge_queries(shape):
    """Queries of zero (a padded request) weigh all keys alike; bf16 queries at both ends of the type's range, with a
    scale that brings the scores back (or keys that do), are as precise as any."""
    hq, h, d = shape
    g = gen(62)
    cache, kq, vq, table, q = decode_case(g, hq, h, d, torch.bfloat16)
    zero = torch.zeros_like(q)
    out = ops.kv4_attention(zero, cache, table, i32([500]), 0.1)
    assert torch.isfinite(out).all()
    check_decode(out, zero, kq, vq, 32, table, [500], 0.1, 0, 0)
    for power in (-110, -60, 60, 110, 120):
        x = (q.float() * 2.0**power).bfloat16()
        out = ops.kv4_attention(x, cache, table, i32([500]), d**-0.5 * 2.0**-power)
        check_decode(out, x, kq, vq, 32, table, [500], d**-0.5 * 2.0**-power, 0, 0)
    # Small keys against large queries at an ordinary scale.
    small = ops.kv4_cache(cache.shape[0], 32, h, d)
    n = cache.shape[0] * 32
    k, v = (randn(g, n, h, d) * 2.0**-119).bfloat16(), randn(g, n, h, d, dtype=torch.bfloat16)
    ops.kv4_store(k, v, torch.arange(n, device="cuda", dtype=torch.int32), small)
    x = (q.float() * 2.0**119).bfloat16()
    out = ops.kv4_attention(x, small, table, i32([500]), d**-0.5)
    check_decode(out, x, serving.kv4_quantise(k), serving.kv4_quantise(v), 32, table, [500], d**-0.5, 0, 0)


# ---- windows that leave nothing out ----------------------------------------------------------------


@pytest.mark.parametrize("variant", [0, 2])
@pytest.mark.parametrize("window", [200, 2**31 - 2, 2**31 - 1, 2**31, 2**63 - 1])
@pytest.mark.parametrize("sinks", [0, 4, 2**31 - 1, 2**63 - 1])
def test_windows_past_every_key_are_no_window(window, sinks, variant):
    """A window that says "unlimited", with queries in front of the first key: the same bits as no window."""
    g = gen(63)
    lq, lk = [70, 40, 5], [40, 49, 0]
    cu_q, cu_k = cu(lq), cu(lk)
    q, k, v = randn(g, 115, 4, 64, dtype=torch.bfloat16), randn(g, 89, 2, 64, dtype=torch.bfloat16), randn(g, 89, 2, 64, dtype=torch.bfloat16)
    run = lambda **kw: ops.window_attention(q, k, v, cu_q.cuda(), 0.125, cu_seqlens_k=cu_k.cuda(), variant=variant, **kw)
    out = run(window=window, sinks=sinks)
    check_window(out, q, k, v, cu_q, cu_k, 0.125, 0, 0, variant)
    assert not out[:30].any() and not out[110:].any() and torch.equal(out, run())


@pytest.mark.parametrize("window", [2**31 - 1, 2**63 - 1])
def test_decoding_with_a_window_past_every_key(window):
    cache, kq, vq, table, q = decode_case(gen(64), 8, 2, 64, torch.bfloat16)
    for sinks in (0, 2**63 - 1):
        for variant in (0, 1, 3):
            out = ops.kv4_attention(q, cache, table, i32([500]), 0.125, window=window, sinks=sinks, variant=variant)
            check_decode(out, q, kq, vq, 32, table, [500], 0.125, 0, 0)


# ---- the weights' precision ------------------------------------------------------------------------


def check_precise(out, q, k, v, cu_q, cu_k, scale, window, sinks):
    """As check_window, with the weights held in two 16-bit parts: a bf16 high part leaves less than 2^-7 of the weight,
    whose own half step is 2^-8 of that; fp16 2^-11 and 2^-11, and 2^-25 of 2^-7 of the largest at the least."""
    inside, r = serving.window_attention(q, k, v, cu_q.tolist(), cu_k.tolist(), scale, window, sinks)
    half = q.dtype == torch.float16
    n = int((cu_k[1:] - cu_k[:-1]).max())
    slack = attention_slack(r, q.shape[2], n, 2.0**-22 if half else 2.0**-15) + (n * 2.0**-32 * r.peak if half else 0)
    close(out[inside], r.value[inside], slack[inside])


PRECISE = WINDOW + SPLIT + LAST_ROUND


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("case", PRECISE, ids=[f"{'_'.join(map(str, c[0]))}+{'_'.join(map(str, c[1]))}-{'x'.join(map(str, c[2:]))}" for c in PRECISE])
def test_window_attention_keeps_the_weights_precision(case, dtype):
    """The result is the definition's to its own rounding, in one piece and split over the keys."""
    lq, ctx, hq, hk, d, window, sinks = case
    g, dt = gen(65), TD[dtype]
    lk = [max(0, a + b) for a, b in zip(lq, ctx)]
    cu_q, cu_k = cu(lq), cu(lk)
    q, k, v = randn(g, sum(lq), hq, d, dtype=dt), randn(g, sum(lk), hk, d, dtype=dt), randn(g, sum(lk), hk, d, dtype=dt)
    for variant in (0, 4):
        out = ops.window_attention(q, k, v, cu_q.cuda(), d**-0.5, window=window, sinks=sinks, cu_seqlens_k=cu_k.cuda(), variant=variant)
        check_precise(out, q, k, v, cu_q, cu_k, d**-0.5, window, sinks)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_window_attention_keeps_small_weights_precision(dtype):
    """Many keys of little weight each (2^-14 of the largest and less), all on one side: their sum keeps its bits."""
    g, dt = gen(66), TD[dtype]
    n, d = 3000, 64
    q, k = torch.zeros(4, 2, d, device="cuda", dtype=dt), torch.zeros(n, 1, d, device="cuda", dtype=dt)
    q[:, :, 0], k[:, 0, 0] = 1, -10 - torch.rand(n, device="cuda", generator=g) * 4
    k[7, 0, 0] = 0
    v = (1 + randn(g, n, 1, d).abs()).to(dt)
    v[7] = 0
    out = ops.window_attention(q, k, v, cu([4]).cuda(), 1.0, cu_seqlens_k=cu([n]).cuda())
    check_precise(out, q, k, v, cu([4]), cu([n]), 1.0, 0, 0)


@pytest.mark.parametrize("variant", [0, 1, 3])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("shape", [(8, 2, 64), (32, 4, 128), (24, 2, 64), (40, 2, 128)], ids=["8x2x64", "32x4x128", "24x2x64", "40x2x128"])
def test_kv4_attention_keeps_the_weights_precision(shape, dtype, variant):
    """The error's mean square is that of the output's own rounding.  What else there is, is some 2^-18 of a result (sums
    in fp32 of whole bytes, 17 times a code, in steps of 2^-24) and the weights' rounding: 2^-22 (fp16) or 2^-11 of a
    bf16 step of 2^-8, at most 1/64 of its square.  Weights of 11 bits would double it in fp16."""
    hq, h, d = shape
    g, dt, n, page, b = gen(67), TD[dtype], 900, 32, 3
    cache = ops.kv4_cache(30 * b, page, h, d)
    # Values about zero, so that results are as small as the weights' errors can make them.
    kx, vx = randn(g, 30 * b * page, h, d, dtype=dt), randn(g, 30 * b * page, h, d, dtype=dt)
    ops.kv4_store(kx, vx, torch.arange(30 * b * page, device="cuda", dtype=torch.int32), cache)
    table = torch.randperm(30 * b, device="cuda", generator=g).view(b, 30).to(torch.int32)
    q = randn(g, b, hq, d, dtype=dt)
    out = ops.kv4_attention(q, cache, table, i32([n] * b), d**-0.5, variant=variant)
    kv, vv = serving.kv4_values(*serving.kv4_quantise(kx)), serving.kv4_values(*serving.kv4_quantise(vx))
    at = torch.arange(n, device="cuda")
    rows = table.long()[:, at // page] * page + at % page
    k, v = (x[rows].transpose(1, 2).repeat_interleave(hq // h, 1) for x in (kv, vv))
    want = (torch.softmax(torch.einsum("bhd,bhnd->bhn", q.double(), k) * d**-0.5, -1)[:, :, None] @ v)[:, :, 0]
    own, error = ((x.double() - want).square().mean() for x in (want.to(dt), out))
    assert error <= 1.1 * own


# ---- the workspace of a split ----------------------------------------------------------------------


def test_a_chunk_split_in_its_last_round_writes_what_it_asked_for():
    """1200 tokens behind 3000 and a short neighbour, 32 heads on 8: the workspace holds the last round's rows alone, all
    of them, and nothing behind it is touched."""
    g, hq, hk, d = gen(68), 32, 8, 128
    cu_q, cu_k = cu([1200, 37]), cu([4200, 3037])
    q, k, v = randn(g, 1240, hq, d, dtype=torch.bfloat16), randn(g, 7237, hk, d, dtype=torch.bfloat16), randn(g, 7237, hk, d, dtype=torch.bfloat16)
    need = ops.window_attention_workspace_bytes(1240, 7237, 2, hq, hk, d)
    assert 0 < need < 1240 * hq * (d + 2) * 4
    ws = torch.full((need + 4096,), 0xFF, dtype=torch.uint8, device="cuda")
    before = torch.full_like(q, 7.5)
    out = ops.window_attention(q, k, v, cu_q.cuda(), 0.09, cu_seqlens_k=cu_k.cuda(), workspace=ws[:need], out=before.clone())
    assert (ws[need:] == 0xFF).all() and torch.equal(out[1237:], before[1237:])
    check_precise(out[:1237], q[:1237], k, v, cu_q, cu_k, 0.09, 0, 0)
    for small in (ws[: need - 16], ws[:0]):
        whole = ops.window_attention(q, k, v, cu_q.cuda(), 0.09, cu_seqlens_k=cu_k.cuda(), workspace=small, out=before.clone())
        check_precise(whole[:1237], q[:1237], k, v, cu_q, cu_k, 0.09, 0, 0)


# ---- values that are not finite --------------------------------------------------------------------


SPECIAL = [
    # query lengths, contexts in front, Hq, Hk, D, window, sinks
    ([300, 40], [0, 33], 4, 2, 128, 0, 0),
    ([300, 150], [20, 0], 8, 1, 64, 90, 0),
    ([260], [100], 5, 1, 128, 70, 6),
    ([400], [0], 2, 2, 64, 40, 150),
    ([3], [2000], 4, 2, 128, 0, 0),             # split over the keys
    ([9, 2], [3333, 2500], 3, 1, 64, 1500, 4),
    ([650, 3], [1300, 1400], 64, 1, 64, 0, 0),  # in the last round
]


@pytest.mark.parametrize("variant", [0, 2, 4])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("case", SPECIAL, ids=[f"{'_'.join(map(str, c[0]))}-{'x'.join(map(str, c[2:]))}" for c in SPECIAL])
def test_infinite_values_come_out_as_the_definition_has_them(case, dtype, variant):
    """An element of the result whose column holds infinities among the values seen is that infinity (NaN with both signs
    or a NaN); every other element is as ever, in the same row and beside values that the row does not see."""
    lq, ctx, hq, hk, d, window, sinks = case
    g, dt = gen(69), TD[dtype]
    lk = [a + b for a, b in zip(lq, ctx)]
    cu_q, cu_k = cu(lq), cu(lk)
    q, k, v = randn(g, sum(lq), hq, d, dtype=dt), randn(g, sum(lk), hk, d, dtype=dt), randn(g, sum(lk) + 1, hk, d, dtype=dt)
    n = lk[0]
    for row, col, value in ((0, 3, math.inf), (n // 2, 3, math.inf), (n // 3, 5, -math.inf), (n - 1, 5, math.inf), (n - 2, 7, math.nan), (n // 2 + 1, 8, -math.inf),
                            (n - 3, d - 1, math.inf), (n // 4, slice(40, 44), math.inf), (n, 9, math.nan)):
        v[row, 0, col] = value
    v[n // 5, hk - 1, 1] = math.nan
    out = ops.window_attention(q, k, v[: sum(lk)], cu_q.cuda(), d**-0.5, window=window, sinks=sinks, cu_seqlens_k=cu_k.cuda(), variant=variant)
    inside, r = serving.window_attention(q, k, v[: sum(lk)], cu_q.tolist(), cu_k.tolist(), d**-0.5, window, sinks)
    assert torch.isinf(r.value).any() and torch.isnan(r.value).any()
    half = dt == torch.float16
    close(out, r.value, attention_slack(r, d, max(lk), 2.0**-22 if half else 2.0**-15) + (max(lk) * 2.0**-32 * r.peak if half else 0))


def test_one_bad_token_does_not_slow_the_whole_prompt_down():
    """A NaN key and value, or an infinite value alone, that every query sees: what comes out is known without going over
    each row's keys again (hundreds of times the work)."""
    g = gen(70)
    n = 6144
    q, k, v = (randn(g, n, h, 128, dtype=torch.bfloat16) for h in (8, 1, 1))
    table = cu([n]).cuda()

    def time():
        best = math.inf
        for _ in range(3):
            start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            start.record()
            out = ops.window_attention(q, k, v, table, 0.09)
            end.record()
            torch.cuda.synchronize()
            best = min(best, start.elapsed_time(end))
        return out, best

    _, clean = time()
    v[0] = math.inf
    out, infinite = time()
    assert torch.isposinf(out).all()
    k[0], v[0] = math.nan, math.nan
    out, bad = time()
    assert torch.isnan(out).all()
    assert infinite < 20 * clean and bad < 5 * clean, (clean, infinite, bad)


# ---- workspaces of calls that overlap --------------------------------------------------------------


def overlap_calls(g):
    """(call(i, **keywords) of two inputs each, workspace bytes): the line of kv4_attention in one shape that takes it by
    itself and one that is told to, window_attention split in all its row tiles and in the last round's."""
    cache, _, _ = filled_cache(g, 128, 64, 2, 128, torch.bfloat16)
    small = torch.randperm(128, device="cuda", generator=g).to(torch.int32).view(2, 64)
    many = torch.randint(128, (24, 64), device="cuda", generator=g).to(torch.int32)
    q2, q24 = ([randn(g, b, 8, 128, dtype=torch.bfloat16) for _ in range(2)] for b in (2, 24))
    n2, n24 = i32([4000, 3333]), torch.randint(1, 4097, (24,), device="cuda", generator=g).to(torch.int32)
    size = ops.kv4_attention_workspace_bytes
    yield lambda i, **kw: ops.kv4_attention(q2[i], cache, small, n2, 0.09, variant=1, **kw), size(2, 8, 2, 128, 64, 64, variant=1)
    yield lambda i, **kw: ops.kv4_attention(q24[i], cache, many, n24, 0.09, **kw), size(24, 8, 2, 128, 64, 64)
    for lq, n, hq, hk in ((7, 3000, 8, 2), (650, 1950, 64, 1)):
        q = [randn(g, lq, hq, 64, dtype=torch.bfloat16) for _ in range(2)]
        k, v = randn(g, n, hk, 64, dtype=torch.bfloat16), randn(g, n, hk, 64, dtype=torch.bfloat16)
        a, b = cu([lq]).cuda(), cu([n]).cuda()
        yield (lambda i, q=q, k=k, v=v, a=a, b=b, **kw: ops.window_attention(q[i], k, v, a, 0.1, cu_seqlens_k=b, **kw),
               ops.window_attention_workspace_bytes(lq, n, 1, hq, hk, 64))


@pytest.mark.parametrize("which", range(4))
def test_overlapping_calls_have_workspaces_of_their_own(which):
    """Two streams at once, allocating or given a workspace each: what they give alone."""
    call, need = list(overlap_calls(gen(71)))[which]
    assert need > 0
    want = [call(i) for i in range(2)]
    assert not torch.equal(*want)
    spaces = [torch.full((need,), 0xFF, dtype=torch.uint8, device="cuda") for _ in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    for turn in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(call(i, **(dict(workspace=spaces[i]) if turn % 2 else {})))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in outs[i])


@pytest.mark.parametrize("which", range(4))
def test_graphs_have_workspaces_of_their_own(which):
    """Two graphs captured one after the other and replayed at once on two streams, beside eager calls."""
    call, need = list(overlap_calls(gen(72)))[which]
    assert need > 0
    want = [call(i) for i in range(2)]
    torch.cuda.synchronize()
    graphs = []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = [call(i) for _ in range(3)]
        graphs.append((graph, out))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        for graph, out in graphs:
            for o in out:
                o.zero_()
        torch.cuda.synchronize()
        for (graph, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        eager = [call(i) for i in range(2)]
        torch.cuda.synchronize()
        for i, (_, out) in enumerate(graphs):
            assert all(torch.equal(o, want[i]) for o in (*out, eager[i]))


# ---- the quantiser's arithmetic --------------------------------------------------------------------


@pytest.mark.parametrize("sign", [1, -1])
def test_codes_are_those_of_fp32_arithmetic(sign):
    """x - minimum and its quotient are IEEE fp32 operations: an element a little past a tie that fp32 does not tell from
    the tie goes where the tie goes, to the even code."""
    x = torch.zeros(1, 1, 64, device="cuda", dtype=torch.bfloat16)
    x[0, 0, 0], x[0, 0, 1], x[0, 0, 2] = -6.5, 8.5, sign * 2.0**-30   # scale 1; 6.5 +- 2^-30 is 6.5 in fp32
    cache = ops.kv4_cache(1, 16, 1, 64)
    ops.kv4_store(x, x, i32([0]), cache)
    k, v = ops.kv4_load(cache, i32([0]))
    assert torch.equal(k, v) and k[0, 0, :3].tolist() == [-6.5, 8.5, -0.5]
    codes, scale, low = serving.kv4_quantise(x)
    assert codes[0, 0, 0, :3].tolist() == [0, 15, 6] and scale.item() == 1 and low.item() == -6.5
