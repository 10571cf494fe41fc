"""The serving operators on the host: refusals before any launch, workspace sizes, and the 64-bit
definitions against themselves (the cache layout is one to one, the mask's corner cases)."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import serving
from shapeforge_b200 import _native, ops

BF16, F16, F32 = 1, 0, 2


def refused(name, fields):
    with pytest.raises(_native.SfError) as exc:
        _native.call_args(name, 0, *fields)
    assert exc.value.code == _native.SF_EINVAL
    return exc.value.message


def norm_args(t=4, hq=2, hk=1, d=64, strides=(128, 64, 64, 64) * 2, rotary=64, base=1e4, eps=1e-6, dtype=BF16, variant=0, ptr=16):
    return (ptr,) * 7 + (t, hq, hk, d, rotary, *strides, base, eps, dtype, variant)


@pytest.mark.parametrize("bad, word", [
    (dict(t=-1), "T"), (dict(d=0), "D"), (dict(rotary=63), "rotary"), (dict(rotary=66), "rotary"), (dict(rotary=-2), "rotary"),
    (dict(base=0.0), "base"), (dict(base=-2.0), "base"), (dict(base=math.nan), "base"), (dict(base=math.inf), "base"),
    (dict(eps=-1.0), "eps"), (dict(eps=math.nan), "eps"), (dict(dtype=F32), "dtype"), (dict(ptr=0), "null"),
    (dict(strides=(128, -1, 64, 64) * 2), "stride"), (dict(ptr=2, variant=1), "vectorised"), (dict(rotary=24, variant=1), "vectorised"),
    (dict(strides=(129, 64, 64, 64) * 2, variant=1), "vectorised"),
])
def test_qk_norm_rope_refusals(bad, word):
    assert word in refused("sf_qk_norm_rope", norm_args(**bad))


def cache_args(t=4, h=2, d=64, pages=3, page=32, strides=(128, 64, 128, 64), dtype=BF16, ptr=16, slots=16):
    return (ptr, ptr, slots, ptr, t, h, d, pages, page, *strides, dtype, 0)


@pytest.mark.parametrize("bad, word", [
    (dict(t=-1), "negative"), (dict(d=96), "64 or 128"), (dict(page=24), "multiple of 16"), (dict(page=0), "multiple of 16"),
    (dict(pages=1 << 30), "2^31"), (dict(dtype=F32), "dtype"), (dict(ptr=0), "null"), (dict(slots=0), "null"), (dict(ptr=8), "aligned"),
    (dict(h=70000), "heads"), (dict(strides=(128, 64, 100, 64)), "multiples of 8"), (dict(strides=(128, -64, 128, 64)), "multiples of 8"),
])
@pytest.mark.parametrize("name", ["sf_kv4_store", "sf_kv4_load"])
def test_kv4_cache_refusals(name, bad, word):
    assert word in refused(name, cache_args(**bad))


def decode_args(b=2, hq=4, hk=2, d=64, pages=3, page=32, width=2, table_stride=2, strides=(256, 64, 256, 64), scale=0.1, window=0, sinks=0,
                dtype=BF16, variant=0, ptr=16, ws=0, ws_bytes=0):
    return (ptr,) * 5 + (ws, ws_bytes, b, hq, hk, d, pages, page, width, table_stride, *strides, window, sinks, scale, dtype, variant)


@pytest.mark.parametrize("bad, word", [
    (dict(b=-1), "negative"), (dict(d=80), "64 or 128"), (dict(page=8), "multiple of 16"), (dict(hq=3), "multiple of the cache"),
    (dict(hk=0), "multiple of the cache"), (dict(scale=0.0), "scale"), (dict(scale=math.nan), "scale"), (dict(scale=math.inf), "scale"),
    (dict(scale=1e-60), "scale"), (dict(window=-1), "window"), (dict(sinks=-1), "sinks"), (dict(dtype=F32), "dtype"), (dict(ptr=0), "null"),
    (dict(ptr=4), "aligned"), (dict(strides=(256, 4, 256, 64)), "multiples of 8"), (dict(table_stride=-2), "stride"),
    (dict(width=1000), "workspace"), (dict(width=1000, ws=16, ws_bytes=8), "workspace"), (dict(width=1000, ws=8, ws_bytes=1 << 40), "workspace"),
    (dict(pages=1 << 29), "2^31"), (dict(width=1 << 29), "2^31"), (dict(b=1 << 25, width=1 << 10), "too large"),
])
def test_kv4_attention_refusals(bad, word):
    assert word in refused("sf_kv4_attention", decode_args(**bad))


def window_args(tq=4, tk=4, seqs=1, hq=4, hk=2, d=64, strides=(256, 64, 128, 64, 128, 64, 256, 64), scale=0.1, window=0, sinks=0, dtype=BF16,
                variant=0, ptr=16):
    return (ptr,) * 6 + (0, 0, tq, tk, seqs, hq, hk, d, *strides, window, sinks, scale, dtype, variant)


@pytest.mark.parametrize("bad, word", [
    (dict(tq=-1), "sizes"), (dict(d=0), "sizes"), (dict(hq=3), "multiple"), (dict(hk=0), "multiple"), (dict(scale=0.0), "scale"),
    (dict(scale=-1.0), "scale"), (dict(scale=math.inf), "scale"), (dict(window=-1), "window"), (dict(sinks=-4), "sinks"),
    (dict(dtype=F32), "dtype"), (dict(ptr=0), "null"), (dict(tq=1 << 31), "2^31"), (dict(d=320), "256"),
    (dict(strides=(256, 64, 128, -64, 128, 64, 256, 64)), "stride"), (dict(d=96, variant=1), "tensor-core"),
    (dict(ptr=8, variant=1), "tensor-core"), (dict(strides=(257, 64, 128, 64, 128, 64, 256, 64), variant=1), "tensor-core"),
    (dict(hq=258, hk=2, variant=1), "tensor-core"),
])
def test_window_attention_refusals(bad, word):
    assert word in refused("sf_window_attention", window_args(**bad))


def test_calls_without_work_are_accepted_without_a_device():
    """Empty inputs return before any CUDA call, null pointers included."""
    _native.call_args("sf_qk_norm_rope", 0, *norm_args(t=0, ptr=0))
    _native.call_args("sf_kv4_store", 0, *cache_args(t=0, ptr=0))
    _native.call_args("sf_kv4_load", 0, *cache_args(t=0, ptr=0))
    _native.call_args("sf_kv4_attention", 0, *decode_args(b=0, ptr=0))
    _native.call_args("sf_window_attention", 0, *window_args(tq=0, ptr=0))
    _native.call_args("sf_window_attention", 0, *window_args(seqs=0, ptr=0))


def test_workspace_sizes():
    size = ops.kv4_attention_workspace_bytes
    assert size(4, 32, 8, 128, 64, 4) == 0            # 256 keys at most: a CTA a (request, head)
    assert size(4, 32, 8, 128, 64, 1000, window=128, sinks=4) == 0
    big = size(4, 32, 8, 128, 64, 1000)
    assert big > 0 and big % 4 == 0
    assert size(1, 32, 8, 128, 64, 1000) <= big       # never more than one resident wave's pieces
    assert size(0, 32, 8, 128, 64, 1000) == 0
    assert size(4, 32, 8, 128, 64, 4, variant=1) > 0 and size(4, 32, 8, 128, 64, 1000, variant=3) == 0


def test_window_workspace_sizes():
    """Split only where CTAs are few and keys are many."""
    size = ops.window_attention_workspace_bytes
    assert size(16384, 16384, 1, 16, 2, 128, window=4096, sinks=4) == 0 and size(1203, 1203, 9, 32, 8, 128, window=128, sinks=4) == 0
    one = size(1, 32768, 1, 32, 8, 128)
    assert one > 0 and one % (32 * 130 * 4) == 0 and 8 <= one // (32 * 130 * 4) <= 32
    assert size(1, 32768, 1, 32, 8, 96) == 0 and size(1, 32768, 1, 129, 1, 64) == 0 and size(0, 9, 1, 8, 8, 64) == 0
    assert size(1, 32768, 1, 32, 8, 128, window=100) == 0


def fake_cuda(t, index=0):
    """A CPU tensor that reports itself on GPU `index`, for the checks that run before a launch."""

    class Fake(torch.Tensor):
        def get_device(self):
            return index

    return torch.Tensor._make_subclass(Fake, t)


def fk(*shape, dtype=torch.bfloat16, index=0):
    return fake_cuda(torch.zeros(*shape, dtype=dtype), index)


def test_python_refusals():
    q, k, w, pos = fk(4, 2, 64), fk(4, 1, 64), fk(64), fk(4, dtype=torch.int32)
    cu = fk(2, dtype=torch.int32)
    cache, slots = fk(3, 1, 2, 18 * 64, dtype=torch.uint8), fk(4, dtype=torch.int32)
    table, lens = fk(4, 2, dtype=torch.int32), fk(4, dtype=torch.int32)
    cases = [
        (TypeError, lambda: ops.qk_norm_rope(q, fk(4, 1, 64, dtype=torch.float16), w, w, pos)),
        (ValueError, lambda: ops.qk_norm_rope(torch.zeros(4, 2, 64), k, w, w, pos)),
        (ValueError, lambda: ops.qk_norm_rope(q, fk(3, 1, 64), w, w, pos)),
        (ValueError, lambda: ops.qk_norm_rope(q, k, fk(32), w, pos)),
        (TypeError, lambda: ops.qk_norm_rope(q, k, w, w, fk(4, dtype=torch.int64))),
        (ValueError, lambda: ops.qk_norm_rope(q, k, w, w, fk(5, dtype=torch.int32))),
        (ValueError, lambda: ops.qk_norm_rope(fake_cuda(torch.zeros(4, 64, 2, dtype=torch.bfloat16).transpose(1, 2)), k, w, w, pos)),
        (ValueError, lambda: ops.qk_norm_rope(q, k, w, w, pos, q_out=fake_cuda(torch.zeros(1, 2, 64, dtype=torch.bfloat16).expand(4, 2, 64)))),
        (ValueError, lambda: ops.qk_norm_rope(q, k, w, w, pos, q_out=fk(4, 1, 64))),
        (ValueError, lambda: ops.qk_norm_rope(fk(4, 128), k, w, w, pos)),
        (ValueError, lambda: ops.kv4_store(k, fk(4, 2, 64), slots, cache)),
        (ValueError, lambda: ops.kv4_store(fk(4, 1, 128), fk(4, 1, 128), slots, cache)),
        (TypeError, lambda: ops.kv4_store(k, k, fk(4, dtype=torch.int64), cache)),
        (ValueError, lambda: ops.kv4_store(k, k, fk(3, dtype=torch.int32), cache)),
        (ValueError, lambda: ops.kv4_store(k, k, slots, fk(3, 1, 2, 18 * 80, dtype=torch.uint8))),
        (TypeError, lambda: ops.kv4_store(k, k, slots, fk(3, 1, 2, 18 * 64, dtype=torch.int8))),
        (ValueError, lambda: ops.kv4_load(cache, slots, k_out=fk(4, 2, 64))),
        (TypeError, lambda: ops.kv4_load(cache, slots, k_out=fk(4, 1, 64), v_out=fk(4, 1, 64, dtype=torch.float16))),
        (ValueError, lambda: ops.kv4_attention(fk(4, 2, 128), cache, table, lens, 0.1)),
        (ValueError, lambda: ops.kv4_attention(fk(4, 3, 64), fk(3, 2, 2, 18 * 64, dtype=torch.uint8), table, lens, 0.1)),
        (ValueError, lambda: ops.kv4_attention(q, cache, fk(3, 2, dtype=torch.int32), lens, 0.1)),
        (TypeError, lambda: ops.kv4_attention(q, cache, fk(4, 2, dtype=torch.int64), lens, 0.1)),
        (ValueError, lambda: ops.kv4_attention(q, cache, table, fk(5, dtype=torch.int32), 0.1)),
        (ValueError, lambda: ops.kv4_attention(q, cache, table, lens, 0.1, out=fk(4, 1, 64))),
        (ValueError, lambda: ops.window_attention(q, k, fk(4, 2, 64), cu, 0.1)),
        (ValueError, lambda: ops.window_attention(fk(4, 3, 64), fk(4, 2, 64), fk(4, 2, 64), cu, 0.1)),
        (ValueError, lambda: ops.window_attention(q, k, k, cu, 0.1, cu_seqlens_k=fk(3, dtype=torch.int32))),
        (ValueError, lambda: ops.window_attention(q, k, k, fk(0, dtype=torch.int32), 0.1)),
        (TypeError, lambda: ops.window_attention(q, k, k, fk(2, dtype=torch.int64), 0.1)),
        (ValueError, lambda: ops.window_attention(q, fk(5, 1, 64), fk(5, 1, 64), cu, 0.1)),
        (ValueError, lambda: ops.kv4_cache(4, 24, 2, 64, device="cpu")),
        (ValueError, lambda: ops.kv4_cache(4, 32, 2, 96, device="cpu")),
    ]
    for i, (kind, call) in enumerate(cases):
        with pytest.raises(kind):
            call()
            pytest.fail(f"call {i} was not refused")


def test_tensors_on_two_gpus_are_refused():
    q, k, w, pos = fk(4, 2, 64), fk(4, 1, 64), fk(64), fk(4, dtype=torch.int32)
    out = fk(4, 2, 64), fk(4, 1, 64)
    cache, slots = fk(3, 1, 2, 18 * 64, dtype=torch.uint8), fk(4, dtype=torch.int32, index=1)
    cu = fk(2, dtype=torch.int32, index=1)
    for call in (lambda: ops.qk_norm_rope(q, k, w, fk(64, index=1), pos, q_out=out[0], k_out=out[1]),
                 lambda: ops.kv4_store(k, k, slots, cache), lambda: ops.kv4_load(cache, slots, k_out=k, v_out=fk(4, 1, 64)),
                 lambda: ops.kv4_attention(q, cache, fk(4, 2, dtype=torch.int32), slots, 0.1, out=out[0]),
                 lambda: ops.window_attention(q, k, k, cu, 0.1, out=out[0])):
        with pytest.raises(ValueError, match="more than one device"):
            call()


def test_output_rows_that_overlap_are_refused():
    base = fake_cuda(torch.zeros(1000, dtype=torch.bfloat16))
    for size, stride in (((4, 2, 64), (64, 64, 1)), ((4, 2, 64), (128, 32, 1)), ((4, 2, 64), (100, 64, 1)), ((2, 4, 64), (64, 96, 1))):
        with pytest.raises(ValueError, match="overlap"):
            ops._check_rows(base.as_strided(size, stride), "out", written=True)
    for size, stride in (((4, 2, 64), (128, 64, 1)), ((4, 2, 64), (64, 256, 1)), ((1, 2, 64), (0, 64, 1)), ((4, 1, 64), (64, 0, 1)), ((3, 2, 64), (160, 72, 1))):
        ops._check_rows(base.as_strided(size, stride), "out", written=True)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("which", [0, 1])
def test_cache_layout_is_one_to_one(dim, which):
    for row in range(16):
        at = serving.kv4_positions(dim, which, row)
        assert sorted(at) == [(b, s) for b in range(dim // 2) for s in (0, 4)]


def test_quantiser_error_bound():
    """|x - value| <= scale / 2 plus what the pair's rounding to bf16 moves the ends by."""
    gen = torch.Generator().manual_seed(0)
    x = (torch.randn(50, 3, 128, generator=gen) * torch.rand(50, 3, 1, generator=gen) * 10 + 3).half()
    codes, scale, low = serving.kv4_quantise(x)
    err = (x.double() - serving.kv4_values(codes, scale, low)).abs().unflatten(-1, (-1, 64)).amax(-1)
    ends = x.double().abs().unflatten(-1, (-1, 64)).amax(-1)
    assert (err <= scale / 2 + 2.0**-9 * (15 * scale + ends) * 1.01).all()


def test_mask_definition():
    m = serving.window_mask(3, 5, 2, 1)
    assert m.tolist() == [[True, True, True, False, False], [True, False, True, True, False], [True, False, False, True, True]]
    assert not serving.window_mask(3, 1, 0, 0)[0].any()      # a query in front of the first key
    assert serving.window_mask(1, 4, 0, 9).all()


def test_unknown_variants_are_refused():
    for name, args, bad in (("sf_qk_norm_rope", norm_args, (-1, 3)), ("sf_kv4_attention", decode_args, (-1, 2, 4)),
                            ("sf_window_attention", window_args, (-1, 3, 5))):
        for variant in bad:
            assert f"no variant {variant}" in refused(name, args(variant=variant))


def test_numbers_that_are_no_sizes_are_refused():
    q, k, cu = fk(4, 2, 64), fk(4, 1, 64), fk(2, dtype=torch.int32)
    cache, table, lens = fk(3, 1, 2, 18 * 64, dtype=torch.uint8), fk(4, 2, dtype=torch.int32), fk(4, dtype=torch.int32)
    for kind, extra in ((TypeError, dict(window=1.5)), (TypeError, dict(sinks=None)), (ValueError, dict(sinks=1 << 70)), (ValueError, dict(window=-1))):
        with pytest.raises(kind):
            ops.kv4_attention(q, cache, table, lens, 0.1, out=fk(4, 2, 64), workspace=fk(16, dtype=torch.uint8), **extra)
        with pytest.raises(kind):
            ops.window_attention(q, k, k, cu, 0.1, out=fk(4, 2, 64), workspace=fk(16, dtype=torch.uint8), **extra)
    with pytest.raises(ValueError, match="sf_qk_norm_rope"):
        _native.call_args("sf_qk_norm_rope", 0, *norm_args(rotary=6.4))


def test_above_1024_requests_a_cta_takes_a_whole_one():
    assert ops.kv4_attention_workspace_bytes(1024, 4, 2, 64, 16, 400) > 0 and ops.kv4_attention_workspace_bytes(1025, 4, 2, 64, 16, 400) == 0


def test_a_few_requests_of_moderate_length_need_no_workspace():
    size = ops.kv4_attention_workspace_bytes
    assert size(1, 32, 8, 128, 64, 65) == 0 and size(4, 32, 8, 128, 64, 32) == 0
    assert size(1, 32, 8, 128, 64, 256) > 0 and size(64, 32, 8, 128, 64, 128) > 0     # long, many
    assert size(1, 32, 8, 128, 64, 65, variant=1) > 0 and size(1, 32, 8, 128, 64, 65, variant=3) == 0
