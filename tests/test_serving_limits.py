"""The serving operators on the host at the edges of what a call may hold: sizes, workspaces and plans."""

from __future__ import annotations

import pytest
import torch

from shapeforge_b200 import ops


@pytest.mark.parametrize("far", [1 << 16, (1 << 31) - 1, 1 << 31, (1 << 63) - 16, (1 << 63) - 1])
def test_windows_past_every_key_are_no_window(far):
    """The plan of a window (or of sinks) that leaves nothing out is the one of no window, however large the number."""
    size = ops.kv4_attention_workspace_bytes
    for shape in ((1, 32, 8, 128, 64, 1000), (32, 64, 8, 128, 64, 256), (4, 32, 8, 128, 64, 4), (17, 24, 2, 64, 16, 313)):
        assert size(*shape, window=far) == size(*shape) == size(*shape, window=16, sinks=far)
        assert size(*shape, window=far, variant=1) == size(*shape, variant=1) > 0
    wide = ops.window_attention_workspace_bytes
    for shape in ((1, 32768, 1, 32, 8, 128), (1536, 26136, 3, 28, 4, 128), (4, 70, 1, 8, 2, 64)):
        assert wide(*shape, window=far) == wide(*shape) == wide(*shape, window=far, sinks=far)


def test_window_workspace_stays_small():
    """The states of a split are those of the rows that are split, and only where that is worth it: 100 MB at most."""
    size = ops.window_attention_workspace_bytes
    for chunk, context, hq, hk in ((8192, 57344, 128, 8), (16384, 65536, 64, 8), (16384, 131072, 64, 8), (11264, 16384, 64, 8)):
        assert size(chunk, chunk + context, 1, hq, hk, 128) == 0    # below a twentieth of the time
    assert 0 < size(1536, 26136, 3, 28, 4, 128) < 20e6
    for d in (64, 128):
        for hq, hk in ((8, 8), (32, 8), (28, 4), (64, 8), (128, 8), (64, 1), (96, 96)):
            for chunk in (1, 7, 64, 500, 1000, 1536, 2048, 4096, 11264, 16384, 65536):
                for context in (0, 4096, 65536, 131072, 500000):
                    for seqs in (1, 3, 32):
                        for window in (0, 1024, 30000):
                            assert size(chunk, chunk + context * seqs, seqs, hq, hk, d, window=window, sinks=4) <= 100e6


def test_workspace_sizes_are_those_of_the_tensors_gpu(monkeypatch):
    """GPUs may have different numbers of SMs, which the plans go by."""
    current = [0]

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.before, current[0] = current[0], self.index

        def __exit__(self, *_):
            current[0] = self.before

    monkeypatch.setattr(torch.cuda, "device", Device)
    for need, query in (("_kv4_attention_need", "kv4_attention_workspace_bytes"), ("_window_attention_need", "window_attention_workspace_bytes")):
        monkeypatch.setattr(ops, query, lambda *sizes: 1000 * current[0] + sizes[0])
        getattr(ops, need).cache_clear()
        assert [getattr(ops, need)(dev, 7) for dev in (0, 2, 1, 2)] == [7, 2007, 1007, 2007] and current == [0]
        getattr(ops, need).cache_clear()


def test_the_line_is_one_resident_wave():
    """Its grid, and so its workspace, is what the SMs hold at once: three CTAs each, two where the prefix of the
    requests' costs leaves room for no more (74 KB and 4 bytes a request of 228 KB)."""
    size = ops.kv4_attention_workspace_bytes
    full, less = (size(b, 32, 8, 128, 64, 200) for b in (700, 800))
    assert full % 3 == 0 and less == full // 3 * 2 == size(1024, 32, 8, 128, 64, 200)
    assert size(700, 32, 8, 64, 64, 200) == size(1024, 32, 8, 64, 64, 200)
