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
