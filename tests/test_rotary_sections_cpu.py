"""Sections of the multi-axis rotary are checked on every call, also after equal ones have been seen."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from ats_v2_b200.rope import MultiAxisRotaryEmbedding, apply_multi_axis_rotary, axis_of_pairs


@pytest.mark.parametrize("interleaved", [False, True])
def test_counts_of_another_type_are_refused_after_equal_ones(interleaved):
    q, pos, inv = torch.randn(1, 2, 3, 8), torch.zeros(2, 1, 3, dtype=torch.int64), torch.ones(4)
    want, _ = apply_multi_axis_rotary(q, None, pos, inv, (3, 1), interleaved)
    assert torch.equal(apply_multi_axis_rotary(q, None, pos, inv, [3, 1], interleaved)[0], want)
    for bad in ((3.0, 1), (3, 1.0), (np.float64(3), 1), (np.int64(3), 1), ("3", 1), (None, 4)):
        for _ in range(2):
            with pytest.raises(ValueError, match="sections"):
                axis_of_pairs(bad, interleaved)
            with pytest.raises(ValueError, match="sections"):
                apply_multi_axis_rotary(q, None, pos, inv, bad, interleaved)
            with pytest.raises(ValueError, match="sections"):
                MultiAxisRotaryEmbedding(8, bad, interleaved=interleaved)
    assert axis_of_pairs((3, 1), interleaved) == (bytes([0, 1, 0, 0]) if interleaved else bytes([0, 0, 0, 1]))
