"""Rotary.scale: 0 is refused (the C argument block's 0 stands for 1, so it would leave the rows unscaled)."""
import pytest
import torch

from leankv_b200 import ops


@pytest.mark.parametrize("zero", [0, 0.0, -0.0])
def test_scale_zero_is_refused(zero):
    positions = torch.zeros(2, 3, dtype=torch.int32)
    rope = ops.Rotary(ops.rotary_frequencies(64, device="cpu"), scale=zero)
    with pytest.raises(ValueError, match="scale"):
        ops._rope_fields(rope, 2, 3, positions, False)
    for scale in (1.0, 0.5, -2.0):
        assert ops._rope_fields(rope._replace(scale=scale), 2, 3, positions, False)[-1] == scale
