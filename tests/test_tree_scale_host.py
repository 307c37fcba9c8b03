"""Scales that fp32 does not hold are refused ahead of any launch (on the CPU)."""

from __future__ import annotations

import pytest
import torch

from engine import _native, paged_ops
from test_tree_host import attend_args


@pytest.mark.parametrize("scale", [1e39, 1e300, 3e38, 1e-50])
def test_attention_refuses_scales_beyond_fp32(scale):
    """What passes fp32 becomes inf or 0 on its way to the kernels (in base 2: scale * log2 e); inf * 0 is no score."""
    with pytest.raises(ValueError, match="scale"):
        paged_ops.paged_tree(**{**attend_args(), "scale": scale})


def test_the_c_entry_refuses_them_too():
    lib, p = _native.load(), 256

    def attend(scale):
        return lib.mip_paged_tree(p, 256, 64, p, 256, 64, p, p, 9, p, 4, p, p, p, 1, 1, 0, 3, 4, 2, 64, 16, 4, scale, None, 0,
                                  _native.MIP_F16, None)

    assert attend(1.0) == attend(2.0**126) == attend(1e-45) == _native.MIP_OK  # no sequences: nothing is launched
    for scale in (float("inf"), 3e38, 0.0, -1.0, float("nan")):
        assert attend(scale) == _native.MIP_EINVAL, scale
    assert torch.finfo(torch.float32).max < 3e38 * 1.4427
