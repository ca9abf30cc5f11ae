"""How a model groups its MXFP4 products, on the CPU: no call here reaches a launch."""
from __future__ import annotations

import pytest
import torch

import mx_reference as mx


def _linears(seed=0, **last):
    """Three MXFP4 linears; the last one with ``bias``, ``codes`` or ``scales`` of its own."""
    from rwkv7mi import MXFP4Linear
    from rwkv7mi.model import BlockFloatLinear

    codes, scales = mx.random_weight(32, 64, torch.Generator().manual_seed(seed))
    mods = [MXFP4Linear.from_packed(codes, scales, torch.zeros(32, dtype=torch.float16)) for _ in range(3)]
    for name, t in last.items():
        setattr(mods[2], name, t)
    return [BlockFloatLinear(m) for m in mods]


@pytest.mark.parametrize("last", [dict(bias=torch.zeros(32)), dict(bias=torch.zeros(64, dtype=torch.float16)[::2]),
                                  dict(codes=torch.zeros(32 * 32 + 1, dtype=torch.uint8)[1:].view(32, 32)),
                                  dict(codes=torch.zeros(32, 64, dtype=torch.uint8)[:, :32]),
                                  dict(scales=torch.zeros(65, dtype=torch.uint8)[1:].view(32, 2)),
                                  dict(scales=torch.zeros(32, 4, dtype=torch.uint8)[:, ::2])])
def test_what_a_group_cannot_take_runs_by_itself(last):
    """A bias of another type or with gaps, codes and scales with gaps or off their boundary: the
    single product converts or copies them, so the group is declined and not refused."""
    from rwkv7mi.model import BlockFloatLinear

    xs = [torch.zeros(2, 64, dtype=torch.float16) for _ in range(3)]
    outs = [torch.empty(2, 32, dtype=torch.float16) for _ in range(3)]
    assert BlockFloatLinear.apply_group(_linears(**last), xs, outs) is False
    with pytest.raises(RuntimeError, match="GPU only"):  # (alike linears go on to the launch)
        BlockFloatLinear.apply_group(_linears(), xs, outs)
