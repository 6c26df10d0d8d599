"""Stores of heads that are not finite, into an int8 cache."""
import math

import pytest
import torch

import shady_thinker_amd as sta

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("dt", [torch.float32, torch.float16])
def test_store_int8_infinities(gpu, hd, dt):
    """An infinity reads back as itself, by its sign; a head's other values
    have no proportion to it and read as NaN."""
    x = torch.randn(3, hd, generator=torch.Generator().manual_seed(hd))
    x[0, 3] = math.inf
    x[1, 5], x[1, hd - 1] = math.inf, -math.inf
    x = x.to(dt).to(gpu.device)
    c = sta.KvCache(gpu, 1, 16, 1, hd, torch.int8)
    slots = torch.arange(3, dtype=torch.int32, device=gpu.device)
    sta.qk_norm_rope_store(gpu, c, None, x, x, None, slots)
    ko, vo = (torch.empty(3, 1, hd, device=gpu.device) for _ in range(2))
    sta.kv_read(gpu, c, slots, ko, vo)
    for o in (ko[:, 0], vo[:, 0]):
        assert torch.equal(o[:2].isinf(), x[:2].isinf()) and (o[:2].isnan() | o[:2].isinf()).all()
        assert torch.equal(o[:2].isposinf(), x[:2].isposinf())
        # (half a step of the head's scale, and a little for f32)
        assert ((o[2] - x[2].float()).abs() <= x[2].float().abs().max() / 127 * 0.501).all()
