"""The operators together in a captured decoder step (examples/decode.py)."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "examples"))

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cache", [torch.float16, torch.int8])
@pytest.mark.parametrize("batch", [1, 3])
def test_captured_decode(gpu, cache, batch):
    """Replayed as the sequences grow over page ends: the tokens and log
    probabilities of the same steps run eagerly, and of torch's log_softmax."""
    import decode as ex

    stack, embedding = ex.build(gpu)
    prompts = torch.arange(batch * 5, dtype=torch.int32, device=gpu.device).view(batch, 5) * 37 % ex.VOCAB
    ids, lps, logits = ex.decode(gpu, stack, embedding, prompts, 40, cache)
    want_ids, want_lps, want_logits = ex.decode(gpu, stack, embedding, prompts, 40, cache, graph=False)
    assert torch.equal(ids, want_ids) and torch.equal(lps, want_lps) and torch.equal(logits, want_logits)
    assert torch.equal(ids[:, -1].long(), logits.argmax(-1))
    want = torch.log_softmax(logits.cpu().double(), -1).gather(1, ids[:, -1:].cpu().long())[:, 0]
    # (f32 sums over 4096 logits of up to about 10 in size: 2^-24 of them)
    assert (lps[:, -1].cpu().double() - want).abs().max() < 1e-5


def test_loads_past_the_caches(gpu):
    """A cache larger than what is kept between calls is read by loads of its
    own; the result is the same as of a call that does not."""
    import shady_thinker_amd as sta

    g = torch.Generator(device=gpu.device).manual_seed(3)
    nkv, hd, page, pages = 8, 128, 64, 768
    for dtype in (torch.float16, torch.int8):
        c = sta.KvCache(gpu, pages, page, nkv, hd, dtype)
        if dtype is torch.int8:
            for t in (c.k, c.v):
                t.copy_(torch.randint(-127, 128, t.shape, device=gpu.device, generator=g))
            c.k_scale.fill_(0.01), c.v_scale.fill_(0.01)
        else:
            for t in (c.k, c.v):
                t.copy_(torch.randn(t.shape, device=gpu.device, generator=g))
        table = torch.arange(pages, dtype=torch.int32, device=gpu.device).view(4, -1)
        q = torch.randn(4, 16 * hd, device=gpu.device, generator=g)
        kv_len = torch.tensor([page * pages // 4 - 5, 1, 700, 40], dtype=torch.int32, device=gpu.device)
        out, want = torch.empty_like(q), torch.empty_like(q)
        sta.paged_attention(gpu, c, q, out, table, kv_len)
        sta.paged_attention(gpu, c, q, want, table, kv_len, torch.arange(5, dtype=torch.int32, device=gpu.device))
        assert torch.equal(out, want)
