"""DecoderStack.capture with hooks that keep a state: recording a step is not
a step (examples/decode.py's model)."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "examples"))

pytestmark = pytest.mark.gpu


class Outer:
    """A program that advances by itself, before the step."""

    def __init__(self, hooks):
        self.hooks = hooks
        self.pre, self.attention, self.post_attention, self.final = hooks.pre_attention, hooks.attention, hooks.post_attention, hooks.final
        self.warm_up = hooks.warm_up

    def pre_attention(self, i, b):
        advance, self.hooks.advance = self.hooks.advance, lambda: None
        self.pre(i, b)
        self.hooks.advance = advance


@pytest.mark.parametrize("outside", [False, True])
@pytest.mark.parametrize("cache", [torch.float16, torch.int8])
def test_capture_after_some_tokens(gpu, cache, outside):
    """Some tokens eagerly, then a capture, then replays: lengths and caches
    stay through the capture, and the replays are the eager steps. At the
    capture the first sequence is at the end of its page and the next one is
    not in its table yet (its 0 there is another sequence's page)."""
    import decode as ex

    stack, embedding = ex.build(gpu)
    B, before, after = 2, 16, 5
    prompts = (torch.arange(B * (before + after), dtype=torch.int32, device=gpu.device).view(B, -1) * 37) % ex.VOCAB

    def make():
        table = torch.tensor([[1, 0], [0, 3]], dtype=torch.int32, device=gpu.device)
        h = ex.Hooks(gpu, embedding, table, cache)
        for c in h.caches:
            for t in (c.k, c.v, c.k_scale, c.v_scale):
                if t is not None:
                    t.zero_()
        return h, stack.buffers(gpu, B)

    def held(h):
        return [t.clone() for c in h.caches for t in (c.k, c.v, c.k_scale, c.v_scale) if t is not None] + [h.kv_len.clone()]

    def eager(h, b, i):
        h.tokens.copy_(prompts[:, i])
        stack.step(gpu, b, h)

    h, b = make()
    other, ob = make()
    for i in range(before):
        eager(h, b, i), eager(other, ob, i)
    kept = held(h)
    hooks = Outer(h) if outside else h
    run = stack.capture(gpu, b, hooks)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(kept, held(h)))
    for x in (h, other):
        x.table[0, 1] = 2
    for i in range(before, before + after):
        h.tokens.copy_(prompts[:, i])
        if outside:
            h.advance()
        run.replay()
        torch.cuda.synchronize()
        eager(other, ob, i)
        assert h.kv_len.tolist() == [i + 1] * B
        assert torch.equal(b.logits, ob.logits)
    run.release()


def test_answers_inside_the_step(gpu):
    """Nothing but replays after the prompt: each finds the next tokens and
    takes them on, with their log probabilities, as the eager loop does."""
    import decode as ex

    stack, embedding = ex.build(gpu)
    prompts = torch.arange(3 * 4, dtype=torch.int32, device=gpu.device).view(3, 4) * 37 % ex.VOCAB
    want_ids, want_lps, _ = ex.decode(gpu, stack, embedding, prompts, 20, graph=False)
    table = torch.arange(6, dtype=torch.int32, device=gpu.device).view(3, 2)
    h = ex.Hooks(gpu, embedding, table, torch.float16)
    b = stack.buffers(gpu, 3)
    run = stack.capture(gpu, b, h)
    for i in range(4):
        h.tokens.copy_(prompts[:, i])
        run.replay()
    ids, lps = [], []
    for i in range(20):
        ids.append(h.top[:, 0].clone()), lps.append(h.logprob[:, 0].clone())
        run.replay()
        torch.cuda.synchronize()
    run.release()
    assert torch.equal(torch.stack(ids, 1), want_ids) and torch.equal(torch.stack(lps, 1), want_lps)
