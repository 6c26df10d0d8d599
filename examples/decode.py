"""A whole decoder step from the framework's parts: GPTQ linears, paged cache,
attention and token log probabilities, captured as one HIP graph and replayed
for each token of a batch (greedy; every token with its log probability).

    python examples/decode.py [--tokens 16] [--batch 4] [--int8]

The weights are random, of a small self-attention model; what a model adds of
its own (norms, residual adds, the embedding) are torch operations in hooks.
"""
import argparse
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
import shady_thinker_amd as sta

HIDDEN, INTER, VOCAB, HEADS, KV_HEADS, DIM, LAYERS = 512, 1024, 4096, 8, 2, 64, 3


def linear(gpu, rng, k, n):
    qw = rng.integers(0, 2**32, (k // 8, n), dtype=np.uint32)
    scales = rng.uniform(0.5, 1.0, (k // 128, n)) * (0.2 / np.sqrt(k))
    return sta.GptqWeight.upload(gpu, qw, scales.astype(np.float16), 128)


def build(gpu, seed=0):
    rng = np.random.default_rng(seed)
    mk = lambda k, n: linear(gpu, rng, k, n)
    q, kv = HEADS * DIM, KV_HEADS * DIM
    layers = [sta.DecoderLinears(mk(HIDDEN, q), mk(HIDDEN, kv), mk(HIDDEN, kv), mk(q, HIDDEN), mk(HIDDEN, INTER), mk(HIDDEN, INTER),
                                 mk(INTER, HIDDEN)) for _ in range(LAYERS)]
    embedding = torch.from_numpy(rng.standard_normal((VOCAB, HIDDEN), dtype=np.float32)).to(gpu.device)
    return sta.DecoderStack(layers, mk(HIDDEN, VOCAB)), embedding


def rotation(gpu, n):
    f = 10000.0 ** (-torch.arange(0, DIM, 2, dtype=torch.float64) / DIM)
    a = torch.arange(n, dtype=torch.float64)[:, None] * f
    return a.cos().float().to(gpu.device), a.sin().float().to(gpu.device)


class Hooks(sta.PagedAttention):
    """The model's own operations around the linears; the attention hook is
    PagedAttention's. `tokens` [B] goes in; the next ones come out in `top`,
    and in `tokens`."""

    def __init__(self, gpu, embedding, table, cache_dtype):
        caches = [sta.KvCache(gpu, table.numel(), 16, KV_HEADS, DIM, cache_dtype) for _ in range(LAYERS)]
        cos, sin = rotation(gpu, table.shape[1] * 16)
        w = torch.ones(DIM, device=gpu.device)
        super().__init__(gpu, caches, HEADS, table, cos, sin, norms=[(w, w)] * LAYERS)
        B = table.shape[0]
        self.embedding = embedding
        self.tokens = torch.zeros(B, dtype=torch.int32, device=gpu.device)
        self.top = torch.zeros(B, 1, dtype=torch.int32, device=gpu.device)
        self.logprob = torch.zeros(B, 1, device=gpu.device)
        self.entropy = torch.zeros(B, device=gpu.device)

    @staticmethod
    def norm(x):
        return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)

    def pre_attention(self, i, b):
        if i == 0:
            self.advance()
            self.residual = self.embedding[self.tokens.long()]
        else:
            self.residual = self.residual + b.down
        b.x.copy_(self.norm(self.residual))

    def post_attention(self, i, b):
        self.residual = self.residual + b.o
        b.xm.copy_(self.norm(self.residual))

    def final(self, b):
        b.x.copy_(self.norm(self.residual + b.down))

    def after_logits(self, b):
        """The likeliest next token of every row, its log probability and the
        row's entropy; the next step's input."""
        sta.token_logprobs(self.gpu, b.logits, entropy=self.entropy, top_ids=self.top, top_logprobs=self.logprob)
        self.tokens.copy_(self.top[:, 0])


def decode(gpu, stack, embedding, prompts, tokens, cache_dtype=torch.float16, graph=True):
    """prompts [B, n] int32: `tokens` more of each, their log probabilities,
    and the last step's logits."""
    B, n = prompts.shape
    pages = -(-(n + tokens) // 16)
    table = torch.randperm(B * pages, generator=torch.Generator().manual_seed(1)).view(B, pages)
    h = Hooks(gpu, embedding, table.to(gpu.device, torch.int32), cache_dtype)
    b = stack.buffers(gpu, B)
    run = stack.capture(gpu, b, h) if graph else None
    ids, lps = [], []
    for i in range(n + tokens - 1):
        if i < n:
            h.tokens.copy_(prompts[:, i])
        run.replay() if graph else stack.step(gpu, b, h)
        if i >= n - 1:
            ids.append(h.top[:, 0].clone()), lps.append(h.logprob[:, 0].clone())
    if graph:
        run.release()
    return torch.stack(ids, 1), torch.stack(lps, 1), b.logits.clone()


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--tokens", type=int, default=16)
    ap.add_argument("--batch", type=int, default=4)
    ap.add_argument("--int8", action="store_true", help="int8 cache")
    a = ap.parse_args()
    gpu = sta.GpuContext(0)
    stack, embedding = build(gpu)
    prompts = torch.arange(a.batch * 5, dtype=torch.int32, device=gpu.device).view(a.batch, 5) * 37 % VOCAB
    ids, lps, _ = decode(gpu, stack, embedding, prompts, a.tokens, torch.int8 if a.int8 else torch.float16)
    for row, lp in zip(ids.tolist(), lps.tolist()):
        print(" ".join(f"{t}({p:.2f})" for t, p in zip(row, lp)))


if __name__ == "__main__":
    main()
