"""GPU parity of st_token_logprobs against float64.

Tolerances: sums of f32 exponentials whose arguments are rounded at 2^-24 of
up to 30 (2e-6 of a small term): 1e-5 relative 2-norm of the log
probabilities and entropies; ids and ranks are compared exactly.
"""
import math

import pytest
import torch

import shady_thinker_amd as sta

pytestmark = pytest.mark.gpu
TOL = 1e-5


def run(gpu, x, tokens, top):
    M = x.shape[0]
    dev = gpu.device
    e = lambda *s, dt=torch.float32: torch.full(s, -99, dtype=dt, device=dev)
    o = dict(logprob=e(M), entropy=e(M), rank=e(M, dt=torch.int32), top_ids=e(M, top, dt=torch.int32), top_logprobs=e(M, top))
    sta.token_logprobs(gpu, x, tokens.to(dev, torch.int32), **o)
    return {k: v.cpu() for k, v in o.items()}


def want(x, tokens, top):
    x = x.double().cpu()
    lp = torch.log_softmax(x, -1)
    t = tokens.long()[:, None]
    xt = x.gather(1, t)
    j = torch.arange(x.shape[1])
    ids = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :top]
    return dict(logprob=lp.gather(1, t)[:, 0], entropy=-torch.where(lp > -math.inf, lp.exp() * lp, 0.0).sum(-1),
                rank=((x > xt) | ((x == xt) & (j < t))).sum(-1), top_ids=ids, top_logprobs=lp.gather(1, ids))


def check(got, ref):
    for k in ("rank", "top_ids"):
        assert torch.equal(got[k].long(), ref[k].long()), k
    for k in ("logprob", "entropy", "top_logprobs"):
        a, b = got[k].double(), ref[k]
        assert torch.equal(a.isinf(), b.isinf()) and not a.isnan().any(), k
        f = b.isfinite()
        if f.any():
            n = torch.linalg.vector_norm(b[f]).clamp(min=1e-30)
            assert torch.linalg.vector_norm(a[f] - b[f]) / n < TOL, k


@pytest.mark.parametrize("dt", [torch.float32, torch.float16])
@pytest.mark.parametrize("M,V,top", [(1, 1, 1), (1, 2, 2), (3, 31, 20), (2, 255, 32), (5, 2047, 20), (2, 2049, 1), (1, 8193, 0), (1, 151936, 20),
                                     (33, 50257, 5), (1, 151935, 32), (600, 9001, 3), (2, 2**20, 32)])
def test_logprobs(gpu, M, V, top, dt):
    g = torch.Generator(device=gpu.device)
    g.manual_seed(M + V)
    x = torch.randn(M, V, device=gpu.device, generator=g) * 3
    x[:, V // 3] += 6
    tokens = torch.randint(0, V, (M,))
    tokens[0] = V // 3
    tokens[M - 1] = V - 1
    x = x.to(dt)
    check(run(gpu, x, tokens, top), want(x, tokens, top))


@pytest.mark.parametrize("dt", [torch.float32, torch.float16])
@pytest.mark.parametrize("first,stride", [(0, 1003), (1, 1001), (3, 1008), (5, 1017)])
def test_logprobs_strides(gpu, dt, first, stride):
    """Rows that start and end anywhere in a 16-byte piece."""
    M, V = 4, 1000
    buf = (torch.randn(M * stride + 8, generator=torch.Generator().manual_seed(first)) * 2).to(gpu.device, dt)
    x = torch.as_strided(buf, (M, V), (stride, 1), first)
    tokens = torch.tensor([0, 999, 500, 3])
    check(run(gpu, x, tokens, 20), want(x, tokens, 20))


@pytest.mark.parametrize("V", [40, 5000, 20000])
def test_logprobs_equal_values(gpu, V):
    """Rows of one value, of two, of few: ties go to the lowest index."""
    x = torch.zeros(4, V)
    x[1, ::2] = 1.0
    x[2] = (torch.arange(V) * 7919 % 5).float()
    x[3, ::3] = -0.0  # equals 0
    tokens = torch.tensor([V - 1, 1, 7, 4])
    check(run(gpu, x.to(gpu.device), tokens, 32), want(x, tokens, 32))


def test_logprobs_masked_tokens(gpu):
    """-inf logits: probability 0; whole chunks of them; all but one."""
    V = 30000
    g = torch.Generator().manual_seed(3)
    x = torch.randn(3, V, generator=g)
    x[0, ::2] = -math.inf
    x[1, :20000] = -math.inf
    x[2] = -math.inf
    x[2, 12345] = -3.5
    tokens = torch.tensor([0, 25000, 12345])
    got, ref = run(gpu, x.to(gpu.device), tokens, 5), want(x, tokens, 5)
    check(got, ref)
    assert got["logprob"][0] == -math.inf and got["logprob"][2] == 0 and got["entropy"][2] == 0


def test_logprobs_no_distribution(gpu):
    """A NaN, a +inf, nothing but -inf: NaN; the rows beside them are right."""
    for V in (50, 9000):
        x = torch.randn(5, V, generator=torch.Generator().manual_seed(V))
        x[1, V // 2] = math.nan
        x[2, 3] = math.inf
        x[3] = -math.inf
        tokens = torch.tensor([1, 2, 3, 4, 5])
        got = run(gpu, x.to(gpu.device), tokens, 4)
        for r in (1, 2, 3):
            for k in ("logprob", "entropy", "top_logprobs"):
                assert got[k][r].isnan().all(), (k, r)
        assert got["top_ids"][1, 0] == V // 2 and got["top_ids"][2, 0] == 3
        assert got["top_ids"][3].tolist() == [0, 1, 2, 3]
        ok = [0, 4]
        check({k: v[ok] for k, v in got.items()}, want(x[ok], tokens[ok], 4))


def test_logprobs_likely_token(gpu):
    """-log p of a token with nearly all of the probability, to f32's relative precision."""
    V = 10000
    x = torch.zeros(3, V)
    x[:, 77] = torch.tensor([25.0, 40.0, 60.0])
    tokens = torch.full((3,), 77)
    got = run(gpu, x.to(gpu.device), tokens, 1)
    d = torch.tensor([25.0, 40.0, 60.0], dtype=torch.float64)
    ref = -torch.log1p((V - 1) * torch.exp(-d))
    assert (((got["logprob"].double() - ref) / ref).abs() < 1e-5).all()
    assert torch.equal(got["top_logprobs"][:, 0], got["logprob"])


def test_logprobs_tokens_outside(gpu):
    x = torch.randn(3, 5000, device=gpu.device)
    got = run(gpu, x, torch.tensor([-1, 5000, 2**31 - 1]), 2)
    assert got["logprob"].isnan().all() and (got["rank"] == -1).all()
    assert got["entropy"].isfinite().all() and got["top_logprobs"].isfinite().all()


def test_logprobs_many_rows(gpu):
    """More rows of several chunks than there are counters; parts left out."""
    M, V = 5000, 2100
    x = torch.randn(M, V, device=gpu.device, generator=torch.Generator(device=gpu.device).manual_seed(1))
    tokens = torch.arange(M) % V
    check(run(gpu, x, tokens, 2), want(x, tokens, 2))
    lp = torch.empty(M, device=gpu.device)
    sta.token_logprobs(gpu, x, tokens.to(gpu.device, torch.int32), logprob=lp)
    ent = torch.empty(M, device=gpu.device)
    sta.token_logprobs(gpu, x, entropy=ent)
    ref = want(x, tokens, 2)
    assert torch.linalg.vector_norm(lp.cpu() - ref["logprob"]) / torch.linalg.vector_norm(ref["logprob"]) < TOL
    assert torch.linalg.vector_norm(ent.cpu() - ref["entropy"]) / torch.linalg.vector_norm(ref["entropy"]) < TOL


def test_logprobs_graph_replays(gpu):
    M, V = 3, 40000
    dev = gpu.device
    x = torch.zeros(M, V, device=dev)
    tokens = torch.tensor([5, 600, 39999], dtype=torch.int32, device=dev)
    o = dict(logprob=torch.empty(M, device=dev), entropy=torch.empty(M, device=dev), top_ids=torch.empty(M, 4, dtype=torch.int32, device=dev))
    s = torch.cuda.Stream(device=dev)
    s.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(s):
        sta.token_logprobs(gpu, x, tokens, **o)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            sta.token_logprobs(gpu, x, tokens, **o)
    torch.cuda.current_stream(dev).wait_stream(s)
    for i in range(4):
        x.copy_(torch.randn(M, V, generator=torch.Generator().manual_seed(i)))
        graph.replay()
        torch.cuda.synchronize()
        got = {k: v.clone() for k, v in o.items()}
        sta.token_logprobs(gpu, x, tokens, **o)
        torch.cuda.synchronize()
        assert all(torch.equal(got[k], o[k]) for k in o)
        ref = want(x, tokens.cpu(), 4)
        assert torch.equal(got["top_ids"].cpu().long(), ref["top_ids"])
