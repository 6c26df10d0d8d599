"""Attention where something is not finite, out of all proportion or past an
end: in the rows that see it, and nowhere else, whatever kernel a call takes
and however it is cut.

Tolerances (relative 2-norm) as in test_gpu_attention.py: f16 output and
weights 1e-3, f32 1e-5.
"""
import math

import pytest
import torch

from attn_util import attention, indices, rel
from test_gpu_attention import F16, F32, I8, Batch, as_prompt

pytestmark = pytest.mark.gpu


def slot_of(b, p, seq=0):
    page = b.cache.page_size
    return (b.table[seq, p // page] * page + p % page).reshape(1)


# ------------------------------------------------- rows with a NaN, in chunks
@pytest.mark.parametrize("hd,cd", [(128, F16), (64, F16), (256, F16), (128, I8)])
@pytest.mark.parametrize("rows,kv", [(100, 4000), (16, 3000), (100, 100)])
def test_nan_query(gpu, hd, cd, rows, kv):
    """A NaN query's row and head are NaN, over a long cache (chunks) as over
    a short one; the others are what they are without it."""
    b = Batch(gpu, [(rows, kv)], 4, 2, hd, 16, cd, F16, wide=1 << 15)
    r, h = rows // 3, 3
    b.q[r, h, 5] = math.nan
    got, want = as_prompt(b), b.want()
    bad = torch.zeros(want.shape, dtype=torch.bool)
    bad[r, h] = True
    assert got[bad].isnan().all()
    assert rel(got[~bad], want[~bad]) < 1e-3


@pytest.mark.parametrize("hd,cd", [(128, F16), (256, F16), (64, I8)])
@pytest.mark.parametrize("window", [0, 40])
def test_nan_key_alone_in_a_chunk(gpu, hd, cd, window):
    """A NaN key (int8: key scale) at a chunk's first place is all that its
    own row sees of the chunk."""
    rows, kv, nkv, nh = 600, 4000, 1, 2
    b = Batch(gpu, [(rows, kv)], nh, nkv, hd, 16, cd, F16, wide=1 << 15)
    p = 3584  # (a multiple of 256 and 512 keys, as the chunks are)
    ki, _, si = indices(slot_of(b, p), nkv, 16, hd)
    t, at = (b.cache.k, ki[0, 0, 7]) if cd is F16 else (b.cache.k_scale, si[0, 0])
    t.view(-1)[at] = math.nan
    got, want = b.run(window=window), b.want(window=window)
    at_row = torch.arange(rows) + kv - rows
    see = (at_row >= p) & ((at_row < p + window) if window else True)
    assert got[see].isnan().all()
    assert got[~see].isfinite().all()
    assert rel(got[~see], want[~see]) < 1e-3
