"""KvCache.slots and PagedAttention's own bookkeeping (CPU)."""
import pytest
import torch

import shady_thinker_amd as sta

I32 = torch.int32
PAGES, PAGE, NKV, HD, NH = 10, 16, 1, 64, 2


class NoGpu:
    handle = None
    device = "cpu"


G = NoGpu()


def outside(slots, cache):
    return (slots < 0) | (slots >= cache.num_pages * cache.page_size)


def test_slots():
    c = sta.KvCache(G, PAGES, PAGE, NKV, HD)
    table = torch.tensor([[7, 2], [5, 9]], dtype=I32)
    assert c.slots(table, torch.tensor([0, 17], dtype=I32)).tolist() == [7 * 16, 9 * 16 + 1]
    got = c.slots(table, torch.tensor([[15, 16, 31], [0, 15, 31]], dtype=I32))
    assert got.dtype is I32 and got.tolist() == [[127, 32, 47], [80, 95, 159]]


@pytest.mark.parametrize("p", [32, 33, 48, 2**31 - 1, -1, -16, -2**31])
def test_slots_past_the_table(p):
    """A position that the table has no page for has no slot, in any row."""
    c = sta.KvCache(G, PAGES, PAGE, NKV, HD)
    table = torch.tensor([[7, 2], [5, 9]], dtype=I32)
    for at in ([p, 3], [3, p], [p, p]):
        got = c.slots(table, torch.tensor(at, dtype=I32))
        for b in range(2):
            want = -1 if at[b] == p else int(table[b, 0]) * 16 + 3
            assert got[b] == want
    assert (c.slots(table, torch.tensor([[p, 3], [3, p]], dtype=I32)) == torch.tensor([[-1, 115], [83, -1]])).all()


@pytest.mark.parametrize("page", [-1, -7, -2**31, PAGES, 2**27, 2**27 + 1, 2**28 + 3, 2**31 - 1])
def test_slots_of_pages_outside(page):
    """Every place of a page outside the cache is outside it (no 32-bit product
    of page and page size comes round to a page that is in it)."""
    c = sta.KvCache(G, PAGES, PAGE, NKV, HD)
    table = torch.tensor([[page, 2]], dtype=I32)
    got = c.slots(table, torch.arange(32, dtype=I32)[None])[0]
    assert outside(got[:16], c).all() and got[16:].tolist() == list(range(32, 48))


def test_advance_stops_at_the_table():
    """A sequence whose table is full keeps its length and gets no slot; the
    others go on."""
    c = sta.KvCache(G, PAGES, PAGE, NKV, HD)
    table = torch.tensor([[7, 2], [5, 9]], dtype=I32)
    p = sta.PagedAttention(G, [c], NH, table)
    p.kv_len.copy_(torch.tensor([31, 3]))
    for n in range(4):
        p.advance()
        assert p.kv_len.tolist() == [32, 4 + n]
        assert p.slots.tolist() == [47 if n == 0 else -1, 83 + n]
        assert p.positions.tolist() == [31 if n == 0 else 32, 3 + n]


@pytest.mark.parametrize("window", [0, 7, 2**31 - 1, 2**31, 2**32, 2**32 + 5, 2**40])
def test_window_of_any_size(monkeypatch, window):
    """A window wider than 32 bits is as good as the widest of them, not what
    its lower 32 bits say."""
    from shady_thinker_amd import attention

    class Gpu(NoGpu):
        def sync_stream(self):
            pass

    got = []
    monkeypatch.setattr(attention, "call", lambda name, *args: got.append(dict(zip(
        ("gpu", "cache", "q", "q_dtype", "table", "pages", "kv_len", "q_start", "scale", "cap", "window"), args))))
    c = sta.KvCache(G, PAGES, PAGE, NKV, HD)
    q = torch.zeros(1, NH * HD)
    sta.paged_attention(Gpu(), c, q, torch.empty_like(q), torch.zeros(1, 2, dtype=I32), torch.ones(1, dtype=I32), window=window)
    assert got[0]["window"] == min(window, 2**31 - 1)
