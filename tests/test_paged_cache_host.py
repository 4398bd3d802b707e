"""PagedKVCache's own bookkeeping on the CPU: the device operators are replaced by their 64-bit restatements (oracle/decoding_oracle.py)."""
import numpy as np
import pytest
import torch

from multimodal_amd import ops
from multimodal_amd.modules.layers.paged_cache import PagedKVCache
from oracle import decoding_oracle as od


@pytest.fixture
def on_cpu(monkeypatch):
    """ops.paged_* on host tensors."""

    def fork(pages, table, lengths, refcounts, parents, reserve=0):
        after, t, n, c, short = od.paged_fork(pages.float().numpy(), table.numpy(), lengths.numpy(), refcounts.numpy(), parents.numpy(),
                                              reserve if isinstance(reserve, int) else reserve.numpy())
        pages.copy_(torch.from_numpy(after))
        return ops.PagedState(*(torch.from_numpy(np.ascontiguousarray(x)) for x in (t, n, c)), torch.tensor([short], dtype=torch.int32))

    def append(k, v, key_pages, value_pages, table, start, counts=None):
        kp, vp = od.paged_append(k.float().numpy(), v.float().numpy(), key_pages.float().numpy(), value_pages.float().numpy(), table.numpy(), start.numpy(),
                                 None if counts is None else counts.numpy())
        key_pages.copy_(torch.from_numpy(kp))
        value_pages.copy_(torch.from_numpy(vp))

    def attention(q, key_pages, value_pages, table, lengths, k=None, v=None, scale=None, out=None):
        o, kp, vp, _ = od.paged_attention(*(x.float().numpy() for x in (q, key_pages, value_pages)), table.numpy(), lengths.numpy(),
                                          *(None if x is None else x.float().numpy() for x in (k, v)), scale=scale)
        key_pages.copy_(torch.from_numpy(kp))
        value_pages.copy_(torch.from_numpy(vp))
        return torch.from_numpy(o).to(q.dtype)

    def compact(pages, table, refcounts):
        after, t, c, live = od.paged_compact(pages.float().numpy(), table.numpy(), refcounts.numpy())
        pages.copy_(torch.from_numpy(after))
        return ops.CompactedPages(torch.from_numpy(t), torch.from_numpy(c), torch.tensor([live], dtype=torch.int32))

    for name, f in (("paged_fork", fork), ("paged_append", append), ("paged_attention", attention), ("paged_compact", compact)):
        monkeypatch.setattr(ops, name, f)


def cache(pages, max_tokens, page_size=16, dim=64):
    return PagedKVCache(1, 1, dim, pages, max_tokens, page_size, dtype=torch.float32, device="cpu")


def test_the_oracle_says_that_two_spare_pages_a_row_do_not_suffice_for_larger_reserves(on_cpu):
    """Pages that were reserved and hold no token are taken anew at every fork, while the old ones still count."""
    c = cache(8 * (16 + 2), 256)
    c.fork(torch.full((8,), -1, dtype=torch.int32), reserve=256)
    assert int(c.shortage) == 0
    c.fork(torch.arange(8, dtype=torch.int32), reserve=256)
    assert int(c.shortage) == 8 * 16 - 16


@pytest.mark.parametrize("page,tokens,reserve,rows", [(16, 256, 1, 8), (16, 256, 16, 4), (16, 256, 64, 8), (16, 256, 128, 8), (16, 256, 256, 8), (4, 30, 7, 5), (1, 9, 3, 3), (64, 40, 100, 2)])
def test_pages_for_is_enough(on_cpu, page, tokens, reserve, rows):
    """Beams reordered at every token, with `reserve` tokens asked for at every fork, and prompts in the place of full rows: nothing is ever short."""
    g = torch.Generator().manual_seed(rows)
    c = cache(PagedKVCache.pages_for(rows, tokens, page, reserve), tokens, page)
    assert PagedKVCache.pages_for(rows, tokens, page) <= c.pages.shape[0] <= 2 * rows * -(-tokens // page)
    c.fork(torch.full((rows,), -1, dtype=torch.int32), reserve=reserve)
    for t in range(tokens):
        assert int(c.shortage) == 0, t
        assert (c.page_table[torch.arange(rows), c.lengths // page] >= 0).all()
        c.advance(1)
        c.fork(torch.randint(0, rows, (rows,), generator=g, dtype=torch.int32) if t % 3 else torch.arange(rows, dtype=torch.int32), reserve=reserve)
    assert int(c.shortage) == 0
    full = cache(PagedKVCache.pages_for(rows, tokens, page, tokens), tokens, page)
    for _ in range(3):
        full.add_rows(rows, tokens)
        assert int(full.shortage) == 0


def test_pages_for_refuses_nonsense():
    for bad in ((0, 4, 4, 1), (2, 0, 4, 1), (2, 4, 0, 1), (2, 4, 4, -1)):
        with pytest.raises(ValueError):
            PagedKVCache.pages_for(*bad)


def test_losses_stay_on_record(on_cpu):
    """A page that could not be had is not forgotten by the next fork, which has nothing to report."""
    c = cache(5, 32, 4)
    c.fork(torch.tensor([-1, -1], dtype=torch.int32), reserve=9)
    assert int(c.shortage) == 1 and int(c.lost) == 1
    c.advance(9)
    c.fork(torch.tensor([0], dtype=torch.int32), reserve=0)
    assert int(c.shortage) == 0 and int(c.lost) == 1
    c.fork(torch.tensor([0, 0, 0, 0], dtype=torch.int32), reserve=1)  # three copies of the partial page for two free ones
    assert int(c.shortage) == 1 and int(c.lost) == 2
    c.reserve(1)
    assert int(c.shortage) == 0 and int(c.lost) == 2
    assert c.shared_rows(torch.tensor([0])).lost is c.lost
    c.reset()
    assert int(c.lost) == 0
