"""Page tables at the edges of their arguments: no sequence at all, lists and tables that do not fit each other."""
import numpy as np
import pytest

from test_gpu_pages import dev, host

pytestmark = pytest.mark.gpu

I32 = np.int32


@pytest.mark.parametrize("M", [1, 70, 20000])
def test_no_sequence(ctx, nnhip, M):
    """Offsets of no token, every token of no sequence; the list stays as it is."""
    table, none = dev(np.zeros((0, 4), I32)), dev(np.zeros(0, I32))
    for pages in (0, 5):
        free, count = dev(np.arange(pages, dtype=I32)), dev(np.array([pages], I32))
        cu, pos, slots = dev(np.array([77], I32)), dev(np.full(M, 99, I32)), dev(np.full(M, 99, I32))
        got = ctx.pages_assign(table, 16, free, count, none, none, cu=cu, pos=pos, slots=slots)
        assert host(got[0]).tolist() == [0] and got[1].shape == (0,)
        assert np.all(host(pos) == -1) and np.all(host(slots) == -1)
        assert int(host(count)[0]) == pages and np.array_equal(host(free), np.arange(pages))
        pos, slots = dev(np.full(M, 99, I32)), dev(np.full(M, 99, I32))
        ctx.pages_slots(table, 16, max(pages, 1), got[0], pos=pos, slots=slots)
        assert np.all(host(pos) == -1) and np.all(host(slots) == -1)
        only = dev(np.full(M, 99, I32))
        ctx.pages_slots(table, 16, max(pages, 1), got[0], slots=only)
        assert np.all(host(only) == -1)
        ctx.pages_release(table, 16, free, count, none, none)
        assert int(host(count)[0]) == pages


@pytest.mark.parametrize("B", [18, 300])
def test_release_of_too_many(ctx, nnhip, B):
    """Rows that hold more pages than there are, 2^31 of them in all: the list is full then, of pages that the rows name."""
    import torch
    page, width = 8, 2 ** 31 // B + 8000
    table = (torch.arange(width, dtype=torch.int32, device="cuda") % 40)[None, :].repeat(B, 1)
    free, count = dev(np.arange(40, dtype=I32)), dev(np.array([10], I32))
    lens, keep = dev(np.full(B, page * width, I32)), dev(np.zeros(B, I32))
    assert B * width > 2 ** 31 and page * width <= 2 ** 30
    ctx.pages_release(table, page, free, count, lens, keep)
    assert int(host(count)[0]) == 40 and not host(lens).any()
    got = host(free)
    assert np.array_equal(got[:10], np.arange(10)) and got.min() >= 0 and got.max() < 40
    # the last of them were the last to be put down: the last sequence's last pages, upwards
    assert np.array_equal(got[10:], (width - 1 - np.arange(30)) % 40)
    del table
    torch.cuda.empty_cache()
