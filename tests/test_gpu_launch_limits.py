"""Sizes whose launch would pass 2^32 threads are refused by name, before anything is launched: the pointers here hold no such tensors."""
import numpy as np
import pytest

from test_gpu_pages import dev

pytestmark = pytest.mark.gpu


def test_refused(ctx, nnhip):
    L = nnhip.lib()
    x = dev(np.zeros(64, np.float32)).data_ptr()
    for M, H, dk, tokens in ((2 ** 29, 1, 64, 1), (2 ** 24, 8, 256, 1), (2 ** 29, 1, 64, 0)):
        assert L.nnhip_qk_norm_rope(ctx.h, x, None, M, H, 0, dk, None, None, 1e-5, None, None, None, 0, tokens, x, None) == 1
        assert "2^35" in L.nnhip_last_error().decode()
    cache = nnhip.KVPagesI8.empty(2, 1, 16, 64, 16, dev(np.zeros((1, 1), np.int32)))
    cu = dev(np.zeros(2, np.int32))
    for M in (2 ** 29 - 64, 2 ** 30):
        assert L.nnhip_kv_pages_fill_i8(ctx.h, cache.ref, x, x, M, cu.data_ptr(), None, 1, None, None, 0) == 1
        assert "too large" in L.nnhip_last_error().decode()
