"""Blocks of an 8-bit cache whose scale is NaN, as a caller may have left them, when further tokens join them: the scale stays, the
new tokens' codes are 0, and the block's positions stand for NaN, by whichever kernel the tokens are written."""
import numpy as np
import pytest

from test_gpu_pages import dev, host
from test_gpu_pages_i8 import CacheI8, check_decode, fill, tokens_of

pytestmark = pytest.mark.gpu

F32 = np.float32


@pytest.mark.parametrize("name", ["k", "v"])
@pytest.mark.parametrize("lens", [[5, 20, 3], [300, 140, 200]])  # by columns, by windows of positions
@pytest.mark.parametrize("dk,block", [(64, 16), (128, 32), (256, 64)])
def test_fill_goes_on_with_nan(ctx, nnhip, dk, block, lens, name):
    print(f"fill dk={dk} block={block} lens={lens} {name}", flush=True)
    rng = np.random.default_rng(dk + len(name) + lens[0])
    Hkv, page, pos0 = 2, 64, [37, 70, 11]
    c = CacheI8(rng, np.array(lens) + np.array(pos0), Hkv, page, dk, block)
    for b, p in enumerate(pos0):
        c.put(b, 0, tokens_of(rng, p, Hkv, dk), tokens_of(rng, p, Hkv, dk))
    for b, g in ((0, 1), (1, 0)):
        c.scales[name][c.table[b, pos0[b] // page], g, pos0[b] % page // block] = np.nan
    cache = c.on_device(nnhip)
    M = sum(lens)
    fill(ctx, cache, c, tokens_of(rng, M, Hkv, dk), tokens_of(rng, M, Hkv, dk), lens, pos0, nnhip.rope_table(dk, 400))
    c.check(cache)
    n = [a + b for a, b in zip(lens, pos0)]
    cu = np.concatenate(([0], np.cumsum(n))).astype(np.int32)
    got = dict(zip("kv", (host(x) for x in ctx.kv_pages_read(cache, dev(cu), sum(n)))))
    for x in "kv":
        want = np.zeros((sum(n), Hkv), bool)
        if x == name:
            for b, g in ((0, 1), (1, 0)):
                first = pos0[b] // block * block
                want[cu[b] + first:cu[b] + min(first + block, n[b]), g] = True
        assert np.array_equal(np.isnan(got[x].T.reshape(sum(n), Hkv, dk)), np.broadcast_to(want[..., None], (sum(n), Hkv, dk)))


@pytest.mark.parametrize("H,Hkv,dk", [(8, 2, 64), (32, 2, 64), (8, 2, 256), (10, 2, 128)])  # the second and third append in a launch of their own
@pytest.mark.parametrize("pos", [[40, 200, 14], [3000, 1500, 14]])
def test_decode_goes_on_with_nan(ctx, nnhip, H, Hkv, dk, pos):
    """The step that joins such a block and the next one, which only reads, agree."""
    base = dict(B=3, H=H, Hkv=Hkv, dk=dk, page=16, block=16, pos=pos, rope=False)
    for name, b, g in (("k", 0, 0), ("v", 1, 1), ("v", 2, 0)):
        def edit(c, q, k, v):
            c.scales[name][c.table[b, pos[b] // 16], g, 0] = np.nan

        _, cache, out = check_decode(ctx, nnhip, **base, edit=edit)
        heads = np.arange(H) // (H // Hkv) == g
        assert np.isnan(out[b][heads]).all() and np.isfinite(out[b][~heads]).all()
        q = dev(np.random.default_rng(1).standard_normal((3, H * dk)).astype(F32))
        again = host(ctx.attention_pages_decode(cache, q, None, None, H, dev(np.array(pos, np.int32)), max(pos) + 1, 0.1,
                                                tokens=True)).reshape(3, H, dk)
        assert np.array_equal(np.isnan(again), np.isnan(out))
