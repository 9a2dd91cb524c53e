"""Paged attention at sizes where the work is cut otherwise than for ordinary batches: more sequences than a wave has
lanes, more than the kernel sizes chunks for, bounds past 2^31 positions in all, long prompts in one call, head
ratios that are no power of two."""
import numpy as np
import pytest

from test_gpu_pages import U, check_decode, check_prompt, dev, host, same

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("B", [64, 65, 129, 700, 1024, 1030])
def test_decode_many_sequences(ctx, nnhip, B, f16):
    """Chunks sized by the lengths of up to 1024 sequences, found 64 at a time; one size for more. Long, short and empty
    sequences, the long ones among the last."""
    rng = np.random.default_rng(B)
    pos = rng.integers(-1, 24, B)
    pos[rng.integers(0, B, 4)] = rng.integers(130, 700, 4)
    pos[-2:] = 517, 0
    check_decode(ctx, nnhip, B, 2, 1, 64, 16, pos, f16, rope=False, seed=50)


@pytest.mark.parametrize("H,f16", [(2, False), (8, True)])
def test_decode_bound_past_31_bits(ctx, nnhip, H, f16):
    """Three sequences with a bound of 2^30 positions: one size of chunks, 2^22 here. The first has three of them, over
    four pages again and again (pages that no call writes may be shared), so its result is that of the pages' rows
    with their number of times as weights."""
    import torch
    print(f"bound 2^30 H={H} f16={f16}", flush=True)
    rng = np.random.default_rng(60)
    dk, page, bound = 64, 1024, 1 << 30
    pos = np.array([2 * (1 << 22) + 5000, 1500, -1], np.int32)
    dt = np.float16 if f16 else np.float32
    k, v = (rng.standard_normal((8, 1, page, dk)).astype(dt) for _ in range(2))
    table = np.full((3, bound // page), -1, np.int32)
    n0 = pos[0] // page
    table[0, :n0] = rng.integers(0, 4, n0)
    table[0, n0] = 4
    table[1, :2] = 5, 6
    q = rng.standard_normal((3, H, dk)).astype(np.float32)
    kn, vn = (rng.standard_normal((3, 1, dk)).astype(np.float32) for _ in range(2))
    cache = nnhip.KVPages(dev(k), dev(v), dev(table))
    out = host(ctx.attention_pages_decode(cache, dev(q.reshape(3, -1)), dev(kn.reshape(3, -1)), dev(vn.reshape(3, -1)), H,
                                          dev(pos), bound, 0.125, tokens=True)).astype(np.float64).reshape(3, H, dk)
    assert np.all(out[2] == 0)
    for b in (0, 1):
        i, s = table[b, pos[b] // page], pos[b] % page
        k[i, 0, s], v[i, 0, s] = kn[b, 0].astype(dt), vn[b, 0].astype(dt)
    assert same(host(cache.k), k) and same(host(cache.v), v)
    K, V = k[:, 0].astype(np.float64), v[:, 0].astype(np.float64)
    for b in (0, 1):
        n = int(pos[b]) + 1
        times = np.zeros((8, page))
        for i in range(8):
            times[i] = np.sum(table[b, :n // page] == i)
        times[table[b, n // page], :n % page] += 1
        assert times.sum() == n
        for h in range(H):
            x = q[b, h].astype(np.float64)
            s = K @ x * 0.125
            w = times * np.exp(s - s.max())
            w /= w.sum()
            ref = (w[..., None] * V).sum((0, 1))
            # attend64's bound, the sums over n positions
            mag = 4 * np.sqrt(dk + 8) * np.max(np.abs(K) @ np.abs(x)) * 0.125
            delta = U * (mag + 8 * np.max(np.abs(s)) + 8)
            tol = (2 * delta + U * (4 * np.sqrt(n) + 40)) * (w[..., None] * np.abs(V)).sum((0, 1)) + 1e-30
            off = np.abs(out[b, h] - ref) / tol
            assert np.all(off <= 1), f"b={b} h={h}: {off.max()} times the bound"


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("H,Hkv", [(5, 1), (7, 1), (10, 2), (15, 1)])
def test_prompt_head_ratios(ctx, nnhip, H, Hkv, f16):
    check_prompt(ctx, nnhip, [70, 1, 33], [0, 300, 17], H, Hkv, 64, 16, f16, seed=51)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("H,Hkv,dk,slopes", [(4, 1, 128, False), (2, 1, 64, True)])
def test_long_prompt_in_one_call(ctx, nnhip, H, Hkv, dk, slopes, f16):
    """One prompt of 12 K tokens behind another's 500 positions, a short one beside it."""
    check_prompt(ctx, nnhip, [12000, 5], [500, 3], H, Hkv, dk, 64, f16, slopes=slopes, seed=52, sample=12)


@pytest.mark.parametrize("width", [8, 64])  # 128 positions: a work-group a block of queries; 1024: equal spans
def test_prompt_constant_bound(ctx, nnhip, width):
    """A server's constant bound of 32 K tokens with 64 slots and 64 heads, most of a packing's columns behind its last
    sequence: the outputs of the tight bound, and the other columns as they were."""
    import torch
    print(f"constant bound width={width}", flush=True)
    rng = np.random.default_rng(70)
    B, H, Hkv, dk, page, M = 64, 64, 8, 64, 16, 1 << 15
    lens = rng.integers(0, 5, B)
    lens[[3, 40]] = 128, 77
    cu = np.concatenate(([0], np.cumsum(lens))).astype(np.int32)
    k, v = (torch.randn(B * width, Hkv, page, dk, device="cuda") for _ in range(2))
    cache = nnhip.KVPages(k, v, dev(rng.permutation(B * width).astype(np.int32).reshape(B, width)))
    q = torch.randn(H * dk, M, device="cuda")
    n = int(cu[-1])
    tight = ctx.attention_pages_prefill(cache, q[:, :n].contiguous(), dev(cu), 128, H, 0.125)
    out = ctx.attention_pages_prefill(cache, q, dev(cu), M, H, 0.125, out=torch.full((H * dk, M), 7.0, device="cuda"))
    assert torch.equal(out[:, :n], tight) and bool(torch.isfinite(tight).all()) and bool((out[:, n:] == 7.0).all())
