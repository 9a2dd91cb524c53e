"""Attention over an 8-bit cache where one position takes nearly all of the weight and thousands of equal ones share the rest:
their part of the sum is there as far as f32 holds it.

All scores are 0 but that of position 0, which is gap log2 units above them; its value is 0. So an output is the others' share
times their values, and what is lost of their weights shows by itself. Bound: attend64's, relative to the share, and what the
kernels' own roundings leave out. Decode holds a weight times its block's scale to 2^-31 of the largest such product in its tile of 64
positions, prompts a weight to 2^-22 of itself, and to 2^-32 of the largest over up to 8192 keys or 2^-25 of the largest in its tile of 64; values
are up to 127 times the scale."""
import math

import numpy as np
import pytest

from test_gpu_pages import attend64, dev, host

pytestmark = pytest.mark.gpu

F32 = np.float32


def sink(nnhip, n, gap, B, Hkv, dk, page=256, block=64, at=0):
    """A cache of n positions that B sequences share, a query, and the keys and values of a head, in 64 bits."""
    import torch
    pages, scale = n // page, 1 / math.sqrt(dk)
    k = np.zeros((n, dk), np.int8)
    k[at] = 127
    v = np.where(np.arange(dk) % 2, 100, -77).astype(np.int8) * np.ones((n, 1), np.int8)
    v[at] = 0
    ks, vs = np.full(n // block, gap * math.log(2) / (dk * 127 * scale), F32), np.full(n // block, 0.5, F32)
    kc = np.broadcast_to(k.reshape(pages, 1, page // 16, 16, dk // 16, 16).transpose(0, 1, 2, 4, 3, 5), (pages, Hkv, page // 16, dk // 16, 16, 16))
    vc = np.broadcast_to(v.reshape(pages, 1, page // 16, 16, dk).transpose(0, 1, 2, 4, 3), (pages, Hkv, page // 16, dk, 16))
    sc = lambda s: dev(np.broadcast_to(s.reshape(pages, 1, -1), (pages, Hkv, page // block)).copy())  # noqa: E731
    table = dev(np.broadcast_to(np.arange(pages, dtype=np.int32), (B, pages)).copy())
    cache = nnhip.KVPagesI8(dev(kc.copy()), dev(vc.copy()), sc(ks), sc(vs), table)
    K = k.astype(np.float64) * np.repeat(ks, block)[:, None].astype(np.float64)
    V = v.astype(np.float64) * 0.5
    return cache, K, V, float(F32(scale))


def expected(K, V, dk, scale, n, run, weight):
    """The result for a query of ones over the first n positions, and its bound."""
    q = np.ones(dk)
    want, tol = attend64(q, K[:n], V[:n], scale, 0.0, 0.0, np.zeros(n), np.ones(n, bool))
    s = (K[:n] @ q) * scale
    p = np.exp(s - s.max())
    p /= p.sum()
    runs = np.add.reduceat(np.ones(n), np.arange(0, n, run)) * np.maximum.reduceat(p, np.arange(0, n, run))
    return want, tol + weight * runs.sum() * 127 * 0.5 + 2.0 ** -22 * (p @ np.abs(V[:n]))


@pytest.mark.parametrize("H,Hkv,dk", [(1, 1, 64), (8, 1, 128), (4, 1, 256)])
@pytest.mark.parametrize("n,B,gap,at", [(1024, 2, 28.0, 0), (1024, 2, 40.0, 700), (16384, 600, 31.0, 0), (16384, 600, 31.0, 9000), (4096, 1, 35.0, 5)])
def test_decode_of_a_sink(ctx, nnhip, H, Hkv, dk, n, B, gap, at):
    print(f"decode H={H} Hkv={Hkv} dk={dk} n={n} B={B} gap={gap} at={at}", flush=True)
    cache, K, V, scale = sink(nnhip, n, gap, B, Hkv, dk, at=at)
    q = dev(np.ones((B, H * dk), F32))
    out = host(ctx.attention_pages_decode(cache, q, None, None, H, dev(np.full(B, n - 1, np.int32)), n, scale, tokens=True))
    out = out.reshape(B, H, dk).astype(np.float64)
    assert np.isfinite(out).all()
    want, tol = expected(K, V, dk, scale, n, 64, 2.0 ** -31)
    worst = float(np.max(np.abs(out - want) / tol))
    print(f"  share {abs(want[0]) / 38.5:.2e}, bound {np.max(tol / np.abs(want)):.2e} of it, worst {worst:.3f} of the bound", flush=True)
    assert worst <= 1.0


def test_decode_of_a_large_value_without_weight(ctx, nnhip):
    """A block with a value 2^40 times the others' and 2^-60 of their weight: the others' weights keep their bits beside it in a tile."""
    n, dk = 512, 64
    cache, K, V, scale = sink(nnhip, n, 0.0, 1, 1, dk, block=16, page=64)
    # positions 16 .. 31: scores 60 log2 units below the others', values of 100 * 2^40 at position 20 and of 0
    k = host(cache.k).copy()
    v = host(cache.v).copy()
    vs = host(cache.v_scale).copy()
    ks = host(cache.k_scale).copy()
    k[0, 0, 1] = -127
    ks[0, 0, 1] = 60 * math.log(2) / (dk * 127 * scale)
    v[0, 0, 1] = 0
    v[0, 0, 1, :, 4] = 100
    vs[0, 0, 1] = 2.0 ** 40
    rng = np.random.default_rng(3)
    for x, y in ((cache.k, k), (cache.v, v), (cache.k_scale, ks), (cache.v_scale, vs)):
        x.copy_(dev(y))
    K, V = K.copy(), V.copy()
    K[16:32], V[16:32] = -127.0 * float(F32(ks[0, 0, 1])), 0.0
    V[20] = 100 * 2.0 ** 40
    q = (1 + 0.3 * rng.standard_normal(dk)).astype(F32)
    out = host(ctx.attention_pages_decode(cache, dev(q[:, None]), None, None, 1, dev(np.array([n - 1], np.int32)), n, scale))[:, 0].astype(np.float64)
    want, tol = attend64(q.astype(np.float64), K, V, scale, 0.0, 0.0, np.zeros(n), np.ones(n, bool))
    # of the tile's largest weight times scale, 2^-1 / 496 (2^40 2^-60 / 496 in that block)
    tol = tol + 2.0 ** -31 * n * 127 * 0.5 / 496
    worst = float(np.max(np.abs(out - want) / tol))
    print(f"  worst {worst:.3f} of the bound", flush=True)
    assert worst <= 1.0


@pytest.mark.parametrize("slopes", [False, True])
@pytest.mark.parametrize("H,Hkv,dk,B,T", [(32, 32, 64, 8, 5), (32, 32, 64, 2, 200), (16, 2, 128, 8, 40), (4, 4, 128, 1, 64)])
@pytest.mark.parametrize("gap,at", [(32.0, 0), (37.0, 0), (33.0, 20000)])
def test_prompt_of_a_sink(ctx, nnhip, H, Hkv, dk, B, T, gap, at, slopes):
    print(f"prompt H={H} Hkv={Hkv} dk={dk} B={B} T={T} gap={gap} at={at} slopes={slopes}", flush=True)
    n = 65536
    cache, K, V, scale = sink(nnhip, n, gap, B, Hkv, dk, at=at)
    q = dev(np.ones((H * dk, B * T), F32))
    cu = dev(np.arange(B + 1, dtype=np.int32) * T)
    out = host(ctx.attention_pages_prefill(cache, q, cu, T, H, scale, pos0=dev(np.full(B, n - T, np.int32)),
                                           slopes=dev(np.zeros(H, F32)) if slopes else None))
    out = out.T.reshape(B, T, H, dk).astype(np.float64)
    assert np.isfinite(out).all()
    worst = 0.0
    for t in {0, T // 2, T - 1}:
        want, tol = expected(K, V, dk, scale, n - T + t + 1, 64, 2.0 ** -25)
        tol = tol + 8192 * 2.0 ** -32 * 127 * 0.5
        worst = max(worst, float(np.max(np.abs(out[:, t] - want) / tol)))
    print(f"  share {abs(want[0]) / 38.5:.2e}, bound {np.max(tol / np.abs(want)):.2e} of it, worst {worst:.3f} of the bound", flush=True)
    assert worst <= 1.0
