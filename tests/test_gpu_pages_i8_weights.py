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
