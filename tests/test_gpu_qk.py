"""RMSNorm of every head of queries and keys with the rotation, against its formula in 64 bits.

Bound (u = 2^-24): the sum of squares has only positive terms, so in any order it is off by at most (dk - 1) u of itself, in
the mean by about sqrt(dk) u; 1/sqrt halves that, and the square root, the division, the two products with x and the gain and
the sum with eps are half a step each, about 6 u in all. A rotated element is a sum of two rounded products: 2 u of |y0 c| + |y1 s|. At four
deviations of the sum: (2 sqrt(dk) + 8) u (|y0 c| + |y1 s|)."""
import math

import numpy as np
import pytest

from test_gpu_pages import U, dev, host

pytestmark = pytest.mark.gpu

F32 = np.float32


def formula(x, gain, eps, cos, sin, pos):
    """x (M, heads, dk) -> outputs and their bound in 64 bits; NaN past the tables."""
    x = x.astype(np.float64)
    dk, half = x.shape[-1], x.shape[-1] // 2
    with np.errstate(all="ignore"):
        y = x / np.sqrt((x * x).sum(-1, keepdims=True) / dk + eps)
    y = y * (1.0 if gain is None else gain.astype(np.float64))
    if cos is None:
        return y, (2 * math.sqrt(dk) + 8) * U * np.abs(y)
    past = pos >= cos.shape[0]
    p = np.where((pos < 0) | past, 0, pos)
    c, s = cos[p].astype(np.float64)[:, None], sin[p].astype(np.float64)[:, None]
    a, b = y[..., :half], y[..., half:]
    out = np.concatenate((a * c - b * s, b * c + a * s), -1)
    tol = np.concatenate((np.abs(a * c) + np.abs(b * s), np.abs(b * c) + np.abs(a * s)), -1)
    out[past] = np.nan
    return out, (2 * math.sqrt(dk) + 8) * U * tol


def lay(x, tokens):
    return np.ascontiguousarray(x.reshape(x.shape[0], -1) if tokens else x.reshape(x.shape[0], -1).T)


def check(ctx, nnhip, M, H, Hkv, dk, tokens, rope=True, gains=True, eps=1e-5, seed=0, edit=None, inplace=False):
    print(f"qk M={M} H={H} Hkv={Hkv} dk={dk} tokens={tokens} rope={rope} gains={gains}", flush=True)
    rng = np.random.default_rng(seed + M + dk + H)
    x = {"q": (3 * rng.standard_normal((M, H, dk))).astype(F32), "k": (0.1 * rng.standard_normal((M, Hkv, dk))).astype(F32)}
    rows = 500
    pos = rng.integers(0, rows, M).astype(np.int32)
    if edit is not None:
        edit(x, pos)
    gain = {n: (1 + 0.3 * rng.standard_normal(dk)).astype(F32) if gains else None for n in "qk"}
    cos, sin = nnhip.rope_table(dk, rows) if rope else (None, None)
    put = {n: dev(lay(v, tokens)) if v.shape[1] else None for n, v in x.items()}
    out = {n: None if t is None else t if inplace else dev(np.full(tuple(t.shape), 7.0, F32)) for n, t in put.items()}
    q, k = ctx.qk_norm_rope(put["q"], put["k"], dk, eps, *(None if g is None else dev(g) for g in gain.values()),
                            pos=dev(pos) if rope else None, cos=None if cos is None else dev(cos),
                            sin=None if sin is None else dev(sin), q_out=out["q"], k_out=out["k"], tokens=tokens)
    for name, t in (("q", q), ("k", k)):
        if t is None:
            assert x[name].shape[1] == 0
            continue
        got = host(t) if tokens else host(t).T
        got = got.reshape(M, -1, dk).astype(np.float64)
        want, tol = formula(x[name], gain[name], eps, cos, sin, pos)
        gone = pos < 0 if rope else np.zeros(M, bool)
        assert np.all(got[gone] == (x[name][gone] if inplace else 7.0))
        got, want, tol = got[~gone], want[~gone], tol[~gone]
        nan = np.isnan(want)
        assert np.array_equal(nan, np.isnan(got))
        assert np.all(np.abs(got - want)[~nan] <= tol[~nan] + 1e-37)


@pytest.mark.parametrize("tokens", [False, True])
@pytest.mark.parametrize("M,H,Hkv,dk", [(1, 1, 1, 64), (16, 20, 5, 128), (3, 7, 7, 256), (64, 4, 1, 64), (65, 3, 2, 128),
                                        (1000, 20, 5, 128), (333, 2, 1, 256), (129, 16, 2, 64), (4099, 1, 1, 64)])
def test_qk(ctx, nnhip, M, H, Hkv, dk, tokens):
    check(ctx, nnhip, M, H, Hkv, dk, tokens)


@pytest.mark.parametrize("tokens", [False, True])
def test_qk_forms(ctx, nnhip, tokens):
    """Without tables, without gains, queries or keys alone, in place; tokens of no sequence and past the tables; zeros,
    NaN and infinities in one head."""
    check(ctx, nnhip, 70, 4, 2, 128, tokens, rope=False)
    check(ctx, nnhip, 70, 4, 2, 64, tokens, gains=False)
    check(ctx, nnhip, 70, 0, 3, 128, tokens)
    check(ctx, nnhip, 70, 3, 0, 128, tokens)
    check(ctx, nnhip, 130, 5, 2, 128, tokens, inplace=True)

    def odd(x, pos):
        pos[[0, 7, 69]] = [-1, -5, -2 ** 31]
        pos[[3, 68]] = [500, 2 ** 31 - 1]
        x["q"][10, 1] = 0
        x["q"][11, 0, 5] = np.nan
        x["k"][12, 1] = F32(1e-30)

    check(ctx, nnhip, 70, 3, 2, 128, tokens, edit=odd)
    check(ctx, nnhip, 70, 3, 2, 128, tokens, edit=odd, inplace=True)

    def zero(x, pos):
        x["q"][4, 0] = 0

    check(ctx, nnhip, 20, 2, 1, 64, tokens, edit=zero, eps=0.0)  # 0 / 0


def test_qk_is_rmsnorm_then_rotation(ctx, nnhip):
    """Without gains' help: one head, no tables, against nnhip_rmsnorm (another order of the sum: 2 steps of the result)."""
    rng = np.random.default_rng(3)
    x = dev(rng.standard_normal((128, 500)).astype(F32))
    g = dev((1 + rng.standard_normal(128)).astype(F32))
    q, _ = ctx.qk_norm_rope(x, None, 128, 1e-6, g)
    want = host(ctx.rmsnorm(x, g, 1e-6)).astype(np.float64)
    assert np.all(np.abs(host(q) - want) <= (2 * math.sqrt(128) + 8) * U * np.abs(want))


def test_qk_refusals(ctx, nnhip):
    x = dev(np.zeros((128, 4), F32))
    cos, sin = (dev(t) for t in nnhip.rope_table(128, 8))
    for kw, what in ((dict(cos=cos, sin=sin), "positions"), (dict(cos=cos), "go together"),
                     (dict(pos=dev(np.zeros(5, np.int32))), "shape"), (dict(gamma_q=dev(np.zeros(64, F32))), "shape")):
        with pytest.raises(nnhip.NNHipError, match=what):
            ctx.qk_norm_rope(x, None, 128, 1e-5, **kw)
    with pytest.raises(nnhip.NNHipError, match="heads of 48"):
        ctx.qk_norm_rope(x, None, 48, 1e-5)
    with pytest.raises(nnhip.NNHipError, match="dk must be"):
        ctx.qk_norm_rope(x, None, 32, 1e-5)
    with pytest.raises(nnhip.NNHipError, match="must be given"):
        ctx.qk_norm_rope(None, None, 128, 1e-5)
    with pytest.raises(nnhip.NNHipError, match="k_out without"):
        ctx.qk_norm_rope(x, None, 128, 1e-5, k_out=x)
    q, k = ctx.qk_norm_rope(dev(np.zeros((128, 0), F32)), None, 128, 1e-5)
    assert k is None and q.shape == (128, 0)
