"""Prompts that reach past a model's positions (max_len) in a page table that goes further: with norms of queries and keys as
without, positions from max_len on are not written, and the sequence's outputs are NaN."""
import dataclasses

import numpy as np
import pytest

from test_gpu_pages import dev, host
from test_gpu_pages_i8 import CacheI8, tokens_of
from test_gpu_prefill import _gpu_model

pytestmark = pytest.mark.gpu

F32 = np.float32


@pytest.mark.parametrize("normed", [False, True])
@pytest.mark.parametrize("kind", ["i8", "f32"])
def test_prompt_past_max_len(ctx, nnhip, kind, normed):
    from nnhip_py import decoder as dmod
    print(f"prompt past max_len kind={kind} normed={normed}", flush=True)
    rng = np.random.default_rng(7)
    cfg = dmod.Config(d=256, H=4, Hkv=2, F=320, vocab=97, max_len=50, act=0, eps=1e-5)
    B, L, page, block, lens, pos0 = 3, 2, 32, 32, [20, 30, 8], [0, 25, 42]
    base = _gpu_model(ctx, nnhip, cfg, L, B, 0x51, subln=True)[0]
    gains = lambda: dev((1 + 0.2 * rng.standard_normal(cfg.dk)).astype(F32))  # noqa: E731
    blocks = [dataclasses.replace(b, g_q=gains(), g_k=gains()) for b in base.blocks] if normed else base.blocks
    mirrors = []
    for _ in range(L):
        c = CacheI8(rng, [64] * B, cfg.Hkv, page, cfg.dk, block)
        for b in range(B):
            c.put(b, 0, tokens_of(rng, pos0[b], cfg.Hkv, cfg.dk), tokens_of(rng, pos0[b], cfg.Hkv, cfg.dk))
        mirrors.append(c)
    if kind == "i8":
        caches = [c.on_device(nnhip) for c in mirrors]
    else:
        shape = (mirrors[0].codes["k"].shape[0], cfg.Hkv, page, cfg.dk)
        caches = [nnhip.KVPages(dev(np.full(shape, 7.0, F32)), dev(np.full(shape, 7.0, F32)), dev(c.table)) for c in mirrors]
    dec = dmod.Decoder(ctx, cfg, blocks, base.emb, base.g_final, base.head, B, caches=caches)
    cu = np.concatenate(([0], np.cumsum(lens))).astype(np.int32)
    seen = {}
    dec.prefill_packed(dev(rng.integers(0, cfg.vocab, sum(lens)).astype(np.int32)), dev(cu), max(lens),
                       pos0=dev(np.array(pos0, np.int32)), hook=lambda i, n, x: seen.setdefault((i, n), host(x)))
    for i in range(L):
        a = seen[i, "a"]
        assert np.isfinite(a[:, :20]).all() and np.isfinite(a[:, 50:]).all()
        assert np.isnan(a[:, 20:50]).all()  # positions 25 .. 54 of the second
    c, cache = mirrors[0], caches[0]
    kept = [n if p + n <= cfg.max_len else cfg.max_len - p for n, p in zip(lens, pos0)]
    if kind == "f32":
        k, v = host(cache.k), host(cache.v)
        for b in range(B):
            at = np.arange(64)
            written = (at >= pos0[b]) & (at < pos0[b] + kept[b])
            for x in (k, v):
                rows = x[c.table[b, at // page], :, at % page]
                assert np.array_equal((rows != 7.0).any((1, 2)), written)
        return
    if normed:  # (keys as they were seen: rotated already)
        for b in range(B):
            cols = range(cu[b], cu[b] + kept[b])
            c.put(b, pos0[b], np.stack([seen[0, "k"][:, m].reshape(cfg.Hkv, cfg.dk) for m in cols]),
                  np.stack([seen[0, "v"][:, m].reshape(cfg.Hkv, cfg.dk) for m in cols]))
        c.check(cache)


def test_limit_alone(ctx, nnhip):
    """Fill and attention of keys that were rotated before, with a limit in place of tables; refusals."""
    rng = np.random.default_rng(8)
    Hkv, H, dk, page, n = 1, 2, 64, 16, 40
    c = CacheI8(rng, [n], Hkv, page, dk, 16)
    k, v = tokens_of(rng, n, Hkv, dk), tokens_of(rng, n, Hkv, dk)
    cu = dev(np.array([0, n], np.int32))
    lay = lambda x: dev(np.ascontiguousarray(x.reshape(n, -1).T))  # noqa: E731
    q = dev(rng.standard_normal((H * dk, n)).astype(F32))
    for limit in (0, 21, 40, 100):
        cache = c.on_device(nnhip)
        ctx.kv_pages_fill(cache, lay(k), lay(v), cu, limit=limit)
        host_cache = CacheI8(np.random.default_rng(8), [n], Hkv, page, dk, 16)
        m = n if limit == 0 else min(n, limit)
        host_cache.put(0, 0, k[:m], v[:m])
        host_cache.check(cache)
        out = host(ctx.attention_pages_prefill(cache, q, cu, n, H, 0.125, limit=limit))
        assert np.isnan(out).all() if limit == 21 else np.isfinite(out).all()
    cos, sin = (dev(t) for t in nnhip.rope_table(dk, n))
    cache = c.on_device(nnhip)
    for kw in (dict(cos=cos, sin=sin, limit=5), dict(limit=-1)):
        with pytest.raises(nnhip.NNHipError, match="limit"):
            ctx.kv_pages_fill(cache, lay(k), lay(v), cu, **kw)
        with pytest.raises(nnhip.NNHipError, match="limit"):
            ctx.attention_pages_prefill(cache, q, cu, n, H, 0.125, **kw)


def test_one_gain_alone(ctx, nnhip):
    """A block with one of the two gains is refused with the decoder, before any block has run."""
    from nnhip_py import decoder as dmod
    cfg = dmod.Config(d=256, H=4, Hkv=2, F=320, vocab=97, max_len=50, act=0, eps=1e-5)
    base = _gpu_model(ctx, nnhip, cfg, 2, 2, 0x52, subln=True)[0]
    g = dev(np.ones(cfg.dk, F32))
    for kw in (dict(g_q=g), dict(g_k=g)):
        with pytest.raises(nnhip.NNHipError, match="go together"):
            dmod.Decoder(ctx, cfg, [base.blocks[0], dataclasses.replace(base.blocks[1], **kw)], base.emb, base.g_final, base.head, 2)
