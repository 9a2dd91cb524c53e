"""The decoder over 8-bit pages whose table is kept on the GPU, with norms of queries and keys: prompts of unlike lengths in
one packed pass, then steps with a sequence that ends and one that moves in, as a server runs them.

The int8 stages are checked elsewhere, so here each block's queries and keys are held to the norm's formula, its
attention to an evaluation in 64 bits on the block's own q, k and v (the bounds of test_gpu_qk.py and test_gpu_pages_i8.py),
the pools to the definition bit for bit, and the tables to the sequences' lengths."""
import dataclasses

import numpy as np
import pytest

from test_gpu_pages import attend64, dev, host, rotate
from test_gpu_pages_i8 import CacheI8, own_bound
from test_gpu_prefill import _gpu_model
from test_gpu_qk import formula

pytestmark = pytest.mark.gpu


class Server:
    """Caches of every block with one table, its free list, and a mirror of all of it on the host."""

    def __init__(self, nnhip, cfg, L, rows, page, block, width, rng, spare=2):
        self.nnhip, self.cfg, self.page, self.rows = nnhip, cfg, page, rows
        pages = rows * width + spare
        self.table = dev(np.full((rows, width), -1, np.int32))
        self.free, self.count = dev(rng.permutation(pages).astype(np.int32)), dev(np.array([pages], np.int32))
        self.lens = dev(np.zeros(rows, np.int32))
        self.host = []
        for _ in range(L):
            c = CacheI8(rng, [0], cfg.Hkv, page, cfg.dk, block, extra=pages)
            self.host.append(c)
        on = [c.on_device(nnhip) for c in self.host]
        self.caches = [nnhip.KVPagesI8(c.k, c.v, c.k_scale, c.v_scale, self.table) for c in on]

    def assign(self, ctx, add, **kw):
        got = ctx.pages_assign(self.table, self.page, self.free, self.count, self.lens, dev(np.array(add, np.int32)), **kw)
        for c in self.host:
            c.table = host(self.table)
        return got

    def check(self, i, b, p, q, a, factor=1, turned=True, cos=None, sin=None):
        cfg, c = self.cfg, self.host[i]
        K, V = c.rows(b, p + 1)
        at = np.arange(p + 1)
        q = q.reshape(cfg.H, cfg.dk).astype(np.float64)
        q = q if turned else rotate(q, cos.astype(np.float64), sin.astype(np.float64), p)
        for h in range(cfg.H):
            g = h // (cfg.H // cfg.Hkv)
            ref, tol = attend64(q[h], K[:, g], V[:, g], cfg.scale, 0.0, 0.0, at - float(p), np.ones(p + 1, bool))
            tol = tol + own_bound(q[h], K[:, g], V[:, g], cfg.scale, p + 1, 2.0 ** -24)
            assert np.all(np.abs(a.reshape(cfg.H, cfg.dk)[h] - ref) <= factor * tol), f"block {i} b={b} p={p} h={h}"

    def same_pools(self):
        for c, d in zip(self.host, self.caches):
            c.check(d)


def model(ctx, nnhip, cfg, L, B, seed, normed, rng):
    base = _gpu_model(ctx, nnhip, cfg, L, B, seed, subln=True)[0]
    if normed:
        gains = lambda: dev((1 + 0.2 * rng.standard_normal(cfg.dk)).astype(np.float32))  # noqa: E731
        base.blocks = [dataclasses.replace(b, g_q=gains(), g_k=gains()) for b in base.blocks]
    return base


@pytest.mark.parametrize("B,normed,page,block", [(4, True, 16, 16), (3, False, 32, 16), (18, True, 32, 32)])
def test_server(ctx, nnhip, B, normed, page, block):
    """B = 18 runs the unfused step."""
    from nnhip_py import decoder as dmod
    print(f"server B={B} normed={normed}", flush=True)
    rng = np.random.default_rng(400 + B)
    cfg = dmod.Config(d=256, H=4, Hkv=2, F=320, vocab=97, max_len=96, act=0, eps=1e-5)
    L = 2
    base = model(ctx, nnhip, cfg, L, B, 0x8A + B, normed, rng)
    s = Server(nnhip, cfg, L, B, page, block, 96 // page, rng)
    cos, sin = nnhip.rope_table(cfg.dk, cfg.max_len)
    dec = dmod.Decoder(ctx, cfg, base.blocks, base.emb, base.g_final, base.head, B, caches=s.caches)
    assert dec.paged
    lens = [int(x) for x in rng.integers(1, 60, B)]
    lens[0], lens[-1] = 33, 1
    cu, pos0 = s.assign(ctx, lens)
    assert np.array_equal(host(cu), np.concatenate(([0], np.cumsum(lens)))) and np.all(host(pos0) == 0)
    assert np.array_equal(host(s.lens), lens)
    prompt = rng.integers(0, cfg.vocab, sum(lens)).astype(np.int32)
    seen = {}

    def hook(i, name, t):
        seen[i, name] = host(t)

    def key(k, p):  # as the cache gets it
        k = k.reshape(cfg.Hkv, cfg.dk)
        return k if normed else rotate(k, cos, sin, p)

    logits, ids = dec.prefill_packed(dev(prompt), cu, max(lens), pos0=pos0, hook=hook)
    first = host(ids).copy()
    assert np.array_equal(first, host(logits).argmax(0))
    at = host(cu)
    for i in range(L):
        for b in range(B):
            cols = range(at[b], at[b + 1])
            s.host[i].put(b, 0, np.stack([key(seen[i, "k"][:, c], c - at[b]) for c in cols]),
                          np.stack([seen[i, "v"][:, c].reshape(cfg.Hkv, cfg.dk) for c in cols]))
            for t in sorted({0, lens[b] // 2, lens[b] - 1}):
                s.check(i, b, t, seen[i, "q"][:, at[b] + t], seen[i, "a"][:, at[b] + t], turned=normed, cos=cos, sin=sin)
    s.same_pools()
    if normed:
        # the first block's projections without norms are the normed ones' inputs
        bare = [dataclasses.replace(b, g_q=None, g_k=None) for b in base.blocks]
        t = Server(nnhip, cfg, L, B, page, block, 96 // page, np.random.default_rng(1))
        cu2, pos2 = t.assign(ctx, lens)
        raw = {}
        dmod.Decoder(ctx, cfg, bare, base.emb, base.g_final, base.head, B, caches=t.caches).prefill_packed(
            dev(prompt), cu2, max(lens), pos0=pos2, hook=lambda i, n, x: raw.setdefault((i, n), host(x)))
        place = np.concatenate([np.arange(n) for n in lens])
        for name, heads, gain in (("q", cfg.H, base.blocks[0].g_q), ("k", cfg.Hkv, base.blocks[0].g_k)):
            want, tol = formula(raw[0, name].T.reshape(-1, heads, cfg.dk), host(gain), cfg.eps, cos, sin, place)
            assert np.all(np.abs(seen[0, name].T.reshape(want.shape) - want) <= tol)

    # steps: sequence 1 ends after the first, another moves into its slot two steps later
    live = np.ones(B, bool)
    length = np.array(lens)
    ids_d = dev(first)
    for step in range(5):
        if step == 1:
            keep = length.copy()
            keep[1] = 0
            ctx.pages_release(s.table, page, s.free, s.count, s.lens, dev(keep.astype(np.int32)))
            length[1], live[1] = 0, False
        if step == 3:
            live[1] = True
        _, pos = s.assign(ctx, live.astype(int))
        want = np.where(live, length, -1)
        assert np.array_equal(host(pos), want)

        def attn_hook(i, a):
            tm = dec._tok and dec.fused_ok()
            q, k, v = (host(x) if tm else host(y).T for x, y in
                       (((dec.q_t if dec._tok else dec.q), dec.q), ((dec.k_t if dec._tok else dec.k), dec.k),
                        ((dec.v_t if dec._tok else dec.v), dec.v)))
            a = host(a).T
            for b in range(B):
                if want[b] < 0:
                    assert np.all(a[b] == 0)
                    continue
                s.host[i].put(b, int(want[b]), key(k[b], want[b])[None], v[b].reshape(1, cfg.Hkv, cfg.dk))
                s.check(i, b, int(want[b]), q[b], a[b], turned=normed, cos=cos, sin=sin)

        logits, got = dec.step(ids_d, pos, cfg.max_len, attn_hook=attn_hook)
        assert np.array_equal(host(got)[live], host(logits).argmax(0)[live])
        ids_d = got.clone()
        length[live] += 1
        s.same_pools()
    held = sum(-(-int(n) // page) for n in length)
    assert int(host(s.count)[0]) == s.free.shape[0] - held
    ids_held = [int(host(s.table)[b, i]) for b in range(B) for i in range(-(-int(length[b]) // page))]
    assert sorted(ids_held + host(s.free)[:s.free.shape[0] - held].tolist()) == list(range(s.free.shape[0]))


def test_captured_server_step(nnhip):
    """A step with its pages, norms and choice, captured once and replayed between eager work, goes on as eager steps do."""
    import torch
    from nnhip_py import decoder as dmod
    ctx = nnhip.Context(0)
    cfg = dmod.Config(d=256, H=4, Hkv=1, F=320, vocab=97, max_len=320, act=1, eps=1e-5)
    B = 3
    base = model(ctx, nnhip, cfg, 2, B, 0xCA8, True, np.random.default_rng(50))
    runs = []
    for captured in (False, True):
        s = Server(nnhip, cfg, 2, B, 16, 16, 20, np.random.default_rng(51))
        dec = dmod.Decoder(ctx, cfg, base.blocks, base.emb, base.g_final, base.head, B, caches=s.caches)
        lens = [250, 3, 127]
        prompt = dev(np.random.default_rng(52).integers(0, 97, sum(lens)).astype(np.int32))
        one, cu, pos = dev(np.ones(B, np.int32)), dev(np.zeros(B + 1, np.int32)), dev(np.zeros(B, np.int32))
        side = torch.cuda.Stream()

        def step():
            ctx.pages_assign(s.table, 16, s.free, s.count, s.lens, one, cu=cu, pos0=pos)
            _, got = dec.step(ids, pos, cfg.max_len)
            ids.copy_(got)

        with torch.cuda.stream(side):
            c0, p0 = s.assign(ctx, lens)
            _, ids = dec.prefill_packed(prompt, c0, 250, pos0=p0)
            ids = ids.clone()
            step()
        torch.cuda.synchronize()
        trace = [host(ids).copy()]
        if captured:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                step()
        for _ in range(6):
            if captured:
                g.replay()
            else:
                with torch.cuda.stream(side):
                    step()
            torch.cuda.synchronize()
            ctx.argmax_rows(torch.randn(3, 50, device="cuda"))
            trace.append(host(ids).copy())
        runs.append((np.array(trace), host(s.lens), host(pos), host(s.table), host(s.caches[1].k), host(s.caches[1].v_scale)))
    for a, b in zip(*runs):
        assert np.array_equal(a, b, equal_nan=a.dtype.kind == "f")
    ctx.close()


@pytest.mark.parametrize("rope", [True, False])
def test_norms_over_contiguous_caches(ctx, nnhip, rope):
    """prefill() and step() over f32 caches of equal prompts with norms: queries and keys by the formula, keys in the cache
    as they are, attention in 64 bits."""
    from nnhip_py import decoder as dmod
    rng = np.random.default_rng(9)
    cfg = dmod.Config(d=256, H=4, Hkv=2, F=320, vocab=97, max_len=40, act=0, eps=1e-5, rope=rope)
    B, T = 2, 11
    base = model(ctx, nnhip, cfg, 2, B, 0x31, True, rng)
    cos, sin = nnhip.rope_table(cfg.dk, cfg.max_len)
    prompt = dev(rng.integers(0, cfg.vocab, B * T).astype(np.int32))
    seen, raw = {}, {}
    bare = [dataclasses.replace(b, g_q=None, g_k=None) for b in base.blocks]
    dmod.Decoder(ctx, cfg, bare, base.emb, base.g_final, base.head, B).prefill(
        prompt, T, pos0=2, hook=lambda i, n, x: raw.setdefault((i, n), host(x)))
    dec = dmod.Decoder(ctx, cfg, base.blocks, base.emb, base.g_final, base.head, B)
    for c in dec.caches:
        c[0].normal_()
        c[1].normal_()
    _, ids = dec.prefill(prompt, T, pos0=2, hook=lambda i, n, x: seen.setdefault((i, n), host(x)))
    place = np.tile(np.arange(2, 2 + T), B)
    for name, heads, gain in (("q", cfg.H, base.blocks[0].g_q), ("k", cfg.Hkv, base.blocks[0].g_k)):
        want, tol = formula(raw[0, name].T.reshape(-1, heads, cfg.dk), host(gain), cfg.eps, cos if rope else None, sin, place)
        assert np.all(np.abs(seen[0, name].T.reshape(want.shape) - want) <= tol)
    for i in range(2):
        for b in range(B):
            k = host(dec.caches[i][0])[b, 2:2 + T].reshape(T, -1)
            assert np.array_equal(k, seen[i, "k"][:, b * T:(b + 1) * T].T)
    pos = dev(np.full(B, 2 + T, np.int32))

    def attn_hook(i, a):
        K, V = (host(x).reshape(B, cfg.max_len, cfg.Hkv, cfg.dk)[:, :3 + T].astype(np.float64) for x in dec.caches[i])
        q = (host(dec.q_t) if dec._tok and dec.fused_ok() else host(dec.q).T).reshape(B, cfg.H, cfg.dk)
        for b in range(B):
            for h in range(cfg.H):
                ref, tol = attend64(q[b, h].astype(np.float64), K[b, :, h // 2], V[b, :, h // 2], cfg.scale, 0.0, 0.0,
                                    np.zeros(3 + T), np.ones(3 + T, bool))
                assert np.all(np.abs(host(a).T.reshape(B, cfg.H, cfg.dk)[b, h] - ref) <= tol)

    dec.step(ids, pos, cfg.max_len, attn_hook=attn_hook)


def test_refusals(ctx, nnhip):
    from nnhip_py import decoder as dmod
    rng = np.random.default_rng(60)
    cfg = dmod.Config(d=256, H=4, Hkv=2, F=320, vocab=97, max_len=96, act=0, eps=1e-5)
    base = model(ctx, nnhip, cfg, 1, 2, 0x77, True, rng)
    s = Server(nnhip, cfg, 1, 2, 16, 16, 8, rng)
    ids, pos = dev(np.zeros(2, np.int32)), dev(np.zeros(2, np.int32))
    dec = dmod.Decoder(ctx, cfg, base.blocks, base.emb, base.g_final, base.head, 2, caches=s.caches)
    with pytest.raises(nnhip.NNHipError, match="prefill_packed"):
        dec.prefill(ids, 1)
    with pytest.raises(nnhip.NNHipError, match="len_bound"):
        dec.step(ids, pos, 97)
    dec.blocks = [dataclasses.replace(base.blocks[0], g_k=None)]
    with pytest.raises(nnhip.NNHipError, match="go together"):
        dec.step(ids, pos, 96)
