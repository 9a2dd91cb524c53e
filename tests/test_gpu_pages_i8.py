"""The paged KV cache in 8 bits on the GPU: its fill, the values read back, and the attention of one new token per
sequence and of packed prompts, against evaluations in 64 bits.

What the cache holds (codes, scales, and that nothing else of the pools changes) is compared bit for bit with the
definition: s = fl(max|x| fl(1/127)), q = round_half_away(clamp(fl(x/s))), a larger value raises a block's scale and its
older values are quantized again. Attention is held to test_gpu_pages.attend64's bound over the values that the cache
holds, and to the roundings of its own that come on top. Decode (n positions): queries to 2^-31 of their largest element,
at most dk 2^-31 max|q| max|K| |scale| of a score; weights to 2^-31 where the largest is between 2^-4 and 1, times a power of
two at most twice a scale, so 2^-26 of the largest weight and value each, 4 sqrt(n) of them in all. Prompts: weights to 2^-22
of themselves, and to 2^-25 where the largest is 2^6 times at least 2^-6 of the largest value's scale, or 2^-24 of the largest
weight and value each, again 4 sqrt(n) of them."""
import math

import numpy as np
import pytest

from test_gpu_pages import U, attend64, dev, host, rotate

pytestmark = pytest.mark.gpu

F32 = np.float32


def quantized(x, s):
    """round_half_away(clamp(fl(x / s))), 0 for NaN and where s is 0, as int8 (arrays of float32)."""
    with np.errstate(all="ignore"):
        y = (x.astype(F32) / s.astype(F32)).astype(F32)
    y = np.where((s == 0) | np.isnan(y), F32(0), y)
    y = np.clip(y, F32(-127), F32(127)).astype(np.float64)
    return (np.sign(y) * np.floor(np.abs(y) + 0.5)).astype(np.int8)


class CacheI8:
    """A cache on the host: codes (pages, Hkv, page, dk), scales (pages, Hkv, page / block), both full of noise where no
    sequence has been written, and sequences of given lengths at pages of their own."""

    def __init__(self, rng, lens, Hkv, page, dk, block, extra=3, width=None):
        need = [-(-int(n) // page) for n in lens]
        self.Hkv, self.page, self.dk, self.block = Hkv, page, dk, block
        total = sum(need) + extra
        places = rng.permutation(total)[:sum(need)].astype(np.int32)
        self.table = np.full((len(lens), max(1, max(need)) if width is None else width), -1, np.int32)
        self.codes = {n: rng.integers(-128, 128, (total, Hkv, page, dk)).astype(np.int8) for n in "kv"}
        # scales that nobody has set: NaN, infinities, large values
        self.scales = {n: rng.choice(np.array([np.nan, np.inf, 1e30, 1.0], F32), (total, Hkv, page // block)) for n in "kv"}
        at = 0
        for b in range(len(lens)):
            self.table[b, :need[b]] = places[at:at + need[b]]
            at += need[b]

    def put(self, b, p0, k, v):
        """Tokens k, v (n, Hkv, dk) from position p0 of sequence b on, as the definition says."""
        G = self.block
        for name, x in (("k", k), ("v", v)):
            n = x.shape[0]
            for j in range(p0 // G, (p0 + n - 1) // G + 1 if n else p0 // G):
                lo, hi = max(j * G, p0), min((j + 1) * G, p0 + n)
                page, slot = self.table[b, j * G // self.page], j * G % self.page
                new = x[lo - p0:hi - p0]
                with np.errstate(invalid="ignore"):
                    s = (np.nanmax(np.where(np.isnan(new), 0, np.abs(new)), axis=(0, 2)).astype(F32) * F32(1 / 127)).astype(F32)
                for g in range(self.Hkv):
                    step = s[g]
                    if lo > j * G:
                        old = self.scales[name][page, g, slot // G]
                        if s[g] > old:
                            here = self.codes[name][page, g, slot:slot + lo - j * G]
                            with np.errstate(all="ignore"):
                                here[:] = quantized(here.astype(F32) * old, np.broadcast_to(step, here.shape))
                        else:
                            step = old
                    self.scales[name][page, g, slot // G] = step
                    self.codes[name][page, g, slot + lo - j * G:slot + hi - j * G] = quantized(new[:, g], np.broadcast_to(step, new[:, g].shape))

    def rows(self, b, n):
        """Keys and values of positions 0 .. n - 1, (n, Hkv, dk) in 64 bits."""
        i, s = self.table[b, np.arange(n) // self.page], np.arange(n) % self.page
        with np.errstate(all="ignore"):
            return tuple(self.codes[x][i, :, s].astype(np.float64) * self.scales[x][i, :, s // self.block][..., None].astype(np.float64)
                         for x in "kv")

    def on_device(self, nnhip):
        P, H, page, dk = self.codes["k"].shape
        k = self.codes["k"].reshape(P, H, page // 16, 16, dk // 16, 16).transpose(0, 1, 2, 4, 3, 5)
        v = self.codes["v"].reshape(P, H, page // 16, 16, dk).transpose(0, 1, 2, 4, 3)
        return nnhip.KVPagesI8(dev(k), dev(v), dev(self.scales["k"]), dev(self.scales["v"]), dev(self.table))

    def check(self, cache):
        """The device's cache holds the same bits."""
        P, H, page, dk = self.codes["k"].shape
        k = host(cache.k).transpose(0, 1, 2, 4, 3, 5).reshape(P, H, page, dk)
        v = host(cache.v).transpose(0, 1, 2, 4, 3).reshape(P, H, page, dk)
        for name, got in (("k", k), ("v", v)):
            wrong = np.argwhere(got != self.codes[name])
            assert wrong.size == 0, f"codes {name} at {wrong[:4].tolist()} of {len(wrong)}"
        for name, got in (("k", host(cache.k_scale)), ("v", host(cache.v_scale))):
            assert np.array_equal(got.view(np.uint32), self.scales[name].view(np.uint32)), f"scales {name}"


def tokens_of(rng, n, Hkv, dk, spread=True):
    """(n, Hkv, dk), each token and head of a size of its own."""
    x = rng.standard_normal((n, Hkv, dk))
    return (x * np.exp(rng.standard_normal((n, Hkv, 1))) if spread else x).astype(F32)


def columns(x):
    """(n, Hkv, dk) as (Hkv*dk, n)."""
    return np.ascontiguousarray(x.reshape(x.shape[0], -1).T)


def fill(ctx, cache, host_cache, k, v, lens, pos0, tables, skip=0):
    """Both caches get the packed tokens (host: those of sequences whose pages are there)."""
    cu = np.concatenate(([0], np.cumsum(lens))).astype(np.int32)
    cos, sin = tables
    ctx.kv_pages_fill(cache, dev(columns(k)), dev(columns(v)), dev(cu), pos0=dev(np.array(pos0, np.int32)),
                      cos=None if cos is None else dev(cos), sin=None if sin is None else dev(sin))
    for b, n in enumerate(lens):
        rk = np.stack([rotate(k[cu[b] + t], cos, sin, pos0[b] + t) for t in range(n)]) if n else k[:0]
        host_cache.put(b, pos0[b], rk, v[cu[b]:cu[b + 1]])


@pytest.mark.parametrize("dk", [64, 128, 256])
@pytest.mark.parametrize("page,block,lens,pos0", [
    (16, 16, [1], [0]), (16, 16, [100], [0]), (64, 64, [64, 64], [0, 0]), (64, 64, [200, 1, 0, 63, 65], [0, 5, 9, 1, 130]),
    (32, 16, [7, 90, 33], [3, 17, 0]), (128, 32, [1] * 70, list(range(70))), (1024, 64, [130, 127], [63, 64]),
    (64, 32, [0, 0, 300], [0, 1, 31]), (16, 16, [150], [13]), (64, 64, [400, 1, 0, 203, 210], [0, 5, 9, 1, 130]),
    (32, 32, [257], [49]), (128, 32, [0, 0, 500], [0, 1, 31])])
def test_fill(ctx, nnhip, dk, page, block, lens, pos0):
    print(f"fill dk={dk} page={page} block={block} lens={lens[:6]} pos0={pos0[:6]}", flush=True)
    rng = np.random.default_rng(dk + page + block + len(lens))
    Hkv, M = 3, sum(lens)
    c = CacheI8(rng, np.array(lens) + np.array(pos0), Hkv, page, dk, block)
    for b, p in enumerate(pos0):
        c.put(b, 0, tokens_of(rng, p, Hkv, dk), tokens_of(rng, p, Hkv, dk))
    cache = c.on_device(nnhip)
    fill(ctx, cache, c, tokens_of(rng, M, Hkv, dk), tokens_of(rng, M, Hkv, dk), lens, pos0,
         nnhip.rope_table(dk, max(n + p for n, p in zip(lens, pos0))))
    c.check(cache)
    # and every value of every sequence read back
    n = [a + b for a, b in zip(lens, pos0)]
    cu = np.concatenate(([0], np.cumsum(n))).astype(np.int32)
    k, v = ctx.kv_pages_read(cache, dev(cu), sum(n))
    for b in range(len(n)):
        for got, want in zip((host(k), host(v)), c.rows(b, n[b])):
            assert np.array_equal(got[:, cu[b]:cu[b + 1]].T.reshape(n[b], Hkv, dk), want.astype(F32))


def test_fill_grows(ctx, nnhip):
    """Tokens one at a time and in small runs, of sizes that go up and down: every scale and code as the definition says."""
    rng = np.random.default_rng(5)
    Hkv, page, dk, block = 2, 32, 64, 32
    c = CacheI8(rng, [200, 200, 200], Hkv, page, dk, block)
    cache = c.on_device(nnhip)
    pos = [0, 0, 0]
    for step in range(40):
        lens = [int(x) for x in rng.integers(0, 6, 3)]
        if step == 7:
            lens = [31, 33, 1]
        size = 10.0 ** rng.uniform(-3, 3)
        k, v = (tokens_of(rng, sum(lens), Hkv, dk) * F32(size) for _ in range(2))
        if sum(lens):
            fill(ctx, cache, c, k, v, lens, pos, (None, None))
        pos = [p + n for p, n in zip(pos, lens)]
        c.check(cache)


def test_fill_values(ctx, nnhip):
    """Zeros, the smallest and largest magnitudes, ties, NaN and infinities."""
    rng = np.random.default_rng(6)
    Hkv, page, dk, block = 1, 64, 64, 16
    n = 16 * 8
    k, v = tokens_of(rng, n, Hkv, dk, spread=False), tokens_of(rng, n, Hkv, dk, spread=False)
    k[0:16] = 0
    v[16:32] *= F32(1e-40)
    k[32:48] *= F32(1e37)
    v[48:64] = rng.integers(-254, 255, (16, Hkv, dk)).astype(F32) / 2  # halves, with a scale of 1
    v[48, 0, 0] = 127.0
    k[64:80, 0, 3] = np.nan
    v[80, 0, 5] = np.inf
    k[97, 0, 9] = -np.inf
    v[112:128] = F32(-0.0)
    c = CacheI8(rng, [n], Hkv, page, dk, block)
    cache = c.on_device(nnhip)
    fill(ctx, cache, c, k, v, [n], [0], (None, None))
    c.check(cache)
    # a token after an infinity, and an infinity after tokens
    c2 = CacheI8(rng, [20], Hkv, page, dk, block)
    cache = c2.on_device(nnhip)
    for t in range(20):
        x = tokens_of(rng, 1, Hkv, dk)
        if t in (7, 18):
            x[0, 0, 2] = np.inf
        fill(ctx, cache, c2, x, x[..., ::-1].copy(), [1], [t], (None, None))
        c2.check(cache)


def test_fill_leaves_out(ctx, nnhip):
    """Tokens of no sequence, past the table or the rope tables and of pages outside the pool are not written; read gives
    NaN where there is no place and leaves other columns."""
    rng = np.random.default_rng(7)
    Hkv, page, dk, block, M = 2, 16, 64, 16, 90
    c = CacheI8(rng, [40, 40], Hkv, page, dk, block)
    bad = c.table.copy()
    bad[1, 1] = c.codes["k"].shape[0]
    c.put(0, 0, tokens_of(rng, 20, Hkv, dk), tokens_of(rng, 20, Hkv, dk))
    k, v = tokens_of(rng, M, Hkv, dk), tokens_of(rng, M, Hkv, dk)
    cu = dev(np.array([0, 30, 80], np.int32))  # the second ends past the table; 10 columns are no one's
    cos, sin = nnhip.rope_table(dk, 46)
    turned = lambda lo, hi, p: np.stack([rotate(k[m], cos, sin, p + m - lo) for m in range(lo, hi)])  # noqa: E731
    cache = c.on_device(nnhip)
    cache.table.copy_(dev(bad))
    ctx.kv_pages_fill(cache, dev(columns(k)), dev(columns(v)), cu, pos0=dev(np.array([20, 0], np.int32)), cos=dev(cos), sin=dev(sin))
    c.put(0, 20, turned(0, 26, 20), v[0:26])           # up to the end of the tables (46)
    c.put(1, 0, turned(30, 46, 0), v[30:46])           # page 0 of the second
    c.put(1, 32, turned(30, 76, 0)[32:46], v[62:76])   # page 2
    c.check(cache)
    out = [dev(np.full((Hkv * dk, M), 7.0, F32)) for _ in range(2)]
    ctx.kv_pages_read(cache, cu, M, pos0=dev(np.array([20, 0], np.int32)), k=out[0], v=out[1])
    got = host(out[0])
    assert np.all(got[:, 80:] == 7.0) and np.isnan(got[:, 28:30]).all()           # positions 48, 49: past the table
    assert np.isnan(got[:, 46:62]).all() and np.isnan(got[:, 78:80]).all()        # the bad page; past the table
    assert np.isfinite(got[:, :26]).all() and np.isfinite(got[:, 30:46]).all()


@pytest.mark.parametrize("dk,block", [(64, 16), (128, 64), (256, 32)])
def test_fill_alone_and_among_empty_sequences(ctx, nnhip, dk, block):
    """A long prompt behind columns of no one, past a bad page and the end of the rope tables, onto older tokens that it
    outgrows: by windows of positions alone, by columns among empty sequences, the same bits, and the definition's."""
    rng = np.random.default_rng(8 + dk)
    Hkv, page, M, p0, n, rows = 2, 64, 330, 37, 300, 320
    k, v = (tokens_of(rng, M, Hkv, dk) * F32(3.0) for _ in range(2))
    old = [tokens_of(rng, p0, Hkv, dk) for _ in range(2)]
    cos, sin = nnhip.rope_table(dk, rows)
    found = []
    for empty in (0, 5):
        c = CacheI8(np.random.default_rng(9), [p0 + n], Hkv, page, dk, block)
        c.put(0, 0, *old)
        bad = np.repeat(c.table, 1 + empty, 0)
        bad[0, 2] = -1  # positions 128 .. 191
        cache = nnhip.KVPagesI8(*(getattr(c.on_device(nnhip), x) for x in ("k", "v", "k_scale", "v_scale")), dev(bad))
        cu = dev(np.array([20] + [20 + n] * (1 + empty), np.int32))
        ctx.kv_pages_fill(cache, dev(columns(k)), dev(columns(v)), cu, pos0=dev(np.array([p0] + [0] * empty, np.int32)),
                          cos=dev(cos), sin=dev(sin))
        turned = np.stack([rotate(k[20 + i], cos, sin, p0 + i) for i in range(rows - p0)])
        c.put(0, p0, turned[:128 - p0], v[20:20 + 128 - p0])
        c.put(0, 192, turned[192 - p0:], v[20 + 192 - p0:20 + rows - p0])
        c.check(cache)
        found.append([host(x) for x in (cache.k, cache.v, cache.k_scale, cache.v_scale)])
    for a, b in zip(*found):
        assert np.array_equal(a.view(np.uint8), b.view(np.uint8))


def check_decode(ctx, nnhip, B, H, Hkv, dk, page, block, pos, rope=True, cap=0.0, slopes=False, tokens=True, seed=0,
                 len_bound=None, append=True, edit=None, spread=True):
    print(f"decode B={B} H={H} Hkv={Hkv} dk={dk} page={page} block={block} pos={list(pos)[:8]} cap={cap} slopes={slopes} "
          f"tokens={tokens} append={append}", flush=True)
    rng = np.random.default_rng(seed + 1000 * dk + H)
    pos = np.array(pos, np.int32)
    bound = int(pos.max()) + 1 if len_bound is None else len_bound
    c = CacheI8(rng, np.maximum(pos + 1, 0), Hkv, page, dk, block, width=-(-max(bound, int(pos.max()) + 1) // page))
    for b, p in enumerate(pos):
        n = max(int(p) + (0 if append else 1), 0)
        c.put(b, 0, tokens_of(rng, n, Hkv, dk, spread), tokens_of(rng, n, Hkv, dk, spread))
    q = rng.standard_normal((B, H, dk)).astype(F32)
    k, v = tokens_of(rng, B, Hkv, dk), tokens_of(rng, B, Hkv, dk)
    if edit is not None:
        edit(c, q, k, v)
    cos, sin = nnhip.rope_table(dk, bound) if rope else (None, None)
    sl = (2.0 ** (-8.0 * (np.arange(H) + 1) / H)).astype(F32) if slopes else None
    scale = float(F32(1 / math.sqrt(dk)))
    cache = c.on_device(nnhip)
    lay = (lambda x: x.reshape(B, -1)) if tokens else (lambda x: x.reshape(B, -1).T)
    new = (dev(lay(k)), dev(lay(v))) if append else (None, None)
    out = ctx.attention_pages_decode(cache, dev(lay(q)), *new, H, dev(pos), bound, scale,
                                     cos=None if cos is None else dev(cos), sin=None if sin is None else dev(sin),
                                     softcap=cap, slopes=None if sl is None else dev(sl), tokens=tokens)
    out = host(out).astype(np.float64)
    out = (out if tokens else out.T).reshape(B, H, dk)
    worst = 0.0
    for b, p in enumerate(pos):
        if p < 0:
            assert np.all(out[b] == 0)
            continue
        if p >= bound:
            assert np.isnan(out[b]).all()
            continue
        if append:
            c.put(b, int(p), rotate(k[b], cos, sin, p)[None], v[b][None])
        K, V = c.rows(b, p + 1)
        at = np.arange(p + 1)
        qr = rotate(q[b].astype(np.float64), None if cos is None else cos.astype(np.float64),
                    None if sin is None else sin.astype(np.float64), p)
        for h in range(H):
            g = h // (H // Hkv)
            if not (np.isfinite(K[:, g]).all() and np.isfinite(V[:, g]).all() and np.isfinite(qr[h]).all()):
                assert np.isnan(out[b, h]).all()
                continue
            want, tol = attend64(qr[h], K[:, g], V[:, g], scale, cap, 0.0 if sl is None else float(sl[h]), at - p, at >= 0)
            tol = tol + own_bound(qr[h], K[:, g], V[:, g], scale, p + 1, 2.0 ** -26)
            err = np.abs(out[b, h] - want)
            worst = max(worst, float(np.max(err / tol)))
    print(f"  worst {worst:.3f} of the bound", flush=True)
    assert worst <= 1.0
    c.check(cache)
    return c, cache, out


def own_bound(q, K, V, scale, n, weights):
    """What the kernels' parts leave out on top of attend64's bound (at the top of the file)."""
    delta = len(q) * 2.0 ** -31 * float(np.max(np.abs(q))) * float(np.max(np.abs(K))) * abs(scale)
    top = float(np.max(np.abs(V)))
    return 2 * delta * top + 4 * math.sqrt(n) * weights * top + 1e-30


@pytest.mark.parametrize("case", [
    dict(B=1, H=1, Hkv=1, dk=64, page=16, block=16, pos=[0]),
    dict(B=1, H=20, Hkv=5, dk=128, page=16, block=16, pos=[99]),
    dict(B=4, H=20, Hkv=5, dk=128, page=64, block=64, pos=[0, 63, 64, 200]),
    dict(B=5, H=16, Hkv=2, dk=64, page=32, block=16, pos=[-1, 15, 16, 1030, -7], cap=20.0, slopes=True),
    dict(B=3, H=8, Hkv=1, dk=256, page=64, block=32, pos=[31, 32, 700], slopes=True),
    dict(B=2, H=7, Hkv=7, dk=128, page=128, block=64, pos=[127, 128], tokens=False),
    dict(B=2, H=10, Hkv=2, dk=128, page=16, block=16, pos=[300, 47], cap=50.0, tokens=False),
    dict(B=2, H=16, Hkv=1, dk=64, page=16, block=16, pos=[77, 300]),
    dict(B=2, H=24, Hkv=2, dk=128, page=64, block=32, pos=[129, 400], rope=False),
    dict(B=2, H=16, Hkv=1, dk=256, page=64, block=32, pos=[129, 255]),
    dict(B=3, H=6, Hkv=2, dk=64, page=1024, block=64, pos=[5, 2000, 1023]),
    dict(B=2, H=4, Hkv=2, dk=256, page=32, block=16, pos=[300, 511], cap=30.0),
    dict(B=33, H=4, Hkv=4, dk=256, page=128, block=64, pos=[30 * b + 3 for b in range(33)]),
    dict(B=2, H=4, Hkv=1, dk=128, page=64, block=64, pos=[5000, 12345]),
    dict(B=17, H=4, Hkv=2, dk=64, page=16, block=16, pos=list(range(17)), slopes=True),
    dict(B=3, H=20, Hkv=5, dk=128, page=64, block=32, pos=[99, 300, -1], append=False),
    dict(B=2, H=16, Hkv=1, dk=64, page=16, block=16, pos=[0, 130], append=False, cap=5.0),
    dict(B=2, H=4, Hkv=1, dk=64, page=16, block=16, pos=[9, 100], len_bound=60, append=False),
])
def test_decode(ctx, nnhip, case):
    check_decode(ctx, nnhip, **case)


def test_decode_edges(ctx, nnhip):
    """Infinities, NaN and zeros: in the query of one head, in the cache, in the new token; noise behind the last position."""
    base = dict(B=3, H=8, Hkv=2, dk=64, page=16, block=16, pos=[40, 200, 15], rope=False)

    def query(c, q, k, v):
        q[0, 3, 5] = np.inf
        q[1, 6, 0] = np.nan
        q[2, 1] = 0.0

    check_decode(ctx, nnhip, **base, edit=query)

    def held(c, q, k, v):
        c.scales["k"][c.table[0, 1], 0, 0] = np.inf
        c.codes["k"][c.table[0, 1], 0, 0:16] = 0
        c.scales["v"][c.table[1, 4], 1, 0] = np.nan
        c.codes["v"][c.table[1, 4], 1, 0:16] = 0

    check_decode(ctx, nnhip, **base, edit=held)

    def new(c, q, k, v):
        k[0, 0, 7] = np.nan   # left out: a code of 0
        v[1, 1, 7] = np.inf   # its block stands for NaN
        v[2] = 0.0

    check_decode(ctx, nnhip, **base, edit=new)

    def zeros(c, q, k, v):
        for x in "kv":
            for b in range(3):
                for i in range(-(-(base["pos"][b] + 1) // 16)):
                    c.scales[x][c.table[b, i], :, 0] = 0.0
                    c.codes[x][c.table[b, i]] = 0
        k[:] = 0.0
        v[:] = 0.0

    _, _, out = check_decode(ctx, nnhip, **base, edit=zeros)
    assert np.all(out == 0)

    def sizes(c, q, k, v):  # scales of values 2^40 apart from block to block, large and small queries
        for b in range(3):
            for i in range(-(-(base["pos"][b] + 1) // 16)):
                c.scales["v"][c.table[b, i], :, 0] *= F32(2.0 ** (20 if i % 2 else -20))
        q[0] *= F32(1e-20)
        q[1] *= F32(8.0)

    check_decode(ctx, nnhip, **base, edit=sizes)


def test_decode_bad_pages(ctx, nnhip):
    """A page outside the pool among the positions: NaN for that sequence, nothing written there; others as they were."""
    rng = np.random.default_rng(9)
    H, Hkv, dk, page, block = 4, 2, 64, 16, 16
    pos = np.array([40, 40, 33], np.int32)
    for at, bad in ((0, -1), (1, 100000), (2, 2 ** 31 - 1)):
        c = CacheI8(rng, pos + 1, Hkv, page, dk, block)
        for b, p in enumerate(pos):
            c.put(b, 0, tokens_of(rng, p, Hkv, dk), tokens_of(rng, p, Hkv, dk))
        cache = c.on_device(nnhip)
        t = c.table.copy()
        t[1, at] = bad
        cache.table.copy_(dev(t))
        q, k, v = (rng.standard_normal((3, h * dk)).astype(F32) for h in (H, Hkv, Hkv))
        out = host(ctx.attention_pages_decode(cache, dev(q), dev(k), dev(v), H, dev(pos), 41, 0.125, tokens=True))
        assert np.isnan(out[1]).all() and np.isfinite(out[[0, 2]]).all()
        for b in (0, 2) if at == 2 else (0, 1, 2):
            c.put(b, int(pos[b]), k[b].reshape(1, Hkv, dk), v[b].reshape(1, Hkv, dk))
        c.check(cache)


def prompt_case(ctx, nnhip, lens, pos0, H, Hkv, dk, page, block, rope=True, cap=0.0, slopes=False, prefix=None, distance=False,
                seed=0, edit=None, t_bound=None, stride=1, q_size=1.0):
    print(f"prompt lens={lens} pos0={pos0} H={H} Hkv={Hkv} dk={dk} page={page} block={block} cap={cap} slopes={slopes} "
          f"prefix={prefix} distance={distance}", flush=True)
    rng = np.random.default_rng(seed + dk + H)
    B, M = len(lens), sum(lens)
    ends = [n + p for n, p in zip(lens, pos0)]
    c = CacheI8(rng, ends, Hkv, page, dk, block)
    for b in range(B):
        c.put(b, 0, tokens_of(rng, ends[b], Hkv, dk), tokens_of(rng, ends[b], Hkv, dk))
    q = (q_size * rng.standard_normal((M, H, dk))).astype(F32)
    if edit is not None:
        edit(c, q)
    cu = np.concatenate(([0], np.cumsum(lens))).astype(np.int32)
    cos, sin = nnhip.rope_table(dk, max(ends)) if rope else (None, None)
    sl = (2.0 ** (-8.0 * (np.arange(H) + 1) / H)).astype(F32) if slopes else None
    scale = float(F32(1 / math.sqrt(dk)))
    cache = c.on_device(nnhip)
    pre = None if prefix is None else np.array(prefix, np.int32)
    out = ctx.attention_pages_prefill(cache, dev(columns(q)), dev(cu), max(lens) if t_bound is None else t_bound, H, scale,
                                      pos0=dev(np.array(pos0, np.int32)), cos=None if cos is None else dev(cos),
                                      sin=None if sin is None else dev(sin), softcap=cap,
                                      slopes=None if sl is None else dev(sl), prefix=None if pre is None else dev(pre),
                                      distance=distance)
    out = host(out).T.reshape(M, H, dk).astype(np.float64)
    worst = 0.0
    for b in range(B):
        K, V = c.rows(b, ends[b])
        at = np.arange(ends[b])
        for t in list(range(0, lens[b], stride)) + ([lens[b] - 1] if lens[b] else []):
            p = pos0[b] + t
            qr = rotate(q[cu[b] + t].astype(np.float64), None if cos is None else cos.astype(np.float64),
                        None if sin is None else sin.astype(np.float64), p)
            see = (at <= p) | (at < (0 if pre is None else pre[b]))
            for h in range(H):
                g = h // (H // Hkv)
                if not (np.isfinite(K[see, g]).all() and np.isfinite(V[see, g]).all() and np.isfinite(qr[h]).all()):
                    assert np.isnan(out[cu[b] + t, h]).all(), (b, t, h)
                    continue
                Ks, Vs = K[see, g], V[see, g]
                dist = (at - p)[see]
                want, tol = attend64(qr[h], Ks, Vs, scale, cap, 0.0 if sl is None else float(sl[h]),
                                     -np.abs(dist) if distance else dist, np.ones(len(dist), bool))
                tol = tol + own_bound(qr[h], Ks, Vs, scale, len(dist), 2.0 ** -24) + 2.0 ** -22 * np.max(np.abs(Vs))
                worst = max(worst, float(np.max(np.abs(out[cu[b] + t, h] - want) / tol)))
    print(f"  worst {worst:.3f} of the bound", flush=True)
    assert worst <= 1.0
    return out


@pytest.mark.parametrize("case", [
    dict(lens=[1], pos0=[0], H=1, Hkv=1, dk=64, page=16, block=16),
    dict(lens=[5, 40, 17], pos0=[200, 0, 63], H=20, Hkv=5, dk=128, page=16, block=16, stride=3),
    dict(lens=[33, 0, 64, 1], pos0=[0, 7, 1, 130], H=8, Hkv=8, dk=64, page=64, block=32, stride=5),
    dict(lens=[150, 40], pos0=[0, 500], H=16, Hkv=2, dk=64, page=32, block=32, cap=50.0, slopes=True, prefix=[60, 520], stride=11),
    dict(lens=[100, 300], pos0=[40, 0], H=8, Hkv=1, dk=128, page=64, block=64, slopes=True, prefix=[70, 200], distance=True, stride=17),
    dict(lens=[70], pos0=[0], H=7, Hkv=7, dk=128, page=128, block=64, rope=False, stride=7),
    dict(lens=[90, 31], pos0=[16, 1], H=6, Hkv=2, dk=128, page=16, block=16, cap=3.0, stride=7),
    dict(lens=[600, 200, 333], pos0=[0, 1500, 77], H=4, Hkv=1, dk=128, page=64, block=64, stride=61),
    dict(lens=[1000], pos0=[3000], H=2, Hkv=2, dk=64, page=32, block=16, slopes=True, stride=97),
])
def test_prompt(ctx, nnhip, case):
    prompt_case(ctx, nnhip, **case)


@pytest.mark.parametrize("case", [
    dict(lens=[1, 32, 33, 64], pos0=[600, 1000, 90, 64], H=20, Hkv=5, dk=128, page=64, block=32, stride=13),
    dict(lens=[20], pos0=[3000], H=4, Hkv=1, dk=128, page=32, block=16, cap=20.0, stride=6),
    dict(lens=[64, 65, 3], pos0=[0, 333, 2000], H=16, Hkv=8, dk=128, page=16, block=16, rope=False, stride=21),
    dict(lens=[128, 129, 200, 2], pos0=[100, 0, 31, 700], H=4, Hkv=4, dk=64, page=64, block=64, cap=5.0, slopes=True,
         prefix=[150, 129, 0, 300], distance=True, stride=29),
    dict(lens=[30, 10], pos0=[0, 40], H=2, Hkv=2, dk=64, page=16, block=16, slopes=True, prefix=[30, 45], stride=4),
    dict(lens=[b % 4 for b in range(70)], pos0=[37 * b % 190 for b in range(70)], H=4, Hkv=1, dk=64, page=32, block=32),
    dict(lens=[256], pos0=[64], H=8, Hkv=1, dk=128, page=64, block=64, cap=30.0, slopes=True, stride=51),
])
def test_prompt_few_queries(ctx, nnhip, case):
    """At most half of a work-group's queries: its waves share the keys."""
    prompt_case(ctx, nnhip, **case)


def test_prompt_few_queries_edges(ctx, nnhip):
    """Scales that differ by any factor from block to block, infinite ones in sight and behind, zeros, over the waves' halves."""
    base = dict(lens=[20, 9], pos0=[200, 330], H=4, Hkv=1, dk=128, page=32, block=16, stride=3)

    def sizes(c, q):
        for b, n in ((0, 220), (1, 339)):
            for i in range(-(-n // 16)):
                at = (c.table[b, i // 2], slice(None), i % 2)
                c.scales["v"][at] *= F32(2.0 ** (30 if i % 4 == 1 else -30 if i % 4 == 2 else 0))
                c.scales["k"][at] *= F32(2.0 ** (1 if i % 3 else -10))

    prompt_case(ctx, nnhip, **base, edit=sizes)

    def odd(c, q):
        c.scales["v"][c.table[0, 6], 0, 1] = np.inf   # positions 208 .. 223: of some queries
        c.scales["k"][c.table[1, 10], 0, 1] = np.nan  # 336 .. 351
        for i in range(0, 10, 2):
            c.scales["v"][c.table[1, i], 0] = 0.0
            c.codes["v"][c.table[1, i]] = 0
        q[25, 2, 7] = np.inf

    prompt_case(ctx, nnhip, **base, edit=odd)


@pytest.mark.parametrize("cap", [0.0, 20.0])
@pytest.mark.parametrize("dk", [64, 128])
def test_prompt_whole_tiles_edges(ctx, nnhip, dk, cap):
    """Tiles that every query sees: infinities, NaN and zeros among queries and scales, scales that differ by any factor within
    a tile and from tile to tile."""
    base = dict(lens=[40, 33], pos0=[260, 192], H=8, Hkv=1, dk=dk, page=32, block=16, cap=cap, slopes=cap > 0, stride=5)

    def odd(c, q):
        c.scales["k"][c.table[0, 3], 0, 1] = np.inf   # positions 112 .. 127 of the first
        c.codes["k"][c.table[0, 3], 0, 16:] = 0
        q[45, 2, 7] = np.inf
        q[60, 1, 0] = np.nan
        q[40] = 0.0

    prompt_case(ctx, nnhip, **base, edit=odd)

    def values(c, q):
        c.scales["v"][c.table[0, 1], 0, 0] = np.nan
        for i in range(0, 6, 2):
            c.scales["v"][c.table[1, i], 0] = 0.0
            c.codes["v"][c.table[1, i]] = 0

    prompt_case(ctx, nnhip, **base, edit=values)

    def sizes(c, q):
        for b, n in ((0, 300), (1, 225)):
            for i in range(-(-n // 16)):
                at = (c.table[b, i // 2], slice(None), i % 2)
                c.scales["v"][at] *= F32(2.0 ** (0, 3, -7, 9, 20, -20, 1, 0, 40, 41, 39, 45)[i % 12])
                c.scales["k"][at] *= F32(2.0 ** (1, 0, -10)[i % 3])
        q[:20] *= F32(1e-30)

    prompt_case(ctx, nnhip, **base, edit=sizes)


def test_prompt_edges(ctx, nnhip):
    base = dict(lens=[60, 50], pos0=[0, 100], H=4, Hkv=2, dk=64, page=16, block=16, rope=False)

    def query(c, q):
        q[3, 1, 5] = np.inf
        q[70, 2, 0] = np.nan
        q[5] = 0.0

    prompt_case(ctx, nnhip, **base, edit=query)

    def held(c, q):
        # blocks that some queries see and others do not, and one in every query's past
        c.scales["k"][c.table[0, 2], 0, 0] = np.inf
        c.codes["k"][c.table[0, 2], 0] = 0
        c.scales["v"][c.table[0, 1], 1, 0] = np.nan
        c.scales["v"][c.table[1, 8], 0, 0] = np.inf
        c.scales["k"][c.table[1, 0], 1, 0] = np.nan

    prompt_case(ctx, nnhip, **base, edit=held)

    def zeros(c, q):
        for x in "kv":
            for b, n in ((0, 4), (1, 10)):
                for i in range(0, n, 2):
                    c.scales[x][c.table[b, i], :, 0] = 0.0
                    c.codes[x][c.table[b, i]] = 0

    prompt_case(ctx, nnhip, **base, edit=zeros)

    def sizes(c, q):
        for b, n in ((0, 4), (1, 10)):
            for i in range(n):
                c.scales["v"][c.table[b, i], :, 0] *= F32(2.0 ** (20 if i % 2 else -20))
                c.scales["k"][c.table[b, i], :, 0] *= F32(2.0 ** (1 if i % 3 else -10))
        q[:30] *= F32(1e-30)

    prompt_case(ctx, nnhip, **base, edit=sizes)
    prompt_case(ctx, nnhip, **dict(base, dk=128, block=16, page=32), edit=lambda c, q: q.__imul__(F32(20.0)))


def test_prompt_bad_sequences(ctx, nnhip):
    """As over f32 pages: sequences that do not fit get NaN, a page outside the pool shows in the queries that see it."""
    rng = np.random.default_rng(27)
    H, Hkv, dk, page = 2, 1, 64, 16
    lens = [40, 40, 40, 20]
    c = CacheI8(rng, lens, Hkv, page, dk, 16)
    for b, n in enumerate(lens):
        c.put(b, 0, tokens_of(rng, n, Hkv, dk), tokens_of(rng, n, Hkv, dk))
    M = 140
    q = dev(rng.standard_normal((H * dk, M)).astype(F32))
    cu = np.concatenate(([0], np.cumsum(lens))).astype(np.int32)

    def run(cu=cu, t_bound=40, pos0=None, table=None):
        cache = c.on_device(nnhip)
        if table is not None:
            cache.table.copy_(dev(table))
        return host(ctx.attention_pages_prefill(cache, q, dev(np.array(cu, np.int32)), t_bound, H, 0.125,
                                                pos0=None if pos0 is None else dev(np.array(pos0, np.int32))))

    ref = run()
    assert np.all(np.isfinite(ref))
    got = run(t_bound=39)
    assert np.isnan(got[:, :120]).all() and np.array_equal(got[:, 120:], ref[:, 120:])
    got = run(pos0=[0, 9, -1, 0])  # the second ends past its table's 48 positions
    assert np.array_equal(got[:, :40], ref[:, :40]) and np.isnan(got[:, 40:120]).all()
    for bad in (-1, c.codes["k"].shape[0], 2 ** 31 - 1):
        t = c.table.copy()
        t[1, 2] = bad  # positions 32 .. 39
        t[3, 2] = bad  # past its length
        got = run(table=t)
        assert np.isnan(got[:, 72:80]).all()
        keep = [m for m in range(M) if not 40 <= m < 80]
        assert np.array_equal(got[:, keep], ref[:, keep])
    # columns of no sequence are left
    out = dev(np.full((H * dk, M), 7.0, F32))
    ctx.attention_pages_prefill(c.on_device(nnhip), q, dev(np.array([0, 40, 80], np.int32)), 40, H, 0.125, out=out)
    assert np.all(host(out)[:, 80:] == 7.0) and np.array_equal(host(out)[:, :40], ref[:, :40])


@pytest.mark.parametrize("decode", [True, False])
def test_error_in_norm(ctx, nnhip, decode):
    """Outputs for normal inputs against 64 bits, in norm. A score of about 1 is off by its sum's roundings (dk = 128 products
    of values about 1 over sqrt(dk): under 2 u), its scaling and the exponential by 4 u, its weight's parts by 1 u; sums of n
    weighted values by 0.5 u sqrt(steps) of independent roundings, a step for 8 positions: 8 u + sqrt(n / 8) u / 2 with a margin of 2."""
    import torch
    rng = np.random.default_rng(70)
    n, H, Hkv, dk, page = 3000, 8, 2, 128, 64
    c = CacheI8(rng, [n], Hkv, page, dk, 32)
    c.put(0, 0, rng.standard_normal((n, Hkv, dk)).astype(F32), rng.standard_normal((n, Hkv, dk)).astype(F32))
    T = 1 if decode else 64
    q = rng.standard_normal((T, H, dk)).astype(F32)
    scale = float(F32(1 / math.sqrt(dk)))
    cache = c.on_device(nnhip)
    if decode:
        out = host(ctx.attention_pages_decode(cache, dev(columns(q)), None, None, H, dev(np.array([n - 1], np.int32)), n, scale))
    else:
        out = host(ctx.attention_pages_prefill(cache, dev(columns(q)), dev(np.array([0, T], np.int32)), T, H, scale,
                                               pos0=dev(np.array([n - T], np.int32))))
    out = out.T.reshape(T, H, dk).astype(np.float64)
    K, V = c.rows(0, n)
    err = norm = 0.0
    for t in range(T):
        m = n - T + t + 1
        for h in range(H):
            x = K[:m, h // 4] @ q[t, h].astype(np.float64) * scale
            p = np.exp(x - x.max())
            want = p @ V[:m, h // 4] / p.sum()
            err += float(np.sum((out[t, h] - want) ** 2))
            norm += float(np.sum(want ** 2))
    rel = math.sqrt(err / norm)
    print(f"  {rel / U:.2f} u", flush=True)
    assert rel <= (8 + 0.5 * math.sqrt(n / 8)) * U * 2


def test_captured_and_streams(nnhip):
    """Fill, decode and prompt captured on a stream of their own and replayed between eager calls of other sizes, the lengths
    changing on the device: each replay gives what eager calls give, in both pools and outputs."""
    import torch
    ctx = nnhip.Context(0)
    rng = np.random.default_rng(71)
    H, Hkv, dk, page = 8, 2, 64, 16
    lens = [700, 500]
    c = CacheI8(rng, lens, Hkv, page, dk, 16)
    for b, n in enumerate(lens):
        c.put(b, 0, tokens_of(rng, n, Hkv, dk), tokens_of(rng, n, Hkv, dk))
    state = [dev(rng.standard_normal(s).astype(F32)) for s in ((H * dk, 2), (Hkv * dk, 2), (Hkv * dk, 2), (H * dk, 90),
                                                               (Hkv * dk, 90), (Hkv * dk, 90))]
    side = torch.cuda.Stream()
    found = []
    for captured in (False, True):
        cache = c.on_device(nnhip)
        pos, cu, pos0 = dev(np.array([99, 300], np.int32)), dev(np.array([0, 40, 90], np.int32)), dev(np.array([100, 301], np.int32))
        out, prompt = torch.zeros(H * dk, 2, device="cuda"), torch.zeros(H * dk, 90, device="cuda")

        def call():
            ctx.attention_pages_decode(cache, state[0], state[1], state[2], H, pos, 700, 0.125, out=out)
            ctx.kv_pages_fill(cache, state[4], state[5], cu, pos0=pos0)
            ctx.attention_pages_prefill(cache, state[3], cu, 90, H, 0.125, pos0=pos0, out=prompt)

        with torch.cuda.stream(side):
            call()
        torch.cuda.synchronize()
        trace = []
        if captured:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                call()
        for p, split, p0 in (([150, 360], 50, [151, 361]), ([5, -1], 0, [6, 0]), ([600, 400], 90, [601, 2]), ([250, 77], 17, [251, 78])):
            pos.copy_(dev(np.array(p, np.int32)))
            cu.copy_(dev(np.array([0, split, 90], np.int32)))
            pos0.copy_(dev(np.array(p0, np.int32)))
            torch.cuda.synchronize()
            if captured:
                g.replay()
            else:
                with torch.cuda.stream(side):
                    call()
            torch.cuda.synchronize()
            ctx.attention_pages_decode(c.on_device(nnhip), state[0], None, None, H, dev(np.array([40, 20], np.int32)), 41, 0.1)
            trace += [host(x).copy() for x in (out, prompt, cache.k, cache.v, cache.k_scale, cache.v_scale)]
        found.append(trace)
    for a, b in zip(*found):
        assert np.array_equal(a, b, equal_nan=a.dtype.kind == "f")
    ctx.close()


def test_refusals(ctx, nnhip):
    t = dev(np.zeros((2, 4), np.int32))
    cache = nnhip.KVPagesI8.empty(4, 2, 16, 64, 16, t)
    q, k = dev(np.zeros((256, 2), F32)), dev(np.zeros((128, 2), F32))
    cu, pos = dev(np.array([0, 1, 2], np.int32)), dev(np.zeros(2, np.int32))
    with pytest.raises(nnhip.NNHipError, match="k and v"):
        ctx.attention_pages_decode(cache, q, k, None, 4, pos, 8, 0.1)
    with pytest.raises(nnhip.NNHipError, match="len_bound"):
        ctx.attention_pages_decode(cache, q, k, k, 4, pos, 65, 0.1)
    with pytest.raises(nnhip.NNHipError, match="multiple of Hkv"):
        ctx.attention_pages_decode(cache, dev(np.zeros((192, 2), F32)), k, k, 3, pos, 8, 0.1)
    with pytest.raises(nnhip.NNHipError, match="softcap"):
        ctx.attention_pages_prefill(cache, q, cu, 1, 4, 0.1, softcap=-1.0)
    with pytest.raises(nnhip.NNHipError, match="t_bound"):
        ctx.attention_pages_prefill(cache, q, cu, 3, 4, 0.1)
    with pytest.raises(nnhip.NNHipError, match="dtype"):
        ctx.kv_pages_fill(cache, k.half(), k, cu)
    with pytest.raises(nnhip.NNHipError, match="shape"):
        ctx.kv_pages_read(cache, cu, 5, k=k)
    with pytest.raises(nnhip.NNHipError, match="KVPagesI8"):
        pool = dev(np.zeros((4, 2, 16, 64), F32))
        ctx.kv_pages_read(nnhip.KVPages(pool, pool.clone(), t), cu, 2)
    with pytest.raises(nnhip.NNHipError, match="null"):
        pool = dev(np.zeros((4, 2, 16, 64), F32))
        ctx.attention_pages_decode(nnhip.KVPages(pool, pool.clone(), t), q, None, None, 4, pos, 8, 0.1)
    wide = nnhip.KVPagesI8.empty(4, 1, 32, 256, 16, t)
    with pytest.raises(nnhip.NNHipError, match="64 or 128"):
        ctx.attention_pages_prefill(wide, dev(np.zeros((256, 2), F32)), cu, 1, 1, 0.1)
    for page, dk, block, what in ((128, 64, 128, "block"), (16, 48, 16, "dk must be"), (48, 64, 16, "power of two"), (2048, 64, 16, "power of two")):
        odd = nnhip.KVPagesI8.empty(2, 1, page, dk, block, t)
        with pytest.raises(nnhip.NNHipError, match=what):
            ctx.kv_pages_fill(odd, dev(np.zeros((dk, 2), F32)), dev(np.zeros((dk, 2), F32)), cu)
    # nothing to do
    ctx.kv_pages_fill(cache, dev(np.zeros((128, 0), F32)), dev(np.zeros((128, 0), F32)), dev(np.zeros(3, np.int32)))
    assert ctx.kv_pages_read(cache, dev(np.zeros(1, np.int32)), 2)[0].shape == (128, 2)


def test_rope_tables_without_rows(ctx, nnhip):
    """No position has a place then: nothing is written, and nothing is read behind the tables' beginning."""
    t = dev(np.array([[1]], np.int32))
    cache = nnhip.KVPagesI8.empty(2, 1, 16, 64, 16, t)
    x, cos, cu = dev(np.ones((64, 9), F32)), dev(np.ones((1, 32), F32)), dev(np.array([0, 9], np.int32))
    assert nnhip.lib().nnhip_kv_pages_fill_i8(ctx.h, cache.ref, x.data_ptr(), x.data_ptr(), 9, cu.data_ptr(), None, 1,
                                              cos.data_ptr(), cos.data_ptr(), 0) == 0
    ctx.sync()
    assert not host(cache.k).any() and not host(cache.k_scale).any()
    with pytest.raises(nnhip.NNHipError, match="rope tables are empty"):
        ctx.qk_norm_rope(x, None, 64, 1e-5, pos=dev(np.zeros(9, np.int32)), cos=cos[:0], sin=cos[:0])


def everything(ctx, cache, k, v, cu, q, pos, H, max_len):
    """A fill, the values read back, attention of the prompts and of a further token."""
    M = k.shape[1]
    ctx.kv_pages_fill(cache, k, v, cu)
    prompt = ctx.attention_pages_prefill(cache, q, cu, M, H, 0.1)
    B = cu.shape[0] - 1
    first = q[:, :B].contiguous()
    one = ctx.attention_pages_decode(cache, first, k[:, :B].contiguous(), v[:, :B].contiguous(), H, pos, max_len, 0.1)
    return [prompt, one, *ctx.kv_pages_read(cache, cu, M)]


@pytest.mark.parametrize("dk", [64, 128])
def test_large_pool(ctx, nnhip, dk):
    """Pages past 2^31 bytes of a pool: as in a small one."""
    import torch
    rng = np.random.default_rng(90)
    H, Hkv, page, lens = 8, 4, 128, [300, 1500, 70]
    need = [-(-(n + 1) // page) for n in lens]
    total = (2 ** 31 + 2 ** 28) // (Hkv * page * dk)
    cu = dev(np.concatenate(([0], np.cumsum(lens))).astype(np.int32))
    k, v, q = (dev(rng.standard_normal((h * dk, sum(lens))).astype(F32)) for h in (Hkv, Hkv, H))
    pos = dev(np.array(lens, np.int32))
    found = []
    for pages in (sum(need), total):
        table = np.full((3, max(need)), -1, np.int32)
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = pages - 1 - at - np.arange(n)  # from the pool's end
            at += n
        cache = nnhip.KVPagesI8.empty(pages, Hkv, page, dk, 32, dev(table))
        found.append([host(x) for x in everything(ctx, cache, k, v, cu, q, pos, H, max(lens) + 1)])
        del cache
    torch.cuda.empty_cache()
    for a, b in zip(*found):
        assert np.isfinite(a).all() and np.array_equal(a, b)


def test_two_streams_at_once(nnhip):
    """Calls of unlike sizes on two streams, each over a cache of its own, with records in scratch of their own: as alone."""
    import torch
    ctx = nnhip.Context(0)
    rng = np.random.default_rng(91)
    H, Hkv, dk, page = 8, 2, 128, 32
    sets = []
    for lens in ([1800, 40, 700], [90, 2500]):
        need = [-(-(n + 1) // page) for n in lens]
        table = np.zeros((len(lens), max(need)), np.int32)
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = at + np.arange(n)
            at += n
        cu = dev(np.concatenate(([0], np.cumsum(lens))).astype(np.int32))
        k, v, q = (dev(rng.standard_normal((h * dk, sum(lens))).astype(F32)) for h in (Hkv, Hkv, H))
        cache = nnhip.KVPagesI8.empty(at, Hkv, page, dk, 16, dev(table))
        sets.append((cache, k, v, cu, q, dev(np.array(lens, np.int32)), H, max(lens) + 1))
    alone = [[host(x) for x in everything(ctx, *s)] for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for _ in range(5):
        outs = [[], []]
        for _ in range(3):
            for i, s in enumerate(sets):
                with torch.cuda.stream(streams[i]):
                    outs[i].append(everything(ctx, *s))
        torch.cuda.synchronize()
        for i in range(2):
            for got in outs[i]:
                for a, b in zip(alone[i], got):
                    assert np.array_equal(a, host(b))
    ctx.close()


def test_derived_handle(ctx, nnhip):
    """A class made from KVPagesI8 is one."""
    class Mine(nnhip.KVPagesI8):
        pass

    found = []
    for cls in (nnhip.KVPagesI8, Mine):
        cache = cls.empty(8, 2, 16, 64, 16, dev(np.arange(8, dtype=np.int32).reshape(2, 4)))
        r = np.random.default_rng(93)
        k, v, q = (dev(r.standard_normal((h * 64, 50)).astype(F32)) for h in (2, 2, 4))
        cu = dev(np.array([0, 20, 50], np.int32))
        found.append([host(x) for x in everything(ctx, cache, k, v, cu, q, dev(np.array([20, 30], np.int32)), 4, 40)])
    for a, b in zip(*found):
        assert np.array_equal(a, b)
