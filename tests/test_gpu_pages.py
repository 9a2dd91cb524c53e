"""The paged KV cache on the GPU: its fill from packed prompts and the attention of one new token per
sequence, against evaluations in 64 bits.

What the cache stores is compared bit for bit. Attention outputs are held to a bound of their own
roundings (attention_bound): with u = 2^-24, a score is a sum of dk rounded products of rotated
queries (2 roundings each), so it is off by about sqrt(dk) u of its largest partial sums; at four
deviations, 4 sqrt(dk + 8) u sum|q||K| |scale|. The cap, the bias and the change to log2 add a few
roundings of the score itself. A relative change e of every weight moves an output by at most 2 e
sum p|v|; the sums over n positions add 4 sqrt(n) u and the joins of partial sums a constant."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def host(t):
    return t.cpu().numpy()


def same(a, b):
    """Equal bits but for NaN's payload."""
    w = {2: np.uint16, 4: np.uint32}[a.dtype.itemsize]
    n = np.isnan(a)
    return a.shape == b.shape and np.array_equal(n, np.isnan(b)) and np.array_equal(a[~n].view(w), b[~n].view(w))


def rotate(x, cos, sin, p):
    """x (heads, dk) at position p as the cache rotates it: rounded products, a rounded sum."""
    if cos is None:
        return x.copy()
    h = x.shape[-1] // 2
    a, b = x[..., :h], x[..., h:]
    return np.concatenate((a * cos[p] + (-b) * sin[p], b * cos[p] + a * sin[p]), -1)


class Cache:
    """A paged cache on the host: sequences of the given lengths at pages of their own, NaN elsewhere."""

    def __init__(self, rng, lens, Hkv, page, dk, f16, extra=3, width=None):
        need = [-(-int(n) // page) for n in lens]
        self.page, self.dt = page, np.float16 if f16 else np.float32
        total = sum(need) + extra
        places = rng.permutation(total)[:sum(need)].astype(np.int32)
        self.table = np.full((len(lens), max(1, max(need)) if width is None else width), -1, np.int32)
        self.k = np.full((total, Hkv, page, dk), np.nan, self.dt)
        self.v = np.full((total, Hkv, page, dk), np.nan, self.dt)
        at = 0
        for b, n in enumerate(lens):
            self.table[b, :need[b]] = places[at:at + need[b]]
            at += need[b]
            for t in range(int(n)):
                self.set(b, t, rng.standard_normal((Hkv, dk)), rng.standard_normal((Hkv, dk)))

    def set(self, b, t, k, v):
        i, s = self.table[b, t // self.page], t % self.page
        self.k[i, :, s], self.v[i, :, s] = k.astype(np.float32).astype(self.dt), v.astype(np.float32).astype(self.dt)

    def rows(self, b, n):
        i, s = self.table[b, np.arange(n) // self.page], np.arange(n) % self.page
        return self.k[i, :, s].astype(np.float64), self.v[i, :, s].astype(np.float64)  # (n, Hkv, dk)

    def on_device(self, nnhip):
        return nnhip.KVPages(dev(self.k), dev(self.v), dev(self.table))


def attend64(q, K, V, scale, cap, slope, dist, see):
    """One query's output over K, V (n, dk) and the bound on its f32 evaluation (at the top of the file)."""
    with np.errstate(invalid="ignore"):
        s = (K @ q) * scale
        mag = 4 * math.sqrt(len(q) + 8) * float(np.max((np.abs(K) @ np.abs(q))[see])) * abs(scale)
        if cap > 0:
            s = cap * np.tanh(s / cap)
        s = s + slope * dist
    s = np.where(see, s, -np.inf)
    p = np.exp(s - s.max())
    p /= p.sum()
    p = np.where(see, p, 0.0)
    V = np.where(see[:, None], V, 0.0)
    near = p > 1e-9
    delta = U * (mag + 8 * float(np.max(np.abs(s[near]))) + (4 * cap if cap > 0 else 0) +
                 2 * abs(slope) * float(np.max(np.abs(dist[near]))) + 8)
    return p @ V, (2 * delta + U * (4 * math.sqrt(len(s)) + 40)) * (p @ np.abs(V)) + 1e-30


def check_decode(ctx, nnhip, B, H, Hkv, dk, page, pos, f16, rope=True, cap=0.0, slopes=False, tokens=True, seed=0,
                 len_bound=None, spread=1.0):
    print(f"decode B={B} H={H} Hkv={Hkv} dk={dk} page={page} pos={list(pos)[:8]} f16={f16} cap={cap} slopes={slopes} "
          f"tokens={tokens}", flush=True)
    rng = np.random.default_rng(seed + 1000 * dk + H)
    pos = np.array(pos, np.int32)
    bound = int(pos.max()) + 1 if len_bound is None else len_bound
    c = Cache(rng, np.maximum(pos + 1, 0), Hkv, page, dk, f16, width=-(-bound // page))
    for b, p in enumerate(pos):  # the new row is the call's to write
        if p >= 0:
            c.set(b, p, np.full((Hkv, dk), np.nan), np.full((Hkv, dk), np.nan))
    q = (spread * rng.standard_normal((B, H, dk))).astype(np.float32)
    k, v = (rng.standard_normal((B, Hkv, dk)).astype(np.float32) for _ in range(2))
    cos, sin = nnhip.rope_table(dk, bound) if rope else (None, None)
    sl = (2.0 ** (-8.0 * (np.arange(H) + 1) / H)).astype(np.float32) if slopes else None
    scale = float(np.float32(1 / math.sqrt(dk)))
    cache = c.on_device(nnhip)
    lay = (lambda x: x.reshape(B, -1)) if tokens else (lambda x: x.reshape(B, -1).T)
    out = ctx.attention_pages_decode(cache, dev(lay(q)), dev(lay(k)), dev(lay(v)), H, dev(pos), bound, scale,
                                     cos=None if cos is None else dev(cos), sin=None if sin is None else dev(sin),
                                     softcap=cap, slopes=None if sl is None else dev(sl), tokens=tokens)
    out = host(out).astype(np.float64)
    out = (out if tokens else out.T).reshape(B, H, dk)
    for b, p in enumerate(pos):
        if p < 0:
            assert np.all(out[b] == 0)
            continue
        c.set(b, p, rotate(k[b], cos, sin, p), v[b])
        K, V = c.rows(b, p + 1)
        qr = rotate(q[b].astype(np.float64), cos, sin, p)
        for h in range(H):
            g = h // (H // Hkv)
            ref, tol = attend64(qr[h], K[:, g], V[:, g], scale, cap, 0.0 if sl is None else float(sl[h]),
                                np.arange(p + 1) - float(p), np.ones(p + 1, bool))
            off = np.abs(out[b, h] - ref)
            assert np.all(off <= tol), f"b={b} p={p} h={h}: {np.max(off / tol)} times the bound"
    assert same(host(cache.k), c.k) and same(host(cache.v), c.v), "the pools differ"


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("dk", [64, 128, 256])
@pytest.mark.parametrize("H,Hkv", [(1, 1), (4, 2), (8, 2), (6, 2), (8, 1), (12, 1)])
def test_decode_head_layouts(ctx, nnhip, H, Hkv, dk, f16):
    check_decode(ctx, nnhip, 3, H, Hkv, dk, 16, [0, 37, 300], f16, seed=1)


@pytest.mark.parametrize("page", [1, 2, 8, 64, 1024])
@pytest.mark.parametrize("f16", [False, True])
def test_decode_page_sizes(ctx, nnhip, page, f16):
    # lengths on and beside the edges of tiles (16), waves' turns (64), chunks (128) and pages
    check_decode(ctx, nnhip, 13, 4, 1, 64, page, [0, 1, 15, 16, 17, 63, 64, 127, 128, 129, 255, 256, 257], f16, seed=2)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("cap,slopes", [(20.0, False), (0.0, True), (5.0, True)])
def test_decode_shaped_scores(ctx, nnhip, cap, slopes, f16):
    check_decode(ctx, nnhip, 4, 8, 2, 128, 32, [5, 130, 400, 777], f16, cap=cap, slopes=slopes, seed=3, spread=4.0)


@pytest.mark.parametrize("tokens", [False, True])
def test_decode_layouts_slots_no_rope(ctx, nnhip, tokens):
    # empty slots among the sequences, a bound past every position
    check_decode(ctx, nnhip, 6, 4, 2, 64, 16, [-1, 40, -7, 0, 129, -1], False, rope=False, tokens=tokens, seed=4,
                 len_bound=1000)


def test_decode_large_scores(ctx, nnhip):
    """Scores of hundreds: the softmax is nearly a choice, the sums move their reference often."""
    check_decode(ctx, nnhip, 2, 4, 1, 128, 64, [200, 1500], True, seed=5, spread=60.0)
    check_decode(ctx, nnhip, 2, 4, 1, 128, 64, [200, 1500], False, seed=6, spread=60.0)


def test_decode_long(ctx, nnhip):
    """Many chunks to join: one sequence of 20 K beside short ones."""
    check_decode(ctx, nnhip, 3, 4, 1, 64, 64, [20000, 7, 4097], True, seed=7)


def test_decode_bad_pages_and_positions(ctx, nnhip):
    """A page outside the pool: NaN for its sequence alone. A position past the bound: NaN, nothing
    written. Entries past a sequence's length are never looked at."""
    rng = np.random.default_rng(8)
    B, H, Hkv, dk, page = 5, 4, 2, 64, 16
    pos = np.array([40, 40, 300, 40, 199], np.int32)
    c = Cache(rng, pos + 1, Hkv, page, dk, False)
    for b, p in enumerate(pos):
        c.set(b, p, np.full((Hkv, dk), 7.0), np.full((Hkv, dk), 7.0))
    good = c.on_device(nnhip)
    q, k, v = (dev(rng.standard_normal((B, n * dk)).astype(np.float32)) for n in (H, Hkv, Hkv))
    ref = host(ctx.attention_pages_decode(good, q, k, v, H, dev(pos), 301, 0.125, tokens=True))
    assert np.all(np.isfinite(ref))
    for bad in (-1, c.k.shape[0], 2 ** 31 - 1, -2 ** 31):
        t = c.table.copy()
        t[1, 1], t[2, 18], t[3, 3:] = bad, bad, bad  # inside, last page of the longest, past the length
        cache = nnhip.KVPages(dev(c.k), dev(c.v), dev(t))
        out = host(ctx.attention_pages_decode(cache, q, k, v, H, dev(pos), 301, 0.125, tokens=True))
        assert np.all(np.isnan(out[[1, 2]])) and np.array_equal(out[[0, 3, 4]], ref[[0, 3, 4]])
    # bound 200: sequence 2 is past it
    cache = c.on_device(nnhip)
    out = host(ctx.attention_pages_decode(cache, q, k, v, H, dev(pos), 200, 0.125, tokens=True))
    assert np.all(np.isnan(out[2])) and np.all(np.isfinite(out[[0, 1, 3, 4]]))
    i, s = c.table[2, 300 // page], 300 % page
    assert np.all(host(cache.k)[i, :, s] == 7.0)


def test_decode_nonfinite_inputs(ctx, nnhip):
    """A NaN or an infinity in a visible row shows in its own sequence and KV head only; rows behind a
    sequence's end (NaN in every test here) never do; a row whose scores are all -infinity gives 0."""
    rng = np.random.default_rng(9)
    B, H, Hkv, dk, page = 3, 4, 2, 64, 16
    pos = np.array([70, 70, 70], np.int32)
    c = Cache(rng, pos + 1, Hkv, page, dk, True)
    q = np.abs(rng.standard_normal((B, H * dk))).astype(np.float32)
    k, v = (rng.standard_normal((B, Hkv * dk)).astype(np.float32) for _ in range(2))
    c.v[c.table[0, 2], 1, 3, 5] = np.nan
    for t in range(70):
        c.k[c.table[1, t // page], 0, t % page] = -np.inf
    k[1, :dk] = -np.inf
    out = host(ctx.attention_pages_decode(c.on_device(nnhip), dev(q), dev(k), dev(v), H, dev(pos), 71, 0.125,
                                          tokens=True)).reshape(B, H, dk)
    n = np.isnan(out)
    assert n[0, 2:, 5].all() and n.sum() == 2
    assert np.all(out[1, :2] == 0) and np.all(out[1, 2:] != 0)


@pytest.mark.parametrize("dk", [64, 128, 256])
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("rope", [False, True])
def test_fill(ctx, nnhip, dk, f16, rope):
    """Packed prompts of unlike lengths (an empty one, one token, page and tile edges) at unlike positions;
    columns behind the last sequence, positions past the table and pages outside the pool are not written."""
    rng = np.random.default_rng(10 + dk)
    Hkv, page = 3, 16
    lens, pos0 = [1, 0, 33, 64, 16, 5, 70], [0, 9, 15, 0, 16, 95, 33]
    cu = np.concatenate(([0], np.cumsum(lens))).astype(np.int32)
    M = int(cu[-1]) + 21
    c = Cache(rng, [p + n for p, n in zip(pos0, lens)], Hkv, page, dk, f16)
    c.table = c.table[:, :6].copy()  # 96 positions: sequences 5 and 6 reach past it
    c.table[3, 1] = c.k.shape[0]     # a page outside the pool
    k, v = (rng.standard_normal((Hkv * dk, M)).astype(np.float32) for _ in range(2))
    cos, sin = nnhip.rope_table(dk, 100) if rope else (None, None)
    cache = c.on_device(nnhip)
    ctx.kv_pages_fill(cache, dev(k), dev(v), dev(cu), dev(np.array(pos0, np.int32)), None if cos is None else dev(cos),
                      None if sin is None else dev(sin))
    for b, n in enumerate(lens):
        for t in range(n):
            p, m = pos0[b] + t, cu[b] + t
            if p < 96 and 0 <= c.table[b, p // page] < c.k.shape[0]:
                c.set(b, p, rotate(k[:, m].reshape(Hkv, dk), cos, sin, p), v[:, m].reshape(Hkv, dk))
    assert same(host(cache.k), c.k) and same(host(cache.v), c.v)


def test_fill_matches_contiguous_fill(ctx, nnhip):
    """Equal prompts into pages of 8 and into contiguous caches: the same bits."""
    rng = np.random.default_rng(11)
    B, T, Hkv, dk, page = 3, 40, 2, 128, 8
    k, v = (dev(rng.standard_normal((Hkv * dk, B * T)).astype(np.float32)) for _ in range(2))
    cos, sin = (dev(x) for x in nnhip.rope_table(dk, 64))
    kc, vc = (dev(np.zeros((B, 64, Hkv * dk), np.float32)) for _ in range(2))
    ctx.kv_cache_fill(k, v, B, T, Hkv, dk, 0, kc, vc, cos, sin)
    table = rng.permutation(B * 5).astype(np.int32).reshape(B, 5)
    kp, vp = (dev(np.zeros((B * 5, Hkv, page, dk), np.float32)) for _ in range(2))
    ctx.kv_pages_fill(nnhip.KVPages(kp, vp, dev(table)), k, v, dev(np.arange(B + 1, dtype=np.int32) * T), cos=cos, sin=sin)
    for pool, ref in ((kp, kc), (vp, vc)):
        got = host(pool)[table].transpose(0, 1, 3, 2, 4).reshape(B, T, Hkv * dk)
        assert same(got, host(ref)[:, :T])


def test_refusals(ctx, nnhip):
    import torch
    f = dict(dtype=torch.float32, device="cuda")
    i = dict(dtype=torch.int32, device="cuda")
    pool, table = torch.zeros(4, 2, 16, 64, **f), torch.zeros(2, 2, **i)
    c = nnhip.KVPages(pool, pool.clone(), table)
    q, k, pos = torch.zeros(2, 256, **f), torch.zeros(2, 128, **f), torch.zeros(2, **i)

    def decode(cache=c, q=q, k=k, v=k, H=4, pos=pos, bound=32, **kw):
        return ctx.attention_pages_decode(cache, q, k, v, H, pos, bound, 0.125, tokens=True, **kw)

    decode()
    for kw in (dict(bound=33), dict(bound=0), dict(softcap=-1.0), dict(softcap=math.inf), dict(softcap=math.nan),
               dict(H=3, q=torch.zeros(2, 192, **f)), dict(q=q.double()), dict(k=k[:, :64]), dict(pos=pos.long()),
               dict(cos=torch.zeros(31, 32, **f), sin=torch.zeros(31, 32, **f)), dict(cos=torch.zeros(32, 32, **f)),
               dict(slopes=torch.zeros(3, **f)), dict(pos=torch.zeros(3, **i)), dict(q=torch.zeros(4, 256, **f)[::2]),
               dict(out=torch.zeros(2, 256, **f).t()), dict(q=q.cpu())):
        with pytest.raises(nnhip.NNHipError):
            decode(**kw)
    for shape in ((4, 2, 16, 96), (4, 2, 24, 64), (4, 2, 2048, 64)):
        p = torch.zeros(shape, **f)
        with pytest.raises(nnhip.NNHipError):
            decode(cache=nnhip.KVPages(p, p.clone(), table))
    with pytest.raises(nnhip.NNHipError):
        nnhip.KVPages(pool, pool.half(), table)
    off = torch.zeros(4 * 2 * 16 * 64 + 1, **f)[1:].view(4, 2, 16, 64)
    with pytest.raises(nnhip.NNHipError, match="16-byte"):
        decode(cache=nnhip.KVPages(off, pool, table))
    cu = torch.tensor([0, 3], **i)
    kk = torch.zeros(128, 3, **f)
    ctx.kv_pages_fill(c, kk, kk, cu)
    for a in ((kk[:64], kk, cu), (kk, kk.half(), cu), (kk, kk, cu.long()), (kk, kk, torch.zeros(4, **i))):
        with pytest.raises(nnhip.NNHipError):
            ctx.kv_pages_fill(c, *a)
    with pytest.raises(nnhip.NNHipError):
        ctx.kv_pages_fill(c, kk, kk, cu, pos0=torch.zeros(2, **i))
    ctx.kv_pages_fill(c, kk[:, :0], kk[:, :0], cu)  # no columns: nothing to do
    ctx.sync()


def test_streams_graphs_and_workspace(nnhip):
    """A captured call replays with new inputs between eager calls of larger sizes (whose workspace must not
    take the captured one's), calls on two streams at once keep to their own scratch, and a capture that
    would have to grow the workspace is refused."""
    import torch
    ctx = nnhip.Context(0)
    rng = np.random.default_rng(12)
    H, Hkv, dk, page = 8, 2, 64, 16

    def problem(B, length, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        n = -(-length // page)
        pools = [torch.randn(B * n, Hkv, page, dk, generator=g, device="cuda") for _ in range(2)]
        table = torch.randperm(B * n, generator=g, device="cuda").int().view(B, n)
        x = [torch.randn(B, h * dk, generator=g, device="cuda") for h in (H, Hkv, Hkv)]
        pos = torch.full((B,), length - 1, dtype=torch.int32, device="cuda")
        return nnhip.KVPages(*pools, table), x, pos, length, torch.empty_like(x[0])

    def call(p):
        cache, x, pos, length, out = p
        return ctx.attention_pages_decode(cache, *x, H, pos, length, 0.125, out=out, tokens=True)

    small, large = problem(2, 700, 1), problem(5, 3000, 2)
    refs = [call(p).clone() for p in (small, large)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        call(small)
        call(small)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        call(small)
    for i in range(4):
        small[1][0].mul_(1.5)
        with torch.cuda.stream(side):
            if i == 1:
                call(large)  # grows the side stream's workspace
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = small[4].clone()
        want = call(small).clone()
        assert torch.equal(got, want)
    # two streams at once
    a, b = problem(3, 2500, 3), problem(3, 2500, 4)
    want = [call(p).clone() for p in (a, b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(10):
        for s, p in zip(streams, (a, b)):
            with torch.cuda.stream(s):
                call(p)
    torch.cuda.synchronize()
    assert torch.equal(a[4], want[0]) and torch.equal(b[4], want[1])
    fresh = torch.cuda.Stream()
    g2 = torch.cuda.CUDAGraph()
    with pytest.raises(nnhip.NNHipError, match="capture"):
        with torch.cuda.graph(g2, stream=fresh):
            small[4].zero_()
            call(small)
    torch.cuda.synchronize()
    assert torch.equal(call(large), refs[1])
    ctx.close()
