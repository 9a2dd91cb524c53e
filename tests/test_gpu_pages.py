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
                 len_bound=None, spread=1.0, edit=None):
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
    if edit is not None:
        edit(c, q, k)
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


@pytest.mark.parametrize("page", [8, 16, 64, 1024])
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


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("H,Hkv,dk", [(8, 1, 64), (16, 2, 128), (6, 1, 64), (4, 1, 128)])
def test_decode_query_range(ctx, nnhip, H, Hkv, dk, f16):
    """Heads of all magnitudes, and in each an element far above the others where the keys are 0: the score is
    that of the small elements, held to their own size (no term of the bound knows the large one)."""

    def edit(c, q, k):
        c.k[..., 0] *= 0  # (NaN stays where nothing is)
        k[..., 0] = 0
        q *= (10.0 ** np.linspace(-30, 1, H))[None, :, None].astype(np.float32)
        q[..., 0] = 2.0 ** 18 * np.abs(q).max(-1)

    check_decode(ctx, nnhip, 2, H, Hkv, dk, 16, [140, 517], f16, rope=False, seed=8, edit=edit)


@pytest.mark.parametrize("f16", [False, True])
def test_decode_infinite_query(ctx, nnhip, f16):
    """An infinite element of a head's query against keys of one sign: all scores -infinity give zeros, all +infinity
    NaN, and the other heads do not see it."""
    import torch
    rng = np.random.default_rng(9)
    B, H, dk, n = 1, 8, 64, 300
    c = Cache(rng, [n + 1], 1, 16, dk, f16)
    c.k[..., 0] = np.abs(c.k[..., 0]) + c.dt(0.1)
    q, k, v = (rng.standard_normal((B, h, dk)).astype(np.float32) for h in (H, 1, 1))
    k[..., 0] = 1.0
    ref = None
    for q3, q5 in ((0.5, 0.5), (-np.inf, np.inf)):
        q[0, 3, 0], q[0, 5, 0] = q3, q5
        out = host(ctx.attention_pages_decode(c.on_device(nnhip), dev(q.reshape(B, -1)), dev(k.reshape(B, -1)),
                                              dev(v.reshape(B, -1)), H, dev(np.array([n], np.int32)), n + 1, 0.125,
                                              tokens=True)).reshape(H, dk)
        if ref is None:
            ref = out
    rest = [h for h in range(H) if h not in (3, 5)]
    assert np.all(out[3] == 0) and np.all(np.isnan(out[5])) and same(out[rest], ref[rest])


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


@pytest.mark.parametrize("lens", [[1] + [0] * 8 + [4], [3] + [0] * 62 + [2], [1] + [0] * 63 + [5], [2] + [0] * 150 + [1, 0, 1],
                                  [0] * 70 + [65] + [0] * 40 + [7] + [0] * 5])
def test_fill_sequences_without_tokens(ctx, nnhip, lens):
    """Runs of empty sequences between tokens of one block, no column behind the last token."""
    rng = np.random.default_rng(12)
    Hkv, dk, page = 2, 64, 8
    cu = np.concatenate(([0], np.cumsum(lens))).astype(np.int32)
    M = int(cu[-1])
    c = Cache(rng, lens, Hkv, page, dk, False)
    k, v = (rng.standard_normal((Hkv * dk, M)).astype(np.float32) for _ in range(2))
    cache = c.on_device(nnhip)
    ctx.kv_pages_fill(cache, dev(k), dev(v), dev(cu))
    for b, n in enumerate(lens):
        for t in range(n):
            c.set(b, t, k[:, cu[b] + t].reshape(Hkv, dk), v[:, cu[b] + t].reshape(Hkv, dk))
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


# ------------------------------------------------------------------------------------------ prompts

# The prompt attention's products are sums of f16 and bf16 parts (or f32 products) that hold f32 operands to
# 2^-22 of a term, so its outputs are held to the decode form's bound with 4 u for each u of a product.

def check_prompt(ctx, nnhip, lens, pos0, H, Hkv, dk, page, f16, rope=True, cap=0.0, slopes=False, prefix=None, seed=0,
                 spread=1.0, t_bound=None, edit=None, sample=None):
    print(f"prompt lens={lens} pos0={pos0} H={H} Hkv={Hkv} dk={dk} page={page} f16={f16} cap={cap} slopes={slopes} "
          f"prefix={prefix}", flush=True)
    rng = np.random.default_rng(seed + 7 * dk + H)
    B, M = len(lens), sum(lens) + 3
    cu = np.concatenate(([0], np.cumsum(lens))).astype(np.int32)
    c = Cache(rng, [p + n for p, n in zip(pos0, lens)], Hkv, page, dk, f16)
    q = (spread * rng.standard_normal((H, dk, M))).astype(np.float32)
    if edit is not None:
        edit(c, q)
    cos, sin = nnhip.rope_table(dk, max(p + n for p, n in zip(pos0, lens))) if rope else (None, None)
    sl = (2.0 ** (-8.0 * (np.arange(H) + 1) / H)).astype(np.float32) if slopes else None
    scale = float(np.float32(1 / math.sqrt(dk)))
    out = dev(np.full((H * dk, M), 77.0, np.float32))
    ctx.attention_pages_prefill(c.on_device(nnhip), dev(q.reshape(H * dk, M)), dev(cu), t_bound or max(lens), H, scale,
                                pos0=dev(np.array(pos0, np.int32)), cos=None if cos is None else dev(cos),
                                sin=None if sin is None else dev(sin), softcap=cap, slopes=None if sl is None else dev(sl),
                                prefix=None if prefix is None else dev(np.array(prefix, np.int32)), out=out)
    out = host(out).astype(np.float64).reshape(H, dk, M)
    assert np.all(out[:, :, cu[-1]:] == 77.0), "columns of no sequence were written"
    worst = 0.0
    for b, n in enumerate(lens):
        if n == 0:
            continue
        K, V = c.rows(b, pos0[b] + n)
        at = np.arange(pos0[b] + n)
        for t in range(n) if sample is None else sorted({0, n - 1, *rng.integers(0, n, sample).tolist()}):
            i, m = pos0[b] + t, cu[b] + t
            see = at <= i
            if prefix is not None:
                see |= at < prefix[b]
            qr = rotate(q[:, :, m].astype(np.float64), cos, sin, i)
            for h in range(H):
                ref, tol = attend64(qr[h], K[:, h // (H // Hkv)], V[:, h // (H // Hkv)], scale, cap,
                                    0.0 if sl is None else float(sl[h]), at - float(i), see)
                got = out[h, :, m]
                nan = np.isnan(ref)
                assert np.array_equal(nan, np.isnan(got)), f"b={b} t={t} h={h}: NaN"
                off = np.abs(got - ref)[~nan] / tol[~nan]
                if off.size:
                    worst = max(worst, float(off.max()))
                    assert worst <= 4, f"b={b} t={t} h={h}: {worst} times the bound"
    print(f"  {worst:.3f} of the bound", flush=True)
    return out


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("dk", [64, 128])
@pytest.mark.parametrize("H,Hkv", [(1, 1), (4, 2), (4, 1), (8, 1), (6, 2), (12, 1)])
def test_prompt_head_layouts(ctx, nnhip, H, Hkv, dk, f16):
    check_prompt(ctx, nnhip, [1, 37, 0, 65], [0, 0, 5, 11], H, Hkv, dk, 16, f16, seed=20)


@pytest.mark.parametrize("page", [8, 64, 1024])
@pytest.mark.parametrize("f16", [False, True])
def test_prompt_page_sizes(ctx, nnhip, page, f16):
    # lengths and starts on and beside the edges of tiles (32) and pages
    check_prompt(ctx, nnhip, [31, 32, 33, 8, 7, 1], [0, 32, 31, 56, 1, 127], 2, 1, 64, page, f16, seed=21)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("cap,slopes,prefix", [(20.0, False, None), (0.0, True, None), (5.0, True, [40, 0, 200]),
                                               (0.0, False, [200, 33, 1])])
def test_prompt_shaped_scores(ctx, nnhip, cap, slopes, prefix, f16):
    check_prompt(ctx, nnhip, [70, 45, 33], [0, 20, 100], 4, 2, 128, 32, f16, cap=cap, slopes=slopes, prefix=prefix, seed=22,
                 spread=3.0)


def test_prompt_bounds_and_no_rope(ctx, nnhip):
    check_prompt(ctx, nnhip, [5, 90], [0, 0], 4, 4, 64, 16, False, rope=False, seed=23, t_bound=93)
    check_prompt(ctx, nnhip, [3], [700], 4, 1, 64, 16, True, seed=24)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("cap", [0.0, 10.0])
def test_prompt_nonfinite(ctx, nnhip, f16, cap):
    """A NaN or an infinity in a key or a value reaches the queries that see it, and no other of the same
    tile, work-group or sequence; scores of f32 range take the f32 products."""
    def values(c, q):
        c.v[c.table[0, 2], 0, 3, 5] = np.nan        # position 35
        c.v[c.table[1, 0], 0, 9, 6] = np.inf        # position 9: infinite where it is seen
        c.k[c.table[2, 1], 0, 4] = np.nan           # position 20

    rng_lens = [60, 40, 50]
    out = check_prompt_nonfinite(ctx, nnhip, rng_lens, f16, cap, values)
    nan = np.isnan(out)
    assert nan[:, 5, 35:60].all() and not nan[:, :, :35].any() and not nan[:, :5, 35:60].any()
    assert np.isinf(out[:, 6, 69:100]).all() and np.isfinite(out[:, :, 60:69]).all()
    assert nan[:, :, 120:150].all() and not nan[:, :, 100:120].any()
    assert np.all(np.isfinite(out[:, 7, 60:100]))

    def large(c, q):
        q *= 1e4
    if not f16:
        check_prompt(ctx, nnhip, [40], [3], 2, 1, 64, 16, f16, cap=cap, seed=26, edit=large)


def check_prompt_nonfinite(ctx, nnhip, lens, f16, cap, edit):
    rng = np.random.default_rng(25)
    H, dk, page = 2, 64, 16
    c = Cache(rng, lens, 1, page, dk, f16)
    M = sum(lens)
    q = rng.standard_normal((H * dk, M)).astype(np.float32)
    edit(c, q)
    cu = np.concatenate(([0], np.cumsum(lens))).astype(np.int32)
    return host(ctx.attention_pages_prefill(c.on_device(nnhip), dev(q), dev(cu), max(lens), H, 0.125, softcap=cap)).reshape(H, dk, M)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("H,Hkv,dk", [(4, 1, 128), (8, 1, 64), (2, 2, 64), (12, 1, 128)])
def test_prompt_shared_items(ctx, nnhip, H, Hkv, dk, f16):
    """Few queries over long caches: work-groups share the keys of a block of queries and join, at every number of
    them to a block, beside sequences of one tile and an empty one."""
    check_prompt(ctx, nnhip, [5, 1, 0, 40, 70], [3000, 1023, 9, 4090, 0], H, Hkv, dk, 64, f16, seed=30, sample=3)
    check_prompt(ctx, nnhip, [1], [9000], H, Hkv, dk, 64, f16, seed=31)


@pytest.mark.parametrize("f16", [False, True])
def test_prompt_shared_items_shaped(ctx, nnhip, f16):
    check_prompt(ctx, nnhip, [300, 33, 2], [400, 2000, 5], 4, 2, 64, 16, f16, cap=8.0, slopes=True, prefix=[650, 0, 7], seed=32,
                 spread=3.0, sample=6)
    check_prompt(ctx, nnhip, [700], [0], 8, 4, 64, 16, f16, seed=33, prefix=[512], sample=12)


def test_prompt_shared_items_many_sequences(ctx, nnhip):
    """More sequences than a wave has lanes, most of them of a token or none."""
    rng = np.random.default_rng(34)
    lens = [int(x) for x in rng.integers(0, 3, 150)]
    lens[70], lens[149] = 900, 65
    check_prompt(ctx, nnhip, lens, [int(x) for x in rng.integers(0, 40, 150)], 2, 1, 64, 16, True, seed=34, sample=4)


@pytest.mark.parametrize("seed", range(8))
def test_prompt_random_packings(ctx, nnhip, seed):
    """Spans of a few tiles: cuts at any tile of an item, beside empty sequences, prefixes and items of one tile."""
    rng = np.random.default_rng(600 + seed)
    B = int(rng.integers(1, 10))
    lens = [int(x) for x in rng.integers(0, 120, B)]
    lens[int(rng.integers(0, B))] = 33
    pos0 = [int(x) for x in rng.integers(0, [1, 700, 700][seed % 3], B)]
    H, Hkv, dk = [(20, 5, 128), (16, 2, 64), (4, 4, 64), (6, 3, 128)][seed % 4]
    prefix = [int(x) for x in rng.integers(0, 300, B)] if seed % 3 == 1 else None
    check_prompt(ctx, nnhip, lens, pos0, H, Hkv, dk, [8, 32, 64][seed % 3], seed % 2 == 0, cap=[0.0, 25.0][seed // 4],
                 slopes=seed % 4 == 1, prefix=prefix, seed=600 + seed, sample=5)


@pytest.mark.parametrize("f16", [False, True])
def test_prompt_shared_items_nonfinite(ctx, nnhip, f16):
    """What one work-group of an item meets (a NaN, an infinity, keys of f32 range, a page outside the pool) and
    the others do not."""
    rng = np.random.default_rng(35)
    H, dk, page, n, past = 4, 64, 16, 40, 3000
    total = past + n
    q = rng.standard_normal((H * dk, n)).astype(np.float32)

    def run(edit):
        c = Cache(np.random.default_rng(36), [total], 1, page, dk, f16)
        edit(c)
        return host(ctx.attention_pages_prefill(c.on_device(nnhip), dev(q), dev(np.array([0, n], np.int32)), n, H, 0.125,
                                                pos0=dev(np.array([past], np.int32)))).reshape(H, dk, n)

    def at(c, t):
        return c.table[0, t // page], t % page

    ref = run(lambda c: None)

    def v_nan(c):
        i, s = at(c, 1500)
        c.v[i, 0, s, 5] = np.nan

    def v_late(c):
        i, s = at(c, past + 20)
        c.v[i, 0, s, 5] = np.inf

    def k_nan(c):
        i, s = at(c, past + 20)
        c.k[i, 0, s, 0] = np.nan

    def bad(c):
        c.table[0, 1500 // page] = c.k.shape[0]

    got = run(v_nan)
    assert np.isnan(got[:, 5]).all() and np.isfinite(np.delete(got, 5, 1)).all()
    got = run(v_late)
    assert np.isinf(got[:, 5, 20:]).all() and np.isfinite(got[:, 5, :20]).all()
    got = run(k_nan)
    assert np.isnan(got[:, :, 20:]).all() and np.isfinite(got[:, :, :20]).all()
    assert np.isnan(run(bad)).all()

    # keys so large that one work-group takes the f32 products; their scores decide the softmax
    def large(c):
        for t in range(1500, 1510):
            i, s = at(c, t)
            c.k[i, 0, s] *= 2.0 ** 9
    c = Cache(np.random.default_rng(36), [total], 1, page, dk, f16)
    large(c)
    got = run(large).astype(np.float64)
    K, V = c.rows(0, total)
    for t in (0, 17, 39):
        see = np.arange(total) <= past + t
        for h in range(H):
            r, tol = attend64(q.reshape(H, dk, n)[h, :, t].astype(np.float64), K[:, 0], V[:, 0], 0.125, 0.0, 0.0,
                              np.arange(total) - float(past + t), see)
            assert np.all(np.abs(got[h, :, t] - r) <= 4 * tol)
    assert np.isfinite(ref).all()


def test_prompt_bad_sequences_in_spans(ctx, nnhip):
    """As test_prompt_bad_sequences where work-groups share items: room for 3000 positions in the table."""
    rng = np.random.default_rng(37)
    H, dk, page, lens = 2, 64, 16, [40, 900, 20]
    c = Cache(rng, lens, 1, page, dk, False, width=200)
    M = sum(lens) + 5
    q = dev(rng.standard_normal((H * dk, M)).astype(np.float32))

    def run(cu, t_bound, pos0=None):
        return host(ctx.attention_pages_prefill(c.on_device(nnhip), q, dev(np.array(cu, np.int32)), t_bound, H, 0.125,
                                                pos0=None if pos0 is None else dev(np.array(pos0, np.int32)),
                                                out=dev(np.full((H * dk, M), 7.0, np.float32))))

    ref = run([0, 40, 940, 960], 900)
    assert np.isfinite(ref).all() and np.all(ref[:, 960:] == 7.0)
    got = run([0, 40, 940, 960], 899)
    assert np.isnan(got[:, 40:940]).all() and np.array_equal(got[:, :40], ref[:, :40]) and np.array_equal(got[:, 940:], ref[:, 940:])
    got = run([0, 40, 940, 960], 900, [0, 0, 3190])
    assert np.isnan(got[:, 940:960]).all() and np.array_equal(got[:, :940], ref[:, :940])
    got = run([0, 0, 0, 0], 900)
    assert np.all(got == 7.0)


def test_prompt_captured_in_spans(nnhip):
    """A captured prompt call replays with new lengths (the work-groups find their shares on the device)."""
    import torch
    ctx = nnhip.Context(0)
    rng = np.random.default_rng(38)
    H, dk, page = 4, 64, 16
    c = Cache(rng, [2000, 2000], 1, page, dk, True)
    cache = c.on_device(nnhip)
    q = dev(rng.standard_normal((H * dk, 300)).astype(np.float32))
    cu, pos0 = dev(np.array([0, 100, 300], np.int32)), dev(np.array([1500, 0], np.int32))
    out = torch.zeros_like(q)
    side = torch.cuda.Stream()

    def call():
        ctx.attention_pages_prefill(cache, q, cu, 300, H, 0.125, pos0=pos0, out=out)

    with torch.cuda.stream(side):
        call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        call()
    for a, b, p in ((100, 1500, 0), (7, 1993, 1700), (290, 0, 30), (0, 5, 1000)):
        cu.copy_(torch.tensor([0, a, 300], dtype=torch.int32))
        pos0.copy_(torch.tensor([b, p], dtype=torch.int32))
        torch.cuda.synchronize()
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        got = out.clone()
        out.zero_()
        call()
        torch.cuda.synchronize()
        assert torch.equal(got, out) and bool(torch.isfinite(out).all())
    ctx.close()


def test_prompt_bad_sequences(ctx, nnhip):
    """Sequences that do not fit get NaN in the columns that are there; a page outside the pool shows in
    the queries that see it; the others keep their outputs."""
    rng = np.random.default_rng(27)
    H, Hkv, dk, page = 2, 1, 64, 16
    lens = [40, 40, 40, 20]
    c = Cache(rng, lens, Hkv, page, dk, False)
    M = 140
    q = dev(rng.standard_normal((H * dk, M)).astype(np.float32))
    cu = np.concatenate(([0], np.cumsum(lens))).astype(np.int32)

    def run(cu=cu, t_bound=40, pos0=None, table=None):
        cache = nnhip.KVPages(dev(c.k), dev(c.v), dev(c.table if table is None else table))
        return host(ctx.attention_pages_prefill(cache, q, dev(np.array(cu, np.int32)), t_bound, H, 0.125,
                                                pos0=None if pos0 is None else dev(np.array(pos0, np.int32))))

    ref = run()
    assert np.all(np.isfinite(ref))
    got = run(t_bound=39)
    assert np.isnan(got[:, :120]).all() and np.array_equal(got[:, 120:], ref[:, 120:])
    got = run(pos0=[0, 9, -1, 0])  # the second ends past its table's 48 positions
    assert np.array_equal(got[:, :40], ref[:, :40]) and np.isnan(got[:, 40:120]).all()
    got = run(cu=[0, 40, 80, 120, 200], t_bound=80)
    assert np.array_equal(got[:, :120], ref[:, :120]) and np.isnan(got[:, 120:]).all()
    for bad in (-1, c.k.shape[0], 2 ** 31 - 1):
        t = c.table.copy()
        t[1, 2] = bad  # positions 32 .. 39
        t[3, 2] = bad  # past its length
        got = run(table=t)
        assert np.isnan(got[:, 72:80]).all()
        keep = [m for m in range(M) if not 40 <= m < 80]
        assert np.array_equal(got[:, keep], ref[:, keep])


def test_prompt_matches_contiguous_prefill(ctx, nnhip):
    """Equal prompts over pages against nnhip_attention_prefill on contiguous caches: over f32 the same
    arithmetic; over f16 each weight is held to 2^-22 in either form, and both sum 96 terms."""
    rng = np.random.default_rng(28)
    for f16 in (False, True):
        B, T, H, Hkv, dk, page, past = 2, 70, 8, 2, 128, 16, 26
        dt = np.float16 if f16 else np.float32
        kc, vc = (rng.standard_normal((B, 96, Hkv * dk)).astype(dt) for _ in range(2))
        q = dev(rng.standard_normal((H * dk, B * T)).astype(np.float32))
        cos, sin = (dev(x) for x in nnhip.rope_table(dk, 96))
        want = ctx.attention_prefill(q, dev(kc), dev(vc), B, T, H, Hkv, dk, past, 0.1, cos, sin)
        table = rng.permutation(B * 6).astype(np.int32).reshape(B, 6)
        pools = []
        for x in (kc, vc):
            pool = np.zeros((B * 6, Hkv, page, dk), dt)
            pool[table] = x.reshape(B, 6, page, Hkv, dk).transpose(0, 1, 3, 2, 4)
            pools.append(dev(pool))
        got = ctx.attention_pages_prefill(nnhip.KVPages(*pools, dev(table)), q, dev(np.arange(B + 1, dtype=np.int32) * T), T, H,
                                          0.1, pos0=dev(np.full(B, past, np.int32)), cos=cos, sin=sin)
        if f16:
            assert np.max(np.abs(host(got) - host(want))) <= 64 * U * np.max(np.abs(vc))
        else:
            assert same(host(got), host(want))


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("gap", [8.0, 13.0, 20.0, 40.0, 55.0])
def test_prompt_spread_weights(ctx, nnhip, gap, f16):
    """A key that takes nearly all weight and whose values are 0, beside keys that are e^-gap of it: the outputs are
    those keys' alone, and hold to the bound of their own weights and values."""
    def edit(c, q):
        q *= 0.3
        q[:, 0] += 8.0
        c.k[c.table[0, 0], 0, 0] = 0
        c.k[c.table[0, 0], 0, 0, 0] = gap * 8.0 / 8.0  # scale 1/8, q 8: a score of gap
        c.v[c.table[0, 0], 0, 0] = 0
        for t in range(1, 70):
            i, s = c.table[0, t // 16], t % 16
            c.k[i, 0, s, 0] = 0.02 * (t % 7)
            c.v[i, 0, s, :8] *= np.float32(10.0) ** (t % 5 - 2)
    check_prompt(ctx, nnhip, [70], [0], 2, 1, 64, 16, f16, rope=False, seed=40, edit=edit)


def test_prompt_then_decode(ctx, nnhip):
    """A prompt in one call and its last token alone by the decode form agree; fill, prompt and decode in turn."""
    rng = np.random.default_rng(29)
    H, Hkv, dk, page, lens = 8, 2, 64, 16, [50, 7, 33]
    B, M = len(lens), sum(lens)
    cu = np.concatenate(([0], np.cumsum(lens))).astype(np.int32)
    table = dev(rng.permutation(B * 5).astype(np.int32).reshape(B, 5))
    cache = nnhip.KVPages(*(dev(np.zeros((B * 5, Hkv, page, dk), np.float32)) for _ in range(2)), table)
    q, k, v = (dev(rng.standard_normal((n * dk, M)).astype(np.float32)) for n in (H, Hkv, Hkv))
    cos, sin = (dev(x) for x in nnhip.rope_table(dk, 80))
    ctx.kv_pages_fill(cache, k, v, dev(cu), cos=cos, sin=sin)
    before = host(cache.k)
    out = host(ctx.attention_pages_prefill(cache, q, dev(cu), 50, H, 0.125, cos=cos, sin=sin))
    last = [int(x) - 1 for x in cu[1:]]
    one = host(ctx.attention_pages_decode(cache, q[:, last].contiguous(), k[:, last].contiguous(), v[:, last].contiguous(),
                                          H, dev(np.array(lens, np.int32) - 1), 50, 0.125, cos=cos, sin=sin))
    assert same(host(cache.k), before)  # the same rows again
    # both within a few roundings of the same value: scores up to about 4, 50 terms
    assert np.max(np.abs(one - out[:, last])) <= 64 * U * np.max(np.abs(host(v)))


@pytest.mark.parametrize("f16", [False, True])
def test_pools_past_32_bits(ctx, nnhip, f16):
    """Pages whose elements lie past 2^31 and 2^32 of the pool's: the same bits as from a pool of those pages alone."""
    import torch
    rng = np.random.default_rng(52)
    dt = torch.float16 if f16 else torch.float32
    B, H, Hkv, dk, page, n = 2, 8, 2, 128, 64, 300
    need = -(-(n + 1) // page)
    many = 2 ** 32 // (Hkv * page * dk) + 2 * B * need
    assert many * Hkv * page < 2 ** 31
    few = rng.permutation(B * need).astype(np.int32).reshape(B, need)
    places = (few * ((many - 1) // (B * need - 1))).astype(np.int32)  # from the first to the last of the pool
    cu = dev(np.arange(B + 1, dtype=np.int32) * n)
    q, k, v = (dev(rng.standard_normal((h * dk, B * n)).astype(np.float32)) for h in (H, Hkv, Hkv))
    qd, kd, vd = (dev(rng.standard_normal((h * dk, B)).astype(np.float32)) for h in (H, Hkv, Hkv))
    pos = dev(np.full(B, n, np.int32))
    cos, sin = (dev(x) for x in nnhip.rope_table(dk, n + 1))
    found = []
    for pages, table in ((B * need, few), (many, places)):
        pools = [torch.empty(pages, Hkv, page, dk, dtype=dt, device="cuda") for _ in range(2)]
        cache = nnhip.KVPages(*pools, dev(table))
        ctx.kv_pages_fill(cache, k, v, cu, cos=cos, sin=sin)
        a = host(ctx.attention_pages_prefill(cache, q, cu, n, H, 0.09, cos=cos, sin=sin))
        d = host(ctx.attention_pages_decode(cache, qd, kd, vd, H, pos, n + 1, 0.09, cos=cos, sin=sin))
        rows = [host(p[torch.from_numpy(table.reshape(-1).astype(np.int64)).cuda()])[:, :, :] for p in pools]
        last = (n + 1) % page or page
        kept = [r.reshape(B, need, Hkv, page, dk) for r in rows]
        found.append((a, d, [r[:, :-1] for r in kept], [r[:, -1, :, :last] for r in kept]))
        del pools, cache
    assert same(found[0][0], found[1][0]) and same(found[0][1], found[1][1])
    for i in (2, 3):
        for x, y in zip(found[0][i], found[1][i]):
            assert same(np.ascontiguousarray(x), np.ascontiguousarray(y))


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
    for shape in ((4, 2, 16, 96), (4, 2, 24, 64), (4, 2, 4, 64), (4, 2, 2048, 64)):
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
    qq = torch.zeros(256, 3, **f)
    ctx.attention_pages_prefill(c, qq, cu, 3, 4, 0.125)
    for a, kw in (((qq, cu, 4, 4), {}), ((qq, cu, 3, 3), {}), ((qq, cu, 3, 2), {}), ((qq.half(), cu, 3, 4), {}),
                  ((qq, cu, 3, 4), dict(softcap=-1.0)), ((qq, cu, 3, 4), dict(prefix=torch.zeros(2, **i))),
                  ((qq, cu, 3, 4), dict(out=qq.t().contiguous())), ((qq, cu, 3, 4), dict(cos=torch.zeros(3, 32, **f)))):
        with pytest.raises(nnhip.NNHipError):
            ctx.attention_pages_prefill(c, *a, 0.125, **kw)
    wide = torch.zeros(2, 1, 16, 256, **f)
    with pytest.raises(nnhip.NNHipError, match="64 or 128"):
        ctx.attention_pages_prefill(nnhip.KVPages(wide, wide.clone(), table), torch.zeros(256, 3, **f), cu, 3, 1, 0.1)
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
