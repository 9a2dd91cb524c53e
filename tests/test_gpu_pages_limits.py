"""Paged decode attention at the ends of what its inputs may hold: infinite keys (an f16 pool gets them from every
key past 65504), queries and caps of extreme sizes. A score is the sum of its products as f32 adds them: an
infinite key makes it infinite where the query's element is not 0, NaN where it is; a score of -infinity
weighs nothing, +infinity and NaN make the head's output NaN. Finite outputs are held to the bound of
test_gpu_pages.py over the keys that weigh something."""
import numpy as np
import pytest

from test_gpu_pages import Cache, attend64, dev, host

pytestmark = pytest.mark.gpu


def scores_of(q, K):
    """The products' sums with infinities, for (H, dk) queries of one KV head and (n, dk) keys."""
    with np.errstate(invalid="ignore"):
        return (q[:, None, :] * K[None, :, :]).sum(-1)


def check_head(out, q, K, V, scale):
    """One head's output against its formula; returns what became of it."""
    s = scores_of(q[None], K)[0] * scale
    if np.isnan(s).any() or (s == np.inf).any():
        assert np.all(np.isnan(out)), out
        return "nan"
    see = s > -np.inf
    if not see.any():
        assert np.all(out == 0), out
        return "zero"
    ref, tol = attend64(q, K[see], V[see], scale, 0.0, 0.0, np.zeros(int(see.sum())), np.ones(int(see.sum()), bool))
    off = np.abs(out - ref)
    assert np.all(off <= tol), f"{np.max(off / tol)} times the bound"
    return "finite"


@pytest.mark.parametrize("new", [False, True])
@pytest.mark.parametrize("exact", [False, True])
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("dk", [64, 128])
@pytest.mark.parametrize("R", [2, 5, 8])
def test_decode_infinite_keys(ctx, nnhip, R, dk, f16, exact, new):
    """Infinite keys among the cached ones, or the new one, against queries of mixed signs, exact: ones that f16 holds
    (nothing is left for a second part). Sequence 0: an infinity that some heads weigh -infinity and others +infinity;
    1: one against query elements far below their head's largest; 2: every key, -infinity for heads of one
    sign; 3: one against an element that is 0; 4: none."""
    print(f"infinite keys R={R} dk={dk} f16={f16} exact={exact} new={new}", flush=True)
    rng = np.random.default_rng(100 + R)
    B, Hkv, page, n = 5, 2, 16, 300
    H = R * Hkv
    pos = np.full(B, n, np.int32)
    c = Cache(rng, pos + 1, Hkv, page, dk, f16)
    q = rng.standard_normal((B, H, dk)).astype(np.float32)
    if exact:
        q = (np.round(q * 64) / 64).astype(np.float32)
    q[0, :, 5] = np.where(np.arange(H) % 2 == 0, -0.5, 0.75)
    q[1, :, 9] = 2.0 ** -44 * np.where(np.arange(H) % 3 == 0, 1.0, -1.0)
    q[2, :, 0] = np.where(np.arange(H) % 2 == 0, -1.0, 1.0)
    q[3, :, 7] = np.where(np.arange(H) % 2 == 0, 0.0, -1.0)
    k, v = (rng.standard_normal((B, Hkv, dk)).astype(np.float32) for _ in range(2))

    def put(b, t, e):
        if new and t == n:
            k[b, :, e] = np.inf if not f16 else 1e6  # f16: past its largest
        else:
            c.k[c.table[b, t // page], :, t % page, e] = np.inf

    put(0, n if new else 130, 5)
    put(1, n if new else 17, 9)
    for t in range(n + 1):
        put(2, t, 0)
    if not new:
        k[2, :, 0] = np.inf
    put(3, n if new else 299, 7)
    out = host(ctx.attention_pages_decode(c.on_device(nnhip), dev(q.reshape(B, -1)), dev(k.reshape(B, -1)),
                                          dev(v.reshape(B, -1)), H, dev(pos), n + 1, 0.125,
                                          tokens=True)).astype(np.float64).reshape(B, H, dk)
    found = set()
    for b in range(B):
        with np.errstate(over="ignore"):
            c.set(b, n, k[b], v[b])
        K, V = c.rows(b, n + 1)
        for h in range(H):
            g = h // R
            found.add((b, check_head(out[b, h], q[b, h].astype(np.float64), K[:, g], V[:, g], 0.125)))
    assert found == {(0, "finite"), (0, "nan"), (1, "finite"), (1, "nan"), (2, "zero"), (2, "nan"), (3, "nan"),
                     (3, "finite"), (4, "finite")}


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("H,Hkv,dk", [(4, 2, 64), (8, 1, 64), (10, 2, 128), (8, 1, 256)])
@pytest.mark.parametrize("size,cap,scale", [(1e15, 1e-30, 0.125), (1e30, 0.0, 1e20), (1e-30, 1e30, 0.125)])
def test_decode_extreme_queries_and_caps(ctx, nnhip, H, Hkv, dk, f16, size, cap, scale):
    """Queries, caps and scales whose quotient or product passes f32's range on the way: sequence 0's keys are 0, so all
    its scores are, and its output is the mean of the values; under the smallest cap sequence 1's is, too (scores of
    1e-30 at most), and under the largest its scores are those of queries of 1e-30."""
    print(f"extreme H={H} Hkv={Hkv} dk={dk} f16={f16} size={size} cap={cap} scale={scale}", flush=True)
    rng = np.random.default_rng(200 + dk)
    B, page, n = 2, 16, 200
    pos = np.full(B, n, np.int32)
    c = Cache(rng, pos + 1, Hkv, page, dk, f16)
    q = (size * rng.standard_normal((B, H, dk))).astype(np.float32)
    k, v = (rng.standard_normal((B, Hkv, dk)).astype(np.float32) for _ in range(2))
    k[0] = 0
    for t in range(n):
        c.k[c.table[0, t // page], :, t % page] = 0
    out = host(ctx.attention_pages_decode(c.on_device(nnhip), dev(q.reshape(B, -1)), dev(k.reshape(B, -1)),
                                          dev(v.reshape(B, -1)), H, dev(pos), n + 1, scale, softcap=cap,
                                          tokens=True)).astype(np.float64).reshape(B, H, dk)
    for b in range(1 if cap == 0 else 2):
        c.set(b, n, k[b], v[b])
        V = c.rows(b, n + 1)[1]
        for h in range(H):
            x = V[:, h // (H // Hkv)]
            # equal weights (scores below 1e-28 change none): attend64's bound of the sums, nothing of the scores
            tol = 2.0 ** -24 * (4 * np.sqrt(n + 1) + 40 + 16) * np.abs(x).mean(0)
            assert np.all(np.abs(out[b, h] - x.mean(0)) <= tol), (b, h)


def test_workspace_queries(ctx, nnhip):
    """Of no sequence, of short rows and short caches (nothing), of long ones (per sequence), of arguments that fit
    nothing."""
    for B in (0, 1, 64, 65535):
        assert ctx.logits_workspace_bytes(0, B) == ctx.logits_workspace_bytes(10000, B) == 0
        assert ctx.attention_pages_workspace_bytes(B, 8, 2, 64, 128) == 0
        assert ctx.attention_pages_workspace_bytes(B, 8, 2, 64, 0) == ctx.attention_pages_workspace_bytes(B, 8, 3, 64, 999) == 0
        assert ctx.attention_pages_workspace_bytes(B, 0, 2, 64, 999) == ctx.attention_pages_workspace_bytes(B, 8, 0, 64, 999) == 0
    assert ctx.logits_workspace_bytes(131071, 0) == ctx.attention_pages_workspace_bytes(0, 8, 2, 64, 9999) == 0
    for B in (1, 64, 1024):
        assert ctx.logits_workspace_bytes(131071, B) >= 16 * B  # two slices a row at least
        assert ctx.attention_pages_workspace_bytes(B, 8, 2, 64, 9999) >= B * 8 * 64 * 4  # a record a head at least
    assert ctx.logits_workspace_bytes(131071, 65535) == 0  # a row a work-group


@pytest.mark.parametrize("width", [8, 40])  # 128 positions: a work-group a block of queries; 640: equal spans
@pytest.mark.parametrize("dk,f16", [(64, False), (128, True)])
def test_prompt_bound_of_no_tokens(ctx, nnhip, width, dk, f16):
    """t_bound = 0 over sequences without tokens: nothing is written; over sequences with some: theirs are NaN, as any
    that has more than the bound."""
    import torch
    rng = np.random.default_rng(31)
    H, Hkv, page, M = 4, 2, 16, 20
    c = Cache(rng, [64, 64, 64], Hkv, page, dk, f16, width=width)
    q = dev(rng.standard_normal((H * dk, M)).astype(np.float32))
    for cu, bad in (([0, 0, 0, 0], []), ([3, 3, 4, 9], list(range(3, 9)))):
        out = torch.full((H * dk, M), 7.0, device="cuda")
        ctx.attention_pages_prefill(c.on_device(nnhip), q, dev(np.array(cu, np.int32)), 0, H, 0.125, out=out)
        got = host(out)
        rest = [m for m in range(M) if m not in bad]
        assert np.all(np.isnan(got[:, bad])) and np.all(got[:, rest] == 7.0)


def distance_ref(c, b, q, i, n, slope, cap, scale, prefix):
    at = np.arange(n)
    K, V = c.rows(b, n)
    return attend64(q, K[:, 0], V[:, 0], scale, cap, slope, -np.abs(at - float(i)), (at <= i) | (at < prefix))


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("dk", [64, 128])
@pytest.mark.parametrize("cap", [0.0, 5.0])
def test_prompt_distance_bias(ctx, nnhip, cap, dk, f16):
    """Biases that fall with the distance on both sides of the query, inside prefixes longer and shorter than a tile, than
    the sequence, and of none; the first query of a prefix weighs its far end least, not most."""
    print(f"distance bias cap={cap} dk={dk} f16={f16}", flush=True)
    rng = np.random.default_rng(300 + dk)
    H, lens, pos0, prefix = 4, [300, 40, 90, 33], [0, 20, 0, 100], [256, 50, 1000, 0]
    cu = np.concatenate(([0], np.cumsum(lens))).astype(np.int32)
    M = int(cu[-1])
    c = Cache(rng, [p + n for p, n in zip(pos0, lens)], 1, 16, dk, f16)
    q = rng.standard_normal((H, dk, M)).astype(np.float32)
    slopes = (2.0 ** -np.array([0.5, 2.0, 5.0, 8.0])).astype(np.float32)
    scale = float(np.float32(1 / np.sqrt(dk)))

    def run(prefix, distance):
        return host(ctx.attention_pages_prefill(
            c.on_device(nnhip), dev(q.reshape(H * dk, M)), dev(cu), max(lens), H, scale, pos0=dev(np.array(pos0, np.int32)),
            softcap=cap, slopes=dev(slopes), prefix=None if prefix is None else dev(np.array(prefix, np.int32)),
            distance=distance)).reshape(H, dk, M)

    out = run(prefix, True).astype(np.float64)
    worst = 0.0
    for b, n in enumerate(lens):
        for t in sorted({0, 1, 31, 32, n // 2, n - 1}):
            for h in range(H):
                ref, tol = distance_ref(c, b, q[h, :, cu[b] + t].astype(np.float64), pos0[b] + t, pos0[b] + n,
                                        float(slopes[h]), cap, scale, prefix[b])
                worst = max(worst, float(np.max(np.abs(out[h, :, cu[b] + t] - ref) / tol)))
                assert worst <= 4, f"b={b} t={t} h={h}: {worst} times the bound"  # 4 u of a product, as the prompts' tests
    for p in (None, [0, 0, 0, 0]):  # nothing is ahead: the linear bias, bit for bit
        assert np.array_equal(run(p, True), run(p, False))
    assert not np.array_equal(run(prefix, True), run(prefix, False))


@pytest.mark.parametrize("f16", [False, True])
def test_prompt_distance_bias_f32_products(ctx, nnhip, f16):
    """The same from the products that inputs beyond the parts' range take: a query of 1e16 against keys of 0 beside an
    ordinary one."""
    rng = np.random.default_rng(310)
    dk, n, prefix = 64, 200, 150
    c = Cache(rng, [n], 1, 16, dk, f16)
    c.k[..., 3] *= 0
    q = rng.standard_normal((1, dk, n)).astype(np.float32)
    q[0, 3, ::7] = 1e16
    out = host(ctx.attention_pages_prefill(c.on_device(nnhip), dev(q.reshape(dk, n)), dev(np.array([0, n], np.int32)), n, 1,
                                           0.125, slopes=dev(np.array([0.3], np.float32)),
                                           prefix=dev(np.array([prefix], np.int32)), distance=True)).astype(np.float64)
    for t in (0, 7, 8, 70, 149, 150, 196, 199):
        x = q[0, :, t].astype(np.float64)
        x[3] = 0  # its keys are
        ref, tol = distance_ref(c, 0, x, t, n, float(np.float32(0.3)), 0.0, 0.125, prefix)
        assert np.all(np.abs(out[:, t] - ref) <= 4 * tol), t


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("R,dk", [(2, 64), (5, 64), (8, 64), (8, 128)])
def test_decode_infinite_keys_under_a_cap(ctx, nnhip, R, dk, f16):
    """Under a cap an infinite score is the cap or its negative, and a key like any other: several of them among the cached
    keys and the new one, with a distance bias. One against an element that is 0 leaves the head NaN."""
    rng = np.random.default_rng(120 + R)
    B, page, n, cap, scale = 4, 16, 300, 3.0, 0.125
    H = R
    pos = np.full(B, n, np.int32)
    c = Cache(rng, pos + 1, 1, page, dk, f16)
    q = rng.standard_normal((B, H, dk)).astype(np.float32)
    q[:, :, 9] = 2.0 ** -44 * np.where(np.arange(H) % 3 == 0, 1.0, -1.0)
    q[3, 0, 7] = 0
    k, v = (rng.standard_normal((B, 1, dk)).astype(np.float32) for _ in range(2))

    def put(b, t, e, x):
        c.k[c.table[b, t // page], :, t % page, e] = x

    for b, e in ((0, 5), (1, 9)):
        for t in (3, 64, 65, 131, 280, 299):
            put(b, t, e, np.inf if t % 2 else -np.inf)
    k[0, 0, 5], k[1, 0, 9] = 1e6, -1e6  # f16: past its largest
    put(3, 250, 7, np.inf)
    slopes = np.linspace(0.001, 0.02, H).astype(np.float32)
    out = host(ctx.attention_pages_decode(c.on_device(nnhip), dev(q.reshape(B, -1)), dev(k.reshape(B, -1)),
                                          dev(v.reshape(B, -1)), H, dev(pos), n + 1, scale, softcap=cap,
                                          slopes=dev(slopes), tokens=True)).astype(np.float64).reshape(B, H, dk)
    dist = np.arange(n + 1) - float(n)
    for b in range(B):
        with np.errstate(over="ignore"):
            c.set(b, n, k[b], v[b])
        K, V = c.rows(b, n + 1)
        for h in range(H):
            x = q[b, h].astype(np.float64)
            s = scores_of(x[None], K[:, 0])[0] * scale
            if np.isnan(s).any():
                assert b == 3 and h == 0 and np.all(np.isnan(out[b, h]))
                continue
            assert not (b == 3 and h == 0)
            s = cap * np.tanh(s / cap) + float(slopes[h]) * dist
            p = np.exp(s - s.max())
            p /= p.sum()
            # attend64's bound; an infinite score's value is the cap itself
            near = np.isfinite(K[:, 0]).all(1)
            mag = 4 * np.sqrt(dk + 8) * np.max(np.abs(K[near, 0]) @ np.abs(x)) * scale
            delta = 2.0 ** -24 * (mag + 8 * np.max(np.abs(s)) + 4 * cap + 2 * float(slopes[h]) * n + 8)
            tol = (2 * delta + 2.0 ** -24 * (4 * np.sqrt(n + 1) + 40)) * (p @ np.abs(V[:, 0])) + 1e-30
            off = np.abs(out[b, h] - p @ V[:, 0])
            assert np.all(off <= tol), f"b={b} h={h}: {np.max(off / tol)} times the bound"


def test_decode_infinite_keys_before_bad_pages(ctx, nnhip):
    """An infinite key in an early tile, a page outside the pool in a later one: NaN for that sequence alone."""
    rng = np.random.default_rng(140)
    B, H, dk, page, n = 3, 8, 64, 16, 500
    pos = np.full(B, n, np.int32)
    c = Cache(rng, pos + 1, 1, page, dk, True)
    q = rng.standard_normal((B, H, dk)).astype(np.float32)
    q[:, :, 5] = -0.5
    q[:, :, 9] = 2.0 ** -44
    k, v = (dev(rng.standard_normal((B, dk)).astype(np.float32)) for _ in range(2))
    for b in range(2):
        for t in (0, 130, 270, 400):
            c.k[c.table[b, t // page], 0, t % page, 5] = np.inf
            c.k[c.table[b, t // page], 0, t % page, 9] = -np.inf
    call = lambda t: host(ctx.attention_pages_decode(nnhip.KVPages(dev(c.k), dev(c.v), dev(t)), dev(q.reshape(B, -1)), k, v, H,
                                                     dev(pos), n + 1, 0.125, tokens=True))
    good = call(c.table)
    assert np.all(np.isfinite(good))
    for entry in (7, 15, 24, 30):
        table = c.table.copy()
        table[1, entry] = c.k.shape[0]
        out = call(table)
        assert np.all(np.isnan(out[1])) and np.array_equal(out[[0, 2]], good[[0, 2]])
