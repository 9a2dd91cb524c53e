"""Adjusted logits and the greedy choice behind them on the GPU, against the rules in numpy: the steps are
single f32 operations in a given order, so outputs are compared bit for bit, and ids and counts exactly."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def dev(a):
    import torch
    a = np.ascontiguousarray(a)
    return torch.from_numpy(a.view(np.int32) if a.dtype == np.uint32 else a).cuda()


def host(t):
    return t.cpu().numpy()


def rules(x, counts=None, repeat=None, presence=None, frequency=None, bias=None, allowed=None):
    """Adjusted logits and ids of the rules, in f32 as the header orders them."""
    B, V = x.shape
    y = x.astype(np.float32).copy()
    f = np.float32
    with np.errstate(all="ignore"):
        for b in range(B):
            if counts is not None:
                c = np.maximum(counts[b], 0)
                seen = c > 0
                if repeat is not None:
                    y[b] = np.where(seen, np.where(y[b] > 0, y[b] / f(repeat[b]), y[b] * f(repeat[b])), y[b])
                if frequency is not None:
                    y[b] = np.where(seen, y[b] - f(frequency[b]) * c.astype(f), y[b])
                if presence is not None:
                    y[b] = np.where(seen, y[b] - f(presence[b]), y[b])
            if bias is not None:
                y[b] = y[b] + bias[b if len(bias) > 1 else 0]
        ok = np.ones((B, V), bool)
        if allowed is not None:
            w = allowed if len(allowed) > 1 else np.repeat(allowed, B, 0)
            v = np.arange(V)
            ok = (w[:, v // 32] >> (v % 32).astype(np.uint32)) & 1 != 0
        y = np.where(ok, y, f(-np.inf))
    ids = np.full(B, -1, np.int32)
    for b in range(B):
        best = -1
        for v in np.flatnonzero(ok[b]):
            if best < 0 or y[b, v] > y[b, best]:
                best = v
        ids[b] = best
    return y, ids


def same(a, b):
    n = np.isnan(a)
    return np.array_equal(n, np.isnan(b)) and np.array_equal(a[~n].view(np.uint32), b[~n].view(np.uint32))


def make(rng, B, V, hist=60, density=0.5):
    x = (3 * rng.standard_normal((B, V))).astype(np.float32)
    counts = np.zeros((B, V), np.int32)
    for b in range(B):
        np.add.at(counts[b], (V * rng.random(hist) ** 3).astype(int), 1)
    r = dict(repeat=(1 + rng.random(B)).astype(np.float32), presence=rng.random(B).astype(np.float32),
             frequency=rng.random(B).astype(np.float32))
    bias = rng.standard_normal((B, V)).astype(np.float32)
    bits = rng.random((B, (V + 31) // 32, 32)) < density
    allowed = (bits * (np.uint64(1) << np.arange(32, dtype=np.uint64))).sum(-1).astype(np.uint32)
    return x, counts, r, bias, allowed


def run(ctx, nnhip, x, write=True, pos=None, choice=True, **r):
    import torch
    print(f"logits {x.shape} {sorted(k for k in r if r[k] is not None)} write={write}", flush=True)
    t = {k: None if v is None else dev(v) for k, v in r.items()}
    L = dev(x)
    obj = nnhip.LogitRules(x.shape[1], count_choice=choice and t.get("counts") is not None, **t)
    out = torch.empty_like(L) if write else None
    p = None if pos is None else dev(pos)
    ids = torch.full((x.shape[0],), 99, dtype=torch.int32, device="cuda")
    ctx.logits_adjust_rows(L, obj, ids=ids, out=out, pos=p)
    ids = host(ids)
    y, want = rules(x, **r)
    assert np.array_equal(ids, want)
    if write:
        assert same(host(out), y)
    assert same(host(L), x)
    chosen = want >= 0
    if r.get("counts") is not None:
        c = r["counts"].copy()
        if choice:
            c[np.flatnonzero(chosen), want[chosen]] += 1
        assert np.array_equal(host(t["counts"]), c)
    if pos is not None:
        assert np.array_equal(host(p), pos + chosen)
    return ids


@pytest.mark.parametrize("V", [1, 3, 4, 31, 33, 127, 1000, 4097, 16384, 16387, 70001])
@pytest.mark.parametrize("B", [1, 5])
def test_every_rule(ctx, nnhip, B, V):
    rng = np.random.default_rng(V + B)
    x, counts, r, bias, allowed = make(rng, B, V)
    run(ctx, nnhip, x, counts=counts, **r, bias=bias, allowed=allowed, pos=np.arange(B, dtype=np.int32))


@pytest.mark.parametrize("what", ["none", "counts", "repeat", "presence", "frequency", "bias", "shared_bias", "allowed",
                                  "shared_allowed"])
def test_single_rules(ctx, nnhip, what):
    rng = np.random.default_rng(5)
    x, counts, r, bias, allowed = make(rng, 3, 777)
    kw = {"none": {}, "counts": dict(counts=counts), "bias": dict(bias=bias), "shared_bias": dict(bias=bias[:1]),
          "allowed": dict(allowed=allowed), "shared_allowed": dict(allowed=allowed[:1])}.get(
              what, dict(counts=counts, **({what: r[what]} if what in r else {})))
    run(ctx, nnhip, x, write=False, **kw)
    run(ctx, nnhip, x, choice=False, **kw)


def test_large_batch(ctx, nnhip):
    rng = np.random.default_rng(6)
    x, counts, r, bias, allowed = make(rng, 300, 2050)
    run(ctx, nnhip, x, counts=counts, **r, bias=bias[:1], allowed=allowed)


def test_nothing_allowed_and_ties(ctx, nnhip):
    """Rows that allow nothing give -1 and leave counts and positions; the lowest index wins a tie; an
    allowed -infinity is chosen before a forbidden token."""
    V = 20000
    x = np.zeros((5, V), np.float32)
    allowed = np.full((5, 625), 0xFFFFFFFF, np.uint32)
    allowed[1] = 0
    x[2, [7, 19999]] = 3.0
    x[3] = -np.inf
    allowed[3] = 0
    allowed[3, 600] = 1 << 5
    x[4] = np.inf
    allowed[4, :3] = 0
    counts = np.zeros((5, V), np.int32)
    ids = run(ctx, nnhip, x, counts=counts, allowed=allowed, pos=np.full(5, 4, np.int32))
    assert list(ids) == [0, -1, 7, 19205, 96]
    # bits past V do not make a token
    V = 33
    w = np.array([[0, 0xFFFFFFFE]], np.uint32)
    assert list(run(ctx, nnhip, np.zeros((1, V), np.float32), allowed=w)) == [-1]


def test_nonfinite(ctx, nnhip):
    """NaN is never chosen but where it is the first allowed token (the reference's loop); a forbidden NaN
    becomes -infinity; infinite logits and penalties keep IEEE's results."""
    rng = np.random.default_rng(7)
    x, counts, r, bias, allowed = make(rng, 6, 3001)
    x[0, 0] = np.nan
    x[1, 100:200] = np.nan
    x[2, 5] = np.inf
    x[3] = np.nan
    x[4, :50] = -np.inf
    allowed[0, 0] |= 1
    r["repeat"][5] = np.inf
    ids = run(ctx, nnhip, x, counts=counts, **r, bias=bias, allowed=allowed)
    assert ids[0] == 0
    run(ctx, nnhip, x, counts=-counts, **r)  # negative counts are none


def test_in_place_and_out_only(ctx, nnhip):
    import torch
    rng = np.random.default_rng(8)
    x, counts, r, bias, allowed = make(rng, 2, 40001)
    y, want = rules(x, counts=counts, **r, bias=bias)
    obj = nnhip.LogitRules(40001, counts=dev(counts), bias=dev(bias), **{k: dev(v) for k, v in r.items()})
    L = dev(x)
    assert ctx.logits_adjust_rows(L, obj, out=torch.empty_like(L)) is None
    ids = ctx.logits_adjust_rows(L, obj, ids=torch.zeros(2, dtype=torch.int32, device="cuda"), out=L)
    assert same(host(L), y) and np.array_equal(host(ids), want)


def test_argmax_without_rules(ctx, nnhip):
    rng = np.random.default_rng(9)
    for V in (10, 5000, 50001):
        x = dev(rng.standard_normal((7, V)).astype(np.float32))
        assert np.array_equal(host(ctx.logits_adjust_rows(x)), host(ctx.argmax_rows(x)))


def test_unaligned_and_rows(ctx, nnhip):
    """Operands that start 4 bytes past a 16-byte boundary."""
    import torch
    rng = np.random.default_rng(10)
    x, counts, r, bias, allowed = make(rng, 3, 1001)

    def off(a):
        t = dev(a)
        s = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape)
        return s.copy_(t)

    obj = nnhip.LogitRules(1001, counts=off(counts), bias=off(bias), allowed=off(allowed),
                           **{k: off(v) for k, v in r.items()})
    out = off(np.zeros_like(x))
    ids = ctx.logits_adjust_rows(off(x), obj, ids=off(np.zeros(3, np.int32)), out=out)
    y, want = rules(x, counts=counts, **r, bias=bias, allowed=allowed)
    assert same(host(out), y) and np.array_equal(host(ids), want)


def test_rows_past_32_bits(ctx, nnhip):
    """More than 2^31 logits: the last rows' choices and adjusted logits."""
    import torch
    V, B = 131071, 16500
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.empty(B, V, dtype=torch.float32, device="cuda")
    x.uniform_(-1, 1, generator=g)
    bias = torch.zeros(1, V, dtype=torch.float32, device="cuda")
    bias[0, ::2] = -3.0
    ids = torch.empty(B, dtype=torch.int32, device="cuda")
    ctx.logits_adjust_rows(x, nnhip.LogitRules(V, bias=bias), ids=ids, out=x)
    tail = x[-300:]
    assert torch.equal(ids[-300:].long(), tail.argmax(1)) and bool((ids % 2 == 1).all())
    assert float(tail[:, ::2].max()) <= -2.0 and float(tail[:, ::2].min()) >= -4.0
    assert float(tail[:, 1::2].min()) >= -1.0
    del x, tail
    torch.cuda.empty_cache()


def test_token_counts(ctx, nnhip):
    rng = np.random.default_rng(11)
    lens, V = [0, 1, 700, 0, 33], 50
    cu = np.concatenate(([0], np.cumsum(lens))).astype(np.int32)
    ids = rng.integers(-2, V + 2, int(cu[-1]) + 9).astype(np.int32)
    start = rng.integers(0, 3, (5, V)).astype(np.int32)
    want = start.copy()
    for b in range(5):
        for t in ids[cu[b]:cu[b + 1]]:
            if 0 <= t < V:
                want[b, t] += 1
    assert np.array_equal(host(ctx.token_counts_add(dev(ids), dev(cu), dev(start))), want)


def test_refusals(ctx, nnhip):
    import torch
    i = dict(dtype=torch.int32, device="cuda")
    L = torch.zeros(2, 40, device="cuda")
    counts = torch.zeros(2, 40, **i)
    ok = nnhip.LogitRules(40, counts=counts, count_choice=True)
    ctx.logits_adjust_rows(L, ok, ids=torch.zeros(2, **i))
    bad = [(L, nnhip.LogitRules(41), {}), (torch.zeros(3, 40, device="cuda"), ok, {}), (L.half(), None, {}),
           (L.t(), None, {}), (L, None, dict(ids=torch.zeros(3, **i))), (L, None, dict(out=L[:1])),
           (L, ok, dict(out=torch.empty_like(L))),  # a choice to count, and no ids
           (L, None, dict(out=torch.empty_like(L), pos=torch.zeros(2, **i))), (L.cpu(), None, {}),
           (L, nnhip.LogitRules(40, presence=torch.zeros(2, device="cuda")), {}),
           (L, nnhip.LogitRules(40, count_choice=True), {})]
    for x, r, kw in bad:
        with pytest.raises(nnhip.NNHipError):
            ctx.logits_adjust_rows(x, r, **kw)
    for kw in (dict(counts=torch.zeros(2, 41, **i)), dict(counts=counts.long()), dict(bias=torch.zeros(3, 39, device="cuda")),
               dict(allowed=torch.zeros(2, 1, **i)), dict(counts=counts, repeat=torch.zeros(2, 1, device="cuda"))):
        with pytest.raises(nnhip.NNHipError):
            nnhip.LogitRules(40, **kw)
    with pytest.raises(nnhip.NNHipError):
        ctx.token_counts_add(torch.zeros(3, **i), torch.zeros(2, **i), counts)


def test_captured(nnhip):
    """A captured choice replays with the counts and positions that the replay before left."""
    import torch
    ctx = nnhip.Context(0)
    rng = np.random.default_rng(12)
    B, V = 2, 60000
    x, counts, r, _, _ = make(rng, B, V)
    L, C, pos, ids = dev(x), dev(counts), dev(np.zeros(B, np.int32)), dev(np.zeros(B, np.int32))
    obj = nnhip.LogitRules(V, counts=C, count_choice=True, **{k: dev(v) for k, v in r.items()})
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ctx.logits_adjust_rows(L, obj, ids=ids, pos=pos)
    torch.cuda.synchronize()
    c = host(C).copy()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        ctx.logits_adjust_rows(L, obj, ids=ids, pos=pos)
    for step in range(5):
        g.replay()
        torch.cuda.synchronize()
        _, want = rules(x, counts=c, **r)
        assert np.array_equal(host(ids), want)
        c[np.arange(B), want] += 1
        assert np.array_equal(host(C), c) and np.all(host(pos) == step + 2)
        ctx.argmax_rows(L)
        torch.cuda.synchronize()
    ctx.close()
