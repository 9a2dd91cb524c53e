"""The decoder over paged caches: prompts of unlike lengths in one packed pass, then steps of the whole batch
with a sequence that ends, a slot that stays empty and a sequence that moves in, and the choice under rules.

The int8 stages are the contiguous decoder's (bit-checked elsewhere), so here each block's attention is
held to an evaluation in 64 bits on the block's own q, k and v (the bound of test_gpu_pages.py), the
pools bit for bit, and the ids to the rules on the step's logits."""
import numpy as np
import pytest

from conftest import normal
from test_gpu_logits import rules as apply_rules
from test_gpu_pages import attend64, dev, host, rotate, same
from test_gpu_prefill import _gpu_model

pytestmark = pytest.mark.gpu


class Mirror:
    """The caches of every block on the host, by sequence and position."""

    def __init__(self, nnhip, cfg, L, rows, page, width, f16, rng):
        import torch
        self.cfg, self.page, self.dt = cfg, page, np.float16 if f16 else np.float32
        self.pages = rows * width + 2
        self.table = rng.permutation(self.pages)[:rows * width].astype(np.int32).reshape(rows, width)
        self.table_d = dev(self.table)
        self.cos, self.sin = nnhip.rope_table(cfg.dk, cfg.max_len)
        shape = (self.pages, cfg.Hkv, page, cfg.dk)
        self.k = [np.full(shape, np.nan, self.dt) for _ in range(L)]
        self.v = [np.full(shape, np.nan, self.dt) for _ in range(L)]
        self.caches = [nnhip.KVPages(dev(k), dev(v), self.table_d) for k, v in zip(self.k, self.v)]

    def put(self, i, b, p, k, v):
        cfg = self.cfg
        page, s = self.table[b, p // self.page], p % self.page
        self.k[i][page, :, s] = rotate(k.reshape(cfg.Hkv, cfg.dk), self.cos, self.sin, p).astype(self.dt)
        self.v[i][page, :, s] = v.reshape(cfg.Hkv, cfg.dk).astype(self.dt)

    def check(self, i, b, p, q, a, factor=1):
        cfg = self.cfg
        at = np.arange(p + 1)
        K = self.k[i][self.table[b, at // self.page], :, at % self.page].astype(np.float64)
        V = self.v[i][self.table[b, at // self.page], :, at % self.page].astype(np.float64)
        qr = rotate(q.reshape(cfg.H, cfg.dk).astype(np.float64), self.cos, self.sin, p)
        for h in range(cfg.H):
            g = h // (cfg.H // cfg.Hkv)
            ref, tol = attend64(qr[h], K[:, g], V[:, g], cfg.scale, 0.0, 0.0, at - float(p), np.ones(p + 1, bool))
            assert np.all(np.abs(a.reshape(cfg.H, cfg.dk)[h] - ref) <= factor * tol), f"block {i} b={b} p={p} h={h}"

    def same_pools(self):
        for i, c in enumerate(self.caches):
            assert same(host(c.k), self.k[i]) and same(host(c.v), self.v[i]), f"block {i}: pools differ"


@pytest.mark.parametrize("B,f16,sub", [(4, False, True), (3, True, False), (18, False, True)])
def test_packed_prompts_then_steps(ctx, nnhip, B, f16, sub):
    """B = 18 runs the unfused step."""
    import torch
    from nnhip_py import decoder as dmod
    print(f"paged decoder B={B} f16={f16}", flush=True)
    rng = np.random.default_rng(40 + B)
    cfg = dmod.Config(d=256, H=4, Hkv=2, F=320, vocab=97, max_len=96, act=0, eps=1e-5)
    L, page, width = 2, 16, 6
    base = _gpu_model(ctx, nnhip, cfg, L, B, 0x9A + B, subln=sub)[0]
    m = Mirror(nnhip, cfg, L, B, page, width, f16, rng)
    dec = dmod.Decoder(ctx, cfg, base.blocks, base.emb, base.g_final, base.head, B, caches=m.caches)
    lens = [int(x) for x in rng.integers(1, 60, B)]
    lens[0], lens[-1] = 33, 1
    cu = np.concatenate(([0], np.cumsum(lens))).astype(np.int32)
    M = int(cu[-1])
    prompt = rng.integers(0, cfg.vocab, M).astype(np.int32)
    seen = {}

    def hook(i, name, t):
        seen[i, name] = host(t)

    logits, ids = dec.prefill_packed(dev(prompt), dev(cu), max(lens), hook=hook)
    first = host(ids).copy()
    assert np.array_equal(first, host(logits).argmax(0))
    for i in range(L):
        for b in range(B):
            for t in range(lens[b]):
                c = cu[b] + t
                m.put(i, b, t, seen[i, "k"][:, c], seen[i, "v"][:, c])
            for t in sorted({0, lens[b] // 2, lens[b] - 1}):
                m.check(i, b, t, seen[i, "q"][:, cu[b] + t], seen[i, "a"][:, cu[b] + t], factor=4)
    m.same_pools()

    # steps under penalties and a grammar that forbids the even tokens; sequence 1 ends after the first
    counts = np.zeros((B, cfg.vocab), np.int32)
    for b in range(B):
        np.add.at(counts[b], prompt[cu[b]:cu[b + 1]], 1)
    counts_d = torch.zeros(B, cfg.vocab, dtype=torch.int32, device="cuda")
    ctx.token_counts_add(dev(prompt), dev(cu), counts_d)
    assert np.array_equal(host(counts_d), counts)
    kw = dict(repeat=np.full(B, 1.3, np.float32), presence=np.full(B, 0.2, np.float32),
              frequency=np.full(B, 0.1, np.float32), allowed=np.full((1, 4), 0xAAAAAAAA, np.uint32))
    rule = nnhip.LogitRules(cfg.vocab, counts=counts_d, count_choice=True, **{k: dev(v.view(np.int32) if v.dtype == np.uint32
                                                                                      else v) for k, v in kw.items()})
    pos = np.array(lens, np.int32)
    ids_d, pos_d = dev(first), dev(pos)
    for step in range(4):
        if step == 1:
            pos[1] = -1
            pos_d[1] = -1
        if step == 3:  # another sequence moves into the slot (and its pages), at position 0
            pos[1] = 0
            pos_d[1] = 0

        def attn_hook(i, a):
            tm = dec._tok and dec.fused_ok()
            q, k, v = (host(x) if tm else host(y).T for x, y in
                       (((dec.q_t if dec._tok else dec.q), dec.q), ((dec.k_t if dec._tok else dec.k), dec.k),
                        ((dec.v_t if dec._tok else dec.v), dec.v)))
            a = host(a).T
            for b in range(B):
                if pos[b] < 0:
                    assert np.all(a[b] == 0)
                    continue
                m.put(i, b, pos[b], k[b], v[b])
                m.check(i, b, pos[b], q[b], a[b])

        logits, got = dec.step(ids_d, pos_d, cfg.max_len, attn_hook=attn_hook, advance=True, rules=rule)
        y, want = apply_rules(host(logits).T.copy(), counts=counts, **kw)
        live = pos >= 0
        assert np.array_equal(host(got), want) and np.all(want % 2 == 1)
        counts[np.flatnonzero(live), want[live]] += 1
        pos[live] += 1
        assert np.array_equal(host(pos_d), pos) and np.array_equal(host(counts_d), counts)
        m.same_pools()


def test_packed_prompts_with_empty_slots(ctx, nnhip):
    """Slots without new tokens (the first and the last among them) beside prompts: the prompts' logits, ids and
    cached rows are those of a call of all slots, the empty slots' pages stay."""
    import torch
    from nnhip_py import decoder as dmod
    rng = np.random.default_rng(77)
    cfg = dmod.Config(d=256, H=4, Hkv=2, F=320, vocab=97, max_len=96, act=0, eps=1e-5)
    B, L, lens = 5, 2, [7, 20, 3, 33, 1]
    base = _gpu_model(ctx, nnhip, cfg, L, B, 0x9F, subln=True)[0]
    ids = [rng.integers(0, cfg.vocab, n).astype(np.int32) for n in lens]
    found = []
    for live in ([0, 1, 2, 3, 4], [1, 3]):
        m = Mirror(nnhip, cfg, L, B, 16, 6, False, np.random.default_rng(5))
        dec = dmod.Decoder(ctx, cfg, base.blocks, base.emb, base.g_final, base.head, B, caches=m.caches)
        n = [len(ids[b]) if b in live else 0 for b in range(B)]
        cu = np.concatenate(([0], np.cumsum(n))).astype(np.int32)
        logits, got = dec.prefill_packed(dev(np.concatenate([ids[b] for b in live])), dev(cu), max(n))
        found.append((host(logits)[:, [1, 3]].copy(), host(got)[[1, 3]].copy(), [(host(c.k), host(c.v)) for c in m.caches]))
    assert np.array_equal(found[0][0], found[1][0]) and np.array_equal(found[0][1], found[1][1])
    for (k0, v0), (k1, v1) in zip(found[0][2], found[1][2]):
        for b in range(B):
            for t in range(lens[b]):
                page, s = m.table[b, t // 16], t % 16
                for x, y in ((k0, k1), (v0, v1)):
                    if b in (1, 3):
                        assert same(x[page, :, s], y[page, :, s])
                    else:
                        assert np.all(np.isnan(y[page, :, s]))


def test_captured_step(nnhip):
    """A step over paged caches with its choice, captured once and replayed between eager work, continues as
    the eager steps do."""
    import torch
    from nnhip_py import decoder as dmod
    ctx = nnhip.Context(0)
    rng = np.random.default_rng(50)
    cfg = dmod.Config(d=256, H=4, Hkv=1, F=320, vocab=97, max_len=320, act=1, eps=1e-5)
    B = 3
    base = _gpu_model(ctx, nnhip, cfg, 2, B, 0xCA9)[0]
    runs = []
    for captured in (False, True):
        m = Mirror(nnhip, cfg, 2, B, 16, 20, False, np.random.default_rng(51))
        dec = dmod.Decoder(ctx, cfg, base.blocks, base.emb, base.g_final, base.head, B, caches=m.caches)
        lens = [250, 3, 127]
        cu = np.concatenate(([0], np.cumsum(lens))).astype(np.int32)
        prompt = dev(np.random.default_rng(52).integers(0, 97, int(cu[-1])).astype(np.int32))
        counts = torch.zeros(B, 97, dtype=torch.int32, device="cuda")
        rule = nnhip.LogitRules(97, counts=counts, repeat=dev(np.full(B, 1.2, np.float32)), count_choice=True)
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            _, ids = dec.prefill_packed(prompt, dev(cu), 250)
            ids, pos = ids.clone(), dev(np.array(lens, np.int32))
            dec.step(ids, pos, cfg.max_len, advance=True, rules=rule)
        torch.cuda.synchronize()
        trace = [host(ids).copy()]
        if captured:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                dec.step(ids, pos, cfg.max_len, advance=True, rules=rule)
        for i in range(6):
            if captured:
                g.replay()
            else:
                with torch.cuda.stream(side):
                    dec.step(ids, pos, cfg.max_len, advance=True, rules=rule)
            torch.cuda.synchronize()
            ctx.argmax_rows(torch.randn(3, 50, device="cuda"))
            trace.append(host(ids).copy())
        runs.append((np.array(trace), host(pos).copy(), host(counts).copy(), host(m.caches[1].k)))
    for a, b in zip(*runs):
        assert np.array_equal(a, b, equal_nan=a.dtype.kind == "f")
    ctx.close()


def test_refusals(ctx, nnhip):
    import torch
    from nnhip_py import decoder as dmod
    rng = np.random.default_rng(60)
    cfg = dmod.Config(d=256, H=4, Hkv=2, F=320, vocab=97, max_len=96, act=0, eps=1e-5)
    base = _gpu_model(ctx, nnhip, cfg, 1, 2, 0x77)[0]
    ids = torch.zeros(4, dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda")
    with pytest.raises(nnhip.NNHipError, match="paged"):
        base.prefill_packed(ids, cu, 2)
    m = Mirror(nnhip, cfg, 1, 2, 16, 6, False, rng)
    dec = dmod.Decoder(ctx, cfg, base.blocks, base.emb, base.g_final, base.head, 2, caches=m.caches)
    with pytest.raises(nnhip.NNHipError, match="prefill_packed"):
        dec.prefill(ids, 2)
    with pytest.raises(nnhip.NNHipError, match="cu"):
        dec.prefill_packed(ids, cu[:2].contiguous(), 2)
    dec.prefill_packed(ids, cu, 2)
    with pytest.raises(nnhip.NNHipError, match="len_bound"):
        dec.step(ids[:2].contiguous(), torch.zeros(2, dtype=torch.int32, device="cuda"), 97)
