"""The decoder where the choice or the batch is at an edge, over paged and contiguous caches."""
import numpy as np
import pytest

from test_gpu_logits import rules as apply_rules
from test_gpu_pages import dev, host, same
from test_gpu_pages_decoder import Mirror
from test_gpu_prefill import _gpu_model

pytestmark = pytest.mark.gpu


def model(ctx, nnhip, B, seed, **kw):
    from nnhip_py import decoder as dmod
    cfg = dmod.Config(**{**dict(d=256, H=4, Hkv=2, F=320, vocab=97, max_len=96, act=0, eps=1e-5), **kw})
    return cfg, _gpu_model(ctx, nnhip, cfg, 2, B, seed, subln=True)[0]


def decoder(ctx, nnhip, cfg, base, B, paged=True, page=16, seed=5):
    from nnhip_py import decoder as dmod
    if not paged:
        return dmod.Decoder(ctx, cfg, base.blocks, base.emb, base.g_final, base.head, B)
    m = Mirror(nnhip, cfg, 2, B, page, -(-cfg.max_len // page), False, np.random.default_rng(seed))
    return dmod.Decoder(ctx, cfg, base.blocks, base.emb, base.g_final, base.head, B, caches=m.caches)


def cached(dec, b, n):
    """The cached keys and values of sequence b's first n positions (one page's at most), block by block."""
    if dec.paged:
        return [np.ascontiguousarray(host(t)[host(c.table)[b, 0], :, :n]) for c in dec.caches for t in (c.k, c.v)]
    return [host(t)[b, :n].copy() for c in dec.caches for t in c]


@pytest.mark.parametrize("paged", [True, False])
@pytest.mark.parametrize("B", [3, 18])
def test_step_where_nothing_is_allowed(ctx, nnhip, B, paged):
    """A sequence whose mask allows nothing gets the choice -1 and stays as it is, its input token too: the steps after
    it find the same state (pools, logits and counts bit for bit), and it goes on once tokens are allowed. The
    other sequences are not touched by it. B = 18 runs the unfused step."""
    import torch
    print(f"nothing allowed B={B} paged={paged}", flush=True)
    cfg, base = model(ctx, nnhip, B, 0xB0 + B)
    dec = decoder(ctx, nnhip, cfg, base, B, paged)
    counts = torch.zeros(B, cfg.vocab, dtype=torch.int32, device="cuda")
    words = torch.full((B, 4), -1, dtype=torch.int32, device="cuda")
    rule = nnhip.LogitRules(cfg.vocab, counts=counts, repeat=dev(np.full(B, 1.2, np.float32)), allowed=words,
                            count_choice=True)
    ids = dev(np.arange(B, dtype=np.int32) + 1)
    pos = torch.zeros(B, dtype=torch.int32, device="cuda")
    for _ in range(3):
        dec.step(ids, pos, cfg.max_len, advance=True, rules=rule)
    words[1] = 0
    start = host(ids).copy(), host(pos).copy(), host(counts).copy()
    seen = []
    for i in range(3):
        before = host(ids).copy(), host(pos).copy()
        logits, got = dec.step(ids, pos, cfg.max_len, advance=True, rules=rule)
        got, rest = host(got), [b for b in range(B) if b != 1]
        assert got[1] == -1 and np.all(got[rest] >= 0)
        assert host(ids)[1] == start[0][1] and np.array_equal(host(ids)[rest], got[rest])
        assert host(pos)[1] == 3 and np.array_equal(host(pos)[rest], before[1][rest] + 1)
        assert np.array_equal(host(counts)[1], start[2][1])
        seen.append((host(logits)[:, 1].copy(), cached(dec, 1, 4)))
    for x, rows in seen:
        assert np.all(np.isfinite(x)) and np.array_equal(x, seen[0][0])
        assert all(np.all(np.isfinite(a)) and same(a, b) for a, b in zip(rows, seen[0][1]))
    words[1] = -1
    logits, got = dec.step(ids, pos, cfg.max_len, advance=True, rules=rule)
    assert np.array_equal(host(logits)[:, 1], seen[0][0])
    want = apply_rules(seen[0][0][None].copy(), counts=start[2][1:2], repeat=np.full(1, 1.2, np.float32))[1]
    assert host(got)[1] == want[0] == host(ids)[1] and host(pos)[1] == 4


def test_captured_step_where_nothing_is_allowed(nnhip):
    """The same in a captured step, whose input is the ids it replays into."""
    import torch
    ctx = nnhip.Context(0)
    cfg, base = model(ctx, nnhip, 3, 0xB7)
    runs = []
    for captured in (False, True):
        dec = decoder(ctx, nnhip, cfg, base, 3)
        words = torch.full((3, 4), -1, dtype=torch.int32, device="cuda")
        rule = nnhip.LogitRules(cfg.vocab, allowed=words)
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            _, ids = dec.prefill_packed(dev(np.arange(9, dtype=np.int32)), dev(np.array([0, 2, 5, 9], np.int32)), 4)
            pos = dev(np.array([2, 3, 4], np.int32))
            _, got = dec.step(ids, pos, cfg.max_len, advance=True, rules=rule)
        torch.cuda.synchronize()
        if captured:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                _, got = dec.step(ids, pos, cfg.max_len, advance=True, rules=rule)
        trace = []
        for i in range(6):
            words[2] = 0 if i in (1, 2, 4) else -1
            torch.cuda.synchronize()
            if captured:
                g.replay()
            else:
                with torch.cuda.stream(side):
                    _, got = dec.step(ids, pos, cfg.max_len, advance=True, rules=rule)
            torch.cuda.synchronize()
            assert (host(got)[2] == -1) == (i in (1, 2, 4))
            trace.append(np.concatenate((host(got), host(ids), host(pos))))
        runs.append(np.array(trace))
    assert np.array_equal(*runs)
    ctx.close()


@pytest.mark.parametrize("advance", [False, True])
@pytest.mark.parametrize("B", [3, 18])
def test_empty_slot_is_not_counted(ctx, nnhip, B, advance):
    """A step counts the choices of live sequences only, whether or not it advances them."""
    import torch
    print(f"empty slot B={B} advance={advance}", flush=True)
    cfg, base = model(ctx, nnhip, B, 0xC0 + B)
    dec = decoder(ctx, nnhip, cfg, base, B)
    counts = torch.zeros(B, cfg.vocab, dtype=torch.int32, device="cuda")
    rule = nnhip.LogitRules(cfg.vocab, counts=counts, repeat=dev(np.full(B, 1.2, np.float32)), count_choice=True)
    pos = np.zeros(B, np.int32)
    pos[[0, B - 1]] = -1, -5
    pos_d, ids = dev(pos), dev(np.arange(B, dtype=np.int32))
    _, got = dec.step(ids, pos_d, cfg.max_len, advance=advance, rules=rule)
    want = np.zeros((B, cfg.vocab), np.int32)
    live = np.flatnonzero(pos >= 0)
    want[live, host(got)[live]] = 1
    assert np.array_equal(host(counts), want)
    assert np.array_equal(host(pos_d), np.where(pos >= 0, pos + advance, pos))


def scribble():
    """NaN into whatever the allocators hand out next, small and large."""
    import torch
    return [torch.full((n,), float("nan"), device="cuda") for n in [1 << 8, 1 << 16, 1 << 18, 1 << 20, 1 << 24] * 4]


@pytest.mark.parametrize("paged", [True, False])
def test_captured_step_beside_larger_calls(nnhip, paged):
    """A captured step of 18 sequences (whose feed-forward block uses the context's workspace) goes on as eager steps do
    after eager prompts that outgrow that workspace: the captured calls keep theirs."""
    import torch
    print(f"captured step beside larger calls paged={paged}", flush=True)
    ctx = nnhip.Context(0)
    B = 18
    cfg, base = model(ctx, nnhip, B, 0xF1, max_len=512)
    assert nnhip.lib().nnhip_ffn_glu_workspace_bytes(cfg.d, cfg.F, 400 * B) > 1 << 20  # what it starts with
    runs = []
    for captured in (True, False):
        dec, other = (decoder(ctx, nnhip, cfg, base, B, paged, seed=s) for s in (5, 6))
        ids, pos = dev(np.arange(B, dtype=np.int32)), torch.zeros(B, dtype=torch.int32, device="cuda")
        side = torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            dec.step(ids, pos, cfg.max_len, advance=True)
        torch.cuda.synchronize()
        if captured:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                dec.step(ids, pos, cfg.max_len, advance=True)
        trace, kept = [], []
        for i in range(6):
            if i in (1, 3):
                T = 400 if i == 1 else 510
                prompt = dev(np.arange(B * T, dtype=np.int32) % cfg.vocab)
                if paged:
                    other.prefill_packed(prompt, dev(np.arange(B + 1, dtype=np.int32) * T), T)
                else:
                    other.prefill(prompt, T)
                torch.cuda.synchronize()
                kept.append(scribble())
            if captured:
                g.replay()
            else:
                with torch.cuda.stream(side):
                    dec.step(ids, pos, cfg.max_len, advance=True)
            torch.cuda.synchronize()
            trace.append(np.concatenate((host(ids), host(pos))))
        runs.append(np.array(trace))
    assert np.array_equal(*runs)
    ctx.close()


def test_captured_attention_beside_larger_calls(nnhip):
    """The same for the scratch of the attention over contiguous caches; a capture that would have to grow a
    workspace is refused, and the calls after it work."""
    import torch
    ctx = nnhip.Context(0)
    H, Hkv, dk = 8, 2, 64

    def problem(B, n):
        x = [torch.randn(B, h * dk, device="cuda") for h in (H, Hkv, Hkv)]
        caches = [torch.randn(B, n, Hkv * dk, device="cuda") for _ in range(2)]
        return x, torch.full((B,), n - 1, dtype=torch.int32, device="cuda"), n, caches, torch.empty(B, H * dk, device="cuda")

    def call(p):
        x, pos, n, (kc, vc), out = p
        return ctx.attention_decode(*x, H, Hkv, dk, pos, n, kc, vc, 0.125, None, None, out=out, tokens=True)

    small, large = problem(2, 2000), problem(9, 9000)
    assert 0 < nnhip.attention_workspace_bytes(2, H, Hkv, dk, 2000) < nnhip.attention_workspace_bytes(9, H, Hkv, dk, 9000)
    fresh, g0 = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with pytest.raises(nnhip.NNHipError, match="capture"):
        with torch.cuda.graph(g0, stream=fresh):
            small[4].zero_()
            call(small)
    want = call(small).clone()
    side, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=side):
        call(small)
    kept = []
    for i in range(4):
        if i == 1:
            call(large)
            torch.cuda.synchronize()
            kept.append(scribble())
        small[4].zero_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(small[4], want)
    ctx.close()


@pytest.mark.parametrize("paged", [True, False])
def test_captured_prompt_beside_others(nnhip, paged):
    """A captured prompt (the chunks of a server's loop) replays beside eager ones of fewer and of more tokens, which need
    other views of the decoder's scratch, and larger ones: the logits, ids and cached rows of an eager run."""
    import torch
    print(f"captured prompt beside others paged={paged}", flush=True)
    ctx = nnhip.Context(0)
    B, T = 3, 40
    cfg, base = model(ctx, nnhip, B, 0xF7, max_len=600)
    runs = []
    for captured in (True, False):
        dec = decoder(ctx, nnhip, cfg, base, B, paged, page=64)

        def prompt(ids, n, T):
            if paged:
                return dec.prefill_packed(ids, n, T)
            return dec.prefill(ids, T)

        ids = torch.zeros(B * T, dtype=torch.int32, device="cuda")
        n = dev(np.array([0, 7, 40, B * T], np.int32))
        bound = 80 if paged else T
        side = torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            prompt(ids, n, bound)
        torch.cuda.synchronize()
        if captured:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                logits, got = prompt(ids, n, bound)
        trace, kept = [], []
        for i, other in enumerate((None, 9, None, 200, 501, None, 300)):
            if other:  # an eager prompt of other sizes
                x = dev((np.arange(B * other, dtype=np.int32) * 5 + i) % cfg.vocab)
                prompt(x, dev(np.arange(B + 1, dtype=np.int32) * other), other)
                torch.cuda.synchronize()
                kept.append(scribble())
            ids.copy_(dev((np.arange(B * T, dtype=np.int32) * 3 + i) % cfg.vocab))
            torch.cuda.synchronize()
            if captured:
                g.replay()
            else:
                with torch.cuda.stream(side):
                    logits, got = prompt(ids, n, bound)
            torch.cuda.synchronize()
            trace.append((host(logits).copy(), host(got).copy(), cached(dec, 2, 40)))
        runs.append(trace)
    for (x0, i0, c0), (x1, i1, c1) in zip(*runs):
        assert np.all(np.isfinite(x0)) and np.array_equal(x0, x1) and np.array_equal(i0, i1)
        assert all(same(a, b) for a, b in zip(c0, c1))
    ctx.close()


def test_first_token_under_rules(ctx, nnhip):
    """prefill_packed's choice under rules: penalties, bias and masks as step()'s, the chosen tokens counted,
    nothing counted for a slot without tokens; the ids go on into steps."""
    import torch
    B = 5
    cfg, base = model(ctx, nnhip, B, 0xD1)
    lens = [7, 0, 20, 1, 0]
    rng = np.random.default_rng(3)
    cu = np.concatenate(([0], np.cumsum(lens))).astype(np.int32)
    prompt = rng.integers(0, cfg.vocab, int(cu[-1])).astype(np.int32)
    live = np.flatnonzero(lens)
    counts = np.zeros((B, cfg.vocab), np.int32)
    for b in range(B):
        np.add.at(counts[b], prompt[cu[b]:cu[b + 1]], 1)
    kw = dict(repeat=np.full(B, 1.5, np.float32), presence=np.full(B, 0.3, np.float32),
              frequency=np.full(B, 0.2, np.float32), bias=rng.standard_normal((1, cfg.vocab)).astype(np.float32))
    words = np.full((B, 4), 0xAAAAAAAA, np.uint32)
    words[3] = 0  # nothing is allowed
    dec = decoder(ctx, nnhip, cfg, base, B)
    counts_d = torch.zeros(B, cfg.vocab, dtype=torch.int32, device="cuda")
    ctx.token_counts_add(dev(prompt), dev(cu), counts_d)
    words_d = dev(words.view(np.int32))
    rule = nnhip.LogitRules(cfg.vocab, counts=counts_d, count_choice=True, allowed=words_d,
                            **{k: dev(v) for k, v in kw.items()})
    logits, ids = dec.prefill_packed(dev(prompt), dev(cu), 20, rules=rule)
    want = apply_rules(host(logits).T.copy(), counts=counts, allowed=words, **kw)[1]
    got = host(ids).copy()
    assert np.array_equal(got[live], want[live]) and got[3] == -1 and np.all(got[[0, 2]] % 2 == 1)
    for b in (0, 2):
        counts[b, got[b]] += 1
    assert np.array_equal(host(counts_d), counts)
    plain = decoder(ctx, nnhip, cfg, base, B)
    same_logits, free = plain.prefill_packed(dev(prompt), dev(cu), 20)
    assert np.array_equal(host(same_logits)[:, live], host(logits)[:, live])
    assert np.array_equal(host(free)[live], host(logits).argmax(0)[live])


def test_first_token_under_rules_of_equal_prompts(ctx, nnhip):
    """The same for prefill() into contiguous caches."""
    import torch
    B, T = 3, 11
    cfg, base = model(ctx, nnhip, B, 0xD3)
    prompt = np.random.default_rng(4).integers(0, cfg.vocab, (B, T)).astype(np.int32)
    counts = np.stack([np.bincount(x, minlength=cfg.vocab) for x in prompt]).astype(np.int32)
    words, repeat = np.full((1, 4), 0x55555555, np.uint32), np.full(B, 1.5, np.float32)
    counts_d = dev(counts)
    rule = nnhip.LogitRules(cfg.vocab, counts=counts_d, repeat=dev(repeat), allowed=dev(words.view(np.int32)), count_choice=True)
    logits, ids = decoder(ctx, nnhip, cfg, base, B, paged=False).prefill(dev(prompt.reshape(-1)), T, rules=rule)
    want = apply_rules(host(logits).T.copy(), counts=counts, repeat=repeat, allowed=words)[1]
    assert np.array_equal(host(ids), want) and np.all(want % 2 == 0)
    counts[np.arange(B), want] += 1
    assert np.array_equal(host(counts_d), counts)


def test_prompt_bound_past_the_tokens(ctx, nnhip):
    """t_bound only bounds the sequences' tokens: a constant one of a server is no error for a short packing."""
    cfg, base = model(ctx, nnhip, 2, 0xE1)
    ids, cu = dev(np.arange(5, dtype=np.int32)), dev(np.array([0, 2, 5], np.int32))
    outs = [decoder(ctx, nnhip, cfg, base, 2).prefill_packed(ids, cu, t) for t in (3, 5, 6, 4096)]
    for logits, got in outs[1:]:
        assert np.array_equal(host(logits), host(outs[0][0])) and np.array_equal(host(got), host(outs[0][1]))


def test_prompts_without_tokens_are_refused(ctx, nnhip):
    cfg, base = model(ctx, nnhip, 2, 0xE5)
    none, cu = dev(np.zeros(0, np.int32)), dev(np.zeros(3, np.int32))
    with pytest.raises(nnhip.NNHipError, match="token"):
        decoder(ctx, nnhip, cfg, base, 2, paged=False).prefill(none, 0)
    with pytest.raises(nnhip.NNHipError, match="token"):
        decoder(ctx, nnhip, cfg, base, 2).prefill_packed(none, cu, 0)
