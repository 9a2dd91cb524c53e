"""Performance cases of the operators around a paged KV cache held in 8 bits: the cache itself (fill and
read, decode attention, prompt attention), norms of queries and keys with the rotation, and the page tables
and slot maps that a server keeps on the GPU.

A case is a dict of plain values with an "op":

  decode   one new token for each of B sequences (the last `idle` of them without one) over an 8-bit cache:
           rotation, quantized append, attention; positions spread from lo to hi. Returned beside the
           outputs: the values of the block of tokens that each new one has joined, all that a call changes
  prompt   attention of packed prompts (lo to hi tokens each, `past` positions before them) over an 8-bit
           cache that holds their keys; causal, or with a bidirectional prefix
  fill     the keys and values of packed tokens rotated, quantized and written behind `past` positions, then
           the values of those tokens and of the block before read back from the cache
  qk       RMSNorm of every head of queries and keys, and the rotation at each token's position
  tables   pages from a free list for the sequences' new tokens, positions and slots of those, and
           the tokens taken back again (`scarce`: the list does not reach for all)

An 8-bit cache holds int8 codes and one f32 scale for every `block` tokens of a head: the scale is the largest
magnitude * fl(1/127), a code the value over the scale rounded half away from zero. A token that joins a
block with a larger value than its scale holds raises the scale, and the block's older values are quantized
again. cap > 0 caps the scores by a tanh; alibi adds a bias that falls with the distance. The shapes are those
of bench.py's decoder (20 heads over 5 KV heads of 128) and generic ones. With `own` false, run()
computes everything by elementary torch operations; with it, by the framework.
"""
import importlib.util
import math
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda"

own = False


def _pkg():
    """The repository's package (its folder name holds a dot, so it is loaded by path)."""
    name = "nnhip_py"
    if name not in sys.modules:
        path = os.path.join(ROOT, "neuralnet.cpp_amd")
        spec = importlib.util.spec_from_file_location(name, os.path.join(path, "__init__.py"),
                                                      submodule_search_locations=[path])
        mod = importlib.util.module_from_spec(spec)
        sys.modules[name] = mod
        spec.loader.exec_module(mod)
    return sys.modules[name]


_context = []


def _ctx():
    if not _context:
        _context.append(_pkg().Context(0))
    return _context[0]


# ------------------------------------------------------------------------------------------ cases

def listed():
    return [
        # one user's chat: a single token over a short cache, where the call's latency counts
        dict(name="decode_1", op="decode", B=1, idle=0, H=20, Hkv=5, dk=128, page=16, block=16, lo=100, hi=100,
             cap=0.0, alibi=False),
        # a server's batch at the decoder benchmark's heads: unlike lengths, two empty slots, capped and biased
        dict(name="decode_16", op="decode", B=16, idle=2, H=20, Hkv=5, dk=128, page=64, block=32, lo=64, hi=4200,
             cap=30.0, alibi=True),
        # long documents: few sequences, caches of up to 128 K positions, 8 heads to a KV head
        dict(name="decode_long", op="decode", B=6, idle=0, H=32, Hkv=4, dk=128, page=64, block=64, lo=50000,
             hi=131072, cap=0.0, alibi=False),
        # short turns of three chats over what they have said: latency
        dict(name="prompt_short", op="prompt", B=3, H=20, Hkv=5, dk=128, page=16, block=16, lo=5, hi=40, past=200,
             cap=0.0, alibi=False, prefix=0),
        # packed prompts of unlike lengths, heads of 64, with a bidirectional prefix of 200 tokens, capped and
        # biased
        dict(name="prompt_packed", op="prompt", B=8, H=16, Hkv=2, dk=64, page=32, block=32, lo=77, hi=1900, past=0,
             cap=50.0, alibi=True, prefix=200),
        # a chunk of long prompts, whose first 6144 positions are cached already
        dict(name="prompt_chunk", op="prompt", B=4, H=20, Hkv=5, dk=128, page=64, block=64, lo=700, hi=1024, past=6144,
             cap=0.0, alibi=False, prefix=0),
        # a few drafted tokens of each sequence of a batch, behind a position inside a block
        dict(name="fill_drafts", op="fill", B=16, Hkv=5, dk=128, page=64, block=32, lo=1, hi=8, past=507),
        # a full prompt batch of the decoder benchmark, ragged
        dict(name="fill_prompts", op="fill", B=16, Hkv=5, dk=128, page=64, block=64, lo=1111, hi=2048, past=0),
        # the queries and keys of a decode step
        dict(name="qk_step", op="qk", B=16, H=20, Hkv=5, dk=128, lo=1, hi=1, past=2111, tokens=True),
        # those of a prompt batch, feature-major as the projections leave them
        dict(name="qk_prompts", op="qk", B=16, H=20, Hkv=5, dk=128, lo=1111, hi=2048, past=0, tokens=False),
        # a decode step of a small server
        dict(name="tables_step", op="tables", B=16, page=64, lo=64, hi=4200, add_lo=1, add_hi=1, scarce=False),
        # a large server takes in prompts beside its running sequences, more than there are pages for
        dict(name="tables_admit", op="tables", B=2000, page=16, lo=1, hi=3000, add_lo=1, add_hi=900, scarce=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _span(rng, lo, hi):
    """A range of lengths: all alike, or spread."""
    a, b = sorted((_log(rng, lo, hi), _log(rng, lo, hi)))
    return (b, b) if rng.random() < 0.3 else (a, b)


def draw(rng):
    op = rng.choice(["decode", "decode", "prompt", "prompt", "fill", "qk", "tables"])
    page = rng.choice([16, 32, 64, 128])
    block = rng.choice([b for b in (16, 32, 64) if b <= page])
    if op == "decode":
        H, Hkv, dk = rng.choice([(20, 5, 128), (16, 16, 64), (16, 2, 64), (32, 8, 128), (8, 1, 256), (12, 4, 128),
                                 (24, 2, 64), (7, 7, 128)])
        B = _log(rng, 1, 64)
        most = max(16, min(131072, 400_000_000 // (B * Hkv * dk * 2)))  # positions within about 0.4 GB of caches
        lo, hi = _span(rng, 1, most)
        return dict(op=op, B=B, idle=rng.choice([0, 0, B // 4]), H=H, Hkv=Hkv, dk=dk, page=page, block=block, lo=lo, hi=hi,
                    cap=rng.choice([0.0, 0.0, 20.0, 50.0]), alibi=rng.random() < 0.3)
    if op == "prompt":
        H, Hkv, dk = rng.choice([(20, 5, 128), (16, 2, 64), (8, 8, 64), (16, 8, 128)])
        B = _log(rng, 1, 8)
        lo, hi = _span(rng, 1, 1024)
        past = rng.choice([0, 0, _log(rng, 1, 4000)])
        return dict(op=op, B=B, H=H, Hkv=Hkv, dk=dk, page=page, block=block, lo=lo, hi=hi, past=past,
                    cap=rng.choice([0.0, 0.0, 20.0, 50.0]), alibi=rng.random() < 0.3,
                    prefix=rng.choice([0, 0, past + _log(rng, 1, 600)]))
    if op == "fill":
        B = _log(rng, 1, 16)
        lo, hi = _span(rng, 1, 2048)
        return dict(op=op, B=B, Hkv=rng.choice([1, 2, 5, 8]), dk=rng.choice([64, 128, 256]), page=page, block=block, lo=lo,
                    hi=hi, past=rng.choice([0, _log(rng, 1, 4000)]))
    if op == "qk":
        H, Hkv, dk = rng.choice([(20, 5, 128), (16, 2, 64), (8, 1, 256), (7, 7, 128)])
        lo, hi = _span(rng, 1, 2048)
        return dict(op=op, B=_log(rng, 1, 16), H=H, Hkv=Hkv, dk=dk, lo=lo, hi=hi, past=rng.choice([0, _log(rng, 1, 60000)]),
                    tokens=rng.random() < 0.5)
    lo, hi = _span(rng, 1, 8192)
    add_lo, add_hi = _span(rng, 1, 700)
    return dict(op=op, B=_log(rng, 1, 2000), page=page, lo=lo, hi=hi, add_lo=add_lo, add_hi=add_hi,
                scarce=rng.random() < 0.5)


def _spread(lo, hi, n):
    """n lengths from lo to hi, spread over their logarithm in a fixed order, the longest among them."""
    got = [int(round(lo * (hi / lo) ** ((0.5 + 0.6180339887 * i) % 1.0))) for i in range(n)]
    got[n // 2] = hi
    return got


def _new_tokens(c):
    """Tokens of each sequence that the call works on."""
    return _spread(c["lo"], c["hi"], c["B"])


def _live(c):
    """decode: lengths with the new token, 0 for empty slots."""
    return [x if i < c["B"] - c["idle"] else 0 for i, x in enumerate(_new_tokens(c))]


def _visible(c, n):
    """Pairs of a prompt's query and a key that it sees, for a sequence of n new tokens."""
    past, pre = c["past"], min(c["prefix"], c["past"] + n)
    full = n * past + n * (n + 1) // 2
    # query t sees max(past + t + 1, pre) keys
    short = max(0, pre - past - 1)  # queries whose causal reach is below the prefix
    short = min(short, n)
    return full + sum(pre - (past + t + 1) for t in range(short))


# ------------------------------------------------------------------------------------------ inputs

def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _offsets(n):
    """(0, n[0], n[0] + n[1], ...)"""
    got = [0]
    for x in n:
        got.append(got[-1] + x)
    return _ints(got)


def _tables(rows, dk):
    """cos and sin of position / 10000^(2j/dk), (rows, dk/2)."""
    theta = torch.arange(rows, device=DEV, dtype=torch.float64)[:, None] / torch.pow(
        torch.tensor(10000.0, device=DEV, dtype=torch.float64),
        torch.arange(0, dk, 2, device=DEV, dtype=torch.float64) / dk)[None, :]
    return theta.cos().float(), theta.sin().float()


def _cache(g, c, lens):
    """Pools of codes with every page of the sequences at a place of its own among a tenth more, their scales, and
    the page table (-1 behind a sequence's last page). Codes are those of normal values: one in 16 tokens or so
    reaches the largest."""
    page, B, Hkv, dk = c["page"], len(lens), c["Hkv"], c["dk"]
    need = [-(-n // page) for n in lens]
    total = sum(need) + max(1, sum(need) // 10)

    def codes(*shape):
        x = torch.randn(total, Hkv, page // 16, *shape, generator=g, device=DEV, dtype=torch.float16)
        return x.mul_(38.0).round_().clamp_(-127.0, 127.0).to(torch.int8)

    def scales():
        return (0.8 + 0.4 * torch.rand(total, Hkv, page // c["block"], generator=g, device=DEV)) / 38.0

    k, v = codes(dk // 16, 16, 16), codes(dk, 16)
    places = torch.randperm(total, generator=g, device=DEV).int()
    table = torch.full((B, max(1, max(need))), -1, dtype=torch.int32, device=DEV)
    valid = torch.arange(table.shape[1], device=DEV)[None, :] < torch.tensor(need, device=DEV)[:, None]
    table[valid] = places[:sum(need)]
    return k, v, scales(), scales(), table


def _slopes(H):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)], device=DEV)


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = dict(c)
    n = _new_tokens(c)
    if c["op"] == "tables":
        return _prepare_tables(s, g, n)
    if c["op"] == "qk":
        M = sum(n)
        lay = (lambda h: (M, h * c["dk"])) if c["tokens"] else (lambda h: (h * c["dk"], M))
        # projections of unlike size in each head, as trained ones are
        s["q"], s["k"] = (_normal(g, *lay(h)) * 3.0 for h in (c["H"], c["Hkv"]))
        s["gq"], s["gk"] = (1.0 + 0.2 * _normal(g, c["dk"]) for _ in range(2))
        s["pos"] = torch.cat([torch.arange(c["past"], c["past"] + x, device=DEV) for x in n]).int()
        s["cos"], s["sin"] = _tables(c["past"] + max(n), c["dk"])
        s["q_out"], s["k_out"] = torch.empty_like(s["q"]), torch.empty_like(s["k"])
        s["eps"] = 1e-5
        return s
    if c["op"] == "decode":
        live = _live(c)
        s["kp"], s["vp"], s["ks"], s["vs"], s["table"] = _cache(g, c, live)
        s["pos"] = _ints([x - 1 for x in live])
        s["len_bound"] = rows = max(live)
        s["q"] = _normal(g, c["B"], c["H"] * c["dk"])
        s["k"], s["v"] = (_normal(g, c["B"], c["Hkv"] * c["dk"]) for _ in range(2))
        # what comes back: the new token's block up to it
        back = [((x - 1) // c["block"] * c["block"], (x - 1) % c["block"] + 1) if x else (0, 0) for x in live]
    else:
        s["kp"], s["vp"], s["ks"], s["vs"], s["table"] = _cache(g, c, [c["past"] + x for x in n])
        s["M"], s["t_bound"] = sum(n), max(n)
        s["cu"], s["pos0"] = _offsets(n), _ints([c["past"]] * c["B"])
        rows = c["past"] + max(n)
        if c["op"] == "fill":
            s["k"], s["v"] = (_normal(g, c["Hkv"] * c["dk"], s["M"]) for _ in range(2))
            old = c["past"] % c["block"]  # tokens of the last block before
            back = [(c["past"] - old, old + x) for x in n]
        else:
            s["q"] = _normal(g, c["H"] * c["dk"], s["M"])
            s["prefix_t"] = _ints([c["prefix"]] * c["B"]) if c["prefix"] else None
    s["cos"], s["sin"] = _tables(rows, c["dk"])
    if c["op"] != "fill":
        s["slopes"] = _slopes(c["H"]) if c["alibi"] else None
        s["scale"] = 1.0 / math.sqrt(c["dk"])
        s["out"] = torch.empty_like(s["q"])
    if c["op"] != "prompt":
        s["back_pos0"], s["back_cu"] = _ints([p for p, _ in back]), _offsets([x for _, x in back])
        s["back_M"] = sum(x for _, x in back)
        s["k_back"], s["v_back"] = (torch.empty(c["Hkv"] * c["dk"], s["back_M"], device=DEV) for _ in range(2))
    if own:
        s["cache"] = _pkg().KVPagesI8(s["kp"], s["vp"], s["ks"], s["vs"], s["table"])
    return s


def _prepare_tables(s, g, n):
    """Running sequences with their pages, the others in the free list in any order; some slots empty."""
    B, page = s["B"], s["page"]
    held = [x if i % 7 != 3 else 0 for i, x in enumerate(n)]  # one in 7 has not begun
    add = _spread(s["add_lo"], s["add_hi"], B)
    add = [x if i % 11 != 5 else 0 for i, x in enumerate(add)]  # one in 11 waits
    pages = [-(-x // page) for x in held]
    need = sum(-(-(x + a) // page) - p for x, a, p in zip(held, add, pages))
    left = need * 4 // 5 if s["scarce"] else need + 5
    width = -(-(max(n) + s["add_hi"]) // page)
    total = sum(pages) + left
    ids = torch.randperm(total, generator=g, device=DEV).int()
    s["table"] = torch.full((B, width), -1, dtype=torch.int32, device=DEV)
    valid = torch.arange(width, device=DEV)[None, :] < torch.tensor(pages, device=DEV)[:, None]
    s["table"][valid] = ids[:sum(pages)]
    s["free"] = torch.full((total,), -1, dtype=torch.int32, device=DEV)
    s["free"][:left] = ids[sum(pages):]
    s["count"], s["lens"], s["add"], s["keep"] = _ints([left]), _ints(held), _ints(add), _ints(held)
    s["M"] = sum(add)  # tokens at most
    s["cu"], s["pos0"] = torch.zeros(B + 1, dtype=torch.int32, device=DEV), torch.zeros(B, dtype=torch.int32, device=DEV)
    s["pos"], s["slots"] = (torch.zeros(s["M"], dtype=torch.int32, device=DEV) for _ in range(2))
    return s


# ------------------------------------------------------------------------------------------ one pass

def run(s):
    if own:
        return _run_own(s)
    return {"decode": _plain_decode, "fill": _plain_fill, "prompt": _plain_prompt, "qk": _plain_qk,
            "tables": _plain_tables}[s["op"]](s)


def _run_own(s):
    ctx = _ctx()
    if s["op"] == "decode":
        out = ctx.attention_pages_decode(s["cache"], s["q"], s["k"], s["v"], s["H"], s["pos"], s["len_bound"],
                                         s["scale"], cos=s["cos"], sin=s["sin"], softcap=s["cap"], slopes=s["slopes"],
                                         out=s["out"], tokens=True)
        k, v = ctx.kv_pages_read(s["cache"], s["back_cu"], s["back_M"], pos0=s["back_pos0"], k=s["k_back"], v=s["v_back"])
        return {"out": out, "k": k, "v": v}
    if s["op"] == "fill":
        ctx.kv_pages_fill(s["cache"], s["k"], s["v"], s["cu"], pos0=s["pos0"], cos=s["cos"], sin=s["sin"])
        k, v = ctx.kv_pages_read(s["cache"], s["back_cu"], s["back_M"], pos0=s["back_pos0"], k=s["k_back"], v=s["v_back"])
        return {"k": k, "v": v}
    if s["op"] == "prompt":
        return ctx.attention_pages_prefill(s["cache"], s["q"], s["cu"], s["t_bound"], s["H"], s["scale"],
                                           pos0=s["pos0"], cos=s["cos"], sin=s["sin"], softcap=s["cap"],
                                           slopes=s["slopes"], prefix=s["prefix_t"], out=s["out"])
    if s["op"] == "qk":
        q, k = ctx.qk_norm_rope(s["q"], s["k"], s["dk"], s["eps"], s["gq"], s["gk"], pos=s["pos"], cos=s["cos"],
                                sin=s["sin"], q_out=s["q_out"], k_out=s["k_out"], tokens=s["tokens"])
        return {"q": q, "k": k}
    ctx.pages_assign(s["table"], s["page"], s["free"], s["count"], s["lens"], s["add"], cu=s["cu"], pos0=s["pos0"],
                     pos=s["pos"], slots=s["slots"])
    ctx.pages_release(s["table"], s["page"], s["free"], s["count"], s["lens"], s["keep"])
    return _tables_out(s)


def _tables_out(s):
    return {x: s[x] for x in ("table", "free", "count", "lens", "cu", "pos0", "pos", "slots")}


def _rotated(x, cos, sin):
    """x (n, heads, dk) rotated with the tables' rows cos, sin (n, dk/2)."""
    h = x.shape[-1] // 2
    a, b, c, d = x[..., :h], x[..., h:], cos[:, None, :], sin[:, None, :]
    return torch.cat((a * c + (-b) * d, b * c + a * d), -1)


def _codes(x, scale):
    """x over scale, rounded half away from zero, within 127; 0 where the scale is 0."""
    y = torch.where(scale > 0, x / scale, torch.zeros_like(x)).clamp(-127.0, 127.0)
    t = y.trunc()
    return t + torch.sign(y) * ((y - t).abs() >= 0.5)


def _places(s, b, p):
    """Page and slot of positions p of sequences b."""
    return s["table"][b, p // s["page"]].long(), p % s["page"]


def _by_position(s):
    """Views of both pools by (page, 16s of slots, slot, head, dimension) and of their scales by (page, block, head)."""
    k, v = s["kp"].permute(0, 2, 4, 1, 3, 5), s["vp"].permute(0, 2, 4, 1, 3)
    return {"k": (k, s["ks"].transpose(1, 2)), "v": (v, s["vs"].transpose(1, 2))}


def _values(pool, scales, at, slot, G):
    """The values at those positions, (n, Hkv, dk), and their scales (n, Hkv, 1)."""
    unit = scales[at, slot // G][:, :, None]
    return pool[at, slot // 16, slot % 16].float().flatten(2) * unit, unit


def _store(s, k, v, b, p, past):
    """Keys and values (n, Hkv, dk) quantized into positions p of sequences b; past: positions that are there already
    of the first sequences, all that get tokens."""
    G, Hkv = s["block"], s["Hkv"]
    R, width = past.shape[0], s["table"].shape[1] * s["page"] // G
    at, slot = _places(s, b, p)
    group = (b * width + p // G)[:, None].expand(-1, Hkv)
    goes_on = (p // G * G < past[b])[:, None]
    # the older positions of the block that a sequence goes on with (in place of the others, its first new one, which
    # is written last)
    op = (past // G * G)[:, None] + torch.arange(G, device=DEV)[None, :]
    op = torch.minimum(op, past[:, None]).flatten()
    oat, oslot = _places(s, torch.arange(R, device=DEV).repeat_interleave(G), op)
    views = _by_position(s)
    for name, x in (("k", k), ("v", v)):
        pool, scales = views[name]
        top = torch.zeros(R * width, Hkv, device=DEV).scatter_reduce(0, group, x.abs().amax(-1), "amax").gather(0, group)
        new = top * (1.0 / 127.0)
        new = torch.where(goes_on, torch.maximum(new, scales[at, slot // G]), new)
        # the older values of the blocks that go on
        here = pool[oat, oslot // 16, oslot % 16]
        values, before = _values(pool, scales, oat, oslot, G)
        scales[at, slot // G] = new
        after = scales[oat, oslot // G][:, :, None]
        again = _codes(values, after).to(torch.int8).view_as(here)
        pool[oat, oslot // 16, oslot % 16] = torch.where((after > before).view(-1, Hkv, *[1] * (here.dim() - 2)), again, here)
        pool[at, slot // 16, slot % 16] = _codes(x, new[:, :, None]).to(torch.int8).view(-1, *here.shape[1:])


def _read(s):
    """The values of positions back_pos0[b] on of each sequence, (Hkv*dk, n) feature-major."""
    m = torch.arange(s["back_M"], device=DEV)
    cu = s["back_cu"].long()
    b = torch.searchsorted(cu, m, right=True) - 1
    at, slot = _places(s, b, s["back_pos0"].long()[b] + m - cu[b])
    return {name: _values(pool, scales, at, slot, s["block"])[0].flatten(1).t().contiguous()
            for name, (pool, scales) in _by_position(s).items()}


def _rows(s, pages):
    """The first pages of every sequence as keys and values (B, Hkv, positions, dk) in 32 bits; -1 reads page 0."""
    B, Hkv, dk, page, G = s["B"], s["Hkv"], s["dk"], s["page"], s["block"]
    at = s["table"][:, :pages].clamp(min=0).long()

    def scaled(x, scales):
        x = x.reshape(B, pages, Hkv, page // G, G, dk).float() * scales[at][..., None, None]
        return x.permute(0, 2, 1, 3, 4, 5).reshape(B, Hkv, pages * page, dk)

    return scaled(s["kp"][at].transpose(4, 5), s["ks"]), scaled(s["vp"][at].transpose(4, 5), s["vs"])


def _attend(q, K, V, visible, distance, s):
    """q (B, H, T, dk) over K, V (B, Hkv, S, dk); visible (B, T, S); distance (B, T, S) = key - query."""
    B, H, T, dk = q.shape
    Hkv, S = K.shape[1], K.shape[2]
    x = torch.matmul(q.reshape(B, Hkv, H // Hkv * T, dk), K.transpose(2, 3).contiguous()) * s["scale"]
    x = x.view(B, H, T, S)
    if s["cap"] > 0:
        x = torch.tanh(x / s["cap"]) * s["cap"]
    if s["slopes"] is not None:
        x = x + s["slopes"][None, :, None, None] * distance[:, None].float()
    x = x.masked_fill(~visible[:, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(-1)
    o = torch.matmul(p.view(B, Hkv, H // Hkv * T, S), V).view(B, H, T, dk)
    return torch.where(total[..., None] > 0, o / total[..., None], torch.zeros_like(o))


def _plain_decode(s):
    B, H, Hkv, dk, page = s["B"], s["H"], s["Hkv"], s["dk"], s["page"]
    n = B - s["idle"]  # sequences with a new token
    p = s["pos"].clamp(min=0).long()
    cos, sin = s["cos"][p], s["sin"][p]
    q = _rotated(s["q"].view(B, H, dk), cos, sin)
    k = _rotated(s["k"].view(B, Hkv, dk), cos, sin)
    _store(s, k[:n], s["v"].view(B, Hkv, dk)[:n], torch.arange(n, device=DEV), p[:n], p[:n])
    pages = -(-s["len_bound"] // page)
    K, V = _rows(s, pages)
    at = torch.arange(pages * page, device=DEV)[None, None, :]
    visible = (at <= s["pos"].long()[:, None, None])
    o = _attend(q.view(B, H, 1, dk), K, V, visible, at - p[:, None, None], s)
    return {"out": o.reshape(B, H * dk), **_read(s)}


def _columns(s):
    """The sequence, token and position of every column."""
    m = torch.arange(s["M"], device=DEV)
    b = torch.searchsorted(s["cu"].long(), m, right=True) - 1
    t = m - s["cu"].long()[b]
    return b, t, s["pos0"].long()[b] + t


def _plain_fill(s):
    Hkv, dk, M = s["Hkv"], s["dk"], s["M"]
    b, _, p = _columns(s)
    k = _rotated(s["k"].t().reshape(M, Hkv, dk), s["cos"][p], s["sin"][p])
    _store(s, k, s["v"].t().reshape(M, Hkv, dk), b, p, s["pos0"].long())
    return _read(s)


def _plain_prompt(s):
    B, H, dk, page, M = s["B"], s["H"], s["dk"], s["page"], s["M"]
    b, t, p = _columns(s)
    T = s["t_bound"]
    q = torch.zeros(B, T, H, dk, device=DEV)
    q[b, t] = _rotated(s["q"].t().reshape(M, H, dk), s["cos"][p], s["sin"][p])
    pages = -(-(s["past"] + T) // page)
    K, V = _rows(s, pages)
    at = torch.arange(pages * page, device=DEV)[None, None, :]
    query = (s["pos0"].long()[:, None] + torch.arange(T, device=DEV))[:, :, None]
    visible = at <= query
    if s["prefix_t"] is not None:
        last = s["pos0"].long() + s["cu"].long()[1:] - s["cu"].long()[:-1]
        visible = visible | (at < torch.minimum(s["prefix_t"].long(), last)[:, None, None])
    o = _attend(q.transpose(1, 2).contiguous(), K, V, visible, at - query, s)  # (B, H, T, dk)
    return o.transpose(1, 2)[b, t].reshape(M, H * dk).t().contiguous()


def _plain_qk(s):
    p = s["pos"].long()
    got = {}
    for name, x, gain in (("q", s["q"], s["gq"]), ("k", s["k"], s["gk"])):
        x = (x if s["tokens"] else x.t()).reshape(p.shape[0], -1, s["dk"])
        y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + s["eps"]) * gain
        y = _rotated(y, s["cos"][p], s["sin"][p]).flatten(1)
        got[name] = y if s["tokens"] else y.t().contiguous()
    return got


def _plain_tables(s):
    B, page = s["B"], s["page"]
    width = s["table"].shape[1]
    lens, add, count = s["lens"].long(), s["add"].long(), s["count"].long()
    # pages for the new tokens, in the sequences' order from the top of the list
    fits = (lens >= 0) & (add > 0) & (lens + add <= width * page)
    held = (lens + page - 1) // page
    need = torch.where(fits, (lens + add + page - 1) // page - held, torch.zeros_like(held))
    total = need.cumsum(0)
    given = fits & ((need == 0) | (total <= count))
    i = torch.arange(width, device=DEV)[None, :]
    mine = given[:, None] & (i >= held[:, None]) & (i < (held + need)[:, None])
    top = count - 1 - ((total - need)[:, None] + i - held[:, None])
    s["table"].copy_(torch.where(mine, s["free"][top.clamp(min=0)], s["table"]))
    taken = torch.where(given, need, torch.zeros_like(need)).sum()
    tokens = torch.where(given, add, torch.zeros_like(add))
    s["cu"][1:] = tokens.cumsum(0)
    s["pos0"].copy_(torch.where(given, lens, torch.full_like(lens, -1)))
    new = lens + tokens
    # positions and slots of the tokens
    m = torch.arange(s["M"], device=DEV)
    cu = s["cu"].long()
    b = (torch.searchsorted(cu, m, right=True) - 1).clamp(max=B - 1)
    there = m < cu[-1]
    p = lens[b] + m - cu[b]
    slot = s["table"][b, (p // page).clamp(0, width - 1)].long() * page + p % page
    s["pos"].copy_(torch.where(there, p, torch.full_like(p, -1)))
    s["slots"].copy_(torch.where(there, slot, torch.full_like(p, -1)))
    # the pages of what is not kept, back on the list in the opposite order
    count = count - taken
    keep = torch.minimum(s["keep"].long(), new)
    left = (keep + page - 1) // page
    back = (new + page - 1) // page - left
    behind = back.flip(0).cumsum(0).flip(0)  # from sequence b to the last
    mine = (i >= left[:, None]) & (i < (left + back)[:, None])
    to = count + behind[:, None] - 1 - (i - left[:, None])
    to = torch.where(mine, to, torch.full_like(to, s["free"].shape[0]))  # (what stays: to a place past the end)
    s["free"].copy_(torch.cat((s["free"], s["count"])).scatter(0, to.flatten(), s["table"].flatten())[:-1])
    s["count"].copy_(count + behind[0])
    s["lens"].copy_(keep)
    return _tables_out(s)


# ------------------------------------------------------------------------------------------ work and truth

def work(case):
    c = case
    n = _new_tokens(c)
    if c["op"] == "tables":
        add = _spread(c["add_lo"], c["add_hi"], c["B"])
        pages = sum(-(-a // c["page"]) for a in add)
        # lengths, counts, offsets and positions of the sequences; ids read, written and put back; the tokens' two
        return {"bytes": 28 * c["B"] + 16 * pages + 8 * sum(add), "flops": 0}
    if c["op"] == "qk":
        M = sum(n)
        x = M * (c["H"] + c["Hkv"]) * c["dk"]
        return {"bytes": 8 * x + 4 * M + 8 * c["dk"] + 4 * c["dk"] * (1 if c["hi"] == 1 else max(n)), "flops": 10 * x}
    row = 2 * c["Hkv"] * c["dk"]          # values of a position
    scale = 2 * c["Hkv"] * 4 / c["block"]  # its share of two scales
    if c["op"] == "decode":
        live = [x for x in _live(c) if x]
        old = sum(x - 1 for x in live)
        back = sum((x - 1) % c["block"] + 1 for x in live)
        b = old * (row + scale) + len(live) * (row * 5 + 4 * c["dk"])           # the cache; the new token; table rows
        b += (len(live) + c["B"]) * c["H"] * c["dk"] * 4                        # queries, outputs
        b += 4 * sum(-(-x // c["page"]) for x in live) + 4 * c["B"]
        b += back * row * 4                                                     # what comes back (its codes were read)
        return {"bytes": int(b), "flops": 4 * c["H"] * c["dk"] * sum(live)}
    M = sum(n)
    tables = 4 * c["dk"] * max(n)
    pages = 4 * sum(-(-(c["past"] + x) // c["page"]) for x in n)
    if c["op"] == "fill":
        old = c["past"] % c["block"] * c["B"]
        # tokens in 32 bits, their codes written, all of it read back and returned in 32 bits
        return {"bytes": int(M * row * 10 + old * row * 5 + M * 3 * scale + tables + pages), "flops": 10 * M * row}
    b = 8 * M * c["H"] * c["dk"] + (M + c["past"] * c["B"]) * (row + scale) + tables + pages
    return {"bytes": int(b), "flops": 4 * c["H"] * c["dk"] * sum(_visible(c, x) for x in n)}


def exact(case, seed):
    s = prepare(dict(case), seed)
    if s["op"] == "tables":
        return None
    d = torch.float64
    dk = s["dk"]
    z = torch.complex(s["cos"].to(d), s["sin"].to(d))  # a pair (x[j], x[j + dk/2]) turned by its angle

    def turned(x, p):
        y = torch.complex(x[..., :dk // 2].to(d), x[..., dk // 2:].to(d)) * z[p][:, None, :]
        return torch.cat((y.real, y.imag), -1)

    if s["op"] == "qk":
        got = {}
        for name, gain in (("q", s["gq"]), ("k", s["gk"])):
            x = s[name] if s["tokens"] else s[name].t()
            x = x.to(d).reshape(x.shape[0], -1, dk)
            x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / dk + s["eps"]) * gain.to(d)
            y = turned(x, s["pos"].long()).flatten(1)
            got[name] = y if s["tokens"] else y.t()
        return got
    Hkv, page, G = s["Hkv"], s["page"], s["block"]
    n = _new_tokens(s)
    # codes as (page, head, slot, dim), scales as (page, head, slot)
    codes = {"k": s["kp"].permute(0, 1, 2, 4, 3, 5).reshape(-1, Hkv, page, dk),
             "v": s["vp"].permute(0, 1, 2, 4, 3).reshape(-1, Hkv, page, dk)}
    unit = {"k": s["ks"].to(d).repeat_interleave(G, 2), "v": s["vs"].to(d).repeat_interleave(G, 2)}

    def once(x, p):
        """A key's rotation as the cache holds it: two rounded products, a rounded sum, f32 each."""
        a, b = x[..., :dk // 2].to(d), x[..., dk // 2:].to(d)
        c, t = s["cos"].to(d)[p][:, None], s["sin"].to(d)[p][:, None]
        r = lambda v: v.float().to(d)  # noqa: E731
        return torch.cat((r(r(a * c) + r(-b * t)), r(r(b * c) + r(a * t))), -1)

    def quantized(x, step):
        y = (x / step.clamp(min=1e-300)).float().to(d).clamp(-127, 127)
        return torch.where(step > 0, torch.floor(y.abs() + 0.5) * torch.sign(y), torch.zeros_like(y))

    def put(b, i0, k, v):
        """Tokens from position i0 of sequence b on, block by block."""
        for name, x in (("k", k), ("v", v)):
            for j in range(i0 // G, (i0 + x.shape[0] - 1) // G + 1):
                lo, hi = max(j * G, i0), min((j + 1) * G, i0 + x.shape[0])
                where, slot = int(s["table"][b, j * G // page]), j * G % page
                new = x[lo - i0:hi - i0].to(d)  # (t, Hkv, dk)
                step = (new.abs().amax((0, 2)) * torch.tensor(1.0 / 127.0).float().to(d).to(DEV)).float().to(d)
                old = unit[name][where, :, slot].clone()
                if lo > j * G:
                    step = torch.maximum(step, old)
                    here = codes[name][where, :, slot:slot + lo - j * G].to(d)  # (Hkv, t, dk)
                    again = quantized((here * old[:, None, None]).float().to(d), step[:, None, None].expand_as(here))
                    here = torch.where((step > old)[:, None, None], again, here)
                    codes[name][where, :, slot:slot + lo - j * G] = here.to(torch.int8)
                unit[name][where, :, slot:slot + G] = step[:, None]
                codes[name][where, :, slot + lo - j * G:slot + hi - j * G] = \
                    quantized(new, step[None, :, None].expand_as(new)).transpose(0, 1).to(torch.int8)

    def held(name, b, i0, i1):
        p = torch.arange(i0, i1, device=DEV)
        at = s["table"][b].long()[p // page]
        return codes[name][at, :, p % page].to(d) * unit[name][at, :, p % page][..., None]  # (t, Hkv, dk)

    if s["op"] == "fill":
        for b, count in enumerate(n):
            m0, p = int(s["cu"][b]), torch.arange(s["past"], s["past"] + count, device=DEV)
            k, v = (s[x][:, m0:m0 + count].t().reshape(count, Hkv, dk) for x in "kv")
            put(b, s["past"], once(k, p), v)
    elif s["op"] == "decode":
        for b in range(s["B"]):
            p = s["pos"][b:b + 1].long()
            if int(p) >= 0:
                put(b, int(p), once(s["k"][b].view(1, Hkv, dk), p), s["v"][b].view(1, Hkv, dk))
    back = {}
    if s["op"] != "prompt":
        cu, pos0 = s["back_cu"].tolist(), s["back_pos0"].tolist()
        for name in "kv":
            back[name] = torch.cat([held(name, b, pos0[b], pos0[b] + cu[b + 1] - cu[b]).flatten(1)
                                    for b in range(s["B"]) if cu[b + 1] > cu[b]]).t()
        if s["op"] == "fill":
            return back
    out = torch.zeros(s["q"].shape, dtype=d, device=DEV)
    for b, count in enumerate(n):
        if s["op"] == "decode":
            i0, count = int(s["pos"][b]), 1
            if i0 < 0:
                continue
            q = s["q"][b].view(1, -1, dk)
        else:
            i0, m0 = s["past"], int(s["cu"][b])
            q = s["q"][:, m0:m0 + count].t().reshape(count, -1, dk)
        p = torch.arange(i0, i0 + count, device=DEV)
        at = torch.arange(i0 + count, device=DEV)
        K, V = held("k", b, 0, i0 + count), held("v", b, 0, i0 + count)
        q = turned(q, p)
        see = at[None, :] <= p[:, None]
        if s["op"] == "prompt":
            see = see | (at[None, :] < s["prefix"])
        for h in range(s["H"]):
            g = h // (s["H"] // Hkv)
            x = (q[:, h] @ K[:, g].t().contiguous()) * s["scale"]
            if s["cap"] > 0:
                x = s["cap"] * torch.tanh(x / s["cap"])
            if s["slopes"] is not None:
                x = x + s["slopes"][h].to(d) * (at[None, :] - p[:, None])
            o = torch.softmax(x.masked_fill(~see, -math.inf), -1) @ V[:, g]
            if s["op"] == "decode":
                out[b, h * dk:(h + 1) * dk] = o[0]
            else:
                out[h * dk:(h + 1) * dk, m0:m0 + count] = o.t()
    return out if s["op"] == "prompt" else {"out": out, **back}
