"""Performance cases of the operators that serve sequences of unlike lengths: the paged KV cache (fill,
prompt attention, decode attention) and the adjustment of logits with the choice of the next token.

A case is a dict of plain values with an "op":

  decode   one new token for each of B sequences (the last `idle` of them without one) over a paged
           cache: rotation, append, attention; positions spread from lo to hi
  fill     the keys and values of packed prompts (lo to hi tokens each) rotated and written to pages
  prompt   attention of packed prompts (lo to hi tokens each, `past` positions already cached) over
           pages that hold their keys; causal, or with a bidirectional prefix
  logits   penalties, bias and grammar mask on a batch's logits, the greedy choice and the counts

cap > 0 caps the scores by a tanh; alibi adds a bias that falls with the distance. The shapes are those
of bench.py's decoder (20 heads over 5 KV heads of 128, vocabulary 10000) and generic ones. With
`own` false, run() computes everything by elementary torch operations; with it, by the framework.
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
        dict(name="decode_1_short", op="decode", B=1, idle=0, H=20, Hkv=5, dk=128, page=16, lo=100, hi=100,
             f16=True, cap=0.0, alibi=False),
        # the decoder benchmark's batch: 16 sequences around position 2112, f32 caches
        dict(name="decode_16", op="decode", B=16, idle=0, H=20, Hkv=5, dk=128, page=64, lo=1920, hi=2176,
             f16=False, cap=0.0, alibi=False),
        # a server's batch: lengths from one token to 16 K, three empty slots, 8 heads to a KV head, capped
        # and biased scores
        dict(name="decode_ragged", op="decode", B=37, idle=3, H=16, Hkv=2, dk=64, page=32, lo=1, hi=16384,
             f16=True, cap=30.0, alibi=True),
        # long documents: few sequences, caches of up to 128 K positions
        dict(name="decode_long", op="decode", B=4, idle=0, H=32, Hkv=8, dk=128, page=64, lo=60000, hi=131072,
             f16=True, cap=0.0, alibi=False),
        # the short prompts that arrive between two decode steps
        dict(name="fill_short", op="fill", B=3, Hkv=5, dk=128, page=16, lo=5, hi=40, past=0, f16=False),
        # a full prompt batch of the decoder benchmark, ragged
        dict(name="fill_prompts", op="fill", B=16, Hkv=5, dk=128, page=64, lo=1111, hi=2048, past=0, f16=True),
        # a handful of short prompts: latency again
        dict(name="prompt_short", op="prompt", B=3, H=20, Hkv=5, dk=128, page=16, lo=5, hi=40, past=0, f16=True,
             cap=0.0, alibi=False, prefix=0),
        # packed prompts of unlike lengths over f32 caches, with a bidirectional prefix of 256 tokens, capped
        # and biased
        dict(name="prompt_packed", op="prompt", B=8, H=16, Hkv=2, dk=64, page=32, lo=77, hi=1900, past=0, f16=False,
             cap=50.0, alibi=True, prefix=256),
        # a chunk of long prompts, whose first 6144 positions are cached already
        dict(name="prompt_chunk", op="prompt", B=4, H=20, Hkv=5, dk=128, page=64, lo=700, hi=1024, past=6144,
             f16=True, cap=0.0, alibi=False, prefix=0),
        # one sequence's choice under a grammar, every rule in use
        dict(name="logits_1", op="logits", B=1, V=10000, hist=700, penalties=True, bias=True, shared=False,
             mask=0.02, empty=0, write=False),
        # a batch under penalties alone; the adjusted logits go on to a sampler
        dict(name="logits_16", op="logits", B=16, V=10000, hist=2048, penalties=True, bias=False, shared=False,
             mask=0.0, empty=0, write=True),
        # a large server's step over a large odd vocabulary: shared bias, masks of which some allow nothing
        dict(name="logits_256", op="logits", B=256, V=131071, hist=4096, penalties=True, bias=True, shared=True,
             mask=0.5, empty=3, write=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _span(rng, lo, hi):
    """A range of lengths: all alike, or spread."""
    a, b = sorted((_log(rng, lo, hi), _log(rng, lo, hi)))
    return (b, b) if rng.random() < 0.3 else (a, b)


def draw(rng):
    op = rng.choice(["decode", "decode", "fill", "prompt", "prompt", "logits"])
    page = rng.choice([8, 16, 32, 64, 128])
    f16 = rng.random() < 0.5
    if op == "decode":
        H, Hkv, dk = rng.choice([(20, 5, 128), (16, 16, 64), (16, 2, 64), (32, 8, 128), (8, 1, 256), (12, 4, 128),
                                 (24, 2, 64), (7, 7, 128)])
        B = _log(rng, 1, 64)
        most = max(16, min(131072, 800_000_000 // (B * Hkv * dk * 8)))  # positions within about 0.8 GB of caches
        lo, hi = _span(rng, 1, most)
        return dict(op=op, B=B, idle=rng.choice([0, 0, B // 4]), H=H, Hkv=Hkv, dk=dk, page=page, lo=lo, hi=hi, f16=f16,
                    cap=rng.choice([0.0, 0.0, 20.0, 50.0]), alibi=rng.random() < 0.3)
    if op == "fill":
        B = _log(rng, 1, 16)
        lo, hi = _span(rng, 1, 2048)
        return dict(op=op, B=B, Hkv=rng.choice([1, 2, 5, 8]), dk=rng.choice([64, 128]), page=page, lo=lo, hi=hi,
                    past=rng.choice([0, _log(rng, 1, 4000)]), f16=f16)
    if op == "prompt":
        H, Hkv, dk = rng.choice([(20, 5, 128), (16, 2, 64), (8, 8, 64), (16, 8, 128)])
        B = _log(rng, 1, 8)
        lo, hi = _span(rng, 1, 1024)
        past = rng.choice([0, 0, _log(rng, 1, 4000)])
        return dict(op=op, B=B, H=H, Hkv=Hkv, dk=dk, page=page, lo=lo, hi=hi, past=past, f16=f16,
                    cap=rng.choice([0.0, 0.0, 20.0, 50.0]), alibi=rng.random() < 0.3,
                    prefix=rng.choice([0, 0, past + _log(rng, 1, 600)]))
    B = _log(rng, 1, 256)
    return dict(op=op, B=B, V=_log(rng, 300, 131071), hist=_log(rng, 1, 4096), penalties=rng.random() < 0.8,
                bias=rng.random() < 0.5, shared=rng.random() < 0.5, mask=rng.choice([0.0, 0.001, 0.3, 0.9]),
                empty=rng.choice([0, B // 8]), write=rng.random() < 0.5)


def _spread(lo, hi, n):
    """n lengths from lo to hi, spread over their logarithm in a fixed order, the longest among them."""
    got = [int(round(lo * (hi / lo) ** ((0.5 + 0.6180339887 * i) % 1.0))) for i in range(n)]
    got[n // 2] = hi
    return got


def _new_tokens(c):
    """Tokens of each sequence that the call works on."""
    return _spread(c["lo"], c["hi"], c["B"])


def _visible(c, n):
    """Pairs of a prompt's query and a key that it sees, for a sequence of n new tokens."""
    past, pre = c["past"], min(c["prefix"], c["past"] + n)
    full = n * past + n * (n + 1) // 2
    # query t sees max(past + t + 1, pre) keys
    short = max(0, pre - past - 1)  # queries whose causal reach is below the prefix
    short = min(short, n)
    return full + sum(pre - (past + t + 1) for t in range(short))


# ------------------------------------------------------------------------------------------ inputs

def _normal(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32).to(dtype)


def _tables(rows, dk):
    """cos and sin of position / 10000^(2j/dk), (rows, dk/2)."""
    theta = torch.arange(rows, device=DEV, dtype=torch.float64)[:, None] / torch.pow(
        torch.tensor(10000.0, device=DEV, dtype=torch.float64),
        torch.arange(0, dk, 2, device=DEV, dtype=torch.float64) / dk)[None, :]
    return theta.cos().float(), theta.sin().float()


def _cache(g, c, lens):
    """Pools with every page of the sequences at a place of its own among a tenth more, and the page table
    (-1 behind a sequence's last page)."""
    page, B = c["page"], len(lens)
    need = [-(-n // page) for n in lens]
    total = sum(need) + max(1, sum(need) // 10)
    dt = torch.float16 if c["f16"] else torch.float32
    k = _normal(g, total, c["Hkv"], page, c["dk"], dtype=dt)
    v = _normal(g, total, c["Hkv"], page, c["dk"], dtype=dt)
    places = torch.randperm(total, generator=g, device=DEV).int()
    table = torch.full((B, max(1, max(need))), -1, dtype=torch.int32, device=DEV)
    valid = torch.arange(table.shape[1], device=DEV)[None, :] < torch.tensor(need, device=DEV)[:, None]
    table[valid] = places[:sum(need)]
    return k, v, table


def _slopes(H):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)], device=DEV)


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = dict(c)
    if c["op"] == "logits":
        B, V = c["B"], c["V"]
        s["logits"] = 2.0 * _normal(g, B, V)
        s["counts"] = s["repeat"] = s["presence"] = s["frequency"] = s["bias_t"] = s["allowed"] = None
        if c["penalties"]:
            # tokens so far, the low ids much more often, as in text
            hist = (V * torch.rand(B, c["hist"], generator=g, device=DEV) ** 3).long().clamp_(max=V - 1)
            s["counts"] = torch.zeros(B, V, dtype=torch.int32, device=DEV)
            s["counts"].scatter_add_(1, hist, torch.ones_like(hist, dtype=torch.int32))
            s["repeat"] = 1.0 + 0.5 * torch.rand(B, generator=g, device=DEV)
            s["presence"] = 0.8 * torch.rand(B, generator=g, device=DEV)
            s["frequency"] = 0.3 * torch.rand(B, generator=g, device=DEV)
        if c["bias"]:
            b = _normal(g, 1 if c["shared"] else B, V)
            s["bias_t"] = torch.where(b.abs() > 2.0, 4.0 * b, torch.zeros_like(b))
        if c["mask"] > 0:
            words = (V + 31) // 32
            bits = torch.rand(B, words, 32, generator=g, device=DEV) < c["mask"]
            if c["empty"]:
                bits[-c["empty"]:] = False
            weight = torch.ones(32, dtype=torch.int64, device=DEV) << torch.arange(32, device=DEV)
            w = (bits.long() * weight).sum(-1)
            s["allowed"] = torch.where(w >= 1 << 31, w - (1 << 32), w).int()
        if own:
            s["rules"] = _pkg().LogitRules(V, counts=s["counts"], repeat=s["repeat"], presence=s["presence"],
                                           frequency=s["frequency"], bias=s["bias_t"], allowed=s["allowed"],
                                           count_choice=s["counts"] is not None)
        s["ids"] = torch.zeros(B, dtype=torch.int32, device=DEV)
        s["out"] = torch.empty(B, V, device=DEV) if c["write"] else None
        return s
    n = _new_tokens(c)
    if c["op"] == "decode":
        live = [x if i < c["B"] - c["idle"] else 0 for i, x in enumerate(n)]  # lengths with the new token
        s["k_pages"], s["v_pages"], s["table"] = _cache(g, c, live)
        s["pos"] = torch.tensor([x - 1 for x in live], dtype=torch.int32, device=DEV)
        s["len_bound"] = max(live)
        s["q"] = _normal(g, c["B"], c["H"] * c["dk"])
        s["k"], s["v"] = (_normal(g, c["B"], c["Hkv"] * c["dk"]) for _ in range(2))
        rows = max(live)
    else:
        s["k_pages"], s["v_pages"], s["table"] = _cache(g, c, [c["past"] + x for x in n])
        M = sum(n)
        s["M"], s["t_bound"] = M, max(n)
        s["cu"] = torch.tensor([sum(n[:i]) for i in range(len(n) + 1)], dtype=torch.int32, device=DEV)
        s["pos0"] = torch.full((c["B"],), c["past"], dtype=torch.int32, device=DEV)
        rows = c["past"] + max(n)
        if c["op"] == "fill":
            s["k"], s["v"] = (_normal(g, c["Hkv"] * c["dk"], M) for _ in range(2))
        else:
            s["q"] = _normal(g, c["H"] * c["dk"], M)
            s["prefix_t"] = torch.full((c["B"],), c["prefix"], dtype=torch.int32, device=DEV) if c["prefix"] else None
    s["cos"], s["sin"] = _tables(rows, c["dk"])
    if c["op"] != "fill":
        s["slopes"] = _slopes(c["H"]) if c["alibi"] else None
        s["scale"] = 1.0 / math.sqrt(c["dk"])
        s["out"] = torch.empty_like(s["q"])
    if own:
        s["cache"] = _pkg().KVPages(s["k_pages"], s["v_pages"], s["table"])
    return s


# ------------------------------------------------------------------------------------------ one pass

def run(s):
    if own:
        return _run_own(s)
    return {"decode": _plain_decode, "fill": _plain_fill, "prompt": _plain_prompt, "logits": _plain_logits}[s["op"]](s)


def _run_own(s):
    ctx = _ctx()
    if s["op"] == "decode":
        out = ctx.attention_pages_decode(s["cache"], s["q"], s["k"], s["v"], s["H"], s["pos"], s["len_bound"],
                                         s["scale"], cos=s["cos"], sin=s["sin"], softcap=s["cap"], slopes=s["slopes"],
                                         out=s["out"], tokens=True)
        return {"out": out, "k": s["k_pages"], "v": s["v_pages"]}
    if s["op"] == "fill":
        ctx.kv_pages_fill(s["cache"], s["k"], s["v"], s["cu"], pos0=s["pos0"], cos=s["cos"], sin=s["sin"])
        return {"k": s["k_pages"], "v": s["v_pages"]}
    if s["op"] == "prompt":
        return ctx.attention_pages_prefill(s["cache"], s["q"], s["cu"], s["t_bound"], s["H"], s["scale"],
                                           pos0=s["pos0"], cos=s["cos"], sin=s["sin"], softcap=s["cap"],
                                           slopes=s["slopes"], prefix=s["prefix_t"], out=s["out"])
    ctx.logits_adjust_rows(s["logits"], s["rules"], ids=s["ids"], out=s["out"])
    return {"ids": s["ids"], "out": s["out"], "counts": s["counts"]}


def _rotated(x, cos, sin):
    """x (n, heads, dk) rotated with the tables' rows cos, sin (n, dk/2)."""
    h = x.shape[-1] // 2
    a, b, c, d = x[..., :h], x[..., h:], cos[:, None, :], sin[:, None, :]
    return torch.cat((a * c + (-b) * d, b * c + a * d), -1)


def _rows(pool, table, pages):
    """The first pages of every sequence as (B, Hkv, positions, dk) in 32 bits; -1 reads page 0."""
    B, Hkv, dk = table.shape[0], pool.shape[1], pool.shape[3]
    x = pool[table[:, :pages].clamp(min=0).long()]  # (B, pages, Hkv, page, dk)
    return x.permute(0, 2, 1, 3, 4).reshape(B, Hkv, -1, dk).float()


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
    at = s["table"].gather(1, (p // page)[:, None])[:n, 0].long()
    slot = (p % page)[:n]
    s["k_pages"][at, :, slot] = k[:n].to(s["k_pages"].dtype)
    s["v_pages"][at, :, slot] = s["v"].view(B, Hkv, dk)[:n].to(s["v_pages"].dtype)
    pages = -(-s["len_bound"] // page)
    K, V = _rows(s["k_pages"], s["table"], pages), _rows(s["v_pages"], s["table"], pages)
    at = torch.arange(pages * page, device=DEV)[None, None, :]
    visible = (at <= s["pos"].long()[:, None, None])
    o = _attend(q.view(B, H, 1, dk), K, V, visible, at - p[:, None, None], s)
    return {"out": o.reshape(B, H * dk), "k": s["k_pages"], "v": s["v_pages"]}


def _columns(s):
    """The sequence, token and position of every column."""
    m = torch.arange(s["M"], device=DEV)
    b = torch.searchsorted(s["cu"].long(), m, right=True) - 1
    t = m - s["cu"].long()[b]
    return b, t, s["pos0"].long()[b] + t


def _plain_fill(s):
    Hkv, dk, page, M = s["Hkv"], s["dk"], s["page"], s["M"]
    b, _, p = _columns(s)
    k = _rotated(s["k"].t().reshape(M, Hkv, dk), s["cos"][p], s["sin"][p])
    at, slot = s["table"][b, p // page].long(), p % page
    s["k_pages"][at, :, slot] = k.to(s["k_pages"].dtype)
    s["v_pages"][at, :, slot] = s["v"].t().reshape(M, Hkv, dk).to(s["v_pages"].dtype)
    return {"k": s["k_pages"], "v": s["v_pages"]}


def _plain_prompt(s):
    B, H, Hkv, dk, page, M = s["B"], s["H"], s["Hkv"], s["dk"], s["page"], s["M"]
    b, t, p = _columns(s)
    T = s["t_bound"]
    q = torch.zeros(B, T, H, dk, device=DEV)
    q[b, t] = _rotated(s["q"].t().reshape(M, H, dk), s["cos"][p], s["sin"][p])
    pages = -(-(s["past"] + T) // page)
    K, V = _rows(s["k_pages"], s["table"], pages), _rows(s["v_pages"], s["table"], pages)
    at = torch.arange(pages * page, device=DEV)[None, None, :]
    query = (s["pos0"].long()[:, None] + torch.arange(T, device=DEV))[:, :, None]
    visible = at <= query
    if s["prefix_t"] is not None:
        last = s["pos0"].long() + s["cu"].long()[1:] - s["cu"].long()[:-1]
        visible = visible | (at < torch.minimum(s["prefix_t"].long(), last)[:, None, None])
    o = _attend(q.transpose(1, 2).contiguous(), K, V, visible, at - query, s)  # (B, H, T, dk)
    return o.transpose(1, 2)[b, t].reshape(M, H * dk).t().contiguous()


def _plain_logits(s):
    x, c = s["logits"], s["counts"]
    if c is not None:
        seen = c > 0
        x = torch.where(seen, torch.where(x > 0, x / s["repeat"][:, None], x * s["repeat"][:, None]), x)
        x = torch.where(seen, (x - s["frequency"][:, None] * c.float()) - s["presence"][:, None], x)
    if s["bias_t"] is not None:
        x = x + s["bias_t"]
    ok = torch.ones_like(x, dtype=torch.bool)
    if s["allowed"] is not None:
        v = torch.arange(s["V"], device=DEV)
        ok = (s["allowed"][:, v // 32] >> (v % 32).int()[None, :]) & 1 != 0
        x = x.masked_fill(~ok, -math.inf)
    # the lowest allowed index of the largest allowed value; -1 where nothing is allowed
    best = x.masked_fill(~ok, -math.inf).amax(1, keepdim=True)
    v = torch.arange(s["V"], device=DEV)[None, :]
    first = torch.where(ok & (x == best), v, s["V"]).amin(1)
    s["ids"].copy_(torch.where(first < s["V"], first, -1))
    if c is not None:
        c.scatter_add_(1, first.clamp(max=s["V"] - 1)[:, None], (first < s["V"]).int()[:, None])
    if s["out"] is not None:
        s["out"].copy_(x)
    return {"ids": s["ids"], "out": s["out"], "counts": c}


# ------------------------------------------------------------------------------------------ work and truth

def work(case):
    c = case
    if c["op"] == "logits":
        B, V = c["B"], c["V"]
        b = 4 * B * V + 4 * B
        b += 4 * B * V + 12 * B + 8 * B if c["penalties"] else 0
        b += 4 * V * (1 if c["shared"] else B) if c["bias"] else 0
        b += 4 * B * ((V + 31) // 32) if c["mask"] > 0 else 0
        b += 4 * B * V if c["write"] else 0
        return {"bytes": b, "flops": 4 * B * V}
    es = 2 if c["f16"] else 4
    n = _new_tokens(c)
    if c["op"] == "decode":
        live = n[:c["B"] - c["idle"]]
        old = sum(x - 1 for x in live)
        b = 2 * old * c["Hkv"] * c["dk"] * es                                  # cached keys and values
        b += len(live) * 2 * c["Hkv"] * c["dk"] * (4 + es) + len(live) * 4 * c["dk"]  # the new ones; table rows
        b += len(live) * c["H"] * c["dk"] * 4 + c["B"] * c["H"] * c["dk"] * 4  # queries, outputs
        b += 4 * sum(-(-x // c["page"]) for x in live) + 4 * c["B"]
        return {"bytes": b, "flops": 4 * c["H"] * c["dk"] * sum(live)}
    M = sum(n)
    tables = 4 * c["dk"] * max(n)
    pages = 4 * sum(-(-(c["past"] + x) // c["page"]) for x in n)
    if c["op"] == "fill":
        return {"bytes": 2 * M * c["Hkv"] * c["dk"] * (4 + es) + tables + pages, "flops": 6 * M * c["Hkv"] * c["dk"]}
    b = 8 * M * c["H"] * c["dk"] + 2 * es * (M + c["past"] * c["B"]) * c["Hkv"] * c["dk"] + tables + pages
    return {"bytes": b, "flops": 4 * c["H"] * c["dk"] * sum(_visible(c, x) for x in n)}


def exact(case, seed):
    s = prepare(dict(case), seed)
    if s["op"] == "logits":
        return _exact_logits(s)
    d = torch.float64
    Hkv, dk, page = s["Hkv"], s["dk"], s["page"]
    n, es = _new_tokens(s), s["k_pages"].dtype
    past = s["past"] if s["op"] != "decode" else None
    kp, vp = s["k_pages"].to(d), s["v_pages"].to(d)
    z = torch.complex(s["cos"].to(d), s["sin"].to(d))  # a pair (x[j], x[j + dk/2]) turned by its angle

    def turned(x, p):
        y = torch.complex(x[..., :dk // 2].to(d), x[..., dk // 2:].to(d)) * z[p][:, None, :]
        return torch.cat((y.real, y.imag), -1)

    out = torch.zeros(s["q"].shape, dtype=d, device=DEV) if s["op"] != "fill" else None
    for b, count in enumerate(n):
        if s["op"] == "decode":
            i0, count = int(s["pos"][b]), 1
            if i0 < 0:
                continue
        else:
            i0, m0 = past, int(s["cu"][b])
        p = torch.arange(i0, i0 + count, device=DEV)
        if s["op"] != "prompt":  # the new keys and values, as the cache's type holds them
            if s["op"] == "decode":
                k, v = (s[x][b].view(1, Hkv, dk) for x in "kv")
            else:
                k, v = (s[x][:, m0:m0 + count].t().reshape(count, Hkv, dk) for x in "kv")
            at = s["table"][b, p // page].long()
            k = turned(k, p)
            kp[at, :, p % page] = k.float().to(es).to(d) if s["f16"] else k
            vp[at, :, p % page] = v.to(es).to(d)
        if s["op"] == "fill":
            continue
        S = i0 + count
        at = torch.arange(S, device=DEV)
        pages = s["table"][b].long()[at // page]
        K, V = kp[pages, :, at % page], vp[pages, :, at % page]  # (S, Hkv, dk)
        q = s["q"][b].view(1, -1, dk) if s["op"] == "decode" else s["q"][:, m0:m0 + count].t().reshape(count, -1, dk)
        q = turned(q, p)
        for h in range(s["H"]):
            g = h // (s["H"] // Hkv)
            x = (q[:, h] @ K[:, g].t().contiguous()) * s["scale"]
            if s["cap"] > 0:
                x = s["cap"] * torch.tanh(x / s["cap"])
            if s["slopes"] is not None:
                x = x + s["slopes"][h].to(d) * (at[None, :] - p[:, None])
            see = at[None, :] <= p[:, None]
            if s["op"] == "prompt":
                see = see | (at[None, :] < s["prefix"])
            o = torch.softmax(x.masked_fill(~see, -math.inf), -1) @ V[:, g]
            if s["op"] == "decode":
                out[b, h * dk:(h + 1) * dk] = o[0]
            else:
                out[h * dk:(h + 1) * dk, m0:m0 + count] = o.t()
    if s["op"] == "prompt":
        return out
    return {"k": kp, "v": vp} if s["op"] == "fill" else {"out": out, "k": kp, "v": vp}


def _exact_logits(s):
    if s["out"] is None:
        return None
    d = torch.float64
    x = s["logits"].to(d)
    if s["counts"] is not None:
        c = s["counts"].to(d)
        r, f, q = (s[n].to(d)[:, None] for n in ("repeat", "frequency", "presence"))
        factor = torch.where(c > 0, torch.where(x > 0, 1.0 / r, r), torch.ones_like(x))
        x = x * factor - f * c - q * (c > 0)
    if s["bias_t"] is not None:
        x = x + s["bias_t"].to(d)
    if s["allowed"] is not None:
        bits = torch.stack([(s["allowed"].long() >> i) & 1 for i in range(32)], -1).flatten(1)[:, :s["V"]]
        x = torch.where(bits == 1, x, torch.full_like(x, -math.inf))
    return {"ids": None, "out": x, "counts": None}
