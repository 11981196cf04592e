"""Measured calls of a decoding step around the paged key / value cache, with their plain forms:
functs::rotary (rotary positions), kv_append (rotated keys and values into the cache), beam_select (the best
continuations of a beam search), kv_fork and kv_copy (the cache's pages after it).

Rotary positions: of a head's D columns the first R = 2 * len(frequencies) are pairs, column i with i + R / 2, or 2 i with
2 i + 1 (interleaved); pair i of a token at position p turns by the angle p * frequencies[i] and is multiplied by `magnitude`.

The cache: pages of P tokens, k_cache [N, H, P, D], v_cache [N, H, P / 16, D, 16] (codes of 8 bits: e4m3 or
int8), k_scale and v_scale [N, H] (fp32 powers of two); a value is its code times the scale of its page and head.
"""
import math
import random

import torch

own = False

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
MOST = {"e4m3": 448.0, "int8": 127.0}          # largest code
TOP = {"e4m3": 119, "int8": 121}               # largest exponent of a scale
LEAST = -100                                   # smallest exponent of a scale
DEVICE = "cuda"


# ---- cases ----
# rotary: batch 0: rows [tokens, heads, depth] out of a wider product; batch > 0: [batch, tokens, heads, depth], as `order` says
# ("tokens": a batch's tokens side by side, "heads": its heads).  turned: columns that turn.  stretch: frequencies divided by it
# (a context that much longer).  train: a backward pass too.
# append: requests with past_lo..past_hi cached tokens and new_lo..new_hi new ones, group query heads to a key head.
# select: masked: share of the vocabulary that may not follow.  ended: share of beams that are at their end.
# fork: lens lo..hi; first: the step after the prompts, whose beams all continue from one.  copy: layers whose pages are copied.

def listed():
    return [
        # a server's step: queries and keys of one token each, side by side as one product gives them
        dict(name="rotary_step", op="rotary", batch=0, tokens=61, heads=40, depth=128, turned=128, type="bf16", inter=False, start=0, spread=4001,
             stretch=1.0, order="tokens", train=False),
        # one long document behind what is cached of it, half of a head's columns turning in neighbouring pairs, a stretched context
        dict(name="rotary_document", op="rotary", batch=0, tokens=30001, heads=24, depth=64, turned=32, type="fp16", inter=True, start=100003, spread=0,
             stretch=8.0, order="tokens", train=False),
        # training: forward and backward
        dict(name="rotary_train", op="rotary", batch=3, tokens=1999, heads=40, depth=128, turned=128, type="bf16", inter=False, start=0, spread=0,
             stretch=1.0, order="tokens", train=True),
        # a server's step: 64 requests of all lengths, a token each
        dict(name="append_step", op="append", requests=64, past_lo=0, past_hi=4001, new_lo=1, new_hi=1, heads=8, group=4, depth=128, page=64,
             held="e4m3", type="bf16", turned=128, inter=False),
        # the prompts of a few requests
        dict(name="append_prompts", op="append", requests=5, past_lo=0, past_hi=0, new_lo=131, new_hi=4095, heads=8, group=4, depth=128, page=64,
             held="int8", type="fp16", turned=64, inter=True),
        # one request, four beams
        dict(name="select_one", op="select", requests=1, beams=4, words=32000, count=4, type="fp32", masked=0.0, ended=0.0),
        # a server's step, twice as many continuations as beams, an odd vocabulary
        dict(name="select_step", op="select", requests=16, beams=4, words=50001, count=8, type="fp16", masked=0.1, ended=0.0),
        # many requests of a large vocabulary, some beams at their end
        dict(name="select_many", op="select", requests=61, beams=8, words=128001, count=8, type="bf16", masked=0.0, ended=0.2),
        # a step of 32 requests of four beams
        dict(name="fork_step", op="fork", groups=32, beams=4, lo=100, hi=2000, page=64, first=False),
        # long requests of many beams, after their prompts
        dict(name="fork_long", op="fork", groups=61, beams=8, lo=1000, hi=30001, page=32, first=True),
        # a step's partly filled pages in all layers of a small model
        dict(name="copy_step", op="copy", groups=16, beams=4, layers=12, heads=12, depth=64, page=16, held="int8", first=False),
        # after the prompts: each one's last page for all its beams, in all layers
        dict(name="copy_first", op="copy", groups=8, beams=8, layers=24, heads=8, depth=128, page=64, held="e4m3", first=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "rotary", "append", "append", "select", "select", "fork", "copy"])
    kind = rng.choice(sorted(TYPES))
    if op == "rotary":
        depth = rng.choice([32, 64, 64, 72, 80, 96, 100, 128, 128, 128, 192, 256])
        turned = rng.choice([depth, depth, depth // 2, depth // 4, 2 * rng.randint(1, depth // 2)]) // 2 * 2
        heads, train, batch = rng.randint(1, 64), rng.random() < 0.4, rng.choice([0, 0, 1, 2, 5])
        most = 30_000_000 // (heads * depth * max(1, batch) * (2 if kind == "fp32" else 1) * (1 if train else 2))
        return dict(op=op, batch=batch, tokens=_log(rng, 1, max(2, min(60000, most))), heads=heads, depth=depth, turned=turned, type=kind,
                    inter=rng.random() < 0.5, start=rng.choice([0, rng.randint(0, 1_000_000)]), spread=rng.choice([0, 0, rng.randint(1, 200_000)]),
                    stretch=rng.choice([1.0, 4.0, 32.0]), order=rng.choice(["tokens", "heads"]), train=train)
    if op == "append":
        tokens, heads, depth = _log(rng, 1, 9000), rng.randint(1, 8), rng.choice([32, 64, 64, 80, 96, 128, 128, 192, 256])
        requests = min(tokens, _log(rng, 1, 200))
        hi, past = max(1, tokens // requests), rng.randint(0, 5000)
        return dict(op=op, requests=requests, past_lo=0, past_hi=past, new_lo=max(1, hi // rng.randint(1, 4)), new_hi=hi, heads=heads,
                    group=rng.randint(1, 8), depth=depth, page=rng.choice([16, 32, 64, 128, 256]), held=rng.choice(sorted(MOST)), type=kind,
                    turned=rng.choice([depth, depth, depth // 2, 2 * rng.randint(1, depth // 2)]), inter=rng.random() < 0.5)
    if op == "select":
        words, beams = _log(rng, 50, 200000), rng.randint(1, 16)
        requests = _log(rng, 1, max(1, min(128, 60_000_000 // (words * beams * (2 if kind == "fp32" else 1)))))
        return dict(op=op, requests=requests, beams=beams, words=words, count=rng.choice([beams, beams, 2 * beams, rng.randint(1, 2 * beams)]),
                    type=kind, masked=rng.choice([0.0, 0.0, 0.1, 0.9]), ended=rng.choice([0.0, 0.0, 0.3]))
    beams, page = rng.choice([1, 2, 3, 4, 4, 5, 8, 8, 12, 16]), rng.choice([16, 32, 64, 128, 256])
    if op == "fork":
        groups = _log(rng, 1, 600 // beams)
        hi = _log(rng, 1, 30000)
        return dict(op=op, groups=groups, beams=beams, lo=rng.randint(0, hi), hi=hi, page=page, first=rng.random() < 0.4)
    heads, depth = rng.randint(1, 12), rng.choice([32, 64, 64, 80, 96, 128, 128, 256])
    pages = max(1, 4500 * 8 * 64 * 128 // (heads * depth * page))
    layers = _log(rng, 1, 40)
    return dict(op=op, groups=_log(rng, 1, max(1, min(600, pages // layers // 2) // beams)), beams=beams, layers=layers, heads=heads, depth=depth, page=page,
                held=rng.choice(sorted(MOST)), first=rng.random() < 0.4)


def _spread(lo, hi, i, n):
    return lo + (hi - lo) * i // max(1, n - 1)


def _lengths(case):
    """(past, new) of each request of an append: the same pairs whatever the seed, which only shuffles them."""
    n = case["requests"]
    return [(_spread(case["past_lo"], case["past_hi"], i, n), _spread(case["new_lo"], case["new_hi"], i * 7919 % n if n > 1 else 0, n)) for i in range(n)]


def _lens(case):
    """Cached tokens of each group of beams of a fork or copy."""
    if case["op"] == "copy":
        return [(i * 29 + 7) % (case["page"] - 1) + 1 + 3 * case["page"] for i in range(case["groups"])]
    return [_spread(case["lo"], case["hi"], i, case["groups"]) for i in range(case["groups"])]


# ---- inputs ----

def _exponent(amax, held):
    """The least e with amax <= MOST 2^e, held to its range."""
    m, x = torch.frexp(amax)
    tm, tx = math.frexp(MOST[held])
    e = x - tx + (m > tm).to(x.dtype)
    return torch.where(amax > 0, e.clamp(LEAST, TOP[held]), torch.full_like(e, LEAST))


def _scale(amax, held):
    return torch.ldexp(torch.ones_like(amax), _exponent(amax, held))


def _codes(x, held):
    """x (fp32, already divided by its scale) as codes: uint8 bits of e4m3 or of int8."""
    if held == "e4m3":
        return x.clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8)
    return x.round().clamp(-127.0, 127.0).to(torch.int8).view(torch.uint8)


def _values(bits, held):
    return bits.view(torch.float8_e4m3fn if held == "e4m3" else torch.int8).float()


def _frequencies(turned, stretch=1.0):
    return (10000.0 ** (-torch.arange(0, turned, 2, dtype=torch.float64) / turned) / stretch).to(DEVICE)


def _parents(case, g):
    """[groups, beams]: which beam of its group each one continues from: all from the first after the prompts, else the good ones more than once."""
    G, K = case["groups"], case["beams"]
    if case["first"]:
        return torch.zeros(G, K, dtype=torch.int32, device=DEVICE)
    skill = torch.rand(G, K, generator=g, device=DEVICE)
    return torch.multinomial(skill.square() + 0.05, K, replacement=True, generator=g).to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    normal = lambda *size: torch.randn(*size, generator=g, device=DEVICE)  # noqa: E731
    op = case["op"]
    if op == "rotary":
        T, H, D, B, kind = case["tokens"], case["heads"], case["depth"], case["batch"], TYPES[case["type"]]
        steps = torch.arange(T, dtype=torch.int32, device=DEVICE) + case["start"]
        if B == 0:
            x = normal(T, H + max(1, H // 4), D).to(kind)[:, :H]            # values lie behind the queries and keys
            moved = torch.randint(0, case["spread"] + 1, (T,), generator=g, device=DEVICE).to(torch.int32)
            positions = case["start"] + moved if case["spread"] else steps
        else:
            x = normal(B, T, H, D).to(kind) if case["order"] == "tokens" else normal(B, H, T, D).to(kind).transpose(1, 2)
            moved = torch.randint(0, case["spread"] + 1, (B, 1), generator=g, device=DEVICE).to(torch.int32)
            positions = steps + moved if case["spread"] else steps
        s = dict(op=op, x=x, positions=positions, frequencies=_frequencies(case["turned"], case["stretch"]), inter=case["inter"], train=case["train"],
                 magnitude=1.0 if case["stretch"] == 1.0 else 0.1 * math.log(case["stretch"]) + 1.0)
        if case["train"]:
            s["grad"] = torch.randn(x.shape, generator=g, device=DEVICE).to(kind)
            s["leaf"] = x.detach().requires_grad_()
        return s
    if op == "select":
        B, K, V, kind = case["requests"], case["beams"], case["words"], TYPES[case["type"]]
        x = normal(B, K, V).mul_(2.0)
        n = max(1, min(20, V // 4))
        likely = torch.randint(0, V // n, (B, K, n), generator=g, device=DEVICE) + torch.arange(n, device=DEVICE) * (V // n)
        x.scatter_add_(2, likely, 6.0 + 3.0 * normal(*likely.shape))       # a few words stand out
        if case["masked"]:
            x.masked_fill_(torch.rand(1, 1, V, generator=g, device=DEVICE) < case["masked"], -math.inf)
        scores = (normal(B, K).mul_(2.0) - 30.0).sort(1, descending=True).values
        s = dict(op=op, logits=x.to(kind), scores=scores, count=case["count"], ended=None, end=V - 1)
        if case["ended"]:
            s["ended"] = torch.rand(B, K, generator=g, device=DEVICE) < case["ended"]
        return s
    if op in ("fork", "copy"):
        G, K, P = case["groups"], case["beams"], case["page"]
        order = _lens(case)
        random.Random(seed).shuffle(order)
        one = torch.tensor(order, dtype=torch.int32, device=DEVICE)
        parents = _parents(case, g)
        if op == "copy":
            # what kv_fork says of these beams, where each has its own last page
            L, H, D, held = case["layers"], case["heads"], case["depth"], case["held"]
            N = 3 * G * K
            pages = torch.randperm(N, generator=g, device=DEVICE)[:2 * G * K].to(torch.int32).view(2, G, K)
            tail = torch.gather(pages[0], 1, parents.long())
            again = (parents[:, :, None] == parents[:, None, :]).tril(-1).any(2)
            filled = (one % P)[:, None].expand(G, K)
            copies = torch.stack([torch.where(again, tail, -1), torch.where(again, pages[1], -1), torch.where(again, filled, 0)], 2).view(G * K, 3).contiguous()
            shape = (L, N, H, P, D), (L, N, H, P // 16, D, 16)
            caches = [torch.randint(0, 0x7f, z, generator=g, device=DEVICE, dtype=torch.uint8) for z in shape]
            scales = [torch.exp2(torch.randint(-9, 3, (L, N, H), generator=g, device=DEVICE).float()) for _ in shape]
            dtype = torch.float8_e4m3fn if held == "e4m3" else torch.int8
            return dict(op=op, page=P, copies=copies, caches=[c.view(dtype) for c in caches] + scales,
                        layers=[[t[i] for i in range(L)] for t in [c.view(dtype) for c in caches] + scales])
        lens = one[:, None].repeat(1, K)
        if case["first"]:
            lens[:, 1:] = 0
        M = case["hi"] // P + 2
        used = -(-lens // P)
        full = lens // P
        column = torch.arange(M, device=DEVICE)
        N = G * K * M + 2 * G * K
        pages = torch.randperm(N, generator=g, device=DEVICE).to(torch.int32)
        table = pages[:G * K * M].view(G, K, M)
        # beams have the pages of their common past in common, up to a third of it behind the prompt
        shared = (full[:, :1] - (full[:, :1] // 3 * torch.rand(G, K, generator=g, device=DEVICE)).int()) if not case["first"] else torch.zeros_like(lens)
        table = torch.where(column < shared[..., None], table[:, :1], table)
        table = torch.where(column < used[..., None], table, -1).view(G * K, M).contiguous()
        return dict(op=op, page=P, parents=parents, lens=lens.reshape(-1).contiguous(), table=table, free=pages[G * K * M:].contiguous())
    # append
    order = _lengths(case)
    random.Random(seed).shuffle(order)
    P, B, H, D, held, kind, G = case["page"], len(order), case["heads"], case["depth"], case["held"], TYPES[case["type"]], case["group"]
    used = [-(-(p + n) // P) - p // P for p, n in order]                     # pages that the step writes to
    tokens, N = sum(n for _, n in order), sum(used) + 3
    pages = torch.randperm(N, generator=g, device=DEVICE)
    at = [sum(used[:b]) for b in range(B)]
    column_k = torch.exp(0.7 * normal(H, 1, D))
    k, v = normal(N, H, P, D) * column_k * torch.exp(0.3 * normal(N, H, 1, 1)), normal(N, H, P, D) * torch.exp(0.5 * normal(N, H, 1, 1))
    ks, vs = _scale(k.abs().amax((2, 3)), held), _scale(v.abs().amax((2, 3)), held)
    dtype = torch.float8_e4m3fn if held == "e4m3" else torch.int8
    kc = _codes(k / ks[:, :, None, None], held).view(dtype)
    vc = _codes(v / vs[:, :, None, None], held).view(N, H, P // 16, 16, D).transpose(3, 4).contiguous().view(dtype)
    slots = lambda b, lo, hi: pages[at[b] + torch.arange(lo, hi, device=DEVICE) // P - order[b][0] // P] * P + torch.arange(lo, hi, device=DEVICE) % P  # noqa: E731
    qkv = normal(tokens, (G + 2) * H, D)
    qkv[:, G * H:(G + 1) * H] *= column_k[:, 0] * torch.exp(0.5 * normal(tokens, H, 1))
    qkv = qkv.to(kind)                                                       # as one product gives them
    return dict(op=op, page=P, held=held, runs=sum(used), q=qkv[:, :G * H], k=qkv[:, G * H:(G + 1) * H], v=qkv[:, (G + 1) * H:],
                cache=(kc, vc, ks, vs), frequencies=_frequencies(case["turned"]), inter=case["inter"], magnitude=1.0,
                slots=torch.cat([slots(b, p, p + n) for b, (p, n) in enumerate(order)]),
                seen=torch.cat([slots(b, p // P * P, p + n) for b, (p, n) in enumerate(order)]),   # what lies in the pages that the call writes to
                positions=torch.cat([torch.arange(p, p + n, device=DEVICE) for p, n in order]).to(torch.int32), order=order)


# ---- plain forms ----

def _turn(x, s, back=False):
    """x [..., heads, depth] turned (or, for gradients, turned back), in fp32."""
    angle = s["positions"].double()[..., None] * s["frequencies"]
    c = (angle.cos() * s["magnitude"]).float()[..., None, :]
    d = (angle.sin() * (-s["magnitude"] if back else s["magnitude"])).float()[..., None, :]
    n = 2 * s["frequencies"].numel()
    x = x.float()
    a, b = (x[..., 0:n:2], x[..., 1:n:2]) if s["inter"] else (x[..., :n // 2], x[..., n // 2:n])
    u, w = a * c - b * d, b * c + a * d
    y = torch.stack([u, w], -1).flatten(-2) if s["inter"] else torch.cat([u, w], -1)
    return torch.cat([y, x[..., n:]], -1)


def _append_one(x, cache, scales, page, off, first, runs, held, P, transposed):
    """One of the two caches. x [T, H, D] fp32; first [N]: least offset written of each page (P: none); runs: the pages written."""
    H = scales.size(1)
    bits = cache.view(torch.uint8)
    amax = torch.zeros_like(scales).scatter_reduce(0, page[:, None].expand(-1, H), x.abs().amax(2), "amax")[runs]
    was, old, at = bits[runs], scales[runs], first[runs][:, None]
    scale = _scale(amax, held)
    scale = torch.where(at == 0, scale, torch.maximum(old, scale))
    scales[runs] = scale
    # what a page holds already, under its new scale
    more = [1] * (was.dim() - 2)
    again = _codes(_values(was, held) * (old / scale).view([-1, H] + more), held)
    offs = torch.arange(P, device=x.device).view((1, 1, P // 16, 1, 16) if transposed else (1, 1, P, 1))
    bits[runs] = torch.where(offs < at.view([-1, 1] + more), again, was)
    codes = _codes(x / scales[page][:, :, None], held)
    if transposed:
        bits[page, :, off // 16, :, off % 16] = codes
    else:
        bits[page, :, off] = codes


def _append_plain(s):
    P, slots, held = s["page"], s["slots"], s["held"]
    kc, vc, ks, vs = s["cache"]
    N = ks.size(0)
    page, off = slots // P, slots % P
    first = torch.full((N,), P, dtype=torch.long, device=slots.device).scatter_reduce(0, page, off, "amin")
    leads = first[page] == off
    place = torch.where(leads, leads.long().cumsum(0) - 1, s["runs"])
    runs = torch.zeros(s["runs"] + 1, dtype=torch.long, device=slots.device).scatter(0, place, page)[:s["runs"]]
    _append_one(_turn(s["k"], s), kc, ks, page, off, first, runs, held, P, False)
    _append_one(s["v"].float(), vc, vs, page, off, first, runs, held, P, True)
    return (_turn(s["q"], s).to(s["q"].dtype),) + _held_plain(s)


def _held_plain(s):
    """The values of the pages written, which bf16 holds exactly."""
    P, held, slots = s["page"], s["held"], s["seen"]
    kc, vc, ks, vs = s["cache"]
    page, off = slots // P, slots % P
    k = _values(kc.view(torch.uint8)[page, :, off], held) * ks[page][:, :, None]
    v = _values(vc.view(torch.uint8)[page, :, off // 16, :, off % 16], held) * vs[page][:, :, None]
    return k.to(torch.bfloat16), v.to(torch.bfloat16)


def _select_plain(s):
    """Continuations in the order of their scores in 64 bits; equal ones in the order of their beams, in a beam of logits, then of words."""
    x, scores, count = s["logits"], s["scores"].double(), s["count"]
    B, K, V = x.shape
    n = min(count, V)
    top = x.amax(2, keepdim=True).double()
    lse = (x.double() - top).exp_().sum(2, keepdim=True).log_() + top
    # a logit and its word as one whole number: larger logits first, then lower words
    bits = (x.float() + 0.0).view(torch.int32)
    bits = torch.where(bits < 0, bits ^ 0x7fffffff, bits).long()
    words = torch.arange(V, device=x.device)
    words = (V - 1) - ((bits << 32) + (V - 1 - words)).topk(n, dim=2).values.bitwise_and(0xffffffff)
    best = torch.gather(x, 2, words).double()
    total = scores[..., None] + (best - lse)
    if s["ended"] is not None:
        only = torch.arange(n, device=x.device) == 0
        total = torch.where(s["ended"][..., None], torch.where(only, scores[..., None], -math.inf), total)
        words = torch.where(s["ended"][..., None], s["end"], words)
    total = torch.where(total > -math.inf, total, -math.inf).view(B, K * n)
    total, at = total.sort(dim=1, descending=True, stable=True)
    m = min(count, K * n)
    total, at = total[:, :m], at[:, :m]
    there = total > -math.inf
    out = torch.full((B, count), -math.inf, device=x.device), torch.full((B, count), -1, dtype=torch.int32, device=x.device), \
        torch.full((B, count), -1, dtype=torch.long, device=x.device)
    out[0][:, :m] = total.float()
    out[1][:, :m] = torch.where(there, at // n, -1).int()
    out[2][:, :m] = torch.where(there, torch.gather(words.reshape(B, K * n), 1, at), -1)
    return out


def _fork_plain(s):
    parents, table, P, free = s["parents"].long(), s["table"], s["page"], s["free"]
    G, K = parents.shape
    M, F = table.size(1), free.numel()
    lens = s["lens"].long().view(G, K)
    lens = torch.where((lens >= 0) & (lens <= M * P), lens, 0)
    old = table.view(G, K, M)
    column = torch.arange(M, device=table.device)
    cols, full = (lens + P - 1) // P, lens // P
    tail = torch.where(lens % P > 0, torch.gather(old, 2, full.clamp(max=M - 1)[..., None])[..., 0], -1)
    has = (parents >= 0) & (parents < K)
    p = parents.clamp(0, K - 1)
    n = torch.where(has, torch.gather(lens, 1, p), 0)
    t = torch.where(has, torch.gather(tail, 1, p), -1)
    # of the beams that continue a partly filled page the first has it, the others get copies
    need = ((t[:, :, None] == t[:, None, :]).tril(-1).any(2)) & (t >= 0)
    spare = (tail >= 0) & ~(t[:, None, :] == tail[:, :, None]).any(2) & ~(tail[:, :, None] == tail[:, None, :]).tril(-1).any(2)
    rank, spares = need.cumsum(1) - need.long(), spare.sum(1, keepdim=True)
    asked = (need.sum(1, keepdim=True) - spares).clamp(min=0)
    index = asked.cumsum(0) - asked + rank - spares                          # of the free pages
    order = torch.where(spare, spare.cumsum(1) - 1, K)
    spare_pages = torch.full((G, K + 1), -1, dtype=table.dtype, device=table.device).scatter(1, order, tail)
    granted = ~need | (rank < spares) | (index < F)
    fresh = free[index.clamp(0, max(0, F - 1))] if F else torch.full_like(tail, -1)
    page = torch.where(rank < spares, torch.gather(spare_pages, 1, rank.clamp(max=K)), fresh)
    copied = need & granted
    # tables
    new = torch.gather(old, 1, p[..., None].expand(G, K, M))
    last = torch.where(need, page, t)
    here = (has & granted)[..., None]
    whole = (n // P)[..., None]
    moved = torch.where(here & (column < whole), new, torch.where(here & (column == whole) & (n % P > 0)[..., None], last[..., None], old))
    # pages that no beam has any more
    alive = (here[..., 0][:, None, :] & (p[:, None, :] == torch.arange(K, device=table.device)[:, None])).any(2)
    reused = spare & (spare.cumsum(1) <= need.sum(1, keepdim=True))
    holds = (column < cols[..., None]) & (old >= 0)
    same = (old[:, :, None] == old[:, None, :]) & holds[:, :, None] & holds[:, None, :]   # [G, K (i), K (other), M]
    before = torch.ones(K, K, dtype=torch.bool, device=table.device).tril(-1)
    kept = (same & (alive[:, None, :] | (before & ~alive[:, None, :]))[..., None]).any(2)
    gone = holds & ~alive[..., None] & ~kept & ~((column == full[..., None]) & reused[..., None])
    gone = gone.transpose(1, 2).reshape(-1)
    place = torch.where(gone, gone.long().cumsum(0) - 1, G * K * M)
    freed = torch.full((G * K * M + 1,), -1, dtype=torch.int32, device=table.device).scatter(0, place, old.transpose(1, 2).reshape(-1))[:-1]
    table.copy_(moved.view(G * K, M))
    copies = torch.stack([torch.where(copied, t, -1), torch.where(copied, page, -1), torch.where(copied, n % P, 0)], 2)
    taken = (copied & (rank >= spares)).sum().to(torch.int32).view(1)
    return (torch.where(granted, n, 0).to(torch.int32).view(-1), copies.to(torch.int32).view(G * K, 3), taken, freed, gone.sum().to(torch.int32).view(1), table)


def _copy_plain(s):
    kc, vc, ks, vs = s["caches"]
    src, dst, filled = s["copies"].long().unbind(1)
    N, P = ks.size(1), s["page"]
    # rows that copy nothing do what one that does is doing; with none of those the first page becomes itself
    live = dst >= 0
    one = live.long().argmax()
    some, come, fill = (torch.where(live, t, t[one]) for t in (dst, src, filled))
    some, come = some.clamp(0, N - 1), come.clamp(0, N - 1)
    token = torch.arange(P, device=kc.device)
    keys, values = kc.view(torch.uint8), vc.view(torch.uint8)
    seen = (token < fill[:, None]).view(1, -1, 1, P, 1)
    keys[:, some] = torch.where(seen, keys[:, come], keys[:, some])
    seen = (token < ((fill + 15) // 16 * 16)[:, None]).view(1, -1, 1, P // 16, 1, 16)    # values: whole groups of 16 tokens
    values[:, some] = torch.where(seen, values[:, come], values[:, some])
    ks[:, some], vs[:, some] = ks[:, come], vs[:, come]
    return kc, vc, ks, vs


def run(s):
    op = s["op"]
    if own:
        import functs_amd.jit  # noqa: F401  (registers the operators)
        ops = torch.ops.functs
        if op == "rotary":
            if not s["train"]:
                return ops.rotary(s["x"], s["positions"], s["frequencies"], s["magnitude"], s["inter"])
            y = ops.rotary(s["leaf"], s["positions"], s["frequencies"], s["magnitude"], s["inter"])
            return y.detach(), torch.autograd.grad(y, s["leaf"], s["grad"])[0]
        if op == "append":
            q = ops.kv_append(s["q"], s["k"], s["v"], *s["cache"], s["slots"], s["positions"], s["frequencies"], s["magnitude"], s["inter"])
            return (q,) + ops.kv_read(*s["cache"], s["seen"], torch.bfloat16)
        if op == "select":
            return ops.beam_select(s["logits"], s["scores"], s["count"], s["ended"], s["end"])
        if op == "fork":
            return ops.kv_fork(s["parents"], s["lens"], s["table"], s["free"], s["page"]) + (s["table"],)
        ops.kv_copy(*s["layers"], s["copies"])
        return tuple(s["caches"])
    if op == "rotary":
        y = _turn(s["x"], s).to(s["x"].dtype)
        return (y, _turn(s["grad"], s, back=True).to(y.dtype)) if s["train"] else y
    if op == "append":
        return _append_plain(s)
    if op == "select":
        return _select_plain(s)
    return _fork_plain(s) if op == "fork" else _copy_plain(s)


# ---- what a pass cannot do without ----

def work(case):
    op = case["op"]
    if op == "rotary":
        n = case["tokens"] * max(1, case["batch"])
        size, passes = TYPES[case["type"]].itemsize, 2 if case["train"] else 1
        return {"bytes": passes * (2 * n * case["heads"] * case["depth"] * size + 4 * n), "flops": passes * 3 * n * case["heads"] * case["turned"]}
    if op == "append":
        order, P, H, D, G, size = _lengths(case), case["page"], case["heads"], case["depth"], case["group"], TYPES[case["type"]].itemsize
        tokens, seen = sum(n for _, n in order), sum(p + n - p // P * P for p, n in order)
        return {"bytes": tokens * (2 * G * H * D * size + 2 * H * D * (size + 1) + 12) + seen * (2 * H * D * 3 + 8),
                "flops": tokens * ((G + 1) * 3 * H * case["turned"] + 4 * H * D) + 2 * H * D * seen}
    if op == "select":
        rows = case["requests"] * case["beams"]
        rows *= 1 - case["ended"]                                             # (a beam at its end has one continuation, whatever its logits are)
        return {"bytes": rows * case["words"] * TYPES[case["type"]].itemsize + 4 * rows + 16 * case["requests"] * case["count"],
                "flops": 4 * rows * case["words"]}
    lens, P, K = _lens(case), case["page"], case["beams"]
    if op == "fork":
        return {"bytes": sum(K * (-(-n // P) * 8 + 24) for n in lens), "flops": 0}
    copies = K - 1 if case["first"] else K // 3                                # (about: a third of the beams have no page of their own)
    return {"bytes": case["layers"] * sum(copies * case["heads"] * (case["depth"] * 2 * (n % P + -(-(n % P) // 16) * 16) + 16) for n in lens) + 12 * K * len(lens),
            "flops": 0}


# ---- from the definition, in 64 bits ----

def _exact_turn(x, s, back=False):
    """Pairs as complex numbers times magnitude e^(i p f)."""
    n = 2 * s["frequencies"].numel()
    angle = s["positions"].double().unsqueeze(-1) * s["frequencies"]
    z = torch.polar(torch.full_like(angle, s["magnitude"]), -angle if back else angle).unsqueeze(-2)
    y = x.double().clone()
    if s["inter"]:
        y[..., :n] = torch.view_as_real(torch.view_as_complex(y[..., :n].unflatten(-1, (-1, 2)).contiguous()) * z).flatten(-2)
    else:
        w = torch.complex(y[..., :n // 2], y[..., n // 2:n]) * z
        y[..., :n // 2], y[..., n // 2:n] = w.real, w.imag
    return y


def _exact_code(x, held):
    """x (already divided by its scale) rounded to the nearest code, ties to even."""
    if held == "int8":
        return torch.round(x).clamp(-127, 127)
    x = x.clamp(-448, 448)
    step = torch.exp2(torch.frexp(x)[1].clamp(min=-5).to(x.dtype) - 4.0)     # of x's binade: three bits behind the first
    return torch.round(x / step) * step


def _exact_append(s):
    P, held, order = s["page"], s["held"], s["order"]
    kc, vc, ks, vs = s["cache"]
    answer = []
    for name, codes, scales in (("k", kc, ks), ("v", vc, vs)):
        new = _exact_turn(s["k"], s) if name == "k" else s["v"].double()
        page, off = s["seen"] // P, s["seen"] % P
        codes = codes.float().double()
        before = (codes[page, :, off] if name == "k" else codes[page, :, off // 16, :, off % 16]) * scales.double()[page][:, :, None]
        at, t, parts = 0, 0, []
        for p, n in order:
            lead = p % P
            rows = torch.cat([before[at:at + lead], new[t:t + n]])
            pages = (s["seen"][at:at + lead + n:P] // P).tolist()
            at, t = at + lead + n, t + n
            for c, here in zip(range(0, lead + n, P), pages):
                part, fresh = rows[c:c + P], lead if c == 0 else 0
                amax = part[fresh:].abs().amax((0, 2))
                e = torch.frexp(amax / MOST[held])[1].double()                # a / most in [2^(e - 1), 2^e)
                e = torch.where(MOST[held] * torch.exp2(e - 1) >= amax, e - 1, e)
                e = torch.where(amax > 0, e.clamp(LEAST, TOP[held]), float(LEAST))
                scale = torch.exp2(e)
                if fresh:
                    scale = torch.maximum(scale, scales[here].double())
                parts.append(_exact_code(part / scale[:, None], held) * scale[:, None])
        answer.append(torch.cat(parts))
    return _exact_turn(s["q"], s), answer[0], answer[1]


def _exact_select(s):
    """Of each request all continuations in 64 bits, one request after the other."""
    answer = []
    for b in range(s["logits"].size(0)):
        total = torch.log_softmax(s["logits"][b].double(), 1) + s["scores"][b].double()[:, None]
        if s["ended"] is not None:
            total[s["ended"][b]] = -math.inf
            total[s["ended"][b], s["end"]] = s["scores"][b][s["ended"][b]].double()
        best = total.flatten().topk(min(s["count"], total.numel())).values
        answer.append(torch.cat([best, best.new_full((s["count"] - best.numel(),), -math.inf)]))
    return torch.stack(answer), None, None


def _exact_copy(s):
    """One copy after the other; codes as the numbers that they are."""
    kc, vc, ks, vs = s["caches"]
    keys, values, ks, vs = kc.float(), vc.float(), ks.clone(), vs.clone()
    for src, dst, n in s["copies"].tolist():
        if dst >= 0:
            keys[:, dst, :, :n] = keys[:, src, :, :n]
            values[:, dst, :, :-(-n // 16)] = values[:, src, :, :-(-n // 16)]
            ks[:, dst], vs[:, dst] = ks[:, src], vs[:, src]
    return (None, None, ks, vs) if kc.dtype == torch.int8 else (keys, values, ks, vs)   # (int8 codes are compared for equality)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        return (_exact_turn(s["x"], s), _exact_turn(s["grad"], s, back=True)) if s["train"] else _exact_turn(s["x"], s)
    if case["op"] == "append":
        return _exact_append(s)
    if case["op"] == "select":
        return _exact_select(s)
    return _exact_copy(s) if case["op"] == "copy" else None                   # (a fork gives whole numbers alone)
