"""Measured calls of the paged 8-bit key / value cache: functs::kv_plan, kv_store, kv_read and
kv_attention, with their plain forms.

The cache: pages of P tokens, k_cache [N, H, P, D], v_cache [N, H, P / 16, D, 16] (codes of 8 bits:
e4m3 or int8), k_scale and v_scale [N, H] (fp32 powers of two); a value is its code times the scale of
its page and head.  Request b's tokens j lie in page table[b, j // P] at offset j % P.
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
# requests: how many; past / new: lengths from (lo) to (hi), spread evenly over the requests; heads: key / value
# heads, group: query heads to each; window 0: all tokens before a row

def listed():
    return [
        # the step of a small server: 17 requests, a token each
        dict(name="plan_step", op="plan", requests=17, past_lo=0, past_hi=1000, new_lo=1, new_hi=1, page=64),
        # many requests at once, some idle, some with whole prompts
        dict(name="plan_prompts", op="plan", requests=700, past_lo=0, past_hi=3001, new_lo=0, new_hi=255, page=32),
        # one token of each of 96 requests, in pages that hold others already
        dict(name="store_step", op="store", requests=96, past_lo=3, past_hi=500, new_lo=1, new_hi=1, heads=8, depth=128, page=16,
             held="e4m3", type="bf16"),
        # the prompts of a few requests, of any length
        dict(name="store_prompts", op="store", requests=9, past_lo=0, past_hi=0, new_lo=131, new_hi=4095, heads=8, depth=128, page=64,
             held="int8", type="fp16"),
        # the cache of the attention program (12 heads of 64, 50 rows, fp32) as values again
        dict(name="read_short", op="read", requests=1, past_lo=0, past_hi=0, new_lo=50, new_hi=50, heads=12, depth=64, page=16,
             held="int8", type="fp32"),
        # a long prefix handed to a path that takes bf16
        dict(name="read_prefix", op="read", requests=3, past_lo=0, past_hi=0, new_lo=1001, new_hi=16001, heads=8, depth=128, page=128,
             held="e4m3", type="bf16"),
        # a step of the attention program: one row, 12 heads of 64, 50 cached rows, fp32
        dict(name="attend_short", op="attention", requests=1, past_lo=49, past_hi=49, new_lo=1, new_hi=1, heads=12, group=1, depth=64,
             page=16, held="int8", type="fp32", window=0),
        # a step of a server: 64 requests of all lengths
        dict(name="attend_step", op="attention", requests=64, past_lo=0, past_hi=4001, new_lo=1, new_hi=1, heads=8, group=4, depth=128,
             page=64, held="e4m3", type="bf16", window=0),
        # one long document
        dict(name="attend_long", op="attention", requests=1, past_lo=130001, past_hi=130001, new_lo=1, new_hi=1, heads=8, group=8, depth=128,
             page=128, held="e4m3", type="fp16", window=0),
        # a few drafted tokens each, checked at once, within a window, an odd depth
        dict(name="attend_drafts", op="attention", requests=24, past_lo=5, past_hi=2500, new_lo=1, new_hi=7, heads=4, group=5, depth=80,
             page=32, held="int8", type="fp16", window=1000),
        # prompts in pieces behind what is cached of them
        dict(name="attend_prompts", op="attention", requests=4, past_lo=0, past_hi=6001, new_lo=511, new_hi=2047, heads=8, group=4, depth=128,
             page=64, held="e4m3", type="bf16", window=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "store", "read", "attention", "attention"])
    page = rng.choice([16, 32, 64, 128, 256])
    if op == "plan":
        requests = _log(rng, 1, 1500)
        most = max(1, min(2000, 150000 // requests))
        lo, hi = sorted((rng.randint(0, most), rng.randint(1, most)))
        past = rng.randint(0, 5000)
        return dict(op=op, requests=requests, past_lo=rng.randint(0, past), past_hi=past, new_lo=lo, new_hi=hi, page=page)
    heads, depth, held, kind = rng.randint(1, 12), rng.choice([32, 64, 64, 80, 96, 128, 128, 128, 192, 256]), rng.choice(sorted(MOST)), rng.choice(sorted(TYPES))
    if op in ("store", "read"):
        tokens = _log(rng, 1, 16000)
        requests = min(tokens, _log(rng, 1, 200))
        hi = max(1, tokens // requests)
        past = rng.randint(0, 600) if op == "store" else 0
        return dict(op=op, requests=requests, past_lo=0, past_hi=past, new_lo=max(1, hi // rng.randint(1, 4)), new_hi=hi, heads=heads,
                    depth=depth, page=page, held=held, type=kind)
    form = rng.choice(["single", "single", "few", "prompt"])
    requests = _log(rng, 1, 100) if form != "prompt" else rng.randint(1, 3)
    new = 1 if form == "single" else rng.randint(2, 12) if form == "few" else _log(rng, 20, 700)
    past = _log(rng, 1, 60000 // requests) if form != "prompt" else _log(rng, 1, 2500)
    return dict(op=op, requests=requests, past_lo=rng.randint(0, past), past_hi=past, new_lo=rng.randint(1, new), new_hi=new, heads=min(heads, 8),
                group=rng.choice([1, 1, 2, 3, 4, 5, 7, 8, 12, 16]) if form != "prompt" else rng.choice([1, 2, 4, 5]), depth=depth, page=page, held=held, type=kind,
                window=rng.choice([0, 0, 0, rng.randint(1, 2000)]))


def _lengths(case):
    """(past, new) of each request: the same pairs whatever the seed, which only shuffles them."""
    n = case["requests"]
    spread = lambda lo, hi, i: lo + (hi - lo) * i // max(1, n - 1)  # noqa: E731
    return [(spread(case["past_lo"], case["past_hi"], i), spread(case["new_lo"], case["new_hi"], i * 7919 % n if n > 1 else 0)) for i in range(n)]


# ---- inputs ----

def _exponent(amax, held):
    """The least e with amax <= MOST 2^e, held to its range."""
    top = MOST[held]
    m, x = torch.frexp(amax)
    tm, tx = math.frexp(top)
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


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    order = _lengths(case)
    random.Random(seed).shuffle(order)
    P, B = case["page"], len(order)
    past = torch.tensor([p for p, _ in order], dtype=torch.int32, device=DEVICE)
    new = torch.tensor([n for _, n in order], dtype=torch.int32, device=DEVICE)
    tokens = sum(n for _, n in order)
    starts = torch.zeros(B + 1, dtype=torch.int32, device=DEVICE)
    starts[1:] = new.cumsum(0)
    width = max(-(-(p + n) // P) for p, n in order) or 1
    used = [-(-(p + n) // P) for p, n in order]
    held_before = [-(-p // P) for p, _ in order]
    N = sum(used) + 3
    pages = torch.randperm(N, generator=g, device=DEVICE).to(torch.int32)   # pages lie in no order
    first = torch.zeros(B, dtype=torch.long, device=DEVICE)
    first[1:] = torch.tensor(used, device=DEVICE).cumsum(0)[:-1]
    column = torch.arange(width, device=DEVICE)
    place = (first[:, None] + column).clamp(max=N - 1)
    whole = torch.where(column < torch.tensor(used, device=DEVICE)[:, None], pages[place], -1).contiguous()
    s = dict(op=case["op"], page=P, past=past, new=new, starts=starts, tokens=tokens, requests=B, max_new=max(n for _, n in order))
    if case["op"] == "plan":
        # the table holds the pages of what is cached; the free ones are the others
        s["table"] = torch.where(column < torch.tensor(held_before, device=DEVICE)[:, None], whole, -1).contiguous()
        taken = torch.cat([whole[i, held_before[i]:used[i]] for i in range(B)] + [pages[sum(used):]])
        s["free"] = taken[torch.randperm(taken.numel(), generator=g, device=DEVICE)].contiguous()
        return s
    H, D, held, kind = case["heads"], case["depth"], case["held"], TYPES[case["type"]]
    normal = lambda *size: torch.randn(*size, generator=g, device=DEVICE)  # noqa: E731
    # keys have a few strong columns, values are even
    column_k = torch.exp(0.7 * normal(H, 1, D))
    s |= dict(held=held, kind=kind, heads=H, depth=D, table=whole, lens=past + new)
    kv = torch.empty(N, H, P, D, dtype=torch.uint8, device=DEVICE)
    vv = torch.empty(N, H, P // 16, D, 16, dtype=torch.uint8, device=DEVICE)
    ks, vs = torch.empty(N, H, device=DEVICE), torch.empty(N, H, device=DEVICE)
    step = max(1, (1 << 26) // (H * P * D))
    for i in range(0, N, step):
        n = min(step, N - i)
        k = normal(n, H, P, D) * column_k * torch.exp(0.3 * normal(n, H, 1, 1))
        v = normal(n, H, P, D) * torch.exp(0.5 * normal(n, H, 1, 1))
        ks[i:i + n], vs[i:i + n] = _scale(k.abs().amax((2, 3)), held), _scale(v.abs().amax((2, 3)), held)
        kv[i:i + n] = _codes(k / ks[i:i + n, :, None, None], held)
        vv[i:i + n] = _codes(v / vs[i:i + n, :, None, None], held).view(n, H, P // 16, 16, D).transpose(3, 4)
    dtype = torch.float8_e4m3fn if held == "e4m3" else torch.int8
    s |= dict(k_cache=kv.view(dtype), v_cache=vv.view(dtype), k_scale=ks, v_scale=vs)
    slots = lambda b, lo, hi: whole[b, torch.arange(lo, hi, device=DEVICE) // P].long() * P + torch.arange(lo, hi, device=DEVICE) % P  # noqa: E731
    if case["op"] == "attention":
        hq = H * case["group"]
        qkv = normal(tokens, hq + 2 * H, D)                       # queries beside new keys and values, as one product gives them
        s |= dict(q=qkv.to(kind)[:, :hq], scale=D ** -0.5, window=case["window"], group=case["group"])
        return s
    s["slots"] = torch.cat([slots(b, p, p + n) for b, (p, n) in enumerate(order)])
    if case["op"] == "store":
        kvn = torch.stack([normal(tokens, H, D) * column_k[:, 0] * torch.exp(0.5 * normal(tokens, H, 1)), normal(tokens, H, D)], dim=1).to(kind)
        s |= dict(k=kvn[:, 0], v=kvn[:, 1], runs=sum(-(-(p + n) // P) - p // P for p, n in order if n))
        # what lies in the pages that the call writes to, up to the last token
        s["seen"] = torch.cat([slots(b, p // P * P, p + n) for b, (p, n) in enumerate(order) if n])
    return s


# ---- plain forms ----

def _plan_plain(s):
    past, new, table, free, P = s["past"].long(), s["new"].long(), s["table"], s["free"], s["page"]
    B, M, most = table.size(0), table.size(1), s["tokens"]
    ends = new.cumsum(0)
    starts = torch.cat([ends.new_zeros(1), ends]).clamp(max=most)
    had, have = (past + P - 1) // P, (past + new + P - 1) // P
    fits = (past >= 0) & (new >= 0) & (past + new <= M * P) & (ends <= most)
    need = torch.where(fits, have - had, 0)
    upto = need.cumsum(0)
    granted = fits & ((need == 0) | (upto <= free.numel()))
    off = upto - need
    # tokens
    t = torch.arange(most, device=past.device)
    b = (starts[1:, None] <= t).sum(0)
    live = b < B
    b = b.clamp(max=B - 1)
    pos = past[b] + t - starts[b]
    live = live & granted[b]
    col = pos // P
    fresh = (off[b] + col - had[b]).clamp(0, max(0, free.numel() - 1))
    page = torch.where(col < had[b], table[b, col.clamp(0, M - 1)], free[fresh] if free.numel() else -1)
    slots = torch.where(live, page.long() * P + pos % P, -1)
    positions = torch.where(live, pos, -1).to(torch.int32)
    # new pages of the table
    column = torch.arange(M, device=past.device)
    here = granted[:, None] & (column >= had[:, None]) & (column < have[:, None])
    given = free[(off[:, None] + column - had[:, None]).clamp(0, max(0, free.numel() - 1))] if free.numel() else table
    table.copy_(torch.where(here, given, table))
    return (slots, positions, starts.to(torch.int32), torch.where(granted, past + new, 0).to(torch.int32),
            torch.where(granted, need, 0).sum().to(torch.int32).view(1), table)


def _store_plain_one(x, cache, scales, page, off, first, runs, held, P, transposed):
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


def _store_plain(s):
    P, slots, N, held = s["page"], s["slots"], s["k_scale"].size(0), s["held"]
    page, off = slots // P, slots % P
    first = torch.full((N,), P, dtype=torch.long, device=slots.device).scatter_reduce(0, page, off, "amin")
    leads = first[page] == off
    place = torch.where(leads, leads.long().cumsum(0) - 1, s["runs"])
    runs = torch.zeros(s["runs"] + 1, dtype=torch.long, device=slots.device).scatter(0, place, page)[:s["runs"]]
    _store_plain_one(s["k"].float(), s["k_cache"], s["k_scale"], page, off, first, runs, held, P, False)
    _store_plain_one(s["v"].float(), s["v_cache"], s["v_scale"], page, off, first, runs, held, P, True)
    return _read_plain(s, s["seen"]) + (s["k_scale"], s["v_scale"])


def _read_plain(s, slots):
    P, held = s["page"], s["held"]
    page, off = slots // P, slots % P
    k = _values(s["k_cache"].view(torch.uint8)[page, :, off], held) * s["k_scale"][page][:, :, None]
    v = _values(s["v_cache"].view(torch.uint8)[page, :, off // 16, :, off % 16], held) * s["v_scale"][page][:, :, None]
    return k.to(s["kind"]), v.to(s["kind"])


def _attention_plain(s):
    q, table, lens, starts, P, H, D, G = s["q"], s["table"], s["lens"].long(), s["starts"].long(), s["page"], s["heads"], s["depth"], s["group"]
    B, M, n, T = table.size(0), table.size(1), s["max_new"], q.size(0)
    N, L = s["k_scale"].size(0), table.size(1) * P
    inside = (table >= 0) & (table < N)
    pages = torch.where(inside, table, 0).long()
    j = torch.arange(L, device=q.device)
    cached = (j < lens[:, None]) & inside.repeat_interleave(P, 1)                                   # [B, L]
    k = _values(s["k_cache"].view(torch.uint8)[pages], s["held"]) * s["k_scale"][pages][..., None, None]   # [B, M, H, P, D]
    k = k.transpose(1, 2).reshape(B, H, L, D)
    v = _values(s["v_cache"].view(torch.uint8)[pages], s["held"]) * s["v_scale"][pages][..., None, None, None]
    v = v.permute(0, 2, 1, 3, 5, 4).reshape(B, H, L, D)
    k, v = (torch.where(cached[:, None, :, None], x, 0.0) for x in (k, v))
    # rows of each request side by side, padded to the longest
    i = torch.arange(n, device=q.device)
    count = starts[1:] - starts[:-1]
    live = i < count[:, None]                                                                      # [B, n]
    row = (starts[:-1, None] + i).clamp(max=max(0, T - 1))
    x = q.float()[row].view(B, n, H, G, D).permute(0, 2, 3, 1, 4).reshape(B, H, G * n, D)
    scores = torch.matmul(x, k.transpose(2, 3)).mul_(s["scale"]).view(B, H, G, n, L)
    pos = (lens - count)[:, None] + i                                                              # [B, n]
    sees = cached[:, None, :] & (j <= pos[..., None]) & live[..., None]
    if s["window"]:
        sees = sees & (j > pos[..., None] - s["window"])
    scores.masked_fill_(~sees[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, H, G * n, L), v).view(B, H, G, n, D) / torch.where(total > 0, total, 1.0)
    lse = (total.log() + top).squeeze(-1)
    # back to the packed rows
    t = torch.arange(T, device=q.device)
    b = (starts[1:, None] <= t).sum(0).clamp(max=B - 1)
    out = o.permute(0, 3, 1, 2, 4).reshape(B, n, H * G, D)[b, t - starts[b]]
    return out.to(q.dtype), lse.permute(0, 3, 1, 2).reshape(B, n, H * G)[b, t - starts[b]]


def run(s):
    if own:
        import functs_amd.jit  # noqa: F401  (registers the operators)
        ops = torch.ops.functs
        if s["op"] == "plan":
            return ops.kv_plan(s["past"], s["new"], s["table"], s["free"], s["page"], s["tokens"]) + (s["table"],)
        cache = (s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"])
        if s["op"] == "store":
            ops.kv_store(s["k"], s["v"], *cache, s["slots"])
            return ops.kv_read(*cache, s["seen"], s["kind"]) + cache[2:]
        if s["op"] == "read":
            return ops.kv_read(*cache, s["slots"], s["kind"])
        return ops.kv_attention(s["q"], *cache, s["table"], s["lens"], s["starts"], s["scale"], s["window"], s["max_new"])
    if s["op"] == "plan":
        return _plan_plain(s)
    if s["op"] == "store":
        return _store_plain(s)
    if s["op"] == "read":
        return _read_plain(s, s["slots"])
    return _attention_plain(s)


# ---- what a pass cannot do without ----

def work(case):
    order, P = _lengths(case), case["page"]
    tokens = sum(n for _, n in order)
    fresh = sum(-(-(p + n) // P) - -(-p // P) for p, n in order)
    if case["op"] == "plan":
        return {"bytes": 16 * len(order) + 12 * tokens + 8 * fresh, "flops": 0}
    H, D, size = case["heads"], case["depth"], TYPES[case["type"]].itemsize
    if case["op"] == "read":
        return {"bytes": 2 * tokens * H * D * (1 + size) + 8 * tokens, "flops": 2 * tokens * H * D}
    if case["op"] == "store":
        seen = sum(p + n - p // P * P for p, n in order if n)
        return {"bytes": 2 * H * D * (tokens * (size + 1) + seen * (1 + size)) + 8 * (tokens + seen), "flops": 2 * H * D * (2 * tokens + seen)}
    G, w = case["group"], case["window"]
    keys = pairs = 0
    for p, n in order:
        if not n:
            continue
        lowest = max(0, p - w + 1) if w else 0
        keys += p + n - lowest
        pairs += sum(min(p + i + 1, w) for i in range(n)) if w else n * p + n * (n + 1) // 2
    return {"bytes": 2 * keys * H * D + tokens * H * G * (2 * D * size + 4), "flops": 4 * pairs * H * G * D}


# ---- from the definition, in 64 bits ----

def _exact_code(x, held):
    """x (already divided by its scale) rounded to the nearest code, ties to even."""
    if held == "int8":
        return torch.round(x).clamp(-127, 127)
    x = x.clamp(-448, 448)
    e = torch.frexp(x)[1].clamp(min=-5).to(x.dtype) - 4.0       # the step of x's binade: three bits behind the first
    step = torch.exp2(e)
    return torch.round(x / step) * step


def _exact_held(s, slots, name):
    P = s["page"]
    page, off = slots // P, slots % P
    c = s[name + "_cache"]
    c = c.double() if c.dtype == torch.int8 else c.float().double()
    rows = c[page, :, off] if name == "k" else c[page, :, off // 16, :, off % 16]
    return rows * s[name + "_scale"].double()[page][:, :, None]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "plan":
        return None
    if case["op"] == "read":
        return _exact_held(s, s["slots"], "k"), _exact_held(s, s["slots"], "v")
    P, held = s["page"], s["held"]
    past, new, table = s["past"].tolist(), s["new"].tolist(), s["table"].tolist()
    if case["op"] == "store":
        answer = []
        for name in ("k", "v"):
            before, scales, parts, t = _exact_held(s, s["seen"], name), s[name + "_scale"].double(), [], 0
            r = 0
            for b, (p, n) in enumerate(zip(past, new)):
                x = s[name][t:t + n].double()
                t += n
                if not n:
                    continue
                lead = p % P
                rows = torch.cat([before[r:r + lead], x])
                r += lead + n
                for c in range(0, lead + n, P):
                    part = rows[c:c + P]
                    fresh = lead if c == 0 else 0
                    amax = part[fresh:].abs().amax((0, 2)).tolist()
                    for h, a in enumerate(amax):
                        e = LEAST
                        if a > 0:
                            e = math.frexp(a / MOST[held])[1]                       # a / most in [2^(e - 1), 2^e)
                            e = e - 1 if math.ldexp(MOST[held], e - 1) >= a else e
                            e = min(max(e, LEAST), TOP[held])
                        at = table[b][(p - lead + c) // P]
                        if fresh:
                            e = max(e, int(math.log2(float(scales[at, h]))))
                        scales[at, h] = math.ldexp(1.0, e)
                        part[:, h] = _exact_code(part[:, h] / math.ldexp(1.0, e), held) * math.ldexp(1.0, e)
                parts.append(rows)
            answer += [torch.cat(parts), scales]
        return answer[0], answer[2], answer[1], answer[3]
    outs, lses, t = [], [], 0
    G, H = s["group"], s["heads"]
    for b, (p, n) in enumerate(zip(past, new)):
        q = s["q"][t:t + n].double()
        t += n
        lo = max(0, p - s["window"] + 1) if s["window"] else 0
        j = torch.arange(lo, p + n, device=DEVICE)
        slots = s["table"][b][j // P].long() * P + j % P
        page, off = slots // P, slots % P
        u8 = lambda c: c.view(torch.uint8)  # noqa: E731
        value = lambda bits: bits.view(s["k_cache"].dtype).to(torch.float32).double()  # noqa: E731
        k = value(u8(s["k_cache"])[page, :, off]) * s["k_scale"].double()[page][:, :, None]
        v = value(u8(s["v_cache"])[page, :, off // 16, :, off % 16]) * s["v_scale"].double()[page][:, :, None]
        i = torch.arange(n, device=DEVICE)
        hidden = (j > p + i[:, None])
        if s["window"]:
            hidden = hidden | (j <= p + i[:, None] - s["window"])
        o, l = [], []
        for h in range(H * G):
            z = (q[:, h] @ k[:, h // G].t().contiguous() * s["scale"]).masked_fill(hidden, -math.inf)
            l.append(torch.logsumexp(z, -1))
            o.append(torch.softmax(z, -1) @ v[:, h // G].contiguous())
        outs.append(torch.stack(o, 1))
        lses.append(torch.stack(l, 1))
    return torch.cat(outs), torch.cat(lses)
