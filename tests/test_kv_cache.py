"""The paged 8-bit key / value cache (functs::kv_plan, kv_store, kv_read, kv_attention; functs_amd/kv_cache.py,
functs_amd/csrc/fxhip/fx_kv*.h).

CPU: refusals, how calls are cut into parts and what becomes of bad lengths and pages.
GPU: the operators against plain implementations in Python integers and 64 bits."""
import ctypes
import math
import os
import random
import subprocess

import pytest
import torch

import functs_amd.jit as fj  # noqa: F401
from functs_amd import _lib
from functs_amd._lib import C, FxError, lib
from functs_amd.kv_cache import KvCache

E4M3, INT8 = torch.float8_e4m3fn, torch.int8
TOP = {E4M3: 448.0, INT8: 127.0}


# ---- plain implementations ----

def plan_plain(past, new, table, free, P, most, free_start=0):
    """kv_plan, one request after the other."""
    B, M = len(past), len(table[0]) if table else 0
    table = [list(r) for r in table]
    slots, positions, starts, lens = [-1] * most, [-1] * most, [0], []
    free = free[min(max(free_start, 0), len(free)):]
    at = asked = taken = 0
    for b in range(B):
        n = max(new[b], 0)
        begin, at = at, at + n
        starts.append(min(at, most))
        had, have = -(-past[b] // P), -(-(past[b] + new[b]) // P)
        fits = past[b] >= 0 and new[b] >= 0 and past[b] + new[b] <= M * P and at <= most
        need = have - had if fits else 0
        if not fits or (need and asked + need > len(free)):
            lens.append(0)
            asked += need
            continue
        for i in range(need):
            table[b][had + i] = free[asked + i]
        asked += need
        taken += need
        lens.append(past[b] + new[b])
        for j in range(n):
            p = past[b] + j
            page = table[b][p // P]
            slots[begin + j] = page * P + p % P if page >= 0 else -1
            positions[begin + j] = p
    return slots, positions, starts, lens, [taken], table


def scale_plain(amax, held):
    if amax == 0:
        return 2.0 ** -100
    e = math.frexp(amax)[1] - 12
    while TOP[held] * 2.0 ** e < amax:
        e += 1
    return 2.0 ** min(max(e, -100), 119 if held == E4M3 else 121)


def code_plain(x, held):
    """x (64 bits, divided by the scale) to the number of the nearest code."""
    if held == INT8:
        return torch.where(torch.isnan(x), 0.0, torch.round(x).clamp(-127, 127))
    y = x.clamp(-448, 448)
    step = torch.exp2(torch.frexp(torch.where(torch.isnan(y), 0.0, y))[1].clamp(min=-5).double() - 4)
    return torch.where(torch.isnan(x), x, torch.round(y / step) * step)


class PlainCache:
    """Numbers (64 bits) instead of codes: k, v [pages, heads, page, depth] in units of their scales."""

    def __init__(self, cache):
        self.held = cache.k.dtype
        num = lambda t: t.cpu().to(torch.float32).double()  # noqa: E731
        N, H, P, D = cache.k.shape
        self.k, self.v = num(cache.k), num(cache.v).permute(0, 1, 2, 4, 3).reshape(N, H, P, D)
        self.ks, self.vs = cache.k_scale.cpu().double(), cache.v_scale.cpu().double()

    def store(self, k, v, slots):
        N, H, P, D = self.k.shape
        slots = slots.tolist()
        t = 0
        while t < len(slots):
            if not 0 <= slots[t] < N * P:
                t += 1
                continue
            page, n = slots[t] // P, 1
            while t + n < len(slots) and 0 <= slots[t + n] < N * P and slots[t + n] // P == page:
                n += 1
            first = slots[t] % P
            for x, codes, scales in ((k, self.k, self.ks), (v, self.v, self.vs)):
                rows = x[t:t + n].cpu().double()
                fine = torch.where(torch.isfinite(rows), rows, 0.0).abs()
                for h in range(H):
                    s = scale_plain(float(fine[:, h].max()), self.held)
                    old = float(scales[page, h])
                    if first > 0 and old > s:
                        s = old
                    elif first > 0 and 0 < old < s:
                        codes[page, h, :first] = code_plain(codes[page, h, :first] * (old / s), self.held)
                    scales[page, h] = s
                    for j in range(n):
                        codes[page, h, slots[t + j] % P] = code_plain(rows[j, h] / s, self.held)
            t += n

    def read(self, slots):
        N, H, P, D = self.k.shape
        ok = (slots >= 0) & (slots < N * P)
        s = torch.where(ok, slots, 0)
        at = lambda c, sc: torch.where(ok[:, None, None], c[s // P, :, s % P] * sc[s // P][:, :, None], 0.0)  # noqa: E731
        return at(self.k, self.ks), at(self.v, self.vs)

    def attention(self, q, table, lens, starts, scale, window):
        """out, lse and what their tolerances need: sum of weights times |values|, the largest sum of |products| of a row's scores."""
        N, H, P, D = self.k.shape
        T, hq = q.shape[:2]
        out, lse = torch.zeros(T, hq, D, dtype=torch.double), torch.full((T, hq), -math.inf, dtype=torch.double)
        spread, size = torch.zeros(T, hq, D, dtype=torch.double), torch.zeros(T, hq, dtype=torch.double)
        q = q.cpu().double()
        for b in range(len(lens)):
            n, L = starts[b + 1] - starts[b], lens[b]
            if n <= 0 or L <= 0:
                continue
            j = torch.arange(L)
            pages = torch.tensor(table[b])[j // P]
            ok = (pages >= 0) & (pages < N)
            pages = torch.where(ok, pages, 0)
            k = self.k[pages, :, j % P] * self.ks[pages][:, :, None]
            v = self.v[pages, :, j % P] * self.vs[pages][:, :, None]
            p = L - n + torch.arange(n)[:, None]
            sees = ok & (j <= p) & ((j > p - window) if window else True)
            k, v = torch.where(ok[:, None, None], k, 0.0), torch.where(ok[:, None, None], v, 0.0)
            heads = lambda x: x.permute(1, 0, 2).repeat_interleave(hq // H, 0)  # noqa: E731
            rows = slice(starts[b], starts[b] + n)
            qb, kb, vb = q[rows].permute(1, 0, 2).contiguous(), heads(k).transpose(1, 2).contiguous(), heads(v).contiguous()
            s = torch.where(sees, torch.bmm(qb, kb) * scale, -math.inf)
            w = torch.nan_to_num(torch.softmax(s, 2), nan=0.0)               # (rows that see nothing)
            size[rows] = torch.where(sees, torch.bmm(qb.abs(), kb.abs()) * scale, 0.0).amax(2).t()
            lse[rows] = torch.logsumexp(s, 2).t()
            out[rows], spread[rows] = torch.bmm(w, vb).permute(1, 0, 2), torch.bmm(w, vb.abs()).permute(1, 0, 2)
        return out, lse, spread, size


def filled(pages, heads, page, depth, held, seed, dev="cuda"):
    """A cache whose every page holds numbers (their scales differ), codes of all kinds among them."""
    g = torch.Generator().manual_seed(seed)
    c = KvCache.empty(pages, heads, page, depth, held, dev)
    for codes, scales in ((c.k, c.k_scale), (c.v, c.v_scale)):
        x = torch.randn(codes.shape, generator=g) * (40.0 if held == INT8 else 60.0)
        codes.copy_(x.round().clamp(-127, 127).to(INT8) if held == INT8 else x.clamp(-448, 448).to(E4M3))
        scales.copy_(torch.exp2(torch.randint(-7, -3, scales.shape, generator=g).float()))
    return c


def requests(spec, page, pages, seed, extra=0):
    """spec: (tokens in all, rows) a request.  Their tables (pages in no order, -1 behind the last), lens, starts."""
    order = list(range(pages))
    random.Random(seed).shuffle(order)
    width = max([-(-L // page) for L, _ in spec] + [1]) + extra
    table, starts = [], [0]
    for L, n in spec:
        need = -(-L // page)
        table.append(order[:need] + [-1] * (width - need))
        order = order[need:]
        starts.append(starts[-1] + n)
    return table, [L for L, _ in spec], starts


def i32(x, dev="cuda"):
    return torch.tensor(x, dtype=torch.int32, device=dev)


# ---- CPU ----

@pytest.fixture(scope="module")
def split(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("kv") / "libkv_split.so")
    src = os.path.join(os.path.dirname(os.path.abspath(__file__)), "support", "kv_split.cpp")
    subprocess.check_call(["g++", "-O2", "-std=c++17", "-fPIC", "-shared", src, "-o", so])
    return ctypes.CDLL(so)


@pytest.mark.parametrize("rows,least", [(16, 4), (128, 4), (64, 2), (256, 8), (256, 4)])
def test_every_step_is_taken_once_and_the_parts_fit_the_workspace(split, rows, least):
    rng = random.Random(rows)
    for case in range(400):
        B = rng.choice([0, 1, 1, 2, 5, 30, 300])
        most = rng.choice([1, 70, 3000, 60000])
        new = [rng.choice([0, 1, 1, rng.randint(0, 40)]) for _ in range(B)]
        if case % 7 == 0 and B:
            new[rng.randrange(B)] = 700
        lens = [rng.choice([0, n, rng.randint(0, most)]) for n in new]
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        tokens, room = starts[-1], most
        if case % 5 == 0 and B:   # what a table may hold by mistake
            lens[rng.randrange(B)] = rng.choice([-5, 2 ** 31 - 1, -2 ** 31])
            starts[rng.randrange(B + 1)] = rng.choice([-1, 2 ** 31 - 1, -2 ** 31, tokens + 3])
            room = rng.randint(0, most)
        out = (ctypes.c_longlong * 3)()
        a, l = (ctypes.c_int * (B + 1))(*starts), (ctypes.c_int * max(B, 1))(*(lens or [0]))
        group, window, heads = rng.choice([1, 2, 5, 8, 16, 71]), rng.choice([0, 0, 1, 64, 777]), rng.choice([1, 3, 8])
        assert split.fx_kv_split_check(B, a, l, tokens, room, group, window, heads, rows, least, out) == 0, (case, starts[:9], lens[:9], group, window)


def test_units_of_requests_that_overlap_stay_inside(tmp_path):
    """Offsets that fall let requests overlap: their units may be more than 31 bits count.  Whatever the sums come to then, a unit that is found is one
    of its request's and nothing is cut."""
    so = str(tmp_path / "libkv_units.so")
    subprocess.check_call(["g++", "-O2", "-std=c++17", "-fPIC", "-shared", os.path.join(os.path.dirname(os.path.abspath(__file__)), "support", "kv_units.cpp"), "-o", so])
    check, shared = ctypes.CDLL(so).fx_kv_units_check, ctypes.c_int()
    rng = random.Random(1)

    def run(starts, lens, tokens, room, group, heads):
        a, l = (ctypes.c_int * len(starts))(*starts), (ctypes.c_int * len(lens))(*lens)
        return check(len(lens), a, l, tokens, room, group, heads, 16, 4, 1 << 20, ctypes.byref(shared))

    for B, tokens, group, heads in ((2000, 1 << 20, 16, 4), (700, 1 << 22, 4, 16), (100, 5000, 8, 8)):
        for falls in (True, False):
            starts = [rng.randint(0, tokens) for _ in range(B + 1)]
            starts[1], starts[2] = 0, tokens
            lens = [rng.choice([0, 0, 1]) for _ in range(B)]
            lens[B // 2], starts[B // 2 + 1] = 1 << 20, starts[B // 2] + 1      # one row and many tokens
            assert run(starts if falls else sorted(starts), lens, tokens, 1 << 20, group, heads) == 0
            assert not falls or shared.value == 0


def test_entries_of_a_table_that_are_no_page(split):
    for entry, page in ((0, 0), (6, 6), (7, -1), (-1, -1), (2 ** 31 - 1, -1), (-2 ** 31, -1)):
        assert split.fx_kv_page_of(entry, 7) == page


def test_sizes_of_a_cache_are_refused():
    for bad in (dict(page_size=48), dict(page_size=8), dict(page_size=512), dict(depth=24), dict(depth=0), dict(depth=272), dict(pages=0), dict(heads=0),
                dict(dtype=torch.float16), dict(dtype=torch.float8_e5m2)):
        with pytest.raises(FxError):
            KvCache.empty(**{**dict(pages=2, heads=2, page_size=16, depth=64, device="cpu"), **bad})


def test_tensors_on_the_host_are_refused():
    c = KvCache.empty(2, 2, 16, 64, device="cpu")
    q, slots = torch.zeros(3, 4, 64), torch.zeros(3, dtype=torch.long)
    for call in (lambda: c.store(q[:, :2], q[:, :2], slots), lambda: c.read(slots), lambda: c.attention(q, i32([[0]], "cpu"), i32([1], "cpu"), i32([0, 3], "cpu")),
                 lambda: c.plan(i32([0], "cpu"), i32([1], "cpu"), i32([[0]], "cpu"), i32([0], "cpu"), 1)):
        with pytest.raises(RuntimeError, match="runs on the GPU only"):
            call()


def refuse_empty_caches(dev):
    c = KvCache.empty(2, 2, 16, 64, device=dev)
    q, slots = torch.zeros(3, 4, 64, device=dev), torch.zeros(3, dtype=torch.long, device=dev)
    for part in ((slice(None), slice(0, 0)), (slice(0, 0),), (slice(0, 0), slice(0, 0))):
        x = KvCache(c.k[part], c.v[part], c.k_scale[part], c.v_scale[part])
        k = q[:, :x.k.size(1)]
        for call in (lambda: x.attention(q, i32([[0]], dev), i32([1], dev), i32([0, 3], dev)), lambda: x.attention(q[:0], i32([[0]], dev), i32([1], dev), i32([0, 0], dev)),
                     lambda: x.store(k, k, slots), lambda: x.read(slots)):
            with pytest.raises(RuntimeError, match="at least one page and one head"):
                call()


def test_caches_of_no_heads_or_pages_are_refused():
    refuse_empty_caches("cpu")


@pytest.mark.gpu
def test_caches_of_no_heads_or_pages_are_refused_on_the_gpu():
    refuse_empty_caches("cuda")


class Cache(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("k", "v", "k_scale", "v_scale")] + [(n, ctypes.c_int64) for n in ("ks", "vs", "kss", "vss")] + \
               [(n, ctypes.c_int32) for n in ("pages", "heads", "page_size", "depth", "held", "reserved")]


class Rows(ctypes.Structure):
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p)] + [(n, ctypes.c_int64) for n in ("kt", "kh", "vt", "vh")] + \
               [("slots", ctypes.c_void_p), ("tokens", ctypes.c_int32), ("dtype", ctypes.c_int32)]


class Plan(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("past", "added", "free_pages", "free_start", "table")] + [("table_stride", ctypes.c_int64)] + \
               [(n, ctypes.c_void_p) for n in ("slots", "positions", "starts", "lens", "taken")] + \
               [(n, ctypes.c_int32) for n in ("requests", "columns", "n_free", "page_size", "tokens", "reserved")]


class Attention(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("q", "out", "lse")] + [(n, ctypes.c_int64) for n in ("qt", "qh")] + [("table", ctypes.c_void_p), ("table_stride", ctypes.c_int64)] + \
               [(n, ctypes.c_void_p) for n in ("lens", "starts")] + \
               [(n, ctypes.c_int32) for n in ("tokens", "requests", "columns", "q_heads", "dtype", "window", "max_new", "clear_rest")] + \
               [("scale", ctypes.c_float), ("reserved", ctypes.c_int32), ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_size_t)]


def test_the_c_abi_refuses_before_it_launches():
    """Descriptors that no kernel may see (addresses here are never read: each call returns from its checks)."""
    at = 4096
    ok = dict(k=at, v=at, k_scale=at, v_scale=at, ks=2 * 16 * 64, vs=2 * 16 * 64, kss=2, vss=2, pages=2, heads=2, page_size=16, depth=64, held=0)
    rows = dict(k=at, v=at, kt=128, kh=64, vt=128, vh=64, slots=at, tokens=3, dtype=C["FX_DT_BF16"])
    for change, code in ((dict(held=2), "FX_E_UNSUPPORTED"), (dict(page_size=17), "FX_E_UNSUPPORTED"), (dict(depth=40), "FX_E_UNSUPPORTED"), (dict(pages=0), "FX_E_INVALID"),
                         (dict(k=None), "FX_E_INVALID"), (dict(k=at + 8), "FX_E_INVALID"), (dict(ks=2 * 16 * 64 - 16), "FX_E_INVALID"), (dict(kss=1), "FX_E_INVALID"),
                         (dict(heads=70000), "FX_E_LIMIT")):
        c = Cache(**{**ok, **change})
        for call in (lib.fx_kv_store, lib.fx_kv_read):
            assert call(ctypes.byref(c), ctypes.byref(Rows(**rows)), None) == C[code], change
            assert b"fx_kv_" in lib.fx_last_error()
    for change, code in ((dict(dtype=C["FX_DT_I64"]), "FX_E_UNSUPPORTED"), (dict(tokens=-1), "FX_E_INVALID"), (dict(slots=None), "FX_E_INVALID"), (dict(tokens=1 << 30), "FX_E_LIMIT")):
        assert lib.fx_kv_store(ctypes.byref(Cache(**ok)), ctypes.byref(Rows(**{**rows, **change})), None) == C[code], change
    plan = dict(past=at, added=at, free_pages=at, table=at, table_stride=4, slots=at, positions=at, starts=at, lens=at, taken=at, requests=2, columns=4, n_free=3, page_size=16, tokens=5)
    for change, code in ((dict(page_size=20), "FX_E_UNSUPPORTED"), (dict(requests=-1), "FX_E_INVALID"), (dict(taken=None), "FX_E_INVALID"), (dict(table_stride=3), "FX_E_INVALID"),
                         (dict(tokens=1 << 30), "FX_E_LIMIT"), (dict(columns=1 << 27, table_stride=1 << 27), "FX_E_LIMIT")):
        assert lib.fx_kv_plan(ctypes.byref(Plan(**{**plan, **change})), None) == C[code], change
    att = dict(q=at, out=at, lse=at, qt=256, qh=64, table=at, table_stride=4, lens=at, starts=at, tokens=3, requests=2, columns=4, q_heads=4, dtype=C["FX_DT_BF16"], scale=1.0,
               workspace=at, workspace_bytes=1 << 40)
    for change, code in ((dict(dtype=7), "FX_E_UNSUPPORTED"), (dict(q_heads=3), "FX_E_INVALID"), (dict(scale=0.0), "FX_E_INVALID"), (dict(scale=math.inf), "FX_E_INVALID"),
                         (dict(scale=math.nan), "FX_E_INVALID"), (dict(window=-1), "FX_E_INVALID"), (dict(lse=None), "FX_E_INVALID"), (dict(out=at + 4), "FX_E_INVALID"),
                         (dict(workspace=None), "FX_E_INVALID"), (dict(workspace_bytes=100), "FX_E_INVALID"), (dict(workspace=at + 16), "FX_E_INVALID"),
                         (dict(columns=1 << 27), "FX_E_LIMIT"), (dict(tokens=1 << 29), "FX_E_LIMIT")):
        assert lib.fx_kv_attention(ctypes.byref(Cache(**ok)), ctypes.byref(Attention(**{**att, **change})), None) == C[code], change
    for call in (lib.fx_kv_store, lib.fx_kv_read):
        assert call(None, ctypes.byref(Rows(**rows)), None) == C["FX_E_INVALID"]
        assert call(ctypes.byref(Cache(**ok)), ctypes.byref(Rows(**{**rows, "tokens": 0})), None) == 0   # nothing to do
    assert lib.fx_kv_attention(ctypes.byref(Cache(**ok)), ctypes.byref(Attention(**{**att, "tokens": 0})), None) == 0


@pytest.mark.parametrize("heads,tokens", [(2, 1 << 28), (64, 63 << 17), (65536, 63 << 7), (1, 63 << 23)])
def test_more_rows_than_a_launch_holds_are_refused(heads, tokens):
    """A launch has fewer than 2^32 threads: 512 for the 63 tokens of a workgroup and each head (addresses here are never read)."""
    at = 4096
    c = Cache(k=at, v=at, k_scale=at, v_scale=at, ks=heads * 256, vs=heads * 256, kss=heads, vss=heads, pages=2, heads=heads, page_size=16, depth=16, held=0)
    rows = Rows(k=at, v=at, kt=heads * 16, kh=16, vt=heads * 16, vh=16, slots=at, tokens=tokens, dtype=C["FX_DT_BF16"])
    assert -(-tokens // 63) * heads * 512 >= 2 ** 32
    for call in (lib.fx_kv_store, lib.fx_kv_read):
        assert call(ctypes.byref(c), ctypes.byref(rows), None) == C["FX_E_LIMIT"]


def test_mutated_arguments_are_in_the_schemas():
    for name, written in (("kv_plan", {"block_table"}), ("kv_store", {"k_cache", "v_cache", "k_scale", "v_scale"}), ("kv_read", set()), ("kv_attention", set())):
        schema = getattr(torch.ops.functs, name).default._schema
        assert {a.name for a in schema.arguments if a.alias_info is not None and a.alias_info.is_write} == written


# ---- GPU: plan ----

def check_plan(past, new, table, free, P, most, free_start=None, stride=0):
    M = len(table[0]) if table else 0
    dev_table = torch.full((len(table), M + stride), -7, dtype=torch.int32, device="cuda")
    dev_table[:, :M] = i32(table) if table else 0
    view = dev_table[:, :M]
    c = KvCache.empty(1, 1, P, 16)
    got = c.plan(i32(past), i32(new), view, i32(free), most, None if free_start is None else i32([free_start]))
    want = plan_plain(past, new, table, free, P, most, free_start or 0)
    for name, g, w in zip(("slots", "positions", "starts", "lens", "taken", "table"), got + (view,), want):
        assert g.tolist() == w, name
    assert bool((dev_table[:, M:] == -7).all())


@pytest.mark.gpu
@pytest.mark.parametrize("requests_,most_past,most_new,P", [(1, 0, 1, 16), (1, 1000, 1, 64), (5, 70, 40, 16), (257, 300, 9, 32), (1025, 90, 3, 256), (2300, 40, 2, 16), (3, 5000, 3000, 128)])
def test_plan(requests_, most_past, most_new, P):
    rng = random.Random(requests_)
    past = [rng.randint(0, most_past) for _ in range(requests_)]
    new = [rng.randint(0, most_new) for _ in range(requests_)]
    M = max(-(-(p + n) // P) for p, n in zip(past, new)) + 2
    ids = iter(range(10 ** 7))
    table = [[next(ids) if c < -(-p // P) else -1 for c in range(M)] for p in past]
    need = sum(-(-(p + n) // P) - -(-p // P) for p, n in zip(past, new))
    free = [10 ** 6 + i for i in range(need + 5)]
    rng.shuffle(free)
    check_plan(past, new, table, free, P, sum(new))
    check_plan(past, new, table, free, P, sum(new) + 1500, stride=3)                   # rows behind the last token
    check_plan(past, new, table, free[:need // 2], P, sum(new))                        # too few pages
    check_plan(past, new, table, free, P, sum(new) // 2)                               # too few rows
    check_plan(past, new, table, free, P, sum(new), free_start=need // 3 + 1)          # some are given already


@pytest.mark.gpu
def test_plan_of_lengths_that_do_not_fit():
    check_plan([], [], [], [], 16, 0)
    check_plan([], [], [], [3], 16, 5)
    check_plan([0, -1, 16, 40, 2, 5], [0, 3, 17, 3, -4, 1], [[-1, -1], [1, -1], [2, -1], [3, 4], [5, -1], [6, -1]], [9, 8, 7], 16, 40)
    check_plan([2 ** 31 - 1, 5, 3], [2 ** 31 - 1, 1, 2 ** 31 - 1], [[0, -1], [1, -1], [2, -1]], [9], 16, 10)
    check_plan([15, 15], [1, 2], [[4], [5]], [], 16, 3)                                # no free pages, one needs none
    check_plan([15, 15], [2, 1], [[4, -1], [5, -1]], [7], 16, 3, free_start=-3)
    check_plan([15, 15], [2, 1], [[4, -1], [5, -1]], [7], 16, 3, free_start=100)


# ---- GPU: store and read ----

def rows_of(kind, tokens, heads, depth, seed, strided=False):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(tokens, 2, heads, depth + (8 if strided else 0), generator=g) * torch.exp(2 * torch.randn(tokens, 1, heads, 1, generator=g))
    x = x.to(kind).cuda()[..., :depth]
    return x[:, 0], x[:, 1]


def assert_cache(cache, plain):
    again = PlainCache(cache)
    for name in ("ks", "vs", "k", "v"):
        g, w = getattr(again, name), getattr(plain, name)
        assert torch.equal(torch.nan_to_num(g, nan=1e9), torch.nan_to_num(w, nan=1e9)), name


@pytest.mark.gpu
@pytest.mark.parametrize("held", [E4M3, INT8])
@pytest.mark.parametrize("kind", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("P,H,D", [(16, 3, 64), (64, 2, 128), (256, 1, 16), (32, 2, 80), (128, 1, 256)])
def test_store_and_read(held, kind, P, H, D):
    """Prompts and single tokens behind them, step by step: codes and scales are exactly those of the definition, and everything that is
    not written stays (equal bits: the codes of both sides as numbers)."""
    cache = filled(9, H, P, D, held, 5)
    cache.k_scale[7] = math.nan                        # a page that nobody has used yet
    plain = PlainCache(cache)
    order = [4, 7, 1, 2, 0, 8]
    first, second = 2 * P + P // 2 + 3, P + 1          # tokens of two requests
    at = lambda pages, lo, hi: [pages[p // P] * P + p % P for p in range(lo, hi)]  # noqa: E731
    steps = [at(order[:4], 0, first) + at(order[4:], 0, second)]
    steps += [at(order[:4], first + i, first + i + 1) + at(order[4:], second + i, second + i + 1) for i in range(3)]
    steps += [at(order[:4], first + 3, first + 8) + [-1, 9 * P, 2 ** 40] + at(order[4:], second + 3, second + 4)]
    for i, s in enumerate(steps):
        slots = torch.tensor(s, dtype=torch.long)
        k, v = rows_of(kind, len(s), H, D, 7 * i + 1, strided=i % 2 == 1)
        cache.store(k, v, slots.cuda())
        plain.store(k, v, slots)
        assert_cache(cache, plain)
    everything = torch.tensor(at(order[:4], 0, first + 8) + [-1, 5, 9 * P] + list(range(17, 40)) + at(order[4:], 0, second + 4) + [3, 3, 2, 2 ** 45, 0])
    k, v = cache.read(everything.cuda(), kind)
    wk, wv = plain.read(everything)
    finite = [torch.where(torch.isnan(x), 0.0, x) for x in (k.cpu().double(), v.cpu().double(), wk.to(kind).double(), wv.to(kind).double())]
    assert k.dtype == kind and torch.equal(finite[0], finite[2]) and torch.equal(finite[1], finite[3])


@pytest.mark.gpu
@pytest.mark.parametrize("held", [E4M3, INT8])
def test_store_of_strange_numbers(held):
    """Infinities, NaN, zeros, the largest and the smallest: for the first row of a page and behind others."""
    H, P, D = 2, 16, 32
    cache = filled(4, H, P, D, held, 6)
    plain = PlainCache(cache)
    g = torch.Generator().manual_seed(3)
    specials = torch.tensor([0.0, -0.0, math.inf, -math.inf, math.nan, 3.4028234e38, -3.4028234e38, 1e-45, 1.2e-38, 448.0, 449.0, 464.0, 465.0, 127.0, 127.5, 1.0])
    for i, slots in enumerate(([0, 1, 2], [3, 4], [16, 17], [18], [32], [33], [34, 35], [48, 49, 50, 51])):
        x = torch.randn(len(slots), 2, H, D, generator=g)
        if i in (0, 3, 6):
            x.view(-1)[:: 3] = specials[torch.randint(0, 16, (len(x.view(-1)[::3]),), generator=g)]
        if i in (2, 4):
            x.zero_()
        if i == 5:
            x *= 1e-37
        if i == 7:
            x = torch.full_like(x, math.inf)
        k, v = x[:, 0].cuda(), x[:, 1].cuda()
        cache.store(k, v, torch.tensor(slots).cuda())
        plain.store(k, v, torch.tensor(slots))
        assert_cache(cache, plain)


@pytest.mark.gpu
def test_store_of_slots_in_no_order():
    """Neighbours of one page in any order, one slot twice (the later row stays), a page rolled back and written again."""
    cache = filled(3, 2, 32, 64, E4M3, 8)
    plain = PlainCache(cache)
    for i, slots in enumerate(([5, 3, 9, 9, 4], [40, 41, 45, 70, 64, 65], [33, 34], [6, 7, 7])):
        k, v = rows_of(torch.float32, len(slots), 2, 64, i)
        cache.store(k, v, torch.tensor(slots).cuda())
        plain.store(k, v, torch.tensor(slots))
        assert_cache(cache, plain)
    cache.store(k[:0], v[:0], torch.empty(0, dtype=torch.long, device="cuda"))
    assert_cache(cache, plain)
    assert [t.shape[0] for t in cache.read(torch.empty(0, dtype=torch.long, device="cuda"))] == [0, 0]


@pytest.mark.gpu
@pytest.mark.parametrize("held", [E4M3, INT8])
@pytest.mark.parametrize("kind", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("P,H,D", [(64, 1, 128), (256, 1, 64), (128, 2, 16), (256, 1, 256), (32, 2, 144), (128, 1, 80)])
def test_store_of_long_runs(held, kind, P, H, D):
    """Runs that several waves share: from the middle of a page on, with larger numbers than before (its codes are rounded again) and smaller ones,
    with infinities and NaN in one wave's part, ends inside a group of 16, a run in reverse, rows that are not aligned."""
    cache = filled(6, H, P, D, held, 7)
    plain = PlainCache(cache)
    at = lambda page, lo, hi: list(range(page * P + lo, page * P + hi))  # noqa: E731
    steps = [(at(0, 0, 5) + at(1, 0, P) + at(2, 0, P // 2 + 3), 0.01, False), (at(0, 5, P) + at(2, P // 2 + 3, P - 1) + at(3, 0, 18), 3.0, False),
             (at(3, 18, P - 5 if P > 32 else P) + at(4, 0, 17), 0.1, True), (at(4, 17, P) + at(5, 0, P - 1)[::-1], 9.0, True)]
    for i, (slots, size, strange) in enumerate(steps):
        k, v = rows_of(kind, len(slots), H, D, 5 * i + 2, strided=i == 1)
        k, v = k * size, v * size
        if strange:
            for x, t in ((k, 1), (v, len(slots) - 2)):
                x[t, 0, 3], x[t, 0, 4], x[t // 2, 0, 5] = math.inf, math.nan, -math.inf
        cache.store(k, v, torch.tensor(slots).cuda())
        plain.store(k, v, torch.tensor(slots))
        assert_cache(cache, plain)
    every = torch.arange(6 * P)
    k, v = cache.read(every.cuda(), torch.float32)
    for got, want in zip((k, v), plain.read(every)):
        assert torch.equal(torch.nan_to_num(got.cpu().double(), nan=1e9), torch.nan_to_num(want, nan=1e9))


# ---- GPU: attention ----

def tolerance(kind, ref, lse, spread, size, tokens, depth, many=False):
    """Bounds of |out - ref| and |lse - ref lse| (64 bits), from the arithmetic:
    result rounding           half a step of its type, relative to the value
    a score                   sums of `depth` products in fp32, and two roundings more: (depth + 4) 2^-24 of the sum of |products|
    a weight                  the score's error (the weight and the sum it is divided by: twice), the exponential (2^-22), the number it is cut to
                              (2^-16 in two bf16, 2^-23 in three, and their products' roundings in the matrix cores; `many` rows of a bf16
                              call: one bf16, off by at most half a step, 2^-8)
    the sums over tokens      one addition for each 32 tokens and 4 for joining them: (tokens / 32 + 40) 2^-24
    All but the first are relative to the sum of weights times |values|."""
    e = 2.0 ** -24
    score = (depth + 4) * e * size
    weight = 2 * score + 2.0 ** -22 + (2.0 ** -22 if kind == torch.float32 else 2.0 ** -8 if many and kind == torch.bfloat16 else 2.0 ** -15) + (tokens / 32 + 40) * e
    step = torch.finfo(kind).eps / 2
    tiny = torch.finfo(kind).smallest_normal * torch.finfo(kind).eps
    out = step * ref.abs() + weight[:, :, None] * spread * (1 + step) + tiny
    return out, score + (tokens / 32 + 40) * e + 2.0 ** -22 + 2.0 ** -23 * lse.abs()


def check_attention(spec, held, kind, P, H, G, D, window=0, max_new=0, seed=1, cache=None, table=None, scale=None, strided=False, pad=0):
    pages = sum(-(-L // P) for L, _ in spec) + 2
    cache = cache or filled(pages, H, P, D, held, seed)
    t, lens, starts = requests(spec, P, pages, seed, extra=seed % 3)
    table = table or t
    g = torch.Generator().manual_seed(seed + 1)
    T = starts[-1] + pad
    q = torch.randn(T, H * G + 1, D + (3 if strided else 0), generator=g).to(kind)[:, :H * G, :D]
    scale = scale or D ** -0.5
    out, lse = cache.attention(q.cuda() if not strided else q.as_strided(q.shape, q.stride()).cuda(), i32(table), i32(lens), i32(starts), scale, window, max_new)
    ref, rl, spread, size = PlainCache(cache).attention(q, table, lens, starts, scale, window)
    o, l = out.cpu().double(), lse.cpu().double()
    assert out.dtype == kind and lse.dtype == torch.float32 and bool(torch.isfinite(o).all())
    assert torch.equal(torch.isinf(l), torch.isinf(rl)) and bool((l[torch.isinf(rl)] < 0).all())
    assert bool((o[torch.isinf(rl)] == 0).all())
    fine = torch.isfinite(rl)
    most, lmost = tolerance(kind, ref, torch.where(fine, rl, 0.0), spread, size, max(lens + [1]), D, T * H * G >= 49152 and any(n * G > 128 for _, n in spec))
    worst = ((o - ref).abs() / most).max() if o.numel() else 0
    assert float(worst) <= 1, "out %.3g times its bound" % worst
    lw = ((l - rl).abs()[fine] / lmost[fine]).max() if bool(fine.any()) else 0
    assert float(lw) <= 1, "lse %.3g times its bound" % lw
    return out, lse


KINDS = [torch.float32, torch.float16, torch.bfloat16]


@pytest.mark.gpu
@pytest.mark.parametrize("held", [E4M3, INT8])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("P,H,G,D", [(16, 12, 1, 64), (64, 2, 4, 128), (128, 1, 8, 256), (32, 2, 5, 80), (256, 1, 3, 16), (16, 1, 16, 192), (64, 3, 2, 32)])
def test_single_tokens(held, kind, P, H, G, D):
    check_attention([(1, 1), (50, 1), (63, 1), (64, 1), (65, 1), (257, 1), (0, 1), (700, 1), (16, 0)], held, kind, P, H, G, D, max_new=1)


@pytest.mark.gpu
@pytest.mark.parametrize("held", [E4M3, INT8])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("window", [0, 1, 37, 200])
def test_a_few_rows_and_windows(held, kind, D, window):
    check_attention([(9, 4), (3, 3), (2, 5), (200, 7), (321, 2), (0, 2), (130, 1)], held, kind, 32, 2, 3, D, window=window, max_new=7, seed=window + D)


@pytest.mark.gpu
@pytest.mark.parametrize("held", [E4M3, INT8])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("G,D,window", [(1, 64, 0), (4, 128, 0), (5, 80, 100), (2, 256, 0), (3, 128, 17)])
def test_prompts(held, kind, G, D, window):
    check_attention([(150, 150), (400, 133), (65, 1), (10, 30), (257, 129), (64, 64)], held, kind, 64, 2, G, D, window=window, seed=G)


@pytest.mark.gpu
@pytest.mark.parametrize("held", [E4M3, INT8])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("P,G,D,window", [(16, 1, 64, 0), (32, 2, 128, 70), (128, 1, 48, 0), (256, 3, 80, 300), (16, 1, 256, 40), (128, 2, 192, 0), (256, 1, 128, 0)])
def test_prompts_on_pages_of_all_sizes(held, kind, P, G, D, window):
    """Requests of more rows than a tile beside short ones, on pages smaller and larger than a step of 64 tokens."""
    check_attention([(300, 140), (320, 270), (200, 1), (131, 129), (77, 60)], held, kind, P, 2, G, D, window=window, seed=P + D)
    check_attention([(700, 260)], held, kind, P, 1, G, D, window=window, seed=P + D + 1, strided=True)


@pytest.mark.gpu
@pytest.mark.parametrize("held", [E4M3, INT8])
@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("P,H,G,D,window", [(16, 90, 1, 64, 0), (32, 2, 45, 128, 70), (64, 3, 30, 128, 0), (128, 90, 1, 48, 33), (256, 9, 10, 80, 300), (16, 30, 3, 256, 40),
                                            (64, 2, 47, 192, 0), (256, 90, 1, 128, 0), (64, 10, 9, 64, 1)])
def test_many_rows(held, kind, P, H, G, D, window):
    """Calls of so many rows that the long requests get large tiles: beside short ones and one that has nothing, with rows of no request."""
    spec = [(300, 140), (320, 270), (200, 1), (0, 0), (131, 129), (77, 60), (5, 9)]
    check_attention(spec, held, kind, P, H, G, D, window=window, seed=P + D, pad=3)
    check_attention([(700, 600)], held, kind, P, H, G, D, window=window, seed=P + D + 1, strided=True, max_new=600)


@pytest.mark.gpu
@pytest.mark.parametrize("held,kind", [(E4M3, torch.bfloat16), (INT8, torch.float16)])
@pytest.mark.parametrize("P,H,G,D,window", [(16, 2, 45, 128, 0), (64, 1, 90, 64, 100), (256, 3, 30, 256, 7)])
def test_many_rows_that_come_before_their_tokens(held, kind, P, H, G, D, window):
    """Requests of more rows than tokens, in large tiles: the first rows see nothing, whole tiles of them too."""
    check_attention([(100, 300), (200, 201), (1, 150)], held, kind, P, H, G, D, window=window, seed=P)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [64, 65, 300])
def test_many_requests_some_of_many_rows(n):
    """Both kernels and their parts in one call, for more requests than a wave has lanes; the same bits in every call."""
    rng = random.Random(n)
    spec = [(L, min(L, rng.choice([0, 1, 1, 2, 7]))) for L in (rng.choice([0, 1, 17, 90, 200]) for _ in range(n))]
    spec[n // 3], spec[n // 2], spec[n - 1], spec[5] = (1500, 300), (2600, 1), (900, 250), (400, 150)
    first = check_attention(spec, INT8, torch.bfloat16, 32, 4, 16, 64, seed=n)
    for _ in range(3):
        again = check_attention(spec, INT8, torch.bfloat16, 32, 4, 16, 64, seed=n)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.gpu
@pytest.mark.parametrize("kind,H", [(torch.float32, 1), (torch.bfloat16, 42)])
@pytest.mark.parametrize("n", [3, 70])
def test_offsets_that_fall(kind, H, n):
    """Requests that overlap by mistake: rows that are one request's alone have its results.  Rows behind the last offset are of no request, whatever the
    offsets before it say, and may be cleared: 590 here."""
    spec = [(900, 600), (700, 1), (300, 3)]
    cache = filled(40, H, 64, 64, INT8, 5)
    table, lens, starts = requests(spec, 64, 40, 1)
    q = torch.randn(starts[-1], H * 2, 64, generator=torch.Generator().manual_seed(1)).to(kind).cuda()
    table, lens = table + [[-1] * len(table[0])] * (n - 3), lens + [0] * (n - 3)
    args = (q, i32(table), i32(lens))
    rising = cache.attention(*args, i32(starts + [starts[-1]] * (n - 3)))
    falling = cache.attention(*args, i32(starts[:3] + [590] + [590] * (n - 3)))         # the third request's end is in the first: it has no rows
    ref, rl, spread, size = PlainCache(cache).attention(q, table, lens, starts + [starts[-1]] * (n - 3), 0.125, 0)
    most, lmost = tolerance(kind, ref, rl, spread, size, 900, 64, True)
    for (out, lse), rows in ((rising, starts[-1]), (falling, 590)):
        assert bool(((out.cpu().double() - ref).abs() <= most)[:rows].all()) and bool(((lse.cpu().double() - rl).abs() <= lmost)[:rows].all())
    wild = cache.attention(*args, i32([0, starts[1], 0, starts[1]] + [0] * (n - 3)))
    assert bool(torch.isfinite(wild[0][:starts[1]].float()).all())


@pytest.mark.gpu
@pytest.mark.parametrize("kind,heads,requests_,columns,launches", [(torch.float32, 2, 64, 5, 2), (torch.float32, 2, 65, 5, 3), (torch.float32, 2, 65, 4, 2),
                                                                   (torch.bfloat16, 90, 64, 5, 3), (torch.bfloat16, 90, 65, 5, 5), (torch.bfloat16, 90, 1, 5, 2)])
def test_every_launch_is_counted(kind, heads, requests_, columns, launches):
    """fx_kv_rows, fx_kv_tiles beside it (16-bit calls of 49 152 rows and more of several requests), fx_kv_offsets ahead of either for more
    than 64 requests, fx_kv_join where a table holds more than 256 tokens."""
    c = filled(2, 2, 64, 64, E4M3, 1)
    starts = [0] + [600] * requests_
    q, table = torch.zeros(600, heads, 64, dtype=kind, device="cuda"), torch.zeros(requests_, columns, dtype=torch.int32, device="cuda")
    counts = [ctypes.c_uint64(), ctypes.c_uint64()]
    lib.fx_launch_stats(ctypes.byref(counts[0]), None)
    c.attention(q, table, i32([columns * 64] * requests_), i32(starts))
    lib.fx_launch_stats(ctypes.byref(counts[1]), None)
    assert counts[1].value - counts[0].value == launches


@pytest.mark.gpu
@pytest.mark.parametrize("max_new", [0, 1, 3, 500])
def test_max_new_is_a_matter_of_speed(max_new):
    """Whatever it says, every row has its result."""
    check_attention([(300, 1), (290, 90), (40, 3)], E4M3, torch.float32, 16, 2, 2, 64, max_new=max_new)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
def test_long_caches_are_shared_by_workgroups(kind):
    check_attention([(6000, 1), (64, 1), (3001, 2), (1, 1)], E4M3, kind, 128, 2, 4, 64, seed=9)
    check_attention([(9000, 1)], INT8, kind, 16, 1, 1, 128, seed=10)
    check_attention([(5000, 40), (33, 2), (3000, 90)], E4M3, kind, 64, 1, 3, 64, seed=11)
    check_attention([(4100, 131)], INT8, kind, 32, 2, 1, 128, seed=12, window=2500)
    check_attention([(5000, 1), (64, 1), (3001, 2), (0, 1)], E4M3, kind, 128, 4, 4, 128, seed=13)
    check_attention([(4000, 3)], INT8, kind, 64, 5, 7, 80, seed=14, window=3300)
    check_attention([(1500, 1), (900, 1)], E4M3, kind, 64, 8, 1, 256, seed=15)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [64, 65, 200, 256, 257, 1000])
def test_many_requests(n):
    """More than a lane, a wave and a workgroup has: none, short and long ones among them, of one row, of a few and of many."""
    rng = random.Random(n)
    spec = [(L, min(L, rng.choice([0, 1, 1, 1, 2]))) for L in (rng.choice([0, 1, 17, 40, 90]) for _ in range(n))]
    spec[n // 2], spec[n - 1], spec[3] = (4000, 1), (2500, 60), (700, 30)
    check_attention(spec, E4M3, torch.float32, 16, 1, 2, 64, seed=n)


@pytest.mark.gpu
def test_pages_outside_the_cache_are_not_seen():
    """-1, the first number behind the cache and garbage in a table: their tokens are left out, wherever they lie."""
    spec, P = [(300, 2), (128, 1), (90, 40), (64, 1)], 64
    pages = sum(-(-L // P) for L, _ in spec) + 2
    for seed in range(4):
        table, _, _ = requests(spec, P, pages, 1, extra=1)
        rng = random.Random(seed)
        for row in table:
            for c in range(len(row)):
                if rng.random() < 0.4:
                    row[c] = rng.choice([-1, pages, pages + 1000000, -2 ** 31, 2 ** 31 - 1])
        table[3] = [-1] * len(table[3])
        check_attention(spec, E4M3, torch.float32, P, 2, 2, 64, table=table, window=seed % 2 * 70)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 6, 70])
@pytest.mark.parametrize("window", [0, 20])
def test_what_a_row_does_not_see_has_no_influence(n, window):
    """NaN codes and NaN scales behind the last token, before the window and in pages of others: nothing of it arrives.  NaN among
    the tokens of a row's own request arrives at the rows that see it, and at no others."""
    P, H, G, D, L = 32, 2, 2, 64, 130
    cache = filled(8, H, P, D, E4M3, 3)
    table, lens, starts = [[3, 1, 6, 0, 5]], [L], [0, n]
    q = torch.randn(n, H * G, D, generator=torch.Generator().manual_seed(n)).cuda()
    args = (q, i32(table), i32(lens), i32(starts), 0.125, window)
    out, lse = cache.attention(*args)
    nan = torch.full((1,), 0x7F, dtype=torch.uint8, device="cuda")
    k8, v8 = cache.k.view(torch.uint8), cache.v.view(torch.uint8)
    k8[5, :, L % P:], cache.k_scale[[2, 4, 7]], cache.v_scale[[2, 4, 7]] = nan, math.nan, math.inf
    for t in range(L % P, P):
        v8[5, :, t // 16, :, t % 16] = nan
    lowest = L - n + 1 - window if window else 0       # the first token that any row sees
    for t in range(max(lowest, 0)):
        k8[table[0][t // P], :, t % P] = nan
        v8[table[0][t // P], :, t % P // 16, :, t % 16] = 0xFF
    again, lse2 = cache.attention(*args)
    assert torch.equal(out, again) and torch.equal(lse, lse2)
    if n == 1:
        return
    # the token before the last: its value in column 9 of head 1 is NaN; the row of the token before it does not see it
    t = L - 2
    v8[table[0][t // P], 1, t % P // 16, 9, t % 16] = nan
    got, _ = cache.attention(*args)
    want = out.clone()
    want[n - 2:, G:, 9] = math.nan
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))
    k8[table[0][t // P], 0, t % P] = nan               # a key: its scores, so whole rows
    got, l = cache.attention(*args)
    assert bool(torch.isnan(got[n - 2:, :G]).all()) and bool(torch.isnan(l[n - 2:, :G]).all())
    assert torch.equal(got[:n - 2], out[:n - 2]) and torch.equal(l[:n - 2], lse[:n - 2])


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("P", [16, 64, 256])
@pytest.mark.parametrize("n,G", [(6, 2), (150, 2), (150, 330)])
def test_nan_that_is_not_seen_and_nan_that_is(kind, P, n, G):
    """The same on pages of all kinds: codes behind the last token and before the window are NaN, then one value that some rows see."""
    H, D, L, window = 1, 128, 330, 100
    pages = -(-L // P)
    cache = filled(pages + 1, H, P, D, E4M3, 4)
    order = torch.randperm(pages + 1, generator=torch.Generator().manual_seed(P))[:pages].tolist()
    q = torch.randn(n, H * G, D, generator=torch.Generator().manual_seed(n)).to(kind).cuda()
    args = (q, i32([order + [-1]]), i32([L]), i32([0, n]), 0.125, window)
    out, lse = cache.attention(*args)
    k8, v8 = cache.k.view(torch.uint8), cache.v.view(torch.uint8)

    def spoil(t, columns=slice(None)):
        v8[order[t // P], :, t % P // 16, columns, t % 16] = 0x7F

    for t in list(range(max(L - n + 1 - window, 0))) + list(range(L, pages * P)):
        k8[order[t // P], :, t % P] = 0xFF
        spoil(t)
    again, lse2 = cache.attention(*args)
    assert torch.equal(out, again) and torch.equal(lse, lse2)
    spoil(L - 3, 77)                                   # seen by the last three rows
    got, lse2 = cache.attention(*args)
    assert bool(torch.isnan(got[n - 3:, :, 77]).all()) and int(torch.isnan(got).sum()) == 3 * G and torch.equal(lse, lse2)
    assert torch.equal(torch.where(torch.isnan(got), 0.0, got), torch.where(torch.isnan(got), 0.0, out))


@pytest.mark.gpu
@pytest.mark.parametrize("held", [E4M3, INT8])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("P", [16, 32, 64])
@pytest.mark.parametrize("n,G", [(1, 2), (6, 2), (150, 2), (150, 330)])
def test_scales_that_are_not_seen(held, kind, P, n, G):
    """Scales of every kind on pages that the table names and no row sees (before the window, in its first step of 64 tokens too, and
    behind the last token), then an infinite scale of values that the last rows see and the others do not: the same bits."""
    D, L, window = 64, 330, 80
    pages = -(-L // P) + 1
    cache = filled(pages, 1, P, D, held, 4)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(P)).tolist()
    q = torch.randn(n, G, D, generator=torch.Generator().manual_seed(n)).to(kind).cuda()
    args = (q, i32([order]), i32([L]), i32([0, n]), 0.125, window)
    out, lse = cache.attention(*args)
    hidden = [order[p] for p in range(pages) if (p + 1) * P <= L - n + 1 - window or p * P >= L]
    assert any((p + 1) * P > (L - n + 1 - window) // 64 * 64 for p in range(pages) if order[p] in hidden and p * P < L) or P == 64
    for value in (math.inf, -math.inf, math.nan, 3.4e38, 0.0, -1.0):
        for scales in (cache.k_scale, cache.v_scale):
            scales[hidden] = value
            again, lse2 = cache.attention(*args)
            assert torch.equal(out, again) and torch.equal(lse, lse2), value
    last = (L - 1) // P
    see = L - last * P                                  # rows that see some of the last page
    if n > see:
        cache.v_scale[order[last]] = math.inf
        again, lse2 = cache.attention(*args)
        assert torch.equal(out[:n - see], again[:n - see]) and torch.equal(lse[:n - see], lse2[:n - see])


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 70])
def test_memory_that_nobody_has_written(n):
    """A cache of zeros, its scales too, as a warm-up may have it: results are finite, and next to nothing."""
    c = KvCache(*[torch.zeros_like(t.view(torch.uint8) if t.element_size() == 1 else t) for t in (lambda c: (c.k, c.v, c.k_scale, c.v_scale))(KvCache.empty(4, 2, 32, 64))])
    c.k, c.v = c.k.view(E4M3), c.v.view(E4M3)
    out, lse = c.attention(torch.randn(n, 4, 64).cuda(), i32([[0, 1, 2, 3]]), i32([100]), i32([0, n]))
    assert float(out.abs().max()) < 1e-30
    seen = torch.arange(100 - n + 1, 101).double()[:, None].expand(n, 4)
    assert bool(((lse.cpu().double() - seen.log()).abs() < 1e-5).all())


@pytest.mark.gpu
def test_scores_far_apart():
    """Scores of up to some thousands: one token takes everything, sums do not overflow."""
    c = filled(6, 1, 64, 64, E4M3, 11)
    c.k_scale *= 64.0
    check_attention([(300, 1), (50, 4)], E4M3, torch.float32, 64, 1, 2, 64, cache=c, scale=4.0)


@pytest.mark.gpu
def test_rows_of_no_request():
    """Behind the last request: zeros and -inf in results of the call's own, untouched in those given to it."""
    spec = [(40, 1), (70, 2)]
    check_attention(spec, E4M3, torch.bfloat16, 16, 2, 2, 64, pad=9)
    cache = filled(9, 2, 16, 64, E4M3, 1)
    table, lens, starts = requests(spec, 16, 9, 1)
    q = torch.randn(12, 4, 64).cuda()
    out, lse = torch.full_like(q, 7.0), torch.full((12, 4), 5.0, device="cuda")
    got = cache.attention(q, i32(table), i32(lens), i32(starts), out=out, lse=lse)
    want = cache.attention(q, i32(table), i32(lens), i32(starts))
    assert got[0].data_ptr() == out.data_ptr() and got[1].data_ptr() == lse.data_ptr()
    assert torch.equal(out[:3], want[0][:3]) and torch.equal(lse[:3], want[1][:3])
    assert bool((out[3:] == 7).all()) and bool((lse[3:] == 5).all()) and bool((want[0][3:] == 0).all()) and bool((want[1][3:] == -math.inf).all())
    empty = cache.attention(q[:0], i32(table), i32(lens), i32([0, 0, 0]))
    assert empty[0].shape == (0, 4, 64) and empty[1].shape == (0, 4)
    none = cache.attention(q, torch.empty(0, 3, dtype=torch.int32, device="cuda"), i32([]), i32([0]))
    assert bool((none[0] == 0).all()) and bool((none[1] == -math.inf).all())
    out.fill_(7)
    cache.attention(q, torch.empty(2, 0, dtype=torch.int32, device="cuda"), i32(lens), i32(starts), out=out, lse=lse)   # tables of no pages
    assert bool((out[:3] == 0).all()) and bool((out[3:] == 7).all()) and bool((lse[:3] == -math.inf).all())


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D,heads", [(64, 90), (128, 90), (256, 90), (64, 2)])
def test_rows_that_have_no_tokens(kind, D, heads):
    """Tables of no columns, tables of one behind lengths of 0, and a request of many rows without tokens beside one that has some: zeros and
    -inf, in calls of few rows (fx_kv_rows) and of many (16-bit ones of 49 152 rows and more: fx_kv_tiles)."""
    n = 600
    cache = filled(4, 2, 64, D, E4M3, 1)
    q = torch.randn(n + 5, heads, D, generator=torch.Generator().manual_seed(1)).to(kind).cuda()
    for table, lens, starts in (([[]], [700], [0, n]), ([[], []], [700, 3], [0, n, n + 2]), ([[1]], [0], [0, n]), ([[1], [-1]], [0, 0], [0, n, n + 2])):
        table = torch.tensor(table, dtype=torch.int32).view(len(lens), len(table[0])).cuda()
        out, lse = torch.full_like(q, 7.0), torch.full((n + 5, heads), 5.0, device="cuda")
        for o, l, rest in (cache.attention(q, table, i32(lens), i32(starts)) + ((0.0, -math.inf),), cache.attention(q, table, i32(lens), i32(starts), out=out, lse=lse) + ((7.0, 5.0),)):
            assert bool((o[:starts[-1]] == 0).all()) and bool((l[:starts[-1]] == -math.inf).all())
            assert bool((o[starts[-1]:] == rest[0]).all()) and bool((l[starts[-1]:] == rest[1]).all())
    check_attention([(0, 300), (200, 200), (0, 200)], E4M3, kind, 64, 2, heads // 2, D)


@pytest.mark.gpu
def test_views_and_strides():
    """A cache that is a layer of a larger one, queries that are a part of a joined product, a table that is a part of a wider one."""
    P, H, D, N = 32, 2, 64, 10
    big_k = torch.zeros(N, 3, H, P, D, dtype=torch.uint8, device="cuda").view(E4M3)
    big_v = torch.zeros(N, 3, H, P // 16, D, 16, dtype=torch.uint8, device="cuda").view(E4M3)
    scales = torch.zeros(N, 3, 2, H, device="cuda")
    src = filled(N, H, P, D, E4M3, 2)
    layer = KvCache(big_k[:, 1], big_v[:, 1], scales[:, 1, 0], scales[:, 1, 1])
    for a, b in ((layer.k.view(torch.uint8), src.k.view(torch.uint8)), (layer.v.view(torch.uint8), src.v.view(torch.uint8)), (layer.k_scale, src.k_scale), (layer.v_scale, src.v_scale)):
        a.copy_(b)
    table, lens, starts = requests([(70, 1), (100, 3)], P, N, 1)
    wide = torch.full((2, 9), -1, dtype=torch.int32, device="cuda")
    wide[:, :len(table[0])] = i32(table)
    qkv = torch.randn(4, 4 + 2 + 2, D, device="cuda")
    want = src.attention(qkv[:, :4].contiguous(), i32(table), i32(lens), i32(starts))
    got = layer.attention(qkv[:, :4], wide[:, :len(table[0])], i32(lens), i32(starts))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    turned = layer.attention(qkv[:, :4].transpose(1, 2).contiguous().transpose(1, 2), wide.t().contiguous().t(), i32(lens), i32(starts))
    assert torch.equal(turned[0], want[0])
    slots = torch.tensor([table[0][2] * P + 6, table[1][3] * P + 4, table[1][3] * P + 5]).cuda()
    for c in (layer, src):
        c.store(qkv[:3, 4:6], qkv[:3, 6:].transpose(1, 2).contiguous().transpose(1, 2), slots)
    assert torch.equal(layer.k.view(torch.uint8), src.k.view(torch.uint8)) and torch.equal(layer.v.view(torch.uint8), src.v.view(torch.uint8))
    assert torch.equal(layer.k_scale, src.k_scale) and bool((big_k[:, 0].view(torch.uint8) == 0).all()) and bool((big_v[:, 2].view(torch.uint8) == 0).all())


@pytest.mark.gpu
def test_refusals():
    c = filled(4, 2, 16, 64, E4M3, 1)
    table, lens, starts, slots = i32([[0, 1]]), i32([20]), i32([0, 2]), torch.tensor([3, 4]).cuda()
    q, k = torch.zeros(2, 4, 64, device="cuda"), torch.zeros(2, 2, 64, device="cuda")
    bad = [lambda: c.attention(q[:, :3], table, lens, starts), lambda: c.attention(q[..., :32], table, lens, starts), lambda: c.attention(q.double(), table, lens, starts),
           lambda: c.attention(q, table.long(), lens, starts), lambda: c.attention(q, table[0], lens, starts), lambda: c.attention(q, table, lens.long(), starts),
           lambda: c.attention(q, table, i32([1, 2]), starts), lambda: c.attention(q, table, lens, i32([0])), lambda: c.attention(q, table, lens, starts, 0.0),
           lambda: c.attention(q, table, lens, starts, -1.0), lambda: c.attention(q, table, lens, starts, math.nan), lambda: c.attention(q, table, lens, starts, window=-1),
           lambda: c.attention(q, table, lens, starts, max_new=-1), lambda: c.attention(q, table.cpu(), lens, starts), lambda: c.attention(q.cpu(), table, lens, starts),
           lambda: c.attention(q.clone().requires_grad_(), table, lens, starts), lambda: c.attention(q, table, lens, starts, out=q.clone()),
           lambda: c.attention(q, table, lens, starts, out=q.half(), lse=torch.zeros(2, 4, device="cuda")),
           lambda: c.attention(q, table, lens, starts, out=q.clone(), lse=torch.zeros(2, 3, device="cuda")),
           lambda: c.store(k, k, slots.int()), lambda: c.store(k[:1], k, slots), lambda: c.store(k, k.half(), slots), lambda: c.store(k.double(), k.double(), slots),
           lambda: c.store(k.clone().requires_grad_(), k, slots), lambda: c.store(k, k, slots.cpu()), lambda: c.store(k, k, slots[None]),
           lambda: c.read(slots.int()), lambda: c.read(slots, torch.int8), lambda: c.read(slots.cpu()),
           lambda: c.plan(i32([0, 0]), i32([1]), table.clone(), i32([2]), 1), lambda: c.plan(i32([0]), i32([1]), table.long(), i32([2]), 1),
           lambda: c.plan(i32([0]), i32([1]), table.clone(), i32([2]), -1), lambda: c.plan(i32([0]), i32([1]), table.clone(), i32([2]), 1, i32([0, 0])),
           lambda: c.plan(i32([0]), i32([1]), i32([[0, 1], [0, 1]]).t()[:1], i32([2]), 1), lambda: torch.ops.functs.kv_plan(i32([0]), i32([1]), table, i32([2]), 24, 1, None)]
    shapes = [KvCache(c.k[:, :, :8], c.v, c.k_scale, c.v_scale), KvCache(c.k, c.v[:, :, :, :32], c.k_scale, c.v_scale), KvCache(c.k, c.v, c.k_scale[:3], c.v_scale),
              KvCache(c.k, c.v, c.k_scale.double(), c.v_scale), KvCache(c.k.view(INT8), c.v, c.k_scale, c.v_scale), KvCache(c.k.float(), c.v.float(), c.k_scale, c.v_scale),
              KvCache(c.k.cpu(), c.v, c.k_scale, c.v_scale), KvCache(c.k, c.v, c.k_scale, c.v_scale.t().contiguous().t()), KvCache(c.k[:0], c.v[:0], c.k_scale[:0], c.v_scale[:0]),
              KvCache(c.k.view(torch.uint8).transpose(2, 3).contiguous().transpose(2, 3).view(E4M3), c.v, c.k_scale, c.v_scale)]
    bad += [lambda x=x: x.read(slots) for x in shapes] + [lambda x=x: x.store(k, k, slots) for x in shapes] + [lambda x=x: x.attention(q, table, lens, starts) for x in shapes]
    for i, call in enumerate(bad):
        with pytest.raises((RuntimeError, TypeError)):
            call()
            pytest.fail("call %d was not refused" % i)
    with torch.no_grad():
        c.attention(q.clone().requires_grad_(), table, lens, starts)


@pytest.mark.gpu
def test_more_refusals():
    """Scales that would leave the range of normal numbers with a page's, and gradients asked of what is written."""
    c = filled(4, 2, 16, 64, E4M3, 1)
    table, lens, starts, slots = i32([[0, 1]]), i32([20]), i32([0, 2]), torch.tensor([3, 4]).cuda()
    q, k = torch.zeros(2, 4, 64, device="cuda"), torch.zeros(2, 2, 64, device="cuda")
    grown = KvCache(c.k, c.v, c.k_scale.clone().requires_grad_(), c.v_scale)
    for call in (lambda: c.attention(q, table, lens, starts, 2.0 ** -27), lambda: c.attention(q, table, lens, starts, 33.0), lambda: grown.attention(q, table, lens, starts),
                 lambda: grown.store(k, k, slots), lambda: grown.read(slots),
                 lambda: c.attention(q, table, lens, starts, out=torch.zeros_like(q).requires_grad_(), lse=torch.zeros(2, 4, device="cuda"))):
        with pytest.raises(RuntimeError):
            call()
    with torch.no_grad():
        grown.store(k, k, slots)


@pytest.mark.gpu
def test_derivatives_are_refused():
    """Tangents of forward-mode differentiation on any operand, and codes that require a gradient."""
    c = filled(4, 2, 16, 64, E4M3, 1)
    table, lens, starts, slots = i32([[0, 1]]), i32([20]), i32([0, 2]), torch.tensor([3, 4]).cuda()
    q, k, lse = torch.zeros(2, 4, 64, device="cuda"), torch.zeros(2, 2, 64, device="cuda"), torch.zeros(2, 4, device="cuda")

    def refused(word, caches, store=(), attention=()):
        for x in caches:
            for call in (lambda: x.store(k, k, slots), lambda: x.read(slots), lambda: x.attention(q, table, lens, starts)):
                with pytest.raises(RuntimeError, match=word):
                    call()
        for a in store:
            with pytest.raises(RuntimeError, match=word):
                c.store(*a, slots)
        for a, kw in attention:
            with pytest.raises(RuntimeError, match=word):
                c.attention(a, table, lens, starts, **kw)

    with torch.autograd.forward_ad.dual_level():
        dual = lambda t: torch.autograd.forward_ad.make_dual(t.clone(), torch.ones_like(t))  # noqa: E731
        refused("carries a tangent", (KvCache(c.k, c.v, dual(c.k_scale), c.v_scale), KvCache(c.k, c.v, c.k_scale, dual(c.v_scale))), ((dual(k), k), (k, dual(k))),
                ((dual(q), {}), (q, dict(out=dual(q), lse=lse)), (q, dict(out=q.clone(), lse=dual(lse)))))
        with torch.no_grad():
            refused("carries a tangent", (), ((dual(k), k),), ((dual(q), {}),))
    grown = lambda t: t.clone().requires_grad_()  # noqa: E731
    caches = (KvCache(grown(c.k), c.v, c.k_scale, c.v_scale), KvCache(c.k, grown(c.v), c.k_scale, c.v_scale))
    refused("requires a gradient", caches)
    with torch.no_grad():
        caches[0].read(slots), caches[1].attention(q, table, lens, starts)


@pytest.mark.gpu
@pytest.mark.parametrize("held,top", [(E4M3, 119), (INT8, 121)])
@pytest.mark.parametrize("n", [1, 140])
def test_the_smallest_and_largest_scales(held, top, n):
    """Pages under the ends of the range of scales, and scale at its own: scores of ordinary size from numbers that are not."""
    for e, scale, size in ((-100, 2.0 ** -26, 2.0 ** 112), (top, 2.0 ** -20, 2.0 ** -105), (0, 32.0, 2.0 ** -8)):
        c = filled(6, 1, 64, 64, held, 3)
        c.k_scale.fill_(2.0 ** e)
        q = torch.randn(n, 2, 64, generator=torch.Generator().manual_seed(n)) * size
        table, lens, starts = [[4, 1, 2, 0]], [200], [0, n]
        out, lse = c.attention(q.cuda(), i32(table), i32(lens), i32(starts), scale)
        ref, rl, spread, most = PlainCache(c).attention(q, table, lens, starts, scale, 0)
        bound, lbound = tolerance(torch.float32, ref, rl, spread, most, 200, 64)
        assert bool(((out.cpu().double() - ref).abs() <= bound).all()) and bool(((lse.cpu().double() - rl).abs() <= lbound).all())


# n rows and query heads of a key head: one row, a few tiles of fx_kv_rows, and 49 152 rows and more (fx_kv_tiles, 16-bit queries)
ROWS = [(1, 2), (140, 2), (150, 330)]


@pytest.mark.gpu
@pytest.mark.parametrize("held", [E4M3, INT8])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,G", ROWS)
def test_small_weights_count_whatever_their_values_scale(held, kind, n, G):
    """One token whose score is 18.375 above the 5 999 others (2^-26.5 of its weight each, 1.1e-4 together of those that pages of zeros hold),
    whose pages hold zeros under scales from 0 to the largest.  Queries and keys have one column and a score is a product of two numbers of
    few bits: 6 roundings of it (scale, log2(e) twice, the sum with the maximum, the way back by ln(2)), then sums as in tolerance()."""
    L, P, D, scale = 6000, 64, 64, 147 / 64
    for vs in (2.0 ** -100, 0.0, 2.0 ** -64, 1.0, 2.0 ** 64, 2.0 ** 100, 2.0 ** (119 if held == E4M3 else 121)):
        c = filled(-(-L // P), 1, P, D, held, 5)
        c.k.view(torch.uint8).zero_(), c.k_scale.fill_(1.0)
        c.k.view(torch.uint8)[0, 0, 3, 0] = torch.tensor([8.0]).to(held).view(torch.uint8).item()
        c.v.view(torch.uint8)[1:].zero_(), c.v_scale[1:].fill_(vs)
        q = torch.zeros(n, 1, D)
        q[:, :, 0] = 1.0
        table, lens, starts = [list(range(c.k.size(0)))], [L], [0, n]
        out, lse = c.attention(q.expand(n, G, D).to(kind).cuda(), i32(table), i32(lens), i32(starts), scale)
        ref, rl, spread, size = PlainCache(c).attention(q, table, lens, starts, scale, 0)
        bound, _ = tolerance(kind, ref, rl, spread, size, L, D, n * G >= 49152)
        e = 2.0 ** -24
        assert bool(((out.cpu().double() - ref).abs() <= bound).all()), vs
        assert float((lse.cpu().double() - rl).abs().max()) <= 6 * e * 18.375 + 2.0 ** -22 + (L / 32 + 40) * e, vs


@pytest.mark.gpu
@pytest.mark.parametrize("held", [E4M3, INT8])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,G", ROWS)
def test_the_smallest_and_largest_scales_of_values(held, kind, n, G):
    """Pages under the ends of the range, alone and beside each other.  At the upper end codes are 0, 1 and -1, as values of more than 2^127
    over the number of tokens may become infinite; what a token adds below 2^-126 may be lost, of sums whose weights are 2^-8 at least."""
    L, P, D = 200, 64, 64
    top = 119 if held == E4M3 else 121
    small = kind == torch.float16                      # (its largest number is 65504)
    for exps, most in (((-100,) * 4, 448), ((-100, -64, -10, -65), 448), ((top,) * 4, 0)) + (() if small else (((119,) * 4, 1), ((-100, 64, 0, 90), 448), ((65, -63, 100, 119), 1))):
        c = filled(6, 1, P, D, held, 3)
        codes = c.v.float()
        c.v.copy_((codes.clamp(-most, most) if most != 1 else codes.sign() * (codes.abs() > 20)).to(held))
        table, lens, starts = [[4, 1, 2, 0]], [L], [0, n]
        for page, x in zip(table[0], exps):
            c.v_scale[page] = 2.0 ** x
        q = torch.randn(n, 1, D, generator=torch.Generator().manual_seed(n)).to(kind)
        out, lse = c.attention(q.expand(n, G, D).cuda(), i32(table), i32(lens), i32(starts))
        ref, rl, spread, size = PlainCache(c).attention(q, table, lens, starts, D ** -0.5, 0)
        bound, lbound = tolerance(kind, ref, rl, spread, size, L, D, n * G >= 49152)
        bound = bound + L * 448 * 2.0 ** -126 * 2.0 ** 8
        assert bool(((out.cpu().double() - ref).abs() <= bound).all()), exps
        assert bool(((lse.cpu().double() - rl).abs() <= lbound).all()), exps


# ---- GPU: together ----

def serve(steps, cache, table, free, tokens, seed, layers=1):
    """A small server: requests of different lengths get prompts, then a token a step; its caches against what was stored."""
    H, D = cache.k.size(1), cache.k.size(3)
    B = table.size(0)
    g = torch.Generator().manual_seed(seed)
    lens = i32([0] * B)
    free_start = i32([0])
    outs = []
    for new in steps:
        q, k, v = (torch.randn(tokens, h, D, generator=g).to(torch.bfloat16).cuda() for h in (2 * H, H, H))
        step = cache.plan(lens, i32(new), table, free, tokens, free_start)
        cache.store(k, v, step.slots)
        outs.append((step, cache.attention(q, table, step.lens, step.starts), q, k, v))
        free_start += step.taken
        lens = step.lens
    return outs


@pytest.mark.gpu
@pytest.mark.parametrize("held", [E4M3, INT8])
def test_plan_store_and_attention_together(held):
    """A server of four requests, some steps idle: every row of the last step sees its own request's tokens as they were stored step after
    step (the plain cache gets the same rows)."""
    P, H, D, tokens = 16, 2, 64, 64
    cache = KvCache.empty(20, H, P, D, held)
    cache.k.view(torch.uint8).fill_(0x7F), cache.v.view(torch.uint8).fill_(0x7F), cache.k_scale.fill_(math.nan), cache.v_scale.fill_(math.nan)
    plain = PlainCache(cache)
    table, free = torch.full((4, 6), -1, dtype=torch.int32, device="cuda"), torch.randperm(20, generator=torch.Generator().manual_seed(2)).int().cuda()
    steps = [[17, 0, 40, 3]] + [[1, 1, 1, 1]] * 3 + [[5, 20, 0, 1]] + [[1, 1, 1, 1]] * 14
    for i, (step, (out, lse), q, k, v) in enumerate(serve(steps, cache, table, free, tokens, 4)):
        plain.store(k, v, step.slots.cpu())
    last, (out, lse), q, k, v = serve(steps, cache, table.fill_(-1), free, tokens, 4)[-1]
    ref, rl, spread, size = plain.attention(q, table.tolist(), last.lens.tolist(), last.starts.tolist(), D ** -0.5, 0)
    assert last.lens.tolist() == [sum(s[b] for s in steps) for b in range(4)]
    most, lmost = tolerance(torch.bfloat16, ref, torch.where(torch.isfinite(rl), rl, 0.0), spread, size, 80, D)
    assert bool(((out.cpu().double() - ref).abs() <= most).all())
    fine = torch.isfinite(rl)
    assert torch.equal(fine, torch.isfinite(lse.cpu())) and bool(((lse.cpu().double() - rl).abs()[fine] <= lmost[fine]).all())


def scripted_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                  table: torch.Tensor, free: torch.Tensor, past: torch.Tensor, new: torch.Tensor, bias: torch.Tensor):
    slots, _, starts, lens, taken = torch.ops.functs.kv_plan(past, new, table, free, k_cache.size(2), q.size(0))
    torch.ops.functs.kv_store(k, v, k_cache, v_cache, k_scale, v_scale, slots)
    turned = q.clone()
    turned[:, :, :8] = turned[:, :, :8] * bias
    out, lse = torch.ops.functs.kv_attention(turned, k_cache, v_cache, k_scale, v_scale, table, lens, starts, 0.25)
    keys, values = torch.ops.functs.kv_read(k_cache, v_cache, k_scale, v_scale, slots, torch.float32)
    return out, lse, keys, values, lens, taken


def test_a_scripted_step_keeps_its_calls():
    """Script and functionalization leave the calls in their order (two of them write to tensors that they are given)."""
    names = [n.kind() for n in fj.script(scripted_step).graph.nodes() if n.kind().startswith("functs::kv_")]
    assert names == ["functs::kv_plan", "functs::kv_store", "functs::kv_attention", "functs::kv_read"]


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [6, 90])
def test_a_scripted_step(tokens):
    """The four calls in one built program, beside a region that is fused, against the same calls made one by one."""
    g = torch.Generator().manual_seed(tokens)
    q, k, v = (torch.randn(tokens, h, 64, generator=g).cuda() for h in (4, 2, 2))
    bias, free, past, new = torch.randn(8, generator=g).cuda(), torch.randperm(12, generator=g).int().cuda(), i32([0, 0, 0]), i32([tokens - 4, 0, 3])

    def inputs():
        c = filled(12, 2, 16, 64, E4M3, 3)
        return [q, k, v, c.k, c.v, c.k_scale, c.v_scale, torch.full((3, 8), -1, dtype=torch.int32, device="cuda"), free, past, new, bias]

    built = fj.build(fj.script(scripted_step), inputs())
    for _ in range(2):
        theirs, ours = inputs(), inputs()
        want, got = scripted_step(*theirs), built(*ours)
        for a, b in zip(want, got):
            assert torch.equal(a, b)
        for a, b in zip(theirs[3:8], ours[3:8]):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.gpu
def test_a_captured_step_serves_other_lengths():
    """Plan, store and attention in one graph: replayed with other lengths and rows in its tensors, with eager calls and waits in between, each
    replay gives what eager calls give."""
    P, H, D, tokens, B = 16, 2, 64, 40, 3
    eager, graphed = KvCache.empty(40, H, P, D), KvCache.empty(40, H, P, D)
    state = {}
    for name, c in (("eager", eager), ("graph", graphed)):
        c.k.view(torch.uint8).zero_(), c.v.view(torch.uint8).zero_(), c.k_scale.fill_(1.0), c.v_scale.fill_(1.0)
        state[name] = dict(past=i32([0] * B), new=i32([1] * B), table=torch.full((B, 30), -1, dtype=torch.int32, device="cuda"), start=i32([0]),
                           q=torch.zeros(tokens, 4, D, device="cuda"), k=torch.zeros(tokens, H, D, device="cuda"), v=torch.zeros(tokens, H, D, device="cuda"))
    free = torch.arange(40, dtype=torch.int32, device="cuda")

    def step(c, s):
        p = c.plan(s["past"], s["new"], s["table"], free, tokens, s["start"])
        c.store(s["k"], s["v"], p.slots)
        out, lse = c.attention(s["q"], s["table"], p.lens, p.starts)
        s["start"].add_(p.taken)
        s["past"].copy_(p.lens)
        return out, lse, p.slots

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(graphed, state["graph"])
    torch.cuda.current_stream().wait_stream(side)
    step(eager, state["eager"])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(graphed, state["graph"])
    g = torch.Generator().manual_seed(1)
    for new in ([1, 1, 1], [20, 0, 3], [1, 1, 1], [0, 30, 10], [1, 0, 1], [13, 13, 13]):
        for s in state.values():
            s["new"].copy_(i32(new))
        for name in ("q", "k", "v"):
            x = torch.randn(state["eager"][name].shape, generator=g).cuda()
            for s in state.values():
                s[name].copy_(x)
        graph.replay()
        want = step(eager, state["eager"])
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b), new
        assert torch.equal(state["eager"]["table"], state["graph"]["table"])
        assert torch.equal(eager.k.view(torch.uint8), graphed.k.view(torch.uint8)) and torch.equal(eager.v_scale, graphed.v_scale)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [3, 70])
def test_a_captured_call_of_both_kernels(n):
    """A call of 49 152 rows and more, recorded once and replayed with other lengths, offsets, tables and queries, eager calls and waits in between: requests
    that were long are short, empty or behind others, rows come before their tokens do, and every replay gives what an eager call gives."""
    H, G, P, pages, rows = 2, 90, 32, 200, 300
    cache = filled(pages, H, P, 64, E4M3, 3)
    q, table, lens, starts = torch.zeros(rows, H * G, 64, dtype=torch.bfloat16, device="cuda"), i32([[-1] * 40] * n), i32([0] * n), i32([0] * (n + 1))
    cache.attention(q, table, lens, starts, window=500)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = cache.attention(q, table, lens, starts, window=500)
    for i, spec in enumerate(([(1200, 200), (1, 1), (900, 90)], [(0, 150), (100, 140), (3, 1)], [(5, 0)] * 3, [(1280, 1), (0, 0), (700, 299)], [(64, 1)] * 2 + [(1100, 260)])):
        t, l, st = requests(spec, P, pages, i)
        for b in range(3):
            table[b] = i32(t[b][:40] + [-1] * (40 - len(t[b])))
        lens.copy_(i32(l + [0] * (n - 3))), starts.copy_(i32(st + [st[-1]] * (n - 3)))
        q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(i)).to(torch.bfloat16))
        want = cache.attention(q, table, lens, starts, window=500)
        for _ in range(2):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), spec
        tb, ref = table.tolist(), PlainCache(cache)
        part = slice(0, 2)                                # (two heads of each key head's: as many as a reference needs)
        few = torch.cat([q[:, part], q[:, G:G + 2]], 1)
        o, rl, spread, size = ref.attention(few, tb, lens.tolist(), starts.tolist(), 0.125, 500)
        most, _ = tolerance(torch.bfloat16, o, torch.where(torch.isfinite(rl), rl, 0.0), spread, size, 1280, 64, True)
        assert bool(((torch.cat([got[0][:, part], got[0][:, G:G + 2]], 1).cpu().double() - o).abs() <= most).all()), spec


@pytest.mark.gpu
@pytest.mark.parametrize("heads", [2, 4])
def test_two_streams_at_once(heads):
    """Calls on two streams, and two captured graphs that run side by side, keep their results apart (each has its own scratch memory)."""
    cache = filled(300, heads, 64, 64, E4M3, 4)
    table, lens, starts = requests([(9000, 1), (5000, 1)], 64, 300, 1)
    table, lens, starts = i32(table), i32(lens), i32(starts)
    qs = [torch.randn(2, heads * 4, 64, generator=torch.Generator().manual_seed(i)).cuda() for i in range(2)]
    want = [cache.attention(q, table, lens, starts)[0] for q in qs]
    torch.cuda.synchronize()
    streams, graphs, outs = [torch.cuda.Stream() for _ in qs], [], []
    for _ in range(20):
        got = []
        for q, s in zip(qs, streams):
            with torch.cuda.stream(s):
                got.append(cache.attention(q, table, lens, starts)[0])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    for q in qs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(cache.attention(q, table, lens, starts)[0])
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


@pytest.mark.gpu
@pytest.mark.parametrize("heads", [2, 8])
def test_results_do_not_change_from_call_to_call(heads):
    cache = filled(200, heads, 64, 128, E4M3, 4)
    table, lens, starts = requests([(9000, 1), (500, 3), (64, 1)], 64, 200, 1)
    q = torch.randn(5, heads * 4, 128).half().cuda()
    first = cache.attention(q, i32(table), i32(lens), i32(starts))
    for _ in range(10):
        again = cache.attention(q, i32(table), i32(lens), i32(starts))
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.gpu
def test_a_cache_of_more_than_two_to_the_32_bytes():
    """Pages whose offsets pass 32 bits: the last page of a cache of 4.3 GB (keys and values each)."""
    P, H, D = 256, 64, 256
    N = (1 << 32) // (P * H * D) + 2
    cache = KvCache.empty(N, H, P, D, INT8)
    page = N - 1
    slots = torch.arange(page * P, page * P + 20, device="cuda")
    k, v = rows_of(torch.float32, 20, H, D, 1)
    cache.store(k, v, slots)
    gk, gv = cache.read(slots, torch.float32)
    small = KvCache.empty(1, H, P, D, INT8)
    small.store(k, v, torch.arange(20, device="cuda"))
    wk, wv = small.read(torch.arange(20, device="cuda"), torch.float32)
    assert torch.equal(gk, wk) and torch.equal(gv, wv)
    q = torch.randn(1, H, D).cuda()
    a = cache.attention(q, i32([[page]]), i32([20]), i32([0, 1]))
    b = small.attention(q, i32([[0]]), i32([20]), i32([0, 1]))
    assert torch.equal(a[0], b[0])
