"""Pages of the paged cache behind a beam search's selection (functs::kv_fork, kv_copy; functs_amd/csrc/fxhip/fx_kv_fork*).

CPU: refusals.  GPU: the operators against a plain implementation in Python's own numbers, and a whole beam search on a small model, whose cache is
shared, copied and freed by them, against one whose every beam is computed anew in 64 bits."""
import ctypes
import math
import random

import pytest
import torch

import functs_amd.jit as fj  # noqa: F401
from functs_amd import beam, rotary
from functs_amd._lib import C, lib
from functs_amd.kv_cache import KvCache, copy_pages
from tests.test_kv_cache import E4M3, INT8, Cache, PlainCache, filled, i32
from tests.test_rotary import plain as turned


def fork_plain(parents, lens, table, free, P, start=0):
    """kv_fork, group by group, in Python's own numbers."""
    G, K, M = len(parents), len(parents[0]), len(table[0])
    old = [list(r) for r in table]
    table = [list(r) for r in table]
    free = free[min(max(start, 0), len(free)):]
    asked = taken = 0
    new_lens, copies, freed = [], [], []
    for g in range(G):
        rows = range(g * K, g * K + K)
        n_old = [lens[r] if 0 <= lens[r] <= M * P else 0 for r in rows]
        pages = [old[r][:-(-n // P)] for r, n in zip(rows, n_old)]
        tail = [pg[-1] if n % P else -1 for pg, n in zip(pages, n_old)]
        at = [p if 0 <= p < K else None for p in parents[g]]
        wanted = [tail[p] if p is not None else -1 for p in at]
        need = [w >= 0 and w in wanted[:j] for j, w in enumerate(wanted)]
        spare = []
        owner = {}
        for i in range(K):
            if tail[i] >= 0 and tail[i] not in wanted and tail[i] not in tail[:i]:
                owner[i] = len(spare)
                spare.append(tail[i])
        k = used = 0
        kept, alive = [], set()
        for j, r in enumerate(rows):
            p = at[j]
            n = n_old[p] if p is not None else 0
            own, page, got = [], None, True
            if p is not None:
                own = list(pages[p])
                if need[j]:
                    if k < len(spare):
                        page = spare[k]
                        used += 1
                    elif asked + k - len(spare) < len(free):
                        page = free[asked + k - len(spare)]
                        taken += 1
                    else:
                        got = False
                    k += 1
                if need[j] and got:
                    own[-1] = page
            if p is None or not got:
                new_lens.append(0)
                copies.append([-1, -1, 0])
                continue
            alive.add(p)
            new_lens.append(n)
            copies.append([tail[p], page, n % P] if need[j] else [-1, -1, 0])
            table[r][:len(own)] = own
        asked += max(0, k - len(spare))
        for c in range(M):
            for i in range(K):
                if i in alive or c >= len(pages[i]) or pages[i][c] < 0:
                    continue
                v = pages[i][c]
                if any(c < len(pages[o]) and pages[o][c] == v and (o in alive or o < i) for o in range(K) if o != i):
                    continue
                if i in owner and owner[i] < used and c == len(pages[i]) - 1:
                    continue
                freed.append(v)
    return new_lens, copies, [taken], freed, [len(freed)], table


def group_of(rng, G, K, P, M, same=0.6, first=False):
    """Tables of G groups whose beams share pages at the front, parents, lengths; pages 0 to N - 1 are theirs."""
    ids = list(range(G * K * M))
    rng.shuffle(ids)
    ids = iter(ids)
    parents, lens, table = [], [], []
    for g in range(G):
        n = rng.randint(0, M * P)
        common = rng.randint(0, n // P)
        shared = [next(ids) for _ in range(common)]
        for k in range(K):
            held = 0 if first and k else n if rng.random() < same else rng.randint(common * P, M * P)
            own = [next(ids) for _ in range(max(0, -(-held // P) - common))]
            row = (shared + own)[:-(-held // P)]
            table.append(row + [-1] * (M - len(row)))
            lens.append(held)
        parents.append([0] * K if first else [rng.choice([rng.randint(0, K - 1), rng.randint(0, (K - 1) // 2), k]) for k in range(K)])
    return parents, lens, table


def check_fork(parents, lens, table, free, P, start=None, stride=0):
    G, K, M = len(parents), len(parents[0]) if parents else 1, len(table[0]) if table else 0
    dev = torch.full((G * K, M + stride), -7, dtype=torch.int32, device="cuda")
    if G and M:
        dev[:, :M] = i32(table)
    view = dev[:, :M]
    c = KvCache.empty(1, 1, P, 16)
    got = c.fork(i32(parents).view(G, K), i32(lens), view, i32(free), None if start is None else i32([start]))
    want = fork_plain(parents, lens, table, free, P, start or 0) if G else ([], [], [0], [], [0], [])
    assert got.lens.tolist() == want[0] and got.copies.tolist() == want[1] and got.taken.tolist() == want[2] and got.n_freed.tolist() == want[4]
    n = want[4][0]
    assert got.freed.tolist()[:n] == want[3] and got.freed.shape == (G * K * M,) and bool((got.freed[n:] == -1).all())
    assert view.tolist() == want[5] and bool((dev[:, M:] == -7).all())
    return got, want


# ---- CPU ----

def test_tensors_on_the_host_are_refused():
    c = KvCache.empty(2, 2, 16, 64, device="cpu")
    z = lambda *n: torch.zeros(*n, dtype=torch.int32)  # noqa: E731
    for call in (lambda: c.fork(z(1, 2), z(2), z(2, 3), z(1)), lambda: copy_pages([c], z(2, 3)), lambda: copy_pages([], z(2, 3))):
        with pytest.raises(RuntimeError, match="runs on the GPU only"):
            call()


def test_mutated_arguments_are_in_the_schemas():
    for name, written in (("kv_fork", {"block_table"}), ("kv_copy", {"k_caches", "v_caches", "k_scales", "v_scales"})):
        schema = getattr(torch.ops.functs, name).default._schema
        assert {a.name for a in schema.arguments if a.alias_info is not None and a.alias_info.is_write} == written


class Desc(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("parents", "lens", "table")] + [("table_stride", ctypes.c_int64)] + \
               [(n, ctypes.c_void_p) for n in ("free_pages", "free_start", "out_lens", "copies", "taken", "freed", "n_freed")] + \
               [(n, ctypes.c_int32) for n in ("groups", "beams", "columns", "n_free", "page_size", "reserved")] + [("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_size_t)]


def test_the_c_abi_refuses_before_it_launches():
    at = 4096   # never read: each call returns from its checks
    ok = dict(parents=at, lens=at, table=at, table_stride=5, free_pages=at, out_lens=at, copies=at, taken=at, freed=at, n_freed=at, groups=2, beams=4, columns=5, n_free=3, page_size=16,
              workspace=at, workspace_bytes=1 << 30)
    lib.fx_kv_fork_workspace_bytes.restype = ctypes.c_size_t
    for change, code in ((dict(page_size=20), "FX_E_UNSUPPORTED"), (dict(beams=0), "FX_E_UNSUPPORTED"), (dict(beams=33), "FX_E_UNSUPPORTED"), (dict(groups=-1), "FX_E_INVALID"),
                         (dict(columns=-1), "FX_E_INVALID"), (dict(n_free=-1), "FX_E_INVALID"), (dict(parents=None), "FX_E_INVALID"), (dict(table=None), "FX_E_INVALID"),
                         (dict(copies=None), "FX_E_INVALID"), (dict(freed=None), "FX_E_INVALID"), (dict(n_freed=None), "FX_E_INVALID"), (dict(free_pages=None), "FX_E_INVALID"),
                         (dict(table_stride=4), "FX_E_INVALID"), (dict(workspace=None), "FX_E_INVALID"), (dict(workspace=at + 4), "FX_E_INVALID"), (dict(workspace_bytes=100), "FX_E_INVALID"),
                         (dict(groups=1 << 24), "FX_E_LIMIT"), (dict(columns=1 << 28, table_stride=1 << 28), "FX_E_LIMIT"), (dict(groups=1 << 20, columns=1 << 10, table_stride=1 << 10), "FX_E_LIMIT")):
        d = Desc(**{**ok, **change})
        assert lib.fx_kv_fork(ctypes.byref(d), None) == C[code], change
        assert b"fx_kv_fork" in lib.fx_last_error()
    assert lib.fx_kv_fork(None, None) == C["FX_E_INVALID"] and lib.fx_kv_fork_workspace_bytes(None) == 0
    cache = dict(k=at, v=at, k_scale=at, v_scale=at, ks=2 * 16 * 64, vs=2 * 16 * 64, kss=2, vss=2, pages=2, heads=2, page_size=16, depth=64, held=0)

    def copy(*changes, n=None, copies=at, rows=3):
        caches = (Cache * max(1, len(changes)))(*[Cache(**{**cache, **c}) for c in changes])
        return lib.fx_kv_copy(caches, len(changes) if n is None else n, ctypes.c_void_p(copies), rows, None)

    for call, code in ((lambda: copy(dict(held=3)), "FX_E_UNSUPPORTED"), (lambda: copy({}, dict(depth=40)), "FX_E_UNSUPPORTED"), (lambda: copy({}, dict(depth=32)), "FX_E_INVALID"),
                       (lambda: copy({}, dict(held=1)), "FX_E_INVALID"), (lambda: copy({}, {}, dict(vs=2 * 16 * 64 + 16)), "FX_E_INVALID"), (lambda: copy({}, dict(pages=3)), "FX_E_INVALID"),
                       (lambda: copy({}, n=-1), "FX_E_INVALID"), (lambda: copy({}, rows=-1), "FX_E_INVALID"), (lambda: copy({}, copies=None), "FX_E_INVALID"),
                       (lambda: copy({}, rows=1 << 26), "FX_E_LIMIT")):
        assert call() == C[code]
        assert b"fx_kv_copy" in lib.fx_last_error()
    assert copy() == 0 and copy({}, rows=0) == 0   # nothing to do


# ---- GPU: fork ----

@pytest.mark.gpu
@pytest.mark.parametrize("G,K,P,M", [(1, 1, 16, 1), (1, 4, 16, 5), (3, 2, 32, 9), (32, 4, 64, 33), (70, 8, 16, 40), (5, 32, 128, 7), (2, 3, 16, 700), (300, 7, 256, 3), (1100, 1, 16, 4),
                                     (128, 8, 16, 6), (146, 7, 32, 6), (1, 8, 16, 768), (5, 3, 16, 409), (1, 8, 16, 4097), (1024, 1, 64, 4)])
@pytest.mark.parametrize("first", [False, True])
def test_fork(G, K, P, M, first):
    rng = random.Random(G + 100 * K + M)
    parents, lens, table = group_of(rng, G, K, P, M, first=first)
    free = list(range(10 ** 6, 10 ** 6 + G * K))
    rng.shuffle(free)
    got, want = check_fork(parents, lens, table, free, P)
    check_fork(parents, lens, table, free[:max(0, want[2][0] // 2)], P, stride=3)      # too few free pages
    check_fork(parents, lens, table, free, P, start=G * K - max(1, want[2][0] - 1))    # some are given already
    check_fork(parents, lens, table, [], P)
    # a step later: every row has a last page of its own, rows behind their tokens as they were
    lens, table = want[0], want[5]
    again = [[rng.randint(-1, K) for _ in range(K)] for _ in range(G)]
    check_fork(again, lens, table, free[want[2][0]:], P)


@pytest.mark.gpu
def test_fork_of_what_makes_no_sense():
    check_fork([], [], [], [3, 4], 16)
    check_fork([[0, 0]], [0, 0], [[], []], [], 16)
    check_fork([[0, 0]], [5, 0], [[], []], [1], 16)                                            # more tokens than columns
    check_fork([[1, 0, 7], [-5, 2, 2 ** 31 - 1]], [-3, 40, 33, 2 ** 31 - 1, 16, 5], [[1, 2], [3, 4], [5, 6], [7, 8], [9, -1], [10, -1]], [20, 21], 16)
    check_fork([[0, 0, 0, 1]], [20, 20, 20, 3], [[1, 2], [1, 2], [1, 2], [4, -1]], [9], 16)   # a partly filled page in the tables of three rows
    check_fork([[0, 1, 2]], [20, 20, 20], [[1, 2], [1, 2], [1, 2]], [9, 8], 16)               # each gets one of its own
    check_fork([[1, 1, 1]], [20, 20, 20], [[1, 2], [1, -1], [-4, 3]], [9, 8], 16)             # entries that are no pages
    check_fork([[1, 1]], [20, 20], [[1, 2], [1, 3]], [-1, -1], 16)                             # a free page that is none: spare ones go first
    check_fork([[1, 1, 1]], [0, 20, 0], [[1, 2], [1, 3], [4, 5]], [-1, 7], 16)
    for start in (-5, 1, 100):
        check_fork([[0, 0, 0]], [7, 0, 0], [[1], [-1], [-1]], [30, 31], 16, start=start)


@pytest.mark.gpu
def test_pages_are_conserved():
    """Over many steps: every page is in some row, free, or neither twice."""
    rng = random.Random(7)
    G, K, P, M = 4, 5, 16, 12
    pool = list(range(G * K * M))
    rng.shuffle(pool)
    lens = [0] * (G * K)
    table = [[-1] * M for _ in range(G * K)]
    c = KvCache.empty(1, 1, P, 16)
    for g in range(G):                               # prompts, in the first row of each group
        n = rng.randint(1, 60)
        lens[g * K] = n
        for i in range(-(-n // P)):
            table[g * K][i] = pool.pop()
    dev = i32(table)
    for step in range(40):
        parents = [[0] * K for _ in range(G)] if step == 0 else [[rng.randint(0, K - 1) for _ in range(K)] for _ in range(G)]
        want = fork_plain(parents, lens, dev.tolist(), pool, P)
        got = c.fork(i32(parents), i32(lens), dev, i32(pool))
        assert got.lens.tolist() == want[0] and dev.tolist() == want[5]
        pool = pool[int(got.taken):] + got.freed.tolist()[:int(got.n_freed)]
        lens = got.lens.tolist()
        used = [set(r[:-(-n // P)]) for r, n in zip(dev.tolist(), lens)]
        whole = set().union(*used)
        assert len(pool) == len(set(pool)) and not whole & set(pool) and len(whole) + len(pool) == G * K * M
        tails = [dev[r, n // P].item() for r, n in enumerate(lens) if n % P]
        assert len(tails) == len(set(tails)) and not set(tails) & set().union(*[set(r[:n // P]) for r, n in zip(dev.tolist(), lens)])
        new = [1 if n < M * P else 0 for n in lens]
        plan = c.plan(i32(lens), i32(new), dev, i32(pool), G * K)
        pool = pool[int(plan.taken):]
        lens = plan.lens.tolist()


@pytest.mark.gpu
def test_fork_refusals():
    c = KvCache.empty(1, 1, 16, 16)
    p, n, t, f = i32([[0, 1]]), i32([3, 3]), i32([[0, 1], [2, 3]]), i32([5])
    for call, word in ((lambda: c.fork(p.long(), n, t, f), "parents must be"), (lambda: c.fork(p[0], n, t, f), "parents must be"), (lambda: c.fork(p, n[:1], t, f), "lens must be"),
                       (lambda: c.fork(p, n, t[:1], f), "block_table must be"), (lambda: c.fork(p, n, t.long(), f), "block_table must be"), (lambda: c.fork(p, n, t.t(), f), "block_table must be"),
                       (lambda: c.fork(p, n, t, f.long()), "free_pages must be"), (lambda: c.fork(p, n, t, f, i32([0, 1])), "free_start"), (lambda: c.fork(p.cpu(), n, t, f), "GPU only"),
                       (lambda: c.fork(p.expand(1, 2).repeat(1, 17), i32([0] * 34), t.repeat(17, 1), f), "beams a group"), (lambda: torch.ops.functs.kv_fork(p, n, t, f, 48), "page_size"),
                       (lambda: c.fork(p, n, t[:1].expand(2, 2), f), "overlap")):
        with pytest.raises(RuntimeError, match=word):
            call()


# ---- GPU: copy ----

def check_copy(caches, copies):
    P = caches[0].k.size(2)
    want = []
    for c in caches:
        k, v, ks, vs = (t.view(torch.uint8).clone() if t.element_size() == 1 else t.clone() for t in (c.k, c.v, c.k_scale, c.v_scale))
        for src, dst, n in copies:
            if 0 <= src < k.size(0) and 0 <= dst < k.size(0):
                n = min(max(n, 0), P)
                k[dst, :, :n] = k[src, :, :n]
                v[dst, :, :-(-n // 16)] = v[src, :, :-(-n // 16)]
                ks[dst], vs[dst] = ks[src], vs[src]
        want.append((k, v, ks, vs))
    copy_pages(caches, i32(copies).view(-1, 3))
    for c, w in zip(caches, want):
        for t, x in zip((c.k, c.v, c.k_scale, c.v_scale), w):
            assert torch.equal(t.view(torch.uint8) if t.element_size() == 1 else t, x)


@pytest.mark.gpu
@pytest.mark.parametrize("held", [E4M3, INT8])
@pytest.mark.parametrize("layers,P,H,D", [(1, 16, 1, 16), (3, 64, 8, 128), (33, 32, 3, 80), (2, 256, 2, 256), (40, 16, 12, 64), (1, 128, 130, 16)])
def test_copy(layers, P, H, D, held):
    N = 12
    caches = [filled(N, H, P, D, held, i) for i in range(layers)]
    rng = random.Random(P + D)
    order = list(range(N))
    rng.shuffle(order)
    src, dst = order[:5], order[5:11]
    copies = [(rng.choice(src), d, rng.choice([0, 1, 15, 16, 17, P - 1, P])) for d in dst]
    rows = copies[:3] + [(-1, -1, 0), (-1, order[11], 5), (src[0], -1, 5), (src[0], N, 5), (N, order[11], 5), (2 ** 31 - 1, -2 ** 31, 3), (src[1], src[1], 9)] + copies[3:]
    check_copy(caches, rows)
    check_copy(caches, [(src[0], dst[0], -5), (src[1], dst[1], 10 ** 9)])
    check_copy(caches, [])


@pytest.mark.gpu
def test_copy_of_many_rows_and_views():
    """Rows of more than one list, most of which copy nothing; pages of a wider cache; layers in one tensor."""
    P, H, D = 16, 2, 32
    whole = [filled(700, 4, P, D, E4M3, i) for i in range(2)]
    caches = [KvCache(c.k[:, 1:3], c.v[:, 1:3], c.k_scale[:, 1:3], c.v_scale[:, 1:3]) for c in whole]
    rng = random.Random(3)
    order = list(range(700))
    rng.shuffle(order)
    rows = [(-1, -1, 0)] * 2500
    for i, at in enumerate(rng.sample(range(2500), 300)):
        rows[at] = (order[i % 200], order[300 + i], rng.randint(1, P))
    before = [c.k.clone() for c in whole]
    check_copy(caches, rows)
    for c, b in zip(whole, before):
        assert torch.equal(c.k.view(torch.uint8)[:, [0, 3]], b.view(torch.uint8)[:, [0, 3]])


@pytest.mark.gpu
def test_copy_refusals():
    a, b = filled(3, 2, 16, 32, E4M3, 1), filled(3, 2, 16, 32, INT8, 1)
    rows = i32([[0, 1, 3]])
    for call, word in ((lambda: copy_pages([a], rows.long()), "copies must be"), (lambda: copy_pages([a], rows[0]), "copies must be"), (lambda: copy_pages([a], rows[:, :2]), "copies must be"),
                       (lambda: copy_pages([a, b], rows), "same sizes, types"), (lambda: copy_pages([a, filled(4, 2, 16, 32, E4M3, 1)], rows), "same sizes, types"),
                       (lambda: copy_pages([a], rows.cpu()), "GPU only"), (lambda: torch.ops.functs.kv_copy([a.k], [a.v], [a.k_scale], [], rows), "as many")):
        with pytest.raises(RuntimeError, match=word):
            call()


@pytest.mark.gpu
def test_a_cache_of_more_than_two_to_the_32_bytes():
    P, H, D = 256, 32, 256
    N = (1 << 32) // (H * P * D) + 40
    c = KvCache.empty(N, H, P, D)
    for t in (c.k, c.v):
        t.view(torch.uint8)[N - 20:] = torch.randint(0, 100, t[N - 20:].shape, dtype=torch.uint8, device="cuda")
    c.k_scale[N - 20:], c.v_scale[N - 20:] = 2.0, 4.0
    copy_pages([c], i32([[N - 1, 3, 100], [N - 7, N - 30, 256]]))
    assert torch.equal(c.k.view(torch.uint8)[3, :, :100], c.k.view(torch.uint8)[N - 1, :, :100]) and torch.equal(c.v.view(torch.uint8)[3, :, :7], c.v.view(torch.uint8)[N - 1, :, :7])
    assert torch.equal(c.k.view(torch.uint8)[N - 30], c.k.view(torch.uint8)[N - 7]) and float(c.k_scale[3, 0]) == 2.0 and float(c.v_scale[N - 30, 5]) == 4.0


@pytest.mark.gpu
def test_launches():
    total, special = ctypes.c_uint64(), ctypes.c_uint64()

    def launches(call):
        lib.fx_launch_stats(ctypes.byref(total), ctypes.byref(special))
        before = total.value
        call()
        lib.fx_launch_stats(ctypes.byref(total), ctypes.byref(special))
        return total.value - before

    c = filled(3, 1, 16, 16, E4M3, 1)
    assert launches(lambda: c.fork(i32([[0, 1]]), i32([3, 3]), i32([[0, 1], [2, 3]]), i32([5]))) == 1
    for G, K, M, n in ((128, 8, 6, 1), (128, 8, 7, 3), (129, 8, 3, 3), (1, 9, 2, 3), (1, 8, 768, 1), (1, 8, 769, 3), (341, 3, 6, 1), (342, 3, 2, 3), (1024, 1, 6, 1), (1024, 1, 7, 3)):
        assert launches(lambda: c.fork(torch.zeros(G, K, dtype=torch.int32, device="cuda"), i32([3] * (G * K)), i32([[0] * M] * (G * K)), i32([5]))) == n, (G, K, M)
    assert launches(lambda: c.fork(i32([]).view(0, 2), i32([]), i32([]).view(0, 3), i32([5]))) == 1
    assert launches(lambda: copy_pages([c] * 5, i32([[0, 1, 3]]))) == 1 and launches(lambda: copy_pages([c] * 33, i32([[0, 1, 3]]))) == 2 and launches(lambda: copy_pages([], i32([[0, 1, 3]]))) == 0


# ---- GPU: a beam search ----

class Model:
    """Two layers of rotary attention over a vocabulary, random weights, no norms: enough for every operator of a step to matter."""

    def __init__(self, V, H, G, D, seed):
        g = torch.Generator().manual_seed(seed)
        W = H * G * D
        normal = lambda *n: torch.randn(*n, generator=g, dtype=torch.double) / math.sqrt(n[0])  # noqa: E731
        self.V, self.H, self.G, self.D = V, H, G, D
        self.embed = torch.randn(V, W, generator=g, dtype=torch.double)
        self.qkv = [normal(W, (G + 2) * H * D) for _ in range(2)]
        self.out = [normal(W, W) for _ in range(2)]
        self.head = normal(W, V) * 1.5
        self.frequencies, self.magnitude = rotary.frequencies(D // 2, device="cpu")

    def to(self, dtype):
        m = Model.__new__(Model)
        m.__dict__.update(self.__dict__)
        move = lambda t: t.to(dtype).cuda()  # noqa: E731
        m.embed, m.qkv, m.out, m.head, m.frequencies = move(self.embed), [move(t) for t in self.qkv], [move(t) for t in self.out], move(self.head), self.frequencies.cuda()
        return m

    def run(self, words, attend):
        """words [tokens]; attend(layer, q, k, v) -> [tokens, query heads, depth]"""
        x, H, G, D = self.embed[words], self.H, self.G, self.D
        for l in range(2):
            qkv = (x @ self.qkv[l]).view(-1, (G + 2) * H, D)
            x = x + attend(l, qkv[:, :G * H], qkv[:, G * H:(G + 1) * H], qkv[:, (G + 1) * H:]).reshape(x.shape) @ self.out[l]
        return x @ self.head


def logits_plain(model, words, held, P):
    """Logits of the last of `words`, everything computed anew in 64 bits, keys and values as codes under their pages' scales, stored as the search stores them: the prompt
    at once, then a token at a time."""
    words = torch.tensor(words)
    prompt, words = words[:held["prompt"]], words
    n = len(words)
    caches = [KvCache.empty(-(-n // P), model.H, P, model.D, held["dtype"], "cpu") for _ in range(2)]
    for c in caches:
        c.k_scale.fill_(1.0), c.v_scale.fill_(1.0)
        c.k.view(torch.uint8).zero_(), c.v.view(torch.uint8).zero_()
    plains = [PlainCache(c) for c in caches]
    done = 0
    for size in [len(prompt)] + [1] * (n - len(prompt)):
        positions = torch.arange(done, done + size)
        table = [list(range(-(-n // P)))]

        def attend(l, q, k, v):
            k, q = turned(k, positions, model.frequencies, model.magnitude)[0], turned(q, positions, model.frequencies, model.magnitude)[0]
            plains[l].store(k, v, positions)
            return plains[l].attention(q, table, [done + size], [0, size], model.D ** -0.5, 0)[0]

        logits = model.run(words[done:done + size], attend)
        done += size
    return logits[-1]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [E4M3, INT8])
@pytest.mark.parametrize("P,K,seed", [(16, 4, 1), (32, 3, 2)])
def test_a_beam_search(dtype, P, K, seed):
    """Prompts of two requests, then steps of K beams: plan, append, attention, logits, select, fork, copy, all on the device.  Every step's totals are those of each beam's words
    computed anew in 64 bits (no other beam, page or copy in it): off by fp32 products, 2^-24 a term and some 2^8 terms a number, weights off by 2^-22, and by codes that fall
    on the other side of a rounding, which are 2^-4 of a value each and few; so totals agree to 0.02 of values of size 1 to 10, and a beam that read another's page would be off by as
    much as its logits differ, which is more than that."""
    model = Model(61, 2, 2, 32, seed)
    m = model.to(torch.float32)
    prompts = [[5, 3, 60, 7, 22, 31, 8, 9, 10, 11, 50, 49, 2, 1, 0, 17, 18][:11 + 6 * (seed % 2)], [4, 4, 8, 15, 16, 23, 42, 1, 9]]
    R, steps = len(prompts), 24
    pages = R * K * 4
    caches = [KvCache.empty(pages, model.H, P, model.D, dtype) for _ in range(2)]
    table = torch.full((R * K, 4), -1, dtype=torch.int32, device="cuda")
    free = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).int().cuda()
    zero = i32([0])

    def step(past, new, words, most):
        nonlocal free
        plan = caches[0].plan(past, new, table, free, most, zero)
        free = free[int(plan.taken):]

        def attend(l, q, k, v):
            q = caches[l].append(q, k, v, plan.slots, plan.positions, m.frequencies, m.magnitude)
            return caches[l].attention(q, table, plan.lens, plan.starts, max_new=0)[0]

        return plan, m.run(words, attend)

    # the prompts, in the first beam of each request
    new = i32([len(p) if k == 0 else 0 for p in prompts for k in range(K)])
    plan, logits = step(torch.zeros_like(new), new, torch.tensor(sum(prompts, [])).cuda(), sum(map(len, prompts)))
    last = torch.stack([logits[len(prompts[0]) - 1], logits[-1]])
    logits = last[:, None].expand(R, K, model.V)
    scores, lens = beam.first_scores(R, K), plan.lens
    texts = [[list(p)] + [None] * (K - 1) for p in prompts]
    totals = [[0.0] + [-math.inf] * (K - 1) for _ in range(R)]
    freed = 0
    for t in range(steps):
        chosen = beam.select(logits, scores)
        # the plain search's totals of what was chosen, and that nothing better was passed over
        beams, words, got = chosen.beams.tolist(), chosen.words.tolist(), chosen.scores.tolist()
        for r in range(R):
            if t in (0, 1, 2, 9, steps - 1):
                every = {}
                for k in range(K):
                    if texts[r][k] is not None:
                        y = logits_plain(model, texts[r][k], dict(prompt=len(prompts[r]), dtype=dtype), P)
                        for w, x in enumerate((y - torch.logsumexp(y, 0)).tolist()):
                            every[k, w] = totals[r][k] + x
                best = sorted(every.values(), reverse=True)[:K]
                for i in range(K):
                    assert abs(every[beams[r][i], words[r][i]] - got[r][i]) <= 0.02, (t, r, i)
                    assert abs(best[i] - got[r][i]) <= 0.02, (t, r, i)
            texts[r] = [texts[r][b] + [w] for b, w in zip(beams[r], words[r])]
        totals = got
        fork = caches[0].fork(chosen.beams, lens, table, free, zero)
        copy_pages(caches, fork.copies)
        free = torch.cat([free[int(fork.taken):], fork.freed[:int(fork.n_freed)]])
        freed += int(fork.n_freed)
        ones = torch.ones(R * K, dtype=torch.int32, device="cuda")
        plan, logits = step(fork.lens, ones, chosen.words.view(-1), R * K)
        scores, lens, logits = chosen.scores, plan.lens, logits.view(R, K, model.V)
        assert lens.tolist() == [len(texts[r][0]) for r in range(R) for _ in range(K)]
        rows = table.tolist()
        used = set().union(*[set(rows[i][:-(-n // P)]) for i, n in enumerate(lens.tolist())])
        assert len(used) + len(free) == pages and not used & set(free.tolist())


@pytest.mark.gpu
def test_a_captured_step_of_a_beam_search():
    """Select, fork and copy in one graph, replayed on other logits, against the same calls made eagerly."""
    R, K, V, P, H, D = 3, 4, 500, 16, 2, 32
    rng = random.Random(5)
    parents, lens_, table_ = group_of(rng, R, K, P, 6, same=1.0)
    pages = R * K * 6 + 40
    cache = [filled(pages, H, P, D, E4M3, i) for i in range(3)]
    logits, scores = torch.zeros(R, K, V, device="cuda"), torch.zeros(R, K, device="cuda")
    table, lens, free = i32(table_), i32(lens_), torch.arange(pages - 40, pages).int().cuda()

    def calls(caches, table):
        chosen = beam.select(logits, scores)
        fork = caches[0].fork(chosen.beams, lens, table, free)
        copy_pages(caches, fork.copies)
        return tuple(chosen) + tuple(fork)

    twin = [KvCache(c.k.clone(), c.v.clone(), c.k_scale.clone(), c.v_scale.clone()) for c in cache]
    twin_table = table.clone()
    calls(twin, twin_table)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = calls(cache, table)
    graph.replay()
    for seed in range(4):
        torch.cuda.synchronize()
        assert torch.equal(table, twin_table)
        for a, b in zip(cache, twin):
            for x, y in ((a.k, b.k), (a.v, b.v)):
                assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
            assert torch.equal(a.k_scale, b.k_scale) and torch.equal(a.v_scale, b.v_scale)
        logits.copy_(torch.randn(R, K, V, generator=torch.Generator().manual_seed(seed)) * 3)
        lens.copy_(out[3])
        eager = calls(twin, twin_table)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager))
