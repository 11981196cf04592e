"""functs::kv_append: rotated keys and values into the paged cache, rotated queries beside them (functs_amd/csrc/fxhip/fx_kv_append.hip,
fx_kv_store.h).

Its result is defined by two other operators: fp32 rows turned by functs::rotary, stored by functs::kv_store, bit for bit; both are compared with
64 bits in their own tests.  What is read again is compared with 64 bits here as well."""
import ctypes
import math

import pytest
import torch

import functs_amd.jit as fj  # noqa: F401
from functs_amd import rotary
from functs_amd._lib import C, lib
from functs_amd.kv_cache import KvCache
from tests.test_kv_cache import E4M3, INT8, Cache, Rows, filled, i32, rows_of
from tests.test_rotary import Desc, plain


def copied(c):
    return KvCache(c.k.clone(), c.v.clone(), c.k_scale.clone(), c.v_scale.clone())


def same_cache(a, b):
    for name in ("k", "v", "k_scale", "v_scale"):
        x, y = getattr(a, name), getattr(b, name)
        x, y = (t.view(torch.uint8) if t.element_size() == 1 else t.view(torch.int32) for t in (x, y))
        assert torch.equal(x, y), name


def check(cache, q, k, v, slots, positions, f, magnitude=1.0, interleaved=False):
    two = copied(cache)
    turned = rotary.rotary(k.float(), positions, f, magnitude, interleaved)
    two.store(turned, v.float(), slots)
    want = rotary.rotary(q, positions, f, magnitude, interleaved)
    got = cache.append(q, k, v, slots, positions, f, magnitude, interleaved)
    assert got.dtype == q.dtype and got.is_contiguous() and torch.equal(got.view(torch.int32 if q.dtype == torch.float32 else torch.int16),
                                                                       want.view(torch.int32 if q.dtype == torch.float32 else torch.int16))
    same_cache(cache, two)
    return turned


def queries(kind, tokens, heads, depth, seed):
    return torch.randn(tokens, heads, depth, generator=torch.Generator().manual_seed(seed)).to(kind).cuda()


# ---- CPU ----

def test_tensors_on_the_host_are_refused():
    c = KvCache.empty(2, 2, 16, 64, device="cpu")
    q, n = torch.zeros(3, 4, 64), torch.zeros(3, dtype=torch.long)
    with pytest.raises(RuntimeError, match="runs on the GPU only"):
        c.append(q, q[:, :2], q[:, :2], n, n, rotary.frequencies(64, device="cpu")[0])


def test_mutated_arguments_are_in_the_schema():
    schema = torch.ops.functs.kv_append.default._schema
    assert {a.name for a in schema.arguments if a.alias_info is not None and a.alias_info.is_write} == {"k_cache", "v_cache", "k_scale", "v_scale"}


def test_the_c_abi_refuses_before_it_launches():
    at = 4096   # never read: each call returns from its checks
    cache = dict(k=at, v=at, k_scale=at, v_scale=at, ks=2 * 16 * 64, vs=2 * 16 * 64, kss=2, vss=2, pages=2, heads=2, page_size=16, depth=64, held=0)
    rows = dict(k=at, v=at, kt=128, kh=64, vt=128, vh=64, slots=at, tokens=3, dtype=C["FX_DT_BF16"])
    turn = dict(x=at, y=at, positions=at, frequencies=at, xt=256, xh=64, yt=256, yh=64, batch=1, tokens=3, heads=4, depth=64, pairs=32, dtype=C["FX_DT_BF16"], magnitude=1.0)

    def call(c={}, r={}, t={}):
        return lib.fx_kv_append(ctypes.byref(Cache(**{**cache, **c})), ctypes.byref(Rows(**{**rows, **r})), ctypes.byref(Desc(**{**turn, **t})), None)

    for change, code in ((dict(c=dict(held=2)), "FX_E_UNSUPPORTED"), (dict(c=dict(depth=40)), "FX_E_UNSUPPORTED"), (dict(c=dict(k=None)), "FX_E_INVALID"),
                         (dict(r=dict(dtype=C["FX_DT_I64"])), "FX_E_UNSUPPORTED"), (dict(r=dict(tokens=-1)), "FX_E_INVALID"), (dict(r=dict(tokens=1 << 30)), "FX_E_LIMIT"),
                         (dict(t=dict(pairs=33)), "FX_E_INVALID"), (dict(t=dict(x=None)), "FX_E_INVALID"), (dict(t=dict(batch=2)), "FX_E_INVALID"), (dict(t=dict(back=1)), "FX_E_INVALID"),
                         (dict(t=dict(tokens=2)), "FX_E_INVALID"), (dict(t=dict(depth=128)), "FX_E_INVALID"), (dict(t=dict(dtype=C["FX_DT_F16"])), "FX_E_INVALID"),
                         (dict(t=dict(batch=0, tokens=3)), "FX_E_INVALID"), (dict(r=dict(tokens=1 << 28), t=dict(tokens=1 << 28)), "FX_E_LIMIT")):
        assert call(**change) == C[code], change
        assert b"fx_kv_append" in lib.fx_last_error()
    assert call(r=dict(tokens=0), t=dict(tokens=0)) == 0   # nothing to do
    assert lib.fx_kv_append(None, None, None, None) == C["FX_E_INVALID"]


# ---- GPU ----

@pytest.mark.gpu
@pytest.mark.parametrize("held", [E4M3, INT8])
@pytest.mark.parametrize("kind", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("P,H,G,D,turned", [(16, 3, 4, 64, 64), (64, 2, 1, 128, 128), (256, 1, 2, 16, 16), (32, 2, 3, 80, 80), (128, 1, 1, 256, 256), (64, 2, 2, 128, 64),
                                            (32, 1, 8, 48, 34), (16, 1, 1, 16, 2), (256, 2, 1, 96, 10), (64, 1, 5, 144, 144)])
def test_prompts_and_single_tokens(held, kind, interleaved, P, H, G, D, turned):
    cache = filled(9, H, P, D, held, 5)
    cache.k_scale[7] = math.nan                        # a page that nobody has used yet
    f, _ = rotary.frequencies(turned)
    order = [4, 7, 1, 2, 0, 8]
    first, second = 2 * P + P // 2 + 3, P + 1          # tokens of two requests
    at = lambda pages, lo, hi: [pages[p // P] * P + p % P for p in range(lo, hi)]  # noqa: E731
    steps = [(at(order[:4], 0, first) + at(order[4:], 0, second), list(range(first)) + list(range(second)))]
    steps += [(at(order[:4], first + i, first + i + 1) + at(order[4:], second + i, second + i + 1), [first + i, second + i]) for i in range(3)]
    steps += [(at(order[:4], first + 3, first + 8) + [-1, 9 * P, 2 ** 40] + at(order[4:], second + 3, second + 4), list(range(first + 3, first + 8)) + [-1, -1, 7, second + 3])]
    for i, (s, p) in enumerate(steps):
        slots, p = torch.tensor(s, dtype=torch.long), torch.tensor(p, dtype=torch.int64 if i % 2 else torch.int32).cuda()
        k, v = rows_of(kind, len(s), H, D, 7 * i + 1, strided=i % 2 == 1)
        q = queries(kind, len(s), H * G, D, i)
        fine = check(cache, q, k, v, slots.cuda(), p, f, 1.0 if i % 2 else 1.125, interleaved)
        # half a step of a code from the turned keys in 64 bits: 2^-4 of an e4m3 number (2^-10 of the scale below its least), half of int8's, and 2^-21 of the numbers that turned
        live = (slots >= 0) & (slots < 9 * P)
        want, size = plain(k, p, f, 1.0 if i % 2 else 1.125, interleaved)
        got = cache.read(slots.cuda(), torch.float32)[0].cpu().double()
        scale = cache.k_scale.cpu().double()[slots[live] // P][:, :, None]
        step = (want[live].abs() * 2.0 ** -4).clamp(min=2.0 ** -10 * scale) if held == E4M3 else 0.5 * scale
        assert bool(((got - want).abs()[live] <= step * (1 + 2.0 ** -20) + 2.0 ** -21 * size[live]).all())
        assert float((fine.cpu().double() - want).abs().max()) <= 2.0 ** -21 * float(size.max())


@pytest.mark.gpu
@pytest.mark.parametrize("held", [E4M3, INT8])
@pytest.mark.parametrize("kind", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("P,H,D,turned,interleaved", [(64, 1, 128, 128, False), (256, 1, 64, 64, True), (128, 2, 16, 16, False), (256, 1, 256, 256, False), (32, 2, 144, 100, True),
                                                      (128, 1, 80, 50, False), (256, 2, 48, 48, False)])
def test_long_runs(held, kind, P, H, D, turned, interleaved):
    """Runs that several waves share, larger numbers than before, infinities and NaN in one wave's part, a run in reverse, rows that are not aligned."""
    cache = filled(6, H, P, D, held, 7)
    f, _ = rotary.frequencies(turned)
    at = lambda page, lo, hi: list(range(page * P + lo, page * P + hi))  # noqa: E731
    steps = [(at(0, 0, 5) + at(1, 0, P) + at(2, 0, P // 2 + 3), 0.01, False), (at(0, 5, P) + at(2, P // 2 + 3, P - 1) + at(3, 0, 18), 3.0, False),
             (at(3, 18, P - 5 if P > 32 else P) + at(4, 0, 17), 0.1, True), (at(4, 17, P) + at(5, 0, P - 1)[::-1], 9.0, True), ([9, 9, 8, 70 % (6 * P)], 1.0, False)]
    for i, (slots, size, strange) in enumerate(steps):
        k, v = rows_of(kind, len(slots), H, D, 5 * i + 2, strided=i == 1)
        k, v = k * size, v * size
        if strange:
            for x, t in ((k, 1), (v, len(slots) - 2)):
                x[t, 0, 3], x[t, 0, 4], x[t // 2, 0, 5] = math.inf, math.nan, -math.inf
        p = torch.arange(len(slots), device="cuda") * 3 + 100 * i
        check(cache, queries(kind, len(slots), 3, D, i), k, v, torch.tensor(slots).cuda(), p, f, 1.0, interleaved)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,heads", [(3000, 8), (20000, 1)])
def test_many_tokens(tokens, heads):
    """Several workgroups a head, queries and keys and values out of one product; the positions of a plan, with rows behind the last token."""
    P, D, G = 64, 128, 4
    cache = filled(-(-tokens // P) + 4, heads, P, D, E4M3, 3)
    lens = [tokens // 3, 1, tokens - tokens // 3 - 1]
    table = i32([list(range(40)) + [-1] * 400] * 3)
    table.fill_(-1)
    step = cache.plan(i32([0, 0, 0]), i32(lens), table, torch.randperm(-(-tokens // P) + 3, generator=torch.Generator().manual_seed(1)).int().cuda(), tokens + 5)
    assert step.lens.tolist() == lens
    qkv = torch.randn(tokens + 5, (G + 2) * heads, D, generator=torch.Generator().manual_seed(2)).bfloat16().cuda()
    f, _ = rotary.frequencies(D)
    check(cache, qkv[:, :G * heads], qkv[:, G * heads:(G + 1) * heads], qkv[:, (G + 1) * heads:], step.slots, step.positions, f)


@pytest.mark.gpu
def test_the_cache_of_the_views_that_kv_store_takes():
    """Pages apart, a part of a wider cache, k and v with a stride in the depth, expanded heads, frequencies in fp32, no tokens."""
    wide = filled(6, 4, 16, 32, INT8, 4)
    cache = KvCache(wide.k[1:, 1:3], wide.v[1:, 1:3], wide.k_scale[1:, 1:3], wide.v_scale[1:, 1:3])
    f, _ = rotary.frequencies(32)
    x = torch.randn(20, 2, 64, generator=torch.Generator().manual_seed(1)).cuda()
    slots = torch.arange(3, 23).cuda()
    p = torch.arange(40, device="cuda")[::2]
    check(cache, x[..., ::2], x[..., 1::2], x[:, :1, :32].expand(20, 2, 32), slots, p, f.float())
    before = copied(cache)
    assert cache.append(x[:0, :, :32], x[:0, :, :32], x[:0, :, :32], slots[:0], p[:0], f).shape == (0, 2, 32)
    same_cache(cache, before)


@pytest.mark.gpu
def test_refusals():
    c = filled(2, 2, 16, 32, E4M3, 1)
    f, _ = rotary.frequencies(32)
    x, n = torch.zeros(3, 2, 32, device="cuda"), torch.arange(3, device="cuda")
    ok = dict(q=x, k=x, v=x, slots=n, positions=n, frequencies=f)
    for change, word in ((dict(q=x[:2]), "q must be"), (dict(q=x[:, :0]), "q must be"), (dict(q=x[..., :16]), "q must be"), (dict(q=x.half()), "one type"), (dict(v=x.half()), "one type"),
                         (dict(k=x[:, :1]), "k must be"), (dict(q=x.double(), k=x.double(), v=x.double()), "float32, float16 or bfloat16"), (dict(slots=n.int()), "slots must be"),
                         (dict(positions=n[:2]), "positions must be"), (dict(positions=n[:, None]), "positions must be"), (dict(positions=n.float()), "int32 or int64"),
                         (dict(positions=n.cpu()), "GPU only"), (dict(frequencies=f.cpu()), "GPU only"), (dict(frequencies=f.half()), "float64 or float32"),
                         (dict(frequencies=torch.ones(17, device="cuda")), "pairs"), (dict(magnitude=math.nan), "finite"), (dict(q=x.clone().requires_grad_()), "no backward pass"),
                         (dict(k=x.clone().requires_grad_()), "no backward pass"), (dict(frequencies=f.clone().requires_grad_()), "no backward pass")):
        with pytest.raises(RuntimeError, match=word):
            c.append(**{**ok, **change})


@pytest.mark.gpu
def test_a_captured_call_serves_other_tokens():
    P, H, G, D = 16, 2, 3, 64
    f, _ = rotary.frequencies(D)
    cache = filled(8, H, P, D, E4M3, 2)
    k, v = (t.clone() for t in rows_of(torch.bfloat16, 5, H, D, 1))
    q = queries(torch.bfloat16, 5, G * H, D, 2)
    slots, p = torch.arange(5).cuda(), torch.arange(5).int().cuda()
    eager = copied(cache)
    eager.append(q, k, v, slots, p, f)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cache.append(q, k, v, slots, p, f)
    graph.replay()
    torch.cuda.synchronize()
    same_cache(cache, eager)
    for i in range(3):
        nk, nv = rows_of(torch.bfloat16, 5, H, D, 10 + i)
        k.copy_(nk), v.copy_(nv), slots.copy_(torch.tensor([5 + i, 40 + i, 16, 17, -1])), p.copy_(torch.tensor([5 + i, 300, 0, 1, -1]))
        want = eager.append(q, k, v, slots, p, f)
        graph.replay()
        torch.cuda.synchronize()
        same_cache(cache, eager)
        assert torch.equal(out, want)


@pytest.mark.gpu
def test_one_launch():
    total, special = ctypes.c_uint64(), ctypes.c_uint64()
    c, f, x, n = filled(2, 2, 16, 32, E4M3, 1), rotary.frequencies(32)[0], torch.zeros(3, 2, 32, device="cuda"), torch.arange(3, device="cuda")
    lib.fx_launch_stats(ctypes.byref(total), ctypes.byref(special))
    before = total.value
    c.append(x, x, x, n, n, f)
    lib.fx_launch_stats(ctypes.byref(total), ctypes.byref(special))
    assert total.value == before + 1


@pytest.mark.gpu
def test_rows_that_are_negative_lazily():
    P, H, D = 16, 2, 32
    f, _ = rotary.frequencies(D)
    cache = filled(4, H, P, D, INT8, 2)
    other = copied(cache)
    q, k, v = (torch.view_as_complex(torch.randn(7, H, D, 2, generator=torch.Generator().manual_seed(i)).cuda()).conj().imag for i in range(3))
    packed = [torch._neg_view(t.resolve_neg().neg().contiguous()) for t in (q, k, v)]   # the same numbers, side by side
    assert all(t.is_neg() for t in (q, k, v, *packed))
    p = torch.arange(7, device="cuda")
    want = cache.append(*(t.resolve_neg().contiguous() for t in (q, k, v)), p, p, f)
    for rows, turn in (((q, k, v), f), (packed, f), (packed, torch._neg_view(f.neg()))):
        again = copied(other)
        assert torch.equal(again.append(*rows, p, p, turn), want)
        same_cache(again, cache)
