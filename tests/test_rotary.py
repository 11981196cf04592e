"""Rotary positions (functs::rotary, functs_amd/rotary.py, functs_amd/csrc/fxhip/fx_rotary*).

CPU: frequencies and refusals.  GPU: the operator and its gradient against complex numbers in 64 bits.

Tolerances: an angle is off by |p| f 2^-52 (two roundings of 64 bits, of the angle and of 2 / pi), its cosine and sine by 2^-23 of 1, the magnitude's
and two products' roundings by 2^-24 each of |a| + |b|: 4 * 2^-24 m (|a| + |b|) in all is more than that, and half a step of the result."""
import ctypes
import math

import pytest
import torch

import functs_amd.jit as fj  # noqa: F401
from functs_amd import _lib, rotary
from functs_amd._lib import C, FxError, lib

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def plain(x, positions, frequencies, magnitude=1.0, interleaved=False, back=False):
    """In 64 bits on the CPU: the result, and |a| + |b| of each number's pair (the number itself where nothing turns)."""
    x, f = x.detach().cpu().double(), frequencies.detach().cpu().double()
    n = 2 * f.numel()
    angle = positions.cpu().double().unsqueeze(-1) * f
    z = magnitude * torch.complex(angle.cos(), -angle.sin() if back else angle.sin()).unsqueeze(-2)
    a, b = (x[..., 0:n:2], x[..., 1:n:2]) if interleaved else (x[..., :n // 2], x[..., n // 2:n])
    w = torch.complex(a, b) * z
    size = (a.abs() + b.abs()) * abs(magnitude)
    both = lambda u, v: torch.stack([u, v], -1).flatten(-2) if interleaved else torch.cat([u, v], -1)  # noqa: E731
    return torch.cat([both(w.real, w.imag), x[..., n:]], -1), torch.cat([both(size, size), x[..., n:].abs() * 0], -1)


def check(got, x, positions, frequencies, magnitude=1.0, interleaved=False, back=False):
    want, size = plain(x, positions, frequencies, magnitude, interleaved, back)
    assert got.dtype == x.dtype and got.shape == x.shape
    got = got.detach().cpu().double()
    off = 4 * 2.0 ** -24 * size + torch.finfo(x.dtype).eps / 2 * (want.abs() + 2.0 ** -22 * size) + torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps
    bad = (got - want).abs() > off
    assert not bool(bad.any()), (int(bad.sum()), float(((got - want).abs() - off).max()))
    assert torch.equal(got[..., 2 * frequencies.numel():], want[..., 2 * frequencies.numel():])   # columns that do not turn


def normal(*size, seed=0, dtype=torch.float32, device="cuda"):
    return torch.randn(*size, generator=torch.Generator().manual_seed(seed)).to(dtype).to(device)


# ---- CPU ----

def test_frequencies():
    f, m = rotary.frequencies(64, device="cpu")
    assert f.dtype == torch.float64 and m == 1.0
    assert torch.allclose(f, torch.tensor([10000.0 ** (-2 * i / 64) for i in range(32)], dtype=torch.float64), rtol=1e-15)
    g, m = rotary.frequencies(64, stretch=8.0, device="cpu")
    assert torch.equal(g, f / 8) and m == 1.0
    g, _ = rotary.frequencies(64, stretch=8.0, how="base", device="cpu")
    assert float(g[0]) == 1.0 and abs(float(g[-1] / f[-1]) * 8 - 1) < 1e-12 and bool((g[1:] < f[1:]).all())
    g, m = rotary.frequencies(64, stretch=8.0, how="parts", length=4096, device="cpu")
    turns = 4096 * f / (2 * math.pi)
    assert abs(m - (0.1 * math.log(8.0) + 1)) < 1e-15 and bool((g <= f).all()) and bool((g >= f / 8 * (1 - 1e-12)).all())
    assert torch.equal(g[turns > 2 * 32], f[turns > 2 * 32]) and torch.allclose(g[turns < 0.5], f[turns < 0.5] / 8, rtol=1e-12)
    g, m = rotary.frequencies(64, base=500000.0, stretch=8.0, how="bands", length=8192, fast=4.0, slow=1.0, device="cpu")
    f, _ = rotary.frequencies(64, base=500000.0, device="cpu")
    turns = 8192 * f / (2 * math.pi)
    assert m == 1.0 and torch.equal(g[turns >= 4], f[turns >= 4]) and torch.allclose(g[turns <= 1], f[turns <= 1] / 8, rtol=1e-14)
    mid = (turns > 1) & (turns < 4)
    assert bool(mid.any()) and bool(((g < f) & (g > f / 8))[mid].all())


@pytest.mark.parametrize("bad", [dict(columns=0), dict(columns=7), dict(columns=64, how="other"), dict(columns=64, stretch=0.5), dict(columns=64, base=1.0),
                                 dict(columns=64, base=math.nan), dict(columns=64, fast=1.0, slow=2.0), dict(columns=64, length=0), dict(columns=2, stretch=2.0, how="base")])
def test_frequencies_that_make_no_sense(bad):
    with pytest.raises(FxError):
        rotary.frequencies(**bad, device="cpu")


def test_tensors_on_the_host_are_refused():
    f, _ = rotary.frequencies(16, device="cpu")
    with pytest.raises(RuntimeError, match="runs on the GPU only"):
        rotary.rotary(torch.zeros(3, 2, 16), torch.arange(3), f)


class Desc(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("x", "y", "positions", "frequencies")] + \
               [(n, ctypes.c_int64) for n in ("xb", "xt", "xh", "yb", "yt", "yh", "pb")] + \
               [(n, ctypes.c_int32) for n in ("batch", "tokens", "heads", "depth", "pairs", "dtype", "positions_64", "frequencies_32", "interleaved", "back")] + \
               [("magnitude", ctypes.c_float), ("reserved", ctypes.c_int32)]


def test_the_c_abi_refuses_before_it_launches():
    at = 4096   # never read: each call returns from its checks
    ok = dict(x=at, y=at, positions=at, frequencies=at, xt=64, xh=16, yt=64, yh=16, batch=1, tokens=3, heads=4, depth=16, pairs=8, dtype=C["FX_DT_BF16"], magnitude=1.0)
    for change, code in ((dict(dtype=C["FX_DT_I64"]), "FX_E_UNSUPPORTED"), (dict(pairs=9), "FX_E_INVALID"), (dict(pairs=0), "FX_E_INVALID"), (dict(heads=0), "FX_E_INVALID"),
                         (dict(tokens=-1), "FX_E_INVALID"), (dict(batch=-1), "FX_E_INVALID"), (dict(x=None), "FX_E_INVALID"), (dict(frequencies=None), "FX_E_INVALID"),
                         (dict(depth=5000, pairs=2049), "FX_E_UNSUPPORTED"), (dict(heads=1 << 24), "FX_E_LIMIT"), (dict(tokens=1 << 30), "FX_E_LIMIT"),
                         (dict(batch=1 << 15, tokens=1 << 15), "FX_E_LIMIT"), (dict(heads=1 << 14, depth=256, pairs=128, tokens=1 << 20), "FX_E_LIMIT")):
        assert lib.fx_rotary(ctypes.byref(Desc(**{**ok, **change})), None) == C[code], change
        assert b"fx_rotary" in lib.fx_last_error()
    assert lib.fx_rotary(None, None) == C["FX_E_INVALID"]
    for change in (dict(tokens=0), dict(batch=0), dict(tokens=0, x=None, y=None, positions=None)):
        assert lib.fx_rotary(ctypes.byref(Desc(**{**ok, **change})), None) == 0   # nothing to do


def test_the_schema_writes_to_nothing():
    schema = torch.ops.functs.rotary.default._schema
    assert not any(a.alias_info is not None and a.alias_info.is_write for a in schema.arguments)


# ---- GPU ----

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,depth,turned", [(1, 1, 2, 2), (1, 12, 64, 64), (61, 40, 128, 128), (5, 3, 80, 80), (7, 5, 100, 100), (33, 2, 72, 30),
                                                       (9, 1, 7, 4), (3, 7, 256, 64), (130, 1, 96, 96), (700, 6, 64, 34), (2, 70, 128, 126), (4, 2, 20, 18),
                                                       (3, 1, 9, 8), (1100, 3, 33, 16)])
def test_forward_and_backward(tokens, heads, depth, turned, interleaved, dtype):
    f, _ = rotary.frequencies(turned)
    x, g = normal(tokens, heads, depth, seed=1, dtype=dtype), normal(tokens, heads, depth, seed=2, dtype=dtype)
    p = torch.randint(-3, 5000, (tokens,), generator=torch.Generator().manual_seed(3)).int().cuda()
    x.requires_grad_()
    y = rotary.rotary(x, p, f, 1.25, interleaved)
    check(y, x, p, f, 1.25, interleaved)
    y.backward(g)
    check(x.grad, g, p, f, 1.25, interleaved, back=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("f32", [False, True])
def test_far_positions(dtype, f32):
    """Angles up to 2^31: off by 2^31 * 2^-52 = 2^-21, which the tolerance of fp32 does not hold; so far positions are compared with that added."""
    f, _ = rotary.frequencies(32)
    f = f.float() if f32 else f
    p = torch.tensor([0, 1, -1, 131071, 1 << 20, 16777217, -16777219, (1 << 31) - 1, -(1 << 31)], dtype=dtype).cuda()
    x = normal(p.numel(), 2, 32, seed=4)
    y = rotary.rotary(x, p, f)
    near = p.abs().long() <= 1 << 20
    check(y[near], x[near], p[near], f)
    want, size = plain(x, p, f)
    assert bool(((y.cpu().double() - want).abs() <= (4 * 2.0 ** -24 + 2.0 ** -20) * size + 2.0 ** -24 * want.abs()).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_batches_views_and_orders(dtype):
    B, S, H, D = 3, 37, 4, 48
    f, _ = rotary.frequencies(48)
    each = torch.randint(0, 3000, (B, S + 2), generator=torch.Generator().manual_seed(5)).cuda()
    x = normal(B, S, 3 * H, D + 8, seed=6, dtype=dtype)
    for t in (x[:, :, :H, :D], x[:, :, H:2 * H, 5:5 + D], x[:, :, :H, :D].transpose(1, 2).contiguous().transpose(1, 2), x[:, ::2, :H, :D], x[:1, :, :H, :D].expand(B, S, H, D),
              x[:, :, :1, :D].expand(B, S, H, D), x[..., :H, ::1][..., :D].transpose(2, 3).contiguous().transpose(2, 3), x[:, :, :H, :2 * (D // 2)].neg()):
        n = t.size(1)
        for p in (each[0, :n], each[:, 1:n + 1], each[:, :n].int(), each[:1, :n].expand(B, n), each.t().contiguous().t()[:, :n]):
            check(rotary.rotary(t, p, f), t, p, f)
    t = x[:, :, :H, :D].transpose(1, 2).contiguous().transpose(1, 2)
    assert rotary.rotary(t, each[0, :S], f).stride() == t.stride()         # an order of dimensions is kept
    assert rotary.rotary(x[:, :, :H, :D], each[0, :S], f).is_contiguous()  # a part of something wider becomes whole
    z = torch.view_as_complex(normal(5, 2, 16, 2, seed=7)).conj().imag      # lazily negative
    assert z.is_neg()
    f, _ = rotary.frequencies(16)
    check(rotary.rotary(z, each[0, :5], f), z.resolve_neg(), each[0, :5], f)


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
def test_gradients_of_broadcast_inputs_and_of_gradients(interleaved):
    f, _ = rotary.frequencies(12)
    p = torch.arange(5).cuda()
    one = normal(1, 1, 3, 16, seed=8).requires_grad_()
    y = rotary.rotary(one.expand(2, 5, 3, 16), p, f, 0.5, interleaved)
    g = normal(2, 5, 3, 16, seed=9)
    y.backward(g)
    want, size = plain(g, p, f, 0.5, interleaved, back=True)
    off = (want.sum((0, 1), keepdim=True) - one.grad.cpu().double()).abs()
    assert bool((off <= 2.0 ** -20 * (size + want.abs()).sum((0, 1), keepdim=True)).all())   # ten terms of 4 * 2^-24, and their sum's roundings
    # a sum's gradient has strides of 0; a second derivative
    x = normal(5, 3, 16, seed=10).requires_grad_()
    (d,) = torch.autograd.grad(rotary.rotary(x, p, f, 0.5, interleaved).sum(), x)
    check(d, torch.ones(5, 3, 16), p, f, 0.5, interleaved, back=True)
    w = normal(5, 3, 16, seed=11).requires_grad_()
    (d,) = torch.autograd.grad(rotary.rotary(x, p, f, 0.5, interleaved), x, w, create_graph=True)
    v = normal(5, 3, 16, seed=12)
    (e,) = torch.autograd.grad(d, w, v)
    check(e, v, p, f, 0.5, interleaved)


@pytest.mark.gpu
def test_the_gradient_against_differences():
    """The operator is linear, so a difference over any step is the derivative, but for roundings: 2 * 4 * 2^-24 of sums of up to 16 numbers of size 4."""
    f, _ = rotary.frequencies(8)
    p = torch.tensor([3, 1000]).cuda()
    x, g = normal(2, 1, 10, seed=13).requires_grad_(), normal(2, 1, 10, seed=14)
    rotary.rotary(x, p, f, 1.5).backward(g)
    for i in range(2):
        for c in range(10):
            e = torch.zeros(2, 1, 10, device="cuda")
            e[i, 0, c] = 1.0
            up, down = rotary.rotary(x.detach() + e, p, f, 1.5), rotary.rotary(x.detach() - e, p, f, 1.5)
            slope = float(((up.double() - down.double()) * g.double()).sum()) / 2
            assert abs(slope - float(x.grad[i, 0, c])) <= 16 * 8 * 2.0 ** -24 * 16


@pytest.mark.gpu
def test_infinities_and_nan_stay_where_they_are():
    f, _ = rotary.frequencies(16)
    x = normal(3, 2, 24, seed=15)
    p = torch.arange(3).cuda()
    was = rotary.rotary(x, p, f)
    x[1, 0, 3], x[2, 1, 20] = math.nan, math.inf
    y = rotary.rotary(x, p, f)
    touched = torch.zeros(3, 2, 24, dtype=torch.bool, device="cuda")
    touched[1, 0, [3, 11]] = True
    assert bool(torch.isnan(y[touched]).all()) and float(y[2, 1, 20]) == math.inf
    touched[2, 1, 20] = True
    assert torch.equal(y[~touched], was[~touched])


@pytest.mark.gpu
def test_nothing_to_turn():
    f, _ = rotary.frequencies(16)
    for shape, p in (((0, 2, 16), torch.zeros(0)), ((2, 0, 3, 16), torch.zeros(0)), ((0, 4, 3, 16), torch.zeros(4))):
        x = torch.zeros(shape, device="cuda", requires_grad=True)
        y = rotary.rotary(x, p.int().cuda(), f)
        assert y.shape == x.shape
        y.sum().backward()
        assert x.grad.shape == x.shape


@pytest.mark.gpu
def test_refusals():
    f, _ = rotary.frequencies(16)
    x, p = torch.zeros(3, 2, 16, device="cuda"), torch.arange(3).cuda()
    for call, word in ((lambda: rotary.rotary(x.double(), p, f), "float32, float16 or bfloat16"), (lambda: rotary.rotary(x[0], p, f), "must be"),
                       (lambda: rotary.rotary(x[:, :0], p, f), "must be"), (lambda: rotary.rotary(x, p[:2], f), "positions must be"), (lambda: rotary.rotary(x, p.float(), f), "int32 or int64"),
                       (lambda: rotary.rotary(x[None], p.expand(2, 3), f), "positions must be"), (lambda: rotary.rotary(x, p[None], f), "positions must be"),
                       (lambda: rotary.rotary(x, p.cpu(), f), "runs on the GPU only"), (lambda: rotary.rotary(x, p, f.cpu()), "runs on the GPU only"),
                       (lambda: rotary.rotary(x, p, f.half()), "float64 or float32"), (lambda: rotary.rotary(x, p, f[None]), "float64 or float32"),
                       (lambda: rotary.rotary(x, p, f[:0]), "pairs"), (lambda: rotary.rotary(x[..., :14], p, f), "pairs"),
                       (lambda: rotary.rotary(x, p, f, math.inf), "finite"), (lambda: rotary.rotary(x, p, f, math.nan), "finite"), (lambda: rotary.rotary(x, p, f, 1e39), "finite"),
                       (lambda: rotary.rotary(x, p, f.clone().requires_grad_()), "no backward pass")):
        with pytest.raises(RuntimeError, match=word):
            call()
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level(), pytest.raises(RuntimeError, match="tangent"):
        rotary.rotary(fwd.make_dual(x, x), p, f)


@pytest.mark.gpu
def test_positions_that_change_before_the_backward_pass_are_noticed():
    f, _ = rotary.frequencies(16)
    x, p = normal(3, 2, 16, seed=16).requires_grad_(), torch.arange(3).cuda()
    y = rotary.rotary(x, p, f)
    p += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


@pytest.mark.gpu
def test_a_scripted_call():
    def program(x: torch.Tensor, p: torch.Tensor, f: torch.Tensor):
        y = torch.ops.functs.rotary(x, p, f)
        return torch.ops.functs.rotary(y, -p, f)

    f, _ = rotary.frequencies(64)
    x, p = normal(19, 4, 64, seed=17), torch.arange(19).cuda()
    back = torch.jit.script(program)(x, p, f)
    assert bool(((back - x).abs() <= 2.0 ** -20 * (x[..., :32].abs() + x[..., 32:].abs()).repeat(1, 1, 2)).all())


@pytest.mark.gpu
def test_two_streams_and_captured_calls():
    f, _ = rotary.frequencies(128)
    x, p = normal(61, 8, 128, seed=18, dtype=torch.bfloat16), torch.arange(61).int().cuda()
    want = rotary.rotary(x, p, f)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got += [rotary.rotary(x, p, f) for _ in range(5)]
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)
    # forward and backward captured, replayed on other numbers
    leaf, g = x.clone().requires_grad_(), normal(61, 8, 128, seed=19, dtype=torch.bfloat16)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = rotary.rotary(leaf, p, f)
        (d,) = torch.autograd.grad(y, leaf, g)
    for seed in (20, 21, 22):
        with torch.no_grad():
            leaf.copy_(normal(61, 8, 128, seed=seed, dtype=torch.bfloat16))
        p.copy_(torch.randint(0, 9000, (61,), generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        eager = rotary.rotary(leaf.detach(), p, f)
        torch.cuda.synchronize()
        assert torch.equal(y, eager)
        check(y, leaf, p, f)
        check(d, g, p, f, back=True)


@pytest.mark.gpu
def test_a_capture_beside_a_living_graph_of_the_leaf_is_refused():
    f, _ = rotary.frequencies(16)
    x, p = normal(3, 2, 16, seed=23).requires_grad_(), torch.arange(3).cuda()
    alive = rotary.rotary(x, p, f)
    graph, said = torch.cuda.CUDAGraph(), ""
    with torch.cuda.graph(graph):
        torch.zeros(1, device="cuda")
        try:
            rotary.rotary(x, p, f)
        except RuntimeError as e:
            said = str(e)
    assert "drop its results" in said
    del alive
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        y = rotary.rotary(x, p, f)
    assert y.shape == x.shape


@pytest.mark.gpu
def test_more_than_two_to_the_31_numbers():
    """Offsets beyond 32 bits: rows far apart in memory."""
    f, _ = rotary.frequencies(8)
    wide = torch.empty(3, (1 << 30) + 8, dtype=torch.float16, device="cuda")
    x = wide[:, -8:].unflatten(1, (1, 8))
    x.copy_(normal(3, 1, 8, seed=24))
    p = torch.tensor([1, 20, 300]).cuda()
    check(rotary.rotary(x, p, f), x, p, f)


@pytest.mark.gpu
def test_every_launch_is_counted():
    total, special = ctypes.c_uint64(), ctypes.c_uint64()
    f, _ = rotary.frequencies(16)
    x, p = normal(3, 2, 16), torch.arange(3).cuda()
    lib.fx_launch_stats(ctypes.byref(total), ctypes.byref(special))
    before = total.value
    rotary.rotary(x, p, f)
    lib.fx_launch_stats(ctypes.byref(total), ctypes.byref(special))
    assert total.value == before + 1


@pytest.mark.gpu
def test_a_captured_backward_pass_to_a_leaf_of_a_living_graph_is_refused():
    """Through views of the leaf, which are no leaves: the pass is refused where it would come to the leaf, and only there."""
    f, _ = rotary.frequencies(16)
    x, p, g = normal(3, 4, 16, seed=25).requires_grad_(), torch.arange(3).cuda(), normal(3, 2, 16, seed=26)
    alive = rotary.rotary(x[:, :2], p, f)
    graph, said = torch.cuda.CUDAGraph(), ""
    with torch.cuda.graph(graph):
        y = rotary.rotary(x[:, 2:], p, f)
        try:
            torch.autograd.grad(y, x, g)
        except RuntimeError as e:
            said = str(e)
    assert "drop its results" in said
    graph.replay()
    check(y, x[:, 2:], p, f)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        part = x[:, 2:]
        y = rotary.rotary(part, p, f)
        (d,) = torch.autograd.grad(y, part, g)   # (does not come to the leaf)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        check(y, x[:, 2:], p, f)
        check(d, g, p, f, back=True)
    del alive, y, part
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        (d,) = torch.autograd.grad(rotary.rotary(x[:, 2:], p, f), x, g)
    for seed in (27, 28, 29):
        g.copy_(normal(3, 2, 16, seed=seed))
        graph.replay()
        torch.cuda.synchronize()
        check(d[:, 2:], g, p, f, back=True)
        assert not bool(d[:, :2].any())
