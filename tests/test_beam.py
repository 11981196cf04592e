"""A beam search's selection (functs::beam_select, functs_amd/beam.py, functs_amd/csrc/fxhip/fx_beam*).

CPU: refusals.  GPU: the operator against a plain selection in 64 bits.

Words and beams have to be equal wherever the totals that decide are further apart than the kernel's are off.  A term is 2 to the power of x c - r, c being log2 e in fp32
(1.3e-8 too large) and r the whole number next to the largest x c: a product and a difference rounded once, by half a step of the result, which is about (x - top) c.
From tops of 2^22 on it is (x - top) c itself, an exact difference and a rounded product.  So it is off by 2^-24 |x - top| c + 1.3e-8 |x - top| + 2^-23 (the power's own
rounding) of itself: with x - top of 30, beyond which no term matters, 2^-18 at most, and far less in their sum.  2^-18 in all; a total is rounded to fp32 once."""
import ctypes
import math

import pytest
import torch

import functs_amd.jit as fj  # noqa: F401
from functs_amd import beam
from functs_amd._lib import C, lib

TYPES = [torch.float32, torch.bfloat16, torch.float16]
OFF = 2.0 ** -18


def plain(logits, scores, count, ended=None, end=-1):
    """Of each request: (total, beam, word) of the candidates, best first, by the rules of include/fxhip.h in 64 bits."""
    logits, scores = logits.cpu().double(), scores.cpu().double()
    B, K, V = logits.shape
    answer = []
    for b in range(B):
        found = []
        for k in range(K):
            s = float(scores[b, k])
            if not s > -math.inf:
                continue
            if ended is not None and bool(ended[b, k]):
                found.append((s, k, 0.0, end))
                continue
            x = logits[b, k]
            top = float(x.max())
            if bool(torch.isnan(x).any()) or not math.isfinite(top):
                continue
            lse = float((x - top).exp().sum().log()) + top
            best = torch.sort(x, descending=True, stable=True)
            for i in range(min(count, V)):
                if float(best.values[i]) > -math.inf:
                    found.append((s + (float(best.values[i]) - lse), k, float(best.values[i]), int(best.indices[i])))
        found.sort(key=lambda f: (-f[0], f[1], -f[2], f[3]))
        answer.append(found)
    return answer


def check(logits, scores, count=0, ended=None, end=-1):
    got = beam.select(logits, scores, count, ended, end)
    count = count or logits.size(1)
    want = plain(logits, scores, count, ended, end)
    B = logits.size(0)
    assert got.scores.shape == got.beams.shape == got.words.shape == (B, count)
    assert got.scores.dtype == torch.float32 and got.beams.dtype == torch.int32 and got.words.dtype == torch.int64
    s, k, w = got.scores.tolist(), got.beams.tolist(), got.words.tolist()
    swaps = 0
    for b in range(B):
        n = min(count, len(want[b]))
        for i in range(count):
            if i >= n:
                assert (s[b][i], k[b][i], w[b][i]) == (-math.inf, -1, -1), (b, i)
                continue
            total, beam_, _, word = want[b][i]
            assert abs(s[b][i] - total) <= OFF + 2.0 ** -23 * abs(total), (b, i, s[b][i], total)
            if (k[b][i], w[b][i]) != (beam_, word):   # only candidates of other beams that are as near
                near = [f for f in want[b] if abs(f[0] - total) <= 2 * OFF]
                assert (k[b][i], w[b][i]) in [(f[1], f[3]) for f in near] and len({f[1] for f in near}) > 1, (b, i, k[b][i], w[b][i], want[b][i])
                swaps += 1
        for i in range(1, n):
            assert s[b][i] <= s[b][i - 1]
    assert swaps <= 2
    return got


def logits_of(B, K, V, seed, dtype=torch.float32, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, K, V, generator=g) * spread
    s = torch.randn(B, K, generator=g) * 2 - 20
    return x.to(dtype).cuda(), s.cuda()


# ---- CPU ----

def test_tensors_on_the_host_are_refused():
    with pytest.raises(RuntimeError, match="runs on the GPU only"):
        beam.select(torch.zeros(1, 2, 5), torch.zeros(1, 2))


def test_the_schema_writes_to_nothing():
    assert not any(a.alias_info is not None and a.alias_info.is_write for a in torch.ops.functs.beam_select.default._schema.arguments)


def test_scores_to_start_with():
    assert beam.first_scores(2, 3, "cpu").tolist() == [[0.0, -math.inf, -math.inf]] * 2


class Desc(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("logits", "scores", "ended")] + [(n, ctypes.c_int64) for n in ("rs", "bs", "end")] + \
               [(n, ctypes.c_void_p) for n in ("out_scores", "out_beams", "out_words")] + \
               [(n, ctypes.c_int32) for n in ("requests", "beams", "words", "count", "dtype", "reserved")] + [("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_size_t)]


def test_the_c_abi_refuses_before_it_launches():
    at = 4096   # never read: each call returns from its checks
    ok = dict(logits=at, scores=at, rs=40, bs=10, out_scores=at, out_beams=at, out_words=at, requests=2, beams=4, words=10, count=4, dtype=C["FX_DT_BF16"], workspace=at,
              workspace_bytes=1 << 30)
    lib.fx_beam_select_workspace_bytes.restype = ctypes.c_size_t
    for change, code in ((dict(dtype=C["FX_DT_I64"]), "FX_E_UNSUPPORTED"), (dict(beams=0), "FX_E_UNSUPPORTED"), (dict(beams=33), "FX_E_UNSUPPORTED"), (dict(count=0), "FX_E_UNSUPPORTED"),
                         (dict(count=65), "FX_E_UNSUPPORTED"), (dict(words=0), "FX_E_UNSUPPORTED"), (dict(words=262145), "FX_E_UNSUPPORTED"), (dict(requests=-1), "FX_E_INVALID"),
                         (dict(logits=None), "FX_E_INVALID"), (dict(scores=None), "FX_E_INVALID"), (dict(out_words=None), "FX_E_INVALID"), (dict(workspace=None), "FX_E_INVALID"),
                         (dict(workspace=at + 8), "FX_E_INVALID"), (dict(workspace_bytes=15), "FX_E_INVALID"), (dict(requests=1 << 22), "FX_E_LIMIT"),
                         (dict(requests=1 << 21, beams=32), "FX_E_LIMIT")):
        d = Desc(**{**ok, **change})
        assert lib.fx_beam_select(ctypes.byref(d), None) == C[code], change
        assert b"fx_beam_select" in lib.fx_last_error()
        if code in ("FX_E_UNSUPPORTED", "FX_E_LIMIT"):
            assert lib.fx_beam_select_workspace_bytes(ctypes.byref(d)) == 0
    assert lib.fx_beam_select(None, None) == C["FX_E_INVALID"] and lib.fx_beam_select_workspace_bytes(None) == 0
    assert lib.fx_beam_select(ctypes.byref(Desc(**{**ok, "requests": 0})), None) == 0   # nothing to do
    # each 256 loads of 16 bytes of a row: 16 bytes, and 4 for each of 8 segments
    for words, dtype, parts in ((10, "FX_DT_BF16", 1), (2049, "FX_DT_BF16", 2), (131072, "FX_DT_F16", 64), (131073, "FX_DT_F16", 65), (262144, "FX_DT_F32", 256), (1025, "FX_DT_F32", 2)):
        d = Desc(**{**ok, "words": words, "dtype": C[dtype]})
        assert lib.fx_beam_select_workspace_bytes(ctypes.byref(d)) == 8 * parts * (16 + 4 * 8)


# ---- GPU ----

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,K,V,count", [(1, 1, 1, 1), (1, 4, 3, 4), (2, 3, 7, 64), (3, 2, 8, 5), (1, 4, 33, 8), (2, 5, 511, 5), (1, 1, 2048, 64), (3, 4, 2049, 4), (2, 8, 5003, 16),
                                         (1, 32, 1025, 64), (1, 16, 32000, 16), (4, 2, 50001, 2), (1, 3, 70001, 33), (1, 2, 131073, 7), (1, 2, 262144, 64), (40, 4, 1000, 8), (130, 1, 257, 3)])
def test_select(B, K, V, count, dtype):
    x, s = logits_of(B, K, V, V + K, dtype)
    check(x, s, count)
    check(x, s, count, spread_ended(B, K), V - 1)


def spread_ended(B, K):
    return (torch.arange(B * K).view(B, K) % 3 == 1).cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [300, 2100])
def test_many_rows(rows, dtype):
    """More rows than the shorter parts are for: longer ones, whose last is not whole."""
    V = 8192 + 5 if dtype != torch.float32 else 4096 + 3
    x, s = logits_of(rows, 4, V, 1, dtype)
    got = beam.select(x, s, 4)
    some = torch.tensor([0, 1, rows // 2, rows - 1]).cuda()
    check(x[some], s[some], 4)
    alone = beam.select(x[some], s[some], 4)                                  # (parts of another size: lse differs in its last bits)
    assert torch.equal(got.words[some], alone.words) and torch.equal(got.beams[some], alone.beams)
    assert float((got.scores[some] - alone.scores).abs().max()) <= OFF + 2.0 ** -23 * 60


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [9, 64, 2048, 2500, 20000])
def test_equal_logits(V, dtype):
    """Lower words go first, and beams whose rows and scores are equal in their order; as many equal words as there may be."""
    for x in (torch.zeros(2, 3, V), torch.full((2, 3, V), -7.5), (torch.arange(V) % 2).float().expand(2, 3, V).clone(), (torch.arange(V) // (V // 2 + 1)).float().expand(2, 3, V).clone(),
              torch.where(torch.arange(V) % 3 == 0, 0.0, -0.0).expand(2, 3, V).clone(), torch.arange(V).float().flip(0).clamp(max=300.0).expand(2, 3, V).clone(),
              torch.arange(V).float().clamp(max=300.0).expand(2, 3, V).clone()):
        for count in (1, 5, 64):
            x, s = x.to(dtype).cuda(), torch.zeros(2, 3).cuda()
            got = check(x, s, count)
            one = torch.sort(x[0, 0].float(), descending=True, stable=True).indices[:count]
            mine = [w for w, k in zip(got.words[0].tolist(), got.beams[0].tolist()) if k == 0]
            assert got.beams[0].tolist()[0] == 0 and mine == one.tolist()[:len(mine)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_masked_words(dtype):
    x, s = logits_of(2, 3, 4099, 5, dtype)
    low = torch.finfo(dtype).min
    for value in (-math.inf, low):
        y = x.clone()
        y[0, 0, :] = value                       # nothing is left (all of the lowest value: all as likely)
        y[0, 1, 7:] = value                      # a few
        y[0, 2, :4098] = value                   # the last word
        y[1, 0, torch.randperm(4099)[:4000].cuda()] = value
        y[1, 1, 64:] = value
        check(y, s, 4)
        check(y, s, 64)
    y = torch.full_like(x, -math.inf)
    got = check(y, s, 3)
    assert got.beams.tolist() == [[-1] * 3] * 2
    y[1, 2, 4000] = 1.0
    got = check(y, s, 3)
    assert got.words.tolist() == [[-1] * 3, [4000, -1, -1]] and abs(float(got.scores[1, 0]) - float(s[1, 2])) <= 1e-6


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [50, 3000, 20000])
def test_rows_with_nan_and_infinity_have_no_candidates(V, dtype):
    x, s = logits_of(1, 5, V, 6, dtype)
    x[0, 1, V - 1], x[0, 2, 3], x[0, 3, :] = math.nan, math.inf, math.nan
    got = check(x, s, 8)
    assert set(got.beams[0].tolist()) <= {0, 4}
    s[0, 0], s[0, 4] = math.nan, -math.inf
    assert check(x, s, 8).beams[0].tolist() == [-1] * 8


@pytest.mark.gpu
def test_the_first_step_and_beams_at_their_end():
    x, _ = logits_of(3, 4, 1000, 7)
    s = beam.first_scores(3, 4)
    got = check(x, s, 4)
    assert got.beams.tolist() == [[0] * 4] * 3
    ended = torch.tensor([[True, False, False, True], [True] * 4, [False] * 4]).cuda()
    s = torch.tensor([[-1.0, -2.0, -30.0, -math.inf], [-4.0, -3.0, -3.0, -5.0], [-1.0, -1.0, -1.0, -1.0]]).cuda()
    x[0, 0] = math.nan                            # what has ended is not looked at
    got = check(x, s, 4, ended, 999)
    assert (int(got.beams[0, 0]), int(got.words[0, 0]), float(got.scores[0, 0])) == (0, 999, -1.0)
    assert got.beams[1].tolist() == [1, 2, 0, 3] and got.words[1].tolist() == [999] * 4 and got.scores[1].tolist() == [-3.0, -3.0, -4.0, -5.0]
    got = beam.select(x, s, 8, ended.to(torch.uint8), -100)
    assert got.words[1].tolist() == [-100] * 4 + [-1] * 4


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_far_apart_and_long_sums(dtype):
    """One word far above the others; thousands of equal ones (the sum of 262 144 terms); scores of any size."""
    V = 262144
    x = torch.zeros(1, 2, V)
    x[0, 0, 77] = 60.0
    check(x.to(dtype).cuda(), torch.tensor([[-1e4, -3.0]]).cuda(), 3)
    check(x.to(dtype).cuda(), torch.tensor([[0.0, 1e5]]).cuda(), 3)
    big = torch.finfo(dtype).max
    x[0, 1, :] = -big
    x[0, 1, V - 1] = big
    check(x.to(dtype).cuda(), torch.tensor([[0.0, -1.0]]).cuda(), 3)


@pytest.mark.gpu
def test_views():
    wide, s = logits_of(6, 8, 400, 8, torch.bfloat16)
    for x in (wide[::2, 1:5, 3:300], wide[:3, ::2, :], wide[:3, :4].transpose(0, 1)[:4].transpose(0, 1), wide[:3, :1].expand(3, 4, 400), wide[:3, :4, ::2],
              wide.transpose(1, 2)[:3, :4], wide[:3, :4, 399:]):
        check(x, s[:3, :4], 4)
    check(wide[:3, :4], s.t().contiguous().t()[:3, :4], 4, (s > 0)[:3, :4])
    for x in (wide[:0], wide[:0, :, :5]):
        assert beam.select(x, s[:0]).beams.shape == (0, 8)


@pytest.mark.gpu
def test_refusals():
    x, s = torch.zeros(2, 3, 10, device="cuda"), torch.zeros(2, 3, device="cuda")
    for call, word in ((lambda: beam.select(x[0], s), "logits must be"), (lambda: beam.select(x.double(), s), "float32, float16 or bfloat16"), (lambda: beam.select(x, s[:1]), "scores must be"),
                       (lambda: beam.select(x, s.half()), "scores must be"), (lambda: beam.select(x, s.cpu()), "GPU only"), (lambda: beam.select(x, s, -1), "count"),
                       (lambda: beam.select(x, s, 65), "continuations"), (lambda: beam.select(x[:, :0], s[:, :0], 1), "beams"), (lambda: beam.select(x[:, :, :0], s), "words"),
                       (lambda: beam.select(x[:, :1].expand(2, 33, 10), s[:, :1].expand(2, 33)), "beams"), (lambda: beam.select(x, s, 3, s), "ended must be"),
                       (lambda: beam.select(x[:, :, :1].expand(2, 3, 262145), s), "words"), (lambda: beam.select(x, s, 3, s.bool()[:1]), "ended must be"),
                       (lambda: beam.select(x, s, 3, s.bool().cpu()), "GPU only"), (lambda: beam.select(x.clone().requires_grad_(), s), "no backward pass"),
                       (lambda: beam.select(x, s.clone().requires_grad_()), "no backward pass")):
        with pytest.raises(RuntimeError, match=word):
            call()


@pytest.mark.gpu
def test_streams_captures_and_a_script():
    x, s = logits_of(5, 4, 6000, 9, torch.bfloat16)
    want = beam.select(x, s, 8)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for t in streams:
        with torch.cuda.stream(t):
            got += [beam.select(x, s, 8) for _ in range(4)]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    out = []
    for graph in graphs:
        with torch.cuda.graph(graph):
            out.append(beam.select(x, s, 8))
    for seed in (10, 11, 12):
        nx, ns = logits_of(5, 4, 6000, seed, torch.bfloat16)
        x.copy_(nx), s.copy_(ns)
        for graph in graphs:
            graph.replay()
        eager = beam.select(x, s, 8)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for o in out for a, b in zip(o, eager))

    def program(x: torch.Tensor, s: torch.Tensor):
        scores, beams, words = torch.ops.functs.beam_select(x, s, 8)
        return scores, beams, words

    assert all(torch.equal(a, b) for a, b in zip(torch.jit.script(program)(x, s), beam.select(x, s, 8)))


@pytest.mark.gpu
def test_rows_beyond_two_to_the_31_numbers():
    wide = torch.empty(3, 1, (1 << 30) + 64, dtype=torch.float16, device="cuda")
    x = wide[:, :, -50:]
    x.copy_(logits_of(3, 1, 50, 13)[0])
    check(x, torch.zeros(3, 1, device="cuda"), 5)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_two_launches(dtype):
    total, special = ctypes.c_uint64(), ctypes.c_uint64()
    part = 1024 if dtype == torch.float32 else 2048
    for V, n in ((10, 1), (part, 1), (part + 1, 2)):
        x, s = logits_of(2, 3, V, 1, dtype)
        lib.fx_launch_stats(ctypes.byref(total), ctypes.byref(special))
        before = total.value
        beam.select(x, s)
        lib.fx_launch_stats(ctypes.byref(total), ctypes.byref(special))
        assert total.value == before + n


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,K,V,count", [(5, 12, 2706, 24), (3, 11, 579, 22), (2, 17, 700, 64), (1, 16, 130, 9), (2, 9, 15000, 15), (59, 1, 978, 1), (2, 3, 700, 43), (1, 31, 4099, 5)])
def test_rows_of_few_segments_and_many_beams(B, K, V, count, dtype):
    x, s = logits_of(B, K, V, V + K, dtype)
    check(x, s, count)
    x[torch.rand(x.shape, generator=torch.Generator().manual_seed(V)).cuda() < 0.9] = -math.inf
    check(x, s, count, spread_ended(B, K), V - 1)


@pytest.mark.gpu
@pytest.mark.parametrize("K,count", [(4, 8), (13, 26), (32, 64), (3, 64)])
def test_beams_of_the_same_numbers_go_in_order(K, count):
    x, _ = logits_of(1, 1, 900, 6)
    got = beam.select(x.expand(1, K, 900).contiguous(), torch.zeros(1, K, device="cuda"), count)
    words = torch.sort(x[0, 0], descending=True, stable=True).indices
    assert got.beams[0].tolist() == [i % K for i in range(count)]
    assert got.words[0].tolist() == [int(words[i // K]) for i in range(count)]


# Numbers of any size.  A total is s + (x - lse) in 64 bits: lse of 1e10 has steps of 2^-19, one of which is within OFF; lse of 1e20 and more steps of 2^14 and more, in which
# log sum exp(x - top) <= log 262 144 < 13 is lost on either side.  (Sizes in between would need a tolerance of a step of theirs.)
SIZES = [1e9, 2e9, 5e9, 1e10, 1e20, 1e30, 2e30, 1e38]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [700, 8195])     # one part, and several, the last of which is a few words
@pytest.mark.parametrize("size", SIZES)
def test_finite_masks_of_any_size(size, V, dtype):
    part = min(1024 if dtype == torch.float32 else 2048, V // 3)
    x, s = logits_of(3, 3, V, 5, dtype)
    x[0, 0, part:2 * part] = -size              # one whole part, or a third of a row of one part
    x[0, 1, :] = -size                          # all but a part in the middle
    x[0, 1, part:2 * part] = logits_of(1, 1, part, 6, dtype)[0][0, 0]
    x[0, 2, :] = -size                          # nothing is left: all as likely
    x[1, 0, :V - 1] = -size                     # the last word
    x[1, 1, :] = torch.where(torch.arange(V).cuda() % 2 == 0, x[1, 1], -size)
    x[1, 2, 3:] = -size                         # a few
    x[2, :, :] = -size
    for count in (4, 64):
        got = check(x, s, count)
        assert bool((got.beams >= 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [700, 8195])
@pytest.mark.parametrize("size", SIZES)
def test_largest_words_of_any_size(size, V, dtype):
    x, s = logits_of(3, 3, V, 7, dtype)
    x[0, 0, V // 2] = size                      # a word above all others, of its row and of the other rows
    x[1, :, 5] = size
    x[2, 0, :] = size                           # a row of nothing else
    x[2, 1, V - 100:] = size
    for count in (1, 5):
        got = check(x, s, count)
        assert bool((got.beams >= 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("V", [700, 8195])
@pytest.mark.parametrize("sign", [-1.0, 1.0])
@pytest.mark.parametrize("middle", [2.0 ** 21, 2.0 ** 22, 2.0 ** 24, 2.0 ** 28])
def test_parts_on_both_sides_of_a_size(middle, sign, V):
    """Parts whose largest words are a little below and above a power of two, and rows of which one part alone is."""
    x, s = logits_of(2, 3, V, 8)
    step = torch.where(torch.arange(V).cuda() // 1024 % 2 == 0, -1.5, 1.5)
    x[0] = sign * middle + (x[0] + step) * max(1.0, middle * 2.0 ** -23)
    x[1, :, V // 2:] = sign * middle + x[1, :, V // 2:]
    check(x, s, 6)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V,count", [(900, 4), (8197, 4), (50001, 20)])
def test_rows_have_the_same_results_alone_and_among_many(V, count, dtype):
    """Parts go by type and number of words, so a row's sum does not depend on the rows beside it: bit for bit."""
    x, s = logits_of(301, 3, V, 15, dtype)
    got = beam.select(x, s, count)
    for some in ([0], [300], [0, 150, 299, 300]):
        some = torch.tensor(some).cuda()
        alone = beam.select(x[some], s[some], count)
        assert all(torch.equal(a[some], b) for a, b in zip(got, alone))
    order = torch.arange(300, -1, -1).cuda()
    assert all(torch.equal(a[order], b) for a, b in zip(got, beam.select(x[order], s[order], count)))
