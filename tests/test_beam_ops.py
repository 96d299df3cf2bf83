"""Selection over beams and vocabulary (gann_beam_select) and the states that
follow it (gann_reorder_states) against plain implementations in 64 bits."""
import ctypes as C

import numpy as np
import pytest
import torch

from conftest import get_index
from gustann_b200 import api
from gustann_b200.api import GustANNError, beam_select, matmul_i8, quantize_rows, reorder_states

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def ref_values(scores, logits, softmax=False, finished=None, end=0):
    """Every candidate's value in 64 bits, [g, w * v]; -inf where there is none."""
    lg = logits.cpu().double().numpy()
    sc = scores.cpu().double().numpy()
    g, w, v = lg.shape
    out = np.empty((g, w * v))
    for i in range(g):
        c = np.where(np.isfinite(lg[i]), lg[i], -np.inf)
        if softmax:
            m = c.max(1, keepdims=True)
            m = np.where(np.isfinite(m), m, 0)
            with np.errstate(divide="ignore", invalid="ignore"):
                c = (c - m) - np.log(np.exp(c - m).sum(1, keepdims=True))
            c = np.where(np.isnan(c) | (c == np.inf), -np.inf, c)
        if finished is not None:
            for b in np.flatnonzero(finished[i].cpu().numpy()):
                c[b] = -np.inf
                c[b, end] = 0
        out[i] = np.where(np.isfinite(sc[i])[:, None], c + np.where(np.isfinite(sc[i]), sc[i], 0)[:, None],
                          -np.inf).ravel()
    return out


def ref_select(scores, logits, k, softmax=False, finished=None, end=0, values=None):
    c = ref_values(scores, logits, softmax, finished, end) if values is None else values
    g, v = c.shape[0], logits.shape[2]
    val = np.full((g, k), -np.inf)
    par = np.full((g, k), -1)
    tok = np.full((g, k), -1)
    for i in range(g):
        o = np.lexsort((np.arange(c.shape[1]), -c[i]))[:k]
        o = o[np.isfinite(c[i, o])]
        val[i, :o.size], par[i, :o.size], tok[i, :o.size] = c[i, o], o // v, o % v
    return val, par, tok


# with log-softmax the sum of exponentials is off by 2^-22 (2 steps of the
# exponential), 2^-24 times the arguments (at most log of the vocabulary, 21,
# on the sum's average; the constant log2 e and the step's rounding, one each)
# and at most 64 sums in float32: below 2^-17 together, which is the logarithm's
# error, one and the same for all candidates of a row
LSE = 2.0 ** -17


def check_select(scores, logits, k, softmax=False, finished=None, end=0):
    s, p, t = (x.cpu().numpy() for x in
               beam_select(scores, logits, k, log_softmax=softmax, finished=finished, end_token=end))
    values = ref_values(scores, logits, softmax, finished, end)
    rv, rp, rt = ref_select(scores, logits, k, softmax, finished, end, values)
    v = logits.shape[2]
    if softmax:
        # Rows' values are off by LSE at most, so the i-th best by the computed
        # values is within 2 LSE of the i-th best by the exact ones, and only
        # candidates of different rows that near to each other can trade places:
        # as many candidates, none twice, and each row's in exact order.
        assert np.array_equal(p < 0, rp < 0) and np.array_equal(t < 0, rt < 0)
        for i in range(len(p)):
            n = int((p[i] >= 0).sum())
            flat = p[i, :n].astype(np.int64) * v + t[i, :n]
            assert len(set(flat.tolist())) == n
            with np.errstate(invalid="ignore"):
                assert bool((np.abs(values[i, flat] - rv[i, :n]) <= 2 * LSE).all())
            for b in set(p[i, :n].tolist()):
                f = flat[p[i, :n] == b]
                row = np.lexsort((np.arange(v), -values[i, b * v:(b + 1) * v]))[:f.size]
                assert np.array_equal(f - b * v, row)
            rv[i, :n] = values[i, flat]
    else:
        assert np.array_equal(p, rp) and np.array_equal(t, rt)
    s = s.astype(np.float64)
    # the 64-bit value rounded to float32
    with np.errstate(invalid="ignore"):
        bound = 2.0 ** -24 * np.abs(rv) * 1.01 + (LSE if softmax else 0.0)
        lost = np.abs(rv) > np.finfo(np.float32).max
        assert bool(((np.abs(s - rv) <= bound) | (s == rv) | (lost & np.isinf(s))).all())


def make(g, w, v, dtype, seed, spread=3.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    lg = (spread * torch.randn(g, w, v, generator=gen, device="cuda")).to(DT[dtype])
    sc = -4 * torch.rand(g, w, generator=gen, device="cuda")
    return sc, lg


SIZES = [(1, 1, 1, 1), (1, 1, 5, 9), (1, 4, 32001, 8), (3, 2, 17, 4), (2, 4, 4099, 8), (2, 1, 50000, 1),
         (1, 3, 131075, 32), (5, 8, 256, 8), (40, 32, 16, 32), (300, 8, 100, 100), (7, 64, 10, 128), (2, 128, 33, 128),
         (1, 128, 3000, 128), (2, 16, 9000, 33), (1, 2, 70001, 128), (1000, 4, 64, 16), (9, 5, 1023, 64),
         (33, 1, 2048, 2), (3, 7, 8191, 17), (4, 2, 20000, 65), (800, 2, 4000, 8), (800, 2, 9000, 24),
         (760, 3, 700, 90)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("softmax", [False, True])
@pytest.mark.parametrize("g,w,v,k", SIZES)
def test_select_equals_sorted(g, w, v, k, softmax, dtype):
    sc, lg = make(g, w, v, dtype, g * 31 + w * 7 + v + k)
    check_select(sc, lg, k, softmax)


@pytest.mark.gpu
@pytest.mark.parametrize("softmax", [False, True])
@pytest.mark.parametrize("g,w,v,k", [(4, 4, 100, 8), (2, 3, 5000, 6), (3, 8, 20011, 16), (20, 6, 40, 50)])
def test_finished_dead_and_masked_beams(g, w, v, k, softmax):
    sc, lg = make(g, w, v, "f32", 3)
    gen = torch.Generator(device="cuda").manual_seed(9)
    fin = torch.rand(g, w, generator=gen, device="cuda") < 0.4
    check_select(sc, lg, k, softmax, fin, v - 1)
    check_select(sc, lg, k, softmax, fin.to(torch.uint8), 0)
    check_select(sc, lg, k, softmax, torch.ones_like(fin), v // 2)
    # first token: one live beam; dead beams by -inf, inf and NaN
    sc2 = sc.clone()
    sc2[:, 1:] = float("-inf")
    check_select(sc2, lg, k, softmax, fin, 1)
    sc2[0, 0] = float("nan")
    sc2[1, 0] = float("inf")
    check_select(sc2, lg, k, softmax)
    # rows with nothing left, rows with one token, masks of every kind
    lg2 = lg.clone()
    lg2[0] = float("-inf")
    lg2[1, 0] = float("nan")
    lg2[1, 1] = float("inf")
    lg2[-1, :, 1:] = float("-inf")
    check_select(sc, lg2, k, softmax)
    check_select(sc, lg2, k, softmax, fin, 2)
    lg3 = lg.clone()
    hide = torch.rand(v, generator=gen, device="cuda") < 0.95
    for bad in (float("-inf"), float("inf"), float("nan")):
        lg3[:, :, hide] = bad
        check_select(sc, lg3, k, softmax)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("softmax", [False, True])
@pytest.mark.parametrize("g,w,v,k", [(2, 4, 300, 16), (1, 3, 9000, 40), (1, 2, 40000, 128), (50, 8, 64, 20)])
def test_equal_values_go_to_the_lowest_index(g, w, v, k, softmax, dtype):
    sc, lg = make(g, w, v, dtype, 5)
    check_select(torch.zeros_like(sc), torch.zeros_like(lg), k, softmax)
    check_select(sc, torch.zeros_like(lg), k, softmax)
    few = lg.float().round().to(DT[dtype])                       # a handful of distinct values
    if not softmax:
        check_select(sc.round(), few, k)
    # the type's lowest value as a mask: still candidates, behind all others
    low = torch.full_like(lg, torch.finfo(lg.dtype).min)
    low[:, :, 3:6] = lg[:, :, 3:6]
    check_select(sc, low, k, softmax)
    check_select(sc, torch.full_like(lg, torch.finfo(lg.dtype).min), k, softmax)


@pytest.mark.gpu
@pytest.mark.parametrize("order", ["up", "down"])
@pytest.mark.parametrize("w,v,k", [(2, 3000, 16), (1, 40000, 100), (4, 200, 128)])
def test_sorted_input(order, w, v, k):
    lg = torch.linspace(-9, 9, w * v, device="cuda").reshape(1, w, v)
    if order == "down":
        lg = -lg
    check_select(torch.zeros(1, w, device="cuda"), lg.contiguous(), k)
    check_select(torch.zeros(1, w, device="cuda"), lg.contiguous(), k, True)


@pytest.mark.gpu
def test_values_closer_than_float32():
    """Candidates whose sums with the score are equal in float32 but not in 64 bits."""
    lg = torch.zeros(1, 2, 50, device="cuda")
    lg[0, 0, 20], lg[0, 0, 30], lg[0, 1, 10] = 1.0, 1.0 + 2.0 ** -23, 1.0 + 2.0 ** -22
    sc = torch.tensor([[-1000.0, -1000.0]], device="cuda")
    s, p, t = beam_select(sc, lg, 3)
    assert t.tolist() == [[10, 30, 20]] and p.tolist() == [[1, 0, 0]]
    check_select(sc, lg, 10)


def equal_sums(g, w, v, dtype, score, kind):
    """Scores so large beside the logits (or logits so small beside the scores)
    that many different logits have one sum in 64 bits."""
    sc, lg = make(g, w, v, dtype, v)
    if kind == "tiny":
        gen = torch.Generator(device="cuda").manual_seed(v)
        lg = (1e-17 * torch.randint(-40, 41, lg.shape, generator=gen, device="cuda")).to(lg.dtype)
    if kind == "one ordinary beam":
        lg[:, 0, 5:] = float("-inf")      # too few to fill the result
    sc = sc + score if kind == "spread" else torch.full_like(sc, score)
    if kind == "one ordinary beam":
        sc[:, 0] = -1.5
    return sc, lg


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("score", [-5.0, -1e9, 1e12, -1e15, -3.4e38])
@pytest.mark.parametrize("g,w,v,k", [(1, 2, 300, 9), (2, 3, 20011, 8), (1, 2, 40000, 128), (2, 4, 6000, 20)])
def test_equal_sums_of_different_logits(g, w, v, k, score, dtype):
    """Values are compared in 64 bits, whichever way the sizes are run."""
    for kind in ("same", "spread", "tiny", "one ordinary beam"):
        check_select(*equal_sums(g, w, v, dtype, score, kind), k)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("score", [-5.0, -1e9, 1e12, -1e15, -3.4e38])
@pytest.mark.parametrize("g,w,v,k", [(1, 2, 300, 9), (2, 3, 20011, 8), (1, 2, 40000, 128)])
def test_equal_sums_with_log_softmax(g, w, v, k, score, dtype):
    """A beam's own candidates come by score + logit in 64 bits, then token. The
    value is rounded three times in 64 bits beside the logarithm's error, each
    time by half a step of at most 2^-52 of the score (other terms: LSE)."""
    for kind in ("same", "spread", "tiny", "one ordinary beam"):
        sc, lg = equal_sums(g, w, v, dtype, score, kind)
        s, p, t = (x.cpu().numpy() for x in beam_select(sc, lg, k, log_softmax=True))
        values = ref_values(sc, lg, True)
        rv, rp, _ = ref_select(sc, lg, k, True, values=values)
        assert np.array_equal(p < 0, rp < 0)
        sums = sc.cpu().double().numpy()[:, :, None] + lg.cpu().double().numpy()
        off = 2 * (LSE + 4 * 2.0 ** -53 * abs(score))
        for i in range(g):
            n = int((p[i] >= 0).sum())
            assert bool((np.abs(values[i, p[i, :n] * v + t[i, :n]] - rv[i, :n]) <= off).all())
            assert bool((np.abs(s[i, :n] - rv[i, :n]) <= off + 1.01 * 2.0 ** -24 * np.abs(rv[i, :n])).all())
            for b in set(p[i, :n].tolist()):
                f = t[i, :n][p[i, :n] == b]
                assert np.array_equal(f, np.lexsort((np.arange(v), -sums[i, b]))[:f.size])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DT))
def test_select_strides_and_alignment(dtype):
    gen = torch.Generator(device="cuda").manual_seed(2)
    big = torch.randn(6, 5, 3001, generator=gen, device="cuda").to(DT[dtype])
    sc = torch.rand(6, 5, generator=gen, device="cuda")
    for lg in (big[:, :, 1:], big[:, :, 3:2000], big[::2], big[:, ::2, 5:300], big.transpose(0, 1),
               big[:1].expand(4, 5, 3001), big[:, :1, :77].expand(6, 4, 77)):
        s = sc.t()[:lg.shape[0], :lg.shape[1]] if lg.shape[0] == 5 else sc[:lg.shape[0], :lg.shape[1]]
        check_select(s, lg, 7)
        check_select(s, lg, 7, True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,offset", [(d, o) for d, offs in (
    ("f32", (1e4, -65504.0, 1e5, -1.31e5, 1.32e5, -1e6, 1e7, 3e7, -5e7, 1e8, -1e9, 1e10, -1e12, 1e30, -3e38)),
    ("f16", (1e4, 65504.0, -65504.0)), ("bf16", (1e4, -1e5, 1e6, 3e7, -1e9, 1e12, -1e30))) for o in offs])
def test_log_softmax_of_rows_far_from_zero(dtype, offset):
    """A constant added to a row changes no candidate's value: rows around the
    offset, one row of the offset alone (every token masked by a large finite
    number) beside ordinary ones, and a row with a few tokens left. The terms
    are taken relative to the maximum, so the derivation of LSE holds as it is."""
    for g, w, v, k in ((2, 4, 3001, 8), (1, 3, 20000, 40)):
        sc, lg = make(g, w, v, dtype, 11)
        check_select(sc, (lg.float() + offset).clamp(torch.finfo(lg.dtype).min, torch.finfo(lg.dtype).max).to(lg.dtype),
                     k, True)
        one = lg.clone()
        one[:, 1] = offset
        check_select(sc, one, k, True)
        one[:, 2, 5:] = offset
        check_select(sc, one, k, True)


@pytest.mark.gpu
def test_select_offsets_past_32_bits():
    """A group stride that puts the last group 2^31 elements behind the first."""
    lg = torch.zeros(2 ** 31 + 4096, dtype=torch.float16, device="cuda").as_strided((2, 2, 1000), (2 ** 31, 1000, 1))
    lg[1] = torch.randn(2, 1000, device="cuda").half()
    check_select(torch.zeros(2, 2, device="cuda"), lg, 5)


@pytest.mark.gpu
def test_select_is_the_same_every_time_on_any_stream():
    sc, lg = make(8, 4, 20000, "f32", 1)
    want = beam_select(sc, lg, 8, log_softmax=True)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(side):
            a = beam_select(sc, lg, 8, log_softmax=True)
        b = beam_select(sc, lg, 8, log_softmax=True, stream=side.cuda_stream)
        c = beam_select(sc, lg, 8, log_softmax=True)
        torch.cuda.synchronize()
        for got in (a, b, c):
            assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.gpu
def test_two_graphs_of_a_decoding_step():
    """Two captured steps, replayed at the same time on two streams."""
    ins, graphs, outs = [], [], []
    for i in range(2):
        sc, lg = make(4, 4, 30000, "bf16", i)
        hist = torch.randint(0, 99, (4, 4, 12), device="cuda", dtype=torch.int32)
        beam_select(sc, lg, 4, log_softmax=True)
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            s, p, t = beam_select(sc, lg, 4, log_softmax=True)
            h = reorder_states(hist, p)
        ins.append((sc, lg, hist))
        graphs.append(gr)
        outs.append((s, p, t, h))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for rep in range(4):
        for i, (sc, lg, hist) in enumerate(ins):
            lg.copy_(torch.randn(lg.shape, generator=torch.Generator().manual_seed(rep * 2 + i)))
        torch.cuda.synchronize()
        for st, gr in zip(streams, graphs):
            with torch.cuda.stream(st):
                gr.replay()
        torch.cuda.synchronize()
        for (sc, lg, hist), (s, p, t, h) in zip(ins, outs):
            rv, rp, rt = ref_select(sc, lg, 4, True)
            assert np.array_equal(p.cpu().numpy(), rp) and np.array_equal(t.cpu().numpy(), rt)
            assert torch.equal(h, hist[torch.arange(4)[:, None], p.long()])


# ------------------------------------------------------------------- reorder
def ref_reorder(s, p):
    w = s.shape[1]
    ok = (p >= 0) & (p < w)
    out = s[torch.arange(len(p), device=p.device)[:, None], p.long().clamp(0, w - 1)]
    return torch.where(ok.reshape(ok.shape + (1,) * (out.dim() - 2)), out, torch.zeros_like(out))


def states_of(g, w, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def r(*shape, dtype=torch.float32):
        return (100 * torch.randn(*shape, generator=gen, device="cuda")).to(dtype)
    cache = r(g, w, 3, 40, 16, dtype=torch.bfloat16)
    layers = r(2, g, w, 3, 20, 9, dtype=torch.float16)
    return [r(g, w), r(g, w, 7, dtype=torch.int32), r(g, w, 5, dtype=torch.uint8), cache[:, :, :, :33],
            layers.permute(1, 2, 0, 3, 4, 5)[..., :11, :], r(g, w, 13, dtype=torch.int64), r(g, w, 1, 128),
            (r(g, w, 3) > 0), r(g, w, 6, 10)[..., ::2], r(g, w, 0, 4)]


@pytest.mark.gpu
@pytest.mark.parametrize("g,w,k", [(1, 1, 1), (3, 4, 4), (2, 8, 3), (5, 3, 9), (70, 2, 2), (1, 128, 128), (4, 5, 1)])
def test_reorder_equals_indexing(g, w, k):
    states = states_of(g, w, g + w + k)
    gen = torch.Generator(device="cuda").manual_seed(k)
    p = torch.randint(-1, w, (g, k), generator=gen, device="cuda", dtype=torch.int32)
    want = [ref_reorder(s, p) for s in states]
    before = [s.clone() for s in states]
    for got, ref, s, b in zip(reorder_states(states, p), want, states, before):
        assert got.shape == ref.shape and got.dtype == ref.dtype and torch.equal(got, ref)
        assert torch.equal(s, b)
    for s, ref in zip(states, want):
        assert torch.equal(reorder_states(s, p), ref)
        out = torch.zeros((g, k + 2) + s.shape[2:], dtype=s.dtype, device="cuda")
        assert torch.equal(reorder_states(s, p, out=out[:, 1:k + 1]), ref)
        assert not out[:, 0].any() and not out[:, k + 1].any()
    if k <= w:
        got = reorder_states(states, p, out=states)
        for s, ref, b in zip(got, want, before):
            assert torch.equal(s[:, :k], ref) and torch.equal(s[:, k:], b[:, k:])


@pytest.mark.gpu
def test_reorder_in_place_leaves_the_rest_of_a_cache():
    cache = torch.randn(4, 6, 3, 50, 24, device="cuda")
    before = cache.clone()
    p = torch.randint(0, 6, (4, 6), device="cuda", dtype=torch.int32)
    view = cache[:, :, :, 5:37]
    reorder_states(view, p, out=view)
    assert torch.equal(view, ref_reorder(before[:, :, :, 5:37], p))
    assert torch.equal(cache[:, :, :, :5], before[:, :, :, :5]) and torch.equal(cache[:, :, :, 37:], before[:, :, :, 37:])


@pytest.mark.gpu
def test_reorder_parents_that_are_no_beams():
    s = torch.ones(2, 3, 5, device="cuda")
    p = torch.tensor([[0, 3, 2], [-1, -7, 2 ** 31 - 1]], device="cuda", dtype=torch.int32)
    assert torch.equal(reorder_states(s, p), ref_reorder(s, p))
    assert reorder_states(s, p).sum() == 10


@pytest.mark.gpu
def test_reorder_takes_any_iterable():
    """States and targets may come from generators, on a given stream too."""
    states = states_of(3, 4, 1)
    p = torch.randint(0, 4, (3, 4), device="cuda", dtype=torch.int32)
    want = [ref_reorder(s, p) for s in states]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for stream in (None, 0, side.cuda_stream):
        new = reorder_states((s for s in states), p, stream=stream)
        outs = [torch.zeros_like(w) for w in want]
        torch.cuda.synchronize()
        into = reorder_states((s for s in states), p, out=(o for o in outs), stream=stream)
        one = reorder_states(states[0], p, stream=stream)
        torch.cuda.synchronize()
        assert len(new) == len(into) == len(want) and torch.equal(one, want[0])
        for a, b, o, w in zip(new, into, outs, want):
            assert torch.equal(a, w) and torch.equal(b, w) and torch.equal(o, w)


@pytest.mark.gpu
def test_reorder_conjugate_views():
    z = torch.randn(3, 4, 5, dtype=torch.complex64, device="cuda")
    p = torch.randint(-1, 4, (3, 4), device="cuda", dtype=torch.int32)
    for s in (z, z.conj(), z.conj().imag, z.imag):
        got = reorder_states(s, p)
        assert torch.equal(got, ref_reorder(s, p))
    rejects(reorder_states, z.conj(), p, out=torch.zeros_like(z))
    rejects(reorder_states, z.conj().imag, p, out=torch.zeros(3, 4, 5, device="cuda"))
    into = torch.zeros_like(z)
    reorder_states(z.conj(), p, out=into.conj())
    assert torch.equal(into.conj(), ref_reorder(z.conj(), p))


@pytest.mark.gpu
def test_reorder_many_states_and_many_groups():
    g = 70000
    s = torch.randint(0, 99, (g, 2, 3), device="cuda", dtype=torch.int16)
    p = torch.randint(0, 2, (g, 2), device="cuda", dtype=torch.int32)
    assert torch.equal(reorder_states(s, p), ref_reorder(s, p))
    many = [torch.randn(3, 4, i % 7 + 1, device="cuda") for i in range(75)]
    p = torch.randint(0, 4, (3, 4), device="cuda", dtype=torch.int32)
    for got, m in zip(reorder_states(many, p), many):
        assert torch.equal(got, ref_reorder(m, p))
    assert reorder_states([], p) == [] and reorder_states(s[:0], p[:0]).shape == (0, 4, 3)


@pytest.mark.gpu
def test_reorder_offsets_past_32_bits():
    s = torch.zeros(2, 2, 2 ** 30 + 16, dtype=torch.int8, device="cuda")
    s[1, 1, -16:] = 5
    s[1, 0, :16] = 3
    p = torch.tensor([[0, 0], [1, 0]], device="cuda", dtype=torch.int32)
    reorder_states(s, p, out=s)
    assert bool((s[1, 0, -16:] == 5).all() and (s[1, 1, :16] == 3).all()) and int(s[0].any()) == 0
    assert int(s[1, 0].count_nonzero()) == 16 and int(s[1, 1].count_nonzero()) == 16


# ------------------------------------------------------------ used together
@pytest.mark.gpu
def test_scores_of_slices_joined_into_a_top_k():
    """Base vectors in slices: 8-bit scores of each slice, its best k, and the
    slices' lists joined, against one selection over all exact scores."""
    gen = torch.Generator(device="cuda").manual_seed(0)
    n, d, nq, k, slices = 6000, 96, 37, 10, 4
    base, bs = quantize_rows(torch.randn(n, d, generator=gen, device="cuda"))
    q, qs = quantize_rows(torch.randn(nq, d, generator=gen, device="cuda"))
    zero = torch.zeros(nq, 1, device="cuda")
    size = n // slices
    lists_s, lists_i = [], []
    for i in range(slices):
        y = matmul_i8(q, qs, base[i * size:(i + 1) * size], bs[i * size:(i + 1) * size])
        s, _, t = beam_select(zero, y[:, None], k)
        lists_s.append(s)
        lists_i.append(t + i * size)
    s, p, t = beam_select(zero.expand(nq, slices), torch.stack(lists_s, 1), k)
    ids = torch.stack(lists_i, 1)[torch.arange(nq, device="cuda")[:, None], p.long(), t.long()]
    acc = (q.cpu().double() @ base.cpu().double().T).float()          # exact: below 2^24
    full = (acc * qs.cpu()[:, None]) * bs.cpu()[None, :]
    rv, ri = torch.sort(full, dim=1, descending=True, stable=True)
    assert torch.equal(s.cpu(), rv[:, :k]) and torch.equal(ids.cpu(), ri[:, :k])


@pytest.mark.gpu
def test_codes_by_beam_search_over_codebooks():
    """Three levels of codebook entries for every vector: scores of the beams'
    residuals by 8-bit products, the best beams, the states behind them."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    g, d, v, w = 50, 32, 64, 5
    x = torch.randn(g, d, generator=gen, device="cuda")
    books = [torch.randn(v, d, generator=gen, device="cuda") / (i + 1) for i in range(3)]

    def encode(select, reorder, product):
        res = x[:, None].expand(g, w, d).contiguous()
        score = torch.full((g, w), float("-inf"), device="cuda")
        score[:, 0] = -(x * x).sum(1)
        codes = torch.zeros(g, w, 0, dtype=torch.int32, device="cuda")
        for book in books:
            y = product(res.reshape(g * w, d), book)
            score, parent, token = select(score, y.reshape(g, w, v), w)
            res, codes = reorder([res, codes], parent)
            codes = torch.cat([codes, token[..., None]], 2)
            res = res - book[token.long()]
        return score, codes, res

    def product(r, book):
        c, s = quantize_rows(r)
        b, bs = quantize_rows(book)
        return matmul_i8(c, s, b, 2 * bs, bias=-(book * book).sum(1))

    def plain_product(r, book):
        c, s = quantize_rows(r)
        b, bs = quantize_rows(book)
        acc = (c.cpu().double() @ b.cpu().double().T)
        y = (acc.float() * s.cpu()[:, None]).double() * (2 * bs.cpu().double()) - (book * book).sum(1).cpu().double()
        return y.float().cuda()

    def plain_select(score, y, k):
        rv, rp, rt = ref_select(score, y, k)
        return (torch.from_numpy(rv).float().cuda(), torch.from_numpy(rp).int().cuda(),
                torch.from_numpy(rt).int().cuda())

    got = encode(beam_select, reorder_states, product)
    want = encode(plain_select, lambda st, p: [ref_reorder(s, p) for s in st], plain_product)
    assert torch.equal(got[1], want[1]) and torch.equal(got[0], want[0]) and torch.equal(got[2], want[2])


@pytest.mark.gpu
def test_calls_after_another_calls_refused_allocation(index_root):
    """A call that ran out of memory leaves an error with the host thread, which
    is not the next call's."""
    info = get_index(index_root, "u8")
    p = info["paths"]
    g = api.GustANN(info["dtype"])
    g.init_pure_mem(api.GustANNConfig(p["index_file"], p["pq_file_prefix"], p["nav_graph_prefix"]), True)
    one = np.zeros(1, np.float32)
    x = torch.randn(8, 64, device="cuda")
    sc, lg = make(2, 3, 300, "f32", 0)
    c, s = quantize_rows(x)
    par = torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    for call in (lambda: quantize_rows(x), lambda: matmul_i8(c, s, c, s), lambda: matmul_i8(c[:1], s[:1], c, s),
                 lambda: beam_select(sc, lg, 4), lambda: beam_select(sc, lg, 4, log_softmax=True),
                 lambda: reorder_states(lg, par)):
        # 2^40 queries: refused before any is read
        assert api.lib.gann_probe_lut(g._h, one.ctypes.data, 2 ** 40, one.ctypes.data) == api.GANN_ENOMEM
        call()
    g.close()


# ------------------------------------------------------------------ refusals
def rejects(f, *a, **k):
    with pytest.raises(GustANNError) as e:
        f(*a, **k)
    assert e.value.code == api.GANN_EINVAL and str(e.value)


def test_refusals():
    sc, lg = torch.zeros(2, 3), torch.zeros(2, 3, 8)
    rejects(beam_select, sc, lg, 2)                       # not on a GPU
    rejects(beam_select, sc.half(), lg, 2)
    rejects(beam_select, sc[:1], lg, 2)
    rejects(beam_select, sc, lg[0], 2)
    rejects(beam_select, sc, lg.double(), 2)
    rejects(beam_select, sc, lg, 2, finished=torch.zeros(2, 3))
    rejects(beam_select, sc, lg, 2, finished=torch.zeros(2, 2, dtype=torch.bool))
    p = torch.zeros(2, 3, dtype=torch.int32)
    rejects(reorder_states, lg, p)
    rejects(reorder_states, lg, p.long())
    rejects(reorder_states, lg, p[0])


def test_c_entries_refuse_before_touching_the_gpu():
    lib = api.lib
    buf = (C.c_byte * 4096)()
    p = (C.addressof(buf) + 63) // 64 * 64
    need = C.c_int64()

    def sel(dt=api.F32, gs=8, bs=8, sc=p, fin=None, g=1, w=1, v=8, k=1, end=0, lg=p, out=p):
        return lib.gann_beam_select(lg, dt, gs, bs, sc, fin, g, w, v, k, 1, end, out, p, p, p, 4096, 0, None)

    def reo(n=1, g=1, w=2, k=2, par=p, **kw):
        st = api._State(p, p + 1024, 64, 32, (0, 0), 64, 32, (0, 0), (1, 1), 32)
        for a, b in kw.items():
            setattr(st, a, b)
        return lib.gann_reorder_states(C.byref(st), n, par, g, w, k, 0, None)

    two = C.c_int64 * 2
    bad = [sel(dt=0), sel(gs=-1), sel(bs=-1), sel(sc=None), sel(g=-1), sel(w=0), sel(w=129), sel(v=0), sel(k=0),
           sel(k=129), sel(w=128, v=2 ** 24), sel(fin=p, end=8), sel(fin=p, end=-1), sel(lg=None), sel(lg=p + 2),
           sel(out=None), sel(out=p + 1), lib.gann_beam_select_workspace(1, 1, 8, 1, api.F32, 0, None),
           lib.gann_beam_select_workspace(1, 0, 8, 1, api.F32, 0, C.byref(need)),
           lib.gann_beam_select_workspace(1, 1, 8, 1, 0, 0, C.byref(need)), sel(v=20000, g=999),
           reo(n=-1), reo(g=-1), reo(w=0), reo(w=129), reo(k=0), reo(k=129), reo(par=None), reo(par=p + 2),
           reo(src=None), reo(dst=None), reo(row_bytes=-1), reo(size=two(-1, 1)), reo(size=two(2 ** 40, 2 ** 40)),
           reo(dst=p, k=3, w=2), reo(dst=p, dst_beam=16), reo(dst=p, dst_stride=two(0, 8))]
    assert bad == [api.GANN_EINVAL] * len(bad)
    assert sel(g=0) == api.GANN_OK and reo(n=0) == api.GANN_OK and reo(g=0) == api.GANN_OK


def test_state_layouts():
    lay = api._state_layout
    t = torch.zeros(2, 3, 4, 10, 6)
    c = torch.zeros(2, 3, 4, 7, 6)
    assert lay(t, t) == ([1, 1], [0, 0], [0, 0], 960)
    assert lay(t[:, :, :, :7], c) == ([1, 4], [0, 240], [0, 168], 168)
    assert lay(torch.zeros(2, 3), torch.zeros(2, 3)) == ([1, 1], [0, 0], [0, 0], 4)
    u = torch.zeros(5, 2, 3, 4, 10, 6).permute(1, 2, 0, 3, 4, 5)[..., :7, :]
    assert lay(u, torch.zeros(2, 3, 5, 4, 7, 6)) == ([5, 4], [5760, 240], [672, 168], 168)
    assert lay(t[..., ::2], torch.zeros(2, 3, 4, 10, 3)) == ([1, 120], [0, 8], [0, 4], 4)
    assert lay(t[:, :, ::2, ::2, ::2], torch.zeros(2, 3, 2, 5, 3)) is None
    assert api._apart(t) and api._apart(u) and not api._apart(t[:, :1].expand(2, 3, 4, 10, 6))
    assert api._extent(t) == (t.data_ptr(), t.data_ptr() + 4 * t.numel())


def targets(monkeypatch, srcs, dsts, k):
    """The check of targets, on tensors of the host."""
    monkeypatch.setattr(api, "_on_cuda", lambda who, *t: (t[0].device, 0))
    g = srcs[0].shape[0]
    api._check_targets(srcs, dsts, torch.zeros(g, k, dtype=torch.int32), g, k)


def test_targets_that_lie_among_beams_that_are_only_read(monkeypatch):
    # groups that share beams: what one writes another reads
    s = torch.zeros(64).as_strided((2, 4, 8), (16, 8, 1))
    rejects(targets, monkeypatch, [s], [s[:, :2]], 2)
    rejects(targets, monkeypatch, [s], [s], 4)
    # one state's target in another's beams behind its own target
    x = torch.zeros(1, 5, 8)
    rejects(targets, monkeypatch, [x, torch.zeros(1, 5, 8)], [x[:, :2], x[:, 3:]], 2)
    targets(monkeypatch, [x, torch.zeros(1, 5, 8)], [x[:, :2], torch.zeros(1, 2, 8)], 2)
    targets(monkeypatch, [x], [x], 5)
    targets(monkeypatch, [x, x], [torch.zeros(1, 2, 8), torch.zeros(1, 2, 8)], 2)


def test_targets_side_by_side_in_one_array(monkeypatch):
    kv = torch.zeros(2, 3, 2, 4, 5)          # keys and values of one array
    both = [kv[:, :, 0], kv[:, :, 1]]
    targets(monkeypatch, both, both, 3)
    rows = torch.zeros(2, 3, 24)             # parts of each row, of different widths
    parts = [rows[..., :10], rows[..., 10:11], rows[..., 11:]]
    targets(monkeypatch, parts, parts, 3)
    targets(monkeypatch, [kv[:, :, 0]], [kv[:, :, 1]], 3)
    rejects(targets, monkeypatch, [rows[..., :10], rows[..., 9:]], [rows[..., :10], rows[..., 9:]], 3)
    rejects(targets, monkeypatch, [kv[:, :, 0], kv[:, :, 0, 1:]], [kv[:, :, 0], kv[:, :, 0, 1:]], 3)
    rejects(targets, monkeypatch, [kv[..., 1:4]], [kv[..., 2:]], 3)


def test_disjoint_against_every_address():
    """Never true of tensors that share an element, and true of slices side by side."""
    gen = np.random.default_rng(0)
    buf = torch.zeros(4096, dtype=torch.uint8)
    kept = {torch.uint8: buf, torch.int16: buf.view(torch.int16), torch.float32: buf.view(torch.float32)}
    apart = shared = found = 0
    for _ in range(6000):
        two = []
        strides = [int(gen.integers(1, 6)), int(gen.integers(1, 25)), int(gen.integers(1, 90))]
        for dt in [list(kept)[int(gen.integers(3))]] * 2 if gen.random() < 0.8 else [torch.uint8, torch.float32]:
            shape = [int(gen.integers(1, 5)) for _ in strides]
            st = strides if gen.random() < 0.8 else [int(x) for x in gen.permutation(strides)]
            two.append(kept[dt].as_strided(shape, st, int(gen.integers(0, 150))))
        used = []
        for t in two:
            at = torch.zeros(1, dtype=torch.int64)
            for n, st in zip(t.shape, t.stride()):
                at = (at[:, None] + torch.arange(n) * st).flatten()
            first = t.storage_offset() * t.element_size()
            used.append({first + x * t.element_size() + e for x in at.tolist() for e in range(t.element_size())})
        meet = bool(used[0] & used[1])
        said = api._disjoint(*two)
        assert said == api._disjoint(*reversed(two)) or not meet
        assert not (said and meet)
        apart, shared, found = apart + (not meet), shared + meet, found + said
    assert shared > 1000 and apart > 1000 and found > apart // 2
    for a, b in ((buf[:4000].view(10, 20, 20)[:, :, :7], buf[:4000].view(10, 20, 20)[:, :, 7:]),
                 (buf[5:4005].view(10, 20, 20)[1:, :, :7], buf[:4000].view(10, 20, 20)[:, :, 0:5])):
        assert api._disjoint(a, b) and api._disjoint(b, a)


@pytest.mark.gpu
@pytest.mark.parametrize("k", [1, 3, 4])
def test_reorder_slices_of_one_array_in_place(k):
    g, w = 5, 4
    kv = torch.randn(g, w, 3, 2, 7, 6, device="cuda")       # layers, keys and values, positions
    before = kv.clone()
    states = [kv[:, :, layer, i, :5] for layer in range(3) for i in range(2)]
    p = torch.randint(-1, w, (g, k), device="cuda", dtype=torch.int32)
    reorder_states(states, p, out=[s[:, :k] for s in states] if k < w else states)
    assert torch.equal(kv[:, :k, :, :, :5], ref_reorder(before[:, :, :, :, :5], p))
    assert torch.equal(kv[:, k:], before[:, k:]) and torch.equal(kv[:, :, :, :, 5:], before[:, :, :, :, 5:])


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    sc, lg = make(2, 3, 8, "f32", 1)
    rejects(beam_select, sc.cpu(), lg, 2)
    rejects(beam_select, sc, lg, 0)
    rejects(beam_select, sc, lg, 129)
    rejects(beam_select, sc, lg[:, :, ::2], 2)
    rejects(beam_select, sc, lg, 2, finished=sc < 0, end_token=8)
    rejects(beam_select, torch.zeros(1, 129, device="cuda"), torch.zeros(1, 129, 4, device="cuda"), 2)
    p = torch.zeros(2, 3, device="cuda", dtype=torch.int32)
    rejects(reorder_states, lg[:1], p)
    rejects(reorder_states, [lg, lg[:, :2]], p)
    rejects(reorder_states, lg, p, out=torch.zeros(2, 2, 8, device="cuda"))
    rejects(reorder_states, lg, p, out=torch.zeros(2, 3, 8, device="cuda").half())
    rejects(reorder_states, lg, p, out=torch.zeros(1, 3, 8, device="cuda").expand(2, 3, 8))
    rejects(reorder_states, [lg, lg], p, out=[lg, lg])
    rejects(reorder_states, [lg], p, out=[lg, lg])
    two = torch.zeros(2, 4, 8, device="cuda")
    rejects(reorder_states, two[:, :3], p, out=two[:, 1:])
    rejects(reorder_states, lg, p, out=p.view(torch.float32)[:, :, None].expand(2, 3, 8))
    four = torch.zeros(2, 3, 4, 4, 4, device="cuda")
    rejects(reorder_states, four[:, :, ::2, ::2, ::2], p)
    wide = torch.zeros(2, 5, device="cuda", dtype=torch.int32)
    rejects(reorder_states, lg, wide, out=lg)
