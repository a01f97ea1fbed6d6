"""The decode operators (beam_step, reorder_states, tree_attention, tree_accept) on a GPU
against plain 64-bit restatements of their definitions.

Tolerances. u = 2^-24.
- beam scores: a term exp(x - max) of the sum has relative error at most (3 |x - max| + 4) u
  (the difference, its product with log2 e, the constant; ex2's 4 u). Weighted with the
  probabilities the |x - max| average to at most ln V. Summation in fp32 adds at most 20 u
  (short runs, then a tree; the rest is done in 64 bits). So |score - exact| <=
  (3 ln V + 24) u, plus half a step of the fp32 result, u |score|. Parents, tokens and flags
  have to be equal.
- attention: out is rounded to its type (half a step h relative), the weights p once to it
  (h relative each, A = sum p |v|), a score's fp32 dot product is off by at most
  (dim + 4) 2^-23 S, S the largest scale * sum |q| |k|, which moves the weights by that twice;
  running sums in fp32 add (n / 8 + 16) 2^-23 A over n keys; ex2 of an argument up to S adds
  (4 + 3 * 2 S) u, twice.
"""
import copy
import io
import math
import os
import subprocess
import sys

import numpy as np
import pytest

from tests.conftest import gpu_available

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
U = 2.0 ** -24
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(autouse=True)
def _needs_gpu():
    if not gpu_available():
        pytest.skip("no CUDA device")


@pytest.fixture(scope="module")
def tb():
    import tabby_b200

    return tabby_b200


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


# -- beam search's selection ---------------------------------------------------------------
def plain_beam(logits, scores, n_out, finished=None, eos=-1):
    """The definition, prompt by prompt in float64 (numpy)."""
    x = logits.double().cpu().numpy()
    sc = scores.double().cpu().numpy()
    b, k, v = x.shape
    done = np.zeros((b, k), bool) if finished is None else finished.cpu().numpy().astype(bool)
    out = dict(scores=np.full((b, n_out), -np.inf), parents=np.full((b, n_out), -1),
               tokens=np.full((b, n_out), -1), finished=np.ones((b, n_out), bool),
               status=np.zeros(b, int))
    for p in range(b):
        keys = np.full((k, v), -np.inf)
        bad = bool((np.isnan(sc[p]) | (sc[p] == np.inf)).any())
        for i in range(k):
            if sc[p, i] == -np.inf or bad:
                continue
            if done[p, i]:
                keys[i, eos] = sc[p, i]
                continue
            row = x[p, i]
            if np.isnan(row).any() or (row == np.inf).any():
                bad = True
                continue
            m = row.max()
            if m == -np.inf:
                continue
            keys[i] = sc[p, i] + (row - (m + math.log(np.exp(row - m).sum())))
        if bad:
            out["status"][p] = 4
            continue
        flat = keys.reshape(-1)
        cand = np.nonzero(flat > -np.inf)[0]
        if len(cand) > 4 * n_out:
            floor = np.partition(flat[cand], len(cand) - n_out)[len(cand) - n_out]
            cand = cand[flat[cand] >= floor]
        order = cand[np.lexsort((cand, -flat[cand]))][:n_out]
        n = len(order)
        out["scores"][p, :n] = flat[order]
        out["parents"][p, :n] = order // v
        out["tokens"][p, :n] = order % v
        out["finished"][p, :n] = [done[p, o // v] or o % v == eos for o in order]
    return out


def check_beam(r, want, vocab):
    s = r.scores.double().cpu().numpy()
    np.testing.assert_array_equal(r.status.cpu().numpy(), want["status"])
    np.testing.assert_array_equal(r.parents.cpu().numpy(), want["parents"])
    np.testing.assert_array_equal(r.tokens.cpu().numpy(), want["tokens"])
    np.testing.assert_array_equal(r.finished.cpu().numpy(), want["finished"])
    w = want["scores"]
    np.testing.assert_array_equal(np.isneginf(s), np.isneginf(w))
    f = np.isfinite(w)
    tol = (3 * math.log(max(vocab, 2)) + 24) * U + U * np.abs(w[f])
    assert (np.abs(s[f] - w[f]) <= tol).all(), np.abs(s[f] - w[f]).max()


def beam_inputs(batch, beams, vocab, dtype, pad=0, seed=0):
    g = gen(seed)
    x = (4 * torch.randn(batch, beams, vocab + pad, device="cuda", generator=g)).to(DT[dtype])
    scores = -8 * torch.rand(batch, beams, device="cuda", generator=g)
    return x[..., :vocab], scores


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("batch,beams,vocab,n_out,pad", [
    (1, 1, 1, 1, 0), (1, 1, 2, 4, 0), (3, 4, 3, 20, 0), (2, 64, 5, 128, 1), (5, 3, 31, 6, 3),
    (2, 2, 257, 3, 0), (4, 4, 1000, 8, 0), (1, 5, 2047, 10, 5), (2, 3, 4096, 6, 0),
    (1, 4, 4097, 128, 2), (1, 2, 8191, 1, 0), (2, 2, 8192, 16, 0), (3, 1, 8193, 64, 0),
    (2, 8, 16385, 16, 0), (2, 5, 50257, 10, 0), (1, 33, 32001, 66, 0), (1, 1, 151936, 128, 0),
    (7, 4, 151936, 8, 0), (40, 8, 1003, 16, 0), (1, 64, 20011, 128, 0), (200, 2, 300, 4, 0),
])
def test_beam_step_matches_the_definition(tb, batch, beams, vocab, n_out, pad, dtype):
    x, scores = beam_inputs(batch, beams, vocab, dtype, pad, seed=vocab + beams)
    r = tb.beam_step(x, scores, n_out)
    check_beam(r, plain_beam(x, scores, n_out), vocab)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_beam_step_finished_dead_and_banned(tb, dtype):
    batch, beams, vocab, n_out = 6, 6, 5003, 12
    x, scores = beam_inputs(batch, beams, vocab, dtype, 1, seed=5)
    x = x.clone()
    finished = torch.zeros(batch, beams, dtype=torch.bool, device="cuda")
    finished[0, 1] = finished[1, :] = finished[3, 0] = True
    scores[2, 1:] = -math.inf          # a first step
    scores[4, :] = -math.inf           # no beam lives
    scores[3, 0] = -math.inf           # finished and dead: dead
    x[0, 1] = math.nan                 # what is not read may hold anything
    x[2, 3] = math.inf
    x[5, 0] = -math.inf                # a live beam with every token banned
    x[5, 1:, 7:] = -math.inf           # a grammar that leaves a few
    x[3, 2, ::2] = -math.inf
    r = tb.beam_step(x, scores, n_out, finished=finished, eos_id=17)
    want = plain_beam(x, scores, n_out, finished, 17)
    assert (want["parents"][4] == -1).all() and (want["parents"][1][6:] == -1).all()
    check_beam(r, want, vocab)
    r8 = tb.beam_step(x, scores, n_out, finished=finished.to(torch.uint8), eos_id=17)
    assert all(torch.equal(a, b) for a, b in zip(r, r8))


@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("at", [0, 3, 4999, 5002])
def test_beam_step_reports_bad_logits_and_scores(tb, value, at):
    x, scores = beam_inputs(4, 3, 5003, "f32", seed=9)
    x[1, 2, at] = value
    scores[3, 1] = value
    r = tb.beam_step(x, scores, 5)
    want = plain_beam(x, scores, 5)
    assert list(want["status"]) == [0, 4, 0, 4]
    check_beam(r, want, 5003)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("vocab", [40, 9001, 70001])
def test_beam_step_ties_go_to_the_lower_index(tb, dtype, vocab):
    g = gen(3)
    x = torch.randint(-3, 4, (4, 3, vocab), device="cuda", generator=g).to(DT[dtype])
    x[1] = 2.5                                    # every token of every beam alike
    x[2, 0] = x[2, 1] = x[2, 2]                   # beams alike, scores alike below
    x[3] = torch.finfo(DT[dtype]).min             # masks of the type's lowest value
    x[3, :, 11:14] = 1.0
    scores = torch.tensor([[-1.0, -1.5, -9.0], [-2.0] * 3, [-3.0] * 3, [-1.0, -1.0, -4.0]],
                          device="cuda")
    for n_out in (1, 6, 100):
        check_beam(tb.beam_step(x, scores, n_out), plain_beam(x, scores, n_out), vocab)


def test_beam_step_orders_keys_closer_than_fp32(tb):
    """Beams whose keys differ by about 1e-9: far below a step of fp32 at this size. Row 1 is
    row 0 with one tail logit moved a little, so only its log-sum-exp differs."""
    vocab = 30000
    x, _ = beam_inputs(1, 2, vocab, "f32", seed=21)
    x = x.repeat(3, 1, 1)
    x[:, 1] = x[:, 0]
    low = int(x[0, 0].argmin())
    x[0, 1, low] = x[0, 0, low] + 6
    x[1, 0, low] = x[1, 1, low] + 6
    scores = torch.full((3, 2), -2.25, device="cuda")
    want = plain_beam(x, scores, 8)
    assert list(want["parents"][0][:2]) == [0, 1] and list(want["parents"][1][:2]) == [1, 0]
    gap = abs(want["scores"][0][0] - want["scores"][0][1])
    assert 0 < gap < 1e-7
    check_beam(tb.beam_step(x, scores, 8), want, vocab)


@pytest.mark.parametrize("batch", [3, 30, 61, 100, 149, 257])
@pytest.mark.parametrize("beams,vocab,n_out", [(31, 30000, 8), (4, 30000, 64)])
def test_beam_step_clusters_of_every_size(tb, batch, beams, vocab, n_out):
    """The second sums in 64 bits and the choice one by one, with 8, 4, 2 and 1 CTAs a prompt of
    either size: prompts with keys closer than fp32 sums tell apart and prompts that are all tied,
    among ordinary ones, so that clusters differ in whether they need help."""
    x, scores = beam_inputs(3, beams, vocab, "f16", seed=beams)
    x[0, 1] = x[0, 0]                       # keys about 1e-8 apart
    low = int(x[0, 0].argmin())
    x[0, 1, low] = x[0, 0, low] + 16
    scores[0, :2] = -0.25
    x[1] = 1.5                              # more ties than the table holds
    scores[1] = -3.0
    want = plain_beam(x, scores, n_out)
    f = want["scores"][0]
    assert (0 < -np.diff(f)).any() and (-np.diff(f)).min() < 1e-6
    kind = np.random.RandomState(batch).randint(0, 3, batch)
    kind[:3] = [2, 0, 1]
    at = torch.from_numpy(kind).cuda()
    check_beam(tb.beam_step(x[at], scores[at], n_out), {k: w[kind] for k, w in want.items()}, vocab)


def test_beam_step_large_values(tb):
    x, scores = beam_inputs(3, 2, 3001, "f32", seed=2)
    x[0] *= 1e30
    x[1, 0, 5] = 3.0e38
    x[1, 1, 6] = -3.0e38
    scores[2, 1] = -1e30
    check_beam(tb.beam_step(x, scores, 6), plain_beam(x, scores, 6), 3001)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("batch,beams,vocab,n_out", [
    (3, 8, 30000, 16), (2, 32, 20000, 64), (1, 4, 3001, 8), (2, 64, 2000, 128),
])
@pytest.mark.parametrize("offset", [-2.0 ** 12, -1e4, -3e7, 5e5])
def test_beam_step_scores_of_long_sequences(tb, offset, batch, beams, vocab, n_out, dtype):
    """Running scores far from 0, by thousands as after long sequences, and further."""
    x, scores = beam_inputs(batch, beams, vocab, dtype, seed=vocab)
    scores = scores + offset
    check_beam(tb.beam_step(x, scores, n_out), plain_beam(x, scores, n_out), vocab)


def graph_us(call, n=10):
    """The median time of a call among others, in a graph."""
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(n):
            call()
    times = []
    for _ in range(9):
        a, z = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        graph.replay()
        z.record()
        torch.cuda.synchronize()
        times.append(a.elapsed_time(z) * 1e3 / n)
    return sorted(times)[4]


@pytest.mark.parametrize("batch,beams,vocab,n_out,dtype", [
    (4, 32, 49152, 64, "f16"), (2, 32, 49152, 128, "f32"),
])
def test_beam_step_time_does_not_go_by_the_scores(tb, batch, beams, vocab, n_out, dtype):
    """What a step has to look at may not grow with the scores' distance from 0 (where the bound
    on the keys was coarse there, steps took 25 to 45 times as long)."""
    x, scores = beam_inputs(batch, beams, vocab, dtype, seed=3)
    near = graph_us(lambda: tb.beam_step(x, scores, n_out))
    far = graph_us(lambda: tb.beam_step(x, scores - 8000, n_out))
    assert far < 4 * near + 20, (near, far)


@pytest.mark.parametrize("batch", [16, 32, 64])
def test_beam_step_time_of_many_prompts(tb, batch):
    """More of the pick's clusters than find a place at once run in waves of CTAs that only wait:
    with 64 prompts steps took 2.8 times as long as with clusters that fit, with 16 1.6 times. A
    batch's step stays below that of its halves, one after the other."""
    x, scores = beam_inputs(batch, 4, 50257, "bf16", seed=3)
    whole = graph_us(lambda: tb.beam_step(x, scores, 64))
    h = batch // 2
    half = graph_us(lambda: (tb.beam_step(x[:h], scores[:h], 64),
                             tb.beam_step(x[h:], scores[h:], 64)))
    assert whole < 0.8 * half, (whole, half)


def test_beam_step_strides_alignment_and_sharing(tb):
    g = gen(8)
    base = 4 * torch.randn(4 * 3 * 5000 + 64, device="cuda", generator=g)
    scores = -torch.rand(4, 3, device="cuda", generator=g)
    for off in (0, 1, 2, 3):
        x = base[off:off + 4 * 3 * 4999].view(4, 3, 4999)
        check_beam(tb.beam_step(x, scores, 6), plain_beam(x, scores, 6), 4999)
        h = base.to(torch.float16)[off:off + 4 * 3 * 4999].view(4, 3, 4999)
        check_beam(tb.beam_step(h, scores, 6), plain_beam(h, scores, 6), 4999)
    x = base[:3 * 4 * 4999].view(3, 4, 4999).transpose(0, 1)     # beams outermost
    check_beam(tb.beam_step(x, scores, 6), plain_beam(x, scores, 6), 4999)
    x = base[:4 * 4999].view(4, 1, 4999).expand(4, 3, 4999)      # a prompt's logits shared
    check_beam(tb.beam_step(x, scores, 6), plain_beam(x, scores, 6), 4999)
    x = base[:4999 * 12].view(4999, 4, 3).permute(1, 2, 0)       # vocabulary not innermost
    check_beam(tb.beam_step(x, scores, 6), plain_beam(x, scores, 6), 4999)
    s = scores.t().contiguous().t()
    x = base[:4 * 3 * 4999].view(4, 3, 4999)
    check_beam(tb.beam_step(x, s), plain_beam(x, scores, 3), 4999)


def test_beam_step_far_rows(tb):
    """Rows whose offset passes 2^32 elements."""
    row = (1 << 31) + 8
    big = torch.empty(3 * row, dtype=torch.float16, device="cuda")
    x = big.as_strided((3, 1, 2000), (row, 2000, 1))
    x.copy_(torch.randn(3, 1, 2000, device="cuda", generator=gen(4)))
    scores = torch.zeros(3, 1, device="cuda")
    check_beam(tb.beam_step(x, scores, 4), plain_beam(x, scores, 4), 2000)


def test_beam_step_repeats_bit_for_bit_on_other_streams_and_in_graphs(tb):
    x, scores = beam_inputs(6, 8, 20000, "f32", seed=31)
    first = tb.beam_step(x, scores, 16)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    for s in (a, b):
        s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(a):
        ra = [tb.beam_step(x, scores, 16) for _ in range(3)]
    with torch.cuda.stream(b):
        rb = [tb.beam_step(x, scores, 16) for _ in range(3)]
    torch.cuda.synchronize()
    for r in ra + rb:
        assert all(torch.equal(p, q) for p, q in zip(first, r))
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        r1 = tb.beam_step(x, scores, 16)
    with torch.cuda.graph(g2):
        r2 = tb.beam_step(x, scores, 8)
    x.copy_(beam_inputs(6, 8, 20000, "f32", seed=32)[0])
    torch.cuda.synchronize()
    for s, g in ((a, g1), (b, g2)):
        with torch.cuda.stream(s):
            for _ in range(3):
                g.replay()
    torch.cuda.synchronize()
    check_beam(r1, plain_beam(x, scores, 16), 20000)
    check_beam(r2, plain_beam(x, scores, 8), 20000)


def test_beam_step_refusals(tb):
    x, scores = beam_inputs(2, 3, 50, "f32")
    for bad in (dict(n_out=0), dict(n_out=129), dict(eos_id=50)):
        with pytest.raises(RuntimeError):
            tb.beam_step(x, scores, **bad)
    with pytest.raises(RuntimeError):
        tb.beam_step(x, scores, finished=torch.zeros(2, 3, dtype=torch.bool, device="cuda"))
    with pytest.raises(ValueError):
        tb.beam_step(x, scores, eos_id=3 - 2 ** 32)
    with pytest.raises(ValueError):
        tb.beam_step(x[0], scores)
    with pytest.raises(ValueError):
        tb.beam_step(x, scores[:1])
    with pytest.raises(ValueError):
        tb.beam_step(x, scores.cpu())
    with pytest.raises(TypeError):
        tb.beam_step(x.double(), scores)
    with pytest.raises(TypeError):
        tb.beam_step(x, scores.half())
    with pytest.raises(RuntimeError):
        tb.beam_step(x[:, :1].expand(2, 65, 50), torch.zeros(2, 65, device="cuda"))
    e = tb.beam_step(x[:0], scores[:0], 4)
    assert e.scores.shape == (0, 4)


# -- the reorder of states -------------------------------------------------------------------
def plain_reorder(x, parents, lengths=None):
    """x [rows, ...] (with lengths [rows, heads, entries, dim]) after the move."""
    y = x.clone()
    b, k = parents.shape
    par = parents.cpu().tolist()
    lens = None if lengths is None else lengths.cpu().tolist()
    for p in range(b):
        for i in range(k):
            if 0 <= par[p][i] < k:
                src = x[p * k + par[p][i]]
                if lens is None:
                    y[p * k + i] = src
                else:
                    n = max(0, min(lens[p], x.shape[2]))
                    y[p * k + i, :, :n] = src[:, :n]
    return y


def random_parents(batch, beams, seed, wild=False):
    r = np.random.RandomState(seed)
    p = r.randint(0, beams, (batch, beams))
    if wild:
        p[r.rand(batch, beams) < 0.2] = -1
        p[r.rand(batch, beams) < 0.1] = beams
        p[r.rand(batch, beams) < 0.05] = -2 ** 31
        p[r.rand(batch, beams) < 0.05] = 2 ** 31 - 1
    return torch.from_numpy(p.astype(np.int32)).cuda()


def filled(shape, dtype, seed):
    n = int(np.prod(shape)) * torch.empty(0, dtype=dtype).element_size()
    raw = torch.randint(0, 256, (max(n, 1),), dtype=torch.uint8, device="cuda",
                        generator=gen(seed))
    return raw[:n].view(dtype).view(shape)


@pytest.mark.parametrize("beams", [1, 2, 3, 4, 5, 8, 11, 16, 17, 32, 33, 64])
@pytest.mark.parametrize("heads,entries,dim,dtype,major", [
    (2, 33, 64, torch.bfloat16, "head"), (3, 7, 80, torch.float32, "token"),
    (1, 1, 1, torch.uint8, "head"), (5, 19, 3, torch.int16, "token"),
    (1, 130, 5, torch.float32, "head"), (2, 9, 24, torch.float16, "token"),
])
def test_reorder_caches(tb, beams, heads, entries, dim, dtype, major):
    batch = 3
    shape = ((batch * beams, heads, entries, dim) if major == "head"
             else (batch * beams, entries, heads, dim))
    raw = [filled(shape, dtype, s) for s in (1, 2, 3)]
    states = raw if major == "head" else [x.transpose(1, 2) for x in raw]
    parents = random_parents(batch, beams, beams, wild=True)
    for lens in ([entries, entries // 2, 0], [1, entries + 5, -3]):
        lengths = torch.tensor(lens, dtype=torch.int32, device="cuda")
        want = [plain_reorder(x.view(torch.uint8) if dim == 1 else x, parents, lengths)
                for x in states]
        tb.reorder_states(states, parents, lengths)
        for x, w in zip(states, want):
            assert torch.equal(x.contiguous().view(torch.uint8), w.contiguous().view(torch.uint8))


def test_reorder_plain_states_of_several_shapes(tb):
    parents = random_parents(4, 5, 7)
    history = filled((20, 77), torch.int32, 1)
    hidden = filled((20, 3, 50), torch.float32, 2)
    odd = filled((20, 13), torch.uint8, 3)
    one = filled((20,), torch.float64, 4)
    sliced = filled((20, 9, 40), torch.int16, 5)[:, 2:7, 3:30]
    outer = filled((6, 20, 8), torch.int32, 6).transpose(0, 1)     # rows not outermost
    states = [history, hidden, odd, one, sliced, outer]
    want = [plain_reorder(x, parents) for x in states]
    tb.reorder_states(states, parents)
    for x, w in zip(states, want):
        assert torch.equal(x.contiguous().view(torch.uint8), w.contiguous().view(torch.uint8))


def test_reorder_leaves_the_rest_alone(tb):
    """What surrounds a sliced state and the entries behind the lengths keep their bits."""
    big = filled((8, 4, 50, 64), torch.bfloat16, 9)
    view = big[:, 1:3, 5:45, 8:56]
    want = big.clone()
    parents = random_parents(2, 4, 3)
    lengths = torch.tensor([17, 40], dtype=torch.int32, device="cuda")
    want[:, 1:3, 5:45, 8:56] = plain_reorder(view, parents, lengths)
    tb.reorder_states([view], parents, lengths)
    assert torch.equal(big.view(torch.int16), want.view(torch.int16))


def test_reorder_many_states_and_the_stacked_form(tb):
    x = filled((300, 6, 2, 10, 8), torch.float32, 4)
    parents = random_parents(2, 3, 5)
    lengths = torch.tensor([10, 4], dtype=torch.int32, device="cuda")
    want = torch.stack([plain_reorder(y, parents, lengths) for y in x])
    listed = x.clone()
    tb.reorder_states(list(listed), parents, lengths)
    tb.reorder_states(x, parents, lengths)
    assert torch.equal(listed.view(torch.int32), want.view(torch.int32))
    assert torch.equal(x.view(torch.int32), want.view(torch.int32))
    y = filled((5, 6, 4), torch.int32, 6)
    w = torch.stack([plain_reorder(z, parents) for z in y])
    tb.reorder_states(y, parents)
    assert torch.equal(y, w)


def test_reorder_offsets_beyond_32_bits(tb):
    """One state of 6 GB: rows, and entries within a row, lie more than 2^31 bytes apart."""
    entries = 3 << 24
    x = torch.zeros(2, 1, entries, 64, dtype=torch.uint8, device="cuda")
    for t in (0, 1, 12345, entries // 2, entries - 1):
        x[0, 0, t] = t % 251
        x[1, 0, t] = 100
    parents = torch.tensor([[1, 0]], dtype=torch.int32, device="cuda")
    tb.reorder_states([x], parents, torch.tensor([entries - 1], dtype=torch.int32, device="cuda"))
    for t in (0, 1, 12345, entries // 2):
        assert (x[1, 0, t] == t % 251).all() and (x[0, 0, t] == 100).all()
    assert (x[0, 0, -1] == (entries - 1) % 251).all() and (x[1, 0, -1] == 100).all()
    assert int(x[0, 0, 2].sum()) == 0


def test_reorder_refusals(tb):
    p = random_parents(2, 3, 1)
    x = filled((6, 2, 5, 8), torch.float32, 1)
    lens = torch.tensor([1, 2], dtype=torch.int32, device="cuda")
    for states, parents, lengths in (
            ([x[:5]], p, None), ([x.cpu()], p, None), ([x], p[0], None),
            ([x], p.long(), None), ([x[:, 0]], p, lens), ([x], p, lens[:1]),
            ([x.transpose(2, 3)], p, lens), ([x], p, lens.long()), (x[:, :, 0], p, lens)):
        with pytest.raises((TypeError, ValueError)):
            tb.reorder_states(states, parents, lengths)
    with pytest.raises(RuntimeError):
        tb.reorder_states([x[:1].expand(6, 2, 5, 8)], p, lens)
    with pytest.raises(ValueError):
        tb.reorder_states([x, x], p, lens)
    with pytest.raises(RuntimeError):
        tb.reorder_states([filled((65, 4), torch.int32, 1)], random_parents(1, 65, 1))
    tb.reorder_states([], p)
    tb.reorder_states([x[:, :, :0]], p, lens)


def test_stacks_that_overlap_are_refused(tb):
    p = random_parents(2, 3, 1)
    lens = torch.tensor([5, 4], dtype=torch.int32, device="cuda")
    z = torch.zeros(6, 4, dtype=torch.int32, device="cuda")
    x = filled((9, 2, 5, 8), torch.float32, 1)
    start = x.clone()
    for bad in (x[:6].expand(3, 6, 2, 5, 8), x.unfold(0, 6, 1).permute(0, 4, 1, 2, 3),
                x.unfold(2, 4, 1)[:6].permute(3, 0, 1, 2, 4)):
        with pytest.raises(ValueError):
            tb.reorder_states(bad, p, lens)
        with pytest.raises(ValueError):
            tb.tree_accept(z, z, z - 1, torch.zeros(6, dtype=torch.int32, device="cuda"), bad)
    assert torch.equal(x.view(torch.int32), start.view(torch.int32))
    stack = filled((6, 2, 3, 5, 8), torch.float32, 2).transpose(1, 2).permute(2, 0, 1, 3, 4)
    want = torch.stack([plain_reorder(s, p, lens) for s in stack])
    tb.reorder_states(stack, p, lens)  # two states between whose heads the other's lie
    assert torch.equal(stack.contiguous().view(torch.int32), want.view(torch.int32))


def test_reorder_that_is_refused_moves_nothing(tb):
    """A state that cannot be moved, behind others that can: none of them is."""
    p = random_parents(2, 3, 1)
    lens = torch.tensor([5, 4], dtype=torch.int32, device="cuda")
    x = filled((6, 2, 5, 8), torch.float32, 1)
    y = filled((6, 3, 5, 16), torch.bfloat16, 2)
    start = [x.clone(), y.clone()]
    for bad, lengths in ((filled((6, 2, 9, 4), torch.float32, 3).transpose(2, 3), lens),
                         (filled((1, 2, 5, 8), torch.int16, 3).expand(6, 2, 5, 8), lens),
                         (filled((6, 7, 6, 5, 4), torch.int16, 3)[:, ::2, ::2, ::2], None),
                         (filled((6, 2, 5), torch.int16, 3), lens)):
        with pytest.raises((RuntimeError, ValueError)):
            tb.reorder_states([x, y, bad], p, lengths)
        for a, b in zip((x, y), start):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


# -- trees -----------------------------------------------------------------------------------
def chain(parents, i):
    way = [i]
    while parents[way[-1]] != -1:
        q = parents[way[-1]]
        if q < 0 or q >= way[-1]:
            return None
        way.append(q)
    return way


def random_trees(batch, nodes, seed, wild=False):
    r = np.random.RandomState(seed)
    p = np.full((batch, nodes), -1)
    for b in range(batch):
        for i in range(1, nodes):
            p[b, i] = int(i * r.rand() ** 2)
        if r.rand() < 0.4:
            p[b, r.randint(1, nodes + 1):] = -2
        if wild:
            p[b, r.rand(nodes) < 0.1] = -1
            p[b, r.rand(nodes) < 0.1] = -7
            p[b, r.rand(nodes) < 0.05] = nodes + 3
            p[b, r.rand(nodes) < 0.05] = 2 ** 31 - 1
            p[b, r.rand(nodes) < 0.05] = nodes - 1
    return torch.from_numpy(p.astype(np.int32)).cuda()


def plain_attention(q, k, v, lengths, parents, scale, tol=True):
    """(out, tolerance) in 64 bits."""
    b, n, hq, d = q.shape
    hk, entries = k.shape[1], k.shape[2]
    out = torch.zeros(b, n, hq, d, dtype=torch.float64, device="cuda")
    err = torch.zeros_like(out)
    h = torch.finfo(q.dtype).eps / 2
    par, lens = parents.cpu().tolist(), lengths.cpu().tolist()
    for i in range(b):
        if lens[i] < 0:
            continue
        for j in range(n):
            way = chain(par[i], j)
            if way is None or lens[i] + j >= entries:
                continue
            at = list(range(lens[i])) + sorted(lens[i] + w for w in way)
            at = torch.tensor(at, device="cuda")
            kk, vv = k[i][:, at].double(), v[i][:, at].double()
            qq = q[i, j].double().view(hk, hq // hk, d)
            x = scale * torch.einsum("hgd,htd->hgt", qq, kk)
            s_max = abs(scale) * torch.einsum("hgd,htd->hgt", qq.abs(), kk.abs()).amax(-1)
            p = torch.softmax(x, -1)
            o = torch.einsum("hgt,htd->hgd", p, vv)
            a = torch.einsum("hgt,htd->hgd", p, vv.abs())
            s_max = s_max[..., None]
            m = len(at)
            e = h * o.abs() + 2 * h * a + 2 * a * (d + 4) * 2 * U * s_max
            e = e + (m / 8 + 16) * 2 * U * a + 2 * (4 + 6 * s_max) * U * a
            out[i, j] = o.reshape(hq, d)
            err[i, j] = e.reshape(hq, d)
    return out, err + 1e-30


def check_attention(got, q, k, v, lengths, parents, scale=None):
    want, tol = plain_attention(q, k, v, lengths, parents,
                                q.shape[-1] ** -0.5 if scale is None else scale)
    # half a step of the smallest subnormal
    tol = tol + (2.0 ** -25 if q.dtype == torch.float16 else 0)
    d = (got.double() - want).abs()
    assert torch.isfinite(got).all()
    assert (d <= tol).all(), (d - tol).max().item()


def attention_inputs(batch, nodes, heads, kv_heads, dim, entries, dtype, seed, token_major=False):
    g = gen(seed)
    dt = DT[dtype]
    q = torch.randn(batch, nodes, heads, dim, device="cuda", generator=g).to(dt)
    shape = (batch, entries, kv_heads, dim) if token_major else (batch, kv_heads, entries, dim)
    k = torch.randn(shape, device="cuda", generator=g).to(dt)
    v = torch.randn(shape, device="cuda", generator=g).to(dt)
    if token_major:
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    return q, k, v


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("nodes,heads,kv_heads,dim", [
    (1, 1, 1, 64), (1, 14, 2, 64), (2, 15, 5, 64), (5, 8, 8, 128), (26, 14, 2, 64),
    (64, 8, 2, 128), (33, 4, 1, 80), (17, 6, 3, 8), (64, 12, 1, 64), (7, 9, 3, 104),
    (3, 64, 1, 16), (64, 64, 1, 128), (64, 7, 7, 72), (2, 300, 1, 16), (3, 257, 1, 64),
])
def test_tree_attention_matches_the_definition(tb, nodes, heads, kv_heads, dim, dtype):
    lens = [0, 1, 63, 64, 65, 200]
    entries = 200 + nodes
    q, k, v = attention_inputs(6, nodes, heads, kv_heads, dim, entries, dtype, nodes + dim,
                               token_major=nodes % 2 == 0)
    lengths = torch.tensor(lens, dtype=torch.int32, device="cuda")
    parents = random_trees(6, nodes, nodes)
    out = tb.tree_attention(q, k, v, lengths, parents)
    check_attention(out, q, k, v, lengths, parents)


@pytest.mark.parametrize("length", [0, 1, 2, 127, 128, 129, 1000, 5000])
def test_tree_attention_lengths(tb, length):
    q, k, v = attention_inputs(2, 9, 4, 2, 64, length + 20, "bf16", length)
    lengths = torch.tensor([length, max(0, length - 1)], dtype=torch.int32, device="cuda")
    parents = random_trees(2, 9, length)
    check_attention(tb.tree_attention(q, k, v, lengths, parents), q, k, v, lengths, parents)


def test_tree_attention_ragged_batch(tb):
    """Many sequences of very different lengths, some empty, some absent."""
    r = np.random.RandomState(3)
    batch = 37
    lens = (r.rand(batch) ** 4 * 3000).astype(np.int32)
    lens[5] = -1
    lens[9] = -2 ** 31
    lens[11] = 0
    q, k, v = attention_inputs(batch, 6, 4, 2, 64, 3010, "f16", 8)
    lengths = torch.from_numpy(lens).cuda()
    parents = random_trees(batch, 6, 4, wild=True)
    check_attention(tb.tree_attention(q, k, v, lengths, parents), q, k, v, lengths, parents)


@pytest.mark.parametrize("batch,length", [(296, 127), (592, 63), (592, 127), (300, 200),
                                          (700, 90), (149, 500)])
def test_tree_attention_many_sequences(tb, batch, length):
    """More sequences than SMs: a worker goes through several of them, whole and in parts."""
    q, k, v = attention_inputs(batch, 1, 2, 1, 64, length + 1, "bf16", batch)
    lengths = torch.full((batch,), length, dtype=torch.int32, device="cuda")
    lengths[::7] = length // 2
    parents = torch.full((batch, 1), -1, dtype=torch.int32, device="cuda")
    check_attention(tb.tree_attention(q, k, v, lengths, parents), q, k, v, lengths, parents)


def test_tree_attention_unread_entries_may_hold_anything(tb):
    nodes = 12
    q, k, v = attention_inputs(4, nodes, 6, 2, 64, 160, "bf16", 5)
    lengths = torch.tensor([0, 50, 100, 155], dtype=torch.int32, device="cuda")
    parents = random_trees(4, nodes, 5, wild=True)
    par, lens = parents.cpu().tolist(), lengths.cpu().tolist()
    for b in range(4):
        for t in range(lens[b], 160):
            j = t - lens[b]
            if j >= nodes or chain(par[b], j) is None:
                k[b, :, t] = [math.nan, math.inf, -math.inf][t % 3]
                v[b, :, t] = [math.inf, math.nan, -math.inf][t % 3]
    check_attention(tb.tree_attention(q, k, v, lengths, parents), q, k, v, lengths, parents)


def test_tree_attention_near_the_caches_end(tb):
    """Slots past the last entry are unused: their outputs are 0."""
    q, k, v = attention_inputs(3, 10, 4, 4, 64, 64, "bf16", 6)
    lengths = torch.tensor([60, 64, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    parents = torch.tensor([[-1] + list(range(9))] * 3, dtype=torch.int32, device="cuda")
    out = tb.tree_attention(q, k, v, lengths, parents)
    assert (out[0, 4:] == 0).all() and (out[1:] == 0).all()
    check_attention(out, q, k, v, lengths, parents)


def test_tree_attention_large_scores(tb):
    """Scores of some hundreds, the largest last and first: the running maximum moves."""
    q, k, v = attention_inputs(2, 4, 4, 2, 64, 700, "f16", 7)
    k[0, :, :600] *= torch.linspace(0.1, 6, 600, device="cuda").half()[None, :, None]
    k[1, :, :600] *= torch.linspace(6, 0.1, 600, device="cuda").half()[None, :, None]
    lengths = torch.tensor([600, 601], dtype=torch.int32, device="cuda")
    parents = random_trees(2, 4, 1)
    for scale in (0.5, -0.25, 0.0, 2.0):
        out = tb.tree_attention(q, k, v, lengths, parents, scale)
        check_attention(out, q, k, v, lengths, parents, scale)


def test_tree_attention_all_keys_alike(tb):
    q, k, v = attention_inputs(1, 3, 2, 1, 128, 5000, "bf16", 17)
    k[:] = k[:, :, :1]
    lengths = torch.tensor([4990], dtype=torch.int32, device="cuda")
    parents = torch.tensor([-1, 0, 0], dtype=torch.int32, device="cuda")
    out = tb.tree_attention(q, k, v, lengths, parents)
    check_attention(out, q, k, v, lengths, parents.expand(1, 3))


def test_tree_attention_strides_and_shared_trees(tb):
    q, k, v = attention_inputs(3, 8, 6, 2, 64, 90, "bf16", 12)
    lengths = torch.tensor([80, 3, 41], dtype=torch.int32, device="cuda")
    parents = random_trees(1, 8, 2)[0]
    want = tb.tree_attention(q, k, v, lengths, parents)
    check_attention(want, q, k, v, lengths, parents.expand(3, 8))
    wide_q = torch.zeros(3, 8, 6, 96, dtype=q.dtype, device="cuda")
    wide_q[..., 16:80] = q
    big = torch.full((3, 95, 2, 2, 80), math.nan, dtype=q.dtype, device="cuda")
    big[:, 2:92, 0, :, 8:72] = k.transpose(1, 2)      # keys and values in one buffer
    big[:, 2:92, 1, :, 8:72] = v.transpose(1, 2)
    kk, vv = big[:, 2:92, 0, :, 8:72].transpose(1, 2), big[:, 2:92, 1, :, 8:72].transpose(1, 2)
    assert torch.equal(want, tb.tree_attention(wide_q[..., 16:80], kk, vv, lengths, parents))
    assert torch.equal(want, tb.tree_attention(wide_q[..., 15:79].roll(1, -1)[..., :64].copy_(q),
                                               kk, vv, lengths, parents))
    every = parents.expand(3, 8).contiguous().t().contiguous().t()
    assert torch.equal(want, tb.tree_attention(q, kk, vv, lengths, every))


def test_tree_attention_far_entries(tb):
    """A cache whose heads lie more than 2^31 elements apart."""
    entries = (1 << 25) + 8
    k = torch.zeros(1, 2, entries, 64, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros(1, 2, entries, 64, dtype=torch.bfloat16, device="cuda")
    q, sk, sv = attention_inputs(1, 4, 4, 2, 64, 300, "bf16", 3)
    k[:, :, :300], v[:, :, :300] = sk, sv
    lengths = torch.tensor([290], dtype=torch.int32, device="cuda")
    parents = random_trees(1, 4, 9)
    check_attention(tb.tree_attention(q, k, v, lengths, parents), q, sk, sv, lengths, parents)
    # and one token behind 2^25 entries of zeros: with q = 0 every key weighs the same
    lengths = torch.tensor([entries - 4], dtype=torch.int32, device="cuda")
    v[:, :, -4:] = 64.0
    v[:, :, :300] = 0
    out = tb.tree_attention(torch.zeros_like(q), k, v, lengths, parents[:, :4])
    depth = torch.tensor([len(chain(parents[0].tolist(), j) or []) for j in range(4)])
    want = 64.0 * depth / (entries - 4 + depth)
    got = out[0, :, 0, 0].double().cpu()
    assert ((got - want).abs() <= want * 2.0 ** -7 + 1e-12).all(), (got, want)


def test_tree_attention_streams_and_graphs(tb):
    q, k, v = attention_inputs(5, 11, 8, 2, 128, 2100, "bf16", 13)
    lengths = torch.tensor([2000, 5, 700, 1024, 0], dtype=torch.int32, device="cuda")
    parents = random_trees(5, 11, 13)
    first = tb.tree_attention(q, k, v, lengths, parents)
    check_attention(first, q, k, v, lengths, parents)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs += [tb.tree_attention(q, k, v, lengths, parents) for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(first, o) for o in outs)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    res = []
    for g in graphs:
        with torch.cuda.graph(g):
            res.append(tb.tree_attention(q, k, v, lengths, parents))
    q2, k2, v2 = attention_inputs(5, 11, 8, 2, 128, 2100, "bf16", 14)
    q.copy_(q2), k.copy_(k2), v.copy_(v2)
    lengths.copy_(torch.tensor([1, 2000, 65, 0, 333], dtype=torch.int32))
    torch.cuda.synchronize()
    for s, g in zip(streams, graphs):
        with torch.cuda.stream(s):
            for _ in range(3):
                g.replay()
    torch.cuda.synchronize()
    assert torch.equal(res[0], res[1])
    check_attention(res[0], q, k, v, lengths, parents)


@pytest.mark.parametrize("batch,nodes,heads,kv_heads,dim,length", [
    (12, 9, 14, 2, 64, 3000), (6, 26, 32, 8, 128, 1500), (8, 1, 32, 8, 128, 2500),
    (2, 64, 16, 4, 128, 2000),
])
def test_tree_attention_repeats_bit_for_bit(tb, batch, nodes, heads, kv_heads, dim, length):
    """Many runs on ranges of several tiles: what the kernel's warps wait for must not depend
    on how fast each of them is."""
    q, k, v = attention_inputs(batch, nodes, heads, kv_heads, dim, length + nodes, "bf16", 40)
    lengths = torch.randint(0, length, (batch,), device="cuda", generator=gen(2)).int()
    parents = random_trees(batch, nodes, 6)
    first = tb.tree_attention(q, k, v, lengths, parents)
    check_attention(first, q, k, v, lengths, parents)
    for _ in range(150):
        assert torch.equal(first, tb.tree_attention(q, k, v, lengths, parents))


def test_tree_attention_refusals(tb):
    q, k, v = attention_inputs(2, 4, 4, 2, 64, 40, "bf16", 1)
    lengths = torch.tensor([3, 4], dtype=torch.int32, device="cuda")
    parents = random_trees(2, 4, 1)
    for a in ((q[0], k, v, lengths, parents), (q.float(), k, v, lengths, parents),
              (q.half(), k, v, lengths, parents), (q, k[:1], v, lengths, parents),
              (q, k, v[:, :, :30], lengths, parents), (q, k, v, lengths[:1], parents),
              (q, k, v, lengths.long(), parents), (q, k, v, lengths, parents[:, :3]),
              (q, k, v, lengths, parents[0, :3]), (q, k.cpu(), v, lengths, parents),
              (q, k, v, lengths, parents.cpu()),
              (q[..., :60], k[..., 1:61], v[..., 1:61], lengths, parents)):
        with pytest.raises((TypeError, ValueError, RuntimeError)):
            tb.tree_attention(*a)
    for a in ((q[:, :, :3], k, v), (q[..., :60], k[..., :60], v[..., :60]),
              (q[:, :1].expand(2, 65, 4, 64), k, v)):
        n = a[0].shape[1]
        with pytest.raises(RuntimeError):
            tb.tree_attention(*a, lengths, random_trees(2, n, 1))
    with pytest.raises(RuntimeError):  # one cache for all sequences
        tb.tree_attention(q, k[:1].expand(2, 2, 40, 64), v, lengths, parents)
    odd = torch.zeros(2, 2, 40, 68, dtype=torch.bfloat16, device="cuda")[..., :64]
    with pytest.raises(ValueError):
        tb.tree_attention(q, odd, v, lengths, parents)
    assert tb.tree_attention(q[:0], k[:0], v[:0], lengths[:0], parents[:0]).shape == (0, 4, 4, 64)


def plain_accept(sampled, tokens, parents, lengths, caches, entries):
    sampled, tokens = sampled.cpu().tolist(), tokens.cpu().tolist()
    parents, lens = parents.cpu().tolist(), lengths.cpu().tolist()
    out = [x.clone() for x in caches]
    paths, nxt = [], []
    for b in range(len(tokens)):
        n = len(tokens[b])
        used = [lens[b] >= 0 and lens[b] + j < entries and chain(parents[b], j) is not None
                for j in range(n)]
        way = [0] if used[0] and parents[b][0] == -1 else []
        while way:
            fits = [j for j in range(n) if used[j] and parents[b][j] == way[-1]
                    and tokens[b][j] == sampled[b][way[-1]]]
            if not fits:
                break
            way.append(fits[0])
        for x, y in zip(caches, out):
            for r, j in enumerate(way):
                y[b, :, lens[b] + r] = x[b, :, lens[b] + j]
        paths.append(way)
        nxt.append(sampled[b][way[-1]] if way else -1)
    return paths, nxt, out


def check_accept(r, want, lengths, nodes):
    paths, nxt, _ = want
    counts = [len(p) for p in paths]
    assert r.counts.tolist() == counts and r.next_tokens.tolist() == nxt
    assert r.path.tolist() == [p + [-1] * (nodes - len(p)) for p in paths]
    assert r.lengths.tolist() == [a + c for a, c in zip(lengths.tolist(), counts)]


@pytest.mark.parametrize("nodes", [1, 2, 5, 26, 63, 64])
@pytest.mark.parametrize("heads,dim,dtype,token_major", [
    (2, 64, torch.bfloat16, False), (3, 5, torch.float32, True), (1, 1, torch.uint8, False),
    (8, 128, torch.float16, True),
])
def test_tree_accept_matches_the_walk(tb, nodes, heads, dim, dtype, token_major):
    batch, entries = 9, 150
    r = np.random.RandomState(nodes)
    tokens = torch.from_numpy(r.randint(0, 3, (batch, nodes)).astype(np.int32)).cuda()
    sampled = torch.from_numpy(r.randint(0, 3, (batch, nodes)).astype(np.int32)).cuda()
    parents = random_trees(batch, nodes, nodes, wild=True)
    parents[0, 0] = -2
    parents[1:4, 0] = -1
    lens = [7, 0, 80, 20, 149, 145, -1, 150, 30]
    lengths = torch.tensor(lens, dtype=torch.int32, device="cuda")
    shape = (batch, entries, heads, dim) if token_major else (batch, heads, entries, dim)
    raw = [filled(shape, dtype, s) for s in (1, 2)]
    caches = [x.transpose(1, 2) for x in raw] if token_major else raw
    bits = [c.clone() for c in caches]
    want = plain_accept(sampled, tokens, parents, lengths, bits, entries)
    got = tb.tree_accept(sampled, tokens, parents, lengths, caches)
    check_accept(got, want, lengths, nodes)
    for x, w in zip(caches, want[2]):
        assert torch.equal(x.contiguous().view(torch.uint8), w.contiguous().view(torch.uint8))
    assert lengths.tolist() == lens
    alone = tb.tree_accept(sampled, tokens, parents, lengths.clamp(-1, 80))
    check_accept(alone, plain_accept(sampled, tokens, parents, lengths.clamp(-1, 80), [], 1 << 40),
                 lengths.clamp(-1, 80), nodes)


def test_tree_accept_long_path_and_shared_tree(tb):
    """A chain whose every second slot is taken: every accepted entry moves."""
    nodes = 64
    parents = torch.tensor([-1] + [max(0, j - 2 if j % 2 == 0 else j - 1) for j in range(1, nodes)],
                           dtype=torch.int32, device="cuda")
    tokens = torch.arange(nodes, dtype=torch.int32, device="cuda").repeat(3, 1)
    sampled = torch.full((3, nodes), -9, dtype=torch.int32, device="cuda")
    sampled[:, 0:62:2] = torch.arange(2, nodes, 2, dtype=torch.int32, device="cuda")
    x = filled((40, 3, 2, 100, 64), torch.bfloat16, 3)
    lengths = torch.tensor([0, 36, 10], dtype=torch.int32, device="cuda")
    caches = list(x.clone())
    want = plain_accept(sampled, tokens, parents.expand(3, nodes), lengths, caches, 100)
    assert [len(p) for p in want[0]] == [32, 32, 32]
    check_accept(tb.tree_accept(sampled, tokens, parents, lengths, x), want, lengths, nodes)
    assert torch.equal(x.view(torch.int16), torch.stack(want[2]).view(torch.int16))


def test_tree_accept_strided_samples_streams_and_graphs(tb):
    batch, nodes = 4, 10
    r = np.random.RandomState(5)
    wide = torch.from_numpy(r.randint(0, 2, (batch, nodes, 12)).astype(np.int32)).cuda()
    tokens = torch.from_numpy(r.randint(0, 2, (batch, nodes)).astype(np.int32)).cuda()
    parents = random_trees(batch, nodes, 3)
    lengths = torch.tensor([5, 6, 7, 0], dtype=torch.int32, device="cuda")
    x = filled((2, batch, 2, 40, 16), torch.bfloat16, 3)
    start = x.clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    want = plain_accept(wide[..., 0], tokens, parents, lengths, list(start), 40)
    with torch.cuda.stream(s):
        got = tb.tree_accept(wide[..., 0], tokens, parents, lengths, x)
    torch.cuda.synchronize()
    check_accept(got, want, lengths, nodes)
    assert torch.equal(x.view(torch.int16), torch.stack(want[2]).view(torch.int16))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = tb.tree_accept(wide[..., 0], tokens, parents, lengths, x)
    x.copy_(start)
    tokens.copy_(1 - tokens)
    want = plain_accept(wide[..., 0], tokens, parents, lengths, list(start), 40)
    g.replay()
    torch.cuda.synchronize()
    check_accept(got, want, lengths, nodes)
    assert torch.equal(x.view(torch.int16), torch.stack(want[2]).view(torch.int16))


def test_tree_accept_refusals(tb):
    z = torch.zeros(2, 4, dtype=torch.int32, device="cuda")
    lens = torch.zeros(2, dtype=torch.int32, device="cuda")
    c = filled((2, 2, 9, 8), torch.float32, 1)
    for a in ((z[:1], z, z, lens), (z, z.long(), z, lens), (z, z, z[:, :3], lens),
              (z, z, z, lens[:1]), (z.cpu(), z, z, lens), (z, z, z, lens, [c[:1]]),
              (z, z, z, lens, [c[:, 0]]), (z, z, z, lens, [c, c[:, :, :8]]),
              (z, z, z, lens, [c.cpu()]), (z, z, z, lens, [c, c]),
              (z, z, z, lens, [c[:, :, :0]])):
        with pytest.raises((TypeError, ValueError)):
            tb.tree_accept(*a)
    w = torch.zeros(2, 65, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError):
        tb.tree_accept(w, w, w, lens)


def test_tree_accept_refuses_an_empty_cache_among_others(tb):
    z = torch.zeros(2, 4, dtype=torch.int32, device="cuda")
    lens = torch.zeros(2, dtype=torch.int32, device="cuda")
    c = filled((2, 2, 9, 8), torch.float32, 1)
    for caches in ([c, c[:, :, :0]], [c[:, :, :0], c], c[None, :, :, :0]):
        with pytest.raises(ValueError):
            tb.tree_accept(z, z, z, lens, caches)
    none = tb.tree_accept(z, z, z - 1, lens, c[None][:0])  # of no layers: no cache
    assert none.counts.tolist() == [1, 1]


def test_outputs_are_ordinary_tensors(tb):
    """Saved and loaded together, copied, changed in place and used in autograd."""
    x, scores = beam_inputs(2, 3, 50, "f32")
    z = torch.zeros(2, 4, dtype=torch.int32, device="cuda")
    for r in (tb.beam_step(x.requires_grad_(), scores), tb.tree_accept(z, z, z - 1, z[:, 0])):
        f = io.BytesIO()
        torch.save(list(r), f)
        f.seek(0)
        for a, b, c in zip(r, torch.load(f), copy.deepcopy(list(r))):
            assert a.dtype == b.dtype and torch.equal(a, b) and torch.equal(a, c)
            assert not a.requires_grad
        others = [t.clone() for t in r[1:]]
        r[0].fill_(1)
        assert all(torch.equal(a, b) for a, b in zip(others, r[1:]))
    step = tb.beam_step(x, scores)
    (step.scores.requires_grad_() * 2).sum().backward()
    assert (step.scores.grad == 2).all()
    with torch.inference_mode():
        tb.beam_step(x, scores).scores.add_(1)


# -- together --------------------------------------------------------------------------------
def test_beam_search_with_a_cache(tb):
    """Eight steps of a beam search over a toy model whose logits depend on the whole cached
    history; the winners have to be those of a search that keeps token lists on the host."""
    batch, beams, vocab, dim, steps, eos = 3, 4, 500, 16, 8, 7
    g = gen(77)
    embed = torch.randn(vocab, dim, device="cuda", generator=g, dtype=torch.float64)
    head = torch.randn(dim, vocab, device="cuda", generator=g, dtype=torch.float64)
    decay = 0.9 ** torch.arange(steps + 1, device="cuda", dtype=torch.float64)

    def logits_of(tokens):  # [rows, n] -> [rows, vocab], float32 as a model's output
        e = embed[tokens] * decay[:tokens.shape[1], None]
        return (torch.sin(e.sum(1)) @ head).float()

    rows = batch * beams
    cache = torch.full((rows, 1, steps + 1, dim), math.nan, dtype=torch.float64, device="cuda")
    history = torch.full((rows, steps + 1), -1, dtype=torch.int32, device="cuda")
    start = torch.arange(batch, device="cuda", dtype=torch.int32).repeat_interleave(beams)
    history[:, 0] = start
    cache[:, 0, 0] = embed[start.long()]
    scores = torch.full((batch, beams), -math.inf, device="cuda")
    scores[:, 0] = 0
    finished = torch.zeros(batch, beams, dtype=torch.bool, device="cuda")
    host = [[(0.0, [b], False)] + [(-math.inf, [b], False)] * (beams - 1) for b in range(batch)]
    for n in range(1, steps + 1):
        state = torch.sin((cache[:, 0, :n] * decay[:n, None]).sum(1))
        logits = (state @ head).float().view(batch, beams, vocab)
        step = tb.beam_step(logits, scores, finished=finished, eos_id=eos)
        assert (step.status == 0).all()
        lengths = torch.full((batch,), n, dtype=torch.int32, device="cuda")
        tb.reorder_states([cache], step.parents, lengths)
        tb.reorder_states([history], step.parents)
        history[:, n] = step.tokens.view(-1)
        cache[:, 0, n] = embed[step.tokens.view(-1).long()]
        scores, finished = step.scores, step.finished
        for b in range(batch):
            toks = torch.tensor([t for _, t, _ in host[b]], device="cuda")
            lg = logits_of(toks)[None]
            sc = torch.tensor([[s for s, _, _ in host[b]]], device="cuda")
            fin = torch.tensor([[f for _, _, f in host[b]]], device="cuda")
            w = plain_beam(lg, sc, beams, fin, eos)
            host[b] = [(float(scores[b, j]), host[b][p][1] + [t], bool(f)) for j, (p, t, f) in
                       enumerate(zip(w["parents"][0].tolist(), w["tokens"][0].tolist(),
                                     w["finished"][0].tolist()))]
            assert history[b * beams:(b + 1) * beams, :n + 1].tolist() == [t for _, t, _ in host[b]]
            assert np.allclose(step.scores[b].cpu().numpy(), w["scores"][0], rtol=0, atol=1e-4)


def test_drafted_decoding_with_the_sampler(tb):
    """Six steps of drafted decoding of a toy attention model: tree_attention over the cache,
    Sampler on every slot's logits, tree_accept on its outcomes. The caches have to hold the
    keys and values of exactly the emitted tokens, and every emitted token has to be the
    model's (greedy) choice after its prefix by the definition in 64 bits."""
    from tabby_b200 import SamplingParams
    from tabby_b200._lib import OUTCOME_DTYPE
    from tabby_b200.sampler import params_array

    batch, nodes, heads, kv_heads, dim, vocab, steps = 3, 7, 4, 2, 32, 200, 6
    entries, g = 64, gen(5)

    def mat(*shape, by):
        return (torch.randn(*shape, device="cuda", generator=g) * by).to(torch.bfloat16)

    emb, wq = mat(vocab, 64, by=1), mat(64, heads * dim, by=0.2)
    wk, wv = mat(64, kv_heads * dim, by=0.2), mat(64, kv_heads * dim, by=0.2)
    head = torch.randn(heads * dim, vocab, device="cuda", generator=g)
    k = torch.zeros(batch, kv_heads, entries, dim, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    parents = torch.tensor([-1, 0, 0, 1, 1, 2, 3], dtype=torch.int32, device="cuda")
    lengths = torch.zeros(batch, dtype=torch.int32, device="cuda")
    root = torch.arange(batch, dtype=torch.int32, device="cuda")
    sampler = tb.Sampler(0, max_rows=batch * nodes, max_vocab=vocab)
    p = params_array(SamplingParams(0.0, 1, 1.0), batch * nodes)
    pd = torch.from_numpy(p.view(np.uint8)).cuda()
    ud = torch.zeros(batch * nodes, dtype=torch.float64, device="cuda")
    out = torch.zeros(batch * nodes * OUTCOME_DTYPE.itemsize, dtype=torch.uint8, device="cuda")
    texts = [[b] for b in range(batch)]  # emitted tokens, the root last
    r = np.random.RandomState(1)
    accepted = 0

    def model(tokens):  # logits after the last token of a prefix, with the kernel's bounds
        x = emb[torch.tensor(tokens, device="cuda")]
        kk, vv = (x @ wk).view(1, -1, kv_heads, dim), (x @ wv).view(1, -1, kv_heads, dim)
        q = (x[-1:] @ wq).view(1, 1, heads, dim)
        n = len(tokens)
        o, tol = plain_attention(q, kk.transpose(1, 2), vv.transpose(1, 2),
                                 torch.tensor([n - 1]), torch.tensor([[-1]]), dim ** -0.5)
        o, tol = o.view(-1), tol.view(-1)
        return o @ head.double(), tol @ head.double().abs() + 1e-3

    for _ in range(steps):
        tokens = torch.from_numpy(r.randint(0, vocab, (batch, nodes)).astype(np.int32)).cuda()
        tokens[:, 0] = root
        for b in range(batch):  # drafts that a good drafter would make: the model's choices
            first = int(model(texts[b])[0].argmax())
            tokens[b, 2 if b == 1 else 1] = first
            if b != 2:
                second = int(model(texts[b] + [first])[0].argmax())
                tokens[b, 5 if b == 1 else 4] = second
        x = emb[tokens.long()]
        at = lengths.long()[:, None] + torch.arange(nodes, device="cuda")
        rows = torch.arange(batch, device="cuda")[:, None]
        k[rows, :, at] = (x @ wk).view(batch, nodes, kv_heads, dim)
        v[rows, :, at] = (x @ wv).view(batch, nodes, kv_heads, dim)
        o = tb.tree_attention((x @ wq).view(batch, nodes, heads, dim), k, v, lengths, parents)
        logits = o.view(batch * nodes, -1).float() @ head
        sampler.sample_rows_async(logits, pd, ud, out)
        sampled = out.view(torch.int32).view(batch, nodes, 12)[..., 0]
        step = tb.tree_accept(sampled, tokens, parents, lengths, [k, v])
        for b in range(batch):
            path = [j for j in step.path[b].tolist() if j >= 0]
            accepted += len(path) - 1
            texts[b] += [int(tokens[b, j]) for j in path[1:]] + [int(step.next_tokens[b])]
        lengths, root = step.lengths, step.next_tokens
    sampler.close()
    assert accepted >= batch * steps // 2
    for b in range(batch):
        n = int(lengths[b])
        assert n == len(texts[b]) - 1
        x = emb[torch.tensor(texts[b][:-1], device="cuda")]
        assert torch.equal(k[b, :, :n], (x @ wk).view(n, kv_heads, dim).transpose(0, 1))
        assert torch.equal(v[b, :, :n], (x @ wv).view(n, kv_heads, dim).transpose(0, 1))
        for i in range(1, len(texts[b])):
            logits, tol = model(texts[b][:i])
            best = int(logits.argmax())
            got = texts[b][i]
            assert got == best or logits[best] - logits[got] <= tol[best] + tol[got]


FIRST_CAPTURE = """
import torch
import tabby_b200 as tb

g = torch.Generator(device="cuda").manual_seed(1)
x = torch.randn(2, 4, 9000, device="cuda", generator=g)
s = torch.zeros(2, 4, device="cuda")
q = torch.randn(2, 5, 8, 64, device="cuda", generator=g).bfloat16()
kv = torch.randn(2, 2, 2, 300, 64, device="cuda", generator=g).bfloat16()
lengths = torch.tensor([200, 7], dtype=torch.int32, device="cuda")
tree = torch.tensor([-1, 0, 0, 1, 1], dtype=torch.int32, device="cuda")
tokens = torch.tensor([[9, 1, 2, 3, 4]] * 2, dtype=torch.int32, device="cuda")
sampled = torch.tensor([[2, 0, 0, 0, 5], [1, 4, 0, 0, 6]], dtype=torch.int32, device="cuda")
state = torch.arange(8 * 6, device="cuda").view(8, 6)
kv2, state2 = kv.clone(), state.clone()


def run(kv, state):
    beams = tb.beam_step(x, s)
    tb.reorder_states([state], beams.parents)
    out = tb.tree_attention(q, kv[0], kv[1], lengths, tree)
    return (*beams, out, *tb.tree_accept(sampled, tokens, tree, lengths, kv), kv, state)


graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = run(kv, state)
graph.replay()
want = run(kv2, state2)
assert all(torch.equal(a, b) for a, b in zip(got, want))
print("same")
"""


def test_first_calls_captured(tb):
    """A process whose first calls of all are captured into a graph."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    p = subprocess.run([sys.executable, "-c", FIRST_CAPTURE], cwd=root, capture_output=True,
                       text=True, timeout=240)
    assert p.returncode == 0 and "same" in p.stdout, p.stderr[-2000:]


def test_calls_side_by_side(tb):
    """All operators at once on streams of their own, with other work between."""
    x, scores = beam_inputs(8, 4, 30000, "bf16", seed=3)
    q, k, v = attention_inputs(4, 9, 8, 2, 64, 900, "bf16", 4)
    lengths = torch.tensor([800, 3, 500, 64], dtype=torch.int32, device="cuda")
    parents = random_trees(4, 9, 5)
    state = filled((32, 2, 40, 64), torch.bfloat16, 6)
    moves = random_parents(8, 4, 7)
    want_beam, want_tree = tb.beam_step(x, scores, 8), tb.tree_attention(q, k, v, lengths, parents)
    want_state = state.clone()
    for _ in range(5):
        want_state = plain_reorder(want_state, moves)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    beams, trees = [], []
    for _ in range(5):
        with torch.cuda.stream(streams[0]):
            beams.append(tb.beam_step(x, scores, 8))
        with torch.cuda.stream(streams[1]):
            trees.append(tb.tree_attention(q, k, v, lengths, parents))
        with torch.cuda.stream(streams[2]):
            tb.reorder_states([state], moves)
    torch.cuda.synchronize()
    for r in beams:
        assert all(torch.equal(a, b) for a, b in zip(want_beam, r))
    assert all(torch.equal(want_tree, o) for o in trees)
    assert torch.equal(state.view(torch.int16), want_state.view(torch.int16))


def test_tensors_on_a_device_that_is_not_current(tb):
    if torch.cuda.device_count() < 2:
        pytest.skip("one GPU")
    x, scores = beam_inputs(2, 3, 400, "f32")
    want = tb.beam_step(x, scores, 6)
    got = tb.beam_step(x.to("cuda:1"), scores.to("cuda:1"), 6)
    assert torch.cuda.current_device() == 0
    assert all(torch.equal(a, b.to("cuda:0")) for a, b in zip(want, got))
