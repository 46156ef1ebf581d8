"""Beam selection and state reordering on the GPU against plain 64-bit / integer code.

The selection is checked by value: the scores are within the rounding of their 32-bit
arithmetic of the 64-bit ones, and the chosen (beam, token) pairs equal the 64-bit choice
wherever neighbouring candidates lie further apart than that; on logits whose scores are
exact in 32 bits (zero normaliser spread, integer scores) ties must go to the lowest index.
"""
import pytest
import torch

import silogic_b200 as S
from silogic_b200 import _hard, _soft

pytestmark = pytest.mark.gpu
dev = "cuda"
NEG = -float("inf")


def _reference(x, scores, finished, eos, width):
    """Sorted (value, flat index) of every candidate in 64 bits, best first."""
    B, k = scores.shape
    V = x.shape[-1]
    x = x.double().view(B, k, V).clone()
    x[torch.isnan(x)] = NEG
    x = x.clamp(max=torch.finfo(torch.float32).max)
    m = x.amax(2, keepdim=True)
    d = torch.where(m > NEG, x - m, NEG)
    c = d - torch.exp(d).sum(2, keepdim=True).log() + scores.double()[:, :, None]
    c = torch.where(m > NEG, c, NEG)
    if finished is not None:
        only = torch.full_like(c, NEG)
        only[:, :, eos] = scores.double()
        c = torch.where(finished[:, :, None], only, c)
    c = torch.where(torch.isnan(c), NEG, c).view(B, k * V)
    v, i = torch.sort(c, dim=1, descending=True, stable=True)
    return c, v[:, :width], i[:, :width]


def _check(x, scores, finished=None, eos=None, width=None):
    r = S.beam_step(x, scores, finished=finished, eos=eos, width=width)
    B, k = scores.shape
    V = x.shape[-1]
    w = width or k
    c, v, i = _reference(x, scores, finished, eos, w)
    flat = r.parents * V + r.tokens
    assert r.scores.shape == (B, w) and r.parents.dtype == torch.int64 and r.tokens.dtype == torch.int64
    assert bool((r.parents >= 0).all()) and bool((r.parents < k).all())
    assert bool((r.tokens >= 0).all()) and bool((r.tokens < V).all())
    # x - m and the logarithm of the sum (V terms in 32 bits) are each rounded, then two sums
    big = torch.where(torch.isinf(v), 1.0, v.abs()) + scores.abs().where(~torch.isinf(scores), 0).amax(1, keepdim=True)
    tol = 2.0 ** -22 * (big + 40.0) + V ** 0.5 * 2.0 ** -24
    same = torch.isinf(v) & (r.scores.double() == v)
    assert bool((same | ((r.scores.double() - v).abs() <= tol)).all())
    mine = torch.gather(c, 1, flat)
    assert bool(((mine == v) | ((mine - v).abs() <= 2 * tol)).all())        # as good as the best
    gap = torch.full_like(v, 1e30)
    gap[:, 1:] = torch.minimum(gap[:, 1:], (v[:, :-1] - v[:, 1:]).nan_to_num(0.0))
    gap[:, :-1] = torch.minimum(gap[:, :-1], (v[:, :-1] - v[:, 1:]).nan_to_num(0.0))
    sure = (gap > 4 * tol) & ~torch.isinf(v)
    sure[:, -1] = False                                                     # its successor is not in v
    assert bool((flat[sure] == i[sure]).all())
    assert all(len(set(row)) == w for row in flat.tolist())                 # no candidate twice
    if eos is not None:
        was = torch.gather(finished, 1, r.parents) if finished is not None else torch.zeros_like(r.finished)
        assert torch.equal(r.finished, was | (r.tokens == eos))
    else:
        assert r.finished is None
    return r


DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dtype", DTYPES, ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("B,k,V", [(1, 1, 1), (1, 1, 2), (3, 2, 5), (1, 4, 2000), (5, 3, 1023), (2, 8, 8191), (7, 5, 333),
                                   (64, 8, 4100), (2, 32, 257), (1, 16, 40001), (300, 2, 64)])
def test_step_matches_64_bits(B, k, V, dtype):
    g = torch.Generator().manual_seed(B * 7 + k * 3 + V)
    x = (4 * torch.randn(B * k, V, generator=g)).to(dtype).to(dev)
    scores = (-10 * torch.rand(B, k, generator=g)).to(dev)
    _check(x, scores)
    if V >= 5:
        x[torch.rand(B * k, V, generator=g).to(dev) < 0.3] = NEG
        finished = (torch.rand(B, k, generator=g) < 0.3).to(dev)
        _check(x.view(B, k, V), scores, finished, eos=V - 1)
        _check(x, scores, eos=2)


@pytest.mark.parametrize("V", [1, 2, 31, 500, 9001])
def test_ties_go_to_the_lowest_index(V):
    """Uniform logits: log V is the same for every candidate, so order is by score, beam, token."""
    k = min(8, V * 2)
    x = torch.full((2 * k, V), 3.0, device=dev)
    scores = torch.zeros(2, k, device=dev)
    scores[1, -1] = 1.0
    r = S.beam_step(x, scores)
    want = torch.arange(k, device=dev)
    assert torch.equal(r.parents[0] * V + r.tokens[0], want)
    last = [(k - 1) * V + t for t in range(min(V, k))]
    rest = [i for i in range(k * V) if i not in last][:k - len(last)]
    assert (r.parents[1] * V + r.tokens[1]).tolist() == (last + rest)[:k]


def test_counts_with_many_equal_logits():
    g = torch.Generator().manual_seed(2)
    x = (torch.randint(0, 4, (4, 3000), generator=g).float() / 10).to(dev)
    scores = torch.tensor([[0.0, -30.0, -60.0, -90.0]], device=dev)
    r = S.beam_step(x, scores)
    top = torch.nonzero(x[0] == x[0].max()).flatten()[:4]          # the first beam's largest count
    assert r.parents.tolist() == [[0, 0, 0, 0]] and torch.equal(r.tokens[0], top)


def test_masked_rows_and_values_that_are_not_finite():
    k, V = 4, 600
    x = torch.randn(2 * k, V, device=dev)
    x[0] = NEG                                        # a beam with nothing left
    x[1] = float("nan")
    x[2, 100:] = float("nan")
    x[3] = torch.finfo(torch.float32).min             # masked with the type's lowest value
    x[4:] = NEG                                       # an entry with nothing left
    scores = torch.tensor([[0.0, 0.0, -1.0, -50.0], [0.0, -1.0, -2.0, -3.0]], device=dev)
    r = _check(x, scores)
    assert bool((r.parents[0] == 2).all()) and bool((r.tokens[0] < 100).all())
    assert r.scores[1].tolist() == [NEG] * 4 and (r.parents[1] * V + r.tokens[1]).tolist() == [0, 1, 2, 3]
    x[2] = NEG
    r = S.beam_step(x, scores)                        # only the lowest-value row is left: uniform
    assert bool((r.parents[0] == 3).all()) and r.tokens[0].tolist() == [0, 1, 2, 3]
    assert (r.scores[0].double() + 50.0 + torch.log(torch.tensor(600.0)).item()).abs().max() < 1e-4
    x[0, 7] = float("inf")                            # counts as the largest finite value
    r = S.beam_step(x, scores)
    assert (r.parents[0, 0].item(), r.tokens[0, 0].item(), r.scores[0, 0].item()) == (0, 7, 0.0)


def test_beams_that_are_not_in_use_and_all_finished():
    x = torch.randn(4, 50, device=dev)
    scores = torch.tensor([[0.0, NEG, NEG, NEG]], device=dev)
    r = _check(x, scores)
    assert bool((r.parents == 0).all())
    done = torch.ones(1, 4, dtype=torch.bool, device=dev)
    scores = torch.tensor([[-4.0, -1.0, -3.0, -2.0]], device=dev)
    r = S.beam_step(x, scores, finished=done, eos=9)
    assert r.parents.tolist() == [[1, 3, 2, 0]] and bool((r.tokens == 9).all()) and bool(r.finished.all())
    assert r.scores.tolist() == [[-1.0, -2.0, -3.0, -4.0]]


@pytest.mark.parametrize("k,width", [(1, 4), (1, 32), (4, 2), (3, 7), (32, 1)])
def test_width_other_than_the_number_of_beams(k, width):
    g = torch.Generator().manual_seed(k)
    x = torch.randn(5 * k, 777, generator=g).to(dev)
    _check(x, -torch.rand(5, k, generator=g).to(dev), width=width)


def test_strided_logits_and_fewer_tokens_than_beams():
    base = torch.randn(6, 1000, device=dev)
    scores = torch.zeros(2, 3, device=dev)
    for x in (base[:, 3:503], base[:, ::2], base[:, 1:4].t().contiguous().t(), base[:1].expand(6, 1000)):
        a, b = S.beam_step(x, scores), S.beam_step(x.contiguous(), scores)
        assert torch.equal(a.scores, b.scores) and torch.equal(a.parents, b.parents) and torch.equal(a.tokens, b.tokens)
    _check(torch.randn(8, 2, device=dev), torch.zeros(1, 8, device=dev))


def _src(parents, beams):
    B = parents.shape[0]
    return (torch.arange(B, device=dev)[:, None] * beams + parents).reshape(-1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.uint8, torch.int64, torch.bool])
@pytest.mark.parametrize("shape", [(), (1,), (3,), (7, 5), (64,), (1000,)])
@pytest.mark.parametrize("B,k,w", [(1, 1, 1), (3, 4, 4), (5, 2, 6), (65, 8, 8)])
def test_reorder_rows(B, k, w, shape, dtype):
    g = torch.Generator().manual_seed(B + k)
    state = torch.randint(0, 200, (B * k,) + shape, generator=g).to(dtype).to(dev)
    parents = torch.randint(0, k, (B, w), generator=g).to(dev)
    got = S.beam_reorder(state, parents)
    assert got.dtype == dtype and torch.equal(got, state[_src(parents, k)])


@pytest.mark.parametrize("F", [1, 3, 100, 2001])
@pytest.mark.parametrize("B,k,w", [(1, 1, 1), (1, 4, 4), (3, 5, 5), (16, 8, 8), (9, 32, 32), (5, 2, 6), (64, 8, 3)])
def test_reorder_features_and_packed(F, B, k, w):
    g = torch.Generator().manual_seed(F + B + k)
    parents = torch.randint(0, k, (B, w), generator=g).to(dev)
    src = _src(parents, k)
    x = torch.rand(B * k, F, generator=g).to(dev)
    xt = torch.zeros(F, _soft.ldb_for(B * k), device=dev)
    xt[:, :B * k] = x.t()
    got = S.beam_reorder(xt, parents, layout="features", beams=k)
    assert got.shape == (F, _soft.ldb_for(B * w) if w != k else xt.shape[1])
    assert torch.equal(got[:, :B * w], xt[:, src]) and bool((got[:, B * w:] == 0).all())
    bits = (x > 0.5).to(torch.uint8)
    packed = _hard.pack(bits)
    got = S.beam_reorder(packed, parents, layout="packed", beams=k)
    assert torch.equal(_hard.unpack(got, B * w), bits[src])
    assert torch.equal(got, _hard.pack(bits[src].contiguous(), ldw=got.shape[1]))       # padding bits 0


def test_reorder_keeps_a_wider_row_and_takes_strided_state():
    bits = (torch.rand(10, 33, device=dev) > 0.5).to(torch.uint8)
    packed = _hard.pack(bits, ldw=6)
    parents = torch.tensor([[4, 0, 0, 2, 1], [3, 3, 3, 4, 0]], device=dev)
    got = S.beam_reorder(packed, parents, layout="packed")
    assert got.shape == packed.shape and torch.equal(got, _hard.pack(bits[_src(parents, 5)].contiguous(), ldw=6))
    state = torch.rand(8, 10, 3, device=dev).transpose(0, 1)
    assert torch.equal(S.beam_reorder(state, parents), state[_src(parents, 5)])


def test_empty_batches():
    r = S.beam_step(torch.empty(0, 50, device=dev), torch.empty(0, 4, device=dev), eos=3)
    assert r.scores.shape == (0, 4) and r.finished.shape == (0, 4)
    p = torch.empty(0, 4, dtype=torch.int64, device=dev)
    assert S.beam_reorder(torch.empty(0, 7, device=dev), p).shape == (0, 7)
    assert S.beam_reorder(torch.empty(5, 4, device=dev), p, layout="features").shape == (5, 4)
    one = torch.zeros(1, 4, dtype=torch.int64, device=dev)
    assert S.beam_reorder(torch.empty(4, 0, device=dev), one).shape == (4, 0)
    assert S.beam_reorder(torch.empty(0, 4, device=dev), one, layout="features").shape == (0, 4)


def test_step_on_another_stream_and_in_a_graph():
    x, scores = torch.randn(8, 900, device=dev), torch.zeros(2, 4, device=dev)
    state = torch.rand(8, 33, device=dev)

    def both():
        r = S.beam_step(x, scores, eos=3)
        return r.scores, r.parents, r.tokens, r.finished, S.beam_reorder(state, r.parents)
    want = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = both()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = both()
    for seed in range(3):
        torch.manual_seed(seed)
        x.normal_()
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(kept, both()))


def test_equal_rows_tie_across_beams():
    """Beams with the same logits and scores (a decoder's first steps) have equal candidates: the
    lowest beam wins, whatever the rows' alignment and the number of beams."""
    g = torch.Generator().manual_seed(0)
    for V in (777, 8191, 20001):
        for k in (3, 5, 8):
            for dtype in DTYPES:
                x = (3 * torch.randn(1, V, generator=g)).to(dtype).to(dev).expand(2 * k, V).contiguous()
                r = S.beam_step(x, torch.full((2, k), -7.0, device=dev))
                top = x[0].float().max()
                first = torch.nonzero(x[0].float() == top).flatten()
                # the best token of every beam ties: beams in order, tokens in order within a beam
                want = [(b, t) for b in range(k) for t in first.tolist()][:k]
                for e in range(2):
                    assert list(zip(r.parents[e].tolist(), r.tokens[e].tolist())) == want


def test_large_magnitudes():
    """Logits far from zero: the normaliser keeps its accuracy (sums run relative to the maximum)."""
    g = torch.Generator().manual_seed(1)
    base = 4 * torch.randn(6, 3000, generator=g, dtype=torch.float64)
    for shift in (0.0, 1000.0, -1000.0, 60000.0, 1e5, -1e6):
        x = (base + shift).float().to(dev)
        _check(x, -torch.rand(2, 3, generator=g).to(dev))
    big = torch.tensor([[1e30, 2e30, 2e30, -3e38]], device=dev)
    r = S.beam_step(big, torch.zeros(1, 1, device=dev), width=4)
    assert r.tokens.tolist() == [[1, 2, 0, 3]]
    assert (r.scores[0, :2] + 0.6931472).abs().max() < 1e-6 and bool((r.scores[0, 2:] < -1e29).all())


def test_logits_past_2_31_elements():
    V = 70_000_000
    x = torch.full((32, V), -3.0, dtype=torch.bfloat16, device=dev)
    x[31, V - 1] = 40.0
    x[30, V - 2] = 39.0
    r = S.beam_step(x, torch.zeros(1, 32, device=dev), width=2)
    assert r.parents.tolist() == [[30, 31]] or r.parents.tolist() == [[31, 30]]
    assert set(r.tokens[0].tolist()) == {V - 1, V - 2}


def test_example_trains_and_decodes():
    import importlib.util
    import os
    from conftest import ROOT
    spec = importlib.util.spec_from_file_location("token_logic_net", os.path.join(ROOT, "examples", "token_logic_net.py"))
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    torch.manual_seed(0)
    net = ex.TokenLogicNet(12, dim=32, state=128).to(dev)
    first = ex.train(net, 1, batch_size=128, length=6, log=None)
    last = ex.train(net, 120, batch_size=128, length=6, log=None)
    assert last < 0.8 * first
    prompt = ex.batch(5, 4, 12, torch.Generator().manual_seed(1), dev)
    tokens, scores = net.generate(prompt, 5, beams=3)
    assert tokens.shape == (5, 3, 5) and bool((scores[:, :-1] >= scores[:, 1:]).all())
    # one beam is the greedy decoder of the circuit, step by step
    tokens, _ = net.generate(prompt, 5, beams=1)
    step = net.circuit()
    from silogic_b200.bitpacking import pack_bits
    h = pack_bits(torch.zeros((5, 128), dtype=torch.uint8, device=dev))
    for t in range(4):
        logits, h = step(prompt[:, t].contiguous(), h)
    for t in range(5):
        ids = logits.argmax(1)
        assert torch.equal(ids, tokens[:, 0, t])
        logits, h = step(ids, h)


@pytest.mark.parametrize("B,k,w", [(3, 48, 48), (3, 49, 49), (2, 51, 51), (3, 64, 64), (2, 100, 100), (1, 200, 200),
                                   (2, 3, 120), (2, 40, 90), (1, 2100, 7), (2, 5000, 3), (1, 4096, 4096), (9, 33, 5)])
def test_reorder_packed_with_more_beams_than_a_step_has(B, k, w):
    """beam_reorder takes any number of beams: a word's sources then lie in more than four words,
    or further than 16 bits apart."""
    g = torch.Generator().manual_seed(k + w)
    parents = torch.randint(0, k, (B, w), generator=g).to(dev)
    parents[:, -1], parents[:, 0] = 0, k - 1
    bits = (torch.rand(B * k, 37, generator=g) > 0.5).to(torch.uint8).to(dev)
    got = S.beam_reorder(_hard.pack(bits), parents, layout="packed", beams=k)
    want = bits[_src(parents, k)].contiguous()
    assert torch.equal(_hard.unpack(got, B * w), want)
    assert torch.equal(got, _hard.pack(want, ldw=got.shape[1]))


def _exact_order(x, scores, finished, eos, width):
    """The step in 32 bits for rows whose normaliser is exactly 1 (one logit far above the
    others): scores are then single roundings, which torch reproduces bit for bit."""
    B, k = scores.shape
    V = x.shape[-1]
    x = x.float().view(B, k, V)
    c = (x - x.amax(2, keepdim=True)) + scores[:, :, None]
    c = torch.where(torch.isnan(c), NEG, c)
    if finished is not None:
        only = torch.full_like(c, NEG)
        only[:, :, eos] = scores
        c = torch.where(finished[:, :, None], only, c)
    v, i = torch.sort(c.view(B, k * V), dim=1, descending=True, stable=True)
    return v[:, :width], i[:, :width]


@pytest.mark.parametrize("dtype", DTYPES, ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("B,k,width,V", [(1, 1, 1, 50), (1, 1, 1, 40000), (3, 1, 4, 1023), (1, 4, 4, 20001), (70, 4, 4, 3000),
                                         (2, 8, 8, 9000), (1, 32, 32, 2000), (5, 3, 32, 700), (200, 2, 2, 2500)])
@pytest.mark.parametrize("size", [30.0, 3e4, 2e6, 1e9])
def test_equal_scores_of_different_logits_go_to_the_lowest_index(B, k, width, V, dtype, size):
    """Far from zero, scores of different logits round to the same value: the order is that of
    the rounded scores, then of the indices."""
    g = torch.Generator().manual_seed(V + B)
    x = -150.0 - 150.0 * torch.rand(B * k, V, generator=g)
    x[torch.arange(B * k), torch.randint(0, V, (B * k,), generator=g)] = 0.0     # the normaliser is 1
    x[torch.rand(B * k, V, generator=g) < 0.1] = NEG
    x[torch.arange(B * k), torch.randint(0, V, (B * k,), generator=g)] = 0.0
    top = (x == 0).sum(1) > 1
    x[top] = torch.where(x[top] == 0, torch.where((x[top] == 0).cumsum(1) > 1, -200.0, 0.0), x[top])
    x = x.to(dtype).to(dev)
    scores = (-size * (1 + torch.randint(0, 3, (B, k), generator=g))).to(dev)
    scores[torch.rand(B, k, generator=g).to(dev) < 0.1] = NEG
    finished = (torch.rand(B, k, generator=g) < 0.2).to(dev)
    for done, eos in ((None, None), (finished, V - 1)):
        r = S.beam_step(x, scores, finished=done, eos=eos, width=width)
        v, i = _exact_order(x, scores, done, eos, width)
        assert torch.equal(r.scores, v)
        assert torch.equal(r.parents * V + r.tokens, i)
        if eos is not None:
            assert torch.equal(r.finished, torch.gather(done, 1, r.parents) | (r.tokens == eos))


@pytest.mark.parametrize("V", [2, 300, 5000, 40001])
@pytest.mark.parametrize("B", [1, 64, 300])
def test_neighbouring_logits_whose_scores_are_equal(B, V):
    """1 - 2^-24 and 1 are half a unit of the score apart at -20.69: token 0 wins."""
    x = torch.full((B, V), -300.0, device=dev)
    x[:, 0], x[:, V // 2] = 1 - 2.0 ** -24, 1.0
    r = S.beam_step(x, torch.full((B, 1), -20.0, device=dev), width=2)
    assert bool((r.scores == r.scores[0, 0]).all()) and abs(r.scores[0, 0].item() + 20.693148) < 1e-5
    assert bool((r.tokens[:, 0] == 0).all()) and bool((r.tokens[:, 1] == V // 2).all())
    r = S.beam_step(x, torch.full((B, 1), -20.0, device=dev))
    assert bool((r.tokens == 0).all())


@pytest.mark.parametrize("V", [3, 40, 3000, 20001])
def test_entries_with_no_beam_in_use(V):
    """Every candidate scores -inf: the lowest indices, whatever the logits."""
    k = 3
    x = torch.randn(4 * k, V, device=dev)
    scores = torch.full((4, k), NEG, device=dev)
    scores[3] = float("nan")                                    # a NaN score is no better
    r = S.beam_step(x, scores)
    assert bool((r.scores == NEG).all()) and bool((r.parents == 0).all())
    assert torch.equal(r.tokens, torch.arange(k, device=dev).expand(4, k))
    r = S.beam_step(x, scores, width=2 * V if V <= 16 else 32, eos=1)
    at = r.parents * V + r.tokens
    assert torch.equal(at, torch.arange(at.shape[1], device=dev).expand_as(at)) and torch.equal(r.finished, r.tokens == 1)
    scores[1, 2] = -4.0                                         # one beam in use, with one token allowed
    x[5] = NEG
    x[5, V - 1] = 2.0
    r = S.beam_step(x, scores)
    assert r.scores[1].tolist() == [-4.0, NEG, NEG] and r.parents[1].tolist() == [2, 0, 0]
    assert r.tokens[1].tolist() == [V - 1, 0, 1]


def test_unused_beams_at_a_large_negative_score():
    """Beams parked at -1e9, as decoders do: candidates that fill a place tie and go by index."""
    x = torch.randn(4, 2, device=dev)
    scores = torch.tensor([[0.0, -1e9, -1e9, -1e9]], device=dev)
    r = S.beam_step(x, scores, width=6)
    assert sorted(r.tokens[0, :2].tolist()) == [0, 1] and r.parents[0, :2].tolist() == [0, 0]
    assert (r.parents[0, 2:] * 2 + r.tokens[0, 2:]).tolist() == [2, 3, 4, 5]


@pytest.mark.parametrize("allowed", [0, 1, 3, 9])
@pytest.mark.parametrize("dtype", DTYPES, ids=["fp32", "bf16", "fp16"])
def test_constrained_rows(allowed, dtype):
    """All but a few tokens masked (fewer than there are beams): the allowed ones in order, then
    what scores -inf by index; a constant row, whose logits all equal the last of its list."""
    k, V, B = 4, 9001, 3
    g = torch.Generator().manual_seed(allowed)
    x = torch.full((B * k, V), NEG)
    for r in range(B * k):
        x[r, torch.randperm(V, generator=g)[:allowed]] = torch.randn(allowed, generator=g)
    x[5] = 1.5
    x = x.to(dtype).to(dev)
    scores = -torch.rand(B, k, generator=g).to(dev)
    r = _check(x, scores)
    if allowed == 0:
        assert (r.parents[0] * V + r.tokens[0]).tolist() == [0, 1, 2, 3]
        assert r.parents[1].tolist() == [1] * 4 and r.tokens[1].tolist() == [0, 1, 2, 3]
    if allowed == 1:
        left = torch.isinf(r.scores[2])
        assert int(left.sum()) == 0 and sorted(r.parents[2].tolist()) == [0, 1, 2, 3]


@pytest.mark.parametrize("dtype", DTYPES, ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("spread", [1e-6, 1e-4, 1e-2, 1.0, 8.0])
@pytest.mark.parametrize("B,V,width", [(1, 33, 32), (3, 1024, 4), (150, 1000, 32), (300, 1025, 8), (2, 20000, 1), (64, 4097, 2)])
def test_order_is_that_of_the_rounded_scores(B, V, width, spread, dtype):
    """Bit for bit: a step at score 0 tells the normaliser l (its best token scores 0 - l); every
    candidate's score is then three single roundings, (x - max) - l + S."""
    g = torch.Generator().manual_seed(B + V)
    x = (torch.randn(B, V, generator=g) * spread + 1.0)
    x[torch.rand(B, V, generator=g) < 0.1] = NEG
    x[:, V // 3] = 1.0
    x = x.to(dtype).to(dev)
    l = -S.beam_step(x, torch.zeros(B, 1, device=dev), width=1).scores
    d = x.float() - x.float().amax(1, keepdim=True)
    for size in (0.0, 1.0, 20.0, 1000.0, 1e5):
        s = (-size * (1 + torch.rand(B, 1, generator=g))).to(dev)
        r = S.beam_step(x, s, width=width)
        v, i = torch.sort((d - l) + s, dim=1, descending=True, stable=True)
        assert torch.equal(r.scores, v[:, :width]) and torch.equal(r.tokens, i[:, :width])
