"""Token embedding on the GPU against a plain 64-bit implementation.

Tolerances: the lookup rounds scale * w once in 32 bits and once to the type
(u = 2^-24, 2^-8, 2^-11 for fp32, bf16, fp16 as the spacing bound of one rounding); a
gradient row of n terms is summed in 32 bits, (n + 2) 2^-24 of the sum of magnitudes, and
rounded once.
"""
import pytest
import torch

import silogic_b200 as S

pytestmark = pytest.mark.gpu
dev = "cuda"
UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SMALLEST = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
NAMES = ["fp32", "bf16", "fp16"]


def _case(V, D, N, dtype, seed=0, ids=None, idt=torch.int64):
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(V, D, generator=g).to(dtype).to(dev)
    if ids is None:     # frequencies fall as 1 / rank: a few tokens fill most of the batch
        ids = (torch.exp(torch.rand(N, generator=g) * torch.log(torch.tensor(V + 1.0))).long() - 1).clamp(0, V - 1)
    gy = torch.randn(len(ids), D, generator=g).to(dtype).to(dev)
    return ids.to(idt).to(dev), w, gy


def _check_grad(got, ids, gy, V, scale, pad=None):
    ids, g64 = ids.reshape(-1).long(), gy.reshape(ids.numel(), gy.shape[-1]).double()
    keep = (ids >= 0) & (ids < V)
    if pad is not None:
        keep &= ids != pad
    want = torch.zeros(V, g64.shape[1], dtype=torch.float64, device=dev).index_add_(0, ids[keep], g64[keep])
    mag = torch.zeros_like(want).index_add_(0, ids[keep], g64[keep].abs())
    n = torch.bincount(ids[keep], minlength=V).double()[:, None]
    u = UNIT[got.dtype]
    tol = abs(scale) * mag * (n + 2) * 2.0 ** -24 + (abs(scale) * want.abs()) * u + SMALLEST[got.dtype]
    err = (got.double() - scale * want).abs()
    assert got.shape == want.shape and bool((err <= tol).all()), f"worst excess {(err - tol).max().item():.3e}"


@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
@pytest.mark.parametrize("V,D,N", [(1, 1, 1), (7, 3, 5), (50, 64, 33), (256, 128, 257), (255, 331, 1021),
                                   (10000, 784, 4), (1000, 100, 20000), (65536, 40, 3000), (65537, 8, 70001),
                                   (300, 1030, 513)])
def test_lookup_and_gradient_match_64_bits(V, D, N, dtype):
    ids, w, gy = _case(V, D, N, dtype, seed=V + D + N, idt=torch.int32 if N % 2 else torch.int64)
    w.requires_grad_(True)
    scale = D ** 0.5
    y = S.token_embedding(ids, w, scale=scale)
    assert y.dtype == dtype and y.shape == (N, D)
    want = w.detach().double()[ids.long()] * scale
    tol = want.abs() * (UNIT[dtype] + 2.0 ** -23) + SMALLEST[dtype]
    assert bool(((y.double() - want).abs() <= tol).all())
    (gw,) = torch.autograd.grad(y, w, gy)
    assert gw.dtype == dtype
    _check_grad(gw, ids, gy, V, scale)


@pytest.mark.parametrize("N", [0, 1, 31, 1024, 1025, 4096, 4097, 8192, 8193, 9000, 300000])
def test_gradient_of_one_hot_token_and_empty_batch(N):
    """Every token the same: one row takes the whole sum, the others are zero."""
    ids, w, gy = _case(37, 20, N, torch.float32, ids=torch.full((N,), 5))
    w.requires_grad_(True)
    y = S.token_embedding(ids, w, scale=0.5)
    (gw,) = torch.autograd.grad(y, w, gy)
    _check_grad(gw, ids, gy, 37, 0.5)
    assert bool((gw[:5] == 0).all()) and bool((gw[6:] == 0).all())


@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
@pytest.mark.parametrize("D", [64, 65])
def test_padding_and_out_of_range_ids(D, dtype):
    V, N = 100, 5000
    g = torch.Generator().manual_seed(3)
    raw = torch.randint(-3, V + 3, (N,), generator=g)
    ids, w, gy = _case(V, D, N, dtype, ids=raw)
    w.requires_grad_(True)
    y = S.token_embedding(ids, w, padding_idx=7)
    bad = (ids < 0) | (ids >= V)
    assert bool(torch.isnan(y[bad]).all()) and not bool(torch.isnan(y[~bad]).any())
    assert torch.equal(y[ids == 7], w.detach()[7].expand(int((ids == 7).sum()), D))   # read like any row
    (gw,) = torch.autograd.grad(y, w, gy)
    _check_grad(gw, ids, gy, V, 1.0, pad=7)
    assert bool((gw[7] == 0).all())
    with pytest.raises(IndexError):
        S.token_embedding(ids, w, check=True)


def test_ids_of_any_shape_strided_weights_and_gradients():
    base = torch.randn(60, 48, device=dev)
    w = base[::2, ::3].requires_grad_(True)                  # not contiguous
    ids = torch.randint(0, 30, (4, 5, 6), device=dev).transpose(0, 2)
    y = S.token_embedding(ids, w, scale=2.0)
    assert y.shape == (6, 5, 4, 16) and torch.equal(y, 2.0 * w.detach()[ids])
    gy = torch.randn(16, 4, 5, 6, device=dev).permute(3, 2, 1, 0)
    (gw,) = torch.autograd.grad(y, w, gy)
    _check_grad(gw, ids, gy.contiguous(), 30, 2.0)
    one = torch.ones((), device=dev).expand(6, 5, 4, 16)     # a broadcast upstream gradient
    (gw,) = torch.autograd.grad(S.token_embedding(ids, w), w, one)
    _check_grad(gw, ids, one.contiguous(), 30, 1.0)


def test_rows_that_start_on_no_vector_boundary():
    flat = torch.randn(1 + 50 * 64, device=dev)
    w = flat[1:].view(50, 64)                                # 4 bytes past a 16-byte boundary
    ids = torch.randint(0, 50, (333,), device=dev)
    assert torch.equal(S.token_embedding(ids, w), w[ids])
    gflat = torch.randn(1 + 333 * 64, device=dev)
    gy = gflat[1:].view(333, 64)
    w2 = w.clone().requires_grad_(True)
    (gw,) = torch.autograd.grad(S.token_embedding(ids, w2), w2, gy)
    _check_grad(gw, ids, gy, 50, 1.0)


def test_gradient_is_the_same_from_run_to_run_and_on_another_stream():
    ids, w, gy = _case(2000, 256, 50000, torch.float32)
    w.requires_grad_(True)

    def grad():
        return torch.autograd.grad(S.token_embedding(ids, w), w, gy)[0]
    first = grad()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = grad()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, other) and torch.equal(first, grad())


def test_gradient_against_differences():
    """dL/dW of L = sum(c * y^2): the directional derivative equals the difference quotient
    of the (quadratic) loss, which a central difference gives without truncation error."""
    V, D, N = 40, 24, 300
    ids, w, c = _case(V, D, N, torch.float32, seed=5)
    w.requires_grad_(True)
    loss = lambda m: (c.double() * S.token_embedding(ids, m, scale=1.5).double() ** 2).sum()   # noqa: E731
    (gw,) = torch.autograd.grad(loss(w), w)
    d = torch.randn(V, D, generator=torch.Generator().manual_seed(1)).to(dev)
    h = 2.0 ** -6
    with torch.no_grad():
        num = (loss(w + h * d) - loss(w - h * d)) / (2 * h)
    # the terms of both losses, rounded to 32 bits, divided by 2 h; the gradient's own rounding
    scale = (c.abs().double() * (1.5 * (w.detach().abs() + h * d.abs()))[ids].double() ** 2).sum()
    tol = 8 * 2.0 ** -24 * scale / (2 * h)
    assert abs(num - (gw.double() * d.double()).sum()) <= tol


def test_inside_a_cuda_graph():
    ids, w, gy = _case(500, 96, 777, torch.float32)
    w.requires_grad_(True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(S.token_embedding(ids, w), w, gy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = S.token_embedding(ids, w)
        (gw,) = torch.autograd.grad(y, w, gy)
    for seed in (1, 2):
        new, _, _ = _case(500, 96, 777, torch.float32, seed=seed)
        ids.copy_(new)
        graph.replay()
        assert torch.equal(y, w.detach()[ids])
        _check_grad(gw, ids, gy, 500, 1.0)


def test_module_trains_and_keeps_its_padding_row():
    torch.manual_seed(0)
    m = S.TokenEmbedding(50, 16, padding_idx=3).to(dev)
    assert bool((m.weight[3] == 0).all()) and m.scale == 4.0
    ids = torch.randint(0, 50, (8, 9), device=dev)
    ids[0] = 3
    m(ids).sum().backward()
    assert bool((m.weight.grad[3] == 0).all()) and bool((m.weight.grad != 0).any())


def test_offsets_past_32_bits():
    """A table of 2.6e9 values: rows, gradients and carries beyond 2^32 bytes and 2^31 elements."""
    V, D = 50000, 52000
    w = torch.zeros(V, D, dtype=torch.bfloat16, device=dev)
    w[V - 1] = 3.0
    w[V - 2, D - 1] = 5.0
    w.requires_grad_(True)
    ids = torch.tensor([V - 1, 0, V - 2, V - 1], device=dev)
    y = S.token_embedding(ids, w, scale=2.0)
    assert bool((y[0] == 6).all()) and bool((y[1] == 0).all()) and y[2, D - 1] == 10 and bool((y[3] == 6).all())
    gy = torch.ones(4, D, dtype=torch.bfloat16, device=dev)
    (gw,) = torch.autograd.grad(y, w, gy)
    assert bool((gw[V - 1] == 4).all()) and bool((gw[V - 2] == 2).all()) and bool((gw[0] == 2).all())
    assert not bool((gw[1:V - 2] != 0).any())


@pytest.mark.parametrize("N,V,top", [(20000, 50, 0.9), (60000, 30000, 0.5), (140000, 65536, 0.3)])
def test_rows_cut_into_many_chunks(N, V, top):
    """Frequent tokens whose rows span hundreds of chunks beside many rows that span two."""
    g = torch.Generator().manual_seed(N)
    ids = torch.randint(0, V, (N,), generator=g)
    ids[torch.rand(N, generator=g) < top] = V // 2
    for D, dtype in ((136, torch.float32), (264, torch.bfloat16), (130, torch.float16), (600, torch.float32)):
        ids_d, w, gy = _case(V, D, N, dtype, ids=ids)
        w.requires_grad_(True)
        (gw,) = torch.autograd.grad(S.token_embedding(ids_d, w), w, gy)
        _check_grad(gw, ids_d, gy, V, 1.0)


def test_traced_by_torch_compile():
    """Lookup and gradient are torch.library ops with fake implementations: no graph break."""
    m = S.TokenEmbedding(100, 24, padding_idx=0).to(dev)
    ids = torch.randint(0, 100, (6, 7), device=dev)
    f = torch.compile(lambda i: (m(i) ** 2).sum(), backend="aot_eager", fullgraph=True)
    m.zero_grad()
    f(ids).backward()
    got = m.weight.grad.clone()
    m.zero_grad()
    (m(ids) ** 2).sum().backward()
    assert torch.equal(got, m.weight.grad)


@pytest.mark.parametrize("pad", [None, 3])
def test_gradients_of_gradients(pad):
    """A penalty on the embedding's gradient, and a third derivative, against torch's indexing in
    64 bits.  The tolerance is 2^-18 of the sum of magnitudes: each value passes through at
    most three 32-bit sums of at most 60 terms."""
    V, D, N = 11, 6, 60
    g = torch.Generator().manual_seed(4)
    ids = torch.randint(-1, V + 1, (N,), generator=g).to(dev)
    c = torch.randn(N, D, generator=g).to(dev)
    inside = (ids >= 0) & (ids < V)
    counted = inside & (ids != pad) if pad is not None else inside

    def values(w, lookup):
        y = torch.where(inside[:, None], lookup(w), 0.0)
        loss = (c.to(w.dtype) * y ** 3).sum()
        (gw,) = torch.autograd.grad(loss, w, create_graph=True)
        total = loss + (gw ** 2).sum()
        (g2,) = torch.autograd.grad(total, w, create_graph=True)
        (g3,) = torch.autograd.grad((g2 * w.detach()).sum(), w)
        return gw, g2, g3

    def plain(w):
        rows = torch.where(counted[:, None], w[ids.clamp(0, V - 1)], w.detach()[ids.clamp(0, V - 1)])
        return 1.5 * rows
    w = (torch.randn(V, D, generator=g).to(dev)).requires_grad_(True)
    w64 = w.detach().double().requires_grad_(True)
    got = values(w, lambda m: S.token_embedding(ids, m, scale=1.5, padding_idx=pad).nan_to_num(0.0))
    want = values(w64, plain)
    for a, b in zip(got, want):
        assert bool(((a.double() - b).abs() <= 2.0 ** -18 * b.abs().max()).all())


@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_refused(grad):
    """A tangent must not be dropped silently, whether or not the weight takes a gradient."""
    from torch.autograd import forward_ad
    ids = torch.tensor([1, 0, 2], device=dev)
    w = torch.randn(4, 8, device=dev)
    with forward_ad.dual_level():
        assert S.token_embedding(ids, w).shape == (3, 8)                # no tangent: an ordinary lookup
        dual = forward_ad.make_dual(w.requires_grad_(grad), torch.ones(4, 8, device=dev))
        with pytest.raises(RuntimeError):
            S.token_embedding(ids, dual)
        with torch.no_grad(), pytest.raises(RuntimeError):
            S.token_embedding(ids, dual)


def test_eager_calls_run_on_the_native_node():
    """A Python autograd Function cost a small training step more than its kernels; what such a
    Function gives must hold for the native node too."""
    V, D = 40, 24
    ids, w, gy = _case(V, D, 30, torch.float32)
    w.requires_grad_(True)
    y = S.token_embedding(ids, w, scale=2.0)
    assert not isinstance(y.grad_fn, torch.autograd.function.BackwardCFunction)
    ids += 1                                                    # the backward pass would see other ids
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, w, gy)
    ids -= 1
    seen = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: seen.append(t) or t, lambda t: t):
        y = S.token_embedding(ids, w, scale=2.0)
    assert len(seen) == 1 and torch.equal(seen[0], ids)
    (gw,) = torch.autograd.grad(y, w, gy, retain_graph=True)
    _check_grad(gw, ids, gy, V, 2.0)
    assert torch.equal(torch.autograd.grad(y, w, gy)[0], gw)
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(y, w, gy)
    for off in (torch.no_grad, torch.inference_mode):
        with off():
            z = S.token_embedding(ids, w, scale=2.0)
        assert not z.requires_grad and torch.equal(z, y)
    assert not S.token_embedding(ids, w.detach()).requires_grad
    h = S.token_embedding(ids, w.half(), scale=2.0)             # a cast inside the graph
    h.sum().backward()
    assert w.grad.dtype == torch.float32 and bool((w.grad[ids] != 0).all())


def test_backward_of_an_unused_and_of_a_partly_used_lookup():
    ids, w, _ = _case(20, 8, 12, torch.float32)
    w.requires_grad_(True)
    a, b = S.token_embedding(ids, w), S.token_embedding(ids, w)
    (gw,) = torch.autograd.grad(a[:5].sum(), w)                 # a gradient with zero rows
    want = torch.zeros_like(gw).index_add_(0, ids[:5], torch.ones(5, 8, device=dev))
    assert torch.equal(gw, want)
    b.sum().backward()
    b2 = S.token_embedding(ids, w)
    b2.sum().backward()                                         # accumulates
    assert torch.equal(w.grad, 2 * torch.zeros_like(gw).index_add_(0, ids, torch.ones(12, 8, device=dev)))
