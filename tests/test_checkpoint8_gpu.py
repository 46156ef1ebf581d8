"""8-bit activation checkpoints on the GPU.

Stored values: the codes are defined by single IEEE roundings, so they are compared with a
restatement in numpy fp32 bit for bit; against 64 bits a value is within half a step plus
the rounding of the arithmetic.  Layer gradients: 64-bit formulas evaluated at the values
read back, with the tolerance of the soft layers' other gradient tests,
1e-5 (|ref| + max|ref|) + 1e-7.
"""
import numpy as np
import pytest
import torch

import silogic_b200 as S
from silogic_b200 import _soft

pytestmark = pytest.mark.gpu
dev = "cuda"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
NAMES = ["fp32", "bf16", "fp16"]


def _reference(x):
    """(codes, lo, step, values) of [rows, cols] fp32 numpy, block by block."""
    rows, cols = x.shape
    f = np.float32
    codes, vals = np.zeros((rows, cols), np.uint8), np.zeros((rows, cols), f)
    bounds = np.zeros((rows, -(-cols // 128), 2), f)
    with np.errstate(all="ignore"):
        for b in range(bounds.shape[1]):
            p = x[:, b * 128:(b + 1) * 128]
            lo, hi = p.min(1, keepdims=True), p.max(1, keepdims=True)
            rng = hi - lo
            bad = ~np.isfinite(p).all(1, keepdims=True) | ~np.isfinite(rng)
            step = rng * (f(1) / f(255))
            flat = bad | (step < f(2.0 ** -100))
            inv = f(255) / np.where(flat, f(1), rng)
            code = np.where(flat, f(0), np.clip(np.rint((p - lo) * inv), 0, 255))
            step, lo = np.where(flat, f(0), step), np.where(bad, f(np.nan), lo)
            step = np.where(bad, f(np.nan), step)
            codes[:, b * 128:(b + 1) * 128] = code.astype(np.uint8)
            vals[:, b * 128:(b + 1) * 128] = code * step + lo
            bounds[:, b, 0], bounds[:, b, 1] = lo[:, 0], step[:, 0]
    return codes, bounds, vals


@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 4), (5, 127), (5, 128), (5, 129), (7, 331), (64, 1000),
                                       (2000, 64), (10, 4100)])
def test_store_and_restore(rows, cols, dtype):
    g = torch.Generator().manual_seed(rows + cols)
    x = torch.sigmoid(3 * torch.randn(rows, cols, generator=g)).to(dtype)
    x[0] = 0.25                                                     # a constant row
    x[-1] = (torch.rand(cols, generator=g) < 0.3).to(dtype)         # a binary one
    ck = S.checkpoint8_store(x.to(dev))
    codes, bounds, vals = _reference(x.float().numpy())
    np.testing.assert_array_equal(ck.codes[:, :cols].cpu().numpy(), codes)
    np.testing.assert_array_equal(ck.bounds.cpu().numpy(), bounds)
    np.testing.assert_array_equal(ck.restore(torch.float32).cpu().numpy(), vals)
    back = ck.restore()
    assert back.dtype == dtype and torch.equal(back.cpu(), torch.from_numpy(vals).to(dtype))
    assert torch.equal(back[-1].cpu(), x[-1]) and torch.equal(back[0].cpu(), x[0])     # exact
    # half a step, and the rounding of x - lo, of the code times step and of the sum
    x64, step = x.double().numpy(), np.repeat(bounds[:, :, 1], 128, 1)[:, :cols].astype(np.float64)
    assert np.all(np.abs(vals - x64) <= 0.5 * step * (1 + 2.0 ** -14) + 2.0 ** -23 * np.abs(x64))


def test_values_that_are_not_finite_and_tiny_or_huge_ranges():
    x = torch.rand(8, 300)
    x[0, 5] = float("nan")
    x[1, 200] = float("inf")
    x[2, 299] = -float("inf")
    x[3, :128] = torch.linspace(1e-42, 2e-40, 128)                  # below the smallest step
    x[4, :2] = torch.tensor([3e38, -3e38])                          # max - lo overflows
    x[5, :128] = 1e30 * torch.rand(128)
    x[6] = torch.finfo(torch.float32).min
    x[7, :128] = -0.0
    codes, bounds, vals = _reference(x.numpy())
    ck = S.checkpoint8_store(x.to(dev))
    back = ck.restore().cpu()
    np.testing.assert_array_equal(ck.codes[:, :300].cpu().numpy(), codes)
    np.testing.assert_array_equal(back.numpy(), vals)
    assert torch.isnan(back[0, :128]).all() and not torch.isnan(back[0, 128:]).any()
    assert torch.isnan(back[1, 128:256]).all() and torch.isnan(back[2, 256:]).all() and torch.isnan(back[4, :128]).all()
    assert torch.equal(back[6], x[6])


def test_shapes_strides_and_offsets():
    base = torch.rand(40, 333, device=dev)
    for x in (base[:, 1:300], base[::3], base.t(), base[3:4, 7:9], base[:, 5], base.view(5, 8, 333)):
        got = S.checkpoint8_store(x).restore()
        want = S.checkpoint8_store(x.contiguous()).restore()
        assert got.shape == x.shape and torch.equal(got, want)
        rows = x.reshape(-1, x.shape[-1]).cpu().numpy()
        np.testing.assert_array_equal(got.reshape(rows.shape).cpu().numpy(), _reference(np.ascontiguousarray(rows))[2])
    for shape in ((0, 5), (5, 0), (0,)):
        assert S.checkpoint8_store(torch.empty(shape, device=dev)).restore().shape == shape


def test_a_checkpoint_takes_a_quarter_of_the_memory():
    x = torch.rand(1000, 4096, device=dev)
    assert S.checkpoint8_store(x).nbytes() * 3.7 < x.numel() * 4


# ------------------------------------------------------------------ layers
BASIS = S.BASIS_COEFFS.double()


def _layer64(layer, x):
    """The layer's formula in 64 bits on [inputs, B]."""
    conn = layer._conn
    p = layer.node.param.detach().double().requires_grad_(True)
    c = conn.conn.detach().double().requires_grad_(True) if hasattr(conn, "conn") else None
    cand = conn.cand_i32.long()
    xs = x[cand]                                                   # [O, A, K, B]
    if c is not None:
        w = torch.softmax(c, 2)
        if conn.ste:
            hard = torch.nn.functional.one_hot(c.argmax(2), w.shape[2]).double()
            w = hard + w - w.detach()
        xs = xs * w[..., None]
    ops = xs.sum(2)
    kind = layer.node.kind
    if kind == "gate16":
        q = torch.softmax(p, 1) @ BASIS.to(x.device)
        a, b = ops[:, 0], ops[:, 1]
        y = q[:, 0:1] + q[:, 1:2] * a + q[:, 2:3] * b + q[:, 3:4] * a * b
    elif kind == "linear":
        y = torch.sigmoid(p[:, :1] + (p[:, 1:, None] * ops).sum(1))
    else:
        cur = [v[:, None] for v in (p if kind == "walsh" else torch.sigmoid(p)).unbind(1)]
        for j in range(layer.arity):
            a = ops[:, j]
            if kind == "walsh":
                cur = [lo + (2 * a - 1) * hi for lo, hi in zip(cur[0::2], cur[1::2])]
            else:
                cur = [lo + a * (hi - lo) for lo, hi in zip(cur[0::2], cur[1::2])]
        y = torch.sigmoid(cur[0] * layer.node.inv_tau) if kind == "walsh" else cur[0]
    return y, p, c


def _close(got, ref, what):
    tol = 1e-5 * (ref.abs() + ref.abs().max()) + 1e-7
    err = (got.double() - ref).abs()
    assert bool((err <= tol).all()), f"{what}: worst {err.max().item():.3e}, largest value {ref.abs().max().item():.3e}"


LAYERS = [("gate16", 2, "topk", 8), ("gate16", 2, "fixed", 1), ("gate16", 2, "topk", 3), ("walsh", 2, "topk", 8),
          ("walsh", 2, "topk", 16), ("walsh", 2, "fixed", 1), ("walsh", 4, "topk", 4), ("multilinear", 2, "topk", 5),
          ("multilinear", 1, "topk", 4), ("multilinear", 3, "topk", 8), ("multilinear", 4, "topk", 4),
          ("multilinear", 6, "topk", 4), ("linear", 2, "topk", 8), ("linear", 5, "topk", 2), ("hybrid", 2, "topk", 8),
          ("hybrid", 4, "fixed", 1)]


@pytest.mark.parametrize("node,arity,conn,k", LAYERS, ids=["-".join(map(str, v)) for v in LAYERS])
@pytest.mark.parametrize("B", [1, 3, 130, 1027])
def test_layer_gradients_at_the_checkpoint(node, arity, conn, k, B):
    torch.manual_seed(B)
    layer = S.LogicLayer(90, 150, node=node, arity=arity, connectome=conn, k=k, seed=1).to(dev)
    with torch.no_grad():
        for p in layer.parameters():
            p.normal_()
    x = torch.sigmoid(2 * torch.randn(B, 90, device=dev)).requires_grad_(True)
    gy = torch.randn(B, 150, device=dev)
    wanted = [x, layer.node.param] + ([layer._conn.conn] if conn == "topk" else [])
    plain = layer(x)
    with S.checkpoint8():
        y = layer(x)
    assert torch.equal(y, plain)                                    # the forward pass is unchanged
    got = torch.autograd.grad(y, wanted, gy)
    seen = S.checkpoint8_store(x.detach().t()).restore().double().requires_grad_(True)
    y64, p64, c64 = _layer64(layer, seen)
    want = torch.autograd.grad(y64, [seen, p64] + ([c64] if c64 is not None else []), gy.t().double())
    _close(got[0], want[0].t(), "x")
    _close(got[1], want[1], "parameters")
    if c64 is not None:
        _close(got[2], want[2], "connections")


def test_layer_with_one_hot_connections_and_without_input_gradient():
    torch.manual_seed(0)
    layer = S.LogicLayer(64, 100, node="walsh", k=4, gate_select="hard", seed=0).to(dev)
    x = (torch.rand(77, 64, device=dev) < 0.4).float()
    gy = torch.randn(77, 100, device=dev)
    with S.checkpoint8():
        y = layer(x)
    got = torch.autograd.grad(y, [layer.node.param, layer._conn.conn], gy)
    y64, p64, c64 = _layer64(layer, x.double().t())                 # binary inputs are kept exactly
    want = torch.autograd.grad(y64, [p64, c64], gy.t().double())
    _close(got[0], want[0], "parameters")
    _close(got[1], want[1], "connections")


def test_nets_with_wire_residual_and_binary_inputs_have_the_plain_gradients():
    """Binary activations are kept exactly, so the first layer's gradients equal those without
    checkpoints; hidden layers differ by the quantisation alone."""
    torch.manual_seed(0)
    net = S.LogicNet(50, 120, 3, node="walsh", k=8, tau=5.0, wire_residual=0.2, seed=0).to(dev)
    x = (torch.rand(200, 50, device=dev) < 0.3).float()
    r = torch.randn(200, 10, device=dev)

    def grads(on):
        net.zero_grad()
        with S.checkpoint8(on):
            out = net(x)
        (out * r).sum().backward()
        return out.detach(), [p.grad.clone() for p in net.parameters()]
    y0, g0 = grads(False)
    y1, g1 = grads(True)
    assert torch.equal(y0, y1)
    for a, b in zip(g0, g1):
        assert (a - b).norm() <= 0.05 * a.norm()
    assert _soft.CHECKPOINT8 is False


def test_conv_net_from_checkpoints():
    """Conv blocks read their checkpoint back before the backward kernels: the gradients are
    those of a block whose input is the values read back."""
    torch.manual_seed(0)
    conv = S.ConvLogicTree(3, 8, tree_depth=2, k=4, seed=0).to(dev)
    x = torch.rand(37, 3, 8, 8, device=dev)
    gy = torch.randn(37, 8, 8, 8, device=dev)
    seen = S.checkpoint8_store(x.reshape(37, -1).t()).restore().t().reshape(x.shape).contiguous().requires_grad_(True)
    x.requires_grad_(True)
    params = list(conv.parameters())
    with S.checkpoint8():
        y = conv(x)
    assert torch.equal(y, conv(x))
    got = torch.autograd.grad(y, [x] + params, gy)
    want = torch.autograd.grad(conv(seen), [seen] + params, gy)
    for a, b in zip(got, want):
        _close(a, b.double(), "conv")


def test_checkpoints_hold_less_memory_between_forward_and_backward():
    torch.manual_seed(0)
    layers = [S.LogicLayer(500, 500, node="walsh", connectome="fixed", seed=i).to(dev) for i in range(4)]
    x = torch.rand(4096, 500, device=dev, requires_grad=True)

    def held(on):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        with S.checkpoint8(on):
            h = _soft.ToFeatureMajor.apply(x)
            for l in layers:
                h = _soft.fc_layer_fm(l, h)
            del l
        used = torch.cuda.memory_allocated() - before
        h.sum().backward()
        return used
    held(True)
    full, small = held(False), held(True)
    act = 500 * 4096 * 4                    # one layer's activations; the last output is held too
    assert full >= 5 * act and small <= act + 4 * 0.27 * act + (1 << 20)


def test_training_step_in_a_cuda_graph():
    from silogic_b200.train import GraphedTrainStep
    torch.manual_seed(0)
    net = S.LogicNet(64, 200, 2, node="gate16", k=4, tau=3.0, seed=0).to(dev)
    opt = torch.optim.Adam(net.parameters(), lr=torch.tensor(0.05, device=dev), capturable=True)
    x = (torch.rand(128, 64) < 0.5).to(torch.uint8)
    y = x[:, :10].long().argmax(1)
    with S.checkpoint8():
        step = GraphedTrainStep(net, opt, (128, 64), dev)
        losses = [step.step(x.to(dev), y.to(dev)).item() for _ in range(60)]
    assert step.graph is not None and losses[-1] < 0.7 * losses[0]


# -------------------------------------------- the backward that reads codes
KINDS = {"gate16": (0, 16), "walsh": (1, 4), "multilinear": (2, 4), "hybrid": (3, 4)}


@pytest.mark.parametrize("node", list(KINDS))
@pytest.mark.parametrize("K", [1, 2, 4, 5, 8])
@pytest.mark.parametrize("B,wire,ste", [(1, 0, 0), (4, 7, 0), (131, 0, 1), (1020, 33, 0), (1028, 0, 2), (4500, 0, 0)])
def test_backward_from_codes_matches_the_restored_one(node, K, B, wire, ste):
    """The fused kernel against the fp32 kernel on the values read back (the same sums in
    another order: the tolerance of the layers' gradient tests)."""
    from silogic_b200._ops import IMPL
    kind, npar = KINDS[node]
    I, O = 61, 75
    g = torch.Generator().manual_seed(B + K)
    ldb = _soft.ldb_for(B)
    xt = torch.zeros(I, ldb)
    xt[:, :B] = torch.rand(I, B, generator=g)
    gy = torch.zeros(O, ldb)
    gy[:, :B] = torch.randn(O, B, generator=g)
    cand = torch.randint(0, I, (O, 2, K), generator=g, dtype=torch.int32).to(dev)
    conn = torch.randn(O, 2, K, generator=g).to(dev) if K > 1 or ste == 2 else None
    params = torch.randn(O, npar, generator=g).to(dev)
    xt, gy = xt.to(dev), gy.to(dev)
    codes, bounds = IMPL["ckpt_store"](xt[:, :B])
    args = (K, ste, kind, 2, 0, 1.3 if node == "walsh" else 1.0, O, wire)
    got = IMPL["fc_soft_bwd_ckpt"](codes, bounds, ldb, cand, conn, params, *args, gy, True)
    seen = torch.zeros_like(xt)
    seen[:, :B] = IMPL["ckpt_load"](codes, bounds, B, torch.float32)
    want = IMPL["fc_soft_bwd"](seen, cand, conn, params, *args, gy, True)
    for a, b, what in zip(got, want, ("x", "parameters", "connections")):
        if b.numel():
            _close(a[:, :B] if what == "x" else a, (b[:, :B] if what == "x" else b).double(), what)
    again = IMPL["fc_soft_bwd_ckpt"](codes, bounds, ldb, cand, conn, params, *args, gy, False)
    assert again[0].numel() == 0 and torch.equal(again[1], got[1]) and torch.equal(again[2], got[2])


def test_blocks_that_are_not_finite_reach_the_gradients():
    layer = S.LogicLayer(20, 30, node="walsh", k=4, seed=0).to(dev)
    x = torch.rand(256, 20, device=dev)
    x[3, 7] = float("nan")
    x.requires_grad_(True)
    with S.checkpoint8():
        y = layer(x)
    gx, gp = torch.autograd.grad(y, [x, layer.node.param], torch.ones_like(y))
    reads = (layer._conn.cand == 7).any(2).any(1)
    assert bool(torch.isnan(gp[reads]).all()) and not bool(torch.isnan(gp[~reads]).any())
    assert bool(torch.isnan(gx[:128]).any()) and not bool(torch.isnan(gx[128:]).any())


def test_offsets_past_32_bits():
    """4.3e9 activations: codes and gradient rows beyond 2^32 bytes and elements."""
    from silogic_b200._ops import IMPL
    I, B, K = 8300, 524288, 2
    codes = torch.randint(0, 256, (I, B), dtype=torch.uint8, device=dev)
    bounds = torch.rand(I, B // 128, 2, device=dev) * 0.01
    cand = torch.tensor([[[I - 1, 5], [I - 2, I - 1]]], dtype=torch.int32, device=dev)
    conn, params = torch.randn(1, 2, K, device=dev), torch.randn(1, 4, device=dev)
    gy = torch.randn(1, B, device=dev)
    args = (K, 0, 1, 2, 0, 1.0, 1, 0)
    gx, gp, gc = IMPL["fc_soft_bwd_ckpt"](codes, bounds, B, cand, conn, params, *args, gy, True)
    rows = torch.tensor([5, I - 2, I - 1], device=dev)
    small = torch.tensor([[[2, 0], [1, 2]]], dtype=torch.int32, device=dev)
    seen = IMPL["ckpt_load"](codes[rows].contiguous(), bounds[rows].contiguous(), B, torch.float32)
    wx, wp, wc = IMPL["fc_soft_bwd"](seen, small, conn, params, *args, gy, True)
    _close(gx[rows], wx.double(), "x")
    _close(gp, wp.double(), "parameters")
    _close(gc, wc.double(), "connections")
    assert not bool((gx[6:I - 2:97] != 0).any())
    del gx
    x = IMPL["ckpt_load"](codes, bounds, B, torch.bfloat16)
    assert torch.equal(x[rows], seen.to(torch.bfloat16))
    back, b2 = IMPL["ckpt_store"](x)
    assert torch.equal(back[rows], IMPL["ckpt_store"](x[rows])[0]) and torch.equal(b2[rows], IMPL["ckpt_store"](x[rows])[1])


def test_a_net_of_checkpointed_layers_traces_under_torch_compile():
    torch.manual_seed(0)
    net = S.LogicNet(40, 60, 2, node="walsh", k=4, tau=3.0, seed=0).to(dev)
    x = torch.rand(50, 40, device=dev)

    def grads(f):
        net.zero_grad()
        with S.checkpoint8():
            out = f(x)
        (out * torch.arange(10, device=dev)).sum().backward()
        return out.detach(), [p.grad.clone() for p in net.parameters()]
    y0, g0 = grads(net)
    y1, g1 = grads(torch.compile(net, backend="aot_eager", fullgraph=True))
    assert torch.equal(y0, y1)
    for a, b in zip(g0, g1):
        _close(a, b.double(), "compiled")


@pytest.mark.parametrize("B,F", [(1, 1), (3, 70), (5, 64), (127, 65), (128, 63), (130, 200), (1000, 333), (4093, 90)])
def test_transpose_and_store_in_one_pass(B, F):
    """Bit for bit the transpose followed by the store of its first B columns."""
    from silogic_b200._ops import IMPL
    g = torch.Generator().manual_seed(B)
    x = torch.randn(B, F, generator=g)
    x[:, 0] = 0.75
    if F > 2:
        x[B // 2, 1], x[0, 2] = float("nan"), float("inf")
    x = x.to(dev)
    ldb = _soft.ldb_for(B)
    out, codes, bounds = IMPL["to_feature_major_ckpt"](x, ldb)
    want = IMPL["to_feature_major"](x, ldb)
    wc, wb = IMPL["ckpt_store"](want[:, :B])
    eq = lambda a, b: torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))       # noqa: E731
    assert eq(out, want) and eq(bounds, wb) and torch.equal(codes[:, :ldb], wc[:, :ldb])


@pytest.mark.parametrize("on", [False, True])
def test_a_single_layer_traces_under_torch_compile(on):
    torch.manual_seed(0)
    layer = S.LogicLayer(40, 60, node="gate16", k=4, seed=0).to(dev)
    f = torch.compile(layer, backend="aot_eager", fullgraph=True)
    x = torch.rand(50, 40, device=dev, requires_grad=True)
    gy = torch.randn(50, 60, device=dev)
    wanted = [x] + list(layer.parameters())
    with S.checkpoint8(on):
        y0, y1 = layer(x), f(x)
    assert torch.equal(y0, y1)
    for a, b in zip(torch.autograd.grad(y1, wanted, gy), torch.autograd.grad(y0, wanted, gy)):
        _close(a, b.double(), "compiled")


def test_nothing_is_stored_without_a_backward_pass(monkeypatch):
    """Under no_grad (evaluation inside a training context) no codes are written."""
    from silogic_b200 import _ops
    stored = []
    for name in ("ckpt_store", "to_feature_major_ckpt"):
        monkeypatch.setitem(_ops.IMPL, name, lambda *a, f=_ops.IMPL[name], n=name: (stored.append(n), f(*a))[1])
    torch.manual_seed(0)
    layer = S.LogicLayer(20, 30, node="walsh", k=4, seed=0).to(dev)
    net = S.LogicNet(20, 30, 2, node="gate16", k=4, tau=3.0, seed=0).to(dev)
    conv = S.ConvLogicTree(3, 8, tree_depth=2, k=4, seed=0).to(dev)
    x, img = torch.rand(50, 20, device=dev), torch.rand(5, 3, 8, 8, device=dev)
    with S.checkpoint8():
        with torch.no_grad():
            for f, v in ((layer, x), (net, x), (conv, img)):
                f(v)
        assert stored == []
        for f, v in ((layer, x), (net, x), (conv, img)):
            f(v)
    assert stored == ["to_feature_major_ckpt", "ckpt_store", "ckpt_store", "ckpt_store"]


@pytest.mark.parametrize("on", [False, True])
def test_second_derivatives_are_refused(on):
    """A gradient taken with create_graph=True is right, and raises when it is differentiated (it
    had no graph, and a penalty on it vanished from the loss without a word)."""
    torch.manual_seed(0)
    layer = S.LogicLayer(20, 30, node="walsh", k=4, seed=0).to(dev)
    net = S.LogicNet(20, 30, 2, node="gate16", k=4, tau=3.0, seed=0).to(dev)
    conv = S.ConvLogicTree(3, 8, tree_depth=2, k=4, seed=0).to(dev)
    for f, shape in ((layer, (9, 20)), (net, (9, 20)), (conv, (5, 3, 8, 8))):
        x = torch.rand(shape, device=dev, requires_grad=True)
        wanted = [x] + list(f.parameters())

        def loss():
            with S.checkpoint8(on):
                return (f(x) ** 2).sum()
        plain = torch.autograd.grad(loss(), wanted)
        graph = torch.autograd.grad(loss(), wanted, create_graph=True)
        for a, b in zip(graph, plain):
            assert a.requires_grad
            _close(a.detach(), b.double(), "first derivative")
        for g in graph:
            with pytest.raises(RuntimeError, match="second derivatives"):
                (loss() + (g ** 2).sum()).backward()
