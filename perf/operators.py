"""Cases and plain forms of the token and training-memory operators.

Three operators that turn logic-gate networks into token-in, token-out models:

* ``embed``: embedding lookup with scaling, and its gradient by sorted tokens;
* ``store`` and ``layer``: activation checkpoints in 8 bits -- stored and read back, and a
  soft logic layer's training step whose backward pass works from them;
* ``beam``: beam search's selection over beams and vocabulary, with the decoder state
  (bit-packed circuit state, feature-major columns or rows) reordered by it.

``run`` computes a case in elementary torch operations, or (``own``) through the
framework's public entry points.
"""
import math

import numpy as np
import torch

own = False

DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
ES = {"fp32": 4, "bf16": 2, "fp16": 2}
BLOCK = 128                 # columns that share one (lo, step) pair of a checkpoint
TINY = 2.0 ** -100          # a block whose step is below this is constant
INV255 = float(np.float32(1.0) / np.float32(255.0))

# coefficients of (1, a, b, ab) of the 16 two-input gates
GATES = [[0, 0, 0, 0], [0, 0, 0, 1], [0, 1, 0, -1], [0, 1, 0, 0], [0, 0, 1, -1], [0, 0, 1, 0],
         [0, 1, 1, -2], [0, 1, 1, -1], [1, -1, -1, 1], [1, -1, -1, 2], [1, 0, -1, 0],
         [1, 0, -1, 1], [1, -1, 0, 0], [1, -1, 0, 1], [1, 0, 0, -1], [1, 0, 0, 0]]


# -------------------------------------------------------------------- cases
def listed():
    return [
        # the tokens of one decoding step (4 beams): only latency counts
        dict(name="embed 4 tokens", op="embed", train=False, dtype="fp32", vocab=10000, dim=784,
             tokens=4, pad=False),
        # a small ragged training batch: odd row length (rows start on no vector boundary),
        # prime number of tokens, padding tokens without a gradient
        dict(name="embed ragged", op="embed", train=True, dtype="fp16", vocab=8000, dim=331,
             tokens=1021, pad=True),
        # an ordinary training batch: 64 samples of 256 tokens
        dict(name="embed train", op="embed", train=True, dtype="fp32", vocab=10000, dim=784,
             tokens=16384, pad=True),
        # a large training batch over a large vocabulary, 16-bit table
        dict(name="embed large", op="embed", train=True, dtype="bf16", vocab=65536, dim=1024,
             tokens=262144, pad=False),
        # the activations of one small layer (width 2000, 64 samples)
        dict(name="store small", op="store", dtype="fp32", rows=2000, cols=64),
        # one layer's activations at the largest batch (width 10000, 65,536 samples)
        dict(name="store large", op="store", dtype="fp32", rows=10000, cols=65536),
        # first layer of a gate16 net with fixed wiring on binary features
        dict(name="layer first", op="layer", node="gate16", arity=2, k=1, inputs=784, width=8000,
             batch=1024, binary=True),
        # hidden layer of a 10,000-wide Walsh net with Top-8 wiring
        dict(name="layer hidden", op="layer", node="walsh", arity=2, k=8, inputs=10000, width=10000,
             batch=4096, binary=False),
        # lookup-table nodes with four inputs, odd sizes everywhere
        dict(name="layer lut", op="layer", node="multilinear", arity=4, k=4, inputs=1283,
             width=2001, batch=333, binary=False),
        # one sentence, 4 beams: logits are class counts / tau, full of exact ties
        dict(name="beam one", op="beam", dtype="fp32", batch=1, beams=4, vocab=2000, counts=True,
             state="packed", features=2000),
        # odd sizes, 16-bit logits, fp32 activations as the state
        dict(name="beam odd", op="beam", dtype="bf16", batch=7, beams=5, vocab=8191, counts=False,
             state="features", features=1283),
        # a serving batch over a large vocabulary
        dict(name="beam batch", op="beam", dtype="fp32", batch=64, beams=8, vocab=32000,
             counts=False, state="packed", features=10000),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["embed", "store", "layer", "beam"])
    if op == "embed":
        train = rng.random() < 0.75
        vocab, dim = _log(rng, 2000, 65536), _log(rng, 64, 1024)
        return dict(op=op, train=train, dtype=rng.choice(["fp32", "bf16", "fp16"]), vocab=vocab,
                    dim=dim if rng.random() < 0.4 else max(64, dim // 16 * 16),
                    tokens=_log(rng, 1, 262144 if dim <= 512 else 131072), pad=rng.random() < 0.5)
    if op == "store":
        rows = _log(rng, 200, 10000)
        return dict(op=op, dtype=rng.choice(["fp32", "bf16", "fp16"]), rows=rows,
                    cols=_log(rng, 1, 65536))
    if op == "layer":
        node, arity = rng.choice([("gate16", 2), ("walsh", 2), ("walsh", 2), ("multilinear", 2),
                                  ("multilinear", 4)])
        k = rng.choice([1, 4, 8]) if arity == 2 else rng.choice([2, 4])
        return dict(op=op, node=node, arity=arity, k=k, inputs=_log(rng, 64, 10000),
                    width=_log(rng, 200, 10000), batch=_log(rng, 1, 4096 if arity == 2 else 1024),
                    binary=rng.random() < 0.3)
    beams = rng.choice([1, 2, 3, 4, 5, 8])
    return dict(op=op, dtype=rng.choice(["fp32", "bf16", "fp16"]), batch=_log(rng, 1, 64),
                beams=beams, vocab=_log(rng, 200, 32000), counts=rng.random() < 0.4,
                state=rng.choice(["packed", "features", "rows"]), features=_log(rng, 200, 10000))


# ------------------------------------------------------------------- inputs
def prepare(case, seed):
    c, dev = case, "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    rand = lambda *s: torch.rand(*s, generator=g, device=dev)       # noqa: E731
    randn = lambda *s: torch.randn(*s, generator=g, device=dev)     # noqa: E731
    st = dict(c)
    if c["op"] == "embed":
        V, D, N, dt = c["vocab"], c["dim"], c["tokens"], DT[c["dtype"]]
        # token frequencies fall as 1 / rank, as in text; ranks are spread over the vocabulary
        rank = (torch.exp(rand(N) * math.log(V + 1.0)).long() - 1).clamp_(0, V - 1)
        st["ids"] = torch.randperm(V, generator=g, device=dev)[rank]
        st["padding"] = 0 if c["pad"] else None
        if c["pad"]:
            st["ids"][rand(N) < 0.1] = 0
        st["scale"] = math.sqrt(D)
        st["weight"] = (randn(V, D) * (1.0 / D)).to(dt).requires_grad_(c["train"])
        if c["train"]:
            st["grad"] = randn(N, D).to(dt)
    elif c["op"] == "store":
        # soft activations: probabilities, many of them near 0 or 1
        st["x"] = torch.sigmoid(2.0 * randn(c["rows"], c["cols"])).to(DT[c["dtype"]])
    elif c["op"] == "layer":
        I, O, B, A, K = c["inputs"], c["width"], c["batch"], c["arity"], c["k"]
        x = (rand(B, I) < 0.3).float() if c["binary"] else torch.sigmoid(2.0 * randn(B, I))
        st["x"] = x.requires_grad_(True)
        st["gy"] = randn(B, O)
        st["cand"] = torch.randint(0, I, (O, A, K), generator=g, device=dev)
        st["conn"] = randn(O, A, K).requires_grad_(True) if K > 1 else None
        st["params"] = randn(O, 16 if c["node"] == "gate16" else 2 ** A).requires_grad_(True)
        st["layer"] = _user_layer(c, st) if own else None
    else:
        B, k, V, F = c["batch"], c["beams"], c["vocab"], c["features"]
        if c["counts"]:         # class counts of a circuit, divided by tau = 10
            x = torch.floor(rand(B * k, V) * rand(B * k, V) * 40.0) / 10.0
        else:
            x = 4.0 * randn(B * k, V)
        x[rand(B * k, V) < 0.02] = -math.inf             # forbidden tokens
        st["logits"] = x.to(DT[c["dtype"]])
        st["scores"] = -20.0 * rand(B, k)
        st["finished"] = rand(B, k) < 0.15
        st["eos"] = 1
        if c["state"] == "packed":
            words = max(2, (B * k + 127) // 128 * 2)
            bits = torch.randint(-2 ** 63, 2 ** 63 - 1, (F, words), generator=g, device=dev)
            keep = torch.arange(words * 64, device=dev).view(words, 64) < B * k
            one = torch.ones((), dtype=torch.int64, device=dev)
            st["words"] = bits & torch.where(keep, one << torch.arange(64, device=dev), 0).sum(1)
        elif c["state"] == "features":
            cols = (B * k + 3) // 4 * 4
            st["words"] = torch.where(torch.arange(cols, device=dev) < B * k, rand(F, cols), 0.0)
        else:
            st["words"] = rand(B * k, F)
    return st


def _user_layer(c, st):
    """The layer module that a user's program holds.  It is built with one node, and then
    given the case's wiring and parameters: drawing the wiring takes seconds."""
    import silogic_b200 as S
    layer = S.LogicLayer(c["inputs"], 1, node=c["node"], arity=c["arity"], k=c["k"],
                         connectome="topk" if c["k"] > 1 else "fixed", seed=0).cuda()
    conn, node = layer._conn, layer.node
    layer.out_dim = node.out_dim = conn.out_dim = c["width"]
    if c["k"] > 1:
        conn.cand, conn.conn = st["cand"], torch.nn.Parameter(st["conn"].detach())
    else:
        conn.idx = st["cand"][:, :, 0]
    conn.cand_i32 = st["cand"].to(torch.int32)
    setattr(node, node.param_name, torch.nn.Parameter(st["params"].detach()))
    return layer


# --------------------------------------------------------------------- run
def run(st):
    return _RUN[st["op"], own](st)


def _embed_own(st):
    import silogic_b200 as S
    y = S.token_embedding(st["ids"], st["weight"], scale=st["scale"], padding_idx=st["padding"])
    if not st["train"]:
        return y
    return y, torch.autograd.grad(y, st["weight"], st["grad"])[0]


def _embed_plain(st):
    w = st["weight"].detach()
    y = (w[st["ids"]].float() * st["scale"]).to(w.dtype)
    if not st["train"]:
        return y
    g = st["grad"].float()
    if st["padding"] is not None:
        g = torch.where((st["ids"] == st["padding"])[:, None], 0.0, g)
    gw = torch.zeros(w.shape, device=w.device).index_add_(0, st["ids"], g) * st["scale"]
    return y, gw.to(w.dtype)


def _store_own(st):
    import silogic_b200 as S
    return S.checkpoint8_store(st["x"]).restore()


def _blocks(x, fill):
    """[rows, cols] as [rows, blocks, BLOCK], the last block filled up."""
    rows, cols = x.shape
    pad = -cols % BLOCK
    if pad:
        x = torch.cat([x, torch.full((rows, pad), fill, dtype=x.dtype, device=x.device)], 1)
    return x.view(rows, -1, BLOCK)


def _codes(x, inv255=INV255):
    """The 8-bit codes of [rows, cols], and the (lo, step) of each block of a row."""
    lo = _blocks(x, math.inf).amin(2, keepdim=True)
    hi = _blocks(x, -math.inf).amax(2, keepdim=True)
    step = (hi - lo) * inv255
    flat = step < TINY
    inv = torch.full_like(lo, 255.0) / torch.where(flat, 1.0, hi - lo)
    code = torch.where(flat, 0.0, torch.round((_blocks(x, 0.0) - lo) * inv).clamp_(0.0, 255.0))
    return code, lo, torch.where(flat, 0.0, step)


def _values(code, lo, step, cols):
    """The values that 8-bit codes stand for."""
    return (code * step + lo).reshape(code.shape[0], -1)[:, :cols]


def _store_plain(st):
    x = st["x"]
    return _values(*_codes(x.float()), x.shape[1]).to(x.dtype)


def _layer_own(st):
    import silogic_b200 as S
    layer = st["layer"]
    with S.checkpoint8():
        y = layer(st["x"])
    wanted = [st["x"], layer.node.param] + ([layer._conn.conn] if st["conn"] is not None else [])
    return [y.detach()] + list(torch.autograd.grad(y, wanted, st["gy"]))


def _softmax(v):
    e = torch.exp(v - v.amax(-1, keepdim=True))
    return e / e.sum(-1, keepdim=True)


def _mix(x, cand, w):
    """x [inputs, B] -> gathered [out, arity, K, B] and mixed operands [out, arity, B]."""
    xs = x[cand]
    return xs, (xs if w is None else xs * w[..., None]).sum(2)


def _corners(arity, dev):
    """[2^arity, arity] truth values: bit j of the row number."""
    p = torch.arange(2 ** arity, device=dev)
    return (p[:, None] >> torch.arange(arity, device=dev)) & 1


def _terms(node, a):
    """The terms of a node that its parameters multiply, [out, P, B], with their derivatives
    by the operands, [out, P, arity, B]."""
    o, A, B = a.shape
    if node == "multilinear":           # weight of a corner: prod_j (a_j or 1 - a_j)
        on = _corners(A, a.device)[:, :, None] == 1                        # [P, A, 1]
        f = torch.where(on, a[:, None], 1.0 - a[:, None])                  # [o, P, A, B]
        d = torch.where(on, 1.0, -1.0)
    else:                               # monomials: prod of the chosen operands (gate16: a, b;
        on = _corners(A, a.device)[:, :, None] == 1                        # Walsh: 2a - 1)
        u = a if node == "gate16" else 2.0 * a - 1.0
        f = torch.where(on, u[:, None], 1.0)
        d = torch.where(on, 1.0 if node == "gate16" else 2.0, 0.0)
    skip = torch.eye(A, device=a.device, dtype=torch.bool)[None, None, :, :, None]
    rest = torch.where(skip, 1.0, f[:, :, None]).prod(3)                   # [o, P, A, B]
    return f.prod(2), rest * d


def _layer_plain(st):
    node, cand, conn, p = st["node"], st["cand"], st["conn"], st["params"].detach()
    x = st["x"].detach().t().contiguous()                                  # [inputs, B]
    gy = st["gy"].t()                                                      # [out, B]
    w = _softmax(conn.detach()) if conn is not None else None
    if node == "gate16":
        basis = torch.tensor(GATES, dtype=torch.float32, device=p.device)
        probs = _softmax(p)
        coef = (probs[:, :, None] * basis).sum(1)
    else:
        coef = p if node == "walsh" else 1.0 / (1.0 + torch.exp(-p))

    def value(a):
        t, dt = _terms(node, a)
        z = (coef[:, :, None] * t).sum(1)
        return t, dt, (1.0 / (1.0 + torch.exp(-z)) if node == "walsh" else z)

    y = value(_mix(x, cand, w)[1])[2]
    # the backward pass sees the 8-bit checkpoint of x
    xs, a = _mix(_values(*_codes(x), x.shape[1]), cand, w)
    t, dt, v = value(a)
    dz = gy * v * (1.0 - v) if node == "walsh" else gy
    ga = (coef[:, :, None, None] * dt).sum(1) * dz[:, None]                # [out, arity, B]
    gc = (dz[:, None] * t).sum(2)                                          # [out, P]
    gt = ga[:, :, None] * w[..., None] if w is not None else ga[:, :, None]
    gx = torch.zeros_like(x).index_add_(0, cand.reshape(-1), gt.reshape(-1, x.shape[1]))
    if node == "gate16":
        gp = (gc[:, None] * basis).sum(2)
        gp = probs * (gp - (probs * gp).sum(1, keepdim=True))
    else:
        gp = gc if node == "walsh" else gc * coef * (1.0 - coef)
    out = [y.t().contiguous(), gx.t().contiguous(), gp]
    if w is not None:
        gw = (ga[:, :, None] * xs).sum(3)
        out.append(w * (gw - (w * gw).sum(2, keepdim=True)))
    return out


def _beam_own(st):
    import silogic_b200 as S
    r = S.beam_step(st["logits"], st["scores"], finished=st["finished"], eos=st["eos"])
    state = S.beam_reorder(st["words"], r.parents, layout=st["state"])
    return r.scores, r.parents, r.tokens, r.finished, state


def _gather_bits(words, src):
    """Bit r of every row becomes bit src[r]; the bits past the samples stay 0."""
    at = torch.arange(64, device=words.device)
    bits = ((words[:, :, None] >> at) & 1).reshape(words.shape[0], -1)
    out = torch.zeros_like(bits)
    out[:, :src.numel()] = bits[:, src]
    return (out.view(words.shape[0], -1, 64) << at).sum(2)


def _beam_plain(st):
    x, scores, done, eos = st["logits"].float(), st["scores"], st["finished"], st["eos"]
    B, k = scores.shape
    V = x.shape[1]
    x = x.view(B, k, V)
    m = x.amax(2, keepdim=True)
    d = torch.where(m > -math.inf, x - m, -math.inf)
    s = torch.exp(d).sum(2, keepdim=True)
    c = torch.where(s > 0, d - torch.log(s) + scores[:, :, None], -math.inf)
    last = torch.where(torch.arange(V, device=x.device) == eos, scores[:, :, None], -math.inf)
    c = torch.where(done[:, :, None], last, c).reshape(B, k * V)
    best, at = torch.sort(c, dim=1, descending=True, stable=True)
    best, at = best[:, :k].clone(), at[:, :k]
    parents, tokens = at // V, at % V
    finished = torch.gather(done, 1, parents) | (tokens == eos)
    src = (torch.arange(B, device=x.device)[:, None] * k + parents).reshape(-1)
    w = st["words"]
    if st["state"] == "packed":
        state = _gather_bits(w, src)
    elif st["state"] == "features":
        state = torch.zeros_like(w)
        state[:, :B * k] = w[:, src]
    else:
        state = w[src]
    return best, parents, tokens, finished, state


_RUN = {("embed", True): _embed_own, ("embed", False): _embed_plain,
        ("store", True): _store_own, ("store", False): _store_plain,
        ("layer", True): _layer_own, ("layer", False): _layer_plain,
        ("beam", True): _beam_own, ("beam", False): _beam_plain}


# -------------------------------------------------------------------- work
def work(case):
    c = case
    if c["op"] == "embed":
        V, D, N, es = c["vocab"], c["dim"], c["tokens"], ES[c["dtype"]]
        b, f = N * 8 + (min(N, V) + N) * D * es, N * D
        if c["train"]:
            b, f = b + (N + V) * D * es, f + N * D + V * D
    elif c["op"] == "store":
        n = c["rows"] * c["cols"]
        held = n + c["rows"] * -(-c["cols"] // BLOCK) * 8
        b, f = 2 * n * ES[c["dtype"]] + 2 * held, 8 * n
    elif c["op"] == "layer":
        I, O, B, A, K = c["inputs"], c["width"], c["batch"], c["arity"], c["k"]
        P = 4 if c["node"] == "gate16" else 2 ** A
        raw = 16 if c["node"] == "gate16" else P
        held = I * B + I * -(-B // BLOCK) * 8
        par = 4 * O * (A * K * (3 if K > 1 else 1) + 2 * raw)
        b = 4 * B * (2 * I + 2 * O) + 2 * held + par
        # mixing, node, and in the backward pass: again, by candidate, by input
        f = B * O * (A * K * 2 * 4 + P * (A + 2) * 3)
    else:
        n = c["batch"] * c["beams"]
        size = {"packed": max(2, (n + 127) // 128 * 2) * 8, "features": (n + 3) // 4 * 16,
                "rows": n * 4}[c["state"]] * c["features"]
        b = n * c["vocab"] * ES[c["dtype"]] + 2 * size + n * (4 + 1 + 4 + 8 + 8 + 1)
        f = n * c["vocab"] * 4
    return {"bytes": float(b), "flops": float(f)}


# ------------------------------------------------------------------- exact
def exact(case, seed):
    """The operators from their definitions in 64 bits."""
    st = prepare(dict(case), seed)
    return {"embed": _embed_exact, "store": _store_exact, "layer": _layer_exact,
            "beam": _beam_exact}[case["op"]](st)


def _embed_exact(st):
    w = st["weight"].detach().double().requires_grad_(True)
    y = torch.index_select(w, 0, st["ids"]) * st["scale"]
    if not st["train"]:
        return y.detach()
    g = st["grad"].double()
    if st["padding"] is not None:
        g = g.masked_fill((st["ids"] == st["padding"])[:, None], 0.0)
    return y.detach(), torch.autograd.grad(y, w, g)[0]


def _read_back(x):
    """Checkpoint values of [rows, cols] in 64 bits, block by block of columns."""
    out = torch.empty_like(x)
    for c0 in range(0, x.shape[1], BLOCK):
        part = x[:, c0:c0 + BLOCK]
        lo, hi = part.min(1, keepdim=True).values, part.max(1, keepdim=True).values
        width = hi - lo
        code = torch.round((part - lo) / torch.where(width == 0, 1.0, width) * 255.0)
        out[:, c0:c0 + BLOCK] = lo + code * width / 255.0
    return out


def _store_exact(st):
    return _read_back(st["x"].double())


def _layer_exact(st):
    node, cand = st["node"], st["cand"]
    p = st["params"].detach().double().requires_grad_(True)
    conn = st["conn"].detach().double().requires_grad_(True) if st["conn"] is not None else None

    def layer(x):                                                          # x [inputs, B]
        O, A, K = cand.shape
        ops = []
        for j in range(A):
            xs = torch.index_select(x, 0, cand[:, j].reshape(-1)).view(O, K, -1)
            if conn is not None:
                xs = (torch.softmax(conn[:, j], 1)[:, :, None] * xs)
            ops.append(xs.sum(1))
        if node == "gate16":
            q = torch.softmax(p, 1) @ torch.tensor(GATES, dtype=torch.float64, device=p.device)
            a, b = ops
            return q[:, 0:1] + q[:, 1:2] * a + q[:, 2:3] * b + q[:, 3:4] * a * b
        table = p if node == "walsh" else torch.sigmoid(p)
        cur = [table[:, i:i + 1] for i in range(2 ** A)]
        for a in ops:                   # fold in one operand at a time, lowest bit first
            if node == "walsh":
                cur = [lo + (2.0 * a - 1.0) * hi for lo, hi in zip(cur[0::2], cur[1::2])]
            else:
                cur = [lo + a * (hi - lo) for lo, hi in zip(cur[0::2], cur[1::2])]
        return torch.sigmoid(cur[0]) if node == "walsh" else cur[0]

    x = st["x"].detach().double().t().contiguous()
    with torch.no_grad():
        y = layer(x).t()
    seen = _read_back(x).requires_grad_(True)
    wanted = [seen, p] + ([conn] if conn is not None else [])
    g = torch.autograd.grad(layer(seen), wanted, st["gy"].double().t())
    return [y, g[0].t()] + list(g[1:])


def _beam_exact(st):
    x, scores, done = st["logits"].double(), st["scores"].double(), st["finished"]
    B, k = scores.shape
    V = x.shape[1]
    c = torch.log_softmax(x, 1).view(B, k, V) + scores[:, :, None]
    only = torch.full_like(c, -math.inf)
    only[:, :, st["eos"]] = scores
    c = torch.where(done[:, :, None], only, c).view(B, k * V)
    best, at = torch.sort(c, dim=1, descending=True, stable=True)
    at = at[:, :k]
    state = st["words"]
    if state.is_floating_point():
        src = (torch.arange(B, device=x.device)[:, None] * k + at // V).reshape(-1)
        if st["state"] == "rows":
            state = state[src]
        else:
            state = torch.cat([state[:, src], state[:, B * k:]], 1)
    else:
        state = None
    return best[:, :k], at // V, at % V, None, state
