"""Refusals of the token, checkpoint and beam entry points (no GPU needed: arguments are
checked before anything is launched)."""
import ctypes
import os

import pytest
import torch

import silogic_b200 as S
from silogic_b200 import _lib


@pytest.fixture(scope="module")
def L():
    if not os.path.exists(_lib.LIB_PATH):
        from silogic_b200 import build
        build.build()
    return _lib.lib()


def _p(v):
    return ctypes.c_void_p(v)


def test_python_entry_points_refuse_wrong_arguments():
    w, ids = torch.randn(10, 4), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(TypeError, match="weight"):
        S.token_embedding(ids, w.double())
    with pytest.raises(TypeError, match="weight"):
        S.token_embedding(ids, w[0])
    with pytest.raises(TypeError, match="ids"):
        S.token_embedding(ids.float(), w)
    with pytest.raises(RuntimeError, match="CUDA"):
        S.token_embedding(ids, w)
    with pytest.raises(RuntimeError, match="CUDA"):
        S.checkpoint8_store(w)
    with pytest.raises(RuntimeError, match="CUDA"):
        S.beam_step(torch.randn(4, 10), torch.zeros(2, 2))
    with pytest.raises(ValueError, match="scores"):
        S.beam_step(torch.randn(4, 10), torch.zeros(4))
    with pytest.raises(ValueError, match="do not fit"):
        S.beam_step(torch.randn(5, 10), torch.zeros(2, 2))
    with pytest.raises(TypeError, match="logits"):
        S.beam_step(torch.zeros(4, 10, dtype=torch.int64), torch.zeros(2, 2))
    with pytest.raises(ValueError, match="parents"):
        S.beam_reorder(torch.randn(4, 10), torch.zeros(2, 2))
    with pytest.raises(RuntimeError, match="CUDA"):
        S.beam_reorder(torch.randn(4, 10), torch.zeros(2, 2, dtype=torch.int64))


def test_checkpoint8_switch_nests_and_resets_on_errors():
    from silogic_b200 import _soft
    assert _soft.CHECKPOINT8 is False
    with pytest.raises(KeyError):
        with S.checkpoint8():
            assert _soft.CHECKPOINT8 is True
            with S.checkpoint8(False):
                assert _soft.CHECKPOINT8 is False
            assert _soft.CHECKPOINT8 is True
            raise KeyError
    assert _soft.CHECKPOINT8 is False


def test_c_entry_points_refuse_bad_arguments(L):
    # embedding: sizes, types, null pointers, alignment, workspace
    fwd = lambda **k: L.slg_embed_fwd(_p(k.get("ids", 256)), k.get("i64", 1), k.get("N", 4), _p(256),       # noqa: E731
                                      k.get("dt", 0), k.get("V", 10), k.get("D", 8), 1.0, _p(k.get("out", 256)), _p(0))
    assert fwd(N=-1) == 1 and fwd(V=0) == 1 and fwd(D=0) == 1 and fwd(i64=2) == 1
    assert fwd(dt=3) == 3 and fwd(N=1 << 31) == 3 and fwd(V=(1 << 31) - 1) == 3
    assert fwd(ids=0) == 1 and fwd(out=260) == 2 and b"aligned" in L.slg_last_error()
    assert fwd(N=0, ids=0) == 0                                            # nothing to do
    need = L.slg_embed_bwd_workspace_bytes(100, 10, 8, 0)
    assert need > 0 and L.slg_embed_bwd_workspace_bytes(-1, 10, 8, 0) == 0
    bwd = lambda n=100, gw=256, ws=256, size=need, dt=0: L.slg_embed_bwd(                                  # noqa: E731
        _p(256), 1, n, _p(256), dt, 10, 8, 1.0, -1, _p(gw), _p(ws), size, _p(0))
    assert bwd(size=need - 1) == 5 and bwd(gw=0) == 1 and bwd(ws=0) == 1 and bwd(ws=264) == 2
    assert bwd(n=-1) == 1 and bwd(dt=7) == 3
    # checkpoints
    store = lambda x=256, rows=4, cols=10, ldx=10, codes=256, ldc=12, bounds=256, dt=0: L.slg_ckpt_store(  # noqa: E731
        _p(x), dt, rows, cols, ldx, _p(codes), ldc, _p(bounds), _p(0))
    assert store(rows=-1) == 1 and store(ldx=9) == 1 and store(ldc=8) == 1 and store(ldc=11) == 2
    assert store(dt=9) == 3 and store(codes=0) == 1 and store(x=0) == 1 and store(codes=258) == 2 and store(bounds=260) == 2
    assert store(rows=0, codes=0, bounds=0, x=0) == 0
    both = lambda x=256, B=130, F=7, out=256, ldb=132, codes=256, ldc=144, bounds=256: L.slg_to_feature_major_ckpt(  # noqa: E731
        _p(x), B, F, _p(out), ldb, _p(codes), ldc, _p(bounds), _p(0))
    assert both(B=0) == 1 and both(F=-1) == 1 and both(ldb=129) == 1 and both(ldc=131) == 1
    assert both(ldb=260, ldc=272) == 1 and b"last block" in L.slg_last_error()
    assert both(x=0) == 1 and both(out=0) == 1 and both(codes=0) == 1 and both(bounds=0) == 1 and both(bounds=260) == 2
    assert both(F=0, x=0) == 0
    load = lambda x=256, rows=4, cols=10, ldx=10, codes=256, ldc=12, bounds=256, dt=0: L.slg_ckpt_load(    # noqa: E731
        _p(codes), ldc, _p(bounds), rows, cols, _p(x), dt, ldx, _p(0))
    assert load(cols=-1) == 1 and load(ldc=11) == 2 and load(dt=-1) == 3 and load(x=0) == 1
    # beams
    step = lambda B=2, k=4, V=50, ldx=50, w=4, dt=0, fin=0, eos=-1, x=256: L.slg_beam_step(                # noqa: E731
        _p(x), dt, B, k, V, ldx, _p(256), _p(fin), eos, w, _p(256), _p(256), _p(256), _p(0), _p(0))
    assert step(B=-1) == 1 and step(V=0) == 1 and step(ldx=49) == 1 and step(k=33) == 3 and step(w=33) == 3
    assert step(k=1, V=2, ldx=2, w=3) == 1 and step(dt=5) == 3 and step(V=1 << 27, ldx=1 << 27) == 3
    assert step(fin=256, eos=-1) == 1 and step(fin=256, eos=50) == 1 and step(x=0) == 1
    assert step(B=0, x=0) == 0
    rows = lambda i=256, o=512, nb=16, B=2: L.slg_beam_reorder_rows(_p(i), nb, _p(256), B, 4, 4, _p(o), _p(0))   # noqa: E731
    assert rows(i=0) == 1 and rows(o=256) == 1 and rows(nb=-1) == 1 and rows(B=0) == 0 and rows(nb=0) == 0
    assert L.slg_beam_reorder_features(_p(256), 3, 7, _p(256), 2, 4, 4, _p(512), 8, _p(0)) == 1       # rows too short
    assert L.slg_beam_reorder_features(_p(256), 3, 8, _p(256), 2, 4, 4, _p(512), 7, _p(0)) == 1
    assert L.slg_beam_reorder_packed(_p(256), 3, 1, _p(256), 20, 4, 4, _p(512), 2, _p(0)) == 1


def test_checkpoint_backward_refuses_bad_arguments(L):
    need = L.slg_fc_soft_workspace_bytes(512, 8, 1, 2, 100)
    ok = dict(codes=256, ldc=512, bounds=256, I=50, ldb=512, cand=256, conn=256, K=8, ste=0, node=1, ar=2, par=256,
              O=100, wire=0, gy=256, gx=256, gconn=256, gpar=256, ws=256, size=need)

    def call(**k):
        a = dict(ok, **k)
        return L.slg_fc_soft_bwd_ckpt(_p(a["codes"]), a["ldc"], _p(a["bounds"]), a["I"], a["ldb"], _p(a["cand"]),
                                      _p(a["conn"]), a["K"], a["ste"], a["node"], a["ar"], _p(a["par"]), 0, 1.0, a["O"],
                                      a["wire"], _p(a["gy"]), _p(a["gx"]), _p(a["gconn"]), _p(a["gpar"]), _p(a["ws"]),
                                      a["size"], _p(0))
    assert call(I=0) == 1 and call(ldb=0) == 1 and call(K=0) == 1 and call(wire=-1) == 1 and call(O=-1) == 1
    assert call(K=9) == 3 and call(ar=3) == 3 and call(node=4) == 3                # restore instead
    assert call(ldb=510) == 2 and call(ldc=514) == 2 and call(ldc=508) == 1
    assert call(ste=3) == 1 and call(wire=51) == 1 and call(wire=101) == 1
    for name in ("codes", "bounds", "cand", "par", "gy", "gpar", "ws", "gconn"):
        assert call(**{name: 0}) == 1, name
    assert call(gy=264) == 2 and call(gx=264) == 2 and call(codes=258) == 2 and call(bounds=260) == 2
    assert call(size=need - 1) == 5
    assert call(O=0, gx=0) == 0
    for K, node, ar, want in ((8, 0, 2, 1), (1, 3, 2, 1), (9, 0, 2, 0), (4, 1, 3, 0), (4, 4, 2, 0), (4, 5, 2, 0), (0, 1, 2, 0)):
        assert L.slg_fc_soft_bwd_ckpt_built(K, node, ar) == want


@pytest.mark.parametrize("beams", [1, 2, 3, 5, 7, 8, 16, 31, 32])
def test_packed_reorder_sources_lie_in_four_words(beams):
    """The kernel that loads four source words per output word (width >= beams) relies on it."""
    for width in range(beams, 33):
        for word in range(0, 6 * width):
            first = (word * 32 // width * beams) >> 5
            last = ((word * 32 + 31) // width) * beams + beams - 1
            assert last - 32 * first < 128


def test_packed_reorder_refuses_offsets_past_32_bits(L):
    """A word of 32 samples of one-beam results spans 32 entries of the state's beams."""
    beams = 1 << 28
    packed = lambda width, ldi: L.slg_beam_reorder_packed(_p(256), 3, ldi, _p(256), 1, beams, width, _p(512), 1, _p(0))   # noqa: E731
    assert packed(1, beams // 64) == 3 and b"beams per entry" in L.slg_last_error()
    assert packed(1, beams // 64 - 1) == 1                                 # rows too short


def test_checkpoint8_belongs_to_the_thread_that_sets_it():
    """Two threads whose contexts overlap: neither sees nor leaves the other's setting."""
    import threading
    from silogic_b200 import _soft
    inside, left = threading.Event(), threading.Event()
    seen = {}

    def first():
        with S.checkpoint8():
            inside.set()
            assert left.wait(10)
            seen["first, inside"] = _soft.CHECKPOINT8
        seen["first, after"] = _soft.CHECKPOINT8
    t = threading.Thread(target=first)
    t.start()
    assert inside.wait(10)
    seen["other, before"] = _soft.CHECKPOINT8
    with S.checkpoint8(False):
        seen["other, off"] = _soft.CHECKPOINT8
    with S.checkpoint8():
        left.set()
        t.join()
        seen["other, inside"] = _soft.CHECKPOINT8
    seen["other, after"] = _soft.CHECKPOINT8
    assert seen == {"first, inside": True, "first, after": False, "other, before": False, "other, off": False,
                    "other, inside": True, "other, after": False}


def test_checkpoint8_contexts_of_one_thread_may_end_in_any_order():
    """Generators and coroutines interleave contexts in one thread."""
    from silogic_b200 import _soft
    a, b = S.checkpoint8(), S.checkpoint8()
    a.__enter__()
    b.__enter__()
    a.__exit__(None, None, None)
    assert _soft.CHECKPOINT8 is True
    b.__exit__(None, None, None)
    assert _soft.CHECKPOINT8 is False


def test_checkpoint8_is_read_again_by_a_traced_function():
    """torch.compile guards on the thread's setting: a function traced outside is traced again inside."""
    from silogic_b200 import _soft
    f = torch.compile(lambda x: x * 2 if _soft.checkpointing() else x + 1, backend="eager", fullgraph=True)
    x = torch.full((2,), 5.0)
    assert f(x)[0] == 6
    with S.checkpoint8():
        assert f(x)[0] == 10
        with S.checkpoint8(False):
            assert f(x)[0] == 6
    assert f(x)[0] == 6


def test_beams_refuse_tensors_of_two_devices():
    """Shapes alone (fake tensors): the devices are compared before anything is launched."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        make = lambda *s, d, t=torch.float32: torch.empty(s, device=f"cuda:{d}", dtype=t)      # noqa: E731
        with pytest.raises(ValueError, match="scores on cuda:1"):
            S.beam_step(make(4, 10, d=0), make(2, 2, d=1))
        with pytest.raises(ValueError, match="finished on cuda:1"):
            S.beam_step(make(4, 10, d=0), make(2, 2, d=0), finished=make(2, 2, d=1, t=torch.bool), eos=0)
        for layout, state in (("rows", make(4, 7, d=0)), ("features", make(7, 4, d=0)),
                              ("packed", make(7, 1, d=0, t=torch.int64))):
            with pytest.raises(ValueError, match="parents on cuda:1"):
                S.beam_reorder(state, make(2, 2, d=1, t=torch.int64), layout=layout)


def test_reorder_refuses_entries_of_no_beams():
    for layout, state in (("rows", torch.zeros(4, 7)), ("features", torch.zeros(7, 4)),
                          ("packed", torch.zeros(7, 1, dtype=torch.int64))):
        with pytest.raises(ValueError, match="parents"):
            S.beam_reorder(state, torch.zeros(2, 0, dtype=torch.int64), layout=layout)
