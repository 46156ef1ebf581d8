"""Beam search on token logits: one selection step over beams and vocabulary, and the
reordering of the decoder's state -- rows, feature-major activations, or the bit-packed
activations of a hard circuit -- by the chosen beams."""
from collections import namedtuple

import torch

from . import _hard, _soft
from ._lib import call, ptr, require_cuda, stream_ptr
from ._ops import DTYPE_ID

BEAM_MAX = 32           # SLG_BEAM_MAX

#: ``scores`` fp32, ``parents`` and ``tokens`` int64, ``finished`` bool (None without ``eos``),
#: each ``[B, width]``, best first
BeamStep = namedtuple("BeamStep", "scores parents tokens finished")


def beam_step(logits, scores, finished=None, eos=None, width=None):
    """The ``width`` (default: as many as there are) best continuations of each entry's beams.

    ``logits`` ``[B, beams, V]`` or ``[B * beams, V]`` (float32, bfloat16 or float16; class
    counts / tau of a circuit, or soft logits), ``scores`` ``[B, beams]`` = each beam's sum of log
    probabilities (-inf: not in use).  A candidate's score is
    ``log_softmax(logits)[b, v] + scores[b]`` in 32 bits; scores that are equal there (of
    different logits too) go to the lowest beam, then the lowest token.  A beam with ``finished[b]`` goes on with ``eos`` alone, at its score.
    Masked logits (-inf or NaN) and all candidates of a beam at -inf score -inf: they are
    chosen only when nothing else is left, by beam and token too."""
    if scores.dim() != 2:
        raise ValueError(f"beam_step: scores must be [B, beams], got {tuple(scores.shape)}")
    B, beams = scores.shape
    if logits.dtype not in DTYPE_ID:
        raise TypeError(f"beam_step: logits must be float32, bfloat16 or float16, got {logits.dtype}")
    V = logits.shape[-1] if logits.dim() else 0
    if V >= 1 << 27:
        raise ValueError(f"beam_step: vocabulary of {V} (must be below 2**27)")
    if logits.shape != (B * beams, V) and logits.shape != (B, beams, V):
        raise ValueError(f"beam_step: logits {tuple(logits.shape)} do not fit scores {tuple(scores.shape)}")
    if not (logits.is_cuda and scores.is_cuda and (finished is None or finished.is_cuda)):
        require_cuda(logits, scores, finished)
    dev = logits.device
    if scores.device != dev or finished is not None and finished.device != dev:
        raise ValueError(f"beam_step: logits on {dev}, scores on {scores.device}, finished on "
                         f"{finished.device if finished is not None else None}")
    width = beams if width is None else int(width)
    if not 1 <= beams <= BEAM_MAX or not 1 <= width <= BEAM_MAX:
        raise ValueError(f"beam_step: beams and width must be in 1..{BEAM_MAX}, got {beams} and {width}")
    if width > beams * V:
        raise ValueError(f"beam_step: width {width} exceeds the {beams * V} candidates")
    if eos is not None and not 0 <= eos < V:
        raise ValueError(f"beam_step: eos {eos} not in the vocabulary of {V}")
    if finished is not None:
        if eos is None:
            raise ValueError("beam_step: finished needs eos")
        if finished.shape != scores.shape or finished.dtype not in (torch.bool, torch.uint8):
            raise ValueError("beam_step: finished must be bool, of the shape of scores")
        finished = finished.contiguous()
    x = logits if logits.dim() == 2 else logits.reshape(B * beams, V)
    if B and (x.stride(1) != 1 and V > 1 or x.stride(0) < V):
        x = x.contiguous()
    if scores.requires_grad or logits.requires_grad:      # a choice has no gradient
        scores, x = scores.detach(), x.detach()
    scores = scores.float().contiguous()
    out = scores.new_empty((B, width))
    parents, tokens = scores.new_empty((2, B, width), dtype=torch.int64).unbind(0)
    done = scores.new_empty((B, width), dtype=torch.bool) if eos is not None else None
    call("slg_beam_step", x.data_ptr(), DTYPE_ID[x.dtype], B, beams, V, max(x.stride(0), V), scores.data_ptr(),
         ptr(finished), -1 if eos is None else int(eos), width, out.data_ptr(), parents.data_ptr(),
         tokens.data_ptr(), ptr(done), stream_ptr(dev))
    return BeamStep(out, parents, tokens, done)


def beam_reorder(state, parents, layout="rows", beams=None):
    """The decoder state after a step: sample ``e * width + n`` is the state's sample
    ``e * beams + parents[e, n]``, for ``parents`` ``[B, width]`` of :func:`beam_step`.

    ``layout``: ``"rows"`` -- ``[B * beams, ...]`` of any type; ``"features"`` -- feature-major
    fp32 ``[F, ldb]``; ``"packed"`` -- bit-packed ``[F, ldw]`` int64 words, sample s = bit
    ``s % 64`` of word ``s // 64``.  ``beams`` (default: ``width``; rows: from the shape) is
    the number of beams that the state holds per entry."""
    if parents.dim() != 2 or parents.dtype != torch.int64 or parents.shape[1] == 0:
        raise ValueError(f"beam_reorder: parents must be [B, width] int64, got {tuple(parents.shape)} {parents.dtype}")
    if not (state.is_cuda and parents.is_cuda):
        require_cuda(state, parents)
    if state.device != parents.device:
        raise ValueError(f"beam_reorder: state on {state.device}, parents on {parents.device}")
    B, width = parents.shape
    parents = parents.contiguous()
    st = stream_ptr(state.device)
    if state.requires_grad:
        state = state.detach()
    state = state.contiguous()
    if layout == "rows":
        if beams is None:
            beams = state.shape[0] // B if B else width
        if state.dim() < 1 or state.shape[0] != B * beams:
            raise ValueError(f"beam_reorder: {tuple(state.shape)} does not hold {B} entries of {beams} beams")
        out = state.new_empty((B * width,) + tuple(state.shape[1:]))
        nbytes = out.numel() * out.element_size() // (B * width) if B else 0
        call("slg_beam_reorder_rows", state.data_ptr(), nbytes, parents.data_ptr(), B, beams, width, out.data_ptr(), st)
        return out
    beams = width if beams is None else int(beams)
    if layout == "features":
        want, size, ld_for, fn = torch.float32, 1, _soft.ldb_for, "slg_beam_reorder_features"
    elif layout == "packed":
        want, size, ld_for, fn = torch.int64, 64, _hard.ldw_for, "slg_beam_reorder_packed"
    else:
        raise ValueError(f"beam_reorder: unknown layout {layout!r}")
    if state.dim() != 2 or state.dtype != want:
        raise ValueError(f"beam_reorder: {layout} state must be [F, ld] {want}, got {tuple(state.shape)} {state.dtype}")
    F, ld = state.shape
    if beams < 1 or ld * size < B * beams:
        raise ValueError(f"beam_reorder: rows of {ld} do not hold {B} entries of {beams} beams")
    out = torch.empty_like(state) if beams == width else state.new_empty((F, ld_for(B * width)))
    call(fn, state.data_ptr(), F, ld, parents.data_ptr(), B, beams, width, out.data_ptr(), out.shape[1], st)
    return out
