"""Beam search over simulations: selection of continuations and reordering of state.

A group is one planning problem; a beam is one candidate of it, with a score (the
sum of its actions' log-probabilities) and a sim of an env.  A step of a search::

    best = codec.beam_select(logits, scores, codec.mask(obs), finished=done)
    env.reorder(best.parents)                      # the kept beams' sims
    reorder_states([hidden], best.parents)         # the caller's own per-beam state
    history = history.fork(best.parents + first)   # the kept beams' records
    env.step(best.actions ...)

The kernels run on torch's current stream of the inputs' device, neither
synchronise nor read values on the host, and can be captured into CUDA graphs.
Inputs must be CUDA tensors; errors are as in ``carl_b200.carl`` (TypeError for
dtypes, ValueError for devices, shapes and ranges, RuntimeError from CUDA).
"""

from __future__ import annotations

import ctypes
from collections.abc import Sequence
from typing import NamedTuple

import torch

from . import capi

_LOGIT_TYPES = {torch.float32: capi.LOGITS_F32, torch.bfloat16: capi.LOGITS_BF16, torch.float16: capi.LOGITS_F16}
_HEADS = 7


class BeamStep(NamedTuple):
    """The kept continuations of each group, best first."""

    scores: torch.Tensor    # float32 [..., width]
    parents: torch.Tensor   # int64 [..., width], beam index inside the group
    actions: torch.Tensor   # int32 [..., width] ([..., width, 7] over the action heads)


def beam_select(logits: torch.Tensor, scores: torch.Tensor, mask: torch.Tensor | None = None, *,
                width: int | None = None, finished: torch.Tensor | None = None) -> BeamStep:
    """The `width` best continuations of each group over its beams and the vocabulary.

    logits    float32, bfloat16 or float16 [..., beams, vocab]
    scores    float32 [..., beams]
    mask      bool, broadcastable to logits: which actions are allowed
    finished  bool [..., beams]: such a beam has one continuation, action 0 at its own score
    width     continuations kept per group, 1 to 128 (default: beams)

    The total of action v of beam k is ``scores[k] + logits[k, v] - logsumexp`` over
    the allowed logits of the beam.  Totals are ranked as if computed in 64 bits, equal
    ones by the lower beam, then the lower action, and returned in float32.  Logits
    that are not allowed are never looked at (they may be NaN); a logit of -inf is not
    a continuation, and a beam with a score of -inf or NaN, no allowed logit above
    -inf, or an allowed NaN or +inf has none.  Where a group has fewer than `width`,
    the places behind them hold score -inf, parent (place mod beams) and action 0, so
    that parents can always be used as indices.

    Up to 1024 beams, beams * vocab <= 2**30.  No gradient flows through the result.
    """
    return select(logits, scores, mask, width, finished, joint=False)


def select(logits, scores, mask, width, finished, *, joint: bool) -> BeamStep:
    """Both selections: checks the arguments, allocates the outputs and launches."""
    for name, t in (("logits", logits), ("scores", scores), ("mask", mask), ("finished", finished)):
        if t is None and name in ("mask", "finished"):
            continue
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a tensor")
        if t.device.type != "cuda":
            raise ValueError(f"{name} must be on a CUDA device")
        if t.device != logits.device:
            raise ValueError(f"{name} must be on {logits.device}")
    kind = _LOGIT_TYPES.get(logits.dtype)
    if kind is None:
        raise TypeError("logits must have dtype float32, bfloat16 or float16")
    if scores.dtype != torch.float32:
        raise TypeError("scores must have dtype float32")
    if logits.dim() < 2 or logits.shape[-1] < 1 or logits.shape[-2] < 1:
        raise ValueError("logits must have shape [..., beams, vocab] with at least one beam and action")
    shape = logits.shape
    beams, vocab = shape[-2], shape[-1]
    if scores.shape != shape[:-1]:
        raise ValueError("scores must have the shape of logits without its last dimension")
    width = beams if width is None else int(width)
    most_beams, most_width = ((capi.JOINT_MAX_BEAMS, capi.JOINT_MAX_WIDTH) if joint
                              else (capi.BEAM_MAX_BEAMS, capi.BEAM_MAX_WIDTH))
    if beams > most_beams or beams * vocab > capi.BEAM_MAX_CANDIDATES:
        raise ValueError(f"at most {most_beams} beams and {capi.BEAM_MAX_CANDIDATES} continuations of a group")
    if not 1 <= width <= most_width:
        raise ValueError(f"width must be 1 to {most_width}")
    args = capi.BeamArgs()
    x = logits.detach()
    if x.stride(-1) != 1:
        x = x.contiguous()
    x = x.reshape(-1, beams, vocab) if x.dim() != 3 else x
    groups = x.shape[0]
    if groups > 0x7fffffff // beams:
        raise ValueError("too many groups")
    s = scores.detach().contiguous()
    args.logits, args.scores = x.data_ptr(), s.data_ptr()
    args.logits_group_stride, args.logits_beam_stride = x.stride(0), x.stride(1)
    m = f = None
    if mask is not None:
        if mask.dtype != torch.bool:
            raise TypeError("mask must have dtype bool")
        try:
            m = mask.expand(shape)
        except RuntimeError:
            raise ValueError("mask must be broadcastable to logits") from None
        if m.stride(-1) != 1:
            m = m.contiguous()
        m = m.reshape(-1, beams, vocab) if m.dim() != 3 else m
        args.mask = m.data_ptr()
        args.mask_group_stride, args.mask_beam_stride = m.stride(0), m.stride(1)
    if finished is not None:
        if finished.dtype != torch.bool:
            raise TypeError("finished must have dtype bool")
        if finished.shape != shape[:-1]:
            raise ValueError("finished must have the shape of scores")
        f = finished.contiguous()
        args.finished = f.data_ptr()
    out_shape = (*shape[:-2], width)
    device = x.device
    best = BeamStep(torch.empty(out_shape, dtype=torch.float32, device=device),
                    torch.empty(out_shape, dtype=torch.int64, device=device),
                    torch.empty((*out_shape, _HEADS) if joint else out_shape, dtype=torch.int32, device=device))
    args.out_scores, args.out_parents, args.out_actions = (t.data_ptr() for t in best)
    args.groups, args.beams, args.vocab, args.width = groups, beams, vocab, width
    args.logit_type, args.device = kind, device.index
    if groups == 0:
        return best
    lib = capi.load()
    stream = torch.cuda.current_stream(device).cuda_stream
    if joint:
        capi.check(lib.carlb_joint_select(args, stream))
        return best
    size = ctypes.c_int64()
    capi.check(lib.carlb_beam_workspace(args, size))
    if size.value:
        work = torch.empty(size.value, dtype=torch.uint8, device=device)
        args.workspace, args.workspace_bytes = work.data_ptr(), size.value
    capi.check(lib.carlb_beam_select(args, stream))
    return best


def reorder_states(states: Sequence[torch.Tensor], parents: torch.Tensor, dim: int = 0) -> None:
    """Moves every group's state to the slots of the beams it became, in place.

    parents  int64 [..., beams], as `beam_select` returns them; groups and beams are
             flattened to rows g * beams + j
    states   contiguous tensors of any dtype whose dimension `dim` counts those rows
             (groups * beams of them); ``dim=1`` is the simulator's word-major layout
             [words, rows, ...]

    Row g * beams + j takes the content that row g * beams + parents[g, j] had; a value
    outside [0, beams) leaves its row as it is.  The tensors must not overlap one
    another.  Up to 1024 beams.
    """
    if isinstance(states, torch.Tensor):
        raise TypeError("states must be a sequence of tensors")
    if not isinstance(parents, torch.Tensor) or parents.dtype != torch.int64:
        raise TypeError("parents must be an int64 tensor")
    if parents.device.type != "cuda":
        raise ValueError("parents must be on a CUDA device")
    if parents.dim() < 1 or not 1 <= parents.shape[-1] <= capi.BEAM_MAX_BEAMS:
        raise ValueError(f"parents must have shape [..., beams] with 1 to {capi.BEAM_MAX_BEAMS} beams")
    rows, beams = parents.numel(), parents.shape[-1]
    arrays = (capi.StateArray * max(1, len(states)))()
    for a, t in zip(arrays, states):
        if not isinstance(t, torch.Tensor):
            raise TypeError("states must be tensors")
        if t.device != parents.device:
            raise ValueError(f"states must be on {parents.device}")
        if not -t.dim() <= dim < t.dim():
            raise ValueError("dim is out of range")
        d = dim % t.dim()
        if t.shape[d] != rows:
            raise ValueError(f"dimension {dim} of every state must count the {rows} rows of parents")
        if not t.is_contiguous():
            raise ValueError("states must be contiguous")
        if t.requires_grad and torch.is_grad_enabled():
            raise ValueError("states that require a gradient cannot be moved in place")
        if t.numel() == 0:
            continue
        outer = 1
        for n in t.shape[:d]:
            outer *= n
        slab = t.numel() // outer * t.element_size()
        a.data, a.outer, a.outer_stride, a.inner_bytes = t.data_ptr(), outer, slab, slab // rows
    if rows == 0 or not len(states):
        return
    p = parents.contiguous()
    capi.check(capi.load().carlb_reorder_states(arrays, len(states), p.data_ptr(), rows // beams, beams, p.device.index,
                                                torch.cuda.current_stream(p.device).cuda_stream))
