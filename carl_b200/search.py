"""Beam search over simulations: selection of continuations and reordering of state.

A group is one planning problem; a beam is one candidate of it, with a score (the
sum of its actions' log-probabilities) and a sim of an env.  A step of a search::

    torch_stream.wait_stream(env_stream)           # the outputs are written on the env's stream
    over = over | env.get_dones().view(over.shape) # an env step resets a sim that is done
    obs = env.get_obs()[:, 0].contiguous()
    best = codec.beam_select(policy(obs).view(...), scores, codec.mask(obs).view(...), finished=over)
    env.reorder(best.parents)                      # the kept beams' sims
    reorder_states([hidden], best.parents)         # the caller's own per-beam state
    history = history.fork(best.parents + first)   # the kept beams' records
    over = over.gather(1, best.parents)            # a lineage that is over stays so
    history.append(best.actions ..., ~over ...)
    env.step(best.actions ...)

with ``env_stream = torch.cuda.ExternalStream(env.stream)``: the env's inputs are
ordered after torch's current stream, but nothing orders torch after the env, so what
reads an env's output, or writes to a tensor that an env call still reads, has to wait.
At the root all beams but one start with a score of -inf: copies of one sim with equal
scores tie everywhere, which says the same several times and is slow (near totals are
ranked in 64 bits, row by row).

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
    ones by the lower beam, then the lower action, and returned in float32: off by up to
    3.5e-6 beyond that rounding (4.5e-6 over the action heads), since a logarithm is
    computed more exactly only where the order needs it.  The same call gives the same
    bits.

    Logits that are not allowed are never looked at (they may be NaN); a logit of -inf
    is not a continuation, and a beam with a score of -inf or NaN, no allowed logit
    above -inf, or an allowed NaN or +inf has none.  Where a group has fewer than
    `width`, the places behind them hold score -inf, parent (place mod beams) and
    action 0, so that parents can always be used as indices.

    Up to 1024 beams, beams * vocab <= 2**30.  No gradient flows through the result.
    """
    return select(logits, scores, mask, width, finished, joint=False)


def _check_device(name: str, t, device) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be on a CUDA device")
    if t.device != device:
        raise ValueError(f"{name} must be on {device}")


def select(logits, scores, mask, width, finished, *, joint: bool) -> BeamStep:
    """Both selections: checks the arguments, allocates the outputs and launches."""
    if not isinstance(logits, torch.Tensor):
        raise TypeError("logits must be a tensor")
    device = logits.device
    _check_device("logits", logits, device)
    _check_device("scores", scores, device)
    kind = _LOGIT_TYPES.get(logits.dtype)
    if kind is None:
        raise TypeError("logits must have dtype float32, bfloat16 or float16")
    if scores.dtype is not torch.float32:
        raise TypeError("scores must have dtype float32")
    shape = logits.shape
    if len(shape) < 2 or shape[-1] < 1 or shape[-2] < 1:
        raise ValueError("logits must have shape [..., beams, vocab] with at least one beam and action")
    lead, beams, vocab = shape[:-2], shape[-2], shape[-1]
    if scores.shape != shape[:-1]:
        raise ValueError("scores must have the shape of logits without its last dimension")
    width = beams if width is None else int(width)
    most_beams, most_width = ((capi.JOINT_MAX_BEAMS, capi.JOINT_MAX_WIDTH) if joint
                              else (capi.BEAM_MAX_BEAMS, capi.BEAM_MAX_WIDTH))
    if beams > most_beams or beams * vocab > capi.BEAM_MAX_CANDIDATES:
        raise ValueError(f"at most {most_beams} beams and {capi.BEAM_MAX_CANDIDATES} continuations of a group")
    if not 1 <= width <= most_width:
        raise ValueError(f"width must be 1 to {most_width}")
    x, x_group, x_beam = _rows(logits, beams, vocab)
    groups = lead[0] if len(lead) == 1 else logits.numel() // (beams * vocab)
    if groups > 0x7fffffff // beams:
        raise ValueError("too many groups")
    s = scores if scores.is_contiguous() else scores.detach().contiguous()
    m = f = m_ptr = f_ptr = None
    m_group = m_beam = 0
    if mask is not None:
        _check_device("mask", mask, device)
        if mask.dtype is not torch.bool:
            raise TypeError("mask must have dtype bool")
        if mask.shape != shape:
            try:
                mask = mask.expand(shape)
            except RuntimeError:
                raise ValueError("mask must be broadcastable to logits") from None
        m, m_group, m_beam = _rows(mask, beams, vocab)
        m_ptr = m.data_ptr()
    if finished is not None:
        _check_device("finished", finished, device)
        if finished.dtype is not torch.bool:
            raise TypeError("finished must have dtype bool")
        if finished.shape != shape[:-1]:
            raise ValueError("finished must have the shape of scores")
        f = finished if finished.is_contiguous() else finished.contiguous()
        f_ptr = f.data_ptr()
    out_shape = (*lead, width)
    best = BeamStep(torch.empty(out_shape, dtype=torch.float32, device=device),
                    torch.empty(out_shape, dtype=torch.int64, device=device),
                    torch.empty((*out_shape, _HEADS) if joint else out_shape, dtype=torch.int32, device=device))
    if groups == 0:
        return best
    args = capi.BeamArgs(x.data_ptr(), s.data_ptr(), m_ptr, f_ptr, best[0].data_ptr(), best[1].data_ptr(),
                         best[2].data_ptr(), None, 0, x_group, x_beam, m_group, m_beam, groups, beams, vocab, width, kind,
                         device.index)
    lib = capi.load()
    if joint:
        capi.check(lib.carlb_joint_select(args, torch._C._cuda_getCurrentRawStream(device.index)))
        return best
    size = ctypes.c_int64()
    capi.check(lib.carlb_beam_workspace(args, size))
    if size.value:
        work = torch.empty(size.value, dtype=torch.uint8, device=device)
        args.workspace, args.workspace_bytes = work.data_ptr(), size.value
    capi.check(lib.carlb_beam_select(args, torch._C._cuda_getCurrentRawStream(device.index)))
    return best


def _rows(t: torch.Tensor, beams: int, vocab: int) -> tuple[torch.Tensor, int, int]:
    """`t` [..., beams, vocab] with a dense last dimension and one stride between
    groups, and its strides of a group and a beam; a copy where it has no such view."""
    stride = t.stride()
    if stride[-1] != 1:
        t = t.detach().contiguous()
        stride = t.stride()
    if len(stride) == 3:
        return t, stride[0], stride[1]
    if len(stride) == 2:
        return t, 0, stride[0]
    t = t.detach().reshape(-1, beams, vocab)
    return t, t.stride(0), t.stride(1)


def reorder_states(states: Sequence[torch.Tensor], parents: torch.Tensor, dim: int = 0) -> None:
    """Moves every group's state to the slots of the beams it became, in place.

    parents  int64 [..., beams], as `beam_select` returns them; groups and beams are
             flattened to rows g * beams + j
    states   contiguous tensors of any dtype whose dimension `dim` counts those rows
             (groups * beams of them); ``dim=1`` is the simulator's word-major layout
             [words, rows, ...]

    Row g * beams + j takes the content that row g * beams + parents[g, j] had; a value
    outside [0, beams) leaves its row as it is.  The tensors must not overlap one
    another or parents.  To autograd it is an in-place operation: a backward pass that
    has saved one of the states raises.  Up to 1024 beams.
    """
    if isinstance(states, torch.Tensor):
        raise TypeError("states must be a sequence of tensors")
    if not isinstance(parents, torch.Tensor) or parents.dtype is not torch.int64:
        raise TypeError("parents must be an int64 tensor")
    if not parents.is_cuda:
        raise ValueError("parents must be on a CUDA device")
    if parents.dim() < 1 or not 1 <= parents.shape[-1] <= capi.BEAM_MAX_BEAMS:
        raise ValueError(f"parents must have shape [..., beams] with 1 to {capi.BEAM_MAX_BEAMS} beams")
    device, rows, beams, count = parents.device, parents.numel(), parents.shape[-1], len(states)
    if rows // beams > 0x7fffffff:
        raise ValueError("too many groups")
    grad = torch.is_grad_enabled()
    arrays = (capi.StateArray * max(1, count))()
    p = parents if parents.is_contiguous() else parents.contiguous()
    at = p.data_ptr()
    spans = [(at, at + 8 * rows)]
    for i, t in enumerate(states):
        if not isinstance(t, torch.Tensor):
            raise TypeError("states must be tensors")
        if t.device != device:
            raise ValueError(f"states must be on {device}")
        shape = t.shape
        d = dim + len(shape) if dim < 0 else dim
        if not 0 <= d < len(shape):
            raise ValueError("dim is out of range")
        if shape[d] != rows:
            raise ValueError(f"dimension {dim} of every state must count the {rows} rows of parents")
        if not t.is_contiguous():
            raise ValueError("states must be contiguous")
        if grad and t.requires_grad:
            raise ValueError("states that require a gradient cannot be moved in place")
        total = t.numel() * t.element_size()
        if total == 0:
            continue
        outer = 1
        for n in shape[:d]:
            outer *= n
        at = t.data_ptr()
        arrays[i] = (at, outer, total // outer, total // outer // rows)
        spans.append((at, at + total))
    if rows == 0 or not count:
        return
    spans.sort()
    if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
        raise ValueError("states must not overlap one another or parents")
    capi.check(capi.load().carlb_reorder_states(arrays, count, p.data_ptr(), rows // beams, beams, device.index,
                                                torch._C._cuda_getCurrentRawStream(device.index)))
    torch.autograd.graph.increment_version(states)  # a backward pass that has saved one must not use it
