"""Beam selection (flat and over the action heads) and state reordering.

Tolerances of the scores: an output is rounded once to float32 (2^-24 relative),
and the logarithms of the softmax sums that a beam's totals share are computed with
float32 terms.  With u = 2^-24 and d the distance of a logit from its row's largest:

flat   a term is off by d u (the difference), d (u + u / 4) (its product with
       log2(e), and that constant) and 4 u (ex2.approx, 2^-22); d averages at most
       log(vocab) <= log(2^30) = 20.8 under the softmax; partial sums of 8 terms add
       7 u, and are added in 64 bits: 20.8 * 2.25 u + 11 u = 58 u = 3.5e-6.
joint  as above per head with d at most log(3) = 1.1 on average and 2 additions:
       (1.1 * 2.25 + 4 + 2) u = 8.5 u, seven heads and six products 66 u, and logf's
       unit in the last place of at most log(648) = 6.5, 2^-21 = 8 u: 74 u = 4.5e-6.

Parents and actions are whole numbers and equal."""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest

from carl_b200 import _build, capi
from search_oracle import HEADS, best_continuations, joint_actions

SUM_ERROR = 3.5e-6
JOINT_SUM_ERROR = 4.5e-6
DTYPES = ["float32", "bfloat16", "float16"]


# ---- refusals (no GPU) -----------------------------------------------------------------


@pytest.fixture(scope="module")
def lib():
    _build.build()
    return capi.load()


def _args(**kw):
    a = capi.BeamArgs(logits=64, scores=64, out_scores=64, out_parents=64, out_actions=64, workspace=64,
                      workspace_bytes=1 << 40, logits_group_stride=72, logits_beam_stride=18, groups=2, beams=4, vocab=18,
                      width=4)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("joint", [False, True])
@pytest.mark.parametrize("bad, needle", [
    (dict(groups=-1), "groups"), (dict(beams=0), "beams"), (dict(beams=1025), "beams"), (dict(width=0), "width"),
    (dict(width=129), "width"), (dict(logit_type=3), "logit_type"), (dict(vocab=0), "vocab"), (dict(logits=None), "null"),
    (dict(out_actions=None), "null"), (dict(logits=66), "aligned"), (dict(out_parents=68), "aligned"),
    (dict(logits_beam_stride=-1), "strides"),
])
def test_select_refuses_before_launch(lib, joint, bad, needle):
    fn = lib.carlb_joint_select if joint else lib.carlb_beam_select
    assert fn(_args(**bad), None) == capi.ERR_VALUE
    assert needle in lib.carlb_last_error(None).decode()


def test_select_limits_by_kind(lib):
    assert lib.carlb_joint_select(_args(beams=33), None) == capi.ERR_VALUE
    assert lib.carlb_joint_select(_args(width=33), None) == capi.ERR_VALUE
    assert lib.carlb_joint_select(_args(vocab=19), None) == capi.ERR_VALUE
    assert lib.carlb_beam_select(_args(beams=1024, vocab=1 << 21), None) == capi.ERR_VALUE
    # Whether this selection needs a workspace is the library's choice; too little is refused.
    size = ctypes.c_int64()
    big = _args(groups=64, beams=64, vocab=100000)
    assert lib.carlb_beam_workspace(big, size) == capi.OK and size.value > 0
    big.workspace_bytes = size.value - 1
    assert lib.carlb_beam_select(big, None) == capi.ERR_VALUE
    assert "workspace" in lib.carlb_last_error(None).decode()
    assert lib.carlb_beam_select(None, None) == capi.ERR_VALUE
    assert lib.carlb_beam_select(_args(groups=0), None) == capi.OK


def test_reorder_refuses_before_launch(lib):
    ok = capi.StateArray(64, 1, 0, 4)
    call = lambda arr, count, parents, groups, beams: lib.carlb_reorder_states(arr, count, parents, groups, beams, 0, None)  # noqa: E731
    assert call(None, 1, 64, 2, 4) == capi.ERR_VALUE
    assert call(ok, -1, 64, 2, 4) == capi.ERR_VALUE
    assert call(ok, 1, None, 2, 4) == capi.ERR_VALUE
    assert call(ok, 1, 64, 2, 0) == capi.ERR_VALUE
    assert call(ok, 1, 64, 2, 1025) == capi.ERR_VALUE
    assert call(capi.StateArray(None, 1, 0, 4), 1, 64, 2, 4) == capi.ERR_VALUE
    assert call(capi.StateArray(64, 3, 31, 4), 1, 64, 2, 4) == capi.ERR_VALUE
    assert "overlap" in lib.carlb_last_error(None).decode()
    assert call(ok, 1, 64, 0, 4) == capi.OK and call(None, 0, None, 2, 4) == capi.OK
    assert lib.carlb_reorder(None, 64, 4) == capi.ERR_VALUE


def test_python_refuses_cpu_tensors_and_types():
    import torch
    from carl_b200.action import CARLActionCodec
    from carl_b200.search import beam_select, reorder_states

    x, s = torch.zeros(2, 4, 18), torch.zeros(2, 4)
    for select in (beam_select, CARLActionCodec().beam_select):
        with pytest.raises(ValueError, match="CUDA"):
            select(x, s)
        with pytest.raises(TypeError, match="logits"):
            select([1.0], s)
    with pytest.raises(ValueError, match="18"):
        CARLActionCodec().beam_select(x[..., :17], s)
    with pytest.raises(ValueError, match="CUDA"):
        reorder_states([x], torch.zeros(2, 4, dtype=torch.int64))
    with pytest.raises(TypeError, match="int64"):
        reorder_states([x], s)
    with pytest.raises(TypeError, match="sequence"):
        reorder_states(x, torch.zeros(2, 4, dtype=torch.int64))


# ---- selection --------------------------------------------------------------------------


def _inputs(G, K, V, dtype, masked, finished, seed):
    import torch

    rng = np.random.default_rng(seed)
    x = torch.from_numpy(rng.normal(0, 3, (G, K, V)).astype(np.float32)).to(getattr(torch, dtype))
    s = torch.from_numpy((-5 * rng.random((G, K))).astype(np.float32))
    m = torch.from_numpy(rng.random((G, K, V)) < 0.7) if masked else None
    if masked and K > 1:
        m[0, K - 1] = False                      # a beam without a legal action
    f = torch.from_numpy(rng.random((G, K)) < 0.25) if finished else None
    if finished:
        s[:, 0] = -math.inf                      # a dead beam, finished or not
    return x, s, m, f


def _check(x, s, m, f, width, heads=None, fn=None, sum_error=SUM_ERROR):
    import torch
    from carl_b200.action import CARLActionCodec
    from carl_b200.search import beam_select

    fn = fn or (beam_select if heads is None else CARLActionCodec().beam_select)
    cuda = lambda t: None if t is None else t.cuda()  # noqa: E731
    best = fn(cuda(x), cuda(s), cuda(m), width=width, finished=cuda(f))
    m3 = None if m is None else m.expand(x.shape).numpy()
    es, ep, ea = best_continuations(x.float().numpy(), s.numpy(), m3, None if f is None else f.numpy(), width, heads)
    assert best.parents.dtype == torch.int64 and best.actions.dtype == torch.int32 and best.scores.dtype == torch.float32
    np.testing.assert_array_equal(best.parents.cpu().numpy(), ep)
    np.testing.assert_array_equal(best.actions.cpu().numpy(), ea if heads is None else joint_actions(ea))
    got = best.scores.cpu().double().numpy()
    np.testing.assert_array_equal(np.isfinite(got), np.isfinite(es))
    ok = np.isfinite(es)
    assert (np.abs(got[ok] - es[ok]) <= sum_error + 2.0 ** -24 * np.abs(es[ok])).all()
    return best


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("G, K, V, width", [
    (1, 1, 1, 1), (1, 1, 7, 3), (3, 2, 18, 5), (5, 8, 90, 8), (7, 5, 648, 4), (2, 33, 1023, 33), (3, 8, 1025, 64),
    (2, 3, 4099, 128), (1, 8, 50257, 8), (2, 64, 2048, 17), (1, 1024, 33, 128), (300, 4, 31, 4), (2, 2, 131072, 1),
    (4001, 3, 41, 4), (2000, 2, 130, 16), (650, 2, 8003, 8), (600, 9, 1500, 12),
])
@pytest.mark.parametrize("masked, finished", [(False, False), (True, True)])
def test_flat_selection(dtype, G, K, V, width, masked, finished):
    _check(*_inputs(G, K, V, dtype, masked, finished, G + K + V), width)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("G, K, width", [(1, 1, 1), (1, 8, 8), (9, 3, 5), (5, 32, 32), (40, 7, 16), (301, 8, 8), (4, 31, 2),
                                         (1, 1, 32), (130, 2, 4)])
@pytest.mark.parametrize("masked, finished", [(False, False), (True, True)])
def test_joint_selection(dtype, G, K, width, masked, finished):
    x, s, m, f = _inputs(G, K, 18, dtype, masked, finished, G + K)
    if masked:
        m[:, :, [0, 3, 6, 9, 11, 13, 16]] |= True     # the neutral choices
        m[0, K - 1, 9:11] = False                     # a head without a legal choice
    _check(x, s, m, f, width, HEADS, sum_error=JOINT_SUM_ERROR)


@pytest.mark.gpu
@pytest.mark.parametrize("V", [40, 5000])
def test_flat_selection_edge_values(V):
    """NaN and infinities, allowed and masked; empty rows; fewer continuations than places; -0 and +0."""
    import torch

    rng = np.random.default_rng(5)
    x, s, m, _ = _inputs(12, 4, V, "float32", True, False, 9)
    low = torch.finfo(torch.float32).min
    x[0, 0, 3], m[0, 0, 3] = math.nan, True          # kills its beam
    x[1, 1, 4], m[1, 1, 4] = math.inf, True
    x[2, 0, :5], m[2, 0, :5] = math.nan, False       # masked: never looked at
    x[2, 1, :5], m[2, 1, :5] = math.inf, False
    x[3, :, 2:] = -math.inf                          # two continuations a beam at most
    x[4] = low                                       # the type's lowest value everywhere
    m[5] = False                                     # a group without a continuation
    m[6] = False
    m[6, 2, V - 1] = True                            # exactly one
    x[7] = 0.0
    x[7, :, ::2] = -0.0                              # equal to +0: ties by index
    s[7] = -1.0
    m[7] = True
    x[8, 0], m[8, 0] = math.nan, True                # every allowed logit is NaN
    s[9, 1], s[9, 2], s[9, 3] = math.nan, -math.inf, -1e30
    x[10, 0, 0], m[10, 0, 0] = 1e30, True            # one logit takes all
    x[11] = torch.from_numpy(rng.integers(0, 3, (4, V)).astype(np.float32))   # many ties
    _check(x, s, m, None, 16)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("G, K, V, width", [(3, 8, 648, 8), (1300, 3, 700, 16), (2, 5, 30011, 16), (2, 4, 9001, 128),
                                            (1, 33, 5000, 40), (2, 2, 100003, 64)])
def test_equal_logits(dtype, G, K, V, width):
    """Rows that an untrained policy gives: more elements at the bar than there is room for, and the first of them win."""
    import torch

    x = torch.zeros(G, K, V, dtype=getattr(torch, dtype))
    s = -torch.arange(G * K, dtype=torch.float32).view(G, K) % 7
    _check(x, s, None, None, width)
    m = torch.ones(G, K, V, dtype=torch.bool)
    m[:, :, : V // 2] = False                        # the first legal action far into the row
    m[:, 0, 3::5] = True
    f = torch.zeros(G, K, dtype=torch.bool)
    f[:, K - 1] = True
    x[:, :, 1::2] = -0.0
    x[:, :, 7::11] = 0.5                             # many at two levels
    _check(x, torch.full((G, K), -1.0), m, f, width) # equal beams: the lower one


@pytest.mark.gpu
@pytest.mark.parametrize("G, K, V, width", [(3, 8, 30011, 64), (2, 64, 5000, 128), (5, 16, 648, 16), (2, 2, 9000, 100),
                                            (1, 12, 70000, 40)])
def test_one_beam_has_all_the_best(G, K, V, width):
    """The bar that the threads' maxima make is far too low, and is raised; rows ascend, so that what is found first
    is the worst."""
    import torch

    rng = np.random.default_rng(V)
    x = rng.normal(0, 2, (G, K, V)).astype(np.float32)
    x[0] = np.sort(x[0], -1)
    x[0, :, : V // 3] = np.linspace(3, 3.001, V // 3, dtype=np.float32)   # a dense third above most of the rest
    s = np.tile(-4.0 * np.arange(K, dtype=np.float32), (G, 1))
    _check(torch.from_numpy(x), torch.from_numpy(s), None, None, width)


@pytest.mark.gpu
@pytest.mark.parametrize("K, V, width, spread", [(8, 30011, 64, 1e-1), (8, 30011, 64, 1e-3), (16, 9000, 128, 1e-2),
                                                 (6, 648, 16, 1e-3), (64, 5000, 32, 1e-2)])
def test_scores_do_not_depend_on_what_was_found_first(K, V, width, spread):
    """More reaches the bar than there is room for, so that the next bar depends on what came first.  Beams 3 and 4 have
    one of the best places each, and near totals of theirs lie at many places behind the last; beams 1 and 2 are
    near in front.  The scores near zero show the last bits of a normaliser."""
    import torch
    from carl_b200.search import beam_select

    rng = np.random.default_rng(V + K)
    G = 24
    x = rng.normal(0, 1, (G, K, V)).astype(np.float32)
    dense = V // 3
    x[:, 0, :dense] = np.linspace(9, 9 + spread, dense, dtype=np.float32)
    at = rng.permutation(V)[:43]
    for k, top in ((1, 2e-3), (2, 2e-3 + 2e-6), (3, 1e-3), (4, 5e-4)):
        x[:, k, at[0]] = 8.9 + 0.001 * k + top
    # Totals of beams 3 and 4 down beam 0's, from a fifth of the way behind the last place on.
    down = np.linspace(dense - 1.2 * width, max(0, dense - 12 * width), 42).astype(int)
    for g in range(G):
        for j, place in enumerate(down):
            for k in (3, 4):
                x[g, k, at[1 + j]] = (x[g, 0, place] - 9.5) + 8.9 + 0.001 * k
    zero = 8.9 + 0.001 * np.arange(K)                # the logit that makes a total of 0
    zero[0] = 9.5                                    # beam 0's dense totals begin at -0.5
    s = (np.log(np.exp(x.astype(np.float64)).sum(-1)) - zero).astype(np.float32)
    x, s = torch.from_numpy(x).cuda(), torch.from_numpy(s).cuda()
    first = beam_select(x, s, width=width)
    assert all(set(range(5)) <= set(row) for row in first.parents.tolist())
    for _ in range(60):
        again = beam_select(x, s, width=width)
        assert torch.equal(again.scores, first.scores) and torch.equal(again.parents, first.parents)
        assert torch.equal(again.actions, first.actions)
    _check(x.cpu(), s.cpu(), None, None, width)


@pytest.mark.gpu
@pytest.mark.parametrize("V, width", [(30012, 64), (9000, 16), (200000, 128)])
def test_near_totals_behind_the_best_of_a_chunk(V, width):
    """A beam of equal logits, and one with four legal neighbours: one far in front, three within a few float32 steps
    of the equal ones, before or behind them."""
    import torch

    G = 9
    x, m = np.zeros((G, 2, V), np.float32), np.ones((G, 2, V), bool)
    at = V // 8 * 4
    m[:, 1] = False
    m[:, 1, at:at + 4] = True
    x[:, 1, at + 1] = 5
    s = np.zeros((G, 2), np.float32)
    s[:, 1] = np.log(np.exp(5.0) + 3) - np.log(V)
    for g in range(G):
        for _ in range(abs(g - 4)):
            s[g, 1] = np.nextafter(s[g, 1], np.float32(np.sign(g - 4) * 100), dtype=np.float32)
    best = _check(torch.from_numpy(x), torch.from_numpy(s), torch.from_numpy(m), None, width)
    assert sorted(set((best.parents == 1).sum(-1).tolist())) == [1, 4]


@pytest.mark.gpu
def test_near_totals_are_ranked_in_64_bits():
    """Beams whose normalisers differ by less than float32 sums can tell."""
    import torch

    rng = np.random.default_rng(11)
    for V in (600, 20011):
        row = rng.normal(0, 2, V).astype(np.float32)
        x = np.tile(row, (6, 8, 1))
        x[:, :, V // 2] = -8 - 8 * rng.random((6, 8)).astype(np.float32)     # e^-8 .. e^-16 of a sum of about e^2 V
        x[5] = row                                                           # equal beams: ties by index
        s = np.full((6, 8), -2.0, np.float32)
        _check(torch.from_numpy(x), torch.from_numpy(s), None, None, 24)
        fin = np.zeros((6, 8), bool)
        fin[:, 3] = True                             # a finished beam right at another's best total
        es, _, _ = best_continuations(x, s, None, None, 1)
        s2 = s.copy()
        s2[:, 3] = es[:, 0].astype(np.float32)
        _check(torch.from_numpy(x), torch.from_numpy(s2), None, torch.from_numpy(fin), 24)


@pytest.mark.gpu
@pytest.mark.parametrize("K, width", [(8, 8), (8, 5), (3, 16), (32, 32), (2, 4)])
def test_joint_near_totals_are_ranked_in_64_bits(K, width):
    """Beams whose normalisers differ by 1e-3 to 1e-7: in one choice that hardly counts."""
    import torch

    rng = np.random.default_rng(17)
    x = np.tile(rng.normal(0, 2, (40, 1, 18)).astype(np.float32), (1, K, 1))
    x[:, :, 8] = x[:, :, 6:8].max(-1) - 7 - 8 * rng.random((40, K)).astype(np.float32)
    x[20:, :, 8] = x[20:, :1, 8]                     # equal beams: ties by index
    _check(torch.from_numpy(x), torch.full((40, K), -2.0), None, None, width, HEADS, sum_error=JOINT_SUM_ERROR)


def _check_beside_rounding(x, s, width, mask=None, heads=HEADS):
    """A selection where scores and logits of two beams may differ and their totals be the same real number (score -2
    and a sum of 3, score -3 and a sum of 4, or the same logits in another order): which of these comes first is then a
    matter of how each side rounds.  Logits are whole and at most 12, scores 3e8 or more or at most 4: where totals are
    below 32, a normaliser, a base and a total round by at most 2^-49 each; seven tops and logarithms added up (or a sum
    of exponentials whose terms and partial sums are off by as much in relation), the base and the total make 16
    roundings a side, 2.9e-14, and two totals on two sides 1.2e-13.  Far from zero (from 1e3 on) a normaliser's last
    bit vanishes in the score, and totals are equal.  A beam's own continuations have exact sums and keep their order."""
    from carl_b200.action import CARLActionCodec
    from carl_b200.search import beam_select

    ROUNDING = 1.2e-13
    G, K, _ = x.shape
    joint = heads is HEADS
    fn = CARLActionCodec().beam_select if joint else beam_select
    best = fn(x.cuda(), s.cuda(), None if mask is None else mask.cuda(), width=width)
    x, s = x.double().numpy(), s.double().numpy()
    x = x if mask is None else np.where(mask.numpy(), x, -np.inf)
    sums, norm, at = np.zeros((G, K, 1)), 0.0, 0
    for h in heads:
        row = x[..., at:at + h]
        top = row.max(-1, keepdims=True)
        norm = norm + top[..., 0] + np.log(np.exp(row - top).sum(-1))
        sums = (sums[..., None] + row[:, :, None, :]).reshape(G, K, -1)
        at += h
    totals = (s - norm)[..., None] + sums
    want = -np.sort(-totals.reshape(G, -1), -1)[:, :width]
    rounding = np.where(np.abs(want) < 1e3, ROUNDING, 0.0)
    parents = best.parents.cpu().numpy()
    actions = best.actions.cpu().numpy()
    actions = np.ravel_multi_index(tuple(np.moveaxis(actions, -1, 0)), HEADS) if joint else actions
    got = totals[np.arange(G)[:, None], parents, actions]
    assert (np.abs(got - want) <= rounding).all()
    error = JOINT_SUM_ERROR if joint else SUM_ERROR
    assert (np.abs(best.scores.cpu().double().numpy() - want) <= error + rounding + 2.0 ** -24 * np.abs(want)).all()
    order = np.argsort(-totals, -1, kind="stable")           # a beam's continuations are taken in order
    for g in range(G):
        for k in np.unique(parents[g]):
            taken = actions[g][parents[g] == k]
            assert (taken == order[g, k, :taken.size]).all()
        for i in range(1, width):                            # and of totals that are equal far from zero the lower beam's
            assert want[g, i] < want[g, i - 1] or want[g, i] > -1e3 or parents[g, i] >= parents[g, i - 1]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("K", [2, 3, 8, 32])
@pytest.mark.parametrize("width", [1, 2, 3, 5, 8, 16, 32])
def test_joint_near_totals_behind_ties(dtype, K, width):
    """Whole logits tie within a beam, so that the first near total of another beam may lie far behind the last place;
    the normalisers differ in one choice that hardly counts, down to less than float32 sums can tell."""
    import torch

    rng = np.random.default_rng(100 * K + width)
    G = 300
    x = np.tile(rng.integers(-1, 3, (G, 1, 18)).astype(np.float32), (1, K, 1))
    x[:, :, 8] = x[:, :, 6:8].max(-1) - 9 - 7 * rng.random((G, K)).astype(np.float32)   # e^-9 .. e^-16 of the head's sum
    x[200:, :, 17] = x[200:, :, 16] - 9 - 7 * rng.random((100, K)).astype(np.float32)
    x = torch.from_numpy(x).to(getattr(torch, dtype))
    s = torch.full((G, K), -2.0)
    s[100:] -= torch.from_numpy(rng.integers(0, 2, (200, K)).astype(np.float32))   # some beams a whole step behind
    _check_beside_rounding(x, s, width)


@pytest.mark.filterwarnings("ignore:invalid value")
@pytest.mark.gpu
@pytest.mark.parametrize("K, width", [(1, 1), (1, 8), (1, 32), (2, 4), (3, 16), (8, 8), (32, 32)])
def test_joint_equal_totals_of_unequal_sums(K, width):
    """Sums of logits that differ and round to one 64-bit total (or to one sum) go to the lower action: scores that
    swallow the logits, logits that swallow others, and scores of +inf."""
    import torch

    rng = np.random.default_rng(10 * K + width)
    x = rng.normal(0, 2, (40, K, 18)).astype(np.float32)
    s = -20.0 - 4.0 * rng.random((40, K)).astype(np.float32)
    s[:5] = -1e30                                    # every total is the score
    s[5:8, K // 2] = -1e30                           # one beam's are
    x[8:12] = 0.0
    x[8:12, :, 17] = 1e-20                           # below the last bit of any total
    x[12:16] = rng.integers(-1, 2, (4, K, 18))
    x[12:16, :, 0], x[12:16, :, 4] = 1e-20, -1e-25
    x[16:20, :, 2], x[16:18, :, 10] = 1e20, -1e20    # the other heads vanish beside it
    x[20:24] = x[20:24] * 1e-42                      # subnormal logits
    s[24:27] = np.inf
    s[27:30, K - 1] = np.inf
    x[24:30, :, [1, 5, 9]] = -np.inf
    x[30:33, :, 3:6] = 0.0, 1e-20, 2e-20
    s[33:36] = 0.0
    x[33:36] = -0.0
    x[33:36, :, 0] = -3e38
    x, s = torch.from_numpy(x), torch.from_numpy(s)
    m = torch.rand(40, K, 18, generator=torch.Generator().manual_seed(K)) < 0.9
    m[33:36] = True                                  # equal beams: their normalisers too
    for mask in (None, m):
        best = _check(x, s, mask, None, width, HEADS, sum_error=JOINT_SUM_ERROR)
        got = best.scores.cpu()
        assert not torch.isnan(got).any() and not (got[:24] == math.inf).any() and not (got[30:] == math.inf).any()
        if mask is None:
            assert (got[24:30, 0] == math.inf).all()


@pytest.mark.filterwarnings("ignore:invalid value")
@pytest.mark.gpu
def test_flat_scores_of_infinity():
    """A beam whose score is +inf wins with every action it has, in their order."""
    import torch

    for V, width in ((40, 16), (648, 8), (30011, 64), (9001, 100)):
        x, s, m, _ = _inputs(6, 4, V, "float32", True, False, V)
        s[:3, 2] = math.inf
        s[3] = math.inf
        x[0, 2, 3:], x[1, 2, ::2] = -math.inf, -math.inf
        m[0, 2, 0] = True
        best = _check(x, s, m, None, width)
        got = best.scores.cpu()
        assert not torch.isnan(got).any() and (got[:4, 0] == math.inf).all()


@pytest.mark.gpu
@pytest.mark.parametrize("joint", [False, True])
@pytest.mark.parametrize("score", [-1e6, -3e8, -1e10, -1e11, -3e11, -1e12, -1e14, -1e16, -1e20])
def test_scores_far_from_zero(joint, score):
    """Totals whose unit in the last place is from far below to far above a normaliser's error: score - normaliser is
    one of two neighbours, and beams of equal scores differ by that.  Logits are whole, so no total is half way; the
    beams of a group differ in one of them, by 1e-5 and less in the normaliser."""
    import torch

    rng = np.random.default_rng(int(-10 * np.log10(-score)) + 1000)
    G, K = 800, 8
    for V, width in [(18, 8)] if joint else [(40, 8), (40, 16), (1500, 20)]:
        x = np.tile(rng.integers(-3, 4, (G, 1, V)).astype(np.float32), (1, K, 1))
        x[:, :, 8] = -8 - 4 * rng.random((G, K))
        s = np.full((G, K), score, np.float32)
        s[G // 2:, ::2] = -4.0                       # some beams near zero; the others are reached where few logits are left
        m = np.ones((G, K, V), bool)
        if not joint:
            m[G // 2:, ::2, 1:8] = False
            m[G // 2:, ::2, 9:] = False
        _check_beside_rounding(torch.from_numpy(x), torch.from_numpy(s), width, torch.from_numpy(m),
                               HEADS if joint else (V,))


@pytest.mark.gpu
def test_joint_groups_do_not_depend_on_their_neighbours():
    """A group whose totals are near is ranked again; the scores of the others in its warp keep their bits."""
    import torch
    from carl_b200.action import CARLActionCodec

    x, s, _, _ = _inputs(64, 4, 18, "float32", False, False, 8)
    alone = CARLActionCodec().beam_select(x.cuda(), s.cuda())
    x[::2], s[::2] = x[::2, :1].clone(), -1.0        # equal beams: all near
    mixed = CARLActionCodec().beam_select(x.cuda(), s.cuda())
    assert torch.equal(alone.scores[1::2], mixed.scores[1::2]) and torch.equal(alone.actions[1::2], mixed.actions[1::2])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_joint_ties_between_heads(dtype):
    """Small whole logits: many joint actions have exactly the same sum."""
    import torch

    rng = np.random.default_rng(3)
    x = torch.from_numpy(rng.integers(-1, 2, (20, 6, 18)).astype(np.float32)).to(getattr(torch, dtype))
    x[10:] = x[10:, :1]                              # equal beams too
    s = torch.full((20, 6), -3.0)
    _check(x, s, None, None, 32, HEADS, sum_error=JOINT_SUM_ERROR)
    x = x.float()
    x[0, 0, 1], x[1, 1, 5], x[2, 2, 17] = math.nan, math.inf, -math.inf
    x[3, 0, 0:3] = -math.inf
    s[4, 0], s[5, 1] = math.nan, -math.inf
    _check(x.to(getattr(torch, dtype)), s, None, None, 32, HEADS, sum_error=JOINT_SUM_ERROR)


@pytest.mark.gpu
@pytest.mark.parametrize("joint", [False, True])
def test_selection_layouts(joint):
    """Broadcast masks, strided and offset logits, more leading dimensions, none, no groups."""
    import torch
    from carl_b200.action import CARLActionCodec
    from carl_b200.search import beam_select

    fn = CARLActionCodec().beam_select if joint else beam_select
    heads, V = (HEADS, 18) if joint else (None, 77)
    x, s, m, f = _inputs(6, 5, V, "bfloat16", True, True, 21)
    error = JOINT_SUM_ERROR if joint else SUM_ERROR
    _check(x, s, m[:1, :1], None, 5, heads, sum_error=error)                        # [1, 1, V]
    _check(x, s, m[0, 0], f, 5, heads, sum_error=error)                             # [V]
    _check(x, s, torch.ones(6, 5, 1, dtype=torch.bool), f, 5, heads, sum_error=error)
    want = fn(x.cuda(), s.cuda(), m.cuda(), finished=f.cuda())
    wide = torch.full((6, 5, V + 9), 99.0, dtype=torch.bfloat16, device="cuda")
    wide[..., 3:3 + V] = x.cuda()
    wide_m = torch.zeros((6, 5, V + 5), dtype=torch.bool, device="cuda")
    wide_m[..., 1:1 + V] = m.cuda()
    views = [(wide[..., 3:3 + V], wide_m[..., 1:1 + V]),
             (x.cuda().transpose(0, 1).contiguous().transpose(0, 1), m.cuda().transpose(1, 2).contiguous().transpose(1, 2)),
             (x.cuda().transpose(1, 2).contiguous().transpose(1, 2), m.cuda())]
    for vx, vm in views:
        got = fn(vx, s.cuda(), vm, finished=f.cuda())
        assert torch.equal(got.parents, want.parents) and torch.equal(got.actions, want.actions)
        # A row's alignment decides which of its terms are summed together, so each side has the
        # normaliser's error of its own and its own rounding (2 * 2^-24).
        live = torch.isfinite(want.scores)
        assert torch.equal(live, torch.isfinite(got.scores))
        off = (got.scores.double() - want.scores.double())[live].abs()
        assert (off <= 2 * error + 2.0 ** -23 * want.scores[live].abs()).all()
    got = fn(x.cuda().view(2, 3, 5, V), s.cuda().view(2, 3, 5), m.cuda().view(2, 3, 5, V), finished=f.cuda().view(2, 3, 5))
    assert got.parents.shape == (2, 3, 5) and torch.equal(got.parents.view(6, 5), want.parents)
    one = fn(x[2].cuda(), s[2].cuda(), m[2].cuda(), finished=f[2].cuda())
    assert torch.equal(one.parents, want.parents[2]) and torch.equal(one.actions, want.actions[2])
    none = fn(x[:0].cuda(), s[:0].cuda())
    assert none.scores.shape == (0, 5)
    same = fn(x[:1].cuda().expand(4, 5, V), s[:1].cuda().expand(4, 5))   # broadcast groups
    assert torch.equal(same.parents[0], same.parents[3])


@pytest.mark.gpu
def test_selection_refusals_on_the_device():
    import torch
    from carl_b200.search import beam_select

    x, s = torch.zeros(2, 4, 9, device="cuda"), torch.zeros(2, 4, device="cuda")
    for exc, call in [(TypeError, lambda: beam_select(x.double(), s)), (TypeError, lambda: beam_select(x, s.half())),
                      (ValueError, lambda: beam_select(x, s[:1])), (ValueError, lambda: beam_select(x[0, 0], s[0, 0])),
                      (TypeError, lambda: beam_select(x, s, x)), (ValueError, lambda: beam_select(x, s, s.bool())),
                      (ValueError, lambda: beam_select(x, s, width=0)), (ValueError, lambda: beam_select(x, s, width=129)),
                      (TypeError, lambda: beam_select(x, s, finished=s)), (ValueError, lambda: beam_select(x, s.cpu())),
                      (ValueError, lambda: beam_select(x, s, finished=s[:, :2].bool())),
                      (ValueError, lambda: beam_select(x[..., :0], s))]:
        with pytest.raises(exc):
            call()


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """Rows more than 2^31 elements apart, by stride."""
    import torch
    from carl_b200.search import beam_select

    far = 2 ** 31 + 64
    store = torch.empty(far + 2 * 4096, dtype=torch.bfloat16, device="cuda")
    x = torch.as_strided(store, (2, 2, 4096), (far, 4096, 1))
    small = torch.randn(2, 2, 4096, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).bfloat16()
    x.copy_(small)
    s = torch.zeros(2, 2, device="cuda")
    a, b = beam_select(x, s), beam_select(small, s)
    assert all(torch.equal(u, v) for u, v in zip(a, b))


# ---- reordering -------------------------------------------------------------------------


def _reordered(t, parents, dim):
    import torch

    K = parents.shape[-1]
    p = parents.reshape(-1, K)
    own = torch.arange(K, device=p.device)
    p = torch.where((p >= 0) & (p < K), p, own)
    source = (p + torch.arange(0, p.numel(), K, device=p.device)[:, None]).flatten()
    return t.index_select(dim, source)


@pytest.mark.gpu
@pytest.mark.parametrize("G, K", [(1, 1), (1, 8), (5, 3), (64, 8), (2, 64), (1, 1024), (37, 7), (3, 1000)])
def test_reorder_rows_and_words(G, K):
    import torch
    from carl_b200.search import reorder_states

    g = torch.Generator("cuda").manual_seed(G * 1000 + K)
    n = G * K
    parents = torch.randint(-2, K + 2, (G, K), device="cuda", generator=g)     # some name no beam
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    rows = [rand(n, 6, 63), rand(n, 5).bfloat16(), rand(n) > 0, rand(n, 3).half(), rand(n, 1000), rand(n, 7, 13).to(torch.uint8),
            rand(n, 2).double(), rand(n, 0), rand(n, 4099).bfloat16()]
    want = [_reordered(t, parents, 0) for t in rows]
    reorder_states(rows, parents)
    assert all(torch.equal(a, b) for a, b in zip(rows, want))
    words = [rand(76, n, 6), rand(33, n, 1), rand(5, n), rand(3, 2, n, 4).bfloat16().movedim(2, 1).contiguous()]
    want = [_reordered(t, parents, 1) for t in words]
    reorder_states(words, parents, dim=1)
    assert all(torch.equal(a, b) for a, b in zip(words, want))
    odd = torch.randn(n * 6 + 1, device="cuda")[1:].view(n, 6)                 # 4-byte aligned only
    want = _reordered(odd, parents, 0)
    reorder_states([odd], parents)
    assert torch.equal(odd, want)


@pytest.mark.gpu
@pytest.mark.parametrize("G, K", [(4001, 3), (1500, 8), (700, 16), (301, 17), (97, 64), (5001, 2), (11, 1000)])
def test_reorder_large_arrays(G, K):
    """Sizes at which rows go through registers and short rows as dense runs, with odd ends and slabs."""
    import torch
    from carl_b200.search import reorder_states

    g = torch.Generator("cuda").manual_seed(G + K)
    n = G * K
    parents = torch.randint(-1, K + 1, (G, K), device="cuda", generator=g)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    # Runs: slabs of 1, 2, 3, 6 and 7 words a row (odd slab strides too), one slab, 128 words a row.
    words = [rand(29, n, w) for w in (1, 2, 3, 6, 7)] + [rand(1, n, 5), rand(13, n, 2).bfloat16(), rand(2, n, 128)]
    want = [_reordered(t, parents, 1) for t in words]
    reorder_states(words, parents, dim=1)
    assert all(torch.equal(a, b) for a, b in zip(words, want))
    # Rows: 256 bytes to 12 KB, whole columns or not, at an offset.
    store = rand(n + 1, 64)
    rows = [rand(n, 6, 252), rand(n, 64), rand(n, 516).bfloat16(), rand(n, 1030).half(), rand(n, 2500), store[1:], rand(n) > 0]
    want = [_reordered(t, parents, 0) for t in rows]
    first = store[0].clone()
    reorder_states(rows, parents)
    assert all(torch.equal(a, b) for a, b in zip(rows, want)) and torch.equal(store[0], first)


@pytest.mark.gpu
def test_reorder_many_arrays_and_neighbours():
    """More arrays than one launch takes; nothing around an array is touched."""
    import torch
    from carl_b200.search import reorder_states

    g = torch.Generator("cuda").manual_seed(3)
    parents = torch.randint(0, 5, (4, 5), device="cuda", generator=g)
    store = [torch.randn(22, 3 + k, device="cuda", generator=g) for k in range(60)]
    before = [t.clone() for t in store]
    reorder_states([t[1:21] for t in store], parents.view(2, 2, 5))
    for t, b in zip(store, before):
        assert torch.equal(t[0], b[0]) and torch.equal(t[21], b[21])
        assert torch.equal(t[1:21], _reordered(b[1:21], parents, 0))
    reorder_states([], parents)
    reorder_states([torch.zeros(0, 4, device="cuda")], parents[:0])
    with pytest.raises(ValueError, match="overlap"):
        reorder_states([store[0][:20], store[1][1:21], store[0][1:21]], parents)
    with pytest.raises(ValueError, match="overlap"):
        reorder_states([parents.view(20)], parents)
    with pytest.raises(ValueError):
        reorder_states([store[0]], parents)                      # 22 rows
    with pytest.raises(ValueError):
        reorder_states([store[0][:20].t()], parents, dim=1)      # not contiguous
    with pytest.raises(ValueError):
        reorder_states([store[0][:20]], parents, dim=2)
    with pytest.raises(ValueError):
        reorder_states([torch.zeros(20, 2, device="cuda", requires_grad=True)], parents)
    with pytest.raises(ValueError):
        reorder_states([torch.zeros(1025, device="cuda")], torch.zeros(1, 1025, dtype=torch.int64, device="cuda"))


@pytest.mark.gpu
def test_a_backward_pass_does_not_use_reordered_states():
    """A state that a backward pass has saved (for a weight's gradient) is changed: the pass refuses, as after copy_."""
    import torch
    from carl_b200.search import reorder_states

    w = torch.ones(5, device="cuda", requires_grad=True)
    saved, other = torch.randn(6, 5, device="cuda"), torch.randn(6, 5, device="cuda")
    parents = torch.tensor([[1, 0, 2], [2, 2, 2]], device="cuda")
    loss, free = (saved * w).sum(), (other.clone() * w).sum()
    reorder_states([other, saved[:]], parents)           # a view of it counts too
    with pytest.raises(RuntimeError, match="inplace"):
        loss.backward()
    free.backward()
    with torch.inference_mode():
        reorder_states([torch.zeros(6, 2, device="cuda"), saved], parents)


@pytest.mark.gpu
def test_reorder_beyond_32_bits():
    import torch
    from carl_b200.search import reorder_states

    t = torch.zeros(4, 2 ** 31 + 16, dtype=torch.uint8, device="cuda")
    t[:, -1] = torch.arange(4, device="cuda")
    t[:, 7] = 10 + torch.arange(4, device="cuda")
    reorder_states([t], torch.tensor([[1, 0], [1, 1]], device="cuda"))
    assert t[:, -1].tolist() == [1, 0, 3, 3] and t[:, 7].tolist() == [11, 10, 13, 13]


@pytest.mark.gpu
@pytest.mark.parametrize("row, unit", [(2 ** 31 + 17, 1), (2 ** 32 + 2, 2)])
def test_reorder_rows_of_more_units_than_an_int(row, unit):
    """Rows of more than 2^31 bytes, or pairs of bytes, that no wider unit divides: every byte moves, none around."""
    import torch
    from carl_b200.search import reorder_states

    assert row % (2 * unit) and row // unit > 2 ** 31
    store = torch.zeros(2 * row + 128, dtype=torch.uint8, device="cuda")
    t = store[64:64 + 2 * row].view(2, row)
    at = torch.tensor([0, 1, 16383, 16384, 2 ** 30 + 5, 2 ** 31 - 1, 2 ** 31, row - 18, row - 2, row - 1], device="cuda")
    t[0] = 1
    t[1] = 2
    for k in range(2):
        t[k, at] = (10 * k + 20 + torch.arange(10, device="cuda")).to(torch.uint8)
    want = t[:, at].flip(0)
    reorder_states([t], torch.tensor([[1, 0]], device="cuda"))
    for k in range(2):
        assert torch.equal(t[k, at], want[k])
        t[k, at] = 2 - k
        assert bool((t[k] == 2 - k).all())
    assert not store[:64].any() and not store[-64:].any()


@pytest.mark.gpu
def test_reorder_more_slabs_than_a_launch_has_blocks():
    import torch
    from carl_b200.search import reorder_states

    slabs = 2 ** 31 + 3
    t = torch.empty(slabs, 2, dtype=torch.uint8, device="cuda")
    t[:, 0], t[:, 1] = 1, 2
    other = torch.arange(6, device="cuda").view(3, 2)
    reorder_states([t, other], torch.tensor([[1, 0]], device="cuda"), dim=1)
    assert bool((t[:, 0] == 2).all()) and bool((t[:, 1] == 1).all()) and other.tolist() == [[1, 0], [3, 2], [5, 4]]


@pytest.mark.gpu
def test_env_reorder(tmp_path, monkeypatch):
    """Every persistent field and output buffer of a sim becomes its parent's; copies go on alike."""
    import torch
    from box_arena import write_box
    from carl_b200 import carl, workloads

    monkeypatch.setenv("CARL_ARENA_OBJ", str(write_box(tmp_path / "box.obj")))
    n, K, nc = 24, 4, 6
    env = carl.Env(n, 3, 3, 3)
    workloads.mixed_state(env._env, 4)
    rng = np.random.default_rng(5)
    act = lambda: torch.from_numpy(workloads.discrete_actions(rng, n * nc).reshape(n, nc, 7)).cuda()  # noqa: E731
    for _ in range(3):
        env.step(act())
    victim = rng.integers(-1, n * nc, (n * nc, 1)).astype(np.int32)
    env._env.write_field("CAR_CONTACT_IDX", victim)
    parents = torch.from_numpy(rng.integers(-1, K + 1, (n // K, K))).cuda()
    p = parents.cpu().numpy().ravel()
    slot = np.arange(n) % K
    source = np.where((p >= 0) & (p < K), np.arange(n) - slot + p, np.arange(n))
    before = env._env.snapshot()
    torch.cuda.synchronize()
    buffers = [env._buffer(b).clone() for b in range(12)]
    env.reorder(parents)
    after = env._env.snapshot()
    torch.cuda.ExternalStream(env.stream).synchronize()
    for b in range(12):
        assert torch.equal(env._buffer(b), buffers[b][torch.from_numpy(source).cuda()]), b
    for name, words in before.items():
        per = words.shape[0] // n
        if name == "TICK_COUNT":
            assert np.array_equal(after[name], words)
            continue
        want = words.reshape(n, per, -1)[source].reshape(words.shape)
        if name == "CAR_CONTACT_IDX":
            v = want.view(np.int32)[:, 0]
            moved = np.repeat((np.arange(n) - source) * nc, nc)
            want = np.where(v >= 0, v + moved, v).astype(np.int32).view(np.uint32)[:, None]
        assert np.array_equal(after[name], want), name
    # Copies of one parent under the same actions stay bit-identical.
    a = act()
    env.step(a[torch.from_numpy(source).cuda()].contiguous())
    snap = env._env.snapshot()
    twins = [(i, j) for i in range(n) for j in range(i) if source[i] == source[j]]
    assert twins
    for i, j in twins:
        assert np.array_equal(snap["CAR_POS"].reshape(n, -1)[i], snap["CAR_POS"].reshape(n, -1)[j])
        assert np.array_equal(snap["BALL_POS"][i], snap["BALL_POS"][j])
    for bad in (parents.int(), parents.view(-1), parents.cpu(), parents.t(), parents[:2],
                torch.zeros(n // 5, 5, dtype=torch.int64, device="cuda")):
        with pytest.raises((TypeError, ValueError)):
            env.reorder(bad)
    env.close()


# ---- streams and graphs ------------------------------------------------------------------


@pytest.mark.gpu
def test_selection_and_reorder_in_a_graph_and_on_a_stream():
    import torch
    from carl_b200.action import CARLActionCodec
    from carl_b200.search import beam_select, reorder_states

    codec = CARLActionCodec()
    x, s, _, _ = _inputs(5, 8, 3001, "float32", False, False, 2)
    x18 = x[..., :18].contiguous().cuda()
    x, s = x.cuda(), s.cuda()
    hidden = torch.randn(40, 33, device="cuda")

    def step():
        best = beam_select(x, s)
        joint = codec.beam_select(x18, best.scores)
        reorder_states([hidden], joint.parents)
        return best, joint

    start = hidden.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = step()
    torch.cuda.current_stream().wait_stream(side)
    after = hidden.clone()
    hidden.copy_(start)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got = step()
    for k in range(3):
        hidden.copy_(start)
        if k == 1:
            s.sub_(1.0)          # a uniform shift: the same choice
        graph.replay()
        for a, b in zip(want, got):
            assert torch.equal(a.parents, b.parents) and torch.equal(a.actions, b.actions)
        assert torch.equal(hidden, after)
