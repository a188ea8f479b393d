"""Paged history: fork, append with copy on write, free, compact and read against
Python lists, bit for bit (the operators only move data and count)."""

from __future__ import annotations

import numpy as np
import pytest

from carl_b200 import _build, capi
from search_oracle import ListHistory


# ---- refusals (no GPU) -----------------------------------------------------------------


@pytest.fixture(scope="module")
def lib():
    _build.build()
    return capi.load()


def _view(**kw):
    v = dict(pages=64, table=64, lengths=64, refs=64, record_bytes=8, n_rows=4, row_pages=2, n_pages=8, page_len=4, device=0)
    v.update(kw)
    return capi.History(**v)


@pytest.mark.parametrize("bad, needle", [
    (dict(n_rows=-1), "non-negative"), (dict(n_pages=-1), "non-negative"), (dict(row_pages=0), "positive"),
    (dict(page_len=0), "positive"), (dict(record_bytes=0), "positive"), (dict(pages=None), "null"), (dict(refs=66), "refs"),
    (dict(table=None), "table"), (dict(lengths=65), "lengths"), (dict(row_pages=1 << 20, page_len=1 << 20), "long"),
])
def test_history_refuses_before_launch(lib, bad, needle):
    h = _view(**bad)
    calls = [lambda: lib.carlb_history_append(h, 64, 8, None, 64, 64, 1 << 40, None),
             lambda: lib.carlb_history_free(h, 64, None), lambda: lib.carlb_history_compact(h, 64, 64, 1 << 40, None),
             lambda: lib.carlb_history_read(h, None, 4, 3, 64, 64, None), lambda: lib.carlb_history_fork(h, _view(), 64, None, None),
             lambda: lib.carlb_history_fork(_view(), h, 64, None, None)]
    for call in calls:
        assert call() == capi.ERR_VALUE
        assert needle in lib.carlb_last_error(None).decode()


def test_history_refuses_arguments(lib):
    h = _view()
    assert lib.carlb_history_fork(h, _view(), 64, None, None) == capi.ERR_VALUE
    assert "overlap" in lib.carlb_last_error(None).decode()
    assert lib.carlb_history_fork(h, _view(table=128, lengths=128, refs=128, page_len=2), 64, None, None) == capi.ERR_VALUE
    assert lib.carlb_history_fork(h, _view(table=128, lengths=128, refs=128), None, None, None) == capi.ERR_VALUE
    assert lib.carlb_history_append(h, None, 8, None, 64, 64, 1 << 40, None) == capi.ERR_VALUE
    assert lib.carlb_history_append(h, 64, -8, None, 64, 64, 1 << 40, None) == capi.ERR_VALUE
    assert lib.carlb_history_append(h, 64, 8, None, 64, 64, 1, None) == capi.ERR_VALUE
    assert lib.carlb_history_append(h, 64, 8, None, None, 64, 1 << 40, None) == capi.ERR_VALUE
    assert lib.carlb_history_free(h, None, None) == capi.ERR_VALUE
    assert lib.carlb_history_compact(h, None, 64, 1 << 40, None) == capi.ERR_VALUE
    assert lib.carlb_history_compact(h, 64, 72, 1 << 40, None) == capi.ERR_VALUE
    assert lib.carlb_history_read(h, None, 3, 2, 64, 64, None) == capi.ERR_VALUE
    assert lib.carlb_history_read(h, 64, 3, 0, 64, 64, None) == capi.ERR_VALUE
    assert lib.carlb_history_read(h, 64, 3, 2, None, 64, None) == capi.ERR_VALUE
    assert lib.carlb_history_read(h, 64, 0, 2, None, None, None) == capi.OK
    assert lib.carlb_history_append(_view(n_rows=0), None, 8, None, None, None, 0, None) == capi.OK


def test_python_refuses_cpu_tensors():
    import torch
    from carl_b200.history import PagedHistory

    i32 = dict(dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        PagedHistory(torch.zeros(3, 2, 4), torch.zeros(2, 2, **i32), torch.zeros(2, **i32), torch.zeros(3, **i32))
    with pytest.raises(TypeError, match="int32"):
        PagedHistory(torch.zeros(3, 2, 4), torch.zeros(2, 2), torch.zeros(2, **i32), torch.zeros(3, **i32))
    with pytest.raises(ValueError):
        PagedHistory.empty(4, 0, 8, 4, device="cpu")


def test_python_refuses_a_counter_of_another_type():
    """The counter is written to by its address, as the books are."""
    import torch
    from carl_b200.history import PagedHistory

    i32 = dict(dtype=torch.int32)
    args = torch.zeros(3, 2, 4), torch.zeros(2, 2, **i32), torch.zeros(2, **i32), torch.zeros(3, **i32)
    for bad in (torch.zeros(1, dtype=torch.int64), torch.zeros(1), 0):
        with pytest.raises(TypeError, match="dropped"):
            PagedHistory(*args, bad)


@pytest.mark.gpu
def test_counters_that_cannot_be_written_are_refused():
    import torch
    from carl_b200.history import PagedHistory

    h = PagedHistory.empty(2, 2, 3, 4, (2,))
    args = h.pages, h.table, h.lengths, h.refs
    for bad in (torch.zeros(1, dtype=torch.int32), torch.zeros(0, dtype=torch.int32, device="cuda"),
                torch.zeros(2, dtype=torch.int32, device="cuda")):
        with pytest.raises(ValueError, match="dropped"):
            PagedHistory(*args, bad)
    counter = torch.full((1,), 3, dtype=torch.int32, device="cuda")
    assert PagedHistory(*args, counter).dropped is counter


# ---- against lists ------------------------------------------------------------------------


def _same(h, ref):
    import torch

    torch.cuda.synchronize()
    np.testing.assert_array_equal(h.table.cpu().numpy(), ref.table)
    np.testing.assert_array_equal(h.lengths.cpu().numpy(), ref.lengths)
    np.testing.assert_array_equal(h.refs.cpu().numpy(), ref.refs)
    np.testing.assert_array_equal(h.pages.cpu().numpy(), ref.pages)
    assert int(h.dropped) == ref.dropped


def _mirror(h):
    return ListHistory(*(t.cpu().numpy() for t in (h.pages, h.table, h.lengths, h.refs)))


GEOMETRIES = [  # rows, row_pages, pages, page_len, record shape, dtype
    (1, 1, 1, 1, (), "float32"), (3, 2, 5, 1, (3,), "int32"), (8, 3, 20, 4, (7,), "float16"), (12, 4, 30, 3, (2, 5), "uint8"),
    (40, 3, 100, 8, (64,), "float32"), (600, 3, 1500, 2, (4,), "int64"), (2500, 2, 3500, 3, (1,), "float16"),
    (16, 40, 200, 5, (252,), "float32"), (5, 2, 0, 4, (3,), "float32"), (1100, 3, 3300, 9, (300,), "float32"),
    (30, 2, 80, 7, (1500,), "float32"), (4, 600, 2300, 1, (2,), "float16"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("geometry", GEOMETRIES)
def test_history_against_lists(geometry):
    """Random sequences of all operators, until the pages and the rows run out."""
    import torch
    from carl_b200.history import PagedHistory

    n, M, pages, P, record, dtype = geometry
    dt = getattr(torch, dtype)
    rng = np.random.default_rng(n + pages)
    h = PagedHistory.empty(n, M, pages, P, record, dt)
    h.pages.copy_(torch.randint(0, 100, h.pages.shape, device="cuda"))
    ref = _mirror(h)
    for step in range(14):
        do = rng.choice(["append", "append", "append", "fork", "free", "compact"]) if step > 1 else "append"
        if do == "append":
            rec = torch.from_numpy(rng.integers(0, 100, (n, *record))).to(dt).cuda()
            mask = None if rng.random() < 0.5 else torch.from_numpy(rng.random(n) < 0.8).cuda()
            h.append(rec, mask)
            ref.append(rec.cpu().numpy(), None if mask is None else mask.cpu().numpy())
        elif do == "fork":
            parents = rng.integers(0, n, n) if rng.random() < 0.5 else np.arange(n) // 4 * 4 + rng.integers(0, 4, n)
            parents[rng.random(n) < 0.1] = rng.choice([-1, n, 2 ** 40])
            h = h.fork(torch.from_numpy(parents).cuda())
            ref = ref.fork(parents)
        elif do == "free":
            mask = rng.random(n) < 0.3
            h.free(torch.from_numpy(mask).cuda())
            ref.free(mask)
        else:
            assert int(h.compact()) == ref.compact()
        _same(h, ref)
        steps = int(rng.integers(1, M * P + 2))
        rows = rng.integers(-1, n + 1, 9)
        got, counts = h.read(steps, torch.from_numpy(rows).cuda())
        want, want_counts = ref.read(steps, rows)
        np.testing.assert_array_equal(counts.cpu().numpy(), want_counts)
        np.testing.assert_array_equal(got.cpu().numpy(), want)
    got, counts = h.read(M * P)
    want, want_counts = ref.read(M * P, range(n))
    np.testing.assert_array_equal(got.cpu().numpy(), want)
    np.testing.assert_array_equal(counts.cpu().numpy(), want_counts)


@pytest.mark.gpu
def test_append_many_rows_and_pages():
    """More rows and pages than one block counts, most pages in use, so that the free ones are far apart."""
    import torch
    from carl_b200.history import PagedHistory

    rng = np.random.default_rng(8)
    n, M, P, pages = 9000, 2, 2, 40000
    h = PagedHistory.empty(n, M, pages, P, (3,), torch.int32)
    busy = np.sort(rng.choice(pages, pages - 7000, replace=False))
    h.refs[torch.from_numpy(busy).cuda()] = 1          # named by someone else
    ref = _mirror(h)
    for _ in range(3):
        rec = rng.integers(0, 1000, (n, 3)).astype(np.int32)
        h.append(torch.from_numpy(rec).cuda())
        ref.append(rec)
        _same(h, ref)
        parents = np.arange(n) // 3 * 3 + rng.integers(0, 3, n)
        h, ref = h.fork(torch.from_numpy(parents).cuda()), ref.fork(parents)
        _same(h, ref)
    assert int(h.compact()) == ref.compact()
    _same(h, ref)


@pytest.mark.gpu
def test_bad_tables_are_bounded():
    """Entries that name no page, lengths beyond the table or below zero: no access out of range."""
    import torch
    from carl_b200.history import PagedHistory

    n, M, P, pages = 6, 3, 4, 10
    h = PagedHistory.empty(n, M, pages, P, (5,), torch.float32)
    for k in range(6):
        h.append(torch.full((n, 5), float(k), device="cuda"))
    h.table[1, 1], h.table[2, 0], h.table[3, 1] = 10 ** 9, -7, pages
    h.lengths[4], h.lengths[5] = 2 ** 31 - 1, -3
    ref = _mirror(h)
    ref.dropped = int(h.dropped)
    rec = np.full((n, 5), 9.0, np.float32)
    h.append(torch.from_numpy(rec).cuda())
    ref.append(rec)
    _same(h, ref)
    got, counts = h.read(20)
    want, want_counts = ref.read(20, range(n))
    np.testing.assert_array_equal(got.cpu().numpy(), want)
    np.testing.assert_array_equal(counts.cpu().numpy(), want_counts)
    parents = np.arange(n)[::-1].copy()
    h2, ref2 = h.fork(torch.from_numpy(parents).cuda()), ref.fork(parents)
    _same(h2, ref2)
    h2.compact()
    ref2.compact()
    _same(h2, ref2)
    h2.free(torch.ones(n, dtype=torch.bool, device="cuda"))
    ref2.free(np.ones(n, bool))
    _same(h2, ref2)


@pytest.mark.gpu
def test_a_full_pool_never_overwrites_a_sharer():
    """Rows that could not copy their shared page fall behind; the longest of the sharers is the one that writes on."""
    import torch
    from carl_b200.history import PagedHistory

    h = PagedHistory.empty(3, 2, 2, 4, (), torch.int32)
    ref = _mirror(h)
    h.append(torch.tensor([1, 1, 1], dtype=torch.int32, device="cuda"), torch.tensor([True, False, False], device="cuda"))
    ref.append(np.array([1, 1, 1]), [True, False, False])
    parents = np.zeros(3, np.int64)
    h, ref = h.fork(torch.from_numpy(parents).cuda()), ref.fork(parents)
    for k in range(2, 6):                               # one spare page for two copies
        rec = np.array([10 * k, 10 * k + 1, 10 * k + 2], np.int32)
        h.append(torch.from_numpy(rec).cuda())
        ref.append(rec)
        _same(h, ref)
    assert ref.dropped > 0


@pytest.mark.gpu
def test_records_by_stride_and_refusals():
    import torch
    from carl_b200.history import PagedHistory

    h = PagedHistory.empty(4, 2, 8, 2, (6,), torch.float32)
    ref = _mirror(h)
    wide = torch.randn(4, 9, device="cuda")
    for rec in (wide[:, 1:7], wide[:1, 2:8].expand(4, 6), torch.randn(6, 4, device="cuda").t(), wide[:, 3:9].requires_grad_()):
        h.append(rec)
        ref.append(rec.detach().cpu().numpy())
        _same(h, ref)
    rec = h.pages[2:6, 0]                               # records of the history's own pages
    ref.append(rec.cpu().numpy())
    h.append(rec)
    _same(h, ref)
    rec = wide.detach()[:, :6]
    for exc, call in [(TypeError, lambda: h.append(rec.half())), (ValueError, lambda: h.append(rec[:3])),
                      (ValueError, lambda: h.append(rec.cpu())), (TypeError, lambda: h.append(rec, rec[:, 0])),
                      (ValueError, lambda: h.append(rec, rec[:2, 0] > 0)), (TypeError, lambda: h.free(None)),
                      (TypeError, lambda: h.fork(rec[:, 0])), (ValueError, lambda: h.read(0)),
                      (TypeError, lambda: h.read(2, rec[:, 0])),
                      (ValueError, lambda: h.fork(torch.arange(4, device="cuda"), out=h)),
                      (ValueError, lambda: h.fork(torch.arange(4, device="cuda"),
                                                  out=PagedHistory.empty(4, 2, 8, 2, (6,), torch.float32)))]:
        with pytest.raises(exc):
            call()
    _same(h, ref)


@pytest.mark.gpu
def test_pages_beyond_32_bits():
    import torch
    from carl_b200.history import PagedHistory

    size = 2 ** 29
    h = PagedHistory.empty(2, 3, 6, 2, (size,), torch.uint8)         # 6 GB of pages
    rec = torch.zeros(2, size, dtype=torch.uint8, device="cuda")
    for k in range(5):
        rec[:, -1] = torch.tensor([10 + k, 20 + k], device="cuda")
        h.append(rec)
    out, counts = h.read(3)
    assert counts.tolist() == [3, 3] and out[:, :, -1].tolist() == [[12, 13, 14], [22, 23, 24]]
    h = h.fork(torch.tensor([-1, 1], device="cuda"))
    assert int(h.compact()) == 3
    out, _ = h.read(5, torch.tensor([1], device="cuda"))
    assert out[0, :, -1].tolist() == [20, 21, 22, 23, 24]


@pytest.mark.gpu
def test_pages_of_nearly_two_to_the_31_records():
    import torch
    from carl_b200.history import PagedHistory

    P = 2 ** 31 - 1
    h = PagedHistory.empty(1, 1, 1, P, (), torch.uint8)              # 2 GB
    h.append(torch.tensor([5], dtype=torch.uint8, device="cuda"))
    for last, value in ((P - 4097, 6), (P - 1, 7)):
        h.lengths[0] = last
        h.append(torch.tensor([value], dtype=torch.uint8, device="cuda"))
        assert h.lengths.tolist() == [last + 1]
        out, counts = h.read(2)
        assert counts.tolist() == [2] and out.tolist() == [[0, value]]
    assert h.pages[0, 0] == 5 and h.pages[0, P - 4097] == 6 and h.pages[0, -1] == 7
    h.append(torch.tensor([8], dtype=torch.uint8, device="cuda"))
    assert h.lengths.tolist() == [P] and int(h.dropped) == 1 and h.pages[0, -1] == 7


@pytest.mark.gpu
def test_sizes_beyond_32_bits_are_refused():
    """Counts that the entry points take as int32: the host refuses what would wrap, before it allocates."""
    import torch
    from carl_b200.history import PagedHistory
    from carl_b200.search import reorder_states

    h = PagedHistory.empty(2, 2, 3, 4, (), torch.uint8)
    many = torch.zeros(1, dtype=torch.int64, device="cuda").expand(2 ** 32 + 2)
    for call in (lambda: h.read(2 ** 32 + 5, many[:1]), lambda: h.read(2 ** 31, many[:1]), lambda: h.read(1, many),
                 lambda: h.fork(many), lambda: h.fork(many, out=h),
                 lambda: reorder_states([torch.zeros(4, device="cuda")], many[:, None])):
        with pytest.raises(ValueError, match="too many"):
            call()


@pytest.mark.gpu
def test_history_in_graphs():
    """Two captured graphs that fork back and forth between two histories, replayed against lists."""
    import torch
    from carl_b200.history import PagedHistory

    n, M, P, pages = 12, 6, 3, 60
    a = PagedHistory.empty(n, M, pages, P, (4,), torch.float32)
    b = PagedHistory(a.pages, torch.full_like(a.table, -1), torch.zeros_like(a.lengths), torch.zeros_like(a.refs), a.dropped)
    ref = _mirror(a)
    parents = torch.arange(n, device="cuda")
    rec = torch.zeros(n, 4, device="cuda")
    graphs = []
    for src, dst in ((a, b), (b, a)):
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            src.fork(parents, out=dst)
            dst.append(rec)
        graphs.append((g, dst))
    rng = np.random.default_rng(2)
    for step in range(10):
        q = np.arange(n) // 4 * 4 + rng.integers(0, 4, n)
        r = rng.normal(size=(n, 4)).astype(np.float32)
        parents.copy_(torch.from_numpy(q))
        rec.copy_(torch.from_numpy(r))
        g, dst = graphs[step % 2]
        g.replay()
        ref = ref.fork(q)
        ref.append(r)
        _same(dst, ref)


@pytest.mark.gpu
@pytest.mark.parametrize("counted", [False, True])
def test_forks_go_on_with_the_dropped_records(counted):
    """Into a new history and into one with a counter of its own, back and forth."""
    import torch
    from carl_b200.history import PagedHistory

    def books():
        i32 = dict(dtype=torch.int32, device="cuda")
        return torch.full((3, 1), -1, **i32), torch.zeros(3, **i32), torch.zeros(8, **i32)

    pages = torch.zeros(8, 2, device="cuda")
    counter = lambda k: torch.full((1,), k, dtype=torch.int32, device="cuda") if counted else None  # noqa: E731
    a, b = PagedHistory(pages, *books(), counter(2)), PagedHistory(pages, *books(), counter(100))
    parents, rec = torch.arange(3, device="cuda"), torch.ones(3, device="cuda")
    want = 2 if counted else 0
    for step in range(4):                               # two records fit; three rows are dropped from then on
        a.append(rec)
        want += 3 * (step >= 2)
        assert int(a.dropped) == want
        a = a.fork(parents)
        assert int(a.dropped) == want
        a.fork(parents, out=b)
        assert int(b.dropped) == want
        a, b = b, PagedHistory(pages, *books(), counter(100))
    fresh = PagedHistory(pages, *books())               # without a counter, not looked at before
    fresh.fork(parents, out=a)
    assert int(a.dropped) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("change", ["append", "compact", "free", "fork", "count"])
def test_a_backward_pass_does_not_use_a_changed_history(change):
    import torch
    from carl_b200.history import PagedHistory

    for forked in (False, True):                         # books of their own, or in one tensor
        h = PagedHistory.empty(3, 2, 9, 2, (4,))
        spare = PagedHistory(h.pages, torch.full_like(h.table, -1), torch.zeros_like(h.lengths), torch.zeros_like(h.refs))
        if forked:
            h = h.fork(torch.arange(3, device="cuda"))
        h.append(torch.ones(3, 4, device="cuda"))
        w = torch.ones(4, device="cuda", requires_grad=True)
        table = torch.ones(10, device="cuda", requires_grad=True)
        which = {"append": h.pages, "compact": h.pages, "free": h.lengths, "fork": spare.lengths, "count": h.dropped}[change]
        if which is h.pages:
            loss = (h.pages[0] * w).sum()
        else:
            loss = table.index_select(0, which).sum()    # saves the indices
        calls = {"append": lambda: h.append(torch.ones(3, 4, device="cuda")), "compact": h.compact,
                 "free": lambda: h.free(torch.ones(3, dtype=torch.bool, device="cuda")),
                 "fork": lambda: h.fork(torch.arange(3, device="cuda"), out=spare),
                 "count": lambda: h.append(torch.ones(3, 4, device="cuda"))}
        calls[change]()
        with pytest.raises(RuntimeError, match="inplace"):
            loss.backward()
        records, _ = h.read(2)                           # a copy
        loss = (records * w).sum()
        h.append(torch.ones(3, 4, device="cuda"))
        loss.backward()


@pytest.mark.gpu
def test_records_in_the_historys_own_memory():
    """Rows that begin in front of the pages and run into them, the lengths, the table: taken as they were before."""
    import torch
    from carl_b200.history import PagedHistory

    n, P = 600, 2
    i32 = dict(dtype=torch.int32, device="cuda")
    store = torch.arange(1500 * P * 3, **i32).view(1500, P, 3)
    pages = store[500:]
    h = PagedHistory(pages, torch.full((n, 3), -1, **i32), torch.zeros(n, **i32), torch.zeros(1000, **i32))
    ref = _mirror(h)
    for records in (store[400:1000, 1], store[:600, 0], h.table, store[400:1000, 1]):
        want = records.cpu().numpy()
        h.append(records)
        ref.append(want)
        _same(h, ref)
    one = PagedHistory(torch.zeros(900, 4, **i32), torch.full((n, 2), -1, **i32), torch.zeros(n, **i32), torch.zeros(900, **i32))
    ref = _mirror(one)
    for records in (one.lengths, one.lengths, one.refs[100:100 + n], one.dropped.expand(n), one.lengths,
                    one.dropped.expand(n)):                  # a third of the rows drop theirs by then
        want = records.cpu().numpy()
        one.append(records)
        ref.append(want)
        _same(one, ref)
    one = one.fork(torch.arange(n, device="cuda"))           # books in one tensor
    ref = ref.fork(np.arange(n))
    for _ in range(3):
        want = one.lengths.cpu().numpy()
        one.append(one.lengths)
        ref.append(want)
        _same(one, ref)


@pytest.mark.gpu
def test_a_search_with_an_env(tmp_path, monkeypatch):
    """The operators together, as a search uses them: mask, select, reorder, fork, append, step, harvest."""
    import torch
    from box_arena import write_box
    from carl_b200 import carl
    from carl_b200.action import CARLActionCodec
    from carl_b200.history import PagedHistory
    from carl_b200.search import reorder_states
    from search_oracle import HEADS, best_continuations, joint_actions

    monkeypatch.setenv("CARL_ARENA_OBJ", str(write_box(tmp_path / "box.obj")))
    G, K = 6, 4
    n = G * K
    env = carl.Env(n, 1, 1, 7)
    codec = CARLActionCodec()
    weight = torch.randn(env.obs_dim, 18, device="cuda", generator=torch.Generator("cuda").manual_seed(1)) * 0.01
    scores = torch.full((G, K), -torch.inf, device="cuda")
    scores[:, 0] = 0.0                                        # one live beam per problem at the root
    hidden = torch.arange(n, device="cuda", dtype=torch.float32)[:, None].repeat(1, 3)
    first = torch.arange(0, n, K, device="cuda")[:, None]
    history = PagedHistory.empty(n, 4, 4 * n, 2, (7,), torch.int32)
    env_stream = torch.cuda.ExternalStream(env.stream)
    paths = [[[] for _ in range(K)] for _ in range(G)]
    for _ in range(5):
        torch.cuda.current_stream().wait_stream(env_stream)
        obs = env.get_obs()[:, 0].contiguous()                # the first car plans
        logits = (obs @ weight).view(G, K, 18)
        mask = codec.mask(obs).view(G, K, 18)
        best = codec.beam_select(logits, scores, mask)
        es, ep, ea = best_continuations(logits.cpu().numpy(), scores.cpu().numpy(), mask.cpu().numpy(), None, K, HEADS)
        assert np.array_equal(best.parents.cpu().numpy(), ep)
        act = joint_actions(ea)
        assert np.array_equal(best.actions.cpu().numpy(), act)
        paths = [[paths[g][ep[g, j]] + [act[g, j].tolist()] for j in range(K)] for g in range(G)]
        scores = best.scores
        env.reorder(best.parents)
        reorder_states([hidden], best.parents)
        history = history.fork(best.parents + first)
        history.append(best.actions.view(n, 7))
        actions = torch.zeros(n, 2, 7, dtype=torch.int32, device="cuda")
        actions[:, 0] = best.actions.view(n, 7)
        env.step(actions)
    assert torch.equal(hidden[:, 0].view(G, K), first.expand(G, K).float())   # every lineage starts at the root's beam
    records, counts = history.read(5)
    assert counts.tolist() == [5] * n and int(history.dropped) == 0
    assert records.view(G, K, 5, 7).tolist() == paths
    keep = torch.full((n,), -1, device="cuda")
    keep[::K] = torch.arange(0, n, K, device="cuda")
    history = history.fork(keep)
    live = int(history.compact())
    assert live == 3 * G
    records, _ = history.read(5, torch.arange(0, n, K, device="cuda"))
    assert records.tolist() == [p[0] for p in paths]
    env.close()


@pytest.mark.gpu
def test_the_documented_search_loop(tmp_path, monkeypatch):
    """The loop of the integration guide as it stands there, with an env that is slow to step (a delay on its stream
    before every step) and one that is waited for after every call: the same observations, choices and records.
    Episodes end on the way, and a lineage that is over keeps its score and its records."""
    import re
    import torch
    from pathlib import Path

    from box_arena import write_box
    from carl_b200 import carl
    from carl_b200.action import CARLActionCodec

    guide = (Path(__file__).resolve().parents[1] / "INTEGRATION.md").read_text()
    loop, = [c for c in re.findall(r"```python\n(.*?)```", guide, re.S) if "codec.beam_select" in c]
    monkeypatch.setenv("CARL_ARENA_OBJ", str(write_box(tmp_path / "box.obj")))
    G, K, depth = 5, 4, 6
    n = G * K
    codec = CARLActionCodec()
    gen = torch.Generator("cuda").manual_seed(1)
    idx = torch.arange(0, n, K, device="cuda")

    def run(slow):
        env = carl.Env(n, 1, 1, 7)
        env.max_ticks = 1000
        stream = torch.cuda.ExternalStream(env.stream)
        seen, steps = [], []
        weight = torch.randn(env.obs_dim, 18, device="cuda", generator=gen.manual_seed(1)) * 0.01
        zeros = torch.zeros(G, dtype=torch.int32, device="cuda")
        delay = torch.zeros(1 << 26, device="cuda")

        def step(actions):
            # One beam of every group ends with this step.
            env_set(zeros + 1, zeros, zeros + 999, idx + len(steps) % K)   # (a tie would go on)
            if slow:
                with torch.cuda.stream(stream):
                    for _ in range(40):              # a few milliseconds, in which an early read sees the old outputs
                        delay.add_(1.0)
            env_step(actions)
            if not slow:
                torch.cuda.synchronize()
            steps.append(None)

        env_step, env_set, env.step = env.step, env.set_match_state, step

        def policy(obs):
            seen.append(obs.clone())
            return obs @ weight

        scope = dict(torch=torch, env=env, codec=codec, policy=policy, groups=G, beams=K, depth=depth, row_pages=4,
                     n_pages=3 * n, page_len=2, hidden=torch.arange(n, device="cuda"))
        exec(loop, scope)
        torch.cuda.synchronize()
        records, counts = scope["history"].read(8)
        env.close()
        return dict(obs=torch.stack(seen), scores=scope["scores"], over=scope["over"], hidden=scope["hidden"],
                    records=records, counts=counts)

    want, got = run(False), run(True)
    for name in want:
        assert torch.equal(want[name], got[name]), name
    assert (want["obs"][1:] != want["obs"][:-1]).flatten(1).any(1).all()         # every step is seen
    assert torch.equal(want["hidden"].view(G, K), idx[:, None].expand(G, K))     # all from the root's first beam
    counts, over = want["counts"].view(G, K), want["over"]
    assert over.any() and (counts[~over] == depth).all() and (counts[over] < depth).any()
    assert torch.isfinite(want["scores"]).all()
