"""Cases and plain forms of the search and history operators.

A search plans with the simulator: every group of beams is one planning problem,
every beam an arena (a sim) with the actions that led to it.  One step scores all
continuations of all beams, keeps the best, moves the kept beams' states to their
slots and records what they saw; at the end the best lineage of every group is
laid out for training.  The operators are

* select   beam selection over beams and a flat vocabulary of actions;
* joint    the same over the seven action heads (3, 3, 3, 2, 2, 3, 2) of a car;
* reorder  the kept beams' states moved to their slots, in place;
* step     a paged history forked to the kept beams, with one record appended each;
* harvest  the best lineages kept, the pages compacted, their last records read.

``run`` computes a case in plain torch operations where ``own`` is false, and by
the framework's calls where it is true.
"""

import math

import numpy as np
import torch

own = False

HEADS = (3, 3, 3, 2, 2, 3, 2)        # the action heads of a car
LOGITS = sum(HEADS)
OFFSETS = tuple(sum(HEADS[:h]) for h in range(len(HEADS)))
JOINT = math.prod(HEADS)             # 648 joint actions
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
CAR_WORDS, CAR_OUT_WORDS, SIM_WORDS = 76, 33, 66   # 32-bit words of state per car and per sim
DEVICE = "cuda"


# ---- cases ----------------------------------------------------------------------------------------------------------


def listed():
    return [
        # One planning problem over the joint actions of a car: what a single decision costs.
        {"name": "select_one_648", "op": "select", "groups": 1, "beams": 8, "vocab": 648, "width": 8, "dtype": "f32",
         "masked": True, "finished": False},
        # A batch of 32768 arenas as 4096 problems of 8 beams, some episodes over, illegal actions masked.
        {"name": "select_batch_648", "op": "select", "groups": 4096, "beams": 8, "vocab": 648, "width": 8,
         "dtype": "f32", "masked": True, "finished": True},
        # One search over a large odd vocabulary (macro actions, tokens of a generative policy): few long rows.
        {"name": "select_one_50257_bf16", "op": "select", "groups": 1, "beams": 8, "vocab": 50257, "width": 8,
         "dtype": "bf16", "masked": False, "finished": False},
        # The largest: many beams over a large vocabulary.
        {"name": "select_batch_131072_bf16", "op": "select", "groups": 32, "beams": 16, "vocab": 131072, "width": 16,
         "dtype": "bf16", "masked": False, "finished": False},
        # One car's decision from its 18 action logits.
        {"name": "joint_one", "op": "joint", "groups": 1, "beams": 8, "width": 8, "dtype": "f32", "masked": True,
         "finished": False},
        # Every car of 32768 arenas of 3v3 plans on its own: 196608 rows of 18 logits.
        {"name": "joint_batch", "op": "joint", "groups": 24576, "beams": 8, "width": 8, "dtype": "f32",
         "masked": True, "finished": True},
        # What a policy keeps beside one planning problem: observations, hidden state, done flags, actions.
        {"name": "reorder_one_rows", "op": "reorder", "layout": "rows", "groups": 1, "beams": 8, "cars": 6,
         "hidden": 512},
        # The tick state of 32768 arenas of 3v3, word-major as the simulator holds it.
        {"name": "reorder_batch_words", "op": "reorder", "layout": "words", "groups": 4096, "beams": 8, "cars": 6,
         "hidden": 0},
        # One planning problem records the observation of a 3v3 agent.
        {"name": "step_one", "op": "step", "rows": 8, "beams": 8, "page_len": 16, "row_pages": 8, "record": 252,
         "dtype": "f32"},
        # 16384 lineages record theirs; the pages hold 1.1 GB.
        {"name": "step_batch", "op": "step", "rows": 16384, "beams": 8, "page_len": 16, "row_pages": 4,
         "record": 252, "dtype": "f32"},
        # The end of a few searches.
        {"name": "harvest_few", "op": "harvest", "rows": 64, "beams": 8, "page_len": 16, "row_pages": 4,
         "record": 252, "dtype": "f32", "steps": 32},
        # The end of 1024 searches of 8 beams: the survivors' pages move together and are read as a training batch.
        {"name": "harvest_batch", "op": "harvest", "rows": 8192, "beams": 8, "page_len": 16, "row_pages": 8,
         "record": 252, "dtype": "f32", "steps": 64},
    ]


def _spread(rng, lo, hi):
    """A whole number from lo to hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["select", "select", "joint", "reorder", "step", "harvest"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op == "select":
        beams, vocab = _spread(rng, 1, 64), _spread(rng, 18, 150000)
        most = max(1, min(8192, 40_000_000 // (beams * vocab)))
        return {"op": op, "groups": _spread(rng, 1, most), "beams": beams, "vocab": vocab,
                "width": min(beams * vocab, _spread(rng, 1, 64)), "dtype": dtype, "masked": rng.random() < 0.5,
                "finished": rng.random() < 0.5}
    if op == "joint":
        beams = _spread(rng, 1, 32)
        return {"op": op, "groups": _spread(rng, 1, 196608 // beams), "beams": beams, "width": _spread(rng, 1, 32),
                "dtype": dtype, "masked": rng.random() < 0.5, "finished": rng.random() < 0.5}
    if op == "reorder":
        beams, layout = _spread(rng, 2, 64), rng.choice(["rows", "words"])
        return {"op": op, "layout": layout, "groups": _spread(rng, 1, 32768 // beams), "beams": beams,
                "cars": rng.randint(1, 8), "hidden": _spread(rng, 1, 512) if layout == "rows" else 0}
    beams = _spread(rng, 1, 16)
    record, page_len, row_pages = _spread(rng, 1, 600), rng.choice([1, 3, 8, 16, 32]), _spread(rng, 2, 16)
    most = max(1, min(2048, 200_000_000 // (beams * record * page_len * row_pages * BYTES[dtype])))
    case = {"op": op, "rows": beams * _spread(rng, 1, most), "beams": beams, "page_len": page_len,
            "row_pages": row_pages, "record": record, "dtype": dtype}
    if op == "harvest":
        case["steps"] = _spread(rng, 1, page_len * row_pages)
    return case


# ---- inputs ---------------------------------------------------------------------------------------------------------


def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    op = case["op"]
    if op in ("select", "joint"):
        return _prepare_scores(case, g)
    if op == "reorder":
        return _prepare_states(case, g)
    return _prepare_history(case, g)


def _prepare_scores(case, g):
    G, K, V = case["groups"], case["beams"], case["vocab"] if case["op"] == "select" else LOGITS
    logits = torch.randn(G, K, V, generator=g, device=DEVICE).mul_(2.5).to(DTYPES[case["dtype"]])
    # Beams have drifted apart by a few nats of the sequences' log-probabilities.
    scores = -(20.0 + 4.0 * torch.rand(G, K, generator=g, device=DEVICE))
    mask = finished = None
    if case["masked"]:
        mask = torch.rand(G, K, V, generator=g, device=DEVICE) < 0.8
        # A beam in a hundred has no legal action left.
        mask &= (torch.rand(G, K, 1, generator=g, device=DEVICE) >= 0.01)
    if case["finished"]:
        finished = torch.rand(G, K, generator=g, device=DEVICE) < 0.1
        scores = torch.where(torch.rand(G, K, generator=g, device=DEVICE) < 0.05, -math.inf, scores)
    return {"case": case, "logits": logits, "scores": scores, "mask": mask, "finished": finished}


def _prepare_states(case, g):
    G, K, n = case["groups"], case["beams"], case["cars"]
    parents = torch.randint(0, K, (G, K), generator=g, device=DEVICE)
    rand = lambda *shape: torch.randn(*shape, generator=g, device=DEVICE)  # noqa: E731
    if case["layout"] == "words":
        states = [rand(CAR_WORDS, G * K, n), rand(CAR_OUT_WORDS, G * K, n), rand(SIM_WORDS, G * K)]
        dim = 1
    else:
        obs = 9 + 21 * n + 68 + 6 + 6 * (n - 1) + 6 + 2 + 5   # an agent's observation
        states = [rand(G * K, n, obs), rand(G * K, case["hidden"]).bfloat16(),
                  rand(G * K) > 0, torch.randint(0, 3, (G * K, n, len(HEADS)), generator=g, device=DEVICE,
                                                 dtype=torch.int32)]
        dim = 0
    return {"case": case, "states": states, "parents": parents, "dim": dim}


def _prepare_history(case, g):
    """A paged history in mid-search: the beams of a group share the full pages of
    their common past and own the rest; pages lie in no order, those beyond the histories' length are free."""
    n, K, P, M = case["rows"], case["beams"], case["page_len"], case["row_pages"]
    G = n // K
    last = M * P - (1 if case["op"] == "step" else 0)      # a step needs room for its record
    length = torch.randint(1, last + 1, (G,), generator=g, device=DEVICE)
    used = (length + P - 1) // P
    shared = (torch.rand(G, generator=g, device=DEVICE) * (length // P + 1)).long()
    col = torch.arange(M, device=DEVICE)
    first = torch.arange(n, device=DEVICE) % K == 0
    rows_used, rows_shared = used.repeat_interleave(K)[:, None], shared.repeat_interleave(K)[:, None]
    has = col < rows_used
    owns = has & (first[:, None] | (col >= rows_shared))
    n_pages = n * M
    ids = torch.randperm(n_pages, generator=g, device=DEVICE)
    rank = (owns.flatten().cumsum(0) - 1).clamp_(min=0).view(n, M)
    owned = ids[rank]
    leader = owned.view(G, K, M)[:, :1].expand(G, K, M).reshape(n, M)
    table = torch.where(has, torch.where(col < rows_shared, leader, owned), -1).int()
    refs = torch.zeros(n_pages + 1, dtype=torch.int32, device=DEVICE)
    refs.scatter_add_(0, torch.where(has, table, n_pages).long().flatten(),
                      torch.ones(n * M, dtype=torch.int32, device=DEVICE))
    lengths = length.repeat_interleave(K).int()
    pages = torch.randn(n_pages, P, case["record"], generator=g, device=DEVICE).to(DTYPES[case["dtype"]])
    state = {"case": case, "pages": pages, "table": table, "lengths": lengths, "refs": refs[:n_pages].clone()}
    group = torch.arange(n, device=DEVICE) // K * K
    if case["op"] == "step":
        state["parents"] = group + torch.randint(0, K, (n,), generator=g, device=DEVICE)
        state["records"] = torch.randn(n, case["record"], generator=g, device=DEVICE).to(DTYPES[case["dtype"]])
    else:
        best = torch.randint(0, K, (G,), generator=g, device=DEVICE).repeat_interleave(K)
        state["parents"] = torch.where(first, group + best, -1)
        state["rows"] = torch.arange(0, n, K, device=DEVICE)
    return state


# ---- one pass -------------------------------------------------------------------------------------------------------


def run(state):
    op = state["case"]["op"]
    if op == "select":
        return _select(state)
    if op == "joint":
        return _joint(state)
    if op == "reorder":
        return _reorder(state)
    return _step(state) if op == "step" else _harvest(state)


def _select(s):
    width = s["case"]["width"]
    if own:
        from carl_b200.search import beam_select

        best = beam_select(s["logits"], s["scores"], s["mask"], width=width, finished=s["finished"])
        return {"scores": best.scores, "parents": best.parents, "actions": best.actions}
    # 64 bits: an order between near totals is a whole-number output.
    x = s["logits"].double()
    if s["mask"] is not None:
        x = torch.where(s["mask"], x, -math.inf)
    return _plain_best(_log_normaliser(x), x, s["scores"], s["finished"], width)


def _joint(s):
    width = s["case"]["width"]
    if own:
        from carl_b200.action import CARLActionCodec

        best = CARLActionCodec().beam_select(s["logits"], s["scores"], s["mask"], width=width, finished=s["finished"])
        return {"scores": best.scores, "parents": best.parents, "actions": best.actions}
    x = s["logits"].double()
    if s["mask"] is not None:
        x = torch.where(s["mask"], x, -math.inf)
    heads = x.split(HEADS, -1)
    norm = sum(_log_normaliser(h) for h in heads)
    a, b, c, d, e, f, q = (h.reshape(h.shape[:-1] + (1,) * i + (-1,) + (1,) * (6 - i)) for i, h in enumerate(heads))
    total = (a + b + c + d + e + f + q).flatten(-7)
    best = _plain_best(norm, total, s["scores"], s["finished"], width)
    radix = torch.tensor([math.prod(HEADS[h + 1:]) for h in range(len(HEADS))], device=x.device)
    size = torch.tensor(HEADS, device=x.device)
    best["actions"] = (best["actions"].long()[..., None] // radix % size).int()
    return best


def _log_normaliser(x):
    """log(sum(exp(x))) over the last dimension; -inf for a row without a finite value."""
    top = x.amax(-1, keepdim=True)
    top = torch.where(top > -math.inf, top, 0.0)
    return (x - top).exp().sum(-1).log() + top[..., 0]


def _plain_best(norm, x, scores, finished, width):
    """The `width` best of scores - norm + x over beams and actions."""
    G, K, V = x.shape
    total = (scores.double() - norm)[..., None] + x
    total = torch.where(total > -math.inf, total, -math.inf)          # a row without a legal action gives NaN
    if finished is not None:
        stay = torch.full_like(total, -math.inf)
        stay[..., 0] = scores.double()
        total = torch.where(finished[..., None], stay, total)
    flat = total.reshape(G, K * V)
    if width > K * V:
        flat = torch.cat([flat, flat.new_full((G, width - K * V), -math.inf)], -1)
    value, index = flat.sort(dim=-1, descending=True, stable=True)
    value, index = value[:, :width], index[:, :width]
    live = value > -math.inf
    slot = torch.arange(width, device=x.device) % K
    return {"scores": value.float(), "parents": torch.where(live, index // V, slot),
            "actions": torch.where(live, index % V, 0).int()}


def _reorder(s):
    if own:
        from carl_b200.search import reorder_states

        reorder_states(s["states"], s["parents"], dim=s["dim"])
        return s["states"]
    K = s["case"]["beams"]
    source = (s["parents"] + torch.arange(0, s["parents"].numel(), K, device=DEVICE)[:, None]).flatten()
    return [t.copy_(t.index_select(s["dim"], source)) for t in s["states"]]


def _step(s):
    if own:
        from carl_b200.history import PagedHistory

        h = PagedHistory(s["pages"], s["table"], s["lengths"], s["refs"]).fork(s["parents"])
        h.append(s["records"])
        return {"pages": h.pages, "table": h.table, "lengths": h.lengths, "refs": h.refs}
    table, lengths, refs = _plain_fork(s)
    pages = s["pages"]
    n_pages, P = pages.shape[:2]
    n, M = table.shape
    row = torch.arange(n, device=DEVICE)
    slot, col = lengths.long() % P, lengths.long() // P
    room = col < M
    held = table.gather(1, col.clamp(max=M - 1)[:, None])[:, 0].long()      # the row's last page, where slot > 0
    shared = (slot > 0) & (refs[held.clamp(min=0)] > 1)
    # Of the rows that share a page and all append, the longest (the first of those) writes on in it; the others copy it.
    at = torch.where(shared & room, held, n_pages)
    sharers = torch.zeros(n_pages + 1, dtype=torch.int32, device=DEVICE).scatter_add_(0, at, torch.ones_like(lengths))
    order = slot * n + (n - 1 - row)
    leader = torch.full((n_pages + 1,), -1, device=DEVICE).scatter_reduce_(0, at, order, "amax")
    stays = shared & (sharers[at] == refs[held.clamp(min=0)]) & (leader[at] == order)
    needs = room & ((slot == 0) | (shared & ~stays))
    rank = needs.cumsum(0) - 1
    free = (refs > 0).int().argsort(stable=True)                             # free pages first, lowest first
    got = needs & (rank < (refs == 0).sum())
    fresh = free[rank.clamp(0, n_pages - 1)]
    done = room & (~needs | got)
    copies = (got & shared).nonzero()[:, 0]
    which, where = (torch.arange(P, device=DEVICE) < slot[copies][:, None]).nonzero(as_tuple=True)
    pages[fresh[copies][which], where] = pages[held[copies][which], where]
    refs.scatter_add_(0, held[copies], torch.full_like(copies, -1, dtype=torch.int32))
    refs[fresh[got]] = 1
    home = torch.where(got, fresh, held)
    writes = done.nonzero()[:, 0]
    table[writes, col[writes]] = home[writes].int()
    pages[home[writes], slot[writes]] = s["records"][writes]
    lengths[writes] += 1
    return {"pages": pages, "table": table, "lengths": lengths, "refs": refs}


def _plain_fork(s):
    """Table, lengths and reference counts of the rows' new lineages."""
    parents, n_pages = s["parents"], s["pages"].shape[0]
    keep = parents >= 0
    lengths = torch.where(keep, s["lengths"][parents.clamp(min=0)], 0)
    table = torch.where(keep[:, None], s["table"][parents.clamp(min=0)], -1)
    refs = torch.zeros(n_pages + 1, dtype=torch.int32, device=DEVICE)
    refs.scatter_add_(0, torch.where(table >= 0, table, n_pages).long().flatten(),
                      torch.ones(table.numel(), dtype=torch.int32, device=DEVICE))
    return table, lengths, refs[:n_pages]


def _harvest(s):
    steps = s["case"]["steps"]
    if own:
        from carl_b200.history import PagedHistory

        h = PagedHistory(s["pages"], s["table"], s["lengths"], s["refs"]).fork(s["parents"])
        h.compact()
        records, counts = h.read(steps, s["rows"])
        return {"records": records, "counts": counts, "pages": h.pages, "table": h.table, "refs": h.refs}
    table, lengths, refs = _plain_fork(s)
    pages = s["pages"]
    P = pages.shape[1]
    live = refs > 0
    page = torch.arange(refs.numel(), device=DEVICE)
    kept = live.sum()
    holes = (~live & (page < kept)).nonzero()[:, 0]
    moved = (live & (page >= kept)).nonzero()[:, 0].flip(0)                  # the highest goes to the lowest hole
    pages[holes] = pages[moved]
    refs[holes] = refs[moved]
    refs[moved] = 0
    page[moved] = holes
    table = torch.where(table >= 0, page[table.clamp(min=0).long()].int(), -1)
    length = lengths[s["rows"]].long()
    counts = length.clamp(max=steps)
    t = torch.arange(steps, device=DEVICE)
    at = (length - counts)[:, None] + t
    inside = t < counts[:, None]
    at = torch.where(inside, at, 0)
    source = table[s["rows"]].gather(1, at // P).clamp(min=0).long()
    records = torch.where(inside[..., None], pages[source, at % P], torch.zeros((), dtype=pages.dtype, device=DEVICE))
    return {"records": records, "counts": counts.int(), "pages": pages, "table": table, "refs": refs}


# ---- what a pass cannot do without ----------------------------------------------------------------------------------


def work(case):
    op = case["op"]
    if op in ("select", "joint"):
        V, per_action = (case["vocab"], 4) if op == "select" else (LOGITS, 4 * len(HEADS))
        rows = case["groups"] * case["beams"]
        # Finished and dead beams need no logits: 0.9 * 0.95 of the rows are read then.
        read = rows * (0.855 if case["finished"] else 1.0) * V
        out = case["groups"] * case["width"] * (4 + 8 + per_action)
        return {"bytes": read * (BYTES[case["dtype"]] + case["masked"]) + rows * (4 + case["finished"]) + out,
                "flops": 4 * read}
    if op == "reorder":
        n, K, cars = case["groups"] * case["beams"], case["beams"], case["cars"]
        if case["layout"] == "words":
            row = 4 * (cars * (CAR_WORDS + CAR_OUT_WORDS) + SIM_WORDS)
        else:
            row = 4 * cars * (9 + 21 * cars + 68 + 6 + 6 * (cars - 1) + 6 + 2 + 5) + 2 * case["hidden"] + 1 + 28 * cars
        moved, needed = 1 - 1 / K, 1 - (1 - 1 / K) ** (K - 1)                # rows that change, rows another slot takes
        return {"bytes": n * (row * (moved + needed) + 8), "flops": 0}
    n, K, P, M = case["rows"], case["beams"], case["page_len"], case["row_pages"]
    record = case["record"] * BYTES[case["dtype"]]
    entries = n * (M + 1) / 2                                                # table entries in use, on average
    if op == "step":
        # A parent of c beams is copied c - 1 times, up to its (P - 1) / 2 filled slots on average.
        copies = n * (1 - 1 / K) ** K
        return {"bytes": 2 * n * record + 2 * copies * (P - 1) / 2 * record + 8 * entries + 16 * n, "flops": 0}
    G = n // K
    live = G * (M + 1) / 2
    moves = live * (1 - live / (n * M))                                      # live pages beyond the first `live`
    last = sum(min(case["steps"], k) for k in range(1, M * P + 1)) / (M * P)  # records read of a row, on average
    return {"bytes": 2 * moves * P * record + G * record * (last + case["steps"]) + 8 * G * (M + 1) / 2 + 8 * n,
            "flops": 0}


# ---- the definition in 64 bits --------------------------------------------------------------------------------------


def exact(case, seed):
    """Scores, parents and actions of the selections from their definition; the others only move data."""
    if case["op"] not in ("select", "joint"):
        return None
    V = case["vocab"] if case["op"] == "select" else JOINT
    if case["groups"] * case["beams"] * V > 25_000_000:
        return None
    s = prepare(case, seed)
    x = s["logits"].double().cpu().numpy()
    legal = np.ones(x.shape, bool) if s["mask"] is None else s["mask"].cpu().numpy()
    beams = s["scores"].double().cpu().numpy()
    over = np.zeros(beams.shape, bool) if s["finished"] is None else s["finished"].cpu().numpy()
    G, K, W = case["groups"], case["beams"], case["width"]
    size = (x.shape[-1],) if case["op"] == "select" else HEADS
    scores, parents = np.full((G, W), -np.inf), np.tile(np.arange(W) % K, (G, 1))
    actions = np.zeros((G, W, len(size)), np.int64)
    for g in range(G):
        totals, index = [], []
        for k in range(K):
            if not beams[g, k] > -np.inf:
                continue
            if over[g, k]:
                totals.append(beams[g, k:k + 1])
                index.append(np.array([k * V]))
                continue
            sums, norm, at = np.zeros(1), 0.0, 0
            for h in size:                      # the heads' sums, the first head the slowest digit
                row = np.where(legal[g, k, at:at + h], x[g, k, at:at + h], -np.inf)
                top = row.max()
                norm += top + np.log(np.exp(row - top).sum()) if top > -np.inf else 0.0
                sums = np.add.outer(sums, row).ravel()
                at += h
            can = np.nonzero(sums > -np.inf)[0]
            if can.size > W:                    # no more than W of a beam can be among the best, all ties kept
                can = can[sums[can] >= np.partition(sums[can], can.size - W)[can.size - W]]
            totals.append(beams[g, k] - norm + sums[can])
            index.append(k * V + can)
        if not totals:
            continue
        totals, index = np.concatenate(totals), np.concatenate(index)
        best = np.lexsort((index, -totals))[:W]
        scores[g, :best.size] = totals[best]
        parents[g, :best.size] = index[best] // V
        actions[g, :best.size] = np.stack(np.unravel_index(index[best] % V, size), -1)
    if case["op"] == "select":
        actions = actions[..., 0]
    return {"scores": torch.from_numpy(scores), "parents": torch.from_numpy(parents),
            "actions": torch.from_numpy(actions).int()}
