"""The serving operators on moment states, as a list of cases that can be timed and compared.

A case is one pass through an operator of `FastmaxCache`, the cache that keeps one page of moment states per sequence:

  verify    attention of a tree of drafted tokens: every node sees the cached sequence, its ancestors and itself
  accept    the accepted path of such a tree is added to the states
  step      one new token per sequence
  arrange   sequences fork, end and begin: pages change hands, are copied and cleared
  compact   live pages move to the front of the cache

A page is float32 (layers, heads, rows, d + 4).  Rows of a state, for heads of d dims and order 2: for every pair a <= b of 8-wide blocks of
the head dim the 64 products x[8a + i] x[8b + j], then x itself and the constant 1; order 1 has the last d + 1 rows only.  Columns: the sums of
feature times v, the sum of the feature, three of padding.  Scores are q.k / temperature with temperature = 8 sqrt(d); f(s) = 1 + s + s^2 / 2.
"""
import math

import torch

own = False

SEEN = 96   # tokens that every sequence has behind it


def _tree(kind, batch, heads, nodes, d, dtype, order=2, chain=False, absent=0):
    return {"kind": kind, "batch": batch, "heads": heads, "nodes": nodes, "d": d, "dtype": dtype, "order": order, "chain": chain,
            "absent": absent, "layers": 1}


def _pages(kind, batch, layers, heads, d, order=2, **counts):
    return {"kind": kind, "batch": batch, "layers": layers, "heads": heads, "d": d, "order": order, **counts}


def _named(name, case):
    return {"name": name, **case}


def listed():
    return [
        # one user, eight heads, a small tree: latency
        _named("verify_one_user", _tree("verify", 1, 8, 7, 64, "bf16")),
        # the decoding workload's batch with trees of no round size, a few places of the batch empty
        _named("verify_batch", _tree("verify", 32, 16, 25, 64, "bf16", absent=3)),
        # the largest trees
        _named("verify_wide", _tree("verify", 32, 16, 64, 64, "bf16")),
        # narrow float32 heads that check a short draft without branches
        _named("verify_chain_f32", _tree("verify", 24, 12, 5, 32, "f32", chain=True)),
        # one user's accepted path
        _named("accept_one_user", _tree("accept", 1, 8, 7, 64, "bf16")),
        # a batch's accepted paths; some sequences accept nothing
        _named("accept_batch", _tree("accept", 32, 16, 25, 64, "bf16")),
        # one new token for one user
        _named("step_one_user", _tree("step", 1, 8, 1, 64, "bf16")),
        # one new token for a batch that is not full
        _named("step_batch", _tree("step", 32, 16, 1, 64, "f32", absent=5)),
        # beam search of one user: four beams, two of them go on
        _named("arrange_beams", _pages("arrange", 4, 1, 8, 64, forked=2, begun=0, ended=0)),
        # a server between two steps: sequences fork, end and begin, six layers' states in a page
        _named("arrange_server", _pages("arrange", 48, 6, 8, 64, forked=13, begun=5, ended=4)),
        # narrow heads: half of a small batch has ended
        _named("compact_narrow", _pages("compact", 24, 2, 8, 32, ended=12, spare=0)),
        # a large cache after a third of its sequences has ended
        _named("compact_server", _pages("compact", 96, 4, 8, 64, ended=37, spare=5)),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["verify", "verify", "verify", "accept", "accept", "step", "arrange", "compact"])
    d = rng.choice([64, 64, 64, 32, 32, 16])
    heads = rng.choice([4, 6, 8, 12, 16])
    order = rng.choice([2, 2, 2, 2, 1])
    if kind in ("verify", "accept", "step"):
        batch = _log_int(rng, 1, 512 // heads)
        nodes = 1 if kind == "step" else _log_int(rng, 1, 64)
        return _tree(kind, batch, heads, nodes, d, rng.choice(["bf16", "bf16", "f32"]), order=order, chain=rng.random() < 0.3,
                     absent=rng.choice([0, 0, batch // 5]))
    layers = _log_int(rng, 1, 32 // heads)
    batch = _log_int(rng, 2, 48)
    if kind == "compact":
        return _pages(kind, batch, layers, heads, d, order, ended=rng.randrange(batch), spare=rng.randrange(4))
    forked = rng.randrange(batch // 2 + 1)
    begun = rng.randrange((batch - forked) // 2 + 1)
    ended = rng.randrange((batch - forked - begun) // 2 + 1)
    return _pages(kind, batch, layers, heads, d, order, forked=forked, begun=begun, ended=ended)


# ---- sizes ------------------------------------------------------------------------------------------------------------


def _rows(d, order):
    blocks = d // 8
    return (32 * blocks * (blocks + 1) if order == 2 else 0) + d + 1


def _state_bytes(d, order):
    return 4 * _rows(d, order) * (d + 4)


def _counts(case):
    """Nodes per sequence: from all of them down to half."""
    n, b = case["nodes"], case["batch"]
    return [n - (i * (n // 2 + 1) // b) for i in range(b)]


def _path_lengths(case):
    """Accepted tokens per sequence: none, some, up to eight (fewer where its tree is not as deep)."""
    return [min((5 * i + 4) % 9, n) for i, n in enumerate(_counts(case))]


def _live(case):
    """Which places of the batch hold a sequence: the absent ones stand at even distances."""
    b, absent = case["batch"], case["absent"]
    gone = {(2 * i + 1) * b // (2 * absent) for i in range(absent)}
    return [i not in gone for i in range(b)]


def work(case):
    d, order, heads = case["d"], case["order"], case["heads"]
    # operations: every product of two dims once, though the rows of the blocks a = a hold them twice
    features = (d * (d + 1) // 2 if order == 2 else 0) + d + 1
    page = case["layers"] * heads * _state_bytes(d, order)
    if case["kind"] == "arrange":
        return {"bytes": (2 * case["forked"] + case["begun"]) * page + 12 * case["batch"], "flops": 0}
    if case["kind"] == "compact":
        # live pages behind the position that the live ones will fill: the ended sequences stand at the front
        kept = case["batch"] - case["ended"]
        return {"bytes": 2 * min(case["ended"], kept) * page + 8 * case["batch"], "flops": 0}
    size = 2 if case["dtype"] == "bf16" else 4
    live = [i for i, x in enumerate(_live(case)) if x]
    if case["kind"] == "step":
        return {"bytes": len(live) * (2 * page + 4 * heads * d * size), "flops": 4 * len(live) * heads * features * (d + 1)}
    if case["kind"] == "accept":
        taken = [_path_lengths(case)[i] for i in live]
        tokens = sum(taken)
        return {"bytes": 2 * page * sum(t > 0 for t in taken) + 2 * tokens * heads * d * size, "flops": 2 * tokens * heads * features * (d + 1)}
    nodes = sum(_counts(case)[i] for i in live)
    return {"bytes": len(live) * page + 4 * nodes * heads * d * size, "flops": 2 * nodes * heads * features * (d + 1)}


# ---- what a program has in hand ----------------------------------------------------------------------------------------


def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


def _phi(x):
    """Features of order 2 in the state's row order, without weights: (..., d) -> (..., rows)."""
    d = x.shape[-1]
    xb = x.reshape(*x.shape[:-1], d // 8, 8)
    a, b = torch.triu_indices(d // 8, d // 8, device=x.device)
    pairs = xb[..., a, :].unsqueeze(-1) * xb[..., b, :].unsqueeze(-2)
    return torch.cat([pairs.flatten(-3), x, torch.ones_like(x[..., :1])], -1)


def _features(x, order):
    return _phi(x) if order == 2 else torch.cat([x, torch.ones_like(x[..., :1])], -1)


def _states(case, count, gen):
    """Moment states of `count` sequences (layers, heads) that have SEEN tokens behind them."""
    d, order = case["d"], case["order"]
    out = torch.zeros(count, case["layers"], case["heads"], _rows(d, order), d + 4, device="cuda")
    for page in out:
        k = torch.randn(case["layers"], case["heads"], SEEN, d, device="cuda", generator=gen)
        v = torch.randn(case["layers"], case["heads"], SEEN, d, device="cuda", generator=gen)
        v1 = torch.cat([v, torch.ones_like(v[..., :1])], -1)
        page[..., : d + 1] = torch.matmul(_features(k, order).transpose(-1, -2), v1)
    return out


def _tree_inputs(case, seed, gen):
    host = torch.Generator().manual_seed(seed)
    b, h, n, d = case["batch"], case["heads"], case["nodes"], case["d"]
    # what a fused projection leaves: (b, n, 3, h, d), seen as three (b, h, n, d) tensors
    qkv = torch.randn(b, n, 3, h, d, device="cuda", generator=gen).to(_dtype(case))
    q, k, v = (qkv[:, :, i].transpose(1, 2) for i in range(3))
    # a node hangs on one of the few nodes before it: branching trees of depth about n / 3
    ids = torch.arange(n)
    parents = (ids - 1 - (torch.rand(b, n, generator=host) * torch.minimum(ids + 1, torch.tensor(5))).long()).clamp_(min=-1)
    if case["chain"]:
        parents = (ids - 1).expand(b, n).contiguous()
    lengths = torch.tensor(_counts(case))
    live = torch.tensor(_live(case))
    # pages in an order of their own, two more than there are places; absent places have none
    table = torch.where(live, torch.randperm(b + 2, generator=host)[:b], torch.tensor(-1))
    # the accepted path: the wanted number of nodes from some node up to the root, as far as the tree is deep
    depth = torch.zeros(b, n, dtype=torch.long)
    for i in range(n):
        depth[:, i] = torch.where(parents[:, i] < 0, 0, depth.gather(1, parents[:, i : i + 1].clamp(min=0))[:, 0]) + 1
    last = []
    for i, want in enumerate(_path_lengths(case)):
        deep = depth[i, : lengths[i]]
        fit = (deep == min(want, int(deep.max()))).nonzero()[:, 0]
        last.append(int(fit[int(torch.randint(len(fit), (1,), generator=host))]) if want else -1)
    cuda = {name: x.to(torch.int32).cuda() for name, x in (("parents", parents), ("lengths", lengths), ("table", table), ("last", torch.tensor(last)))}
    if case["kind"] == "step":
        q, k, v = q[:, :, 0], k[:, :, 0], v[:, :, 0]
    return {"q": q, "k": k, "v": v, "out": torch.zeros_like(q, memory_format=torch.contiguous_format), **cuda,
            "parents": None if case["chain"] else cuda["parents"]}


def _page_inputs(case, seed):
    host = torch.Generator().manual_seed(seed)
    b = case["batch"]
    if case["kind"] == "compact":
        # the sequences that came first have ended; a few pages were never used
        table = torch.arange(b)
        table[: case["ended"]] = -1
        seats = torch.randperm(b, generator=host)   # which sequence has which page does not matter to the cache
        return {"table": table[seats].to(torch.int32).cuda()}, b + case["spare"]
    # sequences that end hand their places to forks of others and to new ones
    places = torch.randperm(b, generator=host)
    forked, begun, ended = case["forked"], case["begun"], case["ended"]
    sources = torch.arange(b)
    stay = places[forked + begun + ended :]
    sources[places[:forked]] = stay[torch.randint(len(stay), (forked,), generator=host)]
    sources[places[forked : forked + begun]] = -2
    sources[places[forked + begun : forked + begun + ended]] = -1
    table = torch.randperm(b, generator=host)
    return {"table": table.to(torch.int32).cuda(), "sources": sources.to(torch.int32).cuda()}, b


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["kind"] in ("arrange", "compact"):
        state, pages = _page_inputs(case, seed)
    else:
        state, pages = _tree_inputs(case, seed, gen), case["batch"] + 2
    state["case"] = case
    state["pages"] = _states(case, pages, gen)
    state["table0"] = state["table"].clone()
    if own:
        from reproducing_fastmax_results_b200.cache import FastmaxCache

        cache = FastmaxCache(case["batch"], case["heads"], case["d"], p=case["order"], temperature=8.0 * math.sqrt(case["d"]),
                             layers=case["layers"], pages=pages)
        cache.state.copy_(state["pages"])
        cache.table.copy_(state["table"])
        state["cache"], state["pages"], state["table"] = cache, cache.state, cache.table
    return state


# ---- one pass ------------------------------------------------------------------------------------------------------------


def run(state):
    kind = state["case"]["kind"]
    if own:
        return _run_own(state, kind)
    if kind in ("verify", "accept", "step"):
        return _run_tree(state, kind)
    return _run_arrange(state) if kind == "arrange" else _run_compact(state)


def _run_own(state, kind):
    cache = state["cache"]
    if kind == "verify":
        return cache.verify(state["q"], state["k"], state["v"], parents=state["parents"], lengths=state["lengths"], out=state["out"])
    if kind == "accept":
        cache.accept(state["k"], state["v"], state["last"], parents=state["parents"])
        return cache.state
    if kind == "step":
        return {"o": cache.step(state["q"], state["k"], state["v"], out=state["out"]), "state": cache.state}
    # every pass starts from the same table: it is what the cache has to work on
    cache.table.copy_(state["table0"])
    done = cache.arrange(state["sources"]) if kind == "arrange" else cache.compact()
    return {"done": done, "table": cache.table, "state": cache.state}


def _visible(state, n):
    """(b, n, n): whether node j is node i or one of its ancestors."""
    parents = state["parents"]
    if parents is None:
        return torch.ones(1, n, n, dtype=torch.bool, device="cuda").tril()
    # one step up as a matrix; powers of two of it reach all ancestors
    up = (parents.long()[:, :, None] == torch.arange(n, device="cuda")).float()
    seen = up + torch.eye(n, device="cuda")
    for _ in range(max(1, (n - 1).bit_length())):
        seen = (seen @ seen).clamp_(max=1.0)
    return seen > 0


def _run_tree(state, kind):
    case = state["case"]
    d, order = case["d"], case["order"]
    table = state["table"].long()
    live = table >= 0
    page = table.clamp(min=0)
    if kind == "step":
        q, k, v = (state[x].unsqueeze(2).float() for x in "qkv")
        n = 1
    else:
        q, k, v = (state[x].float() for x in "qkv")
        n = case["nodes"]
    t = 1.0 / (8.0 * math.sqrt(d))
    v1 = torch.cat([v, torch.ones_like(v[..., :1])], -1)
    moments = state["pages"][:, 0]                                  # (pages, h, rows, d + 4)
    if kind in ("accept", "step"):
        if kind == "accept":
            last = state["last"].long()
            onpath = _visible(state, n).expand(case["batch"], n, n)[torch.arange(case["batch"], device="cuda"), last.clamp(min=0)] & (last >= 0)[:, None]
        else:
            onpath = torch.ones(case["batch"], 1, dtype=torch.bool, device="cuda")
        taken = (onpath & live[:, None])[:, None, :, None]
        grown = moments[page][..., : d + 1] + torch.matmul((_features(k, order) * taken).transpose(-1, -2), v1)
        moments[page[live], :, :, : d + 1] = grown[live]
        if kind == "accept":
            return state["pages"]
    s = moments[page][..., : d + 1]
    weights = torch.full((s.shape[-2],), t, device="cuda")
    weights[-1] = 1.0
    if order == 2:
        a, b = torch.triu_indices(d // 8, d // 8, device="cuda")
        weights[: 64 * len(a)] = torch.where(a == b, 0.5 * t * t, t * t).repeat_interleave(64)
    sums = torch.matmul(_features(q, order) * weights, s)
    if kind == "verify":
        x = torch.matmul(q, k.transpose(-1, -2)) * t
        f = 1.0 + x + (0.5 * x * x if order == 2 else 0.0)
        sums = sums + torch.matmul(f * _visible(state, n)[:, None], v1)
    o = (sums[..., :d] / sums[..., d:]).to(_dtype(case))
    if kind == "step":
        rows = live[:, None, None]
        state["out"] = torch.where(rows, o[:, :, 0], state["out"])
        return {"o": state["out"], "state": state["pages"]}
    rows = (live[:, None] & (torch.arange(n, device="cuda") < state["lengths"][:, None]))[:, None, :, None]
    state["out"] = torch.where(rows, o, state["out"])
    return state["out"]


def _run_arrange(state):
    pages, table, sources = state["pages"], state["table0"].long(), state["sources"].long()
    b, count = len(table), len(pages)
    ids = torch.arange(b, device="cuda")
    held = torch.where(sources >= 0, table[sources.clamp(min=0)], -1)      # the page that a place goes on from
    first = torch.full((count + 1,), b, device="cuda").scatter_reduce_(0, torch.where(held >= 0, held, count), ids, "amin")[:count]
    keeps = (held >= 0) & (first[held.clamp(min=0)] == ids)
    free = first == b
    wants = (sources == -2) | ((held >= 0) & ~keeps)
    rank = wants.long().cumsum(0) - 1
    freed = torch.sort((~free).long(), stable=True).indices                # free pages first, ascending
    got = wants & (rank < free.sum())
    new = torch.where(keeps, held, torch.where(got, freed[rank.clamp(min=0, max=count - 1)], -1))
    copies = got & (held >= 0)
    fresh = got & (held < 0)
    pages[new[copies]] = pages[held[copies]]
    pages[new[fresh]] = 0.0
    state["table"] = new.to(torch.int32)
    asked = (sources < -2) | (sources >= b) | (wants & ~got)
    return {"done": asked.sum().to(torch.int32).reshape(1), "table": state["table"], "state": pages}


def _run_compact(state):
    pages, table = state["pages"], state["table0"].long()
    count = len(pages)
    live = torch.zeros(count + 1, dtype=torch.bool, device="cuda").scatter_(0, torch.where(table >= 0, table, count), True)[:count]
    total = live.sum()
    ids = torch.arange(count, device="cuda")
    movers = (live & (ids >= total)).nonzero()[:, 0]
    holes = (~live & (ids < total)).nonzero()[:, 0]
    pages[holes] = pages[movers]
    where = ids.clone()
    where[movers] = holes
    state["table"] = torch.where(table >= 0, where[table.clamp(min=0)], -1).to(torch.int32)
    return {"done": total.to(torch.int32).reshape(1), "table": state["table"], "state": pages}


# ---- the definition, in 64 bits ---------------------------------------------------------------------------------------------


def _square(moments, d):
    """(…, rows, d + 4) of order 2 -> the full symmetric (…, d, d, d + 1) sums of x_m x_n [v | 1]."""
    full = torch.zeros(*moments.shape[:-2], d, d, d + 1, dtype=torch.float64, device=moments.device)
    row = 0
    for a in range(0, d, 8):
        for b in range(a, d, 8):
            block = moments[..., row : row + 64, : d + 1].unflatten(-2, (8, 8))
            full[..., a : a + 8, b : b + 8, :] = block
            if a != b:
                full[..., b : b + 8, a : a + 8, :] = block.transpose(-3, -2)
            row += 64
    return full


def _ancestors(parents, node):
    found = []
    while node >= 0:
        found.append(node)
        node = parents[node]
    return found


def _grow(moments, k, v, order):
    """moments (h, rows, d + 4) in float64 and the keys and values (h, t, d) that are added to them, in place."""
    h, t, d = k.shape
    v1 = torch.cat([v, torch.ones_like(v[..., :1])], -1)
    row = 0
    if order == 2:
        for a in range(0, d, 8):
            for b in range(a, d, 8):
                moments[:, row : row + 64, : d + 1] += torch.einsum("htm,htn,htc->hmnc", k[..., a : a + 8], k[..., b : b + 8], v1).flatten(1, 2)
                row += 64
    moments[:, row : row + d, : d + 1] += torch.einsum("htm,htc->hmc", k, v1)
    moments[:, row + d, : d + 1] += v1.sum(1)


def exact(case, seed):
    state = prepare(case, seed)
    b, d, order = case["batch"], case["d"], case["order"]
    pages, table = state["pages"].double(), state["table"].tolist()
    if case["kind"] == "arrange":
        sources = state["sources"].tolist()
        old, new, short = table, [-1] * b, 0
        taken, later = set(), []
        for i, j in enumerate(sources):
            if 0 <= j < b and old[j] >= 0:
                if old[j] in taken:
                    later.append((i, old[j]))
                else:
                    taken.add(old[j])
                    new[i] = old[j]
            elif j == -2:
                later.append((i, -1))
            elif j < -2 or j >= b:
                short += 1
        free = [p for p in range(len(pages)) if p not in taken]
        for (i, source), page in zip(later, free):
            new[i] = page
            pages[page] = pages[source] if source >= 0 else 0.0
        short += max(0, len(later) - len(free))
        return {"done": torch.tensor([short], dtype=torch.int32), "table": torch.tensor(new, dtype=torch.int32), "state": pages}
    if case["kind"] == "compact":
        live = sorted(p for p in table if p >= 0)
        movers = [p for p in live if p >= len(live)]
        holes = [p for p in range(len(live)) if p not in set(live)]
        goes = dict(zip(movers, holes))
        for p, hole in goes.items():
            pages[hole] = pages[p]
        return {"done": torch.tensor([len(live)], dtype=torch.int32),
                "table": torch.tensor([goes.get(p, p) for p in table], dtype=torch.int32), "state": pages}
    t = 1.0 / (8.0 * math.sqrt(d))
    q, k, v = (state[x].double() for x in "qkv")
    if case["kind"] == "step":
        q, k, v = (x.unsqueeze(2) for x in (q, k, v))
    n = q.shape[2]
    parents = state["parents"].tolist() if state["parents"] is not None else [list(range(-1, n - 1))] * b
    lengths, last = state["lengths"].tolist(), state["last"].tolist()
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for i in range(b):
        if table[i] < 0:
            continue
        moments = pages[table[i], 0]
        if case["kind"] == "accept":
            path = _ancestors(parents[i], last[i])
            if path:
                _grow(moments, k[i][:, path], v[i][:, path], order)
            continue
        if case["kind"] == "step":
            _grow(moments, k[i], v[i], order)
        r = moments.shape[-2] - d - 1
        sums = moments[:, None, -1, : d + 1] + torch.einsum("hnm,hmc->hnc", q[i], moments[:, r : r + d, : d + 1]) * t
        if order == 2:
            sums = sums + 0.5 * t * t * torch.einsum("hnm,hnmc->hnc", q[i], torch.einsum("hnl,hmlc->hnmc", q[i], _square(moments, d)))
        if case["kind"] == "verify":
            x = torch.einsum("hnd,hmd->hnm", q[i], k[i]) * t
            f = 1.0 + x + (0.5 * x * x if order == 2 else 0.0)
            sees = torch.zeros(n, n, dtype=torch.float64, device=q.device)
            for node in range(n):
                sees[node, _ancestors(parents[i], node)] = 1.0
            f = f * sees
            sums = sums + torch.cat([torch.einsum("hnm,hmc->hnc", f, v[i]), f.sum(-1, keepdim=True)], -1)
        o = sums[..., :d] / sums[..., d:]
        out[i, :, : lengths[i]] = o[:, : lengths[i]]
    if case["kind"] == "verify":
        return out
    if case["kind"] == "accept":
        return pages
    return {"o": out[:, :, 0], "state": pages}
