"""Trees of drafted tokens over moment states and pages of a cache, against the oracle in 64 bits (tests/serving_oracle.py), whose error
bounds are the tolerances."""
import math

import numpy as np
import pytest
import torch

import serving_oracle as so
from oracle import fastmax_oracle as orc

pytestmark = pytest.mark.gpu

A = (1.1, 0.9, 0.4)


def host(t):
    return t.detach().double().cpu().numpy()


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def states(count, heads, d, order, gen, seen=40, layers=None):
    """States of sequences with `seen` random tokens behind them; float32 (count, heads, rows, d + 4), or with layers behind the pages."""
    rows = (4 * d * (d // 8 + 1) if order == 2 else 0) + d + 1
    shape = (count, heads) if layers is None else (count, layers, heads)
    k, v = (torch.randn(*shape, seen, d, device="cuda", generator=gen) for _ in range(2))
    v1 = torch.cat([v, torch.ones_like(v[..., :1])], -1)
    feats = [torch.ones_like(v[..., :1])]
    feats.insert(0, k)
    if order == 2:
        for b in range(d - 8, -1, -8):
            for a in range(d - 8, b - 1, -8):
                feats.insert(0, (k[..., b:b + 8, None] * k[..., None, a:a + 8]).flatten(-2))
    out = torch.zeros(*shape, rows, d + 4, device="cuda")
    out[..., : d + 1] = torch.cat(feats, -1).transpose(-1, -2) @ v1
    return out


def random_parents(b, n, rng):
    p = np.array([[rng.integers(max(-1, i - 5), i) for i in range(n)] for _ in range(b)], dtype=np.int32)
    return p


def check_tree(o, g, q, k, v, state, table, parents, lengths, order, inv_t, untouched=0.0):
    """Every row of o (b, h, n, d) and g (b, h, n); rows that are not computed hold `untouched`."""
    b, h, n, d = q.shape
    bf16 = q.dtype == torch.bfloat16
    oh, gh, qh, kh, vh, sh = host(o), None if g is None else host(g), host(q), host(k), host(v), host(state)
    for i in range(b):
        page = i if table is None else int(table[i])
        count = n if lengths is None else min(max(int(lengths[i]), 0), n)
        if page < 0 or page >= len(sh):
            count = 0
        assert (oh[i, :, count:] == untouched).all()
        if count == 0:
            continue
        up = np.arange(n) - 1 if parents is None else np.asarray(parents[i])
        for j in range(h):
            ref, gref, size, gsize = so.tree(qh[i, j, :count], kh[i, j, :count], vh[i, j, :count], sh[page, j], up, order, A, inv_t)
            off = np.abs(oh[i, j, :count] - ref) / so.attention_tolerance(ref, size, bf16)
            assert off.max() <= 1.0, (i, j, np.unravel_index(off.argmax(), off.shape), off.max())
            if gh is not None:
                assert (np.abs(gh[i, j, :count] - gref) <= (so.SUMS_BF16 if bf16 else so.SUMS_F32) * gsize).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d,order", [(16, 1), (16, 2), (32, 1), (32, 2), (64, 1), (64, 2)])
@pytest.mark.parametrize("n", [1, 2, 7, 8, 9, 16, 17, 31, 33, 63, 64])
def test_trees(n, d, order, dtype):
    from reproducing_fastmax_results_b200 import _lib as L

    b, h = 2, 3
    rng = np.random.default_rng(1000 * n + d + order)
    gen = torch.Generator(device="cuda").manual_seed(n + d)
    q, k, v = (torch.randn(b, h, n, d, device="cuda", generator=gen).to(dtype) for _ in range(3))
    state = states(b, h, d, order, gen)
    before = state.clone()
    parents = random_parents(b, n, rng)
    inv_t = 1.0 / (2.0 * math.sqrt(d))
    o, g = L.tree_attention(q, k, v, state, inv_t, *A, order, parents=i32(parents))
    check_tree(o, g, q, k, v, state, None, parents, None, order, inv_t)
    assert torch.equal(state, before)
    o, g = L.tree_attention(q, k, v, state, inv_t, *A, order)   # a chain
    check_tree(o, g, q, k, v, state, None, None, None, order, inv_t)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads", [1, 16, 19, 40, 80, 160, 300, 520])   # every split of a head over blocks
def test_trees_of_any_number_of_heads(heads, dtype):
    from reproducing_fastmax_results_b200 import _lib as L

    for d, n in ((64, 11), (32, 40)):
        gen = torch.Generator(device="cuda").manual_seed(heads)
        q, k, v = (torch.randn(1, heads, n, d, device="cuda", generator=gen).to(dtype) for _ in range(3))
        state = states(1, heads, d, 2, gen)
        o, g = L.tree_attention(q, k, v, state, 0.1, *A, 2)
        some = sorted({0, heads // 3, heads - 1})
        check_tree(o[:, some], g[:, some], *(t[:, some] for t in (q, k, v)), state[:, some], None, None, None, 2, 0.1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d,order,n", [(64, 2, 13), (32, 2, 24), (16, 2, 5), (64, 1, 40), (64, 2, 50)])
def test_ragged_trees_on_pages(d, order, n, dtype):
    """Lengths from none to all (and beyond either end), sequences without a page, pages with gaps between them, parents that are no nodes,
    views of a fused projection, results into strided memory whose other rows stay as they were, garbage in all rows that are not there."""
    from reproducing_fastmax_results_b200 import _lib as L

    b, h = 7, 2
    rng = np.random.default_rng(n)
    gen = torch.Generator(device="cuda").manual_seed(n)
    cache = states(9, h, d, order, gen, layers=3)
    table = [8, -1, 0, 3, 9, 5, 2]
    lengths = [n, n, n // 2, 0, n, n + 7, 1]
    parents = random_parents(b, n, rng)
    asked = parents.copy()
    if n > 6:
        asked[0, 3], asked[0, 4], asked[2, 2] = 3, 1000, -7   # not before the node: the sequence itself
        parents[0, 3] = parents[0, 4] = parents[2, 2] = -1
    qkv = torch.randn(b, n, 3, h, d, device="cuda", generator=gen).to(dtype)
    for i in range(b):
        qkv[i, max(0, min(lengths[i], n)):] = float("nan")
        if table[i] in (-1, 9):
            qkv[i] = float("inf")
    q, k, v = (qkv[:, :, j].transpose(1, 2) for j in range(3))
    hold = torch.full((b, n, h, d + 16), 7.0, device="cuda").to(dtype)
    out = hold[..., :d].transpose(1, 2)
    inv_t = 0.15
    o, g = L.tree_attention(q, k, v, cache[:, 1], inv_t, *A, order, table=i32(table), parents=i32(asked), lengths=i32(lengths), out=out)
    check_tree(o, None, q, k, v, cache[:, 1], table, parents, lengths, order, inv_t, untouched=7.0)
    assert (hold[..., d:] == 7.0).all()
    for i in range(b):
        for j in range(h):
            if table[i] not in (-1, 9):
                assert torch.isfinite(g[i, j, : max(0, min(lengths[i], n))]).all()


def test_a_node_without_a_number_stays_its_own():
    """Infinities and NaN in a node reach its descendants and no other node; those in q reach that node alone."""
    from reproducing_fastmax_results_b200 import _lib as L

    for dtype in (torch.float32, torch.bfloat16):
        gen = torch.Generator(device="cuda").manual_seed(2)
        q, k, v = (torch.randn(1, 2, 12, 64, device="cuda", generator=gen).to(dtype) for _ in range(3))
        parents = [-1, 0, 0, 1, 1, 2, -1, 6, 4, 4, 3, 5]
        state = states(1, 2, 64, 2, gen)
        clean, _ = L.tree_attention(q, k, v, state, 0.1, *A, 2, parents=i32([parents]))
        v[:, :, 1, 3] = float("inf")
        k[:, :, 6, 5] = float("nan")
        q[:, :, 5] = float("nan")
        o, _ = L.tree_attention(q, k, v, state, 0.1, *A, 2, parents=i32([parents]))
        for i in range(12):
            nodes = so.path(parents, i)
            if 1 in nodes or 6 in nodes or i == 5:
                assert not torch.isfinite(o[:, :, i]).all(), i
            else:
                assert torch.equal(o[:, :, i], clean[:, :, i]), i


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d,n", [(16, 3), (32, 20), (64, 37)])
def test_rows_of_any_alignment(d, n, dtype):
    """Rows that start anywhere, at odd distances: the same bits as contiguous ones."""
    from reproducing_fastmax_results_b200 import _lib as L

    b, h = 3, 2
    gen = torch.Generator(device="cuda").manual_seed(d)
    odd = [torch.randn(b, n, h, d + 3, device="cuda", generator=gen).to(dtype)[..., 1: d + 1].transpose(1, 2) for _ in range(3)]
    even = [t.contiguous() for t in odd]
    state = states(b, h, d, 2, gen)
    parents = i32(random_parents(b, n, np.random.default_rng(n)))
    wide = torch.zeros(b, h, n, d + 5, device="cuda").to(dtype)
    o, g = L.tree_attention(*odd, state, 0.1, *A, 2, parents=parents, out=wide[..., 3: d + 3])
    ref, gref = L.tree_attention(*even, state, 0.1, *A, 2, parents=parents)
    assert torch.equal(o, ref) and torch.equal(g, gref)
    assert (wide[..., :3] == 0).all() and (wide[..., d + 3:] == 0).all()
    both = [state.clone(), state.clone()]
    for st, (_, k, v) in zip(both, (odd, even)):
        L.tree_accept(k, v, st, i32([n - 1, 0, n // 2]), 2, parents=parents)
    assert torch.equal(*both)
    table = i32([2, 0, 1])
    outs = [L.decode_step_paged(*(t[:, :, 0] for t in x), st, table, 0.1)[0] for x, st in zip((odd, even), both)]
    assert torch.equal(*outs) and torch.equal(*both)


@pytest.mark.parametrize("heads", [3, 200])   # one head over a cluster of blocks, many heads
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_chain_is_that_many_steps(dtype, heads):
    """Drafts without branches, all of them accepted: outputs and states of steps token by token, up to the rounding of either."""
    from reproducing_fastmax_results_b200 import _lib as L

    n, d = 6, 64
    gen = torch.Generator(device="cuda").manual_seed(heads)
    q, k, v = (torch.randn(1, heads, n, d, device="cuda", generator=gen).to(dtype) for _ in range(3))
    stepped = states(1, heads, d, 2, gen)
    taken = stepped.clone()
    o, g = L.tree_attention(q, k, v, taken, 0.1, *A, 2)
    some = [0, heads // 2, heads - 1]
    size = [so.tree(*(host(t[0, j]) for t in (q, k, v)), host(taken[0, j]), np.arange(n) - 1, 2, A, 0.1)[2] for j in some]
    L.tree_accept(k, v, taken, i32([n - 1]))
    for t in range(n):
        x, _ = L.decode_step(q[:, :, t], k[:, :, t], v[:, :, t], stepped, 0.1, *A, 2)
        for j, s in zip(some, size):
            a, b = host(o[0, j, t]), host(x[0, j])
            assert (np.abs(a - b) <= so.attention_tolerance(a, s[t], dtype == torch.bfloat16) + so.attention_tolerance(b, s[t], dtype == torch.bfloat16)).all()
    for j in some:
        a, b = host(taken[0, j]), host(stepped[0, j])
        _, s = so.grown(b, host(k[0, j]), host(v[0, j]), 2)
        assert (np.abs(a - b)[:, : d + 1] <= 2 * so.grown_tolerance(s, n)).all()


def test_an_empty_sequence_has_its_drafts_only():
    from reproducing_fastmax_results_b200 import _lib as L

    gen = torch.Generator(device="cuda").manual_seed(3)
    q, k, v = (torch.randn(2, 4, 10, 32, device="cuda", generator=gen) for _ in range(3))
    o, g = L.tree_attention(q, k, v, L.new_state(2, 4, 32), 0.1)
    ref, gref = orc.fastmax_naive(host(q), host(k), host(v), True, orc.Poly(1.0, 1.0, 0.5, 0.1, 2))
    assert orc.max_norm_err(host(o), ref) < so.SUMS_F32 * 10 and orc.max_norm_err(host(g), gref) < so.SUMS_F32 * 10


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d,order", [(16, 1), (16, 2), (32, 1), (32, 2), (64, 1), (64, 2)])
@pytest.mark.parametrize("n", [1, 5, 20, 64])
def test_taking_a_path(n, d, order, dtype):
    from reproducing_fastmax_results_b200 import _lib as L

    b, h = 6, 2
    rng = np.random.default_rng(n + d)
    gen = torch.Generator(device="cuda").manual_seed(n + d)
    cache = states(8, h, d, order, gen, layers=2)
    before = cache.clone()
    qkv = torch.randn(b, n, 3, h, d, device="cuda", generator=gen).to(dtype)
    k, v = (qkv[:, :, j].transpose(1, 2) for j in range(2))
    table, last = [7, 0, -1, 4, 2, 8], [n - 1, -1, n - 1, n // 2, 0, n - 1]
    for parents in (random_parents(b, n, rng), None):
        L.tree_accept(k, v, cache[:, 0], i32(last), order, table=i32(table), parents=None if parents is None else i32(parents))
        for i in range(b):
            if not 0 <= table[i] < 8:
                continue
            nodes = so.path(np.arange(n) - 1 if parents is None else parents[i], last[i])
            for j in range(h):
                got, old = host(cache[table[i], 0, j]), host(before[table[i], 0, j])
                assert (got[:, d + 1:] == old[:, d + 1:]).all()
                ref, size = so.grown(old, host(k[i, j, nodes]), host(v[i, j, nodes]), order)
                assert (np.abs(got[:, : d + 1] - ref) <= so.grown_tolerance(size, len(nodes))).all()
        rest = [p for p in range(8) if p not in table or last[table.index(p)] < 0]
        assert torch.equal(cache[:, 1], before[:, 1]) and torch.equal(cache[rest], before[rest])
        cache.copy_(before)


def test_a_last_node_that_is_none_takes_nothing():
    from reproducing_fastmax_results_b200 import _lib as L

    gen = torch.Generator(device="cuda").manual_seed(5)
    k, v = (torch.randn(4, 3, 6, 64, device="cuda", generator=gen) for _ in range(2))
    state = states(4, 3, 64, 2, gen)
    before = state.clone()
    L.tree_accept(k, v, state, i32([-1, 6, -(1 << 31), (1 << 31) - 1]))
    assert torch.equal(state, before)


@pytest.mark.parametrize("heads", [1, 8, 37, 150, 600])
def test_taking_one_token_is_the_state_of_a_step(heads):
    from reproducing_fastmax_results_b200 import _lib as L

    for d, order in ((64, 2), (64, 1), (32, 2), (16, 2)):
        gen = torch.Generator(device="cuda").manual_seed(heads)
        q, k, v = (torch.randn(1, heads, 1, d, device="cuda", generator=gen).bfloat16() for _ in range(3))
        a = states(1, heads, d, order, gen, seen=4)
        b = a.clone()
        L.tree_accept(k, v, a, i32([0]), order)
        L.decode_step(q, k, v, b, 0.1, order=order)
        # bf16 keys and values: the products of a feature are exact in float32, feature times v rounds at most once, the sum once
        assert ((a - b).abs() <= 2 * 2.0 ** -24 * (a.abs() + b.abs()) + 1e-30).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads", [1, 2, 7])   # few heads: the dense state's own kernel, bit for bit
def test_steps_on_pages_are_the_steps_of_a_dense_state(heads, dtype):
    from reproducing_fastmax_results_b200 import _lib as L

    for d, order in ((64, 2), (32, 1), (16, 2)):
        gen = torch.Generator(device="cuda").manual_seed(heads)
        cache = states(5, heads, d, order, gen, layers=2)
        before = cache.clone()
        table = [4, -1, 0, 5]
        qkv = torch.randn(4, 3, heads, d, device="cuda", generator=gen).to(dtype)
        q, k, v = qkv.unbind(1)
        out = torch.full((4, heads, d), 3.0, device="cuda").to(dtype)
        o, g = L.decode_step_paged(q, k, v, cache[:, 1], i32(table), 0.1, *A, order, out=out)
        dense = before[[4, 0, 0, 0], 1].contiguous()   # as many heads as the call had: the same split over blocks
        ref, gref = L.decode_step(q, k, v, dense, 0.1, *A, order)
        for place, page in ((0, 4), (2, 0)):
            assert torch.equal(o[place], ref[place]) and torch.equal(g[place], gref[place])
            assert torch.equal(cache[page, 1], dense[place])
        assert (o[1] == 3.0).all() and (o[3] == 3.0).all()
        assert torch.equal(cache[:, 0], before[:, 0]) and torch.equal(cache[1:4], before[1:4])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("batch,heads,d,order", [(9, 16, 64, 2), (4, 19, 64, 2), (17, 8, 32, 2), (40, 13, 64, 1), (9, 16, 32, 1), (60, 16, 16, 2),
                                                   (65, 16, 16, 1)])
def test_steps_of_many_heads_on_pages(batch, heads, d, order, dtype):
    from reproducing_fastmax_results_b200 import _lib as L

    gen = torch.Generator(device="cuda").manual_seed(batch)
    cache = states(batch + 1, heads, d, order, gen, layers=2)
    before = cache.clone()
    table = np.random.default_rng(batch).permutation(batch + 1)[:batch]
    table[[1, batch - 1]] = [-1, batch + 1]
    qkv = torch.randn(batch, 3, heads, d, device="cuda", generator=gen).to(dtype)
    qkv[1] = float("nan")
    q, k, v = qkv.unbind(1)
    out = torch.full((batch, heads, d), 3.0, device="cuda").to(dtype)
    o, g = L.decode_step_paged(q, k, v, cache[:, 0], i32(table), 0.1, *A, order, out=out)
    for i in (0, 1, 2, batch // 2, batch - 2, batch - 1):
        page = int(table[i])
        if not 0 <= page <= batch:
            assert (o[i] == 3.0).all() and (g[i] == 0).all()
            continue
        for j in (0, heads - 1):
            old, new = host(before[page, 0, j]), host(cache[page, 0, j])
            kk, vv, qq = (host(t[i, j])[None] for t in (k, v, q))
            ref, size = so.grown(old, kk, vv, order)
            assert (np.abs(new[:, : d + 1] - ref) <= so.grown_tolerance(size, 1)).all() and (new[:, d + 1:] == old[:, d + 1:]).all()
            oref, gref, osize, gsize = so.tree(qq, kk, vv, old, [-1], order, A, 0.1)
            rounding = 2.0 ** (-8 if dtype == torch.bfloat16 else -24)
            assert (np.abs(host(o[i, j])[None] - oref) <= rounding * np.abs(oref) + so.SUMS_F32 * osize).all()
            assert abs(float(g[i, j]) - gref[0]) <= so.SUMS_F32 * gsize[0]
    rest = sorted(set(range(batch + 1)) - set(table.tolist()))
    assert torch.equal(cache[:, 1], before[:, 1]) and torch.equal(cache[rest], before[rest])
    again = before.clone()   # the same bits on every run
    o2, _ = L.decode_step_paged(q, k, v, again[:, 0], i32(table), 0.1, *A, order, out=torch.full_like(out, 3.0))
    assert torch.equal(o2, o) and torch.equal(again, cache)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("batch,heads,d,order", [(3, 2, 64, 2), (9, 16, 64, 2), (17, 8, 32, 2), (12, 13, 64, 1), (70, 16, 16, 2)])   # few heads, many
def test_a_step_without_a_table(batch, heads, d, order, dtype):
    """No table: sequence i has page i, and the pages behind the last sequence stay as they were.  The same bits as with that table."""
    from reproducing_fastmax_results_b200 import _lib as L

    gen = torch.Generator(device="cuda").manual_seed(d)
    cache = states(batch + 2, heads, d, order, gen, layers=2)
    before, tabled = cache.clone(), cache.clone()
    q, k, v = (torch.randn(batch, heads, d, device="cuda", generator=gen).to(dtype) for _ in range(3))
    o, g = L.decode_step_paged(q, k, v, cache[:, 1], None, 0.1, *A, order)
    ref, gref = L.decode_step_paged(q, k, v, tabled[:, 1], i32(range(batch)), 0.1, *A, order)
    assert torch.equal(o, ref) and torch.equal(g, gref) and torch.equal(cache, tabled)
    assert torch.equal(cache[:, 0], before[:, 0]) and torch.equal(cache[batch:], before[batch:])
    for i in (0, batch - 1):
        j = heads - 1
        old, kk, vv = host(before[i, 1, j]), host(k[i, j])[None], host(v[i, j])[None]
        oref, _, size, _ = so.tree(host(q[i, j])[None], kk, vv, old, [-1], order, A, 0.1)
        rounding = 2.0 ** (-8 if dtype == torch.bfloat16 else -24)
        assert (np.abs(host(o[i, j])[None] - oref) <= rounding * np.abs(oref) + so.SUMS_F32 * size).all()


@pytest.mark.parametrize("heads", [2, 48])   # one launch, two
@pytest.mark.parametrize("which", [0, 1, 2])
def test_a_step_may_write_into_its_inputs(which, heads):
    """The output in the place of q, k or v, views of one projection: what it gives elsewhere."""
    from reproducing_fastmax_results_b200 import FastmaxCache

    gen = torch.Generator(device="cuda").manual_seed(heads)
    qkv = torch.randn(6, 3, heads, 1, 64, device="cuda", generator=gen).bfloat16()
    start = states(6, heads, 64, 2, gen)
    results = []
    for place in (False, True):
        cache = FastmaxCache(6, heads, 64, temperature=10.0)
        assert cache.begin(range(5)).item() == 0
        cache.state[:, 0] = start
        x = qkv.clone()
        out = x[:, which] if place else qkv[:, which].clone()   # the absent place's rows stay as they are
        for _ in range(2):
            x.copy_(qkv)
            o = cache.step(x[:, 0], x[:, 1], x[:, 2], out=out)
            others = [i for i in range(3) if i != which]
            assert torch.equal(x[:, others], qkv[:, others]) and torch.equal(x[5], qkv[5])
        results.append((o.clone(), cache.state.clone()))
    assert torch.equal(results[0][0], results[1][0]) and torch.equal(results[0][1], results[1][1])


# ---- pages -----------------------------------------------------------------------------------------------------------------
def arrange_and_compare(table, sources, pages, floats, seed):
    from reproducing_fastmax_results_b200.attention import _ext

    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = torch.randn(pages, floats, device="cuda", generator=gen)
    before, t = state.clone(), i32(table)
    unserved = _ext().cache_arrange(state, t, i32(sources))
    new, moves, missing = so.arranged(table, sources, pages)
    assert t.tolist() == new and unserved.tolist() == [missing]
    for source, page in moves:
        before[page] = before[source] if source >= 0 else 0.0
    assert torch.equal(state, before)


@pytest.mark.parametrize("floats", [4, 20, 4096, 4100, 16384, 100004])
def test_arranging_small_caches(floats):
    for seed, (table, sources, pages) in enumerate([
            ([0], [0], 1), ([-1], [-2], 1), ([0], [-1], 1), ([0], [-2], 1), ([-1], [0], 1), ([0, 1], [1, 0], 2), ([0, 1], [1, 1], 2),
            ([2, 0, 1], [2, 2, 2], 3), ([3, -1, 0, 2], [2, 0, 2, -1], 4), ([0, 1, 2], [-2, 0, 0], 3), ([0, 1, -1], [1, 1, 1], 2),
            ([0, 1], [5, -3], 3), ([0, 7], [1, 0], 3), ([-5, 1], [0, 1], 2)]):
        arrange_and_compare(table, sources, pages, floats, seed)


@pytest.mark.parametrize("places,pages", [(5, 9), (64, 64), (200, 150), (1024, 1030), (1025, 1024), (3000, 5000), (32768, 32768)])
def test_arranging_large_caches(places, pages):
    rng = np.random.default_rng(places)
    for seed in range(2):
        table = np.full(places, -1)
        held = rng.permutation(places)[: min(places, pages) * 3 // 4]
        table[held] = rng.permutation(pages)[: len(held)]
        sources = np.where(rng.random(places) < 0.5, np.arange(places), rng.integers(-2, places, places))
        arrange_and_compare(table.tolist(), sources.tolist(), pages, 36, seed)


@pytest.mark.parametrize("places,pages,live", [(1, 1, 0), (1, 1, 1), (4, 7, 3), (50, 50, 50), (50, 60, 17), (1500, 2049, 1100), (32768, 32768, 20000)])
def test_compacting(places, pages, live):
    from reproducing_fastmax_results_b200.attention import _ext

    rng = np.random.default_rng(pages)
    table = np.full(places, -1)
    table[rng.permutation(places)[:live]] = rng.permutation(pages)[:live]
    if places > live:
        table[np.flatnonzero(table < 0)[0]] = pages   # no page
    state = torch.randn(pages, 44, device="cuda", generator=torch.Generator(device="cuda").manual_seed(live))
    before, t = state.clone(), i32(table)
    count = _ext().cache_compact(state, t)
    new, moves, n = so.compacted(table.tolist(), pages)
    assert t.tolist() == new and count.tolist() == [n] == [live]
    for source, page in moves:
        before[page] = before[source]
    assert torch.equal(state, before)
    again = t.clone()
    assert _ext().cache_compact(state, t).tolist() == [live] and torch.equal(t, again) and torch.equal(state, before)


def test_copying_pages():
    from reproducing_fastmax_results_b200.attention import _ext

    gen = torch.Generator(device="cuda").manual_seed(1)
    cache = torch.randn(6, 3, 2, 5000, device="cuda", generator=gen)
    layer = cache[:, 1]
    dense = torch.full((4, 2, 5000), 2.0, device="cuda")
    _ext().pages_copy(layer, dense, i32([5, -1, 0, 6]), None, 4)
    assert torch.equal(dense[0], layer[5]) and torch.equal(dense[2], layer[0]) and (dense[[1, 3]] == 2.0).all()
    before = cache.clone()
    _ext().pages_copy(dense, layer, None, i32([3, 6, -1, 2]), 4)
    before[3, 1], before[2, 1] = dense[0], dense[3]
    assert torch.equal(cache, before)
    _ext().pages_copy(layer, dense, None, None, 4)
    assert torch.equal(dense, layer[:4])
    _ext().pages_copy(layer, dense, i32([]), None, 0)
    one = torch.zeros(1, 2, 5000, device="cuda")
    _ext().pages_copy(layer, one, i32([4]), i32([0]), 1)
    assert torch.equal(one[0], layer[4])


def test_pages_beyond_32_bits_of_offset():
    """The last page of a cache whose floats do not count in 32 bits (17 GB), by every operator."""
    from reproducing_fastmax_results_b200 import _lib as L
    from reproducing_fastmax_results_b200.cache import FastmaxCache

    h, d = 8, 64
    pages = 2 ** 32 // (h * 2369 * 68) + 2
    cache = FastmaxCache(2, h, d, pages=pages, temperature=10.0)
    assert cache.state.numel() > 2 ** 32
    gen = torch.Generator(device="cuda").manual_seed(0)
    some = states(1, h, d, 2, gen)
    cache.state[pages - 1, 0] = some[0]
    cache.table.copy_(i32([pages - 1, -1]))
    q, k, v = (torch.randn(2, h, 5, d, device="cuda", generator=gen).bfloat16() for _ in range(3))
    dense = some.clone()
    o = cache.verify(q, k, v)
    ref, _ = L.tree_attention(q[:1], k[:1], v[:1], dense, 0.1)
    assert orc.max_norm_err(host(o[0]), host(ref[0])) < 2.0 ** -7 and (o[1] == 0).all()
    cache.accept(k, v, [2, 2])
    L.tree_accept(k[:1], v[:1], dense, i32([2]))
    assert torch.equal(cache.state[pages - 1, 0], dense[0])
    cache.step(q[:, :, 0], k[:, :, 0], v[:, :, 0])
    L.decode_step(q[:1, :, 0], k[:1, :, 0], v[:1, :, 0], dense, 0.1)
    assert orc.max_norm_err(host(cache.state[pages - 1, 0]), host(dense[0])) < 2.0 ** -22
    last = cache.state[pages - 1].clone()
    assert cache.compact().item() == 1 and cache.table.tolist() == [0, -1]
    assert torch.equal(cache.state[0], last)
    cache.table.copy_(i32([-1, pages - 1]))
    assert cache.arrange([1, 1]).item() == 0 and cache.table.tolist() == [pages - 1, 0]
    assert torch.equal(cache.state[0], last)


# ---- together ----------------------------------------------------------------------------------------------------------------
def causal(q, k, v, inv_t, order=2):
    return orc.fastmax_naive(host(q), host(k), host(v), True, orc.Poly(1.0, 1.0, 0.5, inv_t, order))[0]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d,order", [(64, 2), (32, 1)])
def test_serving(d, order, dtype):
    """Two layers, five places: prompts, drafted trees, accepted paths, steps, forks, endings, a new sequence in a freed place, compaction.  At
    the end every sequence's output is the causal operator's over all of its tokens."""
    from reproducing_fastmax_results_b200 import FastmaxCache

    places, layers, h, inv_t = 5, 2, 3, 0.1
    gen = torch.Generator(device="cuda").manual_seed(d)
    rng = np.random.default_rng(d)
    cache = FastmaxCache(places, h, d, p=order, temperature=1 / inv_t, layers=layers, pages=6)
    tokens = {}   # (place, layer) -> k, v so far
    tol = 1e-4 if dtype == torch.float32 else 2e-2   # the operator's own tolerances

    def draft(n, count=places):
        return [torch.randn(count, h, n, d, device="cuda", generator=gen).to(dtype) for _ in range(3)]

    def expect(place, layer, q, k, v):
        """the last row of the causal operator over the place's tokens and these"""
        kk, vv = (torch.cat([a, b], 1) for a, b in zip(tokens[place, layer], (k, v)))
        return orc.fastmax_naive(host(q), host(kk), host(vv), False, orc.Poly(1.0, 1.0, 0.5, inv_t, order))[0]

    def prompt(which, n, continues=False):
        for layer in range(layers):
            q, k, v = draft(n, len(which))
            o = cache.prefill(q, k, v, which, layer=layer, continues=continues)
            for i, place in enumerate(which):
                old = tokens[place, layer] if continues else (k[i][:, :0], v[i][:, :0])
                tokens[place, layer] = [torch.cat([a, b], 1) for a, b in zip(old, (k[i], v[i]))]
                kk, vv = tokens[place, layer]
                ref = orc.fastmax_naive(host(q[i]), host(kk), host(vv), True, orc.Poly(1.0, 1.0, 0.5, inv_t, order))[0]
                assert orc.max_norm_err(host(o[i]), ref) < tol

    def check_step():
        for layer in range(layers):
            q, k, v = (t[:, :, 0] for t in draft(1))
            o = cache.step(q, k, v, layer=layer)
            for place in range(places):
                if (place, layer) not in tokens:
                    assert (o[place] == 0).all()
                    continue
                ref = expect(place, layer, q[place][:, None], k[place][:, None], v[place][:, None])
                assert orc.max_norm_err(host(o[place][:, None]), ref) < tol
                tokens[place, layer] = [torch.cat([a, b], 1) for a, b in zip(tokens[place, layer], (k[place][:, None], v[place][:, None]))]

    def speculate(n):
        parents = random_parents(places, n, rng)
        lengths = rng.integers(1, n + 1, places)
        last = np.array([rng.integers(-1, m) for m in lengths])
        for layer in range(layers):
            q, k, v = draft(n)
            o = cache.verify(q, k, v, parents=parents, lengths=i32(lengths), layer=layer)
            cache.accept(k, v, i32(last), parents=i32(parents), layer=layer)
            for place in range(places):
                if (place, layer) not in tokens:
                    assert (o[place] == 0).all()
                    continue
                for i in (0, lengths[place] // 2, lengths[place] - 1):
                    nodes = so.path(parents[place], i)
                    ref = expect(place, layer, q[place][:, i: i + 1], k[place][:, nodes], v[place][:, nodes])
                    assert orc.max_norm_err(host(o[place][:, i: i + 1]), ref) < tol
                nodes = so.path(parents[place], last[place])
                tokens[place, layer] = [torch.cat([a, b[:, nodes]], 1) for a, b in zip(tokens[place, layer], (k[place], v[place]))]

    assert cache.begin([0, 1, 2]).item() == 0
    prompt([0, 1, 2], 37)
    check_step()
    speculate(9)
    # place 2 goes on in 2, 3 and 4; place 1 ends
    assert cache.arrange(torch.tensor([0, -1, 2, 2, 2], device="cuda")).item() == 0
    for layer in range(layers):
        tokens.pop((1, layer))
        tokens[3, layer] = tokens[4, layer] = tokens[2, layer]
    check_step()
    assert cache.begin([1]).item() == 0
    prompt([1], 5)
    speculate(17)
    # beams change places
    assert cache.arrange([4, 4, 1, 0, -1]).item() == 0
    old = dict(tokens)
    for layer in range(layers):
        for place, source in enumerate([4, 4, 1, 0]):
            tokens[place, layer] = old[source, layer]
        tokens.pop((4, layer))
    speculate(4)
    cache.end([0])
    for layer in range(layers):
        tokens.pop((0, layer))
    assert cache.compact().item() == 3
    assert sorted(cache.table.tolist()) == [-1, -1, 0, 1, 2]
    prompt([3, 1], 6, continues=True)
    check_step()
    for (place, layer), (k, v) in tokens.items():
        got = host(cache.state[int(cache.table[place]), layer])
        for j in range(h):
            ref, _ = so.grown(np.zeros((got.shape[1], d + 4)), host(k[j]), host(v[j]), order)
            assert orc.max_norm_err(got[j, :, : d + 1], ref) < (1e-5 if dtype == torch.float32 else 5e-3)


def test_prompts_of_mixed_types_and_devices_are_refused():
    """Before anything is launched: the states stay as they are, and the next prompt is right.  No places: no prompts."""
    from reproducing_fastmax_results_b200 import FastmaxCache

    gen = torch.Generator(device="cuda").manual_seed(9)
    x = [torch.randn(2, 2, 9, 32, device="cuda", generator=gen) for _ in range(3)]
    cache = FastmaxCache(3, 2, 32, temperature=10.0)
    assert cache.begin([0, 1, 2]).item() == 0
    cache.state[:, 0] = states(3, 2, 32, 2, gen)
    before = cache.state.clone()
    for i in range(3):
        for other in (x[i].bfloat16(), x[i].cpu(), x[i].transpose(2, 3).contiguous().transpose(2, 3)):
            bad = [other if j == i else t for j, t in enumerate(x)]
            for continues in (False, True):
                with pytest.raises(RuntimeError):
                    cache.prefill(*bad, [0, 2], continues=continues)
    none = [t[:0] for t in x]
    assert tuple(cache.prefill(*none, []).shape) == (0, 2, 9, 32)
    assert torch.equal(cache.state, before)
    o = cache.prefill(*x, [0, 2])
    assert orc.max_norm_err(host(o), causal(*x, 0.1)) < 1e-4
    assert torch.equal(cache.state[1], before[1]) and not torch.equal(cache.state[0], before[0])


def test_a_step_into_memory_of_another_device_is_refused():
    """Before the launch, with a dense state and on pages."""
    from reproducing_fastmax_results_b200 import FastmaxCache, FastmaxDecoder

    x = [torch.ones(2, 2, 16, device="cuda") for _ in range(3)]
    dec, cache = FastmaxDecoder(2, 2, 16), FastmaxCache(2, 2, 16)
    cache.begin([0, 1])
    for serve in (dec, cache):
        with pytest.raises(RuntimeError, match="device"):
            serve.step(*x, out=torch.zeros(2, 2, 16))
        assert (serve.state == 0).all()
    assert dec.tokens_seen == 0
    assert torch.equal(dec.step(*x), cache.step(*x))


def test_numbers_of_any_width_mean_what_they_say():
    """64-bit numbers on the device, among them some that would be others in 32 bits; empty lists of places."""
    from reproducing_fastmax_results_b200 import FastmaxCache

    gen = torch.Generator(device="cuda").manual_seed(3)
    x = [torch.randn(3, 2, 4, 16, device="cuda", generator=gen) for _ in range(3)]
    cache = FastmaxCache(3, 2, 16, temperature=10.0)
    assert cache.begin([]).item() == 0 and cache.begin([0, 1, 2]).item() == 0
    cache.end([])
    cache.state[:, 0] = states(3, 2, 16, 2, gen)
    big = 1 << 32
    parents = torch.tensor([[-1, 0, 1, big], [-1, -1, big + 1, 0], [-1, 0, -big, 2]], device="cuda")
    lengths = torch.tensor([4, 2, big], device="cuda")
    o = cache.verify(*x, parents=parents, lengths=lengths)
    ref = cache.verify(*x, parents=[[-1, 0, 1, -1], [-1, -1, -1, 0], [-1, 0, -1, 2]], lengths=[4, 2, 4])
    assert torch.equal(o, ref) and float(o.abs().sum()) > 0
    before = cache.state.clone()
    cache.accept(x[1], x[2], torch.tensor([big, -big, big + 3], device="cuda"))
    assert torch.equal(cache.state, before)
    assert cache.arrange(torch.tensor([big, 1, -big - 2], device="cuda")).item() == 2
    assert cache.table.tolist() == [-1, 1, -1]


@pytest.mark.parametrize("dtype", [torch.uint8, torch.int8, torch.int16, torch.int64])
def test_device_numbers_of_narrow_types_are_what_they_say(dtype):
    """lengths, last, parents and sources in types that do not hold the bounds they are compared with."""
    from reproducing_fastmax_results_b200 import FastmaxCache

    def narrow(x):
        return torch.tensor(x, dtype=dtype, device="cuda")

    signed = dtype != torch.uint8
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = [torch.randn(200, 1, 4, 16, device="cuda", generator=gen) for _ in range(3)]
    start = states(200, 1, 16, 2, gen)
    caches = [FastmaxCache(200, 1, 16, temperature=10.0) for _ in range(2)]
    for cache in caches:
        assert cache.begin(range(200)).item() == 0
        cache.state[:, 0] = start
    lengths, last = [i % 5 for i in range(200)], [i % 4 for i in range(200)]
    parents = [[-1 if signed else 0, 0, 1, 1 - i % 2] for i in range(200)]
    roots = [[-1, *row[1:]] for row in parents]   # an unsigned 0 at the first node is no node before it: a root
    sources = [min(199 - i, 127) for i in range(200)]   # int8 holds them
    o = caches[0].verify(*x, parents=narrow(parents), lengths=narrow(lengths))
    ref = caches[1].verify(*x, parents=i32(roots), lengths=i32(lengths))
    assert torch.equal(o, ref) and (o[4] != 0).any() and (o[5] == 0).all()
    caches[0].accept(x[1], x[2], narrow(last), parents=narrow(parents))
    caches[1].accept(x[1], x[2], i32(last), parents=i32(roots))
    assert torch.equal(caches[0].state, caches[1].state) and not torch.equal(caches[0].state[:, 0], start)
    assert caches[0].arrange(narrow(sources)).tolist() == caches[1].arrange(i32(sources)).tolist() == [0]
    assert torch.equal(caches[0].table, caches[1].table) and torch.equal(caches[0].state, caches[1].state)


def test_the_decoder_checks_drafts():
    """FastmaxDecoder: prompt, a tree, the accepted path, the next step."""
    from reproducing_fastmax_results_b200 import FastmaxDecoder

    b, h, d, n = 3, 4, 64, 6
    gen = torch.Generator(device="cuda").manual_seed(8)
    q, k, v = (torch.randn(b, h, 30 + n, d, device="cuda", generator=gen) for _ in range(3))
    dec = FastmaxDecoder(b, h, d, temperature=10.0)
    dec.prefill(q[:, :, :30], k[:, :, :30], v[:, :, :30])
    drafts = [t[:, :, 30:].contiguous() for t in (q, k, v)]
    o = dec.verify(*drafts)   # a chain: rows of the causal operator
    assert orc.max_norm_err(host(o), causal(q, k, v, 0.1)[:, :, 30:]) < 1e-4
    dec.accept(drafts[1], drafts[2], [n - 1, 1, -1])
    assert dec.tokens_seen == 30 + n
    x = [torch.randn(b, h, d, device="cuda", generator=gen) for _ in range(3)]
    o = dec.step(*x)
    for i, kept in enumerate((30 + n, 32, 30)):
        rows = [torch.cat([t[i: i + 1, :, :kept], y[i: i + 1, :, None]], 2) for t, y in zip((q, k, v), x)]
        assert orc.max_norm_err(host(o[i: i + 1, :, None]), causal(*rows, 0.1)[:, :, -1:]) < 1e-4
    with pytest.raises(RuntimeError):
        dec.verify(*(torch.zeros(b, h, 65, d, device="cuda") for _ in range(3)))
    with pytest.raises(RuntimeError):
        dec.verify(drafts[0], drafts[1], drafts[2].bfloat16())
    with pytest.raises(RuntimeError):
        dec.verify(drafts[0].half(), drafts[1].half(), drafts[2].half())


def test_serving_calls_replay_from_graphs():
    """A server's step, captured: verify, accept, fork and compact with their inputs in place; two graphs that share the cache replay in turn."""
    from reproducing_fastmax_results_b200 import FastmaxCache

    places, h, d, n = 4, 8, 64, 7

    def setup():
        gen = torch.Generator(device="cuda").manual_seed(12)
        cache = FastmaxCache(places, h, d, temperature=10.0, pages=5)
        cache.begin(range(places))
        cache.state[:, 0] = states(5, h, d, 2, gen)
        inputs = [torch.randn(places, h, n, d, device="cuda", generator=gen).bfloat16() for _ in range(3)]
        return cache, inputs, i32([3, -1, 6, 0]), i32([1, 1, -1, 3]), torch.zeros_like(inputs[0])

    def tree(cache, x, last, sources, out):
        cache.verify(*x, out=out)
        cache.accept(x[1], x[2], last)

    def pages(cache, x, last, sources, out):
        cache.arrange(sources)
        cache.compact()
        cache.step(*(t[:, :, 0] for t in x), out=out[:, :, 1])

    eager, captured = setup(), setup()
    for _ in range(3):
        tree(*eager)
        pages(*eager)
    warm = setup()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        tree(*warm)
        pages(*warm)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = []
    for call in (tree, pages):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call(*captured)
        graphs.append(graph)
    for _ in range(3):
        for graph in graphs:
            graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(eager[0].table, captured[0].table) and torch.equal(eager[0].state, captured[0].state) and torch.equal(eager[4], captured[4])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_captured_calls_of_a_decoder_serve_the_next_prompt(dtype):
    """The state keeps its memory: a step, a tree and its path, captured once, go on from whatever prompt was read last."""
    from reproducing_fastmax_results_b200 import FastmaxDecoder

    gen = torch.Generator(device="cuda").manual_seed(6)
    prompts = [[torch.randn(2, 3, n, 64, device="cuda", generator=gen).to(dtype) for _ in range(3)] for n in (9, 30, 4)]
    x = [torch.randn(2, 3, 5, 64, device="cuda", generator=gen).to(dtype) for _ in range(3)]
    last = i32([3, -1])

    def serve(dec, tree, token):
        dec.verify(*x, out=tree)
        dec.accept(x[1], x[2], last)
        dec.step(*(t[:, :, 0] for t in x), out=token)

    def read(dec, which):
        dec.reset()
        dec.prefill(*prompts[which])
        if which == 1:
            dec.prefill(*prompts[2])   # goes on

    eager, captured = FastmaxDecoder(2, 3, 64, temperature=10.0), FastmaxDecoder(2, 3, 64, temperature=10.0)
    outs = [[torch.zeros_like(x[0]), torch.zeros_like(x[0][:, :, 0])] for _ in range(2)]
    read(eager, 0)
    serve(eager, *outs[0])
    memory = captured.state.data_ptr()
    read(captured, 0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        serve(captured, *outs[1])
    for which in (0, 1, 2):
        read(eager, which)
        serve(eager, *outs[0])
        read(captured, which)
        assert captured.state.data_ptr() == memory
        graph.replay()
        assert torch.equal(eager.state, captured.state)
        assert all(torch.equal(a, b) and float(a.float().abs().sum()) > 0 for a, b in zip(*outs))


def test_numbers_on_the_host_are_refused_during_a_capture():
    """The refusal comes before the copy: the capture goes on without the call, and the cache stays as it was."""
    from reproducing_fastmax_results_b200 import FastmaxCache

    gen = torch.Generator(device="cuda").manual_seed(5)
    cache = FastmaxCache(3, 2, 16, temperature=10.0)
    assert cache.begin([0, 1, 2]).item() == 0
    cache.state[:, 0] = states(3, 2, 16, 2, gen)
    x = [torch.randn(3, 2, 4, 16, device="cuda", generator=gen) for _ in range(3)]
    parents, lengths, last = [[-1, 0, 0, 1]] * 3, [4, 2, 0], [3, -1, 0]
    ref = cache.verify(*x, parents=parents, lengths=lengths)
    before, table = cache.state.clone(), cache.table.clone()
    on_device = i32(parents), i32(lengths), i32(last)
    out = torch.zeros_like(x[0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for call in (lambda: cache.begin([1]), lambda: cache.end([0]), lambda: cache.arrange([0, 0, 1]), lambda: cache.verify(*x, parents=parents),
                     lambda: cache.verify(*x, lengths=torch.tensor(lengths)), lambda: cache.accept(x[1], x[2], last), lambda: cache.prefill(*x, [0, 1, 2])):
            with pytest.raises(RuntimeError, match="graph"):
                call()
        cache.verify(*x, parents=on_device[0], lengths=on_device[1], out=out)
    assert torch.equal(cache.state, before) and torch.equal(cache.table, table)
    graph.replay()
    assert torch.equal(out, ref) and torch.equal(cache.state, before)


def test_calls_on_two_streams_keep_apart():
    from reproducing_fastmax_results_b200 import FastmaxCache

    gen = torch.Generator(device="cuda").manual_seed(4)
    inputs = [torch.randn(6, 8, 20, 64, device="cuda", generator=gen).bfloat16() for _ in range(3)]
    start = states(6, 8, 64, 2, gen)
    last, sources = i32([4, 19, -1, 0, 7, 11]), i32([0, 0, 2, 2, 4, -1])

    def one():
        cache = FastmaxCache(6, 8, 64, temperature=10.0)
        cache.begin(range(6))
        cache.state[:, 0] = start
        return cache

    def serve(cache):
        outs = []
        for _ in range(4):
            outs.append(cache.verify(*inputs))
            cache.accept(inputs[1], inputs[2], last)
            cache.arrange(sources)
            outs.append(cache.step(*(t[:, :, 1] for t in inputs)))
        return outs + [cache.state]

    ref = serve(one())
    caches = [one() for _ in range(3)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in caches]
    got = []
    for cache, stream in zip(caches, streams):
        with torch.cuda.stream(stream):
            got.append(serve(cache))
    torch.cuda.synchronize()
    for outs in got:
        assert all(torch.equal(a, b) for a, b in zip(outs, ref))


def test_a_tree_that_gives_up_is_reported_once_and_the_context_stays_usable():
    """The waits of the tree's kernel: a block whose copy never comes ends by itself after about a millisecond, waits for its other copy, and counts
    as one block at its wait site.  No operator is disturbed."""
    from reproducing_fastmax_results_b200 import _lib as L

    lib = L.load()
    torch.cuda.synchronize()
    assert lib.fastmax_check_status() == 0 and L.wait_histogram() == {}
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.fastmax_debug_tree_wait_selftest(stream) == 0
    torch.cuda.synchronize()
    assert lib.fastmax_check_status() == 5 and lib.fastmax_check_status() == 0   # FASTMAX_ERR_DEVICE_TIMEOUT, once
    assert L.wait_histogram() == {210: 1} and L.wait_histogram() == {}
    # beside another kernel's
    assert lib.fastmax_debug_wait_selftest(stream) == 0 and lib.fastmax_debug_tree_wait_selftest(stream) == 0
    with pytest.raises(L.FastmaxError):
        L.check_status()
    assert lib.fastmax_check_status() == 0
    assert L.wait_histogram() == {99: 1, 210: 1} and L.wait_histogram() == {}
    gen = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (torch.randn(1, 2, 20, 64, device="cuda", generator=gen) for _ in range(3))
    state = states(1, 2, 64, 2, gen)
    o, g = L.tree_attention(q, k, v, state, 0.1, *A, 2)
    check_tree(o, g, q, k, v, state, None, None, None, 2, 0.1)
    L.check_status()
    assert L.wait_histogram() == {}


def test_calls_back_to_back_see_each_other():
    """A kernel starts while the one before it ends: a chain of dependent calls gives the same as with a wait behind each."""
    from reproducing_fastmax_results_b200 import FastmaxCache

    def serve(wait):
        gen = torch.Generator(device="cuda").manual_seed(6)
        cache = FastmaxCache(8, 4, 32, temperature=10.0, pages=9)
        cache.begin(range(8))
        x = [torch.randn(8, 4, 12, 32, device="cuda", generator=gen) for _ in range(3)]
        outs = []
        for i in range(12):
            for call in (lambda: cache.accept(x[1], x[2], i32([i % 12] * 8)), lambda: outs.append(cache.verify(*x)),
                         lambda: cache.arrange([(3 * j + i) % 8 for j in range(8)] if i % 3 else [0, 0, 1, 1, 2, 2, -2, -1]), cache.compact,
                         lambda: outs.append(cache.step(*(t[:, :, 0] for t in x)))):
                call()
                if wait:
                    torch.cuda.synchronize()
        return outs + [cache.state.clone(), cache.table.clone()]

    assert all(torch.equal(a, b) for a, b in zip(serve(False), serve(True)))
