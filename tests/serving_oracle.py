"""The serving operators in 64 bits on the CPU, written from their definitions: attention of a tree over a moment state, taking a path into
it, and who gets which page.  Error bounds beside them."""
import numpy as np


def features(x, order):
    """(n, d) -> (n, rows): the features of a state's rows, in their order, without weights."""
    x = np.asarray(x, np.float64)
    n, d = x.shape
    parts = []
    if order == 2:
        for a in range(0, d, 8):
            for b in range(a, d, 8):
                parts.append((x[:, a:a + 8, None] * x[:, None, b:b + 8]).reshape(n, 64))
    return np.concatenate(parts + [x, np.ones((n, 1))], 1)


def weights(d, order, a, inv_t):
    pairs = []
    if order == 2:
        for m in range(0, d, 8):
            for n in range(m, d, 8):
                pairs.append(np.full(64, a[2] * inv_t * inv_t * (1 if m == n else 2)))
    return np.concatenate(pairs + [np.full(d, a[1] * inv_t), [a[0]]])


def path(parents, node):
    """Nodes from the root down to `node`."""
    out = []
    while node >= 0:
        out.append(node)
        up = int(parents[node])
        node = up if 0 <= up < node else -1
    return out[::-1]


def tree(q, k, v, state, parents, order, a, inv_t):
    """One head.  q, k, v (n, d), state (rows, d + 4).  Returns o (n, d), g (n,) and what the errors scale with: the sums of the terms'
    magnitudes over |g|, for o and relative for g."""
    q, k, v, state = (np.asarray(x, np.float64) for x in (q, k, v, state))
    n, d = q.shape
    s = state[:, : d + 1]
    w = features(q, order) * weights(d, order, a, inv_t)
    sums, size = w @ s, np.abs(w) @ np.abs(s)
    v1 = np.concatenate([v, np.ones((n, 1))], 1)
    for i in range(n):
        for j in path(parents, i):
            x = (q[i] @ k[j]) * inv_t
            ax = (np.abs(q[i]) @ np.abs(k[j])) * inv_t
            f = a[0] + a[1] * x + (a[2] * x * x if order == 2 else 0.0)
            af = abs(a[0]) + abs(a[1]) * ax + (abs(a[2]) * ax * ax if order == 2 else 0.0)
            sums[i] += f * v1[j]
            size[i] += af * np.abs(v1[j])
    g = sums[:, d]
    o = sums[:, :d] / g[:, None]
    return o, g, (size[:, :d] + np.abs(o) * size[:, d:]) / np.abs(g)[:, None], size[:, d]


# Roundings behind one another in an output of the attention: a product of pieces adds up to six products per 16 terms, every block
# of the head dim up to 32 of them, then the rest of a block's warps, a cluster's blocks and the tree's nodes (at most 64).  The tensor cores'
# sums may cut off where they do not round: a whole step, 2^-23.  Together less than 256 half steps of 2^-24, and as many again are left
# for f itself (three roundings) and the division.
SUMS_F32 = 512 * 2.0 ** -24
# bfloat16 tensors: the state enters as two pieces, each rounded to 2^-8 of what is left: 2^-16 of each term
SUMS_BF16 = SUMS_F32 + 2.0 ** -16


def attention_tolerance(o, size, bf16):
    out = np.abs(o) * (2.0 ** -8 if bf16 else 2.0 ** -24)
    return out + (SUMS_BF16 if bf16 else SUMS_F32) * size


def grown(state, k, v, order):
    """One head: state (rows, d + 4) and keys and values (t, d) that are added.  Returns the new sums and the sizes of their terms."""
    d = k.shape[1]
    v1 = np.concatenate([np.asarray(v, np.float64), np.ones((len(v), 1))], 1)
    phi = features(k, order)
    state = np.asarray(state, np.float64)[:, : d + 1]
    return state + phi.T @ v1, np.abs(state) + np.abs(phi).T @ np.abs(v1)


def grown_tolerance(size, tokens):
    # a feature, its product with v and the sum: three roundings a token
    return 3 * tokens * 2.0 ** -24 * size


def arranged(table, sources, pages):
    """(table afterwards, [(source page or -1, destination page)], places that were not served)."""
    new, kept, later, unserved = [-1] * len(table), set(), [], 0
    for i, j in enumerate(sources):
        if j == -2:
            later.append((i, -1))
        elif 0 <= j < len(table):
            page = table[j] if 0 <= table[j] < pages else -1
            if page >= 0 and page not in kept:
                kept.add(page)
                new[i] = page
            elif page >= 0:
                later.append((i, page))
        elif j != -1:
            unserved += 1
    free = [p for p in range(pages) if p not in kept]
    moves = []
    for (i, source), page in zip(later, free):
        new[i] = page
        moves.append((source, page))
    return new, moves, unserved + max(0, len(later) - len(free))


def compacted(table, pages):
    live = sorted({p for p in table if 0 <= p < pages})
    movers = [p for p in live if p >= len(live)]
    holes = [p for p in range(len(live)) if p not in live]
    goes = dict(zip(movers, holes))
    return [goes.get(p, p) if 0 <= p < pages else -1 for p in table], list(zip(movers, holes)), len(live)
