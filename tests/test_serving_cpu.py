"""The serving entry points without a GPU: what they refuse before any launch, their Python checks, and the oracle of their tests."""
import ctypes as C

import numpy as np
import pytest
import torch

import serving_oracle as so
from oracle import fastmax_oracle as orc
from reproducing_fastmax_results_b200 import _lib as L
from reproducing_fastmax_results_b200.decoding import per_sequence, tree_parents

PTR = 1 << 20   # looks like an aligned address; no refused call reads it


def problem(**fields):
    pb = L.Problem(2, 3, 5, 5, 32, 2, 1, L.FASTMAX_F32, 1.0, 1.0, 0.5, 1.0, 0, 0)
    for name, value in fields.items():
        setattr(pb, name, value)
    return pb


def cache(**fields):
    c = L.Pages(PTR, 3 * 673 * 36, 2, 0, PTR)
    for name, value in fields.items():
        setattr(c, name, value)
    return c


def calls(pb, c, missing=None):
    """The three entry points that read pages, with argument `missing` left out: (name, status)."""
    lib = L.load()
    t = L.Tensor(PTR, 3 * 5 * 32, 5 * 32, 32)
    one = L.PagedDecodeArgs()
    one.q = one.k = one.v = one.o = t
    one.cache = c
    tree = L.TreeArgs()
    tree.q = tree.k = tree.v = tree.o = t
    tree.cache = c
    accept = L.AcceptArgs()
    accept.k = accept.v = t
    accept.cache = c
    accept.last = PTR
    for args in (one, tree, accept):
        if missing and hasattr(args, missing):
            setattr(args, missing, L.Tensor() if isinstance(getattr(args, missing), L.Tensor) else None)
    single = L.Problem.from_buffer_copy(pb)
    if pb.nq == pb.nk == 5:
        single.nq = single.nk = 1
    yield "step", lib.fastmax_decode_step_paged(C.byref(single), C.byref(one), PTR, 1 << 40, None)
    yield "verify", lib.fastmax_tree_attention(C.byref(pb), C.byref(tree), None)
    yield "accept", lib.fastmax_tree_accept(C.byref(pb), C.byref(accept), None)


@pytest.mark.parametrize("fields,status", [
    ({"batch": 0}, 1), ({"heads": -1}, 1), ({"dtype": 5}, 1), ({"d": 48}, 2), ({"order": 3}, 2), ({"batch": 30000}, 2), ({"nq": 4}, 2), ({"nk": 6}, 2)])
def test_bad_problems_are_refused(fields, status):
    for name, got in calls(problem(**fields), cache()):
        assert got == status, name


def test_too_many_nodes_and_none_are_refused():
    for nodes, status in ((65, 2), (0, 1), (-3, 1)):
        got = dict(calls(problem(nq=nodes, nk=nodes), cache()))
        assert got["verify"] == got["accept"] == status and got["step"] == 2


@pytest.mark.parametrize("fields,status", [
    ({"state": None}, 1), ({"pages": 0}, 1), ({"pages": 1, "table": None}, 1), ({"page_stride": 3 * 673 * 36 - 4}, 1), ({"page_stride": 3 * 673 * 36 + 2}, 6),
    ({"state": PTR + 8}, 6)])
def test_bad_pages_are_refused(fields, status):
    for name, got in calls(problem(), cache(**fields)):
        assert got == status, name


@pytest.mark.parametrize("missing,by", [("k", {"step", "verify", "accept"}), ("v", {"step", "verify", "accept"}), ("q", {"step", "verify"}),
                                        ("o", {"step", "verify"}), ("last", {"accept"})])
def test_missing_tensors_are_refused(missing, by):
    # the others would be launched: a misaligned state stops them before that
    for name, got in calls(problem(), cache(state=PTR + 8), missing):
        assert got == (1 if name in by else 6), name


def test_a_step_without_its_workspace_is_refused():
    lib = L.load()
    assert lib.fastmax_decode_step_workspace(C.byref(problem())) == lib.fastmax_decode_step_workspace(None) == 0
    many = problem(batch=60, nq=1, nk=1)   # 180 heads
    need = lib.fastmax_decode_step_workspace(C.byref(many))
    assert need >= 180 * 3 * 36 * 4
    args = L.PagedDecodeArgs()
    args.q = args.k = args.v = args.o = L.Tensor(PTR, 96, 32, 0)
    args.cache = cache(pages=60, state=PTR + 8)
    for ws, nbytes, status in ((None, need, 3), (PTR + 8, need, 3), (PTR, need - 1, 3), (PTR, need, 6)):
        assert lib.fastmax_decode_step_paged(C.byref(many), C.byref(args), ws, nbytes, None) == status


def test_page_moves_are_refused():
    lib = L.load()
    need = lib.fastmax_cache_workspace(7)
    assert need >= 12 * 7 and lib.fastmax_cache_workspace(0) == 0

    def both(state=PTR, floats=64, pages=9, table=PTR, places=7, sources=PTR, result=PTR, ws=PTR, nbytes=need):
        return (lib.fastmax_cache_arrange(state, floats, pages, table, places, sources, result, ws, nbytes, None),
                lib.fastmax_cache_compact(state, floats, pages, table, places, result, ws, nbytes, None) if sources else 1)

    for fields, status in (({"state": None}, 1), ({"table": None}, 1), ({"result": None}, 1), ({"sources": None}, 1), ({"floats": 0}, 1), ({"pages": 0}, 1),
                           ({"places": 0}, 1), ({"pages": L.CACHE_PAGES + 1}, 2), ({"places": L.CACHE_PAGES + 1}, 2), ({"state": PTR + 4}, 6),
                           ({"floats": 66}, 6), ({"ws": None}, 3), ({"ws": PTR + 8}, 3), ({"nbytes": need - 1}, 3)):
        assert both(**fields) == (status, status), fields

    def copy(**fields):
        a = L.PagesCopyArgs(PTR, 2 * PTR, 64, 64, 64, 4, 4, None, None, 3, 0)
        for name, value in fields.items():
            setattr(a, name, value)
        return lib.fastmax_pages_copy(C.byref(a), None)

    for fields, status in (({"src": None}, 1), ({"dst": None}, 1), ({"page_floats": 0}, 1), ({"src_pages": 0}, 1), ({"dst_pages": -1}, 1), ({"count": -1}, 1),
                           ({"src_stride": 60}, 1), ({"dst_stride": 0}, 1), ({"src": PTR + 4}, 6), ({"dst": PTR + 8}, 6), ({"src_stride": 66}, 6),
                           ({"dst_stride": 66}, 6), ({"page_floats": 62}, 6), ({"count": 0}, 0)):
        assert copy(**fields) == status, fields
    assert lib.fastmax_pages_copy(None, None) == 1


def test_numbers_on_the_host_are_checked():
    like = torch.zeros(3, 2, 4, 16)
    assert per_sequence(None, like, "x", 0, 4) is None
    assert per_sequence([0, 4, 1], like, "x", 0, 4).tolist() == [0, 4, 1]
    assert per_sequence(torch.tensor([0, 4, 1]), like, "x", 0, 4).dtype == torch.int32
    for bad, error in (([0, 5, 1], ValueError), ([0, -1, 1], ValueError), ([0, 1], ValueError), (torch.zeros(3), TypeError),
                       (torch.zeros(3, dtype=torch.bool), TypeError), (torch.zeros(3, 1, dtype=torch.int32), ValueError)):
        with pytest.raises(error):
            per_sequence(bad, like, "x", 0, 4)
    good = torch.tensor([[-1, 0, 0, 2]] * 3)
    assert tree_parents(None, like) is None and tree_parents(good, like).dtype == torch.int32
    for bad, error in ((good[:, :3], ValueError), (good[:2], ValueError), (good.float(), TypeError), (torch.tensor([[0, 0, 0, 0]] * 3), ValueError),
                       (torch.tensor([[-1, 0, 0, 3]] * 3), ValueError), (torch.tensor([[-1, 0, -2, 0]] * 3), ValueError)):
        with pytest.raises(error):
            tree_parents(bad, like)
    with pytest.raises(ValueError):
        tree_parents(good, like[:, 0])


@pytest.mark.parametrize("dtype", [torch.uint8, torch.int8, torch.int16, torch.uint16, torch.int32, torch.uint32, torch.int64])
def test_host_numbers_of_narrow_types_are_what_they_say(dtype):
    signed = dtype not in (torch.uint8, torch.uint16, torch.uint32)
    like = torch.zeros(3, 2, 4, 16)
    wide = torch.zeros(200, 1, 1, 16)
    top = min(199, torch.iinfo(dtype).max)
    for numbers, low, high in (([3, 0, 1], -1, 3), ([4, 0, 2], 0, 4), ([0, 2, 1], -2, 2)):
        got = per_sequence(torch.tensor(numbers, dtype=dtype), like, "x", low, high)
        assert got.dtype == torch.int32 and got.tolist() == numbers
    got = per_sequence(torch.full((200,), top, dtype=dtype), wide, "x", -2, 199)
    assert got.tolist() == [top] * 200
    rows = [[-1 if signed else 0, 0, 1, 2]] * 3
    if signed:
        assert tree_parents(torch.tensor(rows, dtype=dtype), like).tolist() == rows
    else:   # a root cannot be said in a type without a sign
        with pytest.raises(ValueError):
            tree_parents(torch.tensor(rows, dtype=dtype), like)
    with pytest.raises(ValueError):
        per_sequence(torch.tensor([5, 0, 0], dtype=dtype), like, "x", -1, 4)
    with pytest.raises(TypeError):
        per_sequence(torch.tensor([5, 0, 0], dtype=torch.uint64), like, "x", -1, 9)


def test_caches_that_cannot_be_are_refused():
    from reproducing_fastmax_results_b200 import FastmaxCache

    for bad in ({"d": 48}, {"p": 3}, {"places": 0}, {"pages": 0}, {"layers": 0}, {"heads": 0}, {"pages": L.CACHE_PAGES + 1}):
        with pytest.raises(ValueError):
            FastmaxCache(**{"places": 2, "heads": 2, "d": 16, "device": "cpu", **bad})
    cache = FastmaxCache(3, 2, 16, layers=2, pages=5, device="cpu")
    assert tuple(cache.state.shape) == (5, 2, 2, 209, 20) and cache.table.tolist() == [-1] * 3
    x = torch.zeros(3, 2, 4, 16)
    for call in (lambda: cache.begin([0, 0]), lambda: cache.end([3]), lambda: cache.begin([-1]), lambda: cache.arrange([0, 1]), lambda: cache.arrange([0, 3, 1]),
                 lambda: cache.arrange([0, -3, 1]), lambda: cache.verify(x[:2], x, x), lambda: cache.verify(x, x[:, :1], x), lambda: cache.verify(x, x, x, layer=2),
                 lambda: cache.verify(x, x, x, lengths=[0, 5, 1]), lambda: cache.accept(x, x, [4, 0, 0]), lambda: cache.accept(x, x, [0, 0, 0], layer=-1),
                 lambda: cache.step(x[0], x[0], x[0]), lambda: cache.prefill(x, x, x, [0, 1]), lambda: cache.prefill(x, x, x[:, :, :2], [0, 1, 2])):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(RuntimeError):   # there is no CPU path
        cache.verify(x, x, x)


def test_prompts_on_pages_are_checked_before_any_launch(monkeypatch):
    """One type, one device and unit strides for q, k and v: the binding behind takes all three from q."""
    from reproducing_fastmax_results_b200 import FastmaxCache, cache as module

    def reached(*args, **options):
        raise AssertionError("the prompt was launched")

    monkeypatch.setattr(module._lib, "forward", reached)
    monkeypatch.setattr(module, "_ext", reached)
    cache = FastmaxCache(3, 2, 16, layers=2, device="cpu")
    x, y = torch.zeros(2, 2, 4, 16), torch.zeros(2, 2, 4, 16, dtype=torch.bfloat16)
    apart = torch.zeros(2, 2, 16, 4).transpose(2, 3)
    for continues in (False, True):
        for q, k, v in ((x, y, x), (x, x, y), (y, x, x), (x, y, y), (y, y, x)):
            with pytest.raises(RuntimeError, match="dtypes differ"):
                cache.prefill(q, k, v, [0, 2], layer=1, continues=continues)
        for q, k, v in ((apart, x, x), (x, apart, x), (x, x, apart)):
            with pytest.raises(RuntimeError, match="contiguous"):
                cache.prefill(q, k, v, [0, 2], continues=continues)
        for bad in (x.half(), x.double(), x.int()):
            with pytest.raises(TypeError):
                cache.prefill(bad, bad, bad, [0, 2], continues=continues)
        for q, k, v in ((x, x, x), (y, y, y)):   # on the host
            with pytest.raises(RuntimeError, match="CUDA"):
                cache.prefill(q, k, v, [0, 2], continues=continues)
        for q, k, v in ((x[:, :, :0],) * 3, (x[0],) * 3, (x, x, x[:, :, :3]), (x, x[:, :1], x), (x, x, x[..., :8])):
            with pytest.raises(ValueError):
                cache.prefill(q, k, v, [0, 2], continues=continues)
    with pytest.raises(ValueError):
        cache.prefill(x, x, x, [0, 1], layer=2)


def test_prompts_of_the_decoder_are_checked_before_any_launch(monkeypatch):
    """As on pages; a v shorter than k would be read past its end."""
    from reproducing_fastmax_results_b200 import FastmaxDecoder, decoding as module

    def reached(*args, **options):
        raise AssertionError("the prompt was launched")

    monkeypatch.setattr(module._lib, "forward", reached)
    dec = FastmaxDecoder(2, 3, 16, device="cpu")
    x, y = torch.zeros(2, 3, 4, 16), torch.zeros(2, 3, 4, 16, dtype=torch.bfloat16)
    for q, k, v in ((x, x, x[:, :, :3]), (x, x[:, :, :3], x), (x[0], x, x), (x, x, x[0]), (x, x[:1], x), (x, x, x[..., :8]), (x[:, :, :0],) * 3):
        with pytest.raises(ValueError):
            dec.prefill(q, k, v)
    for q, k, v in ((x, y, x), (x, x, y), (y, x, y)):
        with pytest.raises(RuntimeError, match="dtypes differ"):
            dec.prefill(q, k, v)
    with pytest.raises(RuntimeError, match="contiguous"):
        dec.prefill(x, x, torch.zeros(2, 3, 16, 4).transpose(2, 3))
    with pytest.raises(TypeError):
        dec.prefill(x.half(), x.half(), x.half())
    with pytest.raises(RuntimeError, match="CUDA"):
        dec.prefill(x, x, x)
    assert dec.tokens_seen == 0


def test_outputs_whose_rows_lie_on_one_another_are_refused():
    from reproducing_fastmax_results_b200 import FastmaxCache, FastmaxDecoder

    x = torch.zeros(3, 2, 4, 16)
    cache, dec = FastmaxCache(3, 2, 16, device="cpu"), FastmaxDecoder(3, 2, 16, device="cpu")
    for out in (torch.zeros(1, 2, 4, 16), torch.zeros(3, 1, 4, 16), torch.zeros(3, 2, 1, 16), torch.zeros(1)):
        for serve in (cache, dec):
            with pytest.raises(RuntimeError, match="single memory location"):
                serve.verify(x, x, x, out=out.expand(3, 2, 4, 16))
    for out in (torch.zeros(1, 2, 16), torch.zeros(3, 1, 16), torch.zeros(1)):
        for serve in (cache, dec):
            with pytest.raises(RuntimeError, match="single memory location"):
                serve.step(x[:, :, 0], x[:, :, 0], x[:, :, 0], out=out.expand(3, 2, 16))


def test_the_operator_refuses_sizes_that_do_not_fit_before_any_launch():
    """A v shorter than k, or keys of fewer heads than queries, would be read past their end."""
    from reproducing_fastmax_results_b200 import fastmax_custom

    x = torch.zeros(2, 3, 8, 16)
    for k, v in ((x, x[:, :, :7]), (x[:, :, :7], x), (x[:1], x[:1]), (x[:, :2], x[:, :2]), (x, x[:, :1]), (x[..., :8], x[..., :8])):
        for normalize in (False, True):
            with pytest.raises(RuntimeError, match="as many values as keys"):
                fastmax_custom(x, k, v, None, None, True, 0.0, normalize)
    with pytest.raises(RuntimeError, match="dtypes differ"):
        fastmax_custom(x, x.bfloat16(), x)
    with pytest.raises(RuntimeError, match="CUDA"):
        fastmax_custom(x, x[:, :, :5], x[:, :, :5])


# ---- the oracle ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("order", [1, 2])
@pytest.mark.parametrize("d", [16, 32])
def test_tree_oracle_is_the_operator_on_every_path(d, order):
    """What a node gets is the last row of the causal operator over the sequence and the node's path."""
    rng = np.random.default_rng(d + order)
    n, before = 9, 20
    a, inv_t = (1.1, 0.9, 0.4), 0.2
    k0, v0 = rng.standard_normal((2, before, d))
    q, k, v = rng.standard_normal((3, n, d))
    parents = [-1, 0, 0, 1, -1, 4, 2, 2, 5]
    state, _ = so.grown(np.zeros((so.features(k0[:1], order).shape[1], d + 4)), k0, v0, order)
    state = np.concatenate([state, np.zeros((len(state), 3))], 1)
    o, g, _, _ = so.tree(q, k, v, state, parents, order, a, inv_t)
    poly = orc.Poly(*a, inv_t, order)
    for i in range(n):
        nodes = so.path(parents, i)
        keys, values = np.concatenate([k0, k[nodes]]), np.concatenate([v0, v[nodes]])
        o_ref, g_ref = orc.fastmax_naive(q[i][None, None, None], keys[None, None], values[None, None], False, poly)
        assert np.allclose(o[i], o_ref[0, 0, 0], rtol=1e-11, atol=1e-11) and np.isclose(g[i], g_ref[0, 0, 0], rtol=1e-11)


def test_page_oracle():
    table = [3, -1, 0, 2]
    assert so.arranged(table, [0, 1, 2, 3], 4) == ([3, -1, 0, 2], [], 0)
    assert so.arranged(table, [2, 0, 2, -1], 4) == ([0, 3, 1, -1], [(0, 1)], 0)
    assert so.arranged(table, [-2, 2, 2, 2], 4) == ([1, 0, 2, 3], [(-1, 1), (0, 2), (0, 3)], 0)
    assert so.arranged(table, [-2, 9, -3, 3], 2) == ([0, -1, -1, -1], [(-1, 0)], 2)
    assert so.arranged([0, 1], [0, -2], 1) == ([0, -1], [], 1)
    assert so.compacted([3, -1, 5, 0], 6) == ([1, -1, 2, 0], [(3, 1), (5, 2)], 3)
    assert so.compacted([-1, -1], 3) == ([-1, -1], [], 0)
