# SPDX-License-Identifier: MIT
"""The paged beam cache at the edges of its contract: graphs, adopted state, refused paths, values and
weights at the ends of their ranges. Models and bounds are those of test_cache.py."""

from __future__ import annotations

import ctypes as C
import math
import threading
import time

import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

from beamgrad_b200 import _abi as A
from beamgrad_b200 import cache as cache_module
from beamgrad_b200.cache import PagedCache
from test_cache import DTYPES, Model, attend_exact, check_attend, draft_tree, random_cache, tensors


# -- the workspace ----------------------------------------------------------------------


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, dim", [(torch.bfloat16, 64), (torch.float32, 64), (torch.float16, 200)])
def test_graphs_of_one_cache_replay_in_any_order(dtype, dim):
    """Two graphs of one cache, the second replayed first, in memory that an earlier graph left full of
    ones and zeros: what divided segments are joined by cannot come from either graph."""
    cache = random_cache(1, 4, np.full((1, 4), 900), 1, layers=1, dim=dim, dtype=dtype, seed=6)
    inputs = [tensors(cache, 1, 4, seed) for seed in (1, 2)]
    want = [cache.attend(0, *x) for x in inputs]
    pool = torch.cuda.graph_pool_handle()
    graphs = [torch.cuda.CUDAGraph() for _ in range(3)]
    torch.cuda.synchronize()
    with torch.cuda.graph(graphs[0], pool=pool):
        used = torch.full((64 << 20,), 0x5A, dtype=torch.uint8, device="cuda")
    graphs[0].replay()
    torch.cuda.synchronize()
    del used
    got = []
    for graph, x in zip(graphs[1:], inputs):
        with torch.cuda.graph(graph, pool=pool):
            got.append(cache.attend(0, *x))
    for i in (1, 0, 1):
        graphs[1 + i].replay()
        assert torch.equal(got[i], want[i])


@pytest.mark.gpu
def test_a_cache_has_one_workspace_from_the_start():
    cache = random_cache(1, 2, np.full((1, 2), 40), 1, layers=1)
    x = tensors(cache, 1, 2, 0)
    before = torch.cuda.memory_allocated()
    want = cache.attend(0, *x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = cache.attend(0, *x)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    assert torch.cuda.memory_allocated() - before < 1 << 20  # the outputs


# -- weights at the ends of their range -------------------------------------------------


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("K, N, group, dim", [(1, 20, 1, 64), (1, 16, 4, 64), (1, 20, 4, 128), (1, 70, 2, 64), (3, 70, 2, 64), (1, 20, 2, 200)])
def test_hidden_values_at_the_end_of_their_type(K, N, group, dim, dtype):
    """A weight of zero is zero: a hidden value of the type's largest magnitude shows in no output. The
    drafted tokens that nobody sees, and the rows of the pool that nobody holds, are such values."""
    cache = random_cache(1, K, np.full((1, K), 150), N, layers=1, heads=1, dim=dim, dtype=dtype, seed=2)
    big = torch.finfo(dtype).max
    cache.pages[0, 1, cache.references == 0] = big
    q, k, v = tensors(cache, N, group, 3)
    v[:, :, 1::2] = big
    mask = draft_tree(1, K, N, np.random.RandomState(1))
    mask[..., 1::2] = False
    check_attend(cache, 0, q, k, v, mask)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 200])
@pytest.mark.parametrize("N", [1, 40, 100, 200])
def test_small_weights_in_float16(N, dim):
    """1744 keys of weight 2^-25.5 beside 256 of weight 1 whose values are 0: all of the output comes from
    weights that float16 holds as 0 or as one step, where the largest is 1. With the largest at 2^7 a step of
    2^-24 rounds them by 2^-25 at the most, 2^-32 of the largest: a share of 2^-6.5 of each. The sums and the
    exponentials add 2^-19, the output's rounding 2^-11."""
    B, H, T, low = 20, 8, 2000, -25.5
    cache = random_cache(B, 1, np.full((B, 1), T), N, layers=1, heads=H, dim=dim, page=16, dtype=torch.float16, seed=1)
    cache.pages.zero_()
    others = cache.table[:, 0, 16 : T // 16].long().reshape(-1)
    cache.pages[0, 0, others, :, :, 0] = low
    cache.pages[0, 1, others] = 32768.0
    cache.refresh()
    q = torch.zeros((B, 1, N, H, dim), device="cuda", dtype=torch.float16)
    k, v = q.clone(), q.clone()
    q[..., 0], k[..., 0] = 1, -200  # the new tokens weigh nothing
    out, lse = cache.attend(0, q, k, v, scale=float(np.log(2.0)), return_lse=True)
    want = 32768 * (T - 256) * 2.0**low / 256
    assert float((out.double() / want - 1).abs().max()) <= 2.0**-6.5 + 2.0**-11 + 2.0**-19
    assert float((lse.double() - np.log(256 + (T - 256) * 2.0**low)).abs().max()) <= 2.0**-19 + 2.0**-21 * 6


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("N, dim", [(1, 64), (40, 64), (100, 128), (200, 64), (1, 200), (40, 200)])
def test_scores_that_rise_within_a_row(N, dim, dtype):
    """Every row's maximum rises from tile to tile, by less and by more than the references tolerate, with
    values near the end of float16: weights and sums stay within their types."""
    T = 1500
    cache = random_cache(2, 1, np.full((2, 1), T), N, layers=1, heads=2, dim=dim, page=16, dtype=dtype, seed=3)
    place = torch.arange(T, device="cuda")
    pages = cache.table[:, 0].long()[:, place // 16], place % 16
    q, k, v = tensors(cache, N, 1, 9)
    for rise in (0.05, 0.2):  # of a score in base 2, a position
        cache.pages[0, 0, pages[0], :, pages[1], 0] = (place * rise).to(dtype)[None, :, None]
        cache.pages[0, 1].mul_(30000 / cache.pages[0, 1].abs().max())
        cache.refresh()
        for x in (q, k, v):
            x[..., 0] = 1
        check_attend(cache, 0, q, k, v, scale=float(np.log(2.0)))


# Unit roundoff: 24, 11 and 8 significant bits, rounded to the nearest.
UNIT = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N, group, dim", [(1, 1, 64), (10, 4, 64), (50, 4, 128), (70, 4, 64), (1, 2, 200), (10, 4, 200)])
@pytest.mark.parametrize("kind", ["some", "overflow", "all", "plus", "nan"])
def test_scores_that_are_not_finite(kind, N, group, dim, dtype):
    """A score of -inf (of a key that holds it, or of a sum of products that 32 bits do not hold) weighs nothing, and
    a row with such scores alone is as one that sees nothing. A score of +inf or NaN makes the row NaN, and
    no other row. Bound as in test_cache.py, over the keys that weigh something."""
    T, scale = 300, 1e-3 / math.sqrt(dim) if kind == "overflow" else 1 / math.sqrt(dim)
    cache = random_cache(1, 1, np.full((1, 1), T), N, layers=1, heads=1, dim=dim, dtype=dtype, seed=4)
    q, k, v = tensors(cache, N, group, 5)
    q = q.abs() + 0.25
    if kind == "overflow":
        q = q * 1000  # (float16 has no such sums: -65504 * 1000 * 200 is far above -3e38, and weighs nothing all the same)
    place = torch.arange(T, device="cuda")
    pages, at = cache.table[0, 0].long()[place // 16], place % 16
    hit = torch.zeros(T + N, dtype=torch.bool, device="cuda")
    if kind in ("some", "overflow"):
        hit[:T:3] = True
        cache.pages[0, 0, pages[::3], :, at[::3]] = -torch.finfo(dtype).max
        if kind == "some":
            cache.pages[0, 0, pages[::3], :, at[::3], 3] = -math.inf
    elif kind == "all":
        hit[:] = True
        cache.pages[0, 0, pages, :, at, 0] = -math.inf
        k[..., 0] = -math.inf
    else:  # the new token N // 2, seen by itself and the later ones
        hit[T + N // 2] = True
        k[:, :, N // 2, :, 1] = math.inf if kind == "plus" else math.nan
    keys = torch.cat([cache.pages[0, 0, pages, 0, at], k[0, 0, :, 0]]).double()
    values = torch.cat([cache.pages[0, 1, pages, 0, at], v[0, 0, :, 0]]).double()
    out, lse = (x[0, 0] for x in cache.attend(0, q, k, v, scale=scale, return_lse=True))
    cache.check()
    for i in range(N):
        see = torch.arange(T + N, device="cuda") <= T + i
        if kind in ("plus", "nan") and i >= N // 2:
            assert bool(torch.isnan(out[i]).all()) and bool(torch.isnan(lse[i]).all())
            continue
        see &= ~hit
        if not bool(see.any()):
            assert bool((out[i] == 0).all()) and bool((lse[i] == -math.inf).all())
            continue
        x = (q[0, 0, i].double() @ keys[see].T) * scale  # [group, T]
        z, y = torch.logsumexp(x, 1), torch.softmax(x, 1) @ values[see]
        e = (dim + 4) * 2.0**-24 * scale * float((q[0, 0, i].double().abs() @ keys[see].abs().T).max()) + 2.0**-22 * float(x.abs().max())
        bound = float(values[see].abs().max()) * (2 * UNIT[dtype] + 2 * e + 2.0**-19 + 2 * (T + N) * 2.0**-24)
        assert float((out[i].double() - y).abs().max()) <= bound
        assert bool(((lse[i].double() - z).abs() <= e + 2.0**-19 + (T + N) * 2.0**-24 + 2.0**-22 * z.abs()).all())


# -- values that are not finite ---------------------------------------------------------


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_a_cache_recovers_from_values_that_are_not_finite(dtype):
    """They are forgotten with the beam that held them (refresh) and with everything else (reset); the rest of
    the pool is left as it was."""
    B, K, N, G = 1, 3, 2, 4
    cache = random_cache(B, K, np.full((B, K), 60), N, layers=2, heads=1, dtype=dtype, seed=8)
    q, k, v = tensors(cache, N, G, 2)
    assert not cache.has_nonfinite
    bad = v.clone()
    bad[0, 1, 0, 0, :8] = torch.tensor([np.inf, 1, -np.inf, np.nan, 2, 3, np.nan, np.nan])
    cache.attend(1, q, k, bad)
    assert cache.has_nonfinite
    cache.refresh()
    assert cache.has_nonfinite  # beam 1 holds them
    cache.fork(torch.tensor([[0, 0, 2]], device="cuda"), room=N)
    assert cache.has_nonfinite
    before = cache.pages.clone()
    cache.refresh()
    assert not cache.has_nonfinite
    assert torch.equal(cache.pages, torch.where(torch.isfinite(before), before, 0))
    check_attend(cache, 1, q, k, v)
    cache.attend(1, q, k, bad)
    before = cache.pages.clone()
    assert cache.has_nonfinite
    cache.reset()
    assert not cache.has_nonfinite and cache.lengths.sum() == 0
    assert torch.equal(cache.pages, torch.where(torch.isfinite(before), before, 0))
    cache.check()
    cache.reserve(N)
    check_attend(cache, 1, q, k, v)
    # A pool that was never written may hold anything where nobody looks.
    pages = torch.full((1, 2, 6, 1, 16, 64), float("nan"), device="cuda").to(dtype)
    pages[:, :, 2] = 1
    adopted = PagedCache.from_tensors(pages, torch.tensor([[[2, -1]]], dtype=torch.int32, device="cuda"),
                                      torch.tensor([[16]], dtype=torch.int32, device="cuda"))
    assert not adopted.has_nonfinite
    q, k, v = tensors(adopted, 1, 1, 3)
    adopted.reserve(1)
    before = adopted.pages[0].cpu()  # (check_attend compares the pages too, whose keys are still NaN)
    out, lse = adopted.attend(0, q, k, v, return_lse=True)
    want, z, bound, z_bound = attend_exact(before, adopted.table.cpu(), adopted.lengths.cpu(), q.cpu(), k.cpu(), v.cpu(), None, None, 0.125)
    assert bool(((out.cpu().double() - want).abs().amax(-1) <= bound).all())
    assert bool(((lse.cpu().double() - z).abs() <= z_bound).all())


# -- adopted state ----------------------------------------------------------------------


def adopt(table, lengths, pages=12, page=16, dtype=torch.float32):
    put = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    pool = torch.randn((2, 2, pages, 1, page, 64), device="cuda").to(dtype)
    return PagedCache.from_tensors(pool, put(table), put(lengths))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_adopted_lengths_out_of_range(dtype):
    """Lengths below 0 and above the table are brought into range and reported; nothing is read or written
    outside the pages of the table."""
    held = [[[0, 1, 2], [3, 4, 5]], [[6, 7, 8], [9, 10, 11]]]
    for lengths in ([[-1, 20], [-(2**31), 5]], [[49, 20], [2**31 - 1, 48]], [[-17, 2**30], [7, -3]]):
        cache = adopt(held, lengths, dtype=dtype)
        with pytest.raises(RuntimeError, match="length"):
            cache.check()
        assert cache.lengths.cpu().tolist() == [[min(max(n, 0), 48) for n in row] for row in lengths]
        Model(cache).check_plan(cache)
        q, k, v = tensors(cache, 2, 2, 1)
        check_attend(cache, 0, q, k, v)
    cache = adopt(held, [[0, 48], [16, 47]], dtype=dtype)
    cache.check()


HOLES = [  # table rows of one example, lengths, parents, room; pages of 16
    ([[0, -1, 5, -1], [2, 3, -1, -1]], [3, 20], None, 61),           # a spare page behind a missing one
    ([[0, -1, 5, -1, 7, -1], [1, -1, -1, 8, -1, 2]], [16, 0], None, 80),
    ([[-1, 4, -1, 6], [-1, -1, 3, -1]], [20, 40], None, 30),          # committed positions without a page
    ([[0, -1, 5, -1], [2, 3, -1, 9]], [9, 20], [1, 1], 40),           # the first child keeps them, the other copies
    ([[0, -1, 5, -1], [2, 3, -1, 9]], [9, 20], [0, 0], 55),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", range(len(HOLES)))
def test_adopted_tables_with_holes(case):
    """Every missing column gets a page of its own, whatever pages lie between."""
    rows, lengths, parents, room = HOLES[case]
    cache = adopt([rows, [[-1] * len(rows[0])] * 2], [lengths, [0, 0]], pages=24)
    model = Model(cache)
    by = None if parents is None else np.array([parents, [0, 1]])
    cache.fork(None if by is None else torch.from_numpy(by).cuda(), room=room)
    model.fork(by, 0, room)
    model.check(cache)
    assert int(cache.references.max()) <= (1 if parents is None else 2)
    cache.fork(written=1, room=room + 3)
    model.fork(None, 1, room + 3)
    model.check(cache)


@pytest.mark.gpu
def test_adopted_tables_with_holes_at_random():
    for seed in range(12):
        rng = np.random.RandomState(seed)
        B, K, M, P = 3, int(rng.choice([2, 5, 33])), int(rng.choice([4, 40, 300])), 4000
        K = min(K, P // (2 * B * M) or 1)
        table = rng.permutation(P)[: B * K * M].reshape(B, K, M)
        table[rng.rand(B, K, M) < 0.4] = -1
        lengths = rng.randint(0, M * 16 // 2, (B, K))
        cache = adopt(table.tolist(), lengths.tolist(), pages=P + B * K * M)
        model = Model(cache)
        parents = None if seed % 2 else rng.randint(0, K, (B, K))
        room = M * 8 - int(rng.randint(0, 20))
        cache.fork(None if parents is None else torch.from_numpy(parents).cuda(), room=room)
        model.fork(parents, 0, room)
        model.check(cache)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["another beam", "another example", "another group", "another column", "complete pages", "complete for one"])
def test_adopted_pages_that_are_shared_before_they_are_complete(kind):
    """The next token of one holder would be a token of the other: reported, whoever the other is."""
    B, K = (1, 34) if kind == "another group" else (2, 2)
    table = np.arange(B * K * 3).reshape(B, K, 3)
    lengths = np.full((B, K), 20)
    if kind == "another beam":
        table[0, 1, 1] = table[0, 0, 1]
    elif kind == "another example":
        table[1, 1, 1] = table[0, 0, 1]
    elif kind == "another group":
        table[0, 33, 1] = table[0, 0, 1]
    elif kind == "another column":
        table[0, 0, 2] = table[0, 0, 1]
    elif kind == "complete pages":
        table[:, :, 0] = table[0, 0, 0]
    else:
        lengths[1, 1], table[1, 1, 0] = 9, table[0, 0, 0]
    cache = adopt(table.tolist(), lengths.tolist(), pages=B * K * 3)
    Model(cache).check_plan(cache)
    if kind == "complete pages":
        cache.check()
    else:
        with pytest.raises(RuntimeError, match="shared"):
            cache.check()


# -- paths that are refused -------------------------------------------------------------


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["falls late", "repeats", "below zero", "count above the width", "negative count", "no page", "no column"])
def test_a_refused_path_leaves_its_beam_alone(kind):
    cache = PagedCache(1, 4, 640, num_layers=2, num_kv_heads=1, head_dim=8, page_size=16, dtype=torch.float32)
    cache.pages.normal_()
    cache.fork(room=40)
    cache.fork(torch.tensor([[0, 1, 2, -1]], device="cuda"), written=37, room=400)  # the last beam is empty
    model = Model(cache)
    path = np.tile(np.arange(300) + 2, (1, 4, 1))
    counts = np.array([[3, 5, 300, 4]])
    path[0, 0, 1:] += 1
    good = counts.copy()
    good[0, 1], good[0, 3] = 0, 0
    if kind == "falls late":
        path[0, 1, 280], counts[0, 1] = path[0, 1, 279] - 1, 300
    elif kind == "repeats":
        path[0, 1, 3] = path[0, 1, 2]
    elif kind == "below zero":
        path[0, 1, 0] = -1
    elif kind == "count above the width":
        counts[0, 1] = 301
    elif kind == "negative count":
        counts[0, 1] = -2
    elif kind == "no page":
        path[0, 1, 4] = 450
    else:
        path[0, 1, 4] = 2**31 - 1
    dev = lambda x: torch.from_numpy(x.astype(np.int32)).cuda()  # noqa: E731
    cache.commit(dev(path), dev(counts), room=7)
    model.commit(path, good, 7)
    # The empty beam has no tokens and gets room like the others.
    model.check(cache)
    with pytest.raises(RuntimeError, match="path entry"):
        cache.check()


@pytest.mark.gpu
def test_an_empty_beam_accepts_nothing_without_an_error():
    cache = PagedCache(1, 2, 64, num_layers=1, num_kv_heads=1, head_dim=8, page_size=16, dtype=torch.float32)
    cache.fork(torch.tensor([[0, -1]], device="cuda"), room=6)
    cache.commit(torch.tensor([[[0, 2], [0, 1]]], device="cuda"), torch.tensor([[2, 2]], device="cuda"))
    assert cache.lengths.cpu().tolist() == [[2, 0]]
    cache.check()


# -- the host side ----------------------------------------------------------------------


class _Library:
    """The engine's library with its launches of attend handed to the test."""

    def __init__(self, launch):
        self.real, self.launch = A.load(), launch

    def __getattr__(self, name):
        return getattr(self.real, name)

    def dbs_cuda_cache_attend(self, cache, args, stream):
        self.launch(args._obj)
        return 0


def host_cache(monkeypatch, launch=lambda args: None, **sizes) -> PagedCache:
    """A cache of host memory: everything that attend does before a launch, without a device."""
    monkeypatch.setattr(cache_module, "_on", lambda device: cache_module._HERE)
    monkeypatch.setattr(cache_module, "_raw_stream", lambda index: 0)
    z = lambda *shape: torch.zeros(shape, dtype=torch.int32)  # noqa: E731
    cache = PagedCache.__new__(PagedCache)
    pages = torch.zeros((1, 2, 8, 1, 16, 64), dtype=torch.float16)
    cache._describe(tuple(pages.shape), (1, 2, 4), pages.dtype)
    cache._adopt(pages, z(1, 2, 4), z(1, 2), z(8))
    cache.lib = _Library(launch)
    return cache


def host_inputs(N, heads=1, shape=(1, 2)):
    return [torch.zeros((*shape, N, heads, 64), dtype=torch.float16) for _ in range(3)]


def test_what_attend_remembers_is_bounded(monkeypatch):
    seen = []
    cache = host_cache(monkeypatch, lambda a: seen.append(a.new_tokens))
    for N in range(1, 1001):
        cache.attend(0, *host_inputs(N))
        assert len(cache._calls) <= 256
    assert seen == list(range(1, 1001))


def test_tangents_are_refused(monkeypatch):
    seen = []
    cache = host_cache(monkeypatch, seen.append)
    inputs = host_inputs(2)
    with forward_ad.dual_level(), torch.no_grad():
        for i in range(3):
            dual = [forward_ad.make_dual(x, torch.ones_like(x)) if i == j else x for j, x in enumerate(inputs)]
            with pytest.raises(RuntimeError, match="derivative"):
                cache.attend(0, *dual)
        assert not seen
        cache.attend(0, *inputs)
        cache.attend(0, inputs[0])
    assert len(seen) == 2


def test_two_threads_do_not_mix_their_arguments(monkeypatch):
    wrong, calls = [], []

    def launch(a):
        at = a.q, a.k, a.v, a.out, a.lse
        time.sleep(0.002)  # another thread may run
        wrong.extend(x for x in zip(at, (a.q, a.k, a.v, a.out, a.lse)) if x[0] != x[1])
        calls.append(at[:4])

    cache = host_cache(monkeypatch, launch)
    args = [host_inputs(2) for _ in range(2)]
    outs = [torch.zeros_like(x[0]) for x in args]

    def work(i):
        for _ in range(20):
            cache.attend(0, *args[i], out=outs[i], return_lse=True)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong and len(calls) == 40
    assert set(calls) == {(*(x.data_ptr() for x in args[i]), outs[i].data_ptr()) for i in range(2)}


def test_indexes_that_32_bits_do_not_hold(monkeypatch):
    cache = host_cache(monkeypatch)
    x = torch.tensor([[2**32, 2**31 + 1]])
    assert cache._int32(x, "parents").tolist() == [[2**31 - 1] * 2]
    assert cache._int32(-x, "parents").tolist() == [[-1, -1]]
    x = torch.tensor([[3, -1]])
    assert cache._int32(x, "parents").tolist() == [[3, -1]] and cache._int32(x, "parents").dtype == torch.int32
    y = x.int()
    assert cache._int32(y, "parents") is y


@pytest.mark.gpu
def test_parents_that_32_bits_do_not_hold_are_out_of_range():
    cache = PagedCache(1, 2, 64, num_layers=1, num_kv_heads=1, head_dim=8, page_size=16, dtype=torch.float32)
    cache.fork(torch.tensor([[0, 2**32]], device="cuda"))
    with pytest.raises(RuntimeError, match="out of range"):
        cache.check()
    cache.reset()
    cache.reserve(4)
    cache.commit(torch.tensor([[[0], [2**32]]], device="cuda"), torch.tensor([[1, 1]], device="cuda"))
    with pytest.raises(RuntimeError, match="out of range"):
        cache.check()
    assert cache.lengths.cpu().tolist() == [[1, 0]]


def test_misaligned_arrays_are_refused_before_a_launch():
    """Checked where a launch could not follow: no device here, and on one every call below is refused."""
    lib, base = A.load(), 1 << 20  # addresses that nothing reads
    c = A.Cache(batch_size=1, beam_size=2, max_pages=4, num_pages=8, num_layers=1, num_heads=1, head_dim=64, page_size=16,
                data_type=A.DTYPE_F16, pages=base, table=base, lengths=base, references=base, plan=base, status=base)
    c.plan_bytes = lib.dbs_cuda_cache_plan_bytes(C.byref(c))
    ref = C.byref(c)
    for off in (1, 2, 3):
        for at in range(3):
            x = [base + off if i == at else base for i in range(3)]
            assert lib.dbs_cuda_cache_fork(ref, x[0], x[1], 0, x[2], 0, None) == A.STATUS_INVALID_ARGUMENT
        for x in ((base + off, base), (base, base + off)):
            assert lib.dbs_cuda_cache_commit(ref, x[0], 2, x[1], 0, None) == A.STATUS_INVALID_ARGUMENT
        for name in ("lse", "counts"):
            a = A.AttendArgs(beams=2, new_tokens=1, query_heads=1, scale=1.0, q=base, out=base, workspace=base)
            a.workspace_bytes = lib.dbs_cuda_cache_attend_workspace_size(ref, C.byref(a))
            setattr(a, name, base + off)
            assert lib.dbs_cuda_cache_attend(ref, C.byref(a), None) == A.STATUS_INVALID_ARGUMENT


def test_numbers_of_tokens_are_whole(monkeypatch):
    cache = host_cache(monkeypatch)
    for call in (lambda: cache.fork(written=0.5), lambda: cache.fork(room=1.5), lambda: cache.reserve(0.9),
                 lambda: cache.commit(torch.zeros((1, 2, 1), dtype=torch.int32), torch.zeros((1, 2), dtype=torch.int32), room=0.5)):
        with pytest.raises(TypeError):
            call()
    assert cache_module._number(np.int64(3), "room") == 3


def test_sizes_that_32_bits_do_not_hold():
    sizes = dict(num_layers=1, num_kv_heads=1, head_dim=64, num_pages=4, page_size=16, device="cuda:0")
    for args, change in (((1, 1, (2**32 + 2) * 16), {}), ((2**32 + 1, 1, 64), {}), ((1, 1, 64), dict(num_pages=2**32 + 4)),
                         ((1, 1, 64), dict(head_dim=2**32 + 64))):
        with pytest.raises(ValueError):
            PagedCache(*args, **(sizes | change))


# -- large calls ------------------------------------------------------------------------


@pytest.mark.parametrize("code, dim, new, most", [(A.DTYPE_BF16, 128, 4096, 65536), (A.DTYPE_F16, 64, 4096, 65536), (A.DTYPE_F32, 64, 4096, 4096),
                                                  (A.DTYPE_BF16, 256, 1024, 2048)])
def test_prompts_on_large_caches_are_not_refused(code, dim, new, most):
    """What bounds a call is that its tiles are counted in 31 bits: blocks of rows by tiles of positions as the
    kernels have them (256 by 128, 64 by 64, 32 by 64), over full tables."""
    lib = A.load()
    c = A.Cache(batch_size=32, beam_size=8, max_pages=1024, num_pages=32768, num_layers=1, num_heads=8, head_dim=dim,
                page_size=32, data_type=code)
    size = lambda N: lib.dbs_cuda_cache_attend_workspace_size(C.byref(c), C.byref(A.AttendArgs(  # noqa: E731
        beams=1, new_tokens=N, query_heads=64, scale=1.0)))
    assert size(1) > 0 and size(new) == size(1) and size(most) == size(1)
    assert size(65537) < 0
    c.batch_size, c.num_pages = 4096, 1024  # tables of 2^25 pages
    assert size(most) < 0 and size(1) > 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_a_long_prompt_on_a_large_cache(dtype):
    B, N, H, G, D = 32, 4096, 8, 8, 8
    cache = PagedCache(B, 8, 32768, num_layers=1, num_kv_heads=H, head_dim=D, num_pages=B * N // 32 + 8, dtype=dtype)
    room = torch.zeros((B, 8), dtype=torch.int32, device="cuda")
    room[:, 0] = N
    cache.reserve(room)
    q, k, v = tensors(cache, N, G, 4, beams=1)
    out, lse = cache.attend(0, q, k, v, return_lse=True)
    cache.check()
    rng = np.random.RandomState(0)
    u = UNIT[dtype]
    for b, i, h in [(0, 0, 0), (B - 1, N - 1, H * G - 1), *zip(rng.randint(0, B, 40), rng.randint(0, N, 40), rng.randint(0, H * G, 40))]:
        keys, values = (t[b, 0, : i + 1, h // G].double() for t in (k, v))
        s = keys @ q[b, 0, i, h].double() / math.sqrt(D)
        z, y = torch.logsumexp(s, 0), torch.softmax(s, 0) @ values
        e = (D + 4) * 2.0**-24 * float((keys.abs() @ q[b, 0, i, h].double().abs()).max()) / math.sqrt(D) + 2.0**-22 * float(s.abs().max())
        bound = float(values.abs().max()) * (2 * u + 2 * e + 2.0**-19 + 2 * (i + 1) * 2.0**-24)
        assert float((out[b, 0, i, h].double() - y).abs().max()) <= bound
        assert float((lse[b, 0, i, h].double() - z).abs()) <= e + 2.0**-19 + (i + 1) * 2.0**-24 + 2.0**-22 * abs(float(z))
