# SPDX-License-Identifier: MIT
"""The paged beam cache (beamgrad_b200.cache, include/dbs_cuda_cache.h) against plain models.

State: every operation against a page-by-page model in Python, whole numbers equal and rows bit for
bit. Attention: against the definition in 64 bits, one beam and head at a time, within a bound from
the number formats (below). Refusals: on the CPU where no device is needed.

Bound of an attention output. With u the unit roundoff of the output type (2^-9 bfloat16, 2^-12
float16 rounded up to 2^-11, 2^-24 float32), scores S = scale q.k and V the largest |v| that a row
sees: a score is off by at most e = (D + 4) 2^-24 |scale| max sum|q k| + 2^-22 max|S| (a sum of D
products in 32 bits, and the rounding of the exponential's argument), so a weight is off by a factor
of 1 + e + 2^-21 (the exponential); weights may be rounded to the input type (u), sums of T terms
in 32 bits add T 2^-24 at the most, and the output is rounded once (u). Numerator and denominator
carry the weight's error: |out - exact| <= V (2 u + 2 e + 2^-19 + 2 T 2^-24). The lse: e + 2^-19 +
T 2^-24 + 2^-22 |lse|.
"""

from __future__ import annotations

import ctypes as C
import math
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch

from beamgrad_b200 import _abi as A
from beamgrad_b200.cache import PagedCache

ROOT = Path(__file__).resolve().parents[1]
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
ROUND = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-9}


# -- the boundary -----------------------------------------------------------------------


def test_struct_layout_matches_the_header(tmp_path):
    structs = {"DBSCudaCache": A.Cache, "DBSCudaAttendArgs": A.AttendArgs}
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "dbs_cuda_cache.h"', "int main(void) {"]
    for name, cls in structs.items():
        parts = [f"(int)sizeof({name})"] + [f"(int)offsetof({name}, {f[0]})" for f in cls._fields_]
        lines.append(f'  printf("{" ".join(["%d"] * len(parts))}\\n", {", ".join(parts)});')
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["  return 0;", "}"]))
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-I", str(ROOT / "include"), "-o", str(exe), str(src)], check=True)
    got = [[int(x) for x in line.split()] for line in subprocess.run([str(exe)], capture_output=True, text=True).stdout.splitlines()]
    assert got == [[C.sizeof(c)] + [getattr(c, f[0]).offset for f in c._fields_] for c in structs.values()]


def _sizes(**change) -> A.Cache:
    c = A.Cache()
    good = dict(batch_size=2, beam_size=3, max_pages=4, num_pages=30, num_layers=2, num_heads=2, head_dim=64,
                page_size=16, data_type=A.DTYPE_BF16)
    for name, value in (good | change).items():
        setattr(c, name, value)
    return c


def test_sizes_are_checked_without_a_device():
    lib = A.load()
    assert lib.dbs_cuda_cache_plan_bytes(C.byref(_sizes())) > 0
    for bad in (dict(batch_size=0), dict(beam_size=0), dict(beam_size=1025), dict(max_pages=0), dict(num_pages=-1),
                dict(num_layers=0), dict(num_heads=0), dict(head_dim=0), dict(head_dim=12), dict(head_dim=264),
                dict(page_size=24), dict(page_size=128), dict(data_type=3), dict(reserved0=1),
                dict(max_pages=2**26, page_size=64), dict(num_pages=2**30, num_heads=64)):
        assert lib.dbs_cuda_cache_plan_bytes(C.byref(_sizes(**bad))) < 0, bad
    assert lib.dbs_cuda_cache_plan_bytes(None) < 0
    # Arrays missing: refused before anything is launched.
    c = _sizes()
    assert lib.dbs_cuda_cache_fork(C.byref(c), None, None, 0, None, 0, None) == A.STATUS_INVALID_ARGUMENT
    assert lib.dbs_cuda_cache_compact(C.byref(c), None) == A.STATUS_INVALID_ARGUMENT
    assert lib.dbs_cuda_cache_refresh(C.byref(c), 1, None) == A.STATUS_INVALID_ARGUMENT
    assert lib.dbs_cuda_cache_commit(C.byref(c), None, 1, None, 0, None) == A.STATUS_INVALID_ARGUMENT
    a = A.AttendArgs(layer=0, beams=3, new_tokens=1, query_heads=4, scale=1.0)
    assert lib.dbs_cuda_cache_attend_workspace_size(C.byref(c), C.byref(a)) > 0
    assert lib.dbs_cuda_cache_attend(C.byref(c), C.byref(a), None) == A.STATUS_INVALID_ARGUMENT
    for bad in (dict(layer=2), dict(layer=-1), dict(beams=0), dict(beams=4), dict(new_tokens=0), dict(query_heads=3),
                dict(query_heads=0), dict(scale=math.nan), dict(reserved0=1)):
        good = dict(layer=0, beams=3, new_tokens=1, query_heads=4, scale=1.0)
        a = A.AttendArgs(**(good | bad))
        assert lib.dbs_cuda_cache_attend_workspace_size(C.byref(c), C.byref(a)) < 0, bad


def test_no_cpu_path():
    with pytest.raises(ValueError):
        PagedCache(1, 2, 10, num_layers=1, num_kv_heads=1, head_dim=64, device="cpu")
    with pytest.raises(ValueError):
        PagedCache(1, 2, 10, num_layers=1, num_kv_heads=1, head_dim=64, page_size=24, device="cuda:0")
    with pytest.raises(ValueError):
        PagedCache(1, 2, 10, num_layers=1, num_kv_heads=1, head_dim=64, dtype=torch.float64, device="cuda:0")
    z = torch.zeros
    with pytest.raises(ValueError):
        PagedCache.from_tensors(z(1, 2, 4, 1, 16, 64), z(1, 2, 3, dtype=torch.int32), z(1, 2, dtype=torch.int32))
    with pytest.raises(ValueError):
        PagedCache.from_tensors(z(1, 2, 4, 1, 16), z(1, 2, 3, dtype=torch.int32), z(1, 2, dtype=torch.int32))


# -- the state, page by page ------------------------------------------------------------


class Model:
    """The rules of include/dbs_cuda_cache.h, one page at a time."""

    def __init__(self, cache: PagedCache):
        self.pages = cache.pages.cpu().clone()
        self.table = cache.table.cpu().numpy().astype(np.int64)
        self.lengths = cache.lengths.cpu().numpy().astype(np.int64)
        self.B, self.K, self.M = self.table.shape
        self.P, self.page = cache.num_pages, cache.page_size

    def references(self):
        return np.bincount(self.table[self.table >= 0], minlength=self.P)

    def fork(self, parents=None, written=0, room=0):
        B, K, M, page = self.B, self.K, self.M, self.page
        parents = np.tile(np.arange(K), (B, 1)) if parents is None else parents
        written, room = np.broadcast_to(written, (B, K)), np.broadcast_to(room, (B, K))
        old, lengths = self.table.copy(), np.minimum(self.lengths + written, M * page)
        new, asks = np.full_like(old, -1), []
        for b in range(B):
            for s in range(K):
                r = parents[b, s]
                if r < 0 or r >= K:
                    self.lengths[b, s] = 0
                    continue
                n = self.lengths[b, s] = lengths[b, r]
                heir = r not in parents[b, :s]
                for c in range(min(M, -(-(n + room[b, s]) // page))):
                    if c < n // page or (heir and old[b, r, c] >= 0):
                        new[b, s, c] = old[b, r, c]
                    else:
                        rows = n % page if c == n // page and not heir else 0
                        asks.append((b, s, c, old[b, r, c], rows))
        self.table = new
        free = [p for p in range(self.P) if self.references()[p] == 0]
        before = self.pages.clone()
        for (b, s, c, source, rows), p in zip(asks, free):
            new[b, s, c] = p
            if source >= 0:
                self.pages[:, :, p, :, :rows] = before[:, :, source, :, :rows]

    def commit(self, path, counts, room=0):
        before = self.pages.clone()
        for b in range(self.B):
            for k in range(self.K):
                for a in range(counts[b, k]):
                    x, y = self.lengths[b, k] + path[b, k, a], self.lengths[b, k] + a
                    p, q = self.table[b, k, x // self.page], self.table[b, k, y // self.page]
                    self.pages[:, :, q, :, y % self.page] = before[:, :, p, :, x % self.page]
        self.fork(written=counts, room=room)

    def compact(self):
        refs = self.references()
        n = int((refs > 0).sum())
        holes, movers = [p for p in range(n) if refs[p] == 0], [p for p in range(n, self.P) if refs[p] > 0]
        for a, b in zip(movers, holes):
            self.pages[:, :, b] = self.pages[:, :, a]
            self.table[self.table == a] = b

    def check(self, cache: PagedCache):
        assert np.array_equal(cache.lengths.cpu().numpy(), self.lengths)
        assert np.array_equal(cache.table.cpu().numpy(), self.table)
        assert np.array_equal(cache.references.cpu().numpy(), self.references())
        ints = {4: torch.int32, 2: torch.int16}[self.pages.element_size()]
        assert torch.equal(cache.pages.cpu().view(ints), self.pages.view(ints))
        self.check_plan(cache)

    def check_plan(self, cache: PagedCache):
        """The plan lists every distinct page of each group of 32 beams once, in column order."""
        groups = -(-self.K // 32)
        cap = min(self.K, 32) * self.M
        words = cache._plan.cpu().numpy()
        up = lambda n: (n + 255) // 256 * 256  # noqa: E731
        counts = words[256 : 256 + self.B * groups * 4].view(np.int32)
        at = 256 + up(self.B * groups * 4)
        units = words[at : at + self.B * groups * cap * 16].view(np.int32).reshape(self.B * groups, cap, 4)
        for b in range(self.B):
            for g in range(groups):
                rows = self.table[b, 32 * g : 32 * g + 32]
                want = []
                for c in range(self.M):
                    for k in range(len(rows)):
                        p = rows[k, c]
                        if p < 0 or p in rows[:k, c]:
                            continue
                        held = [j for j in range(len(rows)) if rows[j, c] == p]
                        whole = all((c + 1) * self.page <= self.lengths[b, 32 * g + j] for j in held)
                        mask = sum(1 << j for j in held)
                        want.append((p, c * self.page, mask - (mask >> 31 << 32), -1 if whole else self.lengths[b, 32 * g + k]))
                n = counts[b * groups + g]
                assert [tuple(u) for u in units[b * groups + g, :n].tolist()] == want


def _fill(cache: PagedCache, seed: int):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    cache.pages.normal_(generator=gen)


STATES = [  # B, K, max_length, pages, layers, heads, dim, page, dtype
    (1, 1, 40, 8, 1, 1, 8, 16, torch.float32),
    (3, 4, 100, 90, 2, 3, 64, 16, torch.bfloat16),
    (2, 7, 200, 120, 3, 2, 80, 32, torch.float16),
    (2, 40, 150, 260, 1, 1, 24, 64, torch.float32),
    (5, 3, 1200, 700, 1, 2, 16, 16, torch.bfloat16),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", range(len(STATES)))
def test_a_search_of_forks_commits_and_compactions(case):
    B, K, T, P, L, H, D, page, dtype = STATES[case]
    rng = np.random.RandomState(case)
    cache = PagedCache(B, K, T, num_layers=L, num_kv_heads=H, head_dim=D, num_pages=P, page_size=page, dtype=dtype)
    _fill(cache, case)
    model = Model(cache)
    dev = lambda x: torch.from_numpy(np.ascontiguousarray(x)).cuda()  # noqa: E731
    # A prompt for beam 0 of each example, of another length each (one of them empty).
    prompt = np.zeros((B, K), np.int64)
    prompt[:, 0] = rng.randint(0, T // 2, B)
    cache.fork(room=dev(prompt))
    model.fork(room=prompt)
    model.check(cache)
    cache.fork(dev(np.zeros((B, K), np.int32)), written=dev(prompt.astype(np.int32)), room=1)
    model.fork(np.zeros((B, K), np.int64), prompt, 1)
    model.check(cache)
    for step in range(14):
        parents = rng.randint(0, K, (B, K))
        if step % 3 == 1:
            parents = np.minimum(parents, rng.randint(0, K, (B, K)))
        if step % 5 == 2:
            parents[rng.rand(B, K) < 0.3] = -1
        room = int(rng.choice([1, 1, 2, page, 0]))
        cache.fork(dev(parents), written=1 if step % 4 else 0, room=room)
        model.fork(parents, 1 if step % 4 else 0, room)
        model.check(cache)
        if step % 4 == 3:
            n = min(12, T // 8)
            cache.reserve(n)
            model.fork(room=n)
            counts = rng.randint(0, min(n, 6) + 1, (B, K))
            counts[model.lengths == 0] = 0
            path = np.sort(np.argsort(rng.rand(B, K, n), 2)[..., : max(1, counts.max())], 2)
            cache.commit(dev(path), dev(counts), room=1)
            model.commit(path, counts, 1)
            model.check(cache)
        if step % 5 == 4:
            cache.compact()
            model.compact()
            model.check(cache)
            assert int((cache.references > 0).sum()) == 0 or int((cache.references > 0).nonzero().max()) + 1 == int(
                (cache.references > 0).sum())
    cache.check()
    cache.release(torch.ones(B, dtype=torch.bool, device="cuda"))
    assert int(cache.references.sum()) == 0 and int((cache.table >= 0).sum()) == 0


@pytest.mark.gpu
def test_many_beams_and_long_tables():
    """More beams than a group holds, and more columns than a pass of the kernels takes."""
    for B, K, T, page in ((1, 1024, 64, 16), (2, 33, 9000, 16)):
        cache = PagedCache(B, K, T, num_layers=1, num_kv_heads=1, head_dim=8, num_pages=K * 4 + 6000, page_size=page,
                           dtype=torch.float16)
        _fill(cache, K)
        model = Model(cache)
        dev = lambda x: torch.from_numpy(np.ascontiguousarray(x)).cuda()  # noqa: E731
        rng = np.random.RandomState(K)
        prompt = np.zeros((B, K), np.int64)
        prompt[:, 0] = T // 2 + 3
        zero = np.zeros((B, K), np.int64)
        for parents, written, room in ((None, zero, prompt), (zero, prompt, zero + 1), (rng.randint(0, K, (B, K)), zero + 1, zero + 20)):
            cache.fork(None if parents is None else dev(parents), written=dev(written), room=dev(room))
            model.fork(parents, written, room)
        model.check(cache)
        cache.check()


@pytest.mark.gpu
def test_errors_of_the_device_are_reported():
    mk = lambda pages, T=64: PagedCache(1, 2, T, num_layers=1, num_kv_heads=1, head_dim=16, num_pages=pages, page_size=16)  # noqa: E731
    cache = mk(3)
    cache.reserve(33)  # two beams of three pages, three in the pool
    with pytest.raises(RuntimeError, match="ran out"):
        cache.check()
    assert cache.table.cpu().tolist()[0] == [[0, 1, 2, -1], [-1, -1, -1, -1]]
    cache.reset()
    cache.check()
    cache = mk(9, 32)
    cache.reserve(33)
    with pytest.raises(RuntimeError, match="outgrew"):
        cache.check()
    cache = mk(9)
    cache.fork(torch.tensor([[0, 2]], device="cuda"))
    with pytest.raises(RuntimeError, match="out of range"):
        cache.check()
    assert cache.lengths.cpu().tolist() == [[0, 0]] and cache.references.sum() == 1
    cache = mk(9)
    cache.reserve(8)
    cache.commit(torch.tensor([[[1, 1], [0, 1]]], device="cuda"), torch.tensor([[2, 2]], device="cuda"))
    with pytest.raises(RuntimeError, match="out of range"):
        cache.check()
    shared = torch.zeros((1, 2, 4), dtype=torch.int32, device="cuda")
    cache = PagedCache.from_tensors(mk(9).pages, shared, torch.full((1, 2), 5, dtype=torch.int32, device="cuda"))
    with pytest.raises(RuntimeError, match="shared"):
        cache.check()
    for call in (lambda: cache.fork(written=-1), lambda: cache.fork(room=-1), lambda: cache.fork(torch.zeros(1, 3, dtype=torch.int32, device="cuda")),
                 lambda: cache.fork(torch.zeros(1, 2, device="cuda")), lambda: cache.fork(torch.zeros(1, 2, dtype=torch.int32)),
                 lambda: cache.commit(torch.zeros(1, 2, dtype=torch.int32, device="cuda"), torch.zeros(1, 2, dtype=torch.int32, device="cuda"))):
        with pytest.raises(ValueError):
            call()


# -- the attention ----------------------------------------------------------------------


def attend_exact(pages, table, lengths, q, k, v, mask, counts, scale):
    """(out, lse, bound of out, bound of lse) in 64 bits; pages [2, P, H, page, D] before the call."""
    pages = pages.double()
    (B, K, N, Hq, D), H, page = q.shape, pages.shape[2], pages.shape[3]
    u = ROUND[q.dtype]
    q = q.double()
    out, lse = torch.zeros_like(q), torch.full(q.shape[:-1], -math.inf, dtype=torch.float64)
    bound, lse_bound = torch.zeros(q.shape[:-1], dtype=torch.float64), torch.zeros(q.shape[:-1], dtype=torch.float64)
    for b in range(B):
        for beam in range(K):
            n, fresh = int(lengths[b, beam]), int(counts[b, beam]) if counts is not None else N
            for j in range(fresh):
                col = (n + j) // page
                if k is not None and col < table.shape[2] and table[b, beam, col] >= 0:
                    p = int(table[b, beam, col])
                    pages[0, p, :, (n + j) % page], pages[1, p, :, (n + j) % page] = k[b, beam, j].double(), v[b, beam, j].double()
            held = [(int(table[b, beam, t // page]), t % page) for t in range(n + fresh) if t // page < table.shape[2]]
            if not held:
                continue
            there = torch.tensor([p >= 0 for p, _ in held])
            rows = pages[:, [max(p, 0) for p, _ in held], :, [o for _, o in held]]  # [T, 2, H, D]
            for i in range(fresh):
                see = there.clone()
                for j in range(fresh):
                    if n + j < len(held):
                        see[n + j] &= bool(mask[b, beam, i, j]) if mask is not None else j <= i
                if not see.any():
                    continue
                for h in range(Hq):
                    keys, values = rows[see, 0, h // (Hq // H)], rows[see, 1, h // (Hq // H)]
                    x = (keys @ q[b, beam, i, h]) * scale
                    lse[b, beam, i, h] = torch.logsumexp(x, 0)
                    out[b, beam, i, h] = torch.softmax(x, 0) @ values
                    e = (D + 4) * 2.0**-24 * abs(scale) * float((keys.abs() @ q[b, beam, i, h].abs()).max()) + 2.0**-22 * float(x.abs().max())
                    T = len(x)
                    bound[b, beam, i, h] = float(values.abs().max()) * (2 * u + 2 * e + 2.0**-19 + 2 * T * 2.0**-24)
                    lse_bound[b, beam, i, h] = e + 2.0**-19 + T * 2.0**-24 + 2.0**-22 * abs(float(lse[b, beam, i, h]))
    return out, lse, bound, lse_bound


def check_attend(cache, layer, q, k, v, mask=None, counts=None, scale=None):
    before = cache.pages[layer].cpu().clone()
    out, lse = cache.attend(layer, q, k, v, mask=mask, counts=counts, scale=scale, return_lse=True)
    cpu = lambda x: None if x is None else x.cpu()  # noqa: E731
    want, z, bound, z_bound = attend_exact(before, cache.table.cpu(), cache.lengths.cpu(), cpu(q), cpu(k), cpu(v), cpu(mask),
                                           cpu(counts), 1 / math.sqrt(q.shape[-1]) if scale is None else scale)
    got, got_z = out.cpu().double(), lse.cpu().double()
    empty = torch.isinf(z)
    assert torch.equal(torch.isinf(got_z), empty) and bool((got[empty] == 0).all())
    off = (got - want).abs().amax(-1)
    assert bool((off <= bound).all()), float((off - bound).max())
    off = (got_z - z)[~empty].abs()
    assert bool((off <= z_bound[~empty]).all()), float((off - z_bound[~empty]).max())
    # The new rows are in their pages, and nothing else changed.
    after = cache.pages[layer].cpu()
    table, lengths = cache.table.cpu(), cache.lengths.cpu()
    if k is not None:
        for b in range(q.shape[0]):
            for beam in range(q.shape[1]):
                for j in range(int(counts[b, beam]) if counts is not None else q.shape[2]):
                    t = int(lengths[b, beam]) + j
                    if t // cache.page_size < table.shape[2] and (p := int(table[b, beam, t // cache.page_size])) >= 0:
                        before[0, p, :, t % cache.page_size], before[1, p, :, t % cache.page_size] = k[b, beam, j], v[b, beam, j]
    assert torch.equal(after, before)
    return out, lse


def random_cache(B, K, lengths, new, *, layers=2, heads=2, dim=64, page=16, dtype=torch.bfloat16, seed=0, spare=5):
    """A cache whose beams share pages as a search leaves them: forked at random at several lengths."""
    rng = np.random.RandomState(seed)
    T = int(np.max(lengths)) + new + 2 * page
    cache = PagedCache(B, K, T, num_layers=layers, num_kv_heads=heads, head_dim=dim, page_size=page, dtype=dtype,
                       num_pages=B * K * (-(-T // page)) + spare)
    _fill(cache, seed)
    # Random page numbers: pages are handed out lowest first, so hold some back at first.
    dev = lambda x: torch.from_numpy(np.ascontiguousarray(x)).cuda()  # noqa: E731
    lengths = np.broadcast_to(lengths, (B, K)).astype(np.int32)
    done = np.zeros((B, K), np.int32)
    parts = 4
    for i in range(parts):
        goal = lengths.min(1, keepdims=True) * (i + 1) // parts + np.zeros_like(done) if i + 1 < parts else lengths
        step = np.maximum(goal - done, 0).astype(np.int32)
        cache.reserve(dev(step))
        parents = np.minimum(rng.randint(0, K, (B, K)), rng.randint(0, K, (B, K))) if i + 1 < parts else np.tile(np.arange(K), (B, 1))
        cache.fork(dev(parents), written=dev(step), room=new)
        done = goal
    assert np.array_equal(cache.lengths.cpu().numpy(), lengths)
    cache.check()
    return cache


def draft_tree(B, K, N, rng):
    mask = np.zeros((B, K, N, N), bool)
    for b in range(B):
        for k in range(K):
            for i in range(N):
                if i:
                    mask[b, k, i] = mask[b, k, rng.randint(0, i)] if rng.rand() < 0.9 else False
                mask[b, k, i, i] = True
    return torch.from_numpy(mask).cuda()


def tensors(cache, N, group, seed, beams=None, spread=2.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    shape = (cache.batch_size, beams or cache.beam_size, N)
    mk = lambda h: torch.randn((*shape, h, cache.head_dim), generator=gen, device="cuda")  # noqa: E731
    return [(mk(h) * s).to(cache.dtype) for h, s in ((cache.num_kv_heads * group, spread), (cache.num_kv_heads, 1), (cache.num_kv_heads, 1))]


ATTEND = [  # B, K, length, N, heads, group, dim, page, tree
    (1, 1, 0, 1, 1, 1, 8, 16, False),      # nothing cached, one token
    (1, 4, 1, 1, 2, 4, 64, 16, False),
    (2, 3, 15, 1, 2, 3, 64, 16, False),
    (2, 8, 130, 1, 2, 4, 128, 32, False),
    (3, 5, 700, 1, 1, 8, 128, 64, False),  # 40 rows a group
    (1, 33, 90, 1, 2, 2, 64, 32, False),   # two groups of beams
    (2, 2, 63, 2, 3, 5, 80, 64, False),
    (1, 3, 257, 5, 2, 1, 96, 16, True),
    (2, 1, 300, 16, 2, 4, 128, 32, True),  # 64 rows
    (1, 1, 190, 40, 1, 8, 128, 64, True),  # 320 rows
    (1, 2, 64, 33, 1, 3, 64, 64, False),   # a chain that ends in another page
    (1, 1, 31, 17, 2, 2, 72, 16, True),
    (1, 2, 100, 3, 1, 2, 256, 32, True),
    (1, 4, 70, 1, 1, 16, 200, 16, False),
    (2, 5, 100, 20, 2, 4, 64, 16, True),   # blocks of rows that hold a beam and a part of others
    (1, 3, 530, 70, 1, 2, 128, 32, True),  # a beam fills more than a block
    (1, 32, 40, 33, 1, 4, 64, 16, False),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", range(len(ATTEND)))
def test_attend(case, dtype):
    B, K, T, N, H, G, D, page, tree = ATTEND[case]
    rng = np.random.RandomState(case)
    lengths = np.maximum(0, T - rng.randint(0, max(1, T // 3 + 1), (B, 1)) - rng.randint(0, min(T, 3) + 1, (B, K)) * (case % 2))
    cache = random_cache(B, K, lengths, N, heads=H, dim=D, page=page, dtype=dtype, seed=case)
    q, k, v = tensors(cache, N, G, 100 + case)
    mask = draft_tree(B, K, N, rng) if tree else None
    check_attend(cache, 1, q, k, v, mask)
    out, lse = cache.attend(1, q, mask=mask, return_lse=True)  # the positions hold the tokens already
    again = cache.attend(1, q, k, v, mask=mask, return_lse=True)
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_attend_empty_rows_counts_and_missing_pages(dtype):
    B, K, N, H, G = 2, 3, 4, 2, 2
    lengths = np.array([[0, 40, 17], [33, 0, 0]])
    cache = random_cache(B, K, lengths, N, heads=H, dtype=dtype, seed=3)
    q, k, v = tensors(cache, N, G, 5)
    mask = torch.ones((B, K, N, N), dtype=torch.bool, device="cuda")
    mask[0, 0] = False           # nothing cached either: rows that see nothing
    mask[1, 1, 2] = False
    counts = torch.tensor([[4, 0, 2], [1, 3, 4]], dtype=torch.int32, device="cuda")
    check_attend(cache, 0, q, k, v, mask, counts)
    check_attend(cache, 1, q, k, v, None, counts)
    # An emptied beam has no pages: its new tokens are not written and not seen.
    cache.fork(torch.tensor([[0, -1, 1], [-1, -1, 0]], device="cuda"), room=N)
    out, lse = check_attend(cache, 0, q, k, v, mask)
    assert bool((out[0, 1] == 0).all()) and bool(torch.isinf(lse[1, :2]).all())
    # No pages for the new tokens of the beams that have some cached.
    cache.fork(room=0)
    check_attend(cache, 0, q, k, v)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N", [3, 40])
def test_values_that_are_not_finite_stay_where_they_are_seen(dtype, N):
    """NaN and infinities in keys and values of tokens that a row does not see, of pages that other
    beams hold, and of rows nobody committed."""
    B, K, H, G = 2, 4, 1, 3
    cache = random_cache(B, K, np.full((B, K), 50), N, heads=H, dtype=dtype, seed=9)
    q, k, v = tensors(cache, N, G, 11)
    mask = draft_tree(B, K, N, np.random.RandomState(2))
    mask[:, :, 1:, 0] = False                      # token 0 is seen by itself alone
    mask[0, 1, :, 2] = False                       # token 2 of this beam by nobody
    good = cache.attend(0, q, k, v, mask=mask, return_lse=True)
    bad_k, bad_v = k.clone(), v.clone()
    bad_k[:, 1:, 0], bad_v[:, 1:, 0] = math.nan, math.inf
    bad_k[0, 1, 2], bad_v[0, 1, 2] = -math.inf, math.nan
    bad_v[1, 2, :, :, 3] = math.inf                # one beam's own values: the others do not see it
    out, lse = cache.attend(0, q, bad_k, bad_v, mask=mask, return_lse=True)
    clean = torch.ones((B, K, N), dtype=torch.bool)
    clean[:, 1:, 0] = False
    clean[0, 1, 2] = bool(mask[0, 1, 2, 2])
    clean[1, 2] = False
    tol = {torch.float32: 1e-5, torch.float16: 2e-3, torch.bfloat16: 1.6e-2}[dtype]  # two ways of summing, each rounded once
    assert float((out.cpu()[clean].float() - good[0].cpu()[clean].float()).abs().max()) < tol * 4
    assert float((lse.cpu()[clean] - good[1].cpu()[clean]).abs().max()) < 1e-4
    seen = out[1, 2, 1:].float()
    finite = [d for d in range(cache.head_dim) if d != 3]
    assert not bool(torch.isfinite(seen[..., 3]).any()) and bool(torch.isfinite(seen[..., finite]).all())
    assert bool(torch.isnan(out[0, 2, 0]).all())
    # Rows behind the committed tokens hold them now; the next token's page shows none of it.
    cache.fork(torch.tensor([[0, 0, 0, 0]] * B, device="cuda"), room=1)
    q1, k1, v1 = tensors(cache, 1, G, 12)
    assert bool(torch.isfinite(cache.attend(0, q1, k1, v1)).all())


@pytest.mark.gpu
def test_infinite_scores():
    """Scores of -inf leave a row empty (weight 0 everywhere), as an exact softmax over nothing; very
    large scores do not overflow."""
    cache = random_cache(1, 2, np.full((1, 2), 20), 2, heads=1, dtype=torch.bfloat16, seed=1)
    q, k, v = tensors(cache, 2, 2, 3, spread=300.0)
    check_attend(cache, 0, q, k, v)
    check_attend(cache, 0, q, k, v, scale=0.0)
    check_attend(cache, 0, q, k, v, scale=-0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N, dim", [(1, 128), (16, 64), (31, 256), (40, 64), (64, 128), (72, 200), (130, 128), (300, 64)])
def test_divided_segments_stay_in_their_workspace(N, dim, dtype):
    # 1800 pages by heads: every CTA has parts of segments, and the last one's lie last in the workspace.
    cache = random_cache(1, 1, np.full((1, 1), 14400), N, layers=1, heads=8, dim=dim, page=64, dtype=dtype, seed=N)
    q, k, v = tensors(cache, N, 1, N)
    cache.attend(0, q[:, :, :1], k[:, :, :1], v[:, :, :1])
    (stream, workspace), = cache._workspaces.items()
    behind = 4 << 20
    guarded = torch.zeros(workspace.numel() + behind, dtype=torch.uint8, device="cuda")
    guarded[-behind:] = 0x5A
    cache._workspaces[stream] = guarded[:-behind]
    check_attend(cache, 0, q, k, v)
    assert cache._workspaces[stream].data_ptr() == guarded.data_ptr()
    assert bool((guarded[-behind:] == 0x5A).all())


@pytest.mark.gpu
def test_strides_streams_and_fewer_beams():
    B, K, N, H, G, D = 2, 4, 3, 2, 3, 64
    cache = random_cache(B, K, np.full((B, K), 37), N, heads=H, dtype=torch.float16, seed=4)
    fused = torch.randn((B, N, K, H * (G + 2), D), device="cuda").half().transpose(1, 2)
    q, k, v = fused[..., : H * G, :], fused[..., H * G : H * (G + 1), :], fused[..., H * (G + 1) :, :]
    want, _ = check_attend(cache, 0, q, k, v)
    odd = torch.empty(B * K * N * H * G * D + 1, device="cuda", dtype=torch.float16)[1:].view(q.shape)
    odd.copy_(q)  # not on a 16-byte boundary
    assert torch.equal(cache.attend(0, odd, k, v), want)
    assert torch.equal(cache.attend(0, q.transpose(3, 4).contiguous().transpose(3, 4), k, v), want)
    out = torch.empty_like(want)
    assert cache.attend(0, q, k, v, out=out) is out and torch.equal(out, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = cache.attend(0, q, k, v)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, want)
    check_attend(cache, 1, q[:, :1], k[:, :1], v[:, :1])
    check_attend(cache, 1, q[:, :3], k[:, :3], v[:, :3], draft_tree(B, 3, N, np.random.RandomState(0)))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, N, group", [(torch.bfloat16, 1, 4), (torch.float16, 12, 8), (torch.float32, 5, 3)])
def test_a_step_in_a_cuda_graph(dtype, N, group):
    B, K = 2, 4
    graphed, plain = (random_cache(B, K, np.full((B, K), 700), N, dtype=dtype, seed=6) for _ in range(2))
    inputs = [tensors(graphed, N, group, 40 + i) for i in range(4)]
    parents = [torch.randint(0, K, (B, K), device="cuda", dtype=torch.int32) for _ in range(4)]
    static, static_parents = [x.clone() for x in inputs[0]], parents[0].clone()

    def step(cache, q, k, v, by):
        outs = [cache.attend(layer, q, k, v) for layer in range(2)]
        cache.fork(by, written=1, room=N)
        return outs

    step(graphed, *static, static_parents)  # not in the graph: shapes are checked once
    step(plain, *inputs[0], parents[0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(graphed, *static, static_parents)
    for i in range(1, 4):
        for x, y in zip(static, inputs[i]):
            x.copy_(y)
        static_parents.copy_(parents[i])
        graph.replay()
        want = step(plain, *inputs[i], parents[i])
        for x, y in zip(got, want):
            assert torch.equal(x, y)
        assert torch.equal(graphed.table, plain.table) and torch.equal(graphed.lengths, plain.lengths)
    graphed.check()


@pytest.mark.gpu
def test_attend_refusals():
    cache = PagedCache(2, 3, 64, num_layers=2, num_kv_heads=2, head_dim=64, page_size=16)
    q, k, v = tensors(cache, 2, 2, 0)
    ok = torch.ones((2, 3, 2, 2), dtype=torch.bool, device="cuda")
    for args, options in (((2, q, k, v), {}), ((-1, q, k, v), {}), ((0, q[..., :32], k, v), {}), ((0, q[:, :, :, :3], k, v), {}),
                          ((0, q, k, None), {}), ((0, q, k[:, :2], v[:, :2]), {}), ((0, q.float(), k, v), {}), ((0, q.cpu(), k, v), {}),
                          ((0, q[:1], k[:1], v[:1]), {}), ((0, q[0], k, v), {}), ((0, q, k, v), dict(mask=ok.float())),
                          ((0, q, k, v), dict(mask=ok[..., :1])), ((0, q, k, v), dict(mask=ok.cpu())),
                          ((0, q, k, v), dict(counts=torch.ones(2, 2, dtype=torch.int32, device="cuda"))),
                          ((0, q, k, v), dict(scale=math.inf)), ((0, q, k, v), dict(out=torch.empty_like(q).float()))):
        with pytest.raises(ValueError):
            cache.attend(*args, **options)
    with pytest.raises(RuntimeError, match="backward"):
        cache.attend(0, q.clone().requires_grad_(), k, v)
    cache.check()
