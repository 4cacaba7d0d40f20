# SPDX-License-Identifier: MIT
"""Performance cases of the paged beam cache and its attention.

A case is one pass through one operator: ``fork`` (beams reordered after a search step),
``commit`` (the accepted path of a drafted tree), ``compact`` (defragmentation of the pool) or
``attend`` (new tokens written and attended over the cache). With ``own`` false, :func:`run`
computes it with elementary torch operations in 32 bits; with ``own`` true, by
:class:`beamgrad_b200.cache.PagedCache`.

State of a cache: ``pages`` [L, 2, P, H, page, D] (keys, values), ``table`` [B, K, M] (page of each
column of each beam, -1 for none), ``lengths`` [B, K], ``references`` [P] (table entries that name
the page).
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # One sentence, four beams, a small model: launch latency is all there is.
        dict(name="fork_small", op="fork", dtype="f32", batch=1, beams=4, layers=4, heads=2, dim=64, page=16,
             prompt=20, private=19, ragged=False),
        # The beam decode of a batch of 64 with 8 beams, part of a model's layers.
        dict(name="fork_beams", op="fork", dtype="bf16", batch=64, beams=8, layers=4, heads=8, dim=128, page=32,
             prompt=256, private=40, ragged=True),
        # Wide beams, larger pages, more layers: the copies of partial pages dominate.
        dict(name="fork_wide", op="fork", dtype="f16", batch=16, beams=32, layers=16, heads=4, dim=128, page=64,
             prompt=500, private=50, ragged=True),
        # A short draft of one sequence.
        dict(name="commit_small", op="commit", dtype="bf16", batch=1, beams=1, layers=4, heads=2, dim=64, page=16,
             prompt=77, private=0, new=8, ragged=False),
        # Drafted trees of 32 tokens for a batch of 64, all layers of a mid-sized model.
        dict(name="commit_batch", op="commit", dtype="bf16", batch=64, beams=1, layers=16, heads=8, dim=128, page=32,
             prompt=200, private=0, new=32, ragged=True),
        # A small pool with few holes.
        dict(name="compact_small", op="compact", dtype="f16", batch=2, beams=3, layers=2, heads=2, dim=80, page=16,
             prompt=100, private=25, ragged=True),
        # A pool of about a gigabyte, half of it free.
        dict(name="compact_large", op="compact", dtype="bf16", batch=32, beams=4, layers=8, heads=8, dim=128, page=32,
             prompt=400, private=60, ragged=True),
        # One token a beam over a short cache: the smallest call of a decode loop.
        dict(name="attend_small", op="attend", dtype="f16", batch=1, beams=4, group=4, heads=2, dim=64, page=16,
             prompt=60, private=19, new=1, tree=False, ragged=False),
        # The beam decode of a batch of 64 with 8 beams after a prompt of 512.
        dict(name="attend_beams", op="attend", dtype="bf16", batch=64, beams=8, group=4, heads=8, dim=128, page=32,
             prompt=512, private=64, new=1, tree=False, ragged=True),
        # Few long documents, eight beams each.
        dict(name="attend_long", op="attend", dtype="bf16", batch=4, beams=8, group=4, heads=8, dim=128, page=64,
             prompt=32000, private=100, new=1, tree=False, ragged=True),
        # Drafted trees of 64 tokens checked against a cache of 8000, eight query heads a key head.
        dict(name="attend_tree", op="attend", dtype="bf16", batch=16, beams=1, group=8, heads=8, dim=128, page=64,
             prompt=8000, private=0, new=64, tree=True, ragged=True),
        # Odd everything, in 32 bits: three beams with three drafted tokens each, heads of 80.
        dict(name="attend_odd", op="attend", dtype="f32", batch=5, beams=3, group=3, heads=5, dim=80, page=16,
             prompt=701, private=37, new=3, tree=True, ragged=True),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """A case of the listed ones' ranges, within the largest one's bytes and operations."""
    while True:
        op = rng.choice(("fork", "commit", "compact", "attend", "attend", "attend"))
        case = dict(op=op, dtype=rng.choice(("f32", "f16", "bf16", "bf16")), batch=_log_int(rng, 1, 64),
                    beams=1 if op == "commit" else _log_int(rng, 1, 32), heads=rng.choice((1, 2, 3, 4, 5, 8)),
                    dim=rng.choice((64, 80, 96, 128, 128)), page=rng.choice((16, 32, 64)),
                    prompt=_log_int(rng, 1, 32000 if op == "attend" else 600), private=_log_int(rng, 1, 100),
                    ragged=rng.random() < 0.7)
        if op == "attend":
            case |= dict(group=rng.choice((1, 2, 3, 4, 8)), new=1 if rng.random() < 0.5 else _log_int(rng, 2, 64),
                         tree=rng.random() < 0.7)
            if case["new"] == 1:
                case["tree"] = False
        else:
            case["layers"] = _log_int(rng, 1, 16)
        if op == "commit":
            case |= dict(new=_log_int(rng, 2, 32), private=0)
        lengths, _, owner = _layout(case)
        rows = (owner == np.arange(case["beams"])[None, :, None]).sum() * case["page"]
        room = rows * case.get("layers", 1) * case["heads"] * case["dim"] * 2 * _bytes_of(case)
        gathered = lengths.size * (lengths.max() + 1) * case["heads"] * case["dim"] * 4
        w = work(case)
        limit = 35e9 if case["dtype"] == "f32" else 275e9  # operations: 32-bit products have no tensor cores
        if room < 1.6e9 and gathered < 5e9 and w["bytes"] < 6e8 and w["flops"] < limit:
            return case


def _bytes_of(case):
    return 4 if case["dtype"] == "f32" else 2


def _layout(case):
    """Lengths [B, K], columns in use [B, K] and which beam's page each column is ([B, K, M], -1:
    none): the prompt's pages belong to all beams, then come pages shared by pairs, then each
    beam's own."""
    B, K, page = case["batch"], case["beams"], case["page"]
    b, k = np.arange(B)[:, None], np.arange(K)[None, :]
    prompt = case["prompt"] - ((b * 37) % max(1, case["prompt"] // 4) if case["ragged"] else 0) + 0 * (b + k)
    private = case["private"] - ((b * 5 + k // 2 * 3) % max(1, case["private"] // 3) if case["ragged"] else 0)
    lengths = np.maximum(prompt + private, 1)
    used = -(-(lengths + case.get("new", 1)) // page)
    trunk = np.minimum(prompt, lengths) // page
    pairs = np.maximum(trunk, (prompt + private // 2) // page)
    c = np.arange(int(used.max()))[None, None, :]
    owner = np.where(c < trunk[..., None], 0, np.where(c < pairs[..., None], (k // 2 * 2)[..., None], k[..., None]))
    return lengths, used, np.where(c < used[..., None], owner, -1)


def _tree(case):
    """parent [B * K, N] of every drafted token (-1: none), the same for every seed."""
    S, N = case["batch"] * case["beams"], case["new"]
    r = np.random.RandomState(11)
    i = np.arange(N)[None, :]
    return np.where(i == 0, -1, np.floor(r.rand(S, N) * i)).astype(np.int64)


def _visible(case):
    """mask [B, K, N, N]: whether drafted token i sees drafted token j (its ancestors and itself)."""
    parent = _tree(case)
    S, N = parent.shape
    mask = np.zeros((S, N, N), bool)
    at = np.broadcast_to(np.arange(N), (S, N)).copy()
    s, i = np.arange(S)[:, None], np.arange(N)[None, :]
    for _ in range(N):
        mask[s, i, np.maximum(at, 0)] |= at >= 0
        at = np.where(at >= 0, parent[s, np.maximum(at, 0)], -1)
    return mask.reshape(case["batch"], case["beams"], N, N)


def _counts(case):
    """Accepted tokens [B, K] of a commit."""
    S = case["batch"] * case["beams"]
    return (np.arange(S).reshape(case["batch"], case["beams"]) * 7 + 3) % min(case["new"], 8) + 1


def prepare(case, seed):
    device, dtype = "cuda", _DTYPES[case["dtype"]]
    gen = torch.Generator(device=device).manual_seed(seed)
    host = np.random.RandomState(seed % (1 << 32))
    B, K, H, D, page = case["batch"], case["beams"], case["heads"], case["dim"], case["page"]
    L = case.get("layers", 2)
    lengths, used, owner = _layout(case)
    M = owner.shape[2] + 1
    # Pages at random places of the pool: each distinct one once.
    mine = owner == np.arange(K)[None, :, None]
    live = int(mine.sum())
    P = live * 2 + 3 if case["op"] == "compact" else live + B * K * (1 + -(-case.get("new", 1) // page)) + 3
    number = np.zeros(owner.shape, np.int64)
    number[mine] = host.permutation(P)[:live]
    table = np.full((B, K, M), -1, np.int64)
    table[..., :-1] = np.where(owner >= 0, np.take_along_axis(number, np.maximum(owner, 0), 1), -1)
    references = np.bincount(table[table >= 0], minlength=P)
    pages = torch.empty((L, 2, P, H, page, D), dtype=dtype, device=device)
    pages.normal_(generator=gen)
    put = lambda x, t=torch.int32: torch.from_numpy(np.ascontiguousarray(x)).to(device, t)  # noqa: E731
    s = dict(case=case, pages=pages, table=put(table), lengths=put(lengths), references=put(references))
    if case["op"] == "fork":  # parents as a search gives them: better beams have more children
        s["parents"] = put(np.minimum(host.randint(0, K, (B, K)), host.randint(0, K, (B, K))))
    if case["op"] == "commit":  # a path down the tree, from the root
        counts, N = _counts(case), case["new"]
        ranks = np.sort(np.argsort(host.rand(B, K, N - 1), 2)[..., : max(0, counts.max() - 1)] + 1, 2)
        path = np.concatenate([np.zeros((B, K, 1), np.int64), ranks], 2)
        s |= dict(path=put(path), counts=put(counts))
    if case["op"] == "attend":
        N, G = case["new"], case["group"]
        # One fused projection's output, [B, K, N, (H * G + 2 * H) * D]: q, k, v are views of it.
        qkv = torch.randn((B, K, N, H * (G + 2), D), generator=gen, device=device).to(dtype)
        qkv[..., : H * G, :] *= 2  # scores with a spread of about two
        s |= dict(q=qkv[..., : H * G, :], k=qkv[..., H * G : H * (G + 1), :], v=qkv[..., H * (G + 1) :, :],
                  mask=put(_visible(case), torch.bool) if case["tree"] else None)
    s["start"] = tuple(s[x].clone() for x in ("table", "lengths", "references"))
    if own:
        from beamgrad_b200.cache import PagedCache

        s["cache"] = PagedCache.from_tensors(s["pages"], s["table"], s["lengths"], s["references"])
    return s


def run(s):
    op, layer = s["case"]["op"], 1
    if op == "attend":
        if own:
            out, lse = s["cache"].attend(layer, s["q"], s["k"], s["v"], mask=s["mask"], return_lse=True)
        else:
            out, lse = _attend(s, layer)
        return dict(out=out, lse=lse, pages=s["pages"][layer])
    # The same start for every pass: lengths would grow, and a pool is compact after one pass.
    for x, y in zip(("table", "lengths", "references"), s["start"]):
        s[x].copy_(y)
    if op == "fork":
        if own:
            s["cache"].fork(s["parents"], room=1)
        else:
            _fork(s, s["parents"], 0, 1)
    elif op == "commit":
        if own:
            s["cache"].commit(s["path"], s["counts"], room=s["case"]["new"])
        else:
            _commit(s, s["path"], s["counts"], s["case"]["new"])
    else:
        if own:
            s["cache"].compact()
        else:
            _compact(s)
    return {x: s[x] for x in ("table", "lengths", "references", "pages")}


# -- the operators in elementary operations ---------------------------------------------


def _fork(s, parents, written, room):
    pages, table, lengths, references = s["pages"], s["table"], s["lengths"], s["references"]
    (B, K, M), P, page = table.shape, references.numel(), pages.shape[4]
    S, device = B * K, table.device
    slot, col = torch.arange(S, device=device), torch.arange(M, device=device)
    has = parents.reshape(-1) >= 0
    src = (slot // K * K + parents.reshape(-1)).where(has, slot)
    length = torch.where(has, (lengths + written).reshape(-1)[src], 0)
    need = torch.where(has, (length + room + page - 1) // page, 0)[:, None]
    first = torch.full((S,), S, device=device).scatter_reduce(0, src, torch.where(has, slot, S), "amin")
    first = has & (first[src] == slot)
    old = table.reshape(S, M)[src].long()
    full = (length // page)[:, None]
    kept = torch.where((col < need) & ((col < full) | first[:, None]), old, -1)
    wants = (col >= full) & (col < need) & (kept < 0)
    count = lambda t: torch.zeros(P + 1, dtype=torch.long, device=device).index_add_(  # noqa: E731
        0, torch.where(t >= 0, t, P).reshape(-1), torch.ones(S * M, dtype=torch.long, device=device))[:P]
    taken = count(kept) > 0
    order = torch.argsort(taken.int(), stable=True)  # the free pages first, lowest first
    rank = wants.reshape(-1).cumsum(0).reshape(S, M) - 1
    given = torch.where(rank < P - taken.sum(), order[rank.clamp(0, P - 1)], -1)
    new = torch.where(wants, given, kept)
    rows = length % page
    at = (length // page).clamp(max=M - 1)[:, None]
    a, b = old.gather(1, at)[:, 0], new.gather(1, at)[:, 0]
    pick = (has & ~first & (rows > 0) & (a >= 0) & (b >= 0)).nonzero()[:, 0]
    inside = torch.arange(page, device=device)[:, None] < rows[pick][:, None, None, None]
    pages[:, :, b[pick]] = torch.where(inside, pages[:, :, a[pick]], pages[:, :, b[pick]])
    table.copy_(new.reshape(B, K, M))
    lengths.copy_(length.reshape(B, K))
    references.copy_(count(new))


def _commit(s, path, counts, room):
    pages, table, lengths = s["pages"], s["table"], s["lengths"]
    (B, K, M), page = table.shape, pages.shape[4]
    a = torch.arange(path.shape[2], device=table.device)
    base = lengths.long()[..., None]
    source, target = base + path, base + a
    find = lambda x: table.long().gather(2, (x // page).clamp(max=M - 1))  # noqa: E731
    moves = (a < counts[..., None]) & (find(source) >= 0) & (find(target) >= 0)
    source, target, p, q = source[moves], target[moves], find(source)[moves], find(target)[moves]
    pages[:, :, q, :, target % page] = pages[:, :, p, :, source % page]
    identity = torch.arange(K, device=table.device).expand(B, K)
    _fork(s, identity, counts, room)


def _compact(s):
    pages, table, references = s["pages"], s["table"], s["references"]
    P = references.numel()
    live, index = references > 0, torch.arange(P, device=table.device)
    n = live.sum()
    holes, movers = (~live & (index < n)).nonzero()[:, 0], (live & (index >= n)).nonzero()[:, 0]
    pages[:, :, holes] = pages[:, :, movers]
    to = index.index_copy(0, movers, holes)
    table.copy_(torch.where(table >= 0, to[table.clamp(min=0).long()], -1))
    references[holes] = references[movers]
    references[movers] = 0


def _attend(s, layer):
    pages, table, lengths = s["pages"], s["table"].long(), s["lengths"].long()
    q, k, v = s["q"], s["k"], s["v"]
    (B, K, N, Hq, D), H, page = q.shape, k.shape[3], pages.shape[4]
    M, S, device = table.shape[2], B * K, q.device
    place = lengths[..., None] + torch.arange(N, device=device)  # [B, K, N]
    where = table.gather(2, (place // page).clamp(max=M - 1))
    ok = (where >= 0) & (place // page < M)
    for i, x in enumerate((k, v)):
        pages[layer, i][where[ok], :, place[ok] % page] = x[ok]
    span = int(s["case"]["prompt"] + s["case"]["private"] + N + page)  # no length is above this
    cols = min(M, -(-span // page))
    kv = pages[layer][:, table[..., :cols].reshape(S, cols).clamp(min=0)].float()  # [2, S, cols, H, page, D]
    keys, values = (x.permute(0, 2, 1, 3, 4).reshape(S, H, cols * page, D) for x in kv)
    at = torch.arange(cols * page, device=device)
    j = at - lengths.reshape(S, 1)  # [S, T]: index among the new tokens
    if s["mask"] is None:
        fresh = j[:, None, :] <= torch.arange(N, device=device)[:, None]
    else:
        fresh = s["mask"].reshape(S, N, N).gather(2, j.clamp(0, N - 1)[:, None, :].expand(S, N, -1)) & (j < N)[:, None]
    sees = (fresh | (j < 0)[:, None, :]) & (table[..., :cols].reshape(S, cols, 1) >= 0).expand(S, cols, page).reshape(S, 1, -1)
    rows = q.float().reshape(S, N, H, Hq // H, D).permute(0, 2, 3, 1, 4).reshape(S, H, Hq // H * N, D)
    scores = (rows @ keys.transpose(2, 3)) * (1 / math.sqrt(D))
    scores = scores.view(S, H, Hq // H, N, -1).masked_fill(~sees[:, None, None], float("-inf"))
    top = scores.amax(-1, keepdim=True).clamp(min=-3e38)
    weights = torch.exp(scores - top)
    total = weights.sum(-1, keepdim=True)
    out = (weights.view(S, H, Hq // H * N, -1) @ values).view(S, H, Hq // H, N, D) / total.clamp(min=1e-38)
    lse = (total.log() + top)[..., 0]
    back = lambda x, *d: x.permute(0, 3, 1, 2, *d).reshape(B, K, N, Hq, *x.shape[4:])  # noqa: E731
    return back(out, 4).to(q.dtype), back(lse)


def work(case):
    """Bytes and operations of one pass: state and data in and out once."""
    return {name: float(value) for name, value in _work(case).items()}


def _work(case):
    lengths, used, owner = _layout(case)
    B, K, H, D, page = case["batch"], case["beams"], case["heads"], case["dim"], case["page"]
    size, entries = _bytes_of(case), int(used.sum())
    row = 2 * H * D * size * case.get("layers", 1)  # one token's keys and values
    own_pages = owner == np.arange(K)[None, :, None]
    live = int(own_pages.sum())
    if case["op"] == "fork":
        # On average a beam in three is not the first child of its parent and copies its last page.
        copies = (lengths % page).sum() * _repeats(K)
        return dict(bytes=8 * entries + 8 * live + 2 * copies * row, flops=0)
    if case["op"] == "commit":
        moved = _counts(case).sum() - B * K  # the root stays
        return dict(bytes=8 * entries + 8 * live + 2 * moved * row, flops=0)
    if case["op"] == "compact":  # half of the pool is live, at random: half of that moves
        return dict(bytes=8 * entries + 16 * live + 2 * (live / 2) * page * row, flops=0)
    N, G = case["new"], case["group"]
    # Rows of each distinct page up to the end of its longest beam.
    start = np.arange(owner.shape[2])[None, None, :] * page
    rows = np.clip(lengths[..., None] + N - start, 0, page)[own_pages].sum()
    new = B * K * N
    seen = _visible(case).sum() if case["tree"] else B * K * N * (N + 1) // 2
    pairs = (lengths.sum() * N + seen) * H * G
    return dict(bytes=rows * row + new * (2 * row + 2 * H * G * D * size + 4 * H * G), flops=4 * D * pairs)


def _repeats(K):
    """Expected share of the beams that repeat an earlier beam's parent, for prepare()'s parents."""
    i = np.arange(K)
    p = (2 * (K - i) - 1) / K**2
    return 1 - (1 - (1 - p) ** K).sum() / K


# -- the definitions in 64 bits ---------------------------------------------------------


def exact(case, seed):
    """The floating outputs in 64 bits, one beam at a time from the definitions."""
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if case["op"] == "attend":
        return _exact_attend(s)
    table, lengths = s["table"].cpu().numpy(), s["lengths"].cpu().numpy()
    references = s["references"].cpu().numpy()
    (B, K, M), page = table.shape, case["page"]
    pages = s["pages"].double()
    before = pages.clone()
    if case["op"] == "compact":
        n = int((references > 0).sum())
        holes = [p for p in range(n) if references[p] == 0]
        movers = [p for p in range(n, len(references)) if references[p] > 0]
        for a, b in zip(movers, holes):
            pages[:, :, b] = before[:, :, a]
    if case["op"] == "commit":
        path, counts = s["path"].cpu().numpy(), s["counts"].cpu().numpy()
        for b in range(B):
            for i in range(counts[b, 0]):
                x, y = int(lengths[b, 0] + path[b, 0, i]), int(lengths[b, 0] + i)
                pages[:, :, table[b, 0, y // page], :, y % page] = before[:, :, table[b, 0, x // page], :, x % page]
    if case["op"] == "fork":
        parents = s["parents"].cpu().numpy()
        held, asks = np.zeros(len(references), np.int64), []
        for b in range(B):
            for k in range(K):
                r, older = parents[b, k], parents[b, :k]
                n, full = int(lengths[b, r]), int(lengths[b, r]) // page
                for c in range(-(-(n + 1) // page)):
                    if c < full or (r not in older and table[b, r, c] >= 0):
                        held[table[b, r, c]] += 1
                    else:
                        asks.append((table[b, r, c], n % page if c == full and r in older else 0))
        free = [p for p in range(len(held)) if held[p] == 0]
        for (a, n), p in zip(asks, free):
            pages[:, :, p, :, :n] = before[:, :, a, :, :n]
    return dict(table=None, lengths=None, references=None, pages=pages)


def _exact_attend(s):
    case, layer = s["case"], 1
    pages = s["pages"][layer].double()
    table, lengths = s["table"].long(), s["lengths"].cpu().numpy()
    q, k, v = (s[x].double() for x in "qkv")
    (B, K, N, Hq, D), H, page = q.shape, k.shape[3], case["page"]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.full(q.shape[:-1], float("-inf"), dtype=torch.float64, device=q.device)
    causal = torch.ones((N, N), dtype=torch.bool, device=q.device).tril()
    for b in range(B):
        for beam in range(K):
            n = int(lengths[b, beam])
            for i in range(N):
                p, o = table[b, beam, (n + i) // page], (n + i) % page
                pages[0, p, :, o], pages[1, p, :, o] = k[b, beam, i], v[b, beam, i]
    for b in range(B):
        for beam in range(K):
            n = int(lengths[b, beam])
            held = table[b, beam, : -(-n // page)]
            old = pages[:, held].transpose(2, 3).reshape(2, -1, H, D)[:, :n]  # [2, n, H, D]
            both = torch.cat([old, torch.stack([k[b, beam], v[b, beam]])], 1)
            for h in range(H):
                rows = q[b, beam, :, h * (Hq // H) : (h + 1) * (Hq // H)]  # [N, G, D]
                x = torch.einsum("ngd,td->ngt", rows, both[0, :, h]) / math.sqrt(D)
                seen = causal if s["mask"] is None else s["mask"][b, beam]
                x[..., n:] = x[..., n:].masked_fill(~seen[:, None, :], float("-inf"))
                z = torch.logsumexp(x, -1)
                lse[b, beam, :, h * (Hq // H) : (h + 1) * (Hq // H)] = z
                y = torch.einsum("ngt,td->ngd", torch.exp(x - z[..., None]), both[1, :, h])
                out[b, beam, :, h * (Hq // H) : (h + 1) * (Hq // H)] = y
    return dict(out=out, lse=lse, pages=pages)
