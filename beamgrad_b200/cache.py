# SPDX-License-Identifier: MIT
"""A paged key/value cache for the beams of a search, and the attention that reads it.

:class:`beamgrad_b200.search.DeviceSearch` selects tokens and parents on the device; a transformer
behind it also has to reorder what it remembers of every beam. beamgrad leaves that to the caller
(``step_fn`` gets the parents in its ``BeamState``, python/beamgrad/_search.py:26-48 of beamgrad
2.3.0), who gathers whole caches. :class:`PagedCache` keeps keys and values in pages of a shared
pool instead:

* :meth:`PagedCache.fork` applies a step's parents: complete pages are shared between the children
  of a beam, only its last, incomplete page is copied, and pages nobody holds are free again;
* :meth:`PagedCache.attend` writes the new tokens of a layer and attends over the cache, for one
  token a beam or for a drafted tree of them; a page that several beams share is read once;
* :meth:`PagedCache.commit` keeps the accepted path of a drafted tree and frees the rest;
* :meth:`PagedCache.compact` moves the pages in use to the front of the pool.

All of it runs on the device without a host synchronisation, so a decode loop can be captured in a
CUDA graph. Errors that only the device sees (the pool ran out of pages, a parent out of range) are
sticky bits that :meth:`PagedCache.check` raises. There is no CPU path and no derivative: inputs that ask
for one, backward or forward, are refused.
"""

from __future__ import annotations

import ctypes as C
import math
import operator
import threading

import torch
from torch.autograd import forward_ad

from beamgrad_b200 import _abi as A

_DTYPES = {torch.float32: A.DTYPE_F32, torch.float16: A.DTYPE_F16, torch.bfloat16: A.DTYPE_BF16}
_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else (
    lambda index: torch.cuda.current_stream(index).cuda_stream)
_current_device = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else torch.cuda.current_device
_INT_MAX = (1 << 31) - 1
_MOST_CALLS = 256  # shapes and layouts that a cache remembers
_STATUS = (
    (A.CACHE_STATUS_POOL, "the pool ran out of pages"),
    (A.CACHE_STATUS_CAPACITY, "a beam outgrew the table (max_length)"),
    (A.CACHE_STATUS_INDEX, "a parent, a count, a page, a length or a path entry was out of range"),
    (A.CACHE_STATUS_SHARED, "an incomplete page is shared by several beams"),
    (A.CACHE_STATUS_TIMEOUT, "a bounded wait inside a kernel gave up"),
)


class PagedCache:
    """Keys and values of ``batch_size`` x ``beam_size`` beams in pages of ``page_size`` tokens.

    ``max_length`` bounds the tokens of a beam, ``num_pages`` the pool (by default enough for every
    beam to fill its table without sharing). ``page_size`` is 16, 32 or 64, ``head_dim`` a multiple
    of 8 up to 256, ``dtype`` float32, float16 or bfloat16.

    State, on the device: ``pages`` [num_layers, 2, num_pages, num_kv_heads, page_size, head_dim]
    (keys, values), ``table`` [B, K, columns] int32 (the page of each column of each beam, -1 for
    none), ``lengths`` [B, K] int32 (committed tokens) and ``references`` [num_pages] int32. They
    may be read at any time; after writing any of them, call :meth:`refresh`.

    Calls on one cache have to be ordered: one stream, or streams that wait for one another.
    """

    def __init__(self, batch_size: int, beam_size: int, max_length: int, *, num_layers: int, num_kv_heads: int,
                 head_dim: int, num_pages: int | None = None, page_size: int = 32,
                 dtype: torch.dtype = torch.bfloat16, device: torch.device | str | None = None):
        if min(batch_size, beam_size, max_length, num_layers, num_kv_heads) < 1 or page_size not in (16, 32, 64):
            raise ValueError("sizes must be positive and page_size 16, 32 or 64")
        if dtype not in _DTYPES:
            raise ValueError(f"pages must be float32, float16 or bfloat16, got {dtype}")
        device = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
        if device.type != "cuda":
            raise ValueError("PagedCache runs on a CUDA device; there is no CPU path")
        columns = -(-max_length // page_size)
        if num_pages is None:
            num_pages = batch_size * beam_size * columns
        # The sizes are checked before the pool is allocated.
        self._describe((num_layers, 2, num_pages, num_kv_heads, page_size, head_dim), (batch_size, beam_size, columns),
                       dtype)
        self._adopt(
            torch.zeros((num_layers, 2, num_pages, num_kv_heads, page_size, head_dim), dtype=dtype, device=device),
            torch.full((batch_size, beam_size, columns), -1, dtype=torch.int32, device=device),
            torch.zeros((batch_size, beam_size), dtype=torch.int32, device=device),
            torch.zeros(num_pages, dtype=torch.int32, device=device))

    @classmethod
    def from_tensors(cls, pages: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor,
                     references: torch.Tensor | None = None) -> "PagedCache":
        """A cache over existing tensors (laid out as the class says, used in place).
        ``references`` and the internal plan are computed from ``table`` and ``lengths``, as
        :meth:`refresh` does."""
        if pages.dim() != 6 or pages.shape[1] != 2 or pages.dtype not in _DTYPES:
            raise ValueError("pages must be a float [layers, 2, num_pages, heads, page_size, head_dim] tensor")
        if table.dim() != 3 or tuple(lengths.shape) != tuple(table.shape[:2]):
            raise ValueError("table must be [B, K, columns] and lengths [B, K]")
        if references is None:
            references = torch.zeros(pages.shape[2], dtype=torch.int32, device=pages.device)
        if tuple(references.shape) != (pages.shape[2],):
            raise ValueError("references must be [num_pages]")
        for x in (table, lengths, references):
            if x.dtype != torch.int32 or x.device != pages.device or not x.is_contiguous():
                raise ValueError("table, lengths and references must be contiguous int32 tensors on the pages' device")
        if pages.device.type != "cuda" or not pages.is_contiguous():
            raise ValueError("pages must be a contiguous CUDA tensor")
        self = cls.__new__(cls)
        self._describe(tuple(pages.shape), tuple(table.shape), pages.dtype)
        self._adopt(pages, table, lengths, references)
        self.refresh()
        return self

    def _describe(self, pages: tuple, table: tuple, dtype: torch.dtype) -> None:
        if max(*pages, *table) > _INT_MAX:  # (the structure's fields would wrap)
            raise ValueError("sizes must fit into 31 bits")
        self.lib = A.load()
        c = self._cache = A.Cache()
        c.num_layers, _, c.num_pages, c.num_heads, c.page_size, c.head_dim = pages
        c.batch_size, c.beam_size, c.max_pages = table
        c.data_type = _DTYPES[dtype]
        c.plan_bytes = self.lib.dbs_cuda_cache_plan_bytes(C.byref(c))
        if c.plan_bytes < 0:
            raise ValueError("the engine rejects these cache sizes")

    def _adopt(self, pages, table, lengths, references) -> None:
        self.pages, self.table, self.lengths, self.references = pages, table, lengths, references
        self.device, self.dtype = pages.device, pages.dtype  # the device with its index
        self.num_layers, _, self.num_pages, self.num_kv_heads, self.page_size, self.head_dim = pages.shape
        self.batch_size, self.beam_size, columns = table.shape
        self.max_length = columns * self.page_size
        c = self._cache
        self._plan = torch.zeros(c.plan_bytes, dtype=torch.uint8, device=self.device)
        self._status = torch.zeros(2, dtype=torch.int32, device=self.device)
        c.pages, c.table, c.lengths = pages.data_ptr(), table.data_ptr(), lengths.data_ptr()
        c.references, c.plan, c.status = references.data_ptr(), self._plan.data_ptr(), self._status.data_ptr()
        self._ref = C.byref(c)
        # One workspace a cache (its calls are ordered), made here: made by the first call, it would be cleared
        # by the CUDA graph that happens to capture that call, and by no other. Only its counters have to be zero.
        self._workspaces = {self.device.index: self._new_workspace()}
        self._calls = {}  # shapes and layouts of attend's arguments -> _Call
        self._lock = threading.Lock()
        self._float = torch.empty(0, dtype=torch.float32, device=self.device)

    def _new_workspace(self) -> torch.Tensor:
        a = A.AttendArgs(beams=1, new_tokens=1, query_heads=self.num_kv_heads, scale=1.0)
        with _on(self.device):
            size = max(0, self.lib.dbs_cuda_cache_attend_workspace_size(self._ref, C.byref(a)))  # (refused: no attend)
        workspace = torch.empty(size, dtype=torch.uint8, device=self.device)
        workspace[: A.CACHE_WORKSPACE_ZEROED].zero_()
        return workspace

    # -- state ----------------------------------------------------------------------------
    def reset(self) -> None:
        """An empty cache: no tokens, no pages, no errors, and no values in the pool that are not finite.
        On the device alone, without a host synchronisation."""
        self.table.fill_(-1)
        self.lengths.zero_()
        self.references.zero_()
        self._status[:1].zero_()
        self._recount(A.CACHE_VALUES_IF_SET)

    def refresh(self) -> None:
        """Recounts the references and the plan after a caller wrote the state, and notes whether the
        pool's values hold infinities or NaN (reads all of them; those in pages that no beam holds
        become 0). Pages and lengths out of range are brought into it, which :meth:`check` reports."""
        self._recount(A.CACHE_VALUES_ALL)

    def _recount(self, values: int) -> None:
        with _on(self.device):
            A.check(self.lib.dbs_cuda_cache_refresh(self._ref, values, self._stream()), "cache_refresh")

    def fork(self, parents: torch.Tensor | None = None, *, written: int | torch.Tensor = 0,
             room: int | torch.Tensor = 1) -> None:
        """One step of the beams: ``written`` new tokens of every beam become committed, beam
        (b, k) becomes a copy of beam (b, parents[b, k]) (None: itself; negative: empty), and every
        beam gets pages for ``room`` more tokens. ``written`` and ``room`` are numbers or [B, K]
        int32 tensors; pages a beam held beyond its room are freed. ``parents`` is [B, K]: a search
        step's (``DeviceSearch``), or any int32 / int64 tensor."""
        p = self._int32(parents, "parents")
        w, w_all = self._per_beam(written, "written")
        r, r_all = self._per_beam(room, "room")
        with _on(self.device):
            A.check(self.lib.dbs_cuda_cache_fork(self._ref, _ptr(p), _ptr(w), w_all, _ptr(r), r_all, self._stream()),
                    "cache_fork")

    def reserve(self, room: int | torch.Tensor) -> None:
        """Pages for ``room`` more tokens of every beam (a [B, K] tensor: of each)."""
        self.fork(None, room=room)

    def release(self, beams: torch.Tensor) -> None:
        """Empties the beams where the bool tensor ``beams`` ([B, K], or [B] for whole examples) is
        true. The others keep their tokens; their spare pages are freed."""
        if beams.dim() == 1:
            beams = beams[:, None].expand(-1, self.beam_size)
        keep = torch.arange(self.beam_size, device=self.device, dtype=torch.int32)
        self.fork(torch.where(beams, -1, keep), room=0)

    def commit(self, path: torch.Tensor, counts: torch.Tensor, *, room: int = 0) -> None:
        """Accepts a path through the drafted tokens that the last :meth:`attend` calls wrote:
        tokens path[b, k, :counts[b, k]] (indices into the draft, increasing; [B, K, A] and [B, K]
        int32) become the beam's next committed tokens, the other drafted ones are dropped, and
        there are pages for ``room`` more. Of a beam whose path does not increase, or names tokens
        that there was no room for, nothing is accepted, and :meth:`check` raises; a beam without
        tokens and pages stays empty."""
        if path.dim() != 3 or tuple(path.shape[:2]) != (self.batch_size, self.beam_size) or path.shape[2] < 1:
            raise ValueError(f"path must be [{self.batch_size}, {self.beam_size}, A], got {tuple(path.shape)}")
        p, n = self._int32(path, "path", None), self._int32(counts, "counts")
        with _on(self.device):
            A.check(self.lib.dbs_cuda_cache_commit(self._ref, _ptr(p), p.shape[2], _ptr(n), _number(room, "room"),
                                                   self._stream()), "cache_commit")

    def compact(self) -> None:
        """Moves the pages in use to the front of the pool; the beams keep their contents."""
        with _on(self.device):
            A.check(self.lib.dbs_cuda_cache_compact(self._ref, self._stream()), "cache_compact")

    def check(self) -> None:
        """Raises RuntimeError if an earlier call met an error that only the device saw (a host
        sync). The bits stay until :meth:`reset`."""
        bits = int(self._status[0])
        if bits:
            raise RuntimeError("paged cache: " + "; ".join(text for bit, text in _STATUS if bits & bit))

    @property
    def has_nonfinite(self) -> bool:
        """Whether a value that is not finite was written since the last :meth:`reset` or
        :meth:`refresh` (a host sync). While it is so, :meth:`attend` takes every row for itself, right
        but many times slower; when the beams with such values are gone, :meth:`refresh` ends that."""
        return bool(self._status[1])

    # -- attention ------------------------------------------------------------------------
    def attend(self, layer: int, q: torch.Tensor, k: torch.Tensor | None = None, v: torch.Tensor | None = None, *,
               mask: torch.Tensor | None = None, counts: torch.Tensor | None = None, scale: float | None = None,
               return_lse: bool = False, out: torch.Tensor | None = None):
        """Writes the N new tokens of a layer and attends over the committed tokens and them.

        ``q`` is [B, beams, N, query heads, head_dim], ``k`` and ``v`` [B, beams, N, kv heads,
        head_dim] in the cache's dtype (views with strides are read as they are); beams may be
        fewer than the cache's (a prompt is written for beam 0 alone and then forked). New token j
        of a beam takes position ``lengths + j``, for which :meth:`fork` or :meth:`reserve` made
        room; it becomes committed with the next :meth:`fork` or :meth:`commit`. Without ``k`` and
        ``v`` the positions hold it already.

        Query i sees every committed token of its beam and the new tokens j with mask[b, k, i, j]
        ([B, beams, N, N] bool: a drafted tree's ancestors; None: j <= i). ``counts`` [B, beams]
        int32 limits the new tokens of each beam. A query that sees nothing, or only scores of -inf,
        gives zeros (and an lse of -inf); a score of +inf or NaN makes both NaN. ``scale`` defaults to
        head_dim ** -0.5.

        Returns out [B, beams, N, query heads, head_dim], and with ``return_lse`` also the
        logsumexp of the scaled scores, [B, beams, N, query heads] float32.
        """
        if (k is None) != (v is None):
            raise ValueError("k and v are given together or not at all")
        if torch.is_grad_enabled() and (q.requires_grad or k is not None and (k.requires_grad or v.requires_grad)):
            raise RuntimeError("attend has no backward pass: call it under torch.no_grad()")
        if forward_ad._current_level >= 0 and any(x is not None and forward_ad.unpack_dual(x).tangent is not None for x in (q, k, v)):
            raise RuntimeError("attend has no forward-mode derivative: call it on the primals")
        # Arguments of one shape and layout are checked and written down once.
        key = (q.shape, q.stride(), q.dtype, q.device, mask is None) if k is None else (
            q.shape, q.stride(), q.dtype, q.device, mask is None, k.shape, k.stride(), k.dtype, k.device,
            v.shape, v.stride(), v.dtype, v.device)
        call = self._calls.get(key)
        if call is None:
            call = self._check_shapes(q, k, v)
            if len(self._calls) >= _MOST_CALLS:  # prompts of many lengths: begin again
                self._calls.clear()
            self._calls[key] = call
        if not 0 <= layer < self.num_layers:
            raise ValueError(f"layer {layer} is not one of {self.num_layers}")
        with self._lock:  # the structure of arguments is the shape's, not the call's
            out, lse, status = self._launch_attend(call, layer, q, k, v, mask, counts, scale, return_lse, out)
        if status:
            A.check(status, "cache_attend")
        return (out, lse) if return_lse else out

    def _launch_attend(self, call, layer, q, k, v, mask, counts, scale, return_lse, out):
        a, shape = call.args, call.shape
        if call.copies or (q.data_ptr() | (0 if k is None else k.data_ptr() | v.data_ptr())) % 16:
            q, k, v = self._rows(q), None if k is None else self._rows(k), None if v is None else self._rows(v)
            call = self._check_shapes(q, k, v)
            a = call.args
        a.q = q.data_ptr()
        if k is not None:
            a.k, a.v = k.data_ptr(), v.data_ptr()
        if mask is not None:
            if mask.shape != call.mask_shape or mask.dtype != torch.bool or mask.device != self.device:
                raise ValueError(f"mask must be a bool {call.mask_shape} tensor on {self.device}")
            mask = mask.contiguous()
            a.mask = mask.data_ptr()
        if counts is not None:
            counts = self._int32(counts, "counts", shape[:2])
            a.counts = counts.data_ptr()
        else:
            a.counts = None
        if out is None:
            out = self.pages.new_empty(shape)
        elif out.shape != shape or out.dtype != self.dtype or out.device != self.device or not out.is_contiguous():
            raise ValueError(f"out must be a contiguous {self.dtype} {tuple(shape)} tensor on {self.device}")
        a.out = out.data_ptr()
        lse = None
        if return_lse:
            lse = self._float.new_empty(shape[:4])
            a.lse = lse.data_ptr()
        else:
            a.lse = None
        a.layer = layer
        a.scale = call.scale if scale is None else scale
        with _on(self.device):
            stream = self._stream()
            workspace = self._workspaces[self.device.index]
            a.workspace, a.workspace_bytes = workspace.data_ptr(), workspace.numel()
            status = self.lib.dbs_cuda_cache_attend(self._ref, call.ref, stream)
        return out, lse, status

    def _check_shapes(self, q, k, v) -> "_Call":
        if q.dim() != 5:
            raise ValueError(f"q must be [B, beams, N, query heads, head_dim], got {tuple(q.shape)}")
        B, beams, N, heads, D = shape = q.shape
        if (B != self.batch_size or not 1 <= beams <= self.beam_size or N < 1 or D != self.head_dim
                or heads % self.num_kv_heads or heads < 1):
            raise ValueError(f"q {tuple(shape)} does not fit a cache of {self.batch_size} x {self.beam_size} beams with "
                             f"{self.num_kv_heads} heads of {self.head_dim}")
        for name, x in (("q", q), ("k", k), ("v", v)):
            if x is None:
                continue
            if x.dtype != self.dtype or x.device != self.device:
                raise ValueError(f"{name} must be a {self.dtype} tensor on {self.device}, got {x.dtype} on {x.device}")
            if x is not q and tuple(x.shape) != (B, beams, N, self.num_kv_heads, D):
                raise ValueError(f"{name} must be {(B, beams, N, self.num_kv_heads, D)}, got {tuple(x.shape)}")
        call = _Call()
        a = call.args = A.AttendArgs()
        call.ref = C.byref(a)
        call.shape, call.mask_shape, call.scale = shape, (B, beams, N, N), 1.0 / math.sqrt(D)
        step = 16 // q.element_size()
        call.copies = any(x is not None and (x.stride(4) != 1 or any(n % step for n in x.stride()[:4])) for x in (q, k, v))
        a.q_strides[:] = q.stride()[:4]
        if k is not None:
            a.k_strides[:] = k.stride()[:4]
            a.v_strides[:] = v.stride()[:4]
        a.beams, a.new_tokens, a.query_heads, a.scale = beams, N, heads, 1.0
        if self.lib.dbs_cuda_cache_attend_workspace_size(self._ref, call.ref) < 0:
            raise ValueError("the engine rejects these attention sizes")
        return call

    # -- helpers --------------------------------------------------------------------------
    def _stream(self) -> int:
        return _raw_stream(self.device.index)

    @staticmethod
    def _rows(x: torch.Tensor) -> torch.Tensor:
        """x with rows on 16-byte boundaries (a copy where it is not laid out so)."""
        step = 16 // x.element_size()
        if x.stride(4) == 1 and not any(n % step for n in x.stride()[:4]) and x.data_ptr() % 16 == 0:
            return x
        return x.clone(memory_format=torch.contiguous_format)

    def _int32(self, x: torch.Tensor | None, name: str, shape: tuple | None = ()) -> torch.Tensor | None:
        if x is None:
            return None
        if shape == ():
            shape = self.lengths.shape
        if x.device != self.device or x.dtype not in (torch.int32, torch.int64) or shape and x.shape != shape:
            raise ValueError(f"{name} must be an integer {tuple(shape or ())} tensor on {self.device}")
        if x.dtype == torch.int64:  # what 32 bits do not hold stays out of range
            x = x.clamp(-1, _INT_MAX).to(torch.int32)
        return x.contiguous()

    def _per_beam(self, x: int | torch.Tensor, name: str) -> tuple:
        return (self._int32(x, name), 0) if isinstance(x, torch.Tensor) else (None, _number(x, name))


def _number(x: int, name: str) -> int:
    x = operator.index(x)  # 1.5 tokens are a TypeError
    if not 0 <= x <= _INT_MAX:
        raise ValueError(f"{name} must not be negative, got {x}")
    return x


def _ptr(x: torch.Tensor | None) -> int | None:
    return None if x is None else x.data_ptr()


class _Call:
    """What attend keeps of arguments of one shape and layout."""

    __slots__ = ("args", "ref", "shape", "mask_shape", "scale", "copies")


class _Here:
    def __enter__(self):
        return None

    def __exit__(self, *exc):
        return None


_HERE = _Here()


def _on(device: torch.device):
    """The device as the current one; nothing to do where it is already."""
    return _HERE if _current_device() == device.index else torch.cuda.device(device)
