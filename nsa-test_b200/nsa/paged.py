"""Paged serving of NSA's attention branches: requests of any lengths in one step, keys and values held in 4 bits.

The reference has neither a cache nor batches of different lengths.  What ``NSACache`` holds for sequences of one common length in
bf16, ``PagedCache4`` holds in pages of 64 tokens (the selection's block size) that any request may own, at 4.5 bits a value: 180
bytes a token and group at head dims 192/128 instead of 640.  A step is

    step = block_tables(cached, new, table, free_pages, tokens)      # pages and slots of the new tokens, on the GPU
    cache.append(k, v, step.slots)                                   # their keys and values, quantised
    o, L, M = cache.attend(q, table, step.lengths, step.starts, ...) # all earlier keys, a sliding window, or selected blocks

Nothing here waits for the GPU, so a step can be captured into a graph and replayed with other lengths.  Forward only.
"""
from __future__ import annotations

import functools
import math
from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib, ops

__all__ = ["PAGE_TOKENS", "MAX_SELECTED", "StepTables", "block_tables", "PagedCache4"]

PAGE_TOKENS = 64
MAX_SELECTED = 32
_FLOATS = (torch.bfloat16, torch.float32)
_MOST_TOKENS, _MOST_PAGE_TOKENS = 1 << 30, 1 << 16


class StepTables(NamedTuple):
    """A step's tokens, one request after the other (int32 but for the slots)."""
    slots: torch.Tensor        # [tokens] int64: page * page_tokens + place, -1 for tokens without a page and behind the last
    positions: torch.Tensor    # [tokens]: position in the request, -1 behind the last
    starts: torch.Tensor       # [S + 1]: where each request's tokens begin
    lengths: torch.Tensor      # [S]: tokens each request has once these are in
    pages: torch.Tensor        # [1]: pages the step takes off the free list (more than it holds: some tokens got none)


def _int32(name: str, t: torch.Tensor, want: tuple) -> None:
    """int32 of shape ``want`` (None: any), rows without gaps.  (The checks of a call cost no more than its launch: plain comparisons.)"""
    shape = t.shape
    if t.dtype is torch.int32 and len(shape) == len(want):
        if len(want) == 1:
            if (want[0] is None or shape[0] == want[0]) and (shape[0] < 2 or t.stride(0) == 1):
                return
        elif shape[:-1] == want[:-1] and (t.is_contiguous() if len(want) == 3 else shape[1] < 2 or t.stride(1) == 1):
            return
    raise ValueError(f"{name} must be int32 [{', '.join('*' if n is None else str(n) for n in want)}]"
                     f"{', contiguous' if len(want) == 3 else ' with unit stride along its last dimension'}; "
                     f"got {t.dtype} {tuple(shape)}, strides {t.stride()}")


def block_tables(cached: torch.Tensor, new: torch.Tensor, table: torch.Tensor, free_pages: torch.Tensor, tokens: int,
                 page_tokens: int = PAGE_TOKENS) -> StepTables:
    """Lays out a step in which request r, with ``cached[r]`` tokens in the cache, brings ``new[r]`` more.

    ``table [S,P]`` holds the pages of each request's cached tokens and receives those that the new ones open, taken from the front of
    ``free_pages`` in the order of the requests.  ``tokens`` is the number of new tokens or, where that is not known on the host (a
    captured graph), a bound of it.  Lengths are data on the GPU, so a free list or a table row that is too short raises nothing: the tokens
    without a page get slot -1, which the cache passes over, and ``pages`` says how many the step needed.  At most 16384 requests and 2^30
    tokens a call, pages of 1 to 65536 tokens.
    """
    if table.dim() != 2:
        raise ValueError(f"table must be int32 [S, P], got {tuple(table.shape)}")
    S = table.shape[0]
    _int32("table", table, (S, None))
    _int32("cached", cached, (S,))
    _int32("new", new, (S,))
    _int32("free_pages", free_pages, (None,))
    if S > 1 and table.stride(0) < table.shape[1]:
        raise ValueError("table rows overlap")
    if not 0 <= tokens <= _MOST_TOKENS or not 1 <= page_tokens <= _MOST_PAGE_TOKENS:
        raise ValueError(f"tokens {tokens} and page_tokens {page_tokens} must be 0 to {_MOST_TOKENS} and 1 to {_MOST_PAGE_TOKENS}")
    return StepTables(*ops.block_tables(cached, new, table, free_pages, int(tokens), int(page_tokens)))


@functools.lru_cache(maxsize=None)
def _page_bytes(head_dim_qk: int, head_dim_v: int) -> int:
    nbytes = _lib.lib.nsa_cache4_page_bytes(head_dim_qk, head_dim_v)
    if nbytes == 0:
        raise ValueError(f"PagedCache4: head dims {head_dim_qk}/{head_dim_v} are no multiples of 32 up to 256")
    return nbytes


class PagedCache4:
    """Keys and values of ``pages`` pages of 64 tokens in 4 bits with a scale per 32 dimensions.

    ``storage`` is uint8 ``[pages, G, page_bytes]`` (layout in include/nsa_b200.h); the object keeps nothing else, so it can be made anew
    around the same storage at any time.  Head dims are multiples of 32 up to 256.
    """

    def __init__(self, storage: torch.Tensor, head_dim_qk: int, head_dim_v: int):
        nbytes = _page_bytes(head_dim_qk, head_dim_v)
        if storage.dtype != torch.uint8 or storage.dim() != 3 or storage.shape[2] != nbytes or not storage.is_contiguous():
            raise ValueError(f"PagedCache4: storage must be contiguous uint8 [pages, groups, {nbytes}], got {storage.dtype} {tuple(storage.shape)}")
        self.storage, self.head_dim_qk, self.head_dim_v = storage, head_dim_qk, head_dim_v
        if storage.is_cuda:
            ops.cache4_setup(storage.get_device())

    @classmethod
    def empty(cls, pages: int, n_kv_groups: int, head_dim_qk: int, head_dim_v: int, device="cuda") -> "PagedCache4":
        return cls(torch.zeros(pages, n_kv_groups, _page_bytes(head_dim_qk, head_dim_v), device=device, dtype=torch.uint8), head_dim_qk, head_dim_v)

    def append(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
        """Quantises k ``[N,G,dk]`` and v ``[N,G,dv]`` (any strides) into ``slots [N]``, which are distinct; slots outside the cache (-1)
        are passed over.  Infinities are held as +-57120, the largest magnitude there is, NaN as 0."""
        G = self.storage.shape[1]
        N = k.shape[0]
        if k.shape != (N, G, self.head_dim_qk) or v.shape != (N, G, self.head_dim_v):
            raise ValueError(f"append: k {tuple(k.shape)} and v {tuple(v.shape)} do not fit [N, {G}, {self.head_dim_qk}] and [N, {G}, {self.head_dim_v}]")
        if k.dtype not in _FLOATS or v.dtype != k.dtype:
            raise TypeError(f"append: k and v must both be bfloat16 or float32, got {k.dtype} and {v.dtype}")
        self._check_slots(slots, N)
        ops.cache4_append(k, v, slots, self.storage)

    def read(self, slots: torch.Tensor, dtype=torch.float32) -> Tuple[torch.Tensor, torch.Tensor]:
        """The values that ``slots [N]`` hold, k ``[N,G,dk]`` and v ``[N,G,dv]``: exact in float32, rounded once in bfloat16."""
        if dtype not in _FLOATS:
            raise TypeError(f"read: dtype must be bfloat16 or float32, got {dtype}")
        self._check_slots(slots, slots.numel())
        return ops.cache4_read(self.storage, slots, self.head_dim_qk, self.head_dim_v, dtype)

    def attend(self, q: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, starts: torch.Tensor, *, scale: Optional[float] = None,
               window: Optional[int] = None, indices: Optional[torch.Tensor] = None, max_new: Optional[int] = None,
               out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """Attention of the newest tokens: rows ``starts[r]:starts[r+1]`` of q ``[N,H,dk]`` are request r's last ones, whose keys and values
        (their own among them) are in the cache under ``table [S,P]``, ``lengths [S]``.  Each sees the keys up to its own position;
        with ``window`` the last so many of them; with ``indices [N,G,n]`` (int32, n <= 32) those in the named 64-key blocks of its request,
        negative entries and repetitions not counting.  -> (o ``[N,H,dv]`` in the type of q, L, M ``[N,H]`` fp32: log sum and maximum of
        the logits, as of the other branches); rows that see nothing are 0 with L = M = -inf, rows that see something with a query that holds a
        NaN or an infinity are NaN in all three, rows behind the last request's stay as they were.  ``max_new``: a bound of the requests' numbers of new tokens, where the host knows one.
        """
        dk, dv, G = self.head_dim_qk, self.head_dim_v, self.storage.shape[1]
        if q.dim() != 3 or q.shape[2] != dk or q.shape[1] % G or q.shape[1] == 0:
            raise ValueError(f"attend: q {tuple(q.shape)} does not fit [N, a multiple of {G} heads, {dk}]")
        if q.dtype not in _FLOATS:
            raise TypeError(f"attend: q must be bfloat16 or float32, got {q.dtype}")
        if table.dim() != 2:
            raise ValueError(f"table must be int32 [S, P], got {tuple(table.shape)}")
        S = table.shape[0]
        _int32("table", table, (S, None))
        if S > 1 and table.stride(0) < table.shape[1]:
            raise ValueError("table rows overlap")
        _int32("lengths", lengths, (S,))
        _int32("starts", starts, (S + 1,))
        if window is not None and (window < 1 or indices is not None):
            raise ValueError("attend: window must be positive and does not go together with indices")
        if indices is not None:
            _int32("indices", indices, (q.shape[0], G, None))
            if not 0 < indices.shape[2] <= MAX_SELECTED:
                raise ValueError(f"attend: {indices.shape[2]} selected blocks a token, 1 to {MAX_SELECTED} are supported")
        if out is not None and (out.shape != (*q.shape[:2], dv) or out.dtype != q.dtype or not out.is_contiguous()):
            raise ValueError(f"attend: out must be contiguous {q.dtype} [{q.shape[0]}, {q.shape[1]}, {dv}]")
        if max_new is not None and max_new < 0:
            raise ValueError("attend: negative max_new")
        if scale is not None and not math.isfinite(scale):
            raise ValueError(f"attend: scale {scale} is not finite")
        if q.stride(2) != 1 or (q.dtype == torch.bfloat16 and (q.data_ptr() % 16 or q.stride(0) % 8 or q.stride(1) % 8)):
            q = q.clone(memory_format=torch.contiguous_format)      # the tensor-core kernels load rows 16 bytes at a time
        return ops.cache4_attn(q, self.storage, table, lengths, starts, indices, dk, dv, 0 if window is None else min(int(window), 1 << 30),
                               1.0 / math.sqrt(dk) if scale is None else float(scale), 0 if max_new is None else min(int(max_new), 1 << 30), out)

    def _check_slots(self, slots: torch.Tensor, n: int) -> None:
        if slots.dtype != torch.int64 or slots.dim() != 1 or slots.shape[0] != n or (n > 1 and slots.stride(0) != 1):
            raise ValueError(f"slots must be contiguous int64 [{n}], got {slots.dtype} {tuple(slots.shape)}")
