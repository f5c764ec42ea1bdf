"""A KV cache in pages: block tables and slot maps from request lengths, appends, attention of one new token per sequence.

    import penny_b200.ops as P
    cache = P.PagedKVCache(layers=32, rows=64, max_len=4096, kv_heads=8)          # bf16 pages of 16 positions
    step = cache.advance(new, tokens)                       # new [rows] int32 on the device: tokens that come (or leave)
    for i in range(32):
        qkv = ...                                           # [tokens, (heads + 2 kv_heads) head_dim], rows packed by request
        cache.append(i, qkv, step, heads, theta)            # q and k rotated in place, k and v into the pages
        o = cache.attend(i, qkv[:, :heads * 128].unflatten(1, (heads, 128)))      # a step of one token per row

All state lives on the device and nothing here waits for it: the calls may be captured in a CUDA graph, which keeps counting.
`page_tables`, `paged_append` and `paged_attention` are the same calls on a caller's own tensors.

The reference has no KV cache: it serves the paged ones of vLLM and SGLang (README.md:20-33).
"""
from __future__ import annotations

from typing import List, NamedTuple, Optional

import torch

from .._ext import ops


class PageStep(NamedTuple):
    """Where the tokens of a step go, rows one behind the other."""
    slots: torch.Tensor      # [tokens] int64: page * page_size + offset; -1 behind the last token and where not granted
    positions: torch.Tensor  # [tokens] int32: position in the sequence (0 behind the last token and where not granted)
    offsets: torch.Tensor    # [rows + 1] int32: row r's tokens are [offsets[r], offsets[r + 1])
    granted: torch.Tensor    # [rows] bool


class OutOfPages(RuntimeError):
    """Rows that were not granted a token (no page, or at their longest), and the tokens that the step gave all the same."""

    def __init__(self, said: str, rows: List[int], next_tokens: torch.Tensor):
        super().__init__(said)
        self.rows, self.next_tokens = rows, next_tokens


def page_tables(table, lengths, free, free_count, new, page_size: int, tokens: int, out: Optional[PageStep] = None,
                max_len: Optional[int] = None) -> PageStep:
    """Lets new[r] tokens come to row r, or its last -new[r] leave, and moves the pages that follow from it.

    table [rows, pages of a row] int32, lengths [rows] int32: the sequences; free [pages] int32 with free_count [1] int32: a
    stack of the pages that no row has, its top at free_count - 1.  All four are updated in place.  new: [rows] int32.  No two of
    these tensors and of out's share memory.

    Pages of tokens that leave are put on the stack first, rows and pages in descending order; then pages are taken from it,
    rows and pages ascending (so what comes and leaves again is back in its old place).  A row is granted its new tokens if its
    table row can hold them and it gets no longer than max_len (None: what the table row holds), they end inside `tokens`, and there
    are pages for it and every row before it that passes these tests; one that is not keeps its length, and its slots are -1.  A
    row that gets no tokens is granted.
    At most 8192 rows.  `tokens` may exceed the sum of new (a captured step's fixed number).  Entries of a table row behind its
    pages, and of free from free_count on, say nothing."""
    return PageStep._make(ops.page_tables(table, lengths, free, free_count, new, page_size, tokens, out, max_len))


def paged_append(qkv, k, v, slots, positions, heads: int, theta: float, out=None, k_scale=None, v_scale=None, early: bool = False) -> None:
    """Rotates q and k of every token of qkv [tokens, (heads + 2 kv_heads) dim] (rotate-half form, in place or into out
    [tokens, (heads + kv_heads) dim]) and stores the rotated k and v at the tokens' slots of the pools k, v [pages, page_size,
    kv_heads, dim].  A token whose slot the pool does not have (-1) is left alone, its row of out too; no two tokens have the
    same slot.  Pools of qkv's type, or e4m3: value / k_scale[head] (v_scale), saturated at 448.  Any strides of whole 16 bytes;
    dim a multiple of 16, up to 256.  k and v are apart; out is apart from qkv, or the start of its rows.
    early: as in `paged_attention`, for slots and positions."""
    ops.paged_append(qkv, k, v, slots, positions, heads, theta, out, k_scale, v_scale, early)


def paged_attention(q, k, v, table, lengths, out=None, lse=None, scale: Optional[float] = None, window: int = 0, k_scale=None, v_scale=None,
                    workspace=None, early: bool = False) -> torch.Tensor:
    """softmax(scale q K^T) V of one token per row: q [rows, heads, dim] (bf16 or fp16) over the last `window` (0: all) of
    lengths[r] positions on the row's pages; scale: 1 / sqrt(dim) by default.  Returns out, like q.

    k, v: pools [pages, page_size, kv_heads, dim] of q's type, or e4m3 with k_scale, v_scale [kv_heads] fp32; any page size, any
    strides of whole 16 bytes (k's and v's alike); dim 64, 128 or 256; heads a multiple of kv_heads.  lse: [rows, heads] fp32 for
    the logarithm of the weights' sum, with which parts of a context can be joined.  A row of length 0 (or below) gives
    zeros and -inf; a length past the table row counts as the table row; positions on a page that the pool does not have count as
    not there.  Rows may share pages.  out is q itself or apart from it; out, lse and workspace share nothing with each other or with what
    else the call reads.  workspace: `paged_attention_workspace_bytes(rows, heads, kv_heads, dim, max_len, window)`
    bytes with max_len = table.size(1) * page_size, for callers that must not allocate; its contents mean nothing between calls,
    but two calls that may run at the same time need one each.  early: for a step whose kernels overlap (this library's are launched with
    programmatic dependency): those that may still run when this one starts, back to the last launch without it, write of what
    it reads only q and the keys and values of each row's last position; the other rows, lengths and table are then read before they end."""
    return ops.paged_attention(q, k, v, table, lengths, out, lse, scale, window, k_scale, v_scale, workspace, early)


def paged_attention_workspace_bytes(rows: int, heads: int, kv_heads: int, dim: int, max_len: int, window: int = 0) -> int:
    """Bytes of a workspace for `paged_attention` on the current device, for tables of max_len positions a row (0: none is needed)."""
    return ops.paged_attention_workspace_bytes(rows, heads, kv_heads, dim, max_len, window)


class PagedKVCache:
    """The pools of `layers` layers, one table for all of them, and the pages that are free.

    rows: sequences at a time (a row whose length is 0 is free for the next one); max_len: positions that a row can have;
    pages: of the pool, by default as many as all rows need at their longest.  dtype: bf16, fp16 or e4m3, whose scales
    (k_scale, v_scale [kv_heads] fp32, one for all layers, or a list of them) default to one."""

    def __init__(self, layers: int, rows: int, max_len: int, kv_heads: int, head_dim: int = 128, page_size: int = 16, pages: Optional[int] = None,
                 dtype: torch.dtype = torch.bfloat16, k_scale=None, v_scale=None, device=None):
        if min(layers, rows, max_len, kv_heads, head_dim, page_size) < 1 or (pages is not None and pages < 1):
            raise ValueError("PagedKVCache: layers, rows, max_len, kv_heads, head_dim, page_size and pages above zero")
        if rows > ops.PAGED_MAX_ROWS:
            raise ValueError(f"PagedKVCache: at most {ops.PAGED_MAX_ROWS} rows")
        self.e4m3 = dtype == torch.float8_e4m3fn
        if dtype not in (torch.bfloat16, torch.float16) and not self.e4m3:
            raise ValueError("PagedKVCache: bf16, fp16 or e4m3")
        if not self.e4m3 and (k_scale is not None or v_scale is not None):
            raise ValueError("PagedKVCache: scales beside e4m3 only")
        self.device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        self.rows, self.max_len, self.page_size, self.kv_heads, self.head_dim = rows, max_len, page_size, kv_heads, head_dim
        width = -(-max_len // page_size)
        self.pages = rows * width if pages is None else pages
        new = lambda: torch.zeros(self.pages, page_size, kv_heads, head_dim, dtype=dtype, device=self.device)  # noqa: E731
        self.k: List[torch.Tensor] = [new() for _ in range(layers)]
        self.v: List[torch.Tensor] = [new() for _ in range(layers)]
        scales = []
        for s in (k_scale, v_scale):
            if self.e4m3 and s is None:
                s = torch.ones(kv_heads, dtype=torch.float32, device=self.device)
            scales.append(list(s) if isinstance(s, (list, tuple)) else [s] * layers)
            if len(scales[-1]) != layers:
                raise ValueError("PagedKVCache: one scale tensor for all layers, or one for each")
            if self.e4m3 and any(t.dtype != torch.float32 or t.shape != (kv_heads,) for t in scales[-1]):
                raise ValueError("PagedKVCache: scales [kv_heads] fp32")
        self.k_scale, self.v_scale = scales
        self.table = torch.full((rows, width), -1, dtype=torch.int32, device=self.device)
        self.lengths = torch.zeros(rows, dtype=torch.int32, device=self.device)
        self.free = torch.arange(self.pages - 1, -1, -1, dtype=torch.int32, device=self.device)  # page 0 on top
        self.free_count = torch.full((1,), self.pages, dtype=torch.int32, device=self.device)

    def advance(self, new: torch.Tensor, tokens: int, out: Optional[PageStep] = None) -> PageStep:
        """`page_tables` on this cache: new[r] tokens come to row r or its last -new[r] leave (-lengths[r]: the row is free)."""
        return page_tables(self.table, self.lengths, self.free, self.free_count, new, self.page_size, tokens, out, self.max_len)

    def append(self, layer: int, qkv: torch.Tensor, step: PageStep, heads: int, theta: float, out: Optional[torch.Tensor] = None,
               early: bool = False) -> None:
        """`paged_append` to this cache's `layer` at the step's slots and positions."""
        paged_append(qkv, self.k[layer], self.v[layer], step.slots, step.positions, heads, theta, out, self.k_scale[layer], self.v_scale[layer],
                     early)

    def attend(self, layer: int, q: torch.Tensor, out=None, lse=None, scale: Optional[float] = None, window: int = 0, workspace=None,
               early: bool = False) -> torch.Tensor:
        """`paged_attention` of q [rows, heads, head_dim] over this cache's `layer`, all positions of lengths (those of the
        step that `advance` made room for included: append before)."""
        return paged_attention(q, self.k[layer], self.v[layer], self.table, self.lengths, out, lse, scale, window, self.k_scale[layer],
                               self.v_scale[layer], workspace, early)

    def snapshot(self):
        """Which pages and lengths the rows have, for `restore` (the pages' contents are not kept)."""
        return tuple(t.clone() for t in (self.table, self.lengths, self.free, self.free_count))

    def restore(self, snapshot) -> None:
        for t, old in zip((self.table, self.lengths, self.free, self.free_count), snapshot):
            t.copy_(old)

    def rows_of(self, layer: int, row: int, length: int):
        """(k, v) [kv_heads, length, head_dim] of a row's first positions, e4m3 ones times their scales in fp32: a copy, for looking at."""
        if not 0 <= length <= self.table.shape[1] * self.page_size:
            raise IndexError(f"rows_of: a row has {self.table.shape[1] * self.page_size} positions at most")
        at = torch.arange(length, device=self.device)
        pages, within = self.table[row].long()[at // self.page_size], at % self.page_size
        if bool(((pages < 0) | (pages >= self.pages)).any()):
            raise IndexError("rows_of: positions that are on no page of the pool")
        got = []
        for pool, scale in ((self.k[layer], self.k_scale[layer]), (self.v[layer], self.v_scale[layer])):
            rows = pool.view(torch.uint8)[pages, within].view(pool.dtype) if self.e4m3 else pool[pages, within]
            got.append((rows.float() * scale[:, None] if self.e4m3 else rows).transpose(0, 1).contiguous())
        return tuple(got)

    def workspace(self, heads: int, window: int = 0) -> torch.Tensor:
        """A workspace for `attend` with q of `heads` heads."""
        with torch.cuda.device(self.device):
            n = ops.paged_attention_workspace_bytes(self.rows, heads, self.kv_heads, self.head_dim, self.table.shape[1] * self.page_size, window)
        return torch.empty(n, dtype=torch.uint8, device=self.device)
