"""A paged key-value cache: rotary append into pages, attention over them
(with a sliding window and sinks), and the host side that hands pages out.

riallm keeps one contiguous cache per layer (KVCACHE, src/model.rs:15-38);
the rotary embedding and the attention are its own (src/model.rs:912-1071).
Layout and meaning of the page table: include/riallm_cuda.h.
"""
from __future__ import annotations

import struct
from typing import Dict, List, Optional, Tuple

import torch

from . import ConfigError, Context, MemoryError_, lib

PAGE_SIZES = (16, 32, 64, 128)

# riallm_rope_paged_append_args and riallm_paged_attention_args.
_APPEND, _ATTEND = struct.Struct("@7Pq8i"), struct.Struct("@6Pq10i")


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ConfigError(what)


def _check_cache(what, x, pos, page_table, k_pages, v_pages):
    """The checks both operators share; returns (device, B, T, pages' shape).
    A decode step makes them for every layer, so what holds costs little and
    the message is worked out only for what does not."""
    bf16, i32 = torch.bfloat16, torch.int32
    dev = x.get_device()
    shape, table = k_pages.shape, page_table.shape
    B, rows = pos.shape[0] if pos.dim() == 1 else -1, x.shape[0] if x.dim() == 2 else -1
    if (dev >= 0 and dev == k_pages.get_device() == v_pages.get_device() == pos.get_device()
            == page_table.get_device()
            and x.dtype is bf16 and k_pages.dtype is bf16 and v_pages.dtype is bf16 and pos.dtype is i32
            and page_table.dtype is i32 and B >= 0 and rows >= 0 and len(shape) == 4 and shape == v_pages.shape
            and len(table) == 2 and table[0] == B and (rows % B == 0 if B else rows == 0)
            and x.is_contiguous() and k_pages.is_contiguous() and v_pages.is_contiguous() and pos.is_contiguous()
            and (page_table.is_contiguous() or page_table.stride(1) == 1 or table[1] == 1)):
        return dev, B, (rows // B if B else 0), shape
    _need(x.is_cuda and x.dtype is bf16 and rows >= 0 and x.is_contiguous(),
          f"{what}: rows must be a contiguous 2-D bf16 CUDA tensor")
    for t in (k_pages, v_pages):
        _need(t.dtype is bf16 and t.dim() == 4 and t.is_contiguous() and t.device == x.device,
              f"{what}: pages must be contiguous bf16 [num_pages, kv_heads, page_size, head_dim] on the rows' device")
    _need(k_pages.shape == v_pages.shape, f"{what}: k_pages and v_pages differ in shape")
    _need(pos.dtype is i32 and B >= 0 and pos.is_contiguous() and pos.device == x.device,
          f"{what}: pos must be a contiguous int32 [B] tensor on the rows' device")
    _need(rows == 0 if B == 0 else rows % B == 0, f"{what}: {rows} rows are no multiple of {B} sequences")
    raise ConfigError(f"{what}: page_table must be int32 [B, max_pages] with unit stride along the pages, on the "
                      "rows' device")


def _context(what: str, ctx: Optional[Context], dev: int) -> Context:
    if ctx is None:
        return Context._by_device.get(dev) or Context.get(dev)
    _need(ctx.device == dev, f"{what}: the context is another device's")
    return ctx


# The raw handle of the current stream of a device.
_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else (
    lambda dev: torch.cuda.current_stream(dev).cuda_stream)


def _table_stride(page_table: torch.Tensor) -> int:
    # A table of one sequence has no second row; torch may give it any stride.
    return page_table.stride(0) if page_table.shape[0] > 1 else page_table.shape[1]


def rope_paged_append(qkv: torch.Tensor, pos: torch.Tensor, page_table: torch.Tensor, k_pages: torch.Tensor,
                      v_pages: torch.Tensor, inv_freq: torch.Tensor, q_out: Optional[torch.Tensor] = None,
                      ctx: Optional[Context] = None) -> torch.Tensor:
    """Rotates the q and k heads of qkv [B*T, (nh + 2*nkv) * d] (bf16; row
    b*T + t at position pos[b] + t), writes k and v into the sequences' pages
    and returns the rotated q [B*T, nh*d]. inv_freq is float32 [d/2]."""
    dev, B, T, (num_pages, nkv, ps, d) = _check_cache("rope_paged_append", qkv, pos, page_table, k_pages, v_pages)
    rows, width = qkv.shape
    _need(d > 0 and width % d == 0 and width // d > 2 * nkv,
          "rope_paged_append: qkv rows must hold q heads and 2 * kv_heads more of head_dim")
    nh = width // d - 2 * nkv
    _need(inv_freq.dtype is torch.float32 and inv_freq.numel() == d // 2 and inv_freq.get_device() == dev
          and inv_freq.is_contiguous(), "rope_paged_append: inv_freq must be float32 [head_dim / 2]")
    if q_out is None:
        q_out = torch.empty((rows, nh * d), dtype=torch.bfloat16, device=qkv.device)
    else:
        _need(q_out.dtype is torch.bfloat16 and q_out.shape == (rows, nh * d) and q_out.get_device() == dev
              and q_out.is_contiguous(), "rope_paged_append: q_out must be contiguous bf16 [B*T, heads*head_dim]")
    ctx = _context("rope_paged_append", ctx, dev)
    try:
        args = _APPEND.pack(qkv.data_ptr(), pos.data_ptr(), page_table.data_ptr(), inv_freq.data_ptr(),
                            q_out.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), _table_stride(page_table),
                            page_table.shape[1], num_pages, ps, B, T, nh, nkv, d)
    except struct.error:
        raise ConfigError("rope_paged_append: sizes must be 32-bit integers") from None
    status = lib().riallm_cuda_rope_paged_append(ctx.ptr, args, _stream(dev))
    if status:
        ctx.check(status)
    return q_out


# Workspace bytes by call shape: a pure function of the shape on one kind of device.
_workspace: Dict[Tuple[int, ...], int] = {}


def paged_attention(q: torch.Tensor, pos: torch.Tensor, page_table: torch.Tensor, k_pages: torch.Tensor,
                    v_pages: torch.Tensor, window: int = 0, sinks: int = 0, out: Optional[torch.Tensor] = None,
                    ctx: Optional[Context] = None) -> torch.Tensor:
    """Causal grouped-query attention of q [B*T, nh*d] (bf16; row b*T + t at
    position p = pos[b] + t) over the sequences' pages: positions j <= p, and
    with a window only j > p - window or j < sinks. Rows that see nothing are
    zero. Returns out [B*T, nh*d]."""
    dev, B, T, (num_pages, nkv, ps, d) = _check_cache("paged_attention", q, pos, page_table, k_pages, v_pages)
    width = q.shape[1]
    _need(d > 0 and width % d == 0, "paged_attention: q rows must hold whole heads")
    nh = width // d
    if out is None:
        out = torch.empty_like(q)
    else:
        _need(out.dtype is torch.bfloat16 and out.shape == q.shape and out.get_device() == dev and out.is_contiguous(),
              "paged_attention: out must be contiguous bf16 of q's shape")
    ctx = _context("paged_attention", ctx, dev)
    L = lib()
    max_pages = page_table.shape[1]
    key = (dev, B, T, nh, nkv, d, max_pages, ps)
    size = _workspace.get(key)
    if size is None:
        if len(_workspace) > 4096:
            _workspace.clear()
        size = _workspace[key] = L.riallm_cuda_paged_attention_workspace(ctx.ptr, B, T, nh, nkv, d, max_pages, ps)
    # From the caching allocator, in the order of the call's stream: two calls
    # never share one, whatever streams or graphs they are in.
    ws = q.new_empty((size + 1) // 2) if size else None
    try:
        args = _ATTEND.pack(q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), pos.data_ptr(),
                            page_table.data_ptr(), out.data_ptr(), _table_stride(page_table), max_pages, num_pages, ps,
                            B, T, nh, nkv, d, window, sinks)
    except struct.error:
        raise ConfigError("paged_attention: sizes, window and sinks must be 32-bit integers") from None
    status = L.riallm_cuda_paged_attention(ctx.ptr, args, ws.data_ptr() if size else None, size, _stream(dev))
    if status:
        ctx.check(status)
    return out


class PagedKVCache:
    """Pools of pages for `layers` layers and the page tables of up to
    `max_batch` sequences of up to `max_pages` pages each. One table serves
    every layer: page i of each layer's pools belongs to the same positions.

    The tables live on the device (`table`, int32 [max_batch, max_pages],
    -1 where a sequence holds no page) at a fixed address, so captured graphs
    see later changes; the free list and a copy of the tables are the
    host's."""

    def __init__(self, layers: int, kv_heads: int, head_dim: int, num_pages: int, page_size: int = 64,
                 max_batch: int = 1, max_pages: Optional[int] = None, device: int = 0):
        _need(page_size in PAGE_SIZES, f"page_size must be one of {PAGE_SIZES}")
        _need(head_dim in (64, 128), "head_dim must be 64 or 128")
        _need(layers > 0 and kv_heads > 0 and num_pages > 0 and max_batch > 0, "empty paged cache")
        max_pages = num_pages if max_pages is None else int(max_pages)
        _need(max_pages > 0, "empty paged cache")
        self.page_size, self.num_pages, self.max_pages = page_size, num_pages, max_pages
        dev = torch.device("cuda", device)
        shape = (num_pages, kv_heads, page_size, head_dim)
        self.k_pages = [torch.zeros(shape, dtype=torch.bfloat16, device=dev) for _ in range(layers)]
        self.v_pages = [torch.zeros(shape, dtype=torch.bfloat16, device=dev) for _ in range(layers)]
        self.table = torch.full((max_batch, max_pages), -1, dtype=torch.int32, device=dev)
        self._init_host(max_batch)

    def _init_host(self, max_batch: int):
        self._held: List[List[int]] = [[] for _ in range(max_batch)]  # -1: given back
        self._passed = [0] * max_batch  # pages below this index were looked at by release_before
        self._free = list(range(self.num_pages - 1, -1, -1))

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def _upload(self, b: int, lo: int, hi: int) -> None:
        self.table[b, lo:hi].copy_(torch.tensor(self._held[b][lo:hi], dtype=torch.int32))

    def reserve(self, lengths) -> None:
        """Gives sequence b the pages of positions [0, lengths[b]) that it
        was not given before (those given back by release_before stay away).
        MemoryError_, and nothing is given, when the pool has too few."""
        pages = [-(-int(n) // self.page_size) for n in lengths]
        _need(len(pages) <= len(self._held), f"{len(pages)} sequences, of at most {len(self._held)}")
        for n, want in zip(lengths, pages):
            _need(want <= self.max_pages,
                  f"a sequence of {int(n)} positions needs {want} pages, of at most {self.max_pages}")
        wanted = sum(max(0, want - len(held)) for want, held in zip(pages, self._held))
        if wanted > len(self._free):
            raise MemoryError_(f"paged cache: {wanted} pages wanted, {len(self._free)} free")
        for b, want in enumerate(pages):
            had = len(self._held[b])
            if want > had:
                self._held[b] += [self._free.pop() for _ in range(want - had)]
                self._upload(b, had, want)

    def release_before(self, firsts, sinks: int = 0) -> None:
        """Gives back the pages of sequence b that lie wholly in positions
        [sinks, firsts[b]): a sliding window has passed them."""
        for b, first in enumerate(firsts):
            lo = max(self._passed[b], -(-int(sinks) // self.page_size))
            hi = min(max(0, int(first)) // self.page_size, len(self._held[b]))
            if hi > lo:
                self._free += [p for p in self._held[b][lo:hi] if p >= 0]
                self._held[b][lo:hi] = [-1] * (hi - lo)
                self._passed[b] = hi
                self._upload(b, lo, hi)

    def release(self, b: Optional[int] = None) -> None:
        """Gives back all pages of sequence b (of every sequence)."""
        for s in range(len(self._held)) if b is None else (b,):
            self._free += [p for p in self._held[s] if p >= 0]
            self._held[s] = []
            self._passed[s] = 0
            self.table[s].fill_(-1)
