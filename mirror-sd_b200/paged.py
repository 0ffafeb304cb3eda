"""Paged 4-bit K/V cache shared by many requests: block tables built on the
GPU, rows appended as 4-bit numbers, attention read straight from them.

The cache of one draft sequence (``DFlashKVCache``) is an f16 ring whose length
the host tracks.  A target model's cache grows by what was accepted, a number
that only the GPU knows after ``accept``, and every request's is as long as its
text.  Here the lengths, the block table and the free pages stay on the device;
one step of a batch is

    step = cache.reserve(new_rows)                     # slots of the new rows
    for layer in range(num_layers):
        cache.append(layer, k, v, step)                # [rows, NKV, 128] each
        o = cache.attend(layer, q, step, max_rows)     # [rows, NQ, 128]
    cache.trim(rejected)                               # lengths only
    cache.release()                                    # spare pages go back

without a host synchronisation.  The same operators as plain functions on
tensors are ``paged_reserve``, ``paged_release``, ``q4_append``, ``q4_read``
and ``q4_attention``.  Number format and page layout: ``csrc/q4.cuh``.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Sequence, Union

import torch

from . import _native as N

PAGE_SIZES = (16, 32, 64, 128, 256)
HEAD_DIM = 128
BLOCK_BYTES = 2304                   # 16 rows of one kv head, K and V with their scales
STATUS_BITS = {1: "too few free pages", 2: "a request outgrew its row of the block table",
               4: "more new rows than slots", 8: "more pages came back than were lent",
               16: "a NaN or an infinity was appended", 32: "a device-side wait expired",
               64: "a request brought more query rows than max_rows, or starts do not fit q"}


class PagedStep(NamedTuple):
    """Result of ``paged_reserve``: where each request's packed rows start
    [n + 1], the slot of every new row [num_slots], and the requests' lengths,
    page counts and the free list's head afterwards."""
    starts: torch.Tensor
    slots: torch.Tensor
    lens: torch.Tensor
    pages: torch.Tensor
    head: torch.Tensor


def _raw_stream(index: int) -> int:
    """current_stream().cuda_stream without the Stream object."""
    return torch._C._cuda_getCurrentRawStream(index)     # (a torch without CUDA lacks it, and still imports this package)


# Arguments are checked, and outputs made, in csrc/paged_binding.cpp.


def paged_reserve(lens, new_rows, pages, table, free_pages, head, page_size: int, num_slots: int,
                  status=None, refused=None) -> PagedStep:
    """Pages and cache slots for the rows that each request brings.

    lens, new_rows, pages [n], table [n, max_pages], free_pages [num_pages] and
    head [1] are int32 device tensors; request i holds lens[i] rows on pages[i]
    pages.  New pages come off ``free_pages`` at ``head`` and are written into
    ``table``; the other inputs are only read.  ``num_slots`` bounds the new
    rows of all requests (known on the host); surplus slots are -1.  A request
    that cannot be served keeps its length and sets a bit of ``status``
    (STATUS_BITS) and its entry of ``refused`` [n], which a request that is
    served clears."""
    return PagedStep._make(N.load_paged().reserve(lens, new_rows, pages, table, free_pages, head, page_size, num_slots,
                                                  status, refused))


def paged_release(keep, pages, table, free_pages, head, page_size: int, status=None):
    """Request i keeps the pages of its first keep[i] rows; the others go back
    into ``free_pages`` below ``head``.  Returns (pages, head) afterwards."""
    return N.load_paged().release(keep, pages, table, free_pages, head, page_size, status)


def q4_pool(num_pages: int, num_kv_heads: int, page_size: int = 64, device="cuda") -> torch.Tensor:
    """An empty pool of one layer: uint8 [num_pages, NKV, page_size / 16, 2304]."""
    if page_size not in PAGE_SIZES:
        raise ValueError(f"page_size must be one of {PAGE_SIZES}")
    if num_pages < 1 or num_kv_heads < 1:
        raise ValueError("num_pages and num_kv_heads must be positive")
    return torch.zeros(num_pages, num_kv_heads, page_size // 16, BLOCK_BYTES, dtype=torch.uint8, device=device)


def q4_append(k, v, slots, pool, status=None) -> None:
    """Quantise the rows k, v [rows, NKV, 128] (f16 or bf16, strided rows and
    heads) into their slots [rows] of the pool; slots must be distinct, and a
    row whose slot is outside the pool is skipped."""
    N.load_paged().append(k, v, slots, pool, status)


def q4_read(pool, slots, dtype=torch.float16):
    """What the cache stands for at ``slots``: (k, v) [rows, NKV, 128], exact
    in f16 and bf16; zeros for a slot outside the pool."""
    if dtype is not torch.float16 and dtype is not torch.bfloat16:
        raise ValueError("dtype must be torch.float16 or torch.bfloat16")
    return N.load_paged().read(pool, slots, dtype is torch.bfloat16)


def _workspace_size(max_rows: int, num_heads: int, num_kv_heads: int, device) -> int:
    with torch.cuda.device(device):
        size = N.load().dflash_q4_attention_workspace_size(max_rows, num_heads, num_kv_heads)
    if size == 0:
        raise ValueError(f"no such attention: {max_rows} rows, {num_heads} / {num_kv_heads} heads")
    return size


def q4_attention_workspace(n: int, max_rows: int, num_heads: int, num_kv_heads: int, device="cuda") -> torch.Tensor:
    """Workspace of ``q4_attention`` for up to ``max_rows`` query rows a
    request and any number n of requests; it may serve any number of calls that
    do not overlap."""
    device = torch.device(device)
    if device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    return torch.zeros(_workspace_size(max_rows, num_heads, num_kv_heads, device), dtype=torch.uint8, device=device)


def q4_attention(q, pool, table, lens, starts=None, max_rows: int = 1, causal: bool = False, sink: int = 0,
                 window: int = 0, scale: Optional[float] = None, out=None, status=None, workspace=None):
    """Grouped-query attention of each request's query rows over its cached
    rows.  q [rows, NQ, 128] (f16 or bf16; strided rows and heads) holds the
    requests' rows one after another: request i owns starts[i] ..
    starts[i + 1] - 1 (at most ``max_rows``: a request with more sets a bit of
    ``status``, and its rows are undefined), or ``max_rows`` each without
    ``starts``.  lens [n] counts the cached rows, the new ones included.

    causal: query row j of m sees the keys below lens - m + j + 1 (else below
    lens); window: of those only the first ``sink`` and the last ``window``.
    A row that sees no key gives zeros; rows of q that no request owns leave
    their rows of ``out`` unwritten.  ``out`` must not overlap q.  scale
    (positive) defaults to 128 ** -0.5."""
    if workspace is None:
        if pool.dim() != 4 or q.dim() != 3:
            raise ValueError("q must be [rows, heads, 128] and pool a tensor from q4_pool()")
        workspace = q4_attention_workspace(lens.numel(), max_rows, q.shape[1], pool.shape[1], pool.device)
    return N.load_paged().attention(q, pool, table, lens, starts, max_rows, causal, sink, window,
                                    HEAD_DIM ** -0.5 if scale is None else scale, out, status, workspace)


class PagedKVCacheQ4:
    """Cache of ``max_seqs`` requests over ``num_layers`` layers.  Every
    method enqueues on the current stream; none waits for the device except
    ``check`` and ``free_page_count``.  Calls on different streams are the
    caller's to order (an event between them); the state's memory then stays
    until the last of the streams is done with it.

    ``lens``, ``pages`` and ``head`` are new tensors after every step, which a
    CUDA graph could not follow: it would start each replay from the lengths
    that it was captured with.  With ``capturable`` they are updated in place
    (three small copies a ``reserve``, two a ``release``), so that every replay
    of captured steps goes on where the last one ended; only then may
    ``reserve``, ``attend``, ``trim`` and ``release`` be captured, with row
    counts on the device (or one number).  Replays and calls in between are the
    caller's to order like calls on different streams."""

    def __init__(self, num_layers: int, num_pages: int, num_kv_heads: int, max_seqs: int, max_len: int,
                 page_size: int = 64, device="cuda", capturable: bool = False):
        if num_layers < 1 or max_seqs < 1 or max_len < 1:
            raise ValueError("num_layers, max_seqs and max_len must be positive")
        self.page_size, self.max_seqs, self.nkv = page_size, max_seqs, num_kv_heads
        self.pools = [q4_pool(num_pages, num_kv_heads, page_size, device) for _ in range(num_layers)]
        self.device = self.pools[0].device
        i32 = dict(dtype=torch.int32, device=self.device)
        self.table = torch.full((max_seqs, -(-max_len // page_size)), -1, **i32)
        self.lens = torch.zeros(max_seqs, **i32)
        self.pages = torch.zeros(max_seqs, **i32)
        self.free_pages = torch.arange(num_pages, **i32)
        self.head = torch.zeros(1, **i32)
        self.status = torch.zeros(1, **i32)
        self._refused = torch.zeros(max_seqs, **i32)      # turned away when it last brought rows
        self.capturable = capturable
        self._workspace, self._sizes = {}, {}
        self._stream = _raw_stream(self.device.index)
        self._streams = {self._stream}

    def _capturing(self) -> bool:
        return N.load_paged().capturing(self.device.index)

    def _keep(self, **state):
        for name, t in state.items():
            if self.capturable:
                getattr(self, name).copy_(t)
            else:
                setattr(self, name, t)

    def _upload(self, values, name: str):
        """Host numbers on the device, without waiting for it."""
        if self._capturing():
            raise ValueError(f"{name} must be on the device in a CUDA graph, whose replays cannot read the host's")
        values = values if torch.is_tensor(values) else torch.tensor(values, dtype=torch.int32)
        return values.to(self.device, non_blocking=True)

    def _on_stream(self) -> int:
        """The current stream.  Where it is another one than the last call's, the
        allocator learns that it uses the state: ``lens``, ``pages`` and ``head``,
        which are new tensors after each step, and, once for a stream, all others."""
        raw = _raw_stream(self.device.index)
        if raw != self._stream:
            self._stream = raw
            state = [self.lens, self.pages, self.head]
            if raw not in self._streams:
                self._streams.add(raw)
                state += [*self.pools, self.table, self.free_pages, self.status, self._refused]
            for t in state:
                t.record_stream(torch.cuda.current_stream(self.device))
        return raw

    def _enter(self) -> int:
        if not self.capturable and self._capturing():
            raise RuntimeError("a PagedKVCacheQ4 in a CUDA graph must be made with capturable=True")
        return self._on_stream()

    def reserve(self, new_rows: Union[torch.Tensor, Sequence[int]], num_slots: Optional[int] = None) -> PagedStep:
        """Make room for new_rows[i] rows of request i (0 where it sits out).
        ``num_slots`` bounds their sum; it is needed when new_rows is a device
        tensor.  A request that cannot be served (``check`` says why) keeps its
        length; its query rows of this step give nothing of use, and ``trim``
        leaves it alone."""
        self._enter()
        if not torch.is_tensor(new_rows):
            num_slots = sum(new_rows) if num_slots is None else num_slots
            new_rows = self._upload(list(new_rows), "new_rows")
        elif num_slots is None:
            raise ValueError("num_slots is needed with new_rows on the device")
        step = paged_reserve(self.lens, new_rows, self.pages, self.table, self.free_pages, self.head, self.page_size,
                             num_slots, self.status, self._refused)
        self._keep(lens=step.lens, pages=step.pages, head=step.head)
        return step

    def append(self, layer: int, k, v, step: PagedStep) -> None:
        self._on_stream()
        q4_append(k, v, step.slots, self.pools[layer], self.status)

    def attend(self, layer: int, q, step: PagedStep, max_rows: int, causal: bool = True, sink: int = 0,
               window: int = 0, scale: Optional[float] = None, out=None, workspace=None):
        """Attention of the step's query rows over everything cached.  Without a
        ``workspace`` (``q4_attention_workspace``) the object uses one of its own
        for each stream; a call that is captured in a CUDA graph gets one of the
        graph's, zeroed at every replay."""
        stream = self._enter()
        if workspace is None:
            key = (max_rows, q.shape[1])
            size = self._sizes.get(key)
            if size is None:
                size = self._sizes[key] = _workspace_size(*key, self.nkv, self.device)
            # A graph may be replayed on any stream, beside eager calls and other graphs, and long after a larger
            # workspace has taken this one's place: it shares none with them.
            own = None if self.capturable and self._capturing() else self._workspace
            workspace = own.get(stream) if own is not None else None      # calls on different streams may overlap
            if workspace is None or workspace.nbytes < size:
                workspace = torch.zeros(size, dtype=torch.uint8, device=self.device)
                if own is not None:
                    own[stream] = workspace
        return q4_attention(q, self.pools[layer], self.table, self.lens, step.starts, max_rows, causal, sink, window,
                            scale, out, self.status, workspace)

    def trim(self, counts: Union[int, torch.Tensor, Sequence[int]]) -> None:
        """Drop the last counts[i] rows of request i (one number: of every
        request).  Pages stay with the request until ``release``.  A request
        that ``reserve`` turned away has no new rows to drop and keeps those it
        holds, until it is served again or ``check`` has raised."""
        self._enter()
        if not torch.is_tensor(counts):
            counts = counts if isinstance(counts, int) else torch.tensor(list(counts), dtype=torch.int32)
            if counts < 0 if isinstance(counts, int) else bool((counts < 0).any()):
                raise ValueError("trim counts must not be negative")
        if torch.is_tensor(counts):
            if counts.shape != self.lens.shape or counts.is_floating_point():
                raise ValueError(f"counts must be {self.max_seqs} integers, got {counts.dtype} {tuple(counts.shape)}")
            if counts.device != self.device:
                counts = self._upload(counts, "counts")
            if counts.dtype is not torch.int32:
                counts = counts.to(torch.int64).clamp(min=-1, max=2 ** 31 - 1).to(torch.int32)
            counts = counts.contiguous()
        else:
            counts = min(counts, 2 ** 31 - 1)
        # (a negative count on the device, where nobody can raise, trims nothing)
        self.lens = N.load_paged().trim(self.lens, counts, self._refused, self.lens if self.capturable else None)

    def release(self, seqs: Sequence[int] = ()) -> None:
        """Give spare pages back; requests ``seqs`` are finished and emptied."""
        seqs = [int(s) for s in seqs]
        if any(not 0 <= s < self.max_seqs for s in seqs):
            raise ValueError(f"sequences must lie in [0, {self.max_seqs})")
        self._enter()
        if seqs:
            if self._capturing():
                raise ValueError("finished requests cannot be named in a CUDA graph: every replay would empty them")
            self._keep(lens=self.lens.index_fill(0, torch.tensor(seqs).to(self.device, non_blocking=True), 0))
        pages, head = paged_release(self.lens, self.pages, self.table, self.free_pages, self.head, self.page_size,
                                    self.status)
        self._keep(pages=pages, head=head)

    def read(self, layer: int, seq: int, length: int, dtype=torch.float16):
        """The first ``length`` rows of a request, which it must hold, as
        (k, v) [length, NKV, 128]."""
        if not 0 <= seq < self.max_seqs or not 0 <= length <= self.table.shape[1] * self.page_size:
            raise ValueError(f"no rows 0..{length} of request {seq}")
        self._on_stream()
        pos = torch.arange(length, device=self.device)
        slots = self.table[seq][pos // self.page_size] * self.page_size + (pos % self.page_size).to(torch.int32)
        return q4_read(self.pools[layer], slots.to(torch.int32), dtype)

    def free_page_count(self) -> int:
        return self.free_pages.numel() - int(self.head)

    def check(self) -> None:
        """Raise what any call since the last check recorded on the device."""
        bits = int(self.status)
        if bits:
            self.status.zero_()
            self._refused.zero_()
            if bits & 32:
                self._workspace.clear()     # its counters may be left half way
            raise RuntimeError("paged cache: " + "; ".join(m for b, m in STATUS_BITS.items() if bits & b))
