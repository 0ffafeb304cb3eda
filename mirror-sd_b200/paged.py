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

without a host synchronisation.  ``cache.fork`` starts a request from another
one's rows, whose pages both then hold.  The same operators as plain functions on
tensors are ``paged_reserve``, ``paged_release``, ``q4_append``, ``q4_read``
and ``q4_attention``, and, where requests hold pages together, ``paged_fork``,
``paged_reserve_forked``, ``q4_copy_pages`` and ``paged_release_forked``.  Number format and page layout: ``csrc/q4.cuh``.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Sequence, Union

import torch

from . import _native as N

PAGE_SIZES = (16, 32, 64, 128, 256)
HEAD_DIM = 128
# Cached rows, times kv heads, that sharing has to spare to pay for its two more launches.  1 to 8 kv heads, groups of 2 to
# 256 requests of 1 to 16 rows, us shared / on their own: at 2^19 of them 34 shapes of 39 lose (64 requests on 8 kv heads 36 /
# 32, on one 49 / 29), at 2^20 32 of 37 gain (64 requests on 8 kv heads 37 / 47, 16 groups of 16 on one 41 / 50).
LEAST_SPARED = 1 << 20
MAX_GROUP_ROWS = 65536              # query rows that one pass of the attention takes of a request or a group
BLOCK_BYTES = 2304                   # 16 rows of one kv head, K and V with their scales
STATUS_BITS = {1: "too few free pages", 2: "a request outgrew its row of the block table",
               4: "more new rows than slots", 8: "more pages came back than were lent",
               16: "a NaN or an infinity was appended", 32: "a device-side wait expired",
               64: "a request brought more query rows than max_rows, or starts do not fit q",
               128: "a fork named no request, or one that held rows already",
               256: "new rows would have gone into a page of other requests behind the request's rows"}


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


def page_holders(num_pages: int, device="cuda") -> torch.Tensor:
    """Counts of a cache whose pages several requests may hold: int32
    [2, num_pages], row 0 the requests beyond the first that hold each page, row 1
    the operators' own (zero between calls)."""
    if num_pages < 1:
        raise ValueError("num_pages must be positive")
    return torch.zeros(2, num_pages, dtype=torch.int32, device=device)


def paged_fork(src, dst, lens, pages, table, holders, page_size: int, rows=None, status=None, refused=None):
    """Request dst[j] takes over the first rows[j] rows (all without ``rows``)
    of request src[j]: it holds the same pages, and no cached row moves.  src, dst
    and rows are int32 device vectors.  dst[j] must hold nothing and be named once;
    a fork that cannot be made is skipped and sets a bit of ``status``.  The table
    and ``holders`` change in place; returns (lens, pages) afterwards.  From then
    on the cache reserves and releases with the operators below."""
    return N.load_paged().fork(src, dst, rows, lens, pages, table, holders, page_size, status, refused)


def paged_reserve_forked(lens, new_rows, pages, table, free_pages, head, holders, page_size: int, num_slots: int,
                         status=None, refused=None):
    """``paged_reserve`` where requests may hold pages together: one whose new
    rows go into such a page gets a page of its own first.  Returns (PagedStep,
    copies [n, 3]): old page, new page and rows to copy of each request (-1, -1, 0
    where it keeps its page), for ``q4_copy_pages`` before rows are appended.  Pages
    that a trim left behind a request's rows must not be held by others where its
    new rows go (such a request is turned away): ``paged_release_forked`` first."""
    *step, copies = N.load_paged().reserve_forked(lens, new_rows, pages, table, free_pages, head, holders, page_size, num_slots,
                                                  status, refused)
    return PagedStep._make(step), copies


def paged_release_forked(keep, pages, table, free_pages, head, holders, page_size: int, status=None):
    """``paged_release`` where a page goes back once its last holder gives it up."""
    return N.load_paged().release_forked(keep, pages, table, free_pages, head, holders, page_size, status)


def q4_copy_pages(pools: Sequence[torch.Tensor], copies) -> None:
    """Copy pages in every pool of the list: copies [n, 3] int32 on the device
    holds page, page to copy to, and how many of its rows (in whole blocks of 16).
    Entries with -1 are skipped; no page may be copied to twice, or both to and
    from."""
    N.load_paged().copy_pages(list(pools), copies)


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


class PrefixPlan(NamedTuple):
    """What ``paged_prefix_plan`` found, for all layers of a step: per group its
    first packed row, the rows that its members share and whose table row names
    them; per request the pages of those rows and its own rows behind them; and
    what the plan was made for."""
    group_starts: torch.Tensor
    prefix: torch.Tensor
    row_of: torch.Tensor
    skip: torch.Tensor
    own_lens: torch.Tensor
    starts: Optional[torch.Tensor]
    max_rows: int
    max_group: int
    page_size: int
    causal: bool
    shares: bool          # whether any group may share something


def paged_prefix_plan(table, lens, groups, page_size: int, starts=None, max_rows: int = 1, causal: bool = False,
                      max_group: Optional[int] = None, least: int = LEAST_SPARED // 8) -> PrefixPlan:
    """Which cached rows the requests of each group share, found by comparing
    their rows of the block table on the device: whole pages that all members with
    query rows begin with and whose rows all their query rows see.  groups: the
    sizes of consecutive runs of requests, or an int32 device tensor of their
    boundaries [g + 1] with ``max_group``, the requests of a group at most (where one
    has more, the attention's ``status`` says so, its rows are right).  Requests
    of no group are on their own, and where sharing would spare fewer than ``least``
    cached rows from being read, over all groups, all of them are (8 samples of 2,048
    rows each take 18 us on their own, 28 shared).  What is spared is counted in the
    pages found alike; the default is for 8 kv heads, with others 2 ** 20 over their
    number.  lens, starts, max_rows and causal as for ``q4_attention``."""
    if not torch.is_tensor(groups):
        sizes = [int(s) for s in groups]
        if not sizes or any(s < 1 for s in sizes) or sum(sizes) > lens.numel():
            raise ValueError(f"groups must be positive sizes of {lens.numel()} requests at most, got {sizes}")
        bounds = [0]
        for s in sizes:
            bounds.append(bounds[-1] + s)
        max_group = max(sizes) if max_group is None else max_group
        others = sum(sizes) - len(sizes)          # members beyond each group's first
        if lens.is_cuda and N.load_paged().capturing(lens.device.index):
            raise ValueError("groups must be on the device in a CUDA graph, whose replays cannot read the host's")
        groups = torch.tensor(bounds, dtype=torch.int32).to(lens.device, non_blocking=True)
    elif max_group is None:
        raise ValueError("max_group is needed with groups on the device")
    else:
        others = lens.numel() - 1                 # at most: device groups may be empty
    # (known on the host where the table itself is too narrow for `least` rows to be spared; the device, whose groups
    # may not be what the host takes them for, is then told to share nothing either)
    shares = max_group > 1 and others * table.shape[1] * page_size >= max(least, 1)
    least = least if shares else 1 << 62
    return PrefixPlan(*N.load_paged().prefix_plan(table, lens, starts, max_rows, page_size, groups, causal, least), starts,
                      max_rows, max_group, page_size, bool(causal), shares)


def _prefix_group(max_rows: int, max_group: int) -> int:
    """The requests of max_rows rows each that one pass takes of a group of max_group."""
    return min(max_group, max(MAX_GROUP_ROWS // max(max_rows, 1), 1))


def _shared_group(plan: Optional[PrefixPlan], rows: int) -> int:
    """The max_group with which prefix attention takes a plan's groups, 0 where it does not: nothing is shared, or a group
    may have more of the step's rows than one pass takes."""
    if plan is None or not plan.shares:
        return 0
    group = _prefix_group(plan.max_rows, plan.max_group)
    return group if plan.max_rows * group >= min(rows, plan.max_rows * plan.max_group) else 0


def _prefix_workspace_size(rows, max_rows, max_group, num_heads, num_kv_heads, device) -> int:
    with torch.cuda.device(device):
        size = N.load().dflash_q4_prefix_workspace_size(rows, max_rows, _prefix_group(max_rows, max_group), num_heads, num_kv_heads)
    if size == 0:
        raise ValueError(f"no such attention: {rows} rows, groups of {max_group} x {max_rows}, {num_heads} / {num_kv_heads} heads")
    return size


def q4_prefix_workspace(rows: int, max_rows: int, max_group: int, num_heads: int, num_kv_heads: int, device="cuda") -> torch.Tensor:
    """Workspace of ``q4_prefix_attention`` for up to ``rows`` query rows in all,
    ``max_rows`` a request and ``max_group`` requests a group; it may serve any
    number of calls that do not overlap."""
    device = torch.device(device)
    if device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    return torch.zeros(_prefix_workspace_size(rows, max_rows, max_group, num_heads, num_kv_heads, device), dtype=torch.uint8,
                       device=device)


def q4_prefix_attention(q, pool, table, plan: PrefixPlan, scale: Optional[float] = None, out=None, status=None, workspace=None):
    """``q4_attention`` (without a window) of the requests that ``plan`` was made
    for: the rows that a group shares are read once for all its query rows, each
    request's own rows for its own, and both are joined in fp32.  Where max_rows *
    max_group and the rows of q both pass 65,536, every request is read on its own."""
    if pool.dim() != 4 or q.dim() != 3:
        raise ValueError("q must be [rows, heads, 128] and pool a tensor from q4_pool()")
    if pool.shape[2] * 16 != plan.page_size:
        raise ValueError(f"the plan is for pages of {plan.page_size} rows, the pool's have {pool.shape[2] * 16}")
    group = _shared_group(plan, q.shape[0])
    if not group:
        lens = plan.own_lens + plan.skip * plan.page_size if plan.shares else plan.own_lens
        return q4_attention(q, pool, table, lens, plan.starts, plan.max_rows, plan.causal, 0, 0, scale, out, status, workspace)
    if workspace is None:
        workspace = q4_prefix_workspace(q.shape[0], plan.max_rows, group, q.shape[1], pool.shape[1], pool.device)
    return N.load_paged().prefix_attention(q, pool, table, plan.starts, plan.max_rows, plan.group_starts, plan.prefix, plan.row_of,
                                           group, plan.skip, plan.own_lens, plan.causal,
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
    caller's to order like calls on different streams.

    With ``forkable``, ``fork`` lets requests hold pages together: several
    continuations of one prompt, or many prompts that begin alike.  ``reserve``
    then copies a page, in all layers, before a request writes into one that others
    hold, and ``release`` counts holders."""

    def __init__(self, num_layers: int, num_pages: int, num_kv_heads: int, max_seqs: int, max_len: int,
                 page_size: int = 64, device="cuda", capturable: bool = False, forkable: bool = False):
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
        self.holders = page_holders(num_pages, self.device) if forkable else None
        self._trimmed = False
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
                state += [self.holders] if self.holders is not None else []
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
        if self.holders is None:
            step = paged_reserve(self.lens, new_rows, self.pages, self.table, self.free_pages, self.head, self.page_size,
                                 num_slots, self.status, self._refused)
        else:
            if self._trimmed or self.capturable:      # (a graph's replays may follow any trim)
                self._give_back()                     # pages behind the rows may be held with others
            step, copies = paged_reserve_forked(self.lens, new_rows, self.pages, self.table, self.free_pages, self.head,
                                                self.holders, self.page_size, num_slots, self.status, self._refused)
            q4_copy_pages(self.pools, copies)
        self._keep(lens=step.lens, pages=step.pages, head=step.head)
        return step

    def fork(self, src: Union[int, torch.Tensor, Sequence[int]], dst: Union[torch.Tensor, Sequence[int]],
             rows: Union[None, int, torch.Tensor, Sequence[int]] = None) -> None:
        """Request dst[j], which must hold nothing, goes on from the first rows[j]
        rows (default: all) of request src[j] (one number: of that request).  Their
        pages are held together and copied where one is written into; ``check``
        reports what could not be forked.  Device tensors are int32 vectors."""
        if self.holders is None:
            raise RuntimeError("a PagedKVCacheQ4 whose requests fork must be made with forkable=True")
        self._enter()
        if not torch.is_tensor(dst):
            dst = [int(d) for d in dst]
            if any(not 0 <= d < self.max_seqs for d in dst) or len(set(dst)) != len(dst):
                raise ValueError(f"requests to fork into must be distinct and lie in [0, {self.max_seqs})")
        count = len(dst)
        named = {"src": src, "dst": dst, "rows": rows}
        for name, v in named.items():
            if v is None or torch.is_tensor(v):
                continue
            v = [int(v)] * count if isinstance(v, int) else [int(x) for x in v]
            if len(v) != count or (name == "rows" and any(x < 0 for x in v)) or \
                    (name == "src" and any(not 0 <= x < self.max_seqs for x in v)):
                raise ValueError(f"{name} must be {count} numbers, requests in [0, {self.max_seqs}) and rows not negative")
            named[name] = self._upload(v, name)
        if self._trimmed or self.capturable:      # (a request trimmed to nothing holds pages until then)
            self._give_back()
        lens, pages = paged_fork(named["src"], named["dst"], self.lens, self.pages, self.table, self.holders, self.page_size,
                                 named["rows"], self.status, self._refused)
        self._keep(lens=lens, pages=pages)

    def append(self, layer: int, k, v, step: PagedStep) -> None:
        self._on_stream()
        q4_append(k, v, step.slots, self.pools[layer], self.status)

    def prefix_plan(self, step: PagedStep, groups: Union[torch.Tensor, Sequence[int]], max_rows: int, causal: bool = True,
                    max_group: Optional[int] = None, least: Optional[int] = None) -> PrefixPlan:
        """For ``attend``, once a step: the rows that consecutive requests share
        (``paged_prefix_plan``; groups are their numbers, as forks of one prompt lie
        side by side)."""
        self._enter()
        return paged_prefix_plan(self.table, self.lens, groups, self.page_size, step.starts, max_rows, causal, max_group,
                                 LEAST_SPARED // self.nkv if least is None else least)

    def attend(self, layer: int, q, step: PagedStep, max_rows: int, causal: bool = True, sink: int = 0,
               window: int = 0, scale: Optional[float] = None, out=None, workspace=None, plan: Optional[PrefixPlan] = None):
        """Attention of the step's query rows over everything cached; with a
        ``plan`` of the step, what its groups share is read once for all of them.
        Without a ``workspace`` (``q4_attention_workspace``, ``q4_prefix_workspace``)
        the object uses one of its own for each stream; a call that is captured in
        a CUDA graph gets one of the graph's, zeroed at every replay."""
        stream = self._enter()
        if plan is not None and (sink or window or max_rows != plan.max_rows or bool(causal) != plan.causal):
            raise ValueError("a plan goes with the max_rows and causal that it was made for, and without a window")
        group = _shared_group(plan, q.shape[0])
        if workspace is None:
            # (prefix attention keeps sums of every row: sizes by the next power of two)
            key = (1 << max(q.shape[0] - 1, 0).bit_length(), max_rows, group, q.shape[1]) if group else (max_rows, q.shape[1])
            size = self._sizes.get(key)
            if size is None:
                of = _prefix_workspace_size if group else _workspace_size
                size = self._sizes[key] = of(*key, self.nkv, self.device)
            # A graph may be replayed on any stream, beside eager calls and other graphs, and long after a larger
            # workspace has taken this one's place: it shares none with them.
            own = None if self.capturable and self._capturing() else self._workspace
            workspace = own.get(stream) if own is not None else None      # calls on different streams may overlap
            if workspace is None or workspace.nbytes < size:
                workspace = torch.zeros(size, dtype=torch.uint8, device=self.device)
                if own is not None:
                    own[stream] = workspace
        if plan is not None:
            return q4_prefix_attention(q, self.pools[layer], self.table, plan, scale, out, self.status, workspace)
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
        self._trimmed = True
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
        self._give_back()

    def _give_back(self) -> None:
        if self.holders is None:
            pages, head = paged_release(self.lens, self.pages, self.table, self.free_pages, self.head, self.page_size,
                                        self.status)
        else:
            pages, head = paged_release_forked(self.lens, self.pages, self.table, self.free_pages, self.head, self.holders,
                                               self.page_size, self.status)
        self._keep(pages=pages, head=head)
        self._trimmed = False

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
