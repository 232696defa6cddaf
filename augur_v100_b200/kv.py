"""The paged key-value cache of the full-attention layers: pages and who holds them, and the entries that write, read and
move them.

A decoding step of a layer is: projections (``host``), `KvAppend` (rotary positions, optional head norms, the cache
write), `PagedAttention`, output projection. The cache is BF16 (`KvCache`) or in 8 bits (`KvCacheE4m3`); `SharedPrefixAttention` stands in
`PagedAttention`'s place where the sequences begin with the same pages. `KvPagePool` is the host's book of pages: sequences share full pages after a
fork, and what has to be copied (a fork's partly filled page, a compaction's moves) comes back as two lists for
`KvPageCopy`. The reference keeps one contiguous cache per session instead (crates/augur-model-qwen35-runtime); owners
and bindings follow the rules of :mod:`augur_v100_b200.host`: everything is checked once at ``bind``, ``submit`` only
enqueues on the stream it was bound to, and the binding keeps its tensors alive.
"""
from __future__ import annotations

import functools
import heapq
from ctypes import byref, c_uint32, c_uint64
from typing import NamedTuple

import torch

from . import abi
from .host import Plan, Stream, _check, _nbytes, _ptr, allocated, sm_count


def _require(tensor: torch.Tensor, name: str, dtype: torch.dtype, shape: tuple, device: torch.device | None = None) -> torch.Tensor:
    if tensor.dtype != dtype or tuple(tensor.shape) != tuple(shape) or not tensor.is_contiguous():
        raise ValueError(f"{name}: a contiguous {dtype} tensor of shape {tuple(shape)}, not {tensor.dtype} {tuple(tensor.shape)}")
    if device is not None and tensor.device != device:
        raise ValueError(f"{name}: on {device}, not {tensor.device}")
    return tensor


class KvCache:
    """Keys and values of all layers: two BF16 tensors [layers, pages, kv_heads, page_tokens, head_dim]."""

    def __init__(self, keys: torch.Tensor, values: torch.Tensor):
        if keys.dim() != 5:
            raise ValueError("keys: [layers, pages, kv_heads, page_tokens, head_dim]")
        _require(keys, "keys", torch.bfloat16, keys.shape)
        _require(values, "values", torch.bfloat16, keys.shape, keys.device)
        self.keys, self.values = keys, values
        self.layers, self.pages, self.kv_heads, self.page_tokens, self.head_dim = keys.shape

    @classmethod
    def allocate(cls, stream: Stream, layers: int, pages: int, kv_heads: int, page_tokens: int, head_dim: int):
        shape, device = (layers, pages, kv_heads, page_tokens, head_dim), torch.device("cuda", stream.ordinal)
        return cls(*(allocated(stream, torch.empty, shape, dtype=torch.bfloat16, device=device) for _ in range(2)))

    def layer_args(self, layer: int) -> abi.KvLayer:
        if not 0 <= layer < self.layers:
            raise ValueError("no such layer")
        keys, values = self.keys[layer], self.values[layer]
        return abi.KvLayer(_ptr(keys), _ptr(values), _nbytes(keys), self.pages, self.kv_heads, self.page_tokens, self.head_dim)


class KvCacheE4m3:
    """Keys and values of all layers in 8 bits: two tensors of E4M3 codes [layers, pages, kv_heads, page_tokens, head_dim] and
    the scales of every token's heads, E8M0 [layers, pages, kv_heads, page_tokens, 2] (keys, values); an element is code times scale.

    `KvAppend`, `PagedAttention` and `KvPageCopy` take it in a `KvCache`'s place. It holds half the bytes, and attention over it reads half, which makes it
    quicker from some 300 to 1000 tokens a sequence on (one sequence alone: 4000); an element keeps four significant bits (2^-4 relative at most, near a head's largest element as far below it)."""

    def __init__(self, keys: torch.Tensor, values: torch.Tensor, scales: torch.Tensor):
        if keys.dim() != 5:
            raise ValueError("keys: [layers, pages, kv_heads, page_tokens, head_dim]")
        _require(keys, "keys", torch.float8_e4m3fn, keys.shape)
        _require(values, "values", torch.float8_e4m3fn, keys.shape, keys.device)
        _require(scales, "scales", torch.float8_e8m0fnu, (*keys.shape[:4], 2), keys.device)
        self.keys, self.values, self.scales = keys, values, scales
        self.layers, self.pages, self.kv_heads, self.page_tokens, self.head_dim = keys.shape

    @classmethod
    def allocate(cls, stream: Stream, layers: int, pages: int, kv_heads: int, page_tokens: int, head_dim: int):
        shape, device = (layers, pages, kv_heads, page_tokens, head_dim), torch.device("cuda", stream.ordinal)
        codes = [allocated(stream, torch.empty, shape, dtype=torch.float8_e4m3fn, device=device) for _ in range(2)]
        return cls(*codes, allocated(stream, torch.empty, (*shape[:4], 2), dtype=torch.float8_e8m0fnu, device=device))

    def layer_args(self, layer: int) -> abi.KvE4m3Layer:
        if not 0 <= layer < self.layers:
            raise ValueError("no such layer")
        keys, values, scales = self.keys[layer], self.values[layer], self.scales[layer]
        return abi.KvE4m3Layer(_ptr(keys), _ptr(values), _ptr(scales), _nbytes(keys), _nbytes(scales), self.pages, self.kv_heads, self.page_tokens, self.head_dim)


def _entries(cache, name: str, arguments: str):
    """The descriptor and the two entries of an operator for the kind of cache."""
    if isinstance(cache, KvCacheE4m3):
        name, arguments = name + "_e4m3", arguments.replace("Args", "E4m3Args")
    elif not isinstance(cache, KvCache):
        raise ValueError("cache: a KvCache or a KvCacheE4m3")
    lib, prefix = abi.lib(), "augur_cuda_nvfp4_sm100_" + name
    return abi.header(getattr(abi, arguments)), getattr(lib, prefix + "_preflight_v1"), getattr(lib, prefix + "_prevalidated_submit_v1")


def _batch_args(table: torch.Tensor, lengths: torch.Tensor, starts: torch.Tensor, rows: int, device: torch.device) -> abi.KvBatch:
    if table.dim() != 2:
        raise ValueError("page table: [sequences, pages]")
    sequences = table.shape[0]
    _require(table, "page table", torch.int32, table.shape, device)
    _require(lengths, "lengths", torch.int32, (sequences,), device)
    _require(starts, "token starts", torch.int32, (sequences + 1,), device)
    return abi.KvBatch(_ptr(table), _nbytes(table), _ptr(lengths), _nbytes(lengths), _ptr(starts), _nbytes(starts),
                       sequences, table.shape[1], rows, 0)


def _strided(tensor: torch.Tensor, name: str, rows: int, heads: int, head_dim: int, device: torch.device):
    """Address, bytes from the first to the last element, row and head stride of a [rows, heads, head_dim] view."""
    if tensor.dtype != torch.bfloat16 or tuple(tensor.shape) != (rows, heads, head_dim) or tensor.stride(2) != 1 or tensor.device != device:
        raise ValueError(f"{name}: a BF16 tensor of shape {(rows, heads, head_dim)} on {device} with contiguous heads")
    # the stride of a dimension of one element says nothing
    row = tensor.stride(0) if rows > 1 else heads * head_dim
    head = tensor.stride(1) if heads > 1 else head_dim
    return _ptr(tensor), 2 * ((rows - 1) * row + (heads - 1) * head + head_dim), row, head


class KvAppend:
    """Rotary positions on a step's queries and keys, and its keys and values written to one layer's pages.

    `q` [rows, query_heads, head_dim], `k` and `v` [rows, kv_heads, head_dim]: BF16, rows and heads strided as the
    projections leave them. `positions` int32 [3, rows] (time, height, width; equal for text), `frequencies` f32
    [rotary_dim / 2], `sections` how many rotary pairs each axis turns. Optional `q_norm` / `k_norm` f32 [head_dim]: RMSNorm of
    every head first. Rows of sequence b are [starts[b], starts[b + 1]), the last of the lengths[b] tokens that its pages hold
    with them, any number of them."""

    def __init__(self, stream: Stream, cache: KvCache | KvCacheE4m3, layer: int, q, k, v, positions, frequencies, sections, table, lengths, starts,
                 interleaved: bool, q_out, q_norm, k_norm, epsilon: float):
        rows, query_heads, head_dim = q.shape
        device = cache.keys.device
        self.stream, self.cache, self.q_out = stream, cache, q_out
        self._keep = (q, k, v, positions, frequencies, table, lengths, starts, q_norm, k_norm)
        a, self._preflight, enqueue = _entries(cache, "kv_append", "KvAppendArgs")
        a.layer, a.batch = cache.layer_args(layer), _batch_args(table, lengths, starts, rows, device)
        a.query, a.query_len_bytes, a.query_row_stride, a.query_head_stride = _strided(q, "q", rows, query_heads, cache.head_dim, device)
        a.key, a.key_len_bytes, a.key_row_stride, a.key_head_stride = _strided(k, "k", rows, cache.kv_heads, cache.head_dim, device)
        a.value, a.value_len_bytes, a.value_row_stride, a.value_head_stride = _strided(v, "v", rows, cache.kv_heads, cache.head_dim, device)
        _require(positions, "positions", torch.int32, (3, rows), device)
        a.positions, a.positions_len_bytes = _ptr(positions), _nbytes(positions)
        if len(sections) != 3 or min(sections) < 0:
            raise ValueError("sections: three counts of rotary pairs")
        _require(frequencies, "frequencies", torch.float32, (sum(sections),), device)
        a.inv_freq_f32, a.inv_freq_len_bytes = _ptr(frequencies), _nbytes(frequencies)
        for name, norm in (("query_norm_f32", q_norm), ("key_norm_f32", k_norm)):
            if norm is not None:
                _require(norm, name, torch.float32, (head_dim,), device)
                setattr(a, name, _ptr(norm))
                a.norm_len_bytes = _nbytes(norm)
        _require(q_out, "q_out", torch.bfloat16, (rows, query_heads, head_dim), device)
        a.query_out, a.query_out_len_bytes = _ptr(q_out), _nbytes(q_out)
        a.query_heads, a.rotary_dim, a.interleaved, a.epsilon = query_heads, 2 * sum(sections), int(bool(interleaved)), epsilon
        for i, section in enumerate(sections):
            a.sections[i] = section
        self.args = a
        self._enqueue = functools.partial(enqueue, stream.ordinal, stream.handle, byref(a))

    @classmethod
    def bind(cls, stream: Stream, cache: KvCache | KvCacheE4m3, layer: int, q, k, v, positions, frequencies, sections, table, lengths, starts,
             interleaved: bool = False, q_out: torch.Tensor | None = None, q_norm: torch.Tensor | None = None,
             k_norm: torch.Tensor | None = None, epsilon: float = 1e-6):
        if q_out is None:
            q_out = allocated(stream, torch.empty, q.shape, dtype=torch.bfloat16, device=q.device)
        self = cls(stream, cache, layer, q, k, v, positions, frequencies, sections, table, lengths, starts, interleaved, q_out, q_norm, k_norm,
                   epsilon)
        _check("kv_append_preflight", self._preflight(stream.ordinal, stream.handle, byref(self.args)))
        return self

    def submit(self) -> None:
        _check("kv_append_submit", self._enqueue())


def paged_attention_scratch_bytes(query_heads: int, kv_heads: int, head_dim: int, tokens: int = abi.MAX_SMALL_TOKENS, sms: int = 0) -> int:
    """Plan scratch of a `PagedAttention` of up to `tokens` new tokens per sequence. `sms`: `host.sm_count(stream.ordinal)` of the plan's device (0: of the
    current device; a plan on one with more SMs wants more, and binding to it is refused)."""
    out = c_uint64()
    _check("paged_attention_scratch_extent", abi.lib().augur_cuda_nvfp4_sm100_paged_attention_scratch_extent_host_v1(
        query_heads, kv_heads, head_dim, tokens, sms or sm_count(), byref(out)))
    return int(out.value)


class PagedAttention:
    """Attention of up to `tokens` (1..8) new tokens per sequence over one layer's pages, their own keys and values included:
    `q` [rows, query_heads, head_dim] BF16 (what `KvAppend` leaves in `q_out`) -> `out`, the same shape. Rows outside every
    sequence keep what `out` holds. query_heads / kv_heads * tokens is at most 64."""

    def __init__(self, plan: Plan, cache: KvCache | KvCacheE4m3, layer: int, q, table, lengths, starts, tokens: int, out, scale: float):
        rows, query_heads, head_dim = q.shape
        device = cache.keys.device
        _require(q, "q", torch.bfloat16, (rows, query_heads, cache.head_dim), device)
        _require(out, "out", torch.bfloat16, q.shape, device)
        self.plan, self.cache, self.q, self.out = plan, cache, q, out
        self._keep = (table, lengths, starts)
        a, self._preflight, enqueue = _entries(cache, "paged_attention", "PagedAttentionArgs")
        a.layer, a.batch = cache.layer_args(layer), _batch_args(table, lengths, starts, rows, device)
        a.query, a.query_len_bytes = _ptr(q), _nbytes(q)
        a.output, a.output_len_bytes = _ptr(out), _nbytes(out)
        a.query_heads, a.max_new_tokens, a.scale = query_heads, tokens, scale
        self.args = a
        self._enqueue = functools.partial(enqueue, plan.stream.ordinal, plan.stream.handle, plan.handle, byref(a))

    @classmethod
    def bind(cls, plan: Plan, cache: KvCache | KvCacheE4m3, layer: int, q, table, lengths, starts, tokens: int = 1, out: torch.Tensor | None = None,
             scale: float | None = None):
        if out is None:
            out = allocated(plan.stream, torch.zeros_like, q)
        self = cls(plan, cache, layer, q, table, lengths, starts, tokens, out, cache.head_dim ** -0.5 if scale is None else scale)
        s = plan.stream
        _check("paged_attention_preflight", self._preflight(s.ordinal, s.handle, plan.handle, byref(self.args)))
        return self

    def submit_for_plan(self) -> None:
        _check("paged_attention_submit", self._enqueue())


def shared_prefix_attention_scratch_bytes(query_heads: int, kv_heads: int, head_dim: int, rows: int, tokens: int = abi.MAX_SMALL_TOKENS, sms: int = 0) -> int:
    """Plan scratch of a `SharedPrefixAttention` of `rows` token rows and up to `tokens` new tokens per sequence (`sms` as for `paged_attention_scratch_bytes`)."""
    out = c_uint64()
    _check("shared_prefix_attention_scratch_extent", abi.lib().augur_cuda_nvfp4_sm100_shared_prefix_attention_scratch_extent_host_v1(
        query_heads, kv_heads, head_dim, rows, tokens, sms or sm_count(), byref(out)))
    return int(out.value)


class SharedPrefixAttention:
    """`PagedAttention` over a BF16 cache for sequences that begin with the same tokens (a system prompt, the forks of one conversation), whose keys and
    values are read once for all of them. `prefix_pages` int32 [n]: the pages of those tokens (`KvPagePool.shared_prefix` has them);
    `prefix_tokens` int32 [1]: how many they are, counted in whole pages; both device memory. `lengths` count the shared tokens too, and the
    page table has its columns for them, whatever it says there. Behind the prefix everything is as for `PagedAttention`.

    Which of the two to bind is the caller's choice: this one is quicker where it saves some 150 MB of keys and values of a layer ((sequences - 1) times the
    prefix's), rounds the weights to one BF16 term (2^-8 of each, there 2^-16), and takes the longer the more rows `q` has, used or not."""

    def __init__(self, plan: Plan, cache: KvCache, layer: int, q, table, lengths, starts, prefix_pages, prefix_tokens, tokens: int, out, scale: float):
        if not isinstance(cache, KvCache):
            raise ValueError("cache: a KvCache")
        rows, query_heads, _ = q.shape
        device = cache.keys.device
        _require(q, "q", torch.bfloat16, (rows, query_heads, cache.head_dim), device)
        _require(out, "out", torch.bfloat16, q.shape, device)
        if prefix_pages.dim() != 1 or prefix_pages.shape[0] < 1:
            raise ValueError("prefix pages: [n], at least one")
        _require(prefix_pages, "prefix pages", torch.int32, prefix_pages.shape, device)
        _require(prefix_tokens, "prefix tokens", torch.int32, (1,), device)
        self.plan, self.cache, self.q, self.out = plan, cache, q, out
        self._keep = (table, lengths, starts, prefix_pages, prefix_tokens)
        a, self._preflight, enqueue = _entries(cache, "shared_prefix_attention", "SharedPrefixAttentionArgs")
        a.layer, a.batch = cache.layer_args(layer), _batch_args(table, lengths, starts, rows, device)
        a.prefix_pages, a.prefix_pages_len_bytes = _ptr(prefix_pages), _nbytes(prefix_pages)
        a.prefix_tokens, a.prefix_tokens_len_bytes = _ptr(prefix_tokens), _nbytes(prefix_tokens)
        a.query, a.query_len_bytes = _ptr(q), _nbytes(q)
        a.output, a.output_len_bytes = _ptr(out), _nbytes(out)
        a.query_heads, a.max_new_tokens, a.scale = query_heads, tokens, scale
        self.args = a
        self._enqueue = functools.partial(enqueue, plan.stream.ordinal, plan.stream.handle, plan.handle, byref(a))

    @classmethod
    def bind(cls, plan: Plan, cache: KvCache, layer: int, q, table, lengths, starts, prefix_pages, prefix_tokens, tokens: int = 1,
             out: torch.Tensor | None = None, scale: float | None = None):
        if out is None:
            out = allocated(plan.stream, torch.zeros_like, q)
        self = cls(plan, cache, layer, q, table, lengths, starts, prefix_pages, prefix_tokens, tokens, out,
                   cache.head_dim ** -0.5 if scale is None else scale)
        s = plan.stream
        _check("shared_prefix_attention_preflight", self._preflight(s.ordinal, s.handle, plan.handle, byref(self.args)))
        return self

    def submit_for_plan(self) -> None:
        _check("shared_prefix_attention_submit", self._enqueue())


class KvPageCopy:
    """Copies pages of a cache, keys and values (and scales) of all layers: `submit(sources, destinations)` with two lists of page numbers.
    Destinations are distinct and none is a source; anything else is refused with nothing enqueued."""

    def __init__(self, stream: Stream, cache: KvCache | KvCacheE4m3):
        self.stream, self.cache = stream, cache
        a, self._preflight, enqueue = _entries(cache, "kv_page_copy", "KvPageCopyArgs")
        a.keys, a.values, a.len_bytes = _ptr(cache.keys), _ptr(cache.values), _nbytes(cache.keys)
        a.page_bytes = cache.kv_heads * cache.page_tokens * cache.head_dim * cache.keys.element_size()
        if isinstance(cache, KvCacheE4m3):
            a.scales, a.scales_len_bytes, a.scale_page_bytes = _ptr(cache.scales), _nbytes(cache.scales), cache.kv_heads * cache.page_tokens * 2
        a.layers, a.pages = cache.layers, cache.pages
        self.args = a
        self._enqueue = functools.partial(enqueue, stream.ordinal, stream.handle, byref(a))

    @classmethod
    def bind(cls, stream: Stream, cache: KvCache | KvCacheE4m3):
        self = cls(stream, cache)
        _check("kv_page_copy_preflight", self._preflight(stream.ordinal, stream.handle, byref(self.args)))
        return self

    def submit(self, sources, destinations) -> None:
        count = len(sources)
        if len(destinations) != count:
            raise ValueError("one destination for every source")
        if count and (min(min(sources), min(destinations)) < 0 or max(max(sources), max(destinations)) >= self.cache.pages):
            raise ValueError("a page outside the cache")       # ctypes would wrap a negative number round
        array = c_uint32 * count
        _check("kv_page_copy_submit", self._enqueue(array(*sources), array(*destinations), count))


class PageCopies(NamedTuple):
    """Copies that `KvPageCopy` has to make before the pages are used again."""
    sources: list
    destinations: list


class OutOfPages(RuntimeError):
    """The pool holds too few free pages; nothing was changed."""


class KvPagePool:
    """Which sequence holds which pages of a cache (host memory only; no device work happens here).

    A sequence is a number that `create` or `fork` hands out. Full pages are shared between a sequence and its forks and are
    never written again, a partly filled one is copied at the fork. Where a call answers with `PageCopies`, those are to
    be enqueued (`KvPageCopy.submit`) on the stream of the steps before the next step uses the pages: the answer of each call by
    itself and in the order of the calls, since a later call may give away a page that an earlier one copies from."""

    def __init__(self, pages: int, page_tokens: int):
        if pages < 1 or page_tokens < 1:
            raise ValueError("a pool has pages, and a page tokens")
        self.pages, self.page_tokens = pages, page_tokens
        self._free = list(range(pages))          # a heap: the lowest page first, which keeps the cache compact
        self._holders = [0] * pages
        self._pages: dict[int, list[int]] = {}
        self._length: dict[int, int] = {}
        self._next = 0

    def free_pages(self) -> int:
        return len(self._free)

    def sequences(self) -> list[int]:
        return list(self._pages)

    def length(self, sequence: int) -> int:
        return self._length[sequence]

    def page_list(self, sequence: int) -> list[int]:
        return list(self._pages[sequence])

    def _take(self) -> int:
        page = heapq.heappop(self._free)
        self._holders[page] = 1
        return page

    def _drop(self, page: int) -> None:
        self._holders[page] -= 1
        if self._holders[page] == 0:
            heapq.heappush(self._free, page)

    def create(self) -> int:
        sequence = self._next
        self._next += 1
        self._pages[sequence], self._length[sequence] = [], 0
        return sequence

    def extend(self, sequence: int, tokens: int) -> PageCopies:
        """Room for `tokens` more tokens. A partly filled last page that others hold too (after `truncate`) is replaced by a copy."""
        pages, length = self._pages[sequence], self._length[sequence]
        if tokens < 0:
            raise ValueError("a count of tokens")
        needed = -(-(length + tokens) // self.page_tokens) - len(pages)
        copy = tokens > 0 and length % self.page_tokens != 0 and self._holders[pages[-1]] > 1
        if needed + copy > len(self._free):
            raise OutOfPages(f"{needed + copy} pages wanted, {len(self._free)} free")
        copies = PageCopies([], [])
        if copy:
            page = self._take()
            copies.sources.append(pages[-1])
            copies.destinations.append(page)
            self._drop(pages[-1])
            pages[-1] = page
        pages.extend(self._take() for _ in range(needed))
        self._length[sequence] = length + tokens
        return copies

    def truncate(self, sequence: int, length: int) -> None:
        """Takes the tokens behind `length` back, such as speculated ones that were not accepted."""
        if not 0 <= length <= self._length[sequence]:
            raise ValueError("a length of at most the present one")
        pages, keep = self._pages[sequence], -(-length // self.page_tokens)
        for page in pages[keep:]:
            self._drop(page)
        del pages[keep:]
        self._length[sequence] = length

    def fork(self, sequence: int) -> tuple[int, PageCopies]:
        """A second sequence with the same tokens."""
        pages, length = self._pages[sequence], self._length[sequence]
        partly = length % self.page_tokens != 0
        if partly and not self._free:
            raise OutOfPages("1 page wanted, 0 free")
        shared = pages[:-1] if partly else pages
        for page in shared:
            self._holders[page] += 1
        twin, copies = self.create(), PageCopies([], [])
        self._pages[twin], self._length[twin] = list(shared), length
        if partly:
            page = self._take()
            self._pages[twin].append(page)
            copies.sources.append(pages[-1])
            copies.destinations.append(page)
        return twin, copies

    def free(self, sequence: int) -> None:
        for page in self._pages.pop(sequence):
            self._drop(page)
        del self._length[sequence]

    def shared_prefix(self, sequences) -> list[int]:
        """The pages that all of the sequences (None is an idle slot) begin with, in order; all of them are full. For `SharedPrefixAttention`."""
        held = [(self._pages[s], self._length[s]) for s in sequences if s is not None]
        if not held:
            return []
        full = min(length // self.page_tokens for _, length in held)
        first = held[0][0]
        for i in range(full):
            if any(pages[i] != first[i] for pages, _ in held):
                return first[:i]
        return first[:full]

    def compact(self) -> PageCopies:
        """Moves the pages in use to the front of the cache: the highest ones into the lowest free ones. The tables change at once."""
        used = self.pages - len(self._free)
        holes = sorted(page for page in self._free if page < used)
        movers = [page for page in range(self.pages - 1, used - 1, -1) if self._holders[page]]
        moved = dict(zip(movers, holes))
        for source, destination in moved.items():
            self._holders[destination], self._holders[source] = self._holders[source], 0
        for pages in self._pages.values():
            pages[:] = [moved.get(page, page) for page in pages]
        self._free = list(range(used, self.pages))
        return PageCopies(list(moved), list(moved.values()))

    def table(self, sequences, width: int | None = None) -> torch.Tensor:
        """The page table int32 [sequences, width] (host memory) of a step's sequences, -1 behind their pages; None is an idle slot."""
        lists = [[] if sequence is None else self._pages[sequence] for sequence in sequences]
        longest = max((len(pages) for pages in lists), default=0)
        width = max(longest, 1) if width is None else width
        if longest > width:
            raise ValueError(f"a sequence holds {longest} pages")
        return torch.tensor([pages + [-1] * (width - len(pages)) for pages in lists], dtype=torch.int32).reshape(len(lists), width)
