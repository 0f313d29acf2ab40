"""Uncompressed paged cache: decode attention over it, and eviction by accumulated attention weight.

Where the rest of this package makes a cache smaller by coding its tokens, this keeps fewer of them, exactly.
``paged_attention`` attends with one new token per request over pages of 16-bit keys and values (the packed pages'
counterpart is ``inquant_vllm.kernels.paged_decode``), stores that token and keeps up the attention weight that every
cached token has received; ``evict_tokens`` keeps the tokens of most weight.  ``DensePagedCache`` puts both, with
``inquant.prompt``'s attention of whole prompts, behind the bookkeeping of pages and requests.

Pages of one layer are ``[pages, H, page_tokens, D]`` tensors of any strides whose rows start on 16 bytes, D 64 or 128, fp16
or bf16.  Token t of request b lies in page ``block_table[b, t // page_tokens]`` at offset ``t % page_tokens``.
The order of tokens in a cache means nothing to attention, and eviction does not keep it: ``positions`` tells
where in its sequence a cached token stood.  Lengths, tables and positions are read on the device, so that a captured
step serves later lengths.  Scratch comes from PyTorch's allocator, call by call.
"""
from __future__ import annotations

import ctypes

import torch

from . import _native as N
from .prompt import _check_states, _check_window, _rows_apart, _scale, prompt_attention, prompt_weights


def _aligned(t: torch.Tensor) -> bool:
    return t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and all(s % 8 == 0 for s in t.stride()[:-1])


def _check_pages(what: str, key_pages, value_pages, block_table, lengths) -> None:
    N.require_cuda(key_pages, what)
    if key_pages.ndim != 4 or value_pages.shape != key_pages.shape or key_pages.numel() == 0:
        raise ValueError("Expected key and value pages [pages, H, page_tokens, D]")
    if key_pages.dtype not in (torch.float16, torch.bfloat16) or value_pages.dtype != key_pages.dtype:
        raise NotImplementedError(f"{what} takes fp16 or bf16 pages of one dtype")
    if key_pages.shape[3] not in (64, 128):
        raise NotImplementedError(f"{what} requires head_dim 64 or 128")
    if not _aligned(key_pages) or not _aligned(value_pages):
        raise ValueError("the rows of key and value pages must start on 16 bytes and have unit channel stride")
    if block_table.ndim != 2 or block_table.dtype != torch.int32 or block_table.shape[1] < 1 or block_table.stride(1) != 1:
        raise ValueError("block_table must be an int32 tensor [requests, columns] with unit column stride")
    if lengths.shape != (block_table.shape[0],) or lengths.dtype != torch.int32:
        raise ValueError("lengths must be an int32 tensor [requests]")
    if any(t.device != key_pages.device for t in (value_pages, block_table, lengths)):
        raise ValueError("pages, block_table and lengths must share a device")


def _pairs(query: torch.Tensor, key_pages: torch.Tensor) -> int:
    """Pairs of a request and up to 16 query heads of a KV head (of shapes that may not have been checked yet)."""
    if query.ndim != 3 or key_pages.ndim != 4 or key_pages.shape[1] < 1:
        return 1
    heads = key_pages.shape[1]
    return max(query.shape[0] * heads * ((query.shape[1] // heads + 15) // 16), 1)


def _check_state(name: str, t: torch.Tensor, dtype: torch.dtype, requests: int, heads: int, columns: int, device, written: bool = False) -> None:
    if t.ndim != 3 or t.shape[0] != requests or t.shape[1] != heads or t.shape[2] < columns or t.dtype != dtype or t.device != device \
            or (t.shape[2] > 1 and t.stride(2) != 1):
        raise ValueError(f"{name} must be a {dtype} tensor [{requests}, {heads}, >= {columns}] with unit token stride on the pages' device")
    if written and not _rows_apart(t):
        raise ValueError(f"the rows of {name} must share no memory")


def paged_attention(query: torch.Tensor, key_pages: torch.Tensor, value_pages: torch.Tensor, block_table: torch.Tensor,
                    lengths: torch.Tensor, *, scale: float | None = None, new_key: torch.Tensor | None = None,
                    new_value: torch.Tensor | None = None, weights: torch.Tensor | None = None, out_weights: torch.Tensor | None = None,
                    out: torch.Tensor | None = None):
    """Attention of one token per request, ``query`` [B, Hq, D], over the ``lengths`` [B] cached tokens of each.

    ``new_key`` / ``new_value`` [B, H, D]: the token's own row is stored behind the cached ones (``lengths`` is not changed,
    the layers of a model share it) and attended to.  ``weights`` fp32 [B, H, >= columns * page_tokens]: the weight
    that every token received so far; ``out_weights`` (``weights`` itself where it is not given) gets it plus this
    step's, summed over the query heads of a KV head; the new token starts from zero.  ``out_weights`` alone gets this
    step's.  Entries behind a request's tokens are left as they were.

    A negative length marks an unused row (zeros, nothing stored); a request without tokens gives zeros, one whose logits are
    all -infinity NaN, as the formula does.  A page id
    outside the pool is never used as an address: its tokens are left out, a new one among them is not stored, and
    ``STATUS_BAD_INDEX`` is set in the device's status word, as it is for a length beyond the table.  Two requests may share pages as long as neither
    stores into them.  With weights the call takes scratch of 4 bytes per query head and token that the table can
    hold.  Returns the output [B, Hq, D], and with weights ``(output, out_weights)``."""
    host = N.native_call(query)      # the ordinary call in native code, the rest takes the checks and copies below
    if host is not None:
        device = query.device
        counters = N.launch_counters(device, _pairs(query, key_pages))
        result = host.paged_attention(query, key_pages, value_pages, block_table, lengths, scale, new_key, new_value, weights, out_weights, out,
                                      N.status_word(device).data_ptr(), counters)
        if type(result) is int:
            N.check(result, "inq_paged_attention")
        if result is not None:
            return result
    return _paged_attention(query, key_pages, value_pages, block_table, lengths, scale, new_key, new_value, weights, out_weights, out)


@torch.no_grad()
def _paged_attention(query, key_pages, value_pages, block_table, lengths, scale, new_key, new_value, weights, out_weights, out):
    _check_pages("paged_attention", key_pages, value_pages, block_table, lengths)
    pages, heads, page_tokens, dim = key_pages.shape
    requests, device = block_table.shape[0], key_pages.device
    if query.ndim != 3 or query.shape[0] != requests or query.shape[2] != dim or query.shape[1] < 1 or query.shape[1] % heads:
        raise ValueError("Expected query [requests, Hq, D] with query heads a multiple of KV heads")
    if query.dtype != key_pages.dtype:
        raise NotImplementedError("paged_attention takes a query of the pages' dtype")
    if query.device != device:
        raise ValueError("query and pages must share a device")
    scale = _scale(scale, dim)
    if (new_key is None) != (new_value is None):
        raise ValueError("new_key and new_value come together")
    rows = [query]
    if new_key is not None:
        for t in (new_key, new_value):
            if t.shape != (requests, heads, dim) or t.dtype != query.dtype or t.device != device:
                raise ValueError("new_key and new_value must be [requests, H, D] tensors of the pages' dtype and device")
        rows += [new_key, new_value]
    rows = [t if _aligned(t) else t.clone(memory_format=torch.contiguous_format) for t in rows]
    if out is None:
        out = torch.empty(query.shape, dtype=query.dtype, device=device)
    elif out.shape != query.shape or out.dtype != query.dtype or out.device != device or not _aligned(out) or not _rows_apart(out):
        raise ValueError("out must be a [requests, Hq, D] tensor of the pages' dtype and device with aligned rows that share no memory")
    if weights is not None:
        _check_state("weights", weights, torch.float32, requests, heads, block_table.shape[1] * page_tokens, device)
        out_weights = weights if out_weights is None else out_weights
    if out_weights is not None:
        _check_state("out_weights", out_weights, torch.float32, requests, heads, block_table.shape[1] * page_tokens, device, written=True)
    if requests == 0:
        return out if out_weights is None else (out, out_weights)
    lengths = lengths.contiguous()
    args = N.PagedAttentionArgs()
    args.q, args.k, args.v, args.out = rows[0].data_ptr(), key_pages.data_ptr(), value_pages.data_ptr(), out.data_ptr()
    args.q_stride_b, args.q_stride_h = rows[0].stride(0), rows[0].stride(1)
    args.o_stride_b, args.o_stride_h = out.stride(0), out.stride(1)
    args.k_stride_p, args.k_stride_h, args.k_stride_t = key_pages.stride()[:3]
    args.v_stride_p, args.v_stride_h, args.v_stride_t = value_pages.stride()[:3]
    if new_key is not None:
        args.new_k, args.new_k_stride_b, args.new_k_stride_h = rows[1].data_ptr(), rows[1].stride(0), rows[1].stride(1)
        args.new_v, args.new_v_stride_b, args.new_v_stride_h = rows[2].data_ptr(), rows[2].stride(0), rows[2].stride(1)
    if weights is not None:
        args.weights, args.w_stride_b, args.w_stride_h = weights.data_ptr(), weights.stride(0), weights.stride(1)
    if out_weights is not None:
        args.out_weights, args.ow_stride_b, args.ow_stride_h = out_weights.data_ptr(), out_weights.stride(0), out_weights.stride(1)
    args.table, args.lengths, args.table_stride, args.pages = block_table.data_ptr(), lengths.data_ptr(), block_table.stride(0), pages
    args.requests, args.q_heads, args.kv_heads, args.head_dim = requests, query.shape[1], heads, dim
    args.page_tokens, args.table_columns, args.dtype, args.scale = page_tokens, block_table.shape[1], N.DTYPE_CODE[query.dtype], scale
    args.status = N.status_word(device).data_ptr()
    with torch.cuda.device(device):
        need = N.library().inq_paged_attention_workspace_bytes(ctypes.byref(args))
        scratch = torch.empty(need, dtype=torch.uint8, device=device)
        args.workspace, args.workspace_bytes = scratch.data_ptr(), need
        counters = N.launch_counters(device, _pairs(query, key_pages))
        args.counters = counters.data_ptr()
        N.check(N.library().inq_paged_attention(ctypes.byref(args), N.stream_pointer(device)), "inq_paged_attention")
    return out if out_weights is None else (out, out_weights)


def evict_tokens(key_pages: torch.Tensor, value_pages: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor,
                 weights: torch.Tensor, positions: torch.Tensor, seen: torch.Tensor, budget: int, *, sink: int = 4, recent: int = 128,
                 out_weights: torch.Tensor | None = None, out_positions: torch.Tensor | None = None,
                 out_lengths: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Cuts every request to ``budget`` tokens per KV head, in place in the pages.

    First the tokens stay whose position is below ``sink`` or among the last ``recent`` of the ``seen`` [B] that the
    request has had, then those of most accumulated ``weights`` [B, H, T] (NaN last; ties: the one that lies first).  A
    kept token behind the budget moves into a place that falls free in front of it, the i-th into the i-th, with its key
    and value row, its weight and its ``positions`` [B, H, T] entry (int32); the others stay in place.  Requests within
    the budget are left alone.

    Returns the new ``(lengths, weights, positions)``, written into ``out_...`` where those are given; each may be its
    input.  The first ``budget`` columns of weights and positions are written, with 0 and -1 where no token is.  ``lengths``
    and ``seen`` are int32 [B]; pages of a request that evicts belong to it alone.  A page id outside the pool is not
    used, and sets ``STATUS_BAD_INDEX``, as does a length beyond the table or the columns of ``weights`` (it
    counts as that)."""
    host = N.native_call(key_pages)
    if host is not None and type(budget) is int and type(sink) is int and type(recent) is int and 0 < budget < 2 ** 31 and abs(sink) + abs(recent) < 2 ** 31:
        result = host.evict_tokens(key_pages, value_pages, block_table, lengths, weights, positions, seen, budget, sink, recent, out_weights,
                                   out_positions, out_lengths, N.status_word(key_pages.device).data_ptr())
        if type(result) is int:
            N.check(result, "inq_evict_tokens")
        if result is not None:
            return result
    return _evict_tokens(key_pages, value_pages, block_table, lengths, weights, positions, seen, budget, sink, recent, out_weights, out_positions,
                         out_lengths)


@torch.no_grad()
def _evict_tokens(key_pages, value_pages, block_table, lengths, weights, positions, seen, budget, sink, recent, out_weights, out_positions,
                  out_lengths):
    _check_pages("evict_tokens", key_pages, value_pages, block_table, lengths)
    pages, heads, page_tokens, dim = key_pages.shape
    requests, device = block_table.shape[0], key_pages.device
    budget, sink, recent = int(budget), int(sink), int(recent)
    if budget < 1 or sink < 0 or recent < 0 or sink + recent > budget:
        raise ValueError("budget must be positive and hold sink and recent tokens")
    if budget > 0x3fffffff:
        raise ValueError("budget exceeds 2^30 - 1")
    if seen.shape != lengths.shape or seen.dtype != torch.int32 or seen.device != device:
        raise ValueError("seen must be an int32 tensor [requests] on the pages' device")
    _check_state("weights", weights, torch.float32, requests, heads, 1, device)
    _check_state("positions", positions, torch.int32, requests, heads, weights.shape[2], device)
    if out_weights is None:
        out_weights = torch.empty((requests, heads, budget), dtype=torch.float32, device=device)
    if out_positions is None:
        out_positions = torch.empty((requests, heads, budget), dtype=torch.int32, device=device)
    if out_lengths is None:
        out_lengths = torch.empty_like(lengths, memory_format=torch.contiguous_format)
    _check_state("out_weights", out_weights, torch.float32, requests, heads, budget, device, written=True)
    _check_state("out_positions", out_positions, torch.int32, requests, heads, budget, device, written=True)
    if out_lengths.shape != lengths.shape or out_lengths.dtype != torch.int32 or out_lengths.device != device or not out_lengths.is_contiguous():
        raise ValueError("out_lengths must be a contiguous int32 tensor [requests] on the pages' device")
    if requests == 0:
        return out_lengths, out_weights, out_positions
    lengths, seen = lengths.contiguous(), seen.contiguous()
    args = N.EvictArgs()
    args.k, args.v = key_pages.data_ptr(), value_pages.data_ptr()
    args.k_stride_p, args.k_stride_h, args.k_stride_t = key_pages.stride()[:3]
    args.v_stride_p, args.v_stride_h, args.v_stride_t = value_pages.stride()[:3]
    args.table, args.lengths, args.seen, args.table_stride = block_table.data_ptr(), lengths.data_ptr(), seen.data_ptr(), block_table.stride(0)
    for name, short, t in (("weights", "w", weights), ("positions", "p", positions), ("out_weights", "ow", out_weights),
                           ("out_positions", "op", out_positions)):
        setattr(args, name, t.data_ptr())
        setattr(args, short + "_stride_b", t.stride(0))
        setattr(args, short + "_stride_h", t.stride(1))
    args.out_lengths, args.pages, args.columns = out_lengths.data_ptr(), pages, weights.shape[2]
    args.requests, args.kv_heads, args.head_dim, args.page_tokens = requests, heads, dim, page_tokens
    args.table_columns, args.budget, args.sink, args.recent = block_table.shape[1], budget, sink, recent
    args.status = N.status_word(device).data_ptr()
    with torch.cuda.device(device):
        need = N.library().inq_evict_workspace_bytes(requests, heads, budget, block_table.shape[1] * page_tokens)
        scratch = torch.empty(need, dtype=torch.uint8, device=device)
        args.workspace, args.workspace_bytes = scratch.data_ptr(), need
        N.check(N.library().inq_evict_tokens(ctypes.byref(args), N.stream_pointer(device)), "inq_evict_tokens")
    return out_lengths, out_weights, out_positions


class PromptStep:
    """The prompts (or chunks of prompts) of one step of a ``DensePagedCache``: what its layers share."""

    def __init__(self, cache: "DensePagedCache", requests: list, tokens: list[int]):
        device = cache.device
        self.cache, self.requests, self.tokens = cache, list(requests), [int(n) for n in tokens]
        if len(set(self.requests)) != len(self.requests) or len(self.requests) != len(self.tokens) or not self.requests:
            raise ValueError("one positive token count per request, every request once")
        if min(self.tokens) < 1:
            raise ValueError("one positive token count per request, every request once")
        self.slots = [cache.slot(r) for r in self.requests]
        self.past = [cache._held[s] for s in self.slots]
        cache._reserve([(slot, past + n) for slot, past, n in zip(self.slots, self.past, self.tokens)])
        self.reserved = [list(cache._pages[s]) for s in self.slots]
        starts, keys = [0], [0]
        for past, n in zip(self.past, self.tokens):
            starts.append(starts[-1] + n)
            keys.append(keys[-1] + past + n)
        self.cu_seqlens = torch.tensor(starts, dtype=torch.int32).to(device)
        self.cu_seqlens_k = self.cu_seqlens if not any(self.past) else torch.tensor(keys, dtype=torch.int32).to(device)
        # where every key row lies (request by request: cached tokens, then new ones), and which rows are new
        pages, offsets, new = [], [], []
        for slot, past, n in zip(self.slots, self.past, self.tokens):
            t = torch.arange(past + n)
            pages.append(torch.tensor(cache._pages[slot])[t // cache.page_tokens])
            offsets.append(t % cache.page_tokens)
            new.append(t >= past)
        self.pages, self.offsets = torch.cat(pages).to(device), torch.cat(offsets).to(device)
        is_new = torch.cat(new).to(device)
        self.new_pages, self.new_offsets = self.pages[is_new], self.offsets[is_new]
        self.done = False

    def _check(self) -> None:
        if self.done:
            raise RuntimeError("state mismatch: this step was finished")
        cache, n = self.cache, [len(p) for p in self.reserved]
        if [cache._slots.get(r) for r in self.requests] != self.slots or [cache._held[s] for s in self.slots] != self.past \
                or [cache._pages[s][:k] for s, k in zip(self.slots, n)] != self.reserved:
            raise RuntimeError("state mismatch: the cache has changed since this step began")

    @torch.no_grad()
    def attend(self, layer: int, query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, *, scale: float | None = None,
               window: int | None = None) -> torch.Tensor:
        """Attention of the step's packed rows ``query`` [T, Hq, D] over what the cache holds and over themselves; ``key`` and
        ``value`` [T, H, D] are stored.  In a cache with weights, what every key received from the last ``window``
        queries of its request (all of them where it is not given) is added to its weight."""
        cache = self.cache
        self._check()
        total = sum(self.tokens)
        if query.ndim != 3 or query.shape[0] != total:
            raise ValueError("Expected query [tokens of the step, Hq, D]")
        if key.shape != (total, cache.kv_heads, cache.head_dim) or value.shape != key.shape or key.dtype != cache.dtype or value.dtype != key.dtype:
            raise ValueError("Expected key/value [tokens of the step, H, D] of the cache's dtype")
        if any(t.device != cache.device for t in (query, key, value)):
            raise ValueError("query, key, value and the cache must share a device")
        # all that the calls below refuse, before the rows are stored
        _check_states("prompt_attention", query, key)
        _scale(scale, cache.head_dim)
        if cache.weights is not None:
            _check_window(window)
        key_pages, value_pages = cache.key_pages[layer], cache.value_pages[layer]
        key_pages[self.new_pages, :, self.new_offsets] = key
        value_pages[self.new_pages, :, self.new_offsets] = value
        if self.cu_seqlens_k is not self.cu_seqlens:
            key, value = key_pages[self.pages, :, self.offsets], value_pages[self.pages, :, self.offsets]
        out, lse = prompt_attention(query, key, value, self.cu_seqlens, self.cu_seqlens_k, scale=scale)
        if cache.weights is not None:
            received = prompt_weights(query, key, lse, self.cu_seqlens, self.cu_seqlens_k, scale=scale, window=window)
            at = 0
            for slot, past, n in zip(self.slots, self.past, self.tokens):
                row = cache.weights[layer, slot]
                row[:, :past] += received[:, at:at + past]
                row[:, past:past + n] = received[:, at + past:at + past + n]
                at += past + n
        return out

    @torch.no_grad()
    def finish(self) -> None:
        """Every layer has attended: the requests hold the step's tokens from now on."""
        cache = self.cache
        self._check()
        self.done = True
        for slot, past, n in zip(self.slots, self.past, self.tokens):
            if cache.positions is not None:
                cache.positions[:, slot, :, past:past + n] = torch.arange(cache._seen[slot], cache._seen[slot] + n, device=cache.device, dtype=torch.int32)
            cache._held[slot] = past + n
            cache._seen[slot] += n
            cache._changes[slot] += 1
        cache._write_lengths()


class DensePagedCache:
    """Uncompressed paged cache of several requests and layers, with an optional budget per KV head.

    ``begin_prompt(requests, tokens)`` opens a step of packed prompts (``attend`` per layer, then ``finish``);
    ``begin_decode()`` opens a step of one token per request, ``decode(layer, query, key, value)`` attends with them, and
    ``advance()`` behind the last layer takes them into account, unless the cache has changed in between;
    ``evict(budget)``, between steps, cuts every request to its budget and gives back the pages that fell
    empty.  Rows of a decode call are slots (``slot(request)``); slots without a request give zeros.  ``lengths``,
    ``seen`` and ``block_table`` live on the device, so that decode calls can be captured into a CUDA graph; pages are
    handed out by ``begin_decode``, which is not captured, and neither is ``advance``.

    ``gather`` returns the tokens of a request as dense rows, for instance for ``InQuantCache.update``: what is left after
    an eviction can be coded like any other cache."""

    def __init__(self, layers: int, kv_heads: int, head_dim: int, *, pages: int, max_requests: int, max_tokens: int, page_tokens: int = 64,
                 dtype: torch.dtype = torch.bfloat16, device="cuda", weights: bool = True):
        if min(layers, kv_heads, pages, max_requests, max_tokens, page_tokens) < 1:
            raise ValueError("layers, heads, pages, requests and tokens must be positive")
        if head_dim not in (64, 128) or dtype not in (torch.float16, torch.bfloat16):
            raise NotImplementedError("the cache holds fp16 or bf16 rows of 64 or 128 channels")
        self.layers, self.kv_heads, self.head_dim, self.page_tokens, self.max_tokens = layers, kv_heads, head_dim, page_tokens, max_tokens
        self.dtype, self.device, self.max_requests = dtype, torch.device(device), max_requests
        if self.device.type == "cuda" and self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        columns = -(-max_tokens // page_tokens)
        shape = (layers, pages, kv_heads, page_tokens, head_dim)
        self.key_pages = torch.empty(shape, dtype=dtype, device=self.device)
        self.value_pages = torch.empty(shape, dtype=dtype, device=self.device)
        self.block_table = torch.full((max_requests, columns), -1, dtype=torch.int32, device=self.device)
        self.lengths = torch.full((max_requests,), -1, dtype=torch.int32, device=self.device)
        self.seen = torch.zeros((max_requests,), dtype=torch.int32, device=self.device)
        self.weights = self.positions = None
        if weights:
            self.weights = torch.zeros((layers, max_requests, kv_heads, columns * page_tokens), dtype=torch.float32, device=self.device)
            self.positions = torch.zeros(self.weights.shape, dtype=torch.int32, device=self.device)
        self._slots: dict = {}                                   # request -> slot
        self._free_slots = list(range(max_requests))[::-1]
        self._free_pages = list(range(pages))[::-1]
        self._pages: list[list[int]] = [[] for _ in range(max_requests)]
        self._held, self._seen = [0] * max_requests, [0] * max_requests
        self._changes = [0] * max_requests                       # of a slot: all that a decode step must not meet on its way
        self._step: dict[int, int] | None = None                 # slots of the open decode step, as many changes as they had had

    # ------------------------------------------------------------------ bookkeeping
    def slot(self, request) -> int:
        if request not in self._slots:
            raise KeyError(f"unknown request {request!r}")
        return self._slots[request]

    def admit(self, request) -> int:
        """Gives a request a slot."""
        if request in self._slots:
            raise ValueError(f"request {request!r} is in the cache already")
        if not self._free_slots:
            raise RuntimeError("no free slot: release a request first")
        self._slots[request] = slot = self._free_slots.pop()
        self._held[slot] = self._seen[slot] = 0
        self._changes[slot] += 1
        self._write_lengths()
        return slot

    def release(self, request) -> None:
        slot = self.slot(request)
        del self._slots[request]
        self._free_pages += self._pages[slot][::-1]
        self._pages[slot] = []
        self._free_slots.append(slot)
        self._write_lengths()
        self._write_table()

    def tokens(self, request) -> int:
        """Cached tokens of a request; ``seen`` counts the evicted ones too."""
        return self._held[self.slot(request)]

    @property
    def free_pages(self) -> int:
        return len(self._free_pages)

    def _reserve(self, wanted: list[tuple[int, int]]) -> None:
        """Pages for (slot, tokens) pairs: all of them, or none and an error."""
        for _, tokens in wanted:
            if tokens > self.max_tokens:
                raise ValueError(f"a request of {tokens} tokens exceeds max_tokens")
        need = [max(-(-tokens // self.page_tokens) - len(self._pages[slot]), 0) for slot, tokens in wanted]
        if sum(need) > len(self._free_pages):
            raise RuntimeError("no free pages: evict tokens or release a request first")
        for (slot, _), n in zip(wanted, need):
            self._pages[slot] += [self._free_pages.pop() for _ in range(n)]
        if any(need):
            self._write_table()

    def _write_table(self) -> None:
        table = torch.full(self.block_table.shape, -1, dtype=torch.int32)      # a place that nobody reserved is nobody's page
        for slot, pages in enumerate(self._pages):
            table[slot, :len(pages)] = torch.tensor(pages, dtype=torch.int32)
        self.block_table.copy_(table)

    def _write_lengths(self) -> None:
        used = set(self._slots.values())
        self.lengths.copy_(torch.tensor([n if s in used else -1 for s, n in enumerate(self._held)], dtype=torch.int32))
        self.seen.copy_(torch.tensor(self._seen, dtype=torch.int32))

    # ------------------------------------------------------------------ steps
    def begin_prompt(self, requests: list, tokens: list[int]) -> PromptStep:
        """A step of packed prompts: ``tokens[i]`` new tokens of ``requests[i]``, behind what it holds.  Pages are reserved here."""
        return PromptStep(self, requests, tokens)

    def begin_decode(self) -> None:
        """Opens a step: reserves a place for one more token of every request."""
        self._reserve([(slot, self._held[slot] + 1) for slot in self._slots.values()])
        self._open_step()

    def _open_step(self) -> None:
        self._step = {slot: self._changes[slot] for slot in self._slots.values()}

    def decode(self, layer: int, query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, *, scale: float | None = None,
               out: torch.Tensor | None = None) -> torch.Tensor:
        """Attention of one new token per slot, ``query`` [max_requests, Hq, D], over the cached ones and itself; ``key`` and
        ``value`` [max_requests, H, D] are stored.  Places come from ``begin_decode``."""
        weights = None if self.weights is None else self.weights[layer]
        got = paged_attention(query, self.key_pages[layer], self.value_pages[layer], self.block_table, self.lengths, scale=scale, new_key=key,
                              new_value=value, weights=weights, out=out)
        if self._step is None:       # without begin_decode: a step whose tokens have room in the pages that there are
            self._open_step()
        return got if weights is None else got[0]

    @torch.no_grad()
    def advance(self) -> None:
        """Every layer has decoded: the requests hold one more token each.  Refused where requests came in, got a chunk of
        their prompt or lost tokens or pages since the step was opened: the step's tokens are not all there, and it is
        begun again.  A request may have been released."""
        step = self._step or {}
        if any(step.get(s) != self._changes[s] or self._held[s] + 1 > len(self._pages[s]) * self.page_tokens for s in self._slots.values()):
            raise RuntimeError("state mismatch: begin_decode reserves the places of a step's tokens, and the cache has changed since")
        self._step = None
        if self.positions is not None:
            place = self.lengths.clamp(0, self.positions.shape[3] - 1).long().view(1, -1, 1, 1).expand(self.layers, -1, self.kv_heads, 1)
            self.positions.scatter_(3, place, self.seen.view(1, -1, 1, 1).expand(self.layers, -1, self.kv_heads, 1))
        for slot in self._slots.values():
            self._held[slot] += 1
            self._seen[slot] += 1
        self._write_lengths()

    def evict(self, budget: int, *, sink: int = 4, recent: int = 128) -> None:
        """Cuts every request to ``budget`` tokens per KV head and layer, see ``evict_tokens``."""
        if self.weights is None:
            raise RuntimeError("the cache was built without weights")
        if budget < 1 or sink < 0 or recent < 0 or sink + recent > budget:
            raise ValueError("budget must be positive and hold sink and recent tokens")
        if all(self._held[s] <= budget for s in self._slots.values()):
            return
        left = torch.empty_like(self.lengths)
        for layer in range(self.layers):
            evict_tokens(self.key_pages[layer], self.value_pages[layer], self.block_table, self.lengths, self.weights[layer],
                         self.positions[layer], self.seen, budget, sink=sink, recent=recent, out_weights=self.weights[layer],
                         out_positions=self.positions[layer], out_lengths=left)
        self.lengths.copy_(left)
        for slot in self._slots.values():
            keep = -(-min(self._held[slot], budget) // self.page_tokens)
            if self._held[slot] > budget or keep < len(self._pages[slot]):
                self._changes[slot] += 1
            self._held[slot] = min(self._held[slot], budget)
            self._free_pages += self._pages[slot][keep:][::-1]
            del self._pages[slot][keep:]
        self._write_table()

    @torch.no_grad()
    def gather(self, layer: int, request) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor | None]:
        """Key and value rows [1, H, tokens, D] of a request as they lie in the cache, and their positions [H, tokens]."""
        slot = self.slot(request)
        n = self._held[slot]
        t = torch.arange(n)
        page = torch.tensor(self._pages[slot], dtype=torch.long)[t // self.page_tokens].to(self.device)
        offset = (t % self.page_tokens).to(self.device)
        rows = [p[layer][page, :, offset].transpose(0, 1).unsqueeze(0).contiguous() for p in (self.key_pages, self.value_pages)]
        return rows[0], rows[1], None if self.positions is None else self.positions[layer, slot, :, :n].clone()
