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
from .prompt import _scale, prompt_attention, prompt_weights


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


def _check_state(name: str, t: torch.Tensor, dtype: torch.dtype, requests: int, heads: int, columns: int, device) -> None:
    if t.ndim != 3 or t.shape[0] != requests or t.shape[1] != heads or t.shape[2] < columns or t.dtype != dtype or t.device != device \
            or (t.shape[2] > 1 and t.stride(2) != 1):
        raise ValueError(f"{name} must be a {dtype} tensor [{requests}, {heads}, >= {columns}] with unit token stride on the pages' device")


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

    A negative length marks an unused row (zeros, nothing stored); a request without tokens gives zeros.  A page id
    outside the pool is never used as an address: its tokens are left out, and ``STATUS_BAD_INDEX`` is set in the
    device's status word, as it is for a length beyond the table.  Two requests may share pages as long as neither
    stores into them.  Returns the output [B, Hq, D], and with weights ``(output, out_weights)``."""
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
    elif out.shape != query.shape or out.dtype != query.dtype or out.device != device or not _aligned(out):
        raise ValueError("out must be a [requests, Hq, D] tensor of the pages' dtype and device with aligned rows")
    if weights is not None:
        _check_state("weights", weights, torch.float32, requests, heads, block_table.shape[1] * page_tokens, device)
        out_weights = weights if out_weights is None else out_weights
    if out_weights is not None:
        _check_state("out_weights", out_weights, torch.float32, requests, heads, block_table.shape[1] * page_tokens, device)
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
    _check_state("out_weights", out_weights, torch.float32, requests, heads, budget, device)
    _check_state("out_positions", out_positions, torch.int32, requests, heads, budget, device)
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
