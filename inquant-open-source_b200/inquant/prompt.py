"""Attention of whole prompts, several requests packed into one launch, and what their keys received.

A serving step hands over the prompts (or chunks of prompts) that arrived since the last one as packed rows:
sequence ``b`` owns rows ``cu_seqlens[b] .. cu_seqlens[b + 1]`` of ``query`` and rows ``cu_seqlens_k[b] ..
cu_seqlens_k[b + 1]`` of ``key`` and ``value``, and its last query sits at its last key.  ``prompt_attention`` is
the causal attention of all of them (``inquant.prefill.prefill_attention`` for one sequence); ``prompt_weights`` adds
up, from the log-sum-exp that it returns, the attention weight every key received, by which
``inquant.dense_paged.evict_tokens`` chooses the tokens that stay in a cache.

The lengths are read on the device: a call makes no host copy of them and can be captured into a CUDA
graph that is replayed for other lengths of the same total.  Scratch comes from PyTorch's allocator, call by
call, so that calls on several streams or in several graphs share none.
"""
from __future__ import annotations

import ctypes

import torch

from . import _native as N


def _rows(t: torch.Tensor) -> torch.Tensor:
    """16-byte aligned rows with unit channel stride; other layouts are copied."""
    ok = t.stride(2) == 1 and t.stride(0) % 8 == 0 and t.stride(1) % 8 == 0 and t.data_ptr() % 16 == 0 \
        and t.stride(0) > 0 and t.stride(1) > 0
    return t if ok else t.clone(memory_format=torch.contiguous_format)


def _rows_apart(t: torch.Tensor) -> bool:
    """Whether no two elements share memory, as it has to be where a kernel writes."""
    end = 1
    for stride, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1):
        if stride < end:
            return False
        end += stride * (size - 1)
    return True


def _check_offsets(name: str, offsets: torch.Tensor, device: torch.device) -> torch.Tensor:
    if offsets.dtype != torch.int32 or offsets.ndim != 1 or offsets.numel() < 2:
        raise ValueError(f"{name} must be an int32 tensor [sequences + 1]")
    if offsets.device != device:
        raise ValueError(f"query and {name} must share a device")
    return offsets.contiguous()


def _check_states(what: str, query: torch.Tensor, key: torch.Tensor) -> None:
    if query.ndim != 3 or key.ndim != 3:
        raise ValueError("Expected query [tokens, Hq, D] and key/value [tokens, H, D]")
    N.require_cuda(query, what)
    if query.dtype not in (torch.float16, torch.bfloat16) or key.dtype != query.dtype:
        raise NotImplementedError(f"{what} takes fp16 or bf16 tensors of one dtype")
    if query.shape[2] not in (64, 128) or key.shape[2] != query.shape[2]:
        raise NotImplementedError(f"{what} requires head_dim 64 or 128")
    if key.shape[1] < 1 or query.shape[1] < 1 or query.shape[1] % key.shape[1]:
        raise ValueError("Query heads must be a multiple of KV heads")
    if key.device != query.device:
        raise ValueError("query, key and value must share a device")


def _scale(scale: float | None, dim: int) -> float:
    scale = dim ** -0.5 if scale is None else float(scale)
    if not scale > 0.0:
        raise ValueError("scale must be positive")
    return scale


def _check_window(window: int | None) -> None:
    if window is not None and window < 1:
        raise ValueError("window must be positive")


def _arguments(query, key, cu_seqlens, cu_seqlens_k, scale, window, weights) -> N.PromptArgs:
    args = N.PromptArgs()
    args.q, args.k = query.data_ptr(), key.data_ptr()
    args.q_stride_t, args.q_stride_h, args.k_stride_t, args.k_stride_h = query.stride(0), query.stride(1), key.stride(0), key.stride(1)
    args.cu_q, args.cu_k, args.n_seq = cu_seqlens.data_ptr(), cu_seqlens_k.data_ptr(), cu_seqlens.numel() - 1
    args.q_rows, args.k_rows = query.shape[0], key.shape[0]
    args.q_heads, args.kv_heads, args.head_dim = query.shape[1], key.shape[1], query.shape[2]
    args.dtype, args.scale, args.window = N.DTYPE_CODE[query.dtype], scale, window
    args.status = N.status_word(query.device).data_ptr()
    need = N.library().inq_prompt_workspace_bytes(args.q_heads, args.kv_heads, args.head_dim, args.q_rows, args.k_rows, args.n_seq,
                                                  int(weights), window)
    if need:
        args.scratch = torch.empty(need, dtype=torch.uint8, device=query.device)     # lives as long as the arguments
        args.workspace, args.workspace_bytes = args.scratch.data_ptr(), need
    return args


def prompt_attention(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, cu_seqlens: torch.Tensor,
                     cu_seqlens_k: torch.Tensor | None = None, *, scale: float | None = None, out: torch.Tensor | None = None,
                     lse: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Causal attention of packed sequences: ``query`` [Tq, Hq, D], ``key`` / ``value`` [Tk, H, D], fp16 or bf16, D 64 or
    128, any strides (rows that do not start on 16 bytes are copied first).  Query i of a sequence with n queries and
    m keys sees its keys 0 .. m - n + i.  Returns the output [Tq, Hq, D] and the natural log-sum-exp of every row's scaled
    logits, fp32 [Hq, Tq].

    ``cu_seqlens_k`` is ``cu_seqlens`` where it is not given (prompts without a history).  A query without a key (n > m)
    gives zeros and -infinity.  Rows that belong to no sequence are left as they were in ``out`` and ``lse``, and a
    value behind a sequence or at a position that a query does not see never reaches that query, infinities and
    NaN included.  Offsets outside the tensors, or falling ones, are cut to what the tensors hold, and set
    ``STATUS_BAD_INDEX`` in the device's status word."""
    host = N.native_call(query)      # the ordinary call in native code, the rest takes the checks and copies below
    if host is not None:
        result = host.prompt_attention(query, key, value, cu_seqlens, cu_seqlens_k, scale, out, lse, N.status_word(query.device).data_ptr())
        if type(result) is int:
            N.check(result, "inq_prompt_attention")
        if result is not None:
            return result
    return _prompt_attention(query, key, value, cu_seqlens, cu_seqlens_k, scale, out, lse)


@torch.no_grad()
def _prompt_attention(query, key, value, cu_seqlens, cu_seqlens_k, scale, out, lse):
    _check_states("prompt_attention", query, key)
    if value.shape != key.shape:
        raise ValueError("Expected query [tokens, Hq, D] and key/value [tokens, H, D]")
    if value.dtype != key.dtype:
        raise NotImplementedError("prompt_attention takes fp16 or bf16 tensors of one dtype")
    if value.device != query.device:
        raise ValueError("query, key and value must share a device")
    scale = _scale(scale, query.shape[2])
    cu_seqlens = _check_offsets("cu_seqlens", cu_seqlens, query.device)
    cu_seqlens_k = cu_seqlens if cu_seqlens_k is None else _check_offsets("cu_seqlens_k", cu_seqlens_k, query.device)
    if cu_seqlens_k.numel() != cu_seqlens.numel():
        raise ValueError("cu_seqlens and cu_seqlens_k must list the same sequences")
    tokens, q_heads, dim = query.shape
    if out is None:
        out = torch.empty((tokens, q_heads, dim), dtype=query.dtype, device=query.device)
    elif out.shape != query.shape or out.dtype != query.dtype or out.device != query.device or (tokens and _rows(out) is not out) \
            or not _rows_apart(out):
        raise ValueError("out must be a [Tq, Hq, D] tensor of the query dtype and device with aligned rows that share no memory")
    if lse is None:
        lse = torch.empty((q_heads, tokens), dtype=torch.float32, device=query.device)
    elif lse.shape != (q_heads, tokens) or lse.dtype != torch.float32 or lse.device != query.device or lse.stride(1) != 1 \
            or not _rows_apart(lse):
        raise ValueError("lse must be an fp32 tensor [Hq, Tq] on the query's device with unit token stride, its rows sharing no memory")
    if tokens == 0:
        return out, lse
    if key.shape[0] == 0:       # no key anywhere: one row that no sequence reaches stands for the tensors
        key = value = torch.zeros((1, key.shape[1], dim), dtype=key.dtype, device=key.device)
        cu_seqlens_k = torch.zeros_like(cu_seqlens)
    query, key, value = _rows(query), _rows(key), _rows(value)
    with torch.cuda.device(query.device):
        args = _arguments(query, key, cu_seqlens, cu_seqlens_k, scale, 0, False)
        args.v, args.out, args.lse = value.data_ptr(), out.data_ptr(), lse.data_ptr()
        args.v_stride_t, args.v_stride_h, args.o_stride_t, args.o_stride_h = value.stride(0), value.stride(1), out.stride(0), out.stride(1)
        args.lse_stride = lse.stride(0)
        N.check(N.library().inq_prompt_attention(ctypes.byref(args), N.stream_pointer(query.device)), "inq_prompt_attention")
    return out, lse


def prompt_weights(query: torch.Tensor, key: torch.Tensor, lse: torch.Tensor, cu_seqlens: torch.Tensor,
                   cu_seqlens_k: torch.Tensor | None = None, *, scale: float | None = None, window: int | None = None,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention weight that every key received: fp32 [H, Tk], the sum over the query heads of a KV head and over the
    queries that see the key of exp(scale * q k - lse), with the ``lse`` that ``prompt_attention`` returned for the same
    arguments.  With ``window`` only the last ``window`` queries of every sequence count (a prompt's end is the
    better judge of what its continuation reads, and costs less).  Sums are fp32 in a fixed order.  Keys that no counted
    query sees get zero; rows of no sequence are left as they were in ``out``."""
    host = N.native_call(query)
    if host is not None and (window is None or type(window) is int and 0 < window <= 0x7fffffff):
        result = host.prompt_weights(query, key, lse, cu_seqlens, cu_seqlens_k, scale, window or 0, out, N.status_word(query.device).data_ptr())
        if type(result) is int:
            N.check(result, "inq_prompt_weights")
        if result is not None:
            return result
    return _prompt_weights(query, key, lse, cu_seqlens, cu_seqlens_k, scale, window, out)


@torch.no_grad()
def _prompt_weights(query, key, lse, cu_seqlens, cu_seqlens_k, scale, window, out):
    _check_states("prompt_weights", query, key)
    scale = _scale(scale, query.shape[2])
    _check_window(window)
    cu_seqlens = _check_offsets("cu_seqlens", cu_seqlens, query.device)
    cu_seqlens_k = cu_seqlens if cu_seqlens_k is None else _check_offsets("cu_seqlens_k", cu_seqlens_k, query.device)
    if cu_seqlens_k.numel() != cu_seqlens.numel():
        raise ValueError("cu_seqlens and cu_seqlens_k must list the same sequences")
    tokens, q_heads, dim = query.shape
    if lse.shape != (q_heads, tokens) or lse.dtype != torch.float32 or lse.device != query.device:
        raise ValueError("lse must be the fp32 tensor [Hq, Tq] that prompt_attention returned")
    if lse.stride(1) != 1:
        lse = lse.contiguous()
    shape = (key.shape[1], key.shape[0])
    if out is None:
        out = torch.empty(shape, dtype=torch.float32, device=query.device)
    elif out.shape != shape or out.dtype != torch.float32 or out.device != query.device or out.stride(1) != 1 or not _rows_apart(out):
        raise ValueError("out must be an fp32 tensor [H, Tk] on the query's device with unit token stride, its rows sharing no memory")
    if key.shape[0] == 0:
        return out
    if tokens == 0:             # no query anywhere: one row that no sequence reaches stands for the tensors
        query = torch.zeros((1, q_heads, dim), dtype=query.dtype, device=query.device)
        lse = torch.zeros((q_heads, 1), dtype=torch.float32, device=query.device)
        cu_seqlens = torch.zeros_like(cu_seqlens_k)
    query, key = _rows(query), _rows(key)
    with torch.cuda.device(query.device):
        args = _arguments(query, key, cu_seqlens, cu_seqlens_k, scale, min(window or 0, 0x7fffffff), True)
        args.lse, args.lse_stride, args.weights, args.weights_stride = lse.data_ptr(), lse.stride(0), out.data_ptr(), out.stride(0)
        N.check(N.library().inq_prompt_weights(ctypes.byref(args), N.stream_pointer(query.device)), "inq_prompt_weights")
    return out
