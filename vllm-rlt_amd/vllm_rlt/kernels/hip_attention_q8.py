"""PyTorch-facing adapter of the 8-bit paged-KV kernels.

A layer of the 8-bit cache is three views:

  key_cache, value_cache  ``[blocks, block_size, kv_heads, head_dim]``, torch.float8_e4m3fn,
                          equal strides, head_dim contiguous
  scales                  ``[blocks, kv_heads, 2]``, torch.uint8, the last dimension contiguous:
                          the biased exponents e of K's and V's scale, 2^(e - 127), of each
                          block of tokens and KV head

and a cached value stands for ``e4m3 * scale``. ``kv_append_q8`` writes it; queries and new rows
are float32, float16 or bfloat16. Host checks, streams, allocation and errors are those of
``hip_attention``: ``ValueError`` for shapes, dtypes and devices, the current stream of the
tensors' device, workspaces from PyTorch's caching allocator, no synchronisation. No counterpart
in the reference, whose cache has the model's dtype.
"""

from __future__ import annotations

import torch

from vllm_rlt.kernels._extension import plain_calls
from vllm_rlt.kernels._hip import library
from vllm_rlt.kernels.hip_attention import _check_int, _on_gpu, dtype_code

CACHE_DTYPE = torch.float8_e4m3fn


def _check_cache_q8(key_cache, value_cache, scales):
    device = key_cache.device
    for name, cache in (("key_cache", key_cache), ("value_cache", value_cache)):
        _on_gpu(name, cache, device)
        if cache.ndim != 4 or cache.dtype != CACHE_DTYPE:
            raise ValueError(f"{name} must be a {CACHE_DTYPE} tensor [blocks, block_size, kv_heads, "
                             "head_dim]")
    if value_cache.shape != key_cache.shape or value_cache.stride() != key_cache.stride():
        raise ValueError("key_cache and value_cache must have the same shape and strides")
    if key_cache.numel() == 0:
        raise ValueError("the cache is empty")
    if key_cache.stride(-1) != 1 and key_cache.shape[-1] > 1:
        raise ValueError("caches must have a contiguous head dimension")
    _on_gpu("scales", scales, device)
    if scales.dtype != torch.uint8 or scales.shape != (key_cache.shape[0], key_cache.shape[2], 2):
        raise ValueError("scales must be a uint8 tensor [blocks, kv_heads, 2]")
    if scales.stride(-1) != 1:
        raise ValueError("scales must have a contiguous last dimension")


def _cache_args(key_cache, value_cache, scales):
    return key_cache.data_ptr(), value_cache.data_ptr(), scales.data_ptr()


def _cache_strides(key_cache, scales):
    return (*key_cache.stride()[:3], *scales.stride()[:2])


def _check_tables(block_tables, context_lengths, device):
    _check_int("block_tables", block_tables, torch.int32, 2, device)
    _check_int("context_lengths", context_lengths, torch.int32, 1, device)
    if block_tables.shape[1] > 1 and block_tables.stride(1) != 1:
        raise ValueError("block_tables rows must be contiguous")
    if context_lengths.shape[0] != block_tables.shape[0]:
        raise ValueError("block_tables and context_lengths must have the same rows")
    return context_lengths.contiguous()


def _check_cu(cu_seqlens_q, sequences, device):
    _check_int("cu_seqlens_q", cu_seqlens_q, torch.int32, 1, device)
    if cu_seqlens_q.shape[0] != sequences + 1:
        raise ValueError("cu_seqlens_q must have one entry more than there are sequences")
    return cu_seqlens_q.contiguous()


def _check_queries(q, key_cache, value_cache, scales, out):
    if q.ndim != 3:
        raise ValueError("q must be [rows, q_heads, head_dim]")
    dtype_code(q.dtype)
    _on_gpu("q", q, q.device)
    _on_gpu("key_cache", key_cache, q.device)
    _check_cache_q8(key_cache, value_cache, scales)
    if key_cache.shape[3] != q.shape[2]:
        raise ValueError("the cache's head_dim differs from the query head_dim")
    if not 0 < q.shape[2] <= 256:
        raise ValueError("the 8-bit cache supports head_dim <= 256")
    if q.shape[1] == 0 or q.shape[1] % key_cache.shape[2]:
        raise ValueError("query heads must be a positive multiple of KV heads")
    if q.stride(-1) != 1:
        q = q.contiguous()
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    elif (out.shape != q.shape or out.dtype != q.dtype or out.device != q.device
          or out.stride(-1) != 1):
        raise ValueError("out must match q's shape, dtype and device, with a contiguous head_dim")
    return q, out


def _workspace(nbytes, device):
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _pointer(tensor):
    return None if tensor is None else tensor.data_ptr()


def _launch(name, device, *args):
    """The entry point on the current stream of the tensors' device, with that device current."""
    lib = library()
    with torch.cuda.device(device):
        lib.check(getattr(lib, name)(*args, torch.cuda.current_stream(device).cuda_stream), name)


def kv_append_q8(key_cache, value_cache, scales, k, v, block_tables, context_lengths,
                 cu_seqlens_q=None):
    """Quantise and append ``k, v : [rows, kv_heads, head_dim]`` to one layer.

    Sequence s holds ``context_lengths[s]`` tokens after the call (its attention's length); rows
    ``cu_seqlens_q[s] : cu_seqlens_q[s + 1]`` are its newest tokens, in order, and go to the last
    positions of its ``block_tables`` row. Without ``cu_seqlens_q`` row s is the one new token of
    sequence s, and a sequence of length 0 appends nothing. A block that holds older tokens of
    the sequence keeps its scale or, where a new value needs more, gets a larger one and its
    older tokens are rounded to it; any other block starts with the scale its new tokens need.
    A block that is written belongs to one of the sequences: shared blocks are copied first.
    """
    plain = plain_calls()
    if plain is not None and plain.append_q8(key_cache, value_cache, scales, k, v, block_tables,
                                             context_lengths, cu_seqlens_q):
        return
    _check_cache_q8(key_cache, value_cache, scales)
    device = key_cache.device
    for name, rows in (("k", k), ("v", v)):
        _on_gpu(name, rows, device)
        if rows.ndim != 3 or rows.shape[1:] != key_cache.shape[2:]:
            raise ValueError(f"{name} must be [rows, {key_cache.shape[2]}, {key_cache.shape[3]}]")
        if rows.stride(-1) != 1 and rows.shape[-1] > 1:
            raise ValueError(f"{name} must have a contiguous head dimension")
    dtype_code(k.dtype)
    if v.dtype != k.dtype or v.shape != k.shape:
        raise ValueError("k and v must have the same shape and dtype")
    context_lengths = _check_tables(block_tables, context_lengths, device)
    sequences = block_tables.shape[0]
    if cu_seqlens_q is not None:
        cu_seqlens_q = _check_cu(cu_seqlens_q, sequences, device)
    elif k.shape[0] != sequences:
        raise ValueError("without cu_seqlens_q, k and v must have one row per sequence")
    if k.shape[0] == 0 or sequences == 0:
        return
    _launch(
        "vrh_kv_append_q8", key_cache.device,
        dtype_code(k.dtype), *_cache_args(key_cache, value_cache, scales),
        *_cache_strides(key_cache, scales), k.data_ptr(), v.data_ptr(), *k.stride()[:2],
        *v.stride()[:2], block_tables.data_ptr(), context_lengths.data_ptr(),
        _pointer(cu_seqlens_q), sequences, k.shape[0], key_cache.shape[2], key_cache.shape[3],
        key_cache.shape[0], key_cache.shape[1], block_tables.shape[1], block_tables.stride(0),
    )


def kv_read_q8(key_cache, value_cache, scales, pages, dtype=torch.bfloat16):
    """The values that ``pages`` (int64 block ids) stand for, rounded to ``dtype``: K and V
    ``[len(pages), block_size, kv_heads, head_dim]``. Ids outside the pool read as zeros."""
    plain = plain_calls()
    if plain is not None:
        read = plain.read_q8(key_cache, value_cache, scales, pages, dtype)
        if read is not None:
            return read
    _check_cache_q8(key_cache, value_cache, scales)
    code = dtype_code(dtype)
    device = key_cache.device
    _check_int("pages", pages, torch.int64, 1, device)
    keys = torch.empty((pages.shape[0], *key_cache.shape[1:]), dtype=dtype, device=device)
    values = torch.empty_like(keys)
    if pages.shape[0] == 0:
        return keys, values
    pages = pages.contiguous()
    _launch(
        "vrh_kv_read_q8", key_cache.device,
        code, keys.data_ptr(), values.data_ptr(), *_cache_args(key_cache, value_cache, scales),
        *_cache_strides(key_cache, scales), pages.data_ptr(), pages.shape[0],
        key_cache.shape[2], key_cache.shape[3], key_cache.shape[0], key_cache.shape[1],
    )
    return keys, values


def paged_attention_q8(q, key_cache, value_cache, scales, block_tables, context_lengths,
                       window: int = 0, *, out=None):
    """Single-query paged attention over the 8-bit cache: ``paged_attention`` with ``scales``;
    ``window`` > 0 keeps the last ``window`` keys. Rows of length 0 give zeros."""
    if type(window) is not int or not 0 <= window < 1 << 31:
        raise ValueError("window must be a nonnegative integer")
    plain = plain_calls()
    if plain is not None and out is None:
        output = plain.decode_q8(q, key_cache, value_cache, scales, block_tables, context_lengths,
                                 window)
        if output is not None:
            return output
    q, out = _check_queries(q, key_cache, value_cache, scales, out)
    context_lengths = _check_tables(block_tables, context_lengths, q.device)
    rows = q.shape[0]
    if block_tables.shape[0] != rows:
        raise ValueError("block_tables and context_lengths must have one row per query row")
    if rows == 0:
        return out
    lib = library()
    nbytes = lib.vrh_paged_decode_q8_workspace_bytes(rows, q.shape[1], q.shape[2],
                                                     key_cache.shape[1], block_tables.shape[1],
                                                     window)
    workspace = _workspace(nbytes, q.device)
    _launch(
        "vrh_paged_decode_q8", key_cache.device,
        dtype_code(q.dtype), out.data_ptr(), q.data_ptr(),
        *_cache_args(key_cache, value_cache, scales), block_tables.data_ptr(),
        context_lengths.data_ptr(), rows, q.shape[1], key_cache.shape[2], q.shape[2],
        key_cache.shape[0], key_cache.shape[1], block_tables.shape[1], block_tables.stride(0),
        *q.stride()[:2], *out.stride()[:2], *_cache_strides(key_cache, scales), window,
        _pointer(workspace), nbytes,
    )
    return out


def paged_prefill_attention_q8(q, key_cache, value_cache, scales, block_tables, context_lengths,
                               cu_seqlens_q, max_seqlen_q, *, out=None):
    """Packed causal prefill over the 8-bit cache, bottom-right aligned per sequence:
    ``paged_prefill_attention`` with ``scales``. Rows of ``out`` that belong to no sequence are
    not written. With ``max_seqlen_q`` <= 8 every query equals its single-query decode bit for
    bit."""
    plain = plain_calls()
    if plain is not None and out is None:
        output = plain.prefill_q8(q, key_cache, value_cache, scales, block_tables, context_lengths,
                                  cu_seqlens_q, max_seqlen_q)
        if output is not None:
            return output
    q, out = _check_queries(q, key_cache, value_cache, scales, out)
    context_lengths = _check_tables(block_tables, context_lengths, q.device)
    sequences = block_tables.shape[0]
    cu_seqlens_q = _check_cu(cu_seqlens_q, sequences, q.device)
    max_seqlen_q = int(max_seqlen_q)
    if q.shape[0] == 0 or sequences == 0:
        return out
    if not 1 <= max_seqlen_q < 1 << 31:
        raise ValueError("max_seqlen_q must be positive")
    lib = library()
    nbytes = lib.vrh_paged_prefill_q8_workspace_bytes(
        dtype_code(q.dtype), sequences, q.shape[0], max_seqlen_q, q.shape[1], key_cache.shape[2],
        q.shape[2], key_cache.shape[1], block_tables.shape[1])
    workspace = _workspace(nbytes, q.device)
    _launch(
        "vrh_paged_prefill_q8", key_cache.device,
        dtype_code(q.dtype), out.data_ptr(), q.data_ptr(),
        *_cache_args(key_cache, value_cache, scales), block_tables.data_ptr(),
        context_lengths.data_ptr(), cu_seqlens_q.data_ptr(), sequences, q.shape[0],
        max_seqlen_q, q.shape[1], key_cache.shape[2], q.shape[2], key_cache.shape[0],
        key_cache.shape[1], block_tables.shape[1], block_tables.stride(0), *q.stride()[:2],
        *out.stride()[:2], *_cache_strides(key_cache, scales), _pointer(workspace), nbytes,
    )
    return out
