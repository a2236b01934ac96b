"""A paged cache of keys and values held in 8 bits, and the decode attention
that reads it: the grouped-query counterpart of the 16-bit K/V pools that
``GatherWorkspace`` reads, in half the bytes.

The cache is four tensors that the caller owns: codes float8_e4m3fn
[pages, kv_heads, 64, 128] and scales float32 [pages, kv_heads], for K and for
V.  A value is code * scale; one scale, a power of two, stands for the 64 tokens
of a page in one head.

``store`` writes new tokens behind the ones a request has.  A page's scale is
the smallest 2^e, -40 <= e <= 40, with 448 * 2^e >= the largest magnitude of the
tokens stored in it, never lowered while the page fills: where a token raises
it, the page's earlier codes are scaled down by the ratio of the scales (a power
of two, so only codes that fall below the format's normal range are rounded
again).  Codes round to nearest even and saturate at 448.

``attend`` is softmax attention of a row's query heads, ``heads / kv_heads`` of
them per K/V head, over its first ``lens[r]`` tokens; it returns ``(out, lse)``
as ``latent_attention`` does.
"""
from __future__ import annotations

import functools

import torch

from . import _lib
from ._lib import ptr, require
from .kernels import status_ptr
from .latent_attention import MAX_SCALE, PAGE, _DTYPES, _index, _one_device, _outputs, _rows16, _step


def _cache(k_cache, k_scale, v_cache, v_scale):
    shape = k_cache.shape
    require(len(shape) == 4 and shape[2:] == (PAGE, 128) and v_cache.shape == shape and shape[1] >= 1,
            "k_cache, v_cache: [pages, kv_heads, 64, 128]")
    require(k_cache.dtype is torch.float8_e4m3fn and v_cache.dtype is torch.float8_e4m3fn and k_cache.is_contiguous()
            and v_cache.is_contiguous() and k_cache.data_ptr() % 16 == 0 and v_cache.data_ptr() % 16 == 0,
            "k_cache, v_cache: contiguous float8_e4m3fn, 16-byte aligned")
    require(k_scale.shape == shape[:2] and v_scale.shape == shape[:2] and k_scale.dtype is torch.float32
            and v_scale.dtype is torch.float32 and k_scale.is_contiguous() and v_scale.is_contiguous(),
            "k_scale, v_scale: contiguous float32 [pages, kv_heads]")
    return shape[0], shape[1]


@functools.lru_cache(maxsize=4096)
def workspace_bytes(rows, heads, kv_heads, table_pages) -> int:
    """Device bytes ``attend`` needs besides its outputs (0: one kernel)."""
    return _lib.lib().v1x_kv8_attend_workspace(rows, heads, kv_heads, table_pages)


def store(k_cache, k_scale, v_cache, v_scale, k, v, table, prefix, offsets):
    """Write the rows offsets[r] .. offsets[r + 1] of k and v [tokens, kv_heads,
    128] (bfloat16 / float16) as the tokens prefix[r], prefix[r] + 1, ... of
    request r, whose page i is ``table[r, i]``.

    prefix int32 [requests], offsets int32 [requests + 1] non-decreasing, table
    int32 [requests, pages].  Tokens past the table, or of a page outside the
    cache, are dropped; places of a page behind the last token are left as they
    are.  A call may write a page for one request and one of its places in the
    table only.  Storing the same tokens again changes nothing."""
    pages, heads = _cache(k_cache, k_scale, v_cache, v_scale)
    code = _DTYPES.get(k.dtype)
    require(k.dim() == 3 and k.shape[1:] == (heads, 128) and v.shape == k.shape and k.dtype is v.dtype
            and code is not None, "k, v: [tokens, kv_heads, 128], both bfloat16 or both float16")
    require(_rows16(k) and _rows16(v), "k, v: unit inner stride, rows 16-byte aligned")
    require(prefix.dtype is torch.int32 and prefix.dim() == 1 and prefix.is_contiguous(),
            "prefix: contiguous int32 [requests]")
    requests = prefix.shape[0]
    require(offsets.dtype is torch.int32 and offsets.shape == (requests + 1,) and offsets.is_contiguous(),
            "offsets: contiguous int32 [requests + 1]")
    require(_index(table, requests), "table: int32 [requests, pages] with unit inner stride")
    require(k.is_cuda, "k must be a CUDA tensor (there is no CPU path)")
    device = k.device
    _one_device(device, k_cache, k_scale, v_cache, v_scale, v, table, prefix, offsets)
    if requests == 0 or k.shape[0] == 0:
        return
    _lib.call("v1x_kv8_store", k_cache.data_ptr(), k_scale.data_ptr(), v_cache.data_ptr(), v_scale.data_ptr(), pages,
              heads, k.data_ptr(), _step(k, 0), _step(k, 1), v.data_ptr(), _step(v, 0), _step(v, 1), code, k.shape[0],
              table.data_ptr(), _step(table, 0), table.shape[1], prefix.data_ptr(), offsets.data_ptr(), requests,
              _lib.stream_of(k), device=device)


def attend(q, k_cache, k_scale, v_cache, v_scale, table, lens, scale, out=None, lse=None):
    """Attention of q [rows, heads, 128] (bfloat16 / float16) over the cache:
    s[h, j] = scale * q[r, h, :] . k_j of head h // (heads / kv_heads), token j < lens[r]
    in page ``table[r, j // 64]``.  lens int32 [rows] (at most pages * 64 count;
    negative is 0).  The tokens of a page outside the cache are no tokens.  Below
    2^25 pages x kv_heads and table columns, at most 2^34 rows x kv_heads x columns."""
    pages, kv_heads = _cache(k_cache, k_scale, v_cache, v_scale)
    code = _DTYPES.get(q.dtype)
    require(code is not None and q.dim() == 3 and q.shape[2] == 128, "q: [rows, heads, 128] bfloat16 or float16")
    rows, heads, _ = q.shape
    require(1 <= heads <= 1024 and heads % kv_heads == 0, "heads: a multiple of kv_heads, at most 1024")
    require(_rows16(q), "q: unit inner stride, rows 16-byte aligned")
    require(_index(table, rows), "table: int32 [rows, pages] with unit inner stride")
    require(lens.dtype is torch.int32 and lens.shape == (rows,) and lens.is_contiguous(),
            "lens: contiguous int32 [rows]")
    scale = float(scale)
    require(abs(scale) < MAX_SCALE, "scale: a finite number below 2^127")
    require(q.is_cuda, "q must be a CUDA tensor (there is no CPU path)")
    device = q.device
    _one_device(device, k_cache, k_scale, v_cache, v_scale, table, lens, out, lse)
    out, lse = _outputs(q, (rows, heads, 128), out, lse)
    if rows == 0:
        return out, lse
    size = workspace_bytes(rows, heads, kv_heads, table.shape[1])
    work = q.new_empty(size, dtype=torch.uint8) if size else None
    _lib.call("v1x_kv8_attend", q.data_ptr(), _step(q, 0), _step(q, 1), k_cache.data_ptr(), k_scale.data_ptr(),
              v_cache.data_ptr(), v_scale.data_ptr(), pages, kv_heads, table.data_ptr(), _step(table, 0),
              table.shape[1], lens.data_ptr(), rows, heads, scale, code, out.data_ptr(), lse.data_ptr(), ptr(work), size,
              status_ptr(device), _lib.stream_of(q), device=device)
    return out, lse
