"""Attention whose keys and values come from one shared latent vector a token:
what a row of the selection path runs next, straight from the latent pool.

A token's pool row is ``dim`` wide: ``latent`` values shared by every head and
the ``dim - latent`` rotary ones (576 = 512 + 64).  Two forms of the same
attention:

absorbed (``attend_slots``, ``attend_pages``): the key projection has been
  multiplied into the query (q is ``dim`` wide per head) and the value projection
  is applied to the output afterwards, so every head reads the same rows,

      s[h, j] = scale * q[r, h, :] . pool[slot_j, :]
      out[r, h, :] = sum_j softmax_j(s[h, :]) pool[slot_j, :latent]

  ``attend_slots`` over a row's own list of slots -- the physical ids that the
  selection writes (``SelectionStep.physical``, ``Indexer.query``); it takes the
  lists that ``GatherWorkspace.gather`` takes and needs no gathered copy.
  ``attend_pages`` over a row's whole context through its native page table.
expanded (``attend_prompt``): keys and values projected per head, for a prompt's
  own tokens, where every query sees many keys,

      s[i, j] = scale * (q[i, h, :dn] . k[j, h, :] + q[i, h, dn:] . k_rope[j, :])

Every function returns ``(out, lse)``: the attention in q's type and the
natural logarithm of the sum of exp(s) per row and head (float32).  A row with
no token has out 0 and lse -inf.  Nothing is synchronised; all work is on the
current stream of q's device, workspaces come from torch's allocator per call,
so calls on several streams and captured graphs share nothing.  A wait inside a
kernel that runs out (2 s) is reported in the device's status word, which
``kernels.check_status`` reads; the call's result is then of no use.
"""
from __future__ import annotations

import functools

import torch

from . import _lib
from ._lib import ptr, require
from .kernels import status_ptr

PAGE = 64                                           # tokens per page of the native pool
MAX_SCALE = 2.0 ** 127                              # so that scale * log2 e is finite in 32 bits
_DTYPES = {torch.bfloat16: 1, torch.float16: 2}     # codes shared with v1x_pack_q


def _rows16(t) -> bool:
    """Unit inner stride and 16-byte aligned rows (16-bit elements)."""
    stride = t.stride()
    if stride[-1] == 1 and t.data_ptr() % 16 == 0:
        for i in range(len(stride) - 1):
            if stride[i] % 8 and t.shape[i] > 1:
                break
        else:
            return True
    return t.numel() == 0


def _step(t, i: int) -> int:
    """The stride of dimension i; 0 where no second element is reached."""
    return t.stride(i) if t.shape[i] > 1 else 0


def _index(t, rows: int) -> bool:
    """int32 [rows, n] with unit inner stride."""
    return (t.dtype is torch.int32 and t.dim() == 2 and t.shape[0] == rows
            and (t.stride(1) == 1 or t.shape[1] <= 1 or rows == 0))


def _one_device(device, *others) -> None:
    for t in others:
        require(t is None or t.device == device, "tensors on different devices")


def _outputs(q, shape, out, lse):
    if out is None:
        out = q.new_empty(shape)
    else:
        require(out.shape == shape and out.dtype is q.dtype and out.is_contiguous() and out.data_ptr() % 16 == 0,
                "out: contiguous, of q's type, 16-byte aligned, [rows, heads, width of a value]")
    if lse is None:
        lse = q.new_empty(shape[:2], dtype=torch.float32)
    else:
        require(lse.shape == shape[:2] and lse.dtype is torch.float32 and lse.is_contiguous(),
                "lse: contiguous float32 [rows, heads]")
    return out, lse


@functools.lru_cache(maxsize=4096)
def workspace_bytes(rows, heads, count, latent, equal) -> int:
    """Device bytes an absorbed call needs besides its outputs (0: one kernel, no
    parts to join); equal: every row has ``count`` places (``attend_slots``)."""
    return _lib.lib().v1x_latent_attention_workspace(rows, heads, count, latent, equal)


def check_absorbed(q, pool, scale, latent: int = 512) -> tuple[int, float]:
    """What every absorbed call requires of its queries, pool and scale; the type's code and the scale."""
    code = _DTYPES.get(q.dtype)
    require(code is not None and q.dim() == 3, "q: [rows, heads, dim] bfloat16 or float16")
    rows, heads, dim = q.shape
    require(pool.dim() == 3 and pool.shape[1] == 1 and pool.shape[2] == dim and pool.dtype is q.dtype,
            "pool: [slots, 1, dim] of q's type, dim wide as q")
    require(latent in (128, 256, 384, 512) and dim - latent in (0, 64),
            "latent: 128, 256, 384 or 512 wide, with dim - latent 0 or 64")
    require(1 <= heads <= 1024, "heads: 1 to 1024")
    require(_rows16(q) and _rows16(pool), "q, pool: unit inner stride, rows 16-byte aligned")
    scale = float(scale)
    require(abs(scale) < MAX_SCALE, "scale: a finite number below 2^127")
    return code, scale


def _absorbed(q, pool, request_slots, index, count, lens, scale, latent, out, lse):
    code, scale = check_absorbed(q, pool, scale, latent)
    rows, heads, dim = q.shape
    require(q.is_cuda, "q must be a CUDA tensor (there is no CPU path)")
    device = q.device
    _one_device(device, pool, request_slots, index, lens, out, lse)
    out, lse = _outputs(q, (rows, heads, latent), out, lse)
    if rows == 0:
        return out, lse
    size = workspace_bytes(rows, heads, count, latent, lens is None)
    work = q.new_empty(size, dtype=torch.uint8) if size else None
    _lib.call("v1x_latent_attention", q.data_ptr(), _step(q, 0), _step(q, 1), pool.data_ptr(), pool.shape[0],
              _step(pool, 0), ptr(request_slots), 0 if request_slots is None else request_slots.shape[0],
              index.data_ptr(), _step(index, 0), count, ptr(lens), rows, heads, dim, latent, scale, code, out.data_ptr(),
              lse.data_ptr(), ptr(work), size, status_ptr(device), _lib.stream_of(q), device=device)
    return out, lse


def attend_slots(q, pool, request_slots, ids, scale, latent: int = 512, out=None, lse=None):
    """Absorbed attention of row r over the slots ``request_slots[ids[r, j]]``
    (or ``ids[r, j]`` without a slot map).

    q [rows, heads, dim] bfloat16 / float16; pool [slots, 1, dim] of the same
    type; ids int32 [rows, top] with unit inner stride; request_slots int32
    [n] or None.  An id that is negative or outside the map, and a slot
    outside the pool, is no token; a slot named twice counts twice."""
    require(_index(ids, q.shape[0]), "ids: int32 [rows, top] with unit inner stride")
    require(request_slots is None or (request_slots.dtype == torch.int32 and request_slots.dim() == 1
                                      and request_slots.is_contiguous()), "request_slots: contiguous int32 [n]")
    return _absorbed(q, pool, request_slots, ids, ids.shape[1], None, scale, latent, out, lse)


def attend_pages(q, pool, table, lens, scale, latent: int = 512, out=None, lse=None):
    """Absorbed attention of row r over its first ``lens[r]`` tokens, token j in
    slot ``table[r, j // 64] * 64 + j % 64``.

    table int32 [rows, pages] with unit inner stride, lens int32 [rows] (at
    most pages * 64 count; negative is 0).  The tokens of a page outside the
    pool are no tokens."""
    require(_index(table, q.shape[0]), "table: int32 [rows, pages] with unit inner stride")
    require(lens.dtype is torch.int32 and lens.shape == (q.shape[0],) and lens.is_contiguous(),
            "lens: contiguous int32 [rows]")
    return _absorbed(q, pool, None, table, table.shape[1] * PAGE, lens, scale, latent, out, lse)


def attend_prompt(q, k, k_rope, v, offsets, scale, kv_offsets=None, out=None, lse=None):
    """Expanded attention of ragged prompts, causal: request r has the queries
    offsets[r] .. offsets[r + 1] and the keys kv_offsets[r] .. kv_offsets[r + 1]
    (offsets without kv_offsets); its i-th query of nq sees its first
    i + 1 + nk - nq keys, so the queries are the last tokens of the context.

    q [tokens, heads, 128 + dr], k and v [keys, heads, 128], k_rope [keys, dr]
    shared by the heads, dr = 64, or None for dr = 0; all of one type
    (bfloat16 / float16), unit inner stride, rows 16-byte aligned -- views of
    one projection's output or of pool rows are taken as they are.  offsets and
    kv_offsets: int32 [requests + 1], non-decreasing, within the tokens; tokens /
    256 + requests is at most 65535.  Rows
    of q that no request covers are not written in out and lse.  A NaN or an
    infinity among a request's values also reaches queries that come before it
    (0 times it is NaN); other requests' keys and values are never read."""
    code = _DTYPES.get(q.dtype)
    require(code is not None and q.dim() == 3, "q: [tokens, heads, 128 + dr] bfloat16 or float16")
    tokens, heads, width = q.shape
    dr = 0 if k_rope is None else 64
    require(width == 128 + dr, "q: [tokens, heads, 128 + dr], dr 64 with k_rope and 0 without")
    keys = k.shape[0]
    require(k.shape == (keys, heads, 128) and v.shape == k.shape, "k, v: [keys, heads, 128], heads as in q")
    require(k_rope is None or k_rope.shape == (keys, 64), "k_rope: [keys, 64]")
    require(k.dtype is q.dtype and v.dtype is q.dtype and (k_rope is None or k_rope.dtype is q.dtype)
            and _rows16(q) and _rows16(k) and _rows16(v) and (k_rope is None or _rows16(k_rope)),
            "q, k, k_rope, v: one type, unit inner stride, rows 16-byte aligned")
    require(1 <= heads <= 1024, "heads: 1 to 1024")
    scale = float(scale)
    require(abs(scale) < MAX_SCALE, "scale: a finite number below 2^127")
    if kv_offsets is None:
        kv_offsets = offsets
    require(offsets.dtype is torch.int32 and kv_offsets.dtype is torch.int32 and offsets.dim() == 1
            and offsets.is_contiguous() and kv_offsets.is_contiguous() and offsets.shape == kv_offsets.shape
            and offsets.shape[0] >= 1, "offsets, kv_offsets: contiguous int32 [requests + 1]")
    require(q.is_cuda, "q must be a CUDA tensor (there is no CPU path)")
    device = q.device
    _one_device(device, k, k_rope, v, offsets, kv_offsets, out, lse)
    out, lse = _outputs(q, (tokens, heads, 128), out, lse)
    requests = offsets.shape[0] - 1
    if tokens == 0 or requests == 0:
        return out, lse
    _lib.call("v1x_prompt_attention", q.data_ptr(), _step(q, 0), _step(q, 1), k.data_ptr(), _step(k, 0), _step(k, 1),
              ptr(k_rope), 0 if k_rope is None else _step(k_rope, 0), v.data_ptr(), _step(v, 0), _step(v, 1),
              offsets.data_ptr(), kv_offsets.data_ptr(), requests, tokens, keys, heads, dr, scale, code, out.data_ptr(),
              lse.data_ptr(), status_ptr(device), _lib.stream_of(q), device=device)
    return out, lse
