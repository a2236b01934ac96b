"""GPU: attention over lines of few tiles, where most of a call's ranges are empty.

The workspaces hold NaN before each call and the outputs lie inside larger buffers,
so that a row joined from parts that nobody left, or written in another's place,
shows."""
import importlib

import numpy as np
import pytest
import torch

import test_gpu_attention as T
from test_gpu_attention import DEV, check, ints, normal, want_slots

pytestmark = pytest.mark.gpu

L = importlib.import_module("10_20_b200.latent_attention")
K = importlib.import_module("10_20_b200.kv8")


def poison(size):
    """The allocator's next block of `size` bytes holds NaN."""
    if size:
        torch.full((size,), 0xFF, dtype=torch.uint8, device=DEV)


def guarded(rows, heads, width, dtype, behind):
    """out and lse of `rows` rows inside buffers of 3's, `behind` rows after them."""
    out = torch.full((rows + 1 + behind, heads, width), 3.0, dtype=dtype, device=DEV)
    lse = torch.full((rows + 1 + behind, heads), 3.0, device=DEV)
    return out, lse, out[1:rows + 1], lse[1:rows + 1]


def untouched(out, lse, rows):
    return all((t[0] == 3).all() and (t[rows + 1:] == 3).all() for t in (out, lse))


def pages_case(lens, width, heads, dtype="bf16", latent=512):
    rows, dim = len(lens), latent + 64
    pool = torch.full(((rows * width + 2) * 64, 1, dim), float("nan"), dtype=T.TYPES[dtype], device=DEV)
    table = torch.randperm(rows * width + 2, generator=torch.Generator().manual_seed(7))[:rows * width]
    table = table.int().view(rows, width).to(DEV)
    pos = torch.arange(width * 64, device=DEV)
    ids = table.long()[:, pos // 64] * 64 + pos % 64
    live = pos < ints(lens)[:, None]
    pool[ids[live], 0] = normal((int(live.sum()), dim), dtype, 8)
    q = normal((rows, heads, dim), dtype, 9)
    out, lse, o, l = guarded(rows, heads, latent, q.dtype, 2)
    poison(L.workspace_bytes(rows, heads, width * 64, latent, False))
    L.attend_pages(q, pool, table, ints(lens), 0.07, latent=latent, out=o, lse=l)
    check(o, l, want_slots(q, pool, torch.where(live, ids, -1).int(), 0.07, latent, dtype), (lens, width, heads))
    assert untouched(out, lse, rows)


@pytest.mark.parametrize("heads", [1, 24, 64, 128])
@pytest.mark.parametrize("n,width", [(1, 2), (30, 16), (50, 2), (64, 8), (64, 40), (1, 400)])
def test_pages_one_short_row_in_a_wide_table(n, width, heads):
    pages_case([n], width, heads)


@pytest.mark.parametrize("heads", [5, 64, 128])
@pytest.mark.parametrize("rows,at,n", [(3, 1, 30), (16, 9, 5), (16, 0, 64), (16, 15, 1), (200, 140, 63), (40, 0, 1)])
def test_pages_one_row_of_a_padded_batch(rows, at, n, heads):
    lens = [0] * rows
    lens[at] = n
    pages_case(lens, 3, heads, dtype="fp16", latent=128)


@pytest.mark.parametrize("total", [0, 2, 3, 147, 148, 149])
def test_pages_totals_around_the_ranges(total):
    """As many tiles as ranges, one less, one more, two, none: in one row and spread."""
    pages_case([64 * total, 0, 0], 150, 3, latent=128)
    lens = [64 if i < total else 0 for i in range(160)]
    pages_case(lens[::-1], 2, 3, latent=128)


def attend_case(lens, width, kv_heads, heads, dtype="bf16"):
    rows = len(lens)
    c = T.new_cache(rows * width + 1, kv_heads)
    table = np.random.default_rng(11).permutation(rows * width + 1)[:rows * width].reshape(rows, width).astype(np.int32)
    T.fill(c, table, lens, 12)
    q = normal((rows, heads, 128), dtype, 13)
    out, lse, o, l = guarded(rows, heads, 128, q.dtype, max(2, 600 - rows))
    poison(K.workspace_bytes(rows, heads, kv_heads, width))
    K.attend(q, *c, ints(table), ints(lens), 0.09, out=o, lse=l)
    check(o, l, T.want_attend(q, c, table, lens, 0.09, dtype), (lens, width, kv_heads, heads))
    assert untouched(out, lse, rows)


@pytest.mark.parametrize("heads", [1, 8, 16])
@pytest.mark.parametrize("n", [1, 63, 64])
@pytest.mark.parametrize("rows,at,width", [(1, 0, 2), (9, 4, 2), (16, 0, 8), (16, 9, 8), (16, 15, 8), (301, 200, 4)])
def test_attend_one_page_of_a_padded_batch(rows, at, width, n, heads):
    """One K/V head and one row that is not empty: a single page of work, both joins."""
    lens = [0] * rows
    lens[at] = n
    attend_case(lens, width, 1, heads)


@pytest.mark.parametrize("kv_heads,heads", [(1, 5), (2, 8), (1, 40), (8, 8)])
@pytest.mark.parametrize("total", [0, 1, 2, 3])
def test_attend_few_pages(total, kv_heads, heads):
    attend_case([64 * total] + [0] * 11, 5, kv_heads, heads, "fp16")
    attend_case([0] * (12 - total) + [64] * total, 2, kv_heads, heads)
    attend_case([0, 64 * total - 1 if total else 0, 0], 30, kv_heads, heads)
