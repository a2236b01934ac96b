"""GPU: the attention operators against their definitions in 64 bits.

Tolerances are the oracle's bound (oracle/attention.py): the score and softmax
error of 32-bit sums, one rounding of the weights to the type they enter the
product in, one rounding of the result."""
import importlib

import numpy as np
import pytest
import torch

from oracle import attention as A

pytestmark = pytest.mark.gpu

L = importlib.import_module("10_20_b200.latent_attention")
K = importlib.import_module("10_20_b200.kv8")
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
DEV = "cuda:0"


def normal(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(TYPES[dtype])


def ints(x):
    return torch.as_tensor(np.asarray(x, np.int32), device=DEV)


def f64(t):
    return t.detach().to("cpu", torch.float64).numpy()


def check(out, lse, want, what=""):
    o, l, to, tl = want
    o2, l2 = f64(out), f64(lse)
    assert np.all(np.isfinite(o2)), what
    assert np.array_equal(np.isinf(l), np.isinf(l2)), what
    bad = np.abs(o2 - o) > to
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} outside, worst {np.max(np.abs(o2 - o) / to):.3g} of the bound"
    fin = np.isfinite(l)
    assert np.all(np.abs(l2[fin] - l[fin]) <= tl[fin]), f"{what}: lse off by {np.abs(l2[fin] - l[fin]).max()}"


def rounding(dtype):
    """The type's half step for the result and for the weights (the latent and prompt kernels hold the
    weights in the inputs' type); f16 weights underflow below 2^-24."""
    u = A.U[dtype]
    return dict(u=u, up=u, tiny=2.0 ** -24 if dtype == "fp16" else 0.0, smallest=A.SMALLEST[dtype])


# -- absorbed form ----------------------------------------------------------------
def want_slots(q, pool, ids, scale, latent, dtype, req=None):
    qs, kv = f64(q), pool[:, 0]
    rows = []
    for r in range(q.shape[0]):
        at = ids[r].long().cpu()
        if req is not None:
            ok = (at >= 0) & (at < req.shape[0])
            at = torch.where(ok, req.cpu().long()[at.clamp(0, req.shape[0] - 1)], -1)
        at = at[(at >= 0) & (at < pool.shape[0])].to(DEV)
        k = f64(kv[at])
        rows.append(A.softmax_rows(qs[r], k, k[:, :latent], scale, **rounding(dtype)))
    return [np.stack(x) for x in zip(*rows)]


@pytest.mark.parametrize("rows,heads,top,latent,rope,dtype", [
    (1, 1, 1, 512, 64, "bf16"), (3, 5, 63, 512, 64, "fp16"), (2, 64, 64, 512, 64, "bf16"), (2, 65, 65, 512, 64, "bf16"),
    (5, 128, 200, 512, 64, "fp16"), (7, 24, 129, 512, 64, "bf16"), (2, 130, 257, 256, 64, "bf16"),
    (3, 16, 500, 384, 0, "fp16"), (2, 33, 320, 128, 64, "bf16"), (4, 8, 96, 128, 0, "fp16"), (2, 12, 2048, 512, 0, "bf16"),
    (300, 3, 70, 512, 64, "bf16"), (1, 64, 2048, 512, 64, "fp16"), (40, 100, 513, 256, 0, "bf16"),
])
def test_slots(rows, heads, top, latent, rope, dtype):
    dim = latent + rope
    q, pool = normal((rows, heads, dim), dtype, 1), normal((3000, 1, dim), dtype, 2)
    rng = np.random.default_rng(top)
    ids = rng.integers(0, 3000, (rows, top))
    ids[rng.random((rows, top)) < 0.1] = -1
    ids = ints(ids)
    scale = dim ** -0.5
    out, lse = L.attend_slots(q, pool, None, ids, scale, latent=latent)
    assert out.dtype == q.dtype and out.shape == (rows, heads, latent) and lse.shape == (rows, heads)
    check(out, lse, want_slots(q, pool, ids, scale, latent, dtype))


@pytest.mark.parametrize("scale", [0.0, -0.05, 0.6])
def test_slots_scales(scale):
    """Equal weights, reversed order, and rows where one token has all the weight and the maximum keeps rising."""
    q, pool = normal((4, 20, 576), "bf16", 3), normal((700, 1, 576), "bf16", 4)
    ids = torch.arange(700, device=DEV, dtype=torch.int32).repeat(4, 1)
    order = (q[0, 0].float() @ pool[:, 0].float().t()).argsort()
    ids[1] = order.int()
    ids[2] = order.flip(0).int()
    check(*L.attend_slots(q, pool, None, ids, scale), want_slots(q, pool, ids, scale, 512, "bf16"))


@pytest.mark.parametrize("rows,heads,top,latent,rope,dtype", [
    (8, 64, 2048, 512, 64, "bf16"), (10, 3, 640, 128, 0, "fp16"), (30, 70, 300, 256, 64, "bf16"), (14, 33, 575, 384, 64, "fp16"),
    (24, 64, 520, 512, 0, "bf16"), (60, 9, 321, 512, 64, "fp16"), (7, 130, 1000, 128, 64, "bf16"),
])
def test_slots_rows_of_clusters(rows, heads, top, latent, rope, dtype):
    """A few rows, whose CTAs join through shared memory (no workspace): parts of unequal size, a row without a
    token, rows whose tokens are all in one part, a part whose scores dwarf the others'."""
    assert L.workspace_bytes(rows, heads, top, latent, True) == 0
    q, pool = normal((rows, heads, latent + rope), dtype, 101), normal((3000, 1, latent + rope), dtype, 102)
    pool[17] *= 8
    ids = np.random.default_rng(103).integers(0, 3000, (rows, top))
    ids[0] = -1
    ids[1, :top - 1] = -1
    ids[2, 1:] = -1
    ids[3, top // 2] = 17
    ids[4, ::2] = 3000
    ids = ints(ids)
    out, lse = L.attend_slots(q, pool, None, ids, 0.06, latent=latent)
    check(out, lse, want_slots(q, pool, ids, 0.06, latent, dtype))
    assert not out[0].any() and torch.isinf(lse[0]).all()
    again = L.attend_slots(q, pool, None, ids, 0.06, latent=latent)
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])


def test_slots_rising_scores_rescale():
    """Scores that rise by hundreds from tile to tile: the running maximum moves far at every step."""
    base = normal((1, 1, 576), "bf16", 5)
    pool = (base * torch.linspace(0.0, 4.0, 640, device=DEV)[:, None, None].to(torch.bfloat16)).contiguous()
    pool[:, :, :512] += normal((640, 1, 512), "bf16", 6, 0.2)
    q = base.expand(2, 70, 576).contiguous()
    ids = torch.arange(640, device=DEV, dtype=torch.int32).repeat(2, 1)
    ids[1] = ids[1].flip(0)
    check(*L.attend_slots(q, pool, None, ids, 0.5), want_slots(q, pool, ids, 0.5, 512, "bf16"))


def test_slots_masks_maps_and_poison():
    """Rows without a token, one token, ids and slots out of range, a slot named twice, a slot map; the rows that
    nobody names hold NaN and infinities."""
    rows, top, dtype = 8, 190, "bf16"
    q, pool = normal((rows, 40, 576), dtype, 7), normal((500, 1, 576), dtype, 8)
    req = torch.randperm(400, generator=torch.Generator().manual_seed(9)).int().to(DEV)
    req[3], req[5] = 500, -7                     # a slot past the pool, and none
    pool[400:450] = float("nan")
    pool[450:] = float("inf")
    rng = np.random.default_rng(10)
    ids = rng.integers(0, 400, (rows, top))
    ids[0] = -1
    ids[1] = -1
    ids[1, 100] = 17
    ids[2, :] = 12                               # one slot 190 times
    ids[3, 5:] = -1
    ids[4, :128] = -1                            # two tiles without a token first
    ids[5, 7], ids[5, 8], ids[5, 9] = 400, 2 ** 31 - 1, -2 ** 31
    ids[6, ::2] = 3
    ids[7, ::3] = 5
    ids = ints(ids)
    out, lse = L.attend_slots(q, pool, req, ids, 0.07)
    check(out, lse, want_slots(q, pool, ids, 0.07, 512, dtype, req))
    assert not out[0].any() and torch.isinf(lse[0]).all()


def test_slots_strides_and_given_outputs():
    dtype = "bf16"
    q = normal((5, 2, 12, 640), dtype, 11)[:, 1, :, 32:608]
    pool = normal((300, 3, 576), dtype, 12)[:, 1:2]
    wide = ints(np.random.default_rng(13).integers(0, 300, (5, 200)))
    ids = wide[:, 7:172]
    out = torch.full((7, 12, 512), 3.0, dtype=torch.bfloat16, device=DEV)
    lse = torch.full((7, 12), 3.0, device=DEV)
    got = L.attend_slots(q, pool, None, ids, 0.06, out=out[1:6], lse=lse[1:6])
    assert got[0].data_ptr() == out[1:6].data_ptr()
    check(out[1:6], lse[1:6], want_slots(q, pool, ids, 0.06, 512, dtype))
    assert (out[[0, 6]] == 3).all() and (lse[[0, 6]] == 3).all()
    one = q[:1].expand(5, 12, 576)               # a query shared by the rows
    check(*L.attend_slots(one, pool, None, ids, 0.06), want_slots(one, pool, ids, 0.06, 512, dtype))


def test_slots_empty_calls():
    pool = normal((64, 1, 576), "bf16", 14)
    out, lse = L.attend_slots(normal((0, 4, 576), "bf16", 1), pool, None, ints(np.zeros((0, 9))), 0.1)
    assert out.shape == (0, 4, 512) and lse.shape == (0, 4)
    for ids, p in ((ints(np.zeros((3, 0))), pool), (ints(np.zeros((3, 70))), pool[:0])):
        out, lse = L.attend_slots(normal((3, 4, 576), "bf16", 1), p, None, ids, 0.1)
        assert not out.any() and torch.isinf(lse).all() and (lse < 0).all()


def test_slots_of_a_large_pool():
    """Slots whose element offset passes 2^31 and whose byte offset passes 2^32."""
    slots = 4_200_000
    pool = torch.empty((slots, 1, 576), dtype=torch.bfloat16, device=DEV)
    at = torch.tensor([0, 1, 3_728_270, 3_728_271, 4_000_001, slots - 1], device=DEV)
    pool[at] = normal((6, 1, 576), "bf16", 15)
    q = normal((2, 9, 576), "bf16", 16)
    ids = at.int().repeat(2, 30)
    check(*L.attend_slots(q, pool, None, ids, 0.05), want_slots(q, pool, ids, 0.05, 512, "bf16"))


@pytest.mark.parametrize("rows,heads,width,dtype", [(1, 64, 40, "bf16"), (9, 24, 5, "fp16"), (6, 128, 3, "bf16"),
                                                    (70, 7, 9, "bf16"), (2, 16, 130, "fp16")])
def test_pages(rows, heads, width, dtype):
    """Lengths of nothing, one, page ends and past the table; pages of the pool in any order; what lies behind the
    last token is NaN."""
    n = rows * width
    pool = torch.full(((n + 3) * 64, 1, 576), float("nan"), dtype=TYPES[dtype], device=DEV)
    table = torch.randperm(n, generator=torch.Generator().manual_seed(17)).int().view(rows, width).to(DEV)
    lens = np.random.default_rng(18).integers(0, width * 64 + 1, rows)
    edge = [width * 64, 0, 1, 63, 64, 65, width * 64 - 1, width * 64 + 100, -5]
    lens[:min(rows, 9)] = edge[:min(rows, 9)]
    fill = normal((n * 64, 576), dtype, 19)
    pos = torch.arange(width * 64, device=DEV)
    for r in range(rows):
        at = (table[r].long()[pos // 64] * 64 + pos % 64)[:max(0, lens[r])]
        pool[at, 0] = fill[at]
    q = normal((rows, heads, 576), dtype, 20)
    out, lse = L.attend_pages(q, pool, table, ints(lens), 0.07)
    ids = (table.long()[:, pos // 64] * 64 + pos % 64)
    ids = torch.where(pos < ints(lens)[:, None], ids, -1).int()
    check(out, lse, want_slots(q, pool, ids, 0.07, 512, dtype))


def test_pages_outside_the_pool():
    pool, q = normal((640, 1, 576), "bf16", 21), normal((3, 10, 576), "bf16", 22)
    table = ints([[0, 10, 3, -1], [2 ** 31 - 1, -2 ** 31, 9, 9], [-1, -1, -1, -1]])
    lens = ints([256, 200, 256])
    pos = torch.arange(256, device=DEV)
    ids = table.long()[:, pos // 64] * 64 + pos % 64
    ids = torch.where((pos < lens[:, None]) & (ids >= 0) & (ids < 640), ids, -1).int()
    check(*L.attend_pages(q, pool, table, lens, 0.07), want_slots(q, pool, ids, 0.07, 512, "bf16"))


def test_row_views_of_one_table():
    """The rows of an extend share one request's table (stride 0) and see a token more each."""
    pool, q = normal((640, 1, 576), "bf16", 23), normal((6, 16, 576), "bf16", 24)
    table = ints([[4, 2, 9, 0]]).expand(6, 4)
    lens = ints([120, 121, 122, 123, 124, 129])
    pos = torch.arange(256, device=DEV)
    ids = torch.where(pos < lens[:, None], table.long()[:, pos // 64] * 64 + pos % 64, -1).int()
    check(*L.attend_pages(q, pool, table, lens, 0.07), want_slots(q, pool, ids, 0.07, 512, "bf16"))


# -- expanded form ------------------------------------------------------------------
def want_prompt(q, k, rope, v, qo, ko, scale, dtype):
    tokens, heads, _ = q.shape
    out, lse = np.zeros((tokens, heads, 128)), np.zeros((tokens, heads))
    to, tl = np.zeros_like(out), np.zeros_like(lse)
    qs, ks, vs = f64(q), f64(k), f64(v)
    if rope is not None:
        ks = np.concatenate([ks, np.repeat(f64(rope)[:, None], heads, 1)], 2)
    for r in range(len(qo) - 1):
        a, b, c, d = qo[r], qo[r + 1], ko[r], ko[r + 1]
        live = np.tril(np.ones((b - a, d - c), bool), (d - c) - (b - a))
        for h in range(heads):
            got = A.softmax_rows(qs[a:b, h], ks[c:d, h], vs[c:d, h], scale, live, **rounding(dtype))
            for x, y in zip((out, lse, to, tl), got):
                x[a:b, h] = y
    return out, lse, to, tl


@pytest.mark.parametrize("counts,extra,heads,rope,dtype", [
    ([1], [0], 1, 64, "bf16"), ([1], [300], 3, 64, "fp16"), ([127, 1, 129], [0, 0, 0], 2, 64, "bf16"),
    ([128], [0], 4, 0, "bf16"), ([256, 255], [1, 127], 1, 64, "bf16"), ([300, 0, 40], [100, 5, 0], 3, 64, "fp16"),
    ([600], [0], 2, 0, "fp16"), ([5, 7, 300, 1, 1, 64], [1000, 3, 0, 640, 0, 128], 2, 64, "bf16"),
    ([257], [-100], 2, 64, "bf16"), ([40, 30], [-40, -10], 1, 64, "bf16"), ([1025], [511], 1, 64, "bf16"),
])
def test_prompt(counts, extra, heads, rope, dtype):
    """Ragged prompts; more keys than queries, and fewer: the first queries then see nothing."""
    qo = np.concatenate([[0], np.cumsum(counts)]).astype(int)
    ko = np.concatenate([[0], np.cumsum(np.add(counts, extra))]).astype(int)
    q = normal((qo[-1], heads, 128 + rope), dtype, 30)
    kv = normal((ko[-1], heads, 256), dtype, 31)
    kr = normal((ko[-1], 576), dtype, 32)[:, 512:] if rope else None
    k, v = kv[..., :128], kv[..., 128:]
    out, lse = L.attend_prompt(q, k, kr, v, ints(qo), 0.08, kv_offsets=ints(ko))
    check(out, lse, want_prompt(q, k, kr, v, qo, ko, 0.08, dtype))


@pytest.mark.parametrize("scale", [0.0, -0.05, 0.9])
def test_prompt_scales(scale):
    """Equal weights, the reversed order, and rows where the maximum keeps moving far."""
    q, kv, kr = normal((300, 2, 192), "bf16", 41), normal((420, 2, 256), "bf16", 42), normal((420, 64), "bf16", 43)
    kv[:, 0, :128] *= torch.linspace(0.0, 3.0, 420, device=DEV)[:, None].to(torch.bfloat16)
    out, lse = L.attend_prompt(q, kv[..., :128], kr, kv[..., 128:], ints([0, 300]), scale, kv_offsets=ints([0, 420]))
    check(out, lse, want_prompt(q, kv[..., :128], kr, kv[..., 128:], [0, 300], [0, 420], scale, "bf16"))


def test_prompt_poison_and_uncovered_rows():
    """NaN and infinities in the keys of nobody; rows of q outside every request stay as they were."""
    q, kv, kr = normal((400, 2, 192), "bf16", 33), normal((900, 2, 256), "bf16", 34), normal((900, 64), "bf16", 35)
    qo, ko = [20, 150, 330], [40, 300, 610]
    kv[:40], kr[:40] = float("nan"), float("nan")
    kv[610:], kr[610:] = float("inf"), float("nan")
    out = torch.full((400, 2, 128), 5.0, dtype=torch.bfloat16, device=DEV)
    lse = torch.full((400, 2), 5.0, device=DEV)
    L.attend_prompt(q, kv[..., :128], kr, kv[..., 128:], ints(qo), 0.08, kv_offsets=ints(ko), out=out, lse=lse)
    o, l, to, tl = want_prompt(q, kv[..., :128], kr, kv[..., 128:], qo, ko, 0.08, "bf16")
    check(out[20:330], lse[20:330], (o[20:330], l[20:330], to[20:330], tl[20:330]))
    keep = torch.cat([torch.arange(20), torch.arange(330, 400)])
    assert (out[keep] == 5).all() and (lse[keep] == 5).all()


def test_prompt_shared_heads_and_strides():
    """Keys and values broadcast over the heads (stride 0), and heads outside the tokens, equal to their copies."""
    q, kv, kr = normal((300, 3, 192), "bf16", 44), normal((300, 1, 256), "bf16", 45), normal((300, 64), "bf16", 46)
    k, v = kv[..., :128].expand(300, 3, 128), kv[..., 128:].expand(300, 3, 128)
    off = ints([0, 300])
    a = L.attend_prompt(q, k, kr, v, off, 0.08)
    check(*a, want_prompt(q, k, kr, v, [0, 300], [0, 300], 0.08, "bf16"))
    swapped = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v)]
    b = L.attend_prompt(swapped[0], swapped[1], kr, swapped[2], off, 0.08)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_prompt_neighbours_do_not_leak():
    """A request's result does not depend on what its neighbours in the same tiles hold."""
    q, kv, kr = normal((300, 2, 192), "fp16", 36), normal((300, 2, 256), "fp16", 37), normal((300, 64), "fp16", 38)
    qo = ints([0, 90, 190, 300])
    a = L.attend_prompt(q, kv[..., :128], kr, kv[..., 128:], qo, 0.08)
    kv[:90], kr[190:] = float("nan"), float("inf")
    b = L.attend_prompt(q, kv[..., :128], kr, kv[..., 128:], qo, 0.08)
    assert torch.equal(a[0][90:190], b[0][90:190]) and torch.equal(a[1][90:190], b[1][90:190])


def test_prompt_offsets_outside_the_tokens():
    q, kv = normal((50, 1, 128), "bf16", 39), normal((60, 1, 256), "bf16", 40)
    a = L.attend_prompt(q, kv[..., :128], None, kv[..., 128:], ints([0, 50]), 0.1, kv_offsets=ints([0, 60]))
    b = L.attend_prompt(q, kv[..., :128], None, kv[..., 128:], ints([-9, 1 << 30]), 0.1, kv_offsets=ints([-1, 1 << 30]))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    out = torch.full((50, 1, 128), 2.0, dtype=torch.bfloat16, device=DEV)
    L.attend_prompt(q, kv[..., :128], None, kv[..., 128:], ints([0]), 0.1, out=out)      # no requests
    assert (out == 2).all()


# -- the 8-bit cache ------------------------------------------------------------------
def new_cache(pages, heads, seed=None):
    codes = [torch.full((pages, heads, 64, 128), 0x7F, dtype=torch.uint8, device=DEV) for _ in range(2)]   # NaN
    if seed is not None:
        for i, c in enumerate(codes):
            g = torch.Generator(device=DEV).manual_seed(seed + i)
            c.copy_((torch.randn(c.shape, generator=g, device=DEV) * 60).to(torch.float8_e4m3fn).view(torch.uint8))
    g = torch.Generator(device=DEV).manual_seed(99)
    scales = [torch.exp2(torch.randint(-9, -5, (pages, heads), generator=g, device=DEV).float()) for _ in range(2)]
    return [codes[0].view(torch.float8_e4m3fn), scales[0], codes[1].view(torch.float8_e4m3fn), scales[1]]


def bytes_of(c):
    return [t.view(torch.uint8).cpu().numpy().copy() if t.dtype != torch.float32 else t.cpu().numpy().copy() for t in c]


def want_store(c, k, v, table, prefix, offsets):
    b = bytes_of(c)
    for i, x in ((0, k), (2, v)):
        s = b[i + 1].astype(np.float64)
        A.kv8_store(b[i], s, f64(x), table, prefix, offsets)
        b[i + 1] = s.astype(np.float32)
    return b


@pytest.mark.parametrize("counts,prefix,heads,dtype", [
    ([1], [0], 1, "bf16"), ([1], [63], 2, "fp16"), ([1], [64], 2, "bf16"), ([64], [0], 1, "bf16"), ([65], [63], 3, "bf16"),
    ([200, 1, 0, 130], [10, 127, 5, 64], 2, "fp16"), ([1] * 70, list(range(0, 210, 3)), 1, "bf16"),
    ([3, 0, 0, 500, 2], [1, 1, 1, 1, 190], 2, "bf16"), ([0] * 40 + [5] + [0] * 30, [9] * 71, 1, "bf16"),
])
def test_store(counts, prefix, heads, dtype):
    offsets = np.concatenate([[0], np.cumsum(counts)]).astype(int)
    width = max(p + c for p, c in zip(prefix, counts)) // 64 + 1
    n = len(counts) * width
    c = new_cache(n + 2, heads, 50)
    table = np.random.default_rng(51).permutation(n + 2)[:n].reshape(len(counts), width).astype(np.int32)
    k, v = normal((offsets[-1], heads, 128), dtype, 52, 2.0), normal((offsets[-1], heads, 128), dtype, 53, 0.01)
    want = want_store(c, k, v, table, prefix, offsets)
    for _ in range(2):                           # storing the same tokens again changes nothing
        K.store(*c, k, v, ints(table), ints(prefix), ints(offsets))
        for got, w in zip(bytes_of(c), want):
            assert np.array_equal(got, w)


def test_store_special_values():
    """Zeros, magnitudes at the scale's borders and past its ends, infinities, NaN, f16's smallest."""
    x = torch.zeros((64 * 9, 1, 128), device=DEV)
    tops = [0.0, 448.0, 450.0, 1.75 * 2.0 ** -8, 1.765625 * 2.0 ** -8, 2.0 ** -60, 1e30, float("inf"), 1.0]
    for i, t in enumerate(tops):
        x[64 * i:64 * i + 64] = torch.linspace(-1, 1, 128, device=DEV) * (t if np.isfinite(t) else 1.0)
        x[64 * i + 5, 0, 127] = t
    x[64 * 8 + 7, 0, 3] = float("nan")
    x = x.to(torch.bfloat16)
    c = new_cache(9, 1)
    table = np.arange(9, dtype=np.int32)[None]
    K.store(*c, x, x, ints(table), ints([0]), ints([0, 64 * 9]))
    finite = x.clone()
    finite[64 * 7:64 * 8][torch.isinf(x[64 * 7:64 * 8])] = 3e38
    want = want_store(new_cache(9, 1), finite, finite, table, [0], [0, 64 * 9])
    for got, w in zip(bytes_of(c), want):
        assert np.array_equal(got, w)


def test_store_token_by_token_and_dropped_tokens():
    """A page filled token by token with rising and falling magnitudes; tokens past the table and in pages outside
    the cache are dropped, and what lies behind the last token stays."""
    c, ref = new_cache(3, 2, 54), new_cache(3, 2, 54)
    want = bytes_of(ref)
    ws = [w.astype(np.float64) for w in (want[1], want[3])]
    table = np.array([[1, 7], [2, -1]], np.int32)
    for t in range(70):
        k, v = normal((2, 2, 128), "bf16", 100 + t, 2.0 ** ((t * 5) % 13 - 6)), normal((2, 2, 128), "bf16", 300 + t)
        K.store(*c, k, v, ints(table), ints([t, t + 50]), ints([0, 1, 2]))
        A.kv8_store(want[0], ws[0], f64(k), table, [t, t + 50], [0, 1, 2])
        A.kv8_store(want[2], ws[1], f64(v), table, [t, t + 50], [0, 1, 2])
    got = bytes_of(c)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[2], want[2])
    assert np.array_equal(got[1], ws[0].astype(np.float32)) and np.array_equal(got[3], ws[1].astype(np.float32))


def test_store_strides_and_foreign_offsets():
    """Views of one projection's output; offsets that begin past 0 and end past the tokens."""
    kv = normal((90, 3, 256), "fp16", 55)
    k, v = kv[..., :128], kv[..., 128:]
    table = np.array([[0, 1], [2, 3]], np.int32)
    c = new_cache(4, 3, 56)
    want = want_store(c, k, v, table, [3, 60], [10, 70, 90])
    K.store(*c, k, v, ints(table), ints([3, 60]), ints([10, 70, 95]))
    for got, w in zip(bytes_of(c), want):
        assert np.array_equal(got, w)
    before = bytes_of(c)
    K.store(*c, k, v, ints(table), ints([3, 60]), ints([40, 40, 40]))
    assert all(np.array_equal(x, y) for x, y in zip(bytes_of(c), before))


def want_attend(q, c, table, lens, scale, dtype):
    codes = [t.view(torch.uint8).cpu().numpy() for t in (c[0], c[2])]
    sc = [f64(t) for t in (c[1], c[3])]
    qs = f64(q)
    rows, heads, _ = q.shape
    kvh = c[0].shape[1]
    # weights and codes meet in f16: 2^-11 per weight, 2^-24 of the largest weight where it underflows; the query is
    # held in f16 under a power of two that puts its largest value in [1, 2)
    r = dict(rounding(dtype), up=2.0 ** -11, tiny=2.0 ** -24, dq=2.0 ** -24)
    res = []
    for i in range(rows):
        n = min(max(int(lens[i]), 0), table.shape[1] * 64)
        pos = np.arange(n)
        page = table[i][pos // 64] if n else np.zeros(0, int)
        ok = (page >= 0) & (page < c[0].shape[0])
        pos, page = pos[ok], page[ok]
        parts = []
        for g in range(kvh):
            k, v = (A.e4m3_decode(codes[j][page, g, pos % 64]) * sc[j][page, g][:, None] for j in (0, 1))
            hs = slice(g * heads // kvh, (g + 1) * heads // kvh)
            parts.append(A.softmax_rows(qs[i, hs], k, v, scale, **r))
        res.append([np.concatenate(x) for x in zip(*parts)])
    return [np.stack(x) for x in zip(*res)]


def fill(c, table, lens, seed):
    """Random codes up to each row's length (the rest stays NaN)."""
    for i in (0, 2):
        codes = c[i].view(torch.uint8)
        g = torch.Generator(device=DEV).manual_seed(seed + i)
        for r in range(table.shape[0]):
            for p in range(table.shape[1]):
                n = min(64, max(0, int(lens[r]) - 64 * p))
                if n and 0 <= table[r, p] < codes.shape[0]:
                    x = torch.randn((codes.shape[1], n, 128), generator=g, device=DEV) * 90
                    codes[int(table[r, p]), :, :n] = x.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)


@pytest.mark.parametrize("rows,heads,kv_heads,width,dtype", [
    (1, 1, 1, 1, "bf16"), (9, 4, 4, 3, "fp16"), (9, 32, 4, 3, "bf16"), (12, 17, 1, 2, "bf16"), (1, 32, 4, 40, "bf16"),
    (3, 40, 2, 20, "fp16"), (60, 8, 8, 5, "bf16"), (10, 21, 7, 4, "bf16"), (2, 160, 8, 9, "fp16"),
])
def test_attend(rows, heads, kv_heads, width, dtype):
    lens = np.random.default_rng(60).integers(0, width * 64 + 1, rows)
    edge = [width * 64, 0, 1, 63, 64, 65, width * 64 - 1, width * 64 + 9, -3]
    lens[:min(rows, 9)] = edge[:min(rows, 9)]
    c = new_cache(rows * width + 1, kv_heads)
    table = np.random.default_rng(61).permutation(rows * width + 1)[:rows * width].reshape(rows, width).astype(np.int32)
    fill(c, table, np.minimum(lens, width * 64), 62)
    q = normal((rows, heads, 128), dtype, 63)
    out, lse = K.attend(q, *c, ints(table), ints(lens), 0.09)
    check(out, lse, want_attend(q, c, table, lens, 0.09, dtype))


def test_attend_far_scales_pages_and_strides():
    """Scales that differ by 2^30 between pages, pages outside the cache, queries of very different sizes as a
    strided view."""
    c = new_cache(6, 2)
    table = np.array([[0, 1, 2], [3, 9, 4], [-1, -1, -2 ** 31], [5, 5, 0]], np.int32)
    lens = np.array([180, 190, 150, 192])
    fill(c, table, np.array([192] * 4), 64)
    c[3][0], c[3][1], c[3][2] = 2.0 ** -25, 2.0 ** 5, 2.0 ** -8
    c[1][4] = 2.0 ** -20
    q = normal((4, 3, 8, 128), "bf16", 65)[:, 1]
    q[1] *= 2.0 ** -30
    q[3, 4] *= 40
    out, lse = K.attend(q, *c, ints(table), ints(lens), 0.09)
    check(out, lse, want_attend(q, c, table, lens, 0.09, "bf16"))
    assert not out[2].any() and torch.isinf(lse[2]).all()


# -- many small weights beside a few large ones ---------------------------------------
# Every 64th token scores 17.5, the others 0: weights e^-17.5 = 2^-25.2 of the largest, below what f16 holds (half
# its smallest step is 2^-25) unless they are lifted into its range.  The large ones' values are 0, so the output
# consists of the small ones alone.  The floor of a weight, relative to the largest: 2^-25 under the lift, 2^7 in the
# latent and prompt kernels, 2^15 in the 8-bit ones; their bf16 weights have none.
def steep(n, dim):
    k = torch.zeros((n, dim), device=DEV)
    k[::64, 0] = 4.0
    v = torch.zeros((n, 128), device=DEV)
    v[:, 3] = 896.0
    v[::64, 3] = 0.0
    q = torch.zeros(dim, device=DEV)
    q[0] = 4.0
    return q, k, v, 17.5 / 16


def steep_want(q, k, v, scale, dtype, tiny, up):
    r = dict(u=A.U[dtype], up=up, tiny=tiny, smallest=A.SMALLEST[dtype])
    return A.softmax_rows(f64(q)[None], f64(k), f64(v), scale, **r)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_small_weights_latent(dtype):
    q, k, v, scale = steep(2048, 192)
    k[:, 1:128] = v[:, 1:128]                      # the pool's row is key and value; the query sees its first element
    floor = 2.0 ** -32 if dtype == "fp16" else 0.0
    want = [np.broadcast_to(x, (3, 2) + x.shape[1:]) for x in steep_want(q, k, k[:, :128], scale, dtype, floor, A.U[dtype])]
    t = TYPES[dtype]
    qs, pool = q.to(t).expand(3, 2, 192).contiguous(), k.to(t)[:, None]
    check(*L.attend_slots(qs, pool, None, ints(np.arange(2048)[None].repeat(3, 0)), scale, latent=128), want, "slots")
    check(*L.attend_pages(qs, pool, ints(np.arange(32)[None].repeat(3, 0)), ints([2048] * 3), scale, latent=128), want, "pages")
    # the third query of three sees every key
    out, lse = L.attend_prompt(q[:128].to(t).expand(3, 2, 128), k[:, :128].to(t)[:, None].expand(2048, 2, 128), None,
                               v.to(t)[:, None].expand(2048, 2, 128), ints([0, 3]), scale, kv_offsets=ints([0, 2048]))
    want = [np.broadcast_to(x, (2,) + x.shape[1:]) for x in steep_want(q[:128], k[:, :128], v, scale, dtype, floor, A.U[dtype])]
    check(out[2], lse[2], want, "prompt")


@pytest.mark.parametrize("dtype,heads", [("bf16", 4), ("fp16", 40)])
def test_small_weights_8bit(dtype, heads):
    q, k, v, scale = steep(2048, 128)
    c = new_cache(32, 1)
    t = TYPES[dtype]
    # exact: 4 and 896 are codes under their pages' scales
    K.store(*c, k.to(t)[:, None], v.to(t)[:, None], ints(np.arange(32)[None]), ints([0]), ints([0, 2048]))
    out, lse = K.attend(q.to(t).expand(1, heads, 128).contiguous(), *c, ints(np.arange(32)[None]), ints([2048]), scale)
    want = [np.broadcast_to(x, (1, heads) + x.shape[1:])
            for x in steep_want(q, k, v, scale, dtype, 2.0 ** -40, 2.0 ** -11)]
    check(out, lse, want)


# -- streams, graphs, the pieces together ---------------------------------------------
def calls():
    """Small calls of every operator: name -> (inputs, function of the inputs)."""
    pool, ids = normal((900, 1, 576), "bf16", 70), ints(np.random.default_rng(71).integers(0, 900, (9, 333)))
    q, table = normal((9, 20, 576), "bf16", 72), ints(np.arange(9 * 1).reshape(9, 1))
    lens = ints([64, 1, 0, 63, 40, 64, 64, 2, 33])
    pq, kv, kr = normal((333, 2, 192), "bf16", 73), normal((333, 2, 256), "bf16", 74), normal((333, 64), "bf16", 75)
    off = ints([0, 100, 333])
    c = new_cache(30, 2, 76)
    t8, q8 = ints(np.arange(30).reshape(3, 10)), normal((3, 8, 128), "bf16", 77)
    x = normal((30, 2, 128), "bf16", 78)
    return {
        "slots": ([q, pool], lambda q, pool: L.attend_slots(q, pool, None, ids, 0.07)),
        "pages": ([q, pool], lambda q, pool: L.attend_pages(q, pool, table, lens, 0.07)),
        "prompt": ([pq, kv], lambda q, kv: L.attend_prompt(q, kv[..., :128], kr, kv[..., 128:], off, 0.08)),
        "kv8": ([q8, x], lambda q, x: (K.store(*c, x, x, t8, ints_70, off_70), K.attend(q, *c, t8, lens_70, 0.09))[1]),
    }


ints_70 = off_70 = lens_70 = None


@pytest.fixture(scope="module", autouse=True)
def shared_ints(request):
    global ints_70, off_70, lens_70
    if torch.cuda.is_available():
        ints_70, off_70, lens_70 = ints([60, 0, 5]), ints([0, 10, 20, 30]), ints([70, 10, 15])


@pytest.mark.parametrize("name", ["slots", "pages", "prompt", "kv8"])
def test_graphs_and_streams(name):
    """The same bits eagerly, on a side stream, and from two graphs captured side by side and replayed in turn on
    changed inputs."""
    args, f = calls()[name]
    first = [t.clone() for t in args]
    other = [t.flip(0).contiguous() for t in args]
    want = {}
    for key, src in (("first", first), ("other", other)):
        want[key] = [t.clone() for t in f(*src)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = f(*first)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(got, want["first"]))
    graphs = []
    for _ in range(2):
        live = [t.clone() for t in first]
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            res = f(*live)
        graphs.append((live, g, res))
    for key, src in (("other", other), ("first", first), ("other", other)):
        for live, g, res in graphs:
            for a, b in zip(live, src):
                a.copy_(b)
            g.replay()
        for live, g, res in graphs:
            assert all(torch.equal(x, y) for x, y in zip(res, want[key])), key


def test_two_calls_at_once():
    """Two large calls on two streams at the same time give what each gives alone."""
    pool = normal((40000, 1, 576), "bf16", 80)
    rng = np.random.default_rng(81)
    ids = [ints(rng.integers(0, 40000, (150, 1000))) for _ in range(2)]
    q = [normal((150, 32, 576), "bf16", 82 + i) for i in range(2)]
    alone = [L.attend_slots(q[i], pool, None, ids[i], 0.07) for i in range(2)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [None, None]
    for _ in range(3):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i] = L.attend_slots(q[i], pool, None, ids[i], 0.07)
    torch.cuda.synchronize()
    for a, b in zip(alone, got):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_prompt_then_selected_decode():
    """A request served through the operators: the prompt in the expanded form and its latent rows into the paged
    pool, then a decode row in the absorbed form over all pages and over the slots of all tokens.  With the
    projections multiplied out in 32 bits all three are one attention."""
    n, heads, g = 150, 4, torch.Generator(device=DEV).manual_seed(90)
    latent = normal((n, 576), "bf16", 91)
    wk = torch.randn((heads, 128, 512), generator=g, device=DEV) * 512 ** -0.5
    wv = torch.randn((heads, 128, 512), generator=g, device=DEV) * 512 ** -0.5
    q = normal((n, heads, 192), "bf16", 92)
    k = torch.einsum("tl,hdl->thd", latent[:, :512].float(), wk).to(torch.bfloat16)
    v = torch.einsum("tl,hdl->thd", latent[:, :512].float(), wv).to(torch.bfloat16)
    scale = 192 ** -0.5
    prompt, plse = L.attend_prompt(q, k, latent[:, 512:], v, ints([0, n]), scale)
    pool = torch.full((64 * 5, 1, 576), float("nan"), dtype=torch.bfloat16, device=DEV)
    table = ints([[3, 0, 4]])
    pos = torch.arange(n, device=DEV)
    slots = table[0].long()[pos // 64] * 64 + pos % 64
    pool[slots, 0] = latent
    last = q[-1:]
    absorbed = torch.cat([torch.einsum("rhd,hdl->rhl", last[..., :128].float(), wk).to(torch.bfloat16),
                          last[..., 128:]], -1)
    a, alse = L.attend_pages(absorbed, pool, table, ints([n]), scale)
    b, blse = L.attend_slots(absorbed, pool, None, torch.cat([slots, slots.new_full((50,), -1)]).int()[None], scale)
    out = torch.einsum("rhl,hdl->rhd", a.float(), wv)
    # the expanded form rounds k and v to bf16, the absorbed one the query and the result: 2^-8 each of a score
    # whose terms sum to |q| |k| scale, and of the values
    mag = (q[-1].float().abs()[:, None] * torch.cat([k.float().abs().transpose(0, 1),
           latent[:, 512:].float().abs().expand(heads, n, 64)], 2)).sum(2).max().item() * scale
    bound = (4 * 2.0 ** -8 * mag + 4 * 2.0 ** -8) * v.float().abs().amax().item()
    assert (out - prompt[-1:].float()).abs().max().item() <= bound
    assert (alse - plse[-1:]).abs().max().item() <= 2 * 2.0 ** -8 * mag
    assert (a.float() - b.float()).abs().max().item() <= 2.0 ** -6 * a.float().abs().max().item()
    assert (alse - blse).abs().max().item() <= 1e-4


def test_prompt_store_then_decode_steps():
    """A request's prompt into the 8-bit cache, then decode steps that store a token and attend."""
    c = new_cache(8, 2)
    table = np.array([[5, 2, 7]], np.int32)
    ref = bytes_of(c)
    ws = [ref[1].astype(np.float64), ref[3].astype(np.float64)]
    n = 0
    for step, count in enumerate([100, 1, 1, 27, 1, 1]):
        k, v = normal((count, 2, 128), "bf16", 200 + step, 1.0 + step), normal((count, 2, 128), "bf16", 220 + step)
        K.store(*c, k, v, ints(table), ints([n]), ints([0, count]))
        A.kv8_store(ref[0], ws[0], f64(k), table, [n], [0, count])
        A.kv8_store(ref[2], ws[1], f64(v), table, [n], [0, count])
        n += count
        q = normal((1, 8, 128), "bf16", 240 + step)
        out, lse = K.attend(q, *c, ints(table), ints([n]), 0.09)
        assert all(np.array_equal(x, y) for x, y in zip(bytes_of(c)[::2], ref[::2]))
        check(out, lse, want_attend(q, c, table, [n], 0.09, "bf16"))


def test_selection_step_attends():
    """SelectionStep with attention: the selected rows attended in place of gathered; equal to attend_slots over the
    step's own physical ids, in a graph too."""
    synth = importlib.import_module("10_20_b200.synth")
    pipeline = importlib.import_module("10_20_b200.pipeline")
    case = synth.make_query_case(3, 64, [4097, 9000, 700], P=256, take=12, window=64, topk=2048, seed=3, device=DEV,
                                 latent_dim=576)
    q = normal((3, 24, 576), "bf16", 93)
    step = pipeline.SelectionStep(case, gather=False, attention=(q, 0.07))
    step.run()
    torch.cuda.synchronize()
    want = L.attend_slots(q, case.latent, None, step.physical, 0.07)
    assert torch.equal(step.attended[0], want[0]) and torch.equal(step.attended[1], want[1])
    check(*step.attended, want_slots(q, case.latent, step.physical, 0.07, 512, "bf16"))
    step.capture()
    step.attended[0].zero_()
    q.copy_(normal((3, 24, 576), "bf16", 94))
    step.replay()
    want = L.attend_slots(q, case.latent, None, step.physical, 0.07)
    assert torch.equal(step.attended[0], want[0]) and torch.equal(step.attended[1], want[1])
    assert step.launches() == 4      # two of the selection, the attention of three rows and its join
