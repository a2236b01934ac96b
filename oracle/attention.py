"""The attention operators' definitions in 64 bits (numpy), with the bound that
rounding puts on a kernel's result.

``softmax_rows`` returns (out, lse, tol_out, tol_lse).  The bound, per element,
from the kernels' arithmetic (u: half a step of the output type, 2^-8 relative
for bf16, 2^-11 for f16; up: the same of the type the weights are rounded to):

  scores   dim products added in 32 bits: |ds_j| <= (dim + 8) 2^-24 scale sum_d |q_d k_jd|
           plus 2^-22 |s_j| for the scale and the base-2 change of variable; where a
           kernel holds the query in a type that underflows, dq max|q| per value of it
  weights  w_j = exp(s_j): relative error 2 max|ds| after the division by their
           sum, 2^-20 for exp2 and the running rescale, up for the rounding
           of the weights that enter the product, and an absolute floor `tiny`
           (relative to the largest weight) where that type underflows
  out      |dout_d| <= (2 max|ds| + 2^-20 + up + n 2^-24) sum_j p_j |v_jd|
                       + tiny sum_j |v_jd| + u |out_d| (+ the type's smallest step)
  lse      |dlse| <= max|ds| + 2^-20 + 2^-22 |lse|
"""
from __future__ import annotations

import numpy as np

U = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11}
SMALLEST = {"bf16": 2.0 ** -133, "fp16": 2.0 ** -24}


def softmax_rows(q, k, v, scale, live=None, u=0.0, up=0.0, tiny=0.0, dq=0.0, smallest=0.0):
    """q [m, d], k [n, d], v [n, e] in 64 bits; live [m, n] or [n] truth values."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    m, n = q.shape[0], k.shape[0]
    live = np.ones((m, n), bool) if live is None else np.broadcast_to(live, (m, n))
    s = q @ k.T * scale
    s = np.where(live, s, -np.inf)
    mag = np.abs(q) @ np.abs(k).T * abs(scale)
    ds = (q.shape[1] + 8) * 2.0 ** -24 * mag + 2.0 ** -22 * np.abs(np.where(live, s, 0.0))
    ds = ds + dq * np.abs(q).max(1, initial=0.0)[:, None] * np.abs(k).sum(1) * abs(scale)
    ds = np.where(live, ds, 0.0).max(1, initial=0.0)
    some = live.any(1)
    top = np.where(some, s.max(1, initial=-np.inf), 0.0)
    w = np.exp(s - top[:, None])
    total = w.sum(1)
    with np.errstate(divide="ignore"):
        lse = np.where(some, top + np.log(total), -np.inf)
    p = w / np.where(some, total, 1.0)[:, None]
    out = p @ v
    spread = p @ np.abs(v)
    used = live.astype(np.float64) @ np.abs(v)
    tol = ((2 * ds[:, None] + 2.0 ** -20 + up + n * 2.0 ** -24) * spread * (1 + 2.0 ** -6) + tiny * used
           + u * np.abs(out) * (1 + 2.0 ** -6) + smallest)
    return out, lse, tol, ds + 2.0 ** -20 + 2.0 ** -22 * np.where(some, np.abs(lse), 0.0)


def page_scale(most):
    """The smallest 2^e, -40 <= e <= 40, with 448 * 2^e >= most."""
    e = -40
    while e < 40 and 448.0 * 2.0 ** e < most:
        e += 1
    return 2.0 ** e


def _e4m3_values():
    v = np.zeros(128)
    for c in range(127):
        e, m = c >> 3, c & 7
        v[c] = m * 2.0 ** -9 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
    v[127] = np.nan
    return v


E4M3 = _e4m3_values()


def e4m3_decode(codes):
    c = np.asarray(codes, np.uint8)
    return np.where(c & 0x80, -1.0, 1.0) * E4M3[c & 0x7F]


def e4m3_encode(x):
    """Round to nearest, ties to the even code, saturating at 448; the sign of zero kept."""
    x = np.asarray(x, np.float64)
    a = np.minimum(np.abs(x), 448.0)
    hi = np.clip(np.searchsorted(E4M3[:127], a, side="left"), 0, 126)
    lo = np.maximum(hi - 1, 0)
    dl, dh = a - E4M3[lo], E4M3[hi] - a
    code = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi).astype(np.uint8)
    code = np.where(np.isnan(x), 0x7F, code)
    return (code | np.where(np.signbit(x), 0x80, 0)).astype(np.uint8)


def kv8_store(cache, scale, x, table, prefix, offsets):
    """In place: the tokens of x [tokens, heads, 128] into cache u8 [pages, heads,
    64, 128] and scale [pages, heads], page by page."""
    for r in range(len(prefix)):
        t0, t1 = int(offsets[r]), int(offsets[r + 1])
        p = int(prefix[r])
        for i in range(p // 64, (p + t1 - t0 - 1) // 64 + 1 if t1 > t0 else 0):
            if i >= table.shape[1] or not 0 <= table[r, i] < cache.shape[0]:
                continue
            page, lo, hi = int(table[r, i]), max(p, i * 64), min(p + t1 - t0, i * 64 + 64)
            new = np.asarray(x[t0 + lo - p:t0 + hi - p], np.float64)
            for h in range(cache.shape[1]):
                now = page_scale(np.nanmax(np.abs(new[:, h]), initial=0.0))
                old = float(scale[page, h])
                if lo > i * 64:
                    now = max(now, old)
                    if now != old:
                        e = cache[page, h, :lo - i * 64]
                        cache[page, h, :lo - i * 64] = e4m3_encode(e4m3_decode(e) * (old / now))
                scale[page, h] = now
                cache[page, h, lo - i * 64:hi - i * 64] = e4m3_encode(new[:, h] / now)
