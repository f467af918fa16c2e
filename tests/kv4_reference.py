"""Plain 64-bit implementations of the 4-bit KV cache, the attention over it and
token sampling, for the tests (numpy, on the host)."""
from __future__ import annotations

import numpy as np

D, GROUP, ROW = 128, 32, 80
LIMIT = np.float32(65408)


def quantize(x: np.ndarray) -> np.ndarray:
    """Rows [..., 128] to cache rows [..., 80] in the 32-bit arithmetic of the format."""
    x = np.asarray(x, dtype=np.float32)
    x = np.where(np.isnan(x), x, np.clip(x, -LIMIT, LIMIT)).reshape(*x.shape[:-1], 4, GROUP)
    lo, hi = x.min(-1), x.max(-1)  # NaN where the group holds one
    m = lo.astype(np.float16)
    mf = m.astype(np.float32)
    d = ((hi - mf) * np.float32(1 / 15)).astype(np.float16)
    df = d.astype(np.float32)
    inv = np.divide(np.float32(1), df, out=np.zeros_like(df), where=df > 0)
    c = np.rint((x - mf[..., None]) * inv[..., None])
    c = np.where(np.isnan(c), 0, np.clip(c, 0, 15)).astype(np.uint8)
    c = c.reshape(*c.shape[:-2], D)
    codes = c[..., 0::2] | (c[..., 1::2] << 4)
    dm = np.stack([d, m], -1).reshape(*d.shape[:-1], 8).view(np.uint8)
    return np.concatenate([codes, dm], -1)


def values(rows: np.ndarray) -> np.ndarray:
    """fp64 values of cache rows [..., 80]."""
    codes = rows[..., :64]
    c = np.stack([codes & 15, codes >> 4], -1).reshape(*rows.shape[:-1], 4, GROUP).astype(np.float64)
    dm = np.ascontiguousarray(rows[..., 64:]).view(np.float16).astype(np.float64)
    dm = dm.reshape(*rows.shape[:-1], 4, 2)
    return (dm[..., 1:] + dm[..., :1] * c).reshape(*rows.shape[:-1], D)


def attention(q, k_rows, v_rows, lens, counts):
    """out [B][T][heads][128] in 64 bits, NaN rows where t >= counts[b]; and per
    output row the bound of sum |q_i k_i| / sqrt(128) over its keys and the
    largest |v| it may meet.  k_rows, v_rows [B][kv heads][capacity][80]."""
    B, T, NH, _ = q.shape
    H = k_rows.shape[1]
    G = NH // H
    out = np.full(q.shape, np.nan)
    smax, vmax = np.zeros((B, T, NH, 1)), np.zeros((B, T, NH, 1))
    for b in range(B):
        for h in range(H):
            k, v = values(k_rows[b, h, :max(lens[b], 0)]), values(v_rows[b, h, :max(lens[b], 0)])
            for t in range(counts[b]):
                n = max(0, lens[b] - counts[b] + t + 1)
                for g in range(h * G, (h + 1) * G):
                    if n == 0:
                        out[b, t, g] = 0
                        continue
                    x = q[b, t, g].astype(np.float64)
                    s = k[:n] @ x / np.sqrt(D)
                    p = np.exp(s - s.max())
                    out[b, t, g] = p @ v[:n] / p.sum()
                    smax[b, t, g] = (np.abs(k[:n]) @ np.abs(x)).max() / np.sqrt(D)
                    vmax[b, t, g] = np.abs(v[:n]).max()
    return out, smax, vmax


def attention_tolerance(ref, smax, vmax, out_eps, rounded_operands, rounded_weights=False):
    """Largest allowed |got - ref|.

    A score is a sum of 128 products: in 32 bits its error is below 128 roundings of
    2^-23 (tensor cores truncate) of sum |q k| / sqrt(128); where K is rounded to fp16
    first, 2^-11 of the same more.  An error e of every score moves the output by at
    most 2 e max|v| (1 + small).  exp, the sums and the division add 2^-18 of max|v|;
    weights and V rounded to fp16 2^-11 of max|v| each.  `rounded_weights`: the weights p and
    then p d rounded to fp16, 2^-11 of p d c each, where d c is at most V's range, 2 max|v|.
    The output itself is rounded by at most half a step."""
    e = smax * (128 * 2.0 ** -23 + (2.0 ** -11 if rounded_operands else 0))
    rel = np.expm1(2 * e) + 2.0 ** -18 + (2 * 2.0 ** -11 if rounded_operands else 0)
    rel += 2 * 2 * 2.0 ** -11 if rounded_weights else 0
    return (out_eps / 2) * np.abs(ref) + (1 + out_eps) * rel * vmax + 2.0 ** -25


def sample(x, temperature, top_k, top_p, min_p, u):
    """(token, prob) of one row in 64 bits."""
    x = np.asarray(x, dtype=np.float64)
    ok = ~np.isnan(x)
    if not ok.any():
        return 0, 0.0
    top = x[ok].max()
    if top == -np.inf:
        return int(np.nonzero(x == -np.inf)[0][0]), 0.0
    if not temperature > 0:
        return int(np.nonzero(x == top)[0][0]), 1.0
    order = np.nonzero(ok)[0]
    order = order[np.argsort(-x[order], kind="stable")]
    if 0 < top_k < len(x):
        order = order[:top_k]
    y = x[order]
    if top == np.inf:
        w = (y == np.inf).astype(np.float64)
    else:
        with np.errstate(invalid="ignore"):
            w = np.where(y == -np.inf, 0.0, np.exp((y - top) * (1.0 / np.float64(np.float32(temperature)))))
    if top_p < 1:
        target = max(float(np.float32(top_p)), 0.0) * w.sum()
        n = max(1, int((np.cumsum(w) - w < target).sum()))
        order, w = order[:n], w[:n]
    floor = min(float(np.float32(min_p)), 1.0) if min_p > 0 else 0.0
    keep = (w >= floor) & (w > 0)
    order, w = order[keep], w[keep]
    by_index = np.argsort(order)
    order, w = order[by_index], w[by_index]
    u = 0.0 if not u > 0 else min(float(np.float32(u)), 1 - 2.0 ** -24)
    at = int(np.searchsorted(np.cumsum(w), u * w.sum(), side="right"))
    at = min(at, len(w) - 1)
    return int(order[at]), float(w[at] / w.sum())
