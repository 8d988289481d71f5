"""CPU restatement of the paged key-value cache: appending tokens (rotation, quantisation) and the attention of new tokens over
the pages.

TEST INFRASTRUCTURE ONLY: imported by tests; never by the product path.

The reference has no paged cache and no position rotation; what a token attends to is row n of its prefill kernel
(cuda/attn_fwd_i8.cuh:368-619): keys n - W' .. n - 1 and the sink, temperature D^-1/2 log2(min(W', n) + 4) temp_h, base-2
softmax. The rotation of FixedI8 codes is integer arithmetic and the scaled form is defined in f32 operations, so both are
restated exactly; the attention is computed in float64."""
import math

import numpy as np

TINY = np.float32(2.0 ** -100)


def rope_table(n, rotary, base=10000.0):
    a = np.arange(n, dtype=np.float64)[:, None] * base ** (-np.arange(0, rotary, 2, dtype=np.float64) / rotary)
    return np.rint(np.stack((np.cos(a), np.sin(a)), axis=-1) * 16384).astype(np.int16)


def _split(x, rotary, adjacent):
    return (x[..., 0:rotary:2], x[..., 1:rotary:2]) if adjacent else (x[..., :rotary // 2], x[..., rotary // 2:rotary])


def rotate(x, cs, rotary, adjacent):
    """x [T, H, D] int8 (integers) or float32, cs [T, rotary / 2, 2] int16."""
    if rotary == 0:
        return x.copy()
    out = x.copy()
    a, b = _split(x, rotary, adjacent)
    u, v = _split(out, rotary, adjacent)   # views
    if x.dtype == np.int8:
        c, s = (cs[:, None, :, i].astype(np.int64) for i in (0, 1))
        a, b = a.astype(np.int64), b.astype(np.int64)
        u[...] = np.clip((a * c - b * s + 8192) >> 14, -127, 127)
        v[...] = np.clip((a * s + b * c + 8192) >> 14, -127, 127)
    else:
        c, s = (cs[:, None, :, i].astype(np.float32) * np.float32(2.0 ** -14) for i in (0, 1))
        u[...] = a * c - b * s
        v[...] = a * s + b * c
    return out


def quantise(x):
    """float32 [.., D] -> codes int8, scales float32 [..]."""
    top = np.abs(x).max(axis=-1)
    live = top > TINY
    inv = np.where(live, np.float32(127) / np.where(live, top, np.float32(1)), np.float32(0)).astype(np.float32)
    codes = np.clip(np.rint(x * inv[..., None]), -127, 127).astype(np.int8)
    return codes, np.where(live, top * np.float32(1 / 127), np.float32(0)).astype(np.float32)


def attend(q, q_scale, k, k_scale, v, v_scale, sink_k, sink_v, temperature, window):
    """One new token over the `n` keys in front of it: q int8 [H, D], q_scale [H], k / v int8 [n, Hk, D], their scales [n, Hk].
    Returns out float64 [H, D], l [H], and for tolerances mean |v| under the weights [H, D] and the largest |score| [H]."""
    h, d = q.shape
    n, hk = k.shape[:2]
    lo = 0 if window == 0 else max(0, n - window)
    kv = slice(lo, n)
    temp = d ** -0.5 * math.log2(n - lo + 4) * np.asarray(temperature, dtype=np.float64) * np.asarray(q_scale, dtype=np.float64)
    kf = (k[kv].astype(np.float64) * np.asarray(k_scale, dtype=np.float64)[kv, :, None]).repeat(h // hk, axis=1)
    vf = (v[kv].astype(np.float64) * np.asarray(v_scale, dtype=np.float64)[kv, :, None]).repeat(h // hk, axis=1)
    x = np.einsum("hd,nhd->hn", q.astype(np.float64), kf) * temp[:, None]
    sink = (q.astype(np.float64) * sink_k).sum(-1) / 8 * temp
    m = np.maximum(sink, x.max(axis=1, initial=-np.inf))
    e, es = np.exp2(x - m[:, None]), np.exp2(sink - m)
    total = e.sum(1) + es
    out = (np.einsum("hn,nhd->hd", e, vf) + es[:, None] * sink_v / 8) / total[:, None]
    mean = (np.einsum("hn,nhd->hd", e, np.abs(vf)) + es[:, None] * np.abs(sink_v.astype(np.float64)) / 8) / total[:, None]
    top = np.maximum(np.abs(sink), np.abs(x).max(axis=1, initial=0))
    return out, np.log2(255 * total) + m, mean, top
