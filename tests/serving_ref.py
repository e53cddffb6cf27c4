"""Plain implementations in 64 bits of the serving operators (rotary layouts, the paged 4-bit KV cache, attention over it,
rules on logits), for the tests: loops and numpy, nothing of the library."""
import collections

import numpy as np

HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # of a rounding, relative to the value


def torch_type(name):
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def pairs(R, layout):
    i = np.arange(R // 2)
    return (i, i + R // 2) if layout == "half" else (2 * i, 2 * i + 1)


def rotate(x, pos, table, layout, inverse=False):
    """x [T, H, D] in 64 bits; also sum |product| per element, what roundings are relative to"""
    R = table.shape[1]
    ia, ib = pairs(R, layout)
    w = table[pos].astype(np.float64)
    c, s = w[:, None, 0::2], (-1.0 if inverse else 1.0) * w[:, None, 1::2]
    y, m = x.astype(np.float64).copy(), np.zeros(x.shape)
    a, b = x[..., ia].astype(np.float64), x[..., ib].astype(np.float64)
    y[..., ia], y[..., ib] = a * c - b * s, a * s + b * c
    m[..., ia], m[..., ib] = abs(a * c) + abs(b * s), abs(a * s) + abs(b * c)
    return y, m


def rms(x, w, eps):
    x = x.astype(np.float64)
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w.astype(np.float64)


def bf16(x):
    """f32 -> the nearest bf16, ties to even, as f32"""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    return ((u + 0x7FFF + ((u >> 16) & 1)) & 0xFFFF0000).astype(np.uint32).view(np.float32)


def quantise(x):
    """x [..., D] f32 -> codes [..., D/2] and scales [..., D/32] f16, by the definition in single precision"""
    x = np.asarray(x, np.float32)
    b = x.reshape(*x.shape[:-1], -1, 32)
    far = np.abs(b).max(-1, keepdims=True)
    mx = np.where((b == far).any(-1, keepdims=True), far, -far)
    d = bf16(np.clip(mx * np.float32(-0.125), -2720, 2720)).astype(np.float16)
    d32 = d.astype(np.float32)
    with np.errstate(divide="ignore", invalid="ignore"):
        c = np.where(d32 == 0, np.float32(8), np.clip(np.floor(b / d32 + np.float32(8.5)), 0, 15)).astype(np.uint8)
    return (c[..., :16] | (c[..., 16:] << 4)).reshape(*x.shape[:-1], -1), d[..., 0]


def values(codes, scales):
    b = codes.reshape(*codes.shape[:-1], codes.shape[-1] // 16, 16)
    c = np.concatenate([b & 15, b >> 4], -1).astype(np.float64) - 8
    return (c * scales.astype(np.float64)[..., None]).reshape(*codes.shape[:-1], 2 * codes.shape[-1])


def attention(q, k, v, first, window, scale):
    """q [n, D] at positions first.., k / v [len, D]: outputs [n, D] and, per element, sum_j p_j |v_j|, the largest
    |scale| * sum |q k| (what the roundings of the sums and of the scores are relative to) and sum_j |v_j|"""
    n, D = q.shape
    o, a, s1, av = np.zeros((n, D)), np.zeros((n, D)), np.zeros((n, 1)), np.zeros((n, D))
    for i in range(n):
        p = first + i
        lo = max(0, p - window + 1) if window else 0
        if p < 0 or p + 1 <= lo:
            continue
        kk, vv = k[lo:p + 1], v[lo:p + 1]
        s = kk @ q[i] * scale
        e = np.exp(s - s.max())
        w = e / e.sum()
        o[i], a[i], s1[i] = w @ vv, w @ np.abs(vv), (np.abs(kk) @ np.abs(q[i])).max() * abs(scale)
        av[i] = np.abs(vv).sum(0)
    return o, a, s1, av


def rules(x, hist=None, n_prompt=0, rep=None, freq=None, pres=None, bias=(), mask=None):
    """one row; also the sum of magnitudes that the roundings are relative to"""
    x = x.astype(np.float64).copy()
    m = np.abs(x)
    V = x.size
    if hist is not None:
        seen = {int(t) for t in hist if 0 <= t < V}
        out = [int(t) for t in hist[max(0, n_prompt):] if 0 <= t < V]
        for t in seen:
            if rep is not None:
                x[t] = x[t] / rep if x[t] > 0 else x[t] * rep
            m[t] = max(m[t], abs(x[t]))
        for t, n in collections.Counter(out).items():
            for term in ((freq or 0.0) * n, pres or 0.0):
                x[t] -= term
                m[t] += abs(term)
    for t, b in dict((t, b) for t, b in bias if 0 <= t < V).items():
        x[t] += b
        m[t] += abs(b)
    if mask is not None:
        x[~np.asarray(mask, bool)] = -np.inf
    return x, m
