"""Rotary positions with several axes, and attention over packed documents, in 64 bits on the CPU."""
from __future__ import annotations

import numpy as np


def rope_axes(x, positions, freqs, axes, nheads, hd, adjacent=False, inverse=False):
    """(y, |x_a| + |x_b| of each element's pair, 0 where it does not turn): float64 [rows, nheads * hd]."""
    x = np.asarray(x, np.float64)
    rows, pairs = x.shape[0], len(freqs)
    y = x[:, :nheads * hd].copy()
    size = np.zeros_like(y)
    for h in range(nheads):
        for i in range(pairs):
            a = h * hd + (2 * i if adjacent else i)
            b = h * hd + (2 * i + 1 if adjacent else i + pairs)
            angle = positions[axes[i]].astype(np.float64) * freqs[i] * (-1.0 if inverse else 1.0)
            y[:, a] = x[:, a] * np.cos(angle) - x[:, b] * np.sin(angle)
            y[:, b] = x[:, b] * np.cos(angle) + x[:, a] * np.sin(angle)
            size[:, a] = size[:, b] = np.abs(x[:, a]) + np.abs(x[:, b])
    return y, size


def attention_docs(q, k, v, offsets, heads, kv_heads, key_offsets=None, max_rows=None, causal=False, prefix=None,
                   softcap=0.0, slopes=None, scale=None, out=None):
    """float64 (out, spread, reach): out over `out`'s values; spread = sum of weight * |v| for each output (how far a
    relative error of the weights can move it); reach [rows, heads] = the largest sum |q_i k_i| * scale plus bias
    that the row's scores were formed from. Only the keys that a row sees are touched."""
    q, k, v = (np.asarray(t, np.float64) for t in (q, k, v))
    key_offsets = offsets if key_offsets is None else key_offsets
    hd = q.shape[1] // heads
    scale = hd ** -0.5 if scale is None else scale
    o = np.zeros((q.shape[0], heads * hd)) if out is None else np.array(out, np.float64)
    spread, reach = np.zeros_like(o), np.zeros((q.shape[0], heads))
    for d in range(len(offsets) - 1):
        q0, k0 = int(offsets[d]), int(key_offsets[d])
        qlen, klen = int(offsets[d + 1]) - q0, int(key_offsets[d + 1]) - k0
        for i in range(qlen if max_rows is None else min(qlen, max_rows)):
            p = i + klen - qlen
            hi = klen if not causal else min(klen, max(p + 1, 0 if prefix is None else int(prefix[d])))
            for h in range(heads):
                col = slice(h * hd, (h + 1) * hd)
                if hi <= 0:
                    o[q0 + i, col] = 0.0
                    continue
                g = h * kv_heads // heads
                kk, vv = k[k0:k0 + hi, g * hd:(g + 1) * hd], v[k0:k0 + hi, g * hd:(g + 1) * hd]
                with np.errstate(all="ignore"):
                    s = kk @ q[q0 + i, col] * scale
                    big = np.abs(kk) @ np.abs(q[q0 + i, col]) * scale
                    if softcap:
                        s = softcap * np.tanh(s / softcap)
                    if slopes is not None:
                        bias = float(slopes[h]) * np.abs(p - np.arange(hi))
                        s, big = s - bias, big + np.abs(bias)
                    w = np.exp(s - s.max())
                    w /= w.sum()
                    o[q0 + i, col] = w @ vv
                    spread[q0 + i, col] = w @ np.abs(vv)
                    reach[q0 + i, h] = big.max()
    return o, spread, reach
