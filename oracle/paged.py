"""Plain restatement (numpy, 64 bits) of the operators over a paged KV cache: the definition that the kernels are tested against.

TEST INFRASTRUCTURE ONLY, like the rest of this package. A cache is indexed [page][token][head][element] here, whatever its layout in
memory; a batch is (table, q_start, kv_len) as the operators take it.
"""
from __future__ import annotations

import numpy as np


def rope_angles(pos, n_dims, theta_scale, freq_scale=1.0, ext_factor=0.0, attn_factor=1.0, corr=(0.0, 0.0), factors=None):
    """cos and sin times the magnitude, [positions][n_dims / 2], every angle in 64 bits."""
    j = np.arange(n_dims // 2)
    far = np.asarray(pos, np.float64)[:, None] * np.float64(np.float32(theta_scale)) ** j
    if factors is not None:
        far = far / np.asarray(factors, np.float64)
    angle, magnitude = far * np.float64(np.float32(freq_scale)), float(attn_factor)
    if ext_factor:
        y = (j - corr[0]) / max(0.001, corr[1] - corr[0])
        ramp = (1.0 - np.clip(y, 0.0, 1.0)) * ext_factor
        angle = angle * (1.0 - ramp) + far * ramp
        magnitude *= 1.0 + 0.1 * np.log(1.0 / freq_scale)
    return np.cos(angle) * magnitude, np.sin(angle) * magnitude


def rotate(x, cos, sin, n_dims, neox):
    """x [tokens][heads][D]."""
    x = np.asarray(x, np.float64)
    y = x.copy()
    a, b = (slice(0, n_dims // 2), slice(n_dims // 2, n_dims)) if neox else (slice(0, n_dims, 2), slice(1, n_dims, 2))
    c, s = cos[:, None], sin[:, None]
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., a] * s + x[..., b] * c
    return y


def places(q_start, kv_len):
    """(sequence, place among its keys) of every token."""
    out = []
    for s, kv in enumerate(kv_len):
        n = q_start[s + 1] - q_start[s]
        out += [(s, kv - n + j) for j in range(n)]
    return out


def attention(q, k_cache, v_cache, table, q_start, kv_len, scale, softcap=0.0, window=0, prefix=None):
    """q [rows][H][D] -> {row: [H][D]} for the rows of the sequences. prefix: pages and number of keys that come before every
    sequence's own. Hidden keys take no part, whatever they hold; a row that sees none is zero."""
    H, D = q.shape[1:]
    P, Hkv = k_cache.shape[1:3]
    G = H // Hkv
    out = {}

    def keys(cache, pages, n, h):
        m = (n + P - 1) // P
        return np.asarray(cache)[np.asarray(pages[:m], np.int64), :, h].reshape(-1, D)[:n].astype(np.float64)

    for s, kv in enumerate(kv_len):
        n = q_start[s + 1] - q_start[s]
        if not n:
            continue
        for h in range(Hkv):
            k, v = keys(k_cache, table[s], kv, h), keys(v_cache, table[s], kv, h)
            if prefix is not None:
                k = np.concatenate([keys(k_cache, prefix[0], prefix[1], h), k])
                v = np.concatenate([keys(v_cache, prefix[0], prefix[1], h), v])
            before = prefix[1] if prefix is not None else 0
            for j in range(n):
                place = kv - n + j
                lo = max(0, place - window + 1) if window else 0
                hi = max(0, place + 1) + before
                lo = lo if prefix is None else 0
                row = out.setdefault(q_start[s] + j, np.zeros((H, D)))
                if hi <= lo:
                    continue
                x = q[q_start[s] + j, h * G:h * G + G].astype(np.float64) @ k[lo:hi].T * scale
                if softcap:
                    x = softcap * np.tanh(x / softcap)
                p = np.exp(x - x.max(axis=1, keepdims=True))
                row[h * G:h * G + G] = p @ v[lo:hi] / p.sum(axis=1, keepdims=True)
    return out
