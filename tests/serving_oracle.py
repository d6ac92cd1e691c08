"""The serving operators in 64 bits, on the CPU, written from their definitions in ``include/bgcuda.h``, and the bounds
their results are held to.

A rounding to a type is off by at most half a step, ``finfo.eps / 2`` relative: HALF below.
"""
from __future__ import annotations

import numpy as np
import torch

TORCH = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
HALF = {n: torch.finfo(t).eps / 2 for n, t in TORCH.items()}


def frequencies(rot, base=10000.0, scaling="none", factor=1.0, low=1.0, high=4.0, original=0.0):
    f = np.float64(base) ** (-2.0 * np.arange(rot // 2) / rot)
    if scaling == "linear":
        f = f / factor
    elif scaling == "ramp":
        g = np.clip((original * f / (2 * np.pi) - low) / (high - low), 0.0, 1.0)
        f = f * (g + (1 - g) / factor)
    return f


def rotary(x, positions, f, interleaved=False, magnitude=1.0, inverse=False):
    """x [b, s, h, d] float64, positions [b, s].  Returns the rotation and, element by element, the bound of a 32-bit
    evaluation before its last rounding: the fraction of a turn is rounded to 2^-25 (0.2 * 10^-6 rad), sine and cosine and
    three operations to 2^-23 or better, each on a and b: 2^-21 (|a| + |b|) covers their sum; the angle's 64-bit product
    adds 2^-52 of the angle."""
    r = 2 * len(f)
    ang = positions[..., None].astype(np.float64) * f * (-1.0 if inverse else 1.0)
    c, s = np.cos(ang)[:, :, None], np.sin(ang)[:, :, None]
    y, err = x.copy(), np.zeros_like(x)
    i, j = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    a, b = x[..., i], x[..., j]
    y[..., i], y[..., j] = magnitude * (a * c - b * s), magnitude * (a * s + b * c)
    e = abs(magnitude) * (np.abs(a) + np.abs(b)) * (2.0 ** -21 + 2.0 ** -51 * np.abs(ang).max(initial=0.0))
    err[..., i] = err[..., j] = e
    return y, err


def visible(b, sq, sk, causal, lengths=None, starts=None, prefixes=None, documents=None):
    """[b, sq, sk] truth values, and the positions [b, sq]."""
    lengths = np.full(b, sk) if lengths is None else np.asarray(lengths)
    starts = lengths - sq if starts is None else np.asarray(starts)
    pos = starts[:, None].astype(np.int64) + np.arange(sq)
    key = np.arange(sk)
    seen = np.broadcast_to((key[None, :] < lengths[:, None])[:, None, :], (b, sq, sk)).copy()
    if causal:
        first = np.zeros(b, np.int64) if prefixes is None else np.asarray(prefixes)
        seen &= (key <= pos[..., None]) | (key < first[:, None, None])
        seen &= ((pos >= 0) & (pos < lengths[:, None]))[..., None]
    if documents is not None and sk:
        doc = np.asarray(documents)
        inside = (pos >= 0) & (pos < sk)
        mine = np.where(inside, np.take_along_axis(doc, np.clip(pos, 0, sk - 1), 1), -1)
        seen &= (mine[..., None] == doc[:, None, :]) & (mine >= 0)[..., None]
    return seen, pos


def attention(q, k, v, dtype, scale, causal=True, softcap=0.0, slopes=None, documents=None, prefixes=None, lengths=None,
              starts=None):
    """q [b, hq, sq, d], k, v [b, hkv, sk, d] float64 -> the result and its bound.

    Bound: the last rounding HALF |o|; a 16-bit probability's rounding HALF sum p |v|; and the exponent's error, which
    moves a probability relatively: the dot product in 32 bits (d terms, for float32 three tf32 products whose dropped
    part is 2^-21 of a term) is off by (d + 16) 2^-23 of sum |q||k|, cap, bias and the scaling by a few 2^-23 of their own
    size, the sums over n keys by n 2^-24, the exponential by 2^-21; a 16-bit tanh by 2^-21 of the cap.  Numerator and
    denominator both carry it, hence twice."""
    b, hq, sq, d = q.shape
    hkv, sk = k.shape[1], k.shape[2]
    seen, pos = visible(b, sq, sk, causal, lengths, starts, prefixes, documents)
    out, err = np.zeros_like(q), np.zeros_like(q)
    u = HALF[dtype]
    for i in range(b):
        for h in range(hq):
            g = h // (hq // hkv)
            s = scale * (q[i, h] @ k[i, g].T)
            size = abs(scale) * (np.abs(q[i, h]) @ np.abs(k[i, g]).T)
            delta = (d + 16) * 2.0 ** -23 * size
            if softcap:
                s = softcap * np.tanh(s / softcap)
                delta = delta + 2.0 ** -21 * softcap
            if slopes is not None:
                bias = slopes[h] * np.abs(pos[i][:, None] - np.arange(sk))
                s = s - bias
                delta = delta + 2.0 ** -22 * np.abs(bias)
            delta = delta + 2.0 ** -22 * np.abs(s)
            m = seen[i]
            s = np.where(m, s, -np.inf)
            top = s.max(-1, keepdims=True, initial=-np.inf)
            p = np.where(m, np.exp(s - np.where(np.isinf(top), 0.0, top)), 0.0)
            total = p.sum(-1, keepdims=True)
            p = p / np.where(total == 0, 1.0, total)
            vv = np.where(m.any(0)[:, None], v[i, g], 0.0)
            out[i, h] = p @ vv
            # only what weighs counts: an error in the exponent of a vanishing probability vanishes with it
            rel = (p * delta).sum(-1, keepdims=True) + sk * 2.0 ** -24 + 2.0 ** -21
            weight = (p * (delta + rel + (u if dtype != "float32" else 0.0))) @ np.abs(vv)
            # a 16-bit probability below the type's normal range is off by half its smallest step instead: 2^-25 of the
            # largest probability of its row (float16; bfloat16 has float32's range)
            floor = (2.0 ** -25 * p.max(-1, keepdims=True, initial=0.0) * m) @ np.abs(vv) if dtype == "float16" else 0.0
            err[i, h] = weight + floor + u * np.abs(out[i, h])
    if dtype == "float16":
        err = err + 2.0 ** -25          # a result below the normal range of float16
    return out, err


def sample(logits, u, temperature, top_k=0, top_p=1.0, min_p=0.0):
    """One row: (token, chance)."""
    x = logits.astype(np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    if not (x > -np.inf).any():
        return -1, 0.0
    if not temperature > 0:
        return int(np.argmax(x)), 1.0
    order = np.argsort(-x, kind="stable")
    top = x[order[0]]
    with np.errstate(invalid="ignore"):
        w = np.where(x == -np.inf, 0.0, np.where(x == top, 1.0, np.exp((x - top) / np.float64(temperature))))
    ws = w[order]
    n = len(ws) if top_k <= 0 else min(top_k, len(ws))
    if top_p < 1:
        sums = np.cumsum(ws[:n])
        n = max(1, int(np.count_nonzero(np.concatenate([[0.0], sums[:-1]]) < max(np.float64(np.float32(top_p)), 0.0) * sums[-1])))
    n = max(1, min(n, int(np.count_nonzero(ws >= np.float64(np.float32(min_p))))))
    kept = np.sort(order[:n])
    sums = np.cumsum(w[kept])
    u = min(max(float(np.float32(u)), 0.0), 1.0)
    at = int(np.searchsorted(sums, u * sums[-1], side="right"))
    at = min(at, int(np.flatnonzero(w[kept] > 0)[-1]))
    return int(kept[at]), float(w[kept[at]] / sums[-1])


def attention_bound(q, k, v, want, dtype, scale, softcap=0.0, smallest=2.0 ** -25, **rules):
    """``attention``'s bound with two parts held closer, for its result ``want`` without a bias.

    The cap: tanh is off by 2^-20 of its value, whatever the cap.  Up to 1 the odd polynomial is off by 6.2e-7 and its eight
    operations by 2^-24 each, together below 2^-20; beyond 1 the form 1 - 2 / (1 + e^2x) is off by at most 2^-21 (the
    quotient lies in [0, 2], division and exponential are good to 2 units), of a value above 0.76.
    float16: a probability too small for its type is off by ``smallest`` of the largest of its row."""
    b, hq, sq, d = q.shape
    group = hq // k.shape[1]
    k, v = np.repeat(k, group, 1), np.repeat(v, group, 1)
    seen, _ = visible(b, sq, k.shape[2], rules.get("causal", True), *(rules.get(n) for n in ("lengths", "starts", "prefixes", "documents")))
    seen = seen[:, None]
    s = scale * (q @ k.swapaxes(-1, -2))
    delta = (d + 16) * 2.0 ** -23 * abs(scale) * (np.abs(q) @ np.abs(k).swapaxes(-1, -2))
    if softcap:
        s = softcap * np.tanh(s / softcap)
        delta = delta + 2.0 ** -20 * np.abs(s)
    delta = delta + 2.0 ** -22 * np.abs(s)
    p = np.where(seen, np.exp(s - np.where(seen, s, -np.inf).max(-1, keepdims=True, initial=-1e300)), 0.0)
    total = p.sum(-1, keepdims=True)
    p = p / np.where(total == 0, 1.0, total)
    rel = (p * delta).sum(-1, keepdims=True) + k.shape[2] * 2.0 ** -24 + 2.0 ** -21
    size = np.abs(v)
    err = (p * (delta + rel + (HALF[dtype] if dtype != "float32" else 0.0))) @ size + HALF[dtype] * np.abs(want)
    if dtype == "float16":
        err = err + (smallest * p.max(-1, keepdims=True, initial=0.0) * seen) @ size + 2.0 ** -25
    return err
