"""Plain restatements, in 64 bits, of the 4-bit format and of the logits rules (include/b200q8.h)."""
from __future__ import annotations

import numpy as np


def round_to_bf16(v: np.ndarray) -> np.ndarray:
    """float64 values rounded once to bfloat16 (8 significant bits, exponents down to 2^-133), ties to even."""
    v = np.asarray(v, np.float64)
    with np.errstate(invalid="ignore", over="ignore"):
        _, e = np.frexp(v)
        step = np.ldexp(1.0, np.maximum(e - 8, -133))
        r = np.rint(v / step) * step
    r = np.where(np.isfinite(v), r, v)
    return np.where(np.abs(r) >= 2.0 ** 128, np.copysign(np.inf, r), r)


def bf16_bits(v: np.ndarray) -> np.ndarray:
    """Bits of values that are bfloat16 already."""
    return (np.asarray(v, np.float32).view(np.uint32) >> 16).astype(np.uint16)


def quantize(w: np.ndarray, group: int):
    """(q int64 [N, K] in -8..7, scales float64 [N, ng]) by the definition."""
    w = np.asarray(w, np.float64)
    N, K = w.shape
    ng = -(-K // group)
    q, s = np.zeros((N, K), np.int64), np.zeros((N, ng))
    for g in range(ng):
        part = w[:, g * group:(g + 1) * group]
        top = np.nanmax(np.where(np.isnan(part), 0.0, np.abs(part)), axis=1)
        sc = round_to_bf16(top / 7.0)
        with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
            r = np.rint(part / sc[:, None])
        r = np.where((sc[:, None] > 0) & ~np.isnan(r), np.clip(r, -8, 7), 0.0)
        q[:, g * group:(g + 1) * group] = r.astype(np.int64)
        s[:, g] = sc
    return q, s


def pack(q: np.ndarray) -> np.ndarray:
    """uint8 [N, ceil(K/2)] codes of integers -8..7."""
    c = (q + 8).astype(np.uint8)
    if c.shape[1] % 2:
        c = np.concatenate([c, np.full((c.shape[0], 1), 8, np.uint8)], axis=1)
    return c[:, 0::2] | (c[:, 1::2] << 4)


def values(q: np.ndarray, s: np.ndarray, group: int) -> np.ndarray:
    """float64 [N, K]."""
    return q * np.repeat(s, group, axis=1)[:, :q.shape[1]]


def linear(x, q, s, group, bias=None, residual=None) -> np.ndarray:
    y = np.asarray(x, np.float64) @ values(q, s, group).T
    if bias is not None:
        y = y + np.asarray(bias, np.float64)
    if residual is not None:
        y = y + np.asarray(residual, np.float64)
    return y


def logits(x, out_dtype, history=None, history_len=None, prompt_len=None, repetition=None, presence=None,
           frequency=None, bias_ids=None, bias_values=None, bias_len=None, allowed=None):
    """(out, token) of the rules, token by token, in float32 as the header states the operations."""
    M, V = x.shape
    f32 = np.float32
    out, token = np.empty((M, V), out_dtype), np.empty(M, np.int32)

    def row(t, m):
        return None if t is None else t[m if t.ndim == 2 and t.shape[0] > 1 else 0] if t.ndim == 2 else t

    with np.errstate(all="ignore"):
        for m in range(M):
            v = x[m].astype(f32)
            h = row(history, m)
            if h is not None:
                n = int(np.clip(history_len[m], 0, len(h)))
                p = 0 if prompt_len is None else int(np.clip(prompt_len[m], 0, n))
                rep = f32(1 if repetition is None else repetition[m])
                for t in set(h[:n].tolist()):
                    if 0 <= t < V:
                        v[t] = v[t] / rep if v[t] > 0 else v[t] * rep
                made = h[p:n].tolist()
                for t in set(made):
                    if 0 <= t < V:
                        v[t] = v[t] - f32(0 if frequency is None else frequency[m]) * f32(made.count(t))
                        v[t] = v[t] - f32(0 if presence is None else presence[m])
            b = row(bias_ids, m)
            if b is not None:
                n = len(b) if bias_len is None else int(np.clip(bias_len[m], 0, len(b)))
                for t, bv in dict(zip(b[:n].tolist(), row(bias_values, m)[:n])).items():
                    if 0 <= t < V:
                        v[t] = v[t] + f32(bv)
            ok = np.ones(V, bool)
            a = row(allowed, m)
            if a is not None:
                ok = (np.ascontiguousarray(a).view(np.uint32)[np.arange(V) // 32] >> (np.arange(V) % 32).astype(np.uint32)) & 1 > 0
                v[~ok] = -np.inf
            out[m] = v.astype(out_dtype)
            cand = np.flatnonzero(ok)
            best = -1
            for i in cand:  # std::max_element: the first stays unless a later one is larger
                if best < 0 or out[m, best] < out[m, i]:
                    best = int(i)
            token[m] = best
    return out, token
