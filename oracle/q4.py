"""TEST INFRASTRUCTURE ONLY. Values held in 4 bits, attention over caches of them and a beam search's step in float64 numpy,
from their definitions (lokinfer_amd/q4_gpu.py, ops.beam_select_f32_gpu)."""
from __future__ import annotations

import numpy as np


def scale_of(hi, lo):
    """The smallest f16 of at most 8 significant bits with 7 s >= hi and 8 s >= -lo, at most 8128 (hi >= 0 >= lo, f64
    arrays): the first of a few neighbours of max(hi / 7, -lo / 8) on that grid that meets the conditions, which f64
    products decide exactly."""
    a = np.maximum(hi / 7, -lo / 8)
    step = np.exp2(np.maximum(np.floor(np.log2(np.where(a > 0, a, 1.0))) - 7, -24))
    s = np.full(a.shape, np.inf)
    for m in range(2, -3, -1):  # the last that holds is the smallest
        t = (np.ceil(a / step) + m) * step
        odd = t / step <= 256  # 256 steps are 128 of the next size
        s = np.where((t >= 0) & odd & (7 * t >= hi) & (8 * t >= -lo), t, s)
    return np.where(a > 0, np.minimum(s, 8128.0), 0.0)


def quantize(x: np.ndarray):
    """x f16[..., G] -> (codes int[..., G], scales f64[...]); a group that is not finite: scale NaN, codes 8."""
    x = np.asarray(x, np.float64)
    ok = np.isfinite(x).all(-1)
    g = np.where(ok[..., None], x, 0.0)
    s = scale_of(np.maximum(g.max(-1), 0.0), np.minimum(g.min(-1), 0.0))
    c = np.floor(g / np.where(s > 0, s, 1.0)[..., None] + 0.5)
    codes = 8 + np.where(s[..., None] > 0, np.clip(c, -8, 7), 0).astype(np.int64)
    return codes, np.where(ok, s, np.nan)


def weight_values(w: np.ndarray, group: int) -> np.ndarray:
    """w f16[K, N] -> the values f64[K, N] that its 4-bit form holds (groups along K)."""
    k, n = w.shape
    out = np.empty((k, n))
    for k0 in range(0, k, group):
        codes, s = quantize(w[k0:k0 + group].T)
        out[k0:k0 + group] = ((codes - 8) * s[:, None]).T
    return out


def cache_values(k: np.ndarray, v: np.ndarray, kvh: int):
    """Keys and values f64[rows, kvh, 128] that rows f16[rows, kvh 128] are held as; a row (of one head) whose key or value
    is not finite: NaN keys, zero values."""
    rows = k.shape[0]
    out = []
    ok = np.isfinite(k.astype(np.float64)).reshape(rows, kvh, 128).all(-1) & \
        np.isfinite(v.astype(np.float64)).reshape(rows, kvh, 128).all(-1)
    for x, bad in ((k, np.nan), (v, 0.0)):
        x = np.where(ok[..., None], x.reshape(rows, kvh, 128), 0).astype(np.float16)
        codes, s = quantize(x.reshape(rows, kvh, 4, 32))
        y = ((codes - 8) * s[..., None]).reshape(rows, kvh, 128)
        out.append(np.where(ok[..., None], y, bad))
    return out


def attention(q: np.ndarray, key: np.ndarray, val: np.ndarray, pos: int):
    """q f16[T, qh, 128] at positions pos + i over key, val f64[P, kvh, 128] -> (f64[T, qh, 128], the largest score error
    term: sqrt(sum (q k)^2) / sqrt(128) and |score|, over the keys seen)."""
    t, qh, _ = q.shape
    kvh = key.shape[1]
    q = q.astype(np.float64)
    out = np.empty(q.shape)
    term = np.zeros((t, qh))
    for h in range(qh):
        kk, vv = key[:, h // (qh // kvh)], val[:, h // (qh // kvh)]
        for i in range(t):
            n = pos + i + 1
            s = kk[:n] @ q[i, h] / np.sqrt(128)
            e = np.exp(s - s.max())
            out[i, h] = (e / e.sum()) @ vv[:n]
            norm = np.sqrt((kk[:n] ** 2) @ (q[i, h] ** 2)) / np.sqrt(128)
            term[i, h] = (np.sqrt(128) * norm + np.abs(s)).max()
    return out, term


def beam_select(logits, scores, done, k, eos):
    """-> (scores f64[k], parents, tokens, done). A beam's own candidates stand in the order of their logits, which 64 bits of a
    candidate may not tell apart."""
    x = np.asarray(logits, np.float64)
    b, v = x.shape
    cand = np.full((b, v), -np.inf)
    for i in range(b):
        if not np.isfinite(scores[i]):
            continue
        if done[i]:
            cand[i, eos[0]] = scores[i]
            continue
        m = x[i].max()
        if np.isfinite(m):
            cand[i] = float(scores[i]) + (x[i] - (m + np.log(np.exp(x[i] - m).sum())))
    cand = np.where(np.isnan(cand), -np.inf, cand).reshape(-1)
    parent, token = np.divmod(np.arange(b * v), v)
    logit = np.where(np.isfinite(cand) & (np.asarray(done)[parent] == 0), x.reshape(-1), 0.0)
    at = np.lexsort((token, -logit, parent, -cand))[:k]
    parent, token = parent[at], token[at]
    return cand[at], parent, token, np.array([int(bool(done[p]) or t in eos) for p, t in zip(parent, token)])


class _Kv:
    """The cache of OracleLm4: what is written is held in 4 bits."""

    def __init__(self, layers, capacity, dk, dt):
        self.a = np.zeros((layers, 2, capacity, dk), dt)
        self.shape = self.a.shape

    def __getitem__(self, at):
        return self.a[at]

    def __setitem__(self, at, rows):
        rows = np.asarray(rows).astype(np.float16)
        codes, s = quantize(rows.reshape(rows.shape[0], -1, 32))
        self.a[at] = ((codes - 8) * s[..., None]).reshape(rows.shape)


def oracle_lm(sd: dict, cfg, ops, capacity: int, group: int):
    """oracle.qwen3.OracleLm over the values that 4-bit weights, LM head and cache hold."""
    from . import qwen3 as Q

    sd = dict(sd)
    for k in list(sd):
        if k.endswith(".w"):
            sd[k] = weight_values(sd[k], group)
    table = weight_values(sd["embed"].T, group).T

    lm = Q.OracleLm(sd, cfg, ops, capacity)
    lm.kv = _Kv(cfg.layers, capacity, cfg.dk, ops.dt)
    ops.lm_head_last = lambda x, _: ops.c(x)[-1:] @ ops.c(table).T
    return lm
