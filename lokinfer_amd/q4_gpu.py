"""`lk.ops.q4_gpu` (MI355X backend; no counterpart in the reference): serving with weights and caches held in 4 bits. f16
activations, f32 sums, one rounding to f16 at each output, as `lk.ops.f16_gpu`, whose ops these stand beside.

A value held in 4 bits is s (c - 8): a code c of 0 .. 15 and its group's scale s, an f16 >= 0 of at most 8 significant
bits, so that the product is exact in f16. A group's scale is the smallest such s with 7 s >= its largest and 8 s >= minus
its smallest value (at most 8128: larger magnitudes than 56896 are clamped); codes are rounded to nearest, halves up. A group
that holds an infinity or a NaN becomes NaN.

Weights (`pack_w4`): groups of 32, 64 or 128 consecutive k of one column, laid out once for the kernels.
Caches (`kv4_cache`): u8[B, 2, kvh, 72 P], 72 bytes a row and kv head where f16 takes 256; groups of 32 of a head's 128
values. B sequences, each at its own position; P is a multiple of 32. The ops write a cache in place, so the Tensor given
must be contiguous memory of the cache (a Tensor made from a strided view is a copy).

All operands lie on the GPU of `GpuContext.shared()`. Ops run on the current stream and take what scratch memory they need
from torch's allocator there, so calls on different streams, or in different captured graphs, share none.
"""
from __future__ import annotations

import numpy as np
import torch

from .graph import current_graph
from .ops import OpError, _launch, check
from .runtime import GpuContext
from .tensor import Tensor, f16, f32, i32, i64, u8

GROUPS = (32, 64, 128)
ROW = 72  # bytes of a cache row: 64 of codes, 4 f16 scales
HD = 128


def _on_gpu(*xs):
    if current_graph() is not None:
        raise OpError("the 4-bit ops run eagerly or in a stream-captured function (lk.capture), not in a traced one")
    for x in xs:
        check(isinstance(x, Tensor), f"expected lk.Tensor, got {type(x).__name__}")
        check(x.device == "gpu", "GPU kernel operands must be on the GPU (use ops.to_gpu)")
    dev = GpuContext.shared().device
    for x in xs:
        check(x.t.device == dev, f"operands must be on {dev}, got one on {x.t.device}")


def _typed(x, dtype, rank, what):
    check(isinstance(x, Tensor) and x.dtype == dtype and x.ndim == rank, f"{what} must be a rank {rank} {dtype.name} tensor")


# ---- weights ------------------------------------------------------------------------------------------------

class PackedWeight4:
    """A weight [K, N] in 4 bits on the device: codes `q` and scales `s` in the kernels' layout; `shape` is the logical
    (K, N), `group` the k that share a scale."""

    def __init__(self, q: Tensor, s: Tensor, shape, group: int):
        k, n = (int(d) for d in shape)
        check(group in GROUPS and k > 0 and n > 0, "group must be 32, 64 or 128, the shape positive")
        tiles = (-(-n // 16), -(-k // 128))
        check(isinstance(q, Tensor) and q.dtype == i32 and tuple(q.shape) == tiles + (256,), "q does not fit the shape")
        check(isinstance(s, Tensor) and s.dtype == f16 and tuple(s.shape) == tiles + (16, 128 // group),
              "s does not fit the shape and group")
        self.q, self.s, self.shape, self.group = q, s, (k, n), group


def _w4_shapes(k, n, group):
    check(group in GROUPS, "group must be 32, 64 or 128")
    check(k > 0 and n > 0, "a weight needs at least one row and column")
    t = (-(-n // 16), -(-k // 128))
    return [t + (256,), t + (16, 128 // group)]


def quantize_w4_f16_gpu(w, group: int = 64, nt: bool = False) -> PackedWeight4:
    """w f16[K, N] (nt: f16[N, K], an embedding table as the LM head's weight) -> PackedWeight4."""
    _on_gpu(w)
    _typed(w, f16, 2, "w")
    k, n = (w.shape[1], w.shape[0]) if nt else w.shape
    q, s = _launch("quantize_w4_f16_gpu", [w], _w4_shapes(k, n, group), dict(group=int(group), nt=int(bool(nt))),
                   out_dtypes=[i32, f16])
    return PackedWeight4(q, s, (k, n), group)


def _scales_ok(s: torch.Tensor) -> bool:
    """Whether every f16 scale is finite, >= 0, at most 8128 and has at most 8 significant bits."""
    bits = s.contiguous().view(torch.int16).to(torch.int32)
    low = torch.where(bits >= 0x400, bits & 7, 0)  # a normal number: the last 3 of its 11 bits
    sub = bits & 0x3FF                             # a subnormal one: an odd part below 256
    odd = torch.where((bits < 0x400) & (sub > 0), sub // (sub & -sub).clamp(min=1), 0)
    return bool(((bits >= 0) & (bits <= 0x6FF0) & (low == 0) & (odd < 256)).all())


def pack_w4(w, scales=None, group: int = 64, nt: bool = False) -> PackedWeight4:
    """A weight into the kernels' layout: w f16[K, N] (numpy array or lk.Tensor; nt: f16[N, K]), quantised here, or its
    codes u8[K, N] (0 .. 15) with scales f16[ceil(K / group), N] (>= 0, at most 8 significant bits and 8128)."""
    def up(a, dtype):
        if isinstance(a, Tensor):
            return a
        return Tensor(torch.from_numpy(np.ascontiguousarray(a, dtype)).to(GpuContext.shared().device))

    if scales is None:
        return quantize_w4_f16_gpu(up(w, np.float16), group, nt)
    check(not nt, "codes are given as u8[K, N]")
    codes, scales = up(w, np.uint8), up(scales, np.float16)
    _on_gpu(codes, scales)
    _typed(codes, u8, 2, "codes")
    _typed(scales, f16, 2, "scales")
    shapes = _w4_shapes(*codes.shape, group)
    check(tuple(scales.shape) == (-(-codes.shape[0] // group), codes.shape[1]), "scales must be f16[ceil(K / group), N]")
    check(bool((codes.t < 16).all()), "codes must be 0 .. 15")
    check(_scales_ok(scales.t), "scales must be >= 0, at most 8128, of at most 8 significant bits")
    q, s = _launch("pack_w4_u8_gpu", [codes, scales], shapes, dict(group=int(group)), out_dtypes=[i32, f16])
    return PackedWeight4(q, s, codes.shape, group)


def unpack_w4_f16_gpu(w: PackedWeight4):
    """The weight's values, f16[K, N] (exact)."""
    _w(w)
    return _launch("unpack_w4_f16_gpu", [w.q, w.s], [w.shape], dict(group=w.group), out_dtypes=[f16])


def _w(w) -> PackedWeight4:
    check(isinstance(w, PackedWeight4), "the weight must be a PackedWeight4 (pack_w4)")
    _on_gpu(w.q, w.s)
    return w


def _gemm_rule(x, *ws):
    _on_gpu(x)
    _typed(x, f16, 2, "x")
    for w in ws:
        _w(w)
        check(x.shape[1] == w.shape[0], f"x [M, K] and w [K, N]: inner dims differ: {x.shape}, {w.shape}")
        check(w.shape == ws[0].shape and w.group == ws[0].group, "both weights must have one shape and group")
    check(x.shape[1] % 8 == 0, "K must be a multiple of 8")
    return x.shape[0], ws[0].shape[1]


def _gemm(name, x, ws, extra=(), norm=None, dtype=f16):
    m, n = _gemm_rule(x, *ws)
    attrs = dict(group=ws[0].group)
    ops = [x]
    if norm is not None:
        ops.append(norm[0])
        attrs["eps"] = float(norm[1])
    for w in ws:
        ops += [w.q, w.s]
    return _launch(name, ops + list(extra), [(m, n)], attrs, out_dtypes=[dtype])


def gemm_w4_f16_gpu(x, w):
    """x f16[M, K] @ w -> f16[M, N] (f32 sums)."""
    return _gemm("gemm_w4_f16_gpu", x, [w])


def gemm_w4_bias_f16_gpu(x, w, b):
    """x @ w + b (b f16[N])."""
    _on_gpu(b)
    _typed(b, f16, 1, "b")
    check(b.shape[0] == _w(w).shape[1], "b must be f16[N]")
    return _gemm("gemm_w4_bias_f16_gpu", x, [w], [b])


def gemm_w4_add_f16_gpu(x, w, res):
    """res + x @ w (res f16[M, N])."""
    _on_gpu(x, res)
    _typed(res, f16, 2, "res")
    check(tuple(res.shape) == (x.shape[0], _w(w).shape[1]), "res must be f16[M, N]")
    return _gemm("gemm_w4_add_f16_gpu", x, [w], [res])


def gemm_w4_swiglu_f16_gpu(x, gate, up):
    """silu(x @ gate) * (x @ up) -> f16[M, N]; both weights of one shape and group."""
    return _gemm("gemm_w4_swiglu_f16_gpu", x, [gate, up])


def lm_head_w4_f16_gpu(x, w):
    """Logits x @ w -> f32[M, V] of every row (w: the table f16[V, D] packed with nt=True)."""
    return _gemm("lm_head_w4_f16_gpu", x, [w], dtype=f32)


def _normed(name, x, g, ws, eps, dtype=f16):
    """rmsnorm(x, g) in front of a product: inside it for one row, else by rmsnorm_f16_gpu; the same bits."""
    from .f16_gpu import rmsnorm_f16_gpu

    _gemm_rule(x, *ws)
    _on_gpu(g)
    _typed(g, f16, 1, "g")
    check(g.shape[0] == x.shape[1], "g must be f16[K]")
    if x.shape[0] == 1:
        return _gemm("rmsnorm_" + name, x, ws, norm=(g, eps), dtype=dtype)
    return _gemm(name, rmsnorm_f16_gpu(x, g, eps), ws, dtype=dtype)


def rmsnorm_gemm_w4_f16_gpu(x, g, w, eps=1e-6):
    """gemm_w4(rmsnorm(x, g), w)."""
    return _normed("gemm_w4_f16_gpu", x, g, [w], eps)


def rmsnorm_gemm_w4_swiglu_f16_gpu(x, g, gate, up, eps=1e-6):
    """gemm_w4_swiglu(rmsnorm(x, g), gate, up)."""
    return _normed("gemm_w4_swiglu_f16_gpu", x, g, [gate, up], eps)


def rmsnorm_lm_head_w4_f16_gpu(x, g, w, eps=1e-6):
    """lm_head_w4(rmsnorm(x, g), w) -> f32[M, V]."""
    return _normed("lm_head_w4_f16_gpu", x, g, [w], eps, dtype=f32)


# ---- caches --------------------------------------------------------------------------------------------------

def kv4_cache(batch: int, kv_heads: int, capacity: int, layers: int | None = None) -> Tensor:
    """A zeroed cache of at least `capacity` rows (rounded up to a multiple of 32): u8[B, 2, kvh, 72 P], with `layers`
    u8[L, B, 2, kvh, 72 P]."""
    check(batch > 0 and kv_heads > 0 and capacity > 0 and (layers is None or layers > 0), "sizes must be positive")
    shape = (batch, 2, kv_heads, ROW * (-(-capacity // 32) * 32))
    return Tensor(torch.zeros(shape if layers is None else (layers,) + shape, dtype=torch.uint8,
                              device=GpuContext.shared().device))


def kv4_capacity(kv: Tensor) -> int:
    """Rows of a cache."""
    check(isinstance(kv, Tensor) and kv.dtype == u8 and kv.shape[-1] > 0 and kv.shape[-1] % (32 * ROW) == 0,
          "a 4-bit cache is u8[..., 72 P] with P a multiple of 32")
    return kv.shape[-1] // ROW


def _kv(kv, pos):
    _on_gpu(kv, pos)
    kv4_capacity(kv)
    check(kv.ndim == 4 and kv.shape[0] > 0 and kv.shape[1] == 2 and kv.shape[2] > 0, "kv must be u8[B, 2, kvh, 72 P]")
    check(pos.dtype == i64 and tuple(pos.shape) == (kv.shape[0],), "pos must be i64[B]")
    return kv.shape[0], kv.shape[2]


def _rows(x, b, what):
    _typed(x, f16, 2, what)
    check(x.shape[0] % b == 0, f"{what} must have B T rows")


def kv4_write_f16_gpu(kv, k, v, pos):
    """Rows pos[b] .. pos[b] + T - 1 of sequence b = k, v f16[B T, kvh 128], quantised (kv in place); rows outside the cache
    are dropped. A row whose key or value is not finite makes every query that sees it NaN."""
    b, kvh = _kv(kv, pos)
    _on_gpu(k, v)
    _rows(k, b, "k")
    check(tuple(v.shape) == tuple(k.shape) and v.dtype == f16 and k.shape[1] == HD * kvh, "k, v must be f16[B T, kvh 128]")
    return _launch("kv4_write_f16_gpu", [kv, k, v, pos], [], outs=[], inout=[0])


def qknorm_rope_kv4_f16_gpu(qkv, qg, kg, pos, kv, eps=1e-6, theta=1e6):
    """QK-norm + RoPE + cache write: qkv f16[B T, (qh + 2 kvh) 128] (q | k | v), row i of sequence b at position pos[b] + i.
    Returns q = rope(rmsnorm_heads(q, qg)) f16[B T, qh 128] and writes k = rope(rmsnorm_heads(k, kg)) and v as
    kv4_write does."""
    b, kvh = _kv(kv, pos)
    _on_gpu(qkv, qg, kg)
    _rows(qkv, b, "qkv")
    for g in (qg, kg):
        _typed(g, f16, 1, "qg, kg")
        check(g.shape[0] == HD, "qg and kg must be f16[128]")
    dq = qkv.shape[1] - 2 * kvh * HD
    check(dq > 0 and dq % HD == 0, "qkv must be f16[B T, (qh + 2 kvh) 128]")
    return _launch("qknorm_rope_kv4_f16_gpu", [qkv, qg, kg, pos, kv], [(qkv.shape[0], dq)],
                   dict(eps=float(eps), theta=float(theta)), out_dtypes=[f16], inout=[4])


def kv4_read_f16_gpu(kv):
    """The values that a cache (or any u8[..., 72 P] part of one) holds: f16[..., P, 128]."""
    _on_gpu(kv)
    cap = kv4_capacity(kv)
    flat = Tensor(kv.t.view(-1, kv.shape[-1]))
    out = _launch("kv4_read_f16_gpu", [flat], [(flat.shape[0], cap, HD)], out_dtypes=[f16])
    return Tensor(out.t.view(*kv.shape[:-1], cap, HD))


def attention_kv4_f16_gpu(q, kv, pos):
    """Causal attention over a 4-bit cache: query i of sequence b (row b T + i of q f16[B T, qh 128], position pos[b] + i)
    attends to rows 0 .. pos[b] + i of its kv head (already written); qh a multiple of the cache's kvh; scale
    1 / sqrt(128) -> f16[B T, qh 128]. A query whose position is outside the cache (with a negative pos[b], every query of
    the sequence) gives NaN and a device error."""
    b, kvh = _kv(kv, pos)
    _on_gpu(q)
    _rows(q, b, "q")
    check(q.shape[1] > 0 and q.shape[1] % (HD * kvh) == 0, "q must be f16[B T, qh 128], qh a multiple of kvh")
    need = GpuContext.shared().lib.lk_hip_kv4_attention_workspace_bytes(b, q.shape[0] // b, q.shape[1] // HD, kvh,
                                                                        kv4_capacity(kv))
    out, _ = _launch("attention_kv4_f16_gpu", [q, kv, pos], [tuple(q.shape), (-(-need // 4),)], out_dtypes=[f16, f32])
    return out


def kv4_reorder_gpu(kv, parents, n):
    """Beam search: rows 0 .. n - 1 of sequence b of kv u8[L, B, 2, kvh, 72 P] become those of sequence parents[b], in
    place (parents i64[B], n i64[1]; B <= 32, L kvh <= 32767). A parent out of range gives NaN rows and a device error."""
    _on_gpu(kv, parents, n)
    kv4_capacity(kv)
    check(kv.ndim == 5 and kv.shape[2] == 2 and 0 < kv.shape[1] <= 32 and kv.shape[0] > 0 and kv.shape[3] > 0,
          "kv must be u8[L, B, 2, kvh, 72 P] with B <= 32")
    check(kv.shape[0] * kv.shape[3] <= 32767, "L kvh must be at most 32767")
    check(parents.dtype == i64 and tuple(parents.shape) == (kv.shape[1],), "parents must be i64[B]")
    check(n.dtype == i64 and tuple(n.shape) == (1,), "n must be i64[1]")
    return _launch("kv4_reorder_gpu", [kv, parents, n], [], outs=[], inout=[0])


__all__ = [n for n in dir() if n.endswith(("_f16_gpu", "_reorder_gpu"))] + ["pack_w4", "PackedWeight4", "kv4_cache",
                                                                            "kv4_capacity"]
