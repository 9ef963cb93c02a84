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

import functools

import numpy as np
import torch

from ._lib import lib
from .graph import current_graph
from .ops import OpError, check
from .runtime import GpuContext
from .tensor import Tensor, f16, i32

GROUPS = (32, 64, 128)
ROW = 72  # bytes of a cache row: 64 of codes, 4 f16 scales
HD = 128

_NO_WORK = torch.empty(0, dtype=torch.float32)
_F16, _F32, _I32, _I64, _U8 = torch.float16, torch.float32, torch.int32, torch.int64, torch.uint8


_index = None  # of the context's GPU


def _arg(x, dtype, rank, what) -> torch.Tensor:
    """The torch tensor of an operand: of this type and rank, on the context's GPU."""
    global _index
    if not isinstance(x, Tensor):
        raise OpError(f"{what}: expected lk.Tensor, got {type(x).__name__}")
    t = x.t
    if t.dtype is not dtype or t.dim() != rank or t.get_device() != _index or _index is None:
        if t.dtype is not dtype or t.dim() != rank:
            raise OpError(f"{what} must be a rank {rank} {str(dtype)[6:]} tensor, got {str(t.dtype)[6:]}{list(t.shape)}")
        if not t.is_cuda:
            raise OpError(f"{what}: GPU kernel operands must be on the GPU (use ops.to_gpu)")
        _index = GpuContext.shared().device.index
        if t.get_device() != _index:
            raise OpError(f"{what} must be on cuda:{_index}, is on {t.device}")
    return t


def _run(name, ptrs, ints, floats=()):
    if current_graph() is not None:
        raise OpError("the 4-bit ops run eagerly or in a stream-captured function (lk.capture), not in a traced one")
    GpuContext.shared().run(name, ptrs, ints, floats)


def _call(name, tensors, attrs=(), floats=()):
    """Registry kernel `name` over torch tensors (operands, then outs) and its int and float attributes."""
    ints: list[int] = []
    for t in tensors:
        ints += t.shape
    ints += attrs
    _run(name, [t.data_ptr() for t in tensors], ints, floats)


@functools.lru_cache(maxsize=1024)
def _attention_bytes(b, t, qh, kvh, cap) -> int:
    return lib().lk_hip_kv4_attention_workspace_bytes(b, t, qh, kvh, cap)


def _empty(shape, dtype=_F16) -> torch.Tensor:
    return torch.empty(shape, dtype=dtype, device=GpuContext.shared().device)


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
        check(q.t.is_cuda and q.t.device == s.t.device, "q and s must be on one GPU")
        self._q, self._s, self.shape, self.group = q.t, s.t, (k, n), group
        self._dims = (*q.shape, *s.shape)

    @property
    def q(self) -> Tensor:
        return Tensor(self._q)

    @property
    def s(self) -> Tensor:
        return Tensor(self._s)


def _w4_empty(k, n, group):
    check(group in GROUPS, "group must be 32, 64 or 128")
    check(k > 0 and n > 0, "a weight needs at least one row and column")
    tiles = (-(-n // 16), -(-k // 128))
    return _empty(tiles + (256,), _I32), _empty(tiles + (16, 128 // group))


def quantize_w4_f16_gpu(w, group: int = 64, nt: bool = False) -> PackedWeight4:
    """w f16[K, N] (nt: f16[N, K], an embedding table as the LM head's weight) -> PackedWeight4."""
    wt = _arg(w, _F16, 2, "w")
    n, k = wt.shape if nt else reversed(wt.shape)
    q, s = _w4_empty(k, n, group)
    _call("quantize_w4_f16_gpu", [wt, q, s], [group, int(bool(nt))])
    return PackedWeight4(Tensor(q), Tensor(s), (k, n), group)


_CODES, _SCALES = "codes must be 0 .. 15", "scales must be >= 0, at most 8128, of at most 8 significant bits"


def _held(a, dtype, said):
    """Host values as `dtype`, which must hold them as they are; an lk.Tensor as it is."""
    if isinstance(a, Tensor):
        return a
    given = np.asarray(a)
    with np.errstate(invalid="ignore", over="ignore"):
        cast = np.ascontiguousarray(given, dtype)
    check(cast.dtype == given.dtype or np.array_equal(cast, given), said)
    return cast


def _up(a, dtype) -> Tensor:
    if isinstance(a, Tensor):
        return a
    return Tensor(torch.from_numpy(np.ascontiguousarray(a, dtype)).to(GpuContext.shared().device))


def pack_w4(w, scales=None, group: int = 64, nt: bool = False) -> PackedWeight4:
    """A weight into the kernels' layout: w f16[K, N] (numpy array or lk.Tensor; nt: f16[N, K]), quantised here, or its
    codes u8[K, N] (0 .. 15) with scales f16[ceil(K / group), N] (>= 0, at most 8 significant bits and 8128); codes and
    scales in arrays of other types must be values that u8 and f16 hold. The weight is ready for every stream."""
    if scales is None:
        packed = quantize_w4_f16_gpu(_up(w, np.float16), group, nt)
        if not torch.cuda.is_current_stream_capturing():  # like an uploaded weight: ready for every stream that may run first
            torch.cuda.current_stream(packed._q.device).synchronize()
        return packed
    check(not nt, "codes are given as u8[K, N]")
    codes, scales = _held(w, np.uint8, _CODES), _held(scales, np.float16, _SCALES)
    codes, scales = _arg(_up(codes, np.uint8), _U8, 2, "codes"), _arg(_up(scales, np.float16), _F16, 2, "scales")
    k, n = codes.shape
    q, s = _w4_empty(k, n, group)
    check(tuple(scales.shape) == (-(-k // group), n), "scales must be f16[ceil(K / group), N]")
    flag = torch.zeros(1, dtype=_I32, device=codes.device)
    _call("pack_w4_u8_gpu", [codes, scales, flag, q, s], [group])
    bad = int(flag)  # waits for the layout: once per weight
    check(not bad & 1, _CODES)
    check(not bad, _SCALES)
    return PackedWeight4(Tensor(q), Tensor(s), (k, n), group)


def unpack_w4_f16_gpu(w: PackedWeight4):
    """The weight's values, f16[K, N] (exact)."""
    out = _empty(_w(w).shape)
    _call("unpack_w4_f16_gpu", [w._q, w._s, out], [w.group])
    return Tensor(out)


def _w(w) -> PackedWeight4:
    if not isinstance(w, PackedWeight4):
        raise OpError("the weight must be a PackedWeight4 (pack_w4)")
    if w._q.get_device() != _index:
        _arg(w.q, _I32, 3, "the weight")
    return w


def _gemm(name, x, w, w2=None, extra=None, norm=None, dtype=_F16):
    """Registry product `name` of x and one or two weights; extra: (tensor, rank, name) of a bias or residual; norm:
    (gain, eps)."""
    xt = _arg(x, _F16, 2, "x")
    (m, k), (wk, n) = xt.shape, _w(w).shape
    if k != wk:
        raise OpError(f"x [M, K] and w [K, N]: inner dims differ: {tuple(xt.shape)}, {w.shape}")
    if k % 8:
        raise OpError("K must be a multiple of 8")
    out = xt.new_empty((m, n), dtype=dtype)
    ptrs, ints, floats = [xt.data_ptr()], [m, k], ()
    if norm is not None:
        g = _arg(norm[0], _F16, 1, "g")
        if g.shape[0] != k:
            raise OpError("g must be f16[K]")
        ptrs.append(g.data_ptr())
        ints.append(k)
        floats = (float(norm[1]),)
    ptrs += (w._q.data_ptr(), w._s.data_ptr())
    ints += w._dims
    if w2 is not None:
        if _w(w2).shape != w.shape or w2.group != w.group:
            raise OpError("both weights must have one shape and group")
        ptrs += (w2._q.data_ptr(), w2._s.data_ptr())
        ints += w2._dims
    if extra is not None:
        t = _arg(extra[0], _F16, extra[1], extra[2])
        if t.shape != ((m, n) if extra[1] == 2 else (n,)):
            raise OpError(f"{extra[2]} must be f16{'[M, N]' if extra[1] == 2 else '[N]'}")
        ptrs.append(t.data_ptr())
        ints += t.shape
    ptrs.append(out.data_ptr())
    ints += (m, n, w.group)
    _run(name, ptrs, ints, floats)
    return Tensor(out)


def gemm_w4_f16_gpu(x, w):
    """x f16[M, K] @ w -> f16[M, N] (f32 sums)."""
    return _gemm("gemm_w4_f16_gpu", x, w)


def gemm_w4_bias_f16_gpu(x, w, b):
    """x @ w + b (b f16[N])."""
    return _gemm("gemm_w4_bias_f16_gpu", x, w, extra=(b, 1, "b"))


def gemm_w4_add_f16_gpu(x, w, res):
    """res + x @ w (res f16[M, N])."""
    return _gemm("gemm_w4_add_f16_gpu", x, w, extra=(res, 2, "res"))


def gemm_w4_swiglu_f16_gpu(x, gate, up):
    """silu(x @ gate) * (x @ up) -> f16[M, N]; both weights of one shape and group."""
    return _gemm("gemm_w4_swiglu_f16_gpu", x, gate, up)


def lm_head_w4_f16_gpu(x, w):
    """Logits x @ w -> f32[M, V] of every row (w: the table f16[V, D] packed with nt=True)."""
    return _gemm("lm_head_w4_f16_gpu", x, w, dtype=_F32)


def _normed(name, x, g, w, w2, eps, dtype=_F16):
    """rmsnorm(x, g) in front of a product: inside it for one row, else by rmsnorm_f16_gpu; the same bits."""
    from .f16_gpu import rmsnorm_f16_gpu

    if _arg(x, _F16, 2, "x").shape[0] == 1:
        return _gemm("rmsnorm_" + name, x, w, w2, norm=(g, eps), dtype=dtype)
    return _gemm(name, rmsnorm_f16_gpu(x, g, eps), w, w2, dtype=dtype)


def rmsnorm_gemm_w4_f16_gpu(x, g, w, eps=1e-6):
    """gemm_w4(rmsnorm(x, g), w)."""
    return _normed("gemm_w4_f16_gpu", x, g, w, None, eps)


def rmsnorm_gemm_w4_swiglu_f16_gpu(x, g, gate, up, eps=1e-6):
    """gemm_w4_swiglu(rmsnorm(x, g), gate, up)."""
    return _normed("gemm_w4_swiglu_f16_gpu", x, g, gate, up, eps)


def rmsnorm_lm_head_w4_f16_gpu(x, g, w, eps=1e-6):
    """lm_head_w4(rmsnorm(x, g), w) -> f32[M, V]."""
    return _normed("lm_head_w4_f16_gpu", x, g, w, None, eps, dtype=_F32)


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
    if not (isinstance(kv, Tensor) and kv.t.dtype is _U8 and kv.t.dim() and kv.t.shape[-1] > 0
            and kv.t.shape[-1] % (32 * ROW) == 0):
        raise OpError("a 4-bit cache is u8[..., 72 P] with P a multiple of 32")
    return kv.t.shape[-1] // ROW


def _kv(kv, pos):
    """(cache u8[B, 2, kvh, 72 P], pos i64[B]) as torch tensors."""
    kt, pt = _arg(kv, _U8, 4, "kv"), _arg(pos, _I64, 1, "pos")
    b, two, kvh, row = kt.shape
    if b <= 0 or two != 2 or kvh <= 0 or row <= 0 or row % (32 * ROW):
        raise OpError("kv must be u8[B, 2, kvh, 72 P], P a multiple of 32")
    if pt.shape[0] != b:
        raise OpError("pos must be i64[B]")
    return kt, pt


def _rows(x, b, what):
    t = _arg(x, _F16, 2, what)
    if t.shape[0] % b:
        raise OpError(f"{what} must have B T rows")
    return t


def kv4_write_f16_gpu(kv, k, v, pos):
    """Rows pos[b] .. pos[b] + T - 1 of sequence b = k, v f16[B T, kvh 128], quantised (kv in place); rows outside the cache
    are dropped. A row whose key or value is not finite makes every query that sees it NaN."""
    kt, pt = _kv(kv, pos)
    key, val = _rows(k, kt.shape[0], "k"), _arg(v, _F16, 2, "v")
    if val.shape != key.shape or key.shape[1] != HD * kt.shape[2]:
        raise OpError("k, v must be f16[B T, kvh 128]")
    b, two, kvh, row = kt.shape
    rows, width = key.shape
    _run("kv4_write_f16_gpu", (kt.data_ptr(), key.data_ptr(), val.data_ptr(), pt.data_ptr()),
         (b, two, kvh, row, rows, width, rows, width, b))


def qknorm_rope_kv4_f16_gpu(qkv, qg, kg, pos, kv, eps=1e-6, theta=1e6):
    """QK-norm + RoPE + cache write: qkv f16[B T, (qh + 2 kvh) 128] (q | k | v), row i of sequence b at position pos[b] + i.
    Returns q = rope(rmsnorm_heads(q, qg)) f16[B T, qh 128] and writes k = rope(rmsnorm_heads(k, kg)) and v as
    kv4_write does."""
    kt, pt = _kv(kv, pos)
    x = _rows(qkv, kt.shape[0], "qkv")
    gains = [_arg(g, _F16, 1, "qg, kg") for g in (qg, kg)]
    if any(g.shape[0] != HD for g in gains):
        raise OpError("qg and kg must be f16[128]")
    dq = x.shape[1] - 2 * kt.shape[2] * HD
    if dq <= 0 or dq % HD:
        raise OpError("qkv must be f16[B T, (qh + 2 kvh) 128]")
    q = _empty((x.shape[0], dq))
    _call("qknorm_rope_kv4_f16_gpu", [x, *gains, pt, kt, q], (), (float(eps), float(theta)))
    return Tensor(q)


def kv4_read_f16_gpu(kv):
    """The values that a cache (or any u8[..., 72 P] part of one) holds: f16[..., P, 128]."""
    cap = kv4_capacity(kv)
    kt = _arg(kv, _U8, kv.t.dim(), "kv")
    out = kt.new_empty((*kt.shape[:-1], cap, HD), dtype=_F16)
    blocks = kt.numel() // (ROW * cap)
    _run("kv4_read_f16_gpu", (kt.data_ptr(), out.data_ptr()), (blocks, ROW * cap, blocks, cap, HD))
    return Tensor(out)


def attention_kv4_f16_gpu(q, kv, pos):
    """Causal attention over a 4-bit cache: query i of sequence b (row b T + i of q f16[B T, qh 128], position pos[b] + i)
    attends to rows 0 .. pos[b] + i of its kv head (already written); qh a multiple of the cache's kvh; scale
    1 / sqrt(128) -> f16[B T, qh 128]. A query whose position is outside the cache (with a negative pos[b], every query of
    the sequence) gives NaN and a device error."""
    kt, pt = _kv(kv, pos)
    b, _, kvh, row = kt.shape
    qt = _rows(q, b, "q")
    rows, width = qt.shape
    if width <= 0 or width % (HD * kvh):
        raise OpError("q must be f16[B T, qh 128], qh a multiple of kvh")
    need = _attention_bytes(b, rows // b, width // HD, kvh, row // ROW)
    out = qt.new_empty((rows, width))
    words = -(-need // 4)
    work = qt.new_empty((words,), dtype=_F32) if need else _NO_WORK
    _run("attention_kv4_f16_gpu", (qt.data_ptr(), kt.data_ptr(), pt.data_ptr(), out.data_ptr(), work.data_ptr()),
         (rows, width, b, 2, kvh, row, b, rows, width, words))
    return Tensor(out)


def kv4_reorder_gpu(kv, parents, n):
    """Beam search: rows 0 .. n - 1 of sequence b of kv u8[L, B, 2, kvh, 72 P] become those of sequence parents[b], in
    place (parents i64[B], n i64[1]; B <= 32, L kvh <= 32767). A parent out of range gives NaN rows and a device error."""
    kt, pt, nt = _arg(kv, _U8, 5, "kv"), _arg(parents, _I64, 1, "parents"), _arg(n, _I64, 1, "n")
    layers, b, two, kvh, row = kt.shape
    if two != 2 or not 0 < b <= 32 or layers <= 0 or kvh <= 0 or row <= 0 or row % (32 * ROW):
        raise OpError("kv must be u8[L, B, 2, kvh, 72 P] with B <= 32, P a multiple of 32")
    if layers * kvh > 32767:
        raise OpError("L kvh must be at most 32767")
    if pt.shape[0] != b or nt.shape[0] != 1:
        raise OpError("parents must be i64[B], n i64[1]")
    _run("kv4_reorder_gpu", (kt.data_ptr(), pt.data_ptr(), nt.data_ptr()), (layers, b, two, kvh, row, b, 1))


__all__ = [n for n in dir() if n.endswith(("_f16_gpu", "_reorder_gpu"))] + ["pack_w4", "PackedWeight4", "kv4_cache",
                                                                            "kv4_capacity"]
