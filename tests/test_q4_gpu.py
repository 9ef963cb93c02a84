"""4-bit serving (lk.ops.q4_gpu) and beam selection on the GPU against float64 definitions (oracle/q4.py).

Quantisation is exact: codes and scales, and so the values read back, must be equal. Tolerances of the others: one f16
rounding of the exact result (U = 2^-11 relative, half a subnormal step) plus an f32 term:
  product     2^-22 sqrt(K) sqrt(sum_k (x_k w_k)^2), f32 logits 2^-23 |ref| more; SwiGLU through its derivative (at most 1.1)
  attention   max|v| (2^-22 (8 + sqrt(P)) + 4 E), E the largest error of a score that its key's row gives: 2^-22 (sqrt(128)
              |q o k| / sqrt(128) + |score|); a weight is off by e^E - 1 and so is their sum
  beam score  2^-24 |ref| + 2^-24 (8 + |ref|): one f32 rounding, and the f32 exponentials in the log-sum
Beam tokens, parents and flags must be equal; their inputs keep candidates further apart than that, or equal."""
import numpy as np
import pytest
import torch

from lokinfer_amd._lib import LokinferError, check_device_errors
from lokinfer_amd.ops import OpError

from oracle import q4 as O

pytestmark = pytest.mark.gpu

U, SUB = 2.0 ** -11, 2.0 ** -25


def G(lk, a):
    return lk.from_numpy(np.ascontiguousarray(a), device="gpu", copy=True)


def I(lk, *v):
    return G(lk, np.array(v, np.int64))


def close(got, ref, extra, what="", unit=U):
    got = np.asarray(got.numpy(), np.float64)
    ref = np.asarray(ref, np.float64)
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    assert np.isfinite(got).all(), f"{what}: non-finite output"
    off = np.abs(got - ref) - (unit * (1 + 2.0 ** -10) * np.abs(ref) + extra + SUB)
    assert (off <= 0).all(), (what, int((off > 0).sum()), off.max())


def rng_of(*key):
    return np.random.default_rng([hash(str(k)) & 0xFFFF if isinstance(k, str) else int(k) for k in key])


# ---- weights ----------------------------------------------------------------------------------------------------

def hard_weight(r, k, n):
    """Columns of very different sizes, among them zeros, subnormals, the largest f16, one sign only."""
    w = r.standard_normal((k, n)) * np.exp2(r.uniform(-18, 8, (1, n)))
    w[:, :: 7] = np.abs(w[:, :: 7])
    w[:, 1:: 11] = -np.abs(w[:, 1:: 11])
    w = w.astype(np.float16)
    if n > 4:
        w[:, 2] = 0
        w[:, 3] = np.float16(2.0 ** -24) * r.integers(-3, 4, k)
        w[: min(k, 8), 4] = [65504, -65504, 60000, -57000, 1, 0, -1, 7][: min(k, 8)]
    return w


@pytest.mark.parametrize("k,n,group", [(8, 1, 32), (40, 5, 32), (128, 16, 128), (200, 33, 64), (264, 50, 128), (1000, 19, 32)])
@pytest.mark.parametrize("nt", [False, True])
def test_quantize_is_exact(gpu, k, n, group, nt):
    lk, q4 = gpu, gpu.ops.q4_gpu
    w = hard_weight(rng_of(1, k, n, group), k, n)
    p = q4.pack_w4(w.T if nt else w, group=group, nt=nt)
    assert p.shape == (k, n)
    assert np.array_equal(q4.unpack_w4_f16_gpu(p).numpy().astype(np.float64), O.weight_values(w, group))
    # the same codes and scales given: the same weight
    pad = -k % group
    codes, s = O.quantize(np.concatenate([w, np.zeros((pad, n), np.float16)]).reshape(-1, group, n).transpose(0, 2, 1))
    again = q4.pack_w4(codes.transpose(0, 2, 1).reshape(-1, n)[:k].astype(np.uint8), s.astype(np.float16), group)
    assert np.array_equal(q4.unpack_w4_f16_gpu(again).numpy(), q4.unpack_w4_f16_gpu(p).numpy())


def test_groups_that_are_not_finite_become_nan(gpu):
    lk, q4 = gpu, gpu.ops.q4_gpu
    w = rng_of(2).standard_normal((96, 20)).astype(np.float16)
    w[40, 3], w[41, 7] = np.inf, np.nan
    v = q4.unpack_w4_f16_gpu(q4.pack_w4(w, group=32)).numpy()
    bad = np.zeros((96, 20), bool)
    bad[32:64, 3] = bad[32:64, 7] = True
    assert np.isnan(v[bad]).all() and np.isfinite(v[~bad]).all()


def product(x, w):
    x = np.asarray(x, np.float64)
    return x @ w, 2.0 ** -22 * np.sqrt(x.shape[1]) * np.sqrt((x * x) @ (w * w))


def test_scales_that_do_not_fit_are_refused(gpu):
    """Every f16 as a scale, and codes over 15."""
    lk, q4 = gpu, gpu.ops.q4_gpu
    every = np.arange(0x10000, dtype=np.uint32).astype(np.uint16).view(np.float16)

    def fits(h):
        if not (0 <= h <= 8128) or np.signbit(h):
            return False
        m = int(float(h) * 2.0 ** 24)
        return (m & -m) * 256 > m or m == 0

    want = np.array([fits(h) for h in every])
    codes = np.full((32, int(want.sum())), 9, np.uint8)
    p = q4.pack_w4(codes, every[want][None, :], 32)
    assert np.array_equal(q4.unpack_w4_f16_gpu(p).numpy(), np.repeat(every[want][None, :], 32, 0))
    one = np.full((32, 1), 9, np.uint8)
    for h in np.concatenate([every[~want][::199], np.float16([8192, -1, np.nan, np.inf, 1 + 2.0 ** -8, 2.0 ** -15 * (1 + 2.0 ** -8)])]):
        with pytest.raises(OpError, match="scales"):
            q4.pack_w4(one, np.array([[h]], np.float16), 32)
    codes = np.zeros((200, 70), np.uint8)
    codes[199, 69] = 16
    with pytest.raises(OpError, match="codes"):
        q4.pack_w4(codes, np.ones((2, 70), np.float16), 128)


W4_CASES = [(1, 2048, 4096, 64), (1, 8, 1, 32), (1, 136, 17, 128), (1, 6144, 48, 128), (2, 2048, 96, 64), (4, 72, 40, 32),
            (5, 1000, 777, 32), (16, 264, 33, 64), (17, 2048, 31, 128), (33, 512, 65, 32), (64, 640, 200, 64),
            (65, 520, 200, 128), (100, 200, 300, 32), (130, 1032, 130, 64), (257, 2048, 96, 32), (409, 384, 515, 128),
            (1030, 136, 260, 64),
            # many columns: weights streamed by persistent waves, x in LDS; 2048 x 16 rows of it are more than 64 KiB
            (1, 264, 32770, 64), (3, 40, 24600, 32), (7, 136, 25000, 128), (16, 2048, 24583, 128),
            # few rows, many columns: tiles, not streamed (x is too long for LDS, or not enough columns for it)
            (6, 200, 22000, 64), (16, 520, 8200, 32), (13, 5128, 24580, 128),
            # tiles of 32 x 64, 64 x 64 and 128 x 256
            (17, 4104, 70, 32), (40, 6152, 200, 64), (100, 2184, 515, 128), (20, 72, 8200, 32), (405, 2056, 2050, 64),
            (450, 3080, 1990, 128), (450, 3080, 1990, 32), (1025, 264, 2100, 32), (700, 1032, 4100, 128), (700, 1032, 4100, 64)]


@pytest.mark.parametrize("m,k,n,group", W4_CASES)
def test_products(gpu, m, k, n, group):
    lk, q4 = gpu, gpu.ops.q4_gpu
    r = rng_of(3, m, k, n)
    x = r.standard_normal((m, k)).astype(np.float16)
    x[:, : min(k, 3)] *= 100  # a few large channels
    w = (r.standard_normal((k, n)) / np.sqrt(k)).astype(np.float16)
    p = q4.pack_w4(w, group=group)
    v = O.weight_values(w, group)
    ref, term = product(x, v)
    gx = G(lk, x)
    close(q4.gemm_w4_f16_gpu(gx, p), ref, term, "gemm")
    close(q4.lm_head_w4_f16_gpu(gx, p), ref, term, "logits", unit=2.0 ** -23)
    b, res = r.standard_normal(n).astype(np.float16), r.standard_normal((m, n)).astype(np.float16)
    close(q4.gemm_w4_bias_f16_gpu(gx, p, G(lk, b)), ref + b, term + 2.0 ** -23 * np.abs(ref + b), "bias")
    close(q4.gemm_w4_add_f16_gpu(gx, p, G(lk, res)), ref + res, term + 2.0 ** -23 * np.abs(ref + res), "add")
    u = (r.standard_normal((k, n)) / np.sqrt(k)).astype(np.float16)
    up, upTerm = product(x, O.weight_values(u, group))
    silu = ref / (1 + np.exp(-ref))
    close(q4.gemm_w4_swiglu_f16_gpu(gx, p, q4.pack_w4(u, group=group)), silu * up,
          1.1 * np.abs(up) * term + np.abs(silu) * upTerm + 2.0 ** -20 * np.abs(silu * up), "swiglu")


def test_no_rows_give_no_rows(gpu):
    lk, q4 = gpu, gpu.ops.q4_gpu
    p = q4.pack_w4(np.ones((64, 20), np.float16), group=32)
    assert q4.gemm_w4_f16_gpu(G(lk, np.zeros((0, 64), np.float16)), p).shape == (0, 20)


@pytest.mark.parametrize("m,k,n", [(1, 2048, 112), (4, 2048, 112), (70, 2048, 112), (1, 6144, 40), (1, 520, 33000)])
def test_rmsnorm_in_front_is_the_norm_and_the_product(gpu, m, k, n):
    lk, q4, F = gpu, gpu.ops.q4_gpu, gpu.ops.f16_gpu
    r = rng_of(4, m)
    x, g = G(lk, r.standard_normal((m, k)).astype(np.float16)), G(lk, (1 + r.standard_normal(k) / 9).astype(np.float16))
    a, b = (q4.pack_w4((r.standard_normal((k, n)) / 45).astype(np.float16)) for _ in range(2))
    h = F.rmsnorm_f16_gpu(x, g)
    assert np.array_equal(q4.rmsnorm_gemm_w4_f16_gpu(x, g, a).numpy(), q4.gemm_w4_f16_gpu(h, a).numpy())
    assert np.array_equal(q4.rmsnorm_gemm_w4_swiglu_f16_gpu(x, g, a, b).numpy(), q4.gemm_w4_swiglu_f16_gpu(h, a, b).numpy())
    assert np.array_equal(q4.rmsnorm_lm_head_w4_f16_gpu(x, g, a).numpy(), q4.lm_head_w4_f16_gpu(h, a).numpy())


def test_rows_do_not_depend_on_their_neighbours(gpu):
    """A row with infinities or NaN leaves the others as they are; an infinite activation gives what f16 weights would."""
    lk, q4 = gpu, gpu.ops.q4_gpu
    r = rng_of(5)
    for m in (3, 20, 80):
        x = r.standard_normal((m, 256)).astype(np.float16)
        p = q4.pack_w4((r.standard_normal((256, 40)) / 16).astype(np.float16), group=32)
        clean = q4.gemm_w4_f16_gpu(G(lk, x), p).numpy()
        x[1, 5], x[2] = np.inf, np.nan
        got = q4.gemm_w4_f16_gpu(G(lk, x), p).numpy()
        assert np.array_equal(np.delete(got, [1, 2], 0), np.delete(clean, [1, 2], 0))
        assert np.isnan(got[2]).all()
        w5 = q4.unpack_w4_f16_gpu(p).numpy()[5]
        assert np.array_equal(np.isnan(got[1]), w5 == 0) and (np.sign(got[1][w5 != 0]) == np.sign(w5[w5 != 0])).all()
        assert np.isinf(got[1][w5 != 0]).all()


def test_weight_op_refusals(gpu):
    lk, q4 = gpu, gpu.ops.q4_gpu
    p = q4.pack_w4(np.ones((64, 20), np.float16), group=32)
    p2 = q4.pack_w4(np.ones((64, 20), np.float16), group=64)
    x = G(lk, np.zeros((2, 64), np.float16))
    for bad in (lambda: q4.pack_w4(np.ones((64, 20), np.float16), group=16),
                lambda: q4.gemm_w4_f16_gpu(G(lk, np.zeros((2, 72), np.float16)), p),
                lambda: q4.gemm_w4_f16_gpu(G(lk, np.zeros((2, 64), np.float32)), p),
                lambda: q4.gemm_w4_f16_gpu(x, x),
                lambda: q4.gemm_w4_swiglu_f16_gpu(x, p, p2),
                lambda: q4.gemm_w4_bias_f16_gpu(x, p, G(lk, np.zeros(21, np.float16))),
                lambda: q4.gemm_w4_add_f16_gpu(x, p, G(lk, np.zeros((1, 20), np.float16))),
                lambda: q4.rmsnorm_gemm_w4_f16_gpu(x, G(lk, np.zeros(63, np.float16)), p),
                lambda: q4.pack_w4(np.full((64, 4), 16, np.uint8), np.ones((2, 4), np.float16), 32),
                lambda: q4.pack_w4(np.full((64, 4), 1, np.uint8), np.full((2, 4), 1 + 2.0 ** -9, np.float16), 32),
                lambda: q4.pack_w4(np.full((64, 4), 1, np.uint8), np.ones((1, 4), np.float16), 32)):
        with pytest.raises(OpError):
            bad()
    # K that is no multiple of 8, and a row that starts off 16 bytes
    with pytest.raises(OpError):
        q4.gemm_w4_f16_gpu(G(lk, np.zeros((2, 60), np.float16)), q4.pack_w4(np.ones((60, 20), np.float16), group=32))
    off = lk.Tensor(torch.zeros(129, dtype=torch.float16, device="cuda")[1:].view(2, 64))
    with pytest.raises(LokinferError, match="aligned"):
        q4.gemm_w4_f16_gpu(off, p)


# ---- caches -----------------------------------------------------------------------------------------------------

def rows_of(r, n, kvh, hard=False):
    k = r.standard_normal((n, kvh * 128)) * np.exp(0.5 * r.standard_normal(kvh * 128))
    v = r.standard_normal((n, kvh * 128))
    if hard:
        k[:, ::5] *= 2.0 ** -20
        k[:, 32:64] = 0
        v *= np.exp2(r.uniform(-26, 8, (n, 1)))
    return k.astype(np.float16), v.astype(np.float16)


@pytest.mark.parametrize("b,t,kvh,cap,pos", [(1, 1, 1, 32, [0]), (1, 70, 2, 96, [5]), (3, 1, 8, 64, [0, 63, 17]),
                                             (2, 9, 4, 64, [60, -4])])
def test_cache_rows_are_exact_and_the_others_stay(gpu, b, t, kvh, cap, pos):
    lk, q4 = gpu, gpu.ops.q4_gpu
    r = rng_of(6, b, t, kvh)
    kv = q4.kv4_cache(b, kvh, cap)
    kv.t.random_(0, 256, generator=torch.Generator(device="cuda").manual_seed(3))
    before = kv.t.cpu().numpy()
    k, v = rows_of(r, b * t, kvh, hard=True)
    q4.kv4_write_f16_gpu(kv, G(lk, k), G(lk, v), I(lk, *pos))
    after, read = kv.t.cpu().numpy(), q4.kv4_read_f16_gpu(kv).numpy().astype(np.float64)
    key, val = O.cache_values(k, v, kvh)
    touched = np.zeros((b, cap), bool)
    for s in range(b):
        for i in range(t):
            row = pos[s] + i
            if not 0 <= row < cap:
                continue
            touched[s, row] = True
            assert np.array_equal(read[s, 0, :, row], key[s * t + i]) and np.array_equal(read[s, 1, :, row], val[s * t + i])
    for s in range(b):  # rows that the call does not name keep every byte
        codes = lambda x: x[s, :, :, : 64 * cap].reshape(2, kvh, cap, 64)[:, :, ~touched[s]]  # noqa: E731
        scales = lambda x: x[s, :, :, 64 * cap:].reshape(2, kvh, 4, cap, 2)[:, :, :, ~touched[s]]   # noqa: E731
        assert np.array_equal(codes(before), codes(after)) and np.array_equal(scales(before), scales(after))


def filled(lk, r, b, kvh, cap, rows, hard=False):
    """A cache whose first rows[s] rows are written, the rest garbage bytes; (kv, keys, values as held)."""
    q4 = lk.ops.q4_gpu
    kv = q4.kv4_cache(b, kvh, cap)
    kv.t.random_(0, 256, generator=torch.Generator(device="cuda").manual_seed(7))
    held = []
    for s in range(b):
        k, v = rows_of(r, rows[s], kvh, hard)
        q4.kv4_write_f16_gpu(lk.Tensor(kv.t[s:s + 1]), G(lk, k), G(lk, v), I(lk, 0))
        held.append(O.cache_values(k, v, kvh))
    return kv, held


ATTN = [  # b, t, qh, kvh, cap, pos
    (1, 1, 1, 1, 32, [0]), (1, 1, 16, 8, 448, [416]), (1, 1, 16, 8, 448, [63]), (1, 1, 8, 8, 96, [64]),
    (5, 1, 16, 8, 320, [0, 319, 64, 127, 200]), (2, 1, 12, 4, 160, [33, 128]), (3, 1, 32, 2, 128, [7, 100, 31]),
    (1, 1, 7, 7, 64, [40]), (1, 1, 64, 1, 96, [90]), (1, 1, 4, 2, 8192, [8000]),
    (1, 2, 16, 8, 64, [0]), (1, 5, 6, 2, 96, [61]), (2, 3, 4, 4, 64, [61, 0]), (1, 33, 4, 2, 96, [0]),
    (1, 64, 8, 2, 128, [64]), (2, 70, 4, 2, 160, [0, 83]), (1, 100, 3, 3, 128, [27]), (1, 129, 16, 8, 512, [300]),
    (1, 40, 16, 1, 64, [20]),
    # key ranges over workgroups, most of them empty; rows past 16 a kv head
    (1, 1, 4, 2, 8192, [5]), (3, 1, 16, 8, 4096, [0, 4095, 64]), (1, 3, 24, 2, 4096, [2500]), (2, 20, 4, 2, 2080, [2060, 30]),
    # more rows: 4 waves a workgroup; 32 rows of 8 waves over a longer cache; 32 rows of 4 waves
    (2, 150, 16, 8, 512, [0, 361]), (1, 300, 16, 8, 2112, [1801]), (2, 401, 16, 8, 448, [0, 40]), (1, 165, 32, 4, 192, [20]),
]


@pytest.mark.parametrize("b,t,qh,kvh,cap,pos", ATTN)
def test_attention(gpu, b, t, qh, kvh, cap, pos):
    lk, q4 = gpu, gpu.ops.q4_gpu
    r = rng_of(8, b, t, qh, cap)
    kv, held = filled(lk, r, b, kvh, cap, [p + t for p in pos])
    q = (r.standard_normal((b * t, qh * 128)) * np.exp(0.3 * r.standard_normal((1, qh * 128)))).astype(np.float16)
    got = q4.attention_kv4_f16_gpu(G(lk, q), kv, I(lk, *pos))
    ref, extra = [], []
    for s in range(b):
        key, val = held[s]
        o, term = O.attention(q[s * t:(s + 1) * t].reshape(t, qh, 128), key, val, pos[s])
        top = np.abs(val).max()
        ref.append(o.reshape(t, -1))
        extra.append(np.repeat(top * (2.0 ** -22 * (8 + np.sqrt(cap)) + 4 * 2.0 ** -22 * term), 128, 1))
    close(got, np.concatenate(ref), np.concatenate(extra), "attention")
    check_device_errors()


@pytest.mark.parametrize("t", [1, 40])
def test_large_scores_and_one_key_taking_all(gpu, t):
    lk, q4 = gpu, gpu.ops.q4_gpu
    r = rng_of(9, t)
    kv, held = filled(lk, r, 1, 2, 128, [100])
    q = (40 * r.standard_normal((t, 4 * 128))).astype(np.float16)
    got = q4.attention_kv4_f16_gpu(G(lk, q), kv, I(lk, 100 - t))
    o, term = O.attention(q.reshape(t, 4, 128), *held[0], 100 - t)
    top = np.abs(held[0][1]).max()
    close(got, o.reshape(t, -1), np.repeat(top * (2.0 ** -22 * (8 + np.sqrt(128)) + 4 * 2.0 ** -22 * term), 128, 1))


@pytest.mark.parametrize("t,qh,kvh", [(1, 4, 2), (1, 16, 1), (48, 4, 2), (89, 64, 8), (90, 128, 16)])
def test_rows_that_are_not_finite_reach_only_queries_that_see_them(gpu, t, qh, kvh):
    lk, q4 = gpu, gpu.ops.q4_gpu
    r = rng_of(10, t, qh)
    n = 90
    k, v = rows_of(r, n, kvh)
    q = r.standard_normal((t, qh * 128)).astype(np.float16)

    def attend(k, v, first):
        kv = q4.kv4_cache(1, kvh, 96)
        q4.kv4_write_f16_gpu(kv, G(lk, k), G(lk, v), I(lk, 0))
        return q4.attention_kv4_f16_gpu(G(lk, q), kv, I(lk, first)).numpy()

    first = n - t if t > 1 else 60
    clean = attend(k, v, first)
    bad = first + t // 2 + 1  # seen by the queries after it only (t = 1: by none)
    for x in (np.nan, np.inf, -np.inf):
        for which in (0, 1):
            kk, vv = k.copy(), v.copy()
            (kk, vv)[which][bad, 3] = x  # head 0
            got = attend(kk, vv, first)
            seen = np.zeros((t, qh * 128), bool)
            seen[bad - first:, : (qh // kvh) * 128] = True
            assert np.isnan(got[seen]).all()
            assert np.array_equal(got[~seen], clean[~seen])


def test_positions_outside_the_cache_are_nan_and_reported(gpu):
    lk, q4 = gpu, gpu.ops.q4_gpu
    r = rng_of(11)
    check_device_errors()
    for t in (1, 5, 40):
        kv, _ = filled(lk, r, 3, 2, 64, [64, 64, 64])
        q = G(lk, r.standard_normal((3 * t, 4 * 128)).astype(np.float16))
        want = q4.attention_kv4_f16_gpu(q, kv, I(lk, 64 - t, 20, 64 - t)).numpy()
        got = q4.attention_kv4_f16_gpu(q, kv, I(lk, 65 - t, 20, -1)).t.cpu().numpy()
        with pytest.raises(LokinferError, match="position"):
            check_device_errors()
        assert np.isnan(got[t - 1]).all() and np.isfinite(got[: t - 1]).all()  # the last query of sequence 0
        assert np.array_equal(got[t:2 * t], want[t:2 * t])
        assert np.isnan(got[2 * t:]).all()
        got = q4.attention_kv4_f16_gpu(q, kv, I(lk, 2 ** 63 - 1, 20, 2 ** 63 - t)).t.cpu().numpy()
        with pytest.raises(LokinferError, match="position"):
            check_device_errors()
        assert np.isnan(got[: t]).all() and np.isnan(got[2 * t:]).all() and np.array_equal(got[t:2 * t], want[t:2 * t])


def test_qknorm_rope_is_the_f16_ops(gpu):
    """q as rmsnorm_heads and rope give it, keys likewise before they are quantised; each sequence at its own position."""
    lk, q4, F = gpu, gpu.ops.q4_gpu, gpu.ops.f16_gpu
    r = rng_of(12)
    for b, t, qh, kvh, cap, pos in ((1, 1, 16, 8, 64, [40]), (3, 1, 4, 2, 32, [0, 31, 9]), (2, 7, 2, 2, 64, [3, 57])):
        qkv = r.standard_normal((b * t, (qh + 2 * kvh) * 128)).astype(np.float16)
        qg, kg = (G(lk, (1 + r.standard_normal(128) / 9).astype(np.float16)) for _ in range(2))
        kv = q4.kv4_cache(b, kvh, cap)
        got = q4.qknorm_rope_kv4_f16_gpu(G(lk, qkv), qg, kg, I(lk, *pos), kv).numpy()
        want = q4.kv4_cache(b, kvh, cap)
        for s in range(b):
            x = qkv[s * t:(s + 1) * t]
            p = I(lk, pos[s])
            q = F.rope_f16_gpu(F.rmsnorm_heads_f16_gpu(G(lk, x[:, : qh * 128]), qg), p)
            k = F.rope_f16_gpu(F.rmsnorm_heads_f16_gpu(G(lk, x[:, qh * 128:(qh + kvh) * 128]), kg), p)
            assert np.array_equal(got[s * t:(s + 1) * t], q.numpy())
            q4.kv4_write_f16_gpu(lk.Tensor(want.t[s:s + 1]), k, G(lk, x[:, (qh + kvh) * 128:]), p)
        assert np.array_equal(kv.t.cpu().numpy(), want.t.cpu().numpy())


@pytest.mark.parametrize("parents", [[0, 1, 2, 3], [0, 0, 0, 0], [3, 2, 1, 0], [1, 2, 3, 0], [2, 2, 0, 3]])
@pytest.mark.parametrize("n", [0, 1, 37, 64])
def test_reorder(gpu, parents, n):
    lk, q4 = gpu, gpu.ops.q4_gpu
    kv = q4.kv4_cache(4, 2, 64, layers=3)
    kv.t.random_(0, 256, generator=torch.Generator(device="cuda").manual_seed(n))
    was = kv.t.cpu().numpy()
    q4.kv4_reorder_gpu(kv, I(lk, *parents), I(lk, n))
    want = was.copy()
    want[..., : n * 64] = was[:, parents, ..., : n * 64]
    for g in range(4):
        at = slice(64 * 64 + g * 2 * 64, 64 * 64 + g * 2 * 64 + 2 * n)
        want[..., at] = was[:, parents, ..., at]
    assert np.array_equal(kv.t.cpu().numpy(), want)


def test_reorder_of_32_and_of_a_parent_that_is_not_there(gpu):
    lk, q4 = gpu, gpu.ops.q4_gpu
    check_device_errors()
    kv = q4.kv4_cache(32, 1, 32, layers=1)
    kv.t.random_(0, 256, generator=torch.Generator(device="cuda").manual_seed(5))
    was = kv.t.cpu().numpy()
    parents = np.random.default_rng(5).integers(0, 32, 32)
    q4.kv4_reorder_gpu(kv, G(lk, parents), I(lk, 32))
    assert np.array_equal(kv.t.cpu().numpy(), was[:, parents])
    kv = q4.kv4_cache(2, 1, 32, layers=1)
    q4.kv4_reorder_gpu(kv, I(lk, 2, 0), I(lk, 9))
    with pytest.raises(LokinferError, match="index"):
        check_device_errors()
    v = q4.kv4_read_f16_gpu(kv).t.cpu().numpy()
    assert np.isnan(v[0, 0, :, :, :9]).all() and (v[0, 0, :, :, 9:] == 0).all() and (v[0, 1] == 0).all()


def test_cache_op_refusals(gpu):
    lk, q4 = gpu, gpu.ops.q4_gpu
    kv, pos = q4.kv4_cache(2, 2, 32), I(lk, 0, 0)
    h = lambda *s: G(lk, np.zeros(s, np.float16))  # noqa: E731
    for bad in (lambda: q4.attention_kv4_f16_gpu(h(3, 256), kv, pos), lambda: q4.attention_kv4_f16_gpu(h(2, 384), kv, pos),
                lambda: q4.attention_kv4_f16_gpu(h(2, 256), kv, I(lk, 0)),
                lambda: q4.attention_kv4_f16_gpu(G(lk, np.zeros((2, 256), np.float32)), kv, pos),
                lambda: q4.kv4_write_f16_gpu(kv, h(2, 256), h(2, 128), pos),
                lambda: q4.kv4_write_f16_gpu(kv, h(2, 128), h(2, 128), pos),
                lambda: q4.qknorm_rope_kv4_f16_gpu(h(2, 512), h(128), h(128), pos, kv),
                lambda: q4.qknorm_rope_kv4_f16_gpu(h(2, 640), h(64), h(128), pos, kv),
                lambda: q4.kv4_reorder_gpu(kv, pos, I(lk, 1)), lambda: q4.kv4_cache(0, 1, 1),
                lambda: q4.kv4_reorder_gpu(q4.kv4_cache(33, 1, 32, layers=1), G(lk, np.arange(33)), I(lk, 1))):
        with pytest.raises(OpError):
            bad()


# ---- beam selection -----------------------------------------------------------------------------------------------

def select(lk, logits, scores, done, k, eos):
    return lk.ops.beam_select_f32_gpu(G(lk, logits), G(lk, scores), G(lk, np.asarray(done, np.int64)), k, eos)


def same_choice(lk, logits, scores, done, k, eos):
    got = [x.numpy() for x in select(lk, logits, scores, done, k, eos)]
    ref = O.beam_select(logits, scores, done, k, eos)
    for a, b in zip(got[1:], ref[1:]):
        assert np.array_equal(a, b), (a, b)
    assert np.array_equal(np.isinf(got[0]), np.isinf(ref[0]))
    fin = np.isfinite(ref[0])
    assert (np.abs(got[0][fin] - ref[0][fin]) <= 2.0 ** -24 * np.abs(ref[0][fin]) + 2.0 ** -24 * (8 + np.abs(ref[0][fin]))).all()


@pytest.mark.parametrize("b,v,k", [(1, 1, 1), (1, 5, 5), (4, 3, 12), (2, 64, 2), (1, 1000, 32), (4, 1024, 4), (4, 1025, 8),
                                   (32, 2000, 32), (4, 151936, 4), (8, 50257, 16), (2, 262144, 7)])
def test_selection(gpu, b, v, k):
    r = rng_of(20, b, v, k)
    logits = (3 * r.standard_normal((b, v))).astype(np.float32)
    scores = (-5 * r.random(b)).astype(np.float32)
    same_choice(gpu, logits, scores, np.zeros(b), k, [v - 1])
    done = (np.arange(b) % 3 == 1).astype(np.int64)
    if b > 1:
        same_choice(gpu, logits, scores, done, k, sorted({0, v // 2, v - 1}))


def test_ties_go_to_the_lowest_index(gpu):
    r = rng_of(21)
    row = r.integers(-3, 4, 5000).astype(np.float32)  # whole numbers: many equal logits
    row[4000] = -0.0
    same_choice(gpu, np.stack([row, row, row]), np.float32([-1, -1, -1]), [0, 0, 0], 32, [7])
    same_choice(gpu, np.zeros((3, 3000), np.float32), np.zeros(3, np.float32), [0, 0, 0], 20, [7])
    same_choice(gpu, np.zeros((2, 5), np.float32), np.float32([-2, -1]), [0, 1], 10, [3])


def test_rows_without_a_value(gpu):
    r = rng_of(22)
    x = r.standard_normal((6, 3000)).astype(np.float32)
    lowest = np.finfo(np.float32).min
    x[0, :] = -np.inf
    x[1, 17] = np.nan
    x[2, 9] = np.inf
    x[3, 10:] = -np.inf
    x[4, 5:] = lowest
    for k in (1, 15, 32):
        same_choice(gpu, x, np.float32([-1, -2, -1, -4, -5, -3]), [0, 0, 0, 0, 0, 0], k, [2999])
    same_choice(gpu, x[:3], np.float32([-1, -2, -1]), [0, 0, 0], 32, [2999])          # nothing has a value
    same_choice(gpu, x[3:], np.float32([-np.inf, np.nan, -3]), [0, 0, 1], 32, [1])    # nor has a beam without a score
    same_choice(gpu, x[3:], np.float32([-1, np.inf, -3]), [1, 1, 1], 8, [2, 1])       # all ended
    same_choice(gpu, np.full((2, 700), lowest, np.float32), np.float32([-1, -1]), [0, 0], 9, [3])


def test_selection_refusals(gpu):
    lk = gpu
    x, s, d = np.zeros((2, 10), np.float32), np.zeros(2, np.float32), [0, 0]
    for bad in (lambda: select(lk, x, s, d, 0, [1]), lambda: select(lk, x, s, d, 21, [1]), lambda: select(lk, x, s, d, 2, [10]),
                lambda: select(lk, x, s, d, 2, []), lambda: select(lk, x, s, d, 2, [1, 2, 3, 4, 5]),
                lambda: select(lk, x, s[:1], d, 2, [1]), lambda: select(lk, np.zeros((33, 10), np.float32), np.zeros(33, np.float32), [0] * 33, 2, [1])):
        with pytest.raises(OpError):
            bad()
