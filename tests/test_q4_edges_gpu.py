"""4-bit serving and beam selection on the GPU where a call's arguments meet: epilogues together, long flat tails of keys, values
that f16 holds as subnormals, weights used on other streams, candidates that 64 bits do not tell apart. Tolerances as in
test_q4_gpu, whose terms are repeated where they apply."""
import ctypes as C

import numpy as np
import pytest
import torch

from lokinfer_amd._lib import lib

from oracle import q4 as O

pytestmark = pytest.mark.gpu

U, SUB = 2.0 ** -11, 2.0 ** -25


def G(lk, a):
    return lk.from_numpy(np.ascontiguousarray(a), device="gpu", copy=True)


def I(lk, *v):
    return G(lk, np.array(v, np.int64))


def product(x, w):
    """x @ w and the f32 term of its tolerance."""
    x = np.asarray(x, np.float64)
    return x @ w, 2.0 ** -22 * np.sqrt(x.shape[1]) * np.sqrt((x * x) @ (w * w))


# one shape for each kernel a product can take: k split over 4 or 8 waves, streamed, 32 rows, tiles of 32 x 64, 64 x 64, 128 x 256
SHAPES = [(2, 264, 40, 32), (3, 4104, 64, 128), (3, 40, 24600, 32), (20, 264, 70, 64), (17, 4104, 70, 32), (405, 2056, 2050, 64),
          (700, 1032, 4100, 128)]


@pytest.mark.parametrize("m,k,n,group", SHAPES)
def test_bias_and_residual_together(gpu, m, k, n, group):
    """The C entry point takes both: (x @ w + bias) + res, whichever kernel runs."""
    lk, q4 = gpu, gpu.ops.q4_gpu
    r = np.random.default_rng([31, m, k, n])
    x = r.standard_normal((m, k)).astype(np.float16)
    w = (r.standard_normal((k, n)) / np.sqrt(k)).astype(np.float16)
    bias, res = r.standard_normal(n).astype(np.float16), r.standard_normal((m, n)).astype(np.float16)
    p = q4.pack_w4(w, group=group)
    gx, gb, gr = G(lk, x), G(lk, bias), G(lk, res)
    out = torch.zeros(m, n, dtype=torch.float16, device="cuda")
    at = [C.c_void_p(t.data_ptr()) for t in (gx.t, p.q.t, p.s.t, gb.t, gr.t, out)]
    call = lib().lk_hip_w4_gemm
    rc = call(at[0], None, at[1], at[2], None, None, at[3], at[4], at[5], C.c_int64(m), C.c_int64(n), C.c_int64(k),
              C.c_int(group), C.c_int(0), C.c_float(0.0), C.c_void_p(torch.cuda.current_stream().cuda_stream))
    assert rc == 0
    ref, term = product(x, O.weight_values(w, group))
    first, ref = ref + bias, ref + bias + res
    # two f32 sums behind the product, one rounding to f16
    off = np.abs(out.cpu().numpy().astype(np.float64) - ref)
    assert (off <= U * (1 + 2.0 ** -10) * np.abs(ref) + term + 2.0 ** -23 * (np.abs(first) + np.abs(ref)) + SUB).all()


@pytest.mark.parametrize("t,qh,kvh", [(48, 4, 2), (90, 128, 16)])
def test_a_row_does_not_depend_on_the_rows_beside_it(gpu, t, qh, kvh):
    """Where one row's running maximum grows, the sums of the others of its workgroup stay as they are: bit for bit."""
    lk, q4 = gpu, gpu.ops.q4_gpu
    r = np.random.default_rng([34, t, qh])
    n = 1000
    k, v = (r.standard_normal((n, kvh * 128)).astype(np.float16) for _ in range(2))
    k *= np.exp(r.standard_normal((n, 1))).astype(np.float16)  # maxima that grow along the keys
    kv = q4.kv4_cache(1, kvh, n)
    q4.kv4_write_f16_gpu(kv, G(lk, k), G(lk, v), I(lk, 0))
    q = r.standard_normal((t, qh * 128)).astype(np.float16)
    want = q4.attention_kv4_f16_gpu(G(lk, q), kv, I(lk, n - t)).numpy()
    other = q.copy()
    other[::2] *= 4
    got = q4.attention_kv4_f16_gpu(G(lk, other), kv, I(lk, n - t)).numpy()
    assert np.array_equal(got[1::2], want[1::2]) and not np.array_equal(got[::2], want[::2])


@pytest.mark.parametrize("t", [4096, 8192, 10400], ids=["16x8", "32x8", "32x4"])  # rows x waves of a workgroup
def test_few_keys_above_a_long_flat_tail(gpu, t):
    """One key of each wave 17.5 above a million equal others: each of these has a weight of 2^-25, all of them together 0.3%
    of the sum, and they alone have a value. The keys of a row lie in one workgroup."""
    lk, q4 = gpu, gpu.ops.q4_gpu
    cap = 1 << 20
    top = 64 * torch.arange(8, device="cuda")
    key, val = torch.zeros(cap, 128, dtype=torch.float16, device="cuda"), torch.full((cap, 128), 0.875, dtype=torch.float16, device="cuda")
    key[top], val[top] = 1.75, 0.0
    kv = q4.kv4_cache(1, 1, cap)
    q4.kv4_write_f16_gpu(kv, lk.Tensor(key), lk.Tensor(val), I(lk, 0))
    assert (q4.kv4_read_f16_gpu(kv).t[0, :, 0] == torch.stack([key, val])).all()  # exact in 4 bits
    q = np.float16(17.5 / (1.75 * np.sqrt(128)))
    got = q4.attention_kv4_f16_gpu(lk.Tensor(torch.full((t, 128), float(q), dtype=torch.float16, device="cuda")), kv, I(lk, cap - t))
    got = got.t.cpu().numpy().astype(np.float64)
    score = 128 * 1.75 * float(q) / np.sqrt(128)
    rest = (cap - t + np.arange(t) + 1 - 8)[:, None] * np.exp(-score)
    ref = 0.875 * rest / (8 + rest)
    # as in test_q4_gpu: E of a score of 128 equal products; a weight is held to 2^-37 of the largest
    e = 2.0 ** -22 * (np.sqrt(128) * score / np.sqrt(128) + score)
    extra = 0.875 * (2.0 ** -22 * (8 + np.sqrt(cap)) + 4 * e + cap * 2.0 ** -37)
    assert (np.abs(got - ref) <= U * (1 + 2.0 ** -10) * ref + extra).all(), (got.min(), got.max(), ref.min(), ref.max())


@pytest.mark.parametrize("t,cap", [(1, 320), (1, 4096), (33, 320), (300, 320), (401, 448)])
@pytest.mark.parametrize("size", [2.0, 600.0, 8000.0, 60000.0])
def test_scores_of_any_size(gpu, t, cap, size):
    """Keys of two sizes, so scores of two values: the larger ones' rows share the weight equally, also where f32 cannot tell
    the scores' neighbours apart any more (2^36 at 60000) and where all of them are negative."""
    lk, q4 = gpu, gpu.ops.q4_gpu
    r = np.random.default_rng([38, t, cap])
    n = cap - 7
    k, v = np.full((n, 256), 0.5 * size, np.float16), r.standard_normal((n, 256)).astype(np.float16)
    top = [3, 9]
    k[top] = size
    kv = q4.kv4_cache(1, 2, cap)
    q4.kv4_write_f16_gpu(kv, G(lk, k), G(lk, v), I(lk, 0))
    key, val = O.cache_values(k, v, 2)
    for sign in (1, -1):
        q = np.full((t, 4 * 128), sign * size, np.float16)
        got = q4.attention_kv4_f16_gpu(G(lk, q), kv, I(lk, n - t)).numpy().astype(np.float64).reshape(t, 4, 128)
        for i in (0, t // 2, t - 1):
            for h in range(4):
                seen = n - t + i + 1
                s = key[:seen, h // 2] @ q[i, h * 128:(h + 1) * 128].astype(np.float64) / np.sqrt(128)
                e = np.exp(s - s.max())
                ref = (e / e.sum()) @ val[:seen, h // 2]
                assert np.isfinite(got[i, h]).all(), (sign, i, h)
                # a weight next to the largest: all or none, or (size 2) scores of 45 at 2^-22
                assert (np.abs(got[i, h] - ref) <= U * (1 + 2.0 ** -10) * np.abs(ref) + np.abs(val).max() * 2.0 ** -22 *
                        (8 + np.sqrt(cap) + 4 * 2 * 46) + SUB).all(), (sign, i, h)


def test_codes_and_scales_of_other_types(gpu):
    """Values that u8 and f16 hold are taken whatever type they come in."""
    lk, q4 = gpu, gpu.ops.q4_gpu
    r = np.random.default_rng(35)
    codes, scales = r.integers(0, 16, (100, 20)), r.integers(1, 256, (4, 20)) * 2.0 ** -12
    want = ((codes - 8) * np.repeat(scales, 32, 0)[:100]).astype(np.float16)
    for c, s in ((np.uint8, np.float16), (np.int64, np.float32), (np.float32, np.float64)):
        assert np.array_equal(q4.unpack_w4_f16_gpu(q4.pack_w4(codes.astype(c), scales.astype(s), 32)).numpy(), want)
    assert np.array_equal(q4.unpack_w4_f16_gpu(q4.pack_w4(codes.tolist(), scales.tolist(), 32)).numpy(), want)


def test_weights_are_ready_on_any_stream(gpu, monkeypatch):
    """A weight laid out on one stream, where that takes long, is used at once on another."""
    lk, q4 = gpu, gpu.ops.q4_gpu
    w = np.random.default_rng(33).standard_normal((256, 96)).astype(np.float16)
    want = q4.unpack_w4_f16_gpu(q4.pack_w4(w)).numpy()
    quantize = q4.quantize_w4_f16_gpu

    def late(*args):
        torch.cuda._sleep(100_000_000)  # some 50 ms on the device
        return quantize(*args)

    monkeypatch.setattr(q4, "quantize_w4_f16_gpu", late)
    with torch.cuda.stream(torch.cuda.Stream()):
        p = q4.pack_w4(w)
    with torch.cuda.stream(torch.cuda.Stream()):
        got = q4.unpack_w4_f16_gpu(p)
        torch.cuda.current_stream().synchronize()
        assert np.array_equal(got.numpy(), want)


def test_logits_that_give_equal_candidates_keep_their_order(gpu):
    """Beside a log-sum of 8, 1e-20 and 0 are one candidate in 64 bits. Within a beam the larger logit still comes first;
    between beams equal candidates go to the lower one."""
    lk = gpu
    row = np.full(9000, -1.0, np.float32)
    row[[50, 100, 200, 8500, 8700]] = [-1e-20, 0.0, 1e-20, 3e-20, -0.0]
    best = [8500, 200, 100, 8700, 50]
    for b, k, parents, tokens in ((1, 3, [0] * 3, best[:3]), (1, 6, [0] * 6, best + [0]), (2, 7, [0] * 5 + [1] * 2, best + best[:2])):
        logits, scores, done = np.stack([row] * b), np.full(b, -2.0, np.float32), np.zeros(b, np.int64)
        got = [x.numpy() for x in lk.ops.beam_select_f32_gpu(G(lk, logits), G(lk, scores), G(lk, done), k, (7,))]
        assert got[1].tolist() == parents and got[2].tolist() == tokens
        ref = O.beam_select(logits, scores, done, k, [7])
        assert ref[1].tolist() == parents and ref[2].tolist() == tokens
