"""4-bit serving without a GPU: the registry's and the Python ops' refusals, and the oracle's quantiser against its
definition."""
import ctypes as C

import numpy as np
import pytest
import torch

import lokinfer_amd as lk
from lokinfer_amd import _lib, ops
from lokinfer_amd import q4_gpu as q4

from oracle import q4 as O


def run(name, ints, floats=()):
    """Registry call with null pointers: only host checks may answer."""
    L = _lib.lib()
    k = L.lk_find_kernel(name.encode())
    assert k, name
    nop, nout = C.c_int(), C.c_int()
    L.lk_kernel_arity(k, C.byref(nop), C.byref(nout))
    n = nop.value + nout.value
    rc = L.lk_run_kernel(k, (C.c_void_p * n)(), n, (C.c_int64 * max(1, len(ints)))(*ints), len(ints),
                         (C.c_double * max(1, len(floats)))(*floats), len(floats), None, 0, None)
    return rc, L.lk_last_error().decode()


P32 = 72 * 32

REFUSED = [
    ("quantize_w4_f16_gpu", [64, 16, 1, 1, 256, 1, 1, 16, 4, 48, 0], "group"),          # no such group
    ("quantize_w4_f16_gpu", [64, 17, 1, 1, 256, 1, 1, 16, 4, 32, 0], "ceil"),           # 17 columns need 2 tiles
    ("pack_w4_u8_gpu", [64, 16, 1, 16, 1, 1, 1, 256, 1, 1, 16, 4, 32], "ceil"),         # 2 groups of 32
    ("pack_w4_u8_gpu", [64, 16, 2, 16, 2, 1, 1, 256, 1, 1, 16, 4, 32], "flag"),
    ("unpack_w4_f16_gpu", [1, 1, 256, 1, 1, 16, 4, 129, 16, 32], "out"),                # K = 129 needs 2 k blocks
    ("gemm_w4_f16_gpu", [1, 64, 1, 1, 256, 1, 1, 16, 4, 1, 17, 32], "weight"),          # N = 17
    ("gemm_w4_f16_gpu", [1, 64, 1, 1, 256, 1, 1, 16, 4, 2, 16, 32], "out"),             # out rows
    ("gemm_w4_f16_gpu", [1, 60, 1, 1, 256, 1, 1, 16, 4, 1, 16, 32], "multiple of 8"),   # K = 60
    ("gemm_w4_bias_f16_gpu", [1, 64, 1, 1, 256, 1, 1, 16, 4, 15, 1, 16, 32], "bias"),
    ("gemm_w4_add_f16_gpu", [2, 64, 1, 1, 256, 1, 1, 16, 4, 1, 16, 2, 16, 32], "res"),
    ("gemm_w4_swiglu_f16_gpu", [1, 64, 1, 1, 256, 1, 1, 16, 4, 1, 1, 256, 1, 1, 16, 2, 1, 16, 32], "weight"),
    ("rmsnorm_gemm_w4_f16_gpu", [2, 64, 64, 1, 1, 256, 1, 1, 16, 4, 2, 16, 32], "one row"),
    ("rmsnorm_gemm_w4_f16_gpu", [1, 64, 63, 1, 1, 256, 1, 1, 16, 4, 1, 16, 32], "g must be"),
    ("kv4_write_f16_gpu", [1, 2, 1, P32 + 72, 1, 128, 1, 128, 1], "P % 32"),            # 33 rows
    ("kv4_write_f16_gpu", [2, 2, 1, P32, 3, 128, 3, 128, 2], "B T"),                    # 3 rows of 2 sequences
    ("kv4_write_f16_gpu", [1, 2, 1, P32, 1, 128, 1, 128, 2], "pos"),
    ("qknorm_rope_kv4_f16_gpu", [1, 384, 128, 64, 1, 1, 2, 1, P32, 1, 128], "gains"),
    ("kv4_read_f16_gpu", [1, P32, 1, 31, 128], "P % 32"),
    ("attention_kv4_f16_gpu", [1, 384, 1, 2, 2, P32, 1, 1, 384, 0], "multiple of kvh"),
    ("attention_kv4_f16_gpu", [1, 256, 1, 2, 2, P32, 2, 1, 256, 0], "pos"),
    ("kv4_reorder_gpu", [1, 33, 2, 1, P32, 33, 1], "B <= 32"),
    ("kv4_reorder_gpu", [1, 4, 2, 1, P32, 3, 1], "parents"),
    ("beam_select_f32_gpu", [2, 100, 2, 2, 33, 33, 33, 33, 4096, 1], "k outputs"),
    ("beam_select_f32_gpu", [2, 100, 2, 2, 4, 4, 4, 4, 4096, 100], "eos"),
    ("beam_select_f32_gpu", [2, 100, 2, 2, 4, 4, 4, 4, 4096], "eos"),
    ("beam_select_f32_gpu", [2, 300000, 2, 2, 4, 4, 4, 4, 4096, 1], "262144"),
    ("beam_select_f32_gpu", [1, 3, 1, 1, 4, 4, 4, 4, 4096, 1], "k <= 32"),               # k > B V
    ("beam_select_f32_gpu", [2, 100, 2, 2, 4, 4, 4, 4, 4, 1], "work"),
]


@pytest.mark.parametrize("name,ints,said", REFUSED, ids=[f"{n}-{i}" for i, (n, _, _) in enumerate(REFUSED)])
def test_registry_refuses_before_any_launch(name, ints, said):
    rc, msg = run(name, ints)
    assert rc != 0 and said in msg, msg


def test_python_ops_refuse_host_tensors_and_bad_handles():
    x = lk.Tensor(torch.zeros(1, 64, dtype=torch.float16))
    kv = lk.Tensor(torch.zeros(1, 2, 1, P32, dtype=torch.uint8))
    pos = lk.Tensor(torch.zeros(1, dtype=torch.int64))
    with pytest.raises(ops.OpError, match="on the GPU"):
        q4.quantize_w4_f16_gpu(x)
    with pytest.raises(ops.OpError, match="on the GPU"):
        q4.attention_kv4_f16_gpu(x, kv, pos)
    with pytest.raises(ops.OpError, match="on the GPU"):
        ops.beam_select_f32_gpu(lk.zeros(1, 8), lk.zeros(1), pos, 1, (0,))
    with pytest.raises(ops.OpError, match="72 P"):
        q4.kv4_capacity(lk.Tensor(torch.zeros(1, 2, 1, 72 * 31, dtype=torch.uint8)))
    with pytest.raises(ops.OpError, match="q does not fit"):
        q4.PackedWeight4(lk.Tensor(torch.zeros(1, 1, 255, dtype=torch.int32)), x, (64, 16), 32)
    with pytest.raises(ops.OpError, match="s does not fit"):
        q4.PackedWeight4(lk.Tensor(torch.zeros(1, 1, 256, dtype=torch.int32)),
                         lk.Tensor(torch.zeros(1, 1, 16, 2, dtype=torch.float16)), (64, 16), 32)


def test_oracle_quantizer_is_exact_in_f16_and_off_by_half_a_step():
    r = np.random.default_rng(1)
    x = (r.standard_normal((200, 32)) * np.exp2(r.uniform(-24, 14, (200, 1)))).astype(np.float16)
    codes, s = O.quantize(x)
    v = (codes - 8) * s[:, None]
    assert (v.astype(np.float16).astype(np.float64) == v).all()
    over = np.abs(x.astype(np.float64)) > 56896
    assert (np.abs(v - x.astype(np.float64))[~over] <= (np.broadcast_to(s[:, None], v.shape) / 2)[~over]).all()


def test_oracle_scale_is_the_smallest_that_holds():
    """Against every f16 of at most 8 significant bits."""
    every = np.arange(0x7C00, dtype=np.uint16).view(np.float16).astype(np.float64)
    m = np.round(every * 2.0 ** 24).astype(np.int64)
    odd = m // np.maximum(m & -m, 1)
    grid = every[(odd < 256) & (every <= 8128)]
    r = np.random.default_rng(2)
    hi = (np.abs(r.standard_normal(4000)) * np.exp2(r.uniform(-26, 15, 4000))).clip(0, 65504).astype(np.float16)
    lo = (-np.abs(r.standard_normal(4000)) * np.exp2(r.uniform(-26, 15, 4000))).clip(-65504, 0).astype(np.float16)
    lo[::5] = 0
    hi[::7] = (grid[r.integers(0, len(grid), len(hi[::7]))] * 7).clip(0, 65504).astype(np.float16)  # scales that fit exactly
    hi, lo = hi.astype(np.float64), lo.astype(np.float64)
    got = O.scale_of(hi, lo)
    for h, l, s in zip(hi, lo, got):
        fits = grid[(7 * grid >= h) & (8 * grid >= -l)]
        assert s == (fits[0] if len(fits) else 8128.0), (h, l, s)
