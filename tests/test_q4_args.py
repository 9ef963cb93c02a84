"""4-bit ops and the launch path without a GPU: what a call is refused for, and where a launch goes."""
import contextlib

import numpy as np
import pytest
import torch

import lokinfer_amd as lk
from lokinfer_amd import ops
from lokinfer_amd import q4_gpu as q4


@pytest.mark.parametrize("bad", [np.full((64, 4), 257, np.int32), np.full((64, 4), -250),
                                 np.full((64, 4), 1.7), np.full((64, 4), np.nan, np.float32), np.full((64, 4), 2 ** 40)],
                         ids=["257", "-250", "1.7", "nan", "2^40"])
def test_codes_are_checked_as_given(bad):
    """Not after a cast to u8, which would turn 257 into 1."""
    codes = np.full(bad.shape, 3, bad.dtype)
    codes[63, 2] = bad[0, 0]
    with pytest.raises(ops.OpError, match="codes must be 0 .. 15"):
        q4.pack_w4(codes, np.ones((2, 4), np.float16), 32)


@pytest.mark.parametrize("bad", [np.float32(1e-9), np.float64(1 + 2.0 ** -12), np.float32(1e6), np.float32(np.nan), 70000],
                         ids=["1e-9", "1 + 2^-12", "1e6", "nan", "70000"])
def test_scales_are_checked_as_given(bad):
    """Not after a cast to f16, which would turn 1e-9 into 0."""
    scales = np.ones((2, 4), np.asarray(bad).dtype)
    scales[1, 3] = bad
    with pytest.raises(ops.OpError, match="scales must be"):
        q4.pack_w4(np.zeros((64, 4), np.uint8), scales, 32)


def test_torch_tensors_are_no_operands():
    """A torch.Tensor has a method `t`, as an lk.Tensor has the attribute: the refusal names the type."""
    h, u8, i64 = (torch.zeros(*s, dtype=d) for s, d in (((1, 128), torch.float16), ((1, 2, 1, 72 * 32), torch.uint8),
                                                        ((1,), torch.int64)))
    w = q4.PackedWeight4.__new__(q4.PackedWeight4)
    for call in (lambda: q4.quantize_w4_f16_gpu(h), lambda: q4.gemm_w4_f16_gpu(h, w), lambda: q4.rmsnorm_gemm_w4_f16_gpu(h, h, w),
                 lambda: q4.kv4_write_f16_gpu(u8, h, h, i64), lambda: q4.attention_kv4_f16_gpu(h, u8, i64),
                 lambda: q4.qknorm_rope_kv4_f16_gpu(h, h, h, i64, u8), lambda: q4.kv4_reorder_gpu(u8, i64, i64),
                 lambda: q4.quantize_w4_f16_gpu(np.zeros((8, 8)))):
        with pytest.raises(ops.OpError, match="expected lk.Tensor"):
            call()


def test_launches_go_to_the_contexts_gpu(monkeypatch):
    """The null stream is that of the current GPU, whichever that is: a launch makes the context's the current one."""
    from lokinfer_amd import _lib, runtime

    current, seen = [1], []

    @contextlib.contextmanager
    def device(of):
        was, current[0] = current[0], getattr(of, "index", of)
        yield
        current[0] = was

    ctx = runtime.GpuContext.__new__(runtime.GpuContext)
    ctx._index, ctx._handles, ctx.slot = 0, {"op": 1}, 0
    ctx.device = torch.device("cuda", 0)
    ctx._ws_by_slot = {0: torch.zeros(1)}
    ctx._run_kernel = lambda *args: seen.append(current[0]) or 0
    monkeypatch.setattr(runtime, "_current_device", lambda: current[0])
    monkeypatch.setattr(runtime, "_raw_stream", lambda index: 0)
    monkeypatch.setattr(torch.cuda, "device", device)
    ctx.run("op", (1, 2), (3,), ())
    current[0] = 0
    ctx.run("op", (1, 2), (3,), (0.5,))
    assert seen == [0, 0]
    # and a data error is read from where the kernels ran
    current[0] = 1
    monkeypatch.setattr(runtime.GpuContext, "_shared", ctx)

    class Lib:
        def lk_take_device_error(self, detail):
            seen.append(current[0])
            return 0

    monkeypatch.setattr(_lib, "lib", Lib)
    _lib.check_device_errors()
    assert seen == [0, 0, 0] and current == [1]
