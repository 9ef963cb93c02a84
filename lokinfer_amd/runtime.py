"""HIP execution context: one stream (torch's current stream on the device), one zero-initialised device
workspace for kernels that merge partial results, and the launch path into the C-ABI registry.

Replaces the reference's GpuContext (src/runtime/gpu_internal.h:53-290): Metal command buffers, arg tables and
the params ring become plain HIP launches on one stream; errors come back as a status + message and are raised
as LokinferError, the binding-level exception the reference raises from Status (python/ext/module.cpp:29-31).
"""
from __future__ import annotations

import contextlib
from array import array

import torch

from ._lib import LokinferError, check_device_errors, lib
from .graph import current_graph

WORKSPACE_BYTES = 64 << 20
_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice


class GpuContext:
    _shared: "GpuContext | None" = None

    def __init__(self):
        if not torch.cuda.is_available():
            raise LokinferError("no HIP device available (the lokinfer GPU kernels need an MI355X / gfx950)")
        self.device = torch.device("cuda", torch.cuda.current_device())
        # First 64 KiB: ticket counters (must start at zero; kernels restore them), rest: partials.
        self.workspace = torch.zeros(WORKSPACE_BYTES // 4, dtype=torch.float32, device=self.device)
        self.lib = lib()
        self._run_kernel, self._index = self.lib.lk_run_kernel, self.device.index
        self._handles: dict[str, int] = {}
        self._ws_by_slot: dict[int, torch.Tensor] = {0: self.workspace}
        self.slot = 0

    def workspace_for(self, slot: int) -> torch.Tensor:
        """Workspace of a branch slot. Kernels on one stream are ordered and share slot 0; a branch that runs
        concurrently on another stream (see `branch`) uses its own slot. A new slot is allocated on first use,
        which happens on a model's eager warm-up run, before any graph capture."""
        ws = self._ws_by_slot.get(slot)
        if ws is None:
            if torch.cuda.is_current_stream_capturing():
                raise LokinferError("no workspace for this branch yet: run the function once outside capture")
            ws = torch.zeros(WORKSPACE_BYTES // 4, dtype=torch.float32, device=self.device)
            self._ws_by_slot[slot] = ws
        return ws

    def branch(self, stream: "torch.cuda.Stream", slot: int):
        """Context manager: run the enclosed launches on `stream` (which first waits for the current stream)
        with workspace slot `slot`. Join with `join(stream)` before consuming the branch's outputs."""
        ctx = self

        class _Branch:
            def __enter__(self):
                cur = torch.cuda.current_stream(ctx.device)
                stream.wait_stream(cur)
                g = current_graph()
                if g is not None:
                    g.stream_wait(stream, cur)
                self._prev = ctx.slot
                self._sc = torch.cuda.stream(stream)
                self._sc.__enter__()
                ctx.slot = slot
                return stream

            def __exit__(self, *exc):
                ctx.slot = self._prev
                self._sc.__exit__(*exc)
                return False

        return _Branch()

    def join(self, stream: "torch.cuda.Stream") -> None:
        cur = torch.cuda.current_stream(self.device)
        cur.wait_stream(stream)
        g = current_graph()
        if g is not None:
            g.stream_wait(cur, stream)

    def mark(self, stream: "torch.cuda.Stream"):
        """An event recorded on `stream` now; `wait_mark(other, m)` makes `other` wait for it. Traced functions
        record the same structure for the compiled runtime's lane schedule."""
        ev = torch.cuda.Event()
        ev.record(stream)
        g = current_graph()
        return (ev, g.mark(stream) if g is not None else None)

    def wait_mark(self, stream: "torch.cuda.Stream", m) -> None:
        stream.wait_event(m[0])
        g = current_graph()
        if g is not None and m[1] is not None:
            g.wait_mark(stream, m[1])

    @classmethod
    def shared(cls) -> "GpuContext":
        if cls._shared is None:
            cls._shared = GpuContext()
        return cls._shared

    def handle(self, name: str) -> int:
        h = self._handles.get(name)
        if h is None:
            h = self.lib.lk_find_kernel(name.encode())
            if not h:
                raise LokinferError(f"unknown kernel '{name}'")
            self._handles[name] = h
        return h

    def run(self, name: str, ptrs, ints, floats) -> None:
        if _current_device() != self._index:  # the null stream is the current device's, whichever that is
            with torch.cuda.device(self._index):
                return self.run(name, ptrs, ints, floats)
        n = len(ptrs)
        words = array("q", (*ptrs, *ints))  # both arrays of lk_run_kernel: one buffer is cheaper to make than two
        at = words.buffer_info()[0]
        fa = array("d", floats) if floats else None
        ws = self._ws_by_slot.get(self.slot)
        if ws is None:
            ws = self.workspace_for(self.slot)
        rc = self._run_kernel(self._handles.get(name) or self.handle(name), at, n, at + 8 * n, len(words) - n,
                              fa.buffer_info()[0] if floats else None, len(floats), ws.data_ptr(), WORKSPACE_BYTES,
                              _raw_stream(self._index))
        if rc != 0:
            raise LokinferError(self.lib.lk_last_error().decode())


def context_device():
    """Context manager: the shared context's GPU is the current one (before there is a context, the one that is)."""
    ctx = GpuContext._shared
    return contextlib.nullcontext() if ctx is None else torch.cuda.device(ctx.device)


def synchronize() -> None:
    """Waits for the GPU and raises LokinferError for a data error a kernel recorded (check_device_errors)."""
    torch.cuda.synchronize()
    check_device_errors()
