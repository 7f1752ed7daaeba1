"""Replays of graphs that are a short chain of kernels: of this library's, and
with a kernel of another's among them (a module's function, which only a graph
launch may replay)."""
import ctypes

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

SOURCE = b"""
extern "C" __global__ void twice(float *p, int n) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i < n) p[i] = 2.0f * p[i];
}
"""


class Module:
    """A kernel compiled at run time and loaded as a module."""

    def __init__(self):
        rtc, self.hip = ctypes.CDLL("libhiprtc.so.7"), ctypes.CDLL("libamdhip64.so.7")
        prog, size = ctypes.c_void_p(), ctypes.c_size_t()
        ok = rtc.hiprtcCreateProgram(ctypes.byref(prog), SOURCE, b"twice.hip", 0, None, None)
        opts = (ctypes.c_char_p * 1)(b"--offload-arch=gfx950")
        assert ok == 0 and rtc.hiprtcCompileProgram(prog, 1, opts) == 0
        assert rtc.hiprtcGetCodeSize(prog, ctypes.byref(size)) == 0
        code = ctypes.create_string_buffer(size.value)
        assert rtc.hiprtcGetCode(prog, code) == 0
        self.module, self.function = ctypes.c_void_p(), ctypes.c_void_p()
        assert self.hip.hipModuleLoadData(ctypes.byref(self.module), code) == 0
        assert self.hip.hipModuleGetFunction(ctypes.byref(self.function), self.module, b"twice") == 0

    def launch(self, stream, buf, n):
        ptr, count = ctypes.c_void_p(buf.ptr), ctypes.c_int(n)
        args = (ctypes.c_void_p * 2)(ctypes.addressof(ptr), ctypes.addressof(count))
        u = ctypes.c_uint
        assert self.hip.hipModuleLaunchKernel(
            self.function, u((n + 255) // 256), u(1), u(1), u(256), u(1), u(1), u(0),
            ctypes.c_void_p(stream), args, None) == 0


@pytest.mark.parametrize("linears,foreign", [(1, False), (3, False), (3, True), (12, False)])
def test_chain_of_kernels(ctx, oracle, q8, linears, foreign):
    """A chain of linears, each on the last one's output, replayed with new
    inputs and eager work in between: every replay the eager bits."""
    rng = np.random.default_rng(linears)
    n = 64
    p4 = oracle.pack_q8_0_p4((rng.standard_normal((n, n)) * 0.2).astype(np.float32))
    w = ctx.upload_p4(p4, n, n)
    bufs = [ctx.alloc(n * 4) for _ in range(linears + 1)]
    module = Module() if foreign else None
    stream = q8.lib().llmcp_q8_ctx_stream(ctx.handle)

    def run():
        for a, b in zip(bufs, bufs[1:]):
            ctx.linear(a, w, b, 1)
        if module:
            module.launch(stream, bufs[-1], n)
    run()
    ctx.sync()
    ctx.graph_begin()
    run()
    g = ctx.graph_end()
    try:
        for rep in range(4):
            x = rng.standard_normal((1, n)).astype(np.float32)
            ctx.sync()
            q8.check(q8.lib().llmcp_q8_memcpy_h2d(ctx.handle, bufs[0].ptr, x.ctypes.data, x.nbytes))
            ctx.graph_launch(g)
            got = ctx.to_host(bufs[-1], (n,), np.float32)
            run()
            assert np.array_equal(got.view(np.uint32), ctx.to_host(bufs[-1], (n,), np.uint32)), rep
            for _ in range(linears):
                x = oracle.linear(x, p4, n, epilogue=ctx.epilogue)
            assert np.array_equal((x[0] * (2 if foreign else 1)).view(np.uint32), got.view(np.uint32))
    finally:
        ctx.graph_destroy(g)
        ctx.release(w)
