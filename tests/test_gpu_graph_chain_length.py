"""Which captured graphs are replayed as launches (short chains of this
library's kernels, as long as that costs the host less than a graph launch), and
graphs over the experts' workspaces once those have grown."""
import ctypes

import numpy as np
import pytest

from test_gpu_graph_chain import Module

pytestmark = pytest.mark.gpu


def chain_of(q8, graph):
    fn = q8.lib().llmcp_q8_test_graph_chain
    fn.argtypes, fn.restype = [ctypes.c_void_p], ctypes.c_int32
    return fn(graph)


@pytest.mark.parametrize("linears,foreign,launches", [
    (1, False, 1), (3, False, 3), (7, False, 7), (8, False, 0), (12, False, 0), (3, True, 0)])
def test_which_graphs_are_launches(ctx, oracle, q8, linears, foreign, launches):
    rng = np.random.default_rng(linears)
    n = 64
    p4 = oracle.pack_q8_0_p4((rng.standard_normal((n, n)) * 0.2).astype(np.float32))
    w = ctx.upload_p4(p4, n, n)
    x = rng.standard_normal((1, n)).astype(np.float32)
    bufs = [ctx.to_device(x)] + [ctx.alloc(n * 4) for _ in range(linears)]
    module = Module() if foreign else None

    def run():
        for a, b in zip(bufs, bufs[1:]):
            ctx.linear(a, w, b, 1)
        if module:
            module.launch(q8.lib().llmcp_q8_ctx_stream(ctx.handle), bufs[-1], n)
    run()
    ctx.sync()
    ctx.graph_begin()
    run()
    g = ctx.graph_end()
    try:
        assert chain_of(q8, g) == launches
        for _ in range(3):
            ctx.graph_launch(g)
        for _ in range(linears):
            x = oracle.linear(x, p4, n, epilogue=ctx.epilogue)
        got = ctx.to_host(bufs[-1], (n,), np.float32)
        assert np.array_equal((x[0] * (2 if foreign else 1)).view(np.uint32), got.view(np.uint32))
    finally:
        ctx.graph_destroy(g)
        ctx.release(w)
    assert chain_of(q8, g) == -1


@pytest.mark.parametrize("m,more", [(1, 2), (1, 400), (6, 60), (100, 400)])
def test_expert_graph_is_stale_once_its_workspace_grew(ctx, oracle, q8, m, more):
    """A larger eager call after the capture takes new memory for the experts'
    outputs (and the plan and the hidden rows): the graph is refused, and one
    captured again gives the eager bits."""
    rng = np.random.default_rng(m + more)
    top_k, e, h, f = 3, 6, 96, 64
    with q8.Context(0) as c:
        c.set_platform(ctx.platform)
        stacks = []
        for n, k in ((f, h), (f, h), (h, f)):
            w = [oracle.pack_q8_0_p4((rng.standard_normal((n, k)) * 0.1).astype(np.float32)) for _ in range(e)]
            stacks.append(c.upload_experts_p4(np.concatenate(w), e, n, k))
        x = c.to_device(rng.standard_normal((more, h)).astype(np.float32))
        ids = c.to_device(rng.integers(-1, e, (more, top_k)).astype(np.int32))
        y, z = c.alloc(more * h * 4), c.alloc(more * h * 4)

        def capture():
            c.expert_mlp(x, ids, None, m, top_k, *stacks, y)
            c.sync()
            c.graph_begin()
            c.expert_mlp(x, ids, None, m, top_k, *stacks, y)
            return c.graph_end()
        g = capture()
        assert (chain_of(q8, g) == 2) == (m == 1)
        c.graph_launch(g)
        c.expert_mlp(x, ids, None, more, top_k, *stacks, z)
        with pytest.raises(q8.Q8Error) as err:
            c.graph_launch(g)
        assert err.value.code == q8.ESTALE
        c.graph_destroy(g)
        g = capture()
        nan = np.full(m * h, np.nan, np.float32)
        for _ in range(3):
            q8.check(q8.lib().llmcp_q8_memcpy_h2d(c.handle, y.ptr, nan.ctypes.data, nan.nbytes))
            c.graph_launch(g)
            c.expert_mlp(x, ids, None, m, top_k, *stacks, z)
            assert np.array_equal(c.to_host(y, (m, h), np.uint32), c.to_host(z, (m, h), np.uint32))
        c.graph_destroy(g)
