"""What the mixture-of-experts and residual-norm entries refuse before any
device is touched."""
import ctypes


def test_null_context_is_refused(q8):
    L = q8.lib()
    d = q8.f32_memref(64, 1, 32)
    r = ctypes.byref(d)
    for t in ("", "_bf16"):
        assert getattr(L, "llmcp_q8_add_rmsnorm" + t)(None, r, r, r, 1e-6, 0, r, r, None) == q8.EINVAL
        assert getattr(L, "llmcp_q8_route" + t)(None, r, 1, 1, 1.0, 64, 64) == q8.EINVAL
        assert getattr(L, "llmcp_q8_expert_linear" + t)(None, r, 64, 1, r, r, 0) == q8.EINVAL
        for name in ("llmcp_q8_expert_mlp", "llmcp_q8_expert_mlp_rows"):
            assert getattr(L, name + t)(None, r, 64, 64, 1, r, r, r, None, r) == q8.EINVAL
    assert L.llmcp_q8_upload_experts_p4(None, 64, 1, 8, 32, None) == q8.EINVAL
    assert L.llmcp_q8_register_device_experts_p4(None, 64, 1, 8, 32, None) == q8.EINVAL
    assert "null" in q8.last_error()


def test_stack_of_experts_concatenates(q8, oracle):
    """A stack's p4 bytes are its experts', one after another: those of the
    tensor of all their rows."""
    import numpy as np
    w = np.random.default_rng(0).standard_normal((3, 16, 64)).astype(np.float32)
    parts = np.concatenate([q8.pack_p4_host(x) for x in w])
    assert np.array_equal(parts, q8.pack_p4_host(w.reshape(48, 64)))
