"""CPU-only checks of sizes that attention over the 4-bit and the latent cache has to refuse."""
import ctypes

import pytest


@pytest.mark.parametrize("batch", [(1 << 30), (1 << 31) - 32, (1 << 31) - 1])
def test_decode_refuses_batches_whose_steps_wrap(batch):
    """With query lengths on the device a batch need not have a token per request; the kernels walk it in steps of a warp."""
    from cascade_kernel import capi as C
    p = C.QuantAttn()
    for k, v in dict(num_tokens=3, num_heads=16, kv_heads=4, head_dim=128, num_blocks=100, block_size=64, batch=batch, block_cols=0,
                     q_seqlen_value=0, scale=0.1, causal=1, dtype=C.BF16, flags=0).items():
        setattr(p, k, v)
    lib = C.load()
    assert lib.cascade_quant_decode(ctypes.byref(p), None, None, None, 0, None) != C.OK and "too large" in C.last_error()
    assert lib.cascade_quant_decode_workspace_size(ctypes.byref(p)) == 0
    p.batch = (1 << 30) - 1
    assert lib.cascade_quant_decode(ctypes.byref(p), None, None, None, 0, None) != C.OK and "null device pointer" in C.last_error()


@pytest.mark.parametrize("batch", [(1 << 30), (1 << 31) - 1])
def test_latent_decode_refuses_batches_whose_steps_wrap(batch):
    from cascade_kernel import capi as C
    shape = dict(num_tokens=3, num_heads=16, latent_dim=512, rope_dim=64, num_blocks=100, block_size=64, batch=batch, block_cols=0)
    lib = C.load()
    p = C.latent_desc(None, None, None, None, None, 0, 0.1, True, shape=shape)
    assert lib.cascade_latent_decode(ctypes.byref(p), None, None, None, 0, None) != C.OK and "too large" in C.last_error()
    p.batch = (1 << 30) - 1
    assert lib.cascade_latent_decode(ctypes.byref(p), None, None, None, 0, None) != C.OK and "null device pointer" in C.last_error()


@pytest.mark.parametrize("kv_heads,num_tokens", [(1, 1), (8, 1), (8, 40), (74, 40), (75, 40), (2000, 40), (3000, 1), (65535, 1)])
def test_decode_workspace_does_not_grow_with_the_heads(kv_heads, num_tokens):
    """Partial rows of at most two units of 256 rows per SM, and 4 bytes per query row: with more kv heads than SMs a unit is
    never cut."""
    from cascade_kernel import capi as C
    p = C.QuantAttn()
    for k, v in dict(num_tokens=num_tokens, num_heads=kv_heads, kv_heads=kv_heads, head_dim=128, num_blocks=100, block_size=64, batch=1,
                     block_cols=50, q_seqlen_value=num_tokens, scale=0.1, causal=1, dtype=C.BF16, flags=0).items():
        setattr(p, k, v)
    need = C.load().cascade_quant_decode_workspace_size(ctypes.byref(p))
    assert 0 < need <= 2 * 148 * 256 * 129 * 4 + num_tokens * kv_heads * 4 + 256
