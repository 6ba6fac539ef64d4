"""CPU-only checks of the paged latent cache's C ABI: what each entry point
refuses before it launches anything, and what it does with nothing to do."""
import ctypes

import pytest


def _desc(**kw):
    from cascade_kernel import capi as C
    extra = {k: kw.pop(k) for k in ("dtype", "flags") if k in kw}
    head = {"q_seqlen_value": 1, "scale": 0.1, "causal": True}
    head.update({k: kw.pop(k) for k in list(kw) if k in head})
    shape = dict(num_tokens=4, num_heads=16, latent_dim=512, rope_dim=64, num_blocks=100, block_size=64, batch=4,
                 block_cols=8)
    shape.update(kw)
    return C.latent_desc(None, None, None, None, None, head["q_seqlen_value"], head["scale"], head["causal"],
                         shape=shape, **extra)


def _refused(rc, text):
    from cascade_kernel import capi as C
    assert rc != C.OK and text in C.last_error(), C.last_error()


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=2), "bf16 or fp16"),
    (dict(latent_dim=256), "512 latent"),
    (dict(rope_dim=32), "64 rotary"),
    (dict(block_size=24), "blockSize"),
    (dict(block_size=1024), "blockSize"),
    (dict(num_tokens=-1), "negative size"),
    (dict(num_tokens=5), "batch * q_seqlen_value"),
    (dict(q_seqlen_value=-1), "q_seqlen_value must be >= 0"),
    (dict(num_blocks=1 << 26), "too large"),
    (dict(num_tokens=1 << 28, batch=1 << 28), "too large"),
    (dict(scale=0.0), "scale must be positive"),
    (dict(scale=float("nan")), "scale must be positive"),
    (dict(flags=1), "unknown flags"),
    (dict(), "null device pointer"),
])
def test_decode_refusals(kw, text):
    from cascade_kernel import capi as C
    d = _desc(**kw)
    _refused(C.load().cascade_latent_decode(ctypes.byref(d), None, None, None, 0, None), text)


def test_decode_nothing_to_do_and_alignment():
    from cascade_kernel import capi as C
    lib = C.load()
    d = _desc(num_tokens=0, batch=0)
    assert lib.cascade_latent_decode(ctypes.byref(d), None, None, None, 0, None) == C.OK
    assert lib.cascade_latent_decode_workspace_size(ctypes.byref(d)) == 0
    _refused(lib.cascade_latent_decode(None, None, None, None, 0, None), "null argument")
    d = _desc()
    for f in ("query", "cache", "block_table", "actual_kv_seqlens"):
        setattr(d, f, 4096)
    d.query = 4104
    _refused(lib.cascade_latent_decode(ctypes.byref(d), 4096, 4096, None, 0, None), "16-byte aligned")


def test_prefill_refusals():
    from cascade_kernel import capi as C
    lib = C.load()

    def desc(**kw):
        p = C.LatentPrefill()
        base = dict(num_tokens=8, num_kv=8, num_heads=2, batch=1, max_q_seqlen=8, key_token_stride=256,
                    key_head_stride=128, rope_token_stride=64, value_token_stride=256, value_head_stride=128, scale=0.1,
                    dtype=C.BF16, query=4096, key=4096, key_rope=4096, value=4096, cu_q_seqlens=4096, cu_kv_seqlens=4096)
        base.update(kw)
        for k, v in base.items():
            setattr(p, k, v)
        return ctypes.byref(p)

    for kw, text in [(dict(dtype=2), "bf16 or fp16"), (dict(num_kv=-1), "negative size"), (dict(num_heads=70000), "too large"),
                     (dict(scale=-1.0), "scale"), (dict(flags=4), "unknown flags"), (dict(max_q_seqlen=0), "max_q_seqlen"),
                     (dict(key_token_stride=12), "multiples of 8"), (dict(value_head_stride=-8), "multiples of 8"),
                     (dict(key=0), "null device pointer"), (dict(key=4100), "16-byte aligned")]:
        _refused(lib.cascade_latent_prefill(desc(**kw), 4096, 4096, None), text)
    assert lib.cascade_latent_prefill(desc(num_tokens=0), None, None, None) == C.OK


def test_page_refusals():
    from cascade_kernel import capi as C
    lib = C.load()
    one = (ctypes.c_void_p * 1)(4096)
    odd = (ctypes.c_void_p * 1)(4097)
    _refused(lib.cascade_page_copy(odd, 1, 10, 64, 4096, 4096, 1, None), "16-byte aligned")
    _refused(lib.cascade_page_copy(one, 1, 10, 60, 4096, 4096, 1, None), "16 bytes")
    _refused(lib.cascade_page_copy(one, 1, 10, 64, None, 4096, 1, None), "null device pointer")
    assert lib.cascade_page_copy(one, 1, 10, 64, None, None, 0, None) == C.OK
    fork = lambda *a: lib.cascade_page_fork(one, 1, 10, *a)  # noqa: E731
    _refused(fork(0, 64, 4096, 1, 1, 4096, 4096, 4096, 1, 4096, 4096, 8192, 4096, 99, None), "block size")
    _refused(fork(16, 64, 4096, 1, 1, 4096, 4096, 4096, 1, 4096, 4096, 4096, 4096, 99, None), "must not be page_refs")
    _refused(fork(16, 64, 4096, 1, 1, 4096, 4096, 4096, 1, 4096, 4096, 8192, None, 0, None), "workspace too small")
    _refused(fork(16, 64, 4096, 1, 1, 4096, 4096, None, 1, 4096, 4096, 8192, 4096, 99, None), "null device pointer")
    assert lib.cascade_page_fork_workspace_size(10, 0) == 0
    _refused(lib.cascade_page_free(4096, 1, 1, 4096, 4096, 10, None, 16, 4096, 4096, 8192, None), "null device pointer")
    _refused(lib.cascade_page_free(4096, -1, 1, 4096, 4096, 10, 4096, 16, 4096, 4096, 8192, None), "negative size")
    _refused(lib.cascade_page_compact(one, 1, 0, 16, 64, 4096, 1, 1, 4096, 4096, 4096, 8192, 4096, 4096, 999, None),
             "no pages")
    _refused(lib.cascade_page_compact(one, 1, 10, 16, 64, 4096, 1, 1, 4096, 4096, 4096, 8192, 4096, 4096, 3, None),
             "workspace too small")


def test_verify_refusals():
    from cascade_kernel import capi as C
    f = C.load().cascade_verify_drafts
    ok = [4096, 4096, 4096, 4096, 4096, 4096, C.FP32, 2, 3, 100, 4096, 4096, None]

    def put(i, v):
        return ok[:i] + [v] + ok[i + 1:]

    for i, v, text in [(6, 7, "bf16, fp16 or fp32"), (7, -1, "negative size"), (9, 0, "must not be empty"),
                       (9, 1 << 32, "too large"), (3, None, "null device pointer"), (3, 4098, "aligned to their elements"),
                       (10, None, "null device pointer")]:
        _refused(f(*put(i, v)), text)
    assert f(*put(7, 0)) == C.OK


def test_verify_refuses_rows_near_the_32_bit_limit():
    """The kernel's 32-bit indices step past the end of a row before they are compared with it."""
    from cascade_kernel import capi as C
    f = C.load().cascade_verify_drafts
    for vocab in ((1 << 31) - 1, 1 << 30):
        _refused(f(4096, 4096, 4096, 4096, 4096, 4096, C.FP32, 2, 3, vocab, 4096, 4096, None), "too large")


def test_schemas():
    import torch
    import cascade_kernel  # noqa: F401
    for name in ("cascade_latent_decode", "cascade_latent_prefill", "cascade_page_copy", "cascade_page_fork",
                 "cascade_page_free", "cascade_page_compact", "cascade_verify_drafts"):
        assert str(getattr(torch.ops.npu, name).default._schema).startswith("npu::" + name)


@pytest.mark.parametrize("batch,tokens,q_seqlen", [(3, 5, 0x5555555555555557), (4, 4, (1 << 62) + 1), (1, 1 << 31, 1 << 31)])
def test_decode_refuses_query_lengths_past_32_bits(batch, tokens, q_seqlen):
    """3 x 0x5555555555555557 is 5 modulo 2^64: the product must not be taken for num_tokens."""
    from cascade_kernel import capi as C
    d = _desc(batch=batch, num_tokens=tokens, q_seqlen_value=q_seqlen)
    _refused(C.load().cascade_latent_decode(ctypes.byref(d), None, None, None, 0, None), "too large")
    assert C.load().cascade_latent_decode_workspace_size(ctypes.byref(d)) == 0
