"""CPU-only checks of the 4-bit cache's and the log probabilities' C ABI: what each entry point refuses before it
launches anything, what it does with nothing to do; the oracle's format."""
import ctypes

import numpy as np
import pytest


def _refused(rc, text):
    from cascade_kernel import capi as C
    assert rc != C.OK and text in C.last_error(), C.last_error()


def _desc(**kw):
    from cascade_kernel import capi as C
    p = C.QuantAttn()
    base = dict(num_tokens=4, num_heads=16, kv_heads=4, head_dim=128, num_blocks=100, block_size=64, batch=4, block_cols=8,
                q_seqlen_value=1, scale=0.1, causal=1, dtype=C.BF16, flags=0)
    base.update(kw)
    for k, v in base.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=2), "bf16 or fp16"),
    (dict(head_dim=64), "head_dim must be 128"),
    (dict(block_size=24), "blockSize"),
    (dict(block_size=8), "blockSize"),
    (dict(num_tokens=-1), "negative size"),
    (dict(kv_heads=0), "multiple of kv_heads"),
    (dict(kv_heads=3), "multiple of kv_heads"),
    (dict(num_tokens=5), "batch * q_seqlen_value"),
    (dict(q_seqlen_value=-1), "q_seqlen_value must be >= 0"),
    (dict(num_blocks=1 << 26), "too large"),
    (dict(num_heads=1 << 17), "too large"),
    (dict(num_tokens=1 << 28, batch=1 << 28), "too large"),
    (dict(batch=3, num_tokens=5, q_seqlen_value=0x5555555555555557), "too large"),  # their product is 5 modulo 2^64
    (dict(scale=0.0), "scale must be positive"),
    (dict(scale=float("nan")), "scale must be positive"),
    (dict(scale=float("inf")), "scale must be positive"),
    (dict(flags=1), "unknown flags"),
    (dict(), "null device pointer"),
    (dict(batch=0, num_tokens=3, q_seqlen_value=0), "no requests"),
])
def test_decode_refusals(kw, text):
    from cascade_kernel import capi as C
    _refused(C.load().cascade_quant_decode(ctypes.byref(_desc(**kw)), None, None, None, 0, None), text)


def test_decode_nothing_to_do_alignment_and_workspace():
    from cascade_kernel import capi as C
    lib = C.load()
    d = _desc(num_tokens=0, batch=0)
    assert lib.cascade_quant_decode(ctypes.byref(d), None, None, None, 0, None) == C.OK
    assert lib.cascade_quant_decode_workspace_size(ctypes.byref(d)) == 0
    _refused(lib.cascade_quant_decode(None, None, None, None, 0, None), "null argument")
    d = _desc()
    for f in ("query", "key_cache", "value_cache", "block_table", "actual_kv_seqlens"):
        setattr(d, f, 4096)
    need = lib.cascade_quant_decode_workspace_size(ctypes.byref(d))
    if need:
        _refused(lib.cascade_quant_decode(ctypes.byref(d), 4096, 4096, 4096, need - 1, None), "workspace too small")
        _refused(lib.cascade_quant_decode(ctypes.byref(d), 4096, 4096, 4104, need, None), "16-byte aligned")
    d.value_cache = 4104
    _refused(lib.cascade_quant_decode(ctypes.byref(d), 4096, 4096, 4096, need, None), "16-byte aligned")


def test_write_and_read_refusals():
    from cascade_kernel import capi as C
    lib = C.load()
    names = ("key", "kts", "khs", "value", "vts", "vhs", "kc", "vc", "slots", "tokens", "heads", "dim", "blocks", "page", "dtype")
    ok = dict(zip(names, (4096, 512, 128, 4096, 512, 128, 4096, 8192, 4096, 6, 4, 128, 10, 16, C.BF16)))

    def write(**kw):
        return lib.cascade_quant_write(*{**ok, **kw}.values(), None)

    for kw, text in [(dict(dtype=C.FP32), "bf16 or fp16"), (dict(dim=64), "head_dim"), (dict(tokens=-1), "negative size"),
                     (dict(page=0), "block size"), (dict(heads=70000), "too large"), (dict(key=None), "null device pointer"),
                     (dict(slots=None), "null device pointer"), (dict(vc=None), "null device pointer"),
                     (dict(value=4100), "16-byte aligned"), (dict(kc=4104), "16-byte aligned"), (dict(vc=4096), "two caches"),
                     (dict(kts=12), "multiples of 8"), (dict(vhs=-8), "multiples of 8")]:
        _refused(write(**kw), text)
    assert write(tokens=0, key=None) == C.OK and write(heads=0) == C.OK

    names = ("kc", "vc", "slots", "key", "value", "tokens", "heads", "dim", "blocks", "page", "dtype")
    ok = dict(zip(names, (4096, 8192, 4096, 4096, 4096, 6, 4, 128, 10, 16, C.FP32)))

    def read(**kw):
        return lib.cascade_quant_read(*{**ok, **kw}.values(), None)

    for kw, text in [(dict(dtype=5), "bf16, fp16 or fp32"), (dict(dim=256), "head_dim"), (dict(blocks=-1), "negative size"),
                     (dict(tokens=1 << 31), "too large"), (dict(value=None), "null device pointer"),
                     (dict(key=4104), "16-byte aligned")]:
        _refused(read(**kw), text)
    assert read(tokens=0, key=None) == C.OK


def test_logprobs_refusals():
    from cascade_kernel import capi as C
    lib = C.load()
    names = ("logits", "stride", "tokens", "dtype", "rows", "vocab", "top", "logprob", "entropy", "rank", "tl", "tt")
    ok = dict(zip(names, (4096, 100, 4096, C.BF16, 3, 100, 5, 4096, 4096, 4096, 4096, 4096)))

    def call(**kw):
        return lib.cascade_token_logprobs(*{**ok, **kw}.values(), None)

    for kw, text in [(dict(dtype=3), "bf16, fp16 or fp32"), (dict(rows=-1), "negative size"), (dict(vocab=0), "must not be empty"),
                     (dict(top=33), "top must be"), (dict(top=-1), "negative size"), (dict(vocab=4, top=5), "top must be"),
                     (dict(vocab=(1 << 30) - 1, stride=1 << 30), "too large"), (dict(rows=1 << 28), "too large"),
                     (dict(stride=99), "row stride"), (dict(logits=4097), "aligned to their elements"),
                     (dict(tokens=None), "null device pointer"), (dict(tt=None), "null device pointer"),
                     (dict(rank=4100), "aligned to their elements")]:
        _refused(call(**kw), text)
    assert call(rows=0, logits=None) == C.OK


def test_schemas():
    import torch
    import cascade_kernel  # noqa: F401
    for name in ("cascade_quant_write", "cascade_quant_read", "cascade_quant_decode", "cascade_token_logprobs"):
        assert str(getattr(torch.ops.npu, name).default._schema).startswith("npu::" + name)


def test_oracle_format():
    """pack and values undo one another to half a step, whatever the group holds."""
    import torch
    from oracle import quant_oracle as Q
    g = torch.Generator().manual_seed(0)
    x = torch.randn((7, 3, 128), generator=g).half()
    x[0] = 0
    x[1, :, 5] = 900
    x[2] = 1.5
    x[3] *= 1e-6
    rows = Q.pack(x)
    assert rows.shape == (7, 3, 80) and rows.dtype == torch.uint8
    v = Q.values(rows)
    group = x.double().unflatten(-1, (4, 32))
    span, top = group.amax(-1) - group.amin(-1), group.abs().amax(-1)
    # half a step of span / 15, and the fp16 roundings of centre (2^-11 |centre|, 2^-25 at least) and scale (7.5 of the same)
    tol = span / 30 * 1.001 + 2.0 ** -11 * top + 8.5 * 2.0 ** -25 + 7.5 * 2.0 ** -11 * span / 15
    assert bool(((v - x.double()).unflatten(-1, (4, 32)).abs().amax(-1) <= tol).all())
    assert bool((v[0] == 0).all()) and bool((v[2] == 1.5).all())
    x[4, 1, 33] = float("nan")
    x[5, 0, 127] = float("-inf")
    v = Q.values(Q.pack(x))
    assert bool(v[4, 1, 32:64].isnan().all()) and int(v.isnan().sum()) == 64 and bool(v[5, 0, 96:].isnan().all())
    # the first value's code is the low nibble of byte 0, value 32's of byte 4, value 8's of byte 16
    y = torch.zeros(128).half()
    y[0], y[32], y[8] = 15.0, 15.0, 15.0
    r = Q.pack(y).numpy()
    assert r[0] == 0x0F and r[4] == 0x0F and r[16] == 0x0F
    assert np.frombuffer(r[64:72].tobytes(), np.float16).tolist() == [7.5, 1.0, 7.5, 1.0]
