"""The paged latent cache's operators together: the speculative example, a shared prefix, and attention calls whose
bounded waits run out."""
import importlib.util
import os
import time

import numpy as np
import pytest

import helpers as Hh
from conftest import ROOT

pytestmark = pytest.mark.gpu


def _example():
    spec = importlib.util.spec_from_file_location("latent_speculative", os.path.join(ROOT, "examples", "latent_speculative.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


@pytest.mark.parametrize("samples,prompt,page", [(6, 700, 64), (3, 64, 16)])
def test_speculative_example(samples, prompt, page):
    import torch
    Hh.need_cuda()
    r = _example().run(samples=samples, prompt=prompt, page=page, log=lambda *_: None)
    # queries, keys, values and two outputs rounded to bf16 (2^-8 each) on sums of hundreds of terms
    assert r["gap"] < 0.05
    cache = r["cache"]
    # the counts are exactly the table's references, the live pages the first ones
    flat = cache.table[cache.table >= 0].long()
    assert torch.equal(torch.bincount(flat, minlength=cache.refs.numel()).int(), cache.refs)
    assert int((cache.refs[: r["live"]] > 0).sum()) == r["live"] == int((cache.refs > 0).sum())
    assert torch.equal(cache.lens, r["keep"])
    for out in r["produced"][1:]:
        assert int((out >= 0).sum(1).min()) >= 1 and int(out.max()) < 2000
    assert Hh.capi().device_error() == 0


def test_shared_prefix_step_equals_each_row_by_itself():
    import torch
    Hh.need_cuda()
    from cascade_kernel.latent import LatentCache
    g = torch.Generator(device="cuda").manual_seed(0)
    page, P, B, H = 32, 320, 5, 16
    cache = LatentCache(1, 60, page, 1, 16)
    cache.grow(torch.tensor([P], device="cuda"))
    cache.write(0, torch.randn((P, 576), generator=g, device="cuda").bfloat16(), [P])
    prefix = cache.table[:, : P // page].contiguous()
    cache.fork(torch.zeros(B, dtype=torch.int64, device="cuda"))
    own = [1, 40, 32, 7, 100]
    cache.grow(torch.tensor(own, device="cuda"))
    cache.write(0, torch.randn((sum(own), 576), generator=g, device="cuda").bfloat16(), own)
    q = torch.randn((B, H, 576), generator=g, device="cuda").bfloat16()
    scale = 192 ** -0.5
    one, _ = cache.attend(0, q, 1, scale)
    two = cache.attend_shared(0, q, prefix, torch.tensor([P], dtype=torch.int64, device="cuda"), scale, P)
    # the same values but for P's and the partial outputs' rounding to bf16, each 2^-8 of sums of |p v| <= max|v| ~ 4
    assert float((one.float() - two.float()).abs().max()) <= 4 * 2.0 ** -8 * 4
    with pytest.raises(ValueError, match="whole pages"):
        cache.attend_shared(0, q, prefix, torch.tensor([P], dtype=torch.int64, device="cuda"), scale, P + 1)
    with pytest.raises(RuntimeError, match="pages needed"):
        cache.grow(torch.full((B,), 10000, device="cuda"))


def _inputs():
    import torch
    g = torch.Generator(device="cuda").manual_seed(1)
    i64 = dict(dtype=torch.int64, device="cuda")
    kv = [900, 64, 3]
    q = torch.randn((3, 16, 576), generator=g, device="cuda").bfloat16()
    cache = torch.randn((45, 64, 576), generator=g, device="cuda").bfloat16()
    bt = torch.arange(45, dtype=torch.int32, device="cuda").view(3, 15)
    return q, cache, bt, torch.ones(3, **i64), torch.tensor(kv, **i64)


def test_stalled_decode_ends_with_an_error_status():
    import torch
    Hh.need_cuda()
    C = Hh.capi()
    args = _inputs()
    out, lse = torch.empty((3, 16, 512), dtype=torch.bfloat16, device="cuda"), torch.empty(48, device="cuda")

    def call(flags):
        d = C.latent_desc(*args, 1, 192 ** -0.5, flags=flags)
        ws = torch.empty(C.latent_decode_workspace_size(d), dtype=torch.uint8, device="cuda")
        C.latent_decode(d, out, lse, ws)
        torch.cuda.synchronize()

    call(0)
    want = out.clone()
    assert C.device_error() == 0
    t = time.perf_counter()
    call(C.FLAG_DEBUG_STALL)
    assert time.perf_counter() - t < 5.0
    assert C.device_error() & 1
    call(0)
    assert C.device_error() == 0 and torch.equal(out, want)


def test_stalled_prefill_ends_with_an_error_status():
    import ctypes
    import torch
    Hh.need_cuda()
    C = Hh.capi()
    g = torch.Generator(device="cuda").manual_seed(2)
    n, H = 300, 2
    q = torch.randn((n, H, 192), generator=g, device="cuda").bfloat16()
    k, v = (torch.randn((n, H, 128), generator=g, device="cuda").bfloat16() for _ in range(2))
    r = torch.randn((n, 64), generator=g, device="cuda").bfloat16()
    cu = torch.tensor([0, n], dtype=torch.int64, device="cuda")
    out, lse = torch.empty((n, H, 128), dtype=torch.bfloat16, device="cuda"), torch.empty(n * H, device="cuda")

    def call(flags):
        d = C.LatentPrefill()
        for name, t in (("query", q), ("key", k), ("key_rope", r), ("value", v), ("cu_q_seqlens", cu), ("cu_kv_seqlens", cu)):
            setattr(d, name, t.data_ptr())
        d.num_tokens = d.num_kv = d.max_q_seqlen = n
        d.num_heads, d.batch = H, 1
        d.key_token_stride = d.value_token_stride = H * 128
        d.key_head_stride = d.value_head_stride = 128
        d.rope_token_stride = 64
        d.scale, d.causal, d.dtype, d.flags = 192 ** -0.5, 1, C.BF16, flags
        C.check(C.load().cascade_latent_prefill(ctypes.byref(d), out.data_ptr(), lse.data_ptr(), C.stream_ptr()))
        torch.cuda.synchronize()

    call(0)
    want = out.clone()
    assert C.device_error() == 0
    t = time.perf_counter()
    call(C.FLAG_DEBUG_STALL)
    assert time.perf_counter() - t < 5.0
    assert C.device_error() & 1
    call(0)
    assert C.device_error() == 0 and torch.equal(out, want)


def test_head_stride_of_zero_shares_keys_and_values():
    """Expanded keys and values broadcast over the heads (stride 0) give what the copies give."""
    import torch
    Hh.need_cuda()
    g = torch.Generator(device="cuda").manual_seed(3)
    n, H = 150, 4
    q = torch.randn((n, H, 192), generator=g, device="cuda").bfloat16()
    k, v = (torch.randn((n, 1, 128), generator=g, device="cuda").bfloat16() for _ in range(2))
    r = torch.randn((n, 64), generator=g, device="cuda").bfloat16()
    cu = torch.tensor([0, n], dtype=torch.int64, device="cuda")
    a = Hh.ops().cascade_latent_prefill(q, k.expand(n, H, 128), r, v.expand(n, H, 128), cu, cu, n, 192 ** -0.5, True)
    b = Hh.ops().cascade_latent_prefill(q, k.expand(n, H, 128).contiguous(), r, v.expand(n, H, 128).contiguous(), cu, cu, n,
                                        192 ** -0.5, True)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert np.isfinite(Hh.dev_to_f64(a[0])).all()
