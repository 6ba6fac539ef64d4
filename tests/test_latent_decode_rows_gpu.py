"""cascade_latent_decode over its query-row counts: 16, 32 and more rows per
request take different kernels, so what depends on one is tested for each. The
formula, the inputs and the tolerances are those of test_latent_attn_gpu.py."""
import numpy as np
import pytest

import helpers as Hh
from test_latent_attn_gpu import _check, _decode, _decode_case, _decode_inputs, _decode_want

pytestmark = pytest.mark.gpu

HEADS = [16, 32, 64]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("heads", [15, 16, 17, 31, 32, 33])
def test_row_counts_around_the_kernels(heads, dtype):
    _decode_case([0, 1, 63, 64, 65, 130, 700], [1] * 7, heads, 16, dtype, seed=heads)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("q_len,heads", [(2, 8), (4, 4), (3, 5), (8, 4), (16, 1), (32, 1), (7, 9)])
def test_drafted_rows_share_a_tile(q_len, heads, causal):
    """Several tokens' rows in one tile: their limits differ within it, some see nothing."""
    kv = [0, 1, q_len - 1, q_len, 63, 64, 65, 64 + q_len, 200]
    _decode_case(kv, [q_len] * len(kv), heads, 32, "bf16", causal=causal, seed=q_len)


@pytest.mark.parametrize("seed", range(4))
@pytest.mark.parametrize("heads", [4, 12, 40])
def test_ragged_tokens_and_lengths(heads, seed):
    """Units of one tile and of many, requests without tokens or cache: every run holds some of them."""
    rng = np.random.default_rng(seed)
    n = int(rng.integers(20, 90))
    kv = np.where(rng.random(n) < 0.3, rng.integers(0, 4, n), rng.integers(0, 900, n)).tolist()
    q = rng.integers(0, 6, n).tolist()
    _decode_case(kv, q, heads, 16, "bf16", uniform=False, seed=seed)


@pytest.mark.parametrize("heads", HEADS)
def test_more_requests_than_threads(heads):
    rng = np.random.default_rng(heads)
    _decode_case(rng.integers(0, 200, 700).tolist(), [1] * 700, heads, 32, "bf16")


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("tokens", [64, 65, 4097, 12001])
def test_one_request_over_many_runs(heads, tokens):
    _decode_case([tokens], [1], heads, 64, "bf16")


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("heads", HEADS)
def test_rising_and_falling_scores(heads, dtype):
    import torch
    Hh.need_cuda()
    n = 700
    q, cache, bt, qs, kvs = _decode_inputs([n, n], [1, 1], heads, 64, dtype, q_scale=1.0)
    ramp = torch.linspace(-30, 30, n, device="cuda")
    flat = cache.view(-1, 576)
    for b in range(2):
        rows = (bt[b].long()[:, None] * 64 + torch.arange(64, device="cuda")).reshape(-1)[:n]
        flat[rows, 5] = (ramp if b == 0 else -ramp).to(cache.dtype)
    q[:, :, 5] = 100.0
    q[:, 1::2, 5] = -100.0  # rows of one tile move at different tiles
    out, lse = _decode(q, cache, bt, qs, kvs, 1)
    _check(Hh.dev_to_f64(out), Hh.dev_to_f64(lse).reshape(2, heads), _decode_want(q, cache, bt, qs, kvs, True, dtype))


@pytest.mark.parametrize("heads", HEADS)
def test_repeats_bit_for_bit(heads):
    import torch
    Hh.need_cuda()
    args = _decode_inputs([900, 64, 2000, 1, 0, 3333], [1] * 6, heads, 64, "bf16")
    out, lse = _decode(*args, 1)
    for _ in range(20):
        o, l = _decode(*args, 1)
        assert torch.equal(o, out) and torch.equal(l, lse)


@pytest.mark.parametrize("heads", HEADS)
def test_bad_page_reads_as_zeros(heads):
    Hh.need_cuda()
    C = Hh.capi()
    q, cache, bt, qs, kvs = _decode_inputs([400, 64], [1, 1], heads, 32, "bf16")
    assert C.device_error() == 0
    keep = int(bt[0, 9])
    bt[0, 9] = -5
    out, lse = _decode(q, cache, bt, qs, kvs, 1)
    assert C.device_error() & 2 and C.device_error() == 0
    zero = cache.clone()
    zero[keep] = 0
    bt[0, 9] = keep
    want = _decode_want(q, zero, bt, qs, kvs, True, "bf16")
    _check(Hh.dev_to_f64(out), Hh.dev_to_f64(lse).reshape(2, heads), want)


@pytest.mark.parametrize("heads", [32, 64])
def test_cache_past_32_bit_offsets(heads):
    import torch
    Hh.need_cuda()
    page, blocks = 64, (1 << 31) // (64 * 576) + 100
    q, small, bt, qs, kvs = _decode_inputs([200, 64], [1, 1], heads, page, "bf16")
    cache = torch.empty((blocks, page, 576), dtype=torch.bfloat16, device="cuda")
    shift = blocks - small.shape[0]
    cache[shift:] = small
    out, lse = _decode(q, cache, torch.where(bt < 0, bt, bt + shift).int(), qs, kvs, 1)
    _check(Hh.dev_to_f64(out), Hh.dev_to_f64(lse).reshape(2, heads), _decode_want(q, small, bt, qs, kvs, True, "bf16"))


@pytest.mark.parametrize("heads", HEADS)
def test_stalled_call_ends_with_an_error_status(heads):
    """A wait that nothing ends runs into its limit; the next call is right again."""
    import torch
    Hh.need_cuda()
    C = Hh.capi()
    q, cache, bt, qs, kvs = _decode_inputs([400, 3, 900], [1] * 3, heads, 32, "bf16")
    out, lse = torch.empty((3, heads, 512), dtype=q.dtype, device="cuda"), torch.empty(3 * heads, device="cuda")

    def call(flags):
        d = C.latent_desc(q, cache, bt, qs, kvs, 1, 192 ** -0.5, flags=flags)
        ws = torch.empty(C.latent_decode_workspace_size(d), dtype=torch.uint8, device="cuda")
        C.latent_decode(d, out, lse, ws)
        torch.cuda.synchronize()

    call(0)
    want = out.clone()
    assert C.device_error() == 0
    call(C.FLAG_DEBUG_STALL)
    assert C.device_error() & 1
    call(0)
    assert C.device_error() == 0 and torch.equal(out, want)
