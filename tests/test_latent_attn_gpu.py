"""Latent attention on the GPU, absorbed (cascade_latent_decode) and expanded
(cascade_latent_prefill), against the formula in 64 bits.

Tolerances, per output element, from the arithmetic the kernels may use:
  * every score is a dot product of n = 576 (192) products summed in fp32 in
    any order: |ds| <= n 2^-24 scale sum|q||k| =: ds, and a softmax weight is
    off by a factor of at most exp(2 ds);
  * the weights may be rounded to the inputs' type before the second product
    (unit roundoff u = 2^-8 for bf16's 8
    significant bits, 2^-11 for fp16's 11): |dO| <= u sum_t p_t |v_t|; exponentials
    and fp32 sums add less than 2^-17 of the same sum;
  * the output is rounded once to its type: u |O|.
The log-sum-exp is off by at most ds + 2^-18 (1 + |lse|).
"""
import numpy as np
import pytest

import helpers as Hh

pytestmark = pytest.mark.gpu

SCALE = 192 ** -0.5
U = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11}


def _dtype(name):
    import torch
    return {"bf16": torch.bfloat16, "fp16": torch.float16}[name]


def _attend(q, k, v, first, causal, scale, dtype):
    """q [n, d], k [m, d], v [m, e] in float64: (out, lse, tol_out, tol_lse)."""
    n, m = q.shape[0], k.shape[0]
    e = v.shape[1]
    out, lse = np.zeros((n, e)), np.full(n, -np.inf)
    tol, tol_l = np.full((n, e), 0.0), np.zeros(n)
    if m == 0:
        return out, lse, tol, tol_l
    s = scale * q @ k.T
    ds = q.shape[1] * 2.0 ** -24 * scale * (np.abs(q) @ np.abs(k).T)
    seen = np.ones((n, m), bool)
    if causal:
        seen = np.arange(m)[None, :] <= first + np.arange(n)[:, None]
    s = np.where(seen, s, -np.inf)
    rows = seen.any(1)
    top = np.where(rows, s.max(1, initial=-np.inf), 0.0)
    p = np.exp(s - top[:, None])
    tot = p.sum(1)
    p /= np.where(rows, tot, 1.0)[:, None]
    ds = np.where(seen, ds, 0).max(1, initial=0.0)
    out = p @ v
    lse = np.where(rows, np.log(np.where(rows, tot, 1.0)) + top, -np.inf)
    u = U[dtype]
    mag = p @ np.abs(v)
    tol = u * np.abs(out) + (u + 2.0 ** -17 + 2 * ds[:, None]) * mag + 2.0 ** -24
    tol_l = np.where(rows, ds + 2.0 ** -18 * (1 + np.abs(np.where(rows, lse, 0))), 0)
    return out, lse, tol, tol_l


def _check(got_o, got_l, want):
    out, lse, tol, tol_l = want
    assert np.isfinite(got_o).all()
    bad = np.abs(got_o - out) > tol
    assert not bad.any(), (int(bad.sum()), float(np.abs(got_o - out).max()), np.argwhere(bad)[:4].tolist())
    inf = np.isinf(lse)
    assert np.array_equal(np.isneginf(got_l), inf)
    assert (np.abs(got_l[~inf] - lse[~inf]) <= tol_l[~inf]).all()


def _decode_inputs(kv_lens, q_lens, heads, page, dtype, seed=0, q_scale=1.5, spare=1, poison=True):
    """Query rows, a shuffled page pool whose unused rows hold NaN and infinities, and the tables."""
    import torch
    rng = np.random.default_rng(seed)
    need = [(n + page - 1) // page for n in kv_lens]
    blocks = sum(need) + spare
    cols = max(1, max(need, default=1))
    order = rng.permutation(blocks)
    bt = np.full((len(kv_lens), cols), -1, np.int32)
    g = torch.Generator(device="cuda").manual_seed(seed)
    cache = torch.randn((blocks, page, 576), generator=g, device="cuda").to(_dtype(dtype))
    used = torch.zeros((blocks, page), dtype=torch.bool)
    c = 0
    for b, n in enumerate(kv_lens):
        for j in range(need[b]):
            bt[b, j] = order[c]
            used[order[c], : min(page, n - j * page)] = True
            c += 1
    if poison:
        free = ~used.cuda()
        cache[free] = float("nan")
        free[:, ::2] = False
        cache[free] = float("inf")
    q = (torch.randn((sum(q_lens), heads, 576), generator=g, device="cuda") * q_scale).to(_dtype(dtype))
    i64 = dict(dtype=torch.int64, device="cuda")
    return q, cache, torch.from_numpy(bt).cuda(), torch.tensor(q_lens, **i64), torch.tensor(kv_lens, **i64)


def _decode_want(q, cache, bt, q_lens, kv_lens, causal, dtype, scale=SCALE):
    page = cache.shape[1]
    q64, cache = Hh.dev_to_f64(q), cache.float().cpu().numpy().astype(np.float64)
    bt, outs, at = bt.cpu().numpy(), [], 0
    for b, (n, m) in enumerate(zip(q_lens.tolist(), kv_lens.tolist())):
        kv = cache[bt[b, : (m + page - 1) // page]].reshape(-1, 576)[:m]
        H = q64.shape[1]
        mine = [_attend(q64[at : at + n, h], kv, kv[:, :512], m - n, causal, scale, dtype) for h in range(H)]
        outs.append([np.stack([w[i] for w in mine], 1) for i in range(4)])
        at += n
    return [np.concatenate([o[i] for o in outs]) for i in range(4)]


def _decode(q, cache, bt, qs, kvs, q_value, causal=True, scale=SCALE):
    return Hh.ops().cascade_latent_decode(q, cache, bt, qs, kvs, q_value, scale, causal)


def _decode_case(kv_lens, q_lens, heads, page, dtype, causal=True, uniform=True, **kw):
    Hh.need_cuda()
    q, cache, bt, qs, kvs = _decode_inputs(kv_lens, q_lens, heads, page, dtype, **kw)
    out, lse = _decode(q, cache, bt, qs, kvs, q_lens[0] if uniform else 0, causal)
    T, H, _ = q.shape
    assert out.dtype == q.dtype and tuple(out.shape) == (T, H, 512) and tuple(lse.shape) == (T * H,)
    want = _decode_want(q, cache, bt, qs, kvs, causal, dtype)
    _check(Hh.dev_to_f64(out), Hh.dev_to_f64(lse).reshape(T, H), want)


EDGES = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 95, 96, 97, 127, 128, 129, 191, 193, 255, 257]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("page", [16, 64])
def test_decode_lengths_around_tiles(page, dtype):
    _decode_case(EDGES, [1] * len(EDGES), 4, page, dtype)


@pytest.mark.parametrize("heads", [1, 3, 16, 20, 64, 65, 127, 128, 129, 200])
def test_decode_head_counts(heads):
    _decode_case([70, 1, 333], [1, 1, 1], heads, 32, "bf16")


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256, 512])
def test_decode_page_sizes(page):
    _decode_case([1, 700, 513, 64], [1] * 4, 16, page, "bf16", seed=page)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("q_len,heads", [(2, 16), (4, 128), (5, 20), (9, 64), (40, 8)])
def test_decode_drafted_tokens(q_len, heads, causal):
    # lengths below q_len leave the first tokens' rows empty when causal
    kv = [0, 1, q_len - 1, q_len, q_len + 1, 64 + q_len, 211]
    _decode_case(kv, [q_len] * len(kv), heads, 16, "bf16", causal=causal, seed=q_len)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_decode_ragged_queries(dtype):
    _decode_case([100, 3, 0, 65, 400, 1], [3, 1, 2, 7, 0, 1], 24, 32, dtype, uniform=False)


def test_decode_long_sequence_splits_over_the_gpu():
    _decode_case([20011], [1], 16, 64, "bf16")
    _decode_case([9001, 5], [2, 2], 128, 64, "bf16")


def test_decode_many_requests():
    rng = np.random.default_rng(3)
    kv = rng.integers(0, 300, 400).tolist()
    _decode_case(kv, [1] * 400, 4, 32, "bf16")


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_decode_sharp_and_rising_scores(dtype):
    """Scores of hundreds, rising along the sequence: the running maximum moves by far more than an exponent holds."""
    import torch
    Hh.need_cuda()
    n = 700
    q, cache, bt, qs, kvs = _decode_inputs([n, n], [1, 1], 16, 64, dtype, q_scale=1.0)
    ramp = torch.linspace(-30, 30, n, device="cuda")
    flat = cache.view(-1, 576)
    for b in range(2):
        rows = (bt[b].long()[:, None] * 64 + torch.arange(64, device="cuda")).reshape(-1)[:n]
        flat[rows, 5] = (ramp if b == 0 else -ramp).to(cache.dtype)
    q[:, :, 5] = 100.0
    out, lse = _decode(q, cache, bt, qs, kvs, 1)
    _check(Hh.dev_to_f64(out), Hh.dev_to_f64(lse).reshape(2, 16), _decode_want(q, cache, bt, qs, kvs, True, dtype))


def test_decode_empty_calls():
    import torch
    Hh.need_cuda()
    q, cache, bt, qs, kvs = _decode_inputs([5], [1], 4, 16, "bf16")
    out, lse = _decode(q[:0], cache, bt[:0], qs[:0], kvs[:0], 1)
    assert out.shape == (0, 4, 512) and lse.numel() == 0
    out, lse = _decode(q, cache, bt[:, :0], qs, kvs, 1)  # no columns: every length is cut to 0
    assert float(out.abs().max()) == 0 and torch.isneginf(lse).all()


def test_decode_bad_page_reads_as_zeros():
    import torch
    Hh.need_cuda()
    C = Hh.capi()
    q, cache, bt, qs, kvs = _decode_inputs([130, 64], [1, 1], 8, 32, "bf16")
    assert C.device_error() == 0
    keep = int(bt[0, 1])
    bt[0, 1] = cache.shape[0] + 7
    out, lse = _decode(q, cache, bt, qs, kvs, 1)
    assert C.device_error() & 2 and C.device_error() == 0
    zero = cache.clone()
    zero[keep] = 0
    bt[0, 1] = keep
    want = _decode_want(q, zero, bt, qs, kvs, True, "bf16")
    _check(Hh.dev_to_f64(out), Hh.dev_to_f64(lse).reshape(2, 8), want)


def test_decode_cache_past_32_bit_offsets():
    """Pages at the end of a cache of more than 2^31 elements (and 2^32 bytes)."""
    import torch
    Hh.need_cuda()
    page, blocks = 64, (1 << 31) // (64 * 576) + 100
    q, small, bt, qs, kvs = _decode_inputs([200, 64], [1, 1], 16, page, "bf16")
    cache = torch.empty((blocks, page, 576), dtype=torch.bfloat16, device="cuda")
    shift = blocks - small.shape[0]
    cache[shift:] = small
    out, lse = _decode(q, cache, torch.where(bt < 0, bt, bt + shift).int(), qs, kvs, 1)
    _check(Hh.dev_to_f64(out), Hh.dev_to_f64(lse).reshape(2, 16), _decode_want(q, small, bt, qs, kvs, True, "bf16"))


def test_decode_repeats_bit_for_bit_on_streams_and_in_a_graph():
    import torch
    Hh.need_cuda()
    args = _decode_inputs([900, 64, 2000, 1], [2] * 4, 32, 64, "bf16")
    out, lse = _decode(*args, 2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o2, l2 = _decode(*args, 2)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            o3, l3 = _decode(*args, 2)
        g.replay()
    side.synchronize()
    for o, l in ((o2, l2), (o3, l3)):
        assert torch.equal(o, out) and torch.equal(l, lse)


def test_decode_prefix_and_suffix_merge():
    """A prefix shared by a batch (read once, as one request of B query tokens) and each request's own suffix,
    merged by cascade_lse_merge, is attention over both."""
    import torch
    Hh.need_cuda()
    B, H, page, P = 6, 16, 32, 333
    suffix = [0, 1, 40, 64, 100, 7]
    q, cache, bt, qs, kvs = _decode_inputs([P] + suffix, [B] + [0] * B, H, page, "bf16")
    ones = torch.ones(B, dtype=torch.int64, device="cuda")
    o1, l1 = _decode(q, cache, bt[:1], qs[:1], kvs[:1], B, causal=False)
    o2, l2 = _decode(q, cache, bt[1:].contiguous(), ones, kvs[1:].contiguous(), 1)
    out = Hh.ops().cascade_lse_merge(o1, o2, l1, l2, 2)
    c64, bt = cache.float().cpu().numpy().astype(np.float64), bt.cpu().numpy()
    q64 = Hh.dev_to_f64(q)

    def rows(b, n):
        return c64[bt[b, : (n + page - 1) // page]].reshape(-1, 576)[:n]

    for b in range(B):
        kv = np.concatenate([rows(0, P), rows(b + 1, suffix[b])])
        w = _attend(q64[b], kv, kv[:, :512], 0, False, SCALE, "bf16")
        # each side was rounded to bf16 before the merge as well
        assert (np.abs(Hh.dev_to_f64(out)[b] - w[0]) <= 2 * w[2]).all()


@pytest.mark.parametrize("heads,kv", [(16, [90, 200, 5]), (128, [6000, 70, 131])])
@pytest.mark.parametrize("bad", ["nan", "inf"])
def test_decode_nan_in_a_seen_row_reaches_the_output(bad, heads, kv):
    """A NaN key, or a score of +inf, makes the softmax of its request NaN; the others' stay."""
    import torch
    Hh.need_cuda()
    q, cache, bt, qs, kvs = _decode_inputs(kv, [1] * 3, heads, 32, "bf16", poison=False)
    q[:, :, 520] = 1.0
    cache[:, :, 520] = 0.0
    at = kv[0] - 7
    cache[int(bt[0, at // 32]), at % 32, 520] = float(bad)  # a rotary value: the product with V has none
    want = _decode_want(q[1:], cache, bt[1:], qs[1:], kvs[1:], True, "bf16")
    out, lse = _decode(q, cache, bt, qs, kvs, 1)
    lse = lse.view(3, heads)
    assert torch.isnan(out[0]).all() and torch.isnan(lse[0]).all()
    _check(Hh.dev_to_f64(out)[1:], Hh.dev_to_f64(lse)[1:], want)


# ---------------------------------------------------------------- expanded


def _prefill_inputs(pairs, heads, dtype, layout="joint", seed=0, q_scale=1.5):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    T, S = sum(a for a, _ in pairs), sum(b for _, b in pairs)

    def rand(*shape):
        return torch.randn(shape, generator=g, device="cuda").to(_dtype(dtype))

    q = (torch.randn((T, heads, 192), generator=g, device="cuda") * q_scale).to(_dtype(dtype))
    if layout == "joint":        # as one up-projection writes them
        k, v = rand(S, heads, 256).split(128, -1)
        rope = rand(S, 64)
    elif layout == "heads":      # head-major, rope a slice of the cache rows
        k, v = rand(heads, S, 128).transpose(0, 1), rand(heads, S, 128).transpose(0, 1)
        rope = rand(S, 576)[:, 512:]
    else:
        k, v, rope = rand(S, heads, 128), rand(S, heads, 128), rand(S, 64)
    cu = [torch.tensor([0] + [p[i] for p in pairs], dtype=torch.int64).cumsum(0).cuda() for i in (0, 1)]
    return q, k, rope, v, cu[0], cu[1]


def _prefill_want(args, causal, dtype, scale=SCALE):
    q, k, rope, v = (Hh.dev_to_f64(t) for t in args[:4])
    cq, ck = args[4].tolist(), args[5].tolist()
    T, H, _ = q.shape
    want = [np.zeros((T, H, 128)), np.full((T, H), -np.inf), np.zeros((T, H, 128)), np.zeros((T, H))]
    for b in range(len(cq) - 1):
        qs, ks = slice(cq[b], cq[b + 1]), slice(ck[b], ck[b + 1])
        n, m = cq[b + 1] - cq[b], ck[b + 1] - ck[b]
        for h in range(H):
            key = np.concatenate([k[ks, h], rope[ks]], 1)
            w = _attend(q[qs, h], key, v[ks, h], m - n, causal, scale, dtype)
            for i in range(4):
                want[i][qs, h] = w[i]
    return want


def _prefill_case(pairs, heads, dtype, causal=True, layout="joint", **kw):
    Hh.need_cuda()
    args = _prefill_inputs(pairs, heads, dtype, layout, **kw)
    out, lse = Hh.ops().cascade_latent_prefill(*args, max(a for a, _ in pairs), SCALE, causal)
    T = args[0].shape[0]
    assert out.dtype == args[0].dtype and tuple(out.shape) == (T, heads, 128)
    _check(Hh.dev_to_f64(out), Hh.dev_to_f64(lse).reshape(T, heads), _prefill_want(args, causal, dtype))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("causal", [True, False])
def test_prefill_lengths_around_tiles(causal, dtype):
    sizes = [1, 2, 63, 64, 65, 127, 128, 129, 255, 256, 257, 383, 513]
    _prefill_case([(n, n) for n in sizes], 2, dtype, causal)


@pytest.mark.parametrize("causal", [True, False])
def test_prefill_chunks_and_empty_rows(causal):
    """Context before the chunk; fewer keys than queries (rows that see nothing); no keys; no queries."""
    _prefill_case([(5, 300), (130, 131), (300, 5), (129, 128), (7, 0), (0, 9), (1, 777), (256, 1024)], 3, "bf16", causal)


@pytest.mark.parametrize("layout", ["joint", "heads", "plain"])
@pytest.mark.parametrize("heads", [1, 5, 16])
def test_prefill_layouts_and_heads(heads, layout):
    _prefill_case([(100, 100), (33, 200)], heads, "bf16", layout=layout, seed=heads)


def test_prefill_long():
    _prefill_case([(2000, 2000), (900, 1901)], 2, "bf16")


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_prefill_sharp_scores(dtype):
    _prefill_case([(300, 700)], 2, dtype, q_scale=40.0)


def test_prefill_rising_scores():
    import torch
    Hh.need_cuda()
    for sign in (1, -1):
        args = _prefill_inputs([(300, 900)], 2, "bf16", "plain", q_scale=1.0)
        args[1][:, :, 3] = sign * torch.linspace(-30, 30, 900, device="cuda")[:, None]
        args[0][:, :, 3] = 100.0
        out, lse = Hh.ops().cascade_latent_prefill(*args, 300, SCALE, True)
        _check(Hh.dev_to_f64(out), Hh.dev_to_f64(lse).reshape(300, 2), _prefill_want(args, True, "bf16"))


def test_prefill_sequences_do_not_touch_each_other():
    """What another sequence holds, NaN and infinities included, does not reach a sequence's rows."""
    import torch
    Hh.need_cuda()
    pairs = [(70, 70), (50, 61), (90, 90)]
    args = _prefill_inputs(pairs, 2, "bf16", "plain")
    want = _prefill_want(args, True, "bf16")
    for t, bad in ((args[1], float("inf")), (args[2], float("nan")), (args[3], float("nan"))):
        t[70:131] = bad
    args[0][70:120] = float("nan")
    out, lse = Hh.ops().cascade_latent_prefill(*args, 90, SCALE, True)
    keep = np.r_[0:70, 120:210]
    _check(Hh.dev_to_f64(out)[keep], Hh.dev_to_f64(lse).reshape(210, 2)[keep], [w[keep] for w in want])


@pytest.mark.parametrize("at", [0, 2, 3, 66, 130, 255])
def test_prefill_nan_in_a_seen_key_reaches_the_output(at):
    import torch
    Hh.need_cuda()
    args = _prefill_inputs([(256, 256), (40, 40)], 2, "bf16", "plain")
    want = _prefill_want(args, True, "bf16")
    args[2][at, 5] = float("nan")  # rotary key: the values stay finite
    out, lse = Hh.ops().cascade_latent_prefill(*args, 256, SCALE, True)
    lse = lse.view(296, 2)
    assert torch.isnan(out[at:256]).all() and torch.isnan(lse[at:256]).all()
    keep = np.r_[0:at, 256:296]
    _check(Hh.dev_to_f64(out)[keep], Hh.dev_to_f64(lse)[keep], [w[keep] for w in want])


def test_prefill_max_length_may_be_larger():
    import torch
    Hh.need_cuda()
    args = _prefill_inputs([(40, 40), (3, 9)], 2, "bf16")
    a = Hh.ops().cascade_latent_prefill(*args, 40, SCALE, True)
    b = Hh.ops().cascade_latent_prefill(*args, 4000, SCALE, True)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_prefill_repeats_bit_for_bit_on_streams_and_in_a_graph():
    import torch
    Hh.need_cuda()
    args = _prefill_inputs([(300, 500), (20, 20)], 4, "bf16")
    out, lse = Hh.ops().cascade_latent_prefill(*args, 300, SCALE, True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            o2, l2 = Hh.ops().cascade_latent_prefill(*args, 300, SCALE, True)
        g.replay()
    side.synchronize()
    assert torch.equal(o2, out) and torch.equal(l2, lse)


def test_both_forms_agree_on_one_token():
    """The expanded form over up-projected latents is the absorbed form with the projections folded into the query
    and the output (random projections, one sequence)."""
    import torch
    Hh.need_cuda()
    H, n = 4, 150
    g = torch.Generator(device="cuda").manual_seed(1)

    def rand(*shape, s=1.0):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float64) * s

    c, rope, qn, qr = rand(n, 512), rand(n, 64), rand(1, H, 128), rand(1, H, 64)
    wk, wv = rand(H, 128, 512, s=512 ** -0.5), rand(H, 128, 512, s=512 ** -0.5)
    bf = torch.bfloat16
    k = torch.einsum("tc,hdc->thd", c, wk).to(bf)
    v = torch.einsum("tc,hdc->thd", c, wv).to(bf)
    cu = [torch.tensor([0, m], dtype=torch.int64, device="cuda") for m in (1, n)]
    a, la = Hh.ops().cascade_latent_prefill(torch.cat([qn, qr], -1).to(bf), k, rope.to(bf), v, *cu, 1, SCALE, True)
    cache = torch.zeros((10, 16, 576), dtype=bf, device="cuda")
    cache.view(-1, 576)[:n] = torch.cat([c, rope], -1).to(bf)
    q = torch.cat([torch.einsum("thd,hdc->thc", qn, wk), qr], -1).to(bf)
    i64 = dict(dtype=torch.int64, device="cuda")
    b, lb = _decode(q, cache, torch.arange(10, dtype=torch.int32, device="cuda").view(1, 10), torch.ones(1, **i64),
                    torch.tensor([n], **i64), 1)
    b = torch.einsum("thc,hdc->thd", b.double(), wv)
    # inputs, projections and outputs rounded to bf16 (2^-9 each) at score magnitudes of about 20
    assert float((a.double() - b).abs().max()) < 0.1 and float((la - lb).abs().max()) < 0.1


# ---------------------------------------------------------------- refusals


def test_decode_refusals():
    import torch
    Hh.need_cuda()
    q, cache, bt, qs, kvs = _decode_inputs([20, 30], [1, 1], 4, 16, "bf16", poison=False)
    bad = [
        ((q.float(), cache, bt, qs, kvs, 1), "bf16 or fp16"),
        ((q, cache.half(), bt, qs, kvs, 1), "cache must be"),
        ((q[:, :, :512].contiguous(), cache, bt, qs, kvs, 1), "576"),
        ((q, cache[:, :15].contiguous(), bt, qs, kvs, 1), "blockSize"),
        ((q.transpose(0, 1), cache, bt, qs, kvs, 1), "contiguous"),
        ((q, cache, bt.long(), qs, kvs, 1), "block_table must be"),
        ((q, cache, bt[:1], qs, kvs, 1), "row per request"),
        ((q, cache, bt, qs.int(), kvs, 1), "actual_q_seqlens must be"),
        ((q, cache, bt, qs, kvs[:1], 1), "batch entries"),
        ((q, cache, bt, qs, kvs, 2), "batch \\* q_seqlen_value"),
        ((q, cache, bt, qs, kvs, -1), "q_seqlen_value must be >= 0"),
        ((q, cache.cpu(), bt, qs, kvs, 1), "must be on"),
    ]
    for args, text in bad:
        with pytest.raises(RuntimeError, match=text):
            Hh.ops().cascade_latent_decode(*args, SCALE, True)
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(RuntimeError, match="scale must be positive"):
            Hh.ops().cascade_latent_decode(q, cache, bt, qs, kvs, 1, scale, True)
    assert Hh.capi().device_error() == 0


def test_prefill_refusals():
    import torch
    Hh.need_cuda()
    q, k, r, v, cq, ck = _prefill_inputs([(4, 4)], 2, "bf16", "plain")
    odd = torch.zeros((4, 2, 129), dtype=torch.bfloat16, device="cuda")[:, :, :128]
    bad = [
        ((q.float(), k, r, v, cq, ck, 4), "bf16 or fp16"),
        ((q, k.half(), r, v, cq, ck, 4), "query's type"),
        ((q[..., :128].contiguous(), k, r, v, cq, ck, 4), "192"),
        ((q, k[:, :1], r, v, cq, ck, 4), "key must be"),
        ((q, k, r[:3], v, cq, ck, 4), "key_rope must be"),
        ((q, k, r, v[:, :, :64], cq, ck, 4), "value must be"),
        ((q, k, r, v, cq.int(), ck, 4), "cu_q_seqlens must be"),
        ((q, k, r, v, cq, ck[:1], 4), "batch \\+ 1"),
        ((q, odd, r, v, cq, ck, 4), "multiples of 8"),
        ((q, k, r, v, cq, ck, 0), "max_q_seqlen"),
        ((q, k, r, v.transpose(1, 2).contiguous().transpose(1, 2), cq, ck, 4), "last dimension"),
    ]
    for args, text in bad:
        with pytest.raises(RuntimeError, match=text):
            Hh.ops().cascade_latent_prefill(*args, SCALE, True)
