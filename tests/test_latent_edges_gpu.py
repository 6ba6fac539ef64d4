"""Latent attention where its inputs leave the ordinary: scores of +infinity, large values that a weight of 0 has
to hide, lengths that the tables do not hold."""
import numpy as np
import pytest

import helpers as Hh
from test_latent_attn_gpu import SCALE, _check, _decode, _decode_inputs, _decode_want, _prefill_inputs, _prefill_want

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("at", [0, 2, 3, 5, 6, 7, 34, 66, 97, 130, 255])
def test_prefill_infinite_score_makes_its_rows_nan(at, dtype):
    """A score of +inf: inf - inf under the softmax of every row that sees it, wherever the key lies; the rows before it and
    the other sequence keep theirs."""
    import torch
    Hh.need_cuda()
    args = _prefill_inputs([(256, 256), (40, 40)], 2, dtype, "plain")
    args[0][:, :, 128 + 5] = 1.0
    args[2][:, 5] = 0.0
    want = _prefill_want(args, True, dtype)
    args[2][at, 5] = float("inf")  # a rotary value: the values stay finite
    out, lse = Hh.ops().cascade_latent_prefill(*args, 256, SCALE, True)
    lse = lse.view(296, 2)
    assert torch.isnan(out[at:256]).all() and torch.isnan(lse[at:256]).all()
    keep = np.r_[0:at, 256:296]
    _check(Hh.dev_to_f64(out)[keep], Hh.dev_to_f64(lse)[keep], [w[keep] for w in want])


@pytest.mark.parametrize("hidden", ["by the causal mask", "by its score"])
def test_prefill_weight_of_zero_hides_large_values(hidden):
    """Finite values of 1e38 whose weight is 0, or e^-300 (1e38 e^-300 is far below the tolerance), leave nothing."""
    Hh.need_cuda()
    n, first = 300, 200
    args = _prefill_inputs([(n, n)], 2, "bf16", "plain")
    if hidden == "by its score":
        first = n
        args[0][:, :, 128 + 5] = 1.0
        args[2][:, 5] = 0.0
        args[2][1:n:2, 5] = args[2][2:n:4, 5] = -300 / SCALE
        args[3][1:n:2] = args[3][2:n:4] = 1e38
    want = _prefill_want(args, True, "bf16")
    if hidden == "by the causal mask":
        args[3][first:] = 1e38
    out, lse = Hh.ops().cascade_latent_prefill(*args, n, SCALE, True)
    assert np.array_equal(np.isfinite(Hh.dev_to_f64(out)[:first]), np.ones((first, 2, 128), bool))
    _check(Hh.dev_to_f64(out)[:first], Hh.dev_to_f64(lse).reshape(n, 2)[:first], [w[:first] for w in want])


@pytest.mark.parametrize("heads", [4, 12, 64])
def test_decode_lengths_past_the_table_are_cut(heads):
    """A length past the block table's columns counts as all of them, for the causal mask's end too."""
    Hh.need_cuda()
    q, cache, bt, qs, kvs = _decode_inputs([96, 96, 96], [3] * 3, heads, 32, "bf16", poison=False)
    want = _decode_want(q, cache, bt, qs, kvs, True, "bf16")
    for i, n in enumerate((97, 98, 1 << 62)):
        kvs[i] = n
    out, lse = _decode(q, cache, bt, qs, kvs, 3)
    _check(Hh.dev_to_f64(out), Hh.dev_to_f64(lse).reshape(9, heads), want)


@pytest.mark.parametrize("heads", [4, 8, 64])
def test_decode_tokens_of_no_request_keep_their_rows(heads):
    """Query lengths on the device that add up to less than num_tokens, in a workspace that holds what another call might
    have left: the requests' rows are right, the rest of out and lse is not touched."""
    import torch
    Hh.need_cuda()
    C = Hh.capi()
    kv, lens, T = [1000, 300, 2500], [2, 1, 2], 8
    q, cache, bt, qs, kvs = _decode_inputs(kv, [2, 1, 5], heads, 32, "bf16")
    want = _decode_want(q[:5], cache, bt, torch.tensor(lens), kvs, True, "bf16")
    qs = torch.tensor(lens, dtype=torch.int64, device="cuda")
    d = C.latent_desc(q, cache, bt, qs, kvs, 0, SCALE)
    n = C.latent_decode_workspace_size(d)
    for count, first, row in ((2, 0, 0), (2, 0, 15), (3, 1, 127), (100, 40, 31)):
        ws = torch.full((n // 4,), (count << 17) | (first << 7) | row, dtype=torch.int32, device="cuda")
        out, lse = torch.full((T, heads, 512), 7.0, dtype=q.dtype, device="cuda"), torch.full((T * heads,), 7.0, device="cuda")
        C.latent_decode(d, out, lse, ws)
        assert (out[5:] == 7).all() and (lse[5 * heads:] == 7).all()
        _check(Hh.dev_to_f64(out)[:5], Hh.dev_to_f64(lse).reshape(T, heads)[:5], want)
    assert C.device_error() == 0


@pytest.mark.parametrize("tokens,heads", [(8192, 64), (16384, 16)])
def test_decode_query_lengths_past_the_tokens_are_cut(tokens, heads):
    """Every one of `tokens` requests claims all the tokens, 2^32 rows in all: the first one has them, the others none."""
    import torch
    Hh.need_cuda()
    g = torch.Generator(device="cuda").manual_seed(0)
    n, page = 100, 16
    cache = torch.randn((7, page, 576), generator=g, device="cuda").bfloat16()
    q = torch.randn((tokens, heads, 576), generator=g, device="cuda", dtype=torch.bfloat16)
    bt = torch.arange(7, dtype=torch.int32, device="cuda").expand(tokens, 7).contiguous()
    qs, kvs = (torch.full((tokens,), m, dtype=torch.int64, device="cuda") for m in (tokens, n))
    out, lse = _decode(q, cache, bt, qs, kvs, 0, causal=False)
    pick = torch.randint(0, tokens, (40,), generator=g, device="cuda")
    pick[:2] = torch.tensor([0, tokens - 1])
    one = torch.tensor([40], device="cuda")
    want = _decode_want(q[pick], cache, bt[:1], one, kvs[:1], False, "bf16")
    _check(Hh.dev_to_f64(out[pick]), Hh.dev_to_f64(lse.view(tokens, heads)[pick]), want)
    assert Hh.capi().device_error() == 0


def test_decode_query_lengths_past_the_tokens_in_a_batch():
    """The request in which the tokens end gets what is left of them, as the first of its tokens."""
    import torch
    Hh.need_cuda()
    for heads in (4, 10, 48):
        q, cache, bt, qs, kvs = _decode_inputs([300, 90, 40, 7], [3, 2, 1, 0], heads, 32, "bf16", poison=False)
        want = _decode_want(q, cache, bt, qs, kvs, False, "bf16")
        claim = torch.tensor([3, 2, 9, 1 << 40], dtype=torch.int64, device="cuda")
        out, lse = _decode(q, cache, bt, claim, kvs, 0, causal=False)
        _check(Hh.dev_to_f64(out), Hh.dev_to_f64(lse).reshape(6, heads), want)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_prefill_first_rows_without_keys(dtype):
    """Fewer keys than queries: the first 128 rows of a block see none, the next ones do. The query, which must not show in
    the first rows' zeros, is large; many blocks start at once."""
    import torch
    Hh.need_cuda()
    pairs = [(256, 100), (250, 3), (256, 128), (384, 120), (129, 1)]
    args = _prefill_inputs(pairs, 48, dtype, "plain")
    args[0][:, 2:] = 1000.0
    want = _prefill_want([args[0][:, :2], args[1][:, :2], args[2], args[3][:, :2], *args[4:]], True, dtype)
    first = None
    for _ in range(20):
        out, lse = Hh.ops().cascade_latent_prefill(*args, 384, SCALE, True)
        lse = lse.view(-1, 48)
        at = 0
        for n, m in pairs:
            assert float(out[at:at + n - m].abs().max()) == 0 and torch.isneginf(lse[at:at + n - m]).all()
            at += n
        first = out if first is None else first
        assert torch.equal(out, first)
    _check(Hh.dev_to_f64(out[:, :2]), Hh.dev_to_f64(lse[:, :2]), want)


@pytest.mark.parametrize("batch,q_len,heads", [(1, 75, 128), (150, 1, 16)])
def test_decode_units_that_take_longer_than_a_tenth_of_a_second(batch, q_len, heads):
    """Requests of 8 million cached tokens, the same two pages over and over: the query of the unit after one of them waits
    for 150 ms. Attention over r copies of the tokens is attention over the tokens, its log-sum-exp ln r more.

    Tolerance: sums of 8 million terms in fp32, 16 (values) or 64 (weights) at a time, each addition off by at most 2^-23
    (the tensor cores' may truncate) or 2^-24 of the sum: (2^23 / 16) 2^-23 + (2^23 / 64) 2^-24 = 0.0703 of sum |p v|, which
    the tolerance of one copy holds 2^-8 times at least."""
    import torch
    Hh.need_cuda()
    page, cols = 512, 1 << 14
    n, copies = page * cols, cols // 2
    q, cache, bt, qs, kvs = _decode_inputs([2 * page], [batch * q_len], heads, page, "bf16", poison=False)
    out, lse, tol, tol_l = _decode_want(q, cache, bt, qs, kvs, False, "bf16")
    table = bt.repeat(batch, copies)
    kvs = torch.full((batch,), n, dtype=torch.int64, device="cuda")
    got, got_l = _decode(q, cache, table, torch.full_like(kvs, q_len), kvs, q_len, causal=False)
    assert Hh.capi().device_error() == 0
    off = n / 16 * 2.0 ** -23 + n / 64 * 2.0 ** -24
    _check(Hh.dev_to_f64(got), Hh.dev_to_f64(got_l).reshape(batch * q_len, heads),
           (out, lse + np.log(copies), tol * (1 + 256 * off), tol_l + off + 2.0 ** -18 * np.log(copies)))
