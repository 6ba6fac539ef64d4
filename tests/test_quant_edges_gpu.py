"""Attention over a 4-bit cache where its inputs leave the ordinary: queries and scores of any size, NaN among the values,
small scales, long units beside others, every number of query rows; the write's scales over all of fp16."""
import numpy as np
import pytest

import helpers as Hh
from oracle import quant_oracle as Q
from test_quant_decode_gpu import SCALE, _close, _inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("q_len,G", [(1, 4), (40, 4), (200, 2)])
def test_a_call_behind_a_stalled_one(q_len, G):
    """A call whose bounded waits run out ends with its loads landed and its products done: the one behind it in the stream,
    on the same SMs, is right."""
    import torch
    Hh.need_cuda()
    C = Hh.capi()
    q, kc, vc, table, qs, lens = _inputs([3000] * 20, [q_len] * 20, 2, G, 64, seed=31)
    want = Hh.ops().cascade_quant_decode(q, kc, vc, table, qs, lens, q_len, SCALE, True)
    outs = [(torch.empty_like(want[0]), torch.empty_like(want[1])) for _ in range(2)]
    for _ in range(3):
        for flags, (out, lse) in zip((C.FLAG_DEBUG_STALL, 0), outs):
            d = C.quant_desc(q, kc, vc, table, None, lens, q_len, SCALE, flags=flags)
            ws = torch.zeros(C.quant_decode_workspace_size(d), dtype=torch.uint8, device="cuda")
            C.quant_decode(d, out, lse, ws)
        assert torch.equal(outs[1][0], want[0]) and torch.equal(outs[1][1], want[1])
        assert C.device_error() == 1


@pytest.mark.parametrize("dtype,size,keys", [("fp16", 3e4, 1.0), ("fp16", 6e4, 100.0), ("bf16", 1e7, 1.0), ("bf16", 3e9, 1.0),
                                             ("bf16", 1e12, 1.0), ("bf16", 1e20, 30.0), ("bf16", 1e30, 1.0), ("bf16", 1e35, 1.0),
                                             ("bf16", 1e-30, 100.0)])
@pytest.mark.parametrize("q_len,KVH,G,lens", [(1, 2, 4, [40, 1000, 7]), (4, 1, 5, [333, 90]), (4, 2, 8, [700, 31]),
                                              (40, 1, 4, [100, 2000]), (100, 2, 4, [333, 90])])
def test_scores_of_any_size(q_len, KVH, G, lens, dtype, size, keys):
    """Finite scores, whatever their size: with large ones a single token has all the weight.

    The third token's key is 6 (times `keys`) and more in every value against some 1 of the others, and the query positive, so that
    it wins by half of its score at least; a token that half of the queries see beats it in the same way. All their products
    have one sign: a score is the sum of 17 times 16 of them (scales in two parts, centres), one after the other in fp32, each
    addition off by at most 2^-23 (the tensor cores may truncate); its factor and the logarithm's are 2^-22 of it off."""
    import torch
    Hh.need_cuda()
    args = _inputs(lens, [q_len] * len(lens), KVH, G, 16, dtype, seed=q_len + G, loud=False)
    args[0].copy_((args[0].float().abs().clamp(0.1, 1) * size).to(args[0].dtype))
    par = args[1][..., 64:].contiguous().view(torch.float16)
    par = (par.float() * 0.5 * keys).half().unflatten(-1, (4, 2))
    args[1][..., 64:] = par.flatten(-2).contiguous().view(torch.uint8)
    for b, n in enumerate(lens):
        for t, c in ((2, 6.0 * keys), (n - 1 - q_len // 2, 20.0 * keys)):
            if 0 <= t < n and (t != 2 or n > 3):
                par[int(args[3][b, t // 16]), t % 16, ..., 0] = c
    args[1][..., 64:] = par.flatten(-2).contiguous().view(torch.uint8)
    out, lse, (weight, reach) = Q.attend(args[0], *args[1:4], args[4].tolist(), args[5].tolist(), SCALE, True)
    assert bool((lse.abs() < 2.0 ** 127).all() | lse.isinf().any())
    got = Hh.ops().cascade_quant_decode(*args, q_len, SCALE, True)
    o, l = got[0].double(), got[1].double().view(lse.shape)
    half = torch.finfo(args[0].dtype).eps / 2
    # Large scores: weights of 1 and of e^-1000 and less, so that only the value's rounding (2^-11) and the output's are left.
    # Rows too early to see the third token, and small scores: as everywhere.
    sees = torch.cat([torch.arange(n - q_len, n, device="cuda") >= 2 for n in lens])[:, None]
    ds = torch.where(sees & (size > 1e3), 0.0, reach * 17 * 2.0 ** -23 + 2.0 ** -21)
    tol = out.abs() * half * 1.01 + (2 * 2.0 ** -11 + 2 * ds)[..., None] * 1.05 * weight + 2.0 ** -25
    assert bool(o.isfinite().all()), int(o.isnan().sum())
    assert bool(((o - out).abs() <= tol).all()), float(((o - out).abs() / tol).max())
    seen = lse.isfinite()
    assert torch.equal(l.isfinite(), seen)
    tol = reach * 17 * 2.0 ** -23 + 2.0 ** -21 + 2.0 ** -22 * lse.abs() + 2.0 ** -20
    assert bool(((l - lse).abs() <= tol)[seen].all()), float(((l - lse).abs() / tol)[seen].max())


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("power", [-10, -13, -14, -17, -20, -22, -24])
@pytest.mark.parametrize("q_len,KVH,G", [(1, 2, 4), (4, 1, 5), (40, 1, 4), (64, 2, 5)])
def test_keys_of_small_scales(q_len, KVH, G, power, dtype):
    """Key scales down to fp16's smallest number, met by queries that make scores of ordinary size of them.

    Few query rows: mma.sync aligns its products as if an operand below 2^-14 were 2^-14 (measured; the tiles' products do
    not), so each of a row's 16 products of centres and scales is cut at 2^-23 of 2^-14 times the largest 7.5 |sum q|."""
    import torch
    Hh.need_cuda()
    lens = [100, 333]
    args = _inputs(lens, [q_len] * 2, KVH, G, 16, dtype, seed=-power, loud=False)
    par = args[1][..., 64:].contiguous().view(torch.float16).unflatten(-1, (4, 2))
    used = par[..., 1].isfinite()
    g = torch.Generator(device="cuda").manual_seed(power + 100)
    scale = (1 + torch.rand(used.shape, generator=g, device="cuda")) * 2.0 ** power
    centre = torch.randn(used.shape, generator=g, device="cuda") * 2.0 ** power
    par[..., 0][used], par[..., 1][used] = centre.half()[used], scale.half()[used]
    args[1][..., 64:] = par.flatten(-2).contiguous().view(torch.uint8)
    most = 2.0 ** 14 if dtype == "fp16" else 2.0 ** 21
    q = args[0].float() * min(most, 2.0 ** (-2 - power))
    args[0].copy_((q.clamp(-6e4, 6e4) if dtype == "fp16" else q).to(args[0].dtype))
    scale = SCALE * max(1.0, 2.0 ** (-2 - power) / most)
    want = out, lse, (size, reach) = Q.attend(args[0], *args[1:4], args[4].tolist(), args[5].tolist(), scale, True)
    if q_len * G <= 32:
        sums = args[0].double().unflatten(-1, (4, 32)).sum(-1).abs().amax(-1)
        want = out, lse, (size, reach + 2.0 ** 20 * scale * 16 * 2.0 ** -37 * 7.5 * sums)
    _close(Hh.ops().cascade_quant_decode(*args, q_len, scale, True), args, True, scale, want)


@pytest.mark.parametrize("dtype,size,keys", [("bf16", 1.7e35, 1.0), ("bf16", 1e36, 1.0), ("bf16", 5e37, 2.0 ** -8),
                                             ("bf16", 3e38, 2.0 ** -10), ("bf16", 3.3e38, 2.0 ** -14)])
@pytest.mark.parametrize("q_len,KVH,G,lens", [(1, 2, 4, [40, 1000, 7]), (4, 1, 5, [333, 90]), (4, 2, 8, [700, 31]),
                                              (40, 1, 4, [100, 2000])])
def test_the_largest_queries(q_len, KVH, G, lens, dtype, size, keys):
    """Queries up to bf16's largest number whose scores are finite."""
    test_scores_of_any_size(q_len, KVH, G, lens, dtype, size, keys)


@pytest.mark.parametrize("q_len,G", [(1, 4), (4, 5), (4, 8), (40, 4)])
def test_scores_beyond_fp32_make_their_rows_nan(q_len, G):
    """And leave the other rows as they are."""
    import torch
    Hh.need_cuda()
    args = _inputs([100, 333], [q_len] * 2, 2, G, 16, seed=33)
    clean = Hh.ops().cascade_quant_decode(*args, q_len, SCALE, True)
    args[0][q_len :, 1] = 3e38
    out, lse = Hh.ops().cascade_quant_decode(*args, q_len, SCALE, True)
    assert bool(out[q_len:, 1].isnan().all()) and bool(lse.view(2 * q_len, -1)[q_len:, 1].isnan().all())
    out[q_len:, 1], lse.view(2 * q_len, -1)[q_len:, 1] = clean[0][q_len:, 1], clean[1].view(2 * q_len, -1)[q_len:, 1]
    assert torch.equal(out, clean[0]) and torch.equal(lse, clean[1])


@pytest.mark.parametrize("which", ["one", "two tokens", "last", "every group"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("q_len,KVH,G,lens", [(1, 2, 4, [40, 900, 33]), (1, 1, 8, [20000, 64]), (4, 2, 5, [31, 500]), (4, 1, 8, [600]),
                                              (20, 1, 4, [50, 1000]), (100, 2, 4, [333, 90]), (64, 1, 8, [5000, 700])])
def test_nan_values_leave_the_log_sum_exp(q_len, KVH, G, lens, causal, which):
    """A NaN in a value makes its group's 32 values of `out` NaN for the rows that see it, wherever the token lies, and
    nothing else: the scores do not know it."""
    import torch
    Hh.need_cuda()
    args = _inputs(lens, [q_len] * len(lens), KVH, G, 16, seed=41)
    clean, lse = Hh.ops().cascade_quant_decode(*args, q_len, SCALE, causal)
    want = clean.clone().view(len(lens), q_len, KVH, G, 128)
    for b, n in enumerate(lens):
        at = {"one": [n // 3], "two tokens": [5, n - 1 - q_len // 2], "last": [n - 1], "every group": [n // 2]}[which]
        for i, t in enumerate(at):
            if not 0 <= t < n:
                continue
            groups = range(4) if which == "every group" else [(b + 2 * i) % 4]
            head = (b + i) % KVH
            for g in groups:
                args[2][int(args[3][b, t // 16]), t % 16, head, 64 + 4 * g : 68 + 4 * g] = 0xFF
                first = max(0, t - n + q_len) if causal else 0
                want[b, first:, head, :, 32 * g : 32 * g + 32] = float("nan")
    want = want.view(clean.shape)
    out, again = Hh.ops().cascade_quant_decode(*args, q_len, SCALE, causal)
    assert torch.equal(again, lse)
    assert torch.equal(out.isnan(), want.isnan())
    assert torch.equal(out.nan_to_num(7.0), want.nan_to_num(7.0))


@pytest.mark.parametrize("q_lens", [[36, 200], [36, 100, 300]])
def test_units_that_take_longer_than_a_tenth_of_a_second(q_lens):
    """Requests of 8 million cached tokens (one page over and over) with at most 128 query rows, then one with more, in the same run of a
    CTA: the second half of the last one's rows wait while the others are worked on. Attention over r copies of the
    tokens is attention over the tokens, its log-sum-exp ln r more.

    Tolerance: sums of 8 million terms in fp32, 16 (values) or 64 (weights) at a time, each addition off by at most 2^-23
    (the tensor cores' may truncate) or 2^-24 of the sum: (2^23 / 16) 2^-23 + (2^23 / 64) 2^-24 = 0.0703 of sum p |v|."""
    import torch
    Hh.need_cuda()
    page, KVH, cols = 512, 148, 1 << 14
    n = len(q_lens)
    q, kc, vc, table, qs, lens = _inputs([page] * n, q_lens, KVH, 1, page, "bf16", seed=51)
    out, lse, (size, reach) = Q.attend(q, kc, vc, table, q_lens, [page] * n, SCALE, False)
    table = table[:, :1].repeat(1, cols)
    long = torch.tensor([page * cols] * (n - 1) + [page], device="cuda")
    got, got_l = Hh.ops().cascade_quant_decode(q, kc, vc, table, qs, long, 0, SCALE, False)
    assert Hh.capi().device_error() == 0
    copies = torch.repeat_interleave(long // page, qs)
    off = torch.where(copies > 1, page * cols / 16 * 2.0 ** -23 + page * cols / 64 * 2.0 ** -24, 0.0)[:, None]
    ds = reach * 2.0 ** -20 + 2.0 ** -21
    tol = out.abs() * 2.0 ** -8 * 1.01 + (2 * 2.0 ** -11 + 2 * ds + off)[..., None] * 1.05 * size + 2.0 ** -25
    assert bool(((got.double() - out).abs() <= tol).all())
    lse = lse + torch.log(copies.double())[:, None]
    assert bool(((got_l.double().view(lse.shape) - lse).abs() <= ds + off * 1.05 + 2.0 ** -22 * lse.abs() + 2.0 ** -18 * 10).all())


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("q_len,G", [(5, 5), (4, 7), (31, 1), (4, 8), (1, 32), (25, 1)])
@pytest.mark.parametrize("KVH", [1, 2, 3, 8])
def test_four_blocks_of_query_rows(KVH, q_len, G, causal, dtype):
    """25 to 32 query rows per request and kv head, in units that are whole (the short ones) and cut."""
    import torch
    Hh.need_cuda()
    args = _inputs([33, 5, 3000, 700], [q_len] * 4, KVH, G, 16, dtype, seed=KVH)
    got = Hh.ops().cascade_quant_decode(*args, q_len, SCALE, causal)
    _close(got, args, causal)
    assert Hh.capi().device_error() == 0


@pytest.mark.parametrize("KVH,q_len,G", [(5, 3, 3), (6, 2, 5), (10, 4, 4), (7, 1, 16), (18, 4, 5), (18, 3, 8), (9, 1, 32), (11, 8, 3), (70, 2, 8)])
def test_kv_heads_that_fill_no_group(KVH, q_len, G):
    """The last group of kv heads that share tiles is smaller than the others, with two, three and four blocks of rows."""
    Hh.need_cuda()
    args = _inputs([200, 1, 1500], [q_len] * 3, KVH, G, 32, seed=KVH + G)
    got = Hh.ops().cascade_quant_decode(*args, q_len, SCALE, True)
    _close(got, args, True)
    assert Hh.capi().device_error() == 0


@pytest.mark.parametrize("KVH", [1, 3, 8])
@pytest.mark.parametrize("q_lens", [[7, 7, 7, 6], [1, 26, 0, 1], [20, 1, 4, 1, 9, 7], [100, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1]])
def test_query_lengths_whose_mean_is_four_blocks(q_lens, KVH):
    """Lengths on the device: 25 to 32 rows in the mean, from none to 400 in a request."""
    Hh.need_cuda()
    lens = [(i * 611 + 40) % 2000 for i in range(len(q_lens))]
    args = _inputs(lens, q_lens, KVH, 4, 64, "fp16", seed=61)
    assert 24 < sum(q_lens) * 4 / len(q_lens) <= 32
    got = Hh.ops().cascade_quant_decode(*args, 0, SCALE, True)
    _close(got, args, True)
    assert Hh.capi().device_error() == 0


def test_write_with_every_scale():
    """Groups of every fp16 scale up to the largest that values of +-32768 give, their values next to the borders between codes:
    the bytes are the definition's."""
    import torch
    Hh.need_cuda()
    hi = torch.arange(1, 0x7800 + 1, dtype=torch.int16).view(torch.float16)          # positive fp16 numbers up to 32768
    low = torch.cat([hi, torch.arange(2, 0x7800 + 1, dtype=torch.int16).view(torch.float16), hi[-1:]])
    hi = hi.repeat(2)
    # (hi, -hi) and (hi, -the next): 2 hi / 15 and what lies between two of them
    scale = ((hi.float() + low.float()) / np.float32(15)).half()
    want = torch.arange(1, int(scale.max().view(torch.int16)) + 1, dtype=torch.int16).view(torch.float16)
    assert bool(torch.isin(want.view(torch.int16), scale.view(torch.int16)).all())
    centre = ((hi.float() - low.float()) * 0.5).half().double()
    border = centre[:, None] + (torch.arange(15) - 7.0).double() * scale.double()[:, None]     # between codes n and n + 1
    near = border.half()
    step = torch.where(near.double() > border, -1, 1) * torch.where(near.double() < 0, -1, 1)   # to the border's other side
    bits = near.view(torch.int16)
    other = torch.where(bits & 0x7FFF == 0, bits, (bits + step.short())).view(torch.float16)
    x = torch.cat([hi[:, None], -low[:, None], near, other], 1)
    x = torch.minimum(torch.maximum(x, -low[:, None]), hi[:, None])
    x = x[: x.shape[0] // 4 * 4].reshape(-1, 1, 128).contiguous().cuda()
    x = torch.cat([x, x.flip(0)[:1]]) if x.shape[0] % 2 else x
    T = x.shape[0]
    kc, vc = (torch.zeros((T // 16 + 1, 16, 1, 80), dtype=torch.uint8, device="cuda") for _ in range(2))
    Hh.ops().cascade_quant_write(x, x.flip(0), kc, vc, torch.arange(T, device="cuda"))
    want = Q.pack(x)
    assert torch.equal(kc.view(-1, 1, 80)[:T].cpu(), want) and torch.equal(vc.view(-1, 1, 80)[:T].cpu(), want.flip(0))


@pytest.mark.parametrize("KVH,q_len", [(300, 1), (300, 40), (1200, 1)])
def test_more_kv_heads_than_sms(KVH, q_len):
    Hh.need_cuda()
    args = _inputs([70, 5], [q_len] * 2, KVH, 1, 16, seed=71)
    got = Hh.ops().cascade_quant_decode(*args, q_len, SCALE, True)
    _close(got, args, True)
    assert Hh.capi().device_error() == 0
