"""Attention over a 4-bit cache on the GPU (cascade_quant_decode) against its definition in 64 bits."""
import numpy as np
import pytest

import helpers as Hh
from oracle import quant_oracle as Q

pytestmark = pytest.mark.gpu

SCALE = 128 ** -0.5


def _inputs(lens, q_lens, KVH, G, page, dtype="bf16", seed=0, spare=2, fill=0xFF, loud=True):
    """Queries, two caches, table and lengths; what no row may use is filled with 0xFF (centre and scale NaN)."""
    import torch
    t = {"bf16": torch.bfloat16, "fp16": torch.float16}[dtype]
    g = torch.Generator(device="cuda").manual_seed(seed)
    need = [(max(n, 0) + page - 1) // page for n in lens]
    blocks = sum(need) + spare
    cols = max(1, max(need)) + 1
    order = torch.randperm(blocks, generator=g, device="cuda").int()
    table = torch.zeros((len(lens), cols), dtype=torch.int32, device="cuda")
    caches = []
    for c in range(2):
        x = torch.randn((blocks * page, KVH, 128), generator=g, device="cuda")
        if c == 0 and loud:
            x[..., 5] *= 8
            x[..., 70] += 6
        lo, hi = x.unflatten(-1, (4, 32)).amin(-1), x.unflatten(-1, (4, 32)).amax(-1)
        centre, scale = ((lo + hi) / 2).half(), ((hi - lo) / 15).half()
        rows = torch.randint(0, 256, (blocks * page, KVH, 80), generator=g, device="cuda", dtype=torch.uint8)  # any codes
        rows[..., 64:] = torch.stack([centre, scale], -1).flatten(-2).contiguous().view(torch.uint8)
        caches.append(rows)
    used = torch.zeros(blocks * page, dtype=torch.bool, device="cuda")
    at = 0
    for b, n in enumerate(lens):
        ids = order[at : at + need[b]]
        table[b, : need[b]] = ids
        at += need[b]
        slots = (ids.long()[:, None] * page + torch.arange(page, device="cuda")).flatten()[: max(n, 0)]
        used[slots] = True
    for c in caches:
        c[~used] = fill
    q = torch.randn((sum(q_lens), KVH * G, 128), generator=g, device="cuda").to(t)
    i64 = dict(dtype=torch.int64, device="cuda")
    return [q, *(c.view(blocks, page, KVH, 80) for c in caches), table, torch.tensor(q_lens, **i64), torch.tensor(lens, **i64)]


def _close(got, args, causal, scale=SCALE, want=None):
    """Half a step of the type; P and the values are rounded to fp16 (2^-11 each) under sums of p |v|; the scores' sums in
    fp32 are 2^-20 of sum |q k| off, which changes every weight by as much."""
    import torch
    q = args[0]
    want = Q.attend(q, *args[1:4], args[4].tolist(), args[5].tolist(), scale, causal) if want is None else want
    out, lse, (size, reach) = want
    ds = reach * 2.0 ** -20 + 2.0 ** -21
    half = torch.finfo(q.dtype).eps / 2
    tol = out.abs() * half * 1.01 + (2 * 2.0 ** -11 + 2 * ds)[..., None] * 1.05 * size + 2.0 ** -25
    o, l = got[0].double(), got[1].double().view(lse.shape)
    assert bool((o.isnan() == out.isnan()).all()) or bool(out.isnan().any())
    fine = out.isfinite()
    err = (o - out).abs()
    assert bool((err <= tol)[fine].all()), float((err / tol)[fine].max())
    seen = lse.isfinite()
    assert bool(((l - lse).abs() <= ds + 2.0 ** -22 * lse.abs() + 2.0 ** -20)[seen].all())
    assert torch.equal(l.isinf() & (l < 0), lse.isinf())


def _run(args, causal=True, scale=SCALE):
    q_lens = args[4].tolist()
    uniform = q_lens[0] if q_lens and len(set(q_lens)) == 1 else 0
    got = Hh.ops().cascade_quant_decode(*args, uniform, scale, causal)
    _close(got, args, causal, scale)
    assert Hh.capi().device_error() == 0
    return got


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("KVH,G", [(1, 1), (8, 4), (2, 8), (3, 5), (1, 16), (4, 7), (2, 20), (5, 3), (1, 40), (70, 1)])
def test_head_layouts(KVH, G, dtype):
    Hh.need_cuda()
    _run(_inputs([1, 15, 16, 17, 33, 200], [1] * 6, KVH, G, 16, dtype, seed=KVH + G))


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256, 512])
@pytest.mark.parametrize("lens", [[0], [1], [0, 31, 32, 33], [63, 64, 65, 0], [127, 128, 129, 1000], [511, 513, 4097]])
def test_lengths_and_pages(lens, page):
    Hh.need_cuda()
    _run(_inputs(lens, [1] * len(lens), 2, 4, page, seed=len(lens)))


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("q_len,lens,KVH,G", [(2, [2, 1, 0, 40], 2, 4), (3, [100, 31, 3], 1, 5), (4, [5, 77, 640, 33], 8, 4),
                                              (5, [300, 4], 2, 3), (8, [8, 9, 7], 1, 1), (17, [17, 16, 150], 2, 2),
                                              (33, [33, 1, 500], 2, 4), (64, [64, 1000], 1, 8), (130, [130, 129, 700], 2, 4),
                                              (300, [1024], 1, 7), (257, [0, 256], 2, 1)])
def test_several_query_tokens(q_len, lens, KVH, G, causal):
    """Drafted tokens, chunks of prompts and shared prefixes; requests shorter than their queries leave rows empty."""
    Hh.need_cuda()
    _run(_inputs(lens, [q_len] * len(lens), KVH, G, 32, seed=q_len), causal)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("q_lens,lens", [([1, 0, 3], [20, 50, 2]), ([0, 0, 5, 1], [0, 9, 700, 33]), ([40, 1, 2, 0, 1], [64, 3000, 0, 5, 16]),
                                         ([200, 1], [333, 1])])
def test_query_lengths_on_the_device(q_lens, lens, causal):
    Hh.need_cuda()
    args = _inputs(lens, q_lens, 2, 4, 16, seed=9)
    got = Hh.ops().cascade_quant_decode(*args, 0, SCALE, causal)
    _close(got, args, causal)


def test_query_lengths_that_do_not_add_up():
    """Too many are cut where the tokens end; rows of tokens that are no request's stay as they are."""
    import torch
    Hh.need_cuda()
    C = Hh.capi()
    args = _inputs([50, 60, 70], [4, 2, 3], 2, 3, 16, seed=10)
    want = Hh.ops().cascade_quant_decode(*args, 0, SCALE, True)

    def call(q, q_lens, kv):
        out, lse = torch.full_like(q, 7.0), torch.full((q.shape[0] * q.shape[1],), 7.0, device="cuda")
        q_lens, kv = torch.tensor(q_lens, device="cuda"), torch.tensor(kv, device="cuda")
        d = C.quant_desc(q, *args[1:4], q_lens, kv, 0, SCALE)
        ws = torch.full((max(1, C.quant_decode_workspace_size(d)),), 0xFF, dtype=torch.uint8, device="cuda")
        C.quant_decode(d, out, lse, ws)
        return out, lse.view(q.shape[0], -1)

    out, lse = call(args[0], [4, 2, 1], [50, 60, 68])
    assert torch.equal(out[:7], want[0][:7]) and bool((out[7:] == 7).all()) and bool((lse[7:] == 7).all())
    out, lse = call(args[0], [4, 2, 1 << 40], [50, 60, 70])
    assert torch.equal(out, want[0])
    out, lse = call(args[0], [4, 2, -5], [50, 60, 70])
    assert torch.equal(out[:6], want[0][:6]) and bool((out[6:] == 7).all())
    assert C.device_error() == 0


@pytest.mark.parametrize("lens,KVH,G", [([20000], 1, 8), ([30011, 1, 0, 700], 2, 4), ([9000] * 9, 4, 5), ([100000, 99991], 1, 1)])
def test_long_caches(lens, KVH, G):
    Hh.need_cuda()
    _run(_inputs(lens, [1] * len(lens), KVH, G, 64, "fp16", seed=11))


def test_many_requests():
    Hh.need_cuda()
    lens = [(i * 37) % 300 for i in range(700)]
    _run(_inputs(lens, [1] * 700, 2, 4, 16, seed=12))


@pytest.mark.parametrize("KVH,G,q_len,lens", [(2, 4, 1, [40, 100, 1000]), (1, 5, 4, [40, 100, 333]), (1, 8, 40, [100, 444])])
def test_rising_and_falling_scores(KVH, G, q_len, lens):
    """Keys that grow along the sequence move the running maximum at every step; then the other way round."""
    import torch
    Hh.need_cuda()
    args = _inputs(lens, [q_len] * len(lens), KVH, G, 16, "bf16", seed=13, loud=False)
    par = args[1][..., 64:].contiguous().view(torch.float16).view(*args[1].shape[:3], 4, 2)
    place = torch.zeros(args[1].shape[:2], device="cuda")
    for b, n in enumerate(lens):
        ids = args[3][b, : (n + 15) // 16].long()
        place[ids] = (torch.arange(ids.numel() * 16, device="cuda").view(-1, 16) / n)
    for sign in (1.0, -1.0):
        p = par.clone()
        p[..., 0] += (sign * 6 * place)[..., None, None].half()
        args[1][..., 64:] = p.flatten(-2).contiguous().view(torch.uint8)
        args[0].abs_()
        _run(args, True, 0.3)


def test_query_magnitudes_and_scales():
    import torch
    Hh.need_cuda()
    args = _inputs([300, 40, 5], [1] * 3, 2, 4, 32, "bf16", seed=14)
    args[0][0] *= 1e-30
    args[0][1, :4] = 0
    args[0][1, 4:] *= 1e-3
    args[0][2, :, 64:] *= 1e-6   # parts of a row far below its largest value
    _run(args)
    args[0][2] = 3e4             # one token wins everything
    got = Hh.ops().cascade_quant_decode(*args, 1, SCALE, True)
    _close(got, args, True)
    _run(args, True, 1e-4)


@pytest.mark.parametrize("scale", [1e-4, 3e-3, 40.0, 2000.0])
def test_value_magnitudes(scale):
    """The values' centres and scales over fp16's range, in one request beside ordinary ones."""
    import torch
    Hh.need_cuda()
    args = _inputs([500, 77], [1] * 2, 2, 4, 16, "bf16", seed=15)
    for b in range(1):
        ids = args[3][b, :32].long()
        par = args[2][ids][..., 64:].contiguous().view(torch.float16)
        rows = args[2][ids]
        rows[..., 64:] = (par.float() * scale).half().contiguous().view(torch.uint8)
        args[2][ids] = rows
    out, lse, (size, reach) = want = Q.attend(args[0], *args[1:4], [1, 1], [500, 77], SCALE, True)
    got = Hh.ops().cascade_quant_decode(*args, 1, SCALE, True)
    # values are rounded to fp16: 2^-25 at least
    _close(got, args, True, want=(out, lse, (size + 2.0 ** -14, reach)))


def test_what_no_row_sees_may_hold_anything():
    """NaN in keys and values that only the causal mask hides, and past the lengths (every other test as well)."""
    import torch
    Hh.need_cuda()
    for q_len, n, KVH, G in ((4, 40, 2, 4), (20, 50, 1, 4), (100, 333, 2, 4)):
        args = _inputs([n], [q_len], KVH, G, 16, seed=16)
        t = n - q_len // 2     # seen by the last q_len / 2 tokens alone
        page, place = int(args[3][0, t // 16]), t % 16
        clean = Hh.ops().cascade_quant_decode(*args, q_len, SCALE, True)
        for which in (1, 2):
            keep = args[which].clone()
            args[which][page, place, :, 64 + 4 * 2 : 64 + 4 * 3] = 0xFF    # group 2: centre and scale NaN
            out, lse = Hh.ops().cascade_quant_decode(*args, q_len, SCALE, True)
            first = q_len - q_len // 2     # the first token that sees it
            assert torch.equal(out[:first], clean[0][:first])
            assert torch.equal(lse.view(q_len, -1)[:first], clean[1].view(q_len, -1)[:first])
            assert bool(out[first:, :, 64:96].isnan().all())
            if which == 1:
                assert bool(out[first:].isnan().all()) and bool(lse.view(q_len, -1)[first:].isnan().all())
            args[which].copy_(keep)


def test_nan_and_infinity_that_rows_see():
    import torch
    Hh.need_cuda()
    args = _inputs([40, 900, 33, 0], [1] * 4, 2, 4, 16, seed=17)
    clean = Hh.ops().cascade_quant_decode(*args, 1, SCALE, True)
    args[0][0, 3, 100] = float("nan")
    args[0][1, 5, 0] = float("inf")
    args[0][3] = float("nan")                          # sees nothing: zeros all the same
    args[2][int(args[3][2, 1]), 3, 1, 64:68] = 0xFF     # a value's group 0 of kv head 1, token 19 of request 2
    out, lse = Hh.ops().cascade_quant_decode(*args, 1, SCALE, True)
    lse, other = lse.view(4, 8), clean[1].view(4, 8)
    touched = torch.zeros((4, 8), dtype=torch.bool, device="cuda")
    touched[0, 3] = touched[1, 5] = True
    assert bool(out[touched].isnan().all()) and bool(lse[touched].isnan().all())
    assert bool(out[2, 4:, :32].isnan().all())
    touched[2, 4:] = True
    assert torch.equal(out[~touched], clean[0][~touched]) and torch.equal(lse[~touched], other[~touched])
    assert not out[3].any() and bool((lse[3] == float("-inf")).all())


def test_pages_outside_the_cache_read_as_zeros():
    import torch
    Hh.need_cuda()
    for q_len, KVH, G in ((1, 2, 4), (50, 1, 4)):
        args = _inputs([200, 90], [q_len] * 2, KVH, G, 16, seed=18)
        args[3][0, 3], args[3][0, 7], args[3][1, 0] = -5, args[1].shape[0], 1 << 30
        args[3][:, 13:] = -1    # past the lengths: never read
        got = Hh.ops().cascade_quant_decode(*args, q_len, SCALE, True)
        assert Hh.capi().device_error() == 2
        _close(got, args, True)


def test_lengths_past_the_table_are_cut():
    import torch
    Hh.need_cuda()
    args = _inputs([96, 64], [2] * 2, 2, 4, 16, seed=19)
    table = args[3][:, :6].contiguous()
    args[3] = table
    args[3][1, 4:] = args[3][1, :2]
    args[5][:] = torch.tensor([1 << 50, 96], device="cuda")
    got = Hh.ops().cascade_quant_decode(*args, 2, SCALE, True)
    args[5][0] = 96
    _close(got, args, True)
    args[5][:] = -3
    out, lse = Hh.ops().cascade_quant_decode(*args, 2, SCALE, True)
    assert not out.any() and bool((lse == float("-inf")).all())


def test_no_pages_at_all():
    import torch
    Hh.need_cuda()
    q = torch.randn((3, 8, 128), device="cuda").half()
    caches = [torch.empty((0, 16, 2, 80), dtype=torch.uint8, device="cuda") for _ in range(2)]
    i64 = dict(dtype=torch.int64, device="cuda")
    for table in (torch.empty((3, 0), dtype=torch.int32, device="cuda"), torch.zeros((3, 2), dtype=torch.int32, device="cuda")):
        lens = torch.zeros(3, **i64)
        out, lse = Hh.ops().cascade_quant_decode(q, *caches, table, torch.ones(3, **i64), lens, 1, SCALE, True)
        assert not out.any() and bool((lse == float("-inf")).all())
    assert Hh.capi().device_error() == 0


def test_cache_offsets_past_32_bits():
    import torch
    Hh.need_cuda()
    page, KVH = 64, 8
    blocks = (1 << 31) // (page * KVH * 80) + 3000
    small = _inputs([500, 130], [1] * 2, KVH, 4, page, seed=20, spare=1)
    n = small[1].shape[0]
    caches = [torch.zeros((blocks, page, KVH, 80), dtype=torch.uint8, device="cuda") for _ in range(2)]
    ids = torch.cat([torch.arange(n // 2, device="cuda"), blocks - 1 - torch.arange(n - n // 2, device="cuda")])
    for c, s in zip(caches, small[1:3]):
        c[ids] = s
    table = ids[small[3].long()].int()
    want = Hh.ops().cascade_quant_decode(*small, 1, SCALE, True)
    got = Hh.ops().cascade_quant_decode(small[0], *caches, table, *small[4:], 1, SCALE, True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_refusals():
    import torch
    Hh.need_cuda()
    f = Hh.ops().cascade_quant_decode
    a = _inputs([20, 30], [1, 1], 2, 4, 16)

    def put(i, v):
        return a[:i] + [v] + a[i + 1 :]

    for args, text in [(put(0, a[0].float()), "bf16 or fp16"), (put(0, a[0][..., :64].contiguous()), "heads, 128"),
                       (put(0, a[0][:, ::2]), "contiguous"), (put(0, a[0][:, :7].contiguous()), "multiple of kv_heads"),
                       (put(1, a[1][..., :64].contiguous()), "kv heads, 80"), (put(2, a[2][:1]), "equal shapes"),
                       (put(3, a[3].long()), "block_table"), (put(3, a[3][:1]), "row per request"),
                       (put(4, a[4][:1]), "batch entries"), (put(5, a[5].int()), "actual_kv_seqlens"),
                       (put(5, a[5].cpu()), "must be on")]:
        with pytest.raises(RuntimeError, match=text):
            f(*args, 1, SCALE, True)
    with pytest.raises(RuntimeError, match="q_seqlen_value"):
        f(*a, 2, SCALE, True)
    with pytest.raises(RuntimeError, match="scale must be positive"):
        f(*a, 1, 0.0, True)
    with pytest.raises(RuntimeError, match="blockSize"):
        f(a[0], *(c.view(-1, 8, 2, 80) for c in a[1:3]), *a[3:], 1, SCALE, True)
    assert f(a[0][:0], *a[1:3], a[3][:0], a[4][:0], a[5][:0], 1, SCALE, True)[0].shape == (0, 8, 128)


def test_streams_graphs_and_repeats():
    """The same bits in a loop, on another stream, and from two graphs replayed in turn; new lengths in a captured call."""
    import torch
    Hh.need_cuda()
    f = Hh.ops().cascade_quant_decode
    args = _inputs([3000, 1, 500, 64], [1] * 4, 4, 4, 16, seed=21)
    want = [t.clone() for t in f(*args, 1, SCALE, True)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = f(*args, 1, SCALE, True)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(f(*args, 1, SCALE, True))
        graphs.append(g)
    for _ in range(5):
        for g in graphs:
            g.replay()
    for o in outs:
        assert torch.equal(o[0], want[0]) and torch.equal(o[1], want[1])
    short = _inputs([3000, 1, 500, 64], [1] * 4, 4, 4, 16, seed=21)
    short[5] = torch.tensor([17, 0, 499, 33], device="cuda")
    args[5].copy_(short[5])
    graphs[0].replay()
    _close(outs[0], args, True)
    again = f(*args, 1, SCALE, True)
    assert torch.equal(again[0], outs[0][0]) and torch.equal(again[1], outs[0][1])


def test_two_calls_at_once():
    import torch
    Hh.need_cuda()
    f = Hh.ops().cascade_quant_decode
    a, b = _inputs([5000, 400], [1] * 2, 8, 4, 64, seed=22), _inputs([2000] * 8, [4] * 8, 2, 5, 16, "fp16", seed=23)
    want = [f(*a, 1, SCALE, True), f(*b, 4, SCALE, True)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for s, args, n, out in zip(streams, (a, b), (1, 4), got):
            with torch.cuda.stream(s):
                out.append(f(*args, n, SCALE, True))
    torch.cuda.synchronize()
    for w, outs in zip(want, got):
        for o in outs:
            assert torch.equal(o[0], w[0]) and torch.equal(o[1], w[1])
    assert np.isfinite(Hh.dev_to_f64(want[0][0])).all()
