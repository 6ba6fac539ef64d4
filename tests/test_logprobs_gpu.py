"""Log probabilities of tokens on the GPU (cascade_token_logprobs) against their definition in 64 bits."""
import pytest

import helpers as Hh
from oracle import quant_oracle as Q

pytestmark = pytest.mark.gpu


def _logits(N, V, dtype, seed=0, scale=3.0):
    import torch
    t = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}[dtype]
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn((N, V), generator=g, device="cuda") * scale).to(t), torch.randint(0, V, (N,), generator=g, device="cuda")


def _check(x, tokens, top):
    import torch
    got = Hh.ops().cascade_token_logprobs(x, tokens, top)
    want = Q.logprobs(x, tokens, top)
    N, V = x.shape
    assert got[0].shape == got[1].shape == got[2].shape == (N,) and got[3].shape == got[4].shape == (N, top)
    assert got[0].dtype == got[1].dtype == got[3].dtype == torch.float32 and got[2].dtype == got[4].dtype == torch.int64
    assert torch.equal(got[2], want[2]) and torch.equal(got[4], want[4])
    # The sum of positive terms, each 2^-21 off (an exponential of fp32), in chains of at most V / 128 + 64 additions of 2^-24;
    # the logarithm and the last differences 2^-22 of their size. The entropy's terms are |d| times as large.
    rel = 2.0 ** -21 + (V / 128 + 64) * 2.0 ** -24
    d = (x.double() - x.double().amax(-1, keepdim=True)).nan_to_num(0.0, 0.0, 0.0)
    p = torch.softmax(d, -1)
    spread = (p * d.abs()).sum(-1)
    for a, b, tol in ((got[0], want[0], rel + 2.0 ** -22 * (1 + want[0].abs())),
                      (got[1], want[1], (3 * rel + 2.0 ** -21) * (2 + spread)),
                      (got[3], want[3], rel + 2.0 ** -22 * (1 + want[3].abs()))):
        same = (a.double() == b) | (a.isnan() & b.isnan()) | ((a.double() - b).abs() <= tol)
        assert bool(same.all()), (a[~same][:4], b[~same][:4])
    return got


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("N,V,top", [(1, 1, 1), (1, 1, 0), (3, 31, 31), (2, 32, 32), (5, 33, 7), (7, 1000, 5), (64, 4097, 20),
                                     (1, 128256, 32), (9, 32001, 1), (300, 515, 3), (1000, 257, 2), (2, 50304, 0)])
def test_logprobs(N, V, top, dtype):
    Hh.need_cuda()
    _check(*_logits(N, V, dtype, seed=N + V), top)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_many_rows_of_a_large_vocabulary(dtype):
    Hh.need_cuda()
    _check(*_logits(200, 128256, dtype, seed=1), 20)


@pytest.mark.parametrize("dtype", ["fp32", "fp16"])
@pytest.mark.parametrize("N,V", [(48, 40001), (49, 40001), (105, 33000), (145, 33000), (223, 20011), (300, 70000)])
def test_rows_shared_by_clusters_of_every_size(N, V, dtype):
    Hh.need_cuda()
    _check(*_logits(N, V, dtype, seed=N), 32)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("share", [0.001, 0.5, 0.999])
@pytest.mark.parametrize("N", [3, 230])
def test_minus_infinity_among_the_others(N, share, dtype):
    """Also with the token ahead of all others, and behind them."""
    import torch
    Hh.need_cuda()
    x, tokens = _logits(N, 30001, dtype, seed=N)
    gone = torch.rand(x.shape, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda") < share
    gone[:, 17] = False
    x[gone] = -float("inf")
    tokens[0], tokens[1] = x[0].argmax(), x[1].argmin()
    _check(x, tokens, 5)


@pytest.mark.parametrize("V", [40, 1003, 70000])
def test_equal_logits_go_to_the_lowest_index(V):
    import torch
    Hh.need_cuda()
    x, tokens = _logits(6, V, "bf16", seed=2, scale=0.02)   # some hundred different values
    x[1] = 0.0
    x[2] = -0.0
    x[3, ::2] = 0.0
    x[3, 1::2] = -0.0
    tokens[1:4] = torch.tensor([V - 1, V // 2, 3], device="cuda")
    got = _check(x, tokens, 32)
    assert got[2][1] == V - 1 and got[4][3].tolist() == list(range(32))


@pytest.mark.parametrize("order", ["rising", "falling", "last block"])
def test_alternatives_wherever_they_lie(order):
    """Every entry beats all before it, or none does, or the best ones lie together."""
    import torch
    Hh.need_cuda()
    V = 20011
    x = torch.arange(V, device="cuda", dtype=torch.float32)[None] * 0.001
    x = {"rising": x, "falling": x.flip(1), "last block": torch.where(x > 0.001 * (V - 40), x + 5, -x)}[order].repeat(3, 1).contiguous()
    _check(x, torch.tensor([0, V // 2, V - 1], device="cuda"), 32)


def test_masked_vocabularies():
    import torch
    Hh.need_cuda()
    inf = float("inf")
    x, tokens = _logits(8, 3000, "fp32", seed=3)
    x[0, 10:] = -inf                      # a grammar that leaves ten
    x[1, 5:] = -inf
    tokens[1] = 100                       # a masked token
    x[2] = -inf
    x[2, 2999] = 1.5                      # one left: entropy 0
    tokens[2] = 2999
    x[3] = torch.finfo(torch.float32).min  # masked by the type's lowest value
    x[3, 7] = 0
    x[4] = -3e38
    x[5, 1000:] = torch.finfo(torch.float32).min
    got = _check(x, tokens, 20)
    assert got[0][1] == -inf and got[1][2] == 0 and got[0][2] == 0
    assert got[4][0, 10:].tolist() == list(range(10, 20))   # equals of -inf: lowest index first
    y = x[:6].to(torch.bfloat16)
    y[3] = torch.finfo(torch.bfloat16).min
    y[3, 7] = 0
    _check(y, tokens[:6], 20)


@pytest.mark.parametrize("dtype", ["fp32", "fp16"])
def test_nan_infinity_and_rows_of_nothing(dtype):
    import torch
    Hh.need_cuda()
    inf, nan = float("inf"), float("nan")
    x, tokens = _logits(7, 5000, dtype, seed=4)
    x[1, 77] = nan
    x[2, 4999] = inf
    x[3] = -inf
    x[4] = nan
    x[5, [3, 9]] = inf
    tokens[[1, 2]] = torch.tensor([77, 4999], device="cuda")
    got = _check(x, tokens, 5)
    for i in (1, 2, 3, 4, 5):
        assert got[0][i].isnan() and got[1][i].isnan() and bool(got[3][i].isnan().all())
    assert not got[0][[0, 6]].isnan().any()
    assert got[4][2, 0] == 4999 and got[4][5, :2].tolist() == [3, 9] and got[2][3] == int(tokens[3])


def test_tokens_outside_the_vocabulary():
    import torch
    Hh.need_cuda()
    x, tokens = _logits(5, 700, "bf16", seed=5)
    tokens[:4] = torch.tensor([-1, 700, 1 << 40, -(1 << 33)], device="cuda")
    got = _check(x, tokens, 3)
    assert bool((got[0][:4] == float("-inf")).all()) and got[2][:4].tolist() == [-1] * 4


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_row_strides_and_alignment(dtype):
    """Rows inside a wider matrix, starting at any element."""
    Hh.need_cuda()
    for off, V in ((0, 1000), (1, 999), (3, 2051), (5, 64), (8, 4096)):
        x, _ = _logits(6, 4109, dtype, seed=6)
        view = x[:, off : off + V]
        import torch
        _check(view, torch.arange(6, device="cuda") * (V // 7), min(V, 9))


def test_large_values():
    import torch
    Hh.need_cuda()
    x, tokens = _logits(4, 2000, "fp32", seed=7, scale=1e30)
    x[1] = torch.linspace(0, 300, 2000, device="cuda") + 1e6
    x[2] *= 1e-36
    _check(x, tokens, 6)


def test_refusals_and_nothing_to_do():
    import torch
    Hh.need_cuda()
    f = Hh.ops().cascade_token_logprobs
    x, tokens = _logits(3, 50, "fp32")
    assert [t.shape[0] for t in f(x[:0], tokens[:0], 4)] == [0] * 5
    for args, text in [((x.double(), tokens, 1), "bf16, fp16 or fp32"), ((x, tokens[:2], 1), "entry per row"),
                       ((x, tokens.int(), 1), "tokens must be"), ((x, tokens, 33), "top must be"), ((x, tokens, 51), "top must be"),
                       ((x, tokens, -1), "top must be"), ((x[0], tokens, 1), "rows, vocabulary"),
                       ((x.t().contiguous().t(), tokens, 1), "contiguous rows"), ((x, tokens.cpu(), 1), "must be on"),
                       ((x[:, :0], tokens, 0), "must not be empty")]:
        with pytest.raises(RuntimeError, match=text):
            f(*args)


def test_two_graphs_and_a_stream():
    import torch
    Hh.need_cuda()
    f = Hh.ops().cascade_token_logprobs
    x, tokens = _logits(4, 40000, "bf16", seed=8)
    want = [t.clone() for t in f(x, tokens, 5)]
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(f(x, tokens, 5))
        graphs.append(g)
    for _ in range(3):
        for g in graphs:
            g.replay()
    for out in outs:
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = f(x, tokens, 5)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
