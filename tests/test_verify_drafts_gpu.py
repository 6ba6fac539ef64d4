"""Verification of drafted tokens on the GPU (cascade_verify_drafts) against a
plain host version in the same rounded operations (one fp32 product, difference
and quotient each), so tokens and counts have to be equal; and the sampled
distribution against the target's."""
import numpy as np
import pytest

import helpers as Hh

pytestmark = pytest.mark.gpu


def _inputs(B, K, V, dtype="fp32", seed=0, near=0.5, lens=None):
    import torch
    t = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}[dtype]
    g = torch.Generator(device="cuda").manual_seed(seed)
    logits = torch.randn((B, K + 1, V), generator=g, device="cuda") * 2
    target = torch.softmax(logits, -1).to(t)
    draft = torch.softmax(logits[:, :K] + near * torch.randn((B, K, V), generator=g, device="cuda"), -1).to(t)
    tokens = torch.randint(0, V, (B, K), generator=g, device="cuda")
    if K:
        best = draft.float().argmax(-1)
        tokens = torch.where(torch.rand((B, K), generator=g, device="cuda") < 0.8, best, tokens)
    lens = torch.randint(0, K + 1, (B,), generator=g, device="cuda") if lens is None else torch.tensor(lens, device="cuda")
    uniform = torch.rand((B, K), generator=g, device="cuda")
    noise = torch.empty((B, V), device="cuda").exponential_(generator=g).clamp_(min=1e-20)
    return [tokens, lens, draft, target, uniform, noise]


def _want(tokens, lens, draft, target, uniform, noise):
    f = lambda x: x.float().cpu().numpy()  # noqa: E731
    tok, n = tokens.cpu().numpy(), lens.cpu().numpy()
    q, p, u, e = None if draft is None else f(draft), f(target), f(uniform), f(noise)
    B, K = tok.shape
    V = p.shape[2]
    out, acc = np.full((B, K + 1), -1, np.int64), np.zeros(B, np.int64)
    for b in range(B):
        m, i = min(max(int(n[b]), 0), K), 0
        while i < m:
            x = int(tok[b, i])
            ok = 0 <= x < V and np.float32(u[b, i]) * (np.float32(1) if q is None else q[b, i, x]) < p[b, i, x]
            if not ok:
                break
            i += 1
        left = p[b, i].copy()
        if i < m:
            if q is not None:
                left = np.maximum(left - q[b, i], np.float32(0))
            elif 0 <= tok[b, i] < V:
                left[tok[b, i]] = 0
        if not (left > 0).any():
            left = p[b, i]
        out[b, :i] = tok[b, :i]
        out[b, i] = int(np.argmax(left / e[b]))
        acc[b] = i
    return out, acc


def _case(args):
    got = Hh.ops().cascade_verify_drafts(*args)
    want = _want(*args)
    assert np.array_equal(got[1].cpu().numpy(), want[1])
    assert np.array_equal(got[0].cpu().numpy(), want[0])
    return want


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("B,K,V", [(1, 1, 1), (3, 2, 31), (5, 4, 1000), (64, 3, 4097), (7, 5, 32001), (2, 40, 515),
                                   (300, 2, 999), (1, 3, 128256), (4, 0, 700)])
def test_verify(B, K, V, dtype):
    Hh.need_cuda()
    _case(_inputs(B, K, V, dtype, seed=B + V))


@pytest.mark.parametrize("V", [1001, 20000])
def test_verify_without_draft_probabilities(V):
    Hh.need_cuda()
    args = _inputs(40, 3, V)
    args[2] = None
    args[4] *= 0.05   # some are accepted
    acc = _case(args)[1]
    assert 0 < acc.sum() < 120


def test_verify_ties_and_empty_residuals():
    """Equal distributions leave nothing (the target's row stands in); equal quotients take the lowest index."""
    import torch
    Hh.need_cuda()
    args = _inputs(6, 3, 5000)
    args[2] = args[3][:, :3].clone()
    args[4][:] = 1.0                  # u q < p is false: every first draft is refused
    args[1][:] = 3
    _case(args)
    args[3][:] = 1.0 / 5000
    args[2] = args[3][:, :3] * 0.5
    args[5][:] = 0.25
    args[4][:] = 2.5
    out, acc = _case(args)
    assert (acc == 0).all() and (out[:, 0] == 0).all()
    args[3][0], args[2][0] = 0.0, 0.0  # a row of zeros
    _case(args)


def test_verify_edge_lengths_and_tokens():
    import torch
    Hh.need_cuda()
    args = _inputs(6, 3, 900, lens=[0, 3, -2, 9, 1, 2])
    args[0][1, 0], args[0][3, 0] = 900, -1       # outside the vocabulary: refused
    args[4][5, :] = 0.0                           # accepted wherever the target is positive
    _case(args)


def test_verify_samples_the_target():
    """Over many draws the first token is distributed as the target, whatever the drafts were taken from."""
    import torch
    Hh.need_cuda()
    N, V = 60000, 7
    g = torch.Generator(device="cuda").manual_seed(5)
    p = torch.softmax(torch.randn(V, generator=g, device="cuda"), 0)
    q = torch.softmax(torch.randn(V, generator=g, device="cuda"), 0)
    tokens = torch.multinomial(q.expand(N, V), 1, generator=g)
    out, _ = Hh.ops().cascade_verify_drafts(
        tokens, torch.ones(N, dtype=torch.int64, device="cuda"), q.expand(N, 1, V).contiguous(),
        p.expand(N, 2, V).contiguous(), torch.rand((N, 1), generator=g, device="cuda"),
        torch.empty((N, V), device="cuda").exponential_(generator=g))
    seen = torch.bincount(out[:, 0], minlength=V).double() / N
    # five standard deviations of a frequency
    assert ((seen - p.double()).abs() <= 5 * (p.double() * (1 - p.double()) / N).sqrt()).all()


def test_verify_in_a_graph_and_on_a_stream():
    import torch
    Hh.need_cuda()
    args = _inputs(9, 3, 3001)
    want = Hh.ops().cascade_verify_drafts(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            got = Hh.ops().cascade_verify_drafts(*args)
        g.replay()
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_verify_refusals():
    import torch
    Hh.need_cuda()
    t, n, q, p, u, e = _inputs(3, 2, 50)
    bad = [
        ((t, n, q, p.double(), u, e), "bf16, fp16 or fp32"),
        ((t, n, q.half(), p, u, e), "draft_probs must be"),
        ((t, n, q[:, :, :49].contiguous(), p, u, e), "draft_probs must be"),
        ((t, n, q, p[:, :2].contiguous(), u, e), "target_probs must be"),
        ((t.int(), n, q, p, u, e), "draft_tokens must be"),
        ((t, n[:2], q, p, u, e), "draft_lens must be"),
        ((t, n, q, p, u[:, :1].contiguous(), e), "uniform must be"),
        ((t, n, q, p, u, e[:, :49].contiguous()), "noise must be"),
        ((t, n, q, p.transpose(0, 1).contiguous().transpose(0, 1), u, e), "contiguous"),
    ]
    for args, text in bad:
        with pytest.raises(RuntimeError, match=text):
            Hh.ops().cascade_verify_drafts(*args)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("V", [4, 8, 1020, 1028, 4096, 8192, 16388, 40004])
def test_verify_rows_of_whole_groups(V, dtype):
    """Rows that are read in groups of four, around whole rounds."""
    _case(_inputs(9, 3, V, dtype, seed=V))


@pytest.mark.parametrize("which", [2, 3, 5])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_verify_tensors_off_the_group_alignment(which, dtype):
    """One tensor an element past 16 bytes: the same answer from single entries."""
    import torch
    args = _inputs(7, 3, 5000, dtype, seed=which)
    x = args[which]
    room = torch.empty(x.numel() + 1, dtype=x.dtype, device="cuda")
    off = room[1:].view(x.shape)
    off.copy_(x)
    want = _case(args)
    args[which] = off
    assert np.array_equal(_case(args)[0], want[0])


def test_verify_equal_quotients_take_the_lowest_index():
    """Equal best quotients in different rounds, lanes, warps and CTAs."""
    import torch
    V = 40000
    target = torch.full((6, 1, V), 1e-6, device="cuda")
    noise = torch.ones((6, V), device="cuda")
    places = [[39999, 20000], [33, 32], [16384, 8191, 30000], [7, 6, 5, 4], [12345, 12345 + 8192], [39998]]
    for b, p in enumerate(places):
        target[b, 0, p] = 0.25
    empty = torch.zeros((6, 0), device="cuda")
    out, acc = Hh.ops().cascade_verify_drafts(empty.long(), torch.zeros(6, dtype=torch.int64, device="cuda"), None, target,
                                              empty, noise)
    assert out[:, 0].tolist() == [min(p) for p in places] and acc.tolist() == [0] * 6


@pytest.mark.parametrize("token", [(1 << 32) + 5, (1 << 33) + 5, -(1 << 32) + 5, 900, -1])
def test_verify_tokens_outside_the_vocabulary_leave_nothing_out(token):
    """Without draft probabilities a refused token is left out of the target's row; one that is no entry leaves the
    row whole, whatever its low 32 bits are."""
    Hh.need_cuda()
    args = _inputs(4, 2, 900, lens=[1, 2, 1, 2])
    args[2] = None
    args[0][:, 0] = token
    args[5][:, 5] = 1e-12  # the best entry
    out, acc = _case(args)
    assert (acc == 0).all() and (out[:, 0] == 5).all()


@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_verify_nan_probabilities_accept_and_sample_nothing(dtype, draft):
    """A NaN refuses its draft and counts as 0 in what is left, in the target's row that stands in too."""
    import torch
    Hh.need_cuda()
    B, V = 6, 900
    args = _inputs(B, 2, V, dtype, lens=[2] * B)
    args[4][:] = 0.0                      # accepted wherever the target is positive
    args[3][0, 0, args[0][0, 0]] = float("nan")
    args[3][1, 2, ::2] = float("nan")     # the row after the last draft
    args[3][2, 1] = float("nan")          # nothing but NaN: index 0
    args[3][3, 1, args[0][3, 1]] = 0.0
    args[3][3, 1, 1::3] = float("nan")
    if draft:
        args[2][4, 0, 7::2] = float("nan")
        args[4][4, 0] = 2.0               # refused, whatever the draft's probability is
        args[2][5, 0] = args[3][5, 0]     # nothing is left but what NaN hides: the target's row stands in
        args[4][5, 0] = 2.0
        args[3][5, 0, ::2] = float("nan")
    else:
        args[2] = None
    got = Hh.ops().cascade_verify_drafts(*args)
    f = lambda x: x.float().cpu().numpy()  # noqa: E731
    p, q, e, tok = f(args[3]), f(args[2]) if draft else None, f(args[5]), args[0].cpu().numpy()
    u = f(args[4])
    for b in range(B):
        i = 0
        while i < 2 and np.float32(u[b, i]) * (q[b, i, tok[b, i]] if draft else np.float32(1)) < p[b, i, tok[b, i]]:
            i += 1
        left = p[b, i].copy()
        if i < 2 and draft:
            left = left - q[b, i]
        elif i < 2:
            left[tok[b, i]] = 0
        left = np.where(left > 0, left, 0)
        if not left.any():
            left = np.where(p[b, i] > 0, p[b, i], 0)
        assert got[1][b] == i and got[0][b].tolist() == tok[b, :i].tolist() + [int(np.argmax(left / e[b]))] + [-1] * (2 - i)
