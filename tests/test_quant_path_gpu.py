"""The 4-bit cache's operators together: the example, the page operators on its pools, a shared prefix, captured steps,
and attention calls whose bounded waits run out."""
import importlib.util
import os
import time

import pytest

import helpers as Hh
from conftest import ROOT
from oracle import quant_oracle as Q

pytestmark = pytest.mark.gpu

SCALE = 128 ** -0.5


def _example():
    spec = importlib.util.spec_from_file_location("quantised_cache", os.path.join(ROOT, "examples", "quantised_cache.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


@pytest.mark.parametrize("samples,prompt,chunk,page", [(6, 700, 256, 64), (3, 65, 16, 16)])
def test_example(samples, prompt, chunk, page):
    import torch
    Hh.need_cuda()
    r = _example().run(samples=samples, prompt=prompt, chunk=chunk, page=page, log=lambda *_: None)
    cache = r["cache"]
    # two partial outputs rounded to bf16 (2^-8 each), merged, against one rounding
    assert r["gap"] < 3 * 2.0 ** -8
    flat = cache.table[cache.table >= 0].long()
    assert torch.equal(torch.bincount(flat, minlength=cache.refs.numel()).int(), cache.refs)
    assert int((cache.refs[: r["live"]] > 0).sum()) == r["live"] == int((cache.refs > 0).sum())
    for tokens, logprob, entropy, rank, top, alternatives in r["answers"]:
        assert bool((logprob <= 0).all()) and bool((entropy >= 0).all()) and bool((top[:, 1:] <= top[:, :-1]).all())
        first = rank < 5    # a token among the alternatives is found there, with its log probability
        at = rank.clamp(max=4)[:, None]
        assert torch.equal(alternatives.gather(1, at)[first, 0], tokens[first]) and torch.equal(top.gather(1, at)[first, 0], logprob[first])
    # the kept samples' last keys, read back: half a step of their group's span, and the fp16 and bf16 roundings
    kept = r["keys"][::2].double()
    got = r["back"].view(len(range(0, samples, 2)), -1, *kept.shape[1:])[:, -1].double()
    group = kept.unflatten(-1, (4, 32))
    tol = (group.amax(-1) - group.amin(-1)) / 30 * 1.01 + 2.0 ** -8 * group.abs().amax(-1)
    assert bool(((got - kept).unflatten(-1, (4, 32)).abs().amax(-1) <= tol).all())
    assert Hh.capi().device_error() == 0


def _filled(lens, KVH=2, page=16, blocks=80, cols=20, seed=0):
    import torch
    from cascade_kernel.quant import QuantCache
    g = torch.Generator(device="cuda").manual_seed(seed)
    cache = QuantCache(2, blocks, page, len(lens), cols, KVH)
    cache.grow(torch.tensor(lens, device="cuda"))
    kv = torch.randn((sum(lens), 2, KVH, 128), generator=g, device="cuda").bfloat16()
    slots = cache.slots(lens)
    for layer in range(2):
        cache.write(layer, kv[:, layer], kv[:, 1 - layer], slots)
    return cache, kv, g


def test_pages_of_a_quantised_cache():
    """Forked, truncated and compacted rows hold what was written, in every layer."""
    import torch
    Hh.need_cuda()
    lens = [37, 5, 64, 100]
    cache, kv, g = _filled(lens)
    want = [Q.values(Q.pack(kv[:, i]).cuda()).float().bfloat16() for i in range(2)]
    for layer in range(2):
        k, v = cache.read(layer, lens)
        assert torch.equal(k, want[layer]) and torch.equal(v, want[1 - layer])
    parents = [3, 0, 0, 2, 3]
    cache.fork(torch.tensor(parents, device="cuda"))
    start = [sum(lens[:i]) for i in range(4)]
    rows = torch.cat([torch.arange(start[p], start[p] + lens[p]) for p in parents]).cuda()
    assert torch.equal(cache.read(1, [lens[p] for p in parents])[0], want[1][rows])
    keep = [50, 37, 0, 64, 33]
    cache.truncate(torch.tensor(keep, device="cuda"))
    live = int(cache.compact())
    assert live == int((cache.refs > 0).sum())
    rows = torch.cat([torch.arange(start[p], start[p] + n) for p, n in zip(parents, keep)]).cuda()
    for layer in range(2):
        k, v = cache.read(layer, keep)
        assert torch.equal(k, want[layer][rows]) and torch.equal(v, want[1 - layer][rows])
    # a row that goes on inside a shared page gets its own copy
    more = torch.tensor([3, 1, 2, 0, 20], device="cuda")
    cache.grow(more)
    x = torch.randn((int(more.sum()), 2, 2, 128), generator=g, device="cuda").bfloat16()
    cache.write(0, x[:, 0], x[:, 1], more.tolist())
    got = cache.read(0, [n + m for n, m in zip(keep, more.tolist())])[0].split([n + m for n, m in zip(keep, more.tolist())])
    for i, (n, m) in enumerate(zip(keep, more.tolist())):
        assert torch.equal(got[i][:n], want[0][start[parents[i]] : start[parents[i]] + n])
    with pytest.raises(RuntimeError, match="QuantCache"):
        cache.grow(torch.full((5,), 10000, device="cuda"))
    with pytest.raises(RuntimeError, match="QuantCache.slots"):
        cache.slots([1000] * 5)


@pytest.mark.parametrize("B,H", [(5, 8), (3, 2), (40, 8)])
def test_shared_prefix_equals_each_row_by_itself(B, H):
    import torch
    Hh.need_cuda()
    from cascade_kernel.quant import QuantCache
    g = torch.Generator(device="cuda").manual_seed(1)
    page, P, KVH = 32, 320, 2
    cache = QuantCache(1, 400, page, 1, 16, KVH)

    def kv(n):
        return [torch.randn((n, KVH, 128), generator=g, device="cuda").bfloat16() for _ in range(2)]

    cache.grow(torch.tensor([P], device="cuda"))
    cache.write(0, *kv(P), [P])
    prefix = cache.table[:, : P // page].contiguous()
    cache.fork(torch.zeros(B, dtype=torch.int64, device="cuda"))
    own = [1 + (i * 37) % 100 for i in range(B)]
    cache.grow(torch.tensor(own, device="cuda"))
    cache.write(0, *kv(sum(own)), own)
    q = torch.randn((B, H, 128), generator=g, device="cuda").bfloat16()
    one, _ = cache.attend(0, q, 1, SCALE)
    lens = torch.tensor([P], dtype=torch.int64, device="cuda")
    two = cache.attend_shared(0, q, prefix, lens, SCALE, P)
    # the same sums but for the partial outputs' rounding to bf16 (2^-8 each of values up to 4) and one more at the end
    assert float((one.float() - two.float()).abs().max()) <= 3 * 2.0 ** -8 * 4
    with pytest.raises(ValueError, match="whole pages"):
        cache.attend_shared(0, q, prefix, lens, SCALE, P + 1)


def test_a_captured_step():
    """Write, attend and score in one graph, replayed with new tokens and lengths."""
    import torch
    Hh.need_cuda()
    npu = Hh.ops()
    lens = [30, 7, 64]
    cache, _, g = _filled(lens)
    cache.grow(torch.ones(3, dtype=torch.int64, device="cuda"))
    slots = cache.slots([1, 1, 1])
    x = torch.randn((3, 8, 128), generator=g, device="cuda").bfloat16()     # queries of 4 heads, keys, values of 2
    head = torch.randn((512, 1000), generator=g, device="cuda").bfloat16() * 0.05
    tokens = torch.tensor([1, 2, 3], device="cuda")
    table, kv_lens = cache.table.clone(), cache.lens.clone()

    def step():
        npu.cascade_quant_write(x[:, 4:6], x[:, 6:8], *cache.pools[:2], slots)
        o, lse = npu.cascade_quant_decode(x[:, :4].contiguous(), *cache.pools[:2], table, torch.ones_like(kv_lens), kv_lens, 1, SCALE)
        return (o, lse, *npu.cascade_token_logprobs(o.view(3, 512) @ head, tokens, 4))

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for seed in range(3):
        x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
        tokens.copy_(torch.randint(0, 1000, (3,), generator=g, device="cuda"))
        kv_lens.copy_(torch.tensor([[31, 8, 65], [31, 0, 65], [5, 8, 65]][seed], device="cuda"))
        graph.replay()
        got = [t.clone() for t in outs]
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


@pytest.mark.parametrize("q_len,G", [(1, 4), (3, 5), (40, 4)])
def test_stalled_attention_ends_with_an_error_status(q_len, G):
    import torch
    Hh.need_cuda()
    C = Hh.capi()
    cache, _, g = _filled([290, 64, 40])
    q = torch.randn((3 * q_len, 2 * G, 128), generator=g, device="cuda").bfloat16()
    out, lse = torch.empty_like(q), torch.empty(q.shape[0] * q.shape[1], device="cuda")

    def call(flags):
        d = C.quant_desc(q, *cache.pools[:2], cache.table, None, cache.lens, q_len, SCALE, flags=flags)
        ws = torch.zeros(C.quant_decode_workspace_size(d), dtype=torch.uint8, device="cuda")
        C.quant_decode(d, out, lse, ws)
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
