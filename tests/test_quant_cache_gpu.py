"""Rows of a 4-bit cache on the GPU: written bytes equal the oracle's, values read back are the oracle's to half a step."""
import numpy as np
import pytest

import helpers as Hh
from oracle import quant_oracle as Q

pytestmark = pytest.mark.gpu


def _rows(T, KVH, dtype, seed=0, scale=1.0):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = {"bf16": torch.bfloat16, "fp16": torch.float16}[dtype]
    return [(torch.randn((T, KVH, 128), generator=g, device="cuda") * scale).to(t) for _ in range(2)]


def _caches(blocks, page, KVH, fill=0):
    import torch
    return [torch.full((blocks, page, KVH, 80), fill, dtype=torch.uint8, device="cuda") for _ in range(2)]


@pytest.mark.parametrize("T,KVH,page,dtype", [(1, 1, 16, "bf16"), (3, 5, 16, "fp16"), (17, 8, 32, "bf16"), (64, 2, 16, "fp16"),
                                              (1000, 4, 64, "bf16"), (333, 3, 512, "fp16"), (4097, 8, 128, "bf16"),
                                              (20, 70, 16, "bf16"), (50, 1, 1, "fp16")])
def test_write_is_the_definition_bit_for_bit(T, KVH, page, dtype):
    import torch
    Hh.need_cuda()
    k, v = _rows(T, KVH, dtype, seed=T)
    k[:, :, 7] *= 30
    v[T // 2] = 0
    blocks = (T + page - 1) // page + 3
    kc, vc = _caches(blocks, page, KVH, fill=0xA5)
    g = torch.Generator(device="cuda").manual_seed(1)
    slots = torch.randperm(blocks * page, generator=g, device="cuda")[:T]
    Hh.ops().cascade_quant_write(k, v, kc, vc, slots)
    for x, c in ((k, kc), (v, vc)):
        flat = c.view(-1, KVH, 80)
        assert torch.equal(flat[slots].cpu(), Q.pack(x))
        rest = torch.ones(blocks * page, dtype=torch.bool, device="cuda")
        rest[slots] = False
        assert bool((flat[rest] == 0xA5).all())
    assert Hh.capi().device_error() == 0


@pytest.mark.parametrize("scale", [1e-7, 1e-5, 1e-3, 300.0, 9000.0])
def test_write_over_the_range(scale):
    import torch
    Hh.need_cuda()
    k, v = _rows(100, 4, "fp16" if scale < 1 else "bf16", seed=3, scale=scale)
    k, v = k.clamp(-32768, 32768), v.clamp(-32768, 32768)
    k[5] += scale * 50
    kc, vc = _caches(7, 16, 4)
    slots = torch.arange(100, device="cuda")
    Hh.ops().cascade_quant_write(k.clamp(-32768, 32768), v, kc, vc, slots)
    assert torch.equal(kc.view(-1, 4, 80)[:100].cpu(), Q.pack(k.clamp(-32768, 32768)))
    assert torch.equal(vc.view(-1, 4, 80)[:100].cpu(), Q.pack(v))


@pytest.mark.parametrize("bad", ["nan", "inf", "-inf", "33000"])
def test_a_group_that_cannot_be_held_reads_back_as_nan(bad):
    import torch
    Hh.need_cuda()
    k, v = _rows(40, 2, "bf16", seed=4)
    k[3, 1, 64 + 17] = float(bad)
    v[39, 0, 0] = float(bad)
    kc, vc = _caches(3, 16, 2)
    slots = torch.arange(40, device="cuda")
    Hh.ops().cascade_quant_write(k, v, kc, vc, slots)
    assert torch.equal(kc.view(-1, 2, 80)[:40].cpu(), Q.pack(k))
    rk, rv = Hh.ops().cascade_quant_read(kc, vc, slots, torch.float32)
    assert bool(rk[3, 1, 64:96].isnan().all()) and int(rk.isnan().sum()) == 32
    assert bool(rv[39, 0, :32].isnan().all()) and int(rv.isnan().sum()) == 32


def test_write_takes_views_and_passes_slots_by():
    import torch
    Hh.need_cuda()
    T, KVH, H = 37, 4, 12
    g = torch.Generator(device="cuda").manual_seed(5)
    qkv = torch.randn((T, H + 2 * KVH, 128), generator=g, device="cuda").half()     # one projection's rows
    k, v = qkv[:, H : H + KVH], qkv[:, H + KVH :]
    kc, vc = _caches(4, 16, KVH, fill=0x11)
    slots = torch.arange(T, device="cuda") + 20
    slots[[0, 9]] = torch.tensor([-1, -(1 << 40)], device="cuda")
    slots[[12, 36]] = torch.tensor([64, 1 << 50], device="cuda")                    # past the cache
    Hh.ops().cascade_quant_write(k, v, kc, vc, slots)
    assert Hh.capi().device_error() == 2
    kept = torch.tensor([i for i in range(T) if i not in (0, 9, 12, 36)], device="cuda")
    assert torch.equal(kc.view(-1, KVH, 80)[slots[kept]].cpu(), Q.pack(k[kept]))
    assert torch.equal(vc.view(-1, KVH, 80)[slots[kept]].cpu(), Q.pack(v[kept]))
    untouched = torch.ones(64, dtype=torch.bool, device="cuda")
    untouched[slots[kept]] = False
    assert bool((kc.view(-1, KVH, 80)[untouched] == 0x11).all()) and bool((vc.view(-1, KVH, 80)[untouched] == 0x11).all())
    rk, rv = Hh.ops().cascade_quant_read(kc, vc, slots, torch.float16)
    assert Hh.capi().device_error() == 2
    for i in (0, 9, 12, 36):
        assert not rk[i].any() and not rv[i].any()
    # heads in another order than the tokens', one key row for all tokens
    k2, v2 = qkv[:, :KVH].transpose(0, 1).contiguous().transpose(0, 1), qkv[:1, :KVH].expand(T, KVH, 128)
    slots = torch.arange(T, device="cuda")
    Hh.ops().cascade_quant_write(k2, v2, kc, vc, slots)
    assert torch.equal(kc.view(-1, KVH, 80)[:T].cpu(), Q.pack(k2)) and torch.equal(vc.view(-1, KVH, 80)[:T].cpu(), Q.pack(v2))


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("T,KVH,page", [(1, 1, 16), (5, 3, 32), (700, 8, 16), (3001, 2, 128)])
def test_read(T, KVH, page, dtype):
    import torch
    Hh.need_cuda()
    k, v = _rows(page * 40, KVH, "fp16", seed=6)
    caches = [Q.pack(x).cuda().view(40, page, KVH, 80) for x in (k, v)]
    t = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}[dtype]
    g = torch.Generator(device="cuda").manual_seed(7)
    slots = torch.randint(0, 40 * page, (T,), generator=g, device="cuda")   # some more than once
    got = Hh.ops().cascade_quant_read(*caches, slots, t)
    for x, c in zip(got, caches):
        want = Q.values(c.view(-1, KVH, 80)[slots])
        assert x.dtype == t and x.shape == (T, KVH, 128)
        # one fp32 rounding, then one to the type: half a step each, and the type's smallest number
        tol = want.abs() * (torch.finfo(t).eps / 2 + 2.0 ** -24) * 1.001 + torch.finfo(t).smallest_normal * torch.finfo(t).eps
        assert bool(((x.double() - want).abs() <= tol).all())


def test_offsets_past_32_bits():
    """A cache of 2.7 GB: rows at its start and end."""
    import torch
    Hh.need_cuda()
    page, KVH = 64, 8
    blocks = (1 << 31) // (page * KVH * 80) + 15000
    k, v = _rows(64, KVH, "bf16", seed=8)
    kc, vc = _caches(blocks, page, KVH)
    slots = torch.cat([torch.arange(32, device="cuda"), blocks * page - 1 - torch.arange(32, device="cuda")])
    Hh.ops().cascade_quant_write(k, v, kc, vc, slots)
    assert torch.equal(kc.view(-1, KVH, 80)[slots].cpu(), Q.pack(k)) and torch.equal(vc.view(-1, KVH, 80)[slots].cpu(), Q.pack(v))
    rk, rv = Hh.ops().cascade_quant_read(kc, vc, slots, torch.float32)
    assert torch.equal(rk, Q.values(Q.pack(k).cuda()).float()) and torch.equal(rv, Q.values(Q.pack(v).cuda()).float())


def test_nothing_to_do_and_refusals():
    import torch
    Hh.need_cuda()
    ops = Hh.ops()
    kc, vc = _caches(2, 16, 4)
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    k, v = _rows(3, 4, "bf16")
    ops.cascade_quant_write(k[:0], v[:0], kc, vc, none)
    rk, rv = ops.cascade_quant_read(kc, vc, none, torch.bfloat16)
    assert rk.shape == rv.shape == (0, 4, 128)
    s = torch.arange(3, device="cuda")
    for args, text in [((k.float(), v.float(), kc, vc, s), "bf16 or fp16"), ((k, v.half(), kc, vc, s), "its type"),
                       ((k[:, :3], v[:, :3], kc, vc, s), "kv heads, 128"), ((k, v[:2], kc, vc, s), "key's shape"),
                       ((k, v, kc, vc[:1], s), "equal shapes"), ((k, v, kc, vc, s.int()), "slots must be"),
                       ((k, v, kc, vc, s[:2]), "per token"), ((k, v, kc, kc, s), "two caches"),
                       ((k, v, kc.view(2, 16, 2, 160), vc.view(2, 16, 2, 160), s), "kv heads, 80"),
                       ((k, v, kc.cpu(), vc, s), "must be on"), ((k.cpu(), v.cpu(), kc, vc, s), "CUDA"),
                       ((k.transpose(1, 2).contiguous().transpose(1, 2), v, kc, vc, s), "last dimension")]:
        with pytest.raises((RuntimeError, NotImplementedError), match=None if text == "CUDA" else text):
            ops.cascade_quant_write(*args)
    with pytest.raises(RuntimeError, match="bf16, fp16 or fp32"):
        ops.cascade_quant_read(kc, vc, s, torch.float64)
    assert not kc.any() and not vc.any()


def test_another_stream_and_a_graph():
    import torch
    Hh.need_cuda()
    k, v = _rows(300, 8, "bf16", seed=9)
    kc, vc = _caches(20, 16, 8)
    slots = torch.randperm(320, device="cuda")[:300]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        Hh.ops().cascade_quant_write(k, v, kc, vc, slots)
        got = Hh.ops().cascade_quant_read(kc, vc, slots, torch.bfloat16)
    torch.cuda.current_stream().wait_stream(side)
    want = [Q.values(Q.pack(x).cuda()).float().bfloat16() for x in (k, v)]
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        Hh.ops().cascade_quant_write(k, v, kc, vc, slots)
        again = Hh.ops().cascade_quant_read(kc, vc, slots, torch.bfloat16)
    kc.zero_(), vc.zero_()
    k.copy_(k.flip(0))
    slots.copy_(torch.arange(320, device="cuda")[20:])
    graph.replay()
    assert torch.equal(again[0], want[0].flip(0)) and torch.equal(again[1], want[1])
    assert not kc.view(-1)[: 20 * 640].any() and np.isfinite(Hh.dev_to_f64(again[0])).all()
