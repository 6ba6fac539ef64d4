"""Pages of a cache on the GPU (cascade_page_copy / _fork / _free / _compact)
against a plain host version; every result is whole numbers or copied bytes, so
everything has to be equal."""
import numpy as np
import pytest

import helpers as Hh

pytestmark = pytest.mark.gpu


def _state(seed, lens, page, blocks, cols=None, layers=2, width=24, shared=0):
    """Pools, table, lengths and counts: rows own random pages; `shared` rows repeat an earlier row's full pages."""
    import torch
    rng = np.random.default_rng(seed)
    need = [(n + page - 1) // page for n in lens]
    cols = max(1, max(need, default=1)) if cols is None else cols
    order = rng.permutation(blocks)
    bt = np.full((len(lens), cols), -1, np.int32)
    refs = np.zeros(blocks, np.int32)
    c = 0
    for r in range(len(lens)):
        for j in range(need[r]):
            src = r - 1 if r and r <= shared and j < min(lens[r], lens[r - 1]) // page else None
            bt[r, j] = bt[src, j] if src is not None else order[c]
            c += src is None
            refs[bt[r, j]] += 1
    g = torch.Generator(device="cuda").manual_seed(seed)
    pools = [torch.randint(-9999, 9999, (blocks, page, width), generator=g, device="cuda", dtype=torch.int16)
             for _ in range(layers)]
    return pools, torch.from_numpy(bt).cuda(), torch.tensor(lens, dtype=torch.int64).cuda(), torch.from_numpy(refs).cuda()


def _fork_want(pools, bt, lens, refs, parents):
    pools, bt, lens, refs = [p.cpu().numpy().copy() for p in pools], bt.cpu().numpy(), lens.cpu().numpy(), refs.cpu().numpy().copy()
    page = pools[0].shape[1]
    free = [i for i in range(len(refs)) if refs[i] == 0]
    old = [p.copy() for p in pools]
    table = np.full((len(parents), bt.shape[1]), -1, np.int32)
    out = np.full(len(parents), -1, np.int64)
    for i, p in enumerate(parents):
        if not 0 <= p < len(lens):
            continue
        n = int(lens[p])
        full, tail = n // page, n % page
        if tail and not free:
            continue
        out[i] = n
        table[i, :full] = bt[p, :full]
        np.add.at(refs, bt[p, :full], 1)
        if tail:
            new = free.pop(0)
            table[i, full] = new
            refs[new] = 1
            for a, b in zip(pools, old):
                a[new, :tail] = b[bt[p, full], :tail]
    return table, out, refs, pools


def _fork_case(state, parents):
    import torch
    want = _fork_want(*state, parents)
    got = Hh.ops().cascade_page_fork(*state, torch.tensor(parents, dtype=torch.int64, device="cuda"))
    for g, w in zip(got, want[:3]):
        assert np.array_equal(g.cpu().numpy(), w)
    for g, w in zip(state[0], want[3]):
        assert np.array_equal(g.cpu().numpy(), w)


@pytest.mark.parametrize("page", [16, 64, 7])
@pytest.mark.parametrize("layers", [1, 3])
def test_fork(page, layers):
    Hh.need_cuda()
    lens = [0, 1, page - 1, page, page + 1, 5 * page, 5 * page + 3, 300]
    rng = np.random.default_rng(page)
    parents = rng.integers(0, len(lens), 50).tolist()
    _fork_case(_state(page, lens, page, 400, layers=layers), parents)


@pytest.mark.parametrize("spare", [0, 1, 5])
def test_fork_runs_out_of_pages(spare):
    Hh.need_cuda()
    lens = [33, 16, 50, 5]
    used = sum((n + 15) // 16 for n in lens)
    _fork_case(_state(spare, lens, 16, used + spare), [0, 1, 2, 3, 3, 1, 0, 2, 2, 0])


def test_fork_bad_parents_and_no_children():
    Hh.need_cuda()
    _fork_case(_state(1, [20, 40], 16, 30), [0, -1, 2, 1, 1 << 40])
    _fork_case(_state(1, [20, 40], 16, 30), [])


def test_fork_large_tables():
    Hh.need_cuda()
    rng = np.random.default_rng(0)
    lens = rng.integers(0, 4000, 120).tolist()
    _fork_case(_state(2, lens, 16, 40000, layers=1), rng.integers(0, 120, 700).tolist())


def test_fork_more_pools_than_one_launch_takes():
    Hh.need_cuda()
    _fork_case(_state(3, [20, 33], 16, 12, layers=131, width=8), [1, 0, 1])


@pytest.mark.parametrize("shared", [0, 3])
@pytest.mark.parametrize("page", [16, 64, 5])
def test_free(page, shared):
    import torch
    Hh.need_cuda()
    lens = [0, 1, page, page + 1, 9 * page, 9 * page + 2, 200, 3]
    pools, bt, kv, refs = _state(page, lens, page, 300, shared=shared)
    keep = [0, 1, 0, 1, 4 * page, 4 * page + 1, 500, -5]
    table, out, got = Hh.ops().cascade_page_free(bt, kv, refs, torch.tensor(keep, dtype=torch.int64, device="cuda"), page)
    w_refs, w_table = refs.cpu().numpy().copy(), bt.cpu().numpy().copy()
    w_len = np.minimum(np.maximum(keep, 0), lens)
    for r, (n, k) in enumerate(zip(lens, w_len)):
        hold, have = -(-k // page), -(-n // page)
        np.subtract.at(w_refs, w_table[r, hold:have], 1)
        w_table[r, hold:] = -1
    assert np.array_equal(out.cpu().numpy(), w_len) and np.array_equal(table.cpu().numpy(), w_table)
    assert np.array_equal(got.cpu().numpy(), w_refs)


def test_free_undoes_fork():
    import torch
    Hh.need_cuda()
    state = _state(4, [100, 37, 0, 64], 16, 60)
    child, n, refs = Hh.ops().cascade_page_fork(*state, torch.tensor([0, 1, 2, 3, 1], device="cuda"))
    _, _, back = Hh.ops().cascade_page_free(child, n, refs, torch.zeros_like(n), 16)
    assert torch.equal(back, state[3])


def _compact_case(state):
    pools, bt, lens, refs = state
    w_pools, w_bt, w_refs = [p.cpu().numpy().copy() for p in pools], bt.cpu().numpy(), refs.cpu().numpy()
    page = pools[0].shape[1]
    live = [i for i in range(len(w_refs)) if w_refs[i] > 0]
    n = len(live)
    src, dst = [i for i in live if i >= n], [i for i in range(n) if w_refs[i] <= 0]
    to = np.arange(len(w_refs))
    to[src] = dst
    new = np.zeros_like(w_refs)
    new[to[live]] = w_refs[live]
    for p in w_pools:
        p[dst] = p[src]
    table = np.full_like(w_bt, -1)
    for r, m in enumerate(lens.cpu().tolist()):
        have = -(-m // page)
        table[r, :have] = to[w_bt[r, :have]]
    got = Hh.ops().cascade_page_compact(pools, bt, lens, refs)
    assert np.array_equal(got[0].cpu().numpy(), table)
    assert np.array_equal(got[1].cpu().numpy(), new) and int(got[2]) == n
    for g, w in zip(pools, w_pools):
        assert np.array_equal(g.cpu().numpy(), w)


@pytest.mark.parametrize("blocks", [40, 41, 100, 5000, 30001])
@pytest.mark.parametrize("shared", [0, 2])
def test_compact(blocks, shared):
    Hh.need_cuda()
    _compact_case(_state(blocks, [100, 120, 130, 1, 0, 200], 16, blocks, shared=shared))


def test_compact_edges():
    Hh.need_cuda()
    _compact_case(_state(0, [0, 0], 16, 9))            # nothing live
    _compact_case(_state(0, [160], 16, 10))            # everything live
    _compact_case(_state(0, [1], 16, 1))


def test_copy():
    import torch
    Hh.need_cuda()
    pools = _state(5, [16], 16, 64, layers=3, width=40)[0]
    want = [p.clone() for p in pools]
    src = torch.tensor([3, 3, 7, 60], dtype=torch.int64, device="cuda")
    dst = torch.tensor([10, 11, 63, 0], dtype=torch.int64, device="cuda")
    for w in want:
        w[dst] = w[src]
    Hh.ops().cascade_page_copy(pools, src, dst)
    for p, w in zip(pools, want):
        assert torch.equal(p, w)
    C = Hh.capi()
    for w in want:
        w[20] = w[5]
    C.page_copy(pools, torch.tensor([5, 64, -1], device="cuda"), torch.tensor([20, 1, 2], device="cuda"))
    assert C.device_error() & 2 and C.device_error() == 0   # two ids outside the pools, skipped
    for p, w in zip(pools, want):
        assert torch.equal(p, w)


def test_copy_of_large_pools_past_32_bits():
    import torch
    Hh.need_cuda()
    pool = torch.zeros((1 << 17, 64, 600), dtype=torch.int8, device="cuda")   # 5 GB, rows of 600 bytes: refused
    src, dst = torch.tensor([1], device="cuda"), torch.tensor([(1 << 17) - 1], device="cuda")
    with pytest.raises(RuntimeError, match="16 bytes"):
        Hh.ops().cascade_page_fork([pool], torch.zeros((1, 1), dtype=torch.int32, device="cuda"), src,
                                   torch.zeros(1 << 17, dtype=torch.int32, device="cuda"), src)
    pool[1] = torch.randint(-100, 100, (64, 600), dtype=torch.int8, device="cuda")
    Hh.ops().cascade_page_copy([pool], src, dst)              # whole pages are a multiple of 16
    assert torch.equal(pool[-1], pool[1]) and int(pool[-2].abs().max()) == 0


def test_pages_in_a_graph():
    import torch
    Hh.need_cuda()
    state = _state(6, [100, 37, 20], 16, 60)
    parents = torch.tensor([0, 1, 1], device="cuda")
    want = Hh.ops().cascade_page_fork(*state, parents)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            got = Hh.ops().cascade_page_fork(*state, parents)
        g.replay()
    side.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a, b)


def test_refusals():
    import torch
    Hh.need_cuda()
    npu = Hh.ops()
    pools, bt, kv, refs = _state(7, [20, 40], 16, 30)
    par = torch.zeros(2, dtype=torch.int64, device="cuda")
    bad = [
        (lambda: npu.cascade_page_fork([], bt, kv, refs, par), "at least one pool"),
        (lambda: npu.cascade_page_fork([pools[0], pools[1][:-1]], bt, kv, refs, par), "equal shapes"),
        (lambda: npu.cascade_page_fork(pools, bt, kv, refs[:-1].contiguous(), par), "entry per page"),
        (lambda: npu.cascade_page_fork(pools, bt, kv, refs, par.int()), "parents must be"),
        (lambda: npu.cascade_page_fork(pools, bt.long(), kv, refs, par), "block_table must be"),
        (lambda: npu.cascade_page_fork(pools, bt, kv[:1], refs, par), "have its rows"),
        (lambda: npu.cascade_page_fork([p.transpose(0, 1) for p in pools], bt, kv, refs, par), "contiguous"),
        (lambda: npu.cascade_page_free(bt, kv, refs, par[:1], 16), "entry per row"),
        (lambda: npu.cascade_page_free(bt, kv, refs, par, 0), "block size"),
        (lambda: npu.cascade_page_compact(pools, bt, kv, refs.long()), "page_refs must be"),
        (lambda: npu.cascade_page_copy(pools, par, par[:1]), "equally long"),
    ]
    for call, text in bad:
        with pytest.raises(RuntimeError, match=text):
            call()


def test_lengths_near_the_end_of_64_bits():
    """A length that no table holds: no child can be made of such a row, freeing and compacting see all its columns."""
    import torch
    Hh.need_cuda()
    for n in ((1 << 63) - 1, (1 << 63) - 16, 1 << 62):
        pools, bt, lens, refs = _state(3, [64, 40], 16, 9, cols=4)
        lens[0] = n
        table, out, counts = Hh.ops().cascade_page_fork(pools, bt, lens, refs, torch.tensor([0, 1, 0], device="cuda"))
        assert out.tolist() == [-1, 40, -1] and (table[0] == -1).all() and (table[2] == -1).all()
        assert torch.equal(counts, refs + torch.bincount(table[1, :3].long(), minlength=9).int())
        keep = torch.tensor([n, 40], device="cuda")
        table, out, counts = Hh.ops().cascade_page_free(bt, lens, refs, keep, 16)
        assert torch.equal(table, bt) and out.tolist() == [n, 40] and torch.equal(counts, refs)
        table, out, counts = Hh.ops().cascade_page_free(bt, lens, refs, torch.tensor([17, 40], device="cuda"), 16)
        assert torch.equal(table[0, :2], bt[0, :2]) and (table[0, 2:] == -1).all() and out.tolist() == [17, 40]
        assert int(counts.sum()) == int(refs.sum()) - 2
        old = [p.clone() for p in pools]
        table, counts, live = Hh.ops().cascade_page_compact(pools, bt, lens, refs)
        assert int(live) == 7 and (table[0] >= 0).all()
        for p, o in zip(pools, old):
            assert torch.equal(p[table[0].long()], o[bt[0].long()])
    assert Hh.capi().device_error() == 0
