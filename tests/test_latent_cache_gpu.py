"""LatentCache against a host model that keeps every row's tokens by themselves: no row sees another's writes, and the
counts are the table's references."""
import numpy as np
import pytest

import helpers as Hh

pytestmark = pytest.mark.gpu


class Model:
    """A cache of `layers` pools and, per row, the tokens it should hold (None: a row that could not be made)."""

    def __init__(self, layers=2, blocks=60, page=16, rows=1, cols=8, seed=0):
        import torch
        from cascade_kernel.latent import LatentCache
        self.cache = LatentCache(layers, blocks, page, rows, cols)
        self.rows = [np.zeros((layers, 0, 576), np.float32) for _ in range(rows)]
        self.g = torch.Generator(device="cuda").manual_seed(seed)
        self.layers = layers

    def grow(self, counts):
        import torch
        self.cache.grow(torch.tensor(counts, dtype=torch.int64, device="cuda"))
        new = [torch.randn((sum(counts), 576), generator=self.g, device="cuda").bfloat16() for _ in range(self.layers)]
        for i, x in enumerate(new):
            self.cache.write(i, x, counts)
        x = np.stack([t.float().cpu().numpy() for t in new])
        at = 0
        for r, n in enumerate(counts):
            if n:
                self.rows[r] = np.concatenate([self.rows[r], x[:, at:at + n]], 1)
            at += n

    def fork(self, parents):
        import torch
        self.cache.fork(torch.tensor(parents, dtype=torch.int64, device="cuda"))
        made = (self.cache.lens >= 0).tolist()
        self.rows = [self.rows[p] if ok else None for p, ok in zip(parents, made)]

    def truncate(self, keep):
        import torch
        self.cache.truncate(torch.tensor(keep, dtype=torch.int64, device="cuda"))
        self.rows = [x if x is None else x[:, :max(k, 0)] for x, k in zip(self.rows, keep)]

    def check(self):
        import torch
        c = self.cache
        assert c.lens.tolist() == [-1 if x is None else x.shape[1] for x in self.rows]
        flat = c.table[c.table >= 0].long()
        assert torch.equal(torch.bincount(flat, minlength=c.refs.numel()).int(), c.refs)
        for r, x in enumerate(self.rows):
            n = 0 if x is None else x.shape[1]
            pages = (n + c.page - 1) // c.page
            assert (c.table[r] >= 0).tolist() == [j < pages for j in range(c.table.shape[1])]
            for i in range(self.layers if n else 0):
                got = c.pools[i][c.table[r, :pages].long()].reshape(-1, 576)[:n]
                assert np.array_equal(got.float().cpu().numpy(), x[i]), (r, i)


def test_row_cut_inside_a_shared_page_grows_into_its_own():
    """Row 1 is cut to 40 of the 64 tokens that four rows share, and goes on: the others keep tokens 40 to 47."""
    Hh.need_cuda()
    m = Model()
    m.grow([64])
    m.fork([0, 0, 0, 0])
    m.truncate([64, 40, 64, 64])
    m.grow([0, 5, 0, 0])
    m.check()
    assert int(m.cache.refs[m.cache.table[1, 2].long()]) == 1


def test_rows_cut_inside_one_page_part():
    """All holders of a page go on from inside it: one keeps the page, the others get copies, before any of them writes."""
    Hh.need_cuda()
    m = Model(blocks=7)
    m.grow([48])
    m.fork([0, 0, 0])
    m.truncate([41, 35, 48])
    m.truncate([41, 35, 46])
    m.grow([3, 1, 2])  # 3 pages of the prompt and 2 copies
    m.check()
    assert int((m.cache.refs > 0).sum()) == 5
    # a holder that does not go on keeps what it sees
    m.fork([0, 0])
    m.truncate([40, 30])
    m.grow([0, 7])
    m.check()


def test_copies_of_shared_pages_count_as_pages():
    import torch
    Hh.need_cuda()
    m = Model(blocks=4)
    m.grow([64])
    m.fork([0, 0])
    m.truncate([64, 40])
    with pytest.raises(RuntimeError, match="1 pages needed, 0 free"):
        m.cache.grow(torch.tensor([0, 1], device="cuda"))
    m.check()  # a refused growth leaves everything as it was


@pytest.mark.parametrize("seed", range(4))
def test_random_steps_leave_every_row_its_own_tokens(seed):
    Hh.need_cuda()
    rng = np.random.default_rng(seed)
    m = Model(blocks=200, page=16, cols=12, seed=seed)
    m.grow([int(rng.integers(1, 100))])
    m.fork([0] * 4)
    for _ in range(12):
        lens = [x.shape[1] for x in m.rows]
        step = rng.integers(0, 3)
        if step == 0:
            m.fork(rng.integers(0, len(lens), int(rng.integers(1, 6))).tolist())
        elif step == 1:
            m.truncate([int(rng.integers(0, n + 1)) if rng.random() < 0.5 else n for n in lens])
        else:
            m.grow([int(rng.integers(0, min(20, 192 - n) + 1)) for n in lens])
        m.check()
    assert Hh.capi().device_error() == 0


def test_row_that_could_not_be_made_stays_so():
    """A fork that runs out of pages leaves a row of length -1: it cannot grow, be written or become an empty row by itself."""
    import torch
    Hh.need_cuda()
    m = Model(blocks=4, cols=4)
    m.grow([20])
    m.fork([0, 0, 0])  # 2 pages, 2 free ones for the last page's copies
    assert m.cache.lens.tolist() == [20, 20, -1]
    m.check()
    with pytest.raises(RuntimeError, match="row 2"):
        m.cache.grow(torch.tensor([0, 0, 1], device="cuda"))
    with pytest.raises(RuntimeError, match="no token"):
        m.cache.write(0, torch.ones((1, 576), dtype=torch.bfloat16, device="cuda"), [0, 0, 1])
    m.check()
    m.grow([1, 2, 0])
    m.truncate([21, 21, 30])
    m.check()
    m.fork([1, 2])
    assert m.cache.lens.tolist() == [21, -1]
    m.check()
    m.truncate([21, 0])  # an empty row, from now on like any other
    m.rows[1] = m.rows[0][:, :0]
    m.grow([0, 3])
    m.check()


def test_write_refuses_places_outside_the_rows():
    import torch
    Hh.need_cuda()
    m = Model()
    m.grow([3])
    with pytest.raises(RuntimeError, match="no token"):
        m.cache.write(0, torch.ones((4, 576), dtype=torch.bfloat16, device="cuda"), [4])
    with pytest.raises(RuntimeError, match="row 0"):
        m.cache.grow(torch.tensor([-1], device="cuda"))
    m.check()
