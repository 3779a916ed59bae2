"""GPU parity of assign_pages / release_pages with the oracle: whole numbers, so every output
and the whole pool must be equal."""
import numpy as np
import pytest
import torch

from fast_v2_amd import ops
from oracle import paged_step as ps

pytestmark = pytest.mark.gpu


class _Pool:
    """The same pool twice: the oracle's and the GPU's."""

    def __init__(self, gpu, lens, max_pages, page, spare, rng, stride=0):
        B = len(lens)
        have = [-(-max(n, 0) // page) for n in lens]
        self.page, self.size = page, sum(have) + spare
        ids = rng.permutation(self.size)
        self.table = np.full((B, max_pages), -7, np.int64)
        at = 0
        for b, h in enumerate(have):
            self.table[b, :h] = ids[at:at + h]
            at += h
        self.lens, self.free = [int(n) for n in lens], ids[at:].tolist()
        self.g_lens = torch.tensor(self.lens, dtype=torch.int32, device=gpu)
        wide = torch.full((B, max(stride, max_pages)), -9, dtype=torch.int32, device=gpu)
        wide[:, :max_pages] = torch.from_numpy(self.table).int().to(gpu)
        self.g_wide, self.g_table = wide, wide[:, :max_pages]
        self.g_free = torch.full((self.size + 3,), -5, dtype=torch.int32, device=gpu)
        self.g_free[:len(self.free)] = torch.tensor(self.free, dtype=torch.int32)
        self.g_count = torch.tensor([len(self.free)], dtype=torch.int32, device=gpu)

    def gpu(self):
        return self.g_lens, self.g_table, self.g_free, self.g_count, self.page

    def check(self):
        assert self.g_lens.tolist() == self.lens
        assert int(self.g_count) == len(self.free)
        assert self.g_free[:len(self.free)].tolist() == self.free
        assert np.array_equal(self.g_table.cpu().numpy(), self.table)
        assert (self.g_wide[:, self.g_table.shape[1]:] == -9).all() and (self.g_free[self.size:] == -5).all()

    def assign(self, new, width=0, rows=0, as_given=None):
        want = ps.assign_pages_np(new, self.lens, self.table, self.free, self.page, width, rows)
        given = torch.tensor(new, dtype=torch.int32, device=self.g_lens.device) if as_given is None else as_given
        got = ops.assign_pages(given, *self.gpu(), width=width, rows=rows)
        for name in ("slots", "positions", "starts", "seqlens", "granted"):
            assert np.array_equal(getattr(got, name).flatten().cpu().numpy(), want[name]), name
        if width:
            assert got.slots.shape == (len(new), width) and got.sequences is None and got.row_starts is None
        else:
            assert np.array_equal(got.sequences.cpu().numpy(), want["sequences"])
            assert got.row_starts.tolist() == want["row_starts"]
        assert got.slots.dtype == torch.int64 and got.positions.dtype == torch.int32
        self.check()
        return got, want

    def release(self, keep):
        ps.release_pages_np(keep, self.lens, self.table, self.free, self.page)
        ops.release_pages(torch.tensor(keep, dtype=torch.int32, device=self.g_lens.device), *self.gpu())
        self.check()


@pytest.mark.parametrize("page", [1, 16, 32, 64])
@pytest.mark.parametrize("B", [1, 7, 64, 300, 1024, 1025, 2500, 8192])
@pytest.mark.parametrize("width", [0, 1, 8])
def test_steps(gpu, B, page, width):
    """Several steps with releases between; the pool runs out on the way."""
    print(f"case pages B={B} page={page} width={width}", flush=True)
    rng = np.random.default_rng(B * 100 + page + width)
    most = 70 if page == 1 else 9
    lens = rng.integers(0, 5 * page if page > 1 else 40, B)
    pool = _Pool(gpu, lens, most, page, spare=max(3, B * 3 if page == 1 else B // 2), rng=rng, stride=most + 3)
    for step in range(4):
        if width:
            new = rng.integers(-1, width + 2, B)
            pool.assign(new.tolist(), width=width)
        else:
            new = np.where(rng.random(B) < 0.1, rng.integers(0, 3 * page + 2, B), rng.integers(0, 3, B))
            pool.assign(new.tolist(), rows=max(1, int(new.sum()) + (-5, 0, 7, 100)[step]))
        keep = np.where(rng.random(B) < 0.3, rng.integers(-2, 4 * page, B), 2 ** 31 - 1)
        pool.release(keep.tolist())
    pool.release([0] * B)


def test_a_step_taken_back(gpu):
    rng = np.random.default_rng(3)
    pool = _Pool(gpu, rng.integers(0, 500, 200).tolist(), 24, 32, 400, rng)
    before = [t.clone() for t in pool.gpu()[:4]]
    got, _ = pool.assign(rng.integers(0, 60, 200).tolist(), width=64)
    pool.release(got.starts.tolist())
    for a, b, name in zip(before, pool.gpu()[:4], ("lens", "table", "free", "count")):
        if name != "table":
            assert torch.equal(a, b), name


def test_long_prompts(gpu):
    """Whole prompts beside single tokens: pages of one request spread over all threads."""
    rng = np.random.default_rng(4)
    pool = _Pool(gpu, [0, 100, 0, 31, 7], 5000, 16, 9000, rng)
    new = [65000, 1, 40001, 1, 0]
    pool.assign(new, rows=sum(new) + 11)
    pool.release([1, 101, 20000, 0, 7])


def test_numbers_at_their_limits(gpu):
    rng = np.random.default_rng(5)
    big = 2 ** 31 - 1
    pool = _Pool(gpu, [5, -3, 0, 12, 16], 3, 16, 2, rng)
    pool.assign([big, big, -big, 4, 1], rows=40)       # what cannot be held asks for nothing
    pool.assign([big, 1, big, big, 0], rows=big // 2 ** 16)
    pool.release([big, -big, 0, 3, 2])
    # 64-bit requests beyond 32 bits are not taken for small ones
    new = torch.tensor([2 ** 32 + 1, -2 ** 40, 2, 0, 0], device=gpu)
    pool.assign([big, -big, 2, 0, 0], width=8, as_given=new)


def test_large_page_ids(gpu):
    """Slots past 32 bits: page ids near their type's end."""
    rng = np.random.default_rng(10)
    pool = _Pool(gpu, [70, 0, 64], 4, 64, 5, rng)
    far = 2 ** 31 - 1 - np.arange(pool.size)
    pool.free = far[:len(pool.free)].tolist()
    pool.g_free[:len(pool.free)] = torch.tensor(pool.free, dtype=torch.int32, device=gpu)
    got, want = pool.assign([100, 1, 1], rows=102)
    assert got.slots.max() > 2 ** 36
    pool.release([0, 0, 0])


def test_no_pages_no_room(gpu):
    rng = np.random.default_rng(6)
    pool = _Pool(gpu, [30, 32, 0], 2, 32, 0, rng)
    got, _ = pool.assign([2, 1, 1], width=2)
    assert got.granted.tolist() == [2, 0, 0]
    pool.g_count.fill_(-4)  # a count outside of the list counts as its nearest end
    got = ops.assign_pages(torch.tensor([0, 1, 1], dtype=torch.int32, device=gpu), *pool.gpu(), width=1)
    assert got.granted.tolist() == [0, 0, 0] and int(pool.g_count) == 0


def test_empty_batch(gpu):
    i = torch.zeros(0, dtype=torch.int32, device=gpu)
    one = torch.zeros(1, dtype=torch.int32, device=gpu)
    got = ops.assign_pages(i, i, torch.zeros(0, 4, dtype=torch.int32, device=gpu), one, one, 16, width=8)
    assert got.slots.shape == (0, 8)
    ops.release_pages(i, i, torch.zeros(0, 4, dtype=torch.int32, device=gpu), one, one, 16)


@pytest.mark.parametrize("width", [0, 8])
def test_captured(gpu, width):
    """A captured step and its release, replayed on changing lengths."""
    rng = np.random.default_rng(7)
    pool = _Pool(gpu, rng.integers(0, 90, 40).tolist(), 16, 16, 300, rng)
    new, keep = (torch.zeros(40, dtype=torch.int32, device=gpu) for _ in range(2))
    args = dict(width=width) if width else dict(rows=256)
    saved = [t.clone() for t in pool.gpu()[:4]]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ops.assign_pages(new, *pool.gpu(), **args)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = ops.assign_pages(new, *pool.gpu(), **args)
            ops.release_pages(keep, *pool.gpu())
    torch.cuda.synchronize()
    for a, b in zip(saved, pool.gpu()):
        b.copy_(a)
    for step in range(4):
        n, k = rng.integers(0, 9, 40), rng.integers(0, 100, 40)
        new.copy_(torch.from_numpy(n))
        keep.copy_(torch.from_numpy(k))
        graph.replay()
        want = ps.assign_pages_np(n.tolist(), pool.lens, pool.table, pool.free, 16, width, 0 if width else 256)
        ps.release_pages_np(k.tolist(), pool.lens, pool.table, pool.free, 16)
        torch.cuda.synchronize()
        assert np.array_equal(got.slots.flatten().cpu().numpy(), want["slots"])
        pool.check()


def test_on_another_stream(gpu):
    rng = np.random.default_rng(8)
    pool = _Pool(gpu, rng.integers(0, 90, 40).tolist(), 16, 16, 300, rng)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        pool.assign(rng.integers(0, 9, 40).tolist(), width=8)
        pool.release(rng.integers(0, 100, 40).tolist())


def test_refusals(gpu):
    rng = np.random.default_rng(9)
    pool = _Pool(gpu, [3, 4], 4, 16, 4, rng)
    new = torch.ones(2, dtype=torch.int32, device=gpu)
    lens, table, free, count, _ = pool.gpu()
    for args, kw in [((new, *pool.gpu()), dict()), ((new, *pool.gpu()), dict(width=1, rows=2)),
                     ((new, *pool.gpu()), dict(width=-1)), ((new, *pool.gpu()[:4], 24), dict(width=1)),
                     ((new, *pool.gpu()[:4], 0), dict(width=1)),
                     ((new[:1], *pool.gpu()), dict(width=1)), ((new.float(), *pool.gpu()), dict(width=1)),
                     ((new, lens.long(), table, free, count, 16), dict(width=1)),
                     ((new, lens, table.long(), free, count, 16), dict(width=1)),
                     ((new, lens, table[0], free, count, 16), dict(width=1)),
                     ((new, lens, table[:1].expand(2, -1), free, count, 16), dict(width=1)),
                     ((new, lens, table.T.contiguous().T, free, count, 16), dict(width=1)),
                     ((new, lens, table, free[::2], count, 16), dict(width=1)),
                     ((new, lens, table, free, free, 16), dict(width=1)),
                     ((new.cpu(), *pool.gpu()), dict(width=1))]:
        with pytest.raises(RuntimeError):
            ops.assign_pages(*args, **kw)
    with pytest.raises(RuntimeError):
        ops.release_pages(new[:1], *pool.gpu())
    pool.check()
