"""GPU tests of the pages dealt out to sequences and taken back (paged_append, paged_truncate), against lists of Python's."""
import pytest

from test_gpu_mixers import _gen, _torch

pytestmark = pytest.mark.gpu


def _ints(v, dev):
    torch = _torch()
    return torch.tensor(v, dtype=torch.int32, device=dev)


class _Pool:
    """Block tables, lengths and a free list on the host, and what the calls do to them."""

    def __init__(self, seed, B, width, page, pages):
        torch = _torch()
        self.B, self.width, self.page = B, width, page
        self.free = torch.randperm(pages, generator=_gen(seed)).tolist()
        self.count = pages
        self.table = [[-9] * width for _ in range(B)]
        self.lens = [0] * B

    def pages(self, n):
        return -(-n // self.page)

    def append(self, n, T, first=0, complete=False):
        """slots and positions of T rows, the sequences' from row `first` on.  complete: the table has its pages already."""
        slots, positions, taken = [-1] * first, [0] * first, 0
        for b, m in enumerate(n):
            want = min(self.lens[b] + m, self.width * self.page)
            old, need = self.pages(self.lens[b]), 0 if complete else self.pages(want) - self.pages(self.lens[b])
            got = max(0, min(need, self.count - taken))
            for i in range(got):
                self.table[b][old + i] = self.free[self.count - 1 - taken - i]
            taken += need
            end = want if got == need else (old + got) * self.page
            for pos in range(self.lens[b], self.lens[b] + m):
                positions.append(pos)
                slots.append(self.table[b][pos // self.page] * self.page + pos % self.page if pos < end else -1)
            self.lens[b] = end
        self.count -= taken
        return slots + [-1] * (T - len(slots)), positions + [0] * (T - len(positions))

    def truncate(self, keep):
        for b in range(self.B):
            k = max(0, min(keep[b], self.lens[b]))
            for p in self.table[b][self.pages(k):self.pages(self.lens[b])]:
                if self.count < len(self.free):
                    self.free[self.count] = p
                self.count += 1
            self.lens[b] = k

    def on(self, dev):
        return _ints(self.table, dev), _ints(self.lens, dev), _ints(self.free, dev), _ints([self.count], dev)


def _cu(n, dev, first=0):
    at = [first]
    for m in n:
        at.append(at[-1] + m)
    return _ints(at, dev)


def _same(pool, table, lens, free, count, what=""):
    assert table.tolist() == pool.table, what
    assert lens.tolist() == pool.lens and count.item() == pool.count, what
    assert free.tolist()[:max(0, pool.count)] == pool.free[:max(0, pool.count)], what


@pytest.mark.parametrize("B,width,page,most,seed", [(1, 8, 16, 40, 1), (3, 10, 16, 70, 2), (64, 6, 16, 3, 3), (40, 60, 16, 300, 4), (300, 9, 32, 100, 5),
                                                    (1500, 5, 16, 12, 6), (5, 400, 16, 3000, 7), (7, 20, 5, 30, 8), (2, 3, 1, 2, 9), (1100, 3, 128, 40, 10)])
def test_a_run_of_calls(mcv, cuda, B, width, page, most, seed):
    """Sequences grow, shrink and end for a while, in place, on tables that stay on the device."""
    torch = _torch()
    gen = _gen(seed)
    pool = _Pool(seed, B, width, page, B * width)
    table, lens, free, count = pool.on(cuda)
    for turn in range(4):
        n = (torch.rand(B, generator=gen) ** 2 * (most + 1)).int().tolist()
        T = sum(n) + turn
        slots, positions, same = mcv.paged_append(table, lens, _cu(n, cuda), page, tokens=T, free_pages=free, free_count=count)
        assert same is lens
        want = pool.append(n, T)
        assert slots.tolist() == want[0] and positions.tolist() == want[1]
        _same(pool, table, lens, free, count, turn)
        live = [s for s in want[0] if s >= 0]
        assert len(set(live)) == len(live)
        keep = [(m if r < 0.5 else m - 3 if r < 0.8 else 0) for m, r in zip(pool.lens, torch.rand(B, generator=gen).tolist())]
        assert mcv.paged_truncate(table, lens, _ints(keep, cuda), page, free, count) is lens
        pool.truncate(keep)
        _same(pool, table, lens, free, count, turn)
    mcv.paged_truncate(table, lens, None, page, free, count)
    pool.truncate([0] * B)
    _same(pool, table, lens, free, count)
    assert count.item() == B * width and sorted(free.tolist()) == list(range(B * width))


@pytest.mark.parametrize("B,n,page", [(3, 40, 16), (30, 300, 16)])
def test_state_apart(mcv, cuda, B, n, page):
    """seq_lens_out and free_count_out given: what was read stays, and the call may be made again."""
    torch = _torch()
    pool = _Pool(1, B, 30, page, 40 * B)
    table, lens, free, count = pool.on(cuda)
    lens_out, count_out = torch.empty_like(lens), torch.empty_like(count)
    slots, positions = (torch.empty(B * n, dtype=torch.int64, device=cuda) for _ in range(2))
    want = pool.append([n] * B, B * n)
    for _ in range(2):
        got = mcv.paged_append(table, lens, None, page, free_pages=free, free_count=count, seq_lens_out=lens_out,
                               free_count_out=count_out, slots=slots, positions=positions)
        assert got[0] is slots and got[1] is positions and got[2] is lens_out
        assert slots.tolist() == want[0] and positions.tolist() == want[1] and (lens == 0).all() and count.item() == 40 * B
        _same(pool, table, lens_out, free, count_out)
    keep = [5 * b % (n + 9) for b in range(B)]
    pool.truncate(keep)
    again = torch.empty_like(lens)
    for _ in range(2):
        left = torch.empty_like(count)
        assert mcv.paged_truncate(table, lens_out, _ints(keep, cuda), page, free, count_out, seq_lens_out=again, free_count_out=left) is again
        _same(pool, table, again, free, left)
    keep = _ints(keep, cuda)                                     # in the place of what is kept
    mcv.paged_truncate(table, lens_out, keep, page, free, count_out, seq_lens_out=keep)
    _same(pool, table, keep, free, count_out)


@pytest.mark.parametrize("B,n,pages", [(1, 100, 3), (4, 50, 0), (5, 33, 9), (40, 300, 500)])
def test_pages_that_run_out(mcv, cuda, B, n, pages):
    """The first sequences get what there is; lengths end where the room does, and a count below zero says what was lacking."""
    torch = _torch()
    pool = _Pool(2, B, 30, 16, max(pages, 1))
    pool.count = pages
    table, lens, free, count = pool.on(cuda)
    slots, positions, _ = mcv.paged_append(table, lens, None, 16, tokens=B * n, free_pages=free, free_count=count)
    want = pool.append([n] * B, B * n)
    assert slots.tolist() == want[0] and positions.tolist() == want[1] and pool.count < 0
    _same(pool, table, lens, free, count)
    before = table.tolist()
    pool.count = 0                                               # a count below zero is none
    slots, _, _ = mcv.paged_append(table, lens, None, 16, tokens=B * n, free_pages=free, free_count=count)
    want = pool.append([n] * B, B * n)
    assert slots.tolist() == want[0] and table.tolist() == before
    _same(pool, table, lens, free, count)


def test_rows_that_are_full(mcv, cuda):
    pool = _Pool(3, 3, 2, 16, 20)
    table, lens, free, count = pool.on(cuda)
    for n in ([40, 3, 32], [1, 40, 0], [5, 5, 5]):
        slots, positions, _ = mcv.paged_append(table, lens, _cu(n, cuda), 16, tokens=sum(n), free_pages=free, free_count=count)
        want = pool.append(n, sum(n))
        assert slots.tolist() == want[0] and positions.tolist() == want[1]
        _same(pool, table, lens, free, count)
    assert lens.tolist() == [32, 32, 32] and count.item() == 14


def test_complete_tables(mcv, cuda):
    """Without a free list: slots, positions and lengths of tables that have their pages, one row for all sequences too."""
    torch = _torch()
    pool = _Pool(4, 5, 12, 16, 60)
    pool.append([190] * 5, 950)
    pool.lens = [0, 10, 16, 100, 185]
    table, lens, _, _ = pool.on(cuda)
    n = [20, 0, 1, 60, 7]
    before = table.clone()
    slots, positions, _ = mcv.paged_append(table, lens, _cu(n, cuda, 2), 16, tokens=95)
    want = pool.append(n, 95, 2, complete=True)
    assert slots.tolist() == want[0] and positions.tolist() == want[1] and lens.tolist() == pool.lens and (table == before).all()
    shared = table[3:4].expand(4, -1)
    slots, _, out = mcv.paged_append(shared, _ints([0, 5, 64, 191], cuda), None, 16, tokens=8)
    assert slots.tolist() == [pool.table[3][p // 16] * 16 + p % 16 if p < 192 else -1 for p in (0, 1, 5, 6, 64, 65, 191, 192)]
    assert out.tolist() == [2, 7, 66, 192]
    table[3, 1] = -1                                             # a page that is not there
    slots, _, _ = mcv.paged_append(table[3:4], _ints([14], cuda), None, 16, tokens=5)
    assert slots.tolist() == [pool.table[3][0] * 16 + 14, pool.table[3][0] * 16 + 15, -1, -1, -1]


@pytest.mark.parametrize("T", [8, 5000])
def test_offsets_and_lengths_out_of_range(mcv, cuda, T):
    """Lengths, counts and offsets that make no sense stay inside what there is."""
    pool = _Pool(5, 3, 4, 16, 30)
    pool.append([64] * 3, 192)
    table, _, free, _ = pool.on(cuda)
    slots, positions, out = mcv.paged_append(table, _ints([-7, 10 ** 9, 60], cuda), _ints([-3, 4, T, 2 * T], cuda), 16, tokens=T, free_pages=free,
                                             free_count=_ints([10 ** 9], cuda))
    assert out.tolist()[1:] == [64, 60] and out[0].item() == 4 and (slots[4:] == -1).all()
    slots, positions, out = mcv.paged_append(table, _ints([5, 5, 5], cuda), _ints([7, 5, 3, 0], cuda), 16, tokens=T)
    assert (slots == -1).all() and out.tolist() == [5, 5, 5] and (positions == 0).all()
    for count, left in ((-5, 8), (30, 38), (10 ** 9, 38)):       # from no page, or past the end of the list
        at = _ints([count], cuda)
        mcv.paged_truncate(table, _ints([64, 10 ** 9, -1], cuda), _ints([-4, -4, 9], cuda), 16, free, at)
        assert at.item() == left
    mcv.paged_truncate(table, _ints([64, 64, 64], cuda), _ints([10 ** 9, 63, 48], cuda), 16, free, at := _ints([0], cuda))
    assert at.item() == 1 and free[0].item() == table[2, 3].item()


def test_nothing_to_do(mcv, cuda):
    torch = _torch()
    slots, positions, lens = mcv.paged_append(_ints([], cuda).view(0, 4), _ints([], cuda))
    assert slots.shape == positions.shape == lens.shape == (0,)
    pool = _Pool(6, 2, 4, 16, 8)
    table, lens, free, count = pool.on(cuda)
    slots, _, _ = mcv.paged_append(table, lens, _ints([0, 0, 0], cuda), 16, tokens=0, free_pages=free, free_count=count)
    assert slots.numel() == 0 and count.item() == 8 and lens.tolist() == [0, 0]
    slots, _, _ = mcv.paged_append(table, lens, _ints([0, 0, 0], cuda), 16, tokens=3, free_pages=free, free_count=count)
    assert slots.tolist() == [-1] * 3


@pytest.mark.parametrize("B,n", [(3, 40), (30, 300)])
def test_in_a_graph_and_on_another_stream(mcv, cuda, B, n):
    """Captured in place: every replay is one more step of the same sequences."""
    torch = _torch()
    pool = _Pool(7, B, 200, 16, 200 * B)
    table, lens, free, count = pool.on(cuda)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        slots, positions, _ = mcv.paged_append(table, lens, None, 16, tokens=B * n, free_pages=free, free_count=count)
    for turn in range(4):
        graph.replay()
        torch.cuda.synchronize()
        want = pool.append([n] * B, B * n)
        assert slots.tolist() == want[0] and positions.tolist() == want[1], turn
        _same(pool, table, lens, free, count, turn)
    side.wait_stream(torch.cuda.current_stream())
    slots, positions, _ = mcv.paged_append(table, lens, None, 16, tokens=B, free_pages=free, free_count=count, stream=side)
    mcv.paged_truncate(table, lens, None, 16, free, count, stream=side)
    side.synchronize()
    want = pool.append([1] * B, B)
    assert slots.tolist() == want[0] and positions.tolist() == want[1]
    pool.truncate([0] * B)
    _same(pool, table, lens, free, count)
