"""Pages handed out and taken back on the GPU against a list of free numbers on the host: every value
is a whole number, so all comparisons are for equality."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module', autouse=True)
def cuda():
    if not torch.cuda.is_available():
        pytest.fail('CUDA device required for -m gpu tests')


def ints(values, **kw):
    return torch.tensor(values, dtype=torch.int32, device='cuda', **kw)


class Plain:
    """The pool as Python lists: `free` (last first) and the sequences' tables."""

    def __init__(self, free, page, table):
        self.free, self.page, self.table = list(free), page, [list(t) for t in table]

    def used(self, n):
        return -(-n // self.page)

    def grow(self, held, new, rows):
        starts, positions, slots = [0], [], []
        for b, (h, n) in enumerate(zip(held, new)):
            for j in range(self.used(h), self.used(h + n)):
                self.table[b][j] = self.free.pop()
            for t in range(h, h + n):
                positions.append(t)
                slots.append(self.table[b][t // self.page] * self.page + t % self.page)
            starts.append(len(positions))
        more = [-1] * (rows - len(positions))
        return [h + n for h, n in zip(held, new)], starts, positions + more, slots + more

    def release(self, held, keep):
        for b in reversed(range(len(held))):
            for j in reversed(range(self.used(keep[b]), self.used(held[b]))):
                self.free.append(self.table[b][j])


def check_same(pool, plain, table, got=None, want=None):
    if got is not None:
        for name, x in zip(got._fields, want):
            assert getattr(got, name).tolist() == x, name
    assert table.tolist() == plain.table
    count = pool.count.item()
    assert count == len(plain.free)
    assert pool.free[:count].tolist() == plain.free
    held = torch.ones(pool.pages, dtype=torch.int32)
    held[plain.free] = 0
    assert pool._marks.tolist() == held.tolist()


@pytest.mark.parametrize('seqs,page,most', [(1, 16, 5), (3, 1, 40), (33, 64, 700), (257, 32, 90), (5000, 16, 33),
                                            (2, 1024, 5000), (16384, 128, 3)])
def test_growing_and_shrinking(seqs, page, most):
    from rapidtinyrec_b200.page_pool import PagePool
    g = torch.Generator().manual_seed(seqs)
    width = 3 * most // page + 4
    pages = seqs * width + 7
    order = torch.randperm(pages, generator=g)
    pool = PagePool(pages, page, free=order.cuda())
    table = torch.full((seqs, width + 3), -5, dtype=torch.int32, device='cuda')
    plain = Plain(order.tolist(), page, table.tolist())
    held = [0] * seqs
    for step in range(3):
        new = torch.randint(0, most + 1, (seqs,), generator=g).tolist()
        rows = sum(new) + step * 5
        got = pool.grow(table, ints(held), ints(new), rows=rows)
        want = plain.grow(held, new, rows)
        check_same(pool, plain, table, got, want)
        held = want[0]
        keep = [int(h * x) for h, x in zip(held, torch.rand(seqs, generator=g).tolist())]
        if step == 1:
            keep[seqs // 2] = held[seqs // 2]
        pool.release(table, ints(held), ints(keep))
        plain.release(held, keep)
        check_same(pool, plain, table)
        held = keep
    got = pool.grow(table, ints(held), 1)  # a step's tokens
    want = plain.grow(held, [1] * seqs, seqs)
    check_same(pool, plain, table, got, want)
    pool.release(table, got.lens)
    plain.release(want[0], [0] * seqs)
    check_same(pool, plain, table)
    pool.check()


def test_growing_again_takes_the_same_pages():
    from rapidtinyrec_b200.page_pool import PagePool
    pool = PagePool(100, 16)
    table = torch.zeros(3, 9, dtype=torch.int32, device='cuda')
    first = pool.grow(table, ints([0, 0, 0]), ints([40, 0, 100]), rows=140)
    assert table[0, :3].tolist() == [0, 1, 2] and table[2, :7].tolist() == [3, 4, 5, 6, 7, 8, 9]
    assert first.starts.tolist() == [0, 40, 40, 140]
    more = pool.grow(table, first.lens, ints([20, 1, 0]), rows=21)
    kept, version = table.clone(), table._version
    pool.release(table, more.lens, first.lens)
    assert table._version == version
    again = pool.grow(table, first.lens, ints([20, 1, 0]), rows=21)
    assert torch.equal(table, kept) and torch.equal(again.slots, more.slots) and table._version > version
    pool.check()


def test_tables_in_a_wider_one_and_nothing_to_do():
    from rapidtinyrec_b200.page_pool import PagePool
    pool = PagePool(50, 16)
    whole = torch.full((5, 12), -1, dtype=torch.int32, device='cuda')
    table = whole[1:4, 2:8]
    got = pool.grow(table, ints([0, 0, 0]), ints([17, 96, 0]), rows=113)
    assert whole[1, 2:4].tolist() == [0, 1] and whole[2, 2:8].tolist() == [2, 3, 4, 5, 6, 7]
    assert (whole == -1).sum().item() == 60 - 8
    none = pool.grow(table, got.lens, 0)
    assert none.slots.numel() == 0 and torch.equal(none.lens, got.lens) and none.starts.tolist() == [0, 0, 0, 0]
    empty = pool.grow(table[:0], got.lens[:0], 1, rows=3)
    assert empty.slots.tolist() == [-1, -1, -1] and empty.starts.tolist() == [0] and empty.lens.numel() == 0
    pool.release(table, got.lens, got.lens)
    pool.release(table[:0], got.lens[:0])
    assert pool.count.item() == 42
    pool.check()


@pytest.mark.parametrize('held,new,rows,says', [
    ([0, 16, 5], [16, 80, 1], 97, 'fewer free pages'),         # six pages, five are free
    ([0, 16, 5], [16, 1, 124], 141, 'does not fit'),           # 129 tokens in a row of 8 pages
    ([0, 16, 5], [16, -1, 3], 40, 'does not fit'),
    ([0, -16, 5], [16, 1, 3], 40, 'does not fit'),
    ([0, 16, 5], [2, 3, 4], 8, 'does not fit'),                # nine tokens in eight rows
    ([0, 2**31 - 1, 5], [2, 2**31 - 1, 4], 100, 'does not fit')])
def test_a_call_that_does_not_fit_changes_nothing(held, new, rows, says):
    from rapidtinyrec_b200 import _native
    from rapidtinyrec_b200.page_pool import PagePool
    pool = PagePool(7, 16, free=ints([6, 1, 2, 5, 4]))
    table = ints([[-1] * 8, [0] + [-1] * 7, [3] + [-1] * 7])
    before = table.clone(), pool.free.clone(), pool.count.clone(), pool._marks.clone()
    got = pool.grow(table, ints(held), ints(new), rows=rows)
    assert got.lens.tolist() == held and got.starts.tolist() == [0] * 4
    assert (got.positions == -1).all() and (got.slots == -1).all()
    for x, y in zip(before, (table, pool.free, pool.count, pool._marks)):
        assert torch.equal(x, y)
    with pytest.raises(_native.NativeError, match=says):
        pool.check()
    pool.check()  # forgotten
    got = pool.grow(table, ints([0, 16, 5]), ints([16, 17, 11]), rows=44)  # the pool works on: three pages
    assert pool.count.item() == 2 and got.slots[0].item() == 4 * 16
    pool.check()


@pytest.mark.parametrize('table,held,keep,says', [
    ([[3, 3], [1, 0]], [32, 16], [0, 0], 'no sequence held'),      # one page twice in a call
    ([[3, 2], [3, 0]], [32, 16], [0, 0], 'no sequence held'),
    ([[3, 4], [1, 0]], [32, 16], [0, 0], 'no sequence held'),      # 4 is free
    ([[3, 9], [1, 0]], [32, 16], [0, 0], 'outside the pool'),
    ([[-1, 2], [1, 0]], [32, 16], [0, 0], 'outside the pool'),
    ([[3, 2], [1, 0]], [33, 16], [0, 0], 'does not fit'),
    ([[3, 2], [1, 0]], [32, 16], [0, 17], 'does not fit'),
    ([[3, 2], [1, 0]], [32, 16], [-1, 0], 'does not fit')])
def test_pages_that_are_not_held_are_not_taken_back(table, held, keep, says):
    from rapidtinyrec_b200 import _native
    from rapidtinyrec_b200.page_pool import PagePool
    pool = PagePool(6, 16, free=ints([4, 5]))
    before = pool.free.clone(), pool.count.clone(), pool._marks.clone()
    pool.release(ints(table), ints(held), ints(keep))
    for x, y in zip(before, (pool.free, pool.count, pool._marks)):
        assert torch.equal(x, y)
    with pytest.raises(_native.NativeError, match=says):
        pool.check()
    pool.release(ints([[3, 2], [1, 0]]), ints([32, 16]))
    assert pool.free[:5].tolist() == [4, 5, 1, 2, 3]
    pool.release(ints([[3, 2], [1, 0]]), ints([32, 16]))
    with pytest.raises(_native.NativeError, match='no sequence held'):
        pool.check()
    assert pool.count.item() == 5


def test_many_pages_given_back_twice():
    """The same through a cluster of blocks: a table of more entries than one block takes."""
    from rapidtinyrec_b200 import _native
    from rapidtinyrec_b200.page_pool import PagePool
    pool = PagePool(40000, 1)
    table = torch.zeros(40, 1000, dtype=torch.int32, device='cuda')
    got = pool.grow(table, ints([0] * 40), 900)
    state = pool.free.clone(), pool._marks.clone()
    broken = table.clone()
    broken[31, 7] = broken[2, 800]
    pool.release(broken, got.lens)
    assert torch.equal(pool.free, state[0]) and torch.equal(pool._marks, state[1]) and pool.count.item() == 4000
    with pytest.raises(_native.NativeError, match='no sequence held'):
        pool.check()
    pool.release(table, got.lens)
    assert pool.count.item() == 40000 and not pool._marks.any()
    assert pool.free.tolist() == list(range(39999, -1, -1))
    pool.check()


def test_a_row_whose_page_is_outside_the_pool():
    from rapidtinyrec_b200 import _native
    from rapidtinyrec_b200.page_pool import PagePool
    pool = PagePool(6, 16)
    table = ints([[9, 0, 0], [0, 0, 0]])
    got = pool.grow(table, ints([10, 0]), ints([8, 1]), rows=9)
    assert got.slots.tolist() == [-1] * 6 + [0, 1, 16] and got.positions.tolist() == [-1] * 6 + [16, 17, 0]
    with pytest.raises(_native.NativeError, match='outside the pool'):
        pool.check()


def test_captured_and_replayed():
    from rapidtinyrec_b200.page_pool import PagePool
    pool, plain = PagePool(400, 16), None
    table = torch.zeros(6, 20, dtype=torch.int32, device='cuda')
    held, new = ints([0] * 6), ints([0] * 6)
    pool.grow(table, held, new, rows=64)  # loads the kernel
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got = pool.grow(table, held, new, rows=64)
        held.copy_(got.lens)
    plain = Plain(range(399, -1, -1), 16, table.tolist())
    at = [0] * 6
    for step in range(4):
        counts = [(3 * step + 5 * b) % 11 for b in range(6)]
        new.copy_(ints(counts))
        graph.replay()
        want = plain.grow(at, counts, 64)
        check_same(pool, plain, table, got, want)
        at = want[0]
    pool.check()


def test_on_another_stream():
    from rapidtinyrec_b200.page_pool import PagePool
    pool = PagePool(64, 16)
    table = torch.zeros(4, 6, dtype=torch.int32, device='cuda')
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = pool.grow(table, ints([0, 0, 0, 0]), 40)
        pool.release(table, got.lens, ints([16, 0, 40, 17]))
    stream.synchronize()
    assert pool.count.item() == 64 - 12 + 2 + 3 + 0 + 1
    pool.check()


def test_pages_serve_the_cache():
    """Tables, lens and starts as KvCache8 takes them: rows written through them read back."""
    from rapidtinyrec_b200.kv_cache import KvCache8
    from rapidtinyrec_b200.page_pool import PagePool
    g = torch.Generator(device='cuda').manual_seed(3)
    cache, pool = KvCache8.allocate(40, 2, 16, 64), PagePool(40, 16)
    table = torch.zeros(3, 9, dtype=torch.int32, device='cuda')
    parts = []
    held = ints([0, 0, 0])
    for new in ([20, 1, 33], [1, 0, 1], [30, 7, 0]):
        got = pool.grow(table, held, ints(new), rows=sum(new))
        x = torch.randint(-3, 4, (sum(new), 2, 64), generator=g, device='cuda').float()  # small whole numbers: exact codes
        cache.write(x, -x, table, got.lens, starts=got.starts)
        # the slots name the same places
        codes = cache.k.transpose(1, 2).reshape(-1, 2, 64)[got.slots].float()
        assert torch.equal(codes * cache.k_scale[got.slots // 16][:, :, None], x)
        parts.append(x.split(new))
        held = got.lens
    k, v = cache.read(93, table, held, starts=ints([0, 51, 59, 93]))
    want = torch.cat([p[b] for b in range(3) for p in parts])
    assert torch.equal(k, want) and torch.equal(v, -want)
    cache.check()
    pool.check()
