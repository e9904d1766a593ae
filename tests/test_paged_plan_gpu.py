"""The plan of a step on the device against the same bookkeeping on the host."""

import random

import pytest
import torch

from persona import ops

pytestmark = pytest.mark.gpu


class Host:
    """What ``paged_plan`` has to do, in lists."""

    def __init__(self, B, page, max_pages, pool):
        self.page, self.max_pages = page, max_pages
        self.lengths, self.pages, self.free = [0] * B, [[] for _ in range(B)], list(range(pool))

    def step(self, new, keep, rows, seq_slots):
        ps = self.page
        keep = list(self.lengths) if keep is None else keep
        up = lambda n: -(-n // ps)  # noqa: E731
        ok = all(0 <= k <= L and n >= 0 for k, L, n in zip(keep, self.lengths, new)) and sum(new) <= rows and \
            all(up(k + n) <= self.max_pages for k, n in zip(keep, new))
        if ok:
            back = sum(up(L) - up(k) for L, k in zip(self.lengths, keep))
            ok = sum(up(k + n) - up(k) for k, n in zip(keep, new)) <= len(self.free) + back
        if not ok:
            return False, [0] * (len(new) + 1), [-1] * rows, [-1] * rows
        for b in reversed(range(len(new))):
            while len(self.pages[b]) > up(keep[b]):
                self.free.append(self.pages[b].pop())
        indptr, places, slots = [0], [], []
        for b, n in enumerate(new):
            while len(self.pages[b]) < up(keep[b] + n):
                self.pages[b].append(self.free.pop())
            self.lengths[b] = keep[b] + n
            indptr.append(indptr[-1] + n)
            places += [self.pages[b][p // ps] * ps + p % ps for p in range(keep[b], keep[b] + n)]
            slots += [seq_slots[b]] * n
        fill = [-1] * (rows - len(places))
        return True, indptr, places + fill, slots + fill


class Device:
    def __init__(self, B, page, max_pages, pool, rows):
        i32 = dict(dtype=torch.int32, device="cuda")
        self.page = page
        self.lengths = torch.zeros(B, **i32)
        self.table = torch.full((B, max_pages), 1 << 29, **i32)
        self.free = torch.arange(pool, **i32)
        self.num_free = torch.tensor([pool], **i32)
        self.indptr = torch.full((B + 1,), 77, **i32)
        self.places = torch.full((rows,), 77, dtype=torch.int64, device="cuda")
        self.slots, self.row_slots = torch.zeros(B, **i32), torch.full((rows,), 77, **i32)

    def step(self, new, keep=None, slots=True):
        new = torch.tensor(new, dtype=torch.int32, device="cuda")
        keep = None if keep is None else torch.tensor(keep, dtype=torch.int32, device="cuda")
        more = dict(seq_slots=self.slots, row_slots=self.row_slots) if slots else {}
        ops.paged_plan(new, self.lengths, self.table, self.free, self.num_free, self.page, self.indptr, self.places, keep=keep,
                       **more)


def _same(h, d, indptr, places, slots):
    assert d.lengths.tolist() == h.lengths
    assert d.indptr.tolist() == indptr
    assert d.places.tolist() == places
    assert d.row_slots.tolist() == slots
    n = int(d.num_free)
    assert d.free[:n].tolist() == h.free
    table = d.table.tolist()
    for b, p in enumerate(h.pages):
        assert table[b][:len(p)] == p


@pytest.mark.parametrize("B,page,top,rows", [(1, 16, 40, 64), (8, 16, 5, 50), (33, 1, 7, 300), (300, 24, 9, 3000),
                                             (1500, 32, 3, 5000), (8192, 64, 2, 20000), (3, 8, 2500, 8000), (2, 128, 5000, 10500)])
def test_steps_follow_the_host(B, page, top, rows):
    rng = random.Random(B)
    max_pages = -(-4 * top // page) + 2
    pool = B * max(2, max_pages // 2)
    h, d = Host(B, page, max_pages, pool), Device(B, page, max_pages, pool, rows)
    d.slots.copy_(torch.tensor([rng.randrange(-1, 8) for _ in range(B)], dtype=torch.int32))
    seq_slots = d.slots.tolist()
    made = 0
    for step in range(12):
        new = [rng.randint(0, top) if rng.random() < 0.8 else 0 for _ in range(B)]
        keep = None if step % 3 == 0 else [rng.choice([L, L, max(0, L - rng.randint(0, 5)), 0]) for L in h.lengths]
        ok, *want = h.step(new, keep, rows, seq_slots)
        d.step(new, keep)
        if ok:
            made += 1
            ops.check_errors(torch.device("cuda"))
        else:
            with pytest.raises(RuntimeError, match="no room for a planned step|segment"):
                ops.check_errors(torch.device("cuda"))
        _same(h, d, *want)
    assert made >= 4


def test_a_step_made_again_gets_its_pages_again():
    d = Device(5, 16, 10, 40, 100)
    d.step([20, 1, 33, 0, 16])
    table, free, num = d.table.clone(), d.free.clone(), d.num_free.clone()
    keep = [20, 1, 33, 0, 16]
    d.step([17, 16, 3, 40, 1])
    places = d.places.clone()
    d.step([17, 16, 3, 40, 1], keep=keep)
    assert torch.equal(places, d.places)
    d.step([0] * 5, keep=keep)
    assert torch.equal(num, d.num_free) and torch.equal(free, d.free)
    for b, n in enumerate([2, 1, 3, 0, 1]):
        assert torch.equal(table[b, :n], d.table[b, :n])
    assert d.places.tolist() == [-1] * 100


@pytest.mark.parametrize("break_it,match", [
    (lambda d: d.num_free.fill_(-1), "outside the paged cache"), (lambda d: d.num_free.fill_(41), "outside the paged cache"),
    (lambda d: d.lengths.fill_(-3), "segment"), (lambda d: d.lengths.fill_(1 << 30), "outside the paged cache")])
def test_state_that_does_not_fit(break_it, match):
    d = Device(3, 16, 5, 40, 20)
    break_it(d)
    before = [t.clone() for t in (d.lengths, d.table, d.free, d.num_free)]
    d.step([1, 2, 3])
    with pytest.raises(RuntimeError, match=match):
        ops.check_errors(torch.device("cuda"))
    assert all(torch.equal(a, b) for a, b in zip(before, (d.lengths, d.table, d.free, d.num_free)))
    assert d.indptr.tolist() == [0] * 4 and torch.all(d.places == -1) and torch.all(d.row_slots == -1)


@pytest.mark.parametrize("new,keep", [([-1, 0, 0], None), ([0, 0, 0], [0, 1, 0]), ([0, 0, 0], [-1, 0, 0]),
                                      ([2147483647, 2147483647, 2], None), ([1, 0, 0], [2147483647, 0, 0])])
def test_steps_that_are_no_steps(new, keep):
    d = Device(3, 16, 5, 40, 20)
    d.step(new, keep)
    with pytest.raises(RuntimeError, match="segment|no room"):
        ops.check_errors(torch.device("cuda"))
    assert d.indptr.tolist() == [0] * 4 and int(d.num_free) == 40 and d.lengths.tolist() == [0] * 3


def test_without_slots_rows_or_sequences():
    d = Device(2, 16, 3, 6, 9)
    d.step([4, 5], slots=False)
    assert d.places[:4].tolist() == [5 * 16 + i for i in range(4)] and torch.all(d.row_slots == 77)
    e = Device(2, 16, 3, 6, 0)
    e.step([0, 0])
    assert e.indptr.tolist() == [0, 0, 0]
    z = Device(0, 16, 3, 6, 4)
    z.step([])
    assert z.indptr.tolist() == [0] and z.places.tolist() == [-1] * 4
    ops.check_errors(torch.device("cuda"))


def test_captured_steps_follow_their_buffers():
    """Two graphs over two states, replayed in turn: a step of one token each, pages as the lengths need them."""
    states, graphs, news = [], [], []
    for i in range(2):
        d = Device(4, 4, 8, 32, 4)
        new = torch.ones(4, dtype=torch.int32, device="cuda")
        args = (new, d.lengths, d.table, d.free, d.num_free, 4, d.indptr, d.places)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ops.paged_plan(*args)
        states.append(d)
        graphs.append(g)
        news.append(new)
    news[1][2] = 0
    for _ in range(9):
        for g in graphs:
            g.replay()
    ops.check_errors(torch.device("cuda"))
    assert states[0].lengths.tolist() == [9] * 4 and states[1].lengths.tolist() == [9, 9, 0, 9]
    assert int(states[0].num_free) == 32 - 12 and int(states[1].num_free) == 32 - 9
    held = states[0].table[:, :3].flatten().tolist()
    assert len(set(held)) == 12


def test_refusals():
    d = Device(3, 16, 5, 40, 20)
    new = torch.zeros(3, dtype=torch.int32, device="cuda")
    base = [new, d.lengths, d.table, d.free, d.num_free, 16, d.indptr, d.places]

    def call(i, x, match, **kw):
        a = list(base)
        if i is not None:
            a[i] = x
        with pytest.raises(RuntimeError, match=match):
            ops.paged_plan(*a, **kw)

    call(0, new.long(), "int32")
    call(0, new[:2], "int32")
    call(1, torch.zeros(6, dtype=torch.int32, device="cuda")[::2], "contiguous")
    call(2, d.table[:2], "page_table")
    call(2, d.table[:1].expand(3, 5), "page_table")
    call(4, torch.zeros(2, dtype=torch.int32, device="cuda"), "one element")
    call(5, 0, "page_size")
    call(6, d.indptr[:3], "indptr")
    call(7, d.places.int(), "int64")
    call(None, None, "go together", seq_slots=d.slots)
    call(None, None, "go together", row_slots=d.row_slots)
    call(None, None, "overlaps", keep=d.lengths)
    call(0, d.lengths, "overlaps")
    call(3, d.table.flatten()[:10], "overlaps")
    call(None, None, "overlaps", seq_slots=d.slots, row_slots=d.free[:20])
    assert d.places.tolist() == [77] * 20
