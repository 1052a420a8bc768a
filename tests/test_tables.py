"""Block tables made on the GPU (BlockTables.step / .trim) against a request by
request restatement in Python, and the calls that are refused.  Every output is
a whole number, so all comparisons are equalities."""
import random

import pytest
import torch

from locks import _lib
from locks.backend.tables import BlockTables


class Plain:
    """The pool one request at a time."""

    def __init__(self, num_blocks, page, max_reqs, max_pages):
        self.page, self.max_pages, self.NB = page, max_pages, num_blocks
        self.table = [[] for _ in range(max_reqs)]
        self.lens = [0] * max_reqs
        self.free = list(range(num_blocks))
        self.head = 0

    def step(self, rows, new):
        total, start, pos, slots, bt, unserved = [], [0], [], [], [], 0
        seen, want = set(), 0
        for w, n in zip(rows, new):
            if w < 0:
                total.append(0), start.append(start[-1]), bt.append(None)
                continue
            n = max(n, 0)
            ok = w < len(self.lens) and w not in seen
            seen.add(w)
            c = self.lens[w] if ok else 0
            pages = -(-(c + n) // self.page)
            ok = ok and pages <= self.max_pages
            if ok:
                need = pages - len(self.table[w])
                want += need
                ok = need == 0 or want <= self.NB - self.head0
            if ok:
                for _ in range(need):
                    self.table[w].append(self.free[self.head])
                    self.head += 1
                self.lens[w] = c + n
            unserved += not ok
            total.append(c + n if ok else 0)
            bt.append(list(self.table[w]) if ok else None)
            start.append(start[-1] + n)
            for p in range(c, c + n):
                pos.append(p)
                slots.append(self.table[w][p // self.page] * self.page + p % self.page if ok else -1)
        return total, start, pos, slots, bt, unserved

    def begin(self):
        self.head0 = self.head

    def trim(self, rows, keep):
        seen, back = set(), []
        for w, k in zip(rows, keep):
            if w < 0 or w >= len(self.lens) or w in seen:
                continue
            seen.add(w)
            k = min(max(k, 0), self.lens[w])
            n = -(-k // self.page)
            back += self.table[w][n:]
            self.table[w] = self.table[w][:n]
            self.lens[w] = k
        self.head -= len(back)
        self.free[self.head:self.head + len(back)] = back


def _dev(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _check(t, plain, rows, new, n_tokens):
    """One step on both sides; the entries past each output stay as they were."""
    t.block_table.fill_(-7), t.seq_lens.fill_(-7), t.query_start_loc.fill_(-7)
    t.positions.fill_(-7), t.slot_mapping.fill_(-7)
    plain.begin()
    total, start, pos, slots, bt, unserved = plain.step(rows, new)
    t.step(_dev(rows), _dev(new), n_req=len(rows), n_tokens=n_tokens)
    n, T = len(rows), len(pos)
    pos, slots = (pos + [0] * n_tokens)[:n_tokens], (slots + [-1] * n_tokens)[:n_tokens]
    assert t.seq_lens.tolist() == total + [-7] * (t.max_reqs - n)
    assert t.query_start_loc.tolist() == start + [-7] * (t.max_reqs - n)
    assert t.positions.tolist() == pos + [-7] * (t.max_tokens - n_tokens)
    assert t.slot_mapping.tolist() == slots + [-7] * (t.max_tokens - n_tokens)
    want = torch.full((t.max_reqs, t.max_pages), -7, dtype=torch.int32)
    for r, ids in enumerate(bt):
        if ids:
            want[r, :len(ids)] = torch.tensor(ids, dtype=torch.int32)
    assert torch.equal(t.block_table.cpu(), want)
    _state(t, plain)
    assert t.state.tolist()[1:] == [unserved, 0, 0]
    return T


def _state(t, plain):
    assert t.state[0].item() == plain.head
    assert t.lens.tolist() == plain.lens
    assert t.free[plain.head:].tolist() == plain.free[plain.head:]
    for w, ids in enumerate(plain.table):
        assert t.table[w, :len(ids)].tolist() == ids


def _pair(num_blocks, page, max_reqs, max_pages, max_tokens):
    return (BlockTables("cuda", num_blocks=num_blocks, page=page, max_reqs=max_reqs, max_pages=max_pages,
                        max_tokens=max_tokens), Plain(num_blocks, page, max_reqs, max_pages))


@pytest.mark.gpu
@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("max_reqs, max_pages, most", [(1, 1, 16), (7, 13, 90), (300, 41, 200), (2048, 5, 33)])
def test_steps_and_trims(page, max_reqs, max_pages, most):
    """Requests arrive, grow, roll back and end, in batches of any order, with
    padding among them; pools that run out on the way."""
    rng = random.Random(page * 1000 + max_reqs)
    t, plain = _pair(max_reqs * max_pages // 2 + 2, page, max_reqs, max_pages, 20000)
    for _ in range(12):
        rows = rng.sample(range(max_reqs), rng.randint(1, max_reqs))
        new = [rng.choice([0, 1, 1, rng.randint(1, most)]) for _ in rows]
        while sum(new) > 19000:
            new = [n // 2 for n in new]
        if len(rows) > 3:
            rows[rng.randrange(len(rows))] = -1
        _check(t, plain, rows, new, min(20000, sum(new) + rng.choice([0, 5])))
        back = rng.sample(range(max_reqs), rng.randint(1, max_reqs))
        keep = [rng.choice([0, plain.lens[w], max(0, plain.lens[w] - rng.randint(0, 40)), 1 << 30]) for w in back]
        plain.trim(back, keep)
        t.trim(_dev(back), _dev(keep), n_req=len(back))
        _state(t, plain)


@pytest.mark.gpu
def test_long_rows():
    """A table of more ids than one workgroup copies at once, lengths at both
    sides of a page's end, one request of 1M tokens."""
    t, plain = _pair(70000, 16, 4, 65537, 70000)
    _check(t, plain, [2, 0], [40000, 16 * 1024], 60000)
    _check(t, plain, [0, 3, 2], [1, 16 * 1023, 0], 16385)
    for _ in range(15):
        _check(t, plain, [2, 0], [63999, 17], 64020)
    _check(t, plain, [0, 2], [15, 1], 16)


@pytest.mark.gpu
@pytest.mark.parametrize("rows, new, served", [
    ([3, 1, 3, 0], [20, 5, 7, 1], [1, 1, 0, 1]),             # a row twice: the first keeps it
    ([0, 9, 1], [1, 4, 2], [1, 0, 1]),                       # no such row
    ([0, 1], [16 * 6 + 1, 16 * 6], [0, 1]),                  # more pages than the table holds
    ([0, 1, 2], [16 * 5, 16 * 6, 16], [1, 0, 0]),            # the free blocks end within the second
    ([0, 1, 2], [16 * 6, 16 * 4, 0], [1, 1, 1]),             # all of them, to the last
    ([-1, -1, 2], [5, 3, 4], [0, 0, 1]),                     # padding first
    ([0, 1], [-3, 2], [1, 1]),                               # a negative length is none
])
def test_unserved(rows, new, served):
    t, plain = _pair(10, 16, 4, 6, 300)
    _check(t, plain, rows, new, 300)
    assert [int(x > 0 or (n <= 0 and w >= 0)) for x, n, w in zip(t.seq_lens.tolist(), new, rows)] == served
    _check(t, plain, [2, 3], [1, 1], 2)                      # and the pool goes on


@pytest.mark.gpu
def test_replayed():
    """A step and its roll-back captured once and replayed, with other lengths
    written between the replays and eager calls in between."""
    t, plain = _pair(500, 16, 8, 60, 600)
    rows, new, keep = _dev([5, 2, 7]), _dev([0, 0, 0]), _dev([0, 0, 0])
    t.step(rows, new, n_req=3, n_tokens=600)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        t.step(rows, new, n_req=3, n_tokens=600)
        t.trim(rows, keep, n_req=3)
    rng = random.Random(4)
    for i in range(6):
        n = [rng.randint(0, 190) for _ in range(3)]
        k = [rng.randint(0, 400) for _ in range(3)]
        new.copy_(_dev(n)), keep.copy_(_dev(k))
        plain.begin()
        total, start, pos, slots, *_ = plain.step([5, 2, 7], n)
        g.replay()
        assert t.seq_lens[:3].tolist() == total and t.query_start_loc[:4].tolist() == start
        assert t.positions[:len(pos)].tolist() == pos and t.slot_mapping[:len(pos)].tolist() == slots
        plain.trim([5, 2, 7], k)
        _state(t, plain)
        _check(t, plain, [1, 5], [3, 0], 9)
        plain.trim([1], [0])
        t.trim(_dev([1]), _dev([0]), n_req=1)


@pytest.mark.gpu
def test_empty_batch():
    t, plain = _pair(10, 16, 4, 6, 20)
    t.step(_dev([]), _dev([]), n_req=0, n_tokens=4)
    t.trim(_dev([]), _dev([]), n_req=0)
    assert t.positions[:4].tolist() == [0] * 4 and t.slot_mapping[:4].tolist() == [-1] * 4
    assert t.query_start_loc[0].item() == 0
    _state(t, plain)


def test_refusals():
    ok = dict(num_blocks=10, page=16, max_reqs=4, max_pages=6, max_tokens=20)
    for bad in (dict(page=8), dict(max_reqs=0), dict(max_reqs=2049), dict(num_blocks=0), dict(num_blocks=(1 << 22) + 1),
                dict(max_pages=0), dict(max_tokens=0), dict(reserved=11), dict(max_pages=1 << 27)):
        with pytest.raises(ValueError):
            BlockTables("cpu", **{**ok, **bad})
    t = BlockTables("cpu", **ok, reserved=3)
    assert t.state.tolist() == [3, 0, 0, 0] and t.free[3:].tolist() == list(range(3, 10))
    i = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    for args in ((i(0), i(1), 5, 1), (i(0), i(1), 1, 21), (i(0), i(1), -1, 1), (i(0), i(1), 2, 2), (i(0, 1), i(1), 2, 2),
                 (i(0), i(1), 1, 1)):                        # the last: tables on the CPU
        with pytest.raises(ValueError):
            t.step(*args)
    for rows in (torch.tensor([0]), i(0, 1, 2, 3)[::2], i(0)[None]):
        with pytest.raises(TypeError):
            t.step(rows, i(1, 1), n_req=1, n_tokens=1)
    with pytest.raises(ValueError):
        t.trim(i(0), i(0), n_req=5)
    with pytest.raises(ValueError):
        t.set_free(11)


def test_c_entry_refusals():
    """The C entries turn bad arguments into errors before they touch a GPU."""
    lib = _lib.load()
    step = dict(rows=16, new=16, n_req=1, n_tokens=1, lens=16, table=16, ts=8, max_reqs=4, max_pages=8, free=16, nb=10,
                state=16, bt=16, bs=8, sl=16, qsl=16, pos=16, slots=16, page=16, stream=0)
    for bad in (dict(page=8), dict(max_reqs=2049), dict(n_req=5), dict(n_req=-1), dict(n_tokens=-1), dict(max_pages=9),
                dict(ts=9), dict(bs=4), dict(table=8), dict(nb=0), dict(nb=1 << 23), dict(rows=0), dict(slots=0)):
        assert lib.locks_tables_step(*{**step, **bad}.values()) == -1, bad
        assert lib.locks_last_error()
    trim = dict(rows=16, keep=16, n_req=1, lens=16, table=16, ts=8, max_reqs=4, max_pages=8, free=16, nb=10, state=16,
                page=16, stream=0)
    for bad in (dict(page=0), dict(max_reqs=0), dict(n_req=5), dict(max_pages=9), dict(nb=0), dict(keep=0)):
        assert lib.locks_tables_trim(*{**trim, **bad}.values()) == -1, bad
