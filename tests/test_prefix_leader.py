"""Shared-prefix attention whose group starts with a request that does not hold
the prefix: padding, a request that a step could not serve (its block table row is
an earlier batch's), one shorter than the prefix.  The other members read the
prefix through a row that holds it.

Oracle and tolerances are those of tests/test_window.py."""
import pytest
import torch

from locks.attention import prefix_decode
from tests.test_window import _agree, _case, _empty_row, _exact, _no_rows, _outs, _ws


def _reordered(c, order):
    at = torch.tensor(order, device="cuda")
    pick = lambda x: [x[i] for i in order]  # noqa: E731
    return {**c, "q": c["q"][at].contiguous(), "bt": c["bt"][at].contiguous(), "sl": c["sl"][at].contiguous(),
            "k": pick(c["k"]), "v": pick(c["v"]), "lens": pick(c["lens"])}


def _check(c, starts, pages, want=None, **kw):
    i = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    out, lse = _outs(c)
    prefix_decode(c["q"], c["kv"], c["bt"], c["sl"], i(starts), i(pages), out, _ws(c), n_req=len(c["lens"]),
                  n_groups=len(pages), scale=c["scale"], lse=lse, **kw)
    _agree(out, lse, want or _empty_row(c, _exact(_no_rows(c), 0, 0)))


@pytest.mark.gpu
@pytest.mark.parametrize("first", [[], [40], [1, 300], [319, 0, 320]])
@pytest.mark.parametrize("d, page, n_kv, G", [(128, 16, 8, 4), (64, 32, 1, 16), (256, 64, 2, 3)])
def test_first_member_without_the_prefix(d, page, n_kv, G, first):
    """Length 0, with another request's pages in its row, and `first` ahead of the
    members that hold the 320 tokens; a request outside the group."""
    own = [320 + 77, 320 + 1, 320 + 500]
    n = len(own) + len(first) + 1
    c = _case(own + first + [0, 900], [1] * (n + 1), n_kv, G, d, page, seed=len(first), shared=[(0, n - 1, 320 // page)])
    c["bt"][n - 1] = c["bt"][n]                              # the padding row: pages of the request outside
    c = _reordered(c, [n - 1, *range(len(own), n - 1), *range(len(own)), n])
    _check(c, [0, n], [320 // page])
    _check(c, [0, n], [320 // page], max_prefix_pages=320 // page, max_seq_len=1000)


@pytest.mark.gpu
def test_no_member_holds_the_prefix():
    """A prefix longer than all members: the longest one's row; a group of padding;
    a prefix past the table."""
    c = _case([500, 130, 16, 0, 0, 0, 700], [1] * 7, 2, 4, 128, 16, shared=[(0, 3, 40)])
    c = _reordered(c, [3, 2, 1, 0, 4, 5, 6])
    c["bt"][0] = c["bt"][6]
    _check(c, [0, 4, 6, 7], [40, 3, 1 << 20])


@pytest.mark.gpu
def test_holder_behind_many():
    """Groups of more members than lanes, the prefix in the rows of the last one, or
    of one in the middle."""
    lens = [2000, 1999] + [(r * 37) % 900 for r in range(200)]
    c = _case(lens, [1] * len(lens), 2, 4, 128, 16, shared=[(0, 202, 120)])
    short = list(range(2, 202))
    for at in (0, 63, 64, 130, 200):
        order = short[:at] + [0] + short[at:at + 30] + [1] + short[at + 30:]
        _check(_reordered(c, order), [0, 202], [120])


@pytest.mark.gpu
def test_unserved_first_request_of_a_batch():
    """The pool is empty and the group's first request needs a block: BlockTables.step
    leaves its batch row as it was, and the others, which need none, are served."""
    from tests.test_gpu_serving_step import D, G, N_KV, Model
    m = Model()
    t, p = m.t, m.plain
    i = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731

    def step(rows, new):
        p.begin()
        p.step(rows, new)
        t.step(i(*rows), i(*new), n_req=len(rows), n_tokens=sum(new))

    step([0], [96])                                          # six pages to share
    for w in (1, 2, 3):
        p.table[w], p.lens[w] = list(p.table[0]), 96
        t.table[w, :6] = t.table[0, :6]
        t.lens[w] = 96
    step([0, 1, 2, 3], [16, 5, 7, 9])                        # the first one's pages are full
    for w in (4, 5):
        step([w], [380])
        step([w], [100])
    assert t.state[0].item() == m.NB                         # and the pool is empty
    rows = [0, 1, 2, 3]
    step(rows, [1] * 4)
    assert t.state[1].item() == 1 and t.seq_lens[:4].tolist() == [0, 102, 104, 106]
    for kv in m.caches:
        kv.copy_(torch.randn(kv.shape, generator=m.g, device="cuda"))
    q = torch.randn(4, N_KV * G, D, generator=m.g, device="cuda").to(torch.bfloat16)
    out, lse = torch.empty_like(q), torch.zeros(4, N_KV * G, device="cuda")
    m.eng.forward_prefix(q, m.caches[0], t.block_table[:4], t.seq_lens[:4], i(0, 4), i(6), 4, 1, D ** -0.5, out, lse=lse)
    assert not bool(out[0].any()) and bool((lse[0] == -torch.inf).all())
    _agree(out[1:], lse[1:], _exact(m._case(rows[1:], [1] * 3, m.caches[0], q[1:], D ** -0.5), 0, 0))
