"""A serving step whose batch holds padding rows, and the variant whose tier takes
the keys too."""
import pytest
import torch

from tests import test_gpu_serving_step as S
from tests.test_window import _agree, _exact


@pytest.mark.gpu
def test_requests_come_and_go_mem_kv():
    S.test_requests_come_and_go("mem-kv")


def _stepped(m, rows, new):
    i = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    m.plain.begin()
    m.plain.step(rows, new)
    m.t.step(i(rows), i(new), n_req=len(rows), n_tokens=sum(n for w, n in zip(rows, new) if w >= 0))
    return i


@pytest.mark.gpu
def test_padding_behind_the_requests():
    """Single-token calls read row r of q for request r: padding (row -1) takes no
    token, and stands behind the requests."""
    m = S.Model()
    _stepped(m, [3, 0, 2], [70, 33, 129])
    kv, t = m.caches[0], m.t
    kv.copy_(torch.randn(kv.shape, generator=m.g, device="cuda"))
    rows, n = [2, 3, 0, -1, -1], 5
    i = _stepped(m, rows, [1, 1, 1, 1, 0])
    assert t.query_start_loc[:n + 1].tolist() == [0, 1, 2, 3, 3, 3]
    q = torch.randn(n, S.N_KV * S.G, S.D, generator=m.g, device="cuda").to(torch.bfloat16)
    scale = S.D ** -0.5
    c = m._case(rows[:3], [1] * 3, kv, q[:3], scale)
    for window in (0, 40):
        out, lse = torch.full_like(q, 7.0), torch.zeros(n, S.N_KV * S.G, device="cuda")
        m.eng.forward_dense(q, kv, t.block_table[:n], t.seq_lens[:n], n, scale, out, window=window, lse=lse)
        _agree(out[:3], lse[:3], _exact(c, window, 0))
        assert not bool(out[3:].any()) and bool((lse[3:] == -torch.inf).all())
    out, lse = torch.full_like(q, 7.0), torch.zeros(n, S.N_KV * S.G, device="cuda")
    m.eng.forward_prefix(q, kv, t.block_table[:n], t.seq_lens[:n], i([3, 5]), i([4]), n, 1, scale, out, lse=lse)
    _agree(out[:3], lse[:3], _exact(c, 0, 0))
    assert not bool(out[3:].any()) and bool((lse[3:] == -torch.inf).all())


@pytest.mark.gpu
def test_padding_between_the_requests():
    """With query_start_loc a request's rows are where it says, wherever padding or
    a request without a new token stands."""
    m = S.Model()
    _stepped(m, [3, 0, 2], [70, 33, 129])
    kv, t = m.caches[0], m.t
    kv.copy_(torch.randn(kv.shape, generator=m.g, device="cuda"))
    rows, new, n = [-1, 2, -1, 3, 0, -1], [0, 1, 1, 0, 2, 0], 6
    _stepped(m, rows, new)
    assert t.query_start_loc[:n + 1].tolist() == [0, 0, 1, 1, 1, 3, 3]
    q = torch.randn(4, S.N_KV * S.G, S.D, generator=m.g, device="cuda").to(torch.bfloat16)
    out, lse = torch.full_like(q, 7.0), torch.full((4, S.N_KV * S.G), 7.0, device="cuda")
    m.eng.forward_dense(q, kv, t.block_table[:n], t.seq_lens[:n], n, S.D ** -0.5, out,
                        query_start_loc=t.query_start_loc[:n + 1], window=40, sinks=3, lse=lse)
    _agree(out[:3], lse[:3], _exact(m._case([2, 0], [1, 2], kv, q[:3], S.D ** -0.5), 40, 3))
    assert bool((out[3] == 7).all()) and bool((lse[3] == 7).all())
