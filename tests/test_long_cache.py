"""Blocks whose offset in the cache passes 32 bits (a cache of 8.7 GB), and requests
that a step could not serve (rows without a key)."""
import pytest
import torch

from locks.attention import attn_workspace, prefix_decode, qk_norm_rope_write, window_decode, window_prefill
from tests.test_window import _agree, _exact


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["nb2", "2nb"])
def test_far_blocks(layout):
    page, n_kv, G, d, NB = 64, 16, 1, 256, 8300
    shape = (NB, 2, page, n_kv, d) if layout == "nb2" else (2, NB, page, n_kv, d)
    kv = torch.empty(shape, dtype=torch.bfloat16, device="cuda")
    K, V = (kv[:, 0], kv[:, 1]) if layout == "nb2" else (kv[0], kv[1])
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").to(torch.bfloat16)  # noqa: E731
    i = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    lens, new = [300, 200], [40, 30]
    bt = i([[8299, 8297, 1, 8200, 8298], [8299, 8297, 8000, 8250, 0]])
    # the rows written by the cache write itself, one request after the other
    q, k, v = r(500, n_kv * G, d), r(500, n_kv, d), r(500, n_kv, d)
    qo = torch.empty_like(q)
    slots = torch.cat([bt[j].long()[torch.arange(n, device="cuda") // page] * page + torch.arange(n, device="cuda") % page
                       for j, n in enumerate(lens)])
    keep = torch.cat([torch.ones(300), (torch.arange(200) >= 128)]).bool().cuda()       # the shared pages once
    slots = torch.where(keep, slots, -1)
    qk_norm_rope_write(q, k, v, i(list(range(500))), slots, kv, None, qo)
    assert torch.equal(qo, q)
    ks, vs = [k[:300], torch.cat([k[:128], k[428:]])], [v[:300], torch.cat([v[:128], v[428:]])]
    for j, n in enumerate(lens):
        t = torch.arange(n, device="cuda")
        assert torch.equal(K[bt[j].long()[t // page], t % page], ks[j])
        assert torch.equal(V[bt[j].long()[t // page], t % page], vs[j])
    c = dict(k=ks, v=vs, lens=lens, n_kv=n_kv, G=G, d=d, page=page, scale=d ** -0.5)
    ws = attn_workspace("cuda", max_tokens=70, n_kv=n_kv, G=G, head_dim=d)
    sl = i(lens)
    rows = torch.cat([torch.arange(260, 300), torch.arange(470, 500)]).cuda()
    qp = q[rows].contiguous()
    out, lse = torch.empty_like(qp), torch.empty(70, n_kv * G, device="cuda")
    for window in (0, 50):
        window_prefill(qp, kv, bt, sl, i([0, 40, 70]), out, ws, n_req=2, window=window, scale=c["scale"], lse=lse)
        _agree(out, lse, _exact({**c, "q": qp, "new": new}, window, 0))
    q1 = qp[[39, 69]].contiguous()
    out, lse = torch.empty_like(q1), torch.empty(2, n_kv * G, device="cuda")
    one = {**c, "q": q1, "new": [1, 1]}
    window_decode(q1, kv, bt, sl, out, ws, n_req=2, window=150, sinks=3, scale=c["scale"], lse=lse)
    _agree(out, lse, _exact(one, 150, 3))
    prefix_decode(q1, kv, bt, sl, i([0, 2]), i([2]), out, ws, n_req=2, n_groups=1, scale=c["scale"], lse=lse)
    _agree(out, lse, _exact(one, 0, 0))


@pytest.mark.gpu
@pytest.mark.parametrize("long", [50, 9000])
def test_rows_of_an_unserved_request(long):
    """Length 0 with rows in the batch (no block was left for it): zeros and -inf,
    whole and split calls alike; the request behind it as ever."""
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").to(torch.bfloat16)  # noqa: E731
    i = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    pages = -(-long // 16)
    kv = r(pages, 2, 16, 2, 128)
    bt = torch.arange(pages, device="cuda", dtype=torch.int32).expand(2, pages).contiguous()
    q = r(8, 8, 128)
    out, lse = torch.full_like(q, 7.0), torch.zeros(8, 8, device="cuda")
    ws = attn_workspace("cuda", max_tokens=8, n_kv=2, G=4, head_dim=128)
    window_prefill(q, kv, bt, i([0, long]), i([0, 3, 8]), out, ws, n_req=2, scale=0.09, lse=lse)
    assert not bool(out[:3].any()) and bool((lse[:3] == -torch.inf).all())
    k, v = kv[:, 0].flatten(0, 1)[:long], kv[:, 1].flatten(0, 1)[:long]
    want = _exact(dict(q=q[3:], k=[k], v=[v], lens=[long], new=[5], n_kv=2, G=4, d=128, page=16, scale=0.09), 0, 0)
    _agree(out[3:], lse[3:], want)
