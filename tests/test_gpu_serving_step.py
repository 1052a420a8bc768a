"""The operators of a serving step together, as LocksEngine offers them: block
tables and slots from lengths, norm + rotation + cache write, page selection with
its sparse decode, dense and window attention, a shared prefix.

Two layers: one whose decode steps select pages (with a budget that covers all, so
that every token counts), one that keeps a window.  Every step is checked against
plain tables, the formulas of the cache rows and 64-bit attention over them (the
tolerances of the operators' own tests; the selected decode rounds its weights to
fp16, finer than the bf16 they allow)."""
import random

import pytest
import torch

from tests.test_qkv import _close, _formula
from tests.test_tables import Plain
from tests.test_window import _agree, _exact

N_KV, G, D, PAGE = 2, 4, 128, 16
WINDOW, SINKS, EPS = 48, 5, 1e-6


class Model:
    def __init__(self, variant="fast", max_tokens=400):
        from locks import LocksConfig
        from locks.backend.engine import LocksEngine
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(9)
        self.NB, self.R, self.MP = 70, 6, 30
        self.caches = [torch.full((self.NB, 2, PAGE, N_KV, D), 0.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
        self.eng = LocksEngine(LocksConfig(budget_pages=64, variant=variant), self.caches, num_heads_q=N_KV * G,
                               num_heads_kv=N_KV, head_dim=D, block_size=PAGE, max_num_seqs=self.R,
                               max_model_len=self.MP * PAGE, max_num_batched_tokens=max_tokens)
        self.t = self.eng.block_tables()
        self.plain = Plain(self.NB, PAGE, self.R, self.MP)
        r = lambda *s: torch.randn(*s, generator=self.g, device="cuda")  # noqa: E731
        ang = torch.arange(self.MP * PAGE, dtype=torch.float64, device="cuda")[:, None] * (
            10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64, device="cuda") / D))
        self.cs = torch.cat([ang.cos(), ang.sin()], 1).float()
        self.qw, self.kw = [(1 + 0.2 * r(D)).to(torch.bfloat16) for _ in range(2)]
        self.v_kept = [{}, {}]

    def step(self, rows, new, extra_pad=3):
        """One step of requests `rows`; returns nothing, checks everything."""
        i = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
        n, T = len(rows), sum(new)
        n_dec = next((k for k, m in enumerate(new) if m != 1), n)
        self.plain.begin()
        total, starts, pos, slots, bt, unserved = self.plain.step(rows, new)
        assert not unserved
        t, eng = self.t, self.eng
        t.step(i(rows), i(new), n_req=n, n_tokens=T + extra_pad)
        assert t.seq_lens[:n].tolist() == total and t.slot_mapping[:T].tolist() == slots
        sl, qsl, btab = t.seq_lens[:n], t.query_start_loc[:n + 1], t.block_table[:n]
        scale = D ** -0.5
        eng.prologue(btab, sl, qsl, n, torch.tensor(total), torch.tensor(starts))
        for layer in range(2):
            packed = torch.randn(T + extra_pad, (N_KV * (G + 2)) * D, generator=self.g, device="cuda").to(torch.bfloat16)
            q, k, v = (x.view(T + extra_pad, -1, D) for x in packed.split([N_KV * G * D, N_KV * D, N_KV * D], dim=1))
            qo = torch.empty(T + extra_pad, N_KV * G, D, dtype=torch.bfloat16, device="cuda")
            eng.write_qkv(layer, q, k, v, t.positions, t.slot_mapping, self.cs, qo, q_weight=self.qw, k_weight=self.kw,
                          eps=EPS)
            kv = self.caches[layer]
            p = torch.tensor(pos, device="cuda")
            want_q = _formula(q[:T], self.qw, p, self.cs, EPS, False)
            want_k = _formula(k[:T], self.kw, p, self.cs, EPS, False)
            _close(qo[:T], want_q, "q")
            at = torch.tensor(slots, device="cuda")
            _close(kv[at // PAGE, 0, at % PAGE], want_k, "k")
            assert torch.equal(kv[at // PAGE, 1, at % PAGE], v[:T])
            window, sinks = (WINDOW, SINKS) if layer else (0, 0)
            out = torch.full_like(qo, 7.0)
            lse = torch.zeros(T + extra_pad, N_KV * G, device="cuda")
            eng.forward_dense(qo, kv, btab, sl, n, scale, out, query_start_loc=qsl, n_decode=n_dec, window=window,
                              sinks=sinks, lse=lse)
            c = self._case(rows, new, kv, qo[:T], scale)
            want = _exact(c, window, sinks)
            _agree(out[:T], lse[:T], want)
            assert bool((out[T:] == 7).all())
            if layer == 0 and n_dec == n:                    # a pure decode step: the selected pages
                sel = torch.empty_like(out)
                eng.forward(qo, kv, btab, sl, n, scale, sel)
                _agree(sel[:n], lse[:n], want)

    def _case(self, rows, new, kv, q, scale):
        ks, vs, lens = [], [], []
        for w in rows:
            m = self.plain.lens[w]
            at = torch.tensor(self.plain.table[w], device="cuda")[:, None] * PAGE + torch.arange(PAGE, device="cuda")
            at = at.flatten()[:m]
            ks.append(kv[at // PAGE, 0, at % PAGE])
            vs.append(kv[at // PAGE, 1, at % PAGE])
            lens.append(m)
        return dict(q=q, k=ks, v=vs, lens=lens, new=new, n_kv=N_KV, G=G, d=D, page=PAGE, scale=scale)

    def trim(self, rows, keep):
        i = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
        self.plain.trim(rows, keep)
        self.t.trim(i(rows), i(keep), n_req=len(rows))


@pytest.mark.gpu
@pytest.mark.parametrize("variant", ["fast", "mem-v"])
def test_requests_come_and_go(variant):
    """Prompts, chunks beside decoding requests, rejected drafts, a request that
    ends and whose blocks and row serve the next one."""
    m = Model(variant)
    m.step([4, 1, 2], [70, 33, 129])
    for _ in range(3):
        m.step([1, 2, 4], [1, 1, 1])
    m.step([2, 4, 0], [1, 1, 150])                           # a prompt beside two decoding requests
    m.step([2, 4, 1, 0], [1, 1, 5, 40])                      # drafts and the next chunk
    m.trim([1], [m.plain.lens[1] - 3])                       # three of the drafts rejected
    m.step([0, 1, 2, 4], [1, 1, 1, 1])
    m.trim([2], [0])
    m.step([1, 2], [1, 64])                                  # row 2 again, on its old blocks
    rng = random.Random(1)
    for _ in range(18):                                      # over several page ends
        rows = rng.sample([0, 1, 2, 4], rng.randint(1, 4))
        m.step(rows, [1] * len(rows))


@pytest.mark.gpu
def test_shared_prefix_of_a_batch():
    """One prompt's pages in the rows of several requests, each of which goes on by
    itself; decode over the prefix once, and with a request beside the group."""
    m = Model()
    m.step([0, 5], [96, 20])                                 # six pages to share; another request
    t, p = m.t, m.plain
    for w in (1, 2, 3):
        p.table[w], p.lens[w] = list(p.table[0]), 96
        t.table[w, :6] = t.table[0, :6]
        t.lens[w] = 96
    m.step([0, 1, 2, 3], [1, 30, 2, 17])
    for k in range(3):
        rows, n = [1, 0, 3, 2, 5], 5
        m.step(rows, [1] * n)
        i = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
        q = torch.randn(n, N_KV * G, D, generator=m.g, device="cuda").to(torch.bfloat16)
        out, lse = torch.empty_like(q), torch.zeros(n, N_KV * G, device="cuda")
        for layer in range(2):
            m.eng.forward_prefix(q, m.caches[layer], t.block_table[:n], t.seq_lens[:n], i(0, 4), i(6), n, 1, D ** -0.5,
                                 out, lse=lse)
            _agree(out, lse, _exact(m._case(rows, [1] * n, m.caches[layer], q, D ** -0.5), 0, 0))
    m.trim([1, 2], [96, 96])                                 # members end: their own blocks return, the shared stay
    t.lens[1:3] = 0
    for w in (1, 2):
        p.table[w], p.lens[w] = [], 0
    assert t.state[0].item() == p.head and t.free[p.head:].tolist() == p.free[p.head:]


@pytest.mark.gpu
def test_captured_step():
    """Tables, cache write, window and prefix attention of a decode step in one
    graph, replayed over page ends with eager work between."""
    m = Model()
    m.step([0, 1, 2], [40, 60, 31])
    i = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    rows, new, n = i([2, 0, 1]), i([1, 1, 1]), 3
    packed = torch.zeros(n, (N_KV * (G + 2)) * D, dtype=torch.bfloat16, device="cuda")
    q, k, v = (x.view(n, -1, D) for x in packed.split([N_KV * G * D, N_KV * D, N_KV * D], dim=1))
    qo, o1, o2 = (torch.zeros(n, N_KV * G, D, dtype=torch.bfloat16, device="cuda") for _ in range(3))
    z1, z2 = (torch.zeros(n, N_KV * G, device="cuda") for _ in range(2))
    gs, gp, kv, t = i([0, 0]), i([0]), m.caches[0], m.t

    def step():
        t.step(rows, new, n_req=n, n_tokens=n)
        m.eng.write_qkv(0, q, k, v, t.positions, t.slot_mapping, m.cs, qo, q_weight=m.qw, k_weight=m.kw)
        m.eng.forward_dense(qo, kv, t.block_table, t.seq_lens, n, D ** -0.5, o1, window=WINDOW, sinks=SINKS, lse=z1)
        m.eng.forward_prefix(qo, kv, t.block_table, t.seq_lens, gs, gp, n, 1, D ** -0.5, o2, lse=z2)

    def plain():
        m.plain.begin()
        m.plain.step([2, 0, 1], [1, 1, 1])

    step(), plain()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for _ in range(20):
        packed.copy_(torch.randn(packed.shape, generator=m.g, device="cuda"))
        g.replay()
        plain()
        assert t.seq_lens[:n].tolist() == [m.plain.lens[w] for w in (2, 0, 1)]
        c = m._case([2, 0, 1], [1, 1, 1], kv, qo, D ** -0.5)
        _agree(o1, z1, _exact(c, WINDOW, SINKS))
        _agree(o2, z2, _exact(c, 0, 0))
