"""The paged cache in 4 bits at the edges of its documentation: memory that nobody wrote,
and weights and angles of any size.  Tolerances: those of tests/test_kv4.py."""
import pytest
import torch

from locks.attention import RopeAxes, qk_norm_rope_write
from tests.test_kv4 import _blank, _decode, _prefill, _read, case, quantised
from tests.test_rope_axes import formula, inputs
from tests.test_window import _agree, _exact


def _unwritten(c, fill):
    """The case with `fill` in every byte where no token lies (not what a cache's rows hold)."""
    page, cache = c["page"], c["kv"]
    whole = cache.clone()
    cache.fill_(fill)
    for r, n in enumerate(c["lens"]):
        t = torch.arange(n, device="cuda")
        slots = c["bt"][r].long()[t // page] * page + t % page
        k, v = _read(whole, slots)
        qk_norm_rope_write(k, k, v, t.int(), slots, cache, None, torch.empty_like(k))
    return c


@pytest.mark.gpu
@pytest.mark.parametrize("fill", [0, 127, 252, 253, 254, 255])
@pytest.mark.parametrize("d, page, n_kv, G", [(64, 32, 1, 8), (128, 16, 2, 4), (256, 64, 1, 4)])
def test_bytes_that_nobody_wrote(d, page, n_kv, G, fill):
    """Scales that no write makes (253 and 254: entries past bf16's range) lie in masked
    places only, and reach no row there."""
    c = _unwritten(case([130, 300, 65], [40, 7, 65], n_kv, G, d, page), fill)
    for window, sinks in ((0, 0), (50, 3)):
        _agree(*_prefill(c, window, sinks), _exact(c, window, sinks))
    c = _unwritten(case([130, 300, 65], [1, 1, 1], n_kv, G, d, page), fill)
    for window, sinks in ((0, 0), (50, 3)):
        _agree(*_decode(c, window, sinks), _exact(c, window, sinks))


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T", [150, 6000])
@pytest.mark.parametrize("weight, table", [(2.0 ** 59, 1.0), (2.0 ** 30, 1.0), (1.0, 2.0 ** 59), (2.0 ** 15, 2.0 ** 5)])
def test_large_weights_over_small_entries(weight, table, T, interleaved):
    """Blocks whose normed entries lie below fp32's normal numbers, where weights or angles
    bring them back: the codes are those of 64 bits."""
    d, n_kv = 128, 1
    x = inputs(T, 2, n_kv, d, d, 1, w=torch.float32)
    x["kw"], x["cs"] = torch.full_like(x["kw"], weight), x["cs"] * table
    # one block in two of a pair's halves (or of adjacent pairs) tiny, the norm that of the others
    tiny = torch.arange(d, device="cuda") // 32 % 2 == 0
    x["k"] = torch.where(tiny, x["k"].float() * 2.0 ** -110, x["k"].float() * 2.0 ** 35).to(torch.bfloat16)
    cache = _blank(x["blocks"], n_kv, d, 16)
    qk_norm_rope_write(x["q"], x["k"], x["v"], x["pos"][0], x["slots"], cache, x["cs"], torch.zeros_like(x["q"]),
                       k_weight=x["kw"], interleaved=interleaved)
    k64 = formula(x["k"], x["kw"], x["pos"], x["cs"], RopeAxes([0] * (d // 2)), float(torch.tensor(1e-6)), interleaved)[0]
    _, _, want, near = quantised(k64)
    k, _ = _read(cache, x["slots"])
    assert torch.equal(torch.where(near, 0, k.double()), torch.where(near, 0, want)) and int(near.sum()) < 3


def _put(c, request, key, k=None, v=None):
    """Writes K and V of one key of a request again (heads of (n_kv, d)), others as they were."""
    page = c["page"]
    slot = c["bt"][request, key // page].long() * page + key % page
    k = c["k"][request][key:key + 1] if k is None else k[None]
    v = c["v"][request][key:key + 1] if v is None else v[None]
    qk_norm_rope_write(k, k, v, slot[None].int() * 0, slot[None], c["kv"], None, torch.empty_like(k))


@pytest.mark.gpu
@pytest.mark.parametrize("d, G", [(64, 8), (64, 5), (128, 4), (256, 2)])
@pytest.mark.parametrize("where", [20, 300, 2900, 2955])
def test_nan_values_in_split_prompts(d, G, where):
    """A NaN block of V under a few new tokens of a long row, whose keys are split over
    workgroups: in a tile that every row sees, one that the window's edge or the last rows
    cut, and one of the sinks."""
    n_kv = 2
    c = case([3000, 2980], [50, 3], n_kv, G, d, 16, seed=where)
    v = c["v"][0][where].clone()
    v[1, d - 1] = torch.nan
    _put(c, 0, where, v=v)
    c["v"][0][where, 1, d - 32:] = torch.nan
    for window, sinks in ((0, 0), (2660, 0), (100, 21), (47, 0), (2700, 300)):
        _agree(*_prefill(c, window, sinks), _exact(c, window, sinks))


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("lens, new", [([300, 300], [60, 7]), ([3000, 2000], [30, 7])])
def test_nan_keys_in_prompts(d, lens, new):
    """A written K block that is not finite: the rows that see it are NaN; it stands behind
    the window of others, between it and the sinks, or past them."""
    n_kv, G = 2, 4
    c = case(lens, new, n_kv, G, d, 16)
    n, m = lens[0], new[0]
    for bad, value in ((n - m // 2, torch.nan), (n - 100, torch.inf), (10, -torch.inf)):
        k = c["k"][0][bad].clone()
        k[0, 33] = value
        _put(c, 0, bad, k=k)
        for window, sinks in ((0, 0), (90, 0), (90, 4), (90, 11), (m // 2, 10), (n, 0)):
            out, lse = _prefill(c, window, sinks)
            pos = torch.arange(n - m, n, device="cuda")
            sees = (pos >= bad) & ((pos - bad < (window or n)) | (bad < sinks))
            assert bool(out[:m][sees][:, :G].isnan().all()) and bool(lse[:m][sees][:, :G].isnan().all())
            # the other rows and heads: as without the bad block
            o, z, to, tz = _exact(c, window, sinks)
            out[:m][sees, :G], lse[:m][sees, :G] = 0.0, 0.0
            for x in (o, z, to, tz):
                x[:m][sees, :G] = 0.0
            _agree(out, lse, (o, z, to, tz))
        _put(c, 0, bad)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128, 256])
def test_prompt_bounds_of_lengths(d):
    """A bound of the lengths that is exact, and one that is too low, on a wide table: what
    the call splits by, not what it attends to."""
    c = case([2100, 5, 777], [9, 5, 200], 2, 4, d, 16, width=4000)
    for window, sinks in ((0, 0), (700, 4)):
        want = _exact(c, window, sinks)
        for bound in (0, 2100, 300, 1):
            _agree(*_prefill(c, window, sinks, max_seq_len=bound), want)


@pytest.mark.gpu
@pytest.mark.parametrize("d, G", [(64, 8), (128, 4), (256, 4)])
def test_the_same_call_twice(d, G):
    """The same bits from the same call, whatever the workspace holds."""
    c = case([9000, 40, 3000, 0, 700], [1] * 5, 2, G, d, 16)
    p = case([9000, 40, 3000, 700], [30, 40, 1, 200], 2, G, d, 16)
    for call, x in ((_decode, c), (_prefill, p)):
        one = call(x)
        for _ in range(3):
            assert all(torch.equal(a, b) for a, b in zip(call(x), one))


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 64, 65])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_prompts_of_each_count_of_tiles(d, n):
    """One tile of keys to six, odd and even counts, for a tile of rows that sees them all or
    some; more rows than one workgroup's."""
    lens = [n + 64 * k for k in range(6)]
    c = case(lens, [min(m, 70) for m in lens], 3, 4, d, 16, seed=n)
    for window, sinks in ((0, 0), (65, 0), (64, 65)):
        _agree(*_prefill(c, window, sinks), _exact(c, window, sinks))


def test_engine_passes_the_bound_of_lengths(monkeypatch):
    """Both calls of a mixed step get the caller's bound (the table's width sizes them else)."""
    from locks.backend import engine
    got = []
    for name in ("window_decode", "window_prefill"):
        monkeypatch.setattr(engine, name, lambda *a, name=name, **kw: got.append((name, kw["max_seq_len"])))
    eng = engine.LocksEngine.__new__(engine.LocksEngine)
    eng._dense_ws = object()
    rows = torch.zeros(4, 8, dtype=torch.int32)
    for bound in (0, 500):
        eng.forward_dense(None, None, rows, rows[:, 0], 4, 1.0, None, query_start_loc=rows[0], n_decode=2,
                          **({"max_seq_len": bound} if bound else {}))
    assert got == [("window_decode", 0), ("window_prefill", 0), ("window_decode", 500), ("window_prefill", 500)]


@pytest.mark.gpu
@pytest.mark.parametrize("four", [False, True])
def test_engine_with_a_wide_table(four):
    """Short requests in an engine for long ones: the same rows with a bound of the lengths
    (exact, generous or too low) and without."""
    from locks import LocksConfig
    from locks.backend.engine import LocksEngine
    n_kv, G, d, page, blocks = 2, 4, 128, 16, 80
    selected = torch.zeros(blocks, 2, page, n_kv, d, dtype=torch.bfloat16, device="cuda")
    eng = LocksEngine(LocksConfig(budget_pages=8), [selected], num_heads_q=n_kv * G, num_heads_kv=n_kv, head_dim=d,
                      block_size=page, max_num_seqs=4, max_model_len=131072, max_num_batched_tokens=1024)
    cache, t = eng.kv4_cache() if four else selected, eng.block_tables()
    lens, new = [500, 281, 64], [500, 281, 64]
    for n_decode in (0, 3):
        T = sum(new)
        x = inputs(T, n_kv * G, n_kv, d, d, 1, seed=n_decode)
        t.step(torch.arange(3, dtype=torch.int32, device="cuda"), torch.tensor(new, dtype=torch.int32, device="cuda"),
               n_req=3, n_tokens=T)
        assert t.block_table.shape[1] == 8192
        eng.write_qkv(0, x["q"], x["k"], x["v"], x["pos"][0].contiguous(), t.slot_mapping[:T], None, torch.zeros_like(x["q"]),
                      kv_cache=cache)
        at = [torch.arange(n, device="cuda") for n in lens]
        slots = [t.block_table[r].long()[a // page] * page + a % page for r, a in enumerate(at)]
        kv = [_read(cache, s) if four else (cache[s // page, 0, s % page], cache[s // page, 1, s % page]) for s in slots]
        c = dict(q=x["q"], k=[k for k, _ in kv], v=[v for _, v in kv], lens=lens, new=new, n_kv=n_kv, G=G, d=d, scale=0.09)
        want = _exact(c, 0, 0)
        for bound in (0, max(lens), 4000, 16):
            out, lse = torch.zeros_like(x["q"]), torch.zeros(T, n_kv * G, device="cuda")
            eng.forward_dense(x["q"], cache, t.block_table, t.seq_lens, 3, 0.09, out, query_start_loc=t.query_start_loc,
                              n_decode=n_decode, lse=lse, max_seq_len=bound)
            _agree(out, lse, want)
        lens, new = [n + 1 for n in lens], [1, 1, 1]
