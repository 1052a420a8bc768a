"""locks_call takes every word as the entry's own argument would be, or refuses it:
an integer past its argument's 32 bits is an error, not the number that its low half
makes, and no two words change places (nothing reaches a GPU)."""
import pytest

from locks import _lib

ATTN = "q qst qsh k kb kt kh v vb vt vh nb bt bst cols sl".split()
OUT = "out ost osh lse lst ws wsb".split()
NAMES = {
    "locks_tables_step": "rows new n T lens table ts max_reqs max_pages free nb state bt bs sl qsl pos slots page stream",
    "locks_tables_trim": "rows keep n lens table ts max_reqs max_pages free nb state page stream",
    "locks_qkv_write": "q qst qsh k kst ksh v vst vsh pos slots kc kcb kct kch vc vcb vct vch nb cs max_pos rot inter qw "
                       "kw f32 eps qo qost qosh ko kost kosh T H nkv d page stream",
    "locks_window_decode": " ".join(ATTN + ["window", "sinks"] + OUT) + " n nkv G d page maxs scale stream",
    "locks_window_prefill": " ".join(ATTN + ["qsl", "window", "sinks"] + OUT) + " T n nkv G d page maxs scale stream",
    "locks_prefix_decode": " ".join(ATTN + ["gs", "gp", "ng"] + OUT) + " n nkv G d page maxp maxs scale stream",
}
# good values, distinct where an entry takes two of a kind, and what is bad of each
GOOD = dict(nb=40, cols=4096, window=0, sinks=5, n=2, T=6, nkv=8, G=4, d=128, page=16, maxs=900, maxp=7, ng=1, scale=0.5,
            wsb=1 << 30, stream=0, ts=8, bs=12, max_reqs=4, max_pages=8, max_pos=500, rot=64, inter=0, f32=0, eps=1e-6, H=32)
BAD = dict(nb=-41, cols=1 << 27, window=-3, sinks=-5, n=70001, T=-6, nkv=5001, G=19, d=96, page=17, maxs=-900, maxp=-7,
           ng=65599, scale=-0.5, wsb=90, ts=7, bs=5, max_reqs=2051, max_pages=1 << 28, max_pos=-500, rot=68, eps=-1.0, H=5003)


def _entry(name):
    names = NAMES[name].split()
    types = _lib.SIGNATURES[name][1]
    assert len(names) == len(types)
    # a pointer of its own for each (16-byte aligned; never followed)
    return names, types, {n: GOOD.get(n, 16 * (i + 1)) for i, n in enumerate(names)}


def _both(name, values):
    """The messages of the entry called by its arguments and by words."""
    lib, (i, packer) = _lib.load(), _lib._CALLS[name]
    out = []
    for call in (lambda: getattr(lib, name)(*values), lambda: lib.locks_call(i, packer.pack(*values), len(values))):
        assert call() == -1
        out.append(lib.locks_last_error())
    return out


@pytest.mark.parametrize("name", NAMES)
def test_the_same_message_as_the_entry(name):
    names, types, base = _entry(name)
    said = set()
    for n in names:
        bads = [BAD[n]] if n in BAD else []
        bads += [0] if types[names.index(n)] is _lib._p and n not in ("stream", "lse", "qw", "kw", "ko") else []
        for bad in bads:
            direct, words = _both(name, list({**base, n: bad}.values()))
            assert direct == words and direct.startswith(name.encode()), (n, bad, direct)
            said.add(direct)
    assert len(said) > 5


@pytest.mark.parametrize("name", NAMES)
def test_integers_past_32_bits(name):
    lib, (i, packer) = _lib.load(), _lib._CALLS[name]
    names, types, base = _entry(name)
    for at, (n, t) in enumerate(zip(names, types)):
        if t is not _lib._i32:
            continue
        for far in (base[n] + (1 << 32), base[n] - (1 << 32), 1 << 31, -(1 << 31) - 1, (1 << 62) + base[n]):
            values = list({**base, n: far}.values())
            assert lib.locks_call(i, packer.pack(*values), len(values)) == -1, (n, far)
            said = lib.locks_last_error().decode()
            assert "32 bits" in said and str(far) in said and f"word {at} " in said, said
