"""locks_call: the words of an entry reach it as its own arguments would, and a
wrong number of them, or of the entry, is refused (nothing reaches a GPU)."""
from locks import _lib


def test_call_words():
    lib = _lib.load()
    for name, (i, packer) in _lib._CALLS.items():
        args = [0.0 if t is _lib._f32 else 0 for t in _lib.SIGNATURES[name][1]]
        assert getattr(lib, name)(*args) == -1
        want = lib.locks_last_error()
        assert lib.locks_call(i, packer.pack(*args), len(args)) == -1
        assert lib.locks_last_error() == want and want.startswith(name.encode())
        assert lib.locks_call(i, packer.pack(*args), len(args) - 1) == -1
        assert b"arguments" in lib.locks_last_error()
    assert lib.locks_call(99, b"", 0) == -1 and lib.locks_call(0, None, 0) == -1
