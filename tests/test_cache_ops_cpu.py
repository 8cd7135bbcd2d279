"""Arguments of the e4m3 cache, tree attention and path-keeping entry points: what is refused, with which status, before
anything reaches the GPU, and that the native calls and ctypes agree.  The plain forms the GPU tests use are checked here
too."""
import ctypes

import numpy as np
import pytest

import cache_ref as ref

F = 256  # never dereferenced: every call below is refused, or has nothing to do
ST = (4096, 256, 128, 1)


def _expect(fn, exc, status, *args, **kw):
    with pytest.raises(exc) as info:
        fn(*args, **kw)
    assert info.value.status == status, str(info.value)
    return str(info.value)


def test_append_and_read_refusals(q3k):
    IA, OR, OV = q3k.Q3K_ERR_INVALID_ARGUMENT, q3k.Q3K_ERR_OUT_OF_RANGE, q3k.Q3K_ERR_OVERFLOW
    append = lambda *a, **k: q3k.kv_append_e4m3(F, F, F, F, F, *a, **k)  # noqa: E731
    # B, S, Hkv, D, seq_cap, start
    assert "capacity" in _expect(append, IndexError, OR, 2, 5, 8, 128, 8, 4)
    _expect(append, IndexError, OR, 2, 9, 8, 128, 8, 0, starts=F)
    _expect(append, IndexError, OR, 2, 1, 8, 128, 8, -1)
    _expect(append, ValueError, IA, -1, 5, 8, 128, 8, 0)
    _expect(append, ValueError, IA, 2, -5, 8, 128, 8, 0)
    _expect(append, ValueError, IA, 2, 5, 0, 128, 8, 0)
    _expect(append, ValueError, IA, 2, 5, 8, 0, 8, 0)
    _expect(append, ValueError, IA, 2, 5, 8, 128, 0, 0)
    _expect(append, ValueError, IA, 2, 1, 8, 128, 8, 0, starts=F + 2)
    _expect(append, OverflowError, OV, 2**40, 1, 8, 128, 2**20, 0)
    _expect(append, OverflowError, OV, 2**20, 2**10, 8, 128, 2**10, 0)
    for i in range(5):
        args = [F] * 5
        args[i] = None
        _expect(q3k.kv_append_e4m3, ValueError, IA, *args, 2, 5, 8, 128, 8, 0)
    _expect(q3k.kv_append_e4m3, ValueError, IA, F + 1, F, F, F, F, 2, 5, 8, 128, 8, 0)
    q3k.kv_append_e4m3(None, None, None, None, None, 0, 5, 8, 128, 8, 0)
    q3k.kv_append_e4m3(None, None, None, None, None, 3, 0, 8, 128, 8, 8)
    read = lambda *a, **k: q3k.kv_read_e4m3(F, F, F, F, F, *a, **k)  # noqa: E731
    # B, Hkv, D, seq_cap, first, count
    assert "capacity" in _expect(read, IndexError, OR, 2, 8, 128, 8, 4, 5)
    _expect(read, IndexError, OR, 2, 8, 128, 8, -1, 5)
    _expect(read, ValueError, IA, 2, 8, 128, 8, 0, -1)
    _expect(read, ValueError, IA, 2, 8, 128, 8, 0, 1, lengths=F + 1)
    _expect(q3k.kv_read_e4m3, ValueError, IA, F, F, None, F, F, 2, 8, 128, 8, 0, 1)
    _expect(q3k.kv_read_e4m3, ValueError, IA, F, F, F, F, F + 1, 2, 8, 128, 8, 0, 1)
    q3k.kv_read_e4m3(None, None, None, None, None, 2, 8, 128, 8, 8, 0)


def test_attention_refusals(q3k):
    IA, OV = q3k.Q3K_ERR_INVALID_ARGUMENT, q3k.Q3K_ERR_OVERFLOW

    def causal(B, S, Hq, Hkv, D, cap, cached, p=(F,) * 5, **kw):
        return q3k.gqa_attention_e4m3(*p, B, S, Hq, Hkv, D, cap, cached, **kw)

    def tree8(B, S, Hq, Hkv, D, cap, cached, p=(F,) * 5, parents=F, stride=None, **kw):
        return q3k.gqa_tree_attention_e4m3(*p, parents, S if stride is None else stride, B, S, Hq, Hkv, D, cap, cached, **kw)

    def tree16(B, S, Hq, Hkv, D, cap, cached, p=(F,) * 4, parents=F, stride=None, ks=ST, vs=ST, **kw):
        return q3k.gqa_tree_attention(*p[:4], parents, S if stride is None else stride, B, S, Hq, Hkv, D, cached, ks, vs, **kw)

    for call in (causal, tree8, tree16):
        _expect(call, ValueError, IA, -1, 1, 4, 2, 128, 16, 8)
        _expect(call, ValueError, IA, 1, -1, 4, 2, 128, 16, 8)
        assert "divisible" in _expect(call, ValueError, IA, 1, 1, 3, 2, 128, 16, 8)
        _expect(call, ValueError, IA, 1, 1, 4, 0, 128, 16, 8)
        _expect(call, ValueError, IA, 1, 1, 4, 2, 257, 16, 8)
        _expect(call, ValueError, IA, 1, 1, 4, 2, 0, 16, 8)
        _expect(call, ValueError, IA, 1, 1, 4, 2, 128, 16, -1)
        assert "hold" in _expect(call, ValueError, IA, 1, 9, 4, 2, 128, 16, 8)   # no lengths: the queries are in the cache
        _expect(call, ValueError, IA, 1, 1, 4, 2, 128, 16, 8, lengths=F + 2)
        _expect(call, OverflowError, OV, 2**22, 200, 4, 2, 128, 2**10, 2**10)
        _expect(call, OverflowError, OV, 1, 1, 4, 2, 128, 2**33, 2**32)
        for i in range(4):
            p = [F] * 5
            p[i] = None
            _expect(call, ValueError, IA, 1, 1, 4, 2, 128, 16, 8, p=p)
        call(0, 1, 4, 2, 128, 16, 8, p=(None,) * 5)
        call(1, 0, 4, 2, 128, 16, 8, p=(None,) * 5)
    for call in (causal, tree8):
        _expect(call, ValueError, IA, 1, 1, 4, 2, 128, 16, 17)
        _expect(call, ValueError, IA, 1, 1, 4, 2, 128, 0, 0, lengths=F)
        _expect(call, ValueError, IA, 1, 1, 4, 2, 128, 16, 8, p=(F + 1,) + (F,) * 4)
        _expect(call, OverflowError, OV, 1, 1, 4, 2, 128, 2**60, 8)
    for call in (tree8, tree16):
        _expect(call, ValueError, IA, 1, 4, 4, 2, 128, 16, 8, parents=None)
        assert "256 nodes" in _expect(call, ValueError, IA, 1, 257, 4, 2, 128, 512, 512)
        _expect(call, ValueError, IA, 2, 4, 4, 2, 128, 16, 8, stride=3)
        _expect(call, ValueError, IA, 2, 4, 4, 2, 128, 16, 8, stride=-4)
        _expect(call, ValueError, IA, 2, 4, 4, 2, 128, 16, 8, parents=F + 2)
    _expect(tree16, ValueError, IA, 1, 4, 4, 2, 128, 16, 8, ks=(4096, -256, 128, 1))
    _expect(tree16, ValueError, IA, 1, 4, 4, 2, 128, 16, 8, p=(F, F + 1, F, F))


def test_keep_refusals(q3k):
    IA, OR, OV = q3k.Q3K_ERR_INVALID_ARGUMENT, q3k.Q3K_ERR_OUT_OF_RANGE, q3k.Q3K_ERR_OVERFLOW

    def keep(layers, cap_b, heads, seq, row, B, start, n, kc=F, vc=F, sc=None, path=F, **kw):
        return q3k.kv_keep_path(kc, vc, sc, layers, cap_b, heads, seq, row, B, start, path, n, **kw)

    _expect(keep, ValueError, IA, -1, 4, 1, 16, 64, 2, 0, 4)
    _expect(keep, ValueError, IA, 2, 4, 1, 16, 64, -2, 0, 4)
    _expect(keep, ValueError, IA, 2, 4, 1, 16, 64, 2, 0, -4)
    for dims in ((0, 1, 16, 64), (4, 0, 16, 64), (4, 1, 0, 64), (4, 1, 16, 0)):
        _expect(keep, ValueError, IA, 2, *dims, 0, 0, 0)
    _expect(keep, IndexError, OR, 2, 4, 1, 16, 64, 5, 0, 4)
    _expect(keep, IndexError, OR, 2, 4, 1, 16, 64, 2, 13, 4)
    _expect(keep, IndexError, OR, 2, 4, 1, 16, 64, 2, -1, 4)
    _expect(keep, OverflowError, OV, 2**40, 2**20, 1, 16, 64, 2, 0, 4)
    _expect(keep, OverflowError, OV, 2, 4, 1, 16, 2**31, 2, 0, 4)
    for name in ("kc", "vc", "path"):
        _expect(keep, ValueError, IA, 2, 4, 1, 16, 64, 2, 0, 4, **{name: None})
    for kw in ({"path": F + 1}, {"starts": F + 2}, {"counts": F + 3}, {"sc": F + 1}):
        _expect(keep, ValueError, IA, 2, 4, 1, 16, 64, 2, 0, 4, **kw)
    keep(0, 4, 1, 16, 64, 2, 0, 4, kc=None)
    keep(2, 4, 1, 16, 64, 0, 0, 4, kc=None)
    keep(2, 4, 1, 16, 64, 2, 0, 0, kc=None)


def test_workspace_query_of_nothing(q3k):
    ws = q3k.cache_attention_workspace_bytes
    for args in ((0, 1, 4, 2, 128, 100), (1, 0, 4, 2, 128, 100), (1, 1, 3, 2, 128, 100), (1, 1, 4, 0, 128, 100),
                 (1, 1, 4, 2, 64, 5000), (1, 1, 4, 2, 128, 0), (2**20, 2**12, 4, 2, 128, 2**12), (1, 1, 4, 2, 128, 2**40)):
        assert ws(*args) == 0


class _HandsBack:
    def __getattr__(self, name):
        return lambda *args: None


def test_native_calls_take_what_ctypes_takes(q3k, monkeypatch):
    p8 = (None, F, F, F, F)
    cases = [
        (q3k.kv_append_e4m3, (None, F, F, F, F, 1, True, 8, 128, 8, 0)),
        (q3k.kv_append_e4m3, (F, F, F, F, F, np.int64(-1), 1, 8, 128, 8, 0)),
        (q3k.kv_read_e4m3, (F, F, F, None, F, 1, 8, 128, np.int32(8), 0, 1)),
        (q3k.gqa_attention_e4m3, p8 + (1, 1, 2, 1, 128, 8, 4)),
        (q3k.gqa_attention_e4m3, p8 + (1, 1, 2, 1, 128, 8, 4, ctypes.c_void_p(None))),
        (q3k.gqa_tree_attention_e4m3, p8 + (F, 1, 1, 1, 2, 1, 128, 8, 4)),
        (q3k.gqa_tree_attention_e4m3, p8 + (F, 1, 1, 1, 2, 1, 128, "8", 4)),
        (q3k.gqa_tree_attention, p8[:4] + (F, 1, 1, 1, 2, 1, 128, 4, ST, ST)),
        (q3k.gqa_tree_attention, p8[:4] + (F, 1, 1, 1, 2, 1, 128, 4, list(ST), np.array(ST))),
        (q3k.gqa_tree_attention, p8[:4] + (F, 1, 1, 1, 2, 1, 128, 4, ST[:3], ST)),
        (q3k.kv_keep_path, (None, F, None, 1, 1, 1, 8, 64, 1, 0, F, True)),
        (q3k.kv_keep_path, (F, F, None, 1, 1, 1, 8, 64, 1, 9.0, F, 1)),
    ]

    def outcome(fn, args):
        try:
            return fn(*args)
        except Exception as e:  # noqa: BLE001
            return type(e), getattr(e, "status", None), str(e)

    native = [outcome(*c) for c in cases]
    q3k.load()
    monkeypatch.setattr(q3k, "_calls", _HandsBack())
    for c, got in zip(cases, native):
        assert got is not None and got == outcome(*c), f"{c[0].__name__}{c[1]}"


# ---- the plain forms -------------------------------------------------------------------

def test_plain_encoding():
    """Every code encodes to itself; a tie goes to the even code; the step is half an e4m3 step, 2^-4, at most."""
    finite = np.array([c for c in range(256) if (c & 127) != 127])
    assert np.array_equal(ref.encode(ref.CODE[finite]), finite)
    mid = (ref.CODE[1:127] + ref.CODE[0:126]) / 2
    got = ref.encode(mid)
    assert np.all(got % 2 == 0) and np.all(np.abs(got.astype(int) - np.arange(126) - 0.5) == 0.5)
    rng = np.random.default_rng(1)
    x = rng.uniform(2.0**-6, 448, 10000)
    assert np.all(np.abs(ref.CODE[ref.encode(x)] - x) <= x * 2.0**-4)
    assert list(ref.encode(np.array([np.inf, -np.inf, np.nan]))) == [0x7F] * 3


def test_plain_scale():
    """448 * 2^e holds exactly up to the boundary, zeros and subnormals take the least scale, the largest bf16 fits."""
    rows = np.zeros((6, 8), np.uint16)
    rows[1, 0] = 0x43E0          # 448
    rows[2, 0] = 0x43E1          # one bf16 step above it
    rows[3, 0] = 0x7F7F          # the largest bf16
    rows[4, 0] = 0x0001          # the smallest subnormal
    rows[5, :2] = 0x7F80, 0x43E0  # an infinity does not count
    codes, byte = ref.quantise(rows)
    assert byte.tolist() == [1, 127, 128, 247, 1, 127]
    assert codes[5, 0] == 0x7F and codes[5, 1] == 0x7E and codes[1, 0] == 0x7E
    assert np.isfinite(ref.dequantise(codes[3], byte[3])).all()


def test_plain_tree():
    states, seen = ref.ancestors([-1, 0, 0, 2, -1, -2, 5, 9, -3])
    assert states == ["sees"] * 5 + ["empty"] * 2 + ["bad"] * 2
    assert [np.flatnonzero(r).tolist() for r in seen[:5]] == [[0], [0, 1], [0, 2], [0, 2, 3], [4]]
    # a chain of nodes is causal attention
    rng = np.random.default_rng(2)
    q, k, v = rng.standard_normal((4, 4, 8)), rng.standard_normal((9, 2, 8)), rng.standard_normal((9, 2, 8))
    a, _ = ref.attention(q, k, v, 9, 4)
    b, _ = ref.attention(q, k, v, 9, 4, [-1, 0, 1, 2])
    assert np.array_equal(a, b)
