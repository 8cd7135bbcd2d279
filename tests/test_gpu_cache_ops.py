"""The e4m3 KV cache, attention over a cache with a length for each sequence, trees of drafted tokens and the accepted
path, against plain 64-bit forms (cache_ref): codes and copies exactly, attention within half a bf16 step and the bound
that cache_ref.attention derives.  Rows that a call must not read hold NaN, rows that it must not write are compared."""
import numpy as np
import pytest

import cache_ref as ref
from gpu_util import Guarded, announce

pytestmark = pytest.mark.gpu


def _up(hip, *arrays):
    return [hip.DeviceBuffer.from_array(a) for a in arrays]


# ---- quantising append, reading back ---------------------------------------------------

def _rows(rng, B, S, Hkv, D):
    """bf16 rows of magnitudes from 2^-130 to 2^120, zero rows, rows with an infinity or a NaN."""
    x = rng.standard_normal((B, S, Hkv, D)).astype(np.float64) * np.exp2(rng.integers(-12, 12, (B, S, Hkv, 1)).astype(float))
    flat = x.reshape(-1, D)
    for i, p in enumerate((0.0, 2.0**-130, 2.0**120, 2.0**-60)):
        if i < len(flat):
            flat[(5 * i + 1) % len(flat)] *= p
    bits = (x.astype(np.float32).view(np.uint32) >> 16).astype(np.uint16)
    for i, special in enumerate((0x7F80, 0xFF80, 0x7FC1, 0x43E0, 0x8000)):
        bits.reshape(-1, D)[(7 * i + 3) % len(flat), (11 * i + 1) % D] = special
    return bits


@pytest.mark.parametrize("offset", [0, 2])
@pytest.mark.parametrize("B,S,Hkv,D,cap,start", [
    (1, 1, 8, 128, 16, 5), (3, 7, 8, 128, 16, 9), (2, 65, 1, 128, 70, 0), (2, 5, 3, 64, 8, 1), (2, 5, 2, 256, 8, 1),
    (2, 4, 2, 80, 9, 3), (1, 3, 5, 1, 4, 0), (1, 2, 2, 300, 4, 2), (4, 700, 2, 128, 700, 0)])
def test_append(q3k, hip, B, S, Hkv, D, cap, start, offset):
    announce(f"kv_append_e4m3 {B}x{S} heads {Hkv} D {D} cap {cap} start {start} offset {offset}")
    rng = np.random.default_rng(B * 1000 + S + D)
    k, v = _rows(rng, B, S, Hkv, D), _rows(rng, B, S, Hkv, D)
    bk, bv = Guarded(hip, k, offset=offset), Guarded(hip, v, offset=offset)
    shape = (B, Hkv, cap, D)
    old = rng.integers(0, 256, shape, dtype=np.uint8)
    sold = rng.integers(0, 256, (B, Hkv, cap, 2), dtype=np.uint8)
    kc, vc, sc = (Guarded(hip, a, offset=o) for a, o in ((old, offset // 2), (old, 0), (sold, offset // 2)))
    q3k.kv_append_e4m3(bk, bv, kc, vc, sc, B, S, Hkv, D, cap, start)
    hip.synchronize()
    want_k, want_v, want_s = old.copy(), old.copy(), sold.copy()
    for i, (x, w) in enumerate(((k, want_k), (v, want_v))):
        codes, byte = ref.quantise(x)
        w[:, :, start:start + S] = codes.transpose(0, 2, 1, 3)
        want_s[:, :, start:start + S, i] = byte.transpose(0, 2, 1)
    assert np.array_equal(sc.get(np.uint8, sold.shape), want_s)
    assert ref.same_codes(kc.get(np.uint8, shape), want_k) and ref.same_codes(vc.get(np.uint8, shape), want_v)
    assert all(b.guards_intact() for b in (bk, bv, kc, vc, sc))


@pytest.mark.parametrize("D", [128, 72])
def test_append_starts_and_read(q3k, hip, D):
    """Rows at a start of each sequence's own, some partly or wholly outside the cache (nothing is written there), then
    read back: exactly code * scale, rows at or past a length left alone."""
    announce(f"kv_append_e4m3 with starts, kv_read_e4m3, D {D}")
    B, S, Hkv, cap = 7, 3, 2, 10
    starts = np.array([0, 7, 8, 9, -1, 10, 2**31 - 2], np.int32)
    rng = np.random.default_rng(D)
    k, v = _rows(rng, B, S, Hkv, D), _rows(rng, B, S, Hkv, D)
    codes = rng.integers(0, 0x7F, (B, Hkv, cap, D), dtype=np.uint8)
    scales = rng.integers(100, 150, (B, Hkv, cap, 2), dtype=np.uint8)
    kc, vc, sc = (Guarded(hip, a) for a in (codes, codes, scales))
    bk, bv, bs = _up(hip, k, v, starts)
    q3k.kv_append_e4m3(bk, bv, kc, vc, sc, B, S, Hkv, D, cap, 999, starts=bs)
    hip.synchronize()
    want_k, want_v, want_s = codes.copy(), codes.copy(), scales.copy()
    (ck, ek), (cv, ev) = ref.quantise(k), ref.quantise(v)
    for b in range(B):
        for s in range(S):
            pos = int(starts[b]) + s
            if 0 <= pos < cap:
                want_k[b, :, pos], want_v[b, :, pos] = ck[b, s], cv[b, s]
                want_s[b, :, pos, 0], want_s[b, :, pos, 1] = ek[b, s], ev[b, s]
    assert ref.same_codes(kc.get(np.uint8, codes.shape), want_k) and ref.same_codes(vc.get(np.uint8, codes.shape), want_v)
    assert np.array_equal(sc.get(np.uint8, scales.shape), want_s)
    assert all(b.guards_intact() for b in (kc, vc, sc))
    first, count = 1, 8
    lengths = np.array([10, 9, 5, 1, 0, -3, 100], np.int32)
    bl, = _up(hip, lengths)
    for given in (None, bl):
        ko, vo = (Guarded(hip, np.full((B, count, Hkv, D), 0x1234, np.uint16)) for _ in range(2))
        q3k.kv_read_e4m3(kc, vc, sc, ko, vo, B, Hkv, D, cap, first, count, lengths=given)
        hip.synchronize()
        for i, (out, c) in enumerate(((ko, want_k), (vo, want_v))):
            got = out.get(np.uint16, (B, count, Hkv, D))
            x = ref.dequantise(c, want_s[..., i])[:, :, first:first + count].transpose(0, 2, 1, 3)
            n = lengths if given is not None else np.full(B, cap)
            left = np.broadcast_to((first + np.arange(count))[None, :] >= n[:, None], (B, count))
            assert np.all(got[left] == 0x1234)
            want = x[~left]
            # exact down to 2^-126; below it half of bf16's smallest step, 2^-133
            ok = (ref.bf16(got[~left]) == want) | ((np.abs(want) < 2.0**-126) & (np.abs(ref.bf16(got[~left]) - want) <= 2.0**-134))
            assert np.all(ok | (np.isnan(want) & np.isnan(ref.bf16(got[~left]))))
            assert out.guards_intact()


# ---- attention -------------------------------------------------------------------------

class _Cache:
    """A cache of B sequences of the given lengths; rows past a length hold NaN (and scale bytes 255)."""

    def __init__(self, hip, rng, e4m3, B, Hkv, D, cap, lengths, std=1.0, strides=None):
        self.e4m3, self.cap, self.hip = e4m3, cap, hip
        past = np.arange(cap)[None, :] >= np.asarray(lengths)[:, None]
        x = [(rng.standard_normal((B, cap, Hkv, D)) * std).astype(np.float32) for _ in range(2)]
        bits = [(a.view(np.uint32) >> 16).astype(np.uint16) for a in x]
        self.values, stored = [], []
        if e4m3:
            self.bytes = np.empty((B, Hkv, cap, 2), np.uint8)
            for i, b in enumerate(bits):
                codes, byte = ref.quantise(b)
                self.values.append(ref.dequantise(codes, byte))
                codes[past], byte[past] = 0x7F, 255
                stored.append(np.ascontiguousarray(codes.transpose(0, 2, 1, 3)))
                self.bytes[..., i] = byte.transpose(0, 2, 1)
        else:
            for b in bits:
                self.values.append(ref.bf16(b))
                b[past] = 0x7FC0
                if strides == "head-major":
                    b = np.ascontiguousarray(b.transpose(0, 2, 1, 3))
                elif strides == "odd":  # rows of D + 3 elements
                    b = np.concatenate([b, np.full(b.shape[:3] + (3,), 0x7FC0, np.uint16)], -1)
                stored.append(b)
            w = D + 3 if strides == "odd" else D
            self.strides = (cap * Hkv * w, w, cap * w, 1) if strides == "head-major" else (cap * Hkv * w, Hkv * w, w, 1)
        self.stored = stored
        self.upload()

    def upload(self):
        self.k, self.v = (Guarded(self.hip, a) for a in self.stored)
        self.s = Guarded(self.hip, self.bytes) if self.e4m3 else None

    def poison(self, b, row, bits16=0x7FC0, value=np.nan):
        """K and V of one row (all heads) become `value`."""
        for x, s in zip(self.values, self.stored):
            x[b, row] = value
            if self.e4m3:
                s[b, :, row] = 0x7F
            else:
                s[b, row] = bits16
        self.upload()


def _run(q3k, hip, c, q, B, S, Hq, Hkv, D, cached, lengths, parents, ws, stream=None, out=None):
    """One call; lengths and parents are device buffers or None, ws (buffer, bytes)."""
    out = Guarded(hip, np.full((B, S, Hq, D), 0x1234, np.uint16)) if out is None else out
    buf, n = ws if ws is not None else (None, 0)
    kw = dict(lengths=lengths, workspace=buf, workspace_bytes=n, stream=stream)
    if parents is None:
        q3k.gqa_attention_e4m3(q, c.k, c.v, c.s, out, B, S, Hq, Hkv, D, c.cap, cached, **kw)
    elif c.e4m3:
        q3k.gqa_tree_attention_e4m3(q, c.k, c.v, c.s, out, parents[0], parents[1], B, S, Hq, Hkv, D, c.cap, cached, **kw)
    else:
        q3k.gqa_tree_attention(q, c.k, c.v, out, parents[0], parents[1], B, S, Hq, Hkv, D, cached, c.strides, c.strides, **kw)
    return out


def _workspace(q3k, hip, B, S, Hq, Hkv, D, cached):
    n = q3k.cache_attention_workspace_bytes(B, S, Hq, Hkv, D, cached)
    if n == 0:
        return None
    buf = Guarded(hip, nbytes=n)
    return buf, n


def _reference(c, q, lengths, cached, S, parents):
    outs = []
    for b in range(q.shape[0]):
        n = cached if lengths is None else int(lengths[b])
        bad = n < 0 or n > cached or (parents is not None and 0 < n < S)
        if bad:
            outs.append((np.full(q.shape[1:], np.nan), np.zeros(q.shape[1:])))
            continue
        p = None if parents is None else parents[b]
        if n == 0:
            outs.append((np.zeros(q.shape[1:]), np.zeros(q.shape[1:])))
            continue
        outs.append(ref.attention(q[b], c.values[0][b, :n], c.values[1][b, :n], n, S, p))
    return np.stack([o[0] for o in outs]), np.stack([o[1] for o in outs])


def _queries(rng, B, S, Hq, D, std=2.0):
    x = (rng.standard_normal((B, S, Hq, D)) * std).astype(np.float32)
    return (x.view(np.uint32) >> 16).astype(np.uint16)


def _compare(q3k, hip, name, e4m3, B, S, Hq, Hkv, D, cap, cached, lengths=None, parents=None, stride=None, seed=0, strides=None,
             workspaces=(False, True), edit=None):
    announce(name)
    rng = np.random.default_rng(seed + B + 31 * S + cached)
    real = [cached] * B if lengths is None else [min(max(int(n), 0), cached) for n in lengths]
    c = _Cache(hip, rng, e4m3, B, Hkv, D, cap, real, strides=strides)
    if edit is not None:
        edit(c)
    q = _queries(rng, B, S, Hq, D)
    bq, = _up(hip, q)
    bl = _up(hip, np.asarray(lengths, np.int32))[0] if lengths is not None else None
    bp, trees = None, None
    if parents is not None:
        table = np.asarray(parents, np.int32)
        bp = (_up(hip, table)[0], S if stride is None else stride)
        trees = [table.reshape(-1)[b * bp[1]:b * bp[1] + S] for b in range(B)]
    want = _reference(c, ref.bf16(q).reshape(q.shape), lengths, cached, S, trees)
    for with_ws in workspaces:
        ws = _workspace(q3k, hip, B, S, Hq, Hkv, D, cached) if with_ws else None
        out = _run(q3k, hip, c, bq, B, S, Hq, Hkv, D, cached, bl, bp, ws)
        hip.synchronize()
        ref.check_attention(f"{name} workspace {ws is not None}", out.get(np.uint16, q.shape), *want)
        assert out.guards_intact() and (ws is None or ws[0].guards_intact())


@pytest.mark.parametrize("B,S,Hq,Hkv,cached,lengths", [
    (1, 1, 4, 2, 1, None),
    (1, 1, 16, 8, 777, None),
    (5, 1, 8, 2, 130, [130, 129, 64, 1, 0]),
    (6, 1, 5, 1, 260, [260, 65, 63, 33, 32, 31]),
    (4, 1, 8, 8, 2049, [2049, 2048, 1000, 17]),
    (3, 1, 64, 8, 600, [600, 0, 599]),
    (2, 1, 40, 1, 300, None),               # 40 query heads to a KV head: more columns than a wave
    (3, 2, 8, 2, 100, [100, 1, 2]),         # a query before the first row
    (2, 3, 10, 2, 97, [97, 40]),
    (2, 8, 8, 2, 200, [200, 5]),
    (1, 17, 8, 8, 17, None),
    (2, 33, 5, 1, 500, [500, 20]),
    (1, 130, 4, 1, 1000, None),
    (2, 100, 8, 2, 164, [164, 99]),
    (1, 200, 16, 2, 200, None),
    (4, 1, 4, 1, 64, [65, -1, 64, 10]),     # lengths out of range
    (3, 40, 4, 1, 64, [65, -1, 64])])
def test_causal_e4m3(q3k, hip, B, S, Hq, Hkv, cached, lengths):
    _compare(q3k, hip, f"attention e4m3 {B}x{S} heads {Hq}/{Hkv} rows {cached} {lengths}", True, B, S, Hq, Hkv, 128, cached + 3,
             cached, lengths)


# Lengths that the blocks' order has to cope with: below 0 and above the cache's, equal ones, the last of more than 64
# sequences among themselves.
LOWEST, HIGHEST = -2**31, 2**31 - 1
ORDERS = {
    "below": [-5, LOWEST, 40, -2, 17], "all-below": [LOWEST, -2, -3], "above": [HIGHEST, 64, 65, LOWEST, 64],
    "equal": [33] * 6, "67": [(37 * i) % 65 for i in range(64)] + [12, LOWEST, 64],
    "130": [64 - i % 65 for i in range(128)] + [-7, 3]}


@pytest.mark.parametrize("form", ["causal", "tree", "tree-bf16"])
@pytest.mark.parametrize("S", [1, 40])
@pytest.mark.parametrize("order", sorted(ORDERS))
def test_order_of_lengths(q3k, hip, order, S, form):
    lengths = ORDERS[order]
    B, trees = len(lengths), None
    if form != "causal":
        lengths = [n if n <= 0 else max(n, S) for n in lengths]
        trees = _random_trees(np.random.default_rng(S + B), B, S)
    _compare(q3k, hip, f"order of lengths {order} S {S} {form}", form != "tree-bf16", B, S, 4, 2, 128, 66, 64, lengths, trees)


@pytest.mark.parametrize("D", [1, 64, 80, 256])
def test_causal_e4m3_other_widths(q3k, hip, D):
    _compare(q3k, hip, f"attention e4m3 D {D}", True, 2, 3, 4, 2, D, 40, 37, [37, 2], workspaces=(True,))


def _random_trees(rng, B, T, pad=True):
    """Random parents; with pad some trees are smaller and one node of each larger tree names a wrong parent."""
    p = np.full((B, T), -1, np.int32)
    for b in range(B):
        for t in range(1, T):
            p[b, t] = rng.integers(-1, t)
        if pad and b % 2 == 1:
            p[b, max(1, T // 2):] = -2
        if pad and b % 3 == 2 and T > 3:
            p[b, T // 3] = T
    return p


TREES = [
    (1, 1, 4, 2, 1, None), (1, 5, 8, 2, 5, None), (3, 4, 8, 2, 70, [70, 4, 33]), (2, 7, 4, 1, 200, [200, 64]),
    (4, 8, 8, 8, 131, [131, 8, 0, 7]), (2, 26, 8, 2, 300, [300, 90]), (3, 33, 5, 1, 129, [129, 33, 65]),
    (2, 64, 8, 2, 1000, [1000, 64]), (1, 100, 4, 1, 163, None), (2, 256, 4, 2, 400, [400, 256]), (1, 31, 40, 1, 95, None),
    (3, 6, 64, 8, 50, [51, -1, 5])]


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("B,T,Hq,Hkv,cached,lengths", TREES)
def test_tree(q3k, hip, B, T, Hq, Hkv, cached, lengths, e4m3):
    trees = _random_trees(np.random.default_rng(T), B, T)
    _compare(q3k, hip, f"tree e4m3 {e4m3} {B}x{T} heads {Hq}/{Hkv} rows {cached} {lengths}", e4m3, B, T, Hq, Hkv, 128, cached + 2,
             cached, lengths, trees)


def _long_ways(T):
    """Chains, ways that jump far back, and wrong parents and padding whose descendants lie far behind them."""
    chain = np.arange(-1, T - 1, dtype=np.int32)
    broken, padded, jumps, below = chain.copy(), chain.copy(), chain.copy(), chain.copy()
    broken[T // 3] = T - 1                       # a later node
    padded[T // 2] = -2
    jumps[T // 4:] = np.arange(T - T // 4) % (T // 4)
    below[T // 5] = -3
    below[T // 4:] = np.arange(T // 4, T) // 2
    below[-1] = -2**31
    return np.stack([chain, broken, padded, jumps, below])


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("T,Hq,Hkv", [(7, 4, 1), (32, 2, 2), (33, 2, 1), (64, 2, 1), (65, 4, 2), (128, 2, 1), (200, 4, 1), (256, 2, 2)])
def test_tree_long_ways(q3k, hip, T, Hq, Hkv, e4m3):
    trees = _long_ways(T)
    _compare(q3k, hip, f"tree long ways e4m3 {e4m3} T {T} heads {Hq}/{Hkv}", e4m3, 5, T, Hq, Hkv, 128, T + 40, T + 35,
             [T + 35, T, T + 3, T + 34, T + 20], trees)


@pytest.mark.parametrize("strides,D", [("head-major", 128), ("odd", 128), ("odd", 96), (None, 64)])
def test_tree_strides(q3k, hip, strides, D):
    trees = _random_trees(np.random.default_rng(3), 2, 9)
    _compare(q3k, hip, f"tree strides {strides} D {D}", False, 2, 9, 4, 2, D, 80, 77, [77, 30], trees, strides=strides)


@pytest.mark.parametrize("e4m3", [False, True])
def test_tree_shared_and_strided_parents(q3k, hip, e4m3):
    """One tree for all sequences (stride 0), and rows of a wider table."""
    T = 12
    tree = _random_trees(np.random.default_rng(4), 1, T, pad=False)
    _compare(q3k, hip, "tree shared parents", e4m3, 3, T, 8, 2, 128, 100, 90, [90, 50, 12], tree, stride=0)
    table = np.full((3, T + 5), -7, np.int32)
    table[:, :T] = _random_trees(np.random.default_rng(5), 3, T, pad=False)
    _compare(q3k, hip, "tree strided parents", e4m3, 3, T, 8, 2, 128, 100, 90, [90, 50, 12], table, stride=T + 5)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("T", [6, 40])
def test_tree_nan_rows_reach_only_their_descendants(q3k, hip, e4m3, T):
    """K and V of one node are NaN: the nodes that do not descend from it are as if it were finite."""
    def edit(c):
        c.poison(0, 70 - T + 2)
        c.poison(1, 50 - T + 3)

    trees = np.array([[-1, 0, 0, 1, 1, 2] + list(range(5, T - 1)), [-1, 0, 0, -2, 1, 2] + list(range(5, T - 1))], np.int32)[:, :T]
    _compare(q3k, hip, f"tree NaN rows e4m3 {e4m3} T {T}", e4m3, 2, T, 8, 2, 128, 80, 70, [70, 50], trees, edit=edit)


@pytest.mark.parametrize("bits,value", [(0x7F80, np.inf), (0xFF80, -np.inf)])
def test_tree_infinite_values(q3k, hip, bits, value):
    """V of one node is infinite (K finite): its descendants get that infinity, the others what they had."""
    def edit(c):
        c.values[1][0, 70 - 6 + 2] = value
        c.stored[1][0, 70 - 6 + 2] = bits
        c.upload()

    _compare(q3k, hip, f"tree infinite V {value}", False, 1, 6, 8, 2, 128, 80, 70, None, [[-1, 0, 0, 1, 1, 2]], edit=edit)


@pytest.mark.parametrize("S,cached", [(3, 70), (40, 100)])
def test_causal_nan_rows_reach_only_later_queries(q3k, hip, S, cached):
    def edit(c):
        c.poison(0, cached - 2)

    _compare(q3k, hip, f"causal NaN row S {S}", True, 1, S, 8, 2, 128, cached + 5, cached, None, edit=edit)


def test_nan_in_the_context_reaches_every_query_but_empty_ones(q3k, hip):
    def edit(c):
        c.poison(0, 3)

    for T in (4, 30):
        tree = [[-1, 0, -2, 1] + [3] * (T - 4)]
        _compare(q3k, hip, f"tree NaN context T {T}", False, 1, T, 8, 2, 128, 300, 280, None, tree, edit=edit)


def test_large_scores(q3k, hip):
    """Rows far apart in magnitude: the running maximum moves often, and most weights vanish."""
    announce("attention e4m3 large scores")
    rng = np.random.default_rng(8)
    B, Hq, Hkv, D, cached = 2, 8, 2, 128, 700
    c = _Cache(hip, rng, True, B, Hkv, D, cached, [cached] * B, std=6.0)
    q = _queries(rng, B, 1, Hq, D, std=6.0)
    bq, = _up(hip, q)
    want = _reference(c, ref.bf16(q).reshape(q.shape), None, cached, 1, None)
    for ws in (None, _workspace(q3k, hip, B, 1, Hq, Hkv, D, cached)):
        out = _run(q3k, hip, c, bq, B, 1, Hq, Hkv, D, cached, None, None, ws)
        hip.synchronize()
        ref.check_attention("large scores", out.get(np.uint16, q.shape), *want)


# ---- keeping the accepted path -----------------------------------------------------------

@pytest.mark.parametrize("heads,row,dtype,scaled,offset", [
    (1, 2048, np.uint8, False, 0), (8, 128, np.uint8, True, 0), (2, 80, np.uint8, True, 1), (1, 12, np.uint8, False, 4),
    (3, 7, np.uint8, True, 0)])
def test_keep_path(q3k, hip, heads, row, dtype, scaled, offset):
    """Rows move down along each sequence's path, in every layer; overlapping moves read before they write; entries that
    point up, past the cache or past the count leave their rows; other batch rows and layers are untouched."""
    announce(f"kv_keep_path heads {heads} row {row} scales {scaled}")
    L, cap_b, B, seq, n = 3, 6, 5, 40, 12
    rng = np.random.default_rng(row)
    k, v = (rng.integers(0, 256, (L, cap_b, heads, seq, row), dtype=np.uint8) for _ in range(2))
    s = rng.integers(0, 256, (L, cap_b, heads, seq, 2), dtype=np.uint8)
    starts = np.array([0, 20, 35, 3, 40], np.int32)      # the third runs past the cache, the last is outside
    path = np.sort(np.argsort(rng.random((B, 20)), 1)[:, :n], 1).astype(np.int32)
    path[0] = np.arange(n) + 1                          # every row from its neighbour
    path[3, 2:6] = [0, -1, 9, 9]                        # up, negative, the same node twice
    counts = np.array([n, 7, n, n, n], np.int32)
    for given_counts in (True, False):
        bufs = [Guarded(hip, a, offset=offset) for a in (k, v)] + [Guarded(hip, s) if scaled else None]
        bp, bs, bc = _up(hip, path, starts, counts)
        q3k.kv_keep_path(*bufs, L, cap_b, heads, seq, row, B, 0, bp, n, starts=bs, counts=bc if given_counts else None)
        hip.synchronize()
        for buf, a in zip(bufs, (k, v, s)):
            if buf is None:
                continue
            want = a.copy()
            for b in range(B):
                for i in range(int(counts[b]) if given_counts else n):
                    p, at = int(path[b, i]), int(starts[b])
                    if p >= i and at < seq and at + p < seq:
                        want[:, b, :, at + i] = a[:, b, :, at + p]
            assert np.array_equal(buf.get(np.uint8, a.shape), want) and buf.guards_intact()


def test_keep_path_scalar_start_of_a_long_path(q3k, hip):
    announce("kv_keep_path scalar start")
    k = np.random.default_rng(2).integers(0, 256, (2, 2, 1, 300, 64), dtype=np.uint8)
    bk, bv = Guarded(hip, k), Guarded(hip, k)
    path = np.stack([np.arange(100) * 2, np.arange(100)]).astype(np.int32)
    bp, = _up(hip, path)
    q3k.kv_keep_path(bk, bv, None, 2, 2, 1, 300, 64, 2, 50, bp, 100)
    hip.synchronize()
    want = k.copy()
    want[:, 0, :, 50:150] = k[:, 0, :, 50:250:2]
    for b in (bk, bv):
        assert np.array_equal(b.get(np.uint8, k.shape), want) and b.guards_intact()


def test_keep_path_starts_and_counts_out_of_range(q3k, hip):
    """A start outside the cache or a count below 0 leaves a sequence alone, a count past the path ends with it."""
    announce("kv_keep_path starts and counts out of range")
    B, seq, n = 8, 20, 3
    k = np.random.default_rng(5).integers(0, 256, (2, B, 2, seq, 128), dtype=np.uint8)
    s = np.random.default_rng(6).integers(0, 256, (2, B, 2, seq, 2), dtype=np.uint8)
    starts = np.array([-1, LOWEST, HIGHEST, HIGHEST - 1, 20, 17, 4, 6], np.int32)
    counts = np.array([n, n, n, n, n, n, -1, HIGHEST], np.int32)
    path = np.tile(np.array([2, 3, HIGHEST], np.int32), (B, 1))
    path[7] = [1, 1, 4]
    bk, bv, bs = Guarded(hip, k), Guarded(hip, k), Guarded(hip, s)
    bp, bst, bc = _up(hip, path, starts, counts)
    q3k.kv_keep_path(bk, bv, bs, 2, B, 2, seq, 128, B, 0, bp, n, starts=bst, counts=bc)
    hip.synchronize()
    for bufs, a in (((bk, bv), k), ((bs,), s)):
        want = a.copy()
        want[:, 5, :, 17] = a[:, 5, :, 19]              # row 17 + 3 lies past the cache
        want[:, 7, :, 6], want[:, 7, :, 8] = a[:, 7, :, 7], a[:, 7, :, 10]
        for b in bufs:
            assert np.array_equal(b.get(np.uint8, a.shape), want) and b.guards_intact()


@pytest.mark.parametrize("S", [1, 40])
def test_small_and_large_values(q3k, hip, S):
    """Rows of 2^-60 to 2^60 in one cache: each row's scale is its own."""
    def edit(c):
        powers = np.exp2(np.random.default_rng(8).integers(-60, 61, (c.values[1].shape[0], c.cap, 1, 1)).astype(float))
        rows = c.values[1] * powers                     # V of each row scaled by a power of two: codes stay, bytes move
        finite = np.isfinite(rows)
        c.values[1] = np.where(finite, rows, c.values[1])
        move = np.log2(powers[..., 0, 0]).astype(int)
        for b in range(c.bytes.shape[0]):
            for row in range(c.cap):
                byte = c.bytes[b, :, row, 1].astype(int)
                c.bytes[b, :, row, 1] = np.where(byte < 255, byte + move[b, row], 255)
        c.upload()

    _compare(q3k, hip, f"values of 2^-60 to 2^60 S {S}", True, 2, S, 4, 2, 128, 90, 88, [88, 57], edit=edit)
