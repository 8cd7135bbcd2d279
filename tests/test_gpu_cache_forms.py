"""Every form of the attention over a cache (cache_forms) against the plain 64-bit form, at several tiles, query blocks and
slices: finite values, and NaN in rows past the first tile that some queries see and others do not."""
import numpy as np
import pytest

import cache_forms
import cache_ref as ref
from gpu_util import announce
from test_gpu_cache_ops import _Cache, _queries, _random_trees, _run, _up, _workspace

pytestmark = pytest.mark.gpu
D = 128


def _id(c):
    return f"{c[0]}-{c[1]}x{c[2]}-{c[3]}.{c[4]}-{c[5]}{'r' if c[6] else ''}-{c[7].replace('/', 's')}"


class _CodesCache(_Cache):
    """An e4m3 cache of codes drawn as such (a normal distribution's), scale bytes of 2^-8 to 2^-6: about 1 in size."""

    def __init__(self, hip, rng, B, Hkv, cap, lengths):
        self.e4m3, self.cap, self.hip = True, cap, hip
        pool = ref.encode(np.clip(rng.standard_normal(1 << 16) * 100, -448, 448))
        past = (np.arange(cap)[None, :] >= np.asarray(lengths)[:, None])
        self.bytes = rng.integers(119, 122, (B, Hkv, cap, 2), dtype=np.uint8)
        self.values, self.stored = [], []
        for i in range(2):
            codes = pool[rng.integers(0, 1 << 16, (B, Hkv, cap, D), dtype=np.uint16)]
            self.values.append(ref.dequantise(codes, self.bytes[..., i]).transpose(0, 2, 1, 3))
            codes.transpose(0, 2, 1, 3)[past] = 0x7F
            self.stored.append(codes)
        self.bytes.transpose(0, 2, 1, 3)[past] = 255
        self.upload()


class _Call:
    """One of cache_forms.FORMS with its inputs; rows of the cache past a sequence's length hold NaN."""

    def __init__(self, hip, form, seed=0, edit=None, lengths=None):
        self.hip = hip
        kind, self.B, self.S, self.Hq, self.Hkv, self.cached, ragged = form[:7]
        B, S = self.B, self.S
        rng = np.random.default_rng(seed + B + 31 * S + self.cached)
        self.lengths = lengths if lengths is not None else cache_forms.lengths_of(B, S, self.cached, ragged)
        given = np.full(B, self.cached) if self.lengths is None else np.asarray(self.lengths)
        self.bad = (given < 0) | (given > self.cached) | ((given > 0) & (given < S) & (kind != "causal"))
        self.n = np.where(self.bad, 0, given)
        if kind == "tree-bf16":
            self.cache = _Cache(hip, rng, False, B, self.Hkv, D, self.cached + 3, self.n)
        else:
            self.cache = _CodesCache(hip, rng, B, self.Hkv, self.cached + 3, self.n)
        self.trees = _random_trees(rng, B, S) if kind != "causal" else None
        self.q = _queries(rng, B, S, self.Hq, D)
        if edit is not None:
            edit(self)
        self.bq, = _up(hip, self.q)
        self.bl = _up(hip, np.asarray(self.lengths, np.int32))[0] if self.lengths is not None else None
        self.bp = (_up(hip, self.trees)[0], S) if self.trees is not None else None

    def shape(self):
        return self.B, self.S, self.Hq, self.Hkv, D, self.cached

    def run(self, q3k, ws):
        out = _run(q3k, self.hip, self.cache, self.bq, self.B, self.S, self.Hq, self.Hkv, D, self.cached, self.bl, self.bp, ws)
        self.hip.synchronize()
        assert out.guards_intact() and (ws is None or ws[0].guards_intact())
        return out.get(np.uint16, self.q.shape)

    def want(self):
        x = ref.bf16(self.q).reshape(self.q.shape)
        k, v = self.cache.values
        out, bound = np.zeros(x.shape), np.zeros(x.shape)
        out[self.bad] = np.nan
        for b, n in enumerate(self.n):
            if n > 0:
                tree = None if self.trees is None else self.trees[b]
                out[b], bound[b] = cache_forms.attention(x[b], k[b, :n], v[b, :n], int(n), self.S, tree)
        return out, bound


def _check(q3k, hip, name, form, **kw):
    announce(f"{name} {_id(form)}")
    call = _Call(hip, form, **kw)
    want = call.want()
    ws = _workspace(q3k, hip, *call.shape())
    for w in (None, ws) if ws is not None else (None,):
        got = call.run(q3k, w)
        ref.check_attention(f"{name} {_id(form)} workspace {w is not None}", got, *want)
        assert np.array_equal(call.run(q3k, w), got), "a second call gives other bits"


@pytest.mark.parametrize("form", cache_forms.FORMS, ids=_id)
def test_form(q3k, hip, form):
    _check(q3k, hip, "form", form)


@pytest.mark.parametrize("form", [c for c in cache_forms.FORMS if c[2] > 1], ids=_id)
def test_form_with_nan_rows(q3k, hip, form):
    """K and V of a query's own row are NaN in half the sequences, in another tile in each (the lengths differ, or the
    row): what does not see it is as if it were finite.  Of every third sequence a row of the context, which all see."""
    def edit(call):
        for b in range(0, call.B, 2):
            call.cache.poison(b, int(call.n[b]) - call.S + (b + call.S // 2) % call.S)
        for b in range(1, call.B, 3):
            if call.n[b] > call.S + 70:
                call.cache.poison(b, int(call.n[b]) - call.S - 1)

    _check(q3k, hip, "NaN rows", form, seed=1, edit=edit)


@pytest.mark.parametrize("form", [c for c in cache_forms.FORMS if c[0] == "tree-bf16"] + [
    ("tree-bf16", 3, 1, 8, 2, 200, True, "w4", "w4"), ("tree-bf16", 1, 1, 4, 1, 1, False, "w1", "w1"),
    ("tree-bf16", 2, 40, 40, 1, 300, True, "generic", "generic")], ids=_id)
def test_infinite_values(q3k, hip, form):
    """Infinities of V in rows of the context, in the first and in later tiles, and of nodes: who sees the row gets the
    infinity in that dim (NaN where two signs meet), and finite values in all others."""
    def edit(call):
        bits, values = call.cache.stored[1], call.cache.values[1]
        for b in range(call.B):
            n = int(call.n[b])
            for i, row in enumerate(sorted({0, n // 3, n - call.S - 1, n - call.S, n - 1 - call.S // 2, n - 1} & set(range(n)))):
                for dim, sign in (((29 * i + 3 * b) % D, 1), ((29 * i + 64 + b) % D, -1), (127, 1 if row % 2 else -1)):
                    bits[b, row, :, dim] = 0x7F80 if sign > 0 else 0xFF80
                    values[b, row, :, dim] = sign * np.inf
        call.cache.upload()

    _check(q3k, hip, "infinite V", form, seed=2, edit=edit)


@pytest.mark.parametrize("form", [c for c in cache_forms.FORMS if c[6] and c[1] >= 12], ids=_id)
def test_form_with_odd_lengths(q3k, hip, form):
    """No rows, one, fewer than the queries (before whose first row some see nothing), below 0, past the cache's."""
    kind, B, S, cached = form[0], form[1], form[2], form[5]
    lengths = cache_forms.lengths_of(B, S, cached, True)
    lengths[:8] = [0, 1, -1, cached + 1, S // 2, S, cached - 1, -2**31]
    _check(q3k, hip, f"odd lengths {kind}", form, seed=5, lengths=lengths)


@pytest.mark.parametrize("kind", ["causal", "tree", "tree-bf16"])
@pytest.mark.parametrize("S", [1, 5, 40])
def test_one_long_sequence_among_short_ones(q3k, hip, kind, S):
    lengths = np.full(40, S + 19, np.int32)
    lengths[::3] = S + 50
    lengths[23] = 9001
    _check(q3k, hip, "one long", (kind, 40, S, 8, 2, 9001, True, "", ""), seed=6, lengths=lengths)


def test_whole_prompt(q3k, hip):
    """Thousands of queries: every causal query block of a long prompt, the first of which sees one tile."""
    _check(q3k, hip, "prompt", ("causal", 1, 4099, 8, 2, 4099, False, "", ""), seed=7)


def _scale_v(call, power):
    """V times 2^power: the scale bytes, or the exponents."""
    c = call.cache
    if c.e4m3:
        c.bytes[..., 1] = np.where(c.bytes[..., 1] < 255, c.bytes[..., 1].astype(int) + power, 255)
        v = ref.dequantise(c.stored[1], c.bytes[..., 1]).transpose(0, 2, 1, 3)
    else:
        bits = c.stored[1]
        bits[:] = np.where((bits & 0x7FFF) > 0x7F80, bits, bits.astype(int) + power * 128)
        v = ref.bf16(bits)
    c.values[1] = np.where(np.isnan(v), 0.0, v)
    c.upload()


GENERIC = [(kind, 2, 3, 40, 1, 300, True, "generic", "generic") for kind in ("causal", "tree-bf16")]


@pytest.mark.parametrize("form", [c for c in cache_forms.FORMS if c[5] <= 1500] + GENERIC, ids=_id)
def test_largest_values(q3k, hip, form):
    """V up to 2^119 over the number of rows, the least that overflows no sum of weights of up to 2^8, and of one sign in
    half the dims."""
    def edit(call):
        c = call.cache
        if c.e4m3:
            c.stored[1][..., :64] &= 0x7F
            _scale_v(call, int(np.floor(119 - np.log2(call.cached))) - 9 + 127 - 121)      # codes of up to 448 * 2^(121 - 127)
        else:
            c.stored[1][..., :64] &= 0x7FFF
            _scale_v(call, int(np.floor(119 - np.log2(call.cached))) - 3)
        most = np.abs(c.values[1]).max() * call.cached
        assert 2.0**115 < most <= 2.0**119

    _check(q3k, hip, "largest V", form, seed=3, edit=edit)


@pytest.mark.parametrize("form", [c for c in cache_forms.FORMS if c[5] <= 1500] + GENERIC, ids=_id)
def test_small_values(q3k, hip, form):
    """V of rows whose largest value is about 2^-83: as exact as any other.  (Weights of 2^-16 of the largest and more have
    their 16 bits there; what smaller ones lose, 2^-117 a row at most, is below 2^-20 of the result.)"""
    _check(q3k, hip, "small V", form, seed=4, edit=lambda call: _scale_v(call, -84))


@pytest.mark.parametrize("what", ["V", "Q"])
@pytest.mark.parametrize("S", [1, 5, 40])
def test_nan_everywhere(q3k, hip, S, what):
    """V, or the queries, NaN as a whole, and empty nodes that stay zeros."""
    def edit(call):
        if what == "Q":
            call.q[:] = 0x7FC0
            return
        for b in range(call.B):
            call.cache.stored[1][b, :call.n[b]] = 0x7FC0
        call.cache.values[1][:] = np.nan
        call.cache.upload()

    _check(q3k, hip, f"NaN {what}", ("tree-bf16", 2, S, 8, 2, 1500, False, "", ""), seed=8, edit=edit)
