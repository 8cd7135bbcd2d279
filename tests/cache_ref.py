"""Plain 64-bit forms of the e4m3 KV cache, of attention over a cache with a length for each sequence and of trees of
drafted tokens, in numpy: what the GPU tests of these operators compare with."""
import numpy as np

NAN_CODE = 0x7F


def _code_values():
    c = np.arange(256)
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e > 0, (1 + m / 8.0) * np.exp2(e - 7.0), m / 8.0 * np.exp2(-6.0))
    v = np.where((c & 127) == 127, np.nan, v)
    return np.where(c >= 128, -v, v)


CODE = _code_values()
_STEPS = CODE[:127]                     # the non-negative values in order; the index is the code
_MIDDLES = (_STEPS[1:] + _STEPS[:-1]) / 2


def bf16(x):
    return (np.asarray(x, np.uint16).astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def encode(x):
    """RNE of float64 values of at most 448 in magnitude to e4m3 codes (ties to the even code); NaN for the others."""
    a = np.abs(x)
    below = np.searchsorted(_MIDDLES, a, side="left")      # a tie with a middle stays below it
    tie = (below < 126) & (a == _MIDDLES[np.minimum(below, 125)])
    code = np.where(tie & (below % 2 == 1), below + 1, below)
    code = np.where(np.isfinite(x), code, NAN_CODE)
    return (code | np.where(np.signbit(x) & np.isfinite(x), 128, 0)).astype(np.uint8)


def quantise(bits):
    """bf16 patterns [..., D] -> (codes, scale bytes [...]): the smallest 2^e, e >= -126, with max finite |x| <= 448 * 2^e."""
    x = bf16(bits)
    top = np.where(np.isfinite(x), np.abs(x), 0.0).max(-1)
    e = np.full(top.shape, -126)
    for p in range(-126, 121):
        e = np.where(top > 448.0 * np.exp2(float(p)), p + 1, e)
    return encode(x / np.exp2(e[..., None].astype(np.float64))), (e + 127).astype(np.uint8)


def dequantise(codes, byte):
    return CODE[codes] * np.exp2(byte[..., None].astype(np.float64) - 127.0)


def same_codes(a, b):
    """Equal codes; any NaN code equals any other."""
    nan_a, nan_b = (a & 127) == 127, (b & 127) == 127
    return np.array_equal(nan_a, nan_b) and np.array_equal(np.where(nan_a, 0, a), np.where(nan_b, 0, b))


def ancestors(parents):
    """(states, [T, T]): state 'sees', 'empty' or 'bad' of each node, and whether column u is row t or one of its ancestors."""
    T = len(parents)
    states, seen = [], np.zeros((T, T), bool)
    for t in range(T):
        u, state = t, "sees"
        while True:
            p = int(parents[u])
            if p == -2 or p < -2 or p >= u:
                state = "empty" if p == -2 else "bad"
                break
            seen[t, u] = True
            if p == -1:
                break
            u = p
        states.append(state)
    return states, seen


def attention(q, k, v, n, S, parents=None):
    """One sequence: q [S, Hq, D], k and v [n, Hkv, D] float64 -> (out [S, Hq, D], bound [S, Hq, D]).

    bound is what the kernels' arithmetic may be off by before the output's rounding: scores are fp32 sums of D
    products (D + 8 roundings, each 2^-24 of at most the sum of magnitudes), so a weight is off by twice that, by 2^-16
    from its two bf16 parts and by 2^-21 from the exponential; sums over n keys add n * 2^-24; all of it times the sum of
    p |v|."""
    Hq, D = q.shape[1:]
    G = Hq // k.shape[1]
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    if parents is not None:
        states, seen = ancestors(parents)
    for s in range(S):
        if parents is None:
            rows = np.arange(max(0, n - S + s + 1))
        elif states[s] == "bad":
            out[s] = np.nan
            continue
        elif states[s] == "empty" or n == 0:
            continue
        else:
            rows = np.concatenate([np.arange(n - S), n - S + np.flatnonzero(seen[s])])
        if len(rows) == 0:
            continue
        for h in range(Hq):
            kk, vv = k[rows, h // G], v[rows, h // G]
            with np.errstate(invalid="ignore", over="ignore"):
                score = kk @ q[s, h] / np.sqrt(D)
                most = (np.abs(kk) @ np.abs(q[s, h])).max() / np.sqrt(D)
                p = np.exp(score - score.max())
                p /= p.sum()
                out[s, h] = p @ vv
                rel = 2 * (D + 8) * 2.0**-24 * most + 2.0**-16 + 2.0**-21 + (len(rows) + 64) * 2.0**-24
                bound[s, h] = rel * (p @ np.abs(vv))
    return out, bound


def check_attention(name, got_bits, out, bound):
    """got (bf16 patterns) within half a bf16 step (2^-8 of the value) and the arithmetic's bound of out."""
    got = bf16(got_bits).reshape(out.shape)
    nan = np.isnan(out)
    assert np.array_equal(np.isnan(got), nan), f"{name}: NaN at {np.argwhere(np.isnan(got) != nan)[:5].tolist()}"
    with np.errstate(invalid="ignore"):
        off = np.abs(got - out)
        most = 2.0**-8 * np.abs(out) + 1.01 * bound + 2.0**-133
        same = got == out          # infinities
        wrong = ~nan & ~same & ~(off <= most)
    assert not wrong.any(), (f"{name}: {int(wrong.sum())} of {wrong.size} outside; first at {np.argwhere(wrong)[0].tolist()}: "
                             f"got {got[wrong][0]} want {out[wrong][0]} +- {most[wrong][0]}")
