"""Calls that between them take every form of the attention over a cache (tests/test_cache_forms_cpu.py holds the plans to
that): the decode kernel in blocks of 1, 4 and 8 waves, the block kernel in its two shapes over several tiles and query
blocks, whole and in slices, both merges, each mask and cache.  And their plain 64-bit form, of matrix products."""
import numpy as np

import cache_ref as ref

# mask and cache, B, S, Hq, Hkv, cached, whether the lengths differ, and the form taken with and without a workspace:
# "w" waves of a decode block or "g" key groups of the block kernel, "/" the slices, "r" those that 16 lanes a row merge
FORMS = [
    ("causal", 1, 1, 4, 1, 30, False, "w1", "w1"),
    ("causal", 1, 1, 4, 1, 260, False, "w4", "w4"),
    ("causal", 1, 2, 4, 1, 450, False, "w4/4", "w8"),
    ("causal", 12, 5, 40, 8, 700, True, "w4/3r", "w8"),
    ("causal", 12, 1, 32, 8, 1200, True, "w8/3", "w8"),
    ("causal", 12, 5, 40, 8, 1000, False, "w8/2r", "w8"),
    ("causal", 1, 17, 5, 1, 450, False, "g4/4", "g4"),
    ("causal", 1, 130, 16, 4, 450, True, "g4/4r", "g4"),
    ("causal", 12, 40, 40, 8, 330, False, "g1", "g1"),
    ("causal", 1, 26, 40, 8, 12000, False, "g1/32", "g4"),
    ("causal", 12, 41, 32, 8, 700, True, "g1/3r", "g4"),
    ("causal", 2, 300, 32, 8, 3001, False, "g1/3r", "g1"),
    ("tree", 1, 3, 4, 1, 30, False, "w1", "w1"),
    ("tree", 1, 3, 4, 1, 260, False, "w4", "w4"),
    ("tree", 1, 2, 4, 1, 450, False, "w4/4", "w8"),
    ("tree", 12, 5, 40, 8, 700, True, "w4/3r", "w8"),
    ("tree", 12, 1, 32, 8, 1200, True, "w8/3", "w8"),
    ("tree", 12, 5, 40, 8, 1000, False, "w8/2r", "w8"),
    ("tree", 1, 17, 5, 1, 450, False, "g4/4", "g4"),
    ("tree", 2, 255, 16, 8, 1200, False, "g4/2r", "g4"),
    ("tree", 12, 40, 40, 8, 330, False, "g1", "g1"),
    ("tree", 1, 26, 40, 8, 12000, False, "g1/32", "g4"),
    ("tree", 12, 41, 32, 8, 700, True, "g1/3r", "g4"),
    ("tree", 4, 201, 16, 4, 3001, True, "g1/4r", "g4"),
    ("tree-bf16", 1, 3, 4, 1, 30, False, "w1", "w1"),
    ("tree-bf16", 1, 3, 4, 1, 260, False, "w4", "w4"),
    ("tree-bf16", 1, 2, 4, 1, 450, False, "w4/5", "w4"),
    ("tree-bf16", 12, 5, 40, 8, 700, False, "w4/2r", "w4"),
    ("tree-bf16", 1, 17, 5, 1, 450, False, "g4/4", "g4"),
    ("tree-bf16", 1, 130, 16, 4, 450, True, "g4/4r", "g4"),
    ("tree-bf16", 12, 40, 40, 8, 330, False, "g1", "g1"),
    ("tree-bf16", 1, 26, 40, 8, 12000, False, "g1/32", "g4"),
    ("tree-bf16", 12, 41, 32, 8, 700, True, "g1/3r", "g4"),
    ("tree-bf16", 16, 64, 40, 8, 1500, True, "g1", "g1"),
]


def lengths_of(B, S, cached, ragged):
    """None, or lengths from the longest down to the queries' own rows, the second longer sequence's among the tiles' ends."""
    if not ragged:
        return None
    n = np.linspace(cached, S, B).round().astype(int)
    if B > 2:
        n[1] = cached // 64 * 64
    return np.random.default_rng(B + S).permutation(n).astype(np.int32)


def attention(q, k, v, n, S, parents=None):
    """cache_ref.attention of one sequence as a few matrix products: q [S, Hq, D], k and v [n, Hkv, D] float64 -> (out,
    bound), by its formulas.  Infinities and NaN of v reach the queries that see their rows, and no others."""
    Hq, D = q.shape[1:]
    Hkv = k.shape[1]
    G = Hq // Hkv
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    seen = np.arange(n)[None, :] <= n - S + np.arange(S)[:, None]
    bad = np.zeros(S, bool)
    if parents is not None:
        states, tree = ref.ancestors(parents)
        seen = np.zeros((S, n), bool)
        seen[:, :n - S] = True
        seen[:, n - S:] = tree
        seen[[s != "sees" for s in states]] = False
        bad = np.array([s == "bad" for s in states])
    rows, some = seen.sum(1), seen.any(1)
    mask = np.repeat(seen, G, 0)                                  # [(s, g), n]
    for h in range(Hkv):
        qh = q[:, h * G:(h + 1) * G].reshape(S * G, D)
        kh, vh = k[:, h], v[:, h]
        wild = ~np.isfinite(vh)
        finite = np.where(wild, 0.0, vh)
        with np.errstate(invalid="ignore", over="ignore"):
            score = np.where(mask, qh @ kh.T / np.sqrt(D), -np.inf)
            most = np.where(mask, np.abs(qh) @ np.abs(kh).T, 0.0).max(1) / np.sqrt(D)
            top = score.max(1, keepdims=True)
            p = np.exp(score - np.where(top == -np.inf, 0.0, top))
            total = p.sum(1, keepdims=True)
            p = np.where(total == 0, 0.0, p / np.where(total == 0, 1.0, total))
            o = p @ finite
            for j in np.flatnonzero(wild.any(1)):
                o[mask[:, j]] += np.where(wild[j], vh[j], 0.0)
            rel = 2 * (D + 8) * 2.0**-24 * most + 2.0**-16 + 2.0**-21 + (np.repeat(rows, G) + 64) * 2.0**-24
            e = rel[:, None] * (p @ np.abs(finite))
        o[~np.repeat(some, G)] = 0.0
        out[:, h * G:(h + 1) * G] = o.reshape(S, G, D)
        bound[:, h * G:(h + 1) * G] = np.where(np.isfinite(e), e, 0.0).reshape(S, G, D)
    out[bad] = np.nan
    return out, bound
