"""The calls of cache_forms take the forms that they name, and between them every form there is; and their plain form agrees
with cache_ref's."""
import os
import subprocess

import numpy as np

import cache_forms
import cache_ref as ref
from test_cpp import BIN


def _forms(calls):
    """"w4/3r" and the like of calls (mask and cache, B, S, Hq, Hkv, cached, ragged, can_split)."""
    lines = "".join(f"{B} {S} {Hq} {Hkv} {cached} {int(kind != 'tree-bf16')} {int(kind != 'causal')} {int(ragged)} {int(split)}\n"
                    for kind, B, S, Hq, Hkv, cached, ragged, split in calls)
    done = subprocess.run([os.path.join(BIN, "cache_plan_forms")], input=lines, capture_output=True, text=True, timeout=60, check=True)
    out = []
    for line in done.stdout.splitlines():
        waves, groups, splits, by_rows = map(int, line.split())
        out.append((f"w{waves}" if waves else f"g{groups}") + (f"/{splits}" + "r" * by_rows if splits > 1 else ""))
    return out


def test_calls_take_their_forms():
    for split in (True, False):
        got = _forms([c[:7] + (split,) for c in cache_forms.FORMS])
        assert [(c[:7], f) for c, f in zip(cache_forms.FORMS, got)] == [(c[:7], c[7 if split else 8]) for c in cache_forms.FORMS]


def test_calls_cover_every_form():
    """Each kernel of each mask and cache, whole, in slices merged by a block a row and by 16 lanes a row, where a plan
    takes it so at all; of the block kernels over three tiles or more, with a full query block and a lighter one."""
    kinds = {c[0] for c in cache_forms.FORMS}
    assert kinds == {"causal", "tree", "tree-bf16"}
    for kind in kinds:
        taken = set()
        for _, B, S, Hq, Hkv, cached, _, with_ws, without in (c for c in cache_forms.FORMS if c[0] == kind):
            for f in (with_ws, without):
                taken.add(f.split("/")[0] + ("" if "/" not in f else "/r" if f.endswith("r") else "/"))
                if f[0] == "g":
                    cols, block = S * (Hq // Hkv), 128 if f[1] == "1" else 64
                    assert cached > 3 * 64 and cols > block and cols % block != 0
        want = {"w1", "w4", "w4/", "w4/r", "g1", "g1/", "g1/r", "g4", "g4/", "g4/r"} | ({"w8", "w8/", "w8/r"} if kind != "tree-bf16" else set())
        assert taken == want


def test_no_plan_takes_another_form():
    """Over a sweep of shapes there is no form that the calls above leave out."""
    calls = [(kind, B, S, Hq, Hkv, cached, ragged, split)
             for kind in ("causal", "tree", "tree-bf16") for B in (1, 2, 4, 12, 33, 100) for S in (1, 2, 5, 16, 24, 33, 64, 129, 256)
             for Hq, Hkv in ((4, 1), (8, 2), (5, 1), (32, 8), (40, 8), (16, 8), (32, 1))
             for cached in (20, 33, 65, 130, 260, 700, 2000, 9000, 33000) if cached >= S
             for ragged in (False, True) for split in (False, True)]
    covered = {(c[0], f.split("/")[0], "/" in f, f.endswith("r")) for c in cache_forms.FORMS for f in c[7:]}
    for call, f in zip(calls, _forms(calls)):
        assert (call[0], f.split("/")[0], "/" in f, f.endswith("r")) in covered, (call, f)


def test_plain_form_agrees_with_the_other():
    rng = np.random.default_rng(3)
    q, k, v = rng.standard_normal((7, 6, 16)), rng.standard_normal((19, 2, 16)), rng.standard_normal((19, 2, 16))
    v[4, 1, 3], v[15, 0, 2], v[16, 0, 2], k[17, 1, 5] = np.nan, np.inf, -np.inf, np.nan
    for n, parents in ((19, None), (4, None), (19, [-1, 0, 0, 1, -2, 4, 2]), (19, [-1, 0, 7, 2, 0, -5, 1]), (7, [-1, 0, 1, 2, 3, 4, 5])):
        want, most = ref.attention(q, k[:n], v[:n], n, 7, parents)
        got, bound = cache_forms.attention(q, k[:n], v[:n], n, 7, parents)
        assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(got[np.isinf(want)], want[np.isinf(want)])
        some = np.isfinite(want) & np.isfinite(most)
        assert some.sum() > 100 and np.abs(got - want)[some].max() < 1e-13 and np.abs(bound - most)[some].max() < 1e-13


def test_workspace_query_of_calls_that_never_split(q3k):
    """The generic kernel takes more than 32 query heads a KV head, other widths and lengths whose tiles' ends pass 2^31;
    it cuts no keys, so its calls need no workspace."""
    ws = q3k.cache_attention_workspace_bytes
    assert ws(1, 1, 32, 1, 128, 8192) > 0
    for args in ((1, 1, 33, 1, 128, 8192), (1, 1, 40, 1, 128, 8192), (2, 30, 128, 2, 128, 5000), (1, 1, 32, 1, 96, 8192),
                 (1, 1, 32, 1, 128, 2**31 - 1)):
        assert ws(*args) == 0
