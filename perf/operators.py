"""The operators of an 8-bit KV cache and of speculative decoding, as they are measured.

append  bf16 K and V rows quantised as they are written into an e4m3 cache: one power-of-two scale a row (token and
        KV head), the smallest 2^e with max |x| <= 448 * 2^e; codes are [B, KV heads, rows, D], scale bytes [B, KV heads,
        rows, 2] for K and V
read    rows of an e4m3 cache read back as bf16
attend  causal grouped-query attention over an e4m3 cache, sequences of different lengths in one call
tree    attention of a tree of drafted tokens: each node over the context, its ancestors and itself; bf16 or e4m3 cache
keep    the rows of the accepted path moved to the end of the context, in every layer of a cache at once

With ``own`` false a pass is computed in elementary torch operations, with it true by the library's entry points.
Everything is bf16 with head width 128; lengths, parents and paths are int32 tensors on the GPU.
"""
import importlib
import math

import torch

own = False

D = 128
HEADS = [(16, 8), (32, 8), (40, 8), (64, 8)]  # query and KV heads of the model widths; / 8: a tensor-parallel shard


# ---- cases ----------------------------------------------------------------------

def _write(name, kind, B, S, Hkv, cap, ragged):
    """append: S new rows a sequence; read: the first S rows.  ragged: every sequence at a length of its own."""
    return {"name": name, "kind": kind, "B": B, "S": S, "Hkv": Hkv, "cap": cap, "ragged": ragged}


def _attend(name, kind, B, S, cached, Hq, Hkv, cap, ragged, e4m3=True):
    """cached: rows of the longest sequence, its S queries' among them."""
    return {"name": name, "kind": kind, "B": B, "S": S, "cached": cached, "Hq": Hq, "Hkv": Hkv, "cap": cap,
            "ragged": ragged, "e4m3": e4m3}


def _keep(name, layers, B, nodes, kept, Hkv, cap, e4m3):
    return {"name": name, "kind": "keep", "layers": layers, "B": B, "S": nodes, "kept": kept, "Hkv": Hkv, "cap": cap,
            "e4m3": e4m3}


def listed():
    return [
        # one token of each of 64 users, each at a length of its own: what a decode step appends in a layer
        _write("append_decode_64", "append", 64, 1, 8, 1024, True),
        # a prefill batch: bound by memory
        _write("append_prefill_4x2048", "append", 4, 2048, 8, 2048, False),
        # a shard's rows of one prompt of odd length, read back to move it to another engine
        _write("read_1x1001_shard", "read", 1, 1001, 1, 1024, False),
        # every sequence of a batch read back as far as it goes
        _write("read_16x4096", "read", 16, 4096, 8, 4096, True),
        # one user with a long context, and a full serving batch of ragged lengths
        _attend("attend_decode_1x8191", "attend", 1, 1, 8191, 16, 8, 16384, False),
        _attend("attend_decode_64x4096", "attend", 64, 1, 4096, 32, 8, 4096, True),
        # a later chunk of a long prompt
        _attend("attend_chunk_512_at_7680", "attend", 1, 512, 8192, 32, 8, 16384, False),
        # a small drafted tree of one user, bf16 cache
        _attend("tree_26_at_2000", "tree", 1, 26, 2026, 32, 8, 4096, False, False),
        # four drafted tokens (a chain with a branch) for each user of a batch, 8-bit cache
        _attend("tree_5_of_64", "tree", 64, 5, 2053, 32, 8, 2304, True),
        # wide trees for a batch at the width with five query heads a KV head
        _attend("tree_64_of_16", "tree", 16, 64, 4160, 40, 8, 4224, True, False),
        # the accepted tokens of one user, and of a full batch over an 8-bit cache
        _keep("keep_1_of_26", 28, 1, 26, 4, 8, 2100, False),
        _keep("keep_64_of_64", 36, 64, 64, 8, 8, 512, True),
    ]


def _spread(rng, lo, hi):
    """An integer of [lo, hi], spread evenly over the logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "read", "attend", "attend", "attend", "tree", "tree", "tree", "keep"])
    hq, hkv = rng.choice(HEADS)
    if rng.random() < 0.3:
        hq, hkv = hq // 8, hkv // 8
    ragged = rng.random() < 0.5
    e4m3 = rng.random() < 0.5
    if kind in ("append", "read"):
        B = _spread(rng, 1, 64)
        S = _spread(rng, 1, max(1, 16384 // B)) if rng.random() < 0.7 else 1
        case = _write("", kind, B, S, hkv, S + rng.choice([0, 1, 37, 512]), ragged)
    elif kind == "keep":
        B, nodes = _spread(rng, 1, 64), _spread(rng, 4, 64)
        case = _keep("", rng.choice([1, 28, 36]), B, nodes, _spread(rng, 1, max(1, nodes // 4)), hkv,
                     nodes + rng.choice([5, 129, 400]), e4m3)
    elif kind == "attend":
        if rng.random() < 0.6:
            B, S = _spread(rng, 1, 64), 1
            cached = _spread(rng, 1, min(32768, 2 ** 17 // B))
        else:
            B, S = rng.choice([1, 1, 2, 3, 4]), _spread(rng, 2, 512)
            pairs = 1.2e8 // (hq * B)  # (query, key) pairs of one head, to stay below the largest listed case
            cached = min(_spread(rng, S, 8192), max(S, int(pairs // S)))
        case = _attend("", kind, B, S, cached, hq, hkv, cached + rng.choice([0, 1, 37, 512]), ragged)
    else:
        B, S = _spread(rng, 1, 64), _spread(rng, 1, 64)
        S = min(S, max(1, 1024 // B))
        cached = S + _spread(rng, 1, min(16384, 2 ** 15 // B))
        case = _attend("", kind, B, S, cached, hq, hkv, cached + rng.choice([0, 1, 37, 512]), ragged, e4m3)
    del case["name"]
    return case


# ---- inputs -----------------------------------------------------------------------

def _quantise(x):
    """Rows of x (last dimension) as e4m3 codes and scale bytes: 2^(byte - 127) * code."""
    x = x.float()
    part, power = torch.frexp(x.abs().amax(-1, keepdim=True))  # part in [0.5, 1); 448 = 0.875 * 2^9
    e = torch.where(part <= 0.875, power - 9, power - 8).clamp(min=-126)
    codes = torch.ldexp(x, -e).to(torch.float8_e4m3fn)
    return codes, (e.squeeze(-1) + 127).to(torch.uint8)


def _lengths(case, gen):
    """int32 [B]: evenly spaced from a quarter of the longest up to it, in random order."""
    B, S = case["B"], case["S"]
    longest = case["S"] if case["kind"] == "read" else case["cap"] - S if case["kind"] == "append" else case["cached"]
    least = S if case["kind"] == "tree" else min(longest, 1)
    n = torch.linspace(max(least, longest // 4), longest, B, device="cuda", dtype=torch.float64).round()
    return n[torch.randperm(B, generator=gen, device="cuda")].to(torch.int32)


def _parents(case, gen):
    """int32 [B, S]: node 0 the root, a node's parent before it, more often a late one; -2: no node (a smaller tree)."""
    B, T = case["B"], case["S"]
    t = torch.arange(T, device="cuda")
    p = (t * torch.rand((B, T), generator=gen, device="cuda").sqrt()).to(torch.int32).clamp(max=(t - 1).clamp(min=0))
    p[:, 0] = -1
    if case["ragged"]:
        nodes = torch.randint((T + 1) // 2, T + 1, (B, 1), generator=gen, device="cuda")
        p[t[None, :] >= nodes] = -2
    return p.contiguous()


class _State:
    pass


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape: torch.randn(shape, generator=gen, device="cuda", dtype=torch.bfloat16)  # noqa: E731
    s = _State()
    s.case, kind = case, case["kind"]
    B, S, Hkv, cap = case["B"], case["S"], case["Hkv"], case["cap"]
    s.lengths = _lengths(case, gen) if case.get("ragged") else None
    if kind == "keep":
        L, n = case["layers"], case["kept"]
        if case["e4m3"]:
            codes = torch.randint(0, 0x7f, (2, L, B, Hkv, cap, D), generator=gen, device="cuda", dtype=torch.uint8)
            s.kc, s.vc = codes.view(torch.float8_e4m3fn)
            s.scales = torch.randint(100, 140, (L, B, Hkv, cap, 2), generator=gen, device="cuda", dtype=torch.uint8)
        else:
            s.kc, s.vc, s.scales = normal(L, B, cap, Hkv, D), normal(L, B, cap, Hkv, D), None
        s.starts = torch.randint(0, cap - S + 1, (B,), generator=gen, device="cuda", dtype=torch.int32)
        # the root stays where it is; the others come from behind the kept rows, as in a tree numbered by depth
        path = torch.rand((B, S - n), generator=gen, device="cuda").argsort(1)[:, :n].sort(1).values + n
        s.path = path.to(torch.int32)
        s.path[:, 0] = 0
        s.counts = torch.randint((n + 1) // 2, n + 1, (B,), generator=gen, device="cuda", dtype=torch.int32)
        return s
    if kind == "append":
        s.k, s.v = normal(B, S, Hkv, D), normal(B, S, Hkv, D)
        s.kc = torch.zeros((B, Hkv, cap, D), device="cuda", dtype=torch.float8_e4m3fn)
        s.vc = torch.zeros_like(s.kc)
        s.scales = torch.full((B, Hkv, cap, 2), 127, device="cuda", dtype=torch.uint8)
        return s
    if kind != "read":
        s.q = normal(B, S, case["Hq"], D) * 2
        s.parents = _parents(case, gen) if kind == "tree" else None
    if kind == "read" or case["e4m3"]:
        s.kc, ks = _quantise(normal(B, Hkv, cap, D))
        s.vc, vs = _quantise(normal(B, Hkv, cap, D))
        s.scales = torch.stack([ks, vs], -1)
    else:
        s.kc, s.vc, s.scales = normal(B, cap, Hkv, D), normal(B, cap, Hkv, D), None
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "read":
        s.k = torch.zeros((case["B"], case["S"], case["Hkv"], D), device="cuda", dtype=torch.bfloat16)
        s.v = torch.zeros_like(s.k)
    s.ws, s.ws_bytes = None, 0
    if own:  # a program keeps its workspace, its output and its stream's handle
        s.q3k = importlib.import_module("qwen3-runtime-byyourself_amd")
        s.stream = torch.cuda.current_stream().cuda_stream
        if case["kind"] in ("attend", "tree"):
            s.out = torch.empty_like(s.q)
            if s.parents is not None:
                s.parents = s.parents.to(torch.int32)  # as the call takes them
            s.ws_bytes = s.q3k.cache_attention_workspace_bytes(case["B"], case["S"], case["Hq"], case["Hkv"], D,
                                                               case["cached"])
            s.ws = torch.empty(s.ws_bytes, device="cuda", dtype=torch.uint8) if s.ws_bytes else None
        s.ptr = {k: v.data_ptr() for k, v in s.__dict__.items() if isinstance(v, torch.Tensor)}
    return s


# ---- the plain forms ------------------------------------------------------------------

def _dequantise(codes, scale_bytes):
    """float32 values [B, Hkv, rows, D] of codes and their scale bytes [B, Hkv, rows]."""
    return torch.ldexp(codes.float(), scale_bytes.unsqueeze(-1).int() - 127)


def _plain_append(s, c):
    B, S = c["B"], c["S"]
    kc, ks = _quantise(s.k)
    vc, vs = _quantise(s.v)
    start = s.lengths.long() if c["ragged"] else torch.zeros(B, device="cuda", dtype=torch.long)
    rows = start[:, None] + torch.arange(S, device="cuda")
    b = torch.arange(B, device="cuda")[:, None]
    s.kc.view(torch.uint8).transpose(1, 2)[b, rows] = kc.view(torch.uint8)
    s.vc.view(torch.uint8).transpose(1, 2)[b, rows] = vc.view(torch.uint8)
    s.scales.transpose(1, 2)[b, rows] = torch.stack([ks, vs], -1)
    return {"k": s.kc, "v": s.vc, "scales": s.scales.view(torch.float8_e8m0fnu)}


def _plain_read(s, c):
    n = c["S"]
    k = _dequantise(s.kc[:, :, :n], s.scales[:, :, :n, 0]).to(torch.bfloat16).transpose(1, 2)
    v = _dequantise(s.vc[:, :, :n], s.scales[:, :, :n, 1]).to(torch.bfloat16).transpose(1, 2)
    if c["ragged"]:  # the rows behind a sequence stay as they are
        behind = (torch.arange(n, device="cuda") >= s.lengths[:, None])[:, :, None, None]
        k, v = torch.where(behind, s.k, k), torch.where(behind, s.v, v)
    s.k.copy_(k)
    s.v.copy_(v)
    return {"k": s.k, "v": s.v}


def _ancestors(parents):
    """[B, T, T]: whether column u is row t's node itself or one of its ancestors; an empty row where there is no node.
    (1 + A)^T, with A the parent relation, counts the ways up: in float64, where T of 256 still fits."""
    B, T = parents.shape
    t = torch.arange(T, device="cuda")
    up = (parents[:, :, None] == t).double() + torch.eye(T, device="cuda", dtype=torch.float64)
    return (torch.linalg.matrix_power(up, T) > 0) & (parents >= -1)[:, :, None]


def _visible(s, c):
    """[B, S, cached]: the keys that a query attends to."""
    B, S, cached = c["B"], c["S"], c["cached"]
    n = s.lengths.long() if c["ragged"] else torch.full((B,), cached, device="cuda")
    key = torch.arange(cached, device="cuda")
    if c["kind"] == "attend":
        return key <= (n[:, None] - S + torch.arange(S, device="cuda"))[:, :, None]
    node = key - (n[:, None] - S)  # the node of a key, below 0 in the context
    tree = _ancestors(s.parents).gather(2, node.clamp(0, S - 1)[:, None, :].expand(B, S, cached))
    context = (node < 0)[:, None, :] & (s.parents >= -1)[:, :, None]
    return context | (tree & ((node >= 0) & (node < S))[:, None, :])


def _plain_attend(s, c):
    B, S, cached, Hq, Hkv = c["B"], c["S"], c["cached"], c["Hq"], c["Hkv"]
    G = Hq // Hkv
    if c["e4m3"]:
        k = _dequantise(s.kc[:, :, :cached], s.scales[:, :, :cached, 0])
        v = _dequantise(s.vc[:, :, :cached], s.scales[:, :, :cached, 1])
    else:
        k = s.kc[:, :cached].float().transpose(1, 2)
        v = s.vc[:, :cached].float().transpose(1, 2).contiguous()
    k = k.transpose(2, 3).contiguous()                                   # [B, Hkv, D, cached]
    q = s.q.float().view(B, S, Hkv, G, D).permute(0, 2, 1, 3, 4).reshape(B, Hkv, S * G, D)
    scores = torch.matmul(q, k).view(B, Hkv, S, G, cached) / math.sqrt(D)
    seen = _visible(s, c)[:, None, :, None, :]
    scores = torch.where(seen, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, Hkv, S * G, cached), v).view(B, Hkv, S, G, D)
    o = torch.where(total > 0, o / total, 0.0)                           # a row without a key: zeros
    return o.permute(0, 2, 1, 3, 4).reshape(B, S, Hq, D).to(torch.bfloat16)


def _plain_keep(s, c):
    B, n = c["B"], c["kept"]
    i = torch.arange(n, device="cuda")
    keep = i < s.counts[:, None]
    dst = s.starts[:, None].long() + i
    src = torch.where(keep, s.starts[:, None].long() + s.path.long(), dst)
    b = torch.arange(B, device="cuda")[:, None]
    bits = torch.uint8 if c["e4m3"] else torch.bfloat16
    kc, vc = s.kc.view(bits), s.vc.view(bits)
    if c["e4m3"]:
        kc, vc, scales = kc.transpose(2, 3), vc.transpose(2, 3), s.scales.transpose(2, 3)  # [layers, B, rows, Hkv, ..]
        scales[:, b, dst] = scales[:, b, src]
    kc[:, b, dst] = kc[:, b, src]
    vc[:, b, dst] = vc[:, b, src]
    return _kept(s, c)


def _kept(s, c):
    out = {"k": s.kc, "v": s.vc}
    if c["e4m3"]:
        out["scales"] = s.scales.view(torch.float8_e8m0fnu)
    return out


# ---- a pass ---------------------------------------------------------------------------

def _own(s, c):
    q3k, p, st, kind = s.q3k, s.ptr, s.stream, c["kind"]
    B, S, Hkv, cap = c["B"], c["S"], c["Hkv"], c["cap"]
    if kind == "append":
        q3k.kv_append_e4m3(p["k"], p["v"], p["kc"], p["vc"], p["scales"], B, S, Hkv, D, cap, 0, starts=p.get("lengths"),
                           stream=st)
        return {"k": s.kc, "v": s.vc, "scales": s.scales.view(torch.float8_e8m0fnu)}
    if kind == "read":
        q3k.kv_read_e4m3(p["kc"], p["vc"], p["scales"], p["k"], p["v"], B, Hkv, D, cap, 0, S, lengths=p.get("lengths"),
                         stream=st)
        return {"k": s.k, "v": s.v}
    if kind == "keep":
        heads, row = (Hkv, D) if c["e4m3"] else (1, 2 * Hkv * D)
        q3k.kv_keep_path(p["kc"], p["vc"], p.get("scales"), c["layers"], B, heads, cap, row, B, 0, p["path"], c["kept"],
                         starts=p["starts"], counts=p["counts"], stream=st)
        return _kept(s, c)
    cached, Hq = c["cached"], c["Hq"]
    if kind == "attend":
        q3k.gqa_attention_e4m3(p["q"], p["kc"], p["vc"], p["scales"], p["out"], B, S, Hq, Hkv, D, cap, cached,
                               lengths=p.get("lengths"), stream=st, workspace=p.get("ws"), workspace_bytes=s.ws_bytes)
    elif c["e4m3"]:
        q3k.gqa_tree_attention_e4m3(p["q"], p["kc"], p["vc"], p["scales"], p["out"], p["parents"], S, B, S, Hq, Hkv, D, cap,
                                    cached, lengths=p.get("lengths"), stream=st, workspace=p.get("ws"),
                                    workspace_bytes=s.ws_bytes)
    else:
        strides = (cap * Hkv * D, Hkv * D, D, 1)
        q3k.gqa_tree_attention(p["q"], p["kc"], p["vc"], p["out"], p["parents"], S, B, S, Hq, Hkv, D, cached, strides,
                               strides, lengths=p.get("lengths"), stream=st, workspace=p.get("ws"),
                               workspace_bytes=s.ws_bytes)
    return s.out


def run(s):
    c = s.case
    if own:
        return _own(s, c)
    return {"append": _plain_append, "read": _plain_read, "attend": _plain_attend, "tree": _plain_attend,
            "keep": _plain_keep}[c["kind"]](s, c)


# ---- what a pass cannot do without ----------------------------------------------------

def _total(longest, least, B, ragged):
    """The sum of _lengths()."""
    if not ragged:
        return B * longest
    lo = max(least, longest // 4)
    return sum(round(lo + (longest - lo) * i / max(1, B - 1)) for i in range(B))


def work(case):
    kind, B, S, Hkv = case["kind"], case["B"], case["S"], case["Hkv"]
    if kind == "append":
        return {"bytes": 2 * B * S * Hkv * (2 * D + D + 1) + (4 * B if case["ragged"] else 0), "flops": 0}
    if kind == "read":
        rows = _total(S, min(S, 1), B, case["ragged"])
        return {"bytes": 2 * rows * Hkv * (D + 1 + 2 * D) + (4 * B if case["ragged"] else 0), "flops": 0}
    if kind == "keep":
        row = Hkv * (D + 1 if case["e4m3"] else 2 * D)
        rows = B * ((case["kept"] + 1) // 2 + case["kept"]) // 2
        return {"bytes": 2 * 2 * case["layers"] * rows * row + 4 * B * (case["kept"] + 2), "flops": 0}
    Hq = case["Hq"]
    keys = _total(case["cached"], S if kind == "tree" else min(case["cached"], 1), B, case["ragged"])
    # (query, key) pairs: the context, and of the S rows the causal half; a tree's own part is smaller
    pairs = max(0, keys - B * S) * S + B * S * (S + 1) // 2 if kind == "attend" else (keys - B * S) * S + B * S
    row = D + 1 if case["e4m3"] else 2 * D
    total = 2 * keys * Hkv * row + 2 * 2 * B * S * Hq * D + (4 * B * S if kind == "tree" else 0)
    return {"bytes": total + (4 * B if case["ragged"] else 0), "flops": 4 * D * Hq * pairs}


# ---- the same in 64 bits, each step from the definition ---------------------------------

def _scale64(x):
    """2^e of rows x, from comparisons with 448 * 2^e alone."""
    top = x.abs().amax(-1)
    e = torch.floor(torch.log2(torch.where(top > 0, top, 1.0) / 448.0)) - 1
    for _ in range(3):
        e = torch.where(top > 448.0 * torch.exp2(e), e + 1, e)
    return torch.exp2(torch.where(top > 0, e, -126.0).clamp(min=-126.0))


def _values64(s, b, h, n, which):
    x = (s.kc, s.vc)[which][b]
    if s.scales is None:
        return x[:n, h].double()
    return x[h, :n].double() * torch.exp2(s.scales[b, h, :n, which].double() - 127.0).unsqueeze(-1)


def _chain(parents):
    """The rows of one tree's ancestors, by walking up from each node."""
    p = parents.tolist()
    seen = torch.zeros((len(p), len(p)), dtype=torch.bool)
    for t in range(len(p)):
        u = t if p[t] >= -1 else -1
        while u >= 0:
            seen[t, u] = True
            u = p[u]
    return seen.to("cuda")


def exact(case, seed):
    s = _inputs(case, seed)
    kind, B, S, Hkv, cap = case["kind"], case["B"], case["S"], case["Hkv"], case["cap"]
    n = s.lengths.tolist() if s.lengths is not None else [0 if kind == "append" else S if kind == "read" else
                                                          case.get("cached", 0)] * B
    if kind == "append":
        out = {"k": s.kc.double(), "v": s.vc.double(), "scales": torch.ones((B, Hkv, cap, 2), device="cuda", dtype=torch.float64)}
        for i, (name, x) in enumerate((("k", s.k.double()), ("v", s.v.double()))):
            scale = _scale64(x)
            for b in range(B):
                out[name][b, :, n[b]:n[b] + S] = (x[b] / scale[b].unsqueeze(-1)).transpose(0, 1)
                out["scales"][b, :, n[b]:n[b] + S, i] = scale[b].t()
        return out
    if kind == "read":
        out = {"k": torch.zeros((B, S, Hkv, D), device="cuda", dtype=torch.float64)}
        out["v"] = torch.zeros_like(out["k"])
        for b in range(B):
            for h in range(Hkv):
                out["k"][b, :n[b], h] = _values64(s, b, h, n[b], 0)
                out["v"][b, :n[b], h] = _values64(s, b, h, n[b], 1)
        return out
    if kind == "keep":
        start, path, counts = s.starts.tolist(), s.path.tolist(), s.counts.tolist()
        for b in range(B):
            for i in range(counts[b]):
                to, at = start[b] + i, start[b] + path[b][i]
                for x in (s.kc, s.vc, s.scales) if case["e4m3"] else (s.kc, s.vc):
                    rows = x[:, b].transpose(1, 2) if case["e4m3"] else x[:, b]
                    rows[:, to] = rows[:, at].clone()
        out = {"k": s.kc.double(), "v": s.vc.double()}
        if case["e4m3"]:
            out["scales"] = torch.exp2(s.scales.double() - 127.0)
        return out
    Hq = case["Hq"]
    G = Hq // Hkv
    out = torch.zeros((B, S, Hq, D), device="cuda", dtype=torch.float64)
    for b in range(B):
        if kind == "tree":
            seen = torch.zeros((S, n[b]), device="cuda", dtype=torch.bool)
            seen[:, n[b] - S:] = _chain(s.parents[b])
            seen[:, :n[b] - S] = (s.parents[b] >= -1)[:, None]
        else:
            seen = torch.ones((S, n[b]), device="cuda", dtype=torch.bool).tril(n[b] - S)
        some = seen.any(1)
        for h in range(Hkv):
            k, v = _values64(s, b, h, n[b], 0), _values64(s, b, h, n[b], 1)
            q = s.q[b, :, h * G:(h + 1) * G].double().transpose(0, 1).reshape(G * S, D)
            scores = (q @ k.t().contiguous()).view(G, S, n[b]) / math.sqrt(D)
            p = torch.softmax(scores.masked_fill(~seen, -math.inf), -1)
            p = torch.where(some[:, None], p, 0.0)
            out[b, :, h * G:(h + 1) * G] = (p.view(G * S, -1) @ v).view(G, S, D).transpose(0, 1)
    return out
