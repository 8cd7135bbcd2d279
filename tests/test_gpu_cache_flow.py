"""The 8-bit KV cache and the speculative operators run together, as a serving loop does: ragged decode steps captured in
a graph and replayed while the lengths grow on the device, a speculative step on a stream of its own, two graphs that share
a workspace, two calls at once, and caches past 4 GiB."""
import numpy as np
import pytest

import cache_ref as ref
from gpu_util import Guarded, announce

pytestmark = pytest.mark.gpu
D = 128


def _normal(rng, *shape, std=1.0):
    x = (rng.standard_normal(shape) * std).astype(np.float32)
    return (x.view(np.uint32) >> 16).astype(np.uint16)


class _Serving:
    """An empty e4m3 cache layer of B sequences and the values it should hold, kept by the test itself."""

    def __init__(self, hip, B, Hkv, cap, lengths):
        self.B, self.Hkv, self.cap = B, Hkv, cap
        self.kc, self.vc = (hip.DeviceBuffer(B * Hkv * cap * D) for _ in range(2))
        self.sc = hip.DeviceBuffer(B * Hkv * cap * 2)
        for b in (self.kc, self.vc, self.sc):
            b.fill_bytes(0xFF)                      # NaN codes, bytes that are never written
        self.k, self.v = (np.full((B, cap, Hkv, D), np.nan) for _ in range(2))
        self.lengths = np.array(lengths, np.int32)  # rows held

    def note(self, starts, k, v):
        """k, v [B, S, Hkv, D] bf16 patterns went to rows starts[b] .."""
        for dst, x in ((self.k, k), (self.v, v)):
            values = ref.dequantise(*ref.quantise(x))
            for b in range(self.B):
                dst[b, starts[b]:starts[b] + x.shape[1]] = values[b]

    def want(self, q, lengths, S, parents=None):
        outs = [ref.attention(ref.bf16(q[b]).reshape(S, -1, D), self.k[b, :n], self.v[b, :n], int(n), S,
                              None if parents is None else parents[b]) for b, n in enumerate(lengths)]
        return np.stack([o[0] for o in outs]), np.stack([o[1] for o in outs])


def test_ragged_decode_replayed_while_the_lengths_grow(q3k, hip):
    """A decode step (append at each sequence's length, attention over it) captured once; before each replay the host sets
    new K, V, Q and lengths.  Every replay equals the eager calls bit for bit and the 64-bit form within its bound."""
    announce("ragged decode from a graph")
    B, Hq, Hkv, cap = 5, 8, 2, 700
    rng = np.random.default_rng(1)
    s = _Serving(hip, B, Hkv, cap, [640, 300, 0, 31, 64])
    first = int(s.lengths.max())
    prompt = [_normal(rng, B, first, Hkv, D) for _ in range(2)]
    zero = hip.DeviceBuffer.from_array(np.zeros(B, np.int32))
    bufs = [hip.DeviceBuffer.from_array(a) for a in prompt]
    q3k.kv_append_e4m3(*bufs, s.kc, s.vc, s.sc, B, first, Hkv, D, cap, 0, starts=zero)
    hip.synchronize()
    s.note(np.zeros(B, int), *prompt)
    # rows past a sequence's length hold its prompt's rest here: they must not be seen
    k, v, q = (hip.DeviceBuffer(B * h * D * 2) for h in (Hkv, Hkv, Hq))
    starts, lengths = hip.DeviceBuffer(4 * B), hip.DeviceBuffer(4 * B)
    out = hip.DeviceBuffer(B * Hq * D * 2)
    n = q3k.cache_attention_workspace_bytes(B, 1, Hq, Hkv, D, cap)
    assert n > 0
    ws = hip.DeviceBuffer(n)
    stream = hip.Stream()

    def step(st):
        q3k.kv_append_e4m3(k, v, s.kc, s.vc, s.sc, B, 1, Hkv, D, cap, 0, starts=starts, stream=st)
        q3k.gqa_attention_e4m3(q, s.kc, s.vc, s.sc, out, B, 1, Hq, Hkv, D, cap, cap, lengths=lengths, stream=st, workspace=ws,
                               workspace_bytes=n)

    graph = hip.Graph(stream, lambda: step(stream))
    try:
        for i in range(5):
            new = [_normal(rng, B, 1, Hkv, D) for _ in range(2)]
            qs = _normal(rng, B, 1, Hq, D, std=2.0)
            for buf, a in ((k, new[0]), (v, new[1]), (q, qs), (starts, s.lengths), (lengths, s.lengths + 1)):
                buf.upload(a)
            s.note(s.lengths, *new)
            s.lengths = s.lengths + 1
            ws.fill_bytes(0xFF)
            graph.launch(stream)
            stream.synchronize()
            got = out.download(np.uint16, (B, 1, Hq, D))
            ref.check_attention(f"replay {i}", got, *s.want(qs, s.lengths, 1))
            out.fill_bytes(0)
            step(None)                              # the same step eagerly: the append writes the same rows again
            hip.synchronize()
            assert np.array_equal(out.download(np.uint16, got.shape), got)
    finally:
        graph.destroy()


def test_speculative_step_on_a_stream(q3k, hip):
    """Append a drafted tree at each sequence's length, tree attention, keep the accepted path, decode on, all on one
    stream, with sequences of different lengths and trees of different sizes."""
    announce("speculative step on a stream")
    B, Hq, Hkv, cap, T = 4, 16, 4, 400, 9
    rng = np.random.default_rng(2)
    s = _Serving(hip, B, Hkv, cap, [300, 17, 128, 1])
    stream = hip.Stream()
    first = int(s.lengths.max())
    prompt = [_normal(rng, B, first, Hkv, D) for _ in range(2)]
    tree_kv = [_normal(rng, B, T, Hkv, D) for _ in range(2)]
    qs, q1 = _normal(rng, B, T, Hq, D, std=2.0), _normal(rng, B, 1, Hq, D, std=2.0)
    parents = np.array([[-1, 0, 0, 1, 1, 2, 3, 5, 5], [-1, 0, 1, 2, 3, 4, 5, 6, 7], [-1, 0, 0, 0, -2, -2, -2, -2, -2],
                        [-1, -1, 1, 0, 2, 3, 4, 4, 4]], np.int32)
    path = np.array([[0, 2, 5, 8], [0, 1, 2, 3], [0, 3, 0, 0], [1, 2, 4, 7]], np.int32)
    counts = np.array([4, 3, 2, 4], np.int32)
    one = [_normal(rng, B, 1, Hkv, D) for _ in range(2)]
    up = hip.DeviceBuffer.from_array
    bufs = {n: up(a) for n, a in (("k0", prompt[0]), ("v0", prompt[1]), ("kt", tree_kv[0]), ("vt", tree_kv[1]), ("q", qs),
                                  ("q1", q1), ("par", parents), ("path", path), ("cnt", counts), ("k1", one[0]), ("v1", one[1]),
                                  ("at", s.lengths), ("n", s.lengths + T), ("kept", s.lengths + counts),
                                  ("n1", s.lengths + counts + 1))}
    out, out1 = hip.DeviceBuffer(qs.nbytes), hip.DeviceBuffer(q1.nbytes)
    nbytes = max(q3k.cache_attention_workspace_bytes(B, S, Hq, Hkv, D, cap) for S in (1, T))
    ws = hip.DeviceBuffer(nbytes)
    b = bufs
    q3k.kv_append_e4m3(b["k0"], b["v0"], s.kc, s.vc, s.sc, B, first, Hkv, D, cap, 0, stream=stream)
    q3k.kv_append_e4m3(b["kt"], b["vt"], s.kc, s.vc, s.sc, B, T, Hkv, D, cap, 0, starts=b["at"], stream=stream)
    q3k.gqa_tree_attention_e4m3(b["q"], s.kc, s.vc, s.sc, out, b["par"], T, B, T, Hq, Hkv, D, cap, cap, lengths=b["n"],
                                stream=stream, workspace=ws, workspace_bytes=nbytes)
    q3k.kv_keep_path(s.kc, s.vc, s.sc, 1, B, Hkv, cap, D, B, 0, b["path"], 4, starts=b["at"], counts=b["cnt"], stream=stream)
    q3k.kv_append_e4m3(b["k1"], b["v1"], s.kc, s.vc, s.sc, B, 1, Hkv, D, cap, 0, starts=b["kept"], stream=stream)
    q3k.gqa_attention_e4m3(b["q1"], s.kc, s.vc, s.sc, out1, B, 1, Hq, Hkv, D, cap, cap, lengths=b["n1"], stream=stream,
                           workspace=ws, workspace_bytes=nbytes)
    stream.synchronize()
    s.note(np.zeros(B, int), *prompt)
    s.note(s.lengths, *tree_kv)
    ref.check_attention("tree", out.download(np.uint16, qs.shape), *s.want(qs, s.lengths + T, T, parents))
    for x in (s.k, s.v):
        for i in range(B):
            at = int(s.lengths[i])
            x[i, at:at + counts[i]] = x[i, at + path[i, :counts[i]]].copy()
    s.note(s.lengths + counts, *one)
    ref.check_attention("decode after", out1.download(np.uint16, q1.shape), *s.want(q1, s.lengths + counts + 1, 1))
    # what the cache holds, read back
    n = int((s.lengths + counts + 1).max())
    ko, vo = hip.DeviceBuffer(B * n * Hkv * D * 2), hip.DeviceBuffer(B * n * Hkv * D * 2)
    q3k.kv_read_e4m3(s.kc, s.vc, s.sc, ko, vo, B, Hkv, D, cap, 0, n, lengths=b["n1"])
    hip.synchronize()
    for buf, x in ((ko, s.k), (vo, s.v)):
        got = ref.bf16(buf.download(np.uint16, (B, n, Hkv, D)))
        for i in range(B):
            m = int(s.lengths[i] + counts[i] + 1)
            assert np.array_equal(got[i, :m], x[i, :m])


def test_two_graphs_share_a_workspace(q3k, hip):
    """A tree step and a decode step captured with one workspace and replayed in turn on one stream."""
    announce("two graphs, one workspace")
    B, Hq, Hkv, cached, T = 2, 8, 2, 1500, 12
    rng = np.random.default_rng(3)
    k, v = _normal(rng, B, cached, Hkv, D), _normal(rng, B, cached, Hkv, D)
    qs = [_normal(rng, B, S, Hq, D, std=2.0) for S in (1, T)]
    parents = np.tile(np.array([-1] + [t // 2 for t in range(T - 1)], np.int32), (B, 1))
    s = _Serving(hip, B, Hkv, cached, [cached] * B)
    up = hip.DeviceBuffer.from_array
    bk, bv, bp = up(k), up(v), up(parents)
    bq = [up(q) for q in qs]
    outs = [hip.DeviceBuffer(q.nbytes) for q in qs]
    sizes = [q3k.cache_attention_workspace_bytes(B, S, Hq, Hkv, D, cached) for S in (1, T)]
    assert min(sizes) > 0
    ws = hip.DeviceBuffer(max(sizes))
    q3k.kv_append_e4m3(bk, bv, s.kc, s.vc, s.sc, B, cached, Hkv, D, cached, 0)
    hip.synchronize()
    s.note([0] * B, k, v)
    stream = hip.Stream()

    def decode():
        q3k.gqa_attention_e4m3(bq[0], s.kc, s.vc, s.sc, outs[0], B, 1, Hq, Hkv, D, cached, cached, stream=stream, workspace=ws,
                               workspace_bytes=max(sizes))

    def tree():
        q3k.gqa_tree_attention_e4m3(bq[1], s.kc, s.vc, s.sc, outs[1], bp, T, B, T, Hq, Hkv, D, cached, cached, stream=stream,
                                    workspace=ws, workspace_bytes=max(sizes))

    graphs = [hip.Graph(stream, f) for f in (decode, tree)]
    try:
        want = [s.want(qs[0], [cached] * B, 1), s.want(qs[1], [cached] * B, T, parents)]
        for _ in range(3):
            for o in outs:
                o.fill_bytes(0)
            for g in graphs:
                g.launch(stream)
            stream.synchronize()
            for o, q, w in zip(outs, qs, want):
                ref.check_attention("shared workspace", o.download(np.uint16, q.shape), *w)
    finally:
        for g in graphs:
            g.destroy()


def test_two_calls_at_once(q3k, hip):
    """Split calls on two streams, each with a workspace of its own, give what they give alone."""
    announce("two calls at once")
    B, Hq, Hkv, cached, T = 1, 16, 2, 4000, 6
    rng = np.random.default_rng(9)
    s = _Serving(hip, B, Hkv, cached, [cached] * B)
    up = hip.DeviceBuffer.from_array
    bk, bv = up(_normal(rng, B, cached, Hkv, D)), up(_normal(rng, B, cached, Hkv, D))
    q3k.kv_append_e4m3(bk, bv, s.kc, s.vc, s.sc, B, cached, Hkv, D, cached, 0)
    parents = up(np.arange(-1, T - 1, dtype=np.int32))
    q = [up(_normal(rng, B, S, Hq, D, std=2.0)) for S in (1, T)]
    size = [q3k.cache_attention_workspace_bytes(B, S, Hq, Hkv, D, cached) for S in (1, T)]
    assert min(size) > 0
    ws = [hip.DeviceBuffer(n) for n in size]
    streams = [hip.Stream() for _ in range(2)]

    def call(i, out, stream):
        kw = dict(stream=stream, workspace=ws[i], workspace_bytes=size[i])
        if i == 0:
            q3k.gqa_attention_e4m3(q[0], s.kc, s.vc, s.sc, out, B, 1, Hq, Hkv, D, cached, cached, **kw)
        else:
            q3k.gqa_tree_attention_e4m3(q[1], s.kc, s.vc, s.sc, out, parents, 0, B, T, Hq, Hkv, D, cached, cached, **kw)

    shapes = [(B, 1, Hq, D), (B, T, Hq, D)]
    outs = [[hip.DeviceBuffer(int(np.prod(shape)) * 2) for _ in range(20)] for shape in shapes]
    alone = [hip.DeviceBuffer(int(np.prod(shape)) * 2) for shape in shapes]
    hip.synchronize()
    for i in range(2):
        call(i, alone[i], None)
        hip.synchronize()
    for n in range(20):
        for i in range(2):
            call(i, outs[i][n], streams[i])
    for stream in streams:
        stream.synchronize()
    for i, shape in enumerate(shapes):
        want = alone[i].download(np.uint16, shape)
        assert all(np.array_equal(o.download(np.uint16, shape), want) for o in outs[i])


def test_rows_past_4_gib(q3k, hip):
    """One KV head of 2^25 + 40 rows a sequence: codes past 4 GiB inside a sequence and across sequences.  Scores are 0
    for all rows but the last few, whose weight is e^40 of the others'.  Those rows' scores are one product each, the
    same for all, so their weights are equal; what is left are the sums' roundings and the weight of the other rows."""
    announce("e4m3 cache past 4 GiB")
    cap, B, Hq, Hkv, T = 2**25 + 40, 2, 4, 1, 4
    n = 2**25 + 33
    kc, vc, sc = (hip.DeviceBuffer(B * cap * w) for w in (D, D, 2))
    for buf, byte in ((kc, 0), (vc, 0), (sc, 127)):
        buf.fill_bytes(byte)
    rng = np.random.default_rng(4)
    rows = np.zeros((B, T, Hkv, D), np.uint16)
    rows[..., 0] = 0x4180                                     # K: 16 in the first dim
    vals = _normal(rng, B, T, Hkv, D)
    q = np.zeros((B, T, Hq, D), np.uint16)
    q[..., 0] = 0x41E3                                        # 28.375: a score of 16 * 28.375 / sqrt(128) = 40.1
    bk, bv, bq = (hip.DeviceBuffer.from_array(a) for a in (rows, vals, q))
    out = hip.DeviceBuffer(q.nbytes)
    q3k.kv_append_e4m3(bk, bv, kc, vc, sc, B, T, Hkv, D, cap, n - T)
    ws_bytes = max(q3k.cache_attention_workspace_bytes(B, S, Hq, Hkv, D, n) for S in (1, T))
    ws = hip.DeviceBuffer(ws_bytes)
    chain = hip.DeviceBuffer.from_array(np.arange(-1, T - 1, dtype=np.int32))
    v = ref.dequantise(*ref.quantise(vals))[:, :, 0]
    want = np.stack([v[:, :t + 1].mean(1) for t in range(T)], 1)[:, :, None, :].repeat(Hq, 2)
    bound = (2.0**-14 + n * np.exp(-40.0)) * np.abs(v).max() * np.ones_like(want)
    for call in ("causal", "tree"):
        out.fill_bytes(0)
        if call == "causal":
            q3k.gqa_attention_e4m3(bq, kc, vc, sc, out, B, T, Hq, Hkv, D, cap, n, workspace=ws, workspace_bytes=ws_bytes)
        else:
            q3k.gqa_tree_attention_e4m3(bq, kc, vc, sc, out, chain, 0, B, T, Hq, Hkv, D, cap, n, workspace=ws,
                                        workspace_bytes=ws_bytes)
        hip.synchronize()
        ref.check_attention(f"past 4 GiB, {call}", out.download(np.uint16, q.shape), want, bound)
    # the second and the fourth of the rows are kept, then read back
    path = hip.DeviceBuffer.from_array(np.array([[1, 3]] * B, np.int32))
    q3k.kv_keep_path(kc, vc, sc, 1, B, Hkv, cap, D, B, n - T, path, 2)
    ko, vo = Guarded(hip, nbytes=B * 2 * D * 2), Guarded(hip, nbytes=B * 2 * D * 2)
    q3k.kv_read_e4m3(kc, vc, sc, ko, vo, B, Hkv, D, cap, n - T, 2)
    hip.synchronize()
    assert np.array_equal(ref.bf16(vo.get(np.uint16, (B, 2, D))), v[:, [1, 3]])
    assert ko.guards_intact() and vo.guards_intact()
    for buf in (kc, vc, sc):
        buf.free()
