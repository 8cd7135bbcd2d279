"""The e4m3 KV cache, the attention over a cache with a length for each
sequence, trees of drafted tokens and the accepted path, each alone at one
size, for profiling under rocprofv3: Qwen3-8B heads (32 query, 8 key/value,
head_dim 128) unless named otherwise, lengths spread evenly from a quarter of
the cache to all of it where a case is ragged.  (The reference has a bf16
cache of one length only: src/model/kv_cache.cpp:76-204,
src/ops/gqa_attention.cu:304-345.)

Inputs rotate over more memory than the 256 MB Infinity Cache holds.  Prints
one line per case: microseconds per call, and GB/s of the bytes and TFLOP/s of
the products that the case cannot do without (4 * head_dim flops per visible
pair of a query and a row).

Usage: python3 cache_ops.py [--calls 10] [--only NAME,NAME]
"""
import argparse
import importlib
import os
import sys

import numpy as np

PKG_PARENT = os.path.dirname(os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
HKV, D = 8, 128
ROTATE_BYTES = 1 << 29


def ragged(B, most):
    return np.linspace(most // 4, most, B).round().astype(np.int32)[np.random.default_rng(B).permutation(B)]


class Layer:
    """Sets of one cache layer, codes or bf16 values of 0.3 and the like."""

    def __init__(self, hip, e4m3, B, cap):
        row = D if e4m3 else 2 * D
        n = B * HKV * cap * row
        self.sets = []
        for _ in range(max(2, min(8, -(-ROTATE_BYTES // (2 * n))))):
            k, v = hip.DeviceBuffer(n), hip.DeviceBuffer(n)
            scales = hip.DeviceBuffer(B * HKV * cap * 2) if e4m3 else None
            for b, byte in ((k, 0x31), (v, 0x2E), (scales, 126)):
                if b is not None:
                    b.fill_bytes(byte)
            self.sets.append((k, v, scales))
        self.at = 0

    def next(self):
        self.at = (self.at + 1) % len(self.sets)
        return self.sets[self.at]


def cases(q3k, hip, synth, stream):
    """(name, call, bytes, flops)"""
    def attention(name, B, S, Hq, cached, lengths=None, tree=False, e4m3=True):
        def make():
            layer = Layer(hip, e4m3, B, cached)
            q = hip.DeviceBuffer.from_array(synth.normal_bf16(8, B + S, (B, S, Hq, D)))
            out = hip.DeviceBuffer(B * S * Hq * D * 2)
            ws_bytes = q3k.cache_attention_workspace_bytes(B, S, Hq, HKV, D, cached)
            ws = hip.DeviceBuffer(max(ws_bytes, 16))
            ln = None if lengths is None else hip.DeviceBuffer.from_array(lengths)
            parents = hip.DeviceBuffer.from_array(np.tile(np.arange(-1, S - 1, dtype=np.int32), (B, 1)))
            kw = dict(lengths=ln, stream=stream, workspace=ws, workspace_bytes=ws_bytes)
            n = np.full(B, cached, np.int64) if lengths is None else lengths.astype(np.int64)
            pairs = int((S * (n - S) + S * (S + 1) // 2).sum()) * Hq
            nbytes = int(n.sum()) * HKV * 2 * (D + 1 if e4m3 else 2 * D) + 4 * B * S * Hq * D

            def call():
                k, v, s = layer.next()
                if not tree:
                    q3k.gqa_attention_e4m3(q, k, v, s, out, B, S, Hq, HKV, D, cached, cached, **kw)
                elif e4m3:
                    q3k.gqa_tree_attention_e4m3(q, k, v, s, out, parents, S, B, S, Hq, HKV, D, cached, cached, **kw)
                else:
                    st = (cached * HKV * D, HKV * D, D, 1)
                    q3k.gqa_tree_attention(q, k, v, out, parents, S, B, S, Hq, HKV, D, cached, st, st, **kw)
            return call, nbytes, 4 * D * pairs
        return name, make

    def rows(name, write, B, S):
        def make():
            layer = Layer(hip, True, B, S)
            x = [[hip.DeviceBuffer.from_array(synth.normal_bf16(9, i, (B, S, HKV, D))) for i in range(2)] for _ in range(2)]
            at = [0]

            def call():
                k, v, s = layer.next()
                a, b = x[at[0] % 2]
                at[0] += 1
                if write:
                    q3k.kv_append_e4m3(a, b, k, v, s, B, S, HKV, D, S, 0, stream=stream)
                else:
                    q3k.kv_read_e4m3(k, v, s, a, b, B, HKV, D, S, 0, S, stream=stream)
            return call, B * S * HKV * 2 * (3 * D + 1), 0
        return name, make

    def keep(name, layers, B, n, cap):
        def make():
            size = layers * B * HKV * cap * D
            k, v, s = hip.DeviceBuffer(size), hip.DeviceBuffer(size), hip.DeviceBuffer(size // D * 2)
            for b in (k, v, s):
                b.fill_bytes(0x31)
            path = hip.DeviceBuffer.from_array(np.tile(2 * np.arange(n, dtype=np.int32), (B, 1)))
            moved = layers * B * HKV * (n - 1) * 2 * (D + 1)  # row 0 stays where it is

            def call():
                q3k.kv_keep_path(k, v, s, layers, B, HKV, cap, D, B, 100, path, n, stream=stream)
            return call, 2 * moved, 0
        return name, make

    return [rows("append_16x4096", True, 16, 4096), rows("append_64x1", True, 64, 1), rows("read_16x4096", False, 16, 4096),
            attention("decode_64_ragged_to_4096", 64, 1, 32, 4096, ragged(64, 4096)),
            attention("decode_1x8192", 1, 1, 32, 8192),
            attention("chunk_512_at_7680", 1, 512, 32, 8192),
            attention("tree_5_of_64_ragged_to_2053", 64, 5, 32, 2053, ragged(64, 2053), tree=True),
            attention("tree_26_at_2000_bf16", 1, 26, 32, 2026, tree=True, e4m3=False),
            attention("tree_64_of_16_ragged_to_4160_bf16_40_heads", 16, 64, 40, 4160, ragged(16, 4160), tree=True, e4m3=False),
            keep("keep_4_of_64_in_36_layers", 36, 64, 4, 512)]


def main() -> int:
    ap = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    ap.add_argument("--calls", type=int, default=10)
    ap.add_argument("--only", default="")
    args = ap.parse_args()
    sys.path.insert(0, PKG_PARENT)
    q3k = importlib.import_module("qwen3-runtime-byyourself_amd")
    hip = importlib.import_module("qwen3-runtime-byyourself_amd.hip")
    synth = importlib.import_module("qwen3-runtime-byyourself_amd.synth")
    q3k.load()
    stream = hip.Stream()
    only = set(filter(None, args.only.split(",")))
    for name, make in cases(q3k, hip, synth, stream):
        if only and name not in only:
            continue
        call, nbytes, flops = make()
        for _ in range(3):
            call()
        stream.synchronize()
        best = None
        for _ in range(3):
            e0, e1 = hip.Event(), hip.Event()
            e0.record(stream)
            for _ in range(args.calls):
                call()
            e1.record(stream)
            e1.synchronize()
            us = e0.elapsed_ms(e1) * 1e3 / args.calls
            best = us if best is None or us < best else best
        print(f"{name}: {best:.2f} us/call, {nbytes / best / 1e3:.0f} GB/s, {flops / best / 1e6:.1f} TFLOP/s", flush=True)
    stream.synchronize()
    stream.destroy()
    return 0


if __name__ == "__main__":
    sys.exit(main())
