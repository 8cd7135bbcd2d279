// qwen3::QuantizedKvCache, attention over it, tree_attention and keep_path on the
// GPU, run together as a speculative step goes: prefill, a drafted tree appended
// to every layer, its attention, the accepted path kept, a decode step.  The
// attention is compared with the oracle over the values read back (exactly what
// the codes stand for), the 8-bit cache and a bf16 cache of those values with each
// other.
#include "gpu_util.hpp"
#include "qwen3/model/kv_cache.h"
#include "qwen3/model/quantized_kv_cache.h"
#include "qwen3/ops/cache_attention.h"
#include "qwen3/ops/gqa_attention.h"

#include <cmath>

using qwen3::Device;
using qwen3::DType;
using qwen3::KvCache;
using qwen3::QuantizedKvCache;
using qwen3::Shape;
using qwen3::Tensor;
using test::require;
using test::require_throws;

namespace
{
    constexpr std::int64_t B = 2, D = 128, Hq = 8, Hkv = 2, cap = 160;
    constexpr std::int32_t kLayers = 2;

    Tensor rows(std::int64_t s, std::int64_t heads, uint64_t seed)
    {
        return test::to_gpu(test::values(static_cast<std::size_t>(B * s * heads * D), seed), Shape{B, s, heads * D}, DType::BFloat16);
    }

    // The oracle's causal attention of `q` over k, v [B, n, Hkv, D].
    void require_causal(const Tensor &q, const Tensor &got, const std::vector<uint16_t> &k, const std::vector<uint16_t> &v,
                        std::int64_t n, const std::string &what)
    {
        const std::int64_t S = q.shape()[1], st[4] = {n * Hkv * D, Hkv * D, D, 1};
        const auto qh = test::to_host<uint16_t>(q), gh = test::to_host<uint16_t>(got);
        std::vector<uint16_t> prim(gh.size()), lo(gh.size()), hi(gh.size());
        require(q3o_gqa_attention(qh.data(), k.data(), v.data(), B, S, Hq, Hkv, D, n, n - S, st, st, nullptr, 0, prim.data(),
                                  lo.data(), hi.data(), 2) == 0,
                "oracle attention");
        test::require_band(gh, prim, lo, hi, what);
    }

    void speculative_step()
    {
        const Device gpu = Device::cuda(0);
        QuantizedKvCache cache{kLayers, B, cap, Hkv, D, gpu};
        KvCache plain{kLayers, B, cap, Hkv, D, DType::BFloat16, gpu};
        require(cache.key_codes().dtype() == DType::Float8E4M3 && cache.scales().dtype() == DType::ScaleE8M0, "storage types");
        constexpr std::int64_t prompt = 100, nodes = 6;
        // the prompt, and the same values as a bf16 cache
        for (std::int32_t l = 0; l < kLayers; ++l)
        {
            cache.append(l, 0, rows(prompt, Hkv, 10 + l), rows(prompt, Hkv, 20 + l));
            const auto kv = cache.read(l, 0, prompt);
            require(kv.key.shape() == (Shape{B, prompt, Hkv, D}), "read shape");
            Tensor k = test::to_gpu(test::to_host<uint16_t>(kv.key), Shape{B, prompt, Hkv * D}, DType::BFloat16);
            Tensor v = test::to_gpu(test::to_host<uint16_t>(kv.value), Shape{B, prompt, Hkv * D}, DType::BFloat16);
            plain.append(l, 0, k, v);
        }
        Tensor q = rows(prompt, Hq, 3);
        Tensor out = qwen3::ops::grouped_query_attention(q, cache, 1, Hq, 0);
        {
            const auto kv = cache.read(1, 0, prompt);
            require_causal(q, out, test::to_host<uint16_t>(kv.key), test::to_host<uint16_t>(kv.value), prompt, "8-bit prefill");
        }
        // a drafted tree: 0 - (1 - (3, 4), 2 - 5)
        const std::vector<int32_t> parents{-1, 0, 0, 1, 1, 2};
        for (std::int32_t l = 0; l < kLayers; ++l)
        {
            cache.append(l, prompt, rows(nodes, Hkv, 30 + l), rows(nodes, Hkv, 40 + l));
            const auto kv = cache.read(l, prompt, nodes);
            plain.append(l, prompt, test::to_gpu(test::to_host<uint16_t>(kv.key), Shape{B, nodes, Hkv * D}, DType::BFloat16),
                         test::to_gpu(test::to_host<uint16_t>(kv.value), Shape{B, nodes, Hkv * D}, DType::BFloat16));
        }
        Tensor tq = rows(nodes, Hq, 4);
        Tensor shared = test::to_gpu(parents, Shape{nodes}, DType::Int32);
        std::vector<int32_t> twice(parents);
        twice.insert(twice.end(), parents.begin(), parents.end());
        Tensor each = test::to_gpu(twice, Shape{B, nodes}, DType::Int32);
        const auto t8 = test::to_host<uint16_t>(qwen3::ops::tree_attention(tq, cache, 0, shared, Hq));
        require(t8 == test::to_host<uint16_t>(qwen3::ops::tree_attention(tq, cache, 0, each, Hq)), "one tree for all, or one each");
        const auto t16 = test::to_host<uint16_t>(qwen3::ops::tree_attention(tq, plain.key_view(0), plain.value_view(0), each, Hq));
        // the same values through the two kernels: each within half a bf16 step and its own sums of the truth
        for (std::size_t i = 0; i < t8.size(); ++i)
            require(std::fabs(test::f32(t8[i]) - test::f32(t16[i])) <= 0.0079F * std::fabs(test::f32(t16[i])) + 1e-3F,
                    "trees over the two caches differ");
        // every node's path is causal attention over the context and that path: node 5 through 0, 2, 5
        {
            const auto kv = cache.read(0, 0, prompt + nodes);
            const auto k = test::to_host<uint16_t>(kv.key), v = test::to_host<uint16_t>(kv.value);
            const std::int64_t n = prompt + 3;
            std::vector<uint16_t> kp, vp, qp;
            const auto tqh = test::to_host<uint16_t>(tq);
            for (std::int64_t b = 0; b < B; ++b)
                for (std::int64_t r = 0; r < n; ++r)
                {
                    const std::int64_t path[3] = {0, 2, 5}, at = r < prompt ? r : prompt + path[r - prompt];
                    const auto row = static_cast<std::size_t>((b * (prompt + nodes) + at) * Hkv * D);
                    kp.insert(kp.end(), k.begin() + row, k.begin() + row + Hkv * D);
                    vp.insert(vp.end(), v.begin() + row, v.begin() + row + Hkv * D);
                }
            std::vector<uint16_t> got;
            for (std::int64_t b = 0; b < B; ++b)
            {
                const auto row = static_cast<std::size_t>((b * nodes + 5) * Hq * D);
                qp.insert(qp.end(), tqh.begin() + row, tqh.begin() + row + Hq * D);
                got.insert(got.end(), t8.begin() + row, t8.begin() + row + Hq * D);
            }
            require_causal(test::to_gpu(qp, Shape{B, 1, Hq * D}, DType::BFloat16), test::to_gpu(got, Shape{B, 1, Hq * D}, DType::BFloat16),
                           kp, vp, n, "the path of a node");
        }
        // sequence 0 accepts 0, 2, 5 and sequence 1 accepts 0, 1, 4
        const std::vector<int32_t> path{0, 2, 5, 0, 1, 4};
        Tensor kept = test::to_gpu(path, Shape{B, 3}, DType::Int32);
        const auto before = cache.read(1, prompt, nodes);
        const auto bk = test::to_host<uint16_t>(before.key), bv = test::to_host<uint16_t>(before.value);
        cache.keep_path(prompt, kept);
        plain.keep_path(prompt, kept);
        for (std::int32_t l = 0; l < kLayers; ++l)
            require(cache.cached_length(l) == prompt + 3 && plain.cached_length(l) == prompt + 3, "kept length");
        const auto after = cache.read(1, prompt, 3);
        const auto ak = test::to_host<uint16_t>(after.key), av = test::to_host<uint16_t>(after.value);
        const auto pk = test::to_host<uint16_t>(plain.key_storage());
        for (std::int64_t b = 0; b < B; ++b)
            for (std::int64_t i = 0; i < 3; ++i)
                for (std::int64_t c = 0; c < Hkv * D; ++c)
                {
                    const std::int64_t to = (b * 3 + i) * Hkv * D + c, from = (b * nodes + path[b * 3 + i]) * Hkv * D + c;
                    require(ak[to] == bk[from] && av[to] == bv[from], "kept rows");
                    require(pk[((B + b) * cap + prompt + i) * Hkv * D + c] == ak[to], "kept rows of the bf16 cache");
                }
        // and decoding goes on
        cache.append(0, prompt + 3, rows(1, Hkv, 51), rows(1, Hkv, 52));
        Tensor dq = rows(1, Hq, 5);
        Tensor dout = qwen3::ops::grouped_query_attention(dq, cache, 0, Hq, prompt + 3);
        const auto kv = cache.read(0, 0, prompt + 4);
        require_causal(dq, dout, test::to_host<uint16_t>(kv.key), test::to_host<uint16_t>(kv.value), prompt + 4, "8-bit decode");
    }

    void refusals()
    {
        const Device gpu = Device::cuda(0);
        require_throws<std::invalid_argument>([&] { QuantizedKvCache(0, B, cap, Hkv, D, gpu); }, "no layers accepted");
        require_throws<std::invalid_argument>([&] { QuantizedKvCache(1, B, cap, Hkv, D, Device::cpu()); }, "host cache accepted");
        QuantizedKvCache cache{2, B, 8, Hkv, D, gpu};
        Tensor k = rows(3, Hkv, 1), v = rows(3, Hkv, 2), q = rows(3, Hq, 3);
        require_throws<std::logic_error>([&] { cache.append(0, 1, k, v); }, "append past the length accepted");
        require_throws<std::out_of_range>([&] { cache.append(2, 0, k, v); }, "layer out of range accepted");
        require_throws<std::out_of_range>([&] { cache.append(0, 0, rows(9, Hkv, 1), rows(9, Hkv, 2)); }, "append past the capacity");
        require_throws<std::invalid_argument>([&] { cache.append(0, 0, q, q); }, "projection size accepted");
        cache.append(0, 0, k, v);
        require_throws<std::out_of_range>([&] { (void)cache.read(0, 1, 3); }, "read past the length accepted");
        require_throws<std::invalid_argument>([&] { (void)qwen3::ops::grouped_query_attention(q, cache, 0, Hq, 1); },
                                              "start that does not fit the length accepted");
        require_throws<std::invalid_argument>([&] { (void)qwen3::ops::grouped_query_attention(q, cache, 1, Hq, 0); },
                                              "attention over an empty layer accepted");
        Tensor par = test::to_gpu(std::vector<int32_t>{-1, 0}, Shape{2}, DType::Int32);
        require_throws<std::invalid_argument>([&] { (void)qwen3::ops::tree_attention(q, cache, 0, par, Hq); }, "short parents accepted");
        require_throws<std::invalid_argument>([&] { (void)qwen3::ops::tree_attention(q, cache, 0, k, Hq); }, "parents' type accepted");
        Tensor path = test::to_gpu(std::vector<int32_t>{0, 0}, Shape{B, 1}, DType::Int32);
        require_throws<std::logic_error>([&] { cache.keep_path(0, path); }, "layers of different lengths accepted");
        cache.append(1, 0, k, v);
        require_throws<std::out_of_range>([&] { cache.keep_path(3, path); }, "path past the length accepted");
        require_throws<std::invalid_argument>([&] { cache.keep_path(0, par); }, "path of another shape accepted");
        cache.keep_path(2, path);
        require(cache.cached_length(0) == 3 && cache.cached_length(1) == 3, "length after keeping one row");
        cache.reset();
        require(cache.cached_length(0) == 0 && cache.active_batch_size() == 0, "reset");
    }

    void body()
    {
        test::require_gpu();
        const int before = test::current_device();
        speculative_step();
        refusals();
        require(test::current_device() == before, "a cache call changed the current device");
    }
} // namespace

int main() { return test::run("GPU quantized KV cache test", body); }
