// qwen3::ops::grouped_query_attention over an 8-bit cache and tree_attention
// over the gfx950 cache attention kernels.
#include "qwen3/ops/cache_attention.h"

#include "../core/block_cache.hpp"
#include "../kernels/dispatch.hpp"
#include "ops_common.hpp"

#include <limits>

namespace qwen3::ops
{
    namespace
    {
        struct Heads
        {
            std::int32_t query;
            std::int32_t key_value;
            std::int32_t dim;
        };

        // The checks of grouped_query_attention on the query; `rows` cached rows of `batch` sequences.
        void validate_query(const Tensor &query, const Device &device, const Heads &h, std::int64_t batch, std::int64_t rows)
        {
            detail::require(query.dtype() == DType::BFloat16, "GQA currently requires bfloat16 tensors");
            detail::require(query.device().is_cuda(), "GQA tensors must be on CUDA");
            detail::require(query.device() == device, "GQA tensors must be on the same CUDA device");
            detail::require(query.shape().rank() == 3, "GQA query must have rank 3");
            const std::int64_t sequence = query.shape()[1];
            detail::require(query.shape()[0] > 0 && sequence > 0, "GQA batch and sequence dimensions must be positive");
            detail::require(query.shape()[0] == batch, "GQA query/cache batch sizes must match");
            detail::require(h.query > 0 && h.key_value > 0, "GQA head counts must be positive");
            detail::require(h.query % h.key_value == 0, "GQA query heads must be divisible by key/value heads");
            detail::require(h.dim > 0 && h.dim <= 256, "GQA head_dim must be between 1 and 256");
            detail::require(query.shape()[2] == static_cast<std::int64_t>(h.query) * h.dim, "GQA query projection size is incorrect");
            detail::require(rows >= sequence, "GQA cache must hold the query's positions");
            if (batch * sequence * h.query > std::numeric_limits<int>::max())
                throw std::overflow_error("GQA grid is too large");
        }

        std::int64_t parents_stride(const Tensor &query, const Tensor &parents)
        {
            const std::int64_t batch = query.shape()[0], nodes = query.shape()[1];
            detail::require(parents.dtype() == DType::Int32, "tree attention parents must have Int32 dtype");
            detail::require(parents.device() == query.device(), "tree attention parents must be on the query's GPU");
            detail::require(nodes <= q3k::kTreeMaxNodes, "tree attention holds at most 256 nodes a sequence");
            if (parents.shape().rank() == 1)
            {
                detail::require(parents.shape()[0] == nodes, "tree attention parents must have shape [nodes] or [batch, nodes]");
                return 0;
            }
            detail::require(parents.shape().rank() == 2 && parents.shape()[0] == batch && parents.shape()[1] == nodes,
                            "tree attention parents must have shape [nodes] or [batch, nodes]");
            return nodes;
        }

        // call(output, workspace, bytes, stream) -> status, with the workspace of this call's own split.
        template <typename Call>
        Tensor run(const Tensor &query, const Heads &h, std::int64_t rows, bool e4m3, bool tree, Call call)
        {
            Tensor output = Tensor::empty(query.shape(), DType::BFloat16, query.device());
            const std::int64_t batch = query.shape()[0], sequence = query.shape()[1];
            std::int64_t bytes = 0;
            if (h.dim == q3k::kAttHeadDim && h.query / h.key_value <= q3k::kAttColsPerWave)
                bytes = q3k::plan_cache_attention(batch, sequence, h.query, h.key_value, rows, e4m3, tree, false, true).bytes;
            const qwen3::detail::DeviceWorkspace workspace(static_cast<std::size_t>(bytes), query.device().index());
            detail::launch_on(query.device(), [&](q3k_stream_t stream) {
                return call(detail::bf16_ptr(output), workspace.data(), bytes, stream);
            });
            return output;
        }
    } // namespace

    Tensor grouped_query_attention(const Tensor &query, const QuantizedKvCache &kv_cache, std::int32_t layer_index,
                                   std::int32_t num_query_heads, std::int64_t start_position)
    {
        const QuantizedKvCache::Layer l = kv_cache.layer(layer_index);
        const Heads h{num_query_heads, kv_cache.num_key_value_heads(), kv_cache.head_dim()};
        validate_query(query, kv_cache.device(), h, l.batch, l.cached);
        const std::int64_t B = query.shape()[0], S = query.shape()[1];
        detail::require(start_position >= 0, "GQA start_position cannot be negative");
        detail::require(start_position <= l.cached && S == l.cached - start_position,
                        "GQA cache length must equal start_position + sequence_length");
        return run(query, h, l.cached, true, false, [&](uint16_t *out, void *workspace, std::int64_t bytes, q3k_stream_t stream) {
            return q3k_gqa_attention_e4m3_bf16(detail::bf16_ptr(query), l.key_codes, l.value_codes, l.scales, out, B, S, h.query,
                                               h.key_value, h.dim, l.sequence_capacity, l.cached, nullptr, workspace, bytes, stream);
        });
    }

    Tensor tree_attention(const Tensor &query, const TensorView &key_cache, const TensorView &value_cache, const Tensor &parents,
                          std::int32_t num_query_heads)
    {
        detail::require(key_cache.dtype() == DType::BFloat16 && value_cache.dtype() == DType::BFloat16,
                        "GQA currently requires bfloat16 tensors");
        detail::require(key_cache.device() == value_cache.device(), "GQA tensors must be on the same CUDA device");
        detail::require(key_cache.shape().rank() == 4 && value_cache.shape().rank() == 4, "GQA cache views must have rank 4");
        detail::require(key_cache.shape() == value_cache.shape(), "GQA key/value cache shapes must match");
        detail::require(key_cache.shape()[2] <= std::numeric_limits<std::int32_t>::max() && key_cache.shape()[3] <= 256,
                        "GQA head_dim must be between 1 and 256");
        const Heads h{num_query_heads, static_cast<std::int32_t>(key_cache.shape()[2]), static_cast<std::int32_t>(key_cache.shape()[3])};
        const std::int64_t cached = key_cache.shape()[1];
        validate_query(query, key_cache.device(), h, key_cache.shape()[0], cached);
        const std::int64_t stride = parents_stride(query, parents), B = query.shape()[0], T = query.shape()[1];
        const std::int64_t ks[4] = {key_cache.stride(0), key_cache.stride(1), key_cache.stride(2), key_cache.stride(3)};
        const std::int64_t vs[4] = {value_cache.stride(0), value_cache.stride(1), value_cache.stride(2), value_cache.stride(3)};
        return run(query, h, cached, false, true, [&](uint16_t *out, void *workspace, std::int64_t bytes, q3k_stream_t stream) {
            return q3k_gqa_tree_attention_bf16(detail::bf16_ptr(query), static_cast<const uint16_t *>(key_cache.data()),
                                               static_cast<const uint16_t *>(value_cache.data()), out,
                                               static_cast<const int32_t *>(parents.data()), stride, B, T, h.query, h.key_value,
                                               h.dim, cached, nullptr, ks, vs, workspace, bytes, stream);
        });
    }

    Tensor tree_attention(const Tensor &query, const QuantizedKvCache &kv_cache, std::int32_t layer_index, const Tensor &parents,
                          std::int32_t num_query_heads)
    {
        const QuantizedKvCache::Layer l = kv_cache.layer(layer_index);
        const Heads h{num_query_heads, kv_cache.num_key_value_heads(), kv_cache.head_dim()};
        validate_query(query, kv_cache.device(), h, l.batch, l.cached);
        const std::int64_t stride = parents_stride(query, parents), B = query.shape()[0], T = query.shape()[1];
        return run(query, h, l.cached, true, true, [&](uint16_t *out, void *workspace, std::int64_t bytes, q3k_stream_t stream) {
            return q3k_gqa_tree_attention_e4m3_bf16(detail::bf16_ptr(query), l.key_codes, l.value_codes, l.scales, out,
                                                    static_cast<const int32_t *>(parents.data()), stride, B, T, h.query, h.key_value,
                                                    h.dim, l.sequence_capacity, l.cached, nullptr, workspace, bytes, stream);
        });
    }
} // namespace qwen3::ops
