#pragma once

// Attention over an 8-bit KV cache, and of trees of drafted tokens over a bf16
// or an 8-bit one.

#include "qwen3/core/tensor.h"
#include "qwen3/core/tensor_view.h"
#include "qwen3/model/quantized_kv_cache.h"

#include <cstdint>

namespace qwen3::ops
{
    // grouped_query_attention (qwen3/ops/gqa_attention.h) over layer_index of an
    // 8-bit cache: query [batch, sequence, num_query_heads * head_dim]
    // (BFloat16), its cached length start_position + sequence.
    [[nodiscard]] Tensor grouped_query_attention(const Tensor &query, const QuantizedKvCache &kv_cache,
                                                 std::int32_t layer_index, std::int32_t num_query_heads,
                                                 std::int64_t start_position);

    // Attention of a tree of drafted tokens for each sequence.  query [batch,
    // nodes, num_query_heads * head_dim] (BFloat16); the last `nodes` of the
    // cached rows are the nodes' own, in their order, those before them the
    // context.  parents: Int32 [batch, nodes], or [nodes] for one tree for all,
    // on the same GPU: a node's parent, an earlier node, or -1 for a node right
    // after the context; -2 where there is no node.  A node attends to the
    // context, its ancestors and itself.  Returns [batch, nodes, num_query_heads
    // * head_dim] (BFloat16); zeros where there is no node, NaN where the way up
    // from a node meets any other number.  At most 256 nodes.
    [[nodiscard]] Tensor tree_attention(const Tensor &query, const TensorView &key_cache, const TensorView &value_cache,
                                        const Tensor &parents, std::int32_t num_query_heads);

    // The same over layer_index of an 8-bit cache.
    [[nodiscard]] Tensor tree_attention(const Tensor &query, const QuantizedKvCache &kv_cache, std::int32_t layer_index,
                                        const Tensor &parents, std::int32_t num_query_heads);
} // namespace qwen3::ops
