#pragma once

// KvCache in 8 bits: e4m3 codes with a power-of-two scale for each position and
// KV head (the layout and the rounding stand in q3k_abi.h), half the memory and
// half the bytes of a decode step's attention.  The rules of append, the
// lengths and their exceptions are those of qwen3::KvCache.

#include "qwen3/core/tensor.h"

#include <cstdint>
#include <vector>

namespace qwen3
{
    class QuantizedKvCache final
    {
    public:
        QuantizedKvCache(std::int32_t num_layers, std::int64_t max_batch_size, std::int64_t max_sequence_length,
                         std::int32_t num_key_value_heads, std::int32_t head_dim, Device device);
        ~QuantizedKvCache() = default;
        QuantizedKvCache(const QuantizedKvCache &) = delete;
        QuantizedKvCache &operator=(const QuantizedKvCache &) = delete;
        QuantizedKvCache(QuantizedKvCache &&) noexcept = default;
        QuantizedKvCache &operator=(QuantizedKvCache &&) noexcept = default;

        // key / value [batch, sequence, num_key_value_heads * head_dim]
        // (BFloat16) are quantised into positions start_position .. + sequence - 1
        // of layer_index; start_position must equal that layer's cached length.
        void append(std::int32_t layer_index, std::int64_t start_position, const Tensor &key, const Tensor &value);

        // Positions first .. first + count - 1 of the active batch as BFloat16
        // [batch, count, num_key_value_heads, head_dim]: exactly code * scale.
        struct KeyValue
        {
            Tensor key;
            Tensor value;
        };
        [[nodiscard]] KeyValue read(std::int32_t layer_index, std::int64_t first, std::int64_t count) const;

        // As KvCache::keep_path.
        void keep_path(std::int64_t start_position, const Tensor &path);

        // Logical reset: lengths to 0, batch size unset; memory is not cleared.
        void reset() noexcept;

        [[nodiscard]] std::int64_t cached_length(std::int32_t layer_index) const;
        [[nodiscard]] std::int64_t active_batch_size() const noexcept { return active_batch_size_; }

        // One layer as the attention reads it: codes [batch_cap, H, seq_cap, D],
        // scales [batch_cap, H, seq_cap, 2].
        struct Layer
        {
            const std::uint8_t *key_codes;
            const std::uint8_t *value_codes;
            const std::uint8_t *scales;
            std::int64_t batch;
            std::int64_t cached;
            std::int64_t sequence_capacity;
        };
        [[nodiscard]] Layer layer(std::int32_t layer_index) const;

        [[nodiscard]] const Tensor &key_codes() const noexcept { return key_codes_; }
        [[nodiscard]] const Tensor &value_codes() const noexcept { return value_codes_; }
        [[nodiscard]] const Tensor &scales() const noexcept { return scales_; }
        [[nodiscard]] std::int32_t num_layers() const noexcept { return num_layers_; }
        [[nodiscard]] std::int64_t max_batch_size() const noexcept { return max_batch_size_; }
        [[nodiscard]] std::int64_t max_sequence_length() const noexcept { return max_sequence_length_; }
        [[nodiscard]] std::int32_t num_key_value_heads() const noexcept { return num_key_value_heads_; }
        [[nodiscard]] std::int32_t head_dim() const noexcept { return head_dim_; }
        [[nodiscard]] const Device &device() const noexcept { return device_; }

    private:
        void validate_layer_index(std::int32_t layer_index) const;
        [[nodiscard]] std::int64_t layer_rows() const noexcept;

        std::int32_t num_layers_ = 0;
        std::int64_t max_batch_size_ = 0;
        std::int64_t max_sequence_length_ = 0;
        std::int32_t num_key_value_heads_ = 0;
        std::int32_t head_dim_ = 0;
        Device device_ = Device::cpu();
        Tensor key_codes_;   // [layers, batch, heads, sequence, head_dim] Float8E4M3
        Tensor value_codes_; // the same
        Tensor scales_;      // [layers, batch, heads, sequence, 2] ScaleE8M0
        std::vector<std::int64_t> cached_lengths_;
        std::int64_t active_batch_size_ = 0;
    };
} // namespace qwen3
