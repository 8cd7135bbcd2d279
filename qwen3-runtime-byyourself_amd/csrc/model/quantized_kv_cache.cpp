// qwen3::QuantizedKvCache over the gfx950 quantising append, read and path
// kernels.  The checks of append follow qwen3::KvCache's (csrc/model/kv_cache.cpp).
#include "qwen3/model/quantized_kv_cache.h"

#include "../ops/ops_common.hpp"
#include "kept_path.hpp"

#include <algorithm>
#include <stdexcept>
#include <string>

namespace qwen3
{
    namespace
    {
        template <typename T>
        T positive(T value, const char *name)
        {
            if (value <= 0)
                throw std::invalid_argument(std::string(name) + " must be positive");
            return value;
        }

        Device on_gpu(Device device)
        {
            if (!device.is_cuda())
                throw std::invalid_argument("KV cache must be stored on CUDA");
            return device;
        }

        std::uint8_t *bytes(Tensor &t) { return static_cast<std::uint8_t *>(t.data()); }
        const std::uint8_t *bytes(const Tensor &t) { return static_cast<const std::uint8_t *>(t.data()); }
    } // namespace

    QuantizedKvCache::QuantizedKvCache(std::int32_t num_layers, std::int64_t max_batch_size, std::int64_t max_sequence_length,
                                       std::int32_t num_key_value_heads, std::int32_t head_dim, Device device)
        : num_layers_(positive(num_layers, "num_layers")),
          max_batch_size_(positive(max_batch_size, "max_batch_size")),
          max_sequence_length_(positive(max_sequence_length, "max_sequence_length")),
          num_key_value_heads_(positive(num_key_value_heads, "num_key_value_heads")),
          head_dim_(positive(head_dim, "head_dim")),
          device_(on_gpu(device)),
          key_codes_(Tensor::empty(Shape{num_layers_, max_batch_size_, num_key_value_heads_, max_sequence_length_, head_dim_},
                                   DType::Float8E4M3, device_)),
          value_codes_(Tensor::empty(key_codes_.shape(), DType::Float8E4M3, device_)),
          scales_(Tensor::empty(Shape{num_layers_, max_batch_size_, num_key_value_heads_, max_sequence_length_, 2},
                                DType::ScaleE8M0, device_)),
          cached_lengths_(static_cast<std::size_t>(num_layers_), 0)
    {
    }

    void QuantizedKvCache::append(std::int32_t layer_index, std::int64_t start_position, const Tensor &key, const Tensor &value)
    {
        validate_layer_index(layer_index);
        if (key.dtype() != DType::BFloat16 || value.dtype() != DType::BFloat16)
            throw std::invalid_argument("quantized KV cache inputs must be BFloat16");
        if (key.device() != device_ || value.device() != device_)
            throw std::invalid_argument("KV cache inputs must be on the cache device");
        if (key.shape().rank() != 3 || value.shape().rank() != 3)
            throw std::invalid_argument("KV cache inputs must have rank 3");
        if (key.shape() != value.shape())
            throw std::invalid_argument("KV cache key and value shape must match");
        const std::int64_t batch = key.shape()[0], sequence = key.shape()[1];
        if (batch <= 0 || sequence <= 0)
            throw std::invalid_argument("KV cache input batch and sequence dimensions must be positive");
        if (batch > max_batch_size_)
            throw std::out_of_range("KV cache batch size exceeds capacity");
        if (key.shape()[2] != static_cast<std::int64_t>(num_key_value_heads_) * head_dim_)
            throw std::invalid_argument("KV cache projection size does not match num_key_value_heads * head_dim");
        std::int64_t &cached = cached_lengths_[static_cast<std::size_t>(layer_index)];
        if (start_position != cached)
            throw std::logic_error("KV cache append must start at the current cached length");
        if (sequence > max_sequence_length_ - start_position)
            throw std::out_of_range("KV cache append exceeds sequence capacity");
        if (active_batch_size_ != 0 && batch != active_batch_size_)
            throw std::invalid_argument("KV cache batch size cannot change before reset");
        const std::int64_t rows = layer_index * layer_rows();
        ops::detail::launch_on(device_, [&](q3k_stream_t stream) {
            return q3k_kv_append_e4m3_bf16(ops::detail::bf16_ptr(key), ops::detail::bf16_ptr(value),
                                           bytes(key_codes_) + rows * head_dim_, bytes(value_codes_) + rows * head_dim_,
                                           bytes(scales_) + 2 * rows, batch, sequence, num_key_value_heads_, head_dim_,
                                           max_sequence_length_, start_position, nullptr, stream);
        });
        active_batch_size_ = batch;
        cached += sequence;
    }

    QuantizedKvCache::KeyValue QuantizedKvCache::read(std::int32_t layer_index, std::int64_t first, std::int64_t count) const
    {
        const Layer l = layer(layer_index);
        if (first < 0 || count < 0 || first > l.cached || count > l.cached - first)
            throw std::out_of_range("KV cache read exceeds the cached length");
        const Shape shape{l.batch, count, num_key_value_heads_, head_dim_};
        KeyValue out{Tensor::empty(shape, DType::BFloat16, device_), Tensor::empty(shape, DType::BFloat16, device_)};
        ops::detail::launch_on(device_, [&](q3k_stream_t stream) {
            return q3k_kv_read_e4m3_bf16(l.key_codes, l.value_codes, l.scales, ops::detail::bf16_ptr(out.key),
                                         ops::detail::bf16_ptr(out.value), l.batch, num_key_value_heads_, head_dim_,
                                         max_sequence_length_, first, count, nullptr, stream);
        });
        return out;
    }

    void QuantizedKvCache::keep_path(std::int64_t start_position, const Tensor &path)
    {
        const std::int64_t accepted = detail::check_kept_path(cached_lengths_, active_batch_size_, device_, start_position, path);
        ops::detail::launch_on(device_, [&](q3k_stream_t stream) {
            return q3k_kv_keep_path(key_codes_.data(), value_codes_.data(), bytes(scales_), num_layers_, max_batch_size_,
                                    num_key_value_heads_, max_sequence_length_, head_dim_, active_batch_size_, start_position,
                                    static_cast<const int32_t *>(path.data()), accepted, nullptr, nullptr, stream);
        });
        std::fill(cached_lengths_.begin(), cached_lengths_.end(), start_position + accepted);
    }

    void QuantizedKvCache::reset() noexcept
    {
        std::fill(cached_lengths_.begin(), cached_lengths_.end(), 0);
        active_batch_size_ = 0;
    }

    std::int64_t QuantizedKvCache::cached_length(std::int32_t layer_index) const
    {
        validate_layer_index(layer_index);
        return cached_lengths_[static_cast<std::size_t>(layer_index)];
    }

    QuantizedKvCache::Layer QuantizedKvCache::layer(std::int32_t layer_index) const
    {
        validate_layer_index(layer_index);
        const std::int64_t rows = layer_index * layer_rows();
        return Layer{bytes(key_codes_) + rows * head_dim_,
                     bytes(value_codes_) + rows * head_dim_,
                     bytes(scales_) + 2 * rows,
                     active_batch_size_,
                     cached_lengths_[static_cast<std::size_t>(layer_index)],
                     max_sequence_length_};
    }

    void QuantizedKvCache::validate_layer_index(std::int32_t layer_index) const
    {
        if (layer_index < 0 || layer_index >= num_layers_)
            throw std::out_of_range("KV cache layer index is out of range");
    }

    std::int64_t QuantizedKvCache::layer_rows() const noexcept
    {
        return max_batch_size_ * num_key_value_heads_ * max_sequence_length_;
    }
} // namespace qwen3
