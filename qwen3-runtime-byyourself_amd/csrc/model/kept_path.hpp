// The checks of keep_path, shared by the bf16 and the 8-bit KV cache.
#pragma once

#include "qwen3/core/tensor.h"

#include <cstdint>
#include <stdexcept>
#include <vector>

namespace qwen3::detail
{
    // Returns the number of accepted tokens.
    inline std::int64_t check_kept_path(const std::vector<std::int64_t> &cached_lengths, std::int64_t active_batch_size,
                                        const Device &device, std::int64_t start_position, const Tensor &path)
    {
        if (path.dtype() != DType::Int32)
            throw std::invalid_argument("KV cache path must have Int32 dtype");
        if (path.device() != device)
            throw std::invalid_argument("KV cache path must be on the cache device");
        if (path.shape().rank() != 2 || path.shape()[0] != active_batch_size)
            throw std::invalid_argument("KV cache path must have shape [batch, accepted]");
        for (const std::int64_t length : cached_lengths)
            if (length != cached_lengths.front())
                throw std::logic_error("KV cache path needs one cached length in all layers");
        const std::int64_t accepted = path.shape()[1], length = cached_lengths.front();
        if (start_position < 0 || start_position > length || accepted > length - start_position)
            throw std::out_of_range("KV cache path exceeds the cached length");
        return accepted;
    }
} // namespace qwen3::detail
