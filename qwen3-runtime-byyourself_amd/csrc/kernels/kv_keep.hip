// Keeping the accepted path of drafted tokens, for gfx950: in every layer of a
// KV cache, row start + path[b, i] of sequence b moves to row start + i.
//
// A thread owns one word of the rows of one (layer, sequence, head), K's or V's
// (or the two scale bytes of an e4m3 cache), and moves it for the whole path,
// kPathStep entries at a time: their loads, then their stores.  Because an entry
// is only followed where path[b, i] >= i, a word is read before any store
// reaches it: the stores so far went to rows below the step's first entry, and
// every later source is at least its own index.  So rows may overlap and no
// second buffer is needed.  What bounds it is latency for one sequence (a read
// of the path, a read of the rows, a store) and memory for many.
#include "q3k_common.hpp"

namespace q3k
{
    namespace
    {
        constexpr int kPathStep = 8;

        struct KeepShape
        {
            int64_t items;     // layers * B * heads * words of a row (K's, V's and one for the scales)
            uint32_t words;    // words of a row
            uint32_t per_row;  // 2 * words, one more with scales
            uint32_t B;
            uint32_t heads;
            int64_t batch_cap;
            int64_t seq_cap;
            int64_t start;
            const int32_t *path;
            int64_t path_len;
            const int32_t *starts;
            const int32_t *counts;
        };

        // Moves the word at base (rows `stride` words apart) along the path.
        template <typename W>
        __device__ __forceinline__ void keep_word(W *base, int64_t stride, const KeepShape &s, const int32_t *path, int64_t n,
                                                  int64_t start)
        {
            for (int64_t i0 = 0; i0 < n; i0 += kPathStep)
            {
                W val[kPathStep];
                bool move[kPathStep];
#pragma unroll
                for (int u = 0; u < kPathStep; ++u)
                {
                    const int64_t i = i0 + u;
                    const int64_t p = i < n ? path[i] : -1;
                    // also false for i past the end: p is -1 there
                    move[u] = p > i && start + p < s.seq_cap;
                    if (move[u])
                        val[u] = base[(start + p) * stride];
                }
#pragma unroll
                for (int u = 0; u < kPathStep; ++u)
                    if (move[u])
                        base[(start + i0 + u) * stride] = val[u];
            }
        }

        template <typename W>
        __global__ __launch_bounds__(kBlock) void keep_path_kernel(W *k, W *v, uint8_t *scales, KeepShape s)
        {
            const int64_t threads = static_cast<int64_t>(gridDim.x) * kBlock;
            for (int64_t item = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x; item < s.items; item += threads)
            {
                const int64_t outer = item / s.per_row;
                const uint32_t w = static_cast<uint32_t>(item - outer * s.per_row);
                const int64_t lb = outer / s.heads;
                const uint32_t h = static_cast<uint32_t>(outer - lb * s.heads);
                const int64_t layer = lb / s.B;
                const uint32_t b = static_cast<uint32_t>(lb - layer * s.B);
                const int64_t start = s.starts != nullptr ? s.starts[b] : s.start;
                int64_t n = s.path_len;
                if (s.counts != nullptr)
                    n = s.counts[b] < n ? s.counts[b] : n;
                if (start < 0 || start >= s.seq_cap)
                    continue;
                const int32_t *path = s.path + b * s.path_len;
                const int64_t row0 = ((layer * s.batch_cap + b) * s.heads + h) * s.seq_cap;
                if (w < s.words)
                    keep_word(k + row0 * s.words + w, s.words, s, path, n, start);
                else if (w < 2 * s.words)
                    keep_word(v + row0 * s.words + (w - s.words), s.words, s, path, n, start);
                else
                {
                    // the two scale bytes of a row, which may lie at an odd address
                    struct Pair
                    {
                        uint8_t k, v;
                    };
                    keep_word(reinterpret_cast<Pair *>(scales) + row0, int64_t{1}, s, path, n, start);
                }
            }
        }

        template <typename W>
        void launch_keep(void *k, void *v, uint8_t *scales, KeepShape s, int64_t outer, int64_t row_bytes, hipStream_t stream)
        {
            s.words = static_cast<uint32_t>(row_bytes / static_cast<int64_t>(sizeof(W)));
            s.per_row = 2 * s.words + (scales != nullptr ? 1u : 0u);
            s.items = outer * s.per_row;
            const int64_t blocks = blocks_for(s.items, kBlock), most = int64_t{1} << 22;
            keep_path_kernel<W><<<dim3(static_cast<unsigned>(blocks < most ? blocks : most)), dim3(kBlock), 0, stream>>>(
                static_cast<W *>(k), static_cast<W *>(v), scales, s);
        }
    } // namespace
} // namespace q3k

extern "C" int q3k_kv_keep_path(void *key_cache, void *value_cache, uint8_t *scales, int64_t layers, int64_t batch_cap,
                                int32_t heads, int64_t seq_cap, int64_t row_bytes, int64_t B, int64_t start, const int32_t *path,
                                int64_t path_len, const int32_t *starts, const int32_t *counts, q3k_stream_t stream)
{
    using namespace q3k;
    if (layers < 0 || B < 0 || path_len < 0)
        return set_error(Q3K_ERR_INVALID_ARGUMENT, "KV keep layer, batch and path sizes cannot be negative");
    if (batch_cap <= 0 || heads <= 0 || seq_cap <= 0 || row_bytes <= 0)
        return set_error(Q3K_ERR_INVALID_ARGUMENT, "KV keep cache dimensions must be positive");
    if (B > batch_cap)
        return set_error(Q3K_ERR_OUT_OF_RANGE, "KV keep batch size exceeds capacity");
    if (starts == nullptr && (start < 0 || start > seq_cap || path_len > seq_cap - start))
        return set_error(Q3K_ERR_OUT_OF_RANGE, "KV keep exceeds sequence capacity");
    if (row_bytes > INT32_MAX / 2 - 1 || B > INT32_MAX)
        return set_error(Q3K_ERR_OVERFLOW, "KV keep row or batch is too large");
    if (layers > 0 && (batch_cap > INT64_MAX / layers || heads > INT64_MAX / (layers * batch_cap) ||
                       seq_cap > INT64_MAX / (layers * batch_cap * heads) ||
                       2 * row_bytes + 1 > INT64_MAX / (layers * batch_cap * heads * seq_cap)))
        return set_error(Q3K_ERR_OVERFLOW, "KV keep cache size overflows");
    if (B > 0 && path_len > INT64_MAX / 4 / B)
        return set_error(Q3K_ERR_OVERFLOW, "KV keep path overflows");
    if (layers == 0 || B == 0 || path_len == 0)
        return Q3K_OK;
    if (key_cache == nullptr || value_cache == nullptr || path == nullptr)
        return set_error(Q3K_ERR_INVALID_ARGUMENT, "KV keep received a null pointer");
    if (!aligned_to(path, 4) || !aligned_to(starts, 4) || !aligned_to(counts, 4))
        return set_error(Q3K_ERR_INVALID_ARGUMENT, "KV keep index pointers must be 4-byte aligned");
    KeepShape s{};
    s.B = static_cast<uint32_t>(B);
    s.heads = static_cast<uint32_t>(heads);
    s.batch_cap = batch_cap;
    s.seq_cap = seq_cap;
    s.start = start;
    s.path = path;
    s.path_len = path_len;
    s.starts = starts;
    s.counts = counts;
    const int64_t outer = layers * B * heads;
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    const auto fits = [&](int64_t w) {
        return row_bytes % w == 0 && aligned_to(key_cache, static_cast<uintptr_t>(w)) &&
               aligned_to(value_cache, static_cast<uintptr_t>(w));
    };
    if (fits(16))
        launch_keep<Vec8>(key_cache, value_cache, scales, s, outer, row_bytes, st);
    else if (fits(4))
        launch_keep<uint32_t>(key_cache, value_cache, scales, s, outer, row_bytes, st);
    else
        launch_keep<uint8_t>(key_cache, value_cache, scales, s, outer, row_bytes, st);
    return check_launch("kv_keep_path");
}
