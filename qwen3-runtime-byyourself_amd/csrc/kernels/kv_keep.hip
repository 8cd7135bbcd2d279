// Keeping the accepted path of drafted tokens, for gfx950: in every layer of a
// KV cache, row start + path[b, i] of sequence b moves to row start + i.
//
// A wave owns a few chunks of one (layer, sequence): a chunk is up to 64 words of a
// head's K or V rows, and where a row is narrower (128 bytes of codes: 8 words) the
// lanes hold that many entries of the path side by side.  It moves eight entries of one
// chunk at a time, or where rows are narrow one step of entries of eight chunks, all
// loads before the stores.  An entry is only followed where
// path[b, i] >= i, so whatever is read from row i belongs to an entry at or before
// i: its load was issued with or before that of entry i, and the store to row i
// waits for that one.  So rows may overlap and no second buffer is needed.
// What bounds it is latency for one sequence (the path beside its count and start, a
// read of the rows, a store; 28 layers of bf16 4.1 us) and scattered rows of 128 bytes
// for many (64 sequences, 36 layers of e4m3, 4 rows of 8 heads: 16 us, 31 MB at 2 TB/s;
// with plain stores 31.5 us where streaming ones took 19.0).
#include "q3k_common.hpp"

namespace q3k
{
    namespace
    {
        struct KeepShape
        {
            int64_t waves;     // layers * B * groups
            uint32_t groups;   // of chunks of a (layer, sequence)
            uint32_t chunks;   // heads * 2 * chunks of a row
            uint32_t per_row;  // chunks of a row
            uint32_t words;    // words of a row
            uint32_t shift;    // log2 of the lanes of a row
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

        // Which row an entry comes from, below 0 where it stays.  The path is read
        // whatever the count is, so that the two are read together.
        __device__ __forceinline__ int64_t entry_row(const KeepShape &s, const int32_t *path, int64_t i, int64_t n, int64_t start)
        {
            const int64_t p = i < s.path_len ? path[i] : -1;
            return i < n && p > i && start + p < s.seq_cap ? start + p : -1;
        }

        template <typename W>
        __device__ __forceinline__ W load_word(const W *p)
        {
            if constexpr (sizeof(W) == 16)
                return load8<true>(p);
            else
                return *p;
        }
        template <typename W>
        __device__ __forceinline__ void store_word(W *p, const W &w)
        {
            if constexpr (sizeof(W) == 16)
                store8<kStoreStream>(p, w);
            else
                *p = w;
        }

        // U chunks and N entries a lane at once.
        template <typename W, int U, int N>
        __global__ __launch_bounds__(kBlock) void keep_path_kernel(W *__restrict__ k, W *__restrict__ v, uint16_t *__restrict__ scales,
                                                                   KeepShape s)
        {
            const int64_t wave = static_cast<int64_t>(blockIdx.x) * (kBlock / kWave) +
                                 __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
            if (wave >= s.waves)
                return;
            const int lane = threadIdx.x % kWave;
            // layers, sequences and groups are below 2^31 together (checked by the launcher)
            const uint32_t w32 = static_cast<uint32_t>(wave);
            const uint32_t lb = w32 / s.groups, group = w32 - lb * s.groups;
            const uint32_t layer = lb / s.B, b = lb - layer * s.B;
            const int32_t *path = s.path + b * s.path_len;
            const int64_t start = s.starts != nullptr ? s.starts[b] : s.start;
            const int64_t count = s.counts != nullptr ? s.counts[b] : s.path_len;
            const int64_t n = start < 0 ? 0 : count < s.path_len ? count : s.path_len;
            const int64_t row0 = (static_cast<int64_t>(layer) * s.batch_cap + b) * s.heads * s.seq_cap;

            const int entries = kWave >> s.shift, entry = lane >> s.shift;
            const uint32_t sub = static_cast<uint32_t>(lane) & ((1u << s.shift) - 1u);
            W *base[U];
            bool have[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
            {
                const uint32_t c = group * U + u, row = (c / 2) / s.per_row, word = ((c / 2) % s.per_row << s.shift) + sub;
                have[u] = c < s.chunks && word < s.words;
                base[u] = (c % 2 == 0 ? k : v) + (row0 + row * s.seq_cap) * s.words + word;
            }
            for (int64_t i0 = 0; i0 < n; i0 += entries * N)
            {
                W val[U][N];
                int64_t from[N];
#pragma unroll
                for (int x = 0; x < N; ++x)
                    from[x] = entry_row(s, path, i0 + x * entries + entry, n, start);
#pragma unroll
                for (int x = 0; x < N; ++x)
#pragma unroll
                    for (int u = 0; u < U; ++u)
                        if (have[u] && from[x] >= 0)
                            val[u][x] = load_word(base[u] + from[x] * s.words);
#pragma unroll
                for (int x = 0; x < N; ++x)
#pragma unroll
                    for (int u = 0; u < U; ++u)
                        if (have[u] && from[x] >= 0)
                            store_word(base[u] + (start + i0 + x * entries + entry) * s.words, val[u][x]);
            }
            // the scale pairs: eight heads by eight entries, the heads dealt to the groups
            if (scales == nullptr)
                return;
            for (uint32_t h0 = group * 8; h0 < s.heads; h0 += s.groups * 8)
            {
                const uint32_t h = h0 + lane / 8;
                uint16_t *at = scales + row0 + h * s.seq_cap;
                for (int64_t i0 = 0; i0 < n; i0 += 8)
                {
                    const int64_t i = i0 + lane % 8, from = entry_row(s, path, i, n, start);
                    if (h < s.heads && from >= 0)
                        at[start + i] = at[from];
                }
            }
        }

        template <typename W>
        int launch_keep(void *k, void *v, uint8_t *scales, KeepShape s, int64_t lb, int64_t row_bytes, hipStream_t stream)
        {
            s.words = static_cast<uint32_t>(row_bytes / static_cast<int64_t>(sizeof(W)));
            while ((1u << s.shift) < s.words && (1u << s.shift) < static_cast<uint32_t>(kWave))
                ++s.shift;
            s.per_row = static_cast<uint32_t>(blocks_for(s.words, int64_t{1} << s.shift));
            // rows of a wave's width or more: one chunk and eight entries a wave; narrower
            // ones: the entries lie side by side, and eight chunks are moved at once
            const bool wide = s.shift == 6;
            const int64_t chunks = static_cast<int64_t>(s.heads) * 2 * s.per_row;
            const int64_t groups = wide ? chunks : blocks_for(chunks, 8);
            if (chunks > INT32_MAX || groups > INT32_MAX / lb || !launch_fits(blocks_for(lb * groups, kBlock / kWave), kBlock))
                return set_error(Q3K_ERR_OVERFLOW, "KV keep grid is too large");
            s.chunks = static_cast<uint32_t>(chunks);
            s.groups = static_cast<uint32_t>(groups);
            s.waves = lb * groups;
            const dim3 grid(static_cast<unsigned>(blocks_for(s.waves, kBlock / kWave))), block(kBlock);
            W *kw = static_cast<W *>(k), *vw = static_cast<W *>(v);
            uint16_t *sc = reinterpret_cast<uint16_t *>(scales);
            if (wide)
                keep_path_kernel<W, 1, 8><<<grid, block, 0, stream>>>(kw, vw, sc, s);
            else
                keep_path_kernel<W, 8, 1><<<grid, block, 0, stream>>>(kw, vw, sc, s);
            return check_launch("kv_keep_path");
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
    if (!aligned_to(scales, 2))
        return set_error(Q3K_ERR_INVALID_ARGUMENT, "KV keep scales must be 2-byte aligned");
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
    if (layers > INT32_MAX / B)
        return set_error(Q3K_ERR_OVERFLOW, "KV keep grid is too large");
    const int64_t lb = layers * B;
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    const auto fits = [&](int64_t w) {
        return row_bytes % w == 0 && aligned_to(key_cache, static_cast<uintptr_t>(w)) &&
               aligned_to(value_cache, static_cast<uintptr_t>(w));
    };
    if (fits(16))
        return launch_keep<Vec8>(key_cache, value_cache, scales, s, lb, row_bytes, st);
    if (fits(4))
        return launch_keep<uint32_t>(key_cache, value_cache, scales, s, lb, row_bytes, st);
    return launch_keep<uint8_t>(key_cache, value_cache, scales, s, lb, row_bytes, st);
}
