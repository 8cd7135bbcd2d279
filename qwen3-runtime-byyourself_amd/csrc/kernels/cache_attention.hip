// Attention over a KV cache with a length of its own for each sequence: causal
// over the e4m3 cache, and of trees of drafted tokens over a bf16 or an e4m3
// cache.
//
//   out[b, s, h] = sum_j p_j v_j,  p = softmax_j(q[b, s, h] . k_j / sqrt(D))
// over the rows j of sequence b that query s sees: with n = lengths[b] rows, 0 ..
// n - S + s (causal), or the context 0 .. n - T - 1, the node's own row
// n - T + t and those of its ancestors (tree).  A query that sees no row gets
// zeros, a sequence whose length is out of range NaN.
//
// Generic path (any head_dim <= 256, any strides and alignment): one wave per
// query row, its rows in order, lanes over the head dimension, the running
// maximum and sum of the softmax in fp32.
#include "dispatch.hpp"
#include "kv_e4m3.hpp"

namespace q3k
{
    namespace
    {
        struct CacheArgs
        {
            const uint16_t *q;
            const void *k; // bf16 values or e4m3 codes
            const void *v;
            const uint8_t *scales; // [.., 2] of each row, e4m3 only
            uint16_t *out;
            const int32_t *lengths; // null: cached
            const int32_t *parents; // null: causal
            int64_t parents_stride;
            int64_t S; // queries or nodes of a sequence
            int64_t cached;
            int64_t ks0, ks1, ks2, ks3; // element strides of K (batch, position, head, dim)
            int64_t vs0, vs1, vs2, vs3;
            int64_t ss0, ss1, ss2; // strides of the scale pairs (batch, position, head)
            int32_t Hq;
            int32_t Hkv;
            int32_t D;
            float scale;
            int64_t rows;
        };

        constexpr int kTreeWords = kTreeMaxNodes / 64;

        // What becomes of a query.
        enum class Query
        {
            Sees,  // attends to what its mask leaves it
            Empty, // gets zeros
            Bad    // gets NaN
        };

        // The rows of sequence b (0 when its length is out of range), and whether
        // that is so: outside [0, cached], or too short for the nodes of a tree.
        __device__ __forceinline__ int32_t sequence_rows(const CacheArgs &a, int64_t b, bool &bad)
        {
            const int64_t n = a.lengths != nullptr ? a.lengths[b] : a.cached;
            bad = n < 0 || n > a.cached || (a.parents != nullptr && n > 0 && n < a.S);
            return bad ? 0 : static_cast<int32_t>(n);
        }

        // Walks up from node t and calls visit(u) for the node and each ancestor.
        // A parent is smaller than its child, so the walk ends.
        template <typename Visit>
        __device__ __forceinline__ Query walk_up(const int32_t *parents, int32_t t, Visit visit)
        {
            for (;;)
            {
                const int32_t up = parents[t];
                if (up == -2)
                    return Query::Empty;
                if (up < -2 || up >= t)
                    return Query::Bad;
                visit(t);
                if (up < 0)
                    return Query::Sees;
                t = up;
            }
        }

        template <bool E4M3>
        __device__ __forceinline__ float element(const void *base, int64_t i)
        {
            if constexpr (E4M3)
                return e4m3_value(static_cast<const uint8_t *>(base)[i]);
            else
                return bf_to_f(static_cast<const uint16_t *>(base)[i]);
        }

        template <bool E4M3>
        __global__ __launch_bounds__(kBlock) void cache_generic_kernel(CacheArgs a)
        {
            const int64_t row = static_cast<int64_t>(blockIdx.x) * (kBlock / kWave) +
                                __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
            if (row >= a.rows)
                return;
            const int lane = threadIdx.x % kWave;
            const int h = static_cast<int>(row % a.Hq);
            const int64_t bs = row / a.Hq;
            const int64_t s = bs % a.S, b = bs / a.S;
            const int kvh = h / (a.Hq / a.Hkv);
            const int D = a.D;
            bool bad;
            const int32_t n = sequence_rows(a, b, bad);
            Query state = bad ? Query::Bad : n == 0 ? Query::Empty : Query::Sees;
            uint64_t tree[kTreeWords] = {};
            if (a.parents != nullptr && state == Query::Sees)
                state = walk_up(a.parents + b * a.parents_stride, static_cast<int32_t>(s), [&](int32_t u) {
#pragma unroll
                    for (int w = 0; w < kTreeWords; ++w)
                        tree[w] |= u / 64 == w ? uint64_t{1} << (u % 64) : 0;
                });
            float qv[4], acc[4];
#pragma unroll
            for (int x = 0; x < 4; ++x)
            {
                const int d = lane + 64 * x;
                qv[x] = d < D ? bf_to_f(a.q[row * D + d]) : 0.0f;
                acc[x] = 0.0f;
            }
            const int64_t kb = b * a.ks0 + kvh * a.ks2, vb = b * a.vs0 + kvh * a.vs2, sb = b * a.ss0 + kvh * a.ss2;
            float m = -__builtin_huge_valf(), l = 0.0f;
            auto attend = [&](int64_t j) {
                float part = 0.0f;
#pragma unroll
                for (int x = 0; x < 4; ++x)
                {
                    const int d = lane + 64 * x;
                    if (d < D)
                        part = __builtin_fmaf(qv[x], element<E4M3>(a.k, kb + j * a.ks1 + d * a.ks3), part);
                }
                float score = group_sum<64>(part) * a.scale, vscale = 1.0f;
                if constexpr (E4M3)
                {
                    const uint8_t *sc = a.scales + 2 * (sb + j * a.ss1);
                    score *= e4m3_scale(sc[0]);
                    vscale = e4m3_scale(sc[1]);
                }
                const float nm = fmaxf(m, score);
                const float m_use = nm == -__builtin_huge_valf() ? 0.0f : nm;
                const float ow = __expf(m - m_use);
                const float nw = __expf(score - m_use);
                l = __builtin_fmaf(l, ow, nw);
#pragma unroll
                for (int x = 0; x < 4; ++x)
                {
                    const int d = lane + 64 * x;
                    if (d < D)
                        acc[x] = __builtin_fmaf(element<E4M3>(a.v, vb + j * a.vs1 + d * a.vs3) * vscale, nw, acc[x] * ow);
                }
                m = nm;
            };
            if (state == Query::Sees)
            {
                if (a.parents == nullptr)
                {
                    for (int64_t j = 0; j <= n - a.S + s; ++j)
                        attend(j);
                }
                else
                {
                    const int64_t context = n - a.S;
                    for (int64_t j = 0; j < context; ++j)
                        attend(j);
                    for (int w = 0; w < kTreeWords; ++w)
                        for (uint64_t bits = tree[w]; bits != 0; bits &= bits - 1)
                            attend(context + 64 * w + __builtin_ctzll(bits));
                }
            }
#pragma unroll
            for (int x = 0; x < 4; ++x)
            {
                const int d = lane + 64 * x;
                if (d < D)
                    a.out[row * D + d] = state == Query::Bad ? 0x7fc0 : l == 0.0f ? 0 : f_to_bf(acc[x] / l);
            }
        }

        // The checks that the three calls share, in the order of the bf16
        // attention's; `strides` are K's and V's, non-negative.
        int validate(const char *what, const CacheArgs &a, int64_t B, int64_t bound)
        {
            if (B < 0 || a.S < 0)
                return set_error(Q3K_ERR_INVALID_ARGUMENT, "%s batch and sequence sizes cannot be negative", what);
            if (a.Hq <= 0 || a.Hkv <= 0)
                return set_error(Q3K_ERR_INVALID_ARGUMENT, "%s head counts must be positive", what);
            if (a.Hq % a.Hkv != 0)
                return set_error(Q3K_ERR_INVALID_ARGUMENT, "%s query heads must be divisible by key/value heads", what);
            if (a.D <= 0 || a.D > 256)
                return set_error(Q3K_ERR_INVALID_ARGUMENT, "%s head_dim must be between 1 and 256", what);
            if (a.cached < 0 || a.cached > bound)
                return set_error(Q3K_ERR_INVALID_ARGUMENT, "%s cached length must be between 0 and the capacity", what);
            if (a.lengths == nullptr && B > 0 && a.cached < a.S)
                return set_error(Q3K_ERR_INVALID_ARGUMENT, "%s cached length must hold the sequence", what);
            if (B == 0 || a.S == 0)
                return Q3K_OK;
            if (a.cached > INT32_MAX)
                return set_error(Q3K_ERR_OVERFLOW, "%s cached length is too large", what);
            if (a.q == nullptr || a.k == nullptr || a.v == nullptr || a.out == nullptr)
                return set_error(Q3K_ERR_INVALID_ARGUMENT, "%s received a null pointer", what);
            if (!aligned_to(a.q, 2) || !aligned_to(a.out, 2) || !aligned_to(a.lengths, 4) || !aligned_to(a.parents, 4))
                return set_error(Q3K_ERR_INVALID_ARGUMENT, "%s pointers must be aligned to their element size", what);
            if (a.S > INT64_MAX / B || B * a.S > INT64_MAX / a.Hq || B * a.S * a.Hq > INT32_MAX)
                return set_error(Q3K_ERR_OVERFLOW, "%s grid is too large", what);
            return Q3K_OK;
        }

        int validate_tree(const char *what, const CacheArgs &a)
        {
            if (a.S > kTreeMaxNodes)
                return set_error(Q3K_ERR_INVALID_ARGUMENT, "%s holds at most %d nodes a sequence", what, kTreeMaxNodes);
            if (a.parents == nullptr)
                return set_error(Q3K_ERR_INVALID_ARGUMENT, "%s received a null pointer", what);
            if (a.parents_stride != 0 && a.parents_stride < a.S)
                return set_error(Q3K_ERR_INVALID_ARGUMENT, "%s parents stride must be 0 or at least the nodes of a tree", what);
            return Q3K_OK;
        }

        // Strides of an e4m3 cache layer and its scale pairs.
        int e4m3_strides(const char *what, CacheArgs &a, int64_t B, int64_t seq_cap)
        {
            if (seq_cap <= 0)
                return set_error(Q3K_ERR_INVALID_ARGUMENT, "%s sequence capacity must be positive", what);
            if (a.Hkv > 0 && a.D > 0 && B > 0 &&
                (seq_cap > INT64_MAX / a.Hkv || seq_cap * a.Hkv > INT64_MAX / (a.D > 2 ? a.D : 2) ||
                 seq_cap * a.Hkv * (a.D > 2 ? a.D : 2) > INT64_MAX / B))
                return set_error(Q3K_ERR_OVERFLOW, "%s layer size overflows", what);
            a.ss1 = 1;
            a.ss2 = seq_cap;
            a.ss0 = seq_cap * a.Hkv;
            a.ks3 = a.vs3 = 1;
            a.ks1 = a.vs1 = a.D;
            a.ks2 = a.vs2 = seq_cap * a.D;
            a.ks0 = a.vs0 = seq_cap * a.Hkv * a.D;
            return Q3K_OK;
        }

        int launch(const char *what, CacheArgs a, int64_t B, bool e4m3, void *, int64_t, hipStream_t stream)
        {
            a.scale = 1.0f / __builtin_sqrtf(static_cast<float>(a.D));
            a.rows = B * a.S * a.Hq;
            const int64_t blocks = blocks_for(a.rows, kBlock / kWave);
            if (!launch_fits(blocks, kBlock))
                return set_error(Q3K_ERR_OVERFLOW, "%s grid is too large", what);
            const dim3 grid(static_cast<unsigned>(blocks)), block(kBlock);
            if (e4m3)
                cache_generic_kernel<true><<<grid, block, 0, stream>>>(a);
            else
                cache_generic_kernel<false><<<grid, block, 0, stream>>>(a);
            return check_launch(what);
        }
    } // namespace
} // namespace q3k

extern "C" int q3k_gqa_attention_e4m3_bf16(const uint16_t *q, const uint8_t *k_codes, const uint8_t *v_codes, const uint8_t *scales,
                                           uint16_t *out, int64_t B, int64_t S, int32_t Hq, int32_t Hkv, int32_t D,
                                           int64_t seq_cap, int64_t cached, const int32_t *lengths, void *workspace,
                                           int64_t workspace_bytes, q3k_stream_t stream)
{
    using namespace q3k;
    constexpr const char *what = "e4m3 GQA";
    CacheArgs a{};
    a.q = q;
    a.k = k_codes;
    a.v = v_codes;
    a.scales = scales;
    a.out = out;
    a.lengths = lengths;
    a.S = S;
    a.cached = cached;
    a.Hq = Hq;
    a.Hkv = Hkv;
    a.D = D;
    if (const int st = validate(what, a, B, seq_cap))
        return st;
    if (const int st = e4m3_strides(what, a, B, seq_cap))
        return st;
    if (B == 0 || S == 0)
        return Q3K_OK;
    if (scales == nullptr)
        return set_error(Q3K_ERR_INVALID_ARGUMENT, "%s received a null pointer", what);
    return launch(what, a, B, true, workspace, workspace_bytes, reinterpret_cast<hipStream_t>(stream));
}

extern "C" int q3k_gqa_tree_attention_bf16(const uint16_t *q, const uint16_t *k_cache, const uint16_t *v_cache, uint16_t *out,
                                           const int32_t *parents, int64_t parents_stride, int64_t B, int64_t T, int32_t Hq,
                                           int32_t Hkv, int32_t D, int64_t cached, const int32_t *lengths,
                                           const int64_t *k_strides, const int64_t *v_strides, void *workspace,
                                           int64_t workspace_bytes, q3k_stream_t stream)
{
    using namespace q3k;
    constexpr const char *what = "tree attention";
    CacheArgs a{};
    a.q = q;
    a.k = k_cache;
    a.v = v_cache;
    a.out = out;
    a.lengths = lengths;
    a.parents = parents;
    a.parents_stride = parents_stride;
    a.S = T;
    a.cached = cached;
    a.Hq = Hq;
    a.Hkv = Hkv;
    a.D = D;
    if (const int st = validate(what, a, B, INT64_MAX))
        return st;
    if (B == 0 || T == 0)
        return Q3K_OK;
    if (const int st = validate_tree(what, a))
        return st;
    if (k_strides == nullptr || v_strides == nullptr)
        return set_error(Q3K_ERR_INVALID_ARGUMENT, "%s stride arrays are null", what);
    for (int i = 0; i < 4; ++i)
        if (k_strides[i] < 0 || v_strides[i] < 0)
            return set_error(Q3K_ERR_INVALID_ARGUMENT, "%s cache strides cannot be negative", what);
    if (!aligned_to(k_cache, 2) || !aligned_to(v_cache, 2))
        return set_error(Q3K_ERR_INVALID_ARGUMENT, "%s pointers must be aligned to their element size", what);
    a.ks0 = k_strides[0], a.ks1 = k_strides[1], a.ks2 = k_strides[2], a.ks3 = k_strides[3];
    a.vs0 = v_strides[0], a.vs1 = v_strides[1], a.vs2 = v_strides[2], a.vs3 = v_strides[3];
    return launch(what, a, B, false, workspace, workspace_bytes, reinterpret_cast<hipStream_t>(stream));
}

extern "C" int q3k_gqa_tree_attention_e4m3_bf16(const uint16_t *q, const uint8_t *k_codes, const uint8_t *v_codes,
                                                const uint8_t *scales, uint16_t *out, const int32_t *parents,
                                                int64_t parents_stride, int64_t B, int64_t T, int32_t Hq, int32_t Hkv, int32_t D,
                                                int64_t seq_cap, int64_t cached, const int32_t *lengths, void *workspace,
                                                int64_t workspace_bytes, q3k_stream_t stream)
{
    using namespace q3k;
    constexpr const char *what = "e4m3 tree attention";
    CacheArgs a{};
    a.q = q;
    a.k = k_codes;
    a.v = v_codes;
    a.scales = scales;
    a.out = out;
    a.lengths = lengths;
    a.parents = parents;
    a.parents_stride = parents_stride;
    a.S = T;
    a.cached = cached;
    a.Hq = Hq;
    a.Hkv = Hkv;
    a.D = D;
    if (const int st = validate(what, a, B, seq_cap))
        return st;
    if (const int st = e4m3_strides(what, a, B, seq_cap))
        return st;
    if (B == 0 || T == 0)
        return Q3K_OK;
    if (const int st = validate_tree(what, a))
        return st;
    if (scales == nullptr)
        return set_error(Q3K_ERR_INVALID_ARGUMENT, "%s received a null pointer", what);
    return launch(what, a, B, true, workspace, workspace_bytes, reinterpret_cast<hipStream_t>(stream));
}

extern "C" int64_t q3k_cache_attention_workspace_bytes(int64_t, int64_t, int32_t, int32_t, int32_t, int64_t)
{
    return 0;
}
