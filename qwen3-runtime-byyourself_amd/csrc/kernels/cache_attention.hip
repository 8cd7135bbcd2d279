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
// Matrix-core paths (head_dim 128, 16-byte rows), built from the tile operations of
// attention_tiles.hpp, whose mathematics they share with the causal bf16 attention:
// S^T = K Q^T, online softmax, O^T += V^T P^T, keys in tiles, up to 32 (position,
// head) columns to a wave.
//   Few columns (at most 32 to a (sequence, KV head): decode, small trees): the
//   block's waves divide the keys and stream their own tiles of 32 keys through
//   LDS.  Codes stay 8 bits wide until a fragment is in registers: K's with
//   ds_read_b128, 16 dims of a key, converted to two bf16 fragments with the key's
//   scale (a lane holds one key, so the scale is one register); V's with the 8-bit
//   transpose read, 8 keys of a dim, converted without a scale, which is multiplied
//   into the weights instead (there a lane holds one column and 16 keys of each 32).
//   More columns (larger trees, prefill): a block of waves shares its K and V tiles
//   as bf16; codes are converted once, on their way into LDS.
// A weight meets V as a bf16 part and a bf16 remainder, 2^-18 of it at most away from
// fp32: beside fp32 weights single results move by one bf16 step (6e-5 to 1.1e-4 of the
// norm of a result) and the error against 64 bits stays the output's rounding.  A third
// part would be half as many products again.
// The mask only touches the tiles at a sequence's end.  A masked score is -inf, so
// what K holds in a row that a query does not see never counts.  What V holds there
// meets a weight of zero, and zero times an infinity or a NaN is NaN: so a masked
// tile is looked through for such values, and if there is one its product goes the
// careful way (pv_careful).  An infinity that a query does see is put right at the end
// (see_infinities).
// Range: weights are relative to a reference that the scores may pass by kLazyMax, so
// the sum of a query's n rows is at most 2^8 n max |V|, finite for V up to 2^119 / n.
// (A reference 8 + log2 n higher takes any finite V, but its weights' exponents are
// rounded four times as coarsely, and one user's decode of 8191 rows takes 10.9 us
// for 10.7.)
//
// Generic path (any head_dim <= 256, any strides and alignment): one wave per
// query row, its rows in order, lanes over the head dimension, the running
// maximum and sum of the softmax in fp32.  It is bound by the chain of one row after
// another and reads K and V once for each query head: 60 to 700 times the time of the
// others where both could run (64 ragged sequences of up to 4096 rows: 4674 us, 69; one
// of 8191: 7714 us, 10.7).
#include "attention_tiles.hpp"
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
            int32_t B;
            bool ordered; // decode blocks take the sequences longest first
            // the fast kernels: query heads of a KV head, query blocks of a pair, slices of
            // split_keys rows, their results (unnormalised O^T [splits, rows, D], reference max
            // and sum [splits, rows, 2])
            int32_t g;
            int32_t qblocks;
            int32_t splits;
            int32_t split_keys;
            float *part_o;
            float *part_ml;
            // by (sequence, KV head) pairs; by query blocks, of a tree by those of all their columns
            Divisor by_g, by_hkv, by_pairs, by_b, by_qblocks;
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

        // The sequence that comes `rank`-th by length, or with a.ordered false in the order
        // given; the whole wave calls it.  Decode blocks take sequences of different lengths
        // longest first, so that what starts last is short (64 of 1024 to 4096 rows, 8 KV
        // heads: 66.4 us, 78.0 in a random order; of 4000 to 16000 rows 231 us and 278; their
        // trees of 5 nodes over up to 2053 bf16 rows 64.7 us and 73.8).  Finding the
        // place takes 0.6 to 1 us, more than it gives sequences that are cut into slices (4 of
        // up to 8000 rows: 17.3 us, 18.4 ordered).  In the block kernels it gave nothing where
        // the longest sequence's chain of tiles sets the time (16 trees of 64 nodes, 40 heads,
        // one key group, two blocks to a CU: 124 to 130 us, 122 in a random order); with two
        // key groups it was not tried.  Of more than 64 sequences each 64 are ordered among
        // themselves.
        __device__ __forceinline__ int32_t sequence_at(const CacheArgs &a, int32_t rank, int lane)
        {
            if (!a.ordered)
                return rank;
            const int32_t first = rank / kWave * kWave, r = rank - first;
            // lengths past the cache's count as one more, those below 0 as 0 (errors, but they
            // have a place); lanes past the last sequence come last
            const int32_t most = static_cast<int32_t>(a.cached) + 1;
            int32_t n = first + lane < a.B ? a.lengths[first + lane] : -1;
            n = first + lane >= a.B ? -1 : n < 0 ? 0 : n > most ? most : n;
            // the r-th largest, bit by bit, and of those that have it the one whose turn it is
            // by the order given
            int32_t value = 0;
            for (int bit = 31 - __builtin_clz(static_cast<uint32_t>(most)); bit >= 0; --bit)
            {
                const int32_t with = value | 1 << bit;
                value = __builtin_popcountll(__ballot(n >= with)) > r ? with : value;
            }
            const uint64_t equal = __ballot(n == value);
            const int32_t turn = r - __builtin_popcountll(__ballot(n > value));
            const int32_t before = static_cast<int32_t>(__builtin_amdgcn_mbcnt_hi(
                static_cast<uint32_t>(equal >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(equal), 0)));
            return first + static_cast<int32_t>(__builtin_ctzll(__ballot(n == value && before == turn)));
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

        // ---- masks -----------------------------------------------------------------

        // Nodes base .. base + 63 of a tree of T, one a lane of a wave, with `up` its parent:
        // which of them are the node's ancestors or itself, and where the way up leaves them
        // (an earlier node, or -1, -2, or kBadParent for a parent that cannot be).  Each step
        // joins a node's stretch of the way with that of the node where it ends, so 64 nodes
        // take at most six (a chain of 128 nodes in two waves: 22 us a call of 4 trees, 37
        // when each position went up node by node).
        constexpr int32_t kBadParent = -3;

        template <typename Mask>
        __device__ __forceinline__ void ancestors(int32_t up, int32_t base, int32_t T, int lane, Mask &mask, int32_t &end)
        {
            const int32_t node = base + lane;
            mask = Mask{1} << (lane % (8 * static_cast<int>(sizeof(Mask))));
            end = node >= T ? -2 : up < -2 || up >= node ? kBadParent : up;
            while (__ballot(end >= base) != 0)
            {
                const int src = end >= base ? end - base : lane;
                Mask m;
                if constexpr (sizeof(Mask) == 4)
                    m = static_cast<uint32_t>(__shfl(static_cast<int>(mask), src, kWave));
                else
                    m = static_cast<uint32_t>(__shfl(static_cast<int>(mask), src, kWave)) |
                        static_cast<uint64_t>(static_cast<uint32_t>(__shfl(static_cast<int>(mask >> 32), src, kWave))) << 32;
                const int32_t e = __shfl(end, src, kWave);
                if (end >= base)
                {
                    mask |= m;
                    end = e;
                }
            }
        }
        __device__ __forceinline__ Query query_of(int32_t end)
        {
            return end == -1 ? Query::Sees : end == -2 ? Query::Empty : Query::Bad;
        }

        // The masks of a tree's nodes: word w + 1 of a node holds the bits of nodes 32 w ..
        // + 31 that it sees, word 0 stands for the context before them and the last word for
        // what lies behind.
        template <bool TREE>
        struct TreeMasks
        {
            static constexpr int kWords = kTreeMaxNodes / 32 + 2;
            uint32_t mask[kTreeMaxNodes][kWords];
            int32_t end[kTreeMaxNodes]; // -1, -2 or kBadParent
        };
        template <>
        struct TreeMasks<false>
        {
        };

        // Every wave of the block calls it, `up` the parent of node 64 wave + lane: 64 nodes
        // at a time, which look up the way above them in the nodes before.
        __device__ __forceinline__ void tree_masks(TreeMasks<true> &t, int32_t up, int32_t T, int wave, int lane)
        {
            constexpr int kWords = TreeMasks<true>::kWords;
            const int32_t base = kWave * wave, node = base + lane;
            uint64_t mask = 0;
            int32_t end = -2;
            if (base < T)
                ancestors(up, base, T, lane, mask, end);
            for (int32_t done = 0; done < T; done += kWave)
            {
                if (done == base)
                {
                    const int32_t above = end;
                    if (above >= 0)
                        end = t.end[above];
                    t.end[node] = end;
                    t.mask[node][0] = 0xffffffffu;
                    t.mask[node][kWords - 1] = 0;
#pragma unroll
                    for (int w = 0; w < kWords - 2; ++w)
                    {
                        uint32_t bits = above >= 0 ? t.mask[above][1 + w] : 0u;
                        if (w / 2 == wave)
                            bits = static_cast<uint32_t>(mask >> (32 * (w % 2)));
                        t.mask[node][1 + w] = bits;
                    }
                }
                __syncthreads();
            }
        }

        // Which of the 32 keys from `off` nodes into the tree (below 0: the context) a
        // position sees.
        template <int W>
        __device__ __forceinline__ uint32_t tree_window(const uint32_t (&row)[W], int32_t off)
        {
            int i = (off >> 5) + 1, j = i + 1;
            i = i < 0 ? 0 : i < W ? i : W - 1;
            j = j < 0 ? 0 : j < W ? j : W - 1;
            return __builtin_amdgcn_alignbit(row[j], row[i], static_cast<uint32_t>(off) & 31u);
        }
        // The same for a tree of up to 32 nodes, `mask` those that the position sees.
        __device__ __forceinline__ uint32_t tree_window(uint32_t mask, int32_t off)
        {
            return off >= 0 ? (off < 32 ? mask >> off : 0u)
                            : off > -32 ? __builtin_amdgcn_alignbit(mask, 0xffffffffu, static_cast<uint32_t>(off) & 31u)
                                        : 0xffffffffu;
        }

        // Which of the 32 keys from key0 are at most `last`.
        __device__ __forceinline__ uint32_t causal_window(int32_t key0, int32_t last)
        {
            const int32_t n = last - key0 + 1;
            return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u;
        }

        // Element r of a lane's S^T half is key 8 (r / 4) + 4 lg + r % 4: the window is moved
        // by 4 lg once, and each element tests a bit that is a constant.
        template <int HH>
        __device__ __forceinline__ void mask_scores(f32x16_t (&sacc)[HH], const uint32_t (&seen)[HH], int lg)
        {
#pragma unroll
            for (int hh = 0; hh < HH; ++hh)
            {
                const uint32_t w = seen[hh] >> (4 * lg);
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if ((w >> (8 * (r / 4) + r % 4) & 1u) == 0)
                        sacc[hh][r] = -__builtin_huge_valf();
            }
        }

        // ---- products over e4m3 tiles ------------------------------------------------

        typedef int i32x2_t __attribute__((ext_vector_type(2)));
        typedef __attribute__((address_space(3))) i32x2_t lds_i32x2_t;

        // Slots of the 16-byte chunks of a 128-byte row of codes.  Two rows span the LDS
        // banks, so K's chunks move by the row's pair: 16 consecutive rows put a chunk in
        // 16 places.  V's transpose reads take rows {0..3, 8..11} or {4..7, 12..15} of 16
        // and two chunks at once: bits 1 and 3 of the row spread the four pairs of rows.
        __device__ __forceinline__ int k_slot8(int r, int c) { return c ^ ((r >> 1) & 7); }
        __device__ __forceinline__ int v_slot8(int r, int c) { return c ^ ((r & 2) | ((r >> 1) & 4)); }

        // S^T of the 32 keys of a tile of codes; scale: that of key li.  A lane's 16 codes of
        // chunk 2 c + lg are the dims of Q fragments 2 c and 2 c + 1 (load_q orders them so).
        __device__ __forceinline__ f32x16_t qk_codes(const unsigned char *k_lds, const bf16x8_t (&qf)[kAttD / 16], int li, int lg,
                                                     float scale)
        {
            auto read = [&](int c) __attribute__((always_inline)) {
                return *reinterpret_cast<const uint4 *>(k_lds + li * kAttD + 16 * k_slot8(li, 2 * c + lg));
            };
            f32x16_t sacc = f32x16_t{};
            uint4 codes[2] = {read(0), {}};
#pragma unroll
            for (int c = 0; c < kAttD / 32; ++c)
            {
                if (c + 1 < kAttD / 32)
                    codes[(c + 1) % 2] = read(c + 1);
                __builtin_amdgcn_sched_barrier(0); // keep the reads ahead of these MFMAs
                const uint4 w = codes[c % 2];
                sacc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf8(decode8(make_uint2(w.x, w.y), scale)), qf[2 * c], sacc, 0, 0, 0);
                sacc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf8(decode8(make_uint2(w.z, w.w), scale)), qf[2 * c + 1], sacc, 0,
                                                               0, 0);
            }
            return sacc;
        }

        // Per-lane LDS offsets of V's 8-bit transpose reads: lanes 2 i, 2 i + 1 of each 16
        // give row i of the eight keys 4 lg + 0..3, 8 + 4 lg + 0..3 (those of the P^T
        // elements a lane holds) and 16 dims; a lane gets the eight keys of its dim.
        __device__ __forceinline__ void v_offsets8(int lane, int (&v_off)[kAttD / 32])
        {
            const int j = lane % 16, lg = lane / 32, i = j / 2;
            const int row = 8 * (i / 4) + 4 * lg + i % 4;
#pragma unroll
            for (int dt = 0; dt < kAttD / 32; ++dt)
                v_off[dt] = row * kAttD + 16 * v_slot8(row, 2 * dt + (lane / 16) % 2) + 8 * (j % 2);
        }

        // Fragment of P V step i (16-key chunk i / 4, dims 32 (i % 4) .. + 31), in codes.
        __device__ __forceinline__ uint2 read_v8(const unsigned char *v_lds, const int (&v_off)[kAttD / 32], int i)
        {
            const i32x2_t c = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2_t *)(v_lds + v_off[i % 4] + 16 * (i / 4) * kAttD));
            return make_uint2(static_cast<uint32_t>(c.x), static_cast<uint32_t>(c.y));
        }

        // O^T += V^T P^T over a tile of codes, V's scales in P: a bf16 high part and the
        // remainder, 16 bits together as long as p * 2^e stays above 2^-110.  Of rows whose
        // largest value is below 2^-86 the smallest weights (2^-16 of the largest) lose some
        // of them, at most 2^-117 for each row.  The other end is the file's head's.
        __device__ __forceinline__ void pv_codes(const unsigned char *v_lds, const int (&v_off)[kAttD / 32], const bf16x8_t (&phi)[1][2],
                                                 const bf16x8_t (&plo)[1][2], f32x16_t (&o)[kAttD / 32])
        {
            uint2 vq[kAhead + 1];
#pragma unroll
            for (int x = 0; x < kAhead; ++x)
                vq[x] = read_v8(v_lds, v_off, x);
#pragma unroll
            for (int i = 0; i < 8; ++i)
            {
                if (i + kAhead < 8)
                    vq[(i + kAhead) % (kAhead + 1)] = read_v8(v_lds, v_off, i + kAhead);
                __builtin_amdgcn_sched_barrier(0); // keep the reads ahead of these MFMAs
                const int dt = i % 4, mm = i / 4;
                const bf16x8_t v = as_bf8(decode8(vq[i % (kAhead + 1)], 1.0f));
                o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v, phi[0][mm], o[dt], 0, 0, 0);
                o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v, plo[0][mm], o[dt], 0, 0, 0);
            }
        }

        // ---- masked tiles that hold infinities or NaN ---------------------------------

        // Whether a wave's lanes see such a value among the `bytes` of a V tile.
        template <bool CODES>
        __device__ __forceinline__ bool has_nonfinite(const unsigned char *v_lds, int bytes, int lane)
        {
            constexpr uint32_t kAbs = CODES ? 0x7f7f7f7fu : 0x7f807f80u, kOne = CODES ? 0x01010101u : 0x00800080u;
            constexpr uint32_t kTop = CODES ? 0x80808080u : 0x80008000u;
            uint32_t top = 0;
            for (int i = 16 * lane; i < bytes; i += 16 * kWave)
            {
                const uint4 w = *reinterpret_cast<const uint4 *>(v_lds + i);
                top |= ((w.x & kAbs) + kOne) | ((w.y & kAbs) + kOne) | ((w.z & kAbs) + kOne) | ((w.w & kAbs) + kOne);
            }
            return __any((top & kTop) != 0);
        }

        // O^T += V^T P^T of a masked tile with infinities or NaN in it: the product with
        // those set to zero, then, key by key, each of them added where its column sees
        // the key.  Rare, so it is written for few registers: read(i) is the bf16 fragment
        // of P V step i, values(key, dt, q4) the four V values of a key at dims
        // 32 dt + 8 q4 + 4 lg, those of elements 4 q4 .. + 3 of O^T.
        template <int HH, typename Read, typename Values>
        __device__ __forceinline__ void pv_careful(Read read, Values values, const uint32_t (&seen)[HH], const bf16x8_t (&phi)[HH][2],
                                                   const bf16x8_t (&plo)[HH][2], f32x16_t (&o)[kAttD / 32])
        {
#pragma unroll
            for (int i = 0; i < 8 * HH; ++i)
            {
                const int dt = i % 4, hh = i / 8, mm = (i / 4) % 2;
                Vec8 v = __builtin_bit_cast(Vec8, read(i));
#pragma unroll
                for (int j = 0; j < 4; ++j)
                {
                    const uint32_t bad = ((v.d[j] & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
                    v.d[j] &= ~((bad >> 15) * 0xffffu);
                }
                o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf8(v), phi[hh][mm], o[dt], 0, 0, 0);
                o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf8(v), plo[hh][mm], o[dt], 0, 0, 0);
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll 1
            for (int key = 0; key < 32 * HH; ++key)
            {
                const bool sees = ((key < 32 ? seen[0] : seen[HH - 1]) >> (key % 32) & 1u) != 0;
#pragma unroll
                for (int dt = 0; dt < kAttD / 32; ++dt)
#pragma unroll
                    for (int q4 = 0; q4 < 4; ++q4)
                    {
                        const float4 x = values(key, dt, q4);
                        const float e[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                        for (int u = 0; u < 4; ++u)
                            o[dt][4 * q4 + u] +=
                                sees && (__float_as_uint(e[u]) & 0x7f800000u) == 0x7f800000u ? e[u] : 0.0f;
                        __builtin_amdgcn_sched_barrier(0);
                    }
            }
        }

        // The values argument of pv_careful: of a tile of bf16 rows, and of codes.
        __device__ __forceinline__ float4 v_values(const unsigned char *v_lds, int lg, int key, int dt, int q4)
        {
            const uint2 w = *reinterpret_cast<const uint2 *>(v_lds + key * kRowBytes + 16 * v_slot(key, 4 * dt + q4) + 8 * lg);
            return make_float4(bf_lo(w.x), bf_hi(w.x), bf_lo(w.y), bf_hi(w.y));
        }
        __device__ __forceinline__ float4 v_values8(const unsigned char *v_lds, int lg, int key, int dt, int q4)
        {
            const uint32_t w = *reinterpret_cast<const uint32_t *>(v_lds + key * kAttD + 16 * v_slot8(key, 2 * dt + q4 / 2) +
                                                                   8 * (q4 % 2) + 4 * lg);
            const uint32_t lo = decode2<false>(w, 1.0f), hi = decode2<true>(w, 1.0f);
            return make_float4(bf_lo(lo), bf_hi(lo), bf_lo(hi), bf_hi(hi));
        }

        // Infinities of V that a column does see.  A weight is a bf16 part and a remainder,
        // and a remainder of zero, or below it, times an infinity is NaN, not the infinity.
        // So where dims 32 dt .. + 31 of a result (elements of o as store_dims takes them)
        // are not finite, the wave looks through rows begin .. end - 1 of V again and gives
        // each such element the sum of the infinities and NaN that its column sees, until all
        // are NaN.  What they do not explain has left fp32's range, and stays infinite.  live:
        // whether the lane's column has a result that l does not make NaN anyway.  Only bf16
        // holds infinities.  Looking costs 16 instructions where all is finite, once a result.
        template <typename Sees>
        __device__ __forceinline__ void see_infinities(const unsigned char *vbase, int32_t vstride, int32_t begin, int32_t end,
                                                       int dt, int lane, bool live, Sees sees, f32x16_t &o)
        {
            float zero = 0.0f; // NaN if one is not finite
#pragma unroll
            for (int r = 0; r < 16; ++r)
                zero = __builtin_fmaf(o[r], 0.0f, zero);
            if (!__any(live && zero != 0.0f))
                return;
            const auto finite = [](float x) __attribute__((always_inline)) {
                return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u;
            };
            uint32_t wild = 0;
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if (live && !finite(o[r]))
                {
                    wild |= 1u << r;
                    o[r] = __builtin_copysignf(__FLT_MAX__, o[r]);
                }
            const int lg = lane / 32;
            const unsigned char *dims = vbase + 64 * dt;
#pragma unroll 1
            for (int64_t row0 = begin; row0 < end; row0 += kWave / 4) // four lanes a row
            {
                const int64_t row = row0 + lane / 4;
                uint32_t top = 0;
                if (row < end)
                {
                    const uint4 w = *reinterpret_cast<const uint4 *>(dims + row * vstride + 16 * (lane % 4));
                    constexpr uint32_t kAbs = 0x7f807f80u, kOne = 0x00800080u;
                    top = ((w.x & kAbs) + kOne) | ((w.y & kAbs) + kOne) | ((w.z & kAbs) + kOne) | ((w.w & kAbs) + kOne);
                }
                uint64_t rows = __ballot((top & 0x80008000u) != 0);
                bool open = rows == 0; // whether another row could change an element
                while (rows != 0)
                {
                    const int at = __builtin_ctzll(rows) / 4;
                    rows &= ~(uint64_t{15} << (4 * at));
                    const int64_t key = row0 + at;
                    const bool seen = sees(static_cast<int32_t>(key));
#pragma unroll
                    for (int q4 = 0; q4 < 4; ++q4)
                    {
                        const uint2 w = *reinterpret_cast<const uint2 *>(dims + key * vstride + 16 * q4 + 8 * lg);
                        const float e[4] = {bf_lo(w.x), bf_hi(w.x), bf_lo(w.y), bf_hi(w.y)};
#pragma unroll
                        for (int u = 0; u < 4; ++u)
                            o[4 * q4 + u] += seen && !finite(e[u]) ? e[u] : 0.0f;
                    }
                }
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    open = open || ((wild >> r & 1u) != 0 && o[r] == o[r]);
                if (!__any(open))
                    break;
            }
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if ((wild >> r & 1u) != 0 && finite(o[r]))
                    o[r] = __builtin_copysignf(__builtin_huge_valf(), o[r]);
        }

        // ---- results -------------------------------------------------------------------

        // Q fragments of the lane's column, a padding column's from the last position
        // (its results are not stored).  CODES: in the order of qk_codes.
        template <bool CODES>
        __device__ __forceinline__ void load_q(const CacheArgs &a, int64_t b, int32_t s_col, int h_col, int lg,
                                               bf16x8_t (&qf)[kAttD / 16])
        {
            const int64_t s_row = s_col < a.S ? s_col : a.S - 1;
            const Vec8 *qrow = reinterpret_cast<const Vec8 *>(a.q + ((b * a.S + s_row) * a.Hq + h_col) * kAttD);
#pragma unroll
            for (int c = 0; c < kAttD / 16; ++c)
                qf[c] = as_bf8(qrow[CODES ? 4 * (c / 2) + 2 * lg + c % 2 : 2 * c + lg]);
        }

        // Dims 32 dt .. + 31 of a query's result, quarters first .. first + QUARTERS - 1 of
        // them (O^T elements 0 .. of o): bf16 O / l, or with slices the unnormalised O^T of
        // this one.
        template <int QUARTERS>
        __device__ __forceinline__ void store_dims(const CacheArgs &a, bool split, int sp, int64_t row, int dt, int first, int lg,
                                                   const f32x16_t &o, float inv, float l, Query q)
        {
            if (split)
            {
                float *po = a.part_o + (static_cast<int64_t>(sp) * a.rows + row) * kAttD;
#pragma unroll
                for (int q4 = 0; q4 < QUARTERS; ++q4)
                {
                    float4 w = {o[4 * q4], o[4 * q4 + 1], o[4 * q4 + 2], o[4 * q4 + 3]};
                    if (q != Query::Sees)
                        w = {0.0f, 0.0f, 0.0f, 0.0f};
                    *reinterpret_cast<float4 *>(po + dt * 32 + 8 * (first + q4) + 4 * lg) = w;
                }
                return;
            }
            const bool none = q != Query::Sees || l == 0.0f;
            const uint32_t fill = q == Query::Bad ? 0x7fc07fc0u : 0u;
            uint16_t *orow = a.out + row * kAttD;
#pragma unroll
            for (int q4 = 0; q4 < QUARTERS; ++q4)
            {
                uint2 w;
                w.x = pack_rne(o[4 * q4] * inv, o[4 * q4 + 1] * inv);
                w.y = pack_rne(o[4 * q4 + 2] * inv, o[4 * q4 + 3] * inv);
                if (none)
                    w.x = w.y = fill;
                *reinterpret_cast<uint2 *>(orow + dt * 32 + 8 * (first + q4) + 4 * lg) = w;
            }
        }
        // The slice's reference max and sum: those of a query without a row leave it
        // zeros, those of a bad one NaN.
        __device__ __forceinline__ void store_ml(const CacheArgs &a, int sp, int64_t row, float m, float l, Query q)
        {
            const float2 ml = q == Query::Sees    ? make_float2(m, l)
                              : q == Query::Empty ? make_float2(-__builtin_huge_valf(), 0.0f)
                                                  : make_float2(0.0f, __builtin_nanf(""));
            reinterpret_cast<float2 *>(a.part_ml)[static_cast<int64_t>(sp) * a.rows + row] = ml;
        }

        // Zeros or NaN for columns col0 .. col_end - 1 of a pair (a sequence without
        // rows, or a block whose queries see none).
        __device__ __forceinline__ void fill_columns(const CacheArgs &a, int64_t b, int kvh, int32_t col0, int32_t col_end, bool nan,
                                                     int thread, int threads)
        {
            const uint32_t w = nan ? 0x7fc07fc0u : 0u;
            for (int32_t i = thread; i < (col_end - col0) * (kAttD / 4); i += threads)
            {
                const int32_t col = col0 + i / (kAttD / 4);
                const int64_t row = (b * a.S + col / a.by_g) * a.Hq + kvh * a.g + col % a.by_g;
                reinterpret_cast<uint2 *>(a.out + row * kAttD)[i % (kAttD / 4)] = make_uint2(w, w);
            }
        }

        // ---- few columns ---------------------------------------------------------------

        // At most 32 columns to a (sequence, KV head): one wave holds them all, the
        // block's KW waves divide the keys and share nothing until the merge.  Each
        // streams its own tiles of 32 keys (8 KiB of bf16 K and of V, 4 KiB of codes)
        // through two K and two V buffers with no barrier, as the causal bf16 attention
        // does; the scales of a tile's rows come along, a word a key.
        // What bounds it is memory for many sequences, one wave's chain of tiles for few.  A
        // tile of codes is half the bytes of a bf16 one at the same work, so two waves go on
        // a SIMD (64 KiB of LDS a block, at most 256 registers) and one's conversions and
        // softmax run beside the other's: with 64-key tiles and one wave a SIMD 64 ragged
        // sequences of up to 4096 rows took 73.3 us against 69.2, their trees of 5 nodes 51.3
        // against 39.2.  The two are waves of one block (KW 8) where there is one to a CU or
        // the keys are long (8 sequences of 1000 rows whole: 12.9 us, 15.8 with KW 4; 32
        // ragged ones of up to 2500 29.7 and 38.4), else of two (64 of up to 1000: 23.3 us,
        // 28.0 with KW 8).
        // 64 ragged sequences of 1024 to 4096 rows, 32 / 8 heads: 65 to 72 us, 339 MB at 4.7
        // to 5.2 TB/s of the 5.4 to 5.9 that the access pattern reaches; one of 8191 rows,
        // 16 / 8 heads, cut into slices, 10.8 us, of which the merge takes 2.8.
        template <int KW, bool E4M3, bool TREE>
        __global__ __launch_bounds__(KW *kWave, E4M3 ? 2 : 1) void cache_decode_kernel(CacheArgs a)
        {
            constexpr int RB = E4M3 ? kAttD : kRowBytes, kKeys = kCacheDecodeTile, kTileBytes = kKeys * RB;
            using St = Staging<1, kKeys, RB>;
            constexpr int kL = St::kLoads, kS = E4M3 ? 1 : 0;
            __shared__ __attribute__((aligned(16))) unsigned char k_a[KW * kTileBytes];
            __shared__ __attribute__((aligned(16))) unsigned char k_b[KW * kTileBytes];
            __shared__ __attribute__((aligned(16))) unsigned char v_a[KW * kTileBytes];
            __shared__ __attribute__((aligned(16))) unsigned char v_b[KW * kTileBytes];
            __shared__ uint32_t s_a[E4M3 ? KW * kWave : 1];
            __shared__ uint32_t s_b[E4M3 ? KW * kWave : 1];
            __shared__ __attribute__((aligned(16))) float v_scale[E4M3 ? KW * kWave : 4];
            const int kw = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
            const int lane = threadIdx.x % kWave;
            const int li = lane % 32, lg = lane / 32;
            // Slices outermost: those of whole length first, each spread over the XCDs (4
            // sequences of up to 8000 rows 17.2 us, 19.1 with a pair's slices side by side).
            const int32_t sp = static_cast<int32_t>(blockIdx.x) / a.by_pairs, pair = static_cast<int32_t>(blockIdx.x) % a.by_pairs;
            const int32_t kvh = pair % a.by_hkv;
            const int64_t b = sequence_at(a, pair / a.by_hkv, lane);
            const int32_t S = static_cast<int32_t>(a.S);
            const int g = a.g;
            bool bad;
            const int32_t n_keys = sequence_rows(a, b, bad);
            if (n_keys == 0)
            {
                if (sp == 0)
                    fill_columns(a, b, kvh, 0, S * g, bad, threadIdx.x, KW * kWave);
                return;
            }
            const int64_t slice_begin = static_cast<int64_t>(sp) * a.split_keys;
            if (slice_begin >= n_keys)
                return;
            const int32_t k_begin = static_cast<int32_t>(slice_begin);
            const bool split = n_keys > a.split_keys;
            const int32_t k_end = n_keys - k_begin > a.split_keys ? k_begin + a.split_keys : n_keys;
            const int first = k_begin / kKeys + kw, tile_end = (k_end + kKeys - 1) / kKeys;
            const int mine = first < tile_end ? (tile_end - first + KW - 1) / KW : 0;
            const int32_t context = n_keys - S;                       // rows before the queries' own
            const int32_t all_seen = TREE ? context : context + 1;    // rows every query sees

            int32_t parent = 0;
            if constexpr (TREE)
                parent = a.parents[b * a.parents_stride + (lane < S ? lane : S - 1)];
            // the lane's column; lanes past the last one repeat a row of the last position
            const int32_t s_col = li / a.by_g;
            const int h_col = kvh * g + li % a.by_g;
            const bool col_ok = s_col < S;
            const int32_t s_row = col_ok ? s_col : S - 1;

            constexpr int64_t kElement = E4M3 ? 1 : 2;
            const unsigned char *kbase = static_cast<const unsigned char *>(a.k) + (b * a.ks0 + kvh * a.ks2) * kElement;
            const unsigned char *vbase = static_cast<const unsigned char *>(a.v) + (b * a.vs0 + kvh * a.vs2) * kElement;
            const uint8_t *sbase = a.scales + 2 * (b * a.ss0 + kvh * a.ss2);
            const int32_t kstride = static_cast<int32_t>(a.ks1 * kElement), vstride = static_cast<int32_t>(a.vs1 * kElement);
            const auto kslot = [](int r, int c) __attribute__((always_inline)) { return E4M3 ? k_slot8(r, c) : k_slot(r, c); };
            const auto vslot = [](int r, int c) __attribute__((always_inline)) { return E4M3 ? v_slot8(r, c) : v_slot(r, c); };
            int32_t k_voff[kL], v_voff[kL];
            tile_offsets<1, kKeys, RB>(0, lane, kstride, kslot, k_voff);
            tile_offsets<1, kKeys, RB>(0, lane, vstride, vslot, v_voff);
            auto load_k = [&](int j, unsigned char *buf, uint32_t *sbuf) __attribute__((always_inline)) {
                const int tile = first + KW * j;
                if constexpr (E4M3)
                {
                    const int last = n_keys - 1 - tile * kKeys;
                    __builtin_amdgcn_raw_ptr_buffer_load_lds(tile_rsrc(sbase + 2 * static_cast<int64_t>(tile) * kKeys),
                                                             (lds_void_t *)(sbuf + kw * kWave), 2,
                                                             2 * (lane % kKeys < last ? lane % kKeys : last), 0, 0, 0);
                }
                load_tile_rows<1, kKeys, RB>(tile, buf + kw * kTileBytes, kbase, kstride, n_keys, 0, lane, k_voff, kslot);
            };
            auto load_v = [&](int j, unsigned char *buf) __attribute__((always_inline)) {
                load_tile_rows<1, kKeys, RB>(first + KW * j, buf + kw * kTileBytes, vbase, vstride, n_keys, 0, lane, v_voff, vslot);
            };
            bf16x8_t qf[kAttD / 16];
            load_q<E4M3>(a, b, s_col, h_col, lg, qf);
            __asm__ volatile("" ::: "memory"); // Q first: waiting for it waits for no tile
            if (mine > 0)
            {
                load_k(0, k_a, s_a);
                load_v(0, v_a);
            }
            if (mine > 1)
            {
                load_k(1, k_b, s_b);
                load_v(1, v_b);
            }
            // each wave has the tree to itself, a node a lane
            Query query = Query::Sees;
            uint32_t tree = 0; // the nodes that the lane's column sees
            if constexpr (TREE)
            {
                static_assert(kAttColsPerWave <= 32, "nodes of a word");
                uint32_t mask;
                int32_t end;
                ancestors(parent, 0, S, lane, mask, end);
                tree = static_cast<uint32_t>(__shfl(static_cast<int>(mask), s_row, kWave));
                query = query_of(__shfl(end, s_row, kWave));
            }
            int v_off[kAttD / 32];
            if constexpr (E4M3)
                v_offsets8(lane, v_off);
            else
                v_offsets(lane, v_off);
            f32x16_t o[kAttD / 32];
#pragma unroll
            for (int dt = 0; dt < kAttD / 32; ++dt)
                o[dt] = f32x16_t{};
            float m = -__builtin_huge_valf(), l = 0.0f;
            const float scale2 = a.scale * kLog2e;

            auto step = [&](int j, unsigned char *kb, unsigned char *vb, uint32_t *sb) __attribute__((always_inline)) {
                const unsigned char *k_lds = kb + kw * kTileBytes, *v_lds = vb + kw * kTileBytes;
                float *vs = v_scale + (E4M3 ? kw * kWave : 0);
                // loads by age: K(j) with its scales, V(j), K(j + 1), V(j + 1)
                if (j + 1 < mine)
                    wait_loads<3 * kL + kS>();
                else
                    wait_loads<kL>();
                f32x16_t sacc[1];
                if constexpr (E4M3)
                {
                    // lane i has the scales of key i % 32: K's for the codes it reads of that key,
                    // V's go to LDS.  A row past the end may hold any byte; 254 keeps its scale
                    // finite.
                    const uint32_t pair_bytes = sb[kw * kWave + lane];
                    const uint32_t vbyte = pair_bytes >> 8;
                    vs[lane] = e4m3_scale(vbyte < 254u ? vbyte : 254u);
                    sacc[0] = qk_codes(k_lds, qf, li, lg, e4m3_scale(pair_bytes & 255u));
                }
                else
                    qk_tile<1>(k_lds, qf, li, lg, sacc, [](int) __attribute__((always_inline)) {});
                wait_loads<63>();
                if (j + 2 < mine)
                    load_k(j + 2, kb, sb);
                const int32_t key0 = (first + KW * j) * kKeys;
                const bool masked = key0 + kKeys > all_seen;
                uint32_t seen[1];
                if (masked)
                {
                    if constexpr (TREE)
                        seen[0] = tree_window(tree, key0 - context);
                    else
                        seen[0] = causal_window(key0, context + s_row);
                    mask_scores<1>(sacc, seen, lg);
                }
                bf16x8_t phi[1][2], plo[1][2];
                float alpha;
                if constexpr (E4M3)
                {
                    float4 w[4];
#pragma unroll
                    for (int q4 = 0; q4 < 4; ++q4)
                        w[q4] = *reinterpret_cast<const float4 *>(vs + 8 * q4 + 4 * lg);
                    alpha = softmax_tile<1>(sacc, scale2, m, l, phi, plo, [&](float p, int, int r) __attribute__((always_inline)) {
                        const float4 &x = w[r / 4];
                        return p * (r % 4 == 0 ? x.x : r % 4 == 1 ? x.y : r % 4 == 2 ? x.z : x.w);
                    });
                }
                else
                    alpha = softmax_tile<1>(sacc, scale2, m, l, phi, plo);
                rescale(o, alpha);
                // V(j), then K(j + 1), V(j + 1), K(j + 2)
                if (j + 2 < mine)
                    wait_loads<3 * kL + 2 * kS>();
                else if (j + 1 < mine)
                    wait_loads<2 * kL + kS>();
                else
                    wait_loads<0>();
                // one query sees every row up to its own, and past it only repeats of that row
                if (masked && S > 1 && has_nonfinite<E4M3>(v_lds, kTileBytes, lane))
                {
                    pv_careful<1>(
                        [&](int i) __attribute__((always_inline)) {
                            if constexpr (E4M3)
                                return as_bf8(decode8(read_v8(v_lds, v_off, i), 1.0f));
                            else
                                return read_v(v_lds, v_off, i);
                        },
                        [&](int key, int dt, int q4) __attribute__((always_inline)) {
                            return E4M3 ? v_values8(v_lds, lg, key, dt, q4) : v_values(v_lds, lg, key, dt, q4);
                        },
                        seen, phi, plo, o);
                }
                else if constexpr (E4M3)
                    pv_codes(v_lds, v_off, phi, plo, o);
                else
                {
                    bf16x8_t vq[kAhead + 1];
#pragma unroll
                    for (int x = 0; x < kAhead; ++x)
                        vq[x] = read_v(v_lds, v_off, x);
                    pv_tile<1>(v_lds, v_off, phi, plo, o, vq);
                }
                wait_loads<63>();
                if (j + 2 < mine)
                    load_v(j + 2, vb);
            };
            for (int j = 0; j < mine; j += 2)
            {
                step(j, k_a, v_a, s_a);
                if (j + 1 < mine)
                    step(j + 1, k_b, v_b, s_b);
            }
            const int64_t row = (b * a.S + s_col) * a.Hq + h_col;
            const auto sees = [&](int32_t key) __attribute__((always_inline)) {
                if constexpr (TREE)
                    return key < context || (tree >> ((key - context) & 31) & 1u) != 0;
                else
                    return key <= context + s_row;
            };
            const auto put_dims = [&](int dt, int first, f32x16_t part, float inv, float sum) __attribute__((always_inline)) {
                if constexpr (!E4M3)
                    see_infinities(vbase, vstride, k_begin, k_end, dt, lane, col_ok && query == Query::Sees && sum == sum, sees, part);
                if (col_ok)
                    store_dims<KW == 8 ? 2 : 4>(a, split, sp, row, dt, first, lg, part, inv, sum, query);
            };
            const auto put_ml = [&](float mx, float sum) __attribute__((always_inline)) {
                if (split && col_ok)
                    store_ml(a, sp, row, mx, sum, query);
            };
            if constexpr (KW == 1)
            {
#pragma unroll
                for (int dt = 0; dt < kAttD / 32; ++dt)
                    put_dims(dt, 0, o[dt], 1.0f / l, l);
                if (lg == 0)
                    put_ml(m, l);
            }
            else
            {
                __syncthreads(); // every wave is done with its tiles
                merge_groups<1, KW>(k_a, k_b, v_a, v_b, 0, kw, li, lg, o, m, l, put_dims, put_ml);
            }
        }

        // ---- more columns ---------------------------------------------------------------

        // As the block kernel of the causal bf16 attention: CW waves side by side over the
        // columns, KW groups of them dividing the keys, the P V product of a tile beside
        // the S^T product of the next; with a mask of its own and a length for each
        // sequence.
        //   bf16: two K and two V buffers, filled straight from memory, one barrier a
        //   tile.
        //   e4m3: one K and one V buffer of bf16, filled from staged codes.  Each wave
        //   stages 16 rows of K and of V (2 KiB each, the same lanes that convert them, so
        //   no barrier stands between), a tile ahead.  When every wave is past a step's
        //   products both buffers are free, and K of the next tile and V of this one are
        //   converted into them: two barriers a tile, half the LDS for tiles and no
        //   registers for loads in flight (holding the codes in registers instead spilled
        //   or cost the second block of a CU).
        // What bounds it is the softmax beside the matrix instructions, as in the bf16
        // attention.  512 queries over 8192 rows, 32 / 8 heads, e4m3, in 4 slices: 95 to 101 us
        // and 8 for the merge, together 610 to 640 TFLOP/s of the products, matrix cores busy
        // 44%.  16
        // ragged trees of 64 nodes over up to 4160 bf16 rows, 40 / 8 heads: 116 to 122 us, 440
        // to 465 TFLOP/s, 384 blocks of unequal length, two to a CU.  Four groups with 64 columns
        // are for few blocks (4 trees of 64 nodes over 2000 rows: 38.4 us, 40.7 with 128
        // columns) and lose where there are many (64 of 16 nodes over 1000: 49.2 and 43.2).
        template <int CW, int KW, int HH, bool E4M3, bool TREE>
        __global__ __launch_bounds__(CW *KW *kWave, 2) void cache_block_kernel(CacheArgs a)
        {
            const int g = a.g;
            constexpr int kBlockCols = 32 * CW;
            constexpr int kKeys = 32 * HH;
            constexpr int kTileBytes = kKeys * kRowBytes;
            constexpr int kWaves = CW * KW;
            constexpr int kRows = kKeys / CW, kCodeLoads = kRows / 8, kCodeBytes = kRows * kAttD; // of a wave
            static_assert(kRows == 16, "rows of a wave");
            // the groups' merge takes 4 KiB a wave of each buffer
            constexpr int kSecond = !E4M3 ? KW * kTileBytes : KW > 1 ? kWaves * 4096 : kWaves * kCodeBytes;
            __shared__ __attribute__((aligned(16))) unsigned char k_a[KW * kTileBytes];
            __shared__ __attribute__((aligned(16))) unsigned char k_b[kSecond]; // e4m3: the staged codes
            __shared__ __attribute__((aligned(16))) unsigned char v_a[KW * kTileBytes];
            __shared__ __attribute__((aligned(16))) unsigned char v_b[kSecond];
            __shared__ uint32_t k_scales[E4M3 ? kWaves * kWave : 1];
            __shared__ uint32_t v_scales[E4M3 ? kWaves * kWave : 1];
            __shared__ TreeMasks<TREE> tree;

            const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
            const int cw = wave % CW, kw = wave / CW;
            const int lane = threadIdx.x % kWave;
            const int li = lane % 32, lg = lane / 32;
            // KV heads run fastest, so that with a multiple of 8 of them the blocks of a pair
            // meet on one XCD, whose L2 holds its K and V.  Slices outermost: those of whole
            // length first, and a CU's two blocks are of different ones (6 trees of 200 nodes
            // over up to 5000 rows in 4 slices 74 us, 112 with a sequence's slices side by
            // side).  A tree's query blocks are equally long, but a last one of fewer columns
            // is lighter, and those come after all others; causal ones go longest first.
            int32_t sp, qb, kvh;
            int64_t b;
            if constexpr (TREE)
            {
                int32_t unit = static_cast<int32_t>(blockIdx.x);
                kvh = unit % a.by_hkv;
                unit = unit / a.by_hkv;
                const int32_t whole = static_cast<int32_t>(a.S) * g / kBlockCols;
                const int32_t light = unit - a.B * a.splits * whole;
                qb = light >= 0 ? whole : unit % a.by_qblocks;
                unit = light >= 0 ? light : unit / a.by_qblocks;
                sp = unit / a.by_b;
                b = unit % a.by_b;
            }
            else
            {
                const int32_t pair = static_cast<int32_t>(blockIdx.x) % a.by_pairs, rest = static_cast<int32_t>(blockIdx.x) / a.by_pairs;
                sp = rest / a.by_qblocks;
                qb = a.qblocks - 1 - rest % a.by_qblocks;
                kvh = pair % a.by_hkv;
                b = pair / a.by_hkv;
            }
            const int32_t S = static_cast<int32_t>(a.S);
            const int32_t n_cols = S * g;
            const int32_t block_col = qb * kBlockCols;
            const int32_t block_end = n_cols - block_col > kBlockCols ? block_col + kBlockCols : n_cols;
            const int32_t s_last = (block_end - 1) / a.by_g;
            bool bad;
            const int32_t n = sequence_rows(a, b, bad);
            const int32_t context = n - S;
            // rows the block's queries see between them
            const int32_t n_keys = n == 0 || TREE ? n : context + s_last + 1;
            if (n_keys <= 0)
            {
                if (sp == 0)
                    fill_columns(a, b, kvh, block_col, block_end, bad, threadIdx.x, kWaves * kWave);
                return;
            }
            const int64_t slice_begin = static_cast<int64_t>(sp) * a.split_keys;
            if (slice_begin >= n_keys)
                return;
            const int32_t k_begin = static_cast<int32_t>(slice_begin);
            const bool split = n_keys > a.split_keys;
            const int32_t k_end = n_keys - k_begin < a.split_keys ? n_keys : k_begin + a.split_keys;
            // tiles of the block [tile0, tile_end); this group's: first, first + KW, ...
            const int tile_end = (k_end + kKeys - 1) / kKeys;
            const int tile0 = k_begin / kKeys;
            const int first = tile0 + kw;
            const int steps = (tile_end - tile0 + KW - 1) / KW;
            const int mine = first < tile_end ? (tile_end - first + KW - 1) / KW : 0;

            int32_t parent = 0;
            if constexpr (TREE)
            {
                static_assert(kWaves * kWave >= kTreeMaxNodes, "a thread a node");
                const int32_t node = static_cast<int32_t>(threadIdx.x);
                parent = a.parents[b * a.parents_stride + (node < S ? node : S - 1)];
            }
            // this lane's column
            const int32_t wave_col = block_col + 32 * cw;
            const int32_t col = wave_col + li;
            const bool col_ok = col < n_cols;
            const int32_t s_col = col / a.by_g;
            const int h_col = kvh * g + col % a.by_g;
            const int32_t s_row = col_ok ? s_col : S - 1;
            const bool wave_active = wave_col < n_cols;
            // rows that every query of the wave sees
            const int32_t all_seen = TREE ? context : context + wave_col / a.by_g + 1;

            constexpr int64_t kElement = E4M3 ? 1 : 2;
            const unsigned char *kbase = static_cast<const unsigned char *>(a.k) + (b * a.ks0 + kvh * a.ks2) * kElement;
            const unsigned char *vbase = static_cast<const unsigned char *>(a.v) + (b * a.vs0 + kvh * a.vs2) * kElement;
            const uint8_t *sbase = a.scales + 2 * (b * a.ss0 + kvh * a.ss2);
            const int32_t kstride = static_cast<int32_t>(a.ks1 * kElement), vstride = static_cast<int32_t>(a.vs1 * kElement);
            const auto kslot = [](int r, int c) __attribute__((always_inline)) { return k_slot(r, c); };
            const auto vslot = [](int r, int c) __attribute__((always_inline)) { return v_slot(r, c); };
            // bf16: rows straight into a tile
            int32_t k_voff[Staging<CW, kKeys>::kLoads], v_voff[Staging<CW, kKeys>::kLoads];
            if constexpr (!E4M3)
            {
                tile_offsets<CW, kKeys>(cw, lane, kstride, kslot, k_voff);
                tile_offsets<CW, kKeys>(cw, lane, vstride, vslot, v_voff);
            }
            auto load_k = [&](int tile, unsigned char *buf) __attribute__((always_inline)) {
                load_tile_rows<CW, kKeys>(tile, buf + kw * kTileBytes, kbase, kstride, n_keys, cw, lane, k_voff, kslot);
            };
            auto load_v = [&](int tile, unsigned char *buf) __attribute__((always_inline)) {
                load_tile_rows<CW, kKeys>(tile, buf + kw * kTileBytes, vbase, vstride, n_keys, cw, lane, v_voff, vslot);
            };
            // e4m3: the wave's rows kRows cw .. + 15 of a tile, eight lanes a row of codes; a
            // lane's 16 codes land at 16 * lane and go to chunks 2 (lane % 8) and the next
            auto stage = [&](int tile, const unsigned char *base, unsigned char *codes, uint32_t *scales) __attribute__((always_inline)) {
                const int32_t row0 = tile * kKeys + kRows * cw, end = n_keys - 1;
                // based at the tile's first row, which the sequence has; rows past its end
                // repeat the last
                const int32_t key0 = tile * kKeys;
                auto past = [&](int32_t r) __attribute__((always_inline)) { return (row0 + r < end ? row0 + r : end) - key0; };
                __builtin_amdgcn_raw_ptr_buffer_load_lds(tile_rsrc(sbase + 2 * static_cast<int64_t>(key0)),
                                                         (lds_void_t *)(scales + wave * kWave), 2, 2 * past(lane % 16), 0, 0, 0);
                const __amdgpu_buffer_rsrc_t rs = tile_rsrc(base + static_cast<int64_t>(key0) * kAttD);
#pragma unroll
                for (int x = 0; x < kCodeLoads; ++x)
                    dma16(rs, past(8 * x + lane / 8) * kAttD + 16 * (lane % 8), codes + wave * kCodeBytes + x * 1024);
            };
            auto convert = [&](const unsigned char *codes, const uint32_t *scales, int shift, unsigned char *buf, auto slot)
                __attribute__((always_inline)) {
#pragma unroll
                for (int x = 0; x < kCodeLoads; ++x)
                {
                    const uint4 c = *reinterpret_cast<const uint4 *>(codes + wave * kCodeBytes + x * 1024 + 16 * lane);
                    const uint32_t byte = (scales[wave * kWave + 8 * x + lane / 8] >> shift) & 255u;
                    // a row past the end may hold any byte; 254 keeps its scale finite
                    const float scale = e4m3_scale(byte < 254u ? byte : 254u);
                    const int r = kRows * cw + 8 * x + lane / 8;
                    unsigned char *row = buf + kw * kTileBytes + r * kRowBytes;
                    *reinterpret_cast<Vec8 *>(row + 16 * slot(r, 2 * (lane % 8))) = decode8(make_uint2(c.x, c.y), scale);
                    *reinterpret_cast<Vec8 *>(row + 16 * slot(r, 2 * (lane % 8) + 1)) = decode8(make_uint2(c.z, c.w), scale);
                }
            };
            bf16x8_t qf[kAttD / 16];
            load_q<false>(a, b, s_col, h_col, lg, qf);
            int v_off[kAttD / 32];
            v_offsets(lane, v_off);
            f32x16_t o[kAttD / 32];
#pragma unroll
            for (int dt = 0; dt < kAttD / 32; ++dt)
                o[dt] = f32x16_t{};
            float m = -__builtin_huge_valf(), l = 0.0f;
            const float scale2 = a.scale * kLog2e;
            bf16x8_t phi[HH][2], plo[HH][2]; // P of the tile whose P V is still to be issued
            bool masked = false;             // whether that is a masked tile

            // which of a tile's keys the lane's column sees
            auto seen_keys = [&](int32_t key0, uint32_t (&seen)[HH]) __attribute__((always_inline)) {
#pragma unroll
                for (int hh = 0; hh < HH; ++hh)
                {
                    if constexpr (TREE)
                        seen[hh] = tree_window(tree.mask[s_row], key0 + 32 * hh - context);
                    else
                        seen[hh] = causal_window(key0 + 32 * hh, context + s_row);
                }
            };
            // the careful P V of the previous tile, if it needs it
            auto careful = [&](const unsigned char *v_lds, int32_t key0) __attribute__((always_inline)) {
                if (!masked || !has_nonfinite<false>(v_lds, kTileBytes, lane))
                    return false;
                uint32_t seen[HH];
                seen_keys(key0, seen);
                pv_careful<HH>([&](int i) __attribute__((always_inline)) { return read_v(v_lds, v_off, i); },
                               [&](int key, int dt, int q4) __attribute__((always_inline)) {
                                   return v_values(v_lds, lg, key, dt, q4);
                               },
                               seen, phi, plo, o);
                return true;
            };
            auto pv = [&](const unsigned char *v_lds, bf16x8_t (&vq)[kAhead + 1]) __attribute__((always_inline)) {
                pv_tile<HH>(v_lds, v_off, phi, plo, o, vq);
            };
            // The products of a step: S^T of this tile, P V of the previous one (WITH_PV).
            auto products = [&](auto with_pv, int32_t key0, const unsigned char *k_lds, const unsigned char *v_lds,
                                f32x16_t (&sacc)[HH]) __attribute__((always_inline)) {
                constexpr bool kPv = decltype(with_pv)::value;
                bool done = !kPv;
                if constexpr (kPv)
                    done = careful(v_lds, key0 - KW * kKeys);
                __builtin_amdgcn_s_setprio(1);
                bf16x8_t vq[kAhead + 1];
                qk_tile<HH>(k_lds, qf, li, lg, sacc, [&](int x) __attribute__((always_inline)) {
                    if constexpr (kPv)
                        vq[x] = read_v(v_lds, v_off, x);
                });
                masked = key0 + kKeys > all_seen;
                if (masked)
                {
                    uint32_t seen[HH];
                    seen_keys(key0, seen);
                    mask_scores<HH>(sacc, seen, lg);
                }
                if constexpr (kPv)
                    if (!done)
                        pv(v_lds, vq);
                __builtin_amdgcn_s_setprio(0);
            };
            auto softmax = [&](const f32x16_t (&sacc)[HH]) __attribute__((always_inline)) {
                const float alpha = softmax_tile<HH>(sacc, scale2, m, l, phi, plo);
                // o holds the tiles before this one at the previous reference
                rescale(o, alpha);
            };
            auto masks = [&]() __attribute__((always_inline)) {
                if constexpr (TREE)
                    tree_masks(tree, parent, S, wave, lane);
            };
            using no_pv = std::integral_constant<bool, false>;
            using with_pv = std::integral_constant<bool, true>;
            if constexpr (E4M3)
            {
                auto step = [&](auto pv_too, int j) __attribute__((always_inline)) {
                    const bool active = wave_active && (KW == 1 || j < mine);
                    f32x16_t sacc[HH];
                    if (active)
                        products(pv_too, (first + KW * j) * kKeys, k_a + kw * kTileBytes, v_a + kw * kTileBytes, sacc);
                    wait_loads<0>();
                    __syncthreads(); // every wave is past the products: both tiles are free
                    if (j + 1 < mine)
                        convert(k_b, k_scales, 0, k_a, kslot);
                    if (j < mine)
                        convert(v_b, v_scales, 8, v_a, vslot);
                    wait_loads<63>(); // the staged codes are read
                    if (j + 2 < mine)
                        stage(first + KW * (j + 2), kbase, k_b, k_scales);
                    if (j + 1 < mine)
                        stage(first + KW * (j + 1), vbase, v_b, v_scales);
                    if (active)
                        softmax(sacc);
                    __syncthreads();
                };
                if (mine > 0)
                {
                    stage(first, kbase, k_b, k_scales);
                    stage(first, vbase, v_b, v_scales);
                }
                masks();
                wait_loads<0>();
                if (mine > 0)
                    convert(k_b, k_scales, 0, k_a, kslot);
                wait_loads<63>();
                if (mine > 1)
                    stage(first + KW, kbase, k_b, k_scales);
                __syncthreads();
                step(no_pv{}, 0);
                for (int j = 1; j < steps; ++j)
                    step(with_pv{}, j);
            }
            else
            {
                // K of the next tile loads while this one is computed, V of it after the
                // barrier, into the buffer the step has finished with
                auto step = [&](auto pv_too, int j, unsigned char *k_cur, unsigned char *k_next, unsigned char *v_prev)
                    __attribute__((always_inline)) {
                    const int tile = first + KW * j;
                    if (j + 1 < mine)
                        load_k(tile + KW, k_next);
                    if (wave_active && (KW == 1 || j < mine))
                    {
                        f32x16_t sacc[HH];
                        products(pv_too, tile * kKeys, k_cur + kw * kTileBytes, v_prev + kw * kTileBytes, sacc);
                        softmax(sacc);
                    }
                    wait_loads<0>();
                    __syncthreads();
                    if (j + 1 < mine)
                        load_v(tile + KW, v_prev);
                };
                if (mine > 0)
                {
                    load_k(first, k_a);
                    load_v(first, v_a);
                }
                masks();
                wait_loads<0>();
                __syncthreads();
                // V of step j sits in v_a when j is even, else in v_b
                step(no_pv{}, 0, k_a, k_b, v_b);
                for (int j = 1; j < steps; j += 2)
                {
                    step(with_pv{}, j, k_b, k_a, v_a);
                    if (j + 1 < steps)
                        step(with_pv{}, j + 1, k_a, k_b, v_b);
                }
            }
            if (wave_active && mine > 0)
            {
                const unsigned char *v_lds = (E4M3 || (mine - 1) % 2 == 0 ? v_a : v_b) + kw * kTileBytes;
                if (!careful(v_lds, (first + KW * (mine - 1)) * kKeys))
                {
                    bf16x8_t vq[kAhead + 1];
#pragma unroll
                    for (int x = 0; x < kAhead; ++x)
                        vq[x] = read_v(v_lds, v_off, x);
                    pv(v_lds, vq);
                }
            }

            Query query = Query::Sees;
            if constexpr (TREE)
                query = query_of(tree.end[s_row]);
            const int64_t row = (b * a.S + s_col) * a.Hq + h_col;
            const auto sees = [&](int32_t key) __attribute__((always_inline)) {
                if constexpr (TREE)
                    return key < context || (tree.mask[s_row][1 + (key - context) / 32] >> ((key - context) & 31) & 1u) != 0;
                else
                    return key <= context + s_row;
            };
            const auto put_dims = [&](int dt, int first, f32x16_t part, float inv, float sum) __attribute__((always_inline)) {
                if constexpr (!E4M3)
                    see_infinities(vbase, vstride, k_begin, k_end, dt, lane, col_ok && query == Query::Sees && sum == sum, sees, part);
                if (col_ok)
                    store_dims<KW == 8 ? 2 : 4>(a, split, sp, row, dt, first, lg, part, inv, sum, query);
            };
            const auto put_ml = [&](float mx, float sum) __attribute__((always_inline)) {
                if (split && col_ok)
                    store_ml(a, sp, row, mx, sum, query);
            };
            if constexpr (KW == 1)
            {
#pragma unroll
                for (int dt = 0; dt < kAttD / 32; ++dt)
                    put_dims(dt, 0, o[dt], 1.0f / l, l);
                if (lg == 0)
                    put_ml(m, l);
            }
            else
            {
                __syncthreads(); // every wave is done with the V tiles
                merge_groups<CW, KW>(k_a, k_b, v_a, v_b, cw, kw, li, lg, o, m, l, put_dims, put_ml);
            }
        }

        // ---- merging slices ---------------------------------------------------------------

        struct MergeShape
        {
            Divisor by_hq, by_s, by_split_keys;
            int32_t last_col; // of a query block (its columns are a power of two)
        };

        // How many slices hold a query row's keys; 0: its query block wrote the result.
        // With several positions a row takes the slices its own keys reach (in the others of
        // its query block all its scores are masked).
        __device__ __forceinline__ int row_slices(const CacheArgs &a, const MergeShape &m, int64_t row)
        {
            const int32_t r32 = static_cast<int32_t>(row), bs = r32 / m.by_hq, h = r32 - bs * a.Hq, b = bs / m.by_s;
            const int32_t s = bs - b * static_cast<int32_t>(a.S);
            bool bad;
            const int32_t n = sequence_rows(a, b, bad);
            if (n == 0)
                return 0;
            int32_t own = n, block = n; // rows that this query's slices and its block's reach
            if (a.parents == nullptr)
            {
                const int32_t col = s * a.g + h % a.by_g, last = (col | m.last_col) / a.by_g;
                const int32_t s_last = last < a.S ? last : static_cast<int32_t>(a.S) - 1;
                own = n - static_cast<int32_t>(a.S) + s + 1;
                block = own + s_last - s;
            }
            return block <= a.split_keys ? 0 : own <= 0 ? 1 : (own - 1) / m.by_split_keys + 1;
        }

        // Few rows, many slices: a block of four waves a row (32 rows of 32 slices 2.8 us,
        // 832 of 16 3.9).  Lane i of each wave reads
        // slice i's reference max and sum, wave w the unnormalised O^T of slices w, w + 4,
        // ..., all before any is used; weights 2^(m_i - max m), then sum w O / sum w l.
        constexpr int kMergeWaves = 4;
        constexpr int kMergeRound = kAttMaxSplits / kMergeWaves;

        __global__ __launch_bounds__(kMergeWaves *kWave) void cache_merge_block_kernel(CacheArgs a, MergeShape shape)
        {
            __shared__ float2 wave_acc[kMergeWaves][kWave];
            const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
            const int lane = threadIdx.x % kWave;
            const int64_t row = blockIdx.x;
            const int slices = row_slices(a, shape, row);
            if (slices == 0)
                return;
            float2 ml = make_float2(-__builtin_huge_valf(), 0.0f);
            if (lane < slices)
                ml = reinterpret_cast<const float2 *>(a.part_ml)[static_cast<int64_t>(lane) * a.rows + row];
            float2 v[kMergeRound];
#pragma unroll
            for (int u = 0; u < kMergeRound; ++u)
            {
                const int i = wave + kMergeWaves * u;
                if (i < slices)
                    v[u] = reinterpret_cast<const float2 *>(a.part_o + (static_cast<int64_t>(i) * a.rows + row) * kAttD)[lane];
            }
            float mx = ml.x;
#pragma unroll
            for (int off = kWave / 2; off > 0; off /= 2)
                mx = fmaxf(mx, __shfl_xor(mx, off, kWave));
            mx = mx == -__builtin_huge_valf() ? 0.0f : mx;
            const float w = lane < slices ? __builtin_amdgcn_exp2f(ml.x - mx) : 0.0f;
            float a0 = 0.0f, a1 = 0.0f;
#pragma unroll
            for (int u = 0; u < kMergeRound; ++u)
            {
                const int i = wave + kMergeWaves * u;
                if (i < slices)
                {
                    const float wi = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), i));
                    a0 += wi * v[u].x;
                    a1 += wi * v[u].y;
                }
            }
            const float lsum = group_sum<kWave>(w * ml.y);
            wave_acc[wave][lane] = make_float2(a0, a1);
            __syncthreads();
            if (wave != 0)
                return;
#pragma unroll
            for (int k = 1; k < kMergeWaves; ++k)
            {
                a0 += wave_acc[k][lane].x;
                a1 += wave_acc[k][lane].y;
            }
            const float inv = 1.0f / lsum;
            reinterpret_cast<uint32_t *>(a.out + row * kAttD)[lane] = lsum == 0.0f ? 0u : pack_rne(a0 * inv, a1 * inv);
        }

        // Many rows: 16 lanes a row, 8 dims a lane, four slices at a time; every lane works
        // the weights out for itself, so nothing is exchanged.  Memory bounds it: 16384 rows
        // of 4 slices 7.7 us, 38 MB at 5.0 TB/s.
        constexpr int kMergeSlices = 4;
        constexpr int kMergeRows = kBlock / 16;

        __global__ __launch_bounds__(kBlock) void cache_merge_rows_kernel(CacheArgs a, MergeShape shape)
        {
            const int64_t row = static_cast<int64_t>(blockIdx.x) * kMergeRows + threadIdx.x / 16;
            if (row >= a.rows)
                return;
            const int slices = row_slices(a, shape, row), d = 8 * (threadIdx.x % 16);
            if (slices == 0)
                return;
            float mx = -__builtin_huge_valf(), lsum = 0.0f, acc[8] = {};
            for (int i0 = 0; i0 < slices; i0 += kMergeSlices)
            {
                float2 ml[kMergeSlices];
                float4 v[kMergeSlices][2];
#pragma unroll
                for (int u = 0; u < kMergeSlices; ++u)
                    if (i0 + u < slices)
                    {
                        const int64_t at = static_cast<int64_t>(i0 + u) * a.rows + row;
                        ml[u] = reinterpret_cast<const float2 *>(a.part_ml)[at];
                        const float4 *po = reinterpret_cast<const float4 *>(a.part_o + at * kAttD + d);
                        v[u][0] = po[0];
                        v[u][1] = po[1];
                    }
#pragma unroll
                for (int u = 0; u < kMergeSlices; ++u)
                    if (i0 + u < slices)
                    {
                        const float m = fmaxf(mx, ml[u].x), m_use = m == -__builtin_huge_valf() ? 0.0f : m;
                        const float w0 = __builtin_amdgcn_exp2f(mx - m_use), w = __builtin_amdgcn_exp2f(ml[u].x - m_use);
                        lsum = lsum * w0 + ml[u].y * w;
                        const float e[8] = {v[u][0].x, v[u][0].y, v[u][0].z, v[u][0].w, v[u][1].x, v[u][1].y, v[u][1].z, v[u][1].w};
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            acc[j] = acc[j] * w0 + e[j] * w;
                        mx = m;
                    }
            }
            const float inv = 1.0f / lsum;
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                w[j] = lsum == 0.0f ? 0u : pack_rne(acc[2 * j] * inv, acc[2 * j + 1] * inv);
            uint2 *o = reinterpret_cast<uint2 *>(a.out + row * kAttD + d); // out is 8-byte aligned
            o[0] = make_uint2(w[0], w[1]);
            o[1] = make_uint2(w[2], w[3]);
        }

        int launch_merge(const char *what, const CacheArgs &a, int block_cols, hipStream_t stream)
        {
            if (a.splits > 1)
            {
                const MergeShape m{divisor(a.Hq), divisor(a.S), divisor(a.split_keys), block_cols - 1};
                if (a.rows <= kAttBlockMergeRows)
                    cache_merge_block_kernel<<<dim3(static_cast<unsigned>(a.rows)), dim3(kMergeWaves * kWave), 0, stream>>>(a, m);
                else
                    cache_merge_rows_kernel<<<dim3(static_cast<unsigned>(blocks_for(a.rows, kMergeRows))), dim3(kBlock), 0, stream>>>(a, m);
            }
            return check_launch(what);
        }

        template <int KW, bool E4M3, bool TREE>
        int launch_decode(const char *what, const CacheArgs &a, int64_t B, hipStream_t stream)
        {
            const int64_t blocks = B * a.Hkv * a.splits;
            if (!launch_fits(blocks, KW * kWave) || blocks > INT32_MAX)
                return set_error(Q3K_ERR_OVERFLOW, "%s grid is too large", what);
            cache_decode_kernel<KW, E4M3, TREE><<<dim3(static_cast<unsigned>(blocks)), dim3(KW * kWave), 0, stream>>>(a);
            return launch_merge(what, a, kAttColsPerWave, stream);
        }

        template <int CW, int KW, int HH, bool E4M3, bool TREE>
        int launch_block(const char *what, CacheArgs a, int64_t B, hipStream_t stream)
        {
            constexpr int kBlockCols = 32 * CW, kThreads = CW * KW * kWave;
            a.qblocks = static_cast<int32_t>(blocks_for(a.S * a.g, kBlockCols));
            const int64_t whole = a.S * a.g / kBlockCols;
            a.by_qblocks = divisor(!TREE ? a.qblocks : whole > 0 ? whole : 1);
            const int64_t blocks = B * a.Hkv * a.qblocks * a.splits;
            if (!launch_fits(blocks, kThreads) || blocks > INT32_MAX)
                return set_error(Q3K_ERR_OVERFLOW, "%s grid is too large", what);
            cache_block_kernel<CW, KW, HH, E4M3, TREE><<<dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0, stream>>>(a);
            return launch_merge(what, a, kBlockCols, stream);
        }

        template <bool E4M3, bool TREE>
        int launch_fast(const char *what, const CacheArgs &a, int64_t B, const CacheAttnPlan &p, hipStream_t stream)
        {
            if (p.decode_waves > 0)
            {
                if constexpr (E4M3)
                    if (p.decode_waves == 8)
                        return launch_decode<8, E4M3, TREE>(what, a, B, stream);
                return p.decode_waves == 1 ? launch_decode<1, E4M3, TREE>(what, a, B, stream)
                                           : launch_decode<4, E4M3, TREE>(what, a, B, stream);
            }
            return p.key_groups == 1 ? launch_block<4, 1, 2, E4M3, TREE>(what, a, B, stream)
                                     : launch_block<2, 4, 1, E4M3, TREE>(what, a, B, stream);
        }

        // Whether the matrix-core kernels take calls of these sizes: a position's columns in
        // one wave, tile ends counted in 32 bits.
        bool fast_sizes(int32_t Hq, int32_t Hkv, int32_t D, int64_t cached)
        {
            return D == kAttD && Hq / Hkv <= kAttColsPerWave && cached <= INT32_MAX - 4 * kAttKeyTile;
        }

        // Whether they take the call: rows and Q in 16-byte vectors, a tile's rows within
        // 32-bit byte offsets.
        bool fast(const CacheArgs &a, bool e4m3)
        {
            if (!fast_sizes(a.Hq, a.Hkv, a.D, a.cached))
                return false;
            if (!aligned16(a.q) || !aligned16(a.k) || !aligned16(a.v) || !aligned_to(a.out, 8))
                return false;
            if (e4m3)
                return aligned_to(a.scales, 2);
            const int64_t row_limit = (INT32_MAX - 2 * kAttD) / (2 * kAttKeyTile);
            for (const int64_t s : {a.ks0, a.ks1, a.ks2, a.vs0, a.vs1, a.vs2})
                if (s % 8 != 0)
                    return false;
            return a.ks3 == 1 && a.vs3 == 1 && a.ks1 <= row_limit && a.vs1 <= row_limit;
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

        int launch(const char *what, CacheArgs a, int64_t B, bool e4m3, void *workspace, int64_t workspace_bytes,
                   hipStream_t stream)
        {
            a.scale = 1.0f / __builtin_sqrtf(static_cast<float>(a.D));
            a.rows = B * a.S * a.Hq;
            if (fast(a, e4m3))
            {
                const bool tree = a.parents != nullptr, ragged = a.lengths != nullptr;
                CacheAttnPlan p = plan_cache_attention(B, a.S, a.Hq, a.Hkv, a.cached, e4m3, tree, ragged, true);
                if (p.bytes > 0 && (workspace == nullptr || !aligned16(workspace) || workspace_bytes < p.bytes))
                    p = plan_cache_attention(B, a.S, a.Hq, a.Hkv, a.cached, e4m3, tree, ragged, false);
                a.B = static_cast<int32_t>(B);
                a.ordered = ragged && B > 1 && p.splits == 1 && p.decode_waves > 0;
                a.splits = p.splits;
                a.split_keys = p.split_keys;
                a.g = a.Hq / a.Hkv;
                a.by_g = divisor(a.g);
                a.by_hkv = divisor(a.Hkv);
                a.by_b = divisor(B);
                a.by_pairs = divisor(B * a.Hkv);
                a.part_o = static_cast<float *>(workspace);
                a.part_ml = p.splits > 1 ? a.part_o + static_cast<int64_t>(p.splits) * a.rows * kAttD : nullptr;
                if (tree)
                    return e4m3 ? launch_fast<true, true>(what, a, B, p, stream) : launch_fast<false, true>(what, a, B, p, stream);
                return launch_fast<true, false>(what, a, B, p, stream);
            }
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

extern "C" int64_t q3k_cache_attention_workspace_bytes(int64_t B, int64_t S, int32_t Hq, int32_t Hkv, int32_t D, int64_t cached)
{
    if (B <= 0 || S <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 || cached <= 0 || !q3k::fast_sizes(Hq, Hkv, D, cached) ||
        S > INT64_MAX / B || B * S > INT64_MAX / Hq || B * S * Hq > INT32_MAX)
        return 0;
    return q3k::cache_attention_workspace_bytes(B, S, Hq, Hkv, cached);
}
