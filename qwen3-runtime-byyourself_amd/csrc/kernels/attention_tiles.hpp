// Tile operations of the matrix-core attention kernels (attention.hip,
// cache_attention.hip): K and V rows from HBM into LDS, S^T = K Q^T, the online
// softmax, O^T += V^T P^T.  The layout and the mathematics stand in
// attention.hip.
#pragma once

#include <type_traits>

#include "dispatch.hpp"
#include "q3k_common.hpp"

namespace q3k
{
    typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
    typedef float f32x16_t __attribute__((ext_vector_type(16)));

    typedef __bf16 bf16x4_t __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) bf16x4_t lds_bf16x4_t;
    typedef __attribute__((address_space(3))) void lds_void_t;

    constexpr int kAttD = kAttHeadDim;
    constexpr int kRowBytes = kAttD * 2;                  // one K or V row in LDS
    constexpr int kAhead = 2;                             // LDS fragment reads in flight ahead of use
    constexpr float kLazyMax = 8.0f;                      // log2 headroom before the softmax reference moves
    constexpr float kLog2e = 1.4426950408889634f;

    __device__ __forceinline__ bf16x8_t as_bf8(const Vec8 &v) { return __builtin_bit_cast(bf16x8_t, v); }

    // LDS chunk (16 bytes) holding chunk c of K row r / V row r of a tile.
    // K: lanes 0..31 of a fragment read read rows r..r+31 at one chunk;
    // any 16 consecutive rows put it in 16 different chunk positions.
    // V: a transpose read takes 4 rows x 32 bytes per 16 lanes; rows
    // 4 apart share a bank set.
    __device__ __forceinline__ int k_slot(int r, int c) { return c ^ (r & 15); }
    __device__ __forceinline__ int v_slot(int r, int c) { return c ^ (4 * (r & 3)); }

    // Buffer resource over [base, base + 2 GiB): raw (stride 0), so the
    // offsets the loads give are byte offsets from base.
    __device__ __forceinline__ __amdgpu_buffer_rsrc_t tile_rsrc(const void *base)
    {
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(base), 0, 0x7fffffff, 0x00020000);
    }

    // 16 bytes per lane from rsrc + voffset into LDS at lds_wave + 16 * lane
    // (buffer_load_dwordx4 ... lds: no registers, the wave's LDS base in M0)
    __device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t rsrc, int32_t voffset, unsigned char *lds_wave)
    {
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_void_t *)lds_wave, 16, voffset, 0, 0, 0);
    }

    // max / sum of x over lanes l and l ^ 32, in every lane (one VALU swap,
    // no LDS): after the swap one operand is x and the other its partner
    __device__ __forceinline__ float pair_max(float x)
    {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    }
    __device__ __forceinline__ float pair_sum(float x)
    {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        return __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }

    // Waits until at most N of the wave's vector loads are in flight and its
    // LDS reads are done (s_waitcnt vmcnt(N) lgkmcnt(0); 63: the LDS reads only).
    template <int N>
    __device__ __forceinline__ void wait_loads()
    {
        static_assert(N >= 0 && N < 64, "vmcnt");
        __asm__ volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | ((N >> 4) << 14));
        __asm__ volatile("" ::: "memory");
    }

    // ---- tile operations shared by the kernels ------------------------------

    // Loading a key tile's K (or V) rows of RB bytes (256 of bf16, 128 of e4m3
    // codes) into LDS by CW waves: wave cw fills rows (KEYS / CW) cw .. of a
    // buffer, 1024 / RB rows per load; lane j lands in slot j % (RB / 16) of row
    // j / (RB / 16) and so fetches the chunk that slot holds.  A tile's loads
    // address from a buffer resource based at its first key, so the per-lane
    // byte offsets (tile_offsets) stay fixed: 32-bit, checked by the launcher.
    // Rows past n_keys repeat the last key (readable data, later masked or
    // weighted by zero).
    template <int CW, int KEYS, int RB = kRowBytes>
    struct Staging
    {
        static constexpr int kRows = KEYS / CW;                // rows of a tile per wave
        static constexpr int kChunks = RB / 16;                // 16-byte chunks of a row
        static constexpr int kRowsPerLoad = kWave / kChunks;   // rows one wave-wide 16-byte load fills
        static constexpr int kLoads = kRows / kRowsPerLoad;    // loads per wave per K (or V) tile
    };

    template <int CW, int KEYS, int RB = kRowBytes, typename Slot>
    __device__ __forceinline__ void tile_offsets(int cw, int lane, int32_t byte_stride, Slot slot,
                                                 int32_t (&voff)[Staging<CW, KEYS, RB>::kLoads])
    {
        using St = Staging<CW, KEYS, RB>;
        const int st_row = St::kRows * cw + lane / St::kChunks;
#pragma unroll
        for (int x = 0; x < St::kLoads; ++x)
        {
            const int r = st_row + St::kRowsPerLoad * x;
            voff[x] = r * byte_stride + 16 * slot(r, lane % St::kChunks);
        }
    }

    // base: the first key's row, byte_stride bytes between rows.
    template <int CW, int KEYS, int RB = kRowBytes, typename Slot>
    __device__ __forceinline__ void load_tile_rows(int tile, unsigned char *buf, const void *base, int32_t byte_stride,
                                                   int32_t n_keys, int cw, int lane,
                                                   const int32_t (&voff)[Staging<CW, KEYS, RB>::kLoads], Slot slot)
    {
        using St = Staging<CW, KEYS, RB>;
        const int32_t key0 = tile * KEYS;
        const __amdgpu_buffer_rsrc_t rs =
            tile_rsrc(static_cast<const unsigned char *>(base) + static_cast<int64_t>(key0) * byte_stride);
        unsigned char *dst = buf + St::kRows * cw * RB;
        if (key0 + KEYS <= n_keys)
        {
#pragma unroll
            for (int x = 0; x < St::kLoads; ++x)
                dma16(rs, voff[x], dst + St::kRowsPerLoad * x * RB);
        }
        else
        {
            const int last = n_keys - 1 - key0;
            const int st_row = St::kRows * cw + lane / St::kChunks;
#pragma unroll
            for (int x = 0; x < St::kLoads; ++x)
            {
                const int r = st_row + St::kRowsPerLoad * x;
                const int rr = r < last ? r : last;
                dma16(rs, rr * byte_stride + 16 * slot(r, lane % St::kChunks), dst + St::kRowsPerLoad * x * RB);
            }
        }
    }

    // Per-lane LDS byte offsets of the V transpose reads: the lanes of each
    // 16 give rows 4 lg + j / 4 (+ 8 per 8-key step) and 4 dims
    // 32 dt + 16 ((lane / 16) % 2) + 4 (j % 4) .. + 3, and each lane gets 4
    // consecutive keys of one dim (dim 32 dt + lane % 32).
    __device__ __forceinline__ void v_offsets(int lane, int (&v_off)[kAttD / 32])
    {
        const int tj = lane % 16, lg = lane / 32;
        const int v_row = 4 * lg + tj / 4;
#pragma unroll
        for (int dt = 0; dt < kAttD / 32; ++dt)
            v_off[dt] = v_row * kRowBytes + 16 * v_slot(v_row, 4 * dt + 2 * ((lane / 16) % 2) + (tj % 4) / 2) +
                        8 * (tj % 2);
    }

    // The V^T fragment of P V step i (key chunk i / 4, dims 32 (i % 4) .. + 31):
    // keys 16 (i / 4) + 8 t + 4 lg + 0..3 in elements 4 t .. 4 t + 3, the keys
    // of the P^T elements this lane holds.
    __device__ __forceinline__ bf16x8_t read_v(const unsigned char *v_lds, const int (&v_off)[kAttD / 32], int i)
    {
        const unsigned char *vp = v_lds + v_off[i % 4] + 16 * (i / 4) * kRowBytes;
        const bf16x4_t v0 = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4_t *)(vp));
        const bf16x4_t v1 = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4_t *)(vp + 8 * kRowBytes));
        return __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7);
    }

    // S^T = K Q^T for the 32 HH keys of a tile (sacc[hh]: keys 32 hh .. + 31).
    // The K fragment reads run kAhead steps ahead of the MFMAs that use them.
    // When its own reads have run out it calls next(x), x < kAhead, for the
    // reads of the product that follows.
    template <int HH, typename Next>
    __device__ __forceinline__ void qk_tile(const unsigned char *k_lds, const bf16x8_t (&qf)[kAttD / 16], int li,
                                            int lg, f32x16_t (&sacc)[HH], Next next)
    {
        auto read_k = [&](int c, int hh) __attribute__((always_inline)) {
            return *reinterpret_cast<const Vec8 *>(k_lds + (32 * hh + li) * kRowBytes +
                                                   16 * k_slot(li, 2 * c + lg));
        };
#pragma unroll
        for (int hh = 0; hh < HH; ++hh)
            sacc[hh] = f32x16_t{};
        Vec8 kq[kAhead + 1][HH];
#pragma unroll
        for (int c = 0; c < kAhead; ++c)
#pragma unroll
            for (int hh = 0; hh < HH; ++hh)
                kq[c][hh] = read_k(c, hh);
#pragma unroll
        for (int c = 0; c < kAttD / 16; ++c)
        {
            if (c + kAhead < kAttD / 16)
#pragma unroll
                for (int hh = 0; hh < HH; ++hh)
                    kq[(c + kAhead) % (kAhead + 1)][hh] = read_k(c + kAhead, hh);
            if (c + kAhead >= kAttD / 16)
                next(c + kAhead - kAttD / 16);
            __builtin_amdgcn_sched_barrier(0); // keep the reads ahead of these MFMAs
#pragma unroll
            for (int hh = 0; hh < HH; ++hh)
                sacc[hh] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf8(kq[c % (kAhead + 1)][hh]), qf[c], sacc[hh],
                                                                   0, 0, 0);
        }
    }

    // A weight as it meets V (softmax_tile): unchanged.
    struct PlainWeight
    {
        __device__ __forceinline__ float operator()(float p, int, int) const { return p; }
    };

    // Online softmax of one tile for the lane's column: the weights, split
    // into bf16 high parts and remainders, go to phi / plo, and m, l are
    // updated.  The weights are taken relative to a reference m that moves
    // only when a tile's max exceeds it by more than kLazyMax (log2 units):
    // they stay below 2^kLazyMax, and the rescale of the output is left for
    // the rare tiles that move it.  Returns that rescale factor (1 when m did
    // not move).  An all-masked column keeps m = -inf and weight 0.  The max
    // of the raw scores times the (positive) scale is the max of the scaled
    // ones.  weight(p, hh, r) is what V's values are multiplied by instead of p (V's
    // scale of that key, element r of half hh, where it has one).
    template <int HH, typename Weight = PlainWeight>
    __device__ __forceinline__ float softmax_tile(const f32x16_t (&sacc)[HH], float scale2, float &m, float &l,
                                                  bf16x8_t (&phi)[HH][2], bf16x8_t (&plo)[HH][2],
                                                  Weight weight = {})
    {
        float mloc = sacc[0][0];
#pragma unroll
        for (int hh = 0; hh < HH; ++hh)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                mloc = fmaxf(mloc, sacc[hh][r]);
        mloc = pair_max(mloc);
        const float m_tile = mloc * scale2;
        const bool move = m_tile > m + kLazyMax;
        const float m_new = move ? m_tile : m;
        const float m_use = m_new == -__builtin_huge_valf() ? 0.0f : m_new;
        const float alpha = move ? __builtin_amdgcn_exp2f(m - m_use) : 1.0f;
        float psum = 0.0f;
#pragma unroll
        for (int hh = 0; hh < HH; ++hh)
#pragma unroll
            for (int mm = 0; mm < 2; ++mm)
            {
                Vec8 h8, l8;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                {
                    const float x0 =
                        __builtin_amdgcn_exp2f(__builtin_fmaf(sacc[hh][8 * mm + 2 * j], scale2, -m_use));
                    const float x1 =
                        __builtin_amdgcn_exp2f(__builtin_fmaf(sacc[hh][8 * mm + 2 * j + 1], scale2, -m_use));
                    psum += x0;
                    psum += x1;
                    const float y0 = weight(x0, hh, 8 * mm + 2 * j), y1 = weight(x1, hh, 8 * mm + 2 * j + 1);
                    const uint32_t hp = pack_rne(y0, y1);
                    h8.d[j] = hp;
                    l8.d[j] = pack_rne(y0 - bf_lo(hp), y1 - bf_hi(hp));
                }
                phi[hh][mm] = as_bf8(h8);
                plo[hh][mm] = as_bf8(l8);
            }
        psum = pair_sum(psum);
        l = l * alpha + psum;
        m = m_new;
        return alpha;
    }

    // o *= alpha; multiplying by alpha == 1 changes nothing, so the wave
    // skips it when no lane needs it
    __device__ __forceinline__ void rescale(f32x16_t (&o)[kAttD / 32], float alpha)
    {
        if (__any(alpha != 1.0f))
        {
#pragma unroll
            for (int dt = 0; dt < kAttD / 32; ++dt)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    o[dt][r] *= alpha;
        }
    }

    // O^T += V^T P^T for one tile: step i covers the 16-key chunk i / 4
    // (hh = i / 8, mm = (i / 4) % 2) and dims 32 (i % 4) .. + 31.  The
    // transpose reads run kAhead steps ahead of the MFMAs that use them; the
    // first kAhead are in vq already.
    template <int HH>
    __device__ __forceinline__ void pv_tile(const unsigned char *v_lds, const int (&v_off)[kAttD / 32],
                                            const bf16x8_t (&phi)[HH][2], const bf16x8_t (&plo)[HH][2],
                                            f32x16_t (&o)[kAttD / 32], bf16x8_t (&vq)[kAhead + 1])
    {
#pragma unroll
        for (int i = 0; i < 8 * HH; ++i)
        {
            if (i + kAhead < 8 * HH)
                vq[(i + kAhead) % (kAhead + 1)] = read_v(v_lds, v_off, i + kAhead);
            __builtin_amdgcn_sched_barrier(0); // keep the reads ahead of these MFMAs
            const int dt = i % 4, hh = i / 8, mm = (i / 4) % 2;
            o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vq[i % (kAhead + 1)], phi[hh][mm], o[dt], 0, 0, 0);
            o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vq[i % (kAhead + 1)], plo[hh][mm], o[dt], 0, 0, 0);
        }
    }

    // The KW groups' partial results of a column meet in LDS, in the tile
    // buffers: dims 32 dt .. + 31 of all waves in buffer dt (4 KiB a wave, 16
    // bytes a lane, so lanes hit distinct banks).  Group kw then merges and
    // stores 4 / KW of the four parts, with eight groups half of one:
    // store_dims(part, first, O^T, 1 / sum, sum) for quarters first .. of the
    // part's elements, and one lane a column its reference max and sum: store_ml.
    template <int CW, int KW, typename StoreDims, typename StoreMl>
    __device__ __forceinline__ void merge_groups(unsigned char *b0, unsigned char *b1, unsigned char *b2,
                                                 unsigned char *b3, int cw, int kw, int li, int lg,
                                                 const f32x16_t (&o)[kAttD / 32], float m, float l,
                                                 StoreDims store_dims, StoreMl store_ml)
    {
        static_assert(kAttD / 32 == 4 && (4 % KW == 0 || KW == 8), "parts");
        constexpr int kParts = KW == 8 ? 1 : 4 / KW, kQuarters = KW == 8 ? 2 : 4;
        const int lane = 32 * lg + li, wave = kw * CW + cw;
        __shared__ float2 ml[KW][32 * CW];
        unsigned char *const bufs[4] = {b0, b1, b2, b3};
#pragma unroll
        for (int dt = 0; dt < 4; ++dt)
        {
            float4 *dst = reinterpret_cast<float4 *>(bufs[dt]) + wave * 4 * kWave;
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4)
                dst[q4 * kWave + lane] = {o[dt][4 * q4], o[dt][4 * q4 + 1], o[dt][4 * q4 + 2], o[dt][4 * q4 + 3]};
        }
        if (lg == 0)
            ml[kw][32 * cw + li] = make_float2(m, l);
        __syncthreads();
        float w[KW];
        float mx = -__builtin_huge_valf();
#pragma unroll
        for (int x = 0; x < KW; ++x)
            mx = fmaxf(mx, ml[x][32 * cw + li].x);
        const float m_use = mx == -__builtin_huge_valf() ? 0.0f : mx;
        float lsum = 0.0f;
#pragma unroll
        for (int x = 0; x < KW; ++x)
        {
            const float2 e = ml[x][32 * cw + li];
            w[x] = __builtin_amdgcn_exp2f(e.x - m_use);
            lsum += w[x] * e.y;
        }
        const float inv = 1.0f / lsum;
#pragma unroll
        for (int y = 0; y < kParts; ++y)
        {
            const int dt = KW == 8 ? kw / 2 : kw * kParts + y, first = KW == 8 ? 2 * (kw % 2) : 0;
            const unsigned char *buf = dt == 0 ? b0 : dt == 1 ? b1 : dt == 2 ? b2 : b3;
            f32x16_t r = f32x16_t{};
#pragma unroll
            for (int x = 0; x < KW; ++x)
            {
                const float4 *src = reinterpret_cast<const float4 *>(buf) + (x * CW + cw) * 4 * kWave;
#pragma unroll
                for (int q4 = 0; q4 < kQuarters; ++q4)
                {
                    const float4 e = src[(first + q4) * kWave + lane];
                    r[4 * q4] = __builtin_fmaf(w[x], e.x, r[4 * q4]);
                    r[4 * q4 + 1] = __builtin_fmaf(w[x], e.y, r[4 * q4 + 1]);
                    r[4 * q4 + 2] = __builtin_fmaf(w[x], e.z, r[4 * q4 + 2]);
                    r[4 * q4 + 3] = __builtin_fmaf(w[x], e.w, r[4 * q4 + 3]);
                }
            }
            store_dims(dt, first, r, inv, lsum);
        }
        if (lg == 0 && kw == 0)
            store_ml(mx, lsum);
    }
} // namespace q3k
