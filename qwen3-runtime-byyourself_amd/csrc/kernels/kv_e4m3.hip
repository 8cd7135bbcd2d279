// The e4m3 KV cache for gfx950: K and V rows quantised as they are appended,
// and read back as bf16.
//
// A row (one position, one KV head, D bf16 values x) is held as codes
// RNE_e4m3(x * 2^-e) with e the smallest integer >= -126 for which no finite
// |x| exceeds 448 * 2^e.  With a power-of-two scale both scalings are exact:
// the code's rounding is the only one, a value read back is a bf16 value, and
// the scale is an exponent byte.  Of |x| as a bf16 bit pattern a (exponent
// a >> 7, fraction a & 127), 448 = 1.75 * 2^8 gives the byte
// e + 127 = (a >> 7) - 8, one more where the fraction is past 96: (a + 31 >> 7)
// - 8, at least 1.  The largest |x| is a maximum of 15-bit integers; a row with
// an infinity or a NaN shows as one of 0x7f80 or more and is looked at again
// without them.
//
// What bounds both is memory.  A row of 64, 128 or 256 values takes 8, 16 or 32
// lanes of 8 values (one 16-byte load or store of bf16, 8 bytes of codes); K and
// V of a row go through the same lanes, so that both are in flight.
#include "kv_e4m3.hpp"

namespace q3k
{
    namespace
    {
        struct E4m3Shape
        {
            uint32_t rows; // B * positions * Hkv
            uint32_t S;    // positions of a sequence
            uint32_t Hkv;
            uint32_t D;
            int64_t seq_cap;
            int64_t start;
            const int32_t *starts; // append: first row of each sequence; read: its length
        };

        // Cache row of head h, position pos of sequence b, in rows of D codes.
        __device__ __forceinline__ int64_t cache_row(const E4m3Shape &s, uint32_t b, uint32_t h, int64_t pos)
        {
            return (static_cast<int64_t>(b) * s.Hkv + h) * s.seq_cap + pos;
        }

        // max over aligned groups of G lanes, in every lane
        template <int G>
        __device__ __forceinline__ uint32_t group_max(uint32_t v)
        {
            static_assert(G == 8 || G == 16 || G == 32, "lanes of a row");
            auto up = [&](uint32_t o) __attribute__((always_inline)) { v = v > o ? v : o; };
            up(dpp_u<kDppQuadXor1>(v));
            up(dpp_u<kDppQuadXor2>(v));
            up(dpp_u<kDppHalfMirror>(v));
            if constexpr (G >= 16)
                up(dpp_u<kDppMirror>(v));
            if constexpr (G >= 32)
            {
                const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
                v = r[0] > r[1] ? r[0] : r[1];
            }
            return v;
        }

        // The largest magnitude pattern of eight values, 0 for a value of `limit` or more.
        __device__ __forceinline__ uint32_t max_pattern(const Vec8 &x, uint32_t limit)
        {
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i)
            {
                const uint32_t lo = x.d[i] & 0x7fffu, hi = (x.d[i] >> 16) & 0x7fffu;
                const uint32_t l = lo < limit ? lo : 0u, h = hi < limit ? hi : 0u;
                m = m > l ? m : l;
                m = m > h ? m : h;
            }
            return m;
        }

        __device__ __forceinline__ uint32_t scale_byte(uint32_t pattern)
        {
            const int32_t e = static_cast<int32_t>((pattern + 31u) >> 7) - 8;
            return static_cast<uint32_t>(e > 1 ? e : 1);
        }

        // The scale byte of a row spread over G lanes, in every one of them.
        template <int G>
        __device__ __forceinline__ uint32_t row_scale(const Vec8 &x)
        {
            uint32_t a = group_max<G>(max_pattern(x, 0x8000u));
            if (a >= 0x7f80u) // an infinity or a NaN: rare, and the lanes of a row agree
                a = group_max<G>(max_pattern(x, 0x7f80u));
            return scale_byte(a);
        }

        // 2^-e of a scale byte (1 .. 247): an ordinary fp32 number.
        __device__ __forceinline__ float scale_inverse(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }

        __device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d)
        {
            int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
            r = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
            return static_cast<uint32_t>(r);
        }

        // Eight codes; |x| * inv <= 448, and an infinity or a NaN converts to a NaN code.
        __device__ __forceinline__ uint2 encode8(const Vec8 &x, float inv)
        {
            return make_uint2(encode4(bf_lo(x.d[0]) * inv, bf_hi(x.d[0]) * inv, bf_lo(x.d[1]) * inv, bf_hi(x.d[1]) * inv),
                              encode4(bf_lo(x.d[2]) * inv, bf_hi(x.d[2]) * inv, bf_lo(x.d[3]) * inv, bf_hi(x.d[3]) * inv));
        }

        // Eight codes, streamed past the L2 as the 16-byte stores of q3k_common.hpp are (16 x
        // 4096 positions of 8 heads: 68.0 us, 69.7 with plain stores).
        __device__ __forceinline__ void store_codes(uint2 *p, uint2 codes)
        {
            typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
            u32x2 v;
            v.x = codes.x;
            v.y = codes.y;
            __asm__ volatile("global_store_dwordx2 %0, %1, off nt sc1\n\ts_nop 1" : : "v"(p), "v"(v) : "memory");
        }

        // G lanes a row, grid over the rows (b, s, h) of the input in order.  16 x 4096
        // positions of 8 heads: 68.6 us, 404 MB at 5.88 TB/s; 64 positions 2.4 us and the
        // launch.
        template <int G>
        __global__ __launch_bounds__(kBlock) void append_rows_kernel(const Vec8 *__restrict__ k, const Vec8 *__restrict__ v,
                                                                     uint8_t *__restrict__ kc, uint8_t *__restrict__ vc,
                                                                     uint8_t *__restrict__ scales, E4m3Shape s)
        {
            const uint32_t row = blockIdx.x * (kBlock / G) + threadIdx.x / G;
            if (row >= s.rows)
                return;
            const uint32_t l = threadIdx.x % G;
            const Vec8 xk = load8<true>(k + static_cast<int64_t>(row) * G + l);
            const Vec8 xv = load8<true>(v + static_cast<int64_t>(row) * G + l);
            const uint32_t token = row / s.Hkv, h = row - token * s.Hkv;
            const uint32_t b = token / s.S;
            const int64_t pos = (s.starts != nullptr ? s.starts[b] : s.start) + (token - b * s.S);
            const uint32_t sk = row_scale<G>(xk), sv = row_scale<G>(xv);
            const uint2 ck = encode8(xk, scale_inverse(sk)), cv = encode8(xv, scale_inverse(sv));
            if (pos < 0 || pos >= s.seq_cap)
                return;
            const int64_t at = cache_row(s, b, h, pos);
            store_codes(reinterpret_cast<uint2 *>(kc) + at * G + l, ck);
            store_codes(reinterpret_cast<uint2 *>(vc) + at * G + l, cv);
            if (l < 2)
                scales[2 * at + l] = static_cast<uint8_t>(l == 0 ? sk : sv);
        }

        // Two heads of a position a lane (h and h + half of them), the codes of both before
        // the stores, so that the groups of G lanes of a wave store one run of rows and then
        // the run behind it.  16 x 4096 positions of 8 heads: 67.7 us, 404 MB at 5.96 TB/s; of
        // ragged sequences 44.3 us.  With two positions of a head a lane instead 68.0 to 72.7
        // and 44.2 to 48.1, with four positions 71.5 to 76.2 and 45.9 to 47.4; with rows in
        // the output's order whatever their heads 67.3 to 68.5 and 44.0 to 48.6.
        constexpr int kReadHeads = 2;

        template <int G>
        __global__ __launch_bounds__(kBlock) void read_rows_kernel(const uint8_t *__restrict__ kc, const uint8_t *__restrict__ vc,
                                                                   const uint8_t *__restrict__ scales, Vec8 *__restrict__ k,
                                                                   Vec8 *__restrict__ v, E4m3Shape s)
        {
            // unit: (sequence, position, head of the first half)
            const uint32_t half = (s.Hkv + kReadHeads - 1) / kReadHeads;
            const uint32_t unit = blockIdx.x * (kBlock / G) + threadIdx.x / G, l = threadIdx.x % G;
            const uint32_t token = unit / half, h0 = unit - token * half;
            const uint32_t b = token / s.S;
            const int64_t pos = s.start + (token - b * s.S);
            if (token >= s.rows / s.Hkv || (s.starts != nullptr && pos >= s.starts[b]))
                return;
            uint2 ck[kReadHeads], cv[kReadHeads];
            uint32_t sk[kReadHeads], sv[kReadHeads];
#pragma unroll
            for (int x = 0; x < kReadHeads; ++x)
                if (h0 + x * half < s.Hkv)
                {
                    const int64_t at = cache_row(s, b, h0 + x * half, pos);
                    ck[x] = reinterpret_cast<const uint2 *>(kc)[at * G + l];
                    cv[x] = reinterpret_cast<const uint2 *>(vc)[at * G + l];
                    sk[x] = scales[2 * at];
                    sv[x] = scales[2 * at + 1];
                }
#pragma unroll
            for (int x = 0; x < kReadHeads; ++x)
                if (h0 + x * half < s.Hkv)
                {
                    const int64_t out = (static_cast<int64_t>(token) * s.Hkv + h0 + x * half) * G + l;
                    store8<kStoreStream>(k + out, decode8(ck[x], e4m3_scale(sk[x])));
                    store8<kStoreStream>(v + out, decode8(cv[x], e4m3_scale(sv[x])));
                }
        }

        // Any head_dim and alignment: a wave a row, K then V.
        __global__ __launch_bounds__(kBlock) void append_generic_kernel(const uint16_t *k, const uint16_t *v, uint8_t *kc,
                                                                        uint8_t *vc, uint8_t *scales, E4m3Shape s)
        {
            const int lane = threadIdx.x % kWave;
            const int64_t waves = static_cast<int64_t>(gridDim.x) * (kBlock / kWave);
            for (int64_t row = static_cast<int64_t>(blockIdx.x) * (kBlock / kWave) + threadIdx.x / kWave; row < s.rows; row += waves)
            {
                const uint32_t token = static_cast<uint32_t>(row) / s.Hkv, h = static_cast<uint32_t>(row) - token * s.Hkv;
                const uint32_t b = token / s.S;
                const int64_t pos = (s.starts != nullptr ? s.starts[b] : s.start) + (token - b * s.S);
                if (pos < 0 || pos >= s.seq_cap)
                    continue;
                const int64_t at = cache_row(s, b, h, pos);
                for (int which = 0; which < 2; ++which)
                {
                    const uint16_t *x = (which == 0 ? k : v) + row * s.D;
                    uint8_t *c = (which == 0 ? kc : vc) + at * s.D;
                    uint32_t m = 0;
                    for (uint32_t d = lane; d < s.D; d += kWave)
                    {
                        const uint32_t a = x[d] & 0x7fffu;
                        m = a < 0x7f80u && a > m ? a : m;
                    }
                    for (int off = kWave / 2; off > 0; off /= 2)
                    {
                        const uint32_t o = static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), off, kWave));
                        m = m > o ? m : o;
                    }
                    const uint32_t byte = scale_byte(m);
                    const float inv = scale_inverse(byte);
                    for (uint32_t d = lane; d < s.D; d += kWave)
                        c[d] = static_cast<uint8_t>(encode4(bf_to_f(x[d]) * inv, 0.0f, 0.0f, 0.0f));
                    if (lane == 0)
                        scales[2 * at + which] = static_cast<uint8_t>(byte);
                }
            }
        }

        __global__ __launch_bounds__(kBlock) void read_generic_kernel(const uint8_t *kc, const uint8_t *vc, const uint8_t *scales,
                                                                      uint16_t *k, uint16_t *v, E4m3Shape s)
        {
            const int lane = threadIdx.x % kWave;
            const int64_t waves = static_cast<int64_t>(gridDim.x) * (kBlock / kWave);
            for (int64_t row = static_cast<int64_t>(blockIdx.x) * (kBlock / kWave) + threadIdx.x / kWave; row < s.rows; row += waves)
            {
                const uint32_t token = static_cast<uint32_t>(row) / s.Hkv, h = static_cast<uint32_t>(row) - token * s.Hkv;
                const uint32_t b = token / s.S;
                const int64_t pos = s.start + (token - b * s.S);
                if (s.starts != nullptr && pos >= s.starts[b])
                    continue;
                const int64_t at = cache_row(s, b, h, pos);
                for (uint32_t d = lane; d < s.D; d += kWave)
                {
                    k[row * s.D + d] = f_to_bf(e4m3_value(kc[at * s.D + d]) * e4m3_scale(scales[2 * at]));
                    v[row * s.D + d] = f_to_bf(e4m3_value(vc[at * s.D + d]) * e4m3_scale(scales[2 * at + 1]));
                }
            }
        }

        unsigned generic_grid(const E4m3Shape &s)
        {
            const int64_t blocks = blocks_for(s.rows, kBlock / kWave);
            return static_cast<unsigned>(blocks < 65536 ? blocks : 65536);
        }

        // Lanes of a row of the vector kernels, 0: the generic one.
        int row_lanes(const E4m3Shape &s, bool aligned)
        {
            const int lanes = s.D == 64 || s.D == 128 || s.D == 256 ? static_cast<int>(s.D / 8) : 0;
            return aligned && lanes != 0 && launch_fits(blocks_for(s.rows, kBlock / lanes), kBlock) ? lanes : 0;
        }

        // The checks that the append and the reading back share; S: positions of a sequence.
        int validate(const char *what, const void *a, const void *b, const void *c, const void *d, const void *scales,
                     int64_t B, int64_t S, int32_t Hkv, int32_t D, int64_t seq_cap, int64_t start, const int32_t *starts)
        {
            if (B < 0 || S < 0)
                return set_error(Q3K_ERR_INVALID_ARGUMENT, "%s batch and sequence sizes cannot be negative", what);
            if (Hkv <= 0 || D <= 0)
                return set_error(Q3K_ERR_INVALID_ARGUMENT, "%s head count and head_dim must be positive", what);
            if (seq_cap <= 0)
                return set_error(Q3K_ERR_INVALID_ARGUMENT, "%s sequence capacity must be positive", what);
            if (start < 0 || start > seq_cap || S > seq_cap - start)
                return set_error(Q3K_ERR_OUT_OF_RANGE, "%s exceeds sequence capacity", what);
            if (B > 0 && (B > INT64_MAX / Hkv || seq_cap > INT64_MAX / (B * Hkv) || D > INT64_MAX / (B * Hkv * seq_cap)))
                return set_error(Q3K_ERR_OVERFLOW, "%s layer size overflows", what);
            if (B > 0 && S > 0 && (S > INT32_MAX / B || B * S > INT32_MAX / Hkv))
                return set_error(Q3K_ERR_OVERFLOW, "%s grid is too large", what);
            if (B > 0 && S > 0 && (a == nullptr || b == nullptr || c == nullptr || d == nullptr || scales == nullptr))
                return set_error(Q3K_ERR_INVALID_ARGUMENT, "%s received a null pointer", what);
            if (!aligned_to(a, 2) || !aligned_to(b, 2) || !aligned_to(starts, 4))
                return set_error(Q3K_ERR_INVALID_ARGUMENT, "%s pointers must be aligned to their element size", what);
            return Q3K_OK;
        }
    } // namespace
} // namespace q3k

extern "C" int q3k_kv_append_e4m3_bf16(const uint16_t *key, const uint16_t *value, uint8_t *k_codes, uint8_t *v_codes,
                                       uint8_t *scales, int64_t B, int64_t S, int32_t Hkv, int32_t D, int64_t seq_cap,
                                       int64_t start, const int32_t *starts, q3k_stream_t stream)
{
    using namespace q3k;
    // (rows of sequences with starts of their own are checked by the kernel)
    if (const int st = validate("e4m3 KV cache append", key, value, k_codes, v_codes, scales, B, S, Hkv, D, seq_cap,
                                starts != nullptr ? 0 : start, starts))
        return st;
    if (B == 0 || S == 0)
        return Q3K_OK;
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    const E4m3Shape s{static_cast<uint32_t>(B * S * Hkv), static_cast<uint32_t>(S), static_cast<uint32_t>(Hkv),
                      static_cast<uint32_t>(D), seq_cap, start, starts};
    const Vec8 *k = reinterpret_cast<const Vec8 *>(key), *v = reinterpret_cast<const Vec8 *>(value);
    const dim3 block(kBlock);
    const int lanes = row_lanes(s, aligned16(key) && aligned16(value) && aligned_to(k_codes, 8) && aligned_to(v_codes, 8));
    const dim3 grid(lanes == 0 ? generic_grid(s) : static_cast<unsigned>(blocks_for(s.rows, kBlock / lanes)));
    switch (lanes)
    {
    case 8: append_rows_kernel<8><<<grid, block, 0, st>>>(k, v, k_codes, v_codes, scales, s); break;
    case 16: append_rows_kernel<16><<<grid, block, 0, st>>>(k, v, k_codes, v_codes, scales, s); break;
    case 32: append_rows_kernel<32><<<grid, block, 0, st>>>(k, v, k_codes, v_codes, scales, s); break;
    default: append_generic_kernel<<<grid, block, 0, st>>>(key, value, k_codes, v_codes, scales, s); break;
    }
    return check_launch("kv_append_e4m3");
}

extern "C" int q3k_kv_read_e4m3_bf16(const uint8_t *k_codes, const uint8_t *v_codes, const uint8_t *scales, uint16_t *key,
                                     uint16_t *value, int64_t B, int32_t Hkv, int32_t D, int64_t seq_cap, int64_t first,
                                     int64_t count, const int32_t *lengths, q3k_stream_t stream)
{
    using namespace q3k;
    if (const int st = validate("e4m3 KV cache read", key, value, k_codes, v_codes, scales, B, count, Hkv, D, seq_cap, first, lengths))
        return st;
    if (B == 0 || count == 0)
        return Q3K_OK;
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    const E4m3Shape s{static_cast<uint32_t>(B * count * Hkv), static_cast<uint32_t>(count), static_cast<uint32_t>(Hkv),
                      static_cast<uint32_t>(D), seq_cap, first, lengths};
    Vec8 *k = reinterpret_cast<Vec8 *>(key), *v = reinterpret_cast<Vec8 *>(value);
    const dim3 block(kBlock);
    const int lanes = row_lanes(s, aligned16(key) && aligned16(value) && aligned_to(k_codes, 8) && aligned_to(v_codes, 8));
    const dim3 grid(lanes == 0 ? generic_grid(s) : static_cast<unsigned>(blocks_for(B * count * blocks_for(Hkv, kReadHeads), kBlock / lanes)));
    switch (lanes)
    {
    case 8: read_rows_kernel<8><<<grid, block, 0, st>>>(k_codes, v_codes, scales, k, v, s); break;
    case 16: read_rows_kernel<16><<<grid, block, 0, st>>>(k_codes, v_codes, scales, k, v, s); break;
    case 32: read_rows_kernel<32><<<grid, block, 0, st>>>(k_codes, v_codes, scales, k, v, s); break;
    default: read_generic_kernel<<<grid, block, 0, st>>>(k_codes, v_codes, scales, key, value, s); break;
    }
    return check_launch("kv_read_e4m3");
}
