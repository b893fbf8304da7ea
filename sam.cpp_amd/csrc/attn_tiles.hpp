// What the attention kernels on keys of any length share (prefix_attn.hip,
// cache_attn.hip): operands as hi + lo halves, values read transposed from LDS,
// and the join of partial sums.
#pragma once

#include <type_traits>

#include "q8stage.hpp"

#pragma clang fp contract(off)

namespace samhip {

typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef short short4_t __attribute__((ext_vector_type(4)));

constexpr float LOG2E = 1.44269504088896340736f;

// ds_read_b64_tr_b16: within each group of 16 lanes, lane i receives element
// (i % 4) of the 8-byte rows that lanes 4j + i/4 address, j = 0..3
[[maybe_unused]] __device__ __forceinline__ half4 ds_read_tr(const uint8_t* p) {
#if defined(__HIP_DEVICE_COMPILE__)
    const short4_t v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4_t*)(p));
    return __builtin_bit_cast(half4, v);
#else
    return half4{};
#endif
}

typedef _Float16 half8_at __attribute__((ext_vector_type(8), aligned(2)));
typedef float float4_at __attribute__((ext_vector_type(4), aligned(4)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef float float2_t __attribute__((ext_vector_type(2)));

// Values j and j + 1 as hi + lo: hi two at a time; lo = fp16(x - hi) by a
// mixed-precision fma, whose factor one is kept from the compiler, which
// would fold it away.
__device__ __forceinline__ void split_pair(float2_t x, half8& hi, half8& lo, int j) {
#if defined(__HIP_DEVICE_COMPILE__)
    float one = 1.0f;
    asm("" : "+s"(one));
    const half2_t h = __builtin_convertvector(x, half2_t);
    const float2_t hf = __builtin_convertvector(h, float2_t);
    hi[j] = h[0];
    hi[j + 1] = h[1];
    lo[j] = (_Float16)__builtin_fmaf(x[0], one, -hf[0]);
    lo[j + 1] = (_Float16)__builtin_fmaf(x[1], one, -hf[1]);
#endif
}

// Biased exponent of the largest magnitude, kept where both powers below are
// normal floats.
__device__ __forceinline__ int exponent_of(uint32_t magnitude_bits) {
    return magnitude_bits ? min(max(int(magnitude_bits >> 23), 20), 254) : 141;
}
__device__ __forceinline__ float down(int e) { return __uint_as_float(uint32_t(268 - e) << 23); }   // 2^(141 - e)
__device__ __forceinline__ float up(int e) { return __uint_as_float(uint32_t(e - 14) << 23); }      // 2^(e - 141)

__device__ __forceinline__ uint32_t wave_umax(uint32_t v) { return umax_xor32(umax_xor16(umax_row(umax_quad(v)))); }

// A tile of KEYS keys or values of HD as fp16 rows in LDS, of PARTS 2 as hi
// and, behind them, lo.  Keys are read 16 bytes a row from 16 rows at once,
// values (V) 64 bytes a row from 4: the rows' padding spreads either over the
// 64 banks.
template <int PARTS, int HD, int KEYS, bool V>
struct TileShape {
    static constexpr int STRIDE = !V ? HD * 2 + 16 : HD == 32 ? 64 : HD * 2 + 64;
    static constexpr int BYTES = KEYS * STRIDE * PARTS;
    // piece f (8 values) of the tile; its lo is KEYS * STRIDE bytes behind it
    static __device__ __forceinline__ half8* piece(uint8_t* tile, int f) {
        return reinterpret_cast<half8*>(tile + f / (HD / 8) * STRIDE + f % (HD / 8) * 16);
    }
};

// sc[n] += K Q^T of keys 32n .. + 31 of a tile of keys in LDS
template <int PARTS, int HD, int N>
__device__ __forceinline__ void scores(const uint8_t* kt, const half8 (&q_hi)[HD / 16], const half8 (&q_lo)[HD / 16], floatx16 (&sc)[N]) {
    typedef TileShape<PARTS, HD, 32 * N, false> R;
    const int lane = threadIdx.x & 63, li = lane & 31, hh = lane >> 5;
    const uint8_t* at = kt + li * R::STRIDE + 16 * hh;
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) sc[n][r] = 0.f;
#pragma unroll
    for (int t = 0; t < HD / 16; ++t)
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const half8 kh = *reinterpret_cast<const half8*>(at + 32 * n * R::STRIDE + 32 * t);
            sc[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kh, q_hi[t], sc[n], 0, 0, 0);
            sc[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kh, q_lo[t], sc[n], 0, 0, 0);
            if constexpr (PARTS == 2) {
                const half8 kl = *reinterpret_cast<const half8*>(at + (32 * N + 32 * n) * R::STRIDE + 32 * t);
                sc[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kl, q_hi[t], sc[n], 0, 0, 0);
            }
        }
}

// O^T += V^T P^T with a tile of values in LDS: of 16 keys, lane (li, hh) holds
// keys 4hh .. + 3 and 8 + 4hh .. + 3 of both operands, V^T read transposed.
template <int PARTS, int HD, int N>
__device__ __forceinline__ void values(const uint8_t* vt, const half8 (&hi)[2 * N], const half8 (&lo)[2 * N], floatx16 (&o)[HD / 32]) {
    typedef TileShape<PARTS, HD, 32 * N, true> R;
    const int lane = threadIdx.x & 63, hh = lane >> 5;
    const uint8_t* at = vt + (4 * hh + ((lane & 15) >> 2)) * R::STRIDE + 32 * ((lane >> 4) & 1) + 8 * (lane & 3);
    constexpr int DB = HD / 32, COUNT = 2 * N * DB, AHEAD = HD < 128 ? 1 : 0;   // 128: no registers left
    half8 v[2][PARTS];   // the next one is under way during a product
    const auto fetch = [&](int i) {
        const uint8_t* p = at + 16 * (i / DB) * R::STRIDE + 64 * (i % DB);
#pragma unroll
        for (int part = 0; part < PARTS; ++part) {
            const uint8_t* q = p + part * 32 * N * R::STRIDE;
            v[i & 1][part] = __builtin_shufflevector(ds_read_tr(q), ds_read_tr(q + 8 * R::STRIDE), 0, 1, 2, 3, 4, 5, 6, 7);
        }
    };
    if (AHEAD) fetch(0);
#pragma unroll
    for (int i = 0; i < COUNT; ++i) {
        const int u = i / DB, d = i % DB;
        if (i + AHEAD < COUNT) fetch(i + AHEAD);
        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[i & 1][0], hi[u], o[d], 0, 0, 0);
        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[i & 1][0], lo[u], o[d], 0, 0, 0);
        if constexpr (PARTS == 2) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[i & 1][PARTS - 1], hi[u], o[d], 0, 0, 0);
    }
}

// the sum of weights, of both lanes of a place
__device__ __forceinline__ float pair_sum(float l) {
    const auto other = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
    return __uint_as_float(other[0]) + __uint_as_float(other[1]);
}

// A wave joins the parts of one row and head (ml_apart and o_apart floats from
// one to the next): their maxima and sums one to a lane, then HD / 4 lanes to a
// part's mean.
template <int HD>
__device__ __forceinline__ void merge_parts(const float* part_ml, int64_t ml_apart, const float* part_o, int64_t o_apart, int count, float* out) {
    constexpr int QUADS = HD / 4, AT_ONCE = 64 / QUADS;
    const int lane = threadIdx.x & 63;
    const int d = 4 * (lane % QUADS), slot = lane / QUADS;
    float m = -__builtin_inff(), l = 0.f;
    floatx4 v{0.f, 0.f, 0.f, 0.f};
    for (int p0 = 0; p0 < count; p0 += 64) {
        float mp = -__builtin_inff(), lp = 0.f;
        if (p0 + lane < count) {
            const float* ml = part_ml + (p0 + lane) * ml_apart;
            mp = ml[0];
            lp = ml[1];
        }
        const float mnew = fmaxf(m, wave_max(lp != 0.f ? mp : -__builtin_inff()));
        const float old = m == mnew ? 1.f : __builtin_amdgcn_exp2f(m - mnew);
        float f = lp != 0.f ? lp * __builtin_amdgcn_exp2f(mp - mnew) : 0.f;
        const float before = l * old;
        m = mnew;
        l = before + wave_sum(f);
        const float inv = l == 0.f ? 0.f : 1.f / l;   // v stays a mean
        f = lp != 0.f ? f * inv : -1.f;   // no key in this part
        v = v * (before * inv);
        const int here = min(count - p0, 64);
        const float* parts = part_o + p0 * o_apart + d;
        const auto add = [&](auto at_once, int p1) {   // parts p1 + slot, p1 + slot + AT_ONCE, ..
            constexpr int U = decltype(at_once)::value;
            floatx4 o[U];
            float fp[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int p = p1 + u * AT_ONCE + slot, at = min(p, here - 1);
                o[u] = *reinterpret_cast<const floatx4*>(parts + at * o_apart);
                fp[u] = __shfl(f, at, 64);
                if (p >= here) fp[u] = -1.f;
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] += fp[u] < 0.f ? 0.f : o[u][j] * fp[u];   // without keys its mean may never have been written
        };
        int p1 = 0;
        for (; p1 + 3 * AT_ONCE < here; p1 += 4 * AT_ONCE) add(std::integral_constant<int, 4>{}, p1);
        for (; p1 < here; p1 += AT_ONCE) add(std::integral_constant<int, 1>{}, p1);
    }
#pragma unroll
    for (int off = QUADS; off < 64; off <<= 1)
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] += __shfl_xor(v[j], off, 64);
    if (slot == 0) *reinterpret_cast<float4_at*>(out + d) = v;
}

}  // namespace samhip
