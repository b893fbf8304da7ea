// What the attention kernels on keys of any length share (prefix_attn.hip,
// cache_attn.hip): operands as hi + lo halves, tiles in LDS and their transposed
// reads.
#pragma once

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

// the sum of weights, of both lanes of a place
__device__ __forceinline__ float pair_sum(float l) {
    const auto other = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
    return __uint_as_float(other[0]) + __uint_as_float(other[1]);
}

}  // namespace samhip
