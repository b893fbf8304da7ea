// Attention of a batch of requests that share a prefix of keys, each with
// keys of its own behind it:
//   out = softmax(scale * q K^T) V,  K = [prefix ; the request's own keys]
// The prefix part does not depend on the request, so it is computed for
// tiles of query rows of all requests; the own part for tiles of one
// request's rows.  Either part's keys may be split over workgroups.  Each
// leaves a maximum, a sum of weights and a weighted mean of values (a mean fits
// F32 wherever the values do), which attn_merge_kernel joins (a part that is
// alone writes the output itself).
// Grouped heads: the queries that share a kv head are neighbouring rows of a
// tile (row index = query row * group + head in group).
//
// F32-accurate: queries, weights P and F32 keys and values enter the fp16
// matrix instructions as hi + lo (lo = fp16(v - hi)), with the products
// hi*hi + hi*lo + lo*hi; queries (by row), keys and values (by tile) are
// scaled by powers of two so that the largest magnitude lies in [2^14, 2^15),
// which leaves ~22 bits to those no more than 2^18 times smaller.  F16 keys and
// values enter as they are.
// Bound, with many queries, by vector instructions (softmax, splitting) and by
// waits at barriers and for data with two waves a SIMD, beside the matrix
// instructions (8 prompts of 201 queries on 5184 + 33 F32 keys, 8 heads of 32:
// 49 us, 530 TFLOP/s of hi + lo products, vector instructions 25 us and matrix
// instructions 10 us of it; 64 queries of 16 heads of 128 on 65536 F16 keys: 85
// us, 810 TFLOP/s, and 98 with up to 1024 own keys each), by two launches'
// latency for few queries (8 on 5184: 9.3 us).
#include <algorithm>
#include <type_traits>

#include "internal.hpp"
#include "q8stage.hpp"

#pragma clang fp contract(off)

namespace samhip {

namespace {

typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef short short4_t __attribute__((ext_vector_type(4)));

constexpr float LOG2E = 1.44269504088896340736f;
constexpr int TILE = 32;    // query rows and keys of one wave's step
constexpr int WAVES = 4;

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

constexpr uint32_t INF_BITS = 0x7f800000u;

// Eight neighbouring values as loaded.
template <class T>
struct Raw8;
template <>
struct Raw8<_Float16> {
    half8 v;
    __device__ __forceinline__ void load(const _Float16* p) { v = *reinterpret_cast<const half8_at*>(p); }
    __device__ __forceinline__ bool finite() const {
        typedef uint16_t ushort2_t __attribute__((ext_vector_type(2)));
        typedef uint16_t ushort8 __attribute__((ext_vector_type(8)));
        const ushort8 bits = __builtin_bit_cast(ushort8, v) & (uint16_t)0x7fff;
        ushort2_t m{bits[0], bits[1]};
#pragma unroll
        for (int j = 2; j < 8; j += 2) m = __builtin_elementwise_max(m, ushort2_t{bits[j], bits[j + 1]});
        return m[0] < 0x7c00 && m[1] < 0x7c00;
    }
    __device__ __forceinline__ void clear_non_finite() {   // zeros instead
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = __builtin_fabsf16(v[j]) < (_Float16)__builtin_inff16() ? v[j] : (_Float16)0;
    }
};
template <>
struct Raw8<float> {
    floatx4 a, b;
    __device__ __forceinline__ void load(const float* p) {
        a = *reinterpret_cast<const float4_at*>(p);
        b = *reinterpret_cast<const float4_at*>(p + 4);
    }
    __device__ __forceinline__ uint32_t magnitude() const {
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            m = umax(m, __float_as_uint(a[j]) & 0x7fffffffu);
            m = umax(m, __float_as_uint(b[j]) & 0x7fffffffu);
        }
        return m;
    }
    __device__ __forceinline__ bool finite() const { return magnitude() < INF_BITS; }
    __device__ __forceinline__ void clear_non_finite() {   // zeros instead
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            a[j] = __builtin_fabsf(a[j]) < __builtin_inff() ? a[j] : 0.f;
            b[j] = __builtin_fabsf(b[j]) < __builtin_inff() ? b[j] : 0.f;
        }
    }
    // values * factor as hi + lo
    __device__ __forceinline__ void split(float factor, half8& hi, half8& lo) const {
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            const float2_t x{(j < 4 ? a[j & 3] : b[j & 3]) * factor, (j < 4 ? a[(j & 3) + 1] : b[(j & 3) + 1]) * factor};
            split_pair(x, hi, lo, j);
        }
    }
};

// Biased exponent of the largest magnitude, kept where both powers below are
// normal floats.
__device__ __forceinline__ int exponent_of(uint32_t magnitude_bits) {
    return magnitude_bits ? min(max(int(magnitude_bits >> 23), 20), 254) : 141;
}
__device__ __forceinline__ float down(int e) { return __uint_as_float(uint32_t(268 - e) << 23); }   // 2^(141 - e)
__device__ __forceinline__ float up(int e) { return __uint_as_float(uint32_t(e - 14) << 23); }      // 2^(e - 141)

__device__ __forceinline__ uint32_t wave_umax(uint32_t v) { return umax_xor32(umax_xor16(umax_row(umax_quad(v)))); }

// The largest magnitude of a wave's keys or values.  An infinity or a NaN, which
// stays in its key's scores or its value's dimension, does not set the others'
// scale.
template <int N>
__device__ __forceinline__ uint32_t largest_finite(const Raw8<float> (&v)[N]) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) m = umax(m, v[i].magnitude());
    m = __builtin_amdgcn_readfirstlane(wave_umax(m));
    if (m >= INF_BITS) {
        m = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            Raw8<float> finite = v[i];
            finite.clear_non_finite();
            m = umax(m, finite.magnitude());
        }
        m = __builtin_amdgcn_readfirstlane(wave_umax(m));
    }
    return m;
}

// What a workgroup reads: keys [k0, k1) of one kv head, for query rows
// [q0, q0 + n) in flattened (row, head in group) places.
template <class T>
struct Span {
    const T *k, *v;       // row 0, this kv head
    int64_t ldk, ldv;
    int k0, k1;
    int q0, n, first;     // query rows, and the tile's first place
    int limit0;           // causal: a query row i sees keys below limit0 + i
    bool causal;
};

// One wave's 32 query places: lane (li, hh) holds place li's values
// 16t + 8hh .. + 7 as hi + lo, and c, which takes a product of the scaled
// operands to a score in units of log 2 (the sign of a negative scale is the
// query's; factor() keeps it positive, for a masked product is -inf).
template <int HD>
struct Queries {
    half8 hi[HD / 16], lo[HD / 16];
    float c;
    int row, head, limit;
    bool mine;

    __device__ __forceinline__ float factor(float of_keys) const { return fmaxf(c * of_keys, 0x1p-120f); }

    template <class T>
    __device__ __forceinline__ Queries(const PrefixAttnArgs& a, const Span<T>& s, int kvh, int place) {
        const int hh = (threadIdx.x & 63) >> 5, i = place / a.group;
        mine = i < s.n;
        row = s.q0 + (mine ? i : 0);
        head = kvh * a.group + place - i * a.group;
        limit = s.causal ? min(s.k1, s.limit0 + i) : s.k1;
        Raw8<float> raw[HD / 16];
        uint32_t m = 0;
#pragma unroll
        for (int t = 0; t < HD / 16; ++t) raw[t].load(a.q + row * a.ldq + head * HD + 16 * t + 8 * hh);
#pragma unroll
        for (int t = 0; t < HD / 16; ++t) m = umax(m, raw[t].magnitude());
        const int e = exponent_of(umax_xor32(m));
        const float f = a.scale < 0.f ? -down(e) : down(e);
#pragma unroll
        for (int t = 0; t < HD / 16; ++t) raw[t].split(f, hi[t], lo[t]);
        c = fabsf(a.scale) * LOG2E * up(e);
    }
};

// The base of the weights 2^(score - m), below the running maximum (in units of
// log 2), their sum, and the weighted sums of values of a wave's places: o[d]
// holds, transposed, lane (li, hh)'s dimensions 32d + 8 (r / 4) + 4hh + r % 4 of
// place li, F32 values in units of 2^(e - 141), one e for the wave (NONE: no
// value but zeros yet).
template <int HD>
struct Sums {
    static constexpr int NONE = 0, SLACK = 2;
    floatx16 o[HD / 32];
    float m = -__builtin_inff(), l = 0.f;
    int e = NONE;

    __device__ __forceinline__ Sums() { scale(0.f, true); }
    __device__ __forceinline__ void scale(float f, bool clear = false) {
#pragma unroll
        for (int d = 0; d < HD / 32; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[d][r] = clear ? 0.f : o[d][r] * f;
    }
    __device__ __forceinline__ void shift(int by) {   // times 2^by
#pragma unroll
        for (int d = 0; d < HD / 32; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[d][r] = __builtin_ldexpf(o[d][r], by);
    }

    // Those of a row of values that are not finite
    template <class T>
    __device__ __forceinline__ void add_non_finite(const T* row) {
        const int hh = (threadIdx.x & 63) >> 5;
#pragma unroll
        for (int d = 0; d < HD / 32; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float v = float(row[32 * d + 8 * (r >> 2) + 4 * hh + (r & 3)]);
                if ((__float_as_uint(v) & 0x7fffffffu) >= INF_BITS) o[d][r] += v;
                asm volatile("" ::: "memory");   // one at a time, for the registers
            }
    }

    // F32 values of one tile, whose largest has exponent `to` (0: all zero), come
    // in units of 2^(to - 141).  The sums follow it, down where they leave room:
    // values 2^75 apart keep their digits beside each other.  Returns how many
    // powers of two the weights have to be lowered by, SLACK at most where there
    // is room, so that most steps change nothing.
    __device__ __forceinline__ int follow(int to) {
        if (to == 0) return 0;
        if (e == NONE) e = to;
        if (to > e) {
            shift(e - to);
            e = to;
        } else if (to < e - SLACK) {
            uint32_t most = 0;   // of the finite sums
#pragma unroll
            for (int d = 0; d < HD / 32; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const uint32_t b = __float_as_uint(o[d][r]) & 0x7fffffffu;
                    most = umax(most, b < INF_BITS ? b : 0u);
                }
            const int room = 251 - int(__builtin_amdgcn_readfirstlane(wave_umax(most)) >> 23);   // they stay below 2^125
            const int by = min(e - to, max(room, 0));
            shift(by);
            e -= by;
        }
        return min(e - to, 100);   // past 40 no weight is left as fp16, but in l
    }

    // Weights of N blocks of 32 keys from key `k` on: sc[n] holds products with
    // keys 32n + 8 (r / 4) + 4hh + r % 4, c takes them to scores; hi + lo of the
    // weights, lowered by 2^-low, leave in the order the value operand is read in.
    template <int N>
    __device__ __forceinline__ void weigh(floatx16 (&sc)[N], float c, int k, int limit, int low, half8 (&hi)[2 * N], half8 (&lo)[2 * N]) {
        const int hh = (threadIdx.x & 63) >> 5;
        if (__any(k + 32 * N > limit)) {
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (k + 32 * n + 8 * (r >> 2) + 4 * hh + (r & 3) >= limit) sc[n][r] = -__builtin_inff();
        }
        // IEEE maximum: a NaN score gives a NaN row either way, and fmaxf
        // would first quiet every product
        float mx = sc[0][0];
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int r = 0; r < 16; ++r) mx = __builtin_elementwise_maximum(mx, sc[n][r]);
        const auto other = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
        mx = __builtin_elementwise_maximum(__uint_as_float(other[0]), __uint_as_float(other[1]));
        // The largest weight so far lies in [2^11, 2^15): the base moves only
        // when a score passes it by 15, so that most steps skip the rescaling,
        // and as fp16 halves a weight keeps 22 bits down to 2^(low - 14) of the
        // largest and is off by 2^(low - 36) of it at most.
        if (__any(__builtin_fmaf(mx, c, -m) > 15.0f)) {
            const float mnew = fmaxf(m, __builtin_fmaf(mx, c, -11.0f));
            const float alpha = mnew == m ? 1.f : __builtin_amdgcn_exp2f(m - mnew);
            m = mnew;
            l = l * alpha;
            scale(alpha);
        }
        const float mb = (m == -__builtin_inff() ? 0.f : m) + float(low);   // nothing seen yet: weights 0
        float ps = 0.f;
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                sc[n][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[n][r], c, -mb));
                ps += sc[n][r];
            }
        l = l + ps * __builtin_ldexpf(1.f, low);
#pragma unroll
        for (int u = 0; u < 2 * N; ++u)
#pragma unroll
            for (int j = 0; j < 8; j += 2)
                split_pair(float2_t{sc[u / 2][8 * (u % 2) + j], sc[u / 2][8 * (u % 2) + j + 1]}, hi[u], lo[u], j);
    }
};

// A tile of KEYS keys or values of HD as fp16 rows in LDS, F32 ones as hi
// and, behind them, lo.  Keys are read 16 bytes a row from 16 rows at once,
// values (V) 64 bytes a row from 4: the rows' padding spreads either over the
// 64 banks.
template <class T, int HD, int KEYS, bool V>
struct TileRows {
    static constexpr int PARTS = sizeof(T) == 4 ? 2 : 1, STRIDE = !V ? HD * 2 + 16 : HD == 32 ? 64 : HD * 2 + 64;
    static constexpr int BYTES = KEYS * STRIDE * PARTS;
    // piece f (8 values) of the tile
    static __device__ __forceinline__ void put(uint8_t* tile, int f, const Raw8<T>& raw, float factor) {
        half8* to = reinterpret_cast<half8*>(tile + f / (HD / 8) * STRIDE + f % (HD / 8) * 16);
        if constexpr (sizeof(T) == 4) {
            half8 hi, lo;
            raw.split(factor, hi, lo);
            *to = hi;
            to[KEYS * STRIDE / 16] = lo;
        } else {
            *to = raw.v;
        }
    }
};

// sc[n] += K Q^T of keys 32n .. + 31 of a tile of keys in LDS
template <class T, int HD, int N>
__device__ __forceinline__ void scores(const uint8_t* kt, const Queries<HD>& q, floatx16 (&sc)[N]) {
    typedef TileRows<T, HD, 32 * N, false> R;
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
            sc[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kh, q.hi[t], sc[n], 0, 0, 0);
            sc[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kh, q.lo[t], sc[n], 0, 0, 0);
            if constexpr (R::PARTS == 2) {
                const half8 kl = *reinterpret_cast<const half8*>(at + (32 * N + 32 * n) * R::STRIDE + 32 * t);
                sc[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kl, q.hi[t], sc[n], 0, 0, 0);
            }
        }
}

// O^T += V^T P^T with a tile of values in LDS: of 16 keys, lane (li, hh) holds
// keys 4hh .. + 3 and 8 + 4hh .. + 3 of both operands, V^T read transposed.
template <class T, int HD, int N>
__device__ __forceinline__ void values(const uint8_t* vt, const half8 (&hi)[2 * N], const half8 (&lo)[2 * N], Sums<HD>& sums) {
    typedef TileRows<T, HD, 32 * N, true> R;
    const int lane = threadIdx.x & 63, hh = lane >> 5;
    const uint8_t* at = vt + (4 * hh + ((lane & 15) >> 2)) * R::STRIDE + 32 * ((lane >> 4) & 1) + 8 * (lane & 3);
    constexpr int DB = HD / 32, COUNT = 2 * N * DB, AHEAD = HD < 128 ? 1 : 0;   // 128: no registers left
    half8 v[2][R::PARTS];   // the next one is under way during a product
    const auto fetch = [&](int i) {
        const uint8_t* p = at + 16 * (i / DB) * R::STRIDE + 64 * (i % DB);
#pragma unroll
        for (int part = 0; part < R::PARTS; ++part) {
            const uint8_t* q = p + part * 32 * N * R::STRIDE;
            v[i & 1][part] = __builtin_shufflevector(ds_read_tr(q), ds_read_tr(q + 8 * R::STRIDE), 0, 1, 2, 3, 4, 5, 6, 7);
        }
    };
    if (AHEAD) fetch(0);
#pragma unroll
    for (int i = 0; i < COUNT; ++i) {
        const int u = i / DB, d = i % DB;
        if (i + AHEAD < COUNT) fetch(i + AHEAD);
        sums.o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[i & 1][0], hi[u], sums.o[d], 0, 0, 0);
        sums.o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[i & 1][0], lo[u], sums.o[d], 0, 0, 0);
        if constexpr (R::PARTS == 2) sums.o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[i & 1][R::PARTS - 1], hi[u], sums.o[d], 0, 0, 0);
    }
}

// the sum of weights, of both lanes of a place
__device__ __forceinline__ float pair_sum(float l) {
    const auto other = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
    return __uint_as_float(other[0]) + __uint_as_float(other[1]);
}

// Few query places: all four waves have the same 32, and each takes tiles of
// 32 keys of its own, keys straight from memory, values through LDS that no
// other wave touches.
template <class T, int HD>
struct Narrow {
    static constexpr int VBYTES = TileRows<T, HD, 32, true>::BYTES, OBYTES = TILE * (HD + 4) * 4;   // a wave's tile, and its sums at the end
    uint8_t __attribute__((aligned(16))) lds[WAVES * (VBYTES > OBYTES ? VBYTES : OBYTES)];
    float m[WAVES][TILE], l[WAVES][TILE];
};

template <class T, int HD>
__device__ __forceinline__ void attend_narrow(const PrefixAttnArgs& a, const Span<T>& s, int kvh, int part, Narrow<T, HD>& sh) {
    constexpr int STEPS = HD / 16;
    constexpr bool F32 = sizeof(T) == 4, AHEAD = HD * sizeof(T) <= 128;   // registers for the next tile
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, li = lane & 31, hh = lane >> 5;
    const Queries<HD> q(a, s, kvh, s.first + li);
    Sums<HD> sums;
    uint8_t* vt = sh.lds + wave * Narrow<T, HD>::VBYTES;
    Raw8<T> kr[STEPS], vr[STEPS];
    const int step = TILE * WAVES, kw = s.k0 + TILE * wave;
    const int key = lane / (HD / 8), col = 8 * (lane % (HD / 8));   // of the first 64 pieces of values
    const T *kp = s.k + (kw + li) * s.ldk + 8 * hh, *vp = s.v + (kw + key) * s.ldv + col;
    const auto load = [&](int k) {
        if (k + TILE <= s.k1) {
#pragma unroll
            for (int t = 0; t < STEPS; ++t) kr[t].load(kp + 16 * t);
#pragma unroll
            for (int t = 0; t < STEPS; ++t) vr[t].load(vp + t * (512 / HD) * s.ldv);
            kp += step * s.ldk;
            vp += step * s.ldv;
        } else {   // behind the last key the last one again: its weight is zero there
            const T* last = s.k + min(k + li, s.k1 - 1) * s.ldk + 8 * hh;
#pragma unroll
            for (int t = 0; t < STEPS; ++t) kr[t].load(last + 16 * t);
#pragma unroll
            for (int t = 0; t < STEPS; ++t) vr[t].load(s.v + min(k + key + t * (512 / HD), s.k1 - 1) * s.ldv + col);
        }
    };
    // Keys below this one are seen by every place.  In a tile that reaches
    // further a weight of zero keeps no infinity or NaN out: such values are
    // zeros in it, and are added behind the last tile for those that see them.
    const int seen_by_all = s.causal ? s.limit0 + s.first / a.group : s.k1 + TILE;
    bool non_finite_values = false;
    if (AHEAD && kw < s.k1) load(kw);
    for (int k = kw; k < s.k1; k += step) {
        if (!AHEAD) load(k);
        if (k + TILE > seen_by_all) {
            bool finite = true;
#pragma unroll
            for (int t = 0; t < STEPS; ++t) finite = finite && vr[t].finite();
            if (!__all(finite)) {
                non_finite_values = true;
#pragma unroll
                for (int t = 0; t < STEPS; ++t) vr[t].clear_non_finite();
            }
        }
        floatx16 sc[1];
#pragma unroll
        for (int r = 0; r < 16; ++r) sc[0][r] = 0.f;
        float c = q.factor(1.f), fv = 1.f;
        int low = 0;
        if constexpr (F32) {
            const int e = exponent_of(largest_finite(kr));
            const uint32_t mv = largest_finite(vr);
            fv = down(exponent_of(mv));
            c = q.factor(up(e));
#pragma unroll
            for (int t = 0; t < STEPS; ++t) {
                half8 kh, kl;
                kr[t].split(down(e), kh, kl);
                sc[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kh, q.hi[t], sc[0], 0, 0, 0);
                sc[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kl, q.hi[t], sc[0], 0, 0, 0);
                sc[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kh, q.lo[t], sc[0], 0, 0, 0);
            }
            low = sums.follow(mv ? exponent_of(mv) : 0);
        } else {
#pragma unroll
            for (int t = 0; t < STEPS; ++t) {
                sc[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kr[t].v, q.hi[t], sc[0], 0, 0, 0);
                sc[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kr[t].v, q.lo[t], sc[0], 0, 0, 0);
            }
        }
        wave_lds_handoff();   // the last tile's reads came first
#pragma unroll
        for (int t = 0; t < STEPS; ++t) TileRows<T, HD, 32, true>::put(vt, t * 64 + lane, vr[t], fv);
        wave_lds_handoff();
        if (AHEAD && k + step < s.k1) load(k + step);
        half8 ph[2], pl[2];
        sums.weigh(sc, c, k, q.limit, low, ph, pl);
        values<T, HD, 1>(vt, ph, pl, sums);
    }
    if (non_finite_values)
        for (int k = kw; k < s.k1; k += step)
            for (int n = k + TILE > seen_by_all ? 0 : TILE; n < TILE; ++n)
                if (k + n < q.limit) sums.add_non_finite(s.v + int64_t(k + n) * s.ldv);
    // the four waves' sums, joined through LDS
    sums.l = pair_sum(sums.l);
    if (hh == 0) {
        sh.m[wave][li] = sums.m;
        sh.l[wave][li] = sums.l;
    }
    __syncthreads();   // also: every wave is past its value tiles
    float m = -__builtin_inff(), l = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) m = fmaxf(m, sh.m[w][li]);
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        const float lw = sh.l[w][li];
        if (lw != 0.f) l += lw * __builtin_amdgcn_exp2f(sh.m[w][li] - m);   // a NaN sum stays one
    }
    const float f = sums.l != 0.f ? __builtin_amdgcn_exp2f(sums.m - m) / l : 0.f;
    sums.scale(f);
    if constexpr (F32) sums.shift(sums.e - 141);
    float* all = reinterpret_cast<float*>(sh.lds);
#pragma unroll
    for (int d = 0; d < HD / 32; ++d)
#pragma unroll
        for (int r = 0; r < 16; r += 4)
            *reinterpret_cast<floatx4*>(all + (wave * TILE + li) * (HD + 4) + 32 * d + 2 * r + 4 * hh) =
                floatx4{sums.o[d][r], sums.o[d][r + 1], sums.o[d][r + 2], sums.o[d][r + 3]};
    if (part >= 0 && wave == 0 && hh == 0 && q.mine) {
        float* ml = a.part_ml + ((int64_t(q.row) * a.heads + q.head) * a.parts + part) * 2;
        ml[0] = m;
        ml[1] = l;
    }
    __syncthreads();
    constexpr int QUADS = HD / 4;
    for (int t = tid; t < TILE * QUADS; t += 64 * WAVES) {
        const int p = t / QUADS, d = 4 * (t % QUADS), place = s.first + p, i = place / a.group;
        if (i >= s.n) continue;
        floatx4 v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < WAVES; ++w) v += *reinterpret_cast<const floatx4*>(all + (w * TILE + p) * (HD + 4) + d);
        const int64_t r = s.q0 + i, h = kvh * a.group + place - i * a.group;
        float* to = part < 0 ? a.out + r * a.ldo + h * HD : a.part_o + ((r * a.heads + h) * a.parts + part) * HD;
        *reinterpret_cast<float4_at*>(to + d) = v;
    }
}

// Many query places: 32 to a wave, and tiles of 64 keys and values that the
// four waves share in LDS; the next tile is on its way to registers during a
// tile's products.
template <class T, int HD>
struct Wide {
    uint8_t __attribute__((aligned(16))) k[TileRows<T, HD, 64, false>::BYTES];
    uint8_t __attribute__((aligned(16))) v[TileRows<T, HD, 64, true>::BYTES];
    uint32_t largest[WAVES][2];
};

template <class T, int HD>
__device__ __forceinline__ void attend_wide(const PrefixAttnArgs& a, const Span<T>& s, int kvh, int part, Wide<T, HD>& sh) {
    constexpr int PIECES = HD / 32;   // of 8 values, a thread's part of a tile
    constexpr bool F32 = sizeof(T) == 4;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, li = lane & 31, hh = lane >> 5;
    const int first = s.first + TILE * wave;
    const bool any = first < s.n * a.group;
    const Queries<HD> q(a, s, kvh, first + li);
    Sums<HD> sums;
    Raw8<T> kr[PIECES], vr[PIECES];
    // this thread's piece of the first 256; the others are whole rows of keys on
    const int key = tid / (HD / 8), col = 8 * (tid % (HD / 8));
    const T *kp = s.k + (s.k0 + key) * s.ldk + col, *vp = s.v + (s.k0 + key) * s.ldv + col;
    const auto load = [&](int k) {
        if (k + 64 <= s.k1) {
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
                kr[i].load(kp + i * (2048 / HD) * s.ldk);
                vr[i].load(vp + i * (2048 / HD) * s.ldv);
            }
            kp += 64 * s.ldk;
            vp += 64 * s.ldv;
        } else {   // behind the last key the last one again: its weight is zero there
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
                const int64_t at = min(k + key + i * (2048 / HD), s.k1 - 1);
                kr[i].load(s.k + at * s.ldk + col);
                vr[i].load(s.v + at * s.ldv + col);
            }
        }
    };
    load(s.k0);
    for (int k = s.k0; k < s.k1; k += 64) {
        float c = q.factor(1.f), fk = 1.f, fv = 1.f;
        int low = 0;
        if constexpr (F32) {
            uint32_t mk = 0;
#pragma unroll
            for (int i = 0; i < PIECES; ++i) mk = umax(mk, kr[i].magnitude());
            mk = wave_umax(mk);
            const uint32_t mv = largest_finite(vr);
            if (lane == 0) sh.largest[wave][0] = mk, sh.largest[wave][1] = mv;
        }
        __syncthreads();   // the last tile is read, the largest magnitudes are written
        if constexpr (F32) {
            uint32_t mk = 0, mv = 0;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) mk = umax(mk, sh.largest[w][0]), mv = umax(mv, sh.largest[w][1]);
            mv = __builtin_amdgcn_readfirstlane(mv);
            const int e = exponent_of(__builtin_amdgcn_readfirstlane(mk));
            c = q.factor(up(e));
            fk = down(e);
            fv = down(exponent_of(mv));
            low = sums.follow(mv ? exponent_of(mv) : 0);
        }
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            TileRows<T, HD, 64, false>::put(sh.k, tid + 256 * i, kr[i], fk);
            TileRows<T, HD, 64, true>::put(sh.v, tid + 256 * i, vr[i], fv);
        }
        __syncthreads();
        if (k + 64 < s.k1) load(k + 64);
        if (any) {
            floatx16 sc[2];
            half8 ph[4], pl[4];
            scores<T, HD, 2>(sh.k, q, sc);
            sums.weigh(sc, c, k, q.limit, low, ph, pl);
            values<T, HD, 2>(sh.v, ph, pl, sums);
        }
    }
    const float l = pair_sum(sums.l);
    if (!q.mine) return;
    sums.scale(l == 0.f ? 0.f : 1.f / l);
    if constexpr (F32) sums.shift(sums.e - 141);
    float* to;
    if (part < 0) {
        to = a.out + q.row * a.ldo + q.head * HD;
    } else {
        const int64_t at = (int64_t(q.row) * a.heads + q.head) * a.parts + part;
        to = a.part_o + at * HD;
        if (hh == 0) {
            a.part_ml[2 * at] = sums.m;
            a.part_ml[2 * at + 1] = l;
        }
    }
#pragma unroll
    for (int d = 0; d < HD / 32; ++d)
#pragma unroll
        for (int r = 0; r < 16; r += 4)
            *reinterpret_cast<float4_at*>(to + 32 * d + 2 * r + 4 * hh) =
                floatx4{sums.o[d][r], sums.o[d][r + 1], sums.o[d][r + 2], sums.o[d][r + 3]};
}

// Query rows [from, from + n) of request r, cut to the rows that exist.
__device__ __forceinline__ int rows_of(const PrefixAttnArgs& a, int r, int& from) {
    from = min(max(a.q_start[r], 0), a.rows);
    return min(max(a.q_start[r + 1], 0), a.rows) - from;
}

// The t-th tile of all requests' own parts; false past the last.
__device__ __forceinline__ bool find_tile(const PrefixAttnArgs& a, int t, int& request, int& tile) {
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int r0 = 0; r0 < a.requests; r0 += 64) {
        int tiles = 0;
        if (r0 + lane < a.requests) {
            int from;
            tiles = (max(rows_of(a, r0 + lane, from), 0) * a.group + TILE - 1) / TILE;
        }
        int sum = tiles;
        for (int off = 1; off < 64; off <<= 1) {
            const int x = __shfl_up(sum, off, 64);
            if (lane >= off) sum += x;
        }
        const uint64_t past = __ballot(before + sum > t);
        if (past) {
            const int at = __builtin_ctzll(past);
            request = r0 + at;
            tile = t - before - (__shfl(sum, at, 64) - __shfl(tiles, at, 64));
            return true;
        }
        before += __shfl(sum, 63, 64);
    }
    return false;
}

// Grid: the prefix part's workgroups and the own parts'.  Workgroups are
// dispatched round-robin over the 8 XCDs: the prefix part's are numbered so
// that the query tiles that read the same keys run one behind the other on
// one XCD and share its L2.
template <class T, int HD, bool WIDE>
__global__ __launch_bounds__(64 * WAVES, 2) void prefix_attn_kernel(PrefixAttnArgs a) {
    union Shared {
        Narrow<T, HD> narrow;
        Wide<T, HD> wide;
    };
    __shared__ typename std::conditional<WIDE, Shared, Narrow<T, HD>>::type sh;
    // The prefix part first: behind its products the own parts fill the CUs
    // that end early (in turn with them 60 us against 50 for 8 prompts of 201
    // queries on 5184 keys, 44 against 33 for ragged causal requests).
    int w = blockIdx.x;
    Span<T> s;
    if (w < a.prefix_groups) {
        const int order = w >> 3, set = (w & 7) + 8 * (order / a.prefix_tiles);   // of kv head and split
        const int kvh = set / a.prefix_splits, split = set - kvh * a.prefix_splits;
        if (kvh >= a.kv_heads) return;
        s.q0 = min(max(a.q_start[0], 0), a.rows);
        s.n = min(max(a.q_start[a.requests], 0), a.rows) - s.q0;
        s.first = order % a.prefix_tiles * (WIDE ? TILE * WAVES : TILE);
        if (s.first >= s.n * a.group) return;
        s.k = static_cast<const T*>(a.prefix_k) + kvh * HD;
        s.v = static_cast<const T*>(a.prefix_v) + kvh * HD;
        s.ldk = a.ld_prefix_k;
        s.ldv = a.ld_prefix_v;
        s.k0 = split * a.prefix_chunk;
        s.k1 = min(s.k0 + a.prefix_chunk, a.prefix);
        s.causal = false;
        s.limit0 = 0;
        const int part = a.parts > 1 ? split : -1;
        if constexpr (WIDE) attend_wide<T, HD>(a, s, kvh, part, sh.wide);
        else attend_narrow<T, HD>(a, s, kvh, part, sh);
        return;
    }
    w -= a.prefix_groups;
    const int per_head = a.own_tiles * a.own_splits, kvh = w / per_head, split = (w - kvh * per_head) / a.own_tiles;
    int request, tile;
    if (!find_tile(a, w - kvh * per_head - split * a.own_tiles, request, tile)) return;
    s.n = rows_of(a, request, s.q0);
    s.first = tile * TILE;
    int64_t start = 0;
    int len = 0;
    if (a.own_max > 0) {
        start = a.own_start[request];
        len = min(max(a.own_len[request], 0), a.own_max);
        if (start < 0 || start > a.own_rows) start = len = 0;
        len = int(min(int64_t(len), a.own_rows - start));
    }
    s.k = static_cast<const T*>(a.own_k) + start * a.ld_own_k + kvh * HD;
    s.v = static_cast<const T*>(a.own_v) + start * a.ld_own_v + kvh * HD;
    s.ldk = a.ld_own_k;
    s.ldv = a.ld_own_v;
    s.causal = a.causal;
    s.limit0 = len - s.n + 1;
    s.k0 = split * a.own_chunk;
    s.k1 = min(s.k0 + a.own_chunk, len);
    if (s.causal) s.k1 = min(s.k1, s.limit0 + min(s.n - 1, (s.first + TILE - 1) / a.group));
    const int part = a.parts > 1 ? a.prefix_splits + split : -1;
    if constexpr (WIDE) attend_narrow<T, HD>(a, s, kvh, part, sh.narrow);
    else attend_narrow<T, HD>(a, s, kvh, part, sh);
}

// A wave per (row, head): the parts' maxima and sums one to a lane, then
// HD / 4 lanes to a part's mean.
template <int HD>
__global__ __launch_bounds__(256) void attn_merge_kernel(PrefixAttnArgs a) {
    constexpr int QUADS = HD / 4, AT_ONCE = 64 / QUADS;
    const int lane = threadIdx.x & 63;
    const int64_t item = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6), items = int64_t(a.rows) * a.heads;
    if (item >= items) return;
    const int64_t row = item / a.heads, h = item - row * a.heads;
    if (row < min(max(a.q_start[0], 0), a.rows) || row >= min(max(a.q_start[a.requests], 0), a.rows)) return;
    const int d = 4 * (lane % QUADS), slot = lane / QUADS;
    float m = -__builtin_inff(), l = 0.f;
    floatx4 v{0.f, 0.f, 0.f, 0.f};
    for (int p0 = 0; p0 < a.parts; p0 += 64) {
        float mp = -__builtin_inff(), lp = 0.f;
        if (p0 + lane < a.parts) {
            const float* ml = a.part_ml + (item * a.parts + p0 + lane) * 2;
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
        const int here = min(a.parts - p0, 64);
        const float* parts = a.part_o + (item * a.parts + p0) * HD + d;
        const auto add = [&](auto count, int p1) {   // parts p1 + slot, p1 + slot + AT_ONCE, ..
            constexpr int U = decltype(count)::value;
            floatx4 o[U];
            float fp[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int p = p1 + u * AT_ONCE + slot, at = min(p, here - 1);
                o[u] = *reinterpret_cast<const floatx4*>(parts + at * HD);
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
    if (slot == 0) *reinterpret_cast<float4_at*>(a.out + row * a.ldo + h * HD + d) = v;
}

template <class T, int HD>
void launch_typed(const PrefixAttnArgs& a, hipStream_t stream) {
    const unsigned groups = unsigned(a.prefix_groups) + unsigned(a.own_tiles) * a.own_splits * a.kv_heads;
    if (a.wide) prefix_attn_kernel<T, HD, true><<<groups, 64 * WAVES, 0, stream>>>(a);
    else prefix_attn_kernel<T, HD, false><<<groups, 64 * WAVES, 0, stream>>>(a);
    if (a.parts > 1) attn_merge_kernel<HD><<<unsigned((int64_t(a.rows) * a.heads + 3) / 4), 256, 0, stream>>>(a);
}

}  // namespace

void prefix_attn_plan(PrefixAttnArgs& a, int head_dim, int cus) {
    // The number of key splits for `groups` workgroups a split.  A CU takes
    // ceil(workgroups / CUs) of them, each with its tiles of `step` keys and about
    // three tiles' time to begin and end; one alone reaches some 60 % of
    // what three together do, two 85 %.  A split costs its partial sums' way
    // to memory and back, 3 TB/s, where a tile takes 0.5 us + 6 ns a dimension
    // (constants fitted to a few batches between 8 and 1608 queries, not swept).
    const auto splits = [&](int64_t groups, int64_t keys, int step) {
        const int most = int(std::max<int64_t>(1, std::min<int64_t>((keys + 255) / 256, (4 * cus + groups - 1) / groups)));
        const double tile_us = 0.5 + 0.006 * head_dim, split_us = double(a.rows) * a.heads * head_dim * 8 / 3e6;
        int best = 1;
        double least = 0;
        const auto consider = [&](int64_t candidate) {
            const int n = int(std::max<int64_t>(1, std::min<int64_t>(candidate, most)));
            const int64_t per_cu = (groups * n + cus - 1) / cus, tiles = (keys + int64_t(n) * step - 1) / (int64_t(n) * step);
            const double rate = per_cu == 1 ? 0.6 : per_cu == 2 ? 0.85 : 1.0;
            const double us = per_cu * (tiles + 3) / rate * tile_us + (n > 1 ? n * split_us : 0.0);
            if (least == 0 || us < least) best = n, least = us;
        };
        for (int per_cu = 4; per_cu >= 1; --per_cu) consider(int64_t(per_cu) * cus / groups);   // the most that a level takes
        for (int64_t n = cus / groups / 2; n >= 1; n /= 2) consider(n);
        consider(1);
        return best;
    };
    const auto chunk = [](int64_t keys, int n) { return int(((keys + n - 1) / n + 63) / 64 * 64); };
    a.group = a.heads / a.kv_heads;
    const int64_t places = int64_t(a.rows) * a.group;
    a.wide = a.prefix && places > 2 * TILE;
    const int tile = a.wide ? TILE * WAVES : TILE, step = a.wide ? 64 : TILE * WAVES;
    a.prefix_tiles = a.prefix ? int((places + tile - 1) / tile) : 0;
    a.prefix_splits = a.prefix ? splits(int64_t(a.prefix_tiles) * a.kv_heads, a.prefix, step) : 0;
    a.prefix_groups = 0;
    if (a.prefix) {
        a.prefix_chunk = chunk(a.prefix, a.prefix_splits);
        a.prefix_splits = (a.prefix + a.prefix_chunk - 1) / a.prefix_chunk;
        a.prefix_groups = (a.prefix_splits * a.kv_heads + 7) / 8 * 8 * a.prefix_tiles;
    }
    // without a prefix the own parts write every row, an empty one as zeros
    const bool own = a.own_max > 0 || !a.prefix;
    a.own_tiles = own ? int(places / TILE + std::min<int64_t>(a.requests, a.rows)) : 0;
    a.own_splits = own ? splits(int64_t(a.own_tiles) * a.kv_heads, a.own_max, TILE * WAVES) : 0;
    if (own) {
        a.own_chunk = std::max(chunk(a.own_max, a.own_splits), TILE);
        a.own_splits = std::max(1, (a.own_max + a.own_chunk - 1) / a.own_chunk);
    }
    a.parts = a.prefix_splits + a.own_splits;
}

size_t prefix_attn_scratch_bytes(const PrefixAttnArgs& a, int head_dim) {
    return a.parts > 1 ? size_t(a.parts) * a.rows * a.heads * (head_dim + 2) * 4 : 0;
}

void launch_prefix_attn(PrefixAttnArgs a, int type, int head_dim, void* scratch, hipStream_t stream) {
    a.part_o = static_cast<float*>(scratch);
    a.part_ml = a.part_o + size_t(a.parts) * a.rows * a.heads * head_dim;
    if (type == T_F16) {
        if (head_dim == 32) launch_typed<_Float16, 32>(a, stream);
        else if (head_dim == 64) launch_typed<_Float16, 64>(a, stream);
        else launch_typed<_Float16, 128>(a, stream);
    } else {
        if (head_dim == 32) launch_typed<float, 32>(a, stream);
        else if (head_dim == 64) launch_typed<float, 64>(a, stream);
        else launch_typed<float, 128>(a, stream);
    }
}

}  // namespace samhip
