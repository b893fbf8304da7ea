// Attention of a batch of requests that share a prefix of keys, each with
// keys of its own behind it:
//   out = softmax(scale * q K^T) V,  K = [prefix ; the request's own keys]
// The prefix part does not depend on the request, so it is computed for
// tiles of query rows of all requests; the own part for tiles of one
// request's rows.  Either part's keys may be split over workgroups.  Each
// leaves a maximum, a sum of weights and a weighted sum of values, which
// attn_merge_kernel joins (a part that is alone writes the output itself).
// Grouped heads: the queries that share a kv head are neighbouring rows of a
// tile (row index = query row * group + head in group).
//
// F32-accurate: queries, weights P and F32 keys and values enter the fp16
// matrix instructions as hi + lo (lo = fp16(v - hi)), with the products
// hi*hi + hi*lo + lo*hi; queries (by row), keys and values (by tile) are
// scaled by powers of two so that the largest magnitude lies in [2^14, 2^15)
// and any F32 range keeps ~22 bits.  F16 keys and values enter as they are.
#include <algorithm>

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

struct __attribute__((packed, aligned(2))) Half8At {
    half8 v;
};
struct __attribute__((packed, aligned(4))) Float4At {
    floatx4 v;
};

// Eight neighbouring values as loaded, zeros where the row is not to be read.
template <class T>
struct Raw8;
template <>
struct Raw8<_Float16> {
    half8 v;
    __device__ __forceinline__ void load(const _Float16* p, bool real) {
        v = half8{0, 0, 0, 0, 0, 0, 0, 0};
        if (real) v = reinterpret_cast<const Half8At*>(p)->v;
    }
};
template <>
struct Raw8<float> {
    floatx4 a, b;
    __device__ __forceinline__ void load(const float* p, bool real) {
        a = b = floatx4{0.f, 0.f, 0.f, 0.f};
        if (real) {
            a = reinterpret_cast<const Float4At*>(p)->v;
            b = reinterpret_cast<const Float4At*>(p + 4)->v;
        }
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
    // values * factor as hi + lo
    __device__ __forceinline__ void split(float factor, half8& hi, half8& lo) const {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float x = (j < 4 ? a[j & 3] : b[j & 3]) * factor;
            const _Float16 h = (_Float16)x;
            hi[j] = h;
            lo[j] = (_Float16)(x - (float)h);
        }
    }
};

// Biased exponent of the largest magnitude, kept where both powers below are
// normal floats.
__device__ __forceinline__ int exponent_of(uint32_t magnitude_bits) { return min(max(int(magnitude_bits >> 23), 20), 254); }
__device__ __forceinline__ float down(int e) { return __uint_as_float(uint32_t(268 - e) << 23); }   // 2^(141 - e)
__device__ __forceinline__ float up(int e) { return __uint_as_float(uint32_t(e - 14) << 23); }      // 2^(e - 141)

__device__ __forceinline__ uint32_t wave_umax(uint32_t v) { return umax_xor32(umax_xor16(umax_row(umax_quad(v)))); }

// What a workgroup reads: keys [k0, k1) of one kv head, for query rows
// [q0, q0 + n) in the tile's 32 flattened (row, head in group) places.
template <class T>
struct Span {
    const T *k, *v;       // row 0, this kv head
    int64_t ldk, ldv;
    int k0, k1;
    int q0, n, first;     // query rows, and the tile's first place
    int limit0;           // causal: a query row i sees keys below limit0 + i
    bool causal;
};

template <class T, int HD>
struct Shared {
    static constexpr int PARTS = sizeof(T) == 4 ? 2 : 1;
    static constexpr int STRIDE = HD * 2 + 16;                  // bytes of a key's values
    static constexpr int VBYTES = TILE * STRIDE * PARTS;        // one wave's tile
    static constexpr int OBYTES = TILE * (HD + 4) * 4;          // one wave's sums, at the end
    static constexpr int BYTES = WAVES * (VBYTES > OBYTES ? VBYTES : OBYTES);
};

template <class T, int HD>
__device__ __forceinline__ void attend(const PrefixAttnArgs& a, const Span<T>& s, int kvh, int part, uint8_t* lds, float (*wave_m)[TILE],
                                       float (*wave_l)[TILE], float* total) {
    constexpr int STEPS = HD / 16, DB = HD / 32;
    constexpr bool F32 = sizeof(T) == 4;
    typedef Shared<T, HD> S;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, li = lane & 31, hh = lane >> 5;
    const int place = s.first + li, i = place / a.group;
    const bool mine = i < s.n;
    const int row = s.q0 + i, head = kvh * a.group + place - i * a.group;
    const int limit = s.causal ? min(s.k1, s.limit0 + i) : s.k1;

    // the query row as hi + lo, scaled by its own power of two
    half8 qh[STEPS], ql[STEPS];
    float c;
    {
        Raw8<float> raw[STEPS];
        uint32_t m = 0;
#pragma unroll
        for (int t = 0; t < STEPS; ++t) {
            raw[t].load(a.q + row * a.ldq + head * HD + 16 * t + 8 * hh, mine);
            m = umax(m, raw[t].magnitude());
        }
        const int e = exponent_of(umax_xor32(m));
#pragma unroll
        for (int t = 0; t < STEPS; ++t) raw[t].split(down(e), qh[t], ql[t]);
        c = a.scale * LOG2E * up(e);   // scores in units of log 2
    }

    floatx16 o[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] = 0.f;
    float mrun = -__builtin_inff(), lsum = 0.f;
    int ev = 20;   // F32 values: the exponent that the sums are scaled by
    uint8_t* vt = lds + wave * S::VBYTES;

    for (int k = s.k0 + TILE * wave; k < s.k1; k += TILE * WAVES) {
        Raw8<T> kr[STEPS], vr[STEPS];
#pragma unroll
        for (int t = 0; t < STEPS; ++t) kr[t].load(s.k + (k + li) * s.ldk + 16 * t + 8 * hh, k + li < s.k1);
#pragma unroll
        for (int t = 0; t < STEPS; ++t) {
            const int at = t * 64 + lane, key = at / (HD / 8), col = at % (HD / 8);
            vr[t].load(s.v + (k + key) * s.ldv + 8 * col, k + key < s.k1);
        }
        floatx16 sc;
#pragma unroll
        for (int r = 0; r < 16; ++r) sc[r] = 0.f;
        float ck = c;
        if constexpr (F32) {
            uint32_t m = 0;
#pragma unroll
            for (int t = 0; t < STEPS; ++t) m = umax(m, kr[t].magnitude());
            const int e = exponent_of(__builtin_amdgcn_readfirstlane(wave_umax(m)));
            ck = c * up(e);
#pragma unroll
            for (int t = 0; t < STEPS; ++t) {
                half8 kh, kl;
                kr[t].split(down(e), kh, kl);
                sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(kh, qh[t], sc, 0, 0, 0);
                sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(kl, qh[t], sc, 0, 0, 0);
                sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(kh, ql[t], sc, 0, 0, 0);
            }
        } else {
#pragma unroll
            for (int t = 0; t < STEPS; ++t) {
                sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(kr[t].v, qh[t], sc, 0, 0, 0);
                sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(kr[t].v, ql[t], sc, 0, 0, 0);
            }
        }
        // values to LDS, one row per key
        wave_lds_handoff();   // the last tile's reads came first
        if constexpr (F32) {
            uint32_t m = 0;
#pragma unroll
            for (int t = 0; t < STEPS; ++t) m = umax(m, vr[t].magnitude());
            const int e = exponent_of(__builtin_amdgcn_readfirstlane(wave_umax(m)));
            if (e > ev) {
                const float f = __builtin_ldexpf(1.f, ev - e);
                ev = e;
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int r = 0; r < 16; ++r) o[d][r] = o[d][r] * f;
            }
        }
#pragma unroll
        for (int t = 0; t < STEPS; ++t) {
            const int at = t * 64 + lane, key = at / (HD / 8), col = at % (HD / 8);
            half8* to = reinterpret_cast<half8*>(vt + key * S::STRIDE + col * 16);
            if constexpr (F32) {
                half8 vh, vl;
                vr[t].split(down(ev), vh, vl);
                *to = vh;
                to[TILE * S::STRIDE / 16] = vl;
            } else {
                *to = vr[t].v;
            }
        }
        wave_lds_handoff();
        // softmax: lane (li, hh) holds place li's scores of keys
        // 8 (r / 4) + 4 hh + r % 4
#pragma unroll
        for (int r = 0; r < 16; ++r) sc[r] = sc[r] * ck;
        if (__any(k + TILE > limit)) {
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if (k + 8 * (r >> 2) + 4 * hh + (r & 3) >= limit) sc[r] = -__builtin_inff();
        }
        float mx = sc[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) mx = __builtin_elementwise_maximum(mx, sc[r]);
        const auto other = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
        mx = __builtin_elementwise_maximum(__uint_as_float(other[0]), __uint_as_float(other[1]));
        // the exponent base moves only when a score passes it by 8, so that
        // weights stay below 2^8 and most steps skip the rescaling
        if (__any(mx > mrun + 8.0f)) {
            const float mnew = fmaxf(mrun, mx);
            const float alpha = mnew == mrun ? 1.f : __builtin_amdgcn_exp2f(mrun - mnew);
            mrun = mnew;
            lsum = lsum * alpha;
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[d][r] = o[d][r] * alpha;
        }
        const float mb = mrun == -__builtin_inff() ? 0.f : mrun;   // nothing seen yet: weights 0
        float ps = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            sc[r] = __builtin_amdgcn_exp2f(sc[r] - mb);
            ps += sc[r];
        }
        lsum = lsum + ps;
        half8 ph[2], pl[2];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float p = sc[8 * u + j];
                const _Float16 h = (_Float16)p;
                ph[u][j] = h;
                pl[u][j] = (_Float16)(p - (float)h);
            }
        // O^T += V^T P^T: keys 16u + 4hh .. + 3 and 16u + 8 + 4hh .. + 3
        const uint8_t* at = vt + (4 * hh + ((lane & 15) >> 2)) * S::STRIDE + 32 * ((lane >> 4) & 1) + 8 * (lane & 3);
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int d = 0; d < DB; ++d) {
                const uint8_t* p = at + 16 * u * S::STRIDE + 64 * d;
                const half8 vh = __builtin_shufflevector(ds_read_tr(p), ds_read_tr(p + 8 * S::STRIDE), 0, 1, 2, 3, 4, 5, 6, 7);
                o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vh, ph[u], o[d], 0, 0, 0);
                o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vh, pl[u], o[d], 0, 0, 0);
                if constexpr (F32) {
                    const uint8_t* q = p + TILE * S::STRIDE;
                    const half8 vl = __builtin_shufflevector(ds_read_tr(q), ds_read_tr(q + 8 * S::STRIDE), 0, 1, 2, 3, 4, 5, 6, 7);
                    o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vl, ph[u], o[d], 0, 0, 0);
                }
            }
    }
    // the four waves' sums, joined through LDS
    const auto lother = __builtin_amdgcn_permlane32_swap(__float_as_uint(lsum), __float_as_uint(lsum), false, false);
    lsum = __uint_as_float(lother[0]) + __uint_as_float(lother[1]);
    if (hh == 0) {
        wave_m[wave][li] = mrun;
        wave_l[wave][li] = lsum;
    }
    __syncthreads();   // also: every wave is past its value tiles
    float m = -__builtin_inff(), l = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) m = fmaxf(m, wave_m[w][li]);
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        const float lw = wave_l[w][li];
        if (lw != 0.f) l += lw * __builtin_amdgcn_exp2f(wave_m[w][li] - m);   // a NaN sum stays one
    }
    float f = lsum != 0.f ? __builtin_amdgcn_exp2f(mrun - m) : 0.f;
    if constexpr (F32) f = f * up(ev);
    float* sums = reinterpret_cast<float*>(lds);
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            float* to = sums + (wave * TILE + li) * (HD + 4) + 32 * d + 2 * r + 4 * hh;
            *reinterpret_cast<floatx4*>(to) = floatx4{o[d][r] * f, o[d][r + 1] * f, o[d][r + 2] * f, o[d][r + 3] * f};
        }
    if (part >= 0 && wave == 0 && hh == 0 && mine) {
        float* ml = a.part_ml + (int64_t(part) * a.rows * a.heads + int64_t(row) * a.heads + head) * 2;
        ml[0] = m;
        ml[1] = l;
    }
    if (wave == 0 && hh == 0) total[li] = l;
    __syncthreads();
    constexpr int QUADS = HD / 4;
    for (int t = tid; t < TILE * QUADS; t += 64 * WAVES) {
        const int p = t / QUADS, d = 4 * (t % QUADS), pl = s.first + p, pi = pl / a.group;
        if (pi >= s.n) continue;
        floatx4 v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < WAVES; ++w) v += *reinterpret_cast<const floatx4*>(sums + (w * TILE + p) * (HD + 4) + d);
        const int64_t r = s.q0 + pi, h = kvh * a.group + pl - pi * a.group;
        if (part < 0) {
            const float lt = total[p];
            const float inv = lt == 0.f ? 0.f : 1.f / lt;
            reinterpret_cast<Float4At*>(a.out + r * a.ldo + h * HD + d)->v = v * inv;
        } else {
            *reinterpret_cast<floatx4*>(a.part_o + ((int64_t(part) * a.rows + r) * a.heads + h) * HD + d) = v;
        }
    }
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

// Grid: the prefix part's workgroups (tiles x splits), then the own parts',
// times kv heads.
template <class T, int HD>
__global__ __launch_bounds__(64 * WAVES) void prefix_attn_kernel(PrefixAttnArgs a) {
    __shared__ __attribute__((aligned(16))) uint8_t lds[Shared<T, HD>::BYTES];
    __shared__ float wave_m[WAVES][TILE], wave_l[WAVES][TILE], total[TILE];
    const int kvh = blockIdx.y;
    int w = blockIdx.x;
    Span<T> s;
    int part;
    if (w < a.prefix_tiles * a.prefix_splits) {
        const int split = w / a.prefix_tiles;
        s.q0 = min(max(a.q_start[0], 0), a.rows);
        s.n = min(max(a.q_start[a.requests], 0), a.rows) - s.q0;
        s.first = (w - split * a.prefix_tiles) * TILE;
        if (s.first >= s.n * a.group) return;
        s.k = static_cast<const T*>(a.prefix_k) + kvh * HD;
        s.v = static_cast<const T*>(a.prefix_v) + kvh * HD;
        s.ldk = a.ld_prefix_k;
        s.ldv = a.ld_prefix_v;
        s.k0 = split * a.prefix_chunk;
        s.k1 = min(s.k0 + a.prefix_chunk, a.prefix);
        s.causal = false;
        s.limit0 = 0;
        part = split;
    } else {
        w -= a.prefix_tiles * a.prefix_splits;
        const int split = w / a.own_tiles;
        int request, tile;
        if (!find_tile(a, w - split * a.own_tiles, request, tile)) return;
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
        part = a.prefix_splits + split;
    }
    attend<T, HD>(a, s, kvh, a.parts > 1 ? part : -1, lds, wave_m, wave_l, total);
}

// One (row, head) per HD / 4 lanes.
template <int HD>
__global__ __launch_bounds__(256) void attn_merge_kernel(PrefixAttnArgs a) {
    constexpr int QUADS = HD / 4;
    const int64_t item = (int64_t(blockIdx.x) * 256 + threadIdx.x) / QUADS, items = int64_t(a.rows) * a.heads;
    const int d = 4 * (threadIdx.x % QUADS);
    if (item >= items) return;
    const int64_t row = item / a.heads, h = item - row * a.heads;
    if (row < min(max(a.q_start[0], 0), a.rows) || row >= min(max(a.q_start[a.requests], 0), a.rows)) return;
    float m = -__builtin_inff();
    for (int p = 0; p < a.parts; ++p) m = fmaxf(m, a.part_ml[(p * items + item) * 2]);
    float l = 0.f;
    floatx4 v{0.f, 0.f, 0.f, 0.f};
    for (int p = 0; p < a.parts; ++p) {
        const float lp = a.part_ml[(p * items + item) * 2 + 1];
        if (lp == 0.f) continue;   // no key in this part
        const float f = __builtin_amdgcn_exp2f(a.part_ml[(p * items + item) * 2] - m);
        l += lp * f;
        v += *reinterpret_cast<const floatx4*>(a.part_o + (p * items + item) * HD + d) * f;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    reinterpret_cast<Float4At*>(a.out + row * a.ldo + h * HD + d)->v = v * inv;
}

template <class T, int HD>
void launch_typed(const PrefixAttnArgs& a, hipStream_t stream) {
    const unsigned groups = unsigned(a.prefix_tiles) * a.prefix_splits + unsigned(a.own_tiles) * a.own_splits;
    prefix_attn_kernel<T, HD><<<dim3(groups, a.kv_heads), 64 * WAVES, 0, stream>>>(a);
    if (a.parts > 1) {
        const int64_t threads = int64_t(a.rows) * a.heads * (HD / 4);
        attn_merge_kernel<HD><<<unsigned((threads + 255) / 256), 256, 0, stream>>>(a);
    }
}

}  // namespace

// Two workgroups per CU where the keys allow splits of 256.
void prefix_attn_plan(PrefixAttnArgs& a, int cus) {
    const auto splits = [&](int64_t groups, int64_t keys) {
        return int(std::max<int64_t>(1, std::min<int64_t>((2 * cus + groups - 1) / groups, (keys + 255) / 256)));
    };
    const auto chunk = [](int64_t keys, int n) { return int(((keys + n - 1) / n + TILE * WAVES - 1) / (TILE * WAVES) * (TILE * WAVES)); };
    a.group = a.heads / a.kv_heads;
    const int64_t places = int64_t(a.rows) * a.group;
    a.prefix_tiles = a.prefix ? int((places + TILE - 1) / TILE) : 0;
    a.prefix_splits = a.prefix ? splits(int64_t(a.prefix_tiles) * a.kv_heads, a.prefix) : 0;
    if (a.prefix) {
        a.prefix_chunk = chunk(a.prefix, a.prefix_splits);
        a.prefix_splits = (a.prefix + a.prefix_chunk - 1) / a.prefix_chunk;
    }
    // without a prefix the own parts write every row, an empty one as zeros
    const bool own = a.own_max > 0 || !a.prefix;
    a.own_tiles = own ? int(places / TILE + std::min<int64_t>(a.requests, a.rows)) : 0;
    a.own_splits = own ? splits(int64_t(a.own_tiles) * a.kv_heads, a.own_max) : 0;
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
