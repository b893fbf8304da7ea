// Rotary positions, and the rows of keys and values of a batch of requests to
// and from caches in Q8_0 or Q4_0 pages.
//
// Rotation: pair (x0, x1) by angle = position * frequency:
//   y0 = x0 cos - x1 sin,  y1 = x0 sin + x1 cos.
// The angle is an F64 number (in F32 one of 10^5 would be off by 2^-8), cos and
// sin come from their series on an eighth of a turn, in F64, and are rounded
// once.  A workgroup makes them once for its rows and all of a row's heads.
// All of it is bound by memory: one pass, 16-byte loads and stores.  5184 rows of
// 32 heads of 64, F32: 16.2 us (5.2 TB/s, partly from the MALL); 41472 rows of 16
// heads, F16: 34.0 (5.0).  Rows to a cache: 41472 of 512 F32 values of keys and
// values, keys rotated, Q4_0: 45 us from HBM (4.3 TB/s; 41 from the MALL), Q8_0
// 47; back as F16: 30 (21) of either, as F32 58 and 53.  A call of few rows is one
// launch of 3 to 5 us, a chain of loads: tables, page, block.
#include <algorithm>

#include "kv_cache.hpp"
#include "q8stage.hpp"

#pragma clang fp contract(off)

namespace samhip {

namespace {

constexpr int THREADS = 256;
constexpr int kMaxTable = 1024;   // (cos, sin) of a workgroup's rows, and its most rows
constexpr int kMaxRows = 32;

template <class T, int V>
struct Pack {
    typedef T type __attribute__((ext_vector_type(V), aligned(sizeof(T))));
};
typedef uint32_t u32x2_at __attribute__((ext_vector_type(2), aligned(2)));

// cos and sin of an F64 angle below 2^52, each the F64 value rounded.  Whole
// quarter turns k leave exactly: k and pi / 2's first 53 bits have a product
// of whole 2^-52, and so does what is left of the angle; the bits behind them
// follow.  The series end where their next term is below 2^-49 of the sum.
__device__ __forceinline__ float2 cos_sin(double angle) {
    const double k = __builtin_rint(angle * 0.636619772367581343);
    double a = __builtin_fma(-k, 1.5707963267948965580, angle);
    a = __builtin_fma(-k, 6.1232339957367660359e-17, a);
    const double z = a * a;
    double s = 1.0 / 6227020800.0, c = -1.0 / 87178291200.0;
    s = __builtin_fma(s, z, -1.0 / 39916800.0);
    s = __builtin_fma(s, z, 1.0 / 362880.0);
    s = __builtin_fma(s, z, -1.0 / 5040.0);
    s = __builtin_fma(s, z, 1.0 / 120.0);
    s = __builtin_fma(s, z, -1.0 / 6.0);
    s = __builtin_fma(s * z, a, a);
    c = __builtin_fma(c, z, 1.0 / 479001600.0);
    c = __builtin_fma(c, z, -1.0 / 3628800.0);
    c = __builtin_fma(c, z, 1.0 / 40320.0);
    c = __builtin_fma(c, z, -1.0 / 720.0);
    c = __builtin_fma(c, z, 1.0 / 24.0);
    c = __builtin_fma(c, z, -0.5);
    c = __builtin_fma(c, z, 1.0);
    const int quarter = int(int64_t(k)) & 3;
    const double x = quarter & 1 ? s : c, y = quarter & 1 ? c : s;
    return float2{float(quarter == 1 || quarter == 2 ? -x : x), float(quarter >= 2 ? -y : y)};
}

// table[i * pairs + p] for rows row0 + i
__device__ __forceinline__ void fill_rotations(const RopeArgs& rope, Divisor pairs, int row0, int n, float2* table) {
    for (int t = threadIdx.x; t < n * rope.pairs; t += THREADS) {
        const int i = int(pairs.quotient(t)), p = t - i * rope.pairs;
        const int position = rope.positions[int64_t(row0 + i) * rope.axes + rope.axis[p]];
        table[t] = cos_sin(double(position) * rope.frequency[p]);
    }
}

struct RopeShape {
    int rows_each;              // rows of a workgroup
    int rotated, chunks;        // HALVES: chunks of pairs, then of what is left; ADJACENT: chunks of values
    Divisor per_row, per_head, pairs;   // heads * chunks, chunks
};

// A chunk is 16 bytes of x (HALVES: and 16 of the pairs' second values).
template <class TI, class TO, bool HALVES>
__global__ __launch_bounds__(THREADS) void rope_kernel(RopeRows r, RopeArgs rope, RopeShape s) {
    constexpr int V = 16 / int(sizeof(TI)), AT_ONCE = 4;
    typedef typename Pack<TI, V>::type In;
    typedef typename Pack<TO, V>::type Out;
    __shared__ float2 table[kMaxTable];
    const int row0 = blockIdx.x * s.rows_each, n = min(s.rows_each, r.rows - row0), P = rope.pairs, hd = r.head_dim;
    fill_rotations(rope, s.pairs, row0, n, table);
    __syncthreads();
    const TI* x = static_cast<const TI*>(r.x);
    TO* y = static_cast<TO*>(r.y);
    const int items = n * int(s.per_row.d);
    for (int base = threadIdx.x; base < items; base += THREADS * AT_ONCE) {
        In a[AT_ONCE], b[AT_ONCE];
        int row[AT_ONCE], at[AT_ONCE], d0[AT_ONCE], first[AT_ONCE];   // values of one part: pairs (HALVES) or values
        const auto place = [&](int u) {
            const int t = base + u * THREADS;
            row[u] = int(s.per_row.quotient(t));
            const int in_row = t - row[u] * int(s.per_row.d), head = int(s.per_head.quotient(in_row)), c = in_row - head * s.chunks;
            const bool pairs = HALVES && c < s.rotated;
            d0[u] = pairs ? V * c : HALVES ? 2 * P + V * (c - s.rotated) : V * c;
            first[u] = (pairs ? P : hd) - d0[u];
            at[u] = head * hd + d0[u];
        };
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) {
            if (base + u * THREADS >= items) break;
            place(u);
            const TI* from = x + (row0 + row[u]) * r.ldx + at[u];
            const bool pairs = HALVES && d0[u] < P;
            if (first[u] >= V) {
                a[u] = *reinterpret_cast<const In*>(from);
                if (pairs) b[u] = *reinterpret_cast<const In*>(from + P);
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    a[u][j] = j < first[u] ? from[j] : TI(0);
                    if (pairs) b[u][j] = j < first[u] ? from[P + j] : TI(0);
                }
            }
        }
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) {
            if (base + u * THREADS >= items) break;
            const bool pairs = HALVES && d0[u] < P;
            const float2* cs = table + row[u] * P;
            Out ya, yb;
#pragma unroll
            for (int j = 0; j < V; ++j) ya[j] = TO(a[u][j]);
            yb = ya;
            if (HALVES) {
                if (pairs) {
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        const float2 w = cs[min(d0[u] + j, P - 1)];
                        const float x0 = float(a[u][j]), x1 = float(b[u][j]);
                        ya[j] = TO(x0 * w.x - x1 * w.y);
                        yb[j] = TO(x0 * w.y + x1 * w.x);
                    }
                }
            } else {
#pragma unroll
                for (int j = 0; j < V; j += 2) {
                    const int p = (d0[u] + j) >> 1;
                    if (p < P) {
                        const float2 w = cs[p];
                        const float x0 = float(a[u][j]), x1 = float(a[u][j + 1]);
                        ya[j] = TO(x0 * w.x - x1 * w.y);
                        ya[j + 1] = TO(x0 * w.y + x1 * w.x);
                    }
                }
            }
            TO* to = y + (row0 + row[u]) * r.ldy + at[u];
            if (first[u] >= V) {
                *reinterpret_cast<Out*>(to) = ya;
                if (pairs) *reinterpret_cast<Out*>(to + P) = yb;
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (j < first[u]) {
                        to[j] = ya[j];
                        if (pairs) to[P + j] = yb[j];
                    }
            }
        }
    }
}

// Eight neighbouring values of a key row, turned.
__device__ __forceinline__ void turn8(floatx8& v, const float* head, int d0, const RopeArgs& rope, const float2* cs) {
    const int P = rope.pairs;
    if (d0 >= 2 * P) return;
    if (!rope.halves) {
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            const int p = (d0 + j) >> 1;
            if (p < P) {
                const float2 w = cs[p];
                const float x0 = v[j], x1 = v[j + 1];
                v[j] = x0 * w.x - x1 * w.y;
                v[j + 1] = x0 * w.y + x1 * w.x;
            }
        }
        return;
    }
    floatx8 other;
    if (P % 8 == 0) {
        typedef typename Pack<float, 4>::type F4;
        const float* from = head + (d0 < P ? d0 + P : d0 - P);
        const F4 a = *reinterpret_cast<const F4*>(from), b = *reinterpret_cast<const F4*>(from + 4);
        other = floatx8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int d = d0 + j;
            other[j] = head[d < P ? d + P : d < 2 * P ? d - P : d];
        }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int d = d0 + j;
        if (d < P) v[j] = v[j] * cs[d].x - other[j] * cs[d].y;
        else if (d < 2 * P) v[j] = other[j] * cs[d - P].y + v[j] * cs[d - P].x;
    }
}

// The first value of the largest magnitude of a quad of lanes, NaNs passed over.
__device__ __forceinline__ float quad_first_largest(const floatx8& v) {
    const int lane = threadIdx.x & 63;
    float most = 0.f, value = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (fabsf(v[j]) > most) most = fabsf(v[j]), value = v[j];
    const auto take = [&](float om, float ov, bool behind) {
        if (om > most || (om == most && behind)) most = om, value = ov;
    };
    take(dpp<DPP_XOR1>(most), dpp<DPP_XOR1>(value), lane & 1);
    take(dpp<DPP_XOR2>(most), dpp<DPP_XOR2>(value), lane & 2);
    return value;
}

struct CacheRowShape {
    int rows_each;
    Divisor per_row, per_tensor, pairs;   // items of a row of both tensors, of one
};

// Where a workgroup's rows stand: the last wave's work, for the first has the
// rotations of a few rows.
__device__ __forceinline__ void find_places(const KvCacheArgs& c, int rows, int row0, int n, int* place) {
    static_assert(kMaxRows <= 64, "one wave finds them");
    if (threadIdx.x < THREADS - 64) return;
    const int r = first_above(c.row_start + 1, c.requests, row0), i = threadIdx.x & 63;
    if (i < n) place[i] = place_of_row(c, rows, row0 + i, r);
}

// Eight values to a lane, four lanes to a block, which is stored in pieces: rows
// of two workgroups with one place may leave a mixed one.
template <int TYPE, bool X86>
__global__ __launch_bounds__(THREADS) void cache_write_kernel(KvCacheArgs c, RopeArgs rope, CacheRowShape s, const float* k, int64_t ldk,
                                                              const float* v, int64_t ldv, int rows) {
    typedef typename Pack<float, 4>::type F4;
    __shared__ float2 table[kMaxTable];
    __shared__ int place[kMaxRows];
    const int row0 = blockIdx.x * s.rows_each, n = min(s.rows_each, rows - row0), lane = threadIdx.x & 63;
    const int items = n * int(s.per_row.d);
    struct Item {
        int i = 0, octet = 0;
        bool is = false, of_k = false;
        const float* row = nullptr;
        F4 a{0.f, 0.f, 0.f, 0.f}, b{0.f, 0.f, 0.f, 0.f};
    };
    const auto fetch = [&](int t) {
        Item item;
        item.is = t < items;
        if (!item.is) return item;
        item.i = int(s.per_row.quotient(t));
        const int in_row = t - item.i * int(s.per_row.d);
        item.of_k = in_row < int(s.per_tensor.d);
        item.octet = item.of_k ? in_row : in_row - int(s.per_tensor.d);
        item.row = item.of_k ? k + (row0 + item.i) * ldk : v + (row0 + item.i) * ldv;
        item.a = *reinterpret_cast<const F4*>(item.row + 8 * item.octet);
        item.b = *reinterpret_cast<const F4*>(item.row + 8 * item.octet + 4);
        return item;
    };
    Item next = fetch(threadIdx.x);   // under way beside the tables
    find_places(c, rows, row0, n, place);
    fill_rotations(rope, s.pairs, row0, n, table);
    __syncthreads();
    for (int base = 0; base < items; base += THREADS) {   // whole waves: the lanes of a block talk to each other
        const Item item = next;
        if (base + THREADS < items) next = fetch(base + THREADS + threadIdx.x);
        const int octet = item.octet;
        const bool of_k = item.of_k;
        const int to = item.is ? place[item.i] : -1;
        floatx8 x{item.a[0], item.a[1], item.a[2], item.a[3], item.b[0], item.b[1], item.b[2], item.b[3]};
        if (of_k && rope.pairs) {
            const int d0 = 8 * octet & (c.head_dim - 1);
            turn8(x, item.row + (8 * octet - d0), d0, rope, table + item.i * rope.pairs);
        }
        uint32_t w0 = 0, w1 = 0;
        float d, mul;
        if (TYPE == T_Q8_0) {
            quant8_scale_ordered<T_Q8_0, X86>(x, lane, d, mul);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t code = uint32_t(cvt_i32_nan0(quant8_round<T_Q8_0, X86>(x[j] * mul))) & 0xffu;
                if (j < 4) w0 |= code << (8 * j);
                else w1 |= code << (8 * (j - 4));
            }
        } else {
            d = quad_first_largest(x) * -0.125f;   // exact unless subnormal, and then rounded as the quotient is
            mul = d != 0.f ? 1.f / d : 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float r = x[j] * mul + 8.5f;
                const uint32_t code = r == r ? uint32_t(min(max(cvt_i32_nan0(__builtin_truncf(r)), 0), 15)) : 8u;
                if (j < 4) w0 |= code << (8 * j);
                else w1 |= code << (8 * (j - 4));
            }
            w0 |= uint32_t(dpp<DPP_XOR2>(int(w0))) << 4;   // lanes 0 and 1 of the quad: values 16 on in the high halves
            w1 |= uint32_t(dpp<DPP_XOR2>(int(w1))) << 4;
        }
        if (to < 0) continue;
        uint8_t* block = (of_k ? c.k + int64_t(to) * c.ldk : c.v + int64_t(to) * c.ldv) + (octet >> 2) * block_bytes(TYPE);
        if ((lane & 3) == 0) *reinterpret_cast<uint16_t*>(block) = float_to_half_bits(d);
        if (TYPE == T_Q8_0 || (lane & 2) == 0) *reinterpret_cast<u32x2_at*>(block + 2 + 8 * (octet & (TYPE == T_Q8_0 ? 3 : 1))) = u32x2_at{w0, w1};
    }
}

// Eight bytes of codes to a lane: 8 values of Q8_0, 8 and the 8 that stand 16
// behind them of Q4_0.
template <int TYPE, class TO>
__global__ __launch_bounds__(THREADS) void cache_read_kernel(KvCacheArgs c, CacheRowShape s, TO* k, int64_t ldk, TO* v, int64_t ldv, int rows) {
    typedef typename Pack<TO, 8>::type Out;
    constexpr int EACH = TYPE == T_Q8_0 ? 4 : 2;   // lanes to a block
    __shared__ int place[kMaxRows];
    const int row0 = blockIdx.x * s.rows_each, n = min(s.rows_each, rows - row0);
    find_places(c, rows, row0, n, place);
    __syncthreads();
    const int items = n * int(s.per_row.d);
    constexpr int AT_ONCE = 4;   // loads under way together (24 requests of 512 values a row: 58.7 us, one by one 63.3)
    for (int base = threadIdx.x; base < items; base += AT_ONCE * THREADS) {
        int from[AT_ONCE];
        uint32_t d[AT_ONCE];
        u32x2_at w[AT_ONCE];
        TO* to[AT_ONCE];
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) {
            const int t = base + u * THREADS;
            from[u] = -2;
            d[u] = 0;
            w[u] = u32x2_at{0, 0};
            if (t >= items) continue;
            const int i = int(s.per_row.quotient(t)), in_row = t - i * int(s.per_row.d);
            const bool of_k = in_row < int(s.per_tensor.d);
            const int item = of_k ? in_row : in_row - int(s.per_tensor.d), part = item % EACH;
            from[u] = place[i];
            to[u] = (of_k ? k + (row0 + i) * ldk : v + (row0 + i) * ldv) + 32 * (item / EACH) + 8 * part;
            if (from[u] >= 0) {
                const uint8_t* block = (of_k ? c.k + int64_t(from[u]) * c.ldk : c.v + int64_t(from[u]) * c.ldv) + item / EACH * block_bytes(TYPE);
                d[u] = *reinterpret_cast<const uint16_t*>(block);
                w[u] = *reinterpret_cast<const u32x2_at*>(block + 2 + 8 * part);
            }
        }
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) {
            if (from[u] == -2) continue;
            const float scale = half_bits_to_float(d[u]);
            Out lo, hi;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t byte = w[u][j >> 2] >> (8 * (j & 3)) & 0xffu;
                if (TYPE == T_Q8_0) {
                    lo[j] = TO(scale * float(int8_t(byte)));
                } else {
                    lo[j] = TO(scale * float(int(byte & 15u) - 8));
                    hi[j] = TO(scale * float(int(byte >> 4) - 8));
                }
            }
            if (from[u] < 0) lo = Out(0), hi = Out(0);
            *reinterpret_cast<Out*>(to[u]) = lo;
            if (TYPE == T_Q4_0) *reinterpret_cast<Out*>(to[u] + 16) = hi;
        }
    }
}

// Rows of a workgroup: some 1024 items, or fewer so that every CU has two.
int rows_of_workgroup(int rows, int items, int pairs, int cus) {
    int each = std::max(1, std::min({1024 / std::max(items, 1), kMaxRows, pairs ? kMaxTable / pairs : kMaxRows}));
    return std::max(1, std::min(each, rows / (2 * cus)));
}

template <class TI, class TO>
void launch_rope_typed(const RopeRows& r, const RopeArgs& rope, int cus, hipStream_t stream) {
    constexpr int V = 16 / int(sizeof(TI));
    RopeShape s;
    const auto chunks = [](int n) { return (n + V - 1) / V; };
    s.rotated = rope.halves ? chunks(rope.pairs) : 0;
    s.chunks = rope.halves ? s.rotated + chunks(r.head_dim - 2 * rope.pairs) : chunks(r.head_dim);
    s.per_row = Divisor::of(uint32_t(r.heads) * s.chunks);
    s.per_head = Divisor::of(s.chunks);
    s.pairs = Divisor::of(rope.pairs);
    s.rows_each = rows_of_workgroup(r.rows, r.heads * s.chunks, rope.pairs, cus);
    const unsigned groups = unsigned((r.rows + s.rows_each - 1) / s.rows_each);
    if (rope.halves) rope_kernel<TI, TO, true><<<groups, THREADS, 0, stream>>>(r, rope, s);
    else rope_kernel<TI, TO, false><<<groups, THREADS, 0, stream>>>(r, rope, s);
}

CacheRowShape cache_row_shape(const KvCacheArgs& c, int values, int pairs, int rows, int cus) {
    CacheRowShape s;
    const int items = c.kv_heads * c.head_dim / values;
    s.per_row = Divisor::of(2 * items);
    s.per_tensor = Divisor::of(items);
    s.pairs = Divisor::of(std::max(pairs, 1));
    s.rows_each = rows_of_workgroup(rows, 2 * items, pairs, cus);
    return s;
}

}  // namespace

void launch_rope(const RopeRows& r, int x_type, int y_type, const RopeArgs& rope, int cus, hipStream_t stream) {
    if (x_type == T_F16) {
        if (y_type == T_F16) launch_rope_typed<_Float16, _Float16>(r, rope, cus, stream);
        else launch_rope_typed<_Float16, float>(r, rope, cus, stream);
    } else {
        if (y_type == T_F16) launch_rope_typed<float, _Float16>(r, rope, cus, stream);
        else launch_rope_typed<float, float>(r, rope, cus, stream);
    }
}

void launch_cache_write(const KvCacheArgs& c, int type, bool x86, const RopeArgs& rope, const float* k, int64_t ldk,
                        const float* v, int64_t ldv, int rows, int cus, hipStream_t stream) {
    const CacheRowShape s = cache_row_shape(c, 8, rope.pairs, rows, cus);
    const unsigned groups = unsigned((rows + s.rows_each - 1) / s.rows_each);
    if (type == T_Q4_0) cache_write_kernel<T_Q4_0, false><<<groups, THREADS, 0, stream>>>(c, rope, s, k, ldk, v, ldv, rows);
    else if (x86) cache_write_kernel<T_Q8_0, true><<<groups, THREADS, 0, stream>>>(c, rope, s, k, ldk, v, ldv, rows);
    else cache_write_kernel<T_Q8_0, false><<<groups, THREADS, 0, stream>>>(c, rope, s, k, ldk, v, ldv, rows);
}

void launch_cache_read(const KvCacheArgs& c, int type, void* k, int64_t ldk, void* v, int64_t ldv, int out_type, int rows,
                       int cus, hipStream_t stream) {
    const CacheRowShape s = cache_row_shape(c, type == T_Q8_0 ? 8 : 16, 0, rows, cus);
    const unsigned groups = unsigned((rows + s.rows_each - 1) / s.rows_each);
    const auto go = [&](auto* kernel, auto* kt, auto* vt) { kernel<<<groups, THREADS, 0, stream>>>(c, s, kt, ldk, vt, ldv, rows); };
    if (out_type == T_F16) {
        _Float16 *kt = static_cast<_Float16*>(k), *vt = static_cast<_Float16*>(v);
        if (type == T_Q4_0) go(cache_read_kernel<T_Q4_0, _Float16>, kt, vt);
        else go(cache_read_kernel<T_Q8_0, _Float16>, kt, vt);
    } else {
        float *kt = static_cast<float*>(k), *vt = static_cast<float*>(v);
        if (type == T_Q4_0) go(cache_read_kernel<T_Q4_0, float>, kt, vt);
        else go(cache_read_kernel<T_Q8_0, float>, kt, vt);
    }
}

}  // namespace samhip
