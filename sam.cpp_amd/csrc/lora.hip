// Low-rank adapters of many requests beside a shared projection:
//   y[m] = base[m] + scale[s] * B[s] (A[s] x[m]),  s = ids[m]
// A and B of all adapters stand in banks of equal slots; a row whose id is
// no slot gets base alone.  Rows come in any order: a workgroup takes 16
// neighbouring rows and goes through the distinct slots among them (one for
// a request's run of tokens), each product on all 16 rows with the other
// slots' rows left out, so there is no sorting and no host copy of the ids.
//   lora_down_kernel : t = A x, the K range split over workgroups
//   lora_up_kernel   : y = base + scale * B t
// Products on the F32 matrix instruction: F32 products and sums throughout.
#include <algorithm>

#include "internal.hpp"

#pragma clang fp contract(off)

namespace samhip {

namespace {

constexpr int ROWS = 16;   // rows of a workgroup

__device__ __forceinline__ floatx4 ld4(const float* p) {   // 4-byte aligned
    struct __attribute__((packed, aligned(4))) unaligned4 {
        floatx4 v;
    };
    return reinterpret_cast<const unaligned4*>(p)->v;
}
__device__ __forceinline__ void st4(float* p, floatx4 v) {
    struct __attribute__((packed, aligned(4))) unaligned4 {
        floatx4 v;
    };
    reinterpret_cast<unaligned4*>(p)->v = v;
}

// N values p[0 .. N) as floats, those at or behind `left` zero and not read.
template <int N>
__device__ __forceinline__ void take(const float* p, int64_t left, float (&v)[N]) {
    if (left >= N) {
#pragma unroll
        for (int j = 0; j < N; j += 4) {
            const floatx4 f = ld4(p + j);
            v[j] = f[0], v[j + 1] = f[1], v[j + 2] = f[2], v[j + 3] = f[3];
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = j < left ? p[j] : 0.f;
    }
}
template <int N>
__device__ __forceinline__ void take(const _Float16* p, int64_t left, float (&v)[N]) {
    typedef _Float16 halves __attribute__((ext_vector_type(N)));
    struct __attribute__((packed, aligned(2))) unaligned {
        halves v;
    };
    if (left >= N) {
        const halves h = reinterpret_cast<const unaligned*>(p)->v;
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = (float)h[j];
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = j < left ? (float)p[j] : 0.f;
    }
}

// The distinct slots of a tile's rows: body(slot, mask of its rows), the
// z-th of every Z.  Every wave sees the same ids and takes the same path.
template <class Body>
__device__ __forceinline__ void for_slots(const LoraArgs& a, int64_t row0, int z, int Z, Body body) {
    const int lane = threadIdx.x & 63;
    const int64_t row = row0 + lane;
    const int id = lane < ROWS && row < a.m ? a.ids[row] : -1;
    uint32_t left = uint32_t(__ballot(id >= 0 && id < a.slots));
    for (int i = 0; left; ++i) {
        const int slot = __builtin_amdgcn_readlane(id, __builtin_ctz(left));
        const uint32_t mask = uint32_t(__ballot(id == slot)) & left;
        left &= ~mask;
        if (i % Z == z) body(slot, mask);
    }
}

__device__ __forceinline__ int slot_rank(const LoraArgs& a, int slot) {
    return a.ranks ? min(max(a.ranks[slot], 0), a.rank) : a.rank;
}

// Grid: row tiles x K splits x slot lanes.  The 4 waves share the split's K
// range in steps of 32 values; lane (r, g) of a step holds row r's values
// 8g .. 8g + 7 of both operands, the K order of either being the same.
template <class T, int RT>
__global__ __launch_bounds__(256) void lora_down_kernel(LoraArgs a) {
    __shared__ floatx4 red[3][RT][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = lane & 15, g = lane >> 4;
    const int64_t row0 = int64_t(blockIdx.x) * ROWS;
    const int k0 = blockIdx.y * a.k_len, k1 = min(a.k, k0 + a.k_len);
    for_slots(a, row0, blockIdx.z, gridDim.z, [&](int slot, uint32_t mask) {
        const int rank = slot_rank(a, slot), tiles = (rank + 15) / 16;
        const bool mine = (mask >> r) & 1;
        const float* x = a.x + (row0 + r) * a.ldx;
        const T* w = static_cast<const T*>(a.a) + slot * a.a_slot;
        floatx4 acc[RT];
#pragma unroll
        for (int t = 0; t < RT; ++t) acc[t] = floatx4{0.f, 0.f, 0.f, 0.f};
        for (int k = k0 + 32 * wave + 8 * g; k < k1 + 8 * g; k += 128) {
            float xv[8], av[8];
            take<8>(x + k, mine ? k1 - k : 0, xv);
#pragma unroll
            for (int t = 0; t < RT; ++t) {
                if (t < tiles) {
                    const int q = 16 * t + r;
                    take<8>(w + q * a.a_row + k, q < rank ? k1 - k : 0, av);
#pragma unroll
                    for (int j = 0; j < 8; ++j) acc[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(av[j], xv[j], acc[t], 0, 0, 0);
                }
            }
        }
        // lane (r, g) holds row r's ranks 16t + 4g .. + 3
        if (wave) {
#pragma unroll
            for (int t = 0; t < RT; ++t)
                if (t < tiles) red[wave - 1][t][lane] = acc[t];
        }
        __syncthreads();
        if (wave == 0 && mine) {
            float* out = a.part + ((blockIdx.y * a.m + row0 + r) * a.part_ld + 4 * g);
#pragma unroll
            for (int t = 0; t < RT; ++t)
                if (t < tiles) *reinterpret_cast<floatx4*>(out + 16 * t) = acc[t] + red[0][t][lane] + red[1][t][lane] + red[2][t][lane];
        }
        __syncthreads();
    });
}

// Grid: row tiles x blocks of 256 columns x slot lanes; 64 columns a wave.
template <class T, int RT>
__global__ __launch_bounds__(256) void lora_up_kernel(LoraArgs a) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = lane & 15, g = lane >> 4;
    const int64_t row0 = int64_t(blockIdx.x) * ROWS, row = row0 + r;
    const int n0 = blockIdx.y * 256 + wave * 64;
    // base and y of this lane's row, columns n .. n + 3
    auto put = [&](int n, floatx4 v) {
        if (n + 4 <= a.n) {
            if (a.base) v += ld4(a.base + row * a.ldbase + n);
            st4(a.y + row * a.ldy + n, v);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (n + j < a.n) a.y[row * a.ldy + n + j] = a.base ? v[j] + a.base[row * a.ldbase + n + j] : v[j];
        }
    };
    for_slots(a, row0, blockIdx.z, gridDim.z, [&](int slot, uint32_t mask) {
        const int rank = slot_rank(a, slot), tiles = (rank + 15) / 16;
        const float scale = a.scales ? a.scales[slot] : 1.f;
        const bool mine = (mask >> r) & 1;
        floatx4 t[RT];
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            t[i] = floatx4{0.f, 0.f, 0.f, 0.f};
            if (i < tiles && mine) {
                for (int s = 0; s < a.splits; ++s)
                    t[i] += *reinterpret_cast<const floatx4*>(a.part + (s * a.m + row) * a.part_ld + 16 * i + 4 * g);
#pragma unroll
                for (int j = 0; j < 4; ++j) t[i][j] = 16 * i + 4 * g + j < rank ? t[i][j] * scale : 0.f;
            }
        }
        const T* w = static_cast<const T*>(a.b) + slot * a.b_slot;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const int n = n0 + 16 * c;
            if (n >= a.n) break;
            floatx4 acc{0.f, 0.f, 0.f, 0.f};
            const T* wr = w + min(n + r, a.n - 1) * a.b_row + 4 * g;
#pragma unroll
            for (int i = 0; i < RT; ++i) {
                if (i < tiles) {
                    float bv[4];
                    take<4>(wr + 16 * i, rank - (16 * i + 4 * g), bv);
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(bv[j], t[i][j], acc, 0, 0, 0);
                }
            }
            if (mine) put(n + 4 * g, acc);
        }
    });
    if (blockIdx.z == 0 && row < a.m && (a.base != a.y || a.ldbase != a.ldy)) {   // rows without an adapter
        const int id = a.ids[row];
        if (id < 0 || id >= a.slots)
#pragma unroll
            for (int c = 0; c < 4; ++c) put(n0 + 16 * c + 4 * g, floatx4{0.f, 0.f, 0.f, 0.f});
    }
}

template <class T, int RT>
void launch_ranks(const LoraArgs& a, int slot_lanes, hipStream_t stream) {
    const unsigned tiles = unsigned((a.m + ROWS - 1) / ROWS);
    lora_down_kernel<T, RT><<<dim3(tiles, a.splits, slot_lanes), 256, 0, stream>>>(a);
    lora_up_kernel<T, RT><<<dim3(tiles, (a.n + 255) / 256, slot_lanes), 256, 0, stream>>>(a);
}

template <class T>
void launch_typed(const LoraArgs& a, int slot_lanes, hipStream_t stream) {
    if (a.rank <= 16) launch_ranks<T, 1>(a, slot_lanes, stream);
    else if (a.rank <= 32) launch_ranks<T, 2>(a, slot_lanes, stream);
    else if (a.rank <= 64) launch_ranks<T, 4>(a, slot_lanes, stream);
    else if (a.rank <= 128) launch_ranks<T, 8>(a, slot_lanes, stream);
    else launch_ranks<T, 16>(a, slot_lanes, stream);
}

}  // namespace

// About two workgroups per CU from splits of at least 256 values of K.
int lora_splits(int64_t m, int k, int cus) {
    const int64_t tiles = (m + ROWS - 1) / ROWS;
    return int(std::max<int64_t>(1, std::min<int64_t>((2 * cus + tiles - 1) / tiles, (k + 255) / 256)));
}

size_t lora_part_bytes(int64_t m, int rank, int splits) { return size_t(splits) * size_t(m) * ((rank + 15) / 16 * 16) * 4; }

void launch_lora(LoraArgs a, int type, int cus, hipStream_t stream) {
    const int64_t tiles = (a.m + ROWS - 1) / ROWS;
    a.k_len = ((a.k + a.splits - 1) / a.splits + 127) / 128 * 128;
    a.part_ld = (a.rank + 15) / 16 * 16;
    const int slot_lanes = int(std::max<int64_t>(1, std::min<int64_t>({2 * cus / tiles, ROWS, a.slots})));
    if (type == T_F16) launch_typed<_Float16>(a, slot_lanes, stream);
    else launch_typed<float>(a, slot_lanes, stream);
}

}  // namespace samhip
