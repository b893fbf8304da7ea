// Low-rank adapters of many requests beside a shared projection:
//   y[m] = base[m] + scale[s] * B[s] (A[s] x[m]),  s = ids[m]
// A and B of all adapters stand in banks of equal slots; a row whose id is
// no slot gets base alone.  Rows come in any order and the ids stay on the
// device: a workgroup counts the ids of its block of rows per slot, which
// numbers the block's tiles of 16 or 32 rows of one slot, and picks its own
// tile's rows in row order, so that scattered rows cost no more products
// than sorted ones (777 rows of 24 slots in no order, K = 1001, N = 1359,
// ranks to 40: 54 us with tiles of neighbouring rows that went through
// their slots one by one).  Rows without a slot form tiles of their own
// that only copy base.
//   lora_fused_kernel : few tiles; t = A x and its share of B t in one launch
//   lora_down_kernel  : t = A x, the K range split over workgroups
//   lora_up_kernel    : y = base + scale * B t
// Products on the F32 matrix instruction: F32 products and sums throughout.
// Bound by HBM with many rows (41472 x 1024 -> 4736, rank 32, 8 slots: 419 us,
// 4.1 TB/s, most of it the second launch, from base to y; a copy of the bytes
// takes 364), by one or two launches' latency with few (16 rows 1024 -> 1024,
// rank 16: 6.3 us; 256 rows 1024 -> 4096: 10.0), by A from L2 where K is the
// long side of a high rank (8260 x 3591 -> 273, rank 47, F32: 114 us, 28 of
// bytes), and past rank 64 by tiles too small for the matrix instruction (41472
// x 1024 -> 1024, 8 slots: 387 us at rank 128, 1125 at 256, where the
// instruction takes 126 and 252).
#include <algorithm>

#include "internal.hpp"

#pragma clang fp contract(off)

namespace samhip {

namespace {

typedef float float4_at __attribute__((ext_vector_type(4), aligned(4)));

__device__ __forceinline__ floatx4 ld4(const float* p) { return *reinterpret_cast<const float4_at*>(p); }
// PAST: past the caches (a template's argument: of two stores in the branches
// of a condition the compiler makes an ordinary one)
template <bool PAST>
__device__ __forceinline__ void st4(float* p, floatx4 v) {
    if constexpr (PAST) __builtin_nontemporal_store(v, reinterpret_cast<float4_at*>(p));
    else *reinterpret_cast<float4_at*>(p) = v;
}

typedef _Float16 half4_at __attribute__((ext_vector_type(4), aligned(2)));
__device__ __forceinline__ floatx4 take4(const float* p) { return ld4(p); }
__device__ __forceinline__ floatx4 take4(const _Float16* p) {
    const half4_at h = *reinterpret_cast<const half4_at*>(p);
    return floatx4{(float)h[0], (float)h[1], (float)h[2], (float)h[3]};
}
// v[off ..], zeros behind
template <int N, class V>
__device__ __forceinline__ V shift_down(V v, int off) {
#pragma unroll
    for (int s = 1; s < N; s *= 2)
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = off & s ? (j + s < N ? v[j + s] : 0) : v[j];
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = off >= N ? 0 : v[j];
    return v;
}
// row[n .. n + 4) as floats, those at or behind `end` zero and not read.  A
// branch around a load has it waited for at once, so how a group of loads is
// done is chosen outside of it: WHOLE reads them as they are, SHIFTED (end at
// least 4) the last whole vector again, shifted, GUARDED one by one.
enum class Edge { WHOLE, SHIFTED, GUARDED };
template <Edge E, class T>
__device__ __forceinline__ floatx4 take4(const T* row, int n, int end) {
    if constexpr (E == Edge::WHOLE) return take4(row + n);
    if constexpr (E == Edge::SHIFTED) {
        const int at = min(n, end - 4);
        return shift_down<4>(take4(row + at), n - at);
    }
    floatx4 v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 3; ++j)
        if (n + j < end) v[j] = (float)row[n + j];
    return v;
}
template <Edge E>
struct EdgeTag {
    static constexpr Edge value = E;
};
template <class Body>
__device__ __forceinline__ void with_edge(bool whole, int end, Body body) {   // uniform
    if (whole) body(EdgeTag<Edge::WHOLE>{});
    else if (end >= 4) body(EdgeTag<Edge::SHIFTED>{});
    else body(EdgeTag<Edge::GUARDED>{});
}

__device__ __forceinline__ floatx4 mfma(float a, float b, floatx4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

// Inclusive sums over the wave's lanes: within rows of 16 by shifts, then the
// last lane of each row (15, 31 of the half) onto the rows behind it.
__device__ __forceinline__ int prefix_sum(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);    // row_shr:1
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);   // row_bcast:15 onto rows 1 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);   // row_bcast:31 onto rows 2 and 3
    return v;
}

// The rows of one tile: offsets from the block's first row, -1 where the
// tile has fewer.
template <int TR>
struct Tile {
    int rows[TR];
    int counts[64];   // matches per wave and pass
};

// The p-th tile of a block of `n` rows (at most 4096): its slot (a.slots: rows
// without one), or -1 past the last tile.  hist: slots + 1 counters.
template <int TR, int THREADS, int PASSES>
__device__ __forceinline__ int find_tile(const LoraArgs& a, const int32_t* ids, int n, int p, int* hist, Tile<TR>& tile) {
    constexpr int WAVES = THREADS / 64;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int key[PASSES];   // slots of rows tid, tid + THREADS, ..; -1 where none is to be moved
#pragma unroll
    for (int i = 0; i < PASSES; ++i) key[i] = ids[min(i * THREADS + tid, n - 1)];
    for (int s = tid; s <= a.slots; s += THREADS) hist[s] = 0;
    if (tid < TR) tile.rows[tid] = -1;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        const int id = key[i], s = i * THREADS + tid >= n ? -1 : id >= 0 && id < a.slots ? id : a.copy_bare ? a.slots : -1;
        key[i] = s;
        // one request's rows in a run: one addition for the wave
        const int s0 = __builtin_amdgcn_readfirstlane(s);
        if (__all(s == s0)) {
            if (s0 >= 0 && lane == 0) atomicAdd(&hist[s0], 64);
        } else if (s >= 0) {
            atomicAdd(&hist[s], 1);
        }
    }
    __syncthreads();
    int slot = -1, skip = 0, before = 0;
    for (int s0 = 0; s0 <= a.slots && slot < 0; s0 += 64) {
        const int tiles = s0 + lane <= a.slots ? (hist[s0 + lane] + TR - 1) / TR : 0;
        const int sum = prefix_sum(tiles);
        const uint64_t past = __ballot(before + sum > p);
        if (past) {
            const int at = __builtin_ctzll(past);
            slot = s0 + at;
            skip = (p - before - __builtin_amdgcn_readlane(sum - tiles, at)) * TR;
        }
        before += __builtin_amdgcn_readlane(sum, 63);
    }
    slot = __builtin_amdgcn_readfirstlane(slot);
    if (slot < 0) return -1;
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        const uint64_t same = __ballot(key[i] == slot);
        if (lane == 0) tile.counts[i * WAVES + wave] = __builtin_popcountll(same);
    }
    __syncthreads();
    const int count = lane < PASSES * WAVES ? tile.counts[lane] : 0, first = prefix_sum(count) - count;
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        const uint64_t same = __ballot(key[i] == slot);
        const int ahead = __builtin_amdgcn_readlane(first, i * WAVES + wave) + __builtin_popcountll(same & ((uint64_t(1) << lane) - 1)) - skip;
        if (key[i] == slot && ahead >= 0 && ahead < TR) tile.rows[ahead] = i * THREADS + tid;
    }
    __syncthreads();
    return slot;
}

template <int TR, int THREADS>
__device__ __forceinline__ int find_tile(const LoraArgs& a, const int32_t* ids, int n, int p, int* hist, Tile<TR>& tile) {
    if (n <= THREADS) return find_tile<TR, THREADS, 1>(a, ids, n, p, hist, tile);
    if (n <= 4 * THREADS) return find_tile<TR, THREADS, 4>(a, ids, n, p, hist, tile);
    return find_tile<TR, THREADS, kLoraBlockRows / THREADS>(a, ids, n, p, hist, tile);
}

__device__ __forceinline__ int slot_rank(const LoraArgs& a, int slot) {
    return a.ranks ? min(max(a.ranks[slot], 0), a.rank) : a.rank;
}

// Operands of t = A x through LDS, KC values of K at a time: lanes of the
// matrix instruction's operands stand for rows, so reading them straight
// from memory takes a cache line per lane; here neighbouring lanes read
// neighbouring 16 bytes of a row, and a chunk is under way during the
// products of the one before.
template <class T, int THREADS, int TR, int RT, int KC>
struct Stage {
    static constexpr int VA = 16 / sizeof(T), XC = KC / 4, AC = KC / VA;                   // 16-byte pieces of a row
    static constexpr int XN = (TR * XC + THREADS - 1) / THREADS, AN = (16 * RT * AC + THREADS - 1) / THREADS;   // of a thread
    typedef T vec __attribute__((ext_vector_type(VA)));
    typedef T vec_at __attribute__((ext_vector_type(VA), aligned(sizeof(T))));
    struct Lds {
        __attribute__((aligned(16))) float x[TR][KC + 4];
        __attribute__((aligned(16))) T a[16 * RT][KC + VA];
    };
    floatx4 x[XN];
    vec w[AN];
    const float* xp[XN];   // this thread's pieces at k = 0
    const T* wp[AN];

    // The tile's rows (block0 + rows[]) and A's first `rank` rows.  An absent
    // row's place gets the tile's first row, places behind the rank its last
    // one: what becomes of them is left out of t.
    __device__ __forceinline__ Stage(const LoraArgs& a, int64_t block0, const int* rows, const T* A, int rank) {
        const int first = rows[0], last = max(rank - 1, 0);
#pragma unroll
        for (int i = 0; i < XN; ++i) {
            const int f = threadIdx.x + i * THREADS, row = rows[min(f / XC, TR - 1)];
            xp[i] = a.x + (block0 + (row < 0 ? first : row)) * a.ldx + f % XC * 4;
        }
#pragma unroll
        for (int i = 0; i < AN; ++i) {
            const int f = threadIdx.x + i * THREADS;
            wp[i] = A + min(f / AC, last) * a.a_row + f % AC * VA;
        }
    }
    // Values [k, k + KC), zeros at or behind k1.  No branch lies between the
    // loads of a whole chunk, which the compiler would have wait for each
    // other there.
    __device__ __forceinline__ void load(int k, int k1) {
        if (k + KC <= k1) {
#pragma unroll
            for (int i = 0; i < XN; ++i) x[i] = ld4(xp[i] + k);
#pragma unroll
            for (int i = 0; i < AN; ++i) w[i] = *reinterpret_cast<const vec_at*>(wp[i] + k);
        } else if (k1 >= VA) {   // the last whole vector again, shifted
#pragma unroll
            for (int i = 0; i < XN; ++i) {
                const int over = max(k + int(threadIdx.x + i * THREADS) % XC * 4 + 4 - k1, 0);
                x[i] = shift_down<4>(ld4(xp[i] + k - over), over);
            }
#pragma unroll
            for (int i = 0; i < AN; ++i) {
                const int over = max(k + int(threadIdx.x + i * THREADS) % AC * VA + VA - k1, 0);
                w[i] = shift_down<VA>(*reinterpret_cast<const vec_at*>(wp[i] + k - over), over);
            }
        } else {
#pragma unroll
            for (int i = 0; i < XN; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) x[i][j] = k + int(threadIdx.x + i * THREADS) % XC * 4 + j < k1 ? xp[i][k + j] : 0.f;
#pragma unroll
            for (int i = 0; i < AN; ++i)
#pragma unroll
                for (int j = 0; j < VA; ++j) w[i][j] = k + int(threadIdx.x + i * THREADS) % AC * VA + j < k1 ? wp[i][k + j] : (T)0;
        }
    }
    __device__ __forceinline__ void store(Lds& l) const {
#pragma unroll
        for (int i = 0; i < XN; ++i) {
            const int f = threadIdx.x + i * THREADS;
            if (TR * XC % THREADS == 0 || f < TR * XC) *reinterpret_cast<floatx4*>(&l.x[f / XC][f % XC * 4]) = x[i];
        }
#pragma unroll
        for (int i = 0; i < AN; ++i) {
            const int f = threadIdx.x + i * THREADS;
            if (16 * RT * AC % THREADS == 0 || f < 16 * RT * AC) *reinterpret_cast<vec*>(&l.a[f / AC][f % AC * VA]) = w[i];
        }
    }
};

// acc[i] += A x of subtile `sub` over the chunk's units first, first + step, ..
// of 16 values: lane (r, g) holds values 4g .. 4g + 3 of row r of both operands
// and ends with row r's ranks 16i + 4g .. + 3.
template <int RT, int UNITS, class Lds>
__device__ __forceinline__ void multiply(const Lds& l, int sub, int first, int step, int tiles, floatx4 (&acc)[RT]) {
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
#pragma unroll RT <= 4 ? UNITS : 1
    for (int n = 0; n < UNITS; ++n) {
        const int at = 16 * (first + n * step) + 4 * g;
        const floatx4 x = *reinterpret_cast<const floatx4*>(&l.x[16 * sub + r][at]);
#pragma unroll
        for (int i = 0; i < RT; ++i)
            if (i < tiles) {
                const auto* p = &l.a[16 * i + r][at];
                const floatx4 w{(float)p[0], (float)p[1], (float)p[2], (float)p[3]};
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i] = mfma(w[j], x[j], acc[i]);
            }
    }
}

// Over [k0, k1), every chunk
template <class T, int THREADS, int TR, int RT, int KC, int UNITS>
__device__ __forceinline__ void down(const LoraArgs& a, typename Stage<T, THREADS, TR, RT, KC>::Lds& lds, int64_t block0, const int* rows, const T* A,
                                     int rank, int k0, int k1, int sub, int first, int step, floatx4 (&acc)[RT]) {
    Stage<T, THREADS, TR, RT, KC> stage(a, block0, rows, A, rank);
    const int tiles = (rank + 15) / 16;
#pragma unroll
    for (int i = 0; i < RT; ++i) acc[i] = floatx4{0.f, 0.f, 0.f, 0.f};
    if (k0 < k1) stage.load(k0, k1);
    for (int k = k0; k < k1; k += KC) {
        if (k != k0) __syncthreads();   // the last chunk is read
        stage.store(lds);
        __syncthreads();
        if (k + KC < k1) stage.load(k + KC, k1);
        multiply<RT, UNITS>(lds, sub, first, step, tiles, acc);
    }
}

// One tile's t for the lane's rows: zero behind the rank, times the scale.
template <int RT>
__device__ __forceinline__ void finish_t(const LoraArgs& a, int slot, int rank, floatx4 (&t)[RT]) {
    const int g = (threadIdx.x & 63) >> 4;
    const float scale = a.scales ? a.scales[slot] : 1.f;
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) t[i][j] = 16 * i + 4 * g + j < rank ? t[i][j] * scale : 0.f;
}

// B's rows n .. n + 15, and their products with t: lane (r, g) ends with row
// r's columns n + 4g .. + 3.
template <class T, int RT>
__device__ __forceinline__ void take_b(const LoraArgs& a, const T* w, int n, int rank, floatx4 (&b)[RT]) {
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const T* row = w + min(n + r, a.n - 1) * a.b_row;
    with_edge(a.rank % 4 == 0, RT > 2 ? 4 : a.rank, [&](auto edge) {
        constexpr Edge E = decltype(edge)::value;
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            const int at = 16 * i + 4 * g;
            b[i] = take4<E>(row, E == Edge::WHOLE ? min(at, a.rank - 4) : at, a.rank);
        }
    });
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) b[i][j] = 16 * i + 4 * g + j < rank ? b[i][j] : 0.f;   // what stands there does not count
}
template <int RT, int SUB>
__device__ __forceinline__ void up(int rank, const floatx4 (&b)[RT], const floatx4 (&t)[SUB][RT], floatx4 (&acc)[SUB]) {
#pragma unroll
    for (int s = 0; s < SUB; ++s) acc[s] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < RT; ++i)
        if (16 * i < rank)
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int s = 0; s < SUB; ++s) acc[s] = mfma(b[i][j], t[s][i][j], acc[s]);
}

template <bool PAST>
__device__ __forceinline__ void put4(const LoraArgs& a, int64_t row, int n, floatx4 v) {
    float* y = a.y + row * a.ldy + n;
    if (n + 4 <= a.n) {
        st4<PAST>(y, v);
    } else {
#pragma unroll
        for (int j = 0; j < 3; ++j)
            if (n + j < a.n) y[j] = v[j];
    }
}

// Grid: tiles x blocks of 256 columns.  The 8 waves share each chunk of K,
// then take 32 columns each.
template <class T, int RT>
__global__ __launch_bounds__(512) void lora_fused_kernel(LoraArgs a) {
    constexpr int KC = 512 / RT;
    extern __shared__ int hist[];
    __shared__ Tile<16> tile;
    __shared__ typename Stage<T, 512, 16, RT, KC>::Lds lds;
    __shared__ floatx4 red[8][RT][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = lane & 15, g = lane >> 4;
    const int slot = find_tile<16, 512>(a, a.ids, int(a.m), blockIdx.x, hist, tile);
    if (slot < 0) return;
    const int row = tile.rows[r], n0 = blockIdx.y * 256 + wave * 32;
    const bool mine = row >= 0;
    const int64_t at = max(row, 0);
    floatx4 base[2];   // under way during the products
    if (a.base) {
        const float* from = a.base + (mine ? at : tile.rows[0]) * a.ldbase;
        with_edge(n0 + 32 <= a.n, a.n, [&](auto edge) {
#pragma unroll
            for (int c = 0; c < 2; ++c) base[c] = take4<decltype(edge)::value>(from, n0 + 16 * c + 4 * g, a.n);
        });
    } else {
        base[0] = base[1] = floatx4{0.f, 0.f, 0.f, 0.f};
    }
    if (slot < a.slots) {
        const int rank = slot_rank(a, slot);
        floatx4 t[1][RT], b[2][RT];
#pragma unroll
        for (int c = 0; c < 2; ++c) take_b<T, RT>(a, static_cast<const T*>(a.b) + slot * a.b_slot, n0 + 16 * c, rank, b[c]);
        down<T, 512, 16, RT, KC, KC / 128>(a, lds, 0, tile.rows, static_cast<const T*>(a.a) + slot * a.a_slot, rank, 0, a.k, 0, wave, 8, t[0]);
#pragma unroll
        for (int i = 0; i < RT; ++i) red[wave][i][lane] = t[0][i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            t[0][i] = red[0][i][lane];
#pragma unroll
            for (int w = 1; w < 8; ++w) t[0][i] += red[w][i][lane];
        }
        finish_t(a, slot, rank, t[0]);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            floatx4 acc[1];
            up<RT, 1>(rank, b[c], t, acc);
            if (mine) base[c] += acc[0];
        }
    }
#pragma unroll
    for (int c = 0; c < 2; ++c)
        if (mine) put4<false>(a, at, n0 + 16 * c + 4 * g, base[c]);
}

// Grid: a block's tiles x blocks of rows x K splits.  The waves of a
// workgroup take a subtile of 16 rows each, and share the chunks of K where
// they are more.  The first split writes the tile's slot and rows down for
// lora_up_kernel.
template <class T, int RT, int SUB>
__global__ __launch_bounds__(256) void lora_down_kernel(LoraArgs a) {
    constexpr int TR = 16 * SUB, KC = RT == 1 ? 256 : RT <= 4 ? 128 : 512 / RT;
    constexpr int SHARE = KC / 16 < 4 / SUB ? KC / 16 : 4 / SUB, UNITS = KC / 16 / SHARE;   // waves of a subtile, and their units of a chunk
    extern __shared__ int hist[];
    __shared__ Tile<TR> tile;
    __shared__ typename Stage<T, 256, TR, RT, KC>::Lds lds;
    __shared__ floatx4 red[SHARE - 1][SUB][RT][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = lane & 15, g = lane >> 4;
    const int64_t block0 = int64_t(blockIdx.y) * a.block_rows;
    const int slot = find_tile<TR, 256>(a, a.ids + block0, int(min(int64_t(a.block_rows), a.m - block0)), blockIdx.x, hist, tile);
    if (blockIdx.z == 0) {
        int* out = a.tiles + (int64_t(blockIdx.y) * gridDim.x + blockIdx.x) * (TR + 1);
        if (tid == 0) out[TR] = slot;
        if (tid < TR && slot >= 0) out[tid] = tile.rows[tid];
    }
    if (slot < 0 || slot == a.slots) return;
    const int rank = slot_rank(a, slot), tiles = (rank + 15) / 16;
    const int k0 = blockIdx.z * a.k_len, k1 = min(a.k, k0 + a.k_len);
    const int sub = wave % SUB, part = wave / SUB;   // a part past SHARE does another's work again, unused
    floatx4 acc[RT];
    down<T, 256, TR, RT, KC, UNITS>(a, lds, block0, tile.rows, static_cast<const T*>(a.a) + slot * a.a_slot, rank, k0, k1, sub,
                                    part % SHARE, SHARE, acc);
    if (part && part < SHARE) {
#pragma unroll
        for (int t = 0; t < RT; ++t)
            if (t < tiles) red[part - 1][sub][t][lane] = acc[t];
    }
    __syncthreads();
    const int row = tile.rows[16 * sub + r];
    if (part || row < 0) return;
    float* out = a.part + (blockIdx.z * a.m + block0 + row) * a.part_ld + 4 * g;
#pragma unroll
    for (int t = 0; t < RT; ++t)
        if (t < tiles) {
#pragma unroll
            for (int p = 1; p < SHARE; ++p) acc[t] += red[p - 1][sub][t][lane];
            *reinterpret_cast<floatx4*>(out + 16 * t) = acc[t];
        }
}

// Grid: column splits x a block's tiles x blocks of rows.  A workgroup goes
// through its split in blocks of 256 columns, 64 to a wave; the sums pass
// through LDS, so that base and y move in whole KB of a row, and the next
// block's base is under way as soon as this one's is used.
template <class T, int RT, int SUB, bool PAST>
__global__ __launch_bounds__(256, RT <= 2 ? 3 : RT <= 4 ? 2 : 1) void lora_up_kernel(LoraArgs a) {
    constexpr int TR = 16 * SUB, PITCH = 256 + 4, OWN = TR / 4;   // rows that a wave moves
    __shared__ __attribute__((aligned(16))) float sums[TR][PITCH];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = lane & 15, g = lane >> 4;
    const int* tile = a.tiles + (int64_t(blockIdx.z) * gridDim.y + blockIdx.y) * (TR + 1);
    const int slot = tile[TR];
    if (slot < 0) return;
    const int64_t block0 = int64_t(blockIdx.z) * a.block_rows;
    const int n0 = blockIdx.x * a.n_len, n1 = min(a.n, n0 + a.n_len);
    floatx4 base[OWN];
    int row[OWN];
#pragma unroll
    for (int i = 0; i < OWN; ++i) row[i] = __builtin_amdgcn_readfirstlane(tile[OWN * wave + i]);
    const bool whole = row[OWN - 1] >= 0;   // rows fill from the front
    const int row0 = tile[0];
#pragma unroll
    for (int i = 0; i < OWN; ++i) base[i] = floatx4{0.f, 0.f, 0.f, 0.f};
    const auto fetch = [&](int nb) {   // an absent row's place gets the block's first
        if (a.base)
            with_edge(nb + 256 <= a.n, a.n, [&](auto edge) {
#pragma unroll
                for (int i = 0; i < OWN; ++i)
                    base[i] = take4<decltype(edge)::value>(a.base + (block0 + max(row[i], 0)) * a.ldbase, nb + 4 * lane, a.n);
            });
    };
    fetch(n0);
    const bool product = slot < a.slots;
    const int rank = product ? slot_rank(a, slot) : 0;
    const T* B = static_cast<const T*>(a.b) + (product ? slot : 0) * a.b_slot;
    // B of a whole block is under way before the stores of the one before: a
    // wait for any load is one for every store that was issued ahead of it
    constexpr int AHEAD = RT <= 2 ? 4 : 1;
    floatx4 t[SUB][RT], b[AHEAD][RT];
    const auto fetch_b = [&](int nb) {
#pragma unroll
        for (int c = 0; c < AHEAD; ++c) take_b<T, RT>(a, B, nb + 64 * wave + 16 * c, rank, b[c]);
    };
    if (product) {
        fetch_b(n0);
        // t of a subtile: no branch between a split's loads, an absent row's
        // or rank tile's place reads the first row's or last tile's
        const int last = max((rank + 15) / 16 - 1, 0);
        const int64_t step = a.m * a.part_ld;
#pragma unroll
        for (int s = 0; s < SUB; ++s) {
            const int at = tile[16 * s + r];
            const float* p = a.part + (block0 + (at < 0 ? row0 : at)) * a.part_ld + 4 * g;
#pragma unroll
            for (int i = 0; i < RT; ++i) t[s][i] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll RT <= 2 ? 4 : 2
            for (int k = 0; k < a.splits; ++k, p += step)
#pragma unroll
                for (int i = 0; i < RT; ++i) t[s][i] += *reinterpret_cast<const floatx4*>(p + 16 * min(i, last));
            finish_t(a, slot, rank, t[s]);
        }
    }
    for (int nb = n0; nb < n1; nb += 256) {
        if (product) {
            if (nb != n0) __syncthreads();   // the last block's sums are read
            // a loop where the ranks make it long: the way of 20 KB more code to
            // the CU takes longer than its steps (38 rows 1623 -> 266 of rank 110
            // 18.9 us unrolled, 13.8 so; rank 40, 777 rows 1001 -> 1359, 9.8 and 10.9)
#pragma unroll RT <= 4 ? 4 : 1
            for (int c = 0; c < 4; ++c) {
                floatx4 acc[SUB], now[RT];
#pragma unroll
                for (int i = 0; i < RT; ++i) now[i] = b[c % AHEAD][i];
                if (AHEAD == 1 && c < 3) take_b<T, RT>(a, B, nb + 64 * wave + 16 * (c + 1), rank, b[0]);
                up<RT, SUB>(rank, now, t, acc);
#pragma unroll
                for (int s = 0; s < SUB; ++s) *reinterpret_cast<floatx4*>(&sums[16 * s + r][64 * wave + 16 * c + 4 * g]) = acc[s];
            }
            if (nb + 256 < n1) fetch_b(nb + 256);
            __syncthreads();
        }
        const int n = nb + 4 * lane;
        const auto sum_of = [&](int i) {
            return product ? base[i] + *reinterpret_cast<const floatx4*>(&sums[OWN * wave + i][4 * lane]) : base[i];
        };
        if (whole && nb + 512 <= n1) {   // without a branch, behind which every wait would be for all
#pragma unroll
            for (int i0 = 0; i0 < OWN; i0 += 4) {
                floatx4 v[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    v[i] = sum_of(i0 + i);
                    if (a.base) base[i0 + i] = ld4(a.base + (block0 + row[i0 + i]) * a.ldbase + n + 256);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) st4<PAST>(a.y + (block0 + row[i0 + i]) * a.ldy + n, v[i]);
            }
        } else {
            floatx4 v[OWN];
#pragma unroll
            for (int i = 0; i < OWN; ++i) v[i] = sum_of(i);
            if (nb + 256 < n1) fetch(nb + 256);
#pragma unroll
            for (int i = 0; i < OWN; ++i)
                if (row[i] >= 0 && n < n1) put4<PAST>(a, block0 + row[i], n, v[i]);
        }
    }
}

template <class T, int RT>
void launch_ranks(const LoraArgs& a, hipStream_t stream) {
    const unsigned columns = (a.n + 255) / 256;
    const size_t lds = size_t(a.slots + 1) * 4;
    if constexpr (RT <= 4)
        if (a.fused) {
            lora_fused_kernel<T, RT><<<dim3(a.block_tiles, columns), 512, lds, stream>>>(a);
            return;
        }
    const unsigned blocks = a.tile_count / a.block_tiles;
    const dim3 grid(a.block_tiles, blocks, a.splits), up_grid((a.n + a.n_len - 1) / a.n_len, a.block_tiles, blocks);
    if constexpr (RT <= 8)
        if (a.tile_rows == 32) {
            lora_down_kernel<T, RT, 2><<<grid, 256, lds, stream>>>(a);
            if (a.past_cache) lora_up_kernel<T, RT, 2, true><<<up_grid, 256, 0, stream>>>(a);
            else lora_up_kernel<T, RT, 2, false><<<up_grid, 256, 0, stream>>>(a);
            return;
        }
    lora_down_kernel<T, RT, 1><<<grid, 256, lds, stream>>>(a);
    lora_up_kernel<T, RT, 1, false><<<up_grid, 256, 0, stream>>>(a);
}

template <class T>
void launch_typed(const LoraArgs& a, hipStream_t stream) {
    if (a.rank <= 16) launch_ranks<T, 1>(a, stream);
    else if (a.rank <= 32) launch_ranks<T, 2>(a, stream);
    else if (a.rank <= 64) launch_ranks<T, 4>(a, stream);
    else if (a.rank <= 128) launch_ranks<T, 8>(a, stream);
    else launch_ranks<T, 16>(a, stream);
}

}  // namespace

void lora_plan(LoraArgs& a, int cus) {
    a.copy_bare = a.base != a.y || a.ldbase != a.ldy;
    a.past_cache = a.m * a.n * 4 > (int64_t(32) << 20);   // an output that no L2 would hold (measured at 786 MB only)
    a.part_ld = (a.rank + 15) / 16 * 16;
    const int columns = (a.n + 255) / 256;
    // tiles of a block of `rows` rows: whole ones, and one begun per slot
    const auto tiles_of = [&](int64_t rows, int tile) { return int(std::min<int64_t>(rows, rows / tile + a.slots + 1)); };
    // past one block's rows, blocks of a quarter: a tile is found sooner
    const int64_t few = a.m > kLoraBlockRows ? kLoraBlockRows / 4 : a.m;
    // One launch where a workgroup for every tile and block of columns fits a
    // CU and K takes at most four chunks, so that a second launch costs more
    // than doing A x again for each block: 16 tokens 1024 -> 1024 10.4 -> 6.4
    // us; 777 rows 1001 -> 1359 of rank 40 (438 workgroups of eight chunks)
    // 28.3 fused, 18.7 in two.
    const int rank_tiles = a.rank <= 16 ? 1 : a.rank <= 32 ? 2 : 4;
    a.fused = a.rank <= 64 && a.m <= kLoraBlockRows && int64_t(tiles_of(few, 16)) * columns <= cus && a.k <= 2048 / rank_tiles;
    a.tile_rows = !a.fused && a.rank <= 128 && a.m >= 16 * cus ? 32 : 16;
    a.block_rows = int(few);
    a.block_tiles = tiles_of(few, a.tile_rows);
    a.tile_count = int((a.m + a.block_rows - 1) / a.block_rows) * a.block_tiles;
    // about two workgroups per CU from splits of at least 256 values of K (and
    // three from blocks of columns below: not swept)
    const int64_t full = (a.m + a.tile_rows - 1) / a.tile_rows;
    a.splits = int(std::max<int64_t>(1, std::min<int64_t>((2 * cus + full - 1) / full, (a.k + 255) / 256)));
    a.k_len = ((a.k + a.splits - 1) / a.splits + 127) / 128 * 128;
    a.splits = (a.k + a.k_len - 1) / a.k_len;
    const int column_splits = int(std::min<int64_t>(columns, (3 * cus + full - 1) / full));
    a.n_len = (columns + column_splits - 1) / column_splits * 256;
}

static size_t part_bytes(const LoraArgs& a) { return size_t(a.splits) * a.m * a.part_ld * 4; }

size_t lora_scratch_bytes(const LoraArgs& a) {
    return a.fused ? 0 : part_bytes(a) + size_t(a.tile_count) * (a.tile_rows + 1) * 4;
}

void launch_lora(LoraArgs a, int type, void* scratch, hipStream_t stream) {
    a.part = static_cast<float*>(scratch);
    a.tiles = a.fused ? nullptr : reinterpret_cast<int*>(static_cast<char*>(scratch) + part_bytes(a));
    if (type == T_F16) launch_typed<_Float16>(a, stream);
    else launch_typed<float>(a, stream);
}

}  // namespace samhip
