// Attention of a batch of requests over keys and values held in Q8_0 or Q4_0
// pages:
//   out = softmax(scale * q K^T) V
// Grouped heads: the queries that share a kv head are neighbouring places of a
// tile (place = query row * group + head in group).  A tile's keys may be split
// over workgroups; each part leaves a base b, the sum l of its weights
// 2^(score - b) (scores in units of log 2) and its weighted mean of values,
// which a second launch joins.
//
// F32-accurate on fp16 matrix instructions: a block's codes are exact in fp16
// and queries enter as hi + lo halves, scaled by a power of two per query.
// Weights are held against the largest contribution, weight times value scale,
// and not against the largest weight: of one query the products 2^(score - b) *
// scale stay below 2^15, the largest of a tile that moved b at 2^13, so that
// as hi + lo they keep 22 bits down to 2^-16 of the largest contribution so
// far, wherever its weight or its scale comes from.  A scale of zero counts as
// 2^-80 in this, for its weight has its place in the sum.
// F32 scores of 2^23 and more (FAR) are whole numbers, from which neither a
// scale's log nor 13 can be taken: such a query's base is its largest score, as
// rounded, and so are the others that it is taken from, so that weights are 1 at
// most and products below 2^16.  (With the product and the difference rounded at
// once, a score of 2^30 is 2^5 off its own base.)
//
// Few places: a wave takes 32 keys at a time, their codes through LDS that no
// other wave touches, read transposed for values.  An operand's 16 columns are
// places times blocks: column (place, block) has the query's part of that block
// and zeros for the others, so that the products of all blocks run on into one
// accumulator and a lane scales them by its own block's key scale, and weights
// take one block's value scale in each lane instead of all blocks' in every
// one.  (With hi and lo as columns, and a lane's scores and weights block by
// block, 64 queries of 16 heads of 128 on up to 8192 keys took 84 us.)
// That call now: 72.8 us from HBM (3.1 TB/s), 57.8 from the MALL, of it 5.0 the
// join.  At head_dim 128 twelve waves a CU have 4.6 KB each under way, and the
// vector instructions take 30 us of a SIMD, the matrix instructions 10; the rest
// is parts that end early and HBM's lines one by one.
// Many places: 128 to a workgroup, 64 keys (32 of head_dim 128) at a time as fp16
// codes in LDS for its four waves, the next ones written beside them.  Key scales multiply a block's
// products, value scales the weights.  8 prompts of 201 queries of 8 heads of 32
// on up to 5217 Q8_0 keys: 44.6 us, of it 5.2 the join; vector instructions (about
// 160 for 32 keys and 32 places, 16 of them exponentials at a quarter rate, 16 for
// each key's own value scale; with one scale for a tile, which is wrong where they
// lie far apart, 43.6 us) fill 24 us of a SIMD, matrix instructions 6.
#include <algorithm>

#include "attn_tiles.hpp"
#include "kv_cache.hpp"

#pragma clang fp contract(off)

namespace samhip {

namespace {

constexpr int WAVES = 4;
constexpr int MOST_PARTS = 32;             // of a tile's keys where waves have heads of their own
constexpr float NO_BASE = -0x1.fffffep127f;   // below every score, and finite
constexpr float FAR = 0x1p23f;            // of scores; a base from half of it on is looked at with every tile
constexpr float ROOM = 15.f;              // log 2 of the largest product before the base moves
constexpr int ZERO_SCALE = -80;           // log 2 of what a zero scale counts as: 2^30 weights of 2^(15 + 80) still have an F32 sum
constexpr int DPP_HALF_MIRROR = 0x141;    // lane 7 - i of its eight

typedef uint32_t u32x2_at __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t u32x4_at __attribute__((ext_vector_type(4), aligned(2)));
typedef int int2_t __attribute__((ext_vector_type(2)));

__device__ __forceinline__ bool finite_half(uint32_t bits) { return (bits & 0x7c00u) != 0x7c00u; }

__device__ __forceinline__ float max_xor16(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float max_xor32(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_xor16(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

__device__ __forceinline__ half8 joined(uint32_t a, uint32_t b, uint32_t c, uint32_t d) { return __builtin_bit_cast(half8, u32x4{a, b, c, d}); }

// Bytes 0, 2, 1, 3 of two dwords as fp16 operands: Q8_0 codes, or the low or
// the high halves of Q4_0 bytes less 8.  1024 + u is an fp16 number whose low
// bits are u (with the sign of a Q8_0 code turned, u = code + 128; of a high
// half, 16 code); the rest is taken off again, exactly.  The constants stay in
// registers, for v_and_or_b32 and v_pk_add_f16.
struct Unpack {
    uint32_t bytes = 0x00ff00ffu, low = 0x000f000fu, high = 0x00f000f0u, magic = 0x64006400u;
    half2_t bias8{(_Float16)-1152.f, (_Float16)-1152.f}, bias4{(_Float16)-1032.f, (_Float16)-1032.f};
    half2_t sixteenth{(_Float16)0.0625f, (_Float16)0.0625f}, bias16{(_Float16)-72.f, (_Float16)-72.f};
    __device__ __forceinline__ Unpack() {
#if defined(__HIP_DEVICE_COMPILE__)
        asm("" : "+s"(bytes), "+s"(low), "+s"(high), "+v"(magic));
        asm("" : "+s"(bias8), "+s"(bias4), "+s"(sixteenth), "+v"(bias16));
#endif
    }
    static __device__ __forceinline__ uint32_t bits(half2_t v) { return __builtin_bit_cast(uint32_t, v); }
    __device__ __forceinline__ half2_t number(uint32_t w, uint32_t mask) const { return __builtin_bit_cast(half2_t, (w & mask) | magic); }
    __device__ __forceinline__ uint32_t q8_two(uint32_t w) const { return bits(number(w, bytes) + bias8); }
    __device__ __forceinline__ uint32_t low_two(uint32_t w) const { return bits(number(w, low) + bias4); }
    __device__ __forceinline__ uint32_t high_two(uint32_t w) const { return bits(__builtin_elementwise_fma(number(w, high), sixteenth, bias16)); }
    __device__ __forceinline__ half8 q8(uint32_t w0, uint32_t w1) const {
        w0 ^= 0x80808080u;
        w1 ^= 0x80808080u;
        return joined(q8_two(w0), q8_two(w0 >> 8), q8_two(w1), q8_two(w1 >> 8));
    }
    __device__ __forceinline__ half8 q4_low(uint32_t w0, uint32_t w1) const { return joined(low_two(w0), low_two(w0 >> 8), low_two(w1), low_two(w1 >> 8)); }
    __device__ __forceinline__ half8 q4_high(uint32_t w0, uint32_t w1) const { return joined(high_two(w0), high_two(w0 >> 8), high_two(w1), high_two(w1 >> 8)); }
    __device__ __forceinline__ half8 q4_keys(uint32_t w) const { return joined(low_two(w), low_two(w >> 8), high_two(w), high_two(w >> 8)); }
};
constexpr int ORDER[8] = {0, 2, 1, 3, 4, 6, 5, 7};   // the bytes of an operand's elements

// Sum over the lanes up to and with this one (row shifts, then the last lanes of
// rows 0 and 2, and of row 1, to what lies behind them).
__device__ __forceinline__ int running_sum(int v) {
#if defined(__HIP_DEVICE_COMPILE__)
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
#endif
    return v;
}

// A request's share of the grid: tiles of its places, and parts of its keys.
// Parts are even in work over the whole call: with W the tiles' steps of keys
// of all requests, a part has about W / slots steps, so that a long request has
// more of them and no workgroup much more to do than another (64 requests of
// 4096 to 8192 keys in three parts each: 72 us; so: 68).  The parts of requests
// that have several number at most 2 * slots.
struct Share {
    int request, q0, n, len, tiles, parts;
    int before, kept;   // items (tile, part) of the requests before, and those of them that are kept for the join
};

// Rows, length, tiles and steps of request r.
struct Request {
    int from = 0, n = 0, len = 0, tiles = 0, steps = 0;
    __device__ __forceinline__ Request(const CacheAttnArgs& a, int r) {
        if (r < a.cache.requests) {
            n = max(request_rows(a.cache, a.rows, r, from), 0);
            len = request_len(a.cache, r);
        }
        tiles = int(a.by_places.quotient(n * a.group + a.by_places.d - 1));
        steps = int(a.by_step.quotient(min(len, a.max_len) + a.by_step.d - 1));
    }
    __device__ __forceinline__ int parts(float of_part) const { return max(1, int(__builtin_ceilf(float(steps) * of_part))); }
};

// 1 / steps of a part, from the sums over the requests.
__device__ __forceinline__ float part_of(const CacheAttnArgs& a, float work, float tiles) {
    // every tile's last part is a half too much, on average; a thousandth more, for the sums' roundings
    const float slots = fmaxf(float(a.slots) - 0.5f * tiles, 0.5f * float(a.slots));
    return 1.f / fmaxf(float(a.least_steps), fminf(__builtin_ceilf(work * 1.001f / slots), 1e9f));
}

// The request of an item, or of a row: up to 64 are read at once, a lane to each;
// of more, a launch before has left the sums to be searched (1024 requests of one
// query of 16 heads of 128 on up to 512 keys: every workgroup summing up for itself
// 188 us, so 100).
__device__ __forceinline__ bool find_request(const CacheAttnArgs& a, bool of_row, int value, Share& s) {
    if (a.ends) {
        s.request = first_above(of_row ? a.cache.row_start + 1 : a.ends, a.cache.requests, value);
        if (s.request >= a.cache.requests) return false;
        const Request r(a, s.request);
        s.q0 = r.from;
        s.n = r.n;
        s.len = r.len;
        s.tiles = r.tiles;
        s.parts = r.parts(*a.of_part);
        s.before = a.ends[s.request] - s.tiles * s.parts;
        s.kept = a.kept[s.request];
    } else {
        const Request r(a, threadIdx.x & 63);
        const float of_part = a.slots ? part_of(a, wave_sum(float(r.tiles) * float(r.steps)), wave_sum(float(r.tiles))) : 0.f;
        const int parts = r.parts(of_part), items = r.tiles * parts, to_keep = parts > 1 ? items : 0;
        const int sum = running_sum(items), kept = running_sum(to_keep);
        const uint64_t hit = __ballot((of_row ? r.from + r.n : sum) > value);
        if (!hit) return false;
        const int at = __builtin_ctzll(hit);
        s.request = at;
        s.q0 = __builtin_amdgcn_readlane(r.from, at);
        s.n = __builtin_amdgcn_readlane(r.n, at);
        s.len = __builtin_amdgcn_readlane(r.len, at);
        s.tiles = __builtin_amdgcn_readlane(r.tiles, at);
        s.parts = __builtin_amdgcn_readlane(parts, at);
        s.before = __builtin_amdgcn_readlane(sum - items, at);
        s.kept = __builtin_amdgcn_readlane(kept - to_keep, at);
    }
    // (tables that are not in order have none of these)
    const int first = of_row ? s.q0 : s.before, count = of_row ? s.n : s.tiles * s.parts;
    return value >= first && value - first < count && (s.parts == 1 || (s.kept >= 0 && s.kept + s.tiles * s.parts <= 2 * a.slots));
}

// The sums over more than 64 requests, by one workgroup.
constexpr int SUMS_THREADS = 1024;
__global__ __launch_bounds__(SUMS_THREADS) void cache_attn_sums_kernel(CacheAttnArgs a) {
    __shared__ float works[SUMS_THREADS / 64], counts[SUMS_THREADS / 64];
    __shared__ int items_of[SUMS_THREADS / 64], kept_of[SUMS_THREADS / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    float of_part = 0.f;
    if (a.slots) {
        float work = 0.f, tiles = 0.f;
        for (int r0 = 0; r0 < a.cache.requests; r0 += SUMS_THREADS) {
            const Request r(a, r0 + tid);
            work += float(r.tiles) * float(r.steps);
            tiles += float(r.tiles);
        }
        works[wave] = wave_sum(work);
        counts[wave] = wave_sum(tiles);
        __syncthreads();
        const int w = lane % (SUMS_THREADS / 64);
        of_part = part_of(a, wave_sum(lane == w ? works[w] : 0.f), wave_sum(lane == w ? counts[w] : 0.f));
    }
    int before = 0, kept_before = 0;
    for (int r0 = 0; r0 < a.cache.requests; r0 += SUMS_THREADS) {
        const Request r(a, r0 + tid);
        const int parts = r.parts(of_part), items = r.tiles * parts, to_keep = parts > 1 ? items : 0;
        int sum = running_sum(items), kept = running_sum(to_keep);
        if (lane == 63) items_of[wave] = sum, kept_of[wave] = kept;
        __syncthreads();
        int all = 0, all_kept = 0;
        for (int w = 0; w < SUMS_THREADS / 64; ++w) {
            if (w == wave) sum += before + all, kept += kept_before + all_kept;
            all += items_of[w];
            all_kept += kept_of[w];
        }
        before += all;
        kept_before += all_kept;
        if (r0 + tid < a.cache.requests) {
            a.ends[r0 + tid] = sum;
            a.kept[r0 + tid] = kept - to_keep;
        }
        __syncthreads();
    }
    if (tid == 0) *a.of_part = of_part;
}

// What a workgroup has: places [first, ..) of a request whose n query rows begin
// at q0, and its positions [k0, k1).
struct Span {
    int request, q0, n, first, kvh;
    int k0, k1;
    int end, limit0;      // a query row i sees positions below min(end, limit0 + i)
    int kept;             // the place of its results among those to be joined, -1: the output itself
    __device__ __forceinline__ int limit(bool causal, int i) const { return causal ? min(end, limit0 + i) : end; }
};

// Workgroups are dispatched round-robin over the 8 XCDs: the kv heads of the
// same keys, whose blocks share cache lines, follow each other on one of them.
__device__ __forceinline__ bool find_span(const CacheAttnArgs& a, Span& s) {
    const int order = blockIdx.x >> 3, sets = int(a.by_head_sets.quotient(order)), item = (blockIdx.x & 7) + 8 * sets;
    s.kvh = (order - sets * int(a.by_head_sets.d)) * a.wave_heads;
    Share share;
    if (!find_request(a, false, item, share)) return false;
    const int local = item - share.before, part = local / share.tiles, places = int(a.by_places.d), step = int(a.by_step.d);
    s.request = share.request;
    s.q0 = share.q0;
    s.n = share.n;
    s.first = (local - part * share.tiles) * places;
    s.kept = share.parts > 1 ? share.kept + local : -1;
    s.end = min(share.len, a.max_len);
    s.limit0 = share.len - s.n + 1;
    const int tile_end = max(s.limit(a.causal, min(s.n - 1, a.row_of_place(s.first + places - 1))), 0);
    const int chunk = (int(a.by_step.quotient(tile_end + step - 1)) + share.parts - 1) / share.parts * step;
    s.k0 = min(part * chunk, tile_end);
    s.k1 = min(s.k0 + chunk, tile_end);
    return true;
}

// What shares a SIMD is served oldest first, so that the last workgroup would run
// alone in the end, and slowly; with this, who is behind goes first (8 prompts of
// 201 queries of 8 heads of 32: 48.0 us without, 42.6 with it; 64 queries of 16
// heads of 128 on up to 8192 keys: 66.5, 64.5 then).
struct Progress {
    int k0, quarter;
    __device__ __forceinline__ explicit Progress(const Span& s) : k0(s.k0), quarter((s.k1 - s.k0) / 4) { __builtin_amdgcn_s_setprio(3); }
    __device__ __forceinline__ void at(int k) const {
        const int done = k - k0;
        if (done >= 3 * quarter) __builtin_amdgcn_s_setprio(0);
        else if (done >= 2 * quarter) __builtin_amdgcn_s_setprio(1);
        else if (done >= quarter) __builtin_amdgcn_s_setprio(2);
    }
};

// Where the results of a tile's p-th place go.
__device__ __forceinline__ int64_t kept_place(const CacheAttnArgs& a, int kvh, int kept, int p) {
    return (int64_t(kvh) * 2 * a.slots + kept) * a.by_places.d + p;
}
__device__ __forceinline__ float* result_of(const CacheAttnArgs& a, const Span& s, int kvh, int p, int row, int head, int hd) {
    return s.kept < 0 ? a.out + row * a.ldo + head * hd : a.part_o + kept_place(a, kvh, s.kept, p) * hd;
}
__device__ __forceinline__ void leave_sum(const CacheAttnArgs& a, const Span& s, int kvh, int p, float base, float sum) {
    if (s.kept < 0) return;
    float* ml = a.part_ml + kept_place(a, kvh, s.kept, p) * 2;
    ml[0] = base;
    ml[1] = sum;
}

// --- few places -------------------------------------------------------------

template <int TYPE, int HD>
struct KeyTile {
    static constexpr int KEYS = 32, BB = block_bytes(TYPE), BLOCKS = HD / 32, HALVES = TYPE == T_Q8_0 ? 2 : 1;
    static constexpr int CHUNKS = BLOCKS * HALVES;      // 16 bytes of codes of each key
    // A chunk's 32 keys follow each other, so that reads of 16 keys fill the
    // banks; the padding spreads the blocks that a row's lanes write.
    static constexpr int STRIDE = KEYS * 16 + (TYPE == T_Q8_0 ? 32 : 64);
    static constexpr int VALUES = CHUNKS * STRIDE, SCALES = 2 * VALUES, LOGS = SCALES + 2 * BLOCKS * KEYS * 2, BYTES = LOGS + KEYS * 4;
    static constexpr int PIECES = HD / 32;              // blocks of a lane
};

template <int TYPE>
struct Block {
    uint32_t d;
    u32x4 w[TYPE == T_Q8_0 ? 2 : 1];
    __device__ __forceinline__ void load(const uint8_t* p) {
        d = *reinterpret_cast<const uint16_t*>(p);
        w[0] = *reinterpret_cast<const u32x4_at*>(p + 2);
        if constexpr (TYPE == T_Q8_0) w[1] = *reinterpret_cast<const u32x4_at*>(p + 18);
    }
};

template <int TYPE, int HD>
struct NarrowShared {
    static constexpr int PLACES = 512 / HD;   // an operand's
    static constexpr int TILES = WAVES * KeyTile<TYPE, HD>::BYTES, SUMS = WAVES * PLACES * (HD + 4) * 4;
    uint8_t __attribute__((aligned(16))) lds[TILES > SUMS ? TILES : SUMS];
    float b[WAVES][PLACES], l[WAVES][PLACES];
};

template <int TYPE, int HD>
__global__ __launch_bounds__(64 * WAVES, 3) void cache_attn_narrow_kernel(CacheAttnArgs a) {
    typedef KeyTile<TYPE, HD> T;
    typedef NarrowShared<TYPE, HD> Shared;
    __shared__ Shared sh;
    Span s;
    if (!find_span(a, s)) return;
    const KvCacheArgs& c = a.cache;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 15, quarter = lane >> 4;
    const int wave_head = wave & (a.wave_heads - 1), kvh = s.kvh + wave_head;
    const int g = col / T::BLOCKS, my_blk = col % T::BLOCKS;   // this lane's column
    // row 4 quarter + i of the products with values: its place, and whether it is of block `blk`
    const auto place_of = [&](int i) { return (4 * quarter + i) / T::BLOCKS; };
    const auto is_of = [](int i, int blk) { return i % T::BLOCKS == blk; };
    int limit;
    floatx8 x;   // this column's and quarter's part of the queries
    const auto load_queries = [&] {
        const int place = s.first + g, i = a.row_of_place(place), head = kvh * a.group + place - i * a.group;
        const bool mine = i < s.n;
        limit = mine ? s.limit(a.causal, i) : 0;
        // Q8_0: 8 neighbours; Q4_0: 4 and the 4 that stand 16 behind them
        const float* from = a.q + (s.q0 + (mine ? i : 0)) * a.ldq + head * HD + 32 * my_blk + (TYPE == T_Q8_0 ? 8 : 4) * quarter;
        const float4_at u = *reinterpret_cast<const float4_at*>(from), v = *reinterpret_cast<const float4_at*>(from + (TYPE == T_Q8_0 ? 4 : 16));
        x = floatx8{u[0], u[1], u[2], u[3], v[0], v[1], v[2], v[3]};
    };
    const Unpack unpack;
    half8 q_hi[T::BLOCKS], q_lo[T::BLOCKS];
    float cq;
    const auto split_queries = [&] {
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) m = umax(m, __float_as_uint(x[j]) & 0x7fffffffu);
        if (T::BLOCKS >= 2) m = umax_dpp<DPP_XOR1>(m);
        if (T::BLOCKS == 4) m = umax_dpp<DPP_XOR2>(m);
        const int e = exponent_of(umax_xor32(umax_xor16(m)));
        const float f = a.scale < 0.f ? -down(e) : down(e);
        cq = fmaxf(fabsf(a.scale) * (LOG2E * up(e)), 0x1p-120f);   // a masked score times it is -inf
        half8 hi, lo;
#pragma unroll
        for (int j = 0; j < 8; j += 2) split_pair(float2_t{x[ORDER[j]] * f, x[ORDER[j + 1]] * f}, hi, lo, j);
#pragma unroll
        for (int blk = 0; blk < T::BLOCKS; ++blk) {
            q_hi[blk] = my_blk == blk ? hi : half8{};
            q_lo[blk] = my_blk == blk ? lo : half8{};
        }
    };
    uint8_t* tile = sh.lds + wave * T::BYTES;
    _Float16* scales = reinterpret_cast<_Float16*>(tile + T::SCALES);   // [keys, values][block][key]
    float* logs = reinterpret_cast<float*>(tile + T::LOGS);
    floatx4 o[2 * T::BLOCKS];
    float base = NO_BASE, l = 0.f, room = ROOM;
#pragma unroll
    for (int d = 0; d < 2 * T::BLOCKS; ++d) o[d] = floatx4{0.f, 0.f, 0.f, 0.f};

    float zero = 0.f;   // kept from the compiler, which would make a product with a conversion of the mixed fma
#if defined(__HIP_DEVICE_COMPILE__)
    asm("" : "+s"(zero));
#endif
    const int step = int(a.by_step.d), kw = s.k0 + T::KEYS * (wave >> __builtin_ctz(a.wave_heads));
    // block f = lane + 64 i of a tile: keys' first, a key's blocks side by side
    const auto key_of = [&](int i) { return (lane + 64 * i) % HD / T::BLOCKS; };
    const auto of_values = [&](int i) { return lane + 64 * i >= HD; };
    const int blk_of = lane % T::BLOCKS;
    const uint8_t* k_at = c.k + (kvh * T::BLOCKS + blk_of) * T::BB;
    const uint8_t* v_at = c.v + (kvh * T::BLOCKS + blk_of) * T::BB;
    Block<TYPE> raw[T::PIECES];   // the next tile
    // the cache row of position k + lane (lanes 0 to 31), -1: none
    const auto row_of = [&](int k) { return lane < T::KEYS && k + lane < s.k1 ? cache_row(c, s.request, k + lane) : -1; };
    // 32 rows on end, as pages of many rows have them, are a scalar base and
    // offsets that never change.
    const uint32_t k_off = uint32_t(lane / T::BLOCKS) * uint32_t(c.ldk) + blk_of * T::BB, v_off = uint32_t(lane / T::BLOCKS) * uint32_t(c.ldv) + blk_of * T::BB;
    uint32_t there = 0;           // its keys that have a row
    const auto load = [&](int row) {
        const int first = __builtin_amdgcn_readfirstlane(row);
        there = uint32_t(__ballot(row >= 0));
        if (HD > 32 && a.short_rows && there == 0xffffffffu && __all(lane >= T::KEYS || row == first + lane)) {
            const uint8_t *kb = c.k + int64_t(first) * c.ldk + kvh * (T::BLOCKS * T::BB), *vb = c.v + int64_t(first) * c.ldv + kvh * (T::BLOCKS * T::BB);
#pragma unroll
            for (int i = 0; i < T::PIECES; ++i) {
                constexpr int ROWS = 64 / T::BLOCKS;   // of a piece
                const int before = 64 * i % HD / T::BLOCKS / ROWS * ROWS;
                if (of_values(i)) raw[i].load(vb + before * c.ldv + v_off);
                else raw[i].load(kb + before * c.ldk + k_off);
            }
        } else {
#pragma unroll
            for (int i = 0; i < T::PIECES; ++i) {
                const int64_t r = max(__shfl(row, key_of(i), 64), 0);   // where there is none, row 0's blocks with scales of zero
                raw[i].load(of_values(i) ? v_at + r * c.ldv : k_at + r * c.ldk);
            }
        }
    };
    bool odd_values = false;
    int row = row_of(kw);
    load_queries();   // behind the table's load, before what waits for it
    if (kw < s.k1) load(row);
    row = row_of(kw + step);
    split_queries();
    const Progress progress(s);
    for (int k = kw; k < s.k1; k += step) {
        progress.at(k);
        const uint32_t here = there;
        wave_lds_handoff();   // the last tile's reads came first
        bool odd = false;
#pragma unroll
        for (int i = 0; i < T::PIECES; ++i) odd = odd || !finite_half(raw[i].d);
        if (here != 0xffffffffu || __any(odd)) {
#pragma unroll
            for (int i = 0; i < T::PIECES; ++i) {
                const bool is = here >> key_of(i) & 1, v = of_values(i);
                if (!finite_half(raw[i].d)) {
                    odd_values = odd_values || (v && is);   // added behind the last tile, for those that see them
                    raw[i].d = v ? 0u : 0x7e00u;
                }
                raw[i].d = is ? raw[i].d : 0u;
            }
        }
#pragma unroll
        for (int i = 0; i < T::PIECES; ++i) {
            const int key = key_of(i);
            const bool v = of_values(i);
            uint8_t* to = tile + (v ? T::VALUES : 0) + blk_of * T::HALVES * T::STRIDE + key * 16;
            *reinterpret_cast<u32x4*>(to) = raw[i].w[0];
            if constexpr (TYPE == T_Q8_0) *reinterpret_cast<u32x4*>(to + T::STRIDE) = raw[i].w[1];
            reinterpret_cast<uint16_t*>(scales)[((v ? T::BLOCKS : 0) + blk_of) * T::KEYS + key] = uint16_t(raw[i].d);
            if (T::BLOCKS == 1 || 64 * i >= HD) {   // values: the largest scale of a key's blocks
                uint32_t most = raw[i].d & 0x7fffu;
                if (T::BLOCKS == 2) most = umax_dpp<DPP_XOR1>(most);
                if (T::BLOCKS == 4) most = umax_quad(most);
                if (v && blk_of == 0) logs[key] = fmaxf(__builtin_amdgcn_logf(half_bits_to_float(most)), float(ZERO_SCALE));
            }
        }
        wave_lds_handoff();
        if (k + step < s.k1) {
            load(row);
            row = row_of(k + 2 * step);
        }
        // scores of keys 16n + 4 quarter + i: the block's of this column, then the sum over its place's columns
        float w[8];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            floatx4 sc{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int blk = 0; blk < T::BLOCKS; ++blk) {
                half8 keys;
                if constexpr (TYPE == T_Q8_0) {
                    const u32x2 code = *reinterpret_cast<const u32x2*>(tile + (2 * blk + (quarter >> 1)) * T::STRIDE + (16 * n + col) * 16 + 8 * (quarter & 1));
                    keys = unpack.q8(code[0], code[1]);
                } else {
                    keys = unpack.q4_keys(*reinterpret_cast<const uint32_t*>(tile + blk * T::STRIDE + (16 * n + col) * 16 + 4 * quarter));
                }
                sc = __builtin_amdgcn_mfma_f32_16x16x32_f16(keys, q_hi[blk], sc, 0, 0, 0);
                sc = __builtin_amdgcn_mfma_f32_16x16x32_f16(keys, q_lo[blk], sc, 0, 0, 0);
            }
            const half4 d = *reinterpret_cast<const half4*>(scales + my_blk * T::KEYS + 16 * n + 4 * quarter);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float x = __builtin_fmaf(float(d[i]), sc[i], zero);
                if (T::BLOCKS >= 2) x += dpp<DPP_XOR1>(x);
                if (T::BLOCKS == 4) x += dpp<DPP_XOR2>(x);
                w[4 * n + i] = x;
            }
        }
        const floatx4 log_d[2] = {*reinterpret_cast<const floatx4*>(logs + 4 * quarter), *reinterpret_cast<const floatx4*>(logs + 16 + 4 * quarter)};
        if (here != 0xffffffffu || __any(k + T::KEYS > limit)) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int key = 16 * (j >> 2) + 4 * quarter + (j & 3);
                if (!(here >> key & 1) || k + key >= limit) w[j] = -__builtin_inff();
            }
        }
        float top = __builtin_fmaf(w[0], cq, log_d[0][0]);
#pragma unroll
        for (int j = 1; j < 8; ++j) top = fmaxf(top, __builtin_fmaf(w[j], cq, log_d[j >> 2][j & 3]));
        float c_now = cq;
        if (__any(top > base + room)) {
            top = max_xor32(max_xor16(top));
            const bool far = fabsf(top) >= FAR;
            float moved = top > base + ROOM ? top - 13.f : base;
            if (__any(far)) {
                float most = base;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    w[j] = far ? w[j] * cq : w[j];
                    most = fmaxf(most, w[j]);
                }
                most = max_xor32(max_xor16(most));
                moved = far ? most : moved;
                c_now = far ? 1.f : cq;
            }
            const float f = __builtin_amdgcn_exp2f(base - moved);
            base = moved;
            room = fabsf(base) >= 0.5f * FAR ? -__builtin_inff() : ROOM;
            l *= f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float f_i = __shfl(f, place_of(i) * T::BLOCKS, 64);   // of the query of row i
#pragma unroll
                for (int d = 0; d < 2 * T::BLOCKS; ++d)
                    if (is_of(i, d >> 1)) o[d][i] *= f_i;
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            w[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(w[j], c_now, -base));
            l += w[j];
        }
        // O += P V, P the weights with this column's block's scales; element j is key
        // 4 quarter + j or 16 + 4 quarter + j - 4 in either operand.  Of a block's
        // products only the rows of that block count.
        [[maybe_unused]] const uint8_t* values = tile + T::VALUES + (4 * quarter + (col >> 1 & 3) + (col >> 3) * 16) * 16 + 8 * (col & 1);
        half8 p_hi, p_lo;
        {
            const _Float16* dv = scales + (T::BLOCKS + my_blk) * T::KEYS + 4 * quarter;
            const half4 d0 = *reinterpret_cast<const half4*>(dv), d1 = *reinterpret_cast<const half4*>(dv + 16);
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                const int j0 = ORDER[j], j1 = ORDER[j + 1];
                const float x0 = __builtin_fmaf(w[j0], float(j0 < 4 ? d0[j0 & 3] : d1[j0 & 3]), zero);
                const float x1 = __builtin_fmaf(w[j1], float(j1 < 4 ? d0[j1 & 3] : d1[j1 & 3]), zero);
                split_pair(float2_t{x0, x1}, p_hi, p_lo, j);
            }
        }
#pragma unroll
        for (int blk = 0; blk < T::BLOCKS; ++blk) {
            half8 v[2];
#if defined(__HIP_DEVICE_COMPILE__)
            // lane i of 16 gets byte i of the 8 keys that the lanes address, two lanes to a key
            const auto read = [&](int chunk) {
                return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) int2_t*)(values + chunk * T::STRIDE)));
            };
            if constexpr (TYPE == T_Q8_0) {
                const u32x2 w0 = read(2 * blk), w1 = read(2 * blk + 1);
                v[0] = unpack.q8(w0[0], w0[1]);
                v[1] = unpack.q8(w1[0], w1[1]);
            } else {
                const u32x2 w0 = read(blk);
                v[0] = unpack.q4_low(w0[0], w0[1]);
                v[1] = unpack.q4_high(w0[0], w0[1]);
            }
#endif
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                o[2 * blk + h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(p_hi, v[h], o[2 * blk + h], 0, 0, 0);
                o[2 * blk + h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(p_lo, v[h], o[2 * blk + h], 0, 0, 0);
            }
        }
    }
    if (__any(odd_values)) {
        // values whose scale is no number were zeros: NaN for the queries that see them
        for (int k = kw; k < s.k1; k += step)
            for (int n = 0; n < min(T::KEYS, s.k1 - k); ++n) {
                const int r = cache_row(c, s.request, k + n);
                if (r < 0) continue;
#pragma unroll
                for (int blk = 0; blk < T::BLOCKS; ++blk) {
                    if (finite_half(*reinterpret_cast<const uint16_t*>(c.v + r * c.ldv + (kvh * T::BLOCKS + blk) * T::BB))) continue;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (k + n < __shfl(limit, place_of(i) * T::BLOCKS, 64)) o[2 * blk][i] = o[2 * blk + 1][i] = __builtin_nanf("");
                }
            }
    }
    // the sums of the waves of a head, joined through LDS
    l = pair_sum(sum_xor16(l));
    if (quarter == 0 && my_blk == 0) {
        sh.b[wave][g] = base;
        sh.l[wave][g] = l;
    }
    __syncthreads();   // also: every wave is past its tiles
    float* all = reinterpret_cast<float*>(sh.lds);
    const auto joined_sum = [&](int of_head, int p, float& most) {
        most = NO_BASE;
        float sum = 0.f;
        for (int w = of_head; w < WAVES; w += a.wave_heads) most = fmaxf(most, sh.l[w][p] != 0.f ? sh.b[w][p] : NO_BASE);
        for (int w = of_head; w < WAVES; w += a.wave_heads) sum += sh.l[w][p] != 0.f ? sh.l[w][p] * __builtin_amdgcn_exp2f(sh.b[w][p] - most) : 0.f;
        return sum;
    };
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int p = place_of(i);
        float most;
        const float sum = joined_sum(wave_head, p, most);
        const float f = sh.l[wave][p] != 0.f ? __builtin_amdgcn_exp2f(sh.b[wave][p] - most) / sum : 0.f;
#pragma unroll
        for (int d = 0; d < 2 * T::BLOCKS; ++d)
            if (is_of(i, d >> 1)) all[(wave * Shared::PLACES + p) * (HD + 4) + 16 * d + col] = o[d][i] * f;
    }
    if (tid < Shared::PLACES * a.wave_heads) {
        const int p = tid % Shared::PLACES, of_head = tid / Shared::PLACES;
        float most;
        const float sum = joined_sum(of_head, p, most);
        if (a.row_of_place(s.first + p) < s.n) leave_sum(a, s, s.kvh + of_head, p, most, sum);
    }
    __syncthreads();
    constexpr int QUADS = HD / 4;
    for (int t = tid; t < Shared::PLACES * QUADS * a.wave_heads; t += 64 * WAVES) {
        const int of_head = t / (Shared::PLACES * QUADS), p = t / QUADS % Shared::PLACES, d = 4 * (t % QUADS);
        const int place = s.first + p, i = a.row_of_place(place), out_kvh = s.kvh + of_head;
        if (i >= s.n) continue;
        floatx4 v{0.f, 0.f, 0.f, 0.f};
        for (int w = of_head; w < WAVES; w += a.wave_heads) v += *reinterpret_cast<const floatx4*>(all + (w * Shared::PLACES + p) * (HD + 4) + d);
        *reinterpret_cast<float4_at*>(result_of(a, s, out_kvh, p, s.q0 + i, out_kvh * a.group + place - i * a.group, HD) + d) = v;
    }
}

// --- many places --------------------------------------------------------------

constexpr int TILE = 32;                  // query places of a wave
constexpr int wide_keys(int head_dim) { return head_dim == 128 ? 32 : 64; }

// Eight neighbouring codes of a row, and their block's scale.
template <int TYPE>
struct Octet {
    uint32_t d, w0, w1;
    __device__ __forceinline__ void load(const uint8_t* head_row, int octet) {
        const uint8_t* block = head_row + (octet >> 2) * block_bytes(TYPE);
        d = *reinterpret_cast<const uint16_t*>(block);
        const u32x2_at w = *reinterpret_cast<const u32x2_at*>(block + 2 + 8 * (octet & (TYPE == T_Q8_0 ? 3 : 1)));
        w0 = w[0];
        w1 = w[1];
    }
    // as fp16, in order
    __device__ __forceinline__ half8 codes(const Unpack& unpack, int octet) const {
        const uint32_t c0 = TYPE == T_Q8_0 ? w0 ^ 0x80808080u : w0 >> (2 * (octet & 2)) & 0x0f0f0f0fu;
        const uint32_t c1 = TYPE == T_Q8_0 ? w1 ^ 0x80808080u : w1 >> (2 * (octet & 2)) & 0x0f0f0f0fu;
        const half2_t bias = TYPE == T_Q8_0 ? unpack.bias8 : unpack.bias4;
        // bytes 0 and 1, or 2 and 3, each below a 0x64
        const auto two = [&](uint32_t c, uint32_t select) { return Unpack::bits(__builtin_bit_cast(half2_t, __builtin_amdgcn_perm(unpack.magic, c, select)) + bias); };
        return joined(two(c0, 0x07010700u), two(c0, 0x07030702u), two(c1, 0x07010700u), two(c1, 0x07030702u));
    }
};

// At head_dim 128 the queries' low halves: with them in registers, and 64 keys in
// a tile, one wave has a SIMD (48 requests of 48 places: 170 us; so: 111).
template <int HD>
struct WideLow {};
template <>
struct WideLow<128> {
    half8 q_lo[WAVES][128 / 16][64];
};

template <int HD>
struct WideShared : WideLow<HD> {
    static constexpr int WIDE_KEYS = wide_keys(HD);
    typedef TileShape<1, HD, WIDE_KEYS, false> K;
    typedef TileShape<1, HD, WIDE_KEYS, true> V;
    struct Tile {
        uint8_t __attribute__((aligned(16))) k[K::BYTES];
        uint8_t __attribute__((aligned(16))) v[V::BYTES];
        _Float16 __attribute__((aligned(16))) scales[2][HD / 32][WIDE_KEYS];   // of keys, of values
        float __attribute__((aligned(16))) logs[WIDE_KEYS];                    // log 2 of a key's largest value scale
    } tile[2];
    int rows[4][WIDE_KEYS];
    uint64_t here[4];
};

template <int TYPE, int HD>
__global__ __launch_bounds__(64 * WAVES, 2) void cache_attn_wide_kernel(CacheAttnArgs a) {
    typedef WideShared<HD> Shared;
    constexpr int WIDE_KEYS = wide_keys(HD), PIECES = HD * WIDE_KEYS / 2048, BLOCKS = HD / 32, BB = block_bytes(TYPE);   // of 8 values, a thread's part of a tile
    __shared__ Shared sh;
    Span s;
    if (!find_span(a, s)) return;
    const int kvh = s.kvh;
    const KvCacheArgs& c = a.cache;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), li = lane & 31, hh = lane >> 5;
    const int place = s.first + TILE * wave + li, i_row = a.row_of_place(place), head = kvh * a.group + place - i_row * a.group;
    const bool mine = i_row < s.n;
    const int row = s.q0 + (mine ? i_row : 0), limit = mine ? min(s.limit(a.causal, i_row), s.k1) : 0;

    // Cache rows of a tile, looked up by the first wave three tiles ahead.
    const auto row_at = [&](int k) { return lane < WIDE_KEYS && k + lane < s.k1 ? cache_row(c, s.request, k + lane) : -1; };
    const auto put_rows = [&](int t, int r) {
        const uint64_t here = __ballot(r >= 0);
        if (lane < WIDE_KEYS) sh.rows[t & 3][lane] = r;
        if (lane == 0) sh.here[t & 3] = here;
    };
    int ahead = -1;
    if (wave == 0) {
        const int r0 = row_at(s.k0), r1 = row_at(s.k0 + WIDE_KEYS), r2 = row_at(s.k0 + 2 * WIDE_KEYS);
        put_rows(0, r0);
        put_rows(1, r1);
        put_rows(2, r2);
        ahead = row_at(s.k0 + 3 * WIDE_KEYS);
    }

    // queries: lane (li, hh) has place li's values 16t + 8hh .. + 7
    half8 q_hi[HD / 16], q_lo[HD / 16];
    float cq;
    {
        floatx8 x[HD / 16];
        uint32_t m = 0;
#pragma unroll
        for (int t = 0; t < HD / 16; ++t) {
            const float* from = a.q + row * a.ldq + head * HD + 16 * t + 8 * hh;
            const float4_at u = *reinterpret_cast<const float4_at*>(from), v = *reinterpret_cast<const float4_at*>(from + 4);
            x[t] = floatx8{u[0], u[1], u[2], u[3], v[0], v[1], v[2], v[3]};
#pragma unroll
            for (int j = 0; j < 8; ++j) m = umax(m, __float_as_uint(x[t][j]) & 0x7fffffffu);
        }
        const int e = exponent_of(umax_xor32(m));
        const float f = a.scale < 0.f ? -down(e) : down(e);
        cq = fmaxf(fabsf(a.scale) * (LOG2E * up(e)), 0x1p-120f);   // a masked score times it is -inf
#pragma unroll
        for (int t = 0; t < HD / 16; ++t)
#pragma unroll
            for (int j = 0; j < 8; j += 2) split_pair(float2_t{x[t][j] * f, x[t][j + 1] * f}, q_hi[t], q_lo[t], j);
        if constexpr (HD == 128) {
#pragma unroll
            for (int t = 0; t < HD / 16; ++t) sh.q_lo[wave][t][lane] = q_lo[t];
        }
    }
    const auto low = [&](int u) {
        if constexpr (HD == 128) return sh.q_lo[wave][u][lane];
        else return q_lo[u];
    };
    // o[d] holds, transposed, dimensions 32d + 8 (r / 4) + 4hh + r % 4 of place li
    floatx16 o[BLOCKS];
    float base = NO_BASE, l = 0.f, room = ROOM, zero = 0.f;   // (zero: kept from the compiler, for the mixed fma)
#if defined(__HIP_DEVICE_COMPILE__)
    asm("" : "+s"(zero));
#endif
#pragma unroll
    for (int d = 0; d < BLOCKS; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] = 0.f;

    // this thread's piece of the first 256; the others are whole rows of keys on
    constexpr int EACH = 2048 / HD;
    const int key = tid / (HD / 8), octet = tid % (HD / 8);
    const uint8_t *k_at = c.k + kvh * BLOCKS * BB, *v_at = c.v + kvh * BLOCKS * BB;
    const Unpack unpack;
    Octet<TYPE> kr[PIECES], vr[PIECES];
    uint32_t there = 0;   // of the pieces, whether their key has a row
    const auto load = [&](const int* rows) {
        there = 0;
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const int r = rows[key + i * EACH];
            there |= uint32_t(r >= 0) << i;
            const int64_t at = max(r, 0);   // where there is none, row 0's blocks with scales of zero
            kr[i].load(k_at + at * c.ldk, octet);
            vr[i].load(v_at + at * c.ldv, octet);
        }
    };
    bool odd_values = false;
    const auto put = [&](typename Shared::Tile& tile) {
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const bool is = there >> i & 1;
            uint32_t dk = is ? kr[i].d : 0u, dv = is ? vr[i].d : 0u;
            if (!finite_half(dk)) dk = 0x7e00u;
            if (!finite_half(dv)) {
                odd_values = true;   // added behind the last tile, for those that see them
                dv = 0;
            }
            const int f = tid + 256 * i;
            *Shared::K::piece(tile.k, f) = kr[i].codes(unpack, octet);
            *Shared::V::piece(tile.v, f) = vr[i].codes(unpack, octet);
            if (octet % 4 == 0) {
                reinterpret_cast<uint16_t*>(tile.scales[0][octet / 4])[key + i * EACH] = uint16_t(dk);
                reinterpret_cast<uint16_t*>(tile.scales[1][octet / 4])[key + i * EACH] = uint16_t(dv);
            }
            uint32_t most = dv & 0x7fffu;   // of the key's blocks, a quad of lanes to each
            if (BLOCKS == 2) most = umax_dpp<DPP_HALF_MIRROR>(most);
            if (BLOCKS == 4) most = umax_row(most);
            if (octet == 0) tile.logs[key + i * EACH] = fmaxf(__builtin_amdgcn_logf(half_bits_to_float(most)), float(ZERO_SCALE));
        }
    };
    __syncthreads();
    if (s.k0 < s.k1) {
        load(sh.rows[0]);
        put(sh.tile[0]);
        if (s.k0 + WIDE_KEYS < s.k1) load(sh.rows[1]);
    }
    __syncthreads();
    const int wave_end = [&] {   // no place of this wave sees a key from it on
        int v = limit;
        for (int off = 1; off < 32; off <<= 1) v = max(v, __shfl_xor(v, off, 64));
        return __builtin_amdgcn_readfirstlane(v);
    }();
    const Progress progress(s);
    int t_now = 0;
    for (int k = s.k0; k < s.k1; k += WIDE_KEYS, ++t_now) {
        progress.at(k);
        const typename Shared::Tile& tile = sh.tile[t_now & 1];
        if (k < wave_end) {
            const uint64_t here = sh.here[t_now & 3];
#pragma unroll
            for (int n = 0; n < WIDE_KEYS / 32; ++n) {
                // scores of keys 32n + 8 (r / 4) + 4hh + r % 4, block by block
                const uint8_t* kt = tile.k + (32 * n + li) * Shared::K::STRIDE + 16 * hh;
                floatx16 sc;
#pragma unroll
                for (int blk = 0; blk < BLOCKS; ++blk) {
                    floatx16 p;
#pragma unroll
                    for (int r = 0; r < 16; ++r) p[r] = 0.f;
#pragma unroll
                    for (int u = 2 * blk; u < 2 * blk + 2; ++u) {
                        const half8 keys = *reinterpret_cast<const half8*>(kt + 32 * u);
                        p = __builtin_amdgcn_mfma_f32_32x32x16_f16(keys, q_hi[u], p, 0, 0, 0);
                        p = __builtin_amdgcn_mfma_f32_32x32x16_f16(keys, low(u), p, 0, 0, 0);
                    }
#pragma unroll
                    for (int r = 0; r < 16; r += 4) {
                        const half4 d = *reinterpret_cast<const half4*>(tile.scales[0][blk] + 32 * n + 2 * r + 4 * hh);
#pragma unroll
                        for (int j = 0; j < 4; ++j) sc[r + j] = __builtin_fmaf(float(d[j]), p[r + j], blk ? sc[r + j] : zero);
                    }
                }
                const uint32_t here_n = uint32_t(here >> (32 * n));
                if (here_n != 0xffffffffu || __any(k + 32 * n + 32 > limit)) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int at = 8 * (r >> 2) + 4 * hh + (r & 3);
                        if (!(here_n >> at & 1) || k + 32 * n + at >= limit) sc[r] = -__builtin_inff();
                    }
                }
                // the largest contribution, of each key its own score and scale: one with a
                // large scale may have no weight, or be hidden
                float top = -__builtin_inff();
#pragma unroll
                for (int r = 0; r < 16; r += 4) {
                    const floatx4 log_d = *reinterpret_cast<const floatx4*>(tile.logs + 32 * n + 2 * r + 4 * hh);
#pragma unroll
                    for (int j = 0; j < 4; ++j) top = __builtin_elementwise_maximum(top, __builtin_fmaf(sc[r + j], cq, log_d[j]));
                }
                float c_now = cq;
                if (__any(top > base + room)) {
                    top = max_xor32(top);
                    const bool far = fabsf(top) >= FAR;
                    float moved = top > base + ROOM ? top - 13.f : base;
                    if (__any(far)) {
                        float most = base;
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            sc[r] = far ? sc[r] * cq : sc[r];
                            most = fmaxf(most, sc[r]);
                        }
                        most = max_xor32(most);
                        moved = far ? most : moved;
                        c_now = far ? 1.f : cq;
                    }
                    const float by = __builtin_amdgcn_exp2f(base - moved);
                    base = moved;
                    room = fabsf(base) >= 0.5f * FAR ? -__builtin_inff() : ROOM;
                    l *= by;
#pragma unroll
                    for (int d = 0; d < BLOCKS; ++d)
#pragma unroll
                        for (int r = 0; r < 16; ++r) o[d][r] *= by;
                }
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    sc[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[r], c_now, -base));
                    l += sc[r];
                }
                // O^T += V^T P^T, P the weights with a block's scales: of 16 keys, lane
                // (li, hh) has keys 4hh .. + 3 and 8 + 4hh .. + 3 of both operands
                const uint8_t* vt = tile.v + (32 * n + 4 * hh + ((lane & 15) >> 2)) * Shared::V::STRIDE + 32 * ((lane >> 4) & 1) + 8 * (lane & 3);
#pragma unroll
                for (int d = 0; d < BLOCKS; ++d) {
                    half8 p_hi[2], p_lo[2];
#pragma unroll
                    for (int r = 0; r < 16; r += 4) {
                        const half4 dv = *reinterpret_cast<const half4*>(tile.scales[1][d] + 32 * n + 2 * r + 4 * hh);
#pragma unroll
                        for (int j = 0; j < 4; j += 2)
                            split_pair(float2_t{__builtin_fmaf(sc[r + j], float(dv[j]), zero), __builtin_fmaf(sc[r + j + 1], float(dv[j + 1]), zero)}, p_hi[r >> 3],
                                       p_lo[r >> 3], (r & 7) + j);
                    }
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const uint8_t* at = vt + 16 * u * Shared::V::STRIDE + 64 * d;
                        const half8 v = __builtin_shufflevector(ds_read_tr(at), ds_read_tr(at + 8 * Shared::V::STRIDE), 0, 1, 2, 3, 4, 5, 6, 7);
                        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, p_hi[u], o[d], 0, 0, 0);
                        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, p_lo[u], o[d], 0, 0, 0);
                    }
                }
            }
        }
        if (k + WIDE_KEYS < s.k1) put(sh.tile[(t_now + 1) & 1]);
        if (k + 2 * WIDE_KEYS < s.k1) load(sh.rows[(t_now + 2) & 3]);
        if (wave == 0) {
            put_rows(t_now + 3, ahead);
            ahead = row_at(k + 4 * WIDE_KEYS);
        }
        __syncthreads();   // the next tile is written, this one read
    }
    if (__syncthreads_or(odd_values)) {
        // values whose scale is no number were zeros: NaN for the queries that see them
        for (int k = s.k0; k < s.k1; ++k) {
            const int r = cache_row(c, s.request, k);
            if (r < 0) continue;
#pragma unroll
            for (int d = 0; d < BLOCKS; ++d)
                if (!finite_half(*reinterpret_cast<const uint16_t*>(v_at + r * c.ldv + d * BB)) && k < limit)
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[d][e] = __builtin_nanf("");
        }
    }
    l = pair_sum(l);
    if (!mine) return;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    if (hh == 0) leave_sum(a, s, kvh, TILE * wave + li, base, l);
    float* to = result_of(a, s, kvh, TILE * wave + li, row, head, HD);
#pragma unroll
    for (int d = 0; d < BLOCKS; ++d)
#pragma unroll
        for (int r = 0; r < 16; r += 4)
            *reinterpret_cast<float4_at*>(to + 32 * d + 2 * r + 4 * hh) = floatx4{o[d][r] * inv, o[d][r + 1] * inv, o[d][r + 2] * inv, o[d][r + 3] * inv};
}

// Joins the parts of a row's heads.  HD / 4 lanes have a part's mean, SLOTS such
// groups every SLOTS-th part of a head, and a wave 256 / HD / SLOTS heads of a
// row, for finding the row's request costs it more than a join of few parts
// (1608 rows of 8 heads of 32 in three parts: 4.6 us, a wave to each head 8.0).
template <int HD, int SLOTS>
__global__ __launch_bounds__(256) void cache_attn_merge_kernel(CacheAttnArgs a, Divisor by_sets) {
    constexpr int QUADS = HD / 4, HEADS = 64 / (QUADS * SLOTS), AT_ONCE = 4;
    const uint32_t unit = blockIdx.x * 4 + (threadIdx.x >> 6);
    const int row = int(by_sets.quotient(unit)), lane = threadIdx.x & 63, slot = lane / QUADS % SLOTS, d = 4 * (lane % QUADS);
    if (row >= a.rows) return;
    Share s;
    if (!find_request(a, true, row, s) || s.parts == 1) return;
    const int head = int(unit - row * by_sets.d) * HEADS + lane / (QUADS * SLOTS), h = min(head, a.heads - 1);
    const int kvh = a.row_of_place(h), place = (row - s.q0) * a.group + h - kvh * a.group;   // (heads of a kv head are a group too)
    const int tile = int(a.by_places.quotient(place)), p = place - tile * int(a.by_places.d);
    const int64_t first = kept_place(a, kvh, s.kept + tile, p), apart = int64_t(s.tiles) * a.by_places.d;
    const float *ml = a.part_ml + first * 2, *o = a.part_o + first * HD + d;
    float m = -__builtin_inff(), l = 0.f;
    floatx4 v{0.f, 0.f, 0.f, 0.f};   // a mean
    for (int part = slot; part < s.parts; part += AT_ONCE * SLOTS) {
        float m_of[AT_ONCE], l_of[AT_ONCE];
        floatx4 o_of[AT_ONCE];
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) {
            const int64_t at = min(part + u * SLOTS, s.parts - 1) * apart;
            m_of[u] = ml[2 * at];
            l_of[u] = part + u * SLOTS < s.parts ? ml[2 * at + 1] : 0.f;
            o_of[u] = *reinterpret_cast<const floatx4*>(o + at * HD);
        }
        float top = m;
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) top = fmaxf(top, l_of[u] != 0.f ? m_of[u] : -__builtin_inff());
        const float before = m == top ? l : l * __builtin_amdgcn_exp2f(m - top);
        m = top;
        l = before;
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) {
            m_of[u] = l_of[u] != 0.f ? l_of[u] * __builtin_amdgcn_exp2f(m_of[u] - top) : 0.f;
            l += m_of[u];
        }
        const float inv = l == 0.f ? 0.f : 1.f / l;
        v = v * (before * inv);
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u)
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] += l_of[u] != 0.f ? o_of[u][j] * (m_of[u] * inv) : 0.f;   // without keys its mean may never have been written
    }
    if constexpr (SLOTS > 1) {
        float top = m;
#pragma unroll
        for (int off = QUADS; off < QUADS * SLOTS; off <<= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
        float mine = m == top ? l : l * __builtin_amdgcn_exp2f(m - top), sum = mine;
#pragma unroll
        for (int off = QUADS; off < QUADS * SLOTS; off <<= 1) sum += __shfl_xor(sum, off, 64);
        mine = sum == 0.f ? 0.f : mine / sum;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[j] = v[j] * mine;
#pragma unroll
            for (int off = QUADS; off < QUADS * SLOTS; off <<= 1) v[j] += __shfl_xor(v[j], off, 64);
        }
    }
    if (head < a.heads && slot == 0) *reinterpret_cast<float4_at*>(a.out + row * a.ldo + h * HD + d) = v;
}

template <int HD, int SLOTS>
void launch_merge(const CacheAttnArgs& a, hipStream_t stream) {
    constexpr int HEADS = 256 / (HD * SLOTS);
    const int sets = (a.heads + HEADS - 1) / HEADS;
    cache_attn_merge_kernel<HD, SLOTS><<<unsigned((int64_t(a.rows) * sets + 3) / 4), 256, 0, stream>>>(a, Divisor::of(sets));
}

template <int TYPE, int HD>
void launch_typed(const CacheAttnArgs& a, hipStream_t stream) {
    if (a.ends) cache_attn_sums_kernel<<<1, SUMS_THREADS, 0, stream>>>(a);
    const unsigned groups = unsigned((a.slots + a.tiles + 7) / 8 * 8 * int(a.by_head_sets.d));
    if (a.narrow) cache_attn_narrow_kernel<TYPE, HD><<<groups, 64 * WAVES, 0, stream>>>(a);
    else cache_attn_wide_kernel<TYPE, HD><<<groups, 64 * WAVES, 0, stream>>>(a);
    // A wave to a head where rows are few, or parts many (48 places of each of 8 requests
    // of 32: 19.7 us, with one wave for a row's heads 23.6; 8 prompts of 201 queries of
    // 8 heads of 32: 47.6 and 43.5).
    if (a.slots && (a.narrow || a.slots > 8 * a.tiles)) launch_merge<HD, 256 / HD>(a, stream);
    else if (a.slots) launch_merge<HD, 1>(a, stream);
}

template <int TYPE>
void launch_of_type(const CacheAttnArgs& a, hipStream_t stream) {
    if (a.cache.head_dim == 32) launch_typed<TYPE, 32>(a, stream);
    else if (a.cache.head_dim == 64) launch_typed<TYPE, 64>(a, stream);
    else launch_typed<TYPE, 128>(a, stream);
}

}  // namespace

void cache_attn_plan(CacheAttnArgs& a, int cus) {
    const int64_t places = int64_t(a.rows) * a.group, requests = std::min(a.cache.requests, a.rows);
    const int64_t each = (places + requests - 1) / requests;   // of a request with its share of the rows
    // Where the two forms meet (us for 16, 24, 32, 48 places of each of 48 requests on up
    // to 3000 Q4_0 keys of 4 kv heads, few / many: head_dim 32 21 / 34, 25 / 35, 25 / 30,
    // 32 / 38; 64: 31 / 61, 39 / 62, 47 / 52, 67 / 66; 128: 65 / 111, 94 / 111, 123 / 91,
    // 210 / 111; of 8 on up to 5000, 24, 32 and 48 places: 32 16.4 / 17.3, 16.9 / 17.1, 20.2
    // / 19.1; 64: 23 / 23, 25 / 21, 29 / 26; 128: 37 / 39, 44 / 34, 57 / 41).  In Q8_0 the
    // form for few is slower, and they meet at fewer places than this rule has: 48 requests,
    // head_dim 64 50 / 61, 59 / 52 at 24 and 32, 128 100 / 110, 148 / 111 at 16 and 24.  Two
    // operands of places to a workgroup instead of two workgroups, Q4_0: 34, 41 and 80 at 16
    // places.
    a.narrow = each <= (a.cache.head_dim == 128 ? 24 : 32);
    const int tile = a.narrow ? 512 / a.cache.head_dim : TILE * WAVES, keys = a.narrow ? 32 * WAVES : wide_keys(a.cache.head_dim);
    a.tiles = int(places / tile + requests);
    a.short_rows = std::max(a.cache.ldk, a.cache.ldv) < (int64_t(1) << 26);
    // About as many parts as run at once, which registers decide (us for 2, 3, 4, 5,
    // 6 workgroups a CU: 64 queries on up to 8192 Q4_0 keys, 16 heads of 128 in groups
    // of 4: 69, 62, 83, 74, 71; 8 heads of 64: 99, 79, 73, 92, 87; 8 of 32: 78, 63,
    // 56, 55, 66; many places, 8 prompts of 201 queries of 8 heads of 32 on up to 5217
    // Q8_0 keys: 49, 43, 57, 50, 47; 13 requests of up to 150 queries of 12 heads of
    // 64 on up to 1300: 30, 40, 37, 43, 43).
    a.least_steps = 2;
    const int at_once = !a.narrow ? (a.cache.head_dim == 32 ? 3 : 2) : a.cache.head_dim == 128 ? 3 : 4;
    const bool split = a.max_len > a.least_steps * keys;
    const auto slots = [&](int wave_heads) { return split ? at_once * cus / (a.cache.kv_heads / wave_heads) : 0; };
    // Few places: waves of one workgroup read the kv heads of the same keys, for heads
    // share cache lines, and lines that come one by one come slowly from memory that
    // no cache holds (64 queries of 8 kv heads of 64 on up to 8192 Q4_0 keys: 110
    // us with four waves for a head, 90 with four heads); not where a tile would
    // leave more parts to the join (four queries of 4 kv heads of 128 on 30000: 31.8
    // and 45; 8 of 8 heads of 32 on up to 5217: 16.0, 14.7 with two and 15.0 with four).
    a.wave_heads = 1;
    if (split && a.narrow)
        for (int heads : {2, 4})
            if (a.cache.kv_heads % heads == 0 && slots(heads) <= MOST_PARTS * int64_t(a.tiles)) a.wave_heads = heads;
    a.slots = slots(a.wave_heads);
    if (a.slots < 2) a.slots = 0;   // as many kv heads as run at once: nothing is split
    a.by_group = Divisor::of(a.group);
    a.by_head_sets = Divisor::of(a.cache.kv_heads / a.wave_heads);
    a.by_places = Divisor::of(tile);
    a.by_step = Divisor::of(keys / a.wave_heads);
}

namespace {
size_t kept_places(const CacheAttnArgs& a) { return size_t(2) * a.slots * a.cache.kv_heads * a.by_places.d; }
}  // namespace

size_t cache_attn_scratch_bytes(const CacheAttnArgs& a) {
    return kept_places(a) * (a.cache.head_dim + 2) * 4 + (a.cache.requests > 64 ? 8 * size_t(a.cache.requests) + 4 : 0);
}

void launch_cache_attn(CacheAttnArgs a, int type, void* scratch, hipStream_t stream) {
    a.part_o = static_cast<float*>(scratch);
    a.part_ml = a.part_o + kept_places(a) * a.cache.head_dim;
    if (a.cache.requests > 64) {
        a.ends = reinterpret_cast<int32_t*>(a.part_ml + kept_places(a) * 2);
        a.kept = a.ends + a.cache.requests;
        a.of_part = reinterpret_cast<float*>(a.kept + a.cache.requests);
    }
    if (type == T_Q4_0) launch_of_type<T_Q4_0>(a, stream);
    else launch_of_type<T_Q8_0>(a, stream);
}

}  // namespace samhip
