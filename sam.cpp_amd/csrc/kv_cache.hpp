// The operators on caches of keys and values in Q8_0 or Q4_0 pages
// (kv_cache.hip, cache_attn.hip): what their kernels take, and how a request's
// positions lie in its pages.
#pragma once

#include "internal.hpp"

namespace samhip {

// n / d for 0 <= n < 2^31 by a product: with 2^(s-1) < d <= 2^s and
// m = ceil(2^(31+s) / d) <= 2^32 - 1, n m exceeds n 2^(31+s) / d by less than
// n d / d <= 2^31, which is below the 2^(31+s) / d that would carry the
// quotient past the next whole number.
struct Divisor {
    uint32_t d = 1, m = 0x80000000u, shift = 31;
    __host__ static Divisor of(uint32_t d) {
        Divisor v;
        uint32_t s = 0;
        while ((uint64_t(1) << s) < d) ++s;
        v.d = d;
        v.shift = 31 + s;
        v.m = uint32_t(((uint64_t(1) << v.shift) + d - 1) / d);
        return v;
    }
    __host__ __device__ uint32_t quotient(uint32_t n) const { return uint32_t(uint64_t(n) * m >> shift); }
};

struct KvCacheArgs {
    uint8_t *k, *v;
    int64_t ldk, ldv;                      // bytes from row to row
    const int32_t *pages, *row_start, *len;
    int kv_heads, head_dim, requests, max_pages;
    Divisor page;                          // page_rows
    uint32_t page_count;                   // whole pages in the cache
    int capacity;                          // max_pages * page_rows
};

// The rotation of up to 128 pairs of a head: the frequency (scale *
// theta^-power, the angle a position) and the axis of each.
constexpr int kRopeMaxPairs = 128;
struct RopeArgs {
    const int32_t* positions;
    int axes, pairs;                       // pairs 0: no rotation
    bool halves;
    double frequency[kRopeMaxPairs];
    uint8_t axis[kRopeMaxPairs];
};

#if defined(__HIPCC__)
// Query or cache rows [from, from + n) of request r, cut to the `rows` that exist.
__device__ __forceinline__ int request_rows(const KvCacheArgs& c, int rows, int r, int& from) {
    from = min(max(c.row_start[r], 0), rows);
    return min(max(c.row_start[r + 1], 0), rows) - from;
}

// What a request has in the cache, as said: more than there are positions, too,
// for its rows stand before the end.
__device__ __forceinline__ int request_len(const KvCacheArgs& c, int r) { return max(c.len[r], 0); }

// The cache row of a position below the request's length and the capacity, or -1.
__device__ __forceinline__ int cache_row(const KvCacheArgs& c, int r, int position) {
    const uint32_t p = c.page.quotient(uint32_t(position));
    const uint32_t page = uint32_t(c.pages[int64_t(r) * c.max_pages + p]);
    return page < c.page_count ? int(page * c.page.d + (uint32_t(position) - p * c.page.d)) : -1;
}

// The first of `count` ascending ends that is above `value`, count where none is:
// 64 probes at a time, for a wave that asks for one value.
__device__ __forceinline__ int first_above(const int32_t* ends, int count, int value) {
    const int lane = threadIdx.x & 63;
    int lo = 0, hi = count;
    while (lo < hi) {
        const int stride = (hi - lo + 63) >> 6, at = int(min(int64_t(lo) + int64_t(stride) * (lane + 1) - 1, int64_t(hi) - 1));
        const uint64_t hit = __ballot(ends[at] > value);
        if (!hit) {
            lo = hi;
        } else {
            const int f = __builtin_ctzll(hit);
            hi = __builtin_amdgcn_readlane(at, f);
            lo += stride * f;
        }
    }
    return lo;
}

// The cache row where row `row` of `rows` in the call stands, -1 where it has
// no place, -2 where no request has it; its request is `lo` or, where rows of
// others lie between, not far behind.
__device__ __forceinline__ int place_of_row(const KvCacheArgs& c, int rows, int row, int lo) {
    int hi = lo;
    for (uint32_t step = 1; hi < c.requests && c.row_start[hi + 1] <= row; step *= 2) {
        lo = hi + 1;
        hi = int(min(int64_t(hi) + step, int64_t(c.requests)));
    }
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (c.row_start[mid + 1] <= row) lo = mid + 1;
        else hi = mid;
    }
    if (lo >= c.requests) return -2;
    int from;
    const int n = request_rows(c, rows, lo, from), i = row - from;
    if (i < 0 || i >= n) return -2;
    const int len = request_len(c, lo), position = len - n + i;
    return position >= 0 && position < c.capacity ? cache_row(c, lo, position) : -1;
}
#endif

// Rows of heads * head_dim values; strides in elements, types T_F32 or T_F16.
struct RopeRows {
    const void* x;
    void* y;
    int64_t ldx, ldy;
    int rows, heads, head_dim;
};
void launch_rope(const RopeRows& r, int x_type, int y_type, const RopeArgs& rope, int cus, hipStream_t stream);

// k, v: F32 rows of kv_heads * head_dim values.
void launch_cache_write(const KvCacheArgs& c, int type, bool x86, const RopeArgs& rope, const float* k, int64_t ldk,
                        const float* v, int64_t ldv, int rows, int cus, hipStream_t stream);
void launch_cache_read(const KvCacheArgs& c, int type, void* k, int64_t ldk, void* v, int64_t ldv, int out_type, int rows,
                       int cus, hipStream_t stream);

// cache_attn_plan sets the fields behind `causal` but the scratch pointers, which
// launch_cache_attn sets.
struct CacheAttnArgs {
    KvCacheArgs cache;
    const float* q;
    float* out;
    int64_t ldq, ldo;
    int rows, heads, group;
    int max_len;                           // at most the capacity; 0 where the cache has no page
    float scale;
    bool causal;
    bool short_rows;                       // the bytes of 32 rows fit 31 bits
    bool narrow;                           // 512 / head_dim places to a workgroup; else 128
    int wave_heads;                        // kv heads of a workgroup, each some of its waves': 1, 2 or 4
    Divisor by_group, by_head_sets, by_places, by_step;   // by_places, by_step: a workgroup's places of a head, and its keys at a time
    int tiles;                             // of all requests, at most
    int slots, least_steps;                // parts of keys of a kv head in all, and the steps of the smallest; 0 slots: one part each
    __host__ __device__ int row_of_place(int place) const { return int(by_group.quotient(place)); }   // of a request's
    float *part_o, *part_ml;
    int32_t *ends, *kept;                  // null: at most 64 requests; else items to a request's end, and kept ones before it
    float* of_part;                        // 1 / steps of a part
};
void cache_attn_plan(CacheAttnArgs& a, int cus);
size_t cache_attn_scratch_bytes(const CacheAttnArgs& a);
void launch_cache_attn(CacheAttnArgs a, int type, void* scratch, hipStream_t stream);

}  // namespace samhip
