// Attention of a batch of requests over keys and values held in Q8_0 or Q4_0
// pages:
//   out = softmax(scale * q K^T) V
// A workgroup takes a query row and head, a thread every 256th key, each with a
// running maximum, sum of weights and weighted sum of values of its own.
#include <algorithm>

#include "kv_cache.hpp"
#include "q8stage.hpp"

#pragma clang fp contract(off)

namespace samhip {

namespace {

constexpr float LOG2E = 1.44269504088896340736f;
constexpr int THREADS = 256;

template <int TYPE>
__device__ __forceinline__ float block_value(const uint8_t* block, int i) {
    float d = half_bits_to_float(*reinterpret_cast<const uint16_t*>(block));
    d = d - d == 0.f ? d : __builtin_nanf("");
    if (TYPE == T_Q8_0) return d * float(int8_t(block[2 + i]));
    const int byte = block[2 + (i & 15)];
    return d * float((i < 16 ? byte & 15 : byte >> 4) - 8);
}

template <int TYPE, int HD>
__global__ __launch_bounds__(THREADS) void cache_attn_kernel(CacheAttnArgs a) {
    __shared__ float q[HD], m_of[THREADS], part[THREADS], total;
    const int row = blockIdx.x / a.heads, head = blockIdx.x - row * a.heads, kvh = head / a.group, tid = threadIdx.x;
    const KvCacheArgs& c = a.cache;
    int lo = 0, hi = c.requests;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (c.row_start[mid + 1] <= row) lo = mid + 1;
        else hi = mid;
    }
    if (lo == c.requests) return;
    int from;
    const int n = request_rows(c, a.rows, lo, from), i = row - from;
    if (i < 0 || i >= n) return;
    const int len = request_len(c, lo);
    int end = min(len, a.max_len);
    if (a.causal) end = min(end, len - n + i + 1);
    for (int d = tid; d < HD; d += THREADS) q[d] = a.q[row * a.ldq + head * HD + d];
    __syncthreads();
    float o[HD], m = -__builtin_inff(), l = 0.f;
#pragma unroll
    for (int d = 0; d < HD; ++d) o[d] = 0.f;
    for (int p = tid; p < end; p += THREADS) {
        const int64_t at = cache_row(c, lo, p);   // times a stride: 64 bits
        if (at < 0) continue;
        const uint8_t* k = c.k + at * c.ldk + kvh * (HD / 32) * block_bytes(TYPE);
        const uint8_t* v = c.v + at * c.ldv + kvh * (HD / 32) * block_bytes(TYPE);
        float s = 0.f;
        for (int b = 0; b < HD / 32; ++b)
            for (int d = 0; d < 32; ++d) s += q[32 * b + d] * block_value<TYPE>(k + b * block_bytes(TYPE), d);
        s = s * a.scale * LOG2E;
        const float mnew = fmaxf(m, s), f = m == mnew ? 1.f : __builtin_amdgcn_exp2f(m - mnew), w = __builtin_amdgcn_exp2f(s - mnew);
        m = mnew;
        l = l * f + w;
#pragma unroll
        for (int d = 0; d < HD; ++d) o[d] = o[d] * f + w * block_value<TYPE>(v + d / 32 * block_bytes(TYPE), d & 31);
    }
    m_of[tid] = m;
    __syncthreads();
    float most = -__builtin_inff();
    for (int t = 0; t < THREADS; ++t) most = fmaxf(most, m_of[t]);
    const float f = l == 0.f ? 0.f : __builtin_amdgcn_exp2f(m - most);
    part[tid] = l * f;
    __syncthreads();
    if (tid == 0) {
        float sum = 0.f;
        for (int t = 0; t < THREADS; ++t) sum += part[t];
        total = sum;
    }
    __syncthreads();
    const float inv = total == 0.f ? 0.f : 1.f / total;
    for (int d = 0; d < HD; ++d) {
        float v = 0.f;
#pragma unroll
        for (int e = 0; e < HD; ++e) v = e == d ? o[e] : v;
        __syncthreads();
        part[tid] = l == 0.f ? 0.f : v * f;
        __syncthreads();
        for (int half = THREADS / 2; half > 0; half >>= 1) {
            if (tid < half) part[tid] += part[tid + half];
            __syncthreads();
        }
        if (tid == 0) a.out[row * a.ldo + head * HD + d] = part[0] * inv;
    }
}

template <int TYPE>
void launch_typed(const CacheAttnArgs& a, hipStream_t stream) {
    const unsigned groups = unsigned(a.rows) * a.heads;
    if (a.cache.head_dim == 32) cache_attn_kernel<TYPE, 32><<<groups, THREADS, 0, stream>>>(a);
    else if (a.cache.head_dim == 64) cache_attn_kernel<TYPE, 64><<<groups, THREADS, 0, stream>>>(a);
    else cache_attn_kernel<TYPE, 128><<<groups, THREADS, 0, stream>>>(a);
}

}  // namespace

void launch_cache_attn(const CacheAttnArgs& a, int type, void*, hipStream_t stream) {
    if (type == T_Q4_0) launch_typed<T_Q4_0>(a, stream);
    else launch_typed<T_Q8_0>(a, stream);
}

}  // namespace samhip
