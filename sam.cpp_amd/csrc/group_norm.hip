// Group norm with an activation on channels-last maps (pixel rows of C
// channels, groups of C / G neighbouring channels):
//   y = act((x - mean) / sqrt(var + eps) * w + b)
// with mean and var (biased) over a group's channels of every pixel of one
// image.  The sums of x and x^2 are held in F64, where neither a group of
// millions of values nor a mean far above the deviation costs digits, and
// the mean is subtracted as two floats (hi, then lo), so one pass over the
// data gives the statistics.
//   group_norm_block_kernel : one workgroup per (image, group) with the
//                             group's values in registers: x read once
//   group_norm_stats_kernel, _finish_kernel, _apply_kernel : larger groups
#include "internal.hpp"
#include "q8stage.hpp"

#pragma clang fp contract(off)

namespace samhip {

namespace {

template <class T, int VEC>
struct Vec {
    typedef T type __attribute__((ext_vector_type(VEC)));
};
template <class T>
struct Vec<T, 1> {
    typedef T type;
};

template <class T, int VEC>
__device__ __forceinline__ void load(const T* p, float (&v)[VEC]) {
    const auto r = *reinterpret_cast<const typename Vec<T, VEC>::type*>(p);
    if constexpr (VEC == 1) v[0] = (float)r;
    else
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = (float)r[e];
}

template <class T, int VEC>
__device__ __forceinline__ void store(T* p, const float (&v)[VEC]) {
    typename Vec<T, VEC>::type r;
    if constexpr (VEC == 1) r = (T)v[0];
    else
#pragma unroll
        for (int e = 0; e < VEC; ++e) r[e] = (T)v[e];   // F16: round to nearest even
    *reinterpret_cast<typename Vec<T, VEC>::type*>(p) = r;
}

// one row swap or rotation of a double's two halves
template <int STEP>
__device__ __forceinline__ double partner(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    uint32_t lo = uint32_t(u), hi = uint32_t(u >> 32);
    lo = uint32_t(__shfl_xor(int(lo), STEP, 64));
    hi = uint32_t(__shfl_xor(int(hi), STEP, 64));
    return __builtin_bit_cast(double, uint64_t(hi) << 32 | lo);
}
__device__ __forceinline__ double wave_sum(double v) {
    v += partner<32>(v);
    v += partner<16>(v);
    v += partner<8>(v);
    v += partner<4>(v);
    v += partner<2>(v);
    return v + partner<1>(v);
}

// A group's statistics as the apply step uses them: mean = hi + lo.
struct Moments {
    float hi, lo, rstd;
};

__device__ __forceinline__ Moments moments(double sum, double sq, double n, float eps) {
    const double mean = sum / n;
    double var = sq / n - mean * mean;   // F64: loses (mean / deviation)^2 of 2^-53
    var = var < 0.0 ? 0.0 : var;         // a NaN stays one
    Moments m;
    m.hi = (float)mean;
    m.lo = (float)(mean - (double)m.hi);
    m.rstd = (float)(1.0 / sqrt(var + (double)eps));
    return m;
}

template <int ACT>
__device__ __forceinline__ float activate(float v) {
    if (ACT == ACT_RELU) return v > 0.f || v != v ? v : 0.f;
    if (ACT == ACT_SILU) return v / (1.f + __expf(-v));
    if (ACT == ACT_GELU_ERF) return gelu_erf(v);
    return v;
}
__device__ __forceinline__ float activate(int act, float v) {
    switch (act) {   // uniform
        case ACT_RELU: return activate<ACT_RELU>(v);
        case ACT_SILU: return activate<ACT_SILU>(v);
        case ACT_GELU_ERF: return activate<ACT_GELU_ERF>(v);
        default: return v;
    }
}

__device__ __forceinline__ float normalize(float x, const Moments& m) { return ((x - m.hi) - m.lo) * m.rstd; }

template <class TI, class TO, int VEC, int NV>
__global__ __launch_bounds__(1024) void group_norm_block_kernel(const TI* x, TO* y, GroupNormShape s, const float* __restrict__ w,
                                                                const float* __restrict__ b, float eps, int act) {
    __shared__ double part[16][2];
    const int g = blockIdx.x, image = blockIdx.y, tid = threadIdx.x;
    const int size = s.channels / s.groups, cols = size / VEC, total = s.pixels * cols;
    const TI* xg = x + image * s.x_image + g * size;
    TO* yg = y + image * s.y_image + g * size;
    float v[NV][VEC];
    double sum = 0.0, sq = 0.0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int at = tid + i * 1024;
        if (at < total) {
            const int p = at / cols, c = at - p * cols;
            load<TI, VEC>(xg + p * s.x_pixel + c * VEC, v[i]);
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[i][e] = 0.f;
        }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const double d = (double)v[i][e];
            sum += d;
            sq = __builtin_fma(d, d, sq);
        }
    sum = wave_sum(sum);
    sq = wave_sum(sq);
    if ((tid & 63) == 0) {
        part[tid >> 6][0] = sum;
        part[tid >> 6][1] = sq;
    }
    __syncthreads();
    sum = sq = 0.0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        sum += part[i][0];
        sq += part[i][1];
    }
    const Moments m = moments(sum, sq, double(s.pixels) * size, eps);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int at = tid + i * 1024;
        if (at >= total) break;
        const int p = at / cols, c = at - p * cols, ch = g * size + c * VEC;
        float o[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            o[e] = normalize(v[i][e], m);
            if (w) o[e] = o[e] * w[ch + e];
            if (b) o[e] = o[e] + b[ch + e];
            o[e] = activate(act, o[e]);
        }
        store<TO, VEC>(yg + p * s.y_pixel + c * VEC, o);
    }
}

// Thread t of 256 owns the VEC channels of column t % cols (pass j: column
// t % cols + 256 j) and every rows-th pixel of the chunk.
template <class TI, int VEC>
__global__ __launch_bounds__(256) void group_norm_stats_kernel(const TI* __restrict__ x, GroupNormShape s, int chunk,
                                                               double* __restrict__ partial) {
    extern __shared__ double sums[][2];   // [rows][channels]
    const int tid = threadIdx.x, cols = s.channels / VEC;
    const int width = min(cols, 256), rows = 256 / width, col0 = tid % width, row = tid / width;
    const int p0 = blockIdx.x * chunk, p1 = min(p0 + chunk, s.pixels);
    const TI* xi = x + blockIdx.y * s.x_image;
    if (row < rows) {
        for (int col = col0; col < cols; col += width) {
            double sum[VEC], sq[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) sum[e] = sq[e] = 0.0;
            const TI* xc = xi + col * VEC;
#pragma unroll 4
            for (int p = p0 + row; p < p1; p += rows) {
                float v[VEC];
                load<TI, VEC>(xc + p * s.x_pixel, v);
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const double d = (double)v[e];
                    sum[e] += d;
                    sq[e] = __builtin_fma(d, d, sq[e]);
                }
            }
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                sums[row * s.channels + col * VEC + e][0] = sum[e];
                sums[row * s.channels + col * VEC + e][1] = sq[e];
            }
        }
    }
    __syncthreads();
    const int size = s.channels / s.groups, members = size * rows, lane = tid & 63;
    for (int g = tid >> 6; g < s.groups; g += 4) {
        double sum = 0.0, sq = 0.0;
        for (int i = lane; i < members; i += 64) {
            const int r = i / size, at = r * s.channels + g * size + (i - r * size);
            sum += sums[at][0];
            sq += sums[at][1];
        }
        sum = wave_sum(sum);
        sq = wave_sum(sq);
        if (lane == 0) {
            double* out = partial + ((int64_t(blockIdx.y) * gridDim.x + blockIdx.x) * s.groups + g) * 2;
            out[0] = sum;
            out[1] = sq;
        }
    }
}

__global__ __launch_bounds__(64) void group_norm_finish_kernel(const double* __restrict__ partial, int chunks, int groups,
                                                               double n, float eps, Moments* __restrict__ out) {
    const int g = blockIdx.x, image = blockIdx.y;
    double sum = 0.0, sq = 0.0;
    for (int i = threadIdx.x; i < chunks; i += 64) {
        const double* p = partial + ((int64_t(image) * chunks + i) * groups + g) * 2;
        sum += p[0];
        sq += p[1];
    }
    sum = wave_sum(sum);
    sq = wave_sum(sq);
    if (threadIdx.x == 0) out[image * groups + g] = moments(sum, sq, n, eps);
}

template <class TI, class TO, int VEC>
__global__ __launch_bounds__(256) void group_norm_apply_kernel(const TI* x, TO* y, GroupNormShape s, int chunk,
                                                               const Moments* __restrict__ stats, const float* __restrict__ w,
                                                               const float* __restrict__ b, int act) {
    const int tid = threadIdx.x, cols = s.channels / VEC, size = s.channels / s.groups;
    const int width = min(cols, 256), rows = 256 / width, col0 = tid % width, row = tid / width;
    if (row >= rows) return;
    const int p0 = blockIdx.x * chunk, p1 = min(p0 + chunk, s.pixels);
    const TI* xi = x + blockIdx.y * s.x_image;
    TO* yi = y + blockIdx.y * s.y_image;
    for (int col = col0; col < cols; col += width) {
        Moments m[VEC];
        float ww[VEC], bb[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const int c = col * VEC + e;
            m[e] = stats[blockIdx.y * s.groups + c / size];
            ww[e] = w ? w[c] : 1.f;
            bb[e] = b ? b[c] : 0.f;
        }
        const TI* xc = xi + col * VEC;
        TO* yc = yi + col * VEC;
#pragma unroll 4
        for (int p = p0 + row; p < p1; p += rows) {
            float v[VEC];
            load<TI, VEC>(xc + p * s.x_pixel, v);
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[e] = activate(act, normalize(v[e], m[e]) * ww[e] + bb[e]);
            store<TO, VEC>(yc + p * s.y_pixel, v);
        }
    }
}

struct Launch {
    const GroupNormShape& s;
    const float *w, *b;
    float eps;
    int act;
    void* scratch;
    hipStream_t stream;
};

template <class TI, class TO, int VEC>
void launch_typed(const TI* x, TO* y, const Launch& l) {
    const GroupNormShape& s = l.s;
    const int64_t vectors = int64_t(s.pixels) * (s.channels / s.groups) / VEC;
    if (group_norm_one_launch(s, VEC)) {
        const dim3 grid(s.groups, s.images);
#define SAMHIP_GN_BLOCK(NV) \
    group_norm_block_kernel<TI, TO, VEC, NV><<<grid, 1024, 0, l.stream>>>(x, y, s, l.w, l.b, l.eps, l.act)
        if (vectors <= 1024) SAMHIP_GN_BLOCK(1);
        else if (vectors <= 4096) SAMHIP_GN_BLOCK(4);
        else SAMHIP_GN_BLOCK(16);
#undef SAMHIP_GN_BLOCK
        return;
    }
    const int chunk = group_norm_chunk(s, VEC), chunks = (s.pixels + chunk - 1) / chunk;
    const dim3 grid(chunks, s.images);
    double* partial = static_cast<double*>(l.scratch);
    Moments* stats = reinterpret_cast<Moments*>(partial + int64_t(s.images) * chunks * s.groups * 2);
    const int cols = s.channels / VEC, rows = 256 / std::min(cols, 256);
    group_norm_stats_kernel<TI, VEC><<<grid, 256, size_t(rows) * s.channels * 16, l.stream>>>(x, s, chunk, partial);
    group_norm_finish_kernel<<<dim3(s.groups, s.images), 64, 0, l.stream>>>(
        partial, chunks, s.groups, double(s.pixels) * (s.channels / s.groups), l.eps, stats);
    group_norm_apply_kernel<TI, TO, VEC><<<grid, 256, 0, l.stream>>>(x, y, s, chunk, stats, l.w, l.b, l.act);
}

template <class TI, class TO>
void launch_vec(const void* x, void* y, int vec, const Launch& l) {
    if (vec == 4) launch_typed<TI, TO, 4>(static_cast<const TI*>(x), static_cast<TO*>(y), l);
    else launch_typed<TI, TO, 1>(static_cast<const TI*>(x), static_cast<TO*>(y), l);
}

}  // namespace

int group_norm_vec(const GroupNormShape& s, const void* x, int x_bytes, const void* y, int y_bytes) {
    const auto aligned = [](const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % (4 * size_t(bytes)) == 0; };
    const bool four = (s.channels / s.groups) % 4 == 0 && s.x_pixel % 4 == 0 && s.x_image % 4 == 0 && s.y_pixel % 4 == 0 &&
                      s.y_image % 4 == 0 && aligned(x, x_bytes) && aligned(y, y_bytes);
    return four ? 4 : 1;
}

bool group_norm_one_launch(const GroupNormShape& s, int vec) {
    return int64_t(s.pixels) * (s.channels / s.groups) / vec <= 16 * 1024;
}

int group_norm_chunk(const GroupNormShape& s, int vec) {
    const int cols = s.channels / vec, rows = 256 / std::min(cols, 256);
    const int most = std::max(1, 2048 / s.images);
    const int least = 8 * rows;
    return std::max(least, (s.pixels + most - 1) / most);
}

size_t group_norm_scratch_bytes(const GroupNormShape& s, int vec) {
    if (group_norm_one_launch(s, vec)) return 0;
    const int chunk = group_norm_chunk(s, vec), chunks = (s.pixels + chunk - 1) / chunk;
    return (size_t(chunks) * 16 + sizeof(Moments)) * s.images * s.groups;
}

void launch_group_norm(const void* x, int x_type, void* y, int y_type, const GroupNormShape& s, int vec, const float* w,
                       const float* b, float eps, int act, void* scratch, hipStream_t stream) {
    const Launch l{s, w, b, eps, act, scratch, stream};
    if (x_type == T_F32 && y_type == T_F32) launch_vec<float, float>(x, y, vec, l);
    else if (x_type == T_F32) launch_vec<float, _Float16>(x, y, vec, l);
    else if (y_type == T_F32) launch_vec<_Float16, float>(x, y, vec, l);
    else launch_vec<_Float16, _Float16>(x, y, vec, l);
}

}  // namespace samhip
