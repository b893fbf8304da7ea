// Group norm with an activation on channels-last maps (pixel rows of C
// channels, groups of C / G neighbouring channels):
//   y = act((x - mean) / sqrt(var + eps) * w + b)
// with mean and var (biased) over a group's channels of every pixel of one
// image.  Runs of up to 512 values sum x - shift and its square in F32, the
// shift the mean of the run's first values, and are joined in F64 as sums of
// x - base, the base a group's first value, so that neither a group of millions
// of values nor a mean far above the deviation costs digits; the mean is
// subtracted as two floats (hi, then lo).  So one pass over the data gives the
// statistics.
//   group_norm_block_kernel : one workgroup per (image, group) with the
//                             group's values in registers: x read once
//   group_norm_stats_kernel, _finish_kernel, _apply_kernel : larger groups
// Bound by HBM for large maps (288 x 288 x 256 F32 with ReLU: 43.1 us, 3.9 TB/s
// of x once and y; 16 for the sums and 27 for the rest, whose reads find part
// of x in the last-level cache), by two launches' latency for small ones
// (36 x 36 x 256: 8.4 us).
#include "internal.hpp"
#include "q8stage.hpp"

#pragma clang fp contract(off)

namespace samhip {

namespace {

// Channels of one load: 16 bytes.  Rows need no alignment beyond their
// element's.
template <class T>
constexpr int kVec = 16 / sizeof(T);

template <class T, int N>
struct __attribute__((packed, aligned(sizeof(T)))) Packed {
    typedef T type __attribute__((ext_vector_type(N)));
    type v;
};
template <class T>
using Vector = typename Packed<T, kVec<T>>::type;

// Channels ch .. of a pixel's row; those at or behind `channels` are whatever
// comes, and not read.  A branch around a load has it waited for at once, so
// how a group of loads is done is chosen outside of it: WHOLE reads them as
// they are, SHIFTED (a row holds a vector) the row's last vector again,
// shifted, GUARDED one by one.
enum class Edge { WHOLE, SHIFTED, GUARDED };
template <Edge E, class T>
__device__ __forceinline__ Vector<T> load(const T* row, int ch, int channels) {
    constexpr int VEC = kVec<T>;
    if constexpr (E == Edge::GUARDED) {
        Vector<T> v;
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = row[min(ch + e, channels - 1)];
        return v;
    }
    const int at = E == Edge::WHOLE ? ch : min(ch, channels - VEC);
    Vector<T> v = reinterpret_cast<const Packed<T, VEC>*>(row + at)->v;
    if constexpr (E == Edge::SHIFTED)
#pragma unroll
        for (int s = 1; s < VEC; s *= 2)
#pragma unroll
            for (int e = 0; e + s < VEC; ++e) v[e] = (ch - at) & s ? v[e + s] : v[e];
    return v;
}
template <Edge E>
struct EdgeTag {
    static constexpr Edge value = E;
};
template <bool SAME, class T, class Body>
__device__ __forceinline__ void with_edge(int channels, Body body) {   // uniform
    if constexpr (SAME) {
        body(EdgeTag<Edge::WHOLE>{});
    } else {
        if (channels % kVec<T> == 0) body(EdgeTag<Edge::WHOLE>{});
        else if (channels >= kVec<T>) body(EdgeTag<Edge::SHIFTED>{});
        else body(EdgeTag<Edge::GUARDED>{});
    }
}

// PAST: past the caches (a template's argument: of two stores in the branches
// of a condition the compiler makes an ordinary one).
template <bool PAST, class T, int VEC>
__device__ __forceinline__ void store(T* p, int n, const float (&v)[VEC]) {
    if (n == VEC) {
        Packed<T, VEC> r;
#pragma unroll
        for (int e = 0; e < VEC; ++e) r.v[e] = (T)v[e];   // F16: round to nearest even
        typedef T raw __attribute__((ext_vector_type(VEC), aligned(sizeof(T))));
        if constexpr (PAST) __builtin_nontemporal_store(r.v, reinterpret_cast<raw*>(p));
        else *reinterpret_cast<raw*>(p) = r.v;
        return;
    }
    // in pieces of 4, 2 and 1
    int at = 0;
    float a = v[0], b = v[1], c = v[2];
    if constexpr (VEC == 8) {
        if (n & 4) {
            Packed<T, 4> r;
#pragma unroll
            for (int e = 0; e < 4; ++e) r.v[e] = (T)v[e];
            *reinterpret_cast<Packed<T, 4>*>(p) = r;
            at = 4, a = v[4], b = v[5], c = v[6];
        }
    }
    if (n & 2) {
        Packed<T, 2> r;
        r.v[0] = (T)a;
        r.v[1] = (T)b;
        *reinterpret_cast<Packed<T, 2>*>(p + at) = r;
        at += 2, a = c;
    }
    if (n & 1) p[at] = (T)a;
}

// Sums of x - base and its square: F32 runs of x - shift, so that a mean far
// above the deviation cancels; what a run leaves goes to F64, about a base that
// all runs of a group share.  With the mean of k of the
// run's n values as the shift, s2 is at most 1 + n / k times the run's squared
// deviations, wherever outliers stand (with one value, which may be the
// outlier, 1 + n times: 4e-5 of the variance lost at n = 256).  It need not be
// exact: `inv` is about 1 / k.
struct Run {
    float shift = 0.f, s1 = 0.f, s2 = 0.f;
    __device__ __forceinline__ void aim(float x, float inv) { shift = __builtin_fmaf(x, inv, shift); }
    __device__ __forceinline__ void add(float x) {
        const float d = x - shift;
        s1 += d;
        s2 = __builtin_fmaf(d, d, s2);
    }
    __device__ __forceinline__ void into(float n, float base, double& sum, double& sq) const {
        const double a = (double)shift - (double)base, s = s1;
        sum += __builtin_fma((double)n, a, s);
        sq += __builtin_fma(a, __builtin_fma((double)n, a, 2.0 * s), (double)s2);
    }
};

template <int CTRL>
__device__ __forceinline__ double dpp_double(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double, uint64_t(uint32_t(samhip::dpp<CTRL>(int(u >> 32)))) << 32 | uint32_t(samhip::dpp<CTRL>(int(uint32_t(u)))));
}
// Sum over aligned runs of `lanes` (a power of two): each step adds the other
// half's sum, which a mirror reaches as well as an xor once halves agree.
__device__ __forceinline__ double lane_sum(double v, int lanes) {
    constexpr int HALF_MIRROR = 0x141, MIRROR = 0x140;
    if (lanes >= 2) v += dpp_double<DPP_XOR1>(v);
    if (lanes >= 4) v += dpp_double<DPP_XOR2>(v);
    if (lanes >= 8) v += dpp_double<HALF_MIRROR>(v);
    if (lanes >= 16) v += dpp_double<MIRROR>(v);
    const auto swapped = [&](auto swap) {
        const uint64_t u = __builtin_bit_cast(uint64_t, v);
        const auto lo = swap(uint32_t(u)), hi = swap(uint32_t(u >> 32));
        return __builtin_bit_cast(double, uint64_t(hi[0]) << 32 | lo[0]) + __builtin_bit_cast(double, uint64_t(hi[1]) << 32 | lo[1]);
    };
    if (lanes >= 32) v = swapped([](uint32_t x) { return __builtin_amdgcn_permlane16_swap(x, x, false, false); });
    if (lanes >= 64) v = swapped([](uint32_t x) { return __builtin_amdgcn_permlane32_swap(x, x, false, false); });
    return v;
}
__device__ __forceinline__ double wave_sum(double v) { return lane_sum(v, 64); }

// A group's statistics as the apply step uses them: mean = hi + lo.
struct Moments {
    float hi, lo, rstd;
};

constexpr int kGroupNormInline = 2048;   // partial sums that every workgroup of the last launch adds up itself

// From sums of x - base and its square.  The base is one of the n values, so
// that its distance from the mean is at most sqrt(n) deviations, and the
// variance loses at most n 2^-53 of itself.
__device__ __forceinline__ Moments moments(double sum, double sq, double n, double base, float eps) {
    const double off = sum / n, mean = base + off;
    double var = sq / n - off * off;
    var = var < 0.0 ? 0.0 : var;         // a NaN stays one
    Moments m;
    m.hi = (float)mean;
    m.lo = (float)(mean - (double)m.hi);
    m.rstd = (float)(1.0 / sqrt(var + (double)eps));
    return m;
}

template <int ACT>
__device__ __forceinline__ float activate(float v) {
    if constexpr (ACT == ACT_RELU) return v > 0.f || v != v ? v : 0.f;
    // reciprocal and exponential within an ulp each
    else if constexpr (ACT == ACT_SILU) return v * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(v * -1.4426950408889634f));
    else if constexpr (ACT == ACT_GELU_ERF) return gelu_erf(v);
    else return v;
}
template <int ACT>
struct ActTag {
    static constexpr int value = ACT;
};
template <class Body>
__device__ __forceinline__ void with_activation(int act, Body body) {   // uniform: once per pass, not per value
    switch (act) {
        case ACT_RELU: body(ActTag<ACT_RELU>{}); break;
        case ACT_SILU: body(ActTag<ACT_SILU>{}); break;
        case ACT_GELU_ERF: body(ActTag<ACT_GELU_ERF>{}); break;
        default: body(ActTag<ACT_NONE>{});
    }
}

// Gain and bias of channels c .. (`last` at most), all loads at once: a test
// for null around each would have it waited for there.
template <int VEC>
__device__ __forceinline__ void gain_and_bias(const float* w, const float* b, int c, int last, float (&ww)[VEC], float (&bb)[VEC]) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) ww[e] = 1.f, bb[e] = 0.f;
    if (w)
#pragma unroll
        for (int e = 0; e < VEC; ++e) ww[e] = w[min(c + e, last)];
    if (b)
#pragma unroll
        for (int e = 0; e < VEC; ++e) bb[e] = b[min(c + e, last)];
}

// One workgroup per (image, group).  A thread keeps to one vector of the
// group's channels and takes every rows-th pixel.
template <class TI, class TO, int NV>
__global__ __launch_bounds__(1024) void group_norm_block_kernel(const TI* x, TO* y, GroupNormShape s, const float* __restrict__ w,
                                                                const float* __restrict__ b, float eps, int act) {
    constexpr int VEC = kVec<TI>;
    __shared__ double part[16][2];
    const int g = blockIdx.x, image = blockIdx.y, tid = threadIdx.x;
    const int size = s.channels / s.groups, cols = (size + VEC - 1) / VEC, rows = blockDim.x / cols;
    const int row = tid / cols, c = (tid - row * cols) * VEC, n = min(size - c, VEC);
    const int count = row < rows && row < s.pixels ? (s.pixels - 1 - row) / rows + 1 : 0;   // at most NV
    const int64_t first = min(row, s.pixels - 1), x_step = rows * s.x_pixel, y_step = rows * s.y_pixel;
    const TI* xg = x + image * s.x_image + first * s.x_pixel;
    const float base = (float)x[image * s.x_image + g * size];
    TO* yg = y + image * s.y_image + g * size + c + first * s.y_pixel;
    Vector<TI> v[NV];
    const auto fetch = [&](auto edge) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            v[i] = load<decltype(edge)::value>(xg + max(min(i, count - 1), 0) * x_step, g * size + c, s.channels);
    };
    if (size % VEC == 0) fetch(EdgeTag<Edge::WHOLE>{});
    else if (s.channels >= VEC) fetch(EdgeTag<Edge::SHIFTED>{});
    else fetch(EdgeTag<Edge::GUARDED>{});
    float ww[VEC], bb[VEC];
    gain_and_bias<VEC>(w, b, g * size + c, g * size + size - 1, ww, bb);
    double sum = 0.0, sq = 0.0;
    {
        Run run;
        const float inv = __builtin_amdgcn_rcpf((float)(count * n));
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < VEC; ++e) run.aim(i < count && e < n ? (float)v[i][e] : 0.f, inv);
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < VEC; ++e) run.add(i < count && e < n ? (float)v[i][e] : run.shift);
        if (count) run.into((float)(count * n), base, sum, sq);
    }
    sum = wave_sum(sum);
    sq = wave_sum(sq);
    if ((tid & 63) == 0) {
        part[tid >> 6][0] = sum;
        part[tid >> 6][1] = sq;
    }
    __syncthreads();
    sum = sq = 0.0;
    for (int i = 0; i < int(blockDim.x) / 64; ++i) {
        sum += part[i][0];
        sq += part[i][1];
    }
    const Moments m = moments(sum, sq, double(s.pixels) * size, base, eps);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        ww[e] = ww[e] * m.rstd;
        bb[e] = bb[e] - m.lo * ww[e];
    }
    with_activation(act, [&](auto tag) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (i >= count) continue;
            float o[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) o[e] = activate<decltype(tag)::value>(__builtin_fmaf((float)v[i][e] - m.hi, ww[e], bb[e]));
            store<false>(yg + i * y_step, n, o);
        }
    });
}

constexpr int FLIGHT = 8;   // pixels that a thread has in flight
constexpr int RUN = 8;      // of which batches one F32 run

// Thread t of 256 owns the channels of vector t % cols (pass j: of vector
// t % cols + 256 j) and every rows-th pixel of the chunk.  SAME: the channels
// of a vector are of one group, and one run takes them all.
template <class TI, bool SAME>
__global__ __launch_bounds__(256) void group_norm_stats_kernel(const TI* __restrict__ x, GroupNormShape s, int chunk,
                                                               double* __restrict__ partial) {
    constexpr int VEC = kVec<TI>, RUNS = SAME ? 1 : VEC;
    extern __shared__ double sums[];   // [sum, sum of squares][rows][RUNS][cols]: lanes write neighbouring places
    const int tid = threadIdx.x, cols = (s.channels + VEC - 1) / VEC;
    const int width = min(cols, 256), rows = 256 / width, row = tid / width, col0 = tid - row * width;
    const int p0 = blockIdx.x * chunk + row, p1 = min((blockIdx.x + 1) * chunk, s.pixels);
    const int plane = rows * RUNS * cols, size = s.channels / s.groups;
    const TI* xi = x + blockIdx.y * s.x_image;
    const TI early = xi[min(tid, s.groups - 1) * size];   // a group's base, under way from here
    if (row < rows) {
        for (int col = col0; col < cols; col += width) {
            double sum[RUNS], sq[RUNS];
            TI base[RUNS];
            int first = col * VEC / size * size, behind = first + size;   // the group's channels
#pragma unroll
            for (int e = 0; e < RUNS; ++e) {
                sum[e] = sq[e] = 0.0;
                if (col * VEC + e == behind) first = behind, behind += size;
                base[e] = xi[min(first, s.channels - 1)];
            }
            for (int p = p0; p < p1;) {
                const int q = p;
                Run run[RUNS];
                for (int k = 0; k < RUN && p < p1; ++k, p += FLIGHT * rows) {
                    Vector<TI> v[FLIGHT];   // the last pixel again where there are no more
                    with_edge<SAME, TI>(s.channels, [&](auto edge) {
#pragma unroll
                        for (int u = 0; u < FLIGHT; ++u)
                            v[u] = load<decltype(edge)::value>(xi + min(p + u * rows, p1 - 1) * s.x_pixel, col * VEC, s.channels);
                    });
                    if (k == 0) {
                        int pixels = 1;
#pragma unroll
                        for (int u = 1; u < FLIGHT; ++u) pixels += p + u * rows < p1;
                        const float inv = __builtin_amdgcn_rcpf((float)(SAME ? pixels * VEC : pixels));
#pragma unroll
                        for (int u = 0; u < FLIGHT; ++u)
                            if (p + u * rows < p1)
#pragma unroll
                                for (int e = 0; e < VEC; ++e) run[SAME ? 0 : e].aim((float)v[u][e], inv);
                    }
#pragma unroll
                    for (int u = 0; u < FLIGHT; ++u)
                        if (p + u * rows < p1)
#pragma unroll
                            for (int e = 0; e < VEC; ++e) run[SAME ? 0 : e].add((float)v[u][e]);
                }
                const float count = (float)((min(p, p1) - q + rows - 1) / rows * (SAME ? VEC : 1));
#pragma unroll
                for (int e = 0; e < RUNS; ++e) {
                    TI b = base[e];
#if defined(__HIP_DEVICE_COMPILE__)
                    asm("" : "+v"(b));   // not converted ahead of the loop, which would wait for it there
#endif
                    run[e].into(count, (float)b, sum[e], sq[e]);
                }
            }
#pragma unroll
            for (int e = 0; e < RUNS; ++e) {
                sums[(row * RUNS + e) * cols + col] = sum[e];
                sums[plane + (row * RUNS + e) * cols + col] = sq[e];
            }
        }
    }
    __syncthreads();
    const int members = SAME ? size / VEC : size, all = rows * members;
    // as many lanes per group as leave a place for every group, 64 at most
    int lanes = 64;
    while (lanes > 1 && lanes * s.groups > 256) lanes >>= 1;
    for (int g = tid / lanes; g < s.groups; g += 256 / lanes) {
        double sum = 0.0, sq = 0.0;
        for (int i = tid & (lanes - 1); i < all; i += lanes) {
            const int r = i / members, ch = g * members + i - r * members;
            const int at = SAME ? r * cols + ch : (r * RUNS + ch % VEC) * cols + ch / VEC;
            sum += sums[at];
            sq += sums[plane + at];
        }
        sum = lane_sum(sum, lanes);
        sq = lane_sum(sq, lanes);
        if ((tid & (lanes - 1)) == 0) {
            double* out = partial + ((int64_t(blockIdx.y) * (gridDim.x + 1) + blockIdx.x) * s.groups + g) * 2;
            out[0] = sum;
            out[1] = sq;
        }
    }
    if (blockIdx.x == 0) {
        double* bases = partial + (int64_t(blockIdx.y) * (gridDim.x + 1) + gridDim.x) * s.groups * 2;
        for (int g = tid; g < s.groups; g += 256) bases[2 * g] = (double)(g == tid ? early : xi[g * size]);
    }
}

// An image's partial sums over its chunks, by 256 threads: thread t adds
// every (256 / groups)-th chunk's of group t % groups, neighbours reading
// neighbouring places.  The groups' bases stand behind the last chunk's sums.
// `out` has a place for each group.
__device__ __forceinline__ void finish(const double* __restrict__ partial, int chunks, int groups, double n, float eps,
                                       double (*lds)[2], Moments* out) {
    typedef double double2_t __attribute__((ext_vector_type(2)));
    const int tid = threadIdx.x;
    const double* bases = partial + int64_t(chunks) * groups * 2;
    double base = bases[2 * min(tid, groups - 1)];   // here, not in the loop, which would wait for all loads at its head
    for (int g0 = 0; g0 < groups; g0 += 256) {
        const int here = min(groups - g0, 256), step = 256 / here, c0 = tid / here, g = tid - c0 * here;
        double sum = 0.0, sq = 0.0;
        if (c0 < step) {
#pragma unroll 8
            for (int c = c0; c < chunks; c += step) {
                const double2_t p = *reinterpret_cast<const double2_t*>(partial + (int64_t(c) * groups + g0 + g) * 2);
                sum += p[0];
                sq += p[1];
            }
        }
        lds[tid][0] = sum;
        lds[tid][1] = sq;
        __syncthreads();
        if (tid < here) {
#pragma unroll 8
            for (int i = 1; i < step; ++i) {
                sum += lds[tid + i * here][0];
                sq += lds[tid + i * here][1];
            }
            out[g0 + tid] = moments(sum, sq, n, base, eps);
        }
        if (g0 + 256 < groups) base = bases[2 * min(g0 + 256 + tid, groups - 1)];
        __syncthreads();
    }
}

__global__ __launch_bounds__(256) void group_norm_finish_kernel(const double* __restrict__ partial, int chunks, int groups, double n,
                                                                float eps, Moments* __restrict__ out) {
    __shared__ double lds[256][2];
    finish(partial + int64_t(blockIdx.x) * (chunks + 1) * groups * 2, chunks, groups, n, eps, lds, out + int64_t(blockIdx.x) * groups);
}

// FINISH: the workgroups add up the partial sums themselves.
// The chunks in the other order: the last ones read are still in L2.
template <class TI, class TO, bool SAME, bool PAST, bool FINISH>
__global__ __launch_bounds__(256) void group_norm_apply_kernel(const TI* x, TO* y, GroupNormShape s, int chunk,
                                                               const double* __restrict__ partial, int chunks, const Moments* __restrict__ stats,
                                                               const float* __restrict__ w, const float* __restrict__ b, float eps,
                                                               int act) {
    constexpr int VEC = kVec<TI>;
    __shared__ Moments shared[FINISH ? kGroupNormInline : 1];
    __shared__ double lds[FINISH ? 256 : 1][2];
    const int tid = threadIdx.x, cols = (s.channels + VEC - 1) / VEC, size = s.channels / s.groups;
    const int width = min(cols, 256), rows = 256 / width, row = tid / width, col0 = tid - row * width;
    const int at = gridDim.x - 1 - blockIdx.x;
    const int p0 = at * chunk + row, p1 = min((at + 1) * chunk, s.pixels);
    const bool some = row < rows && p0 < p1;
    const TI* xi = x + blockIdx.y * s.x_image;
    TO* yi = y + blockIdx.y * s.y_image;
    constexpr int U = FLIGHT / 2;   // a batch is under way while the one before it is computed
    Vector<TI> v[U], next[U];
    auto fetch = [&](int col, int p, Vector<TI>(&v)[U]) {
        with_edge<SAME, TI>(s.channels, [&](auto edge) {
#pragma unroll
            for (int u = 0; u < U; ++u)
                v[u] = load<decltype(edge)::value>(xi + min(p + u * rows, p1 - 1) * s.x_pixel, col * VEC, s.channels);
        });
    };
    float ww[VEC], bb[VEC];
    if (some) {   // under way while the sums are finished
        fetch(col0, p0, v);
        gain_and_bias<VEC>(w, b, col0 * VEC, s.channels - 1, ww, bb);
    }
    if constexpr (FINISH) {
        finish(partial + int64_t(blockIdx.y) * (chunks + 1) * s.groups * 2, chunks, s.groups, double(s.pixels) * size, eps, lds, shared);
        __syncthreads();
    }
    const auto moments_of = [&](int g) -> Moments {   // from LDS or from memory, never from either by one pointer
        if constexpr (FINISH) return shared[g];
        else return stats[int64_t(blockIdx.y) * s.groups + g];
    };
    if (!some) return;
    for (int col = col0; col < cols; col += width) {
        float hi[SAME ? 1 : VEC];
        if (col != col0) gain_and_bias<VEC>(w, b, col * VEC, s.channels - 1, ww, bb);
        const int n = SAME ? VEC : min(s.channels - col * VEC, VEC);
        Moments m;
        if (SAME) {
            m = moments_of(col * VEC / size);
            hi[0] = m.hi;
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            if (!SAME) {
                m = moments_of(min(col * VEC + e, s.channels - 1) / size);
                hi[e] = m.hi;
            }
            ww[e] = ww[e] * m.rstd;
            bb[e] = bb[e] - m.lo * ww[e];
        }
        if (col != col0) fetch(col, p0, v);
        with_activation(act, [&](auto tag) {
            for (int p = p0; p < p1; p += U * rows) {
                const bool more = p + U * rows < p1;
                if (more) fetch(col, p + U * rows, next);
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int q = p + u * rows;
                    if (q < p1) {
                        float o[VEC];
#pragma unroll
                        for (int e = 0; e < VEC; ++e)
                            o[e] = activate<decltype(tag)::value>(__builtin_fmaf((float)v[u][e] - hi[SAME ? 0 : e], ww[e], bb[e]));
                        store<PAST>(yi + col * VEC + q * s.y_pixel, n, o);
                    }
                }
                if (more)
#pragma unroll
                    for (int u = 0; u < U; ++u) v[u] = next[u];
            }
        });
    }
}

int chunk_of(const GroupNormShape& s, int vec, int most);

template <class TI, class TO>
void launch_typed(const TI* x, TO* y, const GroupNormShape& s, const float* w, const float* b, float eps, int act, void* scratch,
                  hipStream_t stream) {
    constexpr int VEC = kVec<TI>;
    const int size = s.channels / s.groups;
    if (group_norm_one_launch(s, VEC)) {
        const int cols = (size + VEC - 1) / VEC;
        const dim3 grid(s.groups, s.images);
        const unsigned threads = unsigned(std::min<int64_t>((int64_t(s.pixels) * cols + 63) / 64 * 64, 1024));
        const int rows = int(threads) / cols, most = (s.pixels + rows - 1) / rows;   // vectors of a thread
#define SAMHIP_GN_BLOCK(NV) group_norm_block_kernel<TI, TO, NV><<<grid, threads, 0, stream>>>(x, y, s, w, b, eps, act)
        if (most <= 1) SAMHIP_GN_BLOCK(1);
        else if (most <= 4) SAMHIP_GN_BLOCK(4);
        else SAMHIP_GN_BLOCK(8);
#undef SAMHIP_GN_BLOCK
        return;
    }
    const int chunk = group_norm_stats_chunk(s, VEC), chunks = (s.pixels + chunk - 1) / chunk;
    const dim3 grid(chunks, s.images);
    // A map that no L2 would hold is written past the caches: 288 x 288 x 256
    // F32 57.2 -> 45.3 us (no write-back of the L2s at the launch's end; that
    // is 85 MB, with nothing behind it that reads the map: 32 MiB is a guess)
    const bool past_cache = int64_t(s.images) * s.pixels * s.channels * int64_t(sizeof(TO)) > (int64_t(32) << 20);
    const int apply_chunk = chunk_of(s, VEC, 1024 / s.images);
    const dim3 apply_grid((s.pixels + apply_chunk - 1) / apply_chunk, s.images);
    double* partial = static_cast<double*>(scratch);
    const int cols = (s.channels + VEC - 1) / VEC, rows = 256 / std::min(cols, 256);
    const bool same = size % VEC == 0;
    const size_t lds = size_t(rows) * cols * 16;
    if (same) group_norm_stats_kernel<TI, true><<<grid, 256, lds, stream>>>(x, s, chunk, partial);
    else group_norm_stats_kernel<TI, false><<<grid, 256, lds * VEC, stream>>>(x, s, chunk, partial);
    Moments* stats = nullptr;
    if (int64_t(chunks) * s.groups > kGroupNormInline) {
        stats = reinterpret_cast<Moments*>(partial + int64_t(s.images) * (chunks + 1) * s.groups * 2);
        group_norm_finish_kernel<<<s.images, 256, 0, stream>>>(partial, chunks, s.groups, double(s.pixels) * size, eps, stats);
    }
#define SAMHIP_GN_APPLY(SAME, PAST) \
    if (stats) group_norm_apply_kernel<TI, TO, SAME, PAST, false><<<apply_grid, 256, 0, stream>>>(x, y, s, apply_chunk, partial, chunks, stats, w, b, eps, act); \
    else group_norm_apply_kernel<TI, TO, SAME, PAST, true><<<apply_grid, 256, 0, stream>>>(x, y, s, apply_chunk, partial, chunks, stats, w, b, eps, act)
    if (same && past_cache) {
        SAMHIP_GN_APPLY(true, true);
    } else if (same) {
        SAMHIP_GN_APPLY(true, false);
    } else if (past_cache) {
        SAMHIP_GN_APPLY(false, true);
    } else {
        SAMHIP_GN_APPLY(false, false);
    }
#undef SAMHIP_GN_APPLY
}

}  // namespace

int group_norm_vec(int x_type) { return x_type == T_F16 ? kVec<_Float16> : kVec<float>; }

// Eight vectors of each of 1024 threads are what a workgroup holds; past 8192
// channels of pixels a CU's arithmetic takes longer than another launch,
// unless there are groups for most CUs (limits from a few sizes, not swept).
bool group_norm_one_launch(const GroupNormShape& s, int vec) {
    const int size = s.channels / s.groups, cols = (size + vec - 1) / vec, rows = 1024 / cols;
    return (s.pixels + rows - 1) / rows <= 8 && (int64_t(s.pixels) * size <= 8192 || int64_t(s.groups) * s.images >= 192);
}

namespace {
// Pixels of a workgroup's chunk for at most `most` chunks an image.
int chunk_of(const GroupNormShape& s, int vec, int most) {
    const int rows = 256 / std::min((s.channels + vec - 1) / vec, 256);
    return std::max(4 * rows, (s.pixels + std::max(most, 1) - 1) / std::max(most, 1));
}
}  // namespace

// 1024 workgroups in all, or fewer where their partial sums then are so few
// that the last launch adds them up, but a workgroup for every CU.
int group_norm_stats_chunk(const GroupNormShape& s, int vec) {
    return chunk_of(s, vec, std::min(1024 / s.images, std::max(kGroupNormInline / s.groups, 256 / s.images)));
}

size_t group_norm_scratch_bytes(const GroupNormShape& s, int vec) {
    if (group_norm_one_launch(s, vec)) return 0;
    const int chunk = group_norm_stats_chunk(s, vec), chunks = (s.pixels + chunk - 1) / chunk;
    return ((size_t(chunks) + 1) * 16 + sizeof(Moments)) * s.images * s.groups;
}

void launch_group_norm(const void* x, int x_type, void* y, int y_type, const GroupNormShape& s, const float* w, const float* b,
                       float eps, int act, void* scratch, hipStream_t stream) {
    const auto run = [&](auto* xp, auto* yp) { launch_typed(xp, yp, s, w, b, eps, act, scratch, stream); };
    const float* xf = static_cast<const float*>(x);
    const _Float16* xh = static_cast<const _Float16*>(x);
    float* yf = static_cast<float*>(y);
    _Float16* yh = static_cast<_Float16*>(y);
    if (x_type == T_F32 && y_type == T_F32) run(xf, yf);
    else if (x_type == T_F32) run(xf, yh);
    else if (y_type == T_F32) run(xh, yf);
    else run(xh, yh);
}

}  // namespace samhip
