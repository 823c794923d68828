// Global norm of many gradients, and clipping by it, gfx950.
//
//   norm  = sqrt(sum over every element of every tensor of g^2)
//   scale = 1 where norm <= max_norm, else max_norm / norm
//   out   = scale * g, one rounding to the output's type
//
// Squares and their sums are held in 64 bits: a float32 square leaves float32's
// range for |g| outside about [1e-19, 1e19], and the norm of a large model adds
// 1e9 of them. The partition and the order of every sum depend on the sizes
// alone, so results are bitwise reproducible.
//
// Bound by memory: the norm reads each gradient, the clipping reads it again and
// writes it. grad_sumsq gives each workgroup a chunk of one tensor (the table of
// tensors travels by value as a kernel argument: no device allocation, nothing
// to keep alive for a captured graph) and one 64-bit partial sum; the chunks are
// so long that there are at most about kParts of them. The workgroups of
// grad_scale then each add up the partials themselves while their gradients are
// on the way, in place of a launch between the two that does it for all.
#include "common.hpp"
#include "kernels.hpp"

namespace mc {
namespace {

constexpr int kThreads = 256;

// 16 bytes of T as floats.
template <typename T> struct Vec {
    static constexpr int N = 16 / sizeof(T);
    static __device__ __forceinline__ void unpack(const uint4& q, float (&v)[N]) {
        if constexpr (N == 4) {
            v[0] = __uint_as_float(q.x); v[1] = __uint_as_float(q.y);
            v[2] = __uint_as_float(q.z); v[3] = __uint_as_float(q.w);
        } else {
            v[0] = bf16_lo(q.x); v[1] = bf16_hi(q.x); v[2] = bf16_lo(q.y); v[3] = bf16_hi(q.y);
            v[4] = bf16_lo(q.z); v[5] = bf16_hi(q.z); v[6] = bf16_lo(q.w); v[7] = bf16_hi(q.w);
        }
    }
};

// v of every thread of the workgroup summed in a fixed order, to every thread.
__device__ __forceinline__ double wg_sum64(double v, double* red) {
#pragma unroll
    for (int m = 1; m < kWave; m <<= 1) v += __shfl_xor(v, m, kWave);
    if (lane_id() == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    double t = red[0];
#pragma unroll
    for (int w = 1; w < kThreads / kWave; ++w) t += red[w];
    return t;
}

// The slot of a workgroup: the last whose first workgroup is not past it.
template <typename Batch>
__device__ __forceinline__ int slot_of(const Batch& b, int blk) {
    int lo = 0, hi = b.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (b.slot[mid].blk0 <= blk) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

template <typename T>
__device__ __forceinline__ double sumsq_range(const T* __restrict__ p, int64_t n) {
    constexpr int N = Vec<T>::N, U = 8;
    // elements before the first 16-byte boundary, then whole vectors, then the rest
    const int64_t mis = ((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / sizeof(T);
    const int64_t head = mis < n ? mis : n;
    const int64_t nv = (n - head) / N;
    const uint4* v = reinterpret_cast<const uint4*>(p + head);
    double acc[4] = {0.0, 0.0, 0.0, 0.0};
    int64_t i = threadIdx.x;
    for (; i + (U - 1) * kThreads < nv; i += U * kThreads) {
        uint4 q[U];
#pragma unroll
        for (int u = 0; u < U; ++u) q[u] = v[i + u * kThreads];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float x[N];
            Vec<T>::unpack(q[u], x);
#pragma unroll
            for (int e = 0; e < N; ++e) acc[e & 3] = __builtin_fma((double)x[e], (double)x[e], acc[e & 3]);
        }
    }
    for (; i < nv; i += kThreads) {
        float x[N];
        Vec<T>::unpack(v[i], x);
#pragma unroll
        for (int e = 0; e < N; ++e) acc[e & 3] = __builtin_fma((double)x[e], (double)x[e], acc[e & 3]);
    }
    const int64_t tail = head + nv * N;
    if ((int64_t)threadIdx.x < head) {
        const double x = (double)Elem<T>::load(p, threadIdx.x);
        acc[0] = __builtin_fma(x, x, acc[0]);
    }
    if (tail + threadIdx.x < n) {
        const double x = (double)Elem<T>::load(p, tail + threadIdx.x);
        acc[1] = __builtin_fma(x, x, acc[1]);
    }
    return (acc[0] + acc[1]) + (acc[2] + acc[3]);
}

__global__ __launch_bounds__(kThreads) void grad_sumsq(GradNormBatch b, double* __restrict__ parts) {
    __shared__ double red[kThreads / kWave];
    const GradNormSlot& t = b.slot[slot_of(b, (int)blockIdx.x)];
    const int64_t base = (int64_t)((int)blockIdx.x - t.blk0) * b.chunk;
    const int64_t n = t.n - base < b.chunk ? t.n - base : b.chunk;
    const double s = t.dtype == MC_F32 ? sumsq_range(static_cast<const float*>(t.g) + base, n)
                                       : sumsq_range(static_cast<const uint16_t*>(t.g) + base, n);
    const double total = wg_sum64(s, red);
    if (threadIdx.x == 0) parts[blockIdx.x] = total;
}

// The sum of all partials, the same in every workgroup that forms it.
__device__ __forceinline__ double sum_parts(const double* __restrict__ parts, int n, double* red) {
    double s = 0.0;
    for (int i = threadIdx.x; i < n; i += kThreads) s += parts[i];
    return wg_sum64(s, red);
}
// max_norm / norm in 64 bits, so that a norm past float32's range still scales.
__device__ __forceinline__ float scale_of(double norm, float max_norm) {
    return norm <= (double)max_norm ? 1.f : (float)((double)max_norm / norm);
}

__global__ __launch_bounds__(kThreads) void grad_norm_join(const double* __restrict__ parts, int n, float max_norm,
                                                           float* __restrict__ norm, float* __restrict__ scale) {
    __shared__ double red[kThreads / kWave];
    const double total = sqrt(sum_parts(parts, n, red));
    if (threadIdx.x == 0) {
        *norm = (float)total;
        if (scale) *scale = scale_of(total, max_norm);
    }
}

// out = f g over n elements. N elements at a time where both sides are 16-byte
// aligned at the same element; otherwise one, which still writes whole lines.
template <typename TI, typename TO>
__device__ __forceinline__ void scale_range(const TI* g, TO* out, int64_t n, float f) {
    constexpr int N = 16 / (sizeof(TI) < sizeof(TO) ? sizeof(TI) : sizeof(TO));
    constexpr int VI = N * sizeof(TI) / 16, VO = N * sizeof(TO) / 16, U = 2;
    const int64_t head0 = ((16 - (reinterpret_cast<uintptr_t>(g) & 15)) & 15) / sizeof(TI);
    const int64_t head1 = ((16 - (reinterpret_cast<uintptr_t>(out) & 15)) & 15) / sizeof(TO);
    const bool vec = sizeof(TI) == sizeof(TO) ? head0 == head1
                                              : ((reinterpret_cast<uintptr_t>(g) | reinterpret_cast<uintptr_t>(out)) & 15) == 0;
    if (!vec) {
        for (int64_t i = threadIdx.x; i < n; i += kThreads) Elem<TO>::store(out, i, Elem<TI>::load(g, i) * f);
        return;
    }
    const int64_t head = head0 < n ? head0 : n;
    const int64_t nv = (n - head) / N;
    const uint4* src = reinterpret_cast<const uint4*>(g + head);
    TO* dst = out + head;
    auto emit = [&](int64_t i, const uint4 (&q)[VI]) {
        float x[N];
#pragma unroll
        for (int k = 0; k < VI; ++k) {
            float y[Vec<TI>::N];
            Vec<TI>::unpack(q[k], y);
#pragma unroll
            for (int e = 0; e < Vec<TI>::N; ++e) x[k * Vec<TI>::N + e] = y[e] * f;
        }
#pragma unroll
        for (int k = 0; k < VO; ++k) {
            float y[Vec16<TO>::N];
#pragma unroll
            for (int e = 0; e < Vec16<TO>::N; ++e) y[e] = x[k * Vec16<TO>::N + e];
            Vec16<TO>::store(dst + i * N + k * Vec16<TO>::N, y);
        }
    };
    int64_t i = threadIdx.x;
    for (; i + (U - 1) * kThreads < nv; i += U * kThreads) {
        uint4 q[U][VI];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int k = 0; k < VI; ++k) q[u][k] = src[(i + u * kThreads) * VI + k];
#pragma unroll
        for (int u = 0; u < U; ++u) emit(i + u * kThreads, q[u]);
    }
    for (; i < nv; i += kThreads) {
        uint4 q[VI];
#pragma unroll
        for (int k = 0; k < VI; ++k) q[k] = src[i * VI + k];
        emit(i, q);
    }
    const int64_t tail = head + nv * N;
    if ((int64_t)threadIdx.x < head) Elem<TO>::store(out, threadIdx.x, Elem<TI>::load(g, threadIdx.x) * f);
    if (tail + threadIdx.x < n) Elem<TO>::store(out, tail + threadIdx.x, Elem<TI>::load(g, tail + threadIdx.x) * f);
}

// The scale is given (parts null), or formed from the norm's partials; then the
// first workgroup of the first launch also writes norm and scale.
__global__ __launch_bounds__(kThreads) void grad_scale(GradScaleBatch b, const float* __restrict__ given,
                                                       const double* __restrict__ parts, int nparts, float max_norm,
                                                       float* __restrict__ norm, float* __restrict__ scale) {
    __shared__ double red[kThreads / kWave];
    float f;
    if (parts) {
        const double total = sqrt(sum_parts(parts, nparts, red));
        f = scale_of(total, max_norm);
        if (norm && blockIdx.x == 0 && threadIdx.x == 0) {
            *norm = (float)total;
            *scale = f;
        }
    } else {
        f = *given;
    }
    if (b.count == 0) return;
    // backwards: the norm has left the last gradients that it read in the last-level cache
    const int blk = (int)(gridDim.x - 1 - blockIdx.x);
    const GradScaleSlot& t = b.slot[slot_of(b, blk)];
    if (f == 1.f && t.g == t.out) return;  // in place and nothing to clip
    const int64_t base = (int64_t)(blk - t.blk0) * b.chunk;
    const int64_t n = t.n - base < b.chunk ? t.n - base : b.chunk;
    if (t.dtype == MC_F32) {
        const float* g = static_cast<const float*>(t.g) + base;
        if (t.out_dtype == MC_F32) scale_range(g, static_cast<float*>(t.out) + base, n, f);
        else scale_range(g, static_cast<uint16_t*>(t.out) + base, n, f);
    } else {
        const uint16_t* g = static_cast<const uint16_t*>(t.g) + base;
        if (t.out_dtype == MC_F32) scale_range(g, static_cast<float*>(t.out) + base, n, f);
        else scale_range(g, static_cast<uint16_t*>(t.out) + base, n, f);
    }
}

// Elements per workgroup: 32 KB of float32 at least, and few enough chunks that
// every workgroup of the clipping can add their sums.
constexpr int64_t kMinChunk = 8192, kParts = 1024;

int64_t total_of(const mc_grad_tensor* t, int32_t count) {
    int64_t n = 0;
    for (int32_t i = 0; i < count; ++i) n += t[i].numel;
    return n;
}
int64_t chunk_of(int64_t total, int64_t parts) {
    const int64_t per = (total + parts - 1) / parts;
    return per <= kMinChunk ? kMinChunk : (per + kMinChunk - 1) / kMinChunk * kMinChunk;
}
int64_t blocks_of(int64_t n, int64_t chunk) { return (n + chunk - 1) / chunk; }

}  // namespace

int64_t gradient_parts(const mc_grad_tensor* t, int32_t count) {
    const int64_t chunk = chunk_of(total_of(t, count), kParts);
    int64_t n = 0;
    for (int32_t i = 0; i < count; ++i) n += blocks_of(t[i].numel, chunk);
    return n;
}

static hipError_t launch_sumsq(const mc_grad_tensor* t, int32_t count, double* parts, hipStream_t stream) {
    const int64_t chunk = chunk_of(total_of(t, count), kParts);
    GradNormBatch b;
    b.count = 0;
    b.chunk = chunk;
    int64_t blocks = 0;
    auto flush = [&]() {
        if (b.count == 0) return hipSuccess;
        grad_sumsq<<<dim3((unsigned)blocks), kThreads, 0, stream>>>(b, parts);
        parts += blocks;
        b.count = 0;
        blocks = 0;
        return hipGetLastError();
    };
    for (int32_t i = 0; i < count; ++i) {
        if (t[i].numel == 0) continue;
        b.slot[b.count++] = GradNormSlot{t[i].grad, t[i].numel, (int)blocks, t[i].dtype};
        blocks += blocks_of(t[i].numel, chunk);
        if (b.count == kGradNormSlots) {
            const hipError_t e = flush();
            if (e != hipSuccess) return e;
        }
    }
    return flush();
}

hipError_t launch_gradient_norm(const mc_grad_tensor* t, int32_t count, float max_norm, float* norm, float* scale,
                                double* parts, hipStream_t stream) {
    const hipError_t e = launch_sumsq(t, count, parts, stream);
    if (e != hipSuccess) return e;
    grad_norm_join<<<1, kThreads, 0, stream>>>(parts, (int)gradient_parts(t, count), max_norm, norm, scale);
    return hipGetLastError();
}

static hipError_t launch_scale(const mc_grad_tensor* t, int32_t count, const float* given, const double* parts,
                               int nparts, float max_norm, float* norm, float* scale, hipStream_t stream) {
    // a round or two of the CUs' workgroups
    const int64_t chunk = chunk_of(total_of(t, count), 4096);
    GradScaleBatch b;
    b.count = 0;
    b.chunk = chunk;
    int64_t blocks = 0;
    bool first = true;
    auto flush = [&]() {
        grad_scale<<<dim3((unsigned)(blocks ? blocks : 1)), kThreads, 0, stream>>>(b, given, parts, nparts, max_norm,
                                                                                  first ? norm : nullptr, scale);
        first = false;
        b.count = 0;
        blocks = 0;
        return hipGetLastError();
    };
    for (int32_t i = 0; i < count; ++i) {
        if (t[i].numel == 0) continue;
        b.slot[b.count++] = GradScaleSlot{t[i].grad, t[i].out, t[i].numel, (int)blocks, (int16_t)t[i].dtype,
                                          (int16_t)t[i].out_dtype};
        blocks += blocks_of(t[i].numel, chunk);
        if (b.count == kGradScaleSlots) {
            const hipError_t e = flush();
            if (e != hipSuccess) return e;
        }
    }
    return b.count > 0 || (first && norm) ? flush() : hipSuccess;
}

hipError_t launch_scale_gradients(const mc_grad_tensor* t, int32_t count, const float* scale, hipStream_t stream) {
    return launch_scale(t, count, scale, nullptr, 0, 0.f, nullptr, nullptr, stream);
}

hipError_t launch_clip_gradients(const mc_grad_tensor* t, int32_t count, float max_norm, float* norm, float* scale,
                                 double* parts, hipStream_t stream) {
    const hipError_t e = launch_sumsq(t, count, parts, stream);
    if (e != hipSuccess) return e;
    return launch_scale(t, count, nullptr, parts, (int)gradient_parts(t, count), max_norm, norm, scale, stream);
}

}  // namespace mc
