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
// writes it. 281M bf16 gradients to float32: 97 us for the norm (562 MB, 5.8 TB/s),
// 288 for the clipping (562 MB read, 1.12 GB written, 5.9 TB/s); 1 to 6 MB: 8 us,
// the two launches. The table of tensors travels by value as a kernel argument: no
// device allocation, nothing to keep alive for a captured graph.
//
//  grad_sumsq      a chunk of one tensor per workgroup, one 64-bit partial sum.
//  grad_norm_join  the partials' sum, the norm and the scale. Where there are few
//                  partials the workgroups of grad_scale add them up themselves
//                  while their gradients are on the way, and the launch is saved.
//  grad_scale      one vector per thread: the workgroups of such a launch sweep
//                  memory in order, which writes reach 6.2 TB/s at (workgroups of
//                  32 KB and more 5.0: the device's writes are then spread over as
//                  many places as it runs workgroups).
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

// The slot of a workgroup: the last whose first workgroup is not past it, from a
// coarse index on (few dependent scalar loads: a workgroup lives for 2 us).
template <typename Batch>
__device__ __forceinline__ int slot_of(const Batch& b, uint32_t blk) {
    int s = b.first[blk >> b.shift];
    while (s + 1 < b.count && b.slot[s + 1].blk0 <= blk) ++s;
    return s;
}
// Addresses in the tables carry the tensor's type in their lowest bit (elements
// are 2 bytes or 4): 1 for bf16.
__device__ __forceinline__ bool is_bf16(uint64_t at) { return at & 1; }
template <typename T> __device__ __forceinline__ T* pointer(uint64_t at) {
    return reinterpret_cast<T*>(at & ~(uint64_t)1);
}

template <typename T>
__device__ __forceinline__ double sumsq_range(const T* __restrict__ p, int64_t n) {
    constexpr int N = Vec<T>::N, U = 4;
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
    const GradNormSlot& t = b.slot[slot_of(b, blockIdx.x)];
    const uint32_t base = (blockIdx.x - t.blk0) * b.chunk;
    const int64_t n = t.n - base < b.chunk ? t.n - base : b.chunk;
    const double s = is_bf16(t.g) ? sumsq_range(pointer<const uint16_t>(t.g) + base, n)
                                  : sumsq_range(pointer<const float>(t.g) + base, n);
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

// Four elements as loaded and stored by one thread.
__device__ __forceinline__ void load4(const float* p, float (&v)[4]) { Vec16<float>::load(p, v); }
__device__ __forceinline__ void load4(const uint16_t* p, float (&v)[4]) {
    const uint2 q = *reinterpret_cast<const uint2*>(p);
    v[0] = bf16_lo(q.x); v[1] = bf16_hi(q.x); v[2] = bf16_lo(q.y); v[3] = bf16_hi(q.y);
}
template <bool STREAM, typename V, typename T>
__device__ __forceinline__ void put(T* p, const V& v) {
    if constexpr (STREAM) __builtin_nontemporal_store(v, reinterpret_cast<V*>(p));
    else *reinterpret_cast<V*>(p) = v;
}
template <bool STREAM> __device__ __forceinline__ void store4(float* p, const float (&v)[4]) {
    put<STREAM>(p, f32x4{v[0], v[1], v[2], v[3]});
}
template <bool STREAM> __device__ __forceinline__ void store4(uint16_t* p, const float (&v)[4]) {
    put<STREAM>(p, u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])});
}

// out = f g over the n <= kScaleElems elements of a workgroup. Four at a time where
// both sides are aligned to their four, all of a thread's loads before its stores;
// otherwise one, which still writes whole lines.
constexpr int kScaleVecs = 4, kScaleElems = kThreads * 4 * kScaleVecs;
template <bool STREAM, typename TI, typename TO>
__device__ __forceinline__ void scale_range(const TI* g, TO* out, int n, float f) {
    const uintptr_t gm = reinterpret_cast<uintptr_t>(g) % (4 * sizeof(TI)), om = reinterpret_cast<uintptr_t>(out) % (4 * sizeof(TO));
    if (gm != 0 || om != 0) {
        for (int i = threadIdx.x; i < n; i += kThreads) Elem<TO>::store(out, i, Elem<TI>::load(g, i) * f);
        return;
    }
    const int i0 = (int)threadIdx.x * 4;
    float v[kScaleVecs][4];
    if (n == kScaleElems) {
#pragma unroll
        for (int u = 0; u < kScaleVecs; ++u) load4(g + i0 + u * kThreads * 4, v[u]);
#pragma unroll
        for (int u = 0; u < kScaleVecs; ++u) {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[u][e] *= f;
            store4<STREAM>(out + i0 + u * kThreads * 4, v[u]);
        }
        return;
    }
    for (int i = i0; i < n; i += kThreads * 4) {
        if (i + 4 <= n) {
            load4(g + i, v[0]);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[0][e] *= f;
            store4<STREAM>(out + i, v[0]);
        } else {
            for (int e = i; e < n; ++e) Elem<TO>::store(out, e, Elem<TI>::load(g, e) * f);
        }
    }
}

// The scale is given (parts null), or formed from the norm's partials; then the
// first workgroup of the first launch also writes norm and scale.
template <bool STREAM>
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
    const GradScaleSlot& t = b.slot[slot_of(b, blockIdx.x)];
    if (f == 1.f && t.g == t.out) return;  // in place and nothing to clip
    const uint32_t base = (blockIdx.x - t.blk0) * b.chunk;
    const int n = (int)(t.n - base < b.chunk ? t.n - base : b.chunk);
    if (is_bf16(t.g)) {
        const uint16_t* g = pointer<const uint16_t>(t.g) + base;
        if (is_bf16(t.out)) scale_range<STREAM>(g, pointer<uint16_t>(t.out) + base, n, f);
        else scale_range<STREAM>(g, pointer<float>(t.out) + base, n, f);
    } else {
        const float* g = pointer<const float>(t.g) + base;
        if (is_bf16(t.out)) scale_range<STREAM>(g, pointer<uint16_t>(t.out) + base, n, f);
        else scale_range<STREAM>(g, pointer<float>(t.out) + base, n, f);
    }
}

// Elements per workgroup of the norm: 32 KB of float32 at least, and at most about
// kParts of them, which the join adds up by one workgroup. Norm of 2M / 8M / 64M / 281M
// bf16, us: as it is 5.6 / 7.5 / 29 / 117; at most 1024 parts 7.3 / 7.5 / 27 / 120, 16384
// 6.4 / 7.5 / 31 / 120; at least 2048 elements 6.5 / 11.7 / 28 / 117, 32768 6.9 / 7.3 / 27 /
// 117.
constexpr int64_t kMinChunk = 8192, kParts = 4096;
// Partials that every workgroup of the clipping adds up itself (2 per thread). Added up
// there / by a launch of one workgroup, us: 16 partials 6.2 / 7.2, 128 6.7 / 7.9, 512 12.3 /
// 13.1, 1024 20.6 / 21.4; of 512 tensors, three launches of the clipping, 21.4 / 20.0, of
// 1024 tensors 38.5 / 33.7.
constexpr int64_t kFewParts = 512;
// Elements of a slot: offsets in it stay below 2^32, chunk multiples.
constexpr int64_t kSlotElems = (int64_t)1 << 31;
// Outputs past this go past the caches. bf16 gradients to float32 outputs of 64 / 256 /
// 320 / 512 / 1024 MB, us, through the caches: 30 / 97 / 126 / 221 / 425, past them: 30 / 89 /
// 107 / 168 / 410; with the AdamW step that reads them next 104 / 461 / 573 / 899 / 1784 and
// 100 / 451 / 550 / 871 / 1774. Up to here the two differ by 8% at most, and a reader that
// comes at once may find what it needs in the caches.
constexpr double kStreamBytes = 256.0 * 1048576.0;

int64_t total_of(const mc_grad_tensor* t, int32_t count) {
    int64_t n = 0;
    for (int32_t i = 0; i < count; ++i) n += t[i].numel;
    return n;
}
int64_t chunk_of(int64_t total) {
    const int64_t per = (total + kParts - 1) / kParts;
    int64_t chunk = kMinChunk;  // a power of two: it divides kSlotElems
    while (chunk < per && chunk < kSlotElems) chunk *= 2;
    return chunk;
}
int64_t blocks_of(int64_t n, int64_t chunk) { return (n + chunk - 1) / chunk; }

// Fills batches with the pieces of every tensor and calls launch(batch, blocks)
// for each full one and the last. make(tensor, first element): the slot without
// its size and first workgroup.
template <typename Batch, typename Make, typename Launch>
hipError_t for_batches(const mc_grad_tensor* t, int32_t count, int64_t chunk, Make&& make, Launch&& launch) {
    Batch b;
    b.count = 0;
    b.chunk = (uint32_t)chunk;
    int64_t blocks = 0;
    auto flush = [&]() {
        if (b.count == 0) return hipSuccess;
        b.shift = 0;
        while (((blocks - 1) >> b.shift) >= kGradIndex) ++b.shift;
        int s = 0;
        for (int i = 0; i < kGradIndex; ++i) {
            while (s + 1 < b.count && b.slot[s + 1].blk0 <= (uint64_t)i << b.shift) ++s;
            b.first[i] = (uint8_t)s;
        }
        const hipError_t e = launch(b, (unsigned)blocks);
        b.count = 0;
        blocks = 0;
        return e;
    };
    for (int32_t i = 0; i < count; ++i)
        for (int64_t at = 0; at < t[i].numel; at += kSlotElems) {
            const int64_t n = t[i].numel - at < kSlotElems ? t[i].numel - at : kSlotElems;
            // a launch holds at most 2^32 - 1 work-items
            if (blocks + blocks_of(n, chunk) > 16777215) {
                const hipError_t e = flush();
                if (e != hipSuccess) return e;
            }
            auto slot = make(t[i], at);
            slot.n = (uint32_t)n;
            slot.blk0 = (uint32_t)blocks;
            b.slot[b.count++] = slot;
            blocks += blocks_of(n, chunk);
            if (b.count == Batch::kSlots) {
                const hipError_t e = flush();
                if (e != hipSuccess) return e;
            }
        }
    return flush();
}

uint64_t tagged(const void* p, int64_t at, int32_t dtype) {
    return (reinterpret_cast<uint64_t>(p) + (uint64_t)at * (dtype == MC_F32 ? 4 : 2)) | (dtype == MC_BF16 ? 1 : 0);
}

hipError_t launch_sumsq(const mc_grad_tensor* t, int32_t count, double* parts, hipStream_t stream) {
    return for_batches<GradNormBatch>(
        t, count, chunk_of(total_of(t, count)),
        [](const mc_grad_tensor& x, int64_t at) { return GradNormSlot{tagged(x.grad, at, x.dtype), 0, 0}; },
        [&](const GradNormBatch& b, unsigned blocks) {
            grad_sumsq<<<dim3(blocks), kThreads, 0, stream>>>(b, parts);
            parts += blocks;
            return hipGetLastError();
        });
}

hipError_t launch_join(const double* parts, int64_t n, float max_norm, float* norm, float* scale, hipStream_t stream) {
    grad_norm_join<<<1, kThreads, 0, stream>>>(parts, (int)n, max_norm, norm, scale);
    return hipGetLastError();
}

hipError_t launch_scale(const mc_grad_tensor* t, int32_t count, const float* given, const double* parts, int nparts,
                        float max_norm, float* norm, float* scale, hipStream_t stream) {
    double bytes = 0.0;
    for (int32_t i = 0; i < count; ++i) bytes += (double)t[i].numel * (t[i].out_dtype == MC_F32 ? 4.0 : 2.0);
    return for_batches<GradScaleBatch>(
        t, count, kScaleElems,
        [](const mc_grad_tensor& x, int64_t at) {
            return GradScaleSlot{tagged(x.grad, at, x.dtype), tagged(x.out, at, x.out_dtype), 0, 0};
        },
        [&](const GradScaleBatch& b, unsigned blocks) {
            if (bytes > kStreamBytes)
                grad_scale<true><<<dim3(blocks), kThreads, 0, stream>>>(b, given, parts, nparts, max_norm, norm, scale);
            else
                grad_scale<false><<<dim3(blocks), kThreads, 0, stream>>>(b, given, parts, nparts, max_norm, norm, scale);
            norm = nullptr;  // written by the first launch
            return hipGetLastError();
        });
}

}  // namespace

int64_t gradient_parts(const mc_grad_tensor* t, int32_t count) {
    const int64_t chunk = chunk_of(total_of(t, count));
    int64_t n = 0;
    for (int32_t i = 0; i < count; ++i) n += blocks_of(t[i].numel, chunk);
    return n;
}

hipError_t launch_gradient_norm(const mc_grad_tensor* t, int32_t count, float max_norm, float* norm, float* scale,
                                double* parts, hipStream_t stream) {
    const hipError_t e = launch_sumsq(t, count, parts, stream);
    return e != hipSuccess ? e : launch_join(parts, gradient_parts(t, count), max_norm, norm, scale, stream);
}

hipError_t launch_scale_gradients(const mc_grad_tensor* t, int32_t count, const float* scale, hipStream_t stream) {
    return launch_scale(t, count, scale, nullptr, 0, 0.f, nullptr, nullptr, stream);
}

hipError_t launch_clip_gradients(const mc_grad_tensor* t, int32_t count, float max_norm, float* norm, float* scale,
                                 double* parts, hipStream_t stream) {
    hipError_t e = launch_sumsq(t, count, parts, stream);
    if (e != hipSuccess) return e;
    const int64_t n = gradient_parts(t, count);
    if (n <= kFewParts) return launch_scale(t, count, nullptr, parts, (int)n, max_norm, norm, scale, stream);
    e = launch_join(parts, n, max_norm, norm, scale, stream);
    return e != hipSuccess ? e : launch_scale(t, count, scale, nullptr, 0, 0.f, nullptr, nullptr, stream);
}

}  // namespace mc
