// Token embedding with scaling, and its gradient, gfx950.
//
//   out[t] = scale * table[id_t]                    (0 where id_t is padding, NaN where it is past the table)
//   dtable[v] = scale * sum over t with id_t = v of dout[t]
//
// Both are bound by memory: the forward reads and writes T rows, the backward
// reads T rows and writes the whole table's gradient, most of whose rows are zero.
//
// The sums run in the tokens' order whatever the launch does, without atomics:
// the tokens are sorted by id first (stable), then each row of the gradient adds
// up the run of tokens that its id has.
//
//  embed_sort   one workgroup per kIds ids. Each reads every token's id (they are
//               few beside the rows, and stay in L2), which gives it the place of
//               its own run of tokens without another workgroup's help: counts
//               per (id, wave) in LDS, a scan, and a second pass that places the
//               tokens. One launch, no waiting between workgroups, no partial
//               histograms in memory. 16 waves take a 16th of the tokens each, so
//               that a batch of one repeated token is no slower than another.
//  embed_long   runs of more than two units of the sorted tokens: the units'
//               sums to the workspace, so that a frequent token's rows are read
//               by many CUs.
//  embed_grad   one wave per (id, slab of 256 columns): zeros, the run's sum, or
//               the sum of its units', each row written once.
#include <algorithm>

#include "common.hpp"
#include "kernels.hpp"

namespace mc {
namespace {

// ---------------------------------------------------------------- forward
// VEC elements per lane and step: 16 bytes, or one where rows are not whole
// 16-byte vectors.
template <typename T, int VEC>
__device__ __forceinline__ void load_vec(const T* p, float (&v)[VEC]) {
    if constexpr (VEC == 1) v[0] = Elem<T>::load(p, 0);
    else if constexpr (VEC == Vec16<T>::N) Vec16<T>::load(p, v);
    else {  // 4 bf16
        const uint2 q = *reinterpret_cast<const uint2*>(p);
        v[0] = bf16_lo(q.x); v[1] = bf16_hi(q.x); v[2] = bf16_lo(q.y); v[3] = bf16_hi(q.y);
    }
}

template <typename T, int VEC>
__global__ __launch_bounds__(256) void embed_fwd(const T* __restrict__ table, const int32_t* __restrict__ ids,
                                                 T* __restrict__ out, int64_t tokens, int64_t vocab, int64_t dim,
                                                 int64_t padding, float scale) {
    const int64_t t = (int64_t)blockIdx.x * 4 + wave_id();
    if (t >= tokens) return;
    const int64_t id = ids[t];
    T* dst = out + t * dim;
    const bool pad = padding >= 0 && id == padding;
    if (id < 0 || id >= vocab || pad) {
        const float f = pad ? 0.f : __builtin_nanf("");
        for (int64_t d = lane_id(); d < dim; d += kWave) Elem<T>::store(dst, d, f);
        return;
    }
    const T* src = table + id * dim;
#pragma unroll 4
    for (int64_t d = (int64_t)lane_id() * VEC; d < dim; d += kWave * VEC) {
        float v[VEC];
        load_vec<T, VEC>(src + d, v);
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] *= scale;
        if constexpr (VEC == 1) Elem<T>::store(dst, d, v[0]);
        else Vec16<T>::store(dst + d, v);
    }
}

// --------------------------------------------------------------- backward
constexpr int kIds = 512, kSortWaves = 16, kSortThreads = kSortWaves * kWave;

// order[N]: the N tokens with an id of the table that is not padding, by id, in
// their order within an id; start[v]: the first of id v there, start[vocab] = N.
__global__ __launch_bounds__(kSortThreads) void embed_sort(const int32_t* __restrict__ ids, int32_t tokens,
                                                           int64_t vocab, int64_t padding,
                                                           int32_t* __restrict__ order, int32_t* __restrict__ start) {
    __shared__ int32_t count[kSortWaves][kIds];
    __shared__ int32_t wsum[kSortWaves], before[kSortWaves];
    const int tid = threadIdx.x, lane = lane_id(), wave = wave_id();
    const int64_t first = (int64_t)blockIdx.x * kIds;
    const int32_t last = (int32_t)(first + kIds < vocab ? first + kIds : vocab);  // ids below 2^31
    const int32_t lo = (int32_t)first;
    const int32_t pad = padding < vocab ? (int32_t)padding : -1;
    for (int i = tid; i < kSortWaves * kIds; i += kSortThreads) (&count[0][0])[i] = 0;
    // this wave's tokens, whole wave steps
    const int32_t steps = (int32_t)(((int64_t)tokens + kWave - 1) / kWave);
    const int32_t per = (steps + kSortWaves - 1) / kSortWaves;
    const int32_t s0 = wave * per, s1 = s0 + per < steps ? s0 + per : steps;
    __syncthreads();
    int32_t below = 0;
    constexpr int U = 4;
    for (int32_t s = s0; s < s1; s += U) {
        int32_t id[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t t = (int64_t)(s + u) * kWave + lane;
            id[u] = s + u < s1 && t < tokens ? ids[t] : -1;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool real = id[u] >= 0 && id[u] != pad;
            below += real && id[u] < lo;
            if (real && id[u] >= lo && id[u] < last) atomicAdd(&count[wave][id[u] - lo], 1);
        }
    }
#pragma unroll
    for (int m = 1; m < kWave; m <<= 1) below += __shfl_xor(below, m, kWave);
    if (lane == 0) before[wave] = below;
    __syncthreads();
    // exclusive scan over (id, wave): thread i < kIds owns id lo + i
    int32_t mine = 0;
    if (tid < kIds)
        for (int w = 0; w < kSortWaves; ++w) mine += count[w][tid];
    int32_t scan = mine;
#pragma unroll
    for (int m = 1; m < kWave; m <<= 1) {
        const int32_t up = __shfl_up(scan, m, kWave);
        if (lane >= m) scan += up;
    }
    if (lane == kWave - 1) wsum[wave] = scan;
    __syncthreads();
    int32_t base = 0;
    for (int w = 0; w < kSortWaves; ++w) {
        base += before[w];
        if (w < wave) base += wsum[w];
    }
    base += scan - mine;
    if (tid < kIds) {
        if (lo + (int64_t)tid < last) start[lo + tid] = base;
        if (lo + (int64_t)tid + 1 == vocab) start[vocab] = base + mine;
        for (int w = 0; w < kSortWaves; ++w) {
            const int32_t c = count[w][tid];
            count[w][tid] = base;
            base += c;
        }
    }
    __syncthreads();
    for (int32_t s = s0; s < s1; s += U) {
        int32_t id[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t t = (int64_t)(s + u) * kWave + lane;
            id[u] = s + u < s1 && t < tokens ? ids[t] : -1;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool in = id[u] >= 0 && id[u] != pad && id[u] >= lo && id[u] < last;
            uint64_t left = __ballot(in);
            while (left) {  // one id of this step at a time, its lanes in order
                const int l = __builtin_ctzll(left);
                const int32_t v = __builtin_amdgcn_readlane(id[u], l);
                const uint64_t same = __ballot(in && id[u] == v);
                volatile int32_t* place = &count[wave][v - lo];  // volatile: one lane moves it for the others
                const int32_t at = *place;
                if (in && id[u] == v)
                    order[at + __builtin_popcountll(same & (((uint64_t)1 << lane) - 1))] = (s + u) * kWave + lane;
                if (lane == l) *place = at + __builtin_popcountll(same);
                left &= ~same;
            }
        }
    }
}

// The columns of a wave: 4 per lane from d, one where VEC is 1 (then 64 apart).
constexpr int kSlab = 256;
template <typename T, int VEC>
__device__ __forceinline__ void add_row(const T* row, int64_t d, int64_t dim, float (&acc)[4]) {
    if constexpr (VEC == 4) {
        if (d < dim) {
            float v[4];
            load_vec<T, 4>(row + d, v);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[e] += v[e];
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (d + e * kWave < dim) acc[e] += Elem<T>::load(row, d + e * kWave);
    }
}
template <int VEC>
__device__ __forceinline__ void put_row(float* row, int64_t d, int64_t dim, const float (&v)[4]) {
    if constexpr (VEC == 4) {
        if (d < dim) Vec16<float>::store(row + d, v);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (d + e * kWave < dim) row[d + e * kWave] = v[e];
    }
}

// acc += dout of sorted tokens [from, to), eight rows in flight.
template <typename T, int VEC>
__device__ __forceinline__ void add_run(const T* __restrict__ dout, const int32_t* __restrict__ order, int32_t from,
                                        int32_t to, int64_t d, int64_t dim, float (&acc)[4]) {
    constexpr int U = 8;
    for (; from + U <= to; from += U) {
        float part[U][4];
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int e = 0; e < 4; ++e) part[u][e] = 0.f;
            add_row<T, VEC>(dout + (int64_t)order[from + u] * dim, d, dim, part[u]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
            acc[e] += ((part[0][e] + part[1][e]) + (part[2][e] + part[3][e])) +
                      ((part[4][e] + part[5][e]) + (part[6][e] + part[7][e]));
    }
    for (; from < to; ++from) add_row<T, VEC>(dout + (int64_t)order[from] * dim, d, dim, acc);
}

// part[c][0]: the sum over unit c of the sorted tokens of the run that goes on
// through its start, part[c][1]: of the run that starts inside it and goes on
// through its end; only of runs longer than two units.
template <typename T, int VEC>
__global__ __launch_bounds__(256) void embed_long(const T* __restrict__ dout, const int32_t* __restrict__ ids,
                                                  const int32_t* __restrict__ order,
                                                  const int32_t* __restrict__ start, float* __restrict__ part,
                                                  int64_t vocab, int64_t dim, int32_t unit) {
    const int64_t slabs = (dim + kSlab - 1) / kSlab;
    const int64_t job = (int64_t)blockIdx.x * 4 + wave_id();
    const int64_t c = job / slabs, d0 = job % slabs * kSlab;
    const int32_t n = start[vocab];
    const int64_t from = c * unit;
    if (from >= n) return;
    const int32_t to = (int32_t)(from + unit < n ? from + unit : n);
    const int64_t d = d0 + (VEC == 4 ? 4 * lane_id() : lane_id());
    int32_t id = ids[order[from]];
#pragma unroll
    for (int side = 0; side < 2; ++side) {
        if (side == 1) {
            const int32_t next = ids[order[to - 1]];
            if (next == id) return;
            id = next;
        }
        const int32_t a = start[id], b = start[id + 1];
        if (b - a <= 2 * unit) continue;
        float acc[4] = {0.f, 0.f, 0.f, 0.f};
        add_run<T, VEC>(dout, order, a > from ? a : (int32_t)from, b < to ? b : to, d, dim, acc);
        // a run that starts with the unit goes on through its start as well
        put_row<VEC>(part + (2 * c + (a > from)) * dim, d, dim, acc);
    }
}

constexpr int kRows = 8;  // ids per workgroup of embed_grad

template <typename T, int VEC, bool ADD>
__global__ __launch_bounds__(256) void embed_grad(const T* __restrict__ dout, const int32_t* __restrict__ order,
                                                  const int32_t* __restrict__ start, const float* __restrict__ part,
                                                  float* __restrict__ dtable, int64_t vocab, int64_t dim, float scale,
                                                  int32_t unit) {
    const int64_t v0 = (int64_t)blockIdx.x * kRows;
    const int slabs = (int)((dim + kSlab - 1) / kSlab);
    const int rows = (int)(vocab - v0 < kRows ? vocab - v0 : kRows);
    for (int job = wave_id(); job < rows * slabs; job += 4) {
        const int64_t v = v0 + job / slabs;
        const int64_t d = (int64_t)(job % slabs) * kSlab + (VEC == 4 ? 4 * lane_id() : lane_id());
        const int32_t a = start[v], b = start[v + 1];
        if (ADD && a == b) continue;
        float acc[4] = {0.f, 0.f, 0.f, 0.f};
        if (b - a <= 2 * unit) {
            add_run<T, VEC>(dout, order, a, b, d, dim, acc);
        } else {
            const int32_t c1 = (b - 1) / unit;
            for (int32_t c = a / unit; c <= c1; ++c)
                add_row<float, VEC>(part + (2 * (int64_t)c + (a > (int64_t)c * unit)) * dim, d, dim, acc);
        }
        float* row = dtable + v * dim;
        if constexpr (ADD) {
            float old[4] = {0.f, 0.f, 0.f, 0.f};
            add_row<float, VEC>(row, d, dim, old);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[e] = __builtin_fmaf(acc[e], scale, old[e]);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[e] *= scale;
        }
        put_row<VEC>(row, d, dim, acc);
    }
}

size_t align256(size_t n) { return (n + 255) / 256 * 256; }

// Sorted tokens per unit of a long run: few enough units that one wave adds them
// up, and their sums stay small beside the rows that they come from.
int32_t unit_of(int64_t tokens) {
    const int64_t per = (tokens + 1023) / 1024;
    return (int32_t)(per <= 64 ? 64 : (per + 63) / 64 * 64);
}

}  // namespace

EmbeddingWs embedding_bwd_ws(const mc_embedding_desc& d) {
    EmbeddingWs w{};
    size_t off = 0;
    w.order = off;  off += align256((size_t)d.tokens * 4);
    w.start = off;  off += align256(((size_t)d.vocab + 1) * 4);
    const int64_t unit = unit_of(d.tokens);
    if (d.tokens > 2 * unit) {
        w.part = off;
        off += align256((size_t)((d.tokens + unit - 1) / unit) * 2 * (size_t)d.dim * 4);
    }
    w.total = off;
    return w;
}

hipError_t launch_embedding_fwd(const mc_embedding_desc& d, const void* table, const int32_t* ids, void* out,
                                hipStream_t stream) {
    const dim3 grid((unsigned)((d.tokens + 3) / 4));
    auto go = [&](auto elem, auto vec) {
        typedef decltype(elem) T;
        embed_fwd<T, decltype(vec)::value><<<grid, 256, 0, stream>>>(static_cast<const T*>(table), ids,
                                                                     static_cast<T*>(out), d.tokens, d.vocab, d.dim,
                                                                     d.padding_id, d.scale);
    };
    if (d.dtype == MC_F32) {
        if (d.dim % 4 == 0) go(float{}, std::integral_constant<int, 4>{});
        else go(float{}, std::integral_constant<int, 1>{});
    } else {
        if (d.dim % 8 == 0) go(uint16_t{}, std::integral_constant<int, 8>{});
        else go(uint16_t{}, std::integral_constant<int, 1>{});
    }
    return hipGetLastError();
}

hipError_t launch_embedding_bwd(const mc_embedding_desc& d, const int32_t* ids, const void* dout, float* dtable,
                                bool accumulate, char* ws, hipStream_t stream) {
    const EmbeddingWs w = embedding_bwd_ws(d);
    int32_t* order = reinterpret_cast<int32_t*>(ws + w.order);
    int32_t* start = reinterpret_cast<int32_t*>(ws + w.start);
    float* part = reinterpret_cast<float*>(ws + w.part);
    const int32_t unit = unit_of(d.tokens);
    embed_sort<<<dim3((unsigned)((d.vocab + kIds - 1) / kIds)), kSortThreads, 0, stream>>>(
        ids, (int32_t)d.tokens, d.vocab, d.padding_id, order, start);
    const int64_t slabs = (d.dim + kSlab - 1) / kSlab;
    const dim3 glong((unsigned)(((d.tokens + unit - 1) / unit * slabs + 3) / 4));
    const dim3 ggrad((unsigned)((d.vocab + kRows - 1) / kRows));
    auto go = [&](auto elem, auto vec) {
        typedef decltype(elem) T;
        constexpr int VEC = decltype(vec)::value;
        const T* g = static_cast<const T*>(dout);
        if (d.tokens > 2 * unit)
            embed_long<T, VEC><<<glong, 256, 0, stream>>>(g, ids, order, start, part, d.vocab, d.dim, unit);
        if (accumulate)
            embed_grad<T, VEC, true><<<ggrad, 256, 0, stream>>>(g, order, start, part, dtable, d.vocab, d.dim,
                                                                d.scale, unit);
        else
            embed_grad<T, VEC, false><<<ggrad, 256, 0, stream>>>(g, order, start, part, dtable, d.vocab, d.dim,
                                                                 d.scale, unit);
    };
    if (d.dtype == MC_F32) {
        if (d.dim % 4 == 0) go(float{}, std::integral_constant<int, 4>{});
        else go(float{}, std::integral_constant<int, 1>{});
    } else {
        if (d.dim % 4 == 0) go(uint16_t{}, std::integral_constant<int, 4>{});
        else go(uint16_t{}, std::integral_constant<int, 1>{});
    }
    return hipGetLastError();
}

}  // namespace mc
