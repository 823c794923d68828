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

// The columns of a wave: 4 per lane from d (which may lie past the row), row by
// row through buffer loads, whose range check drops the lanes past the row: no
// branch stands between the loads of several rows. Rows of float32 start at any
// 4 bytes, which a 16-byte buffer access takes; a row that is not whole 16-byte
// vectors keeps its last columns in `rest`, one per lane.
constexpr int kSlab = 256;
struct Columns {
    int d;        // this lane's first column
    int rest;     // its column of the row's last dim % 4, or -1
};
__device__ __forceinline__ Columns columns_of(int64_t slab, int64_t dim) {
    const int64_t d0 = slab * kSlab;
    const int whole = (int)(dim & ~(int64_t)3), lane = lane_id();
    const bool last = d0 + kSlab >= whole;  // of slabs_of(dim) (dim < 2^29)
    return Columns{(int)d0 + 4 * lane, last && whole + lane < dim ? whole + lane : -1};
}
__host__ __device__ inline int64_t slabs_of(int64_t dim) { return dim < 4 ? 1 : ((dim & ~(int64_t)3) + kSlab - 1) / kSlab; }
struct Sum {
    float v[4], rest;
};
// 4 floats of a row at column c.d and the rest's; zeros past the row.
template <typename T, int VEC>
__device__ __forceinline__ Sum load_row(const T* row, const Columns& c, int dim) {
    Sum s;
    const __amdgpu_buffer_rsrc_t r = make_rsrc(row, (int64_t)dim * (int)sizeof(T));
    const uint32_t off = c.d + 4 <= dim ? (uint32_t)c.d * (uint32_t)sizeof(T) : kOOB;
    if constexpr (sizeof(T) == 4) {
        const i32x4 q = buf_load16(r, off);
#pragma unroll
        for (int e = 0; e < 4; ++e) s.v[e] = __int_as_float(q[e]);
        s.rest = VEC == 4 ? 0.f
                          : __int_as_float(__builtin_amdgcn_raw_buffer_load_b32(r, c.rest >= 0 ? 4 * c.rest : (int)kOOB, 0, 0));
    } else if constexpr (VEC == 4) {
        const u32x2 q = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(r, (int)off, 0, 0));
        s.v[0] = bf16_lo(q[0]); s.v[1] = bf16_hi(q[0]); s.v[2] = bf16_lo(q[1]); s.v[3] = bf16_hi(q[1]);
        s.rest = 0.f;
    } else {  // rows of bf16 that start at any 2 bytes: one element at a time
#pragma unroll
        for (int e = 0; e < 4; ++e)
            s.v[e] = bf16_to_f32((uint16_t)__builtin_amdgcn_raw_buffer_load_b16(
                r, (int)(off == kOOB ? kOOB : off + 2u * (uint32_t)e), 0, 0));
        s.rest = bf16_to_f32((uint16_t)__builtin_amdgcn_raw_buffer_load_b16(r, c.rest >= 0 ? 2 * c.rest : (int)kOOB, 0, 0));
    }
    return s;
}
template <int VEC>
__device__ __forceinline__ void store_row(float* row, const Columns& c, int dim, const Sum& s) {
    const __amdgpu_buffer_rsrc_t r = make_rsrc(row, (int64_t)dim * 4);
    const i32x4 q = {__float_as_int(s.v[0]), __float_as_int(s.v[1]), __float_as_int(s.v[2]), __float_as_int(s.v[3])};
    __builtin_amdgcn_raw_buffer_store_b128(q, r, (int)(c.d + 4 <= dim ? (uint32_t)c.d * 4u : kOOB), 0, 0);
    if constexpr (VEC != 4)
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_int(s.rest), r, c.rest >= 0 ? 4 * c.rest : (int)kOOB, 0, 0);
}
__device__ __forceinline__ void add(Sum& x, const Sum& y) {
#pragma unroll
    for (int e = 0; e < 4; ++e) x.v[e] += y.v[e];
    x.rest += y.rest;
}

// acc += dout of sorted tokens [from, to), eight rows in flight.
template <typename T, int VEC>
__device__ __forceinline__ void add_run(const T* __restrict__ dout, const int32_t* __restrict__ order, int32_t from,
                                        int32_t to, const Columns& c, int dim, Sum& acc) {
    constexpr int U = 8;
    for (; from + U <= to; from += U) {
        Sum part[U];
#pragma unroll
        for (int u = 0; u < U; ++u) part[u] = load_row<T, VEC>(dout + (int64_t)order[from + u] * dim, c, dim);
#pragma unroll
        for (int s = 1; s < U; s *= 2)
#pragma unroll
            for (int u = 0; u < U; u += 2 * s) add(part[u], part[u + s]);
        add(acc, part[0]);
    }
    for (; from < to; ++from) add(acc, load_row<T, VEC>(dout + (int64_t)order[from] * dim, c, dim));
}

// part[c][0]: the sum over unit c of the sorted tokens of the run that goes on
// through its start, part[c][1]: of the run that starts inside it and goes on
// through its end; only of runs longer than two units.
template <typename T, int VEC>
__global__ __launch_bounds__(256) void embed_long(const T* __restrict__ dout, const int32_t* __restrict__ ids,
                                                  const int32_t* __restrict__ order,
                                                  const int32_t* __restrict__ start, float* __restrict__ part,
                                                  int64_t vocab, int dim, int32_t unit) {
    const int64_t slabs = slabs_of(dim);
    const int64_t job = (int64_t)blockIdx.x * 4 + wave_id();
    const int64_t c = job / slabs;
    const int32_t n = start[vocab];
    const int64_t from = c * unit;
    if (from >= n) return;
    const int32_t to = (int32_t)(from + unit < n ? from + unit : n);
    const Columns cols = columns_of(job % slabs, dim);
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
        Sum acc{};
        add_run<T, VEC>(dout, order, a > from ? a : (int32_t)from, b < to ? b : to, cols, dim, acc);
        // a run that starts with the unit goes on through its start as well
        store_row<VEC>(part + (2 * c + (a > from)) * dim, cols, dim, acc);
    }
}

constexpr int kRows = 8;  // ids per workgroup of embed_grad

template <typename T, int VEC, bool ADD>
__global__ __launch_bounds__(256) void embed_grad(const T* __restrict__ dout, const int32_t* __restrict__ order,
                                                  const int32_t* __restrict__ start, const float* __restrict__ part,
                                                  float* __restrict__ dtable, int64_t vocab, int dim, float scale,
                                                  int32_t unit) {
    const int64_t v0 = (int64_t)blockIdx.x * kRows;
    const int slabs = (int)slabs_of(dim);
    const int rows = (int)(vocab - v0 < kRows ? vocab - v0 : kRows);
    for (int job = wave_id(); job < rows * slabs; job += 4) {
        const int64_t v = v0 + job / slabs;
        const Columns cols = columns_of(job % slabs, dim);
        const int32_t a = start[v], b = start[v + 1];
        if (ADD && a == b) continue;
        Sum acc{};
        if (b - a <= 2 * unit) {
            add_run<T, VEC>(dout, order, a, b, cols, dim, acc);
        } else {
            const int32_t c1 = (b - 1) / unit;
            for (int32_t c = a / unit; c <= c1; ++c)
                add(acc, load_row<float, VEC>(part + (2 * (int64_t)c + (a > (int64_t)c * unit)) * dim, cols, dim));
        }
        float* row = dtable + v * dim;
        Sum old{};
        if constexpr (ADD) old = load_row<float, VEC>(row, cols, dim);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc.v[e] = __builtin_fmaf(acc.v[e], scale, old.v[e]);
        acc.rest = __builtin_fmaf(acc.rest, scale, old.rest);
        store_row<VEC>(row, cols, dim, acc);
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
    const int64_t slabs = slabs_of(d.dim);
    const dim3 glong((unsigned)(((d.tokens + unit - 1) / unit * slabs + 3) / 4));
    const dim3 ggrad((unsigned)((d.vocab + kRows - 1) / kRows));
    auto go = [&](auto elem, auto vec) {
        typedef decltype(elem) T;
        constexpr int VEC = decltype(vec)::value;
        const T* g = static_cast<const T*>(dout);
        if (d.tokens > 2 * unit)
            embed_long<T, VEC><<<glong, 256, 0, stream>>>(g, ids, order, start, part, d.vocab, (int)d.dim, unit);
        if (accumulate)
            embed_grad<T, VEC, true><<<ggrad, 256, 0, stream>>>(g, order, start, part, dtable, d.vocab, (int)d.dim,
                                                                d.scale, unit);
        else
            embed_grad<T, VEC, false><<<ggrad, 256, 0, stream>>>(g, order, start, part, dtable, d.vocab, (int)d.dim,
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
