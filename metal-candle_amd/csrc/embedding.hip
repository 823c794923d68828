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
//  embed_sort   one workgroup per 16 to 512 ids. Each reads every token's id (they are
//               few beside the rows, and stay in L2), which gives it the place of
//               its own run of tokens without another workgroup's help: counts
//               per (id, wave) in LDS, a scan, and a second pass that places the
//               tokens. One launch, no waiting between workgroups, no partial
//               histograms in memory. The waves take a share of the tokens each,
//               so that a batch of one repeated token is no slower than another.
//               Its other workgroups clear the gradient meanwhile.
//  embed_rows   one wave per sorted token and 256 columns: the first token of a run
//               sums the run. Of runs longer than two units of the sorted tokens the
//               first workgroups write the units' sums to the workspace, so that a
//               frequent token's rows are read by many CUs.
//  embed_join   the rows of those runs, from their units' sums.
//
// 16384 tokens whose ids crowd at the table's start, 151936 x 1536 bf16: forward 21
// us (100 MB, 4.7 TB/s); sort and clearing 136 us (933 MB, 6.8 TB/s: a fill's rate),
// rows 38, join 5. Added to a gradient that is there, with nothing to clear: 2036 tokens
// of 50257 x 893 30 us in place of 67, 4096 of 151936 x 896 35 in place of 147.
// A workgroup per sorted token, its waves taking the slabs of one row in turn: 65 us
// for the rows. Sorted tokens as (token, id) pairs instead of two arrays, whose
// consecutive tokens load at once: 54.
#include <type_traits>

#include "common.hpp"
#include "kernels.hpp"
#include "rules.hpp"

namespace mc {
namespace {

// ---------------------------------------------------------------- forward
// VEC elements per lane and step: 16 bytes, or one where rows are not whole
// 16-byte vectors.
template <typename T, int VEC>
__device__ __forceinline__ void load_vec(const T* p, float (&v)[VEC]) {
    if constexpr (VEC == 1) v[0] = Elem<T>::load(p, 0);
    else Vec16<T>::load(p, v);
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
constexpr int kIds = 512;  // of a sorting workgroup, at most (embedding_sort_ids)

// order[N]: the N tokens with an id of the table that is not padding, by id, in their
// order within an id; sorted[N]: their ids; start[v]: the first of id v there,
// start[vocab] = N.
// AHEAD wave steps of ids are in flight, and stay in registers between the two
// passes where they are all of a wave's. us, 2 / 4 / 8 / 16 ahead: 2036 tokens (2
// steps a wave) 4.4 / 5.9 / 6.2 / 7.2, 16384 (16 steps) 12.3 / 12.0 / 12.0 / 11.1,
// 65536 37.2 / 34.6 / 34.1 / 33.5: then the tests of every id bound it.
//
// The workgroups past sort_blocks clear the gradient meanwhile (`clear` floats of
// it), one vector per thread, so that they sweep memory in order: 933 MB take 137
// us, 155 with four vectors per thread, 172 with 16 or workgroups of 1024, and 165
// in chunks of 64 KB and more. WAVES: workgroups that clear have 4, where the sort
// of 16384 tokens takes 30 us instead of the 11 with 16 and hides behind them.
template <int WAVES, int AHEAD>
__global__ __launch_bounds__(WAVES * kWave) void embed_sort(const int32_t* __restrict__ ids, int32_t tokens,
                                                            int64_t vocab, int64_t padding,
                                                            int32_t* __restrict__ order, int32_t* __restrict__ sorted,
                                                            int32_t* __restrict__ start, int id_block,
                                                            int sort_blocks, float* __restrict__ dtable,
                                                            int64_t clear) {
    constexpr int kSortWaves = WAVES, kSortThreads = WAVES * kWave;
    if ((int)blockIdx.x >= sort_blocks) {
        const int64_t i = (((int64_t)blockIdx.x - sort_blocks) * kSortThreads + threadIdx.x) * 4;
        if (i + 4 <= clear) *reinterpret_cast<f32x4*>(dtable + i) = f32x4{0.f, 0.f, 0.f, 0.f};
        else
            for (int64_t e = i; e < clear; ++e) dtable[e] = 0.f;
        return;
    }
    __shared__ int32_t count[kSortWaves][kIds];
    __shared__ int32_t wsum[kSortWaves], before[kSortWaves];
    const int tid = threadIdx.x, lane = lane_id(), wave = wave_id();
    // this workgroup's ids [lo, lo + width); no token's key is -1 (unsigned)
    const uint32_t lo = blockIdx.x * (uint32_t)id_block;
    const uint32_t width = (uint32_t)(vocab - lo < id_block ? vocab - lo : id_block);
    const uint32_t pad = padding >= 0 && padding < vocab ? (uint32_t)padding : 0xffffffffu;
    for (int i = tid; i < kSortWaves * kIds; i += kSortThreads) (&count[0][0])[i] = 0;
    // this wave's tokens [t0, t1), whole wave steps
    const int32_t per = (int32_t)((((int64_t)tokens + kWave - 1) / kWave + kSortWaves - 1) / kSortWaves);
    const int64_t start0 = (int64_t)wave * per * kWave;
    const int32_t t1 = (int32_t)(start0 + (int64_t)per * kWave < tokens ? start0 + (int64_t)per * kWave : tokens);
    const int32_t t0 = (int32_t)(start0 < t1 ? start0 : t1);
    const __amdgpu_buffer_rsrc_t rid = make_rsrc(ids, (int64_t)tokens * 4);
    // AHEAD steps of tokens from t on: an id of the table, or -1
    uint32_t key[AHEAD];
    auto load_keys = [&](int32_t t) {
        const int32_t mine = t + lane;
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
            key[u] = (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(rid, (mine + u * kWave) * 4, 0, 0);
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
            key[u] = mine + u * kWave < t1 && key[u] != pad && (int32_t)key[u] >= 0 ? key[u] : 0xffffffffu;
    };
    __syncthreads();
    int32_t below = 0;  // tokens of smaller ids, wave-uniform
    for (int32_t t = t0; t < t1; t += AHEAD * kWave) {
        load_keys(t);
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            below += __builtin_popcountll(__ballot(key[u] < lo));
            if (key[u] - lo < width) atomicAdd(&count[wave][key[u] - lo], 1);
        }
    }
    if (lane == 0) before[wave] = below;
    __syncthreads();
    // exclusive scan over (id, wave): a thread owns kOwn ids
    constexpr int kOwn = kIds / kSortThreads > 0 ? kIds / kSortThreads : 1;  // ids per thread
    const bool owner = tid * kOwn < kIds;
    int32_t mine = 0;
    if (owner)
        for (int i = 0; i < kOwn; ++i)
            for (int w = 0; w < kSortWaves; ++w) mine += count[w][tid * kOwn + i];
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
    uint32_t total_at = 0xffffffffu;  // the table's last id
    if (owner)
        for (int i = 0; i < kOwn; ++i) {
            const uint32_t k = (uint32_t)(tid * kOwn + i);
            if (k < width) {
                start[lo + k] = base;
                if ((int64_t)lo + k + 1 == vocab) total_at = k;
            }
            for (int w = 0; w < kSortWaves; ++w) {
                const int32_t c = count[w][k];
                count[w][k] = base;
                base += c;
            }
            if (k == total_at) start[vocab] = base;
        }
    __syncthreads();
    for (int32_t t = t0; t < t1; t += AHEAD * kWave) {
        if (per > AHEAD) load_keys(t);  // otherwise they are still there
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const bool in = key[u] - lo < width;
            uint64_t left = __ballot(in);
            while (left) {  // one id of this step at a time, its lanes in order
                const int l = __builtin_ctzll(left);
                const uint32_t v = (uint32_t)__builtin_amdgcn_readlane((int)key[u], l);
                const uint64_t same = __ballot(in && key[u] == v);
                volatile int32_t* place = &count[wave][v - lo];  // volatile: one lane moves it for the others
                const int32_t at = *place;
                if (in && key[u] == v) {
                    const int32_t p = at + __builtin_popcountll(same & (((uint64_t)1 << lane) - 1));
                    order[p] = t + u * kWave + lane;
                    sorted[p] = (int32_t)v;
                }
                if (lane == l) *place = at + __builtin_popcountll(same);
                left &= ~same;
            }
        }
    }
}

__global__ __launch_bounds__(256) void embed_clear(float* __restrict__ dtable, int64_t clear) {
    const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i + 4 <= clear) *reinterpret_cast<f32x4*>(dtable + i) = f32x4{0.f, 0.f, 0.f, 0.f};
    else
        for (int64_t e = i; e < clear; ++e) dtable[e] = 0.f;
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

// The sum of rows [from, to), row i at row(i): eight in flight, then four, two and
// one.
template <int U, typename T, int VEC, typename Row>
__device__ __forceinline__ Sum sum_group(int64_t from, const Columns& c, int dim, Row&& row) {
    Sum part[U];
#pragma unroll
    for (int u = 0; u < U; ++u) part[u] = load_row<T, VEC>(row(from + u), c, dim);
#pragma unroll
    for (int s = 1; s < U; s *= 2)
#pragma unroll
        for (int u = 0; u < U; u += 2 * s) add(part[u], part[u + s]);
    return part[0];
}
template <typename T, int VEC, typename Row>
__device__ __forceinline__ Sum sum_rows(int64_t from, int64_t to, const Columns& c, int dim, Row&& row) {
    Sum acc{};
    for (; from + 8 <= to; from += 8) add(acc, sum_group<8, T, VEC>(from, c, dim, row));
    const int left = (int)(to - from);
    if (left & 4) add(acc, sum_group<4, T, VEC>(from, c, dim, row)), from += 4;
    if (left & 2) add(acc, sum_group<2, T, VEC>(from, c, dim, row)), from += 2;
    if (left & 1) add(acc, sum_group<1, T, VEC>(from, c, dim, row));
    return acc;
}
// Of dout over sorted tokens [from, to).
template <typename T, int VEC>
__device__ __forceinline__ Sum sum_run(const void* dout, const int32_t* __restrict__ order, int64_t from, int64_t to,
                                       const Columns& c, int dim) {
    return sum_rows<T, VEC>(from, to, c, dim,
                            [&](int64_t i) { return static_cast<const T*>(dout) + (int64_t)order[i] * dim; });
}

// scale * acc, added to what the row holds or in its place.
template <int VEC, bool ADD>
__device__ __forceinline__ void put_sum(float* row, const Columns& cols, int dim, float scale, Sum acc) {
    Sum old{};
    if constexpr (ADD) old = load_row<float, VEC>(row, cols, dim);
#pragma unroll
    for (int e = 0; e < 4; ++e) acc.v[e] = __builtin_fmaf(acc.v[e], scale, old.v[e]);
    acc.rest = __builtin_fmaf(acc.rest, scale, old.rest);
    store_row<VEC>(row, cols, dim, acc);
}

struct GradArgs {
    const void* dout;
    const int32_t *order, *sorted, *start;
    float *part, *dtable;
    int64_t vocab;
    int64_t long_blocks;  // the first workgroups: units of long runs
    int dim, unit;
    float scale;
};

// part[c][0]: the sum over unit c of the sorted tokens of the run that goes on
// through its start, part[c][1]: of the run that starts inside it and goes on
// through its end; only of runs longer than two units.
template <typename T, int VEC>
__device__ __forceinline__ void sum_unit(const GradArgs& a) {
    const int64_t slabs = slabs_of(a.dim);
    const int64_t job = (int64_t)blockIdx.x * 4 + wave_id();
    const int64_t c = job / slabs;
    const int32_t n = a.start[a.vocab];
    const int64_t from = c * a.unit;
    if (from >= n) return;
    const int32_t to = (int32_t)(from + a.unit < n ? from + a.unit : n);
    const Columns cols = columns_of(job % slabs, a.dim);
    int32_t id = a.sorted[from];
#pragma unroll
    for (int side = 0; side < 2; ++side) {
        if (side == 1) {
            const int32_t next = a.sorted[to - 1];
            if (next == id) return;
            id = next;
        }
        const int32_t x = a.start[id], y = a.start[id + 1];
        if (y - x <= 2 * a.unit) continue;
        const Sum acc = sum_run<T, VEC>(a.dout, a.order, x > from ? x : from, y < to ? y : to, cols, a.dim);
        // a run that starts with the unit goes on through its start as well
        store_row<VEC>(a.part + (2 * c + (x > from)) * a.dim, cols, a.dim, acc);
    }
}

// One wave per (sorted token, slab): the first token of a run sums and writes its
// row, the others have nothing to do.
template <typename T, int VEC, bool ADD>
__global__ __launch_bounds__(256) void embed_rows(GradArgs a) {
    if ((int64_t)blockIdx.x < a.long_blocks) {
        sum_unit<T, VEC>(a);
        return;
    }
    const int64_t slabs = slabs_of(a.dim);
    const int64_t job = ((int64_t)blockIdx.x - a.long_blocks) * 4 + wave_id();
    const int32_t p = (int32_t)(job / slabs);
    if (p >= a.start[a.vocab]) return;
    const int32_t id = a.sorted[p];
    if (p > 0 && a.sorted[p - 1] == id) return;
    const int32_t end = a.start[id + 1];
    if (end - p > 2 * a.unit) return;  // long runs: embed_join
    const Columns cols = columns_of(job % slabs, a.dim);
    put_sum<VEC, ADD>(a.dtable + (int64_t)id * a.dim, cols, a.dim, a.scale,
                      sum_run<T, VEC>(a.dout, a.order, p, end, cols, a.dim));
}

// The rows of long runs, one wave per (unit, slab) in which such a run ends.
template <int VEC, bool ADD>
__global__ __launch_bounds__(256) void embed_join(GradArgs a) {
    const int64_t slabs = slabs_of(a.dim);
    const int64_t job = (int64_t)blockIdx.x * 4 + wave_id();
    const int64_t from = job / slabs * a.unit;
    const int32_t n = a.start[a.vocab];
    if (from >= n) return;
    const int32_t to = (int32_t)(from + a.unit < n ? from + a.unit : n);
    // the run at the unit's start is the only long one that can end in it
    const int32_t id = a.sorted[from];
    const int32_t x = a.start[id], y = a.start[id + 1];
    if (y - x <= 2 * a.unit || y > to) return;
    const Columns cols = columns_of(job % slabs, a.dim);
    const int64_t c1 = (y - 1) / a.unit;
    const Sum acc = sum_rows<float, VEC>(x / a.unit, c1 + 1, cols, a.dim, [&](int64_t c) {
        return a.part + (2 * c + (x > c * a.unit)) * a.dim;
    });
    put_sum<VEC, ADD>(a.dtable + (int64_t)id * a.dim, cols, a.dim, a.scale, acc);
}

size_t align256(size_t n) { return (n + 255) / 256 * 256; }

// Sorted tokens per unit of a long run: few enough units that one wave adds them
// up, and their sums stay small beside the rows that they come from. The backward with
// units of 16 / 32 / 64 / 128 / 256, us: 16384 tokens crowding at the start of 151936 x
// 1536 415 / 403 / 397 / 397 / 412, of 50257 x 893 307 / 291 / 289 / 295 / 308; 4096 tokens
// of one id of 32000 x 512 69 / 47 / 38 / 37 / 45, 16384 of 2048 x 512 201 / 115 / 77 / 58 /
// 55. Past 65536 tokens units grow: 262144 crowding at the start of 2048 x 256, in 256
// 703, in 128 736, in 32 1004.
int32_t unit_of(int64_t tokens) {
    const int64_t per = (tokens + 1023) / 1024;
    return (int32_t)(per <= 64 ? 64 : (per + 63) / 64 * 64);
}

}  // namespace

EmbeddingWs embedding_bwd_ws(const mc_embedding_desc& d) {
    EmbeddingWs w{};
    size_t off = 0;
    w.order = off;   off += align256((size_t)d.tokens * 4);
    w.sorted = off;  off += align256((size_t)d.tokens * 4);
    w.start = off;   off += align256(((size_t)d.vocab + 1) * 4);
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
    int32_t* sorted = reinterpret_cast<int32_t*>(ws + w.sorted);
    int32_t* start = reinterpret_cast<int32_t*>(ws + w.start);
    float* part = reinterpret_cast<float*>(ws + w.part);
    const int32_t unit = unit_of(d.tokens);
    const int64_t clear = accumulate ? 0 : d.vocab * d.dim;
    const int id_block = embedding_sort_ids(d.vocab);
    static_assert(embedding_sort_ids((int64_t)1 << 31) == kIds, "a workgroup's counts fit in LDS");
    const int sort_blocks = (int)((d.vocab + id_block - 1) / id_block);
    // the sort in as many waves as it takes, or in those that clear
    const bool together = embedding_sort_while_clearing(d.tokens, clear);
    const int threads = together ? 256 : 1024;
    const int64_t steps = (d.tokens + threads - 1) / threads;  // of a wave
    auto sort = [&](auto ahead) {
        constexpr int AHEAD = decltype(ahead)::value;
        const int64_t beside = together ? (clear + 1023) / 1024 : 0;
        const dim3 grid((unsigned)(sort_blocks + beside));
        if (together)
            embed_sort<4, AHEAD><<<grid, 256, 0, stream>>>(ids, (int32_t)d.tokens, d.vocab, d.padding_id, order, sorted,
                                                          start, id_block, sort_blocks, dtable, clear);
        else
            embed_sort<16, AHEAD><<<grid, 1024, 0, stream>>>(ids, (int32_t)d.tokens, d.vocab, d.padding_id, order, sorted,
                                                            start, id_block, sort_blocks, dtable, 0);
    };
    if (steps <= 2) sort(std::integral_constant<int, 2>{});
    else if (steps <= 4) sort(std::integral_constant<int, 4>{});
    else if (steps <= 8) sort(std::integral_constant<int, 8>{});
    else sort(std::integral_constant<int, 16>{});
    if (clear && !together)
        embed_clear<<<dim3((unsigned)((clear + 1023) / 1024)), 256, 0, stream>>>(dtable, clear);
    const int64_t slabs = slabs_of(d.dim), units = (d.tokens + unit - 1) / unit;
    GradArgs a{};
    a.dout = dout;
    a.order = order;
    a.sorted = sorted;
    a.start = start;
    a.part = part;
    a.dtable = dtable;
    a.vocab = d.vocab;
    a.dim = (int)d.dim;
    a.unit = unit;
    a.scale = d.scale;
    a.long_blocks = d.tokens > 2 * unit ? (units * slabs + 3) / 4 : 0;
    const dim3 grid((unsigned)(a.long_blocks + (d.tokens * slabs + 3) / 4));
    auto go = [&](auto elem, auto vec) {
        typedef decltype(elem) T;
        constexpr int VEC = decltype(vec)::value;
        if (accumulate) embed_rows<T, VEC, true><<<grid, 256, 0, stream>>>(a);
        else embed_rows<T, VEC, false><<<grid, 256, 0, stream>>>(a);
        if (a.long_blocks == 0) return;
        if (accumulate) embed_join<VEC, true><<<dim3((unsigned)a.long_blocks), 256, 0, stream>>>(a);
        else embed_join<VEC, false><<<dim3((unsigned)a.long_blocks), 256, 0, stream>>>(a);
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
