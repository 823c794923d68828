// Attention over rows that hold several documents, with capped scores and a bias
// by distance, gfx950.
//
//   x_ij = scale q_i . k_j
//   x_ij = cap tanh(x_ij / cap)                   (with a cap)
//   x_ij = x_ij - slope_h |i - j|                 (with slopes)
//   o_i  = sum over the keys j that i sees of softmax_j(x_ij) v_j,  0 if it sees none
//
// Every mask here (a causal row, a document of a packed row, a prompt that sees
// itself whole, padding) lets a query see an interval of keys and a key an
// interval of queries: attention_spans writes both per token once, and every
// layer's forward and backward reads them. A tile is then skipped, masked or
// taken whole by comparing four numbers.
//
// The kernels are shaped as the causal ones of attention.hip (the same tiles, LDS
// layouts and fragment orders, attention_tiles.hpp):
//
//  packed_vt    V^T for the forward of longer rows, as there; infinities and NaN are left out of
//               it and their blocks of keys noted, since p = 0 times one of them
//               would be NaN in every row of a tile that shares it. The forward
//               adds them afterwards to the rows that see them.
//  packed_fwd   one workgroup per (b, h, 128 queries).
//  packed_prep  Delta and lse per query; blocks of 64 noted whose Q or dO must be
//               cleared of infinities and NaN before hidden pairs meet them.
//  packed_dkdv  one workgroup per (b, K/V head, group of query heads, 128 keys);
//               stores dS^T of the queries that its keys meet, in blocks of 128.
//  packed_dq    dQ from the stored dS^T, one workgroup per (b, h, 128 queries);
//               past 2^31 bytes of one head's dS^T packed_dq_again forms S and dP
//               once more.
//
// Roundings to bf16, each for the matrix rate of bf16, sixteen times float32's: P before
// P.V and dV (its sum keeps it unrounded, so o is off by at most 2^-8 of sum P |v|), dS
// before dK and dQ, which reads it from memory. Sums, maxima, lse and Delta are float32.
// Of the size of a result that makes 2.4e-3 for dq and dk of random rows, where their
// own rounding is 1.7e-3, and up to 3.4e-3 with Delta from o (packed_prep).
//
// The cap. With r = 1 / (1 + 2^(2 log2 e x / cap)), tanh(x / cap) = 1 - 2 r and
// its slope is 4 (r - r^2): one exponential and one reciprocal more per score.
// tanh grows with x, so the running maximum stays one of unscaled products.
//
// What bounds them, with us per call: (a) 4 x 28 x 4096 x 128, capped, one causal
// document a row; (b) 8 x 12 x 2048 x 128 in documents of 345 tokens, a mean of 24 of
// the 40 blocks of 64 x 128 pairs per CU visible; (c) 3 x 14 x 1021 x 64 in documents
// of 156 tokens with prompts and a bias.
//               (a)    (b)   (c)
//  packed_spans        5.6   4.8   two scans of a row by one workgroup: latency
//  packed_vt    10     7.1   3.6   memory
//  packed_fwd   664    70    17    (a) 725 TFLOP/s: the scores' arithmetic, of whose
//                                  time the cap's exponential and reciprocal are half
//  packed_prep  52     44    14    (a) memory; (b, c) S and dP once more
//  packed_dkdv  1467   155   27    one wave per SIMD: MFMA 31% of its cycles, scores
//                                  37, waits 27, which follow each other (the scores
//                                  of one query tile among the other's MFMAs: 1800
//                                  and more, for what is moved between registers;
//                                  tiles three steps ahead, fragments two or three:
//                                  no change)
//  packed_dq    452    65    12    (a) memory: dS^T, 1.9 GB, at 4.2 TB/s
#include <algorithm>
#include <type_traits>

#include "attention_spans.hpp"
#include "attention_tiles.hpp"
#include "common.hpp"
#include "kernels.hpp"
#include "rules.hpp"

namespace mc {
namespace {

using namespace attn;

// ------------------------------------------------------------------ spans
// One workgroup per row of the batch. A document is a run of equal ids; ids below
// 0 are padding. Two scans over the row, kItems tokens per thread and turn: from
// the end, where each token's document ends, and the first token from it on that
// is no prompt; from the start, where each document begins and where its prompt
// ends. Latency is all there is (8 KB of ids at 2048 tokens), so a row of one
// turn stays in registers between the two.
constexpr int kScanThreads = 1024, kScanWaves = kScanThreads / kWave, kItems = 4;
constexpr int kScanTurn = kScanThreads * kItems;  // tokens per turn

// The latest mark (>= 0; -1: none) of the threads before this one (AFTER: the
// first of those behind it), or the carry where they have none; the carry becomes
// the last (first) of all. `slots` must not be the array of the call before.
template <bool AFTER>
__device__ __forceinline__ int nearest_mark(int mark, int& carry, int* slots) {
    const int lane = lane_id(), wave = wave_id();
    const uint64_t marked = __ballot(mark >= 0);
    const uint64_t there = AFTER ? marked >> lane >> 1 : marked & (((uint64_t)1 << lane) - 1);
    const int from = there == 0 ? lane : AFTER ? lane + 1 + __builtin_ctzll(there) : 63 - __builtin_clzll(there);
    const int near = __shfl(mark, from, kWave);
    // the mark of a wave that others see, and of each wave in lane w of 16
    auto outer = [](int v, uint64_t lanes, int none) {
        const int l = lanes == 0 ? 0 : AFTER ? __builtin_ctzll(lanes) : 63 - __builtin_clzll(lanes);
        const int x = __builtin_amdgcn_readlane(v, l);
        return lanes == 0 ? none : x;
    };
    if (lane == 0) slots[wave] = outer(mark, marked, -1);
    __syncthreads();
    const int of_wave = slots[lane % kScanWaves];
    const uint64_t waves = __ballot(of_wave >= 0) & ((1 << kScanWaves) - 1);
    const uint64_t beyond = AFTER ? waves >> wave >> 1 << wave << 1 : waves & (((uint64_t)1 << wave) - 1);
    const int other = outer(of_wave, beyond, carry);
    carry = outer(of_wave, waves, carry);
    return there == 0 ? other : near;
}

__global__ __launch_bounds__(kScanThreads) void packed_spans(const int32_t* __restrict__ documents,
                                                             const uint8_t* __restrict__ prefix, int S, int causal,
                                                             int4* __restrict__ spans) {
    __shared__ int slots[2][2][kScanWaves];
    const int64_t row = (int64_t)blockIdx.x * S;
    const int32_t* id = documents ? documents + row : nullptr;
    const uint8_t* pre = prefix ? prefix + row : nullptr;
    int4* out = spans + row;
    const int turns = (int)(((int64_t)S + kScanTurn - 1) / kScanTurn);
    // a token's id (0 without documents), t brought inside the row
    auto id_at = [&](int64_t t) { return id ? id[t < 0 ? 0 : t >= S ? S - 1 : t] : 0; };
    // this thread's tokens t0 .. t0 + kItems - 1 of a turn: ids[e + 1] is that of t0 + e
    int ids[kItems + 2], end[kItems], stop[kItems];
    int end_carry = S, stop_carry = S, k = 0;
    for (int turn = turns - 1; turn >= 0; --turn, ++k) {
        const int64_t t0 = (int64_t)turn * kScanTurn + (int64_t)threadIdx.x * kItems;
#pragma unroll
        for (int e = 0; e < kItems + 2; ++e) ids[e] = id_at(t0 + e - 1);
        int first_end = -1, first_stop = -1;
#pragma unroll
        for (int e = kItems - 1; e >= 0; --e) {
            const int64_t t = t0 + e;
            const bool in = t < S, marked = pre ? pre[in ? t : S - 1] != 0 : false;
            const bool last = t == S - 1 || ids[e + 1] != ids[e + 2];  // of its document
            end[e] = in && last ? (int)t + 1 : -1;
            stop[e] = in && !marked ? (int)t : end[e];
            first_end = end[e] >= 0 ? end[e] : first_end;
            first_stop = stop[e] >= 0 ? stop[e] : first_stop;
        }
        int end_in = nearest_mark<true>(first_end, end_carry, slots[k & 1][0]);
        int stop_in = pre ? nearest_mark<true>(first_stop, stop_carry, slots[k & 1][1]) : 0;
#pragma unroll
        for (int e = kItems - 1; e >= 0; --e) {
            end[e] = end_in = end[e] >= 0 ? end[e] : end_in;
            stop[e] = stop_in = stop[e] >= 0 ? stop[e] : stop_in;
            // a row of several turns keeps them in its spans; the same thread reads them again
            if (turns > 1 && t0 + e < S) out[t0 + e] = make_int4(0, end[e], stop[e], 0);
        }
    }
    int begin_carry = 0, prompt_carry = 0;
    for (int turn = 0; turn < turns; ++turn, ++k) {
        const int64_t t0 = (int64_t)turn * kScanTurn + (int64_t)threadIdx.x * kItems;
        if (turns > 1) {
#pragma unroll
            for (int e = 0; e < kItems + 2; ++e) ids[e] = id_at(t0 + e - 1);
#pragma unroll
            for (int e = 0; e < kItems; ++e) {
                const int4 x = t0 + e < S ? out[t0 + e] : make_int4(0, 0, 0, 0);
                end[e] = x.y;
                stop[e] = x.z;
            }
        }
        int begin[kItems], prompt[kItems], last_begin = -1, last_prompt = -1;
#pragma unroll
        for (int e = 0; e < kItems; ++e) {
            const int64_t t = t0 + e;
            const bool first = t < S && (t == 0 || ids[e] != ids[e + 1]);
            begin[e] = first ? (int)t : -1;
            prompt[e] = first ? stop[e] : -1;
            last_begin = first ? begin[e] : last_begin;
            last_prompt = first ? prompt[e] : last_prompt;
        }
        int begin_in = nearest_mark<false>(last_begin, begin_carry, slots[k & 1][0]);
        int prompt_in = pre ? nearest_mark<false>(last_prompt, prompt_carry, slots[k & 1][1]) : 0;
#pragma unroll
        for (int e = 0; e < kItems; ++e) {
            const int t = (int)(t0 + e < S ? t0 + e : S - 1);
            begin_in = begin[e] >= 0 ? begin[e] : begin_in;
            prompt_in = prompt[e] >= 0 ? prompt[e] : prompt_in;
            int4 x = make_int4(begin_in, end[e], begin_in, end[e]);
            if (causal) {
                x.y = prompt_in > t + 1 ? prompt_in : t + 1;
                x.z = t < prompt_in ? begin_in : t;
            }
            if (ids[e + 1] < 0) x = make_int4(0, 0, 0, 0);
            if (t0 + e < S) out[t] = x;
        }
    }
}

// Over the 32 tokens of a wave's lanes l and l ^ 32: the union of their spans
// [lo, hi) and what all of them see, [all_lo, all_hi) (nothing where one is empty).
struct WaveSpan {
    int lo, hi, all_lo, all_hi;
};
template <int CTRL>
__device__ __forceinline__ int dpp_int(int v) {
    return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xf, 0xf, false);
}
// The least (greatest) v of a wave half's 32 lanes, in every lane of it: within
// 16 lanes by DPP as in wave_sum, then the two rows of 16 change places.
template <bool GREATEST>
__device__ __forceinline__ int half_extreme(int v) {
    auto pick = [](int x, int y) { return GREATEST ? (x > y ? x : y) : (x < y ? x : y); };
    v = pick(v, dpp_int<0xB1>(v));   // quad_perm [1,0,3,2]
    v = pick(v, dpp_int<0x4E>(v));   // quad_perm [2,3,0,1]
    v = pick(v, dpp_int<0x141>(v));  // row_half_mirror
    v = pick(v, dpp_int<0x140>(v));  // row_mirror
    const auto r = __builtin_amdgcn_permlane16_swap((unsigned)v, (unsigned)v, false, false);
    return pick((int)r[0], (int)r[1]);
}
__device__ __forceinline__ WaveSpan wave_span(Span s) {
    return WaveSpan{__builtin_amdgcn_readfirstlane(half_extreme<false>(s.lo < s.hi ? s.lo : 0x7fffffff)),
                    __builtin_amdgcn_readfirstlane(half_extreme<true>(s.hi)),
                    __builtin_amdgcn_readfirstlane(half_extreme<true>(s.lo)),
                    __builtin_amdgcn_readfirstlane(half_extreme<false>(s.hi))};
}
// The union over the workgroup's four waves, as [lo, hi), empty as [0, 0).
__device__ __forceinline__ Span workgroup_span(const WaveSpan& w, int (*slots)[2]) {
    if (lane_id() == 0) {
        slots[wave_id()][0] = w.lo;
        slots[wave_id()][1] = w.hi;
    }
    __syncthreads();
    int lo = slots[0][0], hi = slots[0][1];
#pragma unroll
    for (int i = 1; i < 4; ++i) {
        lo = slots[i][0] < lo ? slots[i][0] : lo;
        hi = slots[i][1] > hi ? slots[i][1] : hi;
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    hi = __builtin_amdgcn_readfirstlane(hi);
    return lo < hi ? Span{lo, hi} : Span{0, 0};
}

__device__ __forceinline__ bool nonfinite16(uint32_t h) { return (h & 0x7f80u) == 0x7f80u; }
// Any infinity or NaN among the pairs of bf16 of q.
__device__ __forceinline__ bool any_nonfinite(const uint4& q) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
    bool bad = false;
#pragma unroll
    for (int e = 0; e < 4; ++e) bad |= (w[e] & 0x7f80u) == 0x7f80u || (w[e] & 0x7f800000u) == 0x7f800000u;
    return bad;
}
__device__ __forceinline__ uint32_t clear_nonfinite(uint32_t w) {
    if ((w & 0x7f80u) == 0x7f80u) w &= 0xffff0000u;
    if ((w & 0x7f800000u) == 0x7f800000u) w &= 0x0000ffffu;
    return w;
}
// Clears the infinities and NaN of a tile of `elems` bf16 in LDS; every thread of
// the workgroup takes part.
__device__ __forceinline__ bool clear_tile(uint16_t* tile, int elems) {
    bool found = false;
    for (int i = threadIdx.x; i < elems / 8; i += 256) {
        uint4* p = reinterpret_cast<uint4*>(tile) + i;
        uint4 q = *p;
        if (any_nonfinite(q)) {
            q.x = clear_nonfinite(q.x); q.y = clear_nonfinite(q.y);
            q.z = clear_nonfinite(q.z); q.w = clear_nonfinite(q.w);
            *p = q;
            found = true;
        }
    }
    return found;
}
// Any flag of [from, to) set: the same in every lane of a wave.
__device__ __forceinline__ bool any_flag(const int32_t* flags, int from, int to) {
    bool bad = false;
    for (int i = from + lane_id(); i < to; i += kWave) bad |= flags[i] != 0;
    return __any(bad);
}

// take(dt, j, value) for the infinities and NaN of rows [from, to) of x [S][D] that this
// lane's query sees, at its accumulators j of tile dt (dim 32 dt + 8 (j/4) + 4 half + j%4).
template <int D, typename F>
__device__ __forceinline__ void each_nonfinite(const uint16_t* x, int from, int to, Span sees, int half, F&& take) {
#pragma unroll 1
    for (int key = from; key < to; ++key) {
        if (key < sees.lo || key >= sees.hi) continue;
        const uint16_t* row = x + (int64_t)key * D + 4 * half;
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
            for (int jq = 0; jq < 4; ++jq) {
                const uint2 w = *reinterpret_cast<const uint2*>(row + 32 * dt + 8 * jq);
                const uint32_t e[4] = {w.x & 0xffffu, w.x >> 16, w.y & 0xffffu, w.y >> 16};
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    if (nonfinite16(e[u])) take(dt, 4 * jq + u, __uint_as_float(e[u] << 16));
            }
    }
}

struct PackedArgs {
    const uint16_t* q;     // [B, H, S, D]
    const uint16_t* k;     // [B, Hkv, S, D]
    const uint16_t* v;     // [B, Hkv, S, D]
    const uint16_t* vt;    // forward: [B, Hkv, D, Sp]
    const uint16_t* dout;  // [B, S, H, D]
    const int4* spans;     // [B, S], or null
    const float* slopes;   // [H], or null
    uint16_t* o;           // forward: [B, S, H, D]
    float* lse;            // [B, H, S], or null
    const float* lsd;      // backward: [B, H, Sp / 64, 2, 64]: lse * log2 e, Delta
    int32_t* vflags;       // forward: [B, Hkv, Sp / 64], blocks of V with infinities or NaN
    const int32_t* qflags; // backward: [B, H, Sp / 64], blocks of Q and dO
    int4* kinfo;           // backward: [B, Hkv, nblk], blocks of 128 rows of K: whether they hold infinities
                           // or NaN, and the blocks of 128 queries [y, z) whose dS^T is stored
    uint16_t *dq, *dk, *dv;
    float *dk_part, *dv_part;  // [B, Hkv, ngroups, S, D]
    uint16_t* dst;             // dS^T: [B, H] of head_ds bytes (kDsBlock), or null
    int64_t head_ds, dq_blocks, sum_n8;
    int64_t S, Sp;
    int ngroups, B, H, Hkv, D, nblk, causal;
    float scale;       // of dq and dk (with a cap 4 times the scores')
    float scale_log2;  // scores to log2 units, without a cap
    float cap_in;      // 2 log2 e scale / cap
    float cap_log2;    // cap log2 e
};

// dS^T in memory, in the order in which the dK/dV waves hold it, so that each of their
// stores and each of the dQ pass's loads is 1 KB in a row (as key rows of queries a
// store was 64 pieces of 8 bytes, and a seventh of the kernel's time): per head blocks
// of 32 keys x 64 queries, in a block 16-query steps 2 t + kk, in a step lane (half,
// key), in a lane the 8 queries from 8 half on. The blocks of 128 queries, which one
// dQ workgroup reads, follow each other by keys (all queries of 32 keys together:
// strides of a power of two between its reads, 472 us in place of 452).
constexpr int kDsBlock = 32 * 64 * 2;  // bytes
__device__ __forceinline__ uint32_t ds_block(int q64, int k32, int nblk) {
    return ((uint32_t)((q64 >> 1) * 4 * nblk + k32) * 2u + (uint32_t)(q64 & 1)) * kDsBlock;
}
__host__ __device__ inline int64_t head_ds_bytes(int64_t S) {
    const int64_t nblk = (S + 127) / 128;
    return 4 * nblk * 2 * nblk * kDsBlock;
}

// Scores in log2 units from a product s.
template <bool CAP>
__device__ __forceinline__ float score_log2(float s, const PackedArgs& a) {
    if constexpr (!CAP) return s * a.scale_log2;
    const float r = __builtin_amdgcn_rcpf(1.f + exp2_hw(s * a.cap_in));  // (1 - tanh) / 2
    return __builtin_fmaf(r, -2.f * a.cap_log2, a.cap_log2);
}

// ------------------------------------------------------------ V^T prepass
// As attn_vt_bf16, with infinities and NaN left out and their blocks noted.
template <int D>
__global__ __launch_bounds__(256) void packed_vt(const uint16_t* __restrict__ V, int64_t S, int64_t Sp,
                                                 uint16_t* __restrict__ Vt, int32_t* __restrict__ flags) {
    constexpr int CPR = D / 8;
    __shared__ __attribute__((aligned(16))) uint16_t tile[64][D + 8];
    const int64_t bh = blockIdx.y;
    const int64_t k0 = (int64_t)blockIdx.x * 64;
    const __amdgpu_buffer_rsrc_t rv = make_rsrc(V + bh * S * D, S * D * 2);
    bool bad = false;
    for (int i = threadIdx.x; i < 64 * CPR; i += 256) {
        const int key = i / CPR, c = i % CPR;
        const uint32_t off = k0 + key < S ? (uint32_t)(((k0 + key) * D + 8 * c) * 2) : kOOB;
        uint4 v = __builtin_bit_cast(uint4, buf_load16(rv, off));
        if (any_nonfinite(v)) {
            bad = true;
            v.x = clear_nonfinite(v.x); v.y = clear_nonfinite(v.y);
            v.z = clear_nonfinite(v.z); v.w = clear_nonfinite(v.w);
        }
        *reinterpret_cast<uint4*>(&tile[key][8 * c]) = v;
    }
    bad = __syncthreads_or(bad);
    if (threadIdx.x == 0) flags[bh * (Sp / 64) + blockIdx.x] = bad;
    uint16_t* dst = Vt + bh * D * Sp + k0;
    for (int i = threadIdx.x; i < D * 8; i += 256) {
        const int d = i >> 3, c = i & 7;
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int p0 = 8 * c + 2 * e, p1 = p0 + 1;
            const int key0 = (p0 & ~15) | perm16(p0 & 15), key1 = (p1 & ~15) | perm16(p1 & 15);
            w[e] = (uint32_t)tile[key0][d] | ((uint32_t)tile[key1][d] << 16);
        }
        *reinterpret_cast<uint4*>(dst + (int64_t)d * Sp + 8 * c) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// ------------------------------------------------------- flash forward
// ROWS: V as it is, through transposed reads, cleared of infinities and NaN block by
// block in LDS; otherwise V^T from packed_vt.
template <int D, bool CAP, bool BIAS, bool ROWS>
__global__ __launch_bounds__(256, 2) void packed_fwd(PackedArgs a) {
    constexpr int KB = 64;            // keys per block
    constexpr int QB = 128;           // queries per workgroup, 32 per wave
    constexpr int KS = D / 16;        // MFMA k-steps over the head dim
    constexpr int DT = D / 32;        // 32-row tiles of O^T
    constexpr int K_ELEMS = KB * D;   // K tile [64][D], rows of D bf16
    constexpr int STAGE = 2 * KB * D; // K tile, then V^T tile [D][64] (ROWS: V [64][D])
    constexpr int CPR_K = D / 8, RPI_K = 64 / CPR_K;
    constexpr int LOADS_K = KB / RPI_K / 4, LOADS_V = D / 8 / 4;  // DMA per wave per block
    __shared__ __attribute__((aligned(1024))) uint16_t smem[2 * STAGE];
    __shared__ int slots[4][2];
    const uint32_t smem_byte = (uint32_t)reinterpret_cast<uintptr_t>(smem);

    const int lane = threadIdx.x & 63, wave = wave_id();
    const int col = lane & 31, half = lane >> 5;
    const int nbh = a.B * a.H;
    const int qb = a.nblk - 1 - (int)(blockIdx.x / nbh);  // heaviest (causal) query blocks first
    const int bh = xcd_head_order((int)(blockIdx.x % nbh), nbh);
    const int b = bh / a.H, h = bh % a.H;
    const int hk = h / (a.H / a.Hkv);
    const int64_t S = a.S;
    const int64_t q0 = (int64_t)qb * QB;
    const int64_t qw = q0 + 32 * wave;  // first query of this wave
    const int64_t my_q = qw + col;

    // Q^T fragments (B operand of S^T = K.Q^T): query my_q, dims 16 s + 8 half .. +7.
    const __amdgpu_buffer_rsrc_t rq = make_rsrc(a.q + (int64_t)bh * S * D, S * D * 2);
    bf16x8 qf[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
        const uint32_t off = my_q < S ? (uint32_t)((my_q * D + 16 * s + 8 * half) * 2) : kOOB;
        qf[s] = __builtin_bit_cast(bf16x8, buf_load16(rq, off));
    }

    const int64_t bhk = (int64_t)b * a.Hkv + hk;
    const i32x4 rk = rsrc_words(a.k + bhk * S * D, S * D * 2);
    const i32x4 rv = ROWS ? rsrc_words(a.v + bhk * S * D, S * D * 2)
                          : rsrc_words(a.vt + bhk * D * a.Sp, (int64_t)D * a.Sp * 2);
    uint32_t troff[DT][2];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) troff[dt][hh] = ROWS ? tr_off<D>(lane, 32 * dt, hh) : 0;

    // K rows key0 .. key0+63 into the swizzled [64][D] layout, then V^T rows
    // d = 0 .. D-1 (64 positions each) into [D][64].
    auto issue = [&](int kb, int stage) {
        const uint32_t base = smem_byte + (uint32_t)(stage * STAGE * 2);
        const uint32_t key0 = (uint32_t)kb * KB;
#pragma unroll
        for (int j = 0; j < LOADS_K; ++j) {
            const int blk = wave * LOADS_K + j;
            const int row = blk * RPI_K + lane / CPR_K;
            const uint32_t chunk = (uint32_t)swz<D>(row, lane % CPR_K);
            const uint32_t off = ((key0 + (uint32_t)row) * D + 8u * chunk) * 2u;
            dma16(rk, __builtin_amdgcn_readfirstlane(base + (uint32_t)blk * 1024u), off);
        }
        if constexpr (ROWS) {
            dma_rows<D>(rv, base + K_ELEMS * 2, key0, D, wave, lane);
        } else {
#pragma unroll
            for (int j = 0; j < LOADS_V; ++j) {
                const int blk = wave * LOADS_V + j;
                const int row = blk * 8 + lane / 8;
                const uint32_t chunk = (uint32_t)swz<64>(row, lane % 8);
                const uint32_t off = ((uint32_t)row * (uint32_t)a.Sp + key0 + 8u * chunk) * 2u;
                dma16(rv, __builtin_amdgcn_readfirstlane(base + (uint32_t)(K_ELEMS * 2) + (uint32_t)blk * 1024u), off);
            }
        }
    };

    // Block kd holds this tile's own tokens, which see themselves: its rows are on
    // the way while the spans are read. The others follow in order.
    const int kd = 2 * qb;
    issue(kd, 0);
    // what this lane's query sees, and with it the wave's and the workgroup's blocks of keys
    const Span mine = query_span(a.spans, b, my_q, (int)S, a.causal);
    const WaveSpan ws = wave_span(mine);
    const Span wg = workgroup_span(ws, slots);
    const int kb0 = wg.lo / KB, kb1 = (wg.hi + KB - 1) / KB;
    const int wk0 = ws.lo < ws.hi ? ws.lo / KB : 0, wk1 = ws.lo < ws.hi ? (ws.hi + KB - 1) / KB : 0;
    bool bad_v = ROWS ? false : any_flag(a.vflags + bhk * (a.Sp / 64), wk0, wk1);
    const float slope2 = BIAS ? a.slopes[h] * kLog2e : 0.f;

    f32x16 oacc[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int j = 0; j < 16; ++j) oacc[t][j] = 0.f;
    float m_run = kNegInf, l_run = 0.f;

    int kb = kd, next = 0, stage = 0;
    for (bool more = kb0 < kb1; more; kb = next, stage ^= 1) {
        next = kb == kd ? kb0 : kb + 1;
        next += next == kd;
        more = next < kb1;
        wait_vmcnt<0>();
        __syncthreads();
        if (more) issue(next, stage ^ 1);
        if constexpr (ROWS) bad_v |= __syncthreads_or(clear_tile(smem + stage * STAGE + K_ELEMS, K_ELEMS)) != 0;
        if (kb < wk0 || kb >= wk1) continue;  // wave-uniform: no query of this wave sees the block
        const uint16_t* sk = smem + stage * STAGE;
        const uint16_t* sv = sk + K_ELEMS;

        // S^T tiles t = 0, 1 (keys 32 t .. 32 t + 31) x the wave's 32 queries,
        // K fragments one k-step ahead of their MFMAs
        f32x16 sacc[2];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int j = 0; j < 16; ++j) sacc[t][j] = 0.f;
        bf16x8 kf[2][2];
        auto kread = [&](int s, int slot) {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int row = 32 * t + col;
                kf[slot][t] = *reinterpret_cast<const bf16x8*>(&sk[row * D + 8 * swz<D>(row, 2 * s + half)]);
            }
        };
        kread(0, 0);
        __builtin_amdgcn_sched_group_barrier(kSchedDsRead, 2, 0);
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            if (s + 1 < KS) {
                kread(s + 1, (s + 1) & 1);
                __builtin_amdgcn_sched_group_barrier(kSchedDsRead, 2, 0);
            }
#pragma unroll
            for (int t = 0; t < 2; ++t)
                sacc[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[s & 1][t], qf[s], sacc[t], 0, 0, 0);
            __builtin_amdgcn_sched_group_barrier(kSchedMfma, 2, 0);
        }

        // Accumulator j of tile t is key key0 + 32 t + 8 (j/4) + 4 half + j%4.
        // Without a bias x stays a product until the exponent's fma, since the
        // largest product is the largest score: its score is formed once.
        const int key0 = kb * KB;
        float x[2][16];
        const float dist = (float)((int)my_q - key0 - 4 * half);
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                x[t][j] = BIAS ? score_log2<CAP>(sacc[t][j], a) : sacc[t][j];
                if constexpr (BIAS)
                    x[t][j] = __builtin_fmaf(__builtin_fabsf(dist - (float)(32 * t + 8 * (j >> 2) + (j & 3))), -slope2,
                                             x[t][j]);
            }
        // key offsets in the block against this lane's span; its 4 half moves to
        // the bound, so each test is one subtraction and one unsigned comparison
        const bool edge = !(key0 >= ws.all_lo && key0 + KB <= ws.all_hi);
        const int lo = mine.lo - key0 - 4 * half;
        const uint32_t width = (uint32_t)(mine.hi - mine.lo);
        if (edge) {
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    if ((uint32_t)(32 * t + 8 * (j >> 2) + (j & 3) - lo) >= width) x[t][j] = kNegInf;
        }

        // online softmax over this block's 64 keys (32 here, 32 in lane ^ 32);
        // the reference point moves when the maximum passes it by kMaxSlack
        float mx = x[0][0];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int j = 0; j < 16; ++j) mx = fmaxf(mx, x[t][j]);
        mx = half_pair_max(mx);
        if constexpr (!BIAS) mx = mx == kNegInf ? mx : score_log2<CAP>(mx, a);  // scale > 0
        float alpha = 1.f;
        if (mx > m_run + kMaxSlack) {
            alpha = exp2_hw(m_run - mx);  // m_run = -inf: 0 (O and l are 0 then)
            m_run = mx;
        }
        const float m_use = m_run == kNegInf ? 0.f : m_run;  // a row with no key yet keeps p = 0
        if constexpr (CAP && !BIAS) {
            // x -> r = (1 - tanh) / 2; a hidden score's is +inf, not that of -inf
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int j = 0; j < 16; ++j) x[t][j] = __builtin_amdgcn_rcpf(1.f + exp2_hw(x[t][j] * a.cap_in));
            if (edge) {
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        if ((uint32_t)(32 * t + 8 * (j >> 2) + (j & 3) - lo) >= width) x[t][j] = __builtin_inff();
            }
        }
        const float mul = CAP ? -2.f * a.cap_log2 : a.scale_log2, add = (CAP ? a.cap_log2 : 0.f) - m_use;
        float ps = 0.f;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                x[t][j] = exp2_hw(BIAS ? x[t][j] - m_use : __builtin_fmaf(x[t][j], mul, add));
                ps += x[t][j];
            }
        l_run = l_run * alpha + ps;
        if (__any(alpha != 1.f)) {
#pragma unroll
            for (int t = 0; t < DT; ++t)
#pragma unroll
                for (int j = 0; j < 16; ++j) oacc[t][j] *= alpha;
        }

        // P^T fragments: k-step (t, kk) takes accumulators 8 kk .. 8 kk + 7 of
        // tile t, i.e. keys 32 t + 16 kk + perm16(8 half + e), e = 0..7.
        bf16x8 pf[2][2];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) pf[t][kk] = pack_bf16x8(&x[t][8 * kk]);

        // O^T (d x query) += V^T . P^T, V^T fragments one step ahead
        bf16x8 vf[2][2];
        auto vread = [&](int v, int slot) {
            const int row = 32 * (v >> 1) + col, t = v & 1;
#pragma unroll
            for (int kk = 0; kk < 2; ++kk)
                if constexpr (ROWS)
                    vf[slot][kk] = frag_tr_at(sv + (32 * t + 16 * kk) * D, troff[v >> 1][0], troff[v >> 1][1]);
                else
                    vf[slot][kk] = *reinterpret_cast<const bf16x8*>(&sv[row * KB + 8 * swz<64>(row, 4 * t + 2 * kk + half)]);
        };
        constexpr int kReads = ROWS ? 4 : 2;
        vread(0, 0);
        __builtin_amdgcn_sched_group_barrier(kSchedDsRead, kReads, 0);
#pragma unroll
        for (int v = 0; v < 2 * DT; ++v) {
            if (v + 1 < 2 * DT) {
                vread(v + 1, (v + 1) & 1);
                __builtin_amdgcn_sched_group_barrier(kSchedDsRead, kReads, 0);
            }
            const int dt = v >> 1, t = v & 1;
#pragma unroll
            for (int kk = 0; kk < 2; ++kk)
                oacc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[v & 1][kk], pf[t][kk], oacc[dt], 0, 0, 0);
            __builtin_amdgcn_sched_group_barrier(kSchedMfma, 2, 0);
        }
    }

    // the infinities and NaN that V^T left out, for the rows that see their keys
    if (bad_v) {
#pragma unroll 1
        for (int kb = wk0; kb < wk1; ++kb) {
            if (!ROWS && a.vflags[bhk * (a.Sp / 64) + kb] == 0) continue;
            each_nonfinite<D>(a.v + bhk * S * D, kb * KB, (kb + 1) * KB < (int)S ? (kb + 1) * KB : (int)S, mine, half,
                              [&](int dt, int j, float v) { oacc[dt][j] += v; });
        }
    }

    // a row that sees nothing: o = 0, lse = -inf
    const float l_tot = l_run + __shfl_xor(l_run, 32, kWave);
    const bool sees = mine.lo < mine.hi;
    const float inv = sees ? 1.f / l_tot : 0.f;
    float lse = l_tot > 0.f ? (m_run + __log2f(l_tot)) * kLn2 : __builtin_nanf("");
    if constexpr (CAP) {
        // an infinite score is finite under a cap; the backward clears such a row's Q by its lse
        bool bad = false;
#pragma unroll
        for (int s = 0; s < KS; ++s) bad |= any_nonfinite(__builtin_bit_cast(uint4, qf[s]));
        if (__shfl_xor((int)bad, 32, kWave) || bad) lse = __builtin_nanf("");
    }
    if (a.lse && half == 0 && my_q < S) a.lse[(int64_t)bh * S + my_q] = sees ? lse : kNegInf;

    // O^T accumulator j of tile dt is dim 32 dt + 8 (j/4) + 4 half + j%4 of
    // query my_q: through a per-wave LDS patch to 16-byte row stores
    wait_vmcnt<0>();  // the first DMA has landed also when the loop ran no block
    __syncthreads();
    static_assert(4 * 32 * (D + 8) <= 2 * STAGE, "the patches fit in the stages");
    store_rows<D, uint16_t>(oacc, inv, smem + wave * 32 * (D + 8), a.o + ((int64_t)b * S * a.H + h) * D,
                            (int64_t)a.H * D, qw, S, lane);
}

// --------------------------------------------------------- backward prep
// Per (b, h, 128 queries): Delta and lse * log2 e into a [2][64] fp32 block per 64
// queries, and whether the block's Q or dO may hold infinities or NaN: dO does, or
// a row's lse is not finite (its Q or a key that it sees holds one, or it sees
// nothing and may hold anything). A row that sees nothing gets lse = +inf, which
// makes its P 0; one whose dO is not finite NaN, which reaches every gradient that
// depends on it.
//
// Delta_i = sum_d dO_id O_id carries o's rounding and that of P (bf16 both), which
// dS = P (dP - Delta) does not average away where few keys share it: dq and dk of
// 4 causal tokens were 6e-2 of their size off, of 30 9e-3, of 1021 4.9e-3, of 4096
// 3.6e-3 (their own roundings and dS's to bf16 make 2.4e-3). A query that sees at most
// kExactKeys keys has it as sum_j P_ij dP_ij instead, over sum_j P_ij, which is 1 but
// for lse's rounding (dS of the only key that a query sees is 0): S^T = K.Q^T and
// dP^T = V.dO^T once more, shaped as the forward, over the keys of such queries. With
// 64 / 128 / 256 / 512 / 1024 keys the backward of 8 x 12 x 2048 x 128 in documents of
// 340 takes 222 / 223 / 228 / 241 / 241 us, and dq and dk of a row are 2.36 / 2.35 / 2.35 /
// 2.34 / 2.34e-3 off; in documents of 64 to 1024, 3.0 / 2.6 / 2.4e-3 with 256 / 512 / 1024.
// Formed so for every query of 4 x 28 x 4096 x 128, a call takes 24% longer.
constexpr int kExactKeys = 256;
template <int D, bool CAP, bool BIAS>
__global__ __launch_bounds__(256, 2) void packed_prep(PackedArgs a, const uint16_t* __restrict__ o,
                                                      const float* __restrict__ lse, float* __restrict__ lsd,
                                                      int32_t* __restrict__ flags) {
    constexpr int KB = 64, QB = 128, KS = D / 16;
    constexpr int TILE = 64 * D, STAGE = 2 * TILE;  // K, V [64][D]
    __shared__ __attribute__((aligned(1024))) uint16_t smem[2 * STAGE];
    __shared__ int slots[4][2];
    __shared__ int noted[4];
    const uint32_t smem_byte = (uint32_t)reinterpret_cast<uintptr_t>(smem);
    const int lane = threadIdx.x & 63, wave = wave_id();
    const int col = lane & 31, half = lane >> 5;
    const int nbh = a.B * a.H;
    const int qb = (int)(blockIdx.x / nbh);
    const int bh = xcd_head_order((int)(blockIdx.x % nbh), nbh);
    const int b = bh / a.H, h = bh % a.H;
    const int64_t bhk = (int64_t)b * a.Hkv + h / (a.H / a.Hkv);
    const int64_t S = a.S;
    const int64_t qw = (int64_t)qb * QB + 32 * wave;
    const int64_t my_q = qw + col;

    // dO^T fragments (B operand of dP^T = V.dO^T): query my_q, dims 16 s + 8 half .. +7
    const int64_t ldo = (int64_t)a.H * D;
    const __amdgpu_buffer_rsrc_t rdo = make_rsrc(a.dout + ((int64_t)b * S * a.H + h) * D, (S * a.H - h) * D * 2);
    bf16x8 gf[KS];
    bool bad = false;
#pragma unroll
    for (int s = 0; s < KS; ++s)
        gf[s] = __builtin_bit_cast(
            bf16x8, buf_load16(rdo, my_q < S ? (uint32_t)((my_q * ldo + 16 * s + 8 * half) * 2) : kOOB));
    const float x = my_q < S ? lse[(int64_t)bh * S + my_q] : kNegInf;
    const i32x4 rk = rsrc_words(a.k + bhk * S * D, S * D * 2);
    const i32x4 rv = rsrc_words(a.v + bhk * S * D, S * D * 2);
    auto issue = [&](int kb, int stage) {
        const uint32_t base = smem_byte + (uint32_t)(stage * STAGE * 2);
        dma_rows<D>(rk, base, (uint32_t)kb * KB, D, wave, lane);
        dma_rows<D>(rv, base + TILE * 2, (uint32_t)kb * KB, D, wave, lane);
    };
    // the keys of a query that sees few, and with them the wave's and the workgroup's
    const Span all = query_span(a.spans, b, my_q, (int)S, a.causal);
    const bool few = all.hi - all.lo <= kExactKeys;
    const Span mine = few ? all : Span{0, 0};
    const WaveSpan ws = wave_span(mine);
    const Span wg = workgroup_span(ws, slots);
#pragma unroll
    for (int s = 0; s < KS; ++s) bad |= any_nonfinite(__builtin_bit_cast(uint4, gf[s]));
    bad |= __shfl_xor((int)bad, 32, kWave) != 0;
    const bool empty = x == kNegInf;
    const float lse2 = empty ? __builtin_inff() : bad ? __builtin_nanf("") : x * kLog2e;
    const bool note = __any(my_q < S && (bad || !(__builtin_fabsf(x) < __builtin_inff())));

    float from_o = 0.f, delta = 0.f, sum_p = 0.f;
    if (__any(!few)) {
        const __amdgpu_buffer_rsrc_t ro = make_rsrc(o + ((int64_t)b * S * a.H + h) * D, (S * a.H - h) * D * 2);
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            float u[8], g[8];
            BVec<uint16_t>::unpack(
                buf_load16(ro, my_q < S ? (uint32_t)((my_q * ldo + 16 * s + 8 * half) * 2) : kOOB), u);
            BVec<uint16_t>::unpack(__builtin_bit_cast(i32x4, gf[s]), g);
#pragma unroll
            for (int e = 0; e < 8; ++e) from_o = __builtin_fmaf(u[e], g[e], from_o);
        }
        from_o += __shfl_xor(from_o, 32, kWave);
    }
    if (wg.lo < wg.hi) {  // alike in every wave
        const __amdgpu_buffer_rsrc_t rq = make_rsrc(a.q + (int64_t)bh * S * D, S * D * 2);
        bf16x8 qf[KS];
#pragma unroll
        for (int s = 0; s < KS; ++s)
            qf[s] = __builtin_bit_cast(
                bf16x8, buf_load16(rq, my_q < S ? (uint32_t)((my_q * D + 16 * s + 8 * half) * 2) : kOOB));
        const float slope2 = BIAS ? a.slopes[h] * kLog2e : 0.f;
        uint32_t roff[KS];
#pragma unroll
        for (int s = 0; s < KS; ++s) roff[s] = rows_off<D>(lane, 2 * s + half);
        const int kb0 = wg.lo / KB, kb1 = (wg.hi + KB - 1) / KB;
        issue(kb0, 0);
        for (int kb = kb0; kb < kb1; ++kb) {
            wait_vmcnt<0>();
            __syncthreads();
            if (kb + 1 < kb1) issue(kb + 1, (kb + 1 - kb0) & 1);
            const int key0 = kb * KB;
            if (key0 >= ws.hi || key0 + KB <= ws.lo) continue;  // wave-uniform: no query of this wave sees the block
            const uint16_t* sk = smem + ((kb - kb0) & 1) * STAGE;
            const uint16_t* sv = sk + TILE;
            const bool edge = !(key0 >= ws.all_lo && key0 + KB <= ws.all_hi);
            const float dist = (float)((int)my_q - key0 - 4 * half);
            const int lo = mine.lo - key0 - 4 * half;
            const uint32_t width = (uint32_t)(mine.hi - mine.lo);
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                f32x16 sacc, dpacc;  // products, then P and P dP
#pragma unroll
                for (int j = 0; j < 16; ++j) sacc[j] = dpacc[j] = 0.f;
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    sacc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag_at(sk + 32 * t * D, roff[s]), qf[s], sacc, 0, 0, 0);
                    dpacc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag_at(sv + 32 * t * D, roff[s]), gf[s], dpacc, 0, 0, 0);
                }
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const int ko = 32 * t + 8 * (j >> 2) + (j & 3);
                    float y = score_log2<CAP>(sacc[j], a);
                    if constexpr (BIAS) y = __builtin_fmaf(__builtin_fabsf(dist - (float)ko), -slope2, y);
                    sacc[j] = exp2_hw(y - lse2);
                    dpacc[j] *= sacc[j];
                }
                if (edge) {
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        if ((uint32_t)(32 * t + 8 * (j >> 2) + (j & 3) - lo) >= width) sacc[j] = dpacc[j] = 0.f;
                }
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    sum_p += sacc[j];
                    delta += dpacc[j];
                }
            }
        }
        wait_vmcnt<0>();
    }
    delta += __shfl_xor(delta, 32, kWave);
    sum_p += __shfl_xor(sum_p, 32, kWave);
    if (sum_p > 0.f) delta /= sum_p;
    if (!few) delta = from_o;
    // queries past S have lse = +inf too
    if (half == 0 && my_q < a.Sp) {
        float* blk = lsd + ((int64_t)bh * (a.Sp / 64) + my_q / 64) * 128 + my_q % 64;
        blk[0] = lse2;
        blk[64] = empty ? 0.f : delta;
    }
    if (lane == 0) noted[wave] = note;
    __syncthreads();
    const int64_t blk = (int64_t)qb * 2 + threadIdx.x;
    if (threadIdx.x < 2 && blk < a.Sp / 64)
        flags[(int64_t)bh * (a.Sp / 64) + blk] = noted[2 * threadIdx.x] | noted[2 * threadIdx.x + 1];
}

// ------------------------------------------------------------ dK and dV
template <int D, bool CAP, bool BIAS>
__global__ __launch_bounds__(256, 1) void packed_dkdv(PackedArgs a) {
    constexpr int KS = D / 16, DT = D / 32;
    constexpr int TILE = 64 * D;                 // one [64][D] tile
    constexpr int STAGE = 2 * TILE + 512;        // Q, dO, lse/Delta (1 KB)
    constexpr int kDsStores = 4;                 // of dS^T per step and wave
    constexpr int KV = 2 * 128 * D;              // the workgroup's K and V rows, [128][D] each, after the stages
    constexpr int PATCH = 4 * 32 * (D + 8) * 2;  // the epilogue's, over the stages
    constexpr int SMEM = 2 * STAGE + KV > PATCH ? 2 * STAGE + KV : PATCH;
    __shared__ __attribute__((aligned(1024))) uint16_t smem[SMEM];
    __shared__ int slots[4][2];
    const uint32_t smem_byte = (uint32_t)reinterpret_cast<uintptr_t>(smem);
    const int lane = threadIdx.x & 63, wave = wave_id();
    const int col = lane & 31, half = lane >> 5;
    const int ng = a.ngroups;
    const int nwg = a.B * a.Hkv * ng;
    const int kb = (int)(blockIdx.x / nwg);      // key block 0 meets the most queries of a causal row: dispatched first
    const int grp = (int)(blockIdx.x % nwg) % ng;
    const int64_t bhk = (int64_t)(blockIdx.x % nwg) / ng;  // b * Hkv + K/V head
    const int b = (int)(bhk / a.Hkv);
    const int rep = a.H / a.Hkv, hpg = rep / ng;
    const int h0 = (int)(bhk % a.Hkv) * rep + grp * hpg;  // the group's first query head
    const int64_t S = a.S;
    const int64_t key0 = (int64_t)kb * 128;
    const int64_t kw = key0 + 32 * wave;         // first key of this wave
    const int64_t my_key = kw + col;
    uint32_t roff[KS], troff[DT][2];
#pragma unroll
    for (int s = 0; s < KS; ++s) roff[s] = rows_off<D>(lane, 2 * s + half);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int h = 0; h < 2; ++h) troff[dt][h] = tr_off<D>(lane, 32 * dt, h);

    // K and V rows of the workgroup's 128 keys through LDS; past S they load as zeros.
    const i32x4 rk = rsrc_words(a.k + bhk * S * D, S * D * 2);
    const i32x4 rv = rsrc_words(a.v + bhk * S * D, S * D * 2);
    const uint16_t* sk = smem + 2 * STAGE;
    const uint16_t* sv = sk + 128 * D;
    const uint16_t* skw = sk + 32 * wave * D;  // this wave's 32 keys
    const uint16_t* svw = sv + 32 * wave * D;
    {
        const uint32_t kv_byte = smem_byte + (uint32_t)(2 * STAGE * 2);
        dma_rows<D>(rk, kv_byte, (uint32_t)key0, D, wave, lane);
        dma_rows<D>(rk, kv_byte + 64 * D * 2, (uint32_t)key0 + 64, D, wave, lane);
        dma_rows<D>(rv, kv_byte + 128 * D * 2, (uint32_t)key0, D, wave, lane);
        dma_rows<D>(rv, kv_byte + 192 * D * 2, (uint32_t)key0 + 64, D, wave, lane);
    }

    // step it of head h, query block qb
    auto issue = [&](int h, int qb, int stage) {
        const int64_t bh = (int64_t)b * a.H + h;
        const i32x4 rq = rsrc_words(a.q + bh * S * D, S * D * 2);
        const i32x4 rdo = rsrc_words(a.dout + ((int64_t)b * S * a.H + h) * D, (S * a.H - h) * D * 2);
        const i32x4 rl = rsrc_words(a.lsd + bh * (a.Sp / 64) * 128, (a.Sp / 64) * 128 * 4);
        const uint32_t base = smem_byte + (uint32_t)(stage * STAGE * 2);
        const uint32_t q0 = (uint32_t)qb * 64;
        dma_rows<D>(rq, base, q0, D, wave, lane);
        dma_rows<D>(rdo, base + TILE * 2, q0, (uint32_t)(a.H * D), wave, lane);
        if (wave == 0)  // the [2][64] fp32 lse/Delta block (512 B; lanes 32-63 fall outside and write zeros)
            dma16(rl, __builtin_amdgcn_readfirstlane(base + 2 * TILE * 2),
                  lane < 32 ? (uint32_t)(qb * 512 + lane * 16) : kOOB);
    };

    // Block kd holds the queries of the workgroup's own first keys: every head's
    // steps start there and go round, and the first is on the way while the spans
    // are read.
    const int kd = 2 * kb;
    issue(h0, kd, 0);

    // The queries that the workgroup's keys meet, in whole blocks of 128, by which
    // the dQ pass reads dS^T. kd's are among them; a workgroup whose keys nobody
    // sees stores none. kinfo says which, and dQ reads no others.
    const Span mine = key_span(a.spans, b, my_key, (int)S, a.causal);
    const WaveSpan ws = wave_span(mine);
    const Span wg = workgroup_span(ws, slots);
    const int nqb = (int)((S + 63) / 64);
    int qstart = wg.lo / 128 * 2, qend = (int)(((int64_t)wg.hi + 127) / 128 * 2);
    if (wg.lo < wg.hi) {
        qstart = qstart < kd ? qstart : kd;
        qend = qend > kd ? qend : kd + 2;
    }
    const int stored0 = qstart / 2, stored1 = qend / 2;
    qend = qend < nqb ? qend : nqb;
    const int nq = qend - qstart;       // query blocks per head
    const int nit = hpg * nq;           // (head, query block) steps, head-major

    f32x16 dvacc[DT], dkacc[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int j = 0; j < 16; ++j) dvacc[t][j] = dkacc[t][j] = 0.f;

    bool bad_q = false;
    for (int h = h0; h < h0 + hpg; ++h)
        bad_q |= any_flag(a.qflags + ((int64_t)b * a.H + h) * (a.Sp / 64), qstart, qend);
    // the wave's K and V fragments (B operands of S and dP) stay in AGPRs
    wait_vmcnt<0>();
    __syncthreads();
    bf16x8 kf[KS], vf[KS];
    bool bad_k = false;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
        kf[s] = frag_at(skw, roff[s]);
        vf[s] = frag_at(svw, roff[s]);
        bad_k |= any_nonfinite(__builtin_bit_cast(uint4, kf[s]));
        asm volatile("" : "+a"(kf[s]), "+a"(vf[s]));
    }
    bad_k = __syncthreads_or(bad_k);
    if (threadIdx.x == 0) a.kinfo[bhk * a.nblk + kb] = make_int4(bad_k, stored0, stored1, 0);  // alike from every group
    int h = h0, qb = kd, left = nq;  // of this head
    float slope2 = BIAS ? a.slopes[h0] * kLog2e : 0.f;  // its load waits for every store before it: once per head
    for (int it = 0; it < nit; ++it) {
        // step it has landed: behind it only the last step's stores of dS^T went out
        // (the first's were waited for)
        wait_vmcnt<kDsStores>();
        __syncthreads();
        const bool wrap = --left == 0;
        const int next_h = wrap ? h + 1 : h, next_qb = wrap ? kd : qb + 1 == qend ? qstart : qb + 1;
        left = wrap ? nq : left;
        if (it + 1 < nit) issue(next_h, next_qb, (it + 1) & 1);
        uint16_t* sq = smem + (it & 1) * STAGE;
        uint16_t* sdo = sq + TILE;
        const float* sl = reinterpret_cast<const float*>(sq + 2 * TILE);
        if (bad_q && a.qflags[((int64_t)b * a.H + h) * (a.Sp / 64) + qb]) {  // workgroup-uniform
            clear_tile(sq, 2 * TILE);
            __syncthreads();
        }
        const int64_t bh = (int64_t)b * a.H + h;
        const __amdgpu_buffer_rsrc_t rds =
            make_rsrc(a.dst ? a.dst + bh * (a.head_ds / 2) : nullptr, a.dst ? a.head_ds : 0);
        const uint32_t ds_off = ds_block(qb, 4 * kb + wave, a.nblk) + (uint32_t)lane * 16u;
        // Every wave stores every block's dS^T; a tile is masked where its keys do not meet it.
        const int q0 = qb * 64;
        const bool edge = !(q0 >= ws.all_lo && q0 + 64 <= ws.all_hi);

        // accumulator j of tile t: query q0 + 32 t + 8 (j/4) + 4 half + j%4, key my_key.
        // P and dS of query tile t; EDGE hides what this lane's key does not meet.
        auto scores = [&](auto edge_tag, auto t_tag, const f32x16& sacc, const f32x16& dpacc, bf16x8 (&pb)[2],
                          bf16x8 (&db)[2]) {
            constexpr bool EDGE = decltype(edge_tag)::value;
            constexpr int t = decltype(t_tag)::value;
            // the lane's 4 half moves to the bounds, so each test compares a constant
            const int lo = mine.lo - q0 - 4 * half;
            const uint32_t width = (uint32_t)(mine.hi - mine.lo);
            const float dist = (float)(q0 + 4 * half - (int)my_key);
            float p[16], ds[16];
#pragma unroll
            for (int jq = 0; jq < 4; ++jq) {
                const int qi = 32 * t + 8 * jq + 4 * half;  // first of 4 consecutive queries
                const float4 l2 = *reinterpret_cast<const float4*>(&sl[qi]);
                const float4 dl = *reinterpret_cast<const float4*>(&sl[64 + qi]);
                const float lv[4] = {l2.x, l2.y, l2.z, l2.w}, dv4[4] = {dl.x, dl.y, dl.z, dl.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int j = 4 * jq + e, off = 32 * t + 8 * jq + e;
                    float x, slope = 1.f;  // slope: of tanh, over 4
                    if constexpr (CAP) {
                        const float r = __builtin_amdgcn_rcpf(1.f + exp2_hw(sacc[j] * a.cap_in));
                        x = __builtin_fmaf(r, -2.f * a.cap_log2, a.cap_log2 - lv[e]);
                        slope = __builtin_fmaf(-r, r, r);
                    } else {
                        x = __builtin_fmaf(sacc[j], a.scale_log2, -lv[e]);
                    }
                    if constexpr (BIAS) x = __builtin_fmaf(__builtin_fabsf(dist + (float)off), -slope2, x);
                    float pj = exp2_hw(x), dj = dpacc[j] - dv4[e];
                    if constexpr (CAP) dj *= slope;
                    dj *= pj;
                    if constexpr (EDGE) {
                        const bool hidden = (uint32_t)(off - lo) >= width;
                        pj = hidden ? 0.f : pj;
                        dj = hidden ? 0.f : dj;  // not 0 * dj: dP of a hidden pair may be anything
                    }
                    p[j] = pj;
                    ds[j] = dj;
                }
            }
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
                pb[kk] = pack_bf16x8(&p[8 * kk]);
                db[kk] = pack_bf16x8(&ds[8 * kk]);
            }
        };
        // one 32-query tile at a time: S = Q.K^T and dP = dO.V^T, its P and dS,
        // then its share of dV^T (d x key) += dO^T . P and dK^T += Q^T . dS
        auto tile = [&](auto t_tag) {
            constexpr int t = decltype(t_tag)::value;
            // none of the wave's keys meets the tile: 1 to 2% of documents' time, the
            // workgroup's other waves set a step's
            if (q0 + 32 * t >= ws.hi || q0 + 32 * t + 32 <= ws.lo) {
                const i32x4 zero = {0, 0, 0, 0};
#pragma unroll
                for (int kk = 0; kk < 2; ++kk)
                    __builtin_amdgcn_raw_buffer_store_b128(zero, rds, (int)(ds_off + 1024 * (2 * t + kk)), 0, 0);
                return;
            }
            f32x16 sacc, dpacc;
#pragma unroll
            for (int j = 0; j < 16; ++j) sacc[j] = dpacc[j] = 0.f;
            bf16x8 qf[2], df[2];
            qf[0] = frag_at(sq + 32 * t * D, roff[0]);
            df[0] = frag_at(sdo + 32 * t * D, roff[0]);
            __builtin_amdgcn_sched_group_barrier(kSchedDsRead, 2, 0);
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                if (s + 1 < KS) {
                    qf[(s + 1) & 1] = frag_at(sq + 32 * t * D, roff[s + 1]);
                    df[(s + 1) & 1] = frag_at(sdo + 32 * t * D, roff[s + 1]);
                    __builtin_amdgcn_sched_group_barrier(kSchedDsRead, 2, 0);
                }
                sacc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(qf[s & 1], kf[s], sacc, 0, 0, 0);
                dpacc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(df[s & 1], vf[s], dpacc, 0, 0, 0);
                __builtin_amdgcn_sched_group_barrier(kSchedMfma, 2, 0);
            }
            bf16x8 pb[2], db[2];
            if (edge) scores(std::true_type{}, t_tag, sacc, dpacc, pb, db);
            else scores(std::false_type{}, t_tag, sacc, dpacc, pb, db);
            // dS^T: elements 4 hh .. 4 hh + 3 of db[kk] are queries
            // q0 + 32 t + 16 kk + 8 hh + 4 half + 0..3 of this lane's key. The upper half's
            // hh = 0 changes places with the lower's hh = 1, which gives each lane 8
            // consecutive queries, 8 half from the first (zeros at keys past S). Where
            // packed_dq_again forms dS they fall outside the buffer range and are
            // dropped. kDsStores per step, which its first wait counts on.
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
                const uint4 w4 = __builtin_bit_cast(uint4, db[kk]);
                const auto xz = __builtin_amdgcn_permlane32_swap(w4.x, w4.z, false, false);
                const auto yw = __builtin_amdgcn_permlane32_swap(w4.y, w4.w, false, false);
                const i32x4 v = {(int)xz[0], (int)yw[0], (int)xz[1], (int)yw[1]};
                __builtin_amdgcn_raw_buffer_store_b128(v, rds, (int)(ds_off + 1024 * (2 * t + kk)), 0, 0);
            }
            // dO^T and Q^T fragments one step ahead of their MFMAs; step u = 2 dt + kk
            bf16x8 ot[2], qt[2];
            auto tr_frags = [&](int u, int slot) {
                const int dt = u >> 1, r0 = (32 * t + 16 * (u & 1)) * D;
                ot[slot] = frag_tr_at(sdo + r0, troff[dt][0], troff[dt][1]);
                qt[slot] = frag_tr_at(sq + r0, troff[dt][0], troff[dt][1]);
            };
            tr_frags(0, 0);
            __builtin_amdgcn_sched_group_barrier(kSchedDsRead, 4, 0);
#pragma unroll
            for (int u = 0; u < 2 * DT; ++u) {
                if (u + 1 < 2 * DT) {
                    tr_frags(u + 1, (u + 1) & 1);
                    __builtin_amdgcn_sched_group_barrier(kSchedDsRead, 4, 0);
                }
                const int dt = u >> 1, kk = u & 1;
                dvacc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ot[u & 1], pb[kk], dvacc[dt], 0, 0, 0);
                dkacc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(qt[u & 1], db[kk], dkacc[dt], 0, 0, 0);
                __builtin_amdgcn_sched_group_barrier(kSchedMfma, 2, 0);
            }
        };
        tile(std::integral_constant<int, 0>{});
        tile(std::integral_constant<int, 1>{});
        if constexpr (BIAS)
            if (wrap && it + 1 < nit) slope2 = a.slopes[next_h] * kLog2e;
        h = next_h;
        qb = next_qb;
    }

    wait_vmcnt<0>();  // every DMA has landed (also when the loop ran no block)
    __syncthreads();
    static_assert(32 * (D + 4) * 4 <= 32 * (D + 8) * 2 * 2, "fp32 patch rows fit a wave's share");
    void* patch = smem + wave * 32 * (D + 8) * 2;  // 32 rows of up to D + 4 floats per wave
    if (ng == 1) {
        store_rows<D, uint16_t>(dvacc, 1.f, patch, a.dv + bhk * S * D, D, kw, S, lane);
        store_rows<D, uint16_t>(dkacc, a.scale, patch, a.dk + bhk * S * D, D, kw, S, lane);
    } else {
        const int64_t pg = (bhk * ng + grp) * S * D;  // this group's partial
        store_rows<D, float>(dvacc, 1.f, patch, a.dv_part + pg, D, kw, S, lane);
        store_rows<D, float>(dkacc, a.scale, patch, a.dk_part + pg, D, kw, S, lane);
    }
}

__global__ __launch_bounds__(256) void packed_sum(PackedArgs a) {
    bwd_sum_range(a.dk_part, a.dv_part, a.dk, a.dv, a.ngroups, a.S * a.D, a.sum_n8,
                  (int64_t)blockIdx.x * blockDim.x + threadIdx.x, (int64_t)gridDim.x * blockDim.x);
}

// ------------------------------------------------------------------- dQ
// dQ's share of the infinities and NaN that K's tiles were cleared of: dS of a query
// that sees such a key is NaN, or 0 where its score is minus infinity or at the cap,
// and 0 times an infinity is NaN as well.
template <int D, typename Acc>
__device__ __forceinline__ void nan_of_keys(const PackedArgs& a, int64_t bhk, int kb0, int kb1, Span sees, int half,
                                            Acc& dqacc) {
#pragma unroll 1
    for (int i = kb0 / 2; i < (kb1 + 1) / 2; ++i) {
        if (a.kinfo[bhk * a.nblk + i].x == 0) continue;
        each_nonfinite<D>(a.k + bhk * a.S * D, i * 128, i * 128 + 128 < (int)a.S ? i * 128 + 128 : (int)a.S, sees, half,
                          [&](int dt, int j, float) { dqacc[dt][j] = __builtin_nanf(""); });
    }
}

// From the stored dS^T: per block of 64 keys that the workgroup's queries see, the
// K tile [64][D] and dS^T of the 128 queries, four blocks as they are in memory, go
// into LDS (two stages); dQ^T (d x query) += K^T . dS^T takes both by transposed reads.
// A block between the first and the last of these keys that none of the queries
// sees may have no dS^T in memory: it is left out, by kinfo. A K tile with infinities
// or NaN is cleared of them first, and the rows that see such a key get NaN there
// afterwards (nan_of_keys). Workgroups past dq_blocks sum the groups' dK / dV partials.
template <int D>
__global__ __launch_bounds__(256, 2) void packed_dq(PackedArgs a) {
    if ((int64_t)blockIdx.x >= a.dq_blocks) {
        const int64_t sb = (int64_t)blockIdx.x - a.dq_blocks, nsb = (int64_t)gridDim.x - a.dq_blocks;
        bwd_sum_range(a.dk_part, a.dv_part, a.dk, a.dv, a.ngroups, a.S * D, a.sum_n8, sb * 256 + threadIdx.x,
                      nsb * 256);
        return;
    }
    constexpr int KB = 64, QB = 128, DT = D / 32;
    constexpr int KT = 64 * D, DSTILE = 64 * QB;  // K tile, dS^T tile (elements)
    constexpr int STAGE = KT + DSTILE;
    __shared__ __attribute__((aligned(1024))) uint16_t smem[2 * STAGE];
    __shared__ int slots[4][2];
    static_assert(4 * 32 * (D + 8) <= 2 * STAGE, "the epilogue's bf16 patches fit in the stages");
    const uint32_t smem_byte = (uint32_t)reinterpret_cast<uintptr_t>(smem);
    const int lane = threadIdx.x & 63, wave = wave_id();
    const int nbh = a.B * a.H;
    const int qb = a.nblk - 1 - (int)(blockIdx.x / nbh);
    const int bh = xcd_head_order((int)(blockIdx.x % nbh), nbh);
    const int b = bh / a.H, h = bh % a.H;
    const int64_t bhk = (int64_t)b * a.Hkv + h / (a.H / a.Hkv);
    const int64_t S = a.S;
    const int64_t q0 = (int64_t)qb * QB;
    const int64_t qw = q0 + 32 * wave;

    uint32_t tk[DT][2], td[2];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) tk[dt][hh] = tr_off<D>(lane, 32 * dt, hh);
    // the rows and columns that tr_off takes, in a block's order: of this wave's 32
    // queries step g % 2, half i % 4 / 2, four queries i % 2
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
        const int i = lane & 15, g = lane >> 4, row = 4 * (g >> 1) + (i >> 2) + 8 * hh;
        td[hh] = (uint32_t)((wave >> 1) * kDsBlock + (2 * (wave & 1) + (g & 1)) * 1024 + (32 * ((i >> 1) & 1) + row) * 16 +
                            8 * (i & 1));
    }

    const i32x4 rk = rsrc_words(a.k + bhk * S * D, S * D * 2);
    const i32x4 rds = rsrc_words(a.dst + bh * (a.head_ds / 2), a.head_ds);
    auto issue = [&](int kb, int stage) {
        const uint32_t base = smem_byte + (uint32_t)(stage * STAGE * 2);
        const uint32_t key0 = (uint32_t)kb * KB;
        dma_rows<D>(rk, base, key0, D, wave, lane);
        // two blocks of dS^T for each 32 keys, a wave one of the four
        const uint32_t block = ds_block(2 * qb + (wave & 1), 2 * kb + (wave >> 1), a.nblk);
#pragma unroll
        for (int j = 0; j < kDsBlock / 1024; ++j)
            dma16(rds, __builtin_amdgcn_readfirstlane(base + KT * 2 + (uint32_t)(wave * kDsBlock + j * 1024)),
                  block + (uint32_t)(j * 1024 + lane * 16));
    };
    const int kd = 2 * qb;  // the tile's own keys first, on the way while the spans are read
    issue(kd, 0);
    const Span mine = query_span(a.spans, b, qw + (lane & 31), (int)S, a.causal);
    const Span wg = workgroup_span(wave_span(mine), slots);
    const int kb0 = wg.lo / KB, kb1 = (wg.hi + KB - 1) / KB;
    const int4* kinfo = a.kinfo + bhk * a.nblk;
    bool bad = false, hole = false;
    for (int i = kb0 / 2 + lane; i < (kb1 + 1) / 2; i += kWave) {
        const int4 x = kinfo[i];
        bad |= x.x != 0;
        hole |= qb < x.y || qb >= x.z;
    }
    const bool bad_k = __any(bad), holes = __any(hole);

    f32x16 dqacc[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int j = 0; j < 16; ++j) dqacc[t][j] = 0.f;

    int kb = kd, next = 0, stage = 0;
    for (bool more = kb0 < kb1; more; kb = next, stage ^= 1) {
        next = kb == kd ? kb0 : kb + 1;
        next += next == kd;
        more = next < kb1;
        wait_vmcnt<0>();
        __syncthreads();
        if (more) issue(next, stage ^ 1);
        if (kb < kb0 || kb >= kb1) continue;  // kd may be no key of these queries
        if (holes && (qb < kinfo[kb / 2].y || qb >= kinfo[kb / 2].z)) continue;  // workgroup-uniform, as below
        uint16_t* sk = smem + stage * STAGE;
        const uint16_t* sds = sk + KT;
        if (bad_k && kinfo[kb / 2].x) {
            clear_tile(sk, KT);
            __syncthreads();
        }
#pragma unroll
        for (int kc = 0; kc < KB / 16; ++kc) {
            const bf16x8 bfr = frag_tr_at(sds + ((kc >> 1) * 2 * kDsBlock + (kc & 1) * 256) / 2, td[0], td[1]);
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
                dqacc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag_tr_at(sk + 16 * kc * D, tk[dt][0], tk[dt][1]),
                                                                   bfr, dqacc[dt], 0, 0, 0);
        }
    }

    if (bad_k) nan_of_keys<D>(a, bhk, kb0, kb1, mine, lane >> 5, dqacc);
    wait_vmcnt<0>();  // every DMA has landed (also when the loop ran no block)
    __syncthreads();
    store_rows<D, uint16_t>(dqacc, a.scale, smem + wave * 32 * (D + 8), a.dq + (int64_t)bh * S * D, D, qw, S, lane);
}

// The same with S and dP formed once more, shaped as the forward: S^T = K.Q^T,
// dP^T = V.dO^T (lane = query), dQ^T += K^T.dS^T.
template <int D, bool CAP, bool BIAS>
__global__ __launch_bounds__(256, 1) void packed_dq_again(PackedArgs a) {
    constexpr int KB = 64, QB = 128, KS = D / 16, DT = D / 32;
    constexpr int TILE = 64 * D;
    constexpr int STAGE = 2 * TILE;  // K, V [64][D]
    constexpr int QDO = 2 * QB * D;  // the workgroup's Q and dO rows, [128][D] each, after the stages
    __shared__ __attribute__((aligned(1024))) uint16_t smem[2 * STAGE + QDO];
    __shared__ int slots[4][2];
    static_assert(4 * 32 * (D + 8) <= 2 * STAGE, "the epilogue's bf16 patches fit in the stages");
    const uint32_t smem_byte = (uint32_t)reinterpret_cast<uintptr_t>(smem);
    const int lane = threadIdx.x & 63, wave = wave_id();
    const int col = lane & 31, half = lane >> 5;
    const int nbh = a.B * a.H;
    const int qb = a.nblk - 1 - (int)(blockIdx.x / nbh);
    const int bh = xcd_head_order((int)(blockIdx.x % nbh), nbh);
    const int b = bh / a.H, h = bh % a.H;
    const int64_t bhk = (int64_t)b * a.Hkv + h / (a.H / a.Hkv);
    const int64_t S = a.S;
    const int64_t q0 = (int64_t)qb * QB;
    const int64_t qw = q0 + 32 * wave;
    const int64_t my_q = qw + col;

    uint32_t roff[KS], troff[DT][2];
#pragma unroll
    for (int s = 0; s < KS; ++s) roff[s] = rows_off<D>(lane, 2 * s + half);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) troff[dt][hh] = tr_off<D>(lane, 32 * dt, hh);

    // Q and dO rows of the workgroup's 128 queries stay in LDS for the whole key
    // loop. They reach dQ through S and dP alone, so theirs need no clearing.
    const i32x4 rq = rsrc_words(a.q + (int64_t)bh * S * D, S * D * 2);
    const i32x4 rdo = rsrc_words(a.dout + ((int64_t)b * S * a.H + h) * D, (S * a.H - h) * D * 2);
    const uint16_t* sqw = smem + 2 * STAGE + 32 * wave * D;  // this wave's 32 queries
    const uint16_t* sdow = sqw + QB * D;
    {
        const uint32_t qd_byte = smem_byte + (uint32_t)(2 * STAGE * 2);
        dma_rows<D>(rq, qd_byte, (uint32_t)q0, D, wave, lane);
        dma_rows<D>(rq, qd_byte + 64 * D * 2, (uint32_t)q0 + 64, D, wave, lane);
        dma_rows<D>(rdo, qd_byte + QB * D * 2, (uint32_t)q0, (uint32_t)(a.H * D), wave, lane);
        dma_rows<D>(rdo, qd_byte + (QB + 64) * D * 2, (uint32_t)q0 + 64, (uint32_t)(a.H * D), wave, lane);
    }
    float lse2 = __builtin_inff(), delta = 0.f;
    if (my_q < S) {
        const float* blk = a.lsd + ((int64_t)bh * (a.Sp / 64) + my_q / 64) * 128;
        lse2 = blk[my_q % 64];
        delta = blk[64 + my_q % 64];
    }

    const i32x4 rk = rsrc_words(a.k + bhk * S * D, S * D * 2);
    const i32x4 rv = rsrc_words(a.v + bhk * S * D, S * D * 2);
    const Span mine = query_span(a.spans, b, my_q, (int)S, a.causal);
    const WaveSpan ws = wave_span(mine);
    const Span wg = workgroup_span(ws, slots);
    const int kb0 = wg.lo / KB, kb1 = (wg.hi + KB - 1) / KB;
    const int4* kinfo = a.kinfo + bhk * a.nblk;
    bool bad = false;
    for (int i = kb0 / 2 + lane; i < (kb1 + 1) / 2; i += kWave) bad |= kinfo[i].x != 0;
    const bool bad_k = __any(bad);
    const float slope2 = BIAS ? a.slopes[h] * kLog2e : 0.f;

    auto issue = [&](int kb, int stage) {
        const uint32_t base = smem_byte + (uint32_t)(stage * STAGE * 2);
        const uint32_t key0 = (uint32_t)kb * KB;
        dma_rows<D>(rk, base, key0, D, wave, lane);
        dma_rows<D>(rv, base + TILE * 2, key0, D, wave, lane);
    };

    f32x16 dqacc[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int j = 0; j < 16; ++j) dqacc[t][j] = 0.f;

    if (kb0 < kb1) issue(kb0, 0);
    for (int kb = kb0; kb < kb1; ++kb) {
        wait_vmcnt<0>();
        __syncthreads();
        if (kb + 1 < kb1) issue(kb + 1, (kb + 1 - kb0) & 1);
        uint16_t* sk = smem + ((kb - kb0) & 1) * STAGE;
        const uint16_t* sv = sk + TILE;
        const bool clear = bad_k && kinfo[kb / 2].x;  // K for dQ, not for S
        const int key0 = kb * KB;
        // Every wave runs every block, masked where its queries do not see it.
        const bool edge = !(key0 >= ws.all_lo && key0 + KB <= ws.all_hi);
        const float dist = (float)((int)my_q - key0 - 4 * half);
        const int lo = mine.lo - key0 - 4 * half, hi = mine.hi - key0 - 4 * half;
        auto tile = [&](auto t_tag) {
            constexpr int t = decltype(t_tag)::value;
            f32x16 sacc, dpacc;
#pragma unroll
            for (int j = 0; j < 16; ++j) sacc[j] = dpacc[j] = 0.f;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                sacc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag_at(sk + 32 * t * D, roff[s]), frag_at(sqw, roff[s]),
                                                              sacc, 0, 0, 0);
                dpacc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag_at(sv + 32 * t * D, roff[s]),
                                                               frag_at(sdow, roff[s]), dpacc, 0, 0, 0);
            }
            float ds[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const int ko = 32 * t + 8 * (j >> 2) + (j & 3);
                float x, slope = 1.f;
                if constexpr (CAP) {
                    const float r = __builtin_amdgcn_rcpf(1.f + exp2_hw(sacc[j] * a.cap_in));
                    x = __builtin_fmaf(r, -2.f * a.cap_log2, a.cap_log2 - lse2);
                    slope = __builtin_fmaf(-r, r, r);
                } else {
                    x = __builtin_fmaf(sacc[j], a.scale_log2, -lse2);
                }
                if constexpr (BIAS) x = __builtin_fmaf(__builtin_fabsf(dist - (float)ko), -slope2, x);
                float dj = dpacc[j] - delta;
                if constexpr (CAP) dj *= slope;
                dj *= exp2_hw(x);
                ds[j] = edge && (ko < lo || ko >= hi) ? 0.f : dj;
            }
            bf16x8 db[2];
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) db[kk] = pack_bf16x8(&ds[8 * kk]);
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int kk = 0; kk < 2; ++kk) {
                    bf16x8 kt = frag_tr_at(sk + (32 * t + 16 * kk) * D, troff[dt][0], troff[dt][1]);
                    if (clear) {
                        uint4 w = __builtin_bit_cast(uint4, kt);
                        w.x = clear_nonfinite(w.x); w.y = clear_nonfinite(w.y);
                        w.z = clear_nonfinite(w.z); w.w = clear_nonfinite(w.w);
                        kt = __builtin_bit_cast(bf16x8, w);
                    }
                    dqacc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kt, db[kk], dqacc[dt], 0, 0, 0);
                }
        };
        tile(std::integral_constant<int, 0>{});
        tile(std::integral_constant<int, 1>{});
    }

    if (bad_k) nan_of_keys<D>(a, bhk, kb0, kb1, mine, half, dqacc);
    wait_vmcnt<0>();  // every DMA has landed (also when the loop ran no block)
    __syncthreads();
    store_rows<D, uint16_t>(dqacc, a.scale, smem + wave * 32 * (D + 8), a.dq + (int64_t)bh * S * D, D, qw, S, lane);
}

size_t align256(size_t n) { return (n + 255) / 256 * 256; }

// dS^T is stored where a head's fits 32-bit buffer offsets (S <= 32640).
bool dq_from_ds(const mc_attn_desc& d) {
    return attention_uses_mfma(d) && head_ds_bytes(d.seq) < ((int64_t)1 << 31);
}

// The group rule of the causal kernels, which know the rows' shape; spans are
// taken as causal.
mc_attn_desc shape_of(const mc_packed_attn_desc& p, bool spans) {
    mc_attn_desc d = p.attn;
    if (spans) d.causal = 1;
    return d;
}

PackedArgs packed_args(const mc_packed_attn_desc& p, const void* q, const void* k, const void* v, const int32_t* spans,
                       const float* slopes) {
    const mc_attn_desc& d = p.attn;
    PackedArgs a{};
    a.q = static_cast<const uint16_t*>(q);
    a.k = static_cast<const uint16_t*>(k);
    a.v = static_cast<const uint16_t*>(v);
    a.spans = reinterpret_cast<const int4*>(spans);
    a.slopes = slopes;
    a.S = d.seq;
    a.Sp = (d.seq + 63) / 64 * 64;
    a.B = (int)d.batch; a.H = d.heads; a.Hkv = d.kv_heads; a.D = d.head_dim;
    a.nblk = (int)((d.seq + 127) / 128);
    a.causal = d.causal ? 1 : 0;
    a.scale = p.cap != 0.f ? 4.f * d.scale : d.scale;
    a.scale_log2 = d.scale * kLog2e;
    if (p.cap != 0.f) {
        a.cap_in = 2.f * kLog2e * (d.scale / p.cap);
        a.cap_log2 = p.cap * kLog2e;
    }
    return a;
}

// go(head dim, cap, bias) with the three as types.
template <typename F>
void by_variant(int D, bool cap, bool bias, F&& go) {
    using std::false_type;
    using std::true_type;
    auto pick = [&](auto dim) {
        if (cap && bias) go(dim, true_type{}, true_type{});
        else if (cap) go(dim, true_type{}, false_type{});
        else if (bias) go(dim, false_type{}, true_type{});
        else go(dim, false_type{}, false_type{});
    };
    if (D == 64) pick(std::integral_constant<int, 64>{});
    else pick(std::integral_constant<int, 128>{});
}

}  // namespace

hipError_t launch_attention_spans(const int32_t* documents, const uint8_t* prefix, int64_t batch, int64_t seq,
                                  int causal, int32_t* spans, hipStream_t stream) {
    packed_spans<<<dim3((unsigned)batch), kScanThreads, 0, stream>>>(documents, prefix, (int)seq, causal,
                                                                    reinterpret_cast<int4*>(spans));
    return hipGetLastError();
}

PackedWs packed_fwd_ws(const mc_packed_attn_desc& p) {
    const mc_attn_desc& d = p.attn;
    PackedWs w{};
    if (!attention_uses_mfma(d) || packed_fwd_from_rows(d.seq)) return w;
    const size_t Sp = (size_t)(d.seq + 63) / 64 * 64, bhk = (size_t)d.batch * d.kv_heads;
    w.vt = 0;
    w.flags = align256(bhk * d.head_dim * Sp * 2);
    w.total = w.flags + align256(bhk * (Sp / 64) * 4);
    return w;
}

hipError_t launch_packed_fwd(const mc_packed_attn_desc& p, const void* q, const void* k, const void* v,
                             const int32_t* spans, const float* slopes, void* o, float* lse, char* ws,
                             hipStream_t stream) {
    const mc_attn_desc& d = p.attn;
    if (!attention_uses_mfma(d)) {
        if (attention_f32_mfma_fwd(d)) return launch_packed_f32_fwd(p, q, k, v, spans, slopes, o, lse, stream);
        return launch_packed_rows_fwd(p, q, k, v, spans, slopes, o, lse, stream);
    }
    const PackedWs w = packed_fwd_ws(p);
    PackedArgs a = packed_args(p, q, k, v, spans, slopes);
    uint16_t* vt = reinterpret_cast<uint16_t*>(ws + w.vt);
    a.vt = vt;
    a.vflags = reinterpret_cast<int32_t*>(ws + w.flags);
    a.o = static_cast<uint16_t*>(o);
    a.lse = lse;
    const dim3 gvt((unsigned)(a.Sp / 64), (unsigned)(a.B * a.Hkv));
    const dim3 grid((unsigned)((int64_t)a.nblk * a.B * a.H));
    by_variant(a.D, p.cap != 0.f, slopes != nullptr, [&](auto dim, auto cap, auto bias) {
        constexpr int D = decltype(dim)::value;
        constexpr bool CAP = decltype(cap)::value, BIAS = decltype(bias)::value;
        if (packed_fwd_from_rows(d.seq)) {
            packed_fwd<D, CAP, BIAS, true><<<grid, 256, 0, stream>>>(a);
        } else {
            packed_vt<D><<<gvt, 256, 0, stream>>>(a.v, a.S, a.Sp, vt, a.vflags);
            packed_fwd<D, CAP, BIAS, false><<<grid, 256, 0, stream>>>(a);
        }
    });
    return hipGetLastError();
}

PackedBwdWs packed_bwd_ws(const mc_packed_attn_desc& p, bool spans) {
    const mc_attn_desc d = shape_of(p, spans);
    PackedBwdWs w{};
    const size_t B = (size_t)d.batch, H = (size_t)d.heads, Hkv = (size_t)d.kv_heads, D = (size_t)d.head_dim;
    const size_t S = (size_t)d.seq, Sp = (S + 63) / 64 * 64, nblk = (S + 127) / 128;
    const bool mfma = attention_uses_mfma(d);
    size_t off = 0;
    w.lsd = off;
    off += align256(mfma ? B * H * (Sp / 64) * 128 * 4 : B * H * S * 4);
    if (mfma) {
        w.qflags = off;  off += align256(B * H * (Sp / 64) * 4);
        w.kinfo = off;   off += align256(B * Hkv * nblk * 16);
    }
    const size_t ng = mfma ? (size_t)attn_dkdv_groups(d)
                           : attention_f32_mfma_bwd(d) ? (size_t)attention_f32_groups(d) : 1;
    if (ng > 1) {
        w.dk_part = off;  off += align256(B * Hkv * ng * S * D * 4);
        w.dv_part = off;  off += align256(B * Hkv * ng * S * D * 4);
    }
    w.dst = off;
    if (dq_from_ds(d)) off += B * H * (size_t)head_ds_bytes(d.seq);
    w.total = off;
    return w;
}

hipError_t launch_packed_bwd(const mc_packed_attn_desc& p, const void* q, const void* k, const void* v,
                             const int32_t* spans, const float* slopes, const void* o, const float* lse,
                             const void* dout, void* dq, void* dk, void* dv, char* ws, hipStream_t stream) {
    const mc_attn_desc d = shape_of(p, spans != nullptr);
    const PackedBwdWs w = packed_bwd_ws(p, spans != nullptr);
    float *dk_part = reinterpret_cast<float*>(ws + w.dk_part), *dv_part = reinterpret_cast<float*>(ws + w.dv_part);
    float* lsd = reinterpret_cast<float*>(ws + w.lsd);
    if (!attention_uses_mfma(d)) {
        if (attention_f32_mfma_bwd(d))
            return launch_packed_f32_bwd(p, q, k, v, spans, slopes, o, lse, dout, dq, dk, dv, lsd, dk_part, dv_part,
                                         stream);
        return launch_packed_rows_bwd(p, q, k, v, spans, slopes, o, lse, dout, dq, dk, dv, lsd, stream);
    }
    PackedArgs a = packed_args(p, q, k, v, spans, slopes);
    int32_t* qflags = reinterpret_cast<int32_t*>(ws + w.qflags);
    a.dout = static_cast<const uint16_t*>(dout);
    a.lsd = lsd;
    a.qflags = qflags;
    a.kinfo = reinterpret_cast<int4*>(ws + w.kinfo);
    a.dq = static_cast<uint16_t*>(dq);
    a.dk = static_cast<uint16_t*>(dk);
    a.dv = static_cast<uint16_t*>(dv);
    a.ngroups = attn_dkdv_groups(d);
    a.dk_part = a.ngroups > 1 ? dk_part : nullptr;
    a.dv_part = a.ngroups > 1 ? dv_part : nullptr;
    const bool from_ds = dq_from_ds(d);
    a.dst = from_ds ? reinterpret_cast<uint16_t*>(ws + w.dst) : nullptr;
    a.head_ds = head_ds_bytes(a.S);
    a.dq_blocks = (int64_t)a.nblk * a.B * a.H;
    a.sum_n8 = (int64_t)a.B * a.Hkv * a.S * a.D / 8;
    const dim3 gprep((unsigned)((int64_t)a.nblk * a.B * a.H));
    const dim3 gkv((unsigned)((int64_t)a.nblk * a.B * a.Hkv * a.ngroups));
    by_variant(a.D, p.cap != 0.f, slopes != nullptr, [&](auto dim, auto cap, auto bias) {
        constexpr int D = decltype(dim)::value;
        constexpr bool CAP = decltype(cap)::value, BIAS = decltype(bias)::value;
        packed_prep<D, CAP, BIAS><<<gprep, 256, 0, stream>>>(a, static_cast<const uint16_t*>(o), lse, lsd, qflags);
        packed_dkdv<D, CAP, BIAS><<<gkv, 256, 0, stream>>>(a);
        if (from_ds) {
            // with partials, the dQ launch also sums them (see attn_bwd_dq_ds_bf16)
            const int64_t nsum = a.ngroups > 1 ? std::min<int64_t>((2 * a.sum_n8 + 255) / 256, 512) : 0;
            packed_dq<D><<<dim3((unsigned)(a.dq_blocks + nsum)), 256, 0, stream>>>(a);
        } else {
            if (a.ngroups > 1) {
                const int64_t blocks = std::min<int64_t>((2 * a.sum_n8 + 255) / 256, 4096);
                packed_sum<<<dim3((unsigned)blocks), 256, 0, stream>>>(a);
            }
            packed_dq_again<D, CAP, BIAS><<<dim3((unsigned)a.dq_blocks), 256, 0, stream>>>(a);
        }
    });
    return hipGetLastError();
}

}  // namespace mc
