// Losses over a vocabulary's logits for what comes after supervised
// fine-tuning, gfx950: log-probabilities of given tokens, the preference loss
// over pairs of sequences, the clipped policy loss with its KL term, and
// distillation from a teacher's top logits. They start from the same logits
// [rows, vocab] as the cross entropy (rowops.hip).
//
// Per row, with q = softmax(x / T) and lse = log sum exp(x / T):
//   l = x_t / T - lse, the token's log-probability; dl/dx_j = ([j = t] - q_j) / T.
// Every loss but distillation is a function of the l alone, so one kernel forms
// l and the row's maximum and sum from one read of the logits (lp_rows_k), small
// kernels form the loss and dloss/dl, and one kernel turns dloss/dl into the
// gradient of the logits (lp_bwd_k). Distillation is
// sum_k p_k (log p_k - log q_{id k}) over a teacher's K best, whose gradient is
// (P q_j - sum_{id k = j} p_k) / T with P = sum p: the same dense part with K
// entries taken out of it instead of one. A row that is not counted is never read
// and its gradient is zero.
// A token's part of the policy's and the distillation's gradient depends on its own
// row and on counts alone, so those have one kernel for both that reads the logits
// once (policy_both_k, distill_both_k). The preference's depends on whole
// sequences: its logits are read again.
//
// Bound by HBM throughout: 2 or 4 bytes per logit and pass against about ten
// operations. A copy of 1 GiB runs at 5.0 TB/s here; kernels, three of four rows
// counted:
//   lp_rows_k       f32 2036 x 50257 54.8 us, 5.6 TB/s; bf16, for sums of l, 4072 x 151936 182, 5.1
//   lp_bwd_k        the same 116, 6.2; 386, 5.6
//   policy_both_k   bf16 4096 x 151936 410, 5.3; f32 2036 x 50257 143, 5.0
//   distill_both_k  bf16 2036 x 151936, 64 entries, 219, 5.0; f32 1500 x 50257, 8 entries, 108, 4.9
//   distill_rows_k, distill_bwd_k, nearly all rows counted: bf16 2036 x 151936, 64 entries, 104, 5.6
//                   and 234, 5.1 (gradients elsewhere in a vector 252, 4.7); f32 1500 x 50257, 8
//                   entries, 44.9, 5.6 and 113, 4.9 (112, 4.9)
#include <type_traits>

#include "common.hpp"
#include "kernels.hpp"
#include "log_of.hpp"
#include "rules.hpp"
#include "vocab_rows.hpp"

namespace mc {
namespace {

constexpr float kNegInf = -__builtin_inff();

// An element as its bits, to convert where it is used: a conversion waits for the load.
template <typename T> __device__ __forceinline__ uint32_t raw_load(const T* p, int64_t i) {
    if constexpr (std::is_same<T, float>::value) return __float_as_uint(p[i]);
    else return p[i];
}
template <typename T> __device__ __forceinline__ float from_raw(uint32_t w) {
    return std::is_same<T, float>::value ? __uint_as_float(w) : __uint_as_float(w << 16);
}

// The float wave_sum's steps in 64 bits.
template <int CTRL> __device__ __forceinline__ double dpp64(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, 0xf, 0xf, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), CTRL, 0xf, 0xf, false);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double wave_sum(double v) {
    v += dpp64<0xB1>(v);
    v += dpp64<0x4E>(v);
    v += dpp64<0x141>(v);
    v += dpp64<0x140>(v);
    v += __shfl_xor(v, 16, kWave);
    v += __shfl_xor(v, 32, kWave);
    return v;
}

// ------------------------------------------------------------ row statistics
// m = max x and s = sum 2^((x - m) c), c = log2(e) / T as c_hi + c_lo
// (row_scale): with one float for c every exponent is off by up to 6e-8 of
// itself to the same side, and so is every l of a sequence, which the sums over
// an answer add up instead of averaging out. x - m comes first: x c alone
// overflows where logits hold the type's lowest value. An all -inf row has
// m = -inf and s = 0, a NaN in the row makes s NaN: l and the gradient are NaN in
// both. The backward takes m and s as they are: lse as one float would cost each
// q 2^-24 |lse| of itself.
// S, the sum's type: in float one part in 2^24 of the sum is lost at every
// addition to it, which shows in an l whose token holds nearly all of the row.
template <typename S> struct Stat {
    float m;
    S s;
};
// 2^(d c), d <= 0. The small product goes into the fma: added to a rounded one it
// would be lost.
__device__ __forceinline__ float exp_of(float d, LpScale k) { return exp2_hw(fmaf(d, k.c_hi, d * k.c_lo)); }

// exp2_hw is low by 3.4e-9 of itself on the average of any stretch (2.6e-8 rms); what
// rescales a sum of doubles is put right by that.
constexpr double kExpMean = 1.0 + 3.4e-9;
// A sum relative to `from` as one relative to m >= from; equal ones, -inf among them,
// need no factor.
template <typename S> __device__ __forceinline__ S rescaled(S s, float from, float m, LpScale k) {
    if (from == m) return s;
    const S f = exp_of(from - m, k);
    return std::is_same<S, double>::value ? s * (f * (S)kExpMean) : s * f;
}
template <typename S> __device__ __forceinline__ Stat<S> stat_join(Stat<S> a, Stat<S> b, LpScale k) {
    const float m = fmaxf(a.m, b.m);
    return Stat<S>{m, rescaled(a.s, a.m, m, k) + rescaled(b.s, b.m, m, k)};
}

// Over the workgroup's NT threads in a fixed order: the maximum of each wave, its
// sums relative to that, then the same of the waves with sums of type R (of floats,
// that chain loses the most, and it alone is short enough for doubles). One factor
// per step: joined in pairs, a share would collect the errors of one at every level.
// red: one slot per wave.
template <int NT, typename R, typename S>
__device__ __forceinline__ Stat<R> wg_stat(Stat<S> v, LpScale k, Stat<S>* red) {
    const float wm = wave_max(v.m);
    const S ws = wave_sum(rescaled(v.s, v.m, wm, k));
    if (lane_id() == 0) red[threadIdx.x >> 6] = Stat<S>{wm, ws};
    __syncthreads();
    Stat<R> r{red[0].m, 0};
#pragma unroll
    for (int w = 1; w < NT / 64; ++w) r.m = fmaxf(r.m, red[w].m);
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) r.s += rescaled((R)red[w].s, red[w].m, r.m, k);
    return r;
}

// What a share's terms are relative to: where all of it is -inf, anything finite.
__device__ __forceinline__ float base_of(float m) { return m == kNegInf ? 0.f : m; }
__device__ __forceinline__ float term_of(float x, float base, LpScale k) { return exp_of(x - base, k); }

// One thread's share of a row's vectors from c on: U of them requested and
// reduced at a time, one rescale to their maximum, then one exp2 per element. The
// last of them go together, too: one by one, each would wait for its own load.
// P: of the sums of U vectors. With floats the thread that holds a row's largest
// term, 1, rounds at 2^-24 of it for each term it adds there, and l is off by 4e-8
// (rms) where that term is most of the row; a score of 110 tokens by 5e-7. Doubles
// cost 2.7% of a preference step on 4072 bf16 rows of 151936 (555 / 570 us) and 10%
// of 777 rows alone (51.4 / 56.5), so of bf16 logits they are for l that are summed
// (preference, policy forward) and for shared rows (parts_k); for l of f32 ones, half
// as many per byte, they cost nothing. Distillation's rows and the held ones have floats.
template <typename T, int NT, typename S, int U, typename P = float>
__device__ __forceinline__ Stat<S> vec_stat(const T* __restrict__ xv, int c, int nvec, LpScale k) {
    constexpr int N = Vec16<T>::N;
    float m = kNegInf;
    S s = 0;
    auto group = [&](auto whole) {
        float v[U][N];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int at = c + u * NT;
            Vec16<T>::load(xv + (int64_t)(decltype(whole)::value || at < nvec ? at : c) * N, v[u]);
        }
#pragma unroll
        for (int u = 1; u < U; ++u)
            if (!decltype(whole)::value && c + u * NT >= nvec) {
#pragma unroll
                for (int e = 0; e < N; ++e) v[u][e] = kNegInf;
            }
        float vm = v[0][0];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < N; ++e) vm = fmaxf(vm, v[u][e]);
        if (vm > m) {
            s = rescaled(s, m, vm, k);  // 0 for the first
            m = vm;
        }
        const float base = base_of(m);
        P ps[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            ps[u] = 0;
#pragma unroll
            for (int e = 0; e < N; ++e) ps[u] += (P)term_of(v[u][e], base, k);
        }
#pragma unroll
        for (int u = U; u > 1; u /= 2)
#pragma unroll
            for (int i = 0; i < u / 2; ++i) ps[i] = ps[i] + ps[i + u / 2];
        s += ps[0];
    };
    for (; c < nvec - (U - 1) * NT; c += U * NT) group(std::true_type{});
    if (c < nvec) group(std::false_type{});
    return Stat<S>{m, s};
}
// with the thread's element of the row's edges, if it has one
template <typename T, typename S>
__device__ __forceinline__ Stat<S> edge_stat(const T* __restrict__ xr, int vocab, const RowSpan<T>& span, Stat<S> st,
                                             LpScale k) {
    const int64_t j = span.edge((int)threadIdx.x, vocab);
    if (j < 0) return st;
    const float v = Elem<T>::load(xr, j);
    return stat_join(st, Stat<S>{v, (S)term_of(v, base_of(v), k)}, k);
}
template <typename T, int NT, typename S, typename P>
__device__ __forceinline__ Stat<S> row_stat(const T* __restrict__ xr, int vocab, LpScale k) {
    static_assert(NT >= 2 * Vec16<T>::N, "a thread per edge element");
    const RowSpan<T> span(xr, vocab);
    return edge_stat(xr, vocab, span, vec_stat<T, NT, S, 4, P>(xr + span.head, threadIdx.x, (int)span.nvec, k), k);
}

// ------------------------------------------------- sums over a workgroup
template <int NT, int C> __device__ __forceinline__ void wg_sum_f64(double (&v)[C], double (*red)[C]) {
#pragma unroll
    for (int c = 0; c < C; ++c) v[c] = wave_sum(v[c]);
    __syncthreads();
    if (lane_id() == 0)
#pragma unroll
        for (int c = 0; c < C; ++c) red[threadIdx.x >> 6][c] = v[c];
    __syncthreads();
#pragma unroll
    for (int c = 0; c < C; ++c) {
        v[c] = red[0][c];
#pragma unroll
        for (int w = 1; w < NT / 64; ++w) v[c] += red[w][c];
    }
}

// ------------------------------------------------------------- row kernels
__device__ __forceinline__ bool counted(uint32_t t, int64_t ignore_index) {
    return !(ignore_index >= 0 && (int64_t)t == ignore_index);
}

// Few rows do not fill the CUs, and one CU reads about 30 bytes a ns: then
// gridDim.y workgroups take a share of a row's vectors each, and the kernel that
// follows joins their statistics.
template <typename T, int NT>
__global__ __launch_bounds__(NT) void parts_k(int vocab, const T* __restrict__ logits,
                                              const uint32_t* __restrict__ targets, int64_t ignore_index,
                                              const uint8_t* __restrict__ mask, LpScale k,
                                              Stat<double>* __restrict__ part) {
    __shared__ Stat<double> red[NT / 64];
    const int64_t row = blockIdx.x;
    if (targets ? !counted(targets[row], ignore_index) : mask && mask[row] == 0) return;
    const T* xr = logits + row * vocab;
    const RowSpan<T> span(xr, vocab);
    const int share = ((int)span.nvec + (int)gridDim.y - 1) / (int)gridDim.y, lo = (int)blockIdx.y * share;
    const int hi = lo + share < (int)span.nvec ? lo + share : (int)span.nvec;
    Stat<double> st = vec_stat<T, NT, double, 4, double>(xr + span.head, lo + (int)threadIdx.x, hi, k);
    if (blockIdx.y == 0) st = edge_stat(xr, vocab, span, st, k);
    st = wg_stat<NT, double>(st, k, red);
    if (threadIdx.x == 0) part[row * gridDim.y + blockIdx.y] = st;
}
// The thread's part of a row, for wg_stat.
__device__ __forceinline__ Stat<double> own_part(const Stat<double>* __restrict__ part, int64_t row, int parts) {
    return (int)threadIdx.x < parts ? part[row * parts + threadIdx.x] : Stat<double>{kNegInf, 0.0};
}

__device__ __forceinline__ Stat<float> float_stat(Stat<double> v) { return Stat<float>{v.m, (float)v.s}; }

// l (0 where the row is not counted) and the row's statistics, read from the
// logits or (SPLIT) joined from its parts; a counted target past the vocabulary
// makes its l NaN. L: float, or double for sums over answers; logp32 (may be null):
// those as floats, too.
template <typename T, int NT, typename L, bool SPLIT>
__global__ __launch_bounds__(NT) void lp_rows_k(int vocab, const T* __restrict__ logits,
                                                const uint32_t* __restrict__ targets, int64_t ignore_index, LpScale k,
                                                const Stat<double>* __restrict__ part, int parts, L* __restrict__ logp,
                                                float* __restrict__ logp32, RowStat* __restrict__ stats) {
    __shared__ Stat<double> red[NT / 64];
    const int64_t row = blockIdx.x;
    const uint32_t t = targets[row];
    if (!counted(t, ignore_index)) {
        if (threadIdx.x == 0) {
            logp[row] = 0;
            if (logp32) logp32[row] = 0.f;
            if (stats) stats[row] = RowStat{0.f, 1.f};
        }
        return;
    }
    const T* xr = logits + row * vocab;
    const uint32_t xt = raw_load(xr, t < (uint32_t)vocab ? t : 0);
    Stat<double> v;
    if constexpr (SPLIT) v = own_part(part, row, parts);
    else v = row_stat<T, NT, double, typename std::conditional<sizeof(T) == 4, double, L>::type>(xr, vocab, k);
    v = wg_stat<NT, double>(v, k, red);
    if (threadIdx.x == 0) {
        const double x = t < (uint32_t)vocab ? from_raw<T>(xt) : __builtin_nanf("");
        const double l = (x - (double)v.m) * k.inv_t64 - log(v.s);
        logp[row] = (L)l;
        if (logp32) logp32[row] = (float)l;
        if (stats) stats[row] = RowStat{v.m, (float)v.s};
    }
}

// ------------------------------------------------------------- preference
// A sequence's score and the factor of its tokens, from the sums over its
// counted tokens.
__device__ __forceinline__ void preference_score(const mc_preference_desc& d, int64_t q, double sum, double n,
                                                 double* score, float* inv_n, float* rewards) {
    const double inv = d.average && n > 0.0 ? 1.0 / n : 1.0;
    score[q] = sum * inv;
    inv_n[q] = (float)inv;
    if (rewards) rewards[q] = (float)(d.beta * (sum * inv));
}
// The thread's tokens at, at + step, .. of sequence q, eight loaded together.
__device__ __forceinline__ void preference_sum(const mc_preference_desc& d, int64_t q, int at, int step,
                                               const uint32_t* targets, const double* logp, const float* ref,
                                               double (&v)[2]) {
    constexpr int U = 8;
    const int64_t first = q * d.seq;
    for (int64_t i0 = at; i0 < d.seq; i0 += U * step) {
        uint32_t t[U];
        double l[U];
        float r[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t row = first + (i0 + u * step < d.seq ? i0 + u * step : i0);
            t[u] = targets[row];
            l[u] = logp[row];
            r[u] = ref ? ref[row] : 0.f;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool on = i0 + u * step < d.seq && counted(t[u], d.ignore_index);
            v[0] += on ? l[u] - (double)r[u] : 0.0;
            v[1] += on ? 1.0 : 0.0;
        }
    }
}

// The pairs' losses and each sequence's dloss/dl, by the workgroup's NT threads.
template <int NT>
__device__ __forceinline__ void preference_pairs(const mc_preference_desc& d, const double* score, const float* inv_n,
                                                 double (*red)[2], float* loss, float* dseq) {
    double sum[2] = {0.0, 0.0};
    const double beta = d.beta, eps = d.label_smoothing, pairs = (double)d.pairs;
    for (int64_t i = threadIdx.x; i < d.pairs; i += NT) {
        const double diff = score[i] - score[d.pairs + i];
        double l, dd;
        if (d.kind == MC_PREF_SQUARED) {
            const double off = diff - 0.5 / beta;
            l = off * off;
            dd = 2.0 * off;
        } else {
            const double z = beta * diff - (double)d.margin;
            if (d.kind == MC_PREF_HINGE) {
                l = z < 1.0 ? 1.0 - z : z >= 1.0 ? 0.0 : z;  // a NaN stays one
                dd = z < 1.0 ? -beta : z >= 1.0 ? 0.0 : z;
            } else {
                // -log sigma(z) and -log sigma(-z) without overflow, from exp(-|z|)
                const double e = exp(-fabs(z)), tail = log1p(e);
                const double up = z < 0.0 ? tail - z : tail, down = z > 0.0 ? tail + z : tail;
                const double sig = (z < 0.0 ? e : 1.0) / (1.0 + e), sig_neg = (z < 0.0 ? 1.0 : e) / (1.0 + e);
                l = (1.0 - eps) * up + (eps != 0.0 ? eps * down : 0.0);
                dd = beta * (eps * sig - (1.0 - eps) * sig_neg);
            }
        }
        sum[0] += l;
        if (dseq) {
            dseq[i] = (float)(dd / pairs * (double)inv_n[i]);
            dseq[d.pairs + i] = (float)(-dd / pairs * (double)inv_n[d.pairs + i]);
        }
    }
    wg_sum_f64<NT>(sum, red);
    if (threadIdx.x == 0) loss[0] = (float)(sum[0] / pairs);
}

// All in one workgroup, a wave per sequence or several: for few sequences, whose
// tokens it would walk in rounds else. The whole forward over 64 logits, us, so /
// as scores and pairs: 2 sequences of 128 tokens 7.0 / 8.2, 4 of 500 9.4 / 9.6, 40
// of 50 11.4 / 9.7, 100 of 20 18.5 / 9.8.
constexpr int kOneGroupSeqs = 16;
template <int NT>
__global__ __launch_bounds__(NT) void preference_one_k(mc_preference_desc d, const uint32_t* __restrict__ targets,
                                                       const double* __restrict__ logp, const float* __restrict__ ref,
                                                       float* __restrict__ loss, float* __restrict__ rewards,
                                                       float* __restrict__ dseq) {
    constexpr int W = NT / 64;
    __shared__ double red[W][2];
    __shared__ double score[kOneGroupSeqs];
    __shared__ float inv_n[kOneGroupSeqs];
    if (2 * d.pairs < W) {  // the waves of a sequence, side by side
        const int share = W / (int)(2 * d.pairs), q = wave_id() / share;
        double v[2] = {0.0, 0.0};
        if (q < 2 * d.pairs)
            preference_sum(d, q, wave_id() % share * kWave + lane_id(), share * kWave, targets, logp, ref, v);
        v[0] = wave_sum(v[0]);
        v[1] = wave_sum(v[1]);
        if (lane_id() == 0) {
            red[wave_id()][0] = v[0];
            red[wave_id()][1] = v[1];
        }
        __syncthreads();
        if ((int)threadIdx.x < 2 * d.pairs) {
            v[0] = v[1] = 0.0;
            for (int w = 0; w < share; ++w) {
                v[0] += red[threadIdx.x * share + w][0];
                v[1] += red[threadIdx.x * share + w][1];
            }
            preference_score(d, threadIdx.x, v[0], v[1], score, inv_n, rewards);
        }
        __syncthreads();
        return preference_pairs<NT>(d, score, inv_n, red, loss, dseq);
    }
    for (int64_t q = wave_id(); q < 2 * d.pairs; q += W) {
        double v[2] = {0.0, 0.0};
        preference_sum(d, q, lane_id(), kWave, targets, logp, ref, v);
        v[0] = wave_sum(v[0]);
        v[1] = wave_sum(v[1]);
        if (lane_id() == 0) preference_score(d, q, v[0], v[1], score, inv_n, rewards);
    }
    __syncthreads();
    preference_pairs<NT>(d, score, inv_n, red, loss, dseq);
}

// The scores alone, a workgroup per sequence, and the pairs.
__global__ __launch_bounds__(256) void preference_scores_k(mc_preference_desc d, const uint32_t* __restrict__ targets,
                                                           const double* __restrict__ logp,
                                                           const float* __restrict__ ref, double* __restrict__ score,
                                                           float* __restrict__ inv_n, float* __restrict__ rewards) {
    __shared__ double red[4][2];
    const int64_t q = blockIdx.x;
    double v[2] = {0.0, 0.0};
    preference_sum(d, q, (int)threadIdx.x, 256, targets, logp, ref, v);
    wg_sum_f64<256>(v, red);
    if (threadIdx.x == 0) preference_score(d, q, v[0], v[1], score, inv_n, rewards);
}
template <int NT>
__global__ __launch_bounds__(NT) void preference_pairs_k(mc_preference_desc d, const double* __restrict__ score,
                                                         const float* __restrict__ inv_n, float* __restrict__ loss,
                                                         float* __restrict__ dseq) {
    __shared__ double red[NT / 64][2];
    preference_pairs<NT>(d, score, inv_n, red, loss, dseq);
}

// ------------------------------------------------------------------ policy
// Counted tokens of each sequence: NT = 64, a wave for each, or a workgroup of NT
// threads, which keep eight loads each in flight.
template <int NT>
__global__ __launch_bounds__(NT == 64 ? 256 : NT) void seq_counts_k(int64_t batch, int64_t seq,
                                                                    const uint32_t* __restrict__ targets,
                                                                    int64_t ignore_index, uint32_t* __restrict__ n) {
    constexpr int U = 8;
    __shared__ uint32_t red[NT / 64];
    const int64_t q = NT == 64 ? (int64_t)blockIdx.x * 4 + wave_id() : (int64_t)blockIdx.x;
    if (q >= batch) return;
    const uint32_t* t = targets + q * seq;
    uint32_t c = 0;
    for (int64_t i = NT == 64 ? lane_id() : (int)threadIdx.x; i < seq; i += U * NT) {
        uint32_t v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = t[i + u * NT < seq ? i + u * NT : i];
#pragma unroll
        for (int u = 0; u < U; ++u) c += i + u * NT < seq && counted(v[u], ignore_index) ? 1u : 0u;
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) c += (uint32_t)__shfl_xor((int)c, o, kWave);
    if constexpr (NT > 64) {
        if (lane_id() == 0) red[wave_id()] = c;
        __syncthreads();
        c = 0;
        for (int w = 0; w < NT / 64; ++w) c += red[w];
    }
    if (NT == 64 ? lane_id() == 0 : threadIdx.x == 0) n[q] = c;
}

// A token's terms: -min(r A, clip(r) A) + kl_coef kl, dl, kl and whether the
// clipped side holds (then the surrogate has no gradient).
struct PolicyTerm {
    float term, dl, kl, clipped;
};
struct PolicyInputs {
    float A, old, ref;
    bool has_old, has_ref;
};
// Unconditional, from the targets where there are none: a load under a condition is
// waited for at its end.
__device__ __forceinline__ PolicyInputs policy_inputs(const mc_policy_desc& d, const uint32_t* targets,
                                                      const float* adv, const float* old, const float* ref,
                                                      int64_t row, uint32_t seq) {
    const float* spare = reinterpret_cast<const float*>(targets);
    return PolicyInputs{adv[d.per_token_advantages ? row : seq], (old ? old : spare)[row], (ref ? ref : spare)[row],
                        old != nullptr, ref != nullptr};
}
// l in double: its differences to the other policies' are small against it, the KL
// term's gradient is one of them, and terms of both signs cancel in the loss. The
// kernels for the loss and for the gradient take the same l, or at a border the one
// would clip a token and the other not.
__device__ __forceinline__ PolicyTerm policy_term(const mc_policy_desc& d, double l, const PolicyInputs& in) {
    PolicyTerm p;
    const float A = in.A;
    const float r = in.has_old ? expf((float)(l - (double)in.old)) : l == l ? 1.f : (float)l;
    const float held = fminf(fmaxf(r, 1.f - d.clip_low), 1.f + d.clip_high);
    const bool clipped = held * A < r * A;
    p.clipped = clipped ? 1.f : 0.f;
    p.term = -(clipped ? held * A : r * A);
    p.dl = clipped ? 0.f : -r * A;
    p.kl = 0.f;
    if (in.has_ref) {
        const float u = (float)((double)in.ref - l), g = expm1f(u);
        p.kl = g - u;
        if (d.kl_coef != 0.f) {
            p.term = fmaf(d.kl_coef, p.kl, p.term);
            p.dl = fmaf(-d.kl_coef, g, p.dl);
        }
    }
    return p;
}

__device__ __forceinline__ void policy_finish(const mc_policy_desc& d, bool by_seq, const double (&v)[4],
                                              float* __restrict__ loss, float* __restrict__ metrics,
                                              float* __restrict__ dlp) {
    const double N = by_seq ? (double)d.batch : v[3];  // no token at all: 0 / 0, a NaN loss
    loss[0] = (float)(v[0] / N);
    if (metrics) {
        metrics[0] = (float)(v[1] / N);
        metrics[1] = (float)(v[2] / N);
    }
    if (dlp) dlp[d.batch * d.seq] = (float)(1.0 / N);
}
// Workgroup b: rows b * chunk ..; sums of the terms, the KL, the clipped tokens
// and the counted ones. n: counted tokens of each sequence where the mean runs
// over sequences. dlp: dloss/dl but for the factor at dlp[rows], which is known
// only at the end. One workgroup ends here; of several, policy_join_k adds the
// sums in order.
template <int NT>
__global__ __launch_bounds__(NT) void policy_k(mc_policy_desc d, int64_t chunk, const uint32_t* __restrict__ targets,
                                               const double* __restrict__ logp, const float* __restrict__ adv,
                                               const float* __restrict__ old, const float* __restrict__ ref,
                                               const uint32_t* __restrict__ n, double (*part)[4],
                                               float* __restrict__ loss, float* __restrict__ metrics,
                                               float* __restrict__ dlp) {
    __shared__ double red[NT / 64][4];
    const int64_t rows = d.batch * d.seq, r0 = (int64_t)blockIdx.x * chunk;
    const int64_t r1 = r0 + chunk < rows ? r0 + chunk : rows;
    double v[4] = {0.0, 0.0, 0.0, 0.0};
    constexpr int U = 4;  // rows whose loads are in flight together
    for (int64_t row0 = r0 + threadIdx.x; row0 < r1; row0 += U * NT) {
        uint32_t t[U], nq[U];
        double l[U];
        PolicyInputs in[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t row = row0 + u * NT < r1 ? row0 + u * NT : row0;
            const uint32_t q = (uint32_t)row / (uint32_t)d.seq;
            t[u] = targets[row];
            l[u] = logp[row];
            in[u] = policy_inputs(d, targets, adv, old, ref, row, q);
            nq[u] = (n ? n : targets)[q];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t row = row0 + u * NT;
            if (row >= r1) break;
            float dl = 0.f;
            if (counted(t[u], d.ignore_index)) {
                const PolicyTerm p = policy_term(d, l[u], in[u]);
                const double w = n ? 1.0 / (double)nq[u] : 1.0;
                v[0] += w * (double)p.term;
                v[1] += w * (double)p.kl;
                v[2] += w * (double)p.clipped;
                v[3] += 1.0;
                dl = (float)(w * (double)p.dl);
            }
            if (dlp) dlp[row] = dl;
        }
    }
    wg_sum_f64<NT>(v, red);
    if (threadIdx.x != 0) return;
    if (gridDim.x == 1) return policy_finish(d, n != nullptr, v, loss, metrics, dlp);
#pragma unroll
    for (int c = 0; c < 4; ++c) part[blockIdx.x][c] = v[c];
}
constexpr int kSumGroups = 256;  // at most, a thread of the join for each
__global__ __launch_bounds__(kSumGroups) void policy_join_k(mc_policy_desc d, bool by_seq, int groups,
                                                            const double (*part)[4], float* __restrict__ loss,
                                                            float* __restrict__ metrics, float* __restrict__ dlp) {
    __shared__ double red[kSumGroups / 64][4];
    double v[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) v[c] = (int)threadIdx.x < groups ? part[threadIdx.x][c] : 0.0;
    wg_sum_f64<kSumGroups>(v, red);
    if (threadIdx.x == 0) policy_finish(d, by_seq, v, loss, metrics, dlp);
}

// ------------------------------------------------------------ distillation
// A row's teacher. One wave forms p_k = e_k / s and their sum (Top), a thread per
// entry adds its id and the student's logit (TopEntry), and behind a barrier of the
// kernel one wave forms sum p_k (log p_k - log q_k) from those and the row's
// statistics (teacher_value). Before that barrier the teacher needs no other: one
// behind the loads of a held row would have every wave wait until the last has issued
// its own, which is most of the time that they take (2036 bf16 rows of 151936, 283 us
// in place of 248). An entry is left out where its logit is -inf.
// The logarithms are in double: their difference is small against them, the terms
// cancel until about its square is left, and 1 / T as a float has an error of one
// sign. With floats the loss of 2000 rows 5e-3 from a teacher of logits near 110 at
// T = 1.5 was 1.7e-5 in place of 1.2e-5.
// N: as many entries as the workgroup has threads, and all that there may be at most.
template <int NT> struct Teacher {
    static constexpr int N = NT < kDistillMaxTop ? NT : kDistillMaxTop;
    int id[N];               // -1: left out
    float p[N], t[N], x[N];  // t: the teacher's logit, x the student's
    double s;                // log p_k = (t_k - m) / T - lse - log s
    float m, lse, P;         // P: sum p
    int bad;                 // an id past the vocabulary: the row is NaN
};
// 2^y to a float: of y's leading part, and the rest as a factor.
__device__ __forceinline__ float exp2_of(double y) {
    const float hi = (float)y, e = exp2_hw(hi);
    return hi > -200.f ? fmaf(e, (float)(y - (double)hi) * 0.693147181f, e) : e;  // far below, the rest may be infinite
}
struct TopEntry {
    float t;
    int id;
    // Unconditional: see HeldRow.
    __device__ __forceinline__ void load(const mc_distill_desc& d, int64_t row, const int32_t* __restrict__ ids,
                                         const float* __restrict__ tl) {
        const int64_t at = row * d.top + ((int)threadIdx.x < d.top ? (int)threadIdx.x : 0);
        t = tl[at];
        id = ids[at];
    }
    __device__ __forceinline__ void open() {
        if (t == kNegInf) id = -1;
    }
    // The bits of the student's logit at the entry.
    template <typename T> __device__ __forceinline__ uint32_t logit(const T* __restrict__ xr, int vocab) const {
        return raw_load(xr, (unsigned)id < (unsigned)vocab ? id : 0);
    }
    template <typename Te> __device__ __forceinline__ void put(const mc_distill_desc& d, float x, Te& te) const {
        if ((int)threadIdx.x >= d.top) return;
        te.id[threadIdx.x] = id;
        te.x[threadIdx.x] = x;
    }
};
// The entries lane, lane + 64, .. for the first wave; the others have none.
template <int NT> struct Top {
    typedef Teacher<NT> Te;
    static constexpr int C = Te::N / kWave;
    float t[C];
    int id[C];
    // All past 64 or none of them: without a branch between them they overlap.
    static __device__ __forceinline__ bool here(const mc_distill_desc& d, int c) {
        return c != 1 || (wave_id() == 0 && d.top > kWave);
    }
    // Before the row's loads; the first 64 are the wave's own.
    __device__ __forceinline__ void load(const mc_distill_desc& d, int64_t row, const int32_t* __restrict__ ids,
                                         const float* __restrict__ tl, const TopEntry& own) {
        t[0] = own.t;
        id[0] = own.id;
#pragma unroll
        for (int c = 1; c < C; ++c) {
            if (!here(d, c)) break;
            const int i = c * kWave + lane_id();
            const int64_t at = row * d.top + (i < d.top ? i : 0);
            t[c] = tl[at];
            id[c] = ids[at];
        }
    }
    // lse: the teacher's log-sum-exp, or NULL: over these entries.
    __device__ __forceinline__ void form(const mc_distill_desc& d, const float* lse, int64_t row, LpScale k, Te& te) {
        if (wave_id() != 0) return;
        const double log2e = 1.4426950408889634074, c64 = k.inv_t64 * log2e;
        float m = kNegInf, P = 0.f;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            if (!here(d, c)) break;
            if (c * kWave + lane_id() >= d.top) t[c] = kNegInf;
            m = fmaxf(m, t[c]);  // passes over a NaN, which then stays in the sum
        }
        m = lse ? 0.f : wave_max(m);
        const float l = lse ? lse[row] : 0.f;
        double s = 0.0;
        float e[C];
#pragma unroll
        for (int c = 0; c < C; ++c) {
            if (!here(d, c)) break;
            e[c] = exp2_of(fma((double)t[c] - (double)m, c64, -(double)l * log2e));
            if (t[c] == kNegInf) e[c] = 0.f;
            s += (double)e[c];
        }
        s = lse ? 1.0 : wave_sum(s);
        const float r = 1.f / (float)s;  // its rounding scales every p alike
        bool bad = false;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            if (!here(d, c)) break;
            const int i = c * kWave + lane_id();
            const float p = t[c] == kNegInf ? 0.f : e[c] * r;  // without an entry r is infinite
            te.t[i] = t[c];
            te.p[i] = p;
            P += p;
            bad |= p != 0.f && (id[c] < 0 || id[c] >= (int)d.vocab);
        }
        P = wave_sum(P);
        const int any = __any(bad);
        if (lane_id() == 0) {
            te.s = s;
            te.m = m;
            te.lse = l;
            te.P = P;
            te.bad = any;
        }
    }
};
// By one wave; both differences to a maximum come first, as in the rows' own sums.
template <typename Te>
__device__ __forceinline__ double teacher_value(const mc_distill_desc& d, const Te& te, Stat<double> st, LpScale k) {
    const double rest = log_ratio(te.s, st.s) + (double)te.lse;
    double v = 0.0;
#pragma unroll
    for (int c = 0; c < Te::N / kWave; ++c) {
        const int i = c * kWave + lane_id();
        if (c * kWave >= d.top) break;
        const double p = te.p[i];  // 0 past the last
        const double dt = (double)te.t[i] - (double)te.m, dx = (double)te.x[i] - (double)st.m;
        v += p == 0.0 ? 0.0 : p * fma(dt - dx, k.inv_t64, -rest);
    }
    v = wave_sum(v);
    return te.bad ? __builtin_nan("") : v;
}

// At most 64 registers: a CU then holds two rows of 1024 threads.
template <typename T, int NT, bool SPLIT>
__global__ __launch_bounds__(NT, 8) void distill_rows_k(mc_distill_desc d, const T* __restrict__ logits,
                                                        const int32_t* __restrict__ ids, const float* __restrict__ tl,
                                                        const float* __restrict__ tlse,
                                                        const uint8_t* __restrict__ mask, LpScale k,
                                                        const Stat<double>* __restrict__ part, int parts,
                                                        double* __restrict__ kl, RowStat* __restrict__ stats) {
    typedef typename std::conditional<SPLIT, double, float>::type Sum;
    __shared__ Stat<Sum> red[NT / 64];
    __shared__ Teacher<NT> te;
    const int64_t row = blockIdx.x;
    const int vocab = (int)d.vocab;
    if (mask && mask[row] == 0) {
        if (threadIdx.x == 0) {
            kl[row] = 0.0;
            if (stats) stats[row] = RowStat{0.f, 1.f};
        }
        return;
    }
    const T* xr = logits + row * vocab;
    TopEntry entry;
    entry.load(d, row, ids, tl);
    Top<NT> top;
    top.load(d, row, ids, tl, entry);
    Stat<Sum> own;
    if constexpr (SPLIT) own = own_part(part, row, parts);
    else own = row_stat<T, NT, float, float>(xr, vocab, k);
    entry.open();
    const uint32_t x = entry.logit(xr, vocab);
    top.form(d, tlse, row, k, te);
    entry.put(d, from_raw<T>(x), te);
    Stat<double> st = wg_stat<NT, double>(own, k, red);  // its barrier is the teacher's, too
    if (wave_id() != 0) return;
    asm volatile("" : "+v"(st.s), "+v"(st.m) : : "memory");  // or the next reads are made among wg_stat's
    const double v = teacher_value(d, te, st, k);
    if (threadIdx.x == 0) {
        kl[row] = v;
        if (stats) stats[row] = RowStat{st.m, (float)st.s};
    }
}

// loss = T^2 sum kl / counted rows; scale = T / counted rows. Workgroups as
// policy_k's.
__device__ __forceinline__ void distill_finish(double T, const double (&v)[2], float* __restrict__ loss,
                                               float* __restrict__ scale) {
    loss[0] = (float)(T * T * v[0] / v[1]);  // no row counted: 0 / 0, a NaN loss
    if (scale) scale[0] = (float)(T / v[1]);
}
template <int NT>
__global__ __launch_bounds__(NT) void distill_final_k(int64_t rows, int64_t chunk, float temperature,
                                                      const uint8_t* __restrict__ mask, const double* __restrict__ kl,
                                                      double (*part)[2], float* __restrict__ loss,
                                                      float* __restrict__ scale) {
    __shared__ double red[NT / 64][2];
    const int64_t r0 = (int64_t)blockIdx.x * chunk;
    const int64_t r1 = r0 + chunk < rows ? r0 + chunk : rows;
    double v[2] = {0.0, 0.0};
    constexpr int U = 4;
    for (int64_t row0 = r0 + threadIdx.x; row0 < r1; row0 += U * NT) {
        double x[U];
        bool on[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t row = row0 + u * NT < r1 ? row0 + u * NT : row0;
            x[u] = kl[row];
            on[u] = row0 + u * NT < r1 && (!mask || mask[row] != 0);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            v[0] += on[u] ? x[u] : 0.0;
            v[1] += on[u] ? 1.0 : 0.0;
        }
    }
    wg_sum_f64<NT>(v, red);
    if (threadIdx.x != 0) return;
    if (gridDim.x == 1) return distill_finish(temperature, v, loss, scale);
    part[blockIdx.x][0] = v[0];
    part[blockIdx.x][1] = v[1];
}
__global__ __launch_bounds__(kSumGroups) void distill_join_k(float temperature, int groups, const double (*part)[2],
                                                             float* __restrict__ loss, float* __restrict__ scale) {
    __shared__ double red[kSumGroups / 64][2];
    double v[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) v[c] = (int)threadIdx.x < groups ? part[threadIdx.x][c] : 0.0;
    wg_sum_f64<kSumGroups>(v, red);
    if (threadIdx.x == 0) distill_finish(temperature, v, loss, scale);
}

// ---------------------------------------------------------------- gradients
// A row's gradient is a q, q = 2^((x - m) c) / s, but for the elements of the
// target or of the teacher's entries. Those are stored once more by the thread
// that stored their vector, behind it: stores of a thread stay in order, so that
// needs no barrier, and the loop over the row no test. Rows run backwards, and
// stream stores past the caches, for the reasons of the cross entropy's backward.
struct RowGrad {
    float a, m, c;  // a: with 1 / s
    __device__ __forceinline__ float operator()(float x) const { return a * exp2_hw((x - m) * c); }
};
__device__ __forceinline__ RowGrad row_grad(float a, RowStat st, float c) { return RowGrad{a / st.s, st.m, c}; }

// How vectors are stored: in the caches, past them, or at any element, where the
// gradients do not start at the logits' place in a vector. Then the fwd_bwd calls
// run as a forward and a backward (as a second way to store a held row this cost
// the longest 60 registers): 2036 bf16 rows of 151936 backward 251 us, element by
// element 456, aligned 238; policy 362, 550, 242.
enum class Store { kCached, kStream, kAny };
template <typename T, int N> __device__ __forceinline__ void store16(T* p, const float (&v)[N], Store how) {
    if (how == Store::kStream) store_nt16(p, v);
    else if (how == Store::kAny) store_any16(p, v);
    else Vec16<T>::store(p, v);
}

// The threads of a row: those of the gridDim.y workgroups that share it.
struct RowThreads {
    int self, count;
};
template <int NT> __device__ __forceinline__ RowThreads row_threads() {
    return RowThreads{(int)(blockIdx.y * NT + threadIdx.x), (int)(gridDim.y * NT)};
}

// Vectors c, c - step, .. down to lo: U requested at a time, the last together.
template <typename T, int U>
__device__ __forceinline__ void write_vecs(const T* __restrict__ xv, T* __restrict__ dv, int c, int step, int lo,
                                           Store how, RowGrad grad) {
    constexpr int N = Vec16<T>::N;
    auto group = [&](auto whole) {
        float v[U][N];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int at = c - u * step;
            Vec16<T>::load(xv + (int64_t)(decltype(whole)::value || at >= lo ? at : c) * N, v[u]);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int at = c - u * step;
            if (!decltype(whole)::value && at < lo) break;
#pragma unroll
            for (int e = 0; e < N; ++e) v[u][e] = grad(v[u][e]);
            store16(dv + (int64_t)at * N, v[u], how);
        }
    };
    for (; c >= lo + (U - 1) * step; c -= U * step) group(std::true_type{});
    if (c >= lo) group(std::false_type{});
}
template <typename T>
__device__ __forceinline__ void write_row(const T* __restrict__ xr, T* __restrict__ dr, int vocab, Store how,
                                          RowThreads th, RowGrad grad) {
    const RowSpan<T> span(xr, vocab);
    write_vecs<T, 4>(xr + span.head, dr + span.head, (int)span.nvec - 1 - th.self, th.count, 0, how, grad);
    const int64_t j = span.edge(th.self, vocab);
    if (j >= 0) Elem<T>::store(dr, j, grad(Elem<T>::load(xr, j)));
}
// The thread that stores element j: its vector's, or its edge's.
template <int N> __device__ __forceinline__ int owner_of(int j, int head, int nvec, int threads) {
    if (j < head) return j;
    const int c = (j - head) / N;
    return c < nvec ? (nvec - 1 - c) % threads : N + (j - head - nvec * N);
}

template <typename T>
__device__ __forceinline__ void zero_row(T* __restrict__ dr, int vocab, Store how, RowThreads th) {
    constexpr int N = Vec16<T>::N;
    const RowSpan<T> span(dr, vocab);  // its own vectors
    const float z[N] = {};
    for (int c = th.self; c < (int)span.nvec; c += th.count) {
        T* p = dr + span.head + (int64_t)c * N;
        if (how == Store::kStream) store_nt16(p, z);
        else Vec16<T>::store(p, z);
    }
    const int64_t j = span.edge(th.self, vocab);
    if (j >= 0) Elem<T>::store(dr, j, 0.f);
}

// Which of a teacher's entries each thread stores: a bit for entry k in word
// k / 32 of its owner.
template <int NT> struct TopOwners {
    typedef Teacher<NT> Te;
    static constexpr int W = Te::N / 32;
    uint32_t bits[W * NT];

    // Before the entries are there, with a barrier behind it.
    __device__ __forceinline__ void clear(int top) {
        for (int i = threadIdx.x; i < (top + 31) / 32 * NT; i += NT) bits[i] = 0;
    }
    // Thread k puts in entry k, whose element the row's thread `owner` stores; the
    // workgroup's own are from first on. A barrier before the patch.
    __device__ __forceinline__ void insert(int owner, int first) {
        const int k = threadIdx.x;
        if ((unsigned)(owner - first) < (unsigned)NT) atomicOr(&bits[(k >> 5) * NT + owner - first], 1u << (k & 31));
    }
    // The thread's entries' elements, once the row is stored: w times the entry's p
    // less. Entries of one id come in the order of k, each with the sum so far, so
    // that the last one leaves the whole: of up to four entries the sums before are
    // in registers, more than that (several in one thread's vectors, or one id many
    // times) are searched. Searching for every thread took 108 us in place of 97 for
    // 2000 rows of 50257 bf16 logits and 256 entries, 63 in place of 43 for 4000 of
    // 8000.
    template <typename T>
    __device__ __forceinline__ void patch(const Te& te, int top, T* __restrict__ dr, RowGrad grad, float w) const {
        constexpr int kKept = 3;
        uint32_t own[W];
        int count = 0;
#pragma unroll
        for (int i = 0; i < W; ++i) {
            own[i] = 32 * i < top ? bits[i * NT + threadIdx.x] : 0;
            count += __popc(own[i]);
        }
        int ids[kKept] = {-1, -1, -1};
        float sums[kKept] = {};
#pragma unroll
        for (int i = 0; i < W; ++i)
            for (uint32_t b = own[i]; b; b &= b - 1) {
                const int k = 32 * i + __ffs(b) - 1, id = te.id[k];
                float p = te.p[k];
                if (count <= kKept + 1) {
                    float before = 0.f;
#pragma unroll
                    for (int o = kKept - 1; o >= 0; --o) before = ids[o] == id ? sums[o] : before;
                    p += before;
#pragma unroll
                    for (int o = kKept - 1; o > 0; --o) {
                        ids[o] = ids[o - 1];
                        sums[o] = sums[o - 1];
                    }
                    ids[0] = id;
                    sums[0] = p;
                } else {
                    p = 0.f;
                    for (int o = 0; o <= k; ++o) p += te.id[o] == id ? te.p[o] : 0.f;
                }
                Elem<T>::store(dr, id, grad(te.x[k]) - w * p);
            }
    }
};

// dlogits of a loss over l: g ([j = t] - q_j) / T, g = dl of the row (or of its
// sequence) times the optional device scalars.
template <typename T, int NT>
__global__ __launch_bounds__(NT) void lp_bwd_k(int64_t rows, int vocab, Store how,
                                               const T* __restrict__ logits, const uint32_t* __restrict__ targets,
                                               int64_t ignore_index, LpScale k, const RowStat* __restrict__ stats,
                                               const float* __restrict__ dl, uint32_t seq,
                                               const float* __restrict__ scale, const float* __restrict__ dloss,
                                               T* __restrict__ dlogits) {
    const RowThreads th = row_threads<NT>();
    const int64_t row = rows - 1 - (int64_t)blockIdx.x;
    T* dr = dlogits + row * vocab;
    const uint32_t t = targets[row];
    float g = 0.f;
    if (counted(t, ignore_index)) {
        g = dl[seq ? (uint32_t)row / seq : row];
        if (scale) g *= scale[0];
        if (dloss) g *= dloss[0];
        if (t >= (uint32_t)vocab) g = __builtin_nanf("");
    }
    if (g == 0.f) {
        zero_row(dr, vocab, how, th);
        return;
    }
    g *= k.inv_t;
    const T* xr = logits + row * vocab;
    const RowGrad grad = row_grad(-g, stats[row], k.c);
    write_row(xr, dr, vocab, how, th, grad);
    const RowSpan<T> span(xr, vocab);
    if (t < (uint32_t)vocab &&
        owner_of<Vec16<T>::N>((int)t, (int)span.head, (int)span.nvec, th.count) == th.self)
        Elem<T>::store(dr, t, grad(Elem<T>::load(xr, t)) + g);
}

template <typename T, int NT>
__global__ __launch_bounds__(NT) void distill_bwd_k(mc_distill_desc d, Store how,
                                                    const T* __restrict__ logits, const int32_t* __restrict__ ids,
                                                    const float* __restrict__ tl, const float* __restrict__ tlse,
                                                    const uint8_t* __restrict__ mask, LpScale k,
                                                    const RowStat* __restrict__ stats, const float* __restrict__ scale,
                                                    const float* __restrict__ dloss, T* __restrict__ dlogits) {
    constexpr int N = Vec16<T>::N;
    __shared__ Teacher<NT> te;
    __shared__ TopOwners<NT> owners;
    const RowThreads th = row_threads<NT>();
    const int64_t row = d.rows - 1 - (int64_t)blockIdx.x;
    const int vocab = (int)d.vocab;
    T* dr = dlogits + row * vocab;
    if (mask && mask[row] == 0) {
        zero_row(dr, vocab, how, th);
        return;
    }
    owners.clear(d.top);
    const T* xr = logits + row * vocab;
    const RowSpan<T> span(xr, vocab);
    const RowStat v = stats[row];
    TopEntry entry;
    entry.load(d, row, ids, tl);
    Top<NT> top;
    top.load(d, row, ids, tl, entry);
    entry.open();
    const uint32_t x = entry.logit(xr, vocab);
    __syncthreads();
    if ((int)threadIdx.x < d.top && (unsigned)entry.id < (unsigned)vocab)
        owners.insert(owner_of<N>(entry.id, (int)span.head, (int)span.nvec, th.count), (int)(blockIdx.y * NT));
    top.form(d, tlse, row, k, te);
    entry.put(d, from_raw<T>(x), te);
    __syncthreads();
    float w = scale[0] * (dloss ? dloss[0] : 1.f);
    if (te.bad) w = __builtin_nanf("");
    if (te.P == 0.f || w == 0.f) {
        zero_row(dr, vocab, how, th);
        return;
    }
    const RowGrad grad = row_grad(w * te.P, v, k.c);
    write_row(xr, dr, vocab, how, th, grad);
    owners.patch(te, d.top, dr, grad, w);
}

// ------------------------------------------- value and gradient in one read
// A row held in registers, vector u * NT + t of it in thread t, so that the
// statistics and the gradient come from one read: 1024 threads hold up to 304 KiB, a
// row per CU, the smaller shapes several rows. Bound by HBM, with the reads of some
// CUs beside the writes of others: 2036 bf16 rows of 151936 take 246 us, 325
// as lp_rows_k and lp_bwd_k, whose second read the cache meets in part. All the
// loads are in flight at once, and
// the statistics take them as they come, so whatever else a kernel loads comes
// before them (loads return in order). Loads past the last vector give zeros
// and stores there are dropped. The edges' elements are in the first 2 N
// threads, as their bits.
// Nothing is loaded under a condition, or every wait would be for the path with
// the fewest loads, that is for all of them.
// REST: rows of any length. What lies past NT NV vectors is read twice, its end,
// which the cache still has, first.
template <typename T, int NT, int NV, bool REST> struct HeldRow {
    static constexpr int N = Vec16<T>::N, G = 16 / N;  // vectors reduced at a time
    i32x4 q[NV];
    uint32_t edge;
    int head, nvec, j;  // j: the edge element, or -1
    const T* xv;        // the first vector

    // The thread that stores element `at`: its vector's, or its edge's.
    __device__ __forceinline__ int owner(int at) const {
        if (at < head) return at;
        const int c = (at - head) / N;
        return c < nvec ? c & (NT - 1) : N + (at - head - nvec * N);
    }
    __device__ __forceinline__ void load(const T* __restrict__ xr, int vocab, const Stat<double>*, int64_t,
                                         RowThreads) {
        const RowSpan<T> span(xr, vocab);
        head = (int)span.head;
        nvec = (int)span.nvec;
        j = (int)span.edge((int)threadIdx.x, vocab);
        edge = raw_load(xr, j < 0 ? 0 : j);
        xv = xr + head;
        const __amdgpu_buffer_rsrc_t r = make_rsrc(xv, (int64_t)(REST ? NT * NV : nvec) * 16);
#pragma unroll
        for (int u = 0; u < NV; ++u) {
            __builtin_amdgcn_sched_barrier(0);  // in the order of their use
            q[u] = buf_load16(r, (uint32_t)(u * NT + (int)threadIdx.x) * 16u);
        }
        __builtin_amdgcn_sched_barrier(0);
    }
    __device__ __forceinline__ Stat<float> stat(LpScale k) const {
        float m = kNegInf, s = 0.f;
#pragma unroll
        for (int u0 = 0; u0 < NV; u0 += G) {
            if (!REST && u0 * NT >= nvec) break;
            float v[G][N];
            float vm = kNegInf;
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const int u = u0 + g;
                if (u < NV) BVec<T>::unpack(q[u], v[g]);
                if (u >= NV || (!REST && (u + 1) * NT > nvec && u * NT + (int)threadIdx.x >= nvec)) {
#pragma unroll
                    for (int e = 0; e < N; ++e) v[g][e] = kNegInf;
                }
#pragma unroll
                for (int e = 0; e < N; ++e) vm = fmaxf(vm, v[g][e]);
            }
            if (vm > m) {
                s *= exp_of(m - vm, k);
                m = vm;
            }
            const float base = base_of(m);
            float ps[G];
#pragma unroll
            for (int g = 0; g < G; ++g) {
                ps[g] = 0.f;
#pragma unroll
                for (int e = 0; e < N; ++e) ps[g] += term_of(v[g][e], base, k);
            }
            s += G == 4 ? (ps[0] + ps[1]) + (ps[G - 2] + ps[G - 1]) : ps[0] + ps[1];
        }
        Stat<float> st{m, s};
        if constexpr (REST)
            st = stat_join(st, vec_stat<T, NT, float, G>(xv, NT * NV + (int)threadIdx.x, nvec, k), k);
        if (j >= 0) {
            const float x = from_raw<T>(edge);
            st = stat_join(st, Stat<float>{x, term_of(x, base_of(x), k)}, k);
        }
        return st;
    }
    // into the gradient's row dr, which starts like the logits'
    __device__ __forceinline__ void store(T* __restrict__ dr, Store how, RowGrad grad) const {
        if constexpr (REST)
            write_vecs<T, G>(xv, dr + head, (int)threadIdx.x + (nvec - 1 - (int)threadIdx.x) / NT * NT, NT, NT * NV,
                             how, grad);
        const __amdgpu_buffer_rsrc_t r = make_rsrc(dr + head, (int64_t)(REST ? NT * NV : nvec) * 16);
        uint32_t at = threadIdx.x * 16u;
        asm volatile("" : "+v"(at));  // or the loads' NV offsets are held for the stores
#pragma unroll
        for (int u = 0; u < NV; ++u) {
            if (!REST && u * NT >= nvec) break;
            float v[N];
            BVec<T>::unpack(q[u], v);
#pragma unroll
            for (int e = 0; e < N; ++e) v[e] = grad(v[e]);
            if (how == Store::kStream) BVec<T>::store_nt(r, at + u * NT * 16u, v);
            else BVec<T>::store(r, at + u * NT * 16u, v);
        }
        if (j >= 0) Elem<T>::store(dr, j, grad(from_raw<T>(edge)));
    }
};

// A row of few, shared by gridDim.y workgroups: its statistics from parts_k, its
// logits read again, from the cache as a rule.
template <typename T, int NT> struct SplitRow {
    static constexpr int N = Vec16<T>::N;
    const T* xr;
    RowThreads th;
    int vocab, head, nvec;
    Stat<double> part;

    __device__ __forceinline__ int owner(int at) const { return owner_of<N>(at, head, nvec, th.count); }
    __device__ __forceinline__ void load(const T* __restrict__ xr_, int vocab_, const Stat<double>* __restrict__ parts,
                                         int64_t row, RowThreads th_) {
        const RowSpan<T> span(xr_, vocab_);
        xr = xr_;
        th = th_;
        vocab = vocab_;
        head = (int)span.head;
        nvec = (int)span.nvec;
        part = own_part(parts, row, th.count / NT);
    }
    __device__ __forceinline__ Stat<float> stat(LpScale) const { return float_stat(part); }
    __device__ __forceinline__ void store(T* __restrict__ dr, Store how, RowGrad grad) const {
        write_row(xr, dr, vocab, how, th, grad);
    }
};

// Counted tokens of 64 blocks of rows, for the weight of a token.
constexpr int kCountBlocks = 64;
__global__ __launch_bounds__(256) void counts_k(int64_t rows, int64_t chunk, const uint32_t* __restrict__ targets,
                                                const uint8_t* __restrict__ mask, int64_t ignore_index,
                                                uint32_t* __restrict__ part) {
    __shared__ uint32_t red[4];
    const int64_t r0 = (int64_t)blockIdx.x * chunk;
    const int64_t r1 = r0 + chunk < rows ? r0 + chunk : rows;
    uint32_t c = 0;
    for (int64_t row = r0 + threadIdx.x; row < r1; row += 256)
        c += (targets ? counted(targets[row], ignore_index) : mask[row] != 0) ? 1u : 0u;
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) c += (uint32_t)__shfl_xor((int)c, o, kWave);
    if (lane_id() == 0) red[threadIdx.x >> 6] = c;
    __syncthreads();
    if (threadIdx.x == 0) part[blockIdx.x] = red[0] + red[1] + red[2] + red[3];
}
// How many tokens share a row's weight: the sum of `given` counts, or where four
// loads per thread go over the `len` targets (or the mask) themselves, those, which
// saves a launch (1000 rows of 20000 bf16 23.6 us, 25.6 with it). load before the
// row's loads, put after them, a barrier of the kernel, total.
template <int NT> struct RowCount {
    static constexpr int kPer = 4;
    static_assert(NT >= kCountBlocks, "a thread for each count");
    uint32_t w[kPer], part;
    // value(i): the i-th target or mask byte; called where len is 0, too. given: where
    // n_given is 0, any address.
    template <typename F>
    __device__ __forceinline__ void load(int len, F&& value, const uint32_t* __restrict__ given, int n_given) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) w[i] = value(i * NT + (int)threadIdx.x < len ? i * NT + (int)threadIdx.x : 0);
        part = given[(int)threadIdx.x < n_given ? (int)threadIdx.x : 0];
    }
    template <typename F> __device__ __forceinline__ void put(int len, int n_given, uint32_t* red, F&& on) const {
        uint32_t c = (int)threadIdx.x < n_given ? part : 0u;
#pragma unroll
        for (int i = 0; i < kPer; ++i) c += i * NT + (int)threadIdx.x < len && on(w[i]) ? 1u : 0u;
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) c += (uint32_t)__shfl_xor((int)c, o, kWave);
        if (lane_id() == 0) red[threadIdx.x >> 6] = c;
    }
    static __device__ __forceinline__ uint32_t total(const uint32_t* red) {
        uint32_t c = 0;
#pragma unroll
        for (int k = 0; k < NT / 64; ++k) c += red[k];
        return c;
    }
};

// l, and with the token's weight its gradient. Row: HeldRow, or SplitRow with
// parts. given: n_given counts that add up to the tokens that share the weight
// (by_seq: of each sequence, one number each), or n_given 0: counted here over len
// targets. n (may be null): receives the sequences' counts.
template <typename T, int NT, typename Row>
__global__ __launch_bounds__(NT, 4) void policy_both_k(mc_policy_desc d, Store how, const T* __restrict__ logits,
                                                       const uint32_t* __restrict__ targets,
                                                       const float* __restrict__ adv, const float* __restrict__ old,
                                                       const float* __restrict__ ref,
                                                       const Stat<double>* __restrict__ parts,
                                                       const uint32_t* __restrict__ given, int n_given, int len,
                                                       bool by_seq,
                                                       uint32_t* __restrict__ n, LpScale k,
                                                       const float* __restrict__ dloss, double* __restrict__ logp,
                                                       float* __restrict__ logp32, T* __restrict__ dlogits) {
    __shared__ Stat<float> red[NT / 64];
    __shared__ uint32_t redc[NT / 64];
    const RowThreads th = row_threads<NT>();
    const int64_t row = blockIdx.x;
    const int vocab = (int)d.vocab;
    const bool writer = th.self == 0;
    T* dr = dlogits + row * vocab;
    const uint32_t t = targets[row];
    if (!counted(t, d.ignore_index)) {
        if (writer) {
            logp[row] = 0.0;
            logp32[row] = 0.f;
        }
        zero_row(dr, vocab, how, th);
        return;
    }
    const T* xr = logits + row * vocab;
    const bool in = t < (uint32_t)vocab;
    const uint32_t xt = raw_load(xr, in ? t : 0);
    const uint32_t q = (uint32_t)row / (uint32_t)d.seq;
    const PolicyInputs pin = policy_inputs(d, targets, adv, old, ref, row, q);
    const float up = dloss ? dloss[0] : 1.f;
    const uint32_t* cw = by_seq ? targets + (int64_t)q * d.seq : targets;
    RowCount<NT> count;
    count.load(len, [&](int i) { return cw[i]; }, n_given ? given + (by_seq ? q : 0) : targets, n_given);
    Row held;
    held.load(xr, vocab, parts, row, th);
    count.put(len, n_given, redc, [&](uint32_t w) { return counted(w, d.ignore_index); });
    const Stat<double> st = wg_stat<NT, double>(held.stat(k), k, red);
    const RowStat v{st.m, (float)st.s};
    const uint32_t share = count.total(redc);
    const double l = in ? (from_raw<T>(xt) - (double)v.m) * k.inv_t64 - log_of(st.s) : __builtin_nan("");
    if (writer) {
        logp[row] = l;
        logp32[row] = (float)l;
        if (n) n[q] = share;  // the same from every row of the sequence
    }
    float g = policy_term(d, l, pin).dl / (by_seq ? (float)d.batch * (float)share : (float)share) * up;
    if (g == 0.f) {
        zero_row(dr, vocab, how, th);
    } else {
        g *= k.inv_t;
        const RowGrad grad = row_grad(-g, v, k.c);
        held.store(dr, how, grad);
        if (in && held.owner((int)t) == th.self) Elem<T>::store(dr, t, grad(from_raw<T>(xt)) + g);
    }
}

// given: n_given counts of the mask, or n_given 0: counted here over len of it (0
// without a mask).
template <typename T, int NT, typename Row>
__global__ __launch_bounds__(NT, 4) void distill_both_k(mc_distill_desc d, Store how, const T* __restrict__ logits,
                                                        const int32_t* __restrict__ ids, const float* __restrict__ tl,
                                                        const float* __restrict__ tlse,
                                                        const uint8_t* __restrict__ mask,
                                                        const Stat<double>* __restrict__ parts,
                                                        const uint32_t* __restrict__ given, int n_given, int len,
                                                        LpScale k, const float* __restrict__ dloss,
                                                        double* __restrict__ kl,
                                                        T* __restrict__ dlogits) {
    __shared__ Stat<float> red[NT / 64];
    __shared__ uint32_t redc[NT / 64];
    __shared__ Teacher<NT> te;
    __shared__ TopOwners<NT> owners;
    const RowThreads th = row_threads<NT>();
    const int64_t row = blockIdx.x;
    const int vocab = (int)d.vocab;
    const bool writer = th.self == 0;
    T* dr = dlogits + row * vocab;
    if (mask && mask[row] == 0) {
        if (writer) kl[row] = 0.0;
        zero_row(dr, vocab, how, th);
        return;
    }
    const T* xr = logits + row * vocab;
    TopEntry entry;
    entry.load(d, row, ids, tl);
    Top<NT> top;
    top.load(d, row, ids, tl, entry);
    owners.clear(d.top);
    __syncthreads();
    const float up = dloss ? dloss[0] : 1.f;
    RowCount<NT> count;
    const uint8_t* cw = mask ? mask : reinterpret_cast<const uint8_t*>(xr);
    count.load(len, [&](int i) { return (uint32_t)cw[i]; },
               n_given ? given : reinterpret_cast<const uint32_t*>(ids), n_given);
    Row held;
    held.load(xr, vocab, parts, row, th);
    count.put(len, n_given, redc, [](uint32_t w) { return w != 0; });
    entry.open();
    if ((int)threadIdx.x < d.top && (unsigned)entry.id < (unsigned)vocab)
        owners.insert(held.owner(entry.id), (int)(blockIdx.y * NT));
    const uint32_t x = entry.logit(xr, vocab);
    top.form(d, tlse, row, k, te);
    const Stat<float> own = held.stat(k);
    entry.put(d, from_raw<T>(x), te);
    Stat<double> st = wg_stat<NT, double>(own, k, red);  // its barrier is the teacher's, too
    // or the next reads are made among wg_stat's, for which there are no registers
    asm volatile("" : "+v"(st.s), "+v"(st.m) : : "memory");
    float w = d.temperature / (mask ? (float)count.total(redc) : (float)d.rows) * up;
    if (blockIdx.y == 0 && wave_id() == 0) {  // while the others store
        const double value = teacher_value(d, te, st, k);
        if (writer) kl[row] = value;
    }
    if (te.bad) w = __builtin_nanf("");
    if (te.P == 0.f || w == 0.f) {
        zero_row(dr, vocab, how, th);
        return;
    }
    const RowGrad grad = row_grad(w * te.P, RowStat{st.m, (float)st.s}, k.c);
    held.store(dr, how, grad);
    owners.patch(te, d.top, dr, grad, w);
}

// c = log2(e) / T as a float below it and the rest: with c_lo > 0, x c_lo has the
// sign of x c_hi, so an infinite x gives an infinity and no NaN.
LpScale row_scale(float temperature) {
    const double c = 1.4426950408889634074 / (double)temperature;
    LpScale k;
    k.c = k.c_hi = (float)c;
    if ((double)k.c_hi >= c) k.c_hi = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, k.c_hi) - 1);
    k.c_lo = (float)(c - (double)k.c_hi);
    k.inv_t64 = 1.0 / (double)temperature;
    k.inv_t = (float)k.inv_t64;
    return k;
}

// fn(element type, threads per row)
template <typename F> void by_threads(int threads, int dtype, F&& fn) {
    auto by_dtype = [&](auto threads) {
        if (dtype == MC_F32) fn(float{}, threads);
        else fn(uint16_t{}, threads);
    };
    switch (threads) {
        case 64: return by_dtype(std::integral_constant<int, 64>{});
        case 128: return by_dtype(std::integral_constant<int, 128>{});
        case 512: return by_dtype(std::integral_constant<int, 512>{});
        case 1024: return by_dtype(std::integral_constant<int, 1024>{});
        default: return by_dtype(std::integral_constant<int, 256>{});
    }
}
int64_t row_bytes(int64_t vocab, int dtype) { return vocab * (dtype == MC_F32 ? 4 : 2); }

constexpr int kPartThreads = 256;  // of the workgroups that share a row
// Where a fwd_bwd kernel has a row from.
template <typename T, int NT, int NV, bool REST> struct Held {
    static constexpr int kThreads = NT, kVectors = NV;
    static constexpr bool kRest = REST;
    typedef HeldRow<T, NT, NV, REST> Row;
};
template <typename T> struct Split {
    static constexpr int kThreads = kPartThreads;
    typedef SplitRow<T, kPartThreads> Row;
};
// fn(element type, source): the parts of split rows, the smallest held shape of
// at least `least` threads for a row, or the largest with the rest of the row read
// twice. Policy loss, us, by threads x vectors, bf16:
//   4 KB rows, 400     64x4 11.3, 256x2 8.7        4 KB, 16384   64x4 39.8, 128x4 50.3, 256x2 80.3
//   8 KB rows, 1000    64x8 14.1, 128x8 13.4, 256x4 11.8
//   6 KB rows, 16384   64x8 44.9, 64x16 49.3, 128x8 55.0
//   16 KB rows, 1000   64x16 19.6, 128x8 18.1, 256x4 15.4, 512x2 17.2
//   16 KB rows, 4096   64x16 33.8, 128x8 34.4, 256x4 36.6, 512x2 44.8
//   24 KB rows, 4096   128x16 44.8, 256x8 43.0, 512x4 53.7
//   32 KB rows, 1000   128x16 25.0, 256x8 21.1, 512x4 22.3
//   64 KB rows, 1000   512x8 31.1, 512x13 32.5, 1024x4 41.0
// f32: 98 KB rows, 4096 512x13 155, 1024x8 172. Not the fastest: 64 KB rows, 4000,
// which take 512x8 at 113, 512x13 104.
// The kernel alone, bf16: 201 KB rows, 2036 1024x13 139, 1024x16 140, 1024x19 142.
// Without the last shape, by a forward and a backward: 600 rows of 256000 bf16
// 161 / 169, 300 of 256000 f32 156 / 190.
constexpr int64_t kManyRows = 1536;  // past it a CU's rows fill it whatever their threads
template <typename F>
void by_row_source(int64_t rows, int least, int parts, int64_t vocab, int dtype, F&& fn) {
    if (rows < kManyRows && least < 256) least = 256;
    auto go = [&](auto elem) {
        typedef decltype(elem) T;
        if (parts > 1) return fn(elem, Split<T>{});
        const int64_t vectors = vocab / Vec16<T>::N;
        auto shape = [&](auto s) {
            typedef decltype(s) S;
            if (S::kThreads < least || (!S::kRest && vectors > S::kThreads * S::kVectors)) return false;
            fn(elem, s);
            return true;
        };
        // a rest's vectors need registers of their own, unpacked
        constexpr int kWithRest = Vec16<T>::N == 4 ? 16 : 8;
        shape(Held<T, 64, 4, false>{}) || shape(Held<T, 64, 8, false>{}) || shape(Held<T, 128, 8, false>{}) ||
            shape(Held<T, 256, 4, false>{}) || shape(Held<T, 256, 8, false>{}) || shape(Held<T, 512, 8, false>{}) ||
            shape(Held<T, 512, 13, false>{}) || shape(Held<T, 512, 19, false>{}) || shape(Held<T, 1024, 13, false>{}) ||
            shape(Held<T, 1024, 16, false>{}) || shape(Held<T, 1024, 19, false>{}) ||
            shape(Held<T, 1024, kWithRest, true>{});
    };
    if (dtype == MC_F32) go(float{});
    else go(uint16_t{});
}

Store store_of(const void* logits, const void* dlogits, int64_t rows, int64_t vocab, int dtype) {
    if ((reinterpret_cast<uintptr_t>(logits) ^ reinterpret_cast<uintptr_t>(dlogits)) & 15) return Store::kAny;
    return xent_stream_gradients(rows, vocab, dtype == MC_F32 ? 4 : 2) ? Store::kStream : Store::kCached;
}

// Rows whose sums one workgroup forms by itself; past it up to 256 of them, and a
// launch that joins theirs. A forward over 64 logits, us, one / more and the join:
// policy 2000 rows 8.9 / 10.0, 4000 11.0 / 11.3, 8192 16.2 / 14.0, 16384 26.2 /
// 19.8; distillation 4000 10.3 / 11.5, 16000 23.5 / 21.2. The join as the work of
// whichever workgroup ends last took 35.3 at 16384: its fences cost more than a
// launch. Threads of the one workgroup, 256 / 1024: 256 rows 6.4 / 7.0, 4000 13.4
// / 11.4.
constexpr int64_t kOneGroupRows = 4096;
template <typename F> void by_group_size(int64_t rows, F&& fn) {
    if (rows <= 1024) fn(std::integral_constant<int, 256>{});
    else fn(std::integral_constant<int, 1024>{});
}
template <typename F> void by_sum_kernel(int64_t rows, F&& fn) {
    if (rows <= kOneGroupRows) {
        by_group_size(rows, [&](auto threads) { fn(threads, 1, rows); });
    } else {
        const int64_t even = (rows + kSumGroups - 1) / kSumGroups, chunk = even < 1024 ? 1024 : even;
        fn(std::integral_constant<int, 256>{}, (int)((rows + chunk - 1) / chunk), chunk);
    }
}

size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

}  // namespace

// ------------------------------------------------------------- launchers
size_t loss_parts_ws(int64_t rows, int64_t vocab, int dtype, bool both) {
    const int64_t parts = loss_row_parts(rows, vocab, dtype == MC_F32 ? 4 : 2, both);
    return parts > 1 ? align256((size_t)(rows * parts) * sizeof(Stat<double>)) : 0;
}

namespace {
// The statistics of a row's parts into ws (loss_parts_ws bytes) and their number,
// or 1: not split.
int launch_parts(bool both, int64_t rows, int64_t vocab, int dtype, const void* logits, const uint32_t* targets,
                 int64_t ignore_index, const uint8_t* mask, LpScale k, void* ws, hipStream_t stream) {
    const int parts = loss_row_parts(rows, vocab, dtype == MC_F32 ? 4 : 2, both);
    if (parts == 1) return 1;
    by_threads(kPartThreads, dtype, [&](auto elem, auto threads) {
        typedef decltype(elem) T;
        constexpr int NT = decltype(threads)::value;
        if constexpr (NT == kPartThreads)
            parts_k<T, NT><<<dim3((unsigned)rows, (unsigned)parts), NT, 0, stream>>>(
                (int)vocab, static_cast<const T*>(logits), targets, ignore_index, mask, k,
                static_cast<Stat<double>*>(ws));
    });
    return parts;
}

template <typename L>
hipError_t launch_lp_rows(const mc_logprob_desc& d, const void* logits, const uint32_t* targets, L* logp,
                          float* logp32, float* stats, void* parts_ws, hipStream_t stream) {
    const LpScale k = row_scale(d.temperature);
    const int parts =
        launch_parts(false, d.rows, d.vocab, d.dtype, logits, targets, d.ignore_index, nullptr, k, parts_ws, stream);
    const int threads = parts > 1 ? 64 : loss_row_threads(d.rows, row_bytes(d.vocab, d.dtype));
    by_threads(threads, d.dtype, [&](auto elem, auto threads) {
        typedef decltype(elem) T;
        constexpr int NT = decltype(threads)::value;
        auto go = [&](auto split) {
            constexpr bool SPLIT = decltype(split)::value;
            lp_rows_k<T, NT, L, SPLIT><<<dim3((unsigned)d.rows), NT, 0, stream>>>(
                (int)d.vocab, static_cast<const T*>(logits), targets, d.ignore_index, k,
                static_cast<const Stat<double>*>(parts_ws), parts, logp, logp32,
                reinterpret_cast<RowStat*>(stats));
        };
        if constexpr (NT == 64) {
            if (parts > 1) return go(std::true_type{});
        }
        go(std::false_type{});
    });
    return hipGetLastError();
}
}  // namespace

hipError_t launch_token_logprobs_fwd(const mc_logprob_desc& d, const void* logits, const uint32_t* targets, float* logp,
                                     float* stats, void* ws, hipStream_t stream) {
    return launch_lp_rows(d, logits, targets, logp, nullptr, stats, ws, stream);
}

hipError_t launch_token_logprobs_bwd(const mc_logprob_desc& d, const void* logits, const uint32_t* targets,
                                     const float* stats, const float* dl, int64_t seq, const float* scale,
                                     const float* dloss, void* dlogits, hipStream_t stream) {
    const LpScale k = row_scale(d.temperature);
    const LossGrid grid = loss_grad_grid(d.rows, row_bytes(d.vocab, d.dtype));
    by_threads(grid.threads, d.dtype, [&](auto elem, auto threads) {
        typedef decltype(elem) T;
        constexpr int NT = decltype(threads)::value;
        if constexpr (NT != 128)  // loss_grad_grid has no such rows
            lp_bwd_k<T, NT><<<dim3((unsigned)d.rows, grid.parts), NT, 0, stream>>>(
                d.rows, (int)d.vocab, store_of(logits, dlogits, d.rows, d.vocab, d.dtype),
                static_cast<const T*>(logits), targets, d.ignore_index, k,
                reinterpret_cast<const RowStat*>(stats), dl, (uint32_t)seq, scale, dloss, static_cast<T*>(dlogits));
    });
    return hipGetLastError();
}

PreferenceWs preference_ws(const mc_preference_desc& d) {
    PreferenceWs w;
    size_t at = 0;
    w.logp = at;
    at += align256((size_t)(2 * d.pairs * d.seq) * sizeof(double));
    w.score = at;
    at += align256((size_t)(2 * d.pairs) * sizeof(double));
    w.inv_n = at;
    at += align256((size_t)(2 * d.pairs) * sizeof(float));
    w.parts = at;
    w.total = at + loss_parts_ws(2 * d.pairs * d.seq, d.vocab, d.dtype, false);
    return w;
}

hipError_t launch_preference_fwd(const mc_preference_desc& d, const void* logits, const uint32_t* targets,
                                 const float* ref, float* loss, float* rewards, float* stats, char* ws,
                                 hipStream_t stream) {
    const PreferenceWs w = preference_ws(d);
    const int64_t rows = 2 * d.pairs * d.seq;
    double* logp = reinterpret_cast<double*>(ws + w.logp);
    double* score = reinterpret_cast<double*>(ws + w.score);
    float* inv_n = reinterpret_cast<float*>(ws + w.inv_n);
    float* dseq = stats ? stats + 2 * rows : nullptr;
    const mc_logprob_desc lp{rows, d.vocab, d.ignore_index, 1.0f, d.dtype};
    hipError_t e = launch_lp_rows(lp, logits, targets, logp, nullptr, stats, ws + w.parts, stream);
    if (e != hipSuccess) return e;
    if (rows <= kOneGroupRows && 2 * d.pairs <= kOneGroupSeqs) {
        by_group_size(rows, [&](auto threads) {
            constexpr int NT = decltype(threads)::value;
            preference_one_k<NT><<<dim3(1), NT, 0, stream>>>(d, targets, logp, ref, loss, rewards, dseq);
        });
        return hipGetLastError();
    }
    preference_scores_k<<<dim3((unsigned)(2 * d.pairs)), 256, 0, stream>>>(d, targets, logp, ref, score, inv_n,
                                                                          rewards);
    by_group_size(d.pairs, [&](auto threads) {
        constexpr int NT = decltype(threads)::value;
        preference_pairs_k<NT><<<dim3(1), NT, 0, stream>>>(d, score, inv_n, loss, dseq);
    });
    return hipGetLastError();
}

PolicyWs policy_ws(const mc_policy_desc& d) {
    PolicyWs w;
    size_t at = 0;
    w.part = at;
    at += kSumGroups * 4 * sizeof(double);
    w.logp = at;
    at += align256((size_t)(d.batch * d.seq) * sizeof(double));
    w.counts = at;
    if (d.reduction == MC_MEAN_SEQUENCES) at += align256((size_t)d.batch * sizeof(uint32_t));
    w.parts = at;
    w.total = at + loss_parts_ws(d.batch * d.seq, d.vocab, d.dtype, false);
    return w;
}

namespace {
const uint32_t* policy_counts(const mc_policy_desc& d, const uint32_t* targets, char* ws, hipStream_t stream,
                              hipError_t& e) {
    e = hipSuccess;
    if (d.reduction != MC_MEAN_SEQUENCES) return nullptr;
    uint32_t* n = reinterpret_cast<uint32_t*>(ws + policy_ws(d).counts);
    // us of a forward over 64 logits, a wave per sequence / a workgroup: 20000 of one
    // token 27.1 / 56.6, 8 of 1024 16.7 / 17.1, 2 of 8192 25.4 / 22.3, 1 of 200000 260 / 148
    if (d.seq <= 1024)
        seq_counts_k<64><<<dim3((unsigned)((d.batch + 3) / 4)), 256, 0, stream>>>(d.batch, d.seq, targets,
                                                                                  d.ignore_index, n);
    else
        seq_counts_k<1024><<<dim3((unsigned)d.batch), 1024, 0, stream>>>(d.batch, d.seq, targets, d.ignore_index, n);
    e = hipGetLastError();
    return n;
}

hipError_t launch_policy_sums(const mc_policy_desc& d, const uint32_t* targets, const float* adv, const float* old,
                              const float* ref, const uint32_t* n, char* ws, float* loss, float* metrics, float* dlp,
                              hipStream_t stream) {
    auto* part = reinterpret_cast<double(*)[4]>(ws + policy_ws(d).part);
    const double* logp = reinterpret_cast<const double*>(ws + policy_ws(d).logp);
    by_sum_kernel(d.batch * d.seq, [&](auto threads, int groups, int64_t chunk) {
        constexpr int NT = decltype(threads)::value;
        policy_k<NT><<<dim3((unsigned)groups), NT, 0, stream>>>(d, chunk, targets, logp, adv, old, ref, n, part, loss,
                                                                metrics, dlp);
        if (groups > 1)
            policy_join_k<<<dim3(1), kSumGroups, 0, stream>>>(d, n != nullptr, groups, part, loss, metrics, dlp);
    });
    return hipGetLastError();
}
}  // namespace

hipError_t launch_policy_fwd(const mc_policy_desc& d, const void* logits, const uint32_t* targets, const float* adv,
                             const float* old, const float* ref, float* loss, float* logp, float* metrics,
                             float* stats, char* ws, hipStream_t stream) {
    const int64_t rows = d.batch * d.seq;
    const mc_logprob_desc lp{rows, d.vocab, d.ignore_index, d.temperature, d.dtype};
    hipError_t e;
    const uint32_t* n = policy_counts(d, targets, ws, stream, e);
    if (e != hipSuccess) return e;
    const PolicyWs w = policy_ws(d);
    e = launch_lp_rows(lp, logits, targets, reinterpret_cast<double*>(ws + w.logp), logp, stats, ws + w.parts, stream);
    if (e != hipSuccess) return e;
    return launch_policy_sums(d, targets, adv, old, ref, n, ws, loss, metrics, stats ? stats + 2 * rows : nullptr, stream);
}

DistillWs distill_ws(const mc_distill_desc& d) {
    DistillWs w;
    size_t at = 0;
    w.part = at;
    at += kSumGroups * 2 * sizeof(double);
    w.kl = at;
    at += align256((size_t)d.rows * sizeof(double));
    w.split = at;
    w.total = at + loss_parts_ws(d.rows, d.vocab, d.dtype, false);
    return w;
}

namespace {
hipError_t launch_distill_sums(const mc_distill_desc& d, const uint8_t* mask, const double* kl, char* ws, float* loss,
                               float* scale, hipStream_t stream) {
    auto* part = reinterpret_cast<double(*)[2]>(ws + distill_ws(d).part);
    by_sum_kernel(d.rows, [&](auto threads, int groups, int64_t chunk) {
        constexpr int NT = decltype(threads)::value;
        distill_final_k<NT><<<dim3((unsigned)groups), NT, 0, stream>>>(d.rows, chunk, d.temperature, mask, kl, part,
                                                                       loss, scale);
        if (groups > 1)
            distill_join_k<<<dim3(1), kSumGroups, 0, stream>>>(d.temperature, groups, part, loss, scale);
    });
    return hipGetLastError();
}
}  // namespace

hipError_t launch_distill_fwd(const mc_distill_desc& d, const void* logits, const int32_t* ids, const float* tl,
                              const float* tlse, const uint8_t* mask, float* loss, float* stats, char* ws,
                              hipStream_t stream) {
    const DistillWs w = distill_ws(d);
    const LpScale k = row_scale(d.temperature);
    double* kl = reinterpret_cast<double*>(ws + w.kl);
    const int parts =
        launch_parts(false, d.rows, d.vocab, d.dtype, logits, nullptr, -1, mask, k, ws + w.split, stream);
    int threads = parts > 1 ? kDistillMaxTop : loss_row_threads(d.rows, row_bytes(d.vocab, d.dtype));
    while (threads < d.top) threads *= 2;  // a thread per entry
    by_threads(threads, d.dtype, [&](auto elem, auto threads) {
        typedef decltype(elem) T;
        constexpr int NT = decltype(threads)::value;
        auto go = [&](auto split) {
            constexpr bool SPLIT = decltype(split)::value;
            distill_rows_k<T, NT, SPLIT><<<dim3((unsigned)d.rows), NT, 0, stream>>>(
                d, static_cast<const T*>(logits), ids, tl, tlse, mask, k,
                reinterpret_cast<const Stat<double>*>(ws + w.split), parts, kl, reinterpret_cast<RowStat*>(stats));
        };
        if constexpr (NT == kDistillMaxTop) {
            if (parts > 1) return go(std::true_type{});
        }
        go(std::false_type{});
    });
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    return launch_distill_sums(d, mask, kl, ws, loss, stats ? stats + 2 * d.rows : nullptr, stream);
}

hipError_t launch_distill_bwd(const mc_distill_desc& d, const void* logits, const int32_t* ids, const float* tl,
                              const float* tlse, const uint8_t* mask, const float* stats, const float* dloss,
                              void* dlogits, hipStream_t stream) {
    const LpScale k = row_scale(d.temperature);
    const LossGrid grid = loss_grad_grid(d.rows, row_bytes(d.vocab, d.dtype));
    by_threads(grid.threads < kDistillMaxTop ? kDistillMaxTop : grid.threads, d.dtype, [&](auto elem, auto threads) {
        typedef decltype(elem) T;
        constexpr int NT = decltype(threads)::value;
        if constexpr (NT >= kDistillMaxTop)
            distill_bwd_k<T, NT><<<dim3((unsigned)d.rows, grid.parts), NT, 0, stream>>>(
                d, store_of(logits, dlogits, d.rows, d.vocab, d.dtype), static_cast<const T*>(logits), ids, tl,
                tlse, mask, k, reinterpret_cast<const RowStat*>(stats), stats + 2 * d.rows, dloss,
                static_cast<T*>(dlogits));
    });
    return hipGetLastError();
}

// counts_k over rows into ws; the number of its blocks
namespace {
int launch_counts(int64_t rows, const uint32_t* targets, const uint8_t* mask, int64_t ignore_index, uint32_t* part,
                  hipStream_t stream) {
    int64_t chunk = (rows + kCountBlocks - 1) / kCountBlocks;
    if (chunk < 256) chunk = 256;
    const int blocks = (int)((rows + chunk - 1) / chunk);
    counts_k<<<dim3((unsigned)blocks), 256, 0, stream>>>(rows, chunk, targets, mask, ignore_index, part);
    return blocks;
}
}  // namespace

// The forward's buffers, then 64 counts or, where the two run one after the
// other, the forward's stats; then the parts of shared rows.
namespace {
size_t loss_stats_ws(int64_t n) { return align256((size_t)(n + kCountBlocks) * sizeof(float)); }
}  // namespace
size_t policy_fwd_bwd_ws(const mc_policy_desc& d) {
    const int64_t rows = d.batch * d.seq;
    return policy_ws(d).total + loss_stats_ws(3 * rows) + loss_parts_ws(rows, d.vocab, d.dtype, true);
}

hipError_t launch_policy_fwd_bwd(const mc_policy_desc& d, const void* logits, const uint32_t* targets,
                                 const float* adv, const float* old, const float* ref, const float* dloss, float* loss,
                                 float* logp, float* metrics, void* dlogits, char* ws, hipStream_t stream) {
    const PolicyWs w = policy_ws(d);
    float* stats = reinterpret_cast<float*>(ws + w.total);
    const int64_t rows = d.batch * d.seq;
    const LpScale k = row_scale(d.temperature);
    const Store how = store_of(logits, dlogits, rows, d.vocab, d.dtype);
    hipError_t e;
    if (how != Store::kAny && loss_threads_fit(rows, 1024)) {
        uint32_t* part = reinterpret_cast<uint32_t*>(stats);
        const bool by_seq = d.reduction == MC_MEAN_SEQUENCES;
        uint32_t* n = by_seq ? reinterpret_cast<uint32_t*>(ws + w.counts) : nullptr;
        void* parts_ws = ws + w.total + loss_stats_ws(3 * rows);
        const int parts =
            launch_parts(true, rows, d.vocab, d.dtype, logits, targets, d.ignore_index, nullptr, k, parts_ws, stream);
        e = hipSuccess;
        by_row_source(rows, 1, parts, d.vocab, d.dtype, [&](auto elem, auto source) {
            typedef decltype(elem) T;
            typedef decltype(source) S;
            constexpr int NT = S::kThreads;
            const int64_t span = by_seq ? d.seq : rows;
            const bool here = span <= RowCount<NT>::kPer * NT;
            int n_given = here ? 0 : 1;
            if (!here && by_seq) policy_counts(d, targets, ws, stream, e);
            else if (!here) n_given = launch_counts(rows, targets, nullptr, d.ignore_index, part, stream);
            policy_both_k<T, NT, typename S::Row><<<dim3((unsigned)rows, (unsigned)parts), NT, 0, stream>>>(
                d, how, static_cast<const T*>(logits), targets, adv, old,
                ref, static_cast<const Stat<double>*>(parts_ws), here ? nullptr : by_seq ? n : part, n_given,
                here ? (int)span : 0, by_seq, here ? n : nullptr, k, dloss,
                reinterpret_cast<double*>(ws + w.logp), logp, static_cast<T*>(dlogits));
        });
        if (e != hipSuccess) return e;
        if ((e = hipGetLastError()) != hipSuccess) return e;
        return launch_policy_sums(d, targets, adv, old, ref, n, ws, loss, metrics, nullptr, stream);
    }
    e = launch_policy_fwd(d, logits, targets, adv, old, ref, loss, logp, metrics, stats, ws, stream);
    if (e != hipSuccess) return e;
    const mc_logprob_desc lp{rows, d.vocab, d.ignore_index, d.temperature, d.dtype};
    return launch_token_logprobs_bwd(lp, logits, targets, stats, stats + 2 * rows, 0, stats + 3 * rows, dloss, dlogits,
                                     stream);
}

size_t distill_fwd_bwd_ws(const mc_distill_desc& d) {
    return distill_ws(d).total + loss_stats_ws(2 * d.rows) + loss_parts_ws(d.rows, d.vocab, d.dtype, true);
}

hipError_t launch_distill_fwd_bwd(const mc_distill_desc& d, const void* logits, const int32_t* ids, const float* tl,
                                  const float* tlse, const uint8_t* mask, const float* dloss, float* loss,
                                  void* dlogits, char* ws, hipStream_t stream) {
    const DistillWs w = distill_ws(d);
    float* stats = reinterpret_cast<float*>(ws + w.total);
    const LpScale k = row_scale(d.temperature);
    const Store how = store_of(logits, dlogits, d.rows, d.vocab, d.dtype);
    hipError_t e;
    if (how != Store::kAny && loss_threads_fit(d.rows, 1024)) {
        double* kl = reinterpret_cast<double*>(ws + w.kl);
        uint32_t* part = reinterpret_cast<uint32_t*>(stats);
        void* parts_ws = ws + w.total + loss_stats_ws(2 * d.rows);
        const int parts =
            launch_parts(true, d.rows, d.vocab, d.dtype, logits, nullptr, -1, mask, k, parts_ws, stream);
        by_row_source(d.rows, d.top, parts, d.vocab, d.dtype, [&](auto elem, auto source) {
            typedef decltype(elem) T;
            typedef decltype(source) S;
            constexpr int NT = S::kThreads;
            const bool here = !mask || d.rows <= RowCount<NT>::kPer * NT;
            const int n_given = here ? 0 : launch_counts(d.rows, nullptr, mask, -1, part, stream);
            distill_both_k<T, NT, typename S::Row><<<dim3((unsigned)d.rows, (unsigned)parts), NT, 0, stream>>>(
                d, how, static_cast<const T*>(logits), ids, tl, tlse,
                mask, static_cast<const Stat<double>*>(parts_ws), here ? nullptr : part, n_given,
                mask && here ? (int)d.rows : 0, k, dloss, kl, static_cast<T*>(dlogits));
        });
        if ((e = hipGetLastError()) != hipSuccess) return e;
        return launch_distill_sums(d, mask, kl, ws, loss, nullptr, stream);
    }
    e = launch_distill_fwd(d, logits, ids, tl, tlse, mask, loss, stats, ws, stream);
    if (e != hipSuccess) return e;
    return launch_distill_bwd(d, logits, ids, tl, tlse, mask, stats, dloss, dlogits, stream);
}

}  // namespace mc
