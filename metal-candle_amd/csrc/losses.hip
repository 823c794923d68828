// Losses over a vocabulary's logits for what comes after supervised
// fine-tuning, gfx950: log-probabilities of given tokens, the preference loss
// over pairs of sequences, the clipped policy loss with its KL term, and
// distillation from a teacher's top logits. They start from the same logits
// [rows, vocab] as the cross entropy (rowops.hip).
//
// Per row, with q = softmax(x / T) and lse = log sum exp(x / T):
//   l = x_t / T - lse, the token's log-probability; dl/dx_j = ([j = t] - q_j) / T.
// Every loss but distillation is a function of the l alone, so one kernel forms
// l and the row's maximum and sum from one read of the logits (lp_rows_k), small kernels form the
// loss and dloss/dl, and one kernel turns dloss/dl into the gradient of the
// logits (lp_bwd_k). Distillation is sum_k p_k (log p_k - log q_{id k}) over a
// teacher's K best, whose gradient is (P q_j - sum_{id k = j} p_k) / T with
// P = sum p: the same dense part with K entries taken out of it instead of one.
// A row that is not counted is never read and its gradient is zero.
//
// Bound by HBM throughout: 2 or 4 bytes per logit and pass against about ten
// operations.
#include <type_traits>

#include "common.hpp"
#include "kernels.hpp"
#include "rules.hpp"
#include "vocab_rows.hpp"

namespace mc {
namespace {

constexpr float kNegInf = -__builtin_inff();

// ------------------------------------------------------------ row statistics
// m = max x and s = sum 2^((x - m) c), c = log2(e) / T as c_hi + c_lo
// (row_scale): with one float for c every exponent is off by up to 6e-8 of
// itself to the same side, and so is every l of a sequence, which the sums over
// an answer add up instead of averaging out. x - m comes first: x c alone
// overflows where logits hold the type's lowest value. An all -inf row has
// m = -inf and s = 0, a NaN in the row makes s NaN: l and the gradient are NaN in
// both. The backward takes m and s as they are: lse as one float would cost each
// q 2^-24 |lse| of itself.
__device__ __forceinline__ RowStat stat_join(RowStat a, RowStat b, float c) {
    const float m = fmaxf(a.m, b.m);
    // equal maxima, -inf among them, need no factor
    const float sa = a.m == m ? a.s : a.s * exp2_hw((a.m - m) * c);
    const float sb = b.m == m ? b.s : b.s * exp2_hw((b.m - m) * c);
    return RowStat{m, sa + sb};
}

// Over the workgroup's NT threads in a fixed order: a butterfly over each wave,
// then the waves in order. red: one slot per wave.
template <int NT>
__device__ __forceinline__ RowStat wg_stat(RowStat v, float c, RowStat* red) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1)
        v = stat_join(v, RowStat{__shfl_xor(v.m, o, kWave), __shfl_xor(v.s, o, kWave)}, c);
    if (lane_id() == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int k = 1; k < NT / 64; ++k) v = stat_join(v, red[k], c);
    return v;
}

// What a share's terms are relative to: where all of it is -inf, anything finite.
__device__ __forceinline__ float base_of(float m) { return m == kNegInf ? 0.f : m; }
__device__ __forceinline__ float term_of(float x, float base, LpScale k) {
    const float d = x - base;
    return exp2_hw(fmaf(d, k.c_lo, d * k.c_hi));
}

// One thread's share of a row: four vectors requested and reduced at a time,
// one rescale to their maximum, then one exp2 per element.
template <typename T, int NT>
__device__ __forceinline__ RowStat row_stat(const T* __restrict__ xr, int vocab, LpScale k) {
    constexpr int N = Vec16<T>::N, U = 4;
    float m = kNegInf, s = 0.f;
    const RowSpan<T> span(xr, vocab);
    const T* xv = xr + span.head;
    const int nvec = (int)span.nvec;
    auto group = [&](int c, auto count) {
        constexpr int K = decltype(count)::value;
        float v[K][N];
#pragma unroll
        for (int u = 0; u < K; ++u) Vec16<T>::load(xv + (int64_t)(c + u * NT) * N, v[u]);
        float vm = v[0][0];
#pragma unroll
        for (int u = 0; u < K; ++u)
#pragma unroll
            for (int e = 0; e < N; ++e) vm = fmaxf(vm, v[u][e]);
        if (vm > m) {
            s *= exp2_hw((m - vm) * k.c_hi);  // 0 for the first
            m = vm;
        }
        const float base = base_of(m);
        float ps[K];
#pragma unroll
        for (int u = 0; u < K; ++u) {
            ps[u] = 0.f;
#pragma unroll
            for (int e = 0; e < N; ++e) ps[u] += term_of(v[u][e], base, k);
        }
        if constexpr (K == 4) s += (ps[0] + ps[1]) + (ps[2] + ps[3]);
        else s += ps[0];
    };
    int c = threadIdx.x;
    for (; c < nvec - (U - 1) * NT; c += U * NT) group(c, std::integral_constant<int, U>{});
    for (; c < nvec; c += NT) group(c, std::integral_constant<int, 1>{});
    const int64_t j = span.edge((int)threadIdx.x, vocab);
    if (j >= 0) {
        const float v = Elem<T>::load(xr, j);
        return stat_join(RowStat{m, s}, RowStat{v, term_of(v, base_of(v), k)}, k.c_hi);
    }
    return RowStat{m, s};
}

// -------------------------------------------------- sums over many workgroups
// Each workgroup leaves its partial sums in memory; the last one to arrive adds
// them in workgroup order. The kernel before on the stream clears the counter.
template <int C>
__device__ __forceinline__ void wg_sum_f64(double (&v)[C], double (*red)[C]) {
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) v[c] += __shfl_xor(v[c], o, kWave);
    __syncthreads();
    if (lane_id() == 0)
#pragma unroll
        for (int c = 0; c < C; ++c) red[threadIdx.x >> 6][c] = v[c];
    __syncthreads();
    const int nw = (int)(blockDim.x >> 6);
#pragma unroll
    for (int c = 0; c < C; ++c) {
        v[c] = red[0][c];
        for (int w = 1; w < nw; ++w) v[c] += red[w][c];
    }
}

// True in every thread of the workgroup that arrives last; what the others wrote
// before is visible to it.
__device__ __forceinline__ bool last_to_arrive(uint32_t* counter, uint32_t* slot) {
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) *slot = atomicAdd(counter, 1u);
    __syncthreads();
    const bool last = *slot == gridDim.x - 1;
    if (last) __threadfence();
    return last;
}

// ------------------------------------------------------------- row kernels
__device__ __forceinline__ bool counted(uint32_t t, int64_t ignore_index) {
    return !(ignore_index >= 0 && (int64_t)t == ignore_index);
}

// l (0 where the row is not counted) and the row's statistics; a counted target
// past the vocabulary makes its l NaN. counter: cleared for the kernel that
// follows.
template <typename T, int NT>
__global__ __launch_bounds__(NT) void lp_rows_k(int vocab, const T* __restrict__ logits,
                                                const uint32_t* __restrict__ targets, int64_t ignore_index, LpScale k,
                                                float* __restrict__ logp, RowStat* __restrict__ stats,
                                                uint32_t* __restrict__ counter) {
    __shared__ RowStat red[NT / 64];
    const int64_t row = blockIdx.x;
    if (counter && row == 0 && threadIdx.x == 0) *counter = 0;
    const uint32_t t = targets[row];
    if (!counted(t, ignore_index)) {
        if (threadIdx.x == 0) {
            logp[row] = 0.f;
            if (stats) stats[row] = RowStat{0.f, 1.f};
        }
        return;
    }
    const T* xr = logits + row * vocab;
    const RowStat v = wg_stat<NT>(row_stat<T, NT>(xr, vocab, k), k.c_hi, red);
    if (threadIdx.x == 0) {
        logp[row] = t < (uint32_t)vocab ? (Elem<T>::load(xr, t) - v.m) * k.inv_t - logf(v.s) : __builtin_nanf("");
        if (stats) stats[row] = v;
    }
}

// ------------------------------------------------------------- preference
// A workgroup per sequence; the last one turns the pairs' scores into the loss
// and each sequence's dloss/dl. Scores in 64 bits: they are differences of sums
// over whole answers.
__global__ __launch_bounds__(256) void preference_k(mc_preference_desc d, const uint32_t* __restrict__ targets,
                                                    const float* __restrict__ logp, const float* __restrict__ ref,
                                                    double* __restrict__ score, float* __restrict__ inv_n,
                                                    uint32_t* __restrict__ counter, float* __restrict__ loss,
                                                    float* __restrict__ rewards, float* __restrict__ dseq) {
    __shared__ double red[4][2];
    __shared__ uint32_t slot;
    const int64_t q = blockIdx.x;
    double v[2] = {0.0, 0.0};
    for (int64_t i = threadIdx.x; i < d.seq; i += 256) {
        const int64_t row = q * d.seq + i;
        if (!counted(targets[row], d.ignore_index)) continue;
        v[0] += (double)logp[row] - (ref ? (double)ref[row] : 0.0);
        v[1] += 1.0;
    }
    wg_sum_f64<2>(v, red);
    if (threadIdx.x == 0) {
        const double inv = d.average && v[1] > 0.0 ? 1.0 / v[1] : 1.0;
        score[q] = v[0] * inv;
        inv_n[q] = (float)inv;
        if (rewards) rewards[q] = (float)(d.beta * score[q]);
    }
    if (!last_to_arrive(counter, &slot)) return;
    double sum[2] = {0.0, 0.0};
    const double beta = d.beta, eps = d.label_smoothing, pairs = (double)d.pairs;
    for (int64_t i = threadIdx.x; i < d.pairs; i += 256) {
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
    wg_sum_f64<2>(sum, red);
    if (threadIdx.x == 0) loss[0] = (float)(sum[0] / pairs);
}

// ------------------------------------------------------------------ policy
// Counted tokens of each sequence, a wave for each.
__global__ __launch_bounds__(256) void seq_counts_k(int64_t batch, int64_t seq, const uint32_t* __restrict__ targets,
                                                    int64_t ignore_index, uint32_t* __restrict__ n) {
    const int64_t q = (int64_t)blockIdx.x * 4 + wave_id();
    if (q >= batch) return;
    uint32_t c = 0;
    for (int64_t i = lane_id(); i < seq; i += kWave) c += counted(targets[q * seq + i], ignore_index) ? 1u : 0u;
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) c += (uint32_t)__shfl_xor((int)c, o, kWave);
    if (lane_id() == 0) n[q] = c;
}

// A token's terms: -min(r A, clip(r) A) + kl_coef kl, dl, kl and whether the
// clipped side holds (then the surrogate has no gradient).
struct PolicyTerm {
    float term, dl, kl, clipped;
};
__device__ __forceinline__ PolicyTerm policy_term(const mc_policy_desc& d, float l, float A, const float* old,
                                                  const float* ref, int64_t row) {
    PolicyTerm p;
    const float r = old ? expf(l - old[row]) : (l == l ? 1.f : l);
    const float held = fminf(fmaxf(r, 1.f - d.clip_low), 1.f + d.clip_high);
    const bool clipped = held * A < r * A;
    p.clipped = clipped ? 1.f : 0.f;
    p.term = -(clipped ? held * A : r * A);
    p.dl = clipped ? 0.f : -r * A;
    p.kl = 0.f;
    if (ref) {
        const float u = ref[row] - l, g = expm1f(u);
        p.kl = g - u;
        if (d.kl_coef != 0.f) {
            p.term = fmaf(d.kl_coef, p.kl, p.term);
            p.dl = fmaf(-d.kl_coef, g, p.dl);
        }
    }
    return p;
}

// Workgroup b: rows b * chunk ..; sums of the terms, the KL, the clipped tokens
// and the counted ones. n: counted tokens of each sequence where the mean runs
// over sequences. dlp: dloss/dl but for the factor at dlp[rows], which is known
// only at the end.
__global__ __launch_bounds__(256) void policy_k(mc_policy_desc d, int64_t chunk, const uint32_t* __restrict__ targets,
                                                const float* __restrict__ logp, const float* __restrict__ adv,
                                                const float* __restrict__ old, const float* __restrict__ ref,
                                                const uint32_t* __restrict__ n, double (*part)[4],
                                                uint32_t* __restrict__ counter, float* __restrict__ loss,
                                                float* __restrict__ metrics, float* __restrict__ dlp) {
    __shared__ double red[4][4];
    __shared__ uint32_t slot;
    const int64_t rows = d.batch * d.seq, r0 = (int64_t)blockIdx.x * chunk;
    const int64_t r1 = r0 + chunk < rows ? r0 + chunk : rows;
    double v[4] = {0.0, 0.0, 0.0, 0.0};
    for (int64_t row = r0 + threadIdx.x; row < r1; row += 256) {
        float dl = 0.f;
        if (counted(targets[row], d.ignore_index)) {
            const uint32_t q = (uint32_t)row / (uint32_t)d.seq;
            const PolicyTerm p = policy_term(d, logp[row], adv[d.per_token_advantages ? row : q], old, ref, row);
            const double w = n ? 1.0 / (double)n[q] : 1.0;
            v[0] += w * (double)p.term;
            v[1] += w * (double)p.kl;
            v[2] += w * (double)p.clipped;
            v[3] += 1.0;
            dl = (float)(w * (double)p.dl);
        }
        if (dlp) dlp[row] = dl;
    }
    wg_sum_f64<4>(v, red);
    if (threadIdx.x == 0)
#pragma unroll
        for (int c = 0; c < 4; ++c) part[blockIdx.x][c] = v[c];
    if (!last_to_arrive(counter, &slot)) return;
#pragma unroll
    for (int c = 0; c < 4; ++c) v[c] = threadIdx.x < gridDim.x ? part[threadIdx.x][c] : 0.0;
    wg_sum_f64<4>(v, red);
    if (threadIdx.x == 0) {
        const double N = n ? (double)d.batch : v[3];  // no token at all: 0 / 0, a NaN loss
        loss[0] = (float)(v[0] / N);
        if (metrics) {
            metrics[0] = (float)(v[1] / N);
            metrics[1] = (float)(v[2] / N);
        }
        if (dlp) dlp[rows] = (float)(1.0 / N);
    }
}

// ------------------------------------------------------------ distillation
// The teacher's entries of one row in LDS: ids, probabilities (0 where the entry
// is left out: a logit of -inf), their sum P and sum p log p. bad: an entry
// whose id is past the vocabulary.
struct Teacher {
    int id[kDistillMaxTop];
    float p[kDistillMaxTop];
};
struct TeacherSums {
    float P, plogp;
    bool bad;
};
// All threads of the workgroup; NT >= kDistillMaxTop. red: 4 floats per wave.
template <int NT>
__device__ __forceinline__ TeacherSums load_teacher(Teacher& te, const mc_distill_desc& d, int64_t row,
                                                    const int32_t* __restrict__ ids, const float* __restrict__ tl,
                                                    const float* __restrict__ tlse, float* red) {
    static_assert(NT >= kDistillMaxTop, "an entry per thread");
    const int t = threadIdx.x;
    const bool on = t < d.top;
    const float inv_t = 1.0f / d.temperature;
    const float z = on ? tl[row * d.top + t] * inv_t : kNegInf;
    const int id = on ? ids[row * d.top + t] : 0;
    float logp;
    if (tlse) {
        logp = z - tlse[row];
    } else {
        const float zm = wg_max(z, red);
        // z != z: a NaN, which the maximum passes over, stays in the sum
        const float e = z == kNegInf ? 0.f : expf(z - zm);
        const float sum = wg_sum(e, red + NT / 64);
        logp = (z - zm) - logf(sum);
    }
    const float p = z == kNegInf ? 0.f : expf(logp);
    const float term = p == 0.f ? 0.f : p * logp;
    const bool bad = p != 0.f && (id < 0 || id >= (int)d.vocab);
    if (on) {
        te.id[t] = p != 0.f ? id : -1;
        te.p[t] = p;
    }
    TeacherSums s;
    s.P = wg_sum(p, red + 2 * (NT / 64));
    s.plogp = wg_sum(term, red + 3 * (NT / 64));
    s.bad = __syncthreads_or(bad);
    return s;
}

// sum_k p_k (log p_k - log q_k) of a row with statistics v. red: a float per wave.
template <typename T>
__device__ __forceinline__ float distill_row(const Teacher& te, TeacherSums s, int top, const T* __restrict__ xr,
                                             RowStat v, LpScale k, float* red) {
    float cross = 0.f;  // sum p log q
    const int t = threadIdx.x;
    const float ls = logf(v.s);
    if (t < top && te.p[t] != 0.f && !s.bad) cross = te.p[t] * ((Elem<T>::load(xr, te.id[t]) - v.m) * k.inv_t - ls);
    cross = wg_sum(cross, red);
    return s.bad ? __builtin_nanf("") : s.plogp - cross;
}

template <typename T, int NT>
__global__ __launch_bounds__(NT) void distill_rows_k(mc_distill_desc d, const T* __restrict__ logits,
                                                     const int32_t* __restrict__ ids, const float* __restrict__ tl,
                                                     const float* __restrict__ tlse, const uint8_t* __restrict__ mask,
                                                     LpScale k, float* __restrict__ kl, RowStat* __restrict__ stats,
                                                     uint32_t* __restrict__ counter) {
    __shared__ RowStat red[NT / 64];
    __shared__ float redf[5 * (NT / 64)];
    __shared__ Teacher te;
    const int64_t row = blockIdx.x;
    const int vocab = (int)d.vocab;
    if (row == 0 && threadIdx.x == 0) *counter = 0;
    if (mask && mask[row] == 0) {
        if (threadIdx.x == 0) {
            kl[row] = 0.f;
            if (stats) stats[row] = RowStat{0.f, 1.f};
        }
        return;
    }
    const T* xr = logits + row * vocab;
    const TeacherSums ts = load_teacher<NT>(te, d, row, ids, tl, tlse, redf);
    const RowStat v = wg_stat<NT>(row_stat<T, NT>(xr, vocab, k), k.c_hi, red);
    const float r = ts.P == 0.f ? 0.f : distill_row(te, ts, d.top, xr, v, k, redf + 4 * (NT / 64));
    if (threadIdx.x == 0) {
        kl[row] = r;
        if (stats) stats[row] = v;
    }
}

// loss = T^2 sum kl / counted rows; scale = T / counted rows.
__global__ __launch_bounds__(256) void distill_final_k(int64_t rows, int64_t chunk, float temperature,
                                                       const uint8_t* __restrict__ mask, const float* __restrict__ kl,
                                                       double (*part)[2], uint32_t* __restrict__ counter,
                                                       float* __restrict__ loss, float* __restrict__ scale) {
    __shared__ double red[4][2];
    __shared__ uint32_t slot;
    const int64_t r0 = (int64_t)blockIdx.x * chunk;
    const int64_t r1 = r0 + chunk < rows ? r0 + chunk : rows;
    double v[2] = {0.0, 0.0};
    for (int64_t row = r0 + threadIdx.x; row < r1; row += 256)
        if (!mask || mask[row] != 0) {
            v[0] += (double)kl[row];
            v[1] += 1.0;
        }
    wg_sum_f64<2>(v, red);
    if (threadIdx.x == 0) {
        part[blockIdx.x][0] = v[0];
        part[blockIdx.x][1] = v[1];
    }
    if (!last_to_arrive(counter, &slot)) return;
#pragma unroll
    for (int c = 0; c < 2; ++c) v[c] = threadIdx.x < gridDim.x ? part[threadIdx.x][c] : 0.0;
    wg_sum_f64<2>(v, red);
    if (threadIdx.x == 0) {
        const double T = temperature;
        loss[0] = (float)(T * T * v[0] / v[1]);  // no row counted: 0 / 0, a NaN loss
        if (scale) scale[0] = (float)(T / v[1]);
    }
}

// ---------------------------------------------------------------- gradients
// The row's dense part a q, q = 2^((x - m) c) / s, with `take` adding to the elements j0 ..
// j0 + N of a vector what the loss holds there. Rows run backwards, and stream
// stores past the caches, for the reasons of the cross entropy's backward.
template <typename T, int NT, typename Take>
__device__ __forceinline__ void write_row(const T* __restrict__ xr, T* __restrict__ dr, int vocab, bool vec,
                                          bool stream, float a, float c, RowStat st, const Take& take) {
    constexpr int N = Vec16<T>::N;
    const float m = st.m;
    a /= st.s;
    if (vec) {
        const RowSpan<T> span(xr, vocab);
        const int head = (int)span.head;
        for (int cc = (int)span.nvec - 1 - (int)threadIdx.x; cc >= 0; cc -= NT) {
            const int64_t j0 = head + (int64_t)cc * N;
            float v[N];
            Vec16<T>::load(xr + j0, v);
#pragma unroll
            for (int e = 0; e < N; ++e) v[e] = a * exp2_hw((v[e] - m) * c);
            take(cc, (int)j0, v);
            if (stream) store_nt16(dr + j0, v);
            else Vec16<T>::store(dr + j0, v);
        }
        const int64_t j = span.edge((int)threadIdx.x, vocab);
        if (j >= 0) Elem<T>::store(dr, j, take.at((int)j, a * exp2_hw((Elem<T>::load(xr, j) - m) * c)));
    } else {
        for (int64_t j = threadIdx.x; j < vocab; j += NT)
            Elem<T>::store(dr, j, take.at((int)j, a * exp2_hw((Elem<T>::load(xr, j) - m) * c)));
    }
}

template <typename T, int NT>
__device__ __forceinline__ void zero_row(T* __restrict__ dr, int vocab, bool stream) {
    constexpr int N = Vec16<T>::N;
    const RowSpan<T> span(dr, vocab);
    const float z[N] = {};
    for (int c = threadIdx.x; c < (int)span.nvec; c += NT) {
        T* p = dr + span.head + (int64_t)c * N;
        if (stream) store_nt16(p, z);
        else Vec16<T>::store(p, z);
    }
    const int64_t j = span.edge((int)threadIdx.x, vocab);
    if (j >= 0) Elem<T>::store(dr, j, 0.f);
}

// One target's g.
struct TakeOne {
    int t;
    float g;
    template <int N> __device__ __forceinline__ void operator()(int, int j0, float (&v)[N]) const {
        if ((unsigned)(t - j0) < (unsigned)N) {
#pragma unroll
            for (int e = 0; e < N; ++e) v[e] += j0 + e == t ? g : 0.f;
        }
    }
    __device__ __forceinline__ float at(int j, float v) const { return j == t ? v + g : v; }
};

// A teacher's entries, w p_k each, in the order of k where an id comes twice.
// A bit per vector says whether any entry lies in it (two vectors 2^16 apart
// share a bit), so only those vectors go through the list.
constexpr int kTakeBits = 1 << 16;
struct TakeTop {
    const Teacher& te;
    const uint32_t* bits;
    int top;
    float w;
    template <int N> __device__ __forceinline__ void operator()(int cc, int j0, float (&v)[N]) const {
        const unsigned b = (unsigned)cc & (kTakeBits - 1);
        if (!((bits[b >> 5] >> (b & 31)) & 1u)) return;
        for (int k = 0; k < top; ++k) {
            const int id = te.id[k];
            if ((unsigned)(id - j0) < (unsigned)N) {
#pragma unroll
                for (int e = 0; e < N; ++e) v[e] -= j0 + e == id ? w * te.p[k] : 0.f;
            }
        }
    }
    __device__ __forceinline__ float at(int j, float v) const {
        for (int k = 0; k < top; ++k)
            if (te.id[k] == j) v -= w * te.p[k];
        return v;
    }
};
// The bits of a row's entries (ids in range). All threads; head as in write_row.
template <int NT, int N>
__device__ __forceinline__ void mark_top(const Teacher& te, int top, int head, int nvec, uint32_t* bits) {
    const int words = ((nvec < kTakeBits ? nvec : kTakeBits) + 31) / 32;
    for (int i = threadIdx.x; i < words; i += NT) bits[i] = 0;
    __syncthreads();
    if ((int)threadIdx.x < top) {
        const int id = te.id[threadIdx.x];
        if (id >= head) {
            const int c = (id - head) / N;
            if (c < nvec) atomicOr(&bits[(c & (kTakeBits - 1)) >> 5], 1u << (c & 31));
        }
    }
    __syncthreads();
}

// dlogits of a loss over l: g ([j = t] - q_j) / T, g = dl of the row (or of its
// sequence) times the optional device scalars.
template <typename T, int NT>
__global__ __launch_bounds__(NT) void lp_bwd_k(int64_t rows, int vocab, bool vec, bool stream,
                                               const T* __restrict__ logits, const uint32_t* __restrict__ targets,
                                               int64_t ignore_index, LpScale k, const RowStat* __restrict__ stats,
                                               const float* __restrict__ dl, uint32_t seq,
                                               const float* __restrict__ scale, const float* __restrict__ dloss,
                                               T* __restrict__ dlogits) {
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
        zero_row<T, NT>(dr, vocab, stream);
        return;
    }
    g *= k.inv_t;
    write_row<T, NT>(logits + row * vocab, dr, vocab, vec, stream, -g, k.c_hi, stats[row], TakeOne{(int)t, g});
}

template <typename T, int NT>
__global__ __launch_bounds__(NT) void distill_bwd_k(mc_distill_desc d, bool vec, bool stream,
                                                    const T* __restrict__ logits, const int32_t* __restrict__ ids,
                                                    const float* __restrict__ tl, const float* __restrict__ tlse,
                                                    const uint8_t* __restrict__ mask, LpScale k,
                                                    const RowStat* __restrict__ stats, const float* __restrict__ scale,
                                                    const float* __restrict__ dloss, T* __restrict__ dlogits) {
    __shared__ float redf[4 * (NT / 64)];
    __shared__ Teacher te;
    __shared__ uint32_t bits[kTakeBits / 32];
    const int64_t row = d.rows - 1 - (int64_t)blockIdx.x;
    const int vocab = (int)d.vocab;
    T* dr = dlogits + row * vocab;
    float w = 0.f;
    TeacherSums ts{};
    if (!mask || mask[row] != 0) {
        ts = load_teacher<NT>(te, d, row, ids, tl, tlse, redf);
        w = scale[0] * (dloss ? dloss[0] : 1.f);
        if (ts.bad) w = __builtin_nanf("");
        if (ts.P == 0.f) w = 0.f;
    }
    if (w == 0.f) {
        zero_row<T, NT>(dr, vocab, stream);
        return;
    }
    const T* xr = logits + row * vocab;
    const RowSpan<T> span(xr, vocab);
    mark_top<NT, Vec16<T>::N>(te, d.top, (int)span.head, (int)span.nvec, bits);
    write_row<T, NT>(xr, dr, vocab, vec, stream, w * ts.P, k.c_hi, stats[row], TakeTop{te, bits, d.top, w});
}

// c = log2(e) / T as a float below it and the rest: with c_lo > 0, x c_lo has the
// sign of x c_hi, so an infinite x gives an infinity and no NaN.
LpScale row_scale(float temperature) {
    const double c = 1.4426950408889634074 / (double)temperature;
    LpScale k;
    k.c_hi = (float)c;
    if ((double)k.c_hi >= c) k.c_hi = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, k.c_hi) - 1);
    k.c_lo = (float)(c - (double)k.c_hi);
    k.inv_t = (float)(1.0 / (double)temperature);
    return k;
}

// fn(element type, threads per row)
template <typename F>
hipError_t by_row_kernel(int64_t rows, int64_t vocab, int dtype, F&& fn) {
    auto by_dtype = [&](auto threads) {
        if (dtype == MC_F32) fn(float{}, threads);
        else fn(uint16_t{}, threads);
    };
    if (xent_wide_rows(rows, vocab, dtype == MC_F32 ? 4 : 2)) by_dtype(std::integral_constant<int, 1024>{});
    else by_dtype(std::integral_constant<int, 256>{});
    return hipGetLastError();
}

bool same_start(const void* a, const void* b) {
    return ((reinterpret_cast<uintptr_t>(a) ^ reinterpret_cast<uintptr_t>(b)) & 15) == 0;
}

// Workgroups of the kernels that sum over rows, and rows of each: at most 256
// partial sums, which one workgroup then adds.
int64_t sum_chunk(int64_t rows) {
    const int64_t c = (rows + 255) / 256;
    return c < 256 ? 256 : c;
}

size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

}  // namespace

// ------------------------------------------------------------- launchers
hipError_t launch_token_logprobs_fwd(const mc_logprob_desc& d, const void* logits, const uint32_t* targets, float* logp,
                                     float* stats, uint32_t* counter, hipStream_t stream) {
    const LpScale k = row_scale(d.temperature);
    return by_row_kernel(d.rows, d.vocab, d.dtype, [&](auto elem, auto threads) {
        typedef decltype(elem) T;
        constexpr int NT = decltype(threads)::value;
        lp_rows_k<T, NT><<<dim3((unsigned)d.rows), NT, 0, stream>>>((int)d.vocab, static_cast<const T*>(logits),
                                                                    targets, d.ignore_index, k, logp,
                                                                    reinterpret_cast<RowStat*>(stats), counter);
    });
}

hipError_t launch_token_logprobs_bwd(const mc_logprob_desc& d, const void* logits, const uint32_t* targets,
                                     const float* stats, const float* dl, int64_t seq, const float* scale,
                                     const float* dloss, void* dlogits, hipStream_t stream) {
    const LpScale k = row_scale(d.temperature);
    const bool vec = same_start(logits, dlogits);
    return by_row_kernel(d.rows, d.vocab, d.dtype, [&](auto elem, auto threads) {
        typedef decltype(elem) T;
        constexpr int NT = decltype(threads)::value;
        lp_bwd_k<T, NT><<<dim3((unsigned)d.rows), NT, 0, stream>>>(
            d.rows, (int)d.vocab, vec, xent_stream_gradients(d.rows, d.vocab, sizeof(T)),
            static_cast<const T*>(logits), targets, d.ignore_index, k,
            reinterpret_cast<const RowStat*>(stats), dl, (uint32_t)seq, scale, dloss, static_cast<T*>(dlogits));
    });
}

PreferenceWs preference_ws(const mc_preference_desc& d) {
    PreferenceWs w;
    size_t at = 256;  // the counter
    w.logp = at;
    at += align256((size_t)(2 * d.pairs * d.seq) * sizeof(float));
    w.score = at;
    at += align256((size_t)(2 * d.pairs) * sizeof(double));
    w.inv_n = at;
    w.total = at + align256((size_t)(2 * d.pairs) * sizeof(float));
    return w;
}

hipError_t launch_preference_fwd(const mc_preference_desc& d, const void* logits, const uint32_t* targets,
                                 const float* ref, float* loss, float* rewards, float* stats, char* ws,
                                 hipStream_t stream) {
    const PreferenceWs w = preference_ws(d);
    const int64_t rows = 2 * d.pairs * d.seq;
    float* logp = reinterpret_cast<float*>(ws + w.logp);
    uint32_t* counter = reinterpret_cast<uint32_t*>(ws);
    const mc_logprob_desc lp{rows, d.vocab, d.ignore_index, 1.0f, d.dtype};
    hipError_t e = launch_token_logprobs_fwd(lp, logits, targets, logp, stats, counter, stream);
    if (e != hipSuccess) return e;
    preference_k<<<dim3((unsigned)(2 * d.pairs)), 256, 0, stream>>>(
        d, targets, logp, ref, reinterpret_cast<double*>(ws + w.score), reinterpret_cast<float*>(ws + w.inv_n), counter,
        loss, rewards, stats ? stats + 2 * rows : nullptr);
    return hipGetLastError();
}

PolicyWs policy_ws(const mc_policy_desc& d) {
    PolicyWs w;
    size_t at = 256;  // the counter
    w.part = at;
    at += 256 * 4 * sizeof(double);
    w.counts = at;
    if (d.reduction == MC_MEAN_SEQUENCES) at += align256((size_t)d.batch * sizeof(uint32_t));
    w.total = at;
    return w;
}

namespace {
const uint32_t* policy_counts(const mc_policy_desc& d, const uint32_t* targets, char* ws, hipStream_t stream,
                              hipError_t& e) {
    e = hipSuccess;
    if (d.reduction != MC_MEAN_SEQUENCES) return nullptr;
    uint32_t* n = reinterpret_cast<uint32_t*>(ws + policy_ws(d).counts);
    seq_counts_k<<<dim3((unsigned)((d.batch + 3) / 4)), 256, 0, stream>>>(d.batch, d.seq, targets, d.ignore_index, n);
    e = hipGetLastError();
    return n;
}
}  // namespace

hipError_t launch_policy_fwd(const mc_policy_desc& d, const void* logits, const uint32_t* targets, const float* adv,
                             const float* old, const float* ref, float* loss, float* logp, float* metrics,
                             float* stats, char* ws, hipStream_t stream) {
    const PolicyWs w = policy_ws(d);
    const int64_t rows = d.batch * d.seq, chunk = sum_chunk(rows);
    uint32_t* counter = reinterpret_cast<uint32_t*>(ws);
    const mc_logprob_desc lp{rows, d.vocab, d.ignore_index, d.temperature, d.dtype};
    hipError_t e;
    const uint32_t* n = policy_counts(d, targets, ws, stream, e);
    if (e != hipSuccess) return e;
    e = launch_token_logprobs_fwd(lp, logits, targets, logp, stats, counter, stream);
    if (e != hipSuccess) return e;
    policy_k<<<dim3((unsigned)((rows + chunk - 1) / chunk)), 256, 0, stream>>>(
        d, chunk, targets, logp, adv, old, ref, n, reinterpret_cast<double(*)[4]>(ws + w.part), counter, loss, metrics,
        stats ? stats + 2 * rows : nullptr);
    return hipGetLastError();
}

DistillWs distill_ws(const mc_distill_desc& d) {
    DistillWs w;
    size_t at = 256;  // the counter
    w.part = at;
    at += 256 * 2 * sizeof(double);
    w.kl = at;
    w.total = at + align256((size_t)d.rows * sizeof(float));
    return w;
}

hipError_t launch_distill_fwd(const mc_distill_desc& d, const void* logits, const int32_t* ids, const float* tl,
                              const float* tlse, const uint8_t* mask, float* loss, float* stats, char* ws,
                              hipStream_t stream) {
    const DistillWs w = distill_ws(d);
    const LpScale k = row_scale(d.temperature);
    uint32_t* counter = reinterpret_cast<uint32_t*>(ws);
    float* kl = reinterpret_cast<float*>(ws + w.kl);
    hipError_t e = by_row_kernel(d.rows, d.vocab, d.dtype, [&](auto elem, auto threads) {
        typedef decltype(elem) T;
        constexpr int NT = decltype(threads)::value;
        distill_rows_k<T, NT><<<dim3((unsigned)d.rows), NT, 0, stream>>>(d, static_cast<const T*>(logits), ids, tl,
                                                                         tlse, mask, k, kl,
                                                                         reinterpret_cast<RowStat*>(stats), counter);
    });
    if (e != hipSuccess) return e;
    const int64_t chunk = sum_chunk(d.rows);
    distill_final_k<<<dim3((unsigned)((d.rows + chunk - 1) / chunk)), 256, 0, stream>>>(
        d.rows, chunk, d.temperature, mask, kl, reinterpret_cast<double(*)[2]>(ws + w.part), counter, loss,
        stats ? stats + 2 * d.rows : nullptr);
    return hipGetLastError();
}

hipError_t launch_distill_bwd(const mc_distill_desc& d, const void* logits, const int32_t* ids, const float* tl,
                              const float* tlse, const uint8_t* mask, const float* stats, const float* dloss,
                              void* dlogits, hipStream_t stream) {
    const LpScale k = row_scale(d.temperature);
    const bool vec = same_start(logits, dlogits);
    return by_row_kernel(d.rows, d.vocab, d.dtype, [&](auto elem, auto threads) {
        typedef decltype(elem) T;
        constexpr int NT = decltype(threads)::value;
        distill_bwd_k<T, NT><<<dim3((unsigned)d.rows), NT, 0, stream>>>(
            d, vec, xent_stream_gradients(d.rows, d.vocab, sizeof(T)), static_cast<const T*>(logits), ids, tl, tlse,
            mask, k, reinterpret_cast<const RowStat*>(stats), stats + 2 * d.rows, dloss, static_cast<T*>(dlogits));
    });
}

size_t policy_fwd_bwd_ws(const mc_policy_desc& d) {
    return policy_ws(d).total + align256((size_t)(3 * d.batch * d.seq + 1) * sizeof(float));
}

hipError_t launch_policy_fwd_bwd(const mc_policy_desc& d, const void* logits, const uint32_t* targets,
                                 const float* adv, const float* old, const float* ref, const float* dloss, float* loss,
                                 float* logp, float* metrics, void* dlogits, char* ws, hipStream_t stream) {
    float* stats = reinterpret_cast<float*>(ws + policy_ws(d).total);
    const int64_t rows = d.batch * d.seq;
    hipError_t e = launch_policy_fwd(d, logits, targets, adv, old, ref, loss, logp, metrics, stats, ws, stream);
    if (e != hipSuccess) return e;
    const mc_logprob_desc lp{rows, d.vocab, d.ignore_index, d.temperature, d.dtype};
    return launch_token_logprobs_bwd(lp, logits, targets, stats, stats + 2 * rows, 0, stats + 3 * rows, dloss, dlogits,
                                     stream);
}

size_t distill_fwd_bwd_ws(const mc_distill_desc& d) {
    return distill_ws(d).total + align256((size_t)(2 * d.rows + 1) * sizeof(float));
}

hipError_t launch_distill_fwd_bwd(const mc_distill_desc& d, const void* logits, const int32_t* ids, const float* tl,
                                  const float* tlse, const uint8_t* mask, const float* dloss, float* loss,
                                  void* dlogits, char* ws, hipStream_t stream) {
    float* stats = reinterpret_cast<float*>(ws + distill_ws(d).total);
    hipError_t e = launch_distill_fwd(d, logits, ids, tl, tlse, mask, loss, stats, ws, stream);
    if (e != hipSuccess) return e;
    return launch_distill_bwd(d, logits, ids, tl, tlse, mask, stats, dloss, dlogits, stream);
}

}  // namespace mc
