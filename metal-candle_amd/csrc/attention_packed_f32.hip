// The float32 side of attention over packed rows (attention_packed.hip has the
// formulas), and the row kernels for head dims without tiles, gfx950.
//
// The tile kernels are shaped as those of attention_f32.hip, on whose products and
// LDS tiles they stand (attention_f32_tiles.hpp): a workgroup owns 32 queries
// (dK/dV: 32 keys) of one head, its four waves take every fourth block of 32 keys
// (queries) between the first and the last that any of them sees. They are bound
// by the float32 matrix rate, beside which the arithmetic of the cap is small: it
// is chosen at run time, and its tanh is exact to about 2^-23.
//
// 4 x 12 (2) x 509 x 64 in documents of 75 tokens, capped: forward 25 us, dQ 35, dK/dV
// 46, its groups' sum 5: 768 workgroups each, all resident, whose waves have one or two
// blocks of 32 x 32 pairs: a chain of loads, products, scores and the waves' join.
//
// Row kernels (bf16 head dims other than 64 and 128, float32 ones that are no
// multiple of 4 or past 128, and float32 rows of a few tokens): one wave per row,
// lanes over the head dim, only what the row sees is read. Per key they wait for two
// rows and one or two sums over the lanes: 2 x 8 (4) x 1024 x 256 bf16, causal and capped,
// forward 3.5 ms, backward 8.4; of 96 1.3 and 3.8; 1 x 14 (2) x 300 x 40 0.16 and 1.4.
#include <type_traits>

#include "attention_f32_tiles.hpp"
#include "attention_spans.hpp"
#include "common.hpp"
#include "kernels.hpp"
#include "rules.hpp"

namespace mc {
namespace {

using namespace attn;
using namespace attn32;

// The scores' arithmetic in natural units. cap = 0: none.
struct ScoreMods {
    float scale, cap, inv_cap;
};

// tanh(u): below 0.35 its power series up to u^11 (the next term is 1.2e-8 of the
// value), above 1 - 2 / (e^2|u| + 1).
__device__ __forceinline__ float tanh_f32(float u) {
    const float x = u * u;
    float p = -1382.f / 155925.f;
    p = __builtin_fmaf(p, x, 62.f / 2835.f);
    p = __builtin_fmaf(p, x, -17.f / 315.f);
    p = __builtin_fmaf(p, x, 2.f / 15.f);
    p = __builtin_fmaf(p, x, -1.f / 3.f);
    const float small = __builtin_fmaf(p * x, u, u);
    const float big = 1.f - 2.f * __builtin_amdgcn_rcpf(exp2_hw(2.f * kLog2e * __builtin_fabsf(u)) + 1.f);
    return __builtin_fabsf(u) < 0.35f ? small : __builtin_copysignf(big, u);
}
// The score of a product s at distance far; slope: its derivative by scale s.
__device__ __forceinline__ float score_of(float s, float far, const ScoreMods& m, float bias, float& slope) {
    float x = s * m.scale;
    slope = 1.f;
    if (m.cap != 0.f) {
        const float t = tanh_f32(x * m.inv_cap);
        x = t * m.cap;
        slope = __builtin_fmaf(-t, t, 1.f);
    }
    return __builtin_fmaf(-bias, far, x);
}

struct PackedF32Args {
    const float *q, *k, *v, *o, *dout;
    const int4* spans;
    const float* slopes;
    float *out, *lse;  // forward outputs (lse may be null; the backward's input)
    float* delta;      // backward: rowsum(dO (.) O) [B, H, S]
    float *dq, *dk, *dv;
    int64_t S;
    int B, H, Hkv, D, nblk, causal, groups;
    ScoreMods mods;
};

// The union of the spans of a tile's 32 tokens, lane l holding token l % 32.
__device__ __forceinline__ Span tile_span(Span s) {
    int lo = s.lo < s.hi ? s.lo : 0x7fffffff, hi = s.hi;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
        const int a = __shfl_xor(lo, m, kWave), b = __shfl_xor(hi, m, kWave);
        lo = a < lo ? a : lo;
        hi = b > hi ? b : hi;
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    hi = __builtin_amdgcn_readfirstlane(hi);
    return lo < hi ? Span{lo, hi} : Span{0, 0};
}

// add_nonfinite of attention_f32.hip for any span: rows of the tile are visible
// to this lane inside [lo, hi).
template <int DP>
__device__ __forceinline__ void add_nonfinite_in(float* tile, const f32x16& p, f32x16 (&acc)[DP / 32], int lo, int hi) {
    constexpr int DT = DP / 32, LD = Tile32<DP>::LD;
    const int lane = lane_id(), col = lane & 31, h = lane >> 5;
#pragma unroll 1
    for (int r = 0; r < 32; ++r) {  // row r is register 4 (r / 8) + r % 4 of lane half (r / 4) % 2
        const float pr = __shfl(p[4 * (r >> 3) + (r & 3)], col + 32 * ((r >> 2) & 1), kWave);
        const bool visible = r >= lo && r < hi;
#pragma unroll
        for (int g = 0; g < 16; ++g)
#pragma unroll
            for (int t = 0; t < DT; ++t) {
                const float v = tile[r * LD + DT * acc_row(g, h) + t];
                acc[t][g] += visible && nonfinite(v) ? pr * v : 0.f;
            }
    }
    wave_lds_fence();
#pragma unroll 1
    for (int i = lane; i < Tile32<DP>::FLOATS; i += 64)
        if (nonfinite(tile[i])) tile[i] = 0.f;
    wave_lds_fence();
}

// ---------------------------------------------------------------- forward
template <int DP>
__global__ __launch_bounds__(256, kWgPerCu<DP>) void packed_f32_fwd(PackedF32Args a) {
    typedef Tile32<DP> TL;
    constexpr int DT = TL::DT;
    __shared__ __attribute__((aligned(16))) float tiles[4][TL::FLOATS];
    __shared__ float stat[4][2][32];
    const int lane = lane_id(), wave = wave_id(), col = lane & 31, h = lane >> 5;
    const int nbh = a.B * a.H;
    const int qb = a.nblk - 1 - (int)(blockIdx.x / nbh);  // heaviest (causal) query blocks first
    const int bh = head_of((int)(blockIdx.x % nbh), nbh);
    const int b = bh / a.H, hq = bh % a.H;
    const int64_t S = a.S, D = a.D;
    const int64_t bhk = (int64_t)b * a.Hkv + hq / (a.H / a.Hkv);
    const int64_t q0 = (int64_t)qb * 32, qi = q0 + col;
    const float *kh = a.k + bhk * S * D, *vh = a.v + bhk * S * D;
    const float bias = a.slopes ? a.slopes[hq] : 0.f;
    float* kt = tiles[wave];

    f32x4 qf[DP / 8];
    TL::load_along_d(TL::rsrc(a.q + (int64_t)bh * S * D, q0, S, D, a.D), a.D, a.D, qf);
    const Span mine = query_span(a.spans, b, qi, (int)S, a.causal);
    const Span all = tile_span(mine);
    const int kb0 = all.lo / 32, kb1 = (all.hi + 31) / 32;
    float m = kNegInf, l = 0.f;
    f32x16 acc[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t) acc[t] = zero16();

    f32x4 kr[TL::LOADS];
    if (kb0 + wave < kb1) TL::load(TL::rsrc(kh, (int64_t)(kb0 + wave) * 32, S, D, a.D), a.D, a.D, kr);
    for (int kb = kb0 + wave; kb < kb1; kb += 4) {
        const int64_t k0 = (int64_t)kb * 32;
        TL::store(kt, kr);
        // V rows of this block, one step's operand per register group
        typename TL::vec vr[16];
        {
            const __amdgpu_buffer_rsrc_t rv = TL::rsrc(vh, k0, S, D, a.D);
            const uint32_t d0 = (uint32_t)(DT * col);
#pragma unroll
            for (int q = 0; q < 16; ++q) {
                const int off = (int)(d0 < (uint32_t)a.D ? ((uint32_t)acc_row(q, h) * (uint32_t)a.D + d0) * 4u : kOOB);
                if constexpr (DT == 4)
                    vr[q] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rv, off, 0, 0));
                else if constexpr (DT == 2)
                    vr[q] = __builtin_bit_cast(typename TL::vec, __builtin_amdgcn_raw_buffer_load_b64(rv, off, 0, 0));
                else
                    vr[q][0] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rv, off, 0, 0));
            }
        }
        wave_lds_fence();
        f32x16 s = mma_d<DP>(kt, [&](int j) { return qf[j]; });  // S^T: lane = query, registers = keys
        wave_lds_fence();
        if (kb + 4 < kb1) TL::load(TL::rsrc(kh, k0 + 128, S, D, a.D), a.D, a.D, kr);
        const float dist = (float)(int)(qi - k0 - 4 * h);
        float slope;
#pragma unroll
        for (int q = 0; q < 16; ++q)
            s[q] = score_of(s[q], __builtin_fabsf(dist - (float)acc_row(q, 0)), a.mods, bias, slope);
        const int lo = mine.lo - (int)k0 - 4 * h, hi = mine.hi - (int)k0 - 4 * h;
        const bool edge = __any(lo > -4 * h || hi < 32 - 4 * h);
        if (edge) {
#pragma unroll
            for (int q = 0; q < 16; ++q)
                if (acc_row(q, 0) < lo || acc_row(q, 0) >= hi) s[q] = kNegInf;
        }
        float mb = s[0];
#pragma unroll
        for (int q = 1; q < 16; ++q) mb = fmaxf(mb, s[q]);
        mb = fmaxf(mb, half_swap(mb));
        const float mn = fmaxf(m, mb);
        const float mu = mn == kNegInf ? 0.f : mn;  // no key seen yet: p = 0
        if (__any(mn != m)) {
            const float alpha = exp2_hw((m - mu) * kLog2e);
            l *= alpha;
#pragma unroll
            for (int t = 0; t < DT; ++t)
#pragma unroll
                for (int q = 0; q < 16; ++q) acc[t][q] *= alpha;
            m = mn;
        }
        float lb = 0.f;
#pragma unroll
        for (int q = 0; q < 16; ++q) {
            s[q] = exp2_hw((s[q] - mu) * kLog2e);
            lb += s[q];
        }
        l += lb;
        if (edge) {
            bool bad = false;
#pragma unroll
            for (int q = 0; q < 16; ++q)
#pragma unroll
                for (int t = 0; t < DT; ++t) bad |= nonfinite(vr[q][t]);
            if (__any(bad)) {
#pragma unroll
                for (int q = 0; q < 16; ++q)
                    *reinterpret_cast<typename TL::vec*>(&kt[acc_row(q, h) * TL::LD + DT * col]) = vr[q];
                wave_lds_fence();
                add_nonfinite_in<DP>(kt, s, acc, lo + 4 * h, hi + 4 * h);
#pragma unroll
                for (int q = 0; q < 16; ++q) vr[q] = TL::along_rows(kt, q);
                wave_lds_fence();
            }
        }
#pragma unroll
        for (int q = 0; q < 16; ++q)
#pragma unroll
            for (int t = 0; t < DT; ++t)
                acc[t] = __builtin_amdgcn_mfma_f32_32x32x2f32(vr[q][t], s[q], acc[t], 0, 0, 0);
    }
    l += half_swap(l);
    if (h == 0) {
        stat[wave][0][col] = m;
        stat[wave][1][col] = l;
    }
    wave_lds_fence();
    TL::store_acc(kt, acc);
    __syncthreads();
    // o = sum_w O_w 2^(m_w - M) / sum_w l_w 2^(m_w - M), waves in order
#pragma unroll
    for (int i = 0; i < DT; ++i) {
        const int ch = (int)threadIdx.x + 256 * i, row = ch / TL::CPR, d = 4 * (ch % TL::CPR);
        float M = stat[0][0][row];
#pragma unroll
        for (int w = 1; w < 4; ++w) M = fmaxf(M, stat[w][0][row]);
        const float mu = M == kNegInf ? 0.f : M;
        float L = 0.f;
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float e = exp2_hw((stat[w][0][row] - mu) * kLog2e);
            L += stat[w][1][row] * e;
            const f32x4 x = *reinterpret_cast<const f32x4*>(&tiles[w][row * TL::LD + d]);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] += x[j] * e;
        }
        const int64_t qr = q0 + row;
        if (qr >= S) continue;
        const Span see = query_span(a.spans, b, qr, (int)S, a.causal);
        const bool sees = see.lo < see.hi;  // o = 0 and lse = -inf for a query that sees nothing
        const float inv = sees ? 1.f / L : 0.f;
        if (d < a.D)
            *reinterpret_cast<f32x4*>(&a.out[(((int64_t)b * S + qr) * a.H + hq) * D + d]) =
                f32x4{v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv};
        if (d == 0 && a.lse) a.lse[(int64_t)bh * S + qr] = sees ? M + logf(L) : kNegInf;
    }
}

// ------------------------------------------------------------- dQ (and Delta)
// Shaped like the forward; it runs before dK/dV and also writes Delta.
template <int DP>
__global__ __launch_bounds__(256, kWgPerCu<DP>) void packed_f32_dq(PackedF32Args a) {
    typedef Tile32<DP> TL;
    constexpr int DT = TL::DT;
    __shared__ __attribute__((aligned(16))) float tiles[4][2][TL::FLOATS];
    __shared__ float sdelta[32];
    const int lane = lane_id(), wave = wave_id(), col = lane & 31, h = lane >> 5;
    const int nbh = a.B * a.H;
    const int qb = a.nblk - 1 - (int)(blockIdx.x / nbh);
    const int bh = head_of((int)(blockIdx.x % nbh), nbh);
    const int b = bh / a.H, hq = bh % a.H;
    const int64_t S = a.S, D = a.D, HD = (int64_t)a.H * D;
    const int64_t bhk = (int64_t)b * a.Hkv + hq / (a.H / a.Hkv);
    const int64_t q0 = (int64_t)qb * 32, qi = q0 + col;
    const float *kh = a.k + bhk * S * D, *vh = a.v + bhk * S * D;
    const int64_t obase = (int64_t)b * S * HD + (int64_t)hq * D;
    const float bias = a.slopes ? a.slopes[hq] : 0.f;
    float *kt = tiles[wave][0], *vt = tiles[wave][1];

    {  // Delta: 8 threads per query, in a fixed order
        const int row = (int)threadIdx.x >> 3, part = (int)threadIdx.x & 7;
        float s = 0.f;
        if (q0 + row < S) {
            const int64_t base = obase + (q0 + row) * HD;
            for (int d = 4 * part; d < a.D; d += 32) {
                const f32x4 x = *reinterpret_cast<const f32x4*>(a.o + base + d);
                const f32x4 y = *reinterpret_cast<const f32x4*>(a.dout + base + d);
                s += (x[0] * y[0] + x[1] * y[1]) + (x[2] * y[2] + x[3] * y[3]);
            }
        }
        s += __shfl_xor(s, 1, kWave);
        s += __shfl_xor(s, 2, kWave);
        s += __shfl_xor(s, 4, kWave);
        if (part == 0) {
            sdelta[row] = s;
            if (q0 + row < S) a.delta[(int64_t)bh * S + q0 + row] = s;
        }
    }
    f32x4 qf[DP / 8], gf[DP / 8];
    TL::load_along_d(TL::rsrc(a.q + (int64_t)bh * S * D, q0, S, D, a.D), a.D, a.D, qf);
    TL::load_along_d(TL::rsrc(a.dout + obase, q0, S, HD, a.D), (uint32_t)HD, a.D, gf);
    const float li = qi < S ? a.lse[(int64_t)bh * S + qi] : 0.f;
    const Span mine = query_span(a.spans, b, qi, (int)S, a.causal);
    const Span all = tile_span(mine);
    __syncthreads();
    const float di = sdelta[col];
    const int kb0 = all.lo / 32, kb1 = (all.hi + 31) / 32;
    f32x16 acc[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t) acc[t] = zero16();

    f32x4 kr[TL::LOADS], vr[TL::LOADS];
    if (kb0 + wave < kb1) {
        TL::load(TL::rsrc(kh, (int64_t)(kb0 + wave) * 32, S, D, a.D), a.D, a.D, kr);
        TL::load(TL::rsrc(vh, (int64_t)(kb0 + wave) * 32, S, D, a.D), a.D, a.D, vr);
    }
    for (int kb = kb0 + wave; kb < kb1; kb += 4) {
        const int64_t k0 = (int64_t)kb * 32;
        TL::store(kt, kr);
        TL::store(vt, vr);
        // hidden keys of the block: not before lo, nor from hi on, from row 4 h
        const int lo = mine.lo - (int)k0 - 4 * h, hi = mine.hi - (int)k0 - 4 * h;
        const bool edge = __any(lo > -4 * h || hi < 32 - 4 * h);
        const bool bad = edge && any_nonfinite(kr);
        wave_lds_fence();
        if (kb + 4 < kb1) {
            TL::load(TL::rsrc(kh, k0 + 128, S, D, a.D), a.D, a.D, kr);
            TL::load(TL::rsrc(vh, k0 + 128, S, D, a.D), a.D, a.D, vr);
        }
        f32x16 s = mma_d<DP>(kt, [&](int j) { return qf[j]; });
        const f32x16 dp = mma_d<DP>(vt, [&](int j) { return gf[j]; });
        const float dist = (float)(int)(qi - k0 - 4 * h);
#pragma unroll
        for (int q = 0; q < 16; ++q) {
            float slope;
            const float x = score_of(s[q], __builtin_fabsf(dist - (float)acc_row(q, 0)), a.mods, bias, slope);
            const float ds = exp2_hw((x - li) * kLog2e) * ((dp[q] - di) * slope);
            s[q] = acc_row(q, 0) < lo || acc_row(q, 0) >= hi ? 0.f : ds;
        }
        if (bad) add_nonfinite_in<DP>(kt, s, acc, lo + 4 * h, hi + 4 * h);
        mma_rows<DP>(kt, s, acc);
        wave_lds_fence();
    }
    TL::store_acc(kt, acc);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < DT; ++i) {
        const int ch = (int)threadIdx.x + 256 * i, row = ch / TL::CPR, d = 4 * (ch % TL::CPR);
        f32x4 v = *reinterpret_cast<const f32x4*>(&tiles[0][0][row * TL::LD + d]);
#pragma unroll
        for (int w = 1; w < 4; ++w) v += *reinterpret_cast<const f32x4*>(&tiles[w][0][row * TL::LD + d]);
        if (q0 + row < S && d < a.D)
            *reinterpret_cast<f32x4*>(&a.dq[((int64_t)bh * S + q0 + row) * D + d]) = v * a.mods.scale;
    }
}

// -------------------------------------------------------------------- dK, dV
template <int DP>
__global__ __launch_bounds__(256, kWgPerCu<DP>) void packed_f32_dkdv(PackedF32Args a) {
    typedef Tile32<DP> TL;
    constexpr int DT = TL::DT;
    __shared__ __attribute__((aligned(16))) float tiles[4][2][TL::FLOATS];
    __shared__ __attribute__((aligned(16))) float vtile[TL::FLOATS];  // the workgroup's V rows
    __shared__ __attribute__((aligned(16))) float stat[4][2][32];     // lse, Delta of the wave's queries
    const int lane = lane_id(), wave = wave_id(), col = lane & 31, h = lane >> 5;
    const int ngrp = a.B * a.Hkv * a.groups;
    const int kb = (int)(blockIdx.x / ngrp);  // heaviest (causal) key blocks first
    const int grp = head_of((int)(blockIdx.x % ngrp), ngrp);
    const int b = grp / (a.Hkv * a.groups), hk = grp / a.groups % a.Hkv, g = grp % a.groups;
    const int rep = a.H / a.Hkv, per = rep / a.groups;  // query heads per K/V head, per group
    const int64_t S = a.S, D = a.D, HD = (int64_t)a.H * D;
    const int64_t k0 = (int64_t)kb * 32, bhk = (int64_t)b * a.Hkv + hk, key = k0 + col;
    float *qt = tiles[wave][0], *gt = tiles[wave][1];

    f32x4 kf[DP / 8];
    TL::load_along_d(TL::rsrc(a.k + bhk * S * D, k0, S, D, a.D), a.D, a.D, kf);
    if (wave == 0) {
        f32x4 t[TL::LOADS];
        TL::load(TL::rsrc(a.v + bhk * S * D, k0, S, D, a.D), a.D, a.D, t);
        TL::store(vtile, t);
    }
    const Span mine = key_span(a.spans, b, key, (int)S, a.causal);
    const Span all = tile_span(mine);
    __syncthreads();
    const int first = all.lo / 32, nqb = (all.hi + 31) / 32 - first, total = nqb * per;
    f32x16 ak[DT], av[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t) ak[t] = av[t] = zero16();

    f32x4 qr[TL::LOADS], gr[TL::LOADS];
    float st = 0.f;
    // the next block's rows are requested in two steps, each once the registers
    // of a finished product are free
    auto fetch_q = [&](int it) {
        const int hq = hk * rep + g * per + it / nqb;
        const int64_t bh = (int64_t)b * a.H + hq, q0 = (int64_t)(first + it % nqb) * 32;
        TL::load(TL::rsrc(a.q + bh * S * D, q0, S, D, a.D), a.D, a.D, qr);
        st = q0 + col < S ? (h ? a.delta : a.lse)[bh * S + q0 + col] : 0.f;
    };
    auto fetch_g = [&](int it) {
        const int hq = hk * rep + g * per + it / nqb;
        const int64_t q0 = (int64_t)(first + it % nqb) * 32;
        TL::load(TL::rsrc(a.dout + (int64_t)b * S * HD + (int64_t)hq * D, q0, S, HD, a.D), (uint32_t)HD, a.D, gr);
    };
    if (wave < total) {
        fetch_q(wave);
        fetch_g(wave);
    }
    for (int it = wave; it < total; it += 4) {
        const int64_t q0 = (int64_t)(first + it % nqb) * 32;
        const float bias = a.slopes ? a.slopes[hk * rep + g * per + it / nqb] : 0.f;
        TL::store(qt, qr);
        TL::store(gt, gr);
        stat[wave][h][col] = st;
        // hidden queries of the block: not before lo, nor from hi on, from row 4 h
        const int lo = mine.lo - (int)q0 - 4 * h, hi = mine.hi - (int)q0 - 4 * h;
        const bool edge = __any(lo > -4 * h || hi < 32 - 4 * h);
        const bool bad = edge && (any_nonfinite(qr) || any_nonfinite(gr));
        wave_lds_fence();
        f32x16 s = mma_d<DP>(qt, [&](int j) { return kf[j]; });
        f32x16 dp = mma_d<DP>(gt, [&](int j) { return TL::along_d(vtile, j); });
        if (it + 4 < total) fetch_q(it + 4);
        const float dist = (float)(int)(q0 + 4 * h - key);
#pragma unroll
        for (int g4 = 0; g4 < 4; ++g4) {
            const f32x4 li = *reinterpret_cast<const f32x4*>(&stat[wave][0][8 * g4 + 4 * h]);
            const f32x4 di = *reinterpret_cast<const f32x4*>(&stat[wave][1][8 * g4 + 4 * h]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int q = 4 * g4 + e;
                float slope;
                const float x = score_of(s[q], __builtin_fabsf(dist + (float)acc_row(q, 0)), a.mods, bias, slope);
                const bool off = acc_row(q, 0) < lo || acc_row(q, 0) >= hi;
                const float p = exp2_hw(off ? kNegInf : (x - li[e]) * kLog2e);
                const float ds = p * ((dp[q] - di[e]) * slope);
                s[q] = p;
                dp[q] = off ? 0.f : ds;
            }
            __builtin_amdgcn_sched_barrier(0);  // lse and Delta of one row group at a time
        }
        if (bad) {
            add_nonfinite_in<DP>(gt, s, av, lo + 4 * h, hi + 4 * h);
            add_nonfinite_in<DP>(qt, dp, ak, lo + 4 * h, hi + 4 * h);
        }
        mma_rows<DP>(gt, s, av);
        if (it + 4 < total) fetch_g(it + 4);
        mma_rows<DP>(qt, dp, ak);
        wave_lds_fence();
    }
    TL::store_acc(qt, ak);
    TL::store_acc(gt, av);
    __syncthreads();
    const int64_t part = (bhk * a.groups + g) * S;  // groups == 1: the outputs themselves
#pragma unroll
    for (int i = 0; i < 2 * DT; ++i) {
        const int which = i / DT, ch = (int)threadIdx.x + 256 * (i % DT), row = ch / TL::CPR, d = 4 * (ch % TL::CPR);
        f32x4 v = *reinterpret_cast<const f32x4*>(&tiles[0][which][row * TL::LD + d]);
#pragma unroll
        for (int w = 1; w < 4; ++w) v += *reinterpret_cast<const f32x4*>(&tiles[w][which][row * TL::LD + d]);
        if (which == 0) v *= a.mods.scale;
        if (k0 + row < S && d < a.D)
            *reinterpret_cast<f32x4*>(&(which ? a.dv : a.dk)[(part + k0 + row) * D + d]) = v;
    }
}

__global__ __launch_bounds__(256) void packed_f32_sum(const f32x4* __restrict__ pk, const f32x4* __restrict__ pv,
                                                      f32x4* __restrict__ dk, f32x4* __restrict__ dv, int groups,
                                                      int64_t per_head4, int64_t n4) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= 2 * n4) return;
    const bool second = i >= n4;
    const int64_t j = second ? i - n4 : i;
    const f32x4* src = (second ? pv : pk) + j / per_head4 * per_head4 * groups + j % per_head4;
    f32x4 v = src[0];
    for (int g = 1; g < groups; ++g) v += src[g * per_head4];
    (second ? dv : dk)[j] = v;
}

// ------------------------------------------------------------ row kernels
// One wave per row; lane l holds dims l, l + 64, l + 128, l + 192.
template <typename T> struct Rows {
    const T *q, *k, *v, *dout;
    const int4* spans;
    const float* slopes;
    T *o, *dq, *dk, *dv;
    float *lse, *delta;
    int64_t S;
    int B, H, Hkv, D, causal;
    ScoreMods mods;
};
template <typename T>
__device__ __forceinline__ void row_load(const T* p, int D, float (&v)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int d = lane_id() + 64 * i;
        v[i] = d < D ? Elem<T>::load(p, d) : 0.f;
    }
}
template <typename T>
__device__ __forceinline__ void row_store(T* p, int D, const float (&v)[4], float f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int d = lane_id() + 64 * i;
        if (d < D) Elem<T>::store(p, d, v[i] * f);
    }
}
__device__ __forceinline__ float row_dot(const float (&x)[4], const float (&y)[4]) {
    return wave_sum((x[0] * y[0] + x[1] * y[1]) + (x[2] * y[2] + x[3] * y[3]));
}

template <typename T>
__global__ __launch_bounds__(256) void packed_rows_fwd(Rows<T> a) {
    const int64_t row = (int64_t)blockIdx.x * 4 + wave_id();
    if (row >= (int64_t)a.B * a.H * a.S) return;
    const int64_t bh = row / a.S, qi = row % a.S;
    const int b = (int)(bh / a.H), h = (int)(bh % a.H);
    const int64_t bhk = (int64_t)b * a.Hkv + h / (a.H / a.Hkv);
    const Span see = query_span(a.spans, b, qi, (int)a.S, a.causal);
    const float bias = a.slopes ? a.slopes[h] : 0.f;
    float qv[4], acc[4] = {0.f, 0.f, 0.f, 0.f};
    row_load(a.q + row * a.D, a.D, qv);
    float m = kNegInf, l = 0.f;
    for (int key = see.lo; key < see.hi; ++key) {
        const int64_t kr = (bhk * a.S + key) * a.D;
        float kv[4], vv[4], slope;
        row_load(a.k + kr, a.D, kv);
        row_load(a.v + kr, a.D, vv);
        const float s = score_of(row_dot(qv, kv), __builtin_fabsf((float)((int)qi - key)), a.mods, bias, slope);
        const float mn = fmaxf(m, s), mu = mn == kNegInf ? 0.f : mn;
        const float alpha = exp2_hw((m - mu) * kLog2e), p = exp2_hw((s - mu) * kLog2e);
        l = l * alpha + p;
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] = acc[i] * alpha + p * vv[i];
        m = mn;
    }
    const bool sees = see.lo < see.hi;
    row_store(a.o + (((int64_t)b * a.S + qi) * a.H + h) * a.D, a.D, acc, sees ? 1.f / l : 0.f);
    if (a.lse && lane_id() == 0) a.lse[row] = sees ? m + logf(l) : kNegInf;
}

// Also writes Delta, for packed_rows_dkdv. bf16: as sum P dP / sum P, since o's
// rounding to bf16 would stay in the gradients of queries that see few keys; it is
// known behind the last key, so dq is scale (sum P dP slope k - Delta sum P slope k).
template <typename T>
__global__ __launch_bounds__(256) void packed_rows_dq(Rows<T> a) {
    const int64_t row = (int64_t)blockIdx.x * 4 + wave_id();
    if (row >= (int64_t)a.B * a.H * a.S) return;
    const int64_t bh = row / a.S, qi = row % a.S;
    const int b = (int)(bh / a.H), h = (int)(bh % a.H);
    const int64_t bhk = (int64_t)b * a.Hkv + h / (a.H / a.Hkv);
    const int64_t orow = (((int64_t)b * a.S + qi) * a.H + h) * a.D;
    const Span see = query_span(a.spans, b, qi, (int)a.S, a.causal);
    const float bias = a.slopes ? a.slopes[h] : 0.f;
    constexpr bool kFromP = sizeof(T) == 2;
    float qv[4], gv[4], acc[4] = {0.f, 0.f, 0.f, 0.f}, base[4] = {0.f, 0.f, 0.f, 0.f};
    row_load(a.q + row * a.D, a.D, qv);
    row_load(a.dout + orow, a.D, gv);
    float di = 0.f, sum_p = 0.f;
    if constexpr (!kFromP) {
        float ov[4];
        row_load(a.o + orow, a.D, ov);
        di = row_dot(ov, gv);
    }
    const float li = a.lse[row];
    for (int key = see.lo; key < see.hi; ++key) {
        const int64_t kr = (bhk * a.S + key) * a.D;
        float kv[4], vv[4], slope;
        row_load(a.k + kr, a.D, kv);
        row_load(a.v + kr, a.D, vv);
        const float s = score_of(row_dot(qv, kv), __builtin_fabsf((float)((int)qi - key)), a.mods, bias, slope);
        const float p = exp2_hw((s - li) * kLog2e), dp = row_dot(gv, vv);
        if constexpr (kFromP) {
            sum_p += p;
            di = __builtin_fmaf(p, dp, di);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                acc[i] += p * dp * slope * kv[i];
                base[i] += p * slope * kv[i];
            }
        } else {
            const float ds = p * ((dp - di) * slope);
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[i] += ds * kv[i];
        }
    }
    if constexpr (kFromP) {
        if (sum_p > 0.f) di /= sum_p;
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] = __builtin_fmaf(-di, base[i], acc[i]);
    }
    if (lane_id() == 0) a.delta[row] = di;
    row_store(a.dq + row * a.D, a.D, acc, a.mods.scale);
}

template <typename T>
__global__ __launch_bounds__(256) void packed_rows_dkdv(Rows<T> a) {
    const int64_t row = (int64_t)blockIdx.x * 4 + wave_id();  // (b, hk, j)
    if (row >= (int64_t)a.B * a.Hkv * a.S) return;
    const int64_t bhk = row / a.S, key = row % a.S;
    const int b = (int)(bhk / a.Hkv), hk = (int)(bhk % a.Hkv), rep = a.H / a.Hkv;
    const Span see = key_span(a.spans, b, key, (int)a.S, a.causal);
    float kv[4], vv[4], gk[4] = {0.f, 0.f, 0.f, 0.f}, gvv[4] = {0.f, 0.f, 0.f, 0.f};
    row_load(a.k + row * a.D, a.D, kv);
    row_load(a.v + row * a.D, a.D, vv);
    for (int h = hk * rep; h < (hk + 1) * rep; ++h) {
        const int64_t bh = (int64_t)b * a.H + h;
        const float bias = a.slopes ? a.slopes[h] : 0.f;
        for (int i = see.lo; i < see.hi; ++i) {
            float qv[4], gv[4], slope;
            row_load(a.q + (bh * a.S + i) * a.D, a.D, qv);
            row_load(a.dout + (((int64_t)b * a.S + i) * a.H + h) * a.D, a.D, gv);
            const float s = score_of(row_dot(qv, kv), __builtin_fabsf((float)(i - (int)key)), a.mods, bias, slope);
            const float p = exp2_hw((s - a.lse[bh * a.S + i]) * kLog2e);
            const float ds = p * ((row_dot(gv, vv) - a.delta[bh * a.S + i]) * slope);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                gk[u] += ds * qv[u];
                gvv[u] += p * gv[u];
            }
        }
    }
    row_store(a.dk + row * a.D, a.D, gk, a.mods.scale);
    row_store(a.dv + row * a.D, a.D, gvv, 1.f);
}

ScoreMods mods_of(const mc_packed_attn_desc& d) {
    return ScoreMods{d.attn.scale, d.cap, d.cap != 0.f ? 1.f / d.cap : 0.f};
}

PackedF32Args f32_args(const mc_packed_attn_desc& p, const void* q, const void* k, const void* v, const int32_t* spans,
                       const float* slopes) {
    const mc_attn_desc& d = p.attn;
    PackedF32Args a{};
    a.q = static_cast<const float*>(q);
    a.k = static_cast<const float*>(k);
    a.v = static_cast<const float*>(v);
    a.spans = reinterpret_cast<const int4*>(spans);
    a.slopes = slopes;
    a.S = d.seq;
    a.B = (int)d.batch; a.H = d.heads; a.Hkv = d.kv_heads; a.D = d.head_dim;
    a.nblk = (int)((d.seq + 31) / 32);
    a.causal = d.causal ? 1 : 0;
    a.groups = 1;
    a.mods = mods_of(p);
    return a;
}

template <typename T>
Rows<T> row_args(const mc_packed_attn_desc& p, const void* q, const void* k, const void* v, const int32_t* spans,
                 const float* slopes) {
    const mc_attn_desc& d = p.attn;
    Rows<T> a{};
    a.q = static_cast<const T*>(q);
    a.k = static_cast<const T*>(k);
    a.v = static_cast<const T*>(v);
    a.spans = reinterpret_cast<const int4*>(spans);
    a.slopes = slopes;
    a.S = d.seq;
    a.B = (int)d.batch; a.H = d.heads; a.Hkv = d.kv_heads; a.D = d.head_dim;
    a.causal = d.causal ? 1 : 0;
    a.mods = mods_of(p);
    return a;
}

template <typename F>
void by_dim(int D, F&& go) {
    if (D <= 32) go(std::integral_constant<int, 32>{});
    else if (D <= 64) go(std::integral_constant<int, 64>{});
    else go(std::integral_constant<int, 128>{});
}

}  // namespace

hipError_t launch_packed_f32_fwd(const mc_packed_attn_desc& p, const void* q, const void* k, const void* v,
                                 const int32_t* spans, const float* slopes, void* o, float* lse, hipStream_t stream) {
    PackedF32Args a = f32_args(p, q, k, v, spans, slopes);
    a.out = static_cast<float*>(o);
    a.lse = lse;
    const dim3 grid((unsigned)((int64_t)a.nblk * a.B * a.H));
    by_dim(a.D, [&](auto dp) { packed_f32_fwd<decltype(dp)::value><<<grid, 256, 0, stream>>>(a); });
    return hipGetLastError();
}

hipError_t launch_packed_f32_bwd(const mc_packed_attn_desc& p, const void* q, const void* k, const void* v,
                                 const int32_t* spans, const float* slopes, const void* o, const float* lse,
                                 const void* dout, void* dq, void* dk, void* dv, float* delta, float* dk_part,
                                 float* dv_part, hipStream_t stream) {
    PackedF32Args a = f32_args(p, q, k, v, spans, slopes);
    a.o = static_cast<const float*>(o);
    a.dout = static_cast<const float*>(dout);
    a.lse = const_cast<float*>(lse);
    a.delta = delta;
    a.groups = attention_f32_groups(p.attn);
    a.dq = static_cast<float*>(dq);
    a.dk = a.groups > 1 ? dk_part : static_cast<float*>(dk);
    a.dv = a.groups > 1 ? dv_part : static_cast<float*>(dv);
    const dim3 gq((unsigned)((int64_t)a.nblk * a.B * a.H));
    const dim3 gk((unsigned)((int64_t)a.nblk * a.B * a.Hkv * a.groups));
    by_dim(a.D, [&](auto dp) {
        constexpr int DP = decltype(dp)::value;
        packed_f32_dq<DP><<<gq, 256, 0, stream>>>(a);
        packed_f32_dkdv<DP><<<gk, 256, 0, stream>>>(a);
    });
    if (a.groups > 1) {
        const int64_t per4 = a.S * a.D / 4, n4 = per4 * a.B * a.Hkv;
        packed_f32_sum<<<dim3((unsigned)((2 * n4 + 255) / 256)), 256, 0, stream>>>(
            reinterpret_cast<const f32x4*>(dk_part), reinterpret_cast<const f32x4*>(dv_part),
            static_cast<f32x4*>(dk), static_cast<f32x4*>(dv), a.groups, per4, n4);
    }
    return hipGetLastError();
}

hipError_t launch_packed_rows_fwd(const mc_packed_attn_desc& p, const void* q, const void* k, const void* v,
                                  const int32_t* spans, const float* slopes, void* o, float* lse, hipStream_t stream) {
    const mc_attn_desc& d = p.attn;
    const dim3 grid((unsigned)((d.batch * d.heads * d.seq + 3) / 4));
    auto go = [&](auto elem) {
        typedef decltype(elem) T;
        Rows<T> a = row_args<T>(p, q, k, v, spans, slopes);
        a.o = static_cast<T*>(o);
        a.lse = lse;
        packed_rows_fwd<T><<<grid, 256, 0, stream>>>(a);
    };
    if (d.dtype == MC_F32) go(float{});
    else go(uint16_t{});
    return hipGetLastError();
}

hipError_t launch_packed_rows_bwd(const mc_packed_attn_desc& p, const void* q, const void* k, const void* v,
                                  const int32_t* spans, const float* slopes, const void* o, const float* lse,
                                  const void* dout, void* dq, void* dk, void* dv, float* delta, hipStream_t stream) {
    const mc_attn_desc& d = p.attn;
    const dim3 gq((unsigned)((d.batch * d.heads * d.seq + 3) / 4));
    const dim3 gk((unsigned)((d.batch * d.kv_heads * d.seq + 3) / 4));
    auto go = [&](auto elem) {
        typedef decltype(elem) T;
        Rows<T> a = row_args<T>(p, q, k, v, spans, slopes);
        a.o = static_cast<T*>(const_cast<void*>(o));
        a.dout = static_cast<const T*>(dout);
        a.lse = const_cast<float*>(lse);
        a.delta = delta;
        a.dq = static_cast<T*>(dq);
        a.dk = static_cast<T*>(dk);
        a.dv = static_cast<T*>(dv);
        packed_rows_dq<T><<<gq, 256, 0, stream>>>(a);
        packed_rows_dkdv<T><<<gk, 256, 0, stream>>>(a);
    };
    if (d.dtype == MC_F32) go(float{});
    else go(uint16_t{});
    return hipGetLastError();
}

}  // namespace mc
