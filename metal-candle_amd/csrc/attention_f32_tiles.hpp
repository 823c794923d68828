// Device helpers that the float32 attention kernels share (attention_f32.hip,
// attention_packed_f32.hip): 32-row LDS tiles and the products over them.
#pragma once

#include "common.hpp"

namespace mc {
namespace attn32 {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNegInf = -__builtin_inff();

// Orders a wave's LDS accesses for the compiler (the hardware keeps them in
// order): the tiles below are private to a wave.
__device__ __forceinline__ void wave_lds_fence() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

__device__ __forceinline__ float half_swap(float v) { return __shfl_xor(v, 32, kWave); }

// Row of accumulator register q.
__device__ __forceinline__ int acc_row(int q, int h) { return 8 * (q >> 2) + 4 * h + (q & 3); }

// A 32-row tile [32][DP] of fp32, DP = D rounded up to 32, 64 or 128. Rows in
// LDS are DP + 4 floats apart: 16 consecutive rows of one 16-byte column, and
// one row's consecutive columns, each fall on distinct banks.
template <int DP> struct Tile32 {
    static constexpr int LD = DP + 4, CPR = DP / 4, LOADS = DP / 8, DT = DP / 32;
    static constexpr int FLOATS = 32 * LD;
    typedef float vec __attribute__((ext_vector_type(DT)));

    // Resource over rows row0 .. of an operand whose rows are ld floats apart
    // (`rows` of them in all); rows past the end load as zeros.
    static __device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc(const float* base, int64_t row0, int64_t rows,
                                                                  int64_t ld, int D) {
        const int64_t left = rows - row0;
        return make_rsrc(base + row0 * ld, left > 0 ? ((left - 1) * ld + D) * 4 : 0);
    }
    // Whole row segments: lane l loads 16-byte chunk l % CPR of rows
    // l / CPR + i (64 / CPR); chunks past D load as zeros.
    static __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t r, uint32_t ld, int D, f32x4 (&t)[LOADS]) {
        const int lane = lane_id(), c = lane % CPR;
        uint32_t off = 4 * c < D ? ((uint32_t)(lane / CPR) * ld + 4u * c) * 4u : kOOB;
        asm volatile("" : "+v"(off));  // keeps the LOADS offsets out of registers across the caller's loop
#pragma unroll
        for (int i = 0; i < LOADS; ++i)
            t[i] = __builtin_bit_cast(f32x4, buf_load16(r, off + (uint32_t)i * (64u / CPR) * ld * 4u));
    }
    static __device__ __forceinline__ void store(float* lds, const f32x4 (&t)[LOADS]) {
        const int lane = lane_id(), c = lane % CPR;
#pragma unroll
        for (int i = 0; i < LOADS; ++i)
            *reinterpret_cast<f32x4*>(&lds[(lane / CPR + i * (64 / CPR)) * LD + 4 * c]) = t[i];
    }
    // Operand of a product over the head dim: lane's row l % 32, dims
    // 8 j + 4 h .. + 3 for step group j.
    static __device__ __forceinline__ f32x4 along_d(const float* lds, int j) {
        const int lane = lane_id();
        return *reinterpret_cast<const f32x4*>(&lds[(lane & 31) * LD + 8 * j + 4 * (lane >> 5)]);
    }
    // The same straight from memory (an operand held for the whole kernel).
    static __device__ __forceinline__ void load_along_d(__amdgpu_buffer_rsrc_t r, uint32_t ld, int D,
                                                        f32x4 (&t)[DP / 8]) {
        const int lane = lane_id();
#pragma unroll
        for (int j = 0; j < DP / 8; ++j) {
            const int d = 8 * j + 4 * (lane >> 5);
            t[j] = __builtin_bit_cast(f32x4, buf_load16(r, d < D ? ((uint32_t)(lane & 31) * ld + d) * 4u : kOOB));
        }
    }
    // Operand of step q of a product over the rows: row acc_row(q, h), the
    // DT dims of output row l % 32.
    static __device__ __forceinline__ vec along_rows(const float* lds, int q) {
        const int lane = lane_id();
        return *reinterpret_cast<const vec*>(&lds[acc_row(q, lane >> 5) * LD + DT * (lane & 31)]);
    }
    // acc^T (DT tiles, rows = dims, lane = row l % 32) -> lds rows
    static __device__ __forceinline__ void store_acc(float* lds, const f32x16 (&acc)[DT]) {
        const int lane = lane_id();
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            float v[4 * DT];
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int t = 0; t < DT; ++t) v[e * DT + t] = acc[t][4 * g + e];
            float* dst = &lds[(lane & 31) * LD + DT * (8 * g + 4 * (lane >> 5))];
#pragma unroll
            for (int e = 0; e < DT; ++e)
                *reinterpret_cast<f32x4*>(dst + 4 * e) = f32x4{v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]};
        }
    }
};

__device__ __forceinline__ f32x16 zero16() {
    f32x16 z;
#pragma unroll
    for (int q = 0; q < 16; ++q) z[q] = 0.f;
    return z;
}

// A.B over the head dim: A rows from an LDS tile, B from b(j) (held in
// registers, or read from a second tile). Each step's operand is read one step
// (256 cycles of MFMA) ahead; the scheduling barriers keep the compiler from
// hoisting more of them than the registers hold. Every 8 dims are summed on
// their own, added in pairs and the pairs to the total, so the rounding of a
// score is that of short chains (one chain over the whole head dim was up to
// 1.4 times further from the 64-bit result than the row kernels at short
// sequences).
template <int DP, typename Bf>
__device__ __forceinline__ f32x16 mma_d(const float* lds, Bf&& b) {
    constexpr int NJ = DP / 8;
    f32x16 acc, even;
    f32x4 x = Tile32<DP>::along_d(lds, 0), y = b(0);
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
        f32x4 nx = x, ny = y;
        if (j + 1 < NJ) {
            nx = Tile32<DP>::along_d(lds, j + 1);
            ny = b(j + 1);
        }
        f32x16 part = zero16();
#pragma unroll
        for (int p = 0; p < 4; ++p) part = __builtin_amdgcn_mfma_f32_32x32x2f32(x[p], y[p], part, 0, 0, 0);
        if (j % 2 == 0) {
            even = part;
        } else {
            acc = j == 1 ? even + part : acc + (even + part);
            asm volatile("" : "+v"(acc));  // adds it here, not after the last chain
        }
        x = nx;
        y = ny;
        __builtin_amdgcn_sched_barrier(0);
    }
    return acc;
}

// acc^T += X^T.P over the 32 rows of an LDS tile X, P from an accumulator
// (operands read four steps ahead).
template <int DP>
__device__ __forceinline__ void mma_rows(const float* lds, const f32x16& p, f32x16 (&acc)[DP / 32]) {
    typename Tile32<DP>::vec x[2][4];
#pragma unroll
    for (int e = 0; e < 4; ++e) x[0][e] = Tile32<DP>::along_rows(lds, e);
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        if (g < 3)
#pragma unroll
            for (int e = 0; e < 4; ++e) x[(g + 1) & 1][e] = Tile32<DP>::along_rows(lds, 4 * (g + 1) + e);
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int t = 0; t < DP / 32; ++t)
                acc[t] = __builtin_amdgcn_mfma_f32_32x32x2f32(x[g & 1][e][t], p[4 * g + e], acc[t], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
    }
}

__device__ __forceinline__ bool nonfinite(float v) { return !(__builtin_fabsf(v) <= 3.402823466e38f); }

template <int N>
__device__ __forceinline__ bool any_nonfinite(const f32x4 (&t)[N]) {
    bool bad = false;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) bad |= nonfinite(t[i][e]);
    return __any(bad);
}

// Head of workgroup j of a round of nbh: with the round a multiple of 8 long
// each XCD (workgroup id mod 8) takes a contiguous run of heads, so the heads
// that share a K/V head share an L2.
__device__ __forceinline__ int head_of(int j, int nbh) { return (nbh & 7) ? j : (j & 7) * (nbh >> 3) + (j >> 3); }

// Two waves per SIMD where the registers allow it (D <= 64); D = 128 holds
// twice the operands and accumulators and runs one.
template <int DP> constexpr int kWgPerCu = DP <= 64 ? 2 : 1;

}  // namespace attn32
}  // namespace mc
