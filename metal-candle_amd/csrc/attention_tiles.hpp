// Device helpers that the bf16 attention kernels share (attention.hip,
// attention_packed.hip): LDS tile layouts, transposed fragment reads, row stores.
#pragma once

#include "common.hpp"

namespace mc {
namespace attn {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kNegInf = -__builtin_inff();

// 64-bit integer min / max. (The device min / max templates instantiated at
// int64_t were lowered through double-precision min / max and conversions.)
__device__ __forceinline__ int64_t min64(int64_t x, int64_t y) { return x < y ? x : y; }
__device__ __forceinline__ int64_t max64(int64_t x, int64_t y) { return x > y ? x : y; }

// Instruction classes of __builtin_amdgcn_sched_group_barrier.
constexpr int kSchedMfma = 0x008, kSchedDsRead = 0x100;

// max(v of lane l, v of lane l ^ 32) without LDS. v_permlane32_swap swaps
// lanes 32-63 of its first register with lanes 0-31 of its second; with v in
// both, every lane then holds v of lanes l & 31 and (l & 31) + 32.
__device__ __forceinline__ float half_pair_max(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// Position of a workgroup among the B * H (batch, head) workgroups of its
// query-block round. Workgroups are dispatched round-robin over the 8 XCDs
// (id mod 8); when the round is a multiple of 8 long, each XCD takes a
// contiguous run of (b, h), so the heads that share a K / V head share that
// XCD's L2. The rounds, heaviest query blocks first, keep their order.
__device__ __forceinline__ int xcd_head_order(int j, int nbh) {
    return (nbh & 7) ? j : (j & 7) * (nbh >> 3) + (j >> 3);
}

// Growth of a row's score max (log2 units) that the forward absorbs before it
// moves its softmax reference point and rescales O.
constexpr float kMaxSlack = 8.f;

// Position p of a 16-key group of the transposed V holds key perm16(p): the
// positions 0-3, 4-7, 8-11, 12-15 hold keys 0-3, 8-11, 4-7, 12-15 (bits 2 and
// 3 swapped; the map is its own inverse). This is the order in which a lane
// half of the S^T accumulator holds its keys (rows 8 (j/4) + 4 (l/32) + j%4).
__device__ __forceinline__ int perm16(int p) { return (p & 3) | ((p & 4) << 1) | ((p & 8) >> 1); }

// Position of 16-byte chunk c of row r in the backward's [64][D] LDS tiles.
// Two read patterns must be bank-conflict free (64 banks x 4 B): row reads
// (16 consecutive rows of one chunk per 16 lanes) need the row's low bits to
// permute the chunk; the transposed reads (4 consecutive rows x 4
// consecutive chunks per 32 lanes) need the row's two lowest bits on the
// chunk's bits 2-3. Swapping the row's bit pairs 0-1 and 2-3 into the XOR
// mask serves both (D = 128: 16 chunks per 256-byte row; D = 64: 8 chunks,
// two rows per 256 bytes). The row-major swizzle of the forward (swz) put
// two (row, chunk) pairs of each transposed read on one bank group.
template <int D>
__device__ __forceinline__ int aswz(int r, int c) {
    static_assert(D == 64 || D == 128, "head dims with an MFMA backward");
    if constexpr (D == 128) return c ^ (((r & 3) << 2) | ((r >> 2) & 3));
    else return c ^ ((((r >> 1) & 1) << 2) | ((r >> 2) & 3));
}

// [ROWS][D] tile into the swizzled LDS layout from rows row0 .. row0+ROWS-1
// of a buffer with row stride ld (elements); rows past the buffer load zeros.
// Each of the 4 waves issues LOADS of the tile's 1 KB DMA pieces.
template <int D, int ROWS = 64>
__device__ __forceinline__ void dma_rows(i32x4 r, uint32_t lds_byte, uint32_t row0, uint32_t ld, int wave,
                                         int lane) {
    constexpr int CPR = D / 8, RPI = 64 / CPR, LOADS = ROWS / RPI / 4;
    static_assert(LOADS >= 1 && LOADS * RPI * 4 == ROWS, "whole 1 KB pieces per wave");
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
        const int blk = wave * LOADS + j;
        const int row = blk * RPI + lane / CPR;
        const uint32_t chunk = (uint32_t)aswz<D>(row, lane % CPR);
        const uint32_t off = ((row0 + (uint32_t)row) * ld + 8u * chunk) * 2u;
        dma16(r, __builtin_amdgcn_readfirstlane(lds_byte + (uint32_t)blk * 1024u), off);
    }
}

// ds_read_b64_tr_b16: within each 16-lane group, lane i receives element i % 4
// of the 8-byte pieces addressed by the group's lanes i / 4, 4 + i / 4,
// 8 + i / 4 and 12 + i / 4 (in that order).
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
__device__ __forceinline__ s16x4 ds_read_tr16(const uint16_t* p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p));
}

// MFMA 32x32x16 fragments from a swizzled [rows][D] tile, addressed by
// per-lane byte offsets computed once per kernel. Inside a tile the swizzle
// depends only on a row's low four bits, so the lane's offset is the same for
// every 32-row (row fragments) or 16-row (transposed fragments) step of the
// tile, and the step enters as a constant that folds into the LDS
// instruction's offset field; the kernels hold a handful of offsets rather
// than one address per fragment read.
//
// Row fragment (the A or B operand from rows of the tile): lane l reads row
// 32 k + l % 32, 16-byte chunk c.
template <int D>
__device__ __forceinline__ uint32_t rows_off(int lane, int c) {
    const int col = lane & 31;
    return (uint32_t)((col * D + 8 * aswz<D>(col, c)) * 2);
}
// Transposed fragment (operand of M^T for a row-major tile M): lane l gets
// column dcol + l % 32 of M and the 8 rows 16 k + 4 (l / 32) +
// {0, 1, 2, 3, 8, 9, 10, 11}, the order in which a lane half of an S (or S^T)
// accumulator holds its rows (8 (j/4) + 4 half + j%4). Two transposed reads
// of 4 rows each (h = 0, 1): lane i of 16-lane group g addresses row
// 16 k + 4 (g / 2) + i / 4 + 8 h, columns dcol + 16 (g % 2) + 4 (i % 4) .. +3.
template <int D>
__device__ __forceinline__ uint32_t tr_off(int lane, int dcol, int h) {
    const int i = lane & 15, g = lane >> 4;
    const int r = 4 * (g >> 1) + (i >> 2) + 8 * h;
    const int c = (dcol >> 3) + 2 * (g & 1) + ((i & 3) >> 1);
    return (uint32_t)((r * D + 8 * aswz<D>(r, c) + 4 * (i & 1)) * 2);
}
__device__ __forceinline__ bf16x8 frag_at(const uint16_t* t, uint32_t byte_off) {
    return *reinterpret_cast<const bf16x8*>(reinterpret_cast<const char*>(t) + byte_off);
}
__device__ __forceinline__ bf16x8 frag_tr_at(const uint16_t* t, uint32_t off_lo, uint32_t off_hi) {
    const char* b = reinterpret_cast<const char*>(t);
    const s16x4 v8[2] = {ds_read_tr16(reinterpret_cast<const uint16_t*>(b + off_lo)),
                         ds_read_tr16(reinterpret_cast<const uint16_t*>(b + off_hi))};
    return __builtin_bit_cast(bf16x8, v8);
}

// Rows of a wave's transposed accumulators (acc[dt] element j = dim
// 32 dt + 8 (j/4) + 4 half + j%4 of row `col`) through a per-wave LDS patch
// to 16-byte stores of rows row0 + r (r < 32, row0 + r < nrows) of dst
// (row stride ld elements). OutT: uint16_t (bf16) or float.
template <int D, typename OutT>
__device__ __forceinline__ void store_rows(const f32x16 (&acc)[D / 32], float scale, void* patch_mem, OutT* dst,
                                           int64_t ld, int64_t row0, int64_t nrows, int lane) {
    constexpr int EPC = 16 / sizeof(OutT);    // elements per 16-byte chunk
    constexpr int PROW = D + 16 / sizeof(OutT);  // padded patch row (elements)
    constexpr int CPR = D / EPC;
    OutT* patch = static_cast<OutT*>(patch_mem);
    const int col = lane & 31, half = lane >> 5;
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
        for (int jq = 0; jq < 4; ++jq) {
            const int d = 32 * dt + 8 * jq + 4 * half;
            if constexpr (sizeof(OutT) == 2) {
                const uint32_t lo = pack_bf16x2(acc[dt][4 * jq] * scale, acc[dt][4 * jq + 1] * scale);
                const uint32_t hi = pack_bf16x2(acc[dt][4 * jq + 2] * scale, acc[dt][4 * jq + 3] * scale);
                *reinterpret_cast<uint2*>(&patch[col * PROW + d]) = make_uint2(lo, hi);
            } else {
                *reinterpret_cast<float4*>(&patch[col * PROW + d]) =
                    make_float4(acc[dt][4 * jq] * scale, acc[dt][4 * jq + 1] * scale, acc[dt][4 * jq + 2] * scale,
                                acc[dt][4 * jq + 3] * scale);
            }
        }
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): the wave's patch is written
#pragma unroll
    for (int it = 0; it < 32 * CPR / 64; ++it) {
        const int i = it * 64 + lane;
        const int r = i / CPR, c = i % CPR;
        if (row0 + r < nrows) {
            const uint4 v = *reinterpret_cast<const uint4*>(&patch[r * PROW + EPC * c]);
            *reinterpret_cast<uint4*>(dst + (row0 + r) * ld + EPC * c) = v;
        }
    }
    __builtin_amdgcn_s_waitcnt(0xc07f);  // patch reads done before it is rewritten
}

// dk / dv [B, Hkv, S, D] = sum over the rep query-head groups of each K/V
// head of the fp32 partials, in group order; 8 elements per thread.
__device__ __forceinline__ void bwd_sum_range(const float* __restrict__ dk_part, const float* __restrict__ dv_part,
                                              uint16_t* __restrict__ dk, uint16_t* __restrict__ dv, int rep,
                                              int64_t per_head, int64_t n8, int64_t first, int64_t stride) {
    for (int64_t i = first; i < 2 * n8; i += stride) {
        const bool second = i >= n8;
        const int64_t e = (second ? i - n8 : i) * 8;  // element of [B, Hkv, S, D]
        const int64_t bhk = e / per_head, off = e % per_head;
        const float* src = (second ? dv_part : dk_part) + bhk * rep * per_head + off;
        float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        for (int r = 0; r < rep; ++r) {
            const float4 x0 = *reinterpret_cast<const float4*>(src + r * per_head);
            const float4 x1 = *reinterpret_cast<const float4*>(src + r * per_head + 4);
            acc[0] += x0.x; acc[1] += x0.y; acc[2] += x0.z; acc[3] += x0.w;
            acc[4] += x1.x; acc[5] += x1.y; acc[6] += x1.z; acc[7] += x1.w;
        }
        uint16_t* dst = (second ? dv : dk) + e;
        *reinterpret_cast<uint4*>(dst) = make_uint4(pack_bf16x2(acc[0], acc[1]), pack_bf16x2(acc[2], acc[3]),
                                                    pack_bf16x2(acc[4], acc[5]), pack_bf16x2(acc[6], acc[7]));
    }
}
}  // namespace attn
}  // namespace mc
