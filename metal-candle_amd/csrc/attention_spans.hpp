// What a token of a packed row sees (attention_packed.hip, attention_packed_f32.hip).
#pragma once

#include "common.hpp"

namespace mc {
namespace attn {

// What a lane's token sees of the other side: [lo, hi), empty as [0, 0), inside
// [0, S) whatever the spans hold; from the causal rule without spans.
struct Span {
    int lo, hi;
};
__device__ __forceinline__ Span clamp_span(int lo, int hi, int S) {
    lo = lo < 0 ? 0 : lo;
    hi = hi > S ? S : hi;
    return lo < hi ? Span{lo, hi} : Span{0, 0};
}
__device__ __forceinline__ Span query_span(const int4* spans, int64_t row, int64_t t, int S, int causal) {
    if (t >= S) return Span{0, 0};
    if (!spans) return Span{0, causal ? (int)t + 1 : S};
    const int2 x = reinterpret_cast<const int2*>(spans + row * S + t)[0];
    return clamp_span(x.x, x.y, S);
}
__device__ __forceinline__ Span key_span(const int4* spans, int64_t row, int64_t t, int S, int causal) {
    if (t >= S) return Span{0, 0};
    if (!spans) return Span{causal ? (int)t : 0, S};
    const int2 x = reinterpret_cast<const int2*>(spans + row * S + t)[1];
    return clamp_span(x.x, x.y, S);
}

}  // namespace attn
}  // namespace mc
