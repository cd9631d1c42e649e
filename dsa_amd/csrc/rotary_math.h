// The rotation of one pair, shared by the rotary kernels (rotary.hip) and the
// cache row writer (kv_rows.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace dsa {

// Cosine and sine of position * frequency (radians), times magnitude.  The
// angle reaches 10^6 radians in a long context, where 32 bits hold it to 0.06:
// it is formed in 64 bits in turns, of which only the fraction, at most half a
// turn, is rounded to 32 (2^-25 of a turn at most).
__device__ __forceinline__ float2 rotary_turn(int64_t position, double frequency, float magnitude, float sign) {
    double turns = (double)position * frequency * 0.15915494309189533577;
    turns -= rint(turns);
    float s, c;
    sincospif(2.f * (float)turns, &s, &c);
    return float2{c * magnitude, s * magnitude * sign};
}

__device__ __forceinline__ void rotary_pair(float x0, float x1, float2 cs, float& y0, float& y1) {
    y0 = __builtin_fmaf(x0, cs.x, -(x1 * cs.y));
    y1 = __builtin_fmaf(x0, cs.y, x1 * cs.x);
}

__device__ __forceinline__ int64_t rotary_position(const void* positions, int64_t token, int wide) {
    return wide ? static_cast<const int64_t*>(positions)[token] : static_cast<const int32_t*>(positions)[token];
}

}  // namespace dsa
