// Rotary positions on part of each head (include/dsa_mi355x_cache.h:
// dsa_rotary).  No reference counterpart: the reference takes rotated q_rope
// and k_rope (README.md:19-21).
//
//   y0 = x0 cos - x1 sin,  y1 = x0 sin + x1 cos   for each pair of the rotated part
//
// Bound by HBM (each element read and written once) and, for a decode step, by
// the launch.  A workgroup owns kUnits units of some tokens' heads, a unit two
// 16-byte vectors that hold whole pairs.
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/dsa_mi355x_cache.h"
#include "kernels.h"
#include "rotary_math.h"

namespace dsa {
namespace {

constexpr int kThreads = 256;

template <typename T>
__global__ __launch_bounds__(kThreads) void rotary_simple_kernel(dsa_rotary_args p) {
    const int pairs = p.dim >> 1, rest = p.out == p.x ? 0 : p.width - p.dim, per = pairs + rest;
    const int64_t total = p.groups * p.tokens * p.heads * per;
    const T* x = static_cast<const T*>(p.x);
    T* out = static_cast<T*>(p.out);
    const float sign = p.transposed ? -1.f : 1.f;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < total; i += (int64_t)gridDim.x * kThreads) {
        const int e = (int)(i % per);
        const int64_t row = i / per, tok = row / p.heads;
        const int h = (int)(row % p.heads);
        const int64_t a = tok / p.tokens, t = tok % p.tokens;
        const T* xr = x + a * p.x_stride[0] + t * p.x_stride[1] + h * p.x_stride[2];
        T* yr = out + a * p.out_stride[0] + t * p.out_stride[1] + h * p.out_stride[2];
        if (e >= pairs) {
            int c = e - pairs;
            c += c >= p.start ? p.dim : 0;
            yr[c] = xr[c];
            continue;
        }
        const float2 cs = rotary_turn(rotary_position(p.positions, tok, p.positions_64), p.frequencies[e], p.magnitude,
                                      sign);
        const int e0 = p.start + (p.interleaved ? 2 * e : e), e1 = p.start + (p.interleaved ? 2 * e + 1 : e + pairs);
        float y0, y1;
        rotary_pair((float)xr[e0], (float)xr[e1], cs, y0, y1);
        yr[e0] = (T)y0;
        yr[e1] = (T)y1;
    }
}

template <typename T>
int launch(const dsa_rotary_args& p, hipStream_t stream) {
    const int64_t work = p.groups * p.tokens * p.heads * (p.dim / 2 + (p.out == p.x ? 0 : p.width - p.dim));
    const int64_t want = (work + kThreads - 1) / kThreads;
    hipLaunchKernelGGL(rotary_simple_kernel<T>, dim3((unsigned)(want < 16384 ? want : 16384)), dim3(kThreads), 0, stream,
                       p);
    return (int)hipGetLastError();
}

}  // namespace

int launch_rotary(const dsa_rotary_args& p, hipStream_t stream) {
    if (p.dtype == DSA_BF16) return launch<__bf16>(p, stream);
    if (p.dtype == DSA_F16) return launch<_Float16>(p, stream);
    return launch<float>(p, stream);
}

}  // namespace dsa
