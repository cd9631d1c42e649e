// Rotary positions on part of each head (include/dsa_mi355x_cache.h:
// dsa_rotary).  No reference counterpart: the reference takes rotated q_rope
// and k_rope (README.md:19-21).
//
//   y0 = x0 cos - x1 sin,  y1 = x0 sin + x1 cos   for each pair of the rotated part
//
// Bound by HBM (each element read and written once) and, for a decode step, by
// the launch.  A head is cut into units: of the rotated part 16 bytes that hold
// whole pairs (interleaved) or two times 16 bytes, dim / 2 apart; of the rest 16
// bytes; where sizes, strides or alignment forbid it a pair, or an element.  A
// workgroup owns 256 units, of some tokens or of a part of one token's heads, one
// a thread: it loads them, then forms its tokens' cosines and sines once in LDS,
// for all heads, while the loads are on their way.  (Four units a thread were
// slower throughout: 8 tokens x 128 heads x 64 of 192 bf16 4.1 us for 3.0, 4096
// tokens 35.2 for 32.7 in a graph of them, 4.1 TB/s; 4096 x 64 heads x 64 of 128
// fp32 in the half layout 59.4 for 51.5, 5.2 TB/s.)
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/dsa_mi355x_cache.h"
#include "kernels.h"
#include "rotary_math.h"

namespace dsa {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxAngles = 1024;  // cosines and sines a workgroup forms: four a thread at most, 8 KiB of LDS
static_assert(DSA_ROTARY_MAX_DIM / 2 <= kMaxAngles, "a token's fit");

// n / d, by a multiplication where magic = ceil(2^32 / d) gives it exactly (0: a division).
__device__ __forceinline__ uint32_t quotient(uint32_t n, uint32_t d, uint32_t magic) {
    return magic ? __umulhi(n, magic) : n / d;
}
uint32_t magic_of(uint32_t d, uint64_t most) {  // for n <= most
    return d > 1 && most * d < (uint64_t)1 << 32 ? (uint32_t)((((uint64_t)1 << 32) + d - 1) / d) : 0;
}

struct Shape {
    int units, turning;      // a head's, the first of them of the rotated part
    int tokens;              // of a workgroup
    int chunks;              // workgroups of one token's units (tokens > 1: one)
    uint32_t per_token;      // units of a token
    uint32_t units_magic, token_magic;
    int64_t group0;          // first group of tokens (of `chunks` workgroups) of this launch
};
// Workgroups of a launch: the grid's threads are counted in 32 bits.
constexpr int64_t kMaxGrid = (int64_t)1 << 23;

// W elements at a time: 16 bytes, or as few as a unit can have, which need no alignment.
template <typename T, int W>
struct Vec {
    static constexpr bool kWide = W * sizeof(T) == 16;
    T v[W];
    __device__ __forceinline__ void load(const T* from) {
        if constexpr (kWide) {
            *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(from);
        } else {
#pragma unroll
            for (int i = 0; i < W; ++i) v[i] = from[i];
        }
    }
    __device__ __forceinline__ void store(T* to) const {
        if constexpr (kWide) {
            *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(v);
        } else {
#pragma unroll
            for (int i = 0; i < W; ++i) to[i] = v[i];
        }
    }
};

// WIDE: units of 16 bytes.
template <typename T, bool INTERLEAVED, bool WIDE>
__global__ __launch_bounds__(kThreads) void rotary_kernel(dsa_rotary_args p, Shape s) {
    constexpr int W = WIDE ? 16 / (int)sizeof(T) : INTERLEAVED ? 2 : 1;  // elements of a vector
    constexpr int PAIRS = INTERLEAVED ? W / 2 : W;                       // pairs of a turning unit
    constexpr int COPY = WIDE ? W : 1;                                   // elements of another unit
    __shared__ float2 angles[kMaxAngles];
    const int tid = threadIdx.x, pairs = p.dim >> 1;
    const int64_t all = p.groups * p.tokens;
    const uint32_t group = blockIdx.x / (uint32_t)s.chunks;
    const uint32_t chunk = blockIdx.x - group * s.chunks;
    const int64_t token0 = (s.group0 + group) * s.tokens;
    const int tokens = (int)min((int64_t)s.tokens, all - token0);

    const uint32_t n = chunk * kThreads + tid;
    const bool there = n < s.per_token * (uint32_t)tokens;
    bool turns = false;
    int first = 0;  // its first angle
    int64_t to = 0;
    Vec<T, W> a, b;
    if (there) {
        const uint32_t t = s.tokens == 1 ? 0 : quotient(n, s.per_token, s.token_magic);
        const uint32_t in_token = n - t * s.per_token;
        const uint32_t h = s.units == 1 ? in_token : quotient(in_token, s.units, s.units_magic);
        const int u = (int)(in_token - h * s.units);
        int64_t in_group = token0 + t, outer = 0;
        if (p.groups > 1) {
            outer = in_group / p.tokens;
            in_group -= outer * p.tokens;
        }
        turns = u < s.turning;
        first = (int)t * pairs + u * PAIRS;
        int e = p.start + u * W;
        if (!turns) {
            e = (u - s.turning) * COPY;
            e += e >= p.start ? p.dim : 0;
        }
        to = outer * p.out_stride[0] + in_group * p.out_stride[1] + h * p.out_stride[2] + e;
        const T* from = static_cast<const T*>(p.x) + outer * p.x_stride[0] + in_group * p.x_stride[1] + h * p.x_stride[2] + e;
        if (WIDE || turns) {
            a.load(from);
            if (!INTERLEAVED && turns) b.load(from + pairs);
        } else {
            a.v[0] = from[0];
        }
    }

    const float sign = p.transposed ? -1.f : 1.f;
    for (int k = tid; k < tokens * pairs; k += kThreads) {
        const int t = s.tokens == 1 ? 0 : k / pairs, i = k - t * pairs;
        angles[k] = rotary_turn(rotary_position(p.positions, token0 + t, p.positions_64), p.frequencies[i], p.magnitude,
                                sign);
    }
    __syncthreads();

    if (!there) return;
    T* out = static_cast<T*>(p.out) + to;
    if (!turns) {
        if constexpr (WIDE) a.store(out);
        else out[0] = a.v[0];
        return;
    }
    const float2* cs = angles + first;
    Vec<T, W> y;
    if constexpr (INTERLEAVED) {
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) {
            float y0, y1;
            rotary_pair((float)a.v[2 * i], (float)a.v[2 * i + 1], cs[i], y0, y1);
            y.v[2 * i] = (T)y0;
            y.v[2 * i + 1] = (T)y1;
        }
        y.store(out);
    } else {
        Vec<T, W> z;
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) {
            float y0, y1;
            rotary_pair((float)a.v[i], (float)b.v[i], cs[i], y0, y1);
            y.v[i] = (T)y0;
            z.v[i] = (T)y1;
        }
        y.store(out);
        z.store(out + pairs);
    }
}

bool multiples(const int64_t* strides, int of) {
    return strides[0] % of == 0 && strides[1] % of == 0 && strides[2] % of == 0;
}

template <typename T, bool INTERLEAVED>
int launch(const dsa_rotary_args& p, hipStream_t stream) {
    const int wide = 16 / (int)sizeof(T), pairs = p.dim / 2;
    const bool in_place = p.out == p.x;
    // every vector whole, and none across the border of the rotated part
    const bool is_wide = pairs % (INTERLEAVED ? wide / 2 : wide) == 0 && p.start % wide == 0 &&
                         (in_place || p.width % wide == 0) && multiples(p.x_stride, wide) && multiples(p.out_stride, wide) &&
                         (((uintptr_t)p.x | (uintptr_t)p.out) & 15) == 0;
    Shape s;
    s.turning = !is_wide ? pairs : INTERLEAVED ? p.dim / wide : pairs / wide;
    s.units = s.turning + (in_place ? 0 : (p.width - p.dim) / (is_wide ? wide : 1));
    s.per_token = (uint32_t)p.heads * (uint32_t)s.units;
    const int64_t all = p.groups * p.tokens;
    const int64_t fit = s.per_token < kThreads ? kThreads / s.per_token : 1, angles = kMaxAngles / pairs;
    s.tokens = (int)(fit < angles ? fit : angles);
    s.chunks = (int)(((int64_t)s.per_token * s.tokens + kThreads - 1) / kThreads);
    s.token_magic = magic_of(s.per_token, kThreads);
    s.units_magic = magic_of((uint32_t)s.units, s.per_token);
    auto* kernel = is_wide ? rotary_kernel<T, INTERLEAVED, true> : rotary_kernel<T, INTERLEAVED, false>;
    // heads * width <= 2^31, so a token has at most 2^23 chunks
    const int64_t groups = (all + s.tokens - 1) / s.tokens, most = kMaxGrid / s.chunks;
    for (s.group0 = 0; s.group0 < groups; s.group0 += most) {
        const int64_t n = groups - s.group0 < most ? groups - s.group0 : most;
        hipLaunchKernelGGL(kernel, dim3((unsigned)(n * s.chunks)), dim3(kThreads), 0, stream, p, s);
        if (const int rc = (int)hipGetLastError()) return rc;
    }
    return 0;
}

template <typename T>
int launch(const dsa_rotary_args& p, hipStream_t stream) {
    return p.interleaved ? launch<T, true>(p, stream) : launch<T, false>(p, stream);
}

}  // namespace

int launch_rotary(const dsa_rotary_args& args, hipStream_t stream) {
    dsa_rotary_args p = args;
    const int64_t sizes[3] = {p.groups, p.tokens, p.heads};
    for (int i = 0; i < 3; ++i)  // strides nothing steps by say nothing of the alignment
        if (sizes[i] == 1) p.x_stride[i] = p.out_stride[i] = 0;
    if (p.dtype == DSA_BF16) return launch<__bf16>(p, stream);
    if (p.dtype == DSA_F16) return launch<_Float16>(p, stream);
    return launch<float>(p, stream);
}

}  // namespace dsa
