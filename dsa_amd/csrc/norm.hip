// Root-mean-square norms of a residual stream, and 8-bit codes
// (include/dsa_mi355x_layer.h).  No reference counterpart: the reference takes q
// and kv as given (README.md:19-21).
//
// A row is held in registers by a team of one to sixteen waves, eight values a thread
// (sixteen above 8192), so that it is read once: the sum of squares needs all of it
// before the first output.  Bound by HBM (4095 rows of 4096 with a residual 25.8 to 26.9
// us, 5.0 to 5.2 TB/s; their gradients 25.0, and 3.9 for the weight's; codes of 4095 rows
// of 16384 34.3 us, 5.9 TB/s, of 4096 of 7168 with a norm and a residual 43.6 us, 4.7),
// and in a decode step by the launch and a trip to memory (8 rows of 7168 3.8 us, 192 with
// codes 4.8).
#include <hip/hip_runtime.h>
#include <hip/hip_fp16.h>
#include <stdint.h>

#include "kernels.h"
#include "mla_tiles.h"

namespace dsa {
namespace {

constexpr int kBlock = 128;  // values that share a scale: 16 lanes of eight

typedef _Float16 f16;

template <typename T>
struct Eight {
    uint4 v;
    __device__ __forceinline__ void load(const T* p) { v = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ float at(int i) const {
        const uint32_t w = i < 4 ? (i < 2 ? v.x : v.y) : (i < 6 ? v.z : v.w);
        const uint16_t half = (uint16_t)(i & 1 ? w >> 16 : w);
        return (float)__builtin_bit_cast(T, half);
    }
};
template <>
struct Eight<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const float* p) {
        a = reinterpret_cast<const float4*>(p)[0];
        b = reinterpret_cast<const float4*>(p)[1];
    }
    __device__ __forceinline__ float at(int i) const {
        const float4& v = i < 4 ? a : b;
        return (i & 3) == 0 ? v.x : (i & 3) == 1 ? v.y : (i & 3) == 2 ? v.z : v.w;
    }
};

// Values [e, e + 8) of a row as they lie in memory, zeros behind its end: half the
// registers of their 32-bit values, for what is loaded ahead.
template <typename T>
struct Ahead {
    Eight<T> v;
    __device__ __forceinline__ void load(const T* row, int e, int dim, bool vector) {
        if (vector) {
            if (e < dim) v.load(row + e);
            else v = Eight<T>{};
        } else {
            T t[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) t[i] = e + i < dim ? row[e + i] : (T)0.f;
            __builtin_memcpy(&v, t, sizeof t);
        }
    }
    __device__ __forceinline__ float at(int i) const { return v.at(i); }
};

// Values [e, e + 8) of a row of dim, zeros behind its end.  `vector`: the row is
// 16-byte aligned and dim a multiple of eight.
template <typename T>
__device__ __forceinline__ void load8(float (&f)[8], const T* row, int e, int dim, bool vector) {
    if (vector) {
        if (e < dim) {
            Eight<T> v;
            v.load(row + e);
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = v.at(i);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = 0.f;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = e + i < dim ? (float)row[e + i] : 0.f;
    }
}

template <typename T>
__device__ __forceinline__ void store8(T* row, const float (&f)[8], int e, int dim, bool vector) {
    T t[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = (T)f[i];
    if (vector) {
        if (e < dim) {
            typedef T vec __attribute__((ext_vector_type(16 / sizeof(T))));
            constexpr int N = 16 / sizeof(T);
#pragma unroll
            for (int k = 0; k < 8 / N; ++k) {
                vec v;
#pragma unroll
                for (int i = 0; i < N; ++i) v[i] = t[N * k + i];
                reinterpret_cast<vec*>(row + e)[k] = v;
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (e + i < dim) row[e + i] = t[i];
    }
}

// Over the 16 lanes of a DPP row by rotations, then over the four rows by lane swaps:
// no trip through LDS.
template <int CONTROL>
__device__ __forceinline__ float rotated(float v) {
    return __uint_as_float((uint32_t)__builtin_amdgcn_mov_dpp((int)__float_as_uint(v), CONTROL, 0xf, 0xf, true));
}
__device__ __forceinline__ float wave_sum(float v) {
    v += rotated<0x128>(v);  // row_ror:8
    v += rotated<0x124>(v);
    v += rotated<0x122>(v);
    v += rotated<0x121>(v);
    return sum_xor32(sum_xor16(v));
}

// Sum over a team; `turn` alternates, so that one barrier a sum is enough.
template <int WAVES>
__device__ __forceinline__ float team_sum(float v, float (*parts)[WAVES], int turn) {
    v = wave_sum(v);
    if constexpr (WAVES > 1) {
        if ((threadIdx.x & 63) == 0) parts[turn & 1][threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0.f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) v += parts[turn & 1][w];
    }
    return v;
}

// max over the 16 lanes of this lane's DPP row.
__device__ __forceinline__ uint32_t row16_max(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x128, 0xf, 0xf, true));  // row_ror:8
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x124, 0xf, 0xf, true));
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x122, 0xf, 0xf, true));
    return max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x121, 0xf, 0xf, true));
}

// Max over a team of values that are not negative; a NaN's bits exceed infinity's.
template <int WAVES>
__device__ __forceinline__ float team_max(float v, float (*parts)[WAVES], int turn) {
    uint32_t m = row16_max(__float_as_uint(v));
    m = max(m, (uint32_t)__shfl_xor((int)m, 16));
    m = max(m, (uint32_t)__shfl_xor((int)m, 32));
    if constexpr (WAVES > 1) {
        if ((threadIdx.x & 63) == 0) parts[turn & 1][threadIdx.x >> 6] = __uint_as_float(m);
        __syncthreads();
#pragma unroll
        for (int w = 0; w < WAVES; ++w) m = max(m, __float_as_uint(parts[turn & 1][w]));
    }
    return __uint_as_float(m);
}

// A row whose mean square and eps leave 32 bits' range, or come so near to its end that
// squares lose bits, times a power of two: its largest value, or eps's root, is then 1/2
// to 1.  `mean` becomes what its root is to be taken of; returns the power, and 0 for
// a row that no power helps: of zeros, or with an infinity or a NaN.  From 2^-96 on the
// squares that underflow, 2^-150 each, are 2^-40 of the mean at most.
constexpr float kLeastMean = 0x1p-96f;
template <int WAVES, int CH>
__device__ __forceinline__ int scale_row(float (&h)[CH][8], float& mean, float eps, int dim, float (*parts)[WAVES], int& turn) {
    float top = 0.f;
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) top = __uint_as_float(max(__float_as_uint(top), __float_as_uint(h[c][i]) & 0x7fffffffu));
    top = team_max<WAVES>(top, parts, ++turn);
    if (!(top > 0.f && top < INFINITY)) return 0;
    int power = __builtin_amdgcn_frexp_expf(top);
    if (eps > 0.f) power = max(power, (__builtin_amdgcn_frexp_expf(eps) + 1) >> 1);
    float squares = 0.f;
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            h[c][i] = ldexpf(h[c][i], -power);
            squares = fmaf(h[c][i], h[c][i], squares);
        }
    mean = team_sum<WAVES>(squares, parts, ++turn) / (float)dim + ldexpf(eps, -2 * power);
    return power;
}

// e4m3 code of v clamped to +-448, NaN kept (0x7f with v's sign).
__device__ __forceinline__ uint32_t code_special(float v) {
    if (v != v) return 0x7fu | (__float_as_uint(v) >> 31 << 7);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(fminf(fmaxf(v, -448.f), 448.f), 0.f, 0, false) & 0xffu;
}

// Codes of this lane's eight values and the scale that its 16 lanes share.  The
// quotient by 448 is a product with its rounded reciprocal (1.2e-7 of the scale); by
// the scale, an exponent shift where that is a power of two, and else a product with
// its reciprocal: 2^-23 of a value, so that only one so near to the middle of two
// codes takes the other.  Either stays below 464, and e4m3 rounds that to 448.
__device__ __forceinline__ uint2 encode8(const float (&f)[8], bool pow2, float& scale) {
    uint32_t m = 0;  // |f| as bits: a NaN's exceed infinity's
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(f[i]) & 0x7fffffffu);
    m = row16_max(m);
    const float top = __uint_as_float(m);  // of a block with a NaN a NaN: scale 1, as in an fp8 cache row
    scale = top > 0.f ? top * (1.f / 448.f) : 1.f;
    if (!(scale > 0.f)) scale = __uint_as_float(1);  // the product of the least numbers underflows
    float x[8];
    if (pow2) {
        const int k = __builtin_amdgcn_frexp_expf(scale) - (__builtin_amdgcn_frexp_mantf(scale) == 0.5f ? 1 : 0);
        if (m < 0x7f800000u) scale = ldexpf(1.f, k);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = ldexpf(f[i], -k);
    } else if (scale >= 0x1p-126f) {
        const float by = 1.f / scale;
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = f[i] * by;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = f[i] / scale;
    }
    uint2 c;
    if (__builtin_expect(m >= 0x7f800000u || scale < 0x1p-126f, 0)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = f[i] / scale;
        c.x = code_special(x[0]) | code_special(x[1]) << 8 | code_special(x[2]) << 16 | code_special(x[3]) << 24;
        c.y = code_special(x[4]) | code_special(x[5]) << 8 | code_special(x[6]) << 16 | code_special(x[7]) << 24;
    } else {
        c.x = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(
            x[2], x[3], __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false), true);
        c.y = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(
            x[6], x[7], __builtin_amdgcn_cvt_pk_fp8_f32(x[4], x[5], 0, false), true);
    }
    return c;
}

__device__ __forceinline__ void load_weight(float (&f)[8], const void* weight, int e, int dim, bool f32, bool vector,
                                            const __bf16*) {
    if (f32) load8(f, static_cast<const float*>(weight), e, dim, vector);
    else load8(f, static_cast<const __bf16*>(weight), e, dim, vector);
}
__device__ __forceinline__ void load_weight(float (&f)[8], const void* weight, int e, int dim, bool f32, bool vector,
                                            const f16*) {
    if (f32) load8(f, static_cast<const float*>(weight), e, dim, vector);
    else load8(f, static_cast<const f16*>(weight), e, dim, vector);
}
__device__ __forceinline__ void load_weight(float (&f)[8], const void* weight, int e, int dim, bool, bool vector,
                                            const float*) {
    load8(f, static_cast<const float*>(weight), e, dim, vector);
}

template <typename T, bool CODES, int WAVES, int CH>
__global__ __launch_bounds__(WAVES == 1 ? 256 : WAVES * 64) void norm_kernel(dsa_norm_args p, int vector_) {
    constexpr int TEAM = WAVES * 64, TEAMS = WAVES == 1 ? 4 : 1;
    __shared__ float parts[2][WAVES];
    const bool vector = vector_;
    const int tid = WAVES == 1 ? threadIdx.x & 63 : threadIdx.x;
    const int team = WAVES == 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
    const int dim = p.dim, blocks = (dim + kBlock - 1) / kBlock;
    const bool normed = !CODES || p.weight != nullptr;
    float w[CH][8];
    if (normed) {
#pragma unroll
        for (int c = 0; c < CH; ++c)
            load_weight(w[c], p.weight, (c * TEAM + tid) * 8, dim, p.weight_f32, vector, (const T*)nullptr);
    }
    int turn = 0;
    for (int64_t r = (int64_t)blockIdx.x * TEAMS + team; r < p.rows; r += (int64_t)gridDim.x * TEAMS, ++turn) {
        const T* x = static_cast<const T*>(p.x) + r * p.x_stride;
        float h[CH][8];
#pragma unroll
        for (int c = 0; c < CH; ++c) load8(h[c], x, (c * TEAM + tid) * 8, dim, vector);
        if (p.residual) {
            const T* residual = static_cast<const T*>(p.residual) + r * p.residual_stride;
            T* sum = static_cast<T*>(p.sum) + r * dim;
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                float add[8];
                load8(add, residual, (c * TEAM + tid) * 8, dim, vector);
                // rounded here, as the stream is kept: its norm, its gradients and a
                // model that adds first all see the same values
#pragma unroll
                for (int i = 0; i < 8; ++i) h[c][i] = (float)(T)(h[c][i] + add[i]);
            }
#pragma unroll
            for (int c = 0; c < CH; ++c) store8(sum, h[c], (c * TEAM + tid) * 8, dim, vector);
        }
        if (normed) {
            float squares = 0.f;
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int i = 0; i < 8; ++i) squares = fmaf(h[c][i], h[c][i], squares);
            squares = team_sum<WAVES>(squares, parts, turn);
            float mean = squares / (float)dim + p.eps;
            int power = 0;
            if (__builtin_expect(!(mean >= kLeastMean && mean < INFINITY), 0))  // the same in all of the team
                power = scale_row<WAVES, CH>(h, mean, p.eps, dim, parts, turn);
            const float inverse = 1.f / sqrtf(mean);
            if (!CODES && p.inverse && tid == 0) p.inverse[r] = ldexpf(inverse, -power);
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int i = 0; i < 8; ++i) h[c][i] = h[c][i] * inverse * w[c][i];
        }
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int e = (c * TEAM + tid) * 8;
            if constexpr (CODES) {
                float scale;
                const uint2 code = encode8(h[c], p.pow2_scales, scale);
                if (e < dim) {
                    *reinterpret_cast<uint2*>(static_cast<uint8_t*>(p.out) + r * dim + e) = code;
                    if ((tid & 15) == 0) p.scales[r * blocks + e / kBlock] = scale;
                }
            } else {
                store8(static_cast<T*>(p.out) + r * dim, h[c], e, dim, vector);
            }
        }
    }
}

// Gradients: a team goes over rows team, team + teams, .. and keeps its columns'
// sums of the weight's gradient in registers; they are added up, in a fixed order,
// by norm_weight_kernel.
template <typename T, int WAVES, int CH>
__global__ __launch_bounds__(WAVES == 1 ? 256 : WAVES * 64) void norm_grad_kernel(dsa_norm_grad_args p, int vector_) {
    constexpr int TEAM = WAVES * 64, TEAMS = WAVES == 1 ? 4 : 1;
    __shared__ float parts[2][WAVES];
    const bool vector = vector_;
    const int tid = WAVES == 1 ? threadIdx.x & 63 : threadIdx.x;
    const int64_t team = (int64_t)blockIdx.x * TEAMS + (WAVES == 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0);
    const int64_t teams = (int64_t)gridDim.x * TEAMS;
    const int dim = p.dim;
    float w[CH][8], sums[CH][8];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        load_weight(w[c], p.weight, (c * TEAM + tid) * 8, dim, p.weight_f32, vector, (const T*)nullptr);
#pragma unroll
        for (int i = 0; i < 8; ++i) sums[c][i] = 0.f;
    }
    // a row ahead, where there are registers for it: its loads are on their way while the
    // one before is summed and stored
    constexpr bool AHEAD = WAVES * CH < 32;
    Ahead<T> next_h[CH], next_out[CH], next_sum[CH];
    float next_inverse = 0.f;
    auto fetch = [&](int64_t r) __attribute__((always_inline)) {
        next_inverse = p.inverse[r];
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int e = (c * TEAM + tid) * 8;
            next_h[c].load(static_cast<const T*>(p.h) + r * p.h_stride, e, dim, vector);
            next_out[c].load(static_cast<const T*>(p.grad_out) + r * dim, e, dim, vector);
            if (p.grad_sum) next_sum[c].load(static_cast<const T*>(p.grad_sum) + r * dim, e, dim, vector);
        }
    };
    if (AHEAD && team < p.rows) fetch(team);
    int turn = 0;
    for (int64_t r = team; r < p.rows; r += teams, ++turn) {
        if (!AHEAD) fetch(r);
        const float inverse = next_inverse;
        float u[CH][8], b[CH][8], mean = 0.f;
        Ahead<T> given[CH];
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            given[c] = next_sum[c];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                u[c][i] = next_h[c].at(i) * inverse;
                b[c][i] = next_out[c].at(i);
            }
        }
        if (AHEAD && r + teams < p.rows) fetch(r + teams);
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                sums[c][i] = fmaf(b[c][i], u[c][i], sums[c][i]);
                b[c][i] *= w[c][i];
                mean = fmaf(b[c][i], u[c][i], mean);
            }
        mean = team_sum<WAVES>(mean, parts, turn) / (float)dim;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float v = (b[c][i] - u[c][i] * mean) * inverse;
                if (p.grad_sum) v += given[c].at(i);
                b[c][i] = v;
            }
            store8(static_cast<T*>(p.grad_in) + r * dim, b[c], (c * TEAM + tid) * 8, dim, vector);
        }
    }
    if (p.grad_weight) {
        float* out = static_cast<float*>(p.workspace) + team * dim;
#pragma unroll
        for (int c = 0; c < CH; ++c) store8(out, sums[c], (c * TEAM + tid) * 8, dim, (dim & 3) == 0 && (dim & 7) == 0);
    }
}

// The teams' sums of 32 columns: 32 groups of threads take every 32nd team, and are
// added in their order.
constexpr int kSumColumns = 32, kSumGroups = 32;
template <typename W>
__global__ __launch_bounds__(kSumColumns* kSumGroups) void norm_weight_kernel(const float* parts, W* out, int teams, int dim) {
    __shared__ float sums[kSumGroups][kSumColumns];
    const int column = threadIdx.x % kSumColumns, group = threadIdx.x / kSumColumns, at = blockIdx.x * kSumColumns + column;
    float s = 0.f;
    if (at < dim) {
#pragma unroll 16
        for (int t = group; t < teams; t += kSumGroups) s += parts[(int64_t)t * dim + at];
    }
    sums[group][column] = s;
    __syncthreads();
    if (group == 0 && at < dim) {
#pragma unroll
        for (int g = 1; g < kSumGroups; ++g) s += sums[g][column];
        out[at] = (W)s;
    }
}

// Waves a row: as many as hold it with eight values a thread, sixteen at most (then 16).
// Fewer waves with more values each were slower for 8 to 8192 rows: rows of 7168 with
// a residual, by 16, 8 and 4 waves, 8 rows 3.2, 3.7 and 5.1 us, 400 7.6, 7.9 and 10.4,
// 8192 84, 88 and 97; rows of 4096 by 16, 8 and 4, 8 rows 3.0, 2.8 and 3.5, 8192 57, 49
// and 52; of 1024 by 4, 2 and 1, 8 rows 2.6, 2.6 and 3.2, 8192 16.8, 14.6 and 16.0.
int waves_of(int dim) { return dim <= 512 ? 1 : dim <= 1024 ? 2 : dim <= 2048 ? 4 : dim <= 4096 ? 8 : 16; }

constexpr int64_t kMaxGrid = 4096;

template <typename T, bool CODES>
int launch_typed(const dsa_norm_args& p, int vector, hipStream_t stream) {
    const int waves = waves_of(p.dim);
    const int64_t teams = waves == 1 ? 4 : 1, want = (p.rows + teams - 1) / teams;
    const dim3 grid((unsigned)(want < kMaxGrid ? want : kMaxGrid)), block(waves == 1 ? 256 : 64 * waves);
    auto* kernel = waves == 1   ? norm_kernel<T, CODES, 1, 1>
                   : waves == 2 ? norm_kernel<T, CODES, 2, 1>
                   : waves == 4 ? norm_kernel<T, CODES, 4, 1>
                   : waves == 8 ? norm_kernel<T, CODES, 8, 1>
                   : p.dim <= 8192 ? norm_kernel<T, CODES, 16, 1>
                                   : norm_kernel<T, CODES, 16, 2>;
    hipLaunchKernelGGL(kernel, grid, block, 0, stream, p, vector);
    return (int)hipGetLastError();
}

// Workgroups of the gradient: two a CU keep their columns' sums over 8 rows of 4095.
int64_t grad_groups(int64_t rows, int dim) {
    const int64_t teams = waves_of(dim) == 1 ? 4 : 1, want = (rows + teams - 1) / teams;
    return want < 512 ? want : 512;
}

template <typename T>
int launch_grad_typed(const dsa_norm_grad_args& p, int vector, hipStream_t stream) {
    const int waves = waves_of(p.dim);
    const int64_t groups = grad_groups(p.rows, p.dim);
    const dim3 grid((unsigned)groups), block(waves == 1 ? 256 : 64 * waves);
    auto* kernel = waves == 1   ? norm_grad_kernel<T, 1, 1>
                   : waves == 2 ? norm_grad_kernel<T, 2, 1>
                   : waves == 4 ? norm_grad_kernel<T, 4, 1>
                   : waves == 8 ? norm_grad_kernel<T, 8, 1>
                   : p.dim <= 8192 ? norm_grad_kernel<T, 16, 1>
                                   : norm_grad_kernel<T, 16, 2>;
    hipLaunchKernelGGL(kernel, grid, block, 0, stream, p, vector);
    if (const int rc = (int)hipGetLastError()) return rc;
    if (!p.grad_weight) return 0;
    const int teams = (int)norm_grad_teams(p.rows, p.dim);
    const dim3 columns((unsigned)((p.dim + kSumColumns - 1) / kSumColumns)), threads(kSumColumns * kSumGroups);
    const float* parts = static_cast<const float*>(p.workspace);
    if (p.weight_f32)
        hipLaunchKernelGGL((norm_weight_kernel<float>), columns, threads, 0, stream, parts, static_cast<float*>(p.grad_weight), teams,
                           p.dim);
    else
        hipLaunchKernelGGL((norm_weight_kernel<T>), columns, threads, 0, stream, parts, static_cast<T*>(p.grad_weight), teams, p.dim);
    return (int)hipGetLastError();
}

}  // namespace

int64_t norm_grad_teams(int64_t rows, int dim) {
    return grad_groups(rows, dim) * (waves_of(dim) == 1 ? 4 : 1);
}

int launch_norm(const dsa_norm_args& args, bool codes, bool vector, hipStream_t stream) {
    dsa_norm_args p = args;
    // Codes of rows that follow each other, without a norm, are those of pieces of them:
    // a wave then holds 512 values and waits for no other.
    if (codes && !p.weight && p.dim > 512 && p.dim % 512 == 0 && p.x_stride == p.dim) {
        p.rows *= p.dim / 512;
        p.x_stride = p.dim = 512;
    }
    if (p.dtype == DSA_BF16) return codes ? launch_typed<__bf16, true>(p, vector, stream) : launch_typed<__bf16, false>(p, vector, stream);
    if (p.dtype == DSA_F16) return codes ? launch_typed<f16, true>(p, vector, stream) : launch_typed<f16, false>(p, vector, stream);
    return codes ? launch_typed<float, true>(p, vector, stream) : launch_typed<float, false>(p, vector, stream);
}

int launch_norm_grad(const dsa_norm_grad_args& p, bool vector, hipStream_t stream) {
    if (p.dtype == DSA_BF16) return launch_grad_typed<__bf16>(p, vector, stream);
    if (p.dtype == DSA_F16) return launch_grad_typed<f16>(p, vector, stream);
    return launch_grad_typed<float>(p, vector, stream);
}

}  // namespace dsa
