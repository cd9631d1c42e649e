// Product of 8-bit rows with 8-bit weights, a scale for each 128 of a row and for
// each 128 by 128 of the weights (include/dsa_mi355x_layer.h: dsa_matmul_fp8).  No
// reference counterpart: the reference takes q and kv as given (README.md:19-21).
//
// The weights are the A operand of the matrix instruction and the rows of a its B
// operand: a lane's four results are then four columns of one row of a, which lie in
// one block of weights, and have one scale.  The products of a block of 128 are
// summed by the matrix cores from zero, and added to the result times that scale.
//
// The 8-bit matrix instructions do not keep all bits of their products: sums of 128
// were off by 1.4e-5 (2^-16) of their size, far below the rounding of a 16-bit output
// (2^-9 and 2^-12), far above that of a 32-bit one.  For 32-bit outputs the codes are
// widened to bf16, which holds them exactly, and go through the bf16 instructions,
// whose sums were off by 1.3e-8, at half the rate (2.2 PFLOP/s for 4.6).
#include <hip/hip_runtime.h>
#include <hip/hip_fp16.h>
#include <stdint.h>

#include "kernels.h"

namespace dsa {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((__vector_size__(8 * sizeof(__bf16)))) __bf16 bf16x8;
typedef _Float16 f16;

constexpr int kBlock = 128;

// Eight codes as bf16, exactly.
__device__ __forceinline__ bf16x8 widened(int lo, int hi) {
    const auto a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, false);
    const auto b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, true);
    const auto c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, false);
    const auto d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, true);
    return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Sum over 128 of a 16 x 128 by 16 x 128 product of e4m3 codes.
template <bool EXACT>
__device__ __forceinline__ f32x4 dot128(const i32x8& a, const i32x8& b) {
    f32x4 c = {0.f, 0.f, 0.f, 0.f};
    if constexpr (EXACT) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widened(a[2 * i], a[2 * i + 1]), widened(b[2 * i], b[2 * i + 1]), c, 0, 0, 0);
        return c;
    } else {
        return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, 0, 0, 0);
    }
}

// Lane (r, g)'s part of a row's block of 128: chunks g and 4 + g of 16 bytes.
__device__ __forceinline__ i32x8 load_part(const uint8_t* row, int k, int K, int g) {
    uint4 lo = {0, 0, 0, 0}, hi = {0, 0, 0, 0};
    if (k + 16 * g < K) lo = *reinterpret_cast<const uint4*>(row + k + 16 * g);
    if (k + 64 + 16 * g < K) hi = *reinterpret_cast<const uint4*>(row + k + 64 + 16 * g);
    return i32x8{(int)lo.x, (int)lo.y, (int)lo.z, (int)lo.w, (int)hi.x, (int)hi.y, (int)hi.z, (int)hi.w};
}

template <typename T>
__device__ __forceinline__ void store_out(void* out, int64_t at, float v) {
    static_cast<T*>(out)[at] = (T)v;
}
__device__ __forceinline__ void store_out(void* out, int dtype, int64_t at, float v) {
    if (dtype == DSA_BF16) store_out<__bf16>(out, at, v);
    else if (dtype == DSA_F16) store_out<f16>(out, at, v);
    else store_out<float>(out, at, v);
}

// Few rows of a: a workgroup's waves take the blocks of K in turn, 16 columns by
// 16 MB rows each, and join their sums in LDS.
template <bool EXACT, int MB, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void product_few_kernel(dsa_product_args p) {
    __shared__ f32x4 sums[WAVES][MB][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, g = lane >> 4;
    const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 16 * MB;
    const int blocks = (p.K + kBlock - 1) / kBlock;
    const uint8_t* b = p.b + (int64_t)min(n0 + r, p.N - 1) * p.K;
    const float* b_scale = p.b_scales + (int64_t)(n0 / kBlock) * blocks;
    const uint8_t* a[MB];
    const float* a_scale[MB];
#pragma unroll
    for (int i = 0; i < MB; ++i) {
        const int m = min(m0 + 16 * i + r, p.M - 1);
        a[i] = p.a + (int64_t)m * p.K;
        a_scale[i] = p.a_scales + (int64_t)m * blocks;
    }
    f32x4 acc[MB];
#pragma unroll
    for (int i = 0; i < MB; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int k = wave; k < blocks; k += WAVES) {
        const i32x8 weights = load_part(b, k * kBlock, p.K, g);
        const float sb = b_scale[k];
#pragma unroll
        for (int i = 0; i < MB; ++i) {
            const f32x4 t = dot128<EXACT>(weights, load_part(a[i], k * kBlock, p.K, g));
            const float s = a_scale[i][k] * sb;
            acc[i] += t * s;
        }
    }
#pragma unroll
    for (int i = 0; i < MB; ++i) sums[wave][i][lane] = acc[i];
    __syncthreads();
    for (int i = wave; i < MB; i += WAVES) {
        f32x4 t = sums[0][i][lane];
        for (int w = 1; w < WAVES; ++w) t += sums[w][i][lane];
        const int m = m0 + 16 * i + r, n = n0 + 4 * g;
        if (m < p.M)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (n + j < p.N) store_out(p.out, p.dtype, (int64_t)m * p.N + n + j, t[j]);
    }
}

}  // namespace

int64_t product_ws_bytes(const dsa_product_args&) { return 0; }

int launch_product(const dsa_product_args& p, hipStream_t stream) {
    const dim3 grid((p.N + 15) / 16, (p.M + 63) / 64);
    if (p.dtype == DSA_F32) hipLaunchKernelGGL((product_few_kernel<true, 4, 4>), grid, dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((product_few_kernel<false, 4, 4>), grid, dim3(256), 0, stream, p);
    return (int)hipGetLastError();
}

}  // namespace dsa
