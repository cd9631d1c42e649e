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
#include "mla_tiles.h"

namespace dsa {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
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

// Four bytes a lane straight into LDS: lane l's at lds_base + 4 l.
__device__ __forceinline__ void gather_word(uint32_t lds_base, rsrc_t rsrc, uint32_t off) {
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
    asm volatile(
        "s_mov_b32 m0, %0\n\t"
        "buffer_load_dword %1, %2, 0 offen lds"
        :
        : "s"(__builtin_amdgcn_readfirstlane(lds_base)), "v"(off), "s"(rsrc)
        : "memory", "m0");
#pragma clang diagnostic pop
}

// Lane (r, g)'s part of a row's block of 128: chunks g and 4 + g of 16 bytes.
__device__ __forceinline__ i32x8 load_part(const uint8_t* row, int k, int K, int g) {
    uint4 lo = {0, 0, 0, 0}, hi = {0, 0, 0, 0};
    if (k + 16 * g < K) lo = *reinterpret_cast<const uint4*>(row + k + 16 * g);
    if (k + 64 + 16 * g < K) hi = *reinterpret_cast<const uint4*>(row + k + 64 + 16 * g);
    return i32x8{(int)lo.x, (int)lo.y, (int)lo.z, (int)lo.w, (int)hi.x, (int)hi.y, (int)hi.z, (int)hi.w};
}

// Columns n .. n + 3 of a row of N; `wide`: the four are aligned together.
template <typename OUT>
__device__ __forceinline__ void store4(OUT* row, int n, int N, bool wide, const f32x4& v) {
    typedef OUT out4 __attribute__((ext_vector_type(4)));
    if (wide) {
        if (n < N) *reinterpret_cast<out4*>(row + n) = out4{(OUT)v[0], (OUT)v[1], (OUT)v[2], (OUT)v[3]};
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (n + e < N) row[n + e] = (OUT)v[e];
    }
}

// ------------------------------------------------------------------ few rows
// Up to 128 rows of a: the weights are read once, by one wave, so they go from memory
// straight into registers.  A wave takes 16 NT columns by all 16 MB rows, over every
// WAVES-th block of K, DEPTH blocks ahead; the workgroup's waves join their sums in
// LDS, in the order of the waves.
template <typename OUT, int NT, int MB, int WAVES, int DEPTH>
__global__ __launch_bounds__(64 * WAVES, 1) void product_few_kernel(dsa_product_args p) {
    constexpr bool EXACT = sizeof(OUT) == 4;
    __shared__ f32x4 sums[WAVES][NT * MB][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, g = lane >> 4;
    const int n0 = blockIdx.x * 16 * NT;
    const int K = p.K, blocks = (K + kBlock - 1) / kBlock;
    const auto* b_scale = (const __attribute__((address_space(4))) float*)(uint64_t)p.b_scales + (int64_t)(n0 / kBlock) * blocks;
    const uint8_t* b[NT];
    const uint8_t* a[MB];
    const float* a_scale[MB];
#pragma unroll
    for (int j = 0; j < NT; ++j) b[j] = p.b + (int64_t)min(n0 + 16 * j + r, p.N - 1) * K;
#pragma unroll
    for (int i = 0; i < MB; ++i) {
        const int m = min(16 * i + r, p.M - 1);
        a[i] = p.a + (int64_t)m * K;
        a_scale[i] = p.a_scales + (int64_t)m * blocks;
    }
    f32x4 acc[NT][MB];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < MB; ++i) acc[j][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    struct Ahead {
        i32x8 b[NT], a[MB];
        float s[MB], sb;
    } ahead[DEPTH];
    auto fetch = [&](Ahead& x, int k) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < NT; ++j) x.b[j] = load_part(b[j], k * kBlock, K, g);
#pragma unroll
        for (int i = 0; i < MB; ++i) {
            x.a[i] = load_part(a[i], k * kBlock, K, g);
            x.s[i] = a_scale[i][k];
        }
        x.sb = b_scale[k];
    };
#pragma unroll
    for (int d = 0; d < DEPTH; ++d)
        if (wave + d * WAVES < blocks) fetch(ahead[d], wave + d * WAVES);
    for (int k = wave; k < blocks; k += DEPTH * WAVES) {
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
            const int at = k + d * WAVES;
            if (at >= blocks) break;
            Ahead& x = ahead[d];
#pragma unroll
            for (int i = 0; i < MB; ++i) {
                const float s = x.s[i] * x.sb;
#pragma unroll
                for (int j = 0; j < NT; ++j) acc[j][i] += dot128<EXACT>(x.b[j], x.a[i]) * s;
            }
            if (at + DEPTH * WAVES < blocks) fetch(x, at + DEPTH * WAVES);
        }
    }
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < MB; ++i) sums[wave][j * MB + i][lane] = acc[j][i];
    __syncthreads();
    const bool wide = (p.N & 3) == 0 && ((uintptr_t)p.out & (4 * sizeof(OUT) - 1)) == 0;
#pragma unroll 1
    for (int t = wave; t < NT * MB; t += WAVES) {
        f32x4 v = sums[0][t][lane];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) v += sums[w][t][lane];
        const int m = t % MB * 16 + r;
        if (m < p.M) store4(static_cast<OUT*>(p.out) + (int64_t)m * p.N, n0 + t / MB * 16 + 4 * g, p.N, wide, v);
    }
}

template <typename OUT, int NT, int MB, int WAVES, int DEPTH>
void launch_few(const dsa_product_args& p, hipStream_t stream) {
    const dim3 grid((p.N + 16 * NT - 1) / (16 * NT));
    hipLaunchKernelGGL((product_few_kernel<OUT, NT, MB, WAVES, DEPTH>), grid, dim3(64 * WAVES), 0, stream, p);
}

template <typename OUT, int NT, int MB>
void launch_few(const dsa_product_args& p, hipStream_t stream) {
    constexpr int DEPTH = NT + MB <= 4 ? 4 : NT + MB <= 6 ? 3 : 2;
    if (p.K <= 16 * kBlock) launch_few<OUT, NT, MB, 4, DEPTH>(p, stream);
    else launch_few<OUT, NT, MB, 8, DEPTH>(p, stream);
}

template <typename OUT, int NT>
void launch_few(const dsa_product_args& p, hipStream_t stream) {
    if (p.M <= 16) launch_few<OUT, NT, 1>(p, stream);
    else if (p.M <= 32) launch_few<OUT, NT, 2>(p, stream);
    else if (p.M <= 64) launch_few<OUT, NT, 4>(p, stream);
    else if (p.M <= 96) launch_few<OUT, NT, 6>(p, stream);
    else launch_few<OUT, NT, 8>(p, stream);
}

// ------------------------------------------------------------------ tiles
// Many rows of a: a workgroup of eight waves computes TN columns by TM rows, a wave
// 16 NT by 16 MT of them, from stages of 128 of K in LDS, of which there are two: the
// next one's rows come straight into LDS while one is multiplied.
//
// A row's 128 bytes lie in LDS as eight chunks of 16, chunk c of row r at c ^ swizzle(r):
// a fragment read takes chunks g and 4 + g of 16 rows, and the 16 lanes of a
// ds_read_b128 pass (quads 0, 3, 5, 6 or 1, 2, 4, 7 of a half-wave: rows 0-3 and 12-15
// of one lane group, 4-11 of the next) meet 16 different bank groups.
__device__ __forceinline__ uint32_t swizzle(int row) { return (uint32_t)(row >> 1) & 7u; }

// A workgroup's tile.  Every eighth workgroup is on the same XCD: each XCD gets a run of
// tiles, ordered in bands of up to eight tiles of rows, so that the tiles that run
// there together share rows and columns in its L2.
__device__ __forceinline__ void place(int tiles_m, int tiles_n, int& m, int& n) {
    const uint32_t total = (uint32_t)(tiles_m * tiles_n), each = total / 8, rest = total % 8;
    const uint32_t xcd = blockIdx.x % 8, t = xcd * each + min(xcd, rest) + blockIdx.x / 8;
    const uint32_t band = t / (uint32_t)(8 * tiles_n), in_band = t % (uint32_t)(8 * tiles_n);
    const uint32_t high = min(8u, (uint32_t)tiles_m - 8 * band);
    m = (int)(8 * band + in_band % high);
    n = (int)(in_band / high);
}

template <int NT, int MT, int WN, int WM, int KS, int STAGES>
struct Tile {
    static constexpr int TN = 16 * NT * WN, TM = 16 * MT * WM, GROUP = WN * WM, WAVES = GROUP * KS, THREADS = 64 * WAVES;
    static constexpr int B_LOADS = (TN + 8 * GROUP - 1) / (8 * GROUP), A_LOADS = (TM + 8 * GROUP - 1) / (8 * GROUP);  // a wave, of 8 rows each
    static constexpr int S_WAVES = (TM + 63) / 64;  // loads of 64 scales each
    static constexpr int LOADS = B_LOADS + A_LOADS + 1;
    static constexpr int A_OFF = B_LOADS * GROUP * 8 * kBlock, S_OFF = A_OFF + A_LOADS * GROUP * 8 * kBlock;
    static constexpr int BLOCK = S_OFF + S_WAVES * 256, STAGE = BLOCK * KS;
    static constexpr int JOIN_BYTES = KS > 1 ? WAVES * NT * MT * 1024 : 0;
    static constexpr int LDS_BYTES = STAGES * STAGE > JOIN_BYTES ? STAGES * STAGE : JOIN_BYTES;
    static_assert(S_WAVES <= GROUP, "a scale load a wave");
    static_assert(LDS_BYTES <= 160 * 1024, "LDS budget");
    static_assert((STAGES - 1) * LOADS < 64, "loads in flight are counted in six bits");
    // a wave's columns lie in one block of weights
    static_assert(kBlock % (16 * NT) == 0, "one scale a wave");
};

template <typename OUT, int NT, int MT, int WN, int WM, int KS, int STAGES>
__global__ __launch_bounds__(64 * WN * WM * KS, 1) void product_tile_kernel(dsa_product_args p, int tiles_m, int tiles_n) {
    constexpr bool EXACT = sizeof(OUT) == 4;
    using T = Tile<NT, MT, WN, WM, KS, STAGES>;
    __shared__ __attribute__((aligned(1024))) char smem[T::LDS_BYTES];
    const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)smem;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int group = KS > 1 ? wave / T::GROUP : 0, in_group = KS > 1 ? wave % T::GROUP : wave;
    const int r = lane & 15, g = lane >> 4;
    int tile_m, tile_n;
    place(tiles_m, tiles_n, tile_m, tile_n);
    const int m0 = tile_m * T::TM, n0 = tile_n * T::TN;
    const int K = p.K, blocks = (K + kBlock - 1) / kBlock, steps = (blocks + KS - 1) / KS;
    const int rows_m = min(T::TM, p.M - m0), rows_n = min(T::TN, p.N - n0);
    const char* b_base = reinterpret_cast<const char*>(p.b) + (int64_t)n0 * K;
    const char* a_base = reinterpret_cast<const char*>(p.a) + (int64_t)m0 * K;
    const char* s_base = reinterpret_cast<const char*>(p.a_scales + (int64_t)m0 * blocks);
    // Lane l of a load brings in chunk l % 8 of row l / 8: rows 8 apart have the same
    // swizzle but for bit 2.
    const int in8 = lane >> 3;
    const uint32_t chunk = 16u * ((uint32_t)(lane & 7) ^ swizzle(in8));
    // A group's block of step t: behind the last one nothing is read, but the loads are
    // the same, so that they can be counted on.  Rows behind the last are out of the
    // descriptors' range, and so zeros.
    auto issue = [&](int t) __attribute__((always_inline)) {
        const uint32_t stage = lds + (uint32_t)(t % STAGES) * T::STAGE + (uint32_t)group * T::BLOCK;
        const int k = t * KS + group, at = k * kBlock, left = K - at;  // bytes of a row from here on
        const bool on = k < blocks;
        const rsrc_t rb = make_rsrc(b_base + at, on ? (uint32_t)(rows_n * K - at) : 0u);
        const rsrc_t ra = make_rsrc(a_base + at, on ? (uint32_t)(rows_m * K - at) : 0u);
        auto offset = [&](int first) __attribute__((always_inline)) -> uint32_t {
            const uint32_t c = chunk ^ (first & 8 ? 64u : 0u);
            return (int)c < left ? (uint32_t)((first + in8) * K) + c : 0x80000000u;  // behind the row's end: zeros
        };
#pragma unroll
        for (int i = 0; i < T::B_LOADS; ++i) {
            const int first = (in_group * T::B_LOADS + i) * 8;
            gather_lanes(stage + (uint32_t)first * kBlock, rb, offset(first));
        }
#pragma unroll
        for (int i = 0; i < T::A_LOADS; ++i) {
            const int first = (in_group * T::A_LOADS + i) * 8;
            gather_lanes(stage + T::A_OFF + (uint32_t)first * kBlock, ra, offset(first));
        }
        const int part = in_group % T::S_WAVES;  // some are loaded twice, the same
        gather_word(stage + T::S_OFF + (uint32_t)part * 256u,
                    make_rsrc(s_base + 4 * k, on ? (uint32_t)(4 * (rows_m * blocks - k)) : 0u),
                    (uint32_t)(4 * (64 * part + lane) * blocks));
    };
    const int wn = in_group % WN, wm = in_group / WN;
    const int band = min(n0 + 16 * NT * wn, p.N - 1) / kBlock;
    // a scalar load: the compiler does not count the loads to LDS, and would wait for all of them with one of its own
    const auto* b_scale = (const __attribute__((address_space(4))) float*)(uint64_t)p.b_scales + (int64_t)band * blocks;
    // fragment reads: chunk g (and 4 + g: ^ 64) of row r of a 16-row tile
    const uint32_t frag = (uint32_t)r * kBlock + 16u * ((uint32_t)g ^ swizzle(r));
    const uint32_t b_frag = frag + (uint32_t)wn * NT * 16 * kBlock, a_frag = frag + T::A_OFF + (uint32_t)wm * MT * 16 * kBlock;
    const uint32_t s_frag = T::S_OFF + 4u * (uint32_t)(wm * MT * 16 + r);
    f32x4 acc[NT][MT];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[j][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int t = 0; t < STAGES - 1; ++t) issue(t);
    float sb = b_scale[min(group, blocks - 1)];
#pragma unroll 1
    for (int t = 0; t < steps; ++t) {
        wait_vmcnt<(STAGES - 2) * T::LOADS>();
        lds_barrier();  // stage t is there, and every wave is done with stage t - 1
        issue(t + STAGES - 1);
        const int k = t * KS + group;
        if (KS > 1 && k >= blocks) break;  // the last step, of a group that has none: no barrier follows but the one below
        const uint32_t stage = lds + (uint32_t)(t % STAGES) * T::STAGE + (uint32_t)group * T::BLOCK;
        const uint32_t b_lo = stage + b_frag, b_hi = b_lo ^ 64u, a_lo = stage + a_frag, a_hi = a_lo ^ 64u;
        auto read = [&](uint32_t lo, uint32_t hi, int tile) __attribute__((always_inline)) -> i32x8 {
            const i32x4 l = lds_load<i32x4>(lo + tile * 16 * kBlock), h = lds_load<i32x4>(hi + tile * 16 * kBlock);
            return __builtin_shufflevector(l, h, 0, 1, 2, 3, 4, 5, 6, 7);
        };
        i32x8 af[MT], bf[2];
        float s[MT];
        bf[0] = read(b_lo, b_hi, 0);
#pragma unroll
        for (int i = 0; i < MT; ++i) af[i] = read(a_lo, a_hi, i);
#pragma unroll
        for (int i = 0; i < MT; ++i) s[i] = lds_load<float>(stage + s_frag + 64 * i) * sb;
        sb = b_scale[min(k + KS, blocks - 1)];
        // products of tile j beside the sums of tile j - 1
        f32x4 u[2][MT];
#pragma unroll
        for (int j = 0; j <= NT; ++j) {
            if (j + 1 < NT) bf[(j + 1) & 1] = read(b_lo, b_hi, j + 1);
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                if (j < NT) u[j & 1][i] = dot128<EXACT>(bf[j & 1], af[i]);
                if (j > 0) acc[j - 1][i] += u[(j - 1) & 1][i] * s[i];
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    }
    wait_vmcnt<0>();  // loads behind the last block write zeros into LDS
    const bool wide = (p.N & 3) == 0 && ((uintptr_t)p.out & (4 * sizeof(OUT) - 1)) == 0;
    auto store = [&](int j, int i, const f32x4& v) __attribute__((always_inline)) {
        const int m = m0 + (wm * MT + i) * 16 + r;
        if (m < p.M) store4(static_cast<OUT*>(p.out) + (int64_t)m * p.N, n0 + (wn * NT + j) * 16 + 4 * g, p.N, wide, v);
    };
    if constexpr (KS == 1) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) store(j, i, acc[j][i]);
    } else {  // the groups' sums, in their order: a group joins every KS-th tile
        lds_barrier();
        auto at = [&](int of, int tile) __attribute__((always_inline)) -> uint32_t {
            return lds + (uint32_t)(((of * T::GROUP + in_group) * NT * MT + tile) * 1024 + 16 * lane);
        };
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int i = 0; i < MT; ++i) lds_store<f32x4>(at(group, j * MT + i), acc[j][i]);
        lds_barrier();
#pragma unroll 1
        for (int tile = group; tile < NT * MT; tile += KS) {
            f32x4 v = lds_load<f32x4>(at(0, tile));
#pragma unroll
            for (int of = 1; of < KS; ++of) v += lds_load<f32x4>(at(of, tile));
            store(tile / MT, tile % MT, v);
        }
    }
}

template <typename OUT, int NT, int MT, int WN, int WM, int KS, int STAGES>
void launch_tile(const dsa_product_args& p, hipStream_t stream) {
    using T = Tile<NT, MT, WN, WM, KS, STAGES>;
    const int tiles_m = (p.M + T::TM - 1) / T::TM, tiles_n = (p.N + T::TN - 1) / T::TN;
    hipLaunchKernelGGL((product_tile_kernel<OUT, NT, MT, WN, WM, KS, STAGES>), dim3(tiles_m * tiles_n), dim3(T::THREADS), 0, stream, p,
                       tiles_m, tiles_n);
}

template <typename OUT>
void launch_typed(const dsa_product_args& p, hipStream_t stream) {
    if (p.M > 128) {
        if constexpr (sizeof(OUT) == 4) launch_tile<OUT, 4, 4, 2, 4, 1, 2>(p, stream);
        else launch_tile<OUT, 8, 4, 2, 4, 1, 2>(p, stream);
    } else {
        if (p.N >= 32 * 224) launch_few<OUT, 2>(p, stream);
        else launch_few<OUT, 1>(p, stream);
    }
}

}  // namespace

int64_t product_ws_bytes(const dsa_product_args&) { return 0; }

int launch_product(const dsa_product_args& p, hipStream_t stream) {
    if (p.dtype == DSA_BF16) launch_typed<__bf16>(p, stream);
    else if (p.dtype == DSA_F16) launch_typed<f16>(p, stream);
    else launch_typed<float>(p, stream);
    return (int)hipGetLastError();
}

}  // namespace dsa
