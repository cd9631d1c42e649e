// Product of 8-bit rows with 8-bit weights, a scale for each 128 of a row and for
// each 128 by 128 of the weights (include/dsa_mi355x_layer.h: dsa_matmul_fp8).  No
// reference counterpart: the reference takes q and kv as given (README.md:19-21).
//
// The weights are the A operand of the matrix instruction and the rows of a its B
// operand: a lane's four results are then four columns of one row of a, which lie in
// one block of weights, and have one scale.  The products of a block of 128 are
// summed by the matrix cores from zero, and added to the result times that scale.
//
// The 8-bit matrix instructions do not keep all bits of their products: of eight
// neighbours each is cut, towards zero, to a multiple of 2^-13 of the power of two that
// the largest one's exponents make (seen in sums of a large product, its opposite and
// a third).  Sums of 128 were off by 1.4e-5 (2^-16) of their size, far below the
// rounding of a 16-bit output (2^-9 and 2^-12), far above that of a 32-bit one.  For 32-bit outputs the codes are
// widened to bf16, which holds them exactly, and go through the bf16 instructions,
// whose sums were off by 1.3e-8, at half the rate (2.2 PFLOP/s for 4.6).
//
// One family of tiles, from 16 by 16 with K split over four waves to 256 by 256
// (kVariants: which one, and what the others took).  Times below: weights out of 1 GiB of
// them in turn, so that they come from HBM, and in brackets those of a few in turn, which
// stay in the last cache.  Few rows are bound by the weights' bytes and the latency of the
// steps (8 rows, 2112 columns, K 7168 7.0 to 8.1 us (6.1); 77, 24576, 1536 12.7 (10.4, 4.0
// TB/s); 8, 7168, 16384 24.6, 4.8 TB/s): from HBM a CU gets about 50 GB/s however much is
// under way.  Middle ones (1000, 2112, 7168 27.8 (23.9 to 25.3)) by the same and the steps
// of their smaller tiles.  Many by the matrix cores, 57 % busy, and the clock that is left
// to them under load (8192, 7168, 16384 803 to 846 us, 2.27 to 2.4 PFLOP/s; a library's
// product without these scales 699): products and sums alone of a step of a 256 by 256
// tile, of random codes, take 0.97 us on half the chip and 1.20 on all of it.  32-bit
// outputs: 8, 77, 1000 and 8192 rows 7.2 to 8.1, 16, 54 and 1608 to 1680 us, 1.2 PFLOP/s.
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

// ------------------------------------------------------------------ tiles
// A workgroup computes TN columns by TM rows, a wave 16 NT by 16 MT of them, from a ring
// of STAGES stages in LDS, which rows come into straight from memory.  A stage holds KS
// blocks of 128 of K; KS groups of waves take one each, and join their sums at the end,
// in their order.  LW: waves of their own load, and the others do not.
//
// A row's 128 bytes lie in LDS as eight chunks of 16, chunk c of row r at c ^ swizzle(r):
// a fragment read takes chunks g and 4 + g of 16 rows, and the 16 lanes of a
// ds_read_b128 pass (quads 0, 3, 5, 6 or 1, 2, 4, 7 of a half-wave: rows 0-3 and 12-15
// of one lane group, 4-11 of the next) meet 16 different bank groups.
__device__ __forceinline__ uint32_t swizzle(int row) { return (uint32_t)(row >> 1) & 7u; }

// Workgroup i of `total` counted along the XCDs: every eighth is on the same one, and
// each XCD gets a run of them.
__device__ __forceinline__ uint32_t along_xcds(uint32_t i, uint32_t total) {
    const uint32_t each = total / 8, rest = total % 8, xcd = i % 8;
    return xcd * each + min(xcd, rest) + i / 8;
}
// Tile t, in bands of up to eight tiles of rows, so that the tiles that run together on
// an XCD share rows and columns in its L2.
__device__ __forceinline__ void place(uint32_t t, int tiles_m, int tiles_n, int& m, int& n) {
    const uint32_t band = t / (uint32_t)(8 * tiles_n), in_band = t % (uint32_t)(8 * tiles_n);
    const uint32_t high = min(8u, (uint32_t)tiles_m - 8 * band);
    m = (int)(8 * band + in_band % high);
    n = (int)(in_band / high);
}

template <int NT, int MT, int WN, int WM, int KS, int STAGES, int LW = 0>
struct Tile {
    static constexpr int TN = 16 * NT * WN, TM = 16 * MT * WM, GROUP = WN * WM, WAVES = GROUP * KS, THREADS = 64 * (WAVES + LW);
    static constexpr int LOADING = LW ? LW : GROUP;  // waves that load a block
    static constexpr int B_LOADS = (TN + 8 * LOADING - 1) / (8 * LOADING), A_LOADS = (TM + 8 * LOADING - 1) / (8 * LOADING);  // a wave, of 8 rows each
    static constexpr int LOADS = B_LOADS + A_LOADS;
    static constexpr int A_OFF = B_LOADS * LOADING * 8 * kBlock, BLOCK = A_OFF + A_LOADS * LOADING * 8 * kBlock, STAGE = BLOCK * KS;
    // Scales come 8 or 16 blocks of a row at a time, a row's 32 or 64 bytes, four or eight rows a load.
    static constexpr int S_BLOCKS = KS * (STAGES - 1) > 8 ? 16 : 8, S_STEPS = S_BLOCKS / KS, S_ROWS = 64 / S_BLOCKS;
    // Four rows (two, of 16 blocks) fill 32 banks: the next ones have their blocks in another order.
    static __device__ constexpr int s_swizzle(int row) { return S_BLOCKS == 8 ? row >> 2 & 3 : row >> 1 & 7; }
    static constexpr int S_LOADS = (TM + S_ROWS * LOADING * KS - 1) / (S_ROWS * LOADING * KS);
    static constexpr int S_OFF = STAGES * STAGE, SB_OFF = S_LOADS * LOADING * KS * 256, S_BYTES = SB_OFF + 256;
    static constexpr int JOIN_BYTES = KS > 1 ? WAVES * NT * MT * 1024 : 0;
    static constexpr int RING_BYTES = S_OFF + 2 * S_BYTES, LDS_BYTES = RING_BYTES > JOIN_BYTES ? RING_BYTES : JOIN_BYTES;
    // With two stages, the part of a stage that is read first -- the rows of a, and of
    // the weights half of each wave's -- is loaded again within the step that reads it.
    static constexpr bool HALVES = STAGES == 2 && NT % 2 == 0 && B_LOADS % 2 == 0 && TN % (8 * GROUP) == 0 && KS == 1;
    static constexpr int EARLY = A_LOADS + B_LOADS / 2;
    static constexpr int EARLIEST = (NT / 2 * EARLY + NT / 2) / (NT / 2 + 1);  // of them, those issued before a step's last tile
    static constexpr int AHEAD = HALVES ? EARLIEST : (STAGES - 2) * LOADS;  // loads that may be in flight when a step begins
    // Products that wait to be added (LW): what the registers hold beside the operands.
    static constexpr int BEHIND = NT * MT <= 6 ? NT * MT : NT * MT <= 8 ? 4 : 2;
    static_assert(NT * MT % BEHIND == 0 || LW == 0, "a product has one register");
    static_assert(LW == 0 || (KS == 1 && STAGES > 2), "operands a step ahead");
    static_assert(STAGES > 2 || HALVES, "two stages by halves");
    static_assert(S_BLOCKS % KS == 0 && S_STEPS >= STAGES - (LW ? 0 : 1), "scales have landed by the step that needs them");
    static_assert(LDS_BYTES <= 160 * 1024, "LDS budget");
    static_assert((STAGES - (LW ? 0 : 1)) * LOADS < 64, "loads in flight are counted in six bits");
    // a wave's columns lie in one block of weights
    static_assert(kBlock % (16 * NT) == 0, "one scale a wave");
};

template <typename OUT, int NT, int MT, int WN, int WM, int KS, int STAGES, int LW = 0>
__device__ __forceinline__ void product_tile(const dsa_product_args& p, uint32_t lds, int m0, int n0) {
    constexpr bool EXACT = sizeof(OUT) == 4;
    using T = Tile<NT, MT, WN, WM, KS, STAGES, LW>;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const bool loads = LW == 0 || wave >= T::WAVES;
    const int group = KS > 1 ? wave / T::GROUP : 0, in_group = KS > 1 ? wave % T::GROUP : LW > 0 && loads ? wave - T::WAVES : wave;
    const int r = lane & 15, g = lane >> 4;
    const int K = p.K, blocks = (K + kBlock - 1) / kBlock, steps = (blocks + KS - 1) / KS;
    const int rows_m = min(T::TM, p.M - m0), rows_n = min(T::TN, p.N - n0);
    const char* b_base = reinterpret_cast<const char*>(p.b) + (int64_t)n0 * K;
    const char* a_base = reinterpret_cast<const char*>(p.a) + (int64_t)m0 * K;
    const char* s_base = reinterpret_cast<const char*>(p.a_scales + (int64_t)m0 * blocks);
    // Lane l of a load brings in chunk l % 8 of row l / 8: rows 8 apart have the same
    // swizzle but for bit 2.
    const int in8 = lane >> 3;
    const uint32_t chunk = 16u * ((uint32_t)(lane & 7) ^ swizzle(in8));
    // Load i of a group's block of step t: behind the last one nothing is read, but the
    // loads are the same, so that they can be counted on.  Rows behind the last are out
    // of the descriptors' range, and so zeros.
    struct Next {
        rsrc_t b, a;
        uint32_t stage;
        int left;  // bytes of a row from the block on
    };
    auto next_at = [&](int t, uint32_t stage) __attribute__((always_inline)) -> Next {
        const int k = t * KS + group, at = k * kBlock;
        const bool on = k < blocks;
        return Next{make_rsrc(b_base + at, on ? (uint32_t)(rows_n * K - at) : 0u),
                    make_rsrc(a_base + at, on ? (uint32_t)(rows_m * K - at) : 0u), lds + stage + (uint32_t)group * T::BLOCK, K - at};
    };
    auto issue = [&](const Next& n, int i) __attribute__((always_inline)) {
        const bool of_b = i >= T::A_LOADS;
        int first = of_b ? (in_group * T::B_LOADS + i - T::A_LOADS) * 8 : (in_group * T::A_LOADS + i) * 8;
        if (T::HALVES && of_b) {  // first the rows 0 .. 8 NT - 1 of each 16 NT, then the others
            const int half = i - T::A_LOADS >= T::B_LOADS / 2, at = in_group * (T::B_LOADS / 2) + (i - T::A_LOADS) % (T::B_LOADS / 2);
            first = at / NT * 16 * NT + half * 8 * NT + at % NT * 8;
        }
        const uint32_t c = chunk ^ (first & 8 ? 64u : 0u);
        const uint32_t off = (int)c < n.left ? (uint32_t)((first + in8) * K) + c : 0x80000000u;  // behind the row's end: zeros
        gather_lanes(n.stage + (of_b ? 0 : T::A_OFF) + (uint32_t)first * kBlock, of_b ? n.b : n.a, off);
    };
    const rsrc_t rs = make_rsrc(s_base, (uint32_t)(4 * rows_m * blocks));
    const rsrc_t rsb = make_rsrc(p.b_scales + (int64_t)(n0 / kBlock) * blocks, (uint32_t)(4 * ((rows_n + kBlock - 1) / kBlock) * blocks));
    const int s_row = lane / T::S_BLOCKS, s_block = lane % T::S_BLOCKS;
    auto issue_scales = [&](int c) __attribute__((always_inline)) {  // of blocks c * S_BLOCKS on
        const uint32_t to = lds + T::S_OFF + (uint32_t)(c & 1) * T::S_BYTES;
        const int k = c * T::S_BLOCKS + s_block;
        if (group == 0 && in_group == 0)  // the weights': those of 128 columns as those of a row
            gather_word(to + T::SB_OFF, rsb, k < blocks ? (uint32_t)(4 * (s_row * blocks + k)) : 0x80000000u);
#pragma unroll
        for (int i = 0; i < T::S_LOADS; ++i) {
            const int first = ((group * T::LOADING + in_group) * T::S_LOADS + i) * T::S_ROWS;
            const int of = c * T::S_BLOCKS + (s_block ^ T::s_swizzle(first + s_row));
            gather_word(to + (uint32_t)first * (4 * T::S_BLOCKS), rs,
                        of < blocks ? (uint32_t)(4 * ((first + s_row) * blocks + of)) : 0x80000000u);
        }
    };
    const int wn = in_group % WN, wm = in_group / WN;
    // fragment reads: chunk g (and 4 + g: ^ 64) of row r of a 16-row tile
    const uint32_t frag = (uint32_t)r * kBlock + 16u * ((uint32_t)g ^ swizzle(r));
    const uint32_t b_frag = frag + (uint32_t)wn * NT * 16 * kBlock, a_frag = frag + T::A_OFF + (uint32_t)wm * MT * 16 * kBlock;
    // a row's scale: of block k, its number ^ s_swizzle(row)
    const uint32_t s_frag = lds + T::S_OFF + 4u * T::S_BLOCKS * (uint32_t)(wm * MT * 16 + r) + 4u * (uint32_t)T::s_swizzle(r);
    auto scale_at = [&](int k) __attribute__((always_inline)) -> uint32_t {
        return (s_frag ^ 4u * (uint32_t)(k % T::S_BLOCKS)) + (uint32_t)(k / T::S_BLOCKS & 1) * T::S_BYTES;
    };
    const uint32_t sb_frag = lds + T::S_OFF + T::SB_OFF + 4u * T::S_BLOCKS * (uint32_t)((n0 % kBlock + 16 * NT * wn) / kBlock);
    f32x4 acc[NT][MT];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[j][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto read = [&](uint32_t lo, uint32_t hi, int tile) __attribute__((always_inline)) -> i32x8 {
        const i32x4 l = lds_load<i32x4>(lo + tile * 16 * kBlock), h = lds_load<i32x4>(hi + tile * 16 * kBlock);
        return __builtin_shufflevector(l, h, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    if constexpr (LW > 0) {
        // Waves of their own load, whom a full queue stops alone, and the others read a
        // step's operands in the step before, so that LDS and the matrix cores work beside
        // each other.  Stage t is then free for loads in step t.
        uint32_t at = 0;
        if (loads) {
            issue_scales(0);
#pragma unroll
            for (int t = 0; t < STAGES; ++t) {
                const Next n = next_at(t, (uint32_t)t * T::STAGE);
#pragma unroll
                for (int i = 0; i < T::LOADS; ++i) issue(n, i);
            }
            wait_vmcnt<(STAGES - 1) * T::LOADS>();
            lds_barrier();
#pragma unroll 1
            for (int t = 0; t < steps; ++t) {
                wait_vmcnt<T::AHEAD>();
                lds_barrier();
                if (t % T::S_STEPS == 0) issue_scales(t / T::S_STEPS + 1);
                const Next n = next_at(t + STAGES, at);
#pragma unroll
                for (int i = 0; i < T::LOADS; ++i) issue(n, i);
                at = at + T::STAGE == T::S_OFF ? 0 : at + T::STAGE;
            }
            wait_vmcnt<0>();
            return;
        }
        struct Operands {
            i32x8 a[MT], b[NT];
            float s[MT], sb;
        };
        auto fetch = [&](Operands& o, uint32_t stage, int t, int i) __attribute__((always_inline)) {
            const uint32_t chunk_at = (uint32_t)(t / T::S_BLOCKS & 1) * T::S_BYTES + 4u * (uint32_t)(t % T::S_BLOCKS);
            const uint32_t s_at = scale_at(t);
            const uint32_t b_lo = lds + stage + b_frag, a_lo = lds + stage + a_frag;
            if (i == 0) o.sb = lds_load<float>(sb_frag + chunk_at);
            if (i < NT) {
                o.b[i] = read(b_lo, b_lo ^ 64u, i);
            } else {
                o.a[i - NT] = read(a_lo, a_lo ^ 64u, i - NT);
                o.s[i - NT] = lds_load<float>(s_at + 64 * T::S_BLOCKS * (i - NT));
            }
        };
        // A product is added D products later, so that none is waited for: those of a step's
        // end beside the next step's first.
        constexpr int P = NT * MT, D = T::BEHIND;
        f32x4 u[D];
        float last[MT];  // scales of the step before
        auto add = [&](int i, const float (&s)[MT]) __attribute__((always_inline)) {  // what product i's register holds
            const int of = i < D ? P + i - D : i - D;
            acc[of / MT][of % MT] += u[i % D] * (i < D ? last : s)[of % MT];
        };
        auto step = [&](const Operands& o, Operands& next, int t) __attribute__((always_inline)) {
            lds_barrier();  // stage t + 1 is there, and every wave has read stage t
            at = at + T::STAGE == T::S_OFF ? 0 : at + T::STAGE;
            float s[MT];
#pragma unroll
            for (int i = 0; i < MT; ++i) s[i] = o.s[i] * o.sb;
#pragma unroll
            for (int i = 0; i < P; ++i) {
#pragma unroll
                for (int k = 0; k < NT + MT; ++k)
                    if (k * P / (NT + MT) == i) fetch(next, at, t + 1, k);
                add(i, s);
                u[i % D] = dot128<EXACT>(o.b[i / MT], o.a[i % MT]);
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int i = 0; i < MT; ++i) last[i] = s[i];
        };
        Operands even, odd;
#pragma unroll
        for (int i = 0; i < D; ++i) u[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < MT; ++i) last[i] = 0.f;
        lds_barrier();
#pragma unroll
        for (int k = 0; k < NT + MT; ++k) fetch(even, 0, 0, k);
#pragma unroll 1
        for (int t = 0; t < steps; t += 2) {
            step(even, odd, t);
            if (t + 1 < steps) step(odd, even, t + 1);
        }
#pragma unroll
        for (int i = 0; i < D; ++i) add(i, last);
    } else if constexpr (T::HALVES) {
        // Two stages.  A step's first operands are read beside the last products of the one
        // before, in the place of those that it is done with, so that the matrix cores go
        // on through the barrier: 8192 rows, 2112 columns, K 7168 168 -> 155 us.
        issue_scales(0);
        {
            const Next n = next_at(0, 0), n1 = next_at(1, T::STAGE);
#pragma unroll
            for (int i = 0; i < T::LOADS; ++i) issue(n, i);
#pragma unroll
            for (int i = 0; i < T::EARLY; ++i) issue(n1, i);
        }
        uint32_t at = 0;  // stage t; t + 1: the other one
        i32x8 af[MT], bf[2];
        float next_s[MT], next_sb;
        auto read_b = [&](uint32_t stage, int tile) __attribute__((always_inline)) -> i32x8 {
            return read(lds + stage + b_frag, (lds + stage + b_frag) ^ 64u, tile);
        };
        auto read_a = [&](uint32_t stage, int tile) __attribute__((always_inline)) -> i32x8 {
            return read(lds + stage + a_frag, (lds + stage + a_frag) ^ 64u, tile);
        };
        auto read_scales = [&](int k) __attribute__((always_inline)) {
            const uint32_t chunk_at = (uint32_t)(k / T::S_BLOCKS & 1) * T::S_BYTES + 4u * (uint32_t)(k % T::S_BLOCKS);
            next_sb = lds_load<float>(sb_frag + chunk_at);
#pragma unroll
            for (int i = 0; i < MT; ++i) next_s[i] = lds_load<float>(scale_at(k) + 64 * T::S_BLOCKS * i);
        };
        wait_vmcnt<T::EARLY>();
        lds_barrier();
        bf[0] = read_b(0, 0);
#pragma unroll
        for (int i = 0; i < MT; ++i) af[i] = read_a(0, i);
        read_scales(0);
#pragma unroll 1
        for (int t = 0; t < steps; ++t) {
            const uint32_t other = T::STAGE - at;
            float s[MT];
#pragma unroll
            for (int i = 0; i < MT; ++i) s[i] = next_s[i] * next_sb;
            if (t % T::S_STEPS == 0) issue_scales(t / T::S_STEPS + 1);
            const Next n = next_at(t + 1, other), n2 = next_at(t + 2, at);
            // products of tile j beside the sums of tile j - 1, and a few loads
            f32x4 u[2][MT];
#pragma unroll
            for (int j = 0; j <= NT; ++j) {
                if (j == NT - 1) {  // stage t + 1 is there, and every wave has read stage t: the next step's first operands
                    wait_vmcnt<T::AHEAD>();
                    lds_barrier();
                    bf[0] = read_b(other, 0);
                    read_scales(t + 1);
                }
                if (j + 1 < NT) bf[(j + 1) & 1] = read_b(at, j + 1);
                // the last loads of stage t + 1, then, when all waves have read the first
                // part of stage t (tiles up to NT / 2 - 1 are in registers), those of t + 2
#pragma unroll
                for (int i = T::EARLY; i < T::LOADS; ++i)
                    if (i - T::EARLY == j) issue(n, i);
                if (j == NT / 2 - 1) lds_barrier();
#pragma unroll
                for (int i = 0; i < T::EARLY; ++i)
                    if (j >= NT / 2 - 1 && j < NT && i * (NT / 2 + 1) / T::EARLY == j - (NT / 2 - 1)) issue(n2, i);
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    if (j < NT) u[j & 1][i] = dot128<EXACT>(bf[j & 1], af[i]);
                    if (j > 0) acc[j - 1][i] += u[(j - 1) & 1][i] * s[i];
                    __builtin_amdgcn_sched_barrier(0);
                    if (j == NT - 1) af[i] = read_a(other, i);
                }
            }
            at = other;
        }
    } else {
        issue_scales(0);
#pragma unroll
        for (int t = 0; t < STAGES - 1; ++t) {
            const Next n = next_at(t, (uint32_t)t * T::STAGE);
#pragma unroll
            for (int i = 0; i < T::LOADS; ++i) issue(n, i);
        }
        uint32_t at = 0, ahead = (STAGES - 1) * T::STAGE;
#pragma unroll 1
        for (int t = 0; t < steps; ++t) {
            wait_vmcnt<T::AHEAD>();
            lds_barrier();  // stage t is there, and every wave is done with stage t - 1
            const int k = t * KS + group;
            const uint32_t stage = lds + at + (uint32_t)group * T::BLOCK;
            const uint32_t b_lo = stage + b_frag, b_hi = b_lo ^ 64u, a_lo = stage + a_frag, a_hi = a_lo ^ 64u;
            if (KS > 1 && k >= blocks) break;  // the last step, of a group that has no block: only the barriers of the end follow
            i32x8 af[MT], bf[2];
            float s[MT];
            bf[0] = read(b_lo, b_hi, 0);
#pragma unroll
            for (int i = 0; i < MT; ++i) af[i] = read(a_lo, a_hi, i);
            const uint32_t chunk_at = (uint32_t)(k / T::S_BLOCKS & 1) * T::S_BYTES + 4u * (uint32_t)(k % T::S_BLOCKS);
            const float sb = lds_load<float>(sb_frag + chunk_at);
#pragma unroll
            for (int i = 0; i < MT; ++i) s[i] = lds_load<float>(scale_at(k) + 64 * T::S_BLOCKS * i);
            if (t % T::S_STEPS == 0) issue_scales(t / T::S_STEPS + 1);
            const Next n = next_at(t + STAGES - 1, ahead);
            // products of tile j beside the sums of tile j - 1, and a few loads
            f32x4 u[2][MT];
#pragma unroll
            for (int j = 0; j <= NT; ++j) {
                if (j + 1 < NT) bf[(j + 1) & 1] = read(b_lo, b_hi, j + 1);
#pragma unroll
                for (int i = 0; i < T::LOADS; ++i)
                    if (i * NT / T::LOADS == j) issue(n, i);
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    if (j == 0) s[i] *= sb;
                    if (j < NT) u[j & 1][i] = dot128<EXACT>(bf[j & 1], af[i]);
                    if (j > 0) acc[j - 1][i] += u[(j - 1) & 1][i] * s[i];
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            at = at + T::STAGE == T::S_OFF ? 0 : at + T::STAGE;
            ahead = ahead + T::STAGE == T::S_OFF ? 0 : ahead + T::STAGE;
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
        auto part = [&](int of, int tile) __attribute__((always_inline)) -> uint32_t {
            return lds + (uint32_t)(((of * T::GROUP + in_group) * NT * MT + tile) * 1024 + 16 * lane);
        };
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int i = 0; i < MT; ++i) lds_store<f32x4>(part(group, j * MT + i), acc[j][i]);
        lds_barrier();
#pragma unroll 1
        for (int tile = group; tile < NT * MT; tile += KS) {
            f32x4 v = lds_load<f32x4>(part(0, tile));
#pragma unroll
            for (int of = 1; of < KS; ++of) v += lds_load<f32x4>(part(of, tile));
            store(tile / MT, tile % MT, v);
        }
    }
}

template <typename OUT, int NT, int MT, int WN, int WM, int KS, int STAGES, int LW = 0>
__global__ __launch_bounds__(64 * (WN * WM * KS + LW), 1) void product_tile_kernel(dsa_product_args p, int tiles_m, int tiles_n) {
    using T = Tile<NT, MT, WN, WM, KS, STAGES, LW>;
    __shared__ __attribute__((aligned(1024))) char smem[T::LDS_BYTES];
    const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)smem;
    int m, n;
    place(along_xcds(blockIdx.x, tiles_m * tiles_n), tiles_m, tiles_n, m, n);
    product_tile<OUT, NT, MT, WN, WM, KS, STAGES, LW>(p, lds, m * T::TM, n * T::TN);
}

// Tiles of 256 by 256 for whole rounds of them, and those left over cut in two: a last
// round of 128 columns by 256 rows, of two thirds the time.
using Whole = Tile<8, 4, 2, 4, 1, 2>;
using Half = Tile<4, 4, 2, 4, 1, 2>;
template <typename OUT>
__global__ __launch_bounds__(Whole::THREADS, 1) void product_mixed_kernel(dsa_product_args p, int tiles_m, int tiles_n, int whole) {
    static_assert(Whole::THREADS == Half::THREADS && Whole::TM == Half::TM && Whole::TN == 2 * Half::TN, "two halves");
    __shared__ __attribute__((aligned(1024))) char smem[Whole::LDS_BYTES];
    static_assert(Half::LDS_BYTES <= Whole::LDS_BYTES, "one LDS");
    const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)smem;
    int m, n;
    if ((int)blockIdx.x < whole) {
        place(along_xcds(blockIdx.x, whole), tiles_m, tiles_n, m, n);
        product_tile<OUT, 8, 4, 2, 4, 1, 2>(p, lds, m * Whole::TM, n * Whole::TN);
    } else {
        const uint32_t i = along_xcds(blockIdx.x - whole, 2 * (tiles_m * tiles_n - whole));
        place(whole + i / 2, tiles_m, tiles_n, m, n);
        const int n0 = n * Whole::TN + (int)(i & 1) * Half::TN;
        if (n0 < p.N) product_tile<OUT, 4, 4, 2, 4, 1, 2>(p, lds, m * Half::TM, n0);
    }
}

template <typename OUT, int NT, int MT, int WN, int WM, int KS, int STAGES, int LW = 0>
void launch_tile(const dsa_product_args& p, hipStream_t stream) {
    using T = Tile<NT, MT, WN, WM, KS, STAGES, LW>;
    const int tiles_m = (p.M + T::TM - 1) / T::TM, tiles_n = (p.N + T::TN - 1) / T::TN;
    hipLaunchKernelGGL((product_tile_kernel<OUT, NT, MT, WN, WM, KS, STAGES, LW>), dim3(tiles_m * tiles_n), dim3(T::THREADS), 0, stream, p,
                       tiles_m, tiles_n);
}

template <typename OUT>
void launch_mixed(const dsa_product_args& p, int cus, hipStream_t stream) {
    const int tiles_m = (p.M + Whole::TM - 1) / Whole::TM, tiles_n = (p.N + Whole::TN - 1) / Whole::TN;
    const int tiles = tiles_m * tiles_n, whole = tiles / cus * cus;
    hipLaunchKernelGGL((product_mixed_kernel<OUT>), dim3(whole + 2 * (tiles - whole)), dim3(Whole::THREADS), 0, stream, p, tiles_m,
                       tiles_n, whole);
}

// Tiles by the size of the call: a call takes as many rounds as its tiles fill CUs, and
// a round its steps, and a start and end of about 2 us.  What a step takes was measured
// on 17 to 256 workgroups with K from 1536 to 16384, and, where the stages of two
// workgroups fit a CU's LDS, on 264 to 512.  The smallest split K over their waves, so
// that there are fewer steps; from 64 by 64 on waves of their own load: without them
// (columns, rows, K) 128x64 took 31.6 us for 26.2 at (2112, 512, 7168), 128x96 32.6 for
// 27.9 at (2112, 1000, 7168), 128x128 37.5 for 33.4.  The 32-bit outputs' widened codes
// need more registers than a third wave a SIMD leaves, so that from 128x96 on they load
// themselves.  Whole calls, us (rows, columns, K; columns x rows of a tile; weights from
// HBM; two runs differ by up to 10 % below 10 us):
//   8, 2112, 7168      16x16 7.8 (four stages 7.8), 16x32 8.5, 32x16 9.1, 32x32 9.7, 64x32 15
//   5, 4300, 7168      16x16 12.2 (9.9), 32x16 9.3 (three stages 10.7), 32x32 10.1, 64x32 15
//   32, 2112, 16384    16x16 21.1 (17.5), 16x32 16.0, 32x16 16.9, 32x32 21.0, 64x32 32
//   64, 2112, 7168     16x16 17.1 (14.1), 32x32 11.3, 64x32 15.9, 64x64 20, 128x64 28
//   204, 623, 5648     16x16 10.6 (8.3), 16x32 13.0, 32x16 13.6 (10.9), 32x32 8.8, 64x32 13.2
//   16, 24576, 1536    64x32 12.3, 64x64 10.8, 128x32 9.7, 128x64 9.9, 128x96 10.3
//   448, 2112, 7168    64x32 29.5, 64x64 19.5, 128x32 22.1, 128x64 26.2, 128x96 29.3
//   512, 4096, 7168    64x64 33.2, 128x64 26.9, 128x96 27.3, 128x128 34.7
//   1000, 2112, 7168   64x64 39, 128x64 41, 128x96 27.8, 128x128 33.7, 128x160 35.1
//   2000, 2112, 7168   64x64 63, 128x96 51.5, 128x128 59, 128x160 39.2, 128x256 59
//   1000, 7168, 16384  64x64 203, 128x96 167, 128x128 140, 128x160 155, 128x256 135, 256x256 136
//   8192, 2112, 7168   128x96 159, 128x128 163, 128x160 154, 128x256 172, 256x256 151
// Over 170 calls, most of them drawn from these ranges, the chosen tile took 1.5 % longer
// than the best one (at most 22 %, where few rows meet 24576 by 14240 or 16384).  32-bit
// outputs go by the same step times, though theirs are longer, up to 1.9 times in the
// larger tiles: over 270 calls that choice took 1.3 % longer than the best (at most 20 %,
// the same ones), and 1.2 % with their own medians in place of these.
struct Variant {
    int columns, rows, blocks;  // of a tile, and blocks of K a step
    float step, both;           // us a step, alone on a CU and beside another; 0: does not fit beside another
    void (*launch[3])(const dsa_product_args&, hipStream_t);  // by type
};
#define DSA_TILE(...) {launch_tile<__bf16, __VA_ARGS__>, launch_tile<f16, __VA_ARGS__>, launch_tile<float, __VA_ARGS__>}
const Variant kVariants[] = {
    {16, 16, 4, 0.29f, 0.00f, DSA_TILE(1, 1, 1, 1, 4, 5)},  {16, 16, 4, 0.31f, 0.58f, DSA_TILE(1, 1, 1, 1, 4, 4)},
    {16, 32, 4, 0.45f, 0.00f, DSA_TILE(1, 2, 1, 1, 4, 4)},  {32, 16, 4, 0.49f, 0.00f, DSA_TILE(1, 1, 2, 1, 4, 4)},
    {32, 16, 4, 0.53f, 0.70f, DSA_TILE(1, 1, 2, 1, 4, 3)},  {32, 32, 4, 0.60f, 0.00f, DSA_TILE(1, 2, 2, 1, 4, 4)},  {64, 32, 2, 0.48f, 0.00f, DSA_TILE(1, 2, 4, 1, 2, 4)},
    {64, 64, 1, 0.31f, 0.50f, DSA_TILE(2, 2, 2, 2, 1, 4, 4)},   {128, 32, 1, 0.36f, 0.00f, DSA_TILE(2, 2, 4, 1, 1, 4, 4)},
    {128, 64, 1, 0.45f, 0.00f, DSA_TILE(2, 4, 4, 1, 1, 4, 4)},  {128, 96, 1, 0.47f, 0.00f, {launch_tile<__bf16, 2, 3, 4, 2, 1, 4, 4>, launch_tile<f16, 2, 3, 4, 2, 1, 4, 4>, launch_tile<float, 2, 3, 4, 2, 1, 4>}},
    {128, 128, 1, 0.55f, 0.00f, {launch_tile<__bf16, 2, 4, 4, 2, 1, 4, 4>, launch_tile<f16, 2, 4, 4, 2, 1, 4, 4>, launch_tile<float, 2, 4, 4, 2, 1, 4>}},
    {128, 160, 1, 0.61f, 0.00f, {launch_tile<__bf16, 4, 5, 2, 2, 1, 4, 4>, launch_tile<f16, 4, 5, 2, 2, 1, 4, 4>, nullptr}},
    {128, 256, 1, 1.02f, 0.00f, DSA_TILE(4, 4, 2, 4, 1, 2)},
};
// A grid's threads, up to 768 a tile, are counted in 32 bits.  The 128 by 256 tiles of the
// largest output, 2^37 with at most 2^24 rows and columns, always fit.
constexpr int64_t kMaxTiles = 5 << 20;
static_assert(((int64_t)1 << 37) / (128 * 256) + (1 << 24) / 128 + (1 << 24) / 256 + 1 <= kMaxTiles, "one tile is left");
constexpr float kWholeStep = 1.70f, kHalfStep = 1.02f;  // of the mixed kernel

constexpr int kTiles = sizeof kVariants / sizeof kVariants[0];  // and the mixed kernel's number

}  // namespace

// The number of the tiles that a call takes: kVariants', or kTiles.
int product_tile(const dsa_product_args& p, int cus) {
    const int blocks = (p.K + kBlock - 1) / kBlock;
    int best = -1;
    float least = 0.f;
    for (int i = 0; i < kTiles; ++i) {
        const Variant& v = kVariants[i];
        const int64_t tiles = (int64_t)((p.M + v.rows - 1) / v.rows) * ((p.N + v.columns - 1) / v.columns);
        if (tiles > kMaxTiles || !v.launch[p.dtype]) continue;
        const bool pairs = v.both > 0.f && tiles > cus;
        const int64_t fit = pairs ? 2 * cus : cus;
        const float time = (float)((tiles + fit - 1) / fit) *
                           (2.f + (pairs ? v.both : v.step) * (float)((blocks + v.blocks - 1) / v.blocks));
        if (best < 0 || time < least) best = i, least = time;
    }
    if (p.dtype != DSA_F32) {  // the widened codes of 32-bit outputs would need more registers
        const int64_t tiles = (int64_t)((p.M + 255) / 256) * ((p.N + 255) / 256), rest = tiles % cus;
        const float time = (float)(tiles / cus) * (2.f + kWholeStep * (float)blocks) +
                           (float)((2 * rest + cus - 1) / cus) * (2.f + kHalfStep * (float)blocks);
        if (time < least) best = kTiles;
    }
    return best;
}

unsigned product_tiles(int dtype) {
    unsigned set = dtype == DSA_F32 ? 0u : 1u << kTiles;
    for (int i = 0; i < kTiles; ++i) set |= kVariants[i].launch[dtype] ? 1u << i : 0u;
    return set;
}

int launch_product(const dsa_product_args& p, int cus, hipStream_t stream) {
    const int tile = product_tile(p, cus);
    if (tile < kTiles) kVariants[tile].launch[p.dtype](p, stream);
    else if (p.dtype == DSA_BF16) launch_mixed<__bf16>(p, cus, stream);
    else launch_mixed<f16>(p, cus, stream);
    return (int)hipGetLastError();
}

}  // namespace dsa
