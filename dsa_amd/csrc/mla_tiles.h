// Device pieces the MLA attention kernels share: LDS access, gathers from HBM
// straight into LDS, the swizzled tile layout and cross-lane reductions.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace dsa {
namespace {

typedef __attribute__((__vector_size__(8 * sizeof(__bf16)))) __bf16 bf16x8;
typedef __attribute__((__vector_size__(4 * sizeof(__bf16)))) __bf16 bf16x4;
typedef __attribute__((__vector_size__(4 * sizeof(short)))) short i16x4;
typedef __attribute__((__vector_size__(4 * sizeof(float)))) float f32x4;
typedef __attribute__((__vector_size__(16 * sizeof(float)))) float f32x16;
typedef __attribute__((__vector_size__(4 * sizeof(int)))) int i32x4;

// ---------------------------------------------------------------- LDS access
template <typename T>
__device__ __forceinline__ T lds_load(uint32_t addr) {
    return *reinterpret_cast<__attribute__((address_space(3))) T*>(addr);
}
template <typename T>
__device__ __forceinline__ void lds_store(uint32_t addr, T v) {
    *reinterpret_cast<__attribute__((address_space(3))) T*>(addr) = v;
}
__device__ __forceinline__ void lds_or(uint32_t addr, uint32_t v) {
    __hip_atomic_fetch_or(reinterpret_cast<__attribute__((address_space(3))) uint32_t*>(addr), v, __ATOMIC_RELAXED,
                          __HIP_MEMORY_SCOPE_WORKGROUP);
}
// ds_read_b64_tr_b16: within each 16-lane group, lane l supplies the address
// of 4 consecutive bf16 of "row" l/4, columns 4*(l%4)..+3 of a 4x16 block;
// lane n receives column n of that block (rows 0..3).
__device__ __forceinline__ bf16x4 lds_load_tr(uint32_t addr) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4bf16(
        reinterpret_cast<__attribute__((address_space(3))) bf16x4*>(addr));
}

// Barrier that makes this workgroup's LDS writes visible without waiting for
// outstanding global loads (the gather ring stays in flight across it).
__device__ __forceinline__ void lds_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// s_waitcnt vmcnt(N), other counters untouched (gfx9 encoding).
template <int N>
__device__ __forceinline__ void wait_vmcnt() {
    static_assert(N >= 0 && N < 64, "vmcnt range");
    __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (15 << 8));
}

typedef int rsrc_t __attribute__((ext_vector_type(4)));

// Raw buffer resource over [base, base + bytes) (gfx9 descriptor: no stride,
// 32-bit byte offsets).  All fields are wave-uniform.
__device__ __forceinline__ rsrc_t make_rsrc(const void* base, uint32_t bytes) {
    const uint64_t a = reinterpret_cast<uint64_t>(base);
    rsrc_t r;
    r[0] = __builtin_amdgcn_readfirstlane((int)(uint32_t)a);
    r[1] = __builtin_amdgcn_readfirstlane((int)((a >> 32) & 0xffff));
    r[2] = __builtin_amdgcn_readfirstlane((int)bytes);
    r[3] = 0x00020000;
    return r;
}

// Gathers write LDS with buffer_load_dwordx4 ... lds: lane l's 16 bytes land
// at m0 + 16*l.  They are issued as inline asm so the compiler does not
// serialise later LDS reads behind them; completion is tracked with
// Ring::wait_tile().  m0 and the buffer descriptors are wave-uniform by
// construction.
//
// One kv row: a 1 KiB descriptor at the row's 64-bit address (so the kv
// pool has no 4 GiB limit), lane l loading bytes (16*l) ^ xor16 of it.  The
// XOR is part of the asm so no per-row lane offset is ever kept live.
__device__ __forceinline__ rsrc_t row_rsrc(const char* base, uint32_t row) {
    const uint64_t a = reinterpret_cast<uint64_t>(base) + ((uint64_t)row << 10);
    rsrc_t r;
    r[0] = (int)(uint32_t)a;
    r[1] = (int)((a >> 32) & 0xffff);
    r[2] = 1024;
    r[3] = 0x00020000;
    return r;
}
__device__ __forceinline__ void gather_row(uint32_t lds_base, rsrc_t rsrc, uint32_t lane16, uint32_t xor16) {
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
    uint32_t voff;
    asm volatile(
        "v_xor_b32 %0, %1, %2\n\t"
        "s_mov_b32 m0, %3\n\t"
        "buffer_load_dwordx4 %0, %4, 0 offen lds"
        : "=&v"(voff)
        : "s"(xor16), "v"(lane16), "s"(__builtin_amdgcn_readfirstlane(lds_base)), "s"(rsrc)
        : "memory", "m0");
#pragma clang diagnostic pop
}
// Arbitrary per-lane byte offsets (rope rows: 8 rows per instruction).
__device__ __forceinline__ void gather_lanes(uint32_t lds_base, rsrc_t rsrc, uint32_t voff) {
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
    asm volatile(
        "s_mov_b32 m0, %0\n\t"
        "buffer_load_dwordx4 %1, %2, 0 offen lds"
        :
        : "s"(__builtin_amdgcn_readfirstlane(lds_base)), "v"(voff), "s"(rsrc)
        : "memory", "m0");
#pragma clang diagnostic pop
}

// 16-byte chunk swizzles.  A kv row occupies 1024 contiguous LDS bytes (64
// chunks); logical chunk c of tile row r lives at physical chunk c ^ sw_kv(r)
// (only the low 4 bits move).  sw_kv is a permutation of 0..15 whose values
// differ in bits [3:2] within every group of 4 consecutive rows and in bits
// [3:1] within every group of 8.  LDS has 64 banks (a 256-byte period); a
// ds_read_b128 serves 16 lanes per pass, four quads of lanes: quad q of a
// half-wave (lanes 4q..4q+3) joins pass parity(popcount(q)).  With the QK
// chunk assignment of each variant and the transposed PV reads, every pass
// touches 16 distinct bank groups (rocprofv3 SQ_LDS_BANK_CONFLICT reads 0).
// A rope row occupies 128 bytes (8 chunks): physical = c ^ sw_rope(r).
__device__ __forceinline__ int sw_kv(int r) {
    return ((r & 3) << 2) | (((r >> 2) & 1) << 1) | ((r >> 3) & 1);  // uses r mod 16
}
__device__ __forceinline__ int sw_rope(int r) { return (r >> 1) & 7; }

// QK k-order of the specialised-wave and ping-pong kernels: k-step ks (32 of
// the 512 latent dims) takes logical chunks 4 ks .. 4 ks + 3, lane group g
// holding chunk 4 ks + qk_lane_chunk(g), so that one Q fragment load reads a
// whole 64-byte piece of each of its 16 head rows (16 lines per instruction)
// where chunk 16 g + ks reads 16 bytes of 64 lines.  The permutation
// [0, 3, 1, 2] keeps the low two chunk bits of groups 0 and 1 (and of 2 and
// 3) in the same class {0, 3} or {1, 2}, which is what keeps the K reads of
// one ds_read_b128 pass on 16 distinct bank groups under sw_kv (with g in
// place of qk_lane_chunk(g) a pass would meet 2-way conflicts).  Measured:
// C2 -2.4 %, C5 -0.9 %; the column-split kernel (C4 +0.7 % with it) and the
// narrow kernel keep chunk 16 g + ks.
__device__ __forceinline__ int qk_lane_chunk(int g) { return (0x9C >> (2 * g)) & 3; }

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// Cross-lane reductions over lanes l and l ^ 32 (l ^ 16) with the gfx950
// VALU lane swaps instead of an LDS permute.  v_permlane32_swap on two copies
// of v leaves (v[l], v[l ^ 32]) in the pair on every lane; v_permlane16_swap
// does the same for l ^ 16.
__device__ __forceinline__ float max_xor32(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float max_xor16(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_xor32(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float sum_xor16(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Byte offset of k-group g's 16-byte P chunk of head h (within a 64-head
// buffer).  With 64-byte heads, the lanes of one ds_read_b128 / ds_write_b128
// pass (four quads of a half-wave, chosen by popcount parity) would meet 4
// heads apart on the same banks; XOR-ing the chunk with f(h / 4) =
// {0, 2, 3, 1} gives every pass 16 distinct bank groups.
__device__ __forceinline__ uint32_t pp_pchunk(int h, int g) {
    return (uint32_t)(h * 64 + 16 * (g ^ ((0x78 >> (2 * ((h >> 2) & 3))) & 3)));
}

}  // namespace
}  // namespace dsa
