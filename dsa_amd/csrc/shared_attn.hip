// Dense MLA attention of a batch whose sequences share their first rows
// (include/dsa_mi355x_cache.h: dsa_fwd_shared).  No reference counterpart: the
// reference attends to given indices (dsa/api.py:76-132).
//
// Every head of every sequence reads the same key rows in the prefix, so the
// (token, head) pairs of the whole batch are rows of one product there: a block
// of 64 such rows takes each tile of 32 key rows once from memory, whatever
// sequences the rows belong to.  Three launches:
//
//   plan   tiles of every item (kernels.h: SharedParams) from the lengths, summed
//   main   the tiles of all items, cut evenly over the workgroups: one pass over
//          a piece's keys with the running maximum and sum of the softmax
//   merge  rows of cut items joined (FP32), rows without keys filled in
//
// Tiles are laid out and swizzled in LDS as in the sparse kernels (mla_tiles.h).
#include <hip/hip_runtime.h>
#include <float.h>
#include <stdint.h>

#include "kernels.h"
#include "mla_tiles.h"

namespace dsa {
namespace {

constexpr float kLn2 = 0.69314718055994531f;
constexpr int kRows = kSharedRows, kKeys = kSharedKeys;
constexpr int kFp8Row = 656, kFp8ScaleOff = 512, kFp8RopeOff = 528;
// Fewest tiles a workgroup is given.
constexpr int kMinTiles = 2;

__device__ __forceinline__ int ceil_div(int a, int b) { return (a + b - 1) / b; }

// One block of query rows and its keys: tiles of the prefix (sequence 0) and
// then of the own rows.
struct Item {
    int row0, rows;     // first (token, head) row, and how many (multiples of 16)
    int seq;            // sequence of the own rows
    int first, second;  // tiles over the prefix, over the own rows
};

__device__ __forceinline__ int seen_by(const SharedParams& p, int token) {
    return min(max(p.lengths[token], 0), p.L);
}

// Rows and sequence of item i, without its tiles.
__device__ __forceinline__ Item item_rows(const SharedParams& p, int i) {
    Item it;
    if (i < p.prefix_items) {
        it.row0 = i * kRows;
        it.rows = min(kRows, p.B * p.SQ * p.H - it.row0);
        it.seq = 0;
    } else {
        const int j = i - p.prefix_items, b = j / p.seq_blocks, k = j - b * p.seq_blocks;
        const int seq_rows = p.SQ * p.H;
        it.row0 = b * seq_rows + k * kRows;
        it.rows = min(kRows, seq_rows - k * kRows);
        it.seq = b;
    }
    return it;
}

// Tiles of an item whose longest query sees `most` rows.
__device__ __forceinline__ void item_tiles(const SharedParams& p, int i, int most, Item& it) {
    it.first = p.stacked && i >= p.prefix_items ? 0 : ceil_div(min(most, p.prefix), kKeys);
    it.second = i < p.prefix_items ? 0 : ceil_div(max(most - p.prefix, 0), kKeys);
}

__device__ __forceinline__ int most_seen(const SharedParams& p, const Item& it) {
    int most = 0;
    for (int t = it.row0 / p.H; t <= (it.row0 + it.rows - 1) / p.H; ++t) most = max(most, seen_by(p, t));
    return most;
}

__device__ __forceinline__ int groups_of(const SharedParams& p, int total) {
    return max(1, min(p.workgroups, total / kMinTiles));
}

// The workgroup whose share [w * total / groups, (w + 1) * total / groups) holds tile t.
__device__ __forceinline__ int group_at(int t, int total, int groups) {
    return (int)(((int64_t)(t + 1) * groups + total - 1) / total) - 1;
}

// Slot of the piece of item i that workgroup w computes; `head`: it starts at the item's first tile.
__device__ __forceinline__ int64_t slot_of(const SharedParams& p, int i, int w, bool head) {
    return p.stacked ? (int64_t)i + w : 2 * (int64_t)w + (head ? 1 : 0);
}

// ------------------------------------------------------------------ plan
constexpr int kPlanThreads = 1024;
__global__ __launch_bounds__(kPlanThreads) void shared_plan_kernel(SharedParams p) {
    __shared__ int sums[kPlanThreads / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int base = 0;
    for (int i0 = 0; i0 < p.items; i0 += kPlanThreads) {
        const int i = i0 + tid;
        int n = 0;
        if (i < p.items) {
            Item it = item_rows(p, i);
            item_tiles(p, i, most_seen(p, it), it);
            n = it.first + it.second;
        }
        int scan = n;
        for (int d = 1; d < 64; d <<= 1) {
            const int u = __shfl_up(scan, d);
            if (lane >= d) scan += u;
        }
        if (lane == 63) sums[wave] = scan;
        __syncthreads();
        int before = 0, all = 0;
        for (int w = 0; w < kPlanThreads / 64; ++w) {
            if (w < wave) before += sums[w];
            all += sums[w];
        }
        if (i < p.items) p.tiles[i] = base + before + scan - n;
        base += all;
        __syncthreads();
    }
    if (tid == 0) p.tiles[p.items] = base;
}

// ------------------------------------------------------------------ main
constexpr int kThreads = 256;

// Row of the cache behind key `key` of sequence `seq`, or -1 (masked).
__device__ __forceinline__ int64_t cache_row(const SharedParams& p, int seq, int key) {
    if (p.block_table == nullptr) return (int64_t)seq * p.L + key;
    const int blk = p.block_table[(int64_t)seq * p.max_blocks + key / p.block_size];
    if ((uint32_t)blk >= (uint32_t)p.num_blocks) return -1;
    return (int64_t)blk * p.block_size + key % p.block_size;
}

__global__ __launch_bounds__(kThreads) void shared_main_kernel(SharedParams p) {
    __shared__ __attribute__((aligned(1024))) char smem[kKeys * 1152];
    __shared__ uint32_t valid_rows;
    const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)smem;
    const int lane = threadIdx.x & 63, g = lane >> 4, n16 = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

    const int total = p.tiles[p.items], groups = groups_of(p, total);
    const int w = blockIdx.x;
    if (w >= groups) return;
    int t0 = (int)((int64_t)w * total / groups);
    const int t1 = (int)((int64_t)(w + 1) * total / groups);
    if (t0 >= t1) return;
    int low = 0, high = p.items;  // the item that holds tile t0: tiles[low] <= t0 < tiles[low + 1]
    while (high - low > 1) {
        const int mid = (low + high) >> 1;
        if (p.tiles[mid] <= t0) low = mid;
        else high = mid;
    }
    for (int i = low; t0 < t1; ++i) {
        const int begin = p.tiles[i], end = p.tiles[i + 1];
        if (end <= t0) continue;
        Item it = item_rows(p, i);
        item_tiles(p, i, most_seen(p, it), it);
        const int a = t0 - begin, b = min(t1, end) - begin;  // the item's tiles [a, b)
        const bool live = 16 * wave < it.rows;
        const int row = it.row0 + 16 * wave;
        const int seen = live ? seen_by(p, row / p.H) : 0;
        bf16x8 qf[18];
        if (live) {
            const uint16_t* q = p.q + (int64_t)(row + n16) * 512 + 8 * qk_lane_chunk(g);
            for (int ks = 0; ks < 16; ++ks) qf[ks] = *reinterpret_cast<const bf16x8*>(q + 32 * ks);
            const uint16_t* r = p.q_rope + (int64_t)(row + n16) * 64 + 8 * g;
            qf[16] = *reinterpret_cast<const bf16x8*>(r);
            qf[17] = *reinterpret_cast<const bf16x8*>(r + 32);
        }
        f32x4 o[32];
        for (int cb = 0; cb < 32; ++cb) o[cb] = f32x4{0.f, 0.f, 0.f, 0.f};
        float m = -FLT_MAX, l = 0.f;
        for (int t = a; t < b; ++t) {
            const bool shared = t < it.first;
            const int key0 = shared ? t * kKeys : p.prefix + (t - it.first) * kKeys;
            const int limit = shared ? min(seen, p.prefix) : seen;
            const int key_end = shared ? p.prefix : p.L;
            __syncthreads();
            if (threadIdx.x < kKeys) {
                const int key = key0 + (int)threadIdx.x;
                const bool ok = key < key_end && cache_row(p, shared ? 0 : it.seq, key) >= 0;
                const uint64_t v = __ballot(ok);
                if (threadIdx.x == 0) valid_rows = (uint32_t)v;
            }
            for (int c = threadIdx.x; c < kKeys * 72; c += kThreads) {
                const int r = c / 72, ch = c % 72, key = key0 + r;
                const int64_t src = key < key_end ? cache_row(p, shared ? 0 : it.seq, key) : -1;
                bf16x8 v = {};
                if (src >= 0 && p.kv_fp8) {
                    const char* raw = p.kv + src * kFp8Row;
                    if (ch >= 64) {
                        v = *reinterpret_cast<const bf16x8*>(raw + kFp8RopeOff + 16 * (ch - 64));
                    } else {
                        const float sc = *reinterpret_cast<const float*>(raw + kFp8ScaleOff + 4 * (ch >> 4));
                        const int2 codes = *reinterpret_cast<const int2*>(raw + 8 * ch);
                        for (int d = 0; d < 2; ++d) {
                            const int code = d ? codes.y : codes.x;
                            const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(code, false);
                            const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(code, true);
                            v[4 * d + 0] = (__bf16)(lo[0] * sc);
                            v[4 * d + 1] = (__bf16)(lo[1] * sc);
                            v[4 * d + 2] = (__bf16)(hi[0] * sc);
                            v[4 * d + 3] = (__bf16)(hi[1] * sc);
                        }
                    }
                } else if (src >= 0) {
                    v = ch < 64 ? *reinterpret_cast<const bf16x8*>(p.kv + src * 1024 + 16 * ch)
                                : *reinterpret_cast<const bf16x8*>(p.k_rope + src * 64 + 8 * (ch - 64));
                }
                const uint32_t dst = ch < 64 ? r * 1024 + ((ch ^ sw_kv(r)) << 4)
                                             : kKeys * 1024 + r * 128 + (((ch - 64) ^ sw_rope(r)) << 4);
                lds_store<bf16x8>(lds + dst, v);
            }
            __syncthreads();
            if (!live) continue;
            // rows this wave's query sees: bit r is tile row r
            const int n = min(max(limit - key0, 0), kKeys);
            const uint32_t mask = valid_rows & (n == kKeys ? 0xffffffffu : (1u << n) - 1);
            if (mask == 0) continue;
            f32x4 s[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
            for (int ks = 0; ks < 18; ++ks)
                for (int sub = 0; sub < 2; ++sub) {
                    const int r = 16 * sub + n16;
                    const uint32_t at = ks < 16 ? r * 1024 + (((4 * ks + qk_lane_chunk(g)) ^ sw_kv(r)) << 4)
                                                : kKeys * 1024 + r * 128 + (((4 * (ks - 16) + g) ^ sw_rope(r)) << 4);
                    s[sub] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(lds_load<bf16x8>(lds + at), qf[ks], s[sub], 0, 0, 0);
                }
            // lane: rows 4 g + r (j < 4) and 16 + 4 g + r of head n16
            float x[8], top = m;
            uint32_t keep[4] = {0, 0, 0, 0};
            for (int j = 0; j < 8; ++j) {
                const bool on = mask >> (4 * g + (j & 3) + 16 * (j >> 2)) & 1;
                x[j] = on ? s[j >> 2][j & 3] * p.scale_log2 : -INFINITY;
                top = fmaxf(top, x[j]);
                keep[j >> 1] |= on ? 0xffffu << (16 * (j & 1)) : 0u;
            }
            top = max_xor32(max_xor16(top));
            const float alpha = fast_exp2(m - top);
            m = top;
            float sum = 0.f;
            bf16x8 pk;
            for (int j = 0; j < 8; ++j) {
                const float e = fast_exp2(x[j] - top);
                sum += e;
                pk[j] = (__bf16)e;
            }
            l = l * alpha + sum;
            const int vr = 4 * g + (n16 >> 2);
            for (int cb = 0; cb < 32; ++cb) {
                const uint32_t at = lds + vr * 1024 + (((2 * cb + ((n16 & 3) >> 1)) ^ sw_kv(vr)) << 4) + 8 * (n16 & 1);
                const bf16x4 v0 = lds_load_tr(at), v1 = lds_load_tr(at + 16 * 1024);
                // masked rows have weight 0, and are cleared so that no NaN or infinity in them counts
                i32x4 v = __builtin_bit_cast(i32x4, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
                for (int d = 0; d < 4; ++d) v[d] &= (int)keep[d];
                o[cb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, v), pk, o[cb] * alpha, 0, 0, 0);
            }
        }
        l = sum_xor32(sum_xor16(l));
        if (live) {
            const bool whole = !p.stacked && a == 0 && b == end - begin;
            if (whole) {
                const float inv = l == 0.f ? 0.f : 1.f / l;
                uint16_t* out = p.out + (int64_t)(row + n16) * 512 + 4 * g;
                for (int cb = 0; cb < 32; ++cb) {
                    bf16x4 v;
                    for (int r = 0; r < 4; ++r) v[r] = (__bf16)(o[cb][r] * inv);
                    *reinterpret_cast<bf16x4*>(out + 16 * cb) = v;
                }
                if (g == 0) {
                    p.out_max[row + n16] = l == 0.f ? -INFINITY : m * kLn2;
                    p.out_sum[row + n16] = l;
                }
            } else {
                const int64_t prow = slot_of(p, i, w, a == 0) * kRows + 16 * wave + n16;
                for (int cb = 0; cb < 32; ++cb)
                    *reinterpret_cast<f32x4*>(p.part_o + prow * 512 + 16 * cb + 4 * g) = o[cb];
                if (g == 0) {
                    p.part_m[prow] = m;
                    p.part_l[prow] = l;
                }
            }
        }
        t0 = min(t1, end);
    }
}

// ------------------------------------------------------------------ merge
// One workgroup a row pair; thread t of a row's 128 owns columns 4 t .. 4 t + 3.
__global__ __launch_bounds__(kThreads) void shared_merge_kernel(SharedParams p) {
    const int rows = p.B * p.SQ * p.H;
    const int row = blockIdx.x * 2 + (threadIdx.x >> 7), col = (threadIdx.x & 127) * 4;
    if (row >= rows) return;
    const int total = p.tiles[p.items], groups = groups_of(p, total);
    const int seq_rows = p.SQ * p.H, b = row / seq_rows, in_seq = row - b * seq_rows;
    float m = -FLT_MAX, l = 0.f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int part = p.stacked ? 0 : 1; part < 2; ++part) {
        const int i = part == 0 ? row / kRows : p.prefix_items + b * p.seq_blocks + in_seq / kRows;
        const int hl = part == 0 ? row % kRows : in_seq % kRows;
        const int begin = p.tiles[i], end = p.tiles[i + 1];
        if (begin == end) continue;
        const int w0 = group_at(begin, total, groups), w1 = group_at(end - 1, total, groups);
        if (!p.stacked && w0 == w1) return;  // a whole item: written by the main kernel
        for (int w = w0; w <= w1; ++w) {
            const int64_t prow = slot_of(p, i, w, w == w0) * kRows + hl;
            const float ms = p.part_m[prow], ls = p.part_l[prow];
            const f32x4 u = *reinterpret_cast<const f32x4*>(p.part_o + prow * 512 + col);
            const float top = fmaxf(m, ms), keep = fast_exp2(m - top), add = fast_exp2(ms - top);
            l = l * keep + ls * add;
            acc = acc * keep + u * add;
            m = top;
        }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    bf16x4 v;
    for (int r = 0; r < 4; ++r) v[r] = (__bf16)(acc[r] * inv);
    *reinterpret_cast<bf16x4*>(p.out + (int64_t)row * 512 + col) = v;
    if (col == 0) {
        p.out_max[row] = l == 0.f ? -INFINITY : m * kLn2;
        p.out_sum[row] = l;
    }
}

}  // namespace

int launch_shared(const SharedParams& p, hipStream_t stream) {
    hipLaunchKernelGGL(shared_plan_kernel, dim3(1), dim3(kPlanThreads), 0, stream, p);
    int rc = (int)hipGetLastError();
    if (rc) return rc;
    hipLaunchKernelGGL(shared_main_kernel, dim3(p.workgroups), dim3(kThreads), 0, stream, p);
    rc = (int)hipGetLastError();
    if (rc) return rc;
    const int rows = p.B * p.SQ * p.H;
    hipLaunchKernelGGL(shared_merge_kernel, dim3((rows + 1) / 2), dim3(kThreads), 0, stream, p);
    return (int)hipGetLastError();
}

}  // namespace dsa
