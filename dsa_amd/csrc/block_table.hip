// Block tables and slot maps from request lengths
// (include/dsa_mi355x_cache.h: dsa_extend_block_table).  No reference
// counterpart: the reference takes a contiguous cache (dsa/api.py:30-33).
//
// Bound by its launch (64 sequences 4.1 us, 48 prompts of up to 2047 tokens 4.3 in a
// captured row of calls; 3.6 and 4.6 as traced): a step of 64 sequences moves about a kilobyte, one of
// 98,304 tokens 1.2 MB.  So it is one launch with no second pass: every
// workgroup scans the sequences' token and block counts itself (at most 4096 of
// them, kept in LDS) and then writes its share of the tokens and of the taken
// blocks, each found by a binary search in the scan.  A token reads at most one
// entry that was there before the call, the sequence's partly filled block,
// which the call does not write: entries that are new are taken from
// free_blocks instead, so no workgroup waits for another.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/dsa_mi355x_cache.h"
#include "kernels.h"

namespace dsa {
namespace {

constexpr int kMax = 0x7fffffff;

// Sums of counts, held at 2^31 - 1 (associative, since no count is negative).
__device__ __forceinline__ int sat_add(int a, int b) { return (int)min((uint32_t)a + (uint32_t)b, (uint32_t)kMax); }

// Blocks that hold n tokens.
__device__ __forceinline__ int blocks_of(int n, int block) { return n / block + (n % block != 0); }

struct Counts {
    int tokens, blocks;
};

__device__ __forceinline__ int held_of(const TableParams& p, int b) { return max(p.lengths[b], 0); }

__device__ __forceinline__ Counts counts_of(const TableParams& p, int b) {
    const int held = held_of(p, b), add = max(p.new_tokens[b], 0);
    const int first = min(blocks_of(held, p.block_size), p.max_blocks);
    const int last = min(blocks_of(sat_add(held, add), p.block_size), p.max_blocks);
    return Counts{add, last - first};
}

// The last b with scan[b] <= i (scan[0] = 0 <= i).
__device__ __forceinline__ int owner(const int* scan, int n, int i) {
    int low = 0, high = n;  // scan[low] <= i, high: first known > i or n
    while (high - low > 1) {
        const int mid = (low + high) >> 1;
        if (scan[mid] <= i) low = mid;
        else high = mid;
    }
    return low;
}

template <int kThreads>
__global__ __launch_bounds__(kThreads) void extend_table_kernel(TableParams p) {
    extern __shared__ int smem[];
    int* tokens = smem;                // [B]: tokens of the sequences before
    int* blocks = smem + p.B;          // [B]: blocks taken by them
    int* held = smem + 2 * p.B;        // [B]: tokens that a sequence holds
    __shared__ int wave_tokens[kThreads / 64], wave_blocks[kThreads / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;

    // Exclusive scans: thread t sums its run of sequences, the wave and then the
    // workgroup scan the sums.
    const int run = (p.B + kThreads - 1) / kThreads;
    const int b0 = min(tid * run, p.B), b1 = min(b0 + run, p.B);
    int st = 0, sb = 0;
    for (int b = b0; b < b1; ++b) {
        const Counts c = counts_of(p, b);
        st = sat_add(st, c.tokens);
        sb = sat_add(sb, c.blocks);
    }
    int it = st, ib = sb;
    for (int d = 1; d < 64; d <<= 1) {
        const int ut = __shfl_up(it, d), ub = __shfl_up(ib, d);
        if (lane >= d) {
            it = sat_add(it, ut);
            ib = sat_add(ib, ub);
        }
    }
    if (lane == 63) {
        wave_tokens[wave] = it;
        wave_blocks[wave] = ib;
    }
    int bt = __shfl_up(it, 1), bb = __shfl_up(ib, 1);
    if (lane == 0) bt = bb = 0;
    __syncthreads();
    int total_tokens = 0, total_blocks = 0;
    for (int w = 0; w < kThreads / 64; ++w) {
        if (w == wave) {
            bt = sat_add(bt, total_tokens);
            bb = sat_add(bb, total_blocks);
        }
        total_tokens = sat_add(total_tokens, wave_tokens[w]);
        total_blocks = sat_add(total_blocks, wave_blocks[w]);
    }
    for (int b = b0; b < b1; ++b) {
        const Counts c = counts_of(p, b);
        tokens[b] = bt;
        blocks[b] = bb;
        held[b] = held_of(p, b);
        if (blockIdx.x == 0) {
            p.starts[b] = bt;
            p.totals[b] = sat_add(held_of(p, b), c.tokens);
        }
        bt = sat_add(bt, c.tokens);
        bb = sat_add(bb, c.blocks);
    }
    if (blockIdx.x == 0 && tid == 0) {
        p.starts[p.B] = total_tokens;
        p.used[0] = total_blocks;
    }
    __syncthreads();

    const int stride = gridDim.x * kThreads;
    for (int64_t k = blockIdx.x * kThreads + tid; k < total_blocks; k += stride) {
        const int b = owner(blocks, p.B, (int)k);
        const int column = blocks_of(held[b], p.block_size) + ((int)k - blocks[b]);
        p.block_table[(int64_t)b * p.max_blocks + column] = k < p.num_free ? p.free_blocks[k] : -1;
    }
    for (int64_t i = blockIdx.x * kThreads + tid; i < p.max_tokens; i += stride) {
        int slot = -1, position = 0;
        if (i < total_tokens) {
            const int b = owner(tokens, p.B, (int)i);
            const int first = blocks_of(held[b], p.block_size);
            position = sat_add(held[b], (int)i - tokens[b]);
            const int column = position / p.block_size;
            int entry = -1;
            if (column < p.max_blocks) {
                if (column < first) {
                    entry = p.block_table[(int64_t)b * p.max_blocks + column];
                } else {
                    const int64_t k = (int64_t)blocks[b] + (column - first);
                    entry = k < p.num_free ? p.free_blocks[k] : -1;
                }
            }
            const int64_t row = (int64_t)entry * p.block_size + position % p.block_size;
            slot = entry >= 0 && row <= kMax ? (int)row : -1;
        }
        p.slots[i] = slot;
        p.positions[i] = position;
    }
}

}  // namespace

int launch_extend_table(const TableParams& p, hipStream_t stream) {
    // One token a thread (four, with a quarter of the scans: 48 prompts 5.4 us for
    // 4.3 in a captured row of calls); more threads where each has sequences to
    // sum (2000 sequences 7.7 us with 512, 10.8 with 256; 64 4.15 and 4.06).
    const int threads = p.B > 512 ? 512 : 256;
    const int64_t want = ((int64_t)p.max_tokens + threads - 1) / threads;
    const int grid = want < 1 ? 1 : want < 512 ? (int)want : 512;
    auto* kernel = threads == 512 ? extend_table_kernel<512> : extend_table_kernel<256>;
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(threads), 3 * p.B * sizeof(int), stream, p);
    return (int)hipGetLastError();
}

}  // namespace dsa
