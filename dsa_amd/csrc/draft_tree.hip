// Ancestors and positions of drafted tokens (include/dsa_mi355x_cache.h:
// dsa_draft_tree).  No reference counterpart: the reference attends to given
// indices (dsa/api.py:76-132).
//
// A workgroup a sequence, a thread a token: it goes up its own line, which ends as
// every parent's number is below its child's.  Twice: to see whether the line
// reaches the sequence, and, from the highest token down, to set its bits, a word
// after the other.  Bound by the launch and by the longest line, one LDS read a
// generation (3 sequences of 7 tokens 1.9 to 3.8 us, 32 of 33 and 16 of 60 5.0; the
// attention behind them 28 to 1570).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kernels.h"

namespace dsa {
namespace {

constexpr int kThreads = 256, kMaxTokens = 32 * DSA_TREE_MAX_WORDS;

__global__ __launch_bounds__(kThreads) void draft_tree_kernel(const int32_t* parents, const int32_t* lengths, int32_t* tree,
                                                              int32_t* positions, int SQ, int words) {
    __shared__ int32_t up[kMaxTokens];
    const int64_t first = (int64_t)blockIdx.x * SQ;
    for (int t = threadIdx.x; t < SQ; t += kThreads) up[t] = parents[first + t];
    const int length = max(lengths[blockIdx.x], 0);
    __syncthreads();
    for (int t = threadIdx.x; t < SQ; t += kThreads) {
        int at = t, depth = -1;
        for (;;) {
            const int parent = up[at];
            ++depth;
            if (parent < 0 || parent >= at) {
                if (parent != -1) depth = -1;  // no line to the sequence
                break;
            }
            at = parent;
        }
        positions[first + t] = depth < 0 ? 0 : (int)min((int64_t)length + depth, (int64_t)0x7fffffff);
        at = depth < 0 ? -1 : t;
        for (int w = words - 1; w >= 0; --w) {
            uint32_t bits = 0;
            while (at >= 32 * w) {  // -1: below every word
                bits |= 1u << (at & 31);
                at = up[at];
            }
            tree[(first + t) * words + w] = (int32_t)bits;
        }
    }
}

}  // namespace

int launch_draft_tree(const int32_t* parents, const int32_t* lengths, int32_t* tree, int32_t* positions, int B, int SQ,
                      hipStream_t stream) {
    hipLaunchKernelGGL(draft_tree_kernel, dim3(B), dim3(kThreads), 0, stream, parents, lengths, tree, positions, SQ,
                       (SQ + 31) / 32);
    return (int)hipGetLastError();
}

}  // namespace dsa
