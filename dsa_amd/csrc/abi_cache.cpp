// C ABI of the paged cache's operators (include/dsa_mi355x_cache.h): argument
// checks and launches.  Like abi.cpp it never throws and never allocates.
#include <hip/hip_runtime_api.h>

#include <cmath>
#include <cstdarg>
#include <cstdint>
#include <cstdio>

#include "../../include/dsa_mi355x_cache.h"
#include "kernels.h"

namespace {

int fail(int code, const char* fmt, ...) {
    char text[400];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(text, sizeof text, fmt, ap);
    va_end(ap);
    return dsa::set_error(code, "%s", text);
}

int finish(int rc, const char* what) {
    if (rc) return fail(rc, "%s: %s (hipError_t %d)", what, hipGetErrorString((hipError_t)rc), rc);
    return dsa::set_error(0, "%s", "");
}

bool aligned(const void* p, unsigned bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }

}  // namespace

extern "C" {

int dsa_extend_block_table(int32_t* block_table, const int32_t* lengths, const int32_t* new_tokens,
                           const int32_t* free_blocks, int32_t* slots, int32_t* positions, int32_t* starts,
                           int32_t* totals, int32_t* used, int B, int max_blocks, int block_size, int num_free,
                           int max_tokens, void* stream) {
    if (!block_table || !lengths || !new_tokens || !starts || !totals || !used || (num_free > 0 && !free_blocks) ||
        (max_tokens > 0 && (!slots || !positions)))
        return fail(-1, "NULL pointer argument");
    if (B <= 0 || B > DSA_TABLE_MAX_SEQUENCES || max_blocks <= 0 || block_size <= 0 || num_free < 0 || max_tokens < 0)
        return fail(-1, "B must be in [1, %d], max_blocks and block_size positive, num_free and max_tokens not negative "
                    "(got %d, %d, %d, %d, %d)", DSA_TABLE_MAX_SEQUENCES, B, max_blocks, block_size, num_free, max_tokens);
    const dsa::TableParams p{block_table, lengths, new_tokens, free_blocks, slots, positions, starts, totals, used,
                             B, max_blocks, block_size, num_free, max_tokens};
    return finish(dsa::launch_extend_table(p, static_cast<hipStream_t>(stream)), "block table launch");
}

int dsa_rotary(const dsa_rotary_args* a, void* stream) {
    if (!a || !a->x || !a->out || !a->positions || !a->frequencies) return fail(-1, "NULL pointer argument");
    if (a->dtype != DSA_BF16 && a->dtype != DSA_F16 && a->dtype != DSA_F32)
        return fail(-1, "unknown dtype %d", a->dtype);
    if (a->groups <= 0 || a->tokens <= 0 || a->heads <= 0 || a->width <= 0 || a->groups > (int64_t)1 << 31 ||
        a->tokens > (int64_t)1 << 31 || a->groups * a->tokens > ((int64_t)1 << 40) / a->heads)
        return fail(-1, "groups, tokens, heads and width must be positive, and groups * tokens * heads at most 2^40");
    if (a->dim < 2 || a->dim % 2 || a->dim > DSA_ROTARY_MAX_DIM || a->start < 0 || a->start > a->width - a->dim)
        return fail(-1, "dim must be even, in [2, %d], and start .. start + dim lie inside the head (got dim %d, start %d, "
                    "width %d)", DSA_ROTARY_MAX_DIM, a->dim, a->start, a->width);
    if (!std::isfinite(a->magnitude)) return fail(-1, "magnitude must be finite");
    const unsigned size = a->dtype == DSA_F32 ? 4 : 2;
    if (!aligned(a->x, size) || !aligned(a->out, size) || !aligned(a->frequencies, 8) ||
        !aligned(a->positions, a->positions_64 ? 8 : 4))
        return fail(-1, "pointers must be aligned to their elements");
    return finish(dsa::launch_rotary(*a, static_cast<hipStream_t>(stream)), "rotary launch");
}

int dsa_write_kv_rows(const dsa_write_args* a, void* stream) {
    if (!a || !a->kv || !a->k_rope || !a->slots || !a->cache || (a->frequencies && !a->positions))
        return fail(-1, "NULL pointer argument");
    if (a->kv_format != DSA_KV_BF16 && a->kv_format != DSA_KV_FP8) return fail(-1, "unknown kv_format %d", a->kv_format);
    if ((a->kv_format == DSA_KV_BF16) != (a->rope_cache != nullptr))
        return fail(-1, "rope_cache goes with bf16 rows, and only with them");
    if (a->tokens <= 0 || a->cache_rows <= 0) return fail(-1, "tokens and cache_rows must be positive");
    if (a->kv_stride % 8 || a->rope_stride % 2 || !aligned(a->kv, 16) || !aligned(a->k_rope, 4) ||
        !aligned(a->cache, 16) || !aligned(a->rope_cache, 4) || !aligned(a->slots, 4) || !aligned(a->frequencies, 8) ||
        !aligned(a->positions, a->positions_64 ? 8 : 4))
        return fail(-1, "kv and cache must be 16-byte, k_rope and rope_cache 4-byte aligned, kv_stride a multiple of 8, "
                    "rope_stride of 2");
    if (!std::isfinite(a->magnitude)) return fail(-1, "magnitude must be finite");
    return finish(dsa::launch_write_rows(*a, static_cast<hipStream_t>(stream)), "cache row launch");
}

}  // extern "C"
