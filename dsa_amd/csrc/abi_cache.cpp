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

int ceil_div(int a, int b) { return (a + b - 1) / b; }

// Whether a sequence's query rows fill blocks of their own to seven eighths: then
// those take the prefix too; emptier ones leave it to blocks of all sequences'
// rows (stacked).  Measured with 16 sequences of bf16 rows, paged, 8192 rows
// shared and up to 512 of their own, stacked and not: 16 rows a sequence 39 and
// 44 us, 96 64 and 68, 112 70 and 70, 144 80 and 84, 224 106 and 99, 240 112 and
// 99; with 1024 shared rows and up to 2048 own ones within 3 us of each other.
bool fills_blocks(int64_t rows) {
    const int64_t blocks = (rows + dsa::kSharedRows - 1) / dsa::kSharedRows;
    return rows * 8 >= blocks * dsa::kSharedRows * 7;
}

struct SharedPlan {
    bool stacked;
    int prefix_items, seq_blocks, items, workgroups;
    int own_rows;  // of a piece of a sequence's own rows
    int64_t ends_bytes, part_rows, bytes;
};

int64_t round_256(int64_t n) { return (n + 255) / 256 * 256; }

int shared_plan(const dsa_shared_args* a, SharedPlan* plan) {
    if (!a) return fail(-1, "args is NULL");
    if (a->B <= 0 || a->SQ <= 0 || a->H <= 0 || a->L <= 0)
        return fail(-1, "B, SQ, H, L must be positive (got %d, %d, %d, %d)", a->B, a->SQ, a->H, a->L);
    if (a->H % 16) return fail(-1, "H must be a multiple of 16 (got %d)", a->H);
    if (a->L >= 1 << 25) return fail(-1, "L must be below 33554432 (got %d)", a->L);
    if (a->prefix < 0 || a->prefix > a->L) return fail(-1, "prefix must be in [0, L = %d] (got %d)", a->L, a->prefix);
    if (a->num_cus < 0 || a->num_cus > 1 << 12) return fail(-1, "num_cus must be 0 .. 4096");
    const int64_t seq_rows = (int64_t)a->SQ * a->H, rows = seq_rows * a->B;
    if (seq_rows > 1 << 30 || rows > 1 << 30) return fail(-1, "B * SQ * H must be at most 2^30");
    plan->stacked = a->prefix > 0 && a->B > 1 && !fills_blocks(seq_rows);
    plan->seq_blocks = (int)((seq_rows + dsa::kSharedRows - 1) / dsa::kSharedRows);
    plan->prefix_items = plan->stacked ? (int)((rows + dsa::kSharedRows - 1) / dsa::kSharedRows) : 0;
    const int64_t items = plan->prefix_items + (int64_t)a->B * plan->seq_blocks;
    plan->items = (int)items;
    plan->workgroups = a->num_cus;
    if (plan->workgroups == 0) {
        int device = 0, cus = 0;
        int rc = (int)hipGetDevice(&device);
        if (!rc) rc = (int)hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, device);
        if (rc) return fail(rc, "device query: %s", hipGetErrorString((hipError_t)rc));
        plan->workgroups = cus;
    }
    // Pieces: every cut of an item's tiles starts a new one; a stacked call keeps
    // all of them, another only those of cut items, two at most a workgroup.
    plan->own_rows = (int)(seq_rows < dsa::kSharedRows ? seq_rows : dsa::kSharedRows);
    const int64_t own_items = items - plan->prefix_items, wgs = plan->workgroups;
    plan->part_rows = plan->stacked ? (plan->prefix_items + wgs) * dsa::kSharedRows + (own_items + wgs) * plan->own_rows
                                    : 2 * wgs * plan->own_rows;
    // The kernel's sums: an item of at most 2^20 + 2 tiles costs less than 2^26, at
    // most 2^26 items times 2^12 workgroups stay in 64 bits.
    static_assert(dsa::kSharedMaxCost + (dsa::kSharedPieceCost >> 20) < 1 << 6, "an item's cost");
    plan->ends_bytes = round_256(8 * items);
    plan->bytes = plan->ends_bytes + plan->part_rows * (512 + 2) * 4;
    return 0;
}

bool aligned(const void* p, unsigned bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }

// dsa_fwd_shared, or with a tree dsa_fwd_tree.
int run_shared(const dsa_shared_args* a, const int32_t* tree, int words, void* stream) {
    SharedPlan plan;
    if (const int rc = shared_plan(a, &plan)) return rc;
    if (a->kv_format != DSA_KV_BF16 && a->kv_format != DSA_KV_FP8) return fail(-1, "unknown kv_format %d", a->kv_format);
    const bool fp8 = a->kv_format == DSA_KV_FP8;
    if (!a->q || !a->kv || !a->q_rope || (!fp8 && !a->k_rope) || !a->lengths || !a->out || !a->out_max || !a->out_sum ||
        !a->workspace)
        return fail(-1, "NULL pointer argument");
    if (!aligned(a->q, 16) || !aligned(a->kv, 16) || !aligned(a->q_rope, 16) || (!fp8 && !aligned(a->k_rope, 16)) ||
        !aligned(a->out, 16) || !aligned(a->lengths, 4) || !aligned(a->block_table, 4) || !aligned(a->out_max, 4) ||
        !aligned(a->out_sum, 4) || !aligned(a->workspace, 256))
        return fail(-1, "tensors must be 16-byte (lengths, block_table, max and sum 4-byte, workspace 256-byte) aligned");
    if (!(a->scale >= 0.f) || !std::isfinite(a->scale)) return fail(-1, "scale must be a positive finite number, or 0");
    if (a->block_table) {
        if (a->block_size <= 0 || a->max_blocks <= 0 || a->num_blocks <= 0 ||
            (int64_t)a->block_size * a->max_blocks != a->L)
            return fail(-1, "paged kv: block_size, max_blocks and num_blocks must be positive, L = max_blocks * block_size");
        if ((int64_t)a->num_blocks * a->block_size >= 1 << 25)
            return fail(-1, "paged kv: num_blocks * block_size must be below 33554432");
    }
    if (a->workspace_bytes < plan.bytes)
        return fail(-1, "workspace of %lld bytes is below the %lld needed", (long long)a->workspace_bytes,
                    (long long)plan.bytes);
    dsa::SharedParams p{};
    p.q = a->q;
    p.kv = static_cast<const char*>(a->kv);
    p.q_rope = a->q_rope;
    p.k_rope = a->k_rope;
    p.lengths = a->lengths;
    p.block_table = a->block_table;
    p.tree = tree;
    p.words = words;
    p.out = a->out;
    p.out_max = a->out_max;
    p.out_sum = a->out_sum;
    char* ws = static_cast<char*>(a->workspace);
    p.ends = reinterpret_cast<int2*>(ws);
    p.part_o = reinterpret_cast<float*>(ws + plan.ends_bytes);
    p.part_m = p.part_o + plan.part_rows * 512;
    p.part_l = p.part_m + plan.part_rows;
    p.B = a->B;
    p.SQ = a->SQ;
    p.H = a->H;
    p.L = a->L;
    p.prefix = a->prefix;
    p.block_size = a->block_size;
    p.max_blocks = a->max_blocks;
    p.num_blocks = a->num_blocks;
    // d in (2^s, 2^(s+1)]: ceil(2^(32+s) / d) d < 2^(32+s) + d, so the quotient is exact for keys below 2^31
    if (a->block_table && a->block_size > 1) {
        while ((int64_t)2 << p.block_shift < a->block_size) ++p.block_shift;
        const uint64_t num = (uint64_t)1 << (32 + p.block_shift), d = (uint64_t)a->block_size;
        p.block_magic = (uint32_t)((num + d - 1) / d);
    }
    p.kv_fp8 = fp8;
    p.scale = a->scale == 0.f ? 1.f / 24.f : a->scale;
    p.scale_log2 = p.scale * 1.4426950408889634f;
    p.stacked = plan.stacked;
    p.prefix_items = plan.prefix_items;
    p.seq_blocks = plan.seq_blocks;
    p.items = plan.items;
    p.workgroups = plan.workgroups;
    p.own_rows = plan.own_rows;
    return finish(dsa::launch_shared(p, static_cast<hipStream_t>(stream)), "shared attention launch");
}

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
    if ((int64_t)a->heads * a->width > (int64_t)1 << 31) return fail(-1, "heads * width must be at most 2^31");
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

int64_t dsa_fwd_shared_ws_bytes(const dsa_shared_args* a) {
    SharedPlan plan;
    const int rc = shared_plan(a, &plan);
    if (rc) return rc < 0 ? rc : -rc;
    dsa::set_error(0, "%s", "");
    return plan.bytes;
}

int dsa_fwd_shared(const dsa_shared_args* a, void* stream) { return run_shared(a, nullptr, 0, stream); }

int64_t dsa_fwd_tree_ws_bytes(const dsa_tree_args* a) { return dsa_fwd_shared_ws_bytes(a ? &a->shared : nullptr); }

int dsa_fwd_tree(const dsa_tree_args* a, void* stream) {
    if (!a || !a->tree) return fail(-1, "NULL pointer argument");
    if (a->words <= 0 || a->words > DSA_TREE_MAX_WORDS)
        return fail(-1, "words must be in [1, %d] (got %d)", DSA_TREE_MAX_WORDS, a->words);
    if (!aligned(a->tree, 4)) return fail(-1, "tree must be 4-byte aligned");
    return run_shared(&a->shared, a->tree, a->words, stream);
}

int dsa_draft_tree(const int32_t* parents, const int32_t* lengths, int32_t* tree, int32_t* positions, int B, int SQ,
                   void* stream) {
    if (!parents || !lengths || !tree || !positions) return fail(-1, "NULL pointer argument");
    if (B <= 0 || B > 1 << 20 || SQ <= 0 || SQ > 32 * DSA_TREE_MAX_WORDS)
        return fail(-1, "B must be in [1, 2^20] and SQ in [1, %d] (got %d, %d)", 32 * DSA_TREE_MAX_WORDS, B, SQ);
    if (!aligned(parents, 4) || !aligned(lengths, 4) || !aligned(tree, 4) || !aligned(positions, 4))
        return fail(-1, "pointers must be aligned to their elements");
    return finish(dsa::launch_draft_tree(parents, lengths, tree, positions, B, SQ, static_cast<hipStream_t>(stream)),
                  "draft tree launch");
}

}  // extern "C"
