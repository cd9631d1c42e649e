// Dense MLA attention of a batch whose sequences share their first rows
// (include/dsa_mi355x_cache.h: dsa_fwd_shared), or ends with a tree of drafted
// tokens (dsa_fwd_tree).  No reference counterpart: the reference attends to given
// indices (dsa/api.py:76-132).
//
// Every head of every sequence reads the same key rows in the prefix, so the
// (token, head) pairs of the whole batch are rows of one product there: a block
// of up to 128 such rows takes each tile of 32 key rows once from memory,
// whatever sequences the rows belong to.  Two launches:
//
//   main   the tiles of all items (kernels.h: SharedParams), cut by cost evenly
//          over the workgroups, one a CU: one pass over a piece's keys with the sum
//          of the softmax
//   merge  rows of cut items joined (FP32), rows without keys filled in
//
// With 128 heads bound by the matrix cores (54 % of cycles busy, 1.17 to 1.22
// PFLOP/s over 4 prompts of 512 tokens behind 8192 rows: 2.1 us a tile of 128 rows,
// 1.6 at the rate of a large matrix product), with 16 to 64 rows of their own by HBM
// (256 sequences of 4096 bf16 rows 235 us, 5.1 TB/s), and for a decode step by what
// surrounds a piece's tiles: 4 us until
// its share is found, 5 to 7 until its first tile and Q are there, 2 to 6 for its
// rows, 4 to 16 for the merge.
//
// With a tree a token sees all of its sequence's rows, and of the rows behind them those
// whose bits it has: the tiles that hold such rows are masked by its words, all others
// are as above (16 sequences of 60 tokens, 128 heads, behind 6144 to 8192 rows 1530 us,
// 1.07 PFLOP/s; 32 of 33, 16 heads, fp8, 2048 rows shared, 391 us: 528 query rows a
// sequence are four blocks of 128 and one of 16, which takes half a large one's time).
//
// Tiles are laid out and swizzled in LDS as in the sparse kernels (mla_tiles.h).
#include <hip/hip_runtime.h>
#include <float.h>
#include <stdint.h>
#include <type_traits>

#include "kernels.h"
#include "mla_tiles.h"

namespace dsa {
namespace {

typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

constexpr int kKeys = kSharedKeys;
constexpr int kFp8Row = 656, kFp8ScaleOff = 512, kFp8RopeOff = 528;

__device__ __forceinline__ int ceil_div(int a, int b) { return (a + b - 1) / b; }

// Added to a row's sum for each tile while it has keys but no score above -inf.  Its
// maximum counts as -FLT_MAX there, so that beside any finite score this is scaled
// to 0.  2^20 tiles of 2^12 pieces, eight lanes a row: less than 2^-64 in all, and a
// sum of real weights, whose greatest is 1, stays above.
constexpr float kOnlyMinusInf = 0x1p-100f;

// A row's sum and maximum as they are returned (`top`: the largest product, before
// the scale), and what its weighted rows are to be multiplied by.  Sum 0: no key, all
// zeros and -inf.  Scores that are all -inf, or one of +inf or NaN among them: the
// sum is NaN, by its formula, and the maximum NaN too unless an infinity is it.
struct Returned {
    float max, sum, inv;
};
__device__ __forceinline__ Returned returned(float top, float sum, float scale) {
    if (sum == 0.f) return Returned{-INFINITY, 0.f, 0.f};
    if (sum <= 0x1p-64f) return Returned{-INFINITY, NAN, NAN};
    if (sum != sum && top != INFINITY) return Returned{NAN, sum, sum};
    return Returned{top * scale, sum, 1.f / sum};
}

// The kernel's arguments, read from memory here and now.  As ordinary arguments
// the compiler holds all of them in scalar registers from the start, spills
// those into vector registers, and these, in the loop, into memory -- where the
// wait for a reload is a full wait for the gathers too.  What the loop needs
// (Hot) is passed along, the rest is read where it is used.
typedef const __attribute__((address_space(4))) SharedParams* ArgsPtr;
__device__ __forceinline__ ArgsPtr args_now() {
    uint64_t a = (uint64_t)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(a));
    return (ArgsPtr)a;
}

// One block of query rows and its keys: tiles of the prefix (sequence 0) and
// then of the own rows.
struct Item {
    int row0, rows;     // first (token, head) row, and how many (multiples of 16)
    int seq;            // sequence of the own rows
    int first, second;  // tiles over the prefix, over the own rows
};

// Rows that a token sees: all of the first so many.  With a tree that is its
// sequence's length, and some of the 32 * words rows behind it.
template <bool TREE>
__device__ __forceinline__ int seen_by(ArgsPtr p, int token) {
    return min(max(p->lengths[TREE ? token / p->SQ : token], 0), p->L);
}

// Rows and sequence of item i, without its tiles.
__device__ __forceinline__ Item item_rows(ArgsPtr p, int i) {
    Item it;
    if (i < p->prefix_items) {
        it.row0 = i * kSharedRows;
        it.rows = min(kSharedRows, p->B * p->SQ * p->H - it.row0);
        it.seq = 0;
    } else {
        const int j = i - p->prefix_items, b = j / p->seq_blocks, k = j - b * p->seq_blocks;
        const int seq_rows = p->SQ * p->H;
        it.row0 = b * seq_rows + k * kSharedRows;
        it.rows = min(kSharedRows, seq_rows - k * kSharedRows);
        it.seq = b;
    }
    return it;
}

// Tiles of an item whose longest query sees `most` rows.  Tiles start at
// multiples of 32 keys: one that the prefix ends in is there twice, for either side.
__device__ __forceinline__ void item_tiles(ArgsPtr p, int i, int most, Item& it) {
    it.first = p->stacked && i >= p->prefix_items ? 0 : ceil_div(min(most, p->prefix), kKeys);
    it.second = i < p->prefix_items || most <= p->prefix ? 0 : ceil_div(most, kKeys) - p->prefix / kKeys;
}

// What an item costs, in tenths of a microsecond on a full chip: each tile, and
// once the start and end of a piece (Q, the first tile's latency, the stores).
// Set from the kernel's own clock readings on 64 to 256 sequences of their own rows,
// in blocks of 64.  Whole calls of 256 sequences, a workgroup each (2048 to 4096 rows,
// us a tile; contiguous, blocks, pages): 16 query rows 1.65, 1.60, 1.61 for bf16 and
// 1.06, 1.29, 1.49 for fp8, 64 rows 1.56, 1.60, 2.55 and 1.48, 1.84, 1.90, 128 rows
// 2.37, 2.44, 2.87 and 2.54, 2.53, 3.29.  The items of a call differ in rows only, so
// what counts is the ratio of 128 rows to 16: 1.4 here, 1.5 measured, fp8 1.9 and 2.0;
// of pages 1.8 and 2.2, for which no costs of their own have been tried.
struct Cost {
    int tile, piece;
};
__device__ __forceinline__ Cost cost_of(int rows, int fp8) {
    if (rows > 64) return Cost{fp8 ? 26 : 21, 120};
    if (rows > 32) return Cost{fp8 ? 16 : 20, 105};
    return Cost{fp8 ? 14 : 15, 85};
}
static_assert(kSharedMaxCost >= 27 && kSharedPieceCost >= 2 * 27 + 120, "the host's bound on an item's cost");
// Least cost a workgroup is given, more than a tile's.  At 20, 30, 40 and 60: 3
// sequences of 16 heads behind 500 rows 21.4, 21.3, 22.0 and 22.9 us, 16 of them behind
// 600 29.6, 27.9, 27.8 and 27.7, 8 of 1000 rows 23.2, 22.5, 23.3 and 23.8, one query of
// 300 18.3, 19.1, 19.7 and 20.9, of 2000 21.0, 20.7, 20.0 and 21.0 (in a graph of calls).
constexpr int kMinShare = 30;

// Workgroup w computes the tiles that start in its share [w * total / groups,
// (w + 1) * total / groups) of the summed costs; an item that starts at cost
// `begin` has its tile t at begin + piece + t * tile.
struct Shares {
    int64_t each;
    uint32_t rest, groups;
    __device__ __forceinline__ Shares(int64_t total, uint32_t n) : groups(n) {  // a division of 64 bits only where it needs one
        each = total >> 32 ? total / n : (uint32_t)total / n;
        rest = (uint32_t)(total - each * n);
    }
    __device__ __forceinline__ int64_t start(uint32_t w) const { return w * each + w * rest / groups; }  // groups <= 2^12
};

// What an item's queries see (least and most), and with that its tiles and cost.
struct Look {
    Item it;
    int low, high, cost;
    Cost each;
};
__device__ __forceinline__ void look_at(ArgsPtr p, int i, int low, int high, Look& k) {
    k.it = item_rows(p, i);
    item_tiles(p, i, high, k.it);
    k.low = low;
    k.high = high;
    k.each = cost_of(k.it.rows, p->kv_fp8);
    const int tiles = k.it.first + k.it.second;
    k.cost = tiles == 0 ? 0 : k.each.piece + tiles * k.each.tile;
}
template <bool TREE>
__device__ __forceinline__ void look_at(ArgsPtr p, int i, Look& k) {
    const Item it = item_rows(p, i);
    // a block has eight times 16 rows at most, each of one token: as many lengths, read together
    const int first = it.row0 / p->H, last = (it.row0 + it.rows - 1) / p->H;
    int seen[kSharedRows / 16], most = 0, least = p->L;
#pragma unroll
    for (int n = 0; n < kSharedRows / 16; ++n) {
        const int token = min(first + n, last);
        seen[n] = p->lengths[TREE ? token / p->SQ : token];
    }
#pragma unroll
    for (int n = 0; n < kSharedRows / 16; ++n) {
        const int v = min(max(seen[n], 0), p->L);
        most = max(most, v);
        least = min(least, v);
    }
    if constexpr (TREE) most = min(most + 32 * p->words, p->L);
    look_at(p, i, least, most, k);
}

// First partial row of the piece of item i that workgroup w computes; `head`: it
// starts at the item's first tile.  A stacked call keeps all its pieces, item i's
// behind i - 1's; another only those of cut items, of which a workgroup has two at
// most.  A sequence's own piece has own_rows rows.
__device__ __forceinline__ int64_t piece_row(ArgsPtr p, int i, int w, bool head) {
    if (!p->stacked) return (2 * (int64_t)w + (head ? 1 : 0)) * p->own_rows;
    if (i < p->prefix_items) return ((int64_t)i + w) * kSharedRows;
    return ((int64_t)p->prefix_items + p->workgroups) * kSharedRows + ((int64_t)(i - p->prefix_items) + w) * p->own_rows;
}

// ------------------------------------------------------------------ main
// Eight waves in two groups of four (waves w and w + 4 share a SIMD), half a
// tile apart, so that on every SIMD one wave's softmax (VALU) runs beside the
// other's MFMAs.  A group's turn at a tile is
//
//   QK  S^T = K Q^T and its weights: a wave one block of 16 query rows (Q in
//       registers) and all 32 keys; P (bf16) to the group's LDS buffer
//   PV  O^T += V^T P^T: a wave 128 of the 512 columns (O in registers) and
//       four blocks of 16 rows
//
// with a workgroup barrier at the start of each half.
//
//   up to 64 rows (narrow): both groups own the same rows and take the tiles in
//       turn; their sums are joined at the end.
//       half u:       group u % 2 QK (u)    the other PV (u - 1)
//   up to 128 rows (wide): group k owns rows 64 k ..; both take every tile.
//       half 2 t:     group 0 QK (t)        group 1 PV (t - 1)
//       half 2 t + 1: group 0 PV (t)        group 1 QK (t)
//
// P is formed against a reference maximum, a row's from its first tile, and a
// piece whose scores pass it by 64 (log2 units) is computed once more against
// the exact one, so O is never rescaled in the loop.  The maximum is taken off
// the products and the difference scaled: scaled first, a product of 2^31 and its
// rounded maximum would differ by more than weights of 32 bits hold.
//
// A query row sees keys [0, seen) only, and rows behind a bad block entry are
// masked: their scores become -inf, their weights 0 (see clear_specials).
constexpr int kPPThreads = 512;
constexpr float kRestartLog2 = 64.0f;
constexpr int kPoisonBytes = kSharedRows / 16 * 512 / 8;

// Each wave brings in four rows of every tile.  bf16 rows are gathered straight
// into a ring of four tiles; fp8 rows land as stored (656 bytes) in one of two
// raw tiles, and the wave expands them into a ring of three.
template <bool FP8>
struct PPLds {
    static constexpr int NSTAGE = FP8 ? 3 : 4;
    static constexpr int KV_BYTES = kKeys * 1024, STAGE_BYTES = kKeys * 1152;
    static constexpr int RAW_OFF = NSTAGE * STAGE_BYTES, RAW_BYTES = FP8 ? kKeys * kFp8Row : 0;
    // P of one group, 64 rows x 32 bf16 in the k order of the PV operand (pp_pchunk)
    static constexpr int P_OFF = RAW_OFF + 2 * RAW_BYTES, P_GROUP = 64 * 64;
    static constexpr int FLAG_OFF = P_OFF + 2 * P_GROUP;  // a second pass is needed
    static constexpr int BAD_OFF = FLAG_OFF + 4;          // some block entry of the piece lies outside the pool
    static constexpr int PLAN_OFF = FLAG_OFF + 16;        // the workgroup's first item: number, begin, low, high
    static constexpr int MASK_OFF = PLAN_OFF + 32;        // of either group: the keys of a tile that its four row blocks see
    static constexpr int POISON_OFF = MASK_OFF + 32;      // columns of each row block to become NaN, and whether there is one
    static constexpr int LDS_BYTES = POISON_OFF + kPoisonBytes + 16;
    static constexpr int ML_OFF = P_OFF;  // [3][128] floats, at the end: l, reference and maximum
    static_assert(LDS_BYTES <= 160 * 1024, "LDS budget");
    __device__ static uint32_t stage(uint32_t lds, int u) { return lds + (uint32_t)(u % NSTAGE) * STAGE_BYTES; }
    __device__ static uint32_t raw(uint32_t lds, int u) { return lds + RAW_OFF + (uint32_t)(u % 2) * RAW_BYTES; }
};

// What the main kernel's loop needs of them.
struct Hot {
    const char* kv;
    const char* k_rope;
    const int32_t* block_table;
    int L, prefix, max_blocks, block_size, num_blocks;
    uint32_t block_magic;
    int block_shift;
    float scale_log2;
};

// One tile of a piece: its first key (a multiple of 32), the keys [low, high)
// of it that count, and the sequence they are looked up in.
struct Tile {
    int key0, low, high, seq;
};
struct Piece {
    Item it;
    int a, nt;      // first tile of the item, and how many
    int seen_low, seen_high;  // all rows of the block see the rows below the one, none a row from the other on
};
__device__ __forceinline__ Tile tile_at(const Hot& p, const Piece& c, int u) {
    const int t = c.a + u;
    const bool shared = t < c.it.first;
    Tile k;
    k.key0 = (shared ? t : p.prefix / kKeys + (t - c.it.first)) * kKeys;
    k.low = shared ? 0 : p.prefix;
    k.high = shared ? p.prefix : p.L;
    k.seq = shared ? 0 : c.it.seq;
    return k;
}

// key / block_size, without a division (keys are below 2^25).
__device__ __forceinline__ int block_of(const Hot& p, int key) {
    return p.block_size == 1 ? key : (int)(__umulhi((uint32_t)key, p.block_magic) >> p.block_shift);
}

// 16 bytes a lane, OFFSET + off on, straight into LDS: lane l at m0 + OFFSET + 16 l.
template <int OFFSET>
__device__ __forceinline__ void gather_at(uint32_t lds_base, rsrc_t rsrc, uint32_t off) {
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
    asm volatile(
        "s_mov_b32 m0, %0\n\t"
        "buffer_load_dwordx4 %1, %2, 0 offen offset:%3 lds"
        :
        : "s"(__builtin_amdgcn_readfirstlane(lds_base)), "v"(off), "s"(rsrc), "n"(OFFSET)
        : "memory", "m0");
#pragma clang diagnostic pop
}

// How a tile's rows lie: in one sequence (rows), in blocks of a multiple of
// four rows (blocks), in any blocks (pages).
enum { kRows = 0, kBlocks = 1, kPages = 2 };

// The block table's entry of a key of sequence seq: a scalar load.
__device__ __forceinline__ int table_entry(const Hot& p, int seq, int key) {
    const auto* t = (const __attribute__((address_space(4))) int32_t*)(uint64_t)p.block_table;
    return t[(int64_t)seq * p.max_blocks + block_of(p, key)];
}

// Gathers of one tile by one wave: its rows 4 wave .. 4 wave + 3.  bf16: an
// instruction a row (1 KiB), and one for their rotary parts (kPages: one a row);
// fp8: three instructions, or one a row.  The four rows follow each other unless
// LAYOUT is kPages, so that they have one descriptor (rows past a sequence's end
// are out of its range and read as zeros); of a tile behind the piece (u >= nt)
// nothing is read, but the instructions are the same, so that they can be counted
// on.
//
// They are issued together, behind the first LDS reads of QK or PV: the queue in
// front of the texture path holds that many, and in the chain of MFMAs each
// would cost about 60 clocks (a chain of 36 with its LDS reads: 764 clocks,
// 772 with four gathers in front, 1000 with the four between its steps).
//
// Blocks and pages: all the wave needs of the block table it reads by scalar
// loads, a tile ahead (fetch).
template <bool FP8, int LAYOUT>
struct Gathers {
    static constexpr int N = LAYOUT == kRows ? 0 : LAYOUT == kBlocks ? 1 : 4;  // entries of the four rows
    static constexpr int LOADS = FP8 ? (LAYOUT == kPages ? 4 : 3) : (LAYOUT == kPages ? 8 : 5);
    int64_t first;               // row that the four start with, from the cache's start
    int rows;                    // how many of them can be read
    int row[N == 4 ? 4 : 1];     // kPages: each row, from the cache's start, or -1
    int tile;
    int entry[N == 0 ? 1 : N];   // of the tile prepared next

    __device__ __forceinline__ void fetch(const Hot& p, const Piece& c, int u, int wave) {
        if constexpr (N > 0) {
            const Tile k = tile_at(p, c, u);
#pragma unroll
            for (int i = 0; i < N; ++i) entry[i] = table_entry(p, k.seq, min(k.key0 + 4 * wave + i, p.L - 1));
        }
    }
    // Tile u's gathers, from its entries.  A wave that meets an entry outside the
    // pool, of rows that some query sees, says so at `bad`.
    __device__ __forceinline__ void prepare(const Hot& p, const Piece& c, int u, uint32_t bad, int wave) {
        const Tile k = tile_at(p, c, u);
        const int key = k.key0 + 4 * wave;
        const bool on = u < c.nt;
        tile = u;
        if constexpr (LAYOUT == kRows) {
            first = (int64_t)k.seq * p.L + key;
            rows = on ? min(max(k.high - key, 0), 4) : 0;
        } else if constexpr (LAYOUT == kBlocks) {
            const bool ok = (uint32_t)entry[0] < (uint32_t)p.num_blocks;
            const int at = min(key, p.L - 4);
            first = entry[0] * p.block_size + (at - block_of(p, at) * p.block_size);
            rows = on && ok ? 4 : 0;
            if (__builtin_expect(on && !ok && key < min(c.seen_high, k.high), 0)) lds_store<int>(bad, 1);
        } else {
            bool ok = true;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int at = min(key + i, p.L - 1);
                const bool in = (uint32_t)entry[i] < (uint32_t)p.num_blocks;
                row[i] = on && in ? entry[i] * p.block_size + (at - block_of(p, at) * p.block_size) : -1;
                ok &= in || key + i >= min(c.seen_high, k.high);
            }
            if (__builtin_expect(on && !ok, 0)) lds_store<int>(bad, 1);
        }
    }
    __device__ __forceinline__ void issue(const Hot& p, uint32_t lds, int wave, int lane) const {
        using X = PPLds<FP8>;
        asm volatile("" : "+v"(lane));  // lane offsets kept across the loop would be spilled
        if constexpr (FP8) {
            const uint32_t dst = X::raw(lds, tile) + 4 * wave * kFp8Row, off = (uint32_t)lane << 4;
            if constexpr (LAYOUT == kPages) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (lane < kFp8Row / 16)
                        gather_at<0>(dst + i * kFp8Row,
                                     make_rsrc(p.kv + (int64_t)max(row[i], 0) * kFp8Row, row[i] < 0 ? 0 : kFp8Row), off);
            } else {
                const rsrc_t rs = make_rsrc(p.kv + first * kFp8Row, (uint32_t)rows * kFp8Row);
                gather_at<0>(dst, rs, off);
                gather_at<1024>(dst, rs, off);
                if (lane < (4 * kFp8Row - 2048) / 16) gather_at<2048>(dst, rs, off);
            }
        } else {
            const uint32_t dst = X::stage(lds, tile) + 4 * wave * 1024;
            const uint32_t rope_dst = X::stage(lds, tile) + X::KV_BYTES + 4 * wave * 128;
            // sw_kv(4 wave + i) = sw_kv(4 wave) ^ 4 i
            const uint32_t off = (uint32_t)(lane ^ sw_kv(4 * wave)) << 4;
            if constexpr (LAYOUT == kPages) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    gather_at<0>(dst + i * 1024,
                                 make_rsrc(p.kv + ((int64_t)max(row[i], 0) << 10), row[i] < 0 ? 0 : 1024), off ^ (64u * i));
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (lane < 8)
                        gather_at<0>(rope_dst + i * 128,
                                     make_rsrc(p.k_rope + ((int64_t)max(row[i], 0) << 7), row[i] < 0 ? 0 : 128),
                                     (uint32_t)(lane ^ sw_rope(4 * wave + i)) << 4);
            } else {
                const rsrc_t rs = make_rsrc(p.kv + (first << 10), (uint32_t)rows << 10);
                gather_at<0>(dst, rs, off);
                gather_at<1 * 1024>(dst, rs, off ^ 64u);
                gather_at<2 * 1024>(dst, rs, off ^ 128u);
                gather_at<3 * 1024>(dst, rs, off ^ 192u);
                const int in4 = lane >> 3;
                if (lane < 32)
                    gather_at<0>(rope_dst, make_rsrc(p.k_rope + (first << 7), (uint32_t)rows << 7),
                                 (uint32_t)(in4 << 7) + ((uint32_t)((lane & 7) ^ sw_rope(4 * wave + in4)) << 4));
            }
        }
    }
};

// The wave's four rows of tile u, from raw to the ring: lane l takes the latent
// values 8 l .. 8 l + 7 of each (no bank is met twice), and lane l < 32 16 bytes
// of the rotary part of row l / 8.  kv[d] = bf16(fp32(e4m3) * scale), both
// roundings to nearest even; where all scales are powers of two (2^-100 ..
// 2^100), one conversion a pair gives the same bits.
struct RawRows {
    u32x2 v[4];
    float sc[4];
    __device__ __forceinline__ void read(uint32_t lds, int u, int wave, int lane) {
        asm volatile("" : "+v"(lane));
        const uint32_t raw = PPLds<true>::raw(lds, u) + 4 * wave * kFp8Row;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            v[r] = lds_load<u32x2>(raw + r * kFp8Row + 8 * lane);
            sc[r] = lds_load<float>(raw + r * kFp8Row + kFp8ScaleOff + 4 * (lane >> 4));
        }
    }
};
__device__ __forceinline__ void expand_rows(const RawRows& rows, uint32_t lds, int u, int wave, int lane) {
    using X = PPLds<true>;
    asm volatile("" : "+v"(lane));
    const uint32_t raw = X::raw(lds, u) + 4 * wave * kFp8Row;
    const uint32_t stage = X::stage(lds, u);
    const float(&sc)[4] = rows.sc;
    const u32x2(&v)[4] = rows.v;
    const int in4 = (lane >> 3) & 3, rope = 4 * wave + in4;
    const i32x4 turned = lds_load<i32x4>(raw + in4 * kFp8Row + kFp8RopeOff + 16 * (lane & 7));
    const uint32_t s0 = __float_as_uint(sc[0]), s1 = __float_as_uint(sc[1]), s2 = __float_as_uint(sc[2]);
    const uint32_t s3 = __float_as_uint(sc[3]);
    const bool pow2 = ((s0 | s1 | s2 | s3) & 0x807fffffu) == 0 && min(min(s0, s1), min(s2, s3)) >= 27u << 23 &&
                      max(max(s0, s1), max(s2, s3)) <= 227u << 23;
    const uint32_t dst = stage + 4 * wave * 1024, chunk = (uint32_t)(lane ^ sw_kv(4 * wave)) << 4;
    if (__all(pow2)) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            bf16x8 o;
#pragma unroll
            for (int d = 0; d < 2; ++d) {
                const auto lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)v[r][d], sc[r], false);
                const auto hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)v[r][d], sc[r], true);
                o[4 * d + 0] = lo[0];
                o[4 * d + 1] = lo[1];
                o[4 * d + 2] = hi[0];
                o[4 * d + 3] = hi[1];
            }
            lds_store<bf16x8>(dst + r * 1024 + (chunk ^ (64u * r)), o);  // sw_kv(4 wave + r) = sw_kv(4 wave) ^ 4 r
        }
    } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            bf16x8 o;
#pragma unroll
            for (int d = 0; d < 2; ++d) {
                const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)v[r][d], false);
                const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)v[r][d], true);
                o[4 * d + 0] = (__bf16)(lo[0] * sc[r]);
                o[4 * d + 1] = (__bf16)(lo[1] * sc[r]);
                o[4 * d + 2] = (__bf16)(hi[0] * sc[r]);
                o[4 * d + 3] = (__bf16)(hi[1] * sc[r]);
            }
            lds_store<bf16x8>(dst + r * 1024 + (chunk ^ (64u * r)), o);
        }
    }
    if (lane < 32) lds_store<i32x4>(stage + X::KV_BYTES + rope * 128 + (((lane & 7) ^ sw_rope(rope)) << 4), turned);
}

// Rows of a tile that are in the pool, bit r for row r, from the block table (of pieces with an entry outside it).
__device__ __forceinline__ uint32_t pool_rows(const Hot& p, const Piece& c, int u, int lane) {
    asm volatile("" : "+v"(lane));
    const Tile k = tile_at(p, c, u);
    const int key = min(k.key0 + (lane & 31), p.L - 1);
    const int entry = p.block_table[(int64_t)k.seq * p.max_blocks + block_of(p, key)];
    return (uint32_t)__ballot((uint32_t)entry < (uint32_t)p.num_blocks);
}

// Which of the 32 keys of a tile a query row that sees `seen` rows has: bit r is tile row r.
__device__ __forceinline__ uint32_t key_mask(const Tile& k, int seen, uint32_t valid) {
    const int n = min(max(min(seen, k.high) - k.key0, 0), kKeys), skip = max(k.low - k.key0, 0);  // skip < 32
    return valid & (n == kKeys ? 0xffffffffu : (1u << n) - 1) & (0xffffffffu << skip);
}

// The same with a tree: and the rows `seen` + j of the set bits j of the token's
// words.  A tile takes 32 bits from bit key0 - seen on, from two words.
__device__ __forceinline__ uint32_t tree_mask(ArgsPtr p, const Tile& k, int token, int seen, uint32_t valid) {
    const int at = k.key0 - seen, w = at >> 5;
    const auto* words = (const __attribute__((address_space(4))) int32_t*)(uint64_t)p->tree + (int64_t)token * p->words;
    const uint32_t lo = w >= 0 && w < p->words ? (uint32_t)words[w] : 0u;
    const uint32_t hi = w >= -1 && w + 1 < p->words ? (uint32_t)words[w + 1] : 0u;
    const uint32_t drafted = (uint32_t)(((uint64_t)hi << 32 | lo) >> (at & 31));
    return key_mask(k, seen, valid) | (key_mask(k, p->L, valid) & drafted);
}

// Lane group g's rows of a tile -- 4 g + j (j < 4) and 16 + 4 g + j -- from a key mask: bit j, bit 4 + j.
__device__ __forceinline__ uint32_t lane_rows(uint32_t mask, int g) {
    return (mask >> (4 * g) & 15u) | (mask >> (16 + 4 * g) & 15u) << 4;
}

// Infinities and NaN in a wave's 128 columns of a tile become zeros, where some
// query row does not see all of the tile: a hidden row's weight is 0, which they
// would turn into NaN.  Query rows that do see one have NaN in that column (its
// score may be -inf and so its weight 0, too): the row blocks that do, by their
// masks of the tile's keys, are noted in LDS, a bit a column, and their columns
// made NaN at the end.  All groups that read the columns are past QK of the tile;
// the wave's own LDS accesses are in order, and no other wave writes these columns.
template <int BLOCKS>
__device__ __forceinline__ void clear_specials(uint32_t stage, uint32_t masks, uint32_t poison, int gw, int lane) {
    asm volatile("" : "+v"(lane));
    const uint32_t at = stage + (uint32_t)((lane >> 4) * 1024 + gw * 256 + (lane & 15) * 16);
#pragma unroll 1
    for (int r = 0; r < kKeys; r += 4) {
        i32x4 v = lds_load<i32x4>(at + r * 1024);
        uint32_t any = 0;  // an exponent of all ones carries into its sign bit
#pragma unroll
        for (int d = 0; d < 4; ++d) any |= ((uint32_t)v[d] & 0x7f807f80u) + 0x00800080u;
        if (__builtin_expect((any & 0x80008000u) == 0, 1)) continue;
        uint32_t columns = 0;
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            if ((v[d] & 0x7f80) == 0x7f80) v[d] &= 0xffff0000, columns |= 1u << (2 * d);
            if ((v[d] & 0x7f800000) == 0x7f800000) v[d] &= 0xffff, columns |= 2u << (2 * d);
        }
        lds_store<i32x4>(at + r * 1024, v);
        const int row = r + (lane >> 4), byte = 16 * gw + ((lane & 15) ^ sw_kv(row));  // of the 512 columns' bits
#pragma unroll 1
        for (int b = 0; b < BLOCKS; ++b)
            if (lds_load<uint32_t>(masks + 4 * b) >> row & 1)
                lds_or(poison + 64 * b + (byte & ~3), columns << (8 * (byte & 3)));
        lds_store<int>(poison + kPoisonBytes, 1);
    }
}

// One piece of an item, WIDE: up to 128 rows, else up to 16 NB (NB = 4 if WIDE).
template <bool FP8, int LAYOUT, bool TREE, bool WIDE, int NB>
__device__ __forceinline__ void shared_piece(const Hot& p, const Piece& c, bool whole, int64_t first_row,
                                             uint32_t lds, int wave, int lane) {
    static_assert(!WIDE || NB == 4, "a group's four row blocks");
    using X = PPLds<FP8>;
    using G = Gathers<FP8, LAYOUT>;
    const int grp = wave >> 2, gw = wave & 3;
    const int g = lane >> 4, n16 = lane & 15;
    const int block = (WIDE ? 64 * grp : 0) + 16 * gw;  // this wave's query rows in QK
    const bool live = block < c.it.rows;
    const int row = c.it.row0 + (live ? block : 0);
    const int nt = c.nt;
    const ArgsPtr args = args_now();
    const int token = TREE ? __builtin_amdgcn_readfirstlane(row / args->H) : 0;
    int seen = seen_by<TREE>(args, row / args->H);  // in a scalar register from the first wait on
    const uint32_t p_lds = lds + X::P_OFF + grp * X::P_GROUP, bad = lds + X::BAD_OFF;
    const uint32_t masks = lds + X::MASK_OFF + 16 * grp, poison = lds + X::POISON_OFF;

    bf16x8 qf[18];
    {
        const uint16_t* q = args->q + (int64_t)(row + n16) * 512 + 8 * qk_lane_chunk(g);
#pragma unroll
        for (int ks = 0; ks < 16; ++ks) qf[ks] = *reinterpret_cast<const bf16x8*>(q + 32 * ks);
        const uint16_t* rr = args->q_rope + (int64_t)(row + n16) * 64 + 8 * g;
        qf[16] = *reinterpret_cast<const bf16x8*>(rr);
        qf[17] = *reinterpret_cast<const bf16x8*>(rr + 32);
    }

    f32x4 oacc[NB][8];
    // products, not scaled yet; the maximum of this lane's own
    float m_ref = -FLT_MAX, m_lane = -FLT_MAX, l_run = 0.f;

    // This lane's LDS offsets in the loop, packed as in the sparse ping-pong kernel.
    uint32_t off_kv, off_rope, off_p;
    {
        const uint32_t koff = (uint32_t)(n16 * 1024) | ((uint32_t)(qk_lane_chunk(g) ^ sw_kv(n16)) << 4);
        const int tr_row = 4 * g + (n16 >> 2);
        const uint32_t voff = (uint32_t)(tr_row * 1024 + (gw << 8)) +
                              ((uint32_t)((((n16 & 3) >> 1) ^ sw_kv(tr_row)) << 4) + ((n16 & 1) << 3));
        off_kv = koff | (voff << 16);
        off_rope = (uint32_t)(X::KV_BYTES + n16 * 128) | ((uint32_t)(g ^ sw_rope(n16)) << 4);
        off_p = pp_pchunk(n16, g) | (pp_pchunk(16 * gw + n16, g) << 16);
    }

    uint32_t valid = 0;

    // The keys of tile u that this wave's rows see, where `mask` is not all of them.
    auto seen_mask = [&](int u, uint32_t mask) __attribute__((always_inline)) -> uint32_t {
        if constexpr (TREE) mask = tree_mask(args_now(), tile_at(p, c, u), token, seen, valid);
        return mask;
    };

    // Made ready behind QK, the shorter turn of the two: the gathers (behind:
    // narrow, those of the next QK), and the rows of its next tile that are in
    // the pool.
    G gather, behind;
    auto qk_softmax = [&](int u, bool& overflow) __attribute__((always_inline)) {
        const uint32_t stage = X::stage(lds, u);
        asm volatile("" : "+v"(off_kv), "+v"(off_rope), "+v"(off_p));
        const uint32_t kbase = stage + (off_kv & 0xffffu);
        const uint32_t rbase = stage + off_rope;
        auto kfrag = [&](int step) -> bf16x8 {
            const int ks = step >> 1, sub = step & 1;
            if (ks < 16) return lds_load<bf16x8>((kbase ^ (64u * (ks & 3))) + 256u * (ks >> 2) + sub * 16 * 1024);
            return lds_load<bf16x8>((rbase ^ (64u * (ks - 16))) + sub * 16 * 128);
        };
        constexpr int KD = 6;  // K fragments in flight
        __builtin_amdgcn_s_setprio(2);
        f32x4 sacc[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
        bf16x8 kf[KD];
#pragma unroll
        for (int j = 0; j < KD; ++j) kf[j] = kfrag(j);
        if constexpr (!FP8 && !WIDE) behind.issue(p, lds, wave, lane);
#pragma unroll
        for (int step = 0; step < 36; ++step) {
            sacc[step & 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[step % KD], qf[step >> 1], sacc[step & 1], 0, 0, 0);
            if (step + KD < 36) kf[step % KD] = kfrag(step + KD);
            __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_s_setprio(0);
        float x[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) x[r] = sacc[r >> 2][r & 3];
        uint32_t mask = key_mask(tile_at(p, c, u), seen, valid);
        if (__builtin_expect(mask != 0xffffffffu, 0)) {
            mask = seen_mask(u, mask);
            int ln = lane;
            asm volatile("" : "+v"(ln));
            const uint32_t mine = lane_rows(mask, ln >> 4);
#pragma unroll
            for (int r = 0; r < 8; ++r)
                if (!(mine >> r & 1)) x[r] = -INFINITY;
        }
        float top = -INFINITY;
#pragma unroll
        for (int r = 0; r < 8; ++r) top = fmaxf(top, x[r]);
        m_lane = fmaxf(m_lane, top);
        if (__builtin_expect(__any(m_ref == -FLT_MAX), 0)) {  // a row's first keys: O and l are still zero
            const float m = max_xor32(max_xor16(m_lane));
            if (mask != 0 && m == -FLT_MAX) l_run += kOnlyMinusInf;
            m_ref = m_ref == -FLT_MAX ? m : m_ref;
        }
        const bool ovf = (m_lane - m_ref) * p.scale_log2 > kRestartLog2;
        overflow |= ovf;
        float psum = 0.f;
        bf16x8 pk;
        if (__builtin_expect(__any(ovf), 0)) {  // this pass is to be discarded: the clamp keeps it free of inf
#pragma unroll
            for (int r = 0; r < 8; ++r) x[r] = fminf((x[r] - m_ref) * p.scale_log2, kRestartLog2);
        } else {
#pragma unroll
            for (int r = 0; r < 8; ++r) x[r] = (x[r] - m_ref) * p.scale_log2;
        }
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            const float e = fast_exp2(x[r]);
            psum += e;
            pk[r] = (__bf16)e;
        }
        l_run += psum;
        lds_store<bf16x8>(p_lds + (off_p >> 16), pk);
    };

    // Whether some query row of the block does not see all keys of tile u, the wave's
    // last scored (every wave agrees); which ones its own rows see is left for PV then.
    auto partial = [&](int u) __attribute__((always_inline)) -> bool {
        const Tile k = tile_at(p, c, u);
        const bool some = key_mask(k, c.seen_low, valid) != 0xffffffffu;
        if (__builtin_expect(some, 0)) lds_store<uint32_t>(masks + 4 * gw, seen_mask(u, key_mask(k, seen, valid)));
        return some;
    };

    // fp8, every wave once a tile: its rows of tile u (issued two tiles ago) into
    // the ring, and the gathers of tile u + 2, made ready before, into their place:
    // every value read from there has been converted and stored by then.
    auto expand = [&](int u) __attribute__((always_inline)) {
        if constexpr (FP8) {
            wait_vmcnt<G::LOADS>();
            RawRows landed;
            landed.read(lds, u, wave, lane);  // of a tile behind the piece: not used
            if (u < nt) expand_rows(landed, lds, u, wave, lane);
            gather.issue(p, lds, wave, lane);
        }
    };
    auto advance = [&](int u) __attribute__((always_inline)) {
        if constexpr (FP8) {
            gather.prepare(p, c, u + 2, bad, wave);
            expand(u);
            gather.fetch(p, c, u + 3, wave);
        }
    };

    auto pv = [&](int u, bool clears) __attribute__((always_inline)) {
        const uint32_t stage = X::stage(lds, u);
        asm volatile("" : "+v"(off_kv), "+v"(off_p));
        const uint32_t vbase = stage + (off_kv >> 16);
        auto vfrag = [&](int cb) -> bf16x8 {
            const uint32_t a = vbase ^ (32u * cb);
            const bf16x4 v0 = lds_load_tr(a);
            const bf16x4 v1 = lds_load_tr(a + 16 * 1024);
            return __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7);
        };
        if (__builtin_expect(clears, 0)) {
            if constexpr (!WIDE) clear_specials<NB>(stage, masks, poison, gw, lane);
            else if (grp == 0) clear_specials<8>(stage, masks, poison, gw, lane);  // of both groups' rows
        }
        bf16x8 pf[NB];
#pragma unroll
        for (int hb = 0; hb < NB; ++hb) pf[hb] = lds_load<bf16x8>(p_lds + (off_p & 0xffffu) + 1024 * hb);
        constexpr int VD = NB == 4 ? 3 : 4;  // V fragments in flight
        bf16x8 vf[VD];
#pragma unroll
        for (int j = 0; j < VD; ++j) vf[j] = vfrag(j);
        if constexpr (!FP8) gather.issue(p, lds, wave, lane);
#pragma unroll
        for (int cb = 0; cb < 8; ++cb) {
#pragma unroll
            for (int hb = 0; hb < NB; ++hb)
                oacc[hb][cb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf[cb % VD], pf[hb], oacc[hb][cb], 0, 0, 0);
            if (cb + VD < 8) vf[cb % VD] = vfrag(cb + VD);
            __builtin_amdgcn_sched_barrier(0);
        }
    };

#pragma unroll 1
    for (int pass = 0; pass < 2; ++pass) {
#pragma unroll
        for (int hb = 0; hb < NB; ++hb)
#pragma unroll
            for (int cb = 0; cb < 8; ++cb) oacc[hb][cb] = f32x4{0.f, 0.f, 0.f, 0.f};
        l_run = 0.f;
        if (pass == 1) m_ref = max_xor32(max_xor16(m_lane));
        bool overflow = false;
        // The first two tiles' rows, and Q: a full wait, as the compiler does not
        // count the gathers (it would wait for Q in the loop).
        gather.fetch(p, c, 0, wave);
        behind.fetch(p, c, 1, wave);
        if (threadIdx.x == 0) lds_store<int>(bad, 0);
        if (threadIdx.x <= kPoisonBytes / 4) lds_store<int>(poison + 4 * threadIdx.x, 0);
        lds_barrier();
        gather.prepare(p, c, 0, bad, wave);
        gather.issue(p, lds, wave, lane);
        behind.prepare(p, c, 1, bad, wave);
        behind.issue(p, lds, wave, lane);
        gather.fetch(p, c, 2, wave);
        wait_vmcnt<0>();
        seen = live ? __builtin_amdgcn_readfirstlane(seen) : 0;
        if constexpr (FP8) advance(0);
        else gather.prepare(p, c, 2, bad, wave);
        // Rows of tile u in the pool: all, unless the piece has met a bad entry (every wave is past preparing tile u).
        auto turn_to = [&](int u, auto&& prepare) __attribute__((always_inline)) {
            if constexpr (LAYOUT == kRows) {
                prepare();
                valid = 0xffffffffu;
            } else {
                const int met = lds_load<int>(bad);
                prepare();
                valid = 0xffffffffu;
                if (__builtin_expect(__builtin_amdgcn_readfirstlane(met), 0)) valid = pool_rows(p, c, u, lane);
            }
        };
        auto nothing = [] {};
        if constexpr (!WIDE) {
            // bf16: in half u every wave issues its rows of tile u + 2, into the
            // stage of tile u - 2, which was last read in half u - 1; the half
            // ends with its rows of tile u + 1 landed.
            lds_barrier();
            turn_to(grp, nothing);
            if (grp == 1) {  // half 0, without PV
                if constexpr (FP8) {
                    advance(1);
                } else {
                    gather.issue(p, lds, wave, lane);
                    wait_vmcnt<G::LOADS>();
                    gather.fetch(p, c, 3, wave);
                    gather.prepare(p, c, 3, bad, wave);
                }
                lds_barrier();
            }
            if constexpr (!FP8) {
                behind = gather;
                gather.fetch(p, c, 3 + grp, wave);
                behind.fetch(p, c, 4 + grp, wave);
            }
#pragma unroll 1
            for (int u = grp; u < nt; u += 2) {
                if (live) qk_softmax(u, overflow);
                else if constexpr (!FP8) behind.issue(p, lds, wave, lane);
                const bool clears = partial(u);
                turn_to(u + 2, [&]() __attribute__((always_inline)) {
                    if constexpr (FP8) {
                        advance(u + 1);
                    } else {
                        wait_vmcnt<G::LOADS>();
                        gather.prepare(p, c, u + 3, bad, wave);
                        behind.prepare(p, c, u + 4, bad, wave);
                        gather.fetch(p, c, u + 5, wave);
                        behind.fetch(p, c, u + 6, wave);
                    }
                });
                lds_barrier();
                pv(u, clears);
                if constexpr (FP8) {
                    advance(u + 2);
                } else {
                    wait_vmcnt<G::LOADS>();
                }
                lds_barrier();
            }
            if (((nt ^ grp) & 1) == 0) lds_barrier();  // half nt: the other group's last PV
        } else {
            // bf16: tile t + 3 is issued in PV of tile t, into the stage of tile
            // t - 1, which both groups are past.  A tile in which some row sees
            // less than all has one barrier more, between group 1's QK and group
            // 0's clear_specials of it; group 1 meets it cleared.
            if constexpr (!FP8)
                if (grp == 0) gather.issue(p, lds, wave, lane);
            lds_barrier();
            turn_to(0, nothing);
            if (grp == 1) {  // half 0, without PV
                if constexpr (FP8) advance(1);
                else gather.issue(p, lds, wave, lane);
                lds_barrier();
            }
            if constexpr (!FP8) gather.fetch(p, c, 3, wave);
#pragma unroll 1
            for (int t = 0; t < nt; ++t) {
                if (live) qk_softmax(t, overflow);
                const bool clears = partial(t);
                if (grp == 1) {
                    if (__builtin_expect(clears, 0)) lds_barrier();
                    if constexpr (!FP8) wait_vmcnt<G::LOADS>();
                }
                turn_to(t + 1, [&]() __attribute__((always_inline)) {
                    const int next = FP8 ? t + 3 + grp : t + 3;
                    gather.prepare(p, c, next, bad, wave);
                    gather.fetch(p, c, next + 1, wave);
                });
                lds_barrier();
                if (grp == 0 && __builtin_expect(clears, 0)) lds_barrier();
                pv(t, clears);
                expand(t + 1 + grp);  // fp8: behind PV, when the other group's QK has left the LDS
                if constexpr (!FP8)
                    if (grp == 0) wait_vmcnt<2 * G::LOADS>();
                lds_barrier();
            }
            if (grp == 0) lds_barrier();  // half 2 nt: group 1's last PV
        }
        wait_vmcnt<0>();  // gathers behind the piece write zeros into LDS
        if (pass == 1) break;
        // does any row need the second pass?
        const uint32_t flag = lds + X::FLAG_OFF;
        lds_barrier();
        if (threadIdx.x == 0) lds_store<int>(flag, 0);
        lds_barrier();
        if (__any(overflow) && lane == 0) lds_store<int>(flag, 1);
        lds_barrier();
        if (__builtin_amdgcn_readfirstlane(lds_load<int>(flag)) == 0) break;
    }

    // ---- the QK waves publish (l, reference, maximum) of their rows; the PV waves scale their blocks
    lds_barrier();
    const ArgsPtr out = args_now();
    const uint32_t ml = lds + X::ML_OFF;
    l_run = sum_xor32(sum_xor16(l_run));
    const float m_true = max_xor32(max_xor16(m_lane));
    int eln = lane;
    asm volatile("" : "+v"(eln));
    const int eg = eln >> 4, en16 = eln & 15;
    if (eg == 0) {
        const int hl = 64 * grp + 16 * gw + en16;
        lds_store<float>(ml + 4 * hl, l_run);
        lds_store<float>(ml + 4 * (128 + hl), m_ref);
        lds_store<float>(ml + 4 * (256 + hl), m_true);
    }
    if (__builtin_expect(__builtin_amdgcn_readfirstlane(lds_load<int>(poison + kPoisonBytes)), 0)) {
#pragma unroll
        for (int hb = 0; hb < NB; ++hb)
#pragma unroll
            for (int cb = 0; cb < 8; ++cb) {
                const uint32_t word = lds_load<uint32_t>(poison + 64 * ((WIDE ? 4 * grp : 0) + hb) + 16 * gw + (cb >> 1) * 4);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (word >> (16 * (cb & 1) + 4 * eg + j) & 1) oacc[hb][cb][j] = NAN;
            }
    }
    lds_barrier();
    constexpr int HROW = 1040;      // bytes of a staged bf16 row (16 more: rows spread over the banks)
    constexpr int kPartRow = 2064;  // of a staged fp32 row
    static_assert(128 * HROW <= X::P_OFF && 64 * kPartRow <= X::P_OFF, "staging fits the ring and raw tiles");
    static_assert(3 * 128 * 4 <= 2 * X::P_GROUP, "statistics fit the P buffers");
    auto put_stats = [&](int hl, float top, float sum) __attribute__((always_inline)) {
        if (hl >= c.it.rows) return;
        if (whole) {
            const Returned r = returned(top, sum, out->scale);
            out->out_max[c.it.row0 + hl] = r.max;
            out->out_sum[c.it.row0 + hl] = r.sum;
        } else {
            out->part_m[first_row + hl] = top;
            out->part_l[first_row + hl] = sum;
        }
    };
    // Staged rows [first, first + n) of the block, row r at HROW (bf16) or kPartRow (fp32) * (r - first), stored whole.
    auto store_rows = [&](int first, int n) __attribute__((always_inline)) {
        const int end = min(first + n, c.it.rows);
        if (whole) {
            uint16_t* base = out->out + (int64_t)c.it.row0 * 512 + 8 * eln;
            for (int r = first + wave; r < end; r += 8)
                *reinterpret_cast<bf16x8*>(base + (int64_t)r * 512) = lds_load<bf16x8>(lds + (r - first) * HROW + 16 * eln);
        } else {
            float* base = out->part_o + first_row * 512 + 4 * eln;
            for (int i = 2 * first + wave; i < 2 * end; i += 8)
                *reinterpret_cast<f32x4*>(base + (i >> 1) * 512 + 256 * (i & 1)) =
                    lds_load<f32x4>(lds + (uint32_t)(((i >> 1) - first) * kPartRow + 1024 * (i & 1) + 16 * eln));
        }
    };
    auto stage_block = [&](int r, int col, const f32x4& o) __attribute__((always_inline)) {  // r: row within the staged ones
        if (whole) {
            bf16x4 v;
            v[0] = (__bf16)o[0];
            v[1] = (__bf16)o[1];
            v[2] = (__bf16)o[2];
            v[3] = (__bf16)o[3];
            lds_store<bf16x4>(lds + (uint32_t)(r * HROW + 2 * col), v);
        } else {
            lds_store<f32x4>(lds + (uint32_t)(r * kPartRow + 4 * col), o);
        }
    };
    if constexpr (WIDE) {
        float scale[NB];
#pragma unroll
        for (int hb = 0; hb < NB; ++hb) {
            const int hl = 64 * grp + 16 * hb + en16;
            const float l = lds_load<float>(ml + 4 * hl), mr = lds_load<float>(ml + 4 * (128 + hl));
            const float top = lds_load<float>(ml + 4 * (256 + hl));
            const float to_true = fast_exp2((mr - top) * p.scale_log2), sum = l * to_true;
            scale[hb] = to_true;
            if (whole) scale[hb] *= returned(top, sum, 1.f).inv;
            if (gw == 0 && eg == 0) put_stats(hl, top, sum);
        }
        auto stage = [&](int at) __attribute__((always_inline)) {
#pragma unroll
            for (int hb = 0; hb < NB; ++hb)
#pragma unroll
                for (int cb = 0; cb < 8; ++cb)
                    stage_block(at + 16 * hb + en16, 128 * gw + 16 * cb + 4 * eg, oacc[hb][cb] * scale[hb]);
        };
        if (whole) {
            stage(64 * grp);
            lds_barrier();
            store_rows(0, 128);
        } else {  // fp32 rows: one group's at a time
            if (grp == 0) stage(0);
            lds_barrier();
            store_rows(0, 64);
            lds_barrier();
            if (grp == 1) stage(0);
            lds_barrier();
            store_rows(64, 64);
        }
    } else {
        // Both groups hold O of the same rows over their own tiles: each is scaled
        // to the common maximum, a wave hands half of its column blocks to the wave
        // of the other group with the same columns and adds what it gets.
        constexpr uint32_t kHand = NB * 4 * 1024;  // one wave's half: NB row x 4 column blocks of 64 lanes x 16 bytes
        static_assert(8 * kHand <= X::P_OFF, "handed halves fit");
        const uint32_t give = lds + (uint32_t)wave * kHand + 16u * (uint32_t)eln;
        const uint32_t take = lds + (uint32_t)(wave ^ 4) * kHand + 16u * (uint32_t)eln;
        float scale[NB];
#pragma unroll
        for (int hb = 0; hb < NB; ++hb) {
            const int hl = 16 * hb + en16;
            float l[2], mr[2], mt[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                l[k] = lds_load<float>(ml + 4 * (64 * k + hl));
                mr[k] = lds_load<float>(ml + 4 * (128 + 64 * k + hl));
                mt[k] = lds_load<float>(ml + 4 * (256 + 64 * k + hl));
            }
            const float top = fmaxf(mt[0], mt[1]);
            const float f0 = fast_exp2((mr[0] - top) * p.scale_log2), f1 = fast_exp2((mr[1] - top) * p.scale_log2);
            const float sum = fmaf(l[0], f0, l[1] * f1);
            scale[hb] = grp == 0 ? f0 : f1;
            if (whole) scale[hb] *= returned(top, sum, 1.f).inv;
            if (wave == 0 && eg == 0) put_stats(hl, top, sum);
        }
        auto finish = [&](auto kept) __attribute__((always_inline)) {  // kept: 0 (blocks 0-3) or 4 (blocks 4-7)
            constexpr int KEEP = decltype(kept)::value, GIVE = 4 - KEEP;
#pragma unroll
            for (int hb = 0; hb < NB; ++hb)
#pragma unroll
                for (int cb = 0; cb < 4; ++cb)
                    lds_store<f32x4>(give + 1024u * (4 * hb + cb), oacc[hb][GIVE + cb] * scale[hb]);
            lds_barrier();
#pragma unroll
            for (int hb = 0; hb < NB; ++hb)
#pragma unroll
                for (int cb = 0; cb < 4; ++cb)
                    oacc[hb][KEEP + cb] = oacc[hb][KEEP + cb] * scale[hb] + lds_load<f32x4>(take + 1024u * (4 * hb + cb));
            lds_barrier();  // the halves are read: the ring is free for the staged rows
#pragma unroll
            for (int hb = 0; hb < NB; ++hb)
#pragma unroll
                for (int cb = 0; cb < 4; ++cb)
                    stage_block(16 * hb + en16, 128 * gw + 16 * (KEEP + cb) + 4 * eg, oacc[hb][KEEP + cb]);
        };
        if (grp == 0) finish(std::integral_constant<int, 0>{});
        else finish(std::integral_constant<int, 4>{});
        lds_barrier();
        store_rows(0, 16 * NB);
    }
    lds_barrier();  // LDS is free for the next piece
}

template <bool FP8, int LAYOUT, bool TREE>
__global__ __launch_bounds__(kPPThreads, 1) void shared_main_kernel(SharedParams arguments) {
    using X = PPLds<FP8>;
    __shared__ __attribute__((aligned(1024))) char smem[X::LDS_BYTES];
    const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)smem;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Hot hot{arguments.kv,          reinterpret_cast<const char*>(arguments.k_rope), arguments.block_table,
                  arguments.L,           arguments.prefix,      arguments.max_blocks,   arguments.block_size,
                  arguments.num_blocks,  arguments.block_magic, arguments.block_shift,  arguments.scale_log2};
    ArgsPtr p = args_now();
    // The share: every workgroup sums the costs itself (a launch before this one
    // would take 5 us more), a thread those of a run of items, and finds the item
    // that its share starts in.
    const int w = blockIdx.x;
    int64_t c0, c1;
    {
        const int items = p->items, run = (items + kPPThreads - 1) / kPPThreads;
        const int i0 = min((int)threadIdx.x * run, items), i1 = min(i0 + run, items);
        int64_t sum = 0;
        Look k;
        for (int i = i0; i < i1; ++i) {
            look_at<TREE>(p, i, k);
            sum += k.cost;
            if (w == 0 && k.cost == 0) p->ends[i] = int2{0, -1};  // nobody's: for the merge
        }
        int64_t scan = sum;
        if (run == 1) {  // 64 items cost less than 2^32
            uint32_t s = (uint32_t)sum;
            for (int d = 1; d < 64; d <<= 1) {
                const uint32_t u = __shfl_up(s, d);
                if (lane >= d) s += u;
            }
            scan = s;
        } else {
            for (int d = 1; d < 64; d <<= 1) {
                const int64_t u = __shfl_up(scan, d);
                if (lane >= d) scan += u;
            }
        }
        int64_t* sums = reinterpret_cast<int64_t*>(smem);
        if (lane == 63) sums[wave] = scan;
        __syncthreads();
        int64_t begin = scan - sum, total = 0;
        for (int v = 0; v < kPPThreads / 64; ++v) {
            if (v < wave) begin += sums[v];
            total += sums[v];
        }
        total = (int64_t)__builtin_amdgcn_readfirstlane((int)(total >> 32)) << 32 |
                (uint32_t)__builtin_amdgcn_readfirstlane((int)total);
        const int groups = (int)max((int64_t)1, min((int64_t)p->workgroups, total / kMinShare));
        if (total == 0 || w >= groups) return;
        const Shares shares(total, groups);
        c0 = shares.start(w);
        c1 = shares.start(w + 1);
        if (begin <= c0 && c0 < begin + sum) {
            for (int i = i0; i < i1; ++i) {
                if (run > 1) look_at<TREE>(p, i, k);
                if (c0 < begin + k.cost) {
                    int* plan = reinterpret_cast<int*>(smem + X::PLAN_OFF);
                    plan[0] = i;
                    plan[1] = k.low;
                    plan[2] = k.high;
                    *reinterpret_cast<int64_t*>(plan + 4) = begin;
                    break;
                }
                begin += k.cost;
            }
        }
        __syncthreads();
    }
    const int* plan = reinterpret_cast<const int*>(smem + X::PLAN_OFF);
    int i = __builtin_amdgcn_readfirstlane(plan[0]);
    int low = __builtin_amdgcn_readfirstlane(plan[1]), high = __builtin_amdgcn_readfirstlane(plan[2]);
    // costs from here on: from the first item's begin
    int64_t begin;
    {
        const int64_t first = *reinterpret_cast<const int64_t*>(plan + 4);
        begin = (int64_t)__builtin_amdgcn_readfirstlane((int)(first >> 32)) << 32 |
                (uint32_t)__builtin_amdgcn_readfirstlane((int)first);
    }
#pragma unroll 1
    for (;;) {
        p = args_now();
        Look k;
        look_at(p, i, low, high, k);
        // its first tile that starts at c0 or behind, and at c1
        const int64_t tile0 = begin + k.each.piece, end = begin + k.cost;
        const int tiles = k.it.first + k.it.second;
        const int a = c0 <= tile0 ? 0 : ((int)(c0 - tile0) + k.each.tile - 1) / k.each.tile;
        const int b = c1 <= tile0 ? 0 : ((int)(min(c1, end) - tile0) + k.each.tile - 1) / k.each.tile;
        if (a < b) {
            Piece c;
            c.it = k.it;
            c.it.first = __builtin_amdgcn_readfirstlane(c.it.first);
            c.seen_low = __builtin_amdgcn_readfirstlane(low);
            c.seen_high = __builtin_amdgcn_readfirstlane(high);
            c.a = __builtin_amdgcn_readfirstlane(a);
            c.nt = __builtin_amdgcn_readfirstlane(b - a);
            const bool whole = !p->stacked && c.nt == tiles;
            if (threadIdx.x == 0 && a == 0) p->ends[i].x = w;
            if (threadIdx.x == 0 && b == tiles) p->ends[i].y = w;
            const int64_t first_row = piece_row(p, i, w, c.a == 0);
            if (c.it.rows > 64) shared_piece<FP8, LAYOUT, TREE, true, 4>(hot, c, whole, first_row, lds, wave, lane);
            else if (c.it.rows > 32) shared_piece<FP8, LAYOUT, TREE, false, 4>(hot, c, whole, first_row, lds, wave, lane);
            else if (c.it.rows > 16) shared_piece<FP8, LAYOUT, TREE, false, 2>(hot, c, whole, first_row, lds, wave, lane);
            else shared_piece<FP8, LAYOUT, TREE, false, 1>(hot, c, whole, first_row, lds, wave, lane);
        }
        p = args_now();
        if (end >= c1 || ++i >= p->items) break;
        begin = end;
        look_at<TREE>(p, i, k);
        low = __builtin_amdgcn_readfirstlane(k.low);
        high = __builtin_amdgcn_readfirstlane(k.high);
    }
}

// ------------------------------------------------------------------ merge
// Rows of cut items joined, and rows without keys filled in; rows of whole items
// are there already.  A workgroup owns 2 * turns rows of an item (stacked: of all
// rows), two at a time; thread t of a row's 128 owns columns 4 t .. 4 t + 3.  Six
// pieces are read at a time.  Where rows are few (SPLIT), a workgroup owns one, and
// four groups of 128 threads take its pieces, six at a time, in turn.
constexpr int kMergeBatch = 6, kMergeSplit = 4, kMergeFewRows = 2048;
template <bool STACKED, bool SPLIT>
__global__ __launch_bounds__(SPLIT ? 128 * kMergeSplit : 256) void shared_merge_kernel(SharedParams, int turns, int block0) {
    constexpr int ROWS = SPLIT ? 1 : 2, GROUPS = SPLIT ? kMergeSplit : 1;
    __shared__ f32x4 parts[SPLIT ? 128 * (kMergeSplit - 1) : 1];
    __shared__ float2 stats[SPLIT ? kMergeSplit - 1 : 1];  // maximum, sum
    const ArgsPtr p = args_now();
    const int rows = p->B * p->SQ * p->H, col = (threadIdx.x & 127) * 4;
    const int seq_rows = p->SQ * p->H, block = block0 + (int)blockIdx.x;
    const int half = SPLIT ? 0 : threadIdx.x >> 7, group = SPLIT ? threadIdx.x >> 7 : 0;
    int first, count;  // the workgroup's rows
    if constexpr (STACKED) {
        first = block * ROWS * turns;
        count = min(ROWS * turns, rows - first);
    } else {
        const int chunks = kSharedRows / (ROWS * turns), i = block / chunks, chunk = block % chunks;
        const int2 ends = p->ends[i];
        if (ends.x == ends.y) return;  // a whole item
        const Item it = item_rows(p, i);
        first = it.row0 + chunk * ROWS * turns;
        count = min(ROWS * turns, it.row0 + it.rows - first);
    }
    for (int r = half; r < count; r += ROWS) {
        const int row = __builtin_amdgcn_readfirstlane(first + r), b = row / seq_rows, in_seq = row - b * seq_rows;
        float m = -FLT_MAX, l = 0.f;
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
        auto join = [&](float top_of, float sum, const f32x4& u) __attribute__((always_inline)) {
            const float top = fmaxf(m, top_of);
            const float keep = fast_exp2((m - top) * p->scale_log2), add = fast_exp2((top_of - top) * p->scale_log2);
            l = l * keep + sum * add;
            acc = acc * keep + u * add;
            m = top;
        };
        // its pieces: of the stacked item first, then of the sequence's own
        const int own = p->prefix_items + b * p->seq_blocks + in_seq / kSharedRows, shared = row / kSharedRows;
        int2 e1 = p->ends[own], e0 = STACKED ? p->ends[shared] : int2{0, -1};
        e1.x = __builtin_amdgcn_readfirstlane(e1.x);
        e1.y = __builtin_amdgcn_readfirstlane(e1.y);
        e0.x = __builtin_amdgcn_readfirstlane(e0.x);
        e0.y = __builtin_amdgcn_readfirstlane(e0.y);
        const int n0 = e0.y - e0.x + 1, n = n0 + (e1.y - e1.x + 1);
        for (int j0 = __builtin_amdgcn_readfirstlane(group) * kMergeBatch; j0 < n; j0 += GROUPS * kMergeBatch) {
            float ms[kMergeBatch], ls[kMergeBatch];
            f32x4 u[kMergeBatch];
#pragma unroll
            for (int k = 0; k < kMergeBatch; ++k) {
                const int j = j0 + k;
                if (j >= n) break;
                const int64_t prow = j < n0 ? piece_row(p, shared, e0.x + j, j == 0) + row % kSharedRows
                                            : piece_row(p, own, e1.x + (j - n0), j == n0) + in_seq % kSharedRows;
                ms[k] = p->part_m[prow];
                ls[k] = p->part_l[prow];
                u[k] = *reinterpret_cast<const f32x4*>(p->part_o + prow * 512 + col);
            }
#pragma unroll
            for (int k = 0; k < kMergeBatch; ++k) {
                if (j0 + k >= n) break;
                join(ms[k], ls[k], u[k]);
            }
        }
        if constexpr (SPLIT) {
            if (group > 0) {
                parts[128 * (group - 1) + (threadIdx.x & 127)] = acc;
                if (col == 0) stats[group - 1] = float2{m, l};
            }
            __syncthreads();
            if (group > 0) return;
            for (int g = 0; g < GROUPS - 1; ++g) join(stats[g].x, stats[g].y, parts[128 * g + threadIdx.x]);
        }
        const Returned got = returned(m, l, p->scale);
        bf16x4 v;
        for (int e = 0; e < 4; ++e) v[e] = (__bf16)(acc[e] * got.inv);
        *reinterpret_cast<bf16x4*>(p->out + (int64_t)row * 512 + col) = v;
        if (col == 0) {
            p->out_max[row] = got.max;
            p->out_sum[row] = got.sum;
        }
    }
}

template <bool STACKED>
int launch_merge(const SharedParams& p, hipStream_t stream) {
    const int rows = p.B * p.SQ * p.H;
    // Many rows are a prefill's, most of them there already: sixteen a workgroup (262,144
    // rows: 59 us for 121 with two; from 8192 to 65,536 a call is within 3 % either way:
    // 32,768 stacked 461 and 457 us, whole items 302 and 302).  Few: one, shared by four
    // groups (stacked, behind 8192 rows: 48 rows 20.5 us a call for 21.8, 512 47 for 50,
    // 1024 58 and 58, 2048 82 and 80, 4096 127 for 121; whole items 1024 49 for 46).
    const bool split = rows <= kMergeFewRows;
    const int turns = rows >= 32768 ? 8 : 1, own = split ? 1 : 2 * turns;
    const int grid = STACKED ? (rows + own - 1) / own : p.items * (kSharedRows / own);
    auto* kernel = split ? shared_merge_kernel<STACKED, true> : shared_merge_kernel<STACKED, false>;
    constexpr int kMaxGrid = 1 << 22;  // a grid's threads, 512 a workgroup, are counted in 32 bits
    for (int first = 0; first < grid; first += kMaxGrid) {
        const int n = grid - first < kMaxGrid ? grid - first : kMaxGrid;
        hipLaunchKernelGGL(kernel, dim3(n), dim3(split ? 128 * kMergeSplit : 256), 0, stream, p, turns, first);
        if (const int rc = (int)hipGetLastError()) return rc;
    }
    return 0;
}

}  // namespace

template <bool TREE>
auto* main_kernel(const SharedParams& p) {
    const int layout = !p.block_table ? kRows : p.block_size % 4 == 0 ? kBlocks : kPages;
    return p.kv_fp8 ? (layout == kRows     ? shared_main_kernel<true, kRows, TREE>
                       : layout == kBlocks ? shared_main_kernel<true, kBlocks, TREE>
                                           : shared_main_kernel<true, kPages, TREE>)
                    : (layout == kRows     ? shared_main_kernel<false, kRows, TREE>
                       : layout == kBlocks ? shared_main_kernel<false, kBlocks, TREE>
                                           : shared_main_kernel<false, kPages, TREE>);
}

int launch_shared(const SharedParams& p, hipStream_t stream) {
    auto* kernel = p.tree ? main_kernel<true>(p) : main_kernel<false>(p);
    hipLaunchKernelGGL(kernel, dim3(p.workgroups), dim3(kPPThreads), 0, stream, p);
    const int rc = (int)hipGetLastError();
    if (rc) return rc;
    return p.stacked ? launch_merge<true>(p, stream) : launch_merge<false>(p, stream);
}

}  // namespace dsa
