// How the attention over paged rows is cut into work, shared by its kernels and the kernel that merges split work.
//
// An item is one KV head and a block of up to `block` tokens of a sequence (all query heads of the KV head for each: the rows of a
// product); its work is the tiles of 128 (f16) or 64 (f32) keys from the first key that any of its tokens sees to the last. The items of all sequences
// (sequence by sequence, block by block, KV head by KV head) are laid end to end and cut into ranges of about the same cost, one a CTA,
// so that decode steps over long histories and long blocks over short ones fill the GPU alike. A CTA's range is a few segments, each of
// which costs as much as `segment` tiles beside its tiles (queries, the first tile's latency, outputs); a segment that covers its whole
// item writes the output, another its un-normalised part, and the parts are merged in the order of their keys: sums do not depend on
// timing.
#pragma once
#include "pool.cuh"

namespace mkv {

constexpr uint32_t PLAN_SEQS = 128; // sequences of one launch
constexpr uint32_t PLAN_CTAS = 160;
constexpr uint32_t PLAN_FEW = 32; // rows of an item up to which the f32 kernel has a form of its own

struct PlanSeq {
    uint32_t table, first, pos, ntok, row; // first entry of the page table; first key seen; ...; packed tokens in front
};
struct PlanStart { // where a CTA's range begins, and how many tiles it has
    uint16_t seq, kvh;
    uint32_t block, tile, tiles; // tile: of the item
};
struct PoolPlan {
    uint32_t nseq, ctas;
    uint32_t kv_heads, group, block, window;
    PlanSeq seq[PLAN_SEQS];
    PlanStart start[PLAN_CTAS];
};

// What a block of tokens sees
struct PlanItem {
    uint32_t tok0, ntok;  // tokens of the block, counted from the sequence's first of this call
    uint32_t lo, hi;      // keys that any of its tokens sees: lo <= key < hi
    uint32_t all_lo, all_hi; // keys that each of them sees
    uint32_t tile0, tiles;   // in units of `keys`
};
__host__ __device__ inline uint32_t plan_lowest(const PlanSeq &s, uint32_t window, uint32_t tok) {
    const uint32_t end = s.pos + tok + 1u; // (positions stay below 2^30)
    const uint32_t lo = window != 0u && end > window ? end - window : 0u;
    return lo > s.first ? lo : s.first;
}
__host__ __device__ inline PlanItem plan_item(const PlanSeq &s, uint32_t window, uint32_t block, uint32_t b, uint32_t keys) {
    PlanItem it;
    it.tok0 = b * block;
    it.ntok = s.ntok - it.tok0 < block ? s.ntok - it.tok0 : block;
    it.lo = plan_lowest(s, window, it.tok0);
    it.hi = s.pos + it.tok0 + it.ntok;
    it.all_lo = plan_lowest(s, window, it.tok0 + it.ntok - 1u);
    it.all_hi = s.pos + it.tok0 + 1u;
    if (it.lo >= it.hi) it.lo = it.hi; // nothing seen: one tile, all of it masked
    it.tile0 = (it.lo < it.hi ? it.lo : it.hi - 1u) / keys;
    it.tiles = (it.hi + keys - 1u) / keys - it.tile0;
    return it;
}

struct PlanSegment {
    uint32_t seq, kvh, a, b; // tiles [a, b) of the item
    PlanItem it;
    bool whole;
    uint32_t part; // scratch of a part: 0 = it continues an item, 1 = it begins one (a CTA has at most one of each)
};
// Walks the segments of one CTA.
struct PlanWalk {
    const PoolPlan &p;
    uint32_t keys, seq, kvh, block, tile, left;
    __host__ __device__ __forceinline__ PlanWalk(const PoolPlan &plan, uint32_t cta, uint32_t keys_) : p(plan), keys(keys_) {
        const PlanStart &s = plan.start[cta];
        seq = s.seq;
        kvh = s.kvh;
        block = s.block;
        tile = s.tile;
        left = s.tiles;
    }
    __host__ __device__ __forceinline__ bool next(PlanSegment &s) {
        if (left == 0u) return false;
        s.seq = seq;
        s.kvh = kvh;
        s.it = plan_item(p.seq[seq], p.window, p.block, block, keys);
        s.a = tile;
        s.b = tile + left < s.it.tiles ? tile + left : s.it.tiles;
        s.whole = s.a == 0u && s.b == s.it.tiles;
        s.part = s.a == 0u ? 1u : 0u;
        left -= s.b - s.a;
        tile = 0;
        if (++kvh == p.kv_heads) {
            kvh = 0;
            if (++block * p.block >= p.seq[seq].ntok) {
                block = 0;
                seq++;
            }
        }
        return true;
    }
};

// One split item for the merge: its parts are those of CTAs cta0 .. cta0 + parts - 1.
struct MergeItem {
    uint32_t row, head; // packed row of its first token, first query head
    uint32_t ntok;      // tokens of the block
    uint16_t cta0, parts;
};
struct MergeList {
    uint32_t n, group;
    MergeItem item[PLAN_CTAS];
};

struct PlanCost {
    uint32_t rows;    // of an item: query heads of a KV head times tokens
    uint32_t keys;    // of a tile
    uint32_t segment; // in tiles
    uint32_t whole;   // tiles of an item up to which it is not worth a merge
};
// Plans one launch over the items [i, n) that it takes (i is moved on); rows: packed tokens in front of them, moved on too.
// Returns false when no item with tokens is left.
bool pool_plan(const Pool *p, const mkv_seq_rows *items, int n, int &i, uint32_t &rows, uint32_t window, const PlanCost &cost, PoolPlan &plan, MergeList &merge);

// The floats of a part in scratch memory: [128 rows][dim], then [128 rows][maximum, sum]; two parts a CTA. Behind those of all CTAs the f16 kernel
// has another [128 rows][dim] for each.
__host__ __device__ inline size_t part_floats(uint32_t dim) { return 128u * (size_t)(dim + 2u); }
__host__ __device__ inline size_t part_slot(uint32_t cta, uint32_t part) { return 2u * (size_t)cta + part; }

inline size_t pool_attn_ctas(const Pool *p) { return std::min<uint32_t>((uint32_t)p->ctx->sm_count, PLAN_CTAS); }

mkv_status launch_pool_merge(Pool *p, const MergeList &merge, const PoolAttn &a);
mkv_status pool_attn_f16_setup(Pool *);
mkv_status launch_pool_attn_f16(Pool *p, int layer, const PoolPlan &plan, const PoolAttn &a);
mkv_status pool_attn_f32_setup(Pool *);
mkv_status launch_pool_attn_f32(Pool *p, int layer, const PoolPlan &plan, const PoolAttn &a);

} // namespace mkv
