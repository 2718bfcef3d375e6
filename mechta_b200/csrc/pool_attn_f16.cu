// Attention of blocks of new tokens over f16 pages on the 5th-generation tensor cores: tcgen05.mma with the scores, the weights
// and the output in tensor memory, queries in shared memory, K/V tiles staged by TMA page by page.
//   out_t = sum_k e^(s_k - M) v_k / (sum_k e^(s_k - M) + e^(sink - M)),  s_k = scale q_t . k_k
//
// An item is 128 rows = the query heads of one KV head for 128 / group tokens (row = token * group + head). Per tile of 128 keys:
//   S = Q K^T   A = Q (shared memory), B = the K tile as TMA left it (K-major)
//   P = 2^(S - reference) as f16, back into the columns of S (base-2 exponents throughout)
//   O += P V    A = P (tensor memory), B = the V tile as TMA left it (N-major)
// One pass: the reference of a row lies PA_BIAS2 = 7 below its maximum at the time, and moves only when a tile exceeds that maximum by more
// than PA_LAZY2 = 8 (then O is rescaled). Weights stay below 2^15 (f16 ends at 65,504) and are rounded by 2^-11 of themselves down to 2^-21 of the
// row's largest, by 2^-32 of that below (with the reference at the maximum itself it was 2^-25, and 65,536 keys at 2^-25 of one, 0.2% of the sum,
// were lost). 8 is as seldom exceeded as more would be (ragged blocks under a window with 6, 8, 10 and 11.5: 63.8, 61.4, 61.3 and 61.0 us); scores
// of N(0, 1) grow by about 4 behind their first tile. Sums are kept in f32, and those of the weights run over the rounded ones, so that an output is
// a true mean of the values (the same blocks 63.4 us, 61.4 with sums of the weights in front of their rounding).
// The tensor core's f32 sums truncate, all in one direction: about 2^-23.3 of O for each 16 keys (values of one sign over 300,000 keys came out 1.0e-3
// too small). So every 48 tiles (4.2e-5 by then, a sixth of an output's smallest half step) O is added, with rounding, to what its thread has of it
// in global memory, and starts again; the segment's end adds the two. A fold takes 6,000 clocks, the time that the SM's 128 KB of stores need; the
// long block below takes 1,232 us where it took 1,195 without, 1,280 with a fold every 32 tiles.
// TMEM: O = columns 0 .. DIM - 1, then two (DIM = 256) or three S buffers of 128 columns, so that the scores of the next tiles are there when
// a tile's softmax begins.
//
// Two threads share a row, 64 of a tile's keys each. Scores and outputs are issued by a warp each: the tensor cores hold no more than two
// or three products in advance, so what one issuing thread does between two groups of products would cost their time.
//
// K and V come in units of 32 KB (K: 128 keys x 128 dims, V: 64 keys x 256 dims; heads of 128: whole tiles; of 64: whole tiles of 16 KB)
// through one ring, in the order of their use K0 K1 V0 K2 V1 ..; a unit is filled by one TMA box for each page (at most 64 or 128 rows)
// and 64 dims, issued by as many lanes, which look their pages up a tile ahead. Boxes without a key that the item's tokens see are not
// read.
//
// Masked keys: their scores are replaced, so nothing in a K row that a token does not see matters. Their weights are zero, but zero
// times an infinity or NaN is not: V rows outside the item's keys are zeroed in shared memory (first and last tile), and those that
// only some of its tokens see are searched; one that is not finite is zeroed too and its share added to the rows that see it
// with ordinary arithmetic.
//
// Bound by HBM for few rows (32 sessions of up to 65,536 tokens, 2.18 GB: 345 us in a burst, 6.3 TB/s, and 366 to 390 one after the other, where the
// GPU's power limit takes part of the clock), by the chain of softmax and products for long blocks (2,048 tokens over 32,768: 1.13 TFLOP in
// 1.1 ms in a burst, 1.23 to 1.27 ms one after the other, 0.9 PFLOP/s), by the segments' latencies for small work: about 6 us from the start to
// the last store of a CTA with one tile, of which the page lookup and the first tile's way take 2, softmax and products 3, the part's stores 1;
// the merge is 3 more.
//
// Roles (384 threads, three warpgroups whose register budgets are set with setmaxnreg): warps 0 and 3 = TMA producers, warp 1 = issues
// S = Q K^T and owns the TMEM, warp 2 = issues O += P V, warps 4..11 = softmax. Every wait is bounded; TMEM is
// freed on every path.
#include "pool_plan.cuh"
#include "ptx.cuh"

namespace mkv {
using namespace ptx;

constexpr uint32_t PA_KEYS = 128;
constexpr int PA_THREADS = 384;
constexpr uint32_t PA_SOFTMAX_TID0 = 128;
constexpr long long PA_WAIT_LIMIT = 2000000000ll;
constexpr uint32_t PA_FOLD = 48; // tiles whose products are added up in tensor memory
constexpr float PA_LOG2E = 1.4426950408889634f;
constexpr float PA_BIAS2 = 7.0f; // a row's reference lies so far below its maximum, in base-2 exponents,
constexpr float PA_LAZY2 = 8.0f; // and moves when a tile exceeds that maximum by more than this

template <int DIM> struct PaSizes { // (the tensor maps' boxes go by V_KEYS)
    static constexpr uint32_t UNIT_DIMS = DIM < 128 ? DIM : 128;
    static constexpr uint32_t NUN = DIM / UNIT_DIMS;             // units of a K or V tile
    static constexpr uint32_t BOXES = UNIT_DIMS / 64;            // 64-dim boxes of a unit
    static constexpr uint32_t BOX = PA_KEYS * 128;               // bytes of one of K, [128 keys][64 dims]
    static constexpr uint32_t V_KEYS = PA_KEYS / NUN;            // a unit of V has all dims of so many keys
    static constexpr uint32_t V_BOX = V_KEYS * 128;              // [V_KEYS][64 dims]
    static constexpr uint32_t UNIT = BOXES * BOX;
    static constexpr uint32_t NST = DIM == 256 ? 5 : DIM == 128 ? 6 : 12;
    static constexpr uint32_t OFF_RING = (DIM / 64) * 16384;     // behind Q: [DIM / 64][128 rows][64 dims]
    static constexpr uint32_t NBUF = DIM == 256 ? 2 : 3;         // S buffers
    static constexpr uint32_t LEAD = NBUF - 1;                   // tiles that the scores are ahead of the outputs
    static constexpr uint32_t COL_S = 512 - NBUF * 128;          // behind O
    static constexpr uint32_t OFF_RED = OFF_RING + NST * UNIT;   // [2 halves][128 rows] floats
    static constexpr uint32_t OFF_BAR = OFF_RED + 1024;
    static constexpr uint32_t NBAR = 2 * NST + 3 * NBUF + 1;     // full[NST], empty[NST], s_full[NBUF], p_full[NBUF], pv_done[NBUF], q_full
    static constexpr uint32_t OFF_MISC = OFF_BAR + NBAR * 8;
    static constexpr uint32_t SMEM = OFF_MISC + 64 + 1024;
    static_assert(SMEM <= 232448, "shared memory");
};

struct PaShared {
    uint32_t tmem_base;
    volatile uint32_t abort;
    volatile uint32_t keep; // 1 + the tile whose products are added to O although it is its segment's first
    uint32_t bad[3][4];     // [tile's S buffer]: keys of the tile whose V row is not finite and that not every token sees
};
static_assert(sizeof(PaShared) <= 64, "OFF_MISC");

struct PaArgs {
    const __half *q;
    __half *out;
    int64_t q_stride, out_stride;
    const uint32_t *pages;
    const char *kpages;
    const char *vpages;
    const float *sinks;
    float *scratch;
    float *fold; // of a CTA [DIM / 8][256 threads][4]: O of the tiles that were folded
    uint32_t *status;
    size_t row_bytes;
    float scale2; // scale * log2(e)
    uint32_t page_shift;
};

// Waits for a phase, for a bounded time; false when the time runs out or another thread has given up. The first try is all there is to
// it when the phase is there.
__device__ __forceinline__ bool pa_wait_long(uint32_t bar, uint32_t parity, PaShared *sh, uint32_t *status) {
    const long long t0 = clock64();
    for (;;) {
        if (sh->abort) return false;
#pragma unroll 1
        for (int i = 0; i < 64; i++)
            if (mbar_try_wait(bar, parity)) return true;
        if (clock64() - t0 > PA_WAIT_LIMIT) break;
    }
    sh->abort = 1;
    atomicOr(status, DEV_ERR_WAIT_TIMEOUT);
    return false;
}
__device__ __forceinline__ bool pa_wait(uint32_t bar, uint32_t parity, PaShared *sh, uint32_t *status) {
    return mbar_try_wait(bar, parity) || pa_wait_long(bar, parity, sh, status);
}
// A place of a ring of N and the parity of its current use
template <uint32_t N> struct PaRing {
    uint32_t s = 0, turn = 0;
    __device__ __forceinline__ void next(uint32_t d = 1u) { // d <= N
        s += d;
        if (s >= N) {
            s -= N;
            turn ^= 1u;
        }
    }
};
__device__ __forceinline__ bool half2_not_finite(uint32_t w) { return (w & 0x7c00u) == 0x7c00u || (w & 0x7c000000u) == 0x7c000000u; }

// The tiles of a CTA's segments as one stream.
struct TileStream {
    PlanWalk walk;
    PlanSegment sg;
    uint32_t tile;
    bool more;
    __device__ __forceinline__ TileStream(const PoolPlan &plan) : walk(plan, blockIdx.x, PA_KEYS) { step(); }
    __device__ __forceinline__ void step() {
        more = walk.next(sg);
        tile = sg.a;
    }
    __device__ __forceinline__ bool first() const { return tile == sg.a; }
    __device__ __forceinline__ void next() {
        if (++tile == sg.b) step();
    }
};

template <int DIM>
__global__ void __launch_bounds__(PA_THREADS, 1)
pool_attn_f16_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const __grid_constant__ PoolPlan plan,
                     const __grid_constant__ PaArgs g) {
    using Z = PaSizes<DIM>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t *smem = smem_raw + (smem_base - smem_u32(smem_raw));
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
    const uint32_t ring = smem_base + Z::OFF_RING, bar0 = smem_base + Z::OFF_BAR;
    const uint32_t bar_full = bar0, bar_empty = bar0 + 8u * Z::NST, bar_s_full = bar0 + 16u * Z::NST, bar_p_full = bar_s_full + 8u * Z::NBUF;
    const uint32_t bar_pv_done = bar_p_full + 8u * Z::NBUF, bar_q_full = bar_pv_done + 8u * Z::NBUF;
    PaShared *sh = reinterpret_cast<PaShared *>(smem + Z::OFF_MISC);

    if (tid == 0) {
        for (uint32_t s = 0; s < Z::NST; s++) {
            mbar_init(bar_full + 8u * s, 2); // one arrival per producer
            mbar_init(bar_empty + 8u * s, 1);
        }
        for (uint32_t s = 0; s < Z::NBUF; s++) {
            mbar_init(bar_s_full + 8u * s, 1);
            mbar_init(bar_p_full + 8u * s, 8); // one arrival per softmax warp
            mbar_init(bar_pv_done + 8u * s, 1);
        }
        mbar_init(bar_q_full, 8);
        sh->abort = 0;
        sh->keep = 0;
        for (int i = 0; i < 12; i++) sh->bad[i >> 2][i & 3] = 0;
        fence_barrier_init();
        fence_proxy_async();
    }
    if (warp == 1) tmem_alloc(smem_base + Z::OFF_MISC, 512); // writes sh->tmem_base
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh->tmem_base;
    // Nothing global is touched before the kernel in front has finished. This kernel has begun before that, so what that one may have written (page
    // tables, rotated queries) is not read-only for it, and no load takes the read-only path.
    pdl_wait();
    pdl_launch_dependents();

    // The units of the CTA's T tiles in ring order, whatever segment they belong to: K(0) .. K(LEAD - 1), then K(t + LEAD) and V(t) for
    // each t. In front of K(t) are t + max(t - LEAD, 0) tiles of K and V, in front of V(t) min(t + LEAD + 1, T) + t.
    if (warp < 4u) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == 0 || warp == 3u) {
        // ---------------- TMA producers: every other box of each unit (a page of 16 tokens is 2 KB a box: one warp issues too slowly) ----------------
        // Both go through all units in order: a parity tells a phase from its neighbours only, so whoever waits for a slot has to have
        // waited for its uses before.
        const uint32_t page_tokens = 1u << g.page_shift, box_rows = min(page_tokens, Z::V_KEYS), nrb = PA_KEYS / box_rows, nrbv = Z::V_KEYS / box_rows;
        const uint32_t box = 2u * lane + (warp == 0 ? 0u : 1u), rb = box % nrb, cb = box / nrb, rbv = box % nrbv, cbv = box / nrbv; // this lane's of a unit of K, of V
        PaRing<Z::NST> at;
        uint32_t u = 0;
        TileStream ts(plan);
        struct Tile {
            uint32_t k_row, v_row[Z::NUN]; // in the pool, of this lane's boxes; ~0u where no token of the item sees a key of it
            int x;                         // first column of the head
            bool is;
        };
        auto look_up = [&]() -> Tile { // the stream's tile; the stream moves on
            Tile t;
            t.is = ts.more;
            const PlanItem &it = ts.sg.it;
            const uint32_t key0 = (it.tile0 + ts.tile) * PA_KEYS;
            const uint32_t *pages = g.pages + plan.seq[ts.sg.seq].table;
            auto row = [&](bool mine, uint32_t key) {
                if (!mine || key + box_rows <= it.lo || key >= it.hi) return ~0u;
                return (pages[key >> g.page_shift] << g.page_shift) + (key & (page_tokens - 1u));
            };
            t.k_row = row(t.is && cb < Z::BOXES, key0 + rb * box_rows);
#pragma unroll
            for (uint32_t h = 0; h < Z::NUN; h++) t.v_row[h] = row(t.is && cbv < DIM / 64u, key0 + h * Z::V_KEYS + rbv * box_rows);
            t.x = (int)(ts.sg.kvh * DIM);
            if (t.is) ts.next();
            return t;
        };
        auto load = [&](bool v, const Tile &t) -> bool { // the units of one K or V tile
#pragma unroll
            for (uint32_t h = 0; h < Z::NUN; h++, u++, at.next()) {
                const uint32_t bar = bar_full + 8u * at.s, row = v ? t.v_row[h] : t.k_row;
                if (u >= Z::NST && !__all_sync(0xffffffffu, pa_wait(bar_empty + 8u * at.s, at.turn ^ 1u, sh, g.status))) return false;
                const uint32_t boxes = __popc(__ballot_sync(0xffffffffu, row != ~0u));
                if (lane == 0) mbar_expect_tx(bar, boxes * box_rows * 128u);
                __syncwarp();
                if (row != ~0u)
                    tma_load_2d(ring + at.s * Z::UNIT + (v ? cbv * Z::V_BOX + rbv * box_rows * 128u : cb * Z::BOX + rb * box_rows * 128u), v ? &vmap : &kmap,
                                t.x + (int)(v ? cbv * 64u : h * Z::UNIT_DIMS + cb * 64u), (int)row, bar);
            }
            return true;
        };
        Tile next[Z::LEAD + 2]; // tiles t .. t + LEAD + 1: a page is looked up a tile before it is wanted
        bool ok = true;
#pragma unroll
        for (uint32_t i = 0; i <= Z::LEAD; i++) {
            next[i] = look_up();
            if (i < Z::LEAD && next[i].is) ok = ok && load(false, next[i]);
        }
        while (ok && next[0].is) {
            next[Z::LEAD + 1] = look_up();
            if (next[Z::LEAD].is) ok = load(false, next[Z::LEAD]);
            ok = ok && load(true, next[0]);
#pragma unroll
            for (uint32_t i = 0; i <= Z::LEAD; i++) next[i] = next[i + 1];
        }
    } else if (warp == 1) {
        // ---------------- S = Q K^T ----------------
        if (lane == 0) {
            constexpr uint32_t IDESC = tc_idesc_f16(128, 128, false);
            const uint64_t q_desc = tc_desc_sw128(smem_base, 16, 1024), k_desc = tc_desc_sw128(ring, 16, 1024);
            PaRing<Z::NST> at;
            PaRing<Z::NBUF> buf;
            uint32_t nseg = 0;
            bool ok = true;
            TileStream ts(plan);
            for (uint32_t t = 0; ok && ts.more; t++) {
                if (ts.first()) { // the segment's Q is in shared memory
                    ok = pa_wait(bar_q_full, nseg & 1u, sh, g.status);
                    nseg++;
                }
                // the buffer's weights have been multiplied
                if (t >= Z::NBUF) ok = ok && pa_wait(bar_pv_done + 8u * buf.s, buf.turn ^ 1u, sh, g.status);
                const uint32_t d = tmem + Z::COL_S + 128u * buf.s;
#pragma unroll
                for (uint32_t h = 0; h < Z::NUN; h++) {
                    ok = ok && pa_wait(bar_full + 8u * at.s, at.turn, sh, g.status);
                    tc_fence_after();
                    const uint64_t kd = k_desc + at.s * (Z::UNIT >> 4);
#pragma unroll
                    for (uint32_t ks = 0; ks < Z::UNIT_DIMS / 16u; ks++)
                        tc_mma_f16(d, q_desc + (((h * Z::BOXES + (ks >> 2)) * 16384u + (ks & 3u) * 32u) >> 4), kd + (((ks >> 2) * Z::BOX + (ks & 3u) * 32u) >> 4),
                                   IDESC, (h > 0 || ks > 0) ? 1u : 0u);
                    tc_commit(bar_empty + 8u * at.s);
                    at.next();
                }
                tc_commit(bar_s_full + 8u * buf.s);
                buf.next();
                if (t + 1u > Z::LEAD) at.next(Z::NUN); // over a tile of V
                ts.next();
            }
        }
    } else if (warp == 2) {
        // ---------------- O += P V ----------------
        if (lane == 0) {
            constexpr uint32_t IDESC = tc_idesc_f16(128, DIM, true);
            const uint64_t v_desc = tc_desc_sw128(ring, Z::V_BOX, 1024);
            const uint32_t total = plan.start[blockIdx.x].tiles;
            PaRing<Z::NST> at;
            at.next(min(Z::LEAD + 1u, total) * Z::NUN); // over the first tiles of K
            PaRing<Z::NBUF> buf;
            bool ok = true;
            TileStream ts(plan);
            for (uint32_t t = 0; ok && ts.more; t++) {
                ok = pa_wait(bar_p_full + 8u * buf.s, buf.turn, sh, g.status);
                tc_fence_after();
                const bool over = ts.first() && sh->keep != t + 1u; // the segment's first products overwrite O
                const uint32_t p = tmem + Z::COL_S + 128u * buf.s;
#pragma unroll
                for (uint32_t h = 0; h < Z::NUN; h++) {
                    ok = ok && pa_wait(bar_full + 8u * at.s, at.turn, sh, g.status);
                    tc_fence_after();
                    const uint64_t vd = v_desc + at.s * (Z::UNIT >> 4);
#pragma unroll
                    for (uint32_t ks = 0; ks < Z::V_KEYS / 16u; ks++) { // 16 keys an MMA
                        const uint32_t k16 = h * (Z::V_KEYS / 16u) + ks;
                        tc_mma_f16_ta(tmem, p + 64u * (k16 >> 2) + 8u * (k16 & 3u), vd + ((ks * 2048u) >> 4), IDESC, (!over || k16 > 0) ? 1u : 0u);
                    }
                    tc_commit(bar_empty + 8u * at.s);
                    at.next();
                }
                tc_commit(bar_pv_done + 8u * buf.s);
                buf.next();
                if (t + Z::LEAD + 1u < total) at.next(Z::NUN); // over a tile of K
                ts.next();
            }
        }
    } else if (warp >= 4u) {
        // ---------------- softmax: two threads per row (TMEM lane), 64 keys of a tile and half of the dims of O each ----------------
        asm volatile("setmaxnreg.inc.sync.aligned.u32 224;"); // 128 x 56 + 256 x 224 = the launch's 384 x 168
        const uint32_t q4 = warp & 3u, half = (warp - 4u) >> 2;
        const uint32_t row = 32u * q4 + lane, st = tid - PA_SOFTMAX_TID0; // row: the TMEM lanes this warp may access
        const uint32_t lane_addr = (32u * q4) << 16;
        constexpr uint32_t HD = DIM / 2; // dims of Q and O of a thread
        float *red = reinterpret_cast<float *>(smem + Z::OFF_RED);
        const uint32_t group = plan.group, inv_group = 65536u / group + 1u, tok = row * inv_group >> 16, head = row - tok * group; // (rows < 128, groups <= 64)
        const uint32_t bar_pair = 1u + q4;
        auto arrive = [&](uint32_t bar) { // one arrival per warp, after all its lanes
            __syncwarp();
            if (lane == 0) mbar_arrive(bar);
        };
        auto wait = [&](uint32_t bar, uint32_t parity) {
            pa_wait(bar, parity, sh, g.status);
            __syncwarp();
            tc_fence_after();
        };
        // The products of tile t have completed; for tiles since the newest scores that this warp has waited for. (A parity tells a phase from
        // its neighbours only; those scores were computed behind the products of NBUF tiles earlier.)
        auto wait_pv = [&](uint32_t t) { wait(bar_pv_done + 8u * (t % Z::NBUF), (t / Z::NBUF) & 1u); };
        // Q rows of this quarter, half of the dims; rows beyond the block as zeros where the quarter has rows of it. The first rows are fetched
        // while the scores of the segment in front are still being computed; all go to shared memory once they are.
        constexpr uint32_t CPR = DIM / 16;              // 16-byte chunks of a half row
        constexpr uint32_t RPI = 32 / CPR;              // rows of one access of the warp
        constexpr uint32_t QB = CPR < 8u ? CPR : 8u;    // accesses of a batch
        uint4 qv[QB];
        auto fetch_q = [&](const PlanSegment &sg, uint32_t b) {
            const uint32_t rows = sg.it.ntok * group;
            const __half *src = g.q + (int64_t)(plan.seq[sg.seq].row + sg.it.tok0) * g.q_stride + (size_t)sg.kvh * group * DIM + (half * CPR + lane % CPR) * 8u;
#pragma unroll
            for (uint32_t i = 0; i < QB; i++) {
                const uint32_t r = 32u * q4 + (b * QB + i) * RPI + lane / CPR, t = r * inv_group >> 16;
                qv[i] = make_uint4(0u, 0u, 0u, 0u);
                if (r < rows) qv[i] = *reinterpret_cast<const uint4 *>(src + (int64_t)t * g.q_stride + (r - t * group) * DIM);
            }
        };
        bool clean = false; // this quarter's rows in shared memory are zeros
        auto put_q = [&](const PlanSegment &sg) { // the first batch has been fetched
            const uint32_t c = half * CPR + lane % CPR; // chunk of the row
            // (rows that no segment uses are zeros too: products of nothing draw less power, and the clock is bound by that)
            const bool rows = 32u * q4 < sg.it.ntok * group, write = rows || !clean;
            clean = !rows;
#pragma unroll 1
            for (uint32_t b = 0; b < CPR / QB && write; b++) {
                if (b > 0u) fetch_q(sg, b);
#pragma unroll
                for (uint32_t i = 0; i < QB; i++)
                    *reinterpret_cast<uint4 *>(smem + (c >> 3) * 16384u + swz128(32u * q4 + (b * QB + i) * RPI + lane / CPR, c & 7u)) = qv[i];
            }
            fence_proxy_async();
            arrive(bar_q_full);
        };
        const uint32_t total = plan.start[blockIdx.x].tiles;
        uint32_t t0 = 0; // the segment's first tile
        PlanWalk walk(plan, blockIdx.x, PA_KEYS);
        PlanSegment sg, nx;
        bool more = walk.next(sg);
        fetch_q(sg, 0);
        put_q(sg);
        // The weights of a tile are handed over (finish) when the loads of the next tile's scores are on their way, if those are there.
        PaRing<Z::NBUF> buf;
        uint32_t owed = 0; // the p_full barrier of a tile whose weights are not handed over yet
        auto finish = [&]() {
            if (owed == 0u) return;
            tmem_wait_st();
            tc_fence_before();
            arrive(owed);
            owed = 0;
        };
        // A wait that runs out makes all later ones return at once; the warps go through the same barriers all the same, so that none waits
        // for one that has left.
        while (more) {
            const PlanItem it = sg.it;
            const PlanSeq &sq = plan.seq[sg.seq];
            const uint32_t rows = it.ntok * group;
            const bool active = 32u * q4 < rows; // (warp-uniform, and the same for the two warps of these rows)
            const bool real = row < rows;
            const uint32_t vis = real ? sq.pos + it.tok0 + tok + 1u : 0u; // this row sees klo <= key < vis
            const uint32_t klo = real ? plan_lowest(sq, plan.window, it.tok0 + tok) : 0u;
            // Weights are 2^(s C - m_ref), m_ref = m_raw C - PA_BIAS2 for the score m_raw of a key. l: this thread's keys only.
            float m_raw = NEG_BIG, m_ref = 0.0f, l = 0.0f;
            float m_fold = NEG_BIG; // m_raw of what has been folded
            // this thread's 16-byte piece i of it
            auto folded = [&](uint32_t i) { return reinterpret_cast<float4 *>(g.fold) + ((blockIdx.x * (DIM / 8u) + i) * 256u + threadIdx.x - PA_SOFTMAX_TID0); };
            auto add_folded = [&](uint32_t (&o)[32], uint32_t c0) { // o: 32 dims from c0 on of this thread's
                if (!(m_fold > NEG_TEST)) return; // (none yet, or no key seen)
                const float f = exp2f((m_fold - m_raw) * g.scale2);
#pragma unroll
                for (uint32_t i = 0; i < 8u; i++) {
                    const float4 x = __ldcg(folded(c0 / 4u + i));
                    o[4 * i] = __float_as_uint(fmaf(x.x, f, __uint_as_float(o[4 * i])));
                    o[4 * i + 1] = __float_as_uint(fmaf(x.y, f, __uint_as_float(o[4 * i + 1])));
                    o[4 * i + 2] = __float_as_uint(fmaf(x.z, f, __uint_as_float(o[4 * i + 2])));
                    o[4 * i + 3] = __float_as_uint(fmaf(x.w, f, __uint_as_float(o[4 * i + 3])));
                }
            };
            const uint32_t end = t0 + (sg.b - sg.a);
            more = walk.next(nx);
            for (uint32_t t = t0; t < end; t++, buf.next()) {
                const uint32_t key0 = (it.tile0 + sg.a + (t - t0)) * PA_KEYS, s_col = tmem + lane_addr + Z::COL_S + 128u * buf.s + 64u * half;
                const bool edge = key0 < it.all_lo || key0 + PA_KEYS > it.all_hi; // some row does not see some key
                const bool last = t + 1u == end && more;
                if (last) fetch_q(nx, 0);
                const uint32_t bar_s = bar_s_full + 8u * buf.s;
                if (!__all_sync(0xffffffffu, mbar_test(bar_s, buf.turn))) {
                    finish();
                    wait(bar_s, buf.turn);
                }
                tc_fence_after();
                uint32_t sr[2][32];
                if (active) {
                    tmem_ld32(s_col, sr[0]);
                    tmem_ld32(s_col + 32u, sr[1]);
                }
                finish();
                if (last) put_q(nx); // the segment's scores are all there: its Q may go
                bool bad_any = false;
                if (edge) { // (the same for the eight warps)
                    const uint32_t uv = (min(t + Z::LEAD + 1u, total) + t) * Z::NUN; // units in front of this tile's V
                    // The unit that a slot held before must be known to have come. Those of K(t) and in front have; with fewer than three tiles
                    // of slots that may be one of V(t - 1).
                    if (Z::NST < 3u * Z::NUN && t > 0u) wait_pv(t - 1u);
                    for (uint32_t h = 0; h < Z::NUN; h++) wait(bar_full + 8u * ((uv + h) % Z::NST), ((uv + h) / Z::NST) & 1u);
                    auto v_chunk = [&](uint32_t r, uint32_t c) { // 8 dims of key r
                        const uint32_t unit = (uv + r / Z::V_KEYS) % Z::NST;
                        return reinterpret_cast<uint4 *>(smem + Z::OFF_RING + unit * Z::UNIT + (c >> 3) * Z::V_BOX + swz128(r % Z::V_KEYS, c & 7u));
                    };
                    // rows of the tile: [0, z0) and [z1, 128) are outside the item's keys; [z0, p0) and [p1, z1) are not seen by all
                    auto in_tile = [&](uint32_t key) { return key > key0 ? min(key - key0, PA_KEYS) : 0u; };
                    const uint32_t z0 = in_tile(it.lo), z1 = in_tile(it.hi), p0 = max(z0, min(z1, in_tile(it.all_lo))), p1 = max(p0, min(z1, in_tile(it.all_hi)));
                    for (uint32_t idx = st; idx < (z0 + PA_KEYS - z1) * (DIM / 8u); idx += 256u) {
                        const uint32_t r = idx / (DIM / 8u);
                        *v_chunk(r < z0 ? r : r - z0 + z1, idx % (DIM / 8u)) = make_uint4(0u, 0u, 0u, 0u);
                    }
                    bool found = false;
                    for (uint32_t idx = st; idx < (p0 - z0 + z1 - p1) * (DIM / 8u); idx += 256u) {
                        const uint32_t i = idx / (DIM / 8u), r = i < p0 - z0 ? z0 + i : i - (p0 - z0) + p1;
                        const uint4 v = *v_chunk(r, idx % (DIM / 8u));
                        if (half2_not_finite(v.x) || half2_not_finite(v.y) || half2_not_finite(v.z) || half2_not_finite(v.w)) {
                            atomicOr(&sh->bad[buf.s][r >> 5], 1u << (r & 31u));
                            found = true;
                        }
                    }
                    if (p0 - z0 + z1 - p1 != 0u) {
                        bad_any = named_bar_or(5, 256, found);
                        for (uint32_t idx = st; bad_any && idx < PA_KEYS * (DIM / 8u); idx += 256u) {
                            const uint32_t r = idx / (DIM / 8u);
                            if (sh->bad[buf.s][r >> 5] >> (r & 31u) & 1u) *v_chunk(r, idx % (DIM / 8u)) = make_uint4(0u, 0u, 0u, 0u);
                        }
                    }
                    fence_proxy_async();
                }
                if (active) {
                    tmem_wait_ld();
                    // work in base-2 exponents: e^(s scale) = 2^(s C), C = scale log2(e)
                    float mt[4] = {NEG_BIG, NEG_BIG, NEG_BIG, NEG_BIG};
                    if (edge) {
                        // the keys of this half that the row sees, a bit each
                        const uint32_t k = key0 + 64u * half;
                        auto upto = [&](uint32_t key) { return key <= k ? 0ull : key >= k + 64u ? ~0ull : (1ull << (key - k)) - 1ull; };
                        const uint64_t see = upto(vis) & ~upto(klo);
                        const uint32_t bits[2] = {(uint32_t)see, (uint32_t)(see >> 32)};
#pragma unroll
                        for (int h = 0; h < 2; h++)
#pragma unroll
                            for (int c = 0; c < 32; c++)
                                if (!(bits[h] & (1u << c))) sr[h][c] = 0xff800000u; // -infinity
                    }
#pragma unroll
                    for (int h = 0; h < 2; h++)
#pragma unroll
                        for (int c = 0; c < 32; c += 2) mt[(c >> 1) & 3] = max3(mt[(c >> 1) & 3], __uint_as_float(sr[h][c]), __uint_as_float(sr[h][c + 1]));
                    float mx = max3(fmaxf(mt[0], mt[1]), mt[2], mt[3]);
                    // The reference moves for the first tile with a key and when the tile exceeds it by more than PA_LAZY2. The two warps that share
                    // these 32 rows vote; only then they exchange maxima.
                    float cf = 1.0f;
                    auto moves = [&]() { return mx > NEG_TEST && (m_raw < NEG_TEST || (mx - m_raw) * g.scale2 > PA_LAZY2); };
                    if (pair_bar_or(bar_pair, moves())) {
                        red[128u * half + row] = mx;
                        pair_bar_sync(bar_pair);
                        mx = fmaxf(mx, red[128u * (half ^ 1u) + row]);
                        if (moves()) {
                            cf = m_raw > NEG_TEST ? exp2f((m_raw - mx) * g.scale2) : 1.0f;
                            m_raw = mx;
                            m_ref = mx * g.scale2 - PA_BIAS2;
                        }
                    }
                    float neg_m = -m_ref;
                    // Half a step of m_ref is 2^-5 at 2^20, but with the scores of rows that are thousands long it would take weights out of f16's
                    // range; there the difference of the scores comes first.
                    const bool far = fabsf(m_ref) > 1048576.0f;
                    if (far) {
                        neg_m = PA_BIAS2;
#pragma unroll
                        for (int h = 0; h < 2; h++)
#pragma unroll
                            for (int c = 0; c < 32; c++) sr[h][c] = __float_as_uint(__uint_as_float(sr[h][c]) - m_raw);
                    }
                    const uint64_t c2 = pack2(g.scale2, g.scale2), m2 = pack2(neg_m, neg_m);
                    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f}; // of the weights as the products take them
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        uint32_t ph[16]; // 32 weights as f16 pairs
#pragma unroll
                        for (int c = 0; c < 32; c += 2) {
                            float x0, x1;
                            unpack2(fma2(pack2(__uint_as_float(sr[h][c]), __uint_as_float(sr[h][c + 1])), c2, m2), x0, x1);
                            const __half2 hp = __floats2half2_rn(ex2(x0), ex2(x1));
                            ph[c >> 1] = *reinterpret_cast<const uint32_t *>(&hp);
                            add_f16x2(sum[c & 2], sum[(c & 2) + 1], ph[c >> 1]);
                        }
                        tmem_st16(s_col + 16u * h, ph);
                    }
                    l = l * cf + ((sum[0] + sum[2]) + (sum[1] + sum[3]));
                    const bool moved = t > t0 && __any_sync(0xffffffffu, cf != 1.0f);
                    const bool fold = t > t0 && (t - t0) % PA_FOLD == 0u;
                    if (moved || bad_any || fold) { // this warp's rows of O (rare)
                        if (t > t0) wait_pv(t - 1u);
                        const bool adds = m_fold > NEG_TEST && m_fold == m_raw; // (each piece has one thread, and the order of its additions)
#pragma unroll 1
                        for (uint32_t c0 = HD * half; c0 < HD * half + HD; c0 += 32u) {
                            uint32_t orow[32];
                            if (t > t0) {
                                tmem_ld32(tmem + lane_addr + c0, orow);
                                tmem_wait_ld();
                            }
#pragma unroll
                            for (int c = 0; c < 32; c++) orow[c] = t > t0 ? __float_as_uint(__uint_as_float(orow[c]) * cf) : 0u;
                            if (fold) { // O goes on from zero
                                if (!adds) add_folded(orow, c0 - HD * half);
#pragma unroll
                                for (uint32_t i = 0; i < 8u; i++) {
                                    const float4 x = make_float4(__uint_as_float(orow[4 * i]), __uint_as_float(orow[4 * i + 1]), __uint_as_float(orow[4 * i + 2]),
                                                                 __uint_as_float(orow[4 * i + 3]));
                                    float4 *to = folded((c0 - HD * half) / 4u + i);
                                    if (adds) red_add4(to, x);
                                    else *to = x;
                                }
#pragma unroll
                                for (int c = 0; c < 32; c++) orow[c] = 0u;
                            }
                            // rows of V that are not finite, zero in shared memory: w v for the tokens that see them
                            for (uint32_t r = 0; bad_any && r < PA_KEYS; r++) {
                                const uint32_t key = key0 + r;
                                if (!(sh->bad[buf.s][r >> 5] >> (r & 31u) & 1u) || !real || key < klo || key >= vis) continue;
                                const size_t page = g.pages[sq.table + (key >> g.page_shift)], off = key & ((1u << g.page_shift) - 1u);
                                const __half *v = reinterpret_cast<const __half *>(g.vpages + ((page << g.page_shift) + off) * g.row_bytes) + (size_t)sg.kvh * DIM + c0;
                                const __half *k = reinterpret_cast<const __half *>(g.kpages + ((page << g.page_shift) + off) * g.row_bytes) + (size_t)sg.kvh * DIM;
                                const __half *q = g.q + (int64_t)(sq.row + it.tok0 + tok) * g.q_stride + (size_t)(sg.kvh * group + head) * DIM;
                                float s = 0.0f;
                                for (int d = 0; d < DIM; d++) s = fmaf(__half2float(q[d]), __half2float(k[d]), s);
                                const float w = __half2float(__float2half_rn(exp2f(fmaf(far ? s - m_raw : s, g.scale2, neg_m))));
#pragma unroll
                                for (int c = 0; c < 32; c++) orow[c] = __float_as_uint(fmaf(w, __half2float(v[c]), __uint_as_float(orow[c])));
                            }
                            tmem_st32(tmem + lane_addr + c0, orow);
                        }
                        if (fold) m_fold = m_raw;
                    }
                }
                if (bad_any) {
                    named_bar_sync(5, 256);
                    // Noted again NBUF tiles on: those scores are behind this tile's product, which is behind the p_full of the warp that clears.
                    if (st < 4u) sh->bad[buf.s][st] = 0u;
                    if (t == t0 && st == 0u) sh->keep = t + 1u; // what was put into O stays
                }
                owed = bar_p_full + 8u * buf.s;
            }
            finish();
            // ---------------- end of the segment ----------------
            wait_pv(end - 1u); // (the next segment's first scores are computed meanwhile)
            if (active) {
                red[128u * half + row] = l;
                pair_bar_sync(bar_pair);
                const float l_all = red[row] + red[128u + row];
                const bool seen = real && klo < vis;
                // A lane has 64 bytes of its row at a time. Four lanes exchange them, so that each has 16 bytes of each of their four rows and a
                // store of the warp touches eight lines instead of 32.
                const uint32_t q = lane & 3u;
                auto trade = [&](uint32_t (&w)[4][4]) { // chunk and lane change places, a bit of their numbers at a time
#pragma unroll
                    for (uint32_t m = 1u; m <= 2u; m <<= 1)
#pragma unroll
                        for (uint32_t c = 0; c < 4u; c++) {
                            if (c & m) continue;
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                const uint32_t got = __shfl_xor_sync(0xffffffffu, (q & m) ? w[c][e] : w[c | m][e], m);
                                if (q & m) w[c][e] = got;
                                else w[c | m][e] = got;
                            }
                        }
                };
                if (sg.whole) {
                    // out[token][head][:] = O / (l + sink)
                    float den = l_all;
                    if (g.sinks && real) den += exp2f(g.sinks[sg.kvh * group + head] * PA_LOG2E - m_ref);
                    const float inv = 1.0f / den;
                    __half *dst[4];
#pragma unroll
                    for (uint32_t i = 0; i < 4u; i++) {
                        const uint32_t r = (row & ~3u) + i, t = r * inv_group >> 16;
                        dst[i] = r < rows ? g.out + (int64_t)(sq.row + it.tok0 + t) * g.out_stride + (size_t)(sg.kvh * group + (r - t * group)) * DIM + HD * half + 8u * q : nullptr;
                    }
#pragma unroll 1
                    for (uint32_t c0 = 0; c0 < HD; c0 += 32u) {
                        uint32_t orow[32];
                        tmem_ld32(tmem + lane_addr + HD * half + c0, orow);
                        tmem_wait_ld();
                        add_folded(orow, c0);
                        uint32_t w[4][4]; // [16-byte chunk][word]
#pragma unroll
                        for (int c = 0; c < 32; c += 2) {
                            const __half2 h2 = __floats2half2_rn(seen ? __uint_as_float(orow[c]) * inv : 0.0f, seen ? __uint_as_float(orow[c + 1]) * inv : 0.0f);
                            w[c >> 3][(c >> 1) & 3] = *reinterpret_cast<const uint32_t *>(&h2);
                        }
                        trade(w);
#pragma unroll
                        for (uint32_t i = 0; i < 4u; i++)
                            if (dst[i]) *reinterpret_cast<uint4 *>(dst[i] + c0) = make_uint4(w[i][0], w[i][1], w[i][2], w[i][3]);
                    }
                } else {
                    // a part: maximum, sum and O as they are, for the merge
                    float *ps = g.scratch + part_slot(blockIdx.x, sg.part) * part_floats(DIM);
                    if (half == 0u && real) *reinterpret_cast<float2 *>(ps + 128u * DIM + 2u * row) = make_float2(m_raw > NEG_TEST ? m_ref : NEG_BIG, seen ? l_all : -1.0f);
                    // The exchange pays where many rows are stored (six blocks of up to 109 tokens of six heads: the call takes 14.1 us, without it
                    // 17.3); one token's rows are few lines either way, and sooner stored as they are (12.1 us, with it 13.2).
                    const bool many = rows > 32u;
                    ps += (size_t)(many ? row & ~3u : row) * DIM + HD * half + (many ? 4u * q : 0u);
#pragma unroll 1
                    for (uint32_t c0 = 0; c0 < HD; c0 += 32u) {
                        uint32_t orow[32];
                        tmem_ld32(tmem + lane_addr + HD * half + c0, orow);
                        tmem_wait_ld();
                        add_folded(orow, c0);
                        if (!many) {
                            if (real)
#pragma unroll
                                for (int c = 0; c < 32; c += 4) *reinterpret_cast<uint4 *>(ps + c0 + c) = make_uint4(orow[c], orow[c + 1], orow[c + 2], orow[c + 3]);
                            continue;
                        }
#pragma unroll
                        for (uint32_t k = 0; k < 2u; k++) {
                            uint32_t w[4][4];
#pragma unroll
                            for (int c = 0; c < 16; c++) w[c >> 2][c & 3] = orow[16u * k + c];
                            trade(w);
#pragma unroll
                            for (uint32_t i = 0; i < 4u; i++)
                                if ((row & ~3u) + i < rows) *reinterpret_cast<uint4 *>(ps + i * DIM + c0 + 16u * k) = make_uint4(w[i][0], w[i][1], w[i][2], w[i][3]);
                        }
                    }
                }
                tc_fence_before();
                pair_bar_sync(bar_pair); // O and red[] are free for the next segment
            }
            t0 = end;
            sg = nx;
        }
    }

    // ---------------- teardown ----------------
    tc_fence_before();
    __syncwarp();
    if (sh->abort) { // a wait ran out somewhere: give copies already issued into this CTA's shared memory time to land
        const long long t0 = clock64();
        while (clock64() - t0 < 200000000ll) __nanosleep(1000);
    }
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

template <int DIM> static mkv_status launch_dim(Pool *p, int layer, const PoolPlan &plan, const PaArgs &g) {
    PdlLaunch l(p->ctx, dim3(plan.ctas), PA_THREADS, PaSizes<DIM>::SMEM);
    MKV_CUDA(cudaLaunchKernelEx(&l.cfg, pool_attn_f16_kernel<DIM>, p->maps[2 * (size_t)layer], p->maps[2 * (size_t)layer + 1], plan, g));
    p->ctx->launches++;
    return MKV_OK;
}

mkv_status launch_pool_attn_f16(Pool *p, int layer, const PoolPlan &plan, const PoolAttn &a) {
    PaArgs g;
    g.q = static_cast<const __half *>(a.q);
    g.out = static_cast<__half *>(a.out);
    g.q_stride = a.q_stride;
    g.out_stride = a.out_stride;
    g.pages = p->table;
    g.kpages = p->layer_ptr(layer, 0);
    g.vpages = p->layer_ptr(layer, 1);
    g.sinks = a.sinks;
    g.scratch = p->scratch;
    g.fold = p->scratch + 2u * pool_attn_ctas(p) * part_floats((uint32_t)p->desc.head_dim);
    g.status = p->ctx->dev_status;
    g.row_bytes = p->row_bytes;
    g.scale2 = a.scale * PA_LOG2E;
    g.page_shift = (uint32_t)__builtin_ctz(p->desc.page_tokens);
    switch (p->desc.head_dim) {
    case 64: return launch_dim<64>(p, layer, plan, g);
    case 128: return launch_dim<128>(p, layer, plan, g);
    default: return launch_dim<256>(p, layer, plan, g);
    }
}

mkv_status pool_attn_f16_setup(Pool *) {
    MKV_CUDA(cudaFuncSetAttribute(pool_attn_f16_kernel<64>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)PaSizes<64>::SMEM));
    MKV_CUDA(cudaFuncSetAttribute(pool_attn_f16_kernel<128>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)PaSizes<128>::SMEM));
    MKV_CUDA(cudaFuncSetAttribute(pool_attn_f16_kernel<256>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)PaSizes<256>::SMEM));
    return MKV_OK;
}

} // namespace mkv
