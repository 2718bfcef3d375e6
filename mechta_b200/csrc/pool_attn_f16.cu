// Attention of blocks of new tokens over f16 pages on the 5th-generation tensor cores: tcgen05.mma with the scores, the weights
// and the output in tensor memory, queries in shared memory, K/V tiles staged by TMA page by page.
//   out_t = sum_k e^(s_k - M) v_k / (sum_k e^(s_k - M) + e^(sink - M)),  s_k = scale q_t . k_k
//
// An item is 128 rows = the query heads of one KV head for 128 / group tokens (row = token * group + head). Per tile of 128 keys:
//   S = Q K^T   A = Q (shared memory), B = the K tile as TMA left it (K-major)
//   P = e^(S - reference maximum) as f16, back into the columns of S
//   O += P V    A = P (tensor memory), B = the V tile as TMA left it (N-major)
// One pass: the reference maximum of a row moves only when a tile exceeds it by more than 8 (then O is rescaled; weights stay
// below e^8, far from f16's end), the sum is kept in f32. Two S buffers: the tensor cores compute the scores of a tile while the
// one in front is in softmax. TMEM: O = columns 0 .. DIM - 1, S = 256 .. 383 and 384 .. 511.
//
// K and V come in units of 128 keys x 128 dims (32 KB; 64 dims: 16 KB) through one ring, in the order of their use
// K0 K1 V0 K2 V1 ..; a unit is filled by one TMA box for each page (or half page of 256) and 64 dims, issued by as many lanes, each of
// which looks its page up a tile ahead. Boxes without a key that the item's tokens see are not read.
//
// Masked keys: their scores are replaced, so nothing in a K row that a token does not see matters. Their weights are zero, but zero
// times an infinity or NaN is not: V rows outside the item's keys are zeroed in shared memory (first and last tile), and those that
// only some of its tokens see are searched; one that is not finite is zeroed too and its share added to the rows that see it
// with ordinary arithmetic.
//
// Roles (320 threads): warp 0 = TMA producer, warp 1 = MMA issuer (one thread) and TMEM owner, warps 2..9 = softmax, two threads per
// row (64 of a tile's keys each). Every wait is bounded; TMEM is freed on every path.
#include "pool_plan.cuh"
#include "ptx.cuh"

namespace mkv {
using namespace ptx;

constexpr uint32_t PA_KEYS = 128;
constexpr int PA_THREADS = 320;
constexpr long long PA_WAIT_LIMIT = 2000000000ll;
constexpr float PA_LOG2E = 1.4426950408889634f;
constexpr float PA_LAZY2 = 8.0f * PA_LOG2E;
constexpr uint32_t PA_COL_S = 256;

template <int DIM> struct PaSizes {
    static constexpr uint32_t UNIT_DIMS = DIM < 128 ? DIM : 128;
    static constexpr uint32_t NUN = DIM / UNIT_DIMS;             // units of a K or V tile
    static constexpr uint32_t BOXES = UNIT_DIMS / 64;            // 64-dim boxes of a unit
    static constexpr uint32_t BOX = PA_KEYS * 128;               // bytes of one, [128 keys][64 dims]
    static constexpr uint32_t UNIT = BOXES * BOX;
    static constexpr uint32_t NST = DIM == 256 ? 5 : DIM == 128 ? 6 : 12;
    static constexpr uint32_t OFF_RING = (DIM / 64) * 16384;     // behind Q: [DIM / 64][128 rows][64 dims]
    static constexpr uint32_t OFF_RED = OFF_RING + NST * UNIT;   // [2 halves][128 rows] floats
    static constexpr uint32_t OFF_BAR = OFF_RED + 1024;
    static constexpr uint32_t NBAR = 2 * NST + 6;                // full[NST], empty[NST], s_full[2], p_full[2], pv_done, q_full
    static constexpr uint32_t OFF_MISC = OFF_BAR + NBAR * 8;
    static constexpr uint32_t SMEM = OFF_MISC + 64 + 1024;
    static_assert(SMEM <= 232448, "shared memory");
};

struct PaShared {
    uint32_t tmem_base;
    volatile uint32_t abort;
    uint32_t bad[2][4]; // [tile parity]: keys of the tile whose V row is not finite and that not every token sees
};

struct PaArgs {
    const __half *q;
    __half *out;
    int64_t q_stride, out_stride;
    const uint32_t *pages;
    const char *vpages;
    const float *sinks;
    float *scratch;
    uint32_t *status;
    size_t row_bytes;
    float scale2; // scale * log2(e)
    uint32_t page_shift;
};

__device__ __forceinline__ bool pa_wait(uint32_t bar, uint32_t parity, PaShared *sh, uint32_t *status) {
    if (sh->abort) return false;
    if (mbar_wait_bounded(bar, parity, PA_WAIT_LIMIT)) return true;
    sh->abort = 1;
    atomicOr(status, DEV_ERR_WAIT_TIMEOUT);
    return false;
}
__device__ __forceinline__ bool half2_not_finite(uint32_t w) { return (w & 0x7c00u) == 0x7c00u || (w & 0x7c000000u) == 0x7c000000u; }

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
    const uint32_t bar_full = bar0, bar_empty = bar0 + 8u * Z::NST, bar_s_full = bar0 + 16u * Z::NST, bar_p_full = bar_s_full + 16u;
    const uint32_t bar_pv_done = bar_p_full + 16u, bar_q_full = bar_pv_done + 8u;
    PaShared *sh = reinterpret_cast<PaShared *>(smem + Z::OFF_MISC);

    if (tid == 0) {
        for (uint32_t s = 0; s < 2u * Z::NST; s++) mbar_init(bar0 + 8u * s, 1);
        for (uint32_t s = 0; s < 2u; s++) {
            mbar_init(bar_s_full + 8u * s, 1);
            mbar_init(bar_p_full + 8u * s, 8); // one arrival per softmax warp
        }
        mbar_init(bar_pv_done, 1);
        mbar_init(bar_q_full, 8);
        sh->abort = 0;
        for (int i = 0; i < 8; i++) sh->bad[i >> 2][i & 3] = 0;
        fence_barrier_init();
        fence_proxy_async();
    }
    if (warp == 1) tmem_alloc(smem_base + Z::OFF_MISC, 512); // writes sh->tmem_base
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh->tmem_base;
    pdl_wait(); // nothing global is touched before the kernel in front has finished
    pdl_launch_dependents();

    // The units of a segment of n tiles in ring order: K0, then K(j + 1) and V(j) for each j. u counts units, g_ tiles, both across the
    // CTA's segments.
    if (warp == 0) {
        // ---------------- TMA producer ----------------
        const uint32_t page_tokens = 1u << g.page_shift, box_rows = min(page_tokens, PA_KEYS), nrb = PA_KEYS / box_rows;
        const uint32_t rb = lane % nrb, cb = lane / nrb; // this lane's row box and 64-dim box of a unit
        uint32_t u = 0;
        PlanWalk walk(plan, blockIdx.x, PA_KEYS);
        PlanSegment sg;
        bool ok = true;
        while (ok && walk.next(sg)) {
            const PlanItem &it = sg.it;
            const uint32_t *pages = g.pages + plan.seq[sg.seq].table;
            // the row in the pool of the lane's row box of a tile, ~0u where no token of the item sees a key of it
            auto look_up = [&](uint32_t j) -> uint32_t {
                const uint32_t key = (it.tile0 + j) * PA_KEYS + rb * box_rows;
                if (cb >= Z::BOXES || j >= sg.b || key + box_rows <= it.lo || key >= it.hi) return ~0u;
                return (__ldg(pages + (key >> g.page_shift)) << g.page_shift) + (key & (page_tokens - 1u));
            };
            auto load = [&](const CUtensorMap *map, uint32_t row) -> bool { // the units of one K or V tile
#pragma unroll
                for (uint32_t h = 0; h < Z::NUN; h++, u++) {
                    const uint32_t s = u % Z::NST, bar = bar_full + 8u * s;
                    if (u >= Z::NST && !__all_sync(0xffffffffu, pa_wait(bar_empty + 8u * s, ((u / Z::NST) - 1u) & 1u, sh, g.status))) return false;
                    const uint32_t boxes = __popc(__ballot_sync(0xffffffffu, row != ~0u));
                    if (lane == 0) mbar_expect_tx(bar, boxes * box_rows * 128u);
                    __syncwarp();
                    if (row != ~0u)
                        tma_load_2d(ring + s * Z::UNIT + cb * Z::BOX + rb * box_rows * 128u, map, (int)(sg.kvh * DIM + h * Z::UNIT_DIMS + cb * 64u), (int)row, bar);
                }
                return true;
            };
            uint32_t row = look_up(sg.a), ahead = look_up(sg.a + 1u);
            ok = load(&kmap, row);
            for (uint32_t j = sg.a; ok && j < sg.b; j++) {
                const uint32_t later = look_up(j + 2u);
                if (j + 1u < sg.b) ok = load(&kmap, ahead);
                ok = ok && load(&vmap, row);
                row = ahead;
                ahead = later;
            }
        }
    } else if (warp == 1) {
        // ---------------- MMA issuer ----------------
        if (lane == 0) {
            constexpr uint32_t IDESC_QK = tc_idesc_f16(128, 128, false);
            constexpr uint32_t IDESC_PV = tc_idesc_f16(128, Z::UNIT_DIMS, true);
            uint32_t u = 0, gt = 0, nseg = 0;
            auto qk = [&](uint32_t t) -> bool { // S = Q K^T of tile t
#pragma unroll
                for (uint32_t h = 0; h < Z::NUN; h++, u++) {
                    const uint32_t s = u % Z::NST;
                    if (!pa_wait(bar_full + 8u * s, (u / Z::NST) & 1u, sh, g.status)) return false;
                    tc_fence_after();
#pragma unroll
                    for (uint32_t ks = 0; ks < Z::UNIT_DIMS / 16u; ks++) {
                        const uint64_t a = tc_desc_sw128(smem_base + (h * Z::BOXES + (ks >> 2)) * 16384u + (ks & 3u) * 32u, 16, 1024);
                        const uint64_t b = tc_desc_sw128(ring + s * Z::UNIT + (ks >> 2) * Z::BOX + (ks & 3u) * 32u, 16, 1024);
                        tc_mma_f16(tmem + PA_COL_S + 128u * (t & 1u), a, b, IDESC_QK, (h > 0 || ks > 0) ? 1u : 0u);
                    }
                    tc_commit(bar_empty + 8u * s);
                }
                tc_commit(bar_s_full + 8u * (t & 1u));
                return true;
            };
            PlanWalk walk(plan, blockIdx.x, PA_KEYS);
            PlanSegment sg;
            bool ok = true;
            while (ok && walk.next(sg)) {
                if (!(ok = pa_wait(bar_q_full, nseg & 1u, sh, g.status))) break;
                tc_fence_after();
                nseg++;
                const uint32_t n = sg.b - sg.a;
                if (!(ok = qk(gt))) break;
                for (uint32_t j = 0; j < n; j++, gt++) {
                    if (j + 1u < n && !(ok = qk(gt + 1u))) break; // the next tile's scores while this one is in softmax
                    if (!(ok = pa_wait(bar_p_full + 8u * (gt & 1u), (gt >> 1) & 1u, sh, g.status))) break;
                    tc_fence_after();
                    const uint32_t p = tmem + PA_COL_S + 128u * (gt & 1u);
#pragma unroll
                    for (uint32_t h = 0; h < Z::NUN; h++, u++) {
                        const uint32_t s = u % Z::NST;
                        if (!(ok = pa_wait(bar_full + 8u * s, (u / Z::NST) & 1u, sh, g.status))) break;
                        tc_fence_after();
#pragma unroll
                        for (uint32_t ks = 0; ks < 8u; ks++) { // 16 keys an MMA
                            const uint64_t b = tc_desc_sw128(ring + s * Z::UNIT + ks * 2048u, Z::BOX, 1024);
                            tc_mma_f16_ta(tmem + h * Z::UNIT_DIMS, p + 64u * (ks >> 2) + 8u * (ks & 3u), b, IDESC_PV, (j > 0 || ks > 0) ? 1u : 0u);
                        }
                        tc_commit(bar_empty + 8u * s);
                    }
                    if (!ok) break;
                    tc_commit(bar_pv_done);
                }
            }
        }
    } else {
        // ---------------- softmax: two threads per row (TMEM lane), 64 keys of a tile and half of the dims of O each ----------------
        const uint32_t q4 = warp & 3u, half = (warp - 2u) >> 2;
        const uint32_t row = 32u * q4 + lane; // the TMEM lanes this warp may access
        const uint32_t lane_addr = (32u * q4) << 16;
        constexpr uint32_t HD = DIM / 2;      // dims of O of a thread
        float *red = reinterpret_cast<float *>(smem + Z::OFF_RED);
        const uint32_t group = plan.group, tok = row / group, head = row % group;
        auto arrive = [&](uint32_t bar) { // one arrival per warp, after all its lanes
            __syncwarp();
            if (lane == 0) mbar_arrive(bar);
        };
        // The products of tile t have completed. A parity tells a phase from its neighbours only, and the tile in front need not have been
        // waited for yet.
        auto wait_pv = [&](uint32_t t) {
            if (t > 0u) pa_wait(bar_pv_done, (t - 1u) & 1u, sh, g.status);
            pa_wait(bar_pv_done, t & 1u, sh, g.status);
            __syncwarp();
            tc_fence_after();
        };
        // Q rows of this warp, half of the dims, to shared memory; rows beyond the block as zeros where the warp has rows of it.
        auto load_q = [&](const PlanSegment &sg) {
            constexpr uint32_t CPR = DIM / 16; // 16-byte chunks of a half row
            constexpr uint32_t RPI = 32 / CPR; // rows of one access of the warp
            const uint32_t rows = sg.it.ntok * group;
            if (32u * q4 < rows) {
                const __half *src = g.q + (int64_t)(plan.seq[sg.seq].row + sg.it.tok0) * g.q_stride + (size_t)sg.kvh * group * DIM;
                const uint32_t c = half * CPR + lane % CPR; // chunk of the row
#pragma unroll 8
                for (uint32_t i = 0; i < CPR; i++) {
                    const uint32_t r = 32u * q4 + i * RPI + lane / CPR, t = r / group;
                    uint4 v = make_uint4(0u, 0u, 0u, 0u);
                    if (r < rows) v = __ldg(reinterpret_cast<const uint4 *>(src + (int64_t)t * g.q_stride + (r - t * group) * DIM + c * 8u));
                    *reinterpret_cast<uint4 *>(smem + (c >> 3) * 16384u + swz128(r, c & 7u)) = v;
                }
            }
            fence_proxy_async();
            arrive(bar_q_full);
        };
        uint32_t gt = 0, u = 0;
        PlanWalk walk(plan, blockIdx.x, PA_KEYS);
        PlanSegment sg, nx;
        bool more = walk.next(sg);
        if (more) load_q(sg);
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
            float m_ref = NEG_BIG, l_run = 0.0f; // l_run: this thread's 64 keys of every tile only
            const uint32_t n = sg.b - sg.a;
            for (uint32_t j = 0; j < n; j++, gt++) {
                const uint32_t key0 = (it.tile0 + sg.a + j) * PA_KEYS, s_col = tmem + lane_addr + PA_COL_S + 128u * (gt & 1u);
                // units in front of this tile's V: K(0 .. min(j + 1, n - 1)) and V(0 .. j - 1)
                const uint32_t uv = u + (min(j + 2u, n) + j) * Z::NUN;
                const bool edge = key0 < it.all_lo || key0 + PA_KEYS > it.all_hi; // some row does not see some key
                pa_wait(bar_s_full + 8u * (gt & 1u), (gt >> 1) & 1u, sh, g.status);
                __syncwarp();
                tc_fence_after();
                bool bad_any = false;
                uint32_t bad[4] = {0u, 0u, 0u, 0u};
                if (edge) { // (the same for all eight warps)
                    for (uint32_t h = 0; h < Z::NUN; h++) pa_wait(bar_full + 8u * ((uv + h) % Z::NST), ((uv + h) / Z::NST) & 1u, sh, g.status);
                    __syncwarp();
                    const uint32_t st = tid - 64u;
                    for (uint32_t idx = st; idx < PA_KEYS * (DIM / 8u); idx += 256u) {
                        const uint32_t r = idx / (DIM / 8u), c = idx % (DIM / 8u), key = key0 + r; // chunk of 8 dims of key r
                        const uint32_t unit = (uv + c / (Z::UNIT_DIMS / 8u)) % Z::NST, uc = c % (Z::UNIT_DIMS / 8u);
                        uint4 *at = reinterpret_cast<uint4 *>(smem + Z::OFF_RING + unit * Z::UNIT + (uc >> 3) * Z::BOX + swz128(r, uc & 7u));
                        if (key < it.lo || key >= it.hi) *at = make_uint4(0u, 0u, 0u, 0u);
                        else if (key < it.all_lo || key >= it.all_hi) {
                            const uint4 v = *at;
                            if (half2_not_finite(v.x) || half2_not_finite(v.y) || half2_not_finite(v.z) || half2_not_finite(v.w)) atomicOr(&sh->bad[gt & 1u][r >> 5], 1u << (r & 31u));
                        }
                    }
                    if (it.ntok > 1u) { // (else all its rows see the same keys)
                        named_bar_sync(5, 256);
#pragma unroll
                        for (int i = 0; i < 4; i++) bad[i] = sh->bad[gt & 1u][i];
                        bad_any = (bad[0] | bad[1] | bad[2] | bad[3]) != 0u;
                        if (bad_any) {
                            for (uint32_t idx = st; idx < PA_KEYS * (DIM / 8u); idx += 256u) {
                                const uint32_t r = idx / (DIM / 8u), c = idx % (DIM / 8u);
                                const uint32_t unit = (uv + c / (Z::UNIT_DIMS / 8u)) % Z::NST, uc = c % (Z::UNIT_DIMS / 8u);
                                if (bad[r >> 5] >> (r & 31u) & 1u)
                                    *reinterpret_cast<uint4 *>(smem + Z::OFF_RING + unit * Z::UNIT + (uc >> 3) * Z::BOX + swz128(r, uc & 7u)) = make_uint4(0u, 0u, 0u, 0u);
                            }
                            named_bar_sync(5, 256); // all have read bad[]
                            if (st < 4u) sh->bad[gt & 1u][st] = 0u; // (read again two tiles on, behind this tile's p_full)
                        }
                    }
                    fence_proxy_async();
                }
                uint32_t sr[2][32];
                float cf = 1.0f;
                if (active) {
                    tmem_ld32(s_col + 64u * half, sr[0]);
                    tmem_ld32(s_col + 64u * half + 32u, sr[1]);
                    tmem_wait_ld();
                    const uint32_t key_base = key0 + 64u * half;
                    // work in base-2 exponents: e^(s scale - m) = 2^(s C - m2), C = scale log2(e)
                    float mt[4] = {NEG_BIG, NEG_BIG, NEG_BIG, NEG_BIG};
                    if (edge) {
#pragma unroll
                        for (int h = 0; h < 2; h++)
#pragma unroll
                            for (int c = 0; c < 32; c++) {
                                const uint32_t key = key_base + 32u * h + c;
                                const float v = (key >= klo && key < vis) ? __uint_as_float(sr[h][c]) : -INFINITY;
                                sr[h][c] = __float_as_uint(v);
                                mt[c & 3] = fmaxf(mt[c & 3], v);
                            }
                    } else {
#pragma unroll
                        for (int h = 0; h < 2; h++)
#pragma unroll
                            for (int c = 0; c < 32; c++) mt[c & 3] = fmaxf(mt[c & 3], __uint_as_float(sr[h][c]));
                    }
                    float mx = fmaxf(fmaxf(mt[0], mt[1]), fmaxf(mt[2], mt[3]));
                    mx = mx > NEG_TEST ? mx * g.scale2 : NEG_BIG; // this half row's tile maximum as a base-2 exponent
                    // The reference maximum moves for the first valid tile or when the tile exceeds it by more than 8. The two warps that
                    // share these 32 rows vote; only then they exchange maxima.
                    if (pair_bar_or(1u + q4, mx > NEG_TEST && (m_ref < NEG_TEST || mx > m_ref + PA_LAZY2))) {
                        red[128u * half + row] = mx;
                        pair_bar_sync(1u + q4);
                        mx = fmaxf(mx, red[128u * (half ^ 1u) + row]);
                        if (mx > NEG_TEST && (m_ref < NEG_TEST || mx > m_ref + PA_LAZY2)) {
                            const float m_new = fmaxf(m_ref, mx);
                            cf = m_ref > NEG_TEST ? exp2f(m_ref - m_new) : 1.0f;
                            m_ref = m_new;
                        }
                    }
                    const float neg_m = m_ref > NEG_TEST ? -m_ref : 0.0f;
                    float sum[2] = {0.0f, 0.0f};
                    uint32_t ph[32]; // 64 weights as f16 pairs
#pragma unroll
                    for (int h = 0; h < 2; h++)
#pragma unroll
                        for (int c = 0; c < 32; c += 2) {
                            float w0, w1;
                            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(w0) : "f"(fmaf(__uint_as_float(sr[h][c]), g.scale2, neg_m)));
                            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(w1) : "f"(fmaf(__uint_as_float(sr[h][c + 1]), g.scale2, neg_m)));
                            sum[0] += w0;
                            sum[1] += w1;
                            if (edge) { // kept for the rows of V that are added by hand
                                sr[h][c] = __float_as_uint(w0);
                                sr[h][c + 1] = __float_as_uint(w1);
                            }
                            const __half2 hp = __floats2half2_rn(w0, w1);
                            ph[16 * h + (c >> 1)] = *reinterpret_cast<const uint32_t *>(&hp);
                        }
                    l_run = l_run * cf + (sum[0] + sum[1]);
                    tmem_st32(s_col + 64u * half, ph);
                    if (j > 0 && __any_sync(0xffffffffu, cf != 1.0f)) { // rescale this warp's rows and dims of O (rare)
                        wait_pv(gt - 1u);
#pragma unroll 1
                        for (uint32_t c0 = 0; c0 < HD; c0 += 32u) {
                            uint32_t orow[32];
                            tmem_ld32(tmem + lane_addr + HD * half + c0, orow);
                            tmem_wait_ld();
#pragma unroll
                            for (int c = 0; c < 32; c++) orow[c] = __float_as_uint(__uint_as_float(orow[c]) * cf);
                            tmem_st32(tmem + lane_addr + HD * half + c0, orow);
                        }
                    }
                    tmem_wait_st();
                }
                tc_fence_before();
                arrive(bar_p_full + 8u * (gt & 1u));
                if (bad_any) { // rows of V that are not finite: w v for the tokens that see them, added once the tile's products are there
                    wait_pv(gt);
                    for (uint32_t r = 0; r < PA_KEYS; r++) {
                        if (!(bad[r >> 5] >> (r & 31u) & 1u) || !active) continue;
                        if ((r >> 6) == half) {
                            float w = 0.0f;
#pragma unroll
                            for (uint32_t c = 0; c < 64u; c++)
                                if (c == (r & 63u)) w = __uint_as_float(sr[c >> 5][c & 31u]);
                            red[row] = w;
                        }
                        pair_bar_sync(1u + q4);
                        const float w = red[row];
                        const uint32_t key = key0 + r;
                        const bool sees = real && key >= klo && key < vis;
                        const size_t at = ((size_t)g.pages[sq.table + (key >> g.page_shift)] << g.page_shift) + (key & ((1u << g.page_shift) - 1u));
                        const __half *v = reinterpret_cast<const __half *>(g.vpages + at * g.row_bytes) + (size_t)sg.kvh * DIM + HD * half;
#pragma unroll 1
                        for (uint32_t c0 = 0; c0 < HD; c0 += 32u) {
                            uint32_t orow[32];
                            tmem_ld32(tmem + lane_addr + HD * half + c0, orow);
                            tmem_wait_ld();
#pragma unroll
                            for (int c = 0; c < 32; c++)
                                if (sees) orow[c] = __float_as_uint(fmaf(w, __half2float(v[c0 + c]), __uint_as_float(orow[c])));
                            tmem_st32(tmem + lane_addr + HD * half + c0, orow);
                        }
                        tmem_wait_st();
                        pair_bar_sync(1u + q4); // red[] is free again
                    }
                    tc_fence_before();
                }
            }
            // ---------------- end of the segment: all its MMAs have completed ----------------
            u += 2u * n * Z::NUN;
            wait_pv(gt - 1u);
            more = walk.next(nx);
            if (more) load_q(nx); // the next segment's first scores are computed while this one's epilogue runs
            if (active) {
                red[128u * half + row] = l_run;
                pair_bar_sync(1u + q4);
                const float l_all = red[row] + red[128u + row];
                const bool seen = real && klo < vis;
                if (sg.whole) {
                    // out[token][head][:] = O / (l + sink)
                    float den = l_all;
                    if (g.sinks && real) den += exp2f(g.sinks[sg.kvh * group + head] * PA_LOG2E - (m_ref > NEG_TEST ? m_ref : 0.0f));
                    const float inv = 1.0f / den;
                    __half *dst = g.out + (int64_t)(sq.row + it.tok0 + tok) * g.out_stride + (size_t)(sg.kvh * group + head) * DIM + HD * half;
#pragma unroll 1
                    for (uint32_t c0 = 0; c0 < HD; c0 += 32u) {
                        uint32_t orow[32];
                        tmem_ld32(tmem + lane_addr + HD * half + c0, orow);
                        tmem_wait_ld();
                        if (real) {
#pragma unroll
                            for (int c = 0; c < 32; c += 8) {
                                uint32_t w[4];
#pragma unroll
                                for (int e = 0; e < 4; e++) {
                                    const __half2 h2 = __floats2half2_rn(seen ? __uint_as_float(orow[c + 2 * e]) * inv : 0.0f, seen ? __uint_as_float(orow[c + 2 * e + 1]) * inv : 0.0f);
                                    w[e] = *reinterpret_cast<const uint32_t *>(&h2);
                                }
                                *reinterpret_cast<uint4 *>(dst + c0 + c) = make_uint4(w[0], w[1], w[2], w[3]);
                            }
                        }
                    }
                } else {
                    // a part: maximum, sum and O as they are, for the merge
                    float *ps = g.scratch + part_slot(blockIdx.x, sg.part) * part_floats(DIM);
                    if (half == 0u && real) *reinterpret_cast<float2 *>(ps + 128u * DIM + 2u * row) = make_float2(m_ref, seen ? l_all : -1.0f);
#pragma unroll 1
                    for (uint32_t c0 = 0; c0 < HD; c0 += 32u) {
                        uint32_t orow[32];
                        tmem_ld32(tmem + lane_addr + HD * half + c0, orow);
                        tmem_wait_ld();
                        if (real) {
#pragma unroll
                            for (int c = 0; c < 32; c += 4)
                                *reinterpret_cast<uint4 *>(ps + (size_t)row * DIM + HD * half + c0 + c) = make_uint4(orow[c], orow[c + 1], orow[c + 2], orow[c + 3]);
                        }
                    }
                }
                tc_fence_before();
                pair_bar_sync(1u + q4); // red[] is free for the next segment
            }
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
    g.vpages = p->layer_ptr(layer, 1);
    g.sinks = a.sinks;
    g.scratch = p->scratch;
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

mkv_status pool_attn_f16_setup(Pool *p) {
    MKV_CUDA(cudaFuncSetAttribute(pool_attn_f16_kernel<64>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)PaSizes<64>::SMEM));
    MKV_CUDA(cudaFuncSetAttribute(pool_attn_f16_kernel<128>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)PaSizes<128>::SMEM));
    MKV_CUDA(cudaFuncSetAttribute(pool_attn_f16_kernel<256>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)PaSizes<256>::SMEM));
    const uint64_t rows = (uint64_t)p->desc.n_pages * p->desc.page_tokens, cols = (uint64_t)p->desc.kv_heads * (uint64_t)p->desc.head_dim;
    const uint32_t box_rows = std::min(p->desc.page_tokens, PA_KEYS);
    p->maps.resize(2 * (size_t)p->desc.n_layers);
    for (int l = 0; l < p->desc.n_layers; l++)
        for (int kv = 0; kv < 2; kv++) {
            const mkv_status st = make_tensor_map(&p->maps[2 * (size_t)l + (size_t)kv], MKV_F16, p->layer_ptr(l, kv), rows, cols, box_rows);
            if (st != MKV_OK) return st;
        }
    return MKV_OK;
}

} // namespace mkv
