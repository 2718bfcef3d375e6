// Attention of blocks of new tokens over f32 pages on the 5th-generation tensor cores, with f32-grade arithmetic.
//   out_t = sum_k e^(s_k - M) v_k / (sum_k e^(s_k - M) + e^(sink - M)),  s_k = scale q_t . k_k
//
// Every f32 operand is scaled by a power of two and split into two f16 values, hi = f16(x), lo = f16(x - hi): 22 bits. An item is up
// to 64 rows (the query heads of one KV head for 64 / group tokens, row = token * group + head); the 128 rows of a product are the
// rows' hi parts and, 64 further, their lo parts, so that two products with the hi and the lo tile give all four partial products:
//   S'[r], S'[64 + r]   = (Q hi, Q lo) (K hi + K lo)^T      A = Q' (tensor memory), B = the converted K tile (K-major)
//   O'[r], O'[64 + r]   = (P hi, P lo) (V hi + V lo)        A = P' (shared memory), B = the converted V tile (N-major)
// and a score or an output is the sum of two rows. The tensor core's f32 sums truncate, so a long chain of them drifts (2^-24 a step,
// all in one direction): the O' of every tile of 64 keys starts from zero and is folded into O in registers with a rounded FMA, which
// also takes the rescale by the running maximum and the scale of the V tile.
//
// Conversion in place: TMA brings a tile as blocks of [64 keys][32 dims] (rows of 128 bytes, 128-byte swizzle); two lanes read the 256
// bytes that a key has in two neighbouring blocks and write its 64 hi values into the first block's row and its 64 lo values into the
// second's, so a tile needs no second buffer. The scale of a tile (K and V each their own) is the one in front's as long as each
// converter warp's largest value then lies in [2^8, 2^15) or is zero; otherwise, and where a value is not finite, the tile is converted
// once more, from global memory, with its own scale: no f32 value overflows, and what is lost of a value is 2^-23 of it, or 2^-33 of
// the tile's largest. Values that are not finite are zero in the operands; their keys are noted, and the softmax threads add their
// share with ordinary arithmetic for the rows that see them. Keys that no token of the item sees are zero as well, whatever lies in
// their rows.
//
// Bound by the time that a tile stays in the ring: a K or V tile of 64 KB lands about 3,000 clocks after its load was issued, its four
// converter warps take 3,500 to 4,500 (a unit's chain load - split - store is about 800, whatever a warp's share of it; eight warps on a
// tile measured the same), products and their waits the rest, and shared memory holds three. Eight sessions of up to 32,000 tokens (533 MB)
// take 154 us, 3.5 TB/s; blocks of 300 to 512 tokens over up to 4,096 (46 GFLOP, three f16 products each) 405 us.
//
// Where every item has at most 32 rows (decode steps, drafts; FEW) the four warps that would have rows 32 .. 63 are a second team of
// converters, the first one takes K and it takes V: nine sessions with heads of 128 88 us, with one team 96; heads of 256 154 and 157.
//
// Roles (512 threads, four warpgroups whose register budgets are set with setmaxnreg): warps 0 and 3 = TMA producers, warp 1 =
// issues S' and owns the TMEM, warp 2 = issues O', warps 4..7 = converters, warps 8..15 = softmax and owners of O: two threads per TMEM
// lane, half of the dims each, and of a row's four threads 16 of a tile's keys each. TMEM: O' = columns 0 .. DIM - 1, S' = 256 .. 319 and 320 .. 383, Q' = 384 ...
// Every wait is bounded; TMEM is freed on every path. With heads of 256 a thread spills 380 to 480 bytes, of 128 about 100.
#include <type_traits>

#include "pool_plan.cuh"
#include "ptx.cuh"

namespace mkv {
using namespace ptx;

constexpr uint32_t PF_KEYS32 = 64;
constexpr int PB_THREADS = 512;
constexpr long long PB_WAIT_LIMIT = 2000000000ll;
constexpr float PB_LOG2E = 1.4426950408889634f;
constexpr uint32_t PB_COL_S = 256, PB_COL_Q = 384;
constexpr uint32_t PB_BLK = 8192;          // [64 keys][32 dims] f32, then [64 keys][64 dims] f16
constexpr uint32_t PB_UNIT = 2 * PB_BLK;   // 64 dims of a tile
constexpr uint32_t PB_NST = 12;            // units of the ring: a multiple of a tile's, so that a tile lies in one piece
constexpr uint32_t PB_PBUF = 16384;             // P' [128 rows][64 keys] f16; also where S'[64 + r] changes hands
constexpr uint32_t PB_OFF_P = PB_NST * PB_UNIT; // two of them, in turn
constexpr uint32_t PB_OFF_RED = PB_OFF_P + 2 * PB_PBUF; // [4 quarters of a tile's keys][64 rows] floats, [64 rows] scales of Q'
constexpr uint32_t PB_OFF_BAR = PB_OFF_RED + 1280;
constexpr uint32_t PB_KINDS = 8;           // K tiles, and V tiles, that the ring cannot hold at one time: barriers of each kind
constexpr uint32_t PB_NBAR = PB_NST + 4 * PB_KINDS + 7; // empty[NST], full[2][KINDS], conv[2][KINDS], s_full[2], s_free[2], p_full, pv_done, q_full
constexpr uint32_t PB_OFF_MISC = PB_OFF_BAR + PB_NBAR * 8;
constexpr uint32_t PB_NOTES = 8;           // tiles whose scale and notes are kept: more than the ring holds

struct PbShared {
    uint32_t tmem_base;
    volatile uint32_t abort;
    uint32_t amax[2][4];              // [team][converter warp]
    float unscale[2][PB_NOTES];       // [K, V][tile]
    uint16_t odd[2][PB_NOTES][4];     // keys with a value that is not finite, 16 of each converter warp
};
constexpr uint32_t PB_SMEM = PB_OFF_MISC + sizeof(PbShared) + 1024;
static_assert(PB_SMEM <= 232448, "shared memory");

struct PbArgs {
    const float *q;
    float *out;
    int64_t q_stride, out_stride;
    const uint32_t *pages;
    const float *kpages, *vpages;
    const float *sinks;
    float *scratch;
    uint32_t *status;
    size_t row_floats;
    float scale2; // scale * log2(e)
    uint32_t page_shift;
};

__device__ __forceinline__ bool pb_wait(uint32_t bar, uint32_t parity, PbShared *sh, uint32_t *status) {
    if (mbar_try_wait(bar, parity)) return true;
    const long long t0 = clock64();
    for (;;) {
        if (sh->abort) return false;
#pragma unroll 1
        for (int i = 0; i < 64; i++)
            if (mbar_try_wait(bar, parity)) return true;
        if (clock64() - t0 > PB_WAIT_LIMIT) break;
    }
    sh->abort = 1;
    atomicOr(status, DEV_ERR_WAIT_TIMEOUT);
    return false;
}
// A place of a ring of N and the parity of its current use
template <uint32_t N> struct PbRing {
    uint32_t s = 0, turn = 0;
    __device__ __forceinline__ void next(uint32_t d = 1u) { // d <= N
        s += d;
        if (s >= N) {
            s -= N;
            turn ^= 1u;
        }
    }
};
// The tiles of a CTA's segments as one stream
struct PbStream {
    PlanWalk walk;
    PlanSegment sg;
    uint32_t tile;
    bool more;
    __device__ __forceinline__ PbStream(const PoolPlan &plan) : walk(plan, blockIdx.x, PF_KEYS32) { step(); }
    __device__ __forceinline__ void step() {
        more = walk.next(sg);
        tile = sg.a;
    }
    __device__ __forceinline__ bool first() const { return tile == sg.a; }
    __device__ __forceinline__ void next() {
        if (++tile == sg.b) step();
    }
};
__device__ __forceinline__ bool is_finite_bits(uint32_t b) { return (b & 0x7f800000u) != 0x7f800000u; }
// The power of two that brings `amax` (its bits; finite) to [2^13, 2^14)
__device__ __forceinline__ uint32_t scale_bits(uint32_t amax) {
    const int e = (int)(amax >> 23) - 127;
    return (uint32_t)(min(13 - e, 126) + 127) << 23;
}
// 8 values, times s, to their hi and lo parts
__device__ __forceinline__ void split8(const float (&x)[8], float s, uint4 &hi, uint4 &lo) {
    uint32_t h[4], l[4];
    const uint64_t s2 = pack2(s, s);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint64_t x2 = pack2(x[2 * i], x[2 * i + 1]);
        float y0, y1;
        unpack2(mul2(x2, s2), y0, y1);
        const __half2 a = __floats2half2_rn(y0, y1);
        const float2 f = __half22float2(a);
        unpack2(fma2(x2, s2, pack2(-f.x, -f.y)), y0, y1);
        const __half2 b = __floats2half2_rn(y0, y1);
        h[i] = *reinterpret_cast<const uint32_t *>(&a);
        l[i] = *reinterpret_cast<const uint32_t *>(&b);
    }
    hi = make_uint4(h[0], h[1], h[2], h[3]);
    lo = make_uint4(l[0], l[1], l[2], l[3]);
}

template <int DIM, bool FEW>
__global__ void __launch_bounds__(PB_THREADS, 1)
pool_attn_f32_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const __grid_constant__ PoolPlan plan,
                     const __grid_constant__ PbArgs g) {
    constexpr uint32_t NU = DIM / 64;       // units of a tile
    constexpr uint32_t SOFT = FEW ? 4 : 8;  // softmax warps
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t *smem = smem_raw + (smem_base - smem_u32(smem_raw));
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
    const uint32_t bar0 = smem_base + PB_OFF_BAR;
    const uint32_t bar_empty = bar0, bar_full = bar0 + 8u * PB_NST, bar_conv = bar_full + 16u * PB_KINDS, bar_s_full = bar_conv + 16u * PB_KINDS;
    const uint32_t bar_s_free = bar_s_full + 16u, bar_p_full = bar_s_free + 16u, bar_pv_done = bar_p_full + 8u, bar_q_full = bar_pv_done + 8u;
    // full and conv: of K or V tile t. (Not of a slot of the ring: who waits for K tiles alone would miss a slot's phases for V.)
    auto of_tile = [](bool v, uint32_t t) { return 8u * ((v ? PB_KINDS : 0u) + t % PB_KINDS); };
    PbShared *sh = reinterpret_cast<PbShared *>(smem + PB_OFF_MISC);

    if (tid == 0) {
        for (uint32_t s = 0; s < PB_NST; s++) mbar_init(bar_empty + 8u * s, 1);
        for (uint32_t s = 0; s < 2u * PB_KINDS; s++) {
            mbar_init(bar_full + 8u * s, 2); // one arrival per producer
            mbar_init(bar_conv + 8u * s, 4); // one arrival per converter warp
        }
        for (uint32_t s = 0; s < 2u; s++) {
            mbar_init(bar_s_full + 8u * s, 1);
            mbar_init(bar_s_free + 8u * s, SOFT); // one arrival per softmax warp
        }
        mbar_init(bar_p_full, SOFT);
        mbar_init(bar_pv_done, 1);
        mbar_init(bar_q_full, SOFT);
        sh->abort = 0;
        fence_barrier_init();
        fence_proxy_async();
    }
    if (warp == 1) tmem_alloc(smem_base + PB_OFF_MISC, 512); // writes sh->tmem_base
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh->tmem_base, total = plan.start[blockIdx.x].tiles;
    // Nothing global is touched before the kernel in front has finished. This kernel has begun before that, so what that one may have written (page
    // tables, rotated queries) is not read-only for it, and no load takes the read-only path.
    pdl_wait();
    pdl_launch_dependents();

    // The units of the CTA's T tiles in ring order, whatever segment they belong to: K(0), then K(t + 1) and V(t) for each t. In front of
    // K(t) are t + max(t - 1, 0) tiles of K and V, in front of V(t) min(t + 2, T) + t.
    // ---------------- converters: a warp has 16 keys of every unit, a lane one of a key's two blocks ----------------
    // One team of four warps for K and V, or one for each.
    auto converter = [&](bool k_tiles, bool v_tiles, uint32_t cw) {
        const uint32_t team = k_tiles ? 0u : 1u, bar_team = 3u + team, key_in = 16u * cw + (lane >> 1), j = lane & 1u;
        // chunk of the block's row that x[i] holds: in an order in which a key's two lanes meet no bank together
        auto chunk = [&](uint32_t i) { return i ^ (4u * j); };
        PbRing<PB_NST> at;
        struct Tile {
            uint32_t key0, lo, hi, table, kvh;
        };
        PbStream ts(plan);
        auto take = [&](const Tile &last) -> Tile { // the stream's tile, which follows `last`; the stream moves on
            const PlanItem &it = ts.sg.it;
            Tile t = {(it.tile0 + ts.tile) * PF_KEYS32, last.lo, last.hi, last.table, last.kvh};
            if (ts.first()) t = {t.key0, it.lo, it.hi, plan.seq[ts.sg.seq].table, ts.sg.kvh};
            ts.next();
            return t;
        };
        float k_scale = 1.0f, v_scale = 1.0f;
        auto convert = [&](bool v, const Tile &tl, uint32_t note) {
            const uint32_t key = tl.key0 + key_in;
            const bool in = key >= tl.lo && key < tl.hi, whole = tl.key0 >= tl.lo && tl.key0 + PF_KEYS32 <= tl.hi;
            const PbRing<PB_NST> begin = at;
            float amax = 0.0f;
            bool odd = false; // a value of this lane's is not finite
            float s = v ? v_scale : k_scale;
            auto fetch = [&](uint32_t slot, float4 (&x)[8]) { // this lane's values of a unit
                const uint8_t *u = smem + slot * PB_UNIT + j * PB_BLK;
#pragma unroll
                for (uint32_t i = 0; i < 8u; i++) x[i] = *reinterpret_cast<const float4 *>(u + swz128(key_in, chunk(i)));
            };
            auto put = [&](uint32_t slot, const float4 (&x)[8]) { // to hi and lo
                uint8_t *u = smem + slot * PB_UNIT;
#pragma unroll
                for (uint32_t i = 0; i < 8u; i += 2u) {
                    const float y[8] = {x[i].x, x[i].y, x[i].z, x[i].w, x[i + 1].x, x[i + 1].y, x[i + 1].z, x[i + 1].w};
                    uint4 hi, lo;
                    split8(y, s, hi, lo);
                    const uint32_t at_row = swz128(key_in, 4u * j + (chunk(i) >> 1));
                    *reinterpret_cast<uint4 *>(u + at_row) = hi;
                    *reinterpret_cast<uint4 *>(u + PB_BLK + at_row) = lo;
                }
            };
            auto look = [&](float4 (&x)[8]) { // amax; odd
                if (!whole && !in) // (keys that no token of the item sees)
#pragma unroll
                    for (uint32_t i = 0; i < 8u; i++) x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                uint64_t z[2] = {0ull, 0ull}; // 0 * x is a NaN where x is not finite
                float top[2] = {amax, 0.0f};
#pragma unroll
                for (uint32_t i = 0; i < 8u; i++) {
                    top[i & 1u] = max3(top[i & 1u], fabsf(x[i].x), fabsf(x[i].y));
                    top[i & 1u] = max3(top[i & 1u], fabsf(x[i].z), fabsf(x[i].w));
                    z[i & 1u] = fma2(pack2(x[i].x, x[i].y), 0ull, z[i & 1u]);
                    z[i & 1u] = fma2(pack2(x[i].z, x[i].w), 0ull, z[i & 1u]);
                }
                amax = fmaxf(top[0], top[1]);
                float z0, z1;
                unpack2(add2(z[0], z[1]), z0, z1);
                odd = odd || z0 + z1 != 0.0f;
            };
            auto tile_scale = [&]() -> float { // of the largest of all warps' amax
                const uint32_t mine = __reduce_max_sync(0xffffffffu, __float_as_uint(amax));
                if (lane == 0) sh->amax[team][cw] = mine;
                named_bar_sync(bar_team, 128); // (there is another in front of the next use of amax[])
                uint32_t most = 0u;
                for (uint32_t i = 0; i < 4u; i++) most = max(most, sh->amax[team][i]);
                return most ? __uint_as_float(scale_bits(most)) : 1.0f;
            };
            pb_wait(bar_full + of_tile(v, note), (note / PB_KINDS) & 1u, sh, g.status);
            __syncwarp();
            if (note == 0u) { // the first tile has no scale in front of it: the largest value of its first 64 dims gives it, to [2^11, 2^12)
                float4 x[8];
                fetch(begin.s, x);
                look(x);
                s = (v ? v_scale : k_scale) = 0.25f * tile_scale();
                amax = 0.0f;
            }
#pragma unroll 1
            for (uint32_t h = 0; h < NU; h++) {
                float4 x[8];
                fetch(begin.s + h, x);
                __syncwarp(); // both lanes of a key have read its rows
                look(x);
                put(begin.s + h, x);
            }
            at.next(NU);
            // The scale fits if each warp's largest value lies well inside f16's range under it. Otherwise, and where values are not finite, once
            // more from global memory: the tile's largest finite value, then its values with the scale that this gives, the others as zeros.
            amax = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(amax)));
            if (named_bar_or(bar_team, 128, odd || (amax != 0.0f && !(amax * s >= 256.0f && amax * s < 32768.0f)))) {
                const float *src = v ? g.vpages : g.kpages;
                if (in) {
                    const size_t page = __ldcg(g.pages + tl.table + (key >> g.page_shift));
                    src += ((page << g.page_shift) + (key & ((1u << g.page_shift) - 1u))) * g.row_floats + (size_t)tl.kvh * DIM + 32u * j;
                }
                auto again = [&](uint32_t h, float4 (&x)[8]) {
#pragma unroll
                    for (uint32_t i = 0; i < 8u; i++) {
                        x[i] = in ? *reinterpret_cast<const float4 *>(src + 64u * h + 4u * chunk(i)) : make_float4(0.f, 0.f, 0.f, 0.f);
                        float *e = &x[i].x;
#pragma unroll
                        for (int k = 0; k < 4; k++)
                            if (!is_finite_bits(__float_as_uint(e[k]))) e[k] = 0.0f;
                    }
                };
                amax = 0.0f;
#pragma unroll 1
                for (uint32_t h = 0; h < NU; h++) {
                    float4 x[8];
                    again(h, x);
#pragma unroll
                    for (uint32_t i = 0; i < 8u; i++) amax = fmaxf(amax, fmaxf(fmaxf(fabsf(x[i].x), fabsf(x[i].y)), fmaxf(fabsf(x[i].z), fabsf(x[i].w))));
                }
                s = (v ? v_scale : k_scale) = tile_scale();
#pragma unroll 1
                for (uint32_t h = 0; h < NU; h++) {
                    float4 x[8];
                    again(h, x);
                    put(begin.s + h, x);
                }
                named_bar_sync(bar_team, 128); // amax[] has been read
            }
            const uint32_t odds = __ballot_sync(0xffffffffu, odd);
            if (lane == 0) {
                uint32_t m = 0u;
                if (odds)
                    for (uint32_t i = 0; i < 16u; i++) m |= (odds >> (2u * i) & 3u) ? 1u << i : 0u;
                sh->odd[v ? 1 : 0][note % PB_NOTES][cw] = (uint16_t)m;
                if (cw == 0u) sh->unscale[v ? 1 : 0][note % PB_NOTES] = __uint_as_float((254u << 23) - __float_as_uint(s)); // 1 / s, s being a power of two
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_conv + of_tile(v, note));
        };
        // A wait that runs out makes all later ones return at once; the warps go through the same barriers all the same.
        Tile cur = take(Tile{});
        if (k_tiles) convert(false, cur, 0u);
        else at.next(NU);
        for (uint32_t t = 0; t < total; t++) {
            const Tile ahead = ts.more ? take(cur) : cur;
            if (t + 1u < total) {
                if (k_tiles) convert(false, ahead, t + 1u);
                else at.next(NU);
            }
            if (v_tiles) convert(true, cur, t);
            else at.next(NU);
            cur = ahead;
        }
    };
    if (warp < 4u) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
        if (warp == 0 || warp == 3u) {
            // ---------------- TMA producers: every other box of each unit ----------------
            // Both go through all units in order: a parity tells a phase from its neighbours only, so whoever waits for a slot has to have
            // waited for its uses before.
            const uint32_t page_tokens = 1u << g.page_shift, box_rows = min(page_tokens, PF_KEYS32), nrb = PF_KEYS32 / box_rows;
            const uint32_t box = 2u * lane + (warp == 0 ? 0u : 1u), rb = box % nrb, cb = box / nrb; // this lane's row box and 32-dim box of a unit
            PbRing<PB_NST> at;
            uint32_t u = 0;
            PbStream ts(plan);
            struct Tile {
                uint32_t row; // in the pool, of this lane's box; ~0u where no token of the item sees a key of it
                int x;        // first column of the head
                bool is;
            };
            auto look_up = [&]() -> Tile { // the stream's tile; the stream moves on
                Tile t = {~0u, (int)(ts.sg.kvh * DIM + cb * 32u), ts.more};
                const PlanItem &it = ts.sg.it;
                const uint32_t key = (it.tile0 + ts.tile) * PF_KEYS32 + rb * box_rows;
                if (t.is && cb < 2u && key + box_rows > it.lo && key < it.hi)
                    t.row = (__ldcg(g.pages + plan.seq[ts.sg.seq].table + (key >> g.page_shift)) << g.page_shift) + (key & (page_tokens - 1u));
                if (t.is) ts.next();
                return t;
            };
            auto load = [&](bool v, const Tile &t, uint32_t n) -> bool { // the units of K or V tile n
                const uint32_t boxes = __popc(__ballot_sync(0xffffffffu, t.row != ~0u)), bar = bar_full + of_tile(v, n);
#pragma unroll 1
                for (uint32_t h = 0; h < NU; h++, u++, at.next()) {
                    if (u >= PB_NST && !__all_sync(0xffffffffu, pb_wait(bar_empty + 8u * at.s, at.turn ^ 1u, sh, g.status))) return false;
                    if (h == 0u && lane == 0) mbar_expect_tx(bar, NU * boxes * box_rows * 128u);
                    __syncwarp();
                    if (t.row != ~0u)
                        tma_load_2d(smem_base + at.s * PB_UNIT + cb * PB_BLK + rb * box_rows * 128u, v ? &vmap : &kmap, t.x + (int)(64u * h), (int)t.row, bar);
                }
                return true;
            };
            Tile cur = look_up();
            bool ok = load(false, cur, 0u);
            Tile ahead = look_up();
            for (uint32_t t = 0; ok && cur.is; t++) {
                const Tile later = look_up(); // (its page is there when its turn comes)
                if (ahead.is) ok = load(false, ahead, t + 1u);
                ok = ok && load(true, cur, t);
                cur = ahead;
                ahead = later;
            }
        } else if (warp == 1) {
            // ---------------- S' = Q' (K hi + K lo)^T ----------------
            if (lane == 0) {
                constexpr uint32_t IDESC = tc_idesc_f16(128, 64, false);
                const uint64_t k_desc = tc_desc_sw128(smem_base, 16, 1024);
                PbRing<PB_NST> at;
                uint32_t nseg = 0;
                bool ok = true;
                PbStream ts(plan);
                for (uint32_t t = 0; ok && ts.more; t++) {
                    if (ts.first()) { // the segment's Q' is in tensor memory
                        ok = pb_wait(bar_q_full, nseg & 1u, sh, g.status);
                        nseg++;
                    }
                    if (t >= 2u) ok = ok && pb_wait(bar_s_free + 8u * (t & 1u), ((t >> 1) - 1u) & 1u, sh, g.status);
                    const uint32_t d = tmem + PB_COL_S + 64u * (t & 1u);
                    ok = ok && pb_wait(bar_conv + of_tile(false, t), (t / PB_KINDS) & 1u, sh, g.status);
                    tc_fence_after();
                    // All of K lo first: what a step truncates is 2^-24 of the sum so far, and that is small until K hi comes in.
#pragma unroll
                    for (uint32_t n = 0; n < 2u * NU; n++) {
                        const uint32_t h = n % NU;
                        const uint64_t kd = k_desc + (at.s + h) * (PB_UNIT >> 4) + (n < NU ? PB_BLK >> 4 : 0u);
#pragma unroll
                        for (uint32_t ks = 0; ks < 4u; ks++) // 16 dims an MMA
                            tc_mma_f16_ta(d, tmem + PB_COL_Q + 32u * h + 8u * ks, kd + ((ks * 32u) >> 4), IDESC, (n > 0 || ks > 0) ? 1u : 0u);
                        if (n >= NU) tc_commit(bar_empty + 8u * (at.s + h));
                    }
                    at.next(NU);
                    tc_commit(bar_s_full + 8u * (t & 1u));
                    if (t > 0u) at.next(NU); // over a tile of V
                    ts.next();
                }
            }
        } else {
            // ---------------- O' = P' (V hi + V lo) ----------------
            if (lane == 0) {
                constexpr uint32_t IDESC = tc_idesc_f16(128, DIM, true);
                const uint64_t v_desc = tc_desc_sw128(smem_base, PB_UNIT, 1024), p_desc = tc_desc_sw128(smem_base + PB_OFF_P, 16, 1024);
                PbRing<PB_NST> at;
                at.next(min(2u, total) * NU);
                bool ok = true;
                for (uint32_t t = 0; ok && t < total; t++) {
                    const uint32_t s0 = at.s;
                    ok = ok && pb_wait(bar_conv + of_tile(true, t), (t / PB_KINDS) & 1u, sh, g.status);
                    at.next(NU);
                    ok = ok && pb_wait(bar_p_full, t & 1u, sh, g.status);
                    tc_fence_after();
                    const uint64_t vd = v_desc + s0 * (PB_UNIT >> 4);
#pragma unroll
                    for (uint32_t ks = 0; ks < 8u; ks++) // 16 keys an MMA, V lo first
                        tc_mma_f16(tmem, p_desc + (((t & 1u) * PB_PBUF + (ks & 3u) * 32u) >> 4), vd + (((ks < 4u ? PB_BLK : 0u) + (ks & 3u) * 2048u) >> 4), IDESC,
                                   ks > 0 ? 1u : 0u);
#pragma unroll
                    for (uint32_t h = 0; h < NU; h++) tc_commit(bar_empty + 8u * (s0 + h));
                    tc_commit(bar_pv_done);
                    if (t + 2u < total) at.next(NU); // over a tile of K
                }
            }
        }
    } else if (warp < 8u) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
        converter(true, !FEW, warp - 4u);
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 192;"); // 128 x 48 + 128 x 80 + 256 x 192 = the launch's 512 x 128
        if (FEW && (warp & 1u)) {
            // the lanes of rows 32 .. 63, which no item has: zeros, so that their products draw less power
            const uint32_t z[16] = {};
            const uint32_t q4 = warp & 3u, half = (warp - 8u) >> 2;
            for (uint32_t c = 0; c < DIM / 4u; c += 16u) tmem_st16(tmem + ((32u * q4) << 16) + PB_COL_Q + DIM / 4u * half + c, z);
            tmem_wait_st();
            for (uint32_t c = 0; c < 8u; c++) *reinterpret_cast<uint4 *>(smem + PB_OFF_P + half * PB_PBUF + swz128(32u * q4 + lane, c)) = make_uint4(0u, 0u, 0u, 0u);
            fence_proxy_async();
            tc_fence_before();
            converter(false, true, (warp - 8u) >> 1);
        } else {
        // ---------------- softmax ----------------
        const uint32_t q4 = warp & 3u, half = (warp - 8u) >> 2;
        const uint32_t lane_addr = (32u * q4) << 16;
        const bool hi = q4 < 2u;                             // this lane has a row's hi parts, else its lo parts
        const uint32_t row = 32u * (q4 & 1u) + lane;         // the row, 0 .. 63
        const uint32_t bar_group = 1u + (q4 & 1u);           // the four warps that have these 32 rows
        const uint32_t own = (q4 >> 1) + 2u * half;          // this warp's number among them
        const uint32_t e = hi ? 0u : 1u;
        constexpr uint32_t HD = DIM / 2;                     // dims of Q' and O of a thread
        float *red = reinterpret_cast<float *>(smem + PB_OFF_RED), *q_s = red + 256;
        const uint32_t group = plan.group, tok = row / group, head = row - tok * group;
        auto arrive = [&](uint32_t bar) { // one arrival per warp, after all its lanes
            __syncwarp();
            if (lane == 0) mbar_arrive(bar);
        };
        auto wait = [&](uint32_t bar, uint32_t parity) {
            pb_wait(bar, parity, sh, g.status);
            __syncwarp();
            tc_fence_after();
        };
        // where a thread of row r and this half has its 32 scores or weights in the P' buffer: chunk c of 8 (0..3 in row r, 4..7 in row 64 + r)
        uint8_t *p_buf = smem + PB_OFF_P; // of the tile
        auto p_chunk = [&](uint32_t c) { return p_buf + swz128(row + (c >> 2) * 64u, 4u * half + (c & 3u)); };
        // Q' of a segment, scaled by a power of two of each row's own (its inverse is returned). Four threads fetch a row, 16 of every 64 dims
        // each; the hi and lo parts change hands in `stage` (a P' buffer that no product reads), 64 dims at a time, and go to the tensor memory
        // from the threads that have the lanes. The first segment's values stay in registers between the search for the largest one and
        // the split; later ones are read twice, since the registers are O's.
        auto load_q = [&](const PlanSegment &sg, uint8_t *stage, auto first) -> float {
            constexpr bool FIRST = decltype(first)::value;
            const uint32_t rows = sg.it.ntok * group;
            float unscale = 1.0f;
            if (32u * (q4 & 1u) < rows) {
                const uint32_t fr = 32u * (q4 & 1u) + 8u * own + (lane >> 2), j = lane & 3u, ftok = fr / group;
                const bool there = fr < rows;
                const float *src = g.q + (int64_t)(plan.seq[sg.seq].row + sg.it.tok0 + ftok) * g.q_stride + (size_t)(sg.kvh * group + fr - ftok * group) * DIM + 16u * j;
                auto fetch = [&](uint32_t c, float4 (&x)[4]) {
#pragma unroll
                    for (uint32_t i = 0; i < 4u; i++) x[i] = there ? __ldcg(reinterpret_cast<const float4 *>(src + 64u * c + 4u * i)) : make_float4(0.f, 0.f, 0.f, 0.f);
                };
                uint32_t amax = 0u;
                auto look = [&](const float4 (&x)[4]) {
#pragma unroll
                    for (uint32_t i = 0; i < 4u; i++) {
                        const float e[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
                        for (int n = 0; n < 4; n++) {
                            const uint32_t b = __float_as_uint(e[n]) & 0x7fffffffu;
                            amax = max(amax, b < 0x7f800000u ? b : 0u);
                        }
                    }
                };
                float4 x[FIRST ? NU : 2u][4];
                if constexpr (FIRST) {
#pragma unroll
                    for (uint32_t c = 0; c < NU; c++) fetch(c, x[c]);
#pragma unroll
                    for (uint32_t c = 0; c < NU; c++) look(x[c]);
                } else {
#pragma unroll
                    for (uint32_t c = 0; c < NU; c += 2u) {
                        fetch(c, x[0]);
                        if (c + 1u < NU) fetch(c + 1u, x[1]);
                        look(x[0]);
                        if (c + 1u < NU) look(x[1]);
                    }
                    fetch(0, x[0]);
                }
                amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
                amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
                const float s = amax ? __uint_as_float(scale_bits(amax)) : 1.0f;
                if (j == 0u) q_s[fr] = 1.0f / s;
#pragma unroll
                for (uint32_t c = 0; c < NU; c++) {
                    const float4(&y4)[4] = x[FIRST ? c : c & 1u];
                    if (!FIRST && c + 1u < NU) fetch(c + 1u, x[(c + 1u) & 1u]);
#pragma unroll
                    for (uint32_t i = 0; i < 2u; i++) {
                        const float4 u = y4[2 * i], w = y4[2 * i + 1];
                        const float y[8] = {u.x * s, u.y * s, u.z * s, u.w * s, w.x * s, w.y * s, w.z * s, w.w * s};
                        uint32_t h4[4], l4[4];
#pragma unroll
                        for (uint32_t e = 0; e < 4u; e++) {
                            const __half2 h = __floats2half2_rn(y[2 * e], y[2 * e + 1]);
                            const float2 f = __half22float2(h);
                            const __half2 l = __floats2half2_rn(isfinite(f.x) ? y[2 * e] - f.x : 0.0f, isfinite(f.y) ? y[2 * e + 1] - f.y : 0.0f);
                            h4[e] = *reinterpret_cast<const uint32_t *>(&h);
                            l4[e] = *reinterpret_cast<const uint32_t *>(&l);
                        }
                        *reinterpret_cast<uint4 *>(stage + swz128(fr, 2u * j + i)) = make_uint4(h4[0], h4[1], h4[2], h4[3]);
                        *reinterpret_cast<uint4 *>(stage + swz128(64u + fr, 2u * j + i)) = make_uint4(l4[0], l4[1], l4[2], l4[3]);
                    }
                    named_bar_sync(bar_group, 128);
                    uint32_t w[16];
#pragma unroll
                    for (uint32_t i = 0; i < 4u; i++) {
                        const uint4 v = *reinterpret_cast<const uint4 *>(stage + swz128(row + (hi ? 0u : 64u), 4u * half + i));
                        w[4 * i] = v.x;
                        w[4 * i + 1] = v.y;
                        w[4 * i + 2] = v.z;
                        w[4 * i + 3] = v.w;
                    }
                    tmem_st16(tmem + lane_addr + PB_COL_Q + 32u * c + 16u * half, w);
                    if (c == 0u) unscale = q_s[row];
                    named_bar_sync(bar_group, 128); // the stage is free
                }
                tmem_wait_st();
            }
            tc_fence_before();
            arrive(bar_q_full);
            return unscale;
        };
        // score of a key by ordinary arithmetic, for keys that have values that are not finite
        auto plain_score = [&](const float *q, const float *k) {
            float s = 0.0f;
#pragma unroll 1
            for (int d = 0; d < DIM; d++) s = fmaf(q[d], k[d], s);
            return s * g.scale2;
        };
        float O[HD];
        uint32_t t0 = 0; // the segment's first tile
        PlanWalk walk(plan, blockIdx.x, PF_KEYS32);
        PlanSegment sg, nx;
        bool more = walk.next(sg);
        float q_unscale = load_q(sg, smem + PB_OFF_P, std::true_type{}), q_next = 1.0f;
        while (more) {
            const PlanItem it = sg.it;
            const PlanSeq &sq = plan.seq[sg.seq];
            const uint32_t rows = it.ntok * group;
            const bool active = 32u * (q4 & 1u) < rows; // (the same for the four warps of these rows)
            const bool real = row < rows;
            const uint32_t vis = real ? sq.pos + it.tok0 + tok + 1u : 0u; // this row sees klo <= key < vis
            const uint32_t klo = real ? plan_lowest(sq, plan.window, it.tok0 + tok) : 0u;
            const float *q_row = g.q + (int64_t)(sq.row + it.tok0 + (real ? tok : 0u)) * g.q_stride + (size_t)(sg.kvh * group + head) * DIM;
            auto k_row = [&](const float *base, uint32_t key) {
                const size_t page = g.pages[sq.table + (key >> g.page_shift)];
                return base + ((page << g.page_shift) + (key & ((1u << g.page_shift) - 1u))) * g.row_floats + (size_t)sg.kvh * DIM;
            };
            float m = NEG_BIG, l = 0.0f, cf = 0.0f;
            const uint32_t end = t0 + (sg.b - sg.a);
#pragma unroll
            for (uint32_t d = 0; d < HD; d++) O[d] = 0.0f;
            // O = O * cf + O' of tile t; its weights are against m, as cf is
            auto fold = [&](uint32_t t, float m, float cf) {
                wait(bar_pv_done, t & 1u);
                const uint64_t odd = *reinterpret_cast<const uint64_t *>(sh->odd[1][t % PB_NOTES]);
                if (odd != 0ull && hi) { // values of V that are not finite: w v for the rows that see them, added to O' where it lies (rare)
#pragma unroll 1
                    for (uint32_t c0 = 0; c0 < HD; c0 += 32u) {
                        uint32_t o[32];
                        tmem_ld32(tmem + lane_addr + HD * half + c0, o);
                        tmem_wait_ld();
#pragma unroll 1
                        for (uint32_t r = 0; r < PF_KEYS32; r++) {
                            const uint32_t key = (it.tile0 + sg.a + (t - t0)) * PF_KEYS32 + r;
                            if (!(odd >> r & 1ull) || key < klo || key >= vis) continue;
                            const float w = exp2f(plain_score(q_row, k_row(g.kpages, key)) - m);
                            const float *v = k_row(g.vpages, key) + HD * half + c0;
#pragma unroll
                            for (uint32_t c = 0; c < 32u; c++)
                                if (!is_finite_bits(__float_as_uint(v[c]))) o[c] = __float_as_uint(__uint_as_float(o[c]) + w * v[c]);
                        }
                        tmem_st32(tmem + lane_addr + HD * half + c0, o);
                    }
                    tmem_wait_st();
                }
                const float us = sh->unscale[1][t % PB_NOTES] * 0.00006103515625f; // P' carries 2^14
#pragma unroll
                for (uint32_t c0 = 0; c0 < HD; c0 += 32u) {
                    uint32_t o[32];
                    tmem_ld32(tmem + lane_addr + HD * half + c0, o);
                    tmem_wait_ld();
#pragma unroll
                    for (uint32_t c = 0; c < 32u; c++) O[c0 + c] = fmaf(O[c0 + c], cf, __uint_as_float(o[c]) * us);
                }
            };
            for (uint32_t t = t0; t < end; t++) {
                const uint32_t key0 = (it.tile0 + sg.a + (t - t0)) * PF_KEYS32;
                p_buf = smem + PB_OFF_P + (t & 1u) * PB_PBUF; // (free: the product of two tiles in front has been folded)
                const float m_last = m, cf_last = cf;
                wait(bar_s_full + 8u * (t & 1u), (t >> 1) & 1u);
                // A half row's 32 scores: the thread with the hi parts' products takes the first 16, the other the rest; the other 16 of each change
                // hands in the P' buffer.
                const uint32_t s_col = tmem + lane_addr + PB_COL_S + 64u * (t & 1u) + 32u * half;
                uint32_t w[16];
                if (active) {
                    tmem_ld16(s_col + 16u * (1u - e), w);
                    tmem_wait_ld();
#pragma unroll
                    for (uint32_t c = 0; c < 4u; c++) *reinterpret_cast<uint4 *>(p_chunk(4u * (1u - e) + c)) = make_uint4(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]);
                    tmem_ld16(s_col + 16u * e, w);
                    tmem_wait_ld();
                }
                tc_fence_before();
                arrive(bar_s_free + 8u * (t & 1u));
                if (active) {
                    named_bar_sync(bar_group, 128);
                    const float f = g.scale2 * (q_unscale * sh->unscale[0][t % PB_NOTES]);
                    const uint32_t k0 = key0 + 32u * half + 16u * e, odd = sh->odd[0][t % PB_NOTES][2u * half + e];
                    // the keys of this thread that the row sees, a bit each; not those with values that are not finite
                    uint32_t see = 0xffffu;
                    if (key0 < it.all_lo || key0 + PF_KEYS32 > it.all_hi || !real) {
                        const uint32_t a = klo > k0 ? min(klo - k0, 16u) : 0u, b = vis > k0 ? min(vis - k0, 16u) : 0u;
                        see = ((1u << b) - 1u) & ~((1u << a) - 1u);
                    }
                    const uint32_t plain = see & odd;
                    see &= ~odd;
                    float x[16], mx = NEG_BIG;
#pragma unroll
                    for (uint32_t c = 0; c < 4u; c++) {
                        const float4 y = *reinterpret_cast<const float4 *>(p_chunk(4u * e + c));
                        const float o[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                        for (uint32_t n = 0; n < 4u; n++) x[4 * c + n] = (__uint_as_float(w[4 * c + n]) + o[n]) * f;
                    }
                    if (see != 0xffffu)
#pragma unroll
                        for (uint32_t c = 0; c < 16u; c++) x[c] = see >> c & 1u ? x[c] : -INFINITY;
#pragma unroll 1
                    for (uint32_t left = plain; left != 0u; left &= left - 1u) { // (rare)
                        const uint32_t r = (uint32_t)__ffs((int)left) - 1u;
                        const float y = plain_score(q_row, k_row(g.kpages, k0 + r));
#pragma unroll
                        for (uint32_t c = 0; c < 16u; c++)
                            if (c == r) x[c] = y;
                    }
#pragma unroll
                    for (uint32_t c = 0; c < 16u; c += 2u) mx = max3(mx, x[c], x[c + 1]);
                    red[64u * (2u * half + e) + row] = mx;
                    named_bar_sync(bar_group, 128);
                    const float m_new = max3(max3(m, red[row], red[64u + row]), red[128u + row], red[192u + row]);
                    cf = m > NEG_TEST ? exp2f(m - m_new) : 0.0f; // (O and l are zero until the first key)
                    m = m_new;
                    const float neg_m = m > NEG_TEST ? -m : 0.0f;
                    float sum = 0.0f;
#pragma unroll
                    for (uint32_t c = 0; c < 2u; c++) {
                        float y[8];
#pragma unroll
                        for (uint32_t n = 0; n < 8u; n++) {
                            y[n] = ex2(x[8 * c + n] + neg_m);
                            sum += y[n];
                        }
                        uint4 a, b;
                        split8(y, 16384.0f, a, b); // 2^14: f16's smallest step is then 2^-38 of the largest weight
                        *reinterpret_cast<uint4 *>(p_chunk(2u * e + c)) = a;
                        *reinterpret_cast<uint4 *>(p_chunk(4u + 2u * e + c)) = b;
                    }
                    l = fmaf(l, cf, sum);
                    fence_proxy_async();
                }
                if (t > t0) { // behind the tile's scores, so that they and the product of the tile in front run together
                    if (active) fold(t - 1u, m_last, cf_last);
                    else wait(bar_pv_done, (t - 1u) & 1u);
                }
                tc_fence_before();
                arrive(bar_p_full); // P' is there, and O' is free
            }
            // ---------------- end of the segment ----------------
            more = walk.next(nx);
            if (more) q_next = load_q(nx, smem + PB_OFF_P + (end & 1u) * PB_PBUF, std::false_type{}); // the segment's scores were all there: its Q' may go
            if (active) {
                fold(end - 1u, m, cf);
                red[64u * (2u * half + e) + row] = l;
                named_bar_sync(bar_group, 128); // (P' is free too: its last products have completed)
                const float l_all = (red[row] + red[64u + row]) + (red[128u + row] + red[192u + row]);
                const bool seen = real && klo < vis;
                float *part = nullptr; // a part: maximum, sum and O as they are, for the merge
                float inv = 1.0f;
                if (sg.whole) {
                    float den = l_all;
                    if (g.sinks && real) den += exp2f(g.sinks[sg.kvh * group + head] * PB_LOG2E - (m > NEG_TEST ? m : 0.0f));
                    inv = seen ? 1.0f / den : 0.0f; // (O is zero then, and stays so)
                } else {
                    part = g.scratch + part_slot(blockIdx.x, sg.part) * part_floats(DIM);
                    if (hi && half == 0u && real) *reinterpret_cast<float2 *>(part + 128u * DIM + 2u * row) = make_float2(m, seen ? l_all : -1.0f);
                }
                // The row's hi and lo parts meet in the P' buffers, in turn, 32 dims of each half at a time: the one thread adds up the first 16, the
                // other the rest. All threads store, 128 bytes of a row side by side.
                float *dst[4]; // of the four rows of this thread that are stored
#pragma unroll
                for (uint32_t i = 0; i < 4u; i++) {
                    const uint32_t r = 32u * (q4 & 1u) + 8u * i + 2u * own + (lane >> 4), r_tok = r / group;
                    dst[i] = (part ? part + (size_t)r * DIM
                                   : g.out + (int64_t)(sq.row + it.tok0 + r_tok) * g.out_stride + (size_t)(sg.kvh * group + r - r_tok * group) * DIM) +
                             HD * (lane >> 3 & 1u) + 4u * (lane & 7u);
                }
#pragma unroll
                for (uint32_t c0 = 0; c0 < HD; c0 += 32u) {
                    p_buf = smem + PB_OFF_P + ((c0 >> 5) & 1u) * PB_PBUF;
                    auto give = [&](auto from) { // 16 dims
                        constexpr uint32_t F = decltype(from)::value;
#pragma unroll
                        for (uint32_t c = 0; c < 4u; c++)
                            *reinterpret_cast<float4 *>(p_chunk(F / 4u + c)) = make_float4(O[c0 + F + 4 * c], O[c0 + F + 4 * c + 1], O[c0 + F + 4 * c + 2], O[c0 + F + 4 * c + 3]);
                    };
                    auto sum = [&](auto from) {
                        constexpr uint32_t F = decltype(from)::value;
#pragma unroll
                        for (uint32_t c = 0; c < 4u; c++) {
                            const float4 x = *reinterpret_cast<const float4 *>(p_chunk(F / 4u + c));
                            *reinterpret_cast<float4 *>(p_chunk(F / 4u + c)) = make_float4((O[c0 + F + 4 * c] + x.x) * inv, (O[c0 + F + 4 * c + 1] + x.y) * inv,
                                                                                          (O[c0 + F + 4 * c + 2] + x.z) * inv, (O[c0 + F + 4 * c + 3] + x.w) * inv);
                        }
                    };
                    if (hi) give(std::integral_constant<uint32_t, 16>{});
                    else give(std::integral_constant<uint32_t, 0>{});
                    named_bar_sync(bar_group, 128);
                    if (hi) sum(std::integral_constant<uint32_t, 0>{});
                    else sum(std::integral_constant<uint32_t, 16>{});
                    named_bar_sync(bar_group, 128);
#pragma unroll
                    for (uint32_t i = 0; i < 4u; i++) {
                        const uint32_t r = 32u * (q4 & 1u) + 8u * i + 2u * own + (lane >> 4), c = lane & 7u;
                        const float4 x = *reinterpret_cast<const float4 *>(p_buf + swz128(r + (c >> 2) * 64u, 4u * (lane >> 3 & 1u) + (c & 3u)));
                        if (r < rows) *reinterpret_cast<float4 *>(dst[i] + c0) = x;
                    }
                }
                named_bar_sync(bar_group, 128); // the buffers are free
            } else {
                wait(bar_pv_done, (end - 1u) & 1u);
            }
            q_unscale = q_next;
            t0 = end;
            sg = nx;
        }
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

template <int DIM> static mkv_status launch_dim(Pool *p, int layer, const PoolPlan &plan, const PbArgs &g) {
    PdlLaunch l(p->ctx, dim3(plan.ctas), PB_THREADS, PB_SMEM);
    if (plan.block * plan.group <= PLAN_FEW)
        MKV_CUDA(cudaLaunchKernelEx(&l.cfg, pool_attn_f32_kernel<DIM, true>, p->maps[2 * (size_t)layer], p->maps[2 * (size_t)layer + 1], plan, g));
    else
        MKV_CUDA(cudaLaunchKernelEx(&l.cfg, pool_attn_f32_kernel<DIM, false>, p->maps[2 * (size_t)layer], p->maps[2 * (size_t)layer + 1], plan, g));
    p->ctx->launches++;
    return MKV_OK;
}

mkv_status launch_pool_attn_f32(Pool *p, int layer, const PoolPlan &plan, const PoolAttn &a) {
    PbArgs g;
    g.q = static_cast<const float *>(a.q);
    g.out = static_cast<float *>(a.out);
    g.q_stride = a.q_stride;
    g.out_stride = a.out_stride;
    g.pages = p->table;
    g.kpages = reinterpret_cast<const float *>(p->layer_ptr(layer, 0));
    g.vpages = reinterpret_cast<const float *>(p->layer_ptr(layer, 1));
    g.sinks = a.sinks;
    g.scratch = p->scratch;
    g.status = p->ctx->dev_status;
    g.row_floats = p->row_bytes / sizeof(float);
    g.scale2 = a.scale * PB_LOG2E;
    g.page_shift = (uint32_t)__builtin_ctz(p->desc.page_tokens);
    switch (p->desc.head_dim) {
    case 64: return launch_dim<64>(p, layer, plan, g);
    case 128: return launch_dim<128>(p, layer, plan, g);
    default: return launch_dim<256>(p, layer, plan, g);
    }
}

template <int DIM> static mkv_status setup_dim() {
    MKV_CUDA(cudaFuncSetAttribute(pool_attn_f32_kernel<DIM, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)PB_SMEM));
    MKV_CUDA(cudaFuncSetAttribute(pool_attn_f32_kernel<DIM, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)PB_SMEM));
    return MKV_OK;
}
mkv_status pool_attn_f32_setup(Pool *) {
    mkv_status st = setup_dim<64>();
    if (st == MKV_OK) st = setup_dim<128>();
    return st == MKV_OK ? setup_dim<256>() : st;
}

} // namespace mkv
