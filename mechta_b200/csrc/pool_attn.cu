// Attention of blocks of new tokens over paged rows: the plain kernel.
//   out_t = sum_k e^(s_k - M) v_k / (sum_k e^(s_k - M) + e^(sink - M)),  s_k = scale q_t . k_k, over the keys the token sees
// One block of eight warps for one query head of one token; a warp takes every eighth key, keeps its own running maximum and sum, and
// the eight meet in shared memory.
#include "pool_plan.cuh"
#include "ptx.cuh"

namespace mkv {

constexpr uint32_t ATTN_ITEMS = 128;
struct AttnItems {
    uint32_t n;
    uint32_t table[ATTN_ITEMS], first[ATTN_ITEMS], pos[ATTN_ITEMS];
    uint32_t row[ATTN_ITEMS + 1]; // packed tokens in front of the item
};
struct AttnArgs {
    const void *q;
    void *out;
    int64_t q_stride, out_stride;
    const char *k, *v;
    const uint32_t *pages;
    const float *sinks;
    size_t page_bytes, row_bytes;
    float scale;
    uint32_t window, page_shift, group, row0;
};

__device__ __forceinline__ float as_f32(float x) { return x; }
__device__ __forceinline__ float as_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ void put(float *p, float x) { *p = x; }
__device__ __forceinline__ void put(__half *p, float x) { *p = __float2half_rn(x); }

template <class T, int DIM>
__global__ void __launch_bounds__(256) pool_attn_kernel(const __grid_constant__ AttnItems items, const __grid_constant__ AttnArgs g) {
    constexpr int E = DIM / 32;
    __shared__ float ml[8][2], acc_s[8][DIM];
    ptx::pdl_wait();
    ptx::pdl_launch_dependents();
    const uint32_t r = blockIdx.x, head = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    uint32_t i = 0, end = items.n;
    while (i + 1u < end) {
        const uint32_t mid = (i + end) / 2u;
        if (items.row[mid] <= r) i = mid;
        else end = mid;
    }
    const uint32_t at = items.pos[i] + (r - items.row[i]);
    uint32_t lo = items.first[i];
    if (g.window && at + 1u > g.window && at + 1u - g.window > lo) lo = at + 1u - g.window;
    const T *q = static_cast<const T *>(g.q) + (int64_t)(g.row0 + r) * g.q_stride + head * DIM;
    const size_t head_off = (size_t)(head / g.group) * DIM;
    float qv[E], acc[E], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int e = 0; e < E; e++) {
        qv[e] = as_f32(q[lane + 32 * e]);
        acc[e] = 0.0f;
    }
    for (uint32_t key = lo + warp; key <= at; key += 8u) {
        const uint32_t page = g.pages[items.table[i] + (key >> g.page_shift)];
        const size_t off = (size_t)page * g.page_bytes + (size_t)(key & ((1u << g.page_shift) - 1u)) * g.row_bytes;
        const T *k = reinterpret_cast<const T *>(g.k + off) + head_off, *v = reinterpret_cast<const T *>(g.v + off) + head_off;
        float s = 0.0f;
#pragma unroll
        for (int e = 0; e < E; e++) s = fmaf(qv[e], as_f32(k[lane + 32 * e]), s);
#pragma unroll
        for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        s *= g.scale;
        const float mn = fmaxf(m, s);
        const float c = m == mn ? 1.0f : expf(m - mn), w = s == mn ? 1.0f : expf(s - mn);
        l = l * c + w;
#pragma unroll
        for (int e = 0; e < E; e++) acc[e] = acc[e] * c + w * as_f32(v[lane + 32 * e]);
        m = mn;
    }
    if (lane == 0) {
        ml[warp][0] = m;
        ml[warp][1] = l;
    }
#pragma unroll
    for (int e = 0; e < E; e++) acc_s[warp][lane + 32 * e] = acc[e];
    __syncthreads();
    for (int d = threadIdx.x; d < DIM; d += 256) {
        float M = g.sinks ? g.sinks[head] : -INFINITY;
        for (int w = 0; w < 8; w++) M = fmaxf(M, ml[w][0]);
        float L = g.sinks ? expf(g.sinks[head] - M) : 0.0f, o = 0.0f;
        for (int w = 0; w < 8; w++) {
            if (ml[w][1] == 0.0f) continue; // no key
            const float f = expf(ml[w][0] - M);
            L += f * ml[w][1];
            o += f * acc_s[w][d];
        }
        put(static_cast<T *>(g.out) + (int64_t)(g.row0 + r) * g.out_stride + head * DIM + d, lo <= at ? o / L : 0.0f);
    }
}

// ---- the plan of a launch ------------------------------------------------------------------------------------------
// Cuts the items into ranges of cost `budget`: true if the GPU's CTAs suffice.
static bool plan_cut(PoolPlan &plan, MergeList &merge, const PlanCost &cost, uint32_t most, uint64_t budget) {
    plan.ctas = 0;
    merge.n = 0;
    merge.group = plan.group;
    uint64_t left = 0; // of the current CTA's budget
    for (uint32_t q = 0; q < plan.nseq; q++)
        for (uint32_t b = 0; b * plan.block < plan.seq[q].ntok; b++) {
            const PlanItem it = plan_item(plan.seq[q], plan.window, plan.block, b, cost.keys);
            for (uint32_t h = 0; h < plan.kv_heads; h++) {
                uint32_t at = 0, parts = 0, cta0 = 0;
                while (at < it.tiles) {
                    // the rest of the item whole, or a part that is worth a segment, or a CTA of its own
                    const uint64_t rest = it.tiles - at;
                    if (plan.ctas == 0u || (left < rest + cost.segment && left < 2u * cost.segment + 1u)) {
                        if (plan.ctas == most) return false;
                        plan.start[plan.ctas++] = {(uint16_t)q, (uint16_t)h, b, at, 0u};
                        left = budget;
                    }
                    const uint64_t room = left > cost.segment ? left - cost.segment : 1u;
                    const uint32_t n = (uint32_t)std::min<uint64_t>(rest, room);
                    plan.start[plan.ctas - 1u].tiles += n;
                    if (parts++ == 0u) cta0 = plan.ctas - 1u;
                    left -= std::min<uint64_t>(left, n + cost.segment);
                    at += n;
                    if (at < it.tiles) left = 0; // (a CTA has one part that does not end its item)
                }
                if (parts > 1u) merge.item[merge.n++] = {plan.seq[q].row + it.tok0, h * plan.group, it.ntok, (uint16_t)cta0, (uint16_t)parts};
            }
        }
    return true;
}

bool pool_plan(const Pool *p, const mkv_seq_rows *items, int n, int &i, uint32_t &rows, uint32_t window, const PlanCost &cost, PoolPlan &plan, MergeList &merge) {
    plan.nseq = 0;
    plan.kv_heads = (uint32_t)p->desc.kv_heads;
    plan.group = (uint32_t)(p->desc.q_heads / p->desc.kv_heads);
    plan.block = 128u / plan.group;
    plan.window = window;
    uint64_t total = 0, count = 0;
    for (; i < n && plan.nseq < PLAN_SEQS; i++) {
        if (items[i].ntok == 0u) continue;
        PlanSeq &s = plan.seq[plan.nseq];
        s = {items[i].seq * p->book.max_pages, items[i].first_pos, items[i].pos, items[i].ntok, rows};
        uint64_t tiles = 0, blocks = 0;
        for (; blocks * plan.block < s.ntok; blocks++) tiles += plan_item(s, window, plan.block, (uint32_t)blocks, cost.keys).tiles;
        if (total + tiles * plan.kv_heads > 0x7fffffffull && plan.nseq > 0u) break; // (one sequence alone stays below: mkv_attn_pool refuses more)
        total += tiles * plan.kv_heads;
        count += blocks * plan.kv_heads;
        plan.nseq++;
        rows += s.ntok;
    }
    if (plan.nseq == 0u) return false;
    const uint32_t sms = std::min<uint32_t>((uint32_t)p->ctx->sm_count, PLAN_CTAS);
    // the least that could do, and a little more as often as it takes
    uint64_t budget = std::max<uint64_t>((total + count * cost.segment + sms - 1u) / sms, cost.segment + 1u);
    while (!plan_cut(plan, merge, cost, sms, budget)) budget += budget / 32u + 1u;
    return true;
}

// ---- the merge of split items --------------------------------------------------------------------------------------
// out = sum_s e^(m_s - M) O_s / (sum_s e^(m_s - M) l_s + e^(sink - M)) over an item's parts. A few dozen L2 accesses of a thread one after
// the other are all there is to it, so the parts of a row are spread over up to 16 groups of threads, which meet in shared memory.
struct MergeArgs {
    const float *scratch, *sinks;
    void *out;
    int64_t out_stride;
    uint32_t groups; // of a row
};
template <class T, int DIM>
__global__ void __launch_bounds__(1024) pool_merge_kernel(const __grid_constant__ MergeList list, const __grid_constant__ MergeArgs g) {
    constexpr uint32_t L = DIM / 4; // threads of a row's dims
    __shared__ float4 acc_s[1024];
    __shared__ float2 ml_s[1024 / L];
    ptx::pdl_wait();
    ptx::pdl_launch_dependents();
    const MergeItem &it = list.item[blockIdx.y];
    const uint32_t d = threadIdx.x % L, slot = threadIdx.x / L, grp = slot % g.groups, rpb = blockDim.x / L / g.groups;
    const uint32_t row = blockIdx.x * rpb + slot / g.groups, parts = it.parts;
    const bool real = row < it.ntok * list.group;
    float M = NEG_BIG, l = 0.0f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    bool seen = true;
    for (uint32_t s0 = grp; real && s0 < parts; s0 += 4u * g.groups) {
        float2 ml[4];
        float4 v[4];
#pragma unroll
        for (uint32_t k = 0; k < 4u; k++) {
            const uint32_t s = s0 + k * g.groups;
            const float *ps = g.scratch + part_slot(it.cta0 + min(s, parts - 1u), s == 0u ? 1u : 0u) * part_floats(DIM);
            ml[k] = s < parts ? __ldcg(reinterpret_cast<const float2 *>(ps + 128u * DIM + 2u * row)) : make_float2(NEG_BIG, 0.0f);
            v[k] = s < parts ? __ldcg(reinterpret_cast<const float4 *>(ps + (size_t)row * DIM + 4u * d)) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
        const float mx = fmaxf(fmaxf(ml[0].x, ml[1].x), fmaxf(ml[2].x, ml[3].x));
        if (mx > M) {
            const float f = M > NEG_TEST ? exp2f(M - mx) : 0.0f;
            l *= f;
            acc = make_float4(acc.x * f, acc.y * f, acc.z * f, acc.w * f);
            M = mx;
        }
#pragma unroll
        for (int k = 0; k < 4; k++) {
            seen = seen && ml[k].y >= 0.0f; // (-1: the row sees no key of the item; the sum of NaN weights is NaN and goes on)
            if (ml[k].y != ml[k].y) seen = true;
            const float e = ml[k].x > NEG_TEST ? exp2f(ml[k].x - M) : 0.0f;
            if (e == 0.0f && ml[k].y == ml[k].y) continue;
            l = fmaf(e, ml[k].y, l);
            acc.x = fmaf(e, v[k].x, acc.x);
            acc.y = fmaf(e, v[k].y, acc.y);
            acc.z = fmaf(e, v[k].z, acc.z);
            acc.w = fmaf(e, v[k].w, acc.w);
        }
    }
    acc_s[threadIdx.x] = acc;
    if (d == 0u) ml_s[slot] = make_float2(M, seen ? l : -1.0f);
    __syncthreads();
    if (grp != 0u || !real) return;
    const uint32_t head = it.head + row % list.group;
    const float sink = g.sinks ? g.sinks[head] * 1.4426950408889634f : NEG_BIG;
    float Mr = sink;
    for (uint32_t k = 0; k < g.groups; k++) Mr = fmaxf(Mr, ml_s[slot + k].x);
    float den = sink > NEG_TEST ? exp2f(sink - Mr) : 0.0f;
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
    seen = true;
    for (uint32_t k = 0; k < g.groups; k++) {
        const float2 ml = ml_s[slot + k];
        if (ml.y < 0.0f) seen = false;
        const float e = ml.x > NEG_TEST ? exp2f(ml.x - Mr) : 0.0f;
        if (e == 0.0f && ml.y == ml.y) continue;
        const float4 a = acc_s[threadIdx.x + k * L];
        den = fmaf(e, ml.y, den);
        y.x = fmaf(e, a.x, y.x);
        y.y = fmaf(e, a.y, y.y);
        y.z = fmaf(e, a.z, y.z);
        y.w = fmaf(e, a.w, y.w);
    }
    const float inv = 1.0f / den;
    y = seen ? make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv) : make_float4(0.f, 0.f, 0.f, 0.f);
    T *dst = static_cast<T *>(g.out) + (int64_t)(it.row + row / list.group) * g.out_stride + (size_t)head * DIM + 4u * d;
    if constexpr (sizeof(T) == 2) {
        const __half2 a = __floats2half2_rn(y.x, y.y), b = __floats2half2_rn(y.z, y.w);
        *reinterpret_cast<uint2 *>(dst) = make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
    } else {
        *reinterpret_cast<float4 *>(dst) = y;
    }
}

template <class T, int DIM> static mkv_status launch_merge(Pool *p, const MergeList &list, const PoolAttn &a) {
    uint32_t parts = 0, rows = 0;
    for (uint32_t i = 0; i < list.n; i++) {
        parts = std::max<uint32_t>(parts, list.item[i].parts);
        rows = std::max(rows, list.item[i].ntok * list.group);
    }
    const uint32_t threads = parts > 4u ? 1024u : 256u, slots = threads / (DIM / 4);
    MergeArgs g = {p->scratch, a.sinks, a.out, a.out_stride, 1u};
    while (g.groups < slots && g.groups < 16u && 4u * g.groups < parts) g.groups *= 2u;
    const uint32_t rpb = slots / g.groups;
    PdlLaunch l(p->ctx, dim3((rows + rpb - 1u) / rpb, list.n), threads);
    MKV_CUDA(cudaLaunchKernelEx(&l.cfg, pool_merge_kernel<T, DIM>, list, g));
    p->ctx->launches++;
    return MKV_OK;
}
mkv_status launch_pool_merge(Pool *p, const MergeList &list, const PoolAttn &a) {
    if (list.n == 0u) return MKV_OK;
    const bool f16 = p->desc.fmt == MKV_F16;
    switch (p->desc.head_dim) {
    case 64: return f16 ? launch_merge<__half, 64>(p, list, a) : launch_merge<float, 64>(p, list, a);
    case 128: return f16 ? launch_merge<__half, 128>(p, list, a) : launch_merge<float, 128>(p, list, a);
    default: return f16 ? launch_merge<__half, 256>(p, list, a) : launch_merge<float, 256>(p, list, a);
    }
}

mkv_status pool_attn_setup(Pool *p) {
    if (p->desc.fmt != MKV_F16) return MKV_OK;
    const size_t bytes = 2u * (size_t)std::min<uint32_t>((uint32_t)p->ctx->sm_count, PLAN_CTAS) * part_floats((uint32_t)p->desc.head_dim) * sizeof(float);
    if (cudaMalloc(reinterpret_cast<void **>(&p->scratch), bytes) != cudaSuccess) {
        cudaGetLastError();
        set_error("out of device memory for %zu bytes of scratch", bytes);
        return MKV_ERR_NOMEM;
    }
    return pool_attn_f16_setup(p);
}

template <class T> static mkv_status launch_dim(Pool *p, const AttnItems &it, const AttnArgs &g, uint32_t rows) {
    PdlLaunch l(p->ctx, dim3(rows, (unsigned)p->desc.q_heads), 256);
    switch (p->desc.head_dim) {
    case 64: MKV_CUDA(cudaLaunchKernelEx(&l.cfg, pool_attn_kernel<T, 64>, it, g)); break;
    case 128: MKV_CUDA(cudaLaunchKernelEx(&l.cfg, pool_attn_kernel<T, 128>, it, g)); break;
    default: MKV_CUDA(cudaLaunchKernelEx(&l.cfg, pool_attn_kernel<T, 256>, it, g)); break;
    }
    p->ctx->launches++;
    return MKV_OK;
}

mkv_status launch_pool_attn(Pool *p, int layer, const mkv_seq_rows *items, int n, const PoolAttn &a) {
    if (p->desc.fmt == MKV_F16) {
        PoolPlan plan;
        MergeList merge;
        uint32_t rows = 0;
        for (int i = 0; pool_plan(p, items, n, i, rows, a.window, {128u, 2u}, plan, merge);) {
            mkv_status st = launch_pool_attn_f16(p, layer, plan, a);
            if (st == MKV_OK) st = launch_pool_merge(p, merge, a);
            if (st != MKV_OK) return st;
        }
        return MKV_OK;
    }
    AttnArgs g;
    g.q = a.q;
    g.out = a.out;
    g.q_stride = a.q_stride;
    g.out_stride = a.out_stride;
    g.k = p->layer_ptr(layer, 0);
    g.v = p->layer_ptr(layer, 1);
    g.pages = p->table;
    g.sinks = a.sinks;
    g.page_bytes = p->page_bytes;
    g.row_bytes = p->row_bytes;
    g.scale = a.scale;
    g.window = a.window;
    g.page_shift = (uint32_t)__builtin_ctz(p->desc.page_tokens);
    g.group = (uint32_t)(p->desc.q_heads / p->desc.kv_heads);
    g.row0 = 0;
    for (int i = 0; i < n;) {
        AttnItems it;
        it.n = 0;
        it.row[0] = 0;
        for (; i < n && it.n < ATTN_ITEMS; i++)
            if (items[i].ntok > 0u) {
                it.table[it.n] = items[i].seq * p->book.max_pages;
                it.first[it.n] = items[i].first_pos;
                it.pos[it.n] = items[i].pos;
                it.row[it.n + 1u] = it.row[it.n] + items[i].ntok;
                it.n++;
            }
        if (it.n == 0u) break;
        const mkv_status st = launch_dim<float>(p, it, g, it.row[it.n]);
        if (st != MKV_OK) return st;
        g.row0 += it.row[it.n];
    }
    return MKV_OK;
}

} // namespace mkv
