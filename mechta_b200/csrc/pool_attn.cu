// Attention of blocks of new tokens over paged rows: the plan of a launch, and the merge of the items that it splits. The kernels are
// in pool_attn_f16.cu and pool_attn_f32.cu.
#include "pool_plan.cuh"
#include "ptx.cuh"

namespace mkv {

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
    plan.block = cost.rows / plan.group;
    plan.window = window;
    uint64_t total = 0, count = 0;
    uint32_t longest = 0;
    for (; i < n && plan.nseq < PLAN_SEQS; i++) {
        if (items[i].ntok == 0u) continue;
        PlanSeq &s = plan.seq[plan.nseq];
        s = {items[i].seq * p->book.max_pages, items[i].first_pos, items[i].pos, items[i].ntok, rows};
        uint64_t tiles = 0, blocks = 0;
        for (; blocks * plan.block < s.ntok; blocks++) {
            const uint32_t t = plan_item(s, window, plan.block, (uint32_t)blocks, cost.keys).tiles;
            tiles += t;
            longest = std::max(longest, t);
        }
        if (total + tiles * plan.kv_heads > 0x7fffffffull && plan.nseq > 0u) break; // (one sequence alone stays below: mkv_attn_pool refuses more)
        total += tiles * plan.kv_heads;
        count += blocks * plan.kv_heads;
        plan.nseq++;
        rows += s.ntok;
    }
    if (plan.nseq == 0u) return false;
    const uint32_t sms = (uint32_t)pool_attn_ctas(p);
    // the least that could do, and a little more as often as it takes
    uint64_t budget = std::max<uint64_t>((total + count * cost.segment + sms - 1u) / sms, cost.segment + 1u);
    if (longest <= cost.whole) budget = std::max<uint64_t>(budget, cost.segment + longest); // nothing is split
    while (!plan_cut(plan, merge, cost, sms, budget)) budget += budget / 32u + 1u;
    return true;
}

// ---- the merge of split items --------------------------------------------------------------------------------------
// out = sum_s e^(m_s - M) O_s / (sum_s e^(m_s - M) l_s + e^(sink - M)) over an item's parts. A few dozen L2 accesses of a thread one after
// the other are all there is to it, so the parts of a row are spread over up to 16 groups of threads, which meet in shared memory (one
// token over 4,096, 32 parts of 8 rows: the whole call takes 12.2 us, with one group 19.5), as long as all threads fit the GPU at once (24
// items of 5 to 9 parts of up to 128 rows: 19.7 us with one group, with two, in blocks of 1,024 threads, 24.1).
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
    // (the difference of two infinities is no number: a sink of infinity takes everything; one of NaN makes the row NaN)
    float den = sink <= NEG_TEST ? 0.0f : sink == Mr ? 1.0f : exp2f(sink - Mr);
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
    MergeArgs g = {p->scratch, a.sinks, a.out, a.out_stride, 1u};
    // as many groups as the parts keep busy, while all threads fit the GPU at once
    constexpr uint32_t L = DIM / 4;
    while (g.groups < 16u && 4u * g.groups < parts && (uint64_t)list.n * rows * L * 2u * g.groups <= 2048ull * (uint32_t)p->ctx->sm_count) g.groups *= 2u;
    const uint32_t threads = std::max(256u, g.groups * L), rpb = threads / L / g.groups;
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
    const bool f16 = p->desc.fmt == MKV_F16;
    const size_t bytes = pool_attn_ctas(p) * (2u * part_floats((uint32_t)p->desc.head_dim) + (f16 ? 128u * (size_t)p->desc.head_dim : 0u)) * sizeof(float);
    if (cudaMalloc(reinterpret_cast<void **>(&p->scratch), bytes) != cudaSuccess) {
        cudaGetLastError();
        set_error("out of device memory for %zu bytes of scratch", bytes);
        return MKV_ERR_NOMEM;
    }
    // boxes of one page, or of as many of its rows as a unit of the kernel's ring has
    const uint32_t box_rows = std::min<uint32_t>(p->desc.page_tokens, f16 && p->desc.head_dim != 256 ? 128u : 64u);
    const uint64_t rows = (uint64_t)p->desc.n_pages * p->desc.page_tokens, cols = (uint64_t)p->desc.kv_heads * (uint64_t)p->desc.head_dim;
    p->maps.resize(2 * (size_t)p->desc.n_layers);
    for (int l = 0; l < p->desc.n_layers; l++)
        for (int kv = 0; kv < 2; kv++) {
            const mkv_status st = make_tensor_map(&p->maps[2 * (size_t)l + (size_t)kv], p->desc.fmt, p->layer_ptr(l, kv), rows, cols, box_rows);
            if (st != MKV_OK) return st;
        }
    return f16 ? pool_attn_f16_setup(p) : pool_attn_f32_setup(p);
}

mkv_status launch_pool_attn(Pool *p, int layer, const mkv_seq_rows *items, int n, const PoolAttn &a) {
    const bool f16 = p->desc.fmt == MKV_F16;
    // What a segment costs beside its tiles, measured with 0, 2 and 4 tiles: ragged blocks under a window of 513 in f16 110, 73 and 89 us;
    // f32 blocks (with 1, 2 and 4) 440, 432 and 440; long histories hardly care (32 sessions in f16 338, 340 and 339; eight in f32 171, 168 and
    // 165).
    // Where all items have at most two tiles, a second tile in a row is sooner done than a merge (windows of 23 in f16 heads of 128 11.6 us,
    // split 15.0; in f32 11.5 and 12.7), but not in f32 with heads of 256 (20.7 us, split 16.8).
    PlanCost cost = f16 ? PlanCost{128u, 128u, 2u, 2u} : PlanCost{64u, 64u, 2u, p->desc.head_dim == 256 ? 1u : 2u};
    if (!f16) { // items of at most 32 rows have a form of the kernel of their own
        uint32_t most = 0;
        for (int i = 0; i < n; i++) most = std::max(most, items[i].ntok);
        if ((uint64_t)most * (uint32_t)(p->desc.q_heads / p->desc.kv_heads) <= PLAN_FEW) cost.rows = PLAN_FEW;
    }
    PoolPlan plan;
    MergeList merge;
    uint32_t rows = 0;
    for (int i = 0; pool_plan(p, items, n, i, rows, a.window, cost, plan, merge);) {
        mkv_status st = f16 ? launch_pool_attn_f16(p, layer, plan, a) : launch_pool_attn_f32(p, layer, plan, a);
        if (st == MKV_OK) st = launch_pool_merge(p, merge, a);
        if (st != MKV_OK) return st;
    }
    return MKV_OK;
}

} // namespace mkv
