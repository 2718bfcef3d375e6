// Attention of blocks of new tokens over paged rows: the plain kernel.
//   out_t = sum_k e^(s_k - M) v_k / (sum_k e^(s_k - M) + e^(sink - M)),  s_k = scale q_t . k_k, over the keys the token sees
// One block of eight warps for one query head of one token; a warp takes every eighth key, keeps its own running maximum and sum, and
// the eight meet in shared memory.
#include "pool.cuh"
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

mkv_status pool_attn_setup(Pool *) { return MKV_OK; }

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
        const mkv_status st = p->desc.fmt == MKV_F16 ? launch_dim<__half>(p, it, g, it.row[it.n]) : launch_dim<float>(p, it, g, it.row[it.n]);
        if (st != MKV_OK) return st;
        g.row0 += it.row[it.n];
    }
    return MKV_OK;
}

} // namespace mkv
