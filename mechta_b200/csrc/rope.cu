// Rotary positions as an operator of its own: y = R(position) x for the heads of many tokens, forward or transposed, any layout,
// part of the head, scaled frequencies, f16 or f32 on either side.
//
// Reads x once and writes y once: bound by HBM for long blocks, by the launch for a step's few tokens. A block takes the heads of one
// token: its cosines and sines (one product in f64 and one sincospi a pair) are computed once, in shared memory, while the block's
// loads of x are in flight. Measured: 8,192 tokens of 32 heads of 128 f32 dims (268 MB) in 42.6 us, 6.3 TB/s, 98% of a plain copy's rate;
// the queries of a four-token step 2.3 us.
#include <algorithm>
#include <cmath>
#include <new>

#include "internal.cuh"
#include "ptx.cuh"
#include "rope.cuh"

namespace mkv {

RopeTab rope_tab(const mkv_rope *r, bool backward) {
    RopeTab t;
    t.m = 1.0f;
    t.pairs = t.interleaved = 0u;
    t.sign = backward ? -1.0f : 1.0f;
    if (!r) return t;
    t.m = (float)r->m;
    t.pairs = (uint32_t)r->desc.dims / 2u;
    t.interleaved = r->desc.layout == MKV_ROPE_INTERLEAVED;
    std::copy_n(r->turns, t.pairs, t.turns);
    return t;
}

struct RopeArgs {
    const void *x;
    void *y;
    const int32_t *pos;
    uint32_t heads, units; // units of a head
    int64_t xt, xh, yt, yh;
};

constexpr int ROPE_THREADS = 256;
constexpr uint32_t ROPE_PER = 2; // units of a thread

template <int MODE, class TI, class TO>
__global__ void __launch_bounds__(ROPE_THREADS)
rope_kernel(const __grid_constant__ RopeTab tab, const __grid_constant__ RopeArgs g) {
    __shared__ float2 cs[MKV_ROPE_MAX_DIMS / 2];
    ptx::pdl_wait();
    ptx::pdl_launch_dependents();
    const uint32_t tok = blockIdx.x, total = g.heads * g.units;
    const TI *x = static_cast<const TI *>(g.x) + (int64_t)tok * g.xt;
    TO *y = static_cast<TO *>(g.y) + (int64_t)tok * g.yt;
    float a[ROPE_PER][8], b[ROPE_PER][8];
    uint32_t head[ROPE_PER], unit[ROPE_PER];
#pragma unroll
    for (uint32_t k = 0; k < ROPE_PER; k++) {
        const uint32_t idx = (blockIdx.y * ROPE_PER + k) * ROPE_THREADS + threadIdx.x;
        head[k] = idx / g.units;
        unit[k] = idx % g.units;
        if (idx < total) rope_load<MODE>(x + (int64_t)head[k] * g.xh, unit[k], tab.pairs, tab.interleaved, a[k], b[k]);
    }
    const int32_t p = g.pos[tok];
    for (uint32_t i = threadIdx.x; i < tab.pairs; i += ROPE_THREADS) cs[i] = rope_cs(tab, i, p);
    __syncthreads();
#pragma unroll
    for (uint32_t k = 0; k < ROPE_PER; k++) {
        const uint32_t idx = (blockIdx.y * ROPE_PER + k) * ROPE_THREADS + threadIdx.x;
        if (idx < total) rope_store<MODE>(y + (int64_t)head[k] * g.yh, unit[k], tab.pairs, tab.interleaved, cs, a[k], b[k]);
    }
}

template <class TI, class TO> static mkv_status launch_rope(Ctx *ctx, int mode, const RopeTab &tab, const RopeArgs &g, uint32_t ntok) {
    cudaLaunchConfig_t cfg = {};
    const uint64_t units = (uint64_t)g.heads * g.units, per = ROPE_THREADS * ROPE_PER;
    cfg.gridDim = dim3(ntok, (unsigned)((units + per - 1u) / per));
    cfg.blockDim = dim3(ROPE_THREADS);
    cfg.stream = ctx->stream;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = ctx->pdl ? 1 : 0;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    switch (mode) {
    case ROPE_HALF8: MKV_CUDA(cudaLaunchKernelEx(&cfg, rope_kernel<ROPE_HALF8, TI, TO>, tab, g)); break;
    case ROPE_INTER8: MKV_CUDA(cudaLaunchKernelEx(&cfg, rope_kernel<ROPE_INTER8, TI, TO>, tab, g)); break;
    default: MKV_CUDA(cudaLaunchKernelEx(&cfg, rope_kernel<ROPE_ANY, TI, TO>, tab, g)); break;
    }
    ctx->launches++;
    return MKV_OK;
}

} // namespace mkv

using namespace mkv;

extern "C" {

mkv_status mkv_rope_create(const mkv_rope_desc *d, mkv_rope **out) {
    if (!d || !out) {
        set_error("null argument");
        return MKV_ERR_INVALID;
    }
    *out = nullptr;
    if (d->dims < 2 || d->dims > MKV_ROPE_MAX_DIMS || d->dims % 2 != 0) {
        set_error("rope: %d rotated dims: must be even, 2 to %d", d->dims, MKV_ROPE_MAX_DIMS);
        return MKV_ERR_INVALID;
    }
    if (d->layout != MKV_ROPE_HALF && d->layout != MKV_ROPE_INTERLEAVED) {
        set_error("rope: unknown layout %d", d->layout);
        return MKV_ERR_INVALID;
    }
    if (d->scaling < MKV_SCALE_NONE || d->scaling > MKV_SCALE_YARN) {
        set_error("rope: unknown scaling %d", d->scaling);
        return MKV_ERR_INVALID;
    }
    if (!(d->base > 1.0) || !std::isfinite(d->base)) {
        set_error("rope: base %g must be above 1", d->base);
        return MKV_ERR_INVALID;
    }
    const double s = d->scaling == MKV_SCALE_NONE ? 1.0 : d->factor;
    if (!(s >= 1.0) || !std::isfinite(s)) {
        set_error("rope: factor %g must be at least 1", s);
        return MKV_ERR_INVALID;
    }
    double slow = d->slow, fast = d->fast;
    if (d->scaling == MKV_SCALE_YARN) {
        if (slow == 0.0 && fast == 0.0) {
            slow = 1.0;
            fast = 32.0;
        }
        if (!(d->original > 0.0) || !std::isfinite(d->original) || !(slow >= 0.0) || !(fast > slow) || !std::isfinite(fast)) {
            set_error("rope: original context %g must be above 0 and 0 <= slow %g < fast %g", d->original, slow, fast);
            return MKV_ERR_INVALID;
        }
    }
    mkv_rope *r = new (std::nothrow) mkv_rope();
    if (!r) {
        set_error("out of host memory");
        return MKV_ERR_NOMEM;
    }
    r->desc = *d;
    r->m = d->scaling == MKV_SCALE_YARN ? 0.1 * log(s) + 1.0 : 1.0;
    const double dims = d->dims;
    // (with two dims the one frequency is 1 whatever the base)
    const double base = d->scaling == MKV_SCALE_NTK && d->dims > 2 ? d->base * pow(s, dims / (dims - 2.0)) : d->base;
    for (int i = 0; i < d->dims / 2; i++) {
        double f = pow(base, -2.0 * i / dims);
        if (d->scaling == MKV_SCALE_LINEAR) f /= s;
        if (d->scaling == MKV_SCALE_YARN) {
            const double turns = d->original * f / 6.283185307179586476925286766559;
            const double keep = fmin(1.0, fmax(0.0, (turns - slow) / (fast - slow)));
            f = f / s * (1.0 - keep) + f * keep;
        }
        r->freq[i] = f;
        r->turns[i] = f / 6.283185307179586476925286766559;
    }
    *out = r;
    return MKV_OK;
}

void mkv_rope_destroy(mkv_rope *r) { delete r; }

mkv_status mkv_rope_freqs(const mkv_rope *r, double *freqs, double *m) {
    if (!r || !freqs || !m) {
        set_error("null argument");
        return MKV_ERR_INVALID;
    }
    for (int i = 0; i < r->desc.dims / 2; i++) freqs[i] = r->freq[i];
    *m = r->m;
    return MKV_OK;
}

mkv_status mkv_rope_apply(mkv_ctx *h, const mkv_rope *r, const mkv_rope_rows *in) {
    Ctx *ctx = reinterpret_cast<Ctx *>(h);
    if (!r || !in) {
        set_error("null argument");
        return MKV_ERR_INVALID;
    }
    if ((in->x_fmt != MKV_F16 && in->x_fmt != MKV_F32) || (in->y_fmt != MKV_F16 && in->y_fmt != MKV_F32)) {
        set_error("rope: unknown format");
        return MKV_ERR_INVALID;
    }
    if (in->heads < 1 || in->heads > 16384 || in->head_dim < (uint32_t)r->desc.dims || in->head_dim > 1024) {
        set_error("rope: %u heads of %u dims: heads must be 1 to 16384 and dims %d (the rotated ones) to 1024", in->heads, in->head_dim,
                  r->desc.dims);
        return MKV_ERR_INVALID;
    }
    const size_t xe = in->x_fmt == MKV_F16 ? 2 : 4, ye = in->y_fmt == MKV_F16 ? 2 : 4;
    RopeArgs g;
    g.x = in->x_dev;
    g.y = in->y_dev;
    g.pos = in->pos_dev;
    g.heads = in->heads;
    const int64_t dense = (int64_t)in->heads * in->head_dim;
    g.xh = in->x_head_stride ? in->x_head_stride : in->head_dim;
    g.yh = in->y_head_stride ? in->y_head_stride : in->head_dim;
    g.xt = in->x_token_stride ? in->x_token_stride : dense;
    g.yt = in->y_token_stride ? in->y_token_stride : dense;
    const int64_t most = (int64_t)1 << 30; // so that no offset leaves 64 bits
    for (int64_t v : {g.xh, g.xt, g.yh, g.yt})
        if (v < 0 || v > most) {
            set_error("rope: strides must lie between 0 and 2^30 elements");
            return MKV_ERR_INVALID;
        }
    if (in->ntok > 0x7fffffffu) {
        set_error("rope: %u tokens, at most 2^31 - 1", in->ntok);
        return MKV_ERR_INVALID;
    }
    if (in->ntok == 0) return MKV_OK;
    if (!in->x_dev || !in->y_dev || !in->pos_dev) {
        set_error("null argument");
        return MKV_ERR_INVALID;
    }
    // y's heads and tokens may not fall on one another
    const int64_t D = in->head_dim, H = in->heads;
    if ((H > 1 && g.yh < D) || (in->ntok > 1 && (g.yh <= g.yt ? g.yt < (H - 1) * g.yh + D : (g.yt < D || (H > 1 && g.yh < (int64_t)(in->ntok - 1) * g.yt + D))))) {
        set_error("rope: the output's strides (%lld a token, %lld a head) make its heads overlap", (long long)g.yt, (long long)g.yh);
        return MKV_ERR_INVALID;
    }
    if (((uintptr_t)g.x % xe) || ((uintptr_t)g.y % ye) || ((uintptr_t)g.pos & 3u)) {
        set_error("rope: misaligned pointer");
        return MKV_ERR_INVALID;
    }
    const RowSpan sx = {(uintptr_t)g.x, in->ntok, (uint64_t)g.xt * xe, ((uint64_t)(H - 1) * (uint64_t)g.xh + (uint64_t)D) * xe};
    const RowSpan sy = {(uintptr_t)g.y, in->ntok, (uint64_t)g.yt * ye, ((uint64_t)(H - 1) * (uint64_t)g.yh + (uint64_t)D) * ye};
    // Slices of every head (a query beside its gate) lie between one another's: where one of the two strides is a multiple of the other, all
    // heads of all tokens are among rows at the smaller one.
    auto all_heads = [&](const void *at, int64_t t, int64_t h, size_t e) {
        const int64_t s = H == 1 ? t : in->ntok == 1 ? h : std::min(t, h), span = (int64_t)(in->ntok - 1u) * t + (H - 1) * h;
        if (s < 1 || t % s != 0 || h % s != 0) return RowSpan{(uintptr_t)at, 1u, 1u, (uint64_t)(span + D) * e}; // (all of it)
        return RowSpan{(uintptr_t)at, (uint64_t)(span / s) + 1u, (uint64_t)s * e, (uint64_t)D * e};
    };
    const bool same = g.x == g.y && xe == ye && (in->ntok == 1 || g.xt == g.yt) && (H == 1 || g.xh == g.yh);
    if (!same && sx.meets(sy) && all_heads(g.x, g.xt, g.xh, xe).meets(all_heads(g.y, g.yt, g.yh, ye))) {
        set_error("rope: x and y overlap without being the same memory in the same layout and type");
        return MKV_ERR_INVALID;
    }
    if (sy.meets({(uintptr_t)g.pos, in->ntok, 4u, 4u})) {
        set_error("rope: y overlaps the positions");
        return MKV_ERR_INVALID;
    }
    if (!ctx) {
        set_error("null ctx");
        return MKV_ERR_INVALID;
    }
    DeviceScope dev(ctx);
    if (dev.status != MKV_OK) return dev.status;
    const bool aligned = ((uintptr_t)g.x & 15u) == 0 && ((uintptr_t)g.y & 15u) == 0 && (g.xt * xe) % 16 == 0 && (g.xh * xe) % 16 == 0 &&
                         (g.yt * ye) % 16 == 0 && (g.yh * ye) % 16 == 0;
    const RopeTab tab = rope_tab(r, in->backward != 0);
    const int mode = rope_mode(tab.pairs, tab.interleaved, in->head_dim, aligned);
    g.units = rope_units(mode, tab.pairs, in->head_dim);
    if (in->x_fmt == MKV_F16)
        return in->y_fmt == MKV_F16 ? launch_rope<__half, __half>(ctx, mode, tab, g, in->ntok) : launch_rope<__half, float>(ctx, mode, tab, g, in->ntok);
    return in->y_fmt == MKV_F16 ? launch_rope<float, __half>(ctx, mode, tab, g, in->ntok) : launch_rope<float, float>(ctx, mode, tab, g, in->ntok);
}

} // extern "C"
