// The C entry points of the pool of pages (mkv_pool_*, mkv_seq_*): argument checks, the bookkeeping (pages.hpp), the kernels that
// follow it on the device (page tables, page copies) and the writer of new rows.
#include <new>

#include "pool.cuh"
#include "ptx.cuh"
#include "rope.cuh"

namespace mkv {

// ---- what the books ask for --------------------------------------------------------------------------------------
// Changes of the page tables and copies of pages, in one launch: both lists travel in the parameter space (no staging memory whose reuse
// a captured launch would have to survive), and copies read pages by their numbers, so their order does not matter. Copies are two
// bytes of traffic for each byte and nothing to compute: HBM-bound (30,011 tokens of ten layers copied and compacted: 2.46 GB in
// 375 us, the rate of a plain copy). A block copies 16 KB of one page, of K or V of one layer, four 16-byte loads of a thread in flight.
constexpr uint32_t BOOK_ENTRIES = 160;
// RECORDED: notes that the capture has run; MADE_UP: nothing if it has. (Captures are made up for one by one, so the latest number will do, and an
// older graph that runs again does not take it back.)
enum { BOOK_NOW = 0, BOOK_RECORDED = 1, BOOK_MADE_UP = 2 };
struct BookArgs {
    uint32_t n_copies, n_ops, mode, capture;
    PageCopy c[BOOK_ENTRIES];
    TableOp op[BOOK_ENTRIES];
};
static_assert(sizeof(BookArgs) <= 4000, "kernel parameters");

__global__ void __launch_bounds__(256)
books_kernel(const __grid_constant__ BookArgs list, char *__restrict__ mem, size_t layer_bytes, size_t page_bytes, uint32_t row_bytes, uint32_t *__restrict__ table,
             uint32_t *__restrict__ ran) {
    ptx::pdl_wait();
    ptx::pdl_launch_dependents();
    if (list.mode == BOOK_MADE_UP && __ldcg(ran) >= list.capture) return;
    if (list.mode == BOOK_RECORDED && blockIdx.x + blockIdx.y + blockIdx.z + threadIdx.x == 0u) atomicMax(ran, list.capture);
    if (blockIdx.y >= list.n_copies) {
        if (blockIdx.x != 0u || blockIdx.z != 0u) return;
        const TableOp &o = list.op[blockIdx.y - list.n_copies];
        const uint32_t n = o.n & ~TableOp::COPY;
        for (uint32_t i = threadIdx.x; i < n; i += 256u) table[o.dst + i] = (o.n & TableOp::COPY) ? table[o.val + i] : o.val + i;
        return;
    }
    const PageCopy &c = list.c[blockIdx.y];
    const uint32_t bytes = c.rows * row_bytes; // (a page is at most 256 rows of 64 heads of 256 f32: 16 MB)
    char *base = mem + (size_t)blockIdx.z * layer_bytes;
    const char *src = base + (size_t)c.src * page_bytes;
    char *dst = base + (size_t)c.dst * page_bytes;
    const uint32_t at = blockIdx.x * 16384u + threadIdx.x * 16u;
    uint4 v[4];
#pragma unroll
    for (uint32_t i = 0; i < 4u; i++)
        if (at + 4096u * i < bytes) v[i] = __ldcs(reinterpret_cast<const uint4 *>(src + at + 4096u * i));
#pragma unroll
    for (uint32_t i = 0; i < 4u; i++)
        if (at + 4096u * i < bytes) *reinterpret_cast<uint4 *>(dst + at + 4096u * i) = v[i];
}

static mkv_status launch_books(Pool *p, const std::vector<PageCopy> &cs, const std::vector<TableOp> &ops, uint32_t mode) {
    for (size_t i = 0, j = 0; i < cs.size() || j < ops.size();) {
        BookArgs t;
        t.mode = mode;
        t.capture = p->captures;
        t.n_copies = (uint32_t)std::min<size_t>(BOOK_ENTRIES, cs.size() - i);
        t.n_ops = (uint32_t)std::min<size_t>(BOOK_ENTRIES, ops.size() - j);
        std::copy_n(cs.begin() + (long)i, t.n_copies, t.c);
        std::copy_n(ops.begin() + (long)j, t.n_ops, t.op);
        i += t.n_copies;
        j += t.n_ops;
        uint32_t rows = 0;
        for (uint32_t k = 0; k < t.n_copies; k++) rows = std::max(rows, t.c[k].rows);
        const unsigned chunks = (unsigned)std::max<size_t>(1u, (rows * p->row_bytes + 16383u) / 16384u);
        PdlLaunch l(p->ctx, dim3(chunks, t.n_copies + t.n_ops, t.n_copies ? 2u * (unsigned)p->desc.n_layers : 1u), 256);
        MKV_CUDA(cudaLaunchKernelEx(&l.cfg, books_kernel, t, p->mem, p->layer_bytes, p->page_bytes, (uint32_t)p->row_bytes, p->table, p->table + p->table_entries()));
        p->ctx->launches++;
    }
    return MKV_OK;
}

// Launches what is in the lists and clears them; after an error they stay, for the next call. In a capture the launches are only recorded: the
// pages are the sequences' own from now on, but the graph may never run, and rows written through a table that still has others would land on
// other sequences' pages. So the lists are kept, and the first call outside a capture launches them as work that is left out on the device where the
// graph has run by then. Another capture may not begin before: its graph would either go without, or repeat what belongs to other sequences.
static mkv_status follow_books(Pool *p) {
    std::vector<PageCopy> &cs = p->book.copies;
    std::vector<TableOp> &ops = p->book.ops;
    const bool any = !cs.empty() || !ops.empty();
    if (!any && p->recorded.empty()) return MKV_OK;
    cudaStreamCaptureStatus status;
    unsigned long long id = 0;
    MKV_CUDA(cudaStreamGetCaptureInfo(p->ctx->stream, &status, &id));
    if (status == cudaStreamCaptureStatusNone) id = 0;
    if (!p->recorded.empty() && id == 0) {
        for (const BookWork &w : p->recorded) {
            const mkv_status st = launch_books(p, w.copies, w.ops, BOOK_MADE_UP);
            if (st != MKV_OK) return st;
        }
        p->recorded.clear();
    } else if (!p->recorded.empty() && id != p->capture) {
        set_error("an earlier capture changed pages: a call outside a capture has to come first");
        return MKV_ERR_STATE;
    }
    p->capture = id;
    if (!any) return MKV_OK;
    if (id != 0) {
        p->recorded.reserve(p->recorded.size() + 1u); // (nothing may fail behind the launch)
        if (p->recorded.empty()) p->captures++;
    }
    const mkv_status st = launch_books(p, cs, ops, id != 0 ? BOOK_RECORDED : BOOK_NOW);
    if (st != MKV_OK) return st;
    if (id != 0) p->recorded.push_back({std::move(cs), std::move(ops)});
    cs.clear();
    ops.clear();
    return MKV_OK;
}

// ---- new rows ----------------------------------------------------------------------------------------------------
// K and V of the new tokens into their pages, K rotated on the way, one rounding to the pool's type. Bound by HBM for prefill blocks
// and by the launch for steps. A block takes as many tokens as its threads have units for (two units of 8 values a thread; tokens of very
// many heads are spread over several blocks); the loads are in flight while the tokens' cosines and sines are computed.
// Measured: 7,682 rows of four f32 heads of 128 (63 MB) in 14.8 us, 4.3 TB/s; 128 rows of two f16 heads of 256 3.1 us.
constexpr uint32_t WRITE_ITEMS = 120;
struct WriteItems {
    uint32_t n;
    uint32_t table[WRITE_ITEMS], pos[WRITE_ITEMS]; // first entry of the sequence's table; position of the first row
    uint32_t row[WRITE_ITEMS + 1];                 // packed rows in front of the item
};
struct WriteArgs {
    const void *k, *v;
    int64_t k_stride, v_stride;
    char *kpages, *vpages;
    const uint32_t *pages;
    size_t page_bytes, row_bytes;
    uint32_t page_shift, kv_heads, head_dim, units, row0; // units of a K head; row0: packed row of the launch's first
    uint32_t tokens;                                      // of a block
};
static_assert(sizeof(WriteItems) + sizeof(WriteArgs) + sizeof(RopeTab) <= 4000, "kernel parameters");

constexpr uint32_t WRITE_PER = 2, WRITE_TOKENS = 16; // units of a thread, most tokens of a block

template <int MODE, class TI, class TO>
__global__ void __launch_bounds__(256)
pool_write_kernel(const __grid_constant__ WriteItems items, const __grid_constant__ WriteArgs g, const __grid_constant__ RopeTab tab) {
    extern __shared__ float2 cs[]; // [tokens][pairs]
    __shared__ uint32_t pos_s[WRITE_TOKENS];
    __shared__ size_t at_s[WRITE_TOKENS];
    ptx::pdl_wait();
    ptx::pdl_launch_dependents();
    const uint32_t row0 = blockIdx.x * g.tokens, n = min(g.tokens, items.row[items.n] - row0);
    const uint32_t nk = g.kv_heads * g.units, nv = g.kv_heads * g.head_dim / 8u, units = nk + nv;
    float a[WRITE_PER][8], b[WRITE_PER][8];
    uint32_t tok[WRITE_PER], unit[WRITE_PER];
#pragma unroll
    for (uint32_t w = 0; w < WRITE_PER; w++) {
        const uint32_t idx = (blockIdx.y * WRITE_PER + w) * 256u + threadIdx.x;
        tok[w] = idx / units;
        unit[w] = idx % units;
        if (tok[w] >= n) continue;
        if (unit[w] < nk) {
            const uint32_t head = unit[w] / g.units, u = unit[w] % g.units;
            rope_load<MODE>(static_cast<const TI *>(g.k) + (int64_t)(g.row0 + row0 + tok[w]) * g.k_stride + head * g.head_dim, u, tab.pairs, tab.interleaved, a[w], b[w]);
        } else {
            const TI *v = static_cast<const TI *>(g.v) + (int64_t)(g.row0 + row0 + tok[w]) * g.v_stride + 8u * (unit[w] - nk);
            if constexpr (MODE == ROPE_ANY) load8<false>(v, a[w]);
            else load8<true>(v, a[w]);
        }
    }
    if (threadIdx.x < n) { // where the token's rows go
        const uint32_t r = row0 + threadIdx.x;
        uint32_t i = 0, end = items.n; // the item with row[i] <= r < row[i + 1]
        while (i + 1u < end) {
            const uint32_t mid = (i + end) / 2u;
            if (items.row[mid] <= r) i = mid;
            else end = mid;
        }
        const uint32_t p = items.pos[i] + (r - items.row[i]);
        pos_s[threadIdx.x] = p;
        at_s[threadIdx.x] = (size_t)g.pages[items.table[i] + (p >> g.page_shift)] * g.page_bytes + (size_t)(p & ((1u << g.page_shift) - 1u)) * g.row_bytes;
    }
    __syncthreads();
    if (tab.pairs) {
        for (uint32_t j = threadIdx.x; j < n * tab.pairs; j += 256u) cs[j] = rope_cs(tab, j % tab.pairs, (int32_t)pos_s[j / tab.pairs]);
        __syncthreads();
    }
#pragma unroll
    for (uint32_t w = 0; w < WRITE_PER; w++) {
        if (tok[w] >= n) continue;
        if (unit[w] < nk) {
            const uint32_t head = unit[w] / g.units, u = unit[w] % g.units;
            rope_store<MODE>(reinterpret_cast<TO *>(g.kpages + at_s[tok[w]]) + head * g.head_dim, u, tab.pairs, tab.interleaved, cs + tok[w] * tab.pairs, a[w], b[w]);
        } else {
            store8<true>(reinterpret_cast<TO *>(g.vpages + at_s[tok[w]]) + 8u * (unit[w] - nk), a[w]);
        }
    }
}

template <class TI, class TO> static mkv_status launch_write(Ctx *ctx, int mode, uint32_t rows, const WriteItems &it, const WriteArgs &g, const RopeTab &tab) {
    const uint32_t units = g.kv_heads * (g.units + g.head_dim / 8u), per = 256u * WRITE_PER;
    PdlLaunch l(ctx, dim3((rows + g.tokens - 1u) / g.tokens, (g.tokens * units + per - 1u) / per), 256, (size_t)g.tokens * tab.pairs * sizeof(float2));
    switch (mode) {
    case ROPE_COPY: MKV_CUDA(cudaLaunchKernelEx(&l.cfg, pool_write_kernel<ROPE_COPY, TI, TO>, it, g, tab)); break;
    case ROPE_HALF8: MKV_CUDA(cudaLaunchKernelEx(&l.cfg, pool_write_kernel<ROPE_HALF8, TI, TO>, it, g, tab)); break;
    case ROPE_INTER8: MKV_CUDA(cudaLaunchKernelEx(&l.cfg, pool_write_kernel<ROPE_INTER8, TI, TO>, it, g, tab)); break;
    default: MKV_CUDA(cudaLaunchKernelEx(&l.cfg, pool_write_kernel<ROPE_ANY, TI, TO>, it, g, tab)); break;
    }
    ctx->launches++;
    return MKV_OK;
}

mkv_status launch_pool_write(Pool *p, int layer, const mkv_seq_rows *items, int n, const PoolWrite &w) {
    const size_t ie = w.fmt == MKV_F16 ? 2 : 4;
    const bool aligned = ((uintptr_t)w.k & 15u) == 0 && ((uintptr_t)w.v & 15u) == 0 && (w.k_stride * ie) % 16 == 0 && (w.v_stride * ie) % 16 == 0;
    const RopeTab tab = rope_tab(w.rope, false);
    const int mode = rope_mode(tab.pairs, tab.interleaved, (uint32_t)p->desc.head_dim, aligned);
    WriteArgs g;
    g.k = w.k;
    g.v = w.v;
    g.k_stride = w.k_stride;
    g.v_stride = w.v_stride;
    g.kpages = p->layer_ptr(layer, 0);
    g.vpages = p->layer_ptr(layer, 1);
    g.pages = p->table;
    g.page_bytes = p->page_bytes;
    g.row_bytes = p->row_bytes;
    g.page_shift = (uint32_t)__builtin_ctz(p->desc.page_tokens);
    g.kv_heads = (uint32_t)p->desc.kv_heads;
    g.head_dim = (uint32_t)p->desc.head_dim;
    g.units = rope_units(mode, tab.pairs, g.head_dim);
    g.row0 = 0;
    for (int i = 0; i < n;) {
        WriteItems it;
        it.n = 0;
        it.row[0] = 0;
        for (; i < n && it.n < WRITE_ITEMS; i++)
            if (items[i].ntok > 0u) {
                it.table[it.n] = items[i].seq * p->book.max_pages;
                it.pos[it.n] = items[i].pos;
                it.row[it.n + 1u] = it.row[it.n] + items[i].ntok;
                it.n++;
            }
        if (it.n == 0u) break;
        const uint32_t rows = it.row[it.n], token_units = g.kv_heads * (g.units + g.head_dim / 8u);
        // few rows: a block each, for the latency (128 rows: 3.1 us, in full blocks 3.7); many: blocks that are full (7,682 rows: 14.8 us, in
        // blocks of one row 18.3)
        g.tokens = rows < 2u * (uint32_t)p->ctx->sm_count ? 1u : std::max(1u, std::min(WRITE_TOKENS, 256u * WRITE_PER / token_units));
        const bool o16 = p->desc.fmt == MKV_F16;
        mkv_status st;
        if (w.fmt == MKV_F16)
            st = o16 ? launch_write<__half, __half>(p->ctx, mode, rows, it, g, tab) : launch_write<__half, float>(p->ctx, mode, rows, it, g, tab);
        else
            st = o16 ? launch_write<float, __half>(p->ctx, mode, rows, it, g, tab) : launch_write<float, float>(p->ctx, mode, rows, it, g, tab);
        if (st != MKV_OK) return st;
        g.row0 += rows;
    }
    return MKV_OK;
}

static Pool *pool_of(mkv_pool *h) { return reinterpret_cast<Pool *>(h); }
static const Pool *pool_of(const mkv_pool *h) { return reinterpret_cast<const Pool *>(h); }

static mkv_status no_memory() {
    set_error("out of host memory");
    return MKV_ERR_NOMEM;
}
// Runs a body that may throw for want of host memory; nothing is thrown past a C entry point.
template <class F> static mkv_status guarded(const F &body) {
    try {
        return body();
    } catch (const std::bad_alloc &) {
        return no_memory();
    } catch (...) {
        set_error("unexpected exception");
        return MKV_ERR_INVALID;
    }
}

static mkv_status need_pool(const void *p) {
    if (p) return MKV_OK;
    set_error("null argument");
    return MKV_ERR_INVALID;
}

// A change of the books and what follows it on the device; `undo` takes the change back when that could not be launched.
template <class F, class U> static mkv_status change(Pool *p, const F &body, const U &undo) {
    if (!p->ctx) {
        const mkv_status st = body();
        p->book.ops.clear();
        p->book.copies.clear();
        return st;
    }
    DeviceScope dev(p->ctx);
    if (dev.status != MKV_OK) return dev.status;
    mkv_status st = follow_books(p); // (what an earlier call could not launch: entries of one launch do not depend on each other)
    if (st == MKV_OK) st = body();
    if (st != MKV_OK) return st;
    try {
        st = follow_books(p);
    } catch (const std::bad_alloc &) {
        st = no_memory();
    }
    if (st != MKV_OK) undo();
    return st;
}
template <class F> static mkv_status change(Pool *p, const F &body) {
    return change(p, body, [] {}); // (the next call makes up for it)
}

static mkv_status check_items(const Pool *p, int layer, const mkv_seq_rows *items, int n, uint64_t *rows) {
    if (layer < 0 || layer >= p->desc.n_layers) {
        set_error("layer %d outside [0, %d)", layer, p->desc.n_layers);
        return MKV_ERR_INVALID;
    }
    if (n < 0 || (n > 0 && !items)) {
        set_error("%d items", n);
        return MKV_ERR_INVALID;
    }
    *rows = 0;
    for (int i = 0; i < n; i++) *rows += items[i].ntok;
    if (*rows > 0x3fffffffull) {
        set_error("%llu rows in one call, at most 2^30 - 1", (unsigned long long)*rows);
        return MKV_ERR_INVALID;
    }
    return MKV_OK;
}
static bool stride_ok(int64_t *s, int64_t dense) {
    if (*s == 0) *s = dense;
    return *s >= dense && *s <= (int64_t)1 << 30;
}
static mkv_status no_rows() {
    set_error("a pool without a context has no rows");
    return MKV_ERR_UNSUPPORTED;
}

} // namespace mkv

using namespace mkv;

extern "C" {

mkv_status mkv_pool_create(mkv_ctx *h, const mkv_pool_desc *d, mkv_pool **out) {
    Ctx *ctx = reinterpret_cast<Ctx *>(h);
    if (!d || !out || (ctx && ctx->closing)) {
        set_error("null argument");
        return MKV_ERR_INVALID;
    }
    *out = nullptr;
    if (d->fmt != MKV_F16 && d->fmt != MKV_F32) {
        set_error("unknown format %d", (int)d->fmt);
        return MKV_ERR_INVALID;
    }
    if (d->n_layers < 1 || d->n_layers > 256) {
        set_error("n_layers %d outside [1, 256]", d->n_layers);
        return MKV_ERR_INVALID;
    }
    if (d->page_tokens < 16 || d->page_tokens > 256 || (d->page_tokens & (d->page_tokens - 1u))) {
        set_error("pages of %u tokens: must be 16, 32, 64, 128 or 256", d->page_tokens);
        return MKV_ERR_INVALID;
    }
    if (d->n_pages < 1 || (uint64_t)d->n_pages * d->page_tokens >= 1ull << 31) {
        set_error("%u pages of %u tokens: at least one, and less than 2^31 rows", d->n_pages, d->page_tokens);
        return MKV_ERR_INVALID;
    }
    if (d->max_seqs < 1 || d->max_seqs > 65536 || d->max_tokens < 1 || d->max_tokens > 1u << 30) {
        set_error("%u sequences of up to %u tokens: must be 1 to 65536 and 1 to 2^30", d->max_seqs, d->max_tokens);
        return MKV_ERR_INVALID;
    }
    if (d->kv_heads < 1 || d->kv_heads > 64 || d->q_heads < d->kv_heads || d->q_heads % d->kv_heads != 0 || d->q_heads / d->kv_heads > 64) {
        set_error("%d query heads over %d key heads: a multiple of 1 to 64, of 1 to 64 heads", d->q_heads, d->kv_heads);
        return MKV_ERR_INVALID;
    }
    if (d->head_dim != 64 && d->head_dim != 128 && d->head_dim != 256) {
        set_error("heads of %d dims: must be 64, 128 or 256", d->head_dim);
        return MKV_ERR_INVALID;
    }
    return guarded([&]() -> mkv_status {
        if ((uint64_t)d->max_seqs * std::min<uint64_t>(((uint64_t)d->max_tokens + d->page_tokens - 1u) / d->page_tokens, d->n_pages) >= 1ull << 32) {
            set_error("page tables of %u sequences of up to %u tokens are too large", d->max_seqs, d->max_tokens);
            return MKV_ERR_INVALID;
        }
        Pool *p = new Pool(*d);
        p->elem = d->fmt == MKV_F16 ? 2 : 4;
        p->row_bytes = (size_t)d->kv_heads * (size_t)d->head_dim * p->elem;
        p->page_bytes = p->row_bytes * d->page_tokens;
        p->layer_bytes = p->page_bytes * d->n_pages;
        if (!ctx) {
            *out = reinterpret_cast<mkv_pool *>(p);
            return MKV_OK;
        }
        p->ctx = ctx;
        ctx->live_caches++;
        auto fail = [&](mkv_status s) {
            mkv_pool_destroy(reinterpret_cast<mkv_pool *>(p));
            return s;
        };
        DeviceScope dev(ctx);
        if (dev.status != MKV_OK) return fail(dev.status);
        const size_t bytes = 2u * (size_t)d->n_layers * p->layer_bytes, tb = (p->table_entries() + 1u) * sizeof(uint32_t);
        if (cudaMalloc(reinterpret_cast<void **>(&p->mem), bytes) != cudaSuccess || cudaMalloc(reinterpret_cast<void **>(&p->table), tb) != cudaSuccess) {
            cudaGetLastError();
            set_error("out of device memory for a pool of %zu bytes", bytes + tb);
            return fail(MKV_ERR_NOMEM);
        }
        if (cudaMemsetAsync(p->mem, 0, bytes, ctx->stream) != cudaSuccess || cudaMemsetAsync(p->table, 0, tb, ctx->stream) != cudaSuccess) {
            set_error("clearing the pool failed: %s", cudaGetErrorString(cudaGetLastError()));
            return fail(MKV_ERR_CUDA);
        }
        const mkv_status st = pool_attn_setup(p);
        if (st != MKV_OK) return fail(st);
        *out = reinterpret_cast<mkv_pool *>(p);
        return MKV_OK;
    });
}

void mkv_pool_destroy(mkv_pool *h) {
    Pool *p = pool_of(h);
    if (!p) return;
    Ctx *ctx = p->ctx;
    if (ctx) {
        DeviceScope dev(ctx);
        cudaStreamSynchronize(ctx->stream);
        if (p->mem) cudaFree(p->mem);
        if (p->table) cudaFree(p->table);
        if (p->scratch) cudaFree(p->scratch);
    }
    delete p;
    if (ctx) ctx_release(ctx);
}

mkv_status mkv_pool_buffers(mkv_pool *h, int layer, void **k, void **v) {
    Pool *p = pool_of(h);
    if (!p || layer < 0 || layer >= p->desc.n_layers) {
        set_error("bad pool or layer");
        return MKV_ERR_INVALID;
    }
    if (!p->ctx) return no_rows();
    if (k) *k = p->layer_ptr(layer, 0);
    if (v) *v = p->layer_ptr(layer, 1);
    return MKV_OK;
}

uint32_t mkv_pool_free_pages(const mkv_pool *h) { return h ? pool_of(h)->book.free_count() : 0u; }

mkv_status mkv_seq_create(mkv_pool *h, uint32_t *seq) {
    if (need_pool(h) != MKV_OK || need_pool(seq) != MKV_OK) return MKV_ERR_INVALID;
    return guarded([&] { return pool_of(h)->book.create(seq); });
}

mkv_status mkv_seq_fork(mkv_pool *h, uint32_t seq, uint32_t len, int copy, int n, uint32_t *children) {
    if (need_pool(h) != MKV_OK || need_pool(children) != MKV_OK) return MKV_ERR_INVALID;
    Pool *p = pool_of(h);
    return guarded([&] { return change(p, [&] { return p->book.fork(seq, len, copy != 0, n, children); }, [&] { p->book.free_all(children, n); }); });
}

mkv_status mkv_seq_free(mkv_pool *h, const uint32_t *seqs, int n) {
    if (need_pool(h) != MKV_OK) return MKV_ERR_INVALID;
    if (n < 0 || (n > 0 && !seqs)) {
        set_error("%d sequences", n);
        return MKV_ERR_INVALID;
    }
    return guarded([&] { return pool_of(h)->book.free_all(seqs, n); });
}

mkv_status mkv_seq_truncate(mkv_pool *h, uint32_t seq, uint32_t len) {
    if (need_pool(h) != MKV_OK) return MKV_ERR_INVALID;
    return guarded([&] { return pool_of(h)->book.truncate(seq, len); });
}

mkv_status mkv_seq_set_len(mkv_pool *h, uint32_t seq, uint32_t len) {
    if (need_pool(h) != MKV_OK) return MKV_ERR_INVALID;
    Pool *p = pool_of(h);
    return guarded([&] { return change(p, [&] { return p->book.set_len(seq, len); }); });
}

uint32_t mkv_seq_len(const mkv_pool *h, uint32_t seq) { return h && pool_of(h)->book.alive(seq) ? pool_of(h)->book.seqs[seq].len : 0u; }

mkv_status mkv_seq_pages(const mkv_pool *h, uint32_t seq, uint32_t *pages, uint32_t cap, uint32_t *n) {
    if (need_pool(h) != MKV_OK || need_pool(n) != MKV_OK) return MKV_ERR_INVALID;
    const mkv_status st = pool_of(h)->book.need(seq);
    if (st != MKV_OK) return st;
    const std::vector<uint32_t> &v = pool_of(h)->book.seqs[seq].pages;
    *n = (uint32_t)v.size();
    if (cap > 0u && !v.empty() && need_pool(pages) != MKV_OK) return MKV_ERR_INVALID;
    std::copy_n(v.begin(), std::min<size_t>(cap, v.size()), pages);
    return MKV_OK;
}

mkv_status mkv_pool_compact(mkv_pool *h, uint32_t *moved) {
    if (need_pool(h) != MKV_OK) return MKV_ERR_INVALID;
    Pool *p = pool_of(h);
    return guarded([&] { return change(p, [&] { return p->book.compact(moved); }); });
}

mkv_status mkv_pool_write(mkv_pool *h, int layer, const mkv_seq_rows *items, int n, const mkv_pool_rows *in) {
    if (need_pool(h) != MKV_OK || need_pool(in) != MKV_OK) return MKV_ERR_INVALID;
    Pool *p = pool_of(h);
    uint64_t rows;
    mkv_status st = check_items(p, layer, items, n, &rows);
    if (st != MKV_OK) return st;
    if (in->fmt != MKV_F16 && in->fmt != MKV_F32) {
        set_error("unknown format %d", (int)in->fmt);
        return MKV_ERR_INVALID;
    }
    PoolWrite w = {in->k_dev, in->v_dev, in->fmt, in->k_stride, in->v_stride, in->rope};
    const int64_t dense = (int64_t)p->desc.kv_heads * p->desc.head_dim;
    if (!stride_ok(&w.k_stride, dense) || !stride_ok(&w.v_stride, dense)) {
        set_error("token strides must be 0 or %lld to 2^30", (long long)dense);
        return MKV_ERR_INVALID;
    }
    if (w.rope && w.rope->desc.dims > p->desc.head_dim) {
        set_error("%d rotated dims in heads of %d", w.rope->desc.dims, p->desc.head_dim);
        return MKV_ERR_INVALID;
    }
    const uintptr_t low = w.fmt == MKV_F16 ? 1u : 3u;
    if (rows > 0 && (!w.k || !w.v || ((uintptr_t)w.k & low) || ((uintptr_t)w.v & low))) {
        set_error("k and v must be given, at multiples of their element's size");
        return MKV_ERR_INVALID;
    }
    return guarded([&] {
        if (!p->ctx) {
            const mkv_status checked = p->book.write(layer, items, n, true);
            return checked == MKV_OK ? no_rows() : checked;
        }
        auto undo = [&] { p->book.not_written(layer, items, n); };
        mkv_status st2 = change(p, [&] { return p->book.write(layer, items, n, false); }, undo);
        if (st2 != MKV_OK || rows == 0) return st2;
        DeviceScope dev(p->ctx);
        st2 = dev.status != MKV_OK ? dev.status : launch_pool_write(p, layer, items, n, w);
        if (st2 != MKV_OK) undo();
        return st2;
    });
}

mkv_status mkv_attn_pool(mkv_pool *h, int layer, const mkv_seq_rows *items, int n, const mkv_pool_attn *in) {
    if (need_pool(h) != MKV_OK || need_pool(in) != MKV_OK) return MKV_ERR_INVALID;
    Pool *p = pool_of(h);
    uint64_t rows;
    mkv_status st = check_items(p, layer, items, n, &rows);
    if (st != MKV_OK) return st;
    for (int i = 0; i < n; i++) {
        if ((st = p->book.need(items[i].seq)) != MKV_OK) return st;
        // tiles of the launch are counted in 31 bits: an item's blocks (of 128 rows and keys, f32 64) times its KV heads times its tiles
        const uint64_t side = p->desc.fmt == MKV_F16 ? 128u : 64u;
        if (((uint64_t)items[i].ntok * (uint64_t)p->desc.q_heads / (side / 2u) + (uint64_t)p->desc.kv_heads) *
                (((uint64_t)items[i].pos + items[i].ntok) / side + 2u) > 0x7fffffffull) {
            set_error("item %d: %u tokens at %u are too many for one call", i, items[i].ntok, items[i].pos);
            return MKV_ERR_INVALID;
        }
        const uint64_t end = (uint64_t)items[i].pos + items[i].ntok;
        const uint32_t there = p->book.seqs[items[i].seq].written[(size_t)layer];
        if (items[i].ntok > 0u && end > there) {
            set_error("item %d reads rows up to %llu of sequence %u, layer %d has %u", i, (unsigned long long)end, items[i].seq, layer, there);
            return MKV_ERR_STATE;
        }
    }
    PoolAttn a = {in->q_dev, in->out_dev, in->q_stride, in->out_stride, in->scale, in->window, in->sinks_dev};
    const int64_t dense = (int64_t)p->desc.q_heads * p->desc.head_dim;
    if (!stride_ok(&a.q_stride, dense) || !stride_ok(&a.out_stride, dense) || (a.q_stride * (int64_t)p->elem) % 16 != 0 ||
        (a.out_stride * (int64_t)p->elem) % 16 != 0) {
        set_error("token strides must be 0 or %lld to 2^30, and multiples of 16 bytes", (long long)dense);
        return MKV_ERR_INVALID;
    }
    if (!(a.scale >= 0.0f) || a.scale > 3.0e38f) {
        set_error("scale %g must be finite and not negative", a.scale);
        return MKV_ERR_INVALID;
    }
    if (a.scale == 0.0f) a.scale = 1.0f / sqrtf((float)p->desc.head_dim);
    if (rows > 0 && (!a.q || !a.out || ((uintptr_t)a.q & 15u) || ((uintptr_t)a.out & 15u) || ((uintptr_t)a.sinks & 3u))) {
        set_error("q and out must be given and 16-byte aligned, sinks 4-byte aligned");
        return MKV_ERR_INVALID;
    }
    const uint64_t q_row = (uint64_t)dense * p->elem;
    if (rows > 0 && RowSpan{(uintptr_t)a.q, rows, (uint64_t)a.q_stride * p->elem, q_row}.meets({(uintptr_t)a.out, rows, (uint64_t)a.out_stride * p->elem, q_row})) {
        set_error("q and out overlap");
        return MKV_ERR_INVALID;
    }
    if (!p->ctx) return no_rows();
    if (rows == 0) return MKV_OK;
    DeviceScope dev(p->ctx);
    if (dev.status != MKV_OK) return dev.status;
    return guarded([&]() -> mkv_status {
        mkv_status s = follow_books(p); // (what an earlier call could not launch)
        if (s == MKV_OK) s = prof_begin(p->ctx);
        if (s == MKV_OK) s = launch_pool_attn(p, layer, items, n, a);
        return s == MKV_OK ? prof_end(p->ctx) : s;
    });
}

} // extern "C"
