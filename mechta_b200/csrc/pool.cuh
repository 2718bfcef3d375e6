// A pool of pages on the device and the launchers of the kernels that work on it.
#pragma once
#include "internal.cuh"
#include "pages.hpp"

namespace mkv {

// What one change of the books asks of the device
struct BookWork {
    std::vector<PageCopy> copies;
    std::vector<TableOp> ops;
};

struct Pool {
    Ctx *ctx = nullptr; // null: the bookkeeping alone
    mkv_pool_desc desc = {};
    PageBook book;
    size_t elem = 2, row_bytes = 0, page_bytes = 0, layer_bytes = 0; // layer_bytes: the K (or V) pages of one layer
    char *mem = nullptr;                                            // [layer][K, V][page][row]
    uint32_t *table = nullptr;                                      // [max_seqs][max_pages]
    float *scratch = nullptr;                                       // of the attention: parts of split work, folded outputs (pool_plan.cuh)
    std::vector<CUtensorMap> maps;                                  // [layer][K, V]
    // What was recorded into the capture of that number and may never run; captures that have recorded anything are counted, and a word behind the
    // tables on the device has the latest that ran
    std::vector<BookWork> recorded;
    unsigned long long capture = 0;
    uint32_t captures = 0;
    size_t table_entries() const { return (size_t)desc.max_seqs * book.max_pages; }
    explicit Pool(const mkv_pool_desc &d) : desc(d), book(d.n_pages, d.page_tokens, d.max_seqs, d.max_tokens, d.n_layers) {}
    char *layer_ptr(int layer, int kv) const { return mem + (2u * (size_t)layer + (size_t)kv) * layer_bytes; }
};

// One call's checked arguments
struct PoolWrite {
    const void *k, *v;
    mkv_fmt fmt;
    int64_t k_stride, v_stride;
    const mkv_rope *rope;
};
struct PoolAttn {
    const void *q;
    void *out;
    int64_t q_stride, out_stride;
    float scale;
    uint32_t window;
    const float *sinks;
};
mkv_status launch_pool_write(Pool *p, int layer, const mkv_seq_rows *items, int n, const PoolWrite &w);
mkv_status launch_pool_attn(Pool *p, int layer, const mkv_seq_rows *items, int n, const PoolAttn &a);
mkv_status pool_attn_setup(Pool *p);    // scratch, kernel attributes

// The attributes of a launch that may overlap the end of the kernel in front of it.
struct PdlLaunch {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute at[1];
    PdlLaunch(Ctx *ctx, dim3 grid, unsigned threads, size_t smem = 0) {
        cfg.gridDim = grid;
        cfg.blockDim = dim3(threads);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = ctx->stream;
        at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[0].val.programmaticStreamSerializationAllowed = ctx->pdl ? 1 : 0;
        cfg.attrs = at;
        cfg.numAttrs = 1;
    }
};

} // namespace mkv
