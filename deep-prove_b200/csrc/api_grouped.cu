// C ABI: integer matrix products grouped by expert (include/dpb_forward.h).
#include <algorithm>
#include <atomic>

#include "../../include/dpb_forward.h"
#include "grouped_product.cuh"

namespace dpb {

static uint32_t digits_of(uint32_t bits) { return bits <= 8 ? 1 : 2; }

template <int XD, int WD, int T>
static cudaError_t launch_product(dpb_ctx* ctx, const GroupedArgs& a, uint32_t blocks) {
    const uint32_t smem = GroupedShape<XD, WD, T>::smem(a.n_experts);
    // once per device: the most that any number of experts takes
    static std::atomic<uint64_t> allowed{0};
    const uint64_t bit = ctx->device < 64 ? 1ull << ctx->device : 0;
    if (!(allowed.load(std::memory_order_relaxed) & bit) || !bit) {
        const cudaError_t e = cudaFuncSetAttribute(grouped_product_kernel<XD, WD, T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   (int)GroupedShape<XD, WD, T>::smem(1024));
        if (e != cudaSuccess) return e;
        allowed.fetch_or(bit, std::memory_order_relaxed);
    }
    return launch_early(ctx->stream, blocks, kGroupedThreads, smem, grouped_product_kernel<XD, WD, T>, a);
}
template <int XD, int WD>
static cudaError_t launch_rows(dpb_ctx* ctx, const GroupedArgs& a, uint32_t rows, uint32_t blocks) {
    switch (rows) {
        case 16: return launch_product<XD, WD, 16>(ctx, a, blocks);
        case 32: return launch_product<XD, WD, 32>(ctx, a, blocks);
        case 64: return launch_product<XD, WD, 64>(ctx, a, blocks);
        case 128: return launch_product<XD, WD, 128>(ctx, a, blocks);
        default: return launch_product<XD, WD, 160>(ctx, a, blocks);
    }
}

static int weights_impl(dpb_ctx* ctx, const int64_t* src, int on_device, dpb_expert_weights* w) {
    const uint64_t numel = (uint64_t)w->n_experts * w->inner * w->cols;
    const uint64_t bytes = (uint64_t)w->n_experts * w->col_tiles * w->k_blocks * w->digits * kTileBytes;
    void* p = nullptr;
    DPB_TRY(device_alloc(ctx, bytes, &p));
    w->planes = (int8_t*)p;
    FwdCheck check;
    DPB_TRY(fwd_check_begin(ctx, &check));
    const int64_t* dev = nullptr;
    void* owned = nullptr;
    DPB_TRY(fwd_tensor(ctx, src, on_device, numel, &dev, &owned));
    const uint32_t blocks = (uint32_t)std::min<uint64_t>((uint64_t)w->n_experts * w->k_blocks * w->col_tiles, (uint64_t)ctx->sm_count * 4);
    const int64_t half = 1ll << (w->bits - 1);
    if (w->digits == 1)
        cut_weights_kernel<1><<<blocks, kCutThreads, 0, ctx->stream>>>(dev, w->n_experts, w->inner, w->cols, w->col_tiles, w->k_blocks,
                                                                       half, w->planes, check);
    else
        cut_weights_kernel<2><<<blocks, kCutThreads, 0, ctx->stream>>>(dev, w->n_experts, w->inner, w->cols, w->col_tiles, w->k_blocks,
                                                                       half, w->planes, check);
    const cudaError_t e = cudaGetLastError();
    unsigned int found = 0;
    int rc = e == cudaSuccess ? fwd_check_wait(ctx, check, &found) : fail(DPB_ECUDA, "expert weights: %s", cudaGetErrorString(e));
    device_free(ctx, owned);
    if (rc == DPB_OK && found) rc = fail(DPB_EINVAL, "a weight does not fit %u bits", w->bits);
    return rc;
}

static int product_impl(dpb_ctx* ctx, int dtype, const dpb_row_groups* g, const int64_t* x, int x_on_device, uint32_t x_bits,
                        uint32_t per, const dpb_expert_weights* w, dpb_mle** out) {
    const uint64_t n = g->n;
    dpb_mle* m = nullptr;
    DPB_TRY(new_mle(ctx, dtype, n * w->cols, &m));
    if (n == 0) {
        *out = m;
        return DPB_OK;
    }
    FwdCheck check;
    const int64_t* dev = nullptr;
    void *owned = nullptr, *planes = nullptr;
    int rc = fwd_check_begin(ctx, &check);
    if (rc == DPB_OK) rc = fwd_tensor(ctx, x, x_on_device, n / per * w->inner, &dev, &owned);
    // Rows per tile.  An instruction takes as long for 16 rows as for 128 (about 70 clocks; 85 for 160), so a tile should
    // hold what an expert gets: fewer, fuller tiles read the weights less often.  Small tiles leave room for more stages
    // (few rows: bound by the weights' way from HBM) and, up to 64 rows of two digits, for a second accumulator.
    // The average stands for all experts: their counts stay on the device.
    // Measured, the whole call in us, 8 experts of 2048 x 4096, 14 x 12 bits, balanced routes / routes that prefer some
    // experts: 8 rows per expert 30/31 with 16, 32/32 with 32; 12 rows 31/39 with 16, 31/31 with 32, 33/33 with 64; 16 rows
    // 32/32 with 32, 34/34 with 64; 24 rows 32/42 with 32, 33/34 with 64; 48 rows 34/42 with 64, 39/40 with 128; 64 rows
    // 36/44 with 64, 41/42 with 128; 80 rows 53/53 with 64, 44/44 with 128.  Between 128 and 160 it goes by how the counts
    // fill whole tiles until they are large (experts of 4096 x 11008): 256 rows 324/420 with 128, 372/354 with 160; 320
    // rows 464/462 and 405/465; 512 rows 628/689 and 724/684; 1024 rows 1234/1291 and 1234/1211; 2048 rows 2389/2468 and
    // 2255/2298; with 8 x 8 bits 512 rows 294/311 and 331/310, 2048 rows 1076/1094 and 1022/1038.
    const uint64_t used = std::min<uint64_t>(w->n_experts, n), average = (n + used - 1) / used;
    const uint32_t T = average <= 8 ? 16 : average <= 16 ? 32 : average <= 64 ? 64 : average < 320 ? 128 : 160;
    const uint64_t max_tiles = n / T + used;  // every expert's last tile may be partly filled
    const uint32_t digits = digits_of(x_bits);
    if (rc == DPB_OK) rc = device_alloc(ctx, max_tiles * w->k_blocks * digits * 128 * T, &planes);
    cudaError_t e = cudaSuccess;
    unsigned int found = 0;
    if (rc == DPB_OK) {
        GroupedArgs a;
        memset(&a, 0, sizeof a);
        a.weights = w->planes;
        a.x = (const int8_t*)planes;
        a.offsets = g->offsets;
        a.rows = g->rows;
        a.n_experts = w->n_experts;
        a.col_tiles = w->col_tiles;
        a.k_blocks = w->k_blocks;
        a.cols = w->cols;
        a.out = (int64_t*)m->ptr;
        a.gave_up = fwd_gave_up_word(ctx);
        // When the tiles are fewer than four rounds of the GPU's blocks, the inner dimension is cut as well, into items
        // of at least four stages: a block's last item then costs little, and few tiles still keep every SM reading
        const uint64_t tiles = (n / T + (used + 1) / 2) * w->col_tiles, workers = ctx->sm_count;
        uint64_t splits = std::max<uint64_t>(1, std::min<uint64_t>(w->k_blocks / 4, workers * 4 / std::max<uint64_t>(tiles, 1)));
        splits = std::max<uint64_t>(splits, (w->k_blocks + kMaxSteps - 1) / kMaxSteps);
        a.blocks_per_split = (uint32_t)((w->k_blocks + splits - 1) / splits);
        a.splits = (w->k_blocks + a.blocks_per_split - 1) / a.blocks_per_split;
        // items, and an item's number plus a grid, are 32-bit numbers
        if (max_tiles * w->col_tiles * a.splits >= (1ull << 32) - 4096) {
            device_free(ctx, owned);
            device_free(ctx, planes);
            dpb_mle_free(m);
            return fail(DPB_EINVAL, "%llu work items", (unsigned long long)(max_tiles * w->col_tiles * a.splits));
        }
        const uint64_t cuts = n / per * ((w->k_blocks + 1) / 2), per_block = kCutThreads / 32, clear = a.splits > 1 ? n * w->cols : 0;
        const uint64_t for_cuts = (cuts + per_block - 1) / per_block, for_clear = (clear + 8 * kCutThreads - 1) / (8 * kCutThreads);
        const uint32_t blocks = (uint32_t)std::min<uint64_t>(std::max(for_cuts, for_clear), (uint64_t)ctx->sm_count * 8);
        const size_t smem = (w->n_experts + 1) * 4;
        const int64_t half = 1ll << (x_bits - 1);
        e = launch_early(ctx->stream, blocks, kCutThreads, smem, digits == 1 ? cut_rows_kernel<1> : cut_rows_kernel<2>, dev, g->keys, g->places,
                         g->offsets, n / per, per, w->n_experts, w->inner, w->k_blocks, T, half, (int8_t*)planes, a.out, clear, check);
        const uint32_t grid = (uint32_t)std::min<uint64_t>(max_tiles * w->col_tiles * a.splits, workers);
        if (e == cudaSuccess) {
            if (digits == 1) e = w->digits == 1 ? launch_rows<1, 1>(ctx, a, T, grid) : launch_rows<1, 2>(ctx, a, T, grid);
            else e = w->digits == 1 ? launch_rows<2, 1>(ctx, a, T, grid) : launch_rows<2, 2>(ctx, a, T, grid);
        }
        rc = e == cudaSuccess ? fwd_check_wait(ctx, check, &found) : fail(DPB_ECUDA, "grouped product: %s", cudaGetErrorString(e));
    }
    device_free(ctx, owned);
    device_free(ctx, planes);
    if (rc == DPB_OK) rc = fwd_groups_verdict(g);
    if (rc == DPB_OK && found) rc = fail(DPB_EINVAL, "a value of x does not fit %u bits", x_bits);
    if (rc != DPB_OK) {
        dpb_mle_free(m);
        return rc;
    }
    *out = m;
    return DPB_OK;
}

}  // namespace dpb

using namespace dpb;

extern "C" int dpb_expert_weights_new(dpb_ctx* ctx, const int64_t* weights, int on_device, uint32_t n_experts, uint64_t inner,
                                      uint64_t cols, uint32_t bits, dpb_expert_weights** out) {
    if (!ctx || !weights || !out) return fail(DPB_EINVAL, "null argument");
    if (n_experts < 1 || n_experts > 1024) return fail(DPB_EINVAL, "%u experts (1..1024)", n_experts);
    if (inner < 1 || cols < 1 || inner > (1ull << 24) || cols > (1ull << 24) || (uint64_t)n_experts * inner > (1ull << 40) / cols)
        return fail(DPB_EINVAL, "%u matrices of %llu x %llu entries", n_experts, (unsigned long long)inner, (unsigned long long)cols);
    if (bits < 2 || bits > 15) return fail(DPB_EINVAL, "weights of %u bits (2..15)", bits);
    const FwdDevice dev(ctx);
    DPB_TRY(fwd_ready(ctx, dev));
    dpb_expert_weights* w = new (std::nothrow) dpb_expert_weights();
    if (!w) return fail(DPB_ENOMEM, "host allocation failed");
    w->ctx = ctx;
    w->n_experts = n_experts;
    w->bits = bits;
    w->digits = digits_of(bits);
    w->inner = inner;
    w->cols = cols;
    w->col_tiles = (uint32_t)((cols + kTileCols - 1) / kTileCols);
    w->k_blocks = (uint32_t)((inner + kTileK - 1) / kTileK);
    const int rc = weights_impl(ctx, weights, on_device, w);
    if (rc != DPB_OK) {
        dpb_expert_weights_free(w);
        return rc;
    }
    *out = w;
    return DPB_OK;
}

extern "C" void dpb_expert_weights_free(dpb_expert_weights* w) {
    if (!w) return;
    if (w->planes) device_free(w->ctx, w->planes);
    delete w;
}

extern "C" int dpb_grouped_product(dpb_ctx* ctx, int family_dtype, const dpb_row_groups* g, const int64_t* x, int x_on_device,
                                   uint32_t x_bits, uint32_t rows_per_token, const dpb_expert_weights* w, dpb_mle** out) {
    if (!ctx || !g || !w || !out || (!x && g->n)) return fail(DPB_EINVAL, "null argument");
    if (g->ctx != ctx || w->ctx != ctx) return fail(DPB_EINVAL, "the rows or the weights belong to another context");
    if (!valid_dtype(family_dtype)) return fail(DPB_EINVAL, "unknown dtype %d", family_dtype);
    if (g->n_keys != w->n_experts)
        return fail(DPB_EINVAL, "rows routed to %llu experts, weights of %u", (unsigned long long)g->n_keys, w->n_experts);
    if (g->bad) return fwd_groups_verdict(g);
    if (x_bits < 2 || x_bits > 15) return fail(DPB_EINVAL, "rows of %u bits (2..15)", x_bits);
    if (rows_per_token < 1 || g->n % rows_per_token)
        return fail(DPB_EINVAL, "%llu routed rows are not a multiple of %u per token", (unsigned long long)g->n, rows_per_token);
    if (g->n > (1ull << 40) / w->cols) return fail(DPB_EINVAL, "a result of more than 2^40 entries");
    const FwdDevice dev(ctx);
    DPB_TRY(fwd_ready(ctx, dev));
    return product_impl(ctx, is_gl(family_dtype) ? DPB_GL_I64 : DPB_FR_I64, g, x, x_on_device, x_bits, rows_per_token, w, out);
}
