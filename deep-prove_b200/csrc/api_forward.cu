// C ABI: embedding lookup, rows sorted by key and their sums (include/dpb_forward.h).
#include <algorithm>
#include <atomic>

#include "../../include/dpb_forward.h"
#include "forward_kernels.cuh"

namespace dpb {

// mapped page: 8-byte words; 0 {findings, sequence number} of the last check, 1 set by a kernel that gave up waiting,
// kSlotWord + i the check that holds slot i
constexpr size_t kFwdPage = 1024;
constexpr int kSlotWord = 8, kSlots = 64;
static int fwd_init(dpb_ctx* ctx) {
    if (ctx->fwd_words) return DPB_OK;
    if (!ctx->fwd_host) {
        DPB_CUDA(cudaHostAlloc(&ctx->fwd_host, kFwdPage, cudaHostAllocMapped));
        memset(ctx->fwd_host, 0, kFwdPage);
        DPB_CUDA(cudaHostGetDevicePointer(&ctx->fwd_dev, ctx->fwd_host, 0));
    }
    unsigned int* w = nullptr;
    DPB_CUDA(cudaMalloc((void**)&w, 64));
    cudaError_t e = cudaMemsetAsync(w, 0, 64, ctx->stream);
    if (e != cudaSuccess) {
        cudaFree(w);
        return fail(DPB_ECUDA, "clearing counters: %s", cudaGetErrorString(e));
    }
    ctx->fwd_words = w;
    return DPB_OK;
}

unsigned int* fwd_gave_up_word(dpb_ctx* ctx) { return (unsigned int*)ctx->fwd_dev + 2; }

int fwd_slot_take(dpb_ctx* ctx) {
    for (int i = 0; i < kSlots; i++)
        if (!(ctx->fwd_slots >> i & 1)) {
            ctx->fwd_slots |= 1ull << i;
            return i;
        }
    return -1;
}

int fwd_check_begin(dpb_ctx* ctx, FwdCheck* out, int slot) {
    DPB_TRY(fwd_init(ctx));
    out->words = ctx->fwd_words;
    out->status = (unsigned long long*)ctx->fwd_dev + (slot < 0 ? 0 : kSlotWord + slot);
    out->seq = ++ctx->fwd_seq;
    return DPB_OK;
}

int fwd_check_wait(dpb_ctx* ctx, const FwdCheck& c, unsigned int* found) {
    const volatile uint64_t* status = (const volatile uint64_t*)ctx->fwd_host + (c.status - (unsigned long long*)ctx->fwd_dev);
    const auto t0 = std::chrono::steady_clock::now();
    uint64_t spins = 0;
    for (;;) {
        const uint64_t v = *status;
        if ((unsigned int)(v >> 32) == c.seq) {
            std::atomic_thread_fence(std::memory_order_acquire);
            *found = (unsigned int)v;
            return DPB_OK;
        }
        if ((++spins & 0xFFF) == 0) {
            const cudaError_t e = cudaStreamQuery(ctx->stream);  // our own launch may have failed
            if (e != cudaSuccess && e != cudaErrorNotReady) return fail(DPB_ECUDA, "value check: %s", cudaGetErrorString(e));
            const double dt = std::chrono::duration<double>(std::chrono::steady_clock::now() - t0).count();
            if (dt > 120.0) return fail(DPB_ETIMEOUT, "waited %.1f s for a value check", dt);
        }
    }
}

int fwd_groups_verdict(const dpb_row_groups* g) {
    if (g->slot >= 0) {
        unsigned int found = 0;
        DPB_TRY(fwd_check_wait(g->ctx, g->check, &found));
        g->ctx->fwd_slots &= ~(1ull << g->slot);
        g->slot = -1;
        g->bad = found != 0;
    }
    if (g->bad) return fail(DPB_EINVAL, "a key lies outside 0..%llu", (unsigned long long)(g->n_keys - 1));
    return DPB_OK;
}

int fwd_tensor(dpb_ctx* ctx, const int64_t* src, int on_device, uint64_t numel, const int64_t** dev, void** owned) {
    *owned = nullptr;
    *dev = src;
    if (on_device || numel == 0) return DPB_OK;
    DPB_TRY(device_alloc(ctx, numel * 8, owned));
    const cudaError_t e = cudaMemcpyAsync(*owned, src, numel * 8, cudaMemcpyHostToDevice, ctx->stream);
    if (e != cudaSuccess) {
        device_free(ctx, *owned);
        *owned = nullptr;
        return fail(DPB_ECUDA, "tensor upload: %s", cudaGetErrorString(e));
    }
    *dev = (const int64_t*)*owned;
    return DPB_OK;
}

template <class T, int V>
static void launch_lookup(dpb_ctx* ctx, const LookupArgs& a, bool check_all, bool index32, uint32_t blocks) {
    if (index32) {
        if (check_all) embedding_lookup_kernel<T, V, true, uint32_t><<<blocks, kLookupThreads, 0, ctx->stream>>>(a);
        else embedding_lookup_kernel<T, V, false, uint32_t><<<blocks, kLookupThreads, 0, ctx->stream>>>(a);
    } else {
        if (check_all) embedding_lookup_kernel<T, V, true, uint64_t><<<blocks, kLookupThreads, 0, ctx->stream>>>(a);
        else embedding_lookup_kernel<T, V, false, uint64_t><<<blocks, kLookupThreads, 0, ctx->stream>>>(a);
    }
}

static int lookup_impl(dpb_ctx* ctx, const dpb_mle* table, uint64_t vocab, uint64_t width, uint64_t stride, const int64_t* tokens,
                       int tokens_on_device, uint64_t n, int64_t multiplier, uint32_t shift, int padded, dpb_mle** out) {
    const bool i32 = dtype_size(table->dtype) == 4;
    LookupArgs a;
    memset(&a, 0, sizeof a);
    a.out_rows = padded ? pow2_ceil(std::max<uint64_t>(n, 1)) : n;
    a.out_width = padded ? pow2_ceil(width) : width;
    const uint64_t len = a.out_rows * a.out_width;
    dpb_mle* m = nullptr;
    DPB_TRY(new_mle(ctx, is_gl(table->dtype) ? DPB_GL_I64 : DPB_FR_I64, len, &m));
    if (n == 0) {
        const cudaError_t e = cudaMemsetAsync(m->ptr, 0, len * 8, ctx->stream);
        if (e != cudaSuccess) {
            dpb_mle_free(m);
            return fail(DPB_ECUDA, "embedding lookup: %s", cudaGetErrorString(e));
        }
        *out = m;
        return DPB_OK;
    }
    FwdCheck check;
    void* owned = nullptr;
    int rc = fwd_check_begin(ctx, &check);
    if (rc == DPB_OK) rc = fwd_tensor(ctx, tokens, tokens_on_device, n, &a.tokens, &owned);
    if (rc != DPB_OK) {
        dpb_mle_free(m);
        return rc;
    }
    a.table = table->ptr;
    a.vocab = vocab;
    a.width = width;
    a.stride = stride;
    a.n = n;
    a.multiplier = multiplier;
    a.rounding = shift ? 1ll << (shift - 1) : 0;
    a.shift = shift;
    a.out = (int64_t*)m->ptr;
    a.check = check;
    // A 32-bit entry times a 32-bit multiplier, with the rounding, always fits; other products are checked one by one
    const bool check_all = !i32 || multiplier > 0x7fffffffll || multiplier < -0x7fffffffll;
    const int V = i32 ? 4 : 2;
    const bool vec = a.out_width % V == 0 && stride % V == 0 && ((uintptr_t)table->ptr & 15) == 0 && vocab * stride <= table->len;
    const uint64_t steps = a.out_rows * ((a.out_width + (vec ? V : 1) - 1) / (vec ? V : 1));
    const uint32_t blocks = (uint32_t)std::min<uint64_t>((steps + kLookupThreads - 1) / kLookupThreads, (uint64_t)ctx->sm_count * 4);
    const bool index32 = steps + 2ull * kLookupFlight * blocks * kLookupThreads < (1ull << 31);
    // with l = ceil(log2 d) and m = floor(2^(31 + l) / d) + 1, w m / 2^(31 + l) lies less than 1 / d above w / d
    const uint64_t per_row = a.out_width / (vec ? V : 1), l = log2u(per_row);
    if (index32) {
        a.div_mul = (uint32_t)((1ull << (31 + l)) / per_row + 1);
        a.div_shift = (uint32_t)(31 + l);
    }
    a.check_blocks = check_all ? 0 : (uint32_t)std::min<uint64_t>(blocks, (n + 8 * kLookupThreads - 1) / (8 * kLookupThreads));
    if (i32) {
        if (vec) launch_lookup<int32_t, 4>(ctx, a, check_all, index32, blocks);
        else launch_lookup<int32_t, 1>(ctx, a, check_all, index32, blocks);
    } else {
        if (vec) launch_lookup<int64_t, 2>(ctx, a, check_all, index32, blocks);
        else launch_lookup<int64_t, 1>(ctx, a, check_all, index32, blocks);
    }
    const cudaError_t e = cudaGetLastError();
    unsigned int found = 0;
    rc = e == cudaSuccess ? fwd_check_wait(ctx, check, &found) : fail(DPB_ECUDA, "embedding lookup: %s", cudaGetErrorString(e));
    device_free(ctx, owned);
    if (rc == DPB_OK && (found & kFwdKeyRange))
        rc = fail(DPB_EINVAL, "a token lies outside the table's %llu rows", (unsigned long long)vocab);
    else if (rc == DPB_OK && found)
        rc = fail(DPB_EINVAL, "an entry times the multiplier does not fit 64 bits");
    if (rc != DPB_OK) {
        dpb_mle_free(m);
        return rc;
    }
    *out = m;
    return DPB_OK;
}

static int groups_impl(dpb_ctx* ctx, const int64_t* keys, int on_device, dpb_row_groups* g) {
    const uint32_t n = (uint32_t)g->n, n_keys = (uint32_t)g->n_keys;
    const bool few = n_keys <= kFewKeys && n > kSmallSort && n <= kFewSort, small = n <= kSmallSort || few, dense = n_keys <= kGroupOffsets;
    const uint32_t counters = n_keys + 1, tiles = (counters + kCountTile - 1) / kCountTile;
    // one block: [keys | rows | places | offsets or counters]
    auto up = [](uint64_t words) { return (words + 63) & ~63ull; };
    const uint64_t w_rows = up(n), w_places = 2 * up(n), w_off = 3 * up(n), w_end = w_off + (dense || !small ? up((uint64_t)counters + 1) : 0);
    DPB_TRY(device_alloc(ctx, (w_end ? w_end : 1) * 4, &g->block));
    g->keys = (uint32_t*)g->block;
    g->rows = g->keys + w_rows;
    g->places = g->keys + w_places;
    uint32_t* counts = g->keys + w_off;
    if (dense) g->offsets = counts;
    if (n == 0) {
        if (dense) DPB_CUDA(cudaMemsetAsync(counts, 0, (uint64_t)counters * 4, ctx->stream));
        return DPB_OK;
    }
    const int slot = on_device ? fwd_slot_take(ctx) : -1;  // a host buffer is only read during the call: waited for here
    g->slot = slot;
    DPB_TRY(fwd_check_begin(ctx, &g->check, slot));
    const FwdCheck check = g->check;
    const int64_t* dev = nullptr;
    void *owned = nullptr, *scratch = nullptr;
    DPB_TRY(fwd_tensor(ctx, keys, on_device, n, &dev, &owned));
    int rc = DPB_OK;
    cudaError_t e = cudaSuccess;
    if (few) {
        groups_few_kernel<<<1, kFewThreads, (n_keys + 1) * 128, ctx->stream>>>(dev, n, n_keys, g->keys, g->rows, g->places, g->offsets, check);
        e = cudaGetLastError();
    } else if (small) {
        const uint32_t probes = n + (dense ? n_keys + 1 : 0), per_block = kSmallSortThreads / 8;
        groups_small_kernel<<<(probes + per_block - 1) / per_block, kSmallSortThreads, ((n + 31) & ~31u) * 4, ctx->stream>>>(
            dev, n, n_keys, g->keys, g->rows, g->places, g->offsets, check);
        e = cudaGetLastError();
    } else {
        rc = device_alloc(ctx, tiles * 4, &scratch);
        if (rc == DPB_OK) {
            uint32_t *rank = g->places, *tile_sums = (uint32_t*)scratch;
            e = cudaMemsetAsync(counts, 0, (uint64_t)counters * 4, ctx->stream);
            if (e == cudaSuccess) {
                groups_count_kernel<<<grid_for(ctx, n), kThreads, 0, ctx->stream>>>(dev, n, n_keys, counts, rank, check);
                e = launch_early(ctx->stream, tiles, 1024, 0, groups_scan_kernel, counts, counters, tile_sums);
                if (e == cudaSuccess)
                    e = launch_early(ctx->stream, grid_for(ctx, n), kThreads, 0, groups_scatter_kernel, dev, n, n_keys, counts, tile_sums, tiles,
                                     rank, g->keys, g->rows);
                if (e == cudaSuccess) e = cudaGetLastError();
            }
        }
    }
    if (rc == DPB_OK && e != cudaSuccess) rc = fail(DPB_ECUDA, "sorting rows: %s", cudaGetErrorString(e));
    if (rc == DPB_OK && slot < 0) {
        unsigned int found = 0;
        rc = fwd_check_wait(ctx, check, &found);
        g->bad = found != 0;
        if (rc == DPB_OK) rc = fwd_groups_verdict(g);
    }
    device_free(ctx, owned);
    device_free(ctx, scratch);
    return rc;
}

template <class F>
static typename F::E field_constant(int64_t m) {
    const typename F::E v = F::from_u64(m < 0 ? (uint64_t)0 - (uint64_t)m : (uint64_t)m);
    return m < 0 ? F::neg(v) : v;
}

template <class F>
static int sum_impl(dpb_ctx* ctx, const dpb_row_groups* g, const dpb_mle* weights, const int64_t* rows, int rows_on_device,
                    uint64_t width, uint32_t per, int64_t multiplier, dpb_mle** out) {
    typedef typename F::E E;
    const uint64_t out_keys = pow2_ceil(g->n_keys), out_width = pow2_ceil(width);
    dpb_mle* m = nullptr;
    DPB_TRY(new_mle(ctx, F::kChalDtype, out_keys * out_width, &m));
    RowSumArgs a;
    memset(&a, 0, sizeof a);
    a.keys = g->keys;
    a.rows = g->rows;
    a.n = g->n;
    a.n_keys = g->n_keys;
    a.weights = weights ? weights->ptr : nullptr;
    a.width = width;
    a.per = per;
    a.out_width = out_width;
    a.out = m->ptr;
    const E scale = field_constant<F>(multiplier);
    const bool scaled = multiplier != 1;
    void *owned = nullptr, *parts = nullptr;
    cudaError_t e = cudaSuccess;
    int rc = DPB_OK;
    if (!rows) {
        a.slice = kKeySumSlice;
        const uint64_t slices = (a.n + a.slice - 1) / a.slice;
        const uint32_t key_blocks = (uint32_t)((out_keys + kKeySumThreads - 1) / kKeySumThreads);
        if (slices > 1) rc = device_alloc(ctx, slices * 2 * sizeof(E), &parts);
        if (rc == DPB_OK) {
            a.parts = parts;
            const uint32_t grid = key_blocks + (uint32_t)slices;
            e = launch_early(ctx->stream, grid, kKeySumThreads, 0, weights ? key_sums_kernel<F, true> : key_sums_kernel<F, false>, a, out_keys,
                             key_blocks, scale, scaled);
            if (slices > 1 && e == cudaSuccess)
                e = launch_early(ctx->stream, (uint32_t)((slices * 32 + kKeySumThreads - 1) / kKeySumThreads), kKeySumThreads, 0,
                                 key_sums_join_kernel<F>, a, slices, scale, scaled);
        }
    } else {
        rc = fwd_tensor(ctx, rows, rows_on_device, (a.n + per - 1) / per * width, &a.x, &owned);
        const uint64_t per_block = weights ? 2 * kRowSumThreads : kRowSumThreads, col_blocks = (width + per_block - 1) / per_block;
        // slices of at least 16 rows (8 without products), and as many as make one wave of resident blocks: the reduction at the end of a
        // block's sums, some hundred rows' worth of products, is then paid the fewest times
        const uint64_t resident = weights ? kProductBlocks<F> : 8;
        const uint64_t want = std::min<uint64_t>(65535, std::max<uint64_t>(1, (uint64_t)ctx->sm_count * resident / col_blocks));
        a.slice = std::min<uint64_t>(kRowSumMaxSlice, std::max<uint64_t>(weights ? 16 : 8, (a.n + want - 1) / want));
        const uint64_t slices = (a.n + a.slice - 1) / a.slice;
        if (rc == DPB_OK && slices > 1) rc = device_alloc(ctx, slices * 2 * width * sizeof(E), &parts);
        if (rc == DPB_OK) {
            a.parts = parts;
            // keys without rows, and the padding: by the kernel where the keys' places are kept, which saves a launch
            a.offsets = a.n ? g->offsets : nullptr;
            a.out_keys = out_keys;
            if (!a.offsets) e = cudaMemsetAsync(m->ptr, 0, m->len * sizeof(E), ctx->stream);
            if (e == cudaSuccess && a.n) {
                // more blocks where the zeros would be many for the slices' own: 16 entries per thread, up to four per SM
                const uint64_t for_zeros = std::min<uint64_t>(m->len / (16 * kRowSumThreads), (uint64_t)ctx->sm_count * 4);
                const uint64_t rows_of_blocks = a.offsets ? std::max(slices, (for_zeros + col_blocks - 1) / col_blocks) : slices;
                const dim3 grid((uint32_t)col_blocks, (uint32_t)std::min<uint64_t>(rows_of_blocks, 65535));
                auto kernel = !weights ? row_sums_kernel<F>
                              : (width & 1) == 0 && ((uintptr_t)a.x & 15) == 0 ? row_products_kernel<F, true> : row_products_kernel<F, false>;
                e = launch_early(ctx->stream, grid, kRowSumThreads, 0, kernel, a, scale, scaled);
                if (slices > 1 && e == cudaSuccess) {
                    const dim3 join((uint32_t)((width + kRowSumThreads - 1) / kRowSumThreads), (uint32_t)slices);
                    e = launch_early(ctx->stream, join, kRowSumThreads, 0, row_sums_join_kernel<F>, a, scale, scaled);
                }
            }
        }
    }
    // a host tensor is only read during the call: wait for its copy (device tensors need no wait)
    if (rc == DPB_OK && e == cudaSuccess && owned) e = cudaStreamSynchronize(ctx->stream);
    device_free(ctx, owned);
    device_free(ctx, parts);
    if (rc == DPB_OK && e != cudaSuccess) rc = fail(DPB_ECUDA, "row sums: %s", cudaGetErrorString(e));
    if (rc == DPB_OK) rc = fwd_groups_verdict(g);
    if (rc != DPB_OK) {
        dpb_mle_free(m);
        return rc;
    }
    *out = m;
    return DPB_OK;
}

}  // namespace dpb

using namespace dpb;

extern "C" int dpb_embedding_lookup(dpb_ctx* ctx, const dpb_mle* table, uint64_t vocab, uint64_t width, uint64_t row_stride,
                                    const int64_t* tokens, int tokens_on_device, uint64_t n, int64_t multiplier,
                                    uint32_t right_shift, int padded, dpb_mle** out) {
    if (!ctx || !table || !out || (!tokens && n)) return fail(DPB_EINVAL, "null argument");
    if (table->ctx != ctx) return fail(DPB_EINVAL, "the table belongs to another context");
    if (!is_int_dtype(table->dtype)) return fail(DPB_EINVAL, "the embedding table is an integer table (DPB_*_I32 or DPB_*_I64)");
    if (vocab == 0 || width == 0) return fail(DPB_EINVAL, "an embedding table has at least one row and one column");
    if (row_stride < width) return fail(DPB_EINVAL, "rows of %llu entries %llu apart", (unsigned long long)width, (unsigned long long)row_stride);
    if (width > table->len || (table->len - width) / row_stride < vocab - 1)
        return fail(DPB_EINVAL, "%llu rows of %llu entries, %llu apart, exceed the table's %llu entries", (unsigned long long)vocab,
                    (unsigned long long)width, (unsigned long long)row_stride, (unsigned long long)table->len);
    if (right_shift > 62) return fail(DPB_EINVAL, "right shift %u exceeds 62", right_shift);
    if (n > (1ull << 40) / pow2_ceil(width)) return fail(DPB_EINVAL, "a result of more than 2^40 entries");
    const FwdDevice dev(ctx);
    DPB_TRY(fwd_ready(ctx, dev));
    return lookup_impl(ctx, table, vocab, width, row_stride, tokens, tokens_on_device, n, multiplier, right_shift, padded, out);
}

extern "C" int dpb_row_groups_new(dpb_ctx* ctx, const int64_t* keys, int keys_on_device, uint64_t n, uint64_t n_keys,
                                  dpb_row_groups** out) {
    if (!ctx || !out || (!keys && n)) return fail(DPB_EINVAL, "null argument");
    if (n_keys < 1 || n_keys > (1ull << 22)) return fail(DPB_EINVAL, "%llu keys (1..2^22)", (unsigned long long)n_keys);
    if (n >= (1ull << 31)) return fail(DPB_EINVAL, "%llu rows (below 2^31)", (unsigned long long)n);
    const FwdDevice dev(ctx);
    DPB_TRY(fwd_ready(ctx, dev));
    dpb_row_groups* g = new (std::nothrow) dpb_row_groups();
    if (!g) return fail(DPB_ENOMEM, "host allocation failed");
    g->ctx = ctx;
    g->n = n;
    g->n_keys = n_keys;
    const int rc = groups_impl(ctx, keys, keys_on_device, g);
    if (rc != DPB_OK) {
        dpb_row_groups_free(g);
        return rc;
    }
    *out = g;
    return DPB_OK;
}

extern "C" uint64_t dpb_row_groups_len(const dpb_row_groups* g) { return g ? g->n : 0; }

extern "C" void dpb_row_groups_free(dpb_row_groups* g) {
    if (!g) return;
    // a check still under way publishes into its slot before any later one does, and under its own sequence number
    if (g->slot >= 0) g->ctx->fwd_slots &= ~(1ull << g->slot);
    if (g->block) device_free(g->ctx, g->block);
    delete g;
}

extern "C" int dpb_row_groups_sum(dpb_ctx* ctx, const dpb_row_groups* g, int family_dtype, const dpb_mle* weights, const int64_t* rows,
                                  int rows_on_device, uint64_t width, uint32_t rows_per_token, int64_t multiplier, dpb_mle** out) {
    if (!ctx || !g || !out) return fail(DPB_EINVAL, "null argument");
    if (g->ctx != ctx) return fail(DPB_EINVAL, "the rows belong to another context");
    if (!valid_dtype(family_dtype)) return fail(DPB_EINVAL, "unknown dtype %d", family_dtype);
    if (width == 0 || width > (1ull << 32)) return fail(DPB_EINVAL, "rows of %llu entries (1..2^32)", (unsigned long long)width);
    if (!rows && width != 1) return fail(DPB_EINVAL, "sums without rows have one column, got %llu", (unsigned long long)width);
    if (rows_per_token < 1) return fail(DPB_EINVAL, "rows per token must be at least 1");
    if (weights) {
        if (weights->ctx != ctx) return fail(DPB_EINVAL, "the weights belong to another context");
        if (weights->dtype != chal_dtype(family_dtype))
            return fail(DPB_EINVAL, "weights are challenge elements of the family (dtype %d, got %d)", chal_dtype(family_dtype), weights->dtype);
        if (weights->len < g->n)
            return fail(DPB_EINVAL, "%llu weights for %llu rows", (unsigned long long)weights->len, (unsigned long long)g->n);
    }
    if (g->bad) return fwd_groups_verdict(g);
    if (pow2_ceil(g->n_keys) * pow2_ceil(width) > (1ull << 36)) return fail(DPB_EINVAL, "a result of more than 2^36 entries");
    if (rows && g->n / rows_per_token > (1ull << 40) / width) return fail(DPB_EINVAL, "rows of more than 2^40 entries");
    const FwdDevice dev(ctx);
    DPB_TRY(fwd_ready(ctx, dev));
    return is_gl(family_dtype) ? sum_impl<GlFam>(ctx, g, weights, rows, rows_on_device, width, rows_per_token, multiplier, out)
                               : sum_impl<FrFam>(ctx, g, weights, rows, rows_on_device, width, rows_per_token, multiplier, out);
}

// Tests: the word as a kernel that gave up waiting leaves it.  Not part of the interface.
extern "C" int dpb_forward_give_up(dpb_ctx* ctx) {
    const FwdDevice dev(ctx);
    DPB_TRY(fwd_ready(ctx, dev));
    DPB_TRY(fwd_init(ctx));
    *fwd_gave_up_host(ctx) = 1;
    return DPB_OK;
}
