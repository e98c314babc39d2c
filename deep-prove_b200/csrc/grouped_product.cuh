// Integer matrix products grouped by expert, on the tensor cores' 8-bit integer form.
//
// y = x W exactly, |x| < 2^14, |W| < 2^14: both sides are cut into signed 8-bit digits, x = x0 + 256 x1 (one digit when
// 8 bits suffice), and the products of digits are added up in 32-bit integers by tcgen05.mma kind::i8, one accumulator
// per power of 256:  acc0 = W0 x0,  acc1 = W0 x1 + W1 x0,  acc2 = W1 x1;  y = acc0 + 2^8 acc1 + 2^16 acc2 in 64 bits.
// A digit product is at most 2^14 in magnitude and acc1 takes two per step, so up to 2^15 steps stay below 2^31
// (kMaxSteps); a longer inner dimension is cut, like a short list of tiles, over several work items that add their
// 64-bit results to the output (exact, so their order does not matter).
//
// The weights' 128 columns are the instruction's M (rows of the accumulator = TMEM lanes) and a tile's routed rows its
// N: a warp's lanes then hold neighbouring columns of one output row, which is stored as whole 256-byte runs without a
// transposition, and a tile of few rows (a single token) wastes nothing.
//
// What bounds it.  Many rows: the instruction.  16384 routed rows of 4096 by 8 matrices of 4096 x 11008 take 1.95 ms:
// 5.9e12 digit operations at 3.0e15/s, where twice the measured bf16 rate is 3.3e15/s, with the power cap at work.  (Two
// blocks sharing a tile by cta_group::2 bring less through L2 but took 2.02 ms.)  One token through two experts: the
// weights' 180 MB from HBM, 36 us of this kernel where the copy rate gives 28.
#pragma once
#include "forward.cuh"

struct dpb_expert_weights {
    dpb_ctx* ctx = nullptr;
    uint32_t n_experts = 0, bits = 0, digits = 0;
    uint64_t inner = 0, cols = 0;
    uint32_t col_tiles = 0, k_blocks = 0;
    int8_t* planes = nullptr;  // [expert][column tile][128 of the inner dimension][digit][128 columns x 128 bytes]
};

namespace dpb {

constexpr uint32_t kTileCols = 128, kTileK = 128;  // weight columns per tile; inner entries per stage (bytes of a digit)
constexpr uint32_t kTileBytes = kTileCols * kTileK;
constexpr uint32_t kMaxSteps = 256;  // stages per work item: 2^15 inner entries

// A tile's digits lie as the instruction reads them with the 128-byte swizzle: row r's 128 bytes at r * 128, the
// 16-byte pieces of a row exchanged by xor with r mod 8.  One copy then brings a whole tile, with no tensor map.
__device__ __forceinline__ uint32_t tile_piece(uint32_t row, uint32_t piece) { return row * 128 + ((piece ^ (row & 7)) << 4); }

constexpr uint32_t kCutThreads = 256;
// Weights [expert][inner][cols] -> planes, a tile of 128 columns by 128 inner entries at a time: neighbouring threads
// read neighbouring columns, and the digits go through shared memory so that a tile is written as it lies.  Made once
// per model.
template <int DIGITS>
__global__ void __launch_bounds__(kCutThreads)
    cut_weights_kernel(const int64_t* __restrict__ w, uint32_t n_experts, uint64_t inner, uint64_t cols, uint32_t col_tiles,
                       uint32_t k_blocks, int64_t half, int8_t* __restrict__ planes, FwdCheck check) {
    __shared__ uint4 tile[DIGITS][kTileBytes / 16];
    unsigned int found = 0;
    const uint32_t col = threadIdx.x & 127, side = threadIdx.x >> 7;
    const uint64_t total = (uint64_t)n_experts * col_tiles * k_blocks;
    for (uint64_t t = blockIdx.x; t < total; t += gridDim.x) {
        const uint64_t k0 = t % k_blocks * kTileK, ec = t / k_blocks, c = ec % col_tiles * kTileCols + col, e = ec / col_tiles;
        const int64_t* src = w + (e * inner + k0) * cols + c;
#pragma unroll
        for (uint32_t q = 0; q < 4; q++) {
            const uint32_t piece = 4 * side + q;
            int64_t v[16];
#pragma unroll
            for (uint32_t i = 0; i < 16; i++) {
                const uint32_t k = 16 * piece + i;
                v[i] = c < cols && k0 + k < inner ? __ldcs((const long long*)src + (uint64_t)k * cols) : 0;
            }
            uint32_t d[DIGITS][4];
#pragma unroll
            for (uint32_t i = 0; i < 4; i++) {
                uint32_t d0 = 0, d1 = 0;
#pragma unroll
                for (uint32_t j = 0; j < 4; j++) {
                    const int64_t x = v[4 * i + j];
                    if (x < -half || x >= half) found = kFwdValueRange;
                    const int lo = (int)(int8_t)x;
                    d0 |= (uint32_t)(uint8_t)lo << (8 * j);
                    d1 |= (uint32_t)(uint8_t)(((int)x - lo) >> 8) << (8 * j);
                }
                d[0][i] = d0;
                if (DIGITS == 2) d[DIGITS - 1][i] = d1;
            }
#pragma unroll
            for (int i = 0; i < DIGITS; i++) tile[i][tile_piece(col, piece) / 16] = make_uint4(d[i][0], d[i][1], d[i][2], d[i][3]);
        }
        __syncthreads();
        uint4* out = (uint4*)(planes + t * DIGITS * kTileBytes);
        for (uint32_t i = threadIdx.x; i < DIGITS * kTileBytes / 16; i += kCutThreads) __stcs(out + i, (&tile[0][0])[i]);
        __syncthreads();
    }
    fwd_check_done(check, found, gridDim.x);
}

// first tile of every expert: tiles[e] = sum of ceil(rows / T) over the experts before e
__device__ __forceinline__ void expert_tiles(const uint32_t* offsets, uint32_t n_experts, uint32_t T,
                                             uint32_t* tiles /* shared, n_experts + 1 */) {
    if (threadIdx.x < 32) {
        uint32_t carry = 0;
        for (uint32_t e0 = 0; e0 < n_experts; e0 += 32) {
            const uint32_t e = e0 + threadIdx.x;
            const uint32_t n = e < n_experts ? (__ldcg(offsets + e + 1) - __ldcg(offsets + e) + T - 1) / T : 0;
            uint32_t incl = n;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const uint32_t u = __shfl_up_sync(0xffffffffu, incl, off);
                if (threadIdx.x >= (uint32_t)off) incl += u;
            }
            if (e < n_experts) tiles[e] = carry + incl - n;
            carry += __shfl_sync(0xffffffffu, incl, 31);
        }
        if (threadIdx.x == 0) tiles[n_experts] = carry;
    }
}

// Routed rows in sorted order -> planes [row tile][128 of the inner dimension][digit][T rows x 128 bytes].  A warp cuts
// 256 entries of a row: it reads them as whole lines, whatever their alignment, and turns the digits round in shared
// memory so that a lane writes 16 bytes.  Rows of a tile past the expert's last are left as they are: their products are
// not stored.
constexpr uint32_t kCutEntries = 256;
template <int DIGITS>
__global__ void __launch_bounds__(kCutThreads)
    cut_rows_kernel(const int64_t* x, const uint32_t* keys, const uint32_t* places, const uint32_t* offsets, uint64_t tokens, uint32_t per, uint32_t n_experts, uint64_t inner,
                    uint32_t k_blocks, uint32_t T, int64_t half, int8_t* planes, int64_t* clear, uint64_t n_clear, FwdCheck check) {
    extern __shared__ uint32_t tiles[];
    __shared__ __align__(16) uint8_t cut[kCutThreads / 32][DIGITS][kCutEntries];
    unsigned int found = 0;
    wait_for_previous();
    let_next_start();  // the product's kernel, not before the rows' order is there: it sets itself up and fetches weights
    expert_tiles(offsets, n_experts, T, tiles);
    // the output, when several work items will add to its entries (two per 16 bytes; it starts on a 256-byte boundary)
    for (uint64_t i = (uint64_t)blockIdx.x * kCutThreads + threadIdx.x; i < n_clear / 2; i += (uint64_t)gridDim.x * kCutThreads)
        ((longlong2*)clear)[i] = make_longlong2(0, 0);
    if ((n_clear & 1) && blockIdx.x == 0 && threadIdx.x == 0) clear[n_clear - 1] = 0;
    __syncthreads();
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t per_row = (k_blocks + 1) / 2;  // 256 entries = two stages
    const uint64_t total = tokens * per_row, step = (uint64_t)gridDim.x * (kCutThreads / 32);
    for (uint64_t t = (uint64_t)blockIdx.x * (kCutThreads / 32) + warp; t < total; t += step) {
        const uint64_t token = t / per_row;
        const uint32_t k0 = (uint32_t)(t - token * per_row) * kCutEntries;
        const int64_t* src = x + token * inner;
        int64_t v[kCutEntries / 32];
#pragma unroll
        for (uint32_t i = 0; i < kCutEntries / 32; i++) {
            const uint64_t k = k0 + 32 * i + lane;
            v[i] = k < inner ? src[k] : 0;
        }
#pragma unroll
        for (uint32_t i = 0; i < kCutEntries / 32; i++) {
            if (v[i] < -half || v[i] >= half) found = kFwdValueRange;
            const int lo = (int)(int8_t)v[i];
            cut[warp][0][32 * i + lane] = (uint8_t)lo;
            if (DIGITS == 2) cut[warp][DIGITS - 1][32 * i + lane] = (uint8_t)(((int)v[i] - lo) >> 8);
        }
        __syncwarp();
        const uint32_t piece = lane & 15, digit = lane >> 4, block = k0 / kTileK + piece / 8;
        if (digit < DIGITS && block < k_blocks) {
            const uint4 bytes = *(const uint4*)&cut[warp][digit][16 * piece];
            for (uint32_t j = 0; j < per; j++) {
                const uint32_t p = places[token * per + j], e = keys[p];
                if (e >= n_experts) continue;  // a key out of range: the call will be refused
                const uint32_t at = p - offsets[e], q = at / T;
                const uint64_t tile = (uint64_t)(tiles[e] + q) * k_blocks + block;
                *(uint4*)(planes + (tile * DIGITS + digit) * (T * 128) + tile_piece(at - q * T, piece & 7)) = bytes;
            }
        }
        __syncwarp();
    }
    fwd_check_done(check, found, gridDim.x);
}

// ------------------------------------------------------------------------------------------------ PTX
__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
                 : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
// Waits for the phase; gives up, and tells the block's other roles, after kWaitNs.
constexpr uint64_t kWaitNs = 5ull * 1000 * 1000 * 1000;
__device__ __forceinline__ uint64_t now_ns() {
    uint64_t t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}
template <class Try>
__device__ __forceinline__ bool wait_limited(Try once, volatile int* gave_up) {
    if (once()) return true;
    const uint64_t t0 = now_ns();
    for (uint32_t i = 1;; i++) {
        if (once()) return true;
        if (*gave_up) return false;
        if ((i & 63) == 0 && now_ns() - t0 > kWaitNs) break;
    }
    *gave_up = 1;
    return false;
}
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, volatile int* gave_up) {
    return wait_limited([&]() { return bar_try(bar, parity); }, gave_up);
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src),
                 "r"(bytes), "r"(bar) : "memory");
}
// shared-memory operand, K-major, 128-byte swizzle: 8-row groups 1024 bytes apart
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr) {
    return (uint64_t)((addr & 0x3FFFF) >> 4) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) |
           ((uint64_t)2 << 61);
}
__device__ __forceinline__ void mma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
    asm volatile("{ .reg .pred p; setp.ne.u32 p, %4, 0; tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p; }" ::"r"(d), "l"(a),
                 "l"(b), "r"(idesc), "r"((uint32_t)accumulate) : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// 8 columns of the warp's 32 lanes
__device__ __forceinline__ void tmem_load8(uint32_t addr, uint32_t (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(addr));
}

// ------------------------------------------------------------------------------------------------ the product
struct GroupedArgs {
    const int8_t* weights;
    const int8_t* x;
    const uint32_t* offsets;
    const uint32_t* rows;
    uint32_t n_experts, col_tiles, k_blocks;
    uint32_t splits, blocks_per_split;  // work items along the inner dimension, and their stages
    uint64_t cols;
    int64_t* out;
    unsigned int* gave_up;
};

// XD, WD: digits of x and of the weights; T: rows per tile.
template <int XD, int WD, int T>
struct GroupedShape {
    static constexpr int kAcc = XD + WD - 1;
    static constexpr uint32_t kStageBytes = WD * kTileBytes + XD * T * 128;
    static constexpr uint32_t kStages = 216 * 1024 / kStageBytes < 8 ? 216 * 1024 / kStageBytes : 8;
    static constexpr int kBuffers = 2 * kAcc * T <= 512 ? 2 : 1;  // accumulators: the next tile's while one is stored
    static constexpr uint32_t kCols = kBuffers * kAcc * T;
    static constexpr uint32_t kTmem = kCols <= 32 ? 32 : kCols <= 64 ? 64 : kCols <= 128 ? 128 : kCols <= 256 ? 256 : 512;
    static constexpr uint32_t smem(uint32_t n_experts) { return kStages * kStageBytes + 1024 + (n_experts + 1) * 4; }
};

// The sixteen warps that move a finished tile: warp w reads the accumulators' lanes 32 (w mod 4) .. + 31, that is 32
// columns, and of the rows the eights w / 4, w / 4 + 4, ...  There is room for one large tile's accumulators only, so
// they are turned into results in registers first and given back to the next tile's products, and stored after that
// (512 rows routed to 8 experts: 61 us when they were given back between the stores); the rows' places in the output are
// read before the tile is finished.
constexpr uint32_t kStoreWarps = 16, kGroupedThreads = 32 * (kStoreWarps + 2);
template <int T>
struct TileRows {
    uint32_t row[(T + 31) / 32];  // lane l: rows l, l + 32, ... of the tile
    __device__ __forceinline__ void load(const uint32_t* rows, uint32_t lo, int valid) {
#pragma unroll
        for (int i = 0; i < (T + 31) / 32; i++) {
            const int j = 32 * i + (threadIdx.x & 31);
            row[i] = j < valid ? rows[lo + j] : 0;
        }
    }
};
// accumulators -> 64-bit results; `release` is called when the warp has read its accumulators
template <int ACC, int T, class Release>
__device__ __forceinline__ void store_tile(const GroupedArgs& a, uint32_t acc, const TileRows<T>& rows, int valid, uint64_t c,
                                           uint32_t quarter, Release release) {
    constexpr int kEights = (T + 31) / 32;
    int64_t y[kEights][8];
#pragma unroll
    for (int i = 0; i < kEights; i++) {
        if (32 * i + 8 * (int)quarter >= valid) break;
        uint32_t r[ACC][8];
#pragma unroll
        for (int d = 0; d < ACC; d++) tmem_load8(acc + d * T + 32 * i + 8 * quarter, r[d]);
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
        for (int j = 0; j < 8; j++) {
            y[i][j] = (int32_t)r[0][j];
#pragma unroll
            for (int d = 1; d < ACC; d++) y[i][j] += (int64_t)(int32_t)r[d][j] << (8 * d);
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncwarp();
    release();
#pragma unroll
    for (int i = 0; i < kEights; i++) {
        const int j0 = 32 * i + 8 * (int)quarter;
        if (j0 >= valid) break;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const uint32_t row = __shfl_sync(0xffffffffu, rows.row[i], 8 * quarter + j);
            if (c < a.cols && j0 + j < valid) {
                int64_t* o = a.out + (uint64_t)row * a.cols + c;
                if (a.splits > 1) atomicAdd((unsigned long long*)o, (unsigned long long)y[i][j]);
                else __stcs((long long*)o, (long long)y[i][j]);
            }
        }
    }
}

// After a wait that ran out: the host learns of it, and copies and products in flight must not outlive the block, so it
// stays for a second.  Called by the whole block.
__device__ __forceinline__ void gave_up_wait(unsigned int* word) {
    if (threadIdx.x == 0) {
        *(volatile unsigned int*)word = 1;
        for (uint32_t t = 0; t < (1u << 20); t++) __nanosleep(1000);
    }
    __syncthreads();
}

// Eighteen warps: 0-15 move finished accumulators to the output, 16 brings the operands, 17 issues the products.  One block per
// SM walks the work items blockIdx.x, + gridDim.x, ...; items of one expert are ordered with the row tiles fastest, so
// that the blocks at work at one time share the weights' and rows' tiles in L2.
template <int XD, int WD, int T>
__global__ void __launch_bounds__(kGroupedThreads, 1) grouped_product_kernel(GroupedArgs a) {
    typedef GroupedShape<XD, WD, T> S;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t bars[2 * S::kStages + 4];
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int gave_up;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t ring = (smem_addr(smem_raw) + 1023) & ~1023u;
    uint32_t* tiles = (uint32_t*)(smem_raw + (ring - smem_addr(smem_raw)) + S::kStages * S::kStageBytes);
    const uint32_t bar0 = smem_addr(bars);
    auto full = [&](uint32_t s) { return bar0 + 8 * s; };
    auto empty = [&](uint32_t s) { return bar0 + 8 * (S::kStages + s); };
    auto acc_full = [&](uint32_t b) { return bar0 + 8 * (2 * S::kStages + b); };
    auto acc_empty = [&](uint32_t b) { return bar0 + 8 * (2 * S::kStages + 2 + b); };
    expert_tiles(a.offsets, a.n_experts, T, tiles);
    if (threadIdx.x == 0) {
        gave_up = 0;
        for (uint32_t s = 0; s < S::kStages; s++) {
            bar_init(full(s), 1);
            bar_init(empty(s), 1);
        }
        for (uint32_t b = 0; b < 2; b++) {
            bar_init(acc_full(b), 1);
            bar_init(acc_empty(b), kStoreWarps);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == kStoreWarps + 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_slot)), "r"(S::kTmem)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = tmem_slot;
    const uint32_t per_tile = a.col_tiles * a.splits, items = tiles[a.n_experts] * per_tile;  // below 2^32 (the host's rule)

    // the item's expert (found by walking on from the last item's), its row tile, column tile and stages
    struct Item {
        uint32_t expert, row_tile, col_tile, first, last;
    };
    auto item_at = [&](uint32_t i, uint32_t& e) {
        while (i >= tiles[e + 1] * per_tile) e++;
        const uint32_t mine = tiles[e + 1] - tiles[e], j = i - tiles[e] * per_tile, q = j / mine;
        Item it;
        it.expert = e;
        it.row_tile = j - q * mine;
        it.col_tile = q % a.col_tiles;
        it.first = q / a.col_tiles * a.blocks_per_split;
        it.last = it.first + a.blocks_per_split < a.k_blocks ? it.first + a.blocks_per_split : a.k_blocks;
        return it;
    };

    uint32_t e = 0;
    if (warp == kStoreWarps && lane == 0) {
        uint32_t stage = 0, phase = 0;
        auto weights_of = [&](const Item& it) {
            return a.weights + ((uint64_t)(it.expert * a.col_tiles + it.col_tile) * a.k_blocks) * (WD * kTileBytes);
        };
        auto rows_of = [&](const Item& it) { return a.x + ((uint64_t)(tiles[it.expert] + it.row_tile) * a.k_blocks) * (XD * T * 128); };
        // The rows' digits may still be in the making: the first item's first stages get their weights before that is over
        uint32_t ahead = 0;
        if (blockIdx.x < items) {
            const Item it = item_at(blockIdx.x, e);
            const int8_t* w = weights_of(it);
            ahead = it.last - it.first < S::kStages ? it.last - it.first : S::kStages;
            for (uint32_t s = 0; s < ahead; s++) {
                bar_expect(full(s), S::kStageBytes);
                bulk_load(ring + s * S::kStageBytes, w + (uint64_t)(it.first + s) * (WD * kTileBytes), WD * kTileBytes, full(s));
            }
        }
        wait_for_previous();
        for (uint32_t i = blockIdx.x; i < items; i += gridDim.x) {
            const Item it = item_at(i, e);
            const int8_t *w = weights_of(it), *x = rows_of(it);
            for (uint32_t k = it.first; k < it.last; k++) {
                if (!bar_wait(empty(stage), phase ^ 1, &gave_up)) goto done;
                const uint32_t dst = ring + stage * S::kStageBytes;
                if (ahead) {
                    ahead--;
                } else {
                    bar_expect(full(stage), S::kStageBytes);
                    bulk_load(dst, w + (uint64_t)k * (WD * kTileBytes), WD * kTileBytes, full(stage));
                }
                bulk_load(dst + WD * kTileBytes, x + (uint64_t)k * (XD * T * 128), XD * T * 128, full(stage));
                if (++stage == S::kStages) {
                    stage = 0;
                    phase ^= 1;
                }
            }
        }
        // the last products release their stages before the block may end
        for (uint32_t s = 0; s < S::kStages; s++) {
            if (!bar_wait(empty(stage), phase ^ 1, &gave_up)) goto done;
            if (++stage == S::kStages) {
                stage = 0;
                phase ^= 1;
            }
        }
    } else if (warp == kStoreWarps + 1 && lane == 0) {
        // D = S32, A and B = signed 8 bits, both K-major
        constexpr uint32_t idesc = (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(T >> 3) << 17) | ((kTileCols >> 4) << 24);
        uint32_t stage = 0, phase = 0, buf = 0, buf_phase = 0;
        for (uint32_t i = blockIdx.x; i < items; i += gridDim.x) {
            const Item it = item_at(i, e);
            if (!bar_wait(acc_empty(buf), buf_phase ^ 1, &gave_up)) goto done;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t acc = tmem + buf * (S::kAcc * T);
            for (uint32_t k = it.first; k < it.last; k++) {
                if (!bar_wait(full(stage), phase, &gave_up)) goto done;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t base = ring + stage * S::kStageBytes;
#pragma unroll
                for (int wd = 0; wd < WD; wd++)
#pragma unroll
                    for (int xd = 0; xd < XD; xd++)
#pragma unroll
                        for (int s = 0; s < (int)kTileK / 32; s++) {
                            // the first product into an accumulator overwrites it: digit pairs (0, 0), (0, 1) or (1, 0), (1, 1)
                            const bool first = s == 0 && (wd == 0 || xd == XD - 1);
                            mma_i8(acc + (wd + xd) * T, operand_desc(base + wd * kTileBytes + s * 32),
                                   operand_desc(base + WD * kTileBytes + xd * (T * 128) + s * 32), idesc, !(first && k == it.first));
                        }
                mma_commit(empty(stage));
                if (++stage == S::kStages) {
                    stage = 0;
                    phase ^= 1;
                }
            }
            mma_commit(acc_full(buf));
            if (++buf == S::kBuffers) {
                buf = 0;
                buf_phase ^= 1;
            }
        }
    } else if (warp < kStoreWarps) {
        wait_for_previous();  // which may be clearing the output
        uint32_t buf = 0, buf_phase = 0;
        for (uint32_t i = blockIdx.x; i < items; i += gridDim.x) {
            const Item it = item_at(i, e);
            const uint32_t lo = a.offsets[e] + it.row_tile * T, end = a.offsets[e + 1];
            const int valid = end - lo < T ? (int)(end - lo) : T;
            const uint64_t c = (uint64_t)it.col_tile * kTileCols + (warp & 3) * 32 + lane;
            TileRows<T> rows;
            rows.load(a.rows, lo, valid);
            // the lanes stay together: one of them may see the limit pass where another still sees the tile arrive
            if (!__all_sync(0xffffffffu, bar_wait(acc_full(buf), buf_phase, &gave_up))) goto done;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            store_tile<S::kAcc, T>(a, tmem + buf * (S::kAcc * T) + ((warp & 3) << 21), rows, valid, c, warp >> 2,
                                   [&]() { if (lane == 0) bar_arrive(acc_empty(buf)); });
            if (++buf == S::kBuffers) {
                buf = 0;
                buf_phase ^= 1;
            }
        }
    }
done:
    __syncwarp();
    __syncthreads();
    if (gave_up) gave_up_wait(a.gave_up);
    if (warp == kStoreWarps + 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::kTmem));
    }
}

}  // namespace dpb
