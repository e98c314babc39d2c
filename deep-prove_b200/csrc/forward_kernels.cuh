// Embedding lookup, rows sorted by key, sums of rows by key.
#pragma once
#include "forward.cuh"
#include "lazy_sum.cuh"

namespace dpb {

// ------------------------------------------------------------------------------------------------ embedding lookup
// out[i, c] = (table[token_i, c] * m + r) >> s.  Moves 4 or 8 bytes in and 8 bytes out per entry and computes next to
// nothing: bound by HBM writes.  A thread makes four entries of a row (two entries of 64 bits) so that both sides are
// 16-byte accesses; rows that are not aligned for that take the scalar form.
struct LookupArgs {
    const void* table;
    const int64_t* tokens;
    uint64_t vocab, width, stride, n;  // stride: entries between table rows
    int64_t multiplier, rounding;
    uint32_t shift;
    uint64_t out_rows, out_width;  // what is written: n x width, or the padded sizes
    int64_t* out;
    uint32_t div_mul, div_shift;  // 32-bit steps: w / per_row = (w * div_mul) >> div_shift for w below 2^31
    uint32_t check_blocks;  // blocks that check the tokens; 0: every block, and the products as well
    FwdCheck check;
};

constexpr uint32_t kLookupThreads = 256;

// the entry and the multiplier fit 32 bits, so that the product and the rounding fit 64
__device__ __forceinline__ int64_t lookup_scale(const LookupArgs& a, int32_t x) {
    return ((int64_t)x * (int32_t)a.multiplier + a.rounding) >> a.shift;
}
// any product; whether it leaves 64 bits goes to `over`
__device__ __forceinline__ int64_t lookup_scale(const LookupArgs& a, int64_t x, bool& over) {
    const __int128 v = (__int128)x * a.multiplier + a.rounding;
    over = over || v != (__int128)(int64_t)v;
    return (int64_t)v >> a.shift;
}

// T: the table's integers; V: entries per step (1 or 16 bytes' worth on the narrower side).  I: the index type; 32 bits
// wherever they suffice, since finding a step's row takes a division (by a multiplication then).  kLookupFlight steps per thread are under way
// together: tokens, then table entries, then results; steps of neighbouring threads are neighbours, and a thread's own
// lie a grid apart (next to each other they fill fewer blocks of a short call: 8 us instead of 5).  16384 rows of 4096
// entries of 8 bytes take 168 us: 1.07 GB, of which 0.74 GB from and to HBM (4.4 TB/s) and the rest rows that several
// tokens share.  Neither HBM (57 %) nor the instructions' issue (60 %) is full; the registers hold 46 % of an SM's warps.
constexpr int kLookupFlight = 4;
template <class T, int V, bool CHECK, class I>
__global__ void __launch_bounds__(kLookupThreads, sizeof(I) == 4 ? 4 : 2) embedding_lookup_kernel(LookupArgs a) {
    unsigned int found = 0;
    const bool small = a.multiplier == (int32_t)a.multiplier;
    const I per_row = (I)((a.out_width + V - 1) / V), total = (I)a.out_rows * per_row;
    const I step = (I)gridDim.x * kLookupThreads;
    if (!CHECK && blockIdx.x < a.check_blocks) {
        // the checking blocks look at all tokens first, so that the host need not wait for the rows
        for (uint64_t i = (uint64_t)blockIdx.x * kLookupThreads + threadIdx.x; i < a.n; i += (uint64_t)a.check_blocks * kLookupThreads)
            if ((uint64_t)a.tokens[i] >= a.vocab) found = kFwdKeyRange;
        fwd_check_done(a.check, found, a.check_blocks);
    }
    for (I w0 = (I)blockIdx.x * kLookupThreads + threadIdx.x; w0 < total; w0 += kLookupFlight * step) {
        uint64_t row[kLookupFlight], col[kLookupFlight], tok[kLookupFlight];
        T x[kLookupFlight][V];
#pragma unroll
        for (int f = 0; f < kLookupFlight; f++) {
            const I w = w0 + f * step;  // 32 bits: total + 2 kLookupFlight step stays below 2^31 (the host's rule)
            const I i = sizeof(I) == 4 ? (I)(((uint64_t)w * a.div_mul) >> a.div_shift) : w / per_row;
            row[f] = i;
            col[f] = (uint64_t)(w - i * per_row) * V;
            tok[f] = w < total && row[f] < a.n && col[f] < a.width ? (uint64_t)__ldg((const long long*)a.tokens + i) : ~0ull - 1;
        }
#pragma unroll
        for (int f = 0; f < kLookupFlight; f++) {
#pragma unroll
            for (int v = 0; v < V; v++) x[f][v] = 0;
            if (tok[f] < a.vocab) {
                const T* src = (const T*)a.table + tok[f] * a.stride + col[f];
                if constexpr (V * sizeof(T) == 16) *(int4*)x[f] = __ldg((const int4*)src);
                else x[f][0] = __ldg(src);
            }
        }
#pragma unroll
        for (int f = 0; f < kLookupFlight; f++) {
            if (w0 + f * step >= total) break;
            const bool live = tok[f] < a.vocab;
            if (CHECK && !live && row[f] < a.n && col[f] < a.width) found |= kFwdKeyRange;
            int64_t y[V];
#pragma unroll
            for (int v = 0; v < V; v++) {
                const bool in = live && (V == 1 || col[f] + v < a.width);  // not between the width and the stride
                y[v] = 0;
                if (!CHECK || (small && x[f][v] == (T)(int32_t)x[f][v])) {
                    if (in) y[v] = lookup_scale(a, (int32_t)x[f][v]);
                } else if (in) {
                    bool over = false;
                    y[v] = lookup_scale(a, (int64_t)x[f][v], over);
                    if (over) found |= kFwdValueRange;
                }
            }
            int64_t* o = a.out + (uint64_t)(w0 + f * step) * V;  // rows follow one another: V divides the width written
            if constexpr (V == 1) {
                *o = y[0];
            } else {
#pragma unroll
                for (int v = 0; v < V; v += 2) *(longlong2*)(o + v) = make_longlong2(y[v], y[v + 1]);
            }
        }
    }
    if (CHECK) fwd_check_done(a.check, found, gridDim.x);
}

// ------------------------------------------------------------------------------------------------ rows by key
// Up to kSmallSort rows: the place of a row is the number of rows that go before it (a smaller key, or the same key and
// a smaller row), counted against all keys in shared memory by eight threads per row: n^2 comparisons over many SMs in
// one launch, where a sorting network in one block waits at its barriers (2048 rows: 25 us) and a counting sort takes
// three launches.  The first places of the keys, where they are kept, are counted the same way.
constexpr uint32_t kSmallSort = 4096, kSmallSortThreads = 256;
__global__ void __launch_bounds__(kSmallSortThreads)
    groups_small_kernel(const int64_t* __restrict__ keys, uint32_t n, uint32_t n_keys, uint32_t* __restrict__ out_keys,
                        uint32_t* __restrict__ out_rows, uint32_t* __restrict__ places, uint32_t* __restrict__ offsets, FwdCheck check) {
    extern __shared__ uint4 sh4[];
    let_next_start();
    uint32_t* sh = (uint32_t*)sh4;
    const uint32_t n_up = (n + 31) & ~31u;
    unsigned int found = 0;
    for (uint32_t i = threadIdx.x; i < n_up; i += kSmallSortThreads) {
        uint32_t k = 0xffffffffu;
        if (i < n) {
            const uint64_t k64 = (uint64_t)keys[i];
            if (k64 >= n_keys) found = kFwdKeyRange;
            k = k64 < n_keys ? (uint32_t)k64 : n_keys;
        }
        sh[i] = k;
    }
    if (blockIdx.x == 0) fwd_check_done(check, found, 1);
    __syncthreads();
    const uint32_t t = blockIdx.x * kSmallSortThreads + threadIdx.x, part = t & 7, i = t >> 3;
    const uint32_t probes = n + (offsets ? n_keys + 1 : 0);
    const uint32_t k = i < n ? sh[i] : i - n;  // a row's key, or a key whose first place is asked for
    uint32_t below = 0;
    for (uint32_t q = part; q < n_up / 4; q += 8) {
        const uint4 v = sh4[q];
        // rows before i with the same key count as well: key <= k up to i, key < k from there on
        const uint32_t j = 4 * q;
        if (i < n && j + 4 <= i) {
            below += (v.x <= k) + (v.y <= k) + (v.z <= k) + (v.w <= k);
        } else {
            below += (v.x < k) + (v.y < k) + (v.z < k) + (v.w < k);
            if (i < n && j < i) below += (v.x == k) + (j + 1 < i && v.y == k) + (j + 2 < i && v.z == k);
        }
    }
#pragma unroll
    for (int off = 4; off > 0; off >>= 1) below += __shfl_down_sync(0xffffffffu, below, off);
    if (part == 0 && i < probes) {
        if (i < n) {
            out_keys[below] = k;
            out_rows[below] = i;
            places[i] = below;
        } else {
            offsets[i - n] = below;
        }
    }
}

// Few keys (experts) and up to kFewSort rows: one block, each warp a run of neighbouring rows that it keeps in registers.
// Counts per (key, warp) in shared memory, their prefix sums in that order, then every row's place; rows keep their order
// inside a key.  8192 rows of 8 experts: 3 us less than the three launches below; 1996 rows of 60: 3 us more than the
// comparisons above, which therefore keep what they can take.
constexpr uint32_t kFewKeys = 256, kFewSort = 16384, kFewThreads = 1024, kFewPer = kFewSort / kFewThreads;
__global__ void __launch_bounds__(kFewThreads)
    groups_few_kernel(const int64_t* __restrict__ keys, uint32_t n, uint32_t n_keys, uint32_t* __restrict__ out_keys,
                      uint32_t* __restrict__ out_rows, uint32_t* __restrict__ places, uint32_t* __restrict__ offsets, FwdCheck check) {
    extern __shared__ uint4 sh4[];
    let_next_start();
    uint32_t* count = (uint32_t*)sh4;  // [n_keys + 1][32]: key n_keys holds the rows whose key is out of range
    __shared__ uint32_t warp_sum[32];
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, cells = (n_keys + 1) * 32;
    const uint32_t per_warp = ((n + kFewThreads - 1) / kFewThreads) * 32, first = warp * per_warp;
    uint32_t k[kFewPer];
    unsigned int found = 0;
#pragma unroll
    for (uint32_t q = 0; q < kFewPer; q++) {
        const uint32_t i = first + 32 * q + lane;
        k[q] = 0xffffffffu;  // no row
        if (32 * q < per_warp && i < n) {
            const uint64_t k64 = (uint64_t)keys[i];
            k[q] = k64 < n_keys ? (uint32_t)k64 : n_keys;
            if (k[q] == n_keys) found = kFwdKeyRange;
        }
    }
    for (uint32_t i = threadIdx.x; i < cells; i += kFewThreads) count[i] = 0;
    fwd_check_done(check, found, 1);
    __syncthreads();
    uint32_t before[kFewPer];  // rows of the key before this one, in the warp
#pragma unroll
    for (uint32_t q = 0; q < kFewPer; q++) {
        if (32 * q >= per_warp) break;
        const unsigned peers = __match_any_sync(0xffffffffu, k[q]);
        const uint32_t cell = k[q] == 0xffffffffu ? 0 : k[q] * 32 + warp;
        before[q] = k[q] == 0xffffffffu ? 0 : count[cell] + __popc(peers & ((1u << lane) - 1));
        __syncwarp();
        if (k[q] != 0xffffffffu && (int)lane == __ffs(peers) - 1) count[cell] += __popc(peers);
        __syncwarp();
    }
    __syncthreads();
    // exclusive prefix sums over the cells: a thread sums a run of them, then the block the threads' sums
    const uint32_t per = (cells + kFewThreads - 1) / kFewThreads, c0 = threadIdx.x * per;
    uint32_t sum = 0;
    for (uint32_t c = c0; c < c0 + per && c < cells; c++) sum += count[c];
    uint32_t incl = sum;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const uint32_t t = __shfl_up_sync(0xffffffffu, incl, off);
        if (lane >= (uint32_t)off) incl += t;
    }
    if (lane == 31) warp_sum[warp] = incl;
    __syncthreads();
    if (warp == 0) {
        uint32_t w = warp_sum[lane];
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const uint32_t t = __shfl_up_sync(0xffffffffu, w, off);
            if (lane >= (uint32_t)off) w += t;
        }
        warp_sum[lane] = w;
    }
    __syncthreads();
    uint32_t run = incl - sum + (warp ? warp_sum[warp - 1] : 0);
    for (uint32_t c = c0; c < c0 + per && c < cells; c++) {
        const uint32_t t = count[c];
        count[c] = run;
        run += t;
    }
    __syncthreads();
    for (uint32_t e = threadIdx.x; e <= n_keys; e += kFewThreads) offsets[e] = count[e * 32];
#pragma unroll
    for (uint32_t q = 0; q < kFewPer; q++) {
        const uint32_t i = first + 32 * q + lane;
        if (32 * q < per_warp && i < n) {
            const uint32_t p = count[k[q] * 32 + warp] + before[q];
            out_keys[p] = k[q];
            out_rows[p] = i;
            places[i] = p;
        }
    }
}

// More rows: a counting sort.  rank[i] is the row's place inside its key; equal keys of a warp share one atomic.
__global__ void __launch_bounds__(kThreads)
    groups_count_kernel(const int64_t* __restrict__ keys, uint32_t n, uint32_t n_keys, uint32_t* __restrict__ counts,
                        uint32_t* __restrict__ rank, FwdCheck check) {
    unsigned int found = 0;
    let_next_start();
    const uint32_t stride = gridDim.x * kThreads, lane = threadIdx.x & 31;
    const uint64_t n_up = ((uint64_t)n + 31) & ~31ull;
    for (uint64_t i = (uint64_t)blockIdx.x * kThreads + threadIdx.x; i < n_up; i += stride) {
        const bool live = i < n;
        const uint64_t k64 = live ? (uint64_t)keys[i] : 0;
        const uint32_t k = !live ? 0xffffffffu : k64 < n_keys ? (uint32_t)k64 : n_keys;
        if (live && k == n_keys) found = kFwdKeyRange;
        const unsigned peers = __match_any_sync(0xffffffffu, k);
        const int leader = __ffs(peers) - 1;
        uint32_t base = 0;
        if (live && (int)lane == leader) base = atomicAdd(&counts[k], (uint32_t)__popc(peers));
        base = __shfl_sync(0xffffffffu, base, leader);
        if (live) rank[i] = base + __popc(peers & ((1u << lane) - 1));
    }
    fwd_check_done(check, found, gridDim.x);
}

constexpr uint32_t kCountTile = 4096;  // counters per block of the scan
// exclusive prefix sums inside a tile (in place) and the tiles' sums
__global__ void __launch_bounds__(1024)
    groups_scan_kernel(uint32_t* counts, uint32_t n, uint32_t* tile_sums) {
    __shared__ uint32_t warp_sum[32];
    let_next_start();
    wait_for_previous();
    const uint32_t base = blockIdx.x * kCountTile + threadIdx.x * 4, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t c[4], sum = 0;
#pragma unroll
    for (int u = 0; u < 4; u++) {
        c[u] = base + u < n ? counts[base + u] : 0;
        sum += c[u];
    }
    uint32_t incl = sum;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const uint32_t t = __shfl_up_sync(0xffffffffu, incl, off);
        if (lane >= (uint32_t)off) incl += t;
    }
    if (lane == 31) warp_sum[warp] = incl;
    __syncthreads();
    if (warp == 0) {
        uint32_t w = warp_sum[lane];
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const uint32_t t = __shfl_up_sync(0xffffffffu, w, off);
            if (lane >= (uint32_t)off) w += t;
        }
        warp_sum[lane] = w;
    }
    __syncthreads();
    uint32_t run = incl - sum + (warp ? warp_sum[warp - 1] : 0);
#pragma unroll
    for (int u = 0; u < 4; u++) {
        if (base + u < n) counts[base + u] = run;
        run += c[u];
    }
    if (threadIdx.x == 0) tile_sums[blockIdx.x] = warp_sum[31];
}

// tiles <= 1025: every block adds the tiles' sums up for itself
__global__ void __launch_bounds__(kThreads)
    groups_scatter_kernel(const int64_t* keys, uint32_t n, uint32_t n_keys, const uint32_t* counts, const uint32_t* tile_sums,
                          uint32_t tiles, uint32_t* rank, uint32_t* out_keys, uint32_t* out_rows) {
    __shared__ uint32_t before[1056];
    let_next_start();
    wait_for_previous();
    if (threadIdx.x < 32) {
        uint32_t carry = 0;
        for (uint32_t t0 = 0; t0 < tiles; t0 += 32) {
            const uint32_t s = t0 + threadIdx.x < tiles ? tile_sums[t0 + threadIdx.x] : 0;
            uint32_t incl = s;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const uint32_t u = __shfl_up_sync(0xffffffffu, incl, off);
                if (threadIdx.x >= (uint32_t)off) incl += u;
            }
            before[t0 + threadIdx.x] = carry + incl - s;
            carry += __shfl_sync(0xffffffffu, incl, 31);
        }
    }
    __syncthreads();
    const uint32_t stride = gridDim.x * kThreads;
    for (uint64_t i = (uint64_t)blockIdx.x * kThreads + threadIdx.x; i < n; i += stride) {
        const uint64_t k64 = (uint64_t)keys[i];
        const uint32_t k = k64 < n_keys ? (uint32_t)k64 : n_keys;
        const uint32_t p = before[k / kCountTile] + counts[k] + rank[i];
        out_keys[p] = k;
        out_rows[p] = (uint32_t)i;
        rank[i] = p;  // from here on the row's place in the whole order
    }
}

// ------------------------------------------------------------------------------------------------ sums by key
// S[k, c] = m * sum_{i in k} w_i x[i / per, c] over rows in sorted order.  The order is cut into equal slices; a key that
// lies in one slice is finished by the slice's block, a key that spans several leaves one part per slice (slot 0: it
// began before the slice, slot 1: it begins there), and a second launch adds those up.  Every sum is exact, so neither
// the cut nor the rows' order inside a key changes a result.
struct RowSumArgs {
    const uint32_t* keys;
    const uint32_t* rows;
    uint64_t n, n_keys;  // a row's key is below n_keys; n_keys itself marks rows whose key was out of range: no sum
    uint64_t slice;      // rows per slice
    const void* weights;
    const int64_t* x;
    uint64_t width;
    uint32_t per;  // routed rows per row of x
    uint64_t out_width;
    void* out;
    void* parts;  // [slice][2][width]
    const uint32_t* offsets;  // first places of the keys, where the kernel writes the zeros of the result; null: the host does
    uint64_t out_keys;
};

// The result's entries that no sum goes to: rows of keys without rows, and the padding.  All threads share them; the grid
// has rows of blocks past the slices for this when the slices alone are few.
template <class F>
__device__ __forceinline__ void clear_unsummed(const RowSumArgs& a) {
    if (!a.offsets) return;
    const uint32_t shift = 63 - __clzll((long long)a.out_width);  // a power of two
    const uint64_t entries = a.out_keys << shift, step = (uint64_t)gridDim.x * gridDim.y * blockDim.x;
    for (uint64_t i = ((uint64_t)blockIdx.y * gridDim.x + blockIdx.x) * blockDim.x + threadIdx.x; i < entries; i += step) {
        const uint64_t k = i >> shift, c = i & (a.out_width - 1);
        if (k >= a.n_keys || c >= a.width || a.offsets[k] == a.offsets[k + 1]) F::store(a.out, i, F::zero());
    }
}

// An unreduced sum of (weight) * (integer) products.  A weight's 32-bit words and an entry of up to 16 bits are exact in
// a double, a product is at most 2^47 and kExactRows of them stay within 2^53: the sums run as one fused multiply-add per
// word on the 64-bit floating-point pipe, exactly, and move to signed 64-bit integers every kExactRows rows.  Wide integer
// multiply-adds run at half a double's rate, and came with as many moves: 8192 rows of 4096 over BN254 took 88 us in a
// chain of carries, 76 us in one 64-bit accumulator per word, and take 58 us this way.  What bounds it then is shared
// between the weights' and entries' way through shared memory (64 % of its wavefronts) and the instructions' issue (53 %).
// What an entry has above 16 bits, as quantised activations do not, takes a field product.
constexpr uint32_t kExactRows = 64;
constexpr uint64_t kRowSumMaxSlice = 49152;  // rows per slice: 2^47 times as many stays below 2^63
// an integer below 2^31 in magnitude as a double, by its place next to 2^52
__device__ __forceinline__ double exact_double(int32_t x) {
    return __hiloint2double(0x43300000, x ^ (int32_t)0x80000000) - 4503601774854144.0;  // 2^52 + 2^31
}
__device__ __forceinline__ double exact_double(uint32_t x) { return __hiloint2double(0x43300000, (int32_t)x) - 4503599627370496.0; }
template <class F>
struct RowWords;
template <>
struct RowWords<FrFam> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void cut(const Fr& w, double* out) {
        const frw::F8 v = frw::from_fr(w);
#pragma unroll
        for (int j = 0; j < 8; j++) out[j] = exact_double(v.w[j]);
    }
    // sum_j a_j 2^(32 j), signed: what lies below 2^256, and the signed rest times 2^256, which is the rest's Montgomery form
    static __device__ __forceinline__ Fr value(const int64_t* a) {
        frw::F8 lo;
        int64_t carry = 0;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int64_t v = a[j] + carry;
            lo.w[j] = (uint32_t)v;
            carry = v >> 32;
        }
        return fr_add(frw::to_fr(frw::reduce_256(lo)), fr_from_int_rows(carry));
    }
};
template <>
struct RowWords<GlFam> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void cut(const Gl2& w, double* out) {
        const glw::W2 v = gl2_words(w);
        out[0] = exact_double(v.c0.lo);
        out[1] = exact_double(v.c0.hi);
        out[2] = exact_double(v.c1.lo);
        out[3] = exact_double(v.c1.hi);
    }
    static __device__ __forceinline__ uint64_t component(int64_t a0, int64_t a1) {
        const int64_t v1 = a1 + (a0 >> 32), top = v1 >> 32;  // the number: top 2^64 + (v1's low word, a0's low word)
        const uint64_t mag = top < 0 ? (uint64_t)0 - (uint64_t)top : (uint64_t)top;
        glw::A5 l, h;
        l.w0 = (uint32_t)a0;
        l.w1 = (uint32_t)v1;
        l.w2 = l.w3 = l.w4 = 0;
        h.w0 = h.w1 = h.w4 = 0;
        h.w2 = (uint32_t)mag;
        h.w3 = (uint32_t)(mag >> 32);
        const uint64_t lv = glw::to_u64(glw::canon(glw::acc_reduce(l))), hv = glw::to_u64(glw::canon(glw::acc_reduce(h)));
        return top < 0 ? gl_sub(lv, hv) : gl_add(lv, hv);
    }
    static __device__ __forceinline__ Gl2 value(const int64_t* a) { return gl2_make(component(a[0], a[1]), component(a[2], a[3])); }
};
template <class F>
__device__ __forceinline__ typename F::E field_from_i128(__int128 v) {
    const bool neg = v < 0;
    const unsigned __int128 m = neg ? (unsigned __int128)0 - (unsigned __int128)v : (unsigned __int128)v;
    typename F::E r = F::from_u64((uint64_t)m);
    if ((uint64_t)(m >> 64)) r = F::add(r, F::mul(F::from_u64((uint64_t)(m >> 64)), F::from_u64_pow64()));
    return neg ? F::neg(r) : r;
}

// v + w * (x - its low 16 bits, signed)
template <class F>
__device__ __noinline__ typename F::E add_high(typename F::E v, const typename F::E w, int64_t x) {
    const int64_t hi = (x >> 16) + ((x >> 15) & 1);  // x = its low 16 bits, signed, + 2^16 hi
    const typename F::E t = F::mul(w, F::mul(F::from_u64(hi < 0 ? (uint64_t)0 - (uint64_t)hi : (uint64_t)hi), F::from_u64(1ull << 16)));
    return hi < 0 ? F::sub(v, t) : F::add(v, t);
}

// A block: neighbouring columns of one slice.  Rows come in batches whose places and run ends, and weights, go through
// shared memory.  Without weights a thread loads kRowSumFlight rows' entries ahead of the sums.
constexpr uint32_t kRowSumThreads = 128, kRowSumBatch = 64, kRowSumFlight = 8;

// With weights: two columns per thread (a weight read from shared memory then serves two products).  The entries come
// through a per-thread ring in shared memory, kRingAhead groups of eight rows ahead of the products, so that loads are
// under way all the time (groups of four, three ahead: 3 us more over BN254, 8192 rows of 4096).
constexpr uint32_t kRowRing = 2, kRingAhead = kRowRing - 1, kProductBatch = 128, kGroup = 8;
template <int BYTES>
__device__ __forceinline__ void ring_load(void* dst, const void* src) {
    if constexpr (BYTES == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
}
// blocks per SM that the registers are held down for (BN254, 8192 rows of 4096: 3 us more with three, which spill nothing)
template <class F>
constexpr int kProductBlocks = sizeof(typename F::E) == 32 ? 4 : 5;
// PAIRS: rows of an even number of entries at 16-byte addresses, so that a thread's two columns are one word
template <class F, bool PAIRS>
__global__ void __launch_bounds__(kRowSumThreads, kProductBlocks<F>)
    row_products_kernel(RowSumArgs a, typename F::E multiplier, bool scale) {
    typedef typename F::E E;
    constexpr int C = 2, N = RowWords<F>::N;
    let_next_start();
    wait_for_previous();
    clear_unsummed<F>(a);
    __shared__ __align__(16) double wsh[kProductBatch + 1][N];  // the last weight is zero
    __shared__ longlong2 ring[kRowRing][kGroup][kRowSumThreads];
    __shared__ const int64_t* from[kProductBatch];
    __shared__ uint32_t keys[kProductBatch];
    __shared__ uint32_t ends[kProductBatch / 32];  // a bit per row: the key's run ends here
    const uint32_t tid = threadIdx.x, lane = tid & 31;
    const uint64_t c0 = ((uint64_t)blockIdx.x * kRowSumThreads + tid) * C;
    const uint64_t begin = blockIdx.y * a.slice, end = begin + a.slice < a.n ? begin + a.slice : a.n;
    if (begin >= a.n) return;
    const bool live[C] = {c0 < a.width, c0 + 1 < a.width};
    // columns past the last read some column's entries, and keep the result to themselves
    const uint64_t c_load = live[0] ? c0 : 0, second = live[1] ? 1 : 0;
    if (tid < N) wsh[kProductBatch][tid] = 0.0;
    bool before = begin > 0 && a.keys[begin - 1] == a.keys[begin];  // the current run began before the slice
    double acc[C][N];
    int64_t sum[C][N];
    E wide[C];  // what the entries of more than 16 bits add (seldom any)
    bool any_wide = false;
#pragma unroll
    for (int q = 0; q < C; q++) {
#pragma unroll
        for (int j = 0; j < N; j++) {
            acc[q][j] = 0.0;
            sum[q][j] = 0;
        }
        wide[q] = F::zero();
    }
    auto drain = [&]() {
#pragma unroll
        for (int q = 0; q < C; q++)
#pragma unroll
            for (int j = 0; j < N; j++) {
                sum[q][j] += (int64_t)acc[q][j];
                acc[q][j] = 0.0;
            }
    };
    for (uint64_t p0 = begin; p0 < end; p0 += kProductBatch) {
        const uint32_t m = end - p0 < kProductBatch ? (uint32_t)(end - p0) : kProductBatch;
        __syncthreads();
        {
            const uint64_t p = p0 + (tid < m ? tid : m - 1);
            const uint32_t row = a.rows[p], key = a.keys[p];
            from[tid] = a.x + (uint64_t)(row / a.per) * a.width;
            keys[tid] = key;
            const uint32_t run_ends = __ballot_sync(0xffffffffu, tid < m && (p + 1 == end || a.keys[p + 1] != key));
            if (lane == 0) ends[tid >> 5] = run_ends;
            RowWords<F>::cut(F::load(a.weights, F::kChalDtype, row), wsh[tid]);
        }
        __syncthreads();
        auto issue = [&](uint32_t g) {
            if (kGroup * g < m) {
                longlong2* dst = &ring[g % kRowRing][0][tid];
#pragma unroll
                for (uint32_t u = 0; u < kGroup; u++) {  // rows past the batch's last repeat that one
                    const int64_t* src = from[kGroup * g + u] + c_load;
                    if (PAIRS) {
                        ring_load<16>(dst + u * kRowSumThreads, src);
                    } else {
                        ring_load<8>(&dst[u * kRowSumThreads].x, src);
                        ring_load<8>(&dst[u * kRowSumThreads].y, src + second);
                    }
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
#pragma unroll
        for (uint32_t g = 0; g < kRingAhead; g++) issue(g);
        uint32_t next = 0;  // the first group that was not waited for
        // One run, or the part of it in this batch, after the other.  The loop over its rows holds the products alone: with
        // the ends of runs unrolled into it, it left the instruction cache.
        for (uint32_t s = 0; s < m;) {
            uint32_t h = s >> 5, rest = ends[h] >> (s & 31) << (s & 31);
            while (!rest && ++h < kProductBatch / 32) rest = ends[h];
            const uint32_t t = rest ? 32 * h + __ffs(rest) - 1 : m - 1;  // the run's last row here
            for (uint32_t g = s / kGroup; g <= t / kGroup; g++) {
                if (g == next) {
                    asm volatile("cp.async.wait_group %0;" ::"n"(kRingAhead - 1) : "memory");
                    issue(g + kRingAhead);  // into the group before this one, whose products are done
                    next++;
                }
                bool more = false;  // an entry has more than 16 bits
                const longlong2* x4 = &ring[g % kRowRing][0][tid];
#pragma unroll
                for (uint32_t u = 0; u < kGroup; u++) {
                    const uint32_t i = kGroup * g + u;
                    const double* w = wsh[i >= s && i <= t ? i : kProductBatch];  // other runs' rows: times 0
                    const longlong2 x2 = x4[u * kRowSumThreads];
#pragma unroll
                    for (int q = 0; q < C; q++) {
                        const int64_t x = q ? x2.y : x2.x;
                        more |= x != (int64_t)(int16_t)x;
                        const double d = exact_double((int32_t)(int16_t)x);
#pragma unroll
                        for (int j = 0; j < N; j++) acc[q][j] = fma(w[j], d, acc[q][j]);
                    }
                }
                if (more) {
#pragma unroll 1
                    for (uint32_t i = max(s, kGroup * g); i <= min(t, kGroup * g + kGroup - 1); i++) {
                        const E w = F::load(a.weights, F::kChalDtype, a.rows[p0 + i]);
                        const longlong2 x2 = x4[i % kGroup * kRowSumThreads];
                        wide[0] = add_high<F>(wide[0], w, x2.x);
                        wide[1] = add_high<F>(wide[1], w, x2.y);
                    }
                    any_wide = true;
                }
                if (g % (kExactRows / kGroup) == kExactRows / kGroup - 1) drain();
            }
            drain();
            if (rest) {
                const uint32_t key = keys[t];
                const bool after = p0 + t + 1 == end && end < a.n && a.keys[end] == key;
#pragma unroll
                for (int q = 0; q < C; q++) {
                    if (live[q] && key < a.n_keys) {
                        const uint64_t c = c0 + q;
                        E v = RowWords<F>::value(sum[q]);
                        if (any_wide) v = F::add(v, wide[q]);
                        if (before || after) {
                            F::store(a.parts, ((uint64_t)blockIdx.y * 2 + (before ? 0 : 1)) * a.width + c, v);
                        } else {
                            if (scale) v = F::mul(v, multiplier);
                            F::store(a.out, (uint64_t)key * a.out_width + c, v);
                        }
                    }
#pragma unroll
                    for (int j = 0; j < N; j++) sum[q][j] = 0;
                    if (any_wide) wide[q] = F::zero();
                }
                any_wide = false;
                before = false;
            }
            s = t + 1;
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    }
}

// an integer as a field element: from its two words where it fits 64 bits
template <class F>
__device__ __forceinline__ typename F::E field_from_int(__int128 v);
template <>
__device__ __forceinline__ Fr field_from_int<FrFam>(__int128 v) {
    return v == (__int128)(int64_t)v ? fr_from_int_rows((int64_t)v) : field_from_i128<FrFam>(v);
}
template <>
__device__ __forceinline__ Gl2 field_from_int<GlFam>(__int128 v) {
    return v == (__int128)(int64_t)v ? gl2_from_base(GlFam::base_from_int((int64_t)v)) : field_from_i128<GlFam>(v);
}
template <class F>
__device__ __noinline__ void store_sum(__int128 sum, bool part, bool scale, const typename F::E& multiplier, void* out, uint64_t i) {
    typename F::E v = field_from_int<F>(sum);
    if (scale && !part) v = F::mul(v, multiplier);
    F::store(out, i, v);
}

// the integers alone: 128-bit sums, one column per thread
template <class F>
__global__ void __launch_bounds__(kRowSumThreads)
    row_sums_kernel(RowSumArgs a, typename F::E multiplier, bool scale) {
    typedef typename F::E E;
    let_next_start();
    wait_for_previous();
    clear_unsummed<F>(a);
    __shared__ uint64_t at[kRowSumBatch];
    __shared__ uint32_t ends[kRowSumBatch];
    const uint64_t c = (uint64_t)blockIdx.x * kRowSumThreads + threadIdx.x;
    const uint64_t begin = blockIdx.y * a.slice, end = begin + a.slice < a.n ? begin + a.slice : a.n;
    if (begin >= a.n) return;
    const bool live = c < a.width;
    bool before = begin > 0 && a.keys[begin - 1] == a.keys[begin];
    __int128 acc = 0;
    for (uint64_t p0 = begin; p0 < end; p0 += kRowSumBatch) {
        const uint32_t m = end - p0 < kRowSumBatch ? (uint32_t)(end - p0) : kRowSumBatch;
        __syncthreads();
        if (threadIdx.x < kRowSumBatch) {
            const uint64_t p = p0 + (threadIdx.x < m ? threadIdx.x : m - 1);
            const uint32_t key = a.keys[p];
            at[threadIdx.x] = (uint64_t)(a.rows[p] / a.per) * a.width;
            ends[threadIdx.x] = threadIdx.x < m && (p + 1 == end || a.keys[p + 1] != key) ? key + 1 : 0;
        }
        __syncthreads();
        for (uint32_t i0 = 0; i0 < m; i0 += kRowSumFlight) {
            int64_t x[kRowSumFlight];
#pragma unroll
            for (uint32_t u = 0; u < kRowSumFlight; u++)
                x[u] = live && i0 + u < m ? a.x[at[i0 + u] + c] : 0;
#pragma unroll
            for (uint32_t u = 0; u < kRowSumFlight; u++) {
                const uint32_t i = i0 + u;
                if (i >= m) break;
                acc += x[u];
                if (ends[i]) {
                    const uint32_t key = ends[i] - 1;
                    const bool after = p0 + i + 1 == end && end < a.n && a.keys[end] == key;
                    if (live && key < a.n_keys) {
                        const uint64_t slot = ((uint64_t)blockIdx.y * 2 + (before ? 0 : 1)) * a.width + c;
                        store_sum<F>(acc, before || after, scale, multiplier, before || after ? a.parts : a.out,
                                     before || after ? slot : (uint64_t)key * a.out_width + c);
                    }
                    acc = 0;
                    before = false;
                }
            }
        }
    }
}

// First place whose key is not below `key`, by a warp: 32 probes per step.
__device__ __forceinline__ uint64_t warp_first_at(const uint32_t* keys, uint64_t n, uint64_t key) {
    uint64_t lo = 0, hi = n;  // the answer lies in [lo, hi]
    const uint32_t lane = threadIdx.x & 31;
    while (lo < hi) {
        const uint64_t step = (hi - lo + 31) / 32, at = lo + lane * step;
        const bool below = at < hi && keys[at] < key;
        const uint32_t k = __popc(__ballot_sync(0xffffffffu, below));  // probes 0..k-1 are below
        if (k == 0) return lo;
        const uint64_t next = lo + k * step;
        lo = lo + (uint64_t)(k - 1) * step + 1;
        if (next < hi) hi = next;
    }
    return lo;
}

// Adds up the keys that span slices: block row y looks at slice y, and acts when a key begins there and goes on.
template <class F>
__global__ void __launch_bounds__(kRowSumThreads)
    row_sums_join_kernel(RowSumArgs a, typename F::E multiplier, bool scale) {
    typedef typename F::E E;
    wait_for_previous();
    const uint64_t begin = blockIdx.y * a.slice, end = begin + a.slice;
    if (end >= a.n) return;
    const uint32_t key = a.keys[end - 1];
    if (a.keys[end] != key || key >= a.n_keys) return;  // nothing goes on
    if (begin > 0 && a.keys[begin - 1] == key) return;  // it began before
    const uint64_t last = (warp_first_at(a.keys, a.n, (uint64_t)key + 1) - 1) / a.slice;
    const uint64_t c = (uint64_t)blockIdx.x * kRowSumThreads + threadIdx.x;
    if (c >= a.width) return;
    E v = F::load(a.parts, F::kChalDtype, ((uint64_t)blockIdx.y * 2 + 1) * a.width + c);
    for (uint64_t s = blockIdx.y + 1; s <= last; s += 4) {
        E part[4];
#pragma unroll
        for (int u = 0; u < 4; u++) part[u] = s + u <= last ? F::load(a.parts, F::kChalDtype, ((s + u) * 2) * a.width + c) : F::zero();
#pragma unroll
        for (int u = 0; u < 4; u++) v = F::add(v, part[u]);
    }
    if (scale) v = F::mul(v, multiplier);
    F::store(a.out, (uint64_t)key * a.out_width + c, v);
}

// Sums of the weights alone (one column).  Two kinds of blocks in one launch: the first `key_blocks` own 256 keys each,
// a thread per key, which adds the key's rows when they are few and writes the table's zeros; the others own a slice of
// the sorted order, and their warps add up the keys that have many.
constexpr uint32_t kKeySumThreads = 256, kKeySumFew = 8, kKeySumSlice = 512;
template <class F, bool W>
__global__ void __launch_bounds__(kKeySumThreads)
    key_sums_kernel(RowSumArgs a, uint64_t out_keys, uint32_t key_blocks, typename F::E multiplier, bool scale) {
    typedef typename F::E E;
    let_next_start();
    wait_for_previous();
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    auto first_at = [&](uint64_t lo, uint64_t hi, uint64_t key) {  // first place in [lo, hi) whose key is not below
        while (lo < hi) {
            const uint64_t mid = (lo + hi) >> 1;
            if (a.keys[mid] < key) lo = mid + 1;
            else hi = mid;
        }
        return lo;
    };
    if (blockIdx.x < key_blocks) {
        __shared__ uint64_t range[2];
        const uint64_t k0 = (uint64_t)blockIdx.x * kKeySumThreads, k = k0 + tid;
        if (warp < 2) {
            const uint64_t p = warp_first_at(a.keys, a.n, k0 + warp * kKeySumThreads);
            if (lane == 0) range[warp] = p;
        }
        __syncthreads();
        if (k >= out_keys) return;
        E v = F::zero();
        if (k < a.n_keys && range[0] < range[1]) {
            const uint64_t lo = first_at(range[0], range[1], k);
            uint32_t count = 0;
            uint32_t row[kKeySumFew];
            bool mine = lo < range[1];
#pragma unroll
            for (uint32_t j = 0; j < kKeySumFew; j++) {
                mine = mine && lo + j < range[1] && a.keys[lo + j] == k;
                row[j] = mine ? a.rows[lo + j] : 0xffffffffu;
                count += mine;
            }
            if (mine && lo + kKeySumFew < range[1] && a.keys[lo + kKeySumFew] == k) return;  // the slices' blocks write it
            if (W) {
                E w[kKeySumFew];  // all loads under way before the first sum
#pragma unroll
                for (uint32_t j = 0; j < kKeySumFew; j++) w[j] = row[j] != 0xffffffffu ? F::load(a.weights, F::kChalDtype, row[j]) : F::zero();
#pragma unroll
                for (uint32_t j = 0; j < kKeySumFew; j++)
                    if (j < count) v = F::add(v, w[j]);
            } else {
                v = F::from_u64(count);
            }
            if (scale && count) v = F::mul(v, multiplier);
        }
        F::store(a.out, k, v);
        return;
    }
    const uint64_t s = blockIdx.x - key_blocks, begin = s * a.slice, end = begin + a.slice < a.n ? begin + a.slice : a.n;
    __shared__ uint32_t n_long;
    __shared__ uint32_t starts[kKeySumSlice / (kKeySumFew + 1) + 2];  // runs of more than kKeySumFew rows in the slice
    if (tid == 0) n_long = 0;
    __syncthreads();
    for (uint64_t p = begin + tid; p < end; p += kKeySumThreads) {
        const uint32_t key = a.keys[p];
        if (p > begin && a.keys[p - 1] == key) continue;  // not where a run enters the slice
        bool is_long = p + kKeySumFew < a.n && a.keys[p + kKeySumFew] == key;
        if (!is_long && p == begin && begin > 0 && a.keys[begin - 1] == key) {
            // the tail of a run that entered before: its length decides
            uint64_t hi = p + 1, lo = p;
            while (hi < a.n && a.keys[hi] == key) hi++;                                  // at most kKeySumFew steps
            while (lo > 0 && hi - lo <= kKeySumFew && a.keys[lo - 1] == key) lo--;
            is_long = hi - lo > kKeySumFew;
        }
        if (is_long && key < a.n_keys) starts[atomicAdd(&n_long, 1u)] = (uint32_t)(p - begin);
    }
    __syncthreads();
    const uint32_t count = n_long;
    for (uint32_t r = warp; r < count; r += kKeySumThreads / 32) {
        const uint64_t p = begin + starts[r];
        const uint32_t key = a.keys[p];
        E v = F::zero();
        uint64_t rows = 0;
        for (uint64_t q0 = p; q0 < end; q0 += 128) {
            bool in[4];
            E w[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const uint64_t q = q0 + 32 * j + lane;
                in[j] = q < end && a.keys[q] == key;
                if (W) w[j] = in[j] ? F::load(a.weights, F::kChalDtype, a.rows[q]) : F::zero();
                rows += __popc(__ballot_sync(0xffffffffu, in[j]));
            }
            if (W) {
#pragma unroll
                for (int j = 0; j < 4; j++) v = F::add(v, w[j]);
            }
            if (!__shfl_sync(0xffffffffu, (int)in[3], 31)) break;  // the run ended
        }
        if (W) {
#pragma unroll
            for (int off = 16; off > 0; off >>= 1) v = F::add(v, F::shfl_down(v, off));
        } else {
            v = F::from_u64(rows);
        }
        if (lane == 0) {
            const bool before = p == begin && begin > 0 && a.keys[begin - 1] == key;
            const bool after = p + rows == end && end < a.n && a.keys[end] == key;
            if (before || after) {
                F::store(a.parts, s * 2 + (before ? 0 : 1), v);
            } else {
                if (scale) v = F::mul(v, multiplier);
                F::store(a.out, key, v);
            }
        }
    }
}

// As row_sums_join_kernel for one column: a warp per slice adds the following slices' parts lane by lane.
template <class F>
__global__ void __launch_bounds__(kKeySumThreads)
    key_sums_join_kernel(RowSumArgs a, uint64_t slices, typename F::E multiplier, bool scale) {
    typedef typename F::E E;
    wait_for_previous();
    const uint64_t s = ((uint64_t)blockIdx.x * kKeySumThreads + threadIdx.x) >> 5;
    const uint32_t lane = threadIdx.x & 31;
    if (s >= slices) return;
    const uint64_t begin = s * a.slice, end = begin + a.slice;
    if (end >= a.n) return;
    const uint32_t key = a.keys[end - 1];
    if (a.keys[end] != key || key >= a.n_keys || (begin > 0 && a.keys[begin - 1] == key)) return;
    // a run of few rows is the key blocks' own
    uint64_t lo = end - 1;
    while (lo > begin && lo + kKeySumFew >= end && a.keys[lo - 1] == key) lo--;
    if (!(lo + kKeySumFew < a.n && a.keys[lo + kKeySumFew] == key)) return;
    E v = lane == 0 ? F::load(a.parts, F::kChalDtype, s * 2 + 1) : F::zero();
    for (uint64_t t = s + 1 + lane; t * a.slice < a.n && a.keys[t * a.slice] == key; t += 32)
        v = F::add(v, F::load(a.parts, F::kChalDtype, t * 2));
    for (int off = 16; off > 0; off >>= 1) v = F::add(v, F::shfl_down(v, off));
    if (lane == 0) {
        if (scale) v = F::mul(v, multiplier);
        F::store(a.out, key, v);
    }
}

}  // namespace dpb
