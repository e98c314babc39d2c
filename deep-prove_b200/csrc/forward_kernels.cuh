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
    uint32_t check_blocks;  // blocks that check the tokens; 0: every block, and the products as well
    FwdCheck check;
};

constexpr uint32_t kLookupThreads = 256;

__device__ __forceinline__ int64_t lookup_scale(const LookupArgs& a, int64_t x) {
    return (int64_t)((uint64_t)x * (uint64_t)a.multiplier + (uint64_t)a.rounding) >> a.shift;
}
// whether x * m + r leaves 64 bits
__device__ __forceinline__ bool lookup_overflows(const LookupArgs& a, int64_t x) {
    const __int128 v = (__int128)x * a.multiplier + a.rounding;
    return v != (__int128)(int64_t)v;
}

// T: the table's integers; V: entries per step (1 or 16 bytes' worth on the narrower side)
template <class T, int V, bool CHECK>
__global__ void __launch_bounds__(kLookupThreads) embedding_lookup_kernel(LookupArgs a) {
    unsigned int found = 0;
    const uint64_t per_row = (a.out_width + V - 1) / V, total = a.out_rows * per_row;
    const uint64_t step = (uint64_t)gridDim.x * kLookupThreads;
    if (!CHECK && blockIdx.x < a.check_blocks) {
        // the checking blocks look at all tokens first, so that the host need not wait for the rows
        for (uint64_t i = (uint64_t)blockIdx.x * kLookupThreads + threadIdx.x; i < a.n; i += (uint64_t)a.check_blocks * kLookupThreads)
            if ((uint64_t)a.tokens[i] >= a.vocab) found = kFwdKeyRange;
        fwd_check_done(a.check, found, a.check_blocks);
    }
    for (uint64_t w = (uint64_t)blockIdx.x * kLookupThreads + threadIdx.x; w < total; w += step) {
        const uint64_t i = w / per_row, c = (w - i * per_row) * V;
        int64_t y[V];
#pragma unroll
        for (int v = 0; v < V; v++) y[v] = 0;
        if (i < a.n && c < a.width) {
            const uint64_t t = (uint64_t)a.tokens[i];
            if (t < a.vocab) {
                const T* row = (const T*)a.table + t * a.stride + c;
                T x[V];
                if constexpr (V * sizeof(T) == 16) {
                    *(int4*)x = __ldg((const int4*)row);
                } else {
#pragma unroll
                    for (int v = 0; v < V; v++) x[v] = __ldg(row + v);
                }
#pragma unroll
                for (int v = 0; v < V; v++) {
                    if (V > 1 && c + v >= a.width) break;  // between the width and the stride
                    y[v] = lookup_scale(a, (int64_t)x[v]);
                    if (CHECK && lookup_overflows(a, (int64_t)x[v])) found |= kFwdValueRange;
                }
            } else if (CHECK) {
                found |= kFwdKeyRange;
            }
        }
        int64_t* o = a.out + i * a.out_width + c;
        if constexpr (V == 1) {
            __stcs((long long*)o, (long long)y[0]);
        } else {
#pragma unroll
            for (int v = 0; v < V; v += 2) __stcs((longlong2*)(o + v), make_longlong2(y[v], y[v + 1]));
        }
    }
    if (CHECK) fwd_check_done(a.check, found, gridDim.x);
}

// ------------------------------------------------------------------------------------------------ rows by key
// Up to kSmallSort rows: one block sorts (key, row) in shared memory by a bitonic network, one launch in all.
constexpr uint32_t kSmallSort = 2048, kSmallSortThreads = 1024;
__global__ void __launch_bounds__(kSmallSortThreads)
    groups_small_kernel(const int64_t* __restrict__ keys, uint32_t n, uint32_t n_keys, uint32_t n_pow2, uint32_t* __restrict__ out_keys,
                        uint32_t* __restrict__ out_rows, uint32_t* __restrict__ offsets, FwdCheck check) {
    __shared__ unsigned long long v[kSmallSort];
    unsigned int found = 0;
    for (uint32_t i = threadIdx.x; i < n_pow2; i += kSmallSortThreads) {
        unsigned long long e = ~0ull;
        if (i < n) {
            const uint64_t k = (uint64_t)keys[i];
            if (k >= n_keys) found = kFwdKeyRange;
            e = ((unsigned long long)(k < n_keys ? (uint32_t)k : n_keys) << 32) | i;
        }
        v[i] = e;
    }
    fwd_check_done(check, found, 1);
    __syncthreads();
    for (uint32_t size = 2; size <= n_pow2; size <<= 1)
        for (uint32_t half = size >> 1; half > 0; half >>= 1) {
            for (uint32_t p = threadIdx.x; p < n_pow2 / 2; p += kSmallSortThreads) {
                const uint32_t i = 2 * p - (p & (half - 1)), j = i + half;
                const unsigned long long x = v[i], y = v[j];
                if ((x > y) == ((i & size) == 0)) {
                    v[i] = y;
                    v[j] = x;
                }
            }
            __syncthreads();
        }
    for (uint32_t i = threadIdx.x; i < n; i += kSmallSortThreads) {
        out_keys[i] = (uint32_t)(v[i] >> 32);
        out_rows[i] = (uint32_t)v[i];
    }
    if (offsets)
        for (uint32_t k = threadIdx.x; k <= n_keys; k += kSmallSortThreads) {
            uint32_t lo = 0, hi = n;
            while (lo < hi) {
                const uint32_t mid = (lo + hi) >> 1;
                if ((uint32_t)(v[mid] >> 32) < k) lo = mid + 1;
                else hi = mid;
            }
            offsets[k] = lo;
        }
}

// More rows: a counting sort.  rank[i] is the row's place inside its key; equal keys of a warp share one atomic.
__global__ void __launch_bounds__(kThreads)
    groups_count_kernel(const int64_t* __restrict__ keys, uint32_t n, uint32_t n_keys, uint32_t* __restrict__ counts,
                        uint32_t* __restrict__ rank, FwdCheck check) {
    unsigned int found = 0;
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
    groups_scan_kernel(uint32_t* __restrict__ counts, uint32_t n, uint32_t* __restrict__ tile_sums) {
    __shared__ uint32_t warp_sum[32];
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
    groups_scatter_kernel(const int64_t* __restrict__ keys, uint32_t n, uint32_t n_keys, const uint32_t* __restrict__ counts,
                          const uint32_t* __restrict__ tile_sums, uint32_t tiles, const uint32_t* __restrict__ rank,
                          uint32_t* __restrict__ out_keys, uint32_t* __restrict__ out_rows) {
    __shared__ uint32_t before[1056];
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
    uint64_t n;
    uint64_t slice;  // rows per slice
    const void* weights;
    const int64_t* x;
    uint64_t width;
    uint32_t per;  // routed rows per row of x
    uint64_t out_width;
    void* out;
    void* parts;  // [slice][2][width]
};

// An unreduced sum of (weight) * (integer) products, or of plain integers.
template <class F, bool W>
struct RowAccum;
template <>
struct RowAccum<FrFam, true> {
    FrIntAcc s;
    __device__ __forceinline__ void zero() { s = fr_intacc_zero(); }
    // w: the weight and its negative, 8 words each
    __device__ __forceinline__ void mac(const Fr* w, int64_t x) {
        const uint64_t mag = x < 0 ? (uint64_t)0 - (uint64_t)x : (uint64_t)x;
        frw::intacc_mac(s.a, frw::from_fr(w[x < 0]), mag);
    }
    __device__ __forceinline__ Fr finish() const { return fr_intacc_finish(s); }
};
template <>
struct RowAccum<GlFam, true> {
    glw::A8 s0, s1;
    __device__ __forceinline__ void zero() { s0 = s1 = glw::acc_zero(); }
    __device__ __forceinline__ void mac(const Gl2* w, int64_t x) {
        const uint64_t mag = x < 0 ? (uint64_t)0 - (uint64_t)x : (uint64_t)x;
        const glw::W2 ww = gl2_words(w[x < 0]);
        const glw::W m = glw::make_w((uint32_t)mag, (uint32_t)(mag >> 32));
        glw::acc_mac(s0, m, ww.c0);
        glw::acc_mac(s1, m, ww.c1);
    }
    __device__ __forceinline__ Gl2 finish() const {
        return gl2_make(glw::to_u64(glw::canon(glw::acc_reduce(s0))), glw::to_u64(glw::canon(glw::acc_reduce(s1))));
    }
};
template <class F>
__device__ __forceinline__ typename F::E field_from_i128(__int128 v) {
    const bool neg = v < 0;
    const unsigned __int128 m = neg ? (unsigned __int128)0 - (unsigned __int128)v : (unsigned __int128)v;
    typename F::E r = F::from_u64((uint64_t)m);
    if ((uint64_t)(m >> 64)) r = F::add(r, F::mul(F::from_u64((uint64_t)(m >> 64)), F::from_u64_pow64()));
    return neg ? F::neg(r) : r;
}
template <class F>
struct RowAccum<F, false> {
    __int128 s;
    __device__ __forceinline__ void zero() { s = 0; }
    __device__ __forceinline__ void mac(const typename F::E*, int64_t x) { s += x; }
    __device__ __forceinline__ typename F::E finish() const { return field_from_i128<F>(s); }
};

constexpr uint32_t kRowSumThreads = 128, kRowSumBatch = 64, kRowSumFlight = 8;

template <class F, bool W>
__global__ void __launch_bounds__(kRowSumThreads)
    row_sums_kernel(RowSumArgs a, typename F::E multiplier, bool scale) {
    typedef typename F::E E;
    __shared__ E wsh[W ? kRowSumBatch : 1][2];
    __shared__ uint64_t at[kRowSumBatch];
    __shared__ uint32_t ends[kRowSumBatch];  // key + 1 where the key's run ends here, else 0
    const uint64_t c = (uint64_t)blockIdx.x * kRowSumThreads + threadIdx.x;
    const uint64_t begin = blockIdx.y * a.slice, end = begin + a.slice < a.n ? begin + a.slice : a.n;
    const bool live = c < a.width;
    bool before = begin > 0 && a.keys[begin - 1] == a.keys[begin];  // the current run began before the slice
    RowAccum<F, W> acc;
    acc.zero();
    for (uint64_t p0 = begin; p0 < end; p0 += kRowSumBatch) {
        const uint32_t m = end - p0 < kRowSumBatch ? (uint32_t)(end - p0) : kRowSumBatch;
        __syncthreads();
        if (threadIdx.x < kRowSumBatch) {
            const uint32_t i = threadIdx.x < m ? threadIdx.x : m - 1;
            const uint64_t p = p0 + i;
            const uint32_t row = a.rows[p], key = a.keys[p];
            at[threadIdx.x] = (uint64_t)(row / a.per) * a.width;
            ends[threadIdx.x] = threadIdx.x < m && (p + 1 == end || a.keys[p + 1] != key) ? key + 1 : 0;
            if (W) {
                const E w = F::load(a.weights, F::kChalDtype, row);
                wsh[threadIdx.x][0] = w;
                wsh[threadIdx.x][1] = F::neg(w);
            }
        }
        __syncthreads();
        for (uint32_t i0 = 0; i0 < m; i0 += kRowSumFlight) {
            int64_t x[kRowSumFlight];
#pragma unroll
            for (uint32_t u = 0; u < kRowSumFlight; u++) x[u] = live && i0 + u < m ? __ldg(a.x + at[i0 + u] + c) : 0;
#pragma unroll
            for (uint32_t u = 0; u < kRowSumFlight; u++) {
                if (i0 + u >= m) break;
                acc.mac(wsh[W ? i0 + u : 0], x[u]);
                if (ends[i0 + u]) {
                    const uint32_t key = ends[i0 + u] - 1;
                    const uint64_t p = p0 + i0 + u;
                    const bool after = p + 1 == end && end < a.n && a.keys[end] == key;
                    if (live) {
                        E v = acc.finish();
                        if (before || after) {
                            F::store(a.parts, (blockIdx.y * 2 + (before ? 0 : 1)) * a.width + c, v);
                        } else {
                            if (scale) v = F::mul(v, multiplier);
                            F::store(a.out, (uint64_t)key * a.out_width + c, v);
                        }
                    }
                    acc.zero();
                    before = false;
                }
            }
        }
    }
}

// Adds up the keys that span slices: block row y looks at slice y, and acts when a key begins there and goes on.
template <class F>
__global__ void __launch_bounds__(kRowSumThreads)
    row_sums_join_kernel(RowSumArgs a, typename F::E multiplier, bool scale) {
    typedef typename F::E E;
    const uint64_t begin = blockIdx.y * a.slice, end = begin + a.slice;
    if (end >= a.n) return;
    const uint32_t key = a.keys[end - 1];
    if (a.keys[end] != key) return;                                                // nothing goes on
    if (begin > 0 && a.keys[begin - 1] == key) return;                             // it began before
    const uint64_t c = (uint64_t)blockIdx.x * kRowSumThreads + threadIdx.x;
    if (c >= a.width) return;
    E v = F::load(a.parts, F::kChalDtype, (blockIdx.y * 2 + 1) * a.width + c);
    for (uint64_t s = blockIdx.y + 1; s * a.slice < a.n && a.keys[s * a.slice] == key; s++)
        v = F::add(v, F::load(a.parts, F::kChalDtype, (s * 2) * a.width + c));
    if (scale) v = F::mul(v, multiplier);
    F::store(a.out, (uint64_t)key * a.out_width + c, v);
}

// Sums of the weights alone (one column).  Two kinds of blocks in one launch: the first `key_blocks` own 256 keys each,
// a thread per key, which adds the key's rows when they are few and writes the table's zeros; the others own a slice of
// the sorted order and add up, with all their threads, the keys that have many.
constexpr uint32_t kKeySumThreads = 256, kKeySumFew = 16;
template <class F, bool W>
__global__ void __launch_bounds__(kKeySumThreads)
    key_sums_kernel(RowSumArgs a, uint64_t n_keys, uint64_t out_keys, uint32_t key_blocks, typename F::E multiplier, bool scale) {
    typedef typename F::E E;
    const uint32_t tid = threadIdx.x;
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
        if (tid < 2) range[tid] = first_at(0, a.n, k0 + tid * kKeySumThreads);
        __syncthreads();
        if (k >= out_keys) return;
        E v = F::zero();
        if (k < n_keys && range[0] < range[1]) {
            const uint64_t lo = first_at(range[0], range[1], k), hi = first_at(lo, range[1], k + 1);
            if (hi - lo > kKeySumFew) return;  // the slices' blocks write it
            if (W) {
                for (uint64_t p = lo; p < hi; p++) v = F::add(v, F::load(a.weights, F::kChalDtype, a.rows[p]));
            } else {
                v = F::from_u64(hi - lo);
            }
            if (scale) v = F::mul(v, multiplier);
        }
        F::store(a.out, k, v);
        return;
    }
    const uint64_t s = blockIdx.x - key_blocks, begin = s * a.slice, end = begin + a.slice < a.n ? begin + a.slice : a.n;
    __shared__ uint32_t n_long;
    __shared__ uint64_t starts[64];  // runs of more than kKeySumFew rows that touch the slice: at most slice / 16 + 2
    if (tid == 0) n_long = 0;
    __syncthreads();
    for (uint64_t p = begin + tid; p < end; p += kKeySumThreads) {
        const uint32_t key = a.keys[p];
        if (p > begin && a.keys[p - 1] == key) continue;  // not where a run enters the slice
        bool is_long = p + kKeySumFew < a.n && a.keys[p + kKeySumFew] == key;
        if (!is_long && p == begin && begin > 0 && a.keys[begin - 1] == key) {
            const uint64_t lo = first_at(0, begin, key), hi = first_at(begin, a.n, (uint64_t)key + 1);
            is_long = hi - lo > kKeySumFew;
        }
        if (is_long) starts[atomicAdd(&n_long, 1u)] = p;
    }
    __syncthreads();
    const uint32_t count = n_long;
    for (uint32_t r = 0; r < count; r++) {
        const uint64_t p = starts[r];
        const uint32_t key = a.keys[p];
        uint64_t hi = end;
        if (a.keys[end - 1] != key) hi = first_at(p, end, (uint64_t)key + 1);
        E acc[1] = {F::zero()};
        if (W) {
            for (uint64_t q = p + tid; q < hi; q += kKeySumThreads) acc[0] = F::add(acc[0], F::load(a.weights, F::kChalDtype, a.rows[q]));
            block_sum<F, 1>(acc);
        }
        if (tid == 0) {
            E v = W ? acc[0] : F::from_u64(hi - p);
            const bool before = p == begin && begin > 0 && a.keys[begin - 1] == key;
            const bool after = hi == end && end < a.n && a.keys[end] == key;
            if (before || after) {
                F::store(a.parts, s * 2 + (before ? 0 : 1), v);
            } else {
                if (scale) v = F::mul(v, multiplier);
                F::store(a.out, key, v);
            }
        }
        __syncthreads();
    }
}

// As row_sums_join_kernel for one column: a warp per slice adds the following slices' parts lane by lane.
template <class F>
__global__ void __launch_bounds__(kKeySumThreads)
    key_sums_join_kernel(RowSumArgs a, uint64_t slices, typename F::E multiplier, bool scale) {
    typedef typename F::E E;
    const uint64_t s = ((uint64_t)blockIdx.x * kKeySumThreads + threadIdx.x) >> 5;
    const uint32_t lane = threadIdx.x & 31;
    if (s >= slices) return;
    const uint64_t begin = s * a.slice, end = begin + a.slice;
    if (end >= a.n) return;
    const uint32_t key = a.keys[end - 1];
    if (a.keys[end] != key || (begin > 0 && a.keys[begin - 1] == key)) return;
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
