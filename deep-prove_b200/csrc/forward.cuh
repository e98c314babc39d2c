// What the forward operators' translation units share: the check that a kernel makes of its input values and the host
// waits for, and the handle of rows sorted by key.
#pragma once
#include "common.cuh"

namespace dpb {
enum FwdError : unsigned int { kFwdKeyRange = 1, kFwdValueRange = 2 };

// How a kernel tells the host what it thinks of its input: the checking blocks or their findings into `words[0]`, the
// last of them (a ticket in words[1]) publishes {findings, sequence number} in mapped memory as one 8-byte store and
// clears the words for the next launch; a single checking block publishes at once.  The host polls the sequence number,
// which saves the wait for the kernel's end and for whatever was queued behind it.  Nothing else is published, so the
// store needs no fence: results are ordered by the stream.
struct FwdCheck {
    unsigned int* words;
    unsigned long long* status;  // mapped
    unsigned int seq;
};
}  // namespace dpb

struct dpb_row_groups {
    dpb_ctx* ctx = nullptr;
    uint64_t n = 0, n_keys = 0;
    // Keys on the device are checked there while the host goes on; the first call that uses the rows waits for the
    // findings, behind its own launches.
    mutable dpb::FwdCheck check = {};
    mutable int slot = -1;     // the check's place in the mapped page, -1 once its findings are known
    mutable bool bad = false;  // a key lies outside the range
    void* block = nullptr;
    uint32_t* keys = nullptr;     // the keys, ascending
    uint32_t* rows = nullptr;     // the row at each place of that order
    uint32_t* places = nullptr;   // the place of each row
    uint32_t* offsets = nullptr;  // first place of every key (n_keys + 1 entries); null beyond kGroupOffsets keys
};

namespace dpb {

constexpr uint32_t kGroupOffsets = 1024;  // what grouped products take; with the end, one tile of the counting sort's scan

// Called by every thread of each of the `blocks` checking blocks, once, after its checks; `found` is the thread's.
__device__ __forceinline__ void fwd_check_done(const FwdCheck& c, unsigned int found, unsigned int blocks) {
    const unsigned int all = (__syncthreads_or((int)(found & kFwdKeyRange)) ? kFwdKeyRange : 0u) |
                             (__syncthreads_or((int)(found & kFwdValueRange)) ? kFwdValueRange : 0u);
    if (threadIdx.x != 0) return;
    unsigned int verdict = all;
    if (blocks > 1) {
        if (all) {
            atomicOr(c.words, all);
            __threadfence();  // before the ticket; with nothing found there is nothing to order, and results need not land
        }
        if (atomicAdd(c.words + 1, 1u) != blocks - 1) return;
        verdict = atomicExch(c.words, 0u);
        c.words[1] = 0;
    }
    *(volatile unsigned long long*)c.status = ((unsigned long long)c.seq << 32) | verdict;
}

// A kernel launched with launch_early may start while the stream's previous kernel runs, once all of that kernel's
// blocks have called let_next_start (or ended); what that kernel, or any before it, writes may be read after
// wait_for_previous, which waits for its end.  Such a kernel marks no pointer to that data __restrict__ and reads it with
// no __ldg: loads of data that is constant for a whole kernel may be moved up past the wait.
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
template <class... Params, class... Args>
cudaError_t launch_early(cudaStream_t stream, dim3 blocks, uint32_t threads, size_t smem, void (*kernel)(Params...), Args... args) {
    cudaLaunchConfig_t c = {};
    c.gridDim = blocks;
    c.blockDim = dim3(threads);
    c.dynamicSmemBytes = smem;
    c.stream = stream;
    cudaLaunchAttribute at = {};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    c.attrs = &at;
    c.numAttrs = 1;
    return cudaLaunchKernelEx(&c, kernel, Params(args)...);
}

// Restores the caller's current device (the context's own may be another).
struct FwdDevice {
    int before = -1, own;
    cudaError_t err;
    explicit FwdDevice(const dpb_ctx* ctx) : own(ctx->device) {
        err = cudaGetDevice(&before);
        if (err == cudaSuccess && before != ctx->device) err = cudaSetDevice(ctx->device);
    }
    ~FwdDevice() {
        if (before >= 0 && before != own) cudaSetDevice(before);
    }
};

// What every forward call asks for before it does anything.  Inside a capture of the stream a check's findings would
// never come, and a replay would write into scratch memory that has been handed on since.
inline int fwd_ready(const dpb_ctx* ctx, const FwdDevice& dev) {
    DPB_CUDA(dev.err);
    cudaStreamCaptureStatus capture;
    DPB_CUDA(cudaStreamIsCapturing(ctx->stream, &capture));
    if (capture != cudaStreamCaptureStatusNone) return fail(DPB_ESTATE, "forward calls are made outside captures of the context's stream");
    return fwd_results_hold(ctx);
}

// The next check of the context (api_forward.cu).  With a
// slot (fwd_slot_take) the findings stay readable until the slot is given back; without one, until the next check.
int fwd_check_begin(dpb_ctx* ctx, FwdCheck* out, int slot = -1);
int fwd_slot_take(dpb_ctx* ctx);  // -1: none is free
// What the check of the rows' keys found, waiting for it if need be: DPB_EINVAL for a key outside the range.
int fwd_groups_verdict(const dpb_row_groups* g);
// Waits (bounded) for the check's findings.
int fwd_check_wait(dpb_ctx* ctx, const FwdCheck& c, unsigned int* found);
// The word in mapped memory a kernel that gives up waiting sets (device address).
unsigned int* fwd_gave_up_word(dpb_ctx* ctx);
// A host tensor's copy on the device (*owned, to be freed after the launches), or the device tensor itself.  The host
// buffer may be reused once the stream has passed the copy: fwd_check_wait behind it, or a synchronisation.
int fwd_tensor(dpb_ctx* ctx, const int64_t* src, int on_device, uint64_t numel, const int64_t** dev, void** owned);

inline uint64_t pow2_ceil(uint64_t x) { return 1ull << log2u(x); }

}  // namespace dpb
