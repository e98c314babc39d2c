/*
 * dpb_forward — forward operators of quantised models and their transposes.
 *
 * The provers of dpb.h and dpb_prover.h take integer tensors that are already on the device (dpb_einsum_fix_axes,
 * dpb_einsum_prove, dpb_lookup_witness with tensor_on_device); the operators below make such tensors there, and the
 * tables their sumchecks need:
 *   - embedding rows of a token list with a fixed-point scale, and the transposed lookup (sums of rows by token), which
 *     turns a claim about the embeddings at a row point into the table the embedding sumcheck multiplies with
 *     (zkml/src/layers/transformer/embeddings.rs:395-445);
 *   - integer matrix products grouped by expert (a routed feed-forward layer), and the same sums of rows with experts as
 *     keys, which bind the routed rows of such a product to a row point.
 * Everything is exact: integers, or field elements in the layouts of dpb.h.
 *
 * Conventions are those of dpb.h.  Work is queued on the context's stream (dpb_stream); device inputs must be ready on
 * that stream and stay as they are until it has passed the call, and results are ready on it.  Calls that check values
 * on the device wait for that check before they return; their results may still be in the making.  None of the calls
 * can be made while the context's stream is being captured (DPB_ESTATE, and the capture goes on).  Waits inside kernels are bounded.  When one runs out, the result is not valid, which may
 * show after the call has returned: from then on the calls here, and every call that hands values to the host
 * (dpb_mle_to_host, evaluations, sumcheck rounds and the provers, logup outputs, counters, commitments), fail with
 * DPB_ETIMEOUT until dpb_sync has reported it; what was made from results older than that is to be made again.
 */
#ifndef DPB_FORWARD_H
#define DPB_FORWARD_H

#include "dpb.h"

#ifdef __cplusplus
extern "C" {
#endif

/* out[i, c] = (table[tokens[i], c] * multiplier + r) >> right_shift,  r = 2^(right_shift - 1), or 0 without a shift:
 * the rows of n tokens, rescaled the way dpb_lookup_witness rescales (the shift rounds towards minus infinity).
 * `table` is an integer table (DPB_*_I32 / DPB_*_I64) of vocab rows, row_stride >= width entries apart (the padded
 * matrix a sumcheck takes has the padded width as its stride).  `tokens`: int64 ids, on the host or
 * (tokens_on_device != 0) on the device; n = 0 is allowed and gives no entries.
 * The result has the I64 layout of the table's family: with padded = 0 the n x width row-major tensor that the calls
 * with tensor_on_device take (n * width entries; as a table it is refused unless that is a power of two), with
 * padded != 0 a table of 2^ceil(log2 n) rows of 2^ceil(log2 width) entries, zero outside (n = 0: one zero row).
 * right_shift <= 62.  DPB_EINVAL, and no result, when a token lies outside 0..vocab-1 or a rescaled value does not fit
 * 64 bits before the shift. */
int dpb_embedding_lookup(dpb_ctx* ctx, const dpb_mle* table, uint64_t vocab, uint64_t width, uint64_t row_stride,
                         const int64_t* tokens, int tokens_on_device, uint64_t n, int64_t multiplier,
                         uint32_t right_shift, int padded, dpb_mle** out);

/* n rows sorted by key (token ids, or the expert of every routed row): made once per key list, used by any number of
 * the calls below.  Keys are int64 in 0..n_keys-1; 1 <= n_keys <= 2^22, n < 2^31 (0 allowed).  Results do not depend
 * on the order of the rows inside a key.  DPB_EINVAL when a key lies outside the range: from this call for keys on the
 * host, from the first call that uses the rows (and every later one) for keys on the device, which are checked there
 * while the host goes on (or from this call, when 64 handles' checks are waiting to be asked for). */
typedef struct dpb_row_groups dpb_row_groups;
int dpb_row_groups_new(dpb_ctx* ctx, const int64_t* keys, int keys_on_device, uint64_t n, uint64_t n_keys,
                       dpb_row_groups** out);
uint64_t dpb_row_groups_len(const dpb_row_groups* groups);
void dpb_row_groups_free(dpb_row_groups* groups);

/* out[k, c] = multiplier * sum over rows i with key k of weights[i] * rows[i / rows_per_token, c]
 * as field elements of the family (DPB_GL_EXT or DPB_FR): the transpose of dpb_embedding_lookup (keys = tokens), and
 * the binding of a grouped product's rows (keys = experts, rows_per_token = experts per token).
 * `weights`: a table of at least n challenge elements (an eq table of the row point, its entries past n unused) or
 * NULL for ones.  `rows`: an int64 row-major tensor of ceil(n / rows_per_token) x width entries, on the host or on the device, or NULL
 * for ones (width must be 1 then, and the sums are the weights' sums, or the number of rows).
 * The result is a table of 2^ceil(log2 n_keys) rows of 2^ceil(log2 width) entries (2^36 entries at most, of rows that
 * hold 2^40 at most), zero for keys without rows and outside; its low variables are the columns. */
int dpb_row_groups_sum(dpb_ctx* ctx, const dpb_row_groups* groups, int family_dtype, const dpb_mle* weights,
                       const int64_t* rows, int rows_on_device, uint64_t width, uint32_t rows_per_token,
                       int64_t multiplier, dpb_mle** out);

/* The weights of n_experts matrices of inner x cols entries ([expert, in, out], row-major int64, on the host or on the
 * device), laid out once for dpb_grouped_product: every value is cut into signed 8-bit digits (one for bits <= 8, else
 * two).  Values must lie in -2^(bits-1) .. 2^(bits-1)-1, 2 <= bits <= 15 (DPB_EINVAL otherwise); 1..1024 experts.
 * Takes 1 or 2 bytes per entry (inner and cols rounded up to 128). */
typedef struct dpb_expert_weights dpb_expert_weights;
int dpb_expert_weights_new(dpb_ctx* ctx, const int64_t* weights, int on_device, uint32_t n_experts, uint64_t inner,
                           uint64_t cols, uint32_t bits, dpb_expert_weights** out);
void dpb_expert_weights_free(dpb_expert_weights* weights);

/* out[i, :] = x[i / rows_per_token, :] * W[key of row i], exact in 64 bits: the products of routed rows with their
 * expert's matrix.  `groups` holds the expert of every routed row (its n_keys = the weights' n_experts); `x` is an
 * int64 row-major tensor of n / rows_per_token rows of `inner` entries, on the host or on the device, with values in
 * -2^(x_bits-1) .. 2^(x_bits-1)-1, 2 <= x_bits <= 15 (DPB_EINVAL otherwise); n is a multiple of rows_per_token.
 * The result is the n x cols tensor (padded = 0 form of dpb_embedding_lookup) in the I64 layout of family_dtype's
 * family, rows in the order of the key list. */
int dpb_grouped_product(dpb_ctx* ctx, int family_dtype, const dpb_row_groups* groups, const int64_t* x, int x_on_device,
                        uint32_t x_bits, uint32_t rows_per_token, const dpb_expert_weights* weights, dpb_mle** out);

#ifdef __cplusplus
}
#endif
#endif /* DPB_FORWARD_H */
