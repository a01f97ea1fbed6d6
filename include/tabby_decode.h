/*
 * tabby_decode.h -- C ABI of the B200 decode operators (libtabbydecode.so): the parts of a
 * decode step that carries several hypotheses a sequence.
 *
 *   beam search:    tabby_beam_step_async picks the next beams from the logits,
 *                   tabby_states_reorder_async moves the beams' states to follow them;
 *   drafted trees:  tabby_tree_attention_async attends a tree of drafted tokens over a
 *                   key/value cache, tabby_tree_accept_async keeps the path that the sampled
 *                   tokens (tabby_sample.h) agree with and closes the cache's gaps.
 *
 * Conventions: those of tabby_sample.h. Every function returns a tabby_status; on failure
 * tabby_decode_last_error() returns a message for the calling thread. Pointers named d_* (and
 * those of the argument structs) are device pointers, h_* host pointers; host arrays and
 * structs are read before the call returns. `device` is the CUDA device the pointers live on;
 * the caller's current device is left as it was. `stream` is a cudaStream_t of that device.
 * There are no handles and no state between calls: scratch memory comes from the caller,
 * holds anything before the call and is free again when the call's work on the stream is done,
 * so calls on several streams or in several captured graphs need a workspace each and nothing
 * else. Outputs must not overlap inputs except where a call works in place. Nothing here
 * aborts the process.
 */
#ifndef TABBY_DECODE_H
#define TABBY_DECODE_H

#include <stddef.h>
#include <stdint.h>

#include "tabby_sample.h"

#ifdef __cplusplus
extern "C" {
#endif

#define TABBY_DECODE_ABI_VERSION 1

typedef enum tabby_dtype { TABBY_F32 = 0, TABBY_BF16 = 1, TABBY_F16 = 2 } tabby_dtype;

TABBY_API int32_t tabby_decode_abi_version(void);

/* Thread-local message for the last failing call of this library on this thread. */
TABBY_API const char *tabby_decode_last_error(void);

/*
 * Beam search's selection. For prompt b, beam i with running log-probability
 * s = scores[b][i] and logits x[v], v < vocab:
 *   key(i, v) = s + x[v] - log(sum_u exp(x[u]))          (compared in 64 bits)
 * and the n_out continuations with the largest keys are written in falling order, ties to
 * the lower (beam, token); among one beam's continuations the logits themselves decide. Of
 * prompt b, output j:
 *   next_scores = key rounded to f32, parents = i, tokens = v,
 *   next_finished = 1 where beam i was finished or v == eos_id.
 * - A logit of -inf is a banned token: it is no candidate. Any finite logit is one.
 * - A beam whose score is -inf is dead: it has no candidates and its logits are not read.
 * - A finished beam (finished != 0) has one candidate, (eos_id, its score unchanged); its
 *   logits are not read.
 * - Where fewer than n_out candidates exist the rest is parents = tokens = -1,
 *   next_scores = -inf, next_finished = 1.
 * status[b] is TABBY_OK, or TABBY_EINPUT where a live beam's logits hold NaN or +inf or a
 * score is NaN or +inf; all n_out outputs of such a prompt are the "no candidate" values.
 * d_logits: dtype, element (b, i, v) at b * batch_stride + i * beam_stride + v (elements; the
 * strides may be 0 to share rows), aligned to its type. d_finished may be NULL (none is; then
 * eos_id may be -1: no end token); d_next_finished may be NULL.
 * Scores are exact to (3 ln(vocab) + 24) 2^-24 and their rounding to f32. Parents and tokens are
 * those of keys with log-sum-exps good to 3e-13 and the rounding of 64-bit sums: continuations of
 * different beams whose keys lie closer together than about 1e-12 may change places, unless the
 * beams' logits and scores are alike (then they tie).
 * 1 <= beams <= TABBY_BEAM_MAX, 1 <= n_out <= TABBY_BEAM_MAX_OUT, 1 <= vocab <= 2^30,
 * beams * vocab < 2^31; batch * beams * vocab below 2^42 or so (a launch's 2^31 blocks).
 * d_workspace: tabby_beam_workspace_bytes bytes, 16-byte aligned.
 */
#define TABBY_BEAM_MAX 64
#define TABBY_BEAM_MAX_OUT 128
TABBY_API int tabby_beam_workspace_bytes(int32_t batch, int32_t beams, int32_t vocab,
                                         int32_t n_out, size_t *bytes);
TABBY_API int tabby_beam_step_async(int32_t device, const void *d_logits, int32_t dtype,
                                    int64_t batch_stride, int64_t beam_stride, int32_t batch,
                                    int32_t beams, int32_t vocab, const float *d_scores,
                                    const uint8_t *d_finished, int32_t eos_id, int32_t n_out,
                                    float *d_next_scores, int32_t *d_parents,
                                    int32_t *d_tokens, uint8_t *d_next_finished,
                                    int32_t *d_status, void *d_workspace,
                                    size_t workspace_bytes, void *stream);

/*
 * How the rows of a state lie in memory, in bytes. Element e of entry t of segment g of row r
 * starts at r * row_stride + g * segment_stride + t * entry_stride; an entry is entry_bytes
 * contiguous bytes. A [rows][heads][tokens][dim] cache has heads as segments and tokens as
 * entries; a plain [rows][n] state has one segment with one entry. No two rows, segments or
 * entries may overlap.
 */
typedef struct tabby_state_layout {
  int64_t row_stride;
  int64_t segment_stride;
  int64_t entry_stride;
  int64_t entry_bytes;
  int32_t segments;
  int32_t entries;
} tabby_state_layout; /* 40 bytes */

/*
 * Moves the beams' states in place after a selection: for every state, prompt b and beam i,
 *   row b * beams + i  :=  what row b * beams + parents[b][i] held before the call,
 * in the first lengths[b] entries of every segment (all of them where d_lengths is NULL;
 * lengths are clipped to [0, entries]); later entries are left as they were. A row whose
 * parent is its own or lies outside [0, beams) is left as it was. h_states: n_states device
 * pointers, every state with the same layout, none overlapping another. With n_states == 0 the
 * other arguments are checked and nothing is done.
 * 1 <= beams <= TABBY_BEAM_MAX.
 */
TABBY_API int tabby_states_reorder_async(int32_t device, void *const *h_states,
                                         int32_t n_states, const tabby_state_layout *layout,
                                         int32_t batch, int32_t beams,
                                         const int32_t *d_parents, const int32_t *d_lengths,
                                         void *stream);

/*
 * A drafted tree, for the two calls below: parents[j] of slot j < nodes is the slot it
 * continues, -1 for a root, anything else below 0 for an unused slot. A slot whose way up
 * does not end in a root over ever lower slots is unused too, and so is one whose place in the
 * cache, lengths[b] + j, lies past the last entry. A sequence with lengths[b] < 0 is absent:
 * none of its slots is in use. 1 <= nodes <= TABBY_TREE_MAX_NODES.
 */
#define TABBY_TREE_MAX_NODES 64

/*
 * Attention of a drafted tree over a cache. Sequence b holds lengths[b] entries of context,
 * then, at entries lengths[b] + j, the keys and values of its tree's slots (written before the
 * call). Slot j in use attends to the whole context, to itself and to its ancestors:
 *   out[b][j][h] = sum_t p_t v[b][h'][t],  p = softmax over those t of scale * q[b][j][h].k[b][h'][t]
 * with h' = h / (heads / kv_heads). Scores, statistics and sums are in fp32; the weights (before
 * their division by the sum) are rounded to the type where they meet v, which takes 16-bit
 * operands, and out is rounded to it once. Both together put out off by about 2.2e-3 (bf16) or
 * 2.9e-4 (fp16) relative in the norm, where the rounding of out alone is 1.7e-3 and 2.1e-4.
 * Slots not in use give 0. One slot (nodes == 1) is the ordinary decode step. Keys and values
 * of the context and of the slots in use must be finite; what the cache holds elsewhere does
 * not matter. Element (b, h, t) of k starts at b * k_batch_stride + h * k_head_stride +
 * t * k_entry_stride (elements), its dim values contiguous; likewise v, q and out (b, j, h).
 * TABBY_BF16 or TABBY_F16; dim a multiple of 8 up to TABBY_TREE_MAX_DIM; heads a multiple of
 * kv_heads; pointers 16-byte aligned and strides multiples of 8 elements.
 * A cache's axis longer than one has a stride of its own (no shared sequences or heads).
 * parents_stride is the number of ints between the sequences' trees (0: one tree for all).
 * Should a device-side wait run out of its bound (0.5 s), the outputs it concerns are NaN, and so
 * are those that the same block of threads had still to compute.
 */
#define TABBY_TREE_MAX_DIM 128
typedef struct tabby_tree_attention_args {
  const void *q;
  const void *k;
  const void *v;
  void *out;
  int64_t q_batch_stride, q_node_stride, q_head_stride;
  int64_t k_batch_stride, k_head_stride, k_entry_stride;
  int64_t v_batch_stride, v_head_stride, v_entry_stride;
  int64_t out_batch_stride, out_node_stride, out_head_stride;
  const int32_t *lengths; /* [batch] */
  const int32_t *parents; /* [batch][nodes] */
  int64_t parents_stride;
  int32_t dtype;
  int32_t batch, nodes, heads, kv_heads, dim;
  int32_t entries; /* of the cache */
  float scale;
  void *workspace; /* tabby_tree_workspace_bytes bytes, 16-byte aligned */
  size_t workspace_bytes;
} tabby_tree_attention_args;
TABBY_API int tabby_tree_workspace_bytes(int32_t batch, int32_t nodes, int32_t heads,
                                         int32_t kv_heads, int32_t dim, size_t *bytes);
TABBY_API int tabby_tree_attention_async(int32_t device, const tabby_tree_attention_args *h_args,
                                         void *stream);

/*
 * Acceptance of a drafted tree. sampled[b][j] is the token the model gave after slot j (the
 * `id` of a tabby_sample_outcome, or any other choice; element (b, j) lies at b *
 * sampled_batch_stride + j * sampled_stride ints), tokens[b][j] the drafted token of slot j.
 * Slot 0 is the root: the sequence's last token, accepted already. From it the walk goes to
 * the lowest slot in use whose parent is the current one and whose token is the current one's
 * sampled token, until there is none. Of sequence b:
 *   counts        slots on the path, the root among them (0 where slot 0 is no root in use)
 *   path          those slots in order, then -1
 *   next_tokens   the sampled token of the last one: the next root (-1 where counts is 0)
 *   next_lengths  lengths + counts
 * and in every cache entry lengths[b] + r takes what entry lengths[b] + path[r] held, r <
 * counts, in place; all other entries are left as they were. The caches' rows are the
 * sequences; all have the one layout; n_caches may be 0 (then layout is NULL and no slot lies past the end).
 */
TABBY_API int tabby_tree_accept_async(int32_t device, const int32_t *d_sampled,
                                      int64_t sampled_batch_stride, int64_t sampled_stride,
                                      const int32_t *d_tokens, const int32_t *d_parents,
                                      int64_t parents_stride, int32_t batch, int32_t nodes,
                                      const int32_t *d_lengths, int32_t *d_path,
                                      int32_t *d_counts, int32_t *d_next_tokens,
                                      int32_t *d_next_lengths, void *const *h_caches,
                                      int32_t n_caches, const tabby_state_layout *layout,
                                      void *stream);

#ifdef __cplusplus
}
#endif
#endif /* TABBY_DECODE_H */
