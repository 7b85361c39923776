/*
 * moa_search.h -- C ABI of the choice of tokens from logits (same library, error codes and conventions as moa_ops.h):
 * the verification of drafted trees and the selection of beams, both over the rows that final_norm_and_logits writes.
 *
 * No counterpart in the reference, which copies one row of logits to the host and samples there
 * (FO/src/host/generate.rs:129-134). logits are bf16 [rows][vocab], rows logit_row_stride elements apart (at least
 * vocab); vocab may be any number up to 2^20, rows at most 65535. Results are deterministic. The calls share the paged
 * calls' scratch (moa_paged.h; the first call of either kind allocates its 100 MB): one stream at a time.
 */
#ifndef MOA_SEARCH_H
#define MOA_SEARCH_H

#include <stdint.h>

#include "moa_ops.h"

#ifdef __cplusplus
extern "C" {
#endif

/* The greedy verification of a batch's drafted trees (rows, row_starts and masks as in moa_paged_tree_attention,
 * moa_paged.h). best[row]: the token of the row's largest logit, ties to the lowest token; NaN counts as less than every
 * number. From node 0 of a sequence the walk goes to the lowest child of the node whose token (tokens, device int32
 * [rows]) is the node's best, as long as there is one: a child of x sees itself and the nodes that x sees. leaves[s]:
 * the node where it ends; next_tokens[s]: that node's best. Rows that belong to no sequence are left as they were; a
 * sequence without rows, or whose first row is no node, has leaf and token -1, and so has one whose rows are out of
 * range or more than 64 * mask_words (MOA_DEVERR_PAGED). rows may be 0: the leaves and tokens are then -1. */
int moa_tree_verify(const uint16_t* logits, int64_t logit_row_stride, const int32_t* tokens, const int32_t* row_starts,
                    const uint64_t* masks, int mask_words, int32_t* best, int32_t* leaves, int32_t* next_tokens, int rows,
                    int vocab, int sequences, void* stream);

/* A beam search's step: rows g * beams .. g * beams + beams - 1 (beams 1 to 64) are the beams of group g, with
 * scores[row] the sum of their tokens' log probabilities. A candidate is a beam and a token v, at score + logits[v] -
 * log sum_t e^logits[t]; a finished beam (finished[row] not 0) has the one candidate `eos` at its score, and its logits
 * are not read. The `beams` best of a group, ties to the lowest row and then the lowest token, become its rows in
 * descending order: out_scores, parents (the row that it comes from, as moa_paged_cache_reorder takes it), tokens, and
 * out_finished (1 where the parent is finished or the token is eos, else 0). Candidates at -infinity (a total that rounds
 * to it as a score among them) or NaN are none (so is every one of a row that holds a NaN or +infinity, or no finite
 * logit): a row that is left without one is finished, its own parent, at -infinity, with token max(eos, 0). eos: below
 * vocab, or -1 where no token ends a beam (then no beam may be finished: it has no candidate). out_scores may be scores and
 * out_finished may be finished. f32 arrays and int32 arrays are [groups * beams]. Sums and totals are f64, and the scores
 * are rounded once. Exponentials are f32: that of a logit d below its row's largest is off by at most (d + 6) 2^-22 of
 * itself (below 2^-126 it may be 0), the logarithm of their sum by less than 2^-17, so totals of two rows that lie closer
 * can change places; equal rows have equal sums. Where a row's totals are equal, since its score leaves no bit to its
 * logits, the larger logit comes first. groups may be 0. */
int moa_beam_select(const uint16_t* logits, int64_t logit_row_stride, const float* scores, const int32_t* finished,
                    float* out_scores, int32_t* out_finished, int32_t* parents, int32_t* tokens, int groups, int beams,
                    int vocab, int eos, void* stream);

#ifdef __cplusplus
}
#endif
#endif
