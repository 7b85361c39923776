/*
 * moa_paged.h -- C ABI of the paged KV cache: many sequences over one pool of pages, and the
 * attention that reads it (same library, error codes and conventions as moa_ops.h).
 *
 * No counterpart in the reference, whose runtime serves one sequence (a 1024-slot ring per sliding
 * layer, 512-slot pages per full-attention layer, FO/src/host/runtime.rs:401-530). The cache's head
 * layouts include both of its layer kinds: a page is what sliding_project_qkv's ring holds per slot
 * (8 KV heads of 256), or a full-attention layer's page (one KV head of 512).
 *
 * The cache is caller-owned device memory described by a moa_paged_cache (a host struct that the
 * caller keeps; a call reads it before it returns). Its state -- page table, lengths, reference
 * counts -- lives on the device, and every call that changes it runs there: nothing synchronises,
 * and the calls can be captured into a HIP graph (call moa_init before). The first call on a device
 * allocates the paged calls' scratch (100 MB), also while a stream is captured.
 *   - sequence s holds positions 0 .. seq_lens[s] - 1; position t lies in page
 *     page_table[s][t / slots] at slot t % slots. Table entries behind the last page in use are
 *     never read as pages.
 *   - ref_counts[p] is the number of table entries in use that name page p; 0 is a free page.
 * A call finds a bad device-resident argument on the device: it then leaves out what that argument
 * covers (each call says what), never reads or writes outside the arrays, and raises
 * MOA_DEVERR_PAGED, read back by moa_device_errors().
 */
#ifndef MOA_PAGED_H
#define MOA_PAGED_H

#include <stdint.h>

#include "moa_ops.h"

#ifdef __cplusplus
extern "C" {
#endif

#define MOA_DEVERR_PAGED 8u /* a bad device-resident argument of a paged-cache call */

#define MOA_PAGES_BF16 0 /* K and V as bf16 */
#define MOA_PAGES_E4M3 1 /* K and V as E4M3FN codes, a value is code * scale[layer][head] */

typedef struct moa_paged_cache {
    void* k_pages;        /* [layers][pages][slots][kv_heads][head_dim], strides below, 16-byte aligned */
    void* v_pages;        /* the same shape */
    const float* k_scale; /* E4M3: f32 [layers][kv_heads], positive; bf16: NULL */
    const float* v_scale;
    int32_t* page_table;  /* [sequences][columns], rows table_stride apart */
    int32_t* seq_lens;    /* [sequences] */
    int32_t* ref_counts;  /* [pages] */
    int64_t k_stride[4];  /* in elements: layer, page, slot, head; multiples of 16 bytes */
    int64_t v_stride[4];
    int64_t table_stride; /* in entries */
    int32_t layers;       /* 1 .. 1024 */
    int32_t pages;        /* 1 .. 2^20 */
    int32_t slots;        /* positions per page, 1 .. 65536 */
    int32_t kv_heads;     /* 1 .. 256 */
    int32_t head_dim;     /* 64, 128, 256 or 512 */
    int32_t element;      /* MOA_PAGES_BF16 or MOA_PAGES_E4M3 */
    int32_t sequences;    /* 1 .. 65536 */
    int32_t columns;      /* pages a sequence can have; columns * slots <= 2^30 */
} moa_paged_cache;

/* Grows sequence s by new_tokens[s] positions (device int32 [sequences], 0 or more): the new pages
 * are the lowest-numbered free ones, handed out in the order of the sequences and of their pages,
 * with reference count 1. Their slots keep what they held. All or nothing: a negative number, a
 * length past columns * slots or too few free pages leave the state as it was (MOA_DEVERR_PAGED). */
int moa_paged_cache_reserve(const moa_paged_cache* cache, const int32_t* new_tokens, void* stream);

/* Writes the K and V rows of a step's new tokens of one layer. Rows row_starts[s] ..
 * row_starts[s + 1] - 1 (device int32 [sequences + 1], ascending) are sequence s's last positions:
 * row i of n goes to position seq_lens[s] - n + i. k, v bf16 [rows][kv_heads][head_dim] (heads and dims
 * dense, rows k_row_stride / v_row_stride elements apart, 16-byte aligned). E4M3 pages take the
 * nearest code of x / scale, ties to even, at most +-448. Rows before row_starts[0] or from
 * row_starts[sequences] on belong to no sequence and are not read. A row whose position or page is out of
 * range, or whose sequence's starts descend, is not written (MOA_DEVERR_PAGED). rows may be 0. */
int moa_paged_cache_append(const moa_paged_cache* cache, const uint16_t* k, int64_t k_row_stride, const uint16_t* v,
                           int64_t v_row_stride, const int32_t* row_starts, int rows, int layer, void* stream);

/* Makes sequence children[i] a copy of parents[i] (device int32 [count]) in every layer: it shares the
 * parent's full pages (reference count + 1) and gets a copy of its partly filled last page in the
 * lowest free page, handed out in the order of the list. A parent may be listed many times; append
 * its reserved positions first, since an append to a shared page is seen by all that share it. All or
 * nothing: an index out of range, a child that is listed twice, that is also a parent or that has
 * positions, a parent whose length or whose pages are out of range, or too few free pages leave the state as it was
 * (MOA_DEVERR_PAGED). count may be 0. */
int moa_paged_cache_fork(const moa_paged_cache* cache, const int32_t* parents, const int32_t* children, int count,
                         void* stream);

/* Ends the listed sequences (device int32 [count]): length 0, and one reference fewer on each of their
 * pages. A sequence that is empty or listed again changes nothing; an index out of range and a sequence whose length is out of
 * range are left out, and so is a table entry outside the pool or a page whose count is zero (MOA_DEVERR_PAGED). count may be 0. */
int moa_paged_cache_free(const moa_paged_cache* cache, const int32_t* sequences, int count, void* stream);

/* Moves the live pages (reference count > 0; n of them) to pages 0 .. n - 1: those at n and beyond go,
 * in ascending order, to the free pages below n, in ascending order, in every layer. The page table
 * and the reference counts follow. A length out of range leaves the state as it was; a table entry outside the pool is
 * left as it is (MOA_DEVERR_PAGED for both, for an entry only where some page moves). */
int moa_paged_cache_compact(const moa_paged_cache* cache, void* stream);

/* Attention of a batch's new rows over one layer of the cache, their own positions included (append
 * them first). Rows and sequences as in moa_paged_cache_append: row i of a sequence's n stands at
 * position p = seq_lens[s] - n + i and sees positions 0 .. p, the last `window` of them if window > 0.
 * out[row][h] = sum over them of softmax(scale * (q[row][h] . k_t)) v_t, head h reading KV head
 * h / (q_heads / kv_heads); a row that sees nothing (p < 0) gives zeros.
 * q, out bf16 [rows][q_heads][head_dim] (heads and dims dense, rows q_row_stride / out_row_stride elements
 * apart, multiples of 8; 16-byte aligned; out may be q). q_heads a multiple of kv_heads, at most 128
 * query heads per KV head. max_rows: the most rows a sequence has in this call (it chooses the kernel
 * and its grid; rows itself is always right). Rows that belong to no sequence are left as they were.
 * A sequence whose rows or length are out of range, or that has more than max_rows rows, is left out; so
 * is at least every row that sees a page outside the pool, and row starts that descend may leave out all; rows
 * that two sequences claim by such starts get either's result (MOA_DEVERR_PAGED for each). The entries of the
 * positions before a window have to name pages of the pool too: tiles begin up to 63 positions before it.
 * The result is deterministic; how the positions are split, and with it the order of f32 sums, follows the
 * whole batch, so a row's last bits may differ between calls of other batches. Scores, maxima, sums and outputs
 * are f32; a weight enters the product with V as two bf16 numbers, which hold it to 2^-16 of itself, in every row
 * of every call; the result is rounded once. rows may be 0. */
int moa_paged_attention(const uint16_t* q, int64_t q_row_stride, const moa_paged_cache* cache,
                        const int32_t* row_starts, uint16_t* out, int64_t out_row_stride, int rows, int q_heads,
                        int layer, int window, float scale, int max_rows, void* stream);

/* Drafted trees. A step of speculative decoding appends a tree of drafted tokens to a sequence as its last n positions,
 * n at most 256: node i of sequence s is row row_starts[s] + i of the call and position seq_lens[s] - n + i. masks
 * (device uint64 [rows][mask_words], 1 to 4 words) says what a node sees: bit j % 64 of word j / 64 of a node's row
 * stands for node j of the same sequence, the node itself and its ancestors in a tree (any set is allowed; bits from n
 * on are ignored). A row without bits is no node. A node's depth is the number of nodes that it sees, so it stands depth
 * - 1 positions behind the first node; a node without ancestors stands at position seq_lens[s] - n. */

/* Attention of the nodes: node i sees the positions before the tree (with a window, those less than `window` before its
 * own place as above) and the nodes of its mask. Everything else is as in moa_paged_attention, whose last bits a chain's
 * rows need not have. A row without bits gives zeros; nodes that would stand before position 0 are not there. Sequences
 * without a tree take part with trees of one node. max_rows is at most 64 * mask_words (the lesser of that and rows is
 * always right); window is 0 or at least max_rows. */
int moa_paged_tree_attention(const uint16_t* q, int64_t q_row_stride, const moa_paged_cache* cache,
                             const int32_t* row_starts, const uint64_t* masks, int mask_words, uint16_t* out,
                             int64_t out_row_stride, int rows, int q_heads, int layer, int window, float scale, int max_rows,
                             void* stream);

/* Ends a speculative step: of each sequence that has rows, the nodes that node leaves[s] (device int32 [sequences]) sees
 * become, in ascending order and in every layer, the positions behind those before the tree; the sequence ends behind
 * them, and pages that it no longer reaches are free. -1 keeps no node. Positions behind the new length keep what they
 * held or were moved from. A sequence whose rows, length or leaf are out of range, that is shorter than its rows, or one
 * of whose nodes lies in a page outside the pool or in one with a reference count other than 1, stays as it was
 * (MOA_DEVERR_PAGED). rows may be 0. */
int moa_paged_tree_commit(const moa_paged_cache* cache, const int32_t* row_starts, const uint64_t* masks, int mask_words,
                          const int32_t* leaves, int rows, void* stream);

/* A beam search's step back: sequences 0 .. count - 1 are groups of `beams` (1 to 64; count a multiple of it), and every
 * sequence s of them becomes what parents[s] (device int32 [count], a sequence of its group) was before the call, in
 * every layer. Full pages are shared, reference counts follow. A partly filled last page stays with its parent, if that
 * is its own child, else with the parent's first child; the other children get copies of the slots in use: in ascending
 * order, in the partly filled last pages of the sequences that are nobody's parent (where their reference count is 1),
 * in ascending order, then in the lowest free pages. Pages that no sequence names any more are free. All or nothing: a
 * parent outside the group, a length out of range, a page to copy outside the pool or too few free pages leave the state
 * as it was; another table entry outside the pool moves with its row and is not counted (MOA_DEVERR_PAGED for all).
 * count may be 0. */
int moa_paged_cache_reorder(const moa_paged_cache* cache, const int32_t* parents, int count, int beams, void* stream);

#ifdef __cplusplus
}
#endif
#endif
