/*
 * Upkeep of the page pool on the device: copying pages through all layers, forking and freeing
 * sequences, compacting the pool.  No reference counterpart (its engine side plans on the host);
 * tables and page tensors are the reference's descriptors (kvx_abi.h:92-128).
 *
 * The plans run on device tables and never come back to the host: fork and compact leave the page
 * pairs to be copied in device arrays that kvx_launch_copy_pages reads in stream order.  State:
 *   block table  PACKED, [seq_count, max_blocks_per_seq]; a negative entry is no page
 *   seq_lens     cached tokens per row, same index type
 *   page_refs    S32 [num_blocks]: how many table entries name a page; 0 = free
 * All entry points enqueue on `stream`, synchronise nothing and allocate nothing; results do not
 * depend on timing.  Whole numbers wrap nowhere: counts stop at zero.
 */
#ifndef KVX_PAGES_OPS_H
#define KVX_PAGES_OPS_H

#include "kvx_abi.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Copies page src[i] to page dst[i], K and V, in every one of `cache_count` caches (the layers of a
 * model), bits unchanged, any dtype and layout.  src / dst: DEVICE arrays of `pair_count` page
 * numbers (S32 or S64).  Pairs all read the pages as they were before the call.  Bad data is
 * skipped: a pair takes no part when a number is negative or >= num_blocks, when both are equal,
 * when a later pair that is in range has the same destination, or when its source is the
 * destination of a pair in range.  Caches may differ in everything but num_blocks.
 *
 * `workspace`: DEVICE scratch of kvx_copy_pages_workspace_bytes(pair_count) bytes (0 for short
 * lists: NULL is fine), no initialisation, reusable in stream order.
 * Status: INVALID_ARGUMENT for NULL / undersized descriptors, differing num_blocks, scratch too
 * small; UNSUPPORTED for an unknown layout or dtype; OK without a launch when there is nothing. */
KVX_API size_t kvx_copy_pages_workspace_bytes(uint32_t pair_count);
KVX_API kvx_status_t kvx_launch_copy_pages(const kvx_cache_desc_t *caches, uint32_t cache_count, const void *src,
                                           const void *dst, kvx_dtype_t index_dtype, uint32_t pair_count,
                                           void *workspace, size_t workspace_bytes, void *stream);

/* Frees rows[0 .. row_count): every valid entry of the row gives one reference back (a count never
 * goes below zero), the entries become -1 and the length 0.  rows has the table's index type; a
 * number outside the table is skipped, a repeated one counts once. */
KVX_API kvx_status_t kvx_launch_free_sequences(const kvx_block_table_t *table, const kvx_seq_lens_t *seq_lens,
                                               int32_t *page_refs, uint32_t num_blocks, const void *rows,
                                               uint32_t row_count, void *stream);

/* Forks parents[i] into the row children[i], i < pair_count (same index type as the table).  Pages
 * that are full (block_size tokens) are shared and gain a reference; a page that is partly filled
 * is duplicated: the child gets a free page, in pair order the lowest free numbers, and
 * (copy_src[i], copy_dst[i]) tell kvx_launch_copy_pages what to copy (-1, -1 where there is
 * nothing).  Entries behind the sequence become -1; the child's length is the parent's.  What the
 * child row held is overwritten, not freed.
 * A pair is not forked, and gets (-2, -2) and an untouched child, when a row lies outside the
 * table, when parent and child are the same, when an earlier pair names the same child, when its
 * parent is a child of any pair, or when no page is left for its duplicate.  A partly filled page
 * that is not valid in the parent leaves -1 in the child, without a copy.
 * `workspace`: kvx_fork_workspace_bytes(pair_count) bytes of DEVICE scratch. */
KVX_API size_t kvx_fork_workspace_bytes(uint32_t pair_count);
KVX_API kvx_status_t kvx_launch_fork_sequences(const kvx_block_table_t *table, const kvx_seq_lens_t *seq_lens,
                                               int32_t *page_refs, uint32_t num_blocks, uint32_t block_size,
                                               const void *parents, const void *children, uint32_t pair_count,
                                               void *copy_src, void *copy_dst, void *workspace,
                                               size_t workspace_bytes, void *stream);

/* Moves the live pages (references above zero) to the front of the pool: with n live pages, the
 * k-th live page at or beyond n (in ascending order) moves to the k-th free page below n.  Table
 * entries and references follow; copy_src / copy_dst (num_blocks / 2 entries each, at least one,
 * the table's index type) list the moves, -1 behind the last.  Run kvx_launch_copy_pages on them
 * before anything reads the pages through the table.  Every entry of the table is renamed, used or
 * not; other tables that share the pool are not known here: lay all sequences of a pool out in one
 * table. */
KVX_API kvx_status_t kvx_launch_compact_pages(const kvx_block_table_t *table, int32_t *page_refs, uint32_t num_blocks,
                                              void *copy_src, void *copy_dst, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* KVX_PAGES_OPS_H */
