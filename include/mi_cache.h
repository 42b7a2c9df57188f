/*
 * C ABI of libmi_cache.so: operations on the blocks of a paged KV cache on MI355X (gfx950), and
 * attention over blocks that several rows of a batch share.
 *
 * The reference's cache (kv_cache.py:8-121) gives every sequence blocks of its own, so a history that
 * several conversations continue is prefilled, held and read once for each.  With these a sequence
 * can be forked (its whole blocks shared, the started one copied), blocks can be copied into another
 * cache or moved together, and a step reads the shared blocks once for all rows that hold them.
 *
 * Common rules.  A pool is `planes` planes (a K or V buffer of one layer each) `plane_bytes` apart; block
 * b of a plane is the `block_bytes` contiguous bytes from b * block_bytes on.  Pointers are device
 * pointers; all launches are asynchronous on `stream`, allocate nothing and may be captured in a
 * graph.  Ids read on the device that lie outside their range are skipped: nothing is read or written
 * for them.
 *
 * Status codes as in mi_fa2.h: 0 ok, 1 invalid argument, 2 unsupported, 3 workspace too small,
 * 4 launch failed; mi_cache_last_error() gives the calling thread's last message.
 */
#ifndef MI_CACHE_H
#define MI_CACHE_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define MI_CACHE_API __attribute__((visibility("default")))

MI_CACHE_API const char* mi_cache_last_error(void);

/*
 * dst block pairs[i][1] = src block pairs[i][0] in every plane; pairs [n][2].  dst may be src.  No
 * block may be written twice, nor (in one pool) be both read and written, by one call.
 */
MI_CACHE_API int mi_cache_copy_blocks(const void* src, int64_t src_plane_bytes,
                                      int32_t src_num_blocks, void* dst, int64_t dst_plane_bytes,
                                      int32_t dst_num_blocks, int32_t planes, int64_t block_bytes,
                                      const int32_t* pairs, int32_t n, void* stream);

/*
 * New sequences over another's history.  tables [max_seqs][table_stride], table_width entries of a
 * row used; seq_lens [max_seqs]; children [n][4]: parent slot, child slot, tokens L, new block.  With
 * w = L / block_size and r = L % block_size:
 *   tables[child][0, w) = tables[parent][0, w), seq_lens[child] = L, and where r > 0
 *   tables[child][w] = new block, whose first r tokens in every plane become those of the parent's
 *   block w.  (Where r == 0 the new block is not looked at.)
 * A child whose slots, length, new block or copied block are out of range, or whose two slots are the
 * same, is skipped whole (the entries of whole blocks are copied as they stand).  No child slot or new block may occur twice, and no child slot may be a parent slot.
 */
MI_CACHE_API int mi_cache_fork_rows(void* pool, int64_t plane_bytes, int32_t num_blocks,
                                    int32_t planes, int32_t block_size, int64_t token_bytes,
                                    int32_t* tables, int64_t table_stride, int32_t table_width,
                                    int32_t* seq_lens, int32_t max_seqs, const int32_t* children,
                                    int32_t n, void* stream);

/*
 * Blocks moved and the tables that name them rewritten, in one launch: block pairs[i][1] = block
 * pairs[i][0] in every plane, and tables[rows[i][0]][j] = new_ids[tables[rows[i][0]][j]] for
 * j < rows[i][1]; pairs [n][2], rows [n_rows][2], new_ids [num_blocks].  No block may be both read
 * and written or written twice, and no row may occur twice.
 */
MI_CACHE_API int mi_cache_move_blocks(void* pool, int64_t plane_bytes, int32_t num_blocks,
                                      int32_t planes, int64_t block_bytes, const int32_t* pairs,
                                      int32_t n, int32_t* tables, int64_t table_stride,
                                      int32_t table_width, int32_t max_seqs, const int32_t* rows,
                                      int32_t n_rows, const int32_t* new_ids, void* stream);

/*
 * Attention of packed new tokens over a paged cache whose rows share blocks: the contract of
 * mi_fa2_fwd_paged_varlen (head_dim 128; bf16 0, fp16 1; bottom-right causal; a query that sees no key
 * gives 0 and an lse of -inf; keys at or past kv_lens are never read as data), and the groups:
 * cu_rows [n_groups + 1], prefix_lens [n_groups]: rows [cu_rows[g], cu_rows[g + 1]) hold the same
 * first prefix_lens[g] tokens, which are read for all of them together, through the table of the group's
 * first row.  A prefix is used as far as every query of its group sees it and the first row holds it, and
 * where that costs less than the rows by themselves (not where each has tiles of queries of its own);
 * what is left of it, and a row of no group, is read through the row's own table.  Empty groups may
 * stand anywhere; where groups overlap, a row can only be in the one that begins last before it.
 * A NaN that a query sees shows: a score's in all of its o and in its lse, a value's in that dim.
 *
 * q, o [cu_seqlens_q[batch]][heads_q][128] with strides (token, head), pools [slots][heads_kv][128]
 * with strides (slot, head), lse strides (head, token).  total_q: the tokens of q, at least
 * cu_seqlens_q[batch].  At most 512 rows, 2^25 (token, head) pairs and a max_kv_len of 2^31 - 8193;
 * n_groups <= batch.  workspace: mi_cache_attend_workspace_size bytes, 16-byte aligned, contents
 * arbitrary; not shared by calls that may overlap in time.
 */
MI_CACHE_API size_t mi_cache_attend_workspace_size(int32_t total_q, int32_t heads_q);
MI_CACHE_API int mi_cache_attend(int32_t dtype, const void* q, const void* k_pool,
                                 const void* v_pool, void* o, float* lse,
                                 const int32_t* cu_seqlens_q, const int32_t* block_table,
                                 int64_t block_table_stride, const int32_t* kv_lens,
                                 const int32_t* cu_rows, const int32_t* prefix_lens,
                                 int32_t n_groups, int32_t batch, int32_t total_q, int32_t heads_q,
                                 int32_t heads_kv, int32_t max_kv_len, int32_t head_dim,
                                 int32_t block_size, int32_t num_blocks, const int64_t* q_strides,
                                 const int64_t* pool_strides, const int64_t* o_strides,
                                 const int64_t* lse_strides, int32_t is_causal, float sm_scale,
                                 void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* MI_CACHE_H */
