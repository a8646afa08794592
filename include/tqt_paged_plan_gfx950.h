/*
 * The bookkeeping of one step over a paged cache, on the device: from the number of new tokens of every
 * sequence their pages, block tables, lengths, slots and positions, and for trees of drafted tokens which of them
 * each one sees. What it writes is what tqt_run_kv_append_rope_*, tqt_run_attn_paged_* and tqt_run_attn_tree_*
 * read, so a step may be captured as a whole and replayed as the lengths change. No counterpart in the
 * reference library.
 *
 * Sequence b holds kv_len[b] tokens, whose pages are the first held[b] entries of its row of block_table, and
 * brings new_len[b] more (0: none in this step; negative: it has ended). free_pages[0 .. free_count) is a stack of
 * pages that nobody holds. In this order:
 *   1. The pages of ended sequences go on the stack, sequence by sequence and entry by entry (entries outside
 *      [0, num_pages) are pages that are not kept, and are left out); kv_len_out and held_out become 0.
 *   2. Every other sequence needs need_b = max(0, ceil((kv_len + new_len) / page_size) - held) pages. It is refused
 *      if its rows do not all fit into `tokens` or its pages into ld_table, and then counts with need_b = 0, or if
 *      need_b > 0 and the needs of the sequences up to and with it exceed the stack. A refused one keeps its pages
 *      and its length, and the slots of its rows are -1 (which the append skips); refused[0] is their number.
 *   3. The others take their pages from the stack's top, in the order of the batch, as entries held ... of their
 *      rows of block_table: kv_len_out = kv_len + new_len, held_out = held + need_b.
 *   q_start[b + 1] = min(tokens, new tokens of sequences up to b), refused ones with their rows; row i of sequence
 *   b has slot page * page_size + offset of token kv_len[b] + i (-1 where its page is outside [0, num_pages)) and
 *   position kv_len[b] + i. Rows from q_start[batch] on have slot -1, position 0 and no mask bits.
 * Pages past what a sequence needs (drafted tokens that were not accepted) stay with it and are used first.
 *
 * Trees: parent[row] is the number, within its sequence's new tokens, of the token that this one follows, -1
 * for one that follows the context (an entry that is not below the row's own number counts as -1). Then the
 * position is kv_len[b] + depth, 0 for tokens that follow the context, and bit t of mask[row] (bit t % 32 of word
 * t / 32) says whether token t is this one or one that it descends from; bits from 32 * ld_mask on are left out,
 * and all others of the row's ld_mask words are 0. A row's tokens are found one from the other, so a long chain takes long
 * (8 nodes for 63 sequences and for one more a chain of 64: 8.6 us, of 512: 38, of 4096: 417): prompts are better a step
 * without trees.
 *
 * kv_len_out, held_out and free_count_out may be kv_len, held and free_count; no other two arrays may overlap. A step that
 * tqt_run_kv_keep_* ends takes another array for kv_len_out, from which that call writes kv_len: in place every drafted
 * token would count from the next step on. A slot of -1 does not say that its sequence was refused (its page may be none);
 * that its first row's position is kv_len_out or more does.
 * Lengths count as 0 at least and 2^30 at most (a sequence that would grow past that is refused), held as the pages of
 * kv_len at least and as ld_table at most, free_count as 0 to free_capacity; pages that do not fit on the stack any
 * more are lost. workspace holds at least
 * tqt_get_workspace_size_paged_plan_gfx950 bytes on the 16-byte grid (it may be NULL for size 0), needs no initial
 * value, and is free again when the call has run. Results do not depend on the order in which workgroups run.
 * Pointers are device pointers; conventions as in tqt_rope_gfx950.h.
 */
#ifndef TQT_PAGED_PLAN_GFX950_H
#define TQT_PAGED_PLAN_GFX950_H

#include "tqt_gfx950_common.h"

#ifdef __cplusplus
extern "C" {
#endif

struct tqt_paged_plan_params
{
    size_t batch;
    size_t tokens; /* rows of positions, slots, parent and mask */
    size_t page_size;
    size_t num_pages;
    const int32_t *new_len; /* [batch] */
    const int32_t *kv_len;  /* [batch] */
    int32_t *kv_len_out;
    const int32_t *held; /* [batch] */
    int32_t *held_out;
    int32_t *block_table; /* [batch][ld_table], new entries are written */
    size_t ld_table;
    int32_t *free_pages; /* [free_capacity] */
    size_t free_capacity;
    const int32_t *free_count; /* [1] */
    int32_t *free_count_out;
    int32_t *refused;      /* [1] */
    int32_t *q_start;      /* [batch + 1] */
    int32_t *positions;    /* [tokens] */
    int64_t *slots;        /* [tokens] */
    const int32_t *parent; /* [tokens], or NULL: no trees */
    uint32_t *mask;        /* [tokens][ld_mask]; NULL without trees */
    size_t ld_mask;
    void *workspace;
    size_t workspace_size;
};

/* Depends on batch and tokens only. */
size_t tqt_get_workspace_size_paged_plan_gfx950(const struct tqt_paged_plan_params *params);

const char *tqt_get_error_paged_plan_gfx950(const struct tqt_paged_plan_params *params);
void tqt_run_paged_plan_gfx950(const struct tqt_paged_plan_params *params);
void tqt_run_paged_plan_gfx950_async(const struct tqt_paged_plan_params *params, void *stream);

#ifdef __cplusplus
} /* extern "C" */
#endif

#endif
