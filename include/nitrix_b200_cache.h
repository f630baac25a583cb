/*
 * nitrix_b200_cache.h -- C ABI of the paged key / value cache of the B200 (sm_100a) library and of the attention of one new
 * token over it, behind the same shared library, status codes and dtype codes as the attention path
 * (nitrix_b200_attention.h).
 *
 * The cache.  k_pages and v_pages are (pages, heads, page_size, head_dim), each described by three element strides (page,
 * head, slot; unit stride on head_dim; rows on 16-byte boundaries).  Row i of `table` (rows, width) names the pages of
 * sequence i in order: its position p is slot p % page_size of page table[i][p / page_size], for p < lengths[i].  Entries
 * behind the last page in use are not read.  free_pages[free_range[0] .. free_range[1]) are the pages that no row uses, in
 * the order in which they are given out.
 *
 *   nb200_cache_append    tokens offsets[i] .. offsets[i + 1) of k and v are stored behind sequence i's lengths[i]
 *   nb200_cache_fork      row i of the result is row parents[i] (none: empty); full pages are shared, the page that is
 *                         still open is copied for all but the first child
 *   nb200_cache_compact   the live pages move to the pool's front
 *   nb200_decode          attention of one query token per sequence over the cache
 *
 * Each call reads the cache's small arrays and writes new ones, except for append, which adds entries to `table` behind
 * those in use.  Pages are written in place, but only slots that are free in the state that the call is given; the old
 * arrays therefore describe a valid cache until the next call that writes pages.  Where pages run out (or a row of `table`
 * is full), tokens are dropped from the end of the sequences that got none, lengths say what is stored, and `shortfall`
 * counts the dropped tokens: nothing is reported on the host, which does not wait.  Offsets that leave the new tokens are cut
 * to them, and what a sequence misses by that counts as dropped; offsets that descend store nothing, and all tokens count.
 *
 * Every pointer is a device pointer; all work is enqueued on the caller's stream; nothing is allocated.
 */
#ifndef NITRIX_B200_CACHE_H_
#define NITRIX_B200_CACHE_H_

#include "nitrix_b200_attention.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Tokens that a sequence counts at most: places a few blocks behind its end still fit 32 bits. */
#define NB200_CACHE_MOST_TOKENS 0x7fffff00

typedef struct nb200_cache_pages {
  void* k;
  void* v;
  int64_t k_stride[3], v_stride[3];   /* elements, over (page, head, slot) */
  int32_t pages, heads, page_size, head_dim;
  int32_t dtype;                      /* nb200_dtype */
  int32_t reserved;
} nb200_cache_pages;

typedef struct nb200_cache_params {
  size_t struct_size;        /* sizeof(nb200_cache_params) */
  nb200_cache_pages pages;
  /* the state that the call is given */
  int32_t* table;            /* dense (rows, width); append adds entries */
  const int32_t* lengths;    /* (rows) */
  const int32_t* free_pages; /* (pages) */
  const int32_t* free_range; /* (2) */
  int32_t rows, width;
  /* the state after it */
  int32_t* new_table;        /* fork, compact: dense (new_rows, width) */
  int32_t* new_lengths;      /* append, fork: (new_rows) */
  int32_t* new_free_pages;   /* fork, compact: (pages), -1 behind the free ones */
  int32_t* new_free_range;   /* (2) */
  int32_t* shortfall;        /* (1) */
  /* append */
  const void* new_k;         /* (tokens, heads, head_dim), unit stride on head_dim, rows on 16-byte boundaries */
  const void* new_v;
  int64_t new_k_stride[2], new_v_stride[2];   /* elements, over (token, head) */
  const int32_t* offsets;    /* (rows + 1) */
  int64_t tokens;
  /* fork: parents (new_rows), a negative or too large one leaves the row empty; or, with parents NULL, finished (rows) bytes:
   * rows that are set become empty, the others stay */
  const int32_t* parents;
  const uint8_t* finished;
  int32_t new_rows;
  int32_t reserved;
  /* fork, compact */
  void* workspace;           /* nb200_cache_workspace_bytes */
  size_t workspace_bytes;
} nb200_cache_params;

NB200_API int nb200_cache_append(const nb200_cache_params* p, void* cuda_stream);
NB200_API int nb200_cache_fork(const nb200_cache_params* p, void* cuda_stream);
NB200_API int nb200_cache_compact(const nb200_cache_params* p, void* cuda_stream);
NB200_API int nb200_cache_workspace_bytes(const nb200_cache_params* p, size_t* bytes);

typedef struct nb200_decode_params {
  size_t struct_size;        /* sizeof(nb200_decode_params) */
  nb200_cache_pages pages;
  const int32_t* table;      /* dense (rows, width) */
  const int32_t* lengths;    /* (rows); a sequence without a token gives zeros */
  int32_t rows, width;
  const void* q;             /* (rows, q_heads, head_dim), unit stride on head_dim, of the pages' dtype */
  void* out;                 /* dense (rows, q_heads, head_dim) */
  int64_t q_stride[2];       /* elements, over (row, head) */
  int32_t q_heads;           /* a multiple of pages.heads: query head h reads key head h / (q_heads / pages.heads) */
  float scale;
  void* workspace;           /* nb200_decode_workspace_bytes; 16-byte aligned */
  size_t workspace_bytes;
} nb200_decode_params;

NB200_API int nb200_decode(const nb200_decode_params* p, void* cuda_stream);
NB200_API int nb200_decode_workspace_bytes(const nb200_decode_params* p, size_t* bytes);

#ifdef __cplusplus
}
#endif
#endif /* NITRIX_B200_CACHE_H_ */
