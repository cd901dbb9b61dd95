// Argument blocks shared by the paged-cache kernels and their host launchers.
#pragma once
#include <stdint.h>

struct PagedPlanArgs {
  const int32_t *ctx_lens, *new_lens; // [b]
  int32_t *table;                     // [b, max_pages], row stride table_stride
  const int32_t *free_pages;          // [num_free]
  const int32_t *free_start;          // one value, or null = 0
  int32_t *lens, *cu_new, *slots, *free_end; // [b], [b+1], [max_tokens], [1]
  int64_t table_stride;
  int32_t b, max_pages, num_free, page_size, max_tokens;
};

// One cache as the kernels see it; strides in elements (= bytes of codes), the last dimension contiguous.
struct PagedCacheArgs {
  uint8_t *k, *v, *ks, *vs;
  int64_t k_page, k_head, k_tok, v_page, v_head, v_tok;
  int64_t ks_page, ks_head, vs_page, vs_head;
  int32_t pages, heads, page_size, head_dim;
};

struct PagedWriteArgs {
  PagedCacheArgs c;
  const uint16_t *k, *v; // [tokens, heads, head_dim], 16-bit
  const int32_t *slots;
  int64_t k_tok, k_head, v_tok, v_head;
  int32_t tokens;
  int32_t tile;          // consecutive tokens per workgroup (paged_write_any: per wavefront)
};

struct PagedAttnArgs {
  PagedCacheArgs c;
  const uint16_t *q; // [tokens, heads_q, head_dim]
  uint16_t *o;
  float *lse;        // [tokens, heads_q] contiguous, or null
  const int32_t *table, *lens, *cu_q;
  int64_t table_stride, q_tok, q_head, o_tok, o_head;
  int32_t b, max_pages, tokens, heads_q, group; // group = heads_q / heads
  int32_t causal;
  float qk_scale;    // sm_scale * log2(e)
  uint64_t page_magic;  // ceil(2^36 / (page_size / 16)): n / (page_size / 16) = (n * page_magic) >> 36 for n < 2^27,
                        // page_size <= 8192
  float *part, *rows_part; // partial results of split sequences and of split row tiles
  int32_t whole, rows_whole; // a workgroup for each (sequence, head), (row tile, head) instead of an even share of the keys
  int32_t join_pieces;  // workgroups that join a split sequence of few rows
  int32_t rows_groups;  // workgroups for many rows, in front of those for few
  int32_t few_rows;     // launch for many rows: sequences of at most so many (queries times group) are not its
};
