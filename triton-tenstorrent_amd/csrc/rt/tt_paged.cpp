// tt_paged_plan, tt_paged_write, tt_paged_attn: launch validation and kernel selection for the paged 8-bit cache.
#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstring>

#include "tt_internal.h"
#include "../kernels/paged_args.h"

using namespace ttamd;

namespace {
// A launch may have 2^32 - 1 threads in x: workgroups of `threads`.
constexpr int64_t most_groups(int64_t threads) { return UINT32_MAX / threads; }

bool aligned(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

int check_cache(const char *who, const tt_paged_cache *c, PagedCacheArgs *out) {
  if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale) return fail(RT_ERR_INVALID, "%s: null cache or cache pointer", who);
  if (c->num_pages <= 0 || c->heads <= 0 || c->page_size <= 0 || c->head_dim <= 0)
    return fail(RT_ERR_INVALID, "%s: cache of %d pages, %d heads, page size %d, head dim %d", who, c->num_pages, c->heads,
                c->page_size, c->head_dim);
  if ((int64_t)c->num_pages * c->page_size > INT32_MAX)
    return fail(RT_ERR_UNSUPPORTED, "%s: num_pages * page_size exceeds int32", who);
  // paged_write_any steps a 32-bit index through a page's elements, 64 at a time: its last step has to fit too
  if ((int64_t)c->page_size * c->head_dim > INT32_MAX - 63)
    return fail(RT_ERR_UNSUPPORTED, "%s: page_size * head_dim exceeds 2^31 - 64", who);
  if (c->head_dim > 256) return fail(RT_ERR_UNSUPPORTED, "%s: head dim %d (at most 256)", who, c->head_dim);
  for (int i = 0; i < 3; ++i)
    if (c->k_strides[i] < 0 || c->v_strides[i] < 0) return fail(RT_ERR_INVALID, "%s: negative cache stride", who);
  for (int i = 0; i < 2; ++i)
    if (c->k_scale_strides[i] < 0 || c->v_scale_strides[i] < 0) return fail(RT_ERR_INVALID, "%s: negative scale stride", who);
  *out = {(uint8_t *)c->k, (uint8_t *)c->v, (uint8_t *)c->k_scale, (uint8_t *)c->v_scale,
          c->k_strides[0], c->k_strides[1], c->k_strides[2], c->v_strides[0], c->v_strides[1], c->v_strides[2],
          c->k_scale_strides[0], c->k_scale_strides[1], c->v_scale_strides[0], c->v_scale_strides[1],
          c->num_pages, c->heads, c->page_size, c->head_dim};
  return RT_OK;
}

int check_grid(const char *who, const uint32_t grid[3], int32_t x, int32_t y) {
  if (!grid) return fail(RT_ERR_INVALID, "%s: null grid", who);
  if (grid[0] != (uint32_t)x || grid[1] != (uint32_t)y || grid[2] != 1)
    return fail(RT_ERR_INVALID, "%s: grid (%u,%u,%u), expected (%d,%d,1)", who, grid[0], grid[1], grid[2], x, y);
  return RT_OK;
}
// How tt_paged_attn runs a call of these sizes.
struct Route {
  bool fast = false;
  // few queries of a sequence: paged_attn_one_* (exactly one), paged_attn_few_*, or a part of paged_attn_rows_*; its
  // 16-row tiles, its workgroups, and whether sequences may be split (partial results, joined by a second launch)
  bool one = false, one_whole = false, one_join = false;
  int one_tiles = 1, join_pieces = 1;
  uint32_t one_groups = 0;
  // many: paged_attn_rows_*, its workgroups, and whether each has a 128-row tile of its own
  bool rows = false, rows_whole = false;
  int64_t rows_groups = 0;
  size_t one_bytes = 0, workspace = 0;
};
Route route_of(const PagedCacheArgs &c, int32_t B, int32_t max_pages, int32_t tokens, int32_t heads_q, int32_t max_q) {
  Route r;
  const int D = c.head_dim, group = heads_q / c.heads, cus = props()->multiprocessor_count;
  if ((D != 64 && D != 128 && D != 256) || c.page_size % 16 || c.page_size > 8192) return r;
  const int64_t keys = (int64_t)max_pages * c.page_size;
  // positions and rows, rounded up to a unit or a tile, are 32-bit there
  if ((int64_t)tokens * group > INT32_MAX - 1024 || keys > INT32_MAX - 1024) return r;
  r.fast = true;
  // Sequences of few queries go to their own kernel: queries times group up to 32 rows, or 16 where none can have more,
  // where the head dim is 256, or where it is 128 and the registers are shared with the kernel for many rows (pieces of
  // prompts and single tokens: 95 us against 98 with 32).  It is left out where one sequence is all there is and may
  // have more.
  const int64_t rows = (int64_t)max_q * group;
  const int few = D == 256 || rows <= 16 || (D == 128 && rows > 32) ? 16 : 32;
  r.one = group <= few && (rows <= few || B > 1);
  r.rows = !r.one || rows > few;
  if (r.one) {
    r.one_tiles = few / 16;
    const int64_t unit = D * r.one_tiles >= 128 ? 128 : 256;
    const int64_t most = std::max<int64_t>(cdiv64(keys, unit), 1);
    // A workgroup for each head of a group; the groups fill the chip once (two or three workgroups a CU) or have a unit each.
    // (Behind row tiles of head dim 256, with one workgroup on a CU, they come in two turns.)
    const int64_t slots = std::max((D * r.one_tiles > 128 || max_q > 1 ? 2 : 3) * cus / c.heads, 1);
    r.one_groups = (uint32_t)(std::min<int64_t>(most * std::min(B, tokens), slots) * c.heads);
    // A workgroup for each (sequence, head) instead, without parts to join, where the table allows no long sequence: up to
    // 8 units, up to 16 where there are pairs enough to keep the chip busy.  Calls in a captured graph, 8 heads of 128, whole
    // sequences against split ones: 1 sequence of 6 units 9.4 us against 10.3, of 8 units 13.7 against 10.5; 8 sequences of 8
    // units 14.9 against 16.4, of 10 units 17.5 against 16.6; 64 sequences of 16 units 50 against 65.  (The host, which knows
    // the table's width only, cannot tell one short sequence in a wide table from a long one.)
    // Also where the table allows more units than 32 bits count.
    const int64_t pairs = (int64_t)B * c.heads;
    if (most <= (pairs >= slots * c.heads / 2 ? 16 : 8) || most * std::min(B, tokens) > INT32_MAX) {
      if (pairs > most_groups(256)) return Route();
      r.one_whole = true;
      r.one_groups = (uint32_t)pairs;
    }
    r.one_join = !r.one_whole && most > 1 && r.one_groups > (uint32_t)c.heads;
    // sequences of many parts: their rows are joined by several workgroups (6 sequences of 16 parts: 9 us -> 5; with 2 to 3
    // parts the more workgroups cost 2 us)
    if (r.one_groups / c.heads >= 4 * (uint32_t)B) r.join_pieces = 4;
    if (r.one_join) r.one_bytes = (size_t)r.one_groups * (2 * (16 * r.one_tiles * D + 32 * r.one_tiles) * sizeof(float) + 16);
  }
  r.workspace = r.one_bytes;
  if (r.rows) {
    const int64_t items = ((int64_t)tokens * group / 128 + std::min(B, tokens)) * c.heads, slots = (D == 256 ? 1 : 2) * cus;
    // `items` is what the launch may have to hold: a tile for each sequence, also for those that turn out to be the other
    // kernel's.  As a bound of the work it is high beside many single tokens, but the rows by themselves are a worse one (the
    // rule with tokens * group / 128 in its place: a piece of a prompt beside 120, 199 and 256 single tokens 319, 504 and 561 us
    // instead of 330, 548 and 596, beside 159 441 instead of 426; 128 sequences of up to 20 tokens 111 instead of 95, 200
    // 151 instead of 138).  (The last condition: more steps than 32 bits count.)
    r.rows_whole = items >= 2 * slots || keys <= 64 || items / c.heads * cdiv64(keys, 64) > INT32_MAX;
    r.rows_groups = r.rows_whole ? items : std::max<int64_t>(slots / c.heads, 1) * c.heads;
    if (!r.rows_whole) r.workspace += (size_t)r.rows_groups * (2 * (128 * D + 256) * sizeof(float) + 16);
  }
  return r;
}
} // namespace

extern "C" int tt_paged_plan(const int32_t *ctx_lens, const int32_t *new_lens, int32_t *block_table, int64_t table_stride,
                             int32_t B, int32_t max_pages, const int32_t *free_pages, int32_t num_free,
                             const int32_t *free_start, int32_t page_size, int32_t max_tokens, int32_t *lens,
                             int32_t *cu_new, int32_t *slot_map, int32_t *free_end, const uint32_t grid[3], void *stream) {
  const char *who = "paged_plan";
  if (!props()) return fail(RT_ERR_NOT_INIT, "%s: call rt_init first", who);
  if (B <= 0 || max_pages <= 0 || page_size <= 0 || num_free < 0 || max_tokens < 0)
    return fail(RT_ERR_INVALID, "%s: B %d, max_pages %d, page_size %d, num_free %d, max_tokens %d", who, B, max_pages,
                page_size, num_free, max_tokens);
  if (!ctx_lens || !new_lens || !block_table || (num_free && !free_pages) || !lens || !cu_new || (max_tokens && !slot_map) ||
      !free_end)
    return fail(RT_ERR_INVALID, "%s: null pointer", who);
  if (table_stride < max_pages) return fail(RT_ERR_INVALID, "%s: table stride %lld, %d entries", who, (long long)table_stride, max_pages);
  if ((int64_t)max_pages * page_size > INT32_MAX) return fail(RT_ERR_UNSUPPORTED, "%s: max_pages * page_size exceeds int32", who);
  if (B > (1 << 20)) return fail(RT_ERR_UNSUPPORTED, "%s: %d sequences (at most 2^20)", who, B);
  for (const void *p : {(const void *)ctx_lens, (const void *)new_lens, (const void *)block_table, (const void *)free_pages,
                        (const void *)free_start, (const void *)lens, (const void *)cu_new, (const void *)slot_map,
                        (const void *)free_end})
    if (!aligned(p, 4)) return fail(RT_ERR_INVALID, "%s: pointer not aligned to 4 bytes", who);
  // One workgroup may write its results while another still reads: no output may share memory with anything else.
  const struct { const char *name; const void *p; int64_t n; bool out; } v[] = {
      {"ctx_lens", ctx_lens, B, false}, {"new_lens", new_lens, B, false}, {"free_pages", free_pages, num_free, false},
      {"free_start", free_start, free_start ? 1 : 0, false}, {"block_table", block_table, (B - 1) * table_stride + max_pages, true},
      {"lens", lens, B, true}, {"cu_new", cu_new, (int64_t)B + 1, true}, {"slot_map", slot_map, max_tokens, true},
      {"free_end", free_end, 1, true}};
  for (const auto &x : v)
    for (const auto &y : v)
      if (&x < &y && y.out && x.n && y.n && (uintptr_t)x.p < (uintptr_t)y.p + 4 * y.n && (uintptr_t)y.p < (uintptr_t)x.p + 4 * x.n)
        return fail(RT_ERR_INVALID, "%s: %s and %s overlap", who, x.name, y.name);
  int rc;
  if ((rc = check_grid(who, grid, B, 1))) return rc;
  PagedPlanArgs a{ctx_lens, new_lens, block_table, free_pages, free_start, lens, cu_new, slot_map, free_end,
                  table_stride, B, max_pages, num_free, page_size, max_tokens};
  const uint32_t wgs = (uint32_t)std::clamp<int64_t>(cdiv64(max_tokens, 1024), 1, props()->multiprocessor_count);
  void *args[] = {&a};
  return launch("paged", "paged_plan", dim3(wgs), dim3(1024), 0, stream, args, 1);
}

extern "C" int tt_paged_write(const void *k, const void *v, const int64_t k_strides[2], const int64_t v_strides[2],
                              const int32_t *slot_map, int32_t tokens, const tt_paged_cache *cache, int32_t dtype,
                              const uint32_t grid[3], void *stream) {
  const char *who = "paged_write";
  if (!props()) return fail(RT_ERR_NOT_INIT, "%s: call rt_init first", who);
  PagedWriteArgs a;
  memset(&a, 0, sizeof(a));
  int rc;
  if ((rc = check_cache(who, cache, &a.c))) return rc;
  if (dtype != TT_BF16 && dtype != TT_F16) return fail(RT_ERR_UNSUPPORTED, "%s: dtype %d (bf16 and fp16 are supported)", who, dtype);
  if (tokens <= 0) return fail(RT_ERR_INVALID, "%s: %d tokens", who, tokens);
  if (!k || !v || !k_strides || !v_strides || !slot_map) return fail(RT_ERR_INVALID, "%s: null pointer", who);
  for (int i = 0; i < 2; ++i)
    if (k_strides[i] < 0 || v_strides[i] < 0) return fail(RT_ERR_INVALID, "%s: negative stride", who);
  // the cache is written: no two of its elements may lie in one place because a stride is 0
  const PagedCacheArgs &w = a.c;
  if ((w.pages > 1 && (!w.k_page || !w.v_page || !w.ks_page || !w.vs_page)) || (w.heads > 1 && (!w.k_head || !w.v_head || !w.ks_head || !w.vs_head)) ||
      (w.page_size > 1 && (!w.k_tok || !w.v_tok)))
    return fail(RT_ERR_INVALID, "%s: a cache stride is 0", who);
  if (!aligned(k, 2) || !aligned(v, 2) || !aligned(slot_map, 4)) return fail(RT_ERR_INVALID, "%s: misaligned pointer", who);
  if ((rc = check_grid(who, grid, tokens, 1))) return rc;
  a.k = (const uint16_t *)k; a.v = (const uint16_t *)v; a.slots = slot_map;
  a.k_tok = k_strides[0]; a.k_head = k_strides[1]; a.v_tok = v_strides[0]; a.v_head = v_strides[1];
  a.tokens = tokens;
  void *args[] = {&a};
  const PagedCacheArgs &c = a.c;
  const int D = c.head_dim;
  const bool al = aligned16(k) && aligned16(v) && (a.k_tok | a.k_head | a.v_tok | a.v_head) % 8 == 0 && aligned(c.k, 8) &&
                  aligned(c.v, 8) && (c.k_page | c.k_head | c.k_tok | c.v_page | c.v_head | c.v_tok) % 8 == 0 &&
                  std::max({a.k_tok, a.v_tok, c.k_tok, c.v_tok}) < (1 << 26); // (offsets inside 8 rows fit 32 bits)
  char name[64];
  int64_t wgs;
  if (al && (D == 64 || D == 128 || D == 256)) {
    // Tokens per workgroup.  16 single tokens are what its wavefronts do at once at head dim 128; where that gives more
    // workgroups than the chip takes at a time (6 or 7 a CU), 64 leave fewer that only find out that a run began before them.
    // In a captured graph, 8 heads of 128, 16 against 64: 256 single tokens 3.9 us against 5.9, 1024 4.8 against 6.2, 2048
    // 7.1 against 7.1; a prompt of 2090 tokens 8.3 against 5.7 (and of 1045, which the host cannot tell from single ones, 6.5
    // against 4.6).
    a.tile = cdiv64(tokens, 16) * c.heads * 2 > 8 * props()->multiprocessor_count ? 64 : 16;
    wgs = cdiv64(tokens, a.tile) * c.heads * 2;
    snprintf(name, sizeof(name), "paged_write_%s_d%d", dtype == TT_BF16 ? "bf16" : "f16", D);
  } else {
    a.tile = 1;
    wgs = cdiv64((int64_t)tokens * c.heads * 2, 4);
    snprintf(name, sizeof(name), "paged_write_any_%s", dtype == TT_BF16 ? "bf16" : "f16");
  }
  if (wgs > most_groups(256)) return fail(RT_ERR_UNSUPPORTED, "%s: tokens * heads exceeds the grid", who);
  return launch("paged", name, dim3((uint32_t)wgs), dim3(256), 0, stream, args, 1);
}

extern "C" int tt_paged_attn_workspace(int32_t B, int32_t max_pages, int32_t tokens, int32_t heads_q, int32_t max_q,
                                       const tt_paged_cache *cache, size_t *bytes) {
  const char *who = "paged_attn_workspace";
  if (!props()) return fail(RT_ERR_NOT_INIT, "%s: call rt_init first", who);
  if (!bytes) return fail(RT_ERR_INVALID, "%s: null out pointer", who);
  PagedCacheArgs c;
  int rc;
  if ((rc = check_cache(who, cache, &c))) return rc;
  if (B <= 0 || max_pages <= 0 || tokens <= 0 || heads_q <= 0 || max_q <= 0 || heads_q % c.heads)
    return fail(RT_ERR_INVALID, "%s: B %d, max_pages %d, tokens %d, heads %d over %d, max_q %d", who, B, max_pages, tokens,
                heads_q, c.heads, max_q);
  *bytes = route_of(c, B, max_pages, tokens, heads_q, max_q).workspace;
  return RT_OK;
}

extern "C" int tt_paged_attn(const void *q, const int64_t q_strides[2], const tt_paged_cache *cache, const int32_t *block_table,
                             int64_t table_stride, int32_t B, int32_t max_pages, const int32_t *lens, const int32_t *cu_q,
                             int32_t tokens, int32_t heads_q, int32_t max_q, float sm_scale, int32_t causal, int32_t dtype,
                             void *o, const int64_t o_strides[2], float *lse, void *workspace, size_t workspace_bytes,
                             const uint32_t grid[3], void *stream) {
  const char *who = "paged_attn";
  if (!props()) return fail(RT_ERR_NOT_INIT, "%s: call rt_init first", who);
  PagedAttnArgs a;
  memset(&a, 0, sizeof(a));
  size_t need = 0;
  int rc;
  if ((rc = check_cache(who, cache, &a.c))) return rc;
  if ((rc = tt_paged_attn_workspace(B, max_pages, tokens, heads_q, max_q, cache, &need))) return rc;
  if (dtype != TT_BF16 && dtype != TT_F16) return fail(RT_ERR_UNSUPPORTED, "%s: dtype %d (bf16 and fp16 are supported)", who, dtype);
  if (!q || !q_strides || !o || !o_strides || !block_table || !lens || !cu_q) return fail(RT_ERR_INVALID, "%s: null pointer", who);
  if (table_stride < max_pages) return fail(RT_ERR_INVALID, "%s: table stride %lld, %d entries", who, (long long)table_stride, max_pages);
  if ((int64_t)max_pages * a.c.page_size > INT32_MAX) return fail(RT_ERR_UNSUPPORTED, "%s: max_pages * page_size exceeds int32", who);
  for (int i = 0; i < 2; ++i)
    if (q_strides[i] < 0 || o_strides[i] < 0) return fail(RT_ERR_INVALID, "%s: negative stride", who);
  if ((tokens > 1 && !o_strides[0]) || (heads_q > 1 && !o_strides[1])) return fail(RT_ERR_INVALID, "%s: a stride of o is 0", who);
  if (!aligned(q, 2) || !aligned(o, 2) || !aligned(block_table, 4) || !aligned(lens, 4) || !aligned(cu_q, 4) || !aligned(lse, 4))
    return fail(RT_ERR_INVALID, "%s: misaligned pointer", who);
  if (!std::isfinite(sm_scale)) return fail(RT_ERR_INVALID, "%s: sm_scale is not finite", who);
  if (need && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))
    return fail(RT_ERR_INVALID, "%s: a 16-byte aligned workspace of %zu bytes is needed, got %zu", who, need, workspace ? workspace_bytes : 0);
  if ((rc = check_grid(who, grid, tokens, heads_q))) return rc;
  if (heads_q > 65535) return fail(RT_ERR_UNSUPPORTED, "%s: %d query heads (at most 65535)", who, heads_q);
  a.q = (const uint16_t *)q; a.o = (uint16_t *)o; a.lse = lse;
  a.table = block_table; a.lens = lens; a.cu_q = cu_q; a.table_stride = table_stride;
  a.q_tok = q_strides[0]; a.q_head = q_strides[1]; a.o_tok = o_strides[0]; a.o_head = o_strides[1];
  a.b = B; a.max_pages = max_pages; a.tokens = tokens; a.heads_q = heads_q; a.group = heads_q / a.c.heads;
  a.causal = causal != 0; a.qk_scale = sm_scale * 1.44269504f;
  void *args[] = {&a};
  const char *type = dtype == TT_BF16 ? "bf16" : "f16";
  char name[64];
  const Route r = route_of(a.c, B, max_pages, tokens, heads_q, max_q);
  // 16-byte loads of the cache and of q, 8-byte stores of results, and offsets inside 16 rows that fit 32 bits
  const PagedCacheArgs &c = a.c;
  const bool al = aligned16(c.k) && aligned16(c.v) && (c.k_page | c.k_head | c.k_tok | c.v_page | c.v_head | c.v_tok) % 16 == 0 &&
                  std::max(c.k_tok, c.v_tok) < (1 << 26) && aligned16(a.q) && (a.q_tok | a.q_head) % 8 == 0 &&
                  aligned(a.o, 8) && (a.o_tok | a.o_head) % 4 == 0;
  if (r.fast && al) {
    const uint64_t per = (uint64_t)c.page_size / 16;
    a.page_magic = ((1ull << 36) + per - 1) / per;
    a.few_rows = r.one ? 16 * r.one_tiles : 0;
    a.whole = r.one_whole;
    a.part = r.one_join ? (float *)workspace : nullptr;
    a.join_pieces = r.join_pieces;
    const bool few = r.rows || max_q > 1;
    const char *kernel = r.rows ? "rows" : few ? "few" : "one";
    snprintf(name, sizeof(name), "paged_attn_%s_%s_d%d_r%d", kernel, type, c.head_dim, r.one_tiles);
    if (r.rows) {
      a.rows_whole = r.rows_whole;
      a.rows_part = (float *)((char *)workspace + r.one_bytes);
      a.rows_groups = (int32_t)r.rows_groups;
    }
    if (r.rows_groups + r.one_groups > most_groups(256)) return fail(RT_ERR_UNSUPPORTED, "%s: tokens * heads exceeds the grid", who);
    if ((rc = launch("paged", name, dim3((uint32_t)(r.rows_groups + r.one_groups)), dim3(256), 0, stream, args, 1))) return rc;
    if (r.rows_whole) a.rows_groups = 0; // nothing to join there
    const uint32_t joins = 8 * (uint32_t)a.rows_groups + (r.one_join ? r.one_groups * r.join_pieces : 0);
    if (!joins) return RT_OK;
    snprintf(name, sizeof(name), "paged_attn_%s_%s_d%d_r%d", r.rows ? "rows_join" : "join", type, c.head_dim, r.one_tiles);
    return launch("paged", name, dim3(joins), dim3(256), 0, stream, args, 1);
  }
  if (tokens > most_groups(64)) return fail(RT_ERR_UNSUPPORTED, "%s: %d tokens exceed the grid", who, tokens);
  return launch("paged", dtype == TT_BF16 ? "paged_attn_any_bf16" : "paged_attn_any_f16",
                dim3((uint32_t)tokens, (uint32_t)heads_q), dim3(64), 0, stream, args, 1);
}
