// A paged key/value cache in 8 bits for gfx950: its plan (block tables and slot maps from request lengths), its
// quantising write, and attention over it (paged_attn*.h).
//
// Cache: e4m3 codes [pages, heads, page_size, head_dim] for K and for V, and one scale for each (page, head), held as
// its exponent: code s stands for 2^(s - 127).  A power of two costs e4m3 nothing (a floating-point code has the same
// precision at every scale) and makes the change of a page's scale exact but for codes that become subnormal.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "paged_args.h"

namespace {

constexpr int kMinScale = 27; // 2^-100: the scale of a page of zeros

// ---------------------------------------------------------------------------
// plan
// ---------------------------------------------------------------------------
// Inclusive scan over the 1024 threads of the workgroup; `add` is associative with identity 0.
template <typename F> __device__ __forceinline__ uint32_t scan1024(uint32_t v, uint32_t *part, F add) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t o = __shfl_up(v, d);
    if (lane >= d) v = add(o, v);
  }
  __syncthreads(); // `part` may still be read from an earlier scan
  if (lane == 63) part[wave] = v;
  __syncthreads();
  uint32_t before = 0;
  for (int w = 0; w < wave; ++w) before = add(before, part[w]);
  return add(before, v);
}

__device__ __forceinline__ int32_t clampi(int32_t v, int32_t lo, int32_t hi) { return v < lo ? lo : v > hi ? hi : v; }

} // namespace

// Every workgroup scans all sequences (the lengths are a few KB that the L2 holds) and then does its share of the
// tokens, so that no workgroup waits for another and one launch is enough: a few KB in and out, the time is that of
// dependent loads and two scans (16 sequences 4.8 us; 1000 sequences, 142619 tokens 7.0 us).  Thread i owns `per` consecutive sequences; two scans, the tokens'
// (saturating at max_tokens) and the pages'.  A new token at the start of a page writes that page's table entry.
extern "C" __global__ __launch_bounds__(1024) void paged_plan(PagedPlanArgs a) {
  __shared__ uint32_t part[16];
  __shared__ int32_t tok0[1025], page0[1024]; // first token / first new page of thread i's sequences
  const int tid = threadIdx.x;
  const uint32_t cap = (uint32_t)a.max_tokens;
  const int32_t P = a.page_size, width = a.max_pages * P;
  const int per = (a.b + 1023) / 1024;
  const int b0 = min(tid * per, a.b), b1 = min(b0 + per, a.b);
  auto sat = [cap](uint32_t x, uint32_t y) { return min(x + y, cap); };
  auto plus = [](uint32_t x, uint32_t y) { return x + y; };
  auto ctx_of = [&](int b) { return clampi(a.ctx_lens[b], 0, width); };
  auto fits_of = [&](int b, int32_t ctx) { return min((uint32_t)max(a.new_lens[b], 0), (uint32_t)(width - ctx)); };
  auto pages_of = [P](int32_t n) { return (int32_t)(((uint32_t)n + (uint32_t)P - 1) / (uint32_t)P); };

  uint32_t mine = 0;
  for (int b = b0; b < b1; ++b) mine = sat(mine, min(fits_of(b, ctx_of(b)), cap));
  const uint32_t incl = scan1024(mine, part, sat);
  uint32_t total = 0;
  for (int w = 0; w < 16; ++w) total = sat(total, part[w]);
  // (saturated sums cannot be subtracted: the exclusive value comes from the left neighbour)
  __syncthreads();
  tok0[tid + 1] = (int32_t)incl;
  if (tid == 0) tok0[0] = 0;
  __syncthreads();
  uint32_t cu = (uint32_t)tok0[tid];
  const uint32_t cu_first = cu;
  uint32_t fresh = 0;
  for (int b = b0; b < b1; ++b) {
    const int32_t ctx = ctx_of(b);
    const uint32_t next = sat(cu, min(fits_of(b, ctx), cap));
    fresh += (uint32_t)(pages_of(ctx + (int32_t)(next - cu)) - pages_of(ctx));
    cu = next;
  }
  const uint32_t pincl = scan1024(fresh, part, plus);
  const int32_t start = a.free_start ? a.free_start[0] : 0;
  const int32_t pg = start + (int32_t)(pincl - fresh);
  page0[tid] = pg;
  __syncthreads();

  if (blockIdx.x == 0) {
    cu = cu_first;
    for (int b = b0; b < b1; ++b) {
      const int32_t ctx = ctx_of(b);
      const uint32_t next = sat(cu, min(fits_of(b, ctx), cap));
      a.cu_new[b] = (int32_t)cu;
      a.lens[b] = ctx + (int32_t)(next - cu);
      cu = next;
    }
    if (tid == 1023) {
      a.cu_new[a.b] = (int32_t)total;
      a.free_end[0] = start + (int32_t)pincl;
    }
  }

  for (int64_t t64 = (int64_t)blockIdx.x * 1024 + tid; t64 < a.max_tokens; t64 += (int64_t)gridDim.x * 1024) {
    const int32_t t = (int32_t)t64;
    int32_t slot = -1;
    if ((uint32_t)t < total) {
      int lo = 0, hi = 1023; // the last thread whose first token is at most t
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (tok0[mid] <= t) lo = mid; else hi = mid - 1;
      }
      int32_t c = tok0[lo], page = page0[lo];
      int b = min(lo * per, a.b);
      int32_t ctx = 0, n = 0;
      const int be = min(b + per, a.b);
      for (; b < be; ++b) {
        ctx = ctx_of(b);
        n = (int32_t)(sat((uint32_t)c, min(fits_of(b, ctx), cap)) - (uint32_t)c);
        if (t < c + n) break;
        c += n;
        page += pages_of(ctx + n) - pages_of(ctx);
      }
      const int32_t pos = ctx + (t - c), blk = (int32_t)((uint32_t)pos / (uint32_t)P), had = pages_of(ctx);
      int32_t *entry = a.table + (int64_t)b * a.table_stride + blk;
      int32_t id;
      if (blk >= had) {
        const int32_t at = page + (blk - had);
        id = at >= 0 && at < a.num_free ? a.free_pages[at] : -1;
        if (pos == blk * P) *entry = id;
      } else {
        id = *entry;
      }
      const int64_t s = (int64_t)id * P + (pos - blk * P);
      slot = id >= 0 && s <= INT32_MAX ? (int32_t)s : -1;
    }
    a.slots[t] = slot;
  }
}

// ---------------------------------------------------------------------------
// write
// ---------------------------------------------------------------------------
namespace {

typedef __bf16 w_bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 w_f16x2 __attribute__((ext_vector_type(2)));
typedef short w_s16x2 __attribute__((ext_vector_type(2)));

// The two input types.  codes2: two values, divided by the power of two `scale` and rounded to nearest even, into the
// low or high half of c; they must be finite and at most 448 scale (one v_cvt_scalef32_pk_fp8_*).
struct Bf16 {
  static constexpr uint32_t kInfinite = 0x7f80;
  static __device__ __forceinline__ float get(uint16_t h) { return __builtin_bit_cast(float, (uint32_t)h << 16); }
  template <bool HI> static __device__ __forceinline__ w_s16x2 codes2(w_s16x2 c, uint32_t x, float scale) {
    return __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(c, __builtin_bit_cast(w_bf16x2, x), scale, HI);
  }
};
struct Fp16 {
  static constexpr uint32_t kInfinite = 0x7c00;
  static __device__ __forceinline__ float get(uint16_t h) { return (float)__builtin_bit_cast(_Float16, h); }
  template <bool HI> static __device__ __forceinline__ w_s16x2 codes2(w_s16x2 c, uint32_t x, float scale) {
    return __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(c, __builtin_bit_cast(w_f16x2, x), scale, HI);
  }
};

// bits of |x|, 0 for infinities and NaN: what does not decide a scale
__device__ __forceinline__ uint32_t finite_mag(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x) & 0x7fffffffu;
  return u < 0x7f800000u ? u : 0u;
}
// smallest scale code s with amax <= 448 * 2^(s-127) = 1.75 * 2^(s-119), from the bits of amax
__device__ __forceinline__ int scale_for(uint32_t amax) {
  return max((int)(amax >> 23) - 8 + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0), kMinScale);
}
__device__ __forceinline__ float pow2_code(int s) { return __builtin_bit_cast(float, (uint32_t)s << 23); }
// saturating (an infinity becomes +-448), NaN stays NaN
__device__ __forceinline__ float sat448(float y) { return y != y ? y : fminf(fmaxf(y, -448.0f), 448.0f); }
// The maximum over the wavefront, in a scalar register: within the rows of 16 lanes, then across them.
__device__ __forceinline__ uint32_t max64(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xf, 0xf, false)); // row_shr:1
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xf, 0xf, false)); // row_shr:2
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xf, false)); // row_shr:4
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xf, 0xf, false)); // row_shr:8
  return max(max((uint32_t)__builtin_amdgcn_readlane((int)v, 15), (uint32_t)__builtin_amdgcn_readlane((int)v, 31)),
             max((uint32_t)__builtin_amdgcn_readlane((int)v, 47), (uint32_t)__builtin_amdgcn_readlane((int)v, 63)));
}

// One wavefront writes the runs that begin among its `tile` tokens, for one head of K or of V.  A run is a stretch of
// tokens whose slots follow one another inside one page: it has one scale.  Whatever the alignment: one element per
// lane and step.
template <typename E> __device__ __forceinline__ void write_any(const PagedWriteArgs &a) {
  const int lane = threadIdx.x & 63;
  const int64_t unit = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const bool isv = unit & 1;
  const int head = (int)((unit >> 1) % a.c.heads);
  const int64_t first = (unit >> 1) / a.c.heads * a.tile;
  const int P = a.c.page_size, D = a.c.head_dim;
  const int64_t nslots = (int64_t)a.c.pages * P;
  const uint16_t *x = (isv ? a.v : a.k) + head * (isv ? a.v_head : a.k_head);
  const int64_t x_tok = isv ? a.v_tok : a.k_tok;
  for (int64_t t = first; t < min(first + a.tile, (int64_t)a.tokens); ++t) {
    const int32_t slot = a.slots[t];
    if (slot < 0 || slot >= nslots) continue;
    const int row = slot % P;
    const int64_t page = slot / P;
    if (row && t && a.slots[t - 1] == slot - 1) continue; // inside a run that began before
    int n = 1;
    while (row + n < P && t + n < a.tokens && a.slots[t + n] == slot + n) ++n;
    uint8_t *sp = (isv ? a.c.vs + page * a.c.vs_page + head * a.c.vs_head : a.c.ks + page * a.c.ks_page + head * a.c.ks_head);
    uint8_t *base = isv ? a.c.v + page * a.c.v_page + head * a.c.v_head : a.c.k + page * a.c.k_page + head * a.c.k_head;
    const int64_t c_tok = isv ? a.c.v_tok : a.c.k_tok;
    uint32_t amax = 0;
    for (int i = lane; i < n * D; i += 64) amax = max(amax, finite_mag(E::get(x[(t + i / D) * x_tok + i % D])));
    amax = max64(amax);
    int s = scale_for(amax);
    if (row) {
      const int old = *sp;
      if (s > old) { // the tokens before the run go to the larger scale
        const float f = pow2_code(max(127 + old - s, 0));
        for (int i = lane; i < row * D; i += 64) {
          uint8_t *p = base + (i / D) * c_tok + i % D;
          const float y = __builtin_amdgcn_cvt_f32_fp8(*p, 0) * f;
          *p = (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(y, y, 0, false);
        }
      }
      s = max(s, old);
    }
    const float inv = pow2_code(254 - s);
    for (int i = lane; i < n * D; i += 64) {
      const float y = sat448(E::get(x[(t + i / D) * x_tok + i % D]) * inv);
      base[(row + i / D) * c_tok + i % D] = (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(y, y, 0, false);
    }
    if (lane == 0) *sp = (uint8_t)s;
  }
}

// ---- head dims 64, 128, 256, 16-byte aligned rows ----
// Bound: HBM, 2 bytes read and 1 written a value; measured 48 us for 38171 prompt tokens of 8 heads of 128 (235 MB, 4.8 TB/s
// where a copy reaches 6.7; the chain of slots, values and barrier costs as much as the memory), 3.5 us for 64 single
// tokens.  Six workgroups a CU: at eight the registers spill.  A lane takes 8 values (16 bytes in, 8 out), so a row is D / 8 lanes and
// a wavefront step RPS rows.  A workgroup looks at `tile` tokens for one head of K or of V; its wavefronts share the runs
// that begin there:
//   - a run of several tokens is one wavefront's, a long one all four's, held in registers between the maximum and the
//     conversion (one read; twice beyond 16 * RPS tokens);
//   - single tokens (a decode step) go RPS at a time, one to each group of D / 8 lanes;
//   - where a scale grows, the whole wavefront moves that page's earlier rows to it.
typedef uint32_t w_u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t w_u32x4 __attribute__((ext_vector_type(4)));
typedef float w_f32x2 __attribute__((ext_vector_type(2)));

typedef uint16_t w_u16x2 __attribute__((ext_vector_type(2)));

// The largest magnitude of 8 values, as the bits of a 16-bit float: they order like the magnitudes.
__device__ __forceinline__ uint32_t top_of8(w_u32x4 x) {
  w_u16x2 m = __builtin_bit_cast(w_u16x2, x[0] & 0x7fff7fffu);
#pragma unroll
  for (int i = 1; i < 4; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(w_u16x2, x[i] & 0x7fff7fffu));
  return max((uint32_t)m[0], (uint32_t)m[1]);
}
// The same among the finite ones: for runs that hold an infinity or NaN.
template <typename E> __device__ __forceinline__ uint32_t finite_top_of8(w_u32x4 x) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int h = 0; h < 32; h += 16) {
      const uint32_t u = (x[i] >> h) & 0x7fffu;
      m = max(m, u < E::kInfinite ? u : 0u);
    }
  return m;
}
template <typename E> __device__ __forceinline__ int scale_of_top(uint32_t top) {
  return scale_for(__builtin_bit_cast(uint32_t, E::get((uint16_t)top)));
}
template <typename E> __device__ __forceinline__ w_u32x2 codes_of8(w_u32x4 x, int s, bool wild) {
  w_u32x2 r;
  if (wild) {
    const float inv = pow2_code(254 - s);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      int c = __builtin_amdgcn_cvt_pk_fp8_f32(sat448(E::get((uint16_t)x[2 * i]) * inv), sat448(E::get((uint16_t)(x[2 * i] >> 16)) * inv), 0, false);
      c = __builtin_amdgcn_cvt_pk_fp8_f32(sat448(E::get((uint16_t)x[2 * i + 1]) * inv), sat448(E::get((uint16_t)(x[2 * i + 1] >> 16)) * inv), c, true);
      r[i] = (uint32_t)c;
    }
  } else {
    const float scale = pow2_code(s);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      w_s16x2 c = {0, 0};
      c = E::template codes2<false>(c, x[2 * i], scale);
      c = E::template codes2<true>(c, x[2 * i + 1], scale);
      r[i] = __builtin_bit_cast(uint32_t, c);
    }
  }
  return r;
}
__device__ __forceinline__ w_u32x2 rescale8(w_u32x2 x, float f) {
  w_u32x2 r;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const w_f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)x[i], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)x[i], true);
    int c = __builtin_amdgcn_cvt_pk_fp8_f32(lo[0] * f, lo[1] * f, 0, false);
    r[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(hi[0] * f, hi[1] * f, c, true);
  }
  return r;
}

// Rows [0, rows) of a page to the scale 2^(new - old) times larger; the whole wavefront, all arguments uniform.
template <int D> __device__ __forceinline__ void rescale_rows(uint8_t *base, int64_t tok, int rows, int old, int s) {
  constexpr int LPR = D / 8, RPS = 64 / LPR, N = 4;
  const int lane = threadIdx.x & 63, r0 = lane / LPR, col = lane % LPR * 8;
  const float f = pow2_code(max(127 + old - s, 0));
  for (int r = r0; r < rows; r += N * RPS) {
    w_u32x2 x[N];
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (r + i * RPS < rows) x[i] = *(const w_u32x2 *)(base + (r + i * RPS) * tok + col);
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (r + i * RPS < rows) *(w_u32x2 *)(base + (r + i * RPS) * tok + col) = rescale8(x[i], f);
  }
}

template <typename E, int D> __device__ __forceinline__ void write_rows(const PagedWriteArgs &a, uint8_t *list, uint32_t *tops) {
  constexpr int LPR = D / 8, RPS = 64 / LPR, HOLD = 4;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int side = blockIdx.x % (2 * a.c.heads), head = side >> 1; // K or V of one head
  const bool isv = side & 1;
  const int64_t first = (int64_t)(blockIdx.x / (2 * a.c.heads)) * a.tile;
  const int P = a.c.page_size;
  const int64_t nslots = (int64_t)a.c.pages * P;
  const uint16_t *x = isv ? a.v + head * a.v_head : a.k + head * a.k_head;
  const int64_t x_tok = isv ? a.v_tok : a.k_tok, c_tok = isv ? a.c.v_tok : a.c.k_tok;
  const int64_t c_page = isv ? a.c.v_page : a.c.k_page, s_page = isv ? a.c.vs_page : a.c.ks_page;
  uint8_t *codes = isv ? a.c.v + head * a.c.v_head : a.c.k + head * a.c.k_head;
  uint8_t *scales = isv ? a.c.vs + head * a.c.vs_head : a.c.ks + head * a.c.ks_head;
  const int sub = lane / LPR, col = lane % LPR * 8;
  // a lane's offset from the first row of a step, in bytes; what else an address needs is the same for all lanes
  const uint32_t x_off = (uint32_t)(sub * (int32_t)x_tok + col) * 2, c_off = (uint32_t)(sub * (int32_t)c_tok + col);

  // the runs that begin in this tile: lane i looks at token first + i (every wavefront comes to the same answer)
  const int64_t tt = first + lane;
  int32_t slot = -1, in_page = 0, row_of = 0;
  bool leads = false, single = false, goes_on = false;
  if (lane < a.tile && tt < a.tokens) {
    slot = a.slots[tt];
    const int32_t prev = tt ? a.slots[tt - 1] : -1, next = tt + 1 < a.tokens ? a.slots[tt + 1] : -1;
    if (slot >= 0 && slot < nslots) {
      in_page = (int32_t)((uint32_t)slot / (uint32_t)P);
      const int r = row_of = slot - in_page * P;
      goes_on = r && tt && prev == slot - 1;
      leads = !goes_on;
      single = leads && !(r + 1 < P && next == slot + 1);
    }
  }
  uint64_t many = __ballot(leads && !single);
  const uint64_t ones = __ballot(single), rest = __ballot(goes_on);

  int at = 8; // the half of `tops` that the last shared run used
  for (int turn = 0; many; ++turn, many &= many - 1) {
    const int src = __builtin_ctzll(many);
    const int64_t t = first + src;
    const int32_t s0 = __builtin_amdgcn_readlane(slot, src);
    const int row = __builtin_amdgcn_readlane(row_of, src);
    const int64_t page = __builtin_amdgcn_readlane(in_page, src);
    // the run's tokens: those that go on behind it, past the tile's end if it reaches that
    int n = 1 + (src == 63 ? 0 : __builtin_ctzll(~(rest >> (src + 1))));
    while (src + n >= a.tile) {
      const bool on = row + n + lane < P && t + n + lane < a.tokens && a.slots[t + n + lane] == s0 + n + lane;
      const uint64_t off = ~__ballot(on);
      n += off ? __builtin_ctzll(off) : 64;
      if (off) break;
    }
    // a short run is one wavefront's, a long one all four's
    const bool shared = n > HOLD * RPS;
    if (!shared && (turn & 3) != wave) continue;
    at ^= shared ? 8 : 0;
    const int r0 = shared ? wave * HOLD * RPS : 0, stride = shared ? 4 * HOLD * RPS : HOLD * RPS;
    uint8_t *base = codes + page * c_page, *sp = scales + page * s_page;
    const uint8_t *xr = (const uint8_t *)(x + t * x_tok);
    // Rows r .. of the run, RPS a step.  What lies past its end stands for its last rows again, which leaves the maximum as it is:
    // branches around single loads had the compiler wait for three of them before the fourth (54.5 us instead of 48.4 for 38171 prompt tokens).
    auto load4 = [&](int r) {
      struct { w_u32x4 x[HOLD]; } h;
#pragma unroll
      for (int i = 0; i < HOLD; ++i) {
        const int at = min(r + i * RPS, n - 1);
        h.x[i] = *(const w_u32x4 *)(xr + at * x_tok * 2 + (at + sub < n ? x_off : (uint32_t)col * 2));
      }
      return h;
    };
    const int old = row ? *sp : 0;
    const auto first4 = load4(r0);
    uint32_t amax = 0;
#pragma unroll
    for (int i = 0; i < HOLD; ++i) amax = max(amax, top_of8(first4.x[i]));
    for (int b = r0 + stride; b < n; b += stride) {
      const auto h = load4(b);
#pragma unroll
      for (int i = 0; i < HOLD; ++i) amax = max(amax, top_of8(h.x[i]));
    }
    // the maximum over all lanes that share the run; where it is stored again, two shared runs later, every wavefront has
    // read it (there is a barrier between), so none is needed behind the stores of codes, which would wait for them
    auto over_run = [&](uint32_t m, int to) {
      m = max64(m);
      if (shared) {
        if (lane == 0) tops[to + wave] = m;
        __syncthreads();
        m = max(max(tops[to], tops[to + 1]), max(tops[to + 2], tops[to + 3]));
      }
      return (uint32_t)__builtin_amdgcn_readfirstlane((int)m);
    };
    amax = over_run(amax, at);
    const bool wild = amax >= E::kInfinite;
    if (wild) {
      amax = 0;
      for (int b = r0; b < n; b += stride) {
        const auto h = load4(b);
#pragma unroll
        for (int i = 0; i < HOLD; ++i) amax = max(amax, finite_top_of8<E>(h.x[i]));
      }
      amax = over_run(amax, at + 4);
    }
    const int need = scale_of_top<E>(amax), s = row ? max(need, __builtin_amdgcn_readfirstlane(old)) : need;
    if (row && s > old && (!shared || wave == 0)) rescale_rows<D>(base, c_tok, row, old, s);
    auto store4 = [&](int r, const w_u32x4 *h) {
#pragma unroll
      for (int i = 0; i < HOLD; ++i)
        if (r + i * RPS + sub < n) *(w_u32x2 *)(base + (row + r + i * RPS) * c_tok + c_off) = codes_of8<E>(h[i], s, wild);
    };
    store4(r0, first4.x);
    for (int b = r0 + stride; b < n; b += stride) { // a run longer than the registers is read twice
      const auto h = load4(b);
      store4(b, h.x);
    }
    if (lane == 0 && (!shared || wave == 0)) *sp = (uint8_t)s; // (every wavefront has read the old one: over_run's barrier)
  }

  // single tokens: list[i] = the lane that found the i-th
  if (single) list[wave * 64 + __builtin_amdgcn_mbcnt_hi((uint32_t)(ones >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)ones, 0))] = (uint8_t)lane;
  __builtin_amdgcn_wave_barrier();
  const int count = __builtin_popcountll(ones);
  for (int i0 = wave * RPS; i0 < count; i0 += 4 * RPS) {
    const bool mine = i0 + sub < count;
    const int src = mine ? list[wave * 64 + i0 + sub] : 0;
    const int row = __shfl(row_of, src);
    const int64_t page = __shfl(in_page, src);
    uint8_t *base = codes + page * c_page, *sp = scales + page * s_page;
    w_u32x4 v = {0, 0, 0, 0};
    int old = 0;
    if (mine) {
      v = *(const w_u32x4 *)(x + (first + src) * x_tok + col);
      if (row) old = *sp;
    }
    uint32_t amax = top_of8(v);
#pragma unroll
    for (int d = 1; d < LPR; d <<= 1) amax = max(amax, (uint32_t)__shfl_xor((int)amax, d));
    const bool wild = amax >= E::kInfinite;
    if (__any(wild)) {
      amax = finite_top_of8<E>(v);
#pragma unroll
      for (int d = 1; d < LPR; d <<= 1) amax = max(amax, (uint32_t)__shfl_xor((int)amax, d));
    }
    const int need = scale_of_top<E>(amax), s = row ? max(need, old) : need;
    uint64_t grown = __ballot(mine && row && need > old);
    while (grown) { // a group of lanes at a time
      const int l = __builtin_ctzll(grown);
      grown &= ~((LPR == 64 ? ~0ull : (1ull << LPR) - 1) << l);
      const int64_t pg = __builtin_amdgcn_readlane((int)page, l);
      rescale_rows<D>(codes + pg * c_page, c_tok, __builtin_amdgcn_readlane(row, l), __builtin_amdgcn_readlane(old, l),
                      __builtin_amdgcn_readlane(s, l));
    }
    if (mine) {
      *(w_u32x2 *)(base + row * c_tok + col) = codes_of8<E>(v, s, wild);
      if (col == 0) *sp = (uint8_t)s;
    }
  }
}

#define PAGED_WRITE(T, E, D)                                                                          \
  extern "C" __global__ __launch_bounds__(256, 6) void paged_write_##T##_d##D(PagedWriteArgs a) {      \
    __shared__ uint8_t list[256];                                                                     \
    __shared__ uint32_t tops[16];                                                                     \
    write_rows<E, D>(a, list, tops);                                                                     \
  }
} // namespace

PAGED_WRITE(bf16, Bf16, 64)
PAGED_WRITE(bf16, Bf16, 128)
PAGED_WRITE(bf16, Bf16, 256)
PAGED_WRITE(f16, Fp16, 64)
PAGED_WRITE(f16, Fp16, 128)
PAGED_WRITE(f16, Fp16, 256)
#undef PAGED_WRITE
extern "C" __global__ __launch_bounds__(256) void paged_write_any_bf16(PagedWriteArgs a) { write_any<Bf16>(a); }
extern "C" __global__ __launch_bounds__(256) void paged_write_any_f16(PagedWriteArgs a) { write_any<Fp16>(a); }

// ---------------------------------------------------------------------------
// attention, any shape
// ---------------------------------------------------------------------------
namespace {

// The sequence that owns packed row t, or -1: the last b with cu[b] <= t, if t is before its end.
__device__ __forceinline__ int owner_of(const int32_t *cu, int b, int32_t t) {
  int lo = 0, hi = b - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (cu[mid] <= t) lo = mid; else hi = mid - 1;
  }
  return cu[lo] <= t && t < cu[lo + 1] ? lo : -1;
}

// One wavefront per (row, query head): lane = key for the scores of 64 keys, lane = head dims lane, lane + 64, ... for
// the sum over V.  Any page size, strides and head dim up to 256; everything in fp32.  It runs only where the kernels below
// do not (71 ms for 6 sequences of 20000 to 131000 keys that take them 0.14).
template <typename E> __device__ __forceinline__ void attn_any(const PagedAttnArgs &a, float *qs, uint16_t (*to_out)(float)) {
  const int lane = threadIdx.x;
  const int t = blockIdx.x, hq = blockIdx.y, D = a.c.head_dim, P = a.c.page_size, hk = hq / a.group;
  const int b = owner_of(a.cu_q, a.b, t);
  if (b < 0) return;
  const int32_t len = min(max(a.lens[b], 0), (int32_t)min((int64_t)a.max_pages * P, (int64_t)INT32_MAX));
  // keys the query sees: all, or those up to its own position len - n_q + (t - cu)
  const int64_t last = a.causal ? (int64_t)len - ((int64_t)a.cu_q[b + 1] - t) : (int64_t)len - 1;
  for (int d = lane; d < D; d += 64) qs[d] = E::get(a.q[t * a.q_tok + hq * a.q_head + d]) * a.qk_scale;
  __syncthreads();
  const int32_t *table = a.table + b * a.table_stride;
  float m = -__builtin_inff(), l = 0.0f, acc[4] = {0, 0, 0, 0};
  for (int64_t k0 = 0; k0 <= last; k0 += 64) {
    const int64_t key = k0 + lane;
    int32_t page = -1;
    if (key <= last) page = table[key / P];
    const bool live = page >= 0 && page < a.c.pages;
    float s = -__builtin_inff(), vscale = 0.0f;
    if (live) {
      const uint8_t *kr = a.c.k + page * a.c.k_page + hk * a.c.k_head + (key % P) * a.c.k_tok;
      float dot = 0.0f;
      for (int d = 0; d < D; ++d) dot = fmaf(qs[d], __builtin_amdgcn_cvt_f32_fp8(kr[d], 0), dot);
      s = dot * pow2_code(a.c.ks[page * a.c.ks_page + hk * a.c.ks_head]);
      vscale = pow2_code(a.c.vs[page * a.c.vs_page + hk * a.c.vs_head]);
    }
    float top = s;
#pragma unroll
    for (int d = 32; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
    if (!__any(live)) continue;
    const float m_new = fmaxf(m, top), ref = m_new == -__builtin_inff() ? 0.0f : m_new;
    const float p = live ? __builtin_amdgcn_exp2f(s - ref) : 0.0f;
    const float alpha = __builtin_amdgcn_exp2f(m - ref);
    l = l * alpha + p;
    m = m_new;
#pragma unroll
    for (int r = 0; r < 4; ++r) acc[r] *= alpha;
    const int n = (int)min((int64_t)64, last - k0 + 1);
    for (int j = 0; j < n; ++j) {
      const int32_t pj = __shfl(page, j);
      if (pj < 0 || pj >= a.c.pages) continue;
      const float w = __shfl(p, j) * __shfl(vscale, j);
      const uint8_t *vr = a.c.v + pj * a.c.v_page + hk * a.c.v_head + ((k0 + j) % P) * a.c.v_tok;
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (lane + r * 64 < D) acc[r] = fmaf(w, __builtin_amdgcn_cvt_f32_fp8(vr[lane + r * 64], 0), acc[r]);
    }
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) l += __shfl_xor(l, d);
  const bool none = l == 0.0f && m == -__builtin_inff(); // no key, or no score above -inf
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (lane + r * 64 < D) a.o[t * a.o_tok + hq * a.o_head + lane + r * 64] = to_out(none ? 0.0f : acc[r] / l);
  if (a.lse && lane == 0) a.lse[(int64_t)t * a.heads_q + hq] = none ? -__builtin_inff() : m + __builtin_log2f(l);
}

__device__ __forceinline__ uint16_t out_bf16(float f) { return __builtin_bit_cast(uint16_t, (__bf16)f); }
__device__ __forceinline__ uint16_t out_f16(float f) { return __builtin_bit_cast(uint16_t, (_Float16)f); }

} // namespace

extern "C" __global__ __launch_bounds__(64) void paged_attn_any_bf16(PagedAttnArgs a) {
  __shared__ float qs[256];
  attn_any<Bf16>(a, qs, out_bf16);
}
extern "C" __global__ __launch_bounds__(64) void paged_attn_any_f16(PagedAttnArgs a) {
  __shared__ float qs[256];
  attn_any<Fp16>(a, qs, out_f16);
}

#include "paged_attn_one.h"
#include "paged_attn_rows.h"
