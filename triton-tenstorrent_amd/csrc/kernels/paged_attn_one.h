// Attention over the paged cache, few queries of a sequence: one (a decode step), or some (verification) as long as
// they and their heads fit 16 MT rows.
//
// What bounds it: one pass over the cached codes, HBM.  A wavefront owns all queries and query heads of one cache head
// (row r is query r / group, head r % group; empty rows of the MFMA tile cost nothing here) and streams keys from global memory
// into registers (6 sequences of 20000 to 131000 keys, 8 heads of 128, 782 MB: 131 us, 6.0 TB/s where a copy reaches 6.7; 48 of
// 60 to 8000 keys: 55 to 65 us from one set of inputs to another, at best 5.9 TB/s; the join 5 us), with no LDS between: every code is used once, by one wavefront.
//   S^T[key, r] = K . Q^T       v_mfma_f32_16x16x32, A = 16 rows of K, B = Q; lane l ends with row l%16, keys (l/16)*4+r
//   O^T[d, r]  += V^T . P^T     B = P^T is what the lane already holds; A = V^T, whose lane needs 8 keys of one d: it loads
//                               D/16 consecutive codes of each of its keys and pairs neighbouring keys' bytes with
//                               v_perm_b32, one for two conversions.  MFMA number i takes the lanes' i-th code, so its
//                               row l%16 stands for d = (l%16) * D/16 + i.
// e4m3 -> 16 bits is v_cvt_scalef32_pk_{bf16,f16}_fp8 (exact), K and V without their scales.  K's joins the factor on the
// scores.  V's, a power of two 2^(e - 127), joins the exponent: with x = score + e - 121 the weight w = 2^(x - ref) is what
// a key contributes relative to the row's largest contribution, the sum over V takes w and the sum of probabilities
// w 2^(121 - e).  So weights can be held in fp16 (11 bits where bf16 has 8): fp16 keeps all 11 down to 2^-22 of the largest
// contribution and nothing below 2^-32.  That is nothing beside it, but all that there is in a channel where the larger
// pages hold zeros.  So a sequence whose V scales a workgroup finds more than 2^kSpan apart (pages of ordinary values never
// are; within 2^12, 2^-21 are left) goes to a second pass, FAR: a weight is the sum of two bf16 there, which reach as far as
// fp32 does and leave 2^-16, and costs two products.
//
// Split: a group of workgroups, one for each cache head, takes an even share of the keys of all sequences, in units of
// 64 * NS keys, whatever the lengths.  (All heads of a page are read at about the same time, by neighbouring workgroups:
// their codes lie side by side.)  A workgroup meets at most two sequences that it does not have whole, the first and the
// last.  Those leave partial results (fp32 sum, reference, sum of probabilities) in the workspace and paged_attn_join adds them in order, so results do not change from run to run.  While a sequence's
// four wavefronts are merged, the next one's first loads are under way.
#pragma once

namespace one {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr float kLift = 8.0f;  // weights are held times 2^8: fp16 then reaches down to 2^-32 of the reference
constexpr float kLazy = 7.0f;  // the reference follows a row's maximum when that is 2^7 above it: at most 2^15 < 65504
constexpr int kBase = 121;     // scale code that leaves x = score: that of a page of magnitudes up to 4 .. 7
// what brings a page's weights back to probabilities, 2^(kBase - e)
__device__ __forceinline__ float unweight(int e) { return __builtin_bit_cast(float, (uint32_t)max(kBase + 127 - e, 1) << 23); }
constexpr float kOut = 0x1p-6f; // 2^(kBase - 127): V of scale code kBase
constexpr float kInf = __builtin_inff();
constexpr int kSpan = 12;      // see above

// A sum of probabilities times 2^d, d <= 0 (-inf: 0).  (2^d by itself would end at 2^-126, and a page of zeros, whose keys count
// like any others, can lie 2^220 below the largest page.)
__device__ __forceinline__ float lower(float l, float d) {
  d = fmaxf(d, -512.0f);
  const float n = floorf(d);
  return __builtin_amdgcn_ldexpf(l * __builtin_amdgcn_exp2f(d - n), (int)n);
}
// Sums l and k of references m and r, brought to ref, the larger of these, by the powers f and w; where a power is near the end
// of fp32, by lower().  (A row of NaN scores has reference -inf and a NaN sum: it has to stay, f and w are 1 there.)
__device__ __forceinline__ float add_sums(float l, float m, float f, float k, float r, float w, float ref) {
  if (__builtin_expect((m < ref - 100.0f && m != -kInf) || (r < ref - 100.0f && r != -kInf), 0))
    return (m == -kInf ? l : lower(l, m - ref)) + (r == -kInf ? k : lower(k, r - ref));
  return l * f + k * w;
}

// The smallest and the largest of V's scales that a wavefront has met; the same in all its lanes.
struct Span {
  int32_t low, high;
  __device__ __forceinline__ Span(int32_t l = 255, int32_t h = 0) : low(l), high(h) {}
  __device__ __forceinline__ void meet(int32_t live, int32_t vcode) {
    low = min(low, 255 - (int32_t)max64(live > 0 ? 255 - vcode : 0));
    high = max(high, (int32_t)max64(live > 0 ? vcode : 0));
  }
  __device__ __forceinline__ bool far() const { return high > low + kSpan; }
};

// Subtiles of 16 keys that a wavefront takes in one step.  Two leave room for three workgroups on a CU at head dim 128
// and make finer units than four (calls in a captured graph: 513 keys, 8 heads 8.6 us against 12.5; 48 sequences of 60 to 8000
// keys 73 against 94); at head dim 64 two would be too few bytes in flight.
template <int D, int MT> constexpr int subtiles() { return D * MT >= 128 ? 2 : 4; }

// Sequence b as this kernel sees it: no units where it is not this kernel's (no query, or too many).
struct Seq { int32_t q0, n, len, units; };
template <int UK, int ROWS, bool FEW> __device__ __forceinline__ Seq seq_of(const PagedAttnArgs &a, int b) {
  const int32_t q0 = clampi(a.cu_q[b], 0, a.tokens), q1 = clampi(a.cu_q[b + 1], q0, a.tokens);
  const int32_t len = clampi(a.lens[b], 0, a.max_pages * a.c.page_size), n = q1 - q0;
  const bool mine = FEW ? n > 0 && (int64_t)n * a.group <= ROWS : n == 1;
  return {q0, n, len, mine ? max((len + UK - 1) / UK, 1) : 0};
}

// Where the units of all sequences lie: every wavefront scans the lengths by itself, lane i the sequences i * per and
// up.  Up to 64 sequences stay in registers.
template <int UK, int ROWS, bool FEW> struct Walk {
  const PagedAttnArgs &a;
  int per;
  int32_t base, total;
  Seq own;
  __device__ __forceinline__ Walk(const PagedAttnArgs &args, int lane) : a(args) {
    per = (a.b + 63) / 64;
    int32_t n = 0;
    own = {0, 0, 0, 0};
    base = total = 0;
    if (a.whole) return;
    for (int b = min(lane * per, a.b); b < min(lane * per + per, a.b); ++b) {
      own = seq_of<UK, ROWS, FEW>(a, b);
      n += own.units;
    }
    int32_t v = n;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int32_t o = __shfl_up(v, d);
      if (lane >= d) v += o;
    }
    base = v - n;
    total = __builtin_amdgcn_readlane(v, 63);
  }
  __device__ __forceinline__ Seq at(int b) const {
    if (per != 1) return seq_of<UK, ROWS, FEW>(a, b);
    return {__builtin_amdgcn_readlane(own.q0, b), __builtin_amdgcn_readlane(own.n, b), __builtin_amdgcn_readlane(own.len, b),
            __builtin_amdgcn_readlane(own.units, b)};
  }
  // the sequence that holds unit u, and the units before it
  __device__ __forceinline__ int find(int32_t u, int32_t *before, Seq *sq) const {
    const int l = 63 - __builtin_clzll(__ballot(base <= u));
    int b = l * per;
    *before = __builtin_amdgcn_readlane(base, l);
    *sq = at(b);
    step(u, &b, before, sq);
    return b;
  }
  __device__ __forceinline__ void step(int32_t u, int *b, int32_t *before, Seq *sq) const {
    while (*before + sq->units <= u) { // (u is less than all units: ends before the sequences do)
      *before += sq->units;
      *sq = at(++*b);
    }
  }
};

struct Bf {
  typedef bf16x8 frag;
  static __device__ __forceinline__ f32x4 mfma(frag x, frag y, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, y, c, 0, 0, 0); }
  static __device__ __forceinline__ f32x16 mfma32(frag x, frag y, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, y, c, 0, 0, 0); }
  static __device__ __forceinline__ frag codes(uint32_t lo, uint32_t hi) {
    const u32x4 r = {__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true))};
    return __builtin_bit_cast(frag, r);
  }
  template <bool HI> static __device__ __forceinline__ uint32_t codes2(uint32_t x) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.0f, HI));
  }
  static __device__ __forceinline__ uint16_t out(float f) { return out_bf16(f); }
};
struct Hf {
  typedef f16x8 frag;
  static __device__ __forceinline__ f32x4 mfma(frag x, frag y, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(x, y, c, 0, 0, 0); }
  static __device__ __forceinline__ f32x16 mfma32(frag x, frag y, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(x, y, c, 0, 0, 0); }
  static __device__ __forceinline__ frag codes(uint32_t lo, uint32_t hi) {
    const u32x4 r = {__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true))};
    return __builtin_bit_cast(frag, r);
  }
  template <bool HI> static __device__ __forceinline__ uint32_t codes2(uint32_t x) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 1.0f, HI));
  }
  static __device__ __forceinline__ uint16_t out(float f) { return out_f16(f); }
};
// What V and its weights are held in
template <bool FAR> struct Weights { typedef Hf type; };
template <> struct Weights<true> { typedef Bf type; };

// Codes are read once: non-temporal loads where a row is whole 128-byte lines (782 MB of cache, head dim 128, a call
// in a captured graph: 162 -> 155 us; head dim 64, whose lines two rows share: no gain).
template <int D, typename T> __device__ __forceinline__ T stream(const T *p) {
  if constexpr (D >= 128) return __builtin_nontemporal_load(p);
  return *p;
}
__device__ __forceinline__ int64_t lane64(int32_t lo, int32_t hi, int lane) {
  return (int64_t)(((uint64_t)(uint32_t)__builtin_amdgcn_readlane(hi, lane) << 32) | (uint32_t)__builtin_amdgcn_readlane(lo, lane));
}

// The kernel's argument block as a function that is called (not inlined) gets at it, and its wavefront's own values.
typedef __attribute__((address_space(3))) uint8_t *Lds;
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ PagedAttnArgs args_at(uint64_t p) {
  return *(const __attribute__((address_space(4))) PagedAttnArgs *)((uint64_t)(uint32_t)uniform((int)(p >> 32)) << 32 | (uint32_t)uniform((int)p));
}

// Partial result p of the workspace: rows * D sums, then rows pairs (reference, sum).
template <int D, int MT> constexpr int part_floats() { return 16 * MT * D + 32 * MT; }

// A sequence that is split and whose first units are workgroup i's, for that workgroup's head: the i-th entry behind the
// partial results.  Its parts are slot 2 i + slot of workgroup i, then slot 2 j of the `more` workgroups j = i + heads, ...
struct Split { int32_t q0, more, slot, rows; }; // q0: first packed row of its queries, -1 = none; rows: queries times group

// FEW: sequences may have several queries; without it exactly one, and nothing below looks at a row's own limit.
// Returns whether a sequence was left to FAR, which computes those and passes over the others.
template <class E, int D, int MT, bool FEW, bool FAR>
__device__ __forceinline__ bool body(const PagedAttnArgs &a, float *lds, int wg, int wgs, int tid) {
  typedef typename Weights<FAR>::type W;
  constexpr int NS = subtiles<D, MT>(), UK = 64 * NS, KL = D / 64, VW = D / 64; // 16-byte loads of K, dwords of V per row
  constexpr int VB = D / 16, IB = 64 / NS, LD = D + 4;                      // LD: padded LDS row of the merge
  const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c16 = lane & 15, g = lane >> 4;
  const Walk<UK, 16 * MT, FEW> walk(a, lane);
  Split *split = (Split *)(a.part + 2 * (int64_t)wgs * part_floats<D, MT>()) + wg;
  const int hk = wg % a.c.heads, group = wg / a.c.heads;
  int32_t u, u_end, before;
  int32_t each = 1, extra = 0; // units of a group; the first `extra` groups have one more
  Seq sq;
  int b;
  if (a.whole) { // one sequence each
    b = group;
    sq = seq_of<UK, 16 * MT, FEW>(a, b);
    if (sq.units == 0) return false;
    before = u = 0;
    u_end = sq.units;
  } else {
    const int32_t groups = min(wgs / a.c.heads, walk.total); // fewer units than groups: one each
    if (group >= groups) {
      if (!FAR && a.part && tid == 0) split->q0 = -1;
      return false;
    }
    each = walk.total / groups;
    extra = walk.total - each * groups;
    u = group * each + min(group, extra);
    u_end = u + each + (group < extra);
    b = walk.find(u, &before, &sq);
  }
  const int32_t u_first = u;
  bool noted = false, again = false;
  int32_t *spans = (int32_t *)(lds + 4 * 16 * MT * LD + 4 * 16 * MT * 2); // [wave]: low, high
  const uint8_t *kh = a.c.k + hk * a.c.k_head, *vh = a.c.v + hk * a.c.v_head;

  const uint32_t klane = (uint32_t)(c16 * a.c.k_tok + g * 16);
  uint32_t vlane[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) vlane[r] = (uint32_t)((g * 4 + r) * a.c.v_tok + c16 * VB);

  // the sequence at u: units c0 .. c0 + n of its sq.units
  int c0, n;
  int32_t limit[MT]; // last key that the lane's row attends
  const int32_t *table;
  typename E::frag qf[MT][2 * KL];

  // What lane (it % IB) * NS + s knows of subtile s of step it: where its rows lie, how many count, its scales.
  int32_t ko_lo, ko_hi, vo_lo, vo_hi, live, vcode;
  float kscale;
  auto batch = [&](int it0) {
    const int64_t key = (int64_t)(c0 + it0 + lane / NS) * UK + wave * (16 * NS) + (lane % NS) * 16;
    const uint32_t sub = (uint32_t)(key >> 4);
    const uint32_t blk = (uint32_t)(((uint64_t)sub * a.page_magic) >> 36);
    int32_t page = key < sq.len ? table[blk] : -1;
    const bool ok = page >= 0 && page < a.c.pages;
    page = ok ? page : 0;
    const int64_t row = ok ? ((int64_t)sub - (int64_t)blk * (a.c.page_size >> 4)) * 16 : 0;
    const int64_t ko = page * a.c.k_page + row * a.c.k_tok, vo = page * a.c.v_page + row * a.c.v_tok;
    ko_lo = (int32_t)ko; ko_hi = (int32_t)(ko >> 32); vo_lo = (int32_t)vo; vo_hi = (int32_t)(vo >> 32);
    live = ok ? (int32_t)min((int64_t)sq.len - key, (int64_t)16) : 0;
    kscale = pow2_code(a.c.ks[page * a.c.ks_page + hk * a.c.ks_head]) * a.qk_scale;
    vcode = ok ? a.c.vs[page * a.c.vs_page + hk * a.c.vs_head] : 0;
  };

  // the whole workgroup's span is wide (behind a barrier)
  auto far_spans = [&]() {
    const int32_t low = min(min(spans[0], spans[2]), min(spans[4], spans[6])), high = max(max(spans[1], spans[3]), max(spans[5], spans[7]));
    return high > low + kSpan;
  };
  auto put_span = [&](const Span &x) {
    if (lane == 0) { spans[wave * 2] = x.low; spans[wave * 2 + 1] = x.high; }
  };
  // the wavefront's span, with the batch at hand (in LDS: nothing of it is held during the loop over keys)
  auto widen_span = [&]() {
    Span x(spans[wave * 2], spans[wave * 2 + 1]);
    x.meet(live, vcode);
    put_span(x);
  };

  u32x4 kr[NS][KL];
  uint32_t vr[NS][4][VW];
  auto load_k = [&](int it) {
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      const uint8_t *kp = kh + lane64(ko_lo, ko_hi, (it % IB) * NS + s);
#pragma unroll
      for (int h = 0; h < KL; ++h) kr[s][h] = stream<D>((const u32x4 *)(kp + klane + h * 64));
    }
  };
  auto load_v = [&](int it) {
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      const uint8_t *vp = vh + lane64(vo_lo, vo_hi, (it % IB) * NS + s);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if constexpr (VW == 1) vr[s][r][0] = stream<D>((const uint32_t *)(vp + vlane[r]));
        if constexpr (VW == 2) {
          const u32x2 x = stream<D>((const u32x2 *)(vp + vlane[r]));
          vr[s][r][0] = x[0]; vr[s][r][1] = x[1];
        }
        if constexpr (VW == 4) {
          const u32x4 x = stream<D>((const u32x4 *)(vp + vlane[r]));
          vr[s][r][0] = x[0]; vr[s][r][1] = x[1]; vr[s][r][2] = x[2]; vr[s][r][3] = x[3];
        }
      }
    }
  };

  // one set of registers each for K and V: a step's loads go out as soon as the step before has used them up
  bool skip = false; // FAR: a sequence that the first pass has done
  auto open = [&]() {
    c0 = u - before;
    n = min(sq.units - c0, u_end - u);
    table = a.table + (int64_t)b * a.table_stride;
    if constexpr (FAR) {
      Span span;
      for (int it = 0; it < n; it += IB) {
        batch(it);
        span.meet(live, vcode);
      }
      __syncthreads();
      put_span(span);
      __syncthreads();
      skip = !__builtin_amdgcn_readfirstlane(far_spans());
      if (skip) return;
    }
    batch(0);
    if constexpr (!FAR) {
      load_k(0);
      load_v(0);
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int row = m * 16 + c16, i = FEW ? min(row / a.group, sq.n - 1) : 0;
      limit[m] = a.causal ? sq.len - sq.n + i : sq.len - 1;
      const uint16_t *qr = a.q + (sq.q0 + i) * a.q_tok + (hk * a.group + (FEW ? row % a.group : row)) * a.q_head + g * 16;
#pragma unroll
      for (int s = 0; s < 2 * KL; ++s) {
        u32x4 z = {0, 0, 0, 0};
        if (row < (FEW ? sq.n * a.group : a.group)) z = *(const u32x4 *)(qr + (s >> 1) * 64 + (s & 1) * 8);
        qf[m][s] = __builtin_bit_cast(typename E::frag, z);
      }
    }
  };
  open();
  for (;;) {
    if (skip) {
      u += n;
      if (u >= u_end) break;
      walk.step(u, &b, &before, &sq);
      open();
      continue;
    }
    if constexpr (!FAR) { // (while the first keys are on their way)
      Span span;
      span.meet(live, vcode);
      put_span(span);
    }
    f32x4 acc[MT][VB];
    float mref[MT], lsum[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      mref[m] = -kInf;
      lsum[m] = 0.0f;
#pragma unroll
      for (int i = 0; i < VB; ++i) acc[m][i] = (f32x4){0, 0, 0, 0};
    }
    for (int it = 0; it < n; ++it) {
      if constexpr (FAR) { // (nothing ahead: no more registers than the first pass has)
        if (it > 0 && it % IB == 0) batch(it);
        load_k(it);
        load_v(it);
      }
      int nv[NS], vc[NS];
      float ks[NS];
      int nmin = 16;
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        const int src = (it % IB) * NS + s;
        nv[s] = __builtin_amdgcn_readlane(live, src);
        vc[s] = __builtin_amdgcn_readlane(vcode, src);
        ks[s] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, kscale), src));
        nmin = min(nmin, nv[s]);
      }
      // scores
      f32x4 st[MT][NS];
#pragma unroll
      for (int s = 0; s < NS; ++s) {
#pragma unroll
        for (int m = 0; m < MT; ++m) st[m][s] = (f32x4){0, 0, 0, 0};
#pragma unroll
        for (int h = 0; h < KL; ++h)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const typename E::frag kf = E::codes(kr[s][h][2 * c], kr[s][h][2 * c + 1]);
#pragma unroll
            for (int m = 0; m < MT; ++m) st[m][s] = E::mfma(kf, qf[m][h * 2 + c], st[m][s]);
          }
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int r = 0; r < 4; ++r) st[m][s][r] = fmaf(st[m][s][r], ks[s], (float)(vc[s] - kBase));
      }
      if (!FAR && it + 1 < n) {
        if ((it + 1) % IB == 0) {
          if (it >= IB) widen_span(); // (not right behind its loads)
          batch(it + 1);
        }
        load_k(it + 1);
      }
      // keys behind the end or on no page, and those that some row does not attend
      const int32_t key0 = (c0 + it) * UK + wave * (16 * NS);
      const bool edge = FEW && a.causal && key0 + 16 * NS - 1 > sq.len - sq.n;
      bool nan = false;
      if (nmin < 16 || edge) {
        uint32_t any = 0;
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const bool in = g * 4 + r < nv[s];
#pragma unroll
            for (int m = 0; m < MT; ++m) st[m][s][r] = in && (!FEW || key0 + s * 16 + g * 4 + r <= limit[m]) ? st[m][s][r] : -kInf;
#pragma unroll
            for (int w = 0; w < VW; ++w) { // (what lies in dead rows may be NaN)
              vr[s][r][w] = in ? vr[s][r][w] : 0;
              if (FEW) any |= (vr[s][r][w] & 0x7f7f7f7fu) + 0x01010101u;
            }
          }
        // a NaN in V of a key that some row does not attend must not reach that row
        nan = edge && sq.n > 1 && __any((any & 0x80808080u) != 0);
      }
      // the reference
      float top[MT];
      bool grow = false;
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        top[m] = -kInf;
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
          for (int r = 0; r < 4; ++r) top[m] = fmaxf(top[m], st[m][s][r]);
        grow |= top[m] > mref[m] + kLazy;
      }
      if (__any(grow)) {
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          float x = fmaxf(top[m], __shfl_xor(top[m], 16));
          x = fmaxf(x, __shfl_xor(x, 32));
          const float mn = fmaxf(mref[m], x);
          const float al = mn == -kInf ? 1.0f : __builtin_amdgcn_exp2f(mref[m] - mn);
          lsum[m] = !FAR ? lsum[m] * al : mn == -kInf ? lsum[m] : lower(lsum[m], mref[m] - mn);
          mref[m] = mn;
#pragma unroll
          for (int i = 0; i < VB; ++i) acc[m][i] *= al;
        }
      }
      typename W::frag pf[MT][NS / 2];
      [[maybe_unused]] typename W::frag rest[MT][NS / 2]; // FAR: what rounding to pf took away
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const float ref = (mref[m] == -kInf ? 0.0f : mref[m]) - kLift;
#pragma unroll
        for (int s = 0; s < NS; ++s) {
          float w[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            w[r] = __builtin_amdgcn_exp2f(st[m][s][r] - ref);
            if constexpr (FAR) {
              const __bf16 h = (__bf16)w[r];
              pf[m][s >> 1][(s & 1) * 4 + r] = h;
              rest[m][s >> 1][(s & 1) * 4 + r] = (__bf16)(w[r] - (float)h);
              lsum[m] += __builtin_amdgcn_exp2f(st[m][s][r] - ref + (float)(kBase - vc[s])); // (w can be too small for fp32, the probability is not)
            } else {
              pf[m][s >> 1][(s & 1) * 4 + r] = (_Float16)w[r];
            }
          }
          if constexpr (!FAR) lsum[m] = fmaf((w[0] + w[1]) + (w[2] + w[3]), unweight(vc[s]), lsum[m]);
        }
      }
      // the sum over V
#pragma unroll
      for (int p = 0; p < NS / 2; ++p)
#pragma unroll
        for (int w = 0; w < VW; ++w) {
          uint32_t f[4][4]; // [code of the dword][pair of keys]
#pragma unroll
          for (int j = 0; j < 4; ++j) { // pairs: rows 0-1 and 2-3 of subtile 2p, then of 2p + 1
            const int s = 2 * p + (j >> 1), r = (j & 1) * 2;
            const uint32_t x = __builtin_amdgcn_perm(vr[s][r + 1][w], vr[s][r][w], 0x05010400);
            const uint32_t y = __builtin_amdgcn_perm(vr[s][r + 1][w], vr[s][r][w], 0x07030602);
            f[0][j] = W::template codes2<false>(x);
            f[1][j] = W::template codes2<true>(x);
            f[2][j] = W::template codes2<false>(y);
            f[3][j] = W::template codes2<true>(y);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            typedef typename W::frag frag;
            frag x = __builtin_bit_cast(frag, (u32x4){f[i][0], f[i][1], f[i][2], f[i][3]});
            if (FEW && __builtin_expect(nan, 0)) { // the sum runs without NaN, another product counts those that a row attends
              frag y;
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                const bool bad = x[j] != x[j];
                y[j] = bad ? 1.0f : 0.0f;
                x[j] = bad ? 0.0f : (float)x[j];
              }
#pragma unroll
              for (int m = 0; m < MT; ++m) {
                frag sees;
#pragma unroll
                for (int j = 0; j < 8; ++j) sees[j] = key0 + (2 * p + (j >> 2)) * 16 + g * 4 + (j & 3) <= limit[m] ? 1.0f : 0.0f;
                const f32x4 bad = W::mfma(y, sees, (f32x4){0, 0, 0, 0});
#pragma unroll
                for (int r = 0; r < 4; ++r)
                  if (bad[r] > 0.0f) acc[m][w * 4 + i][r] = __builtin_nanf("");
              }
            }
#pragma unroll
            for (int m = 0; m < MT; ++m) {
              if constexpr (FAR) acc[m][w * 4 + i] = W::mfma(x, rest[m][p], acc[m][w * 4 + i]);
              acc[m][w * 4 + i] = W::mfma(x, pf[m][p], acc[m][w * 4 + i]);
            }
          }
        }
      if (!FAR && it + 1 < n) load_v(it + 1);
    }

    // ---- the next sequence's loads, then the merge of the four wavefronts ----
    if (!FAR && n > IB) widen_span();
    const int32_t q0 = sq.q0, rows = FEW ? sq.n * a.group : a.group;
    const bool whole = n == sq.units;
    // (the first sequence of this workgroup takes slot 0, a later one that is not whole can only be its last: slot 1)
    const int which = u == u_first ? 0 : 1;
    if (!FAR && !whole && c0 == 0) {
      const int32_t last = before + sq.units - 1, larger = extra * (each + 1); // its last unit, and the group that has that
      const int32_t owner = last < larger ? last / (each + 1) : extra + (last - larger) / each;
      if (tid == 0) *split = {q0, owner - group, which, rows};
      noted = true;
    }
    u += n;
    const bool more = u < u_end;
    if (more) {
      walk.step(u, &b, &before, &sq);
      open();
    }
    float *wo = lds, *wml = lds + 4 * 16 * MT * LD;   // sums [wave][row][LD], (reference, sum) [wave][row]
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      float l = lsum[m];
      l += __shfl_xor(l, 16);
      l += __shfl_xor(l, 32);
      const int row = wave * 16 * MT + m * 16 + c16;
      if (g == 0) { wml[row * 2] = mref[m]; wml[row * 2 + 1] = l; }
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int i = 0; i < VB; i += 4)
          *(f32x4 *)(wo + row * LD + (g * 4 + r) * VB + i) = (f32x4){acc[m][i][r], acc[m][i + 1][r], acc[m][i + 2][r], acc[m][i + 3][r]};
    }
    __syncthreads();
    float *slot = a.part + (2 * (int64_t)wg + which) * part_floats<D, MT>();
    const bool left = !FAR && far_spans();
    again |= left;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int row = m * 16 + (tid >> 4), d0 = (tid & 15) * VB;
      float mx = -kInf;
#pragma unroll
      for (int w = 0; w < 4; ++w) mx = fmaxf(mx, wml[(w * 16 * MT + row) * 2]);
      const float mm = mx == -kInf ? 0.0f : mx;
      float l = 0.0f, o[VB];
#pragma unroll
      for (int i = 0; i < VB; ++i) o[i] = 0.0f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float mw = wml[(w * 16 * MT + row) * 2];
        const float f = mw == -kInf ? 1.0f : __builtin_amdgcn_exp2f(mw - mm); // (a row of NaN scores has reference -inf)
        const float lw = wml[(w * 16 * MT + row) * 2 + 1];
        l += !FAR ? lw * f : mw == -kInf ? lw : lower(lw, mw - mm);
#pragma unroll
        for (int i = 0; i < VB; ++i) o[i] += wo[(w * 16 * MT + row) * LD + d0 + i] * f;
      }
      if (whole) {
        if (row < rows && !left) {
          const int64_t t = q0 + (FEW ? row / a.group : 0);
          const int hq = hk * a.group + (FEW ? row % a.group : row);
          const bool none = l == 0.0f && mx == -kInf;
          const float inv = none ? 0.0f : kOut / l;
          uint16_t *op = a.o + t * a.o_tok + hq * a.o_head + d0;
#pragma unroll
          for (int i = 0; i < VB; i += 2)
            *(uint32_t *)(op + i) = (uint32_t)E::out(o[i] * inv) |
                                    (uint32_t)E::out(o[i + 1] * inv) << 16;
          if (a.lse && d0 == 0) a.lse[t * a.heads_q + hq] = none ? -kInf : mx - kLift + __builtin_log2f(l);
        }
      } else if (!left) {
#pragma unroll
        for (int i = 0; i < VB; i += 4) *(f32x4 *)(slot + row * D + d0 + i) = (f32x4){o[i], o[i + 1], o[i + 2], o[i + 3]};
        if (d0 == 0) {
          slot[16 * MT * D + row * 2] = mx;
          slot[16 * MT * D + row * 2 + 1] = l;
        }
      }
    }
    if (!more) break;
    __syncthreads();
  }
  if (!FAR && a.part && !noted && tid == 0) split->q0 = -1;
  return __builtin_amdgcn_readfirstlane(again);
}
// (a function of its own, out of the first pass's register allocation: inlined, 48 sequences of 60 to 8000 keys took 73 us instead of 69)
// OCC, workgroups on a CU, keeps apart the functions of kernels that may use more registers.
template <class E, int D, int MT, bool FEW, int OCC>
__device__ __attribute__((noinline)) void far_pass(uint64_t args, Lds lds, int wg, int wgs) {
  const PagedAttnArgs a = args_at(args);
  body<E, D, MT, FEW, true>(a, (float *)lds, uniform(wg), uniform(wgs), threadIdx.x);
}
template <class E, int D, int MT, bool FEW, int OCC>
__device__ __forceinline__ void both(const PagedAttnArgs &a, float *lds, int wg, int wgs) {
  { // One word of each line of the arguments, asked for at once: with a call in the kernel the compiler loads them in three
    // or four turns, each a wait for memory otherwise (62 rows over 16 encoder states: 20.3 us instead of 19.3).
    static_assert(sizeof(PagedAttnArgs) > 64 * 4, "a word of the fifth line");
    const __attribute__((address_space(4))) uint32_t *p = (const __attribute__((address_space(4))) uint32_t *)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" :: "s"(p[0]), "s"(p[16]), "s"(p[32]), "s"(p[48]), "s"(p[64]));
  }
  if (__builtin_expect(body<E, D, MT, FEW, false>(a, lds, wg, wgs, threadIdx.x), 0)) {
    __syncthreads();
    far_pass<E, D, MT, FEW, OCC>((uint64_t)__builtin_amdgcn_kernarg_segment_ptr(), (Lds)lds, wg, wgs);
  }
}

// Adds the parts of the split sequence that workgroup wg of the launch before noted, if any: one of `join_pieces` pieces
// of its rows.  D / 4 threads a row; what is left of the 256 takes several rows or several parts at once.
template <class E, int D, int MT> __device__ __forceinline__ void join(const PagedAttnArgs &a, f32x4 *lds, int wg, int piece, int wgs) {
  constexpr int TPR = D / 4, SLOTS = 256 / TPR, PF = part_floats<D, MT>();
  const Split sp = ((const Split *)(a.part + 2 * (int64_t)wgs * PF))[wg];
  if (sp.q0 < 0) return;
  const int tid = threadIdx.x, d4 = tid % TPR, at = tid / TPR;
  const int share = (sp.rows + a.join_pieces - 1) / a.join_pieces, row_end = min((piece + 1) * share, sp.rows); // this piece's rows
  int across = 1; // rows at once
  while (across < SLOTS && across < share) across <<= 1;
  const int deep = SLOTS / across, r0 = at % across, p0 = at / across;
  const int parts = sp.more + 1, head = wg % a.c.heads;
  const float *first = a.part + (2 * (int64_t)wg + sp.slot) * PF, *later = a.part + 2 * (int64_t)wg * PF;
  float *lm = (float *)(lds + 256), *ll = lm + 256;
  for (int rb = piece * share; rb < row_end; rb += across) {
    const int row = min(rb + r0, 16 * MT - 1);
    float m = -kInf, l = 0.0f;
    f32x4 o = {0, 0, 0, 0};
    for (int p = p0; p < parts; p += 4 * deep) {
      float pm[4], pl[4];
      f32x4 po[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int j = min(p + i * deep, parts - 1);
        const float *x = j ? later + 2 * (int64_t)j * a.c.heads * PF : first;
        pm[i] = x[16 * MT * D + row * 2];
        pl[i] = x[16 * MT * D + row * 2 + 1];
        po[i] = *(const f32x4 *)(x + row * D + d4 * 4);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (p + i * deep >= parts) break;
        const float mn = fmaxf(m, pm[i]), ref = mn == -kInf ? 0.0f : mn;
        const float f = m == -kInf ? 1.0f : __builtin_amdgcn_exp2f(m - ref), w = pm[i] == -kInf ? 1.0f : __builtin_amdgcn_exp2f(pm[i] - ref);
        l = add_sums(l, m, f, pl[i], pm[i], w, ref);
        o = o * f + po[i] * w;
        m = mn;
      }
    }
    if (deep > 1) {
      lds[tid] = o;
      lm[tid] = m;
      ll[tid] = l;
      __syncthreads();
      if (p0 == 0)
        for (int q = 1; q < deep; ++q) {
          const int y = tid + q * across * TPR;
          const float mn = fmaxf(m, lm[y]), ref = mn == -kInf ? 0.0f : mn;
          const float f = m == -kInf ? 1.0f : __builtin_amdgcn_exp2f(m - ref), w = lm[y] == -kInf ? 1.0f : __builtin_amdgcn_exp2f(lm[y] - ref);
          l = add_sums(l, m, f, ll[y], lm[y], w, ref);
          o = o * f + lds[y] * w;
          m = mn;
        }
      __syncthreads();
    }
    if (p0 == 0 && rb + r0 < row_end) {
      const int64_t t = sp.q0 + row / a.group;
      const int hq = head * a.group + row % a.group;
      const bool none = l == 0.0f && m == -kInf;
      const float inv = none ? 0.0f : kOut / l;
      *(u32x2 *)(a.o + t * a.o_tok + hq * a.o_head + d4 * 4) =
          (u32x2){(uint32_t)E::out(o[0] * inv) | (uint32_t)E::out(o[1] * inv) << 16, (uint32_t)E::out(o[2] * inv) | (uint32_t)E::out(o[3] * inv) << 16};
      if (a.lse && d4 == 0) a.lse[t * a.heads_q + hq] = none ? -kInf : m - kLift + __builtin_log2f(l);
    }
  }
}

template <int D, int MT> constexpr int lds_floats() { return 4 * 16 * MT * (D + 4) + 4 * 16 * MT * 2 + 8; }

} // namespace one

#define PAGED_ONE(T, E, D, MT, OCC)                                                                           \
  extern "C" __global__ __launch_bounds__(256, OCC) void paged_attn_one_##T##_d##D##_r##MT(PagedAttnArgs a) {  \
    __shared__ __align__(16) float lds[one::lds_floats<D, MT>()];                                             \
    one::both<one::E, D, MT, false, OCC>(a, lds, blockIdx.x, gridDim.x);                                      \
  }                                                                                                           \
  extern "C" __global__ __launch_bounds__(256, 2) void paged_attn_few_##T##_d##D##_r##MT(PagedAttnArgs a) {    \
    __shared__ __align__(16) float lds[one::lds_floats<D, MT>()];                                             \
    one::both<one::E, D, MT, true, 2>(a, lds, blockIdx.x, gridDim.x);                                         \
  }                                                                                                           \
  extern "C" __global__ __launch_bounds__(256) void paged_attn_join_##T##_d##D##_r##MT(PagedAttnArgs a) {      \
    __shared__ one::f32x4 lds[256 + 128];                                                                     \
    one::join<one::E, D, MT>(a, lds, blockIdx.x / a.join_pieces, blockIdx.x % a.join_pieces, gridDim.x / a.join_pieces); \
  }
// (the last number: workgroups of paged_attn_one on a CU, which the host's grid counts on too; paged_attn_few has two)
PAGED_ONE(bf16, Bf, 64, 1, 3)
PAGED_ONE(bf16, Bf, 64, 2, 3)
PAGED_ONE(bf16, Bf, 128, 1, 3)
PAGED_ONE(bf16, Bf, 128, 2, 2)
PAGED_ONE(bf16, Bf, 256, 1, 2)
PAGED_ONE(f16, Hf, 64, 1, 3)
PAGED_ONE(f16, Hf, 64, 2, 3)
PAGED_ONE(f16, Hf, 128, 1, 3)
PAGED_ONE(f16, Hf, 128, 2, 2)
PAGED_ONE(f16, Hf, 256, 1, 2)
#undef PAGED_ONE
