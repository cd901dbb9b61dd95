// Attention over the paged cache, several queries of a sequence (prompts, pieces of prompts, verification).
//
// A workgroup owns 128 rows of one (sequence, cache head): row r is query r / group, query head r % group of the head's
// group, so that the heads that share keys share the keys' conversion and LDS tile.  Each of its four wavefronts has 32
// rows and computes both products transposed, so that a row's statistics stay in the two lanes that own it:
//   S^T[key, row] = K . Q^T      v_mfma_f32_32x32x16, A = 32 rows of K, B = Q
//   O^T[d, row]  += V^T . P^T    A = V^T, B = P^T straight from the registers of S^T
// Keys come in tiles of 64.  Wavefront w stages the tile's 16 keys 16 w .. 16 w + 15 (they share a page): codes are loaded
// two tiles ahead, turned to 16 bits on the way into LDS, V transposed there (v_perm_b32 pairs neighbouring keys' bytes
// before the conversion, as in paged_attn_one.h), K and V without their scales, which join the scores as there.  LDS
// holds two tiles; one barrier a tile.
// Bound: instruction issue.  7169 prompt tokens, 32 heads of 128 over 8: 250 us, 848 TFLOP/s (a large product reaches 1593; both
// vary by 6 % from one machine to another); the
// MFMA pipes are busy a third of the time, an instruction is issued in 82 % of the cycles (exponentials, conversions,
// staging).  Two workgroups on a CU, so that one's softmax runs beside the other's products; one wavefront a SIMD with
// twice the rows moves its accumulators between the register files (488 us).
//
// Split: with row tiles enough to fill the chip twice, a workgroup takes one, late rows (which attend most keys) first.
// With fewer, a group of workgroups, one for each cache head, takes an even share of the steps of all row tiles, and
// paged_attn_rows_join adds the parts of those that were cut, as in paged_attn_one.h.
#pragma once

namespace rows {

using one::kBase;
using one::kInf;
using one::kLazy;
using one::kLift;
using one::kOut;
using one::unweight;
using one::u32x2;
using one::u32x4;
using one::f32x16;
using one::f32x4;
using one::Bf;
using one::Hf;

constexpr int kRows = 128;

struct Seq { int32_t q0, n, len, tiles; }; // first packed row, queries, keys, tiles of 128 rows
__device__ __forceinline__ Seq seq_of(const PagedAttnArgs &a, int b) {
  const int32_t q0 = clampi(a.cu_q[b], 0, a.tokens), q1 = clampi(a.cu_q[b + 1], q0, a.tokens);
  const int32_t n = (int64_t)(q1 - q0) * a.group > a.few_rows ? q1 - q0 : 0; // fewer are the other kernel's
  return {q0, n, clampi(a.lens[b], 0, a.max_pages * a.c.page_size), (int32_t)(((int64_t)n * a.group + kRows - 1) / kRows)};
}

// Last key that query i of the sequence attends (-1: none).
__device__ __forceinline__ int32_t last_key(const PagedAttnArgs &a, const Seq &sq, int32_t i) {
  return a.causal ? max(sq.len - sq.n + i, -1) : sq.len - 1;
}

// A tile's steps of 64 keys: one at least, so that rows without a key are written too.
__device__ __forceinline__ int steps_of(const PagedAttnArgs &a, const Seq &sq, int tile) {
  const int32_t r1 = (int32_t)min((int64_t)(tile + 1) * kRows, (int64_t)sq.n * a.group) - 1;
  return max((last_key(a, sq, r1 / a.group) + 64) / 64, 1);
}

__device__ __forceinline__ int32_t scan64(int32_t v, int lane) { // inclusive, over the wavefront
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int32_t o = __shfl_up(v, d);
    if (lane >= d) v += o;
  }
  return v;
}

// Where the units of all sequences lie: tiles (whole tiles a workgroup) or steps.  Every wavefront scans by itself, lane i
// the sequences i * per and up.
struct Walk {
  const PagedAttnArgs &a;
  int lane, per;
  int32_t base, total;
  __device__ __forceinline__ int32_t units_of(const Seq &sq) const {
    if (a.rows_whole) return sq.tiles;
    int32_t n = 0;
    for (int i = 0; i < sq.tiles; ++i) n += steps_of(a, sq, i);
    return n;
  }
  __device__ __forceinline__ Walk(const PagedAttnArgs &args, int lane) : a(args), lane(lane) {
    per = (a.b + 63) / 64;
    int32_t n = 0;
    bool large = false; // a sequence of many tiles, which all lanes count together
    for (int b = min(lane * per, a.b); b < min(lane * per + per, a.b); ++b) {
      const Seq sq = seq_of(a, b);
      large = per == 1 && !a.rows_whole && sq.tiles > 8;
      if (!large) n += units_of(sq);
    }
    for (uint64_t todo = __ballot(large); todo; todo &= todo - 1) {
      const int b = __builtin_ctzll(todo);
      const Seq sq = seq_of(a, b);
      int32_t m = 0;
      for (int i = lane; i < sq.tiles; i += 64) m += steps_of(a, sq, i);
#pragma unroll
      for (int d = 32; d; d >>= 1) m += __shfl_xor(m, d);
      if (lane == b) n = m;
    }
    const int32_t v = scan64(n, lane);
    base = v - n;
    total = __builtin_amdgcn_readlane(v, 63);
  }
  // the sequence that holds unit u, with the units before it
  __device__ __forceinline__ int find(int32_t u, int32_t *before, Seq *sq) const {
    const int l = 63 - __builtin_clzll(__ballot(base <= u));
    int b = l * per;
    *before = __builtin_amdgcn_readlane(base, l);
    *sq = seq_of(a, b);
    while (per > 1) {
      const int32_t n = units_of(*sq);
      if (*before + n > u) break;
      *before += n;
      *sq = seq_of(a, ++b);
    }
    return b;
  }
  // the tile of sequence sq that holds its step `at`, and the steps before that tile
  __device__ __forceinline__ int tile_of(const Seq &sq, int32_t at, int32_t *before) const {
    *before = 0;
    for (int i0 = 0;; i0 += 64) {
      const int32_t n = i0 + lane < sq.tiles ? steps_of(a, sq, i0 + lane) : 0, v = scan64(n, lane);
      const uint64_t past = __ballot(*before + v > at);
      if (past) {
        const int l = __builtin_ctzll(past);
        *before += __builtin_amdgcn_readlane(v - n, l);
        return i0 + l;
      }
      *before += __builtin_amdgcn_readlane(v, 63);
    }
  }
};

// A tile that is split and whose first steps are workgroup i's: the i-th entry behind the partial results, as in
// paged_attn_one.h.
struct Split { int32_t b, more, slot, tile; }; // b: sequence, -1 = none

// Floats of one part: 128 rows of D sums, then (reference, sum) of each row.
template <int D> constexpr int part_floats() { return kRows * D + 2 * kRows; }

// K tile, V^T tile; of each 16-key subtile the score factor, the score offset and what brings weights back to probabilities
// (4 floats each), whether a key of it counts, whether its V holds NaN (4 words each); and where V holds NaN, a bit for
// each code, 16 bits for each (key, staging thread)
constexpr int kMeta = 80;
template <int D> constexpr int stage_bytes() { return (64 * D * 2 * 2 + kMeta + 64 * 16 * 2 + 511) / 512 * 512; }
template <int D> constexpr int lds_bytes() { return 2 * stage_bytes<D>(); }

// Returns whether a tile was left to FAR, as in paged_attn_one.h.
template <class E, int D, bool FAR>
__device__ __forceinline__ bool body(const PagedAttnArgs &a, uint8_t *lds, int wg, int wgs, int tid) {
  typedef typename one::Weights<FAR>::type W;
  constexpr int DK = D / 16, DT = D / 32, KB = D / 4, VB = D / 16, KW = KB / 16, VW = VB / 4;
  constexpr int KROW = D * 2, VOFF = 64 * KROW, FOFF = 2 * VOFF;
  constexpr int KMASK = D == 64 ? 7 : 15, KSH = D == 64 ? 1 : 0; // chunk swizzle of K rows
  const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c32 = lane & 31, hi = lane >> 5;
  const Walk walk(a, lane);
  const int heads = a.c.heads, hk = wg % heads, group = wg / heads;
  Split *split = (Split *)(a.rows_part + 2 * (int64_t)wgs * part_floats<D>()) + wg;
  int32_t u, u_end, before;
  int32_t each = 1, extra = 0; // steps of a group; the first `extra` groups have one more
  if (a.rows_whole) {
    u = walk.total - 1 - group; // late rows, which attend most keys, first
    if (u < 0) return false;
    u_end = u + 1;
  } else {
    const int32_t groups = min(wgs / heads, walk.total);
    if (group >= groups) {
      if (!FAR && tid == 0) split->b = -1;
      return false;
    }
    each = walk.total / groups;
    extra = walk.total - each * groups;
    u = group * each + min(group, extra);
    u_end = u + each + (group < extra);
  }
  Seq sq;
  int b = walk.find(u, &before, &sq), tile;
  if (a.rows_whole) {
    tile = u - before;
  } else {
    int32_t inside;
    tile = walk.tile_of(sq, u - before, &inside);
    before += inside; // from here on: the units before the tile
  }
  const int32_t u_first = u;
  bool noted = false, again = false;

  for (;;) {
    const int R = sq.n * a.group, row0 = tile * kRows;
    const int nsteps = steps_of(a, sq, tile);
    const int k_lo = a.rows_whole ? 0 : u - before, k_hi = a.rows_whole ? nsteps : min(nsteps, k_lo + (u_end - u));

    const int row = row0 + wave * 32 + c32;
    const int qi = min(row, R - 1) / a.group, qg = min(row, R - 1) % a.group;
    const int64_t t = sq.q0 + qi;
    const int hq = hk * a.group + qg;
    const int32_t limit = last_key(a, sq, qi);
    const bool alive = row0 + wave * 32 < R;  // the wavefront has rows
    // keys that all rows of the workgroup attend end here; the wavefront's own rows see nothing from `wave_end` on
    const int32_t all_to = last_key(a, sq, row0 / a.group);
    const int32_t wave_last = __builtin_amdgcn_readfirstlane(last_key(a, sq, min(row0 + wave * 32 + 31, R - 1) / a.group));

    typename E::frag qf[DK];
    {
      const uint16_t *qr = a.q + t * a.q_tok + hq * a.q_head + hi * 8;
  #pragma unroll
      for (int s = 0; s < DK; ++s) // (a negative scale's sign goes into q: factors of scores are positive below)
        qf[s] = __builtin_bit_cast(typename E::frag, *(const u32x4 *)(qr + s * 16) ^ (a.qk_scale < 0.0f ? 0x80008000u : 0u));
    }
    f32x16 acc[DT];
  #pragma unroll
    for (int i = 0; i < DT; ++i) acc[i] = (f32x16){0};
    float mref = -kInf, lsum = 0.0f;

    const int32_t *table = a.table + (int64_t)b * a.table_stride;
    const uint8_t *kh = a.c.k + hk * a.c.k_head, *vh = a.c.v + hk * a.c.v_head;
    // staging: K row tid / 4 of the tile, KB codes from column (tid % 4) * KB; V keys 4 (tid / 16) .. + 3, VB codes from
    // column (tid % 16) * VB.  Both lie in the wavefront's 16 keys.
    const uint32_t kvo = (uint32_t)(((tid >> 2) & 15) * a.c.k_tok + (tid & 3) * KB);
    uint32_t vvo[4];
  #pragma unroll
    for (int r = 0; r < 4; ++r) vvo[r] = (uint32_t)(((((tid >> 4) & 3) * 4 + r)) * a.c.v_tok + (tid & 15) * VB);

    // What lane (k % 16) * 4 + s knows of subtile s of step k (16 steps at a time).
    int32_t ko_lo, ko_hi, vo_lo, vo_hi, live, vcode;
    float kscale;
    one::Span span; // the same in all wavefronts
    auto batch = [&](int k0) {
      const int64_t key = (int64_t)(k0 + (lane >> 2)) * 64 + (lane & 3) * 16;
      const uint32_t sub = (uint32_t)(key >> 4);
      const uint32_t blk = (uint32_t)(((uint64_t)sub * a.page_magic) >> 36);
      int32_t page = key < sq.len ? table[blk] : -1;
      const bool ok = page >= 0 && page < a.c.pages;
      page = ok ? page : 0;
      const int64_t prow = ok ? ((int64_t)sub - (int64_t)blk * (a.c.page_size >> 4)) * 16 : 0;
      const int64_t ko = page * a.c.k_page + prow * a.c.k_tok, vo = page * a.c.v_page + prow * a.c.v_tok;
      ko_lo = (int32_t)ko; ko_hi = (int32_t)(ko >> 32); vo_lo = (int32_t)vo; vo_hi = (int32_t)(vo >> 32);
      live = ok ? (int32_t)min((int64_t)sq.len - key, (int64_t)16) : 0;
      kscale = pow2_code(a.c.ks[page * a.c.ks_page + hk * a.c.ks_head]) * fabsf(a.qk_scale);
      vcode = ok ? a.c.vs[page * a.c.vs_page + hk * a.c.vs_head] : 0;
    };
    u32x4 kr[KW];
    uint32_t vr[4][VW];
    int staged_at, staged_nv; // of the codes in kr and vr: the lane that knows the tile's first subtile, the wavefront's live keys
    auto load = [&](int k, int k_first) {
      const int at = ((k - k_first) & 15) * 4;
      if (((k - k_first) & 15) == 0) {
        if (!FAR && k != k_first) span.meet(live, vcode); // (not right behind their loads)
        batch(k);
      }
      staged_at = at;
      staged_nv = __builtin_amdgcn_readlane(live, at + wave);
      const uint8_t *kp = kh + one::lane64(ko_lo, ko_hi, at + wave), *vp = vh + one::lane64(vo_lo, vo_hi, at + wave);
  #pragma unroll
      for (int i = 0; i < KW; ++i) kr[i] = *(const u32x4 *)(kp + kvo + i * 16);
  #pragma unroll
      for (int r = 0; r < 4; ++r) {
        if constexpr (VW == 1) vr[r][0] = *(const uint32_t *)(vp + vvo[r]);
        if constexpr (VW == 2) {
          const u32x2 x = *(const u32x2 *)(vp + vvo[r]);
          vr[r][0] = x[0]; vr[r][1] = x[1];
        }
        if constexpr (VW == 4) {
          const u32x4 x = *(const u32x4 *)(vp + vvo[r]);
          vr[r][0] = x[0]; vr[r][1] = x[1]; vr[r][2] = x[2]; vr[r][3] = x[3];
        }
      }
    };
    // LDS addresses.  16-byte chunk c of K row r lies at c ^ (r / (256 / KROW) & KMASK), chunk c of V^T row d at
    // c ^ swz(d), which spreads what one instruction touches over the banks; a tile begins on 512 bytes, so that every
    // address below is one of four lane constants ^ a compile-time constant + another.
    auto swz = [](int d) { return ((d >> 1) ^ (d >> 4)) & 7; };
    const uint32_t k_rd = c32 * KROW + ((hi ^ ((c32 >> KSH) & KMASK)) << 4);
    const uint32_t v_rd = VOFF + c32 * 128 + ((hi ^ swz(c32)) << 4);
    const uint32_t k_wr = (tid >> 2) * KROW + ((((tid & 3) * (KB / 8)) ^ (((tid >> 2) >> KSH) & KMASK)) << 4);
    const uint32_t v_wr = VOFF + (tid & 15) * VB * 128 + (((wave * 2 + ((tid >> 4) & 1)) ^ swz((tid & 15) * VB)) << 4) + ((tid >> 5) & 1) * 8;
    // codes in registers -> tile in LDS.  `edge`: some row does not attend some of these keys, so a NaN in V must be told
    // from the others' results (found here, handled by the readers).
    auto store = [&](uint32_t buf, bool edge) {
      // (the batch still is the one these codes came from: load() of a later tile comes after)
      if (wave == 0 && (uint32_t)(lane - staged_at) < 4) {
        float *m = (float *)(lds + buf + FOFF) + (lane - staged_at);
        m[0] = fmaxf(kscale, 1e-37f); // (not 0: a masked score times it has to stay -inf)
        m[4] = (float)(vcode - kBase);
        m[8] = unweight(vcode);
        ((int32_t *)m)[12] = live;
      }
      const uint32_t kw = buf + k_wr, vw = buf + v_wr;
  #pragma unroll
      for (int i = 0; i < KW; ++i)
  #pragma unroll
        for (int h = 0; h < 2; ++h)
          *(u32x4 *)(lds + (kw ^ ((i * 2 + h) << 4))) = __builtin_bit_cast(u32x4, E::codes(kr[i][2 * h], kr[i][2 * h + 1]));
      const int nv = staged_nv;
      const int mm = (tid >> 4) & 3; // 4-key group of the 16
      if (nv < 16) {
  #pragma unroll
        for (int r = 0; r < 4; ++r)
  #pragma unroll
          for (int w = 0; w < VW; ++w) vr[r][w] = mm * 4 + r < nv ? vr[r][w] : 0;
      }
      if (edge) {
        uint32_t nan[4][VW], any = 0;
  #pragma unroll
        for (int r = 0; r < 4; ++r)
  #pragma unroll
          for (int w = 0; w < VW; ++w) {
            nan[r][w] = ((vr[r][w] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
            any |= nan[r][w];
          }
        const bool found = __any(any != 0);
        if (lane == 0) *(int32_t *)(lds + buf + FOFF + 64 + wave * 4) = found;
        if (found) {
  #pragma unroll
          for (int r = 0; r < 4; ++r) {
            uint32_t bits = 0;
  #pragma unroll
            for (int w = 0; w < VW; ++w) {
              // bits 7, 15, 23, 31 -> 0 .. 3
              bits |= (((nan[r][w] >> 7) * 0x00204081u) >> 21 & 15u) << (w * 4);
              vr[r][w] &= ~((nan[r][w] >> 7) * 0xffu);
            }
            ((uint16_t *)(lds + buf + FOFF + kMeta))[(wave * 16 + mm * 4 + r) * 16 + (tid & 15)] = (uint16_t)bits;
          }
        }
      }
  #pragma unroll
      for (int w = 0; w < VW; ++w) {
        const uint32_t x0 = __builtin_amdgcn_perm(vr[1][w], vr[0][w], 0x05010400), x1 = __builtin_amdgcn_perm(vr[3][w], vr[2][w], 0x05010400);
        const uint32_t y0 = __builtin_amdgcn_perm(vr[1][w], vr[0][w], 0x07030602), y1 = __builtin_amdgcn_perm(vr[3][w], vr[2][w], 0x07030602);
        const u32x2 f[4] = {{W::template codes2<false>(x0), W::template codes2<false>(x1)},
                            {W::template codes2<true>(x0), W::template codes2<true>(x1)},
                            {W::template codes2<false>(y0), W::template codes2<false>(y1)},
                            {W::template codes2<true>(y0), W::template codes2<true>(y1)}};
  #pragma unroll
        for (int i = 0; i < 4; ++i) *(u32x2 *)(lds + (vw ^ (((w * 4 + i) >> 1) << 4)) + (w * 4 + i) * 128) = f[i];
      }
    };
    auto edge_of = [&](int k) { return k * 64 + 63 > all_to; };

    bool far = false;
    if constexpr (FAR) {
      for (int k = k_lo; k < k_hi; k += 16) {
        batch(k);
        span.meet(live, vcode);
      }
      far = span.far();
    }
    const int k_to = FAR && !far ? k_lo : k_hi; // (no step of a tile that the first pass has done)
    if (k_lo < k_to) {
      load(k_lo, k_lo);
      store(0, edge_of(k_lo));
    }
    if (k_lo + 1 < k_to) load(k_lo + 1, k_lo);
    __syncthreads();
    for (int k = k_lo; k < k_to; ++k) {
      const uint32_t buf = ((k - k_lo) & 1) * stage_bytes<D>(), next = stage_bytes<D>() - buf;
      if (k + 1 < k_to) {
        store(next, edge_of(k + 1));
        if (k + 2 < k_to) load(k + 2, k_lo);
      }
      __builtin_amdgcn_sched_barrier(0);
      if (alive && k * 64 <= wave_last) {
        const uint32_t kb = buf + k_rd, vb = buf + v_rd;
        f32x16 st[2] = {(f32x16){0}, (f32x16){0}};
        // The order is pinned: left alone, the scheduler reads each fragment right before its product and waits for it.
        // Four reads are on their way at any time.
        u32x4 x[4];
        auto k_frag = [&](int i) { return *(const u32x4 *)(lds + (kb ^ ((i >> 1) << 5)) + (i & 1) * 32 * KROW); };
  #pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = k_frag(i);
  #pragma unroll
        for (int i = 0; i < 2 * DK; ++i) {
          __builtin_amdgcn_sched_barrier(0);
          st[i & 1] = E::mfma32(__builtin_bit_cast(typename E::frag, x[i & 3]), qf[i >> 1], st[i & 1]);
          if (i + 4 < 2 * DK) x[i & 3] = k_frag(i + 4);
        }
        __builtin_amdgcn_sched_barrier(0);
        const f32x4 factor = *(const f32x4 *)(lds + buf + FOFF), offset = *(const f32x4 *)(lds + buf + FOFF + 16);
        const f32x4 back = *(const f32x4 *)(lds + buf + FOFF + 32);
        const bool edge = edge_of(k);
        bool whole_tile = !edge;
        if (!edge) { // (also where every row attends every key a page may be missing)
          const u32x4 nv = *(const u32x4 *)(lds + buf + FOFF + 48);
          whole_tile = __builtin_amdgcn_readfirstlane(nv[0] & nv[1] & nv[2] & nv[3]) == 16;
        }
        if (!whole_tile) {
          const u32x4 nv = *(const u32x4 *)(lds + buf + FOFF + 48);
  #pragma unroll
          for (int s = 0; s < 4; ++s) {
            const int32_t rel = nv[s] ? limit - k * 64 - s * 16 - hi * 4 : -1; // (keys past the end are past the limit)
  #pragma unroll
            for (int r = 0; r < 8; ++r) {
              const float x = st[s >> 1][(s & 1) * 8 + r];
              st[s >> 1][(s & 1) * 8 + r] = (r >> 2) * 8 + (r & 3) <= rel ? x : -kInf;
            }
          }
        }
        // x = score * factor + offset, whose maximum is that of the scores
        float top = -kInf;
  #pragma unroll
        for (int s = 0; s < 4; ++s) {
          float m = st[s >> 1][(s & 1) * 8];
  #pragma unroll
          for (int r = 1; r < 8; ++r) m = fmaxf(m, st[s >> 1][(s & 1) * 8 + r]);
          top = fmaxf(top, fmaf(m, factor[s], offset[s]));
        }
        if (__any(top > mref + kLazy)) {
          const float mn = fmaxf(mref, fmaxf(top, __shfl_xor(top, 32)));
          const float al = mn == -kInf ? 1.0f : __builtin_amdgcn_exp2f(mref - mn);
          lsum = !FAR ? lsum * al : mn == -kInf ? lsum : one::lower(lsum, mref - mn);
          mref = mn;
  #pragma unroll
          for (int i = 0; i < DT; ++i)
  #pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][r] *= al;
        }
        const float ref = (mref == -kInf ? 0.0f : mref) - kLift;
        // weights of a subtile between the products of the one before, V fragments four reads ahead (the sums of weights too as
        // it is written; the compiler moves those, 32 additions, behind the last product)
        typename W::frag pf[4];
        [[maybe_unused]] typename W::frag rest[4]; // FAR: what rounding to pf took away
        float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        auto weights = [&](int s, int r0, int n) {
          const float c = offset[s] - ref;
  #pragma unroll
          for (int r = r0; r < r0 + n; ++r) {
            const float w = __builtin_amdgcn_exp2f(fmaf(st[s >> 1][(s & 1) * 8 + r], factor[s], c));
            if constexpr (FAR) {
              const __bf16 h = (__bf16)w;
              pf[s][r] = h;
              rest[s][r] = (__bf16)(w - (float)h);
              lsum += __builtin_amdgcn_exp2f(fmaf(st[s >> 1][(s & 1) * 8 + r], factor[s], -ref)); // (w can be too small for fp32, the probability is not)
            } else {
              sum[s] += w; // (the sum of probabilities has to be fp32's: the log-sum-exp is a result)
              pf[s][r] = (_Float16)w;
            }
          }
        };
        auto v_frag = [&](int i) { return *(const u32x4 *)(lds + (vb ^ (((i / DT) ^ (i % DT & 3)) << 5)) + i % DT * 32 * 128); };
  #pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = v_frag(i);
        weights(0, 0, 8);
  #pragma unroll
        for (int i = 0; i < 4 * DT; ++i) {
          __builtin_amdgcn_sched_barrier(0);
          if constexpr (FAR) acc[i % DT] = W::mfma32(__builtin_bit_cast(typename W::frag, x[i & 3]), rest[i / DT], acc[i % DT]);
          acc[i % DT] = W::mfma32(__builtin_bit_cast(typename W::frag, x[i & 3]), pf[i / DT], acc[i % DT]);
          if (i + 4 < 4 * DT) x[i & 3] = v_frag(i + 4);
          if (i < 3 * DT) weights(i / DT + 1, i % DT * (8 / DT), 8 / DT);
        }
        __builtin_amdgcn_sched_barrier(0);
  #pragma unroll
        for (int s = 0; s < 4 && !FAR; ++s) lsum = fmaf(sum[s], back[s], lsum);
        if (edge) { // NaN in V, taken out of the tile: it reaches the rows that attend its key
          for (int s = 0; s < 4; ++s) {
            if (!__builtin_amdgcn_readfirstlane(*(const int32_t *)(lds + buf + FOFF + 64 + s * 4))) continue;
            for (int j = 0; j < 16; ++j) {
              if (k * 64 + s * 16 + j > limit) continue;
              const uint16_t *bits = (const uint16_t *)(lds + buf + FOFF + kMeta) + (s * 16 + j) * 16;
  #pragma unroll
              for (int i = 0; i < DT; ++i)
  #pragma unroll
                for (int r = 0; r < 16; ++r) {
                  const int d = i * 32 + (r >> 2) * 8 + hi * 4 + (r & 3);
                  if (bits[d / VB] >> (d % VB) & 1) acc[i][r] = __builtin_nanf("");
                }
            }
          }
        }
      }
      __syncthreads();
    }

    if constexpr (!FAR) {
      span.meet(live, vcode);
      far = span.far();
      again |= far;
    }
    lsum += __shfl_xor(lsum, 32);
    const bool cut = k_lo > 0 || k_hi < nsteps;
    // (the first tile of this workgroup takes slot 0, a later one that is cut can only be its last: slot 1)
    const int which = u == u_first ? 0 : 1;
    if (alive && row < R && far == FAR) {
      if (!cut) {
        const bool none = lsum == 0.0f && mref == -kInf;
        const float inv = none ? 0.0f : kOut / lsum;
        uint16_t *op = a.o + t * a.o_tok + hq * a.o_head + hi * 4;
  #pragma unroll
        for (int i = 0; i < DT; ++i)
  #pragma unroll
          for (int r = 0; r < 4; ++r) {
            uint16_t x[4];
  #pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = E::out(acc[i][r * 4 + j] * inv);
            *(u32x2 *)(op + i * 32 + r * 8) = (u32x2){(uint32_t)x[0] | (uint32_t)x[1] << 16, (uint32_t)x[2] | (uint32_t)x[3] << 16};
          }
        if (a.lse && hi == 0) a.lse[t * a.heads_q + hq] = none ? -kInf : mref - kLift + __builtin_log2f(lsum);
      } else {
        float *p = a.rows_part + (2 * (int64_t)wg + which) * part_floats<D>();
        const int lr = wave * 32 + c32;
  #pragma unroll
        for (int i = 0; i < DT; ++i)
  #pragma unroll
          for (int r = 0; r < 4; ++r)
            *(f32x4 *)(p + lr * D + i * 32 + r * 8 + hi * 4) = (f32x4){acc[i][r * 4], acc[i][r * 4 + 1], acc[i][r * 4 + 2], acc[i][r * 4 + 3]};
        if (hi == 0) { p[kRows * D + lr * 2] = mref; p[kRows * D + lr * 2 + 1] = lsum; }
      }
    }
    if (a.rows_whole) return again;
    if (!FAR && cut && k_lo == 0) {
      const int32_t last = before + nsteps - 1, larger = extra * (each + 1); // the tile's last step, and the group that has it
      const int32_t owner = last < larger ? last / (each + 1) : extra + (last - larger) / each;
      if (tid == 0) *split = {b, owner - group, which, tile};
      noted = true;
    }
    u += k_hi - k_lo;
    if (u >= u_end) break;
    before += nsteps;
    if (++tile == sq.tiles) {
      tile = 0;
      do sq = seq_of(a, ++b);
      while (sq.tiles == 0); // (u is less than all units)
    }
  }
  if (!FAR && !noted && tid == 0) split->b = -1;
  return again;
}
template <class E, int D> __device__ __attribute__((noinline)) void far_pass(uint64_t args, one::Lds lds, int wg, int wgs) {
  const PagedAttnArgs a = one::args_at(args);
  body<E, D, true>(a, (uint8_t *)lds, one::uniform(wg), one::uniform(wgs), threadIdx.x);
}
template <class E, int D> __device__ __forceinline__ void both(const PagedAttnArgs &a, uint8_t *lds, int wg, int wgs) {
  if (__builtin_expect(body<E, D, false>(a, lds, wg, wgs, threadIdx.x), 0)) {
    __syncthreads();
    far_pass<E, D>((uint64_t)__builtin_amdgcn_kernarg_segment_ptr(), (one::Lds)lds, wg, wgs);
  }
}

// Adds the parts of the split tile that workgroup wg of the launch before noted, if any: rows 16 part .. + 15.
template <class E, int D> __device__ __forceinline__ void join(const PagedAttnArgs &a, int wg, int part, int wgs) {
  constexpr int PF = part_floats<D>(), VB = D / 16;
  const Split sp = ((const Split *)(a.rows_part + 2 * (int64_t)wgs * PF))[wg];
  if (sp.b < 0) return;
  const Seq sq = seq_of(a, sp.b);
  const int row0 = sp.tile * kRows, lr = part * 16 + (threadIdx.x >> 4), d0 = (threadIdx.x & 15) * VB;
  if (row0 + lr >= sq.n * a.group) return;
  const int heads = a.c.heads, parts = sp.more + 1;
  const float *first = a.rows_part + (2 * (int64_t)wg + sp.slot) * PF, *later = a.rows_part + 2 * (int64_t)wg * PF;
  float m = -kInf, l = 0.0f;
  f32x4 o[VB / 4];
#pragma unroll
  for (int i = 0; i < VB / 4; ++i) o[i] = (f32x4){0, 0, 0, 0};
  for (int p = 0; p < parts; p += 4) {
    float pm[4], pl[4];
    f32x4 po[4][VB / 4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int j = min(p + i, parts - 1);
      const float *x = j ? later + 2 * (int64_t)j * heads * PF : first;
      pm[i] = x[kRows * D + lr * 2];
      pl[i] = x[kRows * D + lr * 2 + 1];
#pragma unroll
      for (int v = 0; v < VB / 4; ++v) po[i][v] = *(const f32x4 *)(x + lr * D + d0 + v * 4);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (p + i >= parts) break;
      const float mn = fmaxf(m, pm[i]), ref = mn == -kInf ? 0.0f : mn;
      const float f = m == -kInf ? 1.0f : __builtin_amdgcn_exp2f(m - ref), w = pm[i] == -kInf ? 1.0f : __builtin_amdgcn_exp2f(pm[i] - ref);
      l = one::add_sums(l, m, f, pl[i], pm[i], w, ref);
#pragma unroll
      for (int v = 0; v < VB / 4; ++v) o[v] = o[v] * f + po[i][v] * w;
      m = mn;
    }
  }
  const int qi = (row0 + lr) / a.group, hq = wg % heads * a.group + (row0 + lr) % a.group;
  const int64_t t = sq.q0 + qi;
  const bool none = l == 0.0f && m == -kInf;
  const float inv = none ? 0.0f : kOut / l;
#pragma unroll
  for (int v = 0; v < VB / 4; ++v)
    *(u32x2 *)(a.o + t * a.o_tok + hq * a.o_head + d0 + v * 4) =
        (u32x2){(uint32_t)E::out(o[v][0] * inv) | (uint32_t)E::out(o[v][1] * inv) << 16, (uint32_t)E::out(o[v][2] * inv) | (uint32_t)E::out(o[v][3] * inv) << 16};
  if (a.lse && d0 == 0) a.lse[t * a.heads_q + hq] = none ? -kInf : m - kLift + __builtin_log2f(l);
}

} // namespace rows

// Many rows, and beside them, in the workgroups behind, the sequences of few.
#define PAGED_MIXED(T, E, D, MT, OCC)                                                                         \
  extern "C" __global__ __launch_bounds__(256, OCC) void paged_attn_rows_##T##_d##D##_r##MT(PagedAttnArgs a) { \
    constexpr int bytes = rows::lds_bytes<D>() > one::lds_floats<D, MT>() * 4 ? rows::lds_bytes<D>() : one::lds_floats<D, MT>() * 4; \
    __shared__ __align__(512) uint8_t lds[bytes];                                                             \
    if ((int)blockIdx.x < a.rows_groups)                                                                      \
      rows::both<rows::E, D>(a, lds, blockIdx.x, a.rows_groups);                                              \
    else                                                                                                      \
      one::both<one::E, D, MT, true, OCC>(a, (float *)lds, blockIdx.x - a.rows_groups, gridDim.x - a.rows_groups); \
  }                                                                                                           \
  /* 8 workgroups for each that may have split a row tile, then join_pieces for each that may have split a sequence */ \
  extern "C" __global__ __launch_bounds__(256) void paged_attn_rows_join_##T##_d##D##_r##MT(PagedAttnArgs a) { \
    __shared__ one::f32x4 lds[256 + 128];                                                                     \
    if ((int)blockIdx.x < 8 * a.rows_groups)                                                                  \
      rows::join<rows::E, D>(a, blockIdx.x / 8, blockIdx.x % 8, a.rows_groups);                               \
    else                                                                                                      \
      one::join<one::E, D, MT>(a, lds, (blockIdx.x - 8 * a.rows_groups) / a.join_pieces,                      \
                               (blockIdx.x - 8 * a.rows_groups) % a.join_pieces, (gridDim.x - 8 * a.rows_groups) / a.join_pieces); \
  }
PAGED_MIXED(bf16, Bf, 64, 1, 2)
PAGED_MIXED(bf16, Bf, 64, 2, 2)
PAGED_MIXED(bf16, Bf, 128, 1, 2)
PAGED_MIXED(bf16, Bf, 256, 1, 1)
PAGED_MIXED(f16, Hf, 64, 1, 2)
PAGED_MIXED(f16, Hf, 64, 2, 2)
PAGED_MIXED(f16, Hf, 128, 1, 2)
PAGED_MIXED(f16, Hf, 256, 1, 1)
#undef PAGED_MIXED
