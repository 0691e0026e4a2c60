// Attention of new tokens over the paged cache with shaped scores: decode
// rows, prefill chunks and drafted token trees, gfx950.
//
// For a query token at place p and a visible key at place j, head h:
//   s = scale q.k;  s = cap tanh(s / cap) (cap > 0);  s -= slope_h |p - j|
//   out = sum_j softmax_j(s) v_j, 0 for a token that sees no key.
// Chunk tokens sit at the end of their sequence's keys (p = p0 + t, p0 the keys
// before the chunk) and see keys j <= p or j < prefix, within the window (p - j
// < window).  Tree token t sees the context j < p0 and the tree keys named by
// its mask bits; its place is p0 + popcount(mask_t) - 1, its depth in the tree.
//
// Layout of the work.  The G query heads of one kv head and the tokens of a
// block are the columns of S^T = K Q^T (a lane owns one column, so a row's
// softmax never leaves its four lane groups), and P, rounded to bf16 as the
// MFMA takes it, is already the operand of O^T = V^T P^T; logits, sums and O
// are fp32.  An item is one block of columns against the 32-key tiles it sees;
// the tiles of all items, in one row, are cut into equal shares, one workgroup
// each, on the device from the device's lengths, so a call needs no lengths on
// the host and can be captured.  An item cut between shares leaves fp32
// partials that a second launch joins.  Short calls are not cut and have no
// second launch (make_plan).
//
// Two kinds of form share the tile arithmetic:
//   private  up to 32 columns (decode rows, small trees): every wave streams
//            its own tiles through its own LDS slots, without a workgroup
//            barrier; waves differ in kv head and in tile phase.  Bound by HBM
//            in a batch (48 ragged decode rows with a distance bias: 447 MB in
//            71 us, 6.3 TB/s, of about 6.9 that reading alone reaches), by
//            latency for one user (333 keys, 8 us: launch, lengths, table,
//            queries, two rounds of tiles and the join in turn).
//   turns    64 to 256 columns (chunks, larger trees): the waves split the
//            columns and read the same tile from a ring of LDS slots; one half
//            multiplies while the other takes its softmax.  Bound by the issue
//            of both: 2100 cycles a 256-column tile for plain scores, 2600 for
//            capped ones, of which the matrix unit is busy 1024 (64 trees of
//            64 tokens over 4096 keys: 838 TFLOP/s; a chunk of 2048 over 14336
//            keys, capped: 880).
// Tried and not kept in the turns form: V operands read under the softmax
// instead of under the products (chunk 570 -> 620 us), half of the caps taken
// between the products of O (no change).
#include <algorithm>
#include <atomic>
#include <cmath>

#include "kvc_lds.h"

namespace kvc {
namespace {

constexpr int kD = 128;
constexpr int kTile = 32;
constexpr int kTensor = kTile * kD * 2;  // one K or V tile of a head: 8 KiB
constexpr uint32_t kLazyBits = 0x4380u;  // bf16 2^8: a weight past it moves the running reference
// Under a near cap scores lie within 2 cap log2(e) <= 160 binades, so a reference
// kNearAbove over a column's largest score so far mostly serves for good: once
// it is no more than kNearRoom below the cap, no weight can pass 2^30 whatever
// follows, and the reference is not looked at again.  Weights are 2^-54 of what
// they would be, far from fp32's ends: values from 2^-64 to 2^64 are served.
constexpr float kNearAbove = 54.f, kNearRoom = 30.f;
constexpr int kNoKey = 1 << 30;  // a key position that no column sees
constexpr float kLowest = -3.402823466e38f;
constexpr uint32_t kOnes2 = 0x3F803F80u;  // two bf16 ones

enum ScoreMode {
  kPlain = 0,
  kDistance = 1,
  kCapNear = 2,      // cap log2(e) <= kCapNearMax
  kCapFar = 3,
  kCapDistance = 4,
};
// Up to this cap (55) tanh by exp2 and a reciprocal, off by 2^-22 of the cap,
// serves scores of any size: 2^-22 x 55 is 2^-16.  The cap's last product and
// the reference then fold into one fma in front of exp2.
constexpr float kCapNearMax = 80.f;

struct ScoredParams {
  const uint16_t* q;
  int64_t q_st, q_sh;
  uint16_t* out;
  int64_t o_st, o_sh;
  const uint16_t* k;
  const uint16_t* v;
  int64_t k_row, k_head, v_row, v_head;  // elements per token row and kv head
  const int32_t* tables;                 // null: fresh rows at cu_k
  int64_t bt_stride;
  int max_blocks, num_blocks, page;
  int page_tiles;  // page / 32
  float page_rcp;  // 1 / page_tiles
  int64_t fresh_rows;
  const int32_t* cu_q;  // null: q_per_seq tokens each
  int q_per_seq;
  const int32_t* lens;  // keys per sequence (plus the queries, lens_exclude_q), or null
  const int32_t* cu_k;
  int lens_exclude_q;
  const uint32_t* mask;  // tree bits, mask_words 32-bit words a token, or null
  int mask_words;
  const int32_t* places;  // tree depths (popcount - 1) per token, or null
  const int32_t* prefix;
  const float* slopes;
  float scale, cap;
  int window;
  int batch, num_tokens, heads, kv_heads, group;
  float group_rcp;  // 1 / group
  int heads_per_wg, head_groups;
  int tokens_per_block;
  int lane_plan;  // the plan walks sequences across lanes (else blocks)
  int min_share;
  int whole;  // items are not cut: a share counts items
  int4* rec;  // per share, of the item it begins and leaves unfinished: first
              // token, tokens, head group, last share (0: none)
  float* part_o;
  float2* part_ml;
};

struct SeqGeo {
  int q0, sq;
  int sk;  // keys that there are: no more than the table's pages or the fresh rows hold
  int p0;  // place of the first query: by the given lengths, cut or not
};
constexpr int64_t kLongest = int64_t(1) << 29;  // of a length (tables hold fewer keys)

__device__ __forceinline__ SeqGeo seq_geo(const ScoredParams& p, int q0, int q1, int len, int k0,
                                          int k1) {
  SeqGeo g;
  g.q0 = max(0, min(q0, p.num_tokens));
  g.sq = max(0, min(q1, p.num_tokens) - g.q0);
  int64_t keys = p.lens != nullptr ? len : int64_t(k1) - k0;
  keys = max(int64_t(0), min(keys, kLongest)) + (p.lens_exclude_q ? g.sq : 0);
  const int64_t most = p.tables != nullptr ? int64_t(p.max_blocks) * p.page : p.fresh_rows - max(k0, 0);
  g.sk = int(max(int64_t(0), min(keys, most)));
  g.p0 = int(keys) - g.sq;
  return g;
}

// Geometry of sequence i from per-lane (vector) loads or uniform (scalar) ones.
template <bool kUniform>
__device__ __forceinline__ SeqGeo load_seq(const ScoredParams& p, int i) {
  auto at = [&](const int32_t* t, int64_t idx) {
    if constexpr (kUniform) return table_entry(t, idx);
    return t[idx];
  };
  int q0, q1, len = 0, k0 = 0, k1 = 0;
  if (p.cu_q != nullptr) {
    q0 = at(p.cu_q, i);
    q1 = at(p.cu_q, i + 1);
  } else {
    q0 = i * p.q_per_seq;
    q1 = q0 + p.q_per_seq;
  }
  if (p.lens != nullptr) {
    len = at(p.lens, i);
  } else {
    k0 = at(p.cu_k, i);
    k1 = at(p.cu_k, i + 1);
  }
  return seq_geo(p, q0, q1, len, k0, k1);
}

__device__ __forceinline__ int num_blocks_of(const ScoredParams& p, int sq) {
  return (sq + p.tokens_per_block - 1) / p.tokens_per_block;
}

// Key tiles [t0, t1) that block c of a sequence sees.
struct TileRange {
  int t0, t1;
};
__device__ __forceinline__ TileRange block_tiles(const ScoredParams& p, const SeqGeo& g, int pre,
                                                 int c) {
  const int p0 = g.p0;
  const int first = c * p.tokens_per_block;
  const int last = min(g.sq, first + p.tokens_per_block) - 1;
  int lo = 0, hi;
  if (p.mask != nullptr) {
    hi = g.sk;
    if (p.window > 0) lo = max(0, p0 - p.window);  // place >= context - 1
  } else {
    hi = min(g.sk, max(p0 + last + 1, pre));
    if (p.window > 0) lo = max(0, p0 + first + 1 - p.window);
  }
  TileRange r;
  r.t0 = lo / kTile;
  r.t1 = max(r.t0, (max(hi, 0) + kTile - 1) / kTile);
  return r;
}

// ---------------------------------------------------------------------------
// One wave's columns and running state.
// ---------------------------------------------------------------------------
template <int NCB>
struct Columns {
  int first, last;        // the block's tokens
  int col0;               // the wave's first column in the block
  float place[NCB];       // p, for the distance bias
  float slope2[NCB];      // slope log2(e)
  const uint32_t* bits;   // tree: the sequence's masks
  const int32_t* depths;  // tree: the sequence's depths
  int pre;                // two-way prefix
  int p0, sk, sq;         // p0: keys before the sequence's queries
  int full_lo, full_hi;   // a tile inside these keys needs no mask
};

// The token, inside its block, and the query head of column col0 + 16 cb + lm.
// (Worked out where it is needed, which is rarely: kept, it would take
// registers from the loop.)
struct ColumnOf {
  int token, head;
};
__device__ __forceinline__ ColumnOf column_of(const ScoredParams& p, int col0, int cb) {
  int lane = int(threadIdx.x);
  asm volatile("" : "+v"(lane));
  const int col = col0 + 16 * cb + (lane & 15);
  ColumnOf c;
  c.token = div_small(col, p.group, p.group_rcp);
  c.head = col - c.token * p.group;
  return c;
}

template <int NCB>
struct State {
  f32x4_t o[NCB][8];
  float l[NCB];  // over the lane's own keys; of the column once the loop is done
  float mu[NCB];
  int settled;   // a near cap's references serve for good
};

template <int NCB>
__device__ __forceinline__ void reset(State<NCB>& st) {
#pragma unroll
  for (int cb = 0; cb < NCB; ++cb) {
#pragma unroll
    for (int jj = 0; jj < 8; ++jj) st.o[cb][jj] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    st.l[cb] = 0.f;
    st.mu[cb] = kLowest;
  }
  st.settled = 0;
}

__device__ __forceinline__ uint32_t bits_below(int n) {  // bits 0 .. n - 1
  return n >= 32 ? 0xffffffffu : (n <= 0 ? 0u : (1u << n) - 1u);
}

// The visible keys of the lane's column cb in the tile at key j0, as bits.
template <int NCB>
__device__ __forceinline__ uint32_t visible_bits(const ScoredParams& p, const Columns<NCB>& c,
                                                 int cb, int j0) {
  const int t = min(c.first + column_of(p, c.col0, cb).token, c.last);
  if (p.mask == nullptr) {
    uint32_t vis = bits_below(min(c.sk, max(c.p0 + t + 1, c.pre)) - j0);
    if (p.window > 0) vis &= ~bits_below(c.p0 + t + 1 - p.window - j0);
    return vis;
  }
  uint32_t vis = bits_below(min(c.p0, c.sk) - j0);
  const int place = p.window > 0 ? c.p0 + c.depths[t] : 0;
  if (p.window > 0) vis &= ~bits_below(place + 1 - p.window - j0);
  const int u0 = j0 - c.p0;  // tree index of the tile's first key
  if (u0 > -kTile) {
    const uint32_t* m = c.bits + int64_t(t) * p.mask_words;
    uint32_t tree;
    if (u0 >= 0) {
      const int w = u0 >> 5, sh = u0 & 31;
      const uint32_t a = w < p.mask_words ? m[w] : 0u;
      const uint32_t b = w + 1 < p.mask_words ? m[w + 1] : 0u;
      tree = sh ? (a >> sh) | (b << (32 - sh)) : a;
    } else {
      tree = m[0] << (-u0);
    }
    tree &= bits_below(c.sk - j0);
    if (p.window > 0 && p.window <= c.sq) {
      // Only here can two depths of one tree, -1 (no bits) to sq - 1, be a
      // window apart.
      for (int k = max(0, -u0); k < kTile && u0 + k < c.sq; ++k)
        if (place - c.p0 - c.depths[u0 + k] >= p.window) tree &= ~(1u << k);
    }
    vis |= tree;
  }
  return vis;
}

struct Consts {
  float c2;      // scale log2(e)
  float zc;      // 2 log2(e) scale / cap
  float a, a2;   // cap log2(e) and twice that
  float z;       // scale / cap
};
// Caps that kCapNear does not take: 1 - 2 / (e^{2z} + 1) is off by 2^-22 of
// the cap, so below |z| = 1/16 tanh comes from its series, z (1 - z^2 / 3 + 2
// z^4 / 15), off by 17 / 315 z^6 < 2^-28 relative.
constexpr float kSeriesBelow = 1.f / 256;  // z^2

// The key offset of element e (0 .. 7) of a lane's column inside a tile: the
// MFMA's C rows 4 lg + i of the two 16-key halves, which is also the K index
// order of the P operand.
__device__ __forceinline__ int key_of(int e) { return (e & 3) + 16 * (e >> 2); }

// S^T = K Q^T: rows 4 lg + i of the tile's two 16-key halves.
template <int NCB>
__device__ __forceinline__ void logits(const u32x4_t (&k)[2][4], const u32x4_t (&q)[NCB][4],
                                       f32x4_t (&s)[NCB][2]) {
#pragma unroll
  for (int cb = 0; cb < NCB; ++cb) {
    s[cb][0] = s[cb][1] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      s[cb][0] = mfma_bf16(k[0][d], q[cb][d], s[cb][0]);
      s[cb][1] = mfma_bf16(k[1][d], q[cb][d], s[cb][1]);
    }
  }
}

// The score's shape, the mask, the running softmax, and P^T as the bf16
// operand pb.  y comes in as the logits and becomes what the softmax is taken
// of: the raw logit s (log2-unit score c2 s) for plain scores, r = -1 / (e^{2z}
// + 1) (log2-unit score a + 2 a r) under a near cap, the log2-unit score
// otherwise; -inf at keys the column does not see.  tanh(z) = 1 - 2 / (e^{2z} +
// 1): one exp2 and one reciprocal.  Sums are formed of the rounded P, so the
// weights add up to the sum that divides them.
template <int NCB, int MODE>
__device__ __forceinline__ void shape_scores(const Columns<NCB>& c, f32x4_t (&y)[NCB][2], int j0,
                                             int lg, const Consts& cs) {
  constexpr bool kDist = MODE == kDistance || MODE == kCapDistance;
  constexpr bool kCap = MODE == kCapNear || MODE == kCapFar || MODE == kCapDistance;
  if constexpr (!kDist && !kCap) return;
#pragma unroll
  for (int cb = 0; cb < NCB; ++cb) {
    // The bias of a key at or before the query's place.
    const float b0 = kDist ? c.slope2[cb] * (float(j0 + 4 * lg) - c.place[cb]) : 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float s = y[cb][e >> 2][e & 3];
      float x = s;
      if constexpr (kCap) {
        const float w = __builtin_amdgcn_exp2f(s * cs.zc);
        x = __builtin_amdgcn_rcpf(-1.f - w);
        if constexpr (MODE != kCapNear) {
          x = __builtin_fmaf(cs.a2, x, cs.a);
          const float z = s * cs.z, z2 = z * z;
          const float series = __builtin_fmaf(z2, __builtin_fmaf(z2, 2.f / 15, -1.f / 3), 1.f);
          x = z2 < kSeriesBelow ? s * cs.c2 * series : x;
        }
      }
      if constexpr (kDist) {
        const float bias = __builtin_fmaf(c.slope2[cb], float(key_of(e)), b0);
        x = kCap ? x + bias : __builtin_fmaf(s, cs.c2, bias);
      }
      y[cb][e >> 2][e & 3] = x;
    }
  }
}

// (in place: one copy of everything around it)
template <int NCB, int MODE>
__device__ __forceinline__ void mask_scores(const ScoredParams& p, const Columns<NCB>& c,
                                            f32x4_t (&y)[NCB][2], int j0, int lg) {
#pragma unroll
  for (int cb = 0; cb < NCB; ++cb) {
    const uint32_t own = visible_bits<NCB>(p, c, cb, j0) >> (4 * lg);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float x = y[cb][e >> 2][e & 3];
      if constexpr (MODE == kDistance || MODE == kCapDistance) {
        const int j = j0 + 4 * lg + key_of(e);
        int at = j;
        if (p.mask != nullptr && j >= c.p0 && j < c.sk) at = c.p0 + c.depths[j - c.p0];
        x = __builtin_fmaf(-c.slope2[cb],
                           fabsf(c.place[cb] - float(at)) + (float(j) - c.place[cb]), x);
      }
      y[cb][e >> 2][e & 3] = ((own >> key_of(e)) & 1u) ? x : -INFINITY;
    }
  }
}

typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t,
                            __builtin_elementwise_max(__builtin_bit_cast(u16x2_t, a),
                                                      __builtin_bit_cast(u16x2_t, b)));
}

// The log2-unit score of y: unit y + base.
template <int MODE>
__device__ __forceinline__ float unit_of(const Consts& cs) {
  return MODE == kPlain ? cs.c2 : MODE == kCapNear ? cs.a2 : 1.f;
}
template <int MODE>
__device__ __forceinline__ float base_of(const Consts& cs) {
  return MODE == kCapNear ? cs.a : 0.f;
}

// P^T of the tile, relative to each column's reference.
template <int NCB, int MODE>
__device__ __forceinline__ void exponentials(const State<NCB>& st, const f32x4_t (&y)[NCB][2],
                                             const Consts& cs, u32x4_t (&pb)[NCB]) {
#pragma unroll
  for (int cb = 0; cb < NCB; ++cb) {
    float pr[8];
    const float base = base_of<MODE>(cs) - st.mu[cb];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float x = y[cb][e >> 2][e & 3];
      pr[e] = __builtin_amdgcn_exp2f(MODE == kPlain || MODE == kCapNear
                                         ? __builtin_fmaf(x, unit_of<MODE>(cs), base)
                                         : x + base);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t two = pack_bf16x2_fast(pr[2 * i], pr[2 * i + 1]);
      asm volatile("" : "+v"(two));  // (else it is packed anew for every use)
      pb[cb][i] = two;
    }
  }
}

// The columns' references up to the tile's largest scores.
template <int NCB, int MODE>
__device__ __forceinline__ void raise_reference(State<NCB>& st, const f32x4_t (&y)[NCB][2],
                                                const Consts& cs) {
  constexpr float kAbove = MODE == kCapNear ? kNearAbove : 0.f;
#pragma unroll
  for (int cb = 0; cb < NCB; ++cb) {
    float top = y[cb][0][0];
#pragma unroll
    for (int e = 1; e < 8; ++e) top = fmaxf(top, y[cb][e >> 2][e & 3]);
    const float mu = fmaxf(st.mu[cb], __builtin_fmaf(rows4_max(top), unit_of<MODE>(cs),
                                                     base_of<MODE>(cs) + kAbove));
    const float down = __builtin_amdgcn_exp2f(st.mu[cb] - mu);
#pragma unroll
    for (int jj = 0; jj < 8; ++jj) st.o[cb][jj] *= down;
    st.l[cb] *= down;
    st.mu[cb] = mu;
  }
}

// A near cap's, ahead of the weights, until it serves for good.
template <int NCB>
__device__ __forceinline__ void settle_reference(State<NCB>& st, const f32x4_t (&y)[NCB][2],
                                                 const Consts& cs) {
  raise_reference<NCB, kCapNear>(st, y, cs);
  bool serves = true;
#pragma unroll
  for (int cb = 0; cb < NCB; ++cb) serves &= st.mu[cb] >= cs.a - kNearRoom;
  st.settled = uniform(int(__all(serves)));
}

// Otherwise the reference moves only when a weight passes 2^8 (or a column has
// none yet), which the packed weights themselves say; the tile's are then
// formed again.
template <int NCB, int MODE>
__device__ __forceinline__ void follow_reference(State<NCB>& st, const f32x4_t (&y)[NCB][2],
                                                 const Consts& cs, u32x4_t (&pb)[NCB]) {
  uint32_t most = 0u;
#pragma unroll
  for (int cb = 0; cb < NCB; ++cb)
#pragma unroll
    for (int i = 0; i < 4; ++i) most = max_u16x2(most, pb[cb][i]);
  const bool past = (most >> 16) > kLazyBits || (most & 0xffffu) > kLazyBits;
  if (__builtin_expect(__any(past), 0)) {
    raise_reference<NCB, MODE>(st, y, cs);
    exponentials<NCB, MODE>(st, y, cs, pb);
  }
}

template <int NCB>
__device__ __forceinline__ void sum_weights(State<NCB>& st, const u32x4_t (&pb)[NCB]) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int cb = 0; cb < NCB; ++cb) {
      const uint32_t two = pb[cb][i];
      st.l[cb] = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, two),
                                                 __builtin_bit_cast(bf16x2_t, kOnes2), st.l[cb],
                                                 false);
    }
}

template <int NCB, int MODE>
__device__ __forceinline__ void weights(const ScoredParams& p, const Columns<NCB>& c,
                                        State<NCB>& st, f32x4_t (&y)[NCB][2], int j0, int lg,
                                        const Consts& cs, bool masked, u32x4_t (&pb)[NCB]) {
  shape_scores<NCB, MODE>(c, y, j0, lg, cs);
  if constexpr (MODE == kCapNear) {
    if (__builtin_expect(masked || !st.settled, 0)) {
      if (masked) mask_scores<NCB, MODE>(p, c, y, j0, lg);
      if (!st.settled) settle_reference<NCB>(st, y, cs);
    }
    exponentials<NCB, MODE>(st, y, cs, pb);
  } else {
    if (__builtin_expect(masked, 0)) mask_scores<NCB, MODE>(p, c, y, j0, lg);
    exponentials<NCB, MODE>(st, y, cs, pb);
    follow_reference<NCB, MODE>(st, y, cs, pb);
  }
  sum_weights<NCB>(st, pb);
}

__device__ __forceinline__ bool not_finite(uint32_t half) { return (half & 0x7f80u) == 0x7f80u; }
__device__ __forceinline__ uint32_t finite_or_zero(uint32_t w) {
  return (not_finite(w) ? 0u : w & 0xffffu) | (not_finite(w >> 16) ? 0u : w & 0xffff0000u);
}

// LDS image of a K or V tile: row r (key) is 256 bytes; K's 16-byte chunk ch
// lies at chunk ch ^ (r & 15), V's at ch ^ 2 (r & 7).  A K operand read takes
// one chunk of 16 rows per lane group, a V operand read (transposed, 8 bytes a
// lane) 32 bytes of four rows per lane group: either way the lanes served
// together lie on distinct banks without padding, so a tile is eight whole
// 1 KiB loads.  (V rows permuted so that a lane's outputs are 32 consecutive
// dims read two lane groups from the same banks: 2 extra cycles per V read.)
struct LdsAddr {
  int k;  // K operand d: row lm, chunk 4 d + lg, at k ^ (d << 6)
  int v;  // V operand jj: row 4 lg + lm / 4, dims 16 jj + 4 (lm % 4) .., at v ^ (jj << 5)
};
__device__ __forceinline__ LdsAddr lds_addrs(int lm, int lg) {
  LdsAddr a;
  const int vr = 4 * lg + (lm >> 2), piece = lm & 3;
  a.k = lm * 256 + ((lg ^ lm) << 4);
  a.v = vr * 256 + (((piece >> 1) ^ ((vr & 7) << 1)) << 4) + (piece & 1) * 8;
  return a;
}
__device__ __forceinline__ int k_swizzle(int row) { return row & 15; }
__device__ __forceinline__ int v_swizzle(int row) { return (row & 7) << 1; }

__device__ __forceinline__ u32x4_t read_k1(const char* kt, const LdsAddr& a, int h, int d) {
  return *reinterpret_cast<const u32x4_t*>(kt + (a.k ^ (d << 6)) + h * 4096);
}
__device__ __forceinline__ void read_k(u32x4_t (&k)[2][4], const char* kt, const LdsAddr& a) {
#pragma unroll
  for (int d = 0; d < 4; ++d)
#pragma unroll
    for (int h = 0; h < 2; ++h) k[h][d] = read_k1(kt, a, h, d);
}

__device__ __forceinline__ u32x4_t read_v1(const char* vt, const LdsAddr& a, int jj) {
  const char* s = vt + (a.v ^ (jj << 5));
  const u32x2_t lo = lds_read_tr16(s), hi = lds_read_tr16(s + 4096);
  return u32x4_t{lo[0], lo[1], hi[0], hi[1]};
}
__device__ __forceinline__ void read_v(u32x4_t (&v)[8], const char* vt, const LdsAddr& a) {
#pragma unroll
  for (int jj = 0; jj < 8; ++jj) v[jj] = read_v1(vt, a, jj);
}

// In a masked tile a column's P is 0 at keys it does not see, but 0 times an
// infinity or NaN held there would still reach its sum: such values are taken
// out of the operand, and the answer says so (add_not_finite then gives them
// to the columns that see them, after the loop).
__device__ __forceinline__ bool take_out_not_finite(u32x4_t (&v)[8]) {
  uint32_t most = 0u;
#pragma unroll
  for (int jj = 0; jj < 8; ++jj)
#pragma unroll
    for (int i = 0; i < 4; ++i) most = max_u16x2(most, v[jj][i] & 0x7fff7fffu);
  if (__builtin_expect(!__any(not_finite(most) || not_finite(most >> 16)), 1)) return false;
#pragma unroll
  for (int jj = 0; jj < 8; ++jj)
#pragma unroll
    for (int i = 0; i < 4; ++i) v[jj][i] = finite_or_zero(v[jj][i]);
  return true;
}

// O^T += V^T P^T.
template <int NCB>
__device__ __forceinline__ void weigh(State<NCB>& st, const u32x4_t (&v)[8],
                                      const u32x4_t (&pb)[NCB]) {
#pragma unroll
  for (int jj = 0; jj < 8; ++jj)
#pragma unroll
    for (int cb = 0; cb < NCB; ++cb) st.o[cb][jj] = mfma_bf16(v[jj], pb[cb], st.o[cb][jj]);
}

// Infinities and NaN of one tile's V rows, added to the columns that see their
// key: they decide its result whatever their weight.  Rare, so plain: each row
// once, from memory.
template <int NCB>
__device__ __forceinline__ void add_not_finite(const ScoredParams& p, const Columns<NCB>& c,
                                               State<NCB>& st, const uint16_t* v, int rows, int j0,
                                               int lg) {
  uint32_t vis[NCB];
#pragma unroll
  for (int cb = 0; cb < NCB; ++cb) vis[cb] = visible_bits<NCB>(p, c, cb, j0);
#pragma unroll 1
  for (int r = 0; r < rows; ++r) {
#pragma unroll
    for (int jj = 0; jj < 8; ++jj) {
      const u32x2_t w = *reinterpret_cast<const u32x2_t*>(v + r * p.v_row + 16 * jj + 4 * lg);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t half = (w[i >> 1] >> (16 * (i & 1))) & 0xffffu;
        const float add = not_finite(half) ? bf16_bits_to_f32(half) : 0.f;
#pragma unroll
        for (int cb = 0; cb < NCB; ++cb)
          st.o[cb][jj][i] += ((vis[cb] >> r) & 1u) ? add : 0.f;
      }
    }
  }
}

// ---------------------------------------------------------------------------
// The plan: which item and tile a share starts at.  Every wave works it out
// for itself from the device's lengths (no barrier before the first load).
// ---------------------------------------------------------------------------
// Virtual tiles that every item adds to its cost: its query loads, its pipe's
// start, its masked tiles (two to three times an ordinary one) and its
// epilogue.  Measured with 3, 7, 12, 19, 26 of them: four prompts with images
// 267, 252, 239, 248, 259 us, four windowed chunks 60, 55, 52, 55, 57 us, 37
// trees 74, 71, 69, 71, 74 us; long items do not care.
constexpr int kItemCost = 12;

struct Where {
  int seq, grp, block, tile;  // tile: offset inside the item
  int64_t total;              // cost of the whole call
};

__device__ __forceinline__ int block_cost(const ScoredParams& p, const SeqGeo& g, int pre, int c) {
  if (p.whole) return 1;
  const TileRange r = block_tiles(p, g, pre, c);
  return r.t1 - r.t0 + kItemCost;
}

// Cost and column blocks of lane's sequence (lane plan).
__device__ __forceinline__ int lane_seq(const ScoredParams& p, int i, SeqGeo& g, int& pre) {
  g = SeqGeo{};
  pre = 0;
  if (i >= p.batch) return 0;
  g = load_seq<false>(p, i);
  pre = p.prefix != nullptr ? p.prefix[i] : 0;
  const int nb = num_blocks_of(p, g.sq);
  int cost = 0;
  for (int c = 0; c < nb; ++c) cost += block_cost(p, g, pre, c);
  return cost * p.head_groups;
}

// The same for a wave-uniform sequence, its blocks across the lanes.
__device__ __forceinline__ int wave_seq(const ScoredParams& p, int i, int lane, SeqGeo& g,
                                        int& pre) {
  g = load_seq<true>(p, i);
  pre = p.prefix != nullptr ? table_entry(p.prefix, i) : 0;
  const int nb = num_blocks_of(p, g.sq);
  int cost = 0;
  for (int c = 0; c < nb; c += 64)
    cost += wave_sum(c + lane < nb ? block_cost(p, g, pre, c + lane) : 0);
  return cost * p.head_groups;
}

__device__ __forceinline__ int first_lane(uint64_t m) { return __builtin_ctzll(m); }

// Finds position `at` (share * size, size from the total) in the concatenated
// items; false when it lies past the end.
__device__ __forceinline__ bool plan_share(const ScoredParams& p, int lane, int share, int shares,
                                           Where& w, SeqGeo& g, int& pre, int& size) {
  int total = 0, cost = 0;
  SeqGeo mine = {};  // lane_plan: this lane's sequence
  int mine_pre = 0;
  g = SeqGeo{};
  pre = 0;
  if (p.whole && (p.batch == 1 || p.cu_q == nullptr)) {
    // As many items in each sequence: no walk, and (small calls are all
    // latency) no division where the quotient is plain.
    g = load_seq<true>(p, 0);
    const int n = g.sq <= p.tokens_per_block ? min(g.sq, 1) : num_blocks_of(p, g.sq);
    const int each = n * p.head_groups;
    w.total = each * p.batch;
    size = w.total <= shares ? 1 : (w.total + shares - 1) / shares;
    const int64_t at = int64_t(share) * size;
    if (at >= w.total) return false;
    w.seq = p.batch == 1 ? 0 : int(at) / each;
    if (w.seq != 0) g = load_seq<true>(p, w.seq);
    if (p.prefix != nullptr) pre = table_entry(p.prefix, w.seq);
    const int rem = int(at) - w.seq * each;
    w.grp = n == 1 ? rem : rem / n;
    w.block = rem - w.grp * n;
    w.tile = 0;
    return true;
  }
  if (p.lane_plan) {
    for (int i = 0; i < p.batch; i += 64) {
      cost = lane_seq(p, i + lane, mine, mine_pre);
      total += wave_sum(cost);
    }
  } else {
    for (int i = 0; i < p.batch; ++i) total += wave_seq(p, i, lane, g, pre);
  }
  w.total = total;
  size = max(p.whole ? 1 : p.min_share, (total + shares - 1) / shares);
  const int64_t at64 = int64_t(share) * size;
  if (at64 >= total) return false;
  const int at = int(at64);
  int acc = 0, seq = -1, start = 0;
  if (p.lane_plan) {
    for (int i = 0; i < p.batch; i += 64) {
      if (p.batch > 64) cost = lane_seq(p, i + lane, mine, mine_pre);
      const int upto = wave_scan_add(cost);
      const uint64_t hit = __ballot(acc + upto > at);
      if (hit != 0) {
        const int l = first_lane(hit);
        seq = i + l;
        start = acc + __builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(cost, l);
        g.q0 = __builtin_amdgcn_readlane(mine.q0, l);
        g.sq = __builtin_amdgcn_readlane(mine.sq, l);
        g.sk = __builtin_amdgcn_readlane(mine.sk, l);
        g.p0 = __builtin_amdgcn_readlane(mine.p0, l);
        pre = __builtin_amdgcn_readlane(mine_pre, l);
        break;
      }
      acc += __builtin_amdgcn_readlane(upto, 63);
    }
  } else {
    for (int i = 0; i < p.batch; ++i) {
      cost = wave_seq(p, i, lane, g, pre);
      if (acc + cost > at) {
        seq = i;
        start = acc;
        break;
      }
      acc += cost;
    }
  }
  if (seq < 0) return false;
  w.seq = seq;
  // Inside the sequence: head groups in turn, each over all column blocks.
  const int n = num_blocks_of(p, g.sq);
  const int rem = at - start;
  if (n == 1) {
    const int each = block_cost(p, g, pre, 0);
    w.grp = rem / each;
    w.block = 0;
    w.tile = rem - w.grp * each;
    return true;
  }
  int each = 0;
  for (int c = 0; c < n; c += 64)
    each += wave_sum(c + lane < n ? block_cost(p, g, pre, c + lane) : 0);
  w.grp = rem / each;
  int left = rem - w.grp * each;
  for (int c = 0; c < n; c += 64) {
    const int one = c + lane < n ? block_cost(p, g, pre, c + lane) : 0;
    const int upto = wave_scan_add(one);
    const uint64_t hit = __ballot(upto > left);
    if (hit != 0) {
      const int l = first_lane(hit);
      w.block = c + l;
      w.tile = left - (__builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(one, l));
      return true;
    }
    left -= __builtin_amdgcn_readlane(upto, 63);
  }
  return false;
}

// ---------------------------------------------------------------------------
// Tile addresses.
// ---------------------------------------------------------------------------
// The block id of tile's page in a sequence's table (0 for fresh rows), -1
// past the table.
__device__ __forceinline__ int page_entry(const ScoredParams& p, int seq, int tile) {
  if (p.tables == nullptr) return 0;
  const int page = uniform(div_small(tile, p.page_tiles, p.page_rcp));
  return page < p.max_blocks ? table_entry(p.tables, int64_t(seq) * p.bt_stride + page) : -1;
}

struct TileSource {
  const uint16_t* k;
  const uint16_t* v;
  int rows;  // valid rows, 0: reads zeros
};
__device__ __forceinline__ TileSource tile_source(const ScoredParams& p, int64_t fresh0, int sk,
                                                  int head, int tile, int blk) {
  const int j0 = tile * kTile;
  int64_t row;
  int rows = min(kTile, sk - j0);
  if (p.tables != nullptr) {
    if (blk < 0 || blk >= p.num_blocks) rows = 0;
    const int page = uniform(div_small(tile, p.page_tiles, p.page_rcp));
    row = rows > 0 ? int64_t(blk) * p.page + (j0 - page * p.page) : 0;
  } else {
    row = fresh0 + j0;
  }
  TileSource t;
  t.k = p.k + row * p.k_row + head * p.k_head;
  t.v = p.v + row * p.v_row + head * p.v_head;
  t.rows = rows;
  return t;
}

// Lane's byte offset of load m (rows 4 m .. 4 m + 3) of a tile.
struct DmaOffsets {
  int base[4];  // m = 0 .. 3
  int step;     // 16 rows
};
template <bool kV>
__device__ __forceinline__ DmaOffsets dma_offsets(int lane, int64_t row_elems) {
  DmaOffsets o;
  const int lr = lane >> 4, slot = lane & 15;
#pragma unroll
  for (int m = 0; m < 4; ++m) {
    const int r = 4 * m + lr;
    o.base[m] = r * int(row_elems) * 2 + ((slot ^ (kV ? v_swizzle(r) : k_swizzle(r))) << 4);
  }
  o.step = 16 * int(row_elems) * 2;
  return o;
}
__device__ __forceinline__ int tensor_bytes(int rows, int64_t row_elems) {
  return rows > 0 ? (rows - 1) * int(row_elems) * 2 + kD * 2 : 0;
}

template <bool kStream>
__device__ __forceinline__ void load_rows(const i32x4_t& rsrc, const DmaOffsets& o, int m,
                                          uint32_t lds) {
  const int off = o.base[m & 3] + (m >> 2) * o.step;
  if constexpr (kStream) {
    dma_to_lds(rsrc, off, lds + m * 1024);
  } else {
    dma_to_lds_cached(rsrc, off, lds + m * 1024);
  }
}

template <int N>
__device__ __forceinline__ void wait_loads() {  // all but the newest N
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void lds_done() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// ---------------------------------------------------------------------------
// The kernel.  NW waves.  Turns forms: a step has KW tiles, and NW / KW waves
// attend each, 16 NCB columns a wave.  KW = NW is the private form, where waves
// split over heads_per_wg kv heads and tile phases.
// ---------------------------------------------------------------------------
template <int NW, int NCB, int KW>
struct Form {
  static constexpr bool kPrivate = KW == NW;
  static constexpr int kColWaves = kPrivate ? 1 : NW / KW;
  static constexpr int kColumns = 16 * NCB * kColWaves;  // per kv head
  static constexpr int kSlots = 8;  // tiles held: one a wave, or a ring
  static constexpr int kSlotBytes = kSlots * 2 * kTensor;
  // A wave's state while tile phases are joined: [cb][8][64 lanes] of O, then
  // [cb][64] of (reference, sum).
  static constexpr int kStateBytes = NCB * (8 * 64 * 16 + 64 * 8);
  static constexpr int kJoinBytes = KW > 1 ? NW * kStateBytes : 0;
  static constexpr int kLds = kSlotBytes > kJoinBytes ? kSlotBytes : kJoinBytes;
  static_assert(NW == kSlots && (kPrivate || KW <= 2));
  static_assert(kLds <= 160 * 1024, "one workgroup per CU");
};

template <int NCB>
__device__ __forceinline__ void put_state(char* at, const State<NCB>& st, int lane) {
#pragma unroll
  for (int cb = 0; cb < NCB; ++cb) {
#pragma unroll
    for (int jj = 0; jj < 8; ++jj)
      *reinterpret_cast<f32x4_t*>(at + (cb * 8 + jj) * 1024 + lane * 16) = st.o[cb][jj];
    *reinterpret_cast<float2*>(at + NCB * 8192 + cb * 512 + lane * 8) =
        float2{st.mu[cb], st.l[cb]};
  }
}

// Join the states of kPhases waves, kept `step` apart: the wave of phase f
// makes a kPhases-th of the rows of O^T and hands them on.
template <int NCB, int kPhases, class Emit>
__device__ __forceinline__ void join_states(const char* at, int step, int f, int lane,
                                            const Emit& emit) {
#pragma unroll
  for (int cb = 0; cb < NCB; ++cb) {
    float2 ml[kPhases];
    float b[kPhases];
    f32x4_t part[8];
#pragma unroll
    for (int i = 0; i < kPhases; ++i)
      ml[i] = *reinterpret_cast<const float2*>(at + i * step + NCB * 8192 + cb * 512 + lane * 8);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      part[i] = *reinterpret_cast<const f32x4_t*>(
          at + (i % kPhases) * step + (cb * 8 + f * (8 / kPhases) + i / kPhases) * 1024 +
          lane * 16);
    float top = ml[0].x, l = 0.f;
#pragma unroll
    for (int i = 1; i < kPhases; ++i) top = fmaxf(top, ml[i].x);
#pragma unroll
    for (int i = 0; i < kPhases; ++i) {
      b[i] = __builtin_amdgcn_exp2f(ml[i].x - top);
      l += ml[i].y * b[i];
    }
#pragma unroll
    for (int i = 0; i < 8; i += kPhases) {
      f32x4_t o = part[i] * b[0];
#pragma unroll
      for (int j = 1; j < kPhases; ++j) o += part[i + j] * b[j];
      part[i / kPhases] = o;
    }
    emit(cb, f * (8 / kPhases), 8 / kPhases, part, top, l);
  }
}

template <int NW, int NCB, int KW, int MODE>
__global__ void __launch_bounds__(64 * NW)
    __attribute__((amdgpu_waves_per_eu(NW / 4, NW / 4))) scored_kernel(ScoredParams p) {
  using F = Form<NW, NCB, KW>;
  extern __shared__ __align__(1024) char smem[];
  const int lane = threadIdx.x & 63, wave = uniform(int(threadIdx.x >> 6));
  const int lm = lane & 15, lg = lane >> 4;
  // Consecutive shares on one XCD (workgroup b runs on XCD b mod 8).
  const int grid = gridDim.x;
  const int share = grid % 8 == 0 ? (blockIdx.x % 8) * (grid / 8) + blockIdx.x / 8 : blockIdx.x;

  touch_kernel_args(int(sizeof(ScoredParams)));
  // The tables' first line on its way beside the lengths'.
  int warm = p.whole && p.tables != nullptr && p.max_blocks > 0 ? table_entry(p.tables, 0) : 0;
  Where w;
  SeqGeo g;
  int size, pre;
  const bool live = plan_share(p, lane, share, grid, w, g, pre, size);
  if (!live) {
    if (threadIdx.x == 0 && !p.whole) p.rec[share] = int4{0, 0, 0, 0};
    return;
  }

  asm volatile("" ::"s"(warm));
  const int hs = F::kPrivate ? wave % p.heads_per_wg : 0;
  const int phases = F::kPrivate ? NW / p.heads_per_wg : KW;
  const int phase = F::kPrivate ? wave / p.heads_per_wg : wave / F::kColWaves;
  const int cw = F::kPrivate ? 0 : wave % F::kColWaves;
  const LdsAddr la = lds_addrs(lm, lg);
  const uint32_t lds0 = lds_addr(smem);
  Consts cs;
  cs.c2 = p.scale * kLog2e;
  cs.zc = p.cap > 0.f ? 2.f * kLog2e * p.scale / p.cap : 0.f;
  cs.a = p.cap * kLog2e;
  cs.a2 = 2.f * cs.a;
  cs.z = p.cap > 0.f ? p.scale / p.cap : 0.f;

  const int col0 = cw * NCB * 16;
  const int wave_t0 = uniform(div_small(col0, p.group, p.group_rcp));
  const int wave_t1 = min(uniform(div_small(col0 + NCB * 16 - 1, p.group, p.group_rcp)),
                          p.tokens_per_block - 1);

  const int end = int(min(w.total, int64_t(share + 1) * size));
  int pos = share * size;
  int nblocks = g.sq <= p.tokens_per_block ? 1 : num_blocks_of(p, g.sq);
  while (true) {
    const TileRange range = block_tiles(p, g, pre, w.block);
    const int tiles = range.t1 - range.t0;
    const int seg0 = w.tile, seg1 = p.whole ? tiles : min(tiles, w.tile + (end - pos));
    if (!p.whole && pos + tiles + kItemCost - w.tile >= end && threadIdx.x == 0) {
      // The share's last item: where it goes on, if it began here.
      const int last = tiles > 0 ? (pos - w.tile + tiles - 1) / size : share;
      const int b0 = w.block * p.tokens_per_block;
      p.rec[share] = int4{g.q0 + b0, min(g.sq - b0, p.tokens_per_block), w.grp,
                          w.tile == 0 && last > share ? last : 0};
    }
    if (seg0 < seg1 || (tiles == 0 && w.tile == 0)) {
      const int head = w.grp * p.heads_per_wg + hs;
      const int64_t fresh0 =
          p.tables == nullptr ? max(0, table_entry(p.cu_k, w.seq)) : 0;
      const int p0 = g.p0;
      const int b0 = w.block * p.tokens_per_block;  // the block's first token
      const int tmax = min(g.sq, b0 + p.tokens_per_block) - 1;

      Columns<NCB> c;
      const uint16_t* qp[NCB];
#pragma unroll
      for (int cb = 0; cb < NCB; ++cb) {
        // (columns past the block repeat its last token)
        const ColumnOf col = column_of(p, col0, cb);
        const int t = min(b0 + col.token, tmax);
        qp[cb] = p.q + int64_t(g.q0 + t) * p.q_st + int64_t(head * p.group + col.head) * p.q_sh;
        c.place[cb] = c.slope2[cb] = 0.f;
        if constexpr (MODE == kDistance || MODE == kCapDistance) {
          c.place[cb] = float(p0 + (p.mask == nullptr ? t : p.places[g.q0 + t]));
          c.slope2[cb] = p.slopes[head * p.group + col.head] * kLog2e;
        }
      }
      c.first = b0;
      c.last = tmax;
      c.col0 = col0;
      c.bits = p.mask != nullptr ? p.mask + int64_t(g.q0) * p.mask_words : nullptr;
      c.depths = p.places != nullptr ? p.places + g.q0 : nullptr;
      c.pre = pre;
      c.p0 = p0;
      c.sk = g.sk;
      c.sq = g.sq;
      {
        const int ta = min(b0 + wave_t0, tmax), tb = min(b0 + wave_t1, tmax);
        if (p.mask == nullptr) {
          c.full_lo = p.window > 0 ? p0 + tb + 1 - p.window : 0;
          // A two-way prefix makes |p - j| bend inside it.
          c.full_hi = min(g.sk, MODE == kDistance || MODE == kCapDistance
                                    ? p0 + ta + 1 : max(p0 + ta + 1, pre));
        } else {
          c.full_lo = p.window > 0 ? p0 + g.sq - p.window : 0;  // depth < sq
          c.full_hi = min(p0, g.sk);
        }
      }
      u32x4_t q[NCB][4];
#pragma unroll
      for (int cb = 0; cb < NCB; ++cb)
#pragma unroll
        for (int d = 0; d < 4; ++d)
          q[cb][d] = *reinterpret_cast<const u32x4_t*>(qp[cb] + 32 * d + 8 * lg);
      // The queries are waited for once the first tiles are on their way: the
      // compiler's wait for them covers those too.
      auto settle = [&] {
#pragma unroll
        for (int cb = 0; cb < NCB; ++cb) {
          if constexpr (MODE == kDistance || MODE == kCapDistance)
            asm volatile("" : "+v"(c.place[cb]), "+v"(c.slope2[cb]));
#pragma unroll
          for (int d = 0; d < 4; ++d) asm volatile("" : "+v"(q[cb][d]));
        }
      };
      State<NCB> st;
      reset<NCB>(st);
      const int t_begin = range.t0 + seg0, t_end = range.t0 + seg1;
      bool odd = false;  // a masked tile held infinities or NaN
      if constexpr (F::kPrivate) {
        // Wave-private slots: K 8 KiB, V 8 KiB.  The next tile's K load goes
        // out as soon as this tile's K is in registers, its V load likewise.
        const DmaOffsets ko = dma_offsets<false>(lane, p.k_row);
        const DmaOffsets vo = dma_offsets<true>(lane, p.v_row);
        const uint32_t kl = lds0 + wave * (2 * kTensor), vl = kl + kTensor;
        const char* kt = smem + wave * (2 * kTensor);
        const char* vt = kt + kTensor;
        auto issue_k = [&](const TileSource& t) {
          const i32x4_t r = raw_rsrc(t.k, tensor_bytes(t.rows, p.k_row));
#pragma unroll
          for (int m = 0; m < 8; ++m) load_rows<true>(r, ko, m, kl);
        };
        auto issue_v = [&](const TileSource& t) {
          const i32x4_t r = raw_rsrc(t.v, tensor_bytes(t.rows, p.v_row));
#pragma unroll
          for (int m = 0; m < 8; ++m) load_rows<true>(r, vo, m, vl);
        };
        int t = t_begin + phase;
        if (t < t_end) {
          const TileSource src = tile_source(p, fresh0, g.sk, head, t, page_entry(p, w.seq, t));
          issue_k(src);
          issue_v(src);
        }
        settle();
        u32x4_t k[2][4];
        for (; t < t_end; t += phases) {
          const bool more = t + phases < t_end;
          TileSource next = {};
          if (more)
            next = tile_source(p, fresh0, g.sk, head, t + phases,
                               page_entry(p, w.seq, t + phases));
          const int j0 = t * kTile;
          const bool masked = j0 < c.full_lo || j0 + kTile > c.full_hi;
          wait_loads<8>();
          read_k(k, kt, la);
          lds_done();
          if (more) issue_k(next);
          f32x4_t sl[NCB][2];
          u32x4_t v[8], pb[NCB];
          logits<NCB>(k, q, sl);
          weights<NCB, MODE>(p, c, st, sl, j0, lg, cs, masked, pb);
          if (more) {
            wait_loads<8>();
          } else {
            wait_loads<0>();
          }
          read_v(v, vt, la);
          lds_done();
          if (more) issue_v(next);
          if (masked) odd |= take_out_not_finite(v);
          weigh<NCB>(st, v, pb);
        }
      } else {
        // The waves take turns: while the first four (one on each SIMD) run
        // their products and read operands, the other four run a softmax, and
        // a barrier swaps them, so that matrix and vector units work side by
        // side.  Products of a turn: S of the wave's tile of step i and O of
        // its tile of step i - 1.  A step has KW tiles: one that all waves
        // attend, or one for each half.  Step s is last read in the later
        // half's turn s, so its slots are loaded again a turn on, kRing - 1
        // steps ahead.
        constexpr int kRing = F::kSlots / KW;
        const bool later = wave >= NW / 2;
        const int n = t_end - t_begin, steps = (n + KW - 1) / KW;
        const int own = KW == 2 && later ? 1 : 0;  // the wave's tile of a step
        // A wave's part of a tile: rows 4 wave .. + 3 of K and of V.
        const int drow = 4 * wave + (lane >> 4);
        const int kvoff = drow * int(p.k_row) * 2 + (((lane & 15) ^ k_swizzle(drow)) << 4);
        const int vvoff = drow * int(p.v_row) * 2 + (((lane & 15) ^ v_swizzle(drow)) << 4);
        // The loads' resources move along a page by adds; a page's block (the
        // next one's entry is read a page ahead), and a ragged last tile, are
        // set apart, once each.
        const bool paged = p.tables != nullptr;
        const int32_t* table = p.tables + int64_t(w.seq) * p.bt_stride;
        int page = paged ? uniform(div_small(t_begin, p.page_tiles, p.page_rcp)) : 0;
        auto entry = [&](int pg) { return paged && pg < p.max_blocks ? table_entry(table, pg) : -1; };
        int blk = entry(page), ahead = entry(page + 1);
        int to_load = n;  // tiles not yet asked for
        int to_stop;      // of them, before the next special one
        uint32_t at = lds0 + wave * 1024;
        const uint32_t at_end = lds0 + F::kSlots * 2 * kTensor;
        i32x4_t kr, vr;
        const int kstep = kTile * int(p.k_row) * 2, vstep = kTile * int(p.v_row) * 2;
        const int whole = min(n, g.sk / kTile - t_begin);  // tiles with all 32 keys
        auto aim = [&](int first) {  // resources of the tile `first` tiles into the page
          const bool there = !paged || (blk >= 0 && blk < p.num_blocks);
          const int done = n - to_load;
          const int64_t row = paged ? int64_t(there ? blk : 0) * p.page + first * kTile
                                    : fresh0 + int64_t(t_begin + done) * kTile;
          const int rows = !there || to_load <= 0 ? 0
                           : done < whole         ? kTile
                                                  : g.sk - (t_begin + done) * kTile;
          kr = raw_rsrc(p.k + row * p.k_row + head * p.k_head, tensor_bytes(rows, p.k_row));
          vr = raw_rsrc(p.v + row * p.v_row + head * p.v_head, tensor_bytes(rows, p.v_row));
          to_stop = paged ? p.page_tiles - first : 1 << 30;
          to_stop = to_load <= 0 ? 1 << 30 : min(to_stop, done < whole ? whole - done : to_load);
        };
        aim(t_begin - page * p.page_tiles);
        auto load = [&] {  // the next tile's two loads, and where the one after lies
          uint32_t m0;
          asm volatile(
              "s_mov_b32 %0, m0\n\t"
              "s_mov_b32 m0, %3\n\t"
              "s_nop 0\n\t"
              "buffer_load_dwordx4 %1, %4, 0 offen lds\n\t"
              "s_add_u32 m0, m0, %6\n\t"
              "s_nop 0\n\t"
              "buffer_load_dwordx4 %2, %5, 0 offen lds\n\t"
              "s_mov_b32 m0, %0"
              : "=&s"(m0)
              : "v"(kvoff), "v"(vvoff), "s"(at), "s"(kr), "s"(vr), "n"(kTensor)
              : "memory", "scc");
          at += 2 * kTensor;
          if (at >= at_end) at -= F::kSlots * 2 * kTensor;
          --to_load;
          --to_stop;
          const uint64_t ka = (uint64_t(uint32_t(kr[1])) << 32 | uint32_t(kr[0])) + uint32_t(kstep);
          const uint64_t va = (uint64_t(uint32_t(vr[1])) << 32 | uint32_t(vr[0])) + uint32_t(vstep);
          kr[0] = int(uint32_t(ka));
          kr[1] = int(uint32_t(ka >> 32));
          vr[0] = int(uint32_t(va));
          vr[1] = int(uint32_t(va >> 32));
        };
        auto steer = [&] {  // a new page, the ragged tile, or the end (rows 0: zeros)
          if (__builtin_expect(to_stop > 0, 1)) return;
          int first = t_begin + (n - to_load) - page * p.page_tiles;
          if (paged && first >= p.page_tiles) {
            first -= p.page_tiles;
            ++page;
            blk = ahead;
            ahead = entry(page + 1);
            smem_drain();
          }
          aim(first);
        };
        // Loads a wave may still have on the way when what the next turns read
        // (V of step i + 1, K of step i + 2) has to be in place: waited for
        // ahead of the barrier before the first half's turn.  The later half
        // does so after its softmax, a turn early, where the ring is deep
        // enough for that.
        constexpr bool kEarly = KW == 1;
        constexpr int kNewer = 2 * KW * (kRing - (kEarly ? 4 : 3));
#pragma unroll 1
        for (int i = 0; i < KW * (kRing - 1); ++i) {
          load();
          steer();
        }
        settle();
        wait_loads<kNewer>();
        pf_barrier();
        u32x4_t k[2][4];
        read_k(k, smem + own * 2 * kTensor, la);
        lds_done();
        if (later) pf_barrier();
        f32x4_t sl[NCB][2];
        u32x4_t v[8] = {}, pb[NCB] = {};  // (nothing to weigh in the first turn)
        // Tiles that every column sees whole, counted from t_begin.  (Tiles
        // that none of a wave's columns sees are attended with every weight 0.)
        const int full0 = (max(c.full_lo, 0) + kTile - 1) / kTile - t_begin;
        const int full1 = c.full_hi / kTile - t_begin;
        int always = 1;
        asm volatile("" : "+s"(always));
        for (int i = 0; i <= steps; ++i) {
          // The next tile's K and this one's V operands come in under the two
          // products, as these let go of the ones before.
          const int u = KW * i + own;
          const char* vt = smem + (u & (F::kSlots - 1)) * (2 * kTensor) + kTensor;
          const char* next = smem + ((u + KW) & (F::kSlots - 1)) * (2 * kTensor);
          __builtin_amdgcn_s_setprio(1);
          // (the opaque test, always true, only keeps the two products apart:
          // one block would be scheduled as a single chain)
          if (always) {
            load();
            if constexpr (KW == 2) {
              steer();
              load();
            }
#pragma unroll
            for (int d = 0; d < 4; ++d) {
#pragma unroll
              for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int cb = 0; cb < NCB; ++cb)
                  sl[cb][h] = mfma_bf16(k[h][d], q[cb][d],
                                        d == 0 ? f32x4_t{0.f, 0.f, 0.f, 0.f} : sl[cb][h]);
                k[h][d] = read_k1(next, la, h, d);
              }
            }
#pragma unroll
            for (int x = 0; x < 8; ++x) {
              __builtin_amdgcn_sched_group_barrier(0x008, NCB, 0);  // MFMA
              __builtin_amdgcn_sched_group_barrier(0x004, 2, 0);    // SALU
              __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);    // LDS read
            }
          }
#pragma unroll
          for (int jj = 0; jj < 8; ++jj) {
#pragma unroll
            for (int cb = 0; cb < NCB; ++cb)
              st.o[cb][jj] = mfma_bf16(v[jj], pb[cb], st.o[cb][jj]);
            v[jj] = read_v1(vt, la, jj);
          }
#pragma unroll
          for (int jj = 0; jj < 8; ++jj) {
            __builtin_amdgcn_sched_group_barrier(0x008, NCB, 0);  // MFMA
            __builtin_amdgcn_sched_group_barrier(0x002, 1, 0);    // VALU: addresses
            __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);    // LDS reads
          }
          __builtin_amdgcn_s_setprio(0);
          __builtin_amdgcn_sched_barrier(0);
          if constexpr (!kEarly)
            if (later) wait_loads<kNewer>();
          pf_barrier();
          __builtin_amdgcn_sched_barrier(0);
          if (__builtin_expect(i < steps, 1)) {
            steer();
            const bool masked = u < full0 || u >= full1;
            if (__builtin_expect(masked, 0)) odd |= take_out_not_finite(v);
            // (a step's second tile may lie past the segment)
            const bool gone = KW == 2 && u >= n;
            weights<NCB, MODE>(p, c, st, sl, gone ? kNoKey : (t_begin + u) * kTile, lg, cs,
                               masked || gone, pb);
            if (kEarly || !later) wait_loads<kNewer>();
          }
          __builtin_amdgcn_sched_barrier(0);
          pf_barrier();
          __builtin_amdgcn_sched_barrier(0);
        }
        if (!later) pf_barrier();
        wait_loads<0>();
      }

      if (__builtin_expect(odd, 0)) {
        for (int t = t_begin + phase; t < t_end; t += phases) {
          const int j0 = t * kTile;
          if (j0 >= c.full_lo && j0 + kTile <= c.full_hi) continue;
          const TileSource src = tile_source(p, fresh0, g.sk, head, t, page_entry(p, w.seq, t));
          add_not_finite<NCB>(p, c, st, src.v, src.rows, j0, lg);
        }
      }
#pragma unroll
      for (int cb = 0; cb < NCB; ++cb) st.l[cb] = rows4_sum(st.l[cb]);
      // Rows 16 jj .. 16 (jj + n) of a column block of O^T: the item's result,
      // or a partial in slot 2 share + 1 (the piece that begins its item), else
      // 2 share.
      auto emit = [&](int cb, int jj0, int n, const f32x4_t* o, float mu, float l) {
        const ColumnOf co = column_of(p, col0, cb);
        if (co.token >= p.tokens_per_block || b0 + co.token > tmax) return;
        if (seg0 == 0 && seg1 == tiles) {
          const float inv = l != 0.f ? 1.f / l : 0.f;
          uint16_t* dst = p.out + int64_t(g.q0 + b0 + co.token) * p.o_st +
                          int64_t(head * p.group + co.head) * p.o_sh + 4 * lg + 16 * jj0;
#pragma unroll
          for (int i = 0; i < n; ++i) {
            const f32x4_t r = o[i] * inv;
            *reinterpret_cast<u32x2_t*>(dst + 16 * i) =
                u32x2_t{pack_bf16x2_fast(r[0], r[1]), pack_bf16x2_fast(r[2], r[3])};
          }
        } else {
          const int64_t slot = int64_t(2) * share + (seg0 == 0 ? 1 : 0);
          const int64_t col = (slot * p.heads_per_wg + hs) * F::kColumns +
                              (cw * NCB + cb) * 16 + lm;
          float* dst = p.part_o + col * kD + 4 * lg + 16 * jj0;
#pragma unroll
          for (int i = 0; i < n; ++i) *reinterpret_cast<f32x4_t*>(dst + 16 * i) = o[i];
          if (lg == 0 && jj0 == 0) p.part_ml[col] = float2{mu, l};
        }
      };
      if constexpr (KW > 1) {
        const int owners = NW / phases;
        const char* first = smem + (wave % owners) * F::kStateBytes;
        const int step = owners * F::kStateBytes;
        pf_barrier();
        put_state<NCB>(smem + wave * F::kStateBytes, st, lane);
        pf_barrier();
        if (phases == 2) {
          join_states<NCB, 2>(first, step, phase, lane, emit);
        } else if constexpr (F::kPrivate) {
          if (phases == 4) {
            join_states<NCB, 4>(first, step, phase, lane, emit);
          } else {
            join_states<NCB, 8>(first, step, phase, lane, emit);
          }
        }
        pf_barrier();
      } else {
        pf_barrier();  // the ring is free for the next item
#pragma unroll
        for (int cb = 0; cb < NCB; ++cb) emit(cb, 0, 8, st.o[cb], st.mu[cb], st.l[cb]);
      }
    }

    pos += p.whole ? 1 : tiles + kItemCost - w.tile;
    if (pos >= end) break;
    w.tile = 0;
    if (++w.block < nblocks) continue;
    w.block = 0;
    if (++w.grp < p.head_groups) continue;
    w.grp = 0;
    do {
      if (++w.seq >= p.batch) {
        if (threadIdx.x == 0 && !p.whole) p.rec[share] = int4{0, 0, 0, 0};
        return;
      }
      g = load_seq<true>(p, w.seq);
      pre = p.prefix != nullptr ? table_entry(p.prefix, w.seq) : 0;
      nblocks = num_blocks_of(p, g.sq);
    } while (nblocks == 0);
  }
}

// ---------------------------------------------------------------------------
// Join the partials of items cut between shares: workgroup (share, eight
// columns) takes the item that begins in the share and ends in another, 32
// lanes per column.
// ---------------------------------------------------------------------------
constexpr int kMergeColumns = 8;
constexpr int kMergeAhead = 4;  // pieces whose loads are in flight together
__global__ void __launch_bounds__(32 * kMergeColumns)
    scored_merge_kernel(ScoredParams p, int columns) {
  const int share = blockIdx.x;
  const int4 r = p.rec[share];
  if (r.w <= share) return;
  const int per_head = columns / kMergeColumns;
  const int hs = blockIdx.y / per_head;
  const int col = (blockIdx.y - hs * per_head) * kMergeColumns + int(threadIdx.x >> 5);
  const int head = r.z * p.heads_per_wg + hs;
  if (col >= r.y * p.group) return;
  const int lane = threadIdx.x & 31;
  const int64_t cols = int64_t(p.heads_per_wg) * columns, at = hs * columns + col;
  float top = kLowest, l = 0.f;
  f32x4_t o = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = share; s0 <= r.w; s0 += kMergeAhead) {
    float2 ml[kMergeAhead];
    f32x4_t part[kMergeAhead];
#pragma unroll
    for (int i = 0; i < kMergeAhead; ++i) {
      const int s = min(s0 + i, r.w);
      const int64_t c = (int64_t(2) * s + (s == share)) * cols + at;
      ml[i] = p.part_ml[c];
      part[i] = reinterpret_cast<const f32x4_t*>(p.part_o + c * kD)[lane];
    }
#pragma unroll
    for (int i = 0; i < kMergeAhead; ++i) {
      if (s0 + i > r.w) continue;
      const float next = fmaxf(top, ml[i].x);
      const float a = __builtin_amdgcn_exp2f(top - next);
      const float b = __builtin_amdgcn_exp2f(ml[i].x - next);
      top = next;
      l = l * a + ml[i].y * b;
      o = o * a + part[i] * b;
    }
  }
  const float inv = l != 0.f ? 1.f / l : 0.f;
  const int t = col / p.group;
  uint16_t* dst = p.out + int64_t(r.x + t) * p.o_st +
                  int64_t(head * p.group + col - t * p.group) * p.o_sh + 4 * lane;
  *reinterpret_cast<u32x2_t*>(dst) =
      u32x2_t{pack_bf16x2_fast(o[0] * inv, o[1] * inv), pack_bf16x2_fast(o[2] * inv, o[3] * inv)};
}

// Depth of each tree token: its mask's bits inside the tree but its own.
__global__ void __launch_bounds__(64) tree_depth_kernel(ScoredParams p, int32_t* depth) {
  const SeqGeo g = load_seq<true>(p, blockIdx.x);
  for (int t = threadIdx.x; t < g.sq; t += 64) {
    const uint32_t* m = p.mask + int64_t(g.q0 + t) * p.mask_words;
    int n = 0;
    for (int w = 0; w < p.mask_words && 32 * w < g.sq; ++w) n += __popc(m[w] & bits_below(g.sq - 32 * w));
    depth[g.q0 + t] = n - 1;
  }
}

// ---------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------
int cu_count() {
  static std::atomic<int> cached[64];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
  int n = cached[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess ||
        n <= 0)
      n = 256;
    cached[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

constexpr int kFormColumns[] = {16, 32, 64, 128, 256};
constexpr int kForms = 5;

struct Plan {
  int form;  // index of the column count
  int columns, heads_per_wg, head_groups, tokens_per_block;
  int grid;
  bool whole;
  int64_t max_items;
  size_t rec_bytes, ml_bytes, o_bytes;
  size_t bytes() const { return rec_bytes + ml_bytes + o_bytes; }
};

size_t up256(size_t n) { return (n + 255) & ~size_t(255); }

Plan lay_out(int form, bool whole, int64_t tokens, int64_t group, int64_t kv_heads,
             int64_t batch) {
  Plan pl{};
  pl.form = form;
  pl.whole = whole;
  pl.columns = kFormColumns[form];
  // kv heads a private workgroup takes together (neighbours in a token's row,
  // read together): that suits HBM when the items fill the card, more and
  // smaller pieces when they do not.  Measured with 1 / 2 / 4: 16 decode rows of
  // 4 kv heads over 2048 keys 19.8 / 20.7 / 23.8 us, 16 of 8 heads 30.3 / 28.0 /
  // 29.7, 48 ragged rows of 4 heads 80.2 / 78.4 / 77.3.
  const int64_t items = batch * kv_heads;
  int most = form > 1 || whole || items <= cu_count() / 4 ? 1 : items <= cu_count() / 2 ? 2 : 4;
  while (most > 1 && kv_heads % most != 0) most >>= 1;
  pl.heads_per_wg = most;
  pl.head_groups = int(kv_heads / most);
  pl.tokens_per_block = int(pl.columns / group);
  pl.grid = cu_count();
  pl.max_items = (tokens / pl.tokens_per_block + batch) * pl.head_groups;
  const size_t cols = size_t(2) * pl.grid * pl.heads_per_wg * pl.columns;
  pl.rec_bytes = up256(size_t(pl.grid) * sizeof(int4));
  pl.ml_bytes = up256(cols * sizeof(float2));
  pl.o_bytes = up256(cols * kD * sizeof(float));
  return pl;
}

// The narrowest form that holds the longest row, or the last.
int holding_form(int64_t longest, int64_t group) {
  int f = 0;
  while (f + 1 < kForms && kFormColumns[f] < longest * group) ++f;
  return f;
}

// The form and whether items are cut.
//
// Up to 32 columns (the longest row's tokens x query heads per kv head) the
// private forms serve, the narrowest that holds them.  Over at most kWholeKeys
// keys, and with a workgroup for each, their items stay whole: nothing is cut
// and the merge is not launched.  One decode row of 8 kv heads, whole against
// cut: 10.3 / 13 us over 512 keys, 17.4 / 13.6 over 1024 (one CU's loads bound
// it then).
//
// Wider rows take any turns form up to the narrowest that holds them, whole or
// cut, whichever these estimates call cheapest, in tenths of a 256-column
// tile.  A narrower form makes more items of less work each: that spares a
// ragged batch empty columns and lets a short call stay whole on more CUs, but
// every tile is read more often.  Measured, the narrowest form that holds the
// longest row and is cut, against this choice: a prompt of 512 tokens (16 / 8
// heads) 30.2 / 16.6 us, four of 256 (32 / 4) 27.5 / 22.0; four windowed chunks
// 52.4 / 40.3; one tree of 31 tokens over 333 keys (32 / 4) 26.3 / 15.3; 37
// ragged trees 69 / 66.  Over 195 calls of 1 to 64 sequences the times fall by
// a fifth (geometric mean); the worst, four trees of 8 tokens over 1000 keys,
// goes from 21.2 to 23.5.
constexpr int64_t kWholeKeys = 768;
constexpr int kTileCost[] = {0, 0, 4, 6, 10};  // of a form's tile
constexpr int kPieceCost = 80;   // an item's, or a piece's, setup, pipe fill and epilogue
constexpr int kMergeCost[] = {0, 0, 140, 180, 240};  // its launch, partials both ways

// Column blocks of all sequences, of which the host knows the tokens and the
// longest: a sequence fills half of its last one.
int64_t likely_blocks(int64_t tokens, int64_t batch, int64_t longest, int64_t per_block) {
  const int64_t most = batch * ((longest + per_block - 1) / per_block);
  return batch * longest == tokens ? most : std::min(most, (tokens + batch * per_block / 2) / per_block);
}

// max_keys: keys of the longest sequence as far as the host knows; window: a
// window's keys, 0 without one (or where a two-way prefix reaches past it).
// These two decide the form and `whole` alone, never what is computed.
Plan make_plan(int64_t tokens, int64_t heads, int64_t kv_heads, int64_t batch, int64_t max_q,
               int64_t max_keys, int64_t window) {
  const int64_t group = heads / kv_heads;
  const int64_t longest = std::max<int64_t>(1, std::min(max_q, tokens));
  const int widest = holding_form(longest, group);
  if (widest <= 1) {
    const int64_t per_block = kFormColumns[widest] / group;
    const int64_t keys = window > 0 ? std::min(max_keys, window + per_block) : max_keys;
    const bool whole = keys <= kWholeKeys &&
                       likely_blocks(tokens, batch, longest, per_block) * kv_heads <= cu_count();
    return lay_out(widest, whole, tokens, group, kv_heads, batch);
  }
  const int64_t grid = cu_count();
  int form = widest;
  bool uncut = false;
  int64_t least = INT64_MAX;
  for (int f = widest; f >= 2 && kFormColumns[f] >= group; --f) {
    const int64_t per_block = kFormColumns[f] / group;
    const int64_t items = likely_blocks(tokens, batch, longest, per_block) * kv_heads;
    const bool windowed = window > 0 && window + per_block < max_keys;
    const int64_t tiles = (windowed ? window + per_block : max_keys) / kTile + 1;
    // (a prompt's rows see from few keys to all, and lengths differ, if less
    // where a window bounds them: cut, the mean counts, not the longest)
    const int64_t mean = (tiles * (windowed ? 75 : 60) + 99) / 100;
    const int64_t rounds = (items + grid - 1) / grid;
    const int64_t whole = rounds > 1 && !windowed
                              ? INT64_MAX
                              : rounds * (tiles * kTileCost[f] + kPieceCost);
    const int64_t cut = items * (mean * kTileCost[f] + kPieceCost) / grid + kPieceCost +
                        kMergeCost[f];
    if (std::min(whole, cut) < least) {
      least = std::min(whole, cut);
      form = f;
      uncut = whole <= cut;
    }
  }
  return lay_out(form, uncut, tokens, group, kv_heads, batch);
}

// Workspace that holds for whatever make_plan chooses once it knows the keys.
size_t plan_bytes(int64_t tokens, int64_t heads, int64_t kv_heads, int64_t batch, int64_t max_q) {
  const int64_t group = heads / kv_heads;
  const int form = holding_form(std::max<int64_t>(1, std::min(max_q, tokens)), group);
  return lay_out(form, false, tokens, group, kv_heads, batch).bytes();
}

template <int NW, int NCB, int KW, int MODE>
int launch_one(const ScoredParams& p, int grid, hipStream_t st) {
  using F = Form<NW, NCB, KW>;
  static std::atomic<uint64_t> ready{0};  // devices whose LDS limit is set
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  const uint64_t bit = uint64_t(1) << (dev & 63);
  if (e == hipSuccess && !(ready.load(std::memory_order_relaxed) & bit)) {
    e = hipFuncSetAttribute(reinterpret_cast<const void*>(&scored_kernel<NW, NCB, KW, MODE>),
                            hipFuncAttributeMaxDynamicSharedMemorySize, F::kLds);
    if (e == hipSuccess) ready.fetch_or(bit, std::memory_order_relaxed);
  }
  KVC_REQUIRE(e == hipSuccess, KVC_ERR_RUNTIME, "scored attention: LDS limit: %s",
              hipGetErrorString(e));
  scored_kernel<NW, NCB, KW, MODE><<<grid, 64 * NW, F::kLds, st>>>(p);
  return check_launch("scored attention");
}

template <int MODE>
int launch_form(const ScoredParams& p, const Plan& pl, hipStream_t st) {
  switch (pl.form) {
    case 0: return launch_one<8, 1, 8, MODE>(p, pl.grid, st);
    case 1: return launch_one<8, 2, 8, MODE>(p, pl.grid, st);
    case 2: return launch_one<8, 1, 2, MODE>(p, pl.grid, st);
    case 3: return launch_one<8, 2, 2, MODE>(p, pl.grid, st);
    default: return launch_one<8, 2, 1, MODE>(p, pl.grid, st);
  }
}

// One launch over `p`'s sequences and its merge.  what: the entry's name.
int run_rows(ScoredParams p, int64_t max_q, int64_t max_keys, void* ws, hipStream_t st,
             const char* what) {
  // Keys that one sequence's tokens see, as far as the host knows (this only
  // steers the plan): fresh rows hold every sequence's, each as many keys as
  // queries or more.
  int64_t seen = max_keys;
  if (p.tables == nullptr)
    seen = std::min(seen, std::max<int64_t>(0, max_keys - p.num_tokens) + max_q);
  const Plan pl = make_plan(p.num_tokens, p.heads, p.kv_heads, p.batch, max_q, seen,
                            p.prefix == nullptr ? p.window : 0);
  KVC_REQUIRE(pl.max_items * ((max_keys + kTile - 1) / kTile + kItemCost) < (int64_t(1) << 30),
              KVC_ERR_VALUE, "%s: too many query blocks x keys for one call", what);
  p.heads_per_wg = pl.heads_per_wg;
  p.head_groups = pl.head_groups;
  p.tokens_per_block = pl.tokens_per_block;
  const int64_t nb = (std::min<int64_t>(max_q, p.num_tokens) + pl.tokens_per_block - 1) /
                     pl.tokens_per_block;
  p.lane_plan = (p.batch + 63) / 64 * nb <= p.batch + p.num_tokens / pl.tokens_per_block / 64;
  // A share has four tiles at least: with 2 / 4 / 8, one decode row over 2048
  // keys took 20.2 / 17.9 / 20.4 us (8 kv heads, 4 a workgroup), 16.0 / 14.5 /
  // 15.2 (2 kv heads, both in one).
  p.min_share = 4;
  p.whole = pl.whole;
  char* w = static_cast<char*>(ws);
  p.rec = reinterpret_cast<int4*>(w);
  p.part_ml = reinterpret_cast<float2*>(w + pl.rec_bytes);
  p.part_o = reinterpret_cast<float*>(w + pl.rec_bytes + pl.ml_bytes);
  int rc;
  const bool bias = p.slopes != nullptr;
  if (p.cap > 0.f) {
    if (bias) {
      rc = launch_form<kCapDistance>(p, pl, st);
    } else if (p.cap * kLog2e <= kCapNearMax) {
      rc = launch_form<kCapNear>(p, pl, st);
    } else {
      rc = launch_form<kCapFar>(p, pl, st);
    }
  } else {
    rc = bias ? launch_form<kDistance>(p, pl, st) : launch_form<kPlain>(p, pl, st);
  }
  if (rc != KVC_OK || pl.whole) return rc;
  const dim3 mg{unsigned(pl.grid), unsigned(pl.heads_per_wg * pl.columns / kMergeColumns)};
  scored_merge_kernel<<<mg, 32 * kMergeColumns, 0, st>>>(p, pl.columns);
  return check_launch(what);
}

bool rows16(const void* p, int64_t st, int64_t sh) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && st % 8 == 0 && sh % 8 == 0;
}

int check_common(const char* what, const void* q, int64_t q_st, int64_t q_sh, int64_t tokens,
                 int64_t heads, int64_t kv_heads, int64_t head_dim, float scale, float softcap,
                 int64_t window,
                 const void* out, int64_t o_st, int64_t o_sh) {
  KVC_REQUIRE(head_dim == kD, KVC_ERR_VALUE, "%s: head_dim must be 128 (got %lld)", what,
              (long long)head_dim);
  KVC_REQUIRE(heads > 0 && kv_heads > 0 && heads % kv_heads == 0, KVC_ERR_VALUE,
              "%s: num_heads must be a multiple of num_kv_heads", what);
  KVC_REQUIRE(heads / kv_heads <= kFormColumns[kForms - 1], KVC_ERR_VALUE,
              "%s: at most %d query heads per kv head", what, kFormColumns[kForms - 1]);
  KVC_REQUIRE(tokens >= 0 && tokens < (int64_t(1) << 30), KVC_ERR_VALUE, "%s: bad token count",
              what);
  KVC_REQUIRE(scale > 0.f && std::isfinite(4.f * scale), KVC_ERR_VALUE,
              "%s: scale must be finite and > 0", what);
  KVC_REQUIRE(softcap >= 0.f && std::isfinite(softcap), KVC_ERR_VALUE,
              "%s: softcap must be finite and >= 0", what);
  KVC_REQUIRE(softcap == 0.f || std::isfinite(4.f * scale / softcap), KVC_ERR_VALUE,
              "%s: scale / softcap is too large", what);
  KVC_REQUIRE(window >= 0 && window < (int64_t(1) << 30), KVC_ERR_VALUE,
              "%s: window must be >= 0", what);
  KVC_REQUIRE(tokens == 0 || (q != nullptr && out != nullptr), KVC_ERR_VALUE,
              "%s: missing q or out", what);
  KVC_REQUIRE(tokens == 0 || (rows16(q, q_st, q_sh) && rows16(out, o_st, o_sh)), KVC_ERR_ASSERT,
              "%s: q and out rows must be 16-byte aligned", what);
  return KVC_OK;
}

int check_pool(const char* what, const void* k, const void* v, int64_t blocks, int64_t page,
               int64_t kv_heads, const void* tables, int64_t max_blocks) {
  KVC_REQUIRE(k != nullptr && v != nullptr && tables != nullptr, KVC_ERR_VALUE,
              "%s: missing pool or block tables", what);
  KVC_REQUIRE(page > 0 && page % kTile == 0, KVC_ERR_VALUE,
              "%s: page_size must be a multiple of 32", what);
  KVC_REQUIRE(blocks > 0 && blocks < (int64_t(1) << 31) && max_blocks >= 0 &&
                  max_blocks * page < (int64_t(1) << 29),
              KVC_ERR_VALUE, "%s: bad pool or table size", what);
  KVC_REQUIRE(rows16(k, 0, 0) && rows16(v, 0, 0) && kv_heads * kD < (1 << 24), KVC_ERR_ASSERT,
              "%s: pools must be 16-byte aligned", what);
  return KVC_OK;
}

}  // namespace
}  // namespace kvc

using namespace kvc;

extern "C" size_t kvc_scored_workspace_bytes(int64_t num_q_tokens, int64_t num_heads,
                                             int64_t num_kv_heads, int64_t num_decode_rows,
                                             int64_t num_prefill, int64_t max_seqlen_q) {
  if (num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0 || num_q_tokens <= 0 ||
      num_heads / num_kv_heads > kFormColumns[kForms - 1])
    return 0;
  size_t n = 0;
  if (num_decode_rows > 0)
    n = plan_bytes(num_decode_rows, num_heads, num_kv_heads, num_decode_rows, 1);
  if (num_prefill > 0 && num_q_tokens > num_decode_rows)
    n = std::max(n, plan_bytes(num_q_tokens - num_decode_rows, num_heads, num_kv_heads,
                               num_prefill, max_seqlen_q));
  return n;
}

extern "C" int kvc_scored_attention(
    const void* q, int64_t q_stride_t, int64_t q_stride_h, int64_t num_q_tokens, int64_t num_heads,
    const void* k_cache, const void* v_cache, int64_t num_cache_blocks, int64_t page_size,
    int64_t num_kv_heads, int64_t head_dim, const void* k_fresh, int64_t kf_stride_t,
    int64_t kf_stride_h, const void* v_fresh, int64_t vf_stride_t, int64_t vf_stride_h,
    int64_t num_fresh_rows, const int32_t* block_tables, int64_t bt_stride,
    int64_t max_blocks_per_seq, int64_t num_decode_rows, const int32_t* decode_context_lens,
    int64_t num_prefill, const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k,
    int64_t max_seqlen_q, const int32_t* prefix_lens, const float* alibi_slopes, float softcap,
    int64_t window, float scale, void* out, int64_t out_stride_t, int64_t out_stride_h,
    void* workspace, size_t workspace_bytes, kvc_stream_t stream) {
  clear_error();
  const char* what = "scored_attention";
  int rc = check_common(what, q, q_stride_t, q_stride_h, num_q_tokens, num_heads, num_kv_heads,
                        head_dim, scale, softcap, window, out, out_stride_t, out_stride_h);
  if (rc != KVC_OK) return rc;
  KVC_REQUIRE(num_decode_rows >= 0 && num_decode_rows <= num_q_tokens && num_prefill >= 0 &&
                  num_prefill < (int64_t(1) << 30) && max_seqlen_q >= 0,
              KVC_ERR_VALUE, "%s: bad row counts", what);
  if (num_q_tokens == 0) return KVC_OK;
  const bool fresh = block_tables == nullptr;
  if (fresh) {
    KVC_REQUIRE(num_decode_rows == 0, KVC_ERR_VALUE, "%s: decode rows need block tables", what);
    KVC_REQUIRE(num_fresh_rows >= 0 && num_fresh_rows < (int64_t(1) << 29) &&
                    (num_fresh_rows == 0 || (k_fresh != nullptr && v_fresh != nullptr)),
                KVC_ERR_VALUE, "%s: without block tables the keys come from k/v", what);
    KVC_REQUIRE(rows16(k_fresh, kf_stride_t, kf_stride_h) &&
                    rows16(v_fresh, vf_stride_t, vf_stride_h),
                KVC_ERR_ASSERT, "%s: k/v rows must be 16-byte aligned", what);
    KVC_REQUIRE(kf_stride_t >= 0 && vf_stride_t >= 0 && kf_stride_t < (1 << 24) &&
                    vf_stride_t < (1 << 24),
                KVC_ERR_VALUE, "%s: k/v row strides must be below 2^24 elements", what);
  } else {
    rc = check_pool(what, k_cache, v_cache, num_cache_blocks, page_size, num_kv_heads, block_tables,
                    max_blocks_per_seq);
    if (rc != KVC_OK) return rc;
  }
  KVC_REQUIRE(num_decode_rows == 0 || decode_context_lens != nullptr, KVC_ERR_VALUE,
              "%s: missing decode_context_lens", what);
  KVC_REQUIRE(num_prefill == 0 || (cu_seqlens_q != nullptr && cu_seqlens_k != nullptr),
              KVC_ERR_VALUE, "%s: missing cu_seqlens", what);
  const size_t need = kvc_scored_workspace_bytes(num_q_tokens, num_heads, num_kv_heads,
                                                 num_decode_rows, num_prefill, max_seqlen_q);
  KVC_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need), KVC_ERR_WORKSPACE,
              "%s: workspace of %zu bytes needed", what, need);
  ScoredParams p{};
  p.q = static_cast<const uint16_t*>(q);
  p.q_st = q_stride_t;
  p.q_sh = q_stride_h;
  p.out = static_cast<uint16_t*>(out);
  p.o_st = out_stride_t;
  p.o_sh = out_stride_h;
  p.k = static_cast<const uint16_t*>(fresh ? k_fresh : k_cache);
  p.v = static_cast<const uint16_t*>(fresh ? v_fresh : v_cache);
  p.k_row = fresh ? kf_stride_t : num_kv_heads * kD;
  p.k_head = fresh ? kf_stride_h : kD;
  p.v_row = fresh ? vf_stride_t : num_kv_heads * kD;
  p.v_head = fresh ? vf_stride_h : kD;
  p.tables = block_tables;
  p.bt_stride = bt_stride;
  p.max_blocks = int(max_blocks_per_seq);
  p.num_blocks = int(num_cache_blocks);
  p.page = int(page_size);
  p.page_tiles = int(page_size / kTile);
  p.page_rcp = page_size > 0 ? 1.f / float(page_size / kTile) : 0.f;
  p.fresh_rows = num_fresh_rows;
  p.slopes = alibi_slopes;
  p.scale = scale;
  p.cap = softcap;
  p.window = int(window);
  p.heads = int(num_heads);
  p.kv_heads = int(num_kv_heads);
  p.group = int(num_heads / num_kv_heads);
  p.group_rcp = 1.f / float(p.group);
  const int64_t max_keys = fresh ? num_fresh_rows : max_blocks_per_seq * page_size;
  hipStream_t st = as_stream(stream);
  if (num_decode_rows > 0) {
    ScoredParams d = p;
    d.batch = d.num_tokens = int(num_decode_rows);
    d.q_per_seq = 1;
    d.lens = decode_context_lens;
    rc = run_rows(d, 1, max_keys, workspace, st, what);
    if (rc != KVC_OK) return rc;
  }
  if (num_prefill > 0 && num_q_tokens > num_decode_rows) {
    p.q += num_decode_rows * q_stride_t;
    p.out += num_decode_rows * out_stride_t;
    if (!fresh) p.tables += num_decode_rows * bt_stride;
    p.batch = int(num_prefill);
    p.num_tokens = int(num_q_tokens - num_decode_rows);
    p.cu_q = cu_seqlens_q;
    p.cu_k = cu_seqlens_k;
    p.prefix = prefix_lens;
    rc = run_rows(p, max_seqlen_q, max_keys, workspace, st, what);
  }
  return rc;
}

extern "C" size_t kvc_tree_workspace_bytes(int64_t num_q_tokens, int64_t num_heads,
                                           int64_t num_kv_heads, int64_t batch,
                                           int64_t max_seqlen_q) {
  if (num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0 || num_q_tokens <= 0 ||
      num_heads / num_kv_heads > kFormColumns[kForms - 1])
    return 0;
  return plan_bytes(num_q_tokens, num_heads, num_kv_heads, batch, max_seqlen_q) +
         up256(size_t(num_q_tokens) * sizeof(int32_t));
}

extern "C" int kvc_tree_attention(
    const void* q, int64_t q_stride_t, int64_t q_stride_h, int64_t num_q_tokens, int64_t num_heads,
    const void* k_cache, const void* v_cache, int64_t num_cache_blocks, int64_t page_size,
    int64_t num_kv_heads, int64_t head_dim, const int32_t* block_tables, int64_t bt_stride,
    int64_t max_blocks_per_seq, int64_t batch, const int32_t* context_lens,
    const int32_t* cu_seqlens_q, int64_t max_seqlen_q, const int64_t* tree_mask,
    int64_t mask_words, const float* alibi_slopes, float softcap, int64_t window, float scale,
    void* out, int64_t out_stride_t, int64_t out_stride_h, void* workspace,
    size_t workspace_bytes, kvc_stream_t stream) {
  clear_error();
  const char* what = "tree_attention";
  int rc = check_common(what, q, q_stride_t, q_stride_h, num_q_tokens, num_heads, num_kv_heads,
                        head_dim, scale, softcap, window, out, out_stride_t, out_stride_h);
  if (rc != KVC_OK) return rc;
  KVC_REQUIRE(batch >= 0 && batch < (int64_t(1) << 30) && max_seqlen_q >= 0, KVC_ERR_VALUE,
              "%s: bad row counts", what);
  if (num_q_tokens == 0 || batch == 0) return KVC_OK;
  rc = check_pool(what, k_cache, v_cache, num_cache_blocks, page_size, num_kv_heads, block_tables,
                  max_blocks_per_seq);
  if (rc != KVC_OK) return rc;
  KVC_REQUIRE(context_lens != nullptr && tree_mask != nullptr, KVC_ERR_VALUE,
              "%s: missing context_lens or tree_mask", what);
  KVC_REQUIRE(mask_words > 0 && mask_words < (1 << 20) && mask_words * 64 >= max_seqlen_q,
              KVC_ERR_VALUE, "%s: tree_mask has too few words for max_seqlen_q", what);
  KVC_REQUIRE(cu_seqlens_q != nullptr || max_seqlen_q * batch == num_q_tokens, KVC_ERR_VALUE,
              "%s: without cu_seqlens_q every tree has max_seqlen_q tokens", what);
  const size_t need =
      kvc_tree_workspace_bytes(num_q_tokens, num_heads, num_kv_heads, batch, max_seqlen_q);
  KVC_REQUIRE(workspace != nullptr && workspace_bytes >= need, KVC_ERR_WORKSPACE,
              "%s: workspace of %zu bytes needed", what, need);
  ScoredParams p{};
  p.q = static_cast<const uint16_t*>(q);
  p.q_st = q_stride_t;
  p.q_sh = q_stride_h;
  p.out = static_cast<uint16_t*>(out);
  p.o_st = out_stride_t;
  p.o_sh = out_stride_h;
  p.k = static_cast<const uint16_t*>(k_cache);
  p.v = static_cast<const uint16_t*>(v_cache);
  p.k_row = p.v_row = num_kv_heads * kD;
  p.k_head = p.v_head = kD;
  p.tables = block_tables;
  p.bt_stride = bt_stride;
  p.max_blocks = int(max_blocks_per_seq);
  p.num_blocks = int(num_cache_blocks);
  p.page = int(page_size);
  p.page_tiles = int(page_size / kTile);
  p.page_rcp = page_size > 0 ? 1.f / float(page_size / kTile) : 0.f;
  p.cu_q = cu_seqlens_q;
  p.q_per_seq = int(max_seqlen_q);
  p.lens = context_lens;
  p.lens_exclude_q = 1;
  p.mask = reinterpret_cast<const uint32_t*>(tree_mask);
  p.mask_words = int(2 * mask_words);
  p.slopes = alibi_slopes;
  p.scale = scale;
  p.cap = softcap;
  p.window = int(window);
  p.batch = int(batch);
  p.num_tokens = int(num_q_tokens);
  p.heads = int(num_heads);
  p.kv_heads = int(num_kv_heads);
  p.group = int(num_heads / num_kv_heads);
  p.group_rcp = 1.f / float(p.group);
  hipStream_t st = as_stream(stream);
  if (alibi_slopes != nullptr || window > 0) {
    int32_t* depth = reinterpret_cast<int32_t*>(
        static_cast<char*>(workspace) + need - up256(size_t(num_q_tokens) * sizeof(int32_t)));
    tree_depth_kernel<<<unsigned(batch), 64, 0, st>>>(p, depth);
    rc = check_launch(what);
    if (rc != KVC_OK) return rc;
    p.places = depth;
  }
  return run_rows(p, max_seqlen_q, max_blocks_per_seq * page_size, workspace, st, what);
}
