// The 4-bit KV cache: quantise on append, dequantising reads, paged decode
// attention (gfx950; the encoding is in kvc_fp4.h).
//
// Decode: out[b, h] = sum_j softmax_j(scale q[b, h].k_j) v_j over the row's first
// context_lens[b] keys, 0 for a row without keys.
//
// K's codes are the scaled MFMA's operand as they lie in the pool: S^T = K Q^T with a
// kv head's G query heads as columns, a run of 32 dims and its power a lane.  Q comes
// as a sum of two 8-bit operands, exact to 2^-21 of its row.  S^T leaves a lane keys
// of its own column that P's operand of O^T = V^T P^T takes, so weights never move
// between lanes.  V is transposed by LDS reads of 4-bit elements and converted with
// power 1: its powers differ by key, the summed index, so they multiply the weights
// instead, in the exponent fields, once for each run of 32 channels (a power of two
// times a bf16 weight is exact).  Sums are formed of the rounded weights, so the
// weights add up to the sum that divides them; logits, sums and O are fp32.
//
// A wave's tile is 64 rows of codes: 64 keys of one kv head, or 32 keys of two, whose
// rows make whole 128-byte lines (loads alone 5.1 against 6.1 TB/s).  Every wave
// streams its own tiles through its own two LDS slots of 8.5 KiB (direct-to-LDS loads
// two tiles ahead, no workgroup barrier); eight waves a workgroup, one workgroup a CU,
// waves differ in kv head and in tile phase and join once an item.  Bound by HBM reads
// for batches: 64 rows of 4096 keys (4 kv heads, 143 MB) 33 us, of 8192 50 + 5 to join
// (47 with the loads alone), 128 of 4096 51: 7 TB/s for every further byte, and 12 to 16
// us of launch, lengths, table, first tiles and last results.  Single rows are bound by
// that chain: 333 keys 7.3 us.
#include <algorithm>
#include <atomic>
#include <cmath>

#include "kvc_fp4.h"
#include "kvc_lds.h"

namespace kvc {
namespace {

constexpr int kThreads = 256;
constexpr int kD = 128;
constexpr int kLanesPerRow = 16;  // of the append and the dequantising reads
constexpr int kRowsPerBlock = kThreads / kLanesPerRow;

// ---------------------------------------------------------------------------
// Append.  A 16-lane group owns one (token, head) row of K and of V, eight dims
// (16 bytes) a lane; four lanes share a run.  Bound by HBM for prompts (16384 tokens
// of 4 heads, 42 MB, 9.6 us: 4.4 TB/s with the launch in it; two or four rows a group
// take 10.2 and 11.4), by the launch and two dependent reads (slot, row) for a decode
// step (3 us).
// ---------------------------------------------------------------------------
__device__ __forceinline__ uint32_t run_max(uint32_t x) {  // over four lanes
  x = max(x, uint32_t(__shfl_xor(int(x), 1, 64)));
  return max(x, uint32_t(__shfl_xor(int(x), 2, 64)));
}

__device__ __forceinline__ void store_row(const u32x4_t& x, uint8_t* codes, uint8_t* powers,
                                          int64_t row, int lane16) {
  const int power = power_of_top(run_max(top_bits(x)));
  // (a NaN run's values may not convert to anything: its codes are 0)
  const uint32_t c = power == kPowerNaN ? 0u : quant_fp4x8(x, power_f32(power));
  *reinterpret_cast<uint32_t*>(codes + row * kFp4RowBytes + lane16 * 4) = c;
  if ((lane16 & 3) == 0) powers[row * kFp4Powers + (lane16 >> 2)] = uint8_t(power);
}

template <int kIdxBytes>
__global__ void __launch_bounds__(kThreads)
store_fp4_kernel(const uint16_t* __restrict__ key, int64_t k_sn, int64_t k_sh,
                 const uint16_t* __restrict__ value, int64_t v_sn, int64_t v_sh,
                 uint8_t* __restrict__ k_cache, uint8_t* __restrict__ v_cache,
                 uint8_t* __restrict__ k_scale, uint8_t* __restrict__ v_scale, int64_t num_slots,
                 const void* __restrict__ slots, int64_t num_tokens, int kvh) {
  const int lane16 = threadIdx.x & (kLanesPerRow - 1);
  const int64_t row = int64_t(blockIdx.x) * kRowsPerBlock + (threadIdx.x / kLanesPerRow);
  const int64_t n = row / kvh;
  const int h = int(row - n * kvh);
  // Whole 16-lane groups share n, so the early exits keep groups intact.
  if (n >= num_tokens) return;
  const int64_t raw = load_index<kIdxBytes>(slots, n);
  const u32x4_t kw = *reinterpret_cast<const u32x4_t*>(key + n * k_sn + h * k_sh + lane16 * 8);
  const u32x4_t vw = *reinterpret_cast<const u32x4_t*>(value + n * v_sn + h * v_sh + lane16 * 8);
  const int64_t slot = wrap_slot(raw, num_slots);
  if (slot < 0 || slot >= num_slots) return;
  store_row(kw, k_cache, k_scale, slot * kvh + h, lane16);
  store_row(vw, v_cache, v_scale, slot * kvh + h, lane16);
}

// ---------------------------------------------------------------------------
// Dequantising reads: 16 lanes a row, four bytes of codes in, 16 bytes out.  Bound
// like the append (16384 tokens of 4 heads 9.0 us; two or four rows a group were 3 and
// 14 % slower).
// ---------------------------------------------------------------------------
__device__ __forceinline__ u32x4_t read_row(const uint8_t* codes, const uint8_t* powers,
                                            int64_t row, int lane16) {
  const uint32_t c = *reinterpret_cast<const uint32_t*>(codes + row * kFp4RowBytes + lane16 * 4);
  return dequant_fp4x8(c, power_f32(powers[row * kFp4Powers + (lane16 >> 2)]));
}

__global__ void __launch_bounds__(kThreads)
dequant_fp4_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ powers,
                   int64_t rows, uint16_t* __restrict__ out) {
  const int lane16 = threadIdx.x & (kLanesPerRow - 1);
  const int64_t row = int64_t(blockIdx.x) * kRowsPerBlock + (threadIdx.x / kLanesPerRow);
  if (row >= rows) return;
  *reinterpret_cast<u32x4_t*>(out + row * kD + lane16 * 8) =
      read_row(codes, powers, row, lane16);
}

__global__ void __launch_bounds__(kThreads)
gather_fp4_kernel(const uint8_t* __restrict__ k_cache, const uint8_t* __restrict__ v_cache,
                  const uint8_t* __restrict__ k_scale, const uint8_t* __restrict__ v_scale,
                  int64_t num_slots, int page, int kvh, const int32_t* __restrict__ block_tables,
                  int64_t bt_stride, int max_blocks, int64_t bt_row0, int num_prefill,
                  const int32_t* __restrict__ cu_k, int64_t tokens, uint16_t* __restrict__ out_k,
                  uint16_t* __restrict__ out_v) {
  const int lane16 = threadIdx.x & (kLanesPerRow - 1);
  const int64_t row = int64_t(blockIdx.x) * kRowsPerBlock + (threadIdx.x / kLanesPerRow);
  const int64_t t = row / kvh;
  const int h = int(row - t * kvh);
  if (t >= tokens) return;
  // chunk i: the last with cu_k[i] <= t
  int lo = 0, hi = num_prefill - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (cu_k[mid] <= t) lo = mid; else hi = mid - 1;
  }
  const int64_t at = t - cu_k[lo];
  const int64_t bi = at >= 0 ? at / page : max_blocks;
  const int64_t blk = bi < max_blocks ? block_tables[(bt_row0 + lo) * bt_stride + bi] : -1;
  const int64_t slot = blk * page + (at - bi * page);
  u32x4_t k = {0u, 0u, 0u, 0u}, v = {0u, 0u, 0u, 0u};
  if (blk >= 0 && slot < num_slots) {  // a bad table entry reads nothing
    k = read_row(k_cache, k_scale, slot * kvh + h, lane16);
    v = read_row(v_cache, v_scale, slot * kvh + h, lane16);
  }
  // (past the caches: 40 MB of them 10.9 -> 8.6 us)
  __builtin_nontemporal_store(k, reinterpret_cast<u32x4_t*>(out_k + row * kD + lane16 * 8));
  __builtin_nontemporal_store(v, reinterpret_cast<u32x4_t*>(out_v + row * kD + lane16 * 8));
}

// ---------------------------------------------------------------------------
// Paged decode.
// ---------------------------------------------------------------------------
constexpr int kWaves = 8;
constexpr int kTileRows = 64;                         // (key, head) rows of a wave's tile
constexpr int kCodeBytes = kTileRows * kFp4RowBytes;  // of K or V, 4 KiB
constexpr int kPowerBytes = kTileRows * kFp4Powers;   // 256
constexpr int kVAt = kCodeBytes, kKpAt = 2 * kCodeBytes, kVpAt = kKpAt + kPowerBytes;
constexpr int kSlotBytes = kVpAt + kPowerBytes;  // 8.5 KiB
constexpr int kSlots = 2;
constexpr float kLowest = -3.402823466e38f;
// Binades that a score may pass the running reference by: a weight of up to 4
// times the largest power, 2^125, is still finite.
constexpr float kSlack = 2.f;
constexpr int kStateBytes = 8 * 64 * 16 + 64 * 8;  // a wave's O and (reference, sum)
static_assert(kStateBytes <= kSlotBytes);  // (one a head, a slot each)

// An item: a block of up to 16 columns (query token x head) of one kv head group
// and sequence.  What the merge needs of it.
struct ItemRec {
  int first, last;  // shares
  int q0, sq;       // the sequence's query rows
  int group, block;
  int unused[2];
};

struct Fp4Params {
  const uint16_t* q;
  int64_t q_st, q_sh;
  uint16_t* out;
  int64_t o_st, o_sh;
  const uint8_t* k;
  const uint8_t* v;
  const uint8_t* ks;
  const uint8_t* vs;
  const int32_t* tables;
  int64_t bt_stride;
  const int32_t* lens;     // of the decode rows
  const int32_t* cu_q;     // of the chunks
  const int32_t* cu_k;
  int decode_rows, chunks, chunk_tokens;
  int max_blocks, num_blocks, page;
  int page_halves;         // page / 32
  float page_halves_rcp;
  int kv_heads, group;
  float group_rcp;
  int heads_per_wg;        // kv heads of a workgroup
  int head_groups;         // kv_heads / heads_per_wg
  int tile_shift;          // log2 of the keys of a wave's tile
  int cols;                // columns kept of a partial: min(16, columns there can be)
  int min_share;
  int item_cost;           // of an item's setup, in tiles
  float grid_rcp;
  int whole;               // one workgroup an item, no partials
  int row_blocks;          // blocks of a decode row
  int items;               // that there is room for
  float c2;                // |scale| log2(e)
  uint32_t flip;           // sign bits of a bf16 pair where scale is negative
  int* count;              // items
  ItemRec* rec;            // of each item
  float* part_o;
  float2* part_ml;
};

// A sequence: a decode row or a chunk.  Query t sees the keys j < given - sq + t + 1;
// keys counts those that its table can hold.
struct SeqGeo {
  int q0, sq, given, keys;
};
constexpr int kLongest = 1 << 29;  // of a length (tables hold fewer keys)
__device__ __forceinline__ SeqGeo seq_geo(const Fp4Params& p, int q0, int q1, int64_t len) {
  SeqGeo g;
  g.q0 = q0;
  g.sq = max(0, q1 - q0);
  g.given = int(max(int64_t(0), min(len, int64_t(kLongest))));
  g.keys = min(g.given, p.max_blocks * p.page);
  return g;
}
__device__ __forceinline__ SeqGeo load_row(const Fp4Params& p, int i) {  // a decode row
  return i < p.decode_rows ? seq_geo(p, i, i + 1, p.lens[i]) : SeqGeo{0, 0, 0, 0};
}
template <bool kUniform>
__device__ __forceinline__ SeqGeo load_seq(const Fp4Params& p, int i) {
  auto at = [&](const int32_t* t, int64_t idx) {
    if constexpr (kUniform) return table_entry(t, idx);
    return t[idx];
  };
  if (i < p.decode_rows) return seq_geo(p, i, i + 1, at(p.lens, i));
  const int c = i - p.decode_rows;
  const int q0 = max(0, min(at(p.cu_q, c), p.chunk_tokens));
  const int q1 = max(0, min(at(p.cu_q, c + 1), p.chunk_tokens));
  return seq_geo(p, p.decode_rows + q0, p.decode_rows + q1,
                 int64_t(at(p.cu_k, c + 1)) - at(p.cu_k, c));
}
// Its blocks, and the tiles of each: 1 at least, which writes the zeros of rows
// without keys.
__device__ __forceinline__ int blocks_of(const Fp4Params& p, const SeqGeo& g) {
  return int((int64_t(g.sq) * p.group + 15) >> 4);
}
__device__ __forceinline__ int tiles_of(const Fp4Params& p, const SeqGeo& g) {
  return p.whole ? 1 : max(1, (g.keys + (1 << p.tile_shift) - 1) >> p.tile_shift);
}

// floor(x / d) for 0 <= x < 2^31 and quotients below 2^20, given rcp, 1 / d to
// within a few ulp.
__device__ __forceinline__ int div_steps(int x, int d, float rcp) {
  int q = int(float(x) * rcp);
  q -= int64_t(q) * d > x ? 1 : 0;
  q += x - q * d >= d ? 1 : 0;
  return uniform(q);
}

template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

typedef int v2i_t __attribute__((ext_vector_type(2)));
typedef int v8i_t __attribute__((ext_vector_type(8)));
typedef float f32x2v_t __attribute__((ext_vector_type(2)));
typedef unsigned short u16x2v_t __attribute__((ext_vector_type(2)));

// A column's query as the two 8-bit operands (e4m3) of the scaled MFMA: x = hi +
// lo, hi = x rounded to four significant bits, lo the rest, which four bits hold
// as well.  Both count in one power of two for the row, lo 16 times finer.  x is
// met to 2^-21 of the row's largest magnitude (lo's last place), exactly from
// 2^-13 of it up.
struct Query {
  v8i_t hi, lo;     // dims 16 lg .. + 15, then 64 + 16 lg .. + 15
  int hi_power, lo_power;
};
struct QueryRow {  // bf16, dims 16 lg .., 16 lg + 8 .., 64 + 16 lg .., 64 + 16 lg + 8 ..
  u32x4_t x[4];
};
__device__ __forceinline__ QueryRow load_query(const uint16_t* row, int lg) {
  QueryRow r;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    r.x[i] = *reinterpret_cast<const u32x4_t*>(row + 64 * (i >> 1) + 16 * lg + 8 * (i & 1));
  return r;
}
__device__ __forceinline__ Query split_query(const QueryRow& r, uint32_t flip) {
  const u32x4_t(&x)[4] = r.x;
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) top = max(top, top_bits(x[i]));
  top = __float_as_uint(rows4_max(__uint_as_float(top << 16))) >> 16;
  Query q;
  // (a magnitude of 2^e counts 2^7; the low end leaves room for lo's power)
  q.hi_power = max(int(top >> 7) - 7, 5);
  q.lo_power = q.hi_power - 4;
  const float hp = __uint_as_float(uint32_t(q.hi_power) << 23);
  const float lp = __uint_as_float(uint32_t(q.lo_power) << 23);
#pragma unroll
  for (int w = 0; w < 8; ++w) {  // four dims
    const uint32_t a = x[w >> 1][2 * (w & 1)] ^ flip, b = x[w >> 1][2 * (w & 1) + 1] ^ flip;
    typedef short s16x2_t __attribute__((ext_vector_type(2)));
    s16x2_t h = {0, 0}, l = {0, 0};
    h = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(h, __builtin_bit_cast(bf16x2_t, a), hp, false);
    h = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(h, __builtin_bit_cast(bf16x2_t, b), hp, true);
    const int hw = __builtin_bit_cast(int, h);
    const auto back0 = __builtin_bit_cast(
        f32x2v_t, __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(hw, hp, false));
    const auto back1 = __builtin_bit_cast(
        f32x2v_t, __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(hw, hp, true));
    l = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(l, bf16_bits_to_f32(a & 0xffffu) - back0[0],
                                                 bf16_bits_to_f32(a >> 16) - back0[1], lp, false);
    l = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(l, bf16_bits_to_f32(b & 0xffffu) - back1[0],
                                                 bf16_bits_to_f32(b >> 16) - back1[1], lp, true);
    q.hi[w] = hw;
    q.lo[w] = __builtin_bit_cast(int, l);
  }
  return q;
}

typedef const __attribute__((address_space(4))) Fp4Params KernelArgs;
__device__ __forceinline__ KernelArgs* kernel_args() {
  KernelArgs* a = (KernelArgs*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(a));
  return a;
}

struct Carry {  // a wave's running softmax and output, column lane & 15
  f32x4_t o[8];  // channels 16 cb + 4 (lane >> 4) ..
  f32x4_t l;     // the column's sum, in every element
  float m;
};

// S^T += K Q^T: 16 rows of 128 codes with their powers (run lane >> 4).
__device__ __forceinline__ f32x4_t mfma_fp4(const u32x4_t& k, const v8i_t& q, const f32x4_t& c,
                                            int k_power, int q_power) {
  const v8i_t a = {int(k[0]), int(k[1]), int(k[2]), int(k[3]), 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, q, c, 4, 0, 0, k_power, 0, q_power);
}

// A wave's tile is 64 rows of codes: 64 keys of one kv head (NH = 1) or 32 keys of
// two (NH = 2), in two halves h of 32 keys.  Two heads next to each other are a
// whole 128-byte line of the pool, and a wave that reads half lines gets 5.1 TB/s
// of HBM where whole ones give 6.1 (loads alone, 16 rows of 32768 keys, 4 heads).
//
// In LDS: NH = 1, 64-byte rows, K's in the order of the MFMA's rows (16-row part
// 2 h + t: key 8 (r >> 2) + 4 t + (r & 3) of the half), V's in key order.  NH = 2,
// 128-byte rows in key order.  A row's 16-byte parts are turned (by xor) so that
// neither kind of operand read meets a bank twice.
template <int NH>
struct TileLayout;
template <>
struct TileLayout<1> {
  static __device__ int key(int x, int lm, int lg) {  // of 16-row part x = 2 h + t
    return 1024 * x + 64 * lm + 16 * (lg ^ (lm >> 2));
  }
  static __device__ int value(int cb, int lm, int lg) {
    const int h = lm >> 3, k = 8 * lg + (lm & 7);
    return 2048 * h + 64 * k + 16 * ((cb >> 1) ^ (((k >> 2) & 1) + 2 * h)) + 8 * (cb & 1);
  }
  // Offsets of a lane's 16 bytes in the pool, of load m (of 4): K, V.
  static __device__ int load_key(int m, int lane, int row_bytes) {
    const int r = lane >> 2;
    return (8 * (r >> 2) + 4 * (m & 1) + (r & 3)) * row_bytes + 16 * ((lane & 3) ^ (r >> 2));
  }
  static __device__ int load_value(int m, int lane, int row_bytes) {
    return (16 * (m & 1) + (lane >> 2)) * row_bytes +
           16 * ((lane & 3) ^ (((lane >> 4) & 1) + 2 * (m >> 1)));
  }
};
template <>
struct TileLayout<2> {
  static __device__ int key(int x, int lm, int lg) {
    return 1024 * (lm >> 2) + 128 * (4 * (x & 1) + (lm & 3)) +
           16 * ((4 * (x >> 1) + lg) ^ (lm >> 1));
  }
  static __device__ int value(int cb, int lm, int lg) {
    return 1024 * lg + 128 * (lm & 7) + 16 * ((4 * (lm >> 3) + (cb >> 1)) ^ ((lm >> 1) & 3)) +
           8 * (cb & 1);
  }
  static __device__ int load_key(int m, int lane, int row_bytes) {
    return (8 * m + (lane >> 3)) * row_bytes + 16 * ((lane & 7) ^ (2 * m + ((lane >> 4) & 1)));
  }
  static __device__ int load_value(int m, int lane, int row_bytes) {
    return (8 * m + (lane >> 3)) * row_bytes + 16 * ((lane & 7) ^ ((lane >> 4) & 3));
  }
};

// A tile in registers.  K: four operands of 16 rows and the lane's run's power of
// each.  V: of each 16 channels, the lane's 8 keys 8 lg + j of both halves, channel
// lm, and those keys' powers; mine: the powers of key lane & 31 of half lane >> 5.
struct Tile {
  u32x4_t k[4];
  int k_power[4];
  v2i_t v[8];
  u32x4_t v_power[2][2];
  uint32_t mine;
};
template <int NH>
__device__ __forceinline__ void read_tile(Tile& t, const char* at, int lane, int lm, int lg) {
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    t.k[x] = *reinterpret_cast<const u32x4_t*>(at + TileLayout<NH>::key(x, lm, lg));
    const int key = 32 * (x >> 1) + 8 * (lm >> 2) + 4 * (x & 1) + (lm & 3);
    t.k_power[x] = *reinterpret_cast<const uint8_t*>(at + kKpAt + 4 * key + lg);
  }
#pragma unroll
  for (int cb = 0; cb < 8; ++cb)
    t.v[cb] = __builtin_amdgcn_ds_read_tr4_b64_v2i32(
        (__attribute__((address_space(3))) v2i_t*)((__attribute__((address_space(3))) char*)(
            at + kVAt + TileLayout<NH>::value(cb, lm, lg))));
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int i = 0; i < 2; ++i)
      t.v_power[h][i] =
          *reinterpret_cast<const u32x4_t*>(at + kVpAt + 4 * (32 * h + 8 * lg + 4 * i));
  t.mine = *reinterpret_cast<const uint32_t*>(at + kVpAt + 4 * lane);
}

// The keys of a tile that the lane's column, which sees `left` of them, does not:
// scores -infinity, no power (what lies behind a sequence may hold anything).
template <int NH>
__device__ __forceinline__ void mask_tile(Tile& t, f32x4_t (&s)[4], int left, int lg) {
  int first = 8 * lg;  // (opaque: nothing of this is worked out for every tile)
  asm volatile("" : "+v"(first));
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const bool seen = (NH == 1 ? 32 * h : 0) + first + j < left;
      s[2 * h + (j >> 2)][j & 3] = seen ? s[2 * h + (j >> 2)][j & 3] : -INFINITY;
      const uint32_t word = t.v_power[h][j >> 2][j & 3];
      t.v_power[h][j >> 2][j & 3] = seen ? word : 0u;
    }
}

// The weights of N scores of a column (bf16 pairs), the reference and the sum.
template <int N>
__device__ __forceinline__ void weights(const f32x4_t* s, Carry& c, float c2, u32x4_t* w) {
  float top = s[0][0];
#pragma unroll
  for (int e = 1; e < N; ++e) top = fmaxf(top, s[e >> 2][e & 3]);
  top *= c2;
  // The reference moves only when a score passes it by kSlack.
  if (__builtin_amdgcn_ballot_w64(top > c.m + kSlack) != 0) {
    const float next = fmaxf(c.m, rows4_max(top));
    const float a = __builtin_amdgcn_exp2f(c.m - next);
    c.m = next;
    c.l *= a;
#pragma unroll
    for (int cb = 0; cb < 8; ++cb) c.o[cb] *= a;
  }
  const u32x4_t ones = {0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u};
#pragma unroll
  for (int i = 0; i < N / 8; ++i) {
#pragma unroll
    for (int e = 0; e < 8; e += 2)
      w[i][e >> 1] = pack_bf16x2_fast(
          __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * i + (e >> 2)][e & 3], c2, -c.m)),
          __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * i + (e >> 2)][(e & 3) + 1], c2, -c.m)));
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      uint32_t word = w[i][e];
      asm volatile("" : "+v"(word));
      w[i][e] = word;
    }
    c.l = mfma_bf16(ones, w[i], c.l);
  }
}

// O^T += V^T P^T over the eight keys of half h.
__device__ __forceinline__ void weigh(const Tile& t, int h, const u32x4_t& w, Carry& c) {
  // A power of two times a weight adds to the weight's exponent field; a sum
  // below 0 is 0.  One multiply-add and one saturating subtraction a pair: the weights
  // as words and the factor in a register keep the compiler from taking them apart.  A
  // weight of 0 has no exponent to add to (its field would count as 2^-127): what is
  // subtracted is then 65535 instead of the bias, which leaves 0 whatever the power.
  u32x4_t pw = w;
  uint32_t field = 128u * 0x10001u;
  asm volatile("" : "+s"(field));
  u16x2v_t less[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t at = pw[i];
    const u16x2v_t none =
        __builtin_elementwise_sub_sat(u16x2v_t{1, 1}, __builtin_bit_cast(u16x2v_t, at));
    less[i] = none * u16x2v_t{65535 - (127 << 7), 65535 - (127 << 7)} +
              u16x2v_t{127 << 7, 127 << 7};
  }
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    u32x4_t pb;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t bytes = perm(t.v_power[h][i >> 1][(2 * i + 1) & 3],
                                  t.v_power[h][i >> 1][(2 * i) & 3], 0x0c040c00u + 0x00010001u * g);
      const uint32_t at = pw[i];
      const u16x2v_t x = __builtin_bit_cast(u16x2v_t, bytes) * __builtin_bit_cast(u16x2v_t, field) +
                         __builtin_bit_cast(u16x2v_t, at);
      pb[i] = __builtin_bit_cast(uint32_t, __builtin_elementwise_sub_sat(x, less[i]));
    }
#pragma unroll
    for (int x = 0; x < 2; ++x)
      c.o[2 * g + x] =
          mfma_bf16(dequant_fp4x8(uint32_t(t.v[2 * g + x][h]), 1.f), pb, c.o[2 * g + x]);
  }
}

// A run that is NaN makes its channels NaN whatever its key weighs, for the columns
// that see it.
template <int NH>
__device__ __forceinline__ void add_nan_runs(uint32_t mine, int left, Carry (&c)[NH]) {
  const uint32_t inv = ~mine;  // a byte of 0 where the power is 255
  if (__builtin_expect(
          __builtin_amdgcn_ballot_w64(((inv - 0x01010101u) & ~inv & 0x80808080u) != 0) == 0, 1))
    return;
  constexpr int kKeys = kTileRows / NH;
  const uint64_t seen = left >= kKeys ? ~uint64_t(0) >> (64 - kKeys)
                                      : (uint64_t(1) << max(left, 0)) - 1;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const uint64_t at = __builtin_amdgcn_ballot_w64(((mine >> (8 * g)) & 255u) == 255u);
#pragma unroll
    for (int i = 0; i < NH; ++i) {
      const bool nan = (at >> (NH == 1 ? 0 : 32 * i) & seen) != 0;
      const float add = nan ? __uint_as_float(0x7fc00000u) : 0.f;
#pragma unroll
      for (int x = 0; x < 2; ++x) c[i].o[2 * g + x] += add;
    }
  }
}

__device__ __forceinline__ i32x4_t scalar_rsrc(const void* base, int bytes) {
  const uint64_t a = reinterpret_cast<uint64_t>(base);
  return i32x4_t{int(uint32_t(a)), int(uint32_t(a >> 32) & 0xffffu), bytes, kBufWord3};
}
// Two loads of 1 KiB of codes; one of powers (of the active lanes).  Whole lines are
// read past the caches (`nt`); half lines are not: their other halves follow from the
// next workgroups of the XCD (64 rows of 2304 keys 22.6 us with nt, 19.6 without).
#define KVC_LOAD_CODES(HINT)                                                   \
  asm volatile(                                                                \
      "s_mov_b32 %0, m0\n\t"                                                   \
      "s_mov_b32 m0, %3\n\t"                                                   \
      "s_nop 0\n\t"                                                            \
      "buffer_load_dwordx4 %1, %4, %5 offen" HINT " lds\n\t"                   \
      "s_add_u32 m0, m0, 0x400\n\t"                                            \
      "s_nop 0\n\t"                                                            \
      "buffer_load_dwordx4 %2, %4, %6 offen" HINT " lds\n\t"                   \
      "s_mov_b32 m0, %0"                                                       \
      : "=&s"(m0)                                                              \
      : "v"(off0), "v"(off1), "s"(lds), "s"(r), "s"(base0), "s"(base1)         \
      : "memory", "scc")
template <bool kWholeLines>
__device__ __forceinline__ void load_codes(const i32x4_t& r, int off0, int off1, int base0,
                                           int base1, uint32_t lds) {
  uint32_t m0;
  if constexpr (kWholeLines) {
    KVC_LOAD_CODES(" nt");
  } else {
    KVC_LOAD_CODES("");
  }
}
#undef KVC_LOAD_CODES
__device__ __forceinline__ void load_powers(const i32x4_t& r, int off, uint32_t lds) {
  uint32_t m0;
  asm volatile(
      "s_mov_b32 %0, m0\n\t"
      "s_mov_b32 m0, %2\n\t"
      "s_nop 0\n\t"
      "buffer_load_dword %1, %3, 0 offen nt lds\n\t"
      "s_mov_b32 m0, %0"
      : "=&s"(m0)
      : "v"(off), "s"(lds), "s"(r)
      : "memory");
}

// The states of P phases, `apart` in LDS, joined: phase f makes channel blocks f, f +
// P, .. of the lane's column.
template <int P, class Put>
__device__ __forceinline__ void join(const char* at, int apart, int f, int lane, const Put& put) {
  float2 ml[P];
  float b[P];
#pragma unroll
  for (int i = 0; i < P; ++i)
    ml[i] = reinterpret_cast<const float2*>(at + i * apart + 8192)[lane];
  f32x4_t part[8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
    part[i] = *reinterpret_cast<const f32x4_t*>(at + (i % P) * apart +
                                                (f + P * (i / P)) * 1024 + lane * 16);
  float top = ml[0].x, l = 0.f;
#pragma unroll
  for (int i = 1; i < P; ++i) top = fmaxf(top, ml[i].x);
#pragma unroll
  for (int i = 0; i < P; ++i) {
    b[i] = __builtin_amdgcn_exp2f(ml[i].x - top);
    l += ml[i].y * b[i];
  }
#pragma unroll
  for (int i = 0; i < 8 / P; ++i) {
    f32x4_t o = part[P * i] * b[0];
#pragma unroll
    for (int j = 1; j < P; ++j) o += part[P * i + j] * b[j];
    put(f + P * i, o, top, l);
  }
}

template <int NH, bool kChunks>
__global__ void __launch_bounds__(64 * kWaves, 2) fp4_decode_kernel(Fp4Params p) {
  constexpr int kKeys = kTileRows / NH;  // of a tile
  extern __shared__ __align__(1024) char smem[];
  const int lane = threadIdx.x & 63, wave = uniform(int(threadIdx.x >> 6));
  const int lm = lane & 15, lg = lane >> 4;
  // Consecutive shares on one XCD (workgroup b runs on XCD b mod 8).
  const int grid = gridDim.x;
  const int share = grid % 8 == 0 ? (blockIdx.x % 8) * (grid / 8) + blockIdx.x / 8 : blockIdx.x;
  touch_kernel_args(int(sizeof(Fp4Params)));
  const int owners = p.heads_per_wg / NH;  // waves of one phase
  const int own = wave % owners, phase = wave / owners;
  const int phases = kWaves / owners;
  const int seqs = kChunks ? p.decode_rows + p.chunks : p.decode_rows;

  // The share's place: sequence, head group, block, and tiles into the block, whose
  // setup counts `cost` of them; and the number of the item.  (A cold launch pays for
  // every line of code it runs through: decode rows have a path of their own.)
  int seq = 0, grp = 0, blk = 0, item = 0, off = 0, cost = 0;
  int pos = 0, end = 1, size = 1;
  float size_rcp = 1.f;
  SeqGeo g;
  // total units over the grid, rounded up with room for the estimate's error
  auto cut = [&](int total) {
    size = int(float(total) * p.grid_rcp * (1.f + 0x1p-21f)) + 1;
    size -= int64_t(size - 1) * grid >= total ? 1 : 0;
    size = max(p.min_share, size);
    size_rcp = __builtin_amdgcn_rcpf(float(size));
    const int64_t at = int64_t(share) * size;
    pos = int(min(at, int64_t(total)));
    end = int(min(at + size, int64_t(total)));
  };
  if (!kChunks && p.whole) {
    const int per_row = p.head_groups * p.row_blocks;
    seq = share / per_row;
    grp = (share - seq * per_row) / p.row_blocks;
    blk = share - seq * per_row - grp * p.row_blocks;
    g = load_seq<true>(p, seq);
  } else if (!kChunks) {
    const int per_row = p.head_groups * p.row_blocks, rows = p.decode_rows;
    // (the first 64 rows' sizes stay in the lanes: one read of them)
    SeqGeo gl = load_row(p, lane);
    int tiles = lane < rows ? tiles_of(p, gl) : 0;
    int incl = wave_scan_add(tiles);
    int sum = __builtin_amdgcn_readlane(incl, 63);
    cost = p.item_cost;
    if (__builtin_expect(rows > 64, 0)) {
      for (int r0 = 64; r0 < rows; r0 += 64) {
        const int r = r0 + lane;
        sum += wave_sum(r < rows ? tiles_of(p, load_row(p, r)) : 0);
      }
    } else {
      // Items of one length that the shares cut without remainder begin where
      // shares do: no share has more than one, and the setup is everybody's.
      const int one = __builtin_amdgcn_readfirstlane(tiles);
      cut(sum * per_row);
      if (__builtin_amdgcn_ballot_w64(lane < rows && tiles != one) == 0 &&
          div_steps(one, size, size_rcp) * size == one)
        cost = 0;
    }
    cut((sum + cost * rows) * per_row);
    if (share == 0 && threadIdx.x == 0) *p.count = rows * per_row;
    if (pos >= end) return;
    int before = 0;  // units of the rows ahead of r0
    int r0 = 0;
    uint64_t past;
    while ((past = __builtin_amdgcn_ballot_w64(
                before + (incl + cost * (lane + 1)) * per_row > pos && r0 + lane < rows)) == 0) {
      if (r0 + 64 >= rows) return;  // (lengths that changed since their sum)
      before += (__builtin_amdgcn_readlane(incl, 63) + cost * 64) * per_row;
      r0 += 64;
      gl = load_row(p, r0 + lane);
      tiles = r0 + lane < rows ? tiles_of(p, gl) : 0;
      incl = wave_scan_add(tiles);
    }
    const int at = __builtin_ctzll(past);
    const int each = __builtin_amdgcn_readlane(tiles, at) + cost;
    const int in =
        pos - before - (__builtin_amdgcn_readlane(incl, at) - each + cost * (at + 1)) * per_row;
    const int nth = div_steps(in, each, __builtin_amdgcn_rcpf(float(each)));
    off = in - nth * each;
    seq = r0 + at;
    item = seq * per_row + nth;
    grp = p.row_blocks == 1 ? nth : nth / p.row_blocks;
    blk = nth - grp * p.row_blocks;
    g = SeqGeo{seq, 1, __builtin_amdgcn_readlane(gl.given, at),
               __builtin_amdgcn_readlane(gl.keys, at)};
  } else {
    cost = p.whole ? 0 : p.item_cost;
    auto load_lane = [&](int r0, SeqGeo& gl, int& blocks, int& units) {
      gl = SeqGeo{0, 0, 0, 0};
      if (r0 + lane < seqs) gl = load_seq<false>(p, r0 + lane);
      blocks = blocks_of(p, gl);
      units = blocks * (tiles_of(p, gl) + cost);
    };
    SeqGeo gl;
    int blocks, units;
    load_lane(0, gl, blocks, units);
    int incl = wave_scan_add(units), incl_blocks = wave_scan_add(blocks);
    int sum = __builtin_amdgcn_readlane(incl, 63);
    int all_blocks = __builtin_amdgcn_readlane(incl_blocks, 63);
    for (int r0 = 64; r0 < seqs; r0 += 64) {
      SeqGeo other;
      int b, u;
      load_lane(r0, other, b, u);
      sum += wave_sum(u);
      all_blocks += wave_sum(b);
    }
    if (p.whole) {
      pos = min(share, sum * p.head_groups);
      end = min(share + 1, sum * p.head_groups);
    } else {
      if (share == 0 && threadIdx.x == 0) *p.count = all_blocks * p.head_groups;
      cut(sum * p.head_groups);
    }
    if (pos >= end) return;
    int before = 0, items = 0, r0 = 0;
    uint64_t past;
    while ((past = __builtin_amdgcn_ballot_w64(before + incl * p.head_groups > pos)) == 0) {
      if (r0 + 64 >= seqs) return;  // (as above)
      before += __builtin_amdgcn_readlane(incl, 63) * p.head_groups;
      items += __builtin_amdgcn_readlane(incl_blocks, 63);
      r0 += 64;
      load_lane(r0, gl, blocks, units);
      incl = wave_scan_add(units);
      incl_blocks = wave_scan_add(blocks);
    }
    const int at = __builtin_ctzll(past);
    seq = r0 + at;
    g = SeqGeo{__builtin_amdgcn_readlane(gl.q0, at), __builtin_amdgcn_readlane(gl.sq, at),
               __builtin_amdgcn_readlane(gl.given, at), __builtin_amdgcn_readlane(gl.keys, at)};
    const int u = __builtin_amdgcn_readlane(units, at);
    const int nb = __builtin_amdgcn_readlane(blocks, at);
    const int each = tiles_of(p, g) + cost;
    const int in = pos - before - (__builtin_amdgcn_readlane(incl, at) - u) * p.head_groups;
    grp = div_steps(in, u, __builtin_amdgcn_rcpf(float(u)));
    blk = div_steps(in - grp * u, each, __builtin_amdgcn_rcpf(float(each)));
    off = in - grp * u - blk * each;
    item = (items + __builtin_amdgcn_readlane(incl_blocks, at) - nb) * p.head_groups + grp * nb +
           blk;
  }

  const uint32_t lds0 = lds_addr(smem) + wave * (kSlots * kSlotBytes);
  const char* slot0 = smem + wave * (kSlots * kSlotBytes);
  const int row_bytes = p.kv_heads * kFp4RowBytes;
  // (NH = 2: the other loads' offsets differ by rows, and K's by an xor)
  const int k0 = TileLayout<NH>::load_key(0, lane, row_bytes);
  const int k1 = TileLayout<NH>::load_key(1, lane, row_bytes);
  const int v0 = TileLayout<NH>::load_value(0, lane, row_bytes);
  const int v1 = TileLayout<NH>::load_value(1, lane, row_bytes);
  // Of power lane: key lane & 31, head lane >> 5 (NH = 2).
  const int poff = ((lane & 31) * p.kv_heads + (NH == 2 ? lane >> 5 : 0)) * kFp4Powers;

  while (true) {
    const int tiles = p.whole ? 1 << 30 : tiles_of(p, g);
    const int seg0 = max(0, off - cost);
    const int seg1 = p.whole ? tiles : min(tiles, off - cost + (end - pos));
    if (seg1 <= seg0) break;  // (the share ends within the setup)
    const int head = grp * p.heads_per_wg + own * NH;
    // (more items than the host was told of have no record, and stay unjoined)
    if (!p.whole && seg0 == 0 && threadIdx.x == 0 && item < p.items)
      p.rec[item] = ItemRec{share, div_steps(pos - off + cost + tiles - 1, size, size_rcp),
                            g.q0,  g.sq, grp, blk, {0, 0}};

    // The lane's column: its query row, head and how many keys it sees; the most
    // and the fewest that a column of the block sees.
    const int col0 = blk * 16, last_col = g.sq * p.group - 1;
    const int col = min(col0 + lm, last_col);
    const int token = div_small(col, p.group, p.group_rcp);
    const int limit = min(g.keys, g.given - g.sq + token + 1);
    const int most = uniform(
        min(g.keys, g.given - g.sq + 1 +
                        div_small(min(col0 + 15, last_col), p.group, p.group_rcp)));
    const int least =
        uniform(min(g.keys, g.given - g.sq + 1 + div_small(col0, p.group, p.group_rcp)));
    // Tiles of this wave: t = seg0 + phase, then every phases-th.
    const int32_t* table = p.tables + seq * p.bt_stride;
    const int t_end = min(seg1, (max(most, 0) + kKeys - 1) / kKeys);
    int t = seg0 + phase;
    int pages0, pages;  // the lane's table entry, of page pages0 + lane
    // Rows of the pool from half u (32 keys) on, times kv heads, plus the head;
    // negative: nowhere.
    auto place_of = [&](int u) {
      const int pg = uniform(div_small(u, p.page_halves, p.page_halves_rcp));
      if (pg >= pages0 + 64) {
        pages0 = pg;
        pages = pg + lane < p.max_blocks ? table[pg + lane] : -1;
      }
      const int blk = __builtin_amdgcn_readlane(pages, pg - pages0);
      const bool there = blk >= 0 && blk < p.num_blocks;
      return there ? (int64_t(blk) * p.page + (u - pg * p.page_halves) * 32) * p.kv_heads + head
                   : int64_t(-1);
    };
    constexpr int kLoads = NH == 2 ? 10 : 12;  // of a tile
    const int code_bytes = 31 * row_bytes + NH * kFp4RowBytes;
    const int power_bytes = (31 * p.kv_heads + NH) * kFp4Powers;
    auto issue = [&](int tl, uint32_t lds) {
      if constexpr (NH == 2) {
        const int64_t w = place_of(tl);
        const int64_t at = max(w, int64_t(0));
        const int there = w >= 0 ? -1 : 0;
        load_powers(scalar_rsrc(p.ks + at * kFp4Powers, power_bytes & there), poff, lds + kKpAt);
        load_powers(scalar_rsrc(p.vs + at * kFp4Powers, power_bytes & there), poff, lds + kVpAt);
        const i32x4_t kr = scalar_rsrc(p.k + at * kFp4RowBytes, code_bytes & there);
        const i32x4_t vr = scalar_rsrc(p.v + at * kFp4RowBytes, code_bytes & there);
        const int step = 8 * row_bytes;
        load_codes<true>(kr, k0, k0 ^ 32, 0, step, lds);
        load_codes<true>(vr, v0, v0, 0, step, lds + kVAt);
        load_codes<true>(kr, k0 ^ 64, k0 ^ 96, 2 * step, 3 * step, lds + 2048);
        load_codes<true>(vr, v0, v0, 2 * step, 3 * step, lds + kVAt + 2048);
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int64_t w = (2 * tl + h) * 32 < g.keys ? place_of(2 * tl + h) : int64_t(-1);
          const int64_t at = max(w, int64_t(0));
          const int there = w >= 0 ? -1 : 0;
          if ((lane >> 5) == h) {
            load_powers(scalar_rsrc(p.ks + at * kFp4Powers, power_bytes & there), poff,
                        lds + kKpAt);
            load_powers(scalar_rsrc(p.vs + at * kFp4Powers, power_bytes & there), poff,
                        lds + kVpAt);
          }
          load_codes<false>(scalar_rsrc(p.k + at * kFp4RowBytes, code_bytes & there), k0, k1, 0, 0,
                     lds + 2048 * h);
          load_codes<false>(scalar_rsrc(p.v + at * kFp4RowBytes, code_bytes & there),
                     v0 ^ (32 * h), v1 ^ (32 * h), 0, 0, lds + kVAt + 2048 * h);
        }
      }
    };
    // Queries and table entries come in together, then two tiles go on their way
    // and the queries are split behind them.
    QueryRow qr[NH];
#pragma unroll
    for (int i = 0; i < NH; ++i)
      qr[i] = load_query(p.q + int64_t(g.q0 + token) * p.q_st +
                             int64_t((head + i) * p.group + col - token * p.group) * p.q_sh,
                         lg);
    pages0 = uniform(div_small(t * (kKeys / 32), p.page_halves, p.page_halves_rcp));
    pages = pages0 + lane < p.max_blocks ? table[pages0 + lane] : -1;
    asm volatile("" : "+v"(pages));
#pragma unroll
    for (int i = 0; i < NH; ++i)
#pragma unroll
      for (int d = 0; d < 4; ++d) asm volatile("" : "+v"(qr[i].x[d]));
    if (t < t_end) issue(t, lds0);
    if (t + phases < t_end) issue(t + phases, lds0 + kSlotBytes);
    Query q[NH];
    Carry c[NH];
#pragma unroll
    for (int i = 0; i < NH; ++i) {
      q[i] = split_query(qr[i], p.flip);
#pragma unroll
      for (int cb = 0; cb < 8; ++cb) c[i].o[cb] = f32x4_t{0.f, 0.f, 0.f, 0.f};
      c[i].l = f32x4_t{0.f, 0.f, 0.f, 0.f};
      c[i].m = kLowest;
    }
    int slot = 0;
    for (; t < t_end; t += phases) {
      if (t + phases < t_end) {
        wait_loads<kLoads>();
      } else {
        wait_loads<0>();
      }
      Tile x;
      read_tile<NH>(x, slot0 + slot, lane, lm, lg);
      f32x4_t s[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const Query& qi = q[NH == 2 ? i >> 1 : 0];
        s[i] = mfma_fp4(x.k[i], qi.lo, f32x4_t{0.f, 0.f, 0.f, 0.f}, x.k_power[i], qi.lo_power);
        s[i] = mfma_fp4(x.k[i], qi.hi, s[i], x.k_power[i], qi.hi_power);
      }
      if (__builtin_expect(least < (t + 1) * kKeys, 0))
        mask_tile<NH>(x, s, limit - t * kKeys, lg);
      u32x4_t w[2];
#pragma unroll
      for (int i = 0; i < NH; ++i) weights<16 / NH>(s + 2 * i, c[i], p.c2, w + i);
      // (a wave at its products goes ahead of one at its softmax: another 0.7 %)
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int h = 0; h < 2; ++h) weigh(x, h, w[h], c[NH == 2 ? h : 0]);
      __builtin_amdgcn_s_setprio(0);
      add_nan_runs<NH>(x.mine, limit - t * kKeys, c);
      // (The next loads go out here, not once the tile is read: their addresses and
      // issue would stand ahead of the scores.  16 rows of 32768 keys 52.6 -> 51.6 us.)
      smem_drain();
      if (t + 2 * phases < t_end) issue(t + 2 * phases, lds0 + slot);
      slot ^= kSlotBytes;
    }

    // Channels 16 cb .. + 15 of the wave's columns: the result, or a partial in
    // slot 2 share + 1 (the piece that begins its item), else 2 share.
    // (Arguments of the epilogue are read again here: held through the loop, they
    // would take registers from it.)
    const KernelArgs* e = kernel_args();
    const bool done = seg0 == 0 && seg1 == tiles;
    const bool mine_too = col0 + lm <= last_col;  // (else the last column again)
    const int64_t part =
        (int64_t(2) * share + (seg0 == 0 ? 1 : 0)) * e->heads_per_wg * e->cols + lm;
    auto emit = [&](int i, int cb, const f32x4_t& o, float m, float l) {
      if (done) {
        const float inv = l != 0.f ? 1.f / l : 0.f;
        uint16_t* dst = e->out + int64_t(g.q0 + token) * e->o_st +
                        int64_t((head + i) * e->group + col - token * e->group) * e->o_sh +
                        16 * cb + 4 * lg;
        *reinterpret_cast<u32x2_t*>(dst) = u32x2_t{pack_bf16x2_fast(o[0] * inv, o[1] * inv),
                                                   pack_bf16x2_fast(o[2] * inv, o[3] * inv)};
      } else {
        const int64_t at = part + (own * NH + i) * e->cols;
        *reinterpret_cast<f32x4_t*>(e->part_o + at * kD + 16 * cb + 4 * lg) = o;
        if (cb == 0 && lg == 0) e->part_ml[at] = float2{m, l};
      }
    };
    // Phases joined through the waves' own slots, a head to a slot: each wave makes
    // its part of its heads' channel blocks.
    char* mine = smem + wave * (kSlots * kSlotBytes);
    smem_drain();
    if (mine_too) {
#pragma unroll
      for (int i = 0; i < NH; ++i) {
#pragma unroll
        for (int cb = 0; cb < 8; ++cb)
          *reinterpret_cast<f32x4_t*>(mine + i * kSlotBytes + cb * 1024 + lane * 16) = c[i].o[cb];
        *reinterpret_cast<float2*>(mine + i * kSlotBytes + 8192 + lane * 8) =
            float2{c[i].m, c[i].l[0]};
      }
    }
    pf_barrier();
    const char* first = smem + own * (kSlots * kSlotBytes);
    const int apart = owners * (kSlots * kSlotBytes);
    if (mine_too) {
#pragma unroll
      for (int i = 0; i < NH; ++i) {
        auto put = [&](int cb, const f32x4_t& o, float top, float l) { emit(i, cb, o, top, l); };
        if (NH == 1 || phases == 8) {
          join<8>(first + i * kSlotBytes, apart, phase, lane, put);
        } else if (phases == 2) {
          join<2>(first + i * kSlotBytes, apart, phase, lane, put);
        } else {
          join<4>(first + i * kSlotBytes, apart, phase, lane, put);
        }
      }
    }
    pf_barrier();

    if (p.whole) break;
    pos += cost + tiles - off;
    if (pos >= end) break;
    off = 0;
    ++item;
    if (++blk < blocks_of(p, g)) continue;
    blk = 0;
    if (++grp < p.head_groups) continue;
    grp = 0;
    do {
      if (++seq >= seqs) return;  // (pos < end: there is one)
      g = load_seq<true>(p, seq);
    } while (kChunks && g.sq == 0);
  }
}

// ---------------------------------------------------------------------------
// Join the partials of items cut between shares: 32 lanes a column and slice of its
// pieces, kGroups of them a workgroup, which takes kGroups / S columns of an item in S
// slices each (by how many pieces an item has: 1 item in 256 pieces 4.6 us, 64 items
// in 5 pieces each 4).
// ---------------------------------------------------------------------------
constexpr int kGroups = 16;
constexpr int kAhead = 8;  // pieces of a slice whose loads are in flight together
template <int S>
__global__ void __launch_bounds__(32 * kGroups) fp4_merge_kernel(Fp4Params p) {
  __shared__ f32x4_t so[kGroups][32];
  __shared__ float2 sml[kGroups];
  touch_kernel_args(int(sizeof(Fp4Params)));
  // (both read at once; past the count there is room for a record but none)
  const int count = *p.count;
  ItemRec rec = p.rec[blockIdx.x];
  asm volatile("" ::"s"(count), "s"(rec.first), "s"(rec.sq));
  const int2 r = {rec.first, rec.last};
  if (int(blockIdx.x) >= count || r.x >= r.y) return;
  const int lane = threadIdx.x & 31, at_group = threadIdx.x >> 5, slice = at_group % S;
  // The workgroup's at_group / S-th column: of a head of the item's, one of its block's.
  const int nth = blockIdx.y * (kGroups / S) + at_group / S;
  const int hs = div_small(nth, p.cols, __builtin_amdgcn_rcpf(float(p.cols)));
  const int in = nth - hs * p.cols;
  const int col = rec.block * 16 + in;
  const bool live = hs < p.heads_per_wg && col < rec.sq * p.group;
  const int token = div_small(col, p.group, p.group_rcp);
  const int head = (rec.group * p.heads_per_wg + hs) * p.group + col - token * p.group;
  const int64_t cols = int64_t(p.heads_per_wg) * p.cols;
  float top = kLowest, l = 0.f;
  f32x4_t o = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = live ? r.x + slice : r.y + 1; s0 <= r.y; s0 += S * kAhead) {
    float2 ml[kAhead];
    f32x4_t part[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int s = min(s0 + S * i, r.y);
      const int64_t c = (int64_t(2) * s + (s == r.x)) * cols + nth;
      ml[i] = p.part_ml[c];
      part[i] = reinterpret_cast<const f32x4_t*>(p.part_o + c * kD)[lane];
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (s0 + S * i > r.y) continue;
      const float next = fmaxf(top, ml[i].x);
      const float a = __builtin_amdgcn_exp2f(top - next);
      const float b = __builtin_amdgcn_exp2f(ml[i].x - next);
      top = next;
      l = l * a + ml[i].y * b;
      o = o * a + part[i] * b;
    }
  }
  if constexpr (S > 1) {
    so[at_group][lane] = o;
    if (lane == 0) sml[at_group] = float2{top, l};
    __syncthreads();
    if (slice != 0) return;
#pragma unroll
    for (int i = 1; i < S; ++i) top = fmaxf(top, sml[at_group + i].x);
    l = 0.f;
    o = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < S; ++i) {
      const float b = __builtin_amdgcn_exp2f(sml[at_group + i].x - top);
      l += sml[at_group + i].y * b;
      o += so[at_group + i][lane] * b;
    }
  }
  if (!live) return;
  const float inv = l != 0.f ? 1.f / l : 0.f;
  uint16_t* dst = p.out + int64_t(rec.q0 + token) * p.o_st + head * p.o_sh + 4 * lane;
  *reinterpret_cast<u32x2_t*>(dst) =
      u32x2_t{pack_bf16x2_fast(o[0] * inv, o[1] * inv), pack_bf16x2_fast(o[2] * inv, o[3] * inv)};
}

// ---------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------
int cu_count() {
  static std::atomic<int> known[64];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
  int n = known[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess ||
        n <= 0) {
      (void)hipGetLastError();
      n = 256;
    }
    known[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

struct Plan {
  int pair;  // waves take two heads
  int heads_per_wg, head_groups, cols, grid, min_share, item_cost, whole;
  int64_t items;  // at most
  size_t rec_at, ml_at, o_at, bytes;
};

size_t up256(size_t n) { return (n + 255) & ~size_t(255); }

// How the work is cut.  Whole: a workgroup takes an item of one, two, four or eight kv
// heads alone, and there is one launch; its eight waves make one tile each a round, 512
// keys of one head (64 a wave) or 256, 128 or 64 of more (a wave takes two heads and 32
// keys).  Cut: two heads a wave, the tiles of all items in equal shares, one a CU, and a
// second launch joins the pieces.  Estimates in us:
//   whole  the longer of ceil(items / CUs) (7 + 2.2 a round of the longest row) and 7 +
//          the keys' bytes at 4 TB/s (one head: half lines), 6 (two) or 6.4
//   cut    13.5, 7 more as the heads' blocks get to 128 and 6 more for every 256 items
//          (more of them in a share), and the longer of the keys' bytes at 6.6 TB/s and
//          0.9 ns for every 64 keys of a head and block
// The host knows a batch's longest row by its table's width; its keys are taken as 0.8 of
// that for every row, between batches of one length and ragged ones, and as half of it
// where chunks join decode rows (200 rows of 300 to 2000 keys and a chunk over 4000: cut
// 43, whole 64).  Measured, cut / whole by one, two, four and eight heads (rows x keys; 4
// kv heads): 1 x 1000 13.1 / 10.1 / 15.1 / 21.5, 8 x 4096 17 / 23 / 35 / 60, 16 x 8192
// 26 / 40 / 61 / 113, 64 x 300 19 / 8.3 / 10.7 / 12.9, 64 x 4096 35 / 28 / 38 / 62, 64 x
// 8192 56 / 60 / 66 / 114, 48 x 1025 to 8007 32 / 40 / 60 / 107, 128 x 1000 28 / 23 / 19 /
// 23, 128 x 4096 59 / 65 / 52 / 65, 192 x 1000 34 / 34 / 33 / 24, 256 x 300 to 900 34 / 36
// / 30 / 23; 8 kv heads: 128 x 300 to 900 34 / 37 / 31 / 24 / 35, 200 x 1000 54 / 82 / 70 /
// 53 / 44, 400 x 20 to 80 35 / 60 / 43 / 28 / 21.  Of 190 shapes the choice is over 8 % off
// in four, 21 % at worst:
// all with tables as wide as the longest row, over two inputs in turn, so that pools under
// 256 MB lay partly in the cache behind the L2s (64 x 4096 whole, one head, over three:
// 33).  Rows far shorter than their table are taken for long ones and cut: 64 rows of 300
// keys 7.4 us under a table of 512 keys, 16.4 under one of 32768.
Plan make_plan(int64_t decode_rows, int64_t chunks, int64_t chunk_tokens, int64_t chunk_blocks,
               int64_t heads, int64_t kv_heads, int64_t most_keys) {
  Plan pl{};
  const int64_t group = heads / kv_heads;
  const int cus = cu_count();
  pl.cols = int(chunks > 0 ? 16 : std::min<int64_t>(group, 16));
  // (of the chunks at most, where the caller does not know)
  if (chunk_blocks <= 0) chunk_blocks = (chunk_tokens * group + 15 * chunks) / 16;
  const int64_t blocks = decode_rows * ((group + 15) / 16) + chunk_blocks;
  const double heads_of = double(blocks) * double(kv_heads), keys = double(most_keys);
  const double part = decode_rows > 0 && chunks > 0 ? 0.5 : 0.8;
  const double bytes = part * double(decode_rows + chunks) * double(kv_heads) * keys *
                       (2 * (kFp4RowBytes + kFp4Powers));
  int best = 1;
  double whole = 1e30;
  const double rate[] = {4e6, 6e6, 6.4e6, 6.4e6};  // bytes a us
  for (int i = 0; i < 4 && kv_heads % (1 << i) == 0; ++i) {
    const int n = 1 << i;
    const double t = std::max(std::ceil(heads_of / n / cus) * (7 + 2.2 * keys * n / 512),
                              7 + bytes / rate[i]);
    if (t < whole) whole = t, best = n;
  }
  // Cut: few items are cut finer between two heads a workgroup (16 rows of 4096 keys 19.9
  // against 21.9, one row of 4096 13.5 against 15.7); many share a workgroup better
  // among four (128 rows of 500 to 1500 keys 39.0 against 41.5).
  const int apart = kv_heads % 2 != 0 ? 1 : kv_heads % 4 == 0 && heads_of > 128 ? 4 : 2;
  const double cut = 13.5 + 7 * std::min(1., heads_of / 128) +
                     6 * std::max(0., heads_of / apart / cus - 0.5) +
                     std::max(bytes / 6.6e6, part * heads_of * keys / 64 * 0.9e-3);
  pl.whole = whole <= cut;
  pl.heads_per_wg = pl.whole ? best : apart;
  pl.pair = pl.heads_per_wg > 1;
  pl.head_groups = int(kv_heads / pl.heads_per_wg);
  pl.min_share = 2;
  pl.item_cost = pl.pair ? 16 : 8;
  pl.items = blocks * pl.head_groups;
  pl.grid = int(pl.whole ? std::min<int64_t>(pl.items, 1 << 30) : cus);
  size_t at = 0;
  if (!pl.whole) {
    pl.rec_at = 256;  // (the count of items comes first)
    at = up256(pl.rec_at + size_t(pl.items) * sizeof(ItemRec));
    pl.ml_at = at;
    const size_t cols = size_t(2) * pl.grid * pl.heads_per_wg * pl.cols;
    at = up256(at + cols * sizeof(float2));
    pl.o_at = at;
    at = up256(at + cols * kD * sizeof(float));
  }
  pl.bytes = at;
  return pl;
}

// An append's arguments, its checks and its launch.
struct Append {
  const void* key;
  int64_t k_sn, k_sh;
  const void* value;
  int64_t v_sn, v_sh;
  uint8_t *k, *v, *ks, *vs;
  int64_t num_slots;
  const void* slots;
  int slot_bytes;
  int64_t tokens, kv_heads;
};

int check_rows(const char* what, const void* key, int64_t k_sn, int64_t k_sh, const void* value,
               int64_t v_sn, int64_t v_sh, int64_t num_tokens, int64_t kv_heads, int64_t head_dim,
               int slot_index_bytes) {
  KVC_REQUIRE(head_dim == kD, KVC_ERR_VALUE, "%s: head_dim must be 128 (got %lld)", what,
              (long long)head_dim);
  KVC_REQUIRE(num_tokens >= 0 && kv_heads > 0 && kv_heads <= 4096, KVC_ERR_VALUE,
              "%s: bad token or kv head count", what);
  KVC_REQUIRE(slot_index_bytes == 4 || slot_index_bytes == 8, KVC_ERR_VALUE,
              "%s: slot_mapping must be int32 or int64", what);
  KVC_REQUIRE(num_tokens * kv_heads <= (int64_t(1) << 31) * kRowsPerBlock - kRowsPerBlock,
              KVC_ERR_VALUE, "%s: too many rows for one launch", what);
  KVC_REQUIRE(num_tokens == 0 ||
                  (reinterpret_cast<uintptr_t>(key) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(value) % 16 == 0 && k_sn % 8 == 0 &&
                   k_sh % 8 == 0 && v_sn % 8 == 0 && v_sh % 8 == 0),
              KVC_ERR_ASSERT, "%s: key/value rows must be 16-byte aligned", what);
  return KVC_OK;
}

int check_pool(const char* what, const void* k, const void* v, const void* ks, const void* vs) {
  KVC_REQUIRE(k != nullptr && v != nullptr && ks != nullptr && vs != nullptr, KVC_ERR_VALUE,
              "%s: null pool", what);
  KVC_REQUIRE(reinterpret_cast<uintptr_t>(k) % 16 == 0 &&
                  reinterpret_cast<uintptr_t>(v) % 16 == 0 &&
                  reinterpret_cast<uintptr_t>(ks) % 4 == 0 &&
                  reinterpret_cast<uintptr_t>(vs) % 4 == 0,
              KVC_ERR_ASSERT, "%s: pools must be 16-byte aligned, scales 4-byte", what);
  return KVC_OK;
}

int check_append(const char* what, const Append& a, int64_t head_dim) {
  int rc = check_rows(what, a.key, a.k_sn, a.k_sh, a.value, a.v_sn, a.v_sh, a.tokens, a.kv_heads,
                      head_dim, a.slot_bytes);
  if (rc != KVC_OK || a.tokens == 0) return rc;
  rc = check_pool(what, a.k, a.v, a.ks, a.vs);
  if (rc != KVC_OK) return rc;
  KVC_REQUIRE(a.key != nullptr && a.value != nullptr && a.slots != nullptr, KVC_ERR_VALUE,
              "%s: null rows or slots", what);
  return KVC_OK;
}

void launch_append(const Append& a, hipStream_t st) {
  if (a.tokens == 0) return;
  const int64_t rows = a.tokens * a.kv_heads;
  const dim3 grid(unsigned((rows + kRowsPerBlock - 1) / kRowsPerBlock));
  auto kern = a.slot_bytes == 8 ? store_fp4_kernel<8> : store_fp4_kernel<4>;
  kern<<<grid, kThreads, 0, st>>>(
      static_cast<const uint16_t*>(a.key), a.k_sn, a.k_sh, static_cast<const uint16_t*>(a.value),
      a.v_sn, a.v_sh, a.k, a.v, a.ks, a.vs, a.num_slots, a.slots, a.tokens, int(a.kv_heads));
}

}  // namespace
}  // namespace kvc

using namespace kvc;

extern "C" int kvc_store_fp4(const void* key, int64_t key_stride_n, int64_t key_stride_h,
                             const void* value, int64_t value_stride_n, int64_t value_stride_h,
                             uint8_t* k_cache, uint8_t* v_cache, uint8_t* k_scale,
                             uint8_t* v_scale, int64_t num_slots, const void* slot_mapping,
                             int slot_index_bytes, int64_t num_tokens, int64_t num_kv_heads,
                             int64_t head_dim, kvc_stream_t stream) {
  clear_error();
  const Append a{key, key_stride_n, key_stride_h, value, value_stride_n, value_stride_h,
                 k_cache, v_cache, k_scale, v_scale, num_slots,
                 slot_mapping, slot_index_bytes, num_tokens, num_kv_heads};
  const int rc = check_append("store_fp4", a, head_dim);
  if (rc != KVC_OK || num_tokens == 0) return rc;
  launch_append(a, as_stream(stream));
  return check_launch("store_fp4");
}

extern "C" int kvc_dequant_fp4(const uint8_t* codes, const uint8_t* scale, int64_t rows,
                               int64_t head_dim, void* out, kvc_stream_t stream) {
  clear_error();
  KVC_REQUIRE(head_dim == kD && rows >= 0, KVC_ERR_VALUE,
              "dequant_fp4: head_dim must be 128 (got %lld)", (long long)head_dim);
  if (rows == 0) return KVC_OK;
  KVC_REQUIRE(rows <= (int64_t(1) << 31) * kRowsPerBlock - kRowsPerBlock, KVC_ERR_VALUE,
              "dequant_fp4: too many rows for one launch");
  KVC_REQUIRE(codes != nullptr && scale != nullptr && out != nullptr, KVC_ERR_VALUE,
              "dequant_fp4: null buffer");
  KVC_REQUIRE(reinterpret_cast<uintptr_t>(codes) % 4 == 0 &&
                  reinterpret_cast<uintptr_t>(out) % 16 == 0,
              KVC_ERR_ASSERT, "dequant_fp4: codes must be 4-byte aligned, out 16-byte");
  const dim3 grid(unsigned((rows + kRowsPerBlock - 1) / kRowsPerBlock));
  dequant_fp4_kernel<<<grid, kThreads, 0, as_stream(stream)>>>(codes, scale, rows,
                                                               static_cast<uint16_t*>(out));
  return check_launch("dequant_fp4");
}

extern "C" int kvc_gather_kv_fp4(const uint8_t* k_cache, const uint8_t* v_cache,
                                 const uint8_t* k_scale, const uint8_t* v_scale,
                                 int64_t num_cache_blocks, int64_t page_size,
                                 int64_t num_kv_heads, int64_t head_dim,
                                 const int32_t* block_tables, int64_t bt_stride,
                                 int64_t max_blocks_per_seq, int64_t block_table_row0,
                                 int64_t num_prefill, const int32_t* cu_seqlens_k,
                                 int64_t total_keys, void* out_k, void* out_v,
                                 kvc_stream_t stream) {
  clear_error();
  KVC_REQUIRE(head_dim == kD, KVC_ERR_VALUE, "gather_kv_fp4: head_dim must be 128 (got %lld)",
              (long long)head_dim);
  KVC_REQUIRE(num_cache_blocks >= 0 && page_size > 0 && page_size < (int64_t(1) << 30) &&
                  num_kv_heads > 0 && num_kv_heads <= 4096 && max_blocks_per_seq >= 0 &&
                  max_blocks_per_seq < (int64_t(1) << 31) && block_table_row0 >= 0 &&
                  num_prefill >= 0 && num_prefill < (int64_t(1) << 31) && total_keys >= 0,
              KVC_ERR_VALUE, "gather_kv_fp4: bad shape");
  KVC_REQUIRE(total_keys * num_kv_heads <= (int64_t(1) << 31) * kRowsPerBlock - kRowsPerBlock,
              KVC_ERR_VALUE, "gather_kv_fp4: too many rows for one launch");
  if (total_keys == 0 || num_prefill == 0) return KVC_OK;
  const int rc = check_pool("gather_kv_fp4", k_cache, v_cache, k_scale, v_scale);
  if (rc != KVC_OK) return rc;
  KVC_REQUIRE(block_tables != nullptr && cu_seqlens_k != nullptr && out_k != nullptr &&
                  out_v != nullptr,
              KVC_ERR_VALUE, "gather_kv_fp4: null tables, offsets or output");
  KVC_REQUIRE(reinterpret_cast<uintptr_t>(out_k) % 16 == 0 &&
                  reinterpret_cast<uintptr_t>(out_v) % 16 == 0,
              KVC_ERR_ASSERT, "gather_kv_fp4: outputs must be 16-byte aligned");
  const int64_t rows = total_keys * num_kv_heads;
  const dim3 grid(unsigned((rows + kRowsPerBlock - 1) / kRowsPerBlock));
  gather_fp4_kernel<<<grid, kThreads, 0, as_stream(stream)>>>(
      k_cache, v_cache, k_scale, v_scale, num_cache_blocks * page_size, int(page_size),
      int(num_kv_heads), block_tables, bt_stride, int(max_blocks_per_seq), block_table_row0,
      int(num_prefill), cu_seqlens_k, total_keys, static_cast<uint16_t*>(out_k),
      static_cast<uint16_t*>(out_v));
  return check_launch("gather_kv_fp4");
}

namespace {
// append (or null): launched ahead of the rows, once the whole call has been checked.
int run_rows(const char* what, const Append* append, const void* q, int64_t q_st, int64_t q_sh,
             int64_t heads, const uint8_t* k_cache, const uint8_t* v_cache,
             const uint8_t* k_scale, const uint8_t* v_scale, int64_t blocks, int64_t page,
             int64_t kv_heads, int64_t head_dim, const int32_t* tables, int64_t bt_stride,
             int64_t max_blocks, int64_t decode_rows, const int32_t* lens, int64_t chunks,
             int64_t chunk_tokens, int64_t chunk_blocks, const int32_t* cu_q,
             const int32_t* cu_k, float scale, void* out, int64_t o_st, int64_t o_sh,
             void* workspace, size_t workspace_bytes, kvc_stream_t stream) {
  KVC_REQUIRE(head_dim == kD, KVC_ERR_VALUE, "%s: head_dim must be 128 (got %lld)", what,
              (long long)head_dim);
  KVC_REQUIRE(kv_heads > 0 && heads > 0 && heads % kv_heads == 0, KVC_ERR_VALUE,
              "%s: num_heads must be a multiple of num_kv_heads", what);
  KVC_REQUIRE(page > 0 && page % 32 == 0, KVC_ERR_VALUE,
              "%s: page_size must be a multiple of 32 (got %lld)", what, (long long)page);
  // (offsets inside a tile and key counts are 32-bit; div_small's range)
  KVC_REQUIRE(kv_heads <= 4096 && heads <= 65536 && max_blocks >= 0 && blocks >= 0 &&
                  blocks < (int64_t(1) << 31) && page <= (1 << 20) &&
                  page * max_blocks <= (int64_t(1) << 26),
              KVC_ERR_VALUE, "%s: shape out of range (tables of up to 2^26 keys)", what);
  KVC_REQUIRE(decode_rows >= 0 && chunks >= 0 && chunk_tokens >= 0 &&
                  decode_rows + chunks + chunk_tokens < (int64_t(1) << 24) &&
                  chunk_tokens * (heads / kv_heads) < (int64_t(1) << 24),
              KVC_ERR_VALUE, "%s: too many rows", what);
  if (decode_rows + chunk_tokens == 0 || decode_rows + chunks == 0) {
    if (append == nullptr || append->tokens == 0) return KVC_OK;
    launch_append(*append, as_stream(stream));
    return check_launch(what);
  }
  const int rc = check_pool(what, k_cache, v_cache, k_scale, v_scale);
  if (rc != KVC_OK) return rc;
  KVC_REQUIRE(q != nullptr && out != nullptr && (lens != nullptr || decode_rows == 0) &&
                  ((cu_q != nullptr && cu_k != nullptr) || chunks == 0) &&
                  (tables != nullptr || max_blocks == 0),
              KVC_ERR_VALUE, "%s: null pointer", what);
  KVC_REQUIRE(reinterpret_cast<uintptr_t>(q) % 16 == 0 && q_st % 8 == 0 && q_sh % 8 == 0 &&
                  reinterpret_cast<uintptr_t>(out) % 16 == 0 && o_st % 8 == 0 && o_sh % 8 == 0,
              KVC_ERR_ASSERT, "%s: q/out rows must be 16-byte aligned", what);
  const Plan pl = make_plan(decode_rows, chunks, chunk_tokens, chunk_blocks, heads, kv_heads,
                            page * max_blocks);
  // (units of the cut are 32-bit)
  KVC_REQUIRE(pl.items * (page * max_blocks / 32 + 64) < (int64_t(1) << 31), KVC_ERR_VALUE,
              "%s: too many rows for tables of this width", what);
  KVC_REQUIRE(pl.bytes == 0 || (workspace != nullptr && workspace_bytes >= pl.bytes),
              KVC_ERR_WORKSPACE, "%s: workspace of %zu bytes needed", what, pl.bytes);
  KVC_REQUIRE(pl.bytes == 0 || reinterpret_cast<uintptr_t>(workspace) % 16 == 0, KVC_ERR_ASSERT,
              "%s: workspace must be 16-byte aligned", what);
  Fp4Params p{};
  p.q = static_cast<const uint16_t*>(q);
  p.q_st = q_st;
  p.q_sh = q_sh;
  p.out = static_cast<uint16_t*>(out);
  p.o_st = o_st;
  p.o_sh = o_sh;
  p.k = k_cache;
  p.v = v_cache;
  p.ks = k_scale;
  p.vs = v_scale;
  p.tables = tables;
  p.bt_stride = bt_stride;
  p.lens = lens;
  p.cu_q = cu_q;
  p.cu_k = cu_k;
  p.decode_rows = int(decode_rows);
  p.chunks = int(chunks);
  p.chunk_tokens = int(chunk_tokens);
  p.max_blocks = int(max_blocks);
  p.num_blocks = int(blocks);
  p.page = int(page);
  p.page_halves = int(page / 32);
  p.page_halves_rcp = 1.f / float(p.page_halves);
  p.kv_heads = int(kv_heads);
  p.group = int(heads / kv_heads);
  p.group_rcp = 1.f / float(p.group);
  p.heads_per_wg = pl.heads_per_wg;
  p.head_groups = pl.head_groups;
  p.tile_shift = pl.pair ? 5 : 6;
  p.cols = pl.cols;
  p.min_share = pl.min_share;
  p.item_cost = pl.item_cost;
  p.grid_rcp = 1.f / float(pl.grid);
  p.whole = pl.whole;
  p.row_blocks = (p.group + 15) / 16;
  p.items = int(pl.items);
  // (a scale of 0 stays above it: masked scores are -infinity)
  p.c2 = std::max(std::abs(scale) * kLog2e, 1e-37f);
  p.flip = scale < 0.f ? 0x80008000u : 0u;
  char* ws = static_cast<char*>(workspace);
  p.count = reinterpret_cast<int*>(ws);
  p.rec = reinterpret_cast<ItemRec*>(ws + pl.rec_at);
  p.part_ml = reinterpret_cast<float2*>(ws + pl.ml_at);
  p.part_o = reinterpret_cast<float*>(ws + pl.o_at);
  constexpr int kLds = kWaves * kSlots * kSlotBytes;
  hipStream_t st = as_stream(stream);
  static std::atomic<uint64_t> ready{0};  // devices whose LDS limit is set
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  const uint64_t bit = uint64_t(1) << (dev & 63);
  if (e == hipSuccess && !(ready.load(std::memory_order_relaxed) & bit)) {
    for (auto kern : {fp4_decode_kernel<1, false>, fp4_decode_kernel<2, false>,
                      fp4_decode_kernel<1, true>, fp4_decode_kernel<2, true>})
      if (e == hipSuccess)
        e = hipFuncSetAttribute(reinterpret_cast<const void*>(kern),
                                hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
    if (e == hipSuccess) ready.fetch_or(bit, std::memory_order_relaxed);
  }
  KVC_REQUIRE(e == hipSuccess, KVC_ERR_RUNTIME, "%s: LDS limit: %s", what, hipGetErrorString(e));
  auto kern = chunks > 0 ? (pl.pair ? fp4_decode_kernel<2, true> : fp4_decode_kernel<1, true>)
                         : (pl.pair ? fp4_decode_kernel<2, false> : fp4_decode_kernel<1, false>);
  if (append != nullptr) launch_append(*append, st);
  kern<<<pl.grid, 64 * kWaves, kLds, st>>>(p);
  if (!pl.whole) {
    const int64_t pieces = pl.grid / std::max<int64_t>(pl.items, 1) + 2;  // of an item
    const int slices = pieces <= kAhead ? 1 : pieces <= 4 * kAhead ? 4 : kGroups;
    auto merge = slices == 1   ? fp4_merge_kernel<1>
                 : slices == 4 ? fp4_merge_kernel<4>
                               : fp4_merge_kernel<kGroups>;
    const int per_wg = kGroups / slices;
    merge<<<dim3(unsigned(pl.items), unsigned((pl.heads_per_wg * pl.cols + per_wg - 1) / per_wg)),
            32 * kGroups, 0, st>>>(p);
  }
  return check_launch(what);
}
}  // namespace

extern "C" size_t kvc_paged_decode_fp4_workspace_bytes(int64_t batch, int64_t num_heads,
                                                       int64_t num_kv_heads, int64_t page_size,
                                                       int64_t max_blocks_per_seq) {
  if (batch <= 0 || num_kv_heads <= 0 || num_heads <= 0 || num_heads % num_kv_heads != 0) return 0;
  return make_plan(batch, 0, 0, 0, num_heads, num_kv_heads, page_size * max_blocks_per_seq).bytes;
}

extern "C" int kvc_paged_decode_fp4(
    const void* q, int64_t q_stride_b, int64_t q_stride_h, const uint8_t* k_cache,
    const uint8_t* v_cache, const uint8_t* k_scale, const uint8_t* v_scale,
    int64_t num_cache_blocks, int64_t page_size, int64_t num_kv_heads, int64_t head_dim,
    const int32_t* block_tables, int64_t bt_stride, int64_t max_blocks_per_seq,
    const int32_t* context_lens, int64_t batch, int64_t num_heads, float scale, void* out,
    int64_t out_stride_b, int64_t out_stride_h, void* workspace, size_t workspace_bytes,
    kvc_stream_t stream) {
  clear_error();
  return run_rows("paged_decode_fp4", nullptr, q, q_stride_b, q_stride_h, num_heads, k_cache,
                  v_cache, k_scale, v_scale, num_cache_blocks, page_size, num_kv_heads, head_dim,
                  block_tables, bt_stride, max_blocks_per_seq, batch, context_lens, 0, 0, 0,
                  nullptr, nullptr, scale, out, out_stride_b, out_stride_h, workspace,
                  workspace_bytes, stream);
}

extern "C" int kvc_paged_decode_append_fp4(
    const void* q, int64_t q_stride_b, int64_t q_stride_h, const void* key, int64_t key_stride_n,
    int64_t key_stride_h, const void* value, int64_t value_stride_n, int64_t value_stride_h,
    const void* slot_mapping, int slot_index_bytes, int64_t num_tokens, uint8_t* k_cache,
    uint8_t* v_cache, uint8_t* k_scale, uint8_t* v_scale, int64_t num_cache_blocks,
    int64_t page_size, int64_t num_kv_heads, int64_t head_dim, const int32_t* block_tables,
    int64_t bt_stride, int64_t max_blocks_per_seq, const int32_t* context_lens, int64_t batch,
    int64_t num_heads, float scale, void* out, int64_t out_stride_b, int64_t out_stride_h,
    void* workspace, size_t workspace_bytes, kvc_stream_t stream) {
  clear_error();
  const Append a{key, key_stride_n, key_stride_h, value, value_stride_n, value_stride_h,
                 k_cache, v_cache, k_scale, v_scale, num_cache_blocks * page_size,
                 slot_mapping, slot_index_bytes, num_tokens, num_kv_heads};
  const int rc = check_append("paged_decode_append_fp4", a, head_dim);
  if (rc != KVC_OK) return rc;
  return run_rows("paged_decode_append_fp4", &a, q, q_stride_b, q_stride_h, num_heads, k_cache,
                  v_cache, k_scale, v_scale, num_cache_blocks, page_size, num_kv_heads, head_dim,
                  block_tables, bt_stride, max_blocks_per_seq, batch, context_lens, 0, 0, 0,
                  nullptr, nullptr, scale, out, out_stride_b, out_stride_h, workspace,
                  workspace_bytes, stream);
}

extern "C" size_t kvc_varlen_fp4_workspace_bytes(int64_t num_q_tokens, int64_t num_heads,
                                                 int64_t num_kv_heads, int64_t page_size,
                                                 int64_t max_blocks_per_seq,
                                                 int64_t num_decode_rows, int64_t num_prefill,
                                                 int64_t chunk_blocks) {
  if (num_q_tokens <= 0 || num_decode_rows < 0 || num_prefill < 0 ||
      num_decode_rows > num_q_tokens || num_kv_heads <= 0 || num_heads <= 0 ||
      num_heads % num_kv_heads != 0)
    return 0;
  return make_plan(num_decode_rows, num_prefill, num_q_tokens - num_decode_rows, chunk_blocks,
                   num_heads, num_kv_heads, page_size * max_blocks_per_seq)
      .bytes;
}

extern "C" int kvc_varlen_fp4(
    const void* q, int64_t q_stride_t, int64_t q_stride_h, int64_t num_q_tokens,
    int64_t num_heads, const uint8_t* k_cache, const uint8_t* v_cache, const uint8_t* k_scale,
    const uint8_t* v_scale, int64_t num_cache_blocks, int64_t page_size, int64_t num_kv_heads,
    int64_t head_dim, const int32_t* block_tables, int64_t bt_stride, int64_t max_blocks_per_seq,
    int64_t num_decode_rows, const int32_t* decode_context_lens, int64_t num_prefill,
    int64_t chunk_blocks, const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, float scale,
    void* out, int64_t out_stride_t, int64_t out_stride_h, void* workspace,
    size_t workspace_bytes, kvc_stream_t stream) {
  clear_error();
  KVC_REQUIRE(num_decode_rows >= 0 && num_decode_rows <= num_q_tokens, KVC_ERR_VALUE,
              "varlen_fp4: more decode rows than query rows");
  return run_rows("varlen_fp4", nullptr, q, q_stride_t, q_stride_h, num_heads, k_cache, v_cache,
                  k_scale, v_scale, num_cache_blocks, page_size, num_kv_heads, head_dim,
                  block_tables, bt_stride, max_blocks_per_seq, num_decode_rows,
                  decode_context_lens, num_prefill, num_q_tokens - num_decode_rows, chunk_blocks,
                  cu_seqlens_q, cu_seqlens_k, scale, out, out_stride_t, out_stride_h, workspace,
                  workspace_bytes, stream);
}

extern "C" int64_t kvc_varlen_fp4_blocks(const int32_t* cu_seqlens_q_host,
                                         const int32_t* cu_seqlens_k_host, int64_t num_prefill,
                                         int64_t num_heads, int64_t num_kv_heads,
                                         int64_t page_size, int64_t max_blocks_per_seq,
                                         int64_t num_decode_rows) {
  if (num_prefill <= 0 || num_kv_heads <= 0 || num_heads <= 0 || num_heads % num_kv_heads != 0 ||
      cu_seqlens_q_host == nullptr || cu_seqlens_k_host == nullptr)
    return 0;
  const int64_t group = num_heads / num_kv_heads;
  int64_t blocks = 0, longest = 0;
  double products = 0, all_keys = 0, pairs = 0;
  for (int64_t i = 0; i < num_prefill; ++i) {
    auto length = [&](const int32_t* cu) {
      return std::max<int64_t>(0, int64_t(cu[i + 1]) - cu[i]);
    };
    const int64_t n = length(cu_seqlens_q_host), m = length(cu_seqlens_k_host);
    const int64_t b = (n * group + 15) / 16;
    blocks += b;
    longest = std::max(longest, m);
    products += double(b) * double(m);
    all_keys += double(m);
    pairs += double(n) * double(std::max<int64_t>(0, m - n)) + double(n) * double(n) / 2;
  }
  if (blocks == 0) return 0;
  const Plan pl = make_plan(num_decode_rows, num_prefill, cu_seqlens_q_host[num_prefill], blocks,
                            num_heads, num_kv_heads, page_size * max_blocks_per_seq);
  const double heads_of = double(blocks) * double(num_kv_heads);
  const double items = std::ceil(heads_of / pl.heads_per_wg);  // (of a whole plan)
  const double here =
      pl.whole ? std::ceil(items / cu_count()) *
                     (6 + 2.2 * double(longest) * pl.heads_per_wg / 512)
               : 12 + 6 * std::min(1., heads_of / 128) +
                     products * double(num_kv_heads) / 64 * 0.9e-3;
  // Gathered: three launches, the keys written and read once more, the products at the
  // long chunks' rate; and the decode rows in a call of their own.  (Of 371 shapes, 1 to
  // 8 chunks of 4 to 512 tokens over up to 32768 keys, five take the form that is over 10 %
  // slower, 25 % at worst.)
  const double gathered = (longest <= 64 ? 13 : 22) + 3e-4 * all_keys * double(num_kv_heads) +
                          0.38e-6 * pairs * double(num_heads) + (num_decode_rows > 0 ? 12 : 0);
  return here <= gathered ? blocks : 0;
}
