// The 4-bit KV cache: quantise on append, dequantising reads, paged decode
// attention (gfx950; the encoding is in kvc_fp4.h).
//
// Decode: out[b, h] = sum_j softmax_j(scale q[b, h].k_j) v_j over the row's first
// context_lens[b] keys, 0 for a row without keys.
//
// A wave attends tiles of 64 keys of one kv head, whose G query heads are the
// columns of S^T = K Q^T.  A lane's 16 bytes of a K row are one run of 32 dims, so
// it needs one power and converts straight to the MFMA's operand; the dims come
// in that order, and Q's operand is read in the same.  S^T leaves a lane the 16
// keys of its own column that P's operand of O^T = V^T P^T takes, so weights
// never move between lanes.  V is transposed by LDS reads of 4-bit elements and
// converted with power 1: its powers differ by key, the summed index, so they
// multiply the weights instead, once for each run of 32 channels (a power of two
// times a bf16 weight is exact).  Sums are formed of the rounded weights, so the
// weights add up to the sum that divides them; logits, sums and O are fp32.
//
// Every wave streams its own tiles through its own LDS slots (two of 8.5 KiB,
// direct-to-LDS loads a tile ahead, no workgroup barrier); waves differ in kv
// head and in tile phase.  Bound by HBM reads for batches, by the chain of launch,
// lengths, table, tiles and merge for single rows.
#include <algorithm>
#include <atomic>

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
// (16 bytes) a lane; four lanes share a run.  Bound by HBM for prompts, by the
// launch and two dependent reads (slot, row) for a decode step.
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
// Dequantising reads: 16 lanes a row, four bytes of codes in, 16 bytes out.
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
  *reinterpret_cast<u32x4_t*>(out_k + row * kD + lane16 * 8) = k;
  *reinterpret_cast<u32x4_t*>(out_v + row * kD + lane16 * 8) = v;
}

// ---------------------------------------------------------------------------
// Paged decode.
// ---------------------------------------------------------------------------
constexpr int kWaves = 8;
constexpr int kTile = 64;                       // keys
constexpr int kCodeBytes = kTile * kFp4RowBytes;  // of K or V, 4 KiB
constexpr int kPowerBytes = kTile * kFp4Powers;   // 256
constexpr int kVAt = kCodeBytes, kKsAt = 2 * kCodeBytes, kVsAt = kKsAt + kPowerBytes;
constexpr int kSlotBytes = kVsAt + kPowerBytes;  // 8.5 KiB
constexpr int kSlots = 2;
constexpr int kLoads = 12;  // of a tile: K and V in four each, powers in two each
constexpr float kLowest = -3.402823466e38f;
constexpr float kSlack = 8.f;  // binades that a score may pass the running reference by
constexpr int kStateBytes = 8 * 64 * 16 + 64 * 8;  // a wave's O and (reference, sum)
static_assert(kStateBytes <= kSlots * kSlotBytes);

struct Fp4Params {
  const uint16_t* q;
  int64_t q_sb, q_sh;
  uint16_t* out;
  int64_t o_sb, o_sh;
  const uint8_t* k;
  const uint8_t* v;
  const uint8_t* ks;
  const uint8_t* vs;
  const int32_t* tables;
  int64_t bt_stride;
  const int32_t* lens;
  int max_blocks, num_blocks, page;
  int page_halves;         // page / 32
  float page_halves_rcp;
  int batch, kv_heads, group;
  int col_blocks;          // of 16 query heads, of a kv head's
  int heads_per_wg;        // kv heads of a workgroup
  int groups;              // workgroup items of a row: kv head groups x col_blocks
  int cols;                // columns kept of a partial: min(16, group)
  int min_share;
  int whole;               // one workgroup an item, no partials
  float c2;                // scale log2(e)
  int2* rec;               // of each item: first and last share
  float* part_o;
  float2* part_ml;
};

// Keys of row b that the tables can hold; steps of a row (a step is one tile of
// every phase), 1 for a row without keys: it writes zeros.
__device__ __forceinline__ int keys_of(const Fp4Params& p, int len) {
  const int64_t most = int64_t(p.max_blocks) * p.page;
  return int(min(int64_t(max(len, 0)), most));
}
__device__ __forceinline__ int steps_of(int keys, int step_keys) {
  return max(1, (keys + step_keys - 1) / step_keys);
}

__device__ __forceinline__ void dma_dword(const i32x4_t& rsrc, int voff, uint32_t lds) {
  uint32_t saved;
  asm volatile(
      "s_mov_b32 %0, m0\n\t"
      "s_mov_b32 m0, %2\n\t"
      "s_nop 0\n\t"
      "buffer_load_dword %1, %3, 0 offen nt lds\n\t"
      "s_mov_b32 m0, %0"
      : "=&s"(saved)
      : "v"(voff), "s"(lds), "s"(rsrc)
      : "memory");
}

template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

struct Carry {  // a wave's running softmax and output, column lane & 15
  f32x4_t o[8];  // channels 16 cb + 4 (lane >> 4) ..
  float m, l;
};

// One tile in `slot`: keys j0 .. j0 + 63 of a row of n keys.
__device__ __forceinline__ void attend_tile(const char* slot, const u32x4_t (&q)[4], Carry& c,
                                            int j0, int n, int lm, int lg, float c2) {
  f32x4_t s[4];
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    const u32x4_t w =
        *reinterpret_cast<const u32x4_t*>(slot + 1024 * x + 64 * lm + 16 * (lg ^ (lm >> 2)));
    const int key = 32 * (x >> 1) + 8 * (lm >> 2) + 4 * (x & 1) + (lm & 3);
    const float power =
        power_f32(*reinterpret_cast<const uint8_t*>(slot + kKsAt + 4 * key + lg));
    s[x] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int d = 0; d < 4; ++d) s[x] = mfma_bf16(dequant_fp4x8(w[d], power), q[d], s[x]);
  }
  // The lane's keys: 32 h + 8 lg + j for h = 0, 1 and j = 0 .. 7.
  u32x4_t pw[2][2];
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int i = 0; i < 2; ++i)
      pw[h][i] = *reinterpret_cast<const u32x4_t*>(slot + kVsAt + 4 * (32 * h + 8 * lg + 4 * i));
  float y[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) y[e] = s[e >> 2][e & 3] * c2;
  if (j0 + kTile > n) {
    // (what lies behind the row's keys may hold anything: weight 0, power 1)
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const bool seen = j0 + 32 * (e >> 3) + 8 * lg + (e & 7) < n;
      y[e] = seen ? y[e] : -INFINITY;
      const uint32_t word = pw[e >> 3][(e >> 2) & 1][e & 3];
      pw[e >> 3][(e >> 2) & 1][e & 3] = seen ? word : 0x7f7f7f7fu;
    }
  }
  float top = y[0];
#pragma unroll
  for (int e = 1; e < 16; ++e) top = fmaxf(top, y[e]);
  // The reference moves only when a score passes it by 2^kSlack.
  if (__builtin_amdgcn_ballot_w64(top > c.m + kSlack) != 0) {
    const float next = fmaxf(c.m, rows4_max(top));
    const float a = __builtin_amdgcn_exp2f(c.m - next);
    c.m = next;
    c.l *= a;
#pragma unroll
    for (int cb = 0; cb < 8; ++cb) c.o[cb] *= a;
  }
  float w[16];
#pragma unroll
  for (int e = 0; e < 16; e += 2) {
    const uint32_t r = pack_bf16x2_fast(__builtin_amdgcn_exp2f(y[e] - c.m),
                                        __builtin_amdgcn_exp2f(y[e + 1] - c.m));
    w[e] = __uint_as_float(r << 16);
    w[e + 1] = __uint_as_float(r & 0xffff0000u);
    c.l += w[e] + w[e + 1];
  }
  // The row of V that the lane points the transposed reads at.
  const int vkey = lm < 8 ? 8 * lg + lm : 24 + 8 * lg + lm;
  const int vswz = ((vkey >> 2) & 1) + 2 * (vkey >> 5);
  const char* vrow = slot + kVAt + 64 * vkey;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    u32x4_t pb[2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int e = 8 * h + 2 * i;
        const uint32_t s0 = ((pw[h][i >> 1][(2 * i) & 3] >> (8 * g)) & 0xffu) << 23;
        const uint32_t s1 = ((pw[h][i >> 1][(2 * i + 1) & 3] >> (8 * g)) & 0xffu) << 23;
        pb[h][i] = perm(__float_as_uint(w[e + 1] * __uint_as_float(s1)),
                        __float_as_uint(w[e] * __uint_as_float(s0)), kPermHiHi);
      }
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int cb = 2 * g + x;
      typedef int v2i __attribute__((ext_vector_type(2)));
      const v2i t = __builtin_amdgcn_ds_read_tr4_b64_v2i32(
          (__attribute__((address_space(3))) v2i*)((__attribute__((address_space(3))) char*)(
              vrow + 16 * (g ^ vswz) + 8 * x)));
      c.o[cb] = mfma_bf16(dequant_fp4x8(uint32_t(t[0]), 1.f), pb[0], c.o[cb]);
      c.o[cb] = mfma_bf16(dequant_fp4x8(uint32_t(t[1]), 1.f), pb[1], c.o[cb]);
    }
  }
}

__global__ void __launch_bounds__(64 * kWaves, 2) fp4_decode_kernel(Fp4Params p) {
  extern __shared__ __align__(1024) char smem[];
  const int lane = threadIdx.x & 63, wave = uniform(int(threadIdx.x >> 6));
  const int lm = lane & 15, lg = lane >> 4;
  // Consecutive shares on one XCD (workgroup b runs on XCD b mod 8).
  const int grid = gridDim.x;
  const int share = grid % 8 == 0 ? (blockIdx.x % 8) * (grid / 8) + blockIdx.x / 8 : blockIdx.x;
  touch_kernel_args(int(sizeof(Fp4Params)));
  const int hs = wave % p.heads_per_wg, phase = wave / p.heads_per_wg;
  const int phases = kWaves / p.heads_per_wg;
  const int step_keys = phases * kTile;

  // The share's place: row, item of the row, step of the item.
  int row = 0, item = 0, step = 0;
  int64_t pos = 0, end = 1, size = 1;
  if (p.whole) {
    row = share / p.groups;
    item = share - row * p.groups;
  } else {
    int64_t total = 0;
    for (int r0 = 0; r0 < p.batch; r0 += 64) {
      const int r = r0 + lane;
      const int n = r < p.batch ? steps_of(keys_of(p, p.lens[r]), step_keys) : 0;
      total += int64_t(wave_sum(n)) * p.groups;
    }
    size = max(int64_t(p.min_share), (total + grid - 1) / grid);
    pos = share * size;
    end = min(total, pos + size);
    if (pos >= end) return;
    int64_t before = 0;
    for (int r0 = 0; r0 < p.batch; r0 += 64) {
      const int r = r0 + lane;
      const int n = r < p.batch ? steps_of(keys_of(p, p.lens[r]), step_keys) : 0;
      const int incl = wave_scan_add(n);
      const int64_t all = int64_t(__builtin_amdgcn_readlane(incl, 63)) * p.groups;
      if (pos < before + all) {
        const uint64_t past =
            __builtin_amdgcn_ballot_w64(before + int64_t(incl) * p.groups > pos);
        const int at = __builtin_ctzll(past);
        row = r0 + at;
        const int steps = __builtin_amdgcn_readlane(n, at);
        const int64_t in =
            pos - before - int64_t(__builtin_amdgcn_readlane(incl, at) - steps) * p.groups;
        item = int(in / steps);
        step = int(in - int64_t(item) * steps);
        break;
      }
      before += all;
    }
  }

  const uint32_t lds0 = lds_addr(smem) + wave * (kSlots * kSlotBytes);
  const char* slot0 = smem + wave * (kSlots * kSlotBytes);
  // Offsets of the lane's 16 bytes in a tile's half of 32 keys.  K's loads fill
  // LDS in the MFMA's row order, V's in key order; four lanes read a row, its
  // quarters turned so that the operand reads meet no bank twice.
  const int row_bytes = p.kv_heads * kFp4RowBytes;
  int koff[2], voff[4];
  {
    const int r = lane >> 2;
#pragma unroll
    for (int x = 0; x < 2; ++x)
      koff[x] = (8 * (r >> 2) + 4 * x + (r & 3)) * row_bytes + 16 * ((lane & 3) ^ (r >> 2));
#pragma unroll
    for (int x = 0; x < 4; ++x)
      voff[x] = (16 * (x & 1) + r) * row_bytes +
                16 * ((lane & 3) ^ (((lane >> 4) & 1) + 2 * (x >> 1)));
  }
  const int soff = (lane & 31) * p.kv_heads * kFp4Powers;

  while (true) {
    const int keys = keys_of(p, table_entry(p.lens, row));
    const int steps = steps_of(keys, step_keys);
    const int seg0 = step;
    const int seg1 = p.whole ? steps : int(min(int64_t(steps), step + (end - pos)));
    const int head = (item / p.col_blocks) * p.heads_per_wg + hs;
    const int col0 = (item % p.col_blocks) * 16;
    if (!p.whole && seg0 == 0 && threadIdx.x == 0)
      p.rec[int64_t(row) * p.groups + item] = int2{share, int((pos + steps - 1) / size)};

    const int col = min(col0 + lm, p.group - 1);
    const uint16_t* qp = p.q + row * p.q_sb + int64_t(head * p.group + col) * p.q_sh + 32 * lg;
    u32x4_t q[4];
#pragma unroll
    for (int d = 0; d < 4; ++d) q[d] = *reinterpret_cast<const u32x4_t*>(qp + 8 * d);
    Carry c;
#pragma unroll
    for (int cb = 0; cb < 8; ++cb) c.o[cb] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    c.m = kLowest;
    c.l = 0.f;

    // Tiles of this wave: t = seg0 phases + phase, then every phases-th.
    const int32_t* table = p.tables + row * p.bt_stride;
    const int t_end = min(seg1 * phases, (keys + kTile - 1) / kTile);
    int t = seg0 * phases + phase;
    int pages0 = -64, pages = -1;  // the lane's table entry, of page pages0 + lane
    auto issue = [&](int tile, uint32_t lds) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int half = 2 * tile + h;
        const int pg = uniform(div_small(half, p.page_halves, p.page_halves_rcp));
        if (pg >= pages0 + 64) {
          pages0 = pg;
          pages = pg + lane < p.max_blocks ? table[pg + lane] : -1;
        }
        const int blk = __builtin_amdgcn_readlane(pages, pg - pages0);
        const bool there = half * 32 < keys && blk >= 0 && blk < p.num_blocks;
        const int64_t at = there ? (int64_t(blk) * p.page + (half - pg * p.page_halves) * 32) *
                                           p.kv_heads + head : 0;
        const int codes = there ? 31 * row_bytes + kFp4RowBytes : 0;
        const int powers = there ? (31 * p.kv_heads + 1) * kFp4Powers : 0;
        const i32x4_t kr = raw_rsrc(p.k + at * kFp4RowBytes, codes);
        const i32x4_t vr = raw_rsrc(p.v + at * kFp4RowBytes, codes);
        const i32x4_t ksr = raw_rsrc(p.ks + at * kFp4Powers, powers);
        const i32x4_t vsr = raw_rsrc(p.vs + at * kFp4Powers, powers);
        if ((lane >> 5) == h) {
          dma_dword(ksr, soff, lds + kKsAt);
          dma_dword(vsr, soff, lds + kVsAt);
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          dma_to_lds(kr, koff[x], lds + 1024 * (2 * h + x));
          dma_to_lds(vr, voff[2 * h + x], lds + kVAt + 1024 * (2 * h + x));
        }
      }
    };
    int buf = 0;
    if (t < t_end) issue(t, lds0);
    // The queries are waited for with the first tile on its way.
#pragma unroll
    for (int d = 0; d < 4; ++d) asm volatile("" : "+v"(q[d]));
    for (; t < t_end; t += phases) {
      smem_drain();  // the other slot's reads are done
      if (t + phases < t_end) {
        issue(t + phases, lds0 + (buf ^ 1) * kSlotBytes);
        wait_loads<kLoads>();
      } else {
        wait_loads<0>();
      }
      attend_tile(slot0 + buf * kSlotBytes, q, c, t * kTile, keys, lm, lg, p.c2);
      buf ^= 1;
    }
    c.l = rows4_sum(c.l);

    // Channels 16 cb .. + 15 of the wave's columns: the result, or a partial in
    // slot 2 share + 1 (the piece that begins its item), else 2 share.
    const bool done = seg0 == 0 && seg1 == steps;
    const int64_t part = ((int64_t(2) * share + (seg0 == 0 ? 1 : 0)) * p.heads_per_wg + hs) *
                             p.cols + lm;
    auto emit = [&](int cb, const f32x4_t& o, float m, float l) {
      if (col0 + lm >= p.group) return;
      if (done) {
        const float inv = l != 0.f ? 1.f / l : 0.f;
        uint16_t* dst = p.out + row * p.o_sb + int64_t(head * p.group + col0 + lm) * p.o_sh +
                        16 * cb + 4 * lg;
        *reinterpret_cast<u32x2_t*>(dst) = u32x2_t{pack_bf16x2_fast(o[0] * inv, o[1] * inv),
                                                   pack_bf16x2_fast(o[2] * inv, o[3] * inv)};
      } else {
        *reinterpret_cast<f32x4_t*>(p.part_o + part * kD + 16 * cb + 4 * lg) = o;
        if (cb == 0 && lg == 0) p.part_ml[part] = float2{m, l};
      }
    };
    {
      // Phases joined through the waves' own slots: a phase makes 8 / phases of
      // the channel blocks of its head's columns.
      char* own = smem + wave * (kSlots * kSlotBytes);
      smem_drain();
#pragma unroll
      for (int cb = 0; cb < 8; ++cb)
        *reinterpret_cast<f32x4_t*>(own + cb * 1024 + lane * 16) = c.o[cb];
      *reinterpret_cast<float2*>(own + 8192 + lane * 8) = float2{c.m, c.l};
      pf_barrier();
      const char* first = smem + hs * (kSlots * kSlotBytes);
      const int apart = p.heads_per_wg * (kSlots * kSlotBytes);
      float top = kLowest, l = 0.f;
      for (int f = 0; f < phases; ++f)
        top = fmaxf(top, reinterpret_cast<const float2*>(first + f * apart + 8192)[lane].x);
      const int each = 8 / phases;
      f32x4_t o[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
      for (int f = 0; f < phases; ++f) {
        const float2 ml = reinterpret_cast<const float2*>(first + f * apart + 8192)[lane];
        const float b = __builtin_amdgcn_exp2f(ml.x - top);
        l += ml.y * b;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (i < each)
            o[i] += *reinterpret_cast<const f32x4_t*>(first + f * apart +
                                                      (phase * each + i) * 1024 + lane * 16) * b;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i < each) emit(phase * each + i, o[i], top, l);
      pf_barrier();
    }

    pos += seg1 - seg0;
    if (p.whole || pos >= end) break;
    step = 0;
    if (++item < p.groups) continue;
    item = 0;
    ++row;
  }
}

// ---------------------------------------------------------------------------
// Join the partials of items cut between shares: a workgroup per item and
// column, eight slices of 32 lanes over its pieces.
// ---------------------------------------------------------------------------
constexpr int kSlices = 8;
constexpr int kAhead = 4;  // pieces of a slice whose loads are in flight together
__global__ void __launch_bounds__(32 * kSlices) fp4_merge_kernel(Fp4Params p) {
  __shared__ f32x4_t so[kSlices][32];
  __shared__ float2 sml[kSlices];
  const int item = blockIdx.x;
  const int2 r = p.rec[item];
  if (r.x >= r.y) return;
  const int row = item / p.groups, in = item - row * p.groups;
  const int hs = blockIdx.y / p.cols, col = blockIdx.y - hs * p.cols;
  const int head = (in / p.col_blocks) * p.heads_per_wg + hs;
  const int qh = (in % p.col_blocks) * 16 + col;
  if (qh >= p.group) return;
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
  const int64_t at = int64_t(hs) * p.cols + col, cols = int64_t(p.heads_per_wg) * p.cols;
  float top = kLowest, l = 0.f;
  f32x4_t o = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = r.x + slice; s0 <= r.y; s0 += kSlices * kAhead) {
    float2 ml[kAhead];
    f32x4_t part[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int s = min(s0 + kSlices * i, r.y);
      const int64_t c = (int64_t(2) * s + (s == r.x)) * cols + at;
      ml[i] = p.part_ml[c];
      part[i] = reinterpret_cast<const f32x4_t*>(p.part_o + c * kD)[lane];
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (s0 + kSlices * i > r.y) continue;
      const float next = fmaxf(top, ml[i].x);
      const float a = __builtin_amdgcn_exp2f(top - next);
      const float b = __builtin_amdgcn_exp2f(ml[i].x - next);
      top = next;
      l = l * a + ml[i].y * b;
      o = o * a + part[i] * b;
    }
  }
  so[slice][lane] = o;
  if (lane == 0) sml[slice] = float2{top, l};
  __syncthreads();
  if (slice != 0) return;
#pragma unroll
  for (int i = 1; i < kSlices; ++i) top = fmaxf(top, sml[i].x);
  l = 0.f;
  o = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < kSlices; ++i) {
    const float b = __builtin_amdgcn_exp2f(sml[i].x - top);
    l += sml[i].y * b;
    o += so[i][lane] * b;
  }
  const float inv = l != 0.f ? 1.f / l : 0.f;
  uint16_t* dst = p.out + row * p.o_sb + int64_t(head * p.group + qh) * p.o_sh + 4 * lane;
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
  int heads_per_wg, col_blocks, groups, cols, grid, min_share, whole;
  size_t rec_at, ml_at, o_at, bytes;
};

size_t up256(size_t n) { return (n + 255) & ~size_t(255); }

Plan make_plan(int64_t batch, int64_t heads, int64_t kv_heads, int64_t most_keys) {
  Plan pl{};
  const int64_t group = heads / kv_heads;
  pl.col_blocks = int((group + 15) / 16);
  pl.cols = int(std::min<int64_t>(group, 16));
  const int cus = cu_count();
  const int64_t tiles = (most_keys + kTile - 1) / kTile;
  // Waves of a workgroup over kv heads, the rest over tile phases.
  int hpw = 4;
  while (hpw > 1 && kv_heads % hpw != 0) hpw >>= 1;
  pl.whole = tiles <= 16;
  if (pl.whole) hpw = 1;
  pl.heads_per_wg = hpw;
  pl.groups = int(kv_heads / hpw * pl.col_blocks);
  pl.min_share = 1;
  const int64_t items = batch * pl.groups;
  pl.grid = int(pl.whole ? items : cus);
  size_t at = 0;
  if (!pl.whole) {
    pl.rec_at = 0;
    at = up256(size_t(items) * sizeof(int2));
    pl.ml_at = at;
    const size_t cols = size_t(2) * pl.grid * hpw * pl.cols;
    at = up256(at + cols * sizeof(float2));
    pl.o_at = at;
    at = up256(at + cols * kD * sizeof(float));
  }
  pl.bytes = at;
  return pl;
}

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
  KVC_REQUIRE(reinterpret_cast<uintptr_t>(k) % 16 == 0 && reinterpret_cast<uintptr_t>(v) % 16 == 0 &&
                  reinterpret_cast<uintptr_t>(ks) % 4 == 0 &&
                  reinterpret_cast<uintptr_t>(vs) % 4 == 0,
              KVC_ERR_ASSERT, "%s: pools must be 16-byte aligned, scales 4-byte", what);
  return KVC_OK;
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
  int rc = check_rows("store_fp4", key, key_stride_n, key_stride_h, value, value_stride_n,
                      value_stride_h, num_tokens, num_kv_heads, head_dim, slot_index_bytes);
  if (rc != KVC_OK) return rc;
  if (num_tokens == 0) return KVC_OK;
  rc = check_pool("store_fp4", k_cache, v_cache, k_scale, v_scale);
  if (rc != KVC_OK) return rc;
  KVC_REQUIRE(key != nullptr && value != nullptr && slot_mapping != nullptr, KVC_ERR_VALUE,
              "store_fp4: null rows or slots");
  const int64_t rows = num_tokens * num_kv_heads;
  const dim3 grid(unsigned((rows + kRowsPerBlock - 1) / kRowsPerBlock));
  auto kern = slot_index_bytes == 8 ? store_fp4_kernel<8> : store_fp4_kernel<4>;
  kern<<<grid, kThreads, 0, as_stream(stream)>>>(
      static_cast<const uint16_t*>(key), key_stride_n, key_stride_h,
      static_cast<const uint16_t*>(value), value_stride_n, value_stride_h, k_cache, v_cache,
      k_scale, v_scale, num_slots, slot_mapping, num_tokens, int(num_kv_heads));
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

extern "C" size_t kvc_paged_decode_fp4_workspace_bytes(int64_t batch, int64_t num_heads,
                                                       int64_t num_kv_heads, int64_t page_size,
                                                       int64_t max_blocks_per_seq) {
  if (batch <= 0 || num_kv_heads <= 0 || num_heads <= 0 || num_heads % num_kv_heads != 0) return 0;
  return make_plan(batch, num_heads, num_kv_heads, page_size * max_blocks_per_seq).bytes;
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
  KVC_REQUIRE(head_dim == kD, KVC_ERR_VALUE, "paged_decode_fp4: head_dim must be 128 (got %lld)",
              (long long)head_dim);
  KVC_REQUIRE(batch >= 0 && num_kv_heads > 0 && num_heads > 0 && num_heads % num_kv_heads == 0,
              KVC_ERR_VALUE, "paged_decode_fp4: num_heads must be a multiple of num_kv_heads");
  KVC_REQUIRE(page_size > 0 && page_size % 32 == 0, KVC_ERR_VALUE,
              "paged_decode_fp4: page_size must be a multiple of 32 (got %lld)",
              (long long)page_size);
  // (row offsets inside a half tile and key counts are 32-bit; div_small's range)
  KVC_REQUIRE(num_kv_heads <= 4096 && num_heads <= 65536 && max_blocks_per_seq >= 0 &&
                  num_cache_blocks >= 0 && num_cache_blocks < (int64_t(1) << 31) &&
                  page_size <= (1 << 20) && page_size * max_blocks_per_seq <= (int64_t(1) << 26),
              KVC_ERR_VALUE, "paged_decode_fp4: shape out of range (tables of up to 2^26 keys)");
  if (batch == 0) return KVC_OK;
  const int rc = check_pool("paged_decode_fp4", k_cache, v_cache, k_scale, v_scale);
  if (rc != KVC_OK) return rc;
  KVC_REQUIRE(q != nullptr && out != nullptr && context_lens != nullptr &&
                  (block_tables != nullptr || max_blocks_per_seq == 0),
              KVC_ERR_VALUE, "paged_decode_fp4: null pointer");
  KVC_REQUIRE(reinterpret_cast<uintptr_t>(q) % 16 == 0 && q_stride_b % 8 == 0 &&
                  q_stride_h % 8 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0 &&
                  out_stride_b % 8 == 0 && out_stride_h % 8 == 0,
              KVC_ERR_ASSERT, "paged_decode_fp4: q/out rows must be 16-byte aligned");
  const Plan pl = make_plan(batch, num_heads, num_kv_heads, page_size * max_blocks_per_seq);
  const int64_t items = batch * pl.groups;
  KVC_REQUIRE(items < (int64_t(1) << 30), KVC_ERR_VALUE, "paged_decode_fp4: batch too large");
  KVC_REQUIRE(pl.bytes == 0 || (workspace != nullptr && workspace_bytes >= pl.bytes),
              KVC_ERR_WORKSPACE, "paged_decode_fp4: workspace of %zu bytes needed", pl.bytes);
  KVC_REQUIRE(pl.bytes == 0 || reinterpret_cast<uintptr_t>(workspace) % 16 == 0, KVC_ERR_ASSERT,
              "paged_decode_fp4: workspace must be 16-byte aligned");
  Fp4Params p{};
  p.q = static_cast<const uint16_t*>(q);
  p.q_sb = q_stride_b;
  p.q_sh = q_stride_h;
  p.out = static_cast<uint16_t*>(out);
  p.o_sb = out_stride_b;
  p.o_sh = out_stride_h;
  p.k = k_cache;
  p.v = v_cache;
  p.ks = k_scale;
  p.vs = v_scale;
  p.tables = block_tables;
  p.bt_stride = bt_stride;
  p.lens = context_lens;
  p.max_blocks = int(max_blocks_per_seq);
  p.num_blocks = int(num_cache_blocks);
  p.page = int(page_size);
  p.page_halves = int(page_size / 32);
  p.page_halves_rcp = 1.f / float(p.page_halves);
  p.batch = int(batch);
  p.kv_heads = int(num_kv_heads);
  p.group = int(num_heads / num_kv_heads);
  p.col_blocks = pl.col_blocks;
  p.heads_per_wg = pl.heads_per_wg;
  p.groups = pl.groups;
  p.cols = pl.cols;
  p.min_share = pl.min_share;
  p.whole = pl.whole;
  p.c2 = scale * kLog2e;
  char* ws = static_cast<char*>(workspace);
  p.rec = reinterpret_cast<int2*>(ws + pl.rec_at);
  p.part_ml = reinterpret_cast<float2*>(ws + pl.ml_at);
  p.part_o = reinterpret_cast<float*>(ws + pl.o_at);
  constexpr int kLds = kWaves * kSlots * kSlotBytes;
  hipStream_t st = as_stream(stream);
  static std::atomic<uint64_t> ready{0};  // devices whose LDS limit is set
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  const uint64_t bit = uint64_t(1) << (dev & 63);
  if (e == hipSuccess && !(ready.load(std::memory_order_relaxed) & bit)) {
    e = hipFuncSetAttribute(reinterpret_cast<const void*>(&fp4_decode_kernel),
                            hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
    if (e == hipSuccess) ready.fetch_or(bit, std::memory_order_relaxed);
  }
  KVC_REQUIRE(e == hipSuccess, KVC_ERR_RUNTIME, "paged_decode_fp4: LDS limit: %s",
              hipGetErrorString(e));
  fp4_decode_kernel<<<pl.grid, 64 * kWaves, kLds, st>>>(p);
  if (!pl.whole)
    fp4_merge_kernel<<<dim3(unsigned(items), unsigned(pl.heads_per_wg * pl.cols)), 32 * kSlices, 0,
                       st>>>(p);
  return check_launch("paged_decode_fp4");
}
