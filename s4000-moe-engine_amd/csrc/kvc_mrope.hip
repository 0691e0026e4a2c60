// Fused q/k RMSNorm + rotary embedding over several position axes + KV append
// for gfx950: the step in front of the paged cache for prompts whose tokens
// have a time, a height and a width (text: all three alike).
//
//   xf = float(x);  r = 1 / sqrt(sum(xf^2) / 128 + eps);  y = xf r w
//   out_i = y_i c - y_{i+64} s;  out_{i+64} = y_{i+64} c + y_i s
//   c, s = cos, sin of pair i at position[axis(i)]
// in fp32 throughout, rounded to bf16 once, at the end (the single-axis step
// rounds after the norm and after its weight too, as the engine's torch ops
// do; nothing here has to match those).
//
// A workgroup owns TPW tokens.  Its threads first bring each token's 64
// (cos, sin) pairs, every pair from its own axis' table row, into LDS, so the
// layout of the axes (runs or dealt out in turn) costs nothing in the row
// loop; the rows' own loads are in flight meanwhile.  Then 8-lane groups take
// the token's head rows: lane j holds dims 8 j .. 8 j + 7 and 64 + 8 j ..,
// 16 bytes each, so a rotation pair never leaves its lane and the sum of
// squares is three DPP moves.  Bound by HBM: each row is read and written
// once; 16384 tokens of 32 / 4 heads, 344 MB, take 67 us (5.1 TB/s; torch's
// copy of 2 GiB 4.9), 58 where a part of them is cached still.  A decode step of
// 64 tokens takes 4 us, the launch and three dependent reads (position, table,
// row).
#include "kvc_lds.h"

namespace kvc {
namespace {

constexpr int kD = 128;
constexpr int kPairs = kD / 2;
constexpr int kThreads = 256;
constexpr int kMaxAxes = 4;

struct MropeArgs {
  const uint16_t* q;
  int64_t q_st, q_sh;
  const uint16_t* k;
  int64_t k_st, k_sh;
  const uint16_t* v;
  int64_t v_st, v_sh;
  const void* positions;  // [axes][tokens], rows pos_stride apart
  int64_t pos_stride;
  uint64_t axis_lo, axis_hi;  // bits of each pair's axis
  const uint16_t* q_w;        // bf16 [128] or null (no norm)
  const uint16_t* k_w;
  const float* cos_sin;  // fp32 [max_position, 128]
  int64_t max_position;
  float eps;
  uint16_t* q_out;
  int64_t qo_st, qo_sh;
  uint16_t* k_out;  // may be null
  int64_t ko_st, ko_sh;
  uint16_t* k_cache;  // [num_slots, KVH, 128] or null (no append)
  uint16_t* v_cache;
  int64_t num_slots;
  const void* slots;
  int64_t num_tokens;
  int num_heads, num_kv_heads;
};

// Sum over an 8-lane group: quad neighbours, then the other quad.
__device__ __forceinline__ float sum8(float x) {
  x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0xB1, 0xf, 0xf, false));
  x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x4E, 0xf, 0xf, false));
  x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x141, 0xf, 0xf, false));
  return x;
}

template <int TPW, int kRows, int kPosBytes, int kSlotBytes>
__global__ void __launch_bounds__(kThreads) qk_norm_mrope_store_kernel(MropeArgs a) {
  constexpr int kGroups = kThreads / 8 / TPW;  // 8-lane groups per token
  __shared__ __align__(16) float lds[TPW][kD];
  const int j = threadIdx.x & 7;
  const int tok = threadIdx.x / (kThreads / TPW);
  const int g = (threadIdx.x / 8) % kGroups;
  const int64_t n0 = int64_t(blockIdx.x) * TPW, n = n0 + tok;
  const bool live = n < a.num_tokens;
  const int rows = live ? a.num_heads + 2 * a.num_kv_heads : 0;

  // The positions of this thread's table entries, ahead of the rows' loads.
  constexpr int kEntries = TPW * kPairs;
  constexpr int kEach = (kEntries + kThreads - 1) / kThreads;
  int64_t pos[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int e = threadIdx.x + i * kThreads;
    const int64_t m = n0 + e / kPairs;
    const int pair = e % kPairs;
    const int axis = int((a.axis_lo >> pair) & 1u) | (int((a.axis_hi >> pair) & 1u) << 1);
    pos[i] = e < kEntries && m < a.num_tokens
                 ? load_index<kPosBytes>(a.positions, axis * a.pos_stride + m)
                 : 0;
  }
  int64_t sl = -1;
  if (a.k_cache != nullptr && live) {
    sl = wrap_slot(load_index<kSlotBytes>(a.slots, n), a.num_slots);
    if (sl >= a.num_slots) sl = -1;
  }

  bool staged = false;
  float c[8], s[8];
  for (int r0 = 0; r0 == 0 || r0 < rows; r0 += kGroups * kRows) {
    u32x4_t lo[kRows], hi[kRows];
#pragma unroll
    for (int u = 0; u < kRows; ++u) {
      const int r = r0 + g + kGroups * u;
      lo[u] = hi[u] = u32x4_t{0u, 0u, 0u, 0u};
      if (r >= rows) continue;
      const int kr = r - a.num_heads, vr = kr - a.num_kv_heads;
      const uint16_t* src = kr < 0   ? a.q + n * a.q_st + r * a.q_sh
                            : vr < 0 ? a.k + n * a.k_st + kr * a.k_sh
                                     : a.v + n * a.v_st + vr * a.v_sh;
      if (vr >= 0 && sl < 0) continue;
      lo[u] = *reinterpret_cast<const u32x4_t*>(src + 8 * j);
      hi[u] = *reinterpret_cast<const u32x4_t*>(src + kPairs + 8 * j);
    }
    if (!staged) {
      staged = true;
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const int e = threadIdx.x + i * kThreads;
        if (e < kEntries) {
          // A negative position wraps like a Python index; one still outside
          // the table gives NaN.
          const int64_t p = wrap_slot(pos[i], a.max_position);
          const bool ok = p >= 0 && p < a.max_position;
          const float* row = a.cos_sin + (ok ? p : 0) * kD + e % kPairs;
          const float cv = row[0], sv = row[kPairs];
          lds[e / kPairs][e % kPairs] = ok ? cv : __builtin_nanf("");
          lds[e / kPairs][kPairs + e % kPairs] = ok ? sv : __builtin_nanf("");
        }
      }
      pf_barrier();
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float4 cv = *reinterpret_cast<const float4*>(&lds[tok][8 * j + 4 * i]);
        const float4 sv = *reinterpret_cast<const float4*>(&lds[tok][kPairs + 8 * j + 4 * i]);
        c[4 * i] = cv.x, c[4 * i + 1] = cv.y, c[4 * i + 2] = cv.z, c[4 * i + 3] = cv.w;
        s[4 * i] = sv.x, s[4 * i + 1] = sv.y, s[4 * i + 2] = sv.z, s[4 * i + 3] = sv.w;
      }
    }
#pragma unroll
    for (int u = 0; u < kRows; ++u) {
      const int r = r0 + g + kGroups * u;
      if (r >= rows) continue;  // whole 8-lane groups skip together
      const int kr = r - a.num_heads, vr = kr - a.num_kv_heads;
      if (vr >= 0) {
        if (sl >= 0) {
          uint16_t* dst = a.v_cache + (sl * a.num_kv_heads + vr) * kD + 8 * j;
          *reinterpret_cast<u32x4_t*>(dst) = lo[u];
          *reinterpret_cast<u32x4_t*>(dst + kPairs) = hi[u];
        }
        continue;
      }
      float x1[8], x2[8];
      unpack8(lo[u], x1);
      unpack8(hi[u], x2);
      const uint16_t* w = kr < 0 ? a.q_w : a.k_w;
      if (w != nullptr) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss += x1[i] * x1[i] + x2[i] * x2[i];
        const float rinv = 1.f / __fsqrt_rn(sum8(ss) * (1.f / kD) + a.eps);
        float w1[8], w2[8];
        unpack8(*reinterpret_cast<const u32x4_t*>(w + 8 * j), w1);
        unpack8(*reinterpret_cast<const u32x4_t*>(w + kPairs + 8 * j), w2);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x1[i] = x1[i] * rinv * w1[i];
          x2[i] = x2[i] * rinv * w2[i];
        }
      }
      u32x4_t o1, o2;
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        o1[i / 2] = pack_bf16x2_fast(x1[i] * c[i] - x2[i] * s[i],
                                     x1[i + 1] * c[i + 1] - x2[i + 1] * s[i + 1]);
        o2[i / 2] = pack_bf16x2_fast(x2[i] * c[i] + x1[i] * s[i],
                                     x2[i + 1] * c[i + 1] + x1[i + 1] * s[i + 1]);
      }
      if (kr < 0) {
        // Past the caches: q_out is most of what is written, and pushed out of
        // them by itself before attention reads it.  Measured, 16384 tokens of
        // 32 / 4 heads, the same call again: 58 us so, 73 through the caches, 57
        // with the pool's rows past them too; with inputs from HBM 67 so, 72
        // through the caches.  Attention after it takes as long in all three.
        uint16_t* row = a.q_out + n * a.qo_st + r * a.qo_sh;
        __builtin_nontemporal_store(o1, reinterpret_cast<u32x4_t*>(row + 8 * j));
        __builtin_nontemporal_store(o2, reinterpret_cast<u32x4_t*>(row + kPairs + 8 * j));
        continue;
      }
      auto put = [&](uint16_t* row) {
        *reinterpret_cast<u32x4_t*>(row + 8 * j) = o1;
        *reinterpret_cast<u32x4_t*>(row + kPairs + 8 * j) = o2;
      };
      if (a.k_out != nullptr) put(a.k_out + n * a.ko_st + kr * a.ko_sh);
      if (sl >= 0) put(a.k_cache + (sl * a.num_kv_heads + kr) * kD);
    }
  }
}

template <int TPW, int kRows>
void launch(const MropeArgs& a, int pos_bytes, int slot_bytes, hipStream_t st) {
  const dim3 grid{unsigned((a.num_tokens + TPW - 1) / TPW)};
  if (pos_bytes == 8) {
    if (slot_bytes == 8)
      qk_norm_mrope_store_kernel<TPW, kRows, 8, 8><<<grid, kThreads, 0, st>>>(a);
    else
      qk_norm_mrope_store_kernel<TPW, kRows, 8, 4><<<grid, kThreads, 0, st>>>(a);
  } else {
    if (slot_bytes == 8)
      qk_norm_mrope_store_kernel<TPW, kRows, 4, 8><<<grid, kThreads, 0, st>>>(a);
    else
      qk_norm_mrope_store_kernel<TPW, kRows, 4, 4><<<grid, kThreads, 0, st>>>(a);
  }
}

bool rows16(const void* p, int64_t st, int64_t sh) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && st % 8 == 0 && sh % 8 == 0;
}

}  // namespace
}  // namespace kvc

using namespace kvc;

extern "C" int kvc_qk_norm_mrope_store(
    const void* q, int64_t q_stride_t, int64_t q_stride_h, const void* k, int64_t k_stride_t,
    int64_t k_stride_h, const void* v, int64_t v_stride_t, int64_t v_stride_h,
    int64_t num_tokens, int64_t num_heads, int64_t num_kv_heads, int64_t head_dim,
    const void* positions, int64_t position_stride, int position_index_bytes, int64_t num_axes,
    const int32_t* pair_axes_host, const void* q_norm_weight, const void* k_norm_weight, float eps,
    const float* cos_sin_cache, int64_t max_position, void* q_out, int64_t q_out_stride_t,
    int64_t q_out_stride_h, void* k_out, int64_t k_out_stride_t, int64_t k_out_stride_h,
    void* k_cache, void* v_cache, int64_t num_slots, const void* slot_mapping,
    int slot_index_bytes, kvc_stream_t stream) {
  clear_error();
  const char* what = "qk_norm_mrope_store";
  KVC_REQUIRE(head_dim == kD, KVC_ERR_VALUE, "%s: head_dim must be 128 (got %lld)", what,
              (long long)head_dim);
  KVC_REQUIRE(num_tokens >= 0 && num_tokens < (int64_t(1) << 31) && num_heads > 0 &&
                  num_kv_heads > 0 && num_heads < (1 << 20) && num_kv_heads < (1 << 20),
              KVC_ERR_VALUE, "%s: bad token or head counts", what);
  KVC_REQUIRE(num_axes >= 1 && num_axes <= kMaxAxes, KVC_ERR_VALUE, "%s: 1 to %d position axes",
              what, kMaxAxes);
  KVC_REQUIRE(pair_axes_host != nullptr, KVC_ERR_VALUE, "%s: missing pair_axes", what);
  KVC_REQUIRE(position_index_bytes == 4 || position_index_bytes == 8, KVC_ERR_VALUE,
              "%s: positions must be int32 or int64", what);
  MropeArgs a{};
  for (int i = 0; i < kPairs; ++i) {
    const int x = pair_axes_host[i];
    KVC_REQUIRE(x >= 0 && x < num_axes, KVC_ERR_VALUE, "%s: pair %d has axis %d of %lld", what, i,
                x, (long long)num_axes);
    a.axis_lo |= uint64_t(x & 1) << i;
    a.axis_hi |= uint64_t(x >> 1) << i;
  }
  if (num_tokens == 0) return KVC_OK;  // empty tensors may carry null pointers
  KVC_REQUIRE(q != nullptr && k != nullptr && q_out != nullptr && positions != nullptr &&
                  cos_sin_cache != nullptr && max_position > 0,
              KVC_ERR_VALUE, "%s: missing q, k, q_out, positions or cache", what);
  const bool cache = k_cache != nullptr || v_cache != nullptr;
  if (cache) {
    KVC_REQUIRE(k_cache != nullptr && v_cache != nullptr && v != nullptr &&
                    slot_mapping != nullptr && num_slots >= 0,
                KVC_ERR_VALUE, "%s: the append needs v, both caches and slots", what);
    KVC_REQUIRE(slot_index_bytes == 4 || slot_index_bytes == 8, KVC_ERR_VALUE,
                "%s: slot_mapping must be int32 or int64", what);
    KVC_REQUIRE(rows16(v, v_stride_t, v_stride_h) && rows16(k_cache, 0, 0) &&
                    rows16(v_cache, 0, 0),
                KVC_ERR_ASSERT, "%s: v rows and caches must be 16-byte aligned", what);
  }
  KVC_REQUIRE(rows16(q, q_stride_t, q_stride_h) && rows16(k, k_stride_t, k_stride_h) &&
                  rows16(q_out, q_out_stride_t, q_out_stride_h) &&
                  (k_out == nullptr || rows16(k_out, k_out_stride_t, k_out_stride_h)),
              KVC_ERR_ASSERT, "%s: q/k rows must be 16-byte aligned", what);
  KVC_REQUIRE(rows16(q_norm_weight, 0, 0) && rows16(k_norm_weight, 0, 0) &&
                  rows16(cos_sin_cache, 0, 0),
              KVC_ERR_ASSERT, "%s: weights and cache must be 16-byte aligned", what);
  a.q = static_cast<const uint16_t*>(q);
  a.q_st = q_stride_t;
  a.q_sh = q_stride_h;
  a.k = static_cast<const uint16_t*>(k);
  a.k_st = k_stride_t;
  a.k_sh = k_stride_h;
  a.v = static_cast<const uint16_t*>(v);
  a.v_st = v_stride_t;
  a.v_sh = v_stride_h;
  a.positions = positions;
  a.pos_stride = position_stride;
  a.q_w = static_cast<const uint16_t*>(q_norm_weight);
  a.k_w = static_cast<const uint16_t*>(k_norm_weight);
  a.cos_sin = cos_sin_cache;
  a.max_position = max_position;
  a.eps = eps;
  a.q_out = static_cast<uint16_t*>(q_out);
  a.qo_st = q_out_stride_t;
  a.qo_sh = q_out_stride_h;
  a.k_out = static_cast<uint16_t*>(k_out);
  a.ko_st = k_out_stride_t;
  a.ko_sh = k_out_stride_h;
  a.k_cache = static_cast<uint16_t*>(k_cache);
  a.v_cache = static_cast<uint16_t*>(v_cache);
  a.num_slots = num_slots;
  a.slots = slot_mapping;
  a.num_tokens = num_tokens;
  a.num_heads = int(num_heads);
  a.num_kv_heads = int(num_kv_heads);
  hipStream_t st = as_stream(stream);
  const int sb = cache ? slot_index_bytes : 4;
  // Four tokens a workgroup share its position and table loads; up to 1024
  // tokens one each keeps every CU busy.  Measured, 1 / 4 a workgroup (32 / 4
  // heads, q_out through the caches): 64 tokens 5.5 / 6.4 us, 1024 6.1 / 7.6,
  // 2048 11.6 / 10.7, 16384 94.9 / 72.7.
  if (num_tokens > 1024) {
    launch<4, 5>(a, position_index_bytes, sb, st);
  } else {
    launch<1, 2>(a, position_index_bytes, sb, st);
  }
  return check_launch(what);
}
