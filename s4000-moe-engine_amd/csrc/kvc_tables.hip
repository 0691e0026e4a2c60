// A serving step's tables from its requests' lengths, on the GPU (gfx950).
//
// Row b has context_lens[b] tokens in held[b] pages and brings query_lens[b] new
// ones.  Requests that ended give their pages back to the stack of free ones, in
// row order; then every row takes from its top what its new tokens need, in row
// order, as far as they go.  A row that does not fit (pages left, columns of the
// table, tokens of the step) waits: it gets no tokens and takes nothing, and so
// does every later row that needs a page, or comes after the step is full; rows
// that need no page go on.  Slots, positions and offsets of the tokens follow.
//
// One workgroup does all of it, a thread a row: four prefix sums over the rows
// (pages given back; needed; tokens wanted; then pages, tokens and keys granted
// together), from DPP scans and one exchange of wave sums each.  The tokens are
// filled by the same launch up to kOneLaunch of them and else by a second one
// over the chip.  Bound by latency throughout: a decode step of 64 rows moves
// some 4 KB and takes 3.7 us; 512 rows with 66000 tokens 6.2 + 4.3 us (2 MB).
#include <algorithm>

#include "kvc_internal.h"

namespace kvc {
namespace {

constexpr int kMaxThreads = 1024;
constexpr int kMaxWaves = kMaxThreads / 64;
constexpr int kFillThreads = 256;
constexpr int kLdsRows = 4096;         // offsets searched in LDS up to this many rows
constexpr int64_t kOneLaunch = 4096;   // tokens
constexpr int kLongest = 1 << 29;      // of a length
constexpr int kMostWanted = 1 << 25;   // past every max_tokens

struct TablesArgs {
  const int32_t* context_lens;
  const int32_t* query_lens;
  const uint8_t* finished;  // or null
  int32_t* ended;           // lengths set to 0 where finished (context_lens itself, say), or null
  int32_t* tables;
  int64_t bt_stride;
  int width, batch;
  const int32_t* held;
  int32_t* free_blocks;
  int64_t free_size;
  const int32_t* num_free;
  int page, page_shift;  // page_shift -1: no power of two
  int max_tokens, per_row;
  int pad_slot;
  int32_t* slots;
  int64_t* positions;
  int32_t* query_out;
  int32_t* seq_out;
  int32_t* context_out;
  int32_t* held_out;
  int32_t* num_free_out;
  int32_t* cu_q;
  int32_t* cu_k;
};

// The sums over all rows before a thread's, and over the block, of N values.  A wave's
// sum counts up to kMost where waves are added.
template <int N>
struct Sums {
  int before[N], all[N];
};
template <int N, int kMost = 0x7fffffff>
__device__ __forceinline__ Sums<N> block_sums(const int (&x)[N], int (*lds)[kMaxWaves], int lane,
                                              int wave, int waves) {
  Sums<N> s;
  int incl[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    incl[i] = wave_scan_add(x[i]);
    if (lane == 63) lds[i][wave] = min(incl[i], kMost);
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int w = wave_scan_add(lane < waves ? lds[i][lane] : 0);
    const int earlier = __shfl(w, max(wave - 1, 0), 64);
    s.before[i] = incl[i] - x[i] + (wave > 0 ? earlier : 0);
    s.all[i] = __builtin_amdgcn_readlane(w, 63);
  }
  return s;
}

__device__ __forceinline__ int page_of(const TablesArgs& a, int pos) {
  return a.page_shift >= 0 ? pos >> a.page_shift : pos / a.page;
}

// Token t: its slot and position.  at(i): cu_q[i].
template <class At>
__device__ __forceinline__ void fill_token(const TablesArgs& a, int t, const At& at) {
  int row, nth;
  if (a.per_row > 0) {
    row = t / a.per_row;
    nth = t - row * a.per_row;
  } else {
    int lo = 0, hi = a.batch;  // the first row whose end lies past t
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (at(mid + 1) <= t) lo = mid + 1; else hi = mid;
    }
    row = lo;
    nth = row < a.batch ? t - at(row) : 0;
  }
  int slot = a.pad_slot;
  int pos = 0;
  if (row < a.batch) {
    const int got = a.query_out[row];
    if (nth < got) {
      pos = a.seq_out[row] - got + nth;
      const int pg = page_of(a, pos);
      const int64_t blk = a.tables[int64_t(row) * a.bt_stride + pg];
      const int64_t s = blk * a.page + (pos - pg * a.page);
      // (a bad table entry gives no slot)
      if (blk >= 0 && s < (int64_t(1) << 31)) slot = int(s);
    }
  }
  a.slots[t] = slot;
  a.positions[t] = pos;
}

__global__ void __launch_bounds__(kMaxThreads) step_tables_kernel(TablesArgs a, int fill) {
  __shared__ int lds[6][kMaxWaves];
  __shared__ int cu[kLdsRows + 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int threads = blockDim.x, waves = threads >> 6;
  const int free0 = int(max(int64_t(0), min(int64_t(a.num_free[0]), a.free_size)));

  // Pages that come back.
  int64_t top64 = free0;
  if (a.finished != nullptr) {
    for (int r0 = 0; r0 < a.batch; r0 += threads) {
      const int r = r0 + int(threadIdx.x);
      const bool gone = r < a.batch && a.finished[r] != 0;
      const int pages = gone ? min(max(a.held[r], 0), a.width) : 0;
      const int x[1] = {pages};
      const Sums<1> s = block_sums<1>(x, lds, lane, wave, waves);
      uint64_t todo = __builtin_amdgcn_ballot_w64(pages > 0);
      while (todo != 0) {
        const int from = __builtin_ctzll(todo);
        todo &= todo - 1;
        const int n = __builtin_amdgcn_readlane(pages, from);
        const int64_t to = top64 + __builtin_amdgcn_readlane(s.before[0], from);
        const int32_t* src = a.tables + int64_t(r0 + 64 * wave + from) * a.bt_stride;
        for (int j = lane; j < n; j += 64)
          if (to + j < a.free_size) a.free_blocks[to + j] = src[j];
      }
      top64 += s.all[0];
      __syncthreads();  // lds is free again, and the pages are in place
    }
  }
  const int top = int(min(top64, a.free_size));

  int need0 = 0, take0 = 0, got0 = 0, seen0 = 0;
  int64_t want0 = 0;
  for (int r0 = 0; r0 < a.batch; r0 += threads) {
    const int r = r0 + int(threadIdx.x);
    const bool live = r < a.batch;
    const bool gone = live && a.finished != nullptr && a.finished[r] != 0;
    const int ctx = live && !gone ? min(max(a.context_lens[r], 0), kLongest) : 0;
    const int held = live && !gone ? min(max(a.held[r], 0), a.width) : 0;
    const int asked = live ? min(max(a.query_lens[r], 0), kLongest) : 0;
    const int pages = page_of(a, ctx + asked - 1 + a.page);
    bool able = asked > 0 && pages <= a.width;
    const int need = able ? max(pages - held, 0) : 0;
    const int x[1] = {need};
    const Sums<1> sn = block_sums<1>(x, lds, lane, wave, waves);
    able = able && (need == 0 || need0 + sn.before[0] + need <= top);
    const int want = able ? min(asked, a.max_tokens + 1) : 0;
    if (a.per_row > 0) {
      able = able && want <= a.per_row;
    } else {
      // (max_tokens is under 2^24, so a wave's wants are up to 2^30 and sixteen waves'
      // 2^34: each wave's count up to 2^25, past max_tokens like what they were)
      const int y[1] = {want};
      const Sums<1> sw = block_sums<1, kMostWanted>(y, lds + 1, lane, wave, waves);
      able = able && want0 + sw.before[0] + want <= a.max_tokens;
      want0 = min(want0 + sw.all[0], int64_t(kMostWanted));
    }
    const int got = able ? asked : 0, take = able ? need : 0;
    const int seen = able ? ctx + got : 0;
    const int z[3] = {take, got, seen};
    const Sums<3> sg = block_sums<3>(z, lds + 2, lane, wave, waves);
    if (gone && a.ended != nullptr) a.ended[r] = 0;
    if (live) {
      a.query_out[r] = got;
      a.seq_out[r] = seen;
      a.context_out[r] = ctx + got;
      a.held_out[r] = held + take;
      const int q_end = got0 + sg.before[1] + got;
      a.cu_q[r + 1] = q_end;
      a.cu_k[r + 1] = seen0 + sg.before[2] + seen;
      if (fill && r < kLdsRows) cu[r + 1] = q_end;
    }
    // The row's j-th new page is the (taken before + j)-th from the top.
    const int first = top - 1 - (take0 + sg.before[0]);
    if (take == 1) a.tables[int64_t(r) * a.bt_stride + held] = a.free_blocks[first];
    uint64_t todo = __builtin_amdgcn_ballot_w64(take > 1);
    while (todo != 0) {
      const int from = __builtin_ctzll(todo);
      todo &= todo - 1;
      const int n = __builtin_amdgcn_readlane(take, from);
      const int src = __builtin_amdgcn_readlane(first, from);
      int32_t* dst = a.tables + int64_t(r0 + 64 * wave + from) * a.bt_stride +
                     __builtin_amdgcn_readlane(held, from);
      for (int j = lane; j < n; j += 64) dst[j] = a.free_blocks[src - j];
    }
    need0 = min(need0 + sn.all[0], 1 << 30);
    take0 += sg.all[0];
    got0 += sg.all[1];
    seen0 += sg.all[2];
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    a.cu_q[0] = a.cu_k[0] = 0;
    cu[0] = 0;
    a.num_free_out[0] = top - take0;
  }
  if (!fill) return;
  __syncthreads();
  for (int t = threadIdx.x; t < a.max_tokens; t += threads)
    fill_token(a, t, [&](int i) { return cu[i]; });
}

__global__ void __launch_bounds__(kFillThreads) fill_tokens_kernel(TablesArgs a) {
  __shared__ int cu[kLdsRows + 1];
  const bool local = a.per_row == 0 && a.batch <= kLdsRows;
  if (local) {
    for (int i = threadIdx.x; i <= a.batch; i += kFillThreads) cu[i] = a.cu_q[i];
    __syncthreads();
  }
  const int t = int(blockIdx.x) * kFillThreads + int(threadIdx.x);
  if (t >= a.max_tokens) return;
  if (local) {
    fill_token(a, t, [&](int i) { return cu[i]; });
  } else {
    fill_token(a, t, [&](int i) { return a.cu_q[i]; });
  }
}

}  // namespace
}  // namespace kvc

using namespace kvc;

extern "C" int kvc_step_tables_ended(
    const int32_t* context_lens, const int32_t* query_lens, const uint8_t* finished,
    int32_t* ended_lens, int32_t* block_tables, int64_t bt_stride, int64_t max_blocks_per_seq,
    int64_t batch, const int32_t* num_blocks, int32_t* free_blocks, int64_t free_size,
    const int32_t* num_free, int64_t page_size, int64_t max_tokens, int64_t tokens_per_row,
    int32_t pad_slot, int32_t* slot_mapping, int64_t* positions, int32_t* query_lens_out,
    int32_t* seq_lens_out, int32_t* context_lens_out, int32_t* num_blocks_out,
    int32_t* num_free_out, int32_t* cu_seqlens_q, int32_t* cu_seqlens_k, kvc_stream_t stream) {
  clear_error();
  KVC_REQUIRE(batch >= 0 && batch < (1 << 20) && max_blocks_per_seq >= 0 &&
                  batch * max_blocks_per_seq < (int64_t(1) << 30) && free_size >= 0 &&
                  free_size < (int64_t(1) << 30),
              KVC_ERR_VALUE, "step_tables: shape out of range");
  KVC_REQUIRE(page_size > 0 && page_size <= (1 << 20), KVC_ERR_VALUE,
              "step_tables: page_size must be 1 to 2^20 (got %lld)", (long long)page_size);
  KVC_REQUIRE(max_tokens >= 0 && max_tokens < (1 << 24), KVC_ERR_VALUE,
              "step_tables: max_tokens must be below 2^24 (got %lld)", (long long)max_tokens);
  KVC_REQUIRE(tokens_per_row >= 0 &&
                  (tokens_per_row == 0 || max_tokens == batch * tokens_per_row),
              KVC_ERR_VALUE, "step_tables: max_tokens must be batch x tokens_per_row");
  KVC_REQUIRE(num_free != nullptr && num_free_out != nullptr && cu_seqlens_q != nullptr &&
                  cu_seqlens_k != nullptr &&
                  (batch == 0 || (context_lens != nullptr && query_lens != nullptr &&
                                  num_blocks != nullptr && query_lens_out != nullptr &&
                                  seq_lens_out != nullptr && context_lens_out != nullptr &&
                                  num_blocks_out != nullptr)) &&
                  (batch * max_blocks_per_seq == 0 || block_tables != nullptr) &&
                  (free_size == 0 || free_blocks != nullptr) &&
                  (max_tokens == 0 || (slot_mapping != nullptr && positions != nullptr)),
              KVC_ERR_VALUE, "step_tables: null pointer");
  // An output may be the input of its own name, and nothing else of the call's.
  const void* ins[] = {query_lens, context_lens, num_blocks, num_free, block_tables, free_blocks,
                       finished};
  const void* outs[] = {query_lens_out, context_lens_out, num_blocks_out, num_free_out,
                        seq_lens_out,   cu_seqlens_q,     cu_seqlens_k,   slot_mapping,
                        positions};
  for (int i = 0; i < 9 && batch > 0; ++i) {
    for (int j = 0; j < 7; ++j)
      KVC_REQUIRE(outs[i] == nullptr || outs[i] != ins[j] || (i == j && i < 4), KVC_ERR_VALUE,
                  "step_tables: an output over another input");
    for (int j = 0; j < i; ++j)
      KVC_REQUIRE(outs[i] == nullptr || outs[i] != outs[j], KVC_ERR_VALUE,
                  "step_tables: two outputs in one place");
  }
  for (int i = 0; i < 9 && ended_lens != nullptr; ++i)
    KVC_REQUIRE(outs[i] != ended_lens, KVC_ERR_VALUE, "step_tables: ended_lens over an output");
  for (int j = 0; j < 7 && ended_lens != nullptr; ++j)
    KVC_REQUIRE(j == 1 || ins[j] != ended_lens, KVC_ERR_VALUE,
                "step_tables: ended_lens over another input");
  TablesArgs a{};
  a.context_lens = context_lens;
  a.query_lens = query_lens;
  a.finished = finished;
  a.ended = ended_lens;
  a.tables = block_tables;
  a.bt_stride = bt_stride;
  a.width = int(max_blocks_per_seq);
  a.batch = int(batch);
  a.held = num_blocks;
  a.free_blocks = free_blocks;
  a.free_size = free_size;
  a.num_free = num_free;
  a.page = int(page_size);
  a.page_shift = (page_size & (page_size - 1)) == 0 ? __builtin_ctzll(page_size) : -1;
  a.max_tokens = int(max_tokens);
  a.per_row = int(tokens_per_row);
  a.pad_slot = pad_slot;
  a.slots = slot_mapping;
  a.positions = positions;
  a.query_out = query_lens_out;
  a.seq_out = seq_lens_out;
  a.context_out = context_lens_out;
  a.held_out = num_blocks_out;
  a.num_free_out = num_free_out;
  a.cu_q = cu_seqlens_q;
  a.cu_k = cu_seqlens_k;
  const int fill = max_tokens <= kOneLaunch && batch <= kLdsRows;
  const int64_t work = std::max<int64_t>(batch, fill ? max_tokens : 0);
  const int64_t waves = std::max<int64_t>(1, (work + 63) / 64);
  const int threads = int(std::min<int64_t>(kMaxThreads, waves * 64));
  hipStream_t st = as_stream(stream);
  step_tables_kernel<<<1, threads, 0, st>>>(a, fill);
  if (!fill && max_tokens > 0)
    fill_tokens_kernel<<<unsigned((max_tokens + kFillThreads - 1) / kFillThreads), kFillThreads, 0,
                         st>>>(a);
  return check_launch("step_tables");
}

extern "C" int kvc_step_tables(const int32_t* context_lens, const int32_t* query_lens,
                               const uint8_t* finished, int32_t* block_tables, int64_t bt_stride,
                               int64_t max_blocks_per_seq, int64_t batch,
                               const int32_t* num_blocks, int32_t* free_blocks,
                               int64_t free_size, const int32_t* num_free, int64_t page_size,
                               int64_t max_tokens, int64_t tokens_per_row, int32_t pad_slot,
                               int32_t* slot_mapping, int64_t* positions,
                               int32_t* query_lens_out, int32_t* seq_lens_out,
                               int32_t* context_lens_out, int32_t* num_blocks_out,
                               int32_t* num_free_out, int32_t* cu_seqlens_q,
                               int32_t* cu_seqlens_k, kvc_stream_t stream) {
  return kvc_step_tables_ended(context_lens, query_lens, finished, nullptr, block_tables,
                               bt_stride, max_blocks_per_seq, batch, num_blocks, free_blocks,
                               free_size, num_free, page_size, max_tokens, tokens_per_row,
                               pad_slot, slot_mapping, positions, query_lens_out, seq_lens_out,
                               context_lens_out, num_blocks_out, num_free_out, cu_seqlens_q,
                               cu_seqlens_k, stream);
}
