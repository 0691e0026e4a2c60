// The accepted path of a drafted token tree kept: its rows, wherever the tree
// holds them, moved to the end of the context, in every plane of the pool.
//
// Row path[j] of sequence b's tree (pool position context + path[j]) goes to
// position context + j, j = 0, 1, ...  A root-to-leaf path of a tree whose
// parents come before their children is strictly increasing, so path[j] >= j
// and every later source lies past every destination written so far: a lane
// that owns one 16-byte column of a (plane, sequence) moves its rows in order
// without a barrier, a batch of loads ahead of the batch's stores.  A path
// ends at its first entry that does not increase or leaves the table, so that
// order holds whatever the device holds.
//
// Bound by latency (lengths, path, table, row: four dependent reads) for one
// user (4 us), by HBM for a batch: each moved row is read and written once (64
// sequences, K and V of 28 layers, 29 MB both ways: 7.5 us, of which the four
// reads are half).
#include "kvc_internal.h"

namespace kvc {
namespace {

constexpr int kWaves = 4;
constexpr int kBatch = 8;  // rows a lane holds between its loads and stores

struct CommitArgs {
  char* pool;
  int64_t planes, plane_stride;
  int64_t num_blocks, page, row_bytes;
  const int32_t* tables;
  int64_t bt_stride, max_blocks;
  const int32_t* lens;
  const int32_t* paths;
  int64_t path_stride;
  int max_path;
  const int32_t* path_lens;
  int64_t batch;
  int chunks;  // 64-unit column chunks of a row
};

// Byte offset of position pos in a plane, or -1.
__device__ __forceinline__ int64_t row_offset(const CommitArgs& a, int64_t b, int64_t pos) {
  if (pos < 0 || pos >= a.max_blocks * a.page) return -1;
  const int64_t pg = pos / a.page;
  const int blk = a.tables[b * a.bt_stride + pg];
  if (blk < 0 || blk >= a.num_blocks) return -1;
  return (blk * a.page + (pos - pg * a.page)) * a.row_bytes;
}

__device__ __forceinline__ int64_t lane64(int64_t v, int l) {
  const uint32_t lo = uint32_t(__builtin_amdgcn_readlane(int(uint32_t(v)), l));
  const uint32_t hi = uint32_t(__builtin_amdgcn_readlane(int(uint32_t(uint64_t(v) >> 32)), l));
  return int64_t((uint64_t(hi) << 32) | lo);
}

template <typename Unit>
__global__ void __launch_bounds__(64 * kWaves) commit_rows_kernel(CommitArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t w = int64_t(blockIdx.x) * kWaves + uniform(int(threadIdx.x >> 6));
  // Planes fastest: the waves of one sequence share its path and table reads.
  const int64_t b = w / (a.planes * a.chunks);
  if (b >= a.batch) return;
  const int64_t rest = w - b * a.planes * a.chunks;
  const int64_t plane = rest / a.chunks;
  const int64_t unit = (rest - plane * a.chunks) * 64 + lane;
  const bool mine = unit * int64_t(sizeof(Unit)) < a.row_bytes;
  char* base = a.pool + plane * a.plane_stride + unit * int64_t(sizeof(Unit));

  const int n = min(a.path_lens[b], a.max_path);
  const int64_t ctx = a.lens[b];
  int before = -1;  // the entry before this round's first
  for (int j0 = 0; j0 < n; j0 += 64) {
    const int j = j0 + lane;
    const int at = j < n ? a.paths[b * a.path_stride + j] : -1;
    const int up = __shfl_up(at, 1, 64);
    int64_t src = -1, dst = -1;
    if (j < n && at > (lane == 0 ? before : up)) {
      src = row_offset(a, b, ctx + at);
      dst = row_offset(a, b, ctx + j);
    }
    const uint64_t bad = __ballot(src < 0 || dst < 0);
    const int m = bad != 0 ? __builtin_ctzll(bad) : 64;
    for (int r = 0; r < m; r += kBatch) {
      Unit v[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        if (r + i < m) {
          const int64_t s = lane64(src, r + i);
          if (mine && s != lane64(dst, r + i)) v[i] = *reinterpret_cast<const Unit*>(base + s);
        }
      }
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        if (r + i < m) {
          const int64_t d = lane64(dst, r + i);
          if (mine && lane64(src, r + i) != d) *reinterpret_cast<Unit*>(base + d) = v[i];
        }
      }
    }
    if (m < 64) return;
    before = __builtin_amdgcn_readlane(at, 63);
  }
}

}  // namespace
}  // namespace kvc

using namespace kvc;

extern "C" int kvc_commit_rows(void* pool, int64_t planes, int64_t plane_stride,
                               int64_t num_blocks, int64_t page_size, int64_t row_bytes,
                               const int32_t* block_tables, int64_t bt_stride,
                               int64_t max_blocks_per_seq, const int32_t* context_lens,
                               const int32_t* paths, int64_t path_stride, int64_t max_path,
                               const int32_t* path_lens, int64_t batch, kvc_stream_t stream) {
  clear_error();
  KVC_REQUIRE(planes >= 0 && batch >= 0 && max_path >= 0, KVC_ERR_VALUE,
              "commit_rows: negative counts");
  if (planes == 0 || batch == 0 || max_path == 0) return KVC_OK;
  KVC_REQUIRE(pool != nullptr && block_tables != nullptr && context_lens != nullptr &&
                  paths != nullptr && path_lens != nullptr,
              KVC_ERR_VALUE, "commit_rows: missing pool, tables, lengths or paths");
  KVC_REQUIRE(num_blocks > 0 && num_blocks < (int64_t(1) << 31) && page_size > 0 &&
                  row_bytes > 0 && max_blocks_per_seq >= 0 && max_path < (int64_t(1) << 31) &&
                  num_blocks < (int64_t(1) << 62) / (page_size * row_bytes) &&
                  plane_stride >= num_blocks * page_size * row_bytes,
              KVC_ERR_VALUE, "commit_rows: bad pool size");
  CommitArgs a{};
  a.pool = static_cast<char*>(pool);
  a.planes = planes;
  a.plane_stride = plane_stride;
  a.num_blocks = num_blocks;
  a.page = page_size;
  a.row_bytes = row_bytes;
  a.tables = block_tables;
  a.bt_stride = bt_stride;
  a.max_blocks = max_blocks_per_seq;
  a.lens = context_lens;
  a.paths = paths;
  a.path_stride = path_stride;
  a.max_path = int(max_path);
  a.path_lens = path_lens;
  a.batch = batch;
  // The widest unit that rows and planes keep aligned.
  const uint64_t bits = uint64_t(reinterpret_cast<uintptr_t>(pool)) | uint64_t(row_bytes) |
                        uint64_t(plane_stride);
  const int unit = bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : 1;
  const int64_t chunks = (row_bytes / unit + 63) / 64;
  const int64_t waves = batch * planes * chunks;
  KVC_REQUIRE(chunks < (1 << 20) && waves < (int64_t(1) << 31), KVC_ERR_VALUE,
              "commit_rows: too many rows for one call");
  a.chunks = int(chunks);
  const dim3 grid{unsigned((waves + kWaves - 1) / kWaves)};
  hipStream_t st = as_stream(stream);
  if (unit == 16) {
    commit_rows_kernel<u32x4_t><<<grid, 64 * kWaves, 0, st>>>(a);
  } else if (unit == 4) {
    commit_rows_kernel<uint32_t><<<grid, 64 * kWaves, 0, st>>>(a);
  } else {
    commit_rows_kernel<uint8_t><<<grid, 64 * kWaves, 0, st>>>(a);
  }
  return check_launch("commit_rows");
}
