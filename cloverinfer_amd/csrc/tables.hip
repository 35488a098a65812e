// tables.hip - one scheduling step of the paged cache's bookkeeping on the GPU.
//
// The block allocator of KVCacheManager (src/core/memory_manager.py:49-72,
// 95-121, 134-143: a LIFO stack of free blocks, popped from its end) for all
// rows of a block table at once. Row r holds held[r] blocks for len[r] tokens;
// new[r] > 0 tokens join it, 0 leaves it, < 0 ends it. With exclusive prefix
// sums over the rows of
//   tok[r]  = max(new[r], 0)
//   take[r] = max(held[r], ceil((len[r] + new[r] + (held[r] ? 0 : reserve)) / bs)) - held[r]
//                                                        where new[r] > 0, else 0
//   gone[r] = held[r] where new[r] < 0, else 0
// and totals T, K, R, the stack V of a step is free[0, F) followed by the ended
// rows' blocks (row by row, in table order), and the i-th block taken (rows in
// order, each row's columns in order) is V[F + R - 1 - i]: what free() for each
// ended row and then allocate() / append_slot() for each growing one do one
// call at a time. Every entry, slot and pushed block is therefore a closed
// expression of the prefix sums and of what the buffers held before the step,
// and nothing written is read again: all of it runs in parallel, in any order,
// also in place. (Entries at columns >= held[r] are not read; those of rows
// that ended stay as they were.)
//
// A step moves a few KB to a few MB, so it is bound by launch and memory
// latency. Small steps run in one workgroup: it scans the rows (its copy of
// the state in LDS lets the state be written in place), then serves entries
// and slots from LDS. Larger ones run a second launch over the chip.
#include "clover_attn.h"
#include "clv_device.h"

namespace clv {
namespace {

constexpr int kScanThreads = 1024;
constexpr int kFillThreads = 256;

// A step's rows: exclusive prefix sums [rows + 1], and the state before it [rows].
struct StepRows {
  int32_t *tok, *take, *gone;
  int32_t *len, *held;
};

__device__ __host__ __forceinline__ StepRows step_rows(int32_t *base, int rows) {
  StepRows s;
  s.tok = base;
  s.take = s.tok + rows + 1;
  s.gone = s.take + rows + 1;
  s.len = s.gone + rows + 1;
  s.held = s.len + rows;
  return s;
}

// What a step does in all.
struct StepTotals {
  int32_t tokens, take, gone;
  int32_t num_free;  // before the step
  int32_t status;
};

// Last row whose prefix is <= i (0 <= i < prefix[rows]).
__device__ __forceinline__ int row_of(const int32_t *prefix, int rows, int i) {
  int lo = 0, n = rows;
  while (n > 1) {
    const int half = n >> 1;
    const bool right = prefix[lo + half] <= i;
    lo += right ? half : 0;
    n -= half;
    if (!right) n = half;
  }
  return lo;
}

// Scans the rows into s (LDS or global memory), checks the step, and writes
// the state after it. All kScanThreads threads call it.
__device__ StepTotals scan_step(const TablesParams &p, const StepRows &s) {
  __shared__ int64_t s_sum[kScanThreads / 64][3];
  __shared__ int s_flags[kScanThreads / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int per = (p.rows + kScanThreads - 1) / kScanThreads;
  const int b = min(p.rows, tid * per), e = min(p.rows, b + per);
  const int F = p.num_free[0];
  auto row = [&](int r, int &len, int &held, int &n, int64_t &need) {
    len = p.context_lens[r];
    held = p.blocks_held[r];
    n = p.new_lens[r];
    need = held;
    if (n > 0) {
      const int64_t all = (int64_t)len + n + (held == 0 ? p.reserve : 0);
      need = max((int64_t)held, (all + (1 << p.block_shift) - 1) >> p.block_shift);
    }
  };
  // Bit 0: a row longer than its table; bit 1: a state that cannot be.
  int64_t x[3] = {0, 0, 0};
  int flags = F < 0 || F > p.num_blocks ? 2 : 0;
  for (int r = b; r < e; ++r) {
    int len, held, n;
    int64_t need;
    row(r, len, held, n, need);
    if (need > p.width) flags |= 1;
    if (len < 0 || held < 0 || held > p.width || len > ((int64_t)held << p.block_shift)) flags |= 2;
    x[0] += max(n, 0);
    x[1] += need - held;
    x[2] += n < 0 ? held : 0;
  }
  const int64_t own[3] = {x[0], x[1], x[2]};
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      const int64_t y = __shfl_up(x[k], off, 64);
      if (lane >= off) x[k] += y;
    }
    flags |= __shfl_xor(flags, off, 64);
  }
  if (lane == 63) {
#pragma unroll
    for (int k = 0; k < 3; ++k) s_sum[wave][k] = x[k];
    s_flags[wave] = flags;
  }
  __syncthreads();
  int64_t run[3], all[3] = {0, 0, 0};
#pragma unroll
  for (int k = 0; k < 3; ++k) run[k] = x[k] - own[k];
  flags = 0;
  for (int w = 0; w < kScanThreads / 64; ++w) {
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      if (w < wave) run[k] += s_sum[w][k];
      all[k] += s_sum[w][k];
    }
    flags |= s_flags[w];
  }
  StepTotals t;
  if ((flags & 2) || F + all[2] > p.num_blocks) t.status = CLV_TABLES_BAD_STATE;
  else if (all[1] > F + all[2]) t.status = CLV_TABLES_NO_BLOCKS;
  else if (flags & 1) t.status = CLV_TABLES_ROW_FULL;
  else if (all[0] > p.num_tokens) t.status = CLV_TABLES_NO_SLOTS;
  else t.status = CLV_TABLES_OK;
  const bool ok = t.status == CLV_TABLES_OK;
  t.num_free = F;
  t.tokens = ok ? (int32_t)all[0] : 0;
  t.take = ok ? (int32_t)all[1] : 0;
  t.gone = ok ? (int32_t)all[2] : 0;
  // In place, a row's state is read and written by the same thread, and every
  // thread has read the stack's count before the barrier above.
  for (int r = b; r < e; ++r) {
    int len, held, n;
    int64_t need;
    row(r, len, held, n, need);
    s.tok[r] = ok ? (int32_t)run[0] : 0;
    s.take[r] = ok ? (int32_t)run[1] : 0;
    s.gone[r] = ok ? (int32_t)run[2] : 0;
    s.len[r] = len;
    s.held[r] = held;
    p.query_start_loc[r] = ok ? (int32_t)run[0] : 0;
    p.context_lens_out[r] = !ok ? len : n < 0 ? 0 : len + n;
    p.blocks_held_out[r] = !ok ? held : n < 0 ? 0 : (int32_t)need;
    run[0] += max(n, 0);
    run[1] += need - held;
    run[2] += n < 0 ? held : 0;
  }
  if (tid == 0) {
    s.tok[p.rows] = t.tokens;
    s.take[p.rows] = t.take;
    s.gone[p.rows] = t.gone;
    p.query_start_loc[p.rows] = t.tokens;
    p.num_free_out[0] = F + t.gone - t.take;
    p.status[0] = t.status;
  }
  return t;
}

// Thread `at` of `n` serves its share of the step's pushed blocks, table
// entries and slots.
__device__ __forceinline__ void fill_step(const TablesParams &p, const StepRows &s,
                                          const StepTotals &t, int64_t at, int64_t n) {
  const int F = t.num_free, R = t.gone, K = t.take;
  // Block v of the stack V.
  auto stack = [&](int v) {
    if (v < F) return p.free_blocks[v];
    const int r = row_of(s.gone, p.rows, v - F);
    return p.block_tables[(int64_t)r * p.width + (v - F - s.gone[r])];
  };
  for (int64_t i = at; i < R - K; i += n) p.free_blocks[F + i] = stack(F + (int)i);
  for (int64_t i = at; i < K; i += n) {
    const int r = row_of(s.take, p.rows, (int)i);
    p.block_tables[(int64_t)r * p.width + s.held[r] + (i - s.take[r])] = stack(F + R - 1 - (int)i);
  }
  const int mask = (1 << p.block_shift) - 1;
  for (int64_t i = at; i < p.num_tokens; i += n) {
    int64_t slot = -1;
    if (i < t.tokens) {
      const int r = row_of(s.tok, p.rows, (int)i);
      const int pos = s.len[r] + ((int)i - s.tok[r]);
      const int col = pos >> p.block_shift;
      const int blk = col < s.held[r] ? p.block_tables[(int64_t)r * p.width + col]
                                      : stack(F + R - 1 - (s.take[r] + col - s.held[r]));
      slot = ((int64_t)blk << p.block_shift) + (pos & mask);
    }
    p.slot_mapping[i] = slot;
  }
}

__global__ void __launch_bounds__(kScanThreads) tables_step(const TablesParams p) {
  extern __shared__ int32_t s_rows[];
  const StepRows s = step_rows(s_rows, p.rows);
  const StepTotals t = scan_step(p, s);
  __syncthreads();
  fill_step(p, s, t, threadIdx.x, kScanThreads);
}

// The two launches of a larger step: the scan into the workspace (totals, then
// the rows), and the rest of it over the chip.
constexpr int kTotalsInts = 8;

__global__ void __launch_bounds__(kScanThreads) tables_scan(const TablesParams p, int32_t *ws) {
  const StepTotals t = scan_step(p, step_rows(ws + kTotalsInts, p.rows));
  if (threadIdx.x == 0) *reinterpret_cast<StepTotals *>(ws) = t;
}

__global__ void __launch_bounds__(kFillThreads)
tables_fill(const TablesParams p, const int32_t *__restrict__ ws) {
  extern __shared__ int32_t s_rows[];
  const StepTotals t = *reinterpret_cast<const StepTotals *>(ws);
  const int n = 5 * p.rows + 3;
  for (int i = threadIdx.x; i < n; i += kFillThreads) s_rows[i] = ws[kTotalsInts + i];
  __syncthreads();
  fill_step(p, step_rows(s_rows, p.rows), t, (int64_t)blockIdx.x * kFillThreads + threadIdx.x,
            (int64_t)gridDim.x * kFillThreads);
}

size_t rows_bytes(int rows) { return (size_t)(5 * rows + 3) * 4; }

// Steps that one workgroup serves.
constexpr int64_t kSmallTokens = 8192;

}  // namespace

size_t tables_workspace_bytes(const TablesParams &p) {
  return p.num_tokens <= kSmallTokens ? 0 : kTotalsInts * 4 + rows_bytes(p.rows);
}

hipError_t launch_tables(const TablesParams &p, void *workspace, hipStream_t stream) {
  if (tables_workspace_bytes(p) == 0) {
    hipLaunchKernelGGL(tables_step, dim3(1), dim3(kScanThreads), rows_bytes(p.rows), stream, p);
    return hipGetLastError();
  }
  hipLaunchKernelGGL(tables_scan, dim3(1), dim3(kScanThreads), 0, stream, p, (int32_t *)workspace);
  const int64_t groups = (p.num_tokens + 4 * kFillThreads - 1) / (4 * kFillThreads);
  hipLaunchKernelGGL(tables_fill, dim3((unsigned)(groups < 1024 ? groups : 1024)),
                     dim3(kFillThreads), rows_bytes(p.rows), stream, p, (const int32_t *)workspace);
  return hipGetLastError();
}

}  // namespace clv
