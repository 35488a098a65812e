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
// latency: a chain of one read of the rows, a scan, a search in LDS, one read of
// a table or stack entry, one write. Every workgroup scans the rows itself
// rather than wait for a launch that does, and takes an even share of the step's
// slots, entries and pushed blocks. Per launch: 128 rows of one token 4.8 us (5.4
// a call, which the host bounds); 256 rows that end, wait, grow or come new, 33000
// slots, 8.0; 512 prompts, a million slots (9 MB), 8.2. Sums in 64 bits cost 0.7 to
// 1.2 us, a binary search 1 us of the mixed step; workgroups of 512 and 1024
// threads (fewer scans) ran 9.6 and 11.4 against 9.8 then.
#include "clover_attn.h"
#include "clv_device.h"

namespace clv {
namespace {

constexpr int kRun = 4;  // consecutive slots (two 16-byte stores) or pushed blocks of a thread

// A step's rows in LDS: exclusive prefix sums [rows + 1], and the state before
// it [rows].
struct StepRows {
  int32_t *tok, *take, *gone;
  int32_t *len, *held;
  __device__ __forceinline__ StepRows(int32_t *base, int rows)
      : tok(base), take(tok + rows + 1), gone(take + rows + 1), len(gone + rows + 1),
        held(len + rows) {}
};

size_t rows_bytes(int rows) { return (size_t)(5 * rows + 3) * 4; }

// What a step does in all.
struct StepTotals {
  int32_t tokens, take, gone;
  int32_t num_free;  // before the step
};

// Last row whose prefix is <= i (0 <= i < prefix[rows]): three candidates a round,
// as a round is the latency of its reads.
__device__ __forceinline__ int row_of(const int32_t *prefix, int rows, int i) {
  int lo = 0;
  for (int n = rows; n > 1;) {
    n = (n + 3) >> 2;
    int right = 0;
#pragma unroll
    for (int k = 1; k < 4; ++k) right += prefix[min(lo + k * n, rows)] <= i ? 1 : 0;
    lo += right * n;
  }
  return lo;
}

// Sums that stay at the largest value instead of wrapping: past every bound
// that a step is checked against.
__device__ __forceinline__ uint32_t add_sat(uint32_t a, uint32_t b) {
  return __builtin_elementwise_add_sat(a, b);
}
__device__ __forceinline__ uint32_t clamp32(int64_t x) {
  return (uint32_t)min(x, (int64_t)0xffffffff);
}

// Scans the rows into s and checks the step; `write`: also writes the state
// after it. All NT threads of the workgroup call it.
template <int NT>
__device__ StepTotals scan_step(const TablesParams &p, const StepRows &s, bool write) {
  __shared__ uint32_t s_sum[NT / 64][3];
  __shared__ int s_flags[NT / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  constexpr int kPer = (CLV_TABLES_MAX_ROWS + NT - 1) / NT;
  const int per = (p.rows + NT - 1) / NT;
  const int b = min(p.rows, tid * per), e = min(p.rows, b + per);
  const int F = p.num_free[0];
  // The thread's rows b .. e - 1 (past them: rows of nothing), read at once.
  int len[kPer], held[kPer], n[kPer];
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    len[k] = held[k] = n[k] = 0;
    if (b + k < e) {
      len[k] = p.context_lens[b + k];
      held[k] = p.blocks_held[b + k];
      n[k] = p.new_lens[b + k];
    }
  }
  auto need = [&](int k) {  // blocks of row b + k after the step
    const int64_t all = (int64_t)len[k] + n[k] + (held[k] == 0 ? p.reserve : 0);
    const int64_t blocks = (all + (1 << p.block_shift) - 1) >> p.block_shift;
    return n[k] > 0 ? max((int64_t)held[k], blocks) : (int64_t)held[k];
  };
  // Bit 0: a row longer than its table; bit 1: a state that cannot be.
  uint32_t x[3] = {0, 0, 0};
  int flags = F < 0 || F > p.num_blocks ? 2 : 0;
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    if (b + k >= e) break;
    if (need(k) > p.width) flags |= 1;
    if (len[k] < 0 || held[k] < 0 || held[k] > p.width ||
        len[k] > ((int64_t)held[k] << p.block_shift))
      flags |= 2;
    x[0] = add_sat(x[0], (uint32_t)max(n[k], 0));
    x[1] = add_sat(x[1], clamp32(need(k) - held[k]));
    x[2] = add_sat(x[2], (uint32_t)(n[k] < 0 ? max(held[k], 0) : 0));
  }
  const uint32_t own[3] = {x[0], x[1], x[2]};
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      const uint32_t y = __shfl_up(x[k], off, 64);
      if (lane >= off) x[k] = add_sat(x[k], y);
    }
    flags |= __shfl_xor(flags, off, 64);
  }
  if (lane == 63) {
#pragma unroll
    for (int k = 0; k < 3; ++k) s_sum[wave][k] = x[k];
    s_flags[wave] = flags;
  }
  __syncthreads();
  uint32_t run[3], all[3] = {0, 0, 0};  // run: of no use where a sum is at its end
#pragma unroll
  for (int k = 0; k < 3; ++k) run[k] = x[k] - own[k];
  flags = 0;
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) {
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      if (w < wave) run[k] += s_sum[w][k];
      all[k] = add_sat(all[k], s_sum[w][k]);
    }
    flags |= s_flags[w];
  }
  int status = CLV_TABLES_OK;
  if ((flags & 2) || (int64_t)F + all[2] > p.num_blocks) status = CLV_TABLES_BAD_STATE;
  else if ((int64_t)all[1] > (int64_t)F + all[2]) status = CLV_TABLES_NO_BLOCKS;
  else if (flags & 1) status = CLV_TABLES_ROW_FULL;
  else if ((int64_t)all[0] > p.num_tokens) status = CLV_TABLES_NO_SLOTS;
  const bool ok = status == CLV_TABLES_OK;
  StepTotals t;
  t.num_free = F;
  t.tokens = ok ? (int32_t)all[0] : 0;
  t.take = ok ? (int32_t)all[1] : 0;
  t.gone = ok ? (int32_t)all[2] : 0;
  // In place, a row's state is read and written by the same thread, and every
  // thread has read the stack's count before the barrier above.
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const int r = b + k;
    if (r >= e) break;
    s.tok[r] = ok ? (int32_t)run[0] : 0;
    s.take[r] = ok ? (int32_t)run[1] : 0;
    s.gone[r] = ok ? (int32_t)run[2] : 0;
    s.len[r] = len[k];
    s.held[r] = held[k];
    if (write) {
      p.query_start_loc[r] = ok ? (int32_t)run[0] : 0;
      p.context_lens_out[r] = !ok ? len[k] : n[k] < 0 ? 0 : len[k] + n[k];
      p.blocks_held_out[r] = !ok ? held[k] : n[k] < 0 ? 0 : (int32_t)need(k);
    }
    run[0] += max(n[k], 0);
    run[1] += (uint32_t)(need(k) - held[k]);
    run[2] += n[k] < 0 ? held[k] : 0;
  }
  if (tid == 0) {
    s.tok[p.rows] = t.tokens;
    s.take[p.rows] = t.take;
    s.gone[p.rows] = t.gone;
    if (write) {
      p.query_start_loc[p.rows] = t.tokens;
      p.num_free_out[0] = F + t.gone - t.take;
      p.status[0] = status;
    }
  }
  __syncthreads();
  return t;
}

// write: workgroup 0 writes the state; fill: the workgroups share the rest.
template <int NT>
__global__ void __launch_bounds__(NT) tables_step(const TablesParams p, bool write, bool fill) {
  extern __shared__ int32_t s_rows[];
  const StepRows s(s_rows, p.rows);
  const StepTotals t = scan_step<NT>(p, s, write && blockIdx.x == 0);
  if (!fill) return;
  const int F = t.num_free, R = t.gone, K = t.take;
  // Where block v of the stack V stands.
  auto stack = [&](int v) -> const int32_t * {
    if (v < F) return p.free_blocks + v;
    const int r = row_of(s.gone, p.rows, v - F);
    return p.block_tables + (int64_t)r * p.width + (v - F - s.gone[r]);
  };
  const int mask = (1 << p.block_shift) - 1;
  // One index space (slots in runs, taken blocks, pushed ones in runs), so that a
  // thread's items do not wait for each other.
  const int64_t runs = (p.num_tokens + kRun - 1) / kRun;
  const int left = max(0, R - K);
  const int64_t items = runs + K + (left + kRun - 1) / kRun;
  for (int64_t i = (int64_t)blockIdx.x * NT + threadIdx.x; i < items;
       i += (int64_t)gridDim.x * NT) {
    if (i >= runs + K) {
      const int k0 = (int)(i - runs - K) * kRun;
      int r = row_of(s.gone, p.rows, k0);
      int32_t blk[kRun];
#pragma unroll
      for (int u = 0; u < kRun; ++u) {
        const int k = min(k0 + u, left - 1);
        while (s.gone[r + 1] <= k) ++r;
        blk[u] = p.block_tables[(int64_t)r * p.width + (k - s.gone[r])];
      }
#pragma unroll
      for (int u = 0; u < kRun; ++u)
        if (k0 + u < left) p.free_blocks[F + k0 + u] = blk[u];
    } else if (i >= runs) {
      const int k = (int)(i - runs);
      const int r = row_of(s.take, p.rows, k);
      p.block_tables[(int64_t)r * p.width + s.held[r] + (k - s.take[r])] = *stack(F + R - 1 - k);
    } else {
      const int64_t i0 = i * kRun;
      // The entries' places first, so that their loads are in flight together.
      const int32_t *entry[kRun];
      int pos[kRun];
      int r = i0 < t.tokens ? row_of(s.tok, p.rows, (int)i0) : 0;
#pragma unroll
      for (int u = 0; u < kRun; ++u) {
        entry[u] = p.num_free;
        pos[u] = -1;
        if (i0 + u < t.tokens) {
          const int k = (int)i0 + u;
          while (s.tok[r + 1] <= k) ++r;
          pos[u] = s.len[r] + (k - s.tok[r]);
          const int col = pos[u] >> p.block_shift;
          if (u > 0 && col == (pos[u - 1] >> p.block_shift) && s.tok[r] < k)
            entry[u] = entry[u - 1];  // the block of the token before it
          else if (col < s.held[r])
            entry[u] = p.block_tables + (int64_t)r * p.width + col;
          else
            entry[u] = stack(F + R - 1 - (s.take[r] + col - s.held[r]));
        }
      }
      int64_t slot[kRun];
#pragma unroll
      for (int u = 0; u < kRun; ++u) slot[u] = *entry[u];
#pragma unroll
      for (int u = 0; u < kRun; ++u)
        slot[u] = pos[u] < 0 ? -1 : (slot[u] << p.block_shift) + (pos[u] & mask);
      typedef int64_t i64x2 __attribute__((ext_vector_type(2)));
      int64_t *dst = p.slot_mapping + i0;
      if (i0 + kRun <= p.num_tokens && ((uintptr_t)dst & 15u) == 0) {
        store_vec<i64x2>(dst, (i64x2){slot[0], slot[1]});
        store_vec<i64x2>(dst + 2, (i64x2){slot[2], slot[3]});
      } else {
#pragma unroll
        for (int u = 0; u < kRun; ++u)
          if (i0 + u < p.num_tokens) dst[u] = slot[u];
      }
    }
  }
}

// In place, the state may only be written when every workgroup has read it:
// up to this many tokens one workgroup serves the step, above it a second
// launch writes the state. One workgroup / two launches, us, 32 rows: 1024 tokens
// 4.8/6.7, 4096 5.5/6.9, 8192 7.1/7.2, 16384 10.8/7.5; 256 rows the same within 0.8.
constexpr int64_t kInPlaceTokens = 8192;

}  // namespace

hipError_t launch_tables(const TablesParams &p, hipStream_t stream) {
  const bool in_place = p.blocks_held_out == p.blocks_held ||
                        p.context_lens_out == p.context_lens || p.num_free_out == p.num_free;
  const size_t lds = rows_bytes(p.rows);
  if (in_place && p.num_tokens <= kInPlaceTokens) {
    hipLaunchKernelGGL(tables_step<1024>, dim3(1), dim3(1024), lds, stream, p, true, true);
    return hipGetLastError();
  }
  // Workgroups for the slots, and two more for the blocks.
  constexpr int NT = 256;
  int64_t groups = p.num_tokens / (kRun * NT) + 3;
  if (groups > 1024) groups = 1024;
  hipLaunchKernelGGL(tables_step<NT>, dim3((unsigned)groups), dim3(NT), lds, stream, p, !in_place,
                     true);
  if (in_place)
    hipLaunchKernelGGL(tables_step<NT>, dim3(1), dim3(NT), lds, stream, p, true, false);
  return hipGetLastError();
}

}  // namespace clv
