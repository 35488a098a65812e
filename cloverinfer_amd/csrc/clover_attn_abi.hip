// clover_attn_abi.hip - the extern "C" boundary declared in include/clover_attn.h.
//
// Validates every argument block, turns it into the kernels' parameter
// structs and dispatches. Nothing here allocates device memory; the only
// state kept between calls is per-device: the compute-unit count and the
// address of the fixed scratch array of clv_paged_decode_balanced_noalloc.
// Errors come back as status codes.
#include <math.h>
#include <stddef.h>
#include <stdlib.h>

#include <algorithm>
#include <atomic>
#include <mutex>

#include "clover_attn.h"
#include "clv_internal.h"

namespace {

using clv::DType;

bool is_pow2(int64_t x) { return x > 0 && (x & (x - 1)) == 0; }

int log2_int(int64_t x) {
  int r = 0;
  while ((int64_t(1) << r) < x) ++r;
  return r;
}

bool supported_head_dim(int d) {
  return d == 8 || d == 16 || d == 32 || d == 64 || d == 128 || d == 256;
}

int elem_bytes(int dtype) { return dtype == CLV_F32 ? 4 : 2; }

bool aligned16(const void *p) { return ((uintptr_t)p & 15u) == 0; }

bool stride16(int64_t stride, int eb) { return (stride * eb) % 16 == 0; }

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

size_t round256(size_t x) { return (x + 255) & ~(size_t)255; }

// Compute units of the current device, queried once per device and cached
// (the default wave counts depend on it). 0 is "not queried yet"; a failed
// query answers 256 (MI355X) without caching.
constexpr int kMaxDevices = 64;
std::atomic<int> g_device_cus[kMaxDevices];

int device_compute_units() {
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0) return 256;
  if (dev < kMaxDevices) {
    const int c = g_device_cus[dev].load(std::memory_order_relaxed);
    if (c > 0) return c;
  }
  int cus = 0;
  if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess ||
      cus <= 0)
    return 256;
  if (dev < kMaxDevices) g_device_cus[dev].store(cus, std::memory_order_relaxed);
  return cus;
}

// Fixed scratch of clv_paged_decode_balanced_noalloc: the balanced decode's
// workspace (segment prefix sums and per-wave partials) for callers that
// cannot allocate. Every GPU the library runs on holds one copy for the life
// of the process. In host code `scratch` names a host-side stand-in, never
// the device array: only the address hipGetSymbolAddress returns for the
// current device (scratch_address) may reach a kernel.
static __device__ __align__(256) unsigned char scratch[CLV_NOALLOC_SCRATCH_BYTES];

std::atomic<void *> g_scratch_dev[kMaxDevices];
std::mutex g_scratch_mu;

// Device address of the current device's scratch array, looked up once per
// device (with that device current) and kept; CLV_ELAUNCH if the runtime
// cannot resolve it.
int scratch_address(void **out) {
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= kMaxDevices) return CLV_ELAUNCH;
  void *ptr = g_scratch_dev[dev].load(std::memory_order_acquire);
  if (ptr == nullptr) {
    std::lock_guard<std::mutex> lock(g_scratch_mu);
    ptr = g_scratch_dev[dev].load(std::memory_order_relaxed);
    if (ptr == nullptr) {
      if (hipGetSymbolAddress(&ptr, HIP_SYMBOL(scratch)) != hipSuccess || ptr == nullptr)
        return CLV_ELAUNCH;
      g_scratch_dev[dev].store(ptr, std::memory_order_release);
    }
  }
  *out = ptr;
  return CLV_OK;
}

// Validates a decode argument block and fills the kernel parameters.
int fill_decode(const clv_decode_args *a, clv::DecodeParams *p) {
  if (a == nullptr) return CLV_EINVAL;
  if (a->dtype != CLV_F32 && a->dtype != CLV_F16 && a->dtype != CLV_BF16) return CLV_EINVAL;
  if (a->num_seqs < 0 || a->num_heads <= 0 || a->num_kv_heads <= 0 || a->head_dim <= 0)
    return CLV_EINVAL;
  if (a->num_heads % a->num_kv_heads != 0) return CLV_EINVAL;
  if (!is_pow2(a->block_size)) return CLV_EUNSUPPORTED;
  if (!supported_head_dim(a->head_dim)) return CLV_EUNSUPPORTED;
  if (a->max_blocks_per_seq < 0 || a->max_context_len < 0 || a->num_blocks <= 0) return CLV_EINVAL;
  if (!isfinite(a->scale)) return CLV_EINVAL;
  if (a->num_seqs > 65535) return CLV_EUNSUPPORTED;  // grid z limit
  const int eb = elem_bytes(a->dtype);
  if (a->num_seqs > 0) {
    if (!a->out || !a->q || !a->k_cache || !a->v_cache || !a->context_lens) return CLV_EINVAL;
    if (a->max_blocks_per_seq > 0 && !a->block_tables) return CLV_EINVAL;
    if (!aligned16(a->out) || !aligned16(a->q) || !aligned16(a->k_cache) || !aligned16(a->v_cache))
      return CLV_EINVAL;
    if (!stride16(a->q_stride_seq, eb) || !stride16(a->q_stride_head, eb) ||
        !stride16(a->out_stride_seq, eb) || !stride16(a->out_stride_head, eb) ||
        !stride16(a->kv_stride_block, eb) || !stride16(a->kv_stride_token, eb) ||
        !stride16(a->kv_stride_head, eb))
      return CLV_EINVAL;
  }
  *p = clv::DecodeParams{};
  p->out = a->out;
  p->q = a->q;
  p->k_cache = a->k_cache;
  p->v_cache = a->v_cache;
  p->block_tables = a->block_tables;
  p->context_lens = a->context_lens;
  p->q_stride_seq = a->q_stride_seq;
  p->q_stride_head = a->q_stride_head;
  p->out_stride_seq = a->out_stride_seq;
  p->out_stride_head = a->out_stride_head;
  p->kv_stride_block = a->kv_stride_block;
  p->kv_stride_token = a->kv_stride_token;
  p->kv_stride_head = a->kv_stride_head;
  p->num_seqs = a->num_seqs;
  p->num_heads = a->num_heads;
  p->num_kv_heads = a->num_kv_heads;
  p->head_dim = a->head_dim;
  p->group = a->num_heads / a->num_kv_heads;
  p->n_gchunks = (int32_t)ceil_div(p->group, 16);
  p->block_shift = log2_int(a->block_size);
  p->max_blocks_per_seq = a->max_blocks_per_seq;
  p->max_context_len = a->max_context_len;
  p->num_blocks = a->num_blocks;
  p->scale_log2 = a->scale * 1.4426950408889634f;
  return CLV_OK;
}

// Longest context for which clv_paged_decode_append runs the single pass
// (the schedule the Python layer picks for such batches: no merge launch).
constexpr int32_t kAppendSinglePassMaxLen = 512;

int launch_decode(const clv::DecodeParams &p, int dtype, int block_size, hipStream_t stream) {
  const DType dt = (DType)dtype;
  hipError_t err;
  if (clv::decode_mfma_supported(dt, p.head_dim, block_size))
    err = clv::launch_decode_mfma(p, dt, stream);
  else
    err = clv::launch_decode_valu(p, dt, stream);
  return err == hipSuccess ? CLV_OK : CLV_ELAUNCH;
}

}  // namespace

extern "C" {

int clv_abi_version(void) { return CLV_ABI_VERSION; }

const char *clv_status_string(int status) {
  switch (status) {
    case CLV_OK: return "ok";
    case CLV_EINVAL: return "invalid argument (shape, stride, alignment, pointer or dtype)";
    case CLV_EUNSUPPORTED: return "unsupported configuration (head_dim, block_size or size limit)";
    case CLV_ELAUNCH: return "kernel launch failed";
    case CLV_EWORKSPACE: return "split-K workspace missing, misaligned or too small";
    case CLV_ESCRATCH:
      return "problem needs more than the fixed scratch of the no-allocation entry point "
             "(CLV_NOALLOC_SCRATCH_BYTES)";
    default: return "unknown status";
  }
}

int clv_reshape_and_cache(const clv_cache_args *a, clv_stream_t stream) {
  if (a == nullptr) return CLV_EINVAL;
  if (a->dtype != CLV_F32 && a->dtype != CLV_F16 && a->dtype != CLV_BF16) return CLV_EINVAL;
  if (a->num_tokens < 0 || a->num_kv_heads <= 0 || a->head_dim <= 0 || a->num_blocks <= 0)
    return CLV_EINVAL;
  if (!is_pow2(a->block_size)) return CLV_EUNSUPPORTED;
  if (a->num_tokens == 0) return CLV_OK;
  if (!a->key || !a->value || !a->k_cache || !a->v_cache || !a->slot_mapping) return CLV_EINVAL;
  clv::CacheParams p{};
  p.key = a->key;
  p.value = a->value;
  p.k_cache = a->k_cache;
  p.v_cache = a->v_cache;
  p.slot_mapping = a->slot_mapping;
  p.key_stride_token = a->key_stride_token;
  p.key_stride_head = a->key_stride_head;
  p.value_stride_token = a->value_stride_token;
  p.value_stride_head = a->value_stride_head;
  p.kv_stride_block = a->kv_stride_block;
  p.kv_stride_token = a->kv_stride_token;
  p.kv_stride_head = a->kv_stride_head;
  p.num_tokens = a->num_tokens;
  p.num_kv_heads = a->num_kv_heads;
  p.head_dim = a->head_dim;
  p.block_shift = log2_int(a->block_size);
  p.num_blocks = a->num_blocks;
  p.num_slots = (int64_t)a->num_blocks * a->block_size;
  p.elem_bytes = elem_bytes(a->dtype);
  return clv::launch_reshape_and_cache(p, (hipStream_t)stream) == hipSuccess ? CLV_OK
                                                                              : CLV_ELAUNCH;
}

int clv_reshape_and_cache_fp8(const clv_cache_args *a, const float *k_scales,
                              const float *v_scales, clv_stream_t stream) {
  if (a == nullptr) return CLV_EINVAL;
  if (a->dtype != CLV_F32 && a->dtype != CLV_F16 && a->dtype != CLV_BF16) return CLV_EINVAL;
  if (a->num_tokens < 0 || a->num_kv_heads <= 0 || a->head_dim <= 0 || a->num_blocks <= 0)
    return CLV_EINVAL;
  if (!is_pow2(a->block_size)) return CLV_EUNSUPPORTED;
  if (a->head_dim % 8 != 0) return CLV_EUNSUPPORTED;
  if (a->num_tokens == 0) return CLV_OK;
  if (!a->key || !a->value || !a->k_cache || !a->v_cache || !a->slot_mapping || !k_scales ||
      !v_scales)
    return CLV_EINVAL;
  // fp8 pools: one byte per element, rows written 8 bytes at a time.
  if (((uintptr_t)a->k_cache & 7u) || ((uintptr_t)a->v_cache & 7u) || (a->kv_stride_block & 7) ||
      (a->kv_stride_token & 7) || (a->kv_stride_head & 7))
    return CLV_EINVAL;
  clv::CacheParams p{};
  p.key = a->key;
  p.value = a->value;
  p.k_cache = a->k_cache;
  p.v_cache = a->v_cache;
  p.slot_mapping = a->slot_mapping;
  p.key_stride_token = a->key_stride_token;
  p.key_stride_head = a->key_stride_head;
  p.value_stride_token = a->value_stride_token;
  p.value_stride_head = a->value_stride_head;
  p.kv_stride_block = a->kv_stride_block;
  p.kv_stride_token = a->kv_stride_token;
  p.kv_stride_head = a->kv_stride_head;
  p.num_tokens = a->num_tokens;
  p.num_kv_heads = a->num_kv_heads;
  p.head_dim = a->head_dim;
  p.block_shift = log2_int(a->block_size);
  p.num_blocks = a->num_blocks;
  p.num_slots = (int64_t)a->num_blocks * a->block_size;
  p.elem_bytes = elem_bytes(a->dtype);
  return clv::launch_reshape_and_cache_fp8(p, a->dtype, k_scales, v_scales, (hipStream_t)stream) ==
                 hipSuccess
             ? CLV_OK
             : CLV_ELAUNCH;
}

int clv_paged_decode(const clv_decode_args *a, clv_stream_t stream) {
  clv::DecodeParams p;
  const int st = fill_decode(a, &p);
  if (st != CLV_OK) return st;
  if (p.num_seqs == 0) return CLV_OK;
  p.partition_size = 0;
  return launch_decode(p, a->dtype, a->block_size, (hipStream_t)stream);
}

size_t clv_splitk_workspace_bytes(int32_t num_seqs, int32_t num_heads, int32_t head_dim,
                                  int32_t max_context_len, int32_t partition_size) {
  if (num_seqs <= 0 || num_heads <= 0 || head_dim <= 0 || partition_size <= 0 ||
      max_context_len < 0)
    return 0;
  const size_t parts = (size_t)(max_context_len > 0 ? ceil_div(max_context_len, partition_size) : 1);
  const size_t rows = (size_t)num_seqs * (size_t)num_heads * parts;
  return round256(rows * (size_t)head_dim * 4) + 2 * round256(rows * 4);
}

}  // extern "C"

namespace {

// Fills the split-K fields of p from the workspace; CLV_OK or an error.
int head_group(int num_kv_heads, int num_waves);
int stream_depth_setting(int def);

int fill_splitk(const clv_decode_args *a, int32_t partition_size, const void *workspace,
                size_t workspace_bytes, clv::DecodeParams *p) {
  if (partition_size <= 0 || partition_size % 32 != 0) return CLV_EINVAL;
  const size_t need = clv_splitk_workspace_bytes(a->num_seqs, a->num_heads, a->head_dim,
                                                 a->max_context_len, partition_size);
  if (workspace == nullptr || workspace_bytes < need || ((uintptr_t)workspace & 255u) != 0)
    return CLV_EWORKSPACE;
  const int64_t parts = a->max_context_len > 0 ? ceil_div(a->max_context_len, partition_size) : 1;
  if (parts > 65535) return CLV_EUNSUPPORTED;
  const size_t rows = (size_t)a->num_seqs * (size_t)a->num_heads * (size_t)parts;
  char *ws = (char *)workspace;
  p->partition_size = partition_size;
  p->max_parts = (int32_t)parts;
  p->ws_o = (float *)ws;
  p->ws_m = (float *)(ws + round256(rows * (size_t)a->head_dim * 4));
  p->ws_l = (float *)(ws + round256(rows * (size_t)a->head_dim * 4) + round256(rows * 4));
  return CLV_OK;
}

}  // namespace

extern "C" {

int clv_paged_decode_partials(const clv_decode_args *a, int32_t partition_size, void *workspace,
                              size_t workspace_bytes, clv_stream_t stream) {
  clv::DecodeParams p;
  int st = fill_decode(a, &p);
  if (st != CLV_OK) return st;
  if (p.num_seqs == 0) return partition_size > 0 && partition_size % 32 == 0 ? CLV_OK : CLV_EINVAL;
  st = fill_splitk(a, partition_size, workspace, workspace_bytes, &p);
  if (st != CLV_OK) return st;
  // The partitions on the balanced stream kernel where it covers the shape:
  // its waves split the batch's partitions evenly and stream each run of
  // consecutive partitions through one ring (16 x 32K-token fp16, partition
  // 512: 339 -> 316 us), writing the same partials as the grid kernel below.
  const int64_t nseg = (int64_t)p.num_seqs * p.num_kv_heads * p.n_gchunks;
  if (clv::decode_stream_supported((DType)a->dtype, a->head_dim, a->block_size, nseg)) {
    const int nw = clv_default_num_waves();
    const int hg = head_group(p.num_kv_heads, nw);
    p.num_waves = nw;
    p.head_group = hg;
    p.stream_depth = stream_depth_setting(a->dtype == CLV_F32 ? 2 : 3);
    p.stream_run_cost = 0;
    p.num_segments = (int32_t)(nseg / hg);
    return clv::launch_decode_stream(p, (DType)a->dtype, (hipStream_t)stream) == hipSuccess
               ? CLV_OK
               : CLV_ELAUNCH;
  }
  return launch_decode(p, a->dtype, a->block_size, (hipStream_t)stream);
}

int clv_splitk_reduce(const clv_decode_args *a, int32_t partition_size, const void *workspace,
                      size_t workspace_bytes, clv_stream_t stream) {
  clv::DecodeParams p;
  int st = fill_decode(a, &p);
  if (st != CLV_OK) return st;
  if (p.num_seqs == 0) return partition_size > 0 && partition_size % 32 == 0 ? CLV_OK : CLV_EINVAL;
  st = fill_splitk(a, partition_size, workspace, workspace_bytes, &p);
  if (st != CLV_OK) return st;
  return clv::launch_splitk_reduce(p, (DType)a->dtype, (hipStream_t)stream) == hipSuccess
             ? CLV_OK
             : CLV_ELAUNCH;
}

int clv_paged_decode_splitk(const clv_decode_args *a, int32_t partition_size, void *workspace,
                            size_t workspace_bytes, clv_stream_t stream) {
  clv::DecodeParams p;
  const int st = fill_decode(a, &p);
  if (st != CLV_OK) return st;
  if (partition_size <= 0 || partition_size % 32 != 0) return CLV_EINVAL;
  if (p.num_seqs == 0) return CLV_OK;
  // A context that fits one partition needs no merge.
  if (a->max_context_len <= partition_size) {
    p.partition_size = 0;
    return launch_decode(p, a->dtype, a->block_size, (hipStream_t)stream);
  }
  const int rc = clv_paged_decode_partials(a, partition_size, workspace, workspace_bytes, stream);
  if (rc != CLV_OK) return rc;
  return clv_splitk_reduce(a, partition_size, workspace, workspace_bytes, stream);
}

int32_t clv_default_num_waves(void) {
  // One wave per SIMD (4 per compute unit), each keeping three steps of
  // loads in flight: on MI355X this streams the paged cache faster than more
  // waves with shallower pipelines.
  return device_compute_units() * 4;
}

int32_t clv_default_num_waves_fp8(void) { return 2 * clv_default_num_waves(); }

size_t clv_balanced_workspace_bytes(int32_t num_seqs, int32_t num_heads, int32_t num_kv_heads,
                                    int32_t head_dim, int32_t num_waves) {
  if (num_seqs <= 0 || num_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0 ||
      num_heads % num_kv_heads != 0)
    return 0;
  if (num_waves <= 0) num_waves = clv_default_num_waves();
  const int64_t group = num_heads / num_kv_heads;
  const size_t nseg = (size_t)num_seqs * (size_t)num_kv_heads * (size_t)ceil_div(group, 16);
  const size_t rows = ((size_t)num_waves + nseg) * 16;
  return round256((nseg + 1) * 4) + 2 * round256(rows * 4) + round256(rows * (size_t)head_dim * 4);
}

}  // extern "C"

namespace {

// Ring depth of the balanced decode: steps of loads each wave keeps in
// flight (2, 3, 4 or 6): three for 16-bit and fp8 pools, two for fp32 pools
// (twice the bytes per step). Fixed at build time; a tuning build may set
// CLV_STREAM_DEPTH (a preprocessor value) to force one depth for every dtype.
int stream_depth_setting(int def) {
#ifdef CLV_STREAM_DEPTH
  (void)def;
  static_assert(CLV_STREAM_DEPTH == 2 || CLV_STREAM_DEPTH == 3 || CLV_STREAM_DEPTH == 4 ||
                    CLV_STREAM_DEPTH == 6,
                "ring depth 2, 3, 4 or 6");
  return CLV_STREAM_DEPTH;
#else
  return def;
#endif
}

// Phantom steps the balanced decode charges for each segment a wave starts
// (a run start costs one memory latency: measured per-wave durations grow by
// ~2.5 us per extra run). With head groups 4 measured best (GQA-7B batch:
// 172.9 us at 2, 172.3 at 4, 173.5 at 6, 173.9 at 8). Fixed at build time
// (preprocessor value CLV_STREAM_RUN_COST, default 4).
#ifndef CLV_STREAM_RUN_COST
#define CLV_STREAM_RUN_COST 4
#endif
static_assert(CLV_STREAM_RUN_COST >= 0 && CLV_STREAM_RUN_COST <= 64, "run cost 0..64 steps");
constexpr int kStreamRunCost = CLV_STREAM_RUN_COST;

// Steps per group of each dispatch slot of the balanced decode, times 256
// against the last slot, when the grid is two or three workgroups (of four
// waves) per compute unit (see StreamSplit in decode_stream.hip); all 256 is
// the even split. fp8 GQA-7B batch, wave end times read from the realtime
// counter: at 2048 waves and equal spans the second-slot waves end 5.3 us
// after the first-slot ones on average; at 282 (1.10) both slots end within
// 0.5 us of each other, the launch span falls from 87.5 to 86.7 us and
// back-to-back launches from 91.2-92.0 to 89.3-90.3 us (320 and 345: slower
// than 256). At 3072 waves the three slots end at 71.6, 78.8 and 86.4 us on
// average with equal spans; back to back (another box): 99.3-99.6 us at
// 256/256, 98.0-98.7 at 282/269, 96.7-97.1 at 300/278, 96.1-96.2 at
// 320/288, 96.4-96.8 at 345/300 (2048 waves there: 95.4-96.3, and per step
// 0.0981 against 0.1045 ms, the merge reading more partials, so the fp8
// default stays at two slots). Fixed at build time (preprocessor values
// CLV_STREAM_SLOT2_Q8 for the first of two slots, CLV_STREAM_SLOT3_Q8_0 and
// _1 for the first two of three).
#ifndef CLV_STREAM_SLOT2_Q8
#define CLV_STREAM_SLOT2_Q8 282
#endif
#ifndef CLV_STREAM_SLOT3_Q8_0
#define CLV_STREAM_SLOT3_Q8_0 320
#endif
#ifndef CLV_STREAM_SLOT3_Q8_1
#define CLV_STREAM_SLOT3_Q8_1 288
#endif
static_assert(CLV_STREAM_SLOT2_Q8 >= 128 && CLV_STREAM_SLOT2_Q8 <= 512 &&
                  CLV_STREAM_SLOT3_Q8_0 >= 128 && CLV_STREAM_SLOT3_Q8_0 <= 512 &&
                  CLV_STREAM_SLOT3_Q8_1 >= 128 && CLV_STREAM_SLOT3_Q8_1 <= 512,
              "slot weights 0.5..2");
constexpr int kSlotQ8[2][3] = {{CLV_STREAM_SLOT2_Q8, 256, 256},
                               {CLV_STREAM_SLOT3_Q8_0, CLV_STREAM_SLOT3_Q8_1, 256}};

// kv heads that one workgroup of the balanced decode reads together (one
// wave each): all of them up to four (a token's whole row of the pools; GQA-7B
// batch, 4 kv heads: 175.3 -> 173.1 us), else pairs (MHA Llama-7B batch, 32
// kv heads: 329.0 -> 326.9 us with pairs, 336.4 with fours). A tuning build
// may cap the group with the preprocessor value CLV_HEAD_GROUP_MAX.
#ifndef CLV_HEAD_GROUP_MAX
#define CLV_HEAD_GROUP_MAX 4
#endif
static_assert(CLV_HEAD_GROUP_MAX == 1 || CLV_HEAD_GROUP_MAX == 2 || CLV_HEAD_GROUP_MAX == 4,
              "head group 1, 2 or 4");
int head_group(int num_kv_heads, int num_waves) {
  int hg = num_kv_heads <= 4 ? num_kv_heads : 2;
  hg = std::min(hg, CLV_HEAD_GROUP_MAX);
  if (hg == 3 || num_kv_heads % hg != 0) hg = 1;
  while (hg > num_waves) hg /= 2;
  return std::max(hg, 1);
}

// Validates a balanced-decode call and lays the workspace out in p. diff: a
// differential decode, `a` counting the rows of both maps as heads.
int fill_balanced(const clv_decode_args *a, int32_t num_waves, void *workspace,
                  size_t workspace_bytes, clv::DecodeParams *p, bool diff = false) {
  const int st = fill_decode(a, p);
  if (st != CLV_OK) return st;
  if (num_waves <= 0) num_waves = clv_default_num_waves();
  if (num_waves > (1 << 22)) return CLV_EINVAL;
  const int64_t nseg = (int64_t)p->num_seqs * p->num_kv_heads * p->n_gchunks;
  const int hg = head_group(p->num_kv_heads, num_waves);
  if (diff ? !clv::diff_decode_mfma_supported(a->head_dim, a->block_size) ||
                 nseg > clv::kStreamMaxSegments
           : !clv::decode_stream_supported((DType)a->dtype, a->head_dim, a->block_size, nseg))
    return CLV_EUNSUPPORTED;
  if (p->num_seqs == 0) return CLV_OK;
  const size_t need = clv_balanced_workspace_bytes(a->num_seqs, a->num_heads, a->num_kv_heads,
                                                   a->head_dim, num_waves);
  if (workspace == nullptr || workspace_bytes < need || ((uintptr_t)workspace & 255u) != 0)
    return CLV_EWORKSPACE;
  const size_t rows = ((size_t)num_waves + (size_t)nseg) * 16;
  char *ws = (char *)workspace;
  p->num_waves = num_waves;
  p->head_group = hg;
  // fp32 steps are twice the bytes: two steps in flight (a sweep over 2-4).
  p->stream_depth = stream_depth_setting(a->dtype == CLV_F32 ? 2 : 3);
  p->stream_run_cost = kStreamRunCost;
  p->num_segments = (int32_t)(nseg / hg);
  // Two or three workgroups (of four waves) per compute unit: one piece of
  // the split per dispatch slot, the older slots taking more steps
  // (decode_stream.hip, StreamSplit). Partials and merge derive the same
  // split from num_waves.
  const int cus = device_compute_units();
  for (int slots = 2; slots <= 3; ++slots) {
    if (num_waves != slots * 4 * cus) continue;
    p->slot_count = slots;
    p->slot_groups = 4 * cus / hg;
    for (int k = 0; k < slots; ++k) p->slot_q8[k] = kSlotQ8[slots - 2][k];
  }
  p->seg_prefix = (int32_t *)ws;
  ws += round256(((size_t)nseg + 1) * 4);
  p->ws_m = (float *)ws;
  ws += round256(rows * 4);
  p->ws_l = (float *)ws;
  ws += round256(rows * 4);
  p->ws_o = (float *)ws;
  return CLV_OK;
}

}  // namespace

extern "C" {

int clv_balanced_partials(const clv_decode_args *a, int32_t num_waves, void *workspace,
                          size_t workspace_bytes, clv_stream_t stream) {
  clv::DecodeParams p;
  const int st = fill_balanced(a, num_waves, workspace, workspace_bytes, &p);
  if (st != CLV_OK || p.num_seqs == 0) return st;
  return clv::launch_decode_stream(p, (DType)a->dtype, (hipStream_t)stream) == hipSuccess
             ? CLV_OK
             : CLV_ELAUNCH;
}

int clv_balanced_reduce(const clv_decode_args *a, int32_t num_waves, const void *workspace,
                        size_t workspace_bytes, clv_stream_t stream) {
  clv::DecodeParams p;
  const int st = fill_balanced(a, num_waves, const_cast<void *>(workspace), workspace_bytes, &p);
  if (st != CLV_OK || p.num_seqs == 0) return st;
  return clv::launch_stream_reduce(p, (DType)a->dtype, (hipStream_t)stream) == hipSuccess
             ? CLV_OK
             : CLV_ELAUNCH;
}

int clv_paged_decode_balanced(const clv_decode_args *a, int32_t num_waves, void *workspace,
                              size_t workspace_bytes, clv_stream_t stream) {
  const int rc = clv_balanced_partials(a, num_waves, workspace, workspace_bytes, stream);
  if (rc != CLV_OK) return rc;
  return clv_balanced_reduce(a, num_waves, workspace, workspace_bytes, stream);
}

int clv_paged_decode_balanced_noalloc(const clv_decode_args *a, int32_t num_waves,
                                      clv_stream_t stream) {
  if (a == nullptr) return CLV_EINVAL;
  if (num_waves <= 0) num_waves = clv_default_num_waves();
  // 0 for arguments the balanced decode refuses anyway (it reports them).
  const size_t need = clv_balanced_workspace_bytes(a->num_seqs, a->num_heads, a->num_kv_heads,
                                                   a->head_dim, num_waves);
  if (need > (size_t)CLV_NOALLOC_SCRATCH_BYTES) return CLV_ESCRATCH;
  void *ws = nullptr;
  if (need > 0 && a->num_seqs > 0) {
    const int st = scratch_address(&ws);
    if (st != CLV_OK) return st;
  }
  // The stream kernel writes the prefix sums and every partial the merge
  // reads before it reads them: nothing in the scratch has to start at zero.
  return clv_paged_decode_balanced(a, num_waves, ws, (size_t)CLV_NOALLOC_SCRATCH_BYTES, stream);
}

int clv_paged_decode_append(const clv_decode_args *a, const void *key_new, const void *value_new,
                            int64_t new_stride_seq, int64_t new_stride_head, int32_t num_waves,
                            void *workspace, size_t workspace_bytes, clv_stream_t stream) {
  clv::DecodeParams p;
  // Short contexts (the single-pass schedule's range) with at most 16 query
  // heads per kv head: one grid launch that appends and attends, no merge.
  if (a != nullptr && num_waves <= 0 && a->max_context_len <= kAppendSinglePassMaxLen &&
      a->num_kv_heads > 0 && a->num_heads % a->num_kv_heads == 0 &&
      a->num_heads / a->num_kv_heads <= 16 &&
      clv::decode_mfma_supported((DType)a->dtype, a->head_dim, a->block_size)) {
    const int st = fill_decode(a, &p);
    if (st != CLV_OK || p.num_seqs == 0) return st;
    const int eb = elem_bytes(a->dtype);
    if (!key_new || !value_new || !aligned16(key_new) || !aligned16(value_new) ||
        !stride16(new_stride_seq, eb) || !stride16(new_stride_head, eb))
      return CLV_EINVAL;
    p.partition_size = 0;
    p.key_new = key_new;
    p.value_new = value_new;
    p.new_stride_seq = new_stride_seq;
    p.new_stride_head = new_stride_head;
    return clv::launch_decode_mfma_append(p, (DType)a->dtype, (hipStream_t)stream) == hipSuccess
               ? CLV_OK
               : CLV_ELAUNCH;
  }
  const int st = fill_balanced(a, num_waves, workspace, workspace_bytes, &p);
  if (st != CLV_OK || p.num_seqs == 0) return st;
  const int eb = elem_bytes(a->dtype);
  if (!key_new || !value_new || !aligned16(key_new) || !aligned16(value_new) ||
      !stride16(new_stride_seq, eb) || !stride16(new_stride_head, eb))
    return CLV_EINVAL;
  p.key_new = key_new;
  p.value_new = value_new;
  p.new_stride_seq = new_stride_seq;
  p.new_stride_head = new_stride_head;
  const hipStream_t s = (hipStream_t)stream;
  if (clv::stream_appends_in_kernel((DType)a->dtype, a->head_dim, a->block_size, p.group)) {
    p.append_new = 1;
  } else if (clv::launch_append_by_table(p, eb, s) != hipSuccess) {
    return CLV_ELAUNCH;
  }
  if (clv::launch_decode_stream(p, (DType)a->dtype, s) != hipSuccess) return CLV_ELAUNCH;
  return clv::launch_stream_reduce(p, (DType)a->dtype, s) == hipSuccess ? CLV_OK : CLV_ELAUNCH;
}

int clv_balanced_reduce_append(const clv_decode_args *a, const void *key_new,
                               const void *value_new, int64_t new_stride_seq,
                               int64_t new_stride_head, const int64_t *slot_mapping,
                               int32_t num_waves, const void *workspace, size_t workspace_bytes,
                               clv_stream_t stream) {
  clv::DecodeParams p;
  const int st = fill_balanced(a, num_waves, const_cast<void *>(workspace), workspace_bytes, &p);
  if (st != CLV_OK || p.num_seqs == 0) return st;
  const int eb = elem_bytes(a->dtype);
  if (!key_new || !value_new || !slot_mapping || !aligned16(key_new) || !aligned16(value_new) ||
      !stride16(new_stride_seq, eb) || !stride16(new_stride_head, eb))
    return CLV_EINVAL;
  p.key_new = key_new;
  p.value_new = value_new;
  p.new_stride_seq = new_stride_seq;
  p.new_stride_head = new_stride_head;
  p.slot_mapping = slot_mapping;
  return clv::launch_stream_reduce_append(p, (DType)a->dtype, (hipStream_t)stream) == hipSuccess
             ? CLV_OK
             : CLV_ELAUNCH;
}

int clv_paged_decode_fp8(const clv_decode_args *a, const float *k_scales, const float *v_scales,
                         int32_t num_waves, void *workspace, size_t workspace_bytes,
                         clv_stream_t stream) {
  if (num_waves <= 0) num_waves = clv_default_num_waves_fp8();
  const int rc = clv_paged_decode_fp8_partials(a, k_scales, v_scales, num_waves, workspace,
                                               workspace_bytes, stream);
  if (rc != CLV_OK) return rc;
  return clv_balanced_reduce(a, num_waves, workspace, workspace_bytes, stream);
}

int clv_paged_decode_fp8_partials(const clv_decode_args *a, const float *k_scales,
                                  const float *v_scales, int32_t num_waves, void *workspace,
                                  size_t workspace_bytes, clv_stream_t stream) {
  if (a == nullptr) return CLV_EINVAL;
  if (a->dtype != CLV_F16 && a->dtype != CLV_BF16) return CLV_EINVAL;
  if (a->head_dim != 128 || a->block_size < 16) return CLV_EUNSUPPORTED;
  // The wave count sets the partial layout that clv_balanced_reduce reads,
  // whose own default differs: it must be explicit here.
  if (num_waves <= 0) return CLV_EINVAL;
  clv::DecodeParams p;
  const int st = fill_balanced(a, num_waves, workspace, workspace_bytes, &p);
  if (st != CLV_OK || p.num_seqs == 0) return st;
  if (!k_scales || !v_scales) return CLV_EINVAL;
  // fp8 pools: strides are bytes; each lane reads 8-byte row chunks.
  if ((a->kv_stride_block & 15) || (a->kv_stride_token & 15) || (a->kv_stride_head & 15))
    return CLV_EINVAL;
  // Half the bytes per step make the per-step compute the longer part: two
  // waves per SIMD (clv_default_num_waves_fp8) with three steps in flight
  // (GQA-7B batch: step 0.0979 ms at depth 3, 0.0991 at depth 4; 2560 or
  // 3072 waves at depth 3, 3072 or 4096 at depth 2: slower).
  p.stream_depth = stream_depth_setting(3);
  p.kv_fp8 = 1;
  p.k_scales = k_scales;
  p.v_scales = v_scales;
  return clv::launch_decode_stream(p, (DType)a->dtype, (hipStream_t)stream) == hipSuccess
             ? CLV_OK
             : CLV_ELAUNCH;
}

}  // extern "C"

namespace {

// Validates a prefill argument block and fills the kernel parameters.
// num_seqs or num_tokens of 0 (nothing to do) leaves the rest unchecked.
int fill_prefill(const clv_prefill_args *a, clv::PrefillParams *out) {
  if (a == nullptr) return CLV_EINVAL;
  if (a->dtype != CLV_F32 && a->dtype != CLV_F16 && a->dtype != CLV_BF16) return CLV_EINVAL;
  if (a->num_seqs < 0 || a->num_tokens < 0 || a->num_heads <= 0 || a->num_kv_heads <= 0 ||
      a->head_dim <= 0 || a->num_blocks <= 0 || a->max_blocks_per_seq < 0 || a->max_query_len < 0)
    return CLV_EINVAL;
  if (a->num_heads % a->num_kv_heads != 0) return CLV_EINVAL;
  if (!is_pow2(a->block_size)) return CLV_EUNSUPPORTED;
  if (!supported_head_dim(a->head_dim)) return CLV_EUNSUPPORTED;
  if (!isfinite(a->scale)) return CLV_EINVAL;
  if (a->num_seqs > 65535) return CLV_EUNSUPPORTED;
  clv::PrefillParams &p = *out;
  p = clv::PrefillParams{};
  p.num_seqs = a->num_seqs;
  p.num_tokens = a->num_tokens;
  if (a->num_seqs == 0 || a->num_tokens == 0) return CLV_OK;
  const int eb = elem_bytes(a->dtype);
  if (!a->out || !a->q || !a->k_cache || !a->v_cache || !a->context_lens || !a->query_start_loc)
    return CLV_EINVAL;
  if (a->max_blocks_per_seq > 0 && !a->block_tables) return CLV_EINVAL;
  if (!aligned16(a->out) || !aligned16(a->q) || !aligned16(a->k_cache) || !aligned16(a->v_cache))
    return CLV_EINVAL;
  if (!stride16(a->q_stride_token, eb) || !stride16(a->q_stride_head, eb) ||
      !stride16(a->out_stride_token, eb) || !stride16(a->out_stride_head, eb) ||
      !stride16(a->kv_stride_block, eb) || !stride16(a->kv_stride_token, eb) ||
      !stride16(a->kv_stride_head, eb))
    return CLV_EINVAL;
  p.out = a->out;
  p.q = a->q;
  p.k_cache = a->k_cache;
  p.v_cache = a->v_cache;
  p.block_tables = a->block_tables;
  p.context_lens = a->context_lens;
  p.query_start_loc = a->query_start_loc;
  p.q_stride_token = a->q_stride_token;
  p.q_stride_head = a->q_stride_head;
  p.out_stride_token = a->out_stride_token;
  p.out_stride_head = a->out_stride_head;
  p.kv_stride_block = a->kv_stride_block;
  p.kv_stride_token = a->kv_stride_token;
  p.kv_stride_head = a->kv_stride_head;
  p.num_heads = a->num_heads;
  p.num_kv_heads = a->num_kv_heads;
  p.head_dim = a->head_dim;
  p.group = a->num_heads / a->num_kv_heads;
  p.block_shift = log2_int(a->block_size);
  p.max_blocks_per_seq = a->max_blocks_per_seq;
  // No chunk is longer than the rows there are: a loose bound then sizes no
  // grid and overflows no tile count.
  p.max_query_len = std::min(a->max_query_len, a->num_tokens);
  p.num_blocks = a->num_blocks;
  p.scale_log2 = a->scale * 1.4426950408889634f;
  p.cus_per_xcd = device_compute_units() / 8;
  return CLV_OK;
}

// The kernel form of a validated prefill.
enum class PrefillKernel { kValu, kMfma, kF32 };

PrefillKernel prefill_kernel(const clv::PrefillParams &p, DType dt, int block_size) {
  if (dt == DType::F32)
    return clv::prefill_f32_chosen(p, block_size) ? PrefillKernel::kF32 : PrefillKernel::kValu;
  return clv::prefill_mfma_supported(dt, p.head_dim, block_size) ? PrefillKernel::kMfma
                                                                 : PrefillKernel::kValu;
}

clv::PrefillSplitShape split_shape(const clv::PrefillParams &p, PrefillKernel k) {
  switch (k) {
    case PrefillKernel::kF32: return clv::prefill_f32_split_shape(p);
    case PrefillKernel::kMfma: return clv::prefill_mfma_split_shape(p);
    default: return {0, 0};
  }
}

size_t split_bytes(const clv::PrefillParams &p, const clv::PrefillSplitShape &sh) {
  const size_t rows = 2 * (size_t)sh.groups * (size_t)sh.rows;
  return round256((size_t)sh.groups * clv::kPrefillDescBytes) + 2 * round256(rows * 4) +
         round256(rows * (size_t)p.head_dim * 4);
}

clv::PrefillSplit split_workspace(const clv::PrefillSplitShape &sh, void *workspace) {
  const size_t rows = 2 * (size_t)sh.groups * (size_t)sh.rows;
  char *ws = (char *)workspace;
  clv::PrefillSplit sp;
  sp.groups = sh.groups;
  sp.desc = ws;
  ws += round256((size_t)sh.groups * clv::kPrefillDescBytes);
  sp.ws_m = (float *)ws;
  ws += round256(rows * 4);
  sp.ws_l = (float *)ws;
  ws += round256(rows * 4);
  sp.ws_o = (float *)ws;
  return sp;
}

int launch_prefill(const clv::PrefillParams &p, DType dt, PrefillKernel k,
                   const clv::PrefillSplit *sp, hipStream_t stream) {
  hipError_t err = hipErrorInvalidValue;
  switch (k) {
    case PrefillKernel::kF32: err = clv::launch_prefill_f32(p, sp, stream); break;
    case PrefillKernel::kMfma: err = clv::launch_prefill_mfma(p, dt, sp, stream); break;
    case PrefillKernel::kValu: err = clv::launch_prefill_valu(p, dt, stream); break;
  }
  return err == hipSuccess ? CLV_OK : CLV_ELAUNCH;
}

}  // namespace

extern "C" {

int clv_chunked_prefill(const clv_prefill_args *a, clv_stream_t stream) {
  clv::PrefillParams p;
  const int st = fill_prefill(a, &p);
  if (st != CLV_OK || p.num_seqs == 0 || p.num_tokens == 0) return st;
  const DType dt = (DType)a->dtype;
  return launch_prefill(p, dt, prefill_kernel(p, dt, a->block_size), nullptr, (hipStream_t)stream);
}

size_t clv_prefill_workspace_bytes(const clv_prefill_args *a) {
  clv::PrefillParams p;
  if (fill_prefill(a, &p) != CLV_OK || p.num_seqs == 0 || p.num_tokens == 0) return 0;
  const clv::PrefillSplitShape sh = split_shape(p, prefill_kernel(p, (DType)a->dtype, a->block_size));
  return sh.groups > 0 ? split_bytes(p, sh) : 0;
}

int clv_chunked_prefill_split(const clv_prefill_args *a, void *workspace, size_t workspace_bytes,
                              clv_stream_t stream) {
  clv::PrefillParams p;
  const int st = fill_prefill(a, &p);
  if (st != CLV_OK || p.num_seqs == 0 || p.num_tokens == 0) return st;
  const DType dt = (DType)a->dtype;
  const PrefillKernel k = prefill_kernel(p, dt, a->block_size);
  const clv::PrefillSplitShape sh = split_shape(p, k);
  if (sh.groups == 0) return launch_prefill(p, dt, k, nullptr, (hipStream_t)stream);
  if (workspace == nullptr || workspace_bytes < split_bytes(p, sh) ||
      ((uintptr_t)workspace & 255u) != 0)
    return CLV_EWORKSPACE;
  const clv::PrefillSplit sp = split_workspace(sh, workspace);
  return launch_prefill(p, dt, k, &sp, (hipStream_t)stream);
}

}  // extern "C"

namespace {

int fill_diff(const clv_diff_args *d, clv::DiffParams *out) {
  if (d == nullptr) return CLV_EINVAL;
  if (!isfinite(d->out_scale)) return CLV_EINVAL;
  if (d->lambda == nullptr && !isfinite(d->lambda_value)) return CLV_EINVAL;
  if (d->norm_weight != nullptr && !(isfinite(d->norm_eps) && d->norm_eps >= 0.f)) return CLV_EINVAL;
  *out = clv::DiffParams{d->lambda, d->lambda_stride_row, d->lambda_stride_head, d->lambda_value,
                         d->norm_weight, d->norm_eps, d->out_scale};
  return CLV_OK;
}

// Least steps of a group of the balanced differential decode: fewer groups read
// less each, more of them leave more partials to the merge. Four sequences of
// 150..3900 tokens, 14/2 heads of 256, bf16, balanced: 1 step 25.5 us, 2 20.6, 4
// 19.5, 8 22.7, 16 31.5; full batches have more steps a group than this anyway.
constexpr int32_t kDiffMinSteps = 4;

// `a` with the rows of both maps as its heads.
int diff_rows(const clv_decode_args *a, clv_decode_args *rows) {
  if (a == nullptr || a->num_heads <= 0 || a->num_heads > (1 << 20) || a->num_kv_heads <= 0 ||
      a->num_heads % a->num_kv_heads != 0)
    return CLV_EINVAL;
  *rows = *a;
  rows->num_heads = 2 * a->num_heads;
  return CLV_OK;
}

// Segments (sequence x kv head x 16 rows) of a differential decode.
int64_t diff_segments(const clv_decode_args &rows) {
  return (int64_t)rows.num_seqs * rows.num_kv_heads *
         ceil_div(rows.num_heads / rows.num_kv_heads, 16);
}

// Small batches: the tokens of every segment in partitions of a multiple of 64, a
// workgroup of four waves each, about kDiffGrid of them. Against the balanced
// decode there is no scan before the first load, and four waves share a partial.
// Partitions / balanced, us, contexts of 0.25..1 of the bound:
//                           1000        4000        16000
//   2 seqs, 14/2 x 256 bf16 12.2/17.3   13.7/18.3   16.5/25.6
//   8 seqs                  12.9/17.6   16.7/21.7   39.7/43.4
//   32 seqs                 16.8/21.1   37.5/42.0   119/113
//   4 seqs, 28/4 x 128 bf16 11.0/14.8   12.4/17.0   27.7/31.7
//   32 seqs                 17.6/21.6   43.5/40.7   165/115
//   4 seqs, 6/6 x 128 fp32  11.9/18.2   14.9/18.9   48.5/47.0
//   16 seqs                 21.3/18.8   54.2/41.4   233/167
// so where the pools' rows up to the bound are at most kDiffGridBytes and the
// segments at most kDiffGridSegments (fp32: half). With 512 workgroups 256-wide heads
// lose (8 x 4000 21.7, two are resident on a unit), 64-wide ones win (8 x 16000
// 24.8, with 256 34.3, balanced 28.2); smallest partitions of 128 equal those of 64.
// fp8 pools, whose steps are bound by their vector work, want three workgroups a
// unit, and gain up to 256 segments and 256 MiB: 16 seqs of up to 4000 tokens, 28/4
// heads, 256 workgroups 26.6, 512 20.3, 768 20.0, 1024 23.4, balanced 31.9; 64 seqs of
// up to 4000 41.1/46.5, 100 85/61; 16 of up to 16000, 32/8, 69.4/65.9.
constexpr int64_t kDiffGrid = 256, kDiffGridFp8 = 768;
constexpr int64_t kDiffGridBytes = 200 << 20, kDiffGridBytesFp8 = 256 << 20;
constexpr int64_t kDiffGridSegments = 128, kDiffGridSegmentsFp8 = 256;

// Tokens of a partition, 0: no partitions.
int32_t diff_partition(const clv_decode_args &rows, bool fp8, int32_t num_waves) {
  if (num_waves > 0 || rows.num_seqs <= 0 ||
      !clv::diff_decode_mfma_supported(rows.head_dim, rows.block_size))
    return 0;
  const int64_t segments = diff_segments(rows), eb = fp8 ? 1 : elem_bytes(rows.dtype);
  if (segments * eb > (fp8 ? kDiffGridSegmentsFp8 : 2 * kDiffGridSegments) ||
      2 * eb * rows.head_dim * rows.num_kv_heads * rows.num_seqs * rows.max_context_len >
          (fp8 ? kDiffGridBytesFp8 : kDiffGridBytes))
    return 0;
  const int64_t grid = fp8 ? kDiffGridFp8 : rows.head_dim == 64 ? 2 * kDiffGrid : kDiffGrid;
  const int64_t parts = std::max<int64_t>(1, grid / segments);
  return (int32_t)(std::max<int64_t>(1, ceil_div(ceil_div(rows.max_context_len, parts), 64)) * 64);
}

// Longest context for which a differential decode runs as one launch, a
// workgroup per (sequence, kv head, 16 rows), where the caller names no wave
// count (kernels.choose_schedule has the same bound for plain decode). One
// launch / balanced, us, every sequence of the same length:
//                                128        512        1024       2048
//   8 seqs,   6/6 x 128  fp32    8.1/19.0   16.6/20.1  28.1/21.0  51.7/28.6
//   8 seqs,  14/2 x 256  bf16    8.7/17.1   15.9/18.5  26.1/19.6  46.5/22.6
//   64 seqs, 28/4 x 128  bf16    6.8/17.3   14.5/24.9  24.3/34.6  41.9/54.6
//   128 seqs, 14/2 x 256 bf16    9.5/21.6   25.2/37.5  43.6/57.0  81.3/95.8
// Past it one launch would still win for many sequences of one length, but it
// takes as long as its longest sequence, which a ragged batch (what decodes
// there) has alone. Where partitions are the other choice, key rows of 512 bytes
// or more take half of it: one launch / partitions of 8 x 256, 320 and 512 tokens
// 11.0/11.2, 12.4/11.4, 16.1/11.8 us (14/2 x 256 bf16), narrower ones 8.5/11.4,
// 9.4/11.5, 11.6/11.2 (28/4 x 128 bf16).
constexpr int32_t kDiffSinglePassMaxLen = 512;

// Most segments (sequence x kv head x 16 rows) of head_dim 256 that take it. Two
// workgroups of that width are resident on a compute unit (64.5 KiB of LDS for
// the waves' join, as much for 2 rows as for 16), so more of them queue:
// 16/16 x 256 fp16, 128 / 512 tokens: 512 segments 20.0/20.3 and 48.9/50.7 us,
// 1024 38.8/29.6 and 93.3/91.5, 2048 74.1/53.4 and 183/171. head_dim 128 wins at
// every count measured (1024 segments of 32/8 heads: 20.1/26.1 and 47.7/55.1).
constexpr int64_t kDiffSinglePassWideSegments = 512;

bool diff_single_pass(const clv_decode_args &rows, bool fp8, int32_t num_waves) {
  if (!clv::diff_decode_mfma_supported(rows.head_dim, rows.block_size)) return true;
  const int64_t segments = diff_segments(rows);
  const bool wide = !fp8 && rows.head_dim * elem_bytes(rows.dtype) >= 512;
  const int32_t max_len = wide && diff_partition(rows, fp8, num_waves) > 0
                              ? kDiffSinglePassMaxLen / 2
                              : kDiffSinglePassMaxLen;
  if (num_waves <= 0 && rows.max_context_len <= max_len &&
      (rows.head_dim <= 128 || segments <= kDiffSinglePassWideSegments))
    return true;
  // More segments than the balanced decode takes: a workgroup each fills the chip.
  return segments > clv::kStreamMaxSegments;
}

PrefillKernel diff_prefill_kernel(const clv::PrefillParams &p, DType dt) {
  if (dt == DType::F32)
    return clv::diff_prefill_f32_covers(p) ? PrefillKernel::kF32 : PrefillKernel::kValu;
  return clv::diff_prefill_mfma_covers(p, dt) ? PrefillKernel::kMfma : PrefillKernel::kValu;
}

// As split_shape; rows counts those of both maps.
clv::PrefillSplitShape diff_split_shape(const clv::PrefillParams &p, PrefillKernel k) {
  clv::PrefillSplitShape sh = {0, 0};
  if (k == PrefillKernel::kF32) sh = clv::diff_prefill_f32_split_shape(p);
  if (k == PrefillKernel::kMfma) sh = clv::diff_prefill_split_shape(p);
  sh.rows *= 2;
  return sh;
}

int32_t diff_waves(bool fp8, int32_t num_waves) {
  return num_waves > 0 ? num_waves : fp8 ? clv_default_num_waves_fp8() : clv_default_num_waves();
}

}  // namespace

extern "C" {

size_t clv_diff_decode_workspace_bytes(const clv_decode_args *a, int32_t fp8, int32_t num_waves) {
  clv_decode_args r;
  if (diff_rows(a, &r) != CLV_OK || diff_single_pass(r, fp8 != 0, num_waves)) return 0;
  if (const int32_t size = diff_partition(r, fp8 != 0, num_waves))
    return clv_splitk_workspace_bytes(r.num_seqs, r.num_heads, r.head_dim, r.max_context_len, size);
  return clv_balanced_workspace_bytes(r.num_seqs, r.num_heads, r.num_kv_heads, r.head_dim,
                                      diff_waves(fp8 != 0, num_waves));
}

int clv_diff_decode(const clv_decode_args *a, const clv_diff_args *d, const float *k_scales,
                    const float *v_scales, int32_t num_waves, void *workspace,
                    size_t workspace_bytes, clv_stream_t stream) {
  clv_decode_args r;
  clv::DiffParams diff;
  int st = diff_rows(a, &r);
  if (st == CLV_OK) st = fill_diff(d, &diff);
  if (st != CLV_OK) return st;
  if ((k_scales == nullptr) != (v_scales == nullptr)) return CLV_EINVAL;
  const bool fp8 = k_scales != nullptr;
  if (fp8) {
    if (a->dtype != CLV_F16 && a->dtype != CLV_BF16) return CLV_EINVAL;
    if (a->head_dim != 128 || a->block_size < 16) return CLV_EUNSUPPORTED;
    if ((a->kv_stride_block & 15) || (a->kv_stride_token & 15) || (a->kv_stride_head & 15))
      return CLV_EINVAL;
  }
  const hipStream_t s = (hipStream_t)stream;
  const DType dt = (DType)a->dtype;
  clv::DecodeParams p;
  auto set_own = [&] {  // what the fills of plain decode do not know
    p.diff = diff;
    p.stream_min_steps = kDiffMinSteps;
    p.kv_fp8 = fp8 ? 1 : 0;
    p.k_scales = k_scales;
    p.v_scales = v_scales;
  };
  if (diff_single_pass(r, fp8, num_waves)) {
    st = fill_decode(&r, &p);
    if (st != CLV_OK || p.num_seqs == 0) return st;
    if ((int64_t)p.num_kv_heads * p.n_gchunks > 65535) return CLV_EUNSUPPORTED;  // grid y limit
    set_own();
    const hipError_t err = clv::diff_decode_mfma_supported(a->head_dim, a->block_size)
                               ? clv::launch_diff_decode_mfma(p, dt, s)
                               : clv::launch_diff_decode_valu(p, dt, s);
    return err == hipSuccess ? CLV_OK : CLV_ELAUNCH;
  }
  if (const int32_t size = diff_partition(r, fp8, num_waves)) {
    st = fill_decode(&r, &p);
    if (st != CLV_OK || p.num_seqs == 0) return st;
    if ((int64_t)p.num_kv_heads * p.n_gchunks > 65535) return CLV_EUNSUPPORTED;  // grid y limit
    st = fill_splitk(&r, size, workspace, workspace_bytes, &p);
    if (st != CLV_OK) return st;
    set_own();
    if (clv::launch_diff_decode_mfma(p, dt, s) != hipSuccess) return CLV_ELAUNCH;
    return clv::launch_diff_stream_reduce(p, dt, s) == hipSuccess ? CLV_OK : CLV_ELAUNCH;
  }
  st = fill_balanced(&r, diff_waves(fp8, num_waves), workspace, workspace_bytes, &p, true);
  if (st != CLV_OK || p.num_seqs == 0) return st;
  set_own();
  if (clv::launch_diff_decode_stream(p, dt, s) != hipSuccess) return CLV_ELAUNCH;
  return clv::launch_diff_stream_reduce(p, dt, s) == hipSuccess ? CLV_OK : CLV_ELAUNCH;
}

size_t clv_diff_prefill_workspace_bytes(const clv_prefill_args *a) {
  clv::PrefillParams p;
  if (fill_prefill(a, &p) != CLV_OK || p.num_seqs == 0 || p.num_tokens == 0) return 0;
  const clv::PrefillSplitShape sh =
      diff_split_shape(p, diff_prefill_kernel(p, (DType)a->dtype));
  return sh.groups > 0 ? split_bytes(p, sh) : 0;
}

int clv_diff_prefill(const clv_prefill_args *a, const clv_diff_args *d, void *workspace,
                     size_t workspace_bytes, clv_stream_t stream) {
  clv::PrefillParams p;
  clv::DiffParams diff;
  int st = fill_prefill(a, &p);
  if (st == CLV_OK) st = fill_diff(d, &diff);
  if (st != CLV_OK || p.num_seqs == 0 || p.num_tokens == 0) return st;
  p.diff = diff;
  const hipStream_t s = (hipStream_t)stream;
  const DType dt = (DType)a->dtype;
  const PrefillKernel k = diff_prefill_kernel(p, dt);
  const clv::PrefillSplitShape sh = diff_split_shape(p, k);
  clv::PrefillSplit split;
  const clv::PrefillSplit *sp = nullptr;
  if (sh.groups > 0 && (workspace != nullptr || workspace_bytes != 0)) {
    if (workspace == nullptr || workspace_bytes < split_bytes(p, sh) ||
        ((uintptr_t)workspace & 255u) != 0)
      return CLV_EWORKSPACE;
    split = split_workspace(sh, workspace);
    sp = &split;
  }
  hipError_t err = hipErrorInvalidValue;
  switch (k) {
    case PrefillKernel::kF32: err = clv::launch_diff_prefill_f32(p, sp, s); break;
    case PrefillKernel::kMfma: err = clv::launch_diff_prefill_mfma(p, dt, sp, s); break;
    case PrefillKernel::kValu:
      p.group *= 2;  // rows of both maps
      err = clv::launch_diff_prefill_valu(p, dt, s);
      break;
  }
  return err == hipSuccess ? CLV_OK : CLV_ELAUNCH;
}

}  // extern "C"

namespace {

// Validates a step of the block tables. An empty table (no rows) is valid.
int fill_tables(const clv_tables_args *a, clv::TablesParams *p) {
  if (a == nullptr) return CLV_EINVAL;
  if (a->rows < 0 || a->width < 0 || a->num_blocks < 0 || a->num_tokens < 0 || a->reserve < 0)
    return CLV_EINVAL;
  if (a->num_tokens > INT32_MAX) return CLV_EINVAL;
  if (!is_pow2(a->block_size) || a->rows > CLV_TABLES_MAX_ROWS) return CLV_EUNSUPPORTED;
  if ((int64_t)a->width * a->block_size > INT32_MAX) return CLV_EINVAL;
  if (!a->num_free || !a->num_free_out || !a->query_start_loc || !a->status) return CLV_EINVAL;
  if (a->num_blocks > 0 && !a->free_blocks) return CLV_EINVAL;
  if (a->num_tokens > 0 && !a->slot_mapping) return CLV_EINVAL;
  if (a->rows > 0 && (!a->blocks_held || !a->context_lens || !a->new_lens || !a->blocks_held_out ||
                      !a->context_lens_out || (a->width > 0 && !a->block_tables)))
    return CLV_EINVAL;
  // What is written is apart from everything else (a count's output may be its
  // input): many workgroups read while others write.
  struct Range {
    const char *begin, *end;
    bool written;
  } range[12];
  int n = 0;
  auto add = [&](const void *x, int64_t bytes, bool written) {
    if (bytes > 0) range[n++] = Range{(const char *)x, (const char *)x + bytes, written};
  };
  auto add_state = [&](const int32_t *in, const int32_t *out, int64_t count) {
    add(in, 4 * count, out == in);
    if (out != in) add(out, 4 * count, true);
  };
  add_state(a->blocks_held, a->blocks_held_out, a->rows);
  add_state(a->context_lens, a->context_lens_out, a->rows);
  add_state(a->num_free, a->num_free_out, 1);
  add(a->new_lens, 4 * (int64_t)a->rows, false);
  add(a->block_tables, 4 * (int64_t)a->rows * a->width, true);
  add(a->free_blocks, 4 * (int64_t)a->num_blocks, true);
  add(a->slot_mapping, 8 * a->num_tokens, true);
  add(a->query_start_loc, 4 * ((int64_t)a->rows + 1), true);
  add(a->status, 4, true);
  for (int i = 0; i < n; ++i)
    for (int k = 0; k < i; ++k)
      if ((range[i].written || range[k].written) && range[i].begin < range[k].end &&
          range[k].begin < range[i].end)
        return CLV_EINVAL;
  *p = clv::TablesParams{a->block_tables,     a->blocks_held,      a->context_lens,
                         a->new_lens,         a->free_blocks,      a->num_free,
                         a->blocks_held_out,  a->context_lens_out, a->num_free_out,
                         a->slot_mapping,     a->query_start_loc,  a->status,
                         a->num_tokens,       a->rows,             a->width,
                         log2_int(a->block_size), a->num_blocks,   a->reserve};
  return CLV_OK;
}

}  // namespace

extern "C" {

int clv_advance_block_tables(const clv_tables_args *a, clv_stream_t stream) {
  clv::TablesParams p;
  const int st = fill_tables(a, &p);
  if (st != CLV_OK) return st;
  return clv::launch_tables(p, (hipStream_t)stream) == hipSuccess ? CLV_OK : CLV_ELAUNCH;
}

}  // extern "C"
