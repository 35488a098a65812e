// diff_prefill.hip - differential attention of chunked prefill with MFMA
// (fp16/bf16), over paged KV.
//
// Query row i of sequence s sees cached positions p <= context_lens[s] - n_s + i
// through two softmax maps, one per half of the head, which share V:
//   a_m = softmax(scale q_m K_m^T) V,   out = joined(a_1 - lambda a_2).
//
// Work decomposition: a workgroup of 8 waves (two per SIMD) takes up to kPairs =
// 64 kRT rows (row r is token r / G, query head r % G of one kv head) against
// all K/V tiles its last row sees, staged in LDS. Waves w and w + 4 hold the
// same 16 kRT rows, one map each: a wave reads only its half of every key row
// (D/64 k-steps of 32), and the pair meets once, at the end, through LDS, where
// each wave finishes half of the rows. Per 32
// tokens a wave runs
//   S^T[t, r] = K_m[t, :] . Q_m[r, :]   2 x kRT x D/64 MFMAs (16x16x32)
//   O[r, d]  += P[r, t] V[t, d]         kRT x D/16 MFMAs
// with an fp32 online softmax between: 6 D flops per (row, key) and head, of
// which 4 D are products with V.
//
// The pipeline is that of the plain MFMA prefill, for its reasons: the C layout
// of the first product is the A layout of the second, so P stays in registers;
// V's B operand comes from LDS through transposing reads; the two waves of a
// SIMD run their softmax and their MFMAs in opposite phases; LDS reads run ahead
// of the MFMAs they feed; tiles go through a ring of three stages. P.V runs in
// fp16 for both types: P <= 2^8 keeps 11 bits there (a relative error of 2^-11
// at most), and bf16 V is converted exactly unless its magnitude reaches 2^16. An
// accumulator that is not finite makes the workgroup run its tiles again, in a
// pass that keeps bf16 V as it is and P as a bf16 value and its residual, with 0
// in the place of infinities and NaN, which only the rows that see them then take
// (0 * inf is NaN). The running maximum is only raised by more than 2^8.
//
// What bounds it. At head_dim 128: the matrix core with the vector work beside
// it, which adds to its time (16x16x32 products 265 us of the 541 of eight chunks
// of 512 over 4096 tokens, 32/8 heads, bf16; staging, conversion and softmax the
// rest): 810 TFLOP/s. Products of 32x32x16 (558 us), exponentials between the
// products of one wave (584), scores a step ahead (564) and a barrier between
// the waves' phases (553) were no faster; nor were two to eight V operands in
// flight (526..541). At head_dim 256: LDS reads, 24 KiB a wave and 32 tokens for
// 25 products: 320 us for four chunks of 512 over 4096 tokens, 16/4 heads (600
// TFLOP/s). Two row tiles a wave would halve them but spill, and cost small
// calls their rows: 287 us there, 34 -> 53 for a prompt of 777 tokens.
#include "prefill_split.h"

#include <type_traits>

namespace clv {
namespace {

constexpr int kWaves = 8;
constexpr int kThreads = kWaves * 64;
constexpr float kRescaleLog2 = 8.f;  // lazy-rescale threshold (log2 units)

// Shape of the kernel at a head_dim: 16-row MFMA tiles per wave, tokens per tile.
// At 256 a wave's accumulator is twice as wide: one row tile keeps two waves on
// a SIMD, and 32 tokens keep the ring of three stages in LDS.
template <int D> struct Shape {
  static constexpr int kRT = D == 256 ? 1 : 2;
  static constexpr int kBK = D == 256 ? 32 : 64;
  static constexpr int kPairs = kWaves / 2 * 16 * kRT;  // rows per workgroup
};

// The transposing LDS read of an MFMA B operand from row-major V: two reads of
// four rows each, as in the plain prefill kernel.
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
__device__ __forceinline__ u32x4 vt_read(uint32_t lo, uint32_t hi) {
  const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(size_t)lo);
  const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(size_t)hi);
  const u32x2 ua = __builtin_bit_cast(u32x2, a), ub = __builtin_bit_cast(u32x2, b);
  return (u32x4){ua[0], ua[1], ub[0], ub[1]};
}

__device__ __forceinline__ uint32_t bf16x2_to_f16x2(uint32_t w) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
  const float a = __builtin_bit_cast(float, w << 16);
  const float b = __builtin_bit_cast(float, w & 0xffff0000u);
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, f16x2));
}

// Units of the split (prefill_split.h): tiles, full or not (D = 256: 1.26 us with all
// rows, 1.13 with 7 of 64). An item costs what its start (Q, first tile) and end
// (join, or partials and their merge) take, 8..10 us: four tiles of 64 tokens, six
// of 32. Sum over 46 batches (chunks, prompts, mixed steps; head_dim 64, 128, 256):
// items at two tiles, a bound moved by up to 1/16 of a share 4860 us, as below,
// 1/64 4638; the least share six tiles in place of four and a cut five in place of
// ten 4600 (cut 16: 4612, 25: 4624; least share eight: 4638, twelve 4642).
template <int D> struct SplitCfg {
  static constexpr int kBK = Shape<D>::kBK;
  static constexpr int kItemUnits = D == 256 ? 6 : 4;
  static constexpr int kMinShare = 6;
  static constexpr int kCutUnits = 5;
  static __host__ __device__ __forceinline__ int tile_units(int) { return 1; }
  static __host__ __device__ __forceinline__ int snap(int share) {
    return max(kItemUnits, share / 64);
  }
};

// Table width in tokens up to which a call is not split. Items (counted at the
// longest chunk) of up to 9/4 rounds of the device: a cut costs what the evenness
// gives (one prompt of 777 tokens, 16/16 x 256, 35.7 us unsplit and 51.5 split; three
// of 488..663, 528 items, 54 and 60). More of them run long after the others end:
// eight prompts of 17..1000 tokens, 32/8 x 128, 2048 items, 168 and 105; 16 of 30..500
// 142 and 102; 24 of up to 200 behind 700, 16/16 x 256, 121 and 62; five of 285..999,
// 28/4 x 128, 104 and 91.
constexpr int kSplitMinTokens = 1024, kSplitMinTokensMany = 256;

// Eight values of V (token `pos`, columns d0 ..) with 0 in the place of NaN and
// infinities; seen_by[column] remembers the first token with a NaN there,
// seen_by[D + column] with +inf, seen_by[2 D + column] with -inf.
template <typename T, int D>
__device__ __forceinline__ u32x4 finite_v8(u32x4 v, int pos, int d0, int *seen_by) {
  constexpr uint32_t kInf = __is_same(T, _Float16) ? 0x7c00u : 0x7f80u;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t x = (v[e / 2] >> (16 * (e % 2))) & 0xffffu;
    if ((x & kInf) != kInf) continue;
    const int kind = (x & 0x7fffu) != kInf ? 0 : (x & 0x8000u) == 0 ? 1 : 2;
    atomicMin(&seen_by[kind * D + d0 + e], pos);
    v[e / 2] &= 0xffffu << (16 * (1 - e % 2));
  }
  return v;
}

// What a row that sees tokens <= last takes from them in a column, beyond the
// finite values.
template <int D>
__device__ __forceinline__ float seen_v(const int *seen_by, int col, int last) {
  const float inf = __builtin_inff();
  float x = seen_by[col] <= last ? __builtin_nanf("") : 0.f;
  if (seen_by[D + col] <= last) x += inf;
  if (seen_by[2 * D + col] <= last) x -= inf;
  return x;
}

template <typename T, int D, bool SPLIT>
__global__ void __launch_bounds__(kThreads)
diff_prefill_mfma(const PrefillArgs args) {
  typedef Mfma16x16x32<T> MfQK;
  typedef Mfma16x16x32<_Float16> MfPV;
  typedef typename MfQK::op_t qk_t;
  typedef typename MfPV::op_t pv_t;
  constexpr bool kBf16 = !__is_same(T, _Float16);
  constexpr int kRT = Shape<D>::kRT;
  constexpr int kBK = Shape<D>::kBK;
  constexpr int kPairs = Shape<D>::kPairs;
  constexpr int kWaveRows = 16 * kRT;
  constexpr int HS = kBK / 32;            // 32-token steps per tile
  constexpr int NQK = D / 64;             // QK k-steps of a half head
  constexpr int CH = D / 16;              // P.V MFMAs per (step, row tile)
  // LDS row strides (elements): 32 mod 64 bytes, conflict-free for the K reads
  // and the transposing V reads (measured on the plain kernel).
  constexpr int KROW = D + 16;
  constexpr int VROW = D + 16;
  constexpr int CPR = D * 2 / 16;         // 16-byte chunks per row
  constexpr int RPP = kThreads / CPR;     // rows per load pass
  constexpr int PASSES = kBK / RPP;       // load passes per tile
  constexpr int kStage = kBK * KROW;      // elements of a stage of K (and of V)
  constexpr int kLdsK = 3 * kStage * 2, kLdsAll = 2 * kLdsK;
  constexpr int kLdsPair = kWaves * kRT * CH * 64 * 8;  // half of every wave's rows
  static_assert(kLdsPair <= kLdsAll, "the pairs meet in the tile ring's memory");

  __shared__ __attribute__((aligned(16))) char s_mem[kLdsAll];
  __shared__ __attribute__((aligned(4))) uint8_t sValid[3][kBK];  // 1 = the token is readable
  __shared__ int sBad;  // set when an accumulator is not finite
  __shared__ int sSeenBy[3 * D];  // exact pass, see finite_v8
  typedef PrefillSched<SplitCfg<D>> Sched;
  __shared__ int s_pre[SPLIT ? kPrefillSplitItems + 1 : 1];
  __shared__ int s_tmp[3 * kWaves];
  __shared__ int s_cur[kWaves][Sched::kCursorInts];
  T *const sK = (T *)s_mem;                       // [3][kBK][KROW]
  uint16_t *const sV = (uint16_t *)(s_mem + kLdsK);  // [3][kBK][VROW]

  // Consecutive ids go round-robin over the 8 XCDs: each takes a contiguous
  // range of items, so that the query tiles of one kv head share its L2.
  int L = SPLIT ? 0 : (int)(blockIdx.x % 8) * (int)(gridDim.x / 8) + (int)(blockIdx.x / 8);
  int *cur = s_cur[__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)];
  if constexpr (SPLIT) {
    Sched sched;
    sched.template init<kThreads>(args.p, args.bq, args.n_qtiles, args.sp.groups, s_pre, s_tmp);
    L = sched.group_of(blockIdx.x);
    if (L < 0) return;
    sched.start(L, cur);
    if (threadIdx.x == 0) sched.clear_desc(args.sp, L);
  } else if (L >= args.total) {
    return;
  }

  for (bool first = true;; first = false) {
  const PrefillArgs ar0 = SPLIT ? reload_args() : args;
  const PrefillParams &p = ar0.p;
  const int bq = ar0.bq, n_qtiles = ar0.n_qtiles;
  PrefillItem it;
  int t0 = 0, t1, nt;  // this workgroup's tiles of the item, and all of them
  if constexpr (SPLIT) {
    if (!Sched::next(p, bq, n_qtiles, s_pre, cur, it, t0, t1, nt)) break;
  } else {
    if (!first) break;
    const int qt = n_qtiles - 1 - L % n_qtiles;  // longest query tiles first
    const int rest = L / n_qtiles;
    it.set(p, bq, rest / p.num_kv_heads, rest % p.num_kv_heads, qt);
    if (it.q0 >= it.n_new) break;
    nt = t1 = Sched::tiles(it.kv_end);
  }
  const int s = it.s, kvh = it.kvh, qs = it.qs, n_new = it.n_new, q0 = it.q0;
  const int base_pos = it.base_pos, kv_end = it.kv_end;
  const int te = min(t1, (kv_end + kBK - 1) / kBK);  // tiles [t0, te); no tokens: none
  const int G = p.group;

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int map = wave / (kWaves / 2);
  const int wave_row0 = kWaveRows * (wave % (kWaves / 2));
  const int n16 = lane & 15;
  const int j = lane >> 4;

  const char *kbase = (const char *)p.k_cache + (int64_t)kvh * p.kv_stride_head * (int64_t)sizeof(T);
  const char *vbase0 = (const char *)p.v_cache + (int64_t)kvh * p.kv_stride_head * (int64_t)sizeof(T);

  // A negative scale is a sign flip of Q, a zero one 2^-126 (every weight 1 to
  // far below fp32 resolution): the softmax multiplies by c > 0 only.
  const float c = fmaxf(fabsf(p.scale_log2), 0x1p-126f);
  const uint32_t qflip = p.scale_log2 < 0.f ? 0x80008000u : 0u;

  // The map's half of Q (B operand of S^T = K Q^T) for rows wave_row0 + 16rt + n16.
  u32x4 qop[kRT][NQK];
  int lim[kRT];  // last visible position of the lane's softmax row (-1: no row)
#pragma unroll
  for (int rt = 0; rt < kRT; ++rt) {
    const int r = wave_row0 + 16 * rt + n16;
    const int tok = q0 + r / G;
    const bool ok = r < bq * G && tok < n_new;
    lim[rt] = ok ? base_pos + tok : -1;
    const T *qrow = (const T *)p.q + (int64_t)(qs + (ok ? tok : q0)) * p.q_stride_token +
                    (int64_t)(kvh * G + r % G) * p.q_stride_head + map * (D / 2);
#pragma unroll
    for (int i = 0; i < NQK; ++i) {
      u32x4 w = load_vec<u32x4>(qrow + 32 * i + 8 * j);
      w ^= qflip;
      if (!ok) w = (u32x4){0u, 0u, 0u, 0u};
      qop[rt][i] = w;
    }
  }
  // Smallest causal limit over the wave's real rows: tiles ending at or below
  // it need no causal mask. A wave without rows only helps to stage the tiles.
  const int wave_lim = (wave_row0 < bq * G && q0 + wave_row0 / G < n_new)
                           ? base_pos + q0 + wave_row0 / G : -1;
  const bool active = wave_row0 < (it.q_hi - q0) * G;

  // Tile loader: thread handles chunk tid % CPR of rows tid / CPR + RPP * i. The
  // rows of one load instruction lie in one block (the launcher checks it): a
  // scalar block id, and 32-bit offsets inside the block through a buffer
  // resource whose range check gives unreadable tokens zeros.
  constexpr int WROWS = 64 / CPR;
  const int lchunk = tid % CPR;
  const int lrow = tid / CPR;
  const int wrow = WROWS * wave;
  const uint32_t sblk32 = (uint32_t)(p.kv_stride_block * (int64_t)sizeof(T));
  const uint32_t stok32 = (uint32_t)(p.kv_stride_token * (int64_t)sizeof(T));
  const unsigned nblocks = (unsigned)p.num_blocks;
  const int bshift = p.block_shift;
  const uint32_t bmask = (1u << bshift) - 1u;
  const uint32_t lane_off = (uint32_t)(lrow - wrow) * stok32 + (uint32_t)lchunk * 16u;
  typedef const int32_t __attribute__((address_space(4))) *cint_t;
  const cint_t brow = (cint_t)(p.block_tables + (int64_t)s * p.max_blocks_per_seq);
  u32x4 kreg[PASSES], vreg[PASSES];
  bool rvalid[PASSES];
  int rblk[PASSES];  // block of the wave's rows of the tile to load next (-1: none)
  auto fetch_blocks = [&](int tile) {
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const int tok0 = tile * kBK + wrow + RPP * i;
      rblk[i] = (tile < te && tok0 < kv_end) ? brow[tok0 >> bshift] : -1;
    }
  };
  auto load_tile = [&](int tile) {
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const uint32_t tok0 = (uint32_t)(tile * kBK + wrow + RPP * i);
      const bool bok = (unsigned)rblk[i] < nblocks;
      const bool ok = bok && (int)tok0 + (lrow - wrow) < kv_end;
      rvalid[i] = ok;
      const uint64_t boff = (uint64_t)(uint32_t)(bok ? rblk[i] : 0) * sblk32;
      const int nrec = bok ? (int)(stok32 * bmask) + D * 2 : 0;
      const uint32_t voff = ok ? (tok0 & bmask) * stok32 + lane_off : 0x80000000u;
      kreg[i] = buf_load<u32x4>(make_rsrc_range(kbase + boff, nrec), voff);
      vreg[i] = buf_load<u32x4>(make_rsrc_range(vbase0 + boff, nrec), voff);
    }
  };
  auto store_tile = [&](int tile, auto exact_c) {
    constexpr bool EXACT = decltype(exact_c)::value;
    const int buf = tile % 3;
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const int row = lrow + RPP * i;
      store_vec<u32x4>(&sK[buf * kStage + row * KROW + lchunk * 8], kreg[i]);
      u32x4 v = vreg[i];
      if constexpr (EXACT) v = finite_v8<T, D>(v, tile * kBK + row, 8 * lchunk, sSeenBy);
      if constexpr (kBf16 && !EXACT) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = bf16x2_to_f16x2(v[e]);
      }
      store_vec<u32x4>(&sV[buf * kStage + row * VROW + lchunk * 8], v);
      if (lchunk == 0) sValid[buf][row] = rvalid[i] ? 1 : 0;
    }
  };

  f32x4 o[kRT][CH];
  float m_run[kRT];
  float thr[kRT];   // rescale threshold per row
  float msub[kRT];  // m_run * c (0 while m_run is -inf)
  // Row sums of P by MFMA against ones: in the C layout of o, and of the
  // rounded P that P.V uses.
  f32x4 lsum[kRT];

  // One pass over the tiles in 32-token steps g (tile g / HS, step g % HS):
  //   M(g): scores of g, then P.V of g - 1;   V(g): online softmax of g.
  // The waves of the first map run M V, those of the second V M with their
  // softmax one step behind. P.V of g - 1 may read the previous tile. Returns
  // whether an accumulator was not finite (fast pass only).
  auto run_tiles = [&](auto exact_c) -> bool {
    constexpr bool EXACT = decltype(exact_c)::value;
    typedef Mfma16x16x32<__bf16> MfB;
    constexpr bool TWO = EXACT && kBf16;  // P as two bf16 values
    typedef typename std::conditional<TWO, typename MfB::op_t, pv_t>::type p_t;
#pragma unroll
    for (int rt = 0; rt < kRT; ++rt) {
#pragma unroll
      for (int m = 0; m < CH; ++m) o[rt][m] = (f32x4){0.f, 0.f, 0.f, 0.f};
      m_run[rt] = kNegInf;
      thr[rt] = kNegInf;
      msub[rt] = 0.f;
      lsum[rt] = (f32x4){0.f, 0.f, 0.f, 0.f};
    }
    f32x4 sacc[2][kRT];     // scores of the step between M and V
    p_t pa[kRT], pl[kRT];   // P of the step between V and the next M (pl: its residual)

    // Scores of step g: sacc[h][rt][e] = S[row 16rt + n16][token 32 (g % HS) + 16h + 4j + e].
    auto qk = [&](int g) {
      const T *K = sK + ((g / HS) % 3) * kStage + map * (D / 2);
      const int half = g % HS;
      auto kread = [&](int h, int i) {
        return load_vec<u32x4>(&K[(32 * half + 16 * h + n16) * KROW + 32 * i + 8 * j]);
      };
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int rt = 0; rt < kRT; ++rt) sacc[h][rt] = (f32x4){0.f, 0.f, 0.f, 0.f};
      u32x4 now[2] = {kread(0, 0), kread(1, 0)};
#pragma unroll
      for (int i = 0; i < NQK; ++i) {
        u32x4 nxt[2];
        __builtin_amdgcn_sched_barrier(0);
        if (i + 1 < NQK) {
          nxt[0] = kread(0, i + 1);
          nxt[1] = kread(1, i + 1);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int rt = 0; rt < kRT; ++rt)
            sacc[h][rt] = MfQK::run(__builtin_bit_cast(qk_t, now[h]),
                                    __builtin_bit_cast(qk_t, qop[rt][i]), sacc[h][rt]);
        if (i + 1 < NQK) {
          now[0] = nxt[0];
          now[1] = nxt[1];
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    };
    const p_t ones = __builtin_bit_cast(
        p_t, (u32x4){TWO ? 0x3f803f80u : 0x3c003c00u, TWO ? 0x3f803f80u : 0x3c003c00u,
                     TWO ? 0x3f803f80u : 0x3c003c00u, TWO ? 0x3f803f80u : 0x3c003c00u});
    // O += P V for step g.
    auto pv = [&](int g) {
      const uint16_t *vrow = sV + ((g / HS) % 3) * kStage +
                             (32 * (g % HS) + 4 * j + (n16 >> 2)) * VROW + 4 * (n16 & 3);
      // One base register per call, opaque to the compiler, which otherwise
      // keeps an address per read.
      uint32_t vb0 = (uint32_t)(size_t)(const __attribute__((address_space(3))) uint16_t *)vrow;
      asm volatile("" : "+v"(vb0));
      auto vread = [&](int m) {
        return vt_read(vb0 + 32u * m, vb0 + 32u * (VROW + m));  // rows +0 / +16
      };
      constexpr int PVD = 3;  // V operands in flight
      u32x4 vq[PVD];
#pragma unroll
      for (int m = 0; m < PVD; ++m) vq[m] = vread(m);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int rt = 0; rt < kRT; ++rt) {
        if constexpr (!TWO) {
          lsum[rt] = MfPV::run(pa[rt], ones, lsum[rt]);
        } else {
          lsum[rt] = MfB::run(pa[rt], ones, lsum[rt]);
          lsum[rt] = MfB::run(pl[rt], ones, lsum[rt]);
        }
      }
#pragma unroll
      for (int m = 0; m < CH; ++m) {
        const p_t vb = __builtin_bit_cast(p_t, vq[m % PVD]);
        __builtin_amdgcn_sched_barrier(0);
        if (m + PVD < CH) vq[m % PVD] = vread(m + PVD);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int rt = 0; rt < kRT; ++rt) {
          if constexpr (!TWO) {
            o[rt][m] = MfPV::run(pa[rt], vb, o[rt][m]);
          } else {
            o[rt][m] = MfB::run(pa[rt], vb, o[rt][m]);
            o[rt][m] = MfB::run(pl[rt], vb, o[rt][m]);
          }
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    };
    // Scores a row may not see become -inf.
    auto mask_step = [&](int g) {
      const int buf = (g / HS) % 3;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t vf =
            *reinterpret_cast<const uint32_t *>(&sValid[buf][32 * (g % HS) + 16 * h + 4 * j]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int pos = 32 * g + 16 * h + 4 * j + e;
          const bool readable = ((vf >> (8 * e)) & 0xffu) != 0;
#pragma unroll
          for (int rt = 0; rt < kRT; ++rt)
            if (!(readable && pos <= lim[rt])) sacc[h][rt][e] = kNegInf;
        }
      }
    };
    // Online softmax of step g; the running maximum is raised when a score
    // passes thr = m_run + 8 / c, and the four lanes of a row agree on it then.
    auto softmax = [&](int g, bool full) {
      if (!full) mask_step(g);
      float pf[kRT][8];
#pragma unroll
      for (int rt = 0; rt < kRT; ++rt) {
        float mx = kNegInf;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e) mx = fmaxf(mx, sacc[h][rt][e]);
        if (__any(mx > thr[rt])) {
          mx = fmaxf(mx, shfl_xor(mx, 16));
          mx = fmaxf(mx, shfl_xor(mx, 32));
          const float m_new = fmaxf(m_run[rt], mx);
          const float alpha = m_new == kNegInf ? 1.f : fast_exp2((m_run[rt] - m_new) * c);
          m_run[rt] = m_new;
          thr[rt] = m_new == kNegInf ? kNegInf : m_new + kRescaleLog2 / c;
          msub[rt] = m_new == kNegInf ? 0.f : m_new * c;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float a = shfl(alpha, 4 * j + e);
            lsum[rt][e] *= a;
#pragma unroll
            for (int m = 0; m < CH; ++m) o[rt][m][e] *= a;
          }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            pf[rt][4 * h + e] = fast_exp2(__builtin_fmaf(sacc[h][rt][e], c, -msub[rt]));
      }
#pragma unroll
      for (int rt = 0; rt < kRT; ++rt) {
        if constexpr (!TWO) {
          pa[rt] = pack8<_Float16>(pf[rt]);
        } else {
          float lo[8];
          pa[rt] = pack8<__bf16>(pf[rt]);
#pragma unroll
          for (int k = 0; k < 8; ++k) lo[k] = pf[rt][k] - (float)pa[rt][k];
          pl[rt] = pack8<__bf16>(lo);
        }
      }
    };
    auto tile_full = [&](int tile) {
      return __all(sValid[tile % 3][lane % kBK] != 0) && tile * kBK + kBK - 1 <= wave_lim;
    };

    // Cleared by the fast pass only: a clear in the exact pass could race a
    // slower wave's read of it.
    if (!EXACT && tid == 0) sBad = 0;
    if constexpr (EXACT)
      for (int i = tid; i < 3 * D; i += kThreads) sSeenBy[i] = 0x7fffffff;
    fetch_blocks(t0);
    if (t0 < te) {
      load_tile(t0);
      fetch_blocks(t0 + 1);
      __syncthreads();  // sBad or sSeenBy set, the previous pass or item done with LDS
      store_tile(t0, exact_c);
    }
    __syncthreads();

    const bool lag = map != 0;
    bool full_prev = false;
    if (!active) {
      for (int tile = t0; tile < te; ++tile) {
        if (tile + 1 < te) {
          load_tile(tile + 1);
          fetch_blocks(tile + 2);
          store_tile(tile + 1, exact_c);
        }
        __syncthreads();
      }
    } else {
      for (int tile = t0; tile < te; ++tile) {
        const bool more = tile + 1 < te;
        if (more) load_tile(tile + 1);
        const bool full = tile_full(tile);
        const int g = HS * tile;
        // The MFMA phases run at raised wave priority: the other wave's softmax
        // fills the issue slots in between.
        if (lag && tile > t0) softmax(g - 1, full_prev);
        __builtin_amdgcn_s_setprio(1);
        qk(g);
        if (tile > t0) pv(g - 1);
        __builtin_amdgcn_s_setprio(0);
        if (more) fetch_blocks(tile + 2);
        if constexpr (HS == 2) {
          softmax(g, full);
          __builtin_amdgcn_s_setprio(1);
          qk(g + 1);
          pv(g);
          __builtin_amdgcn_s_setprio(0);
        }
        if (!lag) softmax(g + HS - 1, full);
        full_prev = full;

        if (more) store_tile(tile + 1, exact_c);
        __syncthreads();
      }
      if (t0 < te) {
        if (lag) softmax(HS * te - 1, full_prev);
        pv(HS * te - 1);
      }
    }
    if constexpr (!EXACT) {
      // A V value that is infinite or NaN (in fp16, for bf16) makes accumulators
      // of every row of its step infinite or NaN, hidden ones (0 * inf) included.
      float acc = 0.f;
#pragma unroll
      for (int rt = 0; rt < kRT; ++rt)
#pragma unroll
        for (int m = 0; m < CH; ++m)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc += o[rt][m][e] * 0.f;
      if (__any(acc != 0.f)) sBad = 1;  // x * 0 is 0 for every finite x
    }
    __syncthreads();  // sBad final; LDS free for a second pass
    return !EXACT && sBad != 0;
  };

  if (run_tiles(std::false_type{})) {
    run_tiles(std::true_type{});
#pragma unroll
    for (int rt = 0; rt < kRT; ++rt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int last = __shfl(lim[rt], 4 * j + e, 64);
#pragma unroll
        for (int m = 0; m < CH; ++m) o[rt][m][e] += seen_v<D>(sSeenBy, 16 * m + n16, last);
      }
    __syncthreads();  // sSeenBy is set anew by the next pass
  }

  // ---- join the maps of rows wave_row0 + 16rt + 4j + e and store them, or
  // leave each map's rows as a partial (unnormalised) where the split cut the item
  const PrefillArgs ar1 = SPLIT ? reload_args() : args;
  const bool whole = !SPLIT || (t0 == 0 && t1 == nt);
  if (whole) {
    // The two waves of a pair finish half of its rows each: those of the
    // accumulators' elements 0 and 1 the first map's wave, 2 and 3 the second's.
    // Each scales its map (by 1 / l, or lambda / l) and hands the other's half over
    // in its own layout.
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    f32x2 *const meet = (f32x2 *)s_mem + (size_t)wave * kRT * CH * 64 + lane;
    const f32x2 *const from = (const f32x2 *)s_mem + (size_t)(wave ^ (kWaves / 2)) * kRT * CH * 64 + lane;
    const DiffParams &d = ar1.p.diff;
    const int e0 = 2 * map;  // the elements this wave finishes
    if (active) {
#pragma unroll
      for (int rt = 0; rt < kRT; ++rt) {
        f32x4 f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int row = wave_row0 + 16 * rt + 4 * j + e;
          const int tok = q0 + row / G;
          float x = 1.f;
          if (map == 1)
            x = row < ar1.bq * G && tok < n_new ? diff_lambda(d, qs + tok, kvh * G + row % G) : 0.f;
          f[e] = lsum[rt][e] > 0.f ? x / lsum[rt][e] : 0.f;
        }
#pragma unroll
        for (int m = 0; m < CH; ++m) {
          o[rt][m] *= f;
          meet[(rt * CH + m) * 64] =
              map == 0 ? (f32x2){o[rt][m][2], o[rt][m][3]} : (f32x2){o[rt][m][0], o[rt][m][1]};
        }
      }
    }
    __syncthreads();
    if (active) {
      float wt[CH];
#pragma unroll
      for (int m = 0; m < CH; ++m) wt[m] = d.weight != nullptr ? d.weight[16 * m + n16] : 1.f;
#pragma unroll
      for (int rt = 0; rt < kRT; ++rt) {
        f32x2 r[CH], ss = {0.f, 0.f};
#pragma unroll
        for (int m = 0; m < CH; ++m) {
          const f32x2 other = from[(rt * CH + m) * 64];
          r[m] = map == 0 ? (f32x2){o[rt][m][0], o[rt][m][1]} - other
                          : other - (f32x2){o[rt][m][2], o[rt][m][3]};
          ss += r[m] * r[m];
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int off = 1; off < 16; off <<= 1) ss[e] += shfl_xor(ss[e], off);
          const int row = wave_row0 + 16 * rt + 4 * j + e0 + e;
          const int tok = q0 + row / G;
          if (row >= ar1.bq * G || tok >= n_new) continue;
          // A row at or past max_query_len (a caller error) is marked with NaN.
          const float f = tok >= ar1.p.max_query_len ? __builtin_nanf("") : diff_factor(d, ss[e], D);
          T *dst = (T *)ar1.p.out + (int64_t)(qs + tok) * ar1.p.out_stride_token +
                   (int64_t)(kvh * G + row % G) * ar1.p.out_stride_head + n16;
#pragma unroll
          for (int m = 0; m < CH; ++m) dst[16 * m] = (T)(r[m][e] * (f * wt[m]));
        }
      }
    }
  } else {
    const int64_t prow = ((int64_t)(2 * L + (t0 == 0 ? 1 : 0)) * 2 + map) * kPairs;
    if (tid == 0) prefill_note(ar1.sp, L, it, G, t0 == 0, t1 == nt);
#pragma unroll
    for (int rt = 0; rt < kRT; ++rt) {
      if (j == 0) ar1.sp.ws_m[prow + wave_row0 + 16 * rt + n16] = m_run[rt];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = wave_row0 + 16 * rt + 4 * j + e;
        if (row >= ar1.bq * G || q0 + row / G >= n_new) continue;
        if (n16 == 0) ar1.sp.ws_l[prow + row] = lsum[rt][e];
        float *dst = ar1.sp.ws_o + (prow + row) * D + n16;
#pragma unroll
        for (int m = 0; m < CH; ++m) dst[16 * m] = o[rt][m][e];
      }
    }
  }
  if (t1 == nt && it.qt == ar1.n_qtiles - 1 && it.q_hi < n_new)
    prefill_nan_tail<T, D, kThreads>(ar1.p, it);
  // The pairs have been read, and every wave has read sBad, before the next
  // item writes either.
  if constexpr (SPLIT) __syncthreads();
  }
}

template <typename T, int D>
hipError_t launch_td(const PrefillParams &p, const PrefillSplit *sp, hipStream_t stream) {
  constexpr int kPairs = Shape<D>::kPairs;
  PrefillArgs args{};
  args.p = p;
  args.bq = kPairs / p.group;
  args.n_qtiles = max(1, (p.max_query_len + args.bq - 1) / args.bq);
  const int64_t total = (int64_t)p.num_seqs * p.num_kv_heads * args.n_qtiles;
  if (total <= 0) return hipSuccess;
  if (total > (int64_t)1 << 30) return hipErrorInvalidValue;
  if (sp != nullptr) {
    args.sp = *sp;
    hipLaunchKernelGGL((diff_prefill_mfma<T, D, true>), dim3((unsigned)sp->groups), dim3(kThreads),
                       0, stream, args);
    hipLaunchKernelGGL((diff_prefill_merge<T, D, kPairs>),
                       dim3((unsigned)sp->groups, kPairs / diff_merge_rows<D>()), dim3(256), 0, stream,
                       args);
    return hipGetLastError();
  }
  args.total = (int)total;
  hipLaunchKernelGGL((diff_prefill_mfma<T, D, false>), dim3((unsigned)((total + 7) / 8 * 8)),
                     dim3(kThreads), 0, stream, args);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_t(const PrefillParams &p, const PrefillSplit *sp, hipStream_t stream) {
  switch (p.head_dim) {
    case 64: return launch_td<T, 64>(p, sp, stream);
    case 128: return launch_td<T, 128>(p, sp, stream);
    case 256: return launch_td<T, 256>(p, sp, stream);
    default: return hipErrorInvalidValue;
  }
}

int pairs_of(int head_dim) {
  return head_dim == 256 ? Shape<256>::kPairs : Shape<128>::kPairs;
}

}  // namespace

// A wave's load instruction covers 512 / head_dim rows of one block; offsets
// inside a block are 32-bit byte offsets below 2^31; a query tile holds at least
// one token.
bool diff_prefill_mfma_covers(const PrefillParams &p, DType dt) {
  const uint64_t eb = 2, lim = (uint64_t)1 << 31;
  return (dt == DType::F16 || dt == DType::BF16) &&
         (p.head_dim == 64 || p.head_dim == 128 || p.head_dim == 256) &&
         (1 << p.block_shift) >= 512 / p.head_dim && p.group <= pairs_of(p.head_dim) &&
         (uint64_t)p.kv_stride_block * eb < lim &&
         ((uint64_t)p.kv_stride_token * eb << p.block_shift) < lim;
}

PrefillSplitShape diff_prefill_split_shape(const PrefillParams &p) {
  const int bk = p.head_dim == 256 ? Shape<256>::kBK : Shape<128>::kBK;
  const int64_t bq = max(1, pairs_of(p.head_dim) / p.group);
  const int64_t items = (p.max_query_len + bq - 1) / bq * p.num_seqs * p.num_kv_heads;
  const bool many = 4 * items > 9 * 8 * (int64_t)p.cus_per_xcd;
  return prefill_split_shape(p, pairs_of(p.head_dim), bk, 1, 1,
                             (many ? kSplitMinTokensMany : kSplitMinTokens) / bk, true);
}

hipError_t launch_diff_prefill_mfma(const PrefillParams &p, DType dt, const PrefillSplit *sp,
                                    hipStream_t stream) {
  if (dt == DType::BF16) return launch_t<__bf16>(p, sp, stream);
  if (dt == DType::F16) return launch_t<_Float16>(p, sp, stream);
  return hipErrorInvalidValue;
}

}  // namespace clv
