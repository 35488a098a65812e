// diff_prefill_f32.hip - differential attention of chunked prefill with fp32
// MFMAs (fp32 operands and accumulation throughout), over paged KV.
//
// A workgroup (4 waves, two or three workgroups per CU) takes kPairs = 32 rows = bq
// tokens x G query heads of one kv head: waves w and w + 2 hold the same 16
// rows, one map each, and meet through LDS at the end. Tiles of K and V go
// through a two-stage LDS ring, the global loads of tile k + 1 in flight while
// tile k is computed; items are split evenly over the workgroups
// (prefill_split.h). Fragments are those of the plain fp32 prefill, over the
// map's half of every key row: score MFMA (i, e) takes d = 16i + 4j + e of the
// half, o[4w + e] holds columns 64w + 4 n16 + e.
//
// Bound by the matrix core and by the vector instructions beside it, which add
// to its time rather than hide in it: a score is two chains of MFMAs and P.V of
// a tile one chain per column block, which joins the running accumulator once
// per tile (a sum over n tokens has n / 16 roundings in a row at most). Trees over
// chains of two, as in the plain form, cost 100 additions a tile more: 8 prompts
// of 2048 tokens, 6/6 heads of 128, 913 us against 844, 16/4 of 256 2437 and 2122.
// 8 x 1024 tokens of 6/6 heads run 215 us (90 TFLOP/s). Short prompts (17..512
// tokens, 50 us) are bound by what a workgroup waits for before its first tile
// and between items: schedule 2, cursor 3, Q and the first tile 2, an item's
// end 2..4 us, then 2.9 us per tile of 16 tokens with three workgroups per CU.
#include "prefill_split.h"

namespace clv {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * 64;
constexpr int kPairs = kWaves / 2 * 16;  // rows per workgroup

// Tokens per tile and workgroups per CU. At head_dim 128 tiles of 16 leave LDS
// and registers for three workgroups, against two with tiles of 32: 8 x 1024
// tokens 215 and 245 us, 17..512 tokens 52.6 and 52.1. At 64 three fit with 32
// (4 x 1024 tokens of 16/4 heads 166 us, two 177); 256 needs the registers of two.
template <int D> constexpr int tile_tokens() { return D == 64 ? 32 : 16; }
template <int D> constexpr int per_cu() { return D == 256 ? 2 : 3; }

template <int D> struct SplitCfg {
  static constexpr int kBK = tile_tokens<D>();
  // Items at 1/2/3/4 units, 23 batches of all head dims, sum: 2443, 2466, 2492,
  // 2532 us. kMinShare, kCutUnits at 48, 64, 96 and 128 tokens: equal within 0.5 %.
  static constexpr int kItemUnits = 1;
  static constexpr int kMinShare = 96 / kBK;
  static constexpr int kCutUnits = 96 / kBK;
  static __host__ __device__ __forceinline__ int tile_units(int) { return 1; }
  static __host__ __device__ __forceinline__ int snap(int share) { return max(1, share / 16); }
};

// Table width in tokens up to which a call is not split: 8 x 256 tokens of 6/6
// heads of 128 40.5 us unsplit and 43.3 split, 4 of 16/4 of 64 25.0 and 30.0
// (of 256 75.3 and 73.0); 8 x 512 of 6/6 94 and 82.
constexpr int kSplitMinTokens = 256;

__device__ __forceinline__ f32x4 mfma(uint32_t a, uint32_t b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, a),
                                              __builtin_bit_cast(float, b), c, 0, 0, 0);
}

// Four values of V (token `pos`, columns d0 ..) with 0 in the place of NaN and
// infinities, which only rows that see them may take (0 * inf is NaN):
// seen_by[column] remembers the first token with a NaN there, seen_by[D +
// column] with +inf, seen_by[2 D + column] with -inf.
template <int D>
__device__ __forceinline__ u32x4 finite_v4(u32x4 v, int pos, int d0, int *seen_by) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if ((v[e] & 0x7f800000u) != 0x7f800000u) continue;
    const int kind = (v[e] & 0x7fffffffu) != 0x7f800000u ? 0 : (v[e] >> 31) == 0 ? 1 : 2;
    atomicMin(&seen_by[kind * D + d0 + e], pos);
    v[e] = 0u;
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

template <int D, bool SPLIT>
__global__ void __launch_bounds__(kThreads, per_cu<D>())
diff_prefill_f32(const PrefillArgs args) {
  constexpr int kBK = tile_tokens<D>();
  constexpr int H = kBK / 16;            // 16-token steps per tile
  constexpr int NQK = D / 32;            // 16-byte Q / K words per lane of a half head
  constexpr int CH = D / 16;             // output blocks
  constexpr int ROW = D + 4;             // LDS row stride (floats)
  constexpr int CPR = D / 4;             // 16-byte chunks per row
  constexpr int RPP = kThreads / CPR;    // rows per load pass
  constexpr int PASSES = kBK / RPP;
  constexpr int WROWS = 64 / CPR;        // rows of one load instruction of a wave
  constexpr int kStage = kBK * ROW;
  static_assert(kWaves / 2 * CH * 64 * 16 <= 4 * kStage * 4, "the pairs meet in the tiles' memory");
  __shared__ __attribute__((aligned(16))) float s_kv[4 * kStage];  // K, K, V, V
  __shared__ __attribute__((aligned(4))) uint8_t sValid[2][kBK];
  __shared__ int sBad;            // V held a value that is not finite
  __shared__ int sSeenBy[3 * D];  // where, see finite_v4
  typedef PrefillSched<SplitCfg<D>> Sched;
  __shared__ int s_pre[SPLIT ? kPrefillSplitItems + 1 : 1];
  __shared__ int s_tmp[3 * kWaves];
  __shared__ int s_cur[kWaves][Sched::kCursorInts];
  float *const sK = s_kv, *const sV = s_kv + 2 * kStage;

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int map = wave / (kWaves / 2);
  const int wave_row0 = 16 * (wave % (kWaves / 2));
  const int n16 = lane & 15;
  const int j = lane >> 4;
  int L = SPLIT ? 0 : (int)(blockIdx.x % 8) * (int)(gridDim.x / 8) + (int)(blockIdx.x / 8);
  if constexpr (SPLIT) {
    Sched sched;
    sched.template init<kThreads>(args.p, args.bq, args.n_qtiles, args.sp.groups, s_pre, s_tmp);
    L = sched.group_of(blockIdx.x);
    if (L < 0) return;
    sched.start(L, s_cur[wave]);
    if (tid == 0) sched.clear_desc(args.sp, L);
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
      if (!Sched::next(p, bq, n_qtiles, s_pre, s_cur[wave], it, t0, t1, nt)) break;
    } else {
      if (!first) break;
      const int qt = n_qtiles - 1 - L % n_qtiles;  // longest query tiles first
      const int rest = L / n_qtiles;
      it.set(p, bq, rest / p.num_kv_heads, rest % p.num_kv_heads, qt);
      if (it.q0 >= it.n_new) break;
      nt = t1 = Sched::tiles(it.kv_end);
    }
    const int G = p.group;
    // A negative scale flips the sign of Q, a zero one becomes 2^-126: the
    // softmax multiplies by c > 0 only.
    const float c = fmaxf(fabsf(p.scale_log2), 0x1p-126f);
    const uint32_t qflip = p.scale_log2 < 0.f ? 0x80000000u : 0u;

    const char *kbase = (const char *)p.k_cache + (int64_t)it.kvh * p.kv_stride_head * 4;
    const char *vbase = (const char *)p.v_cache + (int64_t)it.kvh * p.kv_stride_head * 4;
    const int kv_end = it.kv_end;
    const int te = min(t1, (kv_end + kBK - 1) / kBK);  // 0 tokens: no tile at all

    // The map's half of Q (B operand) of this lane's row wave_row0 + n16.
    u32x4 q[NQK];
    int lim;  // last visible position of the row (-1: no row)
    {
      const int r = wave_row0 + n16;
      const int tok = it.q0 + r / G;
      const bool ok = r < bq * G && tok < it.n_new;
      lim = ok ? it.base_pos + tok : -1;
      const float *qrow = (const float *)p.q + (int64_t)(it.qs + (ok ? tok : it.q0)) * p.q_stride_token +
                          (int64_t)(it.kvh * G + (ok ? r % G : 0)) * p.q_stride_head +
                          map * (D / 2) + 4 * j;
#pragma unroll
      for (int i = 0; i < NQK; ++i) {
        q[i] = load_vec<u32x4>(qrow + 16 * i);
        q[i] ^= qflip;
        if (!ok) q[i] = (u32x4){0u, 0u, 0u, 0u};
      }
    }
    // Causal limits of the wave's first and last real rows: tiles at or below
    // the first need no mask, tiles past the last are left out by this wave.
    const int rows = (it.q_hi - it.q0) * G;
    int lim_first = -1, te_w = t0;
    if (wave_row0 < rows) {
      lim_first = it.base_pos + it.q0 + wave_row0 / G;
      const int lim_last = it.base_pos + it.q0 + min(wave_row0 + 15, rows - 1) / G;
      te_w = max(t0, min(te, lim_last < 0 ? 0 : lim_last / kBK + 1));
    }

    // Tile loader: thread handles chunk tid % CPR of rows tid / CPR + RPP * i;
    // the rows of one load instruction lie in one block (block_size >= WROWS).
    // Unreadable tokens read zeros from the buffer resource's range check.
    const int lchunk = tid % CPR;
    const int lrow = tid / CPR;
    const int wrow = WROWS * wave;
    const uint32_t sblk32 = (uint32_t)(p.kv_stride_block * 4), stok32 = (uint32_t)(p.kv_stride_token * 4);
    const uint32_t bmask = (1u << p.block_shift) - 1u;
    const uint32_t lane_off = (uint32_t)(lrow - wrow) * stok32 + (uint32_t)lchunk * 16u;
    typedef const int32_t __attribute__((address_space(4))) *cint_t;
    const cint_t brow = (cint_t)(p.block_tables + (int64_t)it.s * p.max_blocks_per_seq);
    u32x4 kreg[PASSES], vreg[PASSES];
    bool rvalid[PASSES];
    int rblk[PASSES];
    auto fetch_blocks = [&](int tile) {
#pragma unroll
      for (int i = 0; i < PASSES; ++i) {
        const int t = tile * kBK + wrow + RPP * i;
        rblk[i] = (tile < te && t < kv_end) ? brow[t >> p.block_shift] : -1;
      }
    };
    auto load_tile = [&](int tile) {
#pragma unroll
      for (int i = 0; i < PASSES; ++i) {
        const uint32_t t = (uint32_t)(tile * kBK + wrow + RPP * i);
        const bool bok = (unsigned)rblk[i] < (unsigned)p.num_blocks;
        const bool ok = bok && (int)t + (lrow - wrow) < kv_end;
        rvalid[i] = ok;
        const uint64_t boff = (uint64_t)(uint32_t)(bok ? rblk[i] : 0) * sblk32;
        const int nrec = bok ? (int)(stok32 * bmask) + D * 4 : 0;
        const uint32_t voff = ok ? (t & bmask) * stok32 + lane_off : 0x80000000u;
        kreg[i] = buf_load<u32x4>(make_rsrc_range(kbase + boff, nrec), voff);
        vreg[i] = buf_load<u32x4>(make_rsrc_range(vbase + boff, nrec), voff);
      }
    };
    auto store_tile = [&](int tile) {
      const int buf = tile & 1;
      bool bad = false;
#pragma unroll
      for (int i = 0; i < PASSES; ++i) {
        const int row = lrow + RPP * i;
        store_vec<u32x4>(&sK[buf * kStage + row * ROW + lchunk * 4], kreg[i]);
        if (lchunk == 0) sValid[buf][row] = rvalid[i] ? 1 : 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) bad |= (vreg[i][e] & 0x7f800000u) == 0x7f800000u;
      }
      if (__any(bad)) {
        sBad = 1;
#pragma unroll
        for (int i = 0; i < PASSES; ++i)
          vreg[i] = finite_v4<D>(vreg[i], tile * kBK + lrow + RPP * i, 4 * lchunk, sSeenBy);
      }
#pragma unroll
      for (int i = 0; i < PASSES; ++i)
        store_vec<u32x4>(&sV[buf * kStage + (lrow + RPP * i) * ROW + lchunk * 4], vreg[i]);
    };

    f32x4 o[CH];
    float m_run = kNegInf, l_run = 0.f;
#pragma unroll
    for (int m = 0; m < CH; ++m) o[m] = (f32x4){0.f, 0.f, 0.f, 0.f};

    fetch_blocks(t0);
    if (tid == 0) sBad = 0;
    for (int i = tid; i < 3 * D; i += kThreads) sSeenBy[i] = 0x7fffffff;
    __syncthreads();
    if (t0 < te) {
      load_tile(t0);
      fetch_blocks(t0 + 1);
      store_tile(t0);  // the item before this one ended with a barrier
    }
    __syncthreads();

    for (int tile = t0; tile < te; ++tile) {
      const int buf = tile & 1;
      const bool more = tile + 1 < te;
      if (more) {
        load_tile(tile + 1);
        fetch_blocks(tile + 2);
      }
      if (tile < te_w) {
        const float *K = sK + buf * kStage + map * (D / 2);
        const float *V = sV + buf * kStage;
        // Scores: two chains of MFMAs.
        f32x4 sacc[H];
#pragma unroll
        for (int h = 0; h < H; ++h) {
          f32x4 ch[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
          for (int i = 0; i < NQK; ++i) {
            const u32x4 k = load_vec<u32x4>(&K[(16 * h + n16) * ROW + 16 * i + 4 * j]);
#pragma unroll
            for (int e = 0; e < 4; ++e) ch[e & 1] = mfma(k[e], q[i][e], ch[e & 1]);
          }
          sacc[h] = ch[0] + ch[1];
        }
        const bool full = __all(sValid[buf][lane % kBK] != 0) && tile * kBK + kBK - 1 <= lim_first;
        // Scores a row may not see become -inf.
        if (!full) {
#pragma unroll
          for (int h = 0; h < H; ++h) {
            const uint32_t vf = *reinterpret_cast<const uint32_t *>(&sValid[buf][16 * h + 4 * j]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const bool readable = ((vf >> (8 * e)) & 1u) != 0;
              if (!(readable && tile * kBK + 16 * h + 4 * j + e <= lim)) sacc[h][e] = kNegInf;
            }
          }
        }
        float mx = kNegInf;
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e) mx = fmaxf(mx, sacc[h][e]);
        mx = fmaxf(mx, shfl_xor(mx, 16));
        mx = fmaxf(mx, shfl_xor(mx, 32));
        const float m_new = fmaxf(m_run, mx);
        const float msub = m_new == kNegInf ? 0.f : m_new;
        const float alpha = fast_exp2((m_run - msub) * c);
        m_run = m_new;
        float pr[H][4], psum = 0.f;
#pragma unroll
        for (int h = 0; h < H; ++h) {
#pragma unroll
          for (int e = 0; e < 4; ++e) pr[h][e] = fast_exp2((sacc[h][e] - msub) * c);
          psum += (pr[h][0] + pr[h][1]) + (pr[h][2] + pr[h][3]);
        }
        l_run = l_run * alpha + psum;
        float ar[4];  // alpha of the accumulator's rows 4j + r
#pragma unroll
        for (int r = 0; r < 4; ++r) ar[r] = shfl(alpha, 4 * j + r);

#pragma unroll
        for (int w = 0; w < CH / 4; ++w) {
          u32x4 v[H][4];
#pragma unroll
          for (int h = 0; h < H; ++h)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              v[h][k] = load_vec<u32x4>(&V[(16 * h + 4 * j + k) * ROW + 64 * w + 4 * n16]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
              for (int h = 0; h < H; ++h)
                sum = mfma(__builtin_bit_cast(uint32_t, pr[h][k]), v[h][k][e], sum);
#pragma unroll
            for (int r = 0; r < 4; ++r)
              o[4 * w + e][r] = __builtin_fmaf(o[4 * w + e][r], ar[r], sum[r]);
          }
        }
      }
      if (more) store_tile(tile + 1);
      __syncthreads();
    }

    if (sBad != 0) {  // the last tile's barrier made it final
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int last = __shfl(lim, 4 * j + r, 64);
#pragma unroll
        for (int m = 0; m < CH; ++m)
          o[m][r] += seen_v<D>(sSeenBy, 64 * (m >> 2) + 4 * n16 + (m & 3), last);
      }
    }
    l_run += shfl_xor(l_run, 16);
    l_run += shfl_xor(l_run, 32);
    // The rest of the arguments are read only now.
    const PrefillArgs ar1 = SPLIT ? reload_args() : args;
    const bool whole = !SPLIT || (t0 == 0 && t1 == nt);
    float lr[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) lr[r] = shfl(l_run, 4 * j + r);
    if (whole) {
      // The second map's rows go to the first map's wave in its own layout.
      const DiffParams &d = ar1.p.diff;
      f32x4 *meet = (f32x4 *)s_kv + (size_t)(wave % (kWaves / 2)) * CH * 64 + lane;
      if (map == 1 && wave_row0 < rows) {
        f32x4 f;  // lambda / l of row 4j + r
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int row = wave_row0 + 4 * j + r;
          const float lam =
              row < rows ? diff_lambda(d, it.qs + it.q0 + row / G, it.kvh * G + row % G) : 0.f;
          f[r] = lr[r] > 0.f ? lam / lr[r] : 0.f;
        }
#pragma unroll
        for (int m = 0; m < CH; ++m) meet[m * 64] = o[m] * f;
      }
      __syncthreads();
      if (map == 0 && wave_row0 < rows) {
        f32x4 inv, ss = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int r = 0; r < 4; ++r) inv[r] = lr[r] > 0.f ? 1.f / lr[r] : 0.f;
#pragma unroll
        for (int m = 0; m < CH; ++m) {
          o[m] = o[m] * inv - meet[m * 64];
          ss += o[m] * o[m];
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
#pragma unroll
          for (int off = 1; off < 16; off <<= 1) ss[r] += shfl_xor(ss[r], off);
          const int row = wave_row0 + 4 * j + r;
          if (row >= rows) continue;
          const int tok = it.q0 + row / G;
          // A row at or past max_query_len (a caller error) is marked with NaN.
          const float f = tok >= ar1.p.max_query_len ? __builtin_nanf("") : diff_factor(d, ss[r], D);
          float *dst = (float *)ar1.p.out + (int64_t)(it.qs + tok) * ar1.p.out_stride_token +
                       (int64_t)(it.kvh * G + row % G) * ar1.p.out_stride_head;
#pragma unroll
          for (int w = 0; w < CH / 4; ++w) {
            f32x4 v = {o[4 * w][r], o[4 * w + 1][r], o[4 * w + 2][r], o[4 * w + 3][r]};
            v *= f;
            if (d.weight != nullptr) v *= load_vec<f32x4>(d.weight + 64 * w + 4 * n16);
            store_vec<f32x4>(dst + 64 * w + 4 * n16, v);
          }
        }
      }
    } else {
      const int64_t prow = ((int64_t)(2 * L + (t0 == 0 ? 1 : 0)) * 2 + map) * kPairs;
      if (tid == 0) prefill_note(ar1.sp, L, it, G, t0 == 0, t1 == nt);
      if (j == 0 && wave_row0 + n16 < rows) {
        ar1.sp.ws_m[prow + wave_row0 + n16] = m_run;
        ar1.sp.ws_l[prow + wave_row0 + n16] = l_run;
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = wave_row0 + 4 * j + r;
        if (row >= rows) continue;
        float *dst = ar1.sp.ws_o + (prow + row) * D;
#pragma unroll
        for (int w = 0; w < CH / 4; ++w)
          store_vec<f32x4>(dst + 64 * w + 4 * n16,
                           (f32x4){o[4 * w][r], o[4 * w + 1][r], o[4 * w + 2][r], o[4 * w + 3][r]});
      }
    }
    if (t1 == nt && it.qt == ar1.n_qtiles - 1 && it.q_hi < it.n_new)
      prefill_nan_tail<float, D, kThreads>(ar1.p, it);
    // The pairs have been read before the next item stages its tiles.
    if constexpr (SPLIT) __syncthreads();
  }
}

template <int D>
hipError_t launch_td(const PrefillParams &p, const PrefillSplit *sp, hipStream_t stream) {
  PrefillArgs args{};
  args.p = p;
  args.bq = kPairs / p.group;
  args.n_qtiles = max(1, (p.max_query_len + args.bq - 1) / args.bq);
  const int64_t total = (int64_t)p.num_seqs * p.num_kv_heads * args.n_qtiles;
  if (total > (int64_t)1 << 30) return hipErrorInvalidValue;
  if (sp != nullptr) {
    args.sp = *sp;
    hipLaunchKernelGGL((diff_prefill_f32<D, true>), dim3((unsigned)sp->groups), dim3(kThreads), 0,
                       stream, args);
    hipLaunchKernelGGL((diff_prefill_merge<float, D, kPairs>),
                       dim3((unsigned)sp->groups, kPairs / diff_merge_rows<D>()), dim3(256), 0, stream,
                       args);
    return hipGetLastError();
  }
  args.total = (int)total;
  hipLaunchKernelGGL((diff_prefill_f32<D, false>), dim3((unsigned)((total + 7) / 8 * 8)),
                     dim3(kThreads), 0, stream, args);
  return hipGetLastError();
}

}  // namespace

// One load instruction of a wave covers 256 / head_dim rows of one block, and
// offsets inside a block are 32-bit bytes.
bool diff_prefill_f32_covers(const PrefillParams &p) {
  const uint64_t lim = (uint64_t)1 << 31;
  return (p.head_dim == 64 || p.head_dim == 128 || p.head_dim == 256) &&
         (1 << p.block_shift) >= 4 && p.group <= kPairs &&
         (uint64_t)p.kv_stride_block * 4 < lim &&
         ((uint64_t)p.kv_stride_token * 4 << p.block_shift) < lim;
}

PrefillSplitShape diff_prefill_f32_split_shape(const PrefillParams &p) {
  const int bk = p.head_dim == 64 ? tile_tokens<64>() : tile_tokens<128>();
  const int per = p.head_dim == 256 ? per_cu<256>() : per_cu<128>();
  return prefill_split_shape(p, kPairs, bk, per, 1, kSplitMinTokens / bk, false);
}

hipError_t launch_diff_prefill_f32(const PrefillParams &p, const PrefillSplit *sp,
                                   hipStream_t stream) {
  switch (p.head_dim) {
    case 64: return launch_td<64>(p, sp, stream);
    case 128: return launch_td<128>(p, sp, stream);
    case 256: return launch_td<256>(p, sp, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace clv
