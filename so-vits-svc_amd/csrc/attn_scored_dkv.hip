// attn_scored_dkv.hip — svc_attn_scored_bwd's walk over the queries: dk and dv.
//
// dv[:, s] = sum_t Z P dO[:, t], dk[:, s] = sum_t dS q[:, t]: four products, k's and v's columns and both results in registers, the query heads that share a
// key head one after the other, so that their sum needs no second pass.  At 128 channels that is a wave a SIMD (376 registers): the vector unit's part
// (1900 cycles of the 32 x 32 scores, against 1024 of the matrix unit) then stands beside the matrix unit's only as far as the compiler interleaves
// them.  Short walks wait behind loads and barriers (documents 52 %, windows 57 % of the waves' cycles).  Measured (kernel traces of passes one behind the other): bf16,
// 128 channels, 16 query and 4 key heads, 4 x 4096 x 4096 causal with a cap 1038 to 1043 us = 528 TFLOP/s of its four products; bf16,
// 64 channels, 9 documents in 4099 with bias and dropout 130 us; fp16, window of 128 in 1501 92 us; fp32, 96 channels, 16 ragged items of up to 790 190 us.
#include "attn_scored.h"

namespace attn {

template <int J> __device__ __forceinline__ unsigned quad(unsigned v) {      // lane J of the own four
  return (unsigned)__builtin_amdgcn_mov_dpp((int)v, J * 0x55, 0xf, 0xf, true);
}

// 128 keys of one key head a workgroup (32 a wave), walking the query tiles of its query heads that see any of them.
template <typename E, int DP, bool EXACT, bool DROP>
__global__ __launch_bounds__(256, (sizeof(E) == 4 ? DP <= 32 : DP <= 64) ? 2 : 1) void dkv_kernel(svc_attn_scored_t a, Ws ws, int n_tiles) {
  constexpr int RB = 128;
  // One wave a SIMD (128 channels' accumulators): dP's product is put before the exponentials, which then need not wait behind it, and the compiler orders
  // the rest as it likes (128 channels, 4096 x 4096 causal: 1320 -> 1040 us).  Two waves fill each other's gaps and have no registers for it.
  constexpr bool EARLY = sizeof(E) == 2 && DP > 64;
  // (DROP is a.seed != null.  Kernels of two waves still ask for it at run time: without the branch the compiler moves the draws' registers across the
  // products, 34 spills, 134 -> 172 us at 64 channels.  Without the draws' code at all the same kernel takes 97 us instead of 102.)
  typedef Tile<E, RB> TL;
  constexpr int N = TL::N, RT = TL::RT;
  __shared__ __align__(16) char tiles_[2 * Staged<E, DP, RB>::BUFS * Staged<E, DP, RB>::SIZE * sizeof(E)];
  __shared__ float win[2][NCOL + N];
  __shared__ __align__(16) float lses[2][N], rows[2][N];
  __shared__ __align__(16) int2 ivs[2][N];
  __shared__ float red[8];
  E* const tiles = (E*)tiles_;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5, n = lane & 31, rep = a.H / a.G;
  const Place at = place_of(blockIdx.x, a.B * a.G, 1, n_tiles);
  if (at.group >= a.B * a.G) return;
  // (under a causal mask the first keys are the heaviest)
  const int bg = at.group, c0 = (n_tiles - 1 - at.tile) * NCOL, b = bg / a.G, kvh = bg % a.G;
  const int w0 = c0 + wave * 32, sl = wave * 32 + n, s = c0 + sl;
  Columns<E, DP, RB> kc, vc;
  kc.fetch((const E*)a.k + b * a.k_bs + (long long)kvh * a.dk * a.k_cs, a.k_cs, a.dk, a.Tk, c0, tid);
  vc.fetch((const E*)a.v + b * a.v_bs + (long long)kvh * a.dk * a.v_cs, a.v_cs, a.dk, a.Tk, c0, tid);
  const int off = item_offset(a, b);
  int tbeg, tend, kbeg, kend;
  live_range(a, b, tbeg, tend, kbeg, kend);
  const ScoreScale sc = score_scale(a);
  unsigned thr = 0;
  float keep = 1.f;
  unsigned long long start = 0;
  const unsigned long long ng = (unsigned long long)((a.Tk + 3) >> 2);
  if (DROP && (EARLY || a.seed)) {
    start = draw_start(a) + ((unsigned long long)(s >> 2) + (unsigned long long)(8 * h + (n & 3)) * ng) * DRAW_STEP;      // row 8 h + (n & 3) of a block
    thr = (unsigned)rintf(a.p_drop * 65536.f);
    keep = 65536.f / (65536.f - (float)thr);
  }
  f32x16 ak[DP / 32], av[DP / 32];
#pragma unroll
  for (int i = 0; i < DP / 32; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) ak[i][r] = av[i][r] = 0.f;

  // The walk: (query head, tile) pairs whose tile has a query that sees a key of the workgroup's.  Which tiles do is the same for every head: lane i looks
  // at tile base + i of 64, and the walk follows the ballot's bits (looking at one tile after the other, each a dependent load, took longer than the
  // work where masks leave few: 9 documents in 4099 queries 143 -> 134 us).
  const int t32 = (a.Tq + 31) / 32, nt = (a.Tq + N - 1) / N;
  const int4* const spans = ws.tiles + (long long)b * t32;
  int base = -64;
  unsigned long long left = 0;
  int4 mine = make_int4(0, 0, 0, 0);
  auto advance = [&](int& hh, int& t0, int4& r) {            // to the next pair; hh = rep: none
    while (left == 0) {
      base += 64;
      if (base >= nt) {
        base = 0;
        if (++hh >= rep) return;
      }
      const int tile = base + lane, i = min(tile * RT, t32 - 1);
      mine = spans[i];
      if (RT == 2) {
        const int4 m1 = spans[min(i + 1, t32 - 1)];
        mine = make_int4(min(mine.x, m1.x), max(mine.y, m1.y), max(mine.z, m1.z), min(mine.w, m1.w));
      }
      left = __ballot(tile < nt && mine.x < c0 + NCOL && mine.y > c0);
    }
    const int bit = __builtin_ctzll(left);
    left &= left - 1;
    t0 = (base + bit) * N;
    r = make_int4(__builtin_amdgcn_readlane(mine.x, bit), __builtin_amdgcn_readlane(mine.y, bit), __builtin_amdgcn_readlane(mine.z, bit),
                  __builtin_amdgcn_readlane(mine.w, bit));
  };
  Source<E, DP, RB> qsrc, gsrc;
  Pre<E, DP, RB> qf, gf;
  float bf = 0.f, lf = 0.f, rf = 0.f;
  int2 vf = make_int2(0, 0);
  auto fetch = [&](int hh, int t0) {
    const int head = kvh * rep + hh;
    const long long bh = (long long)b * a.H + head;
    qsrc.set((const E*)a.q + b * a.q_bs + (long long)head * a.dk * a.q_cs, a.q_cs, a.dk, a.Tq, tid);
    gsrc.set((const E*)a.dout + b * a.do_bs + (long long)head * a.dk * a.do_cs, a.do_cs, a.dk, a.Tq, tid);
    qsrc.fetch(qf, t0, tid);
    gsrc.fetch(gf, t0, tid);
    if (a.bias)
      bf = bias_entry(a.bias + (a.bias_heads > 1 ? (long long)head * (2 * a.bias_w + 1) : 0), a.bias_w, c0 - (off + t0) - (N - 1), tid);
    const int t = min(t0 + (tid & (N - 1)), a.Tq - 1);
    lf = a.lse[bh * a.Tq + t];
    rf = ws.rowsum[bh * a.Tq + t];
    vf = ws.iv[(long long)b * a.Tq + t];
  };
  int hh = 0, t0 = 0, buf = 0;
  int4 r = make_int4(0, 0, 0, 0);
  advance(hh, t0, r);
  if (hh < rep) fetch(hh, t0);
  const float g2 = operand_scale<E>(a, ws, b, kvh, red), pup = exp2f(PUP<E>), gm = g2 / pup;
  typename Frag<E>::template Head<DP> k, v;
  kc.settle(k, tiles, c0, kbeg, kend, tid);
  vc.settle(v, tiles, c0, kbeg, kend, tid);
  __syncthreads();                                           // (the keys' columns have been read from the tiles)
  while (hh < rep) {
    if (Staged<E, DP, RB>::BUFS == 1) __syncthreads();
    E* const qs = tiles + buf * 2 * Staged<E, DP, RB>::SIZE;
    E* const gs = qs + Staged<E, DP, RB>::SIZE;
    qsrc.commit(qs, qf, t0, tbeg, tend, tid);
    gsrc.commit(gs, gf, t0, tbeg, tend, tid);
    if (a.bias && tid < NCOL + N) win[buf][tid] = bias_scaled(bf);
    if (tid < N) {
      const bool in = t0 + tid < a.Tq;
      lses[buf][tid] = in ? lf - PUP<E> : 0.f;
      rows[buf][tid] = in ? rf : 0.f;
      ivs[buf][tid] = in ? vf : make_int2(0, 0);
    }
    __syncthreads();
    const int head = kvh * rep + hh, now = t0;
    const bool work = r.x < w0 + 32 && r.y > w0, whole = w0 >= r.z && w0 + 32 <= r.w && now + N <= a.Tq;
    advance(hh, t0, r);
    fetch(min(hh, rep - 1), t0);                             // (behind the last pair: values that are not used)
    const int cur = buf;
    if (Staged<E, DP, RB>::BUFS == 2) buf ^= 1;
    if (!work) continue;
#pragma unroll 1
    for (int rt = 0; rt < RT; ++rt) {
      const f32x16 u = mul_columns<E, DP, RB>(qs, rt, k, lane);
      f32x16 dp;
      if constexpr (EARLY) dp = mul_columns<E, DP, RB>(gs, rt, v, lane);
      float x[16], th[16], p[16], mul = sc.mul;
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = u[i];
      if (sc.cap) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          th[i] = cap_tanh<EXACT>(x[i], sc);
          x[i] = th[i] * sc.cap_out;
        }
        mul = 1.f;
      }
      if (a.bias) {
        const float* w = win[cur] + (N - 1) - 32 * rt + sl;
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = fmaf(x[i], mul, w[-pos_of(i, h)]);
        mul = 1.f;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = __builtin_amdgcn_exp2f(fmaf(x[i], mul, -lses[cur][32 * rt + pos_of(i, h)]));
      if (!whole) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int2 w = ivs[cur][32 * rt + pos_of(i, h)];
          x[i] = s >= w.x && s < w.y ? x[i] : 0.f;
        }
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) p[i] = x[i];
      unsigned gone = 0;                                     // dropped entries' bits
      if (DROP && (EARLY || a.seed)) {
        // A word holds the draws of four neighbouring keys, which are four neighbouring lanes: lane j of the four works out the word of row 4w + j and
        // all of them read it from there, each its own field (into the upper half, to compare in place).
        const unsigned long long row = (unsigned long long)(((long long)b * a.H + head) * a.Tq + now + 32 * rt) * ng * DRAW_STEP;
        const unsigned field = 0x01000c0cu + (n & 3) * 0x02020000u;      // bytes 2 f + 1, 2 f, zero, zero
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const unsigned long long z = draw_word(start + row + (unsigned long long)(16 * (w >> 1) + 4 * (w & 1)) * ng * DRAW_STEP);
          const unsigned lo = (unsigned)z, hi = (unsigned)(z >> 32);
          auto one = [&](int i, unsigned l, unsigned g) {
            const bool drop = __builtin_amdgcn_perm(g, l, field) < thr << 16;
            p[i] = drop ? 0.f : x[i] * keep;
            if constexpr (!X3<E>) gone |= drop ? 1u << i : 0u;
          };
          one(4 * w, quad<0>(lo), quad<0>(hi));
          one(4 * w + 1, quad<1>(lo), quad<1>(hi));
          one(4 * w + 2, quad<2>(lo), quad<2>(hi));
          one(4 * w + 3, quad<3>(lo), quad<3>(hi));
        }
      }
      // dv's product before dP's: P as an operand takes half the registers that dP will
      if constexpr (!EARLY) __builtin_amdgcn_sched_barrier(0);
      mul_rows<E, DP, 1, RB>(av, gs, rt, p, lane);
      if constexpr (!EARLY) {
        __builtin_amdgcn_sched_barrier(0);
        dp = mul_columns<E, DP, RB>(gs, rt, v, lane);
      }
      if constexpr (X3<E>) {
        // P (Z dP - D) = (Z P) dP - P D needs no dropped bits, at sixteen registers that the 16-bit kernels lack
        // (64 channels with dropout: 13 spills and 138-149 us against 133; fp32 at 96: 199 us against 217)
#pragma unroll
        for (int i = 0; i < 16; ++i) dp[i] = fmaf(p[i], dp[i], -(x[i] * rows[cur][32 * rt + pos_of(i, h)]));
      } else {
        if (DROP && (EARLY || a.seed)) {
#pragma unroll
          for (int i = 0; i < 16; ++i) dp[i] = gone >> i & 1 ? 0.f : dp[i] * keep;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) dp[i] -= rows[cur][32 * rt + pos_of(i, h)];
      }
      if (sc.cap) {
#pragma unroll
        for (int i = 0; i < 16; ++i) dp[i] *= fmaf(-th[i], th[i], 1.f);
      }
      // a masked entry: 0 whatever dO.v and the cap's factor are (no query need see the key, which may then hold anything); a nan P is not one
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float g = X3<E> ? dp[i] : x[i] * dp[i];
        x[i] = whole || x[i] != 0.f ? g : 0.f;
      }
      if constexpr (__is_same(E, f16_t)) {
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] *= gm;
      }
      mul_rows<E, DP, 1, RB>(ak, qs, rt, x, lane);
    }
  }
  if (s >= a.Tk) return;
  const float os = a.scale / g2, ov = 1.f / pup;
  E* dk = (E*)a.dk_ + (long long)bg * a.dk * a.Tk + s;
  E* dv = (E*)a.dv + (long long)bg * a.dk * a.Tk + s;
#pragma unroll
  for (int i = 0; i < DP / 32; ++i)
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const int d = 32 * i + 8 * (j >> 2) + 4 * h + (j & 3);
      if (d < a.dk) {
        dk[(long long)d * a.Tk] = (E)(ak[i][j] * os);
        dv[(long long)d * a.Tk] = (E)(av[i][j] * ov);
      }
    }
}

template <typename E, int DP>
static void go(const svc_attn_scored_t& a, const Ws& w, hipStream_t s) {
  const int n_tiles = (a.Tk + NCOL - 1) / NCOL;
  const unsigned grid = (unsigned)grid_of((long long)a.B * a.G, 1, n_tiles);
  const bool exact = sizeof(E) == 4 || a.dbias || a.softcap > SHORT_CAP;
  if (exact && a.seed) hipLaunchKernelGGL((dkv_kernel<E, DP, true, true>), dim3(grid), dim3(256), 0, s, a, w, n_tiles);
  else if (exact) hipLaunchKernelGGL((dkv_kernel<E, DP, true, false>), dim3(grid), dim3(256), 0, s, a, w, n_tiles);
  else if (a.seed) hipLaunchKernelGGL((dkv_kernel<E, DP, sizeof(E) == 4, true>), dim3(grid), dim3(256), 0, s, a, w, n_tiles);
  else hipLaunchKernelGGL((dkv_kernel<E, DP, sizeof(E) == 4, false>), dim3(grid), dim3(256), 0, s, a, w, n_tiles);
}
template <typename E>
static void pick(const svc_attn_scored_t& a, const Ws& w, hipStream_t s) {
  if (a.dk <= 32) go<E, 32>(a, w, s);
  else if (a.dk <= 64) go<E, 64>(a, w, s);
  else if (a.dk <= 96 || X3<E>) go<E, 96>(a, w, s);
  else go<E, X3<E> ? 96 : 128>(a, w, s);
}
void launch_dkv(const svc_attn_scored_t& a, const Ws& w, hipStream_t s) {
  // (three planes of k's and v's columns at 128 channels do not fit the registers beside both accumulators)
  if (a.dtype == SVC_F32 && a.dk > 96) go<float, 128>(a, w, s);
  else if (a.dtype == SVC_F32) pick<x3_t>(a, w, s);
  else if (a.dtype == SVC_BF16) pick<bf16_t>(a, w, s);
  else pick<f16_t>(a, w, s);
}

}  // namespace attn
