// attn_scored_dq.hip — svc_attn_scored_bwd's walk over the keys: dq and the bias gradient.
//
// P = exp2(x - lse) again from q and k, dP = Z (dO.v), dS = P (dP - D): three products, with q's and dO's columns in registers throughout.  The vector
// unit bounds it on long rows (scores as in the forward, and the mask, D and cap factors of dS); on short walks loads and barriers do (waits 40 to 43 % of the waves'
// cycles).  Measured (kernel traces of passes one behind the other): bf16, 128 channels, 4 x 16 heads, 4096 x 4096 causal with a
// cap 566 to 572 us = 720 to 728 TFLOP/s of its three products; bf16, 64 channels, 9 documents in 4099 with bias and dropout 68 us; fp16, window of 128 in 1501 with
// the bias's gradient 88 us; fp32, 96 channels, 16 ragged items of up to 790 123 us.
#include "attn_scored.h"

namespace attn {

// lane l's value from lane l + 1 (0x130) or l - 1 (0x138), 0 from outside the wave
template <int CTRL> __device__ __forceinline__ float lane_shift(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}

// 128 queries of one head a workgroup (32 a wave), walking the key tiles that any of them sees.
template <typename E, int DP, bool EXACT>
__global__ __launch_bounds__(256, (sizeof(E) == 4 ? DP <= 32 : DP <= 128) ? 2 : 1) void dq_kernel(svc_attn_scored_t a, Ws ws, int n_tiles) {
  constexpr int RB = sizeof(E) == 2 && DP == 128 ? 64 : 128;
  typedef Tile<E, RB> TL;
  constexpr int N = TL::N, RT = TL::RT, NB = N + 32;
  __shared__ __align__(16) char tiles_[2 * Staged<E, DP, RB>::BUFS * Staged<E, DP, RB>::SIZE * sizeof(E)];
  __shared__ float win[2][NCOL + N];
  __shared__ float bin_[4][2][NB];
  __shared__ float red[8];
  E* const tiles = (E*)tiles_;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5, n = lane & 31;
  const Place at = place_of(blockIdx.x, a.B * a.G, a.H / a.G, n_tiles);
  if (at.group >= a.B * a.G) return;
  const int b = at.group / a.G, kvh = at.group % a.G, head = kvh * (a.H / a.G) + at.sub, t0 = at.tile * NCOL;
  const long long bh = (long long)b * a.H + head;

  const int tl = wave * 32 + n, t = t0 + tl, off = item_offset(a, b);
  Columns<E, DP, RB> qc, gc;
  qc.fetch((const E*)a.q + b * a.q_bs + (long long)head * a.dk * a.q_cs, a.q_cs, a.dk, a.Tq, t0, tid);
  gc.fetch((const E*)a.dout + b * a.do_bs + (long long)head * a.dk * a.do_cs, a.do_cs, a.dk, a.Tq, t0, tid);
  const int2 iv = t < a.Tq ? ws.iv[(long long)b * a.Tq + t] : make_int2(0, 0);
  const bool some = iv.y > iv.x;
  // the four waves' key ranges, and the range that every query of this wave sees whole
  const int t32 = (a.Tq + 31) / 32;
  const int4* const spans = ws.tiles + (long long)b * t32;
  int blo = a.Tk, bhi = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const int4 r = spans[min((t0 >> 5) + w, t32 - 1)];
    blo = min(blo, r.x);
    bhi = max(bhi, r.y);
  }
  const int4 mine = (t0 >> 5) + wave < t32 ? spans[min((t0 >> 5) + wave, t32 - 1)] : make_int4(a.Tk, 0, 0, a.Tk);
  const int wlo = __builtin_amdgcn_readfirstlane(mine.x), whi = __builtin_amdgcn_readfirstlane(mine.y);
  const int flo = __builtin_amdgcn_readfirstlane(mine.z), fhi = __builtin_amdgcn_readfirstlane(mine.w);
  // queries that can see a key at all: what q and dO hold for the others is not used
  int cbeg, cend, kbeg, kend;
  live_range(a, b, cbeg, cend, kbeg, kend);
  Source<E, DP, RB> ksrc, vsrc;
  ksrc.set((const E*)a.k + b * a.k_bs + (long long)kvh * a.dk * a.k_cs, a.k_cs, a.dk, a.Tk, tid);
  vsrc.set((const E*)a.v + b * a.v_bs + (long long)kvh * a.dk * a.v_cs, a.v_cs, a.dk, a.Tk, tid);
  Pre<E, DP, RB> kf, vf;
  const int first = blo / N * N;
  if (first < bhi) {
    ksrc.fetch(kf, first, tid);
    vsrc.fetch(vf, first, tid);
  }
  const float lse = some ? a.lse[bh * a.Tq + t] : 0.f, D = some ? ws.rowsum[bh * a.Tq + t] : 0.f;
  const float gs = operand_scale<E>(a, ws, b, kvh, red);
  const ScoreScale sc = score_scale(a);
  const float* table = a.bias ? a.bias + (a.bias_heads > 1 ? (long long)head * (2 * a.bias_w + 1) : 0) : nullptr;
  const int d0 = -(off + t0) - (NCOL - 1);
  unsigned long long draws = 0;
  unsigned thr = 0;
  float keep = 1.f;
  if (a.seed) {
    draws = draw_start(a) + ((unsigned long long)(bh * a.Tq + t) * (unsigned long long)((a.Tk + 3) >> 2) + 2 * h) * DRAW_STEP;
    thr = (unsigned)rintf(a.p_drop * 65536.f);
    keep = 65536.f / (65536.f - (float)thr);
  }
  f32x16 acc[DP / 32];
#pragma unroll
  for (int i = 0; i < DP / 32; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[i][r] = 0.f;

  // Bias gradient.  A 32 x 32 block's entries of one distance lie on a diagonal: register j of eight (neighbouring positions) and lane n belong to
  // distance j - n.  The eight are summed along their diagonals in registers by shifting lanes one step per register, downwards for the lanes n >= j
  // and upwards for the others (neither crosses into the other half of the wave: what would is zero); the two results, 32 and 7 distances, are added to
  // the half's own bins in LDS, 4 additions a block instead of 16 (LDS additions of every register held the kernel: fp16, window of 128 in 1501: 267 us for 96).  The
  // lanes of one addition never meet, nor do waves, so the order is fixed.  As the tiles advance by N keys, a wave's first N bins are complete after
  // each tile and leave; the last 32 stay.  Distances at or beyond +-bias_w share the table's end entries and are summed in registers.
  const int W = a.bias_w;
  float* const bin = bin_[wave][h];
  float* bins = a.dbias ? ws.bins + (bh * ((a.Tq + 31) / 32) + (t0 >> 5) + wave) * (2 * W + 1) : nullptr;
  float end_lo = 0.f, end_hi = 0.f;
  const int p31 = off + t0 + wave * 32 + 31;               // the wave's last query position: bin j of a tile at s0 is distance s0 - p31 + j
  const bool live = a.dbias && (t0 >> 5) + wave < (a.Tq + 31) / 32;
  int first_d = 0, base = 0;                               // distances of the first bin ever and of bin 0 now
  bool begun = false;
  if (a.dbias)
    for (int j = n; j < NB; j += 32) bin[j] = 0.f;

  float bf = 0.f;
  if (first < bhi && table && tid < NCOL + N) bf = bias_entry(table, W, first + d0, tid);
  typename Frag<E>::template Head<DP> q, g;
  qc.settle(q, tiles, t0, cbeg, cend, tid);
  gc.settle(g, tiles, t0, cbeg, cend, tid);
  int buf = 0;
  for (int s0 = first; s0 < bhi; s0 += N, buf = Staged<E, DP, RB>::BUFS == 2 ? buf ^ 1 : 0) {
    E* const ks = tiles + buf * 2 * Staged<E, DP, RB>::SIZE;
    E* const vs = ks + Staged<E, DP, RB>::SIZE;
    if (s0 == first || Staged<E, DP, RB>::BUFS == 1) __syncthreads();
    ksrc.commit(ks, kf, s0, blo, bhi, tid);
    vsrc.commit(vs, vf, s0, blo, bhi, tid);
    if (table && tid < NCOL + N) win[buf][tid] = bias_scaled(bf);
    __syncthreads();
    {                                                             // (behind the last tile: values that are not used)
      ksrc.fetch(kf, s0 + N, tid);
      vsrc.fetch(vf, s0 + N, tid);
      if (table) bf = bias_entry(table, W, s0 + N + d0, tid);
    }
    if (s0 >= whi || s0 + N <= wlo) continue;
#pragma unroll 1
    for (int rt = 0; rt < RT; ++rt) {
      const f32x16 u = mul_columns<E, DP, RB>(ks, rt, q, lane);
      float x[16], th[16];
      float mul = sc.mul;
#pragma unroll
      for (int r = 0; r < 16; ++r) x[r] = u[r];
      if (sc.cap) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          th[r] = cap_tanh<EXACT>(x[r], sc);
          x[r] = th[r] * sc.cap_out;
        }
        mul = 1.f;
      }
      if (table) {
        const float* w = win[buf] + 32 * rt + (NCOL - 1) - tl;
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] = fmaf(x[r], mul, w[pos_of(r, h)]);
        mul = 1.f;
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) x[r] = __builtin_amdgcn_exp2f(fmaf(x[r], mul, -lse));
      __builtin_amdgcn_sched_barrier(0);                            // one product's accumulator at a time
      f32x16 dp = mul_columns<E, DP, RB>(vs, rt, g, lane);
      if (a.seed) {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const unsigned long long z = draw_word(draws + draw_block(s0 + 32 * rt) + draw_group(w));
#pragma unroll
          for (int j = 0; j < 4; ++j) dp[4 * w + j] = dropped(z, j, thr) ? 0.f : dp[4 * w + j] * keep;
        }
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) x[r] *= dp[r] - D;
      if (s0 < flo || s0 + N > fhi) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const unsigned p = s0 + 32 * rt + pos_of(r, h) - iv.x;
          x[r] = p < (unsigned)(iv.y - iv.x) ? x[r] : 0.f;
        }
      }
      if (a.dbias) {
        const int d_lo = s0 + 32 * rt - p31, d_hi = d_lo + 62;      // the 32 x 32 block's distances
        if (d_hi <= -W) {
#pragma unroll
          for (int r = 0; r < 16; ++r) end_lo += x[r];
        } else if (d_lo >= W) {
#pragma unroll
          for (int r = 0; r < 16; ++r) end_hi += x[r];
        } else {
#pragma unroll
          for (int g8 = 0; g8 < 16; g8 += 8) {
            float dn = n >= 7 ? x[g8 + 7] : 0.f, up = n < 1 ? x[g8 + 1] : 0.f;
#pragma unroll
            for (int j = 6; j >= 0; --j) dn = lane_shift<0x130>(dn) + (n >= j ? x[g8 + j] : 0.f);
#pragma unroll
            for (int j = 2; j < 8; ++j) up = lane_shift<0x138>(up) + (n < j ? x[g8 + j] : 0.f);
            float* const at = &bin[32 * rt + pos_of(g8, h) - n + 31];
            __hip_atomic_fetch_add(at, dn, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WAVEFRONT);
            if (n < 7) __hip_atomic_fetch_add(at + 7, up, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WAVEFRONT);
          }
        }
      }
      if (sc.cap) {
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] *= fmaf(-th[r], th[r], 1.f);
      }
      if constexpr (__is_same(E, f16_t)) {
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] *= gs;
      }
      mul_rows<E, DP, 1, RB>(acc, ks, rt, x, lane);
    }
    if (live) {
      // N complete bins leave (N = 64: one a lane; N = 32: the lower half of the lanes), 32 stay
      if (!begun) first_d = s0 - p31;
      begun = true;
      base = s0 - p31 + N;
      if (s0 + N - 1 - p31 + 31 > -W && s0 - p31 < W) {     // (else the tile and what stayed are past the ends: nothing was added to bins that leave)
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        const float v = lane < N ? bin_[wave][0][lane] + bin_[wave][1][lane] : 0.f;
        const float stay = bin[N + n];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        for (int j = n; j < NB; j += 32) bin[j] = j < 32 ? stay : 0.f;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        const int d = s0 - p31 + lane;
        if (lane < N) {
          if (d <= -W) end_lo += v;
          else if (d >= W) end_hi += v;
          else bins[d + W] = v;
        }
      }
    }
  }
  if (live) {
    if (begun && lane < 32) {
      const float v = bin_[wave][0][lane] + bin_[wave][1][lane];
      const int d = base + lane;
      if (d <= -W) end_lo += v;
      else if (d >= W) end_hi += v;
      else bins[d + W] = v;
    }
    for (int e = 1 - W + lane; e < W; e += 64)
      if (!begun || e < first_d || e >= base + 32) bins[e + W] = 0.f;
    for (int o = 32; o > 0; o >>= 1) {
      end_lo += __shfl_xor(end_lo, o);
      end_hi += __shfl_xor(end_hi, o);
    }
    if (lane == 0) {
      bins[0] = W ? end_lo : end_lo + end_hi;
      if (W) bins[2 * W] = end_hi;
    }
  }
  if (t >= a.Tq) return;
  const float os = a.scale / gs;
  E* o = (E*)a.dq + bh * a.dk * a.Tq + t;
#pragma unroll
  for (int i = 0; i < DP / 32; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int d = 32 * i + 8 * (r >> 2) + 4 * h + (r & 3);
      if (d < a.dk) o[(long long)d * a.Tq] = (E)(acc[i][r] * os);
    }
}

template <typename E, int DP>
static void go(const svc_attn_scored_t& a, const Ws& w, hipStream_t s) {
  const int n_tiles = (a.Tq + NCOL - 1) / NCOL;
  const unsigned grid = (unsigned)grid_of((long long)a.B * a.G, a.H / a.G, n_tiles);
  if (sizeof(E) == 4 || a.dbias || a.softcap > SHORT_CAP) hipLaunchKernelGGL((dq_kernel<E, DP, true>), dim3(grid), dim3(256), 0, s, a, w, n_tiles);
  else hipLaunchKernelGGL((dq_kernel<E, DP, sizeof(E) == 4>), dim3(grid), dim3(256), 0, s, a, w, n_tiles);
}
template <typename E>
static void pick(const svc_attn_scored_t& a, const Ws& w, hipStream_t s) {
  if (a.dk <= 32) go<E, 32>(a, w, s);
  else if (a.dk <= 64) go<E, 64>(a, w, s);
  else if (a.dk <= 96 || X3<E>) go<E, 96>(a, w, s);
  else go<E, X3<E> ? 96 : 128>(a, w, s);
}
void launch_dq(const svc_attn_scored_t& a, const Ws& w, hipStream_t s) {
  // (three planes of q's and dO's columns at 128 channels do not fit the registers beside the accumulators)
  if (a.dtype == SVC_F32 && a.dk > 96) go<float, 128>(a, w, s);
  else if (a.dtype == SVC_F32) pick<x3_t>(a, w, s);
  else if (a.dtype == SVC_BF16) pick<bf16_t>(a, w, s);
  else pick<f16_t>(a, w, s);
}

}  // namespace attn
