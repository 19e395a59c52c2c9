// attn_scored_fwd.hip — svc_attn_scored_fwd: attention with capped scores, distance bias, document / prefix / window masks and
// counter-based dropout; one pass over the keys with a running maximum and sum per query.
//
// out[:, t] = sum_s exp2(x_ts - m_t) v_s / sum_s exp2(x_ts - m_t), x the score times log2(e), m the running maximum: two matrix products a key tile
// (4 dk operations a visible pair) with the softmax between them in the registers of the first one's accumulator.  At 64 and 128 channels the vector
// unit is the bound, not the matrix unit: 16 scores a lane cost 32 to 48 transcendental cycles and 8 to 30 ordinary instructions each (cap, bias, mask,
// draws), the products 512 to 1024 cycles for all; two waves a SIMD overlap the two.  128 queries a workgroup share every k and v tile through LDS; a
// tile's loads are in flight while the one before is worked on.  Measured (kernel traces of passes one behind the other): bf16, 128 channels, 4 x 16 heads,
// 4096 x 4096 causal with a cap 511 to 518 us = 531 to 538 TFLOP/s; 2049 x 2049 with a prefix 156 us, and 145 a call = 502 without the tracer; bf16, 64 channels,
// 9 documents in 4099 with bias and dropout 59 us; fp16, window of 128 in 1501 56 us; fp32, 96 channels, 16 ragged items of up to 790 with dropout 88 us.  The short
// walks of documents and windows wait a third of the waves' cycles.
#include "attn_scored.h"

namespace attn {

// A workgroup owns 128 queries of one head (32 a wave) and walks the key tiles that any of them sees.
template <typename E, int DP, int MODE>
__global__ __launch_bounds__(256, X3<E> && DP > 96 ? 1 : 2) void fwd_kernel(svc_attn_scored_t a, int n_tiles) {
  constexpr int N = Tile<E>::N, RT = Tile<E>::RT;
  // a maximum that grows by less than this (a factor 2^LAZY in P) leaves the accumulators as they are: P stays far from any type's range.  (Where P is rounded
  // once, the price is that a row's largest P, 1 against its own maximum, is rounded like the others: prompt of 2049 in bf16 2.3e-3 from 64 bits, of which 1.7e-3 is the
  // output's own rounding.)
  constexpr float LAZY = __is_same(E, f16_t) ? 4.f : 8.f;
  __shared__ __align__(16) char tiles_[2 * Staged<E, DP>::BUFS * Staged<E, DP>::SIZE * sizeof(E)];
  __shared__ float win[2][NCOL + N];
  __shared__ int range[2][4];
  E* const tiles = (E*)tiles_;                                    // [2 buffers][k, v][DP][P]
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5, n = lane & 31;
  const Place at = place_of(blockIdx.x, a.B * a.G, a.H / a.G, n_tiles);
  if (at.group >= a.B * a.G) return;
  const int b = at.group / a.G, kvh = at.group % a.G, head = kvh * (a.H / a.G) + at.sub, t0 = at.tile * NCOL;
  const long long bh = (long long)b * a.H + head;

  Columns<E, DP> qc;
  qc.fetch((const E*)a.q + b * a.q_bs + (long long)head * a.dk * a.q_cs, a.q_cs, a.dk, a.Tq, t0, tid);
  const int tl = wave * 32 + n, t = t0 + tl;
  const int len = item_length(a, b), off = item_offset(a, b);
  int2 iv = make_int2(0, 0);
  if (t < a.Tq && (!a.offsets || (off >= -a.Tq && off < a.Tk))) iv = visible(a, b, len, off + t);
  // the wave's and the workgroup's key range, and the range that every query of the wave sees whole
  const bool some = iv.y > iv.x;
  const int wlo = wave_min(some ? iv.x : a.Tk), whi = wave_max(iv.y);
  const int flo = wave_max(t < a.Tq ? (some ? iv.x : a.Tk) : 0), fhi = wave_min(t < a.Tq ? iv.y : a.Tk);
  if (lane == 0) {
    range[0][wave] = wlo;
    range[1][wave] = whi;
  }
  __syncthreads();
  const int blo = min(min(range[0][0], range[0][1]), min(range[0][2], range[0][3]));
  const int bhi = max(max(range[1][0], range[1][1]), max(range[1][2], range[1][3]));

  const ScoreScale sc = score_scale(a);
  const float* table = a.bias ? a.bias + (a.bias_heads > 1 ? (long long)head * (2 * a.bias_w + 1) : 0) : nullptr;
  const int d0 = -(off + t0) - (NCOL - 1);                        // distance of window entry 0 in a tile at key 0
  unsigned long long draws = 0;
  unsigned thr = 0;
  if (a.seed) {
    draws = draw_start(a) + ((unsigned long long)(bh * a.Tq + t) * (unsigned long long)((a.Tk + 3) >> 2) + 2 * h) * DRAW_STEP;
    thr = (unsigned)rintf(a.p_drop * 65536.f);
  }
  f32x16 acc[DP / 32];
#pragma unroll
  for (int i = 0; i < DP / 32; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[i][r] = 0.f;
  float m = -INFINITY, l = 0.f;

  Source<E, DP> ksrc, vsrc;
  ksrc.set((const E*)a.k + b * a.k_bs + (long long)kvh * a.dk * a.k_cs, a.k_cs, a.dk, a.Tk, tid);
  vsrc.set((const E*)a.v + b * a.v_bs + (long long)kvh * a.dk * a.v_cs, a.v_cs, a.dk, a.Tk, tid);
  Pre<E, DP> kf, vf;
  float bf = 0.f;
  const int first = blo / N * N;
  if (first < bhi) {
    ksrc.fetch(kf, first, tid);
    vsrc.fetch(vf, first, tid);
    if (table && tid < NCOL + N) bf = bias_entry(table, a.bias_w, first + d0, tid);
  }
  typename Frag<E>::template Head<DP> q;
  qc.settle(q, tiles, t0, 0, a.Tq, tid);
  int buf = 0;
  for (int s0 = first; s0 < bhi; s0 += N, buf = Staged<E, DP>::BUFS == 2 ? buf ^ 1 : 0) {
    E* const ks = tiles + buf * 2 * Staged<E, DP>::SIZE;
    E* const vs = ks + Staged<E, DP>::SIZE;
    if (s0 == first || Staged<E, DP>::BUFS == 1) __syncthreads();                             // (q's columns have been read from the tiles)
    ksrc.commit(ks, kf, s0, blo, bhi, tid);
    vsrc.commit(vs, vf, s0, blo, bhi, tid);
    if (table && tid < NCOL + N) win[buf][tid] = bias_scaled(bf);
    __syncthreads();
    {                                                             // (behind the last tile: values that are not used)
      ksrc.fetch(kf, s0 + N, tid);
      vsrc.fetch(vf, s0 + N, tid);
      if (table) bf = bias_entry(table, a.bias_w, s0 + N + d0, tid);
    }
    if (s0 >= whi || s0 + N <= wlo) continue;
    float s[RT][16];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const f32x16 u = mul_columns<E, DP>(ks, rt, q, lane);
#pragma unroll
      for (int r = 0; r < 16; ++r) s[rt][r] = u[r];
    }
    float mul = sc.mul;
    if (sc.cap) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[rt][r] = capped<MODE == 2>(s[rt][r], sc);
      mul = 1.f;
    }
    if (table) {
      const float* w = win[buf] + (NCOL - 1) - tl;
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[rt][r] = fmaf(s[rt][r], mul, w[32 * rt + pos_of(r, h)]);
      mul = 1.f;
    }
    if (s0 < flo || s0 + N > fhi) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const unsigned p = s0 + 32 * rt + pos_of(r, h) - iv.x;
          s[rt][r] = p < (unsigned)(iv.y - iv.x) ? s[rt][r] : -INFINITY;
        }
    }
    float mt = -INFINITY;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int r = 0; r < 16; r += 2) mt = fmaxf(fmaxf(s[rt][r], s[rt][r + 1]), mt);
    mt = fmaxf(mt, __shfl_xor(mt, 32)) * mul;
    if (__any(mt > m + LAZY)) {
      const float m1 = fmaxf(m, mt), alpha = __builtin_amdgcn_exp2f(m1 == -INFINITY ? 0.f : m - m1);
      m = m1;
      l *= alpha;
#pragma unroll
      for (int i = 0; i < DP / 32; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][r] *= alpha;
    }
    const float ms = m == -INFINITY ? 0.f : m - PUP<E>;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float ls = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[rt][r] = __builtin_amdgcn_exp2f(fmaf(s[rt][r], mul, -ms));
        ls += s[rt][r];
      }
      l += ls;
      if (a.seed) {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const unsigned long long z = draw_word(draws + draw_block(s0 + 32 * rt) + draw_group(w));
#pragma unroll
          for (int j = 0; j < 4; ++j) s[rt][4 * w + j] = dropped(z, j, thr) ? 0.f : s[rt][4 * w + j];
        }
      }
      mul_rows<E, DP, P_OPS<E, MODE>>(acc, vs, rt, s[rt], lane);
    }
  }

  l += __shfl_xor(l, 32);
  if (t >= a.Tq) return;
  float inv = l > 0.f ? 1.f / l : 0.f;
  if (l != l) inv = l;                                  // nan scores give nan, as they would in any softmax
  if (a.seed) inv *= 65536.f / (65536.f - (float)thr);
  if (a.lse && h == 0) a.lse[bh * a.Tq + t] = l > 0.f || l != l ? m - PUP<E> + __builtin_amdgcn_logf(l) : 0.f;
  E* op = (E*)a.out + b * a.o_bs + (long long)head * a.dk * a.o_cs + t;
  float* fp = a.out32 ? a.out32 + bh * a.dk * a.Tq + t : nullptr;
#pragma unroll
  for (int i = 0; i < DP / 32; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int d = 32 * i + 8 * (r >> 2) + 4 * h + (r & 3);
      if (d < a.dk) {
        const float v = acc[i][r] * inv;
        op[d * a.o_cs] = (E)v;
        if (fp) fp[(long long)d * a.Tq] = v;
      }
    }
}

// What the sizes alone decide: the workspace's queries ask this too, before anything is divided or multiplied.
int check_sizes(const svc_attn_scored_t* a) {
  SVC_REQUIRE(a, "attn_scored: no arguments");
  SVC_REQUIRE(a->dtype >= 0 && a->dtype <= 2, "attn_scored: dtype %d", a->dtype);
  SVC_REQUIRE(a->B >= 0 && a->Tq >= 0 && a->Tq <= a->Tk && a->Tk < (1 << 30), "attn_scored: B=%d Tq=%d Tk=%d (0 <= Tq <= Tk < 2^30)",
              a->B, a->Tq, a->Tk);
  SVC_REQUIRE(a->G >= 1 && a->H >= a->G && a->H % a->G == 0, "attn_scored: %d query heads, %d key heads", a->H, a->G);
  SVC_REQUIRE(a->dk >= 1 && a->dk <= 128, "attn_scored: head size %d (1..128)", a->dk);
  SVC_REQUIRE(!a->bias || (a->bias_w >= 0 && a->bias_w < (1 << 24) && a->H < 65536 && (a->bias_heads == 1 || a->bias_heads == a->H)),
              "attn_scored: bias of %d heads, width %d", a->bias_heads, a->bias_w);
  // (a launch has fewer than 2^32 threads: the widest has three workgroups of 256 for 128 keys of a head; the product of any three ints fits a double's range)
  const double groups = (double)a->B * a->H * svc::cdiv(a->Tk, 128);
  SVC_REQUIRE(a->Tq == 0 || groups < 5. * (1 << 20), "attn_scored: %.0f tiles of 128 keys (up to 5 2^20)", groups);
  return SVC_OK;
}
int check_args(const svc_attn_scored_t* a, bool backward) {
  if (const int rc = check_sizes(a)) return rc;
  SVC_REQUIRE(a->offsets || (a->offset >= 0 && a->offset <= a->Tk - a->Tq), "attn_scored: offset %d with Tq=%d Tk=%d", a->offset, a->Tq, a->Tk);
  SVC_REQUIRE(a->window >= -1 && a->n_docs >= 0 && (a->n_docs == 0 || a->docs), "attn_scored: window %d, %d documents", a->window, a->n_docs);
  SVC_REQUIRE(!a->prefix || (a->causal && a->window < 0), "attn_scored: a prefix goes with a causal mask and no window");
  SVC_REQUIRE(a->scale > 0.f && a->scale < INFINITY && a->softcap >= 0.f && a->softcap < INFINITY, "attn_scored: scale %g, softcap %g", a->scale, a->softcap);
  // (the kernels' factors: score_scale)
  SVC_REQUIRE(a->scale * LOG2E < INFINITY && a->softcap * LOG2E < INFINITY && (a->softcap == 0.f || a->scale / a->softcap * (2.f * LOG2E) < INFINITY),
              "attn_scored: scale %g with softcap %g: beyond fp32", a->scale, a->softcap);
  SVC_REQUIRE(!a->seed || (a->p_drop >= 0.f && a->p_drop <= 0.99f), "attn_scored: dropout rate %g (0..0.99)", a->p_drop);
  if (a->B == 0 || a->Tq == 0) return SVC_OK;
  SVC_REQUIRE(a->q && a->k && a->v, "attn_scored: q, k, v");
  if (!backward) SVC_REQUIRE(a->out, "attn_scored: out");
  if (backward) {
    SVC_REQUIRE(a->dout && a->lse && a->dq && a->dk_ && a->dv && (a->dtype == SVC_F32 ? a->out != nullptr : a->out32 != nullptr),
                "attn_scored_bwd: dout, lse, %s, dq, dk, dv", a->dtype == SVC_F32 ? "out" : "out32");
    SVC_REQUIRE(!a->dbias || a->bias, "attn_scored_bwd: dbias without bias");
  }
  const long long need = svc_attn_scored_ws_bytes(a, backward);
  SVC_REQUIRE(need == 0 || (a->ws && a->ws_bytes >= need && ((size_t)a->ws & 15) == 0), "attn_scored: workspace of %lld bytes needed, %lld given",
              need, a->ws ? a->ws_bytes : 0LL);
  return SVC_OK;
}

template <typename E, int DP>
static void launch_fwd(const svc_attn_scored_t& a, hipStream_t s) {
  const int n_tiles = (a.Tq + NCOL - 1) / NCOL;
  const unsigned grid = (unsigned)grid_of((long long)a.B * a.G, a.H / a.G, n_tiles);
  constexpr bool F = sizeof(E) == 4;
  if (F || a.exact || a.softcap > SHORT_CAP) hipLaunchKernelGGL((fwd_kernel<E, DP, 2>), dim3(grid), dim3(256), 0, s, a, n_tiles);
  else if (a.out32) hipLaunchKernelGGL((fwd_kernel<E, DP, F ? 2 : 1>), dim3(grid), dim3(256), 0, s, a, n_tiles);
  else hipLaunchKernelGGL((fwd_kernel<E, DP, F ? 2 : 0>), dim3(grid), dim3(256), 0, s, a, n_tiles);
}
template <typename E>
static void pick_fwd(const svc_attn_scored_t& a, hipStream_t s) {
  if (a.dk <= 32) launch_fwd<E, 32>(a, s);
  else if (a.dk <= 64) launch_fwd<E, 64>(a, s);
  else if (a.dk <= 96) launch_fwd<E, 96>(a, s);
  else launch_fwd<E, 128>(a, s);
}

}  // namespace attn

extern "C" {

int svc_attn_scored_fwd(const svc_attn_scored_t* a, void* stream) {
  const int rc = attn::check_args(a, false);
  if (rc != SVC_OK || a->B == 0 || a->Tq == 0) return rc;
  hipStream_t s = (hipStream_t)stream;
  svc::ProfScope prof(s, "attn_scored_fwd", 4.0 * a->B * a->H * (double)a->Tq * a->Tk * a->dk, 0);
  const attn::Split p = attn::split_of(*a);
  if (p.parts) attn::launch_split(*a, p, s);
  else if (a->dtype == SVC_F32) attn::pick_fwd<attn::x3_t>(*a, s);
  else if (a->dtype == SVC_BF16) attn::pick_fwd<attn::bf16_t>(*a, s);
  else attn::pick_fwd<attn::f16_t>(*a, s);
  return svc::check_launch("svc_attn_scored_fwd");
}

}  // extern "C"
