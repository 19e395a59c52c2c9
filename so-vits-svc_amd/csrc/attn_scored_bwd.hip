// attn_scored_bwd.hip — svc_attn_scored_bwd: gradients of svc_attn_scored_fwd.  Two passes, each recomputing the scores it needs (a walk over
// keys for dq and the bias, a walk over queries for dk and dv): seven products instead of five, and in exchange no atomics on
// memory, so that results do not vary from run to run, and no copies of dq that a further launch would have to add up.
#include "attn_scored.h"

namespace attn {

// ---- workspace ------------------------------------------------------------------------------------------------------------------
struct Ws {
  float* rowsum;   // [B*H][Tq]  D = sum_d dO out
  int2* iv;        // [B][Tq]    visible keys
  int4* tiles;     // [B][ceil(Tq/32)]  {min lo, max hi, max lo, min hi} of 32 queries
  float* gmax;     // [B*H][ceil(Tq/64)]  max |dO|
  float* bins;     // [B*H][ceil(Tq/32)][2 bias_w + 1]  bias gradient of 32 queries
  long long bytes;
};
static Ws layout(const svc_attn_scored_t& a) {
  Ws w;
  long long o = 0;
  char* base = (char*)a.ws;
  auto take = [&](long long bytes) {
    char* p = base + o;
    o += (bytes + 15) / 16 * 16;
    return p;
  };
  const long long bh = (long long)a.B * a.H, t32 = (a.Tq + 31) / 32;
  w.rowsum = (float*)take(bh * a.Tq * 4);
  w.iv = (int2*)take((long long)a.B * a.Tq * 8);
  w.tiles = (int4*)take(a.B * t32 * 16);
  w.gmax = (float*)take(bh * ((a.Tq + 63) / 64) * 4);
  w.bins = (float*)take(a.dbias ? bh * t32 * (2LL * a.bias_w + 1) * 4 : 0);
  w.bytes = o;
  return w;
}

// ---- rows: D = sum_d dO[d,t] out[d,t], the largest |dO|, and the visible intervals.  64 queries of one head a workgroup ----------
template <typename E>
__global__ __launch_bounds__(256) void rows_kernel(svc_attn_scored_t a, Ws w, int n_tiles) {
  __shared__ float sum[4][64], big[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int bh = blockIdx.x / n_tiles, tile = blockIdx.x % n_tiles, t = tile * 64 + lane;
  const int b = bh / a.H, head = bh % a.H;
  const int len = item_length(a, b), off = item_offset(a, b);
  int2 iv = make_int2(0, 0);
  if (t < a.Tq && (!a.offsets || (off >= -a.Tq && off < a.Tk))) iv = visible(a, b, len, off + t);
  const bool some = iv.y > iv.x;
  float s = 0.f, g = 0.f;
  if (some) {                           // (what dO and out hold for queries without keys is not used)
    const E* dp = (const E*)a.dout + b * a.do_bs + (long long)head * a.dk * a.do_cs + t;
    const E* op = (const E*)a.out + b * a.o_bs + (long long)head * a.dk * a.o_cs + t;
    const float* fp = a.out32 ? a.out32 + (long long)bh * a.dk * a.Tq + t : nullptr;
    for (int d = wave; d < a.dk; d += 4) {
      const float v = to_f(dp[d * a.do_cs]);
      const float o = fp ? fp[(long long)d * a.Tq] : to_f(op[d * a.o_cs]);
      s = fmaf(v, o, s);
      g = fmaxf(g, fabsf(v));
    }
  }
  sum[wave][lane] = s;
  big[wave][lane] = g;
  __syncthreads();
  if (wave) return;
  s = (sum[0][lane] + sum[1][lane]) + (sum[2][lane] + sum[3][lane]);
  g = fmaxf(fmaxf(big[0][lane], big[1][lane]), fmaxf(big[2][lane], big[3][lane]));
  if (t < a.Tq) w.rowsum[(long long)bh * a.Tq + t] = s;
  for (int o = 32; o > 0; o >>= 1) g = fmaxf(g, __shfl_xor(g, o));
  if (lane == 0) w.gmax[(long long)bh * n_tiles + tile] = g;
  if (head) return;
  if (t < a.Tq) w.iv[(long long)b * a.Tq + t] = iv;
  int4 r = make_int4(some ? iv.x : a.Tk, iv.y, t < a.Tq ? (some ? iv.x : a.Tk) : 0, t < a.Tq ? iv.y : a.Tk);
  for (int o = 16; o > 0; o >>= 1) {
    r.x = min(r.x, __shfl_xor(r.x, o));
    r.y = max(r.y, __shfl_xor(r.y, o));
    r.z = max(r.z, __shfl_xor(r.z, o));
    r.w = min(r.w, __shfl_xor(r.w, o));
  }
  const int t32 = 2 * tile + (lane >> 5);
  if ((lane & 31) == 0 && t32 < (a.Tq + 31) / 32) w.tiles[(long long)b * ((a.Tq + 31) / 32) + t32] = r;
}

// fp16 operands: dS is multiplied by a power of two that brings the largest |dO| of the key head to [1, 2): gradients of any magnitude then
// sit in the middle of the type's range (a loss scale of 2^-12 would otherwise leave dS among its subnormals), and |dS| <= 2 P |dO| |v|
// dk stays below 65504 for |v| up to 250.  The factor is divided out of the fp32 accumulators.
template <typename E> __device__ __forceinline__ float operand_scale(const svc_attn_scored_t& a, const Ws& w, int b, int kvh, float* red) {
  if constexpr (!__is_same(E, f16_t)) return 1.f;
  const int n_tiles = (a.Tq + 63) / 64, rep = a.H / a.G, n = rep * n_tiles;
  const float* g = w.gmax + ((long long)b * a.H + (long long)kvh * rep) * n_tiles;
  float m = 0.f;
  for (int i = threadIdx.x; i < n; i += 256) m = fmaxf(m, g[i]);
  for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
  __syncthreads();
  m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  if (!(m > 0.f) || !(m < INFINITY)) return 1.f;
  int e;
  frexpf(m, &e);
  return ldexpf(1.f, 1 - e);
}

// ---- dq (and the bias): 128 queries of one head a workgroup, walking the key tiles -------------------------------------------------
template <typename E, int DP>
__global__ __launch_bounds__(256) void dq_kernel(svc_attn_scored_t a, Ws ws, int n_tiles) {
  constexpr int N = Tile<E>::N, RT = Tile<E>::RT, NB = N + 32;
  __shared__ __align__(16) char ks_[DP * PITCH], vs_[DP * PITCH];
  __shared__ float win[NCOL + N];
  __shared__ float bin_[4][2][NB];
  __shared__ int range[2][4];
  __shared__ float red[4];
  E* ks = (E*)ks_;
  E* vs = (E*)vs_;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5, n = lane & 31;
  const int bh = blockIdx.x / n_tiles, t0 = (blockIdx.x % n_tiles) * NCOL;
  const int b = bh / a.H, head = bh % a.H, kvh = head / (a.H / a.G);
  const E* kp = (const E*)a.k + b * a.k_bs + (long long)kvh * a.dk * a.k_cs;
  const E* vp = (const E*)a.v + b * a.v_bs + (long long)kvh * a.dk * a.v_cs;
  const E* qp = (const E*)a.q + b * a.q_bs + (long long)head * a.dk * a.q_cs;
  const E* gp = (const E*)a.dout + b * a.do_bs + (long long)head * a.dk * a.do_cs;

  const int tl = wave * 32 + n, t = t0 + tl;
  const int off = item_offset(a, b);
  const int2 iv = t < a.Tq ? ws.iv[(long long)b * a.Tq + t] : make_int2(0, 0);
  const bool some = iv.y > iv.x;
  const int wlo = wave_min(some ? iv.x : a.Tk), whi = wave_max(iv.y);
  const int flo = wave_max(t < a.Tq ? (some ? iv.x : a.Tk) : 0), fhi = wave_min(t < a.Tq ? iv.y : a.Tk);
  if (lane == 0) {
    range[0][wave] = wlo;
    range[1][wave] = whi;
  }
  const float gs = operand_scale<E>(a, ws, b, kvh, red);
  __syncthreads();
  const int blo = min(min(range[0][0], range[0][1]), min(range[0][2], range[0][3]));
  const int bhi = max(max(range[1][0], range[1][1]), max(range[1][2], range[1][3]));

  typename Frag<E>::template Head<DP> q, g;
  load_columns<E, DP>(q, qp, a.q_cs, a.dk, some ? t : -1, a.Tq, h);
  load_columns<E, DP>(g, gp, a.do_cs, a.dk, some ? t : -1, a.Tq, h);
  const float lse = some ? a.lse[(long long)bh * a.Tq + t] : 0.f, D = some ? ws.rowsum[(long long)bh * a.Tq + t] : 0.f;
  const ScoreScale sc = score_scale(a);
  const float* table = a.bias ? a.bias + (a.bias_heads > 1 ? (long long)head * (2 * a.bias_w + 1) : 0) : nullptr;
  unsigned long long draws = 0;
  unsigned thr = 0;
  float keep = 1.f;
  if (a.seed) {
    const unsigned long long row = ((unsigned long long)b * a.H + head) * a.Tq + t;
    draws = draw_start(a) + row * (unsigned long long)((a.Tk + 3) >> 2) * 0xD1B54A32D192ED03ull;
    thr = (unsigned)rintf(a.p_drop * 65536.f);
    keep = 65536.f / (65536.f - (float)thr);
  }
  f32x16 acc[DP / 32];
#pragma unroll
  for (int i = 0; i < DP / 32; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[i][r] = 0.f;

  // Bias gradient.  The tile's entries of one distance lie on a diagonal: lane n of half h adds register r to bin pos(r,h) - n + 31 of its
  // half's own row, so the lanes of one instruction never meet (a half has 32 different n) and neither do waves: LDS adds in a fixed order.
  // As the tiles advance by N keys, a wave's first N bins are complete after each tile and leave; the last 32 stay.  Distances at or
  // beyond +-bias_w share the table's end entries and are summed in registers.
  const int W = a.bias_w;
  float* const bin = bin_[wave][h];
  float* bins = a.dbias ? ws.bins + ((long long)bh * ((a.Tq + 31) / 32) + (t0 >> 5) + wave) * (2 * W + 1) : nullptr;
  float end_lo = 0.f, end_hi = 0.f;
  const int p31 = off + t0 + wave * 32 + 31;               // the wave's last query position: bin j of a tile at s0 is distance s0 - p31 + j
  const bool live = a.dbias && (t0 >> 5) + wave < (a.Tq + 31) / 32;
  int first = 0, base = 0;                                 // distances of the first bin ever and of bin 0 now
  bool begun = false;
  if (a.dbias)
    for (int j = n; j < NB; j += 32) bin[j] = 0.f;

  for (int s0 = blo / N * N; s0 < bhi; s0 += N) {
    __syncthreads();
    stage<E, DP>(ks, kp, a.k_cs, a.dk, s0, blo, bhi, tid);
    stage<E, DP>(vs, vp, a.v_cs, a.dk, s0, blo, bhi, tid);
    if (table) stage_bias(win, table, W, s0 - (off + t0) - (NCOL - 1), NCOL + N, tid);
    __syncthreads();
    const bool work = s0 < whi && s0 + N > wlo;
    if (work) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        f32x16 u, dp;
#pragma unroll
        for (int r = 0; r < 16; ++r) u[r] = dp[r] = 0.f;
        u = mul_columns<E, DP>(ks, rt, q, u, lane);
        dp = mul_columns<E, DP>(vs, rt, g, dp, lane);
        float x[16], th[16];
        if (sc.cap_in > 0.f) {
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            th[r] = tanhf(u[r] * sc.cap_in);
            x[r] = th[r] * sc.cap_out;
          }
        } else {
#pragma unroll
          for (int r = 0; r < 16; ++r) x[r] = u[r] * sc.mul;
        }
        if (table) {
          const float* w = win + 32 * rt + (NCOL - 1) - tl;
#pragma unroll
          for (int r = 0; r < 16; ++r) x[r] += w[pos_of(r, h)];
        }
        if (a.seed) {
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const unsigned long long z = draw_word(draws, (unsigned long long)((s0 + 32 * rt + pos_of(4 * w, h)) >> 2));
#pragma unroll
            for (int j = 0; j < 4; ++j) dp[4 * w + j] = ((unsigned)(z >> (16 * j)) & 0xffffu) < thr ? 0.f : dp[4 * w + j] * keep;
          }
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] = __builtin_amdgcn_exp2f(x[r] - lse) * (dp[r] - D);
        if (s0 < flo || s0 + N > fhi) {
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int p = s0 + 32 * rt + pos_of(r, h);
            x[r] = p >= iv.x && p < iv.y ? x[r] : 0.f;
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
            for (int r = 0; r < 16; ++r) __hip_atomic_fetch_add(&bin[32 * rt + pos_of(r, h) - n + 31], x[r], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WAVEFRONT);
          }
        }
        if (sc.cap_in > 0.f) {
#pragma unroll
          for (int r = 0; r < 16; ++r) x[r] *= 1.f - th[r] * th[r];
        }
        if constexpr (__is_same(E, f16_t)) {
#pragma unroll
          for (int r = 0; r < 16; ++r) x[r] *= gs;
        }
        mul_rows<E, DP>(acc, ks, rt, x, lane);
      }
    }
    if (live && work) {
      // N complete bins leave (N = 64: one a lane; N = 32: the lower half of the lanes), 32 stay
      if (!begun) first = s0 - p31;
      begun = true;
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
      base = s0 - p31 + N;
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
      if (!begun || e < first || e >= base + 32) bins[e + W] = 0.f;
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
  E* o = (E*)a.dq + (long long)bh * a.dk * a.Tq + t;
#pragma unroll
  for (int i = 0; i < DP / 32; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int d = 32 * i + 8 * (r >> 2) + 4 * h + (r & 3);
      if (d < a.dk) o[(long long)d * a.Tq] = (E)(acc[i][r] * os);
    }
}

// ---- dk, dv: 128 keys of one key head a workgroup, walking the query tiles of its query heads --------------------------------------
template <typename E, int DP>
__global__ __launch_bounds__(256) void dkv_kernel(svc_attn_scored_t a, Ws ws, int n_tiles) {
  constexpr int N = Tile<E>::N, RT = Tile<E>::RT;
  __shared__ __align__(16) char qs_[DP * PITCH], gs_[DP * PITCH];
  __shared__ float win[NCOL + N];
  __shared__ float lses[N], rows[N];
  __shared__ int2 ivs[N];
  __shared__ float red[4];
  E* qs = (E*)qs_;
  E* gs = (E*)gs_;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5, n = lane & 31;
  const int bg = blockIdx.x / n_tiles, c0 = (blockIdx.x % n_tiles) * NCOL;
  const int b = bg / a.G, kvh = bg % a.G, rep = a.H / a.G;
  const E* kp = (const E*)a.k + b * a.k_bs + (long long)kvh * a.dk * a.k_cs;
  const E* vp = (const E*)a.v + b * a.v_bs + (long long)kvh * a.dk * a.v_cs;
  const int sl = wave * 32 + n, s = c0 + sl;
  const int off = item_offset(a, b), len = item_length(a, b);
  const float g2 = operand_scale<E>(a, ws, b, kvh, red), pup = exp2f(PUP<E>), gm = g2 / pup;
  // queries that can see a key at all: what lies in the others' columns of q and dO is not used
  int tbeg = max(0, -max(off, -a.Tq)), tend = off < a.Tk ? max(0, min(a.Tq, len - max(off, -a.Tq))) : 0;
  int kbeg = 0, kend = len;
  if (a.n_docs) {
    const int* d = a.docs + (long long)b * (a.n_docs + 1);
    kbeg = max(0, d[0]);
    kend = max(0, min(len, d[a.n_docs]));
    tbeg = max(tbeg, kbeg - max(off, -a.Tq));
    tend = min(tend, kend - max(off, -a.Tq));
  }
  const bool ok = s >= kbeg && s < kend;
  typename Frag<E>::template Head<DP> k, v;
  load_columns<E, DP>(k, kp, a.k_cs, a.dk, ok ? s : -1, a.Tk, h);
  load_columns<E, DP>(v, vp, a.v_cs, a.dk, ok ? s : -1, a.Tk, h);
  const ScoreScale sc = score_scale(a);
  unsigned thr = 0;
  float keep = 1.f;
  unsigned long long start = 0;
  const unsigned long long ng = (unsigned long long)((a.Tk + 3) >> 2);
  if (a.seed) {
    start = draw_start(a);
    thr = (unsigned)rintf(a.p_drop * 65536.f);
    keep = 65536.f / (65536.f - (float)thr);
  }
  f32x16 ak[DP / 32], av[DP / 32];
#pragma unroll
  for (int i = 0; i < DP / 32; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) ak[i][r] = av[i][r] = 0.f;

  for (int hh = 0; hh < rep; ++hh) {
    const int head = kvh * rep + hh;
    const long long bh = (long long)b * a.H + head;
    const E* qp = (const E*)a.q + b * a.q_bs + (long long)head * a.dk * a.q_cs;
    const E* gp = (const E*)a.dout + b * a.do_bs + (long long)head * a.dk * a.do_cs;
    const float* table = a.bias ? a.bias + (a.bias_heads > 1 ? (long long)head * (2 * a.bias_w + 1) : 0) : nullptr;
    for (int t0 = 0; t0 < a.Tq; t0 += N) {
      // does any query of the tile see any key of the workgroup's, and does every one see all of them?
      int4 r = ws.tiles[(long long)b * ((a.Tq + 31) / 32) + (t0 >> 5)];
      if (RT == 2 && t0 + 32 < a.Tq) {
        const int4 r1 = ws.tiles[(long long)b * ((a.Tq + 31) / 32) + (t0 >> 5) + 1];
        r = make_int4(min(r.x, r1.x), max(r.y, r1.y), max(r.z, r1.z), min(r.w, r1.w));
      }
      if (r.x >= c0 + NCOL || r.y <= c0) continue;
      const bool whole = c0 >= r.z && c0 + NCOL <= r.w && t0 + N <= a.Tq;
      __syncthreads();
      stage<E, DP>(qs, qp, a.q_cs, a.dk, t0, tbeg, tend, tid);
      stage<E, DP>(gs, gp, a.do_cs, a.dk, t0, tbeg, tend, tid);
      if (tid < N) {
        const int t = t0 + tid;
        lses[tid] = t < a.Tq ? a.lse[bh * a.Tq + t] - PUP<E> : 0.f;
        rows[tid] = t < a.Tq && t >= tbeg && t < tend ? ws.rowsum[bh * a.Tq + t] : 0.f;
        ivs[tid] = t < a.Tq ? ws.iv[(long long)b * a.Tq + t] : make_int2(0, 0);
      }
      if (table) stage_bias(win, table, a.bias_w, c0 - (off + t0) - (N - 1), NCOL + N, tid);
      __syncthreads();
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        f32x16 u, dp;
#pragma unroll
        for (int r2 = 0; r2 < 16; ++r2) u[r2] = dp[r2] = 0.f;
        u = mul_columns<E, DP>(qs, rt, k, u, lane);
        dp = mul_columns<E, DP>(gs, rt, v, dp, lane);
        float x[16], th[16], p[16];
        if (sc.cap_in > 0.f) {
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            th[i] = tanhf(u[i] * sc.cap_in);
            x[i] = th[i] * sc.cap_out;
          }
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) x[i] = u[i] * sc.mul;
        }
        if (table) {
          const float* w = win + (N - 1) - 32 * rt + sl;
#pragma unroll
          for (int i = 0; i < 16; ++i) x[i] += w[-pos_of(i, h)];
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int tl = 32 * rt + pos_of(i, h);
          x[i] = __builtin_amdgcn_exp2f(x[i] - lses[tl]);
          if (!whole) {
            const int2 w = ivs[tl];
            x[i] = s >= w.x && s < w.y ? x[i] : 0.f;
          }
          p[i] = x[i];
          if (a.seed) {
            const unsigned long long z = draw_word(start, ((unsigned long long)bh * a.Tq + t0 + tl) * ng + (unsigned)(s >> 2));
            const bool drop = ((unsigned)(z >> (16 * (s & 3))) & 0xffffu) < thr;
            p[i] = drop ? 0.f : x[i] * keep;
            dp[i] = drop ? 0.f : dp[i] * keep;
          }
          const float g = x[i] * (dp[i] - rows[tl]);
          x[i] = whole || x[i] > 0.f ? g : 0.f;            // (a masked entry: 0 whatever dO.v is)
        }
        if (sc.cap_in > 0.f) {
#pragma unroll
          for (int i = 0; i < 16; ++i) x[i] *= 1.f - th[i] * th[i];
        }
        if constexpr (__is_same(E, f16_t)) {
#pragma unroll
          for (int i = 0; i < 16; ++i) x[i] *= gm;
        }
        mul_rows<E, DP>(av, gs, rt, p, lane);
        mul_rows<E, DP>(ak, qs, rt, x, lane);
      }
    }
  }
  if (s >= a.Tk) return;
  const float os = a.scale / g2;
  E* ok_ = (E*)a.dk_ + (long long)bg * a.dk * a.Tk + s;
  E* ov = (E*)a.dv + (long long)bg * a.dk * a.Tk + s;
#pragma unroll
  for (int i = 0; i < DP / 32; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int d = 32 * i + 8 * (r >> 2) + 4 * h + (r & 3);
      if (d < a.dk) {
        ok_[(long long)d * a.Tk] = (E)(ak[i][r] * os);
        ov[(long long)d * a.Tk] = (E)(av[i][r] / pup);
      }
    }
}

// ---- dbias[head or 0][j] = sum of the 32-query bins over items (and heads, for a shared table), in fixed order -----------------------
__global__ __launch_bounds__(256) void dbias_kernel(svc_attn_scored_t a, Ws ws) {
  __shared__ double sum[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int nb = 2 * a.bias_w + 1, j = blockIdx.x * 64 + lane, head = blockIdx.y, t32 = (a.Tq + 31) / 32;
  double s = 0.0;
  if (j < nb) {
    if (a.bias_heads > 1) {
      for (int b = 0; b < a.B; ++b)
        for (int i = wave; i < t32; i += 4) s += (double)ws.bins[(((long long)b * a.H + head) * t32 + i) * nb + j];
    } else {
      const long long n = (long long)a.B * a.H * t32;
      for (long long i = wave; i < n; i += 4) s += (double)ws.bins[i * nb + j];
    }
  }
  sum[wave][lane] = s;
  __syncthreads();
  if (wave == 0 && j < nb) a.dbias[(long long)head * nb + j] = (float)((sum[0][lane] + sum[1][lane]) + (sum[2][lane] + sum[3][lane]));
}

template <typename E, int DP>
static void launch_bwd(const svc_attn_scored_t& a, const Ws& w, hipStream_t s) {
  const int nq = (a.Tq + NCOL - 1) / NCOL, nk = (a.Tk + NCOL - 1) / NCOL;
  hipLaunchKernelGGL((dq_kernel<E, DP>), dim3((unsigned)(a.B * a.H * nq)), dim3(256), 0, s, a, w, nq);
  hipLaunchKernelGGL((dkv_kernel<E, DP>), dim3((unsigned)(a.B * a.G * nk)), dim3(256), 0, s, a, w, nk);
}
template <typename E>
static void run_bwd(const svc_attn_scored_t& a, const Ws& w, hipStream_t s) {
  const int n64 = (a.Tq + 63) / 64;
  hipLaunchKernelGGL((rows_kernel<E>), dim3((unsigned)(a.B * a.H * n64)), dim3(256), 0, s, a, w, n64);
  if (a.dk <= 32) launch_bwd<E, 32>(a, w, s);
  else if (a.dk <= 64) launch_bwd<E, 64>(a, w, s);
  else if (a.dk <= 96) launch_bwd<E, 96>(a, w, s);
  else launch_bwd<E, 128>(a, w, s);
  if (a.dbias) hipLaunchKernelGGL(dbias_kernel, dim3((2 * a.bias_w + 64) / 64, a.bias_heads), dim3(256), 0, s, a, w);
}

}  // namespace attn

extern "C" {

long long svc_attn_scored_ws_bytes(const svc_attn_scored_t* a, int backward) {
  if (!a || !backward) return 0;
  return attn::layout(*a).bytes;
}

int svc_attn_scored_bwd(const svc_attn_scored_t* a, void* stream) {
  const int rc = attn::check_args(a, true);
  if (rc != SVC_OK || a->B == 0 || a->Tk == 0) return rc;
  SVC_REQUIRE(a->Tq > 0, "attn_scored_bwd: no queries");
  hipStream_t s = (hipStream_t)stream;
  svc::ProfScope prof(s, "attn_scored_bwd", 14.0 * a->B * a->H * (double)a->Tq * a->Tk * a->dk, 0);
  const attn::Ws w = attn::layout(*a);
  if (a->dtype == SVC_F32) attn::run_bwd<float>(*a, w, s);
  else if (a->dtype == SVC_BF16) attn::run_bwd<attn::bf16_t>(*a, w, s);
  else attn::run_bwd<attn::f16_t>(*a, w, s);
  return svc::check_launch("svc_attn_scored_bwd");
}

}  // extern "C"
