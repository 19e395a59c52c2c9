// dropout_add_layernorm.hip — the residual junction of a transformer layer: y = LayerNorm_C(r + dropout(x)) * gamma + beta (* mask), forward and
// backward, on [B, C, T] with time contiguous (modules/attentions.py:51-55,100-104, modules/modules.py:23-35).
//
// The backward keeps nothing but mean and rstd: h = r + dropout(x) is recomputed from x, r and the counter draws, which moves the same bytes as
// storing h would (one write and one read against two reads in place of one) and takes no memory.
//
// Measured, 32 x 768 x 1499 bf16 with dropout: forward 91 to 95 us (221 MB, 2.3 TB/s), backward 181 to 190 us (368 MB, 2.0 TB/s).  Vector instructions take 65 % of the
// forward's cycles (the draws: two 64-bit multiplications an element, 6 quarter-rate instructions of about 40) and 37 % of the backward's; the rest are waits, because a
// tile's loads, sums and stores stand one behind the other in each workgroup.  16 x 192 x 790 fp32: 14 and 19 us, a tile's
// own length; 8 x 1001 x 2047 fp16 without dropout: 44 and 69 us (98 and 131 MB).
#include "common.h"

namespace {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

// svc_dropout_rng_f32's keep decision (splitmix64's finaliser over a counter; the top 24 bits as a number in [0, 1) against p) on integers: the
// last xor-shift leaves the top 31 bits as they are, and k 2^-24 >= p is k >= ceil(2^24 p), both exactly.
__device__ __forceinline__ bool draw_keep(unsigned long long z, unsigned cut) {
  z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
  z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
  return (unsigned)(z >> 40) >= cut;
}

constexpr unsigned long long STEP = 0xD1B54A32D192ED03ull;
constexpr int THR = 512;
constexpr int V = 4;                   // time steps of a thread: one 16-byte (fp32) or 8-byte (16-bit) access, at any alignment of the type

template <typename E> struct Vec {
  struct __attribute__((packed, aligned(sizeof(E)))) M { E e[V]; };
};
// V values from element `at` of an item's slab, a 32-bit offset from a uniform base (one offset register serves all tensors of a row).  FULL: all V lie
// inside the row; else the first `left` do, and the nearest inside stand for the others (never used).  Loads carry no branch, so that all of a
// thread's loads can be in flight together.
template <typename E, bool FULL>
__device__ __forceinline__ typename Vec<E>::M loadm(const E* base, unsigned at, int left) {
  if (FULL) return *(const typename Vec<E>::M*)((const char*)base + (size_t)(at * (unsigned)sizeof(E)));
  typename Vec<E>::M m;
#pragma unroll
  for (int e = 0; e < V; ++e) m.e[e] = base[at + min(e, left - 1)];
  return m;
}
template <typename E, bool FULL>
__device__ __forceinline__ void load4(float (&v)[V], const E* base, unsigned at, int left) {
  const typename Vec<E>::M m = loadm<E, FULL>(base, at, left);
#pragma unroll
  for (int e = 0; e < V; ++e) v[e] = (float)m.e[e];
}
template <typename E, bool FULL>
__device__ __forceinline__ void store4(E* base, const float (&v)[V], unsigned at, int left) {
  if (FULL) {
    typename Vec<E>::M m;
#pragma unroll
    for (int e = 0; e < V; ++e) m.e[e] = (E)v[e];
    *(typename Vec<E>::M*)((char*)base + (size_t)(at * (unsigned)sizeof(E))) = m;
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (e < left) base[at + e] = (E)v[e];
  }
}

// lane exchanges inside 4 neighbouring lanes without LDS: xor 1, xor 2
template <int CTRL> __device__ __forceinline__ float dpp(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
template <int LPR> __device__ __forceinline__ float row_sum(float v) {      // over the LPR lanes of a row
  v += dpp<0xB1>(v);
  if (LPR > 2) v += dpp<0x4E>(v);
  return v;
}

// A column's sum over all channels: over the wave's lanes of the same column group, then over the waves through LDS, in the same order for every thread.
template <int LPR>
__device__ __forceinline__ void column_sum(float (&s)[V], float (*sh)[LPR * V], int lane, int wave) {
#pragma unroll
  for (int o = LPR; o < 64; o <<= 1)
#pragma unroll
    for (int e = 0; e < V; ++e) s[e] += __shfl_xor(s[e], o);
  __syncthreads();                       // the previous use of sh is over
  if (lane < LPR)
#pragma unroll
    for (int e = 0; e < V; ++e) sh[wave][lane * V + e] = s[e];
  __syncthreads();
#pragma unroll
  for (int e = 0; e < V; ++e) s[e] = 0.f;
#pragma unroll 2
  for (int w = 0; w < THR / 64; ++w)
#pragma unroll
    for (int e = 0; e < V; ++e) s[e] += sh[w][(lane & (LPR - 1)) * V + e];
}

struct Site {
  bool drop;
  unsigned long long start;
  unsigned cut;
  float ks;
};
__device__ __forceinline__ Site site(const svc_dropout_add_layernorm_t& a) {
  Site c;
  c.drop = a.seed != nullptr;
  c.start = c.drop ? (unsigned long long)a.seed[0] + (unsigned long long)((unsigned)a.site + 1u) * 0x9E3779B97F4A7C15ull : 0;
  c.cut = (unsigned)ceilf(a.p * 16777216.f);
  c.ks = 1.f / (1.f - a.p);
  return c;
}

// x -> x's dropped value for V neighbouring elements, the first with counter value z; -> the kept ones' bits
__device__ __forceinline__ unsigned drop4(float (&x)[V], unsigned long long z, const Site& c) {
  unsigned bits = 0;
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const bool keep = draw_keep(z + e * STEP, c.cut);
    x[e] = keep ? x[e] * c.ks : 0.f;
    bits |= keep ? 1u << e : 0u;
  }
  return bits;
}

// The tile of a workgroup: LPR * V time steps of one item, all channels; a thread holds V steps of NR channels in registers, so every tensor is read
// once.  Neighbouring tiles share the cache lines at their borders (rows start anywhere), so tiles go to the XCDs in contiguous runs: XCD x = id % 8
// takes tiles x * n / 8 onwards.
__device__ __forceinline__ long long tile_of(long long id, long long n) {
  const long long per = n >> 3;
  return id < per * 8 ? (id & 7) * per + (id >> 3) : id;
}

template <typename E, int LPR, int NR, bool FULL>
__device__ __forceinline__ void fwd_tile(const svc_dropout_add_layernorm_t& a, int b, int t, float (*sh)[LPR * V]) {
  constexpr int RG = THR / LPR;          // channels in flight
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c0 = tid / LPR;
  const Site st = site(a);
  const long long o = (long long)b * a.C * a.T;
  const E *x = (const E*)a.x + o, *r = (const E*)a.r + o;
  const int left = a.T - t, tc = FULL ? t : min(t, a.T - 1), lc = FULL ? V : max(left, 1);
  unsigned at[NR];
#pragma unroll
  for (int i = 0; i < NR; ++i) at[i] = (unsigned)min(c0 + i * RG, a.C - 1) * (unsigned)a.T + tc;
  const unsigned long long z0 = st.start + (unsigned long long)(o + (long long)c0 * a.T + t) * STEP, dz = (unsigned long long)RG * a.T * STEP;
  float h[NR][V], s[V] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < NR; ++i) load4<E, FULL>(h[i], x, at[i], lc);
  if (st.drop) {
#pragma unroll
    for (int i = 0; i < NR; ++i) drop4(h[i], z0 + i * dz, st);
  }
  if (a.r) {
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      float v[V];
      load4<E, FULL>(v, r, at[i], lc);
#pragma unroll
      for (int e = 0; e < V; ++e) h[i][e] += v[e];
    }
  }
#pragma unroll
  for (int i = 0; i < NR; ++i)
#pragma unroll
    for (int e = 0; e < V; ++e) s[e] += c0 + i * RG < a.C ? h[i][e] : 0.f;
  column_sum<LPR>(s, sh, lane, wave);
  float mu[V], rs[V], m[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    mu[e] = s[e] / a.C;
    s[e] = 0.f;
  }
#pragma unroll
  for (int i = 0; i < NR; ++i)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float d = c0 + i * RG < a.C ? h[i][e] - mu[e] : 0.f;
      s[e] = fmaf(d, d, s[e]);
    }
  column_sum<LPR>(s, sh, lane, wave);
#pragma unroll
  for (int e = 0; e < V; ++e) {
    rs[e] = 1.f / sqrtf(s[e] / a.C + a.eps);
    m[e] = 1.f;
  }
  if (a.mask) load4<float, FULL>(m, a.mask + (long long)b * a.T, tc, lc);
  if (c0 == 0 && a.mean) {
    store4<float, FULL>(a.mean + (long long)b * a.T, mu, tc, left);
    store4<float, FULL>(a.rstd + (long long)b * a.T, rs, tc, left);
  }
  E* y = (E*)a.y + o;
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    const int c = c0 + i * RG;
    if (c >= a.C) break;
    const float g = a.gamma[c], be = a.beta[c];
    float v[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float u = fmaf((h[i][e] - mu[e]) * rs[e], g, be);
      v[e] = m[e] != 0.f ? u * m[e] : 0.f;
    }
    store4<E, FULL>(y, v, at[i], left);
  }
}

template <typename E, int LPR, int NR>
__global__ __launch_bounds__(THR, 4) void junction_fwd_kernel(svc_dropout_add_layernorm_t a, int tiles_t, long long n_tiles) {
  __shared__ float sh[THR / 64][LPR * V];
  const long long tile = tile_of(blockIdx.x, n_tiles);
  const int b = (int)(tile / tiles_t), t0 = (int)(tile % tiles_t) * LPR * V, t = t0 + (threadIdx.x & (LPR - 1)) * V;
  if (t0 + LPR * V <= a.T) fwd_tile<E, LPR, NR, true>(a, b, t, sh);
  else fwd_tile<E, LPR, NR, false>(a, b, t, sh);
}

// Backward.  Between the columns' sums and the results a thread keeps x^ and dy as it was loaded.  The parameters' sums stay in LDS over all tiles of a
// workgroup (a channel belongs to one group of LPR lanes, so it is an ordinary read and write) and leave once, part[workgroup][2][C].
template <typename E, int LPR, int NR, bool FULL>
__device__ __forceinline__ void bwd_tile(const svc_dropout_add_layernorm_t& a, int b, int t, float (*sh)[LPR * V], float* sums) {
  constexpr int RG = THR / LPR;
  typedef typename Vec<E>::M M;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c0 = tid / LPR;
  const Site st = site(a);
  const long long o = (long long)b * a.C * a.T;
  const E *x = (const E*)a.x + o, *r = (const E*)a.r + o, *dy = (const E*)a.dy + o;
  const int left = a.T - t, tc = FULL ? t : min(t, a.T - 1), lc = FULL ? V : max(left, 1);
  unsigned at[NR];
  M xr[NR], gr[NR], rr[NR];
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    at[i] = (unsigned)min(c0 + i * RG, a.C - 1) * (unsigned)a.T + tc;
    xr[i] = loadm<E, FULL>(x, at[i], lc);
    gr[i] = loadm<E, FULL>(dy, at[i], lc);
    if (!FULL) __builtin_amdgcn_sched_barrier(0);
  }
  if (a.r) {
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      rr[i] = loadm<E, FULL>(r, at[i], lc);
      if (!FULL) __builtin_amdgcn_sched_barrier(0);
    }
  } else {
#pragma unroll
    for (int i = 0; i < NR; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) rr[i].e[e] = (E)0.f;
  }
  float mu[V], rs[V], m[V], s1[V] = {0.f, 0.f, 0.f, 0.f}, s2[V] = {0.f, 0.f, 0.f, 0.f};
  load4<float, FULL>(mu, a.mean + (long long)b * a.T, tc, lc);
  load4<float, FULL>(rs, a.rstd + (long long)b * a.T, tc, lc);
#pragma unroll
  for (int e = 0; e < V; ++e) m[e] = 1.f;
  if (a.mask) load4<float, FULL>(m, a.mask + (long long)b * a.T, tc, lc);
  if (!FULL)
#pragma unroll
    for (int e = 0; e < V; ++e) m[e] = e < left ? m[e] : 0.f;
  float xh[NR][V];
  unsigned bits = 0;                     // NR * V <= 32
  unsigned long long z = st.start + (unsigned long long)(o + (long long)c0 * a.T + t) * STEP;
  const unsigned long long dz = (unsigned long long)RG * a.T * STEP;
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    __builtin_amdgcn_sched_barrier(0);   // a row at a time: interleaved rows would need the registers of a second workgroup
    const int c = c0 + i * RG;
    const bool in = c < a.C;
    const float ga = a.gamma[min(c, a.C - 1)];
#pragma unroll
    for (int e = 0; e < V; ++e) xh[i][e] = (float)xr[i].e[e];
    if (st.drop) bits |= drop4(xh[i], z, st) << (i * V);
    z += dz;
    float pg = 0.f, pb = 0.f;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const bool on = in && m[e] != 0.f;
      const float g0 = on ? (float)gr[i].e[e] * m[e] : 0.f, g = g0 * ga;
      xh[i][e] = on ? (xh[i][e] + (float)rr[i].e[e] - mu[e]) * rs[e] : 0.f;
      pg = fmaf(g0, xh[i][e], pg);
      pb += g0;
      s1[e] += g;
      s2[e] = fmaf(g, xh[i][e], s2[e]);
    }
    pg = row_sum<LPR>(pg);
    pb = row_sum<LPR>(pb);
    if (in && (tid & (LPR - 1)) == 0) {
      sums[c] += pg;
      sums[RG * NR + c] += pb;
    }
  }
  // dy is unpacked and multiplied again below: without this the compiler would keep the products, twice the registers
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    union { M m; unsigned u[sizeof(M) / 4]; } k;
    k.m = gr[i];
#pragma unroll
    for (unsigned& u : k.u) asm volatile("" : "+v"(u));
    gr[i] = k.m;
  }
  __builtin_amdgcn_sched_barrier(0);
  column_sum<LPR>(s1, sh, lane, wave);
  column_sum<LPR>(s2, sh, lane, wave);
#pragma unroll
  for (int e = 0; e < V; ++e) {
    s1[e] /= a.C;
    s2[e] /= a.C;
  }
  E *dr = (E*)a.dr + o, *dx = (E*)a.dx + o;
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    const int c = c0 + i * RG;
    if (c >= a.C) break;
    const float ga = a.gamma[c];
    float d[V];
#pragma unroll
    for (int e = 0; e < V; ++e) d[e] = m[e] != 0.f ? rs[e] * ((float)gr[i].e[e] * m[e] * ga - s1[e] - xh[i][e] * s2[e]) : 0.f;
    if (a.dr) store4<E, FULL>(dr, d, at[i], left);
    if (a.dx) {
#pragma unroll
      for (int e = 0; e < V; ++e) d[e] = !st.drop ? d[e] : bits >> (i * V + e) & 1 ? d[e] * st.ks : 0.f;
      store4<E, FULL>(dx, d, at[i], left);
    }
  }
}

template <typename E, int LPR, int NR>
__global__ __launch_bounds__(THR, NR > 4 ? 2 : 4) void junction_bwd_kernel(svc_dropout_add_layernorm_t a, int tiles_t, long long n_tiles, float* part) {
  constexpr int CH = THR / LPR * NR;
  __shared__ float sh[THR / 64][LPR * V];
  __shared__ float sums[2 * CH];
  for (int i = threadIdx.x; i < 2 * CH; i += THR) sums[i] = 0.f;
  __syncthreads();
  // XCD x takes the tiles from x * n / 8 on, its workgroups side by side: neighbours in time share cache lines only while they are worked on together
  // (each workgroup with a run of its own: 534 MB fetched and 282 written for 221 and 147, 768 x 1499 x 32 in bf16)
  const long long id = blockIdx.x, xs = gridDim.x % 8 == 0 ? 8 : 1, x = id % xs, lo = n_tiles * x / xs, hi = n_tiles * (x + 1) / xs;
  for (long long tile = lo + id / xs; tile < hi; tile += gridDim.x / xs) {
    const int b = (int)(tile / tiles_t), t0 = (int)(tile % tiles_t) * LPR * V, t = t0 + (threadIdx.x & (LPR - 1)) * V;
    if (t0 + LPR * V <= a.T) bwd_tile<E, LPR, NR, true>(a, b, t, sh, sums);
    else bwd_tile<E, LPR, NR, false>(a, b, t, sh, sums);
  }
  __syncthreads();
  for (int c = threadIdx.x; c < a.C; c += THR) {
    part[2LL * id * a.C + c] = sums[c];
    part[(2LL * id + 1) * a.C + c] = sums[CH + c];
  }
}

// ---- more channels than a workgroup's registers hold: each pass over the channels reads the tensors again (64 steps x 8 channel groups) --------------
constexpr int TX = 64, TY = 8;
__device__ __forceinline__ float wide_sum(float v, float (*sh)[TX], int tx, int ty) {
  __syncthreads();
  sh[ty][tx] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < TY; ++i) s += sh[i][tx];
  return s;
}
template <typename E>
__device__ __forceinline__ float junction1(const E* x, const E* r, long long i, const Site& c, float& k) {
  k = !c.drop ? 1.f : draw_keep(c.start + (unsigned long long)i * STEP, c.cut) ? c.ks : 0.f;
  const float v = k != 0.f ? (float)x[i] * k : 0.f;
  return r ? (float)r[i] + v : v;
}
template <typename E>
__global__ __launch_bounds__(THR) void junction_wide_fwd_kernel(svc_dropout_add_layernorm_t a, int tiles_t) {
  __shared__ float sh[TY][TX];
  const int tx = threadIdx.x & (TX - 1), ty = threadIdx.x / TX, t = (int)(blockIdx.x % tiles_t) * TX + tx, b = blockIdx.x / tiles_t;
  const bool ok = t < a.T;
  const long long o = (long long)b * a.C * a.T + (ok ? t : a.T - 1);
  const E *x = (const E*)a.x, *r = (const E*)a.r;
  const Site c = site(a);
  float s = 0.f, v = 0.f, k;
  for (int i = ty; i < a.C; i += TY) s += junction1<E>(x, r, o + (long long)i * a.T, c, k);
  const float mu = wide_sum(s, sh, tx, ty) / a.C;
  for (int i = ty; i < a.C; i += TY) {
    const float d = junction1<E>(x, r, o + (long long)i * a.T, c, k) - mu;
    v = fmaf(d, d, v);
  }
  const float rs = 1.f / sqrtf(wide_sum(v, sh, tx, ty) / a.C + a.eps);
  if (!ok) return;
  const float m = a.mask ? a.mask[(long long)b * a.T + t] : 1.f;
  if (ty == 0 && a.mean) {
    a.mean[(long long)b * a.T + t] = mu;
    a.rstd[(long long)b * a.T + t] = rs;
  }
  for (int i = ty; i < a.C; i += TY) {
    const long long j = o + (long long)i * a.T;
    const float u = fmaf((junction1<E>(x, r, j, c, k) - mu) * rs, a.gamma[i], a.beta[i]);
    ((E*)a.y)[j] = (E)(m != 0.f ? u * m : 0.f);
  }
}
template <typename E>
__global__ __launch_bounds__(THR) void junction_wide_bwd_kernel(svc_dropout_add_layernorm_t a, int tiles_t, float* part) {
  __shared__ float sh[TY][TX];
  const int tx = threadIdx.x & (TX - 1), ty = threadIdx.x / TX, t = (int)(blockIdx.x % tiles_t) * TX + tx, b = blockIdx.x / tiles_t;
  const bool ok = t < a.T;
  const int tc = ok ? t : a.T - 1;
  const long long o = (long long)b * a.C * a.T + tc;
  const E *x = (const E*)a.x, *r = (const E*)a.r, *dy = (const E*)a.dy;
  const Site c = site(a);
  const float m = !ok ? 0.f : a.mask ? a.mask[(long long)b * a.T + t] : 1.f;
  const bool on = m != 0.f;
  const float mu = a.mean[(long long)b * a.T + tc], rs = a.rstd[(long long)b * a.T + tc];
  float s1 = 0.f, s2 = 0.f, k;
  for (int i = ty; i < a.C; i += TY) {
    const long long j = o + (long long)i * a.T;
    const float g0 = on ? (float)dy[j] * m : 0.f, xh = on ? (junction1<E>(x, r, j, c, k) - mu) * rs : 0.f, g = g0 * a.gamma[i];
    s1 += g;
    s2 = fmaf(g, xh, s2);
    float pg = g0 * xh, pb = g0;
    for (int q = 32; q > 0; q >>= 1) {
      pg += __shfl_xor(pg, q);
      pb += __shfl_xor(pb, q);
    }
    if (tx == 0) {
      part[(2LL * blockIdx.x) * a.C + i] = pg;
      part[(2LL * blockIdx.x + 1) * a.C + i] = pb;
    }
  }
  s1 = wide_sum(s1, sh, tx, ty) / a.C;
  s2 = wide_sum(s2, sh, tx, ty) / a.C;
  if (!ok) return;
  for (int i = ty; i < a.C; i += TY) {
    const long long j = o + (long long)i * a.T;
    const float xh = on ? (junction1<E>(x, r, j, c, k) - mu) * rs : 0.f;
    if (!on && c.drop) k = 0.f;
    const float d = on ? rs * ((float)dy[j] * m * a.gamma[i] - s1 - xh * s2) : 0.f;
    if (a.dr) ((E*)a.dr)[j] = (E)d;
    if (a.dx) ((E*)a.dx)[j] = (E)(on ? d * k : 0.f);
  }
}

// dgamma[c], dbeta[c]: the workgroups' sums in fixed order; 32 channels x 32 strands a workgroup
__global__ __launch_bounds__(1024) void junction_param_kernel(const float* __restrict__ part, float* __restrict__ dgamma, float* __restrict__ dbeta, int C,
                                                              int blocks) {
  __shared__ double sh[32][33];
  const int cx = threadIdx.x & 31, k = threadIdx.x >> 5, c = blockIdx.x * 32 + cx;      // c over 2 C: gamma's, then beta's
  double s = 0.0;
  if (c < 2 * C)
    for (int i = k; i < blocks; i += 32) s += (double)part[2LL * i * C + c];
  sh[k][cx] = s;
  __syncthreads();
  for (int q = 16; q > 0; q >>= 1) {
    if (k < q) sh[k][cx] += sh[k + q][cx];
    __syncthreads();
  }
  if (k == 0 && c < 2 * C) (c < C ? dgamma : dbeta)[c < C ? c : c - C] = (float)sh[0][cx];
}

// How a launch is cut.  LPR = 4: 16 time steps a workgroup, up to 1024 channels in at most 128 registers a thread, which leaves room for a second workgroup
// on the CU: one loads while the other draws, sums and stores.  LPR = 2: 8 steps, for tensors of so few columns that 16-step tiles would leave
// most CUs without one (1 x 192 x 862 fp32: 6.2 us for 7.9 with 16; 16 x 192 x 790: 19 and 23 us with 8 for 13 and 19 with 16).  NR: channels of a
// thread, the smallest built number that covers C; none: the kernels that read the tensors again (32 x 768 x 1499 bf16: 265 and 360 us for 91 and 188).
struct Plan {
  int lpr, nr, tiles_t, blocks;
  long long n_tiles;
};
static Plan plan_of(int B, int C, int T, bool backward) {
  Plan p;
  p.lpr = (long long)B * svc::cdiv(T, 16) >= 256 ? 4 : 2;
  const int need = svc::cdiv(C, THR / p.lpr);
  static const int built[] = {1, 2, 3, 4, 6, 8};
  p.nr = 0;
  for (int n : built)
    if (n >= need) {
      p.nr = n;
      break;
    }
  if ((p.lpr == 2 && p.nr > 4) || (long long)C * T >= (1LL << 30)) p.nr = 0;      // (the register kernels' offsets are 32-bit bytes)
  p.tiles_t = svc::cdiv(T, p.nr ? p.lpr * V : TX);
  p.n_tiles = (long long)B * p.tiles_t;
  p.blocks = (int)p.n_tiles;
  if (backward && p.nr && p.n_tiles > 512) p.blocks = 512;
  return p;
}

template <typename E, int LPR, int NR>
static void launch(const svc_dropout_add_layernorm_t& a, const Plan& p, bool backward, hipStream_t s) {
  if (backward)
    hipLaunchKernelGGL((junction_bwd_kernel<E, LPR, NR>), dim3(p.blocks), dim3(THR), 0, s, a, p.tiles_t, p.n_tiles, (float*)a.ws);
  else
    hipLaunchKernelGGL((junction_fwd_kernel<E, LPR, NR>), dim3(p.blocks), dim3(THR), 0, s, a, p.tiles_t, p.n_tiles);
}
template <typename E>
static void run(const svc_dropout_add_layernorm_t& a, const Plan& p, bool backward, hipStream_t s) {
  if (p.nr == 0) {
    if (backward) hipLaunchKernelGGL((junction_wide_bwd_kernel<E>), dim3(p.blocks), dim3(THR), 0, s, a, p.tiles_t, (float*)a.ws);
    else hipLaunchKernelGGL((junction_wide_fwd_kernel<E>), dim3(p.blocks), dim3(THR), 0, s, a, p.tiles_t);
  } else if (p.lpr == 2) {
    switch (p.nr) {
      case 1: return launch<E, 2, 1>(a, p, backward, s);
      case 2: return launch<E, 2, 2>(a, p, backward, s);
      case 3: return launch<E, 2, 3>(a, p, backward, s);
      default: return launch<E, 2, 4>(a, p, backward, s);
    }
  } else {
    switch (p.nr) {
      case 1: return launch<E, 4, 1>(a, p, backward, s);
      case 2: return launch<E, 4, 2>(a, p, backward, s);
      case 3: return launch<E, 4, 3>(a, p, backward, s);
      case 4: return launch<E, 4, 4>(a, p, backward, s);
      case 6: return launch<E, 4, 6>(a, p, backward, s);
      default: return launch<E, 4, 8>(a, p, backward, s);
    }
  }
}

// (a launch has fewer than 2^32 threads: 512 for 16 columns, 1024 for 16 channels' sums)
bool sizes_fit(int B, int C, int T) { return B < 65536 && C < (1 << 25) && (long long)B * ((T + 15LL) / 16) < (1LL << 23); }

int check(const svc_dropout_add_layernorm_t* a, bool backward) {
  SVC_REQUIRE(a, "dropout_add_layernorm: no arguments");
  SVC_REQUIRE(a->dtype >= 0 && a->dtype <= 2, "dropout_add_layernorm: dtype %d", a->dtype);
  SVC_REQUIRE(a->B >= 0 && a->B < 65536 && a->C >= 1 && a->T >= 0, "dropout_add_layernorm: B=%d C=%d T=%d", a->B, a->C, a->T);
  SVC_REQUIRE(!a->seed || (a->p >= 0.f && a->p < 1.f), "dropout_add_layernorm: rate %g (0 <= p < 1)", a->p);
  SVC_REQUIRE(a->eps > 0.f, "dropout_add_layernorm: eps %g", a->eps);
  if (a->B == 0 || a->T == 0) return SVC_OK;
  SVC_REQUIRE(sizes_fit(a->B, a->C, a->T), "dropout_add_layernorm: B=%d C=%d T=%d (built for 2^27 columns, 2^25 channels)",
              a->B, a->C, a->T);
  SVC_REQUIRE(a->x && a->gamma && a->beta, "dropout_add_layernorm: x, gamma, beta");
  if (!backward) {
    SVC_REQUIRE(a->y && !a->mean == !a->rstd, "dropout_add_layernorm_fwd: y, and mean with rstd");
  } else {
    SVC_REQUIRE(a->dy && a->mean && a->rstd && (a->dr || a->dx) && a->dgamma && a->dbeta, "dropout_add_layernorm_bwd: dy, mean, rstd, dr or dx, dgamma, dbeta");
    const long long need = svc_dropout_add_layernorm_ws_bytes(a->B, a->C, a->T);
    SVC_REQUIRE(a->ws && a->ws_bytes >= need && ((size_t)a->ws & 15) == 0, "dropout_add_layernorm_bwd: workspace of %lld bytes needed, %lld given", need,
                a->ws ? a->ws_bytes : 0LL);
  }
  return SVC_OK;
}

}  // namespace

extern "C" {

long long svc_dropout_add_layernorm_ws_bytes(int B, int C, int T) {
  return B < 1 || C < 1 || T < 1 || !sizes_fit(B, C, T) ? 0 : 2LL * C * plan_of(B, C, T, true).blocks * 4;
}

int svc_dropout_add_layernorm_fwd(const svc_dropout_add_layernorm_t* a, void* stream) {
  const int rc = check(a, false);
  if (rc != SVC_OK || a->B == 0 || a->T == 0) return rc;
  hipStream_t s = (hipStream_t)stream;
  const double n = (double)a->B * a->C * a->T;
  svc::ProfScope prof(s, "dropout_add_layernorm_fwd", 9 * n, 3 * n * (a->dtype == SVC_F32 ? 4 : 2));
  const Plan p = plan_of(a->B, a->C, a->T, false);
  if (a->dtype == SVC_F32) run<float>(*a, p, false, s);
  else if (a->dtype == SVC_BF16) run<bf16_t>(*a, p, false, s);
  else run<f16_t>(*a, p, false, s);
  return svc::check_launch("svc_dropout_add_layernorm_fwd");
}

int svc_dropout_add_layernorm_bwd(const svc_dropout_add_layernorm_t* a, void* stream) {
  const int rc = check(a, true);
  if (rc != SVC_OK) return rc;
  SVC_REQUIRE(a->B > 0 && a->T > 0, "dropout_add_layernorm_bwd: nothing to differentiate");
  hipStream_t s = (hipStream_t)stream;
  const double n = (double)a->B * a->C * a->T;
  svc::ProfScope prof(s, "dropout_add_layernorm_bwd", 15 * n, (a->dx && a->dr ? 5 : 4) * n * (a->dtype == SVC_F32 ? 4 : 2));
  const Plan p = plan_of(a->B, a->C, a->T, true);
  if (a->dtype == SVC_F32) run<float>(*a, p, true, s);
  else if (a->dtype == SVC_BF16) run<bf16_t>(*a, p, true, s);
  else run<f16_t>(*a, p, true, s);
  hipLaunchKernelGGL(junction_param_kernel, dim3(svc::cdiv(2 * a->C, 32)), dim3(1024), 0, s, (const float*)a->ws, a->dgamma, a->dbeta, a->C, p.blocks);
  return svc::check_launch("svc_dropout_add_layernorm_bwd");
}

}  // extern "C"
