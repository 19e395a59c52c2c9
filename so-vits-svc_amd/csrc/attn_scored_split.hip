// attn_scored_split.hip — svc_attn_scored_fwd for few queries: a token over a cache, a short chunk.
//
// There are few softmax rows and many keys, so the work is cut along the keys: a workgroup takes 32 columns — (query head, query) pairs of one key head, so
// that shared key heads are read once — and one of `parts` equal parts of the keys they see; its four waves take tiles of it in turn, each through LDS
// of its own, with no barrier until their results are joined.  Bandwidth is the bound: the next tile's loads (16 KB a wave at 128 channels) are in
// flight while a tile is worked on.  With more than one part the partial maxima, sums and outputs go through the workspace and a second launch.
// Measured: 16 streams, 16 query and 4 key heads of 128 channels, caches of 8191 keys of different fill, bf16: 54 us = 3.8 TB/s on one set of caches, 63 on two in
// turn, and 7 us to join the parts; 2 heads of 96 channels, 862 keys, fp32: 19 + 4 us, latency of 32 waves: the matrix instructions, of whose 32 columns a single query
// uses one, take 22 % of a wave's cycles, the vector unit 17 %, waits 36 %; and two launches.
#include "attn_scored.h"

namespace attn {

// 16-byte loads of a tile and both its matrices take 2 DP / 16 (64-byte rows) registers x 4
template <typename E> constexpr int SPLIT_RB = sizeof(E) == 2 ? 64 : 128;

template <typename E, int DP, int MODE>
__global__ __launch_bounds__(256, DP > (sizeof(E) == 4 ? 64 : 96) ? 1 : 2) void split_kernel(svc_attn_scored_t a, Split sp) {
  constexpr int RB = SPLIT_RB<E>;
  typedef Tile<E, RB, 64> TL;
  constexpr int N = TL::N;
  static_assert(TL::RT == 1, "a wave's tile is 32 keys");
  // bytes of a wave: its k and v tiles, in whose place its output, DP x 32 floats, and its maxima and sums come
  constexpr int WAVE = 2 * DP * TL::PITCH > DP * 128 + 256 ? 2 * DP * TL::PITCH : DP * 128 + 256;
  __shared__ __align__(16) char lds_[4 * WAVE];
  // (the waves' maxima and sums go behind their outputs)
  auto ms = [&](int w) { return (float*)(lds_ + w * WAVE + DP * 128); };
  auto ls = [&](int w) { return (float*)(lds_ + w * WAVE + DP * 128) + 32; };
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5, n = lane & 31, rep = a.H / a.G;
  const int part = blockIdx.x % sp.parts, blk = blockIdx.x / sp.parts % sp.blocks, bg = blockIdx.x / (sp.parts * sp.blocks);
  const int b = bg / a.G, kvh = bg % a.G, col = blk * 32 + n;
  const bool in = col < sp.cols;
  const int head = kvh * rep + (in ? col / a.Tq : 0), t = in ? col % a.Tq : 0;
  const int len = item_length(a, b), off = item_offset(a, b);
  int2 iv = make_int2(0, 0);
  if (in && (!a.offsets || (off >= -a.Tq && off < a.Tk))) iv = visible(a, b, len, off + t);
  const bool some = iv.y > iv.x;
  const int lo = wave_min(some ? iv.x : a.Tk), hi = wave_max(iv.y);              // the same in every wave
  const int flo = wave_max(in ? (some ? iv.x : a.Tk) : 0), fhi = wave_min(in ? iv.y : a.Tk);
  // this part's tiles, of which wave w takes every fourth
  const int first = lo / N, tiles = hi > lo ? (hi + N - 1) / N - first : 0;
  const int beg = first + (int)((long long)tiles * part / sp.parts), end = first + (int)((long long)tiles * (part + 1) / sp.parts);

  typename Frag<E>::template Head<DP> q;
  {
    const E* x = (const E*)a.q + b * a.q_bs + (long long)head * a.dk * a.q_cs + t;
    if constexpr (sizeof(E) == 4) {
#pragma unroll
      for (int i = 0; i < DP / 2; ++i) q.v[i] = in && 2 * i + h < a.dk ? x[(2 * i + h) * a.q_cs] : 0.f;
    } else if (a.q_cs == 1) {                                     // a single query: its channels are neighbours
#pragma unroll
      for (int i = 0; i < DP / 16; ++i) {
        union { uint4 u; E e[8]; typename Frag<E>::V v; } c;
        c.u = make_uint4(0, 0, 0, 0);
        const int d = 16 * i + 8 * h;
        if (in && d + 8 <= a.dk) {
          const U128 u = *(const U128*)(x + d);
          c.u = make_uint4(u.x, u.y, u.z, u.w);
        } else if (in) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (d + e < a.dk) c.e[e] = x[d + e];
        }
        q.v[i] = c.v;
      }
    } else {
#pragma unroll
      for (int i = 0; i < DP / 16; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int d = 16 * i + 8 * h + e;
          q.v[i][e] = in && d < a.dk ? x[d * a.q_cs] : (E)0.f;
        }
    }
  }
  const ScoreScale sc = score_scale(a);
  const float* table = a.bias ? a.bias + (a.bias_heads > 1 ? (long long)head * (2 * a.bias_w + 1) : 0) + a.bias_w : nullptr;
  unsigned long long draws = 0;
  unsigned thr = 0;
  if (a.seed) {
    draws = draw_start(a) + ((unsigned long long)(((long long)b * a.H + head) * a.Tq + t) * (unsigned long long)((a.Tk + 3) >> 2) + 2 * h) * DRAW_STEP;
    thr = (unsigned)rintf(a.p_drop * 65536.f);
  }
  f32x16 acc[DP / 32];
#pragma unroll
  for (int i = 0; i < DP / 32; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[i][r] = 0.f;
  float m = -INFINITY, l = 0.f;

  E* const ks = (E*)(lds_ + wave * WAVE);
  E* const vs = ks + DP * TL::P;
  Source<E, DP, RB, 64> ksrc, vsrc;
  ksrc.set((const E*)a.k + b * a.k_bs + (long long)kvh * a.dk * a.k_cs, a.k_cs, a.dk, a.Tk, lane);
  vsrc.set((const E*)a.v + b * a.v_bs + (long long)kvh * a.dk * a.v_cs, a.v_cs, a.dk, a.Tk, lane);
  Pre<E, DP, RB, 64> kf, vf;
  ksrc.fetch(kf, (beg + wave) * N, lane);                         // (behind the last tile: values that are not used)
  vsrc.fetch(vf, (beg + wave) * N, lane);
  for (int tile = beg + wave; tile < end; tile += 4) {
    const int s0 = tile * N;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    ksrc.commit(ks, kf, s0, lo, hi, lane);
    vsrc.commit(vs, vf, s0, lo, hi, lane);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    float bias[16];
    if (table) {
#pragma unroll
      for (int r = 0; r < 16; ++r) bias[r] = table[min(max(s0 + pos_of(r, h) - off - t, -a.bias_w), a.bias_w)];
    }
    ksrc.fetch(kf, s0 + 4 * N, lane);
    vsrc.fetch(vf, s0 + 4 * N, lane);
    const f32x16 u = mul_columns<E, DP, RB>(ks, 0, q, lane);
    float s[16], mul = sc.mul;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = u[r];
    if (sc.cap) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = capped<MODE == 2>(s[r], sc);
      mul = 1.f;
    }
    if (table) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = fmaf(s[r], mul, bias_scaled(bias[r]));
      mul = 1.f;
    }
    if (s0 < flo || s0 + N > fhi) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const unsigned p = s0 + pos_of(r, h) - iv.x;
        s[r] = p < (unsigned)(iv.y - iv.x) ? s[r] : -INFINITY;
      }
    }
    float mt = -INFINITY;
#pragma unroll
    for (int r = 0; r < 16; r += 2) mt = fmaxf(fmaxf(s[r], s[r + 1]), mt);
    mt = fmaxf(mt, __shfl_xor(mt, 32)) * mul;
    const float m1 = fmaxf(m, mt), alpha = __builtin_amdgcn_exp2f(m1 == -INFINITY ? 0.f : m - m1), mz = m1 == -INFINITY ? 0.f : m1 - PUP<E>;
    m = m1;
    l *= alpha;
#pragma unroll
    for (int i = 0; i < DP / 32; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][r] *= alpha;
    float lt = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], mul, -mz));
      lt += s[r];
    }
    l += lt;
    if (a.seed) {
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const unsigned long long z = draw_word(draws + draw_block(s0) + draw_group(w));
#pragma unroll
        for (int j = 0; j < 4; ++j) s[4 * w + j] = dropped(z, j, thr) ? 0.f : s[4 * w + j];
      }
    }
    mul_rows<E, DP, P_OPS<E, MODE>, RB>(acc, vs, 0, s, lane);
  }
  l += __shfl_xor(l, 32);

  // the four waves' results: a common maximum, scaled outputs through LDS as [d][column], summed in the order of the waves
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  if (h == 0) {
    ms(wave)[n] = m;
    ls(wave)[n] = l;
  }
  __syncthreads();
  const float mb = fmaxf(fmaxf(ms(0)[n], ms(1)[n]), fmaxf(ms(2)[n], ms(3)[n]));
  const float mine = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mb);
  float* const o = (float*)(lds_ + wave * WAVE);
#pragma unroll
  for (int i = 0; i < DP / 32; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[(32 * i + 8 * (r >> 2) + 4 * h + (r & 3)) * 32 + n] = acc[i][r] * mine;
  __syncthreads();
  const int c = tid & 31, cc = blk * 32 + c;
  if (cc >= sp.cols) return;
  float lsum = 0.f, mc = -INFINITY;
#pragma unroll
  for (int w = 0; w < 4; ++w) mc = fmaxf(mc, ms(w)[c]);
#pragma unroll
  for (int w = 0; w < 4; ++w)          // (a wave without a maximum has the sum 0, or nan where its scores are)
    lsum = fmaf(ls(w)[c], ms(w)[c] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ms(w)[c] - mc), lsum);
  const float* const f = (const float*)lds_ + c;
  constexpr int FW = WAVE / 4;
  if (sp.parts > 1) {
    const long long P = (long long)a.B * a.G * sp.cols * sp.parts, at = ((long long)bg * sp.cols + cc) * sp.parts + part;
    float* w = (float*)a.ws;
    if (tid < 32) {
      w[at] = mc;
      w[P + at] = lsum;
    }
    // [part][channel][column]: neighbouring threads write neighbouring columns
    float* y = w + 2 * P + (((long long)bg * sp.parts + part) * a.dk) * sp.cols + cc;
    for (int d = tid >> 5; d < a.dk; d += 8) y[(long long)d * sp.cols] = (f[d * 32] + f[d * 32 + FW]) + (f[d * 32 + 2 * FW] + f[d * 32 + 3 * FW]);
  } else {
    const int hc = kvh * rep + cc / a.Tq, tc = cc % a.Tq;
    const long long row = ((long long)b * a.H + hc) * a.Tq + tc;
    float inv = lsum > 0.f ? 1.f / lsum : 0.f;
    if (lsum != lsum) inv = lsum;
    if (a.seed) inv *= 65536.f / (65536.f - (float)thr);
    if (a.lse && tid < 32) a.lse[row] = lsum > 0.f || lsum != lsum ? mc - PUP<E> + __builtin_amdgcn_logf(lsum) : 0.f;
    E* y = (E*)a.out + b * a.o_bs + (long long)hc * a.dk * a.o_cs + tc;
    float* y32 = a.out32 ? a.out32 + ((long long)b * a.H + hc) * a.dk * a.Tq + tc : nullptr;
    for (int d = tid >> 5; d < a.dk; d += 8) {
      const float v = ((f[d * 32] + f[d * 32 + FW]) + (f[d * 32 + 2 * FW] + f[d * 32 + 3 * FW])) * inv;
      y[d * a.o_cs] = (E)v;
      if (y32) y32[(long long)d * a.Tq] = v;
    }
  }
}

// The parts' results, in their order: one thread per (column, channel), 32 columns x 8 channels a workgroup.
template <typename E>
__global__ __launch_bounds__(256) void join_kernel(svc_attn_scored_t a, Split sp) {
  const int dblocks = (a.dk + 7) / 8, db = blockIdx.x % dblocks, blk = blockIdx.x / dblocks % sp.blocks, bg = blockIdx.x / (dblocks * sp.blocks);
  const int b = bg / a.G, kvh = bg % a.G, c = blk * 32 + (threadIdx.x & 31), d = db * 8 + (threadIdx.x >> 5);
  if (c >= sp.cols || d >= a.dk) return;
  const long long P = (long long)a.B * a.G * sp.cols * sp.parts, at = ((long long)bg * sp.cols + c) * sp.parts;
  const float* w = (const float*)a.ws;
  float m = -INFINITY, l = 0.f, v = 0.f;
  for (int p = 0; p < sp.parts; ++p) m = fmaxf(m, w[at + p]);
  const float* y = w + 2 * P + ((long long)bg * sp.parts * a.dk + d) * sp.cols + c;
  for (int p = 0; p < sp.parts; ++p) {
    const float f = w[at + p] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(w[at + p] - m);
    l = fmaf(w[P + at + p], f, l);
    v = fmaf(y[(long long)p * a.dk * sp.cols], f, v);
  }
  float inv = l > 0.f ? 1.f / l : 0.f;
  if (l != l) inv = l;
  if (a.seed) inv *= 65536.f / (65536.f - rintf(a.p_drop * 65536.f));
  const int head = kvh * (a.H / a.G) + c / a.Tq, t = c % a.Tq;
  if (a.lse && d == 0) a.lse[((long long)b * a.H + head) * a.Tq + t] = l > 0.f || l != l ? m - PUP<E> + __builtin_amdgcn_logf(l) : 0.f;
  v *= inv;
  ((E*)a.out)[b * a.o_bs + ((long long)head * a.dk + d) * a.o_cs + t] = (E)v;
  if (a.out32) a.out32[(((long long)b * a.H + head) * a.dk + d) * a.Tq + t] = v;
}

// Few queries (up to 64: fwd_kernel's workgroups of 128 would stand half empty), parts so that there are about two workgroups a CU, each wave with two
// tiles at least.  This way against fwd_kernel's: one query over 862 keys fp32 24 us for 105, one for each of 16 streams over 8191 keys 81 for 279 (64
// since), 37 queries over 1500 keys with a window of 200 15.5 for 15.7: even where the columns fill the workgroup.
Split split_of(const svc_attn_scored_t& a) {
  Split p;
  p.cols = a.H / a.G * a.Tq;
  p.blocks = (p.cols + 31) / 32;
  p.parts = 0;
  if (a.Tq > 64) return p;
  const long long groups = (long long)a.B * a.G * p.blocks;
  const long long seen = a.window >= 0 && 2LL * a.window + a.Tq < a.Tk ? 2LL * a.window + a.Tq : a.Tk;       // keys that the columns can see
  const long long most = svc::cdivll(seen, 32 * 4 * 2), want = svc::cdivll(512, groups);
  p.parts = (int)(want < most ? want : most);
  if (p.parts < 1) p.parts = 1;
  return p;
}
long long split_ws_bytes(const svc_attn_scored_t& a, const Split& p) {
  return p.parts > 1 ? (long long)a.B * a.G * p.cols * p.parts * (2 + (long long)a.dk) * 4 : 0;
}

template <typename E, int DP>
static void go(const svc_attn_scored_t& a, const Split& p, hipStream_t s) {
  const dim3 grid((unsigned)((long long)a.B * a.G * p.blocks * p.parts));
  constexpr bool F = sizeof(E) == 4;
  if (F || a.exact || a.softcap > SHORT_CAP) hipLaunchKernelGGL((split_kernel<E, DP, 2>), grid, dim3(256), 0, s, a, p);
  else if (a.out32) hipLaunchKernelGGL((split_kernel<E, DP, F ? 2 : 1>), grid, dim3(256), 0, s, a, p);
  else hipLaunchKernelGGL((split_kernel<E, DP, F ? 2 : 0>), grid, dim3(256), 0, s, a, p);
}
template <typename E>
static void pick(const svc_attn_scored_t& a, const Split& p, hipStream_t s) {
  if (a.dk <= 32) go<E, 32>(a, p, s);
  else if (a.dk <= 64) go<E, 64>(a, p, s);
  else if (a.dk <= 96) go<E, 96>(a, p, s);
  else go<E, 128>(a, p, s);
  if (p.parts > 1) {
    const dim3 grid((unsigned)((long long)a.B * a.G * p.blocks * ((a.dk + 7) / 8)));
    hipLaunchKernelGGL((join_kernel<E>), grid, dim3(256), 0, s, a, p);
  }
}
void launch_split(const svc_attn_scored_t& a, const Split& p, hipStream_t s) {
  if (a.dtype == SVC_F32) pick<float>(a, p, s);
  else if (a.dtype == SVC_BF16) pick<bf16_t>(a, p, s);
  else pick<f16_t>(a, p, s);
}

}  // namespace attn
