// attn_scored_bwd.hip — svc_attn_scored_bwd: gradients of svc_attn_scored_fwd.  Two passes, each recomputing the scores it needs (a walk over
// keys for dq and the bias, a walk over queries for dk and dv): seven products instead of five, and in exchange no atomics on
// memory, so that results do not vary from run to run, and no copies of dq that a further launch would have to add up.  What stands around the passes is
// read once and small: the row sums 49 us at 4 x 16 x 128 x 4096 bf16 (dO and out32, 201 MB: 4.1 TB/s), 11 to 19 us elsewhere; the bias 5 us.
#include "attn_scored.h"

namespace attn {

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
  w.vmax = (float*)take(a.dtype == SVC_F16 ? (long long)a.B * a.G * ((a.Tk + 127) / 128) * 4 : 0);
  w.bins = (float*)take(a.dbias ? bh * t32 * (2LL * a.bias_w + 1) * 4 : 0);
  w.bytes = o;
  return w;
}

// ---- rows: D = sum_d dO[d,t] out[d,t], the largest |dO|, and the visible intervals.  64 queries of one head a workgroup; fp16: and the largest |v|, 128
// keys of one key head a workgroup behind those ----------
template <typename E>
__global__ __launch_bounds__(256) void rows_kernel(svc_attn_scored_t a, Ws w, int n_tiles) {
  __shared__ float sum[4][64], big[4][64];
  if constexpr (__is_same(E, f16_t)) {
    if ((int)blockIdx.x >= a.B * a.H * n_tiles) {
      const int nk = (a.Tk + 127) / 128, at = blockIdx.x - a.B * a.H * n_tiles, s = at % nk * 128 + (threadIdx.x & 127), b = at / nk / a.G, kvh = at / nk % a.G;
      int tbeg, tend, kbeg, kend;
      live_range(a, b, tbeg, tend, kbeg, kend);
      float g = 0.f;
      if (s >= kbeg && s < kend) {
        const E* v = (const E*)a.v + b * a.v_bs + (long long)kvh * a.dk * a.v_cs + s;
#pragma unroll 8
        for (int d = threadIdx.x >> 7; d < a.dk; d += 2) g = fmaxf(g, fabsf(to_f(v[d * a.v_cs])));
      }
      for (int o = 32; o > 0; o >>= 1) g = fmaxf(g, __shfl_xor(g, o));
      if ((threadIdx.x & 63) == 0) big[threadIdx.x >> 6][0] = g;
      __syncthreads();
      if (threadIdx.x == 0) w.vmax[at] = fmaxf(fmaxf(big[0][0], big[1][0]), fmaxf(big[2][0], big[3][0]));
      return;
    }
  }
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

// ---- dbias[head or 0][j] = sum of the 32-query bins over items (and heads, for a shared table), in fixed order: 16 entries x 64 strands a workgroup ------
__global__ __launch_bounds__(1024) void dbias_kernel(svc_attn_scored_t a, Ws ws) {
  __shared__ double sum[64][17];
  const int x = threadIdx.x & 15, k = threadIdx.x >> 4, nb = 2 * a.bias_w + 1, j = blockIdx.x * 16 + x, head = blockIdx.y, t32 = (a.Tq + 31) / 32;
  const bool shared = a.bias_heads == 1;
  const int n = (shared ? a.B * a.H : a.B) * t32;              // rows of bins; the item's (and head's) rows are neighbours
  double s = 0.0;
  if (j < nb)
    for (int i = k; i < n; i += 64) {
      const long long row = shared ? i : ((long long)(i / t32) * a.H + head) * t32 + i % t32;
      s += (double)ws.bins[row * nb + j];
    }
  sum[k][x] = s;
  __syncthreads();
  for (int q = 32; q > 0; q >>= 1) {
    if (k < q) sum[k][x] += sum[k + q][x];
    __syncthreads();
  }
  if (k == 0 && j < nb) a.dbias[(long long)head * nb + j] = (float)sum[0][x];
}

}  // namespace attn

extern "C" {

long long svc_attn_scored_ws_bytes(const svc_attn_scored_t* a, int backward) {
  if (!a || attn::check_sizes(a) != SVC_OK || a->B < 1 || a->Tq < 1) return 0;
  return backward ? attn::layout(*a).bytes : attn::split_ws_bytes(*a, attn::split_of(*a));
}

int svc_attn_scored_bwd(const svc_attn_scored_t* a, void* stream) {
  const int rc = attn::check_args(a, true);
  if (rc != SVC_OK || a->B == 0 || a->Tk == 0) return rc;
  SVC_REQUIRE(a->Tq > 0, "attn_scored_bwd: no queries");
  hipStream_t s = (hipStream_t)stream;
  svc::ProfScope prof(s, "attn_scored_bwd", 14.0 * a->B * a->H * (double)a->Tq * a->Tk * a->dk, 0);
  const attn::Ws w = attn::layout(*a);
  const int n64 = (a->Tq + 63) / 64;
  const int rows = a->B * a->H * n64, keys = a->dtype == SVC_F16 ? a->B * a->G * ((a->Tk + 127) / 128) : 0;      // (together up to 15 2^20 workgroups)
  const dim3 grid((unsigned)(rows + keys));
  if (a->dtype == SVC_F32) hipLaunchKernelGGL((attn::rows_kernel<float>), grid, dim3(256), 0, s, *a, w, n64);
  else if (a->dtype == SVC_BF16) hipLaunchKernelGGL((attn::rows_kernel<attn::bf16_t>), grid, dim3(256), 0, s, *a, w, n64);
  else hipLaunchKernelGGL((attn::rows_kernel<attn::f16_t>), grid, dim3(256), 0, s, *a, w, n64);
  attn::launch_dq(*a, w, s);
  attn::launch_dkv(*a, w, s);
  if (a->dbias) hipLaunchKernelGGL(attn::dbias_kernel, dim3((2 * a->bias_w + 16) / 16, a->bias_heads), dim3(1024), 0, s, *a, w);
  return svc::check_launch("svc_attn_scored_bwd");
}

}  // extern "C"
