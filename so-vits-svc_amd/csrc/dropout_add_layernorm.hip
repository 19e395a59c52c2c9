// dropout_add_layernorm.hip — the residual junction of a transformer layer: y = LayerNorm_C(r + dropout(x)) * gamma + beta (* mask), forward and
// backward, on [B, C, T] with time contiguous (modules/attentions.py:51-55,100-104, modules/modules.py:23-35).
//
// The backward keeps nothing but mean and rstd: h = r + dropout(x) is recomputed from x, r and the counter draws, which moves the same bytes as
// storing h would (one write and one read against two reads in place of one) and takes no memory.
#include "common.h"

namespace {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

// svc_dropout_rng_f32's draw (splitmix64's finaliser over a counter)
__device__ __forceinline__ float draw_uniform(unsigned long long start, unsigned long long idx) {
  unsigned long long z = start + idx * 0xD1B54A32D192ED03ull;
  z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
  z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
  z = z ^ (z >> 31);
  return (float)(unsigned)(z >> 40) * (1.0f / 16777216.0f);
}

constexpr int TX = 64, TY = 8;         // 64 time steps x 8 channel groups a workgroup

__device__ __forceinline__ float column_sum(float part, float (*sh)[TX], int tx, int ty) {
  __syncthreads();
  sh[ty][tx] = part;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < TY; ++i) s += sh[i][tx];
  return s;
}

template <typename E>
struct Cols {
  const E *x, *r;
  unsigned long long start;
  bool drop;
  float p, ks;
  __device__ __forceinline__ float keep(long long i) const { return !drop ? 1.f : draw_uniform(start, (unsigned long long)i) >= p ? ks : 0.f; }
  __device__ __forceinline__ float h(long long i) const {
    const float v = (float)x[i], k = keep(i);
    const float d = k != 0.f ? v * k : 0.f;
    return r ? (float)r[i] + d : d;
  }
};
template <typename E> __device__ __forceinline__ Cols<E> cols(const svc_dropout_add_layernorm_t& a) {
  Cols<E> c;
  c.x = (const E*)a.x;
  c.r = (const E*)a.r;
  c.drop = a.seed != nullptr;
  c.start = c.drop ? (unsigned long long)a.seed[0] + (unsigned long long)((unsigned)a.site + 1u) * 0x9E3779B97F4A7C15ull : 0;
  c.p = a.p;
  c.ks = 1.f / (1.f - a.p);
  return c;
}

template <typename E>
__global__ __launch_bounds__(TX * TY) void junction_fwd_kernel(svc_dropout_add_layernorm_t a) {
  __shared__ float sh[TY][TX];
  const int tx = threadIdx.x & (TX - 1), ty = threadIdx.x / TX, t = blockIdx.x * TX + tx, b = blockIdx.y;
  const bool ok = t < a.T;
  const long long o = (long long)b * a.C * a.T + (ok ? t : a.T - 1);
  const Cols<E> c = cols<E>(a);
  float s = 0.f;
  for (int i = ty; i < a.C; i += TY) s += c.h(o + (long long)i * a.T);
  const float mu = column_sum(s, sh, tx, ty) / a.C;
  float v = 0.f;
  for (int i = ty; i < a.C; i += TY) {
    const float d = c.h(o + (long long)i * a.T) - mu;
    v = fmaf(d, d, v);
  }
  const float rs = 1.f / sqrtf(column_sum(v, sh, tx, ty) / a.C + a.eps);
  if (!ok) return;
  const float m = a.mask ? a.mask[(long long)b * a.T + t] : 1.f;
  if (ty == 0 && a.mean) {
    a.mean[(long long)b * a.T + t] = mu;
    a.rstd[(long long)b * a.T + t] = rs;
  }
  E* y = (E*)a.y;
  for (int i = ty; i < a.C; i += TY) {
    const long long j = o + (long long)i * a.T;
    const float u = fmaf((c.h(j) - mu) * rs, a.gamma[i], a.beta[i]);
    y[j] = (E)(m != 0.f ? u * m : 0.f);
  }
}

template <typename E>
__global__ __launch_bounds__(TX * TY) void junction_bwd_kernel(svc_dropout_add_layernorm_t a, float* part) {
  __shared__ float sh[TY][TX];
  const int tx = threadIdx.x & (TX - 1), ty = threadIdx.x / TX, t = blockIdx.x * TX + tx, b = blockIdx.y;
  const long long blk = (long long)b * gridDim.x + blockIdx.x, blocks = (long long)gridDim.x * gridDim.y;
  const bool ok = t < a.T;
  const int tc = ok ? t : a.T - 1;
  const long long o = (long long)b * a.C * a.T + tc;
  const Cols<E> c = cols<E>(a);
  const E* dy = (const E*)a.dy;
  float m = ok ? 1.f : 0.f;
  if (a.mask && ok) m = a.mask[(long long)b * a.T + t];
  const bool on = m != 0.f;
  const float mu = a.mean[(long long)b * a.T + tc], rs = a.rstd[(long long)b * a.T + tc];
  float s1 = 0.f, s2 = 0.f;
  for (int i = ty; i < a.C; i += TY) {
    const long long j = o + (long long)i * a.T;
    const float g0 = on ? (float)dy[j] * m : 0.f, xh = on ? (c.h(j) - mu) * rs : 0.f, g = g0 * a.gamma[i];
    s1 += g;
    s2 = fmaf(g, xh, s2);
    // the parameters' sums over this workgroup's 64 steps
    float pg = g0 * xh, pb = g0;
    for (int q = 32; q > 0; q >>= 1) {
      pg += __shfl_xor(pg, q);
      pb += __shfl_xor(pb, q);
    }
    if (tx == 0) {
      part[(long long)i * blocks + blk] = pg;
      part[((long long)a.C + i) * blocks + blk] = pb;
    }
  }
  s1 = column_sum(s1, sh, tx, ty) / a.C;
  s2 = column_sum(s2, sh, tx, ty) / a.C;
  if (!ok) return;
  E *dr = (E*)a.dr, *dx = (E*)a.dx;
  for (int i = ty; i < a.C; i += TY) {
    const long long j = o + (long long)i * a.T;
    const float g = on ? (float)dy[j] * m * a.gamma[i] : 0.f, xh = on ? (c.h(j) - mu) * rs : 0.f;
    const float d = on ? rs * (g - s1 - xh * s2) : 0.f;
    if (dr) dr[j] = (E)d;
    if (dx) dx[j] = (E)(d * c.keep(j));
  }
}

// dgamma[c], dbeta[c]: the workgroups' sums in fixed order, one workgroup a value
__global__ __launch_bounds__(256) void junction_param_kernel(const float* __restrict__ part, float* __restrict__ dgamma, float* __restrict__ dbeta,
                                                             int C, long long blocks) {
  __shared__ double sh[256];
  const float* p = part + (long long)blockIdx.x * blocks;
  double s = 0.0;
  for (long long i = threadIdx.x; i < blocks; i += 256) s += (double)p[i];
  sh[threadIdx.x] = s;
  __syncthreads();
  for (int q = 128; q > 0; q >>= 1) {
    if (threadIdx.x < q) sh[threadIdx.x] += sh[threadIdx.x + q];
    __syncthreads();
  }
  if (threadIdx.x == 0) (blockIdx.x < C ? dgamma : dbeta)[blockIdx.x < C ? blockIdx.x : blockIdx.x - C] = (float)sh[0];
}

int check(const svc_dropout_add_layernorm_t* a, bool backward) {
  SVC_REQUIRE(a, "dropout_add_layernorm: no arguments");
  SVC_REQUIRE(a->dtype >= 0 && a->dtype <= 2, "dropout_add_layernorm: dtype %d", a->dtype);
  SVC_REQUIRE(a->B >= 0 && a->B < 65536 && a->C >= 1 && a->T >= 0, "dropout_add_layernorm: B=%d C=%d T=%d", a->B, a->C, a->T);
  SVC_REQUIRE(!a->seed || (a->p >= 0.f && a->p < 1.f), "dropout_add_layernorm: rate %g (0 <= p < 1)", a->p);
  SVC_REQUIRE(a->eps > 0.f, "dropout_add_layernorm: eps %g", a->eps);
  if (a->B == 0 || a->T == 0) return SVC_OK;
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
  return B < 1 || C < 1 || T < 1 ? 0 : 2LL * C * B * svc::cdiv(T, TX) * 4;
}

int svc_dropout_add_layernorm_fwd(const svc_dropout_add_layernorm_t* a, void* stream) {
  const int rc = check(a, false);
  if (rc != SVC_OK || a->B == 0 || a->T == 0) return rc;
  hipStream_t s = (hipStream_t)stream;
  const double n = (double)a->B * a->C * a->T;
  svc::ProfScope prof(s, "dropout_add_layernorm_fwd", 9 * n, 3 * n * (a->dtype == SVC_F32 ? 4 : 2));
  const dim3 g(svc::cdiv(a->T, TX), a->B), blk(TX * TY);
  if (a->dtype == SVC_F32) hipLaunchKernelGGL((junction_fwd_kernel<float>), g, blk, 0, s, *a);
  else if (a->dtype == SVC_BF16) hipLaunchKernelGGL((junction_fwd_kernel<bf16_t>), g, blk, 0, s, *a);
  else hipLaunchKernelGGL((junction_fwd_kernel<f16_t>), g, blk, 0, s, *a);
  return svc::check_launch("svc_dropout_add_layernorm_fwd");
}

int svc_dropout_add_layernorm_bwd(const svc_dropout_add_layernorm_t* a, void* stream) {
  const int rc = check(a, true);
  if (rc != SVC_OK) return rc;
  SVC_REQUIRE(a->B > 0 && a->T > 0, "dropout_add_layernorm_bwd: nothing to differentiate");
  hipStream_t s = (hipStream_t)stream;
  const double n = (double)a->B * a->C * a->T;
  svc::ProfScope prof(s, "dropout_add_layernorm_bwd", 15 * n, (a->dx && a->dr ? 5 : 4) * n * (a->dtype == SVC_F32 ? 4 : 2));
  const dim3 g(svc::cdiv(a->T, TX), a->B), blk(TX * TY);
  float* part = (float*)a->ws;
  if (a->dtype == SVC_F32) hipLaunchKernelGGL((junction_bwd_kernel<float>), g, blk, 0, s, *a, part);
  else if (a->dtype == SVC_BF16) hipLaunchKernelGGL((junction_bwd_kernel<bf16_t>), g, blk, 0, s, *a, part);
  else hipLaunchKernelGGL((junction_bwd_kernel<f16_t>), g, blk, 0, s, *a, part);
  hipLaunchKernelGGL(junction_param_kernel, dim3(2 * a->C), dim3(256), 0, s, part, a->dgamma, a->dbeta, a->C, (long long)g.x * g.y);
  return svc::check_launch("svc_dropout_add_layernorm_bwd");
}

}  // extern "C"
