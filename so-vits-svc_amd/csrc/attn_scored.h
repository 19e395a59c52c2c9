// attn_scored.h — what the kernels of svc_attn_scored_fwd / _bwd share: visible-key intervals, the dropout draws, the score, the
// operand layouts of the matrix instruction and the staging of [channel][time] tiles.
//
// Layout of the work.  Tensors are [B, heads*dk, T] with time contiguous, so for one head a matrix is X[d][t].  Every product is
// arranged so that the COLUMN of the 32 x 32 accumulator (a lane's n = lane & 31) is the index that a softmax row belongs to and the
// accumulator itself is the next product's right operand without leaving its registers:
//   forward, dq      S^T[s,t] = K^T Q   (rows s, columns t)  ->  out[d,t] += V[d,s] P^T[s,t],   dq[d,t] += K[d,s] dS^T[s,t]
//   dk, dv           S[t,s]   = Q^T K   (rows t, columns s)  ->  dv[d,s] += dO[d,t] P[t,s],     dk[d,s] += Q[d,t] dS[t,s]
// The first product's left operand reduces over d, which is strided in memory: 16-bit types read it from LDS with the transposing
// read (ds_read_b64_tr_b16), fp32 needs one value per lane and step and reads it as it lies.  The second product's left operand
// reduces over time, which is contiguous: a plain 16-byte LDS read.
//
// Row order.  Register r of half h of an accumulator holds row 8(r>>2) + 4h + (r&3).  Rows are assigned to tile positions with bits 2
// and 3 swapped (`swap23`), so that the register holds tile position 16(r>>3) + 8h + (r&7): eight neighbouring positions per half,
// which is what the second product's 16-byte operand read, the four-to-a-word dropout draws and the bias window want.
#pragma once
#include "common.h"

namespace attn {

typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16_t;
typedef _Float16 f16_t;
struct __attribute__((packed, aligned(2))) U128 { unsigned x, y, z, w; };     // 16 bytes at any 2-byte alignment

constexpr float LOG2E = 1.44269504088896340736f;
constexpr int NCOL = 128;               // columns of a workgroup: 4 waves x 32
constexpr int PITCH = 144;              // bytes of an LDS row: 128 of data + 16, which spreads both operand reads over all banks

template <typename E> struct Tile {     // positions of a staged tile row (128 bytes)
  static constexpr int N = 128 / (int)sizeof(E);
  static constexpr int RT = N / 32;     // 32-row accumulators a tile feeds
  static constexpr int P = PITCH / (int)sizeof(E);
  static constexpr int V = 16 / (int)sizeof(E);     // positions of a 16-byte chunk
};

__device__ __forceinline__ int swap23(int m) { return (m & ~12) | ((m & 4) << 1) | ((m & 8) >> 1); }
__device__ __forceinline__ int pos_of(int r, int h) { return 16 * (r >> 3) + 8 * h + (r & 7); }

// ---- visible keys of a query: the interval [lo, hi) of key positions, empty as lo = hi = 0 ---------------------------------------
__device__ __forceinline__ int item_length(const svc_attn_scored_t& a, int b) {
  return a.lengths ? min(max(a.lengths[b], 0), a.Tk) : a.Tk;
}
__device__ __forceinline__ int item_offset(const svc_attn_scored_t& a, int b) { return a.offsets ? a.offsets[b] : a.offset; }

__device__ __forceinline__ int2 visible(const svc_attn_scored_t& a, int b, int len, int pos) {
  if (pos < 0 || pos >= len) return make_int2(0, 0);
  int lo = 0, hi = len, start = 0, front = 0, n = 0;
  if (a.n_docs) {
    const int* d = a.docs + (long long)b * (a.n_docs + 1);
    int l = 0, r = a.n_docs + 1;        // number of boundaries <= pos
    while (l < r) {
      const int m = (l + r) >> 1;
      if (d[m] <= pos) l = m + 1;
      else r = m;
    }
    if (l < 1 || l > a.n_docs) return make_int2(0, 0);
    n = l - 1;
    start = max(d[n], 0);
    lo = start;
    hi = min(hi, d[n + 1]);
  }
  if (a.causal) {
    if (a.prefix) front = a.prefix[(long long)b * (a.n_docs ? a.n_docs : 1) + n];
    // (in 64 bits: a prefix length is the caller's data and may be any int32)
    const long long end = (long long)start + front;
    hi = min(hi, end > pos + 1 ? (int)(end < hi ? end : hi) : pos + 1);
  }
  if (a.window >= 0) {
    lo = max(lo, pos - min(a.window, pos));
    hi = a.window < hi - pos ? min(hi, pos + a.window + 1) : hi;
  }
  return lo < hi ? make_int2(lo, hi) : make_int2(0, 0);
}

// ---- dropout draws: the finaliser of splitmix64 over a counter, as svc_dropout_rng_f32's, with the 64 bits of a word used as four
// 16-bit draws of four neighbouring keys: a word costs two 64-bit multiplications, more than the rest of a score's arithmetic, and
// a 16-bit threshold holds a drop rate to 2^-17 (the kept values are scaled by the rate it stands for, so that the mean is exact).
__device__ __forceinline__ unsigned long long draw_word(unsigned long long start, unsigned long long idx) {
  unsigned long long z = start + idx * 0xD1B54A32D192ED03ull;
  z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
  z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
  return z ^ (z >> 31);
}
__device__ __forceinline__ unsigned long long draw_start(const svc_attn_scored_t& a) {
  return (unsigned long long)a.seed[0] + (unsigned long long)((unsigned)a.site + 1u) * 0x9E3779B97F4A7C15ull;
}

// ---- operand types ----------------------------------------------------------------------------------------------------------------
template <typename E> __device__ __forceinline__ float to_f(E v) { return (float)v; }
template <typename E> struct Frag;          // right operand of one matrix step and of a whole head
template <> struct Frag<float> {
  template <int DP> struct Head { float v[DP / 2]; };
};
template <> struct Frag<bf16_t> {
  typedef bf16x8 V;
  template <int DP> struct Head { bf16x8 v[DP / 16]; };
};
template <> struct Frag<f16_t> {
  typedef f16x8 V;
  template <int DP> struct Head { f16x8 v[DP / 16]; };
};
// P enters a product multiplied by 2^PUP: fp16's numbers below 2^-14 lose bits, and a P of 2^-14 is an ordinary one in a long row.  256 times the
// largest P and the largest dropout factor (100) stay below 65504.
template <typename E> constexpr float PUP = __is_same(E, f16_t) ? 8.f : 0.f;
__device__ __forceinline__ f32x16 mfma(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mfma(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mfma(float a, float b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0); }

// The columns t0 .. t0+31 of X[d][t] as a right operand that reduces over d (lane: column, half: d's second half of a step).
template <typename E, int DP>
__device__ __forceinline__ void load_columns(typename Frag<E>::template Head<DP>& f, const E* x, long long cs, int dk, int t, int T, int h) {
  const bool ok = t >= 0 && t < T;
  if constexpr (sizeof(E) == 4) {
#pragma unroll
    for (int i = 0; i < DP / 2; ++i) {
      const int d = 2 * i + h;
      f.v[i] = ok && d < dk ? x[d * cs + t] : 0.f;
    }
  } else {
#pragma unroll
    for (int i = 0; i < DP / 16; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int d = 16 * i + 8 * h + e;
        f.v[i][e] = ok && d < dk ? x[d * cs + t] : (E)0.f;
      }
  }
}

// ---- staging: rows 0..DP-1 of X[d][p0 .. p0+N) into LDS rows of PITCH bytes; zero outside [beg, end) and behind row dk, so what
// lies there (unwritten cache, padding) never reaches a product.  Rows may start at any alignment of their type.
template <typename E>
__device__ __forceinline__ uint4 load_chunk(const E* row, int p, int beg, int end) {
  constexpr int V = Tile<E>::V;
  if (p >= beg && p + V <= end) {
    const U128 u = *(const U128*)(row + p);
    return make_uint4(u.x, u.y, u.z, u.w);
  }
  union { uint4 u; E e[V]; } r;
  r.u = make_uint4(0, 0, 0, 0);
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (p + i >= beg && p + i < end) r.e[i] = row[p + i];
  return r.u;
}
template <typename E, int DP>
__device__ __forceinline__ void stage(E* lds, const E* x, long long cs, int dk, int p0, int beg, int end, int tid) {
#pragma unroll
  for (int i = 0; i < DP * 8 / 256; ++i) {
    const int idx = tid + 256 * i, d = idx >> 3, c = idx & 7;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (d < dk) v = load_chunk<E>(x + d * cs, p0 + c * Tile<E>::V, beg, end);
    *(uint4*)((char*)lds + d * PITCH + c * 16) = v;
  }
}

// acc[row = position, column] += sum_d X[d][position] * f[d][column]: rows = positions 32 rt .. 32 rt + 31 of the staged tile
template <typename E, int DP>
__device__ __forceinline__ f32x16 mul_columns(const E* lds, int rt, const typename Frag<E>::template Head<DP>& f, f32x16 acc, int lane) {
  const int h = lane >> 5;
  if constexpr (sizeof(E) == 4) {
    const float* p = lds + h * Tile<E>::P + 32 * rt + swap23(lane & 31);
#pragma unroll
    for (int i = 0; i < DP / 2; ++i) acc = mfma(p[2 * i * Tile<E>::P], f.v[i], acc);
  } else {
    const int i16 = lane & 15, c = i16 & 3;
    const E* p = lds + (8 * h + (i16 >> 2)) * Tile<E>::P + 32 * rt + 16 * ((lane >> 4) & 1) + 4 * (((c & 1) << 1) | (c >> 1));
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) {
      typedef __attribute__((address_space(3))) s16x4 lds4;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(p + 16 * i * Tile<E>::P));
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(p + (16 * i + 4) * Tile<E>::P));
      const s16x8 v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
      acc = mfma(__builtin_bit_cast(typename Frag<E>::V, v), f.v[i], acc);
    }
  }
  return acc;
}

// out[d, column] += sum_position X[d][position] * w[position, column], w in accumulator layout (rows 32 rt .. of the tile).  16-bit types round w
// to the type; TWO: w goes in as two operands, its rounded value and the rounded rest (u^2 instead of u).
template <typename E, int DP, bool TWO = false>
__device__ __forceinline__ void mul_rows(f32x16 (&out)[DP / 32], const E* lds, int rt, const float (&w)[16], int lane) {
  const int h = lane >> 5;
  const E* p = lds + (lane & 31) * Tile<E>::P + 32 * rt + 8 * h;
  if constexpr (sizeof(E) == 4) {
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int dt = 0; dt < DP / 32; ++dt) {
        const f32x4 v = *(const f32x4*)(p + 32 * dt * Tile<E>::P + 16 * (q >> 1) + 4 * (q & 1));
#pragma unroll
        for (int j = 0; j < 4; ++j) out[dt] = mfma(v[j], w[4 * q + j], out[dt]);
      }
  } else {
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      typename Frag<E>::V b, rest;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        b[e] = (E)w[8 * ks + e];
        if constexpr (TWO) rest[e] = (E)(w[8 * ks + e] - (float)b[e]);
      }
#pragma unroll
      for (int dt = 0; dt < DP / 32; ++dt) {
        const typename Frag<E>::V v = *(const typename Frag<E>::V*)(p + 32 * dt * Tile<E>::P + 16 * ks);
        out[dt] = mfma(v, b, out[dt]);
        if constexpr (TWO) out[dt] = mfma(v, rest, out[dt]);
      }
    }
  }
}

// ---- scores in units of log 2: u = cap * tanh(scale q.k / cap) or scale q.k, times log2(e), plus the (already scaled) bias --------
struct ScoreScale {
  float mul, cap_in, cap_out;      // mul: no cap; else tanh(acc * cap_in) * cap_out
};
__device__ __forceinline__ ScoreScale score_scale(const svc_attn_scored_t& a) {
  ScoreScale s;
  s.mul = a.scale * LOG2E;
  s.cap_in = a.softcap > 0.f ? a.scale / a.softcap : 0.f;
  s.cap_out = a.softcap * LOG2E;
  return s;
}

// The distance bias of a tile: win[j] = table[clamp(d0 + j, -W, W) + W] * log2(e) for j in [0, n): the tile's distances are
// consecutive, so the table's clamped entries become one short row in LDS and a lookup an offset from a lane's own base.
__device__ __forceinline__ void stage_bias(float* win, const float* table, int W, int d0, int n, int tid) {
  for (int j = tid; j < n; j += 256) win[j] = table[min(max(d0 + j, -W), W) + W] * LOG2E;
}

__device__ __forceinline__ int wave_min(int v) {
  for (int o = 32; o > 0; o >>= 1) v = min(v, __shfl_xor(v, o));
  return v;
}
__device__ __forceinline__ int wave_max(int v) {
  for (int o = 32; o > 0; o >>= 1) v = max(v, __shfl_xor(v, o));
  return v;
}

int check_args(const svc_attn_scored_t* a, bool backward);      // attn_scored_fwd.hip

}  // namespace attn
