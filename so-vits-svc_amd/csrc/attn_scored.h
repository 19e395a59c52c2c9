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

// fp32 on the bf16 matrix instruction: a value is the sum of three bf16 numbers (8 + 8 + 8 bits: all of its 24, at fp32's own range), and a product the six
// largest of their nine products, each exact in the instruction's fp32 accumulator; what is left out is 2^-24 of the product.  Six instructions for 16
// channels take 192 cycles where the fp32 instruction's eight take 512.  x3_t is fp32 in memory and three planes of bf16 in LDS and registers.
struct x3_t {
  float v;
  __device__ __forceinline__ explicit x3_t(float f) : v(f) {}
  x3_t() = default;
  __device__ __forceinline__ explicit operator float() const { return v; }
};
template <typename E> constexpr bool X3 = __is_same(E, x3_t);
constexpr int X3_PITCH = 80;            // bytes of a plane's row of 32 positions: 64 + 16
// Two values rounded to bf16 in one word, and what the rounding left of them.  (One value at a time the compiler converts each twice, once for its word.)
__device__ __forceinline__ unsigned pack2(float x, float y) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  typedef __bf16 b2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(unsigned, __builtin_convertvector((f2){x, y}, b2));
}
__device__ __forceinline__ void rest2(float& x, float& y, unsigned u) {
  x -= __builtin_bit_cast(float, u << 16);
  y -= __builtin_bit_cast(float, u & 0xffff0000u);
}
// Two values' parts; `big` collects the largest magnitude.  Where that passes bf16's own (an infinity, or a number that rounds to one) the caller has the parts
// made by split3_large: a test a tile, where a test a value took two instructions of ten.  (nan: all three parts are nan.)
constexpr float BF16_TOP = 0x1.fep127f;
__device__ __forceinline__ void split3(float x, float y, unsigned& a, unsigned& b, unsigned& c, float& big) {
  big = fmaxf(fmaxf(fabsf(x), fabsf(y)), big);
  a = pack2(x, y);
  rest2(x, y, a);
  b = pack2(x, y);
  rest2(x, y, b);
  c = pack2(x, y);
}
// An infinity is 1, 0 and, as its third part, itself with its sign: of the six products only the one with the other operand's first part meets it, so an
// infinite operand gives an infinity of the right sign (as a first part it would meet the other's smaller parts, which are of either sign or 0: nan).  A number that
// would round to infinity is cut to its first part instead.
__device__ __forceinline__ void split3_large(float x, float y, unsigned& a, unsigned& b, unsigned& c) {
  a = pack2(x, y);
  unsigned top[2], third[2];
  float v[2] = {x, y};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const unsigned u = __builtin_bit_cast(unsigned, v[i]);
    const bool inf = (u & 0x7fffffffu) == 0x7f800000u;
    top[i] = inf ? (u >> 16 & 0x8000u) | 0x3f80u : fabsf(v[i]) > BF16_TOP ? u >> 16 : a >> 16 * i & 0xffffu;
    third[i] = inf ? u >> 16 : 0u;
    v[i] = inf ? 0.f : v[i] - __builtin_bit_cast(float, top[i] << 16);
  }
  a = top[0] | top[1] << 16;
  b = pack2(v[0], v[1]);
  rest2(v[0], v[1], b);
  c = pack2(v[0], v[1]) | third[0] | third[1] << 16;
}

// A staged tile: rows of RB bytes of positions.  128-byte rows (64 positions of a 16-bit type, 32 of fp32); 64-byte rows for the backward at 128
// channels in 16 bits, whose accumulators leave no registers for a longer tile's loads.  fp32's rows have 16 bytes more, which spreads their reads over the
// banks.  16-bit types' rows are not padded: chunk c (16 bytes) of row d lies at c ^ turn(d), so that the four rows x 64 bytes of a transposing
// read, and the sixteen rows x 16 bytes of an ordinary one, each fall on all 64 banks once (rows padded by 16 bytes: 6 to 17 % of the cycles in conflicts,
// dq at 128 channels 575 us for 560).
template <typename E, int RB = 128, int TH = 256> struct Tile {
  static constexpr int N = RB / (int)sizeof(E);
  static constexpr int RT = N / 32;     // 32-row accumulators a tile feeds
  static constexpr int PITCH = RB + (sizeof(E) == 2 ? 0 : 16);
  static constexpr int P = PITCH / (int)sizeof(E);
  static constexpr int V = 16 / (int)sizeof(E);     // positions of a 16-byte chunk
  static constexpr int CH = RB / 16;                // chunks (lanes) of a row
  static constexpr int RS = TH / CH;                // rows that TH threads stage in one step
};

template <int RB> __device__ __forceinline__ int turn(int d) { return RB == 128 ? (d & 2) << 1 | (d >> 2 & 3) : d >> 2 & 3; }

template <typename E, int DP, int RB = 128> struct Staged {
  static constexpr int SIZE = X3<E> ? 3 * DP * X3_PITCH / 4 : DP * Tile<E, RB>::P;     // elements of E from one staged matrix to the next
  static constexpr int BUFS = X3<E> ? 1 : 2;          // three planes leave no room for a second buffer beside a second workgroup's
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
    start = d[n];                       // (before the key axis, in a cache whose oldest positions were dropped: a prefix counts from there)
    lo = max(start, 0);
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
constexpr unsigned long long DRAW_STEP = 0xD1B54A32D192ED03ull;      // from one counter to the next
__device__ __forceinline__ unsigned long long draw_word(unsigned long long z) {      // z = start + counter * DRAW_STEP
  z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
  z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
  return z ^ (z >> 31);
}
// The counters of a 32 x 32 block are a lane's first one (its row, and 2 h for its half's eight keys) plus what is the same for all lanes: 64-bit
// multiplications, quarter rate three times over, are left to the scalar unit.
__device__ __forceinline__ unsigned long long draw_block(int s) { return (unsigned long long)(s >> 2) * DRAW_STEP; }
__device__ __forceinline__ constexpr unsigned long long draw_group(int w) { return (unsigned long long)(4 * (w >> 1) + (w & 1)) * DRAW_STEP; }
// draw j of a word falls under the threshold (the odd fields compare in place, the even ones shifted up)
__device__ __forceinline__ bool dropped(unsigned long long z, int j, unsigned thr) {
  const unsigned w = (unsigned)(z >> (32 * (j >> 1)));
  return (j & 1 ? w : w << 16) < thr << 16;
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
template <> struct Frag<x3_t> {
  typedef bf16x8 V;
  template <int DP> struct Head { bf16x8 v[3][DP / 16]; };
};
__device__ __forceinline__ f32x16 mfma(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mfma(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mfma(float a, float b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0); }
// the six products: the first parts' own sum, and the five small ones', which would lose their last bits in the large one step by step
__device__ __forceinline__ void mfma6(const bf16x8 (&a)[3], bf16x8 b0, bf16x8 b1, bf16x8 b2, f32x16& large, f32x16& small) {
  small = mfma(a[1], b1, small);
  large = mfma(a[0], b0, large);
  small = mfma(a[2], b0, small);
  small = mfma(a[0], b2, small);
  small = mfma(a[1], b0, small);
  small = mfma(a[0], b1, small);
}

// ---- staging: rows 0..DP-1 of X[d][p0 .. p0+N) into LDS rows of PITCH bytes, zero outside [beg, end) and behind row dk, so what lies there (unwritten
// cache, padding) never reaches a product.  Rows may start at any alignment of their type.  In two halves, so that a tile's loads are in flight
// while the one before is worked on: `fetch` into registers, `commit` to LDS.  By a workgroup of TH = 256 threads, or a wave by itself.
template <typename E, int DP, int RB = 128, int TH = 256> struct Pre { uint4 v[DP / Tile<E, RB, TH>::RS]; };

template <typename E, int DP, int RB = 128, int TH = 256>
struct Source {                         // one head's matrix as this thread sees it
  static constexpr int CH = Tile<E, RB, TH>::CH, RS = Tile<E, RB, TH>::RS, S = DP / RS, V = Tile<E, RB>::V;
  static constexpr int TAIL = RS < 32 ? 32 / RS : 1;      // dk > DP - 32: the steps whose rows may lie behind dk (the last row stands for them, read and not used)
  static_assert(TAIL <= S, "");
  const E *row, *tail[TAIL];            // its rows of step 0 and of the last steps
  long long step;                       // elements between steps
  int T;                                // positions that exist
  int pad;                              // bit j: its row of the j-th of the last steps lies behind dk
  __device__ __forceinline__ void set(const E* x, long long cs, int dk, int T_, int tid) {
    const int d = tid / CH;
    row = x + (long long)min(d, dk - 1) * cs;
    step = RS * cs;
    T = T_;
    pad = 0;
#pragma unroll
    for (int j = 0; j < TAIL; ++j) {
      const int dl = d + (S - TAIL + j) * RS;
      tail[j] = x + (long long)min(dl, dk - 1) * cs;
      pad |= dl >= dk ? 1 << j : 0;
    }
  }
  __device__ __forceinline__ const E* at(int i) const { return i >= S - TAIL ? tail[i - (S - TAIL)] : row + i * step; }
  // Sixteen bytes a step, from the chunk's place or, at the row's end, from the last place that has sixteen: no branch, because a branch around loads makes
  // the compiler wait for them where its sides meet again.  (Rows of fewer than sixteen bytes are read by `commit`.)
  __device__ __forceinline__ void fetch(Pre<E, DP, RB, TH>& f, int p0, int tid) const {
    if (T < V) return;
    const int p = min(p0 + (tid & (CH - 1)) * V, T - V);
#pragma unroll
    for (int i = 0; i < S; ++i) {
      const U128 u = *(const U128*)(at(i) + p);
      f.v[i] = make_uint4(u.x, u.y, u.z, u.w);
    }
  }
  __device__ __forceinline__ void commit(E* lds, Pre<E, DP, RB, TH>& f, int p0, int beg, int end, int tid) const {
    const int p = p0 + (tid & (CH - 1)) * V;
    if (p0 + Tile<E, RB>::N > T) {          // the chunk may have been read from further left: shift it to its place
      if (T < V) {
#pragma unroll
        for (int i = 0; i < S; ++i) {
          union { uint4 u; E e[V]; } x;
          x.u = make_uint4(0, 0, 0, 0);
          const E* r = at(i);
#pragma unroll
          for (int e = 0; e < V; ++e)
            if (p + e < T) x.e[e] = r[p + e];
          f.v[i] = x.u;
        }
      } else {
        const int by = min(max(p - (T - V), 0), V) * (int)sizeof(E) * 8;
#pragma unroll
        for (int i = 0; i < S; ++i) {
          union { uint4 u; unsigned __int128 q; } x;
          x.u = f.v[i];
          x.q = by < 128 ? x.q >> by : 0;
          f.v[i] = x.u;
        }
      }
    }
    if (p0 < beg || p0 + Tile<E, RB>::N > end) {
      unsigned k[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (sizeof(E) == 4) k[j] = p + j >= beg && p + j < end ? ~0u : 0u;
        else k[j] = (p + 2 * j >= beg && p + 2 * j < end ? 0xffffu : 0u) | (p + 2 * j + 1 >= beg && p + 2 * j + 1 < end ? 0xffff0000u : 0u);
      }
#pragma unroll
      for (int i = 0; i < S; ++i) f.v[i] = make_uint4(f.v[i].x & k[0], f.v[i].y & k[1], f.v[i].z & k[2], f.v[i].w & k[3]);
    }
    if (pad) {
#pragma unroll
      for (int j = 0; j < TAIL; ++j)
        if (TAIL == 1 || pad >> j & 1) f.v[S - TAIL + j] = make_uint4(0, 0, 0, 0);
    }
    if constexpr (X3<E>) {
      static_assert(RB == 128, "32 positions");
      float big = 0.f;
      auto put = [&](int i, uint2 u, uint2 v, uint2 w) {
        char* o = (char*)lds + (tid / CH + i * RS) * X3_PITCH + (tid & (CH - 1)) * 8;
        *(uint2*)o = u;
        *(uint2*)(o + DP * X3_PITCH) = v;
        *(uint2*)(o + 2 * DP * X3_PITCH) = w;
      };
#pragma unroll
      for (int i = 0; i < S; ++i) {
        const f32x4 x = __builtin_bit_cast(f32x4, f.v[i]);
        uint2 u, v, w;
        split3(x[0], x[1], u.x, v.x, w.x, big);
        split3(x[2], x[3], u.y, v.y, w.y, big);
        put(i, u, v, w);
      }
      if (__any(big > BF16_TOP)) {
#pragma unroll
        for (int i = 0; i < S; ++i) {
          const f32x4 x = __builtin_bit_cast(f32x4, f.v[i]);
          uint2 u, v, w;
          split3_large(x[0], x[1], u.x, v.x, w.x);
          split3_large(x[2], x[3], u.y, v.y, w.y);
          put(i, u, v, w);
        }
      }
      return;
    }
    constexpr int PITCH = Tile<E, RB>::PITCH;
    // (a step is a multiple of 16 rows, or fp32's: the turn is the same in all)
    static_assert(sizeof(E) == 4 || RS % 16 == 0, "");
    const int d0 = tid / CH, chunk = tid & (CH - 1);
    char* o = (char*)lds + d0 * PITCH + (sizeof(E) == 2 ? chunk ^ turn<RB>(d0) : chunk) * 16;
#pragma unroll
    for (int i = 0; i < S; ++i) *(uint4*)(o + i * RS * PITCH) = f.v[i];
  }
};

// Four rows (d) of 16 columns each, transposed: lane i of 16 gets column i's four values; and the four rows behind them.
template <typename E> __device__ __forceinline__ typename Frag<E>::V read_transposed(const void* p, const void* p4) {
  typedef __attribute__((address_space(3))) s16x4 lds4;
  const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)p);
  const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)p4);
  return __builtin_bit_cast(typename Frag<E>::V, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}
// byte of (row d, column c) in a 16-bit type's tile
template <int RB> __device__ __forceinline__ int byte_of(int d, int c) { return d * RB + ((c >> 3 ^ turn<RB>(d)) << 4) + (c & 7) * 2; }

// Columns 32 sub .. 32 sub + 31 of a staged tile as a right operand that reduces over d.
template <typename E, int DP, int RB = 128>
__device__ __forceinline__ void read_columns(typename Frag<E>::template Head<DP>& f, const E* lds, int sub, int lane) {
  const int h = lane >> 5, i16 = lane & 15;
  if constexpr (X3<E>) {
    const char* p = (const char*)lds + (8 * h + (i16 >> 2)) * X3_PITCH + 2 * (32 * sub + 16 * ((lane >> 4) & 1) + 4 * (i16 & 3));
#pragma unroll
    for (int k = 0; k < 3; ++k)
#pragma unroll
      for (int i = 0; i < DP / 16; ++i) f.v[k][i] = read_transposed<E>(p + (k * DP + 16 * i) * X3_PITCH, p + (k * DP + 16 * i + 4) * X3_PITCH);
  } else if constexpr (sizeof(E) == 4) {
    const float* p = lds + h * Tile<E, RB>::P + 32 * sub + (lane & 31);
#pragma unroll
    for (int i = 0; i < DP / 2; ++i) f.v[i] = p[2 * i * Tile<E, RB>::P];
  } else {
    const int d = 8 * h + (i16 >> 2), c = 32 * sub + 16 * ((lane >> 4) & 1) + 4 * (i16 & 3);
    const char *p = (const char*)lds + byte_of<RB>(d, c), *p4 = (const char*)lds + byte_of<RB>(d + 4, c);
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) f.v[i] = read_transposed<E>(p + 16 * i * RB, p4 + 16 * i * RB);
  }
}

// A workgroup's 128 columns of X as right operands, through the LDS of its tiles, as many at a time as there are.  In two halves, so that a kernel asks
// for all its columns and its first tile before it waits for any.  [beg, end): columns that are used.
template <typename E, int DP, int RB = 128> struct Columns {
  static constexpr int N = Tile<E, RB>::N, ALL = NCOL / N, ONCE = 2 * Staged<E, DP, RB>::BUFS < ALL ? 2 * Staged<E, DP, RB>::BUFS : ALL;
  Source<E, DP, RB> src;
  Pre<E, DP, RB> pre[ALL];
  __device__ __forceinline__ void fetch(const E* x, long long cs, int dk, int T, int t0, int tid) {
    src.set(x, cs, dk, T, tid);
#pragma unroll
    for (int i = 0; i < ALL; ++i) src.fetch(pre[i], t0 + i * N, tid);
  }
  __device__ __forceinline__ void settle(typename Frag<E>::template Head<DP>& f, E* lds, int t0, int beg, int end, int tid) {
    const int col = (tid >> 6) * 32;
#pragma unroll
    for (int at = 0; at < ALL; at += ONCE) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < ONCE; ++i) src.commit(lds + i * Staged<E, DP, RB>::SIZE, pre[at + i], t0 + (at + i) * N, beg, end, tid);
      __syncthreads();
      if (ONCE == ALL || (col / N >= at && col / N < at + ONCE))
        read_columns<E, DP, RB>(f, lds + (col / N - at) * Staged<E, DP, RB>::SIZE, col % N / 32, tid & 63);
    }
  }
};

// -> [row = position, column]: sum_d X[d][position] * f[d][column]: rows = positions 32 rt .. 32 rt + 31 of the staged tile
template <typename E, int DP, int RB = 128>
__device__ __forceinline__ f32x16 mul_columns(const E* lds, int rt, const typename Frag<E>::template Head<DP>& f, int lane) {
  const int h = lane >> 5, i16 = lane & 15, c4 = 4 * (((i16 & 1) << 1) | ((i16 >> 1) & 1));
  f32x16 acc;
#pragma unroll
  for (int r = 0; r < 16; ++r) acc[r] = 0.f;
  if constexpr (X3<E>) {
    const char* p = (const char*)lds + (8 * h + (i16 >> 2)) * X3_PITCH + 2 * (32 * rt + 16 * ((lane >> 4) & 1) + c4);
    f32x16 other = acc;
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) {
      bf16x8 x[3];
#pragma unroll
      for (int k = 0; k < 3; ++k) x[k] = read_transposed<E>(p + (k * DP + 16 * i) * X3_PITCH, p + (k * DP + 16 * i + 4) * X3_PITCH);
      mfma6(x, f.v[0][i], f.v[1][i], f.v[2][i], acc, other);
      if (i & 1) __builtin_amdgcn_sched_barrier(0);
    }
    acc = acc + other;
  } else if constexpr (sizeof(E) == 4) {
    // two sums of half the channels each: a chain's rounding errors grow with its length and with the sums it passes through
    const float* p = lds + h * Tile<E, RB>::P + 32 * rt + swap23(lane & 31);
    f32x16 other = acc;
#pragma unroll
    for (int i = 0; i < DP / 4; ++i) {
      acc = mfma(p[2 * i * Tile<E, RB>::P], f.v[i], acc);
      other = mfma(p[2 * (i + DP / 4) * Tile<E, RB>::P], f.v[i + DP / 4], other);
    }
    acc = acc + other;
  } else {
    // (columns 32 rt further are the byte's bit 6, the four rows behind are bit 4 and 4 rows: worked out here, from one register that stays)
    int at = byte_of<RB>(8 * h + (i16 >> 2), 16 * ((lane >> 4) & 1) + c4);
    asm volatile("" : "+v"(at));
    at ^= 64 * rt;
    const char *p = (const char*)lds + at, *p4 = (const char*)lds + (at ^ 16) + 4 * RB;
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) {
      acc = mfma(read_transposed<E>(p + 16 * i * RB, p4 + 16 * i * RB), f.v[i], acc);
      if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);
    }
  }
  return acc;
}

// out[d, column] += sum_position X[d][position] * w[position, column], w in accumulator layout (rows 32 rt .. of the tile).  16-bit types round w
// to the type; OPS > 1: w goes in as that many operands, its rounded value, the rounded rest, and the rest of that.
template <typename E, int DP, int OPS = 1, int RB = 128>
__device__ __forceinline__ void mul_rows(f32x16 (&out)[DP / 32], const E* lds, int rt, const float (&w)[16], int lane) {
  const int h = lane >> 5;
  const E* p = lds + (lane & 31) * Tile<E, RB>::P + 32 * rt + 8 * h;
  if constexpr (X3<E>) {
    const char* q = (const char*)lds + (lane & 31) * X3_PITCH + 2 * (32 * rt + 8 * h);
    union { unsigned u[4]; bf16x8 v; } b[2][3];
    float big = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) split3(w[2 * e], w[2 * e + 1], b[e >> 2][0].u[e & 3], b[e >> 2][1].u[e & 3], b[e >> 2][2].u[e & 3], big);
    if (__any(big > BF16_TOP)) {
#pragma unroll
      for (int e = 0; e < 8; ++e) split3_large(w[2 * e], w[2 * e + 1], b[e >> 2][0].u[e & 3], b[e >> 2][1].u[e & 3], b[e >> 2][2].u[e & 3]);
    }
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt) {
      f32x16 small;
#pragma unroll
      for (int r = 0; r < 16; ++r) small[r] = 0.f;
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        bf16x8 x[3];
#pragma unroll
        for (int k = 0; k < 3; ++k) x[k] = *(const bf16x8*)(q + (k * DP + 32 * dt) * X3_PITCH + 32 * ks);
        mfma6(x, b[ks][0].v, b[ks][1].v, b[ks][2].v, out[dt], small);
      }
      out[dt] += small;
      __builtin_amdgcn_sched_barrier(0);
    }
  } else if constexpr (sizeof(E) == 4) {
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int dt = 0; dt < DP / 32; ++dt) {
        const f32x4 v = *(const f32x4*)(p + 32 * dt * Tile<E, RB>::P + 16 * (q >> 1) + 4 * (q & 1));
#pragma unroll
        for (int j = 0; j < 4; ++j) out[dt] = mfma(v[j], w[4 * q + j], out[dt]);
      }
  } else {
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      int at = byte_of<RB>(lane & 31, 8 * h);
      asm volatile("" : "+v"(at));
      const char* const row = (const char*)lds + (at ^ (64 * rt + 32 * ks));
      union { unsigned u[4]; typename Frag<E>::V v; } b[OPS];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float x = w[8 * ks + 2 * e], y = w[8 * ks + 2 * e + 1];
#pragma unroll
        for (int o = 0; o < OPS; ++o) {
          if constexpr (__is_same(E, bf16_t)) {
            b[o].u[e] = pack2(x, y);
            if (o + 1 < OPS) rest2(x, y, b[o].u[e]);
          } else {
            b[o].v[2 * e] = (E)x;
            b[o].v[2 * e + 1] = (E)y;
            x -= (float)b[o].v[2 * e];
            y -= (float)b[o].v[2 * e + 1];
          }
        }
      }
#pragma unroll
      for (int dt = 0; dt < DP / 32; ++dt) {
        const typename Frag<E>::V v = *(const typename Frag<E>::V*)(row + 32 * dt * RB);
#pragma unroll
        for (int o = 0; o < OPS; ++o) out[dt] = mfma(v, b[o].v, out[dt]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
}

// What a forward is for.  0: its output alone; P is rounded to the type once.  1: a 16-bit training pass (out32): the backward's row sums of dO out
// carry P's rounding into every dS, so P goes in as two operands (bf16, 4096 x 4096 causal at 128 channels: dq 2.35e-3 from the exact one instead of
// 2.5e-3, where rounding dq and dS alone leaves 2.3e-3).  2: fp32, or a 16-bit pass whose dbias, an fp32 result, will be wanted: as many operands as 24
// bits take, the library's tanh; and caps above SHORT_CAP, for the tanh.
template <typename E, int MODE> constexpr int P_OPS = sizeof(E) == 4 || MODE == 0 ? 1 : MODE == 1 || __is_same(E, f16_t) ? 2 : 3;

// ---- scores in units of log 2 ------------------------------------------------------------------------------------------------------------
struct ScoreScale {
  float mul, cap_in, cap_exp, cap_out;      // no cap: u * mul; else tanh(u * cap_in) * cap_out; cap_exp = 2 log2(e) cap_in
  bool cap;
};
__device__ __forceinline__ ScoreScale score_scale(const svc_attn_scored_t& a) {
  ScoreScale s;
  s.cap = a.softcap > 0.f;
  s.mul = a.scale * LOG2E;
  s.cap_in = s.cap ? a.scale / a.softcap : 0.f;
  s.cap_exp = s.cap_in * (2.f * LOG2E);
  s.cap_out = a.softcap * LOG2E;
  return s;
}
// tanh for the cap.  EXACT (fp32, and where a fp32 gradient of the bias hangs on it): the library's.  Else 1 - 2 / (exp 2x + 1), two
// transcendental instructions: 1.5e-7 absolute, so 1.5e-7 of the cap in a score, whose P and result are rounded to 2^-8 or 2^-11.  At a cap of 256 that is
// an eighth of the smaller rounding; above it (SHORT_CAP) 16-bit types take the library's too (4 x 16 heads of 128, 2049 causal, bf16: 137 us for 205, a training
// pass 952 us for 1132; at a cap of 2^20 the short form would be off by 0.15).
constexpr float SHORT_CAP = 256.f;
template <bool EXACT> __device__ __forceinline__ float cap_tanh(float u, const ScoreScale& sc) {
  if (EXACT) return tanhf(u * sc.cap_in);
  return fmaf(-2.f, __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(u * sc.cap_exp) + 1.f), 1.f);
}
// cap * tanh(u / cap) * log2(e)
template <bool EXACT> __device__ __forceinline__ float capped(float u, const ScoreScale& sc) {
  if (EXACT) return cap_tanh<true>(u, sc) * sc.cap_out;
  return fmaf(-2.f * sc.cap_out, __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(u * sc.cap_exp) + 1.f), sc.cap_out);
}

// The distance bias of a tile: win[j] = table[clamp(d0 + j, -W, W) + W] * log2(e) for j in [0, n), n <= 256: the tile's distances are consecutive, so the
// table's clamped entries become one short row in LDS and a lookup an offset from a lane's own base.  Thread j fetches and commits entry j
// (times log2(e) when it commits: arithmetic on a fetched value would wait for it).
__device__ __forceinline__ float bias_entry(const float* table, int W, int d0, int j) { return table[min(max(d0 + j, -W), W) + W]; }

// An entry of fp16's lowest value or below masks its distance: against any other score its exponential is 0, and a row of nothing else, whose scores such
// an entry would absorb, counts as one without keys.
__device__ __forceinline__ float bias_scaled(float v) { return v <= -65504.f ? -INFINITY : v * LOG2E; }

// ---- which (item, head, tile) a workgroup works on.  Tiles from the heaviest on (the last, under a causal mask), all heads of one tile index before the
// next; where the key heads divide by the 8 XCDs (or there are so many that it hardly matters), a key head's workgroups share one XCD and its L2 (8 items of 12
// query and 4 key heads, 64 channels, 1501 positions: forward 61 -> 58 us, dq 101 -> 95; 4 items of 4096 positions at 128 channels 1-2 % each).
struct Place { int group, sub, tile; };           // group = item * G + key head; sub: query head of the group
__host__ __device__ __forceinline__ bool by_xcd(int groups) { return groups % 8 == 0 || groups >= 64; }
__device__ __forceinline__ Place place_of(int id, int groups, int rep, int n_tiles) {
  Place p;
  if (by_xcd(groups)) {
    const int per = (groups + 7) / 8 * rep, j = id >> 3, r = j % per;
    p.tile = n_tiles - 1 - j / per;
    p.group = r / rep * 8 + (id & 7);
    p.sub = r % rep;
  } else {
    const int r = id % (groups * rep);
    p.tile = n_tiles - 1 - id / (groups * rep);
    p.group = r / rep;
    p.sub = r % rep;
  }
  return p;
}
// ---- few queries: columns are (query head of the group, query) pairs, 32 a workgroup, and the keys are split -------------------------------------
struct Split {
  int cols, blocks, parts;             // columns of a key head, their workgroups of 32, parts of the keys; parts = 0: fwd_kernel's way
};
Split split_of(const svc_attn_scored_t& a);
void launch_split(const svc_attn_scored_t& a, const Split& p, hipStream_t s);       // attn_scored_split.hip
long long split_ws_bytes(const svc_attn_scored_t& a, const Split& p);

static inline long long grid_of(long long groups, long long rep, long long n_tiles) {
  return (by_xcd((int)groups) ? (groups + 7) / 8 * 8 : groups) * rep * n_tiles;
}

// The wave's smallest / largest, by lane exchanges inside the vector unit (an exchange through LDS takes some hundred cycles, and these stand in front of
// everything else).
template <int CTRL> __device__ __forceinline__ int lane_of(int v) { return __builtin_amdgcn_update_dpp(v, v, CTRL, 0xf, 0xf, false); }
__device__ __forceinline__ int wave_max(int v) {
  v = max(v, lane_of<0x111>(v));      // row_shr 1, 2, 4, 8: lane 15 of each row of 16 has the row's
  v = max(v, lane_of<0x112>(v));
  v = max(v, lane_of<0x114>(v));
  v = max(v, lane_of<0x118>(v));
  return max(max(__builtin_amdgcn_readlane(v, 15), __builtin_amdgcn_readlane(v, 31)), max(__builtin_amdgcn_readlane(v, 47), __builtin_amdgcn_readlane(v, 63)));
}
__device__ __forceinline__ int wave_min(int v) { return -wave_max(-v); }      // (values are positions: never the lowest int)

int check_sizes(const svc_attn_scored_t* a);                    // attn_scored_fwd.hip
int check_args(const svc_attn_scored_t* a, bool backward);

// ---- the backward's workspace -----------------------------------------------------------------------------------------------------------
struct Ws {
  float* rowsum;   // [B*H][Tq]  D = sum_d dO out
  int2* iv;        // [B][Tq]    visible keys
  int4* tiles;     // [B][ceil(Tq/32)]  {min lo, max hi, max lo, min hi} of 32 queries
  float* gmax;     // [B*H][ceil(Tq/64)]  max |dO|
  float* vmax;     // [B*G][ceil(Tk/128)]  max |v| of the keys that can be seen (fp16)
  float* bins;     // [B*H][ceil(Tq/32)][2 bias_w + 1]  bias gradient of 32 queries
  long long bytes;
};
// Queries of item b that can see a key at all, and keys that can be seen (by the lengths and the outer document boundaries).
__device__ __forceinline__ void live_range(const svc_attn_scored_t& a, int b, int& tbeg, int& tend, int& kbeg, int& kend) {
  const int len = item_length(a, b), o = min(max(item_offset(a, b), -a.Tq), a.Tk);
  tbeg = max(0, -o);
  tend = max(0, min(a.Tq, len - o));
  kbeg = 0;
  kend = len;
  if (a.n_docs) {
    const int* d = a.docs + (long long)b * (a.n_docs + 1);
    kbeg = max(0, d[0]);
    kend = max(0, min(len, d[a.n_docs]));
    tbeg = max(tbeg, kbeg - o);
    tend = min(tend, kend - o);
  }
}
void launch_dq(const svc_attn_scored_t& a, const Ws& w, hipStream_t s);        // attn_scored_dq.hip
void launch_dkv(const svc_attn_scored_t& a, const Ws& w, hipStream_t s);       // attn_scored_dkv.hip

// fp16 operands: dS is multiplied by a power of two that brings the largest |dO| of the key head to [1, 2): gradients of any magnitude then
// sit in the middle of the type's range (a loss scale of 2^-12 would otherwise leave dS among its subnormals).  |dS| = P |Z dP - D| is at most `most` = 2 keep dk
// max |dO| max |v|: where that would pass 65504 (max |v| above 128 at 128 channels), the power is the largest that keeps it below.  The factor is divided out of the
// fp32 accumulators.  red: 8 floats.
template <typename E> __device__ __forceinline__ float operand_scale(const svc_attn_scored_t& a, const Ws& w, int b, int kvh, float* red) {
  if constexpr (!__is_same(E, f16_t)) return 1.f;
  const int n_tiles = (a.Tq + 63) / 64, rep = a.H / a.G, n = rep * n_tiles, nk = (a.Tk + 127) / 128;
  const float* g = w.gmax + ((long long)b * a.H + (long long)kvh * rep) * n_tiles;
  const float* gv = w.vmax + ((long long)b * a.G + kvh) * nk;
  float m = 0.f, v = 0.f;
  for (int i = threadIdx.x; i < n; i += 256) m = fmaxf(m, g[i]);
  for (int i = threadIdx.x; i < nk; i += 256) v = fmaxf(v, gv[i]);
  for (int o = 32; o > 0; o >>= 1) {
    m = fmaxf(m, __shfl_xor(m, o));
    v = fmaxf(v, __shfl_xor(v, o));
  }
  if ((threadIdx.x & 63) == 0) {
    red[threadIdx.x >> 6] = m;
    red[4 + (threadIdx.x >> 6)] = v;
  }
  __syncthreads();
  m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  v = fmaxf(fmaxf(red[4], red[5]), fmaxf(red[6], red[7]));
  if (!(m > 0.f) || !(m < INFINITY)) return 1.f;
  int e;
  frexpf(m, &e);
  const float f = ldexpf(1.f, 1 - e), keep = a.seed ? 65536.f / (65536.f - rintf(a.p_drop * 65536.f)) : 1.f, most = 2.f * keep * a.dk * m * v;
  if (!(most * f > 65504.f) || !(most < INFINITY)) return f;
  frexpf(65504.f / most, &e);
  return ldexpf(1.f, e - 1);
}

}  // namespace attn
