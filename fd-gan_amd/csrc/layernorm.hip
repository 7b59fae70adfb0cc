// layernorm.hip -- layer norm over the channels of a row, forward and backward, with the reduction of the weight's gradient.
//
//   forward    m = sum x / C,  s = 1 / sqrt(sum (x - m)^2 / C + eps),  y = (x - m) s w + b
//   backward   h = (x - m) s,  g = dy w,  c1 = sum g / C,  c2 = sum g h / C
//              dx = s (g - c1 - h c2),   dw = sum over rows of dy h,   db = sum over rows of dy
//
// A row is a pixel of an NHWC view (C channels, next to each other; the rows may lie at a pitch wider than C, a channel slice of a
// concatenation) or a row of a matrix.  Sums are in fp32; the variance is formed around the mean (or around a value some roundings beside it, and
// what that adds is taken off: mend_mean), never as a difference of the squares of x.
//
// All of it is bound by memory: 2 C or 3 C values a row against some 10 to 20 operations a value.  So each value is read once:
//  * held rows (ln_fwd_rows, ln_bwd_rows): a row stays in the registers of a group of T lanes, NV vectors of 16 bytes each.  T is a power of
//    two from 1 (three channels: every lane its own row) to 1024; the lanes join their sums by shuffles, waves through LDS.
//  * split rows (ln_fwd_part / _apply, ln_bwd_part / _apply): rows too long for that are cut over many workgroups, whose parts are joined by the
//    pass that applies them.
// The weight's gradient is a sum down the columns, across the rows of every workgroup: each workgroup keeps the sums of its rows in registers,
// writes them once, and ln_bwd_join adds the workgroups' in a fixed order.  No atomics: every result is the same bits every time.
#include "common.h"
#include <limits.h>

namespace {

struct LnFwdArgs {
  const void* x;
  void* y;
  const void *gamma, *beta;
  float *mean, *rstd;
  float* part;                 // split rows: [row][piece]{mean, sum of squares around it}
  long long rows, px, py;
  int c, wdt;
  int piece, pieces;           // split rows: elements of a piece, pieces of a row
  float eps, inv_c;
};

struct LnBwdArgs {
  const void *x, *dy;
  void* dx;
  const void* gamma;
  const float *mean, *rstd;
  float* part;                 // split rows: [row][piece]{sum g, sum g h}
  float* wpart;                // [workgroup]{dw, db}[stride]; null: the weight's gradient is not wanted
  long long rows, px, pdy, pdx;
  int c, wdt, stride;
  int piece, pieces, slab;     // split rows; slab: rows of a workgroup of the applying pass
  float inv_c;
};

struct LnJoinArgs {
  const float* wpart;
  void *dgamma, *dbeta;
  int blocks, c, stride, wdt, accumulate;
};

// ---- element types -------------------------------------------------------------------------------------------------------------
// A vector is 16 bytes.  Rows may begin at any element (an odd pitch), so the accesses are declared as aligned to the element only: the
// hardware takes a 16-byte access at any address, at full speed where it happens to be aligned.
template <int DT> struct El {
  static constexpr int V = DT == FD_F32 ? 4 : 8;      // elements of a vector
  typedef typename FmtSel<DT == FD_BF16>::type F;
  static __device__ __forceinline__ float load1(const void* p, long long i) {
    if constexpr (DT == FD_F32) return static_cast<const float*>(p)[i];
    else return fd_cvt1<F>(static_cast<const unsigned short*>(p)[i]);
  }
  static __device__ __forceinline__ void store1(void* p, long long i, float v) {
    if constexpr (DT == FD_F32) static_cast<float*>(p)[i] = v;
    else static_cast<unsigned short*>(p)[i] = fd_pk1<F>(v);
  }
};

// V elements as they lie in memory: 16 bytes, or 8 (16-bit types in fours)
template <int DT, int V> struct Vec {
  typedef typename FmtSel<DT == FD_BF16>::type F;
  static constexpr int W = DT == FD_F32 ? V : V / 2;      // words
  typedef unsigned int raw_t __attribute__((ext_vector_type(W)));
  typedef unsigned int any_t __attribute__((ext_vector_type(W), aligned(DT == FD_F32 ? 4 : 2)));
  static __device__ __forceinline__ const char* at(const void* p, long long i) { return static_cast<const char*>(p) + i * (DT == FD_F32 ? 4 : 2); }
  // a vector of which `cnt` elements exist (any number, also below 0); what does not exist is 0
  static __device__ __forceinline__ raw_t raw(const void* p, long long i, int cnt) {
    raw_t v = {};
    if (cnt >= V) {
      v = *reinterpret_cast<const any_t*>(at(p, i));
    } else if (cnt > 0) {
#pragma unroll
      for (int e = 0; e < V - 1; ++e)
        if (e < cnt) {
          if constexpr (DT == FD_F32) v[e] = *reinterpret_cast<const unsigned*>(at(p, i + e));
          else v[e >> 1] |= (unsigned)*reinterpret_cast<const unsigned short*>(at(p, i + e)) << (16 * (e & 1));
        }
    }
    return v;
  }
  static __device__ __forceinline__ void open(raw_t raw, float (&f)[V]) {
    if constexpr (DT == FD_F32) {
#pragma unroll
      for (int e = 0; e < V; ++e) f[e] = __builtin_bit_cast(float, (unsigned)raw[e]);
    } else {
#pragma unroll
      for (int q = 0; q < W; ++q) {
        const f32x2 v = fd_cvt2<F>(raw[q]);
        f[2 * q] = v[0], f[2 * q + 1] = v[1];
      }
    }
  }
  static __device__ __forceinline__ void store(void* p, long long i, int cnt, const float (&f)[V]) {
    if (cnt >= V) {
      raw_t v;
#pragma unroll
      for (int q = 0; q < W; ++q) {
        if constexpr (DT == FD_F32) v[q] = __builtin_bit_cast(unsigned, f[q]);
        else v[q] = fd_pk2<F>(f32x2{f[2 * q], f[2 * q + 1]});
      }
      *reinterpret_cast<any_t*>(const_cast<char*>(at(p, i))) = v;
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (e < cnt) El<DT>::store1(p, i + e, f[e]);
    }
  }
};

// V elements of any type: in whole vectors (a branch around every single load would wait for each: 22 us before a workgroup's first row)
template <int DT, int V> __device__ __forceinline__ void load_some(const void* p, long long i, int cnt, float (&f)[V]) {
  constexpr int Q = V < El<DT>::V ? V : El<DT>::V;
  typename Vec<DT, Q>::raw_t raw[V / Q];
#pragma unroll
  for (int q = 0; q < V / Q; ++q) raw[q] = Vec<DT, Q>::raw(p, i + q * Q, cnt - q * Q);
#pragma unroll
  for (int q = 0; q < V / Q; ++q) {
    float g[Q];
    Vec<DT, Q>::open(raw[q], g);
#pragma unroll
    for (int e = 0; e < Q; ++e) f[q * Q + e] = g[e];
  }
}
// weights: any type, chosen at run time (once for all rows of a workgroup)
template <int V> __device__ __forceinline__ void load_weight(const void* p, int dt, long long i, int cnt, float none, float (&f)[V]) {
  if (!p) {
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] = none;
  } else if (dt == FD_F32) {
    load_some<FD_F32, V>(p, i, cnt, f);
  } else if (dt == FD_F16) {
    load_some<FD_F16, V>(p, i, cnt, f);
  } else {
    load_some<FD_BF16, V>(p, i, cnt, f);
  }
}

// ---- sums over a group of T lanes ----------------------------------------------------------------------------------------------
// T <= 64: additions across lanes in the vector unit -- quads by permutation, 8 and 16 by mirroring (the halves are uniform by then): one
// instruction a step, no LDS round trip.  32: one swizzle.  A whole wave: its four rows' sums read as scalars.
template <int CTRL> __device__ __forceinline__ float dpp_add(float v) {
  return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
template <int T> __device__ __forceinline__ float lanes_sum(float v) {
  if constexpr (T >= 2) v = dpp_add<0xB1>(v);       // quad_perm [1, 0, 3, 2]
  if constexpr (T >= 4) v = dpp_add<0x4E>(v);       // quad_perm [2, 3, 0, 1]
  if constexpr (T >= 8) v = dpp_add<0x141>(v);      // row_half_mirror
  if constexpr (T >= 16) v = dpp_add<0x140>(v);     // row_mirror
  if constexpr (T == 32) v += __builtin_bit_cast(float, __builtin_amdgcn_ds_swizzle(__builtin_bit_cast(int, v), 0x401F));      // lane ^ 16
  if constexpr (T == 64) {
    const int i = __builtin_bit_cast(int, v);
    const float a = __builtin_bit_cast(float, __builtin_amdgcn_readlane(i, 0)), b = __builtin_bit_cast(float, __builtin_amdgcn_readlane(i, 16));
    const float c = __builtin_bit_cast(float, __builtin_amdgcn_readlane(i, 32)), d = __builtin_bit_cast(float, __builtin_amdgcn_readlane(i, 48));
    v = (a + b) + (c + d);
  }
  return v;
}
// More: the waves' sums through LDS; two sets in turn, so that one barrier a sum is enough (a wave that is one
// sum ahead writes the other set; to be two ahead it would have to pass a barrier that waits for this one's reads).
template <int T, int N> struct GroupSum {
  static constexpr int W = T > 64 ? T / 64 : 1;
  float (*red)[1024 / 64][N];     // [2][wave of the workgroup][N]
  int turn = 0;
  __device__ __forceinline__ void operator()(float (&v)[N]) {
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = lanes_sum<(T < 64 ? T : 64)>(v[k]);
    if constexpr (T > 64) {
      const int wave = threadIdx.x >> 6;
      if ((threadIdx.x & 63) == 0) {
#pragma unroll
        for (int k = 0; k < N; ++k) red[turn][wave][k] = v[k];
      }
      __syncthreads();
      const int w0 = wave / W * W;
#pragma unroll
      for (int k = 0; k < N; ++k) {
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) s += red[turn][w0 + w][k];
        v[k] = s;
      }
      turn ^= 1;
    }
  }
};

template <int T> constexpr int block_of() { return T > 256 ? T : 256; }

// A row of equal values v has to find its mean v again, to the last bit: its differences are divided by sqrt(eps), so that one rounding of a mean
// of 60000 (0.004) would come out as a y of 0.8 where there is nothing to see.  The sum of n values v is exact where n times v's digits fit the
// 24 of fp32: n up to 8192 for fp16's 11 digits, 65536 for bf16's 8.  Beyond that, and for fp32, the mean is mended: the differences d = x - m
// of the pass that squares them are summed as well, e = sum d / C is what m is off by, and x - (m + e) = d - e.  (In a row of equal values
// all d are the same few steps of v, so that their sum, e, and the square below are exact.)
template <int DT> constexpr bool mend_mean(int n) { return DT == FD_F32 || n > (DT == FD_F16 ? 8192 : 65536); }
// sum of squares around m, and e, to the mean square around m + e (rounding may leave a little below 0; infinity and NaN stay)
__device__ __forceinline__ float around(float mean_square, float e) {
  const float q = e * e;
  return mean_square < INFINITY ? (mean_square > q ? mean_square - q : 0.f) : mean_square;
}

// ---- forward, held rows ---------------------------------------------------------------------------------------------------------
// Bound by memory: 46 us for 128 MB in and out (65536 x 1024 bf16, 5.8 TB/s; a copy of 128 MB runs at 7.2, one of 2 GB at 4.9), 50 us for
// 16384 x 4096 bf16, 17.6 us for 262144 x 72 fp16 (4.3 TB/s: rows of 144 bytes end inside lines).  Two or three vectors a lane because one
// leaves lanes idle: 24 us instead of 17 at 72 channels, 16 lanes of which 9 work.
template <int DT, int T, int NV> __global__ __launch_bounds__(block_of<T>()) void ln_fwd_rows(LnFwdArgs a) {
  constexpr int V = El<DT>::V, R = block_of<T>() / T;      // rows of a workgroup at a time
  constexpr bool MEND = mend_mean<DT>(T * NV * V);
  constexpr int S = MEND ? 2 : 1;
  __shared__ float red[2][16][1], red2[2][16][S];
  GroupSum<T, 1> sum{red};
  GroupSum<T, S> sum2{red2};
  const int lane = threadIdx.x % T, sub = threadIdx.x / T;
  constexpr int H = T < 1024 ? NV : 1;                     // 1024 lanes have 128 registers each: the weights are read again for every row
  float w[H][V], b[H][V];
  if constexpr (T < 1024) {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int i = (k * T + lane) * V;
      load_weight<V>(a.gamma, a.wdt, i, a.c - i, 1.f, w[k]);
      load_weight<V>(a.beta, a.wdt, i, a.c - i, 0.f, b[k]);
    }
  }
  // the next row's vectors are on their way while this one's are worked on
  const long long hop = (long long)gridDim.x * R;
  typename Vec<DT, V>::raw_t xn[NV];
  auto fetch = [&](long long r) {
    const int c = r < a.rows ? a.c : 0;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int i = (k * T + lane) * V;
      xn[k] = Vec<DT, V>::raw(a.x, r * a.px + i, c - i);
    }
  };
  constexpr bool AHEAD = T < 1024;                         // (1024 lanes: no registers for it)
  if constexpr (AHEAD) fetch((long long)blockIdx.x * R + sub);
  for (long long r0 = (long long)blockIdx.x * R; r0 < a.rows; r0 += hop) {
    const long long r = r0 + sub;
    const int c = r < a.rows ? a.c : 0;
    float x[NV][V], s[1] = {0.f};
    if constexpr (!AHEAD) fetch(r);
#pragma unroll
    for (int k = 0; k < NV; ++k) Vec<DT, V>::open(xn[k], x[k]);
    if constexpr (AHEAD) fetch(r + hop);
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int e = 0; e < V; ++e) s[0] += x[k][e];
    sum(s);
    const float m = s[0] / (float)a.c;               // not times 1 / C (see mend_mean)
    float sq[S] = {};                                // squares, differences
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int cnt = c - (k * T + lane) * V;
#pragma unroll
      for (int e = 0; e < V; ++e) x[k][e] -= m;
      if (cnt < V) {
#pragma unroll
        for (int e = 0; e < V; ++e) x[k][e] = e < cnt ? x[k][e] : 0.f;
      }
#pragma unroll
      for (int e = 0; e < V; ++e) {
        sq[0] += x[k][e] * x[k][e];
        if constexpr (MEND) sq[1] += x[k][e];
      }
    }
    sum2(sq);
    float off = 0.f;
    if constexpr (MEND) off = sq[1] / (float)a.c;
    const float rs = rsqrtf((MEND ? around(sq[0] / (float)a.c, off) : sq[0] * a.inv_c) + a.eps);
    if (c && lane == 0) {
      if (a.mean) a.mean[r] = m + off;
      if (a.rstd) a.rstd[r] = rs;
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      int i = (k * T + lane) * V;
      const int q = T < 1024 ? k : 0;
      if constexpr (T == 1024) {
        asm("" : "+v"(i));                                 // else the weights' addresses are kept over the rows, in registers that are not there
        load_weight<V>(a.gamma, a.wdt, i, a.c - i, 1.f, w[0]);
        load_weight<V>(a.beta, a.wdt, i, a.c - i, 0.f, b[0]);
      }
#pragma unroll
      for (int e = 0; e < V; ++e) x[k][e] = (MEND ? x[k][e] - off : x[k][e]) * rs * w[q][e] + b[q][e];
      Vec<DT, V>::store(a.y, r * a.py + i, c - i, x[k]);
    }
  }
}

// ---- forward, split rows --------------------------------------------------------------------------------------------------------
// A piece is 256 lanes x NV vectors.  The first pass leaves each piece's own mean and its sum of squares around that mean; the second
// joins a row's pieces (mean of the means by their lengths; squares around the pieces' means plus the means' own around the row's) and
// applies the norm.  x is read twice, the second time from a cache where it fits one.  8 rows of 196608 fp32: 3.2 + 4.8 us, against 946 us
// for one workgroup a row; both are a launch and one round of memory latency.
template <int DT, int NV> __global__ __launch_bounds__(256) void ln_fwd_part(LnFwdArgs a) {
  constexpr int V = El<DT>::V;
  __shared__ float red[2][16][1], red2[2][16][2];
  GroupSum<256, 1> sum{red};
  GroupSum<256, 2> sum2{red2};
  const long long r = blockIdx.x / a.pieces;
  const int p = blockIdx.x % a.pieces, at = p * a.piece, n = a.c - at < a.piece ? a.c - at : a.piece;
  float x[NV][V], s[1] = {0.f};
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int i = (k * 256 + threadIdx.x) * V;
    load_some<DT, V>(a.x, r * a.px + at + i, n - i, x[k]);
  }
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int e = 0; e < V; ++e) s[0] += x[k][e];
  sum(s);
  const float m = s[0] / (float)n;
  float sq[2] = {0.f, 0.f};
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int cnt = n - (k * 256 + (int)threadIdx.x) * V;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float d = e < cnt ? x[k][e] - m : 0.f;
      sq[0] += d * d;
      sq[1] += d;
    }
  }
  sum2(sq);
  if (threadIdx.x == 0) {
    const float off = sq[1] / (float)n;
    a.part[2 * (r * a.pieces + p)] = m + off;
    a.part[2 * (r * a.pieces + p) + 1] = around(sq[0] / (float)n, off) * (float)n;
  }
}

template <int DT, int NV> __global__ __launch_bounds__(256) void ln_fwd_apply(LnFwdArgs a) {
  constexpr int V = El<DT>::V;
  __shared__ float red[2][16][1], red2[2][16][2];
  GroupSum<256, 1> sum{red};
  GroupSum<256, 2> sum2{red2};
  const long long r = blockIdx.x / a.pieces;
  const int p = blockIdx.x % a.pieces, at = p * a.piece, n = a.c - at < a.piece ? a.c - at : a.piece;
  float x[NV][V];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int i = (k * 256 + threadIdx.x) * V;
    load_some<DT, V>(a.x, r * a.px + at + i, n - i, x[k]);
  }
  const float* pt = a.part + 2 * r * a.pieces;
  float s[1] = {0.f};
  for (int j = threadIdx.x; j < a.pieces; j += 256) s[0] += pt[2 * j] * (float)(j + 1 < a.pieces ? a.piece : a.c - j * a.piece);
  sum(s);
  const float m0 = s[0] / (float)a.c;
  float sq[2] = {0.f, 0.f};
  for (int j = threadIdx.x; j < a.pieces; j += 256) {
    const float d = pt[2 * j] - m0, nj = (float)(j + 1 < a.pieces ? a.piece : a.c - j * a.piece);
    sq[0] += pt[2 * j + 1] + d * d * nj;
    sq[1] += d * nj;
  }
  sum2(sq);
  const float off = sq[1] / (float)a.c, m = m0 + off;      // see mend_mean: the mean of the means is mended the same way
  const float rs = rsqrtf(around(sq[0] / (float)a.c, off) + a.eps);
  if (p == 0 && threadIdx.x == 0) {
    if (a.mean) a.mean[r] = m;
    if (a.rstd) a.rstd[r] = rs;
  }
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int i = (k * 256 + threadIdx.x) * V;
    float w[V], b[V];
    load_weight<V>(a.gamma, a.wdt, at + i, n - i, 1.f, w);
    load_weight<V>(a.beta, a.wdt, at + i, n - i, 0.f, b);
#pragma unroll
    for (int e = 0; e < V; ++e) x[k][e] = (x[k][e] - m) * rs * w[e] + b[e];
    Vec<DT, V>::store(a.y, r * a.py + at + i, n - i, x[k]);
  }
}

// ---- backward, held rows --------------------------------------------------------------------------------------------------------
// An element that does not exist has dy = 0 and h = 0 and so adds nothing anywhere.  What waits for a row's two sums are the vectors as they were
// loaded, converted a second time: half the registers of the converted ones, which is what decides how many waves a CU holds.
// 84 us for 16384 x 4096 bf16 (402 MB, 4.8 TB/s: a large copy's rate), 52 us for 262144 x 144 fp16 (4.3 TB/s; the same with bf16 gradients), 33 for
// 262144 x 72 (3.4).
// Rows of T lanes: one vector a lane up to 512 of them (few registers, many waves), two or three only where a row takes all 512.
template <int T> constexpr int bwd_rows_of() { return T > 256 ? 1 : T > 128 ? 2 : T == 128 ? 4 : 512 / T; }      // a power of two: the sets are joined in halves
template <int DT, int GT, int T, int NV, int V> __global__ __launch_bounds__(T * bwd_rows_of<T>()) void ln_bwd_rows(LnBwdArgs a) {
  constexpr int R = bwd_rows_of<T>(), B = T * R;
  typedef Vec<DT, V> X;
  typedef Vec<GT, V> Y;
  constexpr int GW = T > 64 ? T : 64, G = B / GW;          // lanes that hold one set of column sums, sets of a workgroup
  __shared__ float red[2][16][2];
  __shared__ float cols[G > 1 ? (B / 2) * NV * V : 1];
  GroupSum<T, 2> sum{red};
  const int lane = threadIdx.x % T, sub = threadIdx.x / T;
  float w[NV][V], dw[NV][V], db[NV][V];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int i = (k * T + lane) * V;
    load_weight<V>(a.gamma, a.wdt, i, a.c - i, 1.f, w[k]);
#pragma unroll
    for (int e = 0; e < V; ++e) dw[k][e] = db[k][e] = 0.f;
  }
  // the next row's vectors are on their way while this one's are worked on
  const long long hop = (long long)gridDim.x * R;
  typename X::raw_t xn[NV];
  typename Y::raw_t gn[NV];
  float mn, rn;
  auto fetch = [&](long long r) {
    const int c = r < a.rows ? a.c : 0;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int i = (k * T + lane) * V;
      xn[k] = X::raw(a.x, r * a.px + i, c - i);
      gn[k] = Y::raw(a.dy, r * a.pdy + i, c - i);
    }
    const long long q = r < a.rows ? r : a.rows - 1;
    mn = a.mean[q], rn = a.rstd[q];
  };
  fetch((long long)blockIdx.x * R + sub);
  for (long long r0 = (long long)blockIdx.x * R; r0 < a.rows; r0 += hop) {
    const long long r = r0 + sub;
    const int c = r < a.rows ? a.c : 0;
    const float rs = rn, m = mn;                           // h = (x - m) rs: a fused x rs - m rs would leave m rs's rounding where x is m
    typename X::raw_t xr[NV];
    typename Y::raw_t gr[NV];
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int k = 0; k < NV; ++k) xr[k] = xn[k], gr[k] = gn[k];
    fetch(r + hop);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      float x[V], g[V];
      X::open(xr[k], x);
      Y::open(gr[k], g);
      const int cnt = c - (k * T + lane) * V;
      if (cnt < V) {                                       // what does not exist has h = 0: 0 times an infinite m rs would be NaN
#pragma unroll
        for (int e = 0; e < V; ++e) x[e] = e < cnt ? x[e] : m;
      }
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float h = (x[e] - m) * rs, t = g[e] * w[k][e];
        db[k][e] += g[e];
        dw[k][e] = fmaf(g[e], h, dw[k][e]);
        s[0] += t;
        s[1] = fmaf(t, h, s[1]);
      }
    }
    if (a.dx) {
      sum(s);
      const float c1 = -s[0] * a.inv_c * rs, c2 = -s[1] * a.inv_c * rs;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int i = (k * T + lane) * V;
        float x[V], g[V];
        asm("" : "+v"(xr[k]), "+v"(gr[k]));                // else the compiler keeps the converted values over the sums
        X::open(xr[k], x);
        Y::open(gr[k], g);
#pragma unroll
        for (int e = 0; e < V; ++e) g[e] = fmaf(g[e] * w[k][e], rs, fmaf((x[e] - m) * rs, c2, c1));
        Y::store(a.dx, r * a.pdx + i, c - i, g);
      }
    }
  }
  if (!a.wpart) return;
  // the sets of the lanes' groups inside a wave, then of the waves, in halves
#pragma unroll
  for (int d = T; d < 64; d <<= 1) {
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        dw[k][e] += __shfl_xor(dw[k][e], d, 64);
        db[k][e] += __shfl_xor(db[k][e], d, 64);
      }
  }
  auto halves = [&](float (&v)[NV][V]) {
#pragma unroll
    for (int half = G / 2; half > 0; half >>= 1) {
      const int set = threadIdx.x / GW, at = threadIdx.x - (set >= half ? half * GW : 0);
      __syncthreads();
      if (set >= half && set < 2 * half) {
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
          for (int e = 0; e < V; ++e) cols[(k * V + e) * (B / 2) + at] = v[k][e];
      }
      __syncthreads();
      if (set < half) {
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
          for (int e = 0; e < V; ++e) v[k][e] += cols[(k * V + e) * (B / 2) + at];
      }
    }
  };
  if constexpr (G > 1) {
    halves(dw);
    halves(db);
  }
  if (threadIdx.x < T) {
    float* out = a.wpart + (long long)blockIdx.x * 2 * a.stride;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int i = (k * T + lane) * V;
      if (i < a.c) {                                       // the stride has room for the last vector's whole length
#pragma unroll
        for (int q = 0; q < V; q += 4) {
          *reinterpret_cast<f32x4*>(out + i + q) = f32x4{dw[k][q], dw[k][q + 1], dw[k][q + 2], dw[k][q + 3]};
          *reinterpret_cast<f32x4*>(out + a.stride + i + q) = f32x4{db[k][q], db[k][q + 1], db[k][q + 2], db[k][q + 3]};
        }
      }
    }
  }
}

// The workgroups' column sums: 32 columns a workgroup, 32 lanes down each, joined in LDS.  16 loads in flight a lane: 4 us for 512 workgroups'
// sums, 6 with one.  Few sets of many columns leave most lanes idle: 51 us for one set of 196608, more than the passes that made it.
constexpr int JOINWG = 1 << 20;      // 2^30 lanes: a launch has fewer than 2^32.  Wider rows (above 2^24 values) take several turns
__global__ __launch_bounds__(1024) void ln_bwd_join(LnJoinArgs a) {
  __shared__ float red[32][33];
  const int part = threadIdx.x >> 5;
  for (int c0 = blockIdx.x * 32; c0 < 2 * a.stride; c0 += JOINWG * 32) {
    const int col = c0 + (threadIdx.x & 31);               // columns of {dw, db} side by side
    float s = 0.f;
    if (col < 2 * a.stride) {
#pragma unroll 16
      for (int b = part; b < a.blocks; b += 32) s += a.wpart[(long long)b * 2 * a.stride + col];
    }
    red[part][threadIdx.x & 31] = s;
    __syncthreads();
    if (part == 0 && col < 2 * a.stride) {
      s = 0.f;
#pragma unroll
      for (int k = 0; k < 32; ++k) s += red[k][threadIdx.x];
      const int i = col < a.stride ? col : col - a.stride;
      void* out = col < a.stride ? a.dgamma : a.dbeta;
      if (out && i < a.c) {
        if (a.wdt == FD_F32) El<FD_F32>::store1(out, i, a.accumulate ? El<FD_F32>::load1(out, i) + s : s);
        else if (a.wdt == FD_F16) El<FD_F16>::store1(out, i, a.accumulate ? El<FD_F16>::load1(out, i) + s : s);
        else El<FD_BF16>::store1(out, i, a.accumulate ? El<FD_BF16>::load1(out, i) + s : s);
      }
    }
    __syncthreads();
  }
}

// ---- backward, split rows -------------------------------------------------------------------------------------------------------
// x and dy are read in both passes: 72 + 74 us for 4096 x 16384 fp16 (the passes' own reads and writes at 3.7 and 5.5 TB/s), 30 + 37 us for
// 1024 x 16384 fp32.
template <int DT, int GT, int NV> __global__ __launch_bounds__(256) void ln_bwd_part(LnBwdArgs a) {
  constexpr int V = El<DT>::V;
  __shared__ float red[2][16][2];
  GroupSum<256, 2> sum{red};
  const long long r = blockIdx.x / a.pieces;
  const int p = blockIdx.x % a.pieces, at = p * a.piece, n = a.c - at < a.piece ? a.c - at : a.piece;
  const float m = a.mean[r], rs = a.rstd[r];
  float s[2] = {0.f, 0.f};
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int i = (k * 256 + threadIdx.x) * V;
    float h[V], g[V], w[V];
    load_some<DT, V>(a.x, r * a.px + at + i, n - i, h);
    load_some<GT, V>(a.dy, r * a.pdy + at + i, n - i, g);
    load_weight<V>(a.gamma, a.wdt, at + i, n - i, 1.f, w);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float t = g[e] * w[e];
      s[0] += t;
      s[1] += t * (i + e < n ? (h[e] - m) * rs : 0.f);
    }
  }
  sum(s);
  if (threadIdx.x == 0) {
    a.part[2 * (r * a.pieces + p)] = s[0];
    a.part[2 * (r * a.pieces + p) + 1] = s[1];
  }
}

// A workgroup: one piece of the columns, `slab` rows; it keeps the piece's column sums.  x and dy are read a second time here: no workgroup
// could hold a whole row, and the two sums of a row are known only when all its pieces have been seen.
constexpr int MAXSLAB = 64;
template <int DT, int GT, int NV> __global__ __launch_bounds__(256) void ln_bwd_apply(LnBwdArgs a) {
  constexpr int V = El<DT>::V;
  __shared__ float row[MAXSLAB][4];       // mean, rstd, c1, c2
  const int p = blockIdx.x % a.pieces, at = p * a.piece, n = a.c - at < a.piece ? a.c - at : a.piece;
  const long long r0 = (long long)(blockIdx.x / a.pieces) * a.slab;
  const int nr = (int)(a.rows - r0 < a.slab ? a.rows - r0 : a.slab);
  for (int q = threadIdx.x >> 6; q < nr; q += 4) {
    float s1 = 0.f, s2 = 0.f;
    if (a.dx)
      for (int j = threadIdx.x & 63; j < a.pieces; j += 64) {
        s1 += a.part[2 * ((r0 + q) * a.pieces + j)];
        s2 += a.part[2 * ((r0 + q) * a.pieces + j) + 1];
      }
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) s1 += __shfl_xor(s1, d, 64), s2 += __shfl_xor(s2, d, 64);
    if ((threadIdx.x & 63) == 0) {
      row[q][0] = a.mean[r0 + q], row[q][1] = a.rstd[r0 + q];
      row[q][2] = s1 * a.inv_c, row[q][3] = s2 * a.inv_c;
    }
  }
  __syncthreads();
  float w[NV][V], dw[NV][V], db[NV][V];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int i = (k * 256 + threadIdx.x) * V;
    load_weight<V>(a.gamma, a.wdt, at + i, n - i, 1.f, w[k]);
#pragma unroll
    for (int e = 0; e < V; ++e) dw[k][e] = db[k][e] = 0.f;
  }
  for (int q = 0; q < nr; ++q) {
    const float m = row[q][0], rs = row[q][1], c1 = row[q][2], c2 = row[q][3];
    const long long r = r0 + q;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int i = (k * 256 + threadIdx.x) * V;
      float h[V], g[V];
      load_some<DT, V>(a.x, r * a.px + at + i, n - i, h);
      load_some<GT, V>(a.dy, r * a.pdy + at + i, n - i, g);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        h[e] = (h[e] - m) * rs;
        db[k][e] += g[e];
        dw[k][e] += g[e] * h[e];
        g[e] = rs * (g[e] * w[k][e] - c1 - h[e] * c2);
      }
      if (a.dx) Vec<GT, V>::store(a.dx, r * a.pdx + at + i, n - i, g);
    }
  }
  if (!a.wpart) return;
  float* out = a.wpart + (long long)(blockIdx.x / a.pieces) * 2 * a.stride + at;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int i = (k * 256 + threadIdx.x) * V;
    if (i < n) {
#pragma unroll
      for (int q = 0; q < V; q += 4) {
        *reinterpret_cast<f32x4*>(out + i + q) = f32x4{dw[k][q], dw[k][q + 1], dw[k][q + 2], dw[k][q + 3]};
        *reinterpret_cast<f32x4*>(out + a.stride + i + q) = f32x4{db[k][q], db[k][q + 1], db[k][q + 2], db[k][q + 3]};
      }
    }
  }
}

// ---- which variant --------------------------------------------------------------------------------------------------------------
struct Shape {
  int T, NV, V;                     // held rows: lanes, vectors of a lane, elements of one (backward); T = 0: split
  int pieces, piece, slab;          // split rows
  int blocks, stride;               // sets of column sums of the backward pass, floats of one
  long long floats;                 // workspace
};

// Forward: T lanes x NV vectors with NV = 2 or 3 (1 where there is one): the power of two below n with three vectors a lane if that is
// enough, else its double with two -- at least three lanes in four have work at every n.
void held_fwd(int n, Shape& s) {
  int T = 1;
  while (2 * T < n && T < 1024) T *= 2;
  s.T = T, s.NV = n == 1 ? 1 : 2;
  if (T > 1 && n <= T / 2 * 3) s.T = T / 2, s.NV = 3;
  if (n > 2 * T) s.NV = (n + T - 1) / T;                  // T = 1024
}

// Backward: one vector a lane (a power of two of lanes inside a wave, whole waves beyond, two or three vectors above 512 lanes), or 12 elements
// a lane in three vectors of four, whichever leaves fewer places empty: the pass is as much bound by its instructions as by memory where
// half the lanes idle (144 fp16 channels: 32 lanes x 8 70 us, 16 lanes x 12 52 us for 262144 rows).
void held_bwd(int c, int V, Shape& s) {
  const int n = (c + V - 1) / V;
  s.V = V;
  s.NV = (n + 511) / 512;
  s.T = 1;
  while (s.T < n && s.T < 64) s.T *= 2;
  if (n > 64) s.T = s.NV > 1 ? 512 : (n + 63) / 64 * 64;
  int T = 1;
  while (12 * T < c) T *= 2;
  if (T <= 64 && 12 * T < s.T * s.NV * V) s.T = T, s.NV = 3, s.V = 4;
}

Shape shape_fwd(long long rows, long long c, int V) {
  Shape s{};
  const long long n = (c + V - 1) / V;
  if (n <= 4 * 1024) held_fwd((int)n, s);
  if (s.T) return s;
  s.NV = 4;
  while (s.NV > 1 && rows * ((n + 256 * s.NV - 1) / (256 * s.NV)) < 512) s.NV /= 2;      // enough workgroups for the chip
  s.piece = 256 * s.NV * V;
  s.pieces = (int)((c + s.piece - 1) / s.piece);
  s.floats = 2 * rows * s.pieces;
  return s;
}

Shape shape_bwd(long long rows, long long c, int V) {
  Shape s{};
  const long long n = (c + V - 1) / V;
  s.stride = (int)(n * V);
  if (n <= 3 * 512) held_bwd((int)c, V, s);
  if (s.T) {
    const int R = s.T > 256 ? 1 : s.T > 128 ? 2 : s.T == 128 ? 4 : 512 / s.T;
    const long long b = (rows + R - 1) / R;
    // what the registers let the chip hold at once: 85 to 97 a lane at one vector of 8, 146 and 206 at two and three
    const int most = s.NV > 1 && s.V > 4 ? 256 : 512;
    s.blocks = (int)(b < most ? b : most);      // (768 at one vector: 97 us instead of 83 at 16384 x 4096 bf16, a second round half empty)
    s.floats = 2ll * s.blocks * s.stride;
    return s;
  }
  s.NV = 2;
  if (rows * ((n + 511) / 512) < 512) s.NV = 1;
  s.piece = 256 * s.NV * V;
  s.pieces = (int)((c + s.piece - 1) / s.piece);
  // rows of a workgroup: at least 8 (each workgroup leaves 2 floats a column behind, against the 6 to 12 bytes a value of every row), more where 1024
  // workgroups have them.  Few long rows are few workgroups: 8 x 196608 fp32 are 96 of them, 10 us for the 19 MB of that pass
  long long slab = rows * s.pieces / 1024;
  s.slab = (int)(slab < 8 ? 8 : slab > MAXSLAB ? MAXSLAB : slab);
  s.blocks = (int)((rows + s.slab - 1) / s.slab);
  s.floats = 2 * rows * s.pieces + 2ll * s.blocks * s.stride;
  return s;
}

constexpr long long MAXC = 1ll << 29, MAXROWS = 1ll << 40;      // twice the columns is an int; row times pitch a long long
constexpr long long MAXPIECES = 1ll << 24;                      // of all rows: a workgroup of 256 lanes each, and a launch has fewer than 2^32 lanes

// split rows whose pieces are more than one launch takes
bool too_many(const Shape& s, long long rows) { return s.T == 0 && rows >= (MAXPIECES + s.pieces - 1) / s.pieces; }

bool known(int dt) { return dt == FD_F32 || dt == FD_F16 || dt == FD_BF16; }
int esize(int dt) { return dt == FD_F32 ? 4 : 2; }

// The rows of a view: n * h * w of them at one pitch, channels next to each other
int row_view(const char* what, const FdTensor* t, bool written, long long* rows, long long* pitch) {
  FD_REQUIRE(t, "%s: NULL view", what);
  FD_REQUIRE(t->n >= 0 && t->h >= 0 && t->w >= 0 && t->c >= 1 && t->c <= MAXC && (double)t->n * (double)t->h * (double)t->w <= (double)MAXROWS,
             "%s: %lld x %lld x %lld x %lld", what, (long long)t->n, (long long)t->h, (long long)t->w, (long long)t->c);
  FD_REQUIRE(known(t->dtype), "%s: dtype %d", what, t->dtype);
  FD_REQUIRE(t->c == 1 || t->stride[3] == 1, "%s: channel stride %lld (1 expected)", what, (long long)t->stride[3]);
  *rows = t->n * t->h * t->w;
  *pitch = t->c;
  if (*rows == 0) return FD_OK;
  FD_REQUIRE(t->ptr && ((uintptr_t)t->ptr & (esize(t->dtype) - 1)) == 0, "%s: NULL or not aligned to its element", what);
  const int64_t ext[3] = {t->w, t->h, t->n}, str[3] = {t->stride[2], t->stride[1], t->stride[0]};
  long long have = 1;
  for (int k = 0; k < 3; ++k) {
    if (ext[k] == 1) continue;
    if (have == 1) *pitch = str[k];
    FD_REQUIRE(str[k] == *pitch * have, "%s: the rows do not lie at one pitch", what);
    have *= ext[k];
  }
  FD_REQUIRE(*pitch >= (written && *rows > 1 ? t->c : 0), "%s: row pitch %lld below %lld channels", what, (long long)*pitch, (long long)t->c);
  return FD_OK;
}

template <int V> struct Int { static constexpr int value = V; };

#define FD_LN_CASE(t, nv) \
  if (s.T == t && s.NV == nv) return f(Int<t>{}, Int<nv>{});
template <class Fn> int with_fwd(const Shape& s, Fn f) {
  FD_LN_CASE(1, 1) FD_LN_CASE(1, 2) FD_LN_CASE(1, 3) FD_LN_CASE(2, 2) FD_LN_CASE(2, 3) FD_LN_CASE(4, 2) FD_LN_CASE(4, 3) FD_LN_CASE(8, 2)
  FD_LN_CASE(8, 3) FD_LN_CASE(16, 2) FD_LN_CASE(16, 3) FD_LN_CASE(32, 2) FD_LN_CASE(32, 3) FD_LN_CASE(64, 2) FD_LN_CASE(64, 3) FD_LN_CASE(128, 2)
  FD_LN_CASE(128, 3) FD_LN_CASE(256, 2) FD_LN_CASE(256, 3) FD_LN_CASE(512, 2) FD_LN_CASE(512, 3) FD_LN_CASE(1024, 2) FD_LN_CASE(1024, 3)
  FD_LN_CASE(1024, 4)
  FD_FAIL(FD_EUNSUPPORTED, "layer_norm: no variant for %d lanes x %d vectors", s.T, s.NV);
}
template <class Fn> int with_bwd(const Shape& s, Fn f) {
  FD_LN_CASE(1, 1) FD_LN_CASE(2, 1) FD_LN_CASE(4, 1) FD_LN_CASE(8, 1) FD_LN_CASE(16, 1) FD_LN_CASE(32, 1) FD_LN_CASE(64, 1) FD_LN_CASE(128, 1)
  FD_LN_CASE(192, 1) FD_LN_CASE(256, 1) FD_LN_CASE(320, 1) FD_LN_CASE(384, 1) FD_LN_CASE(448, 1) FD_LN_CASE(512, 1) FD_LN_CASE(512, 2)
  FD_LN_CASE(512, 3) FD_LN_CASE(1, 3) FD_LN_CASE(2, 3) FD_LN_CASE(4, 3) FD_LN_CASE(8, 3) FD_LN_CASE(16, 3) FD_LN_CASE(32, 3) FD_LN_CASE(64, 3)
  FD_FAIL(FD_EUNSUPPORTED, "layer_norm: no variant for %d lanes x %d vectors", s.T, s.NV);
}
#undef FD_LN_CASE

template <int DT> int launch_fwd(LnFwdArgs& a, hipStream_t st) {
  const Shape s = shape_fwd(a.rows, a.c, El<DT>::V);
  if (s.T)
    return with_fwd(s, [&](auto t, auto nv) {
      constexpr int T = decltype(t)::value, NV = decltype(nv)::value, R = block_of<T>() / T;
      // as many workgroups as the registers let the chip hold at once (16-bit types 46, 78 to 86, 107 to 124 a lane at 1, 2 or 3 vectors, fp32
      // 35, 51 to 64, 67 to 79, 86 at 512 lanes x 3; 1024 lanes 50 to 81): a few more than that would take a whole second round for themselves
      constexpr int WAVES = NV == 1 ? 8 : El<DT>::V == 4 ? (NV == 2 ? 8 : NV == 3 && T < 512 ? 6 : 5) : NV == 2 ? (T <= 64 ? 5 : 6) : 4;
      constexpr int MOST = 256 * (WAVES * 256 / block_of<T>());
      const long long b = (a.rows + R - 1) / R;
      return fd_launch(&ln_fwd_rows<DT, T, NV>, "layer_norm_fwd", dim3((unsigned)(b < MOST ? b : MOST)), dim3(block_of<T>()), 0, a, st);
    });
  a.piece = s.piece, a.pieces = s.pieces;
  const long long wgs = a.rows * s.pieces;
  auto both = [&](auto nv) {
    constexpr int NV = decltype(nv)::value;
    const int rc = fd_launch(&ln_fwd_part<DT, NV>, "layer_norm_fwd_part", dim3((unsigned)wgs), dim3(256), 0, a, st);
    return rc != FD_OK ? rc : fd_launch(&ln_fwd_apply<DT, NV>, "layer_norm_fwd_apply", dim3((unsigned)wgs), dim3(256), 0, a, st);
  };
  return s.NV == 4 ? both(Int<4>{}) : s.NV == 2 ? both(Int<2>{}) : both(Int<1>{});
}

template <int DT, int GT> int launch_bwd(LnBwdArgs& a, float* ws, const Shape& s, hipStream_t st) {
  a.stride = s.stride;
  if (s.T) {
    if (a.wpart) a.wpart = ws;
    return with_bwd(s, [&](auto t, auto nv) {
      constexpr int T = decltype(t)::value, NV = decltype(nv)::value, V = NV == 3 && T <= 64 ? 4 : El<DT>::V;
      return fd_launch(&ln_bwd_rows<DT, GT, T, NV, V>, "layer_norm_bwd", dim3((unsigned)s.blocks), dim3(T * bwd_rows_of<T>()), 0, a, st);
    });
  }
  a.piece = s.piece, a.pieces = s.pieces, a.slab = s.slab;
  a.part = ws;
  if (a.wpart) a.wpart = ws + ((2 * a.rows * s.pieces + 3) & ~3ll);
  const long long wgs = a.rows * s.pieces;
  auto both = [&](auto nv) {
    constexpr int NV = decltype(nv)::value;
    if (a.dx) {
      const int rc = fd_launch(&ln_bwd_part<DT, GT, NV>, "layer_norm_bwd_part", dim3((unsigned)wgs), dim3(256), 0, a, st);
      if (rc != FD_OK) return rc;
    }
    return fd_launch(&ln_bwd_apply<DT, GT, NV>, "layer_norm_bwd_apply", dim3((unsigned)(s.blocks * s.pieces)), dim3(256), 0, a, st);
  };
  return s.NV == 2 ? both(Int<2>{}) : both(Int<1>{});
}

}  // namespace

extern "C" int64_t fdgan_layer_norm_workspace(int64_t rows, int64_t c, int backward) {
  if (rows < 0 || rows > MAXROWS || c < 1 || c > MAXC) return -1;
  if (rows == 0) return 0;
  long long most = -1;
  for (int V : {4, 8}) {
    const Shape s = backward ? shape_bwd(rows, c, V) : shape_fwd(rows, c, V);
    if (too_many(s, rows)) continue;      // (the other types' vectors hold more)
    const long long f = s.floats > 0 ? s.floats + 4 : 0;
    most = f > most ? f : most;
  }
  return most;
}

extern "C" int fdgan_layer_norm_fwd(const FdTensor* x, const void* gamma, const void* beta, int wdtype, float eps, const FdTensor* y, float* mean,
                                    float* rstd, float* ws, int64_t ws_floats, FdStream stream) {
  long long rows, yrows, px, py;
  int rc = row_view("layer_norm_fwd: x", x, false, &rows, &px);
  if (rc == FD_OK) rc = row_view("layer_norm_fwd: y", y, true, &yrows, &py);
  if (rc != FD_OK) return rc;
  FD_REQUIRE(rows == yrows && x->c == y->c && x->dtype == y->dtype, "layer_norm_fwd: x and y differ in shape or dtype");
  FD_REQUIRE(known(wdtype), "layer_norm_fwd: weight dtype %d", wdtype);
  FD_REQUIRE(eps >= 0.f, "layer_norm_fwd: eps %g", (double)eps);
  if (rows == 0) return FD_OK;
  FD_REQUIRE(x->ptr != y->ptr, "layer_norm_fwd: y is x");
  const Shape s = shape_fwd(rows, x->c, x->dtype == FD_F32 ? 4 : 8);
  FD_REQUIRE(!too_many(s, rows), "layer_norm_fwd: %lld rows of %lld values are too many for one call", rows, (long long)x->c);
  FD_REQUIRE(s.floats == 0 || (ws && ((uintptr_t)ws & 15) == 0 && ws_floats >= s.floats), "layer_norm_fwd: a workspace of %lld floats at a multiple of 16 bytes", s.floats);
  LnFwdArgs a{x->ptr, y->ptr, gamma, beta, mean, rstd, ws, rows, px, py, (int)x->c, wdtype, 0, 0, eps, 1.f / (float)x->c};
  hipStream_t st = static_cast<hipStream_t>(stream);
  return x->dtype == FD_F32 ? launch_fwd<FD_F32>(a, st) : x->dtype == FD_F16 ? launch_fwd<FD_F16>(a, st) : launch_fwd<FD_BF16>(a, st);
}

extern "C" int fdgan_layer_norm_bwd(const FdTensor* x, const FdTensor* dy, const void* gamma, int wdtype, const float* mean, const float* rstd,
                                    const FdTensor* dx, void* dgamma, void* dbeta, int accumulate, float* ws, int64_t ws_floats, FdStream stream) {
  long long rows, r2, px, pdy, pdx = 0;
  int rc = row_view("layer_norm_bwd: x", x, false, &rows, &px);
  if (rc == FD_OK) rc = row_view("layer_norm_bwd: dy", dy, false, &r2, &pdy);
  if (rc != FD_OK) return rc;
  FD_REQUIRE(rows == r2 && x->c == dy->c, "layer_norm_bwd: x and dy differ in shape");
  FD_REQUIRE(x->dtype == dy->dtype || (x->dtype == FD_F16 && dy->dtype == FD_BF16), "layer_norm_bwd: x of dtype %d with dy of dtype %d", x->dtype, dy->dtype);
  if (dx) {
    rc = row_view("layer_norm_bwd: dx", dx, true, &r2, &pdx);
    if (rc != FD_OK) return rc;
    FD_REQUIRE(rows == r2 && x->c == dx->c && dx->dtype == dy->dtype, "layer_norm_bwd: dx and dy differ in shape or dtype");
    FD_REQUIRE(rows == 0 || (dx->ptr != dy->ptr && dx->ptr != x->ptr), "layer_norm_bwd: dx is x or dy");
  }
  FD_REQUIRE(known(wdtype), "layer_norm_bwd: weight dtype %d", wdtype);
  FD_REQUIRE(dx || dgamma || dbeta, "layer_norm_bwd: no output");
  FD_REQUIRE(rows == 0 || (mean && rstd), "layer_norm_bwd: NULL statistics");
  hipStream_t st = static_cast<hipStream_t>(stream);
  const bool weights = dgamma || dbeta;
  Shape s{};
  if (rows > 0) {
    s = shape_bwd(rows, x->c, x->dtype == FD_F32 ? 4 : 8);
    FD_REQUIRE(!too_many(s, rows), "layer_norm_bwd: %lld rows of %lld values are too many for one call", rows, (long long)x->c);
    FD_REQUIRE(ws && ((uintptr_t)ws & 15) == 0 && ws_floats >= s.floats + 4, "layer_norm_bwd: a workspace of %lld floats at a multiple of 16 bytes", s.floats + 4);
    LnBwdArgs a{x->ptr, dy->ptr, dx ? dx->ptr : nullptr, gamma, mean, rstd, nullptr, weights ? ws : nullptr, rows, px, pdy, pdx, (int)x->c, wdtype, 0, 0, 0, 0,
                1.f / (float)x->c};
    rc = x->dtype == FD_F32    ? launch_bwd<FD_F32, FD_F32>(a, ws, s, st)
         : x->dtype == FD_BF16 ? launch_bwd<FD_BF16, FD_BF16>(a, ws, s, st)
         : dy->dtype == FD_F16 ? launch_bwd<FD_F16, FD_F16>(a, ws, s, st)
                               : launch_bwd<FD_F16, FD_BF16>(a, ws, s, st);
    if (rc != FD_OK) return rc;
    ws = a.wpart;
  } else {
    s.stride = (int)x->c;
  }
  if (!weights) return FD_OK;
  LnJoinArgs j{ws, dgamma, dbeta, s.blocks, (int)x->c, s.stride, wdtype, accumulate ? 1 : 0};
  const long long wgs = (2ll * s.stride + 31) / 32;
  return fd_launch(&ln_bwd_join, "layer_norm_bwd_join", dim3((unsigned)(wgs < JOINWG ? wgs : JOINWG)), dim3(1024), 0, j, st);
}
