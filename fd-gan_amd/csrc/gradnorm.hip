// gradnorm.hip -- the global norm of a list of gradients, clipping by it, and the Adam step that clips on the way.
//
//   norm   = ( sum over all tensors of sum |g|^p )^(1/p),  p = 1, 2;  max |g| for p = infinity
//   factor = min(1, max_norm / (norm + 1e-6));   g <- g * factor
//
// The list goes to the kernel BY VALUE (pointer, length, first chunk of up to MAXT tensors: a 4 KB argument block), so that a call
// copies nothing to the device, can be captured, and leaves nothing behind that a later call could find stale.  A tensor is cut into
// chunks of CHUNK elements; each workgroup takes a contiguous run of chunks -- one stretch of each tensor it touches, read in vectors of 16
// bytes at whatever alignment, eight of them in flight a lane (four where they are written back) -- and writes ONE partial.  Whoever needs
// the norm next (the scaling pass, the Adam pass) reduces the few hundred partials itself, in the same order in every workgroup: there is no atomic, no
// launch in between, and every workgroup of every rank finds the same factor to the last bit.
//
// Sums are in fp64: a gradient of 1e-23 or 1e+23 squares to 0 or infinity in fp32, and the MI355X forms fp64 multiply-adds at the
// rate of fp32 ones, far above what the memory delivers.
#include "common.h"
#include "adam.h"
#include <math.h>

namespace {

constexpr int MAXT = 188;             // 188 * (8 + 8 + 4) bytes + the scalars below stay under 4 KB
constexpr long long CHUNK = 4096;     // elements
constexpr long long MAXN = 1ll << 40; // elements of one tensor: its chunks are an int
// An Adam step over more bytes than this reads and writes past the caches: the 256 MB behind the L2s cannot keep its four tensors for the
// next step, and lines that wait there to be written back slow the reading.  Both passes, us, through the caches / past them, three sets of
// tensors in turn: 100 MB 22.4 / 25.8, 200 MB 47.6 / 48.4, 250 MB 59.9 / 56.6, 600 MB 144 / 128, 1.9 GB 476 / 413.
constexpr long long STREAM = 224ll << 20;
constexpr int MAXWG = 512;            // workgroups (= partials) of one launch: two a CU
constexpr int MAXPART = 1024;         // partials a consumer reduces by itself; more are reduced by norm_finish_kernel first

struct SpanTable {
  void* ptr[MAXT];
  long long n_dt[MAXT];               // length * 4 + FdDtype
  unsigned first[MAXT];               // chunk at which the tensor begins
  int count;
  unsigned chunks;
};

struct NormArgs {
  SpanTable t;
  double* partial;
  int kind;                           // 1, 2: the power; 0: the maximum
};

struct PartialRef {
  const double* partial;
  int count, kind;
  float max_norm;
  float* norm_out;                    // written by the first workgroup; may be null
};

struct ScaleArgs {
  SpanTable t;
  PartialRef r;
};

struct FinishArgs {
  const double* partial;
  int count, kind;
  double* total;                      // one combined partial (may be null)
  float* norm_out;                    // may be null
};

struct AdamClipArgs {
  float *p, *m, *v;
  const float* g;
  long long n;
  AdamUpdate u;
  PartialRef r;
};

// A maximum is taken over the magnitudes' bit patterns, which order as the magnitudes do, with NaN above infinity: a NaN stays.
__device__ __forceinline__ double join(double a, double b, int kind) {
  if (kind != 0) return a + b;
  return (b > a || b != b) ? b : a;
}

// the same value in every thread of a workgroup of W waves
template <int W> __device__ __forceinline__ double block_join(double v, int kind) {
  __shared__ double red[W];
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v = join(v, __shfl_xor(v, d, 64), kind);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = red[0];
#pragma unroll
  for (int w = 1; w < W; ++w) v = join(v, red[w], kind);
  __syncthreads();
  return v;
}

__device__ __forceinline__ float norm_of(double total, int kind) { return (float)(kind == 2 ? sqrt(total) : total); }

// every thread of the workgroup: the factor (and, once, the norm)
__device__ __forceinline__ float clip_factor(const PartialRef& r) {
  double s = 0.0;
  for (int i = threadIdx.x; i < r.count; i += 256) s = join(s, r.partial[i], r.kind);
  const float norm = norm_of(block_join<4>(s, r.kind), r.kind);
  if (r.norm_out && blockIdx.x == 0 && threadIdx.x == 0) r.norm_out[0] = norm;
  const float c = r.max_norm / (norm + 1e-6f);
  return c > 1.f ? 1.f : c;           // a NaN goes through
}

// ---- element types: 16-byte vectors at any element's address, single elements -----------------------------------------------------
typedef unsigned int u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
template <int DT> struct El {
  static constexpr int V = DT == FD_F32 ? 4 : 8;
  typedef typename FmtSel<DT == FD_BF16>::type F;
  static __device__ __forceinline__ char* at(void* p, long long i) { return static_cast<char*>(p) + i * (DT == FD_F32 ? 4 : 2); }
  static __device__ __forceinline__ u32x4 raw_past(void* p, long long i) { return __builtin_nontemporal_load(reinterpret_cast<const u32x4_any*>(at(p, i))); }
  static __device__ __forceinline__ u32x4 raw(void* p, long long i) { return *reinterpret_cast<const u32x4_any*>(at(p, i)); }
  static __device__ __forceinline__ void put(void* p, long long i, u32x4 v) { *reinterpret_cast<u32x4_any*>(at(p, i)) = v; }
  static __device__ __forceinline__ float get1(void* p, long long i) {
    if constexpr (DT == FD_F32) return *reinterpret_cast<const float*>(at(p, i));
    else return fd_cvt1<F>(*reinterpret_cast<const unsigned short*>(at(p, i)));
  }
  static __device__ __forceinline__ void put1(void* p, long long i, float v) {
    if constexpr (DT == FD_F32) *reinterpret_cast<float*>(at(p, i)) = v;
    else *reinterpret_cast<unsigned short*>(at(p, i)) = fd_pk1<F>(v);
  }
  static __device__ __forceinline__ void open(u32x4 raw, float (&f)[V]) {
    if constexpr (DT == FD_F32) {
      const f32x4 v = __builtin_bit_cast(f32x4, raw);
#pragma unroll
      for (int e = 0; e < V; ++e) f[e] = v[e];
    } else {
      const f32x8 v = fd_cvt8<F>(raw);
#pragma unroll
      for (int e = 0; e < V; ++e) f[e] = v[e];
    }
  }
  static __device__ __forceinline__ u32x4 close(const float (&f)[V]) {
    if constexpr (DT == FD_F32) return __builtin_bit_cast(u32x4, f32x4{f[0], f[1], f[2], f[3]});
    else return fd_pk8<F>(f32x8{f[0], f[1], f[2], f[3], f[4], f[5], f[6], f[7]});
  }
};

// index of the tensor that holds `chunk`: every thread looks at one entry
__device__ __forceinline__ int find_span(const SpanTable& t, unsigned chunk) {
  __shared__ int found;
  const int i = threadIdx.x;
  if (i < t.count) {
    const unsigned lo = t.first[i], hi = i + 1 < t.count ? t.first[i + 1] : t.chunks;
    if (chunk >= lo && chunk < hi) found = i;
  }
  __syncthreads();
  const int r = found;
  __syncthreads();
  return r;
}

// f(pointer, first element, end, dtype) for the stretch of every tensor in this workgroup's run of chunks
template <class Fn> __device__ __forceinline__ void each_stretch(const SpanTable& t, Fn f) {
  const unsigned lo = (unsigned)((unsigned long long)t.chunks * blockIdx.x / gridDim.x);
  const unsigned hi = (unsigned)((unsigned long long)t.chunks * (blockIdx.x + 1) / gridDim.x);
  for (int k = find_span(t, lo); k < t.count && t.first[k] < hi; ++k) {
    const long long n = t.n_dt[k] >> 2;
    const unsigned from = lo > t.first[k] ? lo - t.first[k] : 0;
    const long long end = (long long)(hi - t.first[k]) * CHUNK;
    f(t.ptr[k], (long long)from * CHUNK, end < n ? end : n, (int)(t.n_dt[k] & 3));
  }
}

// Bound by memory: 348 MB of bf16 in 87 us (4.0 TB/s), with half of it still behind the L2s from the pass before; 268 MB of fp32 in 82 us read
// through the caches and in 44 us (6 TB/s) past them.  The start of a workgroup (finding its tensor) and its join cost 3 to 4 us, which is what
// lists of a few MB take.
constexpr int NT = 512;               // lanes of a workgroup of the norm pass

// One lane's share of a stretch.  KIND 2, 1: fp64 sums of squares, of magnitudes; 0: the largest magnitude's bits
template <int DT, int KIND, bool PAST> __device__ __forceinline__ void norm_share(void* p, long long i, long long end, double& s, unsigned& m) {
  constexpr int V = El<DT>::V;
  double q[2] = {0.0, 0.0};
  auto one = [&](float g, int e) {
    if (KIND == 2) q[e & 1] = fma((double)g, (double)g, q[e & 1]);
    else if (KIND == 1) q[e & 1] += fabs((double)g);
    else {
      const unsigned b = __builtin_bit_cast(unsigned, g) & 0x7fffffffu;
      m = b > m ? b : m;
    }
  };
  auto vec = [&](u32x4 v) {
    float g[V];
    El<DT>::open(v, g);
#pragma unroll
    for (int e = 0; e < V; ++e) one(g[e], e);
  };
  i += threadIdx.x * V;
  for (; i + 7 * NT * V + V <= end; i += 8 * NT * V) {
    u32x4 v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = PAST ? El<DT>::raw_past(p, i + k * NT * V) : El<DT>::raw(p, i + k * NT * V);
#pragma unroll
    for (int k = 0; k < 8; ++k) vec(v[k]);
  }
  for (; i + V <= end; i += NT * V) vec(El<DT>::raw(p, i));
  for (; i < end; ++i) one(El<DT>::get1(p, i), 0);      // at most one lane: the last vector is not whole
  s += q[0] + q[1];
}

template <int KIND, bool PAST> __device__ __forceinline__ void norm_body(const NormArgs& a) {
  double s = 0.0;
  unsigned m = 0;
  each_stretch(a.t, [&](void* p, long long i, long long end, int dt) {
    if (dt == FD_F32) norm_share<FD_F32, KIND, PAST>(p, i, end, s, m);
    else if (dt == FD_F16) norm_share<FD_F16, KIND, PAST>(p, i, end, s, m);
    else norm_share<FD_BF16, KIND, PAST>(p, i, end, s, m);
  });
  if (KIND == 0) s = (double)__builtin_bit_cast(float, m);
  s = block_join<NT / 64>(s, KIND);
  if (threadIdx.x == 0) a.partial[blockIdx.x] = s;
}

__global__ __launch_bounds__(NT) void grad_norm_kernel(NormArgs a) {
  if (a.kind == 2) norm_body<2, false>(a);
  else if (a.kind == 1) norm_body<1, false>(a);
  else norm_body<0, false>(a);
}
// the 2-norm of a flat tensor whose Adam step streams (see STREAM)
__global__ __launch_bounds__(NT) void grad_norm_past_kernel(NormArgs a) { norm_body<2, true>(a); }

__global__ __launch_bounds__(256) void norm_finish_kernel(FinishArgs a) {
  double s = 0.0;
  for (int i = threadIdx.x; i < a.count; i += 256) s = join(s, a.partial[i], a.kind);
  s = block_join<4>(s, a.kind);
  if (threadIdx.x == 0) {
    if (a.total) a.total[0] = s;
    if (a.norm_out) a.norm_out[0] = norm_of(s, a.kind);
  }
}

// 348 MB of bf16 read and written in 131 us (5.3 TB/s).  The factor is formed by every workgroup for itself: 1000 partials are 8 KB from the L2,
// 1 to 2 us, where a launch between the passes would cost 3 to 4.
template <int DT> __device__ __forceinline__ void scale_share(void* p, long long i, long long end, float f) {
  constexpr int V = El<DT>::V;
  auto vec = [&](u32x4 v, long long at) {
    float g[V];
    El<DT>::open(v, g);
#pragma unroll
    for (int e = 0; e < V; ++e) g[e] *= f;
    El<DT>::put(p, at, El<DT>::close(g));
  };
  i += threadIdx.x * V;
  for (; i + 3 * 256 * V + V <= end; i += 4 * 256 * V) {
    u32x4 v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = El<DT>::raw(p, i + k * 256 * V);
#pragma unroll
    for (int k = 0; k < 4; ++k) vec(v[k], i + k * 256 * V);
  }
  for (; i + V <= end; i += 256 * V) vec(El<DT>::raw(p, i), i);
  for (; i < end; ++i) El<DT>::put1(p, i, El<DT>::get1(p, i) * f);
}

__global__ __launch_bounds__(256) void grad_scale_kernel(ScaleArgs a) {
  const float f = clip_factor(a.r);
  each_stretch(a.t, [&](void* p, long long i, long long end, int dt) {
    if (dt == FD_F32) scale_share<FD_F32>(p, i, end, f);
    else if (dt == FD_F16) scale_share<FD_F16>(p, i, end, f);
    else scale_share<FD_BF16>(p, i, end, f);
  });
}

// 67 million parameters: 28 bytes each in 359 us (5.2 TB/s); 790416: 6 us, of which the factor is 2.
template <bool PAST> __device__ __forceinline__ f32x4 get4(const float* p) {
  return PAST ? __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(p)) : *reinterpret_cast<const f32x4*>(p);
}
template <bool PAST> __device__ __forceinline__ void put4(float* p, f32x4 v) {
  if (PAST) __builtin_nontemporal_store(v, reinterpret_cast<f32x4*>(p));
  else *reinterpret_cast<f32x4*>(p) = v;
}

template <bool PAST> __global__ __launch_bounds__(256) void adam_clip_kernel(AdamClipArgs a) {
  const long long hop = (long long)gridDim.x * 1024;
  long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4;
  f32x4 p, m, v, g;
  auto fetch = [&](long long at) {
    p = get4<PAST>(a.p + at), m = get4<PAST>(a.m + at), v = get4<PAST>(a.v + at), g = get4<PAST>(a.g + at);
  };
  if (i + 4 <= a.n) fetch(i);          // on their way while the factor is formed
  const float f = clip_factor(a.r);
  for (; i + 4 <= a.n; i += hop) {
    f32x4 pn, mn, vn;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float pe = p[e], me = m[e], ve = v[e];
      adam_update(a.u, g[e] * f, pe, me, ve);
      pn[e] = pe, mn[e] = me, vn[e] = ve;
    }
    if (i + hop + 4 <= a.n) fetch(i + hop);
    put4<PAST>(a.p + i, pn);
    put4<PAST>(a.m + i, mn);
    put4<PAST>(a.v + i, vn);
  }
  for (; i < a.n; ++i) adam_update(a.u, a.g[i] * f, a.p[i], a.m[i], a.v[i]);      // one lane: the last group is not whole
}

// Up to SMALL parameters: one workgroup forms the norm and takes the step, its gradients in registers in between -- one launch instead of
// two (us a call, two launches / one: 100 parameters 10.5 / 6.3, 8192 9.7 / 6.5).
constexpr int SMALL = 8192;
__global__ __launch_bounds__(1024) void adam_clip_small_kernel(AdamClipArgs a) {
  constexpr int Q = SMALL / 4096;
  const int n = (int)a.n, whole = n & ~3, tail = whole + (int)threadIdx.x;      // the last one to three: a lane each
  f32x4 g[Q], p[Q], m[Q], v[Q];
#pragma unroll
  for (int q = 0; q < Q; ++q) {
    const int i = (q * 1024 + (int)threadIdx.x) * 4;
    g[q] = p[q] = m[q] = v[q] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (i < whole) g[q] = get4<false>(a.g + i), p[q] = get4<false>(a.p + i), m[q] = get4<false>(a.m + i), v[q] = get4<false>(a.v + i);
  }
  const float gt = tail < n ? a.g[tail] : 0.f;
  double s = (double)gt * (double)gt;
#pragma unroll
  for (int q = 0; q < Q; ++q)
#pragma unroll
    for (int e = 0; e < 4; ++e) s = fma((double)g[q][e], (double)g[q][e], s);
  const float norm = norm_of(block_join<16>(s, 2), 2);
  if (threadIdx.x == 0) a.r.norm_out[0] = norm;
  const float c = a.r.max_norm / (norm + 1e-6f), f = c > 1.f ? 1.f : c;
#pragma unroll
  for (int q = 0; q < Q; ++q) {
    const int i = (q * 1024 + (int)threadIdx.x) * 4;
    if (i < whole) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float pe = p[q][e], me = m[q][e], ve = v[q][e];
        adam_update(a.u, g[q][e] * f, pe, me, ve);
        p[q][e] = pe, m[q][e] = me, v[q][e] = ve;
      }
      put4<false>(a.p + i, p[q]);
      put4<false>(a.m + i, m[q]);
      put4<false>(a.v + i, v[q]);
    }
  }
  if (tail < n) adam_update(a.u, gt * f, a.p[tail], a.m[tail], a.v[tail]);
}

// One launch's share of the list: spans [from, return value) without the empty ones, at most MAXT
int64_t fill_table(const FdGradSpan* s, int64_t from, int64_t n, SpanTable& t) {
  t.count = 0;
  unsigned long long chunks = 0;
  int64_t i = from;
  for (; i < n && t.count < MAXT; ++i) {
    if (s[i].n == 0) continue;
    const unsigned long long c = (unsigned long long)((s[i].n + CHUNK - 1) / CHUNK);
    if (t.count > 0 && chunks + c >= (1ull << 31)) break;      // a next launch
    t.ptr[t.count] = s[i].ptr;
    t.n_dt[t.count] = s[i].n * 4 + s[i].dtype;
    t.first[t.count] = (unsigned)chunks;
    chunks += c;
    ++t.count;
  }
  t.chunks = (unsigned)chunks;
  return i;
}

int check_spans(const char* what, const FdGradSpan* s, int64_t n) {
  FD_REQUIRE(n >= 0 && (n == 0 || s), "%s: bad list", what);
  for (int64_t i = 0; i < n; ++i) {
    FD_REQUIRE(s[i].n >= 0 && s[i].n < MAXN, "%s: tensor %lld has %lld elements", what, (long long)i, (long long)s[i].n);
    FD_REQUIRE(s[i].dtype == FD_F32 || s[i].dtype == FD_F16 || s[i].dtype == FD_BF16, "%s: tensor %lld has dtype %lld", what, (long long)i,
               (long long)s[i].dtype);
    FD_REQUIRE(s[i].n == 0 || (s[i].ptr && ((uintptr_t)s[i].ptr & (s[i].dtype == FD_F32 ? 3 : 1)) == 0), "%s: tensor %lld is NULL or not aligned to its element", what,
               (long long)i);
  }
  return FD_OK;
}

// Partials of the whole list: fills r (a reference that any consumer can reduce by itself)
int norm_partials(const FdGradSpan* s, int64_t n, int kind, double* partial, int64_t capacity, PartialRef& r, hipStream_t st, bool past = false) {
  NormArgs a;
  a.kind = kind;
  int64_t count = 0;
  for (int64_t i = 0; i < n;) {
    i = fill_table(s, i, n, a.t);
    if (a.t.count == 0) break;
    const unsigned wgs = a.t.chunks < (unsigned)MAXWG ? a.t.chunks : (unsigned)MAXWG;
    FD_REQUIRE(count + wgs + 1 <= capacity, "grad_norm: the workspace holds %lld partials, %lld needed", (long long)capacity, (long long)(count + wgs + 1));
    a.partial = partial + count;
    const int rc = fd_launch(past ? &grad_norm_past_kernel : &grad_norm_kernel, "grad_norm", dim3(wgs), dim3(NT), 0, a, st);
    if (rc != FD_OK) return rc;
    count += wgs;
  }
  r.partial = partial;
  r.count = (int)count;
  r.kind = kind;
  if (count > MAXPART) {
    FinishArgs f{partial, (int)count, kind, partial + count, nullptr};
    const int rc = fd_launch(&norm_finish_kernel, "grad_norm_join", dim3(1), dim3(256), 0, f, st);
    if (rc != FD_OK) return rc;
    r.partial = partial + count;
    r.count = 1;
  }
  return FD_OK;
}

}  // namespace

extern "C" int64_t fdgan_grad_norm_workspace(const FdGradSpan* spans, int64_t nspans) {
  if (nspans < 0 || (nspans > 0 && !spans)) return -1;
  for (int64_t i = 0; i < nspans; ++i)
    if (spans[i].n < 0 || spans[i].n >= MAXN) return -1;
  SpanTable t;
  int64_t count = 1;
  for (int64_t i = 0; i < nspans;) {
    i = fill_table(spans, i, nspans, t);
    count += t.chunks < (unsigned)MAXWG ? t.chunks : (unsigned)MAXWG;
  }
  return count;
}

extern "C" int fdgan_grad_norm(const FdGradSpan* spans, int64_t nspans, int norm_type, double* partial, int64_t capacity, float* norm_out,
                               FdStream stream) {
  FD_REQUIRE(norm_out && partial && capacity >= 1, "grad_norm: NULL output or workspace");
  FD_REQUIRE(norm_type >= 0 && norm_type <= 2, "grad_norm: norm type %d (0: maximum, 1, 2)", norm_type);
  int rc = check_spans("grad_norm", spans, nspans);
  if (rc != FD_OK) return rc;
  hipStream_t st = static_cast<hipStream_t>(stream);
  PartialRef r;
  rc = norm_partials(spans, nspans, norm_type, partial, capacity, r, st);
  if (rc != FD_OK) return rc;
  FinishArgs f{r.partial, r.count, norm_type, nullptr, norm_out};
  return fd_launch(&norm_finish_kernel, "grad_norm_finish", dim3(1), dim3(256), 0, f, st);
}

extern "C" int fdgan_grad_clip(const FdGradSpan* spans, int64_t nspans, int norm_type, float max_norm, double* partial, int64_t capacity,
                               float* norm_out, FdStream stream) {
  FD_REQUIRE(norm_out && partial && capacity >= 1, "grad_clip: NULL output or workspace");
  FD_REQUIRE(norm_type >= 0 && norm_type <= 2, "grad_clip: norm type %d (0: maximum, 1, 2)", norm_type);
  FD_REQUIRE(max_norm >= 0.f, "grad_clip: max_norm %g", (double)max_norm);
  int rc = check_spans("grad_clip", spans, nspans);
  if (rc != FD_OK) return rc;
  hipStream_t st = static_cast<hipStream_t>(stream);
  ScaleArgs a;
  rc = norm_partials(spans, nspans, norm_type, partial, capacity, a.r, st);
  if (rc != FD_OK) return rc;
  a.r.max_norm = max_norm;
  a.r.norm_out = norm_out;
  bool any = false;
  for (int64_t i = 0; i < nspans;) {
    i = fill_table(spans, i, nspans, a.t);
    if (a.t.count == 0) break;
    any = true;
    rc = fd_launch(&grad_scale_kernel, "grad_scale", dim3(a.t.chunks < 1024u ? a.t.chunks : 1024u), dim3(256), 0, a, st);
    if (rc != FD_OK) return rc;
    a.r.norm_out = nullptr;
  }
  if (any) return FD_OK;
  FinishArgs f{partial, 0, norm_type, nullptr, norm_out};      // nothing but empty tensors: the norm is 0
  return fd_launch(&norm_finish_kernel, "grad_norm_finish", dim3(1), dim3(256), 0, f, st);
}

extern "C" int fdgan_adam_step_clipped(float* p, const float* g, float* m, float* v, int64_t n, float lr, double beta1, double beta2, float eps,
                                       int64_t step, float max_norm, double* partial, int64_t capacity, float* norm_out, FdStream stream) {
  FD_REQUIRE(p && g && m && v && n > 0 && step >= 1, "adam_step_clipped: bad arguments");
  FD_REQUIRE((((uintptr_t)p | (uintptr_t)g | (uintptr_t)m | (uintptr_t)v) & 15) == 0, "adam_step_clipped: 16-byte aligned flat tensors");
  FD_REQUIRE(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0, "adam_step_clipped: betas %g, %g (0 <= beta < 1)", beta1, beta2);
  FD_REQUIRE(norm_out && partial && max_norm >= 0.f, "adam_step_clipped: NULL output or workspace, or max_norm %g", (double)max_norm);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const FdGradSpan s{const_cast<float*>(g), n, FD_F32};
  AdamClipArgs a{p, m, v, g, n, adam_constants(lr, beta1, beta2, eps, step), {}};
  int rc = check_spans("adam_step_clipped", &s, 1);
  if (rc == FD_OK && n <= SMALL) {
    FD_REQUIRE(capacity >= fdgan_grad_norm_workspace(&s, 1), "adam_step_clipped: the workspace holds %lld partials", (long long)capacity);
    a.r.max_norm = max_norm;
    a.r.norm_out = norm_out;
    return fd_launch(&adam_clip_small_kernel, "adam_step_clipped", dim3(1), dim3(1024), 0, a, st);
  }
  const bool past = 28 * n > STREAM;
  if (rc == FD_OK) rc = norm_partials(&s, 1, 2, partial, capacity, a.r, st, past);
  if (rc != FD_OK) return rc;
  a.r.max_norm = max_norm;
  a.r.norm_out = norm_out;
  const long long wgs = (n + 1023) / 1024;
  return fd_launch(past ? &adam_clip_kernel<true> : &adam_clip_kernel<false>, "adam_step_clipped", dim3((unsigned)(wgs < 2048 ? wgs : 2048)), dim3(256), 0, a, st);
}
