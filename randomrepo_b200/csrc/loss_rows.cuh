// Parts shared by the vocabulary-row kernels with f32 / f16 / bf16 logits
// (losses.cu, top_logits.cu): conversions, a row's aligned body, the running
// log-sum-exp of a row.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <string>
#include <type_traits>

#include "pkv_b200.h"
#include "pkv_device.cuh"
#include "pkv_error.h"

namespace pkv {

// PKV_OK, or the status and error message for rows a call named `who` cannot take.
int32_t check_vocab_rows(const pkv_loss_rows* r, const char* who);

namespace {

constexpr double kLn2d = 0.6931471805599453;
constexpr double kLog2ed = 1.4426950408889634;

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// k = log2(e) / T as a pair of floats: one float's error (up to 6e-8 of k) shows in log p as that much of it, and adds
// up in a sequence's sum.  lo > 0, so that a column of -inf stays -inf in x hi + x lo.
struct Scale2 {
  float hi, lo;
};
inline Scale2 scale_for(float temperature, double* kd) {
  const double k = kLog2ed / (double)temperature;
  float hi = (float)k;
  if ((double)hi >= k) hi = nextafterf(hi, 0.f);
  const float lo = (float)(k - (double)hi);
  *kd = (double)hi + (double)lo;
  return Scale2{hi, lo};
}

__device__ __forceinline__ float ex2(float y) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(y));
  return e;
}

// 2^d for d < 127, to 7e-8 of itself: the Taylor series of e^(r ln 2) around the nearest integer, whose next term is 5e-9.
__device__ __forceinline__ float pow2(float d) {
  const float n = rintf(fmaxf(d, -126.f)), r = d - n;
  float p = 1.52527338e-5f;
  p = fmaf(p, r, 1.54035304e-4f);
  p = fmaf(p, r, 1.33335581e-3f);
  p = fmaf(p, r, 9.61812911e-3f);
  p = fmaf(p, r, 5.55041087e-2f);
  p = fmaf(p, r, 0.240226507f);
  p = fmaf(p, r, 0.693147181f);
  return d < -126.f ? 0.f : fmaf(p, r, 1.f) * __int_as_float(((int)n + 127) << 23);
}

// Columns x of a row are taken as y = x k + c, c = -(max x) hi rounded once:
// one fused multiply-add a column, and what is made of y later starts from
// the same c.  Its rounding and max x lo stay in every y, up to 2^-24 + 2^-23
// of c: 18 at 1e8, which the sums hold.  Rows beyond that (masks of -1e9 or a
// type's lowest value everywhere) take y = (x - max x) k.
__device__ __forceinline__ float center(float m, Scale2 k) { return __fmul_rn(-m, k.hi); }  // (rounded: never part of another FMA)
__device__ __forceinline__ bool far_out(float c) { return !(fabsf(c) < 1e8f); }
// The running sums of a set of columns: m near max x, s = sum 2^y, w = sum 2^y y.  D: s between threads, in whose merges
// 32 bits lose 4e-8 of a row's sum (rms).
template <typename D>
struct RowSum {
  D s;
  float m, w;
};

// d: the exponent that takes sums from a reference m to a larger one.
__device__ __forceinline__ float rescale_exponent(float m, float m_new, Scale2 k) {
  const float c = center(m_new, k), from = center(m, k);
  if (!far_out(c) && (!far_out(from) || m == -INFINITY)) return c - from;
  if (far_out(c) && (far_out(from) || m == -INFINITY)) return (m - m_new) * k.hi;
  // One on each side: what stays in c is in the y of one of them alone.
  const float n = far_out(c) ? m : m_new, in_c = far_out(c) ? from : c, stays = fmaf(n, k.lo, fmaf(n, k.hi, in_c));
  return (m - m_new) * k.hi + (far_out(c) ? -stays : stays);
}

template <typename D>
__device__ __forceinline__ void sum_rescale(RowSum<D>& a, float m_new, float d, D f) {
  a.w = f > 0 ? (float)f * fmaf(d, (float)a.s, a.w) : 0.f;  // (a NaN stays in s)
  a.s *= f;
  a.m = m_new;
}

// log2 of a row's sum to about 1e-8: the exponent apart, so that a large sum costs no digits.  The approximate 2^y
// behind the sum is 5e-8 of itself low on average (measured for y from -42 to -1/2; exact at y = 0, at least one
// column's), which would add up in a sequence's log-probability: its share is put back.
__device__ __forceinline__ double log2_sum(float s) {
  int e;
  const float f = frexpf(s, &e);
  return (double)e + (double)log2f(f) + (double)(7.2e-8f * (1.f - 1.f / s));
}
__device__ __forceinline__ double log2_sum(double s) { return log2(s) + 7.2e-8 * (1.0 - 1.0 / s); }

// Columns [0, head) and [head + VE nvec, vocab) of a row are outside its 16-byte-aligned body.
template <typename T>
struct RowSplit {
  static constexpr int VE = 16 / sizeof(T);
  int head, nvec;
  __device__ RowSplit(const T* row, int vocab) {
    head = min(vocab, (int)(((16 - ((uintptr_t)row & 15)) & 15) / sizeof(T)));
    nvec = (vocab - head) / VE;
  }
};

template <typename T>
__device__ __forceinline__ void unpack(uint4 v, float (&f)[16 / sizeof(T)]) {
  if constexpr (sizeof(T) == 4) {
    f[0] = __uint_as_float(v.x);
    f[1] = __uint_as_float(v.y);
    f[2] = __uint_as_float(v.z);
    f[3] = __uint_as_float(v.w);
  } else {
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        f[2 * i] = __uint_as_float(u[i] << 16);
        f[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
      } else {
        const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
        f[2 * i] = p.x;
        f[2 * i + 1] = p.y;
      }
    }
  }
}

template <typename T>
__device__ __forceinline__ uint4 pack(const float (&f)[16 / sizeof(T)]) {
  uint4 v;
  if constexpr (sizeof(T) == 4) {
    v = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  } else {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        const __nv_bfloat162 p = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
        u[i] = *reinterpret_cast<const uint32_t*>(&p);
      } else {
        const __half2 p = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
        u[i] = *reinterpret_cast<const uint32_t*>(&p);
      }
    }
    v = make_uint4(u[0], u[1], u[2], u[3]);
  }
  return v;
}

// Two columns at once (sm_100's packed float32 operations).
using f32x2 = unsigned long long;

__device__ __forceinline__ f32x2 pair(float a, float b) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpair(f32x2 v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// The largest of N columns.  16-bit ones are compared two at a time as they come.
template <typename T, int N>
__device__ __forceinline__ float top_of(const uint4 (&v)[N]) {
  if constexpr (sizeof(T) == 4) {
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < N; ++i)
      m = fmaxf(m, fmaxf(fmaxf(__uint_as_float(v[i].x), __uint_as_float(v[i].y)),
                         fmaxf(__uint_as_float(v[i].z), __uint_as_float(v[i].w))));
    return m;
  } else {
    using T2 = std::conditional_t<std::is_same<T, __half>::value, __half2, __nv_bfloat162>;
    auto as2 = [](const uint32_t& u) { return *reinterpret_cast<const T2*>(&u); };
    T2 m = as2(v[0].x);
#pragma unroll
    for (int i = 0; i < N; ++i) m = __hmax2(m, __hmax2(__hmax2(as2(v[i].x), as2(v[i].y)), __hmax2(as2(v[i].z), as2(v[i].w))));
    return fmaxf(as_float(m.x), as_float(m.y));
  }
}

// The running sums of a thread.  m is a column near the largest so far: as long as no column's 2^y passes 2^20 it
// stays, so that the sums are rarely rescaled.  c is its center, +inf where there is none (no column yet, or far out).
// The lanes of a warp that add whole chunks share their m: their sums then merge without the approximate 2^d.
//
// EXACT: a column that is most of its row must not cost the small ones added after it their digits, nor be an approximate
// 2^y itself (1.1e-7 of the row's sum, rms).  m gives way from 2^4 on, and the sums of the columns that it is taken from
// go to a 64-bit one at once.  (Others are not most of a row: m is the largest of a thousand columns.)
template <bool ENT, bool EXACT = false>
struct Fold {
  static_assert(!(ENT && EXACT), "w is of 32 bits");
  using Sum = std::conditional_t<EXACT, double, float>;
  float m = -INFINITY, c = INFINITY;
  f32x2 s0 = 0ull, s1 = 0ull, w = 0ull;
  double kept = 0.0;

  __device__ __forceinline__ RowSum<float> lanes() const {
    const float2 t = unpair(add2(s0, s1)), u = unpair(w);
    return RowSum<float>{t.x + t.y, m, ENT ? u.x + u.y : 0.f};
  }
  __device__ __forceinline__ RowSum<Sum> sum() const {
    const RowSum<float> a = lanes();
    if constexpr (EXACT) return RowSum<Sum>{(double)a.s + kept, a.m, a.w};
    return RowSum<Sum>{(Sum)a.s, a.m, a.w};
  }

  // Add columns whose largest is `top`.  WHOLE: all lanes of the warp do.
  template <bool WHOLE, int N>
  __device__ __forceinline__ void add(const float (&x)[N], float top, Scale2 k) {
    const bool passed = !(fmaf(top, k.hi, c) <= (EXACT ? 4.f : 20.f));
    const bool refers = WHOLE ? __any_sync(0xffffffffu, passed) : passed;
    if (refers) {
      refer<WHOLE>(x, top, k);
      if (c == INFINITY) return;
    }
    add_columns(x, k);
    if (EXACT && refers) keep();
  }

  // Move the sums to the 64-bit one.
  __device__ __forceinline__ void keep() {
    const float2 a = unpair(add2(s0, s1));
    kept += (double)a.x + (double)a.y;
    s0 = s1 = 0ull;
  }

  // Take a reference of which `top` is within reach.  Far out, with the columns' sums.
  template <bool WHOLE, int N>
  __device__ __forceinline__ void refer(const float (&x)[N], float top, Scale2 k) {
    RowSum<float> a = lanes();
    if (WHOLE) {
      top = fmaxf(top, m);
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
    }
    if (!(top > -INFINITY)) {  // nothing but -inf, or NaN
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (x[i] != x[i]) a.s = NAN;
    } else {
      if (top > m) {
        const float d = rescale_exponent(m, top, k), f = EXACT ? pow2(d) : ex2(d);
        sum_rescale(a, top, d, f);
        if (EXACT) kept *= (double)f;
      }
      m = a.m;
      const float at = center(m, k);
      c = far_out(at) ? INFINITY : at;
      if (far_out(at)) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float y = (x[i] - m) * k.hi, e = ex2(y);
          a.s += e;
          if (ENT) a.w = fmaf(e, fmaxf(y, -1e30f), a.w);
        }
      }
    }
    s0 = pair(EXACT ? 0.f : a.s, 0.f), s1 = 0ull, w = pair(a.w, 0.f);
    if (EXACT && a.s != 0.f) kept += (double)a.s;
  }

  template <int N>
  __device__ __forceinline__ void add_columns(const float (&x)[N], Scale2 k) {
    if constexpr (N == 1) {
      const float y = fmaf(x[0], k.lo, fmaf(x[0], k.hi, c));
      const float e = ex2(y);
      s0 = add2(s0, pair(e, 0.f));
      if (ENT) w = add2(w, pair(e * fmaxf(y, -1e30f), 0.f));
    } else {
      static_assert(N % 4 == 0, "columns go in pairs, to two sums");
      const f32x2 cc = pair(c, c), hi = pair(k.hi, k.hi), lo = pair(k.lo, k.lo);
#pragma unroll
      for (int i = 0; i < N; i += 2) {
        const f32x2 xx = pair(x[i], x[i + 1]);
        const float2 y = unpair(fma2(xx, lo, fma2(xx, hi, cc)));
        const f32x2 e = pair(ex2(y.x), ex2(y.y));
        if (i & 2)
          s1 = add2(s1, e);
        else
          s0 = add2(s0, e);
        if (ENT) w = fma2(e, pair(fmaxf(y.x, -1e30f), fmaxf(y.y, -1e30f)), w);
      }
    }
  }

  // Add N vectors of a row's body; their largest column.
  template <bool WHOLE, typename T, int N>
  __device__ __forceinline__ float add_vecs(const uint4 (&v)[N], Scale2 k) {
    constexpr int VE = 16 / sizeof(T);
    float f[N * VE];
#pragma unroll
    for (int i = 0; i < N; ++i) unpack<T>(v[i], *reinterpret_cast<float (*)[VE]>(f + i * VE));
    const float top = top_of<T>(v);
    add<WHOLE>(f, top, k);
    return top;
  }
};

// ---------------------------------------------------------------------------
// Rows through a shared-memory ring, by a CTA or a cluster.

constexpr int kMaxCluster = 8;

// Shape of a launch: threads that work on the columns, 16-byte vectors of a ring slot each takes, ring slots, CTAs an SM.
template <int THREADS, int VECS, int SLOTS, int CTAS>
struct Shape {
  static constexpr int kGroup = THREADS, kVecs = VECS, kSlots = SLOTS, kCtas = CTAS;
  static constexpr int kChunk = VECS * THREADS;  // vectors of a slot
  static constexpr int kWarps = THREADS / 32;
  static constexpr int kCopyWarp = kWarps, kTeacherWarp = kWarps + 1, kTermsWarp = kWarps + 2;
  static constexpr int kThreads = THREADS + 96;
  static constexpr int kRingBytes = SLOTS * kChunk * 16;
};
// mbar_try_wait that also sees what other CTAs of the cluster sent.
__device__ __forceinline__ bool mbar_try_wait_cluster(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}

// Waits are bounded.  One that gives up marks the CTA: every later wait of it passes at once, so that all roles run
// to their ends (their barriers included) and the loss is made NaN.
template <bool CLUSTER = false, typename Sh>
__device__ __forceinline__ void wait_or_mark(uint64_t* bar, uint32_t parity, Sh& sh) {
  auto passed = [&] { return CLUSTER ? mbar_try_wait_cluster(bar, parity) : mbar_try_wait(bar, parity); };
  if (passed()) return;
  const long long start = clock64();
  while (!passed()) {
    if (*(volatile int*)&sh.gave_up) return;
    if (clock64() - start > kWaitLimitCycles) {
      *(volatile int*)&sh.gave_up = 1;
      return;
    }
  }
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// The same shared-memory object of CTA `rank` of the cluster.
template <typename T>
__device__ __forceinline__ const T* cluster_peer(const T* p, uint32_t rank) {
  uint64_t q;
  asm("mapa.u64 %0, %1, %2;" : "=l"(q) : "l"(reinterpret_cast<uint64_t>(p)), "r"(rank));
  return reinterpret_cast<const T*>(q);
}

__device__ __forceinline__ double warp_sum_d(double v) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}

// The sums of `width` lanes (a power of two), on a common reference.  The factors are exact ones: the approximate 2^d is
// 5e-8 low on average, and a row's sum passes here up to three times.
template <typename D>
__device__ __forceinline__ RowSum<D> warp_merge(RowSum<D> a, int width, Scale2 k) {
  float m = a.m;
  for (int off = width / 2; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
  if (a.m != m) {  // (no column anywhere: s is 0, or the NaN of a NaN column)
    const float d = rescale_exponent(a.m, m, k);
    sum_rescale(a, m, d, (D)exp2((double)d));
  }
  for (int off = width / 2; off > 0; off >>= 1) {
    a.s += __shfl_xor_sync(0xffffffffu, a.s, off);
    a.w += __shfl_xor_sync(0xffffffffu, a.w, off);
  }
  return a;
}

// A row's place in memory and the part of it this CTA of its cluster has.
template <typename T, int CHUNK>
struct RowPart {
  int row, b, t;
  const T* x;
  int head, nvec;      // the row's aligned body, in vectors
  int v0, nv, chunks;  // this CTA's vectors
  template <typename Args>
  __device__ RowPart(const Args& A, int row_, int rank, int size) {
    row = row_;
    b = row / A.length, t = row - b * A.length;
    x = (const T*)A.x + b * A.xb + t * A.xr;
    const RowSplit<T> sp(x, A.vocab);
    head = sp.head, nvec = sp.nvec;
    const int per = (nvec + size - 1) / size;
    v0 = min(nvec, rank * per);
    nv = min(nvec, v0 + per) - v0;
    chunks = (nv + CHUNK - 1) / CHUNK;
  }
  __device__ const uint4* body() const { return reinterpret_cast<const uint4*>(x + head) + v0; }
};

// A place in the ring.  Slots are filled, looked at and freed strictly in turn: a row's chunks 0 .. n-1, and, where
// the row is needed twice, the last min(n, SLOTS) of them stay in their slots for the second time, which takes them
// first; then, behind those, the others again (from L2).
template <int SLOTS>
struct Ring {
  int slot = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next() {
    if (++slot == SLOTS) slot = 0, phase ^= 1;
  }
  __device__ __forceinline__ void back(int n) {  // n <= SLOTS
    slot -= n;
    if (slot < 0) slot += SLOTS, phase ^= 1;
  }
};

// ---------------------------------------------------------------------------
// Host.

inline int32_t fail(int32_t status, const std::string& msg) {
  pkv_set_error(msg);
  return status;
}

inline int32_t cuda_status(const char* what) {
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) return PKV_OK;
  return fail(PKV_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
}

inline int32_t sm_count(int* sms) {
  static int counts[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return cuda_status("device query");
  if (dev < 64 && counts[dev]) {
    *sms = counts[dev];
    return PKV_OK;
  }
  if (cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return cuda_status("device query");
  if (dev < 64) counts[dev] = *sms;
  return PKV_OK;
}

// Launch `kernel` behind the kernel before it on the stream (it waits for that one itself).
template <typename K, typename Args>
int32_t launch_after(K kernel, int grid, int threads, int cluster, int smem, const Args& a, cudaStream_t st,
                     const char* what) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = cluster, at[1].val.clusterDim.y = 1, at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  cudaLaunchKernelEx(&cfg, kernel, a);
  return cuda_status(what);
}

// CTAs that share a row: few rows are spread over the SMs by columns, as long as a CTA keeps at least 16 KB.
inline int row_cluster(int64_t rows, int64_t row_bytes, int ctas) {
  int c = 1;
  while (c < kMaxCluster && rows * (2 * c) <= ctas && row_bytes / (2 * c) >= 16384) c *= 2;
  return c;
}

}  // namespace
}  // namespace pkv
