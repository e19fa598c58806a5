// Parts shared by the vocabulary-row kernels with f32 / f16 / bf16 logits
// (losses.cu, top_logits.cu): conversions, a row's aligned body, the running
// log-sum-exp of a row.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "pkv_b200.h"

namespace pkv {

// PKV_OK, or the status and error message for rows a call named `who` cannot take.
int32_t check_vocab_rows(const pkv_loss_rows* r, const char* who);

constexpr double kLn2d = 0.6931471805599453;
constexpr double kLog2ed = 1.4426950408889634;

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// k = log2(e) / T, as a pair of floats where one is off by more than 2e-8 of
// it (at T = 1 it is not): a sum over many columns shows the scale's error as
// that much of log p, which is up to about 20.
struct Scale2 {
  float hi, lo;
};
inline Scale2 scale_for(float temperature, double* kd) {
  const double k = kLog2ed / (double)temperature;
  Scale2 s{(float)k, 0.f};
  if ((double)s.hi > k) s.hi = nextafterf(s.hi, 0.f);  // lo >= 0: a column of -inf stays -inf in x hi + x lo
  if (k - (double)s.hi > 2e-8 * k) s.lo = (float)(k - (double)s.hi);
  *kd = (double)s.hi + (double)s.lo;
  return s;
}

__device__ __forceinline__ float ex2(float y) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(y));
  return e;
}

// Columns x of a row are taken as y = x k + c, c = -(max x) k rounded once:
// one fused multiply-add a column, and what is made of y later starts from
// the same c.  Where max x k leaves the range in which that is safe (masks of
// a type's lowest value everywhere), y = (x - max x) k.
__device__ __forceinline__ float center(float m, Scale2 k) { return __fmul_rn(-m, k.hi); }  // (rounded: never part of another FMA)
__device__ __forceinline__ bool far_out(float c) { return !(fabsf(c) < 1e30f); }
// The running sums of a set of columns: m = max x, s = sum 2^y, w = sum 2^y y.
struct RowSum {
  float m, s, w;
};

__device__ __forceinline__ void sum_rescale(RowSum& a, float m_new, Scale2 k) {
  const float c = center(m_new, k);
  const float d = far_out(c) ? (a.m - m_new) * k.hi : c - center(a.m, k), f = ex2(d);
  a.w = f > 0.f ? f * fmaf(d, a.s, a.w) : 0.f;  // (a NaN stays in s)
  a.s *= f;
  a.m = m_new;
}

__device__ __forceinline__ void sum_merge(RowSum& a, RowSum b, Scale2 k) {
  const float mn = fmaxf(a.m, b.m);
  if (mn == -INFINITY) {
    a.s += b.s;  // 0, or the NaN of a NaN column
    return;
  }
  // (the larger one's factor is 2^0: exact)
  sum_rescale(a, mn, k);
  sum_rescale(b, mn, k);
  a.s += b.s;
  a.w += b.w;
}

// log2 of a positive float to about 1e-7 absolute: the exponent apart, so that a large sum costs no digits.
__device__ __forceinline__ double log2_of(float s) {
  int e;
  const float f = frexpf(s, &e);
  return (double)e + (double)log2f(f);
}

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

// Add columns whose largest is `top` to the running sums.  LO: the scale has a second float.
template <bool ENT, bool LO, int N>
__device__ __forceinline__ void fold_near(RowSum& a, const float (&x)[N], float c, Scale2 k) {
  if constexpr (N == 1) {
    float y = fmaf(x[0], k.hi, c);
    if (LO) y = fmaf(x[0], k.lo, y);
    const float e = ex2(y);
    a.s += e;
    if (ENT) a.w = fmaf(e, fmaxf(y, -1e30f), a.w);
  } else {
    static_assert(N % 2 == 0, "columns go in pairs");
    const f32x2 cc = pair(c, c), hi = pair(k.hi, k.hi), lo = pair(k.lo, k.lo);
    f32x2 s[2] = {pair(a.s, 0.f), 0ull}, w = pair(a.w, 0.f);
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const f32x2 xx = pair(x[i], x[i + 1]);
      f32x2 y2 = fma2(xx, hi, cc);
      if (LO) y2 = fma2(xx, lo, y2);
      const float2 y = unpair(y2);
      const f32x2 e = pair(ex2(y.x), ex2(y.y));
      s[(i / 2) & 1] = add2(s[(i / 2) & 1], e);
      if (ENT) w = fma2(e, pair(fmaxf(y.x, -1e30f), fmaxf(y.y, -1e30f)), w);
    }
    const float2 t = unpair(add2(s[0], s[1])), u = unpair(w);
    a.s = t.x + t.y;
    if (ENT) a.w = u.x + u.y;
  }
}

template <bool ENT, int N>
__device__ __forceinline__ void fold(RowSum& a, const float (&x)[N], float top, Scale2 k) {
  if (!(top > -INFINITY)) {  // nothing but -inf, or NaN
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (x[i] != x[i]) a.s = NAN;
    return;
  }
  if (top > a.m) sum_rescale(a, top, k);
  const float c = center(a.m, k);
  if (far_out(c)) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float y = (x[i] - a.m) * k.hi, e = ex2(y);
      a.s += e;
      if (ENT) a.w = fmaf(e, fmaxf(y, -1e30f), a.w);
    }
  } else if (k.lo == 0.f) {
    fold_near<ENT, false>(a, x, c, k);
  } else {
    fold_near<ENT, true>(a, x, c, k);
  }
}

// N vectors of a row's body.
template <bool ENT, typename T, int N>
__device__ __forceinline__ void fold_vecs(RowSum& a, const uint4 (&v)[N], Scale2 k) {
  constexpr int VE = 16 / sizeof(T);
  float f[N * VE];
#pragma unroll
  for (int i = 0; i < N; ++i) unpack<T>(v[i], *reinterpret_cast<float (*)[VE]>(f + i * VE));
  fold<ENT>(a, f, top_of<T>(v), k);
}

}  // namespace pkv
