// The k largest logits of vocabulary rows, with their columns and the rows'
// log-sum-exp, for sm_100a.
//
// Values are compared as ordered 32-bit keys (NaN the largest, -0 as 0);
// a column's full key puts its complemented index below, so that keys are
// unique and "largest key" means "largest value, lowest column".
//
// A CTA takes a row.  Its first pass keeps each thread's largest key (and the
// log-sum-exp); a threshold that at least k threads' maxima reach is reached
// by at least k columns, so the second pass collects the columns that reach
// it -- little more than k of them on ordinary rows, since the threshold is
// near the k-th largest of kTopThreads group maxima -- and ranks them by
// counting.  Rows where too many reach it (long ties, runs of large values in
// few threads' columns) collect the columns above it and take the ties in
// column order; should even those be too many, the k-th value is found
// exactly, by its digits.
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <string>

#include "loss_rows.cuh"
#include "pkv_b200.h"
#include "pkv_error.h"

namespace pkv {
namespace {

constexpr int kTopThreads = 512;
constexpr int kTopWarps = kTopThreads / 32;
constexpr int kTopCap = 2048;  // candidates a row may have

struct TopArgs {
  const void* x;
  int64_t xb, xr;
  int32_t batch, length, vocab, k;
  Scale2 ks;
  double kd;
  float* values;
  int64_t* tokens;
  float* lse;
};

__device__ __forceinline__ uint32_t ordered(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ float unordered(uint32_t o) {
  if (o == 0xffffffffu) return __uint_as_float(0x7fffffffu);
  return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}

struct TopShared {
  uint64_t keys[kTopCap];
  RowSum sum[kTopWarps];
  uint32_t part[2 * kTopWarps];
  int hist[256];
  int count, base;
};

// f(column, value) for every column of the row, in no order.
template <typename T, typename F>
__device__ __forceinline__ void each_column(const T* x, const RowSplit<T>& sp, int vocab, F f) {
  constexpr int VE = RowSplit<T>::VE;
  const uint4* body = reinterpret_cast<const uint4*>(x + sp.head);
  for (int j = threadIdx.x; j < sp.nvec; j += kTopThreads) {
    float v[VE];
    unpack<T>(body[j], v);
#pragma unroll
    for (int q = 0; q < VE; ++q) f(sp.head + j * VE + q, v[q]);
  }
  const int edge = vocab - sp.nvec * VE;
  if ((int)threadIdx.x < edge) {
    const int c = (int)threadIdx.x < sp.head ? threadIdx.x : threadIdx.x + sp.nvec * VE;
    f(c, as_float(x[c]));
  }
}

// The columns whose key is at least `low` go into sh.keys (as many as fit); their number.
template <typename T>
__device__ int collect(const T* x, const RowSplit<T>& sp, int vocab, uint32_t low, TopShared& sh) {
  __syncthreads();
  if (threadIdx.x == 0) sh.count = 0;
  __syncthreads();
  each_column<T>(x, sp, vocab, [&](int c, float v) {
    const uint32_t o = ordered(v);
    if (o >= low) {
      const int at = atomicAdd(&sh.count, 1);
      if (at < kTopCap) sh.keys[at] = (uint64_t)o << 32 | (0xffffffffu - (uint32_t)c);
    }
  });
  __syncthreads();
  return sh.count;
}

// The k-th largest value's key, digit by digit.
template <typename T>
__device__ uint32_t kth_key(const T* x, const RowSplit<T>& sp, int vocab, int k, TopShared& sh) {
  uint32_t prefix = 0;
  int left = k;
  for (int shift = 24; shift >= 0; shift -= 8) {
    __syncthreads();
    for (int i = threadIdx.x; i < 256; i += kTopThreads) sh.hist[i] = 0;
    __syncthreads();
    const uint32_t fixed = shift == 24 ? 0u : 0xffffffffu << (shift + 8);
    each_column<T>(x, sp, vocab, [&](int, float v) {
      const uint32_t o = ordered(v);
      if ((o & fixed) != prefix) return;
      // One addition for all lanes with the same digit: rows that come here are full of ties.
      const uint32_t d = (o >> shift) & 255u, lanes = __match_any_sync(__activemask(), d);
      if ((threadIdx.x & 31) == __ffs(lanes) - 1) atomicAdd(&sh.hist[d], __popc(lanes));
    });
    __syncthreads();
    int d = 255;
    for (; d > 0 && sh.hist[d] < left; --d) left -= sh.hist[d];
    prefix |= (uint32_t)d << shift;
  }
  return prefix;
}

template <typename T>
__global__ void __launch_bounds__(kTopThreads) top_logits_kernel(const TopArgs A) {
  __shared__ TopShared sh;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int n = A.batch * A.length;
  for (int row = blockIdx.x; row < n; row += gridDim.x) {
    const int b = row / A.length, t = row - b * A.length;
    const T* x = (const T*)A.x + b * A.xb + t * A.xr;
    const RowSplit<T> sp(x, A.vocab);
    RowSum r{-INFINITY, 0.f, 0.f};
    uint32_t top = 0;
    constexpr int VE = RowSplit<T>::VE;
    const uint4* body = reinterpret_cast<const uint4*>(x + sp.head);
    for (int j = tid; j < sp.nvec; j += kTopThreads) {
      float v[VE];
      unpack<T>(body[j], v);
      const uint4 raw[1] = {body[j]};
      fold_vecs<false, T>(r, raw, A.ks);
#pragma unroll
      for (int q = 0; q < VE; ++q) top = max(top, ordered(v[q]));
    }
    const int edge = A.vocab - sp.nvec * VE;
    if (tid < edge) {
      const float v[1] = {as_float(x[tid < sp.head ? tid : tid + sp.nvec * VE])};
      fold<false>(r, v, v[0], A.ks);
      top = max(top, ordered(v[0]));
    }
    // The log-sum-exp, and the range of the threads' maxima.
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
      RowSum o;
      o.m = __shfl_xor_sync(0xffffffffu, r.m, off);
      o.s = __shfl_xor_sync(0xffffffffu, r.s, off);
      o.w = 0.f;
      sum_merge(r, o, A.ks);
    }
    const uint32_t hi_w = __reduce_max_sync(0xffffffffu, top), lo_w = __reduce_min_sync(0xffffffffu, top);
    __syncthreads();
    if (lane == 0) {
      sh.sum[warp] = r;
      sh.part[warp] = hi_w;
      sh.part[kTopWarps + warp] = lo_w;
    }
    __syncthreads();
    uint32_t lo = 0xffffffffu, hi = 0;
    r = sh.sum[0];
    for (int i = 1; i < kTopWarps; ++i) sum_merge(r, sh.sum[i], A.ks);
    for (int i = 0; i < kTopWarps; ++i) hi = max(hi, sh.part[i]), lo = min(lo, sh.part[kTopWarps + i]);
    // A threshold that k to k + k/4 + 8 threads' maxima reach, if there is one (ties may leave more).
    // Invariant: at least k maxima reach lo (or lo = 0, which every column does), fewer than k reach hi + 1.
    if (__syncthreads_count(top >= lo && top > 0) < A.k) lo = 0;
    while (lo < hi) {
      const uint32_t mid = lo + (hi - lo + 1) / 2;
      const int c = __syncthreads_count(top >= mid);
      if (c >= A.k) {
        lo = mid;
        if (c <= A.k + A.k / 4 + 8) break;
      } else {
        hi = mid - 1;
      }
    }
    int m = collect<T>(x, sp, A.vocab, lo, sh);
    if (m > kTopCap) {
      m = lo == 0xffffffffu ? 0 : collect<T>(x, sp, A.vocab, lo + 1, sh);
      if (m > kTopCap) {
        lo = kth_key<T>(x, sp, A.vocab, A.k, sh);
        m = lo == 0xffffffffu ? 0 : collect<T>(x, sp, A.vocab, lo + 1, sh);
      }
      const int m0 = m;
      // Columns equal to lo, the lowest first.
      for (int c0 = 0; c0 < A.vocab && m < A.k; c0 += kTopThreads) {
        const int c = c0 + tid;
        const bool tie = c < A.vocab && ordered(as_float(x[c])) == lo;
        const uint32_t vote = __ballot_sync(0xffffffffu, tie);
        __syncthreads();
        if (lane == 0) sh.part[warp] = __popc(vote);
        __syncthreads();
        int at = m + __popc(vote & ((1u << lane) - 1u));
        for (int i = 0; i < kTopWarps; ++i) {
          if (i < warp) at += sh.part[i];
          m += sh.part[i];
        }
        if (tie && at < A.k) sh.keys[at] = (uint64_t)lo << 32 | (0xffffffffu - (uint32_t)c);
      }
      if (m0 < A.k) m = min(m, A.k);
    }
    __syncthreads();
    for (int i = tid; i < m; i += kTopThreads) {
      const uint64_t key = sh.keys[i];
      int rank = 0;
      for (int j = 0; j < m; ++j) rank += sh.keys[j] > key;
      if (rank < A.k) {
        A.values[(int64_t)row * A.k + rank] = unordered((uint32_t)(key >> 32));
        A.tokens[(int64_t)row * A.k + rank] = (int64_t)(0xffffffffu - (uint32_t)key);
      }
    }
    if (tid == 0) A.lse[row] = (float)((log2_of(r.s) + (far_out(center(r.m, A.ks)) ? (double)r.m * A.kd : -(double)center(r.m, A.ks))) * kLn2d);
    __syncthreads();
  }
}

}  // namespace
}  // namespace pkv

using namespace pkv;

extern "C" int32_t pkv_top_logits(const pkv_loss_rows* r, int32_t k, float* values_out, int64_t* tokens_out,
                                  float* lse_out, void* stream) {
  pkv_clear_error();
  const int32_t st = check_vocab_rows(r, "top_logits");
  if (st != PKV_OK) return st;
  if (k < 1 || k > PKV_MAX_TOP || k > r->vocab) {
    pkv_set_error("top_logits: k must be from 1 to min(vocab, 256)");
    return PKV_ERR_ARG;
  }
  const int64_t n = (int64_t)r->batch * r->length;
  if (n == 0) return PKV_OK;
  if (!values_out || !tokens_out || !lse_out) {
    pkv_set_error("top_logits: value, token and log-sum-exp outputs are required");
    return PKV_ERR_ARG;
  }
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) {
    pkv_set_error("top_logits: device query failed");
    return PKV_ERR_CUDA;
  }
  TopArgs a{r->logits, r->batch_stride, r->row_stride, r->batch, r->length, r->vocab, k, {0.f, 0.f}, 0.0,
            values_out, tokens_out, lse_out};
  a.ks = scale_for(r->temperature, &a.kd);
  const int grid = (int)std::min<int64_t>(n, 4ll * sms);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (r->dtype == PKV_F32)
    top_logits_kernel<float><<<grid, kTopThreads, 0, s>>>(a);
  else if (r->dtype == PKV_F16)
    top_logits_kernel<__half><<<grid, kTopThreads, 0, s>>>(a);
  else
    top_logits_kernel<__nv_bfloat16><<<grid, kTopThreads, 0, s>>>(a);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    pkv_set_error(std::string("top_logits launch: ") + cudaGetErrorString(e));
    return PKV_ERR_CUDA;
  }
  return PKV_OK;
}
