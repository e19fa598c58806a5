// The k largest logits of vocabulary rows, with their columns and the rows'
// log-sum-exp, for sm_100a.
//
// Values are compared as ordered 32-bit keys (NaN the largest, -0 as 0);
// a column's full key puts its complemented index below, so that keys are
// unique and "largest key" means "largest value, lowest column".
//
// A row streams once through a ring of bulk copies.  On the way each thread
// notes the largest value of every group of columns that it sees (and the
// log-sum-exp).  A threshold that at least k groups' largest values reach is
// reached by at least k columns, all of them in such groups: only those (a
// little over k of thousands) are looked at again.  The columns that reach
// the threshold are ranked by counting.  Rows where too many reach it (long
// ties) collect the columns above it and take the ties in column order;
// should even those be too many, and in rows with NaN or infinities, the k-th
// value is found exactly, by its digits.  Few rows are spread over clusters;
// a cluster's first CTA merges the parts' lists.
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

// Three CTAs an SM of 128 threads with a 48 KB ring (as the losses' sums; a third CTA's lists fit no fourth).
using TopShape = Shape<128, 8, 3, 3>;
constexpr int kTopThreads = TopShape::kGroup;
constexpr int kTopWarps = TopShape::kWarps;
constexpr int kTopCap = 1024;   // candidates a row may have
constexpr int kTopGroups = 24;  // groups a thread notes

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

struct alignas(128) TopShared {
  uint64_t full[TopShape::kSlots], empty[TopShape::kSlots];
  uint64_t keys[kTopCap];
  uint64_t best[PKV_MAX_TOP];             // this CTA's list, largest first
  float tops[kTopGroups][kTopThreads];    // a group's largest value
  RowSum sum[kTopWarps], all;
  int part[2][kTopWarps];
  int hist[256];
  int count, best_n, gave_up;
};

__device__ __forceinline__ void top_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kTopThreads) : "memory"); }

// The sum of v over the threads; `flip` alternates from call to call.
__device__ __forceinline__ int top_sum(int v, int& flip, TopShared& sh) {
  v = __reduce_add_sync(0xffffffffu, v);
  flip ^= 1;
  if ((threadIdx.x & 31) == 0) sh.part[flip][threadIdx.x >> 5] = v;
  top_sync();
  v = 0;
  for (int i = 0; i < kTopWarps; ++i) v += sh.part[flip][i];
  return v;
}

template <typename T>
using TopPart = RowPart<T, TopShape::kChunk>;

// f(column, value) for this thread's vector j of the CTA's part, and for its edge column.
template <typename T, typename F>
__device__ __forceinline__ void vector_columns(const TopPart<T>& p, int j, F f) {
  constexpr int VE = RowSplit<T>::VE;
  float v[VE];
  unpack<T>(p.body()[j], v);
#pragma unroll
  for (int q = 0; q < VE; ++q) f(p.head + (p.v0 + j) * VE + q, v[q]);
}
template <typename T, typename F>
__device__ __forceinline__ void edge_column(const TopPart<T>& p, int edge, F f) {
  if ((int)threadIdx.x < edge) {
    const int c = (int)threadIdx.x < p.head ? threadIdx.x : threadIdx.x + p.nvec * RowSplit<T>::VE;
    f(c, as_float(p.x[c]));
  }
}

// f(column, value) for every column of the CTA's part of the row, in no order.
template <typename T, typename F>
__device__ __forceinline__ void each_column(const TopPart<T>& p, int edge, F f) {
  for (int j = threadIdx.x; j < p.nv; j += kTopThreads) vector_columns<T>(p, j, f);
  edge_column<T>(p, edge, f);
}

__device__ __forceinline__ void take(int c, float v, uint32_t low, TopShared& sh) {
  const uint32_t o = ordered(v);
  if (o >= low) {
    const int at = atomicAdd(&sh.count, 1);
    if (at < kTopCap) sh.keys[at] = (uint64_t)o << 32 | (0xffffffffu - (uint32_t)c);
  }
}

// The columns whose key is at least `low` go into sh.keys (as many as fit); their number.
template <typename T>
__device__ int collect(const TopPart<T>& p, int edge, uint32_t low, TopShared& sh) {
  top_sync();
  if (threadIdx.x == 0) sh.count = 0;
  top_sync();
  each_column<T>(p, edge, [&](int c, float v) { take(c, v, low, sh); });
  top_sync();
  return sh.count;
}

// The k-th largest value's key, digit by digit (0 if there are fewer columns).
template <typename T>
__device__ uint32_t kth_key(const TopPart<T>& p, int edge, int k, TopShared& sh) {
  uint32_t prefix = 0;
  int left = k;
  for (int shift = 24; shift >= 0; shift -= 8) {
    top_sync();
    for (int i = threadIdx.x; i < 256; i += kTopThreads) sh.hist[i] = 0;
    top_sync();
    const uint32_t fixed = shift == 24 ? 0u : 0xffffffffu << (shift + 8);
    each_column<T>(p, edge, [&](int, float v) {
      const uint32_t o = ordered(v);
      if ((o & fixed) != prefix) return;
      // One addition for all lanes with the same digit: rows that come here are full of ties.
      const uint32_t d = (o >> shift) & 255u, lanes = __match_any_sync(__activemask(), d);
      if ((threadIdx.x & 31) == __ffs(lanes) - 1) atomicAdd(&sh.hist[d], __popc(lanes));
    });
    top_sync();
    int d = 255;
    for (; d > 0 && sh.hist[d] < left; --d) left -= sh.hist[d];
    prefix |= (uint32_t)d << shift;
  }
  return prefix;
}

// This CTA's min(k, columns) best columns of its part into sh.best, largest first; their number.
template <typename T>
__device__ int part_list(const TopPart<T>& p, int edge, int k, const RowSum& a, TopShared& sh) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr int VE = RowSplit<T>::VE;
  const int columns = p.nv * VE + edge;
  k = min(k, columns);
  if (k == 0) {
    top_sync();
    return 0;
  }
  const int per = (p.chunks + kTopGroups - 1) / kTopGroups;  // chunks a group spans
  const int groups = per ? (p.chunks + per - 1) / per : 0;
  int flip = 0;
  uint32_t low = 0;
  int m = kTopCap + 1;
  const bool plain = top_sum(a.s == a.s ? 0 : 1, flip, sh) == 0;  // no NaN (of a NaN or infinite column)
  if (plain) {
    // A threshold that k to k + k / 4 + 8 groups reach, if there is one (ties may leave more).  Invariant: at least k
    // groups (or, for -inf, all columns) reach low, fewer than k reach high + 1.
    auto reached = [&](uint32_t key) {
      int c = 0;
      for (int g = 0; g < groups; ++g) c += ordered(sh.tops[g][tid]) >= key;
      return top_sum(c, flip, sh);
    };
    uint32_t high = ordered(INFINITY);
    low = ordered(-INFINITY);
    if (reached(low + 1) >= k) {  // (a group notes -inf where it has no column)
      ++low;
      while (low < high) {
        const uint32_t mid = low + (high - low + 1) / 2;
        const int c = reached(mid);
        if (c >= k) {
          low = mid;
          if (c <= k + k / 4 + 8) break;
        } else {
          high = mid - 1;
        }
      }
      if (tid == 0) sh.count = 0;
      top_sync();
      auto look = [&](int c, float v) { take(c, v, low, sh); };
      for (int g = 0; g < groups; ++g) {
        if (ordered(sh.tops[g][tid]) < low) continue;
        const int j1 = min(p.nv, (g + 1) * per * TopShape::kChunk);
        for (int j = g * per * TopShape::kChunk + tid; j < j1; j += kTopThreads) vector_columns<T>(p, j, look);
      }
      edge_column<T>(p, edge, look);
      top_sync();
      m = sh.count;
    }
    // Too many, or fewer groups than k with a column above -inf: the columns above, then the ties.
    if (m > kTopCap) m = collect<T>(p, edge, low + 1, sh);
  }
  if (m > kTopCap) {
    low = kth_key<T>(p, edge, k, sh);
    m = low == 0xffffffffu ? 0 : collect<T>(p, edge, low + 1, sh);
  }
  if (m < k) {
    // Columns equal to low, the lowest first: the part's body, with the row's edges (all in one CTA) around it.
    const int c0 = edge ? 0 : p.head + p.v0 * VE, c1 = p.head + (p.v0 + p.nv) * VE;
    const int tail = p.head + p.nvec * VE, end = edge ? c1 + (edge - p.head) : c1;
    for (int at0 = c0; at0 < end && m < k; at0 += kTopThreads) {
      const int c = at0 + tid < c1 ? at0 + tid : tail + (at0 + tid - c1);
      const bool tie = at0 + tid < end && ordered(as_float(p.x[c])) == low;
      const uint32_t vote = __ballot_sync(0xffffffffu, tie);
      top_sync();
      if (lane == 0) sh.part[0][warp] = __popc(vote);
      top_sync();
      int at = m + __popc(vote & ((1u << lane) - 1u));
      for (int i = 0; i < kTopWarps; ++i) {
        if (i < warp) at += sh.part[0][i];
        m += sh.part[0][i];
      }
      if (tie && at < k) sh.keys[at] = (uint64_t)low << 32 | (0xffffffffu - (uint32_t)c);
    }
    m = min(m, k);
    top_sync();
  }
  for (int i = tid; i < m; i += kTopThreads) {
    const uint64_t key = sh.keys[i];
    int rank = 0;
    for (int j = 0; j < m; ++j) rank += sh.keys[j] > key;
    if (rank < k) sh.best[rank] = key;
  }
  top_sync();
  return k;
}

// Bound by HBM: the row is read once (16-bit columns: and by the exponentials of its log-sum-exp).
template <typename T>
__global__ void __launch_bounds__(kTopThreads + 32, TopShape::kCtas) top_logits_kernel(const TopArgs A) {
  extern __shared__ __align__(128) uint8_t dyn[];
  uint4* slots = reinterpret_cast<uint4*>(dyn);
  TopShared& sh = *reinterpret_cast<TopShared*>(dyn + TopShape::kRingBytes);
  constexpr int VE = RowSplit<T>::VE;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = cluster_rank(), size = cluster_size();
  if (tid == 0) {
    for (int i = 0; i < TopShape::kSlots; ++i) mbar_init(&sh.full[i], 1), mbar_init(&sh.empty[i], kTopWarps);
    sh.gave_up = 0;
    fence_barrier_init();
  }
  __syncthreads();
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int n = A.batch * A.length, first = blockIdx.x / size, step = gridDim.x / size;
  auto write = [&](int row, const RowSum& a, uint64_t key, int at) {
    const bool bad = *(volatile int*)&sh.gave_up;  // (a wait that ran out: no list)
    A.values[(int64_t)row * A.k + at] = bad ? NAN : unordered((uint32_t)(key >> 32));
    A.tokens[(int64_t)row * A.k + at] = bad ? -1 : (int64_t)(0xffffffffu - (uint32_t)key);
    if (at == 0) {
      const float c = center(a.m, A.ks);
      A.lse[row] = bad ? NAN : (float)((log2_of(a.s) + (far_out(c) ? (double)a.m * A.kd : -(double)c)) * kLn2d);
    }
  };
  if (warp == kTopWarps) {
    if (lane == 0) {
      Ring<TopShape::kSlots> r;
      int filled = 0;
      const uint64_t policy = l2_evict_first_policy();
      for (int row = first; row < n; row += step) {
        const TopPart<T> p(A, row, rank, size);
        for (int c = 0; c < p.chunks; ++c) {
          if (filled == TopShape::kSlots)
            wait_or_mark(&sh.empty[r.slot], r.phase ^ 1, sh);
          else
            ++filled;
          if (*(volatile int*)&sh.gave_up) break;
          const int nv = min(TopShape::kChunk, p.nv - c * TopShape::kChunk);
          mbar_arrive_expect_tx(&sh.full[r.slot], nv * 16);
          bulk_copy_g2s_hint(slots + r.slot * TopShape::kChunk, p.body() + c * TopShape::kChunk, nv * 16, &sh.full[r.slot],
                             policy);
          r.next();
        }
      }
      if (*(volatile int*)&sh.gave_up)  // copies still in flight end before the CTA's shared memory goes
        for (int k = 0; k < TopShape::kSlots; ++k)
          if (k < r.slot || filled == TopShape::kSlots) mbar_wait_bounded(&sh.full[k], k < r.slot ? r.phase : r.phase ^ 1);
    }
  } else {
    Ring<TopShape::kSlots> r;
    for (int row = first; row < n; row += step) {
      const TopPart<T> p(A, row, rank, size);
      const int edge = rank == 0 ? A.vocab - p.nvec * VE : 0;
      const int per = (p.chunks + kTopGroups - 1) / kTopGroups;
      RowSum a{-INFINITY, 0.f, 0.f};
      float top = -INFINITY;
      for (int c = 0; c < p.chunks; ++c) {
        wait_or_mark(&sh.full[r.slot], r.phase, sh);
        const uint4* in = slots + r.slot * TopShape::kChunk;
        const int nv = min(TopShape::kChunk, p.nv - c * TopShape::kChunk);
        if (nv == TopShape::kChunk) {
#pragma unroll
          for (int h = 0; h < TopShape::kVecs; h += 4) {
            uint4 v[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) v[u] = in[tid + (h + u) * kTopThreads];
            top = fmaxf(top, fold_vecs<false, T>(a, v, A.ks));
          }
        } else {
          for (int j = tid; j < nv; j += kTopThreads) {
            const uint4 v[1] = {in[j]};
            top = fmaxf(top, fold_vecs<false, T>(a, v, A.ks));
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.empty[r.slot]);
        r.next();
        if ((c + 1) % per == 0 || c + 1 == p.chunks) {
          sh.tops[c / per][tid] = top;
          top = -INFINITY;
        }
      }
      if (tid < edge) {
        const float f[1] = {as_float(p.x[tid < p.head ? tid : tid + p.nvec * VE])};
        fold<false>(a, f, f[0], A.ks);
      }
      const RowSum w = warp_merge(a, 32, A.ks);
      if (lane == 0) sh.sum[warp] = w;
      const int m = part_list<T>(p, edge, A.k, a, sh);
      RowSum all = sh.sum[0];
      for (int i = 1; i < kTopWarps; ++i) sum_merge(all, sh.sum[i], A.ks);
      if (size == 1) {
        for (int i = tid; i < A.k; i += kTopThreads) write(row, all, sh.best[i], i);
      } else if (tid == 0) {
        sh.all = all;
        sh.best_n = m;
      }
      top_sync();  // (sh.sum and sh.best are read before the next row's)
    }
  }
  if (size == 1) return;
  // A cluster has one row: its first CTA merges the parts' lists, each sorted.  A key's place is the number of keys
  // above it in every list.
  __syncwarp();
  cluster_sync_all();
  if (rank == 0) {
    __shared__ int s_n[kMaxCluster];
    uint64_t* lists = reinterpret_cast<uint64_t*>(dyn);  // (the ring is done)
    RowSum all = sh.all;
    for (int q = 0; q < size; ++q) {
      const TopShared* peer = cluster_peer(&sh, q);
      if (q > 0) sum_merge(all, peer->all, A.ks);
      if (tid == 0) s_n[q] = peer->best_n;
      for (int i = tid; i < peer->best_n; i += kTopThreads + 32) lists[q * PKV_MAX_TOP + i] = peer->best[i];
      if (tid == 0 && peer->gave_up) sh.gave_up = 1;
    }
    __syncthreads();
    for (int i = tid; i < size * A.k; i += kTopThreads + 32) {
      const int q = i / A.k, at = i - q * A.k;
      if (at >= s_n[q]) continue;
      const uint64_t key = lists[q * PKV_MAX_TOP + at];
      int place = at;
      for (int o = 0; o < size; ++o) {
        if (o == q) continue;
        int lo = 0, hi = s_n[o];  // the first index whose key is below
        while (lo < hi) {
          const int mid = (lo + hi) / 2;
          if (lists[o * PKV_MAX_TOP + mid] > key)
            lo = mid + 1;
          else
            hi = mid;
        }
        place += lo;
      }
      if (place < A.k) write(first, all, key, place);
    }
  }
  cluster_sync_all();  // no CTA leaves while the first still reads its list
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
  int sms = 0;
  const int32_t e = sm_count(&sms);
  if (e != PKV_OK) return e;
  TopArgs a{r->logits, r->batch_stride, r->row_stride, r->batch, r->length, r->vocab, k, {0.f, 0.f}, 0.0,
            values_out, tokens_out, lse_out};
  a.ks = scale_for(r->temperature, &a.kd);
  constexpr int kBytes = TopShape::kRingBytes + (int)sizeof(TopShared);
  static_assert((kBytes + 1024 + 64) * TopShape::kCtas <= 233472, "an SM's shared memory");
  static_assert(kMaxCluster * PKV_MAX_TOP * 8 <= TopShape::kRingBytes, "a cluster's lists");
  const int64_t row_bytes = (int64_t)r->vocab * (r->dtype == PKV_F32 ? 4 : 2);
  const int c = row_cluster(n, row_bytes, sms * TopShape::kCtas);
  const int grid = (int)std::min<int64_t>(n, sms * TopShape::kCtas / c) * c;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  auto launch = [&](auto* kernel) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes) != cudaSuccess)
      return cuda_status("top_logits shared memory");
    return launch_after(kernel, grid, kTopThreads + 32, c, kBytes, a, s, "top_logits launch");
  };
  if (r->dtype == PKV_F32) return launch(top_logits_kernel<float>);
  if (r->dtype == PKV_F16) return launch(top_logits_kernel<__half>);
  return launch(top_logits_kernel<__nv_bfloat16>);
}
