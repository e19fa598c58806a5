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
#include <float.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <string>

#include "loss_rows.cuh"
#include "pkv_b200.h"
#include "pkv_error.h"

namespace pkv {
namespace {

// Two CTAs an SM: 256 threads read the columns, 128 pick the row before.  4 096 rows of 151 936 16-bit columns and
// k = 64 take 295 us.  (One group doing both was slower, 391 us against 341 with the picking of that time, since the
// columns waited for each row's picking.)
using TopShape = Shape<256, 4, 4, 2>;
constexpr int kTopThreads = TopShape::kGroup;
constexpr int kTopWarps = TopShape::kWarps;
constexpr int kPickThreads = 128;
constexpr int kPickWarps = kPickThreads / 32;
constexpr int kTopCta = kTopThreads + kPickThreads + 32;
constexpr int kTopCap = 1024;   // candidates a row may have
constexpr int kTopGroups = 12;  // groups a thread notes

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
  uint64_t full[TopShape::kSlots], empty[TopShape::kSlots], row_full[2], row_empty[2];
  alignas(16) uint64_t keys[kTopCap];
  uint64_t best[PKV_MAX_TOP];                 // this CTA's list, largest first
  alignas(16) float tops[2][kTopGroups][kTopThreads];  // a group's largest value
  RowSum<float> sum[2][kTopWarps], all;
  uint16_t hits[kTopCap];                     // groups that reach the threshold
  float4 range[kPickWarps];
  uint32_t part[kPickWarps];
  int hist[256];
  int count, n_hits, best_n, gave_up;
};

// The threads that pick; `pick_id` is a thread's place among them.
__device__ __forceinline__ void pick_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kPickThreads) : "memory"); }
__device__ __forceinline__ int pick_id() { return (int)threadIdx.x - kTopThreads; }

// The least lo, the largest hi and the sum of n over them.
__device__ __forceinline__ void pick_range(float& lo, float& hi, int& n, TopShared& sh) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, off));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, off));
  }
  n = __reduce_add_sync(0xffffffffu, n);
  if ((threadIdx.x & 31) == 0) sh.range[pick_id() >> 5] = make_float4(lo, hi, __int_as_float(n), 0.f);
  pick_sync();
  n = 0;
  for (int i = 0; i < kPickWarps; ++i) {
    const float4 v = sh.range[i];
    lo = fminf(lo, v.x), hi = fmaxf(hi, v.y), n += __float_as_int(v.z);
  }
}

template <typename T>
using TopPart = RowPart<T, TopShape::kChunk>;

// log2 of the chunks that a group of the part spans.
template <typename T>
__device__ __forceinline__ int group_shift(const TopPart<T>& p) {
  const int per = (p.chunks + kTopGroups - 1) / kTopGroups;
  return per > 1 ? 32 - __clz(per - 1) : 0;
}

// A part of less than a chunk: its vectors go round the threads, so that there are more groups.
template <typename T>
__device__ __forceinline__ bool lone_chunk(const TopPart<T>& p) { return p.nv < TopShape::kChunk; }

// f(column, value) for the columns of vector at(i) (< 0: none) of the CTA's part, i = pick_id(), + kPickThreads, ...
// below n, where the vector's largest value is not below `from` (NaN: all of them).  BATCH vectors are on their way at
// once (f's writes would keep a loop's loads apart).
template <typename T, int BATCH, typename At, typename F>
__device__ __forceinline__ void vectors(const TopPart<T>& p, int n, At at, float from, F f) {
  constexpr int VE = RowSplit<T>::VE;
  for (int i0 = pick_id(); i0 < n; i0 += BATCH * kPickThreads) {
    uint4 v[BATCH];
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      const int i = i0 + u * kPickThreads, j = i < n ? at(i) : -1;
      v[u] = make_uint4(0u, 0u, 0u, 0u);
      if (j >= 0) v[u] = p.body()[j];
    }
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      const uint4 one[1] = {v[u]};
      const int i = i0 + u * kPickThreads;
      if (i >= n || top_of<T>(one) < from) continue;
      const int j = at(i);
      if (j < 0) continue;
      float x[VE];
      unpack<T>(v[u], x);
#pragma unroll
      for (int q = 0; q < VE; ++q) f(p.head + (p.v0 + j) * VE + q, x[q]);
    }
  }
}
template <typename T, typename F>
__device__ __forceinline__ void edge_column(const TopPart<T>& p, int edge, F f) {
  if (pick_id() < edge) {
    const int c = pick_id() < p.head ? pick_id() : pick_id() + p.nvec * RowSplit<T>::VE;
    f(c, as_float(p.x[c]));
  }
}

// f(column, value) for every column of the CTA's part of the row, in no order.
template <typename T, typename F>
__device__ __forceinline__ void each_column(const TopPart<T>& p, int edge, F f) {
  vectors<T, 4>(p, p.nv, [](int i) { return i; }, NAN, f);
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
__device__ __noinline__ int collect(const TopPart<T>& p, int edge, uint32_t low, TopShared& sh) {
  pick_sync();
  if (pick_id() == 0) sh.count = 0;
  pick_sync();
  each_column<T>(p, edge, [&](int c, float v) { take(c, v, low, sh); });
  pick_sync();
  return sh.count;
}

// The k-th largest value's key, digit by digit (0 if there are fewer columns).
template <typename T>
__device__ __noinline__ uint32_t kth_key(const TopPart<T>& p, int edge, int k, TopShared& sh) {
  uint32_t prefix = 0;
  int left = k;
  for (int shift = 24; shift >= 0; shift -= 8) {
    pick_sync();
    for (int i = pick_id(); i < 256; i += kPickThreads) sh.hist[i] = 0;
    pick_sync();
    const uint32_t fixed = shift == 24 ? 0u : 0xffffffffu << (shift + 8);
    each_column<T>(p, edge, [&](int, float v) {
      const uint32_t o = ordered(v);
      if ((o & fixed) != prefix) return;
      // One addition for all lanes with the same digit: rows that come here are full of ties.
      const uint32_t d = (o >> shift) & 255u, lanes = __match_any_sync(__activemask(), d);
      if ((threadIdx.x & 31) == __ffs(lanes) - 1) atomicAdd(&sh.hist[d], __popc(lanes));
    });
    pick_sync();
    int d = 255;
    for (; d > 0 && sh.hist[d] < left; --d) left -= sh.hist[d];
    prefix |= (uint32_t)d << shift;
  }
  return prefix;
}

// This CTA's min(k, columns) best columns of its part into sh.best, largest first; their number.  `plain`: no column is
// NaN or +inf.
template <typename T>
__device__ __forceinline__ int part_list(const TopPart<T>& p, int edge, int k, bool plain, int par, TopShared& sh) {
  const int tid = pick_id(), lane = tid & 31, warp = tid >> 5;
  constexpr int VE = RowSplit<T>::VE;
  const int columns = p.nv * VE + edge;
  k = min(k, columns);
  if (k == 0) {
    pick_sync();
    return 0;
  }
  const int shift = group_shift<T>(p), groups = (p.chunks + (1 << shift) - 1) >> shift;
  uint32_t low = 0;
  int m = kTopCap + 1;
  if (plain) {
    // The threshold is one that k to k + k / 2 + 16 groups reach, if ties allow it, from a histogram of the groups'
    // values between `lo`, which at least k groups reach (the least of 128 or 512 maxima, each over some of a
    // thread's groups), and the largest; the bin that holds the k-th is cut again while it is too full.
    // (Every instruction of these few warps is waited for: the groups' values are read four at a time.)
    constexpr int kReads = kTopGroups * kTopThreads / (4 * kPickThreads);
    const float4* tops = reinterpret_cast<const float4*>(sh.tops[par]);
    const int reads = (groups * kTopThreads / 4 - tid + kPickThreads - 1) / kPickThreads;
    auto each_top = [&](auto f) {
#pragma unroll 6
      for (int r = 0; r < reads; ++r) {
        const float4 v = tops[r * kPickThreads + tid];
        f(v.x, 4 * (r * kPickThreads + tid)), f(v.y, 4 * (r * kPickThreads + tid) + 1);
        f(v.z, 4 * (r * kPickThreads + tid) + 2), f(v.w, 4 * (r * kPickThreads + tid) + 3);
      }
    };
    static_assert(kReads * 4 * kPickThreads == kTopGroups * kTopThreads, "whole reads");
    const int subs = groups * kTopThreads / 4 >= kPickThreads && k <= kPickThreads ? 1 : 4;  // (values a thread)
    float best[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};  // (also what a group notes where it has no column)
    each_top([&](float t, int g) { best[g & 3] = fmaxf(best[g & 3], t); });
    float hi = fmaxf(fmaxf(best[0], best[1]), fmaxf(best[2], best[3]));
    if (subs == 1) best[0] = hi;
    float lo = INFINITY;
    int some = 0;
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (q < subs && best[q] > -INFINITY) lo = fminf(lo, best[q]), ++some;
    pick_range(lo, hi, some, sh);
    float from = -FLT_MAX;  // all above -inf
    if (some >= k) {
      from = lo;
      for (int level = 0; level < 4 && hi > lo; ++level) {
        const float scale = 255.f / (hi - lo);
        for (int b = tid; b < 256; b += kPickThreads) sh.hist[b] = 0;
        pick_sync();
        each_top([&](float t, int) {
          if (t >= lo) atomicAdd(&sh.hist[min(255, (int)((t - lo) * scale))], 1);
        });
        pick_sync();
        // Every warp finds the last bin that k groups reach: a lane has 8 bins, and the sum of the lanes above it.
        int mine = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) mine += sh.hist[8 * lane + e];
        int above = mine;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
          const int o = __shfl_down_sync(0xffffffffu, above, off);
          if (lane + off < 32) above += o;
        }
        const int at_lane = 31 - __clz(__ballot_sync(0xffffffffu, above >= k));
        int bin = 0, reached = 0;
        if (lane == at_lane) {
          reached = above - mine;
          for (bin = 8 * lane + 7; bin > 8 * lane; --bin) {
            if (reached + sh.hist[bin] >= k) break;
            reached += sh.hist[bin];
          }
          reached += sh.hist[bin];
        }
        bin = __shfl_sync(0xffffffffu, bin, at_lane);
        reached = __shfl_sync(0xffffffffu, reached, at_lane);
        // The bin's lower end, and a little below for the roundings of a value's bin: no value of the bin is lost.
        const float width = 1.f / scale, slack = 4e-6f * (hi - lo) + 4e-7f * fmaxf(fabsf(lo), fabsf(hi));
        const float end = lo + (float)bin * width;
        from = bin ? fmaxf(lo, end - slack) : lo;
        if (reached <= k + k / 2 + 16 || width < 4.f * slack) break;
        hi = fminf(hi, end + width);
        lo = from;
      }
    }
    if (tid == 0) sh.count = sh.n_hits = 0;
    pick_sync();
    low = ordered(from);
    // The groups that reach it: their number first, so that a warp takes its places at once.
    int n_mine = 0;
    each_top([&](float t, int) { n_mine += t >= from; });
    int place = n_mine;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, place, off);
      if (lane >= off) place += o;
    }
    int base = 0;
    if (lane == 31) base = atomicAdd(&sh.n_hits, place);
    place += __shfl_sync(0xffffffffu, base, 31) - n_mine;
    if (n_mine)
      each_top([&](float t, int g) {
        if (t < from) return;
        if (place < kTopCap) sh.hits[place] = (uint16_t)g;
        ++place;
      });
    auto look = [&](int c, float v) { take(c, v, low, sh); };
    edge_column<T>(p, edge, look);
    pick_sync();
    // All threads share the hit groups' vectors.
    constexpr int kLogVecs = 2;
    static_assert(TopShape::kVecs == 1 << kLogVecs, "a thread's vectors");
    const int hits = sh.n_hits, log_vecs = shift + kLogVecs;
    const bool lone = lone_chunk<T>(p);
    if (hits <= kTopCap) {
      vectors<T, 8>(p, hits << log_vecs, [&](int i) {
        const int group = sh.hits[i >> log_vecs], u = i & ((1 << log_vecs) - 1);
        const int chunk = (group / kTopThreads << shift) + (u >> kLogVecs), t = group % kTopThreads;
        const int j = lone ? t + u * kTopThreads
                           : chunk * TopShape::kChunk + t * TopShape::kVecs + (u & (TopShape::kVecs - 1));
        return j < p.nv ? j : -1;
      }, from, look);
      pick_sync();
      m = sh.count;
    }
    if (m > kTopCap)
      m = collect<T>(p, edge, low + 1, sh);  // the columns above, then the ties
    else if (m < k)
      low = ordered(-INFINITY);  // all there is above it
  }
  if (m > kTopCap) {
    low = kth_key<T>(p, edge, k, sh);
    m = low == 0xffffffffu ? 0 : collect<T>(p, edge, low + 1, sh);
  }
  if (m < k) {
    // Columns equal to low, the lowest first: the part's body, with the row's edges (all in one CTA) around it.
    const int c0 = edge ? 0 : p.head + p.v0 * VE, c1 = p.head + (p.v0 + p.nv) * VE;
    const int tail = p.head + p.nvec * VE, end = edge ? c1 + (edge - p.head) : c1;
    for (int at0 = c0; at0 < end && m < k; at0 += kPickThreads) {
      const int c = at0 + tid < c1 ? at0 + tid : tail + (at0 + tid - c1);
      const bool tie = at0 + tid < end && ordered(as_float(p.x[c])) == low;
      const uint32_t vote = __ballot_sync(0xffffffffu, tie);
      pick_sync();
      if (lane == 0) sh.part[warp] = __popc(vote);
      pick_sync();
      int at = m + __popc(vote & ((1u << lane) - 1u));
      for (int i = 0; i < kPickWarps; ++i) {
        if (i < warp) at += (int)sh.part[i];
        m += (int)sh.part[i];
      }
      if (tie && at < k) sh.keys[at] = (uint64_t)low << 32 | (0xffffffffu - (uint32_t)c);
    }
    m = min(m, k);
    pick_sync();
  }
  if (tid == 0 && (m & 1)) sh.keys[m] = 0;  // (no column's key)
  pick_sync();
  const ulonglong2* pairs = reinterpret_cast<const ulonglong2*>(sh.keys);
  for (int i = tid; i < m; i += kPickThreads) {
    const uint64_t key = sh.keys[i];
    int rank = 0;
#pragma unroll 4
    for (int j = 0; j < (m + 1) / 2; ++j) {
      const ulonglong2 two = pairs[j];
      rank += (two.x > key) + (two.y > key);
    }
    if (rank < k) sh.best[rank] = key;
  }
  pick_sync();
  return k;
}

// Bound by HBM: the row is read once (16-bit columns: and by the exponentials of its log-sum-exp).
template <typename T>
__global__ void __launch_bounds__(kTopCta, TopShape::kCtas) top_logits_kernel(const TopArgs A) {
  extern __shared__ __align__(128) uint8_t dyn[];
  uint4* slots = reinterpret_cast<uint4*>(dyn);
  TopShared& sh = *reinterpret_cast<TopShared*>(dyn + TopShape::kRingBytes);
  constexpr int VE = RowSplit<T>::VE;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = cluster_rank(), size = cluster_size();
  if (tid == 0) {
    for (int i = 0; i < TopShape::kSlots; ++i) mbar_init(&sh.full[i], 1), mbar_init(&sh.empty[i], kTopWarps);
    for (int i = 0; i < 2; ++i) mbar_init(&sh.row_full[i], kTopWarps), mbar_init(&sh.row_empty[i], kPickWarps);
    sh.gave_up = 0;
    fence_barrier_init();
  }
  __syncthreads();
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int n = A.batch * A.length, first = blockIdx.x / size, step = gridDim.x / size;
  auto write = [&](int row, const RowSum<float>& a, uint64_t key, int at) {
    const bool bad = *(volatile int*)&sh.gave_up;  // (a wait that ran out: no list)
    A.values[(int64_t)row * A.k + at] = bad ? NAN : unordered((uint32_t)(key >> 32));
    A.tokens[(int64_t)row * A.k + at] = bad ? -1 : (int64_t)(0xffffffffu - (uint32_t)key);
    if (at == 0) {
      const float c = center(a.m, A.ks);
      A.lse[row] = bad ? NAN : (float)((log2_sum(a.s) + (far_out(c) ? (double)a.m * A.kd : -(double)c)) * kLn2d);
    }
  };
  if (warp == kTopWarps + kPickWarps) {
    if (lane == 0) {
      Ring<TopShape::kSlots> r;
      int filled = 0;
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
          bulk_copy_g2s(slots + r.slot * TopShape::kChunk, p.body() + c * TopShape::kChunk, nv * 16, &sh.full[r.slot]);
          r.next();
        }
      }
      if (*(volatile int*)&sh.gave_up)  // copies still in flight end before the CTA's shared memory goes
        for (int k = 0; k < TopShape::kSlots; ++k)
          if (k < r.slot || filled == TopShape::kSlots) mbar_wait_bounded(&sh.full[k], k < r.slot ? r.phase : r.phase ^ 1);
    }
  } else if (warp < kTopWarps) {
    Ring<TopShape::kSlots> r;
    for (int row = first, it = 0; row < n; row += step, ++it) {
      const TopPart<T> p(A, row, rank, size);
      const int edge = rank == 0 ? A.vocab - p.nvec * VE : 0;
      const int per = 1 << group_shift<T>(p), par = it & 1;
      if (it >= 2) wait_or_mark(&sh.row_empty[par], ((it >> 1) & 1) ^ 1, sh);
      Fold<false> fold;
      float top = -INFINITY;
      for (int c = 0, in_group = 0, group = 0; c < p.chunks; ++c) {
        wait_or_mark(&sh.full[r.slot], r.phase, sh);
        const uint4* in = slots + r.slot * TopShape::kChunk;
        const int nv = min(TopShape::kChunk, p.nv - c * TopShape::kChunk);
        // A thread's vectors lie together, so that a group is 64 bytes of a chunk; each pair of threads starts at
        // another of them, which keeps the reads off each other's banks.
        constexpr int kVecs = TopShape::kVecs;
        const int at = tid * kVecs, turn = tid >> 1;
        if (nv == TopShape::kChunk) {
          uint4 v[kVecs];
#pragma unroll
          for (int u = 0; u < kVecs; ++u) v[u] = in[at + ((u + turn) & (kVecs - 1))];
          top = fmaxf(top, fold.template add_vecs<true, T>(v, A.ks));
        } else {
          const bool lone = lone_chunk<T>(p);
          for (int u = 0; u < kVecs; ++u) {
            const int j = lone ? tid + u * kTopThreads : at + u;
            if (j >= nv) break;
            const uint4 v[1] = {in[j]};
            top = fmaxf(top, fold.template add_vecs<false, T>(v, A.ks));
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.empty[r.slot]);
        r.next();
        if (++in_group == per || c + 1 == p.chunks) {
          sh.tops[par][group++][tid] = top;
          top = -INFINITY;
          in_group = 0;
        }
      }
      if (tid < edge) {
        const float f[1] = {as_float(p.x[tid < p.head ? tid : tid + p.nvec * VE])};
        fold.template add<false>(f, f[0], A.ks);
      }
      const RowSum<float> a = warp_merge(fold.sum(), 32, A.ks);
      if (lane == 0) sh.sum[par][warp] = a;
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.row_full[par]);
    }
  } else {
    for (int row = first, it = 0; row < n; row += step, ++it) {
      const TopPart<T> p(A, row, rank, size);
      const int edge = rank == 0 ? A.vocab - p.nvec * VE : 0, par = it & 1;
      wait_or_mark(&sh.row_full[par], (it >> 1) & 1, sh);
      const RowSum<float> all = warp_merge(lane < kTopWarps ? sh.sum[par][lane] : RowSum<float>{0.f, -INFINITY, 0.f}, 32, A.ks);
      const int m = part_list<T>(p, edge, A.k, all.s == all.s, par, sh);
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.row_empty[par]);
      if (size == 1) {
        for (int i = pick_id(); i < A.k; i += kPickThreads) write(row, all, sh.best[i], i);
      } else if (pick_id() == 0) {
        sh.all = all;
        sh.best_n = m;
      }
      pick_sync();  // (sh.best is read before the next row's)
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
    const RowSum<float> all = warp_merge(lane < size ? cluster_peer(&sh, lane)->all : RowSum<float>{0.f, -INFINITY, 0.f}, 32, A.ks);
    for (int q = 0; q < size; ++q) {
      const TopShared* peer = cluster_peer(&sh, q);
      if (tid == 0) s_n[q] = peer->best_n;
      for (int i = tid; i < peer->best_n; i += kTopCta) lists[q * PKV_MAX_TOP + i] = peer->best[i];
      if (tid == 0 && peer->gave_up) sh.gave_up = 1;
    }
    __syncthreads();
    for (int i = tid; i < size * A.k; i += kTopCta) {
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
    return launch_after(kernel, grid, kTopCta, c, kBytes, a, s, "top_logits launch");
  };
  if (r->dtype == PKV_F32) return launch(top_logits_kernel<float>);
  if (r->dtype == PKV_F16) return launch(top_logits_kernel<__half>);
  return launch(top_logits_kernel<__nv_bfloat16>);
}
