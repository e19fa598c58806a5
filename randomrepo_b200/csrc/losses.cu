// Losses over vocabulary rows and their gradients, for sm_100a: the clipped
// policy loss (with KL and entropy terms), the preference loss over pairs of
// sequences, and distillation from a teacher's top logits.
//
// A row is one position's `vocab` logits x.  With z = x / T everything a loss
// needs of a row is its base-2 log-sum-exp pair (m, s): m = max x, y_j =
// x_j k - m k, k = log2(e) / T, e_j = 2^y_j, s = sum e_j, p_j = e_j / s (and
// w = sum e_j y_j where the entropy H = ln 2 (log2 s - w / s) is asked for), plus a few
// single logits (the token's, the teacher's list).  The gradient of every
// loss here has the form
//     dx_j = e_j (a + b y_j) + [j in a short list] h_j
// with a, b, h per row:
//   policy, preference   a = -g / (T s), h = g / T at the token, g = dl/dlogp
//   entropy bonus        a += c (H - ln 2 log2 s) / s, b = c ln2 / s, c = w ent / T
//   distillation         a = w T Q / s, h_k = -w T q_k
// so a row is read once for its pair, and once more (from L2 or shared
// memory) to write its gradient.
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <string>

#include "loss_rows.cuh"
#include "pkv_b200.h"
#include "pkv_device.cuh"
#include "pkv_error.h"

namespace pkv {
namespace {

constexpr float kLn2 = 0.6931471805599453f;

enum Kind { kPolicy = 0, kPreference = 1, kDistill = 2 };
enum Pass { kForward = 0, kBackward = 1, kFused = 2 };

// A [batch][length] array with element strides (stride 0 broadcasts).
template <typename T>
struct Tokens2 {
  const T* p;
  int64_t sb, st;
  __device__ __forceinline__ T at(int b, int t) const { return p[b * sb + t * st]; }
};

struct LossHeader {
  int32_t n_active;
  int32_t ticket;
  int32_t error;  // a bounded wait gave up: the loss, and gradients made after it, become NaN
};

struct LossArgs {
  const void* x;
  int64_t xb, xr;
  void* g;
  int64_t gb, gr;
  int32_t batch, length, vocab;
  LossHeader* hdr;
  const int32_t* list;    // rows b * length + t: the scored ones in order, then the others
  const float* seq_w;     // [batch] what a scored row's loss counts
  const float* seq_g;     // [batch] dl/dlogp of a sequence's rows (preference), or null
  Scale2 ks;              // log2(e) / T
  double kd;              // the same
  float inv_t, temperature;
  double inv_td;
  Tokens2<int64_t> tokens;
  Tokens2<float> adv, old, ref;
  float ratio_low, ratio_high, kl_coef, ent_coef;
  const int64_t* ids;     // teacher's list
  const float* tl;
  int64_t ids_b, ids_t, tl_b, tl_t;
  int32_t k;
  Tokens2<float> tlse;
  float *logprobs, *kl_out, *entropy, *loss;
  double* row_val;        // [rows]: weighted loss (policy, distillation) or log-probability (preference)
  float4* rec;            // [rows] {m, a, b, h} for a later backward pass (distillation: {m, a, w T, -}) of x's type
  const float* upstream;  // device scalar the gradient is multiplied by, or null
};

// What a row's gradient needs: dx_j = e_j (a + b y_j), + h at the token.
struct RowGrad {
  float m, a, b, h;
  int tok;
  bool zero;  // the gradient is zero whatever the logits
};

// log2 of a column's probability, in 64 bits.
template <typename D>
__device__ __forceinline__ double log2_prob(const LossArgs& A, const RowSum<D>& r, float x) {
  const float c = center(r.m, A.ks);
  return (far_out(c) ? ((double)x - (double)r.m) * A.kd : (double)x * A.kd + (double)c) - log2_sum(r.s);
}

// A scored row's own inputs, loaded before its sums are made.
struct RowTerms {
  int64_t tok;
  float x_tok, w, adv, old, ref;
};

// A row's values beside its gradient: log p, d = ref - log p, the loss without its KL term, the entropy.
struct PolicyRow {
  double lp, d;
  float l, h;
};

template <bool ENT, typename D>
__device__ __forceinline__ RowGrad policy_tail(const LossArgs& A, const RowSum<D>& r, const RowTerms& q, PolicyRow& v) {
  const int64_t tok = q.tok;
  const bool known = tok >= 0 && tok < A.vocab;
  const double log2s = log2_sum(r.s);
  const double lp = known ? log2_prob(A, r, q.x_tok) * kLn2d : (double)NAN;
  const float w = q.w, adv = q.adv;
  const float ratio = A.old.p ? expf((float)(lp - (double)q.old)) : (lp == lp ? 1.f : NAN);
  // -min(r A, clip(r) A): the clipped branch is the smaller one above the border for A > 0, below it for A < 0.
  const bool cut = (adv > 0.f && ratio > A.ratio_high) || (adv < 0.f && ratio < A.ratio_low);
  const float used = cut ? (adv > 0.f ? A.ratio_high : A.ratio_low) : ratio;
  float l = adv == 0.f ? 0.f : -used * adv;
  float g = (cut || adv == 0.f) ? 0.f : -ratio * adv;
  if (!(lp == lp)) l = g = NAN;
  v.lp = lp, v.d = (double)q.ref - lp, v.h = 0.f;
  if (A.ref.p) g = fmaf(-A.kl_coef, expm1f((float)v.d), g);
  g *= w * A.inv_t;
  const float inv_s = 1.f / (float)r.s;
  RowGrad o{r.m, -g * inv_s, 0.f, g, known ? (int)tok : -1, false};
  if (ENT) {
    const double mean = (double)r.w / (double)r.s;
    v.h = (float)((log2s - mean) * kLn2d);
    const float c = A.ent_coef * w * A.inv_t;
    l = fmaf(-A.ent_coef, v.h, l);
    o.a = fmaf(c * inv_s, (float)(-kLn2d * mean), o.a);  // H - ln2 log2 s = -ln2 w / s
    o.b = c * kLn2 * inv_s;
  }
  o.zero = !ENT && g == 0.f;
  v.l = l;
  return o;
}

// Written when the gradient's coefficients are on their way.  The KL estimate e^d - d - 1 in 64 bits: near the
// reference it is d^2 / 2, of which a float32 difference has no digits left below d = 1e-7 (and 1e-4 of it at 1e-3).
template <bool ENT>
__device__ __forceinline__ void write_policy(const LossArgs& A, int row, float w, const PolicyRow& v) {
  float l = v.l, kl = 0.f;
  if (A.ref.p) {
    kl = (float)(expm1(v.d) - v.d);
    l = fmaf(A.kl_coef, kl, l);
  }
  A.logprobs[row] = (float)v.lp;
  if (A.kl_out) A.kl_out[row] = kl;
  if (ENT && A.entropy) A.entropy[row] = v.h;
  A.row_val[row] = (double)w * (double)l;
}

// ---------------------------------------------------------------------------
// Plan: the scored rows, and what each sequence's rows count in the loss.

struct PlanArgs {
  const uint8_t* mask;
  int64_t mb, mt;
  int32_t batch, length, reduction;
  float scale;
  LossHeader* hdr;
  int32_t* list;
  float* seq_w;
  int32_t* seq_n;
};

// One CTA: each thread has a run of rows, whose mask it reads once (into bits, 64 rows at a time, eight reads on their
// way; latency is all there is to this kernel).
__global__ void __launch_bounds__(1024) loss_plan_kernel(const PlanArgs A) {
  __shared__ int s_warp[32], s_full, s_total;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int n = A.batch * A.length;
  const int per = (n + 1023) / 1024, r0 = min(n, tid * per), r1 = min(n, r0 + per);
  for (int b = tid; b < A.batch; b += 1024) A.seq_n[b] = 0;
  if (tid == 0) s_full = 0;
  // 64 rows from r, as bits; b and t of row r go on to the row behind them.
  auto bits_of = [&](int r, int& b, int& t) {
    const int m = min(64, r1 - r);
    uint64_t bits = 0;
#pragma unroll 8
    for (int k = 0; k < m; ++k) {
      if (A.mask == nullptr || A.mask[b * A.mb + t * A.mt] != 0) bits |= 1ull << k;
      if (++t == A.length) t = 0, ++b;
    }
    return bits;
  };
  const int b0 = r0 < r1 ? r0 / A.length : 0, t0 = r0 < r1 ? r0 - b0 * A.length : 0;
  uint64_t first = 0;  // (the only bits of a run of 64 rows)
  int mine = 0;
  {
    int b = b0, t = t0;
    for (int r = r0; r < r1; r += 64) {
      const uint64_t bits = bits_of(r, b, t);
      if (r == r0) first = bits;
      mine += __popcll(bits);
    }
  }
  int incl = mine;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, off);
    if (lane >= off) incl += v;
  }
  if (lane == 31) s_warp[warp] = incl;
  __syncthreads();
  if (warp == 0) {
    int v = s_warp[lane], w = v;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, w, off);
      if (lane >= off) w += u;
    }
    s_warp[lane] = w - v;
    if (lane == 31) s_total = w;
  }
  __syncthreads();
  const int total = s_total;
  int at = s_warp[warp] + incl - mine, rest = total + r0 - at;
  int b = b0, t = t0, seq = b0, in_seq = 0;
  int mb = b0, mt = t0;  // the mask's own place, where it is read again
  auto count = [&]() {
    if (in_seq) atomicAdd(A.seq_n + seq, in_seq);
  };
  for (int r = r0; r < r1; r += 64) {
    const uint64_t bits = per <= 64 ? first : bits_of(r, mb, mt);
    const int m = min(64, r1 - r);
    for (int k = 0; k < m; ++k) {
      if (b != seq) {
        count();
        seq = b, in_seq = 0;
      }
      if (bits >> k & 1) {
        A.list[at++] = r + k;
        ++in_seq;
      } else {
        A.list[rest++] = r + k;
      }
      if (++t == A.length) t = 0, ++b;
    }
  }
  if (r0 < r1) count();
  __threadfence_block();
  __syncthreads();
  if (A.reduction == PKV_SEQUENCE_MEAN) {
    int full = 0;
    for (int q = tid; q < A.batch; q += 1024) full += __ldcg(A.seq_n + q) > 0;
    if (full) atomicAdd(&s_full, full);
    __syncthreads();
  }
  for (int q = tid; q < A.batch; q += 1024) {
    const int c = __ldcg(A.seq_n + q);
    float w = A.scale;
    if (A.reduction == PKV_TOKEN_MEAN) w = (float)((double)A.scale / max(total, 1));
    if (A.reduction == PKV_SEQUENCE_MEAN) w = (float)((double)A.scale / ((double)max(c, 1) * max(s_full, 1)));
    A.seq_w[q] = w;
  }
  if (tid == 0) {
    A.hdr->n_active = total;
    A.hdr->ticket = 0;
    A.hdr->error = 0;
  }
}

// ---------------------------------------------------------------------------
// Rows.

// 16-bit gradients leave x k.lo out of a column's y, which the sum s has: e comes out smaller by 2^(x k.lo), the same
// factor for all columns that count (those near m: (x - m) k.lo is at most 2^-23 of a y of 30 or so).  It goes into the
// row's a and b, for at a column of a large h or q, where p is near it, half a step of 16 bits would not hide it.
template <typename T>
__device__ __forceinline__ void fold_low(RowGrad& o, Scale2 k) {
  if (sizeof(T) == 4) return;
  const float y = far_out(center(o.m, k)) ? 0.f : o.m * k.lo, f = ex2(y);
  o.a = fmaf(o.b, y, o.a) * f;
  o.b *= f;
}

// N columns of the gradient, the list's columns apart.
template <bool ENT, typename T, int N>
__device__ __forceinline__ void grad_columns(float (&x)[N], const RowGrad& o, Scale2 k) {
  const float c = center(o.m, k);
  if (far_out(c)) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float y = (x[i] - o.m) * k.hi;
      x[i] = ex2(y) * (ENT ? fmaf(o.b, fmaxf(y, -1e30f), o.a) : o.a);
    }
    return;
  }
  const f32x2 cc = pair(c, c), hi = pair(k.hi, k.hi), lo = pair(k.lo, k.lo), a = pair(o.a, o.a), b = pair(o.b, o.b);
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    const f32x2 xx = pair(x[i], i + 1 < N ? x[i + 1] : 0.f);
    f32x2 y2 = fma2(xx, hi, cc);
    if (sizeof(T) == 4) y2 = fma2(xx, lo, y2);  // (16 bits: in a and b)
    const float2 y = unpair(y2);
    const f32x2 e = pair(ex2(y.x), ex2(y.y));
    const float2 v = unpair(mul2(e, ENT ? fma2(b, pair(fmaxf(y.x, -1e30f), fmaxf(y.y, -1e30f)), a) : a));
    x[i] = v.x;
    if (i + 1 < N) x[i + 1] = v.y;
  }
}

template <bool ENT, typename T>
__device__ __forceinline__ float grad_of(float x, const RowGrad& o, Scale2 k) {
  float v[1] = {x};
  grad_columns<ENT, T>(v, o, k);
  return v[0];
}

__device__ __forceinline__ float teacher_logit(const LossArgs& A, int b, int t, int i, int64_t& id) {
  id = A.ids[b * A.ids_b + t * A.ids_t + i];
  const float v = A.tl[b * A.tl_b + t * A.tl_t + i];
  return id < 0 ? -INFINITY : v;  // an absent entry
}

// A row's teacher list as its warp leaves it for the others (X: with the columns' logits).
template <bool X>
struct TeacherRow {
  double q_sum, qx, qlogq; // sums over the list of q, q x[id] and q log q (a NaN: an id past the vocabulary)
  int32_t id[PKV_MAX_TOP]; // -1: not a column, or one that an entry before has
  float q[PKV_MAX_TOP];    // the column's share, of all its entries
  float x[X ? PKV_MAX_TOP : 1];
};
constexpr int kIdTable = 2 * PKV_MAX_TOP;

// Measured on rows of 151 936 columns.  Sums or gradient alone: four CTAs of 128 threads that take 8 vectors at a time
// (16-bit sums of 4 096 rows 210 us; 160 threads x 3 CTAs 234, 96 x 5 251, 512 threads x 4 vectors x 1 CTA 275).  Both in
// one launch: one CTA an SM, whose rows in flight stay in L2 until their second pass; 16 bits 454 us (512 threads 464,
// 768 480, two CTAs of 384 threads 512, a row to a pair of CTAs 530), where two exponentials and their conversions a
// column cost as much as HBM.  float32, half the exponentials a byte: fewer threads and more slots (8 192 rows 1.58 ms;
// 512 threads 1.61).  A row to a pair of CTAs where the rows in flight would not stay in L2; us of 4 096 rows with /
// without: float32 116 000 columns 690 / 675, 128 000 725 / 764, 152 064 845 / 950; 16 bits 232 000 696 / 684,
// 256 000 775 / 773 (with an entropy term 890 / 805), 288 000 850 / 914; 2 048 of 512 000 776 / 929.
template <typename T, int PASS> struct ShapeOf : Shape<128, 8, 3, 4> {};
template <typename T> struct ShapeOf<T, kFused> : Shape<640, 4, 5, 1> {};
template <> struct ShapeOf<float, kFused> : Shape<384, 4, 8, 1> {};
// Short rows, sums and gradient: four CTAs an SM, for each row is a chain of latencies.  8 192 rows against the shapes
// above: 1 000 16-bit columns 63 / 176 us, 10 000 127 / 212, 50 000 367 / 402, 80 000 559 / 546; float32 1 000 63 / 153,
// 20 000 246 / 305, 35 000 469 / 423.
using ShortShape = Shape<128, 4, 5, 4>;
constexpr int64_t kShortRow = 112 << 10;   // bytes
constexpr int64_t kRowsInL2 = 72 << 20;    // bytes of rows in flight that come back from L2

template <typename S, bool X, typename D>
struct alignas(128) LossShared {
  uint64_t full[S::kSlots], empty[S::kSlots];
  uint64_t part_full[2], part_empty[2], grad_full[2], grad_empty[2], teacher_full[2], teacher_empty[2], peers[2];
  float4 peer[2][kMaxCluster];
  RowSum<D> part[2][32];
  RowGrad grad[2];
  float grad_wt[2];
  double sum[32];
  int last, gave_up;
  TeacherRow<X> teacher[2];
  int32_t ids[kIdTable];  // the ids of a list, by their hash
};

// The preference loss adds a row's log-probability up over its sequence: its sums are exact ones.  Others' errors (1e-7 at
// the most, rms) are below the rounding of the float32 outputs that they end in.
template <int KIND, int PASS>
constexpr bool kExactSums = KIND == kPreference && PASS == kForward;
template <int KIND, int PASS>
using SumOf = std::conditional_t<kExactSums<KIND, PASS>, double, float>;

template <typename D>
__device__ __forceinline__ float4 sum_bits(const RowSum<D>& a) {
  if constexpr (sizeof(D) == 4) return make_float4(a.m, a.s, a.w, 0.f);
  const double s = a.s;
  return make_float4(a.m, __int_as_float(__double2loint(s)), a.w, __int_as_float(__double2hiint(s)));
}
template <typename D>
__device__ __forceinline__ RowSum<D> sum_of_bits(float4 v) {
  if constexpr (sizeof(D) == 4) return RowSum<D>{v.y, v.x, v.z};
  return RowSum<D>{(D)__hiloint2double(__float_as_int(v.w), __float_as_int(v.y)), v.x, v.z};
}

// 16 bytes into the same shared-memory place of CTA `rank` of the cluster, counted on its barrier.
__device__ __forceinline__ void send_peer(void* dst, uint64_t* bar, uint32_t rank, float4 v) {
  uint32_t d, b;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(d) : "r"(smem_u32(dst)), "r"(rank));
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(b) : "r"(smem_u32(bar)), "r"(rank));
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(d),
               "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w), "r"(b)
               : "memory");
}

// The order of copies, which the column warps follow.  Sums or gradient alone: a row's chunks in turn.  Both: a row's
// chunks for its sums, then the first chunk of the row behind it (whose sums begin while this row's coefficients are
// made), then the chunks that did not stay in the ring, again, for its gradient.
//
// Copy l waits for the chunk of copy l - kSlots, so none may be waited for before it can be free.  `whole`: a row has at
// most kSlots - 1 chunks, all stay, and kSlots copies before the next row's first one lies the row before.  Else the
// last kSlots - 1 chunks stay, but never the first one (rows at another offset in their 16 bytes may have a chunk less):
// it is free when its sums are made, as are all that lie kSlots or more before the next row's first one.
template <typename T, typename S>
__device__ __forceinline__ bool rows_whole(int vocab, int size) {
  const int nvec = vocab / RowSplit<T>::VE, per = (nvec + size - 1) / size;
  return (per + S::kChunk - 1) / S::kChunk <= S::kSlots - 1;
}
// How many chunks of a row are copied twice.
template <int PASS, typename S>
__device__ __forceinline__ int chunks_again(int chunks, bool whole) {
  return PASS == kFused && !whole ? max(chunks - (S::kSlots - 1), min(chunks, 1)) : 0;
}

// The copying warp (one lane of it).
template <typename T, int PASS, typename S, typename Sh>
__device__ __forceinline__ void copy_rows(const LossArgs& A, Sh& sh, uint4* slots, int rank, int size, int first,
                                          int step, int n_active, int row0) {
  Ring<S::kSlots> r;
  int filled = 0;
  const bool whole = rows_whole<T, S>(A.vocab, size);
  // Chunks read twice are asked to stay in L2 until then; the others leave it first.
  uint64_t keep_policy;
  asm volatile("createpolicy.fractional.L2::evict_last.b64 %0, 1.0;" : "=l"(keep_policy));
  const uint64_t once_policy = l2_evict_first_policy();
  // False: a wait gave up.
  auto copy = [&](const RowPart<T, S::kChunk>& p, int at, bool keep) {
    if (filled == S::kSlots)
      wait_or_mark(&sh.empty[r.slot], r.phase ^ 1, sh);
    else
      ++filled;
    if (*(volatile int*)&sh.gave_up) {
      // Copies still in flight end before the CTA's shared memory goes.
      for (int k = 0; k < S::kSlots; ++k)
        if (k < r.slot || filled == S::kSlots) mbar_wait_bounded(&sh.full[k], k < r.slot ? r.phase : r.phase ^ 1);
      return false;
    }
    const int nv = min(S::kChunk, p.nv - at * S::kChunk);
    mbar_arrive_expect_tx(&sh.full[r.slot], nv * 16);
    bulk_copy_g2s_hint(slots + r.slot * S::kChunk, p.body() + at * S::kChunk, nv * 16, &sh.full[r.slot],
                       keep ? keep_policy : once_policy);
    r.next();
    return true;
  };
  int row = row0;
  for (int i = first; i < n_active; i += step) {
    const RowPart<T, S::kChunk> p(A, row, rank, size);
    if (i + step < n_active) row = A.list[i + step];
    const int again = chunks_again<PASS, S>(p.chunks, whole);
    for (int c = PASS == kFused && i != first ? 1 : 0; c < p.chunks; ++c)
      if (!copy(p, c, c < again)) return;
    if (PASS != kFused) continue;
    if (i + step < n_active) {
      const RowPart<T, S::kChunk> next(A, row, rank, size);
      if (next.chunks && !copy(next, 0, chunks_again<PASS, S>(next.chunks, whole) > 0)) return;
    }
    for (int c = 0; c < again; ++c)
      if (!copy(p, c, false)) return;
  }
}

// The teacher's warp: q and its sums, a row or two ahead.
template <typename T, int PASS, typename S, typename Sh>
__device__ __forceinline__ void teacher_rows(const LossArgs& A, Sh& sh, int rank, int size, int first, int step,
                                             int n_active, int row0, int lane) {
  int row = row0;
  for (int i = first, it = 0; i < n_active; i += step, ++it) {
    const RowPart<T, S::kChunk> p(A, row, rank, size);
    if (i + step < n_active) row = A.list[i + step];
    auto& o = sh.teacher[it & 1];
    if (it >= 2) wait_or_mark(&sh.teacher_empty[it & 1], ((it >> 1) & 1) ^ 1, sh);
    constexpr int kPer = PKV_MAX_TOP / 32;
    float v[kPer], x[kPer];
    int ids[kPer];
    float top = -INFINITY;
    for (int j = lane; j < kIdTable; j += 32) sh.ids[j] = -1;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const int j = lane + 32 * e;
      v[e] = -INFINITY, x[e] = 0.f, ids[e] = -1;
      if (j < A.k) {
        int64_t id;
        v[e] = teacher_logit(A, p.b, p.t, j, id);
        if (id >= 0 && id < A.vocab)
          ids[e] = (int)id, x[e] = PASS == kBackward ? 0.f : as_float(p.x[id]);
        else if (v[e] != -INFINITY)
          x[e] = NAN;
        top = fmaxf(top, v[e]);
      }
    }
    // Does an id come twice?  (A column is written once, with all its shares; lists hardly ever need that.)
    __syncwarp();
    bool twice = false;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      if (32 * e >= A.k || ids[e] < 0) continue;
      for (int at = ids[e] & (kIdTable - 1);; at = (at + 1) & (kIdTable - 1)) {
        const int there = atomicCAS(&sh.ids[at], -1, ids[e]);
        if (there == -1) break;
        if (there == ids[e]) {
          twice = true;
          break;
        }
      }
    }
    twice = __any_sync(0xffffffffu, twice);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
    // log q = (v - base) / T - norm, in 64 bits (it would lose digits to a rounded norm) and from the largest entry (an
    // entry may be a type's lowest value, in all of which the norm's logarithm would be lost).
    double base = 0.0, norm = 0.0;
    if (A.tlse.p) {
      norm = (double)A.tlse.at(p.b, p.t);
    } else if (top > -INFINITY) {
      double sum = 0.0;
#pragma unroll
      for (int e = 0; e < kPer; ++e)
        if (v[e] != -INFINITY) sum += (double)expf((float)(((double)v[e] - (double)top) * A.inv_td));
      base = (double)top;
      norm = log(warp_sum_d(sum));
    }
    double qs = 0.0, qx = 0.0, ql = 0.0;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const int j = lane + 32 * e;
      float q = 0.f;
      if (v[e] != -INFINITY) {
        const double lq = ((double)v[e] - base) * A.inv_td - norm;
        q = expf((float)lq);
        qs += (double)q;
        if (q != 0.f || x[e] != x[e]) {
          qx += (double)q * (double)x[e];
          ql += (double)q * lq;
        }
      }
      if (j < A.k) {
        o.q[j] = q, o.id[j] = ids[e];
        if (PASS == kFused) o.x[j] = x[e];
      }
    }
    if (twice) {
      __syncwarp();
      float all[kPer];
      bool later[kPer];
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        const int j = lane + 32 * e;
        all[e] = 0.f, later[e] = false;
        if (j >= A.k) continue;
        for (int f = 0; f < A.k; ++f)
          if (o.id[f] == ids[e]) all[e] += o.q[f], later[e] |= f < j;
      }
      __syncwarp();
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        const int j = lane + 32 * e;
        if (j < A.k) o.q[j] = all[e], o.id[j] = later[e] ? -1 : ids[e];
      }
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {  // (the three together: latency is this warp's cost)
      const double a = __shfl_xor_sync(0xffffffffu, qs, off), b = __shfl_xor_sync(0xffffffffu, qx, off);
      const double c = __shfl_xor_sync(0xffffffffu, ql, off);
      qs += a, qx += b, ql += c;
    }
    if (lane == 0) o.q_sum = qs, o.qx = qx, o.qlogq = ql;
    __syncwarp();
    if (lane == 0) mbar_arrive(&sh.teacher_full[it & 1]);
  }
}

// The warp of the rows' terms: it has a row's own inputs in hand when its sums are done, and hands on its gradient's
// coefficients (in the backward pass, those the forward pass left).
template <typename T, int KIND, bool ENT, int PASS, typename S, typename Sh>
__device__ __forceinline__ void term_rows(const LossArgs& A, Sh& sh, int rank, int size, int first, int step,
                                          int n_active, int n, int row0, int lane) {
  const bool write = lane == 0 && rank == 0;
  const Scale2 ks = A.ks;
  // (records that a launch left without all its sums give no gradient)
  const float up = PASS == kBackward && *(volatile int32_t*)&A.hdr->error ? NAN : A.upstream ? *A.upstream : 1.f;
  int row_next = row0;
  int64_t tok_next = 0;
  if (KIND != kDistill && first < n_active) tok_next = A.tokens.at(row_next / A.length, row_next % A.length);
  for (int i = first, it = 0; i < n_active; i += step, ++it) {
    const int row = row_next, b = row / A.length, t = row - b * A.length, par = it & 1;
    const uint32_t phase = (it >> 1) & 1;
    if (i + step < n_active) row_next = A.list[i + step];
    RowTerms q{tok_next, 0.f, 0.f, 0.f, 0.f, 0.f};
    const bool known = q.tok >= 0 && q.tok < A.vocab;
    if (KIND != kDistill && i + step < n_active) tok_next = A.tokens.at(row_next / A.length, row_next % A.length);
    RowGrad o{0.f, 0.f, 0.f, 0.f, -1, false};
    float wt = 0.f;
    PolicyRow val;
    if (PASS == kBackward) {
      const float4 rec = A.rec[row];
      const float f = up * (A.seq_g ? A.seq_g[b] : 1.f);
      if (KIND == kDistill) {
        wt = rec.z * f;
        o = RowGrad{rec.x, rec.y * f, 0.f, 0.f, -1, false};
        o.zero = f == 0.f || (o.a == 0.f && wt == 0.f);  // (the second: no share in the list)
      } else {
        o = RowGrad{rec.x, rec.y * f, rec.z * f, rec.w * f, known ? (int)q.tok : -1, false};
        o.zero = o.a == 0.f && o.b == 0.f && o.h == 0.f;
      }
    } else {
      const T* x = (const T*)A.x + b * A.xb + t * A.xr;
      if (KIND != kPreference) q.w = A.seq_w[b];
      if (KIND != kDistill) q.x_tok = known ? as_float(x[q.tok]) : NAN;
      if (KIND == kPolicy) {
        q.adv = A.adv.at(b, t);
        if (A.old.p) q.old = A.old.at(b, t);
        if (A.ref.p) q.ref = A.ref.at(b, t);
      }
      wait_or_mark(&sh.part_full[par], phase, sh);
      using D = SumOf<KIND, PASS>;
      constexpr int kWide = S::kWarps > 16 ? 32 : S::kWarps > 4 ? 16 : 4;  // (as few rounds as there are sums)
      const int part = lane & (kWide - 1);
      RowSum<D> a = warp_merge(part < S::kWarps ? sh.part[par][part] : RowSum<D>{0, -INFINITY, 0.f}, kWide, ks);
      if (lane == 0) mbar_arrive(&sh.part_empty[par]);
      if (size > 1) {
        if (lane == 0 && !*(volatile int*)&sh.gave_up) {  // (a CTA that gave up leaves its peers to do so)
          mbar_arrive_expect_tx(&sh.peers[par], 16 * size);
          for (int c = 0; c < size; ++c)
            send_peer(&sh.peer[par][rank], &sh.peers[par], c, sum_bits(a));
        }
        __syncwarp();
        wait_or_mark<true>(&sh.peers[par], phase, sh);
        const float4 v = sh.peer[par][lane & (size - 1)];
        a = warp_merge(sum_of_bits<D>(v), size, ks);
      }
      if (KIND == kPolicy) {
        o = policy_tail<ENT>(A, a, q, val);
      } else if (KIND == kPreference) {
        o = RowGrad{a.m, -1.f / (float)a.s, 0.f, 1.f, 0, false};
        if (write) A.row_val[row] = known ? log2_prob(A, a, q.x_tok) * kLn2d : (double)NAN;
      } else {
        wait_or_mark(&sh.teacher_full[par], phase, sh);
        const auto& te = sh.teacher[par];
        // sum q (log q - log p), log p = (x k + c - log2 s) ln 2.  Where no entry has a share (none is there, or all
        // underflow) that is 0 and so is the gradient, whatever the row's columns are.
        const double w = (double)q.w, tt = (double)A.temperature;
        const bool none = te.q_sum == 0.0 && te.qx == te.qx;
        const float c = center(a.m, ks);
        double qp = te.qx * A.kd + te.q_sum * ((double)c - log2_sum(a.s));  // sum q log2 p
        if (far_out(c) && te.qx == te.qx) {
          qp = 0.0;
          for (int f = 0; f < A.k; ++f)
            if (te.id[f] >= 0 && te.q[f] > 0.f) qp += (double)te.q[f] * log2_prob(A, a, as_float(x[te.id[f]]));
        }
        const double l = none ? 0.0 : tt * tt * (te.qlogq - qp * kLn2d);
        wt = none ? 0.f : (float)(w * tt);
        o = RowGrad{a.m, l == l ? wt * (float)te.q_sum / (float)a.s : NAN, 0.f, 0.f, -1, none};
        if (none) o.a = 0.f;  // (not 0 / s)
        if (write) {
          A.kl_out[row] = (float)l;
          A.row_val[row] = w * l;
        }
      }
      fold_low<T>(o, ks);
      if (PASS == kForward) {
        if (write && A.rec)
          A.rec[row] = KIND == kDistill ? make_float4(o.m, o.a, wt, 0.f) : make_float4(o.m, o.a, o.b, o.h);
        if (KIND == kPolicy && write) write_policy<ENT>(A, row, q.w, val);
        if (KIND == kDistill) {
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh.teacher_empty[par]);
        }
        continue;
      }
    }
    if (it >= 2) wait_or_mark(&sh.grad_empty[par], phase ^ 1, sh);
    if (lane == 0) {
      sh.grad[par] = o;
      sh.grad_wt[par] = wt;
      mbar_arrive(&sh.grad_full[par]);
    }
    if (KIND == kPolicy && PASS == kFused && write) write_policy<ENT>(A, row, q.w, val);
  }
  // Rows that are not scored have zeros.
  if (PASS != kBackward && rank == 0) {
    for (int i = n_active + first + step * lane; i < n; i += 32 * step) {
      const int row = A.list[i];
      if (A.logprobs) A.logprobs[row] = 0.f;
      if (A.kl_out) A.kl_out[row] = 0.f;
      if (ENT && A.entropy) A.entropy[row] = 0.f;
      A.row_val[row] = 0.0;
    }
  }
}

// The warps that work on the columns: a row's sums, then its gradient.
template <typename T, int KIND, bool ENT, int PASS, typename S, typename Sh>
__device__ __forceinline__ void column_rows(const LossArgs& A, Sh& sh, const uint4* slots, int rank, int size,
                                            int first, int step, int n_active, int n, int row0, int tid) {
  constexpr int VE = 16 / sizeof(T);
  const int lane = tid & 31, warp = tid >> 5;
  const Scale2 ks = A.ks;
  Ring<S::kSlots> r, zero;  // the next copy; the row's first chunk
  const bool whole = rows_whole<T, S>(A.vocab, size);
  const int end = PASS == kForward ? n_active : n;
  using Sums = Fold<ENT, kExactSums<KIND, PASS>>;
  // Chunk c of a row, at r, into its sums.
  auto sum_chunk = [&](Sums& fold, const RowPart<T, S::kChunk>& p, int c, bool done) {
    wait_or_mark(&sh.full[r.slot], r.phase, sh);
    const uint4* in = slots + r.slot * S::kChunk;
    const int nv = min(S::kChunk, p.nv - c * S::kChunk);
    if (nv == S::kChunk) {
      constexpr int kAtOnce = 4;
      static_assert(S::kVecs % kAtOnce == 0, "vectors are taken four at a time");
#pragma unroll
      for (int h = 0; h < S::kVecs; h += kAtOnce) {
        uint4 v[kAtOnce];
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) v[u] = in[tid + (h + u) * S::kGroup];
        fold.template add_vecs<true, T>(v, ks);
      }
    } else {
      for (int j = tid; j < nv; j += S::kGroup) {
        const uint4 v[1] = {in[j]};
        fold.template add_vecs<false, T>(v, ks);
      }
    }
    if (done) {
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.empty[r.slot]);
    }
    r.next();
  };
  Sums fold;
  int begun = 0;  // chunks of the row that are in its sums already (0 or 1)
  int row = row0;
  for (int i = first, it = 0; i < end; i += step) {
    const RowPart<T, S::kChunk> p(A, row, rank, size);
    if (i + step < end) row = A.list[i + step];
    // The columns outside the body are the cluster's first CTA's.
    const int edge = rank == 0 ? A.vocab - p.nvec * VE : 0;
    const int edge_col = tid < p.head ? tid : tid + p.nvec * VE;
    const int par = it & 1;
    const uint32_t phase = (it >> 1) & 1;
    const int again = chunks_again<PASS, S>(p.chunks, whole);
    Ring<S::kSlots> at_zero = zero;
    if (PASS != kBackward && i < n_active) {
      if (!begun) {
        fold = Sums();
        at_zero = r;
      }
      for (int c = begun; c < p.chunks; ++c) sum_chunk(fold, p, c, PASS == kForward || c < again);
      if (tid < edge) {
        const float f[1] = {as_float(p.x[edge_col])};
        fold.template add<false>(f, f[0], ks);
      }
      const auto a = warp_merge(fold.sum(), 32, ks);
      if (it >= 2) wait_or_mark(&sh.part_empty[par], phase ^ 1, sh);
      if (lane == 0) {
        sh.part[par][warp] = a;
        mbar_arrive(&sh.part_full[par]);
      }
      begun = 0;
      if (PASS == kFused && i + step < n_active) {
        const RowPart<T, S::kChunk> next(A, row, rank, size);
        if (next.chunks) {
          fold = Sums();
          zero = r;
          sum_chunk(fold, next, 0, chunks_again<PASS, S>(next.chunks, whole) > 0);
          begun = 1;
        }
      }
    }
    if (PASS == kForward) {
      ++it;
      continue;
    }
    T* g = (T*)A.g + p.b * A.gb + p.t * A.gr;
    uint4* out = reinterpret_cast<uint4*>(g + p.head) + p.v0;
    const bool vec = ((uintptr_t)out & 15) == 0;
    // (Rows whose gradient starts elsewhere in its 16 bytes are stored a column at a time.)
    auto store = [&](int j, uint4 v) {
      if (vec) {
        __stcs(out + j, v);
      } else {
        const T* f = reinterpret_cast<const T*>(&v);
#pragma unroll
        for (int q = 0; q < VE; ++q) g[p.head + (p.v0 + j) * VE + q] = f[q];
      }
    };
    if (i >= n_active) {
      for (int j = tid; j < p.nv; j += S::kGroup) store(j, make_uint4(0u, 0u, 0u, 0u));
      if (tid < edge) put(g + edge_col, 0.f);
      continue;
    }
    ++it;
    wait_or_mark(&sh.grad_full[par], phase, sh);
    const RowGrad o = sh.grad[par];
    const float wt = KIND == kDistill ? sh.grad_wt[par] : 0.f;
    const int hot_vec = o.tok < p.head ? -1 : (o.tok - p.head) / VE - p.v0;
    // Both passes: the chunks that stayed, which lie before the next row's first one (a row that stayed whole: its
    // first chunk where it was begun), then the others behind it.
    const int stayed = p.chunks - again;
    Ring<S::kSlots> from = r;
    if (PASS == kFused) {
      if (again)
        from.back(begun + stayed);
      else
        from = at_zero;
    }
    for (int c = 0; c < p.chunks; ++c) {
      const int at = c + again < p.chunks ? c + again : c + again - p.chunks;
      if (PASS == kFused && c == (again ? stayed : 1)) {
        from = r;
        if (!again) from.back(begun + stayed - 1);
      }
      wait_or_mark(&sh.full[from.slot], from.phase, sh);
      const uint4* in = slots + from.slot * S::kChunk;
      const int j0 = at * S::kChunk, nv = min(S::kChunk, p.nv - j0);
      const bool hot_here = (unsigned)(hot_vec - j0) < (unsigned)nv;
      if (vec && !o.zero && nv == S::kChunk && !hot_here) {
#pragma unroll
        for (int u = 0; u < S::kVecs; ++u) {
          float f[VE];
          unpack<T>(in[tid + u * S::kGroup], f);
          grad_columns<ENT, T>(f, o, ks);
          __stcs(out + j0 + tid + u * S::kGroup, pack<T>(f));
        }
      } else {
        for (int j = tid; j < nv; j += S::kGroup) {
          float f[VE] = {};
          if (!o.zero) {
            unpack<T>(in[j], f);
            grad_columns<ENT, T>(f, o, ks);
            if (j0 + j == hot_vec) {
              const int hot = (o.tok - p.head) % VE;
#pragma unroll
              for (int q = 0; q < VE; ++q)
                if (q == hot) f[q] += o.h;
            }
          }
          store(j0 + j, pack<T>(f));
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.empty[from.slot]);
      from.next();
    }
    if (PASS == kBackward || again) r = from;
    if (tid < edge) {
      float v = o.zero ? 0.f : grad_of<ENT, T>(as_float(p.x[edge_col]), o, ks);
      if (!o.zero && edge_col == o.tok) v += o.h;
      put(g + edge_col, v);
    }
    if (KIND == kDistill) {
      // The list's columns, over what their vectors wrote.
      if (PASS == kBackward) wait_or_mark(&sh.teacher_full[par], phase, sh);
      asm volatile("bar.sync 1, %0;" ::"n"(S::kGroup) : "memory");
      const auto& q = sh.teacher[par];
      const int c0 = p.head + p.v0 * VE, c1 = c0 + p.nv * VE;
      for (int e = tid; e < A.k && !o.zero; e += S::kGroup) {
        const int id = q.id[e];
        if (id >= 0 && ((id >= c0 && id < c1) || (rank == 0 && (id < p.head || id >= p.head + p.nvec * VE))))
          put(g + id, grad_of<false, T>(PASS == kFused ? q.x[e] : as_float(p.x[id]), o, ks) - wt * q.q[e]);
      }
    }
    __syncwarp();
    if (lane == 0) {
      mbar_arrive(&sh.grad_empty[par]);
      if (KIND == kDistill) mbar_arrive(&sh.teacher_empty[par]);
    }
  }
}

// Rows of a loss: sums, terms, gradient.
//
// Bound by HBM and the exponentials: a scored row is read once and its gradient written once, with two exponentials a
// column.  A CTA keeps its rows in a ring of bulk copies: the gradient is made mostly from the chunks still in the
// ring, the rest is read again while it is in L2.  One warp copies, one takes a finished row's sums to its
// coefficients, the others work on the columns.  Few rows are spread over clusters: each CTA has a part of the
// columns, and the parts' sums cross by distributed shared memory.
template <typename T, int KIND, bool ENT, int PASS, typename S>
__global__ void __launch_bounds__(S::kThreads, S::kCtas) loss_rows_kernel(const LossArgs A) {
  using Sh = LossShared<S, PASS == kFused, SumOf<KIND, PASS>>;
  extern __shared__ __align__(128) uint8_t dyn[];
  uint4* slots = reinterpret_cast<uint4*>(dyn);
  Sh& sh = *reinterpret_cast<Sh*>(dyn + S::kRingBytes);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = cluster_rank(), size = cluster_size();
  if (tid == 0) {
    for (int i = 0; i < S::kSlots; ++i) mbar_init(&sh.full[i], 1), mbar_init(&sh.empty[i], S::kWarps);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.part_full[i], S::kWarps), mbar_init(&sh.part_empty[i], 1);
      mbar_init(&sh.grad_full[i], 1), mbar_init(&sh.grad_empty[i], S::kWarps);
      mbar_init(&sh.teacher_full[i], 1), mbar_init(&sh.teacher_empty[i], PASS == kForward ? 1 : S::kWarps);
      mbar_init(&sh.peers[i], 1);
    }
    sh.gave_up = 0;
    fence_barrier_init();
  }
  __syncthreads();
  if (size > 1) cluster_sync_all();
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (PASS != kBackward) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int n = A.batch * A.length, first = blockIdx.x / size, step = gridDim.x / size;
  const int row0 = first < n ? A.list[first] : 0;  // (on its way beside the count)
  const int n_active = A.hdr->n_active;
  if (warp == S::kCopyWarp) {
    if (lane == 0) copy_rows<T, PASS, S>(A, sh, slots, rank, size, first, step, n_active, row0);
  } else if (warp == S::kTeacherWarp) {
    if (KIND == kDistill) teacher_rows<T, PASS, S>(A, sh, rank, size, first, step, n_active, row0, lane);
  } else if (warp == S::kTermsWarp) {
    term_rows<T, KIND, ENT, PASS, S>(A, sh, rank, size, first, step, n_active, n, row0, lane);
  } else {
    column_rows<T, KIND, ENT, PASS, S>(A, sh, slots, rank, size, first, step, n_active, n, row0, tid);
  }
  __syncwarp();
  __syncthreads();
  if (size > 1) cluster_sync_all();  // no CTA leaves while its peers may still send to it
  if (tid == 0 && *(volatile int*)&sh.gave_up) {
    atomicExch(&A.hdr->error, 1);
    if (PASS != kForward && first < n) {  // (a gradient without a loss has no other sign)
      const int row = A.list[first], b = row / A.length;
      put((T*)A.g + b * A.gb + (row - b * A.length) * A.gr, NAN);
    }
  }
  if (PASS != kBackward && KIND != kPreference) {
    // The last CTA adds the rows' losses, always in the same order.
    if (tid == 0) {
      __threadfence();
      sh.last = atomicAdd(&A.hdr->ticket, 1) == (int)gridDim.x - 1;
    }
    __syncthreads();
    if (sh.last) {
      __threadfence();
      double sum = 0.0;
      for (int i = tid; i < n; i += S::kThreads) sum += __ldcg(A.row_val + i);  // (0 where a row is not scored)
      sum = warp_sum_d(sum);
      if (lane == 0) sh.sum[warp] = sum;
      __syncthreads();
      if (tid == 0) {
        for (int i = 1; i < S::kThreads / 32; ++i) sum += sh.sum[i];
        *A.loss = __ldcg(&A.hdr->error) ? NAN : (float)sum;
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Preference: sequence sums, margins, the loss and each sequence's dl/dlogp.

struct PairArgs {
  const uint8_t* mask;
  int64_t mb, mt;
  int32_t batch, length, normalised;
  const LossHeader* hdr;
  const float* ref;
  float beta, smoothing, scale;
  const double* row_val;
  const int32_t* seq_n;
  double* seq_sum;
  float *seq_g, *logprobs, *margins, *loss;
};

__global__ void __launch_bounds__(1024) loss_pair_kernel(const PairArgs A) {
  __shared__ double s_d[32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const double start = A.hdr->error ? (double)NAN : 0.0;  // (a NaN goes from the sums into all there is)
  for (int b = warp; b < A.batch; b += 32) {
    double sum = start;
    for (int t = lane; t < A.length; t += 32)
      if (A.mask == nullptr || A.mask[b * A.mb + t * A.mt] != 0) sum += A.row_val[b * A.length + t];
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    if (A.normalised) sum /= (double)max(A.seq_n[b], 1);
    if (lane == 0) {
      A.seq_sum[b] = sum;
      A.logprobs[b] = (float)sum;
    }
  }
  __syncthreads();
  const int pairs = A.batch / 2;
  double loss = 0.0;
  for (int p = tid; p < pairs; p += 1024) {
    const double rc = A.ref ? (double)A.ref[p] : 0.0, rr = A.ref ? (double)A.ref[p + pairs] : 0.0;
    const double m = (double)A.beta * ((A.seq_sum[p] - rc) - (A.seq_sum[p + pairs] - rr));
    const double eps = (double)A.smoothing;
    const double soft = log1p(exp(-fabs(m)));  // -log sigmoid(|m|)
    // (a term of weight 0 adds nothing, also where a sequence of probability 0 makes it infinite)
    if (eps < 1.0) loss += (1.0 - eps) * (soft + fmax(-m, 0.0));
    if (eps > 0.0) loss += eps * (soft + fmax(m, 0.0));
    if (m != m) loss = m;  // (fmax drops a NaN)
    const double sig = m >= 0.0 ? 1.0 / (1.0 + exp(-m)) : exp(m) / (1.0 + exp(m));
    const double neg = m >= 0.0 ? exp(-m) / (1.0 + exp(-m)) : 1.0 / (1.0 + exp(m));  // 1 - sig, without the loss of digits
    const double slope = (eps * sig - (1.0 - eps) * neg) * (double)A.beta * (double)A.scale / pairs;
    A.margins[p] = (float)m;
    A.seq_g[p] = (float)(slope / (A.normalised ? max(A.seq_n[p], 1) : 1));
    A.seq_g[p + pairs] = (float)(-slope / (A.normalised ? max(A.seq_n[p + pairs], 1) : 1));
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) loss += __shfl_xor_sync(0xffffffffu, loss, off);
  if (lane == 0) s_d[warp] = loss;
  __syncthreads();
  if (tid == 0) {
    double sum = 0.0;
    for (int i = 0; i < 32; ++i) sum += s_d[i];
    *A.loss = (float)(sum * (double)A.scale / max(pairs, 1));
  }
}

// ---------------------------------------------------------------------------
// Host.

int64_t up256(int64_t n) { return (n + 255) / 256 * 256; }

struct Layout {
  int64_t list, row_val, rec, seq_n, seq_w, seq_g, seq_sum, total;
};

Layout layout(int64_t batch, int64_t length) {
  const int64_t n = batch * length;
  Layout l;
  int64_t at = 256;
  l.row_val = at, at += up256(8 * n);
  l.rec = at, at += up256(16 * n);
  l.list = at, at += up256(4 * n);
  l.seq_sum = at, at += up256(8 * batch);
  l.seq_n = at, at += up256(4 * batch);
  l.seq_w = at, at += up256(4 * batch);
  l.seq_g = at, at += up256(4 * batch);
  l.total = at;
  return l;
}

template <typename T, int KIND, bool ENT, int PASS, typename S>
int32_t launch_shape(const LossArgs& a, cudaStream_t st) {
  constexpr int kBytes = S::kRingBytes + (int)sizeof(LossShared<S, PASS == kFused, SumOf<KIND, PASS>>);
  static_assert((kBytes + 1024) * S::kCtas <= 233472, "an SM's shared memory");
  int sms = 0;
  const int32_t e = sm_count(&sms);
  if (e != PKV_OK) return e;
  auto* kernel = loss_rows_kernel<T, KIND, ENT, PASS, S>;
  static bool ready[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 64 || !ready[dev]) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes) != cudaSuccess)
      return cuda_status("loss rows shared memory");
    if (dev < 64) ready[dev] = true;
  }
  const int64_t rows = (int64_t)a.batch * a.length;
  const int64_t row_bytes = (int64_t)a.vocab * sizeof(T);
  int c = row_cluster(rows, row_bytes, sms * S::kCtas);
  if (PASS == kFused && S::kCtas == 1 && c == 1 && rows > sms && sms * row_bytes > kRowsInL2) c = 2;
  const int grid = (int)std::min<int64_t>(rows, sms * S::kCtas / c) * c;
  return launch_after(kernel, grid, S::kThreads, c, kBytes, a, st, "loss rows launch");
}

template <typename T, int KIND, bool ENT, int PASS>
int32_t launch_typed(const LossArgs& a, cudaStream_t st) {
  if constexpr (PASS == kFused)
    if ((int64_t)a.vocab * (int64_t)sizeof(T) <= kShortRow) return launch_shape<T, KIND, ENT, PASS, ShortShape>(a, st);
  return launch_shape<T, KIND, ENT, PASS, ShapeOf<T, PASS>>(a, st);
}

template <int KIND, bool ENT, int PASS>
int32_t launch_rows(const LossArgs& a, int32_t dtype, cudaStream_t st) {
  if (dtype == PKV_F32) return launch_typed<float, KIND, ENT, PASS>(a, st);
  if (dtype == PKV_F16) return launch_typed<__half, KIND, ENT, PASS>(a, st);
  return launch_typed<__nv_bfloat16, KIND, ENT, PASS>(a, st);
}

LossArgs row_args(const pkv_loss_rows* r, const Layout& l, uint8_t* ws) {
  LossArgs a{};
  a.x = r->logits, a.xb = r->batch_stride, a.xr = r->row_stride;
  a.g = r->grad, a.gb = r->grad_batch_stride, a.gr = r->grad_row_stride;
  a.batch = r->batch, a.length = r->length, a.vocab = r->vocab;
  a.hdr = reinterpret_cast<LossHeader*>(ws);
  a.list = reinterpret_cast<const int32_t*>(ws + l.list);
  a.seq_w = reinterpret_cast<const float*>(ws + l.seq_w);
  a.row_val = reinterpret_cast<double*>(ws + l.row_val);
  a.rec = reinterpret_cast<float4*>(ws + l.rec);
  a.ks = scale_for(r->temperature, &a.kd);
  a.inv_t = (float)(1.0 / (double)r->temperature), a.temperature = r->temperature;
  a.inv_td = 1.0 / (double)r->temperature;
  return a;
}

int32_t launch_plan(const pkv_loss_rows* r, const Layout& l, uint8_t* ws, int32_t reduction, float scale,
                    cudaStream_t st) {
  PlanArgs p{r->mask, r->mask_batch_stride, r->mask_row_stride, r->batch, r->length, reduction, scale,
             reinterpret_cast<LossHeader*>(ws), reinterpret_cast<int32_t*>(ws + l.list),
             reinterpret_cast<float*>(ws + l.seq_w), reinterpret_cast<int32_t*>(ws + l.seq_n)};
  loss_plan_kernel<<<1, 1024, 0, st>>>(p);
  return cuda_status("loss plan launch");
}

template <typename T>
Tokens2<T> token_array(const pkv_token_array& t) {
  return Tokens2<T>{static_cast<const T*>(t.data), t.batch_stride, t.row_stride};
}

int32_t check_workspace(const pkv_loss_rows* r, const void* ws, int64_t bytes, const char* who) {
  if (!ws || (uintptr_t)ws % 256 || bytes < layout(r->batch, r->length).total)
    return fail(PKV_ERR_ARG, std::string(who) + ": the workspace is missing, unaligned or too small");
  return PKV_OK;
}

bool empty_rows(const pkv_loss_rows* r) { return (int64_t)r->batch * r->length == 0; }

}  // namespace

int32_t check_vocab_rows(const pkv_loss_rows* r, const char* who) {
  const std::string w(who);
  if (!r) return fail(PKV_ERR_ARG, w + ": no rows");
  if (r->batch < 0 || r->length < 0 || r->vocab < 1) return fail(PKV_ERR_ARG, w + ": invalid sizes");
  if ((int64_t)r->batch * r->length > INT32_MAX / 2) return fail(PKV_ERR_UNSUPPORTED, w + ": more than 2^30 rows");
  if (r->vocab > (1 << 30)) return fail(PKV_ERR_UNSUPPORTED, w + ": more than 2^30 columns");
  if (r->dtype != PKV_F32 && r->dtype != PKV_F16 && r->dtype != PKV_BF16)
    return fail(PKV_ERR_ARG, w + ": unknown dtype");
  if (!(r->temperature >= 1e-6f && r->temperature <= 1e6f))
    return fail(PKV_ERR_ARG, w + ": the temperature must lie in [1e-6, 1e6]");
  const int64_t size = r->dtype == PKV_F32 ? 4 : 2;
  if ((int64_t)r->batch * r->length > 0) {
    if (!r->logits || (uintptr_t)r->logits % size) return fail(PKV_ERR_ARG, w + ": logits pointer");
    if ((uintptr_t)r->grad % size) return fail(PKV_ERR_ARG, w + ": gradient pointer");
    if ((r->length > 1 && r->row_stride < 0) || (r->batch > 1 && r->batch_stride < 0))
      return fail(PKV_ERR_ARG, w + ": negative strides");
    if (r->grad) {
      // Every gradient row has a place of its own.
      const int64_t rs = r->length > 1 ? r->grad_row_stride : r->vocab;
      const int64_t span = (r->length - 1) * rs + r->vocab;
      if (rs < r->vocab || (r->batch > 1 && r->grad_batch_stride < span))
        return fail(PKV_ERR_ARG, w + ": gradient rows overlap");
      auto extent = [&](int64_t bs, int64_t rst) {
        return ((r->batch - 1) * (r->batch > 1 ? bs : 0) + (r->length - 1) * (r->length > 1 ? rst : 0) + r->vocab) * size;
      };
      const uintptr_t x0 = (uintptr_t)r->logits, g0 = (uintptr_t)r->grad;
      if (g0 < x0 + extent(r->batch_stride, r->row_stride) && x0 < g0 + extent(r->grad_batch_stride, r->grad_row_stride))
        return fail(PKV_ERR_ARG, w + ": the gradient overlaps the logits");
    }
  }
  return PKV_OK;
}

}  // namespace pkv

using namespace pkv;

extern "C" int64_t pkv_loss_workspace_bytes(int32_t batch, int32_t length) {
  if (batch < 0 || length < 0 || (int64_t)batch * length > INT32_MAX / 2) return -1;
  return layout(batch, length).total;
}

extern "C" int32_t pkv_policy_loss(const pkv_loss_rows* r, const pkv_policy_terms* p, float* loss, float* logprobs,
                                   float* kl, float* entropy, void* workspace, int64_t workspace_bytes, void* stream) {
  pkv_clear_error();
  int32_t st = check_vocab_rows(r, "policy_loss");
  if (st != PKV_OK) return st;
  if (!p || !loss) return fail(PKV_ERR_ARG, "policy_loss: terms and a loss output are required");
  if (p->reduction < PKV_TOKEN_MEAN || p->reduction > PKV_SUM) return fail(PKV_ERR_ARG, "policy_loss: unknown reduction");
  if (!(p->clip_low >= 0.f) || !(p->clip_high >= 0.f)) return fail(PKV_ERR_ARG, "policy_loss: clip ranges are >= 0");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (empty_rows(r)) {
    cudaMemsetAsync(loss, 0, 4, s);
    return cuda_status("policy_loss");
  }
  if ((st = check_workspace(r, workspace, workspace_bytes, "policy_loss")) != PKV_OK) return st;
  if (!p->tokens.data || !p->advantages.data || !logprobs)
    return fail(PKV_ERR_ARG, "policy_loss: tokens, advantages and a log-probability output are required");
  const Layout l = layout(r->batch, r->length);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  LossArgs a = row_args(r, l, ws);
  a.tokens = token_array<int64_t>(p->tokens);
  a.adv = token_array<float>(p->advantages);
  a.old = token_array<float>(p->old_logprobs);
  a.ref = token_array<float>(p->ref_logprobs);
  a.ratio_low = (float)(1.0 - (double)p->clip_low), a.ratio_high = (float)(1.0 + (double)p->clip_high);
  a.kl_coef = p->kl_coef, a.ent_coef = p->entropy_coef;
  a.logprobs = logprobs, a.kl_out = kl, a.entropy = entropy, a.loss = loss;
  if ((st = launch_plan(r, l, ws, p->reduction, p->scale, s)) != PKV_OK) return st;
  const bool ent = p->entropy_coef != 0.f || entropy;
  if (r->grad) return ent ? launch_rows<kPolicy, true, kFused>(a, r->dtype, s) : launch_rows<kPolicy, false, kFused>(a, r->dtype, s);
  return ent ? launch_rows<kPolicy, true, kForward>(a, r->dtype, s) : launch_rows<kPolicy, false, kForward>(a, r->dtype, s);
}

extern "C" int32_t pkv_preference_loss(const pkv_loss_rows* r, const pkv_preference_terms* p, float* loss,
                                       float* logprobs, float* margins, void* workspace, int64_t workspace_bytes,
                                       void* stream) {
  pkv_clear_error();
  int32_t st = check_vocab_rows(r, "preference_loss");
  if (st != PKV_OK) return st;
  if (!p || !loss) return fail(PKV_ERR_ARG, "preference_loss: terms and a loss output are required");
  if (r->batch % 2) return fail(PKV_ERR_ARG, "preference_loss: chosen and rejected sequences, an even number of them");
  if (!(p->label_smoothing >= 0.f && p->label_smoothing <= 1.f))
    return fail(PKV_ERR_ARG, "preference_loss: the label smoothing lies in [0, 1]");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (r->batch == 0) {
    cudaMemsetAsync(loss, 0, 4, s);
    return cuda_status("preference_loss");
  }
  if ((st = check_workspace(r, workspace, workspace_bytes, "preference_loss")) != PKV_OK) return st;
  if (!logprobs || !margins || (!p->tokens.data && r->length))
    return fail(PKV_ERR_ARG, "preference_loss: tokens, log-probability and margin outputs are required");
  const Layout l = layout(r->batch, r->length);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  LossArgs a = row_args(r, l, ws);
  a.tokens = token_array<int64_t>(p->tokens);
  if ((st = launch_plan(r, l, ws, PKV_SUM, 1.f, s)) != PKV_OK) return st;
  if (!empty_rows(r) && (st = launch_rows<kPreference, false, kForward>(a, r->dtype, s)) != PKV_OK) return st;
  PairArgs q{r->mask, r->mask_batch_stride, r->mask_row_stride, r->batch, r->length, p->length_normalised,
             a.hdr, p->ref_logprobs, p->beta, p->label_smoothing, p->scale,
             reinterpret_cast<const double*>(ws + l.row_val), reinterpret_cast<const int32_t*>(ws + l.seq_n),
             reinterpret_cast<double*>(ws + l.seq_sum), reinterpret_cast<float*>(ws + l.seq_g), logprobs, margins, loss};
  if ((st = launch_after(loss_pair_kernel, 1, 1024, 1, 0, q, s, "preference pairs launch")) != PKV_OK) return st;
  if (!r->grad || empty_rows(r)) return PKV_OK;
  a.seq_g = q.seq_g;
  return launch_rows<kPreference, false, kBackward>(a, r->dtype, s);
}

extern "C" int32_t pkv_distillation_loss(const pkv_loss_rows* r, const pkv_distillation_terms* p, float* loss,
                                         float* kl, void* workspace, int64_t workspace_bytes, void* stream) {
  pkv_clear_error();
  int32_t st = check_vocab_rows(r, "distillation_loss");
  if (st != PKV_OK) return st;
  if (!p || !loss) return fail(PKV_ERR_ARG, "distillation_loss: terms and a loss output are required");
  if (p->reduction < PKV_TOKEN_MEAN || p->reduction > PKV_SUM)
    return fail(PKV_ERR_ARG, "distillation_loss: unknown reduction");
  if (p->k < 1 || p->k > PKV_MAX_TOP) return fail(PKV_ERR_UNSUPPORTED, "distillation_loss: 1 to 256 teacher entries a row");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (empty_rows(r)) {
    cudaMemsetAsync(loss, 0, 4, s);
    return cuda_status("distillation_loss");
  }
  if ((st = check_workspace(r, workspace, workspace_bytes, "distillation_loss")) != PKV_OK) return st;
  if (!p->ids || !p->teacher_logits || !kl)
    return fail(PKV_ERR_ARG, "distillation_loss: teacher ids, teacher logits and a per-row output are required");
  const Layout l = layout(r->batch, r->length);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  LossArgs a = row_args(r, l, ws);
  a.ids = p->ids, a.ids_b = p->ids_batch_stride, a.ids_t = p->ids_row_stride;
  a.tl = p->teacher_logits, a.tl_b = p->logits_batch_stride, a.tl_t = p->logits_row_stride;
  a.k = p->k, a.tlse = token_array<float>(p->teacher_lse);
  a.kl_out = kl, a.loss = loss;
  if ((st = launch_plan(r, l, ws, p->reduction, p->scale, s)) != PKV_OK) return st;
  return r->grad ? launch_rows<kDistill, false, kFused>(a, r->dtype, s) : launch_rows<kDistill, false, kForward>(a, r->dtype, s);
}

extern "C" int32_t pkv_policy_loss_backward(const pkv_loss_rows* r, const pkv_policy_terms* p, const float* upstream,
                                            void* workspace, int64_t workspace_bytes, void* stream) {
  pkv_clear_error();
  int32_t st = check_vocab_rows(r, "policy_loss_backward");
  if (st != PKV_OK || empty_rows(r)) return st;
  if ((st = check_workspace(r, workspace, workspace_bytes, "policy_loss_backward")) != PKV_OK) return st;
  if (!p || !r->grad || !p->tokens.data) return fail(PKV_ERR_ARG, "policy_loss_backward: tokens and a gradient output are required");
  LossArgs a = row_args(r, layout(r->batch, r->length), static_cast<uint8_t*>(workspace));
  a.tokens = token_array<int64_t>(p->tokens);
  a.upstream = upstream;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return p->entropy_coef != 0.f ? launch_rows<kPolicy, true, kBackward>(a, r->dtype, s)
                                : launch_rows<kPolicy, false, kBackward>(a, r->dtype, s);
}

extern "C" int32_t pkv_preference_loss_backward(const pkv_loss_rows* r, const pkv_preference_terms* p,
                                                const float* upstream, void* workspace, int64_t workspace_bytes,
                                                void* stream) {
  pkv_clear_error();
  int32_t st = check_vocab_rows(r, "preference_loss_backward");
  if (st != PKV_OK || empty_rows(r)) return st;
  if ((st = check_workspace(r, workspace, workspace_bytes, "preference_loss_backward")) != PKV_OK) return st;
  if (!p || !r->grad || !p->tokens.data)
    return fail(PKV_ERR_ARG, "preference_loss_backward: tokens and a gradient output are required");
  const Layout l = layout(r->batch, r->length);
  LossArgs a = row_args(r, l, static_cast<uint8_t*>(workspace));
  a.tokens = token_array<int64_t>(p->tokens);
  a.seq_g = reinterpret_cast<const float*>(static_cast<uint8_t*>(workspace) + l.seq_g);
  a.upstream = upstream;
  return launch_rows<kPreference, false, kBackward>(a, r->dtype, static_cast<cudaStream_t>(stream));
}

extern "C" int32_t pkv_distillation_loss_backward(const pkv_loss_rows* r, const pkv_distillation_terms* p,
                                                  const float* upstream, void* workspace, int64_t workspace_bytes,
                                                  void* stream) {
  pkv_clear_error();
  int32_t st = check_vocab_rows(r, "distillation_loss_backward");
  if (st != PKV_OK || empty_rows(r)) return st;
  if ((st = check_workspace(r, workspace, workspace_bytes, "distillation_loss_backward")) != PKV_OK) return st;
  if (!p || !r->grad || !p->ids || !p->teacher_logits)
    return fail(PKV_ERR_ARG, "distillation_loss_backward: the teacher's list and a gradient output are required");
  if (p->k < 1 || p->k > PKV_MAX_TOP)
    return fail(PKV_ERR_UNSUPPORTED, "distillation_loss_backward: 1 to 256 teacher entries a row");
  LossArgs a = row_args(r, layout(r->batch, r->length), static_cast<uint8_t*>(workspace));
  a.ids = p->ids, a.ids_b = p->ids_batch_stride, a.ids_t = p->ids_row_stride;
  a.tl = p->teacher_logits, a.tl_b = p->logits_batch_stride, a.tl_t = p->logits_row_stride;
  a.k = p->k, a.tlse = token_array<float>(p->teacher_lse);
  a.upstream = upstream;
  return launch_rows<kDistill, false, kBackward>(a, r->dtype, static_cast<cudaStream_t>(stream));
}
