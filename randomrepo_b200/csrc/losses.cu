// Losses over vocabulary rows and their gradients, for sm_100a: the clipped
// policy loss (with KL and entropy terms), the preference loss over pairs of
// sequences, and distillation from a teacher's top logits.
//
// A row is one position's `vocab` logits x.  With z = x / T everything a loss
// needs of a row is its base-2 log-sum-exp pair (m, s): m = max x, y_j =
// (x_j - m) k, k = log2(e) / T, e_j = 2^y_j, s = sum e_j, p_j = e_j / s (and
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
#include "pkv_error.h"

namespace pkv {
namespace {

constexpr int kLossThreads = 512;
constexpr int kLossWarps = kLossThreads / 32;
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
  float4* rec;            // [rows] {m, a, b, h} for a later backward pass (distillation: {m, a, w T, log q's norm})
  const float* upstream;  // device scalar the gradient is multiplied by, or null
};

__device__ __forceinline__ RowSum cta_sum(RowSum a, RowSum* smem, Scale2 k) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    RowSum b;
    b.m = __shfl_xor_sync(0xffffffffu, a.m, off);
    b.s = __shfl_xor_sync(0xffffffffu, a.s, off);
    b.w = __shfl_xor_sync(0xffffffffu, a.w, off);
    sum_merge(a, b, k);
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) smem[threadIdx.x >> 5] = a;
  __syncthreads();
  a = smem[0];
  for (int i = 1; i < kLossWarps; ++i) sum_merge(a, smem[i], k);
  return a;
}

// What a row's gradient needs: dx_j = e_j (a + b y_j), + h at the token.
struct RowGrad {
  float m, a, b, h;
  int tok;
  bool zero;  // the gradient is zero whatever the logits
};

template <bool ENT>
__device__ RowGrad policy_tail(const LossArgs& A, int row, int b, int t, RowSum r, float x_tok, int64_t tok, bool write) {
  const bool known = tok >= 0 && tok < A.vocab;
  const double log2s = log2_of(r.s);
  const double lp = known ? (((double)x_tok - (double)r.m) * A.kd - log2s) * kLn2d : (double)NAN;
  const float w = A.seq_w[b], adv = A.adv.at(b, t);
  const float ratio = A.old.p ? expf((float)(lp - (double)A.old.at(b, t))) : (lp == lp ? 1.f : NAN);
  // -min(r A, clip(r) A): the clipped branch is the smaller one above the border for A > 0, below it for A < 0.
  const bool cut = (adv > 0.f && ratio > A.ratio_high) || (adv < 0.f && ratio < A.ratio_low);
  const float used = cut ? (adv > 0.f ? A.ratio_high : A.ratio_low) : ratio;
  float l = adv == 0.f ? 0.f : -used * adv;
  float g = (cut || adv == 0.f) ? 0.f : -ratio * adv;
  if (!(lp == lp)) l = g = NAN;
  float kl = 0.f;
  if (A.ref.p) {
    const float d = (float)((double)A.ref.at(b, t) - lp);
    const float em = expm1f(d);
    kl = em - d;
    l = fmaf(A.kl_coef, kl, l);
    g = fmaf(-A.kl_coef, em, g);
  }
  g *= w * A.inv_t;
  const float inv_s = 1.f / r.s;
  RowGrad o{r.m, -g * inv_s, 0.f, g, known ? (int)tok : -1, false};
  float h = 0.f;
  if (ENT) {
    const double mean = (double)r.w / (double)r.s;
    h = (float)((log2s - mean) * kLn2d);
    const float c = A.ent_coef * w * A.inv_t;
    l = fmaf(-A.ent_coef, h, l);
    o.a = fmaf(c * inv_s, (float)(-kLn2d * mean), o.a);  // H - ln2 log2 s = -ln2 w / s
    o.b = c * kLn2 * inv_s;
  }
  o.zero = !ENT && g == 0.f;
  if (write) {
    A.logprobs[row] = (float)lp;
    if (A.kl_out) A.kl_out[row] = kl;
    if (ENT && A.entropy) A.entropy[row] = h;
    A.row_val[row] = (double)w * (double)l;
  }
  return o;
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

__global__ void __launch_bounds__(1024) loss_plan_kernel(const PlanArgs A) {
  __shared__ int s_warp[33], s_full, s_total;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int n = A.batch * A.length;
  auto scored = [&](int b, int t) { return A.mask == nullptr || A.mask[b * A.mb + t * A.mt] != 0; };
  if (tid == 0) s_full = 0;
  __syncthreads();
  for (int b = warp; b < A.batch; b += 32) {
    int c = 0;
    for (int t = lane; t < A.length; t += 32) c += scored(b, t);
    c = __reduce_add_sync(0xffffffffu, c);
    if (lane == 0) {
      A.seq_n[b] = c;
      if (c > 0) atomicAdd(&s_full, 1);
    }
  }
  // Each thread's run of rows: count, exclusive scan, then their places.
  const int per = (n + 1023) / 1024, r0 = min(n, tid * per), r1 = min(n, r0 + per);
  int mine = 0;
  for (int r = r0; r < r1; ++r) mine += scored(r / A.length, r % A.length);
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
  for (int r = r0; r < r1; ++r) {
    if (scored(r / A.length, r % A.length))
      A.list[at++] = r;
    else
      A.list[rest++] = r;
  }
  for (int b = tid; b < A.batch; b += 1024) {
    const int c = A.seq_n[b];
    float w = A.scale;
    if (A.reduction == PKV_TOKEN_MEAN) w = (float)((double)A.scale / max(total, 1));
    if (A.reduction == PKV_SEQUENCE_MEAN) w = (float)((double)A.scale / ((double)max(c, 1) * max(s_full, 1)));
    A.seq_w[b] = w;
  }
  if (tid == 0) {
    A.hdr->n_active = total;
    A.hdr->ticket = 0;
  }
}

// ---------------------------------------------------------------------------
// Rows.

template <bool ENT>
__device__ __forceinline__ float grad_of(float x, const RowGrad& o, Scale2 k) {
  const float d = x - o.m, y = fmaf(d, k.lo, d * k.hi);
  return ex2(y) * (ENT ? fmaf(o.b, fmaxf(y, -1e30f), o.a) : o.a);
}

__device__ __forceinline__ float teacher_logit(const LossArgs& A, int b, int t, int i, int64_t& id) {
  id = A.ids[b * A.ids_b + t * A.ids_t + i];
  const float v = A.tl[b * A.tl_b + t * A.tl_t + i];
  return id < 0 ? -INFINITY : v;  // an absent entry
}

__device__ double cta_sum_d(double v, double* smem) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) smem[threadIdx.x >> 5] = v;
  __syncthreads();
  v = smem[0];
  for (int i = 1; i < kLossWarps; ++i) v += smem[i];
  return v;
}

// The log-sum-exp of a row's teacher logits / T over its list, or the teacher's own.  Computed in 64 bits: log q
// would lose digits to a rounded norm.
__device__ double teacher_norm(const LossArgs& A, int b, int t, double* smem) {
  if (A.tlse.p) return (double)A.tlse.at(b, t);
  int64_t id;
  float top = -INFINITY;
  for (int e = 0; e < A.k; ++e) top = fmaxf(top, teacher_logit(A, b, t, e, id));
  if (top == -INFINITY) return 0.0;
  double sum = 0.0;
  for (int e = threadIdx.x; e < A.k; e += kLossThreads) {
    const float v = teacher_logit(A, b, t, e, id);
    if (v != -INFINITY) sum += (double)expf((float)(((double)v - (double)top) * A.inv_td));
  }
  sum = cta_sum_d(sum, smem);
  return (double)top * A.inv_td + log(sum);
}

template <typename T, int KIND, bool ENT, int PASS>
__global__ void __launch_bounds__(kLossThreads) loss_rows_kernel(const LossArgs A) {
  constexpr int VE = 16 / sizeof(T);
  __shared__ RowSum s_sum[kLossWarps];
  __shared__ double s_d[kLossWarps];
  __shared__ int s_last;
  const int tid = threadIdx.x;
  const int n = A.batch * A.length, n_active = A.hdr->n_active;
  const float up = A.upstream ? *A.upstream : 1.f;
  for (int i = blockIdx.x; i < n; i += gridDim.x) {
    const int row = A.list[i], b = row / A.length, t = row - b * A.length;
    const T* x = (const T*)A.x + b * A.xb + t * A.xr;
    T* g = (T*)A.g + b * A.gb + t * A.gr;
    const RowSplit<T> sp(x, A.vocab);
    const int edge = A.vocab - sp.nvec * VE;  // columns outside the body
    RowGrad o{0.f, 0.f, 0.f, 0.f, -1, i >= n_active};
    float wt = 0.f;
    double qnorm = 0.0;
    if (i >= n_active) {
      if (PASS != kBackward && tid == 0) {
        if (A.logprobs) A.logprobs[row] = 0.f;
        if (A.kl_out) A.kl_out[row] = 0.f;
        if (ENT && A.entropy) A.entropy[row] = 0.f;
        A.row_val[row] = 0.0;
      }
      if (PASS == kForward) continue;
    } else if (PASS == kBackward) {
      const float4 r = A.rec[row];
      const float f = up * (A.seq_g ? A.seq_g[b] : 1.f);
      o = RowGrad{r.x, r.y * f, r.z * f, r.w * f, -1, false};
      if (KIND == kDistill) {
        o.b = 0.f;
        wt = r.z * f;
        qnorm = teacher_norm(A, b, t, s_d);
        o.zero = f == 0.f;
      } else {
        const int64_t tok = A.tokens.at(b, t);
        o.tok = tok >= 0 && tok < A.vocab ? (int)tok : -1;
        o.zero = o.a == 0.f && o.b == 0.f && o.h == 0.f;
      }
    } else {
      RowSum r{-INFINITY, 0.f, 0.f};
      const uint4* body = reinterpret_cast<const uint4*>(x + sp.head);
      for (int j = tid; j < sp.nvec; j += kLossThreads) {
        float f[VE];
        unpack<T>(body[j], f);
        fold<ENT>(r, f, A.ks);
      }
      if (tid < edge) {
        const float f[1] = {as_float(x[tid < sp.head ? tid : tid + sp.nvec * VE])};
        fold<ENT>(r, f, A.ks);
      }
      r = cta_sum(r, s_sum, A.ks);
      if (KIND == kPolicy) {
        const int64_t tok = A.tokens.at(b, t);
        const float xt = tok >= 0 && tok < A.vocab ? as_float(x[tok]) : NAN;
        o = policy_tail<ENT>(A, row, b, t, r, xt, tok, tid == 0);
      } else if (KIND == kPreference) {
        const int64_t tok = A.tokens.at(b, t);
        const bool known = tok >= 0 && tok < A.vocab;
        const double lp = known ? (((double)as_float(x[tok]) - (double)r.m) * A.kd - log2_of(r.s)) * kLn2d
                                : (double)NAN;
        o = RowGrad{r.m, -1.f / r.s, 0.f, 1.f, 0, false};
        if (tid == 0) A.row_val[row] = lp;
      } else {
        // sum q (log q - log p) over the teacher's list.
        qnorm = teacher_norm(A, b, t, s_d);
        double l = 0.0, q_sum = 0.0;
        int64_t id;
        for (int e = tid; e < A.k; e += kLossThreads) {
          const float v = teacher_logit(A, b, t, e, id);
          if (v == -INFINITY) continue;
          const double lq = (double)v * A.inv_td - qnorm;
          const double lp = id < A.vocab ? (((double)as_float(x[id]) - (double)r.m) * A.kd - log2_of(r.s)) * kLn2d : (double)NAN;
          const float q = expf((float)lq);
          l += q == 0.f && lp == lp ? 0.0 : (double)q * (lq - lp);
          q_sum += (double)q;
        }
        l = cta_sum_d(l, s_d);
        q_sum = cta_sum_d(q_sum, s_d);
        const float w = A.seq_w[b];
        wt = w * A.temperature;
        l *= (double)A.temperature * (double)A.temperature;
        o = RowGrad{r.m, wt * (float)q_sum / r.s, 0.f, 0.f, -1, false};
        if (l != l) o.a = NAN;
        if (tid == 0) {
          A.kl_out[row] = (float)l;
          A.row_val[row] = (double)w * l;
        }
      }
      if (PASS == kForward) {
        if (tid == 0 && A.rec)
          A.rec[row] = KIND == kDistill ? make_float4(o.m, o.a, wt, 0.f) : make_float4(o.m, o.a, o.b, o.h);
        continue;
      }
    }
    uint4* out = reinterpret_cast<uint4*>(g + sp.head);
    const bool vec = ((uintptr_t)out & 15) == 0;
    const uint4* body = reinterpret_cast<const uint4*>(x + sp.head);
    for (int j = tid; j < sp.nvec; j += kLossThreads) {
      float f[VE] = {};
      if (!o.zero) {
        unpack<T>(body[j], f);
        const int hot = o.tok - (sp.head + j * VE);
#pragma unroll
        for (int q = 0; q < VE; ++q) f[q] = grad_of<ENT>(f[q], o, A.ks) + (q == hot ? o.h : 0.f);
      }
      if (vec) {
        out[j] = pack<T>(f);
      } else {
#pragma unroll
        for (int q = 0; q < VE; ++q) put(g + sp.head + j * VE + q, f[q]);
      }
    }
    if (tid < edge) {
      const int j = tid < sp.head ? tid : tid + sp.nvec * VE;
      put(g + j, o.zero ? 0.f : grad_of<ENT>(as_float(x[j]), o, A.ks) + (j == o.tok ? o.h : 0.f));
    }
    if (KIND == kDistill && i < n_active && !o.zero) {
      // The list's columns: an id that comes twice is written once, with both its shares.
      __syncthreads();
      for (int e = tid; e < A.k; e += kLossThreads) {
        int64_t id, other;
        const float v = teacher_logit(A, b, t, e, id);
        if (id < 0 || id >= A.vocab) continue;
        float q = expf((float)((double)v * A.inv_td - qnorm));
        bool first = true;
        for (int f = 0; f < A.k; ++f) {
          if (f == e) continue;
          const float u = teacher_logit(A, b, t, f, other);
          if (other != id) continue;
          first = first && f > e;
          q += expf((float)((double)u * A.inv_td - qnorm));
        }
        if (first) put(g + id, grad_of<false>(as_float(x[id]), o, A.ks) - wt * q);
      }
    }
  }
  if (PASS == kBackward || KIND == kPreference) return;
  // The last CTA adds the rows' losses, always in the same order.
  __syncthreads();
  if (tid == 0) {
    __threadfence();
    s_last = atomicAdd(&A.hdr->ticket, 1) == (int)gridDim.x - 1;
  }
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  double sum = 0.0;
  for (int i = tid; i < n_active; i += kLossThreads) sum += __ldcg(A.row_val + A.list[i]);
  sum = cta_sum_d(sum, s_d);
  if (tid == 0) *A.loss = (float)sum;
}

// ---------------------------------------------------------------------------
// Preference: sequence sums, margins, the loss and each sequence's dl/dlogp.

struct PairArgs {
  const uint8_t* mask;
  int64_t mb, mt;
  int32_t batch, length, normalised;
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
  for (int b = warp; b < A.batch; b += 32) {
    double sum = 0.0;
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
    loss += (1.0 - eps) * (soft + fmax(-m, 0.0)) + eps * (soft + fmax(m, 0.0));
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

int32_t fail(int32_t status, const std::string& msg) {
  pkv_set_error(msg);
  return status;
}

int32_t cuda_status(const char* what) {
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) return PKV_OK;
  return fail(PKV_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
}

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

template <int KIND, bool ENT, int PASS>
int32_t launch_rows(const LossArgs& a, int32_t dtype, cudaStream_t st) {
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return cuda_status("device query");
  const int grid = (int)std::min<int64_t>((int64_t)a.batch * a.length, 4ll * sms);
  if (dtype == PKV_F32)
    loss_rows_kernel<float, KIND, ENT, PASS><<<grid, kLossThreads, 0, st>>>(a);
  else if (dtype == PKV_F16)
    loss_rows_kernel<__half, KIND, ENT, PASS><<<grid, kLossThreads, 0, st>>>(a);
  else
    loss_rows_kernel<__nv_bfloat16, KIND, ENT, PASS><<<grid, kLossThreads, 0, st>>>(a);
  return cuda_status("loss rows launch");
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
  a.kd = kLog2ed / (double)r->temperature;
  a.ks.hi = (float)a.kd, a.ks.lo = (float)(a.kd - (double)a.ks.hi);
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
  if (!(r->temperature > 0.f) || !std::isfinite(r->temperature))
    return fail(PKV_ERR_ARG, w + ": the temperature must be positive and finite");
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
             p->ref_logprobs, p->beta, p->label_smoothing, p->scale,
             reinterpret_cast<const double*>(ws + l.row_val), reinterpret_cast<const int32_t*>(ws + l.seq_n),
             reinterpret_cast<double*>(ws + l.seq_sum), reinterpret_cast<float*>(ws + l.seq_g), logprobs, margins, loss};
  loss_pair_kernel<<<1, 1024, 0, s>>>(q);
  if ((st = cuda_status("preference pairs launch")) != PKV_OK) return st;
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
