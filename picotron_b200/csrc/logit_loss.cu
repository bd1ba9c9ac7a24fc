// Post-training losses over vocabulary rows on sm_100a: the log-probability of each row's target
// (forward and backward), the preference loss of chosen / rejected pairs and the clipped policy
// loss with a KL term, each with the gradient of its logits.
//
// For a row x with target t:
//   m = max(x),  s = sum 2^((x - m) log2 e),  log softmax(x)_t = (x_t - m) - ln s.
// x is taken relative to m before it is scaled, so a row of one type's lowest values (a mask
// that leaves nothing) neither overflows nor loses its s; s is held in 32 bits per thread and
// merged in 32 bits, ln s and the differences are taken in 64 bits and the log-probability is
// rounded once. Every loss here depends on the logits through these log-probabilities alone,
// so its gradient is
//   dx = c (onehot(t) - softmax(x)),  softmax(x) = 2^((x - m) log2 e) / s,
// with one coefficient c per row: the forward keeps (m, 1/s) and c, the backward reads the
// logits once more and writes dx. All passes over the logits are bound by HBM bandwidth.
//
// Rows form an [outer, inner] grid addressed by two strides (sequences x positions). Rows whose
// target is ignore_index are not read at all; their gradient is stored as zeros.

#include <algorithm>
#include <cmath>

#include "common.cuh"

namespace pt {

__device__ int g_logit_loss_error = 0;

namespace {

// Rows per CTA and vectors in flight as for the cross-entropy kernels, which read the same
// rows: 128 threads, 8 vectors in flight where rows are only read, 4 where dx is written too.
constexpr int kThreads = 128;
constexpr int kUnrollStats = 8;
constexpr int kUnrollGrad = 4;
constexpr int kSumThreads = 1024;
constexpr float kLog2e = 1.4426950408889634f;  // log2(e): exp(a) = 2^(a log2(e))
constexpr int kErrBadTarget = 2;

// Row r of the [outer, inner] row grid sits at outer index r / inner, inner index r % inner.
struct RowGrid {
  int64_t inner;
  int64_t outer_stride, inner_stride;  // elements
  __device__ __forceinline__ int64_t offset(int64_t r) const {
    const int64_t o = r / inner;
    return o * outer_stride + (r - o * inner) * inner_stride;
  }
};

struct Targets {
  const int64_t* p;
  RowGrid g;
  int64_t ignore;
  __device__ __forceinline__ int64_t at(int64_t r) const { return p[g.offset(r)]; }
};

// A set of values x as (max, sum of e^(x - max)); m = -inf and s = 0 for the empty set.
struct Stat {
  float m, s;
};

// 2^x on the special-function unit (PTX ex2.approx.ftz, relative error below 2^-22).
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float fast_exp(float a) { return fast_exp2(a * kLog2e); }

__device__ __forceinline__ Stat merge(Stat a, Stat b) {
  const float m = fmaxf(a.m, b.m);
  const float fa = a.m == -INFINITY ? 0.0f : fast_exp(a.m - m);
  const float fb = b.m == -INFINITY ? 0.0f : fast_exp(b.m - m);
  // A NaN sum survives even where its factor is 0 (NaN * 0).
  return {m, fmaf(a.s, fa, b.s * fb)};
}

__device__ __forceinline__ Stat warp_merge(Stat v) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1)
    v = merge(v, Stat{__shfl_xor_sync(0xffffffffu, v.m, off),
                      __shfl_xor_sync(0xffffffffu, v.s, off)});
  return v;
}

// Merged over the CTA; valid in warp 0. `red` holds one Stat per warp.
__device__ __forceinline__ Stat block_merge(Stat v, Stat* red) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  v = warp_merge(v);
  if (lane == 0) red[warp] = v;
  __syncthreads();
  if (warp == 0) v = warp_merge(lane < nw ? red[lane] : Stat{-INFINITY, 0.0f});
  return v;
}

// Per-thread running statistics: two partial sums (paired fp32 lanes) relative to m.
struct Running {
  float m = -INFINITY;
  float2 s = make_float2(0.0f, 0.0f);
  __device__ __forceinline__ void raise(float xmax) {
    if (xmax > m) {
      s = __fmul2_rn(s, splat2(m == -INFINITY ? 0.0f : fast_exp(m - xmax)));
      m = xmax;
    }
  }
  // What x is taken relative to. Only -inf (which add 0) or NaN so far: 0 gives those results.
  __device__ __forceinline__ float base() const { return m == -INFINITY ? 0.0f : m; }
  // Adds N values (N even).
  template <int N> __device__ __forceinline__ void add(const float* x) {
    float vmax = x[0];
#pragma unroll
    for (int e = 1; e < N; ++e) vmax = fmaxf(vmax, x[e]);
    raise(vmax);
    const float2 L = splat2(kLog2e), nm = splat2(-base());
#pragma unroll
    for (int e = 0; e < N; e += 2) {
      const float2 t = __fmul2_rn(__fadd2_rn(make_float2(x[e], x[e + 1]), nm), L);
      s = __fadd2_rn(s, make_float2(fast_exp2(t.x), fast_exp2(t.y)));
    }
  }
  __device__ __forceinline__ void add1(float x) {
    raise(x);
    s.x += fast_exp(x - base());
  }
  __device__ __forceinline__ Stat stat() const { return {m, s.x + s.y}; }
};

// log softmax at the value xt. The differences are taken first: m may be as large as the type
// allows, where m + ln s would absorb ln s.
__device__ __forceinline__ double log_softmax(Stat v, float xt) {
  return ((double)xt - (double)v.m) - log((double)v.s);
}

// Elements before the first 16-byte boundary of a row (0 when it is aligned).
template <typename T> __device__ __forceinline__ int head_elems(const T* p, int64_t vocab) {
  const int mis = (int)(reinterpret_cast<uintptr_t>(p) & 15u);
  const int h = mis ? (16 - mis) / (int)sizeof(T) : 0;
  return (int64_t)h < vocab ? h : (int)vocab;
}

// The part of a row that split `k` of `n` takes: whole 16-byte vectors [v0, v1) of the aligned
// body, the unaligned head with the first split and the tail with the last.
struct Part {
  int64_t v0, v1;
  __device__ __forceinline__ Part(int64_t nvec, int k, int n) {
    const int64_t per = (nvec + n - 1) / n;
    v0 = min(nvec, per * k);
    v1 = min(nvec, v0 + per);
  }
};

enum RowKind { kRowIgnored, kRowBad, kRowUsed };
__device__ __forceinline__ RowKind row_kind(int64_t t, int64_t ignore, int64_t vocab) {
  return t == ignore ? kRowIgnored : (t < 0 || t >= vocab) ? kRowBad : kRowUsed;
}

// Per-row outputs of the forward passes, dense [rows]. logps32 and logps64 may be null.
struct RowOut {
  float2* stats;    // (m, 1/s)
  float* logps32;
  double* logps64;
  __device__ __forceinline__ void store(int64_t r, RowKind kind, Stat v, float xt) const {
    double lp = 0.0;
    if (kind == kRowUsed) {
      lp = log_softmax(v, xt);
      stats[r] = make_float2(v.m, 1.0f / v.s);
    } else {
      if (kind == kRowBad) {  // a kernel cannot raise: poison the row and flag it
        lp = NAN;
        atomicExch(&g_logit_loss_error, kErrBadTarget);
      }
      stats[r] = make_float2(0.0f, 0.0f);
    }
    if (logps32) logps32[r] = (float)lp;
    if (logps64) logps64[r] = lp;
  }
};

// Row statistics: one CTA per (row, split). One split writes the row's results; several write
// their Stat to `part` [rows, splits], which finish_kernel merges.
template <typename T>
__global__ void __launch_bounds__(kThreads)
stats_kernel(const T* __restrict__ logits, RowGrid lg, Targets tg, int64_t rows, int64_t vocab,
             int splits, Stat* __restrict__ part, RowOut out) {
  constexpr int V = Vec16<T>::N;
  __shared__ Stat red[kThreads / 32];
  const int64_t items = rows * splits;
  for (int64_t it = blockIdx.x; it < items; it += gridDim.x) {
    const int64_t r = splits == 1 ? it : it / splits;
    const int k = (int)(it - r * splits);
    const int64_t t = tg.at(r);
    const RowKind kind = row_kind(t, tg.ignore, vocab);
    if (kind != kRowUsed) {
      if (splits == 1 && threadIdx.x == 0) out.store(r, kind, Stat{0.0f, 1.0f}, 0.0f);
      continue;
    }
    const T* row = logits + lg.offset(r);
    const float xt = splits == 1 && threadIdx.x == 0 ? to_float(row[t]) : 0.0f;
    const int head = head_elems(row, vocab);
    const T* body = row + head;
    const int64_t nvec = (vocab - head) / V;
    const Part p(nvec, k, splits);
    Running acc;
    if (k == 0 && (int)threadIdx.x < head) acc.add1(to_float(row[threadIdx.x]));
    int64_t v = p.v0 + threadIdx.x;
    for (; v + (kUnrollStats - 1) * kThreads < p.v1; v += kUnrollStats * kThreads) {
      uint4 raw[kUnrollStats];
#pragma unroll
      for (int u = 0; u < kUnrollStats; ++u) raw[u] = ld_stream(body + (v + u * kThreads) * V);
#pragma unroll
      for (int u = 0; u < kUnrollStats; ++u) {
        float x[V];
        unpack<T>(raw[u], x);
        acc.template add<V>(x);
      }
    }
    for (; v < p.v1; v += kThreads) {
      float x[V];
      unpack<T>(ld_stream(body + v * V), x);
      acc.template add<V>(x);
    }
    if (k == splits - 1)
      for (int64_t c = head + nvec * V + threadIdx.x; c < vocab; c += kThreads)
        acc.add1(to_float(row[c]));
    const Stat tot = block_merge(acc.stat(), red);
    if (threadIdx.x == 0) {
      if (splits == 1)
        out.store(r, kind, tot, xt);
      else
        part[it] = tot;
    }
    __syncthreads();  // `red` is reused by the next item
  }
}

// Merges the splits of each row, one warp per row in a fixed order.
template <typename T>
__global__ void __launch_bounds__(kThreads)
finish_kernel(const T* __restrict__ logits, RowGrid lg, Targets tg, int64_t rows, int64_t vocab,
              int splits, const Stat* __restrict__ part, RowOut out) {
  const int lane = threadIdx.x & 31;
  constexpr int kWarps = kThreads / 32;
  for (int64_t r = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5); r < rows;
       r += (int64_t)gridDim.x * kWarps) {
    const int64_t t = tg.at(r);
    const RowKind kind = row_kind(t, tg.ignore, vocab);
    Stat v{-INFINITY, 0.0f};
    float xt = 0.0f;
    if (kind == kRowUsed) {
      xt = to_float(logits[lg.offset(r) + t]);
      for (int k = lane; k < splits; k += 32) v = merge(v, part[r * splits + k]);
      v = warp_merge(v);
    }
    if (lane == 0) out.store(r, kind, v, xt);
  }
}

// dx = c (onehot - softmax), one CTA per (row, split); c = coef[row] * grad. Rows are visited
// from the last to the first: the forward read the last ones last, so they are still in L2.
template <typename T>
__global__ void __launch_bounds__(kThreads)
grad_kernel(const T* __restrict__ logits, RowGrid lg, Targets tg, int64_t rows, int64_t vocab,
            int splits, const float2* __restrict__ stats, const float* __restrict__ coef,
            RowGrid cg, const float* __restrict__ grad, T* __restrict__ dlogits, RowGrid dg) {
  constexpr int V = Vec16<T>::N;
  const float scale = grad != nullptr ? *grad : 1.0f;
  const int64_t items = rows * splits;
  for (int64_t it = blockIdx.x; it < items; it += gridDim.x) {
    const int64_t rr = splits == 1 ? it : it / splits;
    const int k = (int)(it - rr * splits);
    const int64_t r = rows - 1 - rr;
    const T* row = logits + lg.offset(r);
    T* drow = dlogits + dg.offset(r);
    const int64_t t = tg.at(r);
    const bool used = row_kind(t, tg.ignore, vocab) == kRowUsed;
    const int head = head_elems(row, vocab);
    const T* body = row + head;
    T* dbody = drow + head;
    const int64_t nvec = (vocab - head) / V;
    const int64_t tail = head + nvec * V;
    const Part p(nvec, k, splits);
    if (!used) {
      const uint4 z = make_uint4(0, 0, 0, 0);
      if (k == 0 && (int)threadIdx.x < head) drow[threadIdx.x] = from_float<T>(0.0f);
      for (int64_t v = p.v0 + threadIdx.x; v < p.v1; v += kThreads) st_stream(dbody + v * V, z);
      if (k == splits - 1)
        for (int64_t c = tail + threadIdx.x; c < vocab; c += kThreads)
          drow[c] = from_float<T>(0.0f);
      continue;
    }
    const float2 st = stats[r];
    const float c = coef[cg.offset(r)] * scale;
    const float a = -c * st.y, nm = -st.x;
    auto one = [&](int64_t col) {
      const float e = fast_exp(to_float(row[col]) + nm);
      drow[col] = from_float<T>(col == t ? fmaf(a, e, c) : a * e);
    };
    const float2 L = splat2(kLog2e), nm2 = splat2(nm), a2 = splat2(a);
    auto vec = [&](const uint4& raw, int64_t v) {
      float x[V];
      unpack<T>(raw, x);
#pragma unroll
      for (int e = 0; e < V; e += 2) {
        const float2 y = __fmul2_rn(__fadd2_rn(make_float2(x[e], x[e + 1]), nm2), L);
        x[e] = fast_exp2(y.x);
        x[e + 1] = fast_exp2(y.y);
      }
#pragma unroll
      for (int e = 0; e < V; e += 2) {
        const float2 y = __fmul2_rn(make_float2(x[e], x[e + 1]), a2);
        x[e] = y.x;
        x[e + 1] = y.y;
      }
      st_stream(dbody + v * V, pack<T>(x));
      // The thread that stored the target's vector stores the target's element over it.
      if ((uint64_t)(t - (head + v * V)) < (uint64_t)V) one(t);
    };
    if (k == 0 && (int)threadIdx.x < head) one(threadIdx.x);
    int64_t v = p.v0 + threadIdx.x;
    for (; v + (kUnrollGrad - 1) * kThreads < p.v1; v += kUnrollGrad * kThreads) {
      uint4 raw[kUnrollGrad];
#pragma unroll
      for (int u = 0; u < kUnrollGrad; ++u) raw[u] = ld_stream(body + (v + u * kThreads) * V);
#pragma unroll
      for (int u = 0; u < kUnrollGrad; ++u) vec(raw[u], v + u * kThreads);
    }
    for (; v < p.v1; v += kThreads) vec(ld_stream(body + v * V), v);
    if (k == splits - 1)
      for (int64_t col = tail + threadIdx.x; col < vocab; col += kThreads) one(col);
  }
}

// ------------------------------------------------------------------- preference loss --

__device__ __forceinline__ double block_sum(double v, double* red) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  v = warp_sum(v);
  if (lane == 0) red[warp] = v;
  __syncthreads();
  if (warp == 0) v = warp_sum(lane < nw ? red[lane] : 0.0);
  __syncthreads();
  return v;  // valid in warp 0
}

// ratio[q] = sum over the positions of sequence q with a target of (logp - reference), in 64
// bits: the sum of differences, not a difference of long sums. One CTA per sequence.
__global__ void __launch_bounds__(256)
pair_ratio_kernel(const double* __restrict__ logps, const float* __restrict__ ref, RowGrid rg,
                  Targets tg, double* __restrict__ ratio) {
  __shared__ double red[8];
  const int64_t q = blockIdx.x, inner = tg.g.inner;
  double s = 0.0;
  for (int64_t i = threadIdx.x; i < inner; i += 256) {
    const int64_t r = q * inner + i;
    if (tg.at(r) != tg.ignore) s += logps[r] - (double)ref[rg.offset(r)];
  }
  s = block_sum(s, red);
  if (threadIdx.x == 0) ratio[q] = s;
}

// z = beta (ratio_chosen - ratio_rejected); loss = mean((1 - e) softplus(-z) + e softplus(z))
// = mean(softplus(-z) + e z); d loss / d logp is +-beta (e - sigmoid(-z)) / pairs. One CTA,
// pairs in a fixed order. No pairs give NaN (a mean over nothing).
__global__ void __launch_bounds__(kSumThreads)
pair_loss_kernel(const double* __restrict__ ratio, int64_t pairs, double beta, double smoothing,
                 float* __restrict__ loss, float* __restrict__ rewards,
                 float* __restrict__ coef) {
  __shared__ double red[kSumThreads / 32];
  double s = 0.0;
  for (int64_t i = threadIdx.x; i < pairs; i += kSumThreads) {
    const double a = ratio[i], b = ratio[pairs + i];
    const double z = beta * (a - b);
    const double e = exp(-fabs(z));
    s += fmax(-z, 0.0) + log1p(e) + smoothing * z;
    const double sig = z >= 0.0 ? e / (1.0 + e) : 1.0 / (1.0 + e);  // sigmoid(-z)
    const double c = beta * (smoothing - sig) / (double)pairs;
    rewards[i] = (float)(beta * a);
    rewards[pairs + i] = (float)(beta * b);
    coef[i] = (float)c;
    coef[pairs + i] = (float)-c;
  }
  s = block_sum(s, red);
  if (threadIdx.x == 0) *loss = pairs > 0 ? (float)(s / (double)pairs) : NAN;
}

// ----------------------------------------------------------------------- policy loss --

// weight[q]: what each position with a target in sequence q weighs in the mean. Over tokens it
// is 1 / (positions with a target); over sequences 1 / (such positions of q * sequences that
// have any). One CTA of 32 warps.
__global__ void __launch_bounds__(kSumThreads)
policy_weight_kernel(Targets tg, int64_t outer, int by_sequence, double* __restrict__ weight) {
  __shared__ double red[kSumThreads / 32];
  __shared__ double total;
  const int64_t inner = tg.g.inner;
  if (by_sequence) {
    const int lane = threadIdx.x & 31;
    double some = 0.0;
    for (int64_t q = threadIdx.x >> 5; q < outer; q += kSumThreads / 32) {
      double n = 0.0;
      for (int64_t i = lane; i < inner; i += 32) n += tg.at(q * inner + i) != tg.ignore;
      n = warp_sum(n);
      if (lane == 0) {
        weight[q] = n;
        some += n > 0.0;
      }
    }
    some = block_sum(some, red);
    if (threadIdx.x == 0) total = some;
    __syncthreads();  // makes weight[] visible to the whole CTA as well
    for (int64_t q = threadIdx.x; q < outer; q += kSumThreads)
      weight[q] = weight[q] > 0.0 ? 1.0 / (weight[q] * total) : 0.0;
  } else {
    double n = 0.0;
    for (int64_t r = threadIdx.x; r < outer * inner; r += kSumThreads)
      n += tg.at(r) != tg.ignore;
    n = block_sum(n, red);
    if (threadIdx.x == 0) total = n;
    __syncthreads();
    for (int64_t q = threadIdx.x; q < outer; q += kSumThreads)
      weight[q] = total > 0.0 ? 1.0 / total : 0.0;
  }
}

struct PolicyTerms {
  const float* old;
  RowGrid og;
  const float* adv;
  RowGrid ag;
  const float* ref;  // null without a KL term
  RowGrid rg;
  const double* weight;  // [outer]
  float low, high;       // 1 - clip_low, 1 + clip_high
  float kl;
  double* term;     // [rows] weighted loss terms
  float* coef;      // [rows] d loss / d logp
};

// max(-A r, -A clip(r)) + kl (e^g - g - 1) with r = e^(lp - old), g = ref - lp, and its
// derivative to lp; -A r where the unclipped term is the larger one.
__device__ __forceinline__ void policy_term(const PolicyTerms& p, int64_t r, double lp, double w,
                                            double& term, double& coef) {
  const double a = (double)p.adv[p.ag.offset(r)];
  const double ratio = exp(lp - (double)p.old[p.og.offset(r)]);
  const double lo = (double)p.low, hi = (double)p.high;
  const bool inside = a > 0.0 ? ratio <= hi : ratio >= lo;
  const double clipped = fmin(fmax(ratio, lo), hi);
  term = fmax(-a * ratio, -a * clipped);
  coef = inside ? -a * ratio : 0.0;
  if (p.ref != nullptr) {
    const double g = (double)p.ref[p.rg.offset(r)] - lp;
    const double eg = expm1(g);
    term += (double)p.kl * (eg - g);
    coef -= (double)p.kl * eg;
  }
  term *= w;
  coef *= w;
}

// Loss terms and coefficients of every row from the log-probabilities, one thread per row.
__global__ void __launch_bounds__(kThreads)
policy_row_kernel(const double* __restrict__ logps, Targets tg, int64_t rows, PolicyTerms p) {
  for (int64_t r = (int64_t)blockIdx.x * kThreads + threadIdx.x; r < rows;
       r += (int64_t)gridDim.x * kThreads) {
    double term = 0.0, coef = 0.0;
    if (tg.at(r) != tg.ignore)
      policy_term(p, r, logps[r], p.weight[r / tg.g.inner], term, coef);
    p.term[r] = term;
    p.coef[r] = (float)coef;
  }
}

// loss = sum of the weighted terms in a fixed order; NaN when no position has a target.
__global__ void __launch_bounds__(kSumThreads)
policy_sum_kernel(const double* __restrict__ term, int64_t rows, const double* __restrict__ weight,
                  int64_t outer, float* __restrict__ loss) {
  __shared__ double red[kSumThreads / 32];
  double s = 0.0, w = 0.0;
  for (int64_t r = threadIdx.x; r < rows; r += kSumThreads) s += term[r];
  for (int64_t q = threadIdx.x; q < outer; q += kSumThreads) w += weight[q];
  s = block_sum(s, red);
  w = block_sum(w, red);
  if (threadIdx.x == 0) *loss = w > 0.0 ? (float)s : NAN;
}

// ------------------------------------------------------------------------- host side --

struct Rows {  // the checked geometry of a call
  int64_t rows, vocab, outer, inner;
  int splits, sms;
  RowGrid lg;
  Targets tg;
};

// Splits of each row: one CTA a row when the rows alone fill the GPU, else so many that about
// eight CTAs per SM share the work, each with at least one unrolled trip of 16-byte vectors.
int split_count(int64_t rows, int64_t vocab, int elem, int sms) {
  const int64_t trips = vocab * elem / 16 / (kThreads * kUnrollStats);
  const int64_t want = rows > 0 ? ((int64_t)sms * 8 + rows - 1) / rows : 1;
  return (int)std::max<int64_t>(1, std::min(want, trips));
}

int64_t workspace_bytes(int64_t rows, int64_t outer, int splits) {
  // Per row: one Stat per split (when there are several), a log-probability and a loss term;
  // per sequence: a sum or a weight.
  return 8 * ((splits > 1 ? rows * splits : 0) + 2 * rows + outer);
}

int check_sizes(int64_t vocab, int64_t outer, int64_t inner, int64_t* rows) {
  if (outer < 0 || inner < 0 || __builtin_mul_overflow(outer, inner, rows) ||
      *rows > (int64_t(1) << 40))
    return set_error(PT_ERR_SHAPE, "outer and inner must be >= 0 and their product below 2^40");
  if (vocab < 1 || vocab > (int64_t(1) << 31))
    return set_error(PT_ERR_SHAPE, "vocab must be in [1, 2^31] (got %lld)", (long long)vocab);
  return PT_OK;
}

int check_rows(Rows& g, const void* logits, int64_t vocab, int64_t outer, int64_t inner,
               int64_t lo, int64_t li, const int64_t* targets, int64_t to, int64_t ti,
               int64_t ignore, int dtype) {
  if (int st = check_sizes(vocab, outer, inner, &g.rows)) return st;
  const int elem = dtype_size(dtype);
  if (elem == 0) return set_error(PT_ERR_UNSUPPORTED_DTYPE, "unsupported dtype %d", dtype);
  if (int st = current_device_info(nullptr, &g.sms)) return st;
  if (g.rows > 0) {
    if (int st = check_device_ptr(logits, "logits")) return st;
    if (int st = check_device_ptr(targets, "targets")) return st;
    if (reinterpret_cast<uintptr_t>(logits) % elem)
      return set_error(PT_ERR_INVALID_ARGUMENT, "logits are not aligned to their element size");
  }
  g.vocab = vocab;
  g.outer = outer;
  g.inner = inner > 0 ? inner : 1;
  g.splits = split_count(g.rows, vocab, elem, g.sms);
  g.lg = RowGrid{g.inner, lo, li};
  g.tg = Targets{targets, RowGrid{g.inner, to, ti}, ignore};
  return PT_OK;
}

int check_optional(const void* p, const char* name, int64_t rows) {
  return rows > 0 ? check_device_ptr(p, name) : PT_OK;
}

struct Workspace {
  double* logps;
  double* term;
  double* seq;
  Stat* part;
};

int take_workspace(Workspace& w, const Rows& g, void* workspace, int64_t bytes) {
  const int64_t need = workspace_bytes(g.rows, g.outer, g.splits);
  if (bytes < need)
    return set_error(PT_ERR_INVALID_ARGUMENT, "workspace of %lld bytes; %lld are needed",
                     (long long)bytes, (long long)need);
  if (need > 0) {
    if (int st = check_device_ptr(workspace, "workspace")) return st;
    if (reinterpret_cast<uintptr_t>(workspace) % 16)
      return set_error(PT_ERR_INVALID_ARGUMENT, "workspace must be 16-byte aligned");
  }
  w.logps = static_cast<double*>(workspace);
  w.term = w.logps + g.rows;
  w.seq = w.term + g.rows;
  w.part = reinterpret_cast<Stat*>(w.seq + g.outer);
  return PT_OK;
}

int grid_of(int64_t items, int sms, int per_sm) {
  return (int)std::max<int64_t>(1, std::min<int64_t>(items, (int64_t)sms * per_sm));
}

template <typename T>
void launch_stats(const Rows& g, const void* logits, Stat* part, const RowOut& out,
                  cudaStream_t s) {
  const T* x = static_cast<const T*>(logits);
  stats_kernel<T><<<grid_of(g.rows * g.splits, g.sms, 2048 / kThreads), kThreads, 0, s>>>(
      x, g.lg, g.tg, g.rows, g.vocab, g.splits, part, out);
  if (g.splits > 1)
    finish_kernel<T><<<grid_of((g.rows + 3) / 4, g.sms, 2048 / kThreads), kThreads, 0, s>>>(
        x, g.lg, g.tg, g.rows, g.vocab, g.splits, part, out);
}

void row_stats(const Rows& g, const void* logits, int dtype, Stat* part, const RowOut& out,
               cudaStream_t s) {
  if (g.rows == 0) return;
  switch (dtype) {
    case PT_FLOAT32: return launch_stats<float>(g, logits, part, out, s);
    case PT_FLOAT16: return launch_stats<__half>(g, logits, part, out, s);
    default: return launch_stats<__nv_bfloat16>(g, logits, part, out, s);
  }
}

}  // namespace

// Reads and clears this file's device error word (called by pt_take_device_error).
int take_logit_loss_device_error(int* code);
int take_logit_loss_device_error(int* code) {
  int v = 0;
  const int zero = 0;
  if (cudaMemcpyFromSymbol(&v, g_logit_loss_error, sizeof(int)) != cudaSuccess ||
      (v != 0 && cudaMemcpyToSymbol(g_logit_loss_error, &zero, sizeof(int)) != cudaSuccess)) {
    cudaGetLastError();
    return set_error(PT_ERR_CUDA, "cannot read the device error word");
  }
  *code = v;
  return PT_OK;
}

}  // namespace pt

using namespace pt;

extern "C" {

int pt_logit_loss_workspace(int64_t vocab, int64_t outer, int64_t inner, int dtype,
                            int64_t* bytes) {
  if (bytes == nullptr) return set_error(PT_ERR_INVALID_ARGUMENT, "bytes is NULL");
  int64_t rows = 0;
  if (int st = check_sizes(vocab, outer, inner, &rows)) return st;
  const int elem = dtype_size(dtype);
  if (elem == 0) return set_error(PT_ERR_UNSUPPORTED_DTYPE, "unsupported dtype %d", dtype);
  int sms = 0;
  if (int st = current_device_info(nullptr, &sms)) return st;
  *bytes = workspace_bytes(rows, outer, split_count(rows, vocab, elem, sms));
  return ok();
}

int pt_token_logps_fwd(const void* logits, int64_t vocab, int64_t outer, int64_t inner,
                       int64_t logits_outer_stride, int64_t logits_inner_stride,
                       const int64_t* targets, int64_t targets_outer_stride,
                       int64_t targets_inner_stride, int64_t ignore_index, float* logps,
                       float* stats, void* workspace, int64_t workspace_size, int dtype,
                       void* stream) {
  Rows g;
  if (int st = check_rows(g, logits, vocab, outer, inner, logits_outer_stride,
                          logits_inner_stride, targets, targets_outer_stride,
                          targets_inner_stride, ignore_index, dtype))
    return st;
  if (int st = check_optional(logps, "logps", g.rows)) return st;
  if (int st = check_optional(stats, "stats", g.rows)) return st;
  Workspace w;
  if (int st = take_workspace(w, g, workspace, workspace_size)) return st;
  row_stats(g, logits, dtype, w.part, RowOut{reinterpret_cast<float2*>(stats), logps, nullptr},
            as_stream(stream));
  return check_launch("pt_token_logps_fwd");
}

int pt_token_logps_bwd(const void* logits, int64_t vocab, int64_t outer, int64_t inner,
                       int64_t logits_outer_stride, int64_t logits_inner_stride,
                       const int64_t* targets, int64_t targets_outer_stride,
                       int64_t targets_inner_stride, int64_t ignore_index, const float* stats,
                       const float* coef, int64_t coef_outer_stride, int64_t coef_inner_stride,
                       const float* grad, void* dlogits, int64_t dlogits_outer_stride,
                       int64_t dlogits_inner_stride, int dtype, void* stream) {
  Rows g;
  if (int st = check_rows(g, logits, vocab, outer, inner, logits_outer_stride,
                          logits_inner_stride, targets, targets_outer_stride,
                          targets_inner_stride, ignore_index, dtype))
    return st;
  if (g.rows == 0) return ok();
  if (int st = check_device_ptr(stats, "stats")) return st;
  if (int st = check_device_ptr(coef, "coef")) return st;
  if (int st = check_device_ptr(dlogits, "dlogits")) return st;
  if (grad)
    if (int st = check_device_ptr(grad, "grad")) return st;
  const int elem = dtype_size(dtype);
  const bool same = (reinterpret_cast<uintptr_t>(logits) - reinterpret_cast<uintptr_t>(dlogits)) %
                            16 == 0 &&
                    (outer < 2 || (logits_outer_stride - dlogits_outer_stride) * elem % 16 == 0) &&
                    (inner < 2 || (logits_inner_stride - dlogits_inner_stride) * elem % 16 == 0);
  if (!same)
    return set_error(PT_ERR_SHAPE, "rows of logits and dlogits must have the same address modulo "
                                   "16 bytes");
  const RowGrid cg{g.inner, coef_outer_stride, coef_inner_stride};
  const RowGrid dg{g.inner, dlogits_outer_stride, dlogits_inner_stride};
  const float2* st2 = reinterpret_cast<const float2*>(stats);
  const int grid = grid_of(g.rows * g.splits, g.sms, 2048 / kThreads);
  cudaStream_t s = as_stream(stream);
  switch (dtype) {
    case PT_FLOAT32:
      grad_kernel<float><<<grid, kThreads, 0, s>>>(static_cast<const float*>(logits), g.lg, g.tg,
                                                   g.rows, vocab, g.splits, st2, coef, cg, grad,
                                                   static_cast<float*>(dlogits), dg);
      break;
    case PT_FLOAT16:
      grad_kernel<__half><<<grid, kThreads, 0, s>>>(static_cast<const __half*>(logits), g.lg,
                                                    g.tg, g.rows, vocab, g.splits, st2, coef, cg,
                                                    grad, static_cast<__half*>(dlogits), dg);
      break;
    default:
      grad_kernel<__nv_bfloat16><<<grid, kThreads, 0, s>>>(
          static_cast<const __nv_bfloat16*>(logits), g.lg, g.tg, g.rows, vocab, g.splits, st2,
          coef, cg, grad, static_cast<__nv_bfloat16*>(dlogits), dg);
  }
  return check_launch("pt_token_logps_bwd");
}

int pt_preference_loss_fwd(const void* logits, int64_t vocab, int64_t outer, int64_t inner,
                           int64_t logits_outer_stride, int64_t logits_inner_stride,
                           const int64_t* targets, int64_t targets_outer_stride,
                           int64_t targets_inner_stride, int64_t ignore_index,
                           const float* reference, int64_t reference_outer_stride,
                           int64_t reference_inner_stride, double beta, double label_smoothing,
                           float* loss, float* rewards, float* stats, float* coef,
                           void* workspace, int64_t workspace_size, int dtype, void* stream) {
  Rows g;
  if (outer % 2 != 0)
    return set_error(PT_ERR_SHAPE, "chosen and rejected sequences come in pairs (outer is %lld)",
                     (long long)outer);
  if (!std::isfinite(beta) || !(label_smoothing >= 0.0 && label_smoothing <= 1.0))
    return set_error(PT_ERR_INVALID_ARGUMENT,
                     "beta must be finite and label_smoothing in [0, 1]");
  if (int st = check_rows(g, logits, vocab, outer, inner, logits_outer_stride,
                          logits_inner_stride, targets, targets_outer_stride,
                          targets_inner_stride, ignore_index, dtype))
    return st;
  if (int st = check_device_ptr(loss, "loss")) return st;
  if (int st = check_optional(reference, "reference", g.rows)) return st;
  if (int st = check_optional(stats, "stats", g.rows)) return st;
  if (int st = check_optional(rewards, "rewards", outer)) return st;
  if (int st = check_optional(coef, "coef", outer)) return st;
  if (outer > INT32_MAX) return set_error(PT_ERR_SHAPE, "too many sequences");
  Workspace w;
  if (int st = take_workspace(w, g, workspace, workspace_size)) return st;
  cudaStream_t s = as_stream(stream);
  row_stats(g, logits, dtype, w.part, RowOut{reinterpret_cast<float2*>(stats), nullptr, w.logps},
            s);
  if (outer > 0) {
    Targets tg = g.tg;
    tg.g.inner = inner;  // zero positions sum to zero
    pair_ratio_kernel<<<(unsigned)outer, 256, 0, s>>>(
        w.logps, reference, RowGrid{g.inner, reference_outer_stride, reference_inner_stride}, tg,
        w.seq);
  }
  pair_loss_kernel<<<1, kSumThreads, 0, s>>>(w.seq, outer / 2, beta, label_smoothing, loss,
                                             rewards, coef);
  return check_launch("pt_preference_loss_fwd");
}

int pt_policy_loss_fwd(const void* logits, int64_t vocab, int64_t outer, int64_t inner,
                       int64_t logits_outer_stride, int64_t logits_inner_stride,
                       const int64_t* targets, int64_t targets_outer_stride,
                       int64_t targets_inner_stride, int64_t ignore_index,
                       const float* old_logps, int64_t old_outer_stride, int64_t old_inner_stride,
                       const float* advantages, int64_t advantages_outer_stride,
                       int64_t advantages_inner_stride, const float* reference,
                       int64_t reference_outer_stride, int64_t reference_inner_stride,
                       double clip_low, double clip_high, double kl_coef, int by_sequence,
                       float* loss, float* logps, float* stats, float* coef, void* workspace,
                       int64_t workspace_size, int dtype, void* stream) {
  Rows g;
  if (!(clip_low >= 0.0) || !(clip_high >= 0.0) || !std::isfinite(kl_coef))
    return set_error(PT_ERR_INVALID_ARGUMENT,
                     "clip_low and clip_high must be >= 0 and kl_coef finite");
  if (int st = check_rows(g, logits, vocab, outer, inner, logits_outer_stride,
                          logits_inner_stride, targets, targets_outer_stride,
                          targets_inner_stride, ignore_index, dtype))
    return st;
  if (int st = check_device_ptr(loss, "loss")) return st;
  if (int st = check_optional(old_logps, "old_logps", g.rows)) return st;
  if (int st = check_optional(advantages, "advantages", g.rows)) return st;
  if (reference)
    if (int st = check_optional(reference, "reference", g.rows)) return st;
  if (int st = check_optional(logps, "logps", g.rows)) return st;
  if (int st = check_optional(stats, "stats", g.rows)) return st;
  if (int st = check_optional(coef, "coef", g.rows)) return st;
  Workspace w;
  if (int st = take_workspace(w, g, workspace, workspace_size)) return st;
  cudaStream_t s = as_stream(stream);
  PolicyTerms p;
  p.old = old_logps;
  p.og = RowGrid{g.inner, old_outer_stride, old_inner_stride};
  p.adv = advantages;
  p.ag = RowGrid{g.inner, advantages_outer_stride, advantages_inner_stride};
  p.ref = reference;
  p.rg = RowGrid{g.inner, reference_outer_stride, reference_inner_stride};
  p.weight = w.seq;
  p.low = (float)(1.0 - clip_low);
  p.high = (float)(1.0 + clip_high);
  p.kl = (float)kl_coef;
  p.term = w.term;
  p.coef = coef;
  row_stats(g, logits, dtype, w.part, RowOut{reinterpret_cast<float2*>(stats), logps, w.logps},
            s);
  const int64_t sequences = g.rows > 0 ? outer : 0;
  policy_weight_kernel<<<1, kSumThreads, 0, s>>>(g.tg, sequences, by_sequence, w.seq);
  if (g.rows > 0)
    policy_row_kernel<<<grid_of((g.rows + kThreads - 1) / kThreads, g.sms, 2048 / kThreads),
                        kThreads, 0, s>>>(w.logps, g.tg, g.rows, p);
  policy_sum_kernel<<<1, kSumThreads, 0, s>>>(w.term, g.rows, w.seq, sequences, loss);
  return check_launch("pt_policy_loss_fwd");
}

}  // extern "C"
