// Post-training losses over vocabulary rows on sm_100a: the log-probability of each row's target
// (forward and backward), the preference loss of chosen / rejected pairs and the clipped policy
// loss with a KL term, each with the gradient of its logits.
//
// For a row x with target t, relative to a reference m a little above max(x):
//   s = sum 2^((x - m) log2 e),  log softmax(x)_t = (x_t - m) - ln s.
// x is taken relative to m before it is scaled, so a row of one type's lowest values (a mask
// that leaves nothing) neither overflows nor loses its s. Losses sum these over thousands of
// positions, where a bias matters more than a rounding: log2 e is applied in two parts, sums are
// rescaled only when a value passes the reference and once more when threads are merged, and
// the mean error of the exponential unit is taken out of ln s. The differences are taken in 64
// bits and the log-probability is rounded once. Every loss here depends on the
// logits through these log-probabilities alone, so its gradient is
//   dx = c (onehot(t) - softmax(x)),  softmax(x) = 2^((x - m) log2 e) / s,
// with one coefficient c per row: the forward keeps (m, 1/s) and c, the backward reads the
// logits once more and writes dx. All passes over the logits are bound by HBM bandwidth.
//
// Rows form an [outer, inner] grid addressed by two strides (sequences x positions). Rows whose
// target is ignore_index are not read at all; their gradient is stored as zeros.

#include <algorithm>
#include <cmath>
#include <cstddef>

#include "common.cuh"

namespace pt {

__device__ int g_logit_loss_error = 0;

namespace {

// Statistics: 128 threads with 8 vectors in flight each, as for the cross-entropy kernels, which
// read the same rows (0.97 of the HBM peak at 8192 x 128256 bf16; 0.89 with 256 threads).
constexpr int kThreads = 128;
constexpr int kUnrollStats = 8;
// Gradient: 256 threads with 4 vectors in flight, four such trips per CTA (537 us there, 0.99 of
// the peak; 550 to 590 us with 128 threads, 557 with more or wider trips).
constexpr int kGradThreads = 256;
constexpr int kUnrollGrad = 4;
constexpr int kGradTrips = 4;
constexpr int kSumThreads = 1024;
constexpr float kLog2e = 1.4426950408889634f;  // log2(e): exp(a) = 2^(a log2(e))
constexpr float kLog2eLow = (float)(1.4426950408889634 - (double)kLog2e);  // what it lacks
// How far ex2.approx is below the true value on average for arguments below 0 (measured over 10^6
// points of [-20, 0] on B200; its largest error there is 1.4e-7). Above 0 it is 3.3e-8 too high,
// so the reference is kept above every value: by kAbove when it is set, which leaves room for
// larger values to come. References are whole numbers, so that most threads of a row have the
// same one and their sums merge without a factor. What that costs: x - m, up to 9 below 0 at the
// row's maximum, is rounded in fp32, by up to 5e-7 there (either way) where fp32 logits next to 0
// are known to more digits.
constexpr float kExpLow = 5.05e-8f;
constexpr float kAbove = 8.0f;
constexpr int kErrBadTarget = 2;

// Row r of the [outer, inner] row grid sits at outer index r / inner, inner index r % inner. One
// division by a multiplication serves all the tensors that are addressed by the row.
struct RowIndex {
  int64_t outer, inner;
};
struct RowDiv {
  FastDiv div;
  __device__ __forceinline__ RowIndex operator()(int64_t r) const {
    const uint32_t o = div.div((uint32_t)r);
    return {o, (uint32_t)r - o * div.d};
  }
};
struct RowGrid {
  int64_t outer_stride, inner_stride;  // elements
  __device__ __forceinline__ int64_t offset(RowIndex i) const {
    return i.outer * outer_stride + i.inner * inner_stride;
  }
};

struct Targets {
  const int64_t* p;
  RowGrid g;
  int64_t ignore;
  RowDiv index;  // of every per-row tensor of the call
  __device__ __forceinline__ int64_t at(RowIndex i) const { return p[g.offset(i)]; }
};

// A set of values x as (reference m, sum of e^(x - m)); m = -inf and s = 0 for the empty set.
struct Stat {
  float m, s;
};

// 2^x on the special-function unit (PTX ex2.approx.ftz).
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float2 log2_scaled(float2 d) {  // d log2(e)
  return __ffma2_rn(d, splat2(kLog2e), __fmul2_rn(d, splat2(kLog2eLow)));
}
__device__ __forceinline__ float fast_exp(float d) {
  return fast_exp2(fmaf(d, kLog2e, d * kLog2eLow));
}
// e^-k, rounded once, for the whole numbers that references differ by.
constexpr int kWholePowers = 32;
struct WholePowers {
  float p[kWholePowers];
  constexpr WholePowers() : p() {
    double v = 1.0;
    for (int k = 0; k < kWholePowers; ++k, v *= 0.36787944117144233) p[k] = (float)v;
  }
};
__constant__ WholePowers c_powers{};
__device__ __noinline__ float exact_exp(float d) { return (float)exp((double)d); }
// e^-d for two references that are d >= 0 apart.
__device__ __forceinline__ float factor_below(float d) {
  if (d < (float)kWholePowers) return c_powers.p[(int)d];
  return exact_exp(-d);
}

// The sum of v relative to the reference m >= v.m. A NaN sum stays NaN (NaN * 0).
__device__ __forceinline__ float sum_at(Stat v, float m) {
  return v.m == m ? v.s : v.s * (v.m == -INFINITY ? 0.0f : factor_below(m - v.m));
}

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, off));
  return v;
}

// Merged over the CTA; valid in all threads of warp 0. `red` holds one Stat per warp.
__device__ __forceinline__ Stat block_merge(Stat v, Stat* red) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  const float wm = warp_max(v.m);
  if (lane == 0) red[warp].m = wm;
  __syncthreads();
  float m = red[0].m;
  for (int w = 1; w < nw; ++w) m = fmaxf(m, red[w].m);
  const float ws = warp_sum(sum_at(v, m));
  if (lane == 0) red[warp].s = ws;
  __syncthreads();
  return {m, warp == 0 ? warp_sum(lane < nw ? red[lane].s : 0.0f) : 0.0f};
}

// Per-thread running statistics: two partial sums (paired fp32 lanes) relative to m.
struct Running {
  float m = -INFINITY;
  float2 s = make_float2(0.0f, 0.0f);
  __device__ __forceinline__ void raise(float xmax) {
    if (xmax > m) {
      const float above = ceilf(xmax) + kAbove;
      s = __fmul2_rn(s, splat2(m == -INFINITY ? 0.0f : factor_below(above - m)));
      m = above;
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
    const float2 nm = splat2(-base());
#pragma unroll
    for (int e = 0; e < N; e += 2) {
      const float2 t = log2_scaled(__fadd2_rn(make_float2(x[e], x[e + 1]), nm));
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
// allows, where m + ln s would absorb ln s. s = 2^k f with f in [2^-1/2, 2^1/2): k ln 2 is exact in
// 64 bits and the fp32 logarithm of f is within 2^-25 (a 64-bit one took longer than a short
// row's pass).
__device__ __forceinline__ double log_softmax(Stat v, float xt) {
  const int bits = __float_as_int(v.s) - 0x3f3504f3;  // of 2^-1/2
  const int k = bits >> 23;
  const float f = __int_as_float((bits & 0x007fffff) + 0x3f3504f3);
  // s - s is 0, or NaN where s is not finite and has no such k and f.
  const double lp = ((double)xt - (double)v.m) -
                    ((double)k * 0.6931471805599453 + (double)kExpLow) -
                    (double)(logf(f) + (v.s - v.s));
  return lp > 0.0 ? 0.0 : lp;  // a near-certain target is within rounding of 0 on either side
}

// Elements before the first 16-byte boundary of a row (0 when it is aligned).
template <typename T> __device__ __forceinline__ int head_elems(const T* p, int64_t vocab) {
  const int mis = (int)(reinterpret_cast<uintptr_t>(p) & 15u);
  const int h = mis ? (16 - mis) / (int)sizeof(T) : 0;
  return (int64_t)h < vocab ? h : (int)vocab;
}

// The part of a row that split `k` of `n` (or of 2^log2_n) takes: whole 16-byte vectors [v0, v1) of the aligned
// body, the unaligned head with the first split and the tail with the last.
struct Part {
  int64_t v0, v1;
  __device__ __forceinline__ Part(int64_t nvec, int k, int n) {
    const int64_t per = (nvec + n - 1) / n;
    v0 = min(nvec, per * k);
    v1 = min(nvec, v0 + per);
  }
  __device__ __forceinline__ Part(int64_t nvec, int k, int log2_n, std::nullptr_t) {
    const int64_t per = (nvec + (1 << log2_n) - 1) >> log2_n;
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
    const RowIndex index = tg.index(r);
    const int64_t t = tg.at(index);
    const RowKind kind = row_kind(t, tg.ignore, vocab);
    if (kind != kRowUsed) {
      if (splits == 1 && threadIdx.x == 0) out.store(r, kind, Stat{0.0f, 1.0f}, 0.0f);
      continue;
    }
    const T* row = logits + lg.offset(index);
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

// Short rows: one warp per row, without the CTA's meetings. The policy loss holds a row in
// registers: kShortVecs 16-byte vectors (8 KB) at most.
constexpr int kShortVecs = 512;
constexpr int kShortWarps = 4;  // rows per CTA

// The element of an unaligned row's head (lanes below 16) or tail (the others) that a lane takes,
// or -1; there are at most 7 of each.
__device__ __forceinline__ int64_t edge_of(int lane, int head, int64_t tail, int64_t vocab) {
  if (lane < head) return lane;
  return lane >= 16 && tail + lane - 16 < vocab ? tail + lane - 16 : -1;
}

template <typename T>
__global__ void __launch_bounds__(kShortWarps * 32)
stats_short_kernel(const T* __restrict__ logits, RowGrid lg, Targets tg, int64_t rows,
                   int64_t vocab, RowOut out) {
  constexpr int V = Vec16<T>::N;
  const int lane = threadIdx.x & 31;
  const int64_t r = (int64_t)blockIdx.x * kShortWarps + (threadIdx.x >> 5);
  if (r >= rows) return;
  const RowIndex index = tg.index(r);
  const int64_t t = tg.at(index);
  const RowKind kind = row_kind(t, tg.ignore, vocab);
  if (kind != kRowUsed) {
    if (lane == 0) out.store(r, kind, Stat{0.0f, 1.0f}, 0.0f);
    return;
  }
  const T* row = logits + lg.offset(index);
  const float xt = to_float(row[t]);
  const int head = head_elems(row, vocab);
  const T* body = row + head;
  const int nvec = (int)((vocab - head) / V);
  const int64_t edge = edge_of(lane, head, head + (int64_t)nvec * V, vocab);
  Running acc;
  if (edge >= 0) acc.add1(to_float(row[edge]));
  for (int v0 = lane; v0 < nvec; v0 += 32 * kUnrollStats) {
    uint4 raw[kUnrollStats];
#pragma unroll
    for (int u = 0; u < kUnrollStats; ++u)
      if (v0 + 32 * u < nvec) raw[u] = ld_stream(body + (v0 + 32 * u) * V);
#pragma unroll
    for (int u = 0; u < kUnrollStats; ++u) {
      if (v0 + 32 * u < nvec) {
        float x[V];
        unpack<T>(raw[u], x);
        acc.template add<V>(x);
      }
    }
  }
  const Stat v = acc.stat();
  const float m = warp_max(v.m);
  const float sum = warp_sum(sum_at(v, m));
  if (lane == 0) out.store(r, kind, Stat{m, sum}, xt);
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
    const RowIndex index = tg.index(r);
    const int64_t t = tg.at(index);
    const RowKind kind = row_kind(t, tg.ignore, vocab);
    Stat v{-INFINITY, 0.0f};
    float xt = 0.0f;
    if (kind == kRowUsed) {
      xt = to_float(logits[lg.offset(index) + t]);
      for (int k = lane; k < splits; k += 32) v.m = fmaxf(v.m, part[r * splits + k].m);
      v.m = warp_max(v.m);
      for (int k = lane; k < splits; k += 32) v.s += sum_at(part[r * splits + k], v.m);
      v.s = warp_sum(v.s);
    }
    if (lane == 0) out.store(r, kind, v, xt);
  }
}

// How dx of one row is formed: dx = a e^(x - m), a = -c / s, and c more at the target. Whole
// vectors take log2 e in one part: what that leaves out, 1.3e-8 |x - m| relative, is a bias of a
// sum but less than an element's own rounding of the product (6e-8 |x - m|).
struct RowGrad {
  float a, c, nm;
  // V elements; the target, if it is among them, without its c.
  template <typename T> __device__ __forceinline__ uint4 vec(const uint4& raw) const {
    constexpr int V = Vec16<T>::N;
    const float2 nm2 = splat2(nm), a2 = splat2(a), L = splat2(kLog2e);
    float x[V];
    unpack<T>(raw, x);
#pragma unroll
    for (int e = 0; e < V; e += 2) {
      const float2 y = __fmul2_rn(__fadd2_rn(make_float2(x[e], x[e + 1]), nm2), L);
      const float2 d = __fmul2_rn(make_float2(fast_exp2(y.x), fast_exp2(y.y)), a2);
      x[e] = d.x;
      x[e + 1] = d.y;
    }
    return pack<T>(x);
  }
  __device__ __forceinline__ float one(float x, bool target) const {
    const float e = fast_exp(x + nm);
    return target ? fmaf(a, e, c) : a * e;
  }
};

// dx = c (onehot - softmax) of short rows, one warp per row.
template <typename T>
__global__ void __launch_bounds__(kShortWarps * 32)
grad_short_kernel(const T* __restrict__ logits, RowGrid lg, Targets tg, int64_t rows,
                  int64_t vocab, const float2* __restrict__ stats,
                  const float* __restrict__ coef, RowGrid cg, const float* __restrict__ grad,
                  T* __restrict__ dlogits, RowGrid dg) {
  constexpr int V = Vec16<T>::N;
  const int lane = threadIdx.x & 31;
  const int64_t r = (int64_t)blockIdx.x * kShortWarps + (threadIdx.x >> 5);
  if (r >= rows) return;
  const RowIndex index = tg.index(r);
  const int64_t t = tg.at(index);
  const bool used = row_kind(t, tg.ignore, vocab) == kRowUsed;
  const T* row = logits + lg.offset(index);
  T* drow = dlogits + dg.offset(index);
  const int head = head_elems(row, vocab);
  const int nvec = (int)((vocab - head) / V);
  const int64_t edge = edge_of(lane, head, head + (int64_t)nvec * V, vocab);
  const T* body = row + head;
  T* dbody = drow + head;
  if (!used) {
    if (edge >= 0) drow[edge] = from_float<T>(0.0f);
    for (int v = lane; v < nvec; v += 32) st_stream(dbody + v * V, make_uint4(0, 0, 0, 0));
    return;
  }
  const float2 st = stats[r];
  RowGrad f;
  f.c = coef[cg.offset(index)] * (grad != nullptr ? *grad : 1.0f);
  f.a = -f.c * st.y;
  f.nm = -st.x;
  if (edge >= 0) drow[edge] = from_float<T>(f.one(to_float(row[edge]), edge == t));
  const int tv = t >= head && t < head + (int64_t)nvec * V ? (int)((t - head) / V) : -1;
  for (int v0 = lane; v0 < nvec; v0 += 32 * kUnrollGrad) {
    uint4 raw[kUnrollGrad];
#pragma unroll
    for (int u = 0; u < kUnrollGrad; ++u)
      if (v0 + 32 * u < nvec) raw[u] = ld_stream(body + (v0 + 32 * u) * V);
#pragma unroll
    for (int u = 0; u < kUnrollGrad; ++u) {
      const int v = v0 + 32 * u;
      if (v < nvec) {
        st_stream(dbody + v * V, f.vec<T>(raw[u]));
        if (v == tv) drow[t] = from_float<T>(f.one(to_float(row[t]), true));
      }
    }
  }
}

// dx = c (onehot - softmax), one CTA per (row, split); c = coef[row] * grad. A split is kGradTrips
// unrolled trips: rows without a target cost a fraction of the others, so CTAs have to be short
// and handed out as they finish (one row per CTA in a fixed assignment took 1.45 times as long
// at 8192 x 128256 bf16 with a third of the rows ignored). Rows are visited from the last to
// the first: the forward read the last ones last, so they are still in L2.
template <typename T>
__global__ void __launch_bounds__(kGradThreads)
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
    const RowIndex index = tg.index(r);
    const int64_t t = tg.at(index);
    const T* row = logits + lg.offset(index);
    T* drow = dlogits + dg.offset(index);
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
      for (int64_t v = p.v0 + threadIdx.x; v < p.v1; v += kGradThreads) st_stream(dbody + v * V, z);
      if (k == splits - 1)
        for (int64_t c = tail + threadIdx.x; c < vocab; c += kGradThreads)
          drow[c] = from_float<T>(0.0f);
      continue;
    }
    const float2 st = stats[r];
    RowGrad f;
    f.c = coef[cg.offset(index)] * scale;
    f.a = -f.c * st.y;
    f.nm = -st.x;
    auto one = [&](int64_t col) {
      drow[col] = from_float<T>(f.one(to_float(row[col]), col == t));
    };
    auto vec = [&](const uint4& raw, int64_t v) {
      st_stream(dbody + v * V, f.vec<T>(raw));
      // The thread that stored the target's vector stores the target's element over it.
      if ((uint64_t)(t - (head + v * V)) < (uint64_t)V) one(t);
    };
    if (k == 0 && (int)threadIdx.x < head) one(threadIdx.x);
    int64_t v = p.v0 + threadIdx.x;
    for (; v + (kUnrollGrad - 1) * kGradThreads < p.v1; v += kUnrollGrad * kGradThreads) {
      uint4 raw[kUnrollGrad];
#pragma unroll
      for (int u = 0; u < kUnrollGrad; ++u) raw[u] = ld_stream(body + (v + u * kGradThreads) * V);
#pragma unroll
      for (int u = 0; u < kUnrollGrad; ++u) vec(raw[u], v + u * kGradThreads);
    }
    for (; v < p.v1; v += kGradThreads) vec(ld_stream(body + v * V), v);
    if (k == splits - 1)
      for (int64_t col = tail + threadIdx.x; col < vocab; col += kGradThreads) one(col);
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
                  Targets tg, int64_t inner, double* __restrict__ ratio) {
  __shared__ double red[8];
  const int64_t q = blockIdx.x;
  double s = 0.0;
#pragma unroll 2
  for (int64_t i = threadIdx.x; i < inner; i += 256) {
    const RowIndex at{q, i};
    if (tg.at(at) != tg.ignore) s += logps[q * inner + i] - (double)ref[rg.offset(at)];
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
// have any). One CTA counts and writes the weights of a mean over tokens; where there are many
// tokens or sequences have weights of their own, one CTA per sequence counts first (4 sequences of
// 16384: 5 us, against 11 us in the one CTA and 29 with a warp of it per sequence).
constexpr int64_t kCountAtOnce = 16384;

__global__ void __launch_bounds__(kSumThreads)
count_kernel(Targets tg, int64_t inner, double* __restrict__ counts) {
  __shared__ double red[kSumThreads / 32];
  const int64_t q = blockIdx.x;
  double n = 0.0;
#pragma unroll 8
  for (int64_t i = threadIdx.x; i < inner; i += kSumThreads) n += tg.at({q, i}) != tg.ignore;
  n = block_sum(n, red);
  if (threadIdx.x == 0) counts[q] = n;
}

// From counts in weight[], if they are there, else counting all `rows`.
__global__ void __launch_bounds__(kSumThreads)
policy_weight_kernel(Targets tg, int64_t outer, int64_t rows, int counted, int by_sequence,
                     double* __restrict__ weight) {
  __shared__ double red[kSumThreads / 32];
  __shared__ double total;
  double n = 0.0;
  if (counted) {
    for (int64_t q = threadIdx.x; q < outer; q += kSumThreads)
      n += by_sequence ? (double)(weight[q] > 0.0) : weight[q];
  } else {
#pragma unroll 4
    for (int64_t r = threadIdx.x; r < rows; r += kSumThreads)
      n += tg.at(tg.index(r)) != tg.ignore;
  }
  n = block_sum(n, red);
  if (threadIdx.x == 0) total = n;
  __syncthreads();
  for (int64_t q = threadIdx.x; q < outer; q += kSumThreads) {
    const double own = by_sequence ? weight[q] * total : total;
    weight[q] = own > 0.0 ? 1.0 / own : 0.0;
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
  double low, high;      // 1 - clip_low, 1 + clip_high
  double kl;
  double* term;     // [rows] weighted loss terms
  float* coef;      // [rows] d loss / d logp
};

constexpr double kOrdinary = 2.0;
__device__ __noinline__ double far_exp(double x) { return exp(x); }

// What a row's loss term takes besides its log-probability.
struct PolicyRow {
  float old, adv, ref;
  double weight;
  __device__ __forceinline__ void load(const PolicyTerms& p, RowIndex i) {
    old = p.old[p.og.offset(i)];
    adv = p.adv[p.ag.offset(i)];
    ref = p.ref != nullptr ? p.ref[p.rg.offset(i)] : 0.0f;
    weight = p.weight[i.outer];
  }
  // max(-A r, -A clip(r)) + kl (e^g - g - 1) with r = e^(lp - old), g = ref - lp, and its
  // derivative to lp. The clipped term is the larger one where r is above the upper border for a
  // positive A, below the lower one for a negative A: -A times that border, which has no slope;
  // elsewhere it is -A r, its own derivative. That of the KL term is kl (1 - e^g). NaN of any
  // input is kept in both (fmax and fmin would drop it). All is in 64 bits but for the
  // exponentials of up to kOrdinary: expf is within 2^-22 and expm1f within 2^-22 |e^g - 1| there,
  // which is what an error of 2^-22 in the log-probability makes of r and of the KL term. Larger
  // arguments are taken in 64 bits, where e^89 and above are finite, so that a zero advantage
  // weighs nothing.
  __device__ __forceinline__ void term(const PolicyTerms& p, double lp, double& term,
                                       float& coef) const {
    const double d = lp - (double)old, a = (double)adv;
    const double r = fabs(d) <= kOrdinary ? (double)expf((float)d) : far_exp(d);
    const double border = a > 0.0 ? p.high : p.low;
    const bool beyond = a > 0.0 ? r > border : r < border;
    double value = -a * (beyond ? border : r);
    double slope = beyond && value == value ? 0.0 : value;
    if (p.ref != nullptr) {
      const double g = (double)ref - lp;
      const double eg = fabs(g) <= kOrdinary ? (double)expm1f((float)g) : far_exp(g) - 1.0;
      value += p.kl * (eg - g);
      slope -= p.kl * eg;
    }
    term = value * weight;
    coef = (float)(slope * weight);
  }
};

// Loss terms and coefficients of every row from the log-probabilities, one thread per row.
__global__ void __launch_bounds__(kThreads)
policy_row_kernel(const double* __restrict__ logps, Targets tg, int64_t rows, PolicyTerms p) {
  for (int64_t r = (int64_t)blockIdx.x * kThreads + threadIdx.x; r < rows;
       r += (int64_t)gridDim.x * kThreads) {
    double term = 0.0;
    float coef = 0.0f;
    const RowIndex index = tg.index(r);
    if (tg.at(index) != tg.ignore) {
      PolicyRow row;
      row.load(p, index);
      row.term(p, logps[r], term, coef);
    }
    p.term[r] = term;
    p.coef[r] = coef;
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

// One pass for the loss and its gradient (see pt_policy_loss_grad): the coefficient of a row
// depends on that row alone, so a row is read from HBM once, kept in shared memory while its
// statistics form, and turned into dx from there: one read and one write of the logits' size
// where the two-kernel form reads twice.
//
// A cluster of C CTAs takes one row, each a slice of whole 16-byte vectors. Every warp fetches
// its own piece of the slice by one bulk copy, sums it when it has arrived and later turns the
// same piece into dx, so warps meet only to merge their sums. The CTAs exchange theirs by
// asynchronous stores into each other's shared memory, which complete on the receiver's barrier:
// one thread waits for it, not the whole cluster. Several clusters share an SM, so one row's
// loads overlap another's arithmetic and stores.
// 128 threads and slices of up to 32 KB, seven CTAs per SM: 633 us at 8192 x 128256 bf16 with 35 %
// of the rows ignored (680 us with 256 threads and 64 KB, 715 with 64 threads and 16 KB), against
// 753 us for statistics and gradient in two passes.
constexpr int kFusedThreads = 128;
constexpr int kFusedBlocks = 7;
constexpr int kFusedWarps = kFusedThreads / 32;
constexpr int kMaxCluster = 8;  // the portable cluster size
constexpr int kSliceBytes = 32 * 1024;
constexpr int kMaxSliceBytes = 192 * 1024;
constexpr int kErrWait = kDeviceErrWaitTimeout;

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t in_cluster(const void* p, uint32_t rank) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_addr(p)),
               "r"(rank));
  return remote;
}
// Stores v at the place that `p` (in this CTA's shared memory) has in CTA `rank`, counted by the
// barrier that `bar` is there.
__device__ __forceinline__ void store_in_cluster(Stat* p, uint64_t* bar, uint32_t rank, Stat v) {
  asm volatile(
      "st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.b32 [%0], {%1, %2}, [%3];" ::
          "r"(in_cluster(p, rank)),
      "r"(__float_as_uint(v.m)), "r"(__float_as_uint(v.s)), "r"(in_cluster(bar, rank))
      : "memory");
}
// mbar_wait_bounded for data that other CTAs of the cluster have stored.
__device__ __forceinline__ bool cluster_wait_bounded(uint64_t* bar, long long limit) {
  const long long t0 = clock64();
  for (;;) {
    uint32_t done;
    asm volatile(
        "{\n .reg .pred p;\n"
        " mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], 0;\n"
        " selp.u32 %0, 1, 0, p;\n}"
        : "=r"(done)
        : "r"(smem_addr(bar))
        : "memory");
    if (done) return true;
    if (clock64() - t0 > limit) return false;
  }
}

// A wait that gives up (after wait_limit cycles; at once if that is negative) sets the error word
// and makes the row NaN through its sum, whatever the slice then holds. What it waited for gets
// the full time once more: it must not reach shared memory that another CTA has by then.
template <typename T>
__global__ void __launch_bounds__(kFusedThreads, kFusedBlocks)
policy_grad_kernel(const T* __restrict__ logits, RowGrid lg, Targets tg, int64_t vocab,
                   int log2_cluster, PolicyTerms p, float grad, long long wait_limit, RowOut out,
                   T* __restrict__ dlogits, RowGrid dg) {
  constexpr int V = Vec16<T>::N;
  const int cluster = 1 << log2_cluster;
  extern __shared__ __align__(16) unsigned char slice[];
  __shared__ uint64_t bar[kFusedWarps];
  __shared__ uint64_t peer_bar;
  __shared__ Stat red[kFusedWarps];
  __shared__ Stat peer[kMaxCluster];
  __shared__ float3 shared_row;  // reference, 1 / s, coefficient
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = cluster > 1 ? (int)cluster_rank() : 0;
  const int64_t r = blockIdx.x >> log2_cluster;
  const RowIndex index = tg.index(r);
  const int64_t t = tg.at(index);
  const T* row = logits + lg.offset(index);
  T* drow = dlogits + dg.offset(index);
  const RowKind kind = row_kind(t, tg.ignore, vocab);
  const int head = head_elems(row, vocab);
  const int64_t nvec = (vocab - head) / V;
  const int64_t tail = head + nvec * V;
  const Part part(nvec, rank, log2_cluster, nullptr);
  const int n = (int)(part.v1 - part.v0);
  const T* body = row + head + part.v0 * V;
  T* dbody = drow + head + part.v0 * V;
  // This thread's element of the unaligned head or tail, or -1.
  int64_t edge = -1;
  if (rank == 0 && tid < head) edge = tid;
  if (rank == cluster - 1 && tid >= 32 && tail + tid - 32 < vocab) edge = tail + tid - 32;

  if (kind != kRowUsed) {  // the same for every CTA of the cluster: none waits for another
    const uint4 z = make_uint4(0, 0, 0, 0);
    for (int v = tid; v < n; v += kFusedThreads) st_stream(dbody + (int64_t)v * V, z);
    if (edge >= 0) drow[edge] = from_float<T>(0.0f);
    if (rank == 0 && tid == 0) {
      out.store(r, kind, Stat{0.0f, 1.0f}, 0.0f);
      p.term[r] = kind == kRowIgnored ? 0.0 : NAN;
      p.coef[r] = 0.0f;
    }
    return;
  }

  const int per_warp = (n + kFusedWarps - 1) / kFusedWarps;
  const int w0 = min(n, warp * per_warp), w1 = min(n, w0 + per_warp);
  if (lane == 0 && w1 > w0) {
    mbar_init(&bar[warp], 1);
    fence_mbar_init();
    mbar_arrive_expect_tx(&bar[warp], (uint32_t)(w1 - w0) * 16u);
    bulk_load(slice + (size_t)w0 * 16, body + (int64_t)w0 * V, (uint32_t)(w1 - w0) * 16u,
              &bar[warp]);
  }
  if (cluster > 1) {
    if (tid == 0) {
      mbar_init(&peer_bar, 1);
      fence_mbar_init();
      mbar_arrive_expect_tx(&peer_bar, (uint32_t)(cluster * sizeof(Stat)));
    }
    // Says that this CTA runs and its barrier is set (which the fence above has published). All
    // threads arrive here and wait below, each warp as one: the barrier counts warps.
    __syncwarp();
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  }
  float xt = 0.0f;
  PolicyRow terms;
  if (tid == 0) {
    xt = to_float(row[t]);
    terms.load(p, index);
  }
  const float xe = edge >= 0 ? to_float(row[edge]) : 0.0f;
  Running acc;
  if (edge >= 0) acc.add1(xe);
  __syncwarp();
  int v = w0 + lane;
  if (w1 > w0 && (wait_limit < 0 || !mbar_wait_bounded(&bar[warp], 0, wait_limit))) {
    if (lane == 0) atomicExch(&g_logit_loss_error, kErrWait);
    mbar_wait_bounded(&bar[warp], 0);
    acc.s.x = NAN;
    v = w1;  // nothing is summed
  }
  // Two vectors a trip: their loads and exponentials overlap.
  for (; v + 32 < w1; v += 64) {
    float x[2 * V];
    unpack<T>(lds128(slice + (size_t)v * 16), x);
    unpack<T>(lds128(slice + (size_t)(v + 32) * 16), x + V);
    acc.template add<2 * V>(x);
  }
  if (v < w1) {
    float x[V];
    unpack<T>(lds128(slice + (size_t)v * 16), x);
    acc.template add<V>(x);
  }
  if (cluster > 1) {
    __syncwarp();
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
  Stat total = block_merge(acc.stat(), red);
  if (cluster > 1 && tid < cluster) store_in_cluster(&peer[rank], &peer_bar, tid, total);
  if (tid == 0) {
    if (cluster > 1) {
      // All CTAs' stores have arrived after this: none reaches into a CTA that has ended.
      total = Stat{-INFINITY, 0.0f};
      if (wait_limit < 0 || !cluster_wait_bounded(&peer_bar, wait_limit)) {
        atomicExch(&g_logit_loss_error, kErrWait);
        cluster_wait_bounded(&peer_bar, kWaitLimitCycles);
        total.s = NAN;
      }
      for (int c = 0; c < cluster; ++c) total.m = fmaxf(total.m, peer[c].m);
      for (int c = 0; c < cluster; ++c) total.s += sum_at(peer[c], total.m);
    }
    double term;
    float coef;
    terms.term(p, log_softmax(total, xt), term, coef);
    shared_row = make_float3(total.m, 1.0f / total.s, coef * grad);
    if (rank == 0) {
      out.store(r, kind, total, xt);
      p.term[r] = term;
      p.coef[r] = coef;
    }
  }
  __syncthreads();
  const RowGrad f{-shared_row.z * shared_row.y, shared_row.z, -shared_row.x};
  if (edge >= 0) drow[edge] = from_float<T>(f.one(xe, edge == t));
  // The target's vector in this slice, if it is here.
  const int64_t from = t - (head + part.v0 * V);
  const int tv = from >= 0 && from < (int64_t)n * V ? (int)(from / V) : -1;
#pragma unroll 2
  for (int u = w0 + lane; u < w1; u += 32) {
    st_stream(dbody + (int64_t)u * V, f.vec<T>(lds128(slice + (size_t)u * 16)));
    if (u == tv) drow[t] = from_float<T>(f.one(to_float(row[t]), true));
  }
}

// The same for short rows: one warp per row, which stays in registers.
template <typename T>
__global__ void __launch_bounds__(kShortWarps * 32)
policy_short_kernel(const T* __restrict__ logits, RowGrid lg, Targets tg, int64_t rows,
                    int64_t vocab, PolicyTerms p, float grad, RowOut out,
                    T* __restrict__ dlogits, RowGrid dg) {
  constexpr int V = Vec16<T>::N;
  constexpr int kHeld = kShortVecs / 32;  // vectors per lane
  const int lane = threadIdx.x & 31;
  const int64_t r = (int64_t)blockIdx.x * kShortWarps + (threadIdx.x >> 5);
  if (r >= rows) return;
  const RowIndex index = tg.index(r);
  const int64_t t = tg.at(index);
  const RowKind kind = row_kind(t, tg.ignore, vocab);
  const T* row = logits + lg.offset(index);
  T* drow = dlogits + dg.offset(index);
  const int head = head_elems(row, vocab);
  const int nvec = (int)((vocab - head) / V);
  const int64_t edge = edge_of(lane, head, head + (int64_t)nvec * V, vocab);
  const T* body = row + head;
  T* dbody = drow + head;
  if (kind != kRowUsed) {
    if (edge >= 0) drow[edge] = from_float<T>(0.0f);
    for (int v = lane; v < nvec; v += 32) st_stream(dbody + v * V, make_uint4(0, 0, 0, 0));
    if (lane == 0) {
      out.store(r, kind, Stat{0.0f, 1.0f}, 0.0f);
      p.term[r] = kind == kRowIgnored ? 0.0 : NAN;
      p.coef[r] = 0.0f;
    }
    return;
  }
  uint4 raw[kHeld];
#pragma unroll
  for (int u = 0; u < kHeld; ++u)
    if (lane + 32 * u < nvec) raw[u] = ld_stream(body + (lane + 32 * u) * V);
  PolicyRow terms;
  terms.load(p, index);
  const float xt = to_float(row[t]), xe = edge >= 0 ? to_float(row[edge]) : 0.0f;
  Running acc;
  if (edge >= 0) acc.add1(xe);
#pragma unroll
  for (int u = 0; u < kHeld; ++u) {
    if (lane + 32 * u < nvec) {
      float x[V];
      unpack<T>(raw[u], x);
      acc.template add<V>(x);
    }
  }
  const Stat own = acc.stat();
  Stat total;
  total.m = warp_max(own.m);
  total.s = warp_sum(sum_at(own, total.m));
  double term;
  float coef;
  terms.term(p, log_softmax(total, xt), term, coef);
  if (lane == 0) {
    out.store(r, kind, total, xt);
    p.term[r] = term;
    p.coef[r] = coef;
  }
  const float c = coef * grad;
  const RowGrad f{-c * (1.0f / total.s), c, -total.m};
  if (edge >= 0) drow[edge] = from_float<T>(f.one(xe, edge == t));
  const int tv = t >= head && t < head + (int64_t)nvec * V ? (int)((t - head) / V) : -1;
#pragma unroll
  for (int u = 0; u < kHeld; ++u) {
    const int v = lane + 32 * u;
    if (v < nvec) {
      st_stream(dbody + v * V, f.vec<T>(raw[u]));
      if (v == tv) drow[t] = from_float<T>(f.one(xt, true));
    }
  }
}

// dx *= grad / expected, unless they are equal. Zeros stay zeros, also where the factor is not
// finite: rows without a target have no gradient whatever the loss's is.
__device__ __forceinline__ float rescaled(float x, float f) { return x != 0.0f ? x * f : x; }
template <typename T>
__global__ void __launch_bounds__(kThreads)
rescale_kernel(T* __restrict__ dlogits, RowGrid dg, RowDiv index, int64_t rows, int64_t vocab,
               const float* __restrict__ grad, float expected) {
  constexpr int V = Vec16<T>::N;
  if (*grad == expected) return;
  const float f = *grad / expected;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    T* row = dlogits + dg.offset(index(r));
    const int head = head_elems(row, vocab);
    const int64_t nvec = (vocab - head) / V;
    for (int64_t v = threadIdx.x; v < nvec; v += kThreads) {
      uint4* at = reinterpret_cast<uint4*>(row + head + v * V);
      float x[V];
      unpack<T>(*at, x);
#pragma unroll
      for (int e = 0; e < V; ++e) x[e] = rescaled(x[e], f);
      *at = pack<T>(x);
    }
    if ((int)threadIdx.x < head)
      row[threadIdx.x] = from_float<T>(rescaled(to_float(row[threadIdx.x]), f));
    for (int64_t c = head + nvec * V + threadIdx.x; c < vocab; c += kThreads)
      row[c] = from_float<T>(rescaled(to_float(row[c]), f));
  }
}

// ------------------------------------------------------------------------- host side --

struct Rows {  // the checked geometry of a call
  int64_t rows, vocab, outer, inner;
  int splits, sms;
  RowGrid lg;
  Targets tg;
};

// Splits of each row for its statistics: one CTA a row when the rows alone fill the GPU, else so
// many that about eight CTAs per SM share the work, each with at least one unrolled trip of
// 16-byte vectors. (More splits, for a fuller last wave, gained 13 % at 1300 rows of 128256
// bf16 logits and lost 8 to 20 % at other sizes.)
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
      *rows > INT32_MAX || outer > INT32_MAX || inner > INT32_MAX)
    return set_error(PT_ERR_SHAPE, "outer, inner and their product must be in [0, 2^31)");
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
  g.lg = RowGrid{lo, li};
  g.tg = Targets{targets, RowGrid{to, ti}, ignore, RowDiv{FastDiv((uint32_t)g.inner)}};
  return PT_OK;
}

int check_optional(const void* p, const char* name, int64_t rows) {
  return rows > 0 ? check_device_ptr(p, name) : PT_OK;
}

// stats [rows, 2], read and written as pairs.
int check_stats(const float* stats, int64_t rows) {
  if (rows == 0) return PT_OK;
  if (int st = check_device_ptr(stats, "stats")) return st;
  if (reinterpret_cast<uintptr_t>(stats) % 8)
    return set_error(PT_ERR_INVALID_ARGUMENT, "stats must be 8-byte aligned");
  return PT_OK;
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
// One CTA per item, handed out as CTAs finish (items differ in length).
int grid_of(int64_t items) { return (int)std::min<int64_t>(items, INT32_MAX); }

// The longest rows, in 16-byte vectors, that one warp takes. Measured in bf16 against a CTA per row:
// statistics of 65536 x 1000 / 16384 x 8000 / 8192 x 16000 logits 50 / 54 / 52 against 160 / 109 / 72
// us (at 30000 logits even); gradient of 65536 x 1000 / 16384 x 8000 / 8192 x 16000 45 / 85 / 90
// against 159 / 95 / 86 us; policy pass of 65536 x 1000 / 32768 x 4000 108 / 107 against 207 / 157.
constexpr int kShortStatVecs = 2048;
constexpr int kShortGradVecs = 1024;
// Whether a warp takes a row: rows of at most `vecs` vectors that give every SM eight CTAs so.
bool short_rows(const Rows& g, int elem, int vecs) {
  return g.vocab * elem <= (int64_t)vecs * 16 && g.rows >= (int64_t)g.sms * 8 * kShortWarps;
}
unsigned short_grid(const Rows& g) { return (unsigned)((g.rows + kShortWarps - 1) / kShortWarps); }

template <typename T>
void launch_stats(const Rows& g, const void* logits, Stat* part, const RowOut& out,
                  cudaStream_t s) {
  const T* x = static_cast<const T*>(logits);
  if (short_rows(g, sizeof(T), kShortStatVecs)) {
    stats_short_kernel<T><<<short_grid(g), kShortWarps * 32, 0, s>>>(x, g.lg, g.tg, g.rows,
                                                                     g.vocab, out);
    return;
  }
  stats_kernel<T><<<grid_of(g.rows * g.splits), kThreads, 0, s>>>(
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

// Rows of logits and of their gradient have to start at the same place of a 16-byte vector.
int check_same_rows(const Rows& g, const void* logits, int64_t lo, int64_t li, const void* dlogits,
                    int64_t dlo, int64_t dli, int elem) {
  const uintptr_t gap = reinterpret_cast<uintptr_t>(logits) - reinterpret_cast<uintptr_t>(dlogits);
  if (gap % 16 || (g.outer > 1 && (lo - dlo) * elem % 16) ||
      (g.inner > 1 && (li - dli) * elem % 16))
    return set_error(PT_ERR_SHAPE, "rows of logits and dlogits must have the same address modulo "
                                   "16 bytes");
  return PT_OK;
}

struct PolicyInputs {
  const float* old;
  int64_t oo, oi;
  const float* adv;
  int64_t ao, ai;
  const float* ref;
  int64_t ro, ri;
  double low, high, kl;
};

int check_policy(Rows& g, Workspace& w, PolicyTerms& p, const PolicyInputs& in,
                 const void* logits, int64_t vocab, int64_t outer, int64_t inner, int64_t lo,
                 int64_t li, const int64_t* targets, int64_t to, int64_t ti, int64_t ignore,
                 float* loss, float* logps, float* stats, float* coef, void* workspace,
                 int64_t workspace_size, int dtype) {
  if (!(in.low >= 0.0) || !(in.high >= 0.0) || !std::isfinite(in.kl))
    return set_error(PT_ERR_INVALID_ARGUMENT,
                     "clip_low and clip_high must be >= 0 and kl_coef finite");
  if (int st = check_rows(g, logits, vocab, outer, inner, lo, li, targets, to, ti, ignore, dtype))
    return st;
  if (int st = check_device_ptr(loss, "loss")) return st;
  if (int st = check_optional(in.old, "old_logps", g.rows)) return st;
  if (int st = check_optional(in.adv, "advantages", g.rows)) return st;
  if (in.ref)
    if (int st = check_optional(in.ref, "reference", g.rows)) return st;
  if (int st = check_optional(logps, "logps", g.rows)) return st;
  if (int st = check_stats(stats, g.rows)) return st;
  if (int st = check_optional(coef, "coef", g.rows)) return st;
  if (int st = take_workspace(w, g, workspace, workspace_size)) return st;
  p.old = in.old;
  p.og = RowGrid{in.oo, in.oi};
  p.adv = in.adv;
  p.ag = RowGrid{in.ao, in.ai};
  p.ref = in.ref;
  p.rg = RowGrid{in.ro, in.ri};
  p.weight = w.seq;
  p.low = 1.0 - in.low;
  p.high = 1.0 + in.high;
  p.kl = in.kl;
  p.term = w.term;
  p.coef = coef;
  return PT_OK;
}

void launch_weights(const Rows& g, int64_t sequences, int by_sequence, double* weight,
                    cudaStream_t s) {
  const int counted = sequences > 0 && (by_sequence || g.rows > kCountAtOnce);
  if (counted) count_kernel<<<(unsigned)sequences, kSumThreads, 0, s>>>(g.tg, g.inner, weight);
  policy_weight_kernel<<<1, kSumThreads, 0, s>>>(g.tg, sequences, sequences > 0 ? g.rows : 0,
                                                 counted, by_sequence, weight);
}

// CTAs per row of the one-pass policy loss: as few as keep a slice within kSliceBytes, more (down
// to 4 KB a slice) while the rows alone do not give every SM eight CTAs; larger slices where
// the row does not fit eight such, 0 where it does not fit at all.
int cluster_size(int64_t rows, int64_t row_bytes, int sms) {
  if (row_bytes > (int64_t)kMaxCluster * kMaxSliceBytes || rows > INT32_MAX / kMaxCluster) return 0;
  int c = 1;
  while (c < kMaxCluster && (row_bytes > (int64_t)c * kSliceBytes ||
                             (rows * c < (int64_t)sms * 8 && row_bytes >= (int64_t)c * 8192)))
    c *= 2;
  return c;
}

template <typename T>
void launch_grad(const Rows& g, const void* logits, const float2* stats, const float* coef,
                 const RowGrid& cg, const float* grad, void* dlogits, const RowGrid& dg,
                 cudaStream_t s) {
  const T* x = static_cast<const T*>(logits);
  T* dx = static_cast<T*>(dlogits);
  if (short_rows(g, sizeof(T), kShortGradVecs)) {
    grad_short_kernel<T><<<short_grid(g), kShortWarps * 32, 0, s>>>(
        x, g.lg, g.tg, g.rows, g.vocab, stats, coef, cg, grad, dx, dg);
    return;
  }
  // kGradTrips unrolled trips per CTA, fewer (down to one) while that leaves SMs without eight CTAs.
  const int64_t trips = g.vocab / Vec16<T>::N / (kGradThreads * kUnrollGrad);
  const int64_t spread = std::min(trips, ((int64_t)g.sms * 8 + g.rows - 1) / g.rows);
  const int splits = (int)std::max<int64_t>({1, trips / kGradTrips, spread});
  grad_kernel<T><<<grid_of(g.rows * splits), kGradThreads, 0, s>>>(
      x, g.lg, g.tg, g.rows, g.vocab, splits, stats, coef, cg, grad, dx, dg);
}

// How long the next one-pass call of this thread waits (see pt_selftest_policy_wait).
thread_local long long g_next_wait_limit = kWaitLimitCycles;

template <typename T>
int launch_policy_grad(const Rows& g, const void* logits, int cluster, const PolicyTerms& p,
                       float grad, long long wait_limit, const RowOut& out, void* dlogits,
                       const RowGrid& dg, cudaStream_t s) {
  if (short_rows(g, sizeof(T), kShortVecs)) {
    policy_short_kernel<T><<<short_grid(g), kShortWarps * 32, 0, s>>>(
        static_cast<const T*>(logits), g.lg, g.tg, g.rows, g.vocab, p, grad, out,
        static_cast<T*>(dlogits), dg);
    return PT_OK;
  }
  // The largest slice: ceil(vectors / cluster) vectors (an unaligned row has fewer whole ones).
  const int64_t nvec = g.vocab / Vec16<T>::N;
  const size_t smem = (size_t)((nvec + cluster - 1) / cluster) * 16;
  // The limit is the same on every call: calls on two threads must not lower each other's.
  cudaError_t e = cudaFuncSetAttribute(policy_grad_kernel<T>,
                                       cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       kMaxSliceBytes);
  if (e == cudaSuccess) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(g.rows * cluster));
    cfg.blockDim = dim3(kFusedThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)cluster;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int log2_cluster = 0;
    while (1 << log2_cluster < cluster) ++log2_cluster;
    e = cudaLaunchKernelEx(&cfg, policy_grad_kernel<T>, static_cast<const T*>(logits), g.lg, g.tg,
                           g.vocab, log2_cluster, p, grad, wait_limit, out,
                           static_cast<T*>(dlogits), dg);
  }
  if (e != cudaSuccess) {
    cudaGetLastError();
    return set_error(PT_ERR_CUDA, "pt_policy_loss_grad: launch failed: %s",
                     cudaGetErrorString(e));
  }
  return PT_OK;
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
  if (int st = check_stats(stats, g.rows)) return st;
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
  if (int st = check_stats(stats, g.rows)) return st;
  if (int st = check_device_ptr(coef, "coef")) return st;
  if (int st = check_device_ptr(dlogits, "dlogits")) return st;
  if (grad)
    if (int st = check_device_ptr(grad, "grad")) return st;
  if (int st = check_same_rows(g, logits, logits_outer_stride, logits_inner_stride, dlogits,
                               dlogits_outer_stride, dlogits_inner_stride, dtype_size(dtype)))
    return st;
  const RowGrid cg{coef_outer_stride, coef_inner_stride};
  const RowGrid dg{dlogits_outer_stride, dlogits_inner_stride};
  const float2* st2 = reinterpret_cast<const float2*>(stats);
  cudaStream_t s = as_stream(stream);
  switch (dtype) {
    case PT_FLOAT32: launch_grad<float>(g, logits, st2, coef, cg, grad, dlogits, dg, s); break;
    case PT_FLOAT16: launch_grad<__half>(g, logits, st2, coef, cg, grad, dlogits, dg, s); break;
    default: launch_grad<__nv_bfloat16>(g, logits, st2, coef, cg, grad, dlogits, dg, s);
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
  if (int st = check_stats(stats, g.rows)) return st;
  if (int st = check_optional(rewards, "rewards", outer)) return st;
  if (int st = check_optional(coef, "coef", outer)) return st;
  Workspace w;
  if (int st = take_workspace(w, g, workspace, workspace_size)) return st;
  cudaStream_t s = as_stream(stream);
  row_stats(g, logits, dtype, w.part, RowOut{reinterpret_cast<float2*>(stats), nullptr, w.logps},
            s);
  if (outer > 0)
    pair_ratio_kernel<<<(unsigned)outer, 256, 0, s>>>(
        w.logps, reference, RowGrid{reference_outer_stride, reference_inner_stride}, g.tg, inner,
        w.seq);
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
  Workspace w;
  PolicyTerms p;
  const PolicyInputs in{old_logps, old_outer_stride, old_inner_stride,
                        advantages, advantages_outer_stride, advantages_inner_stride,
                        reference, reference_outer_stride, reference_inner_stride,
                        clip_low, clip_high, kl_coef};
  if (int st = check_policy(g, w, p, in, logits, vocab, outer, inner, logits_outer_stride,
                            logits_inner_stride, targets, targets_outer_stride,
                            targets_inner_stride, ignore_index, loss, logps, stats, coef,
                            workspace, workspace_size, dtype))
    return st;
  cudaStream_t s = as_stream(stream);
  row_stats(g, logits, dtype, w.part, RowOut{reinterpret_cast<float2*>(stats), logps, w.logps},
            s);
  const int64_t sequences = g.rows > 0 ? outer : 0;
  launch_weights(g, sequences, by_sequence, w.seq, s);
  if (g.rows > 0)
    policy_row_kernel<<<grid_of((g.rows + kThreads - 1) / kThreads, g.sms, 2048 / kThreads),
                        kThreads, 0, s>>>(w.logps, g.tg, g.rows, p);
  policy_sum_kernel<<<1, kSumThreads, 0, s>>>(w.term, g.rows, w.seq, sequences, loss);
  return check_launch("pt_policy_loss_fwd");
}

int pt_policy_loss_grad_supported(int64_t vocab, int64_t outer, int64_t inner, int dtype,
                                  int* supported) {
  if (supported == nullptr) return set_error(PT_ERR_INVALID_ARGUMENT, "supported is NULL");
  int64_t rows = 0;
  if (int st = check_sizes(vocab, outer, inner, &rows)) return st;
  const int elem = dtype_size(dtype);
  if (elem == 0) return set_error(PT_ERR_UNSUPPORTED_DTYPE, "unsupported dtype %d", dtype);
  *supported = cluster_size(rows, vocab * elem, 1) > 0;
  return ok();
}

int pt_policy_loss_grad(const void* logits, int64_t vocab, int64_t outer, int64_t inner,
                        int64_t logits_outer_stride, int64_t logits_inner_stride,
                        const int64_t* targets, int64_t targets_outer_stride,
                        int64_t targets_inner_stride, int64_t ignore_index,
                        const float* old_logps, int64_t old_outer_stride, int64_t old_inner_stride,
                        const float* advantages, int64_t advantages_outer_stride,
                        int64_t advantages_inner_stride, const float* reference,
                        int64_t reference_outer_stride, int64_t reference_inner_stride,
                        double clip_low, double clip_high, double kl_coef, int by_sequence,
                        double grad, float* loss, float* logps, float* stats, float* coef,
                        void* dlogits, int64_t dlogits_outer_stride, int64_t dlogits_inner_stride,
                        void* workspace, int64_t workspace_size, int dtype, void* stream) {
  const long long wait_limit = g_next_wait_limit;
  g_next_wait_limit = kWaitLimitCycles;
  if (!std::isfinite((float)grad))
    return set_error(PT_ERR_INVALID_ARGUMENT, "grad must be finite in fp32");
  Rows g;
  Workspace w;
  PolicyTerms p;
  const PolicyInputs in{old_logps, old_outer_stride, old_inner_stride,
                        advantages, advantages_outer_stride, advantages_inner_stride,
                        reference, reference_outer_stride, reference_inner_stride,
                        clip_low, clip_high, kl_coef};
  if (int st = check_policy(g, w, p, in, logits, vocab, outer, inner, logits_outer_stride,
                            logits_inner_stride, targets, targets_outer_stride,
                            targets_inner_stride, ignore_index, loss, logps, stats, coef,
                            workspace, workspace_size, dtype))
    return st;
  if (int st = check_optional(dlogits, "dlogits", g.rows)) return st;
  if (g.rows > 0)
    if (int st = check_same_rows(g, logits, logits_outer_stride, logits_inner_stride, dlogits,
                                 dlogits_outer_stride, dlogits_inner_stride, dtype_size(dtype)))
      return st;
  const int cluster = cluster_size(g.rows, vocab * dtype_size(dtype), g.sms);
  if (cluster == 0)
    return set_error(PT_ERR_SHAPE, "rows of %lld logits do not fit on chip (or too many rows)",
                     (long long)vocab);
  cudaStream_t s = as_stream(stream);
  const int64_t sequences = g.rows > 0 ? outer : 0;
  launch_weights(g, sequences, by_sequence, w.seq, s);
  if (g.rows > 0) {
    const RowGrid dg{dlogits_outer_stride, dlogits_inner_stride};
    const RowOut out{reinterpret_cast<float2*>(stats), logps, nullptr};
    int st;
    switch (dtype) {
      case PT_FLOAT32:
        st = launch_policy_grad<float>(g, logits, cluster, p, (float)grad, wait_limit, out,
                                       dlogits, dg, s);
        break;
      case PT_FLOAT16:
        st = launch_policy_grad<__half>(g, logits, cluster, p, (float)grad, wait_limit, out,
                                       dlogits, dg, s);
        break;
      default:
        st = launch_policy_grad<__nv_bfloat16>(g, logits, cluster, p, (float)grad, wait_limit, out,
                                               dlogits, dg, s);
    }
    if (st) return st;
  }
  policy_sum_kernel<<<1, kSumThreads, 0, s>>>(w.term, g.rows, w.seq, sequences, loss);
  return check_launch("pt_policy_loss_grad");
}

int pt_selftest_policy_wait(int64_t limit_cycles) {
  if (limit_cycles < -1 || limit_cycles > kWaitLimitCycles)
    return set_error(PT_ERR_INVALID_ARGUMENT, "limit_cycles must be in [-1, %lld] (got %lld)",
                     kWaitLimitCycles, (long long)limit_cycles);
  g_next_wait_limit = limit_cycles;
  return ok();
}

int pt_rescale_logits_grad(void* dlogits, int64_t vocab, int64_t outer, int64_t inner,
                           int64_t dlogits_outer_stride, int64_t dlogits_inner_stride,
                           const float* grad, double expected, int dtype, void* stream) {
  int64_t rows = 0;
  if (int st = check_sizes(vocab, outer, inner, &rows)) return st;
  if (dtype_size(dtype) == 0)
    return set_error(PT_ERR_UNSUPPORTED_DTYPE, "unsupported dtype %d", dtype);
  // As fp32, which the gradient was formed with: a smaller factor has left nothing to rescale.
  if (!std::isnormal((float)expected))
    return set_error(PT_ERR_INVALID_ARGUMENT, "expected must be a normal fp32 number");
  if (rows == 0) return ok();
  if (int st = check_device_ptr(dlogits, "dlogits")) return st;
  if (int st = check_device_ptr(grad, "grad")) return st;
  int sms = 0;
  if (int st = current_device_info(nullptr, &sms)) return st;
  const RowGrid dg{dlogits_outer_stride, dlogits_inner_stride};
  const RowDiv index{FastDiv((uint32_t)inner)};
  const int grid = grid_of(rows, sms, 2048 / kThreads);
  cudaStream_t s = as_stream(stream);
  switch (dtype) {
    case PT_FLOAT32:
      rescale_kernel<<<grid, kThreads, 0, s>>>(static_cast<float*>(dlogits), dg, index, rows, vocab,
                                               grad, (float)expected);
      break;
    case PT_FLOAT16:
      rescale_kernel<<<grid, kThreads, 0, s>>>(static_cast<__half*>(dlogits), dg, index, rows, vocab,
                                               grad, (float)expected);
      break;
    default:
      rescale_kernel<<<grid, kThreads, 0, s>>>(static_cast<__nv_bfloat16*>(dlogits), dg, index, rows,
                                               vocab, grad, (float)expected);
  }
  return check_launch("pt_rescale_logits_grad");
}

}  // extern "C"
