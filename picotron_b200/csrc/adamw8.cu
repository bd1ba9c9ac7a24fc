// AdamW step with the moments held in 8 bits, for a whole list of tensors per launch (sm_100a).
//
// Moments are kept in blocks of 256 consecutive elements that share one fp32 scale each:
//   exp_avg    = c |c| s   with c in [-127, 127] and s = max |exp_avg| / 127^2,
//   exp_avg_sq = c^4 s     with c in [0, 255]    and s = max exp_avg_sq / 255^4,
// so codes are uniform in the square root of exp_avg and in the fourth root of exp_avg_sq (the
// square root of the update's denominator): small values keep a relative step that grows only
// with the root of their distance to the block's largest. A positive exp_avg_sq under a positive
// scale never takes code 0, which would drop the denominator to eps. The step itself is AdamW in
// fp32:
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g g       (every product and sum rounded)
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// Each new code is the one nearest to the new fp32 moment in the root's domain. The candidate
// comes from the approximate square root; where it lies within 1e-4 of a border between two
// codes (above the 5.7e-5 that reciprocal, product and two square roots, 2^-23 each, can be off
// by at code 255), the border itself,
// ((2c + 1) / 2)^2 s or ((2c + 1) / 2)^4 s, is compared with the moment in 64 bits, so the code
// does not depend on how the root was computed.
//
// One warp per block of 256, eight elements per lane; the block's two maxima by integer max over
// the warp (for values >= 0 the bit patterns order like the values, NaN above all). The parameter's
// update alone takes the approximate square root and reciprocal (2^-23 each): it is within 2^-21
// of its value, less than the rounding of an fp32 parameter of eight times its size or more.
// Bytes per element: 3 parameter widths (parameter read and written, gradient read) + 4. In fp32
// the kernel is bound by HBM (436 M parameters: 1.07 ms, the copy rate); in 16 bits, with 10 bytes
// an element in place of 16 and the same arithmetic, by instruction issue (0.87 ms, 0.77 of it).
#include <algorithm>
#include <cmath>

#include "common.cuh"

namespace pt {

__device__ int g_adamw8_error = 0;

namespace {

constexpr int kThreads = 256;
constexpr int kBlock = 256;            // elements that share a scale

constexpr int kWarps = kThreads / 32;
constexpr int kStages = 2;             // blocks that a warp's copies run ahead (see adamw8_kernel)
constexpr int kMaxWarpBlocks = 16;     // blocks per warp and work item, at most
constexpr int kBatch = 96;             // tensors per launch (10 KB of kernel parameters)
constexpr float kTiny = 1.17549435e-38f;  // smallest normal: a smaller scale is kept as 0
constexpr float kMomentScale = (float)(1.0 / 16129.0);        // 127^-2
constexpr float kSquareScale = (float)(1.0 / 4228250625.0);   // 255^-4
constexpr float kBorder = 0.4999f;
// A block whose largest exp_avg_sq is below 255^4 kTiny = 5e-29 keeps a scale of 0, and eps alone
// is left in the next step's denominator. Its gradients were below sqrt(5e-29 / (1 - b2)), and so
// is m / (1 - b1^t): with an eps of 1e-12 a step is at most 0.22 lr for a b2 of 0.999 (0.7 lr for
// 0.9999). An eps of 1e-15 would let it be 220 lr, and one below kTiny, which the approximate
// square root and reciprocal take for 0, infinite.
constexpr double kLeastEps = 1e-12;


struct Tensor {
  void* param;
  const void* grad;
  int8_t* mc;
  float* ms;
  uint8_t* vc;
  float* vs;
  int64_t numel;
  int64_t item_end;   // work items of this tensor and all before it in the batch
  float step_size;    // lr / (1 - beta1^t)
  float root;         // 1 / sqrt(1 - beta2^t)
  float decay;        // 1 - lr * weight_decay
};

struct Batch {
  Tensor t[kBatch];
  int count;
  int warp_blocks;  // blocks per warp and work item
};

struct Scalars {
  float b1, w1, b2, w2, eps;
  int maximize;
};

__device__ __forceinline__ float approx_sqrt(float x) {
  float y;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float approx_rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The larger of two values >= 0, NaN if either is (fmaxf would drop it).
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ float warp_top(float v) {
  return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v)));
}

// The sum of two pairs of products, each product rounded and then the sum. Packed products and
// sums (mul and add of f32x2, .rn in PTX as well) were contracted into fused multiply-adds, which
// the definition of the moments rules out; scalar sums with explicit rounding are not.
__device__ __forceinline__ float2 sum_of_products(float2 a, float2 wa, float2 b, float2 wb) {
  const float2 x = __fmul2_rn(a, wa), y = __fmul2_rn(b, wb);
  return make_float2(__fadd_rn(x.x, y.x), __fadd_rn(x.y, y.y));
}

// Whole numbers in the low byte of an fp32: x + kWhole is x rounded to the nearest whole number,
// ties to even, whose two's complement is the low bits (|x| < 2^22).
constexpr float kWhole = 12582912.0f;  // 1.5 * 2^23

// Byte e of w as an fp32: 2^23 with the byte in its low bits, less 2^23 and `bias`.
__device__ __forceinline__ float2 bytes_to_float2(uint32_t w, int e, float bias) {
  const uint32_t a = __byte_perm(w, 0x4b000000u, 0x7440 + e);
  const uint32_t b = __byte_perm(w, 0x4b000000u, 0x7441 + e);
  return __fadd2_rn(make_float2(__uint_as_float(a), __uint_as_float(b)), splat2(-8388608.0f - bias));
}
// The low bytes of four values that kWhole was added to.
__device__ __forceinline__ uint32_t low_bytes(float2 a, float2 b) {
  const uint32_t lo = __byte_perm(__float_as_uint(a.x), __float_as_uint(a.y), 0x0040);
  const uint32_t hi = __byte_perm(__float_as_uint(b.x), __float_as_uint(b.y), 0x0040);
  return __byte_perm(lo, hi, 0x5410);
}

// Eight moments of one lane as codes, and the values that codes stand for. Every product that is
// part of the definition is rounded by itself.
__device__ __forceinline__ void moment_values(uint2 codes, float scale, float2 (&m)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    // int8 as a byte with 128 added.
    float2 c = bytes_to_float2((i < 2 ? codes.x : codes.y) ^ 0x80808080u, 2 * (i & 1), 128.0f);
    c = make_float2(c.x * fabsf(c.x), c.y * fabsf(c.y));
    m[i] = __fmul2_rn(c, splat2(scale));
  }
}
__device__ __forceinline__ void square_values(uint2 codes, float scale, float2 (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float2 c = bytes_to_float2(i < 2 ? codes.x : codes.y, 2 * (i & 1), 0.0f);
    c = __fmul2_rn(c, c);
    v[i] = __fmul2_rn(__fmul2_rn(c, c), splat2(scale));
  }
}

// The exact choice between codes lo and lo + 1 for a root next to lo + 1/2: the moment (times
// 2^power) against the border (2 lo + 1)^power s, both exact or within 2^-53; ties to even.
template <int kPower>
__device__ __noinline__ float border_code(float root, float x, float s) {
  const int lo = (int)floorf(root);
  double b = (double)(2 * lo + 1);
  b *= b;
  if (kPower == 4) b *= b;
  const double border = b * (double)s, value = (double)(1 << kPower) * (double)x;
  return (float)(value > border || (value == border && (lo & 1)) ? lo + 1 : lo);
}

// How far a root is from the whole number that it was rounded to in `t`.
__device__ __forceinline__ float off_whole(float root, float t) {
  return fabsf(__fsub_rn(root, __fsub_rn(t, kWhole)));
}
__device__ __forceinline__ float2 to_whole(float2 root, float& worst) {
  const float2 t = __fadd2_rn(root, splat2(kWhole));
  const float2 c = __fadd2_rn(t, splat2(-kWhole));
  const float2 d = __fadd2_rn(root, make_float2(-c.x, -c.y));
  worst = fmaxf(worst, fmaxf(fabsf(d.x), fabsf(d.y)));
  return t;
}

// The codes nearest to eight moments in the root's domain; zeros, which stand for NaN, under a
// scale that is not finite.
__device__ __forceinline__ uint2 moment_codes(const float2 (&m)[4], float s) {
  if (!(s < INFINITY)) return make_uint2(0, 0);
  const float inv = s > 0.0f ? approx_rcp(s) : 0.0f;
  float2 r[4], t[4];
  float worst = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 q = __fmul2_rn(m[i], splat2(inv));
    r[i] = make_float2(copysignf(approx_sqrt(fabsf(q.x)), m[i].x),
                       copysignf(approx_sqrt(fabsf(q.y)), m[i].y));
    t[i] = to_whole(r[i], worst);
  }
  if (worst > kBorder) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (off_whole(r[i].x, t[i].x) > kBorder)
        t[i].x = kWhole + copysignf(border_code<2>(fabsf(r[i].x), fabsf(m[i].x), s), m[i].x);
      if (off_whole(r[i].y, t[i].y) > kBorder)
        t[i].y = kWhole + copysignf(border_code<2>(fabsf(r[i].y), fabsf(m[i].y), s), m[i].y);
    }
  }
  return make_uint2(low_bytes(t[0], t[1]), low_bytes(t[2], t[3]));
}
__device__ __forceinline__ uint2 square_codes(const float2 (&v)[4], float s) {
  if (!(s < INFINITY)) return make_uint2(0, 0);
  const float inv = s > 0.0f ? approx_rcp(s) : 0.0f, least = s > 0.0f ? 1.0f : 0.0f;
  float2 r[4], t[4];
  float worst = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 q = __fmul2_rn(v[i], splat2(inv));
    r[i] = make_float2(approx_sqrt(approx_sqrt(q.x)), approx_sqrt(approx_sqrt(q.y)));
    if (v[i].x > 0.0f) r[i].x = fmaxf(r[i].x, least);
    if (v[i].y > 0.0f) r[i].y = fmaxf(r[i].y, least);
    t[i] = to_whole(r[i], worst);
  }
  if (worst > kBorder) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (off_whole(r[i].x, t[i].x) > kBorder) t[i].x = kWhole + border_code<4>(r[i].x, v[i].x, s);
      if (off_whole(r[i].y, t[i].y) > kBorder) t[i].y = kWhole + border_code<4>(r[i].y, v[i].y, s);
    }
  }
  return make_uint2(low_bytes(t[0], t[1]), low_bytes(t[2], t[3]));
}

struct StepScalars {
  float step_size, root, decay;
};

// The parameters' step on one warp's block, and its new moments: p, g and the codes of this lane
// in registers (elements past the end hold g = 0 and codes 0, so they change no maximum). ms, vs:
// the block's scales, in and out.
__device__ __forceinline__ void step_block(float2 (&p)[4], const float2 (&g)[4], uint2 mc,
                                           uint2 vc, float2 (&m)[4], float2 (&v)[4], float& ms,
                                           float& vs, const Scalars& k, const StepScalars& t) {
  moment_values(mc, ms, m);
  square_values(vc, vs, v);
  float mtop = 0.0f, vtop = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = sum_of_products(m[i], splat2(k.b1), g[i], splat2(k.w1));
    v[i] = sum_of_products(v[i], splat2(k.b2), __fmul2_rn(g[i], g[i]), splat2(k.w2));
    mtop = max_nan(mtop, max_nan(fabsf(m[i].x), fabsf(m[i].y)));
    vtop = max_nan(vtop, max_nan(v[i].x, v[i].y));
    const float2 d = __ffma2_rn(make_float2(approx_sqrt(v[i].x), approx_sqrt(v[i].y)),
                                splat2(t.root), splat2(k.eps));
    const float2 u = __fmul2_rn(m[i], make_float2(approx_rcp(d.x), approx_rcp(d.y)));
    p[i] = __ffma2_rn(u, splat2(-t.step_size), __fmul2_rn(p[i], splat2(t.decay)));
  }
  ms = __fmul_rn(warp_top(mtop), kMomentScale);
  vs = __fmul_rn(warp_top(vtop), kSquareScale);
  ms = ms < kTiny ? 0.0f : ms;
  vs = vs < kTiny ? 0.0f : vs;
}

// Eight elements from shared memory.
template <typename T> __device__ __forceinline__ void lds8(const T* p, float2 (&f)[4]) {
  if constexpr (sizeof(T) == 4) {
    unpack2<T>(lds128(p), f);
    unpack2<T>(lds128(p + 4), f + 2);
  } else {
    unpack2<T>(lds128(p), f);
  }
}
template <typename T> __device__ __forceinline__ void store8(T* p, const float2 (&f)[4]) {
  float t[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    t[2 * i] = f[i].x;
    t[2 * i + 1] = f[i].y;
  }
  if constexpr (sizeof(T) == 4)
    st_global_v8(p, t);
  else
    *reinterpret_cast<uint4*>(p) = pack<T>(t);
}

// The tensor that a work item belongs to (items of tensor i end at t[i].item_end).
template <typename B> __device__ __forceinline__ int tensor_of(const B& batch, int64_t item) {
  int lo = 0, hi = batch.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (item < batch.t[mid].item_end)
      hi = mid;
    else
      lo = mid + 1;
  }
  return lo;
}

// What one warp's block takes from memory, as it lies in shared memory: 256 elements of each.
template <typename T> struct Stage {
  T p[kBlock];
  T g[kBlock];
  int8_t mc[kBlock];
  uint8_t vc[kBlock];
};

// A warp's whole blocks come through a ring of kStages stages in shared memory, filled by bulk
// copies that run ahead: with plain loads the time followed the number of resident warps (2.8,
// 2.1 and 1.7 ms with 2, 3 and 4 CTAs per SM), since a block's loads waited for the arithmetic of
// the one before. 436 M fp32 parameters take 1.07 ms, the time of their bytes at the copy rate,
// with 16 blocks a warp, 2 stages and 3 CTAs per SM (1.08 ms with 8 blocks, 1.25 with 4; 1.09
// with 3 stages; 1.09 with 4 CTAs, 1.10 with 2 CTAs of 3 stages).
template <typename T>
__global__ void __launch_bounds__(kThreads, 3)
adamw8_kernel(const __grid_constant__ Batch batch, Scalars k) {
  extern __shared__ __align__(128) unsigned char shared[];
  __shared__ uint64_t bars[kWarps][kStages];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t item = blockIdx.x;
  const int which = tensor_of(batch, item);
  const Tensor& t = batch.t[which];
  const int64_t first = which > 0 ? batch.t[which - 1].item_end : 0;
  T* const P = static_cast<T*>(t.param);
  const T* const G = static_cast<const T*>(t.grad);
  int8_t* const MC = t.mc;
  uint8_t* const VC = t.vc;
  const int64_t numel = t.numel;
  const StepScalars sc{t.step_size, t.root, t.decay};
  const uintptr_t bits = reinterpret_cast<uintptr_t>(P) | reinterpret_cast<uintptr_t>(G) |
                         reinterpret_cast<uintptr_t>(MC) | reinterpret_cast<uintptr_t>(VC);
  // Whole blocks of arrays on 32-byte boundaries; anything else goes element by element.
  const int64_t whole = bits % 32 == 0 ? numel / kBlock : 0;
  const int64_t blocks = (numel + kBlock - 1) / kBlock;
  const int64_t b0 = ((item - first) * kWarps + warp) * batch.warp_blocks;  // consecutive blocks
  const int n = (int)max((int64_t)0, min((int64_t)batch.warp_blocks, whole - b0));
  Stage<T>* ring = reinterpret_cast<Stage<T>*>(shared) + warp * kStages;
  uint64_t* bar = bars[warp];
  auto fetch = [&](int j) {  // by lane 0
    Stage<T>& s = ring[j % kStages];
    uint64_t* at = &bar[j % kStages];
    const int64_t o = (b0 + j) * kBlock;
    mbar_arrive_expect_tx(at, sizeof(Stage<T>));
    bulk_load(s.p, P + o, sizeof(s.p), at);
    bulk_load(s.g, G + o, sizeof(s.g), at);
    bulk_load(s.mc, MC + o, sizeof(s.mc), at);
    bulk_load(s.vc, VC + o, sizeof(s.vc), at);
  };
  if (lane == 0 && n > 0) {
    for (int j = 0; j < kStages; ++j) mbar_init(&bar[j], 1);
    fence_mbar_init();
    for (int j = 0; j < min(n, kStages); ++j) fetch(j);
  }
  __syncwarp();
  float ms = 0.0f, vs = 0.0f;
  if (n > 0) {
    ms = t.ms[b0];
    vs = t.vs[b0];
  }
#pragma unroll 1
  for (int j = 0; j < n; ++j) {
    const int64_t b = b0 + j;
    float next_ms = 0.0f, next_vs = 0.0f;
    if (j + 1 < n) {
      next_ms = t.ms[b + 1];
      next_vs = t.vs[b + 1];
    }
    if (!mbar_wait_bounded(&bar[j % kStages], (uint32_t)(j / kStages) & 1u)) {
      // Nothing of this block, or of the warp's blocks behind it, is changed; the copies that are
      // still on their way are given their time as well.
      if (lane == 0) atomicExch(&g_adamw8_error, kDeviceErrWaitTimeout);
      for (int i = j + 1; i < min(n, j + kStages); ++i)
        mbar_wait_bounded(&bar[i % kStages], (uint32_t)(i / kStages) & 1u);
      return;
    }
    const Stage<T>& s = ring[j % kStages];
    float2 p[4], g[4], m[4], v[4];
    lds8<T>(s.p + lane * 8, p);
    lds8<T>(s.g + lane * 8, g);
    const uint2 mc = *reinterpret_cast<const uint2*>(s.mc + lane * 8);
    const uint2 vc = *reinterpret_cast<const uint2*>(s.vc + lane * 8);
    __syncwarp();  // all lanes have read the stage
    if (lane == 0 && j + kStages < n) fetch(j + kStages);
    if (k.maximize)
#pragma unroll
      for (int i = 0; i < 4; ++i) g[i] = make_float2(-g[i].x, -g[i].y);
    step_block(p, g, mc, vc, m, v, ms, vs, k, sc);
    const int64_t o = b * kBlock + lane * 8;
    store8<T>(P + o, p);
    *reinterpret_cast<uint2*>(MC + o) = moment_codes(m, ms);
    *reinterpret_cast<uint2*>(VC + o) = square_codes(v, vs);
    if (lane == 0) {
      t.ms[b] = ms;
      t.vs[b] = vs;
    }
    ms = next_ms;
    vs = next_vs;
  }
#pragma unroll 1
  for (int64_t b = max(b0, whole); b < min(b0 + batch.warp_blocks, blocks); ++b) {
    float2 p[4], g[4], m[4], v[4];
    float pe[8], ge[8];
    uint2 mc = make_uint2(0, 0), vc = make_uint2(0, 0);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int64_t o = b * kBlock + e * 32 + lane;
      const bool in = o < numel;
      pe[e] = in ? to_float(P[o]) : 0.0f;
      ge[e] = in ? to_float(G[o]) : 0.0f;
      ge[e] = k.maximize ? -ge[e] : ge[e];
      (e < 4 ? mc.x : mc.y) |= (in ? (uint32_t)(uint8_t)MC[o] : 0u) << (8 * (e & 3));
      (e < 4 ? vc.x : vc.y) |= (in ? (uint32_t)VC[o] : 0u) << (8 * (e & 3));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      p[i] = make_float2(pe[2 * i], pe[2 * i + 1]);
      g[i] = make_float2(ge[2 * i], ge[2 * i + 1]);
    }
    float bms = t.ms[b], bvs = t.vs[b];
    step_block(p, g, mc, vc, m, v, bms, bvs, k, sc);
    mc = moment_codes(m, bms);
    vc = square_codes(v, bvs);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int64_t o = b * kBlock + e * 32 + lane;
      if (o < numel) {
        P[o] = from_float<T>(e & 1 ? p[e / 2].y : p[e / 2].x);
        MC[o] = (int8_t)((e < 4 ? mc.x : mc.y) >> (8 * (e & 3)));
        VC[o] = (uint8_t)((e < 4 ? vc.x : vc.y) >> (8 * (e & 3)));
      }
    }
    if (lane == 0) {
      t.ms[b] = bms;
      t.vs[b] = bvs;
    }
  }
}

// The fp32 moments that codes and scales stand for: 10 bytes per element, most of them written.
// 436 M elements take 0.65 ms, the copy rate (0.68 ms with 8 or 16 blocks a warp).
constexpr int kMomentWarpBlocks = 4;
struct MomentTensor {
  const int8_t* mc;
  const float* ms;
  const uint8_t* vc;
  const float* vs;
  float* m;
  float* v;
  int64_t numel;
  int64_t item_end;
};
struct MomentBatch {
  MomentTensor t[kBatch];
  int count;
  int warp_blocks;
};

__global__ void __launch_bounds__(kThreads)
moments_kernel(const __grid_constant__ MomentBatch batch) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t item = blockIdx.x;
  const int which = tensor_of(batch, item);
  const MomentTensor t = batch.t[which];
  const int64_t first = which > 0 ? batch.t[which - 1].item_end : 0;
  const bool aligned =
      (reinterpret_cast<uintptr_t>(t.mc) | reinterpret_cast<uintptr_t>(t.vc)) % 8 == 0 &&
      (reinterpret_cast<uintptr_t>(t.m) | reinterpret_cast<uintptr_t>(t.v)) % 32 == 0;
  const int64_t blocks = (t.numel + kBlock - 1) / kBlock;
  const int64_t b0 = (item - first) * batch.warp_blocks * kWarps + warp;
#pragma unroll 4
  for (int j = 0; j < batch.warp_blocks; ++j) {
    const int64_t b = b0 + j * kWarps;
    if (b >= blocks) break;
    const float ms = t.ms[b], vs = t.vs[b];
    const int64_t at = b * kBlock;
    if (aligned && at + kBlock <= t.numel) {
      const int64_t o = at + lane * 8;
      float2 m[4], v[4];
      moment_values(*reinterpret_cast<const uint2*>(t.mc + o), ms, m);
      square_values(*reinterpret_cast<const uint2*>(t.vc + o), vs, v);
      store8<float>(t.m + o, m);
      store8<float>(t.v + o, v);
    } else {
      for (int64_t o = at + lane; o < min(at + kBlock, t.numel); o += 32) {
        const int c = t.mc[o], d = t.vc[o];
        const float d2 = (float)(d * d);
        t.m[o] = (float)(c * abs(c)) * ms;
        t.v[o] = __fmul_rn(__fmul_rn(d2, d2), vs);
      }
    }
  }
}

int64_t blocks_of(int64_t numel) { return (numel + kBlock - 1) / kBlock; }

// Blocks per warp: `most` where the tensors have that many for every warp of the GPU four times
// over, fewer for smaller ones (small launches take as long as one warp's share).
int warp_blocks(const int64_t* numels, int num_tensors, int sms, int most) {
  int64_t blocks = 0;
  for (int i = 0; i < num_tensors; ++i) blocks += blocks_of(numels[i]);
  return (int)std::max<int64_t>(1, std::min<int64_t>(most, blocks / (sms * 3 * kWarps * 4)));
}
int64_t items_of(int64_t numel, int warp_blocks) {
  const int64_t per = (int64_t)warp_blocks * kWarps;
  return (blocks_of(numel) + per - 1) / per;
}

int check_state(int i, int64_t numel, const int8_t* mc, const float* ms, const uint8_t* vc,
                const float* vs) {
  if (numel < 0 || numel > (int64_t(1) << 34))
    return set_error(PT_ERR_SHAPE, "tensor %d: numel must be in [0, 2^34]", i);
  if (numel == 0) return PT_OK;
  const char* what[4] = {"exp_avg codes", "exp_avg scales", "exp_avg_sq codes",
                         "exp_avg_sq scales"};
  const void* ptr[4] = {mc, ms, vc, vs};
  for (int k = 0; k < 4; ++k)
    if (int st = check_device_ptr(ptr[k], what[k])) return st;
  return PT_OK;
}

template <typename T>
void launch_step(const Batch& b, const Scalars& k, int64_t items, cudaStream_t s) {
  const int smem = (int)(sizeof(Stage<T>) * kWarps * kStages);
  if (cudaFuncSetAttribute(adamw8_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) ==
      cudaSuccess)
    adamw8_kernel<T><<<(unsigned)items, kThreads, smem, s>>>(b, k);
}

}  // namespace

// Reads and clears this file's device error word (called by pt_take_device_error).
int take_adamw8_device_error(int* code);
int take_adamw8_device_error(int* code) {
  int v = 0;
  const int zero = 0;
  if (cudaMemcpyFromSymbol(&v, g_adamw8_error, sizeof(int)) != cudaSuccess ||
      (v != 0 && cudaMemcpyToSymbol(g_adamw8_error, &zero, sizeof(int)) != cudaSuccess)) {
    cudaGetLastError();
    return set_error(PT_ERR_CUDA, "cannot read the device error word");
  }
  *code = v;
  return PT_OK;
}

}  // namespace pt

using namespace pt;

extern "C" {

int pt_adamw8_step(void* const* params, const void* const* grads, int8_t* const* exp_avg_codes,
                   float* const* exp_avg_scales, uint8_t* const* exp_avg_sq_codes,
                   float* const* exp_avg_sq_scales, const int64_t* numels, const int64_t* steps,
                   const double* lrs, const double* weight_decays, int num_tensors, double beta1,
                   double beta2, double eps, int maximize, int dtype, void* stream) {
  if (num_tensors < 0) return set_error(PT_ERR_INVALID_ARGUMENT, "num_tensors must be >= 0");
  const int elem = dtype_size(dtype);
  if (elem == 0) return set_error(PT_ERR_UNSUPPORTED_DTYPE, "unsupported dtype %d", dtype);
  if (num_tensors == 0) return ok();
  if (!params || !grads || !exp_avg_codes || !exp_avg_scales || !exp_avg_sq_codes ||
      !exp_avg_sq_scales || !numels || !steps || !lrs || !weight_decays)
    return set_error(PT_ERR_INVALID_ARGUMENT, "a tensor list pointer is NULL");
  if (!(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0) || !(eps >= kLeastEps))
    return set_error(PT_ERR_INVALID_ARGUMENT, "betas must be in [0, 1) and eps >= 1e-12");
  // Everything is checked before the first launch: a refused call changes nothing.
  for (int i = 0; i < num_tensors; ++i) {
    if (int st = check_state(i, numels[i], exp_avg_codes[i], exp_avg_scales[i],
                             exp_avg_sq_codes[i], exp_avg_sq_scales[i]))
      return st;
    if (steps[i] < 1)
      return set_error(PT_ERR_INVALID_ARGUMENT, "tensor %d: step must be >= 1", i);
    if (numels[i] == 0) continue;
    if (int st = check_device_ptr(params[i], "param")) return st;
    if (int st = check_device_ptr(grads[i], "grad")) return st;
    if ((reinterpret_cast<uintptr_t>(params[i]) | reinterpret_cast<uintptr_t>(grads[i])) % elem)
      return set_error(PT_ERR_INVALID_ARGUMENT, "tensor %d is not aligned to its element size", i);
  }
  const Scalars k{(float)beta1, (float)(1.0 - beta1), (float)beta2, (float)(1.0 - beta2),
                  (float)eps, maximize != 0};
  cudaStream_t s = as_stream(stream);
  int sms = 0;
  if (int st = current_device_info(nullptr, &sms)) return st;
  const int per_warp = warp_blocks(numels, num_tensors, sms, kMaxWarpBlocks);
  for (int i = 0; i < num_tensors;) {
    Batch b;
    b.count = 0;
    b.warp_blocks = per_warp;
    int64_t items = 0;
    for (; i < num_tensors && b.count < kBatch; ++i) {
      if (numels[i] == 0) continue;
      items += items_of(numels[i], per_warp);
      const double bc1 = 1.0 - std::pow(beta1, (double)steps[i]);
      const double bc2 = 1.0 - std::pow(beta2, (double)steps[i]);
      b.t[b.count++] = Tensor{params[i], grads[i], exp_avg_codes[i], exp_avg_scales[i],
                              exp_avg_sq_codes[i], exp_avg_sq_scales[i], numels[i], items,
                              (float)(lrs[i] / bc1), (float)(1.0 / std::sqrt(bc2)),
                              (float)(1.0 - lrs[i] * weight_decays[i])};
    }
    if (b.count == 0) break;
    switch (dtype) {
      case PT_FLOAT32: launch_step<float>(b, k, items, s); break;
      case PT_FLOAT16: launch_step<__half>(b, k, items, s); break;
      default: launch_step<__nv_bfloat16>(b, k, items, s);
    }
    if (int st = check_launch("pt_adamw8_step")) return st;
  }
  return ok();
}

int pt_adamw8_moments(const int8_t* const* exp_avg_codes, const float* const* exp_avg_scales,
                      const uint8_t* const* exp_avg_sq_codes,
                      const float* const* exp_avg_sq_scales, const int64_t* numels,
                      float* const* exp_avgs, float* const* exp_avg_sqs, int num_tensors,
                      void* stream) {
  if (num_tensors < 0) return set_error(PT_ERR_INVALID_ARGUMENT, "num_tensors must be >= 0");
  if (num_tensors == 0) return ok();
  if (!exp_avg_codes || !exp_avg_scales || !exp_avg_sq_codes || !exp_avg_sq_scales || !numels ||
      !exp_avgs || !exp_avg_sqs)
    return set_error(PT_ERR_INVALID_ARGUMENT, "a tensor list pointer is NULL");
  for (int i = 0; i < num_tensors; ++i) {
    if (int st = check_state(i, numels[i], exp_avg_codes[i], exp_avg_scales[i],
                             exp_avg_sq_codes[i], exp_avg_sq_scales[i]))
      return st;
    if (numels[i] == 0) continue;
    if (int st = check_device_ptr(exp_avgs[i], "exp_avg")) return st;
    if (int st = check_device_ptr(exp_avg_sqs[i], "exp_avg_sq")) return st;
  }
  int sms = 0;
  if (int st = current_device_info(nullptr, &sms)) return st;
  const int per_warp = warp_blocks(numels, num_tensors, sms, kMomentWarpBlocks);
  for (int i = 0; i < num_tensors;) {
    MomentBatch b;
    b.count = 0;
    b.warp_blocks = per_warp;
    int64_t items = 0;
    for (; i < num_tensors && b.count < kBatch; ++i) {
      if (numels[i] == 0) continue;
      items += items_of(numels[i], per_warp);
      b.t[b.count++] = MomentTensor{exp_avg_codes[i], exp_avg_scales[i], exp_avg_sq_codes[i],
                                    exp_avg_sq_scales[i], exp_avgs[i], exp_avg_sqs[i],
                                    numels[i], items};
    }
    if (b.count == 0) break;
    const unsigned grid = (unsigned)items;
    moments_kernel<<<grid, kThreads, 0, as_stream(stream)>>>(b);
    if (int st = check_launch("pt_adamw8_moments")) return st;
  }
  return ok();
}

}  // extern "C"
