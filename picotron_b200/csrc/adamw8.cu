// AdamW step with the moments held in 8 bits, for a whole list of tensors per launch (sm_100a).
//
// Moments are kept in blocks of 256 consecutive elements that share one fp32 scale each:
//   exp_avg    = c |c| s   with c in [-127, 127] and s = max |exp_avg| / 127^2,
//   exp_avg_sq = c^4 s     with c in [0, 255]    and s = max exp_avg_sq / 255^4,
// so codes are uniform in the square root of exp_avg and in the fourth root of exp_avg_sq (the
// square root of the update's denominator): small values keep a relative step that grows only
// with the root of their distance to the block's largest. A positive exp_avg_sq never takes code
// 0, which would drop the denominator to eps. The step itself is AdamW in fp32:
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g g       (every product and sum rounded)
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// Each new code is the one nearest to the new fp32 moment in the root's domain. The candidate
// comes from the approximate square root; where it lies within 2e-4 of a border between two
// codes (above the 6e-5 that the approximations can be off by at code 255), the border itself,
// ((2c + 1) / 2)^2 s or ((2c + 1) / 2)^4 s, is compared with the moment in 64 bits, so the code
// does not depend on how the root was computed.
//
// One warp per block of 256: eight elements per lane in 32-byte loads, the block's two maxima by
// integer max over the warp (for values >= 0 the bit patterns order like the values, NaN above
// all). Bytes per element: 3 parameter widths (parameter read and written, gradient read) + 4;
// the kernel is bound by HBM.
#include <cmath>

#include "common.cuh"

namespace pt {
namespace {

constexpr int kThreads = 256;
constexpr int kBlock = 256;            // elements that share a scale
constexpr int kWarpBlocks = 4;         // quantisation blocks per warp and work item
constexpr int kItemBlocks = kThreads / 32 * kWarpBlocks;  // per work item (8192 elements)
constexpr int kBatch = 96;             // tensors per launch (10 KB of kernel parameters)
constexpr float kTiny = 1.17549435e-38f;  // smallest normal: a smaller scale is kept as 0
constexpr float kMomentScale = (float)(1.0 / 16129.0);        // 127^-2
constexpr float kSquareScale = (float)(1.0 / 4228250625.0);   // 255^-4
constexpr float kBorder = 0.4998f;

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
};

struct Scalars {
  float b1, w1, b2, w2, eps;
  int maximize;
};

__device__ __forceinline__ float approx_sqrt(float x) {
  float y;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The eight codes of one lane's part of a block.
struct Codes {
  int8_t m[8];
  uint8_t v[8];
};

// sqrt(q) rounded to the nearest code, ties to even; x = |moment|, q = x / s approximately.
__device__ __forceinline__ int moment_code(float x, float s, float inv) {
  const float r = approx_sqrt(x * inv);
  float c = rintf(r);
  if (fabsf(r - c) > kBorder) {
    const int lo = (int)floorf(r);
    const double b = (double)(2 * lo + 1);
    const double border = b * b * (double)s, value = 4.0 * (double)x;
    c = (float)(value > border || (value == border && (lo & 1)) ? lo + 1 : lo);
  }
  return min((int)c, 127);
}

__device__ __forceinline__ int square_code(float x, float s, float inv) {
  const float r = approx_sqrt(approx_sqrt(x * inv));
  float c = rintf(r);
  if (fabsf(r - c) > kBorder) {
    const int lo = (int)floorf(r);
    double b = (double)(2 * lo + 1);
    b *= b;
    const double border = b * b * (double)s, value = 16.0 * (double)x;
    c = (float)(value > border || (value == border && (lo & 1)) ? lo + 1 : lo);
  }
  const int code = min((int)c, 255);
  return code == 0 && x > 0.0f && s > 0.0f ? 1 : code;
}

__device__ __forceinline__ float moment_value(int c, float s) { return (float)(c * abs(c)) * s; }
__device__ __forceinline__ float square_value(int c, float s) {
  const float d = (float)(c * c);
  return __fmul_rn(__fmul_rn(d, d), s);
}

// The step of one warp's block: p, g and the codes of this lane in registers (elements past the
// end hold g = 0 and codes 0, so they change no maximum). ms, vs: the block's scales, in and out.
__device__ __forceinline__ void step_block(float (&p)[8], const float (&g)[8], Codes& q, float& ms,
                                           float& vs, const Scalars& k, const Tensor& t) {
  float m[8], v[8];
  uint32_t mtop = 0, vtop = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float ge = k.maximize ? -g[e] : g[e];
    m[e] = __fadd_rn(__fmul_rn(moment_value(q.m[e], ms), k.b1), __fmul_rn(ge, k.w1));
    v[e] = __fadd_rn(__fmul_rn(square_value(q.v[e], vs), k.b2),
                     __fmul_rn(__fmul_rn(ge, ge), k.w2));
    mtop = max(mtop, __float_as_uint(fabsf(m[e])));
    vtop = max(vtop, __float_as_uint(v[e]));
    const float d = fmaf(approx_sqrt(v[e]), t.root, k.eps);
    p[e] = fmaf(-t.step_size, __fdividef(m[e], d), p[e] * t.decay);
  }
  ms = __fmul_rn(__uint_as_float(__reduce_max_sync(0xffffffffu, mtop)), kMomentScale);
  vs = __fmul_rn(__uint_as_float(__reduce_max_sync(0xffffffffu, vtop)), kSquareScale);
  ms = ms < kTiny ? 0.0f : ms;
  vs = vs < kTiny ? 0.0f : vs;
  const float mi = ms > 0.0f ? __fdividef(1.0f, ms) : 0.0f;
  const float vi = vs > 0.0f ? __fdividef(1.0f, vs) : 0.0f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int c = moment_code(fabsf(m[e]), ms, mi);
    q.m[e] = (int8_t)(m[e] < 0.0f ? -c : c);
    q.v[e] = (uint8_t)square_code(v[e], vs, vi);
  }
}

template <typename T> __device__ __forceinline__ void load8(const T* p, float (&f)[8]) {
  if constexpr (sizeof(T) == 4) {
    ld_global_v8(p, f);
  } else {
    unpack<T>(*reinterpret_cast<const uint4*>(p), f);
  }
}
template <typename T> __device__ __forceinline__ void store8(T* p, const float (&f)[8]) {
  if constexpr (sizeof(T) == 4) {
    st_global_v8(p, f);
  } else {
    *reinterpret_cast<uint4*>(p) = pack<T>(f);
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
adamw8_kernel(const __grid_constant__ Batch batch, Scalars k) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t items = batch.t[batch.count - 1].item_end;
  int i = 0;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    while (item >= batch.t[i].item_end) ++i;  // items are visited in increasing order
    const Tensor& t = batch.t[i];
    const int64_t first = i > 0 ? batch.t[i - 1].item_end : 0;
    T* P = static_cast<T*>(t.param);
    const T* G = static_cast<const T*>(t.grad);
    const uintptr_t wide = reinterpret_cast<uintptr_t>(P) | reinterpret_cast<uintptr_t>(G);
    const uintptr_t codes = reinterpret_cast<uintptr_t>(t.mc) | reinterpret_cast<uintptr_t>(t.vc);
    const bool aligned = wide % (8 * sizeof(T)) == 0 && codes % 8 == 0;
    const int64_t blocks = (t.numel + kBlock - 1) / kBlock;
    const int64_t b0 = (item - first) * kItemBlocks + warp;
    for (int j = 0; j < kWarpBlocks; ++j) {
      const int64_t b = b0 + j * (kThreads / 32);
      if (b >= blocks) break;
      float ms = t.ms[b], vs = t.vs[b];
      float p[8], g[8];
      Codes q;
      const int64_t at = b * kBlock;
      if (aligned && at + kBlock <= t.numel) {
        const int64_t o = at + lane * 8;
        load8<T>(P + o, p);
        load8<T>(G + o, g);
        const uint2 mc = *reinterpret_cast<const uint2*>(t.mc + o);
        const uint2 vc = *reinterpret_cast<const uint2*>(t.vc + o);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          q.m[e] = (int8_t)((e < 4 ? mc.x : mc.y) >> (8 * (e & 3)));
          q.v[e] = (uint8_t)((e < 4 ? vc.x : vc.y) >> (8 * (e & 3)));
        }
        step_block(p, g, q, ms, vs, k, t);
        store8<T>(P + o, p);
        uint2 mo = make_uint2(0, 0), vo = make_uint2(0, 0);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          (e < 4 ? mo.x : mo.y) |= (uint32_t)(uint8_t)q.m[e] << (8 * (e & 3));
          (e < 4 ? vo.x : vo.y) |= (uint32_t)q.v[e] << (8 * (e & 3));
        }
        *reinterpret_cast<uint2*>(t.mc + o) = mo;
        *reinterpret_cast<uint2*>(t.vc + o) = vo;
      } else {
        // A short last block, or arrays that are not aligned: lane strides of one element.
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int64_t o = at + e * 32 + lane;
          const bool in = o < t.numel;
          p[e] = in ? to_float(P[o]) : 0.0f;
          g[e] = in ? to_float(G[o]) : 0.0f;
          q.m[e] = in ? t.mc[o] : (int8_t)0;
          q.v[e] = in ? t.vc[o] : (uint8_t)0;
        }
        step_block(p, g, q, ms, vs, k, t);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int64_t o = at + e * 32 + lane;
          if (o < t.numel) {
            P[o] = from_float<T>(p[e]);
            t.mc[o] = q.m[e];
            t.vc[o] = q.v[e];
          }
        }
      }
      if (lane == 0) {
        t.ms[b] = ms;
        t.vs[b] = vs;
      }
    }
  }
}

// The fp32 moments that codes and scales stand for.
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
};

__global__ void __launch_bounds__(kThreads)
moments_kernel(const __grid_constant__ MomentBatch batch) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t items = batch.t[batch.count - 1].item_end;
  int i = 0;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    while (item >= batch.t[i].item_end) ++i;
    const MomentTensor& t = batch.t[i];
    const int64_t first = i > 0 ? batch.t[i - 1].item_end : 0;
    const bool aligned =
        (reinterpret_cast<uintptr_t>(t.mc) | reinterpret_cast<uintptr_t>(t.vc)) % 8 == 0 &&
        (reinterpret_cast<uintptr_t>(t.m) | reinterpret_cast<uintptr_t>(t.v)) % 32 == 0;
    const int64_t blocks = (t.numel + kBlock - 1) / kBlock;
    const int64_t b0 = (item - first) * kItemBlocks + warp;
#pragma unroll
    for (int j = 0; j < kWarpBlocks; ++j) {
      const int64_t b = b0 + j * (kThreads / 32);
      if (b >= blocks) break;
      const float ms = t.ms[b], vs = t.vs[b];
      const int64_t at = b * kBlock;
      if (aligned && at + kBlock <= t.numel) {
        const int64_t o = at + lane * 8;
        const uint2 mc = *reinterpret_cast<const uint2*>(t.mc + o);
        const uint2 vc = *reinterpret_cast<const uint2*>(t.vc + o);
        float m[8], v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          m[e] = moment_value((int8_t)((e < 4 ? mc.x : mc.y) >> (8 * (e & 3))), ms);
          v[e] = square_value((uint8_t)((e < 4 ? vc.x : vc.y) >> (8 * (e & 3))), vs);
        }
        st_global_v8(t.m + o, m);
        st_global_v8(t.v + o, v);
      } else {
        for (int64_t o = at + lane; o < min(at + kBlock, t.numel); o += 32) {
          t.m[o] = moment_value(t.mc[o], ms);
          t.v[o] = square_value(t.vc[o], vs);
        }
      }
    }
  }
}

int64_t items_of(int64_t numel) {
  const int64_t per = (int64_t)kItemBlocks * kBlock;
  return (numel + per - 1) / per;
}

int check_state(int i, int64_t numel, const int8_t* mc, const float* ms, const uint8_t* vc,
                const float* vs) {
  if (numel < 0) return set_error(PT_ERR_SHAPE, "tensor %d has a negative numel", i);
  if (numel == 0) return PT_OK;
  const char* what[4] = {"exp_avg codes", "exp_avg scales", "exp_avg_sq codes",
                         "exp_avg_sq scales"};
  const void* ptr[4] = {mc, ms, vc, vs};
  for (int k = 0; k < 4; ++k)
    if (int st = check_device_ptr(ptr[k], what[k])) return st;
  return PT_OK;
}

}  // namespace
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
  if (!(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0) || !(eps >= 0.0))
    return set_error(PT_ERR_INVALID_ARGUMENT, "betas must be in [0, 1) and eps >= 0");
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
  int sms = 0;
  if (int st = current_device_info(nullptr, &sms)) return st;
  const Scalars k{(float)beta1, (float)(1.0 - beta1), (float)beta2, (float)(1.0 - beta2),
                  (float)eps, maximize != 0};
  cudaStream_t s = as_stream(stream);
  for (int i = 0; i < num_tensors;) {
    Batch b;
    b.count = 0;
    int64_t items = 0;
    for (; i < num_tensors && b.count < kBatch; ++i) {
      if (numels[i] == 0) continue;
      items += items_of(numels[i]);
      const double bc1 = 1.0 - std::pow(beta1, (double)steps[i]);
      const double bc2 = 1.0 - std::pow(beta2, (double)steps[i]);
      b.t[b.count++] = Tensor{params[i], grads[i], exp_avg_codes[i], exp_avg_scales[i],
                              exp_avg_sq_codes[i], exp_avg_sq_scales[i], numels[i], items,
                              (float)(lrs[i] / bc1), (float)(1.0 / std::sqrt(bc2)),
                              (float)(1.0 - lrs[i] * weight_decays[i])};
    }
    if (b.count == 0) break;
    const int grid = (int)std::min<int64_t>(items, (int64_t)sms * (2048 / kThreads));
    switch (dtype) {
      case PT_FLOAT32: adamw8_kernel<float><<<grid, kThreads, 0, s>>>(b, k); break;
      case PT_FLOAT16: adamw8_kernel<__half><<<grid, kThreads, 0, s>>>(b, k); break;
      default: adamw8_kernel<__nv_bfloat16><<<grid, kThreads, 0, s>>>(b, k);
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
  for (int i = 0; i < num_tensors;) {
    MomentBatch b;
    b.count = 0;
    int64_t items = 0;
    for (; i < num_tensors && b.count < kBatch; ++i) {
      if (numels[i] == 0) continue;
      items += items_of(numels[i]);
      b.t[b.count++] = MomentTensor{exp_avg_codes[i], exp_avg_scales[i], exp_avg_sq_codes[i],
                                    exp_avg_sq_scales[i], exp_avgs[i], exp_avg_sqs[i],
                                    numels[i], items};
    }
    if (b.count == 0) break;
    const int grid = (int)std::min<int64_t>(items, (int64_t)sms * (2048 / kThreads));
    moments_kernel<<<grid, kThreads, 0, as_stream(stream)>>>(b);
    if (int st = check_launch("pt_adamw8_moments")) return st;
  }
  return ok();
}

}  // extern "C"
