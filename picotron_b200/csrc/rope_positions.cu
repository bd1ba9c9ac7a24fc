// Rotary embedding by explicit positions, forward and backward (sm_100a).
//
// Query and key [B, H, S, D] of one launch share positions [B, S] and R/2 frequencies (R the
// rotated part of the head, R <= D). The angle of pair i at token (b, s) is
//   a = positions[b, s] * inv_freq[i],
// formed in 64 bits and reduced to within half a turn there (a far position times a frequency
// has lost its fraction in 32 bits: at position 10^6 the product is off by 0.03 radian), so one
// single-precision sincospi of the rest follows: rounding the rest to fp32 moves it by at most
// 2^-25 pi radian, less than the two products and the sum of an output are rounded by. With
// c = scale cos a, s = scale sin a,
//   out_1 = x_1 c - x_2 s,  out_2 = x_1 s + x_2 c
// for the pairs (x[2i], x[2i+1]) (INTERLEAVED) or (x[i], x[i + R/2]) (ROTATE_HALF); x[R:] is
// copied. The backward is the transpose, the same with s negated. Each output is rounded once.
//
// A CTA takes a few whole tokens: all heads of q and k at a token share its R/2 angles, which
// are computed once into shared memory while the first loads are in flight. Tables of positions
// would be read per head or built by another launch; here only positions and frequencies are
// read next to q and k, and the kernel is bound by reading and writing those.
#include <algorithm>

#include "common.cuh"

namespace pt {
namespace {

// 128 threads (64 and 256 took 1.1 and 1.2 times as long at B 8, S 2048, 32 + 8 heads of 128,
// bf16: 54 us, 0.95 of the copy rate). Units in flight per thread: five where a token has that
// many, as there, else three (54 against 60 us there; 3.1 against 3.9 us for 32 decoded tokens).
constexpr int kThreads = 128;
constexpr int kManyUnits = 5;
constexpr int kFewUnits = 3;
constexpr int kTableBytes = 32 * 1024;         // of shared memory for a CTA's angles
constexpr int kMaxTokens = 16;                 // tokens per CTA

struct Geom {
  const void* x[2];
  void* out[2];
  int64_t xb[2], xh[2], xs[2], ob[2], oh[2], os[2];  // strides of B, H, S (elements)
  const int64_t* positions;
  int64_t pb, ps;
  const double* inv_freq;
  uint32_t heads0, heads;    // heads of tensor 0, of both
  uint32_t half;             // R / 2
  uint32_t head_units;       // units per head: rotated ones, then copied ones
  uint32_t rot_units;
  uint32_t token_units;      // heads * head_units
  uint32_t tokens_per_cta;
  uint32_t tokens;           // B * S
  FastDiv div_token, div_head, div_s, div_half;
  float scale, sign;
};

// The angles of `count` tokens from token0 on: (c, s) per pair, by all threads of the CTA.
__device__ __forceinline__ void fill_table(const Geom& g, float2* table, uint32_t token0,
                                           uint32_t count) {
  for (uint32_t i = threadIdx.x; i < count * g.half; i += kThreads) {
    const uint32_t tok = g.div_half.div(i), p = i - tok * g.half;
    const uint32_t b = g.div_s.div(token0 + tok), s = token0 + tok - b * g.div_s.d;
    const double a = (double)g.positions[b * g.pb + s * g.ps] * g.inv_freq[p];
    // a less whole turns, with 2 pi as a sum of two 64-bit numbers: exact to 64 bits for any a
    // whose turns are whole numbers in 64 bits, where a fraction of a / (2 pi) loses |a| 2^-53.
    const double turns = rint(a * 0.15915494309189535);
    const double rest = fma(-turns, 2.4492935982947064e-16, fma(-turns, 6.283185307179586, a));
    float sn, c;
    sincospif((float)(rest * 0.3183098861837907), &sn, &c);
    table[i] = make_float2(c * g.scale, g.sign * (sn * g.scale));
  }
}

// N consecutive elements of T moved as one access of N * sizeof(T) bytes, as fp32.
template <typename T, int N> struct Pack {
  static constexpr int kBytes = N * (int)sizeof(T);
  using Raw = std::conditional_t<
      kBytes == 16, uint4,
      std::conditional_t<kBytes == 8, uint2, std::conditional_t<kBytes == 4, uint32_t, uint16_t>>>;
  Raw raw;
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (kBytes == 16)
      raw = ld_stream(p);
    else
      raw = *reinterpret_cast<const Raw*>(p);
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (kBytes == 16)
      st_stream(p, raw);
    else
      *reinterpret_cast<Raw*>(p) = raw;
  }
  __device__ __forceinline__ void get(float* f) const {
    const T* e = reinterpret_cast<const T*>(&raw);
    if constexpr (kBytes == 16) {
      unpack<T>(raw, f);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = to_float(e[i]);
    }
  }
  __device__ __forceinline__ void set(const float* f) {
    if constexpr (kBytes == 16) {
      raw = pack<T>(f);
    } else {
      T e[N];
#pragma unroll
      for (int i = 0; i < N; ++i) e[i] = from_float<T>(f[i]);
      memcpy(&raw, e, kBytes);
    }
  }
};

// A unit is N elements (two single ones for N = 1 interleaved), or for rotated rotate-half
// units N elements of each half.
// kOne: a CTA takes one token, whose rows' addresses are the same for all its threads.
template <typename T, int N, bool kRotateHalf, bool kOne, int kUnits>
__global__ void __launch_bounds__(kThreads)
rope_positions_kernel(const __grid_constant__ Geom g) {
  extern __shared__ float2 table[];  // [tokens_per_cta][half] (c, s)
  constexpr bool kPairLoads = !kRotateHalf && N == 1;
  constexpr int kSpan = kPairLoads ? 2 : N;  // elements from one unit's start to the next
  const uint32_t token0 = kOne ? blockIdx.x : blockIdx.x * g.tokens_per_cta;
  const uint32_t count = kOne ? 1u : min(g.tokens_per_cta, g.tokens - token0);
  const uint32_t total = count * g.token_units;

  struct Token {
    const T* x[2];
    T* out[2];
  };
  auto token_at = [&](uint32_t tok) {
    const uint32_t b = g.div_s.div(token0 + tok), s = token0 + tok - b * g.div_s.d;
    Token t;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      t.x[i] = static_cast<const T*>(g.x[i]) + (int64_t)b * g.xb[i] + (int64_t)s * g.xs[i];
      t.out[i] = static_cast<T*>(g.out[i]) + (int64_t)b * g.ob[i] + (int64_t)s * g.os[i];
    }
    return t;
  };
  const Token one = kOne ? token_at(0) : Token{};

  struct Where {
    const T* x;
    T* out;
    uint32_t table;  // index of the unit's first pair
    bool rotated;
  };
  auto where = [&](uint32_t u) {
    uint32_t tok = 0, in = u;
    if (!kOne) {
      tok = g.div_token.div(u);
      in = u - tok * g.token_units;
    }
    const Token t = kOne ? one : token_at(tok);
    const uint32_t h = g.div_head.div(in);
    const uint32_t j = in - h * g.head_units;
    const bool second = h >= g.heads0;
    const int64_t hh = second ? h - g.heads0 : h;
    Where w;
    w.rotated = j < g.rot_units;
    // Copied units of a rotate-half head start behind both halves.
    const uint32_t d =
        kRotateHalf ? (w.rotated ? j * kSpan : 2 * g.half + (j - g.rot_units) * kSpan) : j * kSpan;
    w.x = (second ? t.x[1] + hh * g.xh[1] : t.x[0] + hh * g.xh[0]) + d;
    w.out = (second ? t.out[1] + hh * g.oh[1] : t.out[0] + hh * g.oh[0]) + d;
    w.table = tok * g.half + j * (kRotateHalf ? N : kSpan / 2);
    return w;
  };
  struct Data {
    Pack<T, N> a, b;
  };
  auto load = [&](const Where& w, Data& d) {
    d.a.load(w.x);
    if constexpr (kRotateHalf) {
      if (w.rotated) d.b.load(w.x + g.half);
    } else if constexpr (kPairLoads) {
      d.b.load(w.x + 1);
    }
  };
  auto finish = [&](const Where& w, Data& d) {
    if (w.rotated) {
      if constexpr (kRotateHalf || kPairLoads) {
        float e[N], o[N];
        d.a.get(e);
        d.b.get(o);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float2 cs = table[w.table + i];
          const float r = fmaf(e[i], cs.x, -(o[i] * cs.y));
          o[i] = fmaf(e[i], cs.y, o[i] * cs.x);
          e[i] = r;
        }
        d.a.set(e);
        d.b.set(o);
      } else {
        float f[N];
        d.a.get(f);
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
          const float2 cs = table[w.table + i];
          const float r = fmaf(f[2 * i], cs.x, -(f[2 * i + 1] * cs.y));
          f[2 * i + 1] = fmaf(f[2 * i], cs.y, f[2 * i + 1] * cs.x);
          f[2 * i] = r;
        }
        d.a.set(f);
      }
    }
    d.a.store(w.out);
    if constexpr (kRotateHalf) {
      if (w.rotated) d.b.store(w.out + g.half);
    } else if constexpr (kPairLoads) {
      d.b.store(w.out + 1);
    }
  };

  Where w[kUnits];
  Data d[kUnits];
#pragma unroll
  for (int k = 0; k < kUnits; ++k) {
    const uint32_t u = threadIdx.x + k * kThreads;
    if (u < total) {
      w[k] = where(u);
      load(w[k], d[k]);
    }
  }
  fill_table(g, table, token0, count);
  __syncthreads();
  for (uint32_t u0 = threadIdx.x; u0 < total; u0 += kThreads * kUnits) {
    if (u0 != threadIdx.x) {
#pragma unroll
      for (int k = 0; k < kUnits; ++k) {
        const uint32_t u = u0 + k * kThreads;
        if (u < total) {
          w[k] = where(u);
          load(w[k], d[k]);
        }
      }
    }
#pragma unroll
    for (int k = 0; k < kUnits; ++k)
      if (u0 + k * kThreads < total) finish(w[k], d[k]);
  }
}

// Rows path, for heads whose rows are not made of whole 16-byte vectors (head_dim 78 or 226 in
// bf16, a boundary or a half at an odd place): where the heads of a token lie behind one
// another, the token's row of heads x head_dim elements is one run of memory. It goes through
// shared memory in 16-byte vectors, whatever its start, and the pairs are rotated there, one per
// thread. The path above moves such heads in 8 to 2 bytes at a time and is bound by the address
// arithmetic of each: for 16384 tokens of 20 + 5 heads of 78 (66 rotated) in bf16 it took 64
// (interleaved) and 78 us (rotate-half), this one 46; for 10 + 5 heads of 226 107 and 115 us, this
// one 86; for 14 + 2 heads of 96 (40 rotated, rotate-half) 35 us, this one 31. What bounds it now is
// the instruction issue of the pairs. In fp32 the two take equally long, and the other is used.
struct RowGeom {
  uint32_t n[2];       // elements of a row: heads * head_dim
  uint32_t vecs[2];    // vectors that a row touches, at most
  uint32_t slot[2];    // where a token's rows start in shared memory (bytes)
  uint32_t token_bytes;
  uint32_t dim;
  uint32_t step_pairs, step_heads;  // kThreads pairs on: so many whole heads and pairs
  FastDiv div_vecs, div_pairs;  // by the vectors and by the pairs (of all heads) of one token
};

template <typename T, bool kRotateHalf>
__global__ void __launch_bounds__(kThreads)
rope_rows_positions_kernel(const __grid_constant__ Geom g, const __grid_constant__ RowGeom rg) {
  constexpr int V = Vec16<T>::N;
  constexpr int kLoads = 4;
  struct Row {
    const T* x;
    T* out;
    T* held;     // the row's first element in shared memory
    int before;  // elements of its first vector that lie before it
  };
  extern __shared__ __align__(16) unsigned char shared[];
  __shared__ Row rows[kMaxTokens * 2];
  float2* table = reinterpret_cast<float2*>(shared + g.tokens_per_cta * rg.token_bytes);
  const uint32_t token0 = blockIdx.x * g.tokens_per_cta;
  const uint32_t count = min(g.tokens_per_cta, g.tokens - token0);
  if (threadIdx.x < 2 * count) {
    const uint32_t tok = threadIdx.x >> 1, i = threadIdx.x & 1;
    const uint32_t b = g.div_s.div(token0 + tok), s = token0 + tok - b * g.div_s.d;
    Row r;
    r.x = static_cast<const T*>(g.x[i]) + (int64_t)b * g.xb[i] + (int64_t)s * g.xs[i];
    r.out = static_cast<T*>(g.out[i]) + (int64_t)b * g.ob[i] + (int64_t)s * g.os[i];
    r.before = (int)((reinterpret_cast<uintptr_t>(r.x) & 15u) / sizeof(T));
    r.held = reinterpret_cast<T*>(shared + tok * rg.token_bytes + rg.slot[i]) + r.before;
    rows[threadIdx.x] = r;
  }
  __syncthreads();

  // Vector u of the CTA's rows: its row and first element; whole vectors only are moved as such.
  auto whole = [&](uint32_t u, uint32_t& row, int& first) {
    const uint32_t tok = rg.div_vecs.div(u);
    const uint32_t in = u - tok * rg.div_vecs.d, i = in >= rg.vecs[0] ? 1 : 0;
    row = 2 * tok + i;
    first = (int)(in - (i ? rg.vecs[0] : 0)) * V - rows[row].before;
    return first >= 0 && first + V <= (int)rg.n[i];
  };
  // The elements of a row before its first whole vector and behind its last, one per thread:
  // `move` gets the row and the element.
  auto edges = [&](auto move) {
    for (uint32_t q = threadIdx.x; q < 2 * count * 2 * V; q += kThreads) {
      const Row& r = rows[q / (2 * V)];
      const int n = (int)rg.n[(q / (2 * V)) & 1], e = (int)(q % (2 * V));
      const int head = min(n, (V - r.before) % V), tail = (n - head) % V;
      if (e < head)
        move(r, e);
      else if (e >= V && e - V < tail)
        move(r, n - tail + e - V);
    }
  };

  const uint32_t vecs = count * rg.div_vecs.d;
  for (uint32_t u0 = threadIdx.x; u0 < vecs; u0 += kThreads * kLoads) {
    uint4 raw[kLoads];
    T* at[kLoads];
#pragma unroll
    for (int k = 0; k < kLoads; ++k) {
      uint32_t row;
      int first;
      at[k] = nullptr;
      if (u0 + k * kThreads < vecs && whole(u0 + k * kThreads, row, first)) {
        at[k] = rows[row].held + first;
        raw[k] = ld_stream(rows[row].x + first);
      }
    }
#pragma unroll
    for (int k = 0; k < kLoads; ++k)
      if (at[k] != nullptr) *reinterpret_cast<uint4*>(at[k]) = raw[k];
  }
  edges([](const Row& r, int e) { r.held[e] = r.x[e]; });
  fill_table(g, table, token0, count);
  __syncthreads();
  // Pair u = (token, head, pair of the head); the next one of a thread is kThreads further on.
  const uint32_t pairs = count * rg.div_pairs.d;
  uint32_t tok = rg.div_pairs.div(threadIdx.x);
  uint32_t h = g.div_half.div(threadIdx.x - tok * rg.div_pairs.d);
  uint32_t j = threadIdx.x - tok * rg.div_pairs.d - h * g.half;
#pragma unroll 2
  for (uint32_t u = threadIdx.x; u < pairs; u += kThreads) {
    const uint32_t i = h >= g.heads0 ? 1 : 0;
    T* a = rows[2 * tok + i].held + (h - (i ? g.heads0 : 0)) * rg.dim + (kRotateHalf ? j : 2 * j);
    T* b = a + (kRotateHalf ? g.half : 1);
    const float2 cs = table[tok * g.half + j];
    const float x = to_float(*a), y = to_float(*b);
    *a = from_float<T>(fmaf(x, cs.x, -(y * cs.y)));
    *b = from_float<T>(fmaf(x, cs.y, y * cs.x));
    j += rg.step_pairs;
    h += rg.step_heads;
    if (j >= g.half) {
      j -= g.half;
      ++h;
    }
    while (h >= g.heads) {
      h -= g.heads;
      ++tok;
    }
  }
  __syncthreads();
#pragma unroll 4
  for (uint32_t u = threadIdx.x; u < vecs; u += kThreads) {
    uint32_t row;
    int first;
    if (whole(u, row, first)) st_stream(rows[row].out + first, lds128(rows[row].held + first));
  }
  edges([](const Row& r, int e) { r.out[e] = r.held[e]; });
}

struct Side {
  const void* x;
  const int64_t* xst;
  void* out;
  const int64_t* ost;
  const int64_t* sizes;
};

// Whether accesses of n elements fit every row: the offsets of both tensors' heads, the
// boundary of the rotated part and the heads' ends all fall on multiples of n elements.
bool fits(const Side* sides, int64_t D, int64_t R, int n, int elem, bool rh) {
  if (D % n || (rh ? R / 2 : R) % n) return false;
  for (int i = 0; i < 2; ++i) {
    const Side& t = sides[i];
    if (t.sizes[0] * t.sizes[1] * t.sizes[2] == 0) continue;
    if (reinterpret_cast<uintptr_t>(t.x) % (n * elem) ||
        reinterpret_cast<uintptr_t>(t.out) % (n * elem))
      return false;
    for (int a = 0; a < 3; ++a)
      if (t.sizes[a] > 1 && (t.xst[a] % n || t.ost[a] % n)) return false;
  }
  return true;
}

template <typename T, int N>
int launch(Geom& g, int64_t D, int64_t R, bool rh, cudaStream_t s) {
  const int span = !rh && N == 1 ? 2 : N;
  g.half = (uint32_t)(R / 2);
  g.rot_units = (uint32_t)(rh ? R / 2 / N : R / span);
  const int64_t copied = (D - R) / span;
  const int64_t units = (int64_t)g.heads * (g.rot_units + copied);
  if (units > (int64_t)UINT32_MAX / (2 * kMaxTokens))
    return set_error(PT_ERR_SHAPE, "too many heads times head_dim for one token");
  g.head_units = (uint32_t)(g.rot_units + copied);
  g.token_units = (uint32_t)units;
  // Enough tokens per CTA to give every thread its units in flight, as far as the angles fit.
  const int64_t want = std::max<int64_t>(1, kThreads * kFewUnits / units);
  const int64_t room = std::max<int64_t>(1, kTableBytes / ((int64_t)g.half * 8));
  g.tokens_per_cta = (uint32_t)std::min<int64_t>({want, room, kMaxTokens, (int64_t)g.tokens});
  g.div_token = FastDiv(g.token_units);
  g.div_head = FastDiv(g.head_units);
  g.div_half = FastDiv(g.half);
  const unsigned grid = (g.tokens + g.tokens_per_cta - 1) / g.tokens_per_cta;
  const size_t smem = (size_t)g.tokens_per_cta * g.half * sizeof(float2);
  auto kernel = rh ? rope_positions_kernel<T, N, true, false, kFewUnits>
                   : rope_positions_kernel<T, N, false, false, kFewUnits>;
  if (g.tokens_per_cta == 1) {
    if (units > kThreads * kFewUnits)
      kernel = rh ? rope_positions_kernel<T, N, true, true, kManyUnits>
                  : rope_positions_kernel<T, N, false, true, kManyUnits>;
    else
      kernel = rh ? rope_positions_kernel<T, N, true, true, kFewUnits>
                  : rope_positions_kernel<T, N, false, true, kFewUnits>;
  }
  kernel<<<grid, kThreads, smem, s>>>(g);
  return check_launch("pt_rope_positions");
}

// Whether the rows path can take the call: the heads of a token behind one another in inputs and
// outputs, whose rows start at the same place of a 16-byte vector, and one token's rows in kRowBytes.
constexpr int64_t kRowBytes = 40 * 1024;
template <typename T> bool make_rows(RowGeom& rg, const Side* sides, int64_t D, int64_t R) {
  constexpr int elem = (int)sizeof(T);
  int64_t at = 0;
  for (int i = 0; i < 2; ++i) {
    const Side& t = sides[i];
    const int64_t H = t.sizes[1];
    if (H > 0) {
      if (H > 1 && (t.xst[1] != D || t.ost[1] != D)) return false;
      if ((reinterpret_cast<uintptr_t>(t.x) - reinterpret_cast<uintptr_t>(t.out)) % 16) return false;
      for (int a : {0, 2})
        if (t.sizes[a] > 1 && (t.xst[a] - t.ost[a]) * elem % 16) return false;
    }
    if (H > kRowBytes || H * D * elem > kRowBytes) return false;
    rg.n[i] = (uint32_t)(H * D);
    rg.vecs[i] = H > 0 ? (uint32_t)((H * D * elem + 15) / 16 + 1) : 0;
    rg.slot[i] = (uint32_t)at;
    at += (int64_t)rg.vecs[i] * 16;
  }
  if (at + R / 2 * 8 > kRowBytes) return false;
  rg.token_bytes = (uint32_t)at;
  rg.dim = (uint32_t)D;
  rg.div_vecs = FastDiv(rg.vecs[0] + rg.vecs[1]);
  return true;
}

template <typename T>
int launch_rows(Geom& g, RowGeom& rg, int64_t R, bool rh, cudaStream_t s) {
  g.half = (uint32_t)(R / 2);
  g.div_half = FastDiv(g.half);
  rg.div_pairs = FastDiv(g.heads * g.half);
  rg.step_pairs = kThreads % g.half;
  rg.step_heads = kThreads / g.half;
  // Tokens for four vectors a thread, as far as 16 KB (or one token) hold them.
  const int64_t bytes = rg.token_bytes + (int64_t)g.half * 8;
  const int64_t want = kThreads * 4 / rg.div_vecs.d;
  const int64_t room = 16 * 1024 / bytes;
  g.tokens_per_cta = (uint32_t)std::max<int64_t>(
      1, std::min<int64_t>({want, room, kMaxTokens, (int64_t)g.tokens}));
  const unsigned grid = (g.tokens + g.tokens_per_cta - 1) / g.tokens_per_cta;
  const size_t smem = (size_t)(g.tokens_per_cta * bytes);
  if (rh)
    rope_rows_positions_kernel<T, true><<<grid, kThreads, smem, s>>>(g, rg);
  else
    rope_rows_positions_kernel<T, false><<<grid, kThreads, smem, s>>>(g, rg);
  return check_launch("pt_rope_positions");
}

// The widest access that fits: 16 bytes, rows through shared memory (16-bit types), 8 or 4 bytes,
// else single elements.
template <typename T>
int dispatch(Geom& g, const Side* sides, int64_t D, int64_t R, bool rh, cudaStream_t s) {
  constexpr int elem = (int)sizeof(T);
  constexpr int kWide = 16 / elem;
  if (fits(sides, D, R, kWide, elem, rh)) return launch<T, kWide>(g, D, R, rh, s);
  [[maybe_unused]] RowGeom rg;
  if constexpr (elem == 2)
    if (make_rows<T>(rg, sides, D, R)) return launch_rows<T>(g, rg, R, rh, s);
  if (fits(sides, D, R, kWide / 2, elem, rh)) return launch<T, kWide / 2>(g, D, R, rh, s);
  if constexpr (elem == 2) {
    if (fits(sides, D, R, 2, elem, rh)) return launch<T, 2>(g, D, R, rh, s);
  }
  return launch<T, 1>(g, D, R, rh, s);
}

}  // namespace
}  // namespace pt

using namespace pt;

extern "C" {

int pt_rope_positions(const void* q, const int64_t q_strides[4], void* q_out,
                      const int64_t q_out_strides[4], const int64_t q_sizes[4], const void* k,
                      const int64_t k_strides[4], void* k_out, const int64_t k_out_strides[4],
                      const int64_t k_sizes[4], const int64_t* positions,
                      int64_t position_batch_stride, int64_t position_stride,
                      const double* inv_freq, int64_t rotary_dim, double scale, int backward,
                      int layout, int dtype, void* stream) {
  if (layout != PT_ROPE_INTERLEAVED && layout != PT_ROPE_ROTATE_HALF)
    return set_error(PT_ERR_INVALID_ARGUMENT, "unknown layout %d", layout);
  const int elem = dtype_size(dtype);
  if (elem == 0) return set_error(PT_ERR_UNSUPPORTED_DTYPE, "unsupported dtype %d", dtype);
  const Side sides[2] = {{q, q_strides, q_out, q_out_strides, q_sizes},
                         {k, k_strides, k_out, k_out_strides, k_sizes}};
  for (const Side& t : sides) {
    if (!t.xst || !t.ost || !t.sizes)
      return set_error(PT_ERR_INVALID_ARGUMENT, "strides and sizes must not be NULL");
    for (int a = 0; a < 4; ++a)
      if (t.sizes[a] < 0 || t.xst[a] < 0 || t.ost[a] < 0)
        return set_error(PT_ERR_SHAPE, "negative size or stride");
    if (t.xst[3] != 1 || t.ost[3] != 1)
      return set_error(PT_ERR_SHAPE, "the head_dim stride must be 1");
    if (t.sizes[0] > INT32_MAX || t.sizes[1] > INT32_MAX || t.sizes[2] > INT32_MAX)
      return set_error(PT_ERR_SHAPE, "sizes must be below 2^31");
  }
  const int64_t B = q_sizes[0], S = q_sizes[2], D = q_sizes[3];
  if (k_sizes[0] != B || k_sizes[2] != S || k_sizes[3] != D)
    return set_error(PT_ERR_SHAPE, "query and key must share batch, sequence and head_dim");
  if (D < 1 || D > 65536 || rotary_dim < 2 || rotary_dim % 2 != 0 || rotary_dim > D ||
      rotary_dim > 8192)
    return set_error(PT_ERR_SHAPE, "rotary_dim must be even, from 2 to min(head_dim, 8192) (got "
                                   "%lld of %lld)",
                     (long long)rotary_dim, (long long)D);
  if (layout == PT_ROPE_INTERLEAVED && D % 2 != 0)
    return set_error(PT_ERR_SHAPE, "head_dim must be even for interleaved pairs");
  if (position_batch_stride < 0 || position_stride < 0)
    return set_error(PT_ERR_SHAPE, "negative position stride");
  if (B * S == 0 || q_sizes[1] + k_sizes[1] == 0) return ok();
  if (B * S > INT32_MAX || q_sizes[1] + k_sizes[1] > INT32_MAX)
    return set_error(PT_ERR_SHAPE, "B * S and the heads together must be below 2^31");
  for (const Side& t : sides) {
    if (t.sizes[1] == 0) continue;
    if (int st = check_device_ptr(t.x, "x")) return st;
    if (int st = check_device_ptr(t.out, "out")) return st;
    if ((reinterpret_cast<uintptr_t>(t.x) | reinterpret_cast<uintptr_t>(t.out)) % elem)
      return set_error(PT_ERR_INVALID_ARGUMENT, "tensors must be aligned to their element size");
  }
  if (int st = check_device_ptr(positions, "positions")) return st;
  if (int st = check_device_ptr(inv_freq, "inv_freq")) return st;
  Geom g;
  for (int i = 0; i < 2; ++i) {
    const Side& t = sides[i];
    g.x[i] = t.x;
    g.out[i] = t.out;
    g.xb[i] = t.xst[0];
    g.xh[i] = t.xst[1];
    g.xs[i] = t.xst[2];
    g.ob[i] = t.ost[0];
    g.oh[i] = t.ost[1];
    g.os[i] = t.ost[2];
  }
  g.positions = positions;
  g.pb = position_batch_stride;
  g.ps = position_stride;
  g.inv_freq = inv_freq;
  g.heads0 = (uint32_t)q_sizes[1];
  g.heads = (uint32_t)(q_sizes[1] + k_sizes[1]);
  g.tokens = (uint32_t)(B * S);
  g.div_s = FastDiv((uint32_t)S);
  g.scale = (float)scale;
  g.sign = backward ? -1.0f : 1.0f;
  const bool rh = layout == PT_ROPE_ROTATE_HALF;
  cudaStream_t s = as_stream(stream);
  switch (dtype) {
    case PT_FLOAT32: return dispatch<float>(g, sides, D, rotary_dim, rh, s);
    case PT_FLOAT16: return dispatch<__half>(g, sides, D, rotary_dim, rh, s);
    default: return dispatch<__nv_bfloat16>(g, sides, D, rotary_dim, rh, s);
  }
}

}  // extern "C"
