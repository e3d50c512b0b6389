// Rotary positions for queries and keys, forward and backward, in one launch.
//
// Pair i of a head is (x[i], x[i + R/2]) in the half layout and (x[2i], x[2i + 1]) in the
// interleaved one, for i < R/2 with R the rotated part of the head; with c, s the table's cosine
// and sine of (position, i)
//     y0 = x0 c - x1 s,    y1 = x1 c + x0 s,
// and the elements behind R pass through.  The map is linear and a table entry may carry a scale
// (m cos, m sin), so its transpose, the backward pass, is the same kernel with -s.  Products and
// sums are fp32 with one rounding to the output type.
//
// Bound by bytes: x is read once and y written once, the table adds 4 R bytes per token.  A thread owns
// one unit (two vectors of V elements, 16 bytes each where possible) of one token and walks the heads
// with it, so a unit's cosines and sines are read once for several heads and two heads' loads are in
// flight together.  Vectors need R and D - R to be multiples of 2 V and aligned rows; other calls take
// V = 2 or 1.  64 registers: at 122 (four heads in flight, chosen among segments per head) the prefill
// case of 16,384 tokens (407 MB) took 138 us, now 72 us, 5.7 TB/s.
#include "common.cuh"
#include "serving.h"

#include <cuda_fp16.h>

namespace pra {
namespace rotary {

constexpr int NT = 256;
constexpr int64_t L2_BYTES = 126 << 20;

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f(float v) { return v; }
template <>
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16(v); }
template <>
__device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }

template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
  T v[V];
};

// Loads and stores of a call that passes through more than the L2 holds are marked as used once: its
// outputs would evict one another before anyone reads them (prefill case 79.9 -> 73.8 us, a smaller
// call keeps its outputs in L2 for the attention that follows).
template <bool STREAM, typename X>
__device__ __forceinline__ X load(const void* p) {
  if constexpr (STREAM && sizeof(X) == 16) {
    const uint4 v = __ldcs(reinterpret_cast<const uint4*>(p));
    return *reinterpret_cast<const X*>(&v);
  } else {
    return *reinterpret_cast<const X*>(p);
  }
}
template <bool STREAM, typename X>
__device__ __forceinline__ void store(void* p, const X& x) {
  if constexpr (STREAM && sizeof(X) == 16) __stcs(reinterpret_cast<uint4*>(p), *reinterpret_cast<const uint4*>(&x));
  else *reinterpret_cast<X*>(p) = x;
}

template <typename T, int V, bool STREAM>
__global__ void __launch_bounds__(NT, 4) rotary_kernel(const RotaryArgs a, int units, int unit_lanes, int head_lanes,
                                                       int tokens_per_block) {
  const int per = unit_lanes * head_lanes;
  const int lt = threadIdx.x / per;
  const int64_t m = (int64_t)blockIdx.x * tokens_per_block + lt;
  if (lt >= tokens_per_block || m >= a.tokens) return;
  const int rem = threadIdx.x - lt * per;
  const int hl = rem / unit_lanes;
  const int half = a.rot / 2, rot_units = half / V;
  const int64_t pos = a.pos64 ? reinterpret_cast<const int64_t*>(a.pos)[m] : reinterpret_cast<const int*>(a.pos)[m];
  const bool pos_ok = pos >= 0 && pos < a.max_pos;  // outside the table: the rotated part becomes NaN
  int64_t slot = m;
  if (a.slots != nullptr) slot = a.slots[m];
  const bool slot_ok = a.slots == nullptr || (slot >= 0 && slot < a.slot_rows);
  for (int u = rem - hl * unit_lanes; u < units; u += unit_lanes) {
    const bool turns = u < rot_units;
    // the unit's two vectors, the rotated part's (or the rest's) halves apart, so that neighbouring
    // threads touch neighbouring bytes in both layouts; single elements of the interleaved one side by side
    int o0, o1, c0, c1;  // their offsets, and those of the cosines of their first pairs
    if (!turns) {
      o0 = a.rot + (u - rot_units) * V;
      o1 = o0 + (a.head_dim - a.rot) / 2;
    } else if (a.interleaved && V == 1) {
      o0 = u * 2;
      o1 = o0 + 1;
    } else {
      o0 = u * V;
      o1 = half + u * V;
    }
    constexpr int F = V < 4 ? (V > 1 ? V / 2 : 1) : V / 2 < 4 ? V / 2 : 4;  // floats of a table access
    c0 = a.interleaved && V > 1 ? o0 / 2 : u * V;
    c1 = a.interleaved && V > 1 ? o1 / 2 : u * V + V / 2;
    float c[V], s[V];
    if (turns) {
      const int64_t row = (pos_ok ? pos : 0) * half;
#pragma unroll
      for (int j = 0; j < V; j += F) {
        const int64_t at = row + (j < V / 2 || V == 1 ? c0 + j : c1 + j - V / 2);
        const Vec<float, F> cv = *reinterpret_cast<const Vec<float, F>*>(a.cos_t + at);
        const Vec<float, F> sv = *reinterpret_cast<const Vec<float, F>*>(a.sin_t + at);
#pragma unroll
        for (int i = 0; i < F; ++i) {
          c[j + i] = pos_ok ? cv.v[i] : __int_as_float(0x7fffffff);
          s[j + i] = pos_ok ? (a.inverse ? -sv.v[i] : sv.v[i]) : __int_as_float(0x7fffffff);
        }
      }
    }
#pragma unroll
    for (int g = 0; g < 3; ++g) {
      const RotarySegment& q = a.seg[g];
      if (q.heads == 0 || (q.to_slot && !slot_ok)) continue;
      const bool rotate = turns && q.rotate;
      const T* src = reinterpret_cast<const T*>(q.src) + m * q.src_token;
      T* dst = reinterpret_cast<T*>(q.dst) + (q.to_slot ? slot : m) * q.dst_token;
#pragma unroll 2
      for (int h = hl; h < q.heads; h += head_lanes) {
        Vec<T, V> x0 = load<STREAM, Vec<T, V>>(src + h * q.src_head + o0);
        Vec<T, V> x1 = load<STREAM, Vec<T, V>>(src + h * q.src_head + o1);
        if (rotate) {
          if (a.interleaved && V > 1) {  // pair i of each vector is its elements (2i, 2i + 1)
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
              const float p0 = to_f(x0.v[2 * i]), p1 = to_f(x0.v[2 * i + 1 < V ? 2 * i + 1 : 0]);
              const float q0 = to_f(x1.v[2 * i]), q1 = to_f(x1.v[2 * i + 1 < V ? 2 * i + 1 : 0]);
              x0.v[2 * i] = from_f<T>(p0 * c[i] - p1 * s[i]);
              x0.v[2 * i + 1 < V ? 2 * i + 1 : 0] = from_f<T>(p1 * c[i] + p0 * s[i]);
              x1.v[2 * i] = from_f<T>(q0 * c[V / 2 + i] - q1 * s[V / 2 + i]);
              x1.v[2 * i + 1 < V ? 2 * i + 1 : 0] = from_f<T>(q1 * c[V / 2 + i] + q0 * s[V / 2 + i]);
            }
          } else {
#pragma unroll
            for (int i = 0; i < V; ++i) {
              const float p0 = to_f(x0.v[i]), p1 = to_f(x1.v[i]);
              x0.v[i] = from_f<T>(p0 * c[i] - p1 * s[i]);
              x1.v[i] = from_f<T>(p1 * c[i] + p0 * s[i]);
            }
          }
        }
        store<STREAM>(dst + h * q.dst_head + o0, x0);
        store<STREAM>(dst + h * q.dst_head + o1, x1);
      }
    }
  }
}

template <typename T, int V>
cudaError_t launch(const RotaryArgs& a, cudaStream_t st) {
  const int heads = std::max(a.seg[0].heads, std::max(a.seg[1].heads, a.seg[2].heads));
  const int units = a.head_dim / (2 * V);
  const int unit_lanes = std::min(units, NT);
  // one head of the widest segment per thread spreads a small call over more threads; eight share
  // a unit's cosines and sines
  const bool small = a.tokens * (int64_t)units * heads < (int64_t)148 * 2048 * 4;
  const int hpt = small ? 1 : 8;
  const int head_lanes = std::max(1, std::min((heads + hpt - 1) / hpt, NT / unit_lanes));
  const int tpb = std::max(1, NT / (unit_lanes * head_lanes));
  const int64_t blocks = (a.tokens + tpb - 1) / tpb;
  if (blocks > INT32_MAX) return cudaErrorInvalidValue;
  const int64_t bytes = 2 * (int64_t)sizeof(T) * a.tokens * a.head_dim * (a.seg[0].heads + a.seg[1].heads + a.seg[2].heads);
  if (bytes > L2_BYTES)
    rotary_kernel<T, V, true><<<(unsigned)blocks, NT, 0, st>>>(a, units, unit_lanes, head_lanes, tpb);
  else
    rotary_kernel<T, V, false><<<(unsigned)blocks, NT, 0, st>>>(a, units, unit_lanes, head_lanes, tpb);
  return cudaGetLastError();
}

// The widest vector that the rotated part, the rest of the head and every row's alignment allow.
template <typename T, int V>
bool fits(const RotaryArgs& a) {
  if (a.rot % (2 * V) || (a.head_dim - a.rot) % (2 * V)) return false;
  const uintptr_t bytes = V * sizeof(T), table = std::min(V, 4) * 4;
  if (reinterpret_cast<uintptr_t>(a.cos_t) % table || reinterpret_cast<uintptr_t>(a.sin_t) % table) return false;
  for (const RotarySegment& s : a.seg) {
    if (s.heads == 0) continue;
    if (reinterpret_cast<uintptr_t>(s.src) % bytes || reinterpret_cast<uintptr_t>(s.dst) % bytes) return false;
    if (s.src_token % V || s.src_head % V || s.dst_token % V || s.dst_head % V) return false;
  }
  return true;
}

template <typename T>
cudaError_t dispatch(const RotaryArgs& a, cudaStream_t st) {
  constexpr int W = 16 / sizeof(T);
  if (fits<T, W>(a)) return launch<T, W>(a, st);
  if (fits<T, 2>(a)) return launch<T, 2>(a, st);
  return launch<T, 1>(a, st);
}

}  // namespace rotary
}  // namespace pra

cudaError_t pra_rotary(const RotaryArgs& a, int dtype, cudaStream_t st) {
  if (a.tokens == 0) return cudaSuccess;
  switch (dtype) {
    case PRA_BF16: return pra::rotary::dispatch<__nv_bfloat16>(a, st);
    case PRA_FP16: return pra::rotary::dispatch<__half>(a, st);
    case PRA_FP32: return pra::rotary::dispatch<float>(a, st);
    default: return cudaErrorInvalidValue;
  }
}
