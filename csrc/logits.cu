// Rules on logits: penalties for repeated tokens, sparse biases, grammar bit masks; written back, or
// reduced to the greedy token.
//
// For the logit x of token t in a row whose history holds t (prompt or output), whose output part
// holds it n times, with bias entries for t summing to b:
//     z = x > 0 ? x / r : x * r          (seen)
//     z = (z - f * n) - p                (n > 0)
//     z = z + b                          (biased)
//     z = -inf                           (mask bit 0)
// every step rounded to fp32 in this order (no contraction), so a choice by the largest z does not
// depend on the compiler.  The greedy token is the lowest id of the largest z; NaN counts as the
// largest; a row with nothing above -inf gives -1.
//
// Bound by bytes: each logit is read once (and written once), the history read once.  A cluster of
// CL CTAs owns a row, one slice of the vocabulary each.  The history cannot be looked up per logit,
// so it is turned around: a 32-bit word per token of the slice in shared memory counts its
// occurrences (bits 0-19 output count, bit 20 seen, bits 21-31 bias entry + 1), filled by
// shared-memory atomics (integer: any order gives the same counts), and the pass over the logits
// reads the words beside them.
#include "common.cuh"
#include "serving.h"

#include <cooperative_groups.h>
#include <cuda_fp16.h>

namespace cg = cooperative_groups;

namespace pra {
namespace rules {

constexpr int NT = 512;
constexpr uint32_t COUNT = (1u << 20) - 1, SEEN = 1u << 20;

__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float widen(__half v) { return __half2float(v); }
__device__ __forceinline__ void narrow(float v, float& o) { o = v; }
__device__ __forceinline__ void narrow(float v, __nv_bfloat16& o) { o = __float2bfloat16(v); }
__device__ __forceinline__ void narrow(float v, __half& o) { o = __float2half_rn(v); }

// Larger key = better choice: the value's order (NaN above all, -0 as +0), then the lower id.
__device__ __forceinline__ unsigned long long choice_key(float z, uint32_t id) {
  const uint32_t u = __float_as_uint(__fadd_rn(z, 0.f));
  const uint32_t k = z != z ? 0xFFFFFFFFu : (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return ((unsigned long long)k << 32) | (0xFFFFFFFFu - id);
}

template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
  T v[V];
};

// T: type of the logits; V: elements of one access; TABLE: a history or biases are given.
template <typename T, int V, bool TABLE>
__global__ void __launch_bounds__(NT) rules_kernel(const LogitsArgs a, int slice) {
  extern __shared__ uint32_t smem[];
  __shared__ unsigned long long s_best[NT / 32];
  __shared__ unsigned long long s_cluster;  // this CTA's best, read by the cluster's first CTA
  cg::cluster_group cluster = cg::this_cluster();
  const int parts = cluster.num_blocks(), part = cluster.block_rank();
  const int b = blockIdx.y;
  const int v0 = part * slice, v1 = min(a.V, v0 + slice), n = max(v1 - v0, 0);
  uint32_t* words = smem;                                              // [slice]
  int* bias_id = reinterpret_cast<int*>(smem + (TABLE ? slice : 0));   // [n_bias]
  float* bias_sum = reinterpret_cast<float*>(bias_id + a.n_bias);      // [n_bias]
  const float rep = a.repetition ? a.repetition[b] : 1.f;
  const float pres = a.presence ? a.presence[b] : 0.f;
  const float freq = a.frequency ? a.frequency[b] : 0.f;
  const int len = a.ids ? max(0, min(a.hist_len[b], a.capacity)) : 0;
  if constexpr (TABLE) {
    uint4* w4 = reinterpret_cast<uint4*>(words);
    for (int i = threadIdx.x; i < slice / 4; i += NT) w4[i] = make_uint4(0, 0, 0, 0);
    for (int i = threadIdx.x; i < a.n_bias; i += NT) {
      bias_id[i] = a.bias_ids[(int64_t)b * a.n_bias + i] - a.vocab_start - v0;
    }
    __syncthreads();
    const int prompt = a.prompt_len ? a.prompt_len[b] : 0;
    const int* ids = a.ids + (int64_t)b * a.ids_stride;
    for (int i = threadIdx.x; i < len; i += NT) {
      const int64_t t = (int64_t)ids[i] - a.vocab_start - v0;
      if (t < 0 || t >= n) continue;
      if (i < prompt) atomicOr(words + t, SEEN);
      else atomicAdd(words + t, 1u);
    }
    __syncthreads();  // the counts are whole before the bias entries join their words
    // an entry whose id no earlier entry has owns the token and sums all its entries in list order
    for (int i = threadIdx.x; i < a.n_bias; i += NT) {
      const int t = bias_id[i];
      if (t < 0 || t >= n) continue;
      bool first = true;
      for (int j = 0; j < i && first; ++j) first = bias_id[j] != t;
      if (!first) continue;
      float sum = 0.f;
      for (int j = i; j < a.n_bias; ++j)
        if (bias_id[j] == t) sum += a.bias_values[(int64_t)b * a.n_bias + j];
      bias_sum[i] = sum;
      atomicOr(words + t, (uint32_t)(i + 1) << 21);
    }
    __syncthreads();
  }
  // the row's mask as bytes: element e of the slice is bit (vocab_start + v0 + e) % 8 of its byte
  const uint8_t* mask = nullptr;
  bool none = false;  // a mask row outside the masks allows nothing
  if (a.mask) {
    const int r = a.mask_rows ? a.mask_rows[b] : b;
    none = r >= a.mask_count;
    if (r >= 0 && !none)
      mask = reinterpret_cast<const uint8_t*>(a.mask + r * a.mask_words) + (a.vocab_start + v0) / 8;
  }
  const T* x = reinterpret_cast<const T*>(a.logits) + (int64_t)b * a.in_stride + v0;
  T* y = a.out ? reinterpret_cast<T*>(a.out) + (int64_t)b * a.out_stride + v0 : nullptr;
  unsigned long long best = 0;
  auto rule = [&](float z, int e, uint32_t w, bool allowed) {
    if (TABLE && w != 0) {
      if (w & (SEEN | COUNT)) z = z > 0.f ? __fdiv_rn(z, rep) : __fmul_rn(z, rep);
      const uint32_t count = w & COUNT;
      if (count) z = __fsub_rn(__fsub_rn(z, __fmul_rn(freq, (float)count)), pres);
      if (w >> 21) z = __fadd_rn(z, bias_sum[(w >> 21) - 1]);
    }
    if (!allowed) z = -INFINITY;
    if (a.token) {
      const unsigned long long k = choice_key(z, (uint32_t)(a.vocab_start + v0 + e));
      best = k > best ? k : best;
    }
    return z;
  };
  const int vecs = n / V;
  for (int i = threadIdx.x; i < vecs; i += NT) {
    const int e = i * V;
    Vec<T, V> in = *reinterpret_cast<const Vec<T, V>*>(x + e);
    uint32_t bits = none ? 0u : 0xFFu;
    if (mask) bits = mask[e / 8] >> (e & 7);
#pragma unroll
    for (int j = 0; j < V; ++j)
      narrow(rule(widen(in.v[j]), e + j, TABLE ? words[e + j] : 0u, (bits >> j) & 1u), in.v[j]);
    if (y) *reinterpret_cast<Vec<T, V>*>(y + e) = in;
  }
  for (int e = vecs * V + threadIdx.x; e < n; e += NT) {
    const bool allowed = !none && (!mask || (mask[e / 8] >> (e & 7) & 1));
    T o;
    narrow(rule(widen(x[e]), e, TABLE ? words[e] : 0u, allowed), o);
    if (y) y[e] = o;
  }
  if (a.token) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long other = __shfl_xor_sync(0xffffffffu, best, o);
      best = other > best ? other : best;
    }
    if ((threadIdx.x & 31) == 0) s_best[threadIdx.x >> 5] = best;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 1; w < NT / 32; ++w) best = s_best[w] > best ? s_best[w] : best;
      s_cluster = best;
    }
    cluster.sync();
    if (part == 0 && threadIdx.x == 0) {
      for (int p = 1; p < parts; ++p) {
        const unsigned long long other = *cluster.map_shared_rank(&s_cluster, p);
        best = other > best ? other : best;
      }
      const uint32_t k = (uint32_t)(best >> 32);
      const float z = k == 0xFFFFFFFFu ? __int_as_float(0x7fffffff) : __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
      const int64_t id = 0xFFFFFFFFu - (uint32_t)best;
      const bool any = z != -INFINITY;
      a.token[b] = any ? id : -1;
      if (a.value) a.value[b] = z;
      if (a.append_ids && any && len < a.capacity) {  // every CTA of the row has read its length by now
        a.append_ids[(int64_t)b * a.ids_stride + len] = (int)id;
        a.hist_len[b] = len + 1;
      }
    }
    cluster.sync();  // the other CTAs' shared memory lives until it has been read
  }
}

template <typename T, int V, bool TABLE>
cudaError_t launch(const LogitsArgs& a, cudaStream_t st) {
  const int cl = 8;
  const int slice = ((a.V + cl - 1) / cl + 15) / 16 * 16;
  const size_t bytes = TABLE ? (size_t)slice * 4 + (size_t)a.n_bias * 8 : 0;
  if (bytes > 220 * 1024) return cudaErrorInvalidValue;
  auto kernel = rules_kernel<T, V, TABLE>;
  if (bytes > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 220 * 1024);
    if (e != cudaSuccess) return e;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(cl, a.B);
  cfg.blockDim = dim3(NT);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cl;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, a, slice);
}

template <typename T>
cudaError_t dispatch(const LogitsArgs& a, cudaStream_t st) {
  constexpr int W = 16 / sizeof(T);
  bool wide = reinterpret_cast<uintptr_t>(a.logits) % 16 == 0 && a.in_stride % W == 0;
  if (a.out) wide = wide && reinterpret_cast<uintptr_t>(a.out) % 16 == 0 && a.out_stride % W == 0;
  const bool table = a.ids != nullptr || a.bias_ids != nullptr;
  if (wide) return table ? launch<T, W, true>(a, st) : launch<T, W, false>(a, st);
  return table ? launch<T, 1, true>(a, st) : launch<T, 1, false>(a, st);
}

}  // namespace rules
}  // namespace pra

cudaError_t pra_logits_rules(const LogitsArgs& a, int dtype, cudaStream_t st) {
  if (a.B == 0 || a.V == 0) return cudaSuccess;
  switch (dtype) {
    case PRA_BF16: return pra::rules::dispatch<__nv_bfloat16>(a, st);
    case PRA_FP16: return pra::rules::dispatch<__half>(a, st);
    case PRA_FP32: return pra::rules::dispatch<float>(a, st);
    default: return cudaErrorInvalidValue;
  }
}
