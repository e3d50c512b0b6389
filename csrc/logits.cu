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
// reads the words beside them.  Every CTA needs every id of the row: a long history is read once
// per cluster, each CTA bringing its share into shared memory and reading the others' through
// the cluster.  A thread's first logits are loaded before the table is built.
#include "common.cuh"
#include "serving.h"

#include <cooperative_groups.h>
#include <cuda_fp16.h>

namespace cg = cooperative_groups;

namespace pra {
namespace rules {

#ifndef NTT
#define NTT 512
#endif
#ifndef LB
#define LB 2
#endif
constexpr int NT = NTT;
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

__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if either is
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
  return m;
}

constexpr int STAGE = 2048;   // ids of a long history that a CTA holds for its cluster at a time
#ifndef DIR
#define DIR 2048
#endif
constexpr int DIRECT = DIR;  // up to here every CTA reads the whole history itself

// T: type of the logits; V: elements of one access; TABLE: a history or biases are given.
template <typename T, int V, bool TABLE>
__global__ void __launch_bounds__(NT, LB) rules_kernel(const LogitsArgs a, int slice) {
  #ifndef UU
#define UU 2
#endif
  constexpr int U = V == 1 ? 4 : UU;  // accesses of a thread in flight
  extern __shared__ uint4 smem_raw[];
  uint32_t* smem = reinterpret_cast<uint32_t*>(smem_raw);
  __shared__ unsigned long long s_best[NT / 32];
  __shared__ unsigned long long s_cluster;  // this CTA's best, read by the cluster's first CTA
  cg::cluster_group cluster = cg::this_cluster();
  const int parts = cluster.num_blocks(), part = cluster.block_rank();
  const int b = blockIdx.y;
  const int v0 = part * slice, n = max(min(a.V, v0 + slice) - v0, 0);
  const T* x = reinterpret_cast<const T*>(a.logits) + (int64_t)b * a.in_stride + v0;
  T* y = a.out ? reinterpret_cast<T*>(a.out) + (int64_t)b * a.out_stride + v0 : nullptr;
  const int vecs = n / V;
  Vec<T, V> in[U];
  auto load = [&](int i0) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i0 + u * NT < vecs) in[u] = *reinterpret_cast<const Vec<T, V>*>(x + (i0 + u * NT) * V);
  };
  load(threadIdx.x);

  uint32_t* words = smem;                                              // [slice]
  int* stage = reinterpret_cast<int*>(smem + (TABLE ? slice : 0));     // [STAGE], long histories only
  const int len = a.ids ? max(0, min(a.hist_len[b], a.capacity)) : 0;
  const bool staged = a.capacity > DIRECT;  // the same for the whole cluster
  int* bias_id = stage + (staged ? STAGE : 0);                         // [n_bias]
  float* bias_sum = reinterpret_cast<float*>(bias_id + a.n_bias);      // [n_bias]
  const float rep = a.repetition ? a.repetition[b] : 1.f;
  const float pres = a.presence ? a.presence[b] : 0.f;
  const float freq = a.frequency ? a.frequency[b] : 0.f;
  if constexpr (TABLE) {
    const int prompt = a.prompt_len ? a.prompt_len[b] : 0;
    const int* ids = a.ids + (int64_t)b * a.ids_stride;
    const uint32_t base = (uint32_t)a.vocab_start + (uint32_t)v0;
    uint4* w4 = reinterpret_cast<uint4*>(words);
    for (int i = threadIdx.x; i < slice / 4; i += NT) w4[i] = make_uint4(0, 0, 0, 0);
    for (int i = threadIdx.x; i < a.n_bias; i += NT) bias_id[i] = a.bias_ids[(int64_t)b * a.n_bias + i];
    auto count = [&](int id, int i) {
      const uint32_t t = (uint32_t)id - base;
      if (t >= (uint32_t)n) return;
      if (i < prompt) atomicOr(words + t, SEEN);
      else atomicAdd(words + t, 1u);
    };
    if (!staged) {
      __syncthreads();
#pragma unroll 4
      for (int i = threadIdx.x; i < len; i += NT) count(ids[i], i);
    } else {
      for (int i0 = 0; i0 < len; i0 += parts * STAGE) {
        // CTA p of the cluster brings in ids [i0 + p * per, i0 + (p + 1) * per)
        const int per = (min(len - i0, parts * STAGE) + parts - 1) / parts;
        const int lo = i0 + part * per, mine = max(0, min(per, len - lo));
#pragma unroll 4
        for (int i = threadIdx.x; i < mine; i += NT) stage[i] = ids[lo + i];
        cluster.sync();
        for (int q = 0; q < parts; ++q) {
          const int p = (part + q) % parts;  // each CTA begins with its own: not all read one at once
          const int* other = cluster.map_shared_rank(stage, p);
          const int first = i0 + p * per, there = max(0, min(per, len - first));
#pragma unroll 4
          for (int i = threadIdx.x; i < there; i += NT) count(other[i], first + i);
        }
        cluster.sync();  // the stage is refilled, or its CTA goes on
      }
    }
    __syncthreads();  // the counts are whole before the bias entries join their words
    // an entry whose id no earlier entry has owns the token and sums all its entries in list order
    for (int i = threadIdx.x; i < a.n_bias; i += NT) {
      const uint32_t t = (uint32_t)bias_id[i] - base;
      if (t >= (uint32_t)n) continue;
      bool first = true;
      for (int j = 0; j < i && first; ++j) first = bias_id[j] != bias_id[i];
      if (!first) continue;
      float sum = 0.f;
      for (int j = i; j < a.n_bias; ++j)
        if (bias_id[j] == bias_id[i]) sum += a.bias_values[(int64_t)b * a.n_bias + j];
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
  const bool choose = a.token != nullptr;
  float best = -INFINITY;  // largest so far, and its element: strictly larger ones replace it, in ascending order
  int best_e = 0;
  // The rules on V logits at element e of the slice.
  auto apply = [&](Vec<T, V> raw, int e) {
    float z[V];
#pragma unroll
    for (int j = 0; j < V; ++j) z[j] = widen(raw.v[j]);
    bool changed = false;
    if constexpr (TABLE) {
      const Vec<uint32_t, V> w = *reinterpret_cast<const Vec<uint32_t, V>*>(words + e);
      uint32_t any = 0;
#pragma unroll
      for (int j = 0; j < V; ++j) any |= w.v[j];
      if (any) {
        changed = true;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          if (w.v[j] & (SEEN | COUNT)) z[j] = z[j] > 0.f ? __fdiv_rn(z[j], rep) : __fmul_rn(z[j], rep);
          const uint32_t times = w.v[j] & COUNT;
          if (times) z[j] = __fsub_rn(__fsub_rn(z[j], __fmul_rn(freq, (float)times)), pres);
          if (w.v[j] >> 21) z[j] = __fadd_rn(z[j], bias_sum[(w.v[j] >> 21) - 1]);
        }
      }
    }
    uint32_t bits = none ? 0u : 0xFFFFFFFFu;
    if (mask) bits = mask[e / 8] >> (e & 7);
    if ((~bits & ((1u << V) - 1)) != 0) {
      changed = true;
#pragma unroll
      for (int j = 0; j < V; ++j) z[j] = (bits >> j) & 1u ? z[j] : -INFINITY;
    }
    if (choose) {
      float m = z[0];
#pragma unroll
      for (int j = 1; j < V; ++j) m = max_nan(m, z[j]);
      if (!(m <= best) && best == best) {
#pragma unroll
        for (int j = V - 1; j >= 0; --j)
          if (z[j] == m || (m != m && z[j] != z[j])) best_e = e + j;
        best = m;
      }
    }
    if (y) {
      if (changed) {
#pragma unroll
        for (int j = 0; j < V; ++j) narrow(z[j], raw.v[j]);
      }
      *reinterpret_cast<Vec<T, V>*>(y + e) = raw;
    }
  };
  for (int i0 = threadIdx.x; i0 < vecs; i0 += U * NT) {
    if (i0 != (int)threadIdx.x) load(i0);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i0 + u * NT < vecs) apply(in[u], (i0 + u * NT) * V);
  }
  unsigned long long key = choice_key(best, (uint32_t)(a.vocab_start + v0 + best_e));
  for (int e = vecs * V + threadIdx.x; e < n; e += NT) {  // fewer than V elements at the end of the last slice
    float z = widen(x[e]);
    if constexpr (TABLE) {
      const uint32_t w = words[e], times = w & COUNT;
      if (w & (SEEN | COUNT)) z = z > 0.f ? __fdiv_rn(z, rep) : __fmul_rn(z, rep);
      if (times) z = __fsub_rn(__fsub_rn(z, __fmul_rn(freq, (float)times)), pres);
      if (w >> 21) z = __fadd_rn(z, bias_sum[(w >> 21) - 1]);
    }
    if (none || (mask && !(mask[e / 8] >> (e & 7) & 1))) z = -INFINITY;
    const unsigned long long k = choice_key(z, (uint32_t)(a.vocab_start + v0 + e));
    key = k > key ? k : key;
    if (y) narrow(z, y[e]);
  }
  if (choose) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long other = __shfl_xor_sync(0xffffffffu, key, o);
      key = other > key ? other : key;
    }
    if ((threadIdx.x & 31) == 0) s_best[threadIdx.x >> 5] = key;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 1; w < NT / 32; ++w) key = s_best[w] > key ? s_best[w] : key;
      s_cluster = key;
    }
    cluster.sync();
    if (part == 0 && threadIdx.x < 32) {
      unsigned long long other = (int)threadIdx.x < parts ? *cluster.map_shared_rank(&s_cluster, (int)threadIdx.x) : 0;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const unsigned long long k = __shfl_xor_sync(0xffffffffu, other, o);
        other = k > other ? k : other;
      }
      if (threadIdx.x == 0) {
        const uint32_t k = (uint32_t)(other >> 32);
        const float z = k == 0xFFFFFFFFu ? __int_as_float(0x7fffffff) : __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
        const int64_t id = 0xFFFFFFFFu - (uint32_t)other;
        const bool any = z != -INFINITY;
        a.token[b] = any ? id : -1;
        if (a.value) a.value[b] = z;
        if (a.append_ids && any && len < a.capacity) {  // every CTA of the row has read its length by now
          a.append_ids[(int64_t)b * a.ids_stride + len] = (int)id;
          a.hist_len[b] = len + 1;
        }
      }
    }
    cluster.sync();  // the other CTAs' shared memory lives until it has been read
  }
}

template <typename T, int V, bool TABLE>
cudaError_t launch(const LogitsArgs& a, cudaStream_t st) {
  const int cl = 8;
  const int slice = ((a.V + cl - 1) / cl + 15) / 16 * 16;
  const size_t bytes = TABLE ? (size_t)slice * 4 + (a.capacity > DIRECT ? STAGE * 4 : 0) + (size_t)a.n_bias * 8 : 0;
  auto kernel = rules_kernel<T, V, TABLE>;
  if (bytes > 48 * 1024) PRA_RETURN_IF_ERROR(pra::set_max_dynamic_smem(reinterpret_cast<const void*>(kernel), (int)bytes));
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
