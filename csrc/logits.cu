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
// Each logit is read once (and written once), the history by each CTA of its row, once or twice.  A
// cluster of 1 to 8 CTAs owns a row, one slice of the vocabulary each.  The history cannot be looked up
// per logit, so each CTA turns its slice of it around in shared memory: a bit per token that the history or a
// bias names (their ranks by a prefix sum of the bits), and for each such token its id and a word with
// its occurrences (bits 0-19 output count, bit 20 seen, bits 21-31 2,047 less its first bias entry, or
// 0).  Integer atomics fill them, so any order gives the same table; a token's first bias entry sums all
// of its entries (looking for earlier ones from each entry took 203 us for 2,047 biases, now 21).
//
// The pass over all logits then takes maxima on packed 16-bit pairs, and masks and leaves out what is
// named only where a vector may hold a new largest; the named tokens follow, four logits on their way per
// thread (half of the warps at them while the others are at all logits: no shorter).  Where the history
// may name half of a slice, a word per token takes no more room and the history is walked once instead
// of twice (64 rows of 128,256 logits with 100,000 ids each: 368 -> 136 us).  256 rows of 152,064 bf16
// logits with 8,192 ids each take 41 us (16 without a history, 13.9 is what their bytes need; written back
// 69, 29 and 25.8), one row of 128,256 with 512 ids 10.4, with 16,384 23.5: the two walks and the scattered
// logits of the named tokens wait for memory, one after the other.  (Looking the penalties up within the
// pass over all logits took 107 us, a word per token of the slice instead of the table 183 us.)  A thread
// only remembers which vector held its maximum: the element is looked up at the end, by the warps' winners.
// A thread's first logits and mask bytes are loaded before the table is built.
#include <algorithm>
#include <type_traits>

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

// The value of a key's upper half.
__device__ __forceinline__ float key_value(uint32_t k) {
  if (k == 0xFFFFFFFFu) return __int_as_float(0x7fffffff);
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
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

// All ones where bit j of `bits` is set, else 0.
__device__ __forceinline__ uint32_t spread(uint32_t bits, int j) {
  uint32_t m;
  asm("bfe.s32 %0, %1, %2, 1;" : "=r"(m) : "r"(bits), "r"(j));
  return m;
}

// -inf where the element's bit is 0.
template <int V>
__device__ __forceinline__ void mask_vec(Vec<float, V>& x, uint32_t bits) {
#pragma unroll
  for (int j = 0; j < V; ++j) x.v[j] = (bits >> j) & 1u ? x.v[j] : -INFINITY;
}
template <typename T, int V>
__device__ __forceinline__ void mask_vec(Vec<T, V>& x, uint32_t bits) {
  constexpr uint32_t NEG = sizeof(T) == 2 && std::is_same<T, __half>::value ? 0xFC00FC00u : 0xFF80FF80u;
  if constexpr (V == 1) {
    if (!(bits & 1u)) narrow(-INFINITY, x.v[0]);
  } else {
    uint32_t* w = reinterpret_cast<uint32_t*>(&x);
#pragma unroll
    for (int j = 0; j < V / 2; ++j) {
      const uint32_t m = __byte_perm(spread(bits, 2 * j), spread(bits, 2 * j + 1), 0x5410);
      w[j] = (w[j] & m) | (NEG & ~m);
    }
  }
}

// The largest element (NaN if one is).
template <int V>
__device__ __forceinline__ float max_vec(const Vec<float, V>& x) {
  float m = x.v[0];
#pragma unroll
  for (int j = 1; j < V; ++j) m = max_nan(m, x.v[j]);
  return m;
}
__device__ __forceinline__ __nv_bfloat162 max_pair(__nv_bfloat162 a, __nv_bfloat162 b) { return __hmax2_nan(a, b); }
__device__ __forceinline__ __half2 max_pair(__half2 a, __half2 b) { return __hmax2_nan(a, b); }
template <typename T, int V>
__device__ __forceinline__ float max_vec(const Vec<T, V>& x) {
  if constexpr (V == 1) {
    return widen(x.v[0]);
  } else {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    const T2* w = reinterpret_cast<const T2*>(&x);
    T2 m = w[0];
#pragma unroll
    for (int j = 1; j < V / 2; ++j) m = max_pair(m, w[j]);
    return max_nan(widen(m.x), widen(m.y));
  }
}

// 32-bit words of a slice's bits.
__host__ __device__ constexpr int bit_words(int slice) { return (slice + 31) / 32; }

// T: type of the logits; V: elements of one access; TABLE: a history or biases are given; CHOOSE: the
// greedy token is wanted, else the processed logits; PEEL: rows may begin at any element (vectors then
// start at the first aligned one, and their mask bits straddle bytes).
template <typename T, int V, bool TABLE, bool CHOOSE, bool PEEL>
__global__ void __launch_bounds__(NT, 2) rules_kernel(const LogitsArgs a, int slice, int table_words, bool direct) {
  constexpr int U = 3;  // accesses of a batch
  extern __shared__ uint32_t smem[];
  __shared__ uint32_t s_scan[NT / 32];
  __shared__ unsigned long long s_best[NT / 32];
  __shared__ unsigned long long s_cluster;  // this CTA's best, read by the cluster's first CTA
  cg::cluster_group cluster = cg::this_cluster();
  const int parts = cluster.num_blocks(), part = cluster.block_rank();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int b = blockIdx.y;
  const int v0 = part * slice, n = max(min(a.V, v0 + slice) - v0, 0);
  const T* x = reinterpret_cast<const T*>(a.logits) + (int64_t)b * a.in_stride + v0;
  T* y = CHOOSE ? nullptr : reinterpret_cast<T*>(a.out) + (int64_t)b * a.out_stride + v0;
  // the row's mask as bytes: element e of the slice is bit (vocab_start + v0 + e) % 8 of its byte
  const uint8_t* mask = nullptr;
  bool none = false;  // a mask row outside the masks allows nothing
  if (a.mask_words > 0) {  // (an empty set of masks has no address)
    const int r = a.mask_rows ? a.mask_rows[b] : b;
    none = r >= a.mask_count;
    if (r >= 0 && !none)
      mask = reinterpret_cast<const uint8_t*>(a.mask + r * a.mask_words) + (a.vocab_start + v0) / 8;
  }
  // elements in front of the first aligned vector (rows of an odd length begin anywhere), then vectors
  const int head = !PEEL ? 0 : min(n, (int)((0 - reinterpret_cast<uintptr_t>(x)) / sizeof(T) % V));
  const int vecs = (n - head) / V;
  // mask bits of the V elements from e, and named ones
  auto mask_bits = [&](int e) {
    const int s = e & 7;
    uint32_t bits = mask[e >> 3] >> s;
    if constexpr (PEEL) bits |= (uint32_t)mask[(e + V - 1) >> 3] << 8 >> s;  // the same byte again does no harm
    return bits;
  };
  struct Batch {
    Vec<T, V> x[U];
    uint32_t allowed[U];
  } here, next;  // one being worked on, one on its way
  auto load = [&](Batch& q, int i0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * NT;
      q.allowed[u] = none ? 0u : 0xFFu;
      if (i < vecs) {
        q.x[u] = *reinterpret_cast<const Vec<T, V>*>(x + head + i * V);
        if (mask) q.allowed[u] = mask_bits(head + i * V);
      }
    }
  };
  load(here, tid);

  uint32_t* named = smem;                                       // [bit_words(slice)] tokens with a table word
  uint32_t* rank = named + bit_words(slice);                    // [bit_words(slice)] table words before
  uint32_t* table = rank + bit_words(slice);                    // [table_words]
  uint32_t* token = table + table_words;                        // [table_words] their elements of the slice
  int* bias_id = reinterpret_cast<int*>(direct ? token : token + table_words);  // [n_bias] (direct: word t is token t's)
  float* bias_sum = reinterpret_cast<float*>(bias_id + a.n_bias);
  const int len = a.ids ? max(0, min(a.hist_len[b], a.capacity)) : 0;
  const float rep = a.repetition ? a.repetition[b] : 1.f;
  const float pres = a.presence ? a.presence[b] : 0.f;
  const float freq = a.frequency ? a.frequency[b] : 0.f;
  auto entry_of = [&](uint32_t t) { return rank[t >> 5] + __popc(named[t >> 5] & ((1u << (t & 31)) - 1u)); };
  int named_tokens = 0;
  if constexpr (TABLE) {
    const int prompt = a.prompt_len ? a.prompt_len[b] : 0;
    const int* ids = a.ids + (int64_t)b * a.ids_stride;
    const uint32_t base = (uint32_t)a.vocab_start + (uint32_t)v0;
    const int words = bit_words(slice);
    for (int i = tid; i < words; i += NT) named[i] = 0;
    for (int i = tid; i < table_words; i += NT) table[i] = 0;
    for (int i = tid; i < a.n_bias; i += NT) {
      bias_id[i] = a.bias_ids[(int64_t)b * a.n_bias + i];
      bias_sum[i] = 0.f;
    }
    __syncthreads();
    auto name = [&](int id) {
      const uint32_t t = (uint32_t)id - base, bit = 1u << (t & 31);
      if (t < (uint32_t)n && !(named[t >> 5] & bit)) atomicOr(named + (t >> 5), bit);
    };
    // every id of the row, four to a load where the row is aligned (the second walk finds them in L1)
    const bool quads = (reinterpret_cast<uintptr_t>(ids) & 15) == 0;
    auto walk = [&](auto visit) {
      int done = 0;
      if (quads) {
        done = len & ~3;
#pragma unroll 2
        for (int i = tid * 4; i < done; i += NT * 4) {
          const int4 q = *reinterpret_cast<const int4*>(ids + i);
          visit(q.x, i);
          visit(q.y, i + 1);
          visit(q.z, i + 2);
          visit(q.w, i + 3);
        }
      }
#pragma unroll 4
      for (int i = done + tid; i < len; i += NT) visit(ids[i], i);
    };
    if (!direct) {
      walk([&](int id, int) { name(id); });
      for (int i = tid; i < a.n_bias; i += NT) name(bias_id[i]);
      __syncthreads();
      // exclusive prefix sum of the words' bit counts, each thread a run of words
      const int per = (words + NT - 1) / NT, first = min(tid * per, words), last = min(first + per, words);
      uint32_t mine = 0;
      for (int i = first; i < last; ++i) mine += __popc(named[i]);
      uint32_t upto = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
      }
      if (lane == 31) s_scan[warp] = upto;
      __syncthreads();
      uint32_t at = upto - mine;
      for (int w = 0; w < warp; ++w) at += s_scan[w];
      for (int i = first; i < last; ++i) {
        rank[i] = at;
        at += __popc(named[i]);
      }
      for (int w = 0; w < NT / 32; ++w) named_tokens += s_scan[w];
      __syncthreads();
    }
    auto place = [&](uint32_t t) { return direct ? t : entry_of(t); };
    // the table words of biased tokens, before anything else is in them: the smallest entry wins
    for (int i = tid; i < a.n_bias; i += NT) {
      const uint32_t t = (uint32_t)bias_id[i] - base;
      if (t >= (uint32_t)n) continue;
      if (!direct) token[place(t)] = t;
      atomicMax(table + place(t), (uint32_t)(PRA_RULES_MAX_BIASES - i) << 21);
    }
    if (a.n_bias > 0) __syncthreads();
    walk([&](int id, int i) {
      const uint32_t t = (uint32_t)id - base;
      if (t >= (uint32_t)n) return;
      const uint32_t at = place(t);
      if (!direct) token[at] = t;  // every occurrence writes the same
      if (i >= prompt) atomicAdd(table + at, 1u);
      else if (!(table[at] & SEEN)) atomicOr(table + at, SEEN);
    });
    // a token's first entry owns it and sums all its entries in list order
    if (a.n_bias > 0) {
      for (int i = tid; i < a.n_bias; i += NT) {
        const uint32_t t = (uint32_t)bias_id[i] - base;
        if (t >= (uint32_t)n) continue;
        const int first = PRA_RULES_MAX_BIASES - (int)(table[place(t)] >> 21);
        if (first != i) bias_sum[first] = 1.f;  // there are more of it
      }
      __syncthreads();
      const float* values = a.bias_values + (int64_t)b * a.n_bias;
      for (int i0 = warp * 32; i0 < a.n_bias; i0 += NT) {
        const int i = i0 + lane;
        const uint32_t t = i < a.n_bias ? (uint32_t)bias_id[i] - base : 0xFFFFFFFFu;
        const bool owns = t < (uint32_t)n && PRA_RULES_MAX_BIASES - (int)(table[place(t)] >> 21) == i;
        float sum = owns ? 0.f + values[i] : 0.f;
        // the warp looks for the other entries of one token after the other
        for (uint32_t more = __ballot_sync(0xffffffffu, owns && bias_sum[i] != 0.f); more; more &= more - 1) {
          const int of = __ffs(more) - 1, id = bias_id[i0 + of];
          for (int c = i0; c < a.n_bias; c += 32) {
            const int j = c + lane;
            uint32_t found = __ballot_sync(0xffffffffu, j > i0 + of && j < a.n_bias && bias_id[j] == id);
            for (; found; found &= found - 1) {
              const float v = values[c + __ffs(found) - 1];
              if (lane == of) sum += v;
            }
          }
        }
        if (owns) bias_sum[i] = sum;
      }
    }
    __syncthreads();
    if (direct) {
      for (int i = warp; i < words; i += NT / 32) {
        const uint32_t bits = __ballot_sync(0xffffffffu, table[i * 32 + lane] != 0);
        if (lane == 0) named[i] = bits;
      }
      named_tokens = n;
      __syncthreads();
    }
  }
  // The bits of the vector's elements that this pass chooses among: allowed, and not named.
  auto choosable = [&](uint32_t bits, int e) {
    if constexpr (TABLE && PEEL) bits &= ~__funnelshift_r(named[e >> 5], named[(e + V - 1) >> 5], e & 31);
    else if constexpr (TABLE) bits &= ~(named[e >> 5] >> (e & 31));
    return bits;
  };
  unsigned long long key = 0;
  if constexpr (CHOOSE) {
    // Most vectors hold nothing above the largest that the warp has found: they are only compared, masks
    // and names are looked up for the others.  A warp's tokens come in rising order, so an equal one later
    // never wins.
    float best = -INFINITY, bar = -INFINITY;  // this thread's largest (vector best_i), the warp's
    int best_i = 0;
    auto look = [&](Batch& q, int i0) {
      float m[U];
      bool above = false;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        m[u] = max_vec(q.x[u]);
        above = above || (i0 + u * NT < vecs && !(m[u] <= bar));
      }
      if (!__any_sync(0xffffffffu, above && bar == bar)) return;  // NaN: nothing is larger
      float least = bar;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u * NT;
        if (i >= vecs || m[u] <= least || least != least) continue;
        mask_vec(q.x[u], choosable(q.allowed[u], head + i * V));
        const float k = max_vec(q.x[u]);
        if (k <= least) continue;
        best = least = k;
        best_i = i;
      }
      bar = key_value(__reduce_max_sync(0xffffffffu, (uint32_t)(choice_key(best, 0) >> 32)));
    };
    for (int i0 = tid; i0 - lane < vecs; i0 += 2 * U * NT) {
      load(next, i0 + U * NT);
      look(here, i0);
      load(here, i0 + 2 * U * NT);
      look(next, i0 + U * NT);
    }
    // the lanes that have the warp's largest value look for their element
    const uint32_t mine = (uint32_t)(choice_key(best, 0) >> 32);
    if (mine == __reduce_max_sync(0xffffffffu, mine) && best_i < vecs) {
      const int e = head + best_i * V;
      Vec<T, V> raw = *reinterpret_cast<const Vec<T, V>*>(x + e);
      uint32_t bits = none ? 0u : 0xFFu;
      if (mask) bits = mask_bits(e);
      mask_vec(raw, choosable(bits, e));
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const unsigned long long k = choice_key(widen(raw.v[j]), (uint32_t)(a.vocab_start + v0 + e + j));
        key = k > key ? k : key;
      }
    }
  } else {
    auto apply = [&](Batch& q, int i0) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u * NT;
        if (i >= vecs) continue;
        if (mask || none) mask_vec(q.x[u], q.allowed[u]);
        *reinterpret_cast<Vec<T, V>*>(y + head + i * V) = q.x[u];
      }
    };
    for (int i0 = tid; i0 < vecs; i0 += 2 * U * NT) {
      load(next, i0 + U * NT);
      apply(here, i0);
      load(here, i0 + 2 * U * NT);
      apply(next, i0 + U * NT);
    }
  }
  auto is_allowed = [&](int e) { return !none && (!mask || (mask[e / 8] >> (e & 7) & 1)); };
  // fewer than V elements in front of the vectors and behind them
  for (int r = tid; r < n - vecs * V; r += NT) {
    const int e = r < head ? r : r + vecs * V;
    if (TABLE && ((named[e >> 5] >> (e & 31)) & 1u)) continue;
    const float z = is_allowed(e) ? widen(x[e]) : -INFINITY;
    if constexpr (CHOOSE) {
      const unsigned long long k = choice_key(z, (uint32_t)(a.vocab_start + v0 + e));
      key = k > key ? k : key;
    }
    if constexpr (!CHOOSE) narrow(z, y[e]);
  }
  if constexpr (TABLE) {
    // the named tokens, after their vectors have been written (in place, an allowed one is still as it came)
    if constexpr (!CHOOSE) __syncthreads();
    for (int i0 = tid; i0 < named_tokens; i0 += 4 * NT) {
      float z4[4];  // four scattered logits and mask bytes on their way
      int e4[4];
      uint32_t bits4[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = min(i0 + u * NT, named_tokens - 1);
        e4[u] = direct ? i : token[i];
        if (direct && table[i] == 0) continue;
        z4[u] = widen(x[e4[u]]);
        bits4[u] = none ? 0u : 0xFFu;
        if (mask) bits4[u] = mask[e4[u] / 8];
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = i0 + u * NT;
        if (i >= named_tokens) break;
        const uint32_t w = table[i], times = w & COUNT;
        if (w == 0) continue;  // direct: not named
        const int e = e4[u];
        float z = z4[u];
        if (w & (SEEN | COUNT)) z = z > 0.f ? __fdiv_rn(z, rep) : __fmul_rn(z, rep);
        if (times) z = __fsub_rn(__fsub_rn(z, __fmul_rn(freq, (float)times)), pres);
        if (w >> 21) z = __fadd_rn(z, bias_sum[PRA_RULES_MAX_BIASES - (w >> 21)]);
        if (!((bits4[u] >> (e & 7)) & 1u)) z = -INFINITY;
        if constexpr (CHOOSE) {
          const unsigned long long k = choice_key(z, (uint32_t)(a.vocab_start + v0 + e));
          key = k > key ? k : key;
        }
        if constexpr (!CHOOSE) narrow(z, y[e]);
      }
    }
  }
  if constexpr (CHOOSE) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long other = __shfl_xor_sync(0xffffffffu, key, o);
      key = other > key ? other : key;
    }
    if (lane == 0) s_best[warp] = key;
    __syncthreads();
    if (warp == 0) {
      key = lane < NT / 32 ? s_best[lane] : 0;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const unsigned long long other = __shfl_xor_sync(0xffffffffu, key, o);
        key = other > key ? other : key;
      }
      if (lane == 0) s_cluster = key;
    }
    cluster.sync();
    if (part == 0 && warp == 0) {
      unsigned long long other = lane < parts ? *cluster.map_shared_rank(&s_cluster, lane) : 0;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const unsigned long long k = __shfl_xor_sync(0xffffffffu, other, o);
        other = k > other ? k : other;
      }
      if (lane == 0) {
        const float z = key_value((uint32_t)(other >> 32));
        const int64_t id = 0xFFFFFFFFu - (uint32_t)other;
        const bool any = z != -INFINITY;
        a.token[b] = any ? id : -1;
        if (a.value) a.value[b] = z;
        if (a.append_ids && any && len < a.capacity) {  // every CTA of the row has read its history by now
          a.append_ids[(int64_t)b * a.ids_stride + len] = (int)id;
          a.hist_len[b] = len + 1;
        }
      }
    }
    cluster.sync();  // the other CTAs' shared memory lives until it has been read
  }
}

template <typename T, int V, bool TABLE, bool CHOOSE, bool PEEL>
cudaError_t launch(const LogitsArgs& a, cudaStream_t st) {
  // One wave of two CTAs per SM: rows in 8 slices while few, whole rows (every id then read once, no
  // exchange) when many; more slices again where the table would leave one CTA per SM.
  int dev = 0, sms = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  int cl = 8, slice = 0, table_words = 0;
  bool direct = false;
  size_t bytes = 0;
  const auto shape = [&](int c) {
    cl = c;
    slice = ((a.V + cl - 1) / cl + 31) / 32 * 32;
    const int64_t most = std::min<int64_t>(slice, (int64_t)a.capacity + a.n_bias);  // tokens that may be named
    direct = TABLE && 2 * most >= slice;
    table_words = !TABLE ? 0 : direct ? slice : (int)most;
    bytes = TABLE ? (size_t)bit_words(slice) * 8 + (size_t)table_words * (direct ? 4 : 8) + (size_t)a.n_bias * 8 : 0;
  };
  shape(8);
  while (cl > 1 && (int64_t)a.B * cl > 2 * sms) shape(cl / 2);
  while (cl < 8 && bytes > 110 * 1024) shape(cl * 2);
  auto kernel = rules_kernel<T, V, TABLE, CHOOSE, PEEL>;
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
  return cudaLaunchKernelEx(&cfg, kernel, a, slice, table_words, direct);
}

template <typename T>
cudaError_t dispatch(const LogitsArgs& a, cudaStream_t st) {
  constexpr int W = 16 / sizeof(T);
  // Vectors need rows of input and output that begin alike.  Rows that begin anywhere have their own variant: in
  // one for all, aligned rows took longer (256 rows of 152,064 13.3 -> 20.8 us), and with single elements these do
  // (75 rows of 50,257 bf16: the choice 14.0 us, now 7.3, processed with 300 ids 17.3, now 9.4).
  const bool table = a.ids != nullptr || a.bias_ids != nullptr;
  const bool aligned = reinterpret_cast<uintptr_t>(a.logits) % 16 == 0 && a.in_stride % W == 0;
  const bool alike = !a.out || ((reinterpret_cast<uintptr_t>(a.out) - reinterpret_cast<uintptr_t>(a.logits)) % 16 == 0 &&
                                (a.out_stride - a.in_stride) % W == 0);
  const auto choose = [&](auto vec, auto peel) {
    if (table) return a.token ? launch<T, vec, true, true, peel>(a, st) : launch<T, vec, true, false, peel>(a, st);
    return a.token ? launch<T, vec, false, true, peel>(a, st) : launch<T, vec, false, false, peel>(a, st);
  };
  using std::integral_constant;
  if (!alike) return choose(integral_constant<int, 1>(), std::false_type());
  return aligned ? choose(integral_constant<int, W>(), std::false_type()) : choose(integral_constant<int, W>(), std::true_type());
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
