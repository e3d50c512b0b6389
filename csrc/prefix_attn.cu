// Attention of a batch that shares a long prefix, on the 5th-generation tensor cores.
//
// For the query row i (batch row b, token t, head h) one softmax runs over the prefix keys, which are
// the same for every row, and the row's own causal keys:
//     s_ij = scale q_i . k_j,   o_i = sum_j e^{s_ij} v_j / sum_j e^{s_ij},   lse_i = log sum_j e^{s_ij}.
// Attending row by row would read the prefix B times; here the B * T * H / Hkv query rows of one KV
// head are the M dimension of S = Q K^T and O = P V, so each prefix key is read once per 256 of them.
//
// One CTA owns NT = 1 or 2 tiles of 128 query rows of one KV head and a range of 128-key blocks:
//   * one thread brings K and V blocks in with TMA (128-byte swizzle) through a ring of R tiles;
//   * one thread issues the MMAs: S_i = Q_i K^T (both operands in shared memory) and O_i += P_i V
//     (P from TMEM), each committed to an mbarrier;
//   * a warpgroup per tile does the softmax, one thread per query row (TMEM lane): a block's 128 scores
//     come into registers once, the running maximum is raised lazily (only when it grows by more
//     than 2^8, then O is rescaled in TMEM), and P goes back over S's columns as bf16, 96 keys and then 32,
//     so that P V of the first begins while the rest is computed and little is left to wait for after it.
// P shares S's columns (S, P and O of two tiles fill TMEM), so S_{j+1} of a tile is issued only after
// P V_j of that tile has completed; the issuer takes the tiles in turn, which keeps one tile's softmax
// beside the other's products.  P is rounded to bf16 (one half step, 2^-8 relative, of each weight: the
// tensor cores take 16-bit operands); the row sums use the unrounded weights, and S, O, maxima and
// sums stay in fp32.
//
// What bounds it: a tile's chain of about 3,200 cycles per block (softmax 1,800, two products of 512,
// the rest hand-overs of 200 to 300 between the roles), against 2,048 cycles of products and 2,048 of
// exponentials for both tiles: 4 x 512 queries behind 16,384 keys 470 us and 1.18 PFLOP/s in a few calls
// after a pause, 525 to 555 us and 1.0 PFLOP/s under the power cap in hundreds of them (8 x 512: 1.27
// and 1.12).  Measured beside it: an issuer per tile, or one that serves whichever tile is ready, half
// as long again (the tiles fall into step and compete for the tensor cores); two threads per row 2%
// longer; S in two buffers of 64 columns 40% (an MMA of 64 columns takes 57 cycles, one of 128 takes
// 65); a quarter of the exponentials as polynomials as long or longer; only one tile in its exponentials
// at a time 9% longer; 224 registers for the softmax warps (setmaxnreg, with two idle warps) 2% longer.
//
// Keys past the ones any query of the CTA may see are never multiplied: their scores are replaced by
// -inf, and their value rows are zeroed in shared memory (a stale row may hold NaN, and 0 * NaN is
// not 0).  Every wait is bounded; a CTA that times out sets *status, waits (bounded) for its copies
// and MMAs in flight, frees its TMEM and returns.  What it leaves unwritten the merge reads all the same, as
// numbers without meaning: every index it takes from memory is written by CTAs that gave up, too.
#include <algorithm>
#include <map>
#include <mutex>
#include <utility>

#include "serving.h"
#include "tcgen05.cuh"

namespace pra {
namespace prefix {

constexpr int BM = 128;  // query rows of a tile
constexpr int BN = 128;  // keys of a block
constexpr int HEAD = 96;  // of which P V takes these first
static_assert(HEAD % 32 == 0 && HEAD < BN, "weights are stored 32 keys at a time");
constexpr float LOG2E = 1.4426950408889634f;
constexpr float RESCALE_LOG2 = 8.f;
constexpr long long WAIT_CYCLES = 4000000000LL;

template <int D, int NT>
struct Cfg {
  static constexpr int BOXES = D / 64;
  static constexpr int BOX = BN * 128;        // 128 rows x 64 columns
  static constexpr int TILE = BOXES * BOX;    // one K, V or Q tile
  static constexpr int R = NT == 2 ? (D == 128 ? 4 : 6) : (D == 128 ? 2 : 4);
  static constexpr int SOFTMAX = NT * 128;   // softmax threads; then the issuer's and the producer's warp
  static constexpr int THREADS = SOFTMAX + 64;
  static constexpr int OFF_RING = NT * TILE;
  static constexpr int OFF_BAR = OFF_RING + R * TILE;
  static constexpr int OFF_ROW = OFF_BAR + 256;        // [NT][BM] offsets of the rows in global memory
  static constexpr int SMEM = OFF_ROW + NT * BM * 8 + 1024;  // + alignment slack
  static constexpr int O_COL = NT * BN;               // TMEM: S / P of tile i at i * BN, O at O_COL + i * D
  static constexpr uint32_t COLS = NT == 2 ? 512 : 256;
  static constexpr int CTAS = NT == 2 ? 1 : 2;        // per SM
  static constexpr int STAGE = 32 * (D * 4 + 16);     // a warp's outputs on their way out (over queries and ring)
  static_assert(O_COL + NT * D <= (int)COLS, "TMEM");
  static_assert(NT * 4 * STAGE <= (NT + R) * TILE, "output staging");
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float max3(float a, float b, float c) {  // NaN if one is
  float m;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(a), "f"(b), "f"(c));
  return m;
}

// Two fp32 values in one 64-bit register pair, and the packed operations on them.
using f2 = unsigned long long;
__device__ __forceinline__ f2 pack2(float a, float b) {
  f2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack2(f2 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
  f2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f2 add2(f2 a, f2 b) {
  f2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

__device__ __forceinline__ void tma_load3(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n" ::"r"(
          dst),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(smem_u32(bar)) : "memory");
}

// Swizzled shared-memory descriptors (128-byte rows, 8-row groups of 1,024 bytes).  K-major: the
// stride offset is the next 8 rows; MN-major: it is the next 8 K rows, and the leading offset the
// next 64 columns.
__device__ __forceinline__ uint64_t desc_sw128(uint32_t addr, uint32_t lead) {
  uint64_t d = (uint64_t)((addr >> 4) & 0x3FFFu);
  d |= (uint64_t)((lead >> 4) & 0x3FFFu) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}

// Bounded wait that also ends when another role of the CTA has given up.
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, volatile int* abort) {
  if (mbar_try_wait_parity(bar, parity)) return true;
  const long long t0 = clock64();
  while (!mbar_try_wait_parity(bar, parity)) {
    if (*abort || clock64() - t0 > WAIT_CYCLES) {
      *abort = 1;
      return false;
    }
  }
  return true;
}

// What a CTA works on, computed alike by every thread.
struct Item {
  int kvh, b;             // KV head; batch row (-1: packed)
  int row0, rows;         // first query row of the CTA, query rows of the whole row space
  int prefix_seen;        // prefix keys any of the CTA's queries may see
  int own_seen;           // own keys any of them may see
  int prefix_blocks;      // blocks [0, prefix_blocks) are prefix, the rest own
  int lo, hi;             // blocks of this split
};

// The query tile of this CTA and its share of the keys: all of them for the first `whole` tiles, else part
// `split` of `splits`.
struct Share {
  int tile, split, splits;
};
__device__ __forceinline__ Share share_of(const PrefixAttnArgs& a) {
  if (a.whole == 0) return {(int)blockIdx.x, (int)blockIdx.y, a.splits};
  if ((int)blockIdx.x < a.whole) return {(int)blockIdx.x, 0, 1};
  const int behind = ((int)gridDim.x - a.whole) / a.splits, c = (int)blockIdx.x - a.whole;
  return {a.whole + c % behind, c / behind, a.splits};
}

template <int NT>
__device__ __forceinline__ Item item_of(const PrefixAttnArgs& a, const Share& share, int seen) {
  Item it;
  const int G = a.H / a.Hkv;
  it.rows = (a.packed ? a.B : 1) * a.T * G;
  const int tiles = (it.rows + NT * BM - 1) / (NT * BM);
  int x = share.tile;
  it.row0 = (x % tiles) * NT * BM;
  x /= tiles;
  it.kvh = x % a.Hkv;
  it.b = a.packed ? -1 : x / a.Hkv;
  it.prefix_seen = a.use_prefix ? seen : 0;
  it.own_seen = 0;
  if (a.use_own) {  // the CTA's last query sees the most
    const int len = max(0, min(a.len[it.b], a.cap));
    const int t = min(it.row0 + NT * BM, it.rows) - 1;
    it.own_seen = max(0, len - a.T + t / G + 1);
  }
  it.prefix_blocks = (it.prefix_seen + BN - 1) / BN;
  const int n = it.prefix_blocks + (it.own_seen + BN - 1) / BN;
  it.lo = (int)((int64_t)n * share.split / share.splits);
  it.hi = (int)((int64_t)n * (share.split + 1) / share.splits);
  return it;
}

template <int D, int NT>
__global__ void __launch_bounds__(Cfg<D, NT>::THREADS, Cfg<D, NT>::CTAS)
    prefix_kernel(const __grid_constant__ CUtensorMap map_pk, const __grid_constant__ CUtensorMap map_pv,
                  const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                  const PrefixAttnArgs a) {
  using C = Cfg<D, NT>;
  constexpr int R = C::R;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);  // [R] a ring tile has landed
  uint64_t* empty = full + R;                                        // [R] a ring tile has been read
  uint64_t* s_full = empty + R;                                      // [NT] S_i is in TMEM
  uint64_t* p_head = s_full + NT;                                    // [NT] the first HEAD keys' P_i is in TMEM
  uint64_t* p_full = p_head + NT;                                    // [NT] all of P_i is
  uint64_t* o_full = p_full + NT;                                    // [NT] O_i has P_i V
  uint64_t* q_full = o_full + NT;                                    // [NT] Q_i is in shared memory
  uint64_t* drain = q_full + NT;                                     // [1] every MMA issued has completed
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort;
  __shared__ int s_seen;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const Share share = share_of(a);
  pdl_launch_dependents();  // the own part, as this grid's CTAs make room, or the merge
  const int G = a.H / a.Hkv;
  constexpr int ISSUER = C::SOFTMAX / 32, PRODUCER = ISSUER + 1;  // warps
  if (tid == 0) {
    for (int i = 0; i < R; ++i) {
      mbar_init(full + i, 1);
      mbar_init(empty + i, i % 2 == 0 ? NT : 1);  // K: each tile's softmax, V: the issuer
    }
    for (int i = 0; i < NT; ++i) {
      mbar_init(s_full + i, 1);
      mbar_init(p_head + i, 4);
      mbar_init(p_full + i, 4);
      mbar_init(o_full + i, 1);
      mbar_init(q_full + i, 4);
    }
    mbar_init(drain, 1);
    s_abort = 0;
    s_seen = 0;
    tc::fence_mbarrier_init();
  }
  if (warp == PRODUCER) {
    tc::alloc(&s_tmem, C::COLS);
    tc::relinquish();
  }
  __syncthreads();
  // the prefix keys any query row of this CTA may see
  {
    const int rows = (a.packed ? a.B : 1) * a.T * G;
    const int tiles = (rows + NT * BM - 1) / (NT * BM);
    const int row0 = (share.tile % tiles) * NT * BM, b1 = share.tile / (tiles * a.Hkv);
    int seen = 0;
    if (!a.use_prefix) seen = 0;
    else if (a.prefix_len == nullptr) seen = a.P;
    else if (!a.packed) seen = max(0, min(a.prefix_len[b1], a.P));
    else {
      const int b_lo = row0 / (a.T * G), b_hi = (min(rows, row0 + NT * BM) - 1) / (a.T * G);
      for (int b = b_lo + tid; b <= b_hi; b += C::THREADS) seen = max(seen, min(a.prefix_len[b], a.P));
    }
    if (seen > 0) atomicMax(&s_seen, seen);
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const Item it = item_of<NT>(a, share, s_seen);
  const uint32_t tmem = s_tmem;
  const uint32_t ring = smem_u32(smem + C::OFF_RING);
  const int n = it.hi - it.lo;
  int issued = 0;  // ring tiles requested (the producer's count)
  // rows of the block that some query of the CTA may see
  auto block_seen = [&](int j) {
    return j < it.prefix_blocks ? it.prefix_seen - j * BN : it.own_seen - (j - it.prefix_blocks) * BN;
  };

  if (warp == PRODUCER) {
    // ---------------------------------------------------------------- K / V producer
    if (lane == 0 && n > 0) {
      for (int j = it.lo; j < it.hi && !s_abort; ++j) {
        const bool own = j >= it.prefix_blocks;
        const int y = (own ? j - it.prefix_blocks : j) * BN, z = own ? it.b : 0;
        bool ok = true;
        for (int kv = 0; kv < 2 && ok; ++kv) {
          const int r = issued % R;
          if (issued >= R) ok = wait(empty + r, (uint32_t)((issued / R - 1) & 1), &s_abort);
          if (issued + 1 == a.give_up) s_abort = 1, ok = false;
          if (!ok) break;
          const CUtensorMap* map = kv == 0 ? (own ? &map_k : &map_pk) : (own ? &map_v : &map_pv);
          expect_tx(full + r, C::TILE);
#pragma unroll
          for (int x = 0; x < C::BOXES; ++x)
            tma_load3(ring + r * C::TILE + x * C::BOX, map, it.kvh * D + x * 64, y, z, full + r);
          ++issued;
        }
        if (!ok) break;
      }
    }
  } else if (warp >= ISSUER) {
    // ---------------------------------------------------------------- MMA issuer
    constexpr uint32_t ID_S = tc::idesc_bf16(BM, BN, false);
    constexpr uint32_t ID_O = tc::idesc_bf16(BM, D, true);
    const uint32_t q_addr = smem_u32(smem);
    auto issue_s = [&](int i, int r) {
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        const uint32_t off = (kk / 4) * C::BOX + (kk % 4) * 32;
        tc::mma_bf16(tmem + i * BN, desc_sw128(q_addr + i * C::TILE + off, 16), desc_sw128(ring + r * C::TILE + off, 16), ID_S, kk > 0);
      }
    };
    auto issue_o = [&](int i, int r, bool head, bool acc) {
#pragma unroll
      for (int kk = head ? 0 : HEAD / 16; kk < (head ? HEAD : BN) / 16; ++kk)
        tc::mma_bf16_ts(tmem + C::O_COL + i * D, tmem + i * BN + kk * 8,
                        desc_sw128(ring + r * C::TILE + kk * 2048, C::BOX), ID_O, (acc || kk > 0) ? 1u : 0u);
    };
    if (lane == 0 && n > 0) {
      bool ok = wait(full, 0, &s_abort);
      for (int i = 0; i < NT && ok; ++i) {
        ok = wait(q_full + i, 0, &s_abort);
        if (!ok) break;
        tc::fence_after();
        issue_s(i, 0);
        tc::commit(s_full + i);
      }
      for (int j = 0; j < n && ok; ++j) {
        const int vt = 2 * j + 1, kt = 2 * j + 2;  // ring positions of V_j and K_{j+1}
        ok = wait(full + vt % R, (uint32_t)((vt / R) & 1), &s_abort);
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          ok = ok && wait(p_head + i, (uint32_t)(j & 1), &s_abort);
          if (!ok) break;
          tc::fence_after();
          issue_o(i, vt % R, true, j > 0);
          ok = wait(p_full + i, (uint32_t)(j & 1), &s_abort);
          if (!ok) break;
          tc::fence_after();
          issue_o(i, vt % R, false, true);
          tc::commit(o_full + i);
          if (j + 1 == n) continue;
          if (i == 0) ok = wait(full + kt % R, (uint32_t)((kt / R) & 1), &s_abort);
          // P V_j reads the columns that S_{j+1} is about to overwrite
          ok = ok && wait(o_full + i, (uint32_t)(j & 1), &s_abort);
          if (!ok) break;
          tc::fence_after();
          issue_s(i, kt % R);
          tc::commit(s_full + i);
          if (i == NT - 1) mbar_arrive(empty + vt % R);
        }
      }
    }
  } else {
    // ---------------------------------------------------------------- softmax
    const int i = warp >> 2, row = tid & (BM - 1);
    const int qr = it.row0 + i * BM + row;
    const bool live = qr < it.rows;
    const int TG = a.T * G;
    const int b = it.b >= 0 ? it.b : min(qr / TG, a.B - 1);
    const int t = (qr / G) % a.T, h = it.kvh * G + qr % G;
    // This tile's queries into shared memory (rows past the last: zero), all in flight together.  Each
    // thread works out its own row's place once: divisions by G and T for every piece took 3 us.
    int64_t* row_at = reinterpret_cast<int64_t*>(smem + C::OFF_ROW) + i * BM;
    auto tile_sync = [&]() { asm volatile("bar.sync %0, 128;\n" ::"r"(2 + i) : "memory"); };
    row_at[row] = live ? b * a.q_batch + t * a.q_token + (int64_t)h * D : -1;
    tile_sync();
    {
      constexpr int CH = D / 8, STEP = BM / CH;
      const int c = row % CH;
      const uint32_t to = i * C::TILE + (c / 8) * C::BOX;
#pragma unroll 4
      for (int r = row / CH; r < BM; r += STEP) {
        const int64_t at = row_at[r];
        cp_async16(smem + to + r * 128 + (((c & 7) ^ (r & 7)) << 4), at >= 0 ? a.q + at + c * 8 : a.q, at >= 0);
      }
      cp_async_commit();
      cp_async_wait<0>();
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(q_full + i);
    const int prefix_lim = !live ? 0 : a.prefix_len ? max(0, min(a.prefix_len[b], a.P)) : a.P;
    int own_lim = 0;
    if (live && a.use_own) own_lim = max(0, min(max(a.len[b], 0), a.cap) - a.T + t + 1);
    const uint32_t t_lane = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + t_lane + i * BN, t_o = tmem + t_lane + C::O_COL + i * D;
    const float sl2 = a.scale * LOG2E;
    float m_run = -INFINITY, l_run = 0.f;
    // After a wait that gave up (here or in another role) the rest runs through without waiting; nothing
    // is written at the end.
    bool ok = true;
    for (int j = 0; j < n; ++j) {
      const int blk = it.lo + j;
      const bool own = blk >= it.prefix_blocks;
      const int lim = own ? own_lim - (blk - it.prefix_blocks) * BN : prefix_lim - blk * BN;
      ok &= wait(s_full + i, (uint32_t)(j & 1), &s_abort);
      __syncwarp();
      if (lane == 0 && (warp & 3) == 0) mbar_arrive(empty + (2 * j) % R);  // K_j has been read
      tc::fence_after();
      uint32_t s[BN];
      tc::ld128(t_s, s);
      if (__any_sync(0xffffffffu, lim < BN)) {
#pragma unroll
        for (int c = 0; c < BN; ++c) s[c] = c < lim ? s[c] : 0xff800000u;
      }
      auto at = [&](int c) { return __uint_as_float(s[c]); };
      float m8[8];  // eight chains: their latency would show with four
#pragma unroll
      for (int x = 0; x < 8; ++x) m8[x] = max3(at(x), at(x + 8), at(x + 16));
#pragma unroll
      for (int c = 24; c + 16 <= BN; c += 16)
#pragma unroll
        for (int x = 0; x < 8; ++x) m8[x] = max3(m8[x], at(c + x), at(c + x + 8));
#pragma unroll
      for (int x = 0; x < 4; ++x) m8[x] = max3(m8[x], at(BN - 8 + x), at(BN - 4 + x));
      const float mx = max3(max3(m8[0], m8[1], m8[2]), max3(m8[3], m8[4], m8[5]), max3(m8[6], m8[7], m8[7]));
      // Raised lazily: where it grew by more than the margin.  The first maximum costs no rescaling (O has
      // not been written: P V of the first block overwrites it, and rows that saw nothing so far hold
      // zeros).  A NaN score makes the maximum, and with it the row's sum and output, NaN.  The rescaling
      // stays a rolled loop: it is rare, and unrolled it cost the loop its registers (534 -> 496 us).
      const bool rescale = (mx - m_run) * sl2 > RESCALE_LOG2 || mx != mx;
      const float m_old = m_run;
      if (rescale) m_run = mx;
      if (__any_sync(0xffffffffu, rescale)) {
        const float corr = rescale && m_old != -INFINITY ? ex2((m_old - mx) * sl2) : 1.f;
        l_run *= corr;
        if (j > 0) {  // P V_{j-1} has completed: S_j was issued after it
#pragma unroll 1
          for (int c0 = 0; c0 < D; c0 += 16) {
            uint32_t r[16];
            tc::ld16(t_o + c0, r);
#pragma unroll
            for (int c = 0; c < 16; ++c) r[c] = __float_as_uint(__uint_as_float(r[c]) * corr);
            tc::st16(t_o + c0, r);
          }
        }
      }
      const int seen = block_seen(blk);
      if (seen < BN) {  // value rows that no query of the CTA sees: zero, before this tile's weights are handed on
                        // (each tile for itself: with two, both write the same zeros)
        const int vt = 2 * j + 1;
        ok &= wait(full + vt % R, (uint32_t)((vt / R) & 1), &s_abort);
        uint8_t* v = smem + C::OFF_RING + (vt % R) * C::TILE;
        for (int e = seen * (D / 8) + row; e < BN * (D / 8); e += BM) {
          const int r = e / (D / 8), c = e % (D / 8);
          *reinterpret_cast<uint4*>(v + (c / 8) * C::BOX + r * 128 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async_smem();
        __syncwarp();
      }
      const float ms = m_run == -INFINITY ? 0.f : m_run * sl2;
      const f2 sl2x2 = pack2(sl2, sl2), msx2 = pack2(-ms, -ms);
      f2 sum[2] = {pack2(0.f, 0.f), pack2(0.f, 0.f)};
#pragma unroll
      for (int c0 = 0; c0 < BN / 2; c0 += 16) {
        uint32_t w[16];  // two weights each
#pragma unroll
        for (int c = 0; c < 16; ++c) {
          const f2 x = fma2(pack2(at(2 * (c0 + c)), at(2 * (c0 + c) + 1)), sl2x2, msx2);
          float p0, p1;
          unpack2(x, p0, p1);
          p0 = ex2(p0);
          p1 = ex2(p1);
          sum[c & 1] = add2(sum[c & 1], pack2(p0, p1));
          w[c] = pack_bf16(p0, p1);
        }
        tc::st16_async(t_s + c0, w);
        if (2 * c0 + 32 == HEAD || 2 * c0 + 32 == BN) {
          tc::wait_st();
          tc::fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(2 * c0 + 32 == HEAD ? p_head + i : p_full + i);
        }
      }
      float sums[4];
      unpack2(sum[0], sums[0], sums[1]);
      unpack2(sum[1], sums[2], sums[3]);
      l_run += (sums[0] + sums[1]) + (sums[2] + sums[3]);
    }
    if (n > 0) ok &= wait(o_full + i, (uint32_t)((n - 1) & 1), &s_abort);
    // every tile's last product has completed: queries and ring are idle and take the outputs
    asm volatile("bar.sync 1, %0;\n" ::"n"(C::SOFTMAX) : "memory");
    if (__all_sync(0xffffffffu, ok)) {
      tc::fence_after();
      const bool any = m_run != -INFINITY;  // else nothing of this range is visible to the row
      const int64_t bt = (int64_t)b * a.T + t;
      const int64_t place = a.whole > 0 ? (int64_t)(share.tile - a.whole) * (NT * BM) + i * BM + row : bt * a.H + h;
      const int64_t slot = place * a.n_slots + a.slot0 + share.split;
      const bool partial = a.part_o != nullptr && share.tile >= a.whole;
      if (live) {
        if (partial) {
          *reinterpret_cast<float2*>(a.part_ml + 2 * slot) = make_float2(any ? m_run * a.scale : -INFINITY, l_run);
        } else if (a.lse != nullptr) {
          a.lse[((int64_t)b * a.H + h) * a.T + t] = any ? m_run * a.scale + logf(l_run) : -INFINITY;
        }
      }
      // A thread has one row: it goes through shared memory (16 bytes apart, for the banks) and out as one bulk copy,
      // which is read before the CTA ends.  Stores of whole rows by the warp took 1.2 us longer.
      const float inv = partial || !any ? 1.f : 1.f / l_run;
      const int row_bytes = D * (partial ? 4 : 2);
      uint8_t* stage = smem + warp * C::STAGE + lane * (row_bytes + 16);
#pragma unroll 1
      for (int c0 = 0; c0 < D; c0 += 64) {
        uint32_t r[64];
        if (n > 0) tc::ld64(t_o + c0, r);
        auto val = [&](int c) { return n > 0 && any ? __uint_as_float(r[c]) * inv : 0.f; };
        if (partial) {
#pragma unroll
          for (int c = 0; c < 64; c += 4)
            *reinterpret_cast<float4*>(stage + (c0 + c) * 4) = make_float4(val(c), val(c + 1), val(c + 2), val(c + 3));
        } else {
#pragma unroll
          for (int c = 0; c < 64; c += 8)
            *reinterpret_cast<uint4*>(stage + (c0 + c) * 2) =
                make_uint4(pack_bf16(val(c), val(c + 1)), pack_bf16(val(c + 2), val(c + 3)),
                           pack_bf16(val(c + 4), val(c + 5)), pack_bf16(val(c + 6), val(c + 7)));
        }
      }
      fence_proxy_async_smem();
      if (live) {
        uint8_t* to = partial ? reinterpret_cast<uint8_t*>(a.part_o + slot * D) : reinterpret_cast<uint8_t*>(a.out + (bt * a.H + h) * D);
        asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;\n" ::"l"(to), "r"(smem_u32(stage)), "r"(row_bytes)
                     : "memory");
        asm volatile("cp.async.bulk.commit_group;\ncp.async.bulk.wait_group.read 0;\n" ::: "memory");
      }
    }
  }
  __syncwarp();
  tc::fence_before();
  __syncthreads();
  if (s_abort) {
    // Nothing may land in shared memory, and no MMA may read it or TMEM, after the CTA has gone: wait for both.
    // Here and not where the issuer gives up: its own waits may all have been answered while another role's ran out.
    if (tid == 0 && a.status != nullptr) atomicExch(a.status, 1);
    for (int x = max(0, issued - R); x < issued; ++x)
      tc::mbar_wait_cycles(full + x % R, (uint32_t)((x / R) & 1), WAIT_CYCLES);
    if (tid == ISSUER * 32) {  // the thread whose MMAs they are
      tc::commit(drain);
      tc::mbar_wait_cycles(drain, 0, WAIT_CYCLES);
    }
    __syncthreads();
  }
  if (warp == PRODUCER) {
    tc::fence_after();
    tc::dealloc(tmem, C::COLS);
  }
  if (a.after_prefix) pdl_wait();  // what waits for this grid waits for the one before, too
}

// ---------------------------------------------------------------- own keys of few queries
// Up to 16 query rows (t, g) of a (batch row, KV head) against its own keys: bound by reading K and V once.
// A persistent grid of two CTAs per SM (where two fit); each walks its run of 64-key blocks across items without
// draining its pipeline: one thread streams K and V tiles (TMA, 128-byte swizzle) and the items' queries
// (bulk copies) some stages ahead, four warps take 16 keys of every block each, with their own running
// maximum and sum, and join at the end of an item.  The products are transposed, S^T = K Q^T and
// O^T = V^T P^T (mma.sync m16n8k16, keys or features as M, 8 NB query rows as N): with the queries as M
// the 16 rows of a tile were mostly padding and twice the MMAs bound an SM to 44 GB/s of keys, an SM's
// share of HBM.  P^T goes from accumulator to operand layout with movmatrix.  Equal runs of blocks, with
// two more counted per item for its queries and its end (2,100 cycles beside a block's 1,000), keep every
// SM busy to the end whatever the lengths: 36 SMs walk 768 items of 1 to 8 blocks in 60 us, without the two
// in 80.  On all SMs it reads 128 rows of 2,048 keys (8 KV heads of 128) at 6.4 TB/s, 64 rows of 64 to 1,024 keys at
// 4.2.  Of 10 to 16 query rows of head dim 128 only one CTA fits on an SM: 64 rows of 2,048 keys are read at 4.8 to
// 4.9 TB/s then, at 5.9 with 8 query rows.
constexpr int OB = 64;       // keys of a block
constexpr int OWARPS = 4;
constexpr int ITEM = 2;  // blocks' worth of time that beginning and ending an item takes
template <int D>
struct OwnCfg {
  static constexpr int BOXES = D / 64, BOX = OB * 128, TILE = BOXES * BOX, STAGE = 2 * TILE;
  static constexpr int STAGES = D == 128 ? 3 : 6;
  static constexpr int THREADS = OWARPS * 32 + 32;
  static constexpr int RED_LD = D / 2 + 4;  // half of the columns at a time
  static constexpr int smem(int rows) {
    return 1024 + STAGES * STAGE + 2 * rows * D * 2 + OWARPS * rows * RED_LD * 4 + OWARPS * rows * 8 + 256;
  }
};

// Byte offset of (key r, column c) in a swizzled tile.
__device__ __forceinline__ uint32_t tile_off(int r, int c) {
  return (uint32_t)((c >> 6) * (OB * 128) + r * 128 + ((((c & 63) >> 3) ^ (r & 7)) << 4) + ((c & 7) << 1));
}

__device__ __forceinline__ int own_len(const OwnAttnArgs& a, int b) { return max(0, min(a.len[b], a.cap)); }
__device__ __forceinline__ int own_blocks(int len) { return max(1, (len + OB - 1) / OB); }

// The 8 x 8 matrix of 16-bit elements in the mma fragment layout, transposed.
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

template <int D, int NB>  // NB: query rows / 8
__global__ void __launch_bounds__(OwnCfg<D>::THREADS, 2)
    own_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const OwnAttnArgs a) {
  using C = OwnCfg<D>;
  pdl_launch_dependents();        // the merge (it waits for this grid's end)
  if (!a.after_prefix) pdl_wait();  // else the launch before is the prefix part's, which writes none of this one's inputs
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int G = a.H / a.Hkv, rows = a.T * G;
  __nv_bfloat16* sq = reinterpret_cast<__nv_bfloat16*>(smem + C::STAGES * C::STAGE);  // [2][rows][D]
  float* red = reinterpret_cast<float*>(sq + 2 * rows * D);                            // [4][rows][RED_LD]
  float* red_ml = red + OWARPS * rows * C::RED_LD;                                     // [4][rows][2]
  __shared__ uint64_t full[C::STAGES], empty[C::STAGES], q_full[2], q_empty[2];
  __shared__ long long s_part[C::THREADS / 32];
  __shared__ long long s_before[2];
  __shared__ int s_row[2], s_abort;
  if (tid == 0) {
    for (int i = 0; i < C::STAGES; ++i) {
      mbar_init(full + i, 1);
      mbar_init(empty + i, OWARPS);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(q_full + i, 1);
      mbar_init(q_empty + i, OWARPS);
    }
    s_abort = 0;
    s_row[0] = s_row[1] = -1;
    tc::fence_mbarrier_init();
  }
  // Every item weighs its blocks and ITEM more; the CTAs take equal runs of that weight.  Here: all of it,
  // and the rows where this CTA's run begins and ends (a sum, then a scan over the lengths).
  auto block_total = [&](long long v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if (lane == 0) s_part[warp] = v;
    __syncthreads();
    long long all = 0;
    for (int w = 0; w < C::THREADS / 32; ++w) all += s_part[w];
    return all;
  };
  long long mine = 0;
  for (int b = tid; b < a.B; b += C::THREADS) mine += own_blocks(own_len(a, b)) + ITEM;
  const long long total = block_total(mine) * a.Hkv;
  // no CTA between an item's first and last may be without a block of it: at most one CTA per unit
  const long long n = min((long long)a.ctas, total), me = min((long long)blockIdx.x, n);
  const long long u0 = total * me / n, u1 = total * min(me + 1, n) / n;
  for (long long b0 = 0, base = 0; b0 < a.B && u0 < u1; b0 += C::THREADS) {
    const long long nb = b0 + tid < a.B ? (long long)(own_blocks(own_len(a, (int)b0 + tid)) + ITEM) * a.Hkv : 0;
    long long upto = nb;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    __syncthreads();
    if (lane == 31) s_part[warp] = upto;
    __syncthreads();
    long long all = 0;
    for (int w = 0; w < C::THREADS / 32; ++w) {
      if (w < warp) upto += s_part[w];
      all += s_part[w];
    }
#pragma unroll
    for (int x = 0; x < 2; ++x) {  // the last unit of the run, not the one behind it
      const long long at = x == 0 ? u0 : u1 - 1;
      if (nb > 0 && base + upto - nb <= at && at < base + upto) {
        s_row[x] = (int)b0 + tid;
        s_before[x] = base + upto - nb;
      }
    }
    base += all;
    if (base >= u1) break;  // the same for every thread
  }
  __syncthreads();
  int issued = 0, queries = 0;  // stages and query tiles requested (the producer's counts)
  // where a unit is: row and its keys, KV head, block of the item
  struct Place {
    int b, len, kvh, blk, blocks;
  };
  // the place of a unit of weight: in front of an item's blocks (blk = 0) or one of them
  auto place_of = [&](int x, long long unit) {
    Place p;
    p.b = s_row[x];
    p.len = own_len(a, p.b);
    p.blocks = own_blocks(p.len);
    const int at = (int)(unit - s_before[x]);
    p.kvh = at / (p.blocks + ITEM);
    p.blk = at - p.kvh * (p.blocks + ITEM) - ITEM;
    return p;
  };
  auto start = [&]() {
    Place p = place_of(0, u0);
    p.blk = max(p.blk, 0);
    return p;
  };
  int count = 0;  // this CTA's blocks
  if (s_row[0] >= 0 && s_row[1] >= 0) {
    const Place p = place_of(0, u0), q = place_of(1, u1 - 1);
    // weight of the run, less the ITEMs (or what of the first and last lies in it)
    const long long items = (long long)(q.b - p.b) * a.Hkv + q.kvh - p.kvh;  // items begun behind the first
    count = (int)(u1 - u0 - items * ITEM - max(0, -p.blk) + max(0, -(q.blk + 1)));
  }
  auto advance = [&](Place& p) {  // to the next unit; true when it begins an item
    if (++p.blk < p.blocks) return false;
    p.blk = 0;
    if (++p.kvh == a.Hkv) {
      p.kvh = 0;
      if (++p.b < a.B) p.len = own_len(a, p.b), p.blocks = own_blocks(p.len);
    }
    return true;
  };

  if (warp == OWARPS) {
    if (lane == 0 && count > 0) {
      Place p = start();
      bool fresh = true;
      for (int u = 0; u < count && !s_abort; ++u) {
        if (fresh) {  // the item's queries: one run of G heads per token
          const int slot = queries & 1;
          if (queries > 1 && !wait(q_empty + slot, (uint32_t)((queries / 2 - 1) & 1), &s_abort)) break;
          expect_tx(q_full + slot, rows * D * 2);
          for (int t = 0; t < a.T; ++t)
            asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n" ::"r"(
                             smem_u32(sq + (slot * rows + t * G) * D)),
                         "l"(a.q + p.b * a.q_batch + t * a.q_token + (int64_t)p.kvh * G * D), "r"(G * D * 2),
                         "r"(smem_u32(q_full + slot))
                         : "memory");
          ++queries;
        }
        const int st = issued % C::STAGES;
        if (issued >= C::STAGES && !wait(empty + st, (uint32_t)((issued / C::STAGES - 1) & 1), &s_abort)) break;
        if (issued + 1 == a.give_up) {
          s_abort = 1;
          break;
        }
        expect_tx(full + st, C::STAGE);
        const uint32_t to = smem_u32(smem + st * C::STAGE);
#pragma unroll
        for (int x = 0; x < C::BOXES; ++x) {
          tma_load3(to + x * C::BOX, &map_k, p.kvh * D + x * 64, p.blk * OB, p.b, full + st);
          tma_load3(to + C::TILE + x * C::BOX, &map_v, p.kvh * D + x * 64, p.blk * OB, p.b, full + st);
        }
        ++issued;
        fresh = advance(p);
      }
    }
  } else if (count > 0) {
    // After a wait that gave up the rest runs through without waiting (the barriers between warps stay
    // matched) and nothing more is written.
    bool ok = true;
    Place p = start();
    bool fresh = true;
    int item_no = 0;
    uint32_t qb[NB][D / 16][2];                     // Q^T, the B operand of S^T
    float o[NB][D / 16][4], m_run[NB][2], l_run[NB][2];  // O^T; this thread's two query rows of each 8
    int lim[NB][2], len = 0;
    int first_lim[NB][2];  // of a row without own keys: t + 1 - T
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = nb * 8 + (lane & 3) * 2 + e;
        first_lim[nb][e] = row < rows ? row / G + 1 - a.T : -a.cap;
      }
    const float sl2 = a.scale * LOG2E;
    for (int u = 0; u < count; ++u) {
      if (fresh) {
        const int slot = item_no & 1;
        ok &= wait(q_full + slot, (uint32_t)((item_no >> 1) & 1), &s_abort);
        __syncwarp();
        const __nv_bfloat16* qs = sq + slot * rows * D;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          const int r = min(nb * 8 + (lane & 7), rows - 1);  // rows past the last repeat it, their results are not used
#pragma unroll
          for (int kk = 0; kk < D / 16; kk += 2) {
            uint32_t f[4];
            ldmatrix_x4(f, smem_u32(qs + r * D + kk * 16 + (lane >> 3) * 8));
            qb[nb][kk][0] = f[0];
            qb[nb][kk][1] = f[1];
            qb[nb][kk + 1][0] = f[2];
            qb[nb][kk + 1][1] = f[3];
          }
        }
        ++item_no;
        len = p.len;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            lim[nb][e] = max(0, len + first_lim[nb][e]);
            m_run[nb][e] = -INFINITY;
            l_run[nb][e] = 0.f;
          }
#pragma unroll
          for (int d = 0; d < D / 16; ++d) o[nb][d][0] = o[nb][d][1] = o[nb][d][2] = o[nb][d][3] = 0.f;
        }
      }
      const int st = u % C::STAGES;
      ok &= wait(full + st, (uint32_t)((u / C::STAGES) & 1), &s_abort);
      __syncwarp();
      uint8_t* kt = smem + st * C::STAGE;
      const uint32_t k_addr = smem_u32(kt), v_addr = k_addr + C::TILE;
      const int key0 = p.blk * OB + warp * 16;  // this warp's first key
      if (key0 + 16 > len) {  // value rows past the last key: zero (they may hold NaN)
        for (int e = max(0, len - key0) * (D / 8) + lane; e < 16 * (D / 8); e += 32)
          *reinterpret_cast<uint4*>(kt + C::TILE + tile_off(warp * 16 + e / (D / 8), (e % (D / 8)) * 8)) = make_uint4(0, 0, 0, 0);
        fence_proxy_async_smem();  // before a later copy into this stage
        __syncwarp();
      }
      // S^T of this warp's 16 keys, two accumulators so that the MMAs do not wait for one another
      float s[NB][2][4];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int x = 0; x < 2; ++x) s[nb][x][0] = s[nb][x][1] = s[nb][x][2] = s[nb][x][3] = 0.f;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        uint32_t ka[4];
        ldmatrix_x4(ka, k_addr + tile_off(warp * 16 + (lane & 15), kk * 16 + (lane >> 4) * 8));
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) mma_bf16_16816(s[nb][kk & 1], ka, qb[nb][kk]);
      }
      if (fresh) {
        // the MMAs have taken the queries' fragments, so their loads are done and the tile may be filled
        // again (an arrival right behind the loads is not ordered after their reads)
        __syncwarp();
        if (lane == 0) mbar_arrive(q_empty + ((item_no - 1) & 1));
      }
      uint32_t pb[NB][2];  // P^T, the B operand of O^T
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        float z[4];  // keys (lane >> 2) + 8 (e >> 1), query rows 8 nb + 2 (lane & 3) + (e & 1)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          z[e] = s[nb][0][e] + s[nb][1][e];
          if (key0 + (lane >> 2) + 8 * (e >> 1) >= lim[nb][e & 1]) z[e] = -INFINITY;
        }
        float mx[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          mx[e] = max3(z[e], z[e + 2], m_run[nb][e]);
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) {
            const float other = __shfl_xor_sync(0xffffffffu, mx[e], x);
            mx[e] = max3(mx[e], other, other);
          }
        }
        // O is rescaled only when some row's maximum has grown
        if (__any_sync(0xffffffffu, !(mx[0] <= m_run[nb][0]) || !(mx[1] <= m_run[nb][1]))) {
          float corr[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            corr[e] = mx[e] == -INFINITY ? 1.f : ex2((m_run[nb][e] - mx[e]) * sl2);
            m_run[nb][e] = mx[e];
            l_run[nb][e] *= corr[e];
          }
#pragma unroll
          for (int d = 0; d < D / 16; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[nb][d][e] *= corr[e & 1];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float m = m_run[nb][e & 1];
          z[e] = ex2(fmaf(z[e], sl2, m == -INFINITY ? 0.f : -m * sl2));
          l_run[nb][e & 1] += z[e];
        }
        pb[nb][0] = movmatrix_trans(pack_bf16(z[0], z[1]));
        pb[nb][1] = movmatrix_trans(pack_bf16(z[2], z[3]));
      }
#pragma unroll
      for (int d = 0; d < D / 16; ++d) {
        uint32_t va[4];
        ldmatrix_x4_trans(va, v_addr + tile_off(warp * 16 + (lane & 7) + ((lane >> 4) & 1) * 8, d * 16 + ((lane >> 3) & 1) * 8));
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) mma_bf16_16816(o[nb][d], va, pb[nb]);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(empty + st);
      const Place at = p;
      fresh = advance(p);
      if (!fresh && u + 1 < count) continue;
      // the item (or this CTA's part of it) is done: join the four warps' sums, half of the columns at a time
      const int item = at.b * a.Hkv + at.kvh;
      const int64_t piece = (int64_t)(item + (int)blockIdx.x) * rows;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float l = l_run[nb][e];
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
          const int row = nb * 8 + (lane & 3) * 2 + e;
          if ((lane >> 2) == 0 && row < rows)
            *reinterpret_cast<float2*>(red_ml + (warp * rows + row) * 2) = make_float2(m_run[nb][e], l);
        }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int row = nb * 8 + (lane & 3) * 2 + e;
            if (row < rows) {
              float* dst = red + (warp * rows + row) * C::RED_LD + (lane >> 2);
#pragma unroll
              for (int d = 0; d < D / 32; ++d) {
                dst[d * 16] = o[nb][d + half * (D / 32)][e];
                dst[d * 16 + 8] = o[nb][d + half * (D / 32)][e + 2];
              }
            }
          }
        asm volatile("bar.sync 1, %0;\n" ::"n"(OWARPS * 32) : "memory");
        for (int e = tid; e < rows * (D / 8); e += OWARPS * 32) {  // four columns of a row
          const int row = e / (D / 8), col = e % (D / 8) * 4;
          float2 ml[OWARPS];
          float4 part[OWARPS];
#pragma unroll
          for (int w = 0; w < OWARPS; ++w) {
            ml[w] = *reinterpret_cast<const float2*>(red_ml + (w * rows + row) * 2);
            part[w] = *reinterpret_cast<const float4*>(red + (w * rows + row) * C::RED_LD + col);
          }
          const float M = max3(max3(ml[0].x, ml[1].x, ml[2].x), ml[3].x, ml[3].x);
          float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
          float L = 0.f;
#pragma unroll
          for (int w = 0; w < OWARPS; ++w) {
            const float f = ml[w].x == -INFINITY ? 0.f : ex2((ml[w].x - M) * sl2);
            acc.x += part[w].x * f;
            acc.y += part[w].y * f;
            acc.z += part[w].z * f;
            acc.w += part[w].w * f;
            L += ml[w].y * f;
          }
          if (ok) {
            *reinterpret_cast<float4*>(a.piece_o + (piece + row) * D + half * (D / 2) + col) = acc;
            if (half == 0 && col == 0)
              *reinterpret_cast<float2*>(a.piece_ml + (piece + row) * 2) = make_float2(M == -INFINITY ? M : M * a.scale, L);
          }
        }
        asm volatile("bar.sync 1, %0;\n" ::"n"(OWARPS * 32) : "memory");
      }
      if (tid == 0) {  // after a wait that gave up, too: the merge reads the pieces in this range
        if (u >= at.blk) a.first[item] = blockIdx.x;  // the run began at or before the item's first block
        if (at.blk + 1 == at.blocks) a.last[item] = blockIdx.x;
      }
    }
  }
  __syncwarp();
  __syncthreads();
  if (s_abort) {  // nothing may land in shared memory after the CTA has gone: wait for the copies in flight
    if (tid == 0 && a.status != nullptr) atomicExch(a.status, 1);
    for (int x = max(0, issued - C::STAGES); x < issued; ++x)
      tc::mbar_wait_cycles(full + x % C::STAGES, (uint32_t)((x / C::STAGES) & 1), WAIT_CYCLES);
    for (int x = max(0, queries - 2); x < queries; ++x)
      tc::mbar_wait_cycles(q_full + (x & 1), (uint32_t)((x >> 1) & 1), WAIT_CYCLES);
    __syncthreads();
  }
  pdl_wait();  // the prefix part, launched before, has ended when this grid has
}

// One warp per (b, t, h): the parts weighted by their own maxima and summed in order.  Bound by
// latency: lane s finds part s (32 at a time) and holds its weight, and the first AT_ONCE parts' sums are
// on their way while the maxima are still being compared (a part that holds nothing was not written:
// what is read there is dropped).  16 at once where there are more than 8 slots (8 rows behind 2K, 16 slots:
// 15.5 -> 14.1 us in a graph), else 8, for more warps per SM (64 rows behind 8K, 6 slots: 43.7 us, with 16 45.9).
constexpr int MERGE_WARPS = 4;
template <int D, int AT_ONCE>
__global__ void __launch_bounds__(MERGE_WARPS * 32) merge_kernel(const PrefixMergeArgs a) {
  constexpr int E = D / 32;
  struct alignas(4 * E) Piece {
    float v[E];
  };
  const int64_t at = (int64_t)blockIdx.x * MERGE_WARPS + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  int b, t, h;
  bool ok;
  if (a.tiles > 0) {  // row `at` of the split tiles
    const int G = a.H / a.Hkv, rows_all = (a.packed ? a.B : 1) * a.T * G, per = (rows_all + a.tile_rows - 1) / a.tile_rows;
    const int64_t behind = at / a.tile_rows;
    const int tile = a.tile0 + (int)behind, x = tile / per;  // x: KV head, or (batch row, KV head)
    const int64_t qr = (int64_t)(tile - x * per) * a.tile_rows + (at - behind * a.tile_rows);
    ok = behind < a.tiles && qr < rows_all;
    const int bt = (int)(qr / G);
    b = a.packed ? bt / a.T : x / a.Hkv;
    t = bt % a.T;
    h = (a.packed ? x : x % a.Hkv) * G + (int)(qr - (int64_t)bt * G);
  } else {
    const int64_t bt = at / a.H;
    h = (int)(at - bt * a.H), b = (int)(bt / a.T), t = (int)(bt - (int64_t)b * a.T);
    ok = at < (int64_t)a.B * a.T * a.H;
  }
  pdl_wait();
  if (!ok) return;
  const int64_t query = ((int64_t)b * a.T + t) * a.H + h;  // parts: `at`
  // parts [0, n0) are the first set's, [n0, n1) the second's, [n1, n) the pieces
  const int n0 = a.part_o != nullptr ? a.n_slots : 0, n1 = n0 + (a.more_o != nullptr ? a.n_more : 0);
  int n = n1;
  int64_t row0 = 0;
  const int rows = a.T * (a.H / a.Hkv);
  if (a.piece_o != nullptr) {
    const int G = a.H / a.Hkv, item = b * a.Hkv + h / G, first = a.first[item];
    n += a.last[item] - first + 1;
    row0 = (int64_t)(item + first) * rows + t * G + h % G;
  }
  // (max, sum) and sums of part s
  auto find = [&](int s, const float2*& ml, const float*& o) {
    const int64_t i = s < n0 ? at * a.n_slots + s : s < n1 ? at * a.n_more + (s - n0) : row0 + (int64_t)(s - n1) * rows;
    ml = reinterpret_cast<const float2*>(s < n0 ? a.part_ml : s < n1 ? a.more_ml : a.piece_ml) + i;
    o = (s < n0 ? a.part_o : s < n1 ? a.more_o : a.piece_o) + i * D;
  };
  const float2 nothing = make_float2(-INFINITY, 0.f);
  const float2* ml = nullptr;
  const float* o = nullptr;
  float2 mine = nothing;
  if (lane < n) {
    find(lane, ml, o);
    mine = *ml;
  }
  Piece v[AT_ONCE];
  auto fetch = [&](int s0) {  // parts s0 .. s0 + AT_ONCE - 1 of the 32 that the lanes hold
#pragma unroll
    for (int q = 0; q < AT_ONCE; ++q) {
      const float* src = reinterpret_cast<const float*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(o), s0 + q));
      if (src != nullptr) v[q] = *reinterpret_cast<const Piece*>(src + lane * E);
    }
  };
  fetch(0);
  float M = mine.x;
  for (int s = lane + 32; s < n; s += 32) {
    const float2* m2;
    const float* o2;
    find(s, m2, o2);
    M = max3(M, m2->x, m2->x);
  }
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) {  // NaN if one part's is: it must not pass for an empty row
    const float other = __shfl_xor_sync(0xffffffffu, M, x);
    M = max3(M, other, other);
  }
  float L = 0.f, acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
  for (int s0 = 0; s0 < n; s0 += 32) {
    if (s0 > 0) {
      mine = nothing;
      o = nullptr;
      if (s0 + lane < n) {
        find(s0 + lane, ml, o);
        mine = *ml;
      }
    }
    const float w = mine.x == -INFINITY ? 0.f : exp2f((mine.x - M) * LOG2E);
    if (w != 0.f) L += w * mine.y;
    const int m = min(32, n - s0);
    for (int s = 0; s < m; s += AT_ONCE) {
      if (s0 + s > 0) fetch(s);
#pragma unroll
      for (int q = 0; q < AT_ONCE; ++q) {
        const float ws = __shfl_sync(0xffffffffu, w, (s + q) & 31);
        if (s + q < m && ws != 0.f) {  // 0: nothing visible, or too small to count
#pragma unroll
          for (int e = 0; e < E; ++e) acc[e] += ws * v[q].v[e];
        }
      }
    }
  }
  L = warp_sum(L);
  const bool any = M != -INFINITY;
  const float inv = any ? 1.f / L : 0.f;
  if (a.out != nullptr) {
    uint32_t w[E / 2];
#pragma unroll
    for (int e = 0; e < E; e += 2) w[e / 2] = pack_bf16(acc[e] * inv, acc[e + 1] * inv);
    uint32_t* dst = reinterpret_cast<uint32_t*>(a.out + query * D + lane * E);
#pragma unroll
    for (int e = 0; e < E / 2; ++e) dst[e] = w[e];
  }
  if (a.lse != nullptr && lane == 0) a.lse[((int64_t)b * a.H + h) * a.T + t] = any ? M + logf(L) : -INFINITY;
  if (a.joined_o != nullptr) {
#pragma unroll
    for (int e = 0; e < E; ++e) a.joined_o[query * D + lane * E + e] = acc[e];
    if (lane == 0) *reinterpret_cast<float2*>(a.joined_ml + 2 * query) = make_float2(M, L);
  }
}

// Shared memory of a kernel, and the whole of an SM's for it: an SM only runs CTAs of two kernels side
// by side under one split between L1 and shared memory.  Once per kernel and device.
cudaError_t prepare(const void* kernel, int bytes) {
  static std::mutex mu;
  static auto* done = new std::map<std::pair<const void*, int>, int>();  // never freed
  int dev = 0;
  PRA_RETURN_IF_ERROR(cudaGetDevice(&dev));
  std::lock_guard<std::mutex> lock(mu);
  int& have = (*done)[{kernel, dev}];
  if (have >= bytes) return cudaSuccess;
  PRA_RETURN_IF_ERROR(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  PRA_RETURN_IF_ERROR(cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
  have = bytes;
  return cudaSuccess;
}

bool encode(CUtensorMap* map, const void* base, int64_t cols, int64_t rows, int64_t row, int64_t batches, int64_t batch,
            int keys) {
  const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)batches};
  const cuuint64_t strides[2] = {(cuuint64_t)row * 2, (cuuint64_t)batch * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)keys, 1}, elem[3] = {1, 1, 1};
  return cuTensorMapEncodeTiled(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box,
                                elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int rows_of(const PrefixAttnArgs& a) { return (a.packed ? a.B : 1) * a.T * (a.H / a.Hkv); }

template <int D, int NT>
cudaError_t launch(const PrefixAttnArgs& a, cudaStream_t st) {
  using C = Cfg<D, NT>;
  CUtensorMap pk, pv, k, v;
  const int64_t width = (int64_t)a.Hkv * D;
  bool ok = true;
  if (a.use_prefix)
    ok = encode(&pk, a.pk, width, a.P, a.pk_row, 1, a.pk_row * a.P, BN) && encode(&pv, a.pv, width, a.P, a.pv_row, 1, a.pv_row * a.P, BN);
  if (a.use_own)
    ok = ok && encode(&k, a.k, width, a.cap, a.k_row, a.B, a.k_batch, BN) && encode(&v, a.v, width, a.cap, a.v_row, a.B, a.v_batch, BN);
  if (!ok) return cudaErrorInvalidValue;
  if (!a.use_prefix) pk = k, pv = v;
  if (!a.use_own) k = pk, v = pv;
  PRA_RETURN_IF_ERROR(prepare(reinterpret_cast<const void*>(prefix_kernel<D, NT>), C::SMEM));
  const int tiles = (rows_of(a) + NT * BM - 1) / (NT * BM);
  const int64_t items = (int64_t)tiles * a.Hkv * (a.packed ? 1 : a.B);
  const int64_t ctas = a.whole > 0 ? a.whole + (items - a.whole) * a.splits : items;
  if (ctas > INT32_MAX || a.splits > 65535 || a.whole < 0 || a.whole > items) return cudaErrorInvalidValue;
  const dim3 grid((unsigned)ctas, a.whole > 0 ? 1 : a.splits);
  if (a.after_prefix) return pra_launch_pdl(prefix_kernel<D, NT>, grid, dim3(C::THREADS), C::SMEM, st, pk, pv, k, v, a);
  prefix_kernel<D, NT><<<grid, C::THREADS, C::SMEM, st>>>(pk, pv, k, v, a);
  return cudaGetLastError();
}

// Two tiles per CTA read every key block once for 256 queries; one tile leaves room for two CTAs per SM.  Row by
// row two are 2 to 16% faster where they are full, or where there is less than a wave of them (4 x 600 query rows
// behind 16K 112 us, with one 137); one is where the second of the last pair would be empty (122 x 324, head dim 64:
// 472 -> 344 us).
int tiles_per_cta(const PrefixAttnArgs& a) {
  const int64_t rows = rows_of(a), ones = (rows + BM - 1) / BM, pairs = (ones + 1) / 2;
  int dev = 0, sms = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (!a.packed && ones * 115 < 2 * pairs * 100 && pairs * a.Hkv * a.B > sms) return 1;
  return rows > BM ? 2 : 1;
}

}  // namespace prefix
}  // namespace pra

void pra_prefix_attention_shape(const PrefixAttnArgs& a, int* tiles, int* slots, int* tile_rows) {
  using namespace pra::prefix;
  const int nt = tiles_per_cta(a);
  if (tile_rows != nullptr) *tile_rows = nt * BM;
  *tiles = (rows_of(a) + nt * BM - 1) / (nt * BM) * a.Hkv * (a.packed ? 1 : a.B);
  int dev = 0, sms = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  *slots = sms * (nt == 2 ? 1 : 2);
}

cudaError_t pra_prefix_attention(const PrefixAttnArgs& a, cudaStream_t st) {
  using namespace pra::prefix;
  if (a.B == 0 || a.T == 0) return cudaSuccess;
  if ((!a.use_prefix && !a.use_own) || (a.packed && a.use_own) || a.H % a.Hkv || a.splits < 1) return cudaErrorInvalidValue;
  const int nt = tiles_per_cta(a);
  if (a.D == 128) return nt == 2 ? launch<128, 2>(a, st) : launch<128, 1>(a, st);
  if (a.D == 64) return nt == 2 ? launch<64, 2>(a, st) : launch<64, 1>(a, st);
  return cudaErrorInvalidValue;
}

namespace pra {
namespace prefix {

template <int D, int NB>
cudaError_t launch_own(const OwnAttnArgs& a, cudaStream_t st) {
  using C = OwnCfg<D>;
  CUtensorMap k, v;
  const int64_t width = (int64_t)a.Hkv * D;
  if (!encode(&k, a.k, width, a.cap, a.k_row, a.B, a.k_batch, OB) || !encode(&v, a.v, width, a.cap, a.v_row, a.B, a.v_batch, OB))
    return cudaErrorInvalidValue;
  const int smem = C::smem(a.T * (a.H / a.Hkv));
  PRA_RETURN_IF_ERROR(prepare(reinterpret_cast<const void*>(own_kernel<D, NB>), smem));
  return pra_launch_pdl(own_kernel<D, NB>, dim3(a.ctas), dim3(C::THREADS), smem, st, k, v, a);
}

}  // namespace prefix
}  // namespace pra

int pra_own_attention_ctas(const OwnAttnArgs& a) {
  int dev = 0, sms = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const int rows = a.T * (a.H / a.Hkv);
  const int smem = a.D == 128 ? pra::prefix::OwnCfg<128>::smem(rows) : pra::prefix::OwnCfg<64>::smem(rows);
  const int per_sm = smem <= 113 * 1024 ? 2 : 1;
  // no more CTAs than blocks there can be
  const int64_t most = (int64_t)a.B * a.Hkv * ((a.cap + pra::prefix::OB - 1) / pra::prefix::OB);
  return (int)std::max<int64_t>(1, std::min<int64_t>(per_sm * sms, most));
}

cudaError_t pra_own_attention(const OwnAttnArgs& a, cudaStream_t st) {
  using namespace pra::prefix;
  if (a.B == 0 || a.T == 0) return cudaSuccess;
  if (a.cap < 1 || a.H % a.Hkv || a.T * (a.H / a.Hkv) > PRA_OWN_ROWS || a.ctas < 1) return cudaErrorInvalidValue;
  const bool few = a.T * (a.H / a.Hkv) <= 8;
  if (a.D == 128) return few ? launch_own<128, 1>(a, st) : launch_own<128, 2>(a, st);
  if (a.D == 64) return few ? launch_own<64, 1>(a, st) : launch_own<64, 2>(a, st);
  return cudaErrorInvalidValue;
}

cudaError_t pra_prefix_merge(const PrefixMergeArgs& a, cudaStream_t st) {
  using namespace pra::prefix;
  const int64_t rows = a.tiles > 0 ? (int64_t)a.tiles * a.tile_rows : (int64_t)a.B * a.T * a.H;
  if (rows == 0) return cudaSuccess;
  const int64_t blocks = (rows + MERGE_WARPS - 1) / MERGE_WARPS;
  if (blocks > INT32_MAX) return cudaErrorInvalidValue;
  const dim3 grid((unsigned)blocks), block(MERGE_WARPS * 32);
  const bool many = (a.part_o != nullptr ? a.n_slots : 0) + (a.more_o != nullptr ? a.n_more : 0) > 8;
  if (a.D == 128) return pra_launch_pdl(many ? merge_kernel<128, 16> : merge_kernel<128, 8>, grid, block, 0, st, a);
  if (a.D == 64) return pra_launch_pdl(many ? merge_kernel<64, 16> : merge_kernel<64, 8>, grid, block, 0, st, a);
  return cudaErrorInvalidValue;
}
