// Host-visible parameter blocks and launch entry points of the serving operators: rotary
// positions, attention over a shared prefix, rules on logits.  Pure C++ (no torch).
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

enum : int { PRA_BF16 = 0, PRA_FP16 = 1, PRA_FP32 = 2 };

// ---- rotary positions (rotary.cu) --------------------------------------------------------
struct RotarySegment {  // some heads of every token (queries, keys or values)
  const void* src;      // head h of token m at src + m * src_token + h * src_head (elements)
  void* dst;            // head h of token m at dst + row * dst_token + h * dst_head
  int64_t src_token, src_head, dst_token, dst_head;
  int heads;            // 0: no such segment
  int rotate;           // 0: a plain copy (values)
  int to_slot;          // 1: row = slots[m] (a cache), 0: row = m
};
struct RotaryArgs {
  RotarySegment seg[3];
  int64_t tokens;
  const void* pos;      // [tokens] int32 or int64
  int pos64;
  const float* cos_t;   // [max_pos, rot / 2]
  const float* sin_t;
  int64_t max_pos;      // a position outside [0, max_pos) gives NaN in the rotated part
  const int* slots;     // [tokens] cache rows or null; outside [0, slot_rows): not written
  int64_t slot_rows;
  int head_dim, rot;    // both even, rot <= head_dim
  int interleaved, inverse;
};
cudaError_t pra_rotary(const RotaryArgs& a, int dtype, cudaStream_t stream);

// ---- rules on logits (logits.cu) ---------------------------------------------------------
constexpr int PRA_RULES_MAX_BIASES = 2047;         // entries of one row's bias list (11 bits of a table word)
constexpr int64_t PRA_RULES_MAX_HISTORY = 1 << 20;  // history capacity (20-bit counts)
constexpr int64_t PRA_RULES_MAX_VOCAB = 384 * 1024;  // columns of a call with a history or biases
struct LogitsArgs {
  const void* logits;      // [B, V] rows at stride in_stride
  void* out;               // [B, V] rows at stride out_stride, same type (may be logits), or null
  int64_t in_stride, out_stride;
  int B, V, vocab_start;   // logits cover token ids [vocab_start, vocab_start + V); vocab_start % 8 == 0
  const int* ids;          // [B, capacity] token history (rows at ids_stride) or null
  int64_t ids_stride;
  int capacity;
  int* hist_len;           // [B] valid ids of each row
  const int* prompt_len;   // [B] leading ids that are prompt (repetition only), or null: none
  const float* repetition; // [B] or null
  const float* presence;
  const float* frequency;
  const int* bias_ids;     // [B, n_bias] or null; ids outside the vocabulary are skipped
  const float* bias_values;
  int n_bias;
  const uint32_t* mask;    // [mask_count, mask_words] bit t: token id t is allowed
  int mask_count;
  int64_t mask_words;      // 0: no mask
  const int* mask_rows;    // [B] mask of each row (negative: no mask) or null: mask b
  int64_t* token;          // [B] greedy token ids or null
  float* value;            // [B] their processed logits
  int* append_ids;         // the history again when the chosen token is appended to it, or null
};
cudaError_t pra_logits_rules(const LogitsArgs& a, int dtype, cudaStream_t stream);

// ---- attention over a shared prefix (prefix_attn.cu) -------------------------------------
// One softmax over [prefix keys (the same for every batch row) ; the row's own keys (causal)].
// Query (b, t) is the token at own position len[b] - T + t: it sees the first prefix_len[b] prefix keys
// and own keys 0 .. that position.  A launch covers the prefix, the own keys, or both:
//   packed:  query rows (b, t, g) of one KV head are numbered across the batch (prefix only)
//   else:    query rows (t, g) of one batch row and KV head
struct PrefixAttnArgs {
  const __nv_bfloat16* q;         // query (b, t), head h at q + b * q_batch + t * q_token + h * D
  int64_t q_batch, q_token;
  const __nv_bfloat16* pk;        // prefix key j, KV head h at pk + j * pk_row + h * D
  const __nv_bfloat16* pv;
  int64_t pk_row, pv_row;
  int P;                          // prefix rows
  const int* prefix_len;          // [B] or null: P
  const __nv_bfloat16* k;         // own key j of row b, KV head h at k + b * k_batch + j * k_row + h * D
  const __nv_bfloat16* v;
  int64_t k_batch, k_row, v_batch, v_row;
  int cap;                        // own rows per batch row
  const int* len;                 // [B], clamped to [0, cap]
  int B, T, H, Hkv, D;
  float scale;
  int packed, use_prefix, use_own;
  int splits;                     // CTAs along the keys of one query tile
  int whole;                      // > 0: that many tiles take all their keys, to out; the tiles behind are split
  int slot0, n_slots;             // partial s of this launch goes to slot slot0 + s of n_slots
  float* part_o;                  // [B * T, H, n_slots, D] unnormalised, or null: write out / lse (with `whole`
                                  // [tiles behind it * tile rows, n_slots, D])
  float* part_ml;                 // [B * T, H, n_slots, 2] (maximum in natural-log units, sum)
  __nv_bfloat16* out;             // [B, T, H * D] contiguous
  float* lse;                     // [B, H, T] or null
  int* status;                    // set to 1 by a CTA that gave up on a bounded wait
  int give_up;                    // > 0: the producer of every CTA gives up in front of its give_up-th copy
  int after_prefix;               // the launch before it on the stream is such a one, on whose results it does not wait
};
cudaError_t pra_prefix_attention(const PrefixAttnArgs& a, cudaStream_t stream);
// Query tiles of a launch (CTAs before splitting), how many run at once (for choosing splits), rows of a tile.
void pra_prefix_attention_shape(const PrefixAttnArgs& a, int* tiles, int* slots, int* tile_rows = nullptr);

// The own keys of rows with few queries (T * H / Hkv <= PRA_OWN_ROWS per KV head), which a 128-row tile would
// leave mostly empty: every (batch row, KV head) is an item of ceil(len / 64) blocks (at least one), the
// CTAs take equal runs of the blocks of all items, and an item that several CTAs share has a piece in
// each.  CTA c's piece of item i is piece i + c: pieces of an item follow one another.
constexpr int PRA_OWN_ROWS = 16;
struct OwnAttnArgs {
  const __nv_bfloat16* q;         // as in PrefixAttnArgs
  int64_t q_batch, q_token;
  const __nv_bfloat16* k;
  const __nv_bfloat16* v;
  int64_t k_batch, k_row, v_batch, v_row;
  int cap;
  const int* len;
  int B, T, H, Hkv, D;
  float scale;
  int ctas;                       // grid
  int after_prefix;               // the launch before it on the stream is pra_prefix_attention's
  float* piece_o;                 // [B * Hkv + ctas, T * G, D] unnormalised
  float* piece_ml;                // [B * Hkv + ctas, T * G, 2]
  int* first;                     // [B * Hkv] first and last CTA of each item
  int* last;
  int* status;
  int give_up;                    // as in PrefixAttnArgs
};
int pra_own_attention_ctas(const OwnAttnArgs& a);
cudaError_t pra_own_attention(const OwnAttnArgs& a, cudaStream_t stream);

// out / lse, or the joined partial, from the partials of every (b, t, h).
struct PrefixMergeArgs {
  int B, T, H, Hkv, D;
  int tile0, tiles, tile_rows;    // tiles > 0: only the queries of tiles tile0 .. tile0 + tiles - 1 of the attention launch,
  int packed;                     // whose parts are [tiles * tile_rows, n_slots, D]; its `packed`
  const float* part_o;            // [B * T, H, n_slots, D] and (max, sum) pairs, or null
  const float* part_ml;
  int n_slots;
  const float* more_o;            // a second such set [B * T, H, n_more, D], or null
  const float* more_ml;
  int n_more;
  const float* piece_o;           // pieces of pra_own_attention, or null
  const float* piece_ml;
  const int* first;
  const int* last;
  __nv_bfloat16* out;             // [B, T, H * D] or null
  float* lse;                     // [B, H, T] or null
  float* joined_o;                // [B * T, H, D] unnormalised or null
  float* joined_ml;               // [B * T, H, 2]
};
cudaError_t pra_prefix_merge(const PrefixMergeArgs& a, cudaStream_t stream);
