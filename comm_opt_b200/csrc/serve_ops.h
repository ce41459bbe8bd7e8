// Host entry points of the rotary, tree-attention and logits operators (plain CUDA, no torch types).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace cob {

// A [batch, seq, heads, D] operand: element strides of batch, sequence and head, components contiguous.
struct HeadView {
  const void* p = nullptr;
  long long sb = 0, ss = 0, sh = 0;
  int heads = 0;
};

// Rotary positions of up to two operands (queries and keys) sharing the positions, optionally after an RMSNorm
// of every head; the append form also takes v and writes k and v into the paged caches.
struct RotaryParams {
  HeadView in[3];      // q, k, v (v: append form only); heads = 0 leaves one out
  HeadView out[2];     // q, k; the append form writes k and v into the caches instead of out[1]
  HeadView grad[2];    // backward: gradients of q and k outputs
  const void* w[2] = {nullptr, nullptr};  // norm weights [D] of q and k, both or neither
  int w_f32 = 0;       // weights are fp32 (else of the operands' type)
  const void* bias = nullptr;             // append form: [(nq + nk + nv) * D] of the operands' type
  const int32_t* pos = nullptr;           // positions, element strides (pos_sb, pos_ss)
  long long pos_sb = 0, pos_ss = 0;
  const float* cos_t = nullptr;           // [max_pos, rot / 2]
  const float* sin_t = nullptr;
  int max_pos = 0, rot = 0, D = 0, batch = 0, seq = 0;
  int interleaved = 0;  // pairs (2j, 2j + 1); else (j, j + rot / 2)
  int inverse = 0;      // the transpose: sines negated (the gradient of a rotation)
  float eps = 0.f;
  // append form
  int append = 0;
  const int32_t* block_tables = nullptr;  // [batch, max_blocks]
  const int32_t* starts = nullptr;        // [batch] cache slot of a sequence's first row
  const int32_t* lens = nullptr;          // [batch] valid rows, or nullptr: all
  void* k_cache = nullptr;                // [num_blocks, nkv, 16, D]
  void* v_cache = nullptr;
  int max_blocks = 0, num_blocks = 0;
  int dtype = 0;
};
cudaError_t rotary_forward(const RotaryParams& p, cudaStream_t s);
// Backward of norm + rotation: grad -> out (gradients of q and k), and the weight gradients of q and k in `dw`
// (two [D] rows of the weights' type). `ws` holds rotary_backward_blocks(p) rows of D floats.
int rotary_backward_blocks(const RotaryParams& p);
cudaError_t rotary_norm_backward(const RotaryParams& p, float* ws, void* dwq, void* dwk, cudaStream_t s);

// Penalties, biases and grammar masks on the logits of a vocabulary shard, row by row:
//   seen before:  x = x > 0 ? x / repetition : x * repetition
//   c times in the output (c > 0):  x -= frequency * c, x -= presence
//   x += sum of the row's biases of this id;  not allowed by the grammar: x = -inf
// in fp32, rounded once to the logits' type.
struct LogitsParams {
  const void* logits = nullptr;  // [rows, vocab], row stride ld_in
  void* out = nullptr;           // [rows, vocab], row stride ld_out (may be the logits)
  long long ld_in = 0, ld_out = 0;
  int rows = 0, vocab = 0, vocab_offset = 0;
  const int32_t* tokens = nullptr;  // [rows, history], row stride ld_tokens; global ids, others are skipped
  long long ld_tokens = 0;
  int history = 0;
  const int32_t* lens = nullptr;         // [rows] tokens of each row, or nullptr: all
  const int32_t* prompt_lens = nullptr;  // [rows] how many of them are the prompt's, or nullptr: none
  const float* repetition = nullptr;     // [rows] each, or nullptr: no such penalty
  const float* frequency = nullptr;
  const float* presence = nullptr;
  const int32_t* bias_ids = nullptr;     // [rows, biases] global ids, others are skipped
  const float* bias = nullptr;
  int biases = 0;
  const uint32_t* allowed = nullptr;     // [rows, mask_words]: bit i % 32 of word i / 32 is global id i
  long long ld_mask = 0;
  unsigned long long* keys = nullptr;    // [rows] greedy keys (see argmax_local), folded with atomicMax
  int dtype = 0;
};
cudaError_t penalize_logits(const LogitsParams& p, cudaStream_t s);

// Attention of drafted tokens over a paged cache: row t of sequence b sees the cache slots [0, ctx[b]) and, of the
// drafted tokens (cached in slots ctx[b] + j), those whose bit j is set in mask[b, t]. Rows that see nothing are
// zeros; rows t >= tree_lens[b] are left as they were.
struct TreeAttnParams {
  const void* q = nullptr;  // [batch, tree, nq, D], element strides q_sb, q_st, q_sh
  long long q_sb = 0, q_st = 0, q_sh = 0;
  void* out = nullptr;      // [batch, tree, nq, D], element strides o_sb, o_st, o_sh
  long long o_sb = 0, o_st = 0, o_sh = 0;
  const void* k_cache = nullptr;  // [num_blocks, nkv, 16, D]
  const void* v_cache = nullptr;
  const int32_t* block_tables = nullptr;  // [batch, max_blocks]
  const int32_t* ctx_lens = nullptr;      // [batch]
  const int32_t* tree_lens = nullptr;     // [batch] or nullptr: all rows
  const int64_t* mask = nullptr;          // [batch, tree], batch stride mask_sb (0: one mask for all); nullptr: a chain
  long long mask_sb = 0;
  int batch = 0, tree = 0, nq = 0, nkv = 0, head_dim = 0, max_blocks = 0, num_blocks = 0;
  float scale = 1.f;
  unsigned long long timeout_ns = 1000000000ull;  // of every wait inside the kernel; 0: gives up before its first wait
  int dtype = 0;
};
// Where a wait runs out, the rows that were still owed become NaN and the current device's word (its address in *word)
// is set to 1 until the host clears it.
cudaError_t tree_attention_error_word(int** word);
// `scratch`: tree_attention_scratch_bytes(p) bytes, 16-byte aligned, of this call alone; any content.
size_t tree_attention_scratch_bytes(const TreeAttnParams& p);
cudaError_t tree_attention(const TreeAttnParams& p, void* scratch, cudaStream_t s);

}  // namespace cob
