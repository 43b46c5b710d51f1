// Launchers of a ragged batch's operators: rows appended to paged caches with
// their rotation, several prompts' attention, 8-bit projections, sampling. As
// kernels.hpp's: each enqueues on `stream` and returns without synchronising.
#pragma once

#include "serving.hpp"

namespace mi
{

  // ---- rows into paged caches (append.hip) --------------------------------------------
  // A sequence whose cache the host holds: `rows` consecutive rows from position
  // `start` on; `pages` its page table (device addresses), or null where the
  // rows go into pages by another launch.
  struct AppendSequence
  {
    const unsigned long long *pages;
    int page_count;
    int rows;
    int start;
  };
  constexpr int kAppendHeld = 32; // sequences that go in one launch's arguments

  struct AppendRows
  {
    const void *q; // (rows, heads, head_dim) fp16, strides in elements (0: contiguous)
    const void *k; // (rows, kv_heads, head_dim)
    const void *v;
    void *q_out; // contiguous; k_out, v_out may be null
    void *k_out;
    void *v_out;
    long long q_stride;
    long long k_stride;
    long long v_stride;
    // The tables on the device: (batch, max_pages) and (batch), offsets
    // (batch + 1), or null where every sequence has one row; or `held`, `batch`
    // sequences in host memory.
    const unsigned long long *pages;
    const std::uint8_t *tiers;
    const int *lengths;
    const int *offsets;
    const AppendSequence *held;
    int batch;
    int max_pages;
    int page_tokens;
    int rows;
    int heads;
    int kv_heads;
    int head_dim;
    const float *table; // (positions, rotary / 2) cos and sin; null: nothing turns
    int table_positions;
    int rotary; // channels of a head that turn
    bool interleaved; // pairs (2j, 2j + 1), else (j, j + rotary / 2)
  };
  void launch_append(const AppendRows &t, hipStream_t stream);
  // What launch_append refuses, with no launch.
  void check_append(const AppendRows &t);
  // (positions, pairs) cos and sin, times `magnitude`, of position * frequencies[pair].
  void launch_rope_frequencies(float *table, int positions, const double *frequencies, int pairs,
                               double magnitude, hipStream_t stream);

  // ---- several prompts' attention (packed.hip) -----------------------------------------
  struct PackedAttention
  {
    const void *q; // (rows_q, heads, head_dim) fp16
    const void *k; // (rows_k, kv_heads, head_dim)
    const void *v;
    void *out; // (rows_q, heads, head_dim), contiguous
    long long q_stride;
    long long k_stride;
    long long v_stride;
    const int *offsets_q; // (batch + 1) on the device
    const int *offsets_k; // null: offsets_q
    int batch;
    int rows_q;
    int rows_k;
    int heads;
    int kv_heads;
    int head_dim;
    // Null: no row's keys are split over workgroups; else at least
    // packed_attention_floats, used until the launch is done.
    float *partials;
    std::size_t partials_floats;
  };
  std::size_t packed_attention_floats(const PackedAttention &t);
  void launch_packed_attention(const PackedAttention &t, hipStream_t stream);

  // ---- 8-bit rows and weights (int8.hip) -------------------------------------------------
  // Rows (rows, features) fp16, `stride` elements apart (0: features), as codes
  // (rows, features) of a byte and an fp32 scale a row.
  void launch_quantise_rows_int8(const void *x, long long stride, void *codes, float *scales,
                                 int rows, int features, hipStream_t stream);
  struct Int8Linear
  {
    const void *x; // (rows, in) codes
    const float *x_scales;
    const void *w; // (out, in) codes
    const float *w_scales;
    const void *bias; // (out) fp16, or null; none where the output is fp32
    void *out;
    const float *residual; // null: out is fp16; else out (rows, out) fp32 = residual + x W^T
    int rows;
    int in;
    int features;
  };
  void launch_linear_int8(const Int8Linear &t, hipStream_t stream);

  // ---- a token of every row of logits (sample.hip) ----------------------------------------
  struct Sampling
  {
    const void *logits; // (rows, vocab), `stride` elements apart (0: vocab)
    bool half;          // fp16, else fp32
    long long stride;
    const float *uniforms;     // (rows)
    const float *temperature;  // (rows) each, or null
    const int *top_k;
    const float *top_p;
    const float *min_p;
    int *tokens;
    int rows;
    int vocab;
    void *scratch; // sample_scratch_floats
    std::size_t scratch_floats;
  };
  std::size_t sample_scratch_floats(int rows, int vocab);
  void launch_sample(const Sampling &t, hipStream_t stream);

} // namespace mi
