// Launchers of the serving operators' kernels: 4-bit projections, a batch's
// token attention, a prompt's window attention. As kernels.hpp's: each
// enqueues on `stream` and returns without synchronising.
#pragma once

#include "common.hpp"

#include <cstddef>
#include <cstdint>

namespace mi
{

  // ---- what a launch may not write over ----------------------------------------------
  // Memory that a launch reads or writes: `bytes` from `at`, or rows of them
  // `stride` bytes apart. (Null, or no bytes: none.)
  struct Extent
  {
    const void *at;
    std::size_t bytes;
    std::size_t rows = 1;
    std::size_t stride = 0;
  };
  // Whether `a`, one run of bytes, shares a byte with some row of `b`.
  inline bool overlaps(const Extent &a, const Extent &b)
  {
    if (a.at == nullptr || b.at == nullptr || a.bytes == 0 || b.bytes == 0 || b.rows == 0)
    {
      return false;
    }
    const auto from = reinterpret_cast<std::uintptr_t>(a.at), to = from + a.bytes;
    const auto first = reinterpret_cast<std::uintptr_t>(b.at);
    // The first row that ends behind `from`.
    std::size_t row = 0;
    if (first + b.bytes <= from && b.stride > 0)
    {
      row = (from - first - b.bytes) / b.stride + 1;
    }
    return row < b.rows && first + row * b.stride + b.bytes > from && first + row * b.stride < to;
  }

  // ---- 4-bit weights (int4.hip) -----------------------------------------------------
  // A weight (out, in) as codes (out, in / 2) bytes, two a byte, the first in
  // the low bits, and fp16 scales and zeros (out, in / group): group 32, 64
  // or 128, codes and weight 16-byte aligned. Weights are finite.
  void launch_quantise_int4(const void *weight, void *codes, void *scales, void *zeros, int group,
                            int in_features, int out_features, hipStream_t stream);
  // out (rows, out) fp16 = x (rows, in) W^T + bias (may be null), rounded
  // once; or out (rows, out) fp32 += x W^T. x 16-byte aligned.
  void launch_linear_int4(const void *x, const void *codes, const void *scales, const void *zeros,
                          int group, const void *bias, void *out, int rows, int in_features,
                          int out_features, hipStream_t stream);
  void launch_linear_int4_accumulate(const void *x, const void *codes, const void *scales,
                                     const void *zeros, int group, float *out, int rows,
                                     int in_features, int out_features, hipStream_t stream);

  // ---- one token of every sequence of a batch (batch.hip) --------------------------
  // A sequence whose cache the host holds: its page table's row, and where a
  // cache that seals keeps the token's own page (`open` null: in the table).
  struct BatchSequence
  {
    const unsigned long long *pages;
    const std::uint8_t *tiers;
    const std::uint16_t *open; // the page being filled: 32 key rows, 32 value rows
    const std::uint16_t *own_k;
    const std::uint16_t *own_v;
    int length;
  };
  constexpr int kBatchHeld = 32; // sequences that go in one launch's arguments

  struct BatchAttention
  {
    const void *q; // (batch, heads, head_dim) fp16
    void *out;
    // The tables on the device, (batch, max_pages) and (batch); or `held`,
    // `batch` sequences in host memory.
    const unsigned long long *pages;
    const std::uint8_t *tiers;
    const int *lengths;
    const BatchSequence *held;
    int batch;
    int max_pages;
    int page_tokens;
    int heads;
    int kv_heads;
    int head_dim;
    int window; // the last tokens visible; 0: every one
    int sinks;  // the first tokens visible beside a window's
    float *mass; // (batch, heads, max_pages), or null
    // Null: a workgroup a sequence and KV heads, no masses; else at least
    // batch_attention_floats, used until the launch is done.
    float *partials;
    std::size_t partials_floats;
  };
  constexpr int kBatchPageTokens = 32;
  std::size_t batch_attention_floats(const BatchAttention &t, bool with_mass);
  void launch_batch_attention(const BatchAttention &t, hipStream_t stream);

  // ---- a prompt through a sliding window (window.hip) --------------------------------
  struct WindowAttention
  {
    const void *q; // (seq_q, heads, head_dim) fp16, the last of k's positions
    const void *k; // (seq_k, kv_heads, head_dim)
    const void *v;
    void *out; // (seq_q, heads, head_dim), contiguous
    long long q_stride; // elements between tokens; 0: contiguous
    long long k_stride;
    long long v_stride;
    int seq_q;
    int seq_k;
    int heads;
    int kv_heads;
    int head_dim;
    int window; // the last tokens visible, the query's own counted; 0: every one
    int sinks;  // the first tokens visible beside a window's
    // Null: no row's keys are split over workgroups; else at least
    // window_attention_floats, used until the launch is done.
    float *partials;
    std::size_t partials_floats;
  };
  std::size_t window_attention_floats(const WindowAttention &t);
  void launch_window_attention(const WindowAttention &t, hipStream_t stream);

} // namespace mi
