// What the attentions over contiguous keys and values (window.hip, packed.hip)
// have in common: 32 x 32 matrix tiles of scores with the keys as M and the rows
// as N, the places of a step's rows in LDS, V read transposed from there.
#pragma once

#include "common.hpp"
#include "lane_ops.hpp"

namespace mi::attention_tiles
{
  typedef _Float16 half8 __attribute__((ext_vector_type(8)));
  typedef _Float16 half4 __attribute__((ext_vector_type(4)));
  typedef _Float16 half2v __attribute__((ext_vector_type(2)));
  typedef float f32x16 __attribute__((ext_vector_type(16)));
  typedef float f32x4 __attribute__((ext_vector_type(4)));
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
  typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
  typedef short i16x4 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) i16x4 *lds_i16x4;
  typedef __attribute__((address_space(3))) void *lds_void;
  typedef const __attribute__((address_space(1))) void *global_void;

  constexpr float kRise = 6.0f;
  constexpr float kProb = 8.0f; // P x 2^8
  constexpr float kProbUnscale = 1.0f / 256.0f;

  __device__ inline half8 as_half8(u32x4 v) { return __builtin_bit_cast(half8, v); }

  __device__ inline f32x16 mfma32(half8 a, half8 b, f32x16 c)
  {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }

  // Piece c (16 bytes) of row t of a tile in LDS lies at place c ^ swizzle(t), so
  // that lanes which read a piece of many rows meet no bank twice: for rows of 8
  // pieces two rows span the banks, so rows differ by t / 2; bits reversed, so that rows 0-3
  // of a transposing read differ in the bits its four pieces do not use.
  template <int HD>
  __device__ inline int swizzle(int t)
  {
    if constexpr (HD == 64)
    {
      const int u = t >> 1;
      return ((u & 1) << 2) | (u & 2) | ((u >> 2) & 1);
    }
    else
    {
      return ((t & 1) << 3) | ((t & 2) << 1) | ((t >> 1) & 2) | ((t >> 3) & 1);
    }
  }

  // Four keys of the lane's channel: the 16 lanes of a row group address
  // four rows' 16 channels (lane s: row s / 4, channels 4 (s % 4) ..) and
  // lane s receives channel s of the four.
  __device__ inline half4 transposed(const std::uint16_t *p)
  {
    return __builtin_bit_cast(half4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4)(p)));
  }

  __device__ inline bool is_finite(std::uint16_t v) { return (v & 0x7c00u) != 0x7c00u; }

  // Zeros where a value is not finite.
  __device__ inline half8 finite_only(half8 v)
  {
    u32x4 bits = __builtin_bit_cast(u32x4, v);
#pragma unroll
    for (int w = 0; w < 4; ++w)
    {
      const unsigned word = bits[w];
      bits[w] = (is_finite(static_cast<std::uint16_t>(word)) ? word & 0xFFFFu : 0u) |
                (is_finite(static_cast<std::uint16_t>(word >> 16)) ? word & 0xFFFF0000u : 0u);
    }
    return as_half8(bits);
  }

  // Whether every value of a step is finite.
  template <int HD, int kKeys>
  __device__ inline bool finite_values(const std::uint16_t *values, int lane)
  {
    bool fine = true;
#pragma unroll 4
    for (int i = 0; i < kKeys * HD / 512; ++i)
    {
      const u32x4 x = *reinterpret_cast<const u32x4 *>(values + 512 * i + 8 * lane);
#pragma unroll
      for (int w = 0; w < 4; ++w)
      {
        const unsigned word = x[w];
        fine = fine && is_finite(static_cast<std::uint16_t>(word)) &&
               is_finite(static_cast<std::uint16_t>(word >> 16));
      }
    }
    return __all(fine);
  }

  // A wave's 32 rows: weights are 2^(score - m), l is their sum, o x 2^kProb.
  template <int HD>
  struct Rows
  {
    float m;
    float l;
    f32x16 o[HD / 32];
  };
} // namespace mi::attention_tiles
