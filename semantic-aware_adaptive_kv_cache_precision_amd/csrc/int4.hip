// Projections through 4-bit weights: the quantiser that makes them and
// y = x W^T for the rows of a decode step or a few sequences' steps.
//
// A weight (out, in) is held as codes (out, in / 2) bytes, two a byte, the
// first in the low bits, and a scale and a zero in fp16 for every `group`
// consecutive inputs of a row (group 32, 64 or 128). The rule is the page
// quantiser's: zero the group's least value, scale the least fp16 with
// 15 scale >= range, code = rint((w - zero) / scale). A weight stands for
// code * scale + zero, not rounded again, so that
//   y = sum over groups of scale (x . codes) + zero sum(x).
//
// linear_int4_kernel. A wave takes tiles of 16 outputs: the matrix cores form
// x . codes (A: 16 rows of x, B: the codes as fp16 integers, exact) and
// sum(x) (B: ones) of a group in fp32, 32 inputs an instruction, and two fmas
// an output scale them. Nothing is rounded before the one rounding of y. A
// lane reads its row's codes straight from memory, 16 bytes at a time
// where the group is 128 (8 at 64, 4 at 32: an instruction's four lane groups
// must lie in one group of the weight); x goes through LDS, a phase of inputs
// at a time. A code becomes fp16 by the mask that splices it under the
// exponent of 1024 (or, four bits up, 1024 + 16 code), nine instructions for
// eight; this leaves them in the order 0 4 1 5 2 6 3 7, in which x is laid in
// LDS. A tile's inputs are split over up to eight waves, whose sums meet in
// LDS in wave order: the bits do not depend on timing.

#include "kernels.hpp"
#include "quant_core.hpp"

#include <algorithm>
#include <string>

namespace mi
{
  namespace
  {
    typedef _Float16 half8 __attribute__((ext_vector_type(8)));
    typedef _Float16 half2v __attribute__((ext_vector_type(2)));
    typedef float f32x4 __attribute__((ext_vector_type(4)));
    typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
    typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

    // ---- the quantiser ------------------------------------------------------

    // Eight weights a lane, Group / 8 lanes a group. Bound by memory: 2 bytes
    // read and a little over half of one written a weight.
    template <int Group>
    __global__ void __launch_bounds__(256)
        quantise_int4_kernel(const std::uint16_t *weight, unsigned *codes, std::uint16_t *scales,
                             std::uint16_t *zeros, std::size_t count)
    {
      constexpr int kLanes = Group / 8;
      const std::size_t i = static_cast<std::size_t>(blockIdx.x) * 256 + threadIdx.x;
      const bool live = i < count; // whole groups: their lanes are live together
      u32x4 raw = {0u, 0u, 0u, 0u};
      if (live)
      {
        raw = *reinterpret_cast<const u32x4 *>(weight + 8 * i);
      }
      float x[8];
#pragma unroll
      for (int w = 0; w < 4; ++w)
      {
        x[2 * w] = h2f(static_cast<std::uint16_t>(raw[w]));
        x[2 * w + 1] = h2f(static_cast<std::uint16_t>(raw[w] >> 16));
      }
      float lo = x[0], hi = x[0];
#pragma unroll
      for (int e = 1; e < 8; ++e)
      {
        lo = fminf(lo, x[e]);
        hi = fmaxf(hi, x[e]);
      }
#pragma unroll
      for (int offset = 1; offset < kLanes; offset *= 2)
      {
        lo = fminf(lo, __shfl_xor(lo, offset));
        hi = fmaxf(hi, __shfl_xor(hi, offset));
      }
      const std::uint16_t bits = quant_core::scale_bits_fast(lo, hi, 4);
      const float scale = h2f(bits);
      const float inv = scale == 0.0f ? 0.0f : 1.0f / scale;
      float zero8[8], scale8[8], inv8[8], q[8];
#pragma unroll
      for (int e = 0; e < 8; ++e)
      {
        zero8[e] = lo;
        scale8[e] = scale;
        inv8[e] = inv;
      }
      quant_core::quotients_of<4>(x, zero8, scale8, inv8, q);
      unsigned packed = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e)
      {
        packed |= (static_cast<unsigned>(q[e]) & 15u) << (4 * e);
      }
      if (live)
      {
        codes[i] = packed;
        if (i % kLanes == 0)
        {
          scales[i / kLanes] = bits;
          zeros[i / kLanes] = __half_as_ushort(__float2half(lo)); // exact: a weight's own value
        }
      }
    }

    // ---- the projection -----------------------------------------------------

    constexpr int kWaves = 8;
    constexpr int kThreads = 64 * kWaves;
    constexpr int kChunk = 128;               // inputs a wave takes at a time
    constexpr int kStageHalves = 24 * 1024;   // x in LDS: 48 KB, three workgroups a CU
    constexpr int kRowPad = 8;                // halves: 16 rows a read, no bank twice

    enum class Int4Out : int
    {
      kHalf,       // fp16, with the bias if there is one
      kAccumulate, // fp32, added to what is there
    };

    struct Int4Args
    {
      const std::uint16_t *x;
      const std::uint8_t *codes;
      const std::uint16_t *scales;
      const std::uint16_t *zeros;
      const std::uint16_t *bias;
      void *out;
      int rows;
      int in;
      int features;
      int groups;      // a row's
      int splits;      // waves a tile's inputs are split over: 1, 2, 4 or 8
      int phase;       // inputs of a phase, whole chunks
      int row_stride;  // of x in LDS, halves
    };

    // Eight codes, the first in the lowest bits, as fp16 in the order
    // 0 4 1 5 2 6 3 7.
    __device__ inline half8 codes_as_half(unsigned w)
    {
      constexpr unsigned kLow = 0x000F000Fu, kHigh = 0x00F000F0u, kExp = 0x64006400u;
      const _Float16 k1024 = static_cast<_Float16>(1024.0f);
      const _Float16 k64 = static_cast<_Float16>(64.0f);
      const _Float16 k16th = static_cast<_Float16>(0.0625f);
      const unsigned w8 = w >> 8;
      const auto low = [&](unsigned v) {
        return __builtin_bit_cast(half2v, (v & kLow) | kExp) - half2v{k1024, k1024};
      };
      const auto high = [&](unsigned v) { // (1024 + 16 code) / 16 - 64, exact
        return __builtin_elementwise_fma(__builtin_bit_cast(half2v, (v & kHigh) | kExp),
                                         half2v{k16th, k16th}, half2v{-k64, -k64});
      };
      const half2v a = low(w), b = high(w), c = low(w8), d = high(w8);
      return half8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
    }

    // A wave's part of a chunk of 128 inputs: FT tiles' codes, and the scales
    // and zeros of the lane's output (row), Words = group / 32.
    template <int Words, int FT>
    struct Fetched
    {
      static constexpr int kGroups = 4 / Words;
      unsigned w[FT][4];
      std::uint16_t s[FT][kGroups];
      std::uint16_t z[FT][kGroups];
    };

    template <int Words, int FT>
    __device__ inline void fetch(Fetched<Words, FT> &f, const Int4Args &a, const int (&row)[FT],
                                 int chunk, int g)
    {
      constexpr int kGroups = 4 / Words;
#pragma unroll
      for (int t = 0; t < FT; ++t)
      {
        const std::uint8_t *codes = a.codes + static_cast<std::size_t>(row[t]) * (a.in / 2);
        const std::size_t meta = static_cast<std::size_t>(row[t]) * a.groups;
#pragma unroll
        for (int h = 0; h < kGroups; ++h)
        {
          // (Past the row's last group: the first's, multiplied by zeros.)
          const int group = chunk * kGroups + h;
          const bool there = group < a.groups;
          const int at = there ? group : 0;
          const std::uint8_t *p = codes + (at * (32 * Words) + 8 * Words * g) / 2;
          if constexpr (Words == 4)
          {
            const u32x4 v = *reinterpret_cast<const u32x4 *>(p);
            f.w[t][0] = v.x;
            f.w[t][1] = v.y;
            f.w[t][2] = v.z;
            f.w[t][3] = v.w;
          }
          else if constexpr (Words == 2)
          {
            const u32x2 v = *reinterpret_cast<const u32x2 *>(p);
            f.w[t][2 * h] = v.x;
            f.w[t][2 * h + 1] = v.y;
          }
          else
          {
            f.w[t][h] = *reinterpret_cast<const unsigned *>(p);
          }
          f.s[t][h] = there ? a.scales[meta + at] : std::uint16_t{0};
          f.z[t][h] = there ? a.zeros[meta + at] : std::uint16_t{0};
        }
      }
    }

    template <int Words, int NT, int FT, Int4Out Out>
    __global__ void __launch_bounds__(kThreads) linear_int4_kernel(Int4Args a)
    {
      constexpr int kGroups = 4 / Words;
      extern __shared__ __align__(16) std::uint16_t x_lds[];
      const int lane = threadIdx.x & 63;
      const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
      const int n = lane & 15;
      const int g = lane >> 4;
      const int split = wave % a.splits;
      const int tiles = kWaves / a.splits * FT; // of 16 outputs a workgroup
      const int tile0 = (static_cast<int>(blockIdx.x) * tiles + wave / a.splits * FT) * 16;
      const int row0 = static_cast<int>(blockIdx.y) * 16 * NT;
      const int rows = min(a.rows - row0, 16 * NT);
      const std::uint16_t *x = a.x + static_cast<std::size_t>(row0) * a.in;

      int row[FT];
#pragma unroll
      for (int t = 0; t < FT; ++t)
      {
        row[t] = min(tile0 + 16 * t + n, a.features - 1);
      }
      int at[NT]; // the lane's row of x in LDS (a row past the last repeats it)
#pragma unroll
      for (int t = 0; t < NT; ++t)
      {
        at[t] = min(16 * t + n, rows - 1) * a.row_stride + 8 * Words * g;
      }
      f32x4 y[NT][FT];
#pragma unroll
      for (int t = 0; t < NT; ++t)
      {
#pragma unroll
        for (int u = 0; u < FT; ++u)
        {
          y[t][u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
      }
      const _Float16 one = static_cast<_Float16>(1.0f);
      const half8 ones = {one, one, one, one, one, one, one, one};
      const f32x4 none = {0.0f, 0.0f, 0.0f, 0.0f};

      const int chunks = (a.in + kChunk - 1) / kChunk;
      int chunk = split;
      Fetched<Words, FT> next;
      fetch<Words, FT>(next, a, row, min(chunk, chunks - 1), g);
      for (int from = 0; from < a.in; from += a.phase)
      {
        // The phase's inputs of every row, zeros past the last.
        const int width = min(a.phase, (a.in - from + kChunk - 1) / kChunk * kChunk);
        if (from > 0)
        {
          __syncthreads();
        }
        for (int i = threadIdx.x; i < rows * (width / 8); i += kThreads)
        {
          const int r = i / (width / 8);
          const int k = i % (width / 8) * 8;
          u32x4 v = {0u, 0u, 0u, 0u};
          if (from + k < a.in)
          {
            v = *reinterpret_cast<const u32x4 *>(x + static_cast<std::size_t>(r) * a.in + from + k);
          }
          const u32x4 turned = {__builtin_amdgcn_perm(v.z, v.x, 0x05040100u),
                                __builtin_amdgcn_perm(v.z, v.x, 0x07060302u),
                                __builtin_amdgcn_perm(v.w, v.y, 0x05040100u),
                                __builtin_amdgcn_perm(v.w, v.y, 0x07060302u)};
          *reinterpret_cast<u32x4 *>(x_lds + r * a.row_stride + k) = turned;
        }
        __syncthreads();
        const int phase_end = (from + width) / kChunk;
#pragma unroll 2
        for (; chunk < phase_end; chunk += a.splits)
        {
          const Fetched<Words, FT> now = next;
          fetch<Words, FT>(next, a, row, min(chunk + a.splits, chunks - 1), g);
          const int k0 = chunk * kChunk - from;
#pragma unroll
          for (int h = 0; h < kGroups; ++h)
          {
            f32x4 dot[NT][FT], sum[NT];
#pragma unroll
            for (int j = 0; j < Words; ++j)
            {
              half8 xa[NT];
#pragma unroll
              for (int t = 0; t < NT; ++t)
              {
                xa[t] = *reinterpret_cast<const half8 *>(x_lds + at[t] + k0 + 32 * Words * h +
                                                         8 * j);
                sum[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(xa[t], ones, j ? sum[t] : none, 0,
                                                                0, 0);
              }
#pragma unroll
              for (int u = 0; u < FT; ++u)
              {
                const half8 c = codes_as_half(now.w[u][h * Words + j]);
#pragma unroll
                for (int t = 0; t < NT; ++t)
                {
                  dot[t][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(xa[t], c, j ? dot[t][u] : none,
                                                                     0, 0, 0);
                }
              }
            }
#pragma unroll
            for (int u = 0; u < FT; ++u)
            {
              const float s = h2f(now.s[u][h]), z = h2f(now.z[u][h]);
#pragma unroll
              for (int t = 0; t < NT; ++t)
              {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                {
                  y[t][u][i] = __builtin_fmaf(s, dot[t][u][i],
                                              __builtin_fmaf(z, sum[t][i], y[t][u][i]));
                }
              }
            }
          }
        }
      }

      // The splits' sums, added by the tile's first wave in wave order.
      if (a.splits > 1)
      {
        f32x4 *parts = reinterpret_cast<f32x4 *>(x_lds);
        __syncthreads();
        if (split > 0)
        {
#pragma unroll
          for (int t = 0; t < NT; ++t)
          {
#pragma unroll
            for (int u = 0; u < FT; ++u)
            {
              parts[((wave * NT + t) * FT + u) * 64 + lane] = y[t][u];
            }
          }
        }
        __syncthreads();
        if (split > 0)
        {
          return;
        }
        for (int s = 1; s < a.splits; ++s)
        {
#pragma unroll
          for (int t = 0; t < NT; ++t)
          {
#pragma unroll
            for (int u = 0; u < FT; ++u)
            {
              y[t][u] += parts[(((wave + s) * NT + t) * FT + u) * 64 + lane];
            }
          }
        }
      }
#pragma unroll
      for (int u = 0; u < FT; ++u)
      {
        const int feature = tile0 + 16 * u + n;
        if (feature >= a.features)
        {
          continue;
        }
        const float bias = Out == Int4Out::kHalf && a.bias != nullptr ? h2f(a.bias[feature]) : 0.0f;
#pragma unroll
        for (int t = 0; t < NT; ++t)
        {
#pragma unroll
          for (int i = 0; i < 4; ++i)
          {
            const int r = 16 * t + 4 * g + i;
            if (r >= rows)
            {
              continue;
            }
            const std::size_t to =
                static_cast<std::size_t>(row0 + r) * a.features + feature;
            if constexpr (Out == Int4Out::kHalf)
            {
              static_cast<std::uint16_t *>(a.out)[to] =
                  __half_as_ushort(__float2half(y[t][u][i] + bias));
            }
            else
            {
              static_cast<float *>(a.out)[to] += y[t][u][i];
            }
          }
        }
      }
    }

    void check_int4(const void *codes, const void *scales, const void *zeros, int group, int in,
                    int out)
    {
      if (group != 32 && group != 64 && group != 128)
      {
        throw InvalidArgument("int4 weights have groups of 32, 64 or 128 inputs, not " +
                              std::to_string(group));
      }
      if (in < 0 || out < 0 || in % group != 0)
      {
        throw InvalidArgument("in_features " + std::to_string(in) + " and out_features " +
                              std::to_string(out) + " must not be negative, and in_features whole "
                              "groups of " + std::to_string(group));
      }
      if (in > 0 && out > 0 && (codes == nullptr || scales == nullptr || zeros == nullptr))
      {
        throw InvalidArgument("int4 weights need their codes, scales and zeros");
      }
      if (reinterpret_cast<std::uintptr_t>(codes) % 16 != 0 ||
          (reinterpret_cast<std::uintptr_t>(scales) | reinterpret_cast<std::uintptr_t>(zeros)) % 2 != 0)
      {
        throw InvalidArgument("int4 codes must be 16-byte aligned");
      }
    }

    template <int Words, int NT, int FT>
    void project(const Int4Args &a, Int4Out out, hipStream_t stream)
    {
      const int tiles = kWaves / a.splits * FT;
      const dim3 grid((a.features + 16 * tiles - 1) / (16 * tiles),
                      (a.rows + 16 * NT - 1) / (16 * NT));
      const std::size_t stage =
          static_cast<std::size_t>(std::min(a.rows, 16 * NT)) * a.row_stride * 2;
      const std::size_t parts = a.splits > 1 ? sizeof(f32x4) * kWaves * NT * FT * 64 : 0;
      const std::size_t lds = std::max(stage, parts);
      if (out == Int4Out::kHalf)
      {
        linear_int4_kernel<Words, NT, FT, Int4Out::kHalf><<<grid, kThreads, lds, stream>>>(a);
      }
      else
      {
        linear_int4_kernel<Words, NT, FT, Int4Out::kAccumulate><<<grid, kThreads, lds, stream>>>(a);
      }
      hip_check(hipGetLastError(), "linear_int4_kernel");
    }

    template <int Words>
    void project_rows(Int4Args a, Int4Out out, hipStream_t stream)
    {
      const int tiles = (a.features + 15) / 16;
      const int chunks = (a.in + kChunk - 1) / kChunk;
      const int nt = a.rows <= 16 ? 1 : a.rows <= 32 ? 2 : 4;
      const int ft = a.rows <= 16 ? 1 : 2;
      // A tile's inputs are split while the waves would not fill the CUs and
      // each keeps two chunks.
      a.splits = 1;
      while (a.splits < kWaves && (tiles / ft) * a.splits < 2048 && chunks >= 4 * a.splits)
      {
        a.splits *= 2;
      }
      const int rows = std::min(a.rows, 16 * nt);
      a.phase = std::min(chunks, std::max(1, (kStageHalves / rows - kRowPad) / kChunk)) * kChunk;
      a.row_stride = a.phase + kRowPad;
      switch (nt)
      {
      case 1: project<Words, 1, 1>(a, out, stream); break;
      case 2: project<Words, 2, 2>(a, out, stream); break;
      default: project<Words, 4, 2>(a, out, stream); break;
      }
    }

    void linear_int4(const void *x, const void *codes, const void *scales, const void *zeros,
                     int group, const void *bias, void *out, Int4Out kind, int rows, int in,
                     int features, hipStream_t stream)
    {
      check_int4(codes, scales, zeros, group, in, features);
      if (rows < 0)
      {
        throw InvalidArgument("rows must not be negative, got " + std::to_string(rows));
      }
      if (rows == 0 || features == 0)
      {
        return;
      }
      if (out == nullptr || (x == nullptr && in > 0))
      {
        throw InvalidArgument("x and out must not be null");
      }
      if (reinterpret_cast<std::uintptr_t>(x) % 16 != 0)
      {
        throw InvalidArgument("an int4 projection's x must be 16-byte aligned");
      }
      constexpr int kMostRows = 65535 * 64; // grid.y
      if (rows > kMostRows)
      {
        throw InvalidArgument("rows " + std::to_string(rows) + " are more than an int4 projection's " +
                              std::to_string(kMostRows));
      }
      if (in == 0)
      {
        throw InvalidArgument("an int4 projection needs at least one group of inputs");
      }
      Int4Args a{};
      a.x = static_cast<const std::uint16_t *>(x);
      a.codes = static_cast<const std::uint8_t *>(codes);
      a.scales = static_cast<const std::uint16_t *>(scales);
      a.zeros = static_cast<const std::uint16_t *>(zeros);
      a.bias = static_cast<const std::uint16_t *>(bias);
      a.out = out;
      a.rows = rows;
      a.in = in;
      a.features = features;
      a.groups = in / group;
      switch (group)
      {
      case 32: project_rows<1>(a, kind, stream); break;
      case 64: project_rows<2>(a, kind, stream); break;
      default: project_rows<4>(a, kind, stream); break;
      }
    }
  } // namespace

  void launch_quantise_int4(const void *weight, void *codes, void *scales, void *zeros, int group,
                            int in_features, int out_features, hipStream_t stream)
  {
    check_int4(codes, scales, zeros, group, in_features, out_features);
    if (in_features == 0 || out_features == 0)
    {
      return;
    }
    if (weight == nullptr || reinterpret_cast<std::uintptr_t>(weight) % 16 != 0)
    {
      throw InvalidArgument("the weight to quantise must be given, 16-byte aligned");
    }
    const std::size_t count = static_cast<std::size_t>(in_features) * out_features / 8;
    const std::size_t blocks = (count + 255) / 256;
    if (blocks > 0x7fffffffull)
    {
      throw InvalidArgument("a weight of " + std::to_string(8 * count) + " values is too large");
    }
    const dim3 grid(static_cast<unsigned>(blocks));
    const auto *w = static_cast<const std::uint16_t *>(weight);
    auto *c = static_cast<unsigned *>(codes);
    auto *s = static_cast<std::uint16_t *>(scales);
    auto *z = static_cast<std::uint16_t *>(zeros);
    switch (group)
    {
    case 32: quantise_int4_kernel<32><<<grid, 256, 0, stream>>>(w, c, s, z, count); break;
    case 64: quantise_int4_kernel<64><<<grid, 256, 0, stream>>>(w, c, s, z, count); break;
    default: quantise_int4_kernel<128><<<grid, 256, 0, stream>>>(w, c, s, z, count); break;
    }
    hip_check(hipGetLastError(), "quantise_int4_kernel");
  }

  void launch_linear_int4(const void *x, const void *codes, const void *scales, const void *zeros,
                          int group, const void *bias, void *out, int rows, int in_features,
                          int out_features, hipStream_t stream)
  {
    linear_int4(x, codes, scales, zeros, group, bias, out, Int4Out::kHalf, rows, in_features,
                out_features, stream);
  }

  void launch_linear_int4_accumulate(const void *x, const void *codes, const void *scales,
                                     const void *zeros, int group, float *out, int rows,
                                     int in_features, int out_features, hipStream_t stream)
  {
    linear_int4(x, codes, scales, zeros, group, nullptr, out, Int4Out::kAccumulate, rows,
                in_features, out_features, stream);
  }

} // namespace mi
