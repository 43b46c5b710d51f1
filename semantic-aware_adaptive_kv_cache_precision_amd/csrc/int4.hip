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
// One or two rows (int4_rows_kernel): bound by the weight's bytes. A lane
// takes 32 codes, 16 bytes, of one output; sixteen lanes take 256 bytes of a
// row and a wave 4 R rows at a time, so that every line is asked for once and
// whole; v_dot2 multiplies pairs into fp32. 128256 x 2048 in groups of 64, a
// row: 30 us, 4.9 TB/s; 128 x 896: 5.0 us, a launch.
//
// More rows (int4_tiles_kernel): the matrix cores form x . codes (A: 16 rows of
// x, B: 16 outputs' codes as fp16 integers, exact) and sum(x) (B: ones) of 32
// inputs an instruction in fp32, and two fmas an output scale a group. A step
// is 128 inputs: their codes, 64 bytes an output, come four lanes an output
// and turn through the wave's own LDS to a word an instruction, its inputs 32
// in a row: of one group, whatever its size. x comes sixteen lanes a row and
// turns the same way; scales and zeros come four steps at a load. (The lanes
// of an operand lie along the rows, where each sixteen bytes are a request of
// their own, and requests are what a CU runs out of: loaded so, and the next
// step's fetched past the last, 16 rows of 2048 x 8192 took 16.1 us, now 8.0.)
// 27 rows of 8960 -> 1536: 8.3 us, what a CU takes in (its 16 rows of x whole,
// 287 KB, and 72 KB of codes; two steps fetched ahead 9.6); 64 rows of
// 128256 x 2048: 79 us, a third of the matrix cores' rate, the vector units
// making fp16 of codes beside them.
//
// A code becomes fp16 by the mask that splices it under the exponent of 1024
// (or, four bits up, 1024 + 16 code): nine instructions for eight, which
// leaves them in the order 0 4 1 5 2 6 3 7; x is turned to that order, once
// for all the outputs a wave takes. Nothing is rounded before the one
// rounding of y. An output's inputs are split over up to sixteen waves, whose
// sums meet in LDS in wave order: the bits do not depend on timing.

#include "quant_core.hpp"
#include "serving.hpp"

#include <algorithm>
#include <string>
#include <type_traits>

namespace mi
{
  namespace
  {
    typedef _Float16 half8 __attribute__((ext_vector_type(8)));
    typedef _Float16 half2v __attribute__((ext_vector_type(2)));
    typedef float f32x4 __attribute__((ext_vector_type(4)));
    typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

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
      int groups;   // a row's
      int splits;   // waves an output's inputs are split over, a power of two
      int group_32; // log2 of a group's runs of 32
      bool wide_meta; // whole chunks of groups a row, on their own alignment
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

    // Eight inputs in the codes' order.
    __device__ inline u32x4 turned(u32x4 v)
    {
      const unsigned a = v.x, b = v.y, c = v.z, d = v.w;
      return u32x4{__builtin_amdgcn_perm(c, a, 0x05040100u), __builtin_amdgcn_perm(c, a, 0x07060302u),
                   __builtin_amdgcn_perm(d, b, 0x05040100u), __builtin_amdgcn_perm(d, b, 0x07060302u)};
    }

    // One output, stored. (Added to in memory by its one owner.)
    template <Int4Out Out>
    __device__ inline void store(const Int4Args &a, int row, int feature, float y)
    {
      const std::size_t to = static_cast<std::size_t>(row) * a.features + feature;
      if constexpr (Out == Int4Out::kHalf)
      {
        const float bias = a.bias != nullptr ? h2f(a.bias[feature]) : 0.0f;
        static_cast<std::uint16_t *>(a.out)[to] = __half_as_ushort(__float2half(y + bias));
      }
      else
      {
        static_cast<float *>(a.out)[to] += y;
      }
    }

    __device__ inline bool is_finite(float y)
    {
      return (__float_as_uint(y) & 0x7f800000u) != 0x7f800000u;
    }

    // The sum of a row that holds infinities or NaN, from their own terms
    // x (code * scale + zero): the kernels form x code and x zero apart, which
    // makes NaN of an infinity where the code is zero or the zero point has the
    // other sign. (A row that holds none has a scale or zero that is not finite.)
    __device__ inline float sum_of_infinite(const Int4Args &a, int row, int feature)
    {
      const std::uint16_t *x = a.x + static_cast<std::size_t>(row) * a.in;
      const std::uint8_t *codes = a.codes + static_cast<std::size_t>(feature) * (a.in / 2);
      const std::size_t meta = static_cast<std::size_t>(feature) * a.groups;
      float sum = 0.0f;
      bool some = false;
      for (int i = 0; i < a.in; i += 8)
      {
        const u32x4 eight = *reinterpret_cast<const u32x4 *>(x + i);
#pragma unroll
        for (int e = 0; e < 8; ++e)
        {
          const unsigned word = eight[e / 2];
          const auto bits = static_cast<std::uint16_t>(word >> (16 * (e % 2)));
          if ((bits & 0x7c00u) == 0x7c00u)
          {
            const int code = (codes[(i + e) / 2] >> (4 * (e % 2))) & 15;
            const std::size_t group = meta + (i >> (5 + a.group_32));
            sum += h2f(bits) * __builtin_fmaf(static_cast<float>(code), h2f(a.scales[group]),
                                              h2f(a.zeros[group]));
            some = true;
          }
        }
      }
      return some ? sum : __builtin_nanf("");
    }

    // ---- one or two rows ----------------------------------------------------

    constexpr int kRowWaves = 8;

    // The sum over the 16 lanes of a row group, in every lane.
    __device__ inline float row_sum(float v)
    {
      const auto turn = [](float x, auto ctrl) {
        return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), decltype(ctrl)::value,
                                                          0xf, 0xf, true));
      };
      v += turn(v, std::integral_constant<int, 0x128>{}); // row_ror:8
      v += turn(v, std::integral_constant<int, 0x124>{});
      v += turn(v, std::integral_constant<int, 0x122>{});
      v += turn(v, std::integral_constant<int, 0x121>{});
      return v;
    }

    template <int R>
    struct RowFetch
    {
      u32x4 w[R];
      std::uint16_t s[R];
      std::uint16_t z[R];
    };

    template <int Rows, int R, Int4Out Out>
    __global__ void __launch_bounds__(64 * kRowWaves) int4_rows_kernel(Int4Args a)
    {
      __shared__ float parts[kRowWaves][4 * R * Rows];
      const int lane = threadIdx.x & 63;
      const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
      const int f = lane >> 4; // the output of each four
      const int c = lane & 15; // the run of 32 inputs of each sixteen
      const int split = wave & (a.splits - 1);
      const int tile = static_cast<int>(blockIdx.x) * (kRowWaves / a.splits) + wave / a.splits;
      const int runs = a.in / 32;
      const int steps = (runs + 15) / 16;
      const std::uint8_t *codes[R];
      std::size_t meta[R];
#pragma unroll
      for (int u = 0; u < R; ++u)
      {
        const int row = min(tile * 4 * R + 4 * u + f, a.features - 1);
        codes[u] = a.codes + static_cast<std::size_t>(row) * (a.in / 2);
        meta[u] = static_cast<std::size_t>(row) * a.groups;
      }
      const auto fetch = [&](RowFetch<R> &to, int step) {
        const int run = min(16 * step + c, runs - 1);
#pragma unroll
        for (int u = 0; u < R; ++u)
        {
          to.w[u] = *reinterpret_cast<const u32x4 *>(codes[u] + 16 * static_cast<std::size_t>(run));
        }
#pragma unroll
        for (int u = 0; u < R; ++u)
        {
          to.s[u] = a.scales[meta[u] + (run >> a.group_32)];
          to.z[u] = a.zeros[meta[u] + (run >> a.group_32)];
        }
      };
      float y[R][Rows] = {};
      RowFetch<R> next;
      if (split < steps)
      {
        fetch(next, split);
      }
#pragma unroll 2
      for (int step = split; step < steps; step += a.splits)
      {
        const RowFetch<R> now = next;
        fetch(next, min(step + a.splits, steps - 1));
        const int run = 16 * step + c;
        u32x4 x[Rows][4];
        float sum[Rows];
#pragma unroll
        for (int r = 0; r < Rows; ++r)
        {
          const std::uint16_t *from =
              a.x + static_cast<std::size_t>(min(r, a.rows - 1)) * a.in + 32 * min(run, runs - 1);
#pragma unroll
          for (int j = 0; j < 4; ++j)
          {
            x[r][j] = *reinterpret_cast<const u32x4 *>(from + 8 * j);
            x[r][j] = run < runs ? turned(x[r][j]) : u32x4{0u, 0u, 0u, 0u};
          }
        }
        const _Float16 one = static_cast<_Float16>(1.0f);
#pragma unroll
        for (int r = 0; r < Rows; ++r)
        {
          sum[r] = 0.0f;
#pragma unroll
          for (int j = 0; j < 4; ++j)
          {
#pragma unroll
            for (int i = 0; i < 4; ++i)
            {
              const unsigned word = x[r][j][i];
              sum[r] = __builtin_amdgcn_fdot2(__builtin_bit_cast(half2v, word), half2v{one, one},
                                              sum[r], false);
            }
          }
        }
#pragma unroll
        for (int u = 0; u < R; ++u)
        {
          float dot[Rows] = {};
#pragma unroll
          for (int j = 0; j < 4; ++j)
          {
            const unsigned code_word = now.w[u][j];
            const u32x4 q = __builtin_bit_cast(u32x4, codes_as_half(code_word));
#pragma unroll
            for (int i = 0; i < 4; ++i)
            {
              const unsigned pair = q[i];
#pragma unroll
              for (int r = 0; r < Rows; ++r)
              {
                const unsigned word = x[r][j][i];
                dot[r] = __builtin_amdgcn_fdot2(__builtin_bit_cast(half2v, word),
                                                __builtin_bit_cast(half2v, pair), dot[r], false);
              }
            }
          }
          const float s = h2f(now.s[u]), z = h2f(now.z[u]);
#pragma unroll
          for (int r = 0; r < Rows; ++r)
          {
            y[u][r] = __builtin_fmaf(s, dot[r], __builtin_fmaf(z, sum[r], y[u][r]));
          }
        }
      }
      // Lane c keeps the sum of (output set c / Rows, row c % Rows).
      float mine = 0.0f;
#pragma unroll
      for (int u = 0; u < R; ++u)
      {
#pragma unroll
        for (int r = 0; r < Rows; ++r)
        {
          const float total = row_sum(y[u][r]);
          mine = c == u * Rows + r ? total : mine;
        }
      }
      if (a.splits > 1)
      {
        if (c < R * Rows)
        {
          parts[wave][4 * c + f] = mine;
        }
        __syncthreads();
        if (split > 0)
        {
          return;
        }
        if (c < R * Rows)
        {
          for (int p = 1; p < a.splits; ++p)
          {
            mine += parts[wave + p][4 * c + f];
          }
        }
      }
      const int feature = tile * 4 * R + 4 * (c / Rows) + f;
      if (c < R * Rows && c % Rows < a.rows && feature < a.features)
      {
        store<Out>(a, c % Rows, feature,
                   is_finite(mine) ? mine : sum_of_infinite(a, c % Rows, feature));
      }
    }

    // ---- more rows ----------------------------------------------------------

    constexpr int kChunk = 128; // inputs a wave takes at a time

    // Between one wave's writes of LDS and its reads of them by other lanes, and
    // between those reads and the next writes: the wave's operations complete in
    // order, and this keeps the compiler to it. (No instruction.)
    __device__ inline void wave_exchange()
    {
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }

    // NT tiles of 16 rows, FT tiles of 16 outputs a wave; Groups: groups in a
    // chunk.
    // Shared: the waves' tiles of outputs are all different, and x goes through
    // LDS once for all of them, double buffered.
    template <int Groups, int NT, int FT, int Waves, bool Shared, Int4Out Out>
    __global__ void __launch_bounds__(64 * Waves) int4_tiles_kernel(Int4Args a)
    {
      constexpr int kPer = 4 / Groups; // instructions a group
      constexpr int kStage = NT * 256;               // 16-byte pieces of x
      constexpr int kWaveStage = kStage + 64 * FT;   // and of a wave's codes
      extern __shared__ __align__(16) u32x4 stages[];
      const int lane = threadIdx.x & 63;
      const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
      const int n = lane & 15;
      const int g = lane >> 4;
      const int split = wave & (a.splits - 1);
      const int tile0 =
          (static_cast<int>(blockIdx.x) * (Waves / a.splits) + wave / a.splits) * FT * 16;
      const int row0 = static_cast<int>(blockIdx.y) * 16 * NT;
      const int rows = min(a.rows - row0, 16 * NT);
      // Addresses: a scalar base and 32 bits a lane (in is held to kMostInputs).
      const int base = min(tile0, a.features - 1); // (a wave past the last output repeats it)
      const std::uint8_t *codes = a.codes + static_cast<std::size_t>(base) * (a.in / 2);
      const char *scales =
          reinterpret_cast<const char *>(a.scales + static_cast<std::size_t>(base) * a.groups);
      const char *zeros =
          reinterpret_cast<const char *>(a.zeros + static_cast<std::size_t>(base) * a.groups);
      // Codes, scales and zeros are loaded by the lane's fourth: four lanes an
      // output.
      const int quarter = lane & 3;
      unsigned of[FT];
#pragma unroll
      for (int u = 0; u < FT; ++u)
      {
        of[u] = min(16 * u + (lane >> 2), a.features - 1 - base);
      }
      unsigned *words = reinterpret_cast<unsigned *>(
          stages + (Shared ? 2 * kStage + wave * FT * 64 : wave * kWaveStage + kStage));
      // x comes in whole lines, four rows' chunks a load, and turns through the
      // wave's own LDS, piece p of row r at place p ^ r % 16 of its row.
      u32x4 *stage = stages + (Shared ? 0 : wave * kWaveStage);
      const char *x =
          reinterpret_cast<const char *>(a.x + static_cast<std::size_t>(row0) * a.in);
      constexpr int kFetches = Shared ? (4 * NT + Waves - 1) / Waves : 4 * NT; // of four rows
      const auto four_of = [&](int i) { return Shared ? wave + Waves * i : i; };
      unsigned x_at[kFetches]; // (a row past the last repeats it)
#pragma unroll
      for (int i = 0; i < kFetches; ++i)
      {
        x_at[i] = 2u * min(4 * four_of(i) + g, rows - 1) * static_cast<unsigned>(a.in);
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
      // (Inputs past the last, and groups: the first's, which no product takes.)
      const auto fetch = [&](u32x4 (&to)[FT], int chunk) {
        const int k = chunk * kChunk + 32 * quarter;
#pragma unroll
        for (int u = 0; u < FT; ++u)
        {
          to[u] = *reinterpret_cast<const u32x4 *>(
              codes + (of[u] * static_cast<unsigned>(a.in) + (k < a.in ? k : 0)) / 2);
        }
      };
      const auto fetch_x = [&](u32x4 (&to)[kFetches], int chunk) {
        const int k = chunk * kChunk + 8 * n;
#pragma unroll
        for (int i = 0; i < kFetches; ++i)
        {
          if (4 * four_of(i) < rows)
          {
            to[i] = *reinterpret_cast<const u32x4 *>(x + (x_at[i] + 2u * (k < a.in ? k : 0)));
          }
        }
      };
      // (Products of rows past the last are left.)
      const auto stage_x = [&](u32x4 *to, const u32x4 (&from)[kFetches]) {
#pragma unroll
        for (int i = 0; i < kFetches; ++i)
        {
          const int four = four_of(i);
          if (!Shared || four < 4 * NT)
          {
            const int row = 4 * (four % 4) + g;
            to[four / 4 * 256 + 16 * row + (n ^ row)] = turned(from[i]);
          }
        }
      };
      // Scales (low) and zeros of four chunks, quarters q those of chunk + q.
      const auto fetch_meta = [&](unsigned (&to)[FT][Groups], int chunk) {
        const int at_chunk = min(chunk + quarter, chunks - 1);
#pragma unroll
        for (int u = 0; u < FT; ++u)
        {
          std::uint16_t sc[Groups], ze[Groups];
          const unsigned row = of[u] * a.groups;
          if (Groups > 1 && a.wide_meta)
          {
            const unsigned at = 2u * (row + at_chunk * Groups);
            __builtin_memcpy(sc, __builtin_assume_aligned(scales + at, 2 * Groups), 2 * Groups);
            __builtin_memcpy(ze, __builtin_assume_aligned(zeros + at, 2 * Groups), 2 * Groups);
          }
          else
          {
#pragma unroll
            for (int h = 0; h < Groups; ++h)
            {
              const int group = at_chunk * Groups + h;
              const unsigned at = 2u * (row + (group < a.groups ? group : 0));
              sc[h] = *reinterpret_cast<const std::uint16_t *>(scales + at);
              ze[h] = *reinterpret_cast<const std::uint16_t *>(zeros + at);
            }
          }
#pragma unroll
          for (int h = 0; h < Groups; ++h)
          {
            to[u][h] = sc[h] | static_cast<unsigned>(ze[h]) << 16;
          }
        }
      };
      const int per = (chunks + a.splits - 1) / a.splits;
      const int begin = split * per;
      const int end = min(begin + per, chunks);
      u32x4 next[FT], next_x[kFetches] = {};
      unsigned four[FT][Groups], next_four[FT][Groups];
      if (begin < end)
      {
        fetch(next, begin);
        fetch_x(next_x, begin);
        fetch_meta(next_four, begin);
        if constexpr (Shared)
        {
          stage_x(stage, next_x);
        }
      }
      for (int chunk = begin; chunk < end; ++chunk)
      {
        const int of_four = (chunk - begin) & 3;
        wave_exchange();
        // The codes, run p of 32 of output o at place p ^ o / 4 of its four.
#pragma unroll
        for (int u = 0; u < FT; ++u)
        {
          const int o = lane >> 2;
          reinterpret_cast<u32x4 *>(words)[u * 64 + 4 * o + (quarter ^ (o >> 2))] = next[u];
#pragma unroll
          for (int h = 0; h < Groups; ++h)
          {
            four[u][h] = of_four == 0 ? next_four[u][h] : four[u][h];
          }
        }
        if constexpr (Shared)
        {
          stage = stages + ((chunk - begin) & 1) * kStage;
          __syncthreads();
        }
        else
        {
          stage_x(stage, next_x);
          wave_exchange();
        }
        if (chunk + 1 < end)
        {
          fetch(next, chunk + 1);
          fetch_x(next_x, chunk + 1);
          if (of_four == 3)
          {
            fetch_meta(next_four, chunk + 1);
          }
        }
        const int k0 = chunk * kChunk;
#pragma unroll
        for (int h = 0; h < Groups; ++h)
        {
          if (h > 0 && k0 + 32 * kPer * h >= a.in)
          {
            break;
          }
          f32x4 dot[NT][FT], sum[NT];
#pragma unroll
          for (int j = 0; j < kPer; ++j)
          {
            half8 xt[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t)
            {
              xt[t] = __builtin_bit_cast(
                  half8, stage[t * 256 + 16 * n + ((4 * (h * kPer + j) + g) ^ n)]);
              sum[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(xt[t], ones, j ? sum[t] : none, 0, 0,
                                                              0);
            }
#pragma unroll
            for (int u = 0; u < FT; ++u)
            {
              const unsigned word =
                  words[u * 256 + 16 * n + 4 * ((h * kPer + j) ^ (n >> 2)) + g];
              const half8 q = codes_as_half(word);
#pragma unroll
              for (int t = 0; t < NT; ++t)
              {
                dot[t][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(xt[t], q, j ? dot[t][u] : none, 0,
                                                                   0, 0);
              }
            }
          }
#pragma unroll
          for (int u = 0; u < FT; ++u)
          {
            const unsigned both = static_cast<unsigned>(__builtin_amdgcn_ds_bpermute(
                4 * (4 * n + of_four), static_cast<int>(four[u][h])));
            const float s = h2f(static_cast<std::uint16_t>(both));
            const float z = h2f(static_cast<std::uint16_t>(both >> 16));
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
        if constexpr (Shared)
        {
          if (chunk + 1 < end)
          {
            stage_x(stages + ((chunk + 1 - begin) & 1) * kStage, next_x);
          }
        }
      }

      // The splits' sums, added by the tile's first wave in wave order.
      if (a.splits > 1)
      {
        static_assert(Shared || FT <= 4, "a wave's sums in its stage");
        f32x4 *parts = reinterpret_cast<f32x4 *>(stages);
        wave_exchange();
        if (split > 0)
        {
#pragma unroll
          for (int t = 0; t < NT; ++t)
          {
#pragma unroll
            for (int u = 0; u < FT; ++u)
            {
              parts[wave * kWaveStage + (t * FT + u) * 64 + lane] = y[t][u];
            }
          }
        }
        __syncthreads();
        if (split > 0)
        {
          return;
        }
        for (int p = 1; p < a.splits; ++p)
        {
#pragma unroll
          for (int t = 0; t < NT; ++t)
          {
#pragma unroll
            for (int u = 0; u < FT; ++u)
            {
              y[t][u] += parts[(wave + p) * kWaveStage + (t * FT + u) * 64 + lane];
            }
          }
        }
      }
      float odd = 0.0f; // zero while every sum is finite, else NaN
#pragma unroll
      for (int u = 0; u < FT; ++u)
      {
#pragma unroll
        for (int t = 0; t < NT; ++t)
        {
#pragma unroll
          for (int i = 0; i < 4; ++i)
          {
            odd = __builtin_fmaf(y[t][u][i], 0.0f, odd);
          }
        }
      }
      // (Sums that are not finite are left for later, a bit each; a test of each
      // one's own beside its store took 4% of 1,024 rows, 6% of 64 of 8192 x 2048.)
      static_assert(NT <= 4 && FT <= 4);
      unsigned long long left = 0;
      const auto store_all = [&](auto test) {
#pragma unroll
        for (int u = 0; u < FT; ++u)
        {
          const int feature = tile0 + 16 * u + n;
#pragma unroll
          for (int t = 0; t < NT; ++t)
          {
#pragma unroll
            for (int i = 0; i < 4; ++i)
            {
              const int r = 16 * t + 4 * g + i;
              if (r < rows && feature < a.features)
              {
                if (!test || is_finite(y[t][u][i]))
                {
                  store<Out>(a, row0 + r, feature, y[t][u][i]);
                }
                else
                {
                  left |= 1ull << (16 * u + 4 * t + i);
                }
              }
            }
          }
        }
      };
      if (odd == 0.0f)
      {
        store_all(std::false_type{});
        return;
      }
      store_all(std::true_type{});
      for (; left != 0; left &= left - 1)
      {
        const int bit = __builtin_ctzll(left);
        const int row = row0 + 16 * (bit % 16 / 4) + 4 * g + bit % 4;
        const int feature = tile0 + 16 * (bit / 16) + n;
        store<Out>(a, row, feature, sum_of_infinite(a, row, feature));
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

    // The waves an output's inputs are split over: a power of two up to
    // `most`, while the waves would not fill the device twice over and each
    // keeps a step (a step is a trip to memory).
    int splits_of(int tiles, int steps, int most)
    {
      int splits = 1;
      while (splits < most && static_cast<long long>(tiles) * splits < 4096 && steps >= 2 * splits)
      {
        splits *= 2;
      }
      return splits;
    }

    template <int Rows, int R>
    void project_rows(Int4Args a, Int4Out out, hipStream_t stream)
    {
      const int tiles = (a.features + 4 * R - 1) / (4 * R);
      a.splits = splits_of(tiles, (a.in / 32 + 15) / 16, kRowWaves);
      const int per = kRowWaves / a.splits;
      const dim3 grid((tiles + per - 1) / per);
      if (out == Int4Out::kHalf)
      {
        int4_rows_kernel<Rows, R, Int4Out::kHalf><<<grid, 64 * kRowWaves, 0, stream>>>(a);
      }
      else
      {
        int4_rows_kernel<Rows, R, Int4Out::kAccumulate><<<grid, 64 * kRowWaves, 0, stream>>>(a);
      }
      hip_check(hipGetLastError(), "int4_rows_kernel");
    }

    template <int Groups, int NT, int FT, int Waves, bool Shared = false>
    void project_tiles(Int4Args a, Int4Out out, hipStream_t stream)
    {
      const int tiles = (a.features + 16 * FT - 1) / (16 * FT);
      const int row_tiles = (a.rows + 16 * NT - 1) / (16 * NT);
      a.splits = splits_of(static_cast<int>(std::min<long long>(
                               static_cast<long long>(tiles) * row_tiles, 1 << 20)),
                           (a.in + kChunk - 1) / kChunk, Shared ? 1 : Waves);
      const int per = Waves / a.splits;
      const dim3 grid((tiles + per - 1) / per, row_tiles);
      constexpr std::size_t lds =
          sizeof(u32x4) * ((Shared ? 2 : Waves) * NT * 256 + Waves * FT * 64);
      auto kernel = out == Int4Out::kHalf
                        ? int4_tiles_kernel<Groups, NT, FT, Waves, Shared, Int4Out::kHalf>
                        : int4_tiles_kernel<Groups, NT, FT, Waves, Shared, Int4Out::kAccumulate>;
      if constexpr (lds > 64 * 1024)
      {
        hip_check(hipFuncSetAttribute(reinterpret_cast<const void *>(kernel),
                                      hipFuncAttributeMaxDynamicSharedMemorySize,
                                      static_cast<int>(lds)),
                  "hipFuncSetAttribute int4 LDS");
      }
      kernel<<<grid, 64 * Waves, lds, stream>>>(a);
      hip_check(hipGetLastError(), "int4_tiles_kernel");
    }

    template <int Groups>
    void project(const Int4Args &a, Int4Out out, hipStream_t stream)
    {
      const long long tiles = (a.features + 15) / 16;
      const long long work = tiles * ((a.rows + 15) / 16);
      const int steps = (a.in + kChunk - 1) / kChunk;
      const auto groups_of = [&](int outputs, int rows) { // workgroups of tiles of these
        return static_cast<long long>((a.features + outputs - 1) / outputs) *
               ((a.rows + rows - 1) / rows);
      };
      // Whether it takes more than eight waves a tile to make the device full.
      const bool wide = work <= 4096 && splits_of(static_cast<int>(work), steps, 16) > 8;
      // One row by dot products, and two of plenty of outputs or a wide tile
      // (128256 x 2048, two rows 41 us, by tiles 50; 1536 x 8960 7.3 and 7.7;
      // but 8960 x 1536 7.1 and 5.2); four sets of outputs a wave where there
      // are plenty.
      const bool many = a.features >= 16384;
      if (a.rows == 1)
      {
        many ? project_rows<1, 4>(a, out, stream) : project_rows<1, 1>(a, out, stream);
      }
      else if (a.rows == 2 && (many || wide))
      {
        many ? project_rows<2, 4>(a, out, stream) : project_rows<2, 1>(a, out, stream);
      }
      // Little work: a tile a wave, its inputs split over as many waves as
      // make the device full, in workgroups of eight where that is enough
      // (8960 x 1536, 16 rows, in us: sixteen waves 8.3, eight 5.7; 48 rows
      // 10.0, by the tiles below 15.7; 64 rows of 8192 x 2048 13.8 and 12.0).
      // Where workgroups of sixteen waves, one a CU, would take two turns, two
      // row tiles a wave share the codes (1536 x 8960: 64 rows 16.4 and 13.2,
      // 32 rows, one turn, 9.3). Much work: tiles of outputs share x.
      else if (wide && work * steps <= 40960)
      {
        work > 256 ? project_tiles<Groups, 2, 1, 16>(a, out, stream)
                   : project_tiles<Groups, 1, 1, 16>(a, out, stream);
      }
      else if (!wide && (work <= 1024 || work * steps <= 28672))
      {
        project_tiles<Groups, 1, 1, 8>(a, out, stream);
      }
      // Where workgroups of eight different tiles fill most of the device, x
      // goes through LDS once for all of them (128256 x 2048: 16 rows 55 us
      // and shared 49, 32 rows 72 and 57, 64 rows 109 and 80, 1,024 rows 1386
      // and 1073, 501 TFLOP/s; but 64 rows of 16384 x 2048, 64 workgroups, 23
      // and 37).
      else if (a.rows <= 16)
      {
        groups_of(64 * 4, 16) >= 192 ? project_tiles<Groups, 1, 4, 4, true>(a, out, stream)
                                     : project_tiles<Groups, 1, 4, 8>(a, out, stream);
      }
      else if (a.rows <= 32)
      {
        groups_of(32 * 8, 32) >= 192 ? project_tiles<Groups, 2, 2, 8, true>(a, out, stream)
                                     : project_tiles<Groups, 2, 4, 8>(a, out, stream);
      }
      else if (groups_of(32 * 8, 64) < 192)
      {
        project_tiles<Groups, 4, 2, 8>(a, out, stream);
      }
      // One workgroup a CU at a time: tiles of twice the outputs unless they
      // take more turns for it (1,024 rows 8192 x 2048, 256 workgroups: 72 us,
      // the smaller tiles 77; 8960 x 1536, 288: 111 and 76).
      else if (2 * ((groups_of(64 * 8, 64) + 255) / 256) <= (groups_of(32 * 8, 64) + 255) / 256)
      {
        project_tiles<Groups, 4, 4, 8, true>(a, out, stream);
      }
      else
      {
        project_tiles<Groups, 4, 2, 8, true>(a, out, stream);
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
      // 64 rows of x within 32 bits, a grid's threads too.
      constexpr int kMostInputs = 1 << 24, kMostOutputs = 1 << 27;
      if (in > kMostInputs || features > kMostOutputs)
      {
        throw InvalidArgument("an int4 projection takes at most " + std::to_string(kMostInputs) +
                              " in_features and " + std::to_string(kMostOutputs) +
                              " out_features, got " + std::to_string(in) + " and " +
                              std::to_string(features));
      }
      if (in == 0)
      {
        throw InvalidArgument("an int4 projection needs at least one group of inputs");
      }
      const std::size_t outputs = static_cast<std::size_t>(features);
      const std::size_t meta = 2 * outputs * (in / group);
      const Extent written{out, (kind == Int4Out::kHalf ? 2 : 4) * outputs * rows};
      for (const Extent &read : {Extent{x, 2 * static_cast<std::size_t>(rows) * in},
                                 Extent{codes, outputs * (in / 2)}, Extent{scales, meta},
                                 Extent{zeros, meta}, Extent{bias, 2 * outputs}})
      {
        if (overlaps(written, read))
        {
          throw InvalidArgument("an int4 projection cannot write over its input or weight");
        }
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
      a.wide_meta = in % kChunk == 0 && ((reinterpret_cast<std::uintptr_t>(scales) |
                                          reinterpret_cast<std::uintptr_t>(zeros)) % 8) == 0;
      a.group_32 = group == 32 ? 0 : group == 64 ? 1 : 2;
      switch (group)
      {
      case 32: project<4>(a, kind, stream); break;
      case 64: project<2>(a, kind, stream); break;
      default: project<1>(a, kind, stream); break;
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
    const std::size_t meta = 16 * count / group;
    const Extent read{weight, 16 * count}, code_bytes{codes, 4 * count};
    const Extent scale_bytes{scales, meta}, zero_bytes{zeros, meta};
    if (overlaps(code_bytes, read) || overlaps(scale_bytes, read) || overlaps(zero_bytes, read) ||
        overlaps(code_bytes, scale_bytes) || overlaps(code_bytes, zero_bytes) ||
        overlaps(scale_bytes, zero_bytes))
    {
      throw InvalidArgument("codes, scales and zeros cannot write over the weight or one another");
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
