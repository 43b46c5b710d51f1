// Rows and weights in signed bytes with a scale a row, and their products:
// y[m][n] = s_x[m] s_w[n] sum_k c_x[m][k] c_w[n][k] (+ bias, or + a residual).
//
// A row's scale is its largest magnitude / 127 and a code its value / scale,
// both divisions rounded in fp32, the code then to the nearest whole number.
// The sums are whole numbers and stay in 32 bits (in < 2^17), so that their
// order does not matter; y takes three roundings in fp32 (the sum to fp32, the
// two scales) and the bias's, then the one to fp16.
#include "common.hpp"
#include "ragged.hpp"

#include <algorithm>
#include <cmath>
#include <string>

namespace mi
{
  namespace
  {
    typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
    typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
    typedef int i32x4 __attribute__((ext_vector_type(4)));
    typedef int i32x16 __attribute__((ext_vector_type(16)));
    typedef float f32x4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) void *lds_void;
    typedef const __attribute__((address_space(1))) void *global_void;

    // ---- the quantiser ------------------------------------------------------

    // The larger magnitude, as fp16 bits, of each half of two words: infinities
    // and NaN are the largest.
    __device__ inline unsigned larger_halves(unsigned a, unsigned b)
    {
      const unsigned lo = max(a & 0x7FFFu, b & 0x7FFFu);
      const unsigned hi = max(a & 0x7FFF0000u, b & 0x7FFF0000u);
      return lo | hi;
    }

    // x / scale to the nearest whole number: by a product, which is within
    // 2^-15 of the quotient (at most 127 in magnitude), and by the division
    // where that does not settle it.
    __device__ inline int code_of(float x, float scale, float inv)
    {
      const float q = x * inv;
      float c = rintf(q);
      if (fabsf(q - c) > 0.5f - 0x1p-13f)
      {
        c = rintf(x / scale);
      }
      return static_cast<int>(c);
    }

    // Eight values a lane, kLanes lanes a row, kRuns times, held in registers
    // between the largest and the codes; rows of more are read twice (kRuns 0).
    // Bound by memory: 2 bytes read, one written a value (2,048 rows of 8,960 11.6
    // us, 4.7 TB/s; five rows of 896 a launch, 4.5).
    template <int kLanes, int kRuns>
    __global__ void __launch_bounds__(256)
        quantise_rows_kernel(const std::uint16_t *__restrict__ x, long long stride,
                             std::uint8_t *__restrict__ codes, float *__restrict__ scales, int rows,
                             int runs)
    {
      constexpr int kHeld = kRuns == 0 ? 1 : kRuns;
      __shared__ unsigned s_top[4];
      const int row = blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes;
      const int lane = threadIdx.x % kLanes;
      const bool live = row < rows;
      const std::uint16_t *from = x + static_cast<std::size_t>(live ? row : 0) * stride;
      u32x4 held[kHeld];
      unsigned top = 0;
      if constexpr (kRuns > 0)
      {
#pragma unroll
        for (int r = 0; r < kRuns; ++r)
        {
          const int run = lane + r * kLanes;
          held[r] = live && run < runs ? *reinterpret_cast<const u32x4 *>(from + 8 * run)
                                       : u32x4{0u, 0u, 0u, 0u};
        }
#pragma unroll
        for (int r = 0; r < kRuns; ++r)
        {
#pragma unroll
          for (int w = 0; w < 4; ++w)
          {
            top = larger_halves(top, held[r][w]);
          }
        }
      }
      else
      {
        for (int run = lane; live && run < runs; run += kLanes)
        {
          const u32x4 v = *reinterpret_cast<const u32x4 *>(from + 8 * run);
#pragma unroll
          for (int w = 0; w < 4; ++w)
          {
            top = larger_halves(top, v[w]);
          }
        }
      }
      unsigned bits = max(top & 0xFFFFu, top >> 16);
#pragma unroll
      for (int offset = 1; offset < 64; offset *= 2)
      {
        bits = max(bits, static_cast<unsigned>(__shfl_xor(static_cast<int>(bits), offset)));
      }
      if constexpr (kLanes > 64)
      {
        if (threadIdx.x % 64 == 0)
        {
          s_top[threadIdx.x / 64] = bits;
        }
        __syncthreads();
        bits = max(max(s_top[0], s_top[1]), max(s_top[2], s_top[3]));
      }
      const bool finite = bits < 0x7C00u;
      const float scale = finite ? h2f(static_cast<std::uint16_t>(bits)) / 127.0f : NAN;
      const float inv = finite && bits > 0 ? 1.0f / scale : 0.0f;
      const auto store = [&](int run, u32x4 v) {
        unsigned out[2] = {0u, 0u};
        if (finite && bits > 0)
        {
#pragma unroll
          for (int e = 0; e < 8; ++e)
          {
            const auto half = static_cast<std::uint16_t>(v[e / 2] >> (16 * (e % 2)));
            const int c = code_of(h2f(half), scale, inv);
            out[e / 4] |= (static_cast<unsigned>(c) & 255u) << (8 * (e % 4));
          }
        }
        *reinterpret_cast<u32x2 *>(codes + 8 * (static_cast<std::size_t>(row) * runs + run)) =
            u32x2{out[0], out[1]};
      };
      if (!live)
      {
        return;
      }
      if constexpr (kRuns > 0)
      {
#pragma unroll
        for (int r = 0; r < kRuns; ++r)
        {
          const int run = lane + r * kLanes;
          if (run < runs)
          {
            store(run, held[r]);
          }
        }
      }
      else
      {
        for (int run = lane; run < runs; run += kLanes)
        {
          store(run, *reinterpret_cast<const u32x4 *>(from + 8 * run));
        }
      }
      if (lane == 0)
      {
        scales[row] = scale;
      }
    }

    // ---- the projection -----------------------------------------------------

    struct Int8Args
    {
      const std::uint8_t *x;
      const float *x_scales;
      const std::uint8_t *w;
      const float *w_scales;
      const std::uint16_t *bias;
      const float *residual;
      void *out;
      int rows;
      int in;
      int features;
    };

    // One output from its whole-number sum.
    __device__ inline float scaled(int sum, float x_scale, float w_scale)
    {
      return static_cast<float>(sum) * x_scale * w_scale;
    }

    template <bool kHalf>
    __device__ inline void put(const Int8Args &a, int row, int n, int sum)
    {
      float y = scaled(sum, a.x_scales[row], a.w_scales[n]);
      const std::size_t at = static_cast<std::size_t>(row) * a.features + n;
      if constexpr (kHalf)
      {
        if (a.bias != nullptr)
        {
          y += h2f(a.bias[n]);
        }
        static_cast<std::uint16_t *>(a.out)[at] = __half_as_ushort(__float2half(y));
      }
      else
      {
        static_cast<float *>(a.out)[at] = a.residual[at] + y;
      }
    }

    // Few rows: bound by the weight's bytes. A wave takes 16 outputs and MT x
    // 16 rows over its share of the inputs; the workgroup's waves share them,
    // 128 at a time, and meet in LDS. Operands straight from memory: lane l
    // holds the 32 bytes 32 (l / 16) .. of row l % 16 of a step, so that four
    // lanes take a line and a product any 16 of a lane's bytes. (One row 1536 ->
    // 8960 5.6 us, 2048 -> 128256 39, 6.7 TB/s with the weight in the caches.)
    template <int MT, int kWaves, bool kHalf>
    __global__ void __launch_bounds__(64 * kWaves) int8_rows_kernel(Int8Args a)
    {
      __shared__ int s_sums[kWaves][MT][4][64];
      const int lane = threadIdx.x & 63;
      const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
      const int n0 = blockIdx.x * 16;
      const int m0 = blockIdx.y * 16 * MT;
      const int at = 32 * (lane >> 4);
      const std::uint8_t *w = a.w + static_cast<std::size_t>(min(n0 + (lane & 15), a.features - 1)) * a.in;
      const std::uint8_t *x[MT];
      i32x4 acc[MT];
#pragma unroll
      for (int t = 0; t < MT; ++t)
      {
        x[t] = a.x + static_cast<std::size_t>(min(m0 + 16 * t + (lane & 15), a.rows - 1)) * a.in;
        acc[t] = i32x4{0, 0, 0, 0};
      }
      const int whole = a.in / 128; // steps with no end in them
      const int steps = (a.in + 127) / 128;
      const int per = (steps + kWaves - 1) / kWaves;
      const int begin = min(wave * per, steps), end = min(begin + per, steps);
      const auto step_at = [&](int step, i32x4 (&b)[2], i32x4 (&v)[MT][2]) {
        const int k = 128 * step + at;
#pragma unroll
        for (int h = 0; h < 2; ++h)
        {
          b[h] = *reinterpret_cast<const i32x4 *>(w + k + 16 * h);
#pragma unroll
          for (int t = 0; t < MT; ++t)
          {
            v[t][h] = *reinterpret_cast<const i32x4 *>(x[t] + k + 16 * h);
          }
        }
      };
      const auto multiply = [&](const i32x4 (&b)[2], const i32x4 (&v)[MT][2]) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
        {
#pragma unroll
          for (int t = 0; t < MT; ++t)
          {
            acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(v[t][h], b[h], acc[t], 0, 0, 0);
          }
        }
      };
      // Steps asked for together, as registers allow.
      constexpr int kAhead = MT == 1 ? 4 : 2;
      int step = begin;
      for (; step + kAhead <= min(end, whole); step += kAhead)
      {
        i32x4 b[kAhead][2], v[kAhead][MT][2];
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
        {
          step_at(step + i, b[i], v[i]);
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
        {
          multiply(b[i], v[i]);
        }
      }
      for (; step < min(end, whole); ++step)
      {
        i32x4 b[2], v[MT][2];
        step_at(step, b, v);
        multiply(b, v);
      }
      if (step < end)
      {
        // The last inputs, in sixteens: those past the end count as zeros.
        i32x4 b[2], v[MT][2];
#pragma unroll
        for (int h = 0; h < 2; ++h)
        {
          const int k = 128 * step + at + 16 * h;
          const bool there = k < a.in;
          b[h] = *reinterpret_cast<const i32x4 *>(w + (there ? k : 0));
#pragma unroll
          for (int t = 0; t < MT; ++t)
          {
            const i32x4 got = *reinterpret_cast<const i32x4 *>(x[t] + (there ? k : 0));
            v[t][h] = there ? got : i32x4{0, 0, 0, 0};
          }
        }
        multiply(b, v);
      }
#pragma unroll
      for (int t = 0; t < MT; ++t)
      {
#pragma unroll
        for (int i = 0; i < 4; ++i)
        {
          s_sums[wave][t][i][lane] = acc[t][i];
        }
      }
      __syncthreads();
      for (int o = threadIdx.x; o < MT * 256; o += 64 * kWaves)
      {
        // Output o: column o % 16, row o / 16 of the rows; held by lane
        // 16 (row / 4 % 4) + column as its sum row % 4.
        const int n = n0 + o % 16, r = o / 16 % 16, t = o / 256;
        int sum = 0;
#pragma unroll
        for (int v = 0; v < kWaves; ++v)
        {
          sum += s_sums[v][t][r % 4][16 * (r / 4) + o % 16];
        }
        const int row = m0 + 16 * t + r;
        if (row < a.rows && n < a.features)
        {
          put<kHalf>(a, row, n, sum);
        }
      }
    }

    // Many rows: bound by the matrix cores. A workgroup of four waves, two by
    // two, takes 64 TM rows and 64 TN outputs, a wave 32 TM by 32 TN, with the
    // weight as the products' M and the rows as their N: a lane ends up with
    // four consecutive outputs of a row. Steps of 128 inputs, whole lines of
    // memory (steps of 64 ask L2 for each line twice: 8192^3 577 us, and 507),
    // pass through LDS, kStages of them, copied there directly: two stages where
    // two workgroups to a CU hide the copies, three where one is alone (1,777
    // rows 8192 -> 2048 40.4, by two 46.6). Piece c (16 bytes) of row t lies at
    // place c ^ (t / 2 % 8) of its row: sixteen lanes that read a piece of
    // sixteen rows meet no bank twice. A wave reads the operands of the next 32
    // inputs while it multiplies these. 8192^3 takes 507 us, 2,170 TOP/s, where the
    // library's product reaches 2,069; 4,096 rows 1536 -> 8960 (1,504 tiles, 5.9 a
    // CU) 69 to 77 us with the clocks; 1,777 rows 8192 -> 2048, 224 tiles for 256
    // CUs with a wave a SIMD, 40.4, waiting for copies two fifths of it.
    // Where that leaves the device workgroups too few, kGroups such sets of four
    // waves share a tile's inputs, with stages of their own, and the first adds
    // the others' sums up.
    // kTail: the last step is short, or a group's steps end before the others':
    // what is past the inputs counts as zeros.
    constexpr int kStep = 128; // inputs a step
    template <int TM, int TN, int kGroups, int kStages, bool kHalf, bool kTail>
    __global__ void __launch_bounds__(256 * kGroups, 2)
        int8_tiles_kernel(Int8Args a, int m_tiles, int n_tiles)
    {
      constexpr int kM = 64 * TM, kN = 64 * TN; // a workgroup's rows and outputs
      constexpr int kStage = (kM + kN) * kStep; // bytes: rows, then the weight's
      constexpr int kPieces = kStep / 16, kCopyRows = 256 / kPieces, kSame = 256 / kStep;
      constexpr int kCopies = kStage / 4096;    // 16-byte copies a lane a step
      constexpr int kPitch = 32 * TN * 4 + 16;  // bytes of a row of outputs in LDS
      extern __shared__ __align__(16) std::uint8_t all_stages[];
      const int lane = threadIdx.x & 63, thread = threadIdx.x % 256;
      const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6)) % 4;
      const int group = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x / 256));
      std::uint8_t *stages = all_stages + group * kStages * kStage;
      // Workgroups go to the eight XCDs in turn: each XCD takes consecutive
      // tiles, columns of up to eight row tiles, so that its L2 holds the
      // rows and outputs its workgroups share.
      const int total = m_tiles * n_tiles;
      const int xcd = blockIdx.x % 8, local = blockIdx.x / 8;
      int tile = xcd * (total / 8) + min(xcd, total % 8) + local;
      constexpr int kBand = 8;
      const int band = tile / (kBand * n_tiles);
      const int high = min(kBand, m_tiles - band * kBand);
      tile -= band * kBand * n_tiles;
      const int m0 = (band * kBand + tile % high) * kM;
      const int n0 = tile / high * kN;

      // A lane's copies: places i * 256 + thread, rows of eight.
      const std::uint8_t *x0 = a.x + static_cast<std::size_t>(m0) * a.in;
      const std::uint8_t *w0 = a.w + static_cast<std::size_t>(n0) * a.in;
      unsigned row_at[kCopies];
#pragma unroll
      for (int i = 0; i < kCopies; ++i)
      {
        const int t = i * kCopyRows + thread / kPieces;
        const int r = i * kCopyRows < kM ? min(t, a.rows - 1 - m0) : min(t - kM, a.features - 1 - n0);
        row_at[i] = static_cast<unsigned>(r) * a.in;
      }
      // The piece a lane copies: place % 8 of its row, turned by the row.
      const int piece = (thread % kPieces) ^ (thread / kPieces / kSame % kPieces);
      // The group's steps.
      const int steps = ((a.in + kStep - 1) / kStep + kGroups - 1) / kGroups, begin = group * steps;
      const auto copy = [&](int step, int stage) {
        // (Past the last input, of a short last step or those after it: any
        // piece.)
        const unsigned k = min(kStep * (begin + step) + 16 * piece, a.in - 16);
        std::uint8_t *to = stages + stage * kStage + wave * 1024;
#pragma unroll
        for (int i = 0; i < kCopies; ++i)
        {
          const std::uint8_t *from = (i * kCopyRows < kM ? x0 : w0) + (row_at[i] + k);
          __builtin_amdgcn_global_load_lds((global_void)from, (lds_void)(to + i * 4096), 16, 0, 0);
        }
      };

      const int n = lane & 31, half = lane >> 5;
      const int wm = wave / 2, wn = wave % 2;
      i32x16 acc[TN][TM];
#pragma unroll
      for (int j = 0; j < TN; ++j)
      {
#pragma unroll
        for (int i = 0; i < TM; ++i)
        {
#pragma unroll
          for (int e = 0; e < 16; ++e)
          {
            acc[j][i][e] = 0;
          }
        }
      }
      // Where the lane's row lies in a stage, and its pieces' turn.
      const int x_row = (32 * TM * wm + n) * kStep;
      const int w_row = (kM + 32 * TN * wn + n) * kStep;
      const int turn = n / kSame % kPieces;
      i32x4 x[2][TM], w[2][TN];
      // Half c of a step's operands.
      const auto read = [&](int c, int step, int stage) {
        const std::uint8_t *at = stages + stage * kStage;
        const int place = 16 * ((2 * c + half) ^ turn);
#pragma unroll
        for (int j = 0; j < TN; ++j)
        {
          i32x4 &codes = w[c % 2][j];
          codes = *reinterpret_cast<const i32x4 *>(at + w_row + 32 * kStep * j + place);
          if constexpr (kTail)
          {
            codes = kStep * (begin + step) + 16 * (2 * c + half) < a.in ? codes : i32x4{0, 0, 0, 0};
          }
        }
#pragma unroll
        for (int i = 0; i < TM; ++i)
        {
          x[c % 2][i] = *reinterpret_cast<const i32x4 *>(at + x_row + 32 * kStep * i + place);
        }
        __builtin_amdgcn_sched_barrier(0);
      };
      // Products [from, to) of half c.
      const auto multiply = [&](int c, int from, int to) {
#pragma unroll
        for (int p = 0; p < TN * TM; ++p)
        {
          if (p >= from && p < to)
          {
            i32x16 &sums = acc[p / TM][p % TM];
            sums = __builtin_amdgcn_mfma_i32_32x32x32_i8(w[c % 2][p / TM], x[c % 2][p % TM], sums, 0, 0, 0);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      };
#pragma unroll
      for (int i = 0; i < kStages; ++i)
      {
        copy(i, i);
      }
      asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(kCopies * (kStages - 1)) : "memory");
      read(0, 0, 0);
      int stage = 0;
      for (int step = 0; step < steps; ++step)
      {
        // (Operands are asked for behind a first product: its wait for its own
        // would be for them too.)
#pragma unroll
        for (int c = 0; c < kStep / 32 - 1; ++c)
        {
          multiply(c, 0, 1);
          read(c + 1, step, stage);
          multiply(c, 1, TN * TM);
        }
        // The next step's copies have landed, those of the steps after it may be
        // on their way; every wave has its operands of this one, whose stage the
        // next copies go to.
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(kCopies * (kStages - 2)) : "memory");
        multiply(1, 0, 1);
        copy(step + kStages, stage);
        stage = stage == kStages - 1 ? 0 : stage + 1;
        read(0, step + 1, stage);
        multiply(1, 1, TN * TM);
      }
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory"); // the copies past the last

      __syncthreads();
      if constexpr (kGroups > 1)
      {
        constexpr int kSums = 256 * 16 * TM * TN; // of a group
        int *sums = reinterpret_cast<int *>(all_stages) + thread;
        if (group > 0)
        {
          int *to = sums + (group - 1) * kSums;
#pragma unroll
          for (int e = 0; e < 16 * TM * TN; ++e)
          {
            to[256 * e] = acc[e / (16 * TM)][e / 16 % TM][e % 16];
          }
        }
        __syncthreads();
        if (group == 0)
        {
#pragma unroll
          for (int g = 1; g < kGroups; ++g)
          {
#pragma unroll
            for (int e = 0; e < 16 * TM * TN; ++e)
            {
              acc[e / (16 * TM)][e / 16 % TM][e % 16] += sums[(g - 1) * kSums + 256 * e];
            }
          }
        }
        __syncthreads(); // (the sums are read: their place is the outputs')
        if (group > 0)
        {
          return;
        }
      }
      // 32 rows at a time through the wave's own LDS, so that outputs leave
      // eight a lane in rows.
      std::uint8_t *own = stages + wave * (32 * kPitch);
      constexpr int kRowLanes = 32 * TN / 8; // lanes a row
      constexpr int kRowsOnce = 64 / kRowLanes; // (of 12 lanes a row, four lanes take none)
      const int col = n0 + 32 * TN * wn + 8 * (lane % kRowLanes);
      const bool full = col + 8 <= a.features;
      const bool vector = full && a.features % 8 == 0;
      float w_scale[8], bias[8];
#pragma unroll
      for (int e = 0; e < 8; ++e)
      {
        const int c = min(col + e, a.features - 1);
        w_scale[e] = a.w_scales[c];
        bias[e] = kHalf && a.bias != nullptr ? h2f(a.bias[c]) : 0.0f;
      }
#pragma unroll
      for (int i = 0; i < TM; ++i)
      {
#pragma unroll
        for (int j = 0; j < TN; ++j)
        {
#pragma unroll
          for (int g = 0; g < 4; ++g)
          {
            *reinterpret_cast<i32x4 *>(own + n * kPitch + 4 * (32 * j + 8 * g + 4 * half)) =
                i32x4{acc[j][i][4 * g], acc[j][i][4 * g + 1], acc[j][i][4 * g + 2], acc[j][i][4 * g + 3]};
          }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int p = 0; p < (32 + kRowsOnce - 1) / kRowsOnce; ++p)
        {
          const int r = p * kRowsOnce + lane / kRowLanes;
          const int row = m0 + 32 * (TM * wm + i) + r;
          if ((64 % kRowLanes != 0 && (lane >= kRowsOnce * kRowLanes || r >= 32)) || row >= a.rows)
          {
            continue;
          }
          const i32x4 lo = *reinterpret_cast<const i32x4 *>(own + r * kPitch + 32 * (lane % kRowLanes));
          const i32x4 hi = *reinterpret_cast<const i32x4 *>(own + r * kPitch + 32 * (lane % kRowLanes) + 16);
          const float x_scale = a.x_scales[row];
          float y[8];
#pragma unroll
          for (int e = 0; e < 8; ++e)
          {
            y[e] = scaled(e < 4 ? lo[e] : hi[e - 4], x_scale, w_scale[e]);
            if (kHalf && a.bias != nullptr)
            {
              y[e] += bias[e];
            }
          }
          const std::size_t at = static_cast<std::size_t>(row) * a.features + col;
          if constexpr (kHalf)
          {
            auto *out = static_cast<std::uint16_t *>(a.out) + at;
            unsigned bits[8];
#pragma unroll
            for (int e = 0; e < 8; ++e)
            {
              bits[e] = __half_as_ushort(__float2half(y[e]));
            }
            if (vector)
            {
              *reinterpret_cast<u32x4 *>(out) = u32x4{bits[0] | bits[1] << 16, bits[2] | bits[3] << 16,
                                                      bits[4] | bits[5] << 16, bits[6] | bits[7] << 16};
            }
            else
            {
#pragma unroll
              for (int e = 0; e < 8; ++e)
              {
                if (col + e < a.features)
                {
                  out[e] = static_cast<std::uint16_t>(bits[e]);
                }
              }
            }
          }
          else
          {
            auto *out = static_cast<float *>(a.out) + at;
            const float *residual = a.residual + at;
            if (vector)
            {
              const f32x4 r0 = *reinterpret_cast<const f32x4 *>(residual);
              const f32x4 r1 = *reinterpret_cast<const f32x4 *>(residual + 4);
              *reinterpret_cast<f32x4 *>(out) =
                  f32x4{r0[0] + y[0], r0[1] + y[1], r0[2] + y[2], r0[3] + y[3]};
              *reinterpret_cast<f32x4 *>(out + 4) =
                  f32x4{r1[0] + y[4], r1[1] + y[5], r1[2] + y[6], r1[3] + y[7]};
            }
            else
            {
#pragma unroll
              for (int e = 0; e < 8; ++e)
              {
                if (col + e < a.features)
                {
                  out[e] = residual[e] + y[e];
                }
              }
            }
          }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
      }
    }

    template <int MT, int kWaves>
    void rows_by(const Int8Args &a, hipStream_t stream)
    {
      const dim3 grid((a.features + 15) / 16, (a.rows + 16 * MT - 1) / (16 * MT));
      if (a.residual == nullptr)
      {
        int8_rows_kernel<MT, kWaves, true><<<grid, 64 * kWaves, 0, stream>>>(a);
      }
      else
      {
        int8_rows_kernel<MT, kWaves, false><<<grid, 64 * kWaves, 0, stream>>>(a);
      }
      hip_check(hipGetLastError(), "int8_rows_kernel");
    }

    template <int MT>
    void rows_as(const Int8Args &a, hipStream_t stream)
    {
      // As many waves to an output's inputs as fill the device, a step at
      // least each.
      const long long tiles = (a.features + 15ll) / 16 * ((a.rows + 16ll * MT - 1) / (16 * MT));
      const int steps = (a.in + 127) / 128;
      const long long want = std::min<long long>(steps, 4096 / std::max<long long>(1, tiles));
      want >= 16 ? rows_by<MT, 16>(a, stream)
                 : want >= 8 ? rows_by<MT, 8>(a, stream)
                             : want >= 4 ? rows_by<MT, 4>(a, stream) : rows_by<MT, 2>(a, stream);
    }

    template <int TM, int TN, int kGroups, int kStages, bool kHalf, bool kTail>
    void tiles_by(const Int8Args &a, hipStream_t stream)
    {
      constexpr std::size_t stages = kGroups * kStages * (64 * TM + 64 * TN) * kStep;
      constexpr std::size_t outs = 4 * 32 * (32 * TN * 4 + 16);
      constexpr std::size_t sums = (kGroups - 1) * sizeof(int) * 256 * 16 * TM * TN;
      constexpr std::size_t lds = std::max({stages, outs, sums});
      auto kernel = int8_tiles_kernel<TM, TN, kGroups, kStages, kHalf, kTail>;
      if constexpr (lds > 64 * 1024)
      {
        hip_check(hipFuncSetAttribute(reinterpret_cast<const void *>(kernel),
                                      hipFuncAttributeMaxDynamicSharedMemorySize,
                                      static_cast<int>(lds)),
                  "hipFuncSetAttribute int8 LDS");
      }
      const int m_tiles = (a.rows + 64 * TM - 1) / (64 * TM);
      const int n_tiles = (a.features + 64 * TN - 1) / (64 * TN);
      kernel<<<static_cast<unsigned>(m_tiles) * n_tiles, 256 * kGroups, lds, stream>>>(a, m_tiles, n_tiles);
      hip_check(hipGetLastError(), "int8_tiles_kernel");
    }

    template <int TM, int TN, int kGroups, int kStages>
    void tiles_as(const Int8Args &a, hipStream_t stream)
    {
      if (a.in % (kStep * kGroups) == 0)
      {
        a.residual == nullptr ? tiles_by<TM, TN, kGroups, kStages, true, false>(a, stream)
                              : tiles_by<TM, TN, kGroups, kStages, false, false>(a, stream);
      }
      else
      {
        a.residual == nullptr ? tiles_by<TM, TN, kGroups, kStages, true, true>(a, stream)
                              : tiles_by<TM, TN, kGroups, kStages, false, true>(a, stream);
      }
    }

    void check_features(int features, const char *what)
    {
      if (features < 0 || features % 16 != 0)
      {
        throw InvalidArgument(std::string(what) + " " + std::to_string(features) +
                              " must not be negative, and whole sixteens");
      }
    }

    bool aligned(const void *p) { return reinterpret_cast<std::uintptr_t>(p) % 16 == 0; }
  } // namespace

  void launch_quantise_rows_int8(const void *x, long long stride, void *codes, float *scales,
                                 int rows, int features, hipStream_t stream)
  {
    check_features(features, "features");
    if (rows < 0 || stride < 0)
    {
      throw InvalidArgument("rows and stride must not be negative, got " + std::to_string(rows) +
                            " and " + std::to_string(stride));
    }
    if (rows == 0)
    {
      return;
    }
    if (features == 0)
    {
      throw InvalidArgument("rows to quantise have values");
    }
    if (x == nullptr || codes == nullptr || scales == nullptr)
    {
      throw InvalidArgument("rows to quantise need x, codes and scales");
    }
    // A wave a row up to 2,048 values, else a workgroup; a launch has fewer than
    // 2^32 threads.
    const int runs = features / 8;
    const int most_rows = 0xffffff * (runs <= 256 ? 4 : 1);
    if (rows > most_rows)
    {
      throw InvalidArgument("at most " + std::to_string(most_rows) + " rows of " +
                            std::to_string(features) + " values are quantised at once, got " +
                            std::to_string(rows));
    }
    stride = stride > 0 ? stride : features;
    if (stride < features || stride % 8 != 0)
    {
      throw InvalidArgument("rows to quantise are a multiple of 8 elements apart, and their own " +
                            std::to_string(features) + " at least; got " + std::to_string(stride));
    }
    if (!aligned(x) || !aligned(codes) || reinterpret_cast<std::uintptr_t>(scales) % 4 != 0)
    {
      throw InvalidArgument("rows to quantise and their codes must be 16-byte aligned");
    }
    const std::size_t count = static_cast<std::size_t>(rows) * features;
    const Extent read{x, 2 * static_cast<std::size_t>(features), static_cast<std::size_t>(rows),
                      2 * static_cast<std::size_t>(stride)};
    const Extent code_bytes{codes, count}, scale_bytes{scales, 4 * static_cast<std::size_t>(rows)};
    if (overlaps(code_bytes, read) || overlaps(scale_bytes, read) || overlaps(code_bytes, scale_bytes))
    {
      throw InvalidArgument("codes and scales cannot write over the rows or one another");
    }
    const auto *from = static_cast<const std::uint16_t *>(x);
    auto *to = static_cast<std::uint8_t *>(codes);
    const unsigned blocks = static_cast<unsigned>(rows);
    const unsigned fours = (blocks + 3) / 4;
    if (runs <= 64)
    {
      quantise_rows_kernel<64, 1><<<fours, 256, 0, stream>>>(from, stride, to, scales, rows, runs);
    }
    else if (runs <= 128)
    {
      quantise_rows_kernel<64, 2><<<fours, 256, 0, stream>>>(from, stride, to, scales, rows, runs);
    }
    else if (runs <= 256)
    {
      quantise_rows_kernel<64, 4><<<fours, 256, 0, stream>>>(from, stride, to, scales, rows, runs);
    }
    else if (runs <= 1024)
    {
      quantise_rows_kernel<256, 4><<<blocks, 256, 0, stream>>>(from, stride, to, scales, rows, runs);
    }
    else if (runs <= 2048)
    {
      quantise_rows_kernel<256, 8><<<blocks, 256, 0, stream>>>(from, stride, to, scales, rows, runs);
    }
    else
    {
      quantise_rows_kernel<256, 0><<<blocks, 256, 0, stream>>>(from, stride, to, scales, rows, runs);
    }
    hip_check(hipGetLastError(), "quantise_rows_kernel");
  }

  void launch_linear_int8(const Int8Linear &t, hipStream_t stream)
  {
    check_features(t.in, "in_features");
    if (t.rows < 0 || t.features < 0)
    {
      throw InvalidArgument("rows and out_features must not be negative, got " +
                            std::to_string(t.rows) + " and " + std::to_string(t.features));
    }
    if (t.rows == 0 || t.features == 0)
    {
      return;
    }
    constexpr int kMostInputs = 1 << 17; // 2^17 products of up to 2^14 leave 32 bits
    if (t.in == 0 || t.in >= kMostInputs)
    {
      throw InvalidArgument("an int8 projection takes 16 to " + std::to_string(kMostInputs - 16) +
                            " in_features, got " + std::to_string(t.in));
    }
    constexpr int kMostOutputs = 1 << 27, kMostRows = 1 << 21; // a launch's workgroups
    if (t.features > kMostOutputs || t.rows > kMostRows ||
        static_cast<long long>((t.rows + 127) / 128) * ((t.features + 127) / 128) > 0xffffff)
    {
      throw InvalidArgument("an int8 projection takes at most " + std::to_string(kMostRows) +
                            " rows, " + std::to_string(kMostOutputs) +
                            " out_features and 2^24 tiles of 128 by 128 of them, got " +
                            std::to_string(t.rows) + " and " + std::to_string(t.features));
    }
    if (t.x == nullptr || t.x_scales == nullptr || t.w == nullptr || t.w_scales == nullptr ||
        t.out == nullptr)
    {
      throw InvalidArgument("an int8 projection needs x, its scales, the weight, its scales and out");
    }
    const std::uintptr_t words = reinterpret_cast<std::uintptr_t>(t.x_scales) |
                                 reinterpret_cast<std::uintptr_t>(t.w_scales);
    if (!aligned(t.x) || !aligned(t.w) || !aligned(t.out) || !aligned(t.residual) || words % 4 != 0)
    {
      throw InvalidArgument("an int8 projection's codes and outputs must be 16-byte aligned");
    }
    const std::size_t rows = static_cast<std::size_t>(t.rows), outs = static_cast<std::size_t>(t.features);
    const std::size_t in = static_cast<std::size_t>(t.in);
    const Extent written{t.out, (t.residual == nullptr ? 2 : 4) * rows * outs};
    const Extent residual{t.residual != t.out ? t.residual : nullptr, 4 * rows * outs};
    for (const Extent &read : {Extent{t.x, rows * in}, Extent{t.x_scales, 4 * rows},
                               Extent{t.w, outs * in}, Extent{t.w_scales, 4 * outs},
                               Extent{t.bias, 2 * outs}, residual})
    {
      if (overlaps(written, read))
      {
        throw InvalidArgument("an int8 projection cannot write over its input or weight");
      }
    }
    Int8Args a{};
    a.x = static_cast<const std::uint8_t *>(t.x);
    a.x_scales = t.x_scales;
    a.w = static_cast<const std::uint8_t *>(t.w);
    a.w_scales = t.w_scales;
    a.bias = static_cast<const std::uint16_t *>(t.bias);
    a.residual = t.residual;
    a.out = t.out;
    a.rows = t.rows;
    a.in = t.in;
    a.features = t.features;
    // By the workgroups that a tile of 64 by 64 would make. Few tiles of few rows
    // read the weight straight (us as rows and tiles: 1 row 1536 -> 8960 5.6 and
    // 5.8, 8960 -> 1536 7.5 and 15.7, 32 rows 4096 -> 4096 8.0 and 9.8; but 24
    // rows 2048 -> 8192 7.2 and 6.9, 16 rows 2048 -> 32000 17.5 and 14.1). As many
    // workgroups as compute units or fewer want the smallest tile, its inputs
    // shared by two groups (256 rows 8960 -> 1536 16.9, by 64 by 128 24.2); then
    // the tile grows as far as it leaves every CU one: 64 by 128 (1,000 rows 8960
    // -> 1536 26.5, by the smallest 33.1, by 128 by 128 47.2), also where 64 rows
    // are all there are, 128 by 128 (2,048 rows 2048 -> 2048 13.9, by 64 by 128
    // 14.3, by 128 by 192 18.3), and 128 by 192, two to a CU, which reads LDS less
    // for its products (1,000 rows 1536 -> 8960 23.7, by 128 by 128 27.3, by 128 by
    // 256 37; 4,096 rows 1536 -> 8960 69, 73 and 97; 8192^3 507, 554 and 615).
    const long long tiles = (t.rows + 63ll) / 64 * ((t.features + 63ll) / 64);
    if (t.rows <= 64 && t.rows * tiles <= 2048)
    {
      t.rows <= 16 ? rows_as<1>(a, stream) : rows_as<2>(a, stream);
    }
    else if (tiles <= 256)
    {
      tiles_as<1, 1, 2, 3>(a, stream);
    }
    else if (tiles <= 640 || t.rows <= 64)
    {
      tiles_as<1, 2, 1, 3>(a, stream);
    }
    else if ((t.rows + 127ll) / 128 * ((t.features + 127ll) / 128) <= 256)
    {
      tiles_as<2, 2, 1, 3>(a, stream);
    }
    else
    {
      tiles_as<2, 3, 1, 2>(a, stream);
    }
  }

} // namespace mi
