// Attention of a prompt's queries over contiguous keys and values, causal,
// through a sliding window with the first `sinks` tokens kept visible.
//
// Query i of seq_q is at position p = seq_k - seq_q + i and sees key j <= p if
// there is no window, or j > p - window, or j < sinks. out = softmax(q . k /
// sqrt(hd)) v over those; every query sees itself at least.
//
// A workgroup takes one KV head and consecutive (query, head) rows of its
// group, query by query, so that its rows' windows nearly coincide, in tiles of
// 32; a tile's waves share the keys of a step and join their sums at the end.
// Steps of kKeys keys, of which only those some row of the workgroup
// sees are taken (the sink steps, then the window's), pass through LDS, double
// buffered, copied there directly from memory. In the matrix cores' terms,
// with keys as M and rows as N:
//   S^T (32 keys x 32 rows) = K . Q^T      lane l holds row l % 32
//   O^T (32 channels x 32 rows) += V^T . P^T  P from the lane's own scores,
//                                             V^T by transposing LDS reads
// so that the softmax stays in a lane but for one exchange with lane ^ 32.
//
// A key or value in LDS lies in 16-byte pieces, piece c of row t at place
// c ^ swizzle(t) of its row: the 16 lanes that read one piece of 16 rows, and
// the 32 lanes that a transposing read serves at a time (four rows, four
// pieces), meet no bank twice.
//
// P is rounded to fp16 once (half a step is 2^-11 of a weight, as much as the
// output's own rounding; the sums are of the rounded weights, so that the
// output stays an average of the values), held against a reference that is
// moved up only when a score passes it by 2^kRise: P is at most
// 2^(kRise + kProb) = 2^14, and a weight keeps its 11 bits down to 2^-22 of
// the reference.
//
// With few rows the range of keys is split over workgroups, whose parts a
// second launch joins.
//
// Bound by vector and matrix work that take turns. 2,048 queries x 32 heads at
// 14,336 behind a 4,096-token window with 4 sinks, head_dim 64: 103 us, 668
// TFLOP/s; of the 253 M SIMD cycles in it vector instructions take some 166 M
// (28.8 M of them, 4 cycles each, the exponentials, 16 a lane of a 32 x 32 tile,
// at a quarter of that rate) and the products 69 M, together nearly all: the
// waves of a SIMD pass the step's barrier together and do the same kind of work
// at the same time. A prompt of 4,096 x 12 heads of 128 behind 1,024: 57.6 us,
// 393 TFLOP/s, vector work 43 M and products 25 M of 141 M cycles, its 384
// workgroups of unequal ranges leaving half the CUs one instead of two. 100 queries x 14 heads of 64:
// 5.9 us, a launch and a chain of loads. Measured and not taken: 64 rows a
// wave (158 us for the first of these, one wave a SIMD), the next step's first
// product beside this step's exponentials (the same at head_dim 64; 90 us for
// the second, out of registers), addresses a lane keeps instead of making, KV
// heads first in the order of workgroups (the same; 95% of reads meet the L2
// either way).

#include "common.hpp"
#include "lane_ops.hpp"
#include "serving.hpp"

#include <algorithm>
#include <cmath>
#include <string>
#include <type_traits>

namespace mi
{
  namespace
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
    constexpr int kMaxSplits = 256;
    constexpr int kFewSplits = 8; // that a lane joins one after another

    struct WindowArgs
    {
      const std::uint16_t *q;
      const std::uint16_t *k;
      const std::uint16_t *v;
      std::uint16_t *out;
      long long q_stride; // elements between tokens
      long long k_stride;
      long long v_stride;
      int seq_q;
      int seq_k;
      int heads;
      int kv_heads;
      int group;
      int window; // 0: none
      int sinks;
      int splits;
      float scale;    // log2 e / sqrt(hd)
      float *part_ml; // splits > 1: [split][row] maximum and sum (row = query * heads + head),
      float *part_o;  // and hd outputs
    };

    __device__ inline half8 as_half8(u32x4 v) { return __builtin_bit_cast(half8, v); }

    __device__ inline f32x16 mfma32(half8 a, half8 b, f32x16 c)
    {
      return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }

    // The place of piece c of row t (see above): for rows of 8 pieces two rows
    // span the banks, so rows differ by t / 2; bits reversed, so that rows 0-3
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

    // The keys of steps: [0, sink_steps) and from `first` on.
    struct Steps
    {
      int sink_steps;
      int first; // the window's first step
      int count;
      __device__ int key(int i, int keys) const
      {
        return (i < sink_steps ? i : first + i - sink_steps) * keys;
      }
    };

    // Waves a SIMD that a form's registers are held to: four at head_dim 64
    // (128 registers), two at 128 (256); few rows leave a wave alone anyway.
    template <int HD, int kTiles>
    constexpr int kWavesASimd = kTiles == 1 ? 1 : HD == 64 ? 4 : 2;

    template <int HD, int kTiles, int kWays, int kKeys>
    __global__ void __launch_bounds__(64 * kTiles * kWays, (kWavesASimd<HD, kTiles>))
        window_kernel(WindowArgs a)
    {
      constexpr int NW = kTiles * kWays;
      constexpr int kPieces = HD / 8;          // 16-byte pieces a row
      constexpr int kTile = kKeys * HD;        // halves of a step's keys
      constexpr int kStage = 2 * kTile;        // keys, then values
      constexpr int kRows = 32 * kTiles;       // rows a workgroup
      constexpr int kWayKeys = kKeys / kWays;
      constexpr int N = kWayKeys / 32;
      extern __shared__ __align__(16) std::uint16_t stages[]; // two of kStage

      const int lane = threadIdx.x & 63;
      const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
      const int way = wave / kTiles;
      const int n = lane & 31;
      const int half = lane >> 5;
      const int kvh = blockIdx.y;
      const int split = blockIdx.z;
      const int G = a.group;
      const int past = a.seq_k - a.seq_q;
      const long long all_rows = static_cast<long long>(a.seq_q) * G;
      // The last queries, whose ranges are longest, go first.
      const long long row0 = static_cast<long long>(gridDim.x - 1 - blockIdx.x) * kRows;

      // The workgroup's positions, and the steps they see.
      const int lo_pos = past + static_cast<int>(row0 / G);
      const int hi_pos = past + static_cast<int>((min(row0 + kRows, all_rows) - 1) / G);
      Steps steps{0, 0, 0};
      if (a.window > 0 && a.window <= lo_pos)
      {
        steps.first = (lo_pos - a.window + 1) / kKeys;
        steps.sink_steps = min(a.sinks / kKeys + (a.sinks % kKeys > 0 ? 1 : 0), steps.first);
      }
      steps.count = steps.sink_steps + hi_pos / kKeys + 1 - steps.first;
      const int per = (steps.count + a.splits - 1) / a.splits;
      const int begin = min(split * per, steps.count);
      const int end = min(begin + per, steps.count);

      // The wave's rows (a wave past the last computes nothing), and the lane's.
      const long long wave_row = row0 + 32 * (wave % kTiles);
      const bool computes = wave_row < all_rows;
      const int wave_lo = past + static_cast<int>(min(wave_row, all_rows - 1) / G);
      const int wave_hi = past + static_cast<int>((min(wave_row + 32, all_rows) - 1) / G);
      const long long row = wave_row + n;
      const bool valid = row < all_rows;
      const int query = valid ? static_cast<int>(row / G) : 0;
      const int head = kvh * G + (valid ? static_cast<int>(row % G) : 0);
      const int pos = past + query;
      const std::size_t row_at = static_cast<std::size_t>(query) * a.heads + head;
      half8 q[HD / 16];
      const std::uint16_t *q_row = a.q + query * a.q_stride + head * HD + 8 * half;
#pragma unroll
      for (int c = 0; c < HD / 16; ++c)
      {
        q[c] = as_half8(*reinterpret_cast<const u32x4 *>(q_row + 16 * c));
      }
      Rows<HD> run;
      run.m = -INFINITY;
      run.l = 0.0f;
#pragma unroll
      for (int d = 0; d < HD / 32; ++d)
      {
#pragma unroll
        for (int i = 0; i < 16; ++i)
        {
          run.o[d][i] = 0.0f;
        }
      }

      // A step's rows to LDS, 16 bytes a lane; rows past the last repeat it.
      const auto copy = [&](int step, int buf) {
        const int key0 = steps.key(step, kKeys);
        std::uint16_t *stage = stages + buf * kStage;
#pragma unroll
        for (int i = 0; i < kTile / 8 / (64 * NW); ++i)
        {
          const int place = (i * NW + wave) * 64 + lane;
          const int t = place / kPieces;
          const int c = (place % kPieces) ^ swizzle<HD>(t);
          const long long key = min(key0 + t, a.seq_k - 1);
          std::uint16_t *to = stage + (i * NW + wave) * 512;
          __builtin_amdgcn_global_load_lds(
              (global_void)(a.k + key * a.k_stride + kvh * HD + 8 * c), (lds_void)(to), 16, 0, 0);
          __builtin_amdgcn_global_load_lds(
              (global_void)(a.v + key * a.v_stride + kvh * HD + 8 * c), (lds_void)(to + kTile), 16,
              0, 0);
        }
      };
      if (begin < end)
      {
        copy(begin, 0);
      }
      for (int step = begin; step < end; ++step)
      {
        const int buf = (step - begin) & 1;
        // This step's copies have landed (a wave waits for its own before the
        // barrier), and every wave is done with the other buffer.
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_s_waitcnt(0x0F70); // vmcnt(0)
        __syncthreads();
        if (step + 1 < end)
        {
          copy(step + 1, buf ^ 1);
        }
        const int key0 = steps.key(step, kKeys) + way * kWayKeys;
        const bool sees = key0 <= wave_hi &&
                          (a.window == 0 || key0 + kWayKeys - 1 > wave_lo - a.window ||
                           key0 < a.sinks);
        if (!computes || !sees)
        {
          continue;
        }
        const std::uint16_t *keys = stages + buf * kStage + way * kWayKeys * HD;
        const std::uint16_t *values = keys + kTile;
        f32x16 s[N];
#pragma unroll
        for (int j = 0; j < N; ++j)
        {
#pragma unroll
          for (int i = 0; i < 16; ++i)
          {
            s[j][i] = 0.0f;
          }
        }
#pragma unroll
        for (int c = 0; c < HD / 16; ++c)
        {
#pragma unroll
          for (int j = 0; j < N; ++j)
          {
            const int t0 = 32 * j + n;
            const half8 k = as_half8(*reinterpret_cast<const u32x4 *>(
                keys + t0 * HD + 8 * ((2 * c + half) ^ swizzle<HD>(t0))));
            s[j] = mfma32(k, q[c], s[j]);
          }
        }
        // Whether some row of the wave does not see some key of the step.
        const bool edge = key0 + kWayKeys - 1 > wave_lo ||
                          (a.window > 0 && key0 <= wave_hi - a.window &&
                           key0 + kWayKeys > a.sinks);
        if (edge)
        {
          const int from = a.window > 0 ? pos - a.window : -1; // keys after it are seen
#pragma unroll
          for (int j = 0; j < N; ++j)
          {
#pragma unroll
            for (int i = 0; i < 16; ++i)
            {
              const int key = key0 + 32 * j + 8 * (i / 4) + 4 * half + i % 4;
              const bool seen = key <= pos && (key > from || key < a.sinks);
              s[j][i] = seen ? s[j][i] : -INFINITY;
            }
          }
        }
        half8 p[N][2];
        float top = s[0][0];
#pragma unroll
        for (int j = 0; j < N; ++j)
        {
#pragma unroll
          for (int i = 0; i < 16; ++i)
          {
            top = fmaxf(top, s[j][i]);
          }
        }
        top = lane_max32(top) * a.scale;
        if (__any(top > run.m + kRise))
        {
          const float m = fmaxf(run.m, top);
          const float keep = run.m == m ? 1.0f : __builtin_amdgcn_exp2f(run.m - m);
          run.m = m;
          run.l *= keep;
#pragma unroll
          for (int d = 0; d < HD / 32; ++d)
          {
            run.o[d] *= keep;
          }
        }
        const float from = (run.m == -INFINITY ? 0.0f : run.m) - kProb;
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < N; ++j)
        {
#pragma unroll
          for (int i = 0; i < 16; i += 2)
          {
            const f32x2 w = {
                __builtin_amdgcn_exp2f(__builtin_fmaf(s[j][i], a.scale, -from)),
                __builtin_amdgcn_exp2f(__builtin_fmaf(s[j][i + 1], a.scale, -from))};
            const half2v h = __builtin_convertvector(w, half2v);
            const _Float16 one = static_cast<_Float16>(1.0f);
            sum = __builtin_amdgcn_fdot2(h, half2v{one, one}, sum, false);
            p[j][i / 8][i % 8] = h[0];
            p[j][i / 8][i % 8 + 1] = h[1];
          }
        }
        run.l += sum;
        // A value some row does not see may be anything: if one of an edge
        // step's is not finite, the products take it as zero, and the rows
        // that do see it add it after them.
        const bool spoilt = edge && !finite_values<HD, kWayKeys>(values, lane);
        // Lane l's P of a 16-key product: keys 8 e + 4 half + {0..3}, e = 0, 1.
#pragma unroll
        for (int j = 0; j < N; ++j)
        {
#pragma unroll
          for (int u = 0; u < 2; ++u)
          {
#pragma unroll
            for (int d = 0; d < HD / 32; ++d)
            {
              half8 vt;
#pragma unroll
              for (int e = 0; e < 2; ++e)
              {
                const int t0 = 32 * j + 16 * u + 8 * e + 4 * half + (lane % 16) / 4;
                const int ch = 32 * d + 16 * ((lane / 16) & 1) + 4 * (lane % 4);
                const half4 x = transposed(values + t0 * HD +
                                           8 * ((ch / 8) ^ swizzle<HD>(t0)) + ch % 8);
                vt[4 * e] = x[0];
                vt[4 * e + 1] = x[1];
                vt[4 * e + 2] = x[2];
                vt[4 * e + 3] = x[3];
              }
              if (spoilt)
              {
                vt = finite_only(vt);
              }
              run.o[d] = mfma32(vt, p[j][u], run.o[d]);
            }
          }
        }
        if (spoilt)
        {
          for (int key = key0; key < min(key0 + kWayKeys, a.seq_k); ++key)
          {
            const std::uint16_t *spoilt_row = values + (key - key0) * HD;
            const int swap = swizzle<HD>(key - key0);
#pragma unroll
            for (int d = 0; d < HD / 32; ++d)
            {
#pragma unroll
              for (int i = 0; i < 16; ++i)
              {
                const int ch = 32 * d + 8 * (i / 4) + 4 * half + i % 4;
                const std::uint16_t v = spoilt_row[8 * ((ch / 8) ^ swap) + ch % 8];
                const bool seen = key <= pos && (a.window == 0 || key > pos - a.window ||
                                                 key < a.sinks);
                run.o[d][i] += seen && !is_finite(v) ? h2f(v) : 0.0f;
              }
            }
          }
        }
      }

      if constexpr (kWays > 1)
      {
        // The ways' sums joined by the first way's wave.
        constexpr int kHeld = (HD / 2 + 2) * 64; // floats a wave leaves
        float *left = reinterpret_cast<float *>(stages);
        __syncthreads();
        if (way > 0)
        {
          float *to = left + (wave - kTiles) * kHeld + lane;
          to[0] = run.m;
          to[64] = run.l;
#pragma unroll
          for (int i = 0; i < HD / 2; ++i)
          {
            to[64 * (2 + i)] = run.o[i / 16][i % 16];
          }
        }
        __syncthreads();
        if (way > 0)
        {
          return;
        }
        float m[kWays];
        m[0] = run.m;
        float top = run.m;
#pragma unroll
        for (int w = 1; w < kWays; ++w)
        {
          m[w] = left[((w - 1) * kTiles + wave) * kHeld + lane];
          top = fmaxf(top, m[w]);
        }
        const float keep = m[0] == top ? 1.0f : __builtin_amdgcn_exp2f(m[0] - top);
        run.m = top;
        run.l *= keep;
#pragma unroll
        for (int d = 0; d < HD / 32; ++d)
        {
          run.o[d] *= keep;
        }
#pragma unroll
        for (int w = 1; w < kWays; ++w)
        {
          const float *from = left + ((w - 1) * kTiles + wave) * kHeld + lane;
          const float weight = m[w] == top ? 1.0f : __builtin_amdgcn_exp2f(m[w] - top);
          run.l = __builtin_fmaf(from[64], weight, run.l);
#pragma unroll
          for (int i = 0; i < HD / 2; ++i)
          {
            run.o[i / 16][i % 16] =
                __builtin_fmaf(from[64 * (2 + i)], weight, run.o[i / 16][i % 16]);
          }
        }
      }
      const float sum = lane_sum32(run.l) * kProbUnscale;
      if (!valid)
      {
        return;
      }
      if (a.splits == 1)
      {
        const float inv = kProbUnscale / sum;
        std::uint16_t *out = a.out + row_at * HD + 4 * half;
#pragma unroll
        for (int d = 0; d < HD / 32; ++d)
        {
#pragma unroll
          for (int b = 0; b < 4; ++b)
          {
            const f32x16 &o = run.o[d];
            const half2v x = {static_cast<_Float16>(o[4 * b] * inv),
                              static_cast<_Float16>(o[4 * b + 1] * inv)};
            const half2v y = {static_cast<_Float16>(o[4 * b + 2] * inv),
                              static_cast<_Float16>(o[4 * b + 3] * inv)};
            *reinterpret_cast<u32x2 *>(out + 32 * d + 8 * b) =
                u32x2{__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, y)};
          }
        }
        return;
      }
      const std::size_t at = static_cast<std::size_t>(split) * a.seq_q * a.heads + row_at;
      if (half == 0)
      {
        *reinterpret_cast<f32x2 *>(a.part_ml + 2 * at) = f32x2{run.m, sum};
      }
      float *out = a.part_o + at * HD + 4 * half;
#pragma unroll
      for (int d = 0; d < HD / 32; ++d)
      {
#pragma unroll
        for (int b = 0; b < 4; ++b)
        {
          f32x4 x;
#pragma unroll
          for (int i = 0; i < 4; ++i)
          {
            x[i] = run.o[d][4 * b + i] * kProbUnscale;
          }
          *reinterpret_cast<f32x4 *>(out + 32 * d + 8 * b) = x;
        }
      }
    }

    // The splits of a (query, head) row joined, four channels a thread.
    template <int HD>
    __global__ void __launch_bounds__(256) window_join_kernel(WindowArgs a, std::size_t rows)
    {
      constexpr int kLanes = HD / 4;
      const std::size_t i = static_cast<std::size_t>(blockIdx.x) * 256 + threadIdx.x;
      const std::size_t row = i / kLanes;
      const int d = 4 * static_cast<int>(i % kLanes);
      if (row >= rows)
      {
        return;
      }
      float top = -INFINITY;
#pragma unroll 4
      for (int s = 0; s < a.splits; ++s)
      {
        top = fmaxf(top, a.part_ml[2 * (s * rows + row)]);
      }
      const float from = top == -INFINITY ? 0.0f : top;
      float sum = 0.0f;
      f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
      for (int s = 0; s < a.splits; ++s)
      {
        const f32x2 ml = *reinterpret_cast<const f32x2 *>(a.part_ml + 2 * (s * rows + row));
        const f32x4 o = *reinterpret_cast<const f32x4 *>(a.part_o + (s * rows + row) * HD + d);
        const float w = __builtin_amdgcn_exp2f(ml[0] - from);
        sum += ml[1] * w;
        acc += o * w;
      }
      const half2v x = {static_cast<_Float16>(acc[0] / sum), static_cast<_Float16>(acc[1] / sum)};
      const half2v y = {static_cast<_Float16>(acc[2] / sum), static_cast<_Float16>(acc[3] / sum)};
      *reinterpret_cast<u32x2 *>(a.out + row * HD + d) =
          u32x2{__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, y)};
    }

    // The same for many splits: a workgroup a row, its groups of lanes each
    // taking some, with maxima of their own (one query over 7,000 keys, 56 splits:
    // 17.8 us in all with the kernel above, 9.9 with this).
    template <int HD>
    __global__ void __launch_bounds__(256) window_join_row_kernel(WindowArgs a, std::size_t rows)
    {
      constexpr int kLanes = HD / 4, kGroups = 256 / kLanes;
      __shared__ f32x2 s_ml[kGroups];
      __shared__ __align__(16) float s_o[kGroups][HD];
      const std::size_t row = blockIdx.x;
      const int group = threadIdx.x / kLanes;
      const int d = 4 * static_cast<int>(threadIdx.x % kLanes);
      float m = -INFINITY, l = 0.0f;
      f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
      for (int s = group; s < a.splits; s += kGroups)
      {
        const f32x2 ml = *reinterpret_cast<const f32x2 *>(a.part_ml + 2 * (s * rows + row));
        const f32x4 x = *reinterpret_cast<const f32x4 *>(a.part_o + (s * rows + row) * HD + d);
        const float top = fmaxf(m, ml[0]);
        const float from = top == -INFINITY ? 0.0f : top;
        const float keep = __builtin_amdgcn_exp2f(m - from), w = __builtin_amdgcn_exp2f(ml[0] - from);
        l = l * keep + ml[1] * w;
        o = o * keep + x * w;
        m = top;
      }
      if (d == 0)
      {
        s_ml[group] = f32x2{m, l};
      }
      *reinterpret_cast<f32x4 *>(&s_o[group][d]) = o;
      __syncthreads();
      if (threadIdx.x >= HD)
      {
        return;
      }
      float from = -INFINITY;
#pragma unroll
      for (int i = 0; i < kGroups; ++i)
      {
        from = fmaxf(from, s_ml[i][0]);
      }
      from = from == -INFINITY ? 0.0f : from;
      float sum = 0.0f, out = 0.0f;
#pragma unroll
      for (int i = 0; i < kGroups; ++i)
      {
        const float w = __builtin_amdgcn_exp2f(s_ml[i][0] - from);
        sum += s_ml[i][1] * w;
        out += s_o[i][threadIdx.x] * w;
      }
      a.out[row * HD + threadIdx.x] =
          __builtin_bit_cast(std::uint16_t, static_cast<_Float16>(out / sum));
    }

    // A launch's form: the row tiles of a workgroup, the waves that share a
    // tile's keys, and the keys a step. Few rows are a matter of latency, so
    // four waves take a quarter of a step's keys each (100 queries x 14 heads
    // of 64 by one wave 9.1 us, by four 5.9). Many at head_dim 64 have the
    // registers for four waves a SIMD, two to a tile, and one barrier in 128
    // keys (2,048 queries x 32 heads at 14K behind 4,096: one wave to a tile
    // and 64 keys a step 110 us, two 104, and 128 keys 100.5). At 128 a wave's
    // output and queries allow two a SIMD, and tiles of half the rows, or
    // three waves a SIMD, cost more than they balance (4,096 x 12 heads behind
    // 1,024: 57.5 us, 65.6 and 124).
    template <int kTiles_, int kWays_, int kKeys_>
    struct Form
    {
      static constexpr int tiles = kTiles_, ways = kWays_, keys = kKeys_, rows = 32 * kTiles_;
    };
    using Few = Form<1, 4, 128>;
    using Many64 = Form<4, 2, 128>;
    using Many128 = Form<4, 1, 64>;

    // How a launch is cut.
    struct Cut
    {
      bool few;
      int rows; // a workgroup's rows, and keys a step
      int keys;
      int blocks; // workgroups over the rows, a KV head
      int splits; // workgroups over a row's keys
    };

    Cut cut_of(const WindowAttention &t, bool may_split)
    {
      const int group = t.heads / t.kv_heads;
      const long long rows = static_cast<long long>(t.seq_q) * group;
      Cut c{};
      // The keys that a row sees, and the sink steps beside them.
      const long long span =
          t.window > 0 ? std::min<long long>(t.seq_k, static_cast<long long>(t.window) + t.sinks)
                       : t.seq_k;
      // Few: what leaves no CU two of those workgroups; over long spans, where
      // 32 rows are too few to share a step's copies, a half or a quarter of
      // that; at head_dim 64, whose stages leave room, twice as many for short
      // ones. Measured in us, few against many: 1,024 x 14 heads of 64 behind
      // 64 keys 11 and 15; 512 x 32 over 512 keys 10.7 and 12.9; 256 x 32 over
      // 1,256 16.7 and 18.2, over 3,256 34.5 and 23.2; 400 x 12 of 128 over 400
      // 12.7 and 17.6, over 3,400 48.7 and 38.3; 256 x 12 over 3,256 32.3 and
      // 35.6.
      const long long few = (rows + Few::rows - 1) / Few::rows * t.kv_heads;
      const bool narrow = t.head_dim == 64;
      c.few = few <= (span <= 1024 && narrow ? 512 : span <= 2048 ? 256 : narrow ? 64 : 128);
      c.rows = c.few ? Few::rows : t.head_dim == 64 ? Many64::rows : Many128::rows;
      c.keys = c.few ? Few::keys : t.head_dim == 64 ? Many64::keys : Many128::keys;
      c.blocks = static_cast<int>((rows + c.rows - 1) / c.rows);
      c.splits = 1;
      if (may_split && c.blocks > 0)
      {
        // About the steps a workgroup takes.
        const long long reach = t.seq_k - t.seq_q / 2;
        const long long steps = t.window > 0 && span < reach
                                    ? (t.window + c.keys - 1) / c.keys + 1 +
                                          (t.sinks + c.keys - 1) / c.keys
                                    : (reach + c.keys - 1) / c.keys;
        // A workgroup a CU, down to a step each for few rows, a chain of trips
        // otherwise (one query x 14 heads of 64 over 1,000 keys: two steps each
        // 10.2 us, one 9.8; 16 x 12 of 128 over 500 14.5 and 12.9), unless the
        // chain is as short as the join (over 300: whole 8.0, in parts 9.7),
        // and two or more steps for many. Two workgroups a CU for many rows of
        // head_dim 128, whose four waves leave half of it idle, but no more
        // than four parts to join (1,536 x 12 heads behind 1,024 keys: by one
        // part 44 us, by three 33.5; 768 of them by seven 23.5, by four 22). At
        // head_dim 64 a workgroup has the CU's waves busy by itself (1,024 x
        // 32: one part 19.5 us, two 26), and a second part pays over long spans
        // alone (680 x 32 behind 4,096: one 66 us, two 56; 1,400 x 14 over
        // 4,400 57 and 51).
        const bool two = !c.few && t.head_dim == 128;
        const long long groups = static_cast<long long>(c.blocks) * t.kv_heads;
        const long long fill =
            !c.few && narrow && span > 2048 && groups > 128 && groups <= 256
                ? 2
                : (two ? 512 : 256) / groups;
        c.splits = static_cast<int>(std::max<long long>(
            1, std::min<long long>({fill, c.few ? (steps < 4 ? 1 : steps) : steps / 2, two ? 4 : kMaxSplits})));
      }
      return c;
    }

    void check_window(const WindowAttention &t)
    {
      if (t.seq_q < 0 || t.seq_k < 0 || t.window < 0 || t.sinks < 0)
      {
        throw InvalidArgument("seq_q, seq_k, window and sinks must not be negative, got " +
                              std::to_string(t.seq_q) + ", " + std::to_string(t.seq_k) + ", " +
                              std::to_string(t.window) + ", " + std::to_string(t.sinks));
      }
      if (t.seq_q > t.seq_k)
      {
        throw InvalidArgument("seq_q " + std::to_string(t.seq_q) + " exceeds seq_k " +
                              std::to_string(t.seq_k));
      }
      constexpr int kMostKeys = 0x7fffff00; // a step's last key stays a position
      if (t.seq_k > kMostKeys)
      {
        throw InvalidArgument("seq_k " + std::to_string(t.seq_k) + " exceeds window attention's " +
                              std::to_string(kMostKeys));
      }
      if (t.head_dim != 64 && t.head_dim != 128)
      {
        throw InvalidArgument("window attention takes head_dim 64 or 128, got " +
                              std::to_string(t.head_dim));
      }
      if (t.kv_heads <= 0 || t.heads <= 0 || t.heads % t.kv_heads != 0 || t.kv_heads > 65535)
      {
        throw InvalidArgument("window attention takes a whole number of query heads a KV head, got " +
                              std::to_string(t.heads) + " and " + std::to_string(t.kv_heads));
      }
      // A head's offset in its token is 32 bits.
      if (static_cast<long long>(t.heads) * t.head_dim > 0x7fffffff)
      {
        throw InvalidArgument("window attention takes fewer than 2^31 query elements a token, got " +
                              std::to_string(t.heads) + " heads of " + std::to_string(t.head_dim));
      }
    }

    template <int HD, typename F>
    void launch(const WindowArgs &a, const Cut &c, hipStream_t stream)
    {
      constexpr std::size_t lds = std::max(sizeof(std::uint16_t) * 2 * 2 * F::keys * HD,
                                           sizeof(float) * (F::ways - 1) * F::tiles * (HD / 2 + 2) * 64);
      auto kernel = window_kernel<HD, F::tiles, F::ways, F::keys>;
      if constexpr (lds > 64 * 1024)
      {
        hip_check(hipFuncSetAttribute(reinterpret_cast<const void *>(kernel),
                                      hipFuncAttributeMaxDynamicSharedMemorySize,
                                      static_cast<int>(lds)),
                  "hipFuncSetAttribute window LDS");
      }
      kernel<<<dim3(c.blocks, a.kv_heads, c.splits), 64 * F::tiles * F::ways, lds, stream>>>(a);
      hip_check(hipGetLastError(), "window_kernel");
    }

    template <int HD>
    void launch_any(const WindowArgs &a, const Cut &c, hipStream_t stream)
    {
      if (c.few)
      {
        launch<HD, Few>(a, c, stream);
      }
      else
      {
        launch<HD, std::conditional_t<HD == 64, Many64, Many128>>(a, c, stream);
      }
      if (c.splits > 1)
      {
        const std::size_t rows = static_cast<std::size_t>(a.seq_q) * a.heads;
        if (c.splits > kFewSplits)
        {
          window_join_row_kernel<HD><<<static_cast<unsigned>(rows), 256, 0, stream>>>(a, rows);
          hip_check(hipGetLastError(), "window_join_row_kernel");
          return;
        }
        const std::size_t blocks = (rows * (HD / 4) + 255) / 256;
        window_join_kernel<HD><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(a, rows);
        hip_check(hipGetLastError(), "window_join_kernel");
      }
    }
  } // namespace

  std::size_t window_attention_floats(const WindowAttention &t)
  {
    check_window(t);
    const Cut c = cut_of(t, true);
    return c.splits > 1 ? static_cast<std::size_t>(c.splits) * t.seq_q * t.heads * (t.head_dim + 2)
                        : 0;
  }

  void launch_window_attention(const WindowAttention &t, hipStream_t stream)
  {
    check_window(t);
    if (t.seq_q == 0)
    {
      return;
    }
    if (t.q == nullptr || t.k == nullptr || t.v == nullptr || t.out == nullptr)
    {
      throw InvalidArgument("window attention needs q, k, v and out");
    }
    const long long width = static_cast<long long>(t.kv_heads) * t.head_dim;
    const long long q_width = static_cast<long long>(t.heads) * t.head_dim;
    const long long q_stride = t.q_stride > 0 ? t.q_stride : q_width;
    const long long k_stride = t.k_stride > 0 ? t.k_stride : width;
    const long long v_stride = t.v_stride > 0 ? t.v_stride : width;
    if (t.q_stride < 0 || t.k_stride < 0 || t.v_stride < 0 || q_stride < q_width ||
        k_stride < width || v_stride < width)
    {
      throw InvalidArgument("window attention's strides are of a token's " +
                            std::to_string(q_width) + " query and " + std::to_string(width) +
                            " key and value elements at least (0: those); got " +
                            std::to_string(t.q_stride) + ", " + std::to_string(t.k_stride) +
                            " and " + std::to_string(t.v_stride));
    }
    if ((reinterpret_cast<std::uintptr_t>(t.q) | reinterpret_cast<std::uintptr_t>(t.k) |
         reinterpret_cast<std::uintptr_t>(t.v) | reinterpret_cast<std::uintptr_t>(t.out) |
         reinterpret_cast<std::uintptr_t>(t.partials)) % 16 != 0 ||
        (q_stride | k_stride | v_stride) % 8 != 0)
    {
      throw InvalidArgument("window attention's rows and partials must be 16-byte aligned");
    }
    const Cut c = cut_of(t, t.partials != nullptr);
    if (t.partials != nullptr && t.partials_floats < window_attention_floats(t))
    {
      throw InvalidArgument("window attention's partials need " +
                            std::to_string(window_attention_floats(t)) + " floats; got " +
                            std::to_string(t.partials_floats));
    }
    const auto rows_of = [](const void *at, long long width, int tokens, long long stride) {
      return Extent{at, 2 * static_cast<std::size_t>(width), static_cast<std::size_t>(tokens),
                    2 * static_cast<std::size_t>(stride)};
    };
    const Extent out{t.out, 2 * static_cast<std::size_t>(t.seq_q) * q_width};
    const Extent parts{t.partials, t.partials != nullptr ? sizeof(float) * window_attention_floats(t) : 0};
    for (const Extent &read : {rows_of(t.q, q_width, t.seq_q, q_stride),
                               rows_of(t.k, width, t.seq_k, k_stride),
                               rows_of(t.v, width, t.seq_k, v_stride)})
    {
      if (overlaps(out, read) || overlaps(parts, read))
      {
        throw InvalidArgument("window attention cannot write over its queries, keys or values");
      }
    }
    if (overlaps(parts, out))
    {
      throw InvalidArgument("window attention's partials lie over its output");
    }
    WindowArgs a{};
    a.q = static_cast<const std::uint16_t *>(t.q);
    a.k = static_cast<const std::uint16_t *>(t.k);
    a.v = static_cast<const std::uint16_t *>(t.v);
    a.out = static_cast<std::uint16_t *>(t.out);
    a.q_stride = q_stride;
    a.k_stride = k_stride;
    a.v_stride = v_stride;
    a.seq_q = t.seq_q;
    a.seq_k = t.seq_k;
    a.heads = t.heads;
    a.kv_heads = t.kv_heads;
    a.group = t.heads / t.kv_heads;
    a.window = t.window;
    a.sinks = t.sinks;
    a.splits = c.splits;
    a.scale = static_cast<float>(1.4426950408889634 / std::sqrt(static_cast<double>(t.head_dim)));
    if (c.splits > 1)
    {
      const std::size_t rows = static_cast<std::size_t>(t.seq_q) * t.heads;
      a.part_o = t.partials;
      a.part_ml = t.partials + rows * c.splits * t.head_dim;
    }
    t.head_dim == 64 ? launch_any<64>(a, c, stream) : launch_any<128>(a, c, stream);
  }

} // namespace mi
