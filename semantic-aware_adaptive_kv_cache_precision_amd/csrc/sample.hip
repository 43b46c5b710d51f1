// A token of every row of logits, by temperature, top-k, top-p and min-p, from
// a given uniform number.
//
// Logit l weighs w = exp((l - max) / T). The kept tokens are a prefix of the
// row's order, larger logits first and of equal ones the lower index: the
// shortest of the top_k first, of the fewest first of those whose weights sum to
// top_p of theirs, and of those that weigh min_p of the largest. The token is
// the first by index whose kept weights, up to and with its own, exceed the
// uniform's share of all kept.
//
// Four launches:
//   parts   a workgroup 4,096 logits of a row: their largest, and a histogram of
//           the others below it. Buckets of a sixteenth of a nat, floor(16 l / T),
//           on one grid for the whole row, each with its count and its weights' sum.
//   plan    a workgroup a row: the parts' histograms added up, and from them the
//           bucket that each border (k, p, min-p) falls into, or the few it may.
//   gather  a workgroup a part: the logits of those buckets, which are ranges of
//           logits, into the row's list; its kept weights before them.
//   choose  a workgroup a row: the borders, found in the list by histograms of its
//           logits' places in the order until 64 are left to be put in order; with
//           them each part's kept weights, the part that the token is in, and the
//           token, by its weights in turn.
// (One launch for the last three reads the row again by one CU: 27 us for a row
// of 151,936 with 3,000 logits in a border's bucket.)
//
// Sums: a bucket's weights are added as whole numbers of 2^-38 of the part's
// largest, by LDS atomics of 64 bits (13 of them the count), so that the order
// of adding does not matter: 4,096 weights are off by 2^-27 of the part's largest at
// most, and so the sums of kept ones by 2^-27 of themselves, since a part that
// has kept logits has its largest among them. A border's weights are added as
// finer whole numbers, by what they are themselves (unit_exponent: off by 2^-31 of the
// kept at most, however far below the row's largest they lie); everything else in
// fp64, in one order. A weight below 2^-39 of its part's largest may count as none.
//
// One row of 128,256 takes 26 us, four launches that each are a chain of trips
// and barriers (parts 5, plan 8, gather 5, choose 7); 48 rows of 151,936 45 us
// (parts 14.5, where 29 MB are read and some 43 vector instructions a logit,
// fp64 most, weigh as much as that; plan 9, gather 8, choose 14: borders in buckets of
// thousands, of the rows with high temperatures).
#include "common.hpp"
#include "ragged.hpp"

#include <algorithm>
#include <string>
#include <type_traits>

namespace mi
{
  namespace
  {
    typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
    typedef float f32x4 __attribute__((ext_vector_type(4)));

    constexpr int kPart = 4096;   // logits a part
    constexpr int kThreads = 256; // of a part's workgroup
    constexpr int kBuckets = 512; // 32 nats below the largest
    constexpr int kPerNat = 16;
    constexpr int kRowThreads = 512;  // a bucket each
    constexpr int kBinBits = 9;       // and a bin
    constexpr int kList = 4096;       // of a row's list, held in LDS
    constexpr int kFew = 64;          // of them put in order
    constexpr int kMostVocab = 1 << 20;
    constexpr int kMostParts = kMostVocab / kPart;
    constexpr double kUnit = 0x1p38; // of a weight, in the histograms
    constexpr int kCountShift = 51;  // 4,096 weights of at most 2^38 stay below it
    constexpr unsigned long long kSumMask = (1ull << kCountShift) - 1;

    struct SampleArgs
    {
      const void *logits;
      long long stride;
      bool aligned; // rows begin on 16 bytes
      const float *uniforms;
      const float *temperature;
      const int *top_k;
      const float *top_p;
      const float *min_p;
      int *tokens;
      int vocab;
      int parts;
      unsigned long long *sums; // [row][part][bucket] count << 51 | weights
      double *sure;             // [row][part] weights kept before the plan's first bucket
      struct RowPlan *plans;    // [row]
      unsigned long long *lists; // [row][vocab] ranks of the logits gathered
      float *tops;              // [row][part] largest logit
      int *top_at;              // and its index, or vocab
    };

    // A whole number below 2^52.
    __device__ inline double number_of(unsigned long long v)
    {
      return __builtin_bit_cast(double, v | __builtin_bit_cast(unsigned long long, 0x1p52)) - 0x1p52;
    }

    // The nearest whole number to one below 2^52.
    __device__ inline unsigned long long units_of(double units)
    {
      return __builtin_bit_cast(unsigned long long, units + 0x1p52) -
             __builtin_bit_cast(unsigned long long, 0x1p52);
    }
    template <bool kHalf>
    __device__ inline float logit_at(const void *row, int i)
    {
      if constexpr (kHalf)
      {
        return h2f(static_cast<const std::uint16_t *>(row)[i]);
      }
      else
      {
        return static_cast<const float *>(row)[i];
      }
    }

    // Logits a load of 16 bytes takes.
    template <bool kHalf>
    constexpr int kWide = kHalf ? 8 : 4;

    // kWide logits from i on (a multiple of kWide), as they lie; -inf past the last.
    template <bool kHalf>
    __device__ inline u32x4 logits_at(const void *row, int i, int vocab, bool aligned)
    {
      if (aligned && i + kWide<kHalf> <= vocab)
      {
        return *reinterpret_cast<const u32x4 *>(static_cast<const std::uint8_t *>(row) +
                                                static_cast<std::size_t>(i) * (16 / kWide<kHalf>));
      }
      unsigned v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
      {
        if constexpr (kHalf)
        {
          const auto *at = static_cast<const std::uint16_t *>(row) + i + 2 * e;
          const unsigned lo = i + 2 * e < vocab ? at[0] : 0xFC00u;
          const unsigned hi = i + 2 * e + 1 < vocab ? at[1] : 0xFC00u;
          v[e] = lo | hi << 16;
        }
        else
        {
          v[e] = i + e < vocab ? static_cast<const unsigned *>(row)[i + e] : 0xFF800000u;
        }
      }
      return u32x4{v[0], v[1], v[2], v[3]};
    }
    template <bool kHalf>
    __device__ inline float logit_in(u32x4 v, int e)
    {
      if constexpr (kHalf)
      {
        return h2f(static_cast<std::uint16_t>(v[e / 2] >> (16 * (e % 2))));
      }
      else
      {
        const unsigned bits = v[e]; // (a vector's element is no object to cast the bits of)
        return __builtin_bit_cast(float, bits);
      }
    }

    template <bool kHalf>
    __device__ inline const void *row_of(const SampleArgs &a, int row)
    {
      const std::size_t at = static_cast<std::size_t>(row) * a.stride;
      return kHalf ? static_cast<const void *>(static_cast<const std::uint16_t *>(a.logits) + at)
                   : static_cast<const void *>(static_cast<const float *>(a.logits) + at);
    }

    // 1 / T, or less than 0 where the row takes its largest logit.
    __device__ inline double inverse_temperature(const SampleArgs &a, int row)
    {
      const float t = a.temperature != nullptr ? a.temperature[row] : 1.0f;
      return t > 0.0f ? 1.0 / static_cast<double>(t) : -1.0;
    }

    // A logit that weighs anything.
    __device__ inline bool counts(float l) { return l > -INFINITY; }

    // The bucket on the row's grid, floor(l steps) in fp32, with `steps` kPerNat
    // / T: it never falls as l rises, which is all that is asked of it.
    constexpr int kFar = 1 << 29;
    __device__ inline int bucket_of(float l, float steps)
    {
      return l == INFINITY ? 1 << 30
                           : static_cast<int>(__builtin_amdgcn_fmed3f(floorf(l * steps), -1.0f * kFar, 1.0f * kFar));
    }
    __device__ inline float steps_of(double inv_t)
    {
      return static_cast<float>(fmin(kPerNat * inv_t, 3e38));
    }

    // exp(x) for x <= 0 as 2^n exp(y), |y| <= ln 2 / 2, by the first N + 1 terms
    // of exp's series: of 14, what is left out is 2^-57 of it.
    template <int N>
    __device__ inline double exp_series(double y)
    {
      // 1 / N! .. 1 / 0!
      constexpr double kInverse[] = {1.0, 1.0, 1.0 / 2, 1.0 / 6, 1.0 / 24, 1.0 / 120, 1.0 / 720,
                                     1.0 / 5040, 1.0 / 40320, 1.0 / 362880, 1.0 / 3628800,
                                     1.0 / 39916800, 1.0 / 479001600, 1.0 / 6227020800.0};
      double p = kInverse[N];
#pragma unroll
      for (int i = N - 1; i >= 0; --i)
      {
        p = __builtin_fma(p, y, kInverse[i]);
      }
      return p;
    }
    constexpr double kLog2e = 1.4426950408889634;
    constexpr double kLn2High = 0x1.62e42fefa38p-1, kLn2Low = 0x1.ef35793c7673p-45; // their sum ln 2
    __device__ inline double exp_below(double x)
    {
      x = fmax(x, -1400.0); // (2^-1400 and less are 0)
      const double n = rint(x * kLog2e);
      const double y = __builtin_fma(n, -kLn2Low, __builtin_fma(n, -kLn2High, x));
      return ldexp(exp_series<13>(y), static_cast<int>(n));
    }

    __device__ inline double weight_of(float l, float top, double inv_t)
    {
      return l == top          ? 1.0
             : top == INFINITY ? 0.0
                               : exp_below((static_cast<double>(l) - static_cast<double>(top)) * inv_t);
    }

    // The power of two that a logit's weight does not pass, 2^-128 at least (units of
    // less would leave fp64, where a temperature next to 0 makes weights of nothing).
    __device__ inline int power_above(float l, float top, double inv_t)
    {
      return l >= top ? 0
                      : static_cast<int>(ceil(
                            fmax((static_cast<double>(l) - static_cast<double>(top)) * inv_t * kLog2e, -128.0)));
    }
    // The units of 2^-e that n weights of at most 2^high each, some `mass` in all,
    // are counted in: a weight is 2^51 of them at most, and all of them 2^62, by
    // their mass, which may be too small by a factor of two, or by their number.
    // What n halves of a unit make up is 2^-31 of a weight next to 2^high or 2^-42 of
    // the mass at most. (From exponents alone: every pass of a border's search forms it.)
    __device__ inline int unit_exponent(int n, double mass, int high)
    {
      const int many = max(0, min(32 - __clz(n), __builtin_amdgcn_frexp_exp(mass) - high));
      return min(51, 62 - many) - high;
    }

    // A logit's entry of a histogram: one, and exp(x) as a whole number of kUnit.
    // A double below 2^51 added to 1.5 x 2^52 is rounded to a whole one, its low
    // bits: so n of exp(x) = 2^n 2^f, |f| <= 1/2, with which the exponent moves,
    // and the number itself. 2^f by the polynomial of degree 8 with the least
    // relative error, 2^-40.2, found by exchange of its extrema.
    struct Entries
    {
      double c[9] = {0x1.ffffffffff7a3p-1,  0x1.62e42fef8615ep-1,  0x1.ebfbdff9319e1p-3,
                     0x1.c6b08dd46d38fp-5,  0x1.3b2ab5c529251p-7,  0x1.5d87483855cbcp-10,
                     0x1.430acca348ed9p-13, 0x1.00dad250347c9p-16, 0x1.61afceb9107ebp-20};
      double log2e = kLog2e, least = -64.0, whole = 0x1.8p52 + 38 /* of kUnit */, one = 0x1p52;

      // (In scalar registers: else every product takes its constant from two
      // moves to vector ones.)
      __device__ Entries()
      {
#pragma unroll
        for (double &v : c)
        {
          asm volatile("" : "+s"(v));
        }
        asm volatile("" : "+s"(log2e), "+s"(least), "+s"(whole), "+s"(one));
      }
      __device__ unsigned long long of(double x) const
      {
        const double t = fmax(x * log2e, least);
        const double m = t + whole;
        const double f = t - (m - whole);
        double p = __builtin_fma(c[8], f, c[7]);
#pragma unroll
        for (int i = 6; i >= 0; --i)
        {
          p = __builtin_fma(p, f, c[i]);
        }
        const auto n = static_cast<unsigned>(__builtin_bit_cast(unsigned long long, m)); // n + 38
        const double w = __builtin_bit_cast(double, __builtin_bit_cast(unsigned long long, p) +
                                                        (static_cast<unsigned long long>(n) << 52)) +
                         one;
        return __builtin_bit_cast(unsigned long long, w) -
               (__builtin_bit_cast(unsigned long long, 0x1p52) - (1ull << kCountShift));
      }
    };

    // ---- a part's histogram ---------------------------------------------------

    template <bool kHalf>
    __global__ void __launch_bounds__(kThreads) sample_parts_kernel(SampleArgs a)
    {
      __shared__ unsigned long long s_sums[kBuckets];
      __shared__ float s_top[kThreads / 64];
      __shared__ int s_at[kThreads / 64];
      const int part = blockIdx.x, row = blockIdx.y;
      const void *logits = row_of<kHalf>(a, row);
      const int first = part * kPart;
      constexpr int W = kWide<kHalf>, kLoads = kPart / kThreads / W;
      float l[kLoads][W];
      {
        u32x4 raw[kLoads];
#pragma unroll
        for (int c = 0; c < kLoads; ++c)
        {
          raw[c] = logits_at<kHalf>(logits, first + W * (c * kThreads + static_cast<int>(threadIdx.x)),
                                    a.vocab, a.aligned);
        }
#pragma unroll
        for (int c = 0; c < kLoads; ++c)
        {
#pragma unroll
          for (int e = 0; e < W; ++e)
          {
            l[c][e] = logit_in<kHalf>(raw[c], e);
          }
        }
      }
      const double inv_t = inverse_temperature(a, row);
#pragma unroll
      for (int b = 0; b < kBuckets; b += kThreads)
      {
        s_sums[b + threadIdx.x] = 0;
      }
      // The largest, and the lowest index that has it.
      float top = -INFINITY;
      int at = a.vocab;
#pragma unroll
      for (int c = 0; c < kLoads; ++c)
      {
#pragma unroll
        for (int e = 0; e < W; ++e)
        {
          if (l[c][e] > top)
          {
            top = l[c][e];
            at = first + W * (c * kThreads + static_cast<int>(threadIdx.x)) + e;
          }
        }
      }
#pragma unroll
      for (int offset = 1; offset < 64; offset *= 2)
      {
        const float t = __shfl_xor(top, offset);
        const int i = __shfl_xor(at, offset);
        if (t > top || (t == top && i < at))
        {
          top = t;
          at = i;
        }
      }
      if (threadIdx.x % 64 == 0)
      {
        s_top[threadIdx.x / 64] = top;
        s_at[threadIdx.x / 64] = at;
      }
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kThreads / 64; ++w)
      {
        if (s_top[w] > top || (s_top[w] == top && s_at[w] < at))
        {
          top = s_top[w];
          at = s_at[w];
        }
      }
      const std::size_t slot = static_cast<std::size_t>(row) * a.parts + part;
      if (threadIdx.x == 0)
      {
        a.tops[slot] = top;
        a.top_at[slot] = at;
      }
      if (inv_t < 0.0)
      {
        return; // the largest is the token
      }
      if (counts(top))
      {
        const float steps = steps_of(inv_t);
        const int highest = bucket_of(top, steps);
        // (Only the equals of an infinite largest are in its buckets: as the
        // largest finite they weigh one.)
        constexpr float kLargest = 0x1.fffffep127f;
        const double high = static_cast<double>(fminf(top, kLargest));
        const Entries entries;
#pragma unroll
        for (int c = 0; c < kLoads; ++c)
        {
#pragma unroll
          for (int e0 = 0; e0 < W; e0 += 4)
          {
            // (Four at a time, each for all lanes: their steps side by side.)
            unsigned long long entry[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
            {
              entry[e] = entries.of((static_cast<double>(fminf(l[c][e0 + e], kLargest)) - high) * inv_t);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
            {
              asm volatile("" : "+v"(entry[e]));
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
            {
              const int below = highest - bucket_of(l[c][e0 + e], steps);
              if (counts(l[c][e0 + e]) && below < kBuckets)
              {
                atomicAdd(&s_sums[below], entry[e]);
              }
            }
          }
        }
      }
      __syncthreads();
#pragma unroll
      for (int b = 0; b < kBuckets; b += kThreads)
      {
        a.sums[slot * kBuckets + b + threadIdx.x] = s_sums[b + threadIdx.x];
      }
    }

    // ---- the row ------------------------------------------------------------------

    // A logit's place in the row's order as a number: larger is earlier.
    __device__ inline unsigned long long rank_of(float l, int index)
    {
      unsigned bits = __builtin_bit_cast(unsigned, l + 0.0f); // -0 is 0
      bits = bits & 0x80000000u ? ~bits : bits | 0x80000000u;
      return (static_cast<unsigned long long>(bits) << 32) | static_cast<unsigned>(~index);
    }
    __device__ inline float logit_of(unsigned long long rank)
    {
      const unsigned bits = static_cast<unsigned>(rank >> 32);
      return __builtin_bit_cast(float, bits & 0x80000000u ? bits & 0x7FFFFFFFu : ~bits);
    }
    __device__ inline int index_of(unsigned long long rank)
    {
      return static_cast<int>(~static_cast<unsigned>(rank));
    }

    // v of the lane that a DPP pattern names, 0 where it names none.
    template <int kPattern, int kRows>
    __device__ inline int moved(int v)
    {
      return __builtin_amdgcn_update_dpp(0, v, kPattern, kRows, 0xF, false);
    }
    template <int kPattern, int kRows>
    __device__ inline double moved(double v)
    {
      const auto bits = __builtin_bit_cast(unsigned long long, v);
      const unsigned lo = moved<kPattern, kRows>(static_cast<int>(bits));
      const unsigned hi = moved<kPattern, kRows>(static_cast<int>(bits >> 32));
      return __builtin_bit_cast(double, static_cast<unsigned long long>(hi) << 32 | lo);
    }
    // Inclusive sums over a wave: within rows of 16 lanes, then the rows before.
    template <typename T>
    __device__ inline T wave_scan(T v)
    {
      v += moved<0x111, 0xF>(v); // row_shr:1, 2, 4, 8
      v += moved<0x112, 0xF>(v);
      v += moved<0x114, 0xF>(v);
      v += moved<0x118, 0xF>(v);
      v += moved<0x142, 0xA>(v); // row_bcast:15 to rows 1 and 3
      v += moved<0x143, 0xC>(v); // row_bcast:31 to rows 2 and 3
      return v;
    }
    // Inclusive sums over the workgroup's threads, in thread order. (The caller
    // has a barrier between two scans by the same s_waves.)
    template <typename T>
    __device__ inline T waves_before(const T *s_waves)
    {
      const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
      return __shfl(wave_scan(lane < wave ? s_waves[lane] : T(0)), 63);
    }
    template <typename T>
    __device__ inline T scan(T v, T *s_waves)
    {
      v = wave_scan(v);
      if ((threadIdx.x & 63) == 63)
      {
        s_waves[threadIdx.x >> 6] = v;
      }
      __syncthreads();
      return v + waves_before(s_waves);
    }
    __device__ inline void scan(int &count, double &sum, int *s_counts, double *s_sums)
    {
      count = wave_scan(count);
      sum = wave_scan(sum);
      if ((threadIdx.x & 63) == 63)
      {
        s_counts[threadIdx.x >> 6] = count;
        s_sums[threadIdx.x >> 6] = sum;
      }
      __syncthreads();
      count += waves_before(s_counts);
      sum += waves_before(s_sums);
    }

    // The first thread of the row's workgroup that a condition holds for, `none`
    // if none. (An LDS atomic of every thread takes 2 us: they share its address.
    // Between two calls by the same s_waves the caller has a barrier.)
    __device__ inline int first_of(bool holds, int none, int *s_waves)
    {
      const unsigned long long all = __ballot(holds);
      if ((threadIdx.x & 63) == 0)
      {
        s_waves[threadIdx.x >> 6] =
            all != 0 ? static_cast<int>(threadIdx.x) + __ffsll(all) - 1 : none;
      }
      __syncthreads();
      int first = none;
#pragma unroll
      for (int w = kRowThreads / 64 - 1; w >= 0; --w)
      {
        first = s_waves[w] != none ? s_waves[w] : first;
      }
      return first;
    }

    // The last one, -1 if none.
    __device__ inline int last_of(bool holds, int *s_waves)
    {
      const unsigned long long all = __ballot(holds);
      if ((threadIdx.x & 63) == 0)
      {
        s_waves[threadIdx.x >> 6] = all != 0 ? static_cast<int>(threadIdx.x) + 63 - __clzll(all) : -1;
      }
      __syncthreads();
      int last = -1;
#pragma unroll
      for (int w = 0; w < kRowThreads / 64; ++w)
      {
        last = max(last, s_waves[w]);
      }
      return last;
    }

    // What the plan finds of a row.
    struct RowPlan
    {
      double inv_t;
      float steps;
      float top;   // the largest logit,
      int highest; // and its bucket on the grid
      int kind;
      int k_bucket; // top_k's border's, kBuckets: none
      int p_first;  // those that top_p's may be in, p_first > p_last: none
      int p_last;
      int first; // before it every bucket is kept: kBuckets where no border is
      unsigned long long min_rank; // what min_p keeps ranks so at least
      int min_bucket;
      int listed; // logits gathered: those in these ranges
      unsigned from[3]; // of top_k's bucket, top_p's, min_p's, as the upper half of
      unsigned to[3];   // a rank; none where from > to
      int count[kBuckets]; // of the row, up to and with each bucket
      double weight[kBuckets];
      double scale[kMostParts]; // of a part's weights in the row's
      short shift[kMostParts];  // a part's bucket 0 among the row's; kBuckets: none of it
    };
    enum : int
    {
      kChosen, // there is nothing to choose
      kOpen,
    };

    // The least logit, as the upper half of a rank, from which on a condition
    // holds: by 64 pivots at a time.
    template <typename F>
    __device__ inline unsigned first_key(F &&holds)
    {
      const unsigned lane = threadIdx.x & 63;
      unsigned lo = 0x00800000u, hi = 0xFF800001u; // the least finite; past infinity
      while (lo < hi)
      {
        const unsigned step = (hi - lo) / 64 + 1;
        const unsigned long long at = lo + static_cast<unsigned long long>(lane) * step;
        const bool reached = at >= hi || holds(logit_of(at << 32));
        const int before = __popcll(~__ballot(reached));
        const unsigned long long next = lo + static_cast<unsigned long long>(before) * step;
        lo = before > 0 ? static_cast<unsigned>(next - step + 1) : lo;
        hi = static_cast<unsigned>(min(next, static_cast<unsigned long long>(hi)));
      }
      return __builtin_amdgcn_readfirstlane(lo);
    }
    // The same near a logit that it should hold from: 64 of them at once.
    template <typename F>
    __device__ inline unsigned first_key(float near, F &&holds)
    {
      if (near > -3e38f && near < 3e38f)
      {
        const unsigned from = static_cast<unsigned>(rank_of(near, 0) >> 32) - 32;
        const unsigned long long reached =
            __ballot(holds(logit_of(static_cast<unsigned long long>(from + (threadIdx.x & 63)) << 32)));
        if ((reached & 1) == 0 && reached != 0)
        {
          return from + __ffsll(reached) - 1;
        }
      }
      return first_key(holds);
    }
    // The least and the largest logit of a bucket of the row.
    __device__ inline unsigned least_key(const RowPlan &p, int b)
    {
      const int bucket = p.highest - b;
      const float steps = p.steps;
      return first_key(static_cast<float>(bucket) / steps,
                       [&](float l) { return bucket_of(l, steps) >= bucket; });
    }
    __device__ inline unsigned most_key(const RowPlan &p, int b)
    {
      return b == 0 ? static_cast<unsigned>(rank_of(p.top, 0) >> 32) : least_key(p, b - 1) - 1;
    }

    __global__ void __launch_bounds__(kRowThreads) sample_plan_kernel(SampleArgs a)
    {
      static_assert(kRowThreads == kBuckets, "a bucket a thread");
      __shared__ double s_scale[kMostParts], s_waves[kRowThreads / 64], s_weight[kBuckets];
      __shared__ int s_shift[kMostParts], s_int_waves[kRowThreads / 64];
      __shared__ int s_firsts[3][kRowThreads / 64];
      __shared__ unsigned s_keys[7];
      const int row = blockIdx.x;
      const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
      RowPlan &plan = a.plans[row];
      const double inv_t = inverse_temperature(a, row);
      const int k = a.top_k != nullptr ? a.top_k[row] : 0;
      const float p = a.top_p != nullptr ? a.top_p[row] : 1.0f;
      const float m = a.min_p != nullptr ? a.min_p[row] : 0.0f;
      const float *tops = a.tops + static_cast<std::size_t>(row) * a.parts;
      const int *top_at = a.top_at + static_cast<std::size_t>(row) * a.parts;
      // The row's largest logit.
      float top = -INFINITY;
      int at = a.vocab;
      for (int q = threadIdx.x & 63; q < a.parts; q += 64)
      {
        const float t = tops[q];
        const int i = top_at[q];
        if (t > top || (t == top && i < at))
        {
          top = t;
          at = i;
        }
      }
#pragma unroll
      for (int offset = 1; offset < 64; offset *= 2)
      {
        const float t = __shfl_xor(top, offset);
        const int i = __shfl_xor(at, offset);
        if (t > top || (t == top && i < at))
        {
          top = t;
          at = i;
        }
      }
      if (inv_t < 0.0 || !counts(top))
      {
        if (threadIdx.x == 0)
        {
          a.tokens[row] = at;
          plan.kind = kChosen;
        }
        return;
      }
      RowPlan now;
      now.inv_t = inv_t;
      now.steps = steps_of(inv_t);
      now.top = top;
      now.highest = bucket_of(top, now.steps);
      for (int q = threadIdx.x; q < a.parts; q += kRowThreads)
      {
        const float t = tops[q];
        const int shift = counts(t) ? min(now.highest - bucket_of(t, now.steps), kBuckets) : kBuckets;
        const double scale = counts(t) ? weight_of(t, top, inv_t) / kUnit : 0.0;
        s_shift[q] = shift;
        s_scale[q] = scale;
        plan.shift[q] = static_cast<short>(shift);
        plan.scale[q] = scale;
      }
      if (m > 0.0f && wave == kRowThreads / 64 - 1)
      {
        // The least logit that weighs enough for min_p, wherever it lies.
        const double least = static_cast<double>(fminf(m, 1.0f));
        const float near = static_cast<float>(static_cast<double>(top) + log(least) / inv_t);
        s_keys[6] = first_key(
            near, [&](float l) { return l >= top || weight_of(l, top, inv_t) >= least; });
      }
      __syncthreads();
      // Forty parts' counts asked for together.
      const unsigned long long *sums = a.sums + static_cast<std::size_t>(row) * a.parts * kBuckets;
      const int bucket = threadIdx.x;
      int count = 0;
      double weight = 0.0;
      for (int q0 = 0; q0 < a.parts; q0 += 40)
      {
        unsigned long long v[40];
#pragma unroll
        for (int i = 0; i < 40; ++i)
        {
          const int of = q0 + i < a.parts ? bucket - s_shift[q0 + i] : -1;
          v[i] = of >= 0 ? sums[static_cast<std::size_t>(q0 + i) * kBuckets + of] : 0;
        }
#pragma unroll
        for (int i = 0; i < 40; ++i)
        {
          count += static_cast<int>(v[i] >> kCountShift);
          weight += number_of(v[i] & kSumMask) * s_scale[min(q0 + i, a.parts - 1)];
        }
      }
      scan(count, weight, s_int_waves, s_waves);
      s_weight[bucket] = weight;

      // The buckets to gather.
      const int kb = k > 0 ? first_of(count >= k, kBuckets, s_firsts[0]) : kBuckets;
      now.k_bucket = kb;
      now.p_first = kBuckets;
      now.p_last = -1;
      if (p < 1.0f)
      {
        // top_p's share of what top_k keeps: all before its bucket, and some of
        // that (by sums that may differ in their last places).
        __syncthreads(); // s_weight
        const double least = kb == 0 ? 0.0 : s_weight[(kb < kBuckets ? kb : kBuckets) - 1];
        const double most = s_weight[min(kb, kBuckets - 1)];
        const double share = static_cast<double>(fmaxf(p, 0.0f));
        const int bound = min(kb, kBuckets - 1);
        now.p_first = min(bound, first_of(weight >= share * least * (1 - 1e-9), kBuckets, s_firsts[1]));
        now.p_last = min(bound, first_of(weight >= share * most * (1 + 1e-9), kBuckets, s_firsts[2]));
      }
      now.min_rank = 0;
      now.min_bucket = kBuckets;
      if (m > 0.0f)
      {
        now.min_rank = static_cast<unsigned long long>(s_keys[6]) << 32;
        now.min_bucket = min(now.highest - bucket_of(logit_of(now.min_rank), now.steps), kBuckets);
      }
      now.first = min(min(kb, now.p_first), now.min_bucket);
      // Their ranges, an end a wave (min_p's only where it may be the border).
      const int reach = now.p_first < kBuckets ? now.p_last : kb;
      const int from = wave % 3 == 0 ? kb : wave % 3 == 1 ? now.p_first : now.min_bucket;
      const int to = wave % 3 == 1 ? now.p_last : from;
      if (wave < 6)
      {
        const bool wanted = from < kBuckets && (wave % 3 < 2 || from <= reach);
        s_keys[wave] = wave < 3 ? (wanted ? least_key(now, to) : 1u) : (wanted ? most_key(now, from) : 0u);
      }
      plan.count[bucket] = count;
      plan.weight[bucket] = weight;
      __syncthreads();
      if (threadIdx.x == 0)
      {
        plan.inv_t = now.inv_t;
        plan.steps = now.steps;
        plan.top = now.top;
        plan.highest = now.highest;
        plan.k_bucket = now.k_bucket;
        plan.p_first = now.p_first;
        plan.p_last = now.p_last;
        plan.first = now.first;
        plan.min_rank = now.min_rank;
        plan.min_bucket = now.min_bucket;
        plan.listed = 0;
#pragma unroll
        for (int i = 0; i < 3; ++i)
        {
          plan.from[i] = s_keys[i];
          plan.to[i] = s_keys[3 + i];
        }
        plan.kind = kOpen;
      }
    }

    template <bool kHalf>
    __global__ void __launch_bounds__(kThreads) sample_gather_kernel(SampleArgs a)
    {
      __shared__ double s_kept[kThreads / 64];
      const int part = blockIdx.x, row = blockIdx.y;
      RowPlan &plan = a.plans[row];
      const std::size_t slot = static_cast<std::size_t>(row) * a.parts + part;
      const int kind = plan.kind, shift = plan.shift[part];
      const double scale = plan.scale[part];
      const float part_top = a.tops[slot];
      if (kind == kChosen)
      {
        return;
      }
      // The part's weights before the plan's first bucket.
      const int before = min(plan.first - shift, kBuckets);
      unsigned long long kept = 0;
#pragma unroll
      for (int b = 0; b < kBuckets; b += kThreads)
      {
        const int of = b + static_cast<int>(threadIdx.x);
        kept += of < before ? a.sums[slot * kBuckets + of] & kSumMask : 0;
      }
      float from[3], to[3];
      bool wanted = false;
#pragma unroll
      for (int i = 0; i < 3; ++i)
      {
        const bool any = plan.from[i] <= plan.to[i];
        from[i] = any ? logit_of(static_cast<unsigned long long>(plan.from[i]) << 32) : INFINITY;
        to[i] = any ? logit_of(static_cast<unsigned long long>(plan.to[i]) << 32) : -INFINITY;
        wanted = wanted || part_top >= from[i];
      }
      const double own = wave_scan(number_of(kept)); // (512 of at most 2^51 / 2^13)
      if (threadIdx.x % 64 == 63)
      {
        s_kept[threadIdx.x / 64] = own;
      }
      __syncthreads();
      if (threadIdx.x == 0)
      {
        a.sure[slot] = (s_kept[0] + s_kept[1] + s_kept[2] + s_kept[3]) * scale;
      }
      if (!wanted)
      {
        return;
      }
      const void *logits = row_of<kHalf>(a, row);
      constexpr int W = kWide<kHalf>, kLoads = kPart / kThreads / W;
      const int i0 = part * kPart + W * static_cast<int>(threadIdx.x);
      u32x4 raw[kLoads];
#pragma unroll
      for (int c = 0; c < kLoads; ++c)
      {
        raw[c] = logits_at<kHalf>(logits, i0 + W * kThreads * c, a.vocab, a.aligned);
      }
      unsigned found = 0;
#pragma unroll
      for (int i = 0; i < 16; ++i)
      {
        const float l = logit_in<kHalf>(raw[i / W], i % W);
        bool in = false;
#pragma unroll
        for (int j = 0; j < 3; ++j)
        {
          in = in || (l >= from[j] && l <= to[j]);
        }
        // (Buckets past the part's histogram are no part of any sum.)
        in = in && plan.highest - bucket_of(l, plan.steps) - shift < kBuckets;
        found |= (in ? 1u : 0u) << i;
      }
      if (__ballot(found != 0) == 0)
      {
        return;
      }
      // A wave's places in the list from one count.
      const int mine = __popc(found);
      const int upto = wave_scan(mine);
      int at = 0;
      if (threadIdx.x % 64 == 0)
      {
        at = atomicAdd(&plan.listed, __builtin_amdgcn_readlane(upto, 63));
      }
      at = __builtin_amdgcn_readfirstlane(at) + upto - mine;
      unsigned long long *list = a.lists + static_cast<std::size_t>(row) * a.vocab;
#pragma unroll
      for (int i = 0; i < 16; ++i)
      {
        if ((found >> i & 1) != 0)
        {
          list[at++] = rank_of(logit_in<kHalf>(raw[i / W], i % W), i0 + W * kThreads * (i / W) + i % W);
        }
      }
    }

    // The ranks of a bucket.
    struct Ranks
    {
      unsigned long long lo;
      unsigned long long hi;
    };
    __device__ inline Ranks ranks_of(unsigned from, unsigned to)
    {
      return {static_cast<unsigned long long>(from) << 32,
              static_cast<unsigned long long>(to) << 32 | 0xFFFFFFFFull};
    }
    // A border: everything in buckets before `bucket` is kept, and in it what
    // ranks at least `rank`.
    struct Border
    {
      int bucket;
      unsigned long long rank;
      Ranks in;
    };

    struct RowState
    {
      unsigned long long list[kList];
      unsigned long long bins[kRowThreads]; // histograms of ranks
      int bin_counts[kRowThreads];
      unsigned long long few[kFew];
      unsigned long long border[kMostParts]; // each part's kept weights of the border's bucket
      double waves[kRowThreads / 64];
      int int_waves[kRowThreads / 64];
      int firsts[kRowThreads / 64];
      int lasts[kRowThreads / 64];
      int ints[4];
      unsigned long long rank;
      double value;
      double mass;
    };

    struct RowSampler
    {
      RowState &s;
      const RowPlan &plan;
      const unsigned long long *list; // in LDS where it fits
      int listed;

      template <typename F>
      __device__ void each(F &&f) const
      {
        for (int i = threadIdx.x; i < listed; i += kRowThreads)
        {
          f(list[i]);
        }
      }

      // Of the listed ranks in [lo, hi], those above the border are counted as
      // taken, and [lo, hi] becomes the 512th of it (or the 256th) that has the border. n are in
      // it, of some `mass`, before and after.
      __device__ void narrow(long long most, double need, unsigned long long &lo,
                             unsigned long long &hi, long long &taken, double &weight, int &n,
                             double &mass) const
      {
        const int units = unit_exponent(n, mass, power_above(logit_of(hi), plan.top, plan.inv_t));
        const double scale = ldexp(1.0, units), unit = ldexp(1.0, -units);
        // (A power of two: a division of 64 bits a rank is most of a pass.)
        const int shift = max(0, 64 - __clzll(hi - lo) - kBinBits);
        const unsigned long long step = 1ull << shift;
        __syncthreads();
        s.bins[threadIdx.x] = 0;
        s.bin_counts[threadIdx.x] = 0;
        __syncthreads();
        each([&](unsigned long long rank) {
          if (rank >= lo && rank <= hi)
          {
            const int bin = static_cast<int>((hi - rank) >> shift);
            atomicAdd(&s.bin_counts[bin], 1);
            atomicAdd(&s.bins[bin], units_of(weight_of(logit_of(rank), plan.top, plan.inv_t) * scale));
          }
        });
        __syncthreads();
        const int bin = threadIdx.x;
        const int mine = s.bin_counts[bin];
        const double own = static_cast<double>(s.bins[bin]) * unit;
        int count = mine;
        double sum = own;
        scan(count, sum, s.int_waves, s.waves);
        // The first bin that cannot be kept whole has the border.
        const int at = min(first_of(taken + count >= most || (taken + count > 0 && weight + sum >= need),
                                    kRowThreads, s.firsts),
                           kRowThreads - 1);
        if (bin == at)
        {
          s.ints[0] = count - mine;
          s.ints[2] = mine;
          s.value = sum - own;
          s.mass = own + mine * unit; // (a weight's rounding is half a unit)
        }
        __syncthreads();
        taken += s.ints[0];
        weight += s.value;
        n = s.ints[2];
        mass = s.mass;
        const unsigned long long above = hi - step * at;
        lo = above - lo < step ? lo : above - (step - 1);
        hi = above;
      }

      // The border among the logits of bucket b, of which the first are kept: as
      // long as they are fewer than `most` and the weights before them less than
      // `need`; one at least if `need` is not more than nothing. Returns the rank
      // of the last kept (where none is, the one above the first), and to *sum
      // the weights of the kept.
      __device__ unsigned long long cut(int b, Ranks in, long long most, double need, double *sum) const
      {
        unsigned long long lo = in.lo, hi = in.hi;
        long long taken = 0;
        double weight = 0.0;
        int n = plan.count[b] - (b > 0 ? plan.count[b - 1] : 0);
        // (The plan's sums: each weight is off by 2^-39 of the row's largest at most.)
        double mass = plan.weight[b] - (b > 0 ? plan.weight[b - 1] : 0.0) + n * 0x1p-38;
        while (n > kFew)
        {
          narrow(most, need, lo, hi, taken, weight, n, mass);
        }
        // The few in order, by each one's place among them.
        __syncthreads();
        if (threadIdx.x == 0)
        {
          s.ints[0] = 0;
          s.ints[1] = 0;
          s.value = weight;
          s.rank = hi == ~0ull ? hi : hi + 1; // none of them: what ranks above
        }
        __syncthreads();
        each([&](unsigned long long rank) {
          if (rank >= lo && rank <= hi)
          {
            s.bins[min(atomicAdd(&s.ints[0], 1), kFew - 1)] = rank;
          }
        });
        __syncthreads();
        if (threadIdx.x < 64)
        {
          const int lane = threadIdx.x;
          const unsigned long long own = lane < n ? s.bins[lane] : 0;
          int place = 0;
          for (int i = 0; i < n; ++i)
          {
            place += s.bins[i] > own ? 1 : 0;
          }
          if (lane < n)
          {
            s.few[min(place, kFew - 1)] = own;
          }
        }
        __syncthreads();
        if (threadIdx.x < 64)
        {
          const int i = threadIdx.x;
          const double w = i < n ? weight_of(logit_of(s.few[i]), plan.top, plan.inv_t) : 0.0;
          const double upto = weight + wave_scan(w);
          const bool kept = i < n && taken + i < most && (upto - w < need || taken + i == 0);
          const unsigned long long all = __ballot(kept); // a run from the first on
          if (kept && i == __popcll(all) - 1)
          {
            s.value = upto;
            s.rank = s.few[i];
          }
        }
        __syncthreads();
        *sum = s.value;
        return s.rank;
      }
    };

    template <bool kHalf>
    __global__ void __launch_bounds__(kRowThreads) sample_choose_kernel(SampleArgs a)
    {
      __shared__ RowState s;
      __shared__ RowPlan plan;
      const int row = blockIdx.x;
      const unsigned long long *list = a.lists + static_cast<std::size_t>(row) * a.vocab;
      const int k = a.top_k != nullptr ? a.top_k[row] : 0;
      const float p = a.top_p != nullptr ? a.top_p[row] : 1.0f;
      const float uniform = a.uniforms[row];
      // The plan, and the list as far as most go, asked for together.
      {
        constexpr int kWords = sizeof(RowPlan) / 8;
        static_assert(sizeof(RowPlan) % 8 == 0, "in words");
        const auto *from = reinterpret_cast<const unsigned long long *>(a.plans + row);
        auto *to = reinterpret_cast<unsigned long long *>(&plan);
        unsigned long long ranks[2];
#pragma unroll
        for (int i = 0; i < 2; ++i)
        {
          const int at = i * kRowThreads + static_cast<int>(threadIdx.x);
          ranks[i] = at < a.vocab ? list[at] : 0;
        }
#pragma unroll
        for (int i = 0; i < (kWords + kRowThreads - 1) / kRowThreads; ++i)
        {
          const int at = i * kRowThreads + static_cast<int>(threadIdx.x);
          if (at < kWords)
          {
            to[at] = from[at];
          }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
        {
          s.list[i * kRowThreads + threadIdx.x] = ranks[i];
        }
      }
      __syncthreads();
      if (plan.kind == kChosen)
      {
        return;
      }
      const double inv_t = plan.inv_t;
      const float top = plan.top;
      const int listed = plan.listed;
      if (listed <= kList)
      {
        if (listed > 2 * kRowThreads)
        {
          constexpr int kMore = kList / kRowThreads - 2;
          unsigned long long ranks[kMore];
#pragma unroll
          for (int i = 0; i < kMore; ++i)
          {
            const int at = (i + 2) * kRowThreads + static_cast<int>(threadIdx.x);
            ranks[i] = at < listed ? list[at] : 0;
          }
#pragma unroll
          for (int i = 0; i < kMore; ++i)
          {
            s.list[(i + 2) * kRowThreads + threadIdx.x] = ranks[i];
          }
        }
        list = s.list;
      }
      for (int q = threadIdx.x; q < a.parts; q += kRowThreads)
      {
        s.border[q] = 0;
      }
      __syncthreads();
      const RowSampler r{s, plan, list, listed};

      // The border so far: nothing left out.
      Border border{kBuckets, 0, {0, 0}};
      double total = plan.weight[kBuckets - 1]; // of the weights kept by top_k
      if (plan.k_bucket < kBuckets)
      {
        const int b = plan.k_bucket;
        double kept = 0.0;
        border.bucket = b;
        border.in = ranks_of(plan.from[0], plan.to[0]);
        border.rank = r.cut(b, border.in, k - (b > 0 ? plan.count[b - 1] : 0), INFINITY, &kept);
        total = (b > 0 ? plan.weight[b - 1] : 0.0) + kept;
      }
      if (plan.p_first <= plan.p_last)
      {
        const double need = static_cast<double>(fmaxf(p, 0.0f)) * total;
        int b = plan.p_first;
        while (b < plan.p_last && plan.weight[b] < need)
        {
          ++b;
        }
        double kept = 0.0;
        const Ranks in = plan.p_first == plan.p_last ? ranks_of(plan.from[1], plan.to[1])
                                                     : ranks_of(least_key(plan, b), most_key(plan, b));
        const unsigned long long rank =
            r.cut(b, in, 1ll << 40, need - (b > 0 ? plan.weight[b - 1] : 0.0), &kept);
        if (b < border.bucket || rank > border.rank)
        {
          border = {b, rank, in};
        }
      }
      if (plan.min_bucket < border.bucket ||
          (plan.min_bucket == border.bucket && plan.min_rank > border.rank))
      {
        border = {plan.min_bucket, plan.min_rank, ranks_of(plan.from[2], plan.to[2])};
      }

      // Each part's kept weights: those before the plan's first bucket, those of
      // the buckets from there to the border's, and the border's own by their ranks.
      double unit = 1.0; // of the border's weights: a part has 4,096 of them at most
      if (border.bucket < kBuckets)
      {
        const unsigned long long lo = max(border.rank, border.in.lo);
        const int units = 51 - power_above(logit_of(border.in.hi), top, inv_t);
        const double scale = ldexp(1.0, units);
        unit = ldexp(1.0, -units);
        r.each([&](unsigned long long rank) {
          if (rank >= lo && rank <= border.in.hi)
          {
            atomicAdd(&s.border[index_of(rank) / kPart],
                      units_of(weight_of(logit_of(rank), top, inv_t) * scale));
          }
        });
      }
      __syncthreads();
      double part_kept = 0.0;
      const int mine = threadIdx.x;
      const int shift = mine < a.parts ? plan.shift[mine] : kBuckets;
      if (mine < a.parts)
      {
        const std::size_t slot = static_cast<std::size_t>(row) * a.parts + mine;
        unsigned long long more = 0;
        for (int b = max(plan.first, shift); b < border.bucket; ++b)
        {
          more += a.sums[slot * kBuckets + (b - shift)] & kSumMask;
        }
        part_kept = a.sure[slot] + static_cast<double>(more) * plan.scale[mine] +
                    static_cast<double>(s.border[mine]) * unit;
      }
      // The part that holds the uniform's share.
      const double upto = scan(part_kept, s.waves);
      if (threadIdx.x == kRowThreads - 1)
      {
        s.value = upto;
      }
      __syncthreads();
      const double share = (uniform > 0.0f ? fmin(static_cast<double>(uniform), 1.0) : 0.0) * s.value;
      const int part = max(last_of(part_kept > 0.0 && upto - part_kept <= share, s.lasts), 0);
      if (mine == part)
      {
        s.value = share - (upto - part_kept);
      }
      __syncthreads();
      const double left = s.value;
      // Its weights in turn, eight consecutive a thread.
      constexpr int kEach = kPart / kRowThreads, W = kWide<kHalf>;
      const void *logits = row_of<kHalf>(a, row);
      const int i0 = part * kPart + kEach * mine, part_shift = plan.shift[part];
      u32x4 raw[kEach / W];
#pragma unroll
      for (int c = 0; c < kEach / W; ++c)
      {
        raw[c] = logits_at<kHalf>(logits, i0 + W * c, a.vocab, a.aligned);
      }
      double w[kEach], sum = 0.0;
#pragma unroll
      for (int e = 0; e < kEach; ++e)
      {
        const float l = logit_in<kHalf>(raw[e / W], e % W);
        const int below = plan.highest - bucket_of(l, plan.steps);
        const bool kept = counts(l) && below - part_shift < kBuckets &&
                          (below < border.bucket ||
                           (below == border.bucket && rank_of(l, i0 + e) >= border.rank));
        w[e] = kept ? weight_of(l, top, inv_t) : 0.0;
        sum += w[e];
      }
      double before = scan(sum, s.waves) - sum;
      int found = a.vocab, last = -1;
#pragma unroll
      for (int e = 0; e < kEach; ++e)
      {
        before += w[e];
        if (w[e] > 0.0)
        {
          last = i0 + e;
          if (before > left && found == a.vocab)
          {
            found = i0 + e;
          }
        }
      }
      // (The share may pass the part's own sum by a rounding: then its last.)
      const int by = first_of(found < a.vocab, kRowThreads, s.firsts);
      const int end = last_of(last >= 0, s.lasts);
      if (by < kRowThreads ? mine == by : mine == end)
      {
        a.tokens[row] = by < kRowThreads ? found : last;
      }
    }

    int parts_of(int vocab) { return (vocab + kPart - 1) / kPart; }

    void check_sizes(int rows, int vocab)
    {
      if (rows < 0 || vocab < 0)
      {
        throw InvalidArgument("rows and vocab must not be negative, got " + std::to_string(rows) +
                              " and " + std::to_string(vocab));
      }
      if (vocab > kMostVocab || rows > 65535)
      {
        throw InvalidArgument("sampling takes at most 65535 rows of " + std::to_string(kMostVocab) +
                              " logits, got " + std::to_string(rows) + " of " +
                              std::to_string(vocab));
      }
    }
  } // namespace

  std::size_t sample_scratch_floats(int rows, int vocab)
  {
    check_sizes(rows, vocab);
    // In eight bytes: the list, the parts' histograms and numbers, the plan.
    return 2 * static_cast<std::size_t>(rows) *
           (vocab + static_cast<std::size_t>(parts_of(vocab)) * (kBuckets + 2) + sizeof(RowPlan) / 8);
  }

  void launch_sample(const Sampling &t, hipStream_t stream)
  {
    check_sizes(t.rows, t.vocab);
    const long long stride = t.stride > 0 ? t.stride : t.vocab;
    if (t.stride < 0 || stride < t.vocab)
    {
      throw InvalidArgument("a row's logits are " + std::to_string(t.vocab) +
                            " elements apart at least (0: those), got " + std::to_string(t.stride));
    }
    if (t.rows == 0)
    {
      return;
    }
    if (t.vocab == 0)
    {
      throw InvalidArgument("sampling needs a token at least");
    }
    const std::size_t need = sample_scratch_floats(t.rows, t.vocab);
    if (t.scratch == nullptr || t.scratch_floats < need)
    {
      throw InvalidArgument("sampling's scratch needs " + std::to_string(need) + " floats; got " +
                            std::to_string(t.scratch == nullptr ? 0 : t.scratch_floats));
    }
    if (t.logits == nullptr || t.uniforms == nullptr || t.tokens == nullptr)
    {
      throw InvalidArgument("sampling needs logits, uniforms and tokens");
    }
    const auto address = [](const void *p) { return reinterpret_cast<std::uintptr_t>(p); };
    if (address(t.scratch) % 16 != 0 || address(t.logits) % (t.half ? 2 : 4) != 0 ||
        (address(t.uniforms) | address(t.temperature) | address(t.top_k) | address(t.top_p) |
         address(t.min_p) | address(t.tokens)) % 4 != 0)
    {
      throw InvalidArgument("sampling's scratch must be 16-byte aligned, its numbers as they are wide");
    }
    const std::size_t rows = static_cast<std::size_t>(t.rows);
    const std::size_t each = t.half ? 2 : 4;
    const Extent tokens{t.tokens, 4 * rows}, scratch{t.scratch, 4 * need};
    for (const Extent &read : {Extent{t.logits, each * t.vocab, rows, each * stride},
                               Extent{t.uniforms, 4 * rows}, Extent{t.temperature, 4 * rows},
                               Extent{t.top_k, 4 * rows}, Extent{t.top_p, 4 * rows},
                               Extent{t.min_p, 4 * rows}})
    {
      if (overlaps(tokens, read) || overlaps(scratch, read))
      {
        throw InvalidArgument("sampling cannot write over what it reads");
      }
    }
    if (overlaps(tokens, scratch))
    {
      throw InvalidArgument("sampling's scratch lies over its tokens");
    }
    SampleArgs a{};
    a.logits = t.logits;
    a.stride = stride;
    a.aligned = address(t.logits) % 16 == 0 && stride * static_cast<long long>(each) % 16 == 0;
    a.uniforms = t.uniforms;
    a.temperature = t.temperature;
    a.top_k = t.top_k;
    a.top_p = t.top_p;
    a.min_p = t.min_p;
    a.tokens = t.tokens;
    a.vocab = t.vocab;
    a.parts = parts_of(t.vocab);
    static_assert(sizeof(RowPlan) % 8 == 0, "plans lie one after another");
    const std::size_t slots = rows * a.parts;
    a.sums = static_cast<unsigned long long *>(t.scratch);
    a.lists = a.sums + slots * kBuckets;
    a.sure = reinterpret_cast<double *>(a.lists + rows * t.vocab);
    a.plans = reinterpret_cast<RowPlan *>(a.sure + slots);
    a.tops = reinterpret_cast<float *>(a.plans + rows);
    a.top_at = reinterpret_cast<int *>(a.tops + slots);
    const dim3 grid(a.parts, t.rows);
    const auto launch = [&](auto half) {
      constexpr bool kHalf = decltype(half)::value;
      sample_parts_kernel<kHalf><<<grid, kThreads, 0, stream>>>(a);
      sample_plan_kernel<<<t.rows, kRowThreads, 0, stream>>>(a);
      sample_gather_kernel<kHalf><<<grid, kThreads, 0, stream>>>(a);
      sample_choose_kernel<kHalf><<<t.rows, kRowThreads, 0, stream>>>(a);
    };
    t.half ? launch(std::true_type{}) : launch(std::false_type{});
    hip_check(hipGetLastError(), "sample kernels");
  }

} // namespace mi
