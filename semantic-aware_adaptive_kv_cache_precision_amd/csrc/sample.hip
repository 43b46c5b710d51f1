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
// Two launches. The first (a workgroup 4,096 logits of a row) finds its part's
// largest logit and a histogram of the others below it: buckets of a
// thirty-second of a nat, floor(32 l / T), on one grid for the whole row, each
// with its count and its weights' sum. The second (a workgroup a row) adds the
// parts' up, and knows from them the bucket that each border (k, p, min-p)
// falls into. A bucket is a range of logits: only those are looked for again, in
// the parts that have any, and the border found among them, by histograms of
// their ranks until 64 are left to be put in order. With the kept part of every
// bucket known, so is the part that the token is in, whose weights are then
// added in turn.
//
// Sums: a bucket's weights are added as whole numbers of 2^-38 of the part's
// largest, by LDS atomics of 64 bits (13 of them the count), so that the order
// of adding does not matter; everything else in fp64, in one order. A weight
// below 2^-39 of the largest counts as none.
#include "common.hpp"
#include "ragged.hpp"

#include <algorithm>
#include <string>

namespace mi
{
  namespace
  {
    typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
    typedef float f32x4 __attribute__((ext_vector_type(4)));

    constexpr int kPart = 4096;   // logits a part
    constexpr int kThreads = 256; // of a part's workgroup
    constexpr int kBuckets = 1024; // 32 nats below the largest
    constexpr int kPerNat = 32;
    constexpr int kRowThreads = 1024; // a bucket each
    constexpr int kList = 2048;       // logits of a border's bucket held in LDS
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
      const float *uniforms;
      const float *temperature;
      const int *top_k;
      const float *top_p;
      const float *min_p;
      int *tokens;
      int vocab;
      int parts;
      unsigned long long *sums; // [row][part][bucket] count << 51 | weights
      double *whole;            // [row][part] the weights of them all
      float *tops;              // [row][part] largest logit
      int *top_at;              // and its index, or vocab
    };

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

    // The bucket on the row's grid; larger for larger logits.
    __device__ inline int on_grid(double steps)
    {
      constexpr double kFar = 1 << 29;
      return static_cast<int>(fmin(fmax(floor(steps), -kFar), kFar));
    }
    __device__ inline int bucket_of(float l, double inv_t)
    {
      return l == INFINITY ? 1 << 30 : on_grid(kPerNat * (static_cast<double>(l) * inv_t));
    }

    __device__ inline double weight_of(float l, float top, double inv_t)
    {
      return l == top          ? 1.0
             : top == INFINITY ? 0.0
                               : exp((static_cast<double>(l) - static_cast<double>(top)) * inv_t);
    }

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
      const int count = min(kPart, a.vocab - first);
      const double inv_t = inverse_temperature(a, row);
      constexpr int kEach = kPart / kThreads;
      float l[kEach];
#pragma unroll
      for (int e = 0; e < kEach; ++e)
      {
        const int i = e * kThreads + threadIdx.x;
        l[e] = i < count ? logit_at<kHalf>(logits, first + i) : -INFINITY;
      }
#pragma unroll
      for (int b = 0; b < kBuckets; b += kThreads)
      {
        s_sums[b + threadIdx.x] = 0;
      }
      // The largest, and the lowest index that has it.
      float top = -INFINITY;
      int at = a.vocab;
#pragma unroll
      for (int e = 0; e < kEach; ++e)
      {
        if (l[e] > top)
        {
          top = l[e];
          at = first + e * kThreads + static_cast<int>(threadIdx.x);
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
        const int highest = bucket_of(top, inv_t);
#pragma unroll
        for (int e = 0; e < kEach; ++e)
        {
          if (counts(l[e]))
          {
            const int below = highest - bucket_of(l[e], inv_t);
            if (below < kBuckets)
            {
              const double w = weight_of(l[e], top, inv_t) * kUnit;
              atomicAdd(&s_sums[below], (1ull << kCountShift) + static_cast<unsigned long long>(rint(w)));
            }
          }
        }
      }
      __syncthreads();
      unsigned long long whole = 0;
#pragma unroll
      for (int b = 0; b < kBuckets; b += kThreads)
      {
        const unsigned long long v = s_sums[b + threadIdx.x];
        a.sums[slot * kBuckets + b + threadIdx.x] = v;
        whole += v & kSumMask;
      }
#pragma unroll
      for (int offset = 1; offset < 64; offset *= 2)
      {
        whole += __shfl_xor(whole, offset);
      }
      __syncthreads();
      if (threadIdx.x % 64 == 0)
      {
        s_sums[threadIdx.x / 64] = whole;
      }
      __syncthreads();
      if (threadIdx.x == 0)
      {
        a.whole[slot] = static_cast<double>(s_sums[0] + s_sums[1] + s_sums[2] + s_sums[3]);
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

    // Inclusive sums over the workgroup's threads, in thread order.
    template <typename T>
    __device__ inline T scan(T v, T *s_waves)
    {
      const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
      for (int offset = 1; offset < 64; offset *= 2)
      {
        const T before = __shfl_up(v, offset);
        v = lane >= offset ? v + before : v;
      }
      __syncthreads(); // the last scan's sums are read
      if (lane == 63)
      {
        s_waves[wave] = v;
      }
      __syncthreads();
      T before = 0;
      for (int w = 0; w < wave; ++w)
      {
        before += s_waves[w];
      }
      return before + v;
    }

    struct RowState
    {
      int count[kBuckets];      // of the row, up to and with each bucket
      double weight[kBuckets];
      double scale[kMostParts]; // of a part's weights in the row's
      short shift[kMostParts];  // a part's bucket 0 among the row's; kBuckets: none of it
      short with[kMostParts];   // the parts that have logits of a border's bucket
      double kept[kMostParts];  // a part's kept weights
      unsigned long long border[kMostParts]; // of the border's bucket
      unsigned long long list[kList];
      unsigned long long bins[kRowThreads]; // histograms of ranks
      int bin_counts[kRowThreads];
      unsigned long long few[kFew];
      double waves[kRowThreads / 64];
      int int_waves[kRowThreads / 64];
      int ints[4];
      unsigned long long rank;
      double value;
      int listed;
    };

    // A border: everything in buckets before `bucket` is kept, and in it what
    // ranks at least `rank`.
    struct Border
    {
      int bucket;
      unsigned long long rank;
    };

    template <bool kHalf>
    struct RowSampler
    {
      const SampleArgs &a;
      RowState &s;
      const void *logits;
      const unsigned long long *sums; // the row's histograms
      double inv_t;
      float top;
      int highest;
      int held = -1; // the bucket whose logits are all in the list

      // The least logit, as the upper half of a rank, of a bucket on the grid
      // or above: by 64 pivots at a time.
      __device__ unsigned first_key(int bucket) const
      {
        const unsigned lane = threadIdx.x & 63;
        unsigned lo = 0x00800000u, hi = 0xFF800001u; // the least finite; past infinity
        while (lo < hi)
        {
          const unsigned step = (hi - lo) / 64 + 1;
          const unsigned long long at = lo + static_cast<unsigned long long>(lane) * step;
          const bool reached =
              at >= hi ||
              bucket_of(logit_of(at << 32), inv_t) >= bucket;
          const int before = __popcll(~__ballot(reached));
          const unsigned long long next = lo + static_cast<unsigned long long>(before) * step;
          lo = before > 0 ? static_cast<unsigned>(next - step + 1) : lo;
          hi = static_cast<unsigned>(min(next, static_cast<unsigned long long>(hi)));
        }
        return __builtin_amdgcn_readfirstlane(lo);
      }

      // Calls f(rank, logit) for the row's logits of buckets [b, end), which
      // are those from `least` to `most`; the parts that have none are passed over.
      template <typename F>
      __device__ void each(int b, int end, float least, float most, F &&f) const
      {
        __syncthreads();
        if (threadIdx.x == 0)
        {
          s.ints[3] = 0;
        }
        __syncthreads();
        for (int part = threadIdx.x; part < a.parts; part += kRowThreads)
        {
          bool any = false;
          for (int c = b; c < end; ++c)
          {
            const int of = c - s.shift[part];
            any = any || (of >= 0 && of < kBuckets &&
                          sums[static_cast<std::size_t>(part) * kBuckets + of] != 0);
          }
          if (any)
          {
            s.with[atomicAdd(&s.ints[3], 1)] = static_cast<short>(part);
          }
        }
        __syncthreads();
        const int all = s.ints[3] * kPart;
#pragma unroll 4
        for (int i = threadIdx.x; i < all; i += kRowThreads)
        {
          const int part = s.with[i / kPart], at = part * kPart + i % kPart;
          const float l = at < a.vocab ? logit_at<kHalf>(logits, at) : NAN;
          if (l >= least && l <= most)
          {
            f(rank_of(l, at), l);
          }
        }
      }

      // Of the ranks in [lo, hi], `source` calls back with each, those above the
      // border are counted as taken, and [lo, hi] becomes the 1,024th of it that
      // has the border. Returns how many are in it.
      template <typename S>
      __device__ int narrow(S &&source, long long most, double need, double least,
                            unsigned long long &lo, unsigned long long &hi, long long &taken,
                            double &weight) const
      {
        const unsigned long long step = (hi - lo) / kRowThreads + 1;
        s.bins[threadIdx.x] = 0;
        s.bin_counts[threadIdx.x] = 0;
        if (threadIdx.x == 0)
        {
          s.ints[1] = kRowThreads - 1;
        }
        __syncthreads();
        source([&](unsigned long long rank, float l) {
          if (rank >= lo && rank <= hi)
          {
            const int bin = static_cast<int>((hi - rank) / step);
            atomicAdd(&s.bin_counts[bin], 1);
            // (2^20 of at most 2^38 stay below 2^58.)
            atomicAdd(&s.bins[bin],
                      static_cast<unsigned long long>(rint(weight_of(l, top, inv_t) * kUnit)));
          }
        });
        __syncthreads();
        const int bin = threadIdx.x;
        const int mine = s.bin_counts[bin];
        const double own = static_cast<double>(s.bins[bin]) / kUnit;
        const int count = scan(mine, s.int_waves);
        const double sum = scan(own, s.waves);
        // The first bin that cannot be kept whole has the border. (The least
        // rank a bin may hold weighs too little: none after it can weigh enough.)
        const unsigned long long end = step * (bin + 1) - 1;
        const unsigned long long last = hi - lo < end ? lo : hi - end;
        if (taken + count >= most || (taken + count > 0 && weight + sum >= need) ||
            weight_of(logit_of(last), top, inv_t) < least)
        {
          atomicMin(&s.ints[1], bin);
        }
        __syncthreads();
        const int at = s.ints[1];
        if (bin == at)
        {
          s.ints[0] = count - mine;
          s.ints[2] = mine;
          s.value = sum - own;
        }
        __syncthreads();
        taken += s.ints[0];
        weight += s.value;
        const unsigned long long above = hi - step * at;
        lo = above - lo < step ? lo : above - (step - 1);
        hi = above;
        const int in = s.ints[2];
        __syncthreads();
        return in;
      }

      // The border among the logits of buckets [b, end), of which the first are
      // kept: as long as they are fewer than `most`, the weights before them
      // less than `need`, and they weigh `least`; one at least if `need` is not
      // more than nothing. Returns the rank of the last kept (all ones: none
      // is), and to *sum the weights of the kept.
      __device__ unsigned long long cut(int b, int end, long long most, double need, double least,
                                        double *sum)
      {
        const unsigned key_lo = first_key(highest - end + 1);
        const unsigned key_hi = b == 0 ? static_cast<unsigned>(rank_of(top, 0) >> 32)
                                       : first_key(highest - b + 1) - 1;
        const float from = logit_of(static_cast<unsigned long long>(key_lo) << 32);
        const float to = logit_of(static_cast<unsigned long long>(key_hi) << 32);
        unsigned long long lo = static_cast<unsigned long long>(key_lo) << 32;
        unsigned long long hi = static_cast<unsigned long long>(key_hi) << 32 | 0xFFFFFFFFull;
        long long taken = 0;
        double weight = 0.0;
        int n = s.count[end - 1] - (b > 0 ? s.count[b - 1] : 0);
        const auto row = [&](auto &&f) { each(b, end, from, to, f); };
        const bool whole = n <= kList && end == b + 1;
        if (!(whole && held == b))
        {
          held = -1;
          while (n > kList)
          {
            n = narrow(row, most, need, least, lo, hi, taken, weight);
          }
          if (threadIdx.x == 0)
          {
            s.listed = 0;
          }
          row([&](unsigned long long rank, float) {
            if (rank >= lo && rank <= hi)
            {
              s.list[atomicAdd(&s.listed, 1)] = rank;
            }
          });
          held = whole ? b : -1;
          __syncthreads();
        }
        const int listed = s.listed;
        const auto list = [&](auto &&f) {
          for (int i = threadIdx.x; i < listed; i += kRowThreads)
          {
            f(s.list[i], logit_of(s.list[i]));
          }
        };
        while (n > kFew)
        {
          n = narrow(list, most, need, least, lo, hi, taken, weight);
        }
        // The few in order, by each one's place among them.
        if (threadIdx.x == 0)
        {
          s.ints[0] = 0;
          s.ints[1] = 0;
          s.value = weight;
          s.rank = hi == ~0ull ? hi : hi + 1; // none of them: what ranks above
        }
        __syncthreads();
        list([&](unsigned long long rank, float) {
          if (rank >= lo && rank <= hi)
          {
            s.bins[atomicAdd(&s.ints[0], 1)] = rank;
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
            s.few[place] = own;
          }
        }
        __syncthreads();
        const int i = threadIdx.x;
        const double w = i < n ? weight_of(logit_of(s.few[min(i, kFew - 1)]), top, inv_t) : 0.0;
        const double upto = weight + scan(w, s.waves);
        if (i < n && taken + i < most && (upto - w < need || taken + i == 0) && w >= least)
        {
          atomicMax(&s.ints[1], i + 1);
        }
        __syncthreads();
        if (i == s.ints[1] - 1)
        {
          s.value = upto;
          s.rank = s.few[i];
        }
        __syncthreads();
        *sum = s.value;
        const unsigned long long rank = s.rank;
        __syncthreads();
        return rank;
      }
    };

    template <bool kHalf>
    __global__ void __launch_bounds__(kRowThreads) sample_rows_kernel(SampleArgs a)
    {
      __shared__ RowState s;
      const int row = blockIdx.x;
      const double inv_t = inverse_temperature(a, row);
      const float *tops = a.tops + static_cast<std::size_t>(row) * a.parts;
      const int *top_at = a.top_at + static_cast<std::size_t>(row) * a.parts;
      // The row's largest logit.
      float top = -INFINITY;
      int at = a.vocab;
      for (int p = threadIdx.x & 63; p < a.parts; p += 64)
      {
        const float t = tops[p];
        const int i = top_at[p];
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
        }
        return;
      }
      RowSampler<kHalf> r{a, s, row_of<kHalf>(a, row),
                          a.sums + static_cast<std::size_t>(row) * a.parts * kBuckets, inv_t, top,
                          bucket_of(top, inv_t)};
      for (int p = threadIdx.x; p < a.parts; p += kRowThreads)
      {
        const float t = tops[p];
        const int shift = counts(t) ? r.highest - bucket_of(t, inv_t) : kBuckets;
        s.shift[p] = static_cast<short>(min(shift, kBuckets));
        s.scale[p] = counts(t) ? weight_of(t, top, inv_t) / kUnit : 0.0;
      }
      __syncthreads();
      {
        int count = 0;
        double weight = 0.0;
#pragma unroll 8
        for (int p = 0; p < a.parts; ++p)
        {
          const int of = static_cast<int>(threadIdx.x) - s.shift[p];
          const unsigned long long v =
              of >= 0 ? r.sums[static_cast<std::size_t>(p) * kBuckets + of] : 0;
          count += static_cast<int>(v >> kCountShift);
          weight += static_cast<double>(v & kSumMask) * s.scale[p];
        }
        const int count_upto = scan(count, s.int_waves);
        const double weight_upto = scan(weight, s.waves);
        s.count[threadIdx.x] = count_upto;
        s.weight[threadIdx.x] = weight_upto;
      }
      __syncthreads();
      // The first bucket that a condition holds for, kBuckets if none: the
      // condition does not change back.
      const auto first_bucket = [&](auto &&holds) {
        if (threadIdx.x == 0)
        {
          s.ints[0] = kBuckets;
        }
        __syncthreads();
        if (holds(static_cast<int>(threadIdx.x)))
        {
          atomicMin(&s.ints[0], static_cast<int>(threadIdx.x));
        }
        __syncthreads();
        const int b = s.ints[0];
        __syncthreads();
        return b;
      };

      // The border so far: nothing left out.
      Border border{kBuckets, 0};
      const int k = a.top_k != nullptr ? a.top_k[row] : 0;
      const float p = a.top_p != nullptr ? a.top_p[row] : 1.0f;
      const float m = a.min_p != nullptr ? a.min_p[row] : 0.0f;
      double total = s.weight[kBuckets - 1]; // of the weights kept by top_k
      if (k > 0)
      {
        const int b = first_bucket([&](int i) { return s.count[i] >= k; });
        if (b < kBuckets)
        {
          double kept = 0.0;
          border.bucket = b;
          border.rank = r.cut(b, b + 1, k - (b > 0 ? s.count[b - 1] : 0), INFINITY, 0.0, &kept);
          total = (b > 0 ? s.weight[b - 1] : 0.0) + kept;
        }
      }
      if (p < 1.0f)
      {
        const double need = static_cast<double>(fmaxf(p, 0.0f)) * total;
        const int b = min(first_bucket([&](int i) { return s.weight[i] >= need; }),
                          min(border.bucket, kBuckets - 1));
        double kept = 0.0;
        const unsigned long long rank =
            r.cut(b, b + 1, 1ll << 40, need - (b > 0 ? s.weight[b - 1] : 0.0), 0.0, &kept);
        if (b < border.bucket || rank > border.rank)
        {
          border.bucket = b;
          border.rank = rank;
        }
      }
      if (m > 0.0f)
      {
        // The buckets that min_p's border may lie in: one, or two at an edge.
        const double least = static_cast<double>(fminf(m, 1.0f));
        const double edge = kPerNat * (static_cast<double>(top) * inv_t + log(least));
        const int b = top == INFINITY ? 0 : max(r.highest - on_grid(edge + 1e-6), 0);
        const int end = top == INFINITY ? 1 : min(max(r.highest - on_grid(edge - 1e-6), 0), kBuckets - 1) + 1;
        if (b <= border.bucket && b < kBuckets)
        {
          double kept = 0.0;
          const unsigned long long rank = r.cut(b, end, 1ll << 40, INFINITY, least, &kept);
          // The last kept's bucket: with none kept in them, all before them are.
          const int of = rank == ~0ull ? b : r.highest - bucket_of(logit_of(rank), inv_t);
          if (of < border.bucket || (of == border.bucket && rank > border.rank))
          {
            border.bucket = of;
            border.rank = rank;
          }
        }
      }

      // Each part's kept weights: those of the buckets before the border's, a
      // wave a part, and the border's own by their ranks.
      const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
      const double *whole = a.whole + static_cast<std::size_t>(row) * a.parts;
      if (border.bucket >= kBuckets)
      {
        for (int q = threadIdx.x; q < a.parts; q += kRowThreads)
        {
          s.kept[q] = s.shift[q] < kBuckets ? whole[q] * s.scale[q] : 0.0;
          s.border[q] = 0;
        }
      }
      else
      {
        for (int q = threadIdx.x; q < a.parts; q += kRowThreads)
        {
          s.border[q] = 0;
        }
        for (int q = wave; q < a.parts; q += kRowThreads / 64)
        {
          unsigned long long kept = 0;
          const int before = border.bucket - s.shift[q];
#pragma unroll 4
          for (int of = lane; of < before; of += 64)
          {
            kept += r.sums[static_cast<std::size_t>(q) * kBuckets + of] & kSumMask;
          }
#pragma unroll
          for (int offset = 1; offset < 64; offset *= 2)
          {
            kept += __shfl_xor(kept, offset);
          }
          if (lane == 0)
          {
            s.kept[q] = static_cast<double>(kept) * s.scale[q];
          }
        }
        __syncthreads();
        const auto add = [&](unsigned long long rank, float l) {
          if (rank >= border.rank)
          {
            atomicAdd(&s.border[index_of(rank) / kPart],
                      static_cast<unsigned long long>(rint(weight_of(l, top, inv_t) * kUnit)));
          }
        };
        if (r.held == border.bucket)
        {
          for (int i = threadIdx.x; i < s.listed; i += kRowThreads)
          {
            add(s.list[i], logit_of(s.list[i]));
          }
        }
        else
        {
          // (What ranks at least the border's last, and lies in its bucket.)
          const unsigned key_hi = border.bucket == 0
                                      ? static_cast<unsigned>(rank_of(top, 0) >> 32)
                                      : r.first_key(r.highest - border.bucket + 1) - 1;
          const float to = logit_of(static_cast<unsigned long long>(key_hi) << 32);
          const float from = border.rank == ~0ull ? INFINITY : logit_of(border.rank);
          r.each(border.bucket, border.bucket + 1, from, to, add);
        }
      }
      __syncthreads();
      // The part that holds the uniform's share.
      const double part_kept =
          static_cast<int>(threadIdx.x) < a.parts
              ? s.kept[threadIdx.x] + static_cast<double>(s.border[threadIdx.x]) / kUnit
              : 0.0;
      const double upto = scan(part_kept, s.waves);
      if (threadIdx.x == kRowThreads - 1)
      {
        s.value = upto;
        s.ints[2] = 0;
      }
      __syncthreads();
      const float uniform = a.uniforms[row];
      const double share = (uniform > 0.0f ? fmin(static_cast<double>(uniform), 1.0) : 0.0) * s.value;
      if (part_kept > 0.0 && upto - part_kept <= share)
      {
        atomicMax(&s.ints[2], static_cast<int>(threadIdx.x));
      }
      __syncthreads();
      const int part = s.ints[2];
      if (static_cast<int>(threadIdx.x) == part)
      {
        s.value = share - (upto - part_kept);
        s.ints[3] = a.vocab;
        s.ints[1] = -1;
      }
      __syncthreads();
      const double left = s.value;
      // Its weights in turn, four consecutive a thread.
      double w[4], sum = 0.0;
      const int i0 = part * kPart + 4 * static_cast<int>(threadIdx.x);
#pragma unroll
      for (int e = 0; e < 4; ++e)
      {
        w[e] = 0.0;
        if (i0 + e < a.vocab)
        {
          const float l = logit_at<kHalf>(r.logits, i0 + e);
          if (counts(l))
          {
            const int below = r.highest - bucket_of(l, inv_t);
            const bool kept = below < border.bucket ||
                              (below == border.bucket && rank_of(l, i0 + e) >= border.rank);
            w[e] = kept && below - s.shift[part] < kBuckets ? weight_of(l, top, inv_t) : 0.0;
          }
        }
        sum += w[e];
      }
      const double all = scan(sum, s.waves);
      double before = all - sum;
      int found = a.vocab, last = -1;
#pragma unroll
      for (int e = 0; e < 4; ++e)
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
      if (found < a.vocab)
      {
        atomicMin(&s.ints[3], found);
      }
      if (last >= 0)
      {
        atomicMax(&s.ints[1], last);
      }
      __syncthreads();
      if (threadIdx.x == 0)
      {
        // (The share may pass the part's own sum by a rounding: then its last.)
        a.tokens[row] = s.ints[3] < a.vocab ? s.ints[3] : s.ints[1];
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
    return static_cast<std::size_t>(rows) * parts_of(vocab) * (2 * kBuckets + 4);
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
    a.uniforms = t.uniforms;
    a.temperature = t.temperature;
    a.top_k = t.top_k;
    a.top_p = t.top_p;
    a.min_p = t.min_p;
    a.tokens = t.tokens;
    a.vocab = t.vocab;
    a.parts = parts_of(t.vocab);
    const std::size_t slots = rows * a.parts;
    a.sums = static_cast<unsigned long long *>(t.scratch);
    a.whole = reinterpret_cast<double *>(a.sums + slots * kBuckets);
    a.tops = reinterpret_cast<float *>(a.whole + slots);
    a.top_at = reinterpret_cast<int *>(a.tops + slots);
    const dim3 grid(a.parts, t.rows);
    if (t.half)
    {
      sample_parts_kernel<true><<<grid, kThreads, 0, stream>>>(a);
      sample_rows_kernel<true><<<t.rows, kRowThreads, 0, stream>>>(a);
    }
    else
    {
      sample_parts_kernel<false><<<grid, kThreads, 0, stream>>>(a);
      sample_rows_kernel<false><<<t.rows, kRowThreads, 0, stream>>>(a);
    }
    hip_check(hipGetLastError(), "sample kernels");
  }

} // namespace mi
