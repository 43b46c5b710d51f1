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
// largest logit and a histogram of the others below it: buckets of an eighth
// of a nat, floor(8 l / T), on one grid for the whole row, each with its count
// and its weights' sum. The second (a workgroup a row) adds the parts' up, and
// knows from them the bucket that each border (k, p, min-p) falls into. Only
// the logits of such a bucket are looked at again, in the parts that have any:
// they are put in order, and the border found among them. With the kept part of
// every bucket known, so is the part that the token is in, whose weights are
// then added in turn.
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
    constexpr int kBuckets = 256; // an eighth of a nat each: 32 nats below the largest
    constexpr int kPerNat = 8;
    constexpr int kRowThreads = 1024;
    constexpr int kList = 2048;   // logits of a border's bucket held in LDS
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
    __device__ inline int on_grid(double eighths)
    {
      constexpr double kFar = 1 << 29;
      return static_cast<int>(fmin(fmax(floor(eighths), -kFar), kFar));
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
      s_sums[threadIdx.x] = 0;
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
      a.sums[slot * kBuckets + threadIdx.x] = s_sums[threadIdx.x];
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
      int counts4[4][kBuckets]; // of quarters of the parts
      double weights4[4][kBuckets];
      int count[kBuckets];      // of the row, up to and with each bucket
      double weight[kBuckets];
      short with[kMostParts];   // the parts that have logits of a border's bucket
      double scale[kMostParts]; // of a part's weights in the row's
      short shift[kMostParts];  // a part's bucket 0 among the row's; kBuckets: none of it
      double kept[kMostParts];  // a part's kept weights
      unsigned long long list[kList];
      unsigned long long bins[256]; // narrowing a border that is too wide for the list
      double waves[kRowThreads / 64];
      int int_waves[kRowThreads / 64];
      int ints[4];
      double value;
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

      // Calls f(rank, logit) for the logits of buckets [b, end), by threads; the
      // parts that have none are passed over.
      template <typename F>
      __device__ void each(int b, int end, F &&f) const
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
          const float l = at < a.vocab ? logit_at<kHalf>(logits, at) : -INFINITY;
          if (counts(l))
          {
            const int below = highest - bucket_of(l, inv_t);
            if (below >= b && below < end && below - s.shift[part] < kBuckets)
            {
              f(rank_of(l, at), l);
            }
          }
        }
      }

      // The list's first n ranks in order, largest first.
      __device__ void sort(int n) const
      {
        int size = 64;
        while (size < n)
        {
          size *= 2;
        }
        for (int i = n + threadIdx.x; i < size; i += kRowThreads)
        {
          s.list[i] = 0;
        }
        __syncthreads();
        for (int k = 2; k <= size; k *= 2)
        {
          for (int j = k / 2; j > 0; j /= 2)
          {
            for (int i = threadIdx.x; i < size / 2; i += kRowThreads)
            {
              const int lo = 2 * j * (i / j) + i % j, hi = lo + j;
              const unsigned long long x = s.list[lo], y = s.list[hi];
              const bool down = (lo & k) == 0;
              if ((x < y) == down)
              {
                s.list[lo] = y;
                s.list[hi] = x;
              }
            }
            __syncthreads();
          }
        }
      }

      // The border among the logits of buckets [b, end), of which the first are
      // kept: as long as they are fewer than `most` and `reached` of their
      // weights' sum so far (their own not in it) does not hold, and they weigh
      // `least`. One of them is kept at least where `most` and `need` are
      // positive. Returns the rank of the last kept (all ones: none), and to
      // *sum the weights of the kept.
      __device__ unsigned long long cut(int b, int end, long long most, double need, double least,
                                        double *sum) const
      {
        // Ranks in [lo, hi] are looked at; what ranks above hi, within the
        // buckets, is kept: `taken` logits of weight `weight`.
        unsigned long long lo = 0, hi = ~0ull;
        long long taken = 0;
        double weight = 0.0;
        for (;;)
        {
          if (threadIdx.x == 0)
          {
            s.ints[0] = 0;
          }
          __syncthreads();
          each(b, end, [&](unsigned long long rank, float) {
            if (rank >= lo && rank <= hi)
            {
              const int at = atomicAdd(&s.ints[0], 1);
              if (at < kList)
              {
                s.list[at] = rank;
              }
            }
          });
          __syncthreads();
          const int n = s.ints[0];
          if (n <= kList)
          {
            sort(n);
            // Two a thread, in order.
            const int i0 = 2 * threadIdx.x;
            double w[2];
#pragma unroll
            for (int e = 0; e < 2; ++e)
            {
              w[e] = i0 + e < n ? weight_of(logit_of(s.list[i0 + e]), top, inv_t) : 0.0;
            }
            const double upto = scan(w[0] + w[1], s.waves);
            double before = weight + (upto - (w[0] + w[1]));
            if (threadIdx.x == 0)
            {
              s.ints[1] = 0;
              s.value = 0.0;
            }
            __syncthreads();
#pragma unroll
            for (int e = 0; e < 2; ++e)
            {
              const int i = i0 + e;
              if (i < n && taken + i < most && (before < need || taken + i == 0) && w[e] >= least)
              {
                atomicMax(&s.ints[1], i + 1);
              }
              before += w[e];
            }
            __syncthreads();
            const int kept = s.ints[1];
            before = weight + (upto - (w[0] + w[1]));
#pragma unroll
            for (int e = 0; e < 2; ++e)
            {
              before += w[e];
              if (i0 + e == kept - 1)
              {
                s.value = before;
              }
            }
            __syncthreads();
            *sum = kept > 0 ? s.value : weight;
            const unsigned long long rank = kept > 0 ? s.list[kept - 1] : hi == ~0ull ? ~0ull : hi + 1;
            __syncthreads();
            return rank;
          }
          // Too many: 256 equal ranges of [lo, hi], and the one with the border.
          narrow(b, end, most, need, least, lo, hi, taken, weight);
        }
      }

      __device__ void narrow(int b, int end, long long most, double need, double least,
                             unsigned long long &lo, unsigned long long &hi, long long &taken,
                             double &weight) const
      {
        // The ranks there are.
        if (threadIdx.x == 0)
        {
          s.bins[0] = ~0ull;
          s.bins[1] = 0;
        }
        __syncthreads();
        each(b, end, [&](unsigned long long rank, float) {
          if (rank >= lo && rank <= hi)
          {
            atomicMin(&s.bins[0], rank);
            atomicMax(&s.bins[1], rank);
          }
        });
        __syncthreads();
        lo = s.bins[0];
        hi = s.bins[1];
        __syncthreads();
        // (hi > lo: ranks differ, and there are many.)
        const unsigned long long step = (hi - lo) / 256 + 1;
        for (int i = threadIdx.x; i < 256; i += kRowThreads)
        {
          s.bins[i] = 0;
        }
        // Weights as whole numbers again; 2^20 of at most 2^38 stay below 2^58.
        __shared__ int s_counts[256];
        for (int i = threadIdx.x; i < 256; i += kRowThreads)
        {
          s_counts[i] = 0;
        }
        __syncthreads();
        each(b, end, [&](unsigned long long rank, float l) {
          if (rank >= lo && rank <= hi)
          {
            const int bin = static_cast<int>((hi - rank) / step);
            atomicAdd(&s_counts[bin], 1);
            atomicAdd(&s.bins[bin],
                      static_cast<unsigned long long>(rint(weight_of(l, top, inv_t) * kUnit)));
          }
        });
        __syncthreads();
        // The bin with the border: the first that cannot be kept whole.
        int bin = 0;
        for (; bin < 255; ++bin)
        {
          const long long with = taken + s_counts[bin];
          const double sum = weight + static_cast<double>(s.bins[bin]) / kUnit;
          // Its last logit's rank is at least hi - step (bin + 1) + 1: none weighs less.
          const unsigned long long last = hi - lo < step * (bin + 1) - 1 ? lo : hi - (step * (bin + 1) - 1);
          if (with >= most || sum >= need || weight_of(logit_of(last), top, inv_t) < least)
          {
            break;
          }
          taken = with;
          weight = sum;
        }
        const unsigned long long above = hi - step * bin;
        lo = above - lo < step ? lo : above - (step - 1);
        hi = above;
        __syncthreads();
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
        const int bucket = threadIdx.x % kBuckets, quarter = threadIdx.x / kBuckets;
        int count = 0;
        double weight = 0.0;
#pragma unroll 8
        for (int p = quarter; p < a.parts; p += 4)
        {
          const int of = bucket - s.shift[p];
          const unsigned long long v =
              of >= 0 ? r.sums[static_cast<std::size_t>(p) * kBuckets + of] : 0;
          count += static_cast<int>(v >> kCountShift);
          weight += static_cast<double>(v & kSumMask) * s.scale[p];
        }
        s.counts4[quarter][bucket] = count;
        s.weights4[quarter][bucket] = weight;
      }
      __syncthreads();
      {
        const int b = threadIdx.x % kBuckets;
        const bool mine = threadIdx.x < kBuckets;
        const int count = mine ? s.counts4[0][b] + s.counts4[1][b] + s.counts4[2][b] + s.counts4[3][b] : 0;
        const double weight = mine ? (s.weights4[0][b] + s.weights4[1][b]) +
                                         (s.weights4[2][b] + s.weights4[3][b])
                                   : 0.0;
        const int count_upto = scan(count, s.int_waves);
        const double weight_upto = scan(weight, s.waves);
        if (mine)
        {
          s.count[b] = count_upto;
          s.weight[b] = weight_upto;
        }
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
        if (threadIdx.x < kBuckets && holds(static_cast<int>(threadIdx.x)))
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
      for (int q = wave; q < a.parts; q += kRowThreads / 64)
      {
        double kept = 0.0;
#pragma unroll
        for (int c = 0; c < kBuckets / 64; ++c)
        {
          const int of = lane + 64 * c;
          const unsigned long long v = of + s.shift[q] < border.bucket
                                           ? r.sums[static_cast<std::size_t>(q) * kBuckets + of]
                                           : 0;
          kept += static_cast<double>(v & kSumMask);
        }
#pragma unroll
        for (int offset = 1; offset < 64; offset *= 2)
        {
          kept += __shfl_xor(kept, offset);
        }
        if (lane == 0)
        {
          s.kept[q] = kept * s.scale[q];
        }
      }
      __shared__ unsigned long long s_border[kMostParts];
      for (int q = threadIdx.x; q < a.parts; q += kRowThreads)
      {
        s_border[q] = 0;
      }
      __syncthreads();
      if (border.bucket < kBuckets)
      {
        r.each(border.bucket, border.bucket + 1, [&](unsigned long long rank, float l) {
          if (rank >= border.rank)
          {
            atomicAdd(&s_border[index_of(rank) / kPart],
                      static_cast<unsigned long long>(rint(weight_of(l, top, inv_t) * kUnit)));
          }
        });
      }
      __syncthreads();
      // The part that holds the uniform's share.
      const double part_kept =
          static_cast<int>(threadIdx.x) < a.parts
              ? s.kept[threadIdx.x] + static_cast<double>(s_border[threadIdx.x]) / kUnit
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
    return static_cast<std::size_t>(rows) * parts_of(vocab) * (2 * kBuckets + 2);
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
    a.tops = reinterpret_cast<float *>(a.sums + slots * kBuckets);
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
