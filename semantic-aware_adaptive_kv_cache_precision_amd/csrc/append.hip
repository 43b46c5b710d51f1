// The rows of a packed batch's new tokens: queries and keys turned to their
// positions, keys and values written into their sequences' FP16 pages.
//
// Row r of sequence s (offsets[s] <= r < offsets[s + 1]) is at position
// p = lengths[s] - (offsets[s + 1] - r). A pair of channels (a, b), (j, j + R/2)
// or interleaved (2j, 2j + 1) for j < R/2, turns by the angle p f_j:
//   a' = a cos - b sin,  b' = b cos + a sin,
// each product and sum rounded in fp32, then to fp16 once (the RoPE kernels'
// own arithmetic, whose rows these are to the bit where the angles are); the
// channels from R on stay as they are. cos and sin come from a table of fp32
// values formed in fp64.
//
// A workgroup takes consecutive rows. It first finds each row's sequence, by
// a search of the offsets held in LDS, and its place in its page, once a row;
// then its threads take 16 channels of a head each: two 16-byte reads, two
// writes to each place a row goes to.
//
// Bound by memory: 9,001 rows of 32 + 2 x 8 heads of 64 (119 MB read and
// written) 29 us, 4.2 TB/s, where a large copy reaches 5.3; by 32 rows of single
// tokens (4.4 us) by a launch and a chain of trips: offsets, page, row. (A
// thread's channels asked for ahead of the row's place: 32.0 us for 30.3.)
#include "common.hpp"
#include "ragged.hpp"

#include <algorithm>
#include <cmath>
#include <string>
#include <type_traits>

namespace mi
{
  namespace
  {
    typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

    constexpr int kThreads = 256;
    constexpr int kOffsetsHeld = 2048; // offsets that fit the workgroup's LDS
    constexpr int kRowsHeld = 32;      // rows of a workgroup
    constexpr int kMostRows = 0xffffff * kRowsHeld; // a launch has fewer than 2^32 threads

    struct AppendArgs
    {
      const std::uint16_t *q;
      const std::uint16_t *k;
      const std::uint16_t *v;
      std::uint16_t *q_out;
      std::uint16_t *k_out;
      std::uint16_t *v_out;
      long long q_stride;
      long long k_stride;
      long long v_stride;
      const unsigned long long *pages;
      const std::uint8_t *tiers;
      const int *lengths;
      const int *offsets;
      int batch;
      int max_pages;
      int page_tokens;
      int rows;
      int heads;
      int kv_heads;
      int head_dim;
      int rotary;
      const float *table;
      int table_positions;
      int rows_block;
    };

    struct HeldSequences
    {
      const unsigned long long *pages[kAppendHeld];
      int page_count[kAppendHeld];
      int end[kAppendHeld]; // one past the sequence's last row
      int length[kAppendHeld];
    };
    struct NoneHeld
    {
    };

    // Where a row goes.
    struct RowPlace
    {
      std::uint16_t *page_row; // its keys' row in its page, or null
      int position;            // of its angles, within the table
      int live;                // a sequence's row
    };

    // The number of leading entries of offsets[0 .. n) that are at most `row`
    // (entries do not decrease).
    template <typename F>
    __device__ inline int entries_up_to(const F &offsets, int n, int row)
    {
      int lo = 0, hi = n;
      while (lo < hi)
      {
        const int mid = (lo + hi) >> 1;
        if (offsets(mid) <= row)
        {
          lo = mid + 1;
        }
        else
        {
          hi = mid;
        }
      }
      return lo;
    }

    template <bool kWide>
    struct Run; // N channels of a row
    template <>
    struct Run<true>
    {
      static constexpr int N = 8;
      u32x4 x;
      __device__ void load(const std::uint16_t *at) { x = *reinterpret_cast<const u32x4 *>(at); }
      __device__ void store(std::uint16_t *at) const { *reinterpret_cast<u32x4 *>(at) = x; }
      __device__ std::uint16_t get(int i) const
      {
        return static_cast<std::uint16_t>(x[i / 2] >> (16 * (i % 2)));
      }
      __device__ void set(int i, std::uint16_t v)
      {
        x[i / 2] = i % 2 == 0 ? (x[i / 2] & 0xFFFF0000u) | v
                              : (x[i / 2] & 0xFFFFu) | (static_cast<unsigned>(v) << 16);
      }
    };
    template <>
    struct Run<false>
    {
      static constexpr int N = 1;
      std::uint16_t x;
      __device__ void load(const std::uint16_t *at) { x = *at; }
      __device__ void store(std::uint16_t *at) const { *at = x; }
      __device__ std::uint16_t get(int) const { return x; }
      __device__ void set(int, std::uint16_t v) { x = v; }
    };

    // kWide: a thread takes 2 x 8 channels, where rows and the rotated part are
    // whole 16-byte runs; else 2 x 1.
    template <bool kWide, bool kInterleaved, typename Held>
    __global__ void __launch_bounds__(kThreads) append_kernel(AppendArgs a, Held held)
    {
      constexpr bool kHeld = std::is_same_v<Held, HeldSequences>;
      constexpr int N = Run<kWide>::N;
      __shared__ int s_offsets[kHeld ? 1 : kOffsetsHeld + 1];
      __shared__ RowPlace s_rows[kRowsHeld];
      const int first = blockIdx.x * a.rows_block;
      const int count = min(a.rows_block, a.rows - first);
      if constexpr (!kHeld)
      {
        if (a.offsets != nullptr && a.batch <= kOffsetsHeld)
        {
          for (int i = threadIdx.x; i <= a.batch; i += kThreads)
          {
            s_offsets[i] = a.offsets[i];
          }
          __syncthreads();
        }
      }
      if (static_cast<int>(threadIdx.x) < count)
      {
        const int row = first + threadIdx.x;
        RowPlace place{nullptr, 0, 0};
        long long position = -1;
        const unsigned long long *pages = nullptr;
        const std::uint8_t *tiers = nullptr;
        int page_count = 0;
        if constexpr (kHeld)
        {
          const int s = entries_up_to([&](int i) { return held.end[i]; }, a.batch, row);
          if (s < a.batch)
          {
            place.live = 1;
            position = held.length[s] - (held.end[s] - row);
            pages = held.pages[s];
            page_count = held.page_count[s];
          }
        }
        else
        {
          int s = row, end = row + 1;
          place.live = 1;
          if (a.offsets != nullptr)
          {
            const bool near = a.batch <= kOffsetsHeld;
            s = (near ? entries_up_to([&](int i) { return s_offsets[i]; }, a.batch, row)
                      : entries_up_to([&](int i) { return a.offsets[i]; }, a.batch, row)) - 1;
            if (s >= 0)
            {
              end = near ? s_offsets[s + 1] : a.offsets[s + 1];
            }
            place.live = s >= 0 && row < end;
          }
          if (place.live)
          {
            position = static_cast<long long>(a.lengths[s]) - (static_cast<long long>(end) - row);
            page_count = a.max_pages;
            pages = a.pages + static_cast<std::size_t>(s) * a.max_pages;
            tiers = a.tiers + static_cast<std::size_t>(s) * a.max_pages;
          }
        }
        if (pages != nullptr && position >= 0 && position / a.page_tokens < page_count)
        {
          const int page = static_cast<int>(position / a.page_tokens);
          const unsigned long long at = pages[page];
          if ((tiers == nullptr || tiers[page] == kFP16) && at != 0)
          {
            place.page_row = reinterpret_cast<std::uint16_t *>(at) +
                             static_cast<std::size_t>(position % a.page_tokens) * a.kv_heads *
                                 a.head_dim;
          }
        }
        place.position = static_cast<int>(
            max(0ll, min(position, static_cast<long long>(a.table_positions) - 1)));
        s_rows[threadIdx.x] = place;
      }
      __syncthreads();

      const int per = a.head_dim / (2 * N);      // threads a head
      const int turning = a.rotary / (2 * N);    // of them with pairs that turn
      const int units = (a.heads + 2 * a.kv_heads) * per;
      const int width = a.kv_heads * a.head_dim;
      for (int i = threadIdx.x; i < count * units; i += kThreads)
      {
        const int r = i / units, u = i % units;
        const RowPlace place = s_rows[r];
        if (!place.live)
        {
          continue;
        }
        const std::size_t row = static_cast<std::size_t>(first) + r;
        int head = u / per;
        const int unit = u % per;
        const bool is_q = head < a.heads;
        const bool is_v = head >= a.heads + a.kv_heads;
        head -= is_q ? 0 : is_v ? a.heads + a.kv_heads : a.heads;
        const std::uint16_t *from =
            (is_q ? a.q + row * a.q_stride : is_v ? a.v + row * a.v_stride : a.k + row * a.k_stride) +
            static_cast<std::size_t>(head) * a.head_dim;
        const bool turns = !is_v && unit < turning;
        // The two runs' channels.
        int at0 = 2 * N * unit, at1 = at0 + N;
        if (!kInterleaved && turns)
        {
          at0 = N * unit;
          at1 = at0 + a.rotary / 2;
        }
        Run<kWide> x0, x1;
        x0.load(from + at0);
        x1.load(from + at1);
        if (turns)
        {
          const float2 *cs = reinterpret_cast<const float2 *>(a.table) +
                             static_cast<std::size_t>(place.position) * (a.rotary / 2) + N * unit;
          float2 angle[N];
          if constexpr (kWide)
          {
#pragma unroll
            for (int e = 0; e < N; e += 2)
            {
              const float4 two = *reinterpret_cast<const float4 *>(cs + e);
              angle[e] = make_float2(two.x, two.y);
              angle[e + 1] = make_float2(two.z, two.w);
            }
          }
          else
          {
            angle[0] = cs[0];
          }
          Run<kWide> y0 = x0, y1 = x1;
#pragma unroll
          for (int e = 0; e < N; ++e)
          {
            std::uint16_t lo, hi;
            if (!kInterleaved || N == 1)
            {
              rope_pair(h2f(x0.get(e)), h2f(x1.get(e)), angle[e].x, angle[e].y, lo, hi);
              y0.set(e, lo);
              y1.set(e, hi);
            }
            else
            {
              const int c = 2 * e % N;
              const Run<kWide> &x = 2 * e < N ? x0 : x1;
              rope_pair(h2f(x.get(c)), h2f(x.get(c + 1)), angle[e].x, angle[e].y, lo, hi);
              Run<kWide> &y = 2 * e < N ? y0 : y1;
              y.set(c, lo);
              y.set(c + 1, hi);
            }
          }
          x0 = y0;
          x1 = y1;
        }
        const std::size_t in_row = static_cast<std::size_t>(head) * a.head_dim;
        if (is_q)
        {
          std::uint16_t *to = a.q_out + row * a.heads * a.head_dim + in_row;
          x0.store(to + at0);
          x1.store(to + at1);
          continue;
        }
        std::uint16_t *flat = is_v ? a.v_out : a.k_out;
        if (flat != nullptr)
        {
          std::uint16_t *to = flat + row * width + in_row;
          x0.store(to + at0);
          x1.store(to + at1);
        }
        if (place.page_row != nullptr)
        {
          std::uint16_t *to = place.page_row + in_row +
                              (is_v ? static_cast<std::size_t>(a.page_tokens) * width : 0);
          x0.store(to + at0);
          x1.store(to + at1);
        }
      }
    }

    __global__ void __launch_bounds__(kThreads)
        rope_frequencies_kernel(float *__restrict__ table, const double *__restrict__ frequencies,
                                int pairs, double magnitude, std::size_t count)
    {
      for (std::size_t i = static_cast<std::size_t>(blockIdx.x) * kThreads + threadIdx.x; i < count;
           i += static_cast<std::size_t>(gridDim.x) * kThreads)
      {
        double s, c;
        sincos(static_cast<double>(i / pairs) * frequencies[i % pairs], &s, &c);
        table[2 * i] = static_cast<float>(c * magnitude);
        table[2 * i + 1] = static_cast<float>(s * magnitude);
      }
    }

    bool aligned(const void *p) { return reinterpret_cast<std::uintptr_t>(p) % 16 == 0; }

    template <bool kWide, bool kInterleaved>
    void launch_as(AppendArgs a, const AppendSequence *sequences, hipStream_t stream)
    {
      // Rows a workgroup: one, or as many as its threads hold, since a row is a
      // chain of trips (9,001 rows of 32 + 2 x 8 heads of 64 take 29.1 us so, 30.4
      // by three rows, 32.8 by eight, 36.8 by 16); more past 16,384 workgroups.
      const int units = (a.heads + 2 * a.kv_heads) * (a.head_dim / (kWide ? 16 : 2));
      const int whole = std::max(1, kThreads / units);
      a.rows_block = std::min(kRowsHeld, std::max(whole, (a.rows + 16383) / 16384));
      const auto blocks = [&] {
        return static_cast<unsigned>((a.rows + a.rows_block - 1) / a.rows_block);
      };
      if (sequences == nullptr)
      {
        append_kernel<kWide, kInterleaved, NoneHeld><<<blocks(), kThreads, 0, stream>>>(a, NoneHeld{});
        hip_check(hipGetLastError(), "append_kernel");
        return;
      }
      const AppendArgs all = a;
      const int width = a.kv_heads * a.head_dim;
      std::size_t row0 = 0;
      for (int s0 = 0; s0 < all.batch; s0 += kAppendHeld)
      {
        HeldSequences held{};
        int rows = 0;
        a.batch = std::min(kAppendHeld, all.batch - s0);
        for (int i = 0; i < a.batch; ++i)
        {
          const AppendSequence &s = sequences[s0 + i];
          rows += s.rows;
          held.pages[i] = s.pages;
          held.page_count[i] = s.page_count;
          held.end[i] = rows;
          held.length[i] = s.start + s.rows;
        }
        if (rows == 0)
        {
          continue;
        }
        a.rows = rows;
        a.q = all.q + row0 * all.q_stride;
        a.k = all.k + row0 * all.k_stride;
        a.v = all.v + row0 * all.v_stride;
        a.q_out = all.q_out + row0 * all.heads * all.head_dim;
        a.k_out = all.k_out != nullptr ? all.k_out + row0 * width : nullptr;
        a.v_out = all.v_out != nullptr ? all.v_out + row0 * width : nullptr;
        append_kernel<kWide, kInterleaved, HeldSequences><<<blocks(), kThreads, 0, stream>>>(a, held);
        hip_check(hipGetLastError(), "append_kernel");
        row0 += rows;
      }
    }

    struct Strides
    {
      long long q, k, v;
    };
    Strides strides_of(const AppendRows &t)
    {
      const long long width = static_cast<long long>(t.kv_heads) * t.head_dim;
      const long long q_width = static_cast<long long>(t.heads) * t.head_dim;
      return {t.q_stride > 0 ? t.q_stride : q_width, t.k_stride > 0 ? t.k_stride : width,
              t.v_stride > 0 ? t.v_stride : width};
    }
  } // namespace

  void check_append(const AppendRows &t)
  {
    if (t.batch < 0 || t.max_pages < 0 || t.rows < 0)
    {
      throw InvalidArgument("batch, max_pages and rows must not be negative, got " +
                            std::to_string(t.batch) + ", " + std::to_string(t.max_pages) + " and " +
                            std::to_string(t.rows));
    }
    if (t.rows > kMostRows)
    {
      throw InvalidArgument("at most " + std::to_string(kMostRows) + " rows are appended at once, got " +
                            std::to_string(t.rows));
    }
    if (t.heads <= 0 || t.kv_heads <= 0 || t.head_dim <= 0 || t.head_dim % 2 != 0)
    {
      throw InvalidArgument("appended rows have query and KV heads of an even head_dim, got " +
                            std::to_string(t.heads) + ", " + std::to_string(t.kv_heads) + " and " +
                            std::to_string(t.head_dim));
    }
    if ((static_cast<long long>(t.heads) + 2ll * t.kv_heads) * t.head_dim > 0x3ffffff)
    {
      throw InvalidArgument("appended rows have at most 67108863 channels of queries, keys and "
                            "values; got " + std::to_string(t.heads) + " + 2 x " +
                            std::to_string(t.kv_heads) + " heads of " + std::to_string(t.head_dim));
    }
    if (t.rotary < 0 || t.rotary > t.head_dim || t.rotary % 2 != 0)
    {
      throw InvalidArgument("the RoPE table turns " + std::to_string(t.rotary) +
                            " channels of a head; appended heads have " +
                            std::to_string(t.head_dim));
    }
    const Strides st = strides_of(t);
    const long long width = static_cast<long long>(t.kv_heads) * t.head_dim;
    const long long q_width = static_cast<long long>(t.heads) * t.head_dim;
    if (t.q_stride < 0 || t.k_stride < 0 || t.v_stride < 0 || st.q < q_width || st.k < width ||
        st.v < width)
    {
      throw InvalidArgument("appended rows' strides are of a token's " + std::to_string(q_width) +
                            " query and " + std::to_string(width) +
                            " key and value elements at least (0: those); got " +
                            std::to_string(t.q_stride) + ", " + std::to_string(t.k_stride) +
                            " and " + std::to_string(t.v_stride));
    }
    if (t.rows == 0 || t.batch == 0)
    {
      return;
    }
    if (t.q == nullptr || t.k == nullptr || t.v == nullptr || t.q_out == nullptr)
    {
      throw InvalidArgument("appended rows need q, k, v and q_out");
    }
    if (t.held == nullptr)
    {
      if (t.lengths == nullptr || (t.max_pages > 0 && (t.pages == nullptr || t.tiers == nullptr)))
      {
        throw InvalidArgument("appended rows need the sequences' pages, tiers and lengths");
      }
      if (t.offsets == nullptr && t.rows != t.batch)
      {
        throw InvalidArgument("without offsets every sequence has one row; got " +
                              std::to_string(t.rows) + " rows of " + std::to_string(t.batch) +
                              " sequences");
      }
      const long long positions = static_cast<long long>(t.max_pages) * t.page_tokens;
      if (t.rotary > 0 && t.table_positions < positions)
      {
        throw InvalidArgument("the RoPE table covers " + std::to_string(t.table_positions) +
                              " positions; the page tables hold " + std::to_string(positions));
      }
    }
    if (t.rotary > 0 && (t.table == nullptr || t.table_positions <= 0))
    {
      throw InvalidArgument("the RoPE table covers no position");
    }
    const auto rows_of = [&](const void *at, long long wide, long long stride) {
      return Extent{at, 2 * static_cast<std::size_t>(wide), static_cast<std::size_t>(t.rows),
                    2 * static_cast<std::size_t>(stride)};
    };
    const std::size_t rows = static_cast<std::size_t>(t.rows), batch = static_cast<std::size_t>(t.batch);
    const std::size_t table = batch * static_cast<std::size_t>(t.max_pages);
    const std::size_t q_bytes = 2 * rows * q_width, kv_bytes = 2 * rows * width;
    const Extent outs[] = {{t.q_out, q_bytes}, {t.k_out, kv_bytes}, {t.v_out, kv_bytes}};
    const Extent reads[] = {
        rows_of(t.q, q_width, st.q), rows_of(t.k, width, st.k), rows_of(t.v, width, st.v),
        {t.pages, 8 * table}, {t.tiers, table}, {t.lengths, 4 * batch},
        {t.offsets, 4 * (batch + 1)},
        {t.table, 4 * static_cast<std::size_t>(t.table_positions) * static_cast<std::size_t>(t.rotary)}};
    for (int i = 0; i < 3; ++i)
    {
      for (const Extent &read : reads)
      {
        if (overlaps(outs[i], read))
        {
          throw InvalidArgument("appending rows cannot write over what it reads");
        }
      }
      for (int j = 0; j < i; ++j)
      {
        if (overlaps(outs[i], outs[j]))
        {
          throw InvalidArgument("appending rows cannot write q_out, k_out and v_out over one another");
        }
      }
    }
  }

  void launch_append(const AppendRows &t, hipStream_t stream)
  {
    check_append(t);
    if (t.rows == 0 || t.batch == 0)
    {
      return;
    }
    const Strides st = strides_of(t);
    AppendArgs a{};
    a.q = static_cast<const std::uint16_t *>(t.q);
    a.k = static_cast<const std::uint16_t *>(t.k);
    a.v = static_cast<const std::uint16_t *>(t.v);
    a.q_out = static_cast<std::uint16_t *>(t.q_out);
    a.k_out = static_cast<std::uint16_t *>(t.k_out);
    a.v_out = static_cast<std::uint16_t *>(t.v_out);
    a.q_stride = st.q;
    a.k_stride = st.k;
    a.v_stride = st.v;
    a.pages = t.pages;
    a.tiers = t.tiers;
    a.lengths = t.lengths;
    a.offsets = t.offsets;
    a.batch = t.batch;
    a.max_pages = t.max_pages;
    a.page_tokens = t.page_tokens;
    a.rows = t.rows;
    a.heads = t.heads;
    a.kv_heads = t.kv_heads;
    a.head_dim = t.head_dim;
    a.rotary = t.rotary;
    a.table = t.table;
    a.table_positions = t.table_positions;
    // (Pages are 16-byte aligned, as the allocator's slots are.)
    const bool wide = t.head_dim % 16 == 0 && t.rotary % 16 == 0 &&
                      (st.q | st.k | st.v) % 8 == 0 && aligned(t.q) && aligned(t.k) &&
                      aligned(t.v) && aligned(t.q_out) && aligned(t.k_out) && aligned(t.v_out);
    if (wide)
    {
      t.interleaved ? launch_as<true, true>(a, t.held, stream)
                    : launch_as<true, false>(a, t.held, stream);
    }
    else
    {
      t.interleaved ? launch_as<false, true>(a, t.held, stream)
                    : launch_as<false, false>(a, t.held, stream);
    }
  }

  void launch_rope_frequencies(float *table, int positions, const double *frequencies, int pairs,
                               double magnitude, hipStream_t stream)
  {
    const std::size_t count = static_cast<std::size_t>(positions) * pairs;
    if (count == 0)
    {
      return;
    }
    const unsigned blocks = static_cast<unsigned>(std::min<std::size_t>((count + kThreads - 1) / kThreads, 4096));
    rope_frequencies_kernel<<<blocks, kThreads, 0, stream>>>(table, frequencies, pairs, magnitude, count);
    hip_check(hipGetLastError(), "rope_frequencies_kernel");
  }

} // namespace mi
