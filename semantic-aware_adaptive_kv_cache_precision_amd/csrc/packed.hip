// Causal attention of several prompts in one run of rows: queries
// [offsets_q[s], offsets_q[s + 1]) are the last positions of the keys
// [offsets_k[s], offsets_k[s + 1]) of their sequence. Query i of m, of e keys,
// sees the first e - m + i + 1 of them; out = softmax(q . k / sqrt(hd)) v.
//
// Tiles are cut from the run of (query, head of the group) rows, whatever the
// sequences' lengths: a row sees the keys [lo, hi] of the run of keys, and both
// ends only rise along the run, so that a tile's keys are one range, from its
// first row's lo to its last row's hi, and a short sequence costs a share of a
// tile. Which sequence a row is of is found by a search of the offsets, held in
// LDS before the first keys are.
//
// A workgroup takes one KV head and consecutive rows, its waves 32 of them each;
// the keys of a step pass through LDS, double buffered, copied there directly
// from memory; scores and output as attention_tiles.hpp has them, P rounded to
// fp16 once (half a step is 2^-11 of a weight, as much as the output's own
// rounding; the sums are of the rounded weights) against a reference that is
// moved up only when a score passes it by 2^kRise: P is at most
// 2^(kRise + kProb) = 2^14, and keeps its 11 bits down to 2^-22 of the reference.
//
// With few rows the range of keys is split over workgroups, whose parts a
// second launch joins.
#include "attention_tiles.hpp"
#include "ragged.hpp"

#include <algorithm>
#include <climits>
#include <cmath>
#include <string>
#include <type_traits>

namespace mi
{
  namespace
  {
    using namespace attention_tiles;

    constexpr int kMaxSplits = 256;
    constexpr int kOffsetsHeld = 4096; // offsets of each kind that LDS holds

    struct PackedArgs
    {
      const std::uint16_t *q;
      const std::uint16_t *k;
      const std::uint16_t *v;
      std::uint16_t *out;
      long long q_stride; // elements between tokens
      long long k_stride;
      long long v_stride;
      const int *offsets_q;
      const int *offsets_k;
      int batch;
      int rows_q;
      int rows_k;
      int heads;
      int group;
      int splits;
      float scale;    // log2 e / sqrt(hd)
      float *part_ml; // splits > 1: [split][row] maximum and sum (row = query * heads + head),
      float *part_o;  // and hd outputs
    };

    // The keys [lo, hi] that a query sees, none where hi is lo - 1; and whether
    // it is a sequence's.
    struct Seen
    {
      int lo;
      int hi;
      bool live;
    };
    template <typename Q, typename K>
    __device__ inline Seen seen_by(int query, int batch, int rows_k, Q &&at_q, K &&at_k)
    {
      // The last sequence that begins at or before the query.
      int from = 0, to = batch + 1;
      while (from < to)
      {
        const int mid = (from + to) >> 1;
        if (at_q(mid) <= query)
        {
          from = mid + 1;
        }
        else
        {
          to = mid;
        }
      }
      const int s = from - 1;
      if (s < 0 || s >= batch)
      {
        return {0, -1, false};
      }
      // (In 64 bits, and held within the keys: offsets may be anything.)
      const long long begin = min(max(at_k(s), 0), rows_k), end = min(max(at_k(s + 1), 0), rows_k);
      const long long last = end - 1 - (static_cast<long long>(at_q(s + 1)) - 1 - query);
      return {static_cast<int>(begin), static_cast<int>(max(begin - 1, min(last, end - 1))), true};
    }

    __device__ inline int wave_min(int v)
    {
#pragma unroll
      for (int offset = 1; offset < 64; offset *= 2)
      {
        v = min(v, __shfl_xor(v, offset));
      }
      return __builtin_amdgcn_readfirstlane(v);
    }
    __device__ inline int wave_max(int v) { return -wave_min(-v); }

    // Waves a SIMD that a form's registers are held to: four at head_dim 64
    // (128 registers), two at 128 (256); few rows leave a wave alone anyway.
    template <int HD, int kTiles>
    constexpr int kWavesASimd = kTiles == 1 ? 1 : HD == 64 ? 4 : 2;

    template <int HD, int kTiles, int kWays, int kKeys>
    __global__ void __launch_bounds__(64 * kTiles * kWays, (kWavesASimd<HD, kTiles>))
        packed_kernel(PackedArgs a)
    {
      constexpr int NW = kTiles * kWays;
      constexpr int kPieces = HD / 8;    // 16-byte pieces a row
      constexpr int kTile = kKeys * HD;  // halves of a step's keys
      constexpr int kStage = 2 * kTile;  // keys, then values
      constexpr int kRows = 32 * kTiles; // rows a workgroup
      constexpr int kWayKeys = kKeys / kWays;
      constexpr int N = kWayKeys / 32;
      extern __shared__ __align__(16) std::uint16_t stages[]; // two of kStage
      __shared__ int s_lo[NW], s_hi[NW];

      const int lane = threadIdx.x & 63;
      const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
      const int way = wave / kTiles;
      const int n = lane & 31;
      const int half = lane >> 5;
      const int kvh = blockIdx.y;
      const int split = blockIdx.z;
      const int G = a.group;
      const long long all_rows = static_cast<long long>(a.rows_q) * G;
      // The last rows of the run go first: of one prompt, those with most keys.
      const long long row0 = static_cast<long long>(gridDim.x - 1 - blockIdx.x) * kRows;

      // The lane's row and what it sees.
      const long long row = row0 + 32 * (wave % kTiles) + n;
      const bool there = row < all_rows;
      const int query = there ? static_cast<int>(row / G) : 0;
      const int head = kvh * G + (there ? static_cast<int>(row % G) : 0);
      const std::size_t row_at = static_cast<std::size_t>(query) * a.heads + head;
      half8 q[HD / 16];
      const std::uint16_t *q_row = a.q + query * a.q_stride + head * HD + 8 * half;
#pragma unroll
      for (int c = 0; c < HD / 16; ++c)
      {
        q[c] = as_half8(*reinterpret_cast<const u32x4 *>(q_row + 16 * c));
      }
      Seen seen;
      if (a.batch <= kOffsetsHeld)
      {
        int *held_q = reinterpret_cast<int *>(stages), *held_k = held_q + kOffsetsHeld + 1;
        for (int i = threadIdx.x; i <= a.batch; i += 64 * NW)
        {
          held_q[i] = a.offsets_q[i];
          held_k[i] = a.offsets_k[i];
        }
        __syncthreads();
        seen = seen_by(query, a.batch, a.rows_k, [&](int i) { return held_q[i]; },
                       [&](int i) { return held_k[i]; });
      }
      else
      {
        seen = seen_by(query, a.batch, a.rows_k, [&](int i) { return a.offsets_q[i]; },
                       [&](int i) { return a.offsets_k[i]; });
      }
      const bool valid = there && seen.live;
      const int lo = valid ? seen.lo : 0, hi = valid ? seen.hi : -1;
      // The wave's keys, and those that every row of it sees.
      const int wave_lo = wave_min(valid && hi >= lo ? lo : INT_MAX);
      const int wave_hi = wave_max(hi);
      const int all_lo = wave_max(valid ? lo : 0);
      const int all_hi = wave_min(valid ? hi : INT_MAX);
      if (lane == 0)
      {
        s_lo[wave] = wave_lo;
        s_hi[wave] = wave_hi;
      }
      __syncthreads(); // (the offsets are read too)
      int first = INT_MAX, last = -1;
#pragma unroll
      for (int w = 0; w < NW; ++w)
      {
        first = min(first, s_lo[w]);
        last = max(last, s_hi[w]);
      }
      first = __builtin_amdgcn_readfirstlane(first);
      last = __builtin_amdgcn_readfirstlane(last);
      const int steps = last >= first ? (last - first) / kKeys + 1 : 0;
      const int per = (steps + a.splits - 1) / a.splits;
      const int begin = min(split * per, steps);
      const int end = min(begin + per, steps);

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
        const int key0 = first + step * kKeys;
        std::uint16_t *stage = stages + buf * kStage;
#pragma unroll
        for (int i = 0; i < kTile / 8 / (64 * NW); ++i)
        {
          const int place = (i * NW + wave) * 64 + lane;
          const int t = place / kPieces;
          const int c = (place % kPieces) ^ swizzle<HD>(t);
          const long long key = min(key0 + t, a.rows_k - 1);
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
        const int key0 = first + step * kKeys + way * kWayKeys;
        if (key0 > wave_hi || key0 + kWayKeys - 1 < wave_lo)
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
        const bool edge = key0 + kWayKeys - 1 > all_hi || key0 < all_lo;
        if (edge)
        {
#pragma unroll
          for (int j = 0; j < N; ++j)
          {
#pragma unroll
            for (int i = 0; i < 16; ++i)
            {
              const int key = key0 + 32 * j + 8 * (i / 4) + 4 * half + i % 4;
              s[j][i] = key >= lo && key <= hi ? s[j][i] : -INFINITY;
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
          for (int key = key0; key < min(key0 + kWayKeys, a.rows_k); ++key)
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
                run.o[d][i] += key >= lo && key <= hi && !is_finite(v) ? h2f(v) : 0.0f;
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
        // (Of no keys the sum is 0, and the output.)
        const float inv = sum > 0.0f || sum != sum ? kProbUnscale / sum : 0.0f;
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
      const std::size_t at = static_cast<std::size_t>(split) * a.rows_q * a.heads + row_at;
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

    // The parts of a (query, head) row joined by a workgroup, its groups of
    // lanes each taking some.
    template <int HD>
    __global__ void __launch_bounds__(256) packed_join_kernel(PackedArgs a, std::size_t rows)
    {
      constexpr int kLanes = HD / 4, kGroups = 256 / kLanes;
      __shared__ f32x2 s_ml[kGroups];
      __shared__ __align__(16) float s_o[kGroups][HD];
      const std::size_t row = blockIdx.x;
      const long long query = row / a.heads;
      if (query < a.offsets_q[0] || query >= a.offsets_q[a.batch])
      {
        return; // of no sequence
      }
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
      out = sum > 0.0f || sum != sum ? out / sum : 0.0f;
      a.out[row * HD + threadIdx.x] = __builtin_bit_cast(std::uint16_t, static_cast<_Float16>(out));
    }

    // A launch's form: the row tiles of a workgroup, the waves that share a
    // tile's keys, and the keys a step.
    template <int kTiles_, int kWays_, int kKeys_>
    struct Form
    {
      static constexpr int tiles = kTiles_, ways = kWays_, keys = kKeys_, rows = 32 * kTiles_;
    };
    using Few = Form<1, 4, 128>;
    using Many64 = Form<4, 2, 128>;
    using Many128 = Form<4, 1, 64>;

    // How a launch is cut. The lengths are on the device: what is known of them
    // here is how many rows and keys there are.
    struct Cut
    {
      bool few;
      int blocks; // workgroups over the rows, a KV head
      int splits; // workgroups over a row's keys
    };

    Cut cut_of(const PackedAttention &t, bool may_split)
    {
      const int group = t.heads / t.kv_heads;
      const long long rows = static_cast<long long>(t.rows_q) * group;
      // About the keys that a row sees: those of a sequence, a causal half of
      // its own new ones.
      const long long batch = std::max(1, t.batch);
      const long long span = (t.rows_k - t.rows_q / 2 + batch - 1) / batch;
      Cut c{};
      const long long few = (rows + Few::rows - 1) / Few::rows * t.kv_heads;
      c.few = few <= (span <= 1024 && t.head_dim == 64 ? 512 : 256);
      const int tile = c.few ? Few::rows : t.head_dim == 64 ? Many64::rows : Many128::rows;
      const int keys = c.few ? Few::keys : t.head_dim == 64 ? Many64::keys : Many128::keys;
      c.blocks = static_cast<int>((rows + tile - 1) / tile);
      c.splits = 1;
      if (may_split && c.blocks > 0)
      {
        const long long steps = (2 * span + keys - 1) / keys;
        const long long groups = static_cast<long long>(c.blocks) * t.kv_heads;
        const bool two = !c.few && t.head_dim == 128;
        const long long fill = (two ? 512 : 256) / groups;
        c.splits = static_cast<int>(std::max<long long>(
            1, std::min<long long>({fill, steps < 4 ? 1 : steps / 2, two ? 4 : kMaxSplits})));
      }
      return c;
    }

    void check_packed(const PackedAttention &t)
    {
      if (t.batch < 0 || t.rows_q < 0 || t.rows_k < 0)
      {
        throw InvalidArgument("batch, rows_q and rows_k must not be negative, got " +
                              std::to_string(t.batch) + ", " + std::to_string(t.rows_q) + " and " +
                              std::to_string(t.rows_k));
      }
      constexpr int kMost = 0x7fffff00; // a step's last key stays an index
      if (t.rows_q > kMost || t.rows_k > kMost || t.batch > kMost)
      {
        throw InvalidArgument("batch, rows_q and rows_k exceed packed attention's " +
                              std::to_string(kMost));
      }
      if (t.head_dim != 64 && t.head_dim != 128)
      {
        throw InvalidArgument("packed attention takes head_dim 64 or 128, got " +
                              std::to_string(t.head_dim));
      }
      if (t.kv_heads <= 0 || t.heads <= 0 || t.heads % t.kv_heads != 0 || t.kv_heads > 65535)
      {
        throw InvalidArgument("packed attention takes a whole number of query heads a KV head, got " +
                              std::to_string(t.heads) + " and " + std::to_string(t.kv_heads));
      }
      // A head's offset in its token is 32 bits, and a launch's workgroups are.
      if (static_cast<long long>(t.heads) * t.head_dim > 0x7fffffff ||
          static_cast<long long>(t.rows_q) * (t.heads / t.kv_heads) > 0x7fffffffll * 32)
      {
        throw InvalidArgument("packed attention takes fewer than 2^31 query elements a token and "
                              "2^36 rows a KV head, got " + std::to_string(t.heads) + " heads of " +
                              std::to_string(t.head_dim));
      }
    }

    template <int HD, typename F>
    void launch(const PackedArgs &a, const Cut &c, int kv_heads, hipStream_t stream)
    {
      constexpr std::size_t lds =
          std::max({sizeof(std::uint16_t) * 2 * 2 * F::keys * HD,
                    sizeof(float) * (F::ways - 1) * F::tiles * (HD / 2 + 2) * 64,
                    sizeof(int) * 2 * (kOffsetsHeld + 1)});
      auto kernel = packed_kernel<HD, F::tiles, F::ways, F::keys>;
      if constexpr (lds > 63 * 1024)
      {
        hip_check(hipFuncSetAttribute(reinterpret_cast<const void *>(kernel),
                                      hipFuncAttributeMaxDynamicSharedMemorySize,
                                      static_cast<int>(lds)),
                  "hipFuncSetAttribute packed LDS");
      }
      kernel<<<dim3(c.blocks, kv_heads, c.splits), 64 * F::tiles * F::ways, lds, stream>>>(a);
      hip_check(hipGetLastError(), "packed_kernel");
    }

    template <int HD>
    void launch_any(const PackedArgs &a, const Cut &c, int kv_heads, hipStream_t stream)
    {
      if (c.few)
      {
        launch<HD, Few>(a, c, kv_heads, stream);
      }
      else
      {
        launch<HD, std::conditional_t<HD == 64, Many64, Many128>>(a, c, kv_heads, stream);
      }
      if (c.splits > 1)
      {
        const std::size_t rows = static_cast<std::size_t>(a.rows_q) * a.heads;
        packed_join_kernel<HD><<<static_cast<unsigned>(rows), 256, 0, stream>>>(a, rows);
        hip_check(hipGetLastError(), "packed_join_kernel");
      }
    }
  } // namespace

  std::size_t packed_attention_floats(const PackedAttention &t)
  {
    check_packed(t);
    if (t.rows_q == 0 || t.rows_k == 0)
    {
      return 0;
    }
    const Cut c = cut_of(t, true);
    return c.splits > 1 ? static_cast<std::size_t>(c.splits) * t.rows_q * t.heads * (t.head_dim + 2)
                        : 0;
  }

  void launch_packed_attention(const PackedAttention &t, hipStream_t stream)
  {
    check_packed(t);
    if (t.rows_q == 0 || t.batch == 0)
    {
      return;
    }
    if (t.rows_k == 0)
    {
      throw InvalidArgument("packed attention needs keys for its " + std::to_string(t.rows_q) +
                            " queries");
    }
    if (t.q == nullptr || t.k == nullptr || t.v == nullptr || t.out == nullptr ||
        t.offsets_q == nullptr)
    {
      throw InvalidArgument("packed attention needs q, k, v, out and offsets_q");
    }
    const long long width = static_cast<long long>(t.kv_heads) * t.head_dim;
    const long long q_width = static_cast<long long>(t.heads) * t.head_dim;
    const long long q_stride = t.q_stride > 0 ? t.q_stride : q_width;
    const long long k_stride = t.k_stride > 0 ? t.k_stride : width;
    const long long v_stride = t.v_stride > 0 ? t.v_stride : width;
    if (t.q_stride < 0 || t.k_stride < 0 || t.v_stride < 0 || q_stride < q_width ||
        k_stride < width || v_stride < width)
    {
      throw InvalidArgument("packed attention's strides are of a token's " +
                            std::to_string(q_width) + " query and " + std::to_string(width) +
                            " key and value elements at least (0: those); got " +
                            std::to_string(t.q_stride) + ", " + std::to_string(t.k_stride) +
                            " and " + std::to_string(t.v_stride));
    }
    const auto address = [](const void *p) { return reinterpret_cast<std::uintptr_t>(p); };
    if ((address(t.q) | address(t.k) | address(t.v) | address(t.out) | address(t.partials)) % 16 != 0 ||
        (q_stride | k_stride | v_stride) % 8 != 0 ||
        (address(t.offsets_q) | address(t.offsets_k)) % 4 != 0)
    {
      throw InvalidArgument("packed attention's rows and partials must be 16-byte aligned, its "
                            "offsets 4-byte");
    }
    const Cut c = cut_of(t, t.partials != nullptr);
    if (t.partials != nullptr && t.partials_floats < packed_attention_floats(t))
    {
      throw InvalidArgument("packed attention's partials need " +
                            std::to_string(packed_attention_floats(t)) + " floats; got " +
                            std::to_string(t.partials_floats));
    }
    const auto rows_of = [](const void *at, long long width, int tokens, long long stride) {
      return Extent{at, 2 * static_cast<std::size_t>(width), static_cast<std::size_t>(tokens),
                    2 * static_cast<std::size_t>(stride)};
    };
    const std::size_t offsets = 4 * (static_cast<std::size_t>(t.batch) + 1);
    const Extent out{t.out, 2 * static_cast<std::size_t>(t.rows_q) * q_width};
    const Extent parts{t.partials, t.partials != nullptr ? sizeof(float) * packed_attention_floats(t) : 0};
    for (const Extent &read :
         {rows_of(t.q, q_width, t.rows_q, q_stride), rows_of(t.k, width, t.rows_k, k_stride),
          rows_of(t.v, width, t.rows_k, v_stride), Extent{t.offsets_q, offsets},
          Extent{t.offsets_k, offsets}})
    {
      if (overlaps(out, read) || overlaps(parts, read))
      {
        throw InvalidArgument("packed attention cannot write over its queries, keys, values or offsets");
      }
    }
    if (overlaps(parts, out))
    {
      throw InvalidArgument("packed attention's partials lie over its output");
    }
    PackedArgs a{};
    a.q = static_cast<const std::uint16_t *>(t.q);
    a.k = static_cast<const std::uint16_t *>(t.k);
    a.v = static_cast<const std::uint16_t *>(t.v);
    a.out = static_cast<std::uint16_t *>(t.out);
    a.q_stride = q_stride;
    a.k_stride = k_stride;
    a.v_stride = v_stride;
    a.offsets_q = t.offsets_q;
    a.offsets_k = t.offsets_k != nullptr ? t.offsets_k : t.offsets_q;
    a.batch = t.batch;
    a.rows_q = t.rows_q;
    a.rows_k = t.rows_k;
    a.heads = t.heads;
    a.group = t.heads / t.kv_heads;
    a.splits = c.splits;
    a.scale = static_cast<float>(1.4426950408889634 / std::sqrt(static_cast<double>(t.head_dim)));
    if (c.splits > 1)
    {
      const std::size_t rows = static_cast<std::size_t>(t.rows_q) * t.heads;
      a.part_o = t.partials;
      a.part_ml = t.partials + rows * c.splits * t.head_dim;
    }
    t.head_dim == 64 ? launch_any<64>(a, c, t.kv_heads, stream)
                     : launch_any<128>(a, c, t.kv_heads, stream);
  }

} // namespace mi
