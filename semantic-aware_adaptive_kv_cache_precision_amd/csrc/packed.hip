// Causal attention of several prompts in one run of rows: queries
// [offsets_q[s], offsets_q[s + 1]) are the last positions of the keys
// [offsets_k[s], offsets_k[s + 1]) of their sequence. Query i of m, of e keys,
// sees the first e - m + i + 1 of them; out = softmax(q . k / sqrt(hd)) v.
//
// A sequence's rows (query by query, the heads of a KV head's group) are cut into
// tiles, and a workgroup takes a tile of one KV head. Which one, it finds from
// the offsets, which are on the device: tiles with most keys first, as long as
// the sequences are few enough to be ranked (a search for the length that as many
// tiles reach as there are workgroups before this one); else in their order.
//
// The waves of a workgroup take 32 rows each (at head_dim 64 two waves share the
// rows and take the keys in turn); the keys of a step pass through LDS, double
// buffered, copied there directly from memory; scores and output as
// attention_tiles.hpp has them, P rounded to fp16 once (half a step is 2^-11 of a weight, as much as the output's own
// rounding; the sums are of the rounded weights) against a reference that is
// moved up only when a score passes it by 2^kRise: P is at most
// 2^(kRise + kProb) = 2^14, and keeps its 11 bits down to 2^-22 of the reference.
//
// With few rows the range of keys is split over workgroups, whose parts a
// second launch joins.
//
// Bound by the matrix cores and the vector unit in turn, two waves to a SIMD at
// head_dim 128, four at 64: a prompt of 16K runs at 855 TFLOP/s at 128, some 800 at 64,
// where the exponentials and their sums are half of the time; a large product
// reaches 1,323. Ragged ones lose a quarter more to CUs that end early: eight
// prompts of 12K rows (12 heads of 128) 151 us, 870 TFLOP/s; new turns behind
// prefixes (32 heads of 64) 187 us, 650. Nine chats of 413 rows take 7.1 us, a
// launch and a chain of trips.
#include "attention_tiles.hpp"
#include "packed_copies.hpp"
#include "ragged.hpp"

#include <algorithm>
#include <cmath>
#include <string>
#include <type_traits>

namespace mi
{
  namespace
  {
    using namespace attention_tiles;

    constexpr int kMaxSplits = 256;
    constexpr int kFewSplits = 8; // that a lane joins by itself
    constexpr int kMfma = 0x8, kDsRead = 0x100; // instructions, to the scheduler
    constexpr int kOffsetsHeld = 4096; // offsets of each kind that LDS holds
    constexpr int kRanked = 256;       // sequences whose tiles are ranked by their keys
    constexpr int kCus = 256;

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
      int kv_heads;
      int group;
      int splits;
      int ranked;     // whether workgroups take tiles by their keys, and so many of
                      // the first are on the device together
      float scale;    // log2 e / sqrt(hd)
      float *part_ml; // splits > 1: [split][row] maximum and sum (row = query * heads + head),
      float *part_o;  // and hd outputs
    };

    // A wave's sum and extrema: within rows of 16 lanes, then over the rows
    // before, into the last lane. (Moves between registers: a search's steps
    // each wait for one, and through LDS they take five times as long.)
    template <typename F>
    __device__ inline int wave_fold(int v, int none, F &&f)
    {
      v = f(v, __builtin_amdgcn_update_dpp(none, v, 0x111, 0xF, 0xF, false)); // row_shr:1, 2, 4, 8
      v = f(v, __builtin_amdgcn_update_dpp(none, v, 0x112, 0xF, 0xF, false));
      v = f(v, __builtin_amdgcn_update_dpp(none, v, 0x114, 0xF, 0xF, false));
      v = f(v, __builtin_amdgcn_update_dpp(none, v, 0x118, 0xF, 0xF, false));
      v = f(v, __builtin_amdgcn_update_dpp(none, v, 0x142, 0xA, 0xF, false)); // row_bcast:15
      v = f(v, __builtin_amdgcn_update_dpp(none, v, 0x143, 0xC, 0xF, false)); // row_bcast:31
      return __builtin_amdgcn_readlane(v, 63);
    }
    __device__ inline int wave_sum(int v)
    {
      return wave_fold(v, 0, [](int x, int y) { return x + y; });
    }
    __device__ inline int wave_min(int v)
    {
      return wave_fold(v, 0x7fffffff, [](int x, int y) { return min(x, y); });
    }
    __device__ inline int wave_max(int v) { return -wave_min(-v); }

    // A sequence's rows and keys, whatever its offsets hold.
    struct Sequence
    {
      int q0, queries, k0, keys;
    };
    template <typename Q, typename K>
    __device__ inline Sequence sequence_of(const PackedArgs &a, int s, Q &&at_q, K &&at_k)
    {
      const int q0 = min(max(at_q(s), 0), a.rows_q), q1 = min(max(at_q(s + 1), 0), a.rows_q);
      const int k0 = min(max(at_k(s), 0), a.rows_k), k1 = min(max(at_k(s + 1), 0), a.rows_k);
      return {q0, max(q1 - q0, 0), k0, max(k1 - k0, 0)};
    }
    // The row tiles of a sequence, and how many of them (its last) see `keys`
    // keys at least.
    template <int kRows>
    __device__ inline int tiles_of(const Sequence &s, int G)
    {
      return static_cast<int>((static_cast<long long>(s.queries) * G + kRows - 1) / kRows);
    }
    template <int kRows>
    __device__ inline int tiles_that_see(const Sequence &s, int G, int keys)
    {
      // The first query that sees so many, and the tile that its last row is in
      // or that reaches it.
      const int query = keys - 1 - (s.keys - s.queries);
      const int tiles = tiles_of<kRows>(s, G);
      if (query <= 0 || keys <= 0)
      {
        return tiles;
      }
      return query >= s.queries
                 ? 0
                 : tiles - static_cast<int>(static_cast<long long>(query) * G / kRows);
    }

    // A workgroup's tile: its sequence, or none.
    struct Tile
    {
      int sequence;
      int tile;
    };
    // The index-th tile. Every wave finds it by itself.
    template <int kRows, typename Q, typename K>
    __device__ inline Tile tile_at(const PackedArgs &a, int index, Q &&at_q, K &&at_k)
    {
      const int lane = threadIdx.x & 63, G = a.group;
      int least = -1; // keys that the tile sees, if they are ranked by them
      if (a.ranked > 0)
      {
        Sequence mine[kRanked / 64];
        int all = 0, most = 0;
#pragma unroll
        for (int i = 0; i < kRanked / 64; ++i)
        {
          const int s = lane + 64 * i;
          mine[i] = s < a.batch ? sequence_of(a, s, at_q, at_k) : Sequence{0, 0, 0, 0};
          all += tiles_of<kRows>(mine[i], G);
          most = max(most, mine[i].keys);
        }
        if (index >= wave_sum(all))
        {
          return {-1, 0};
        }
        // The most keys that more than `index` tiles see: lo is, hi is not.
        int lo = 0, hi = wave_max(most) + 1;
        while (hi - lo > 1)
        {
          const int keys = lo + (hi - lo) / 2;
          int see = 0;
#pragma unroll
          for (int i = 0; i < kRanked / 64; ++i)
          {
            if (64 * i < a.batch)
            {
              see += tiles_that_see<kRows>(mine[i], G, keys);
            }
          }
          (wave_sum(see) > index ? lo : hi) = keys;
        }
        int more = 0;
#pragma unroll
        for (int i = 0; i < kRanked / 64; ++i)
        {
          if (64 * i < a.batch)
          {
            more += tiles_that_see<kRows>(mine[i], G, lo + 1);
          }
        }
        index -= wave_sum(more); // among those that see so many and no more
        least = lo;
      }
      for (int s0 = 0; s0 < a.batch; s0 += 64)
      {
        const int s = s0 + lane;
        const Sequence mine = s < a.batch ? sequence_of(a, s, at_q, at_k) : Sequence{0, 0, 0, 0};
        const int tiles = tiles_of<kRows>(mine, G);
        const int see = least < 0 ? tiles : tiles_that_see<kRows>(mine, G, least);
        const int count = least < 0 ? tiles : see - tiles_that_see<kRows>(mine, G, least + 1);
        int upto = count;
#pragma unroll
        for (int offset = 1; offset < 64; offset *= 2)
        {
          const int before = __shfl_up(upto, offset);
          upto = lane >= offset ? upto + before : upto;
        }
        const unsigned long long reached = __ballot(upto > index);
        if (reached != 0)
        {
          const int at = __ffsll(reached) - 1;
          const int tile = tiles - see + index - (upto - count);
          return {s0 + at, __builtin_amdgcn_readfirstlane(__shfl(tile, at))};
        }
        index -= __builtin_amdgcn_readfirstlane(__shfl(upto, 63));
      }
      return {-1, 0};
    }

    // An LDS address as an instruction's operand has it.
    __device__ inline unsigned lds_address(const void *p)
    {
      return static_cast<unsigned>(__builtin_amdgcn_readfirstlane(static_cast<int>(
          reinterpret_cast<std::uintptr_t>((lds_void)(const_cast<void *>(p))))));
    }
    // `count` + 1 rows of `width` halves, `step` bytes apart, for buffer loads.
    __device__ inline u32x4 rows_from(const std::uint16_t *at, int count, unsigned step, int width)
    {
      const auto address = reinterpret_cast<std::uintptr_t>(at);
      return u32x4{static_cast<unsigned>(address), static_cast<unsigned>(address >> 32) & 0xFFFFu,
                   packed_copies::rows_bytes(count, step, width), 0x00020000u};
    }
    // 16 bytes a lane from rows + at to the 1,024 bytes at LDS address `to`.
    __device__ inline void copy_to_lds(unsigned to, unsigned at, u32x4 rows)
    {
      asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                   :: "s"(to), "v"(at), "s"(rows)
                   : "memory", "m0");
    }

    // A barrier for what waves leave each other in LDS, copies in flight or not.
    __device__ inline void lds_barrier()
    {
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    }
    __device__ inline bool all_finite(half8 v)
    {
      const u32x4 bits = __builtin_bit_cast(u32x4, v);
      bool fine = true;
#pragma unroll
      for (int w = 0; w < 4; ++w)
      {
        fine = fine && is_finite(static_cast<std::uint16_t>(bits[w])) &&
               is_finite(static_cast<std::uint16_t>(bits[w] >> 16));
      }
      return fine;
    }

    // Waves a SIMD that a form's registers are held to: four at head_dim 64
    // (128 registers), two at 128 (256); few rows leave a wave alone anyway.
    template <int HD, int kTiles>
    constexpr int kWavesASimd = kTiles == 1 ? 1 : HD == 64 ? 4 : 2;

    template <int HD, int kTiles, int kWays, int kKeys>
    __global__ void __launch_bounds__(64 * kTiles * kWays, (kWavesASimd<HD, kTiles>))
        packed_kernel(PackedArgs a)
    {
      constexpr int NW = kTiles * kWays;
      constexpr int kPieces = packed_copies::pieces(HD);
      constexpr int kTile = kKeys * HD;  // halves of a step's keys
      constexpr int kStage = 2 * kTile;  // keys, then values
      constexpr int kRows = 32 * kTiles; // rows a workgroup
      constexpr int kWayKeys = kKeys / kWays;
      constexpr int N = kWayKeys / 32;
      extern __shared__ __align__(16) std::uint16_t stages[]; // two of kStage
      __shared__ int s_fine[NW];

      const int lane = threadIdx.x & 63;
      const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
      const int way = wave / kTiles;
      const int n = lane & 31;
      const int half = lane >> 5;
      // Of the workgroups on the device together, a CU's first, third .. come from
      // the most keys on, its second, fourth .. the other way: 256 sums that are
      // nearly alike (8 prompts of 12K rows: 1.11 of their mean at most, one way 1.35).
      int block = blockIdx.x;
      if ((block / kCus) % 2 == 1 && (block / kCus + 1) * kCus <= a.ranked)
      {
        block = (2 * (block / kCus) + 1) * kCus - 1 - block;
      }
      const int kvh = block % a.kv_heads, index = block / a.kv_heads;
      const int split = blockIdx.y;
      const int G = a.group;

      // The tile, and its sequence.
      Tile tile;
      Sequence of;
      if (a.batch <= kOffsetsHeld)
      {
        int *held_q = reinterpret_cast<int *>(stages), *held_k = held_q + kOffsetsHeld + 1;
        for (int i = threadIdx.x; i <= a.batch; i += 64 * NW)
        {
          held_q[i] = a.offsets_q[i];
          held_k[i] = a.offsets_k[i];
        }
        __syncthreads();
        const auto at_q = [&](int i) { return held_q[i]; };
        const auto at_k = [&](int i) { return held_k[i]; };
        tile = tile_at<kRows>(a, index, at_q, at_k);
        of = sequence_of(a, max(tile.sequence, 0), at_q, at_k);
        __syncthreads(); // the offsets are read
      }
      else
      {
        const auto at_q = [&](int i) { return a.offsets_q[i]; };
        const auto at_k = [&](int i) { return a.offsets_k[i]; };
        tile = tile_at<kRows>(a, index, at_q, at_k);
        of = sequence_of(a, max(tile.sequence, 0), at_q, at_k);
      }
      if (tile.sequence < 0)
      {
        return;
      }
      const int q0 = __builtin_amdgcn_readfirstlane(of.q0), first = __builtin_amdgcn_readfirstlane(of.k0);
      const int queries = __builtin_amdgcn_readfirstlane(of.queries);
      const int past = __builtin_amdgcn_readfirstlane(of.keys) - queries; // less than none: blind queries

      // The lane's row, and the last key it sees: one before the first, if none.
      const long long rows = static_cast<long long>(queries) * G;
      const long long tile_row = static_cast<long long>(tile.tile) * kRows;
      const long long wave_row = tile_row + 32 * (wave % kTiles);
      const long long row = wave_row + n;
      const bool valid = row < rows;
      const auto last_key = [&](long long r) {
        return first + max(-1, past + static_cast<int>(min(r, rows - 1) / G));
      };
      const int query = q0 + (valid ? static_cast<int>(row / G) : 0);
      const int head = kvh * G + (valid ? static_cast<int>(row % G) : 0);
      const int hi = last_key(row);
      const std::size_t row_at = static_cast<std::size_t>(query) * a.heads + head;
      half8 q[HD / 16];
      const std::uint16_t *q_row = a.q + query * a.q_stride + head * HD + 8 * half;
#pragma unroll
      for (int c = 0; c < HD / 16; ++c)
      {
        q[c] = as_half8(*reinterpret_cast<const u32x4 *>(q_row + 16 * c));
      }
      // The wave's last key, the last that all its rows see, and the workgroup's.
      const int wave_hi = wave_row < rows ? last_key(wave_row + 31) : -1;
      const int all_hi = last_key(wave_row);
      const int block_hi = last_key(tile_row);
      const int last = last_key(tile_row + kRows - 1);
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

      // A step's rows to LDS, 16 bytes a lane, asked for without the compiler's
      // knowledge, whose wait for them would come before the first transposing
      // read of the step before: buffer loads from the step's first row, with
      // zeros for what lies past the last key (packed_copies.hpp).
      constexpr int kCopies = packed_copies::copies(HD, NW, kKeys);
      constexpr int kCopyRows = packed_copies::rows_at_once(HD, NW);
      static_assert(kCopyRows % 16 == 0, "rows a copy apart have their pieces in the same places");
      const int copy_row = static_cast<int>(threadIdx.x) / kPieces;
      const int copy_piece = (static_cast<int>(threadIdx.x) % kPieces) ^ swizzle<HD>(copy_row);
      const unsigned k_step = 2u * static_cast<unsigned>(a.k_stride), v_step = 2u * static_cast<unsigned>(a.v_stride);
      const unsigned k_at = packed_copies::lane_at(copy_row, copy_piece, k_step);
      const unsigned v_at = packed_copies::lane_at(copy_row, copy_piece, v_step);
      const auto copy = [&](int step, int buf) {
        const int key0 = first + step * kKeys;
        const unsigned to = lds_address(stages + buf * kStage + wave * 512);
        const u32x4 k_rows = rows_from(a.k + key0 * a.k_stride + kvh * HD, a.rows_k - 1 - key0, k_step, HD);
        const u32x4 v_rows = rows_from(a.v + key0 * a.v_stride + kvh * HD, a.rows_k - 1 - key0, v_step, HD);
#pragma unroll
        for (int i = 0; i < kCopies; ++i)
        {
          copy_to_lds(to + 1024 * NW * i, packed_copies::copy_at(k_at, i, kCopyRows, k_step), k_rows);
          copy_to_lds(to + 2 * kTile + 1024 * NW * i,
                      packed_copies::copy_at(v_at, i, kCopyRows, v_step), v_rows);
        }
      };
      // (The queries are there before the loop: a wait for them inside it would
      // wait for the copies too.)
#pragma unroll
      for (int c = 0; c < HD / 16; ++c)
      {
        asm volatile("" : "+v"(q[c]));
      }
      if (begin < end)
      {
        copy(begin, 0);
      }
      // (Buffers in turn, as constants where registers allow: the places in them
      // are then offsets of the reads' instructions.)
      constexpr bool kInTurn = kTiles == 1 || HD == 128;
      const auto take = [&](auto buf, int step) {
        // This step's copies have landed, and every wave is done with the other
        // buffer.
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (step + 1 < end)
        {
          copy(step + 1, buf ^ 1);
        }
        const int step0 = first + step * kKeys;
        // A value that some row does not see may be anything: where one of such
        // a step's is not finite, the rows that see it add it here, and the
        // products take it as zero.
        if (step0 + kKeys - 1 > block_hi)
        {
          std::uint16_t *brought = stages + buf * kStage + kTile + 8 * threadIdx.x;
          bool fine = true;
#pragma unroll
          for (int i = 0; i < kCopies; ++i)
          {
            const half8 v = as_half8(*reinterpret_cast<const u32x4 *>(brought + 512 * NW * i));
            fine = fine && all_finite(v);
          }
          if (lane == 0)
          {
            s_fine[wave] = 1;
          }
          if (!__all(fine) && lane == 0)
          {
            s_fine[wave] = 0;
          }
          lds_barrier();
          bool all = true;
#pragma unroll
          for (int w = 0; w < NW; ++w)
          {
            all = all && s_fine[w] != 0;
          }
          if (!all)
          {
            if (way == step % kWays) // the ways' sums are added up: one of them adds it
            {
              for (int t = 0; t < min(kKeys, a.rows_k - step0); ++t)
              {
                const std::uint16_t *spoilt_row = stages + buf * kStage + kTile + t * HD;
                const int swap = swizzle<HD>(t);
                const bool sees = step0 + t <= hi;
#pragma unroll
                for (int d = 0; d < HD / 32; ++d)
                {
#pragma unroll
                  for (int i = 0; i < 16; ++i)
                  {
                    const int ch = 32 * d + 8 * (i / 4) + 4 * half + i % 4;
                    const std::uint16_t v = spoilt_row[8 * ((ch / 8) ^ swap) + ch % 8];
                    run.o[d][i] += sees && !is_finite(v) ? h2f(v) : 0.0f;
                  }
                }
              }
            }
            lds_barrier();
#pragma unroll
            for (int i = 0; i < kCopies; ++i)
            {
              u32x4 *at = reinterpret_cast<u32x4 *>(brought + 512 * NW * i);
              *at = __builtin_bit_cast(u32x4, finite_only(as_half8(*at)));
            }
          }
          lds_barrier();
        }
        const int key0 = step0 + way * kWayKeys;
        if (key0 > wave_hi)
        {
          return;
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
        // Four reads ahead of the products.
        constexpr int kReads = N * HD / 16;
        __builtin_amdgcn_sched_group_barrier(kDsRead, 4, 0);
#pragma unroll
        for (int i = 4; i < kReads; ++i)
        {
          __builtin_amdgcn_sched_group_barrier(kMfma, 1, 0);
          __builtin_amdgcn_sched_group_barrier(kDsRead, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(kMfma, 4, 0);
        // Whether some row of the wave does not see some key of the step.
        const bool edge = key0 + kWayKeys - 1 > all_hi;
        if (edge)
        {
#pragma unroll
          for (int j = 0; j < N; ++j)
          {
#pragma unroll
            for (int i = 0; i < 16; ++i)
            {
              const int key = key0 + 32 * j + 8 * (i / 4) + 4 * half + i % 4;
              s[j][i] = key <= hi ? s[j][i] : -INFINITY;
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
              run.o[d] = mfma32(vt, p[j][u], run.o[d]);
            }
          }
        }
      };
      for (int step = begin; step < end; step += kInTurn ? 2 : 1)
      {
        if constexpr (!kInTurn)
        {
          take((step - begin) & 1, step);
          continue;
        }
        take(std::integral_constant<int, 0>{}, step);
        if (step + 1 < end)
        {
          take(std::integral_constant<int, 1>{}, step + 1);
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

    // The parts of a (query, head) row joined, four channels a thread.
    template <int HD>
    __global__ void __launch_bounds__(256) packed_join_few_kernel(PackedArgs a, std::size_t rows)
    {
      constexpr int kLanes = HD / 4;
      const std::size_t i = static_cast<std::size_t>(blockIdx.x) * 256 + threadIdx.x;
      const std::size_t row = i / kLanes;
      const int d = 4 * static_cast<int>(i % kLanes);
      const long long query = row / a.heads;
      if (row >= rows || query < a.offsets_q[0] || query >= a.offsets_q[a.batch])
      {
        return; // of no sequence
      }
      float m[kFewSplits], l[kFewSplits];
      f32x4 o[kFewSplits];
      float top = -INFINITY;
#pragma unroll
      for (int s = 0; s < kFewSplits; ++s)
      {
        const std::size_t at = min(s, a.splits - 1) * rows + row;
        const f32x2 ml = *reinterpret_cast<const f32x2 *>(a.part_ml + 2 * at);
        o[s] = *reinterpret_cast<const f32x4 *>(a.part_o + at * HD + d);
        m[s] = s < a.splits ? ml[0] : -INFINITY;
        l[s] = ml[1];
        top = fmaxf(top, m[s]);
      }
      const float from = top == -INFINITY ? 0.0f : top;
      float sum = 0.0f;
      f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int s = 0; s < kFewSplits; ++s)
      {
        if (s < a.splits)
        {
          const float w = __builtin_amdgcn_exp2f(m[s] - from);
          sum += l[s] * w;
          acc += o[s] * w;
        }
      }
      const float inv = sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f; // of no keys: zeros
      const half2v x = {static_cast<_Float16>(acc[0] * inv), static_cast<_Float16>(acc[1] * inv)};
      const half2v y = {static_cast<_Float16>(acc[2] * inv), static_cast<_Float16>(acc[3] * inv)};
      *reinterpret_cast<u32x2 *>(a.out + row * HD + d) =
          u32x2{__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, y)};
    }

    // The same for many parts: a workgroup a row, its groups of lanes each taking
    // some.
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
      static constexpr int tiles = kTiles_, ways = kWays_, keys = kKeys_, rows = 32 * kTiles_,
                           threads = 64 * kTiles_ * kWays_;
    };
    using Few = Form<1, 4, 128>;
    using Many64 = Form<4, 2, 128>;
    using Many128 = Form<4, 1, 64>;

    // How a launch is cut. The lengths are on the device: what is known of them
    // here is how many rows and keys there are.
    struct Cut
    {
      bool few;
      int blocks; // workgroups over the tiles there may be, a KV head
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
      // Few rows over short spans: what leaves no CU two of those workgroups (at
      // head_dim 64, whose stages leave room, four); a handful over long ones.
      // Measured in us, few against many: 413 x 14 heads of 64 in nine chats 7.5 and
      // 13; 256 x 12 of 128 over 2,000 keys 22.9 and 21.7; 512 x 12 of 128 over
      // 8,192 87.6 and 54.8; 64 x 32 of 64 over 8,192 25.6 and 22.8.
      const long long few = (rows + Few::rows - 1) / Few::rows * t.kv_heads;
      const bool narrow = t.head_dim == 64;
      c.few = few <= (span <= 1024 && narrow ? 512 : span <= 2048 ? 256 : 32);
      const int tile = c.few ? Few::rows : narrow ? Many64::rows : Many128::rows;
      const int keys = c.few ? Few::keys : narrow ? Many64::keys : Many128::keys;
      c.blocks = static_cast<int>(rows / tile + std::min(t.batch, t.rows_q)); // a short tile a sequence
      c.splits = 1;
      if (may_split && c.blocks > 0)
      {
        // Few rows: a workgroup a CU, of two steps at least, unless the chain is as
        // short as the join. Many: the device's workgroups, of eight steps at
        // least, sixteen of the longer ones where they are no handful (512 x 12 of
        // 128 over 8,192 keys: one part 153 us, four 54.8, eight 55.3; 8 x 64 over
        // 2,000 each: one 43.9, three 26.0, eight 34; 8 x 64 x 32 of 64 over 2,000:
        // one 29.2, two 40.5; 512 over 8,192 93.6, three 72.9).
        const long long steps = (span + keys - 1) / keys;
        const long long groups = static_cast<long long>(c.blocks) * t.kv_heads;
        const long long parts = c.few ? std::min(256 / groups, steps < 4 ? 1 : steps / 2)
                                      : std::min<long long>({512 / groups, steps / (narrow && groups >= 64 ? 16 : 8), 16});
        c.splits = static_cast<int>(std::max<long long>(1, std::min<long long>(parts, kMaxSplits)));
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
      if (t.rows_q > kMost || t.rows_k > kMost || t.batch > 65535)
      {
        throw InvalidArgument("packed attention takes at most 65535 sequences and " +
                              std::to_string(kMost) + " rows, got " + std::to_string(t.batch) + ", " +
                              std::to_string(t.rows_q) + " and " + std::to_string(t.rows_k));
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
      // A head's offset in its token is 32 bits, and a launch's workgroups and
      // a join's rows are.
      if (static_cast<long long>(t.heads) * t.head_dim > 0x7fffffff ||
          static_cast<long long>(t.rows_q) * t.heads > 0x7fffffffll - 65535ll * t.kv_heads)
      {
        throw InvalidArgument("packed attention takes fewer than 2^31 query elements a token and "
                              "(query, head) rows, got " + std::to_string(t.rows_q) + " rows of " +
                              std::to_string(t.heads) + " heads of " + std::to_string(t.head_dim));
      }
    }

    template <int HD, typename F>
    void launch(const PackedArgs &a, const Cut &c, hipStream_t stream)
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
      kernel<<<dim3(c.blocks * a.kv_heads, c.splits), F::threads, lds, stream>>>(a);
      hip_check(hipGetLastError(), "packed_kernel");
    }

    template <int HD>
    void launch_any(const PackedArgs &a, const Cut &c, hipStream_t stream)
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
        const std::size_t rows = static_cast<std::size_t>(a.rows_q) * a.heads;
        if (c.splits <= kFewSplits)
        {
          const std::size_t blocks = (rows * (HD / 4) + 255) / 256;
          packed_join_few_kernel<HD><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(a, rows);
          hip_check(hipGetLastError(), "packed_join_few_kernel");
          return;
        }
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
    // (A step's rows within 32 bits.)
    constexpr long long kMostStride = 1 << 24;
    if (t.q_stride < 0 || t.k_stride < 0 || t.v_stride < 0 || q_stride < q_width ||
        k_stride < width || v_stride < width || k_stride >= kMostStride || v_stride >= kMostStride)
    {
      throw InvalidArgument("packed attention's strides are of a token's " +
                            std::to_string(q_width) + " query and " + std::to_string(width) +
                            " key and value elements at least (0: those), of keys and values below " +
                            std::to_string(kMostStride) + "; got " +
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
    const long long groups = static_cast<long long>(c.blocks) * t.kv_heads;
    const int threads = c.few ? Few::threads : t.head_dim == 64 ? Many64::threads : Many128::threads;
    if (groups * threads > 0xffffffffll) // (a launch's)
    {
      throw InvalidArgument("packed attention takes at most " + std::to_string(0xffffffffll / threads) +
                            " tiles of rows and KV heads, got " + std::to_string(groups) + " of " +
                            std::to_string(t.batch) + " sequences, " + std::to_string(t.rows_q) +
                            " rows and " + std::to_string(t.kv_heads) + " KV heads");
    }
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
    a.kv_heads = t.kv_heads;
    a.group = t.heads / t.kv_heads;
    a.splits = c.splits;
    // Where the device holds them all at once, tiles need no order.
    const int held = 2 * kCus;
    a.ranked = t.batch <= kRanked && groups * c.splits > kCus ? static_cast<int>(std::min<long long>(held, groups)) : 0;
    a.scale = static_cast<float>(1.4426950408889634 / std::sqrt(static_cast<double>(t.head_dim)));
    if (c.splits > 1)
    {
      const std::size_t rows = static_cast<std::size_t>(t.rows_q) * t.heads;
      a.part_o = t.partials;
      a.part_ml = t.partials + rows * c.splits * t.head_dim;
    }
    t.head_dim == 64 ? launch_any<64>(a, c, stream)
                     : launch_any<128>(a, c, stream);
  }

} // namespace mi
