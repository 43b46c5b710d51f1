// One new token of every sequence of a batch: attention over paged,
// mixed-precision caches, whole or through a sliding window with the first
// `sinks` tokens kept visible, with the pages' attention masses on request.
//
// For sequence b of n = length[b] tokens and query head h of KV head kv:
//   s_j = q . k_j / sqrt(hd) over the visible keys j < n (all of them, or
//   j >= n - window or j < sinks), p = softmax(s), out = sum p_j v_j,
//   mass[page] = the sum of its keys' p.
// Nothing visible: out 0 and masses 0. A page whose tier is not 0..3 or whose
// address is 0 is not read.
//
// Layout. A sequence's visible pages (the sink pages, then the window's) are
// one list; a workgroup takes a run of it, its four waves sharing the run's
// pages and the KV heads (up to four) among them, so that the KV heads of a
// page, which share its rows' lines, are read on one CU. A wave reads a page
// of a KV head once for all the query heads of that KV head: the keys as M of
// 16x16x32 products, the heads as N, codes made fp16 in registers (the page
// format's own rounding), V transposed by products with a 0/1 matrix, P as
// high and low fp16 parts, the softmax in base 2 with a running maximum. The
// waves of a KV head meet in LDS, phase by phase; each workgroup writes a
// maximum, sum and output a head, which a second launch joins. A launch of one
// run a sequence writes its outputs itself. A visible value that is not finite
// makes the 32 channels of its step not finite in the heads that see it.
//
// Bound by the latency of a page's one dependent chain, some 500 vector and 40
// matrix instructions (a SIMD is busy 40% of the time), with the page's own
// trip to memory before it: 16 sequences to 32,768 tokens (12 x 2 heads of 128,
// mixed tiers) 30 us of which the join is 5, 2.9 TB/s; 32 to 16,640 behind a
// 4,096-token window (32 x 8 heads of 64) 27.5 us, 2.8 TB/s; 8 to 5,000 with
// masses 12.8; one of 33 tokens 5.4 us, one launch. Four waves a workgroup: eight took 54
// and 38 us for the first two. Scalar page bases and 32-bit lane offsets, not
// kept from page to page, leave four waves a SIMD at head_dim 64; two a SIMD,
// evenly, are better than three at 128. The next page fetched ahead into LDS
// costs waves at 64 (34 us) and saves nothing at 128, nor would faster memory
// save much: with every page in the caches the first two take 28.7 of 31.0 us
// and 26.2 of 27.0, each pair from one run.

#include "common.hpp"
#include "dequant.hpp"
#include "lane_ops.hpp"
#include "serving.hpp"

#include <algorithm>
#include <cmath>
#include <string>

namespace mi
{
  namespace
  {
    using dq::dequant_step;
    typedef _Float16 half8 __attribute__((ext_vector_type(8)));
    typedef _Float16 half2v __attribute__((ext_vector_type(2)));
    typedef float f32x4 __attribute__((ext_vector_type(4)));
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
    typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
    typedef const __attribute__((address_space(1))) u32x4 *g_u32x4;
    typedef u32x4 u32x4_anywhere __attribute__((aligned(2))); // a token's row: any view's
    typedef const __attribute__((address_space(1))) u32x4_anywhere *g_u32x4_anywhere;
    typedef const __attribute__((address_space(1))) u32x2 *g_u32x2;
    typedef const __attribute__((address_space(1))) unsigned *g_u32;
    typedef const __attribute__((address_space(1))) unsigned short *g_u16;

    constexpr int kWaves = 4;
    constexpr int kThreads = 64 * kWaves;
    constexpr int kP = kBatchPageTokens;
    constexpr int kMaxGroup = 16;
    constexpr int kMaxSplits = 1024;
    constexpr int kJoinThreads = 512;
    // P is held x 2^14 (exact), so that its fp16 low part stays normal for
    // every weight above 2^-17 of the running maximum.
    constexpr float kPScale = 16384.0f;
    constexpr float kPUnscale = 1.0f / 16384.0f;

    struct BatchArgs
    {
      const std::uint16_t *q; // (batch, heads, hd)
      std::uint16_t *out;
      float *mass;      // (batch, heads, max_pages), or null
      float *mass_from; // the same: the maximum each page's mass is held against
      float *parts_ml;  // splits > 1: [batch][heads][splits] maxima and sums,
      float *parts_o;   // and outputs of hd floats
      const unsigned long long *pages; // (batch, max_pages)
      const std::uint8_t *tiers;
      const int *lengths;
      int max_pages;
      int heads;
      int kv_heads;
      int group;
      int kv_block; // KV heads a workgroup takes: a power of two up to 4
      int window;   // 0: every token
      int sinks;
      int run_pages; // of the visible list a workgroup takes
      int splits;
      float scale; // log2 e / sqrt(hd): scores in base 2
    };

    // The sequences themselves, where the launch brings them (kHeld).
    template <bool kHeld>
    struct Sequences
    {
    };
    template <>
    struct Sequences<true>
    {
      BatchSequence of[kBatchHeld];
    };

    // A sequence's visible pages: [0, sink_pages) and [first, pages).
    struct Reach
    {
      int length;
      int pages;
      int sink_pages;
      int first;
      __device__ int count() const { return sink_pages + pages - first; }
      __device__ int page(int i) const { return i < sink_pages ? i : first + i - sink_pages; }
      __device__ bool has(int page) const
      {
        return page < pages && (page >= first || page < sink_pages);
      }
    };

    __device__ inline Reach reach_of(const BatchArgs &a, int length)
    {
      Reach r;
      r.pages = min(max(length, 0) / kP + (length % kP > 0 ? 1 : 0), a.max_pages);
      r.length = min(max(length, 0), r.pages * kP);
      r.sink_pages = 0;
      r.first = 0;
      if (a.window > 0 && a.window < r.length)
      {
        r.first = (r.length - a.window) / kP;
        r.sink_pages = min(a.sinks / kP + (a.sinks % kP > 0 ? 1 : 0), r.first);
      }
      return r;
    }

    // The page's visible tokens, a bit each.
    __device__ inline unsigned visible_of(const BatchArgs &a, const Reach &r, int page)
    {
      const int t0 = page * kP;
      const int held = r.length - t0; // > 0
      unsigned bits = held >= kP ? ~0u : (1u << held) - 1u;
      const int hidden = a.window > 0 ? r.length - a.window - t0 : 0; // tokens before the window
      if (hidden > 0)
      {
        const unsigned in_window = hidden >= kP ? 0u : ~0u << hidden;
        const int kept = a.sinks - t0;
        bits &= in_window | (kept >= kP ? ~0u : kept > 0 ? (1u << kept) - 1u : 0u);
      }
      return bits;
    }

    __device__ inline half8 as_half8(u32x4 v) { return __builtin_bit_cast(half8, v); }

    __device__ inline f32x4 mfma(half8 a, half8 b, f32x4 c)
    {
      return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }

    // Loads from a base that is the same in every lane (scalar registers) and
    // the lane's 32-bit offset.
    typedef const __attribute__((address_space(1))) std::uint8_t *g_base;

    template <int Bytes>
    __device__ inline void load_words(unsigned *w, g_base base, unsigned offset)
    {
      if constexpr (Bytes >= 16)
      {
#pragma unroll
        for (int i = 0; i < Bytes / 16; ++i)
        {
          const u32x4 v = *((g_u32x4)(base + offset + 16 * i));
          w[4 * i + 0] = v.x;
          w[4 * i + 1] = v.y;
          w[4 * i + 2] = v.z;
          w[4 * i + 3] = v.w;
        }
      }
      else if constexpr (Bytes == 8)
      {
        const u32x2 v = *((g_u32x2)(base + offset));
        w[0] = v.x;
        w[1] = v.y;
      }
      else
      {
        w[0] = *((g_u32)(base + offset));
      }
    }

    // A wave's running softmax and output, lane % 16 the query head: weights
    // are 2^(score - m), o carries kPScale.
    template <int HD>
    struct Running
    {
      float m;
      float l;
      f32x4 o[HD / 16];
    };

    struct PageAt
    {
      int r; // lane % 16: a row of each half of the page, and a query head
      int g; // lane / 16: a quarter of the channels
      unsigned visible;
      float scale;
      bool scored;
      unsigned mass_at; // where head r's sum of the page goes, from the KV head's rows
      float *mass;
      float *mass_from;
    };

    // The lane's first channel in row r of a page's keys, in elements. Opaque,
    // so that no tier's offsets are kept in registers from page to page.
    __device__ inline unsigned opaque(unsigned v)
    {
      asm volatile("" : "+v"(v));
      return v;
    }

    // The two 16-key accumulators as P (high, low), the running softmax
    // moved on. (Scores are scaled inside the subtraction of the maximum, by
    // one fma, so that a weight errs by its distance to the maximum, not by
    // its score.)
    template <int HD>
    __device__ inline void softmax_page(f32x4 (&acc)[2], const PageAt &c, Running<HD> &run,
                                        half8 &p_hi, half8 &p_lo)
    {
      if (c.visible != ~0u)
      {
        const unsigned mine = c.visible >> (4 * c.g); // keys 16 b + 4 g + {0..3}
#pragma unroll
        for (int e = 0; e < 8; ++e)
        {
          acc[e / 4][e % 4] =
              mine & (1u << (e / 4 * 16 + e % 4)) ? acc[e / 4][e % 4] : -INFINITY;
        }
      }
      float top = acc[0][0];
#pragma unroll
      for (int e = 1; e < 8; ++e)
      {
        top = fmaxf(top, acc[e / 4][e % 4]);
      }
      top = lane_max32(lane_max16(top)) * c.scale;
      const float m = fmaxf(run.m, top);
      const float from = m == -INFINITY ? 0.0f : m;
      const float keep = __builtin_amdgcn_exp2f(run.m - from);
      float p[8], sum = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e)
      {
        p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[e / 4][e % 4], c.scale, -from));
        sum += p[e];
      }
      sum = lane_sum32(lane_sum16(sum));
      if (c.scored && c.g == 0)
      {
        c.mass[c.mass_at] = sum;
        c.mass_from[c.mass_at] = from;
      }
      run.l = run.l * keep + sum;
      if (__builtin_amdgcn_ballot_w64(!(top <= run.m)) != 0)
      {
#pragma unroll
        for (int d = 0; d < HD / 16; ++d)
        {
          run.o[d] *= keep;
        }
      }
      run.m = m;
#pragma unroll
      for (int e = 0; e < 8; ++e)
      {
        _Float16 hi, lo;
        split_half(p[e] * kPScale, hi, lo);
        p_hi[e] = hi;
        p_lo[e] = lo;
      }
    }

    __device__ inline unsigned packed(float a, float b)
    {
      return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_pkrtz(a, b));
    }

    // The 0/1 matrix that picks channel r (lo) or 16 + r (hi) of 32: row
    // 8 g + e, column r. Made anew for each page, not kept through it.
    struct Pick
    {
      u32x4 lo;
      u32x4 hi;
      __device__ Pick(int lane_r, int g)
      {
        const unsigned r = opaque(lane_r);
        const unsigned one = r & 1u ? 0x3C000000u : 0x00003C00u;
        const unsigned word = r % 8 / 2;
        const unsigned group = r / 8; // of lo; 2 more of hi
#pragma unroll
        for (unsigned w = 0; w < 4; ++w)
        {
          const unsigned v = w == word ? one : 0u;
          lo[w] = static_cast<unsigned>(g) == group ? v : 0u;
          hi[w] = static_cast<unsigned>(g) == group + 2 ? v : 0u;
        }
      }
    };

    // P.V of 32 channels (8 of each quarter): V^T by products with a 0/1
    // matrix, whose K axis then is the lane's own keys.
    template <int HD>
    __device__ inline void values_step(Running<HD> &run, int s, half8 v0, half8 v1, const Pick &p,
                                       half8 p_hi, half8 p_lo)
    {
      const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int h = 0; h < 2; ++h)
      {
        const half8 pick = as_half8(h == 0 ? p.lo : p.hi);
        const f32x4 t0 = mfma(v0, pick, zero);
        const f32x4 t1 = mfma(v1, pick, zero);
        // (Exact, so that any rounding is the same.)
        const half8 vt = as_half8(u32x4{packed(t0[0], t0[1]), packed(t0[2], t0[3]),
                                        packed(t1[0], t1[1]), packed(t1[2], t1[3])});
        run.o[2 * s + h] = mfma(vt, p_hi, run.o[2 * s + h]);
        run.o[2 * s + h] = mfma(vt, p_lo, run.o[2 * s + h]);
      }
    }

    // The first of o[2 s + h]'s four channels in lane group g.
    template <int HD>
    __device__ inline int channel_of(int s, int h, int g)
    {
      return (2 * h + g / 2) * (HD / 4) + 8 * s + 4 * (g % 2);
    }

    // A value row that is not visible may hold anything: it enters P.V as
    // zeros (its weight is zero, and zero times infinity is not).
    template <int S>
    __device__ inline void hide_rows(half8 (&v)[2][S], const PageAt &c)
    {
#pragma unroll
      for (int b = 0; b < 2; ++b)
      {
        if (!((c.visible >> (16 * b + c.r)) & 1u))
        {
#pragma unroll
          for (int s = 0; s < S; ++s)
          {
            v[b][s] = as_half8(u32x4{0u, 0u, 0u, 0u});
          }
        }
      }
    }

    // A page of FP16 rows, keys then values. `own_row`, if it is not negative,
    // is read from own_k and own_v (a token's row, not yet in the page).
    template <int HD>
    __device__ inline void fp16_page(Running<HD> &run, const PageAt &c, const half8 (&q)[HD / 32],
                                     g_base page, unsigned elem, int width, int own_row = -1,
                                     const std::uint16_t *own_k = nullptr,
                                     const std::uint16_t *own_v = nullptr)
    {
      constexpr int S = HD / 32;
      half8 k[2][S], v[2][S];
      const unsigned at = 2 * opaque(elem);
#pragma unroll
      for (int b = 0; b < 2; ++b)
      {
#pragma unroll
        for (int s = 0; s < S; ++s)
        {
          k[b][s] = as_half8(*((g_u32x4)(page + 32 * b * width + at + 16 * s)));
        }
      }
#pragma unroll
      for (int b = 0; b < 2; ++b)
      {
#pragma unroll
        for (int s = 0; s < S; ++s)
        {
          v[b][s] = as_half8(*((g_u32x4)(page + 2 * (kP + 16 * b) * width + at + 16 * s)));
        }
      }
      if (own_row >= 0)
      {
#pragma unroll
        for (int b = 0; b < 2; ++b)
        {
          if (16 * b + c.r == own_row)
          {
            const unsigned chan = elem - c.r * width;
#pragma unroll
            for (int s = 0; s < S; ++s)
            {
              k[b][s] = as_half8(*((g_u32x4_anywhere)(own_k + chan + 8 * s)));
              v[b][s] = as_half8(*((g_u32x4_anywhere)(own_v + chan + 8 * s)));
            }
          }
        }
      }
      f32x4 acc[2] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
      for (int s = 0; s < S; ++s)
      {
        acc[0] = mfma(k[0][s], q[s], acc[0]);
        acc[1] = mfma(k[1][s], q[s], acc[1]);
      }
      half8 p_hi, p_lo;
      softmax_page<HD>(acc, c, run, p_hi, p_lo);
      const Pick pick(c.r, c.g);
      if (c.visible != ~0u)
      {
        hide_rows<S>(v, c);
      }
#pragma unroll
      for (int s = 0; s < S; ++s)
      {
        values_step<HD>(run, s, v[0][s], v[1][s], pick, p_hi, p_lo);
      }
    }

    // `meta`: the wave's 2 HD halves of LDS, through which the page's key
    // scales and zeros reach the 16 lanes that share them.
    template <int HD, int Bits>
    __device__ inline void quantised_page(Running<HD> &run, const PageAt &c,
                                          const half8 (&q)[HD / 32], g_base page, unsigned elem,
                                          int width, int kvh, int kv_heads, int lane,
                                          unsigned *meta)
    {
      constexpr int S = HD / 32;
      constexpr int kRun = HD / 4;
      constexpr int kRowBytes = kRun * Bits / 8;
      constexpr int kWords = kRowBytes / 4;
      constexpr int kMetaLanes = HD / 4; // 8 bytes a lane, scales then zeros
      // The page's regions back to back, as page_layout lays them.
      const unsigned value_codes = kP * width * Bits / 8;
      const unsigned key_scales = 2 * value_codes;
      const unsigned value_scales = key_scales + 4 * width;
      const unsigned value_zeros = value_scales + 2 * kP * kv_heads;
      unsigned kc[2][kWords], vc[2][kWords];
      unsigned short vs[2], vz[2];
      const unsigned at = opaque(elem) / (8 / Bits);
#pragma unroll
      for (int b = 0; b < 2; ++b)
      {
        load_words<kRowBytes>(kc[b], page + 16 * b * width * Bits / 8, at);
        load_words<kRowBytes>(vc[b], page + value_codes + 16 * b * width * Bits / 8, at);
      }
      u32x2 km = {0u, 0u};
      if (lane < 2 * kMetaLanes)
      {
        // (The zeros lie behind the scales: a lane's eight bytes of a head's
        // scales, or 2 width bytes on.)
        const unsigned piece = 8 * (lane % kMetaLanes) + (lane < kMetaLanes ? 0 : 2 * width);
        km = *((g_u32x2)(page + key_scales + 2 * kvh * HD + opaque(piece)));
      }
#pragma unroll
      for (int b = 0; b < 2; ++b)
      {
        const unsigned row = 2 * (opaque(c.r) * kv_heads);
        vs[b] = *((g_u16)(page + value_scales + 2 * (16 * b * kv_heads + kvh) + row));
        vz[b] = *((g_u16)(page + value_zeros + 2 * (16 * b * kv_heads + kvh) + row));
      }
      // One wave's LDS operations complete in order; the fences keep the
      // compiler from moving the reads above the write, and the write above
      // the last page's reads.
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      if (lane < 2 * kMetaLanes)
      {
        *reinterpret_cast<u32x2 *>(meta + 2 * lane) = km;
      }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
      const auto word = [](const unsigned(&w)[kWords], int s, int second) -> unsigned {
        if constexpr (Bits == 8)
        {
          return w[2 * s + second];
        }
        else if constexpr (Bits == 4)
        {
          return w[s];
        }
        else
        {
          return w[s / 2] >> (16 * (s & 1));
        }
      };
      f32x4 acc[2] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
      for (int s = 0; s < S; ++s)
      {
        const u32x4 s2 = *reinterpret_cast<const u32x4 *>(meta + (c.g * kRun + 8 * s) / 2);
        const u32x4 z2 = *reinterpret_cast<const u32x4 *>(meta + (HD + c.g * kRun + 8 * s) / 2);
#pragma unroll
        for (int b = 0; b < 2; ++b)
        {
          acc[b] = mfma(dequant_step<Bits>(word(kc[b], s, 0), word(kc[b], s, 1), s2, z2), q[s],
                        acc[b]);
        }
      }
      half8 p_hi, p_lo;
      softmax_page<HD>(acc, c, run, p_hi, p_lo);
      const Pick pick(c.r, c.g);
      u32x4 s4[2], z4[2];
#pragma unroll
      for (int b = 0; b < 2; ++b)
      {
        // (A row that is not visible: codes times zero and zero. Its scale and
        // zero may be anything, its codes are finite.)
        const bool see = c.visible == ~0u || ((c.visible >> (16 * b + c.r)) & 1u);
        const unsigned sp = see ? vs[b] | (static_cast<unsigned>(vs[b]) << 16) : 0u;
        const unsigned zp = see ? vz[b] | (static_cast<unsigned>(vz[b]) << 16) : 0u;
        s4[b] = u32x4{sp, sp, sp, sp};
        z4[b] = u32x4{zp, zp, zp, zp};
      }
#pragma unroll
      for (int s = 0; s < S; ++s)
      {
        half8 v[2];
#pragma unroll
        for (int b = 0; b < 2; ++b)
        {
          v[b] = dequant_step<Bits>(word(vc[b], s, 0), word(vc[b], s, 1), s4[b], z4[b]);
        }
        values_step<HD>(run, s, v[0], v[1], pick, p_hi, p_lo);
      }
    }

    // LDS of the pages kernel, in floats: the key metadata a wave, then the
    // waves' joined state (the outputs of every wave but the first phase's, a
    // lane's registers as they are), then the heads' maxima and sums.
    template <int HD>
    constexpr int kMetaFloats = kWaves * HD;
    template <int HD>
    constexpr int kWaveFloats = HD / 16 * 4 * 64;
    constexpr int kHeadFloats = kWaves * kMaxGroup * 2;

    // One page's mass from the sum held against `held_from`, given the row's
    // maximum and sum. (A page that was not read is held against 0, which may
    // lie further above the maximum than 2^x reaches: its zero stays one.)
    __device__ inline float mass_of(float sum, float held_from, float top, float inv)
    {
      return sum == 0.0f ? 0.0f : sum * __builtin_amdgcn_exp2f(held_from - top) * inv;
    }

    template <int HD, bool kHeld>
    __global__ void __launch_bounds__(kThreads, HD == 64 ? 4 : 2) batch_pages_kernel(BatchArgs a,
                                                                                    Sequences<kHeld> held)
    {
      constexpr int S = HD / 32;
      constexpr int kRun = HD / 4;
      extern __shared__ __align__(16) float lds[];
      const int lane = threadIdx.x & 63;
      const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
      const int r = lane & 15;
      const int g = lane >> 4;
      const int b = blockIdx.z;
      const int split = blockIdx.x;
      const int phases = kWaves / a.kv_block;
      const int phase = wave / a.kv_block;
      const int begin = split * a.run_pages;
      BatchSequence sequence{};
      if constexpr (kHeld)
      {
        sequence = held.of[b];
      }
      const unsigned long long *pages =
          kHeld ? sequence.pages : a.pages + static_cast<std::size_t>(b) * a.max_pages;
      const std::uint8_t *tiers =
          kHeld ? sequence.tiers : a.tiers + static_cast<std::size_t>(b) * a.max_pages;
      // Without a window the list is the table itself: the wave's first entries
      // are asked for together with the length, which says whether they count.
      unsigned long long first_address = 0;
      int first_tier = kUnreadPage;
      if (!kHeld && a.window == 0)
      {
        const long long entry = static_cast<long long>(begin) + phase + lane * phases;
        if (lane * phases + phase < a.run_pages && entry < a.max_pages)
        {
          first_address = pages[entry];
          first_tier = tiers[entry];
        }
      }
      const Reach reach = reach_of(a, kHeld ? sequence.length : a.lengths[b]);
      const int count = reach.count();
      if (split > 0 && begin >= count)
      {
        return; // the join reads no part of this split
      }
      const int end = min(begin + a.run_pages, count);
      const int kvh = blockIdx.y * a.kv_block + wave % a.kv_block;
      const int G = a.group;
      const int width = a.kv_heads * HD;

      // The sequence's own page, where a cache that seals keeps it: the rows
      // before the token's in the page being filled, the token's as given.
      const bool open = kHeld && sequence.open != nullptr;
      const int own_page = open ? (reach.length - 1) / kP : -1;

      // Columns past the group repeat its first head and are not stored.
      const std::size_t head0 = static_cast<std::size_t>(b) * a.heads + kvh * G;
      const std::uint16_t *q_row = a.q + (head0 + (r < G ? r : 0)) * HD + g * kRun;
      half8 q[S];
#pragma unroll
      for (int s = 0; s < S; ++s)
      {
        q[s] = as_half8(*((g_u32x4)(q_row + 8 * s)));
      }
      Running<HD> run;
      run.m = -INFINITY;
      run.l = 0.0f;
#pragma unroll
      for (int d = 0; d < HD / 16; ++d)
      {
        run.o[d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      }
      unsigned *meta = reinterpret_cast<unsigned *>(lds) + wave * HD;
      const unsigned elem = static_cast<unsigned>(r * width + kvh * HD + g * kRun);
      const bool scored = a.mass != nullptr && r < G;
      float *mass = a.mass + head0 * a.max_pages;
      float *mass_from = a.mass_from + head0 * a.max_pages;
      const unsigned mass_at = static_cast<unsigned>(r) * static_cast<unsigned>(a.max_pages);

      // The wave's pages, up to 64 at a time: their table entries are one
      // lane's each, asked for together.
      for (int first = begin + phase; first < end; first += 64 * phases)
      {
        unsigned long long address = 0;
        int tier_of = kUnreadPage;
        const int entry = first + lane * phases;
        if (!kHeld && first == begin + phase && a.window == 0)
        {
          address = first_address;
          tier_of = first_tier;
        }
        else if (entry < end && reach.page(entry) != own_page)
        {
          // (The own page of a cache that seals has no entry to read: the
          // table may end before it.)
          address = pages[reach.page(entry)];
          tier_of = tiers[reach.page(entry)];
        }
        if (entry >= end || address == 0)
        {
          tier_of = kUnreadPage;
        }
        const unsigned address_lo = static_cast<unsigned>(address);
        const unsigned address_hi = static_cast<unsigned>(address >> 32);
        const int here = min(64, (end - first + phases - 1) / phases);
        for (int t = 0; t < here; ++t)
        {
          const int page = __builtin_amdgcn_readfirstlane(reach.page(first + t * phases));
          const PageAt c{r, g, visible_of(a, reach, page), a.scale, scored, mass_at + page, mass,
                         mass_from};
          if (kHeld && page == own_page)
          {
            fp16_page<HD>(run, c, q, (g_base)(sequence.open), elem, width,
                          (reach.length - 1) % kP, sequence.own_k, sequence.own_v);
            continue;
          }
          const unsigned long long page_address =
              static_cast<unsigned>(__builtin_amdgcn_readlane(static_cast<int>(address_lo), t)) |
              static_cast<unsigned long long>(static_cast<unsigned>(
                  __builtin_amdgcn_readlane(static_cast<int>(address_hi), t)))
                  << 32;
          const g_base at = (g_base)(page_address);
          switch (__builtin_amdgcn_readlane(tier_of, t))
          {
          case kFP16: fp16_page<HD>(run, c, q, at, elem, width); break;
          case kINT8:
            quantised_page<HD, 8>(run, c, q, at, elem, width, kvh, a.kv_heads, lane, meta);
            break;
          case kINT4:
            quantised_page<HD, 4>(run, c, q, at, elem, width, kvh, a.kv_heads, lane, meta);
            break;
          case kINT2:
            quantised_page<HD, 2>(run, c, q, at, elem, width, kvh, a.kv_heads, lane, meta);
            break;
          default:
            if (scored && g == 0)
            {
              mass[c.mass_at] = 0.0f;
              mass_from[c.mass_at] = 0.0f;
            }
          }
        }
      }

      // The waves of a KV head joined into its first phase's.
      f32x4 *s_o = reinterpret_cast<f32x4 *>(lds + kMetaFloats<HD>);
      float *s_ml = lds + kMetaFloats<HD> + (phases - 1) * a.kv_block * kWaveFloats<HD>;
      if (g == 0)
      {
        *reinterpret_cast<f32x2 *>(s_ml + 2 * (wave * kMaxGroup + r)) = f32x2{run.m, run.l};
      }
      if (phase > 0)
      {
#pragma unroll
        for (int d = 0; d < HD / 16; ++d)
        {
          s_o[((wave - a.kv_block) * (HD / 16) + d) * 64 + lane] = run.o[d];
        }
      }
      __syncthreads();
      if (phase == 0)
      {
        float top = run.m;
        for (int p = 1; p < phases; ++p)
        {
          top = fmaxf(top, s_ml[2 * ((wave + p * a.kv_block) * kMaxGroup + r)]);
        }
        const float from = top == -INFINITY ? 0.0f : top;
        const float keep = __builtin_amdgcn_exp2f(run.m - from);
        float sum = run.l * keep;
#pragma unroll
        for (int d = 0; d < HD / 16; ++d)
        {
          run.o[d] *= keep;
        }
        for (int p = 1; p < phases; ++p)
        {
          const int w = wave + p * a.kv_block;
          const f32x2 ml = *reinterpret_cast<const f32x2 *>(s_ml + 2 * (w * kMaxGroup + r));
          const float f = __builtin_amdgcn_exp2f(ml[0] - from);
          sum += ml[1] * f;
#pragma unroll
          for (int d = 0; d < HD / 16; ++d)
          {
            run.o[d] += s_o[((w - a.kv_block) * (HD / 16) + d) * 64 + lane] * f;
          }
        }
        if (r < G)
        {
          const std::size_t head = head0 + r;
          if (a.splits > 1)
          {
            const std::size_t part = head * a.splits + split;
            if (g == 0)
            {
              *reinterpret_cast<f32x2 *>(a.parts_ml + 2 * part) = f32x2{top, sum};
            }
#pragma unroll
            for (int d = 0; d < HD / 16; ++d)
            {
              *reinterpret_cast<f32x4 *>(a.parts_o + part * HD + channel_of<HD>(d / 2, d % 2, g)) =
                  run.o[d] * kPUnscale;
            }
          }
          else
          {
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum; // (a sum of NaN stays one)
#pragma unroll
            for (int d = 0; d < HD / 16; ++d)
            {
              const f32x4 o = run.o[d] * (kPUnscale * inv);
              const half2v lo = {static_cast<_Float16>(o[0]), static_cast<_Float16>(o[1])};
              const half2v hi = {static_cast<_Float16>(o[2]), static_cast<_Float16>(o[3])};
              *reinterpret_cast<u32x2 *>(a.out + head * HD + channel_of<HD>(d / 2, d % 2, g)) =
                  u32x2{__builtin_bit_cast(unsigned, lo), __builtin_bit_cast(unsigned, hi)};
            }
            if (g == 0)
            {
              *reinterpret_cast<f32x2 *>(s_ml + 2 * (wave * kMaxGroup + r)) = f32x2{from, inv};
            }
          }
        }
      }
      if (a.mass == nullptr || a.splits > 1)
      {
        return;
      }
      __syncthreads();
      const std::size_t row0 = static_cast<std::size_t>(b) * a.heads + blockIdx.y * a.kv_block * G;
      for (int h = wave; h < a.kv_block * G; h += kWaves)
      {
        const f32x2 fi = *reinterpret_cast<const f32x2 *>(s_ml + 2 * (h / G * kMaxGroup + h % G));
        float *mass = a.mass + (row0 + h) * a.max_pages;
        const float *held_from = a.mass_from + (row0 + h) * a.max_pages;
        for (int p = lane; p < a.max_pages; p += 64)
        {
          mass[p] = reach.has(p) ? mass_of(mass[p], held_from[p], fi[0], fi[1]) : 0.0f;
        }
      }
    }

    // A head's splits joined, weights 2^(m_s - max m); then the masses of its
    // pages.
    template <int HD, bool kHeld>
    __global__ void __launch_bounds__(kJoinThreads) batch_join_kernel(BatchArgs a, Sequences<kHeld> held)
    {
      __shared__ f32x2 s_ml[kJoinThreads / (HD / 4)];
      __shared__ __align__(16) float s_o[kJoinThreads / (HD / 4)][HD];
      __shared__ f32x2 s_total;
      const int b = blockIdx.y;
      const std::size_t head = static_cast<std::size_t>(b) * a.heads + blockIdx.x;
      int length;
      if constexpr (kHeld)
      {
        length = held.of[b].length;
      }
      else
      {
        length = a.lengths[b];
      }
      const Reach reach = reach_of(a, length);
      const int live = (reach.count() + a.run_pages - 1) / a.run_pages;
      // Groups of lanes, sixteen bytes a lane of a split's outputs, each with a
      // running maximum of its own, so that nothing waits for a first pass.
      constexpr int kLanes = HD / 4, kGroups = kJoinThreads / kLanes;
      const int group = threadIdx.x / kLanes;
      const int d = 4 * (threadIdx.x % kLanes);
      float m = -INFINITY, l = 0.0f;
      f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 8
      for (int s = group; s < live; s += kGroups)
      {
        const std::size_t part = head * a.splits + s;
        const f32x2 ml = *reinterpret_cast<const f32x2 *>(a.parts_ml + 2 * part);
        const f32x4 x = *reinterpret_cast<const f32x4 *>(a.parts_o + part * HD + d);
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
      // (By the waves that have an output: the others' reads would be in the way.)
      if (threadIdx.x < HD)
      {
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
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        a.out[head * HD + threadIdx.x] = __half_as_ushort(__float2half(out * inv));
        if (threadIdx.x == 0)
        {
          s_total = f32x2{from, inv};
        }
      }
      if (a.mass == nullptr)
      {
        return;
      }
      __syncthreads();
      const float from = s_total[0], inv = s_total[1];
      float *mass = a.mass + head * a.max_pages;
      const float *held_from = a.mass_from + head * a.max_pages;
      for (int p = threadIdx.x; p < a.max_pages; p += kJoinThreads)
      {
        mass[p] = reach.has(p) ? mass_of(mass[p], held_from[p], from, inv) : 0.0f;
      }
    }

    // How a launch is cut: KV heads a workgroup, pages a run, runs a sequence.
    struct Cut
    {
      int kv_block;
      int run_pages;
      int splits;
      long long most_parts; // of a head over the batch, of partials
    };

    Cut cut_of(int batch, int max_pages, int kv_heads, int head_dim, int window, int sinks)
    {
      Cut c{1, 1, 1, 0};
      while (c.kv_block < kWaves && kv_heads % (2 * c.kv_block) == 0)
      {
        c.kv_block *= 2;
      }
      const int phases = kWaves / c.kv_block;
      // The most pages a sequence can see.
      long long most = max_pages;
      if (window > 0)
      {
        most = std::min<long long>(most, (static_cast<long long>(sinks) + kP - 1) / kP +
                                             (static_cast<long long>(window) + kP - 2) / kP + 1);
      }
      most = std::max<long long>(most, 1);
      // Eight workgroups a CU over the batch if every sequence is as long as it
      // can be (six of head_dim 128, which has two at a time), each wave at
      // least a page: a ragged batch fills half of them, and more only adds
      // parts to join (32 behind a window, in us: 1,024 workgroups 35.5, 2,048
      // 29, 4,096 30; of 128, 16 to 32K: 1,408 30.3, 1,536 30.4, 1,792 36.7).
      const long long workgroups = head_dim == 64 ? 2048 : 1536;
      const long long units = most * batch * (kv_heads / c.kv_block);
      long long run = std::max<long long>((units + workgroups - 1) / workgroups,
                                          (most + kMaxSplits - 1) / kMaxSplits);
      run = (run + phases - 1) / phases * phases;
      // Pages a wave walks rather than have a second launch join them, in us (2
      // KV heads): of 64, four pages 7.8 and 8.7, six 10.0 and 8.7; of 128, three
      // 8.4 and 8.7, four 10.0 and 8.7.
      const long long whole = head_dim == 64 ? 4 : 3;
      const long long paged = std::min<long long>((most + phases - 1) / phases, kMaxSplits);
      if (paged <= whole)
      {
        run = most;
      }
      c.run_pages = static_cast<int>(std::min<long long>(run, 0x7fffffc0));
      c.splits = static_cast<int>((most + run - 1) / run);
      // What no cut of fewer sequences or pages passes: a part a wave's page,
      // and the workgroups that fill the device with one more a sequence.
      c.most_parts = paged <= whole
                         ? 0
                         : std::min(batch * paged, workgroups / (kv_heads / c.kv_block) + batch);
      return c;
    }

    void check_batch(const BatchAttention &t)
    {
      if (t.batch < 0 || t.max_pages < 0 || t.window < 0 || t.sinks < 0)
      {
        throw InvalidArgument("batch, max_pages, window and sinks must not be negative, got " +
                              std::to_string(t.batch) + ", " + std::to_string(t.max_pages) + ", " +
                              std::to_string(t.window) + ", " + std::to_string(t.sinks));
      }
      if (t.page_tokens != kP || (t.head_dim != 64 && t.head_dim != 128))
      {
        throw InvalidArgument("batch attention takes 32-token pages of head_dim 64 or 128, got " +
                              std::to_string(t.page_tokens) + " and " + std::to_string(t.head_dim));
      }
      if (t.kv_heads <= 0 || t.heads <= 0 || t.heads % t.kv_heads != 0 ||
          t.heads / t.kv_heads > kMaxGroup || t.heads > 65535)
      {
        throw InvalidArgument("batch attention takes a whole number of query heads a KV head, at "
                              "most " + std::to_string(kMaxGroup) + ", got " +
                              std::to_string(t.heads) + " and " + std::to_string(t.kv_heads));
      }
      if (t.batch > 65535)
      {
        throw InvalidArgument("a batch of " + std::to_string(t.batch) + " sequences; at most 65535");
      }
      if (t.max_pages > 0x7fffffff / kP)
      {
        throw InvalidArgument(std::to_string(t.max_pages) + " pages a sequence; at most " +
                              std::to_string(0x7fffffff / kP));
      }
    }

    template <int HD, bool kHeld>
    void launch(const BatchArgs &a, const Sequences<kHeld> &held, int batch, hipStream_t stream)
    {
      const int phases = kWaves / a.kv_block;
      // At head_dim 128 LDS for no more than two workgroups a CU: the launch
      // order gives some CUs three while others have one, and three take
      // nearly twice two's time (16 to 32K 35.4 us, so 30.4; 8 to 5K 14.1 and
      // 12.9).
      constexpr std::size_t kThirdOfLds = HD == 64 ? 0 : 55 * 1024;
      const std::size_t lds = std::max(
          kThirdOfLds,
          sizeof(float) * (kMetaFloats<HD> + (phases - 1) * a.kv_block * kWaveFloats<HD> +
                           kHeadFloats));
      const dim3 grid(a.splits, a.kv_heads / a.kv_block, batch);
      batch_pages_kernel<HD, kHeld><<<grid, kThreads, lds, stream>>>(a, held);
      hip_check(hipGetLastError(), "batch_pages_kernel");
      if (a.splits > 1)
      {
        batch_join_kernel<HD, kHeld>
            <<<dim3(a.heads, batch), kJoinThreads, 0, stream>>>(a, held);
        hip_check(hipGetLastError(), "batch_join_kernel");
      }
    }
  } // namespace

  namespace
  {
    void check_overlaps(const BatchAttention &t)
    {
      const std::size_t rows = static_cast<std::size_t>(t.batch) * t.heads;
      const std::size_t entries = static_cast<std::size_t>(t.batch) * t.max_pages;
      const Extent q{t.q, 2 * rows * t.head_dim}, out{t.out, 2 * rows * t.head_dim};
      const Extent mass{t.mass, sizeof(float) * rows * t.max_pages};
      const Extent parts{t.partials, t.partials == nullptr
                                         ? 0
                                         : sizeof(float) *
                                               batch_attention_floats(t, t.mass != nullptr)};
      const Extent pages{t.pages, 8 * entries}, tiers{t.tiers, entries};
      const Extent lengths{t.lengths, sizeof(int) * static_cast<std::size_t>(t.batch)};
      const std::size_t row = 2 * static_cast<std::size_t>(t.kv_heads) * t.head_dim;
      for (const Extent &written : {out, mass, parts})
      {
        bool over = overlaps(written, q) || overlaps(written, pages) || overlaps(written, tiers) ||
                    overlaps(written, lengths);
        for (int b = 0; t.held != nullptr && b < t.batch; ++b)
        {
          over = over || overlaps(written, {t.held[b].own_k, row}) ||
                 overlaps(written, {t.held[b].own_v, row});
        }
        if (over)
        {
          throw InvalidArgument("batch attention cannot write over its queries, tables or rows");
        }
      }
      if (overlaps(out, mass) || overlaps(out, parts) || overlaps(mass, parts))
      {
        throw InvalidArgument("batch attention's output, masses and partials write over one another");
      }
    }
  } // namespace

  std::size_t batch_attention_floats(const BatchAttention &t, bool with_mass)
  {
    check_batch(t);
    const std::size_t rows = static_cast<std::size_t>(t.batch) * t.heads;
    const Cut cut = cut_of(t.batch, t.max_pages, t.kv_heads, t.head_dim, t.window, t.sinks);
    return static_cast<std::size_t>(cut.most_parts) * t.heads * (t.head_dim + 2) +
           (with_mass ? rows * t.max_pages : 0);
  }

  void launch_batch_attention(const BatchAttention &t, hipStream_t stream)
  {
    check_batch(t);
    if (t.batch == 0)
    {
      return;
    }
    if (t.q == nullptr || t.out == nullptr ||
        (t.held == nullptr && (t.lengths == nullptr ||
                               (t.max_pages > 0 && (t.pages == nullptr || t.tiers == nullptr)))))
    {
      throw InvalidArgument("batch attention needs q, out, the page tables and the lengths");
    }
    if ((reinterpret_cast<std::uintptr_t>(t.q) | reinterpret_cast<std::uintptr_t>(t.out) |
         reinterpret_cast<std::uintptr_t>(t.partials)) % 16 != 0)
    {
      throw InvalidArgument("batch attention's q, out and partials must be 16-byte aligned");
    }
    if (t.mass != nullptr && t.partials == nullptr && t.max_pages > 0)
    {
      throw InvalidArgument("batch attention's masses need partials");
    }
    Cut cut = cut_of(t.batch, t.max_pages, t.kv_heads, t.head_dim, t.window, t.sinks);
    if (t.partials == nullptr)
    {
      cut.run_pages = std::max(t.max_pages, 1);
      cut.splits = 1;
    }
    else if (t.partials_floats < batch_attention_floats(t, t.mass != nullptr))
    {
      throw InvalidArgument("batch attention's partials need " +
                            std::to_string(batch_attention_floats(t, t.mass != nullptr)) +
                            " floats; got " +
                            std::to_string(t.partials_floats));
    }
    check_overlaps(t);
    BatchArgs a{};
    a.q = static_cast<const std::uint16_t *>(t.q);
    a.out = static_cast<std::uint16_t *>(t.out);
    a.mass = t.mass;
    a.pages = t.pages;
    a.tiers = t.tiers;
    a.lengths = t.lengths;
    a.max_pages = t.max_pages;
    a.heads = t.heads;
    a.kv_heads = t.kv_heads;
    a.group = t.heads / t.kv_heads;
    a.kv_block = cut.kv_block;
    a.window = t.window;
    a.sinks = t.sinks;
    a.run_pages = cut.run_pages;
    a.splits = cut.splits;
    a.scale = static_cast<float>(1.4426950408889634 / std::sqrt(static_cast<double>(t.head_dim)));
    const std::size_t rows = static_cast<std::size_t>(t.batch) * t.heads;
    float *parts = t.partials;
    if (cut.splits > 1)
    {
      a.parts_o = parts;
      a.parts_ml = parts + rows * cut.splits * t.head_dim;
      parts = a.parts_ml + rows * cut.splits * 2;
    }
    a.mass_from = parts;
    if (t.held == nullptr)
    {
      t.head_dim == 64 ? launch<64, false>(a, {}, t.batch, stream)
                       : launch<128, false>(a, {}, t.batch, stream);
      return;
    }
    // The sequences go with the launch, kBatchHeld at a time.
    const std::size_t per = static_cast<std::size_t>(t.heads);
    for (int at = 0; at < t.batch; at += kBatchHeld)
    {
      const int n = std::min(kBatchHeld, t.batch - at);
      BatchArgs part = a;
      part.q += at * per * t.head_dim;
      part.out += at * per * t.head_dim;
      if (part.mass != nullptr)
      {
        part.mass += at * per * t.max_pages;
        part.mass_from += at * per * t.max_pages;
      }
      Sequences<true> held{};
      std::copy(t.held + at, t.held + at + n, held.of);
      t.head_dim == 64 ? launch<64, true>(part, held, n, stream)
                       : launch<128, true>(part, held, n, stream);
    }
  }

} // namespace mi
