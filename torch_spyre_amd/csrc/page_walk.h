// How the attention of drafted tokens shares the pages of ragged sequences over
// the device, and the lane exchanges of its kernels.  The arguments A of such a
// kernel hold
//   ctx, counts (or null)   lengths of the B sequences, on the device
//   T, max_ctx, draft_keys  bounds on them
//   Hkv, by_hkv, row_blocks, by_blocks, ranges, by_ranges, min_per, min_cut, each
#pragma once

#include <hip/hip_runtime.h>

#include "fast_div.h"

namespace spyre_hip {

constexpr int kPage = 64;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

typedef float f32x4_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float xor32_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x), false, false);
  return fmaxf(__builtin_bit_cast(float, static_cast<unsigned>(r[0])), __builtin_bit_cast(float, static_cast<unsigned>(r[1])));
}

__device__ __forceinline__ float xor32_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x), false, false);
  return __builtin_bit_cast(float, static_cast<unsigned>(r[0])) + __builtin_bit_cast(float, static_cast<unsigned>(r[1]));
}

// The same over lanes l and l ^ 16.
__device__ __forceinline__ float xor16_max(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x), false, false);
  return fmaxf(__builtin_bit_cast(float, static_cast<unsigned>(r[0])), __builtin_bit_cast(float, static_cast<unsigned>(r[1])));
}

__device__ __forceinline__ float xor16_sum(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x), false, false);
  return __builtin_bit_cast(float, static_cast<unsigned>(r[0])) + __builtin_bit_cast(float, static_cast<unsigned>(r[1]));
}

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

__host__ __device__ __forceinline__ int pages_of(int tokens) { return tokens / kPage + (tokens % kPage != 0); }
// What a sequence holds.  bad: it breaks the max_context_len contract.
struct Seq {
  int ctx, n, pages;
  bool bad;
};

template <typename A>
__device__ __forceinline__ Seq seq_of(const A& a, int raw, int count) {
  Seq s;
  s.bad = raw > a.max_ctx;
  s.ctx = min(max(raw, 0), a.max_ctx);
  s.n = min(max(count, 0), a.T);
  s.pages = pages_of(s.ctx + (a.draft_keys ? s.n : 0));
  return s;
}

// Sequence b, the same for the wavefront (in scalar registers).
template <typename A>
__device__ __forceinline__ Seq seq_at(const A& a, int b) {
  return seq_of(a, __builtin_amdgcn_readfirstlane(a.ctx[b]),
                a.counts ? __builtin_amdgcn_readfirstlane(a.counts[b]) : a.T);
}

// Inclusive sums over the lanes of a wavefront.
__device__ __forceinline__ int scan64(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr 1, 2, 4, 8: within 16 lanes
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // lane 15 of a row to the next
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // lane 31 to the upper half
  return x;
}

// The largest over the lanes of a wavefront (none negative).
__device__ __forceinline__ int max64(int x) {
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false));
  return __builtin_amdgcn_readlane(x, 63);
}

// How the pages are shared out.  A (sequence, KV head) counts kStart units, what
// its beginning and end cost, and then one for each page; range r of `ranges` is
// the units [r per, (r + 1) per) of all, one (sequence, KV head) after the
// other.  A bound that would leave a piece of few pages moves to the
// (sequence, KV head)'s end: a part costs its join.  The lengths are data of
// the device, so every wavefront works out the sums itself; ragged batches are
// then as even as equal ones.  A range that holds only part of a (sequence, KV
// head) leaves a partial: in slot 1 that of the first part, in slot 0 that of
// any other.
// Lengths that another stream changes meanwhile give wrong results, as in any
// kernel, but no endless walk and no index beyond the buffers: hence the bounds
// that lengths at rest never meet.
// kStart: 64 sequences of 128 to 16384 tokens, longest first, took 237 us
// where pages alone were counted: a workgroup had 60 short ones.
constexpr int kStart = 4;

template <typename A>
struct PageWalk {
  int per, u, end;      // units
  int b, base, size;    // the sequence: its first unit / Hkv, its units a KV head
  Seq seq;              // what it holds
  bool uncut;           // range r is the (sequence, KV head)s [r each, (r + 1) each)
  // A sequence a lane: its lengths as they were given, its units a KV head.
  struct Lane {
    int ctx = 0, count = 0, size = 0;
  };
  __device__ __forceinline__ static Lane lane_of(const A& a, int b) {
    Lane x;
    if (b < a.B) {
      x.ctx = a.ctx[b], x.count = a.counts ? a.counts[b] : a.T;
      x.size = kStart + seq_of(a, x.ctx, x.count).pages;
    }
    return x;
  }
  // Units a KV head of all sequences and the largest one's; the first 64
  // sequences, one a lane.
  __device__ __forceinline__ static int total_of(const A& a, int lane, Lane& first64, int& largest) {
    int sum = 0, top = 0;
    first64 = lane_of(a, lane);
    for (int c = 0; c < a.B; c += 256) {
      int x[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) x[k] = c == 0 && k == 0 ? first64.size : lane_of(a, c + 64 * k + lane).size;
      sum += x[0] + x[1] + x[2] + x[3];
      top = max(max(top, max(x[0], x[1])), max(x[2], x[3]));
    }
    largest = max64(top);
    return __builtin_amdgcn_readlane(scan64(sum), 63);
  }
  // An equal share, but no smaller than a mean (sequence, KV head) cut into
  // parts of min_per pages, or uncut below min_cut.  Where a whole number of (sequence, KV head)s to a
  // range is within an eighth of it, none is cut: 16 x 8 of 8000 to 8192 tokens
  // and 512 rows, whose parts take 20 us to join.
  __device__ __forceinline__ void share(const A& a, int total, int largest) {
    const int mean = total / a.B, pages = mean - kStart, parts = pages < a.min_cut ? 1 : max(1, pages / a.min_per);
    per = max(static_cast<int>(fdiv(total * a.Hkv + a.ranges - 1, a.by_ranges)), (mean + parts - 1) / parts);
    uncut = a.each > 0 && static_cast<int64_t>(largest) * a.each <= per + per / 8;
  }
  // Pages that are too few for a piece.
  __device__ __forceinline__ int few() const { return min(max(per - kStart, 0) / 2, 4); }
  // The sequence of a unit (below the total).
  __device__ __forceinline__ void find(const A& a, int lane, const Lane& first64, int unit) {
    const int target = static_cast<int>(fdiv(unit, a.by_hkv));
    base = 0;
    for (int c = 0;; c += 64) {
      const Lane x = c == 0 ? first64 : lane_of(a, c + lane);
      const int sum = scan64(x.size);
      const uint64_t past = __builtin_amdgcn_ballot_w64(base + sum > target);
      if (past || c + 64 >= a.B) {
        const int i = past ? __builtin_ctzll(past) : (a.B - 1) % 64;
        b = c + i;
        take(a, x, i);
        base += __builtin_amdgcn_readlane(sum, i) - size;
        return;
      }
      base += __builtin_amdgcn_readlane(sum, 63);
    }
  }
  // The sequence of lane i.
  __device__ __forceinline__ void take(const A& a, const Lane& x, int i) {
    seq = seq_of(a, __builtin_amdgcn_readlane(x.ctx, i), __builtin_amdgcn_readlane(x.count, i));
    size = kStart + seq.pages;
  }
  // A bound where it belongs, after find() of it.
  __device__ __forceinline__ int placed(const A& a, int unit) const {
    const uint32_t in = unit - base * a.Hkv, at = in % static_cast<uint32_t>(size);
    const int g0 = unit - static_cast<int>(at), g1 = g0 + size;
    return static_cast<int>(at) - kStart <= few() ? g0 : g1 - unit <= few() ? g1 : unit;
  }
  // Range r; false if it is empty.
  __device__ __forceinline__ bool start(const A& a, int lane, int r) {
    Lane x;
    int largest;
    const int total = total_of(a, lane, x, largest), units = total * a.Hkv;
    share(a, total, largest);
    if (uncut) {
      const int first = r * a.each, at0 = static_cast<int>(fdiv(first, a.by_hkv)), kvh = first - at0 * a.Hkv;
      to(a, lane, x, at0);
      u = base * a.Hkv + kvh * size;
      end = u;
      for (int k = 0, at = at0, h = kvh; k < a.each; ++k) {
        end += at == at0 ? size : kStart + seq_at(a, at).pages;
        if (++h == a.Hkv) h = 0, ++at;
      }
      return true;
    }
    u = r * per;
    if (u >= units) return false;
    end = units;
    if (u + per < units) {
      find(a, lane, x, u + per);
      end = placed(a, u + per);
    }
    find(a, lane, x, u);
    u = placed(a, u);
    if (u >= end) return false;
    if (u == (base + size) * a.Hkv) next_sequence(a);
    return true;
  }
  __device__ __forceinline__ void next_sequence(const A& a) {
    base += size;
    b = min(b + 1, a.B - 1);
    seq = seq_at(a, b);
    size = kStart + seq.pages;
  }
  // To sequence i.
  __device__ __forceinline__ void to(const A& a, int lane, const Lane& first64, int i) {
    int before = 0;
    Lane x;
    for (int c = 0; c <= i; c += 64) {
      x = c == 0 ? first64 : lane_of(a, c + lane);
      before += c + lane < i ? x.size : 0;
    }
    b = i;
    base = __builtin_amdgcn_readlane(scan64(before), 63);
    take(a, x, i % 64);
  }
  // Sequence i and the shares, for parts_of().
  __device__ __forceinline__ void seek(const A& a, int lane, int i) {
    Lane x;
    int largest;
    const int total = total_of(a, lane, x, largest);
    share(a, total, largest);
    to(a, lane, x, i);
  }
  // The ranges that hold parts of a KV head of the sequence: r0 the first one,
  // r0 + 1 .. r1 the others; r1 <= r0 where one range holds it whole.
  __device__ __forceinline__ void parts_of(const A& a, int kvh, int& r0, int& r1) const {
    const int g0 = base * a.Hkv + kvh * size, g1 = g0 + size;
    r0 = min((g0 + kStart + few()) / per, a.ranges - 1);
    r1 = uncut ? r0 : min((g1 - few() - 1) / per, a.ranges - 1);
  }
};

// A piece of a range: pages [page0, page1) of a (sequence, KV head).
struct Piece {
  int kvh, page0, page1;
  bool whole;   // all of them
  int slot;     // else its partial's
};

template <typename A>
__device__ __forceinline__ Piece piece_of(const A& a, const PageWalk<A>& w) {
  Piece p;
  const int in = w.u - w.base * a.Hkv;
  p.kvh = min(static_cast<uint32_t>(in) / static_cast<uint32_t>(w.size), static_cast<uint32_t>(a.Hkv - 1));
  const int at = in - p.kvh * w.size;
  p.page0 = max(at - kStart, 0);
  p.page1 = min(w.size, at + w.end - w.u) - kStart;
  p.whole = at == 0 && p.page1 == w.size - kStart;
  p.slot = at == 0 ? 1 : 0;
  return p;
}

// After it.
template <typename A>
__device__ __forceinline__ void advance(const A& a, PageWalk<A>& w, const Piece& p) {
  w.u = max(w.base * a.Hkv + p.kvh * w.size + kStart + p.page1, w.u + 1);
  if (w.u < w.end && p.kvh == a.Hkv - 1 && p.page1 == w.size - kStart) w.next_sequence(a);
}

// The range and the row block of a workgroup.  The row blocks of one range
// read the same pages: 8 workgroups apart, they meet in one XCD's L2.
template <typename A>
__device__ __forceinline__ void place_of(const A& a, int& range, int& rb) {
  const uint32_t lo8 = blockIdx.x & 7, hi = blockIdx.x >> 3, q = fdiv(hi, a.by_blocks);
  rb = static_cast<int>(hi - q * a.row_blocks);
  range = static_cast<int>(q * 8 + lo8);
}

// Joins the parts r0 .. r1 of 4 features of a row, 8 loads in flight.
template <typename Load>
__device__ __forceinline__ void merge_parts(int r0, int r1, float& M, float& L, f32x4_t& acc, Load load) {
  constexpr int G = 8;
  for (int c = r0; c <= r1; c += G) {
    float m[G], l[G];
    f32x4_t x[G];
#pragma unroll
    for (int k = 0; k < G; ++k) load(min(c + k, r1), m[k], l[k], x[k]);  // past r1 the last one again
    float mc = M;
#pragma unroll
    for (int k = 0; k < G; ++k) mc = fmaxf(mc, m[k]);
    const float f0 = M == -INFINITY ? 0.f : exp2_of(M - mc);
    L *= f0;
    acc *= f0;
#pragma unroll
    for (int k = 0; k < G; ++k) {
      if (c + k > r1) break;
      const float f = m[k] == -INFINITY ? 0.f : exp2_of(m[k] - mc);
      L += m[k] == -INFINITY ? l[k] : l[k] * f;  // l without a reference is 0, or NaN
      if (m[k] != -INFINITY) acc += x[k] * f;
    }
    M = mc;
  }
}

// The same where r0 and r1 are the wavefront's: no part is loaded twice (latent attention of 64 x
// 128-16384 tokens 123.8 us, so 122.9; 600 x 10-900 93.9, 93.3).
template <typename Load>
__device__ __forceinline__ void merge_parts_once(int r0, int r1, float& M, float& L, f32x4_t& acc, Load load) {
  constexpr int G = 4;
  for (int c = r0; c <= r1; c += G) {
    float m[G], l[G];
    f32x4_t x[G];
#pragma unroll
    for (int k = 0; k < G; ++k) {
      m[k] = -INFINITY, l[k] = 0.f, x[k] = f32x4_t{0.f, 0.f, 0.f, 0.f};
      if (c + k <= r1) load(c + k, m[k], l[k], x[k]);
    }
    float mc = M;
#pragma unroll
    for (int k = 0; k < G; ++k) mc = fmaxf(mc, m[k]);
    const float f0 = M == -INFINITY ? 0.f : exp2_of(M - mc);
    L *= f0;
    acc *= f0;
#pragma unroll
    for (int k = 0; k < G; ++k) {
      const float f = m[k] == -INFINITY ? 0.f : exp2_of(m[k] - mc);
      L += m[k] == -INFINITY ? l[k] : l[k] * f;  // l without a reference is 0, or NaN
      if (m[k] != -INFINITY) acc += x[k] * f;
    }
    M = mc;
  }
}

}  // namespace spyre_hip
