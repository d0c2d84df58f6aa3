// Attention of prompts whose keys and values have been expanded from latent vectors
// (spyre_latent_attn): every head has keys of D features and, behind them, the 64
// rotated ones that all heads share, and values of D.
//   score(t) = scale (q_h . k_(t,h) + s_h . r_t),  out = softmax(score) v_h
// Sequence b has ctx[b] keys before its n[b] queries; query i attends the keys t <=
// ctx[b] + i.  Rows from n[b] on are zeros with lse -inf.
//
// A wavefront has 32 query rows of one (sequence, head), a workgroup W of them, which
// share tiles of 64 keys through LDS, the next tile on its way while one is used:
//   S^T[tok, row] = K[tok, :] Q^T[:, row]      K's rows as they lie, the shared ones after the head's
//   O^T[d, row] += V^T[d, tok] P^T[tok, row]   V^T by transposing reads
// K's rows are permuted so that a lane's scores are the 16 tokens that its half of the
// wavefront wants in the second product: P stays where it is.
// A tile's exponentials cost as much time as its products, so the two run side by side: the
// first product of the next tile between the exponentials of this one, the largest score of
// the next one between the second products of this one.  K is a tile ahead of V for it.
// Few rows with many keys are split over the keys and joined by a second kernel.
//
// Measured: 4096 tokens x 32 heads x 128 features 215 us, 4 x 512 rows over 2000-8000 keys 328-345
// us, from device to device (770-810 TFLOP/s).  Counters of the latter: of the cycles in which the device has
// any wavefronts the matrix cores are busy for 37 %, of those in which a SIMD has its own for 49 %
// (row blocks end at different times: 77 %); wavefronts wait in 36 % of their cycles and have an instruction
// that cannot issue in 24 %, 3 % for LDS.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "fast_div.h"
#include "lds_dma.h"
#include "page_walk.h"
#include "spyre_common.h"

namespace {

using namespace spyre_hip;

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr int kRope = 64;
constexpr int kRows = 32;      // query rows of a wavefront
constexpr int kKeys = 64;      // keys of a tile
constexpr int kStick = kKeys * 64 * 2;  // bytes of 64 features of a tile
constexpr int kNoWhere = 0x7fffff00;    // the buffers' extent: an offset from here on reads zeros
// As in the paged latent attention.
constexpr float kBelow = 7.f, kAbove = 15.f;

struct PromptArgs {
  const _Float16 *q, *qr, *k, *kr, *v;
  int64_t q_sb, q_st, q_sh, qr_sb, qr_st, qr_sh, k_sb, k_st, k_sh, kr_sb, kr_st, v_sb, v_st, v_sh;
  const int32_t *ctx, *counts;
  _Float16* out;  // [B, T, H, D]
  float* lse;     // [B, T, H] or null
  float* ws;  // splits > 1: O [splits][B, T, H][D], then (m, l) [splits][B, T, H]
  int B, T, H, keys, pairs, blocks, splits;  // pairs: (sequence, head)s; blocks: of rows, to each
  float scale_log2;  // above 0
  uint32_t q_sign;   // 0x80008000: of the other sign
  FastDiv by_h, by_octets, by_splits;
};

__device__ __forceinline__ int token_of(int m) {
  return 16 * ((m >> 2) & 1) + 8 * (m >> 4) + 4 * ((m >> 3) & 1) + (m & 3);
}

// Unit u (16 bytes) of token t lies at u ^ key(t) of its 128 bytes in LDS: neither the
// reads of K's rows (32 tokens in token_of's order x 2 units) nor the transposing ones of V's (2
// x 4 tokens x 4 units) then meet in a bank: 4 and 2 cycles a read (measured).
__device__ __forceinline__ int key_of(int t) { return (t & 2) << 1 | ((t >> 2) & 1) | ((t >> 3) & 2); }

// A lane index whose addresses are formed where they are used, not kept through the loop.
__device__ __forceinline__ int here(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

template <int D, int W>
__global__ __launch_bounds__(W * 64, 2) void prompt_kernel(PromptArgs a) {
  constexpr int KS = D / 64 + 1, VS = D / 64;  // sticks of K and V
  constexpr int K_TILE = KS * kStick, V_TILE = VS * kStick, V_AT = 2 * K_TILE;
  constexpr int NQ = (D + kRope) / 16;
  constexpr int DT = D / 32;
  constexpr int PARTS = 8 / W;  // chunks (8 tokens of a stick) of a stick to a wavefront
  __shared__ __align__(16) uint8_t s_mem[2 * (K_TILE + V_TILE)];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
  const int col = lane & 31, half = lane >> 5;
  // A (sequence, head) stays in one XCD, the row blocks of most keys first: begun last, they
  // would run on alone (4096 tokens x 32 heads 215 us; one (sequence, head) after the other 285).
  // Equal shares of all tiles, cut within row blocks and joined, measured no better (4 x 512 rows
  // over 2000-8000 keys 338 us, this 335; 4096 tokens 240): a tile then took longer.
  const uint32_t js = blockIdx.x >> 3, j = fdiv(js, a.by_splits), split = js - j * a.splits;
  const uint32_t block = fdiv(j, a.by_octets), pair = (j - block * ((a.pairs + 7) / 8)) * 8 + (blockIdx.x & 7);
  if (pair >= static_cast<uint32_t>(a.pairs)) return;
  const int b = static_cast<int>(fdiv(pair, a.by_h)), h = static_cast<int>(pair) - b * a.H;
  const int block0 = (a.blocks - 1 - static_cast<int>(block)) * (W * kRows);
  const int raw = __builtin_amdgcn_readfirstlane(a.ctx[b]);
  const int n = a.counts ? min(max(__builtin_amdgcn_readfirstlane(a.counts[b]), 0), a.T) : a.T;
  const int ctx = min(max(raw, 0), a.keys), total = min(ctx + n, a.keys);
  const bool bad = max(raw, 0) > a.keys - n;  // fewer keys than the lengths say
  const int row0 = block0 + wave * kRows;
  // Keys of the workgroup's rows, of this wavefront's, and those that all rows of
  // the workgroup attend; tiles [first, tiles) of the split, up to `mine` of this wavefront.
  const int most = block0 < n ? min(total, ctx + block0 + W * kRows) : 0;
  const int all = min(ctx + block0 + 1, total);
  const int every = (most + kKeys - 1) / kKeys;
  const int first = static_cast<int>(static_cast<int64_t>(every) * split / a.splits);
  const int tiles = static_cast<int>(static_cast<int64_t>(every) * (split + 1) / a.splits);
  const int mine = min(tiles, row0 < n ? (min(total, ctx + row0 + kRows) + kKeys - 1) / kKeys : 0);

  const uint32_t lds0 = lds_address(s_mem);
  const _Float16 *kp = a.k + b * a.k_sb + h * a.k_sh, *rp = a.kr + b * a.kr_sb, *vp = a.v + b * a.v_sb + h * a.v_sh;
  // Load x of a wavefront's KL of tile t's K, or (x from KL on) KL + VL of its V: 8 tokens of a
  // stick.  Tokens that do not exist, and all of tiles from `tiles` on, are zeros.
  constexpr int KL = KS * PARTS, VL = VS * PARTS;
  auto load = [&](int x, int t) {
    const bool of_v = x >= KL;
    const int stick = of_v ? (x - KL) / PARTS : x / PARTS, chunk = x % PARTS * W + wave;
    const _Float16* base = of_v ? vp : stick == D / 64 ? rp : kp;
    const int64_t st = of_v ? a.v_st : stick == D / 64 ? a.kr_st : a.k_st;
    const int ln = here(lane), tok = chunk * 8 + ln / 8, left = t < tiles ? total - t * kKeys : 0;
    const uint32_t off = tok * static_cast<uint32_t>(st) * 2 + ((ln & 7) ^ key_of(tok)) * 16;
    const uint32_t to = of_v ? V_AT + (t & 1) * V_TILE : (t & 1) * K_TILE;
    dma16(dma_buffer(base + static_cast<int64_t>(t) * kKeys * st, kNoWhere), lds0 + to + stick * kStick + chunk * 1024,
          tok < left ? off : kNoWhere, !of_v && stick == D / 64 ? 0 : stick * 128);
  };
  auto load_k = [&](int t) {
#pragma unroll
    for (int x = 0; x < KL; ++x) load(x, t);
  };
  auto load_v = [&](int t) {
#pragma unroll
    for (int x = KL; x < KL + VL; ++x) load(x, t);
  };
  if (first < tiles) {
    load_k(first);
    load_v(first);
    load_k(first + 1);
  }

  f16x8 qf[NQ];
  {
    const int64_t qi = row0 + col < n ? row0 + col : 0;
    const _Float16* x = a.q + b * a.q_sb + qi * a.q_st + h * a.q_sh + 8 * half;
    const _Float16* xr = a.qr + b * a.qr_sb + qi * a.qr_st + h * a.qr_sh + 8 * half;
#pragma unroll
    for (int s = 0; s < NQ; ++s)
      qf[s] = __builtin_bit_cast(f16x8, *reinterpret_cast<const u32x4*>(16 * s < D ? x + 16 * s : xr + 16 * s - D) ^ a.q_sign);
#pragma unroll
    for (int s = 0; s < NQ; ++s) asm volatile("" : "+v"(qf[s]));  // waits here: in the loop it would for the tiles on their way
  }
  const int k_tok = token_of(col);
  const int k_lane = k_tok * 128 + ((half ^ key_of(k_tok)) * 16);
  // V^T: 4 features of token 16 half + lane % 16 / 4; the key of tokens 8 and 32 further is the
  // same, odd tiles and tokens 4 further turn the unit's bits 2 and 0.
  const int tv = 16 * half + (lane & 15) / 4;
  const int v_lane = V_AT + tv * 128 + (((2 * ((lane >> 4) & 1) + ((lane >> 1) & 1)) ^ key_of(tv)) * 16) + 8 * (lane & 1);
  auto tr = [&](int at) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(s_mem + at));
  };

  f32x16 o[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int x = 0; x < 16; ++x) o[dt][x] = 0.f;
  float m = -INFINITY, l = 0.f;
  f32x16 sc[2];  // a tile's scores before the scale: x of sc[tb] is token 32 tb + 16 half + x
  f16x8 w[4];    // its weights, in the same order

  // Reading ahead, in this order; the scheduler would read each operand when it is due.
  constexpr int kAhead = 4, kVAhead = 2, NK = 2 * NQ, NV = 4 * DT;
  // The first product of tile t (QK) beside the weights of the one before it (EXP), whose scores
  // are then this one's.  Weights round to fp16 for the second product (a relative 2^-12 on
  // average); their sum stays in fp32.
  // Between them (EXP) go the loads of the tiles that follow, K of t + 1 and V of t: at once they
  // would take the address unit for a quarter of a tile's time, with every wavefront waiting.
  auto products_and_weights = [&](int t, auto qk_tag, auto exp_tag) {
    constexpr bool QK = decltype(qk_tag)::value, EXP = decltype(exp_tag)::value;
    const int kb = (t & 1) * K_TILE + k_lane;
    const int k_at[4] = {kb, kb ^ 32, kb ^ 64, kb ^ 96};
    auto k_of = [&](int x) {
      return *reinterpret_cast<const f16x8*>(s_mem + k_at[x / 2 % 4] + x / 8 * kStick + x % 2 * (32 * 128));
    };
    const float mu = m == -INFINITY ? 0.f : m;  // a row that has attended nothing yet: weights 0
    f32x16 acc[2] = {};
    f16x8 kf[kAhead];
    if constexpr (QK)
#pragma unroll
      for (int x = 0; x < kAhead; ++x) kf[x] = k_of(x);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int x = 0; x < NK; ++x) {
      if constexpr (QK) {
        acc[x % 2] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[x % kAhead], qf[x / 2], acc[x % 2], 0, 0, 0);
        if (x + kAhead < NK) kf[x % kAhead] = k_of(x + kAhead);
      }
      if constexpr (EXP)
#pragma unroll
        for (int y = 32 * x / NK; y < 32 * (x + 1) / NK; ++y) {
          const float e = exp2_of(__builtin_fmaf(sc[y / 16][y % 16], a.scale_log2, -mu));
          l += e;
          w[y / 8][y % 8] = static_cast<_Float16>(e);
        }
      if (EXP && x % 2 == 1 && x / 2 < KL + VL) load(x / 2, x / 2 < KL ? t + 1 : t);
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (QK) sc[0] = acc[0], sc[1] = acc[1];
  };
  // The second product of tile t (PV) beside the largest of the scores (MAX).
  auto second = [&](int t, auto pv_tag, auto max_tag) -> float {
    constexpr bool PV = decltype(pv_tag)::value, MAX = decltype(max_tag)::value;
    const int vb = (t & 1) * V_TILE + v_lane;
    auto v_of = [&](int x) {  // tile x % DT, tokens 32 (x / DT / 2) + 16 half + 8 (x / DT % 2) ..
      const int dt = x % DT, at = dt / 2 * kStick + (32 * (x / DT / 2) + 8 * (x / DT % 2)) * 128;
      const s16x4 lo = tr((dt & 1 ? vb ^ 64 : vb) + at), hi = tr((dt & 1 ? vb ^ 80 : vb ^ 16) + at + 4 * 128);
      return __builtin_bit_cast(f16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    };
    float mx = -INFINITY;
    f16x8 vf[kVAhead];
    if constexpr (PV)
#pragma unroll
      for (int x = 0; x < kVAhead; ++x) vf[x] = v_of(x);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int x = 0; x < NV; ++x) {
      if constexpr (PV) {
        o[x % DT] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[x % kVAhead], w[x / DT], o[x % DT], 0, 0, 0);
        if (x + kVAhead < NV) vf[x % kVAhead] = v_of(x + kVAhead);
      }
      if constexpr (MAX)
#pragma unroll
        for (int y = 32 * x / NV; y < 32 * (x + 1) / NV; ++y) mx = fmaxf(mx, sc[y / 16][y % 16]);
      __builtin_amdgcn_sched_barrier(0);
    }
    return mx;
  };
  static_assert(KL + VL <= NK / 2, "every load has its place");
  std::true_type yes;
  std::false_type no;
  // Of tile t's scores, before their weights: those that rows do not attend, the reference.
  auto settle = [&](int t, float mx) {
    if (t * kKeys + kKeys > all) {
      const int ln = here(lane), last = min(ctx + row0 + ln % 32, total - 1) - t * kKeys - 16 * (ln / 32);
      mx = -INFINITY;
#pragma unroll
      for (int x = 0; x < 32; ++x) {
        sc[x / 16][x % 16] = 32 * (x / 16) + x % 16 > last ? -INFINITY : sc[x / 16][x % 16];
        mx = fmaxf(mx, sc[x / 16][x % 16]);
      }
    }
    mx = xor32_max(mx) * a.scale_log2;
    if (__any(mx > m + kAbove)) {
      const float mn = mx > m + kAbove ? mx - kBelow : m;  // a row's own: what others attend does not turn its roundings
      const float alpha = m == -INFINITY ? 0.f : exp2_of(m - mn);
      m = mn;
      l *= alpha;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int x = 0; x < 16; ++x) o[dt][x] *= alpha;
    }
  };

  // What a row does not attend must not meet its weight of 0 in the second product.  So numbers of
  // such values (`odd`: keys of tile t that hold any) that are a NaN or an infinity are added by
  // themselves to the rows that attend them, and are zeros in LDS from then on.
  auto reach = [&](int t, uint64_t odd) {
    const int ln = here(lane), last = min(ctx + row0 + ln % 32, total - 1) - t * kKeys;
#pragma unroll 1
    for (; odd; odd &= odd - 1) {
      const int tok = __builtin_ctzll(odd), x = 16 * (tok / 32) + tok % 16;
      float p = 0.f;  // the key's weight: in one half of the wavefront
#pragma unroll
      for (int y = 0; y < 32; ++y) p = y == x ? static_cast<float>(w[y / 8][y % 8]) : p;
      p = __shfl(p, ln % 32 + (tok & 16) * 2, 64);
      const uint8_t* v = s_mem + V_AT + (t & 1) * V_TILE + tok * 128 + 8 * (ln / 32);
#pragma unroll
      for (int y = 0; y < 4 * DT; ++y) {
        const f16x4 z = *reinterpret_cast<const f16x4*>(v + y / 8 * kStick + ((y % 8) ^ key_of(tok)) * 16);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float f = static_cast<float>(z[e]);
          o[y / 4][4 * (y % 4) + e] += tok <= last && !(__builtin_fabsf(f) < INFINITY) ? p * f : 0.f;
        }
      }
    }
  };
  auto clear = [&](int t, uint64_t odd) {
    const int tok = here(lane);
    if (!((odd >> tok) & 1)) return;
#pragma unroll 1
    for (int u = 0; u < VS * 64; ++u) {
      uint16_t* x = reinterpret_cast<uint16_t*>(s_mem + V_AT + (t & 1) * V_TILE + tok * 128 + u / 64 * kStick) + u % 64;
      if ((*x & 0x7c00) == 0x7c00) *x = 0;
    }
  };

  for (int t = first; t < tiles; ++t) {
    dma_wait();
    __syncthreads();  // K of t + 1 and V of t are there (at first K of t, too); their places of before are read
    if (t == first && t < mine) {
      products_and_weights(t, yes, no);
      settle(t, second(t, no, yes));
    }
    if (t == first) __syncthreads();
    uint64_t odd = 0;  // keys whose values hold a NaN or an infinity, of those that not all rows attend
    if (t * kKeys + kKeys > all) {
      // Every wavefront looks at all 64 rows, one a lane.
      const int tok = here(lane), at = t * kKeys + tok;
      const uint8_t* x = s_mem + V_AT + (t & 1) * V_TILE + tok * 128;
      uint32_t found = 0;
      if (at >= all && at < total)
        for (int s = 0; s < VS; ++s)
#pragma unroll
          for (int u = 0; u < 8; ++u) {
            const u32x4 y = *reinterpret_cast<const u32x4*>(x + s * kStick + (u ^ (tok & 7)) * 16);
#pragma unroll
            for (int e = 0; e < 4; ++e) found |= (y[e] & 0x7c007c00u) + 0x04000400u;
          }
      odd = __ballot((found & 0x80008000u) != 0);
    }
    const bool more = t + 1 < mine;
    if (t >= mine) {  // none of its rows' keys (the barriers are all of a step's)
      load_k(t + 2);
      load_v(t + 1);
    } else if (more) {
      products_and_weights(t + 1, yes, yes);
    } else {
      products_and_weights(t + 1, no, yes);
    }
    if (odd) {  // the same for all wavefronts
      if (t < mine) reach(t, odd);
      __syncthreads();
      if (wave == 0) clear(t, odd);
      __syncthreads();
    }
    if (t >= mine) continue;
    if (more)
      settle(t + 1, second(t, yes, yes));
    else
      second(t, yes, no);
  }
  dma_wait();  // (those behind the last tile: nothing is on its way into LDS that is given up)
  l = xor32_sum(l);
  const int i = row0 + here(col);
  const bool live = i < n;
  if (!live) l = 0.f;
  if (bad && live) l = NAN;
  if (i >= a.T) return;
  const int64_t rows = static_cast<int64_t>(a.B) * a.T * a.H, at = (static_cast<int64_t>(b) * a.T + i) * a.H + h;
  if (a.splits > 1) {
    float* part = a.ws + (split * rows + at) * D;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int x = 0; x < 4; ++x)
        *reinterpret_cast<f32x4_t*>(part + 32 * dt + 8 * x + 4 * half) =
            f32x4_t{o[dt][4 * x], o[dt][4 * x + 1], o[dt][4 * x + 2], o[dt][4 * x + 3]};
    if (half == 0) {
      float* ml = a.ws + a.splits * rows * D + (split * rows + at) * 2;
      ml[0] = live ? m : -INFINITY, ml[1] = l;
    }
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      f16x4 y;
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = static_cast<_Float16>(l == 0.f ? 0.f : o[dt][4 * x + e] * inv);
      *reinterpret_cast<f16x4*>(a.out + at * D + 32 * dt + 8 * x + 4 * half) = y;
    }
  if (a.lse && half == 0) a.lse[at] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
}

// Joins the splits of a row, a thread 4 features.
template <int D>
__global__ __launch_bounds__(256) void prompt_join_kernel(PromptArgs a) {
  const int64_t rows = static_cast<int64_t>(a.B) * a.T * a.H, u = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (u >= rows * (D / 4)) return;
  const int64_t at = u / (D / 4);
  const int d = 4 * static_cast<int>(u % (D / 4));
  float M = -INFINITY, L = 0.f;
  f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
  merge_parts_once(0, a.splits - 1, M, L, acc, [&](int s, float& m, float& l, f32x4_t& x) {
    const float* ml = a.ws + a.splits * rows * D + (s * rows + at) * 2;
    m = ml[0], l = ml[1];
    x = *reinterpret_cast<const f32x4_t*>(a.ws + (s * rows + at) * D + d);
  });
  const float inv = L == 0.f ? 0.f : 1.f / L;
  f16x4 y;
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = static_cast<_Float16>(L == 0.f ? 0.f : acc[e] * inv);
  *reinterpret_cast<f16x4*>(a.out + at * D + d) = y;
  if (a.lse && d == 0) a.lse[at] = L == 0.f ? -INFINITY : (M + log2f(L)) * kLn2;
}

struct Plan {
  int waves, blocks, splits;
  size_t ws_bytes;
};

Plan plan_of(int B, int T, int H, int D, int keys) {
  Plan p;
  // 8 wavefronts read a tile for 256 rows, 4 leave room for a second workgroup: 512 rows over
  // 2000-8000 keys 335 us (4: 374), 128 rows over the same 125 (4: 118), 16 rows 103 (4: 83).
  p.waves = T <= 4 * kRows ? 4 : 8;
  p.blocks = (T + p.waves * kRows - 1) / (p.waves * kRows);
  const int64_t groups = static_cast<int64_t>(B) * H * p.blocks, slots = p.waves == 8 ? 256 : 512;
  const int64_t tiles = (static_cast<int64_t>(keys) + kKeys - 1) / kKeys;
  p.splits = static_cast<int>(std::max<int64_t>(1, std::min(slots / std::max<int64_t>(groups, 1), tiles / 4)));
  p.ws_bytes = p.splits == 1 ? 0 : static_cast<size_t>(p.splits) * B * T * H * (D + 2) * 4;
  return p;
}

bool sizes_ok(int B, int T, int H, int keys) {
  return B >= 0 && T > 0 && H > 0 && keys >= 0 && keys < (1 << 30) && T < (1 << 30) &&
         static_cast<double>(B) * T * H < 4e9;
}

}  // namespace

extern "C" size_t spyre_latent_attn_workspace_bytes(int B, int T, int H, int D, int keys) {
  if (!sizes_ok(B, T, H, keys)) return 0;
  return plan_of(B, T, H, D, keys).ws_bytes;
}

extern "C" int spyre_latent_attn(const void* q, const int64_t* q_strides, const void* q_rope, const int64_t* q_rope_strides,
                                 const void* k, const int64_t* k_strides, const void* k_rope, const int64_t* k_rope_strides,
                                 const void* v, const int64_t* v_strides, const int32_t* context_lens, const int32_t* new_lens,
                                 void* out, float* lse, void* workspace, size_t workspace_bytes, int B, int T, int H, int D,
                                 int keys, float scale, void* stream) {
  spyre_hip::clear_error();
  SPYRE_REQUIRE(D == 64 || D == 128, SPYRE_EUNSUPPORTED, "head_dim %d not in {64, 128}", D);
  SPYRE_REQUIRE(B >= 0 && T >= 0 && H > 0 && keys >= 0, SPYRE_EINVAL, "bad sizes B=%d T=%d H=%d keys=%d", B, T, H, keys);
  if (B == 0 || T == 0) return SPYRE_OK;
  SPYRE_REQUIRE(q && q_strides && q_rope && q_rope_strides && k_strides && k_rope_strides && v_strides && context_lens && out &&
                    (keys == 0 || (k && k_rope && v)),
                SPYRE_EINVAL, "null pointer argument");
  auto aligned = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  SPYRE_REQUIRE(aligned(q) && aligned(q_rope) && aligned(k) && aligned(k_rope) && aligned(v) && aligned(out), SPYRE_EINVAL,
                "q, k, v and out must be 16-byte aligned");
  for (int i = 0; i < 3; ++i)
    SPYRE_REQUIRE(q_strides[i] % 8 == 0 && q_rope_strides[i] % 8 == 0 && k_strides[i] % 8 == 0 && v_strides[i] % 8 == 0 &&
                      (i == 2 || k_rope_strides[i] % 8 == 0),
                  SPYRE_EINVAL, "strides must be multiples of 8 elements");
  // A tile's offsets in 31 bits.
  constexpr int64_t kMost = (int64_t{1} << 30) / (2 * kKeys);
  SPYRE_REQUIRE(k_strides[1] >= 0 && k_strides[1] < kMost && v_strides[1] >= 0 && v_strides[1] < kMost && k_rope_strides[1] >= 0 &&
                    k_rope_strides[1] < kMost,
                SPYRE_EUNSUPPORTED, "token strides of keys and values must be below 2^23 elements");
  SPYRE_REQUIRE(sizes_ok(B, T, H, keys), SPYRE_EUNSUPPORTED, "too many rows or tokens");
  const Plan p = plan_of(B, T, H, D, keys);
  SPYRE_REQUIRE(p.ws_bytes == 0 || (workspace && workspace_bytes >= p.ws_bytes && aligned(workspace)), SPYRE_ENOSPC,
                "workspace holds %zu bytes, need %zu (16-byte aligned)", workspace ? workspace_bytes : 0, p.ws_bytes);
  PromptArgs a{};
  a.q = static_cast<const _Float16*>(q), a.q_sb = q_strides[0], a.q_st = q_strides[1], a.q_sh = q_strides[2];
  a.qr = static_cast<const _Float16*>(q_rope), a.qr_sb = q_rope_strides[0], a.qr_st = q_rope_strides[1], a.qr_sh = q_rope_strides[2];
  a.k = static_cast<const _Float16*>(k), a.k_sb = k_strides[0], a.k_st = k_strides[1], a.k_sh = k_strides[2];
  a.kr = static_cast<const _Float16*>(k_rope), a.kr_sb = k_rope_strides[0], a.kr_st = k_rope_strides[1];
  a.v = static_cast<const _Float16*>(v), a.v_sb = v_strides[0], a.v_st = v_strides[1], a.v_sh = v_strides[2];
  a.ctx = context_lens, a.counts = new_lens, a.out = static_cast<_Float16*>(out), a.lse = lse;
  a.ws = static_cast<float*>(workspace);
  a.B = B, a.T = T, a.H = H, a.keys = keys, a.blocks = p.blocks, a.splits = p.splits;
  // Scores are masked before the scale, so that it is above 0: its sign goes to q, and 0 is as
  // good as the smallest number.
  a.scale_log2 = std::max(std::fabs(scale) * kLog2e, 1.17549435e-38f);
  if (std::isnan(scale)) a.scale_log2 = scale;
  a.q_sign = std::signbit(scale) ? 0x80008000u : 0u;
  const int64_t pairs = static_cast<int64_t>(B) * H, grid = (pairs + 7) / 8 * 8 * p.blocks * p.splits;
  SPYRE_REQUIRE(grid < (int64_t{1} << 31), SPYRE_EUNSUPPORTED, "too many rows");
  a.pairs = static_cast<int>(pairs);
  a.by_h = make_fastdiv(static_cast<uint32_t>(H)), a.by_octets = make_fastdiv(static_cast<uint32_t>((pairs + 7) / 8));
  a.by_splits = make_fastdiv(static_cast<uint32_t>(a.splits));
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 blocks(static_cast<uint32_t>(grid));
  auto go = [&](auto d) {
    constexpr int DD = decltype(d)::value;
    p.waves == 8 ? prompt_kernel<DD, 8><<<blocks, 512, 0, st>>>(a) : prompt_kernel<DD, 4><<<blocks, 256, 0, st>>>(a);
    if (p.splits > 1) {
      const int64_t units = static_cast<int64_t>(B) * T * H * (DD / 4);
      prompt_join_kernel<DD><<<dim3(static_cast<uint32_t>((units + 255) / 256)), 256, 0, st>>>(a);
    }
  };
  D == 128 ? go(std::integral_constant<int, 128>{}) : go(std::integral_constant<int, 64>{});
  const hipError_t e = hipGetLastError();
  SPYRE_REQUIRE(e == hipSuccess, SPYRE_EHIP, "latent prompt attention launch failed: %s", hipGetErrorString(e));
  return SPYRE_OK;
}
