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

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

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
  int B, T, H, keys, pairs, blocks;  // pairs: (sequence, head)s; blocks: of rows, to each
  float scale_log2;
  FastDiv by_h, by_blocks;
};

__device__ __forceinline__ int token_of(int m) {
  return 16 * ((m >> 2) & 1) + 8 * (m >> 4) + 4 * ((m >> 3) & 1) + (m & 3);
}

// Unit u (16 bytes) of token t lies at u ^ key(t) of its 128 bytes in LDS: neither the
// reads of K's rows (32 tokens in token_of's order x 2 units) nor the transposing ones of V's (2
// x 4 tokens x 4 units) then meet in a bank: 4 and 2 cycles a read (measured).
__device__ __forceinline__ int key_of(int t) { return (t & 2) << 1 | ((t >> 2) & 1) | ((t >> 3) & 2); }

template <int D, int W>
__global__ __launch_bounds__(W * 64, W / 4) void prompt_kernel(PromptArgs a) {
  constexpr int KS = D / 64 + 1, VS = D / 64;  // sticks of K and V
  constexpr int TILE = (KS + VS) * kStick;
  constexpr int NQ = (D + kRope) / 16;
  constexpr int DT = D / 32;
  __shared__ __align__(16) uint8_t s_mem[2 * TILE];
  __shared__ uint32_t s_odd[W];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
  const int col = lane & 31, half = lane >> 5;
  // The row blocks of a (sequence, head) run in one XCD, whose L2 then holds its
  // keys, those of most keys first.
  const uint32_t j = blockIdx.x >> 3, pq = fdiv(j, a.by_blocks), pair = pq * 8 + (blockIdx.x & 7);
  if (pair >= static_cast<uint32_t>(a.pairs)) return;
  const int b = static_cast<int>(fdiv(pair, a.by_h)), h = static_cast<int>(pair) - b * a.H;
  const int block0 = (a.blocks - 1 - static_cast<int>(j - pq * a.blocks)) * (W * kRows);
  const int raw = __builtin_amdgcn_readfirstlane(a.ctx[b]);
  const int n = a.counts ? min(max(__builtin_amdgcn_readfirstlane(a.counts[b]), 0), a.T) : a.T;
  const int ctx = min(max(raw, 0), a.keys), total = min(ctx + n, a.keys);
  const bool bad = raw > a.keys - n;  // fewer keys than the lengths say
  const int row0 = block0 + wave * kRows, i = row0 + col;
  const bool live = i < n;
  // Keys of the workgroup's rows, of this wavefront's, and those that all rows of
  // the workgroup attend.
  const int most = block0 < n ? min(total, ctx + block0 + W * kRows) : 0;
  const int mine = row0 < n ? min(total, ctx + row0 + kRows) : 0;
  const int all = min(ctx + block0 + 1, total);
  const int tiles = (most + kKeys - 1) / kKeys;

  const uint32_t lds0 = lds_address(s_mem);
  auto load = [&](int t, int buf) {
    const int64_t t0 = static_cast<int64_t>(t) * kKeys;
    const int left = total - t * kKeys;
    const dma_rsrc rk = dma_buffer(a.k + b * a.k_sb + h * a.k_sh + t0 * a.k_st, kNoWhere),
                   rr = dma_buffer(a.kr + b * a.kr_sb + t0 * a.kr_st, kNoWhere),
                   rv = dma_buffer(a.v + b * a.v_sb + h * a.v_sh + t0 * a.v_st, kNoWhere);
#pragma unroll
    for (int c = 0; c < (KS + VS) * 8 / W; ++c) {
      const int chunk = c * W + wave, stick = c * W / 8;  // 8 tokens of a stick
      const int tok = (chunk & 7) * 8 + lane / 8;
      const uint32_t unit = ((lane & 7) ^ key_of(tok)) * 16;
      auto go = [&](dma_rsrc r, int64_t st, int feature) {
        dma16(r, lds0 + buf * TILE + chunk * 1024, tok < left ? tok * static_cast<uint32_t>(st) * 2 + unit : kNoWhere, feature * 2);
      };
      if (stick < D / 64)
        go(rk, a.k_st, stick * 64);
      else if (stick == D / 64)
        go(rr, a.kr_st, 0);
      else
        go(rv, a.v_st, (stick - KS) * 64);
    }
  };
  static_assert(W == 4 || W == 8, "a step of the workgroup's chunks lies in one stick");
  static_assert((KS + VS) * 8 % W == 0, "equal shares of a tile's chunks");
  if (tiles) load(0, 0);

  f16x8 qf[NQ];
  {
    const int64_t qi = live ? i : 0;
    const _Float16* x = a.q + b * a.q_sb + qi * a.q_st + h * a.q_sh + 8 * half;
    const _Float16* xr = a.qr + b * a.qr_sb + qi * a.qr_st + h * a.qr_sh + 8 * half;
#pragma unroll
    for (int s = 0; s < NQ; ++s) qf[s] = *reinterpret_cast<const f16x8*>(16 * s < D ? x + 16 * s : xr + 16 * s - D);
#pragma unroll
    for (int s = 0; s < NQ; ++s) asm volatile("" : "+v"(qf[s]));  // waits here: in the loop it would for the tile on its way
  }
  const int k_tok = token_of(col);
  int k_off[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) k_off[u] = k_tok * 128 + (((2 * u + half) ^ key_of(k_tok)) * 16);
  // V^T: 4 features of token 16 half + lane % 16 / 4; the key of tokens 8 and 32 further is the
  // same, odd tiles and tokens 4 further turn the unit's bits 2 and 0.
  const int tv = 16 * half + (lane & 15) / 4;
  const int v_lane = KS * kStick + tv * 128 + (((2 * ((lane >> 4) & 1) + ((lane >> 1) & 1)) ^ key_of(tv)) * 16) + 8 * (lane & 1);
  auto tr = [&](int at) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(s_mem + at));
  };

  f32x16 o[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int x = 0; x < 16; ++x) o[dt][x] = 0.f;
  float m = -INFINITY, l = 0.f;

  for (int t = 0; t < tiles; ++t) {
    const int buf = t & 1, t0 = t * kKeys;
    dma_wait();
    __syncthreads();  // the tile is there, and the other one is read
    if (t + 1 < tiles) load(t + 1, buf ^ 1);
    const bool edge = t0 + kKeys > all;  // some rows do not attend some of its keys
    uint64_t odd = 0;                    // of those, keys that hold a NaN or an infinity
    if (edge) {
      // What a row does not attend must not meet its weight of 0: such keys and values
      // become zeros, and the rows that attend them NaN.
      constexpr int PER = W * 64 / kKeys;  // threads of a token
      const int tok = threadIdx.x / PER;
      uint8_t* x = s_mem + buf * TILE + tok * 128 + (threadIdx.x % PER) * (128 / PER);
      uint32_t found = 0;
      if (t0 + tok >= all && t0 + tok < total)
        for (int s = 0; s < KS + VS; ++s)
#pragma unroll
          for (int u = 0; u < 8 / PER; ++u) {
            const u32x4 w = *reinterpret_cast<const u32x4*>(x + s * kStick + u * 16);
#pragma unroll
            for (int e = 0; e < 4; ++e) found |= (w[e] & 0x7c007c00u) + 0x04000400u;
          }
      const uint64_t lanes = __ballot((found & 0x80008000u) != 0);
      const bool drop = (lanes >> (lane & ~(PER - 1))) & ((1 << PER) - 1);
      if (drop)
        for (int s = 0; s < KS + VS; ++s)
#pragma unroll
          for (int u = 0; u < 8 / PER; ++u) *reinterpret_cast<u32x4*>(x + s * kStick + u * 16) = u32x4{0, 0, 0, 0};
      const uint64_t dropped = __ballot(drop);
      uint32_t bits = 0;
#pragma unroll
      for (int k = 0; k < 64 / PER; ++k) bits |= static_cast<uint32_t>((dropped >> (PER * k)) & 1) << k;
      if (lane == 0) s_odd[wave] = bits;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < W; ++w) odd |= static_cast<uint64_t>(s_odd[w]) << (64 / PER * w);
    }
    if (t0 >= mine) continue;  // none of its rows' keys (the barriers above are all of a step's)

    f32x16 s16[2] = {};
#pragma unroll
    for (int s = 0; s < NQ; ++s)
#pragma unroll
      for (int tb = 0; tb < 2; ++tb) {
        const f16x8 k = *reinterpret_cast<const f16x8*>(s_mem + buf * TILE + k_off[s % 4] + (s / 4) * kStick + tb * (32 * 128));
        s16[tb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, qf[s], s16[tb], 0, 0, 0);
      }
    // kAhead operands on their way at a time
    constexpr int kAhead = 6;
    __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);
#pragma unroll
    for (int x = 0; x < 2 * NQ - kAhead; ++x) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, kAhead, 0);
    float sc[32];
#pragma unroll
    for (int x = 0; x < 32; ++x) sc[x] = s16[x / 16][x % 16];
    float mx = -INFINITY;
#pragma unroll
    for (int x = 0; x < 32; ++x) {
      float y = sc[x] * a.scale_log2;
      if (edge) {
        const int tok = 32 * (x / 16) + 16 * half + x % 16;
        y = t0 + tok > min(ctx + i, total - 1) ? -INFINITY : (odd >> tok) & 1 ? NAN : y;
      }
      sc[x] = y;
      mx = fmaxf(mx, y);
    }
    mx = xor32_max(mx);
    if (__any(mx > m + kAbove)) {
      const float mn = fmaxf(m, mx - kBelow);
      const float alpha = m == -INFINITY ? 0.f : exp2_of(m - mn);
      m = mn;
      l *= alpha;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int x = 0; x < 16; ++x) o[dt][x] *= alpha;
    }
    const float mu = m == -INFINITY ? 0.f : m;  // a row that has attended nothing yet: weights 0
    // Weights round to fp16 for the product (a relative 2^-12 on average); their sum
    // stays in fp32.
    f16x8 w[4];
    const int v_at[2] = {buf * TILE + v_lane, (buf * TILE + v_lane) ^ 64};
#pragma unroll
    for (int x = 0; x < 32; ++x) {
      const float e = exp2_of(sc[x] - mu);
      l += e;
      w[x / 8][x % 8] = static_cast<_Float16>(e);
    }
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const int at = v_at[dt & 1] + dt / 2 * kStick + (32 * (s / 2) + 8 * (s % 2)) * 128;
        const s16x4 lo = tr(at), hi = tr((at ^ 16) + 4 * 128);
        o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(
            __builtin_bit_cast(f16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7)), w[s], o[dt], 0, 0, 0);
      }
  }
  l = xor32_sum(l);
  if (!live) l = 0.f;
  if (bad && live) l = NAN;
  if (i >= a.T) return;
  const int64_t at = (static_cast<int64_t>(b) * a.T + i) * a.H + h;
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

constexpr int kWaves = 8;

}  // namespace

extern "C" int spyre_latent_attn(const void* q, const int64_t* q_strides, const void* q_rope, const int64_t* q_rope_strides,
                                 const void* k, const int64_t* k_strides, const void* k_rope, const int64_t* k_rope_strides,
                                 const void* v, const int64_t* v_strides, const int32_t* context_lens, const int32_t* new_lens,
                                 void* out, float* lse, int B, int T, int H, int D, int keys, float scale, void* stream) {
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
  SPYRE_REQUIRE(keys < (1 << 30) && T < (1 << 30), SPYRE_EUNSUPPORTED, "too many tokens");
  PromptArgs a{};
  a.q = static_cast<const _Float16*>(q), a.q_sb = q_strides[0], a.q_st = q_strides[1], a.q_sh = q_strides[2];
  a.qr = static_cast<const _Float16*>(q_rope), a.qr_sb = q_rope_strides[0], a.qr_st = q_rope_strides[1], a.qr_sh = q_rope_strides[2];
  a.k = static_cast<const _Float16*>(k), a.k_sb = k_strides[0], a.k_st = k_strides[1], a.k_sh = k_strides[2];
  a.kr = static_cast<const _Float16*>(k_rope), a.kr_sb = k_rope_strides[0], a.kr_st = k_rope_strides[1];
  a.v = static_cast<const _Float16*>(v), a.v_sb = v_strides[0], a.v_st = v_strides[1], a.v_sh = v_strides[2];
  a.ctx = context_lens, a.counts = new_lens, a.out = static_cast<_Float16*>(out), a.lse = lse;
  a.B = B, a.T = T, a.H = H, a.keys = keys, a.scale_log2 = scale * kLog2e;
  const int rows = kWaves * kRows;
  a.blocks = (T + rows - 1) / rows;
  const int64_t pairs = static_cast<int64_t>(B) * H, grid = (pairs + 7) / 8 * 8 * a.blocks;
  SPYRE_REQUIRE(grid < (int64_t{1} << 31), SPYRE_EUNSUPPORTED, "too many rows");
  a.pairs = static_cast<int>(pairs);
  a.by_h = make_fastdiv(static_cast<uint32_t>(H)), a.by_blocks = make_fastdiv(static_cast<uint32_t>(a.blocks));
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (D == 128)
    prompt_kernel<128, kWaves><<<dim3(static_cast<uint32_t>(grid)), kWaves * 64, 0, st>>>(a);
  else
    prompt_kernel<64, kWaves><<<dim3(static_cast<uint32_t>(grid)), kWaves * 64, 0, st>>>(a);
  const hipError_t e = hipGetLastError();
  SPYRE_REQUIRE(e == hipSuccess, SPYRE_EHIP, "latent prompt attention launch failed: %s", hipGetErrorString(e));
  return SPYRE_OK;
}
