// Attention over the paged latent cache (spyre_paged_latent_attn).
//
// A cached token is one row for all heads: c (rank features), its latent vector,
// and r (64), its rotated key.  Head h's query in the latent space is (q, s), its
// keys' weights in q already, and the values' come behind the output:
//   score(t) = scale (q . c_t + s . r_t),  out = softmax(score) c,
//   lse the logarithm of the softmax's sum.
// Sequence b holds ctx[b] tokens and, behind them in the same pages, n[b] new ones;
// query i < n[b] attends t < ctx[b], and new j < n[b] where mask[b, i, j] (no mask:
// j <= i).  Rows that attend nothing, and those from n[b] on, are zeros with lse
// -inf.
//
// All T H rows of a sequence have the same keys, and the values are a part of
// them: a page is read once, into LDS, and serves both products of all rows.
//   S^T[tok, row] = K[tok, :] Q^T[:, row]      K as it lies: rows of features
//   O^T[d, row] += C^T[d, tok] P^T[tok, row]   C^T by transposing reads of the same rows
// Four wavefronts have 32 rows.  Each has all of their Q in registers (rank 512: 144
// of them) and takes the scores of 16 of a page's tokens; the weights meet in LDS, and
// each then takes all 64 tokens of a quarter of O's features (64 registers).  With
// O whole in one wavefront (256 registers) two of them do not fit a SIMD, and one
// spills.  Up to 32 rows a workgroup is four wavefronts with one page in LDS, two
// workgroups to a compute unit, one of which loads while the other computes; beyond
// it is eight, 64 rows, and two pages in LDS, the next one on its way.

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
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr int kRope = 64;
constexpr int kTile = 32;   // rows of a wavefront
constexpr int kSplit = 4;   // wavefronts that share them
constexpr int kStick = kPage * 64 * 2;  // bytes of 64 features of a page
// The reference of a row's exponents lies kBelow under its largest score (log2
// units) and moves when a score passes it by kAbove: most pages then leave O as
// it is, and a weight is a normal number of fp16 down to 2^-21 of the largest.
constexpr float kBelow = 7.f, kAbove = 15.f;

struct LatentArgs {
  const _Float16 *q, *qr;
  int64_t q_sb, q_st, q_sh, qr_sb, qr_st, qr_sh;
  const _Float16* pages;
  const int32_t *bt, *ctx, *counts;
  const uint8_t* mask;
  int64_t bt_stride, pages_per_seq, num_pages, m_sb, m_si, m_sj;
  _Float16* out;  // [B, T, H, rank]
  float* lse;     // [B, T, H] or null
  float* ws;
  int B, T, H, Hkv, rows, max_ctx, draft_keys;
  float scale_log2;
  int row_blocks, block_rows, width;
  int ranges, min_per, min_cut, each;  // see PageWalk
  FastDiv by_h, by_hkv, by_blocks, by_ranges;
};
typedef PageWalk<LatentArgs> Walk;

// Partials: O [slots][width][rank], then (m, l) [slots][width]; slots are (range,
// row block, slot 0 / 1).
__device__ __forceinline__ int64_t partial_of(const LatentArgs& a, int range, int rb, int slot, int row) {
  return ((static_cast<int64_t>(range) * a.row_blocks + rb) * 2 + slot) * a.width + row;
}
__device__ __forceinline__ int64_t partials(const LatentArgs& a) {
  return static_cast<int64_t>(a.ranges) * a.row_blocks * 2 * a.width;
}

// 4 features of a finished row.
template <int RANK>
__device__ __forceinline__ void store_row4(const LatentArgs& a, int b, int row, int d, f32x4 x, float m, float l) {
  const int i = static_cast<int>(fdiv(row, a.by_h)), h = row - i * a.H;
  const int64_t at = (static_cast<int64_t>(b) * a.T + i) * a.H + h;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  f16x4 y;
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = static_cast<_Float16>(l == 0.f ? 0.f : x[e] * inv);
  *reinterpret_cast<f16x4*>(a.out + at * RANK + d) = y;
  if (a.lse && d == 0) a.lse[at] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
}

// A sequence's pages from `first` on: 64 table entries at a time, one a lane.  A
// page that the table does not name validly is page 0 (in bounds) and poisons
// the rows.
struct Pages {
  const LatentArgs& a;
  const int32_t* trow;
  int lane, first, ids = 0;
  bool poisoned = false;
  __device__ __forceinline__ Pages(const LatentArgs& args, int b, int lane_, int first_)
      : a(args), trow(args.bt + b * args.bt_stride), lane(lane_), first(first_) {}
  __device__ __forceinline__ int64_t at(int p) {  // first, first + 1, ...
    const int i = p - first;
    if ((i & 63) == 0) {
      ids = p + lane < a.pages_per_seq ? trow[p + lane] : -1;
      asm volatile("" : "+v"(ids));  // waits here, not in every page
    }
    const int64_t phys = __builtin_amdgcn_readlane(ids, i & 63);
    const bool bad = phys < 0 || phys >= a.num_pages;
    poisoned |= bad;
    return bad ? 0 : phys;
  }
};

// A lane index that the compiler forms addresses from where they are used: kept in
// registers through the loops, those of rare paths would spill.
__device__ __forceinline__ int here(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// Rows of a page in LDS are 128 bytes for each stick; unit u (16 bytes) of token t
// lies at u ^ (t & 7).  Neither 8 lanes that read a unit of 8 tokens nor 16 that read
// 2 units of 4 tokens, transposed, then meet in a bank.
template <int RANK, int RG>
__global__ __launch_bounds__(RG * kSplit * 64, 2) void latent_kernel(LatentArgs a) {
  constexpr int WAVES = RG * kSplit;
  constexpr int NS = (RANK + kRope) / 64;  // sticks
  constexpr int DT = RANK / 32 / kSplit;   // tiles of O of a wavefront
  constexpr int NQ = (RANK + kRope) / 32;  // operands of Q of 16 rows
  constexpr int BUF = NS * kStick;
  constexpr int BUFS = RG == 1 ? 1 : 2;
  __shared__ __align__(16) uint8_t s_mem[BUFS * BUF];
  __shared__ __align__(16) _Float16 s_p[RG][kTile * kPage];  // weights: 8 units of 8 tokens a row, unit u at u ^ (row & 7)
  __shared__ float s_max[RG][kSplit][kTile];                 // of a page's scores
  __shared__ float s_ref[RG][kTile], s_sum[RG][kSplit][kTile];
  __shared__ uint32_t s_odd[WAVES];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
  const int col = lane & 31, half = lane >> 5, l16 = lane & 15, g16 = lane >> 4;
  const int rg = wave / kSplit, part = wave % kSplit;
  const uint32_t lds0 = lds_address(s_mem);
  int range, rb;
  place_of(a, range, rb);
  Walk walk;
  if (range >= a.ranges || !walk.start(a, lane, range)) return;

  // Lane offsets: unit g16 (and 4 + g16) of K's row 16 part + l16; 4 features of token
  // 8 half + l16 / 4 (and 4 tokens further) of C^T's tiles.
  const int k_tok = 16 * part + l16;
  const int k_off[2] = {k_tok * 128 + ((g16 ^ (k_tok & 7)) * 16), k_tok * 128 + (((4 + g16) ^ (k_tok & 7)) * 16)};
  // The unit's key is that of token l16 / 4, its bit 2 turned by odd tiles and by tokens 4
  // further: two lane offsets, the rest of an address is constant.
  const int v_lane = DT / 2 * part * kStick + (8 * half + l16 / 4) * 128 + (((2 * (g16 & 1) + ((lane >> 1) & 1)) ^ (l16 / 4)) * 16) + 8 * (lane & 1);
  auto tr = [&](int at) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(s_mem + at));
  };

  for (; walk.u < walk.end;) {
    const Piece pc = piece_of(a, walk);
    const int b = walk.b;
    const Seq sq = walk.seq;
    const int total = sq.ctx + sq.n;
    const int row0 = rb * a.block_rows + kTile * rg;
    // (a workgroup whose rows are all of no new token has nothing to do)
    const int p0 = pc.page0, p1 = rb * a.block_rows < sq.n * a.H ? pc.page1 : pc.page0;
    Pages pages(a, b, lane, p0);

    // A page on its way into buffer `buf`; tokens that do not exist as zeros.
    auto load = [&](int p, int buf) {
      const dma_rsrc r = dma_buffer(a.pages + pages.at(p) * (NS * (kStick / 2)), BUF);
      const int n = total - p * kPage;
      const int t = here(lane) / 8;
      const uint32_t off = t * 128 + (((lane & 7) ^ t) * 16);
      // a wavefront's chunks (8 tokens of a stick): the same tokens in every stick, RG 1 two runs of them
      uint32_t voff[8 / WAVES];
#pragma unroll
      for (int c = 0; c < 8 / WAVES; ++c) voff[c] = (c * WAVES + wave) * 8 + t < n ? off : BUF;
#pragma unroll
      for (int c = 0; c < NS * 8 / WAVES; ++c) {
        const int chunk = c * WAVES + wave;
        dma16(r, lds0 + buf * BUF + chunk * 1024, voff[c % (8 / WAVES)], chunk * 1024);
      }
    };
    static_assert(NS * 8 % WAVES == 0, "equal shares of a page's chunks");
    if (p0 < p1) load(p0, 0);

    // Queries of rows l16 and 16 + l16 of the tile.  (One that is not there is another's.)
    f16x8 qf[2][NQ];
    auto token_of_row = [&](int row) {  // its new token; sq.n or more: none
      return row < a.rows ? static_cast<int>(fdiv(row, a.by_h)) : sq.n;
    };
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const int row = row0 + 16 * n + here(l16), i = token_of_row(row);
      const bool live = i < sq.n;
      const int64_t qi = live ? i : 0, h = live ? row - i * a.H : 0;
      const _Float16* x = a.q + b * a.q_sb + qi * a.q_st + h * a.q_sh + 8 * g16;
      const _Float16* xr = a.qr + b * a.qr_sb + qi * a.qr_st + h * a.qr_sh + 8 * g16;
#pragma unroll
      for (int s = 0; s < NQ; ++s) qf[n][s] = *reinterpret_cast<const f16x8*>(32 * s < RANK ? x + 32 * s : xr + 32 * s - RANK);
    }
#pragma unroll
    for (int s = 0; s < NQ; ++s) asm volatile("" : "+v"(qf[0][s]), "+v"(qf[1][s]));  // waits here: in the loop it would for the page on its way
    f32x16 o[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int x = 0; x < 16; ++x) o[dt][x] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};  // of rows l16 and 16 + l16; l: of this lane's tokens
    if (part == 0 && half == 0) s_ref[rg][col] = -INFINITY;

    for (int p = p0; p < p1; ++p) {
      const int buf = BUFS == 1 ? 0 : (p - p0) & 1;
      dma_wait();
      __syncthreads();  // the page is there, and the other buffer is read
      if (BUFS == 2 && p + 1 < p1) load(p + 1, buf ^ 1);
      const bool edge = (p + 1) * kPage > sq.ctx;  // some tokens are new or do not exist
      uint32_t odd = 0;                            // of this wavefront's 16 tokens, new ones that hold a NaN or an infinity
      if (edge && a.T > 1) {
        // What a row does not attend must not meet its weight of 0: such tokens become
        // zeros, and the rows that attend them NaN.
        constexpr int PER = WAVES * 64 / kPage;  // threads of a token
        const int th = here(threadIdx.x), t = th / PER;
        uint8_t* x = s_mem + buf * BUF + t * 128 + (th % PER) * (128 / PER);
        uint32_t found = 0;
        if (p * kPage + t >= sq.ctx && p * kPage + t < total)
          for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int u = 0; u < 8 / PER; ++u) {
              const u32x4 w = *reinterpret_cast<const u32x4*>(x + s * kStick + u * 16);
#pragma unroll
              for (int e = 0; e < 4; ++e) found |= (w[e] & 0x7c007c00u) + 0x04000400u;
            }
        const uint64_t lanes = __ballot((found & 0x80008000u) != 0);
        const bool bad = (lanes >> (lane & ~(PER - 1))) & ((1 << PER) - 1);
        if (bad)
          for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int u = 0; u < 8 / PER; ++u) *reinterpret_cast<u32x4*>(x + s * kStick + u * 16) = u32x4{0, 0, 0, 0};
        const uint64_t all = __ballot(bad);
        uint32_t bits = 0;
#pragma unroll
        for (int k = 0; k < 64 / PER; ++k) bits |= static_cast<uint32_t>((all >> (PER * k)) & 1) << k;
        if (lane == 0) s_odd[wave] = bits;
        __syncthreads();
        // wavefront w looked at tokens 64 / PER * w on
        odd = RG == 1 ? s_odd[part] : s_odd[2 * part] | s_odd[2 * part + 1] << 8;
        static_assert(RG <= 2, "see odd");
      }

      f32x4 sc[2] = {};
#pragma unroll
      for (int s = 0; s < NQ; ++s) {
        const f16x8 k = *reinterpret_cast<const f16x8*>(s_mem + buf * BUF + k_off[s % 2] + (s / 2) * kStick);
#pragma unroll
        for (int n = 0; n < 2; ++n) sc[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, qf[n][s], sc[n], 0, 0, 0);
      }
      // kAhead operands on their way at a time
      constexpr int kAhead = 4;
      __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);
#pragma unroll
      for (int x = 0; x < NQ - kAhead; ++x) {
        __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x008, 2 * kAhead, 0);
      // sc[n][e]: row 16 n + l16, token 16 part + 4 g16 + e
      float mx[2];
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        uint32_t seen = 15;
        if (edge) {
          const int ln = here(lane), j0 = p * kPage + 16 * part + 4 * (ln / 16) - sq.ctx;
          const int i = min(token_of_row(row0 + 16 * n + ln % 16), sq.n - 1);
          seen = 0;
          if (a.mask) {
            const uint8_t* mask = a.mask + b * a.m_sb + max(i, 0) * a.m_si;
            uint8_t keep[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) keep[e] = mask[min(max(j0 + e, 0), a.T - 1) * a.m_sj];
#pragma unroll
            for (int e = 0; e < 4; ++e) seen |= static_cast<uint32_t>(j0 + e < 0 || (j0 + e < sq.n && keep[e] != 0)) << e;
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) seen |= static_cast<uint32_t>(j0 + e <= i) << e;
          }
        }
        mx[n] = -INFINITY;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float v = sc[n][e] * a.scale_log2;
          if (edge) v = !((seen >> e) & 1) ? -INFINITY : (odd >> (4 * g16 + e)) & 1 ? NAN : v;
          sc[n][e] = v;
          mx[n] = fmaxf(mx[n], v);
        }
        mx[n] = xor32_max(xor16_max(mx[n]));
        if (g16 == n) s_max[rg][part][16 * n + l16] = mx[n];
      }
      // Weights relative to the reference as it is.  They round to fp16 for the product (a
      // relative 2^-12 on average); their sum stays in fp32.
      float add[2];
      const int ln = here(lane), p_write = (ln & 15) * kPage + (((2 * part + ln / 32) ^ (ln & 7)) * 8) + (ln / 16 & 1) * 4;
      auto weigh = [&] {
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const float mu = m[n] == -INFINITY ? 0.f : m[n];  // a row that has attended nothing yet: weights 0
          f16x4 w4;
          add[n] = 0.f;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float w = exp2_of(sc[n][e] - mu);
            add[n] += w;
            w4[e] = static_cast<_Float16>(w);
          }
          *reinterpret_cast<f16x4*>(&s_p[rg][p_write + 16 * n * kPage]) = w4;
        }
      };
      weigh();
      __syncthreads();
      // Where a row's scores pass its reference too far, all move.
      bool moves = false;
#pragma unroll
      for (int r = 0; r < RG; ++r) {
        const int k = 2 * (ln / 32), c = ln & 31;
        moves = moves || fmaxf(s_max[r][k][c], s_max[r][k + 1][c]) > s_ref[r][c] + kAbove;
      }
      if (__any(moves)) {
        const int c = here(col);
        float top = s_max[rg][0][c];
#pragma unroll
        for (int k = 1; k < kSplit; ++k) top = fmaxf(top, s_max[rg][k][c]);
        const float old = s_ref[rg][c], ref = fmaxf(old, top - kBelow);
        const float alpha = old == -INFINITY ? 0.f : exp2_of(old - ref);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int x = 0; x < 16; ++x) o[dt][x] *= alpha;
        __syncthreads();  // the old references and the weights are read
        if (part == 0 && half == 0) s_ref[rg][c] = ref;
        const float r0 = __shfl(ref, l16, 64), r1 = __shfl(ref, 16 + l16, 64);
        l[0] *= m[0] == -INFINITY ? 0.f : exp2_of(m[0] - r0);
        l[1] *= m[1] == -INFINITY ? 0.f : exp2_of(m[1] - r1);
        m[0] = r0, m[1] = r1;
        weigh();
        __syncthreads();
      }
      l[0] += add[0], l[1] += add[1];
      const int v_at[2] = {buf * BUF + v_lane, (buf * BUF + v_lane) ^ 64};
      const int p_read = (ln & 31) * kPage + ((ln / 32) ^ (ln & 7)) * 8;
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const f16x8 w = *reinterpret_cast<const f16x8*>(&s_p[rg][p_read ^ (16 * s)]);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          const int at = dt / 2 * kStick + 16 * s * 128;
          const s16x4 lo = tr(v_at[dt & 1] + at), hi = tr(v_at[(dt & 1) ^ 1] + at + 4 * 128);
          o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(
              __builtin_bit_cast(f16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7)), w, o[dt], 0, 0, 0);
        }
      }
      if (BUFS == 1) {
        __syncthreads();
        if (p + 1 < p1) load(p + 1, 0);
      }
    }
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const int r = 16 * n + here(l16);
      const bool live = token_of_row(row0 + r) < sq.n;
      l[n] = xor32_sum(xor16_sum(l[n]));
      if (!live) l[n] = 0.f;
      if ((pages.poisoned || sq.bad) && live) l[n] = NAN;
      if (g16 == n) s_sum[rg][part][r] = l[n];
    }
    __syncthreads();
    float L = 0.f;
#pragma unroll
    for (int k = 0; k < kSplit; ++k) L += s_sum[rg][k][col];
    const float M = L == 0.f ? -INFINITY : s_ref[rg][col];
    if (row0 + col < a.rows) {
      const int64_t at = partial_of(a, range, rb, pc.slot, kTile * rg + col);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const f32x4 y = {o[dt][4 * x], o[dt][4 * x + 1], o[dt][4 * x + 2], o[dt][4 * x + 3]};
          const int d = 32 * (DT * part + dt) + 8 * x + 4 * half;
          if (pc.whole)
            store_row4<RANK>(a, b, row0 + col, d, y, M, L);
          else
            *reinterpret_cast<f32x4*>(a.ws + at * RANK + d) = y;
        }
      if (!pc.whole && part == 0 && half == 0) {
        float* ml = a.ws + partials(a) * RANK + at * 2;
        ml[0] = M, ml[1] = L;
      }
    }
    advance(a, walk, pc);
    __syncthreads();  // LDS is read before the next piece writes it
  }
}

// Joins the partials of each sequence that several ranges share: a thread 4
// features of a row.
template <int RANK>
__global__ __launch_bounds__(256) void latent_join_kernel(LatentArgs a) {
  const int b = blockIdx.x;
  Walk w;
  w.seek(a, threadIdx.x % 64, b);
  int r0, r1;
  w.parts_of(a, 0, r0, r1);
  if (r1 <= r0) return;
  const Seq sq = w.seq;
  for (int64_t u = blockIdx.y * 256 + threadIdx.x; u < static_cast<int64_t>(a.rows) * (RANK / 4); u += gridDim.y * 256) {
    const int row = static_cast<int>(u / (RANK / 4)), d = 4 * static_cast<int>(u % (RANK / 4));
    const int rb = row / a.block_rows, rl = row - rb * a.block_rows;
    float M = -INFINITY, L = 0.f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    if (row < sq.n * a.H)
      merge_parts(r0, r1, M, L, acc, [&](int r, float& m, float& l, f32x4& x) {
        const int64_t part = partial_of(a, r, rb, r == r0 ? 1 : 0, rl);
        const float* ml = a.ws + partials(a) * RANK + part * 2;
        m = ml[0], l = ml[1];
        x = *reinterpret_cast<const f32x4*>(a.ws + part * RANK + d);
      });
    store_row4<RANK>(a, b, row, d, acc, M, L);
  }
}

struct Plan {
  int groups;  // RG
  int row_blocks, block_rows, width, ranges, min_per, min_cut;
  size_t ws_bytes;
};

Plan plan_of(int B, int T, int H, int rank, int max_tokens) {
  Plan p;
  const int64_t rows = static_cast<int64_t>(T) * H;
  p.groups = rows <= kTile ? 1 : 2;
  p.block_rows = kTile * p.groups;
  p.row_blocks = static_cast<int>((rows + p.block_rows - 1) / p.block_rows);
  p.width = static_cast<int>(std::min<int64_t>(p.block_rows, rows));
  p.min_per = 2, p.min_cut = 4;
  const int64_t pages = std::max(pages_of(max_tokens), 1), parts_of_one = pages < p.min_cut ? 1 : pages / p.min_per;
  const int64_t ranges = std::min(B * parts_of_one, std::max<int64_t>((p.groups == 1 ? 512 : 256) / p.row_blocks, 1));
  p.ranges = static_cast<int>(std::max<int64_t>(ranges, 1));
  p.ws_bytes = static_cast<size_t>(p.ranges) * p.row_blocks * 2 * p.width * (rank + 2) * 4;
  return p;
}

constexpr int kJoinBlocks = 2048;

bool sizes_ok(int B, int T, int H, int max_ctx) {
  return B >= 0 && T > 0 && H > 0 && max_ctx >= 0 && static_cast<int64_t>(T) * H < (int64_t{1} << 31) - 256 &&
         static_cast<int64_t>(max_ctx) + T < (int64_t{1} << 31) - kPage;
}

template <int RANK>
void launch(const LatentArgs& a, int groups, dim3 grid, hipStream_t st) {
  if (groups == 1)
    latent_kernel<RANK, 1><<<grid, kSplit * 64, 0, st>>>(a);
  else
    latent_kernel<RANK, 2><<<grid, 2 * kSplit * 64, 0, st>>>(a);
}

}  // namespace

extern "C" size_t spyre_paged_latent_attn_workspace_bytes(int B, int T, int H, int rank, int max_context_len) {
  if (!sizes_ok(B, T, H, max_context_len) || (rank != 256 && rank != 512)) return 0;
  return plan_of(B, T, H, rank, max_context_len + T).ws_bytes;
}

extern "C" int spyre_paged_latent_attn(const void* q, const int64_t* q_strides, const void* q_rope, const int64_t* q_rope_strides,
                                       const void* cache, const int32_t* block_table, int64_t bt_stride, int64_t pages_per_seq,
                                       const int32_t* context_lens, const int32_t* draft_lens, const void* mask,
                                       const int64_t* mask_strides, void* out, float* lse, void* workspace,
                                       size_t workspace_bytes, int B, int T, int H, int rank, int64_t num_pages,
                                       int max_context_len, float scale, void* stream) {
  spyre_hip::clear_error();
  SPYRE_REQUIRE(rank == 256 || rank == 512, SPYRE_EUNSUPPORTED, "rank %d not in {256, 512}", rank);
  SPYRE_REQUIRE(B >= 0 && T >= 0 && H > 0 && max_context_len >= 0 && pages_per_seq >= 0 && bt_stride >= 0, SPYRE_EINVAL,
                "bad sizes B=%d T=%d H=%d max_context_len=%d", B, T, H, max_context_len);
  if (B == 0 || T == 0) return SPYRE_OK;
  SPYRE_REQUIRE(sizes_ok(B, T, H, max_context_len), SPYRE_EUNSUPPORTED, "too many rows or tokens");
  SPYRE_REQUIRE(num_pages > 0, SPYRE_EINVAL, "bad num_pages");
  SPYRE_REQUIRE(q && q_strides && q_rope && q_rope_strides && cache && block_table && context_lens && out && (!mask || mask_strides),
                SPYRE_EINVAL, "null pointer argument");
  auto aligned = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  SPYRE_REQUIRE(aligned(q) && aligned(q_rope) && aligned(cache) && aligned(out), SPYRE_EINVAL,
                "q, the cache and out must be 16-byte aligned");
  for (int i = 0; i < 3; ++i)
    SPYRE_REQUIRE(q_strides[i] % 8 == 0 && q_rope_strides[i] % 8 == 0, SPYRE_EINVAL, "q strides must be multiples of 8 elements");
  const Plan p = plan_of(B, T, H, rank, max_context_len + T);
  SPYRE_REQUIRE(workspace && workspace_bytes >= p.ws_bytes && aligned(workspace), SPYRE_ENOSPC,
                "workspace holds %zu bytes, need %zu (16-byte aligned)", workspace ? workspace_bytes : 0, p.ws_bytes);
  LatentArgs a{};
  a.q = static_cast<const _Float16*>(q), a.q_sb = q_strides[0], a.q_st = q_strides[1], a.q_sh = q_strides[2];
  a.qr = static_cast<const _Float16*>(q_rope), a.qr_sb = q_rope_strides[0], a.qr_st = q_rope_strides[1], a.qr_sh = q_rope_strides[2];
  a.pages = static_cast<const _Float16*>(cache);
  a.bt = block_table, a.bt_stride = bt_stride, a.pages_per_seq = pages_per_seq, a.num_pages = num_pages;
  a.ctx = context_lens, a.counts = draft_lens, a.draft_keys = 1;
  a.mask = static_cast<const uint8_t*>(mask);
  if (mask) a.m_sb = mask_strides[0], a.m_si = mask_strides[1], a.m_sj = mask_strides[2];
  a.out = static_cast<_Float16*>(out), a.lse = lse, a.ws = static_cast<float*>(workspace);
  a.B = B, a.T = T, a.H = H, a.Hkv = 1, a.rows = T * H;
  a.max_ctx = max_context_len, a.scale_log2 = scale * kLog2e;
  a.row_blocks = p.row_blocks, a.block_rows = p.block_rows, a.width = p.width;
  a.ranges = p.ranges, a.min_per = p.min_per, a.min_cut = p.min_cut;
  a.each = B % p.ranges == 0 ? B / p.ranges : 0;
  const int64_t blocks = static_cast<int64_t>((p.ranges + 7) / 8 * 8) * p.row_blocks;
  SPYRE_REQUIRE(static_cast<int64_t>(B) * (pages_of(max_context_len + T) + kStart + 1) < (int64_t{1} << 30) && blocks < (int64_t{1} << 31),
                SPYRE_EUNSUPPORTED, "too many pages or rows");
  a.by_h = make_fastdiv(static_cast<uint32_t>(H)), a.by_hkv = make_fastdiv(1);
  a.by_blocks = make_fastdiv(static_cast<uint32_t>(p.row_blocks)), a.by_ranges = make_fastdiv(static_cast<uint32_t>(p.ranges));
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid(static_cast<uint32_t>(blocks));
  rank == 512 ? launch<512>(a, p.groups, grid, st) : launch<256>(a, p.groups, grid, st);
  hipError_t e = hipGetLastError();
  SPYRE_REQUIRE(e == hipSuccess, SPYRE_EHIP, "latent attention launch failed: %s", hipGetErrorString(e));
  if (p.ranges > 1) {  // no sequence is cut where one range has them all
    const int64_t n = std::min((static_cast<int64_t>(a.rows) * (rank / 4) + 255) / 256, std::max<int64_t>(kJoinBlocks / B, 1));
    const dim3 join(static_cast<uint32_t>(B), static_cast<uint32_t>(n));
    rank == 512 ? latent_join_kernel<512><<<join, 256, 0, st>>>(a) : latent_join_kernel<256><<<join, 256, 0, st>>>(a);
    e = hipGetLastError();
    SPYRE_REQUIRE(e == hipSuccess, SPYRE_EHIP, "latent attention join launch failed: %s", hipGetErrorString(e));
  }
  return SPYRE_OK;
}
