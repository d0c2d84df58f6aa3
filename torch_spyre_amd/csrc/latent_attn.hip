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
// Up to 32 rows of a sequence are one workgroup's, more are split into blocks of 64; pages, and 32
// tokens of them, come into LDS while the ones before are used.  The first product has 16 x 16 tiles
// with Q in registers, the weights meet in LDS, and the second has 32 x 32 tiles of O in registers.
//
// Measured, rank 512 (a pass among others, from device to device): 32 sequences x 4096 tokens x 128
// heads 61-65 us (36.5 GFLOP, 560-600 TFLOP/s; the first kernel 52-58, the join 9.8).  That kernel has
// wavefronts on the device for 93000 cycles: 32.5 tiles of 32 tokens x 64 rows of 2130 each (0.85 us,
// of which the matrix cores 0.45 and the loads' way into LDS as much), the start of a range 6 us, the
// parts; the matrix cores are busy for 38 % of them.  What the rest of its time goes to, or whether the
// clock falls, is not established.  16 x 500-6000 tokens x 1-7 new x 32 heads 46-48 (39-42 and 9.0;
// 72000 cycles, 29 % busy); 64 x 128-16384 tokens x 16 heads 124 (629 MB; 117, 5.4 TB/s, and 7.3);
// 1 x 700 x 16 heads 17.1-17.5: latency.

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
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr int kRope = 64;
constexpr int kTile = 32;   // rows of a wavefront
constexpr int kParts = 4;   // of O's features, one to a wavefront
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
  int B, T, H, rows, max_ctx, draft_keys;
  float scale_log2;
  int row_blocks, block_rows, block_shift;  // of a sequence with T new tokens; a block's
  int ranges;                               // at most
  FastDiv by_h, by_ranges;
};

// How the work is shared out, as in PageWalk, with row blocks in the place of KV heads: a row
// block that has rows counts kOpen units and one for each page, one behind the sequence's
// new tokens (zeros) one unit.  Range r of R is the units [all r / R, all (r + 1) / R), row block
// after row block, sequence after sequence: with a workgroup to each row block of a range of
// pages half of them had no rows where sequences had 1 to 7 new tokens (16 x 7 x 32 heads 64 us, so
// 57).  A bound that would leave kFew pages or less of a row block moves to its end (fewer where
// a range has few).
struct Walk {
  // kLeast: units of a range, at least: one sequence of 700 tokens and 16 heads 17.4 us (4: 20.5, 6:
  // 24), 4 of 3000 22.4 (23.2, 25.5).  kOpen: 32 x 4096 tokens x 128 heads 66 us with 1, 2 and 4; the
  // drafts above 56, 54, 52.  kFew: 300 x 10-900 tokens x 64 heads 68 us (4: 72).
  static constexpr int kLeast = 3, kOpen = 4, kFew = 2;
  int used;           // ranges that have any units
  int u, end;         // units
  int b, base;        // the sequence, its first unit
  Seq seq;            // what it holds
  int size, live;     // units of a row block that has rows; such row blocks

  __device__ __forceinline__ static int live_of(const LatentArgs& a, int n) { return (n * a.H + a.block_rows - 1) >> a.block_shift; }
  __device__ __forceinline__ static int units_of(const LatentArgs& a, const Seq& s) {
    const int live = live_of(a, s.n);
    return live * (kOpen + s.pages) + a.row_blocks - live;
  }
  __device__ __forceinline__ int units(const LatentArgs& a) const { return live * size + a.row_blocks - live; }
  // A sequence a lane.
  __device__ __forceinline__ static void lane_of(const LatentArgs& a, int b, int& ctx, int& count, int& units) {
    ctx = count = units = 0;
    if (b < a.B) {
      ctx = a.ctx[b], count = a.counts ? a.counts[b] : a.T;
      units = units_of(a, seq_of(a, ctx, count));
    }
  }
  // A bound where it belongs, in its sequence: no piece of few pages.
  __device__ __forceinline__ int placed(int unit, int few) const {
    const int in = unit - base;
    if (in >= live * size) return unit;
    const int at = static_cast<int>(static_cast<uint32_t>(in) % static_cast<uint32_t>(size));
    const int g0 = unit - at, g1 = g0 + size;
    return at - kOpen <= few ? g0 : g1 - unit <= few ? g1 : unit;
  }
  // This workgroup's range; -1: none.  Those that follow one another run in one XCD.  (Loops
  // and one copy of each step: what a kernel runs once, it waits for to be fetched.)
  __device__ __forceinline__ int start(const LatentArgs& a, int lane) {
    int total = 0, ctx, count, sum;
#pragma unroll 1
    for (int c = 0; c < a.B; c += 64) {
      lane_of(a, c + lane, ctx, count, sum);
      sum = scan64(sum);
      total += __builtin_amdgcn_readlane(sum, 63);
    }
    const bool many = total >= kLeast * a.ranges;
    used = many ? a.ranges : max(total / kLeast, 1);
    const int xcd = blockIdx.x & 7, i = blockIdx.x >> 3;
    if (i >= used / 8 + (xcd < used % 8)) return -1;
    const int r = xcd * (used / 8) + min(xcd, used % 8) + i;
    const int share = many ? static_cast<int>(fdiv(total, a.by_ranges)) : kLeast, rest = many ? total - share * a.ranges : 0;
#pragma unroll 1
    for (int k = 1; k >= 0; --k) {
      int unit = (r + k) * share + static_cast<int>(fdiv((r + k) * rest, a.by_ranges));
      if (r + k == used) unit = total;
      if (unit < total) {
        base = 0;
#pragma unroll 1
        for (int c = 0;; c += 64) {
          if (a.B > 64) {
            lane_of(a, c + lane, ctx, count, sum);
            sum = scan64(sum);
          }
          const uint64_t past = __builtin_amdgcn_ballot_w64(base + sum > unit);
          if (past || c + 64 >= a.B) {
            const int l = past ? __builtin_ctzll(past) : (a.B - 1) % 64;
            b = c + l;
            seq = seq_of(a, __builtin_amdgcn_readlane(ctx, l), __builtin_amdgcn_readlane(count, l));
            live = live_of(a, seq.n), size = kOpen + seq.pages;
            base += __builtin_amdgcn_readlane(sum, l) - units(a);
            break;
          }
          base += __builtin_amdgcn_readlane(sum, 63);
        }
        unit = placed(unit, min(max(share - kOpen, 0) / 2, kFew));
      }
      (k ? end : u) = unit;
    }
    if (u < end && u == base + units(a)) next_sequence(a);
    return r;
  }
  __device__ __forceinline__ void next_sequence(const LatentArgs& a) {
    base += units(a);
    b = min(b + 1, a.B - 1);
    const Seq s = seq_at(a, b);
    seq = s, live = live_of(a, s.n), size = kOpen + s.pages;
  }
  // Pages [page0, page1) of a row block.
  struct Piece {
    int rb, page0, page1;
    bool begins, ends;
  };
  __device__ __forceinline__ Piece piece(const LatentArgs& a) const {
    const int in = u - base, of_live = live * size;
    if (in >= of_live) return {min(live + in - of_live, a.row_blocks - 1), 0, 0, true, true};
    Piece p;
    p.rb = min(static_cast<int>(static_cast<uint32_t>(in) / static_cast<uint32_t>(size)), a.row_blocks - 1);
    const int at = in - p.rb * size;
    p.page0 = max(at - kOpen, 0), p.page1 = min(size, at + end - u) - kOpen;
    p.begins = at == 0, p.ends = p.page1 == size - kOpen;
    return p;
  }
  // After it.
  __device__ __forceinline__ void advance(const LatentArgs& a, const Piece& p) {
    u = max(p.rb < live ? base + p.rb * size + kOpen + p.page1 : u + 1, u + 1);
    if (u < end && p.ends && p.rb == a.row_blocks - 1) next_sequence(a);
  }
};

// The parts of a row block that several ranges share, joined by a second kernel (in this
// one, by the last workgroup to arrive, each step of the exchange is a way to memory and
// back: 8 us more for one short sequence, 60 for 32 x 4 parts of 128 rows).  A range leaves
// the part of the row block that it ends in at slot 2 r + 1, that of the one that it begins
// in at 2 r: O as the wavefronts' registers have it, [wave][tile, 4 features][lane] of 4
// floats, so that stores and loads are whole lines, then (m, l) of its rows.  Behind the slots a
// range has the (sequence, row block) that it began and did not end (-1: none) and whether it
// ended the one that it began within; behind those lies the number of ranges.
__host__ __device__ constexpr int64_t slot_floats(int rows, int rank) { return static_cast<int64_t>(rows) * (rank + 2); }
__device__ __forceinline__ float* slot_of(const LatentArgs& a, int slot, int rank) {
  return a.ws + slot * slot_floats(a.block_rows, rank);
}
__device__ __forceinline__ int32_t* bounds_of(const LatentArgs& a, int range, int rank) {
  return reinterpret_cast<int32_t*>(slot_of(a, 2 * a.ranges, rank)) + 4 * range;
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

__device__ __forceinline__ int uniform_here(int x) {
  asm volatile("" : "+s"(x));
  return x;
}

// Waits until no more than N of the wavefront's loads are on their way.
template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// Rows of a page in LDS are 128 bytes for each stick; unit u (16 bytes) of token t
// lies at u ^ key(t).  Of the keys that are linear in t's bits this is the simplest with which
// neither the reads of K's rows (16 tokens x 4 units) nor the transposing ones (4 tokens x 4
// units twice) meet in a bank: 4 and 2 cycles a read (measured; t & 7: 4 and 4).
__device__ __forceinline__ int key_of(int t) { return (t & 2) << 1 | (t & 4) >> 1; }
// That of the weights' rows, whose reads are 32 rows x 2 units.
__device__ __forceinline__ int row_key(int r) { return (r & 2) << 1 | ((r >> 2) & 3); }

// The rows' queries on their way into LDS at `to`, 8 rows to a wavefront: the latent features
// [rows][RANK], then the rotated ones, unit u of row r at u ^ (r & 15), u ^ (r / 2 & 7).  Offsets are
// those from the first row's token, 31 bits.  Rows that are not there have the last one's: what they
// get is given up.
template <int RANK, int WAVES>
__device__ __forceinline__ void load_queries(const LatentArgs& a, int b, int n, int row0, int wave, int lane, uint32_t to) {
  const int last = min(a.rows, n * a.H) - 1, i0 = static_cast<int>(fdiv(row0, a.by_h));
  const dma_rsrc q = dma_buffer(a.q + b * a.q_sb + i0 * a.q_st, 0x7fffff00), qr = dma_buffer(a.qr + b * a.qr_sb + i0 * a.qr_st, 0x7fffff00);
  auto from = [&](int r, int64_t st, int64_t sh) {
    const int row = min(row0 + r, last), i = static_cast<int>(fdiv(row, a.by_h));
    return 2 * (static_cast<uint32_t>(i - i0) * static_cast<uint32_t>(st) + static_cast<uint32_t>(row - i * a.H) * static_cast<uint32_t>(sh));
  };
#pragma unroll 1
  for (int k = 0; k < 8; ++k) {
    const int r = k * WAVES + wave;
    if (lane < RANK / 8) dma16(q, to + r * RANK * 2, (lane ^ (r & 15)) * 16, from(r, a.q_st, a.q_sh));
  }
  const int r = 8 * wave + lane / 8;
  dma16(qr, to + WAVES * 8 * RANK * 2 + wave * 1024, from(r, a.qr_st, a.qr_sh) + ((lane & 7) ^ (r / 2 & 7)) * 16, 0);
}

// Whether a token in LDS, NS sticks of 128 bytes `stride` apart, holds a NaN or an infinity: a decode
// step's own one, which every row attends, so that the rows are NaN.
template <int NS>
__device__ __forceinline__ bool token_odd(const uint8_t* token, int stride, int lane) {
  uint32_t found = 0;
#pragma unroll
  for (int u = 0; u < 8 * NS; u += 64)
    if (u + lane < 8 * NS) {
      const u32x4 w = *reinterpret_cast<const u32x4*>(token + (u + lane) / 8 * stride + (u + lane) % 8 * 16);
#pragma unroll
      for (int e = 0; e < 4; ++e) found |= (w[e] & 0x7c007c00u) + 0x04000400u;
    }
  return __ballot((found & 0x80008000u) != 0) != 0;
}

// Up to 32 rows: four wavefronts, each a SIMD's alone, have 32 rows x 16 tokens of a page of scores,
// and then all 64 tokens of 32 rows x a quarter of O's features, which stay in 64 registers.
template <int RANK>
__global__ __launch_bounds__(kParts * 64, 1) void latent_kernel(LatentArgs a) {
  constexpr int WAVES = kParts, ROWS = kTile;
  constexpr int NS = (RANK + kRope) / 64;     // sticks
  constexpr int OS = RANK / 64 / kParts;      // sticks of O of a wavefront
  constexpr int DT = 2 * OS;                  // tiles of it, 32 features each
  constexpr int NQ = (RANK + kRope) / 32;     // steps of the first product
  constexpr int NR = 2;                       // its tiles of 16 rows
  constexpr int TG = kParts;                  // wavefronts that share a row's tokens in it
  constexpr int NT = 4;                       // scores of a lane's row
  constexpr int BUF = NS * kStick;
  constexpr int SHARE = 8 * NS / WAVES;       // loads of a wavefront for a page
  static_assert(ROWS * (RANK + kRope) * 2 <= BUF, "the rows' queries fit a page's buffer");
  __shared__ __align__(16) uint8_t s_mem[2 * BUF];
  __shared__ __align__(16) _Float16 s_p[ROWS * kPage];  // weights: 8 units of 8 tokens a row, unit u at u ^ row_key
  __shared__ float s_max[TG * ROWS], s_sum[TG * ROWS];  // of a page's scores; of all weights
  __shared__ float s_ref[ROWS];
  __shared__ uint32_t s_odd[WAVES];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
  const int col = lane & 31, half = lane >> 5, l16 = lane & 15, g16 = lane >> 4;
  const int part = wave;  // first product: tokens 16 part ..; second: features
  const uint32_t lds0 = lds_address(s_mem);
  Walk walk;
  const int range = walk.start(a, lane);
  if (range < 0) return;
  if (threadIdx.x == 0 && range == 0) *bounds_of(a, a.ranges, RANK) = walk.used;
  int open_b = -1, open_rb = 0, ended = 0;

  // K's row of a lane (16 tokens further its key is the same), units g16 and 4 + g16.  C^T: 4 features
  // of token 8 half + l16 / 4 of the wavefront's first tile; odd tiles and tokens 4 further turn
  // the unit's bits 2 and 1.
  const int k_tok = 16 * part + l16;
  const int k_lane = k_tok * 128 + ((g16 ^ key_of(k_tok)) * 16);
  const int v_tok = 8 * half + l16 / 4;
  const int v_lane = OS * part * kStick + v_tok * 128 + (((2 * (g16 & 1) + ((lane >> 1) & 1)) ^ key_of(v_tok)) * 16) + 8 * (lane & 1);
  auto tr = [&](int at) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(s_mem + at));
  };

  for (; walk.u < walk.end;) {
    const Walk::Piece pc = walk.piece(a);
    const int b = walk.b;
    const Seq sq = walk.seq;
    const int total = sq.ctx + sq.n;
    const int row0 = pc.rb * a.block_rows, p0 = pc.page0, p1 = pc.page1;
    Pages pages(a, b, lane, p0);

    // `sticks` sticks of a page from s0 on, on their way into buffer `buf`: of their chunks (8
    // tokens of a stick) one of SHARES.  Tokens that do not exist are zeros.
    auto load = [&](int64_t page, int p, int buf, auto sticks, int s0, int share, auto shares) {
      constexpr int STICKS = decltype(sticks)::value, SHARES = decltype(shares)::value;
      const dma_rsrc r = dma_buffer(a.pages + page * (NS * (kStick / 2)), BUF);
      const int t = here(lane) / 8, n = total - p * kPage - 8 * share - t;
      const uint32_t off = t * 128 + (((lane & 7) ^ key_of(t)) * 16);
      const uint32_t at = uniform_here(s0 * kStick + share * 1024), to = lds0 + buf * BUF + at;
      auto go = [&](auto whole) {
#pragma unroll
        for (int c = 0; c < 8 / SHARES; ++c)
#pragma unroll
          for (int s = 0; s < STICKS; ++s)
            dma16(r, to + s * kStick + c * SHARES * 1024, decltype(whole)::value || c * SHARES * 8 < n ? off : BUF,
                  at + s * kStick + c * SHARES * 1024);
      };
      if ((p + 1) * kPage <= total)
        go(std::true_type{});
      else
        go(std::false_type{});
    };
    typedef std::integral_constant<int, 1> One;
    typedef std::integral_constant<int, WAVES> Shared;
    // A wavefront loads the sticks of its features, which only it reads in the second product, and
    // its share of the rotated keys.
    auto load_page = [&](int64_t page, int p, int buf) {
      load(page, p, buf, std::integral_constant<int, OS>{}, OS * part, 0, One{});
      load(page, p, buf, One{}, NS - 1, wave, Shared{});
    };
    auto token_of_row = [&](int row) {  // its new token; sq.n or more: none
      return row < a.rows ? static_cast<int>(fdiv(row, a.by_h)) : sq.n;
    };
    int64_t next = 0;  // the page after the ones on their way
    if (p0 < p1) {
      load_queries<RANK, WAVES>(a, b, sq.n, row0, wave, lane, lds0 + BUF);
      load_page(pages.at(p0), p0, 0);
      if (p0 + 1 < p1) next = pages.at(p0 + 1);
      wait_loads<SHARE>();
    }
    __syncthreads();
    f16x8 qf[NR][NQ];
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
      for (int s = 0; s < NQ; ++s) {
        const int r = 16 * n + here(l16);
        const int at = 32 * s < RANK ? r * RANK * 2 + ((4 * s + g16) ^ (r & 15)) * 16
                                     : ROWS * RANK * 2 + r * kRope * 2 + ((4 * s - RANK / 8 + g16) ^ (r / 2 & 7)) * 16;
        qf[n][s] = *reinterpret_cast<const f16x8*>(s_mem + BUF + at);
      }
#pragma unroll
    for (int s = 0; s < NQ; ++s)
#pragma unroll
      for (int n = 0; n < NR; ++n) asm volatile("" : "+v"(qf[n][s]));  // they are read
    if (threadIdx.x < ROWS) s_ref[threadIdx.x] = -INFINITY;
    __syncthreads();
    if (p0 + 1 < p1) load_page(next, p0 + 1, 1);
    f32x16 o[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int x = 0; x < 16; ++x) o[dt][x] = 0.f;
    float m[NR], l[NR];  // of a lane's rows in the first product; l: of this lane's tokens
#pragma unroll
    for (int n = 0; n < NR; ++n) m[n] = -INFINITY, l[n] = 0.f;

    // EDGE: some of the page's tokens are new or do not exist.  (In a copy of its own: its loads of
    // masks would make every page wait for the ones on their way.)
    auto step = [&](int p, auto edge_tag) {
      constexpr bool EDGE = decltype(edge_tag)::value;
      const int buf = (p - p0) & 1;
      if (p + 1 < p1)
        wait_loads<SHARE>();  // the next page's
      else
        wait_loads<0>();
      __syncthreads();  // the page is there
      const bool more = p + 2 < p1;
      if (more) next = pages.at(p + 2);
      uint32_t odd = 0;                            // of this wavefront's tokens, new ones that hold a NaN or an infinity
      if (EDGE && (a.T > 1 || a.mask)) {
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
        odd = s_odd[wave];  // (wavefront w looked at tokens 16 w ..)
      } else if (EDGE && sq.n > 0) {
        pages.poisoned |= token_odd<NS>(s_mem + buf * BUF + sq.ctx % kPage * 128, kStick, here(lane));
      }

      // The scores: sc[n][x] of row 16 n + l16, token 16 part + tok(x).
      float sc[NR][NT];
      auto tok = [&](int x, int ln) { return 16 * (x / 4) + 4 * (ln / 16) + x % 4; };
      {
        const uint8_t* kb = s_mem + buf * BUF;
        const int k_at[2] = {k_lane, k_lane ^ 64};
        // kAhead operands on their way; in this order, the scheduler would read each when it is due
        constexpr int kAhead = 8;
        f16x8 kf[kAhead];
        auto k_of = [&](int x) { return *reinterpret_cast<const f16x8*>(kb + k_at[x % 2] + x / 2 * kStick); };
#pragma unroll
        for (int x = 0; x < kAhead; ++x) kf[x] = k_of(x);
        f32x4 acc[2][NR] = {};  // four chains: a product waits 64 cycles for the one before it and takes 16
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int x = 0; x < NQ; ++x) {
#pragma unroll
          for (int n = 0; n < NR; ++n)
            acc[x % 2][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[x % kAhead], qf[n][x], acc[x % 2][n], 0, 0, 0);
          if (x + kAhead < NQ) kf[x % kAhead] = k_of(x + kAhead);
          __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int n = 0; n < NR; ++n)
#pragma unroll
          for (int x = 0; x < NT; ++x) sc[n][x] = acc[0][n][x] + acc[1][n][x];
      }
      const int ln = here(lane);
#pragma unroll
      for (int n = 0; n < NR; ++n) {
        uint32_t seen = ~0u;
        if constexpr (EDGE) {
          const int j0 = p * kPage + 16 * part - sq.ctx;
          const int i = min(token_of_row(row0 + 16 * n + ln % 16), sq.n - 1);
          seen = 0;
          if (a.mask) {
            const uint8_t* mask = a.mask + b * a.m_sb + max(i, 0) * a.m_si;
            uint8_t keep[NT];
#pragma unroll
            for (int x = 0; x < NT; ++x) keep[x] = mask[min(max(j0 + tok(x, ln), 0), a.T - 1) * a.m_sj];
#pragma unroll
            for (int x = 0; x < NT; ++x) {
              const int j = j0 + tok(x, ln);
              seen |= static_cast<uint32_t>(j < 0 || (j < sq.n && keep[x] != 0)) << x;
            }
          } else {
#pragma unroll
            for (int x = 0; x < NT; ++x) seen |= static_cast<uint32_t>(j0 + tok(x, ln) <= i) << x;
          }
        }
        float mx = -INFINITY;
#pragma unroll
        for (int x = 0; x < NT; ++x) {
          float v = sc[n][x] * a.scale_log2;
          if (EDGE) v = !((seen >> x) & 1) ? -INFINITY : (odd >> tok(x, ln)) & 1 ? NAN : v;
          sc[n][x] = v;
          mx = fmaxf(mx, v);
        }
        mx = xor32_max(xor16_max(mx));
        if (ln / 16 == n) s_max[part * ROWS + 16 * n + ln % 16] = mx;
      }
      // Weights relative to the reference as it is.  They round to fp16 for the product (a
      // relative 2^-12 on average); their sum stays in fp32.
      float add[NR];
      auto weigh = [&] {
#pragma unroll
        for (int n = 0; n < NR; ++n) {
          const float mu = m[n] == -INFINITY ? 0.f : m[n];  // a row that has attended nothing yet: weights 0
          add[n] = 0.f;
          const int row = 16 * n + ln % 16;
#pragma unroll
          for (int x = 0; x < NT; x += 4) {
            f16x4 w4;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float w = exp2_of(sc[n][x + e] - mu);
              add[n] += w;
              w4[e] = static_cast<_Float16>(w);
            }
            const int t = 16 * part + tok(x, ln);  // of 4
            *reinterpret_cast<f16x4*>(&s_p[row * kPage + (((t / 8) ^ row_key(row)) * 8) + t % 8]) = w4;
          }
        }
      };
      weigh();
      __syncthreads();
      // Where a row's scores pass its reference too far, it moves.
      bool moves = false;
#pragma unroll
      for (int k = 0; k < 2; ++k) moves = moves || s_max[64 * k + ln] > s_ref[(64 * k + ln) % ROWS] + kAbove;
      if (__any(moves)) {
        auto ref_of = [&](int r) {  // a row's new reference
          float top = s_max[r];
#pragma unroll
          for (int k = 1; k < TG; ++k) top = fmaxf(top, s_max[k * ROWS + r]);
          return top > s_ref[r] + kAbove ? top - kBelow : s_ref[r];  // its own: what others attend does not turn its roundings
        };
        auto factor = [](float from, float to) { return from == -INFINITY ? 0.f : exp2_of(from - to); };
        const int c = here(col), th = here(threadIdx.x) % ROWS;
        const float alpha = factor(s_ref[c], ref_of(c)), ref = ref_of(th);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int x = 0; x < 16; ++x) o[dt][x] *= alpha;
#pragma unroll
        for (int n = 0; n < NR; ++n) {
          const float to = ref_of(16 * n + ln % 16);
          l[n] *= factor(m[n], to);
          m[n] = to;
        }
        __syncthreads();  // the old references and the weights are read
        if (threadIdx.x < ROWS) s_ref[th] = ref;
        weigh();
        __syncthreads();
      }
#pragma unroll
      for (int n = 0; n < NR; ++n) l[n] += add[n];
      const int v_at[2] = {buf * BUF + v_lane, (buf * BUF + v_lane) ^ 64};
      // Sticks that no wavefront reads any more take the page after the next.
      if (more) load(next, p + 2, buf, One{}, NS - 1, wave, Shared{});
      f16x8 w[4];
#pragma unroll
      for (int s = 0; s < 4; ++s) w[s] = *reinterpret_cast<const f16x8*>(&s_p[(ln % 32) * kPage + (((2 * s + ln / 32) ^ row_key(ln)) * 8)]);
      // Operand x of C^T: tile v_tile(x) of the wavefront (two to a stick), tokens 16 v_step(x) .. +
      // 15, stick after stick.
      auto v_tile = [](int x) { return x / 8 * 2 + x % 2; };
      auto v_step = [](int x) { return x / 2 % 4; };
      constexpr int kAhead = 6, NV = 8 * OS;
      f16x8 vf[kAhead];
      auto v_of = [&](int x) {
        const int at = v_tile(x) / 2 * kStick + v_step(x) * 16 * 128, odd_tile = v_tile(x) & 1;
        const s16x4 lo = tr(v_at[odd_tile] + at), hi = tr((v_at[odd_tile] ^ 32) + at + 4 * 128);
        return __builtin_bit_cast(f16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
      };
#pragma unroll
      for (int x = 0; x < kAhead; ++x) vf[x] = v_of(x);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int x = 0; x < NV; ++x) {
        f32x16& y = o[v_tile(x)];
        y = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[x % kAhead], w[v_step(x)], y, 0, 0, 0);
        if (x + kAhead < NV) vf[x % kAhead] = v_of(x + kAhead);
        __builtin_amdgcn_sched_barrier(0);
        // a stick is read: this wavefront alone reads it, in this product
        if (x % 8 == 7 && more) load(next, p + 2, buf, One{}, OS * part + x / 8, 0, One{});
      }
    };
    // Every row attends every token below ctx.
    const int whole = min(max(sq.ctx / kPage, p0), p1);
    for (int p = p0; p < whole; ++p) step(p, std::false_type{});
    for (int p = whole; p < p1; ++p) step(p, std::true_type{});
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      const int r = 16 * n + here(l16);
      const bool live = token_of_row(row0 + r) < sq.n;
      l[n] = xor32_sum(xor16_sum(l[n]));
      if (!live) l[n] = 0.f;
      if ((pages.poisoned || sq.bad) && live) l[n] = NAN;
      if (g16 == n) s_sum[part * ROWS + r] = l[n];
    }
    __syncthreads();
    const int out_row = col;
    float L = 0.f;
#pragma unroll
    for (int k = 0; k < TG; ++k) L += s_sum[k * ROWS + out_row];
    const float M = L == 0.f ? -INFINITY : s_ref[out_row];
    if (pc.begins && pc.ends) {
      if (row0 + out_row < a.rows)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int x = 0; x < 4; ++x)
            store_row4<RANK>(a, b, row0 + out_row, 32 * (DT * part + dt) + 8 * x + 4 * half,
                             f32x4{o[dt][4 * x], o[dt][4 * x + 1], o[dt][4 * x + 2], o[dt][4 * x + 3]}, M, L);
    } else {
      float* slot = slot_of(a, 2 * range + (pc.begins ? 1 : 0), RANK);
      if (pc.begins) open_b = b, open_rb = pc.rb;
      if (pc.ends) ended = 1;
      if (row0 + out_row < a.rows)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int x = 0; x < 4; ++x)
            *reinterpret_cast<f32x4*>(slot + ((wave * DT + dt) * 4 + x) * 256 + lane * 4) =
              f32x4{o[dt][4 * x], o[dt][4 * x + 1], o[dt][4 * x + 2], o[dt][4 * x + 3]};
      if (part == 0 && half == 0) {
        float* ml = slot + ROWS * RANK + out_row * 2;
        ml[0] = M, ml[1] = L;
      }
    }
    walk.advance(a, pc);
    wait_loads<0>();  // (those behind the last page, too)
    __syncthreads();  // LDS is read before the next piece writes it
  }
  if (threadIdx.x == 0) {
    int32_t* x = bounds_of(a, range, RANK);
    x[0] = open_b, x[1] = open_rb, x[2] = ended;
  }
}

// 64 rows, in two groups of four wavefronts, one of each on a SIMD: while one group has the scores
// and weights of a tile of 32 tokens, the other multiplies the weights of the tile before it with C,
// so that neither's waits leave the matrix cores idle (in step, 8 wavefronts took 76 us for 32 x 4096
// tokens x 128 heads, so 72).
//   scores: a wavefront has 16 rows x the tile, Q in registers
//   sums:   a wavefront has 64 rows x a quarter of O's features, in 128 registers
// Four tiles lie in LDS: one in each product, two on their way.  A load into LDS of 1 KiB holds up
// its wavefront 25 cycles times those in line, so that the second group has two thirds of them, before
// its products, and the first one the others, behind its weights (between the products 85 us, all
// in the second group 79).
template <int RANK>
__global__ __launch_bounds__(2 * kParts * 64, 2) void latent_rows_kernel(LatentArgs a) {
  constexpr int ROWS = 64, WAVES = 2 * kParts, TOKS = 32;
  constexpr int NS = (RANK + kRope) / 64;     // sticks
  constexpr int OS = RANK / 64 / kParts;      // sticks of O of a wavefront
  constexpr int DT = 2 * OS;                  // tiles of it, 32 features each
  constexpr int NQ = (RANK + kRope) / 32;     // steps of the first product
  constexpr int STICK = TOKS * 128, TILE = NS * STICK;
  constexpr int LOADS_A = NS / 3, LOADS = NS - LOADS_A;  // of a wavefront of the first group for a tile, of the second
  static_assert(ROWS * (RANK + kRope) * 2 == 2 * TILE, "the rows' queries fit the buffers of two tiles");
  __shared__ __align__(16) uint8_t s_mem[4 * TILE];
  __shared__ __align__(16) _Float16 s_p[ROWS * 64];  // weights of two tiles: 4 units of 8 tokens each, unit u of a row at u ^ row_key
  __shared__ float s_alpha[2][ROWS];                 // of two tiles: what O is to be multiplied with before
  __shared__ int s_moved[2][4];                      // whether any of 16 rows is
  __shared__ float s_ref[ROWS], s_sum[ROWS];         // at the end
  __shared__ uint32_t s_odd[WAVES];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
  const int col = lane & 31, half = lane >> 5, l16 = lane & 15, g16 = lane >> 4;
  const bool first = wave < kParts;
  const int part = wave % kParts;  // first group: rows 16 part ..; second: features
  const uint32_t lds0 = lds_address(s_mem);
  Walk walk;
  const int range = walk.start(a, lane);
  if (range < 0) return;
  if (threadIdx.x == 0 && range == 0) *bounds_of(a, a.ranges, RANK) = walk.used;
  int open_b = -1, open_rb = 0, ended = 0;

  for (; walk.u < walk.end;) {
    const Walk::Piece pc = walk.piece(a);
    const int b = walk.b;
    const Seq sq = walk.seq;
    const int total = sq.ctx + sq.n, row0 = pc.rb * ROWS;
    const int t0 = 2 * pc.page0, n = max(min(2 * pc.page1, (total + TOKS - 1) / TOKS) - t0, 0);  // tiles t0 .. t0 + n
    Pages pages(a, b, lane, pc.page0);
    int64_t page = 0;  // of the tile that is loaded next
    auto token_of_row = [&](int row) {  // its new token; sq.n or more: none
      return row < a.rows ? static_cast<int>(fdiv(row, a.by_h)) : sq.n;
    };
    // A group's loads of tile t0 + i: sticks, 8 tokens to a wavefront.  Tokens that do not exist are
    // zeros.
    auto load_tile = [&](int i) {
      if ((t0 + i) % 2 == 0) page = pages.at((t0 + i) / 2);
      const int ln = here(lane), t = ln / 8, at = (t0 + i) % 2 * TOKS + 8 * part;
      const uint32_t off = (t0 + i) * TOKS + 8 * part + t < total ? t * 128 + (((ln & 7) ^ key_of(t)) * 16) : NS * kStick;
      const dma_rsrc r = dma_buffer(a.pages + page * (NS * (kStick / 2)), NS * kStick);
      const uint32_t to = lds0 + (i & 3) * TILE + part * 1024;
      if (first)
#pragma unroll
        for (int k = LOADS; k < NS; ++k) dma16(r, to + k * STICK, off, k * kStick + at * 128);
      else
#pragma unroll
        for (int k = 0; k < LOADS; ++k) dma16(r, to + k * STICK, off, k * kStick + at * 128);
    };
    constexpr int Q_AT = 2 * TILE;  // the queries: in the last two buffers
    if (n > 0) {
      load_queries<RANK, WAVES>(a, b, sq.n, row0, wave, lane, lds0 + Q_AT);
      load_tile(0);
      if (n > 1) load_tile(1);
    }
    wait_loads<0>();
    __syncthreads();

    // What a row does not attend must not meet its weight of 0: new tokens that hold a NaN or an
    // infinity become zeros, and the rows that attend them NaN.  All wavefronts, before a tile's first
    // product; bit t of the result: token t.
    auto odd_of = [&](int i) -> uint32_t {
      const int th = here(threadIdx.x), t = th / 16, at = (t0 + i) * TOKS + t;
      uint8_t* x = s_mem + (i & 3) * TILE + t * 128 + (th % 8) * 16;
      uint32_t found = 0;
      const bool fresh = at >= sq.ctx && at < total;
      for (int s = th / 8 % 2; s < NS && fresh; s += 2) {
        const u32x4 w = *reinterpret_cast<const u32x4*>(x + s * STICK);
#pragma unroll
        for (int e = 0; e < 4; ++e) found |= (w[e] & 0x7c007c00u) + 0x04000400u;
      }
      const uint64_t lanes = __ballot((found & 0x80008000u) != 0);
      const bool bad = (lanes >> (lane & 48)) & 0xffff;
      for (int s = th / 8 % 2; s < NS && bad; s += 2) *reinterpret_cast<u32x4*>(x + s * STICK) = u32x4{0, 0, 0, 0};
      const uint64_t all = __ballot(bad);
      if (lane == 0) s_odd[wave] = (all & 1) | (all >> 15 & 2) | (all >> 30 & 4) | (all >> 45 & 8);
      __syncthreads();
      uint32_t odd = 0;
#pragma unroll
      for (int k = 0; k < WAVES; ++k) odd |= s_odd[k] << (4 * k);
      return odd;
    };
    // Every row attends every token below ctx.
    auto edge_at = [&](int i) { return (t0 + i + 1) * TOKS > sq.ctx; };

    if (first) {
      f16x8 qf[NQ];
#pragma unroll
      for (int s = 0; s < NQ; ++s) {
        const int r = 16 * part + here(l16);
        const int at = 32 * s < RANK ? r * RANK * 2 + ((4 * s + g16) ^ (r & 15)) * 16
                                     : ROWS * RANK * 2 + r * kRope * 2 + ((4 * s - RANK / 8 + g16) ^ (r / 2 & 7)) * 16;
        qf[s] = *reinterpret_cast<const f16x8*>(s_mem + Q_AT + at);
      }
#pragma unroll
      for (int s = 0; s < NQ; ++s) asm volatile("" : "+v"(qf[s]));  // they are read
      __syncthreads();
      const int k_lane = l16 * 128 + ((g16 ^ key_of(l16)) * 16);
      float m = -INFINITY, l = 0.f;  // of a lane's row; l: of this lane's tokens
      auto step = [&](int i, auto edge_tag) {
        constexpr bool EDGE = decltype(edge_tag)::value;
        uint32_t odd = 0;
        if (EDGE && (a.T > 1 || a.mask))
          odd = odd_of(i);
        else if (EDGE && sq.n > 0)
          pages.poisoned |= token_odd<NS>(s_mem + (i & 3) * TILE + sq.ctx % TOKS * 128, STICK, here(lane));
        // The scores: sc[x] of row 16 part + l16, token tok(x).
        auto tok = [&](int x, int ln) { return 16 * (x / 4) + 4 * (ln / 16) + x % 4; };
        float sc[8];
        {
          const int kb = (i & 3) * TILE + k_lane, k_at[2] = {kb, kb ^ 64};
          // kAhead operands on their way; in this order, the scheduler would read each when it is due
          constexpr int kAhead = 8, NK = 2 * NQ;
          f16x8 kf[kAhead];
          auto k_of = [&](int x) { return *reinterpret_cast<const f16x8*>(s_mem + k_at[x / 2 % 2] + x / 4 * STICK + x % 2 * (16 * 128)); };
#pragma unroll
          for (int x = 0; x < kAhead; ++x) kf[x] = k_of(x);
          f32x4 acc[2][2] = {};  // four chains: a product waits 64 cycles for the one before it and takes 16
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int x = 0; x < NK; ++x) {
            acc[x / 2 % 2][x % 2] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[x % kAhead], qf[x / 2], acc[x / 2 % 2][x % 2], 0, 0, 0);
            if (x + kAhead < NK) kf[x % kAhead] = k_of(x + kAhead);
            __builtin_amdgcn_sched_barrier(0);
          }
#pragma unroll
          for (int x = 0; x < 8; ++x) sc[x] = acc[0][x / 4][x % 4] + acc[1][x / 4][x % 4];
        }
        const int ln = here(lane);
        uint32_t seen = ~0u;
        if constexpr (EDGE) {
          const int j0 = (t0 + i) * TOKS - sq.ctx, q = min(token_of_row(row0 + 16 * part + ln % 16), sq.n - 1);
          seen = 0;
          if (a.mask) {
            const uint8_t* mask = a.mask + b * a.m_sb + max(q, 0) * a.m_si;
            uint8_t keep[8];
#pragma unroll
            for (int x = 0; x < 8; ++x) keep[x] = mask[min(max(j0 + tok(x, ln), 0), a.T - 1) * a.m_sj];
#pragma unroll
            for (int x = 0; x < 8; ++x) {
              const int j = j0 + tok(x, ln);
              seen |= static_cast<uint32_t>(j < 0 || (j < sq.n && keep[x] != 0)) << x;
            }
          } else {
#pragma unroll
            for (int x = 0; x < 8; ++x) seen |= static_cast<uint32_t>(j0 + tok(x, ln) <= q) << x;
          }
        }
        float mx = -INFINITY;
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          float v = sc[x] * a.scale_log2;
          if (EDGE) v = !((seen >> x) & 1) ? -INFINITY : (odd >> tok(x, ln)) & 1 ? NAN : v;
          sc[x] = v;
          mx = fmaxf(mx, v);
        }
        mx = xor32_max(xor16_max(mx));
        // Where a row's scores pass its reference too far, it moves.
        const bool moves = mx > m + kAbove;
        float alpha = 1.f;
        if (moves) {
          const float to = mx - kBelow;
          alpha = m == -INFINITY ? 0.f : exp2_of(m - to);
          m = to;
        }
        const int any = __any(moves);
        if (ln < 16) s_alpha[i & 1][16 * part + ln] = alpha;
        if (ln == 0) s_moved[i & 1][part] = any;
        // Weights round to fp16 for the product (a relative 2^-12 on average); their sum stays in fp32.
        const float mu = m == -INFINITY ? 0.f : m;  // a row that has attended nothing yet: weights 0
        float add = 0.f;
        const int row = 16 * part + ln % 16;
#pragma unroll
        for (int x = 0; x < 8; x += 4) {
          f16x4 w4;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float w = exp2_of(sc[x + e] - mu);
            add += w;
            w4[e] = static_cast<_Float16>(w);
          }
          const int t = TOKS * (i & 1) + tok(x, ln);  // of 4
          *reinterpret_cast<f16x4*>(&s_p[row * 64 + (((t / 8) ^ row_key(row)) * 8) + t % 8]) = w4;
        }
        l = l * alpha + add;
        if (i + 2 < n) {
          load_tile(i + 2);
          wait_loads<LOADS_A>();  // tile i + 1 is there
        } else {
          wait_loads<0>();
        }
        __syncthreads();
      };
      int i = 0;
      for (; i < n && !edge_at(i); ++i) step(i, std::false_type{});
      for (; i < n; ++i) step(i, std::true_type{});
      const int r = 16 * part + here(l16);
      const bool live = token_of_row(row0 + r) < sq.n;
      l = xor32_sum(xor16_sum(l));
      if (!live) l = 0.f;
      if ((pages.poisoned || sq.bad) && live) l = NAN;
      if (g16 == 0) s_sum[r] = l, s_ref[r] = l == 0.f ? -INFINITY : m;
      if (n > 0) __syncthreads();  // the second group's last tile
      __syncthreads();
    } else {
      __syncthreads();  // the queries are read
      const int v_tok = 8 * half + l16 / 4;
      const int v_lane = OS * part * STICK + v_tok * 128 + (((2 * (g16 & 1) + ((lane >> 1) & 1)) ^ key_of(v_tok)) * 16) + 8 * (lane & 1);
      auto tr = [&](int at) {
        return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(s_mem + at));
      };
      f32x16 o[2][DT];
#pragma unroll
      for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int x = 0; x < 16; ++x) o[g][dt][x] = 0.f;
      if (n > 0) {
        if (edge_at(0) && (a.T > 1 || a.mask)) odd_of(0);
        if (n > 2) load_tile(2);
        n > 2 ? wait_loads<LOADS>() : wait_loads<0>();  // tile 1 is there
        __syncthreads();
      }
      for (int i = 1; i <= n; ++i) {
        if (i < n && edge_at(i) && (a.T > 1 || a.mask)) odd_of(i);
        const bool more = i + 2 < n;
        {
          const int j = i - 1, ln = here(lane), c = ln % 32;
          int moved = 0;
#pragma unroll
          for (int k = 0; k < 4; ++k) moved |= s_moved[j & 1][k];
          if (__any(moved)) {
#pragma unroll
            for (int g = 0; g < 2; ++g) {
              const float alpha = s_alpha[j & 1][32 * g + c];
#pragma unroll
              for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int x = 0; x < 16; ++x) o[g][dt][x] *= alpha;
            }
          }
          f16x8 w[2][2];
#pragma unroll
          for (int g = 0; g < 2; ++g)
#pragma unroll
            for (int s = 0; s < 2; ++s)
              w[g][s] = *reinterpret_cast<const f16x8*>(&s_p[(32 * g + c) * 64 + (((4 * (j & 1) + 2 * s + ln / 32) ^ row_key(c)) * 8)]);
          // Operand x of C^T: tile x % DT of the wavefront (two to a stick), tokens 16 (x / DT) .. + 15.
          const int vb = (j & 3) * TILE + v_lane;
          constexpr int kAhead = 4, NV = 2 * DT;
          f16x8 vf[kAhead];
          auto v_of = [&](int x) {
            const int at = x % DT / 2 * STICK + x / DT * 16 * 128, turn = x & 1 ? 64 : 0;
            const s16x4 lo = tr((vb ^ turn) + at), hi = tr((vb ^ turn ^ 32) + at + 4 * 128);
            return __builtin_bit_cast(f16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
          };
#pragma unroll
          for (int x = 0; x < kAhead; ++x) vf[x] = v_of(x);
          __builtin_amdgcn_sched_barrier(0);
          if (more) load_tile(i + 2);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int x = 0; x < NV; ++x) {
#pragma unroll
            for (int g = 0; g < 2; ++g)
              o[g][x % DT] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[x % kAhead], w[g][x / DT], o[g][x % DT], 0, 0, 0);
            if (x + kAhead < NV) vf[x % kAhead] = v_of(x + kAhead);
            __builtin_amdgcn_sched_barrier(0);
          }
        }
        more ? wait_loads<LOADS>() : wait_loads<0>();  // tile i + 1 is there
        __syncthreads();
      }
      __syncthreads();  // the rows' sums
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const int out_row = 32 * g + col;
        const float L = s_sum[out_row], M = s_ref[out_row];
        if (pc.begins && pc.ends) {
          if (row0 + out_row < a.rows)
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
              for (int x = 0; x < 4; ++x)
                store_row4<RANK>(a, b, row0 + out_row, 32 * (DT * part + dt) + 8 * x + 4 * half,
                                 f32x4{o[g][dt][4 * x], o[g][dt][4 * x + 1], o[g][dt][4 * x + 2], o[g][dt][4 * x + 3]}, M, L);
        } else {
          float* slot = slot_of(a, 2 * range + (pc.begins ? 1 : 0), RANK);
          if (row0 + out_row < a.rows)
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
              for (int x = 0; x < 4; ++x)
                *reinterpret_cast<f32x4*>(slot + (((g * kParts + part) * DT + dt) * 4 + x) * 256 + lane * 4) =
                    f32x4{o[g][dt][4 * x], o[g][dt][4 * x + 1], o[g][dt][4 * x + 2], o[g][dt][4 * x + 3]};
          if (part == 0 && half == 0) {
            float* ml = slot + ROWS * RANK + out_row * 2;
            ml[0] = M, ml[1] = L;
          }
        }
      }
    }
    if (!(pc.begins && pc.ends)) {
      if (pc.begins) open_b = b, open_rb = pc.rb;
      if (pc.ends) ended = 1;
    }
    walk.advance(a, pc);
    wait_loads<0>();
    __syncthreads();  // LDS is read before the next piece writes it
  }
  if (threadIdx.x == 0) {
    int32_t* x = bounds_of(a, range, RANK);
    x[0] = open_b, x[1] = open_rb, x[2] = ended;
  }
}

// Joins the parts of the row block that a range began and did not end: a thread 4 features of a
// row, numbered as they lie in a slot.
template <int RANK, int RG>
__global__ __launch_bounds__(256) void latent_join_kernel(LatentArgs a) {
  constexpr int ROWS = RG * kTile, DT = RANK / 32 / kParts, BLOCKS = ROWS * RANK / 1024;
  const int range = static_cast<int>(blockIdx.x / BLOCKS), at = static_cast<int>(blockIdx.x % BLOCKS) * 256 + threadIdx.x, lane = at % 64;
  const int used = *bounds_of(a, a.ranges, RANK);
  if (range >= used) return;
  const int32_t* open = bounds_of(a, range, RANK);
  const int b = open[0], rb = open[1];
  if (b < 0) return;
  int last = range + 1;  // the range that it ends in
  for (;; last += 64) {
    const uint64_t ended = __ballot(last + lane >= used - 1 || bounds_of(a, last + lane, RANK)[2] != 0);
    if (ended != 0) {
      last += __builtin_ctzll(ended);
      break;
    }
  }
  const int wave = at / (DT * 256), tile = wave % kParts * DT + at / 256 % DT;
  const int r = wave / kParts * kTile + lane % 32, row = rb * ROWS + r;
  if (row >= a.rows) return;
  float M = -INFINITY, L = 0.f;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  merge_parts_once(range, __builtin_amdgcn_readfirstlane(min(last, used - 1)), M, L, acc, [&](int p, float& m, float& l, f32x4& x) {
    const float* slot = slot_of(a, 2 * p + (p == range ? 1 : 0), RANK);
    const float* ml = slot + ROWS * RANK + r * 2;
    m = ml[0], l = ml[1];
    x = *reinterpret_cast<const f32x4*>(slot + at * 4);
  });
  store_row4<RANK>(a, b, row, 32 * tile + 8 * (at / 64 % 4) + 4 * (lane / 32), acc, M, L);
}

struct Plan {
  int groups;  // of 32 rows to a workgroup
  int row_blocks, block_rows, ranges;
  size_t ws_bytes;
};

Plan plan_of(int B, int T, int H, int rank, int max_tokens) {
  Plan p;
  const int64_t rows = static_cast<int64_t>(T) * H;
  p.groups = rows <= kTile ? 1 : 2;
  p.block_rows = kTile * p.groups;
  p.row_blocks = static_cast<int>((rows + p.block_rows - 1) / p.block_rows);
  // One workgroup to a CU, and no more than there could be work for.
  const double most = static_cast<double>(B) * p.row_blocks * (Walk::kOpen + std::max(pages_of(max_tokens), 1));
  p.ranges = static_cast<int>(std::max(1., std::min(256., most / Walk::kLeast)));
  p.ws_bytes = static_cast<size_t>(2 * p.ranges) * slot_floats(p.block_rows, rank) * 4 + 16 * (static_cast<size_t>(p.ranges) + 1);
  return p;
}

bool sizes_ok(int B, int T, int H, int max_ctx) {
  return B >= 0 && T > 0 && H > 0 && max_ctx >= 0 && static_cast<int64_t>(T) * H < (int64_t{1} << 31) - 256 &&
         static_cast<int64_t>(max_ctx) + T < (int64_t{1} << 31) - kPage;
}

template <int RANK>
void launch(const LatentArgs& a, int groups, dim3 grid, hipStream_t st) {
  if (groups == 1)
    latent_kernel<RANK><<<grid, kParts * 64, 0, st>>>(a);
  else
    latent_rows_kernel<RANK><<<grid, 2 * kParts * 64, 0, st>>>(a);
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
  // The rows of a workgroup are addressed from the first one's token, in 31 bits.
  const int tokens = std::min(T - 1, (p.block_rows + H - 2) / H);
  for (const int64_t* st : {q_strides, q_rope_strides})
    SPYRE_REQUIRE(st[1] >= 0 && st[2] >= 0 && static_cast<double>(tokens) * st[1] + static_cast<double>(H - 1) * st[2] < (1 << 30) - rank,
                  SPYRE_EUNSUPPORTED, "strides of q and q_rope are too large");
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
  a.B = B, a.T = T, a.H = H, a.rows = T * H;
  a.max_ctx = max_context_len, a.scale_log2 = scale * kLog2e;
  a.row_blocks = p.row_blocks, a.block_rows = p.block_rows;
  a.block_shift = p.groups == 1 ? 5 : 6, a.ranges = p.ranges;
  SPYRE_REQUIRE(static_cast<double>(B) * p.row_blocks * (pages_of(max_context_len + T) + Walk::kOpen + 1) < (1 << 30),
                SPYRE_EUNSUPPORTED, "too many pages or rows");
  a.by_h = make_fastdiv(static_cast<uint32_t>(H)), a.by_ranges = make_fastdiv(static_cast<uint32_t>(p.ranges));
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid(static_cast<uint32_t>((p.ranges + 7) / 8 * 8));
  rank == 512 ? launch<512>(a, p.groups, grid, st) : launch<256>(a, p.groups, grid, st);
  hipError_t e = hipGetLastError();
  SPYRE_REQUIRE(e == hipSuccess, SPYRE_EHIP, "latent attention launch failed: %s", hipGetErrorString(e));
  if (p.ranges > 1) {  // nothing is cut where one range has it all
    const dim3 join(static_cast<uint32_t>(p.ranges * (p.block_rows * rank / 1024)));
    auto go = [&](auto r) {
      constexpr int R = decltype(r)::value;
      p.groups == 1 ? latent_join_kernel<R, 1><<<join, 256, 0, st>>>(a) : latent_join_kernel<R, 2><<<join, 256, 0, st>>>(a);
    };
    rank == 512 ? go(std::integral_constant<int, 512>{}) : go(std::integral_constant<int, 256>{});
    e = hipGetLastError();
    SPYRE_REQUIRE(e == hipSuccess, SPYRE_EHIP, "latent attention join launch failed: %s", hipGetErrorString(e));
  }
  return SPYRE_OK;
}
