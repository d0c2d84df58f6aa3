// Attention of drafted tokens over the paged cache (spyre_paged_tree_attn).
//
// Sequence b holds ctx[b] cached tokens and, behind them in the same pages, n[b]
// drafted ones.  Query row (i, h) of drafted token i < n[b] attends
//   t < ctx[b],  and drafted j < n[b] where mask[b, i, j]   (no mask: j <= i)
//   out = softmax(scale q . K^T) V,   lse its logarithm of the sum
// over fp16 pages (K [D/64, 64 tok, 64], V [D, 64 tok]) or 8-bit ones
// (cache8.h).  Rows that attend nothing, and those from n[b] on, are zeros
// with lse -inf.  One query and no drafted keys is a decode step.
//
// The T g rows that share a KV head (g q heads to it) are the columns of the
// products, 32 to a tile:
//   S^T[tok, row] = K[tok, :] Q^T[:, row]      MFMA 32x32x16, M = 32 tokens
//   O^T[d, row] += V^T[d, tok] P^T[tok, row]
// Both operands of a tile come straight from the pages: an operand lane wants
// 8 numbers along the reduction, and both page forms have the reduced
// dimension innermost.  Two orders are free and chosen so that nothing moves
// between lanes: the order of d in Q K^T (lane half H, MFMAs 2 s and 2 s + 1
// take d = 32 s + 16 H .. + 15, one 16-byte unit of the 8-bit pages), and the
// order of the tokens of a tile (token_of), which leaves lane half H the
// scores of its tokens 16 H .. + 15, just the P the second product wants there.
//
// 8-bit V carries a scale for each token.  It is added to the score as its
// logarithm, so the weights that meet the codes are p * scale relative to the
// largest such, whatever the scales' range; the row sum divides it out again.
// A V row of zeros is stored with scale 1, far above that of ordinary rows (2^-7
// for e4m3): attended with 0.999, as an attention sink is, it would press all
// weights that count below fp16's range.  Where a scale is 1 the codes are looked
// at, and a row of zeros then weighs as little as a scale of 0 (2^-60).

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "cache8.h"
#include "decode_dense.h"
#include "fast_div.h"
#include "page_walk.h"
#include "spyre_common.h"

namespace {

using namespace spyre_hip;

typedef c8_f16x8 f16x8;
typedef c8_u32x4 u32x4;
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kTile = 32;  // query rows of a tile, and tokens of an MFMA
constexpr int kF16 = SPYRE_CACHE_F16;
// The running reference of a row's exponents is put kBelow under its largest score
// (log2 units) and moves only when a score passes it by more than kAbove: weights
// up to 2^15 are as exact in fp16 as those up to 1, most steps then skip the
// rescaling of O, and a weight is a normal number of fp16 (a relative 2^-11) down
// to 2^-21 of the largest: many small ones count beside one that takes nearly all
// of a row and whose V adds little, as an attention sink's.
constexpr float kBelow = 7.f, kAbove = 15.f;

struct TreeArgs {
  const _Float16* q;
  int64_t q_sb, q_st, q_sh;
  const uint8_t *k, *v;
  const float *ks, *vs;
  const int32_t *bt, *ctx, *counts;
  const uint8_t* mask;
  int64_t bt_stride, pages_per_seq, num_pages, m_sb, m_si, m_sj;
  _Float16* out;  // [B, T, Hq, D]
  float* lse;     // [B, T, Hq] or null
  float* ws;
  int B, T, Hq, Hkv, g, rows, max_ctx, draft_keys;
  float scale_log2;
  // The rows of a KV head are cut into row_blocks of block_rows; a partial
  // holds `width` of them, the fewer of block_rows and rows.
  int row_blocks, block_rows, width;
  int ranges, min_per, min_cut, each;  // see Walk; each: (sequence, KV head)s a range where that is a whole number, else 0
  uint32_t ticket;      // see finish()
  FastDiv by_g, by_hkv, by_blocks, by_ranges;
};

typedef PageWalk<TreeArgs> Walk;

// The token of MFMA row m of a 32-token tile: row 16 e + 8 a + 4 H + r is token
// 16 H + 8 e + 4 a + r, so that accumulator register i of lane half H is token
// 16 H + i.
__device__ __forceinline__ int token_of(int m) {
  return 16 * ((m >> 2) & 1) + 8 * (m >> 4) + 4 * ((m >> 3) & 1) + (m & 3);
}

// Partials: O [slots][width][D], then (m, l) [slots][width], then an arrival
// flag for each slot; slots are (range, row block, slot 0 / 1).
__device__ __forceinline__ int64_t partial_of(const TreeArgs& a, int range, int rb, int slot, int row) {
  return ((static_cast<int64_t>(range) * a.row_blocks + rb) * 2 + slot) * a.width + row;
}
__device__ __forceinline__ int64_t partials(const TreeArgs& a) {
  return static_cast<int64_t>(a.ranges) * a.row_blocks * 2 * a.width;
}

// 4 features of a finished row.
template <int D>
__device__ __forceinline__ void store_row4(const TreeArgs& a, int b, int i, int head, int d, f32x4 x, float m, float l) {
  const int64_t at = (static_cast<int64_t>(b) * a.T + i) * a.Hq + head;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  f16x4 y;
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = static_cast<_Float16>(l == 0.f ? 0.f : x[e] * inv);
  *reinterpret_cast<f16x4*>(a.out + at * D + d) = y;
  if (a.lse && d == 0) a.lse[at] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
}

// The raw operands of a 32-token step: 8-bit, D / 32 units of 16 codes a lane;
// fp16, twice as many of 8 numbers.
template <int CT, int D>
struct Raw {
  static constexpr int W = CT == kF16 ? 2 : 1;
  u32x4 x[D / 32][W];
};

template <int CT, int W>
__device__ __forceinline__ f16x8 operand(const u32x4 (&x)[W], int e) {
  if constexpr (CT == kF16)
    return __builtin_bit_cast(f16x8, x[e]);
  else
    return codes_to_f16x8<CT>(x[0][2 * e], x[0][2 * e + 1]);
}

// Zeroes the numbers of tokens from n on, of the 16 that a lane's words hold.
template <int CT, int W>
__device__ __forceinline__ void drop_tokens(u32x4 (&x)[W], int n) {
#pragma unroll
  for (int e = 0; e < W; ++e)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      constexpr int PER = CT == kF16 ? 2 : 4, BITS = 32 / PER;  // numbers of a word
      const int keep = n - (4 * e + i) * PER;
      const uint32_t mask = keep <= 0 ? 0u : keep >= PER ? ~0u : (1u << (keep * BITS)) - 1;
      x[e][i] &= mask;
    }
}

// x or-ed over the 16 lanes of a row.
__device__ __forceinline__ uint32_t or16(uint32_t x) {
  x |= static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(x), 0xb1, 0xf, 0xf, false));   // quad_perm 1 0 3 2
  x |= static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(x), 0x4e, 0xf, 0xf, false));   // quad_perm 2 3 0 1
  x |= static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(x), 0x141, 0xf, 0xf, false));  // row_half_mirror
  x |= static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(x), 0x140, 0xf, 0xf, false));  // row_mirror
  return x;
}

// A unit of V's codes (16 tokens of a feature), or-ed over all features: whether
// token t's are all zero (e4m3 has a negative one).
template <int CT>
__device__ __forceinline__ bool zero_row(const u32x4& w, int t) {
  const uint32_t x = t < 8 ? t < 4 ? w[0] : w[1] : t < 12 ? w[2] : w[3];
  return ((x >> (8 * (t % 4))) & (CT == SPYRE_CODES_E4M3 ? 0x7fu : 0xffu)) == 0;
}

// Zeroes a word's infinities and NaNs (int8 has none); whether it held any.
template <int CT>
__device__ __forceinline__ bool drop_odd(uint32_t& w) {
  uint32_t odd = 0;
  if constexpr (CT == kF16)
    odd = ((w & 0x7c00u) == 0x7c00u ? 0xffffu : 0u) | ((w & 0x7c000000u) == 0x7c000000u ? 0xffff0000u : 0u);
  else if constexpr (CT == SPYRE_CODES_E4M3)
    odd = ((((w & 0x7f7f7f7fu) + 0x01010101u) >> 7) & 0x01010101u) * 0xffu;
  w &= ~odd;
  return odd != 0;
}

// Pages are read by buffer loads: the base in scalar registers, 32-bit offsets a
// lane, and every access clamped to the page.
typedef __amdgpu_buffer_rsrc_t Rsrc;
constexpr int kAuxDevice = 16;  // sc1: device scope
constexpr int kAuxOnce = 2;     // non-temporal: read once

__device__ __forceinline__ Rsrc page_rsrc(const void* cache, int64_t head, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(static_cast<const uint8_t*>(cache)) + head * bytes, 0, bytes, 0x00020000);
}

// A wavefront's pages, one after the other from `first` on, as indexes of their
// (page, KV head): 64 table entries at a time, one a lane, so that no page's
// loads wait for its entry.  A page that the table does not name validly is
// page 0 (in bounds) and poisons the rows.
struct Pages {
  const TreeArgs& a;
  const int32_t* trow;
  int kvh, lane, first, ids = 0;
  bool poisoned = false;
  __device__ __forceinline__ Pages(const TreeArgs& args, int b, int kv_head, int lane_, int first_)
      : a(args), trow(args.bt + b * args.bt_stride), kvh(kv_head), lane(lane_), first(first_) {}
  __device__ __forceinline__ int64_t head(int p) {  // p: first, first + 1, ..., each once or again
    const int at = p - first;
    if ((at & 63) == 0) {
      ids = p + lane < a.pages_per_seq ? trow[p + lane] : -1;
      asm volatile("" : "+v"(ids));  // waits here: behind the branch every page would, for all loads in flight
    }
    const int64_t phys = __builtin_amdgcn_readlane(ids, at & 63);
    const bool bad = phys < 0 || phys >= a.num_pages;
    poisoned |= bad;
    return (bad ? 0 : phys) * a.Hkv + kvh;
  }
};

// A lane's row of the T g rows of a KV head.
struct Row {
  int i;      // its drafted token
  int head;   // its q head
  bool live;
  const uint8_t* mask;  // of its token; null: a chain
  // Which of the 16 tokens t + offset(x) the row attends (total: all there
  // are).  Every mask byte is loaded, and none waits for another.
  template <typename Offset>
  __device__ __forceinline__ uint32_t attends16(const TreeArgs& a, const Seq& sq, int t, int total, Offset offset) const {
    uint32_t seen = 0;
    const int j0 = t - sq.ctx, n = total - t;
    if (mask) {
      uint8_t keep[16];
#pragma unroll
      for (int x = 0; x < 16; ++x) keep[x] = mask[min(max(j0 + offset(x), 0), a.T - 1) * a.m_sj];
#pragma unroll
      for (int x = 0; x < 16; ++x)
        seen |= static_cast<uint32_t>(offset(x) < n && (j0 + offset(x) < 0 || keep[x] != 0)) << x;
    } else {
#pragma unroll
      for (int x = 0; x < 16; ++x) seen |= static_cast<uint32_t>(offset(x) < n && j0 + offset(x) <= i) << x;
    }
    return live ? seen : 0u;
  }
};

__device__ __forceinline__ Row row_of(const TreeArgs& a, const Seq& sq, int b, int kvh, int row) {
  Row r;
  r.i = static_cast<int>(fdiv(row, a.by_g));
  r.head = kvh * a.g + row - r.i * a.g;
  r.live = row < a.rows && r.i < sq.n;
  r.mask = a.mask ? a.mask + b * a.m_sb + (r.live ? r.i : 0) * a.m_si : nullptr;
  return r;
}

// Q^T operands of a lane's row: features 32 s + 16 half + 8 e .. + 7.  (A row
// that is not live loads another's.)
template <int DS>
__device__ __forceinline__ void load_q(const TreeArgs& a, int b, const Row& r, int half, f16x8 (&qf)[DS][2]) {
  const _Float16* qp = a.q + b * a.q_sb + (r.live ? r.i * a.q_st + r.head * a.q_sh : 0) + 16 * half;
#pragma unroll
  for (int s = 0; s < DS; ++s)
#pragma unroll
    for (int e = 0; e < 2; ++e) qf[s][e] = *reinterpret_cast<const f16x8*>(qp + 32 * s + 8 * e);
#pragma unroll
  for (int s = 0; s < DS; ++s)
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if (!r.live) qf[s][e] = f16x8{};
}

// The infinities and NaNs of tokens t0 .. t1 - 1 (part 0 / 1: of their pages'
// first / second halves only) that drop_odd left out of O, number by number.
// A lane's numbers of O are those of the features feature(x), x < NR; add(x, f)
// adds to one.
template <int CT, int D, int NR, typename Feature, typename Add>
__device__ __forceinline__ void add_odd(const TreeArgs& a, const Seq& sq, int b, int kvh, const Row& r, int lane, int t0, int t1,
                                        int part, Feature feature, Add add) {
  constexpr int KB = CT == kF16 ? 2 : 1;
  asm volatile("" : "+v"(lane));  // rare: its addresses are not worth registers of the loops before it
  Pages pages(a, b, kvh, lane, t0 / kPage);
  for (int t = t0; t < t1; ++t) {
    const bool attends = r.attends16(a, sq, t, t + 1, [](int x) { return x; }) && (part < 0 || part == (t % kPage) / 32);
    const int64_t head = pages.head(t / kPage);
    const uint8_t* v = a.v + head * (static_cast<int64_t>(kPage) * D * KB);
    float vs = 1.f;  // 8-bit: V's scale if it is not finite
    if constexpr (CT != kF16) {
      const float x = a.vs[head * kPage + t % kPage];
      if (!(__builtin_fabsf(x) <= 0x1.fffffep127f)) vs = x;
    }
#pragma unroll
    for (int x = 0; x < NR; ++x) {
      const int d = feature(x, lane);
      float f;
      if constexpr (CT == kF16) {
        f = static_cast<float>(reinterpret_cast<const _Float16*>(v)[d * kPage + t % kPage]);
      } else {
        float c[4];
        codes_to_f32<CT>(v[(t % kPage / 16) * (D * 16) + d * 16 + t % 16], c);
        f = c[0] * vs;
      }
      if (attends && !(__builtin_fabsf(f) <= 65504.f)) add(x, f);
    }
  }
}

// The end of a piece whose wavefronts' partials are in LDS, O [W][rows][D + 4]
// at s_o and (m, l) [W][rows] at s_ml: every thread folds 4 features of a row
// over the wavefronts, in their order.  A whole (sequence, KV head) is then
// finished.  Any other leaves its part in the workspace, then an arrival flag
// (the call's ticket), and reads the flags of all parts: of two workgroups the
// one whose flag was stored later sees the other's, so at least one sees them
// all; those that do join the parts (to the same bits) and clear the flags,
// so that a replayed call (the same ticket) starts with none.  One launch: a
// second kernel for it costs a decode step 4 us.
template <int D, int W>
__device__ __forceinline__ void finish(const TreeArgs& a, const Walk& walk, const Piece& pc, const Seq& sq, int range, int rb,
                                       int rows, const float* s_o, const float* s_ml) {
  constexpr int ROW = D + 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
  const int row0 = rb * a.block_rows;
  // The host keeps the workspace below 2^31 bytes here.
  const Rsrc ws = __builtin_amdgcn_make_buffer_rsrc(a.ws, 0, 0x7ffffff0, 0x00020000);
  const uint32_t ml0 = static_cast<uint32_t>(partials(a) * D * 4);
  for (int u = threadIdx.x; u < rows * (D / 4); u += W * 64) {
    const int r = u / (D / 4), d = 4 * (u % (D / 4));
    float M = -INFINITY, L = 0.f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < W; ++w) M = fmaxf(M, s_ml[(w * rows + r) * 2]);
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float mw = s_ml[(w * rows + r) * 2], lw = s_ml[(w * rows + r) * 2 + 1];
      const float f = mw == -INFINITY ? 0.f : exp2_of(mw - M);
      L += mw == -INFINITY ? lw : lw * f;  // l without a reference is 0, or NaN
      if (mw != -INFINITY) acc += *reinterpret_cast<const f32x4*>(s_o + (w * rows + r) * ROW + d) * f;
    }
    if (pc.whole) {
      const int i = static_cast<int>(fdiv(row0 + r, a.by_g));
      store_row4<D>(a, walk.b, i, pc.kvh * a.g + row0 + r - i * a.g, d, acc, M, L);
    } else {
      const uint32_t part = static_cast<uint32_t>(partial_of(a, range, rb, pc.slot, r));
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, acc), ws, (part * D + d) * 4, 0, kAuxDevice);
      if (d == 0) {
        typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
        __builtin_amdgcn_raw_buffer_store_b64(u32x2{__builtin_bit_cast(uint32_t, M), __builtin_bit_cast(uint32_t, L)}, ws,
                                              ml0 + part * 8, 0, kAuxDevice);
      }
    }
  }
  if (pc.whole) return;
  __shared__ int s_merge;
  int r0, r1;
  walk.parts_of(a, pc.kvh, r0, r1);
  const uint32_t fl0 = ml0 + static_cast<uint32_t>(partials(a)) * 8;
  auto flag_of = [&](int r) { return fl0 + ((r * a.row_blocks + rb) * 2 + (r == r0 ? 1 : 0)) * 4; };
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();  // every part of the row is stored
  if (wave == 0) {
    if (lane == 0) __builtin_amdgcn_raw_buffer_store_b32(a.ticket, ws, flag_of(range), 0, kAuxDevice);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    bool seen = true;
    for (int r = r0 + lane; r <= r1; r += 64)
      seen = seen && __builtin_amdgcn_raw_buffer_load_b32(ws, flag_of(r), 0, kAuxDevice) == a.ticket;
    const bool all = __all(seen);
    if (lane == 0) s_merge = all ? 1 : 0;
  }
  __syncthreads();
  if (!s_merge) return;
  for (int u = threadIdx.x; u < rows * (D / 4); u += W * 64) {
    const int r = u / (D / 4), d = 4 * (u % (D / 4)), i = static_cast<int>(fdiv(row0 + r, a.by_g));
    float M = -INFINITY, L = 0.f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    if (i < sq.n)
      merge_parts(r0, r1, M, L, acc, [&](int p, float& m, float& l, f32x4& x) {
        typedef float f32x2 __attribute__((ext_vector_type(2)));
        const uint32_t part = static_cast<uint32_t>(partial_of(a, p, rb, p == r0 ? 1 : 0, r));
        const f32x2 ml = __builtin_bit_cast(f32x2, __builtin_amdgcn_raw_buffer_load_b64(ws, ml0 + part * 8, 0, kAuxDevice));
        m = ml[0], l = ml[1];
        x = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(ws, (part * D + d) * 4, 0, kAuxDevice));
      });
    store_row4<D>(a, walk.b, i, pc.kvh * a.g + row0 + r - i * a.g, d, acc, M, L);
  }
  for (int r = r0 + static_cast<int>(threadIdx.x); r <= r1; r += W * 64)
    __builtin_amdgcn_raw_buffer_store_b32(0u, ws, flag_of(r), 0, kAuxDevice);
}

// 17 to 64 rows to a KV head.  W wavefronts share a piece of a (sequence, KV
// head, tile of 32 rows): each takes steps of 32 tokens of its own, and they
// join in LDS at its end.  K of the next step is loaded as soon as the scores
// have used this one's, V as soon as O has.
// 16 sequences x 4096 tokens, 32 / 8 heads: 8 drafted tokens (32 rows) 36 us over
// e4m3 of head_dim 128 (3.7 TB/s), 31 over fp16 of 64 (4.4 TB/s); 16 (two tiles,
// which read the pages twice, the second time from L2) 34 us over e4m3, 501
// TFLOP/s.  Bound by instruction issue over 8-bit pages (a tile's conversions
// cost as much as its products) and by the one step in flight over fp16 ones.
template <int CT, int D, int W>
__global__ __launch_bounds__(W * 64, 2) void tree_rows_kernel(TreeArgs a) {
  constexpr int STEP = 32, PER_PAGE = kPage / STEP;
  constexpr int KB = CT == kF16 ? 2 : 1;  // bytes of an element
  constexpr int DS = D / 32;
  constexpr int ROW = D + 4;  // floats of a row in LDS
  __shared__ __align__(16) float s_mem[W * kTile * (ROW + 2)];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
  const int col = lane & 31, half = lane >> 5;
  int range, tile;
  place_of(a, range, tile);
  Walk walk;
  if (range >= a.ranges || !walk.start(a, lane, range)) return;
  for (; walk.u < walk.end;) {
    const Piece pc = piece_of(a, walk);
    const int b = walk.b, kvh = pc.kvh;
    const Seq sq = walk.seq;
    const int total = sq.ctx + (a.draft_keys ? sq.n : 0);
    // The wavefronts take equal shares of the piece's steps; rows of no drafted token none.
    const int c0 = pc.page0 * PER_PAGE, c1 = tile * kTile < sq.n * a.g ? min(pc.page1 * PER_PAGE, (total + STEP - 1) / STEP) : c0;
    const int s0 = c0 + (c1 - c0) * wave / W, s1 = c0 + (c1 - c0) * (wave + 1) / W;
    const Row row = row_of(a, sq, b, kvh, tile * kTile + col);
    f16x8 qf[DS][2];
    Pages pages(a, b, kvh, lane, s0 / PER_PAGE);
    bool odd = false;

    f32x16 o[DS];
#pragma unroll
    for (int dt = 0; dt < DS; ++dt)
#pragma unroll
      for (int x = 0; x < 16; ++x) o[dt][x] = 0.f;
    float m = -INFINITY, l = 0.f;

    // Lane offsets within a page, bytes.
    const int tok = token_of(col);
    const int k_off = CT == kF16 ? (tok * 64 + 16 * half) * 2 : half * (kPage * 16) + tok * 16;
    const int v_off = CT == kF16 ? (col * kPage + 16 * half) * 2 : half * (D * 16) + col * 16;

    int64_t head = 0;  // physical page * Hkv + KV head, of the step being loaded
    auto locate = [&](int st) { head = pages.head(st / PER_PAGE); };
    Raw<CT, D> kr, vr;
    float scale = 0.f;  // 8-bit: of the step's token `col`, K's in the lower lanes, V's in the upper
    auto load_k = [&](int st) {
      const int hp = st % PER_PAGE;
      const Rsrc r = page_rsrc(a.k, head, kPage * D * KB);
#pragma unroll
      for (int s = 0; s < DS; ++s)
#pragma unroll
        for (int e = 0; e < KB; ++e)
          kr.x[s][e] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
              r, k_off,
              CT == kF16 ? hp * (STEP * 128) + (s / 2) * (kPage * 128) + (s % 2) * 64 + 16 * e
                         : hp * (STEP * 16) + 2 * s * (kPage * 16), 0));
      if constexpr (CT != kF16)
        scale = (half ? a.vs : a.ks)[head * kPage + hp * STEP + col];
    };
    auto load_v = [&](int st) {
      const int hp = st % PER_PAGE;
      const Rsrc r = page_rsrc(a.v, head, kPage * D * KB);
#pragma unroll
      for (int dt = 0; dt < DS; ++dt)
#pragma unroll
        for (int e = 0; e < KB; ++e)
          vr.x[dt][e] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
              r, v_off, CT == kF16 ? hp * (STEP * 2) + dt * (32 * kPage * 2) + 16 * e : 2 * hp * (D * 16) + dt * (32 * 16), 0));
    };
    // 8-bit: this wavefront's step: score factors, V's scales' logarithms and inverses.
    float* s_sc = s_mem + wave * 3 * STEP;

    // MORE: another step follows (as in the few kernel).
    auto step = [&](int st, auto more_tag, auto edge_tag) {
      constexpr bool MORE = decltype(more_tag)::value;
      constexpr bool EDGE = decltype(edge_tag)::value;  // some tokens are drafted or do not exist
      const int tok0 = st * STEP + 16 * half;           // this lane's 16 tokens
      uint32_t seen = 0;                                // those that its row attends
      if constexpr (EDGE) seen = row.attends16(a, sq, tok0, total, [](int x) { return x; });
      uint32_t odd_scale = 0, inf_scale = 0;  // of this lane's 16 tokens, those whose V has no finite scale
      if constexpr (CT != kF16) {
        __builtin_amdgcn_wave_barrier();
        const bool finite = __builtin_fabsf(scale) <= 0x1.fffffep127f;
        odd_scale = static_cast<uint32_t>(__builtin_amdgcn_ballot_w64(half && !finite) >> (32 + 16 * half)) & 0xffffu;
        inf_scale = static_cast<uint32_t>(__builtin_amdgcn_ballot_w64(half && scale == INFINITY) >> (32 + 16 * half)) & 0xffffu;
        bool none = scale < 0x1p-60f;  // codes of no weight
        if (__any(half && scale == 1.f && (!EDGE || st * STEP + col < total))) {  // rows of zeros?
          u32x4 w = vr.x[0][0];
#pragma unroll
          for (int dt = 1; dt < DS; ++dt) w |= vr.x[dt][0];
          u32x4 w0, w1;  // tokens 0 .. 15 and 16 .. 31 of the step
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t x = or16(w[i]);
            const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
            const auto h = __builtin_amdgcn_permlane32_swap(r[0] | r[1], r[0] | r[1], false, false);
            w0[i] = h[0], w1[i] = h[1];
          }
          none = none || (scale == 1.f && zero_row<CT>(col < 16 ? w0 : w1, col % 16));
        }
        const float vc = !finite ? 1.f : none ? 0x1p-60f : scale;
        s_sc[lane] = half ? __builtin_amdgcn_logf(vc) : scale * a.scale_log2;
        if (half) s_sc[2 * STEP + col] = __builtin_amdgcn_rcpf(vc);
        __builtin_amdgcn_wave_barrier();
      }
      f32x16 sc;
#pragma unroll
      for (int x = 0; x < 16; ++x) sc[x] = 0.f;
#pragma unroll
      for (int s = 0; s < DS; ++s)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(operand<CT>(kr.x[s], e), qf[s][e], sc, 0, 0, 0);
      if constexpr (MORE) {
        if ((st + 1) % PER_PAGE == 0) locate(st + 1);
        load_k(st + 1);
      }
      float mx = -INFINITY;
#pragma unroll
      for (int x4 = 0; x4 < 4; ++x4) {
        f32x4 f, lv;
        if constexpr (CT != kF16) {
          f = *reinterpret_cast<const f32x4*>(s_sc + 16 * half + 4 * x4);
          lv = *reinterpret_cast<const f32x4*>(s_sc + STEP + 16 * half + 4 * x4);
        }
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const int x = 4 * x4 + y;
          float v = CT == kF16 ? sc[x] * a.scale_log2 : __builtin_fmaf(sc[x], f[y], lv[y]);
          if constexpr (EDGE) v = (seen >> x) & 1 ? v : -INFINITY;
          sc[x] = v;
          mx = fmaxf(mx, v);
        }
      }
      mx = xor32_max(mx);
      if (__any(mx > m + kAbove)) {
        const float mn = fmaxf(m, mx - kBelow);
        const float alpha = m == -INFINITY ? 0.f : exp2_of(m - mn);
        m = mn;
        l *= alpha;
#pragma unroll
        for (int dt = 0; dt < DS; ++dt)
#pragma unroll
          for (int x = 0; x < 16; ++x) o[dt][x] *= alpha;
      }
      const float mu = m == -INFINITY ? 0.f : m;  // a row that has attended nothing yet: weights 0
      f16x8 p[2];
#pragma unroll
      for (int x4 = 0; x4 < 4; ++x4) {
        f32x4 r;
        if constexpr (CT != kF16) r = *reinterpret_cast<const f32x4*>(s_sc + 2 * STEP + 16 * half + 4 * x4);
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const int x = 4 * x4 + y;
          const float w = exp2_of(sc[x] - mu);
          if constexpr (CT == kF16)
            l += w;
          else
            l = __builtin_fmaf(w, EDGE && !((seen >> x) & 1) ? 0.f : r[y], l);
          p[x / 8][x % 8] = static_cast<_Float16>(w);
        }
      }
      if (CT != kF16 && __any(odd_scale != 0)) {  // weights that leave the codes as the scale does; lse does not know V
#pragma unroll
        for (int x = 0; x < 16; ++x)
          if ((odd_scale >> x) & 1 && (!EDGE || (seen >> x) & 1))
            p[x / 8][x % 8] = static_cast<_Float16>((inf_scale >> x) & 1 ? INFINITY : NAN);
      }
      if constexpr (EDGE) {
        // Numbers of tokens that do not exist are any bits; those of drafted
        // tokens that a row does not attend may be infinite or NaN.  Neither
        // may meet a weight of 0: rows that do attend them take them below.
#pragma unroll
        for (int dt = 0; dt < DS; ++dt) {
          drop_tokens<CT>(vr.x[dt], total - tok0);
#pragma unroll
          for (int e = 0; e < Raw<CT, D>::W; ++e)
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              uint32_t y = vr.x[dt][e][w];
              odd = drop_odd<CT>(y) || odd;
              vr.x[dt][e][w] = y;
            }
        }
      }
#pragma unroll
      for (int dt = 0; dt < DS; ++dt)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(operand<CT>(vr.x[dt], e), p[e], o[dt], 0, 0, 0);
      if constexpr (MORE) load_v(st + 1);
    };

    // Every row attends every token of a step below ctx (rows without a drafted
    // token drop theirs at the end), so only the last steps test tokens.
    const int whole = min(s1, sq.ctx / STEP);
    std::true_type yes;
    std::false_type no;
    auto wait_q = [&] {  // behind the first step's loads; waits here, not in every step
      load_q<DS>(a, b, row, half, qf);
#pragma unroll
      for (int s = 0; s < DS; ++s)
#pragma unroll
        for (int e = 0; e < 2; ++e) asm volatile("" : "+v"(qf[s][e]));
    };
    int st = s0;
    if (st < whole) {
      locate(st);
      load_k(st);
      load_v(st);
      wait_q();
      for (; st < whole - 1; ++st) step(st, yes, no);
      step(st, no, no);
      ++st;
    } else if (st < s1) {
      wait_q();
    }
    for (; st < s1; ++st) {  // the sequence's last steps
      if (st == s0 || st % PER_PAGE == 0) locate(st);
      load_k(st);
      load_v(st);
      step(st, no, yes);
    }
    if (CT != SPYRE_CODES_INT8 && __any(odd))
      add_odd<CT, D, DS * 16>(
          a, sq, b, kvh, row, lane, max(s0, whole) * STEP, min(s1 * STEP, total), -1,
          [](int x, int ln) { return 32 * (x / 16) + 8 * (x % 16 / 4) + 4 * (ln >> 5) + x % 4; },
          [&](int x, float f) { o[x / 16][x % 16] += f; });
    l = xor32_sum(l);
    if (!row.live) m = -INFINITY, l = 0.f;
    if ((pages.poisoned || sq.bad) && row.live) l = NAN;

    // O, m and l of the rows that exist.
    const int rows = min(kTile, a.rows - static_cast<int>(tile) * kTile);
    float* s_o = s_mem;                          // [W][rows][ROW]
    float* s_ml = s_mem + W * rows * ROW;        // [W][rows][2]
    __syncthreads();
    if (col < rows) {
#pragma unroll
      for (int dt = 0; dt < DS; ++dt)
#pragma unroll
        for (int x4 = 0; x4 < 4; ++x4)
          *reinterpret_cast<f32x4*>(s_o + (wave * rows + col) * ROW + 32 * dt + 8 * x4 + 4 * half) =
              f32x4{o[dt][4 * x4], o[dt][4 * x4 + 1], o[dt][4 * x4 + 2], o[dt][4 * x4 + 3]};
      if (half == 0) {
        s_ml[(wave * rows + col) * 2] = m;
        s_ml[(wave * rows + col) * 2 + 1] = l;
      }
    }
    __syncthreads();
    finish<D, W>(a, walk, pc, sq, range, tile, rows, s_o, s_ml);
    advance(a, walk, pc);
    __syncthreads();  // LDS is read before the next piece writes it
  }
}

// ------------------------------------------------------------- few rows --
//
// Up to 16 rows to a KV head (a decode step): MFMA 16x16x32, whose 16 columns
// cost half of what 32 would.  W wavefronts share a piece, each whole pages of
// it:
//   S^T[tok, row] = K[tok, :] Q^T[:, row]      4 x D/32 products of 16 tokens
//   O^T[d, row] += V^T[d, tok] P^T[tok, row]   D/16 x 2
// The same free orders as above, taken so that every load instruction covers
// whole runs of memory.  Lane group G = lane / 16; token tile j's row m is
//   fp16   token 32 (j / 2) + 8 (m / 4) + 4 (j % 2) + m % 4, features 64 s +
//          8 G + 32 e of products 2 s + e: group G ends with the scores of the
//          two runs of 8 tokens of V's 16-byte loads; 64-byte runs of a row.
//   8-bit  token 16 j + m, features 64 s + 16 G + 8 e: 256-byte runs of K's
//          units.  Group G then holds the scores of the tokens 16 j + 4 G + i;
//          its V load is the tokens 16 G .. + 15, so the 4 x 4 words (of 4
//          tokens) of the four groups change places in registers first.
// Bound by memory: K of the next page is loaded as soon as the scores have used
// this one's, V as soon as O has; head_dim 64 has the registers for two pages in
// flight.  A decode step over e4m3, 32 / 8 heads of 128: 32 x 4096 tokens 45 us
// (6.1 TB/s), 64 x 8192 165 us (6.7 TB/s), 64 x 128 to 16384 185 us; one
// sequence of 700 tokens 10.6 us, which is the chain of its loads (lengths, table,
// page) and the join.
template <int CT, int D, int W>
__global__ __launch_bounds__(W * 64, 2) void tree_few_kernel(TreeArgs a) {
  constexpr int KB = CT == kF16 ? 2 : 1, KW = KB;  // bytes of an element; 16-byte words of 16 of them
  constexpr int DQ = D / 64, DV = D / 16;
  constexpr int SETS = D == 128 ? 1 : 2;
  constexpr int ROW = D + 4;
  __shared__ __align__(16) float s_mem[W * 16 * (ROW + 2)];
  static_assert(3 * kPage <= 16 * (ROW + 2), "a wavefront's scales fit its share");
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
  const int col = lane & 15, grp = lane >> 4;
  const int range = blockIdx.x;
  Walk walk;
  if (!walk.start(a, lane, range)) return;
  // Lane offsets within a page, bytes.
  const int k_off = CT == kF16 ? (8 * (col >> 2) + (col & 3)) * 128 + grp * 16 : grp * (kPage * 16) + col * 16;
  const int v_off = CT == kF16 ? col * (kPage * 2) + grp * 16 : grp * (D * 16) + col * 16;
  // This lane's 16 tokens of a page, in the order of its scores: tok_of(0) + offset(x).
  auto offset = [](int x) { return CT == kF16 ? 32 * (x / 8) + x % 8 : 16 * (x / 4) + x % 4; };
  const int tok_of0 = CT == kF16 ? 8 * grp : 4 * grp;
  float* s_sc = s_mem + wave * 3 * kPage;  // 8-bit: score factors, V's scales' logarithms and inverses
  for (; walk.u < walk.end;) {
    const Piece pc = piece_of(a, walk);
    const int b = walk.b, kvh = pc.kvh;
    const Seq sq = walk.seq;
    const int total = sq.ctx + (a.draft_keys ? sq.n : 0);
    const int c1 = sq.n > 0 ? min(pc.page1, sq.pages) : pc.page0, nc = c1 - pc.page0;
    const int p0 = pc.page0 + nc * wave / W, p1 = pc.page0 + nc * (wave + 1) / W;
    const Row row = row_of(a, sq, b, kvh, col);
    f16x8 qf[DQ][2];
    auto load_q = [&] {  // behind the first page's loads; waits for all of them
      const _Float16* qp = a.q + b * a.q_sb + (row.live ? row.i * a.q_st + row.head * a.q_sh : 0) + (CT == kF16 ? 8 : 16) * grp;
#pragma unroll
      for (int s = 0; s < DQ; ++s)
#pragma unroll
        for (int e = 0; e < 2; ++e) qf[s][e] = *reinterpret_cast<const f16x8*>(qp + 64 * s + (CT == kF16 ? 32 : 8) * e);
#pragma unroll
      for (int s = 0; s < DQ; ++s)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          if (!row.live) qf[s][e] = f16x8{};
          asm volatile("" : "+v"(qf[s][e]));
        }
    };
    Pages pages(a, b, kvh, lane, p0);
    bool odd = false;
    f32x4 o[DV];
#pragma unroll
    for (int dt = 0; dt < DV; ++dt) o[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;
    // The raw operands of a page, in sets that take turns.
    struct Operands {
      u32x4 k[4][DQ][KW], v[DV][KW];
      float ks, vs;  // 8-bit: scales of the page's token `lane`
    };
    Operands set[SETS];
    auto load_k = [&](Operands& x, int64_t head) {
      const Rsrc r = page_rsrc(a.k, head, kPage * D * KB);
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int s = 0; s < DQ; ++s)
#pragma unroll
          for (int e = 0; e < KW; ++e)
            x.k[j][s][e] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                r, k_off,
                CT == kF16 ? s * (kPage * 128) + (32 * (j / 2) + 4 * (j % 2)) * 128 + 64 * e : 4 * s * (kPage * 16) + 16 * j * 16,
                kAuxOnce));
      if constexpr (CT != kF16) {
        x.ks = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(page_rsrc(a.ks, head, kPage * 4), 4 * lane, 0, kAuxOnce));
        x.vs = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(page_rsrc(a.vs, head, kPage * 4), 4 * lane, 0, kAuxOnce));
      }
    };
    auto load_v = [&](Operands& x, int64_t head) {
      const Rsrc r = page_rsrc(a.v, head, kPage * D * KB);
#pragma unroll
      for (int dt = 0; dt < DV; ++dt)
#pragma unroll
        for (int e = 0; e < KW; ++e)
          x.v[dt][e] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
              r, v_off, CT == kF16 ? dt * (16 * kPage * 2) + 64 * e : dt * (16 * 16), kAuxOnce));
    };
    // MORE: page p + SETS follows in the same registers.  (A test of it at run
    // time would leave the compiler paths on which K is loaded and V is not, and
    // every page would wait for its V before its first product.)
    auto step = [&](Operands& x, int p, auto more_tag, auto edge_tag) {
      constexpr bool MORE = decltype(more_tag)::value;
      constexpr bool EDGE = decltype(edge_tag)::value;   // some tokens are drafted or do not exist
      const int tok0 = p * kPage + tok_of0;
      uint32_t seen = 0, odd_scale = 0, inf_scale = 0;   // as in the rows kernel
      if constexpr (EDGE) seen = row.attends16(a, sq, tok0, total, offset);
      if constexpr (CT != kF16) {
        __builtin_amdgcn_wave_barrier();
        const bool finite = __builtin_fabsf(x.vs) <= 0x1.fffffep127f;
        const uint64_t not_finite = __builtin_amdgcn_ballot_w64(!finite), infinite = __builtin_amdgcn_ballot_w64(x.vs == INFINITY);
        if (not_finite) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            odd_scale |= (static_cast<uint32_t>(not_finite >> (16 * j + 4 * grp)) & 0xfu) << (4 * j);
            inf_scale |= (static_cast<uint32_t>(infinite >> (16 * j + 4 * grp)) & 0xfu) << (4 * j);
          }
        }
        bool none = x.vs < 0x1p-60f;  // as in the rows kernel
        if (__any(x.vs == 1.f && (!EDGE || p * kPage + lane < total))) {
          u32x4 w = x.v[0][0];
#pragma unroll
          for (int dt = 1; dt < DV; ++dt) w |= x.v[dt][0];
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = or16(w[i]);
          none = none || (x.vs == 1.f && zero_row<CT>(w, col));
        }
        const float vc = !finite ? 1.f : none ? 0x1p-60f : x.vs;
        s_sc[lane] = x.ks * a.scale_log2;
        s_sc[kPage + lane] = __builtin_amdgcn_logf(vc);
        s_sc[2 * kPage + lane] = __builtin_amdgcn_rcpf(vc);
        __builtin_amdgcn_wave_barrier();
      }
      f32x4 sc[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        sc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < DQ; ++s)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            sc[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(operand<CT>(x.k[j][s], e), qf[s][e], sc[j], 0, 0, 0);
      }
      int64_t head = 0;
      if constexpr (MORE) {
        head = pages.head(p + SETS);
        load_k(x, head);
      }
      float mx = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        f32x4 f, lv;
        if constexpr (CT != kF16) {
          f = *reinterpret_cast<const f32x4*>(s_sc + 16 * j + 4 * grp);
          lv = *reinterpret_cast<const f32x4*>(s_sc + kPage + 16 * j + 4 * grp);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float v = CT == kF16 ? sc[j][i] * a.scale_log2 : __builtin_fmaf(sc[j][i], f[i], lv[i]);
          if constexpr (EDGE) v = (seen >> (4 * j + i)) & 1 ? v : -INFINITY;
          sc[j][i] = v;
          mx = fmaxf(mx, v);
        }
      }
      mx = xor32_max(mx);
      mx = xor16_max(mx);
      if (__any(mx > m + kAbove)) {
        const float mn = fmaxf(m, mx - kBelow);
        const float alpha = m == -INFINITY ? 0.f : exp2_of(m - mn);
        m = mn;
        l *= alpha;
#pragma unroll
        for (int dt = 0; dt < DV; ++dt) o[dt] *= alpha;
      }
      const float mu = m == -INFINITY ? 0.f : m;  // a row that has attended nothing yet: weights 0
      f16x8 pw[2];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        f32x4 r;
        if constexpr (CT != kF16) r = *reinterpret_cast<const f32x4*>(s_sc + 2 * kPage + 16 * j + 4 * grp);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float w = exp2_of(sc[j][i] - mu);
          if constexpr (CT == kF16)
            l += w;
          else
            l = __builtin_fmaf(w, EDGE && !((seen >> (4 * j + i)) & 1) ? 0.f : r[i], l);
          pw[j / 2][4 * (j % 2) + i] = static_cast<_Float16>(w);
        }
      }
      if (CT != kF16 && __any(odd_scale != 0)) {
#pragma unroll
        for (int x = 0; x < 16; ++x)
          if ((odd_scale >> x) & 1 && (!EDGE || (seen >> x) & 1))
            pw[x / 8][x % 8] = static_cast<_Float16>((inf_scale >> x) & 1 ? INFINITY : NAN);
      }
      if constexpr (EDGE) {
#pragma unroll
        for (int dt = 0; dt < DV; ++dt) {
          if constexpr (CT == kF16) {
            u32x4 lo[1] = {x.v[dt][0]}, hi[1] = {x.v[dt][1]};  // 8 tokens each
            drop_tokens<CT>(lo, total - tok0);
            drop_tokens<CT>(hi, total - tok0 - 32);
            x.v[dt][0] = lo[0], x.v[dt][1] = hi[0];
          } else {
            drop_tokens<CT>(x.v[dt], total - p * kPage - 16 * grp);
          }
#pragma unroll
          for (int e = 0; e < KW; ++e)
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              uint32_t y = x.v[dt][e][w];
              odd = drop_odd<CT>(y) || odd;
              x.v[dt][e][w] = y;
            }
        }
      }
#pragma unroll
      for (int dt = 0; dt < DV; ++dt) {
        if constexpr (CT != kF16) {
          uint32_t w[4] = {x.v[dt][0][0], x.v[dt][0][1], x.v[dt][0][2], x.v[dt][0][3]};
          transpose4x4_groups(w);  // word j: tokens 16 j + 4 grp ..
          x.v[dt][0] = u32x4{w[0], w[1], w[2], w[3]};
        }
#pragma unroll
        for (int e = 0; e < 2; ++e)
          o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(operand<CT>(x.v[dt], e), pw[e], o[dt], 0, 0, 0);
      }
      if constexpr (MORE) load_v(x, head);
    };
    const int whole = min(p1, sq.ctx / kPage);
    std::true_type yes;
    std::false_type no;
    int p = p0;
    auto load = [&](Operands& x, int page) {
      const int64_t head = pages.head(page);
      load_k(x, head);
      load_v(x, head);
    };
    if (p < whole) {
      load(set[0], p);
      if constexpr (SETS == 2) {
        if (p + 1 < whole) load(set[1], p + 1);
      }
      load_q();
      if constexpr (SETS == 2) {
        for (; p + 3 < whole; p += 2) {
          step(set[0], p, yes, no);
          step(set[1], p + 1, yes, no);
        }
        if (p + 2 < whole) {
          step(set[0], p, yes, no);
          step(set[1], p + 1, no, no);
          step(set[0], p + 2, no, no);
        } else {
          step(set[0], p, no, no);
          if (p + 1 < whole) step(set[1], p + 1, no, no);
        }
        p = whole;
      } else {
        for (; p < whole - 1; ++p) step(set[0], p, yes, no);
        step(set[0], p, no, no);
        ++p;
      }
    } else if (p < p1) {
      load_q();
    }
    for (; p < p1; ++p) {  // the sequence's last pages
      load(set[0], p);
      step(set[0], p, no, yes);
    }
    if (CT != SPYRE_CODES_INT8 && __any(odd))
      add_odd<CT, D, DV * 4>(
          a, sq, b, kvh, row, lane, max(p0, whole) * kPage, min(p1 * kPage, total), -1,
          [](int x, int ln) { return 16 * (x / 4) + 4 * (ln >> 4) + x % 4; }, [&](int x, float f) { o[x / 4][x % 4] += f; });
    l = xor16_sum(xor32_sum(l));
    if (!row.live) m = -INFINITY, l = 0.f;
    if ((pages.poisoned || sq.bad) && row.live) l = NAN;
    const int rows = a.rows;
    float* s_o = s_mem;
    float* s_ml = s_mem + W * rows * ROW;
    __syncthreads();
    if (col < rows) {
#pragma unroll
      for (int dt = 0; dt < DV; ++dt) *reinterpret_cast<f32x4*>(s_o + (wave * rows + col) * ROW + 16 * dt + 4 * grp) = o[dt];
      if (grp == 0) {
        s_ml[(wave * rows + col) * 2] = m;
        s_ml[(wave * rows + col) * 2 + 1] = l;
      }
    }
    __syncthreads();
    finish<D, W>(a, walk, pc, sq, range, 0, rows, s_o, s_ml);
    advance(a, walk, pc);
    __syncthreads();  // LDS is read before the next piece writes it
  }
}

// ---------------------------------------------------------- wide drafts --
//
// 8 wavefronts share every page through LDS: RT = 8 row tiles of 32 rows, each
// wavefront's own, or RT = 4, where a wavefront takes one half of each page's
// tokens and the two of a tile join at the end.  K [D/64, 64 tok, 64] lies in
// KS slots and V [D, 64 tok] in VS, as fp16: fp16 pages are on their way two
// pages ahead, 8-bit ones, converted once on the way in, one.  A 128-byte row is 8 units of 16 bytes; unit u lies at
// u ^ swz(row), so that the 16 lanes that a read serves at once, and a
// conversion's 16 stores, meet 16 different bank groups.
//
// The matrix products of one 32-token half run beside the softmax of another:
// while the weights of half i are formed, the scores of half i + 1 are
// multiplied, and while those weights meet V, the scores' maximum is taken.  K
// therefore runs one page ahead of V.
//
// RT 8: 16 sequences x 8192 tokens, 64 tokens of 64 / 8 heads of 128 (512 rows to
// a KV head): 314 to 320 us over fp16, 865 to 880 TFLOP/s where a large matrix
// product of the same type reaches 1200; 328 us over e4m3.  Bound by the products and the
// softmax's instructions beside them.
// RT 4: 25 tokens of 32 / 8 heads x 4096: 67 + 8 us of joining over e4m3, 77 + 8
// over fp16; 16 tokens x 8192 over fp16 131 us, 4.1 TB/s.  An e4m3 page takes 1.4
// us, 0.9 without its loads and conversions: one step a wavefront between two
// barriers is too little to hide either.  More 8-bit pages in flight, as codes
// in LDS or in a second set of registers, gained nothing (1.9 and 1.3 us).
__device__ __forceinline__ int swz_k(int row) { return ((row >> 1) & 3) | ((((row >> 3) ^ (row >> 4)) & 1) << 2); }
__device__ __forceinline__ int swz_v(int row) { return (row >> 1) & 7; }

constexpr int kWideWaves = 8;

template <int CT, int D, int RT>
__global__ __launch_bounds__(kWideWaves * 64, 2) void tree_wide_kernel(TreeArgs a) {
  constexpr int W = kWideWaves, DS = D / 32;
  constexpr int TILE = kPage * D * 2;  // bytes of a K or a V tile
  constexpr int KU = kPage * D / 16;   // 8-bit: units of a K or a V page, one for each thread (D 64: K's and V's share them)
  static_assert(RT == W || 2 * RT == W, "a wavefront takes a page or a half of it");
  constexpr int KS = CT == kF16 ? 4 : 3, VS = KS - 1;  // K and V slots
  __shared__ __align__(16) char s_kv[(KS + VS) * TILE];
  __shared__ __align__(16) float s_sc[3][3][kPage];  // 8-bit: score factors, V's scales' logarithms and inverses
  __shared__ __align__(16) float s_vs[3][kPage];     // V's scales where they are not finite, else 0
  __shared__ int s_odd[3];                           // whether any is not
  __shared__ float s_ml[RT == W ? 1 : RT * 64 * 2];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
  const int col = lane & 31, half = lane >> 5;
  const int part = RT == W ? 0 : wave & 1;  // RT 4: this wavefront's half of a page
  int range, rb;
  place_of(a, range, rb);
  Walk walk;
  if (range >= a.ranges || !walk.start(a, lane, range)) return;

  // fp16 pages go straight into LDS: load i of a tile fills its bytes 1024 i
  // .., lane by lane, so each lane fetches the unit that belongs at its place.
  const int l8 = lane / 8;
  const int k_src = 1024 * wave + 128 * l8 + (((lane % 8) ^ swz_k(8 * wave + l8)) * 16);
  const int v_src = 1024 * wave + 128 * l8 + (((lane % 8) ^ swz_v(8 * wave + l8)) * 16);
  // Operand addresses in a tile: unit u of a row is (bits of the unroll) ^
  // (bits of the lane).
  const int tok = token_of(col);
  const int k_x = (2 * half) ^ swz_k(tok), v_x = (2 * half) ^ swz_v(col);
  int k_at[2][2];
#pragma unroll
  for (int y = 0; y < 2; ++y)
#pragma unroll
    for (int e = 0; e < 2; ++e) k_at[y][e] = tok * 128 + ((k_x ^ (4 * y + e)) * 16);
  const float c = __builtin_fabsf(a.scale_log2);  // its sign is in q

  for (; walk.u < walk.end;) {
    const Piece pc = piece_of(a, walk);
    const int b = walk.b, kvh = pc.kvh;
    const Seq sq = walk.seq;
    const int total = sq.ctx + (a.draft_keys ? sq.n : 0);
    const int p0 = pc.page0, p1 = min(pc.page1, sq.pages);
    const int local = RT == W ? wave : wave >> 1, tile = rb * RT + local;
    const Row row = row_of(a, sq, b, kvh, tile * kTile + col);
    Pages pages(a, b, kvh, lane, p0);
    bool odd = false;
    const bool block_live = rb * RT * kTile < sq.n * a.g;  // some row of the workgroup is drafted
    const bool wave_live = tile * kTile < sq.n * a.g;
    f16x8 qf[DS][2];
    load_q<DS>(a, b, row, half, qf);
    if (a.scale_log2 < 0.f) {
#pragma unroll
      for (int s = 0; s < DS; ++s)
#pragma unroll
        for (int e = 0; e < 2; ++e) qf[s][e] = -qf[s][e];
    }
    f32x16 o[DS];
#pragma unroll
    for (int dt = 0; dt < DS; ++dt)
#pragma unroll
      for (int x = 0; x < 16; ++x) o[dt][x] = 0.f;
    float m = -INFINITY, l = 0.f;

    // A page's K or V into its slot: fp16 by loads into LDS; 8-bit by way of
    // registers (take, then put a step later).
    auto k_tile = [&](int s3) { return s_kv + s3 * TILE; };
    auto v_tile = [&](int s2) { return s_kv + (KS + s2) * TILE; };
    auto dma = [&](const uint8_t* cache, int64_t head, char* to, int src) {
      const Rsrc r = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(cache + head * TILE), 0, TILE, 0x00020000);
#pragma unroll
      for (int j = 0; j < TILE / 1024 / W; ++j)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)(to + 1024 * (wave + W * j)), 16,
                                                 src, 1024 * W * j, 0, 0);
    };
    // 8-bit: D 128: every thread a unit of K and one of V; D 64: the first
    // wavefronts K's, the others V's.  Scales: K's by wavefront 0, V's by 1.
    u32x4 k_raw, v_raw;
    float scale = 0.f;
    const bool has_k = wave * 64 < KU, has_v = D == 128 || wave * 64 >= KU;
    const int v_unit0 = D == 128 ? wave * 64 : wave * 64 - KU;
    auto take_k = [&](int64_t head) {
      if (has_k) k_raw = *reinterpret_cast<const u32x4*>(a.k + head * (TILE / 2) + (wave * 64 + lane) * 16);
      if (wave < 2) scale = (wave ? a.vs : a.ks)[head * kPage + lane];
    };
    auto take_v = [&](int64_t head) {
      if (has_v) v_raw = *reinterpret_cast<const u32x4*>(a.v + head * (TILE / 2) + (v_unit0 + lane) * 16);
    };
    auto put = [&](char* at, int u, int sw, const u32x4& w) {  // units u and u + 1 of a row
      *reinterpret_cast<f16x8*>(at + ((u ^ sw) * 16)) = codes_to_f16x8<CT>(w[0], w[1]);
      *reinterpret_cast<f16x8*>(at + (((u + 1) ^ sw) * 16)) = codes_to_f16x8<CT>(w[2], w[3]);
    };
    auto put_k = [&](int s3, int page, int64_t head) {  // those of `page`, which lies at `head`
      int ln = lane;
      asm volatile("" : "+v"(ln));  // its addresses are not worth registers of the products
      if (has_k) {
        const int un = wave * 64 / kPage;  // 16 features of token ln
        put(k_tile(s3) + (un / 4) * (kPage * 128) + ln * 128, 2 * (un % 4), swz_k(ln), k_raw);
      }
      if (wave == 0) s_sc[s3][0][ln] = scale * c;
      if (wave == 1) {
        const bool finite = __builtin_fabsf(scale) <= 0x1.fffffep127f;
        bool none = scale < 0x1p-60f;  // codes of no weight
        if (__any(scale == 1.f && page * kPage + ln < total)) {  // rows of zeros?
          const u32x4* v = reinterpret_cast<const u32x4*>(a.v + head * (TILE / 2)) + ln / 16 * D + ln % 16;
          u32x4 w = v[0];
#pragma unroll 1
          for (int f = 16; f < D; f += 16) w |= v[f];
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = or16(w[i]);
          none = none || (scale == 1.f && zero_row<CT>(w, ln % 16));
        }
        const float vc = !finite ? 1.f : none ? 0x1p-60f : scale;
        s_sc[s3][1][ln] = __builtin_amdgcn_logf(vc);
        s_sc[s3][2][ln] = __builtin_amdgcn_rcpf(vc);
        s_vs[s3][ln] = finite ? 0.f : scale;
        if (lane == 0) s_odd[s3] = 0;
        if (!finite) s_odd[s3] = 1;
      }
    };
    auto put_v = [&](int s2) {
      int ln = lane;
      asm volatile("" : "+v"(ln));
      if (has_v) {  // 16 tokens of a feature
        const int x = v_unit0 + ln, q4 = x / D, d = x % D;
        put(v_tile(s2) + d * 128, 2 * q4, swz_v(d), v_raw);
      }
    };
    // 8-bit V whose scales are not finite: their numbers as the scales leave them.
    auto patch_v = [&](int s2, int s3) {
      for (int i = threadIdx.x; i < kPage * D; i += W * 64) {
        const int d = i / kPage, t = i % kPage;
        const float vs = s_vs[s3][t];
        if (!(vs == 0.f)) {
          _Float16* at = reinterpret_cast<_Float16*>(v_tile(s2) + d * 128 + (((t / 8) ^ swz_v(d)) * 16)) + t % 8;
          *at = static_cast<_Float16>(static_cast<float>(*at) * vs);
        }
      }
    };

    // The scores of half t of a K tile.
    auto scores = [&](f32x16& s, const char* kt, int t) {
#pragma unroll
      for (int x = 0; x < 16; ++x) s[x] = 0.f;
#pragma unroll
      for (int i = 0; i < DS; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const f16x8 k = *reinterpret_cast<const f16x8*>(kt + t * (32 * 128) + k_at[i % 2][e] + (i / 2) * (kPage * 128));
          s = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, qf[i][e], s, 0, 0, 0);
        }
    };
    // 8-bit: scores scaled, V's scales added.  The largest, in log2 units.
    auto largest = [&](f32x16& s, int s3, int t) {
      float mx = -INFINITY;
#pragma unroll
      for (int x4 = 0; x4 < 4; ++x4) {
        f32x4 f, lv;
        if constexpr (CT != kF16) {
          f = *reinterpret_cast<const f32x4*>(&s_sc[s3][0][32 * t + 16 * half + 4 * x4]);
          lv = *reinterpret_cast<const f32x4*>(&s_sc[s3][1][32 * t + 16 * half + 4 * x4]);
        }
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          if constexpr (CT != kF16) s[4 * x4 + y] = __builtin_fmaf(s[4 * x4 + y], f[y], lv[y]);
          mx = fmaxf(mx, s[4 * x4 + y]);
        }
      }
      return xor32_max(mx) * (CT == kF16 ? c : 1.f);
    };
    auto rescale = [&](float mx) {
      if (__any(mx > m + kAbove)) {
        const float mn = fmaxf(m, mx - kBelow);
        const float alpha = m == -INFINITY ? 0.f : exp2_of(m - mn);
        m = mn;
        l *= alpha;
#pragma unroll
        for (int dt = 0; dt < DS; ++dt)
#pragma unroll
          for (int x = 0; x < 16; ++x) o[dt][x] *= alpha;
      }
    };
    // The step of a half whose scores are `cur` (half t of the page whose V is
    // vt and whose scales are in slot s3), beside the scores `nxt` of the next
    // half (tn of kt, slot n3); returns the largest of those.  First the next
    // scores' products with the weights, then the values' products with the
    // maximum.  The scheduling barriers keep each product beside its share of
    // the softmax, and operands three products ahead.
    auto step = [&](const f32x16& cur, f32x16& nxt, const char* kt, int tn, int n3, const char* vt, int t, int s3) {
      constexpr int N = 2 * DS, PER = 16 / N, AHEAD = 3;
      const float mu = m == -INFINITY ? 0.f : m;  // scores of -inf only so far: weights 0
      const char* v_at[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) v_at[e] = vt + col * 128 + ((v_x ^ (4 * t + e)) * 16);
      // operands 0 .. N - 1: K's; N .. 2 N - 1: V's
      f16x8 x[2 * N];
      auto read = [&](int i) {
        if (i < N)
          x[i] = *reinterpret_cast<const f16x8*>(kt + tn * (32 * 128) + k_at[(i / 2) % 2][i % 2] + (i / 4) * (kPage * 128));
        else if (i < 2 * N)
          x[i] = *reinterpret_cast<const f16x8*>(v_at[(i - N) / DS] + (i - N) % DS * (32 * 128));
      };
      f32x4 r[4], f[4], lv[4];
      const float *sc0 = &s_sc[s3][2][32 * t + 16 * half], *sc1 = &s_sc[n3][0][32 * tn + 16 * half];
      if constexpr (CT != kF16) {
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = *reinterpret_cast<const f32x4*>(sc0 + 4 * i);
      }
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) read(i);
#pragma unroll
      for (int i = 0; i < 16; ++i) nxt[i] = 0.f;
      f16x8 pw[2];
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        read(i + AHEAD);
        nxt = __builtin_amdgcn_mfma_f32_32x32x16_f16(x[i], qf[i / 2][i % 2], nxt, 0, 0, 0);
#pragma unroll
        for (int y = PER * i; y < PER * (i + 1); ++y) {
          const float w = exp2_of(CT == kF16 ? __builtin_fmaf(cur[y], c, -mu) : cur[y] - mu);
          l = CT == kF16 ? l + w : __builtin_fmaf(w, r[y / 4][y % 4], l);
          pw[y / 8][y % 8] = static_cast<_Float16>(w);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      float mx = -INFINITY;
      auto scale4 = [&](int i) {
        if constexpr (CT != kF16) {
          f[i] = *reinterpret_cast<const f32x4*>(sc1 + 4 * i);
          lv[i] = *reinterpret_cast<const f32x4*>(sc1 + kPage + 4 * i);
        }
      };
      auto max4 = [&](int i) {
#pragma unroll
        for (int y = 4 * i; y < 4 * i + 4; ++y) {
          if constexpr (CT != kF16) nxt[y] = __builtin_fmaf(nxt[y], f[i][y % 4], lv[i][y % 4]);
          mx = fmaxf(mx, nxt[y]);
        }
      };
      if constexpr (N == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) scale4(i);
      }
#pragma unroll
      for (int i = 0; i < N; ++i) {
        read(N + i + AHEAD);
        if (N == 8 && i < 4) scale4(i);
        o[i % DS] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x[N + i], pw[i / DS], o[i % DS], 0, 0, 0);
        if (N == 4 || i >= 4) max4(i % 4);
        __builtin_amdgcn_sched_barrier(0);
      }
      return xor32_max(mx) * (CT == kF16 ? c : 1.f);
    };
    // Half t of a page with drafted tokens, or the sequence's end: one thing
    // after the other, each token tested.
    auto edge = [&](int p, int s3, int s2, int t) {
      const int tok0 = p * kPage + 32 * t + 16 * half;  // this lane's 16 tokens
      const uint32_t seen = row.attends16(a, sq, tok0, total, [](int x) { return x; });
      f32x16 s;
      scores(s, k_tile(s3), t);
      float mx = -INFINITY;
      largest(s, s3, t);
#pragma unroll
      for (int x = 0; x < 16; ++x) {
        const float v = CT == kF16 ? s[x] * c : s[x];
        s[x] = (seen >> x) & 1 ? v : -INFINITY;
        mx = fmaxf(mx, s[x]);
      }
      rescale(xor32_max(mx));
      const float mu = m == -INFINITY ? 0.f : m;  // a row that has attended nothing yet: weights 0
      f16x8 pw[2];
#pragma unroll
      for (int x = 0; x < 16; ++x) {
        const float w = exp2_of(s[x] - mu);
        const float r = CT == kF16 ? 1.f : s_sc[s3][2][32 * t + 16 * half + x];
        l = __builtin_fmaf(w, (seen >> x) & 1 ? r : 0.f, l);
        pw[x / 8][x % 8] = static_cast<_Float16>(w);
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const char* v_at = v_tile(s2) + col * 128 + ((v_x ^ (4 * t + e)) * 16);
#pragma unroll
        for (int dt = 0; dt < DS; ++dt) {
          u32x4 v = *reinterpret_cast<const u32x4*>(v_at + dt * (32 * 128));
          const int keep = total - tok0 - 8 * e;  // as in the rows kernel
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int k = keep - 2 * i;
            uint32_t w = v[i] & (k <= 0 ? 0u : k == 1 ? 0xffffu : ~0u);
            odd = drop_odd<kF16>(w) || odd;
            v[i] = w;
          }
          o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, v), pw[e], o[dt], 0, 0, 0);
        }
      }
    };

    if (block_live && p0 < p1) {
      // Page p's K lies in slot (p - p0) % KS and its V in (p - p0) % VS.  At the
      // top of page p, K of pages p and p + 1 and V of page p have arrived.
      const bool two = p0 + 1 < p1;
      int64_t head = pages.head(p0);
      if constexpr (CT == kF16) {
        dma(a.k, head, k_tile(0), k_src);
        dma(a.v, head, v_tile(0), v_src);
        if (two) {
          head = pages.head(p0 + 1);
          dma(a.k, head, k_tile(1), k_src);
          dma(a.v, head, v_tile(1), v_src);
        }
        if (p0 + 2 < p1) {
          head = pages.head(p0 + 2);
          dma(a.k, head, k_tile(2), k_src);
        }
      } else {
        take_k(head);
        take_v(head);
        put_k(0, p0, head);
        put_v(0);
        if (two) {
          head = pages.head(p0 + 1);
          take_k(head);
          take_v(head);
          put_k(1, p0 + 1, head);
          if (p0 + 2 < p1) {
            head = pages.head(p0 + 2);
            take_k(head);
          }
        }
      }
      const int whole = min(p1, sq.ctx / kPage);
      int s3 = 0, s2 = 0;
      f32x16 sa, sb;
      // The top of page p: its arrivals, and the loads of what comes after.
      auto top = [&](int p) {
        const int kf = s3 == 0 ? KS - 1 : s3 - 1, vf = s2 == 0 ? VS - 1 : s2 - 1;  // the slots that page p - 1 had
        if constexpr (CT == kF16) {
          // K of page p + 1 and V of page p have arrived when no more is on its
          // way than V of p + 1 and K of p + 2.  (__syncthreads() would wait for all.)
          if (p + 2 < p1)
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(2 * (TILE / 1024 / W)) : "memory");
          else
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
          __builtin_amdgcn_s_barrier();  // and every wavefront is done with page p - 1
          asm volatile("" ::: "memory");
          if (p + 2 < p1) dma(a.v, head, v_tile(vf), v_src);
          if (p + 3 < p1) {
            head = pages.head(p + 3);
            dma(a.k, head, k_tile(kf), k_src);
          }
        } else {
          __syncthreads();
          if (p + 1 < p1) put_v(vf);
          if (p + 2 < p1) {
            put_k(kf, p + 2, head);
            take_v(head);
          }
          if (p + 3 < p1) {
            head = pages.head(p + 3);
            take_k(head);
          }
          if (s_odd[s3]) {
            patch_v(s2, s3);
            __syncthreads();
          }
        }
      };
      auto next = [&] {
        s3 = s3 == KS - 1 ? 0 : s3 + 1;
        s2 = s2 == VS - 1 ? 0 : s2 + 1;
      };
      if (wave_live) {
        int p = p0;
        if (p < whole) {  // sa: the scores of the page's first (or only) half
          top(p);
          scores(sa, k_tile(0), part);
          rescale(largest(sa, 0, part));
          for (;;) {
            // (past the last whole page the scores ahead are of no page, and not used)
            const int n3 = s3 == KS - 1 ? 0 : s3 + 1;
            const char *k0 = k_tile(s3), *k1 = k_tile(n3), *v0 = v_tile(s2);
            float mx;
            if constexpr (RT == W) {
              mx = step(sa, sb, k0, 1, s3, v0, 0, s3);
              rescale(mx);
              mx = step(sb, sa, k1, 0, n3, v0, 1, s3);
            } else {
              mx = step(sa, sb, k1, part, n3, v0, part, s3);
              sa = sb;
            }
            next();
            if (++p == whole) break;
            rescale(mx);
            top(p);
          }
        }
        for (; p < p1; ++p, next()) {
          top(p);
          if constexpr (RT == W) {
#pragma unroll 1
            for (int t = 0; t < 2; ++t) edge(p, s3, s2, t);
          } else {
            edge(p, s3, s2, part);
          }
        }
      } else {
        for (int p = p0; p < p1; ++p, next()) top(p);
      }
      if (__any(odd)) {
        const int t0 = max(p0, whole) * kPage, t1 = min(p1 * kPage, total);
        add_odd<CT, D, DS * 16>(
            a, sq, b, kvh, row, lane, t0, t1, RT == W ? -1 : part,
            [](int x, int ln) { return 32 * (x / 16) + 8 * (x % 16 / 4) + 4 * (ln >> 5) + x % 4; },
            [&](int x, float f) { o[x / 16][x % 16] += f; });
      }
    }
    l = xor32_sum(l);
    if (!row.live) m = -INFINITY, l = 0.f;
    if ((pages.poisoned || sq.bad) && row.live) l = NAN;
    if constexpr (RT != W) {  // the second half's wavefront hands over
      f32x4* x = reinterpret_cast<f32x4*>(s_kv) + local * (DS * 4 * 64) + lane;
      __syncthreads();  // the tiles are read
      if (part == 1) {
#pragma unroll
        for (int i = 0; i < DS * 4; ++i)
          x[i * 64] = f32x4{o[i / 4][4 * (i % 4)], o[i / 4][4 * (i % 4) + 1], o[i / 4][4 * (i % 4) + 2], o[i / 4][4 * (i % 4) + 3]};
        s_ml[(local * 64 + lane) * 2] = m;
        s_ml[(local * 64 + lane) * 2 + 1] = l;
      }
      __syncthreads();
      if (part == 0) {
        const float m1 = s_ml[(local * 64 + lane) * 2], l1 = s_ml[(local * 64 + lane) * 2 + 1];
        const float M = fmaxf(m, m1);
        const float f0 = m == -INFINITY ? 0.f : exp2_of(m - M), f1 = m1 == -INFINITY ? 0.f : exp2_of(m1 - M);
        l = (m == -INFINITY ? l : l * f0) + (m1 == -INFINITY ? l1 : l1 * f1);  // l without a reference is 0, or NaN
        m = M;
#pragma unroll
        for (int i = 0; i < DS * 4; ++i) {
          const f32x4 y = x[i * 64];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float z = f0 == 0.f ? 0.f : o[i / 4][4 * (i % 4) + e] * f0;
            if (f1 != 0.f) z += y[e] * f1;
            o[i / 4][4 * (i % 4) + e] = z;
          }
        }
      }
    }
    if (part == 0 && tile * kTile + col < a.rows) {
      const int64_t part_row = partial_of(a, range, rb, pc.slot, local * kTile + col);
      float* x = a.ws + part_row * D + 4 * half;
#pragma unroll
      for (int dt = 0; dt < DS; ++dt)
#pragma unroll
        for (int x4 = 0; x4 < 4; ++x4) {
          const f32x4 y = {o[dt][4 * x4], o[dt][4 * x4 + 1], o[dt][4 * x4 + 2], o[dt][4 * x4 + 3]};
          if (pc.whole)
            store_row4<D>(a, b, row.i, row.head, 32 * dt + 8 * x4 + 4 * half, y, m, l);
          else
            *reinterpret_cast<f32x4*>(x + 32 * dt + 8 * x4) = y;
        }
      if (!pc.whole && half == 0) {
        float* ml = a.ws + partials(a) * D + part_row * 2;
        ml[0] = m, ml[1] = l;
      }
    }
    advance(a, walk, pc);
    __syncthreads();  // LDS is read before the next piece writes it
  }
}

// Joins the partials of each (sequence, KV head) that several ranges share: a
// thread 4 features of a row.  For the wide kernel, whose partials are too many
// for one workgroup (100 rows to each of 16 x 8: 8 us, most of it the launch and
// the chain lengths, references, partials).
template <int D>
__global__ __launch_bounds__(256) void tree_merge_kernel(TreeArgs a) {
  const uint32_t pair = blockIdx.x, b = fdiv(pair, a.by_hkv), kvh = pair - b * a.Hkv;
  Walk w;
  w.seek(a, threadIdx.x % 64, b);
  int r0, r1;
  w.parts_of(a, kvh, r0, r1);
  if (r1 <= r0) return;
  const Seq sq = w.seq;
  for (int u = blockIdx.y * 256 + threadIdx.x; u < a.rows * (D / 4); u += gridDim.y * 256) {
    const int row = u / (D / 4), d = 4 * (u % (D / 4));
    const int i = static_cast<int>(fdiv(row, a.by_g)), rb = row / a.block_rows, rl = row - rb * a.block_rows;
    float M = -INFINITY, L = 0.f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    if (i < sq.n)
      merge_parts(r0, r1, M, L, acc, [&](int r, float& m, float& l, f32x4& x) {
        const int64_t part = partial_of(a, r, rb, r == r0 ? 1 : 0, rl);
        const float* ml = a.ws + partials(a) * D + part * 2;
        m = ml[0], l = ml[1];
        x = *reinterpret_cast<const f32x4*>(a.ws + part * D + d);
      });
    store_row4<D>(a, b, i, kvh * a.g + row - i * a.g, d, acc, M, L);
  }
}

constexpr int kWaves = 8;  // of every workgroup
static_assert(kWaves == kWideWaves, "one workgroup to a compute unit in all three kernels");
constexpr int kFewRows = 16;
// Rows up to here take the rows kernel, whose two tiles read a piece's pages
// twice; but fp16 pages of head_dim 128 (large_pages) go through LDS at once.
// 16 x 8192 tokens, 32 / 8 heads, 8 and 16 drafted (32 and 64 rows), us by rows
// and through LDS: fp16 139, 209 and 119, 131; head_dim 64 51, 70 and 75, 79;
// e4m3 56, 59 and 120 (25 drafted).
constexpr int kNarrowRows = 64;
constexpr bool large_pages(int kind, int D) { return kind == kF16 && D == 128; }  // 32 KiB for K and V

struct Plan {
  int wide;  // row tiles of a workgroup of the wide kernel; 0: the rows kernel; -1: the few, -2: in half workgroups
  int row_blocks, block_rows, width, ranges, min_per, min_cut;
  bool merge;  // a second kernel joins the parts
  size_t ws_bytes;
};

Plan plan_of(int kind, int B, int T, int Hq, int Hkv, int D, int max_tokens) {
  Plan p;
  const int64_t rows = static_cast<int64_t>(T) * (Hq / Hkv);
  // Half workgroups, two to a compute unit, where each has a (sequence, KV
  // head) of its own (64 x 8 x 1024 tokens 28.8 -> 25.5 us, x 8192 168.5 -> 165.5);
  // fewer would be cut for them (32 x 8 x 4096 45.6 -> 50.0).
  p.wide = rows <= kFewRows ? (static_cast<int64_t>(B) * Hkv >= 512 ? -2 : -1) : rows <= kNarrowRows && !large_pages(kind, D) ? 0 : rows <= 128 ? 4 : 8;
  p.block_rows = kTile * std::max(p.wide, 1);
  p.row_blocks = static_cast<int>((rows + p.block_rows - 1) / p.block_rows);
  p.width = static_cast<int>(std::min<int64_t>(p.block_rows, rows));
  // Parts of fewer pages cost more to join than they save (one sequence of 1024
  // tokens, us at 2 / 3 / 4 / 8 pages a part: 64 rows 13.2 / 13.5 / 15 / 17;
  // 256 rows, whose joining is launched in any case, 29 / 31 / 32 / 42).  Nor is
  // a sequence cut whose wavefronts have one page each, or two of 16 KiB
  // (700 tokens, few rows: int8 10.6 whole, 11.7 in parts; fp16 17.8 and 15.2),
  // nor one in LDS whose pages are few where whole ones fill half the device (16 x
  // 25 drafted tokens x 32 / 8 heads over 1000, e4m3: 41.9 whole, 46.4 in parts;
  // over 1500 49.1 and 39.9).
  p.min_per = p.wide > 0 ? 2 : p.wide < 0 ? 3 : 6;
  const int64_t slots = p.wide == -2 ? 512 : 256;
  const bool half = 2 * p.row_blocks * (static_cast<int64_t>(B) * Hkv) >= slots;
  p.min_cut = p.wide > 0 ? (half ? 20 : 4) : p.wide == 0 ? 12 : large_pages(kind, D) ? 9 : 13;
  // One round of the device, or as many parts as there can be.
  const int64_t pages = std::max(pages_of(max_tokens), 1), parts_of_one = pages < p.min_cut ? 1 : pages / p.min_per;
  const int64_t ranges = std::min(B * (Hkv * parts_of_one), std::max<int64_t>(slots / p.row_blocks, 1));
  p.ranges = static_cast<int>(std::max<int64_t>(ranges, 1));
  const int64_t parts = static_cast<int64_t>(p.ranges) * p.row_blocks * 2;
  p.ws_bytes = static_cast<size_t>(parts * p.width * (D + 2) + parts) * 4;
  p.merge = p.wide > 0;
  return p;
}

template <int CT, int D>
void launch(const TreeArgs& a, int wide, dim3 grid, hipStream_t st) {
  if (wide == 8) {
    tree_wide_kernel<CT, D, 8><<<grid, kWideWaves * 64, 0, st>>>(a);
  } else if (wide == 4) {
    tree_wide_kernel<CT, D, 4><<<grid, kWideWaves * 64, 0, st>>>(a);
  } else if (wide == 0) {
    if constexpr (!large_pages(CT, D)) tree_rows_kernel<CT, D, kWaves><<<grid, kWaves * 64, 0, st>>>(a);
  } else if (wide == -1) {
    tree_few_kernel<CT, D, kWaves><<<dim3(a.ranges), kWaves * 64, 0, st>>>(a);
  } else {
    tree_few_kernel<CT, D, kWaves / 2><<<dim3(a.ranges), kWaves / 2 * 64, 0, st>>>(a);
  }
}

// T and the tokens of a sequence that a call may hold.  The merge kernel indexes
// rows x D / 4 in 32 bits, and its loop passes the last by up to kMergeBlocks
// workgroups of 256.
constexpr int kMergeBlocks = 2048;

bool sizes_ok(int B, int T, int Hq, int Hkv, int D, int max_ctx) {
  return B >= 0 && T > 0 && Hkv > 0 && Hq > 0 && Hq % Hkv == 0 && (D == 64 || D == 128) && max_ctx >= 0 &&
         static_cast<int64_t>(T) * (Hq / Hkv) * (D / 4) < (int64_t{1} << 31) - 256 * kMergeBlocks &&
         static_cast<int64_t>(max_ctx) + T < (int64_t{1} << 31) - kPage;
}

}  // namespace

extern "C" size_t spyre_paged_tree_attn_workspace_bytes(int cache_kind, int B, int T, int Hq, int Hkv, int D, int max_context_len,
                                                        int draft_keys) {
  if (!sizes_ok(B, T, Hq, Hkv, D, max_context_len)) return 0;
  return plan_of(cache_kind, B, T, Hq, Hkv, D, max_context_len + (draft_keys ? T : 0)).ws_bytes;
}

extern "C" int spyre_paged_tree_attn(const void* q, const int64_t* q_strides, const void* k_cache, const void* v_cache,
                                     const float* k_scale, const float* v_scale, int cache_kind,
                                     const int32_t* block_table, int64_t bt_stride, int64_t pages_per_seq,
                                     const int32_t* context_lens, const int32_t* draft_lens, int draft_keys,
                                     const void* mask, const int64_t* mask_strides, void* out, float* lse,
                                     void* workspace, size_t workspace_bytes, int B, int T, int Hq, int Hkv, int D,
                                     int page_size, int64_t num_pages, int max_context_len, float scale, void* stream) {
  spyre_hip::clear_error();
  SPYRE_REQUIRE(D == 64 || D == 128, SPYRE_EUNSUPPORTED, "head_dim %d not in {64, 128}", D);
  SPYRE_REQUIRE(page_size == kPage, SPYRE_EUNSUPPORTED, "page_size %d != %d", page_size, kPage);
  SPYRE_REQUIRE(B >= 0 && T >= 0 && Hkv > 0 && Hq > 0 && Hq % Hkv == 0 && max_context_len >= 0 && pages_per_seq >= 0 &&
                    bt_stride >= 0,
                SPYRE_EINVAL, "bad sizes B=%d T=%d Hq=%d Hkv=%d max_context_len=%d", B, T, Hq, Hkv, max_context_len);
  SPYRE_REQUIRE(cache_kind == SPYRE_CACHE_F16 || cache_kind == SPYRE_CODES_E4M3 || cache_kind == SPYRE_CODES_INT8,
                SPYRE_EINVAL, "unknown cache kind %d", cache_kind);
  if (B == 0 || T == 0) return SPYRE_OK;
  SPYRE_REQUIRE(sizes_ok(B, T, Hq, Hkv, D, max_context_len), SPYRE_EUNSUPPORTED, "too many rows or tokens");
  SPYRE_REQUIRE(num_pages > 0, SPYRE_EINVAL, "bad num_pages");
  const bool f16 = cache_kind == SPYRE_CACHE_F16;
  SPYRE_REQUIRE(q && q_strides && k_cache && v_cache && block_table && context_lens && out && (f16 || (k_scale && v_scale)) &&
                    (!mask || mask_strides),
                SPYRE_EINVAL, "null pointer argument");
  auto aligned = [](const void* p, int n) { return reinterpret_cast<uintptr_t>(p) % n == 0; };
  SPYRE_REQUIRE(aligned(q, 16) && aligned(k_cache, 16) && aligned(v_cache, 16) && aligned(out, 16), SPYRE_EINVAL,
                "q, the caches and out must be 16-byte aligned");
  for (int i = 0; i < 3; ++i)
    SPYRE_REQUIRE(q_strides[i] % 8 == 0, SPYRE_EINVAL, "q strides must be multiples of 8 elements");
  const Plan p = plan_of(cache_kind, B, T, Hq, Hkv, D, max_context_len + (draft_keys ? T : 0));
  SPYRE_REQUIRE(p.ws_bytes == 0 || (workspace && workspace_bytes >= p.ws_bytes && aligned(workspace, 16)), SPYRE_ENOSPC,
                "workspace holds %zu bytes, need %zu (16-byte aligned)", workspace ? workspace_bytes : 0, p.ws_bytes);
  TreeArgs a{};
  a.q = static_cast<const _Float16*>(q), a.q_sb = q_strides[0], a.q_st = q_strides[1], a.q_sh = q_strides[2];
  a.k = static_cast<const uint8_t*>(k_cache), a.v = static_cast<const uint8_t*>(v_cache), a.ks = k_scale, a.vs = v_scale;
  a.bt = block_table, a.bt_stride = bt_stride, a.pages_per_seq = pages_per_seq, a.num_pages = num_pages;
  a.ctx = context_lens, a.counts = draft_lens, a.draft_keys = draft_keys != 0;
  a.mask = static_cast<const uint8_t*>(mask);
  if (mask) a.m_sb = mask_strides[0], a.m_si = mask_strides[1], a.m_sj = mask_strides[2];
  a.out = static_cast<_Float16*>(out), a.lse = lse, a.ws = static_cast<float*>(workspace);
  a.B = B, a.T = T, a.Hq = Hq, a.Hkv = Hkv, a.g = Hq / Hkv, a.rows = T * a.g;
  a.max_ctx = max_context_len, a.scale_log2 = scale * kLog2e;
  a.row_blocks = p.row_blocks, a.block_rows = p.block_rows, a.width = p.width;
  a.ranges = p.ranges, a.min_per = p.min_per, a.min_cut = p.min_cut;
  a.each = static_cast<int64_t>(B) * Hkv % p.ranges == 0 ? static_cast<int>(static_cast<int64_t>(B) * Hkv / p.ranges) : 0;
  a.ticket = spyre_hip::next_call_ticket();
  const int64_t pairs = static_cast<int64_t>(B) * Hkv, blocks = static_cast<int64_t>((p.ranges + 7) / 8 * 8) * p.row_blocks;
  SPYRE_REQUIRE(pairs * (pages_of(max_context_len + T) + kStart + 1) < (int64_t{1} << 30) && blocks < (int64_t{1} << 31),
                SPYRE_EUNSUPPORTED, "too many pages or rows");
  a.by_g = make_fastdiv(static_cast<uint32_t>(a.g)), a.by_hkv = make_fastdiv(static_cast<uint32_t>(Hkv));
  a.by_blocks = make_fastdiv(static_cast<uint32_t>(p.row_blocks));
  a.by_ranges = make_fastdiv(static_cast<uint32_t>(p.ranges));
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid(static_cast<uint32_t>(blocks));
  auto go = [&](auto kind) {
    constexpr int CT = decltype(kind)::value;
    D == 128 ? launch<CT, 128>(a, p.wide, grid, st) : launch<CT, 64>(a, p.wide, grid, st);
  };
  if (f16)
    go(std::integral_constant<int, SPYRE_CACHE_F16>{});
  else if (cache_kind == SPYRE_CODES_E4M3)
    go(std::integral_constant<int, SPYRE_CODES_E4M3>{});
  else
    go(std::integral_constant<int, SPYRE_CODES_INT8>{});
  hipError_t e = hipGetLastError();
  SPYRE_REQUIRE(e == hipSuccess, SPYRE_EHIP, "tree attention launch failed: %s", hipGetErrorString(e));
  if (p.merge) {
    // Workgroups whose rows nobody shared leave at once; too many of those cost
    // more than a few long loops (8192 of them 23 us).
    const int64_t n = std::min((static_cast<int64_t>(a.rows) * (D / 4) + 255) / 256, std::max<int64_t>(kMergeBlocks / pairs, 1));
    const dim3 merge(static_cast<uint32_t>(pairs), static_cast<uint32_t>(n));
    if (D == 128)
      tree_merge_kernel<128><<<merge, 256, 0, st>>>(a);
    else
      tree_merge_kernel<64><<<merge, 256, 0, st>>>(a);
    e = hipGetLastError();
    SPYRE_REQUIRE(e == hipSuccess, SPYRE_EHIP, "tree attention merge launch failed: %s", hipGetErrorString(e));
  }
  return SPYRE_OK;
}
