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

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "cache8.h"
#include "fast_div.h"
#include "spyre_common.h"

namespace {

using namespace spyre_hip;

typedef c8_f16x8 f16x8;
typedef c8_u32x4 u32x4;
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kPage = 64;
constexpr int kTile = 32;  // query rows of a tile, and tokens of an MFMA
constexpr int kF16 = SPYRE_CACHE_F16;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// The running reference of a row's exponents moves only when a score passes it
// by more than this (log2 units): weights up to 2^8 are as exact in fp16 as
// those up to 1, and most steps then skip the rescaling of O.
constexpr float kSlack = 8.f;

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
  int B, T, Hq, Hkv, g, rows, tiles, max_ctx, draft_keys, chunk_pages, max_chunks;
  float scale_log2;
  uint32_t pairs;  // B Hkv
  int row_blocks;  // of the wide kernel
  FastDiv by_g, by_hkv, by_tiles, by_pairs, by_blocks;
};

__device__ __forceinline__ float xor32_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x), false, false);
  return fmaxf(__builtin_bit_cast(float, static_cast<unsigned>(r[0])), __builtin_bit_cast(float, static_cast<unsigned>(r[1])));
}

__device__ __forceinline__ float xor32_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x), false, false);
  return __builtin_bit_cast(float, static_cast<unsigned>(r[0])) + __builtin_bit_cast(float, static_cast<unsigned>(r[1]));
}

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

// The token of MFMA row m of a 32-token tile: row 16 e + 8 a + 4 H + r is token
// 16 H + 8 e + 4 a + r, so that accumulator register i of lane half H is token
// 16 H + i.
__device__ __forceinline__ int token_of(int m) {
  return 16 * ((m >> 2) & 1) + 8 * (m >> 4) + 4 * ((m >> 3) & 1) + (m & 3);
}

__host__ __device__ __forceinline__ int pages_of(int tokens) { return tokens / kPage + (tokens % kPage != 0); }
__host__ __device__ __forceinline__ int chunks_of(int pages, int chunk_pages) {
  return pages == 0 ? 1 : (pages + chunk_pages - 1) / chunk_pages;
}

// What a sequence holds.  bad: it breaks the max_context_len contract.
struct Seq {
  int ctx, n, pages;
  bool bad;
};

__device__ __forceinline__ Seq seq_of(const TreeArgs& a, int b) {
  Seq s;
  const int raw = a.ctx[b];
  s.bad = raw > a.max_ctx;
  s.ctx = min(max(raw, 0), a.max_ctx);
  s.n = a.counts ? min(max(a.counts[b], 0), a.T) : a.T;
  s.pages = pages_of(s.ctx + (a.draft_keys ? s.n : 0));
  return s;
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
    if ((at & 63) == 0) ids = p + lane < a.pages_per_seq ? trow[p + lane] : -1;
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
  // Which of the 16 tokens from t on the row attends (total: all there are).
  // Every mask byte is loaded, and none waits for another.
  __device__ __forceinline__ uint32_t attends16(const TreeArgs& a, const Seq& sq, int t, int total) const {
    uint32_t seen = 0;
    const int j0 = t - sq.ctx;
    if (mask) {
      uint8_t keep[16];
#pragma unroll
      for (int x = 0; x < 16; ++x) keep[x] = mask[min(max(j0 + x, 0), a.T - 1) * a.m_sj];
#pragma unroll
      for (int x = 0; x < 16; ++x) seen |= static_cast<uint32_t>(j0 + x < 0 || keep[x] != 0) << x;
    } else {
      const int n = i - j0 + 1;  // tokens of the 16 up to i's own
      seen = n <= 0 ? 0u : n >= 16 ? 0xffffu : (1u << n) - 1;
    }
    const int n = total - t;
    return live && n > 0 ? seen & (n >= 16 ? 0xffffu : (1u << n) - 1) : 0u;
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

// Q^T operands of a lane's row: features 32 s + 16 half + 8 e .. + 7.
template <int DS>
__device__ __forceinline__ void load_q(const TreeArgs& a, int b, const Row& r, int half, f16x8 (&qf)[DS][2]) {
  const _Float16* qp = a.q + b * a.q_sb + r.i * a.q_st + r.head * a.q_sh + 16 * half;
#pragma unroll
  for (int s = 0; s < DS; ++s)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      qf[s][e] = f16x8{};
      if (r.live) qf[s][e] = *reinterpret_cast<const f16x8*>(qp + 32 * s + 8 * e);
    }
}

// The infinities and NaNs of tokens t0 .. t1 - 1 that drop_odd left out of O,
// number by number.
template <int CT, int D>
__device__ void add_odd(const TreeArgs& a, const Seq& sq, int b, int kvh, const Row& r, int lane, int t0, int t1,
                        f32x16 (&o)[D / 32]) {
  constexpr int KB = CT == kF16 ? 2 : 1;
  const int half = lane >> 5;
  Pages pages(a, b, kvh, lane, t0 / kPage);
  for (int t = t0; t < t1; ++t) {
    const bool attends = r.attends16(a, sq, t, t + 1);
    const uint8_t* v = a.v + pages.head(t / kPage) * (static_cast<int64_t>(kPage) * D * KB);
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int x = 0; x < 16; ++x) {
        const int d = 32 * dt + 8 * (x / 4) + 4 * half + x % 4;
        float f = 0.f;
        if constexpr (CT == kF16) {
          f = static_cast<float>(reinterpret_cast<const _Float16*>(v)[d * kPage + t % kPage]);
          if (__builtin_fabsf(f) <= 65504.f) f = 0.f;
        } else {
          if ((v[(t % kPage / 16) * (D * 16) + d * 16 + t % 16] & 0x7f) == 0x7f) f = NAN;
        }
        if (attends) o[dt][x] += f;
      }
  }
}

// W wavefronts share a chunk of a (sequence, KV head, row tile): each takes
// its own steps of it, and they join in LDS.
template <int CT, int D, int W>
__global__ __launch_bounds__(W * 64, 2) void tree_rows_kernel(TreeArgs a) {
  constexpr int STEP = 32, PER_PAGE = kPage / STEP;
  constexpr int KB = CT == kF16 ? 2 : 1;  // bytes of an element
  constexpr int DS = D / 32;
  constexpr int ROW = D + 4;  // floats of a row in LDS
  __shared__ __align__(16) float s_mem[W * kTile * (ROW + 2)];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
  const int col = lane & 31, half = lane >> 5;
  // Row tiles of one chunk read the same pages: 8 blocks apart, so that they
  // meet in one XCD's L2.
  const uint32_t blk = blockIdx.x, lo8 = blk & 7, hi = blk >> 3;
  const uint32_t hi_t = fdiv(hi, a.by_tiles), tile = hi - hi_t * a.tiles, item = hi_t * 8 + lo8;
  const uint32_t chunk = fdiv(item, a.by_pairs), pair = item - chunk * a.pairs;
  if (chunk >= static_cast<uint32_t>(a.max_chunks)) return;
  const uint32_t b = fdiv(pair, a.by_hkv), kvh = pair - b * a.Hkv;
  const Seq sq = seq_of(a, b);
  const int nch = chunks_of(sq.pages, a.chunk_pages);
  if (static_cast<int>(chunk) >= nch) return;
  const int total = sq.ctx + (a.draft_keys ? sq.n : 0);
  // Equal shares of the sequence's steps for the chunks, of a chunk's for the wavefronts.
  const int steps = (total + STEP - 1) / STEP;
  const int c0 = static_cast<int>(static_cast<int64_t>(chunk) * steps / nch);
  const int c1 = static_cast<int>(static_cast<int64_t>(chunk + 1) * steps / nch);
  const int s0 = c0 + (c1 - c0) * wave / W, s1 = c0 + (c1 - c0) * (wave + 1) / W;

  const Row row = row_of(a, sq, b, kvh, tile * kTile + col);
  f16x8 qf[DS][2];
  load_q<DS>(a, b, row, half, qf);
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
    const uint8_t* p = a.k + head * (static_cast<int64_t>(kPage) * D * KB) + k_off;
    if constexpr (CT == kF16) {
#pragma unroll
      for (int s = 0; s < DS; ++s)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          kr.x[s][e] = *reinterpret_cast<const u32x4*>(p + hp * (STEP * 128) + (s / 2) * (kPage * 128) + (s % 2) * 64 + 16 * e);
    } else {
#pragma unroll
      for (int s = 0; s < DS; ++s)
        kr.x[s][0] = *reinterpret_cast<const u32x4*>(p + hp * (STEP * 16) + 2 * s * (kPage * 16));
      scale = (half ? a.vs : a.ks)[head * kPage + hp * STEP + col];
    }
  };
  auto load_v = [&](int st) {
    const int hp = st % PER_PAGE;
    const uint8_t* p = a.v + head * (static_cast<int64_t>(kPage) * D * KB) + v_off;
    if constexpr (CT == kF16) {
#pragma unroll
      for (int dt = 0; dt < DS; ++dt)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          vr.x[dt][e] = *reinterpret_cast<const u32x4*>(p + hp * (STEP * 2) + dt * (32 * kPage * 2) + 16 * e);
    } else {
#pragma unroll
      for (int dt = 0; dt < DS; ++dt)
        vr.x[dt][0] = *reinterpret_cast<const u32x4*>(p + 2 * hp * (D * 16) + dt * (32 * 16));
    }
  };
  // 8-bit: this wavefront's step: score factors, V's scales' logarithms and inverses.
  float* s_sc = s_mem + wave * 3 * STEP;

  auto step = [&](int st, bool more, auto edge_tag) {
    constexpr bool EDGE = decltype(edge_tag)::value;  // some tokens are drafted or do not exist
    const int tok0 = st * STEP + 16 * half;           // this lane's 16 tokens
    uint32_t seen = 0;                                // those that its row attends
    if constexpr (EDGE) seen = row.attends16(a, sq, tok0, total);
    uint32_t odd_scale = 0, inf_scale = 0;  // of this lane's 16 tokens, those whose V has no finite scale
    if constexpr (CT != kF16) {
      __builtin_amdgcn_wave_barrier();
      const bool finite = __builtin_fabsf(scale) <= 0x1.fffffep127f;
      odd_scale = static_cast<uint32_t>(__builtin_amdgcn_ballot_w64(half && !finite) >> (32 + 16 * half)) & 0xffffu;
      inf_scale = static_cast<uint32_t>(__builtin_amdgcn_ballot_w64(half && scale == INFINITY) >> (32 + 16 * half)) & 0xffffu;
      const float vc = !finite ? 1.f : scale < 0x1p-60f ? 0x1p-60f : scale;  // V's scale 0: codes of no weight
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
    if (more) {
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
    if (__any(mx > m + kSlack)) {
      const float mn = fmaxf(m, mx);
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
        if ((odd_scale >> x) & 1 && (!EDGE || (seen >> x) & 1)) p[x / 8][x % 8] = static_cast<_Float16>((inf_scale >> x) & 1 ? INFINITY : NAN);
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
    if (more) load_v(st + 1);
  };

  if (s0 < s1) {
    locate(s0);
    load_k(s0);
    load_v(s0);
  }
  // Every row attends every token of a step below ctx (rows without a drafted
  // token drop theirs at the end), so only the last steps test tokens.
  int st = s0;
  const int whole = min(s1, sq.ctx / STEP);
  for (; st < whole; ++st) step(st, st + 1 < s1, std::false_type{});
  for (; st < s1; ++st) step(st, st + 1 < s1, std::true_type{});
  if (CT != SPYRE_CODES_INT8 && __any(odd))
    add_odd<CT, D>(a, sq, b, kvh, row, lane, max(s0, whole) * STEP, min(s1 * STEP, total), o);
  l = xor32_sum(l);
  if (!row.live) m = -INFINITY, l = 0.f;
  if ((pages.poisoned || sq.bad) && row.live) l = NAN;

  // Join the wavefronts: O, m and l of the rows that exist, then every thread
  // folds elements in wavefront order.
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
  const bool single = nch == 1;
  const int64_t slot = (static_cast<int64_t>(pair) * a.tiles + tile) * a.max_chunks + chunk;
  const int64_t slots = static_cast<int64_t>(a.pairs) * a.tiles * a.max_chunks;
  const int width = min(kTile, a.rows);  // rows of a partial
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
      L += mw == -INFINITY ? lw : lw * f;  // lw without a reference is 0, or NaN
      if (mw != -INFINITY) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(s_o + (w * rows + r) * ROW + d);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] += x[e] * f;
      }
    }
    if (single) {
      const int rr = tile * kTile + r, ii = static_cast<int>(fdiv(rr, a.by_g)), hh = kvh * a.g + rr - ii * a.g;
      const int64_t at = (static_cast<int64_t>(b) * a.T + ii) * a.Hq + hh;
      const float inv = L == 0.f ? 0.f : 1.f / L;
      f16x4 y;
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = static_cast<_Float16>(L == 0.f ? 0.f : acc[e] * inv);
      *reinterpret_cast<f16x4*>(a.out + at * D + d) = y;
      if (a.lse && d == 0) a.lse[at] = L == 0.f ? -INFINITY : (M + log2f(L)) * kLn2;
    } else {
      *reinterpret_cast<f32x4*>(a.ws + (slot * width + r) * D + d) = acc;
      if (d == 0) {
        float* ml = a.ws + slots * width * D + (slot * width + r) * 2;
        ml[0] = M, ml[1] = L;
      }
    }
  }
}

// ---------------------------------------------------------- wide drafts --
//
// W wavefronts, 32 rows each, share every page of a chunk through LDS: K [D/64,
// 64 tok, 64] and V [D, 64 tok] as fp16, in two slots.  8-bit pages are
// converted once on the way in.  A 128-byte row is 8 units of 16 bytes; unit u
// lies at u ^ swz(row), so that the 16 lanes that a read serves at once, and a
// conversion's 16 stores, meet 16 different bank groups.
__device__ __forceinline__ int swz_k(int row) { return ((row >> 1) & 3) | ((((row >> 3) ^ (row >> 4)) & 1) << 2); }
__device__ __forceinline__ int swz_v(int row) { return (row >> 1) & 7; }

typedef __amdgpu_buffer_rsrc_t Rsrc;

template <int CT, int D, int W>
__global__ __launch_bounds__(W * 64, 2) void tree_wide_kernel(TreeArgs a) {
  constexpr int DS = D / 32;
  constexpr int TILE = kPage * D * 2;         // bytes of a K or a V tile
  constexpr int SLOT = 2 * TILE;
  constexpr int KU = kPage * D / 16;            // 8-bit: units of a K or a V page
  constexpr int UNITS = 2 * KU / (W * 64);      // of both, that a thread converts
  static_assert(CT == kF16 || (UNITS >= 1 && KU % 64 == 0), "every thread has a unit, and a wavefront's are all K or all V");
  __shared__ __align__(16) char s_kv[2 * SLOT];
  __shared__ __align__(16) float s_sc[2][3][kPage];  // 8-bit: score factors, V's scales' logarithms and inverses
  __shared__ uint64_t s_odd[2][2];                   // and which of V's scales are not finite, and infinite
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
  const int col = lane & 31, half = lane >> 5;
  const uint32_t blk = blockIdx.x, lo8 = blk & 7, hi = blk >> 3;
  const uint32_t hi_t = fdiv(hi, a.by_blocks), rb = hi - hi_t * a.row_blocks, item = hi_t * 8 + lo8;
  const uint32_t chunk = fdiv(item, a.by_pairs), pair = item - chunk * a.pairs;
  if (chunk >= static_cast<uint32_t>(a.max_chunks)) return;
  const uint32_t b = fdiv(pair, a.by_hkv), kvh = pair - b * a.Hkv;
  const Seq sq = seq_of(a, b);
  const int nch = chunks_of(sq.pages, a.chunk_pages);
  if (static_cast<int>(chunk) >= nch) return;
  const int total = sq.ctx + (a.draft_keys ? sq.n : 0);
  const int p0 = static_cast<int>(static_cast<int64_t>(chunk) * sq.pages / nch);
  const int p1 = static_cast<int>(static_cast<int64_t>(chunk + 1) * sq.pages / nch);
  const int tile = rb * W + wave;
  const Row row = row_of(a, sq, b, kvh, tile * kTile + col);
  Pages pages(a, b, kvh, lane, p0);
  bool odd = false;
  const bool block_live = static_cast<int>(rb) * W * kTile < sq.n * a.g;  // some row of the workgroup is drafted
  const bool wave_live = tile * kTile < sq.n * a.g;
  f16x8 qf[DS][2];
  load_q<DS>(a, b, row, half, qf);
  f32x16 o[DS];
#pragma unroll
  for (int dt = 0; dt < DS; ++dt)
#pragma unroll
    for (int x = 0; x < 16; ++x) o[dt][x] = 0.f;
  float m = -INFINITY, l = 0.f;

  // fp16 pages go straight into LDS: load i of a tile fills its bytes 1024 i
  // .., lane by lane, so each lane fetches the unit that belongs at its place.
  const int l8 = lane / 8;
  const int k_src = 1024 * wave + 128 * l8 + (((lane % 8) ^ swz_k(8 * wave + l8)) * 16);
  const int v_src = 1024 * wave + 128 * l8 + (((lane % 8) ^ swz_v(8 * wave + l8)) * 16);
  static_assert(W % 4 == 0, "the loads of a wavefront share their swizzle");
  // 8-bit: the next page's units and scales, in registers.
  u32x4 raw[CT == kF16 ? 1 : UNITS];
  float scale = 0.f;
  auto fetch = [&](int p, int slot) {
    const int64_t head = pages.head(p);
    if constexpr (CT == kF16) {
      const uint8_t *kp = a.k + head * TILE, *vp = a.v + head * TILE;
      const Rsrc kr = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(kp), 0, TILE, 0x00020000);
      const Rsrc vr = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(vp), 0, TILE, 0x00020000);
#pragma unroll
      for (int j = 0; j < TILE / 1024 / W; ++j) {
        char* dk = s_kv + slot * SLOT + 1024 * (wave + W * j);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(kr, (__attribute__((address_space(3))) void*)dk, 16, k_src, 1024 * W * j, 0, 0);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(vr, (__attribute__((address_space(3))) void*)(dk + TILE), 16, v_src,
                                                 1024 * W * j, 0, 0);
      }
    } else {
#pragma unroll
      for (int j = 0; j < UNITS; ++j) {
        const int w0 = (wave + j * W) * 64;  // this wavefront's first unit, of K's and then V's
        const uint8_t* p8 = w0 < KU ? a.k + head * (TILE / 2) + w0 * 16 : a.v + head * (TILE / 2) + (w0 - KU) * 16;
        raw[j] = *reinterpret_cast<const u32x4*>(p8 + lane * 16);
      }
      if (wave < 2) scale = (wave ? a.vs : a.ks)[head * kPage + lane];
    }
  };
  // 8-bit: what fetch() brought, into a slot.
  auto store = [&](int slot) {
    if constexpr (CT != kF16) {
      char* k0 = s_kv + slot * SLOT;
      auto two = [&](char* at, int u, int sw, const u32x4& w) {  // units u and u + 1 of a row
        *reinterpret_cast<f16x8*>(at + ((u ^ sw) * 16)) = codes_to_f16x8<CT>(w[0], w[1]);
        *reinterpret_cast<f16x8*>(at + (((u + 1) ^ sw) * 16)) = codes_to_f16x8<CT>(w[2], w[3]);
      };
#pragma unroll
      for (int j = 0; j < UNITS; ++j) {
        const int w0 = (wave + j * W) * 64;
        if (w0 < KU) {  // 16 features un of a token
          const int un = w0 / kPage, tok = lane;
          two(k0 + (un / 4) * (kPage * 128) + tok * 128, 2 * (un % 4), swz_k(tok), raw[j]);
        } else {  // 16 tokens q4 of a feature
          const int x = w0 - KU + lane, q4 = x / D, d = x % D;
          two(k0 + TILE + d * 128, 2 * q4, swz_v(d), raw[j]);
        }
      }
      if (wave == 0) s_sc[slot][0][lane] = scale * a.scale_log2;
      if (wave == 1) {
        const bool finite = __builtin_fabsf(scale) <= 0x1.fffffep127f;
        const float vc = !finite ? 1.f : scale < 0x1p-60f ? 0x1p-60f : scale;  // 0: codes of no weight
        s_sc[slot][1][lane] = __builtin_amdgcn_logf(vc);
        s_sc[slot][2][lane] = __builtin_amdgcn_rcpf(vc);
        const uint64_t not_finite = __builtin_amdgcn_ballot_w64(!finite);
        const uint64_t infinite = __builtin_amdgcn_ballot_w64(scale == INFINITY);
        if (lane == 0) s_odd[slot][0] = not_finite, s_odd[slot][1] = infinite;
      }
    }
  };

  // Operand addresses in a slot: unit u of a row is (bits of the unroll) ^
  // (bits of the lane), four of each.
  const int tok = token_of(col);
  const int k_row = tok * 128, v_row = col * 128;
  const int k_x = (2 * half) ^ swz_k(tok), v_x = (2 * half) ^ swz_v(col);
  int k_at[2][2];
#pragma unroll
  for (int y = 0; y < 2; ++y)
#pragma unroll
    for (int e = 0; e < 2; ++e) k_at[y][e] = k_row + ((k_x ^ (4 * y + e)) * 16);

  // The 32 tokens from half t of page p on.
  auto step = [&](int p, int slot, int t, auto edge_tag) {
    constexpr bool EDGE = decltype(edge_tag)::value;
    const char* base = s_kv + slot * SLOT;
    const int s0 = 32 * t + 16 * half, tok0 = p * kPage + s0;  // this lane's 16 tokens
    uint32_t seen = 0;
    if constexpr (EDGE) seen = row.attends16(a, sq, tok0, total);
    f32x16 sc;
#pragma unroll
    for (int x = 0; x < 16; ++x) sc[x] = 0.f;
#pragma unroll
    for (int s = 0; s < DS; ++s)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const f16x8 k = *reinterpret_cast<const f16x8*>(base + t * (32 * 128) + k_at[s % 2][e] + (s / 2) * (kPage * 128));
        sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, qf[s][e], sc, 0, 0, 0);
      }
    float mx = -INFINITY;
#pragma unroll
    for (int x4 = 0; x4 < 4; ++x4) {
      f32x4 f, lv;
      if constexpr (CT != kF16) {
        f = *reinterpret_cast<const f32x4*>(&s_sc[slot][0][s0 + 4 * x4]);
        lv = *reinterpret_cast<const f32x4*>(&s_sc[slot][1][s0 + 4 * x4]);
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
    if (__any(mx > m + kSlack)) {
      const float mn = fmaxf(m, mx);
      const float alpha = m == -INFINITY ? 0.f : exp2_of(m - mn);
      m = mn;
      l *= alpha;
#pragma unroll
      for (int dt = 0; dt < DS; ++dt)
#pragma unroll
        for (int x = 0; x < 16; ++x) o[dt][x] *= alpha;
    }
    const float mu = m == -INFINITY ? 0.f : m;
    f16x8 pw[2];
#pragma unroll
    for (int x4 = 0; x4 < 4; ++x4) {
      f32x4 r;
      if constexpr (CT != kF16) r = *reinterpret_cast<const f32x4*>(&s_sc[slot][2][s0 + 4 * x4]);
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const int x = 4 * x4 + y;
        const float w = exp2_of(sc[x] - mu);
        if constexpr (CT == kF16)
          l += w;
        else
          l = __builtin_fmaf(w, EDGE && !((seen >> x) & 1) ? 0.f : r[y], l);
        pw[x / 8][x % 8] = static_cast<_Float16>(w);
      }
    }
    if constexpr (CT != kF16) {
      const uint32_t not_finite = static_cast<uint32_t>(s_odd[slot][0] >> s0) & 0xffffu;
      if (__any(not_finite != 0)) {
        const uint32_t infinite = static_cast<uint32_t>(s_odd[slot][1] >> s0) & 0xffffu;
#pragma unroll
        for (int x = 0; x < 16; ++x)
          if ((not_finite >> x) & 1 && (!EDGE || (seen >> x) & 1))
            pw[x / 8][x % 8] = static_cast<_Float16>((infinite >> x) & 1 ? INFINITY : NAN);
      }
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const char* v_at = base + TILE + v_row + ((v_x ^ (4 * t + e)) * 16);
#pragma unroll
      for (int dt = 0; dt < DS; ++dt) {
        u32x4 v = *reinterpret_cast<const u32x4*>(v_at + dt * (32 * 128));
        if constexpr (EDGE) {  // as in the rows kernel
          const int keep = total - tok0 - 8 * e;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int k = keep - 2 * i;
            uint32_t w = v[i] & (k <= 0 ? 0u : k == 1 ? 0xffffu : ~0u);
            odd = drop_odd<kF16>(w) || odd;
            v[i] = w;
          }
        }
        o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, v), pw[e], o[dt], 0, 0, 0);
      }
    }
  };

  if (block_live && p0 < p1) {
    fetch(p0, 0);
    if constexpr (CT != kF16) {
      store(0);
      if (p0 + 1 < p1) fetch(p0 + 1, 1);
    }
    const int whole = min(p1, sq.ctx / kPage);
    for (int p = p0; p < p1; ++p) {
      const int slot = (p - p0) & 1;
      if constexpr (CT == kF16) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();  // page p is in its slot, and every wavefront is done with the other one
      if constexpr (CT == kF16) {
        if (p + 1 < p1) fetch(p + 1, slot ^ 1);
      } else {
        if (p + 1 < p1) store(slot ^ 1);
        if (p + 2 < p1) fetch(p + 2, slot);
      }
      if (wave_live) {
        if (p < whole) {
          step(p, slot, 0, std::false_type{});
          step(p, slot, 1, std::false_type{});
        } else {
#pragma unroll 1
          for (int t = 0; t < 2; ++t) step(p, slot, t, std::true_type{});
        }
      }
    }
    if (CT != SPYRE_CODES_INT8 && __any(odd))
      add_odd<CT, D>(a, sq, b, kvh, row, lane, max(p0, whole) * kPage, min(p1 * kPage, total), o);
  }
  l = xor32_sum(l);
  if (!row.live) m = -INFINITY, l = 0.f;
  if ((pages.poisoned || sq.bad) && row.live) l = NAN;
  if (tile * kTile + col >= a.rows) return;
  if (nch == 1) {
    const int64_t at = (static_cast<int64_t>(b) * a.T + row.i) * a.Hq + row.head;
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int dt = 0; dt < DS; ++dt)
#pragma unroll
      for (int x4 = 0; x4 < 4; ++x4) {
        f16x4 y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = static_cast<_Float16>(l == 0.f ? 0.f : o[dt][4 * x4 + e] * inv);
        *reinterpret_cast<f16x4*>(a.out + at * D + 32 * dt + 8 * x4 + 4 * half) = y;
      }
    if (a.lse && half == 0) a.lse[at] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
  } else {
    const int64_t slot = (static_cast<int64_t>(pair) * a.tiles + tile) * a.max_chunks + chunk;
    const int64_t slots = static_cast<int64_t>(a.pairs) * a.tiles * a.max_chunks;
    float* x = a.ws + (slot * kTile + col) * D + 4 * half;
#pragma unroll
    for (int dt = 0; dt < DS; ++dt)
#pragma unroll
      for (int x4 = 0; x4 < 4; ++x4)
        *reinterpret_cast<f32x4*>(x + 32 * dt + 8 * x4) =
            f32x4{o[dt][4 * x4], o[dt][4 * x4 + 1], o[dt][4 * x4 + 2], o[dt][4 * x4 + 3]};
    if (half == 0) {
      float* ml = a.ws + slots * kTile * D + (slot * kTile + col) * 2;
      ml[0] = m, ml[1] = l;
    }
  }
}

// Joins the chunks of sequences that have several: a thread 4 features of a row.
template <int D>
__global__ __launch_bounds__(256) void tree_merge_kernel(TreeArgs a) {
  const int64_t u = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t r_all = u / (D / 4);
  const int d = 4 * static_cast<int>(u % (D / 4));
  if (r_all >= static_cast<int64_t>(a.pairs) * a.rows) return;
  const uint32_t pair = static_cast<uint32_t>(r_all / a.rows), row = static_cast<uint32_t>(r_all % a.rows);
  const uint32_t b = fdiv(pair, a.by_hkv), kvh = pair - b * a.Hkv;
  const Seq sq = seq_of(a, b);
  const int nch = chunks_of(sq.pages, a.chunk_pages);
  if (nch == 1) return;
  const int tile = row / kTile, r = row % kTile, width = min(kTile, a.rows);
  const int64_t slot0 = (static_cast<int64_t>(pair) * a.tiles + tile) * a.max_chunks;
  const int64_t slots = static_cast<int64_t>(a.pairs) * a.tiles * a.max_chunks;
  const float* ml = a.ws + slots * width * D + (slot0 * width + r) * 2;
  const float* x = a.ws + (slot0 * width + r) * D + d;
  float M = -INFINITY, L = 0.f;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int c = 0; c < nch; ++c) M = fmaxf(M, ml[static_cast<int64_t>(c) * width * 2]);
  for (int c = 0; c < nch; ++c) {
    const float mc = ml[static_cast<int64_t>(c) * width * 2], lc = ml[static_cast<int64_t>(c) * width * 2 + 1];
    const float f = mc == -INFINITY ? 0.f : exp2_of(mc - M);
    L += mc == -INFINITY ? lc : lc * f;
    if (mc != -INFINITY) {
      const f32x4 y = *reinterpret_cast<const f32x4*>(x + static_cast<int64_t>(c) * width * D);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] += y[e] * f;
    }
  }
  const int ii = static_cast<int>(fdiv(row, a.by_g)), hh = kvh * a.g + row - ii * a.g;
  const int64_t at = (static_cast<int64_t>(b) * a.T + ii) * a.Hq + hh;
  const float inv = L == 0.f ? 0.f : 1.f / L;
  f16x4 y;
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = static_cast<_Float16>(L == 0.f ? 0.f : acc[e] * inv);
  *reinterpret_cast<f16x4*>(a.out + at * D + d) = y;
  if (a.lse && d == 0) a.lse[at] = L == 0.f ? -INFINITY : (M + log2f(L)) * kLn2;
}

constexpr int kRowWaves = 4;
// Rows up to here take the rows kernel: two tiles read a chunk's pages twice.
constexpr int kNarrowRows = 64;

struct Plan {
  int tiles, waves, row_blocks;  // waves 0: the rows kernel
  int chunk_pages, max_chunks;
  size_t ws_bytes;
};

// Chunks: enough workgroups to fill the device, each wavefront at least a
// page, at most 8 pages a wavefront.
Plan plan_of(int B, int T, int Hq, int Hkv, int D, int max_tokens) {
  Plan p;
  const int64_t rows = static_cast<int64_t>(T) * (Hq / Hkv);
  p.tiles = static_cast<int>((rows + kTile - 1) / kTile);
  p.waves = rows <= kNarrowRows ? 0 : rows <= 128 ? 4 : 8;
  p.row_blocks = p.waves ? (p.tiles + p.waves - 1) / p.waves : p.tiles;
  const int pages = pages_of(max_tokens);
  const int64_t groups = static_cast<int64_t>(B) * Hkv * p.row_blocks;
  if (p.waves == 0) {
    int cp = 8 * kRowWaves;
    while (cp > kRowWaves && groups * chunks_of(pages, cp) < 512) cp /= 2;
    p.chunk_pages = cp;
  } else {
    // Rounds of the device times a workgroup's steps, its start counted as
    // four of them.
    const int64_t slots = p.waves == 8 ? 256 : 512;
    int64_t best = INT64_MAX;
    p.chunk_pages = std::max(pages, 1);
    for (int n = 1; n <= std::max(pages, 1) && n <= 256; ++n) {
      const int cp = (pages + n - 1) / n;
      const int64_t rounds = (groups * n + slots - 1) / slots, cost = rounds * (cp + 4) + (n > 1 ? 4 : 0);
      if (cost < best) best = cost, p.chunk_pages = std::max(cp, 1);
    }
  }
  p.max_chunks = chunks_of(pages, p.chunk_pages);
  const int64_t width = std::min<int64_t>(kTile, rows);
  p.ws_bytes = p.max_chunks == 1 ? 0 : static_cast<size_t>(static_cast<int64_t>(B) * Hkv * p.tiles * p.max_chunks * width * (D + 2)) * 4;
  return p;
}

template <int CT, int D>
void launch(const TreeArgs& a, int waves, dim3 grid, hipStream_t st) {
  if (waves == 8)
    tree_wide_kernel<CT, D, 8><<<grid, 512, 0, st>>>(a);
  else if (waves == 4)
    tree_wide_kernel<CT, D, 4><<<grid, 256, 0, st>>>(a);
  else
    tree_rows_kernel<CT, D, kRowWaves><<<grid, kRowWaves * 64, 0, st>>>(a);
}

// T and the tokens of a sequence that a call may hold.
bool sizes_ok(int B, int T, int Hq, int Hkv, int D, int max_ctx) {
  return B >= 0 && T > 0 && Hkv > 0 && Hq > 0 && Hq % Hkv == 0 && (D == 64 || D == 128) && max_ctx >= 0 &&
         static_cast<int64_t>(T) * (Hq / Hkv) < (int64_t{1} << 30) && static_cast<int64_t>(max_ctx) + T < (int64_t{1} << 31) - kPage;
}

}  // namespace

extern "C" size_t spyre_paged_tree_attn_workspace_bytes(int cache_kind, int B, int T, int Hq, int Hkv, int D, int max_context_len,
                                                        int draft_keys) {
  (void)cache_kind;
  if (!sizes_ok(B, T, Hq, Hkv, D, max_context_len)) return 0;
  return plan_of(B, T, Hq, Hkv, D, max_context_len + (draft_keys ? T : 0)).ws_bytes;
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
  const Plan p = plan_of(B, T, Hq, Hkv, D, max_context_len + (draft_keys ? T : 0));
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
  a.tiles = p.tiles, a.chunk_pages = p.chunk_pages, a.max_chunks = p.max_chunks, a.max_ctx = max_context_len;
  a.scale_log2 = scale * kLog2e;
  const int64_t pairs = static_cast<int64_t>(B) * Hkv;
  const int64_t items = (pairs * p.max_chunks + 7) / 8 * 8;
  SPYRE_REQUIRE(items * p.row_blocks < (int64_t{1} << 31), SPYRE_EUNSUPPORTED, "too many workgroups");
  a.pairs = static_cast<uint32_t>(pairs);
  a.by_g = make_fastdiv(static_cast<uint32_t>(a.g)), a.by_hkv = make_fastdiv(static_cast<uint32_t>(Hkv));
  a.row_blocks = p.row_blocks, a.by_blocks = make_fastdiv(static_cast<uint32_t>(p.row_blocks));
  a.by_tiles = make_fastdiv(static_cast<uint32_t>(p.tiles)), a.by_pairs = make_fastdiv(a.pairs);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid(static_cast<uint32_t>(items * p.row_blocks));
  auto go = [&](auto kind) {
    constexpr int CT = decltype(kind)::value;
    D == 128 ? launch<CT, 128>(a, p.waves, grid, st) : launch<CT, 64>(a, p.waves, grid, st);
  };
  if (f16)
    go(std::integral_constant<int, SPYRE_CACHE_F16>{});
  else if (cache_kind == SPYRE_CODES_E4M3)
    go(std::integral_constant<int, SPYRE_CODES_E4M3>{});
  else
    go(std::integral_constant<int, SPYRE_CODES_INT8>{});
  hipError_t e = hipGetLastError();
  SPYRE_REQUIRE(e == hipSuccess, SPYRE_EHIP, "tree attention launch failed: %s", hipGetErrorString(e));
  if (p.max_chunks > 1) {
    const int64_t n = (pairs * a.rows * (D / 4) + 255) / 256;
    SPYRE_REQUIRE(n < (int64_t{1} << 31), SPYRE_EUNSUPPORTED, "too many rows");
    if (D == 128)
      tree_merge_kernel<128><<<dim3(static_cast<uint32_t>(n)), 256, 0, st>>>(a);
    else
      tree_merge_kernel<64><<<dim3(static_cast<uint32_t>(n)), 256, 0, st>>>(a);
    e = hipGetLastError();
    SPYRE_REQUIRE(e == hipSuccess, SPYRE_EHIP, "tree attention merge launch failed: %s", hipGetErrorString(e));
  }
  return SPYRE_OK;
}
