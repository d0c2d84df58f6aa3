// Writes and reads of the 8-bit paged cache (cache8.h has its layout).
//
// A row x (one token, one KV head, D features) is held as codes and a scale:
//   amax = max |x|,  scale = amax / TOP,  code = rne(x TOP / amax)
// with TOP = 448 (e4m3) or 127 (int8), in fp32.  The product x TOP is exact for
// fp16 rows, so one correctly rounded division decides the code and ties go to
// even as the definition says.  Rows without a value of 2^-100 or more are zeros
// of scale 1; a NaN or an infinity makes the scale NaN or infinite, and the whole
// row reads back as NaN.
//
// Both directions are bound by memory (a large copy 4.88 TB/s).  3 x 2500 tokens
// of 32 heads of 128, int8: written in 48 to 56 us, 3.3 to 3.9 TB/s (54 where the
// last reader's rows are still on their way to memory), read in 30 to 34.  8 x
// 8500 rows of 8 heads, 4500 of them held, e4m3: 73 us, 4.8 TB/s.  A decode step
// of 32 tokens: 6.5 and 4.5 us, the chains of their loads.

#include <hip/hip_runtime.h>

#include <algorithm>

#include "cache8.h"
#include "fast_div.h"
#include "rotary.h"
#include "spyre_common.h"

namespace {

using namespace spyre_hip;

constexpr int kPage = 64;
constexpr int kGroup = 16;   // tokens of a work group: a V unit
constexpr int kWaves = 4;
constexpr int kLdsPairs = 64;  // R / 2 <= D / 2

typedef c8_f16x8 f16x8;
typedef c8_u32x4 u32x4;
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4), aligned(4)));  // scales may lie anywhere

__device__ __forceinline__ uint32_t umax_row(uint32_t x, bool sixteen) {
#define SPYRE_DPP(ctrl) x = max(x, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(x), ctrl, 0xf, 0xf, false)))
  SPYRE_DPP(0xb1);   // quad_perm 1 0 3 2
  SPYRE_DPP(0x4e);   // quad_perm 2 3 0 1
  SPYRE_DPP(0x141);  // row_half_mirror: the other quad of 8 lanes
  if (sixteen) SPYRE_DPP(0x140);  // row_mirror: the other 8 of 16 lanes
#undef SPYRE_DPP
  return x;
}

template <int KIND>
constexpr float kTop = KIND == SPYRE_CODES_E4M3 ? 448.f : 127.f;

// 8 values of a row whose largest magnitude has the bits `top` -> 8 codes.
template <int KIND>
__device__ __forceinline__ float quantise8(const float (&x)[8], uint32_t top, uint32_t (&w)[2]) {
  float amax = __builtin_bit_cast(float, top);
  if (amax < 0x1p-100f) amax = kTop<KIND>;
  float y[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] = x[e] * kTop<KIND> / amax;
  if constexpr (KIND == SPYRE_CODES_E4M3) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      int r = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i], y[4 * i + 1], 0, false);
      w[i] = static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i + 2], y[4 * i + 3], r, true));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      w[i] = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        w[i] |= (static_cast<uint32_t>(static_cast<int>(rintf(y[4 * i + e]))) & 0xffu) << (8 * e);
    }
  }
  return amax / kTop<KIND>;
}

struct AppendArgs {
  const _Float16 *q, *k, *v;
  int64_t q_sb, q_st, q_sh, k_sb, k_st, k_sh, v_sb, v_st, v_sh;
  _Float16* q_out;  // [B, T, Hq, D]
  uint8_t *kc, *vc;
  float *ks, *vs;
  const int32_t *bt, *slots;
  int64_t bt_stride, pages_per_seq, sl_sb, sl_st, num_pages;
  const void* rot_pos;
  int64_t rp_sb, rp_st;
  int rot_wide;
  const double* freq;
  float amplitude;
  int half;  // rotated pairs; 0: none
  int T, Hq, Hkv, groups, rows_per_slice, q_rows, kv_rows;  // rows: 128 features of 128 / D heads
  FastDiv by_groups;
};

// One workgroup: 16 tokens of a sequence (cut so that a run of consecutive
// slots meets the cache's 16-token units), and of their heads the rows of one
// slice.  A wavefront takes a row of 16 lanes x 8 features for 4 x 4 tokens at
// once (lane group g: tokens 4 g .. 4 g + 3), so that a whole V unit turns
// into 16-byte pieces in registers (4 x 4 bytes, then 4 x 4 words over the lane
// groups); quarters of a unit are written as words, other tokens byte by byte.
template <int KIND, int D, bool ROTATE, bool INTERLEAVED>
__global__ __launch_bounds__(kWaves * 64) void append_kernel(AppendArgs a) {
  constexpr int HP = 128 / D;      // heads of a row
  constexpr int LH = 16 / HP;      // lanes of a head
  __shared__ float s_cs[ROTATE ? kGroup * 2 * kLdsPairs : 1];
  const uint32_t b = fdiv(blockIdx.x, a.by_groups);
  const int gi = static_cast<int>(blockIdx.x - b * a.groups);
  const int32_t* sl = a.slots + b * a.sl_sb;
  const int first = sl[0], last = sl[(a.T - 1) * a.sl_st];
  // Any cut is right; this one meets the units of runs padded on either side.
  const int off = first >= 0 ? first % kGroup : last >= 0 ? (last % kGroup + kGroup - (a.T - 1) % kGroup) % kGroup : 0;
  const int t0 = gi * kGroup - off;
  if (t0 >= a.T) return;
  if constexpr (ROTATE) {
    const int lo = max(0, -t0), n = min(kGroup, a.T - t0) - lo;
    for (int i = threadIdx.x; i < n * a.half; i += kWaves * 64) {
      const int t = lo + i / a.half, p = i % a.half;
      const int64_t at = b * a.rp_sb + (t0 + t) * a.rp_st;
      const double pos = a.rot_wide ? static_cast<double>(static_cast<const int64_t*>(a.rot_pos)[at])
                                    : static_cast<double>(static_cast<const int32_t*>(a.rot_pos)[at]);
      float c, s;
      cos_sin_of(pos, a.freq[p], c, s);
      s_cs[t * 2 * kLdsPairs + p] = c * a.amplitude;
      s_cs[t * 2 * kLdsPairs + kLdsPairs + p] = s * a.amplitude;
    }
    __syncthreads();
  }
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
  const int rl = lane % 16, g = lane / 16;
  const int f = 8 * (rl % LH);  // this lane's first feature
  // This lane's tokens 4 g + p: whether they exist, and where they go.
  bool live[4];
  int64_t where[4];  // page * Hkv * 64 + slot, or -1
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const int t = t0 + 4 * g + p;
    live[p] = t >= 0 && t < a.T;
    const int slot = live[p] ? sl[t * a.sl_st] : -1;
    where[p] = -1;
    if (slot >= 0 && slot / kPage < a.pages_per_seq) {
      const int64_t page = a.bt[b * a.bt_stride + slot / kPage];
      if (page >= 0 && page < a.num_pages) where[p] = page * a.Hkv * kPage + slot % kPage;
    }
  }
  const int64_t unit0 = __builtin_amdgcn_readfirstlane(static_cast<int>(where[0] & 0xffffffff)) & 0xffffffffll;
  const int64_t unit = unit0 | static_cast<int64_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(where[0] >> 32))) << 32;
  bool in_unit = unit >= 0 && unit % kGroup == 0;
  bool quad = where[0] >= 0 && where[0] % 4 == 0;  // this lane's tokens are a quarter of a unit
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    in_unit = in_unit && where[p] == unit + 4 * g + p;
    quad = quad && where[p] == where[0] + p;
  }
  const bool whole = __all(in_unit);
  const int row_end = min(a.q_rows + 2 * a.kv_rows, static_cast<int>(blockIdx.y + 1) * a.rows_per_slice);
  for (int r = blockIdx.y * a.rows_per_slice + wave; r < row_end; r += kWaves) {
    // rows: q, then K, then V
    const int what = r < a.q_rows ? 0 : r < a.q_rows + a.kv_rows ? 1 : 2;
    const int row = what == 0 ? r : what == 1 ? r - a.q_rows : r - a.q_rows - a.kv_rows;
    const int h = row * HP + rl / LH;
    const bool head = h < (what == 0 ? a.Hq : a.Hkv);
    const _Float16* src = what == 0 ? a.q : what == 1 ? a.k : a.v;
    const int64_t sb = what == 0 ? a.q_sb : what == 1 ? a.k_sb : a.v_sb;
    const int64_t st = what == 0 ? a.q_st : what == 1 ? a.k_st : a.v_st;
    const int64_t sh = what == 0 ? a.q_sh : what == 1 ? a.k_sh : a.v_sh;
    src += b * sb + h * sh;
    const bool turn = ROTATE && what != 2 && f < 2 * a.half;
    const int fo = INTERLEAVED ? f : f < a.half ? f + a.half : f - a.half;  // the partners'
    f16x8 x[4], xo[4];
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      x[p] = xo[p] = f16x8{};
      if (live[p] && head) {
        const _Float16* at = src + (t0 + 4 * g + p) * st;
        x[p] = *reinterpret_cast<const f16x8*>(at + f);
        if (!INTERLEAVED && turn) xo[p] = *reinterpret_cast<const f16x8*>(at + fo);
      }
    }
    uint32_t w[4][2];
    float scale[4];
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = static_cast<float>(x[p][e]);
      if (turn && live[p]) {
        const float* cs = s_cs + (4 * g + p) * 2 * kLdsPairs;
        if constexpr (INTERLEAVED) {
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            const float c = cs[(f + e) / 2], s = cs[kLdsPairs + (f + e) / 2];
            turn_pair(y[e], y[e + 1], c, s, y[e], y[e + 1]);
          }
        } else {
          const int p0 = f < a.half ? f : f - a.half;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float c = cs[p0 + e], s = cs[kLdsPairs + p0 + e], o = static_cast<float>(xo[p][e]);
            float y1, y2;
            turn_pair(f < a.half ? y[e] : o, f < a.half ? o : y[e], c, s, y1, y2);
            y[e] = f < a.half ? y1 : y2;
          }
        }
      }
      if (what == 0) {
        if (live[p] && head) {
          f16x8 o;
#pragma unroll
          for (int e = 0; e < 8; ++e) o[e] = static_cast<_Float16>(y[e]);
          *reinterpret_cast<f16x8*>(a.q_out + ((static_cast<int64_t>(b) * a.T + t0 + 4 * g + p) * a.Hq + h) * D + f) = o;
        }
        continue;
      }
      uint32_t top = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) top = max(top, __builtin_bit_cast(uint32_t, y[e]) & 0x7fffffffu);
      top = umax_row(top, HP == 1);
      scale[p] = quantise8<KIND>(y, top, w[p]);
    }
    if (what == 0) continue;
    const int64_t hk = static_cast<int64_t>(h) * kPage;
    if (rl % LH == 0 && head) {
      float* sc = what == 1 ? a.ks : a.vs;
      if (quad) {
        *reinterpret_cast<f32x4*>(sc + where[0] + hk) = f32x4{scale[0], scale[1], scale[2], scale[3]};
      } else {
#pragma unroll
        for (int p = 0; p < 4; ++p)
          if (where[p] >= 0) sc[where[p] + hk] = scale[p];
      }
    }
    if (what == 1) {
      // Two lanes hold the halves of a token's units: the even one takes those
      // of its tokens 0 and 1, the odd one those of 2 and 3.
      const bool odd = lane % 2 != 0;
      auto unit_of = [&](uint32_t (&even_w)[2], uint32_t (&odd_w)[2], int64_t even_at, int64_t odd_at) {
        uint32_t mine[2], other[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint32_t x = even_w[j], y = odd_w[j];
          mine[j] = odd ? y : x;
          other[j] = static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(odd ? x : y), 0xb1, 0xf, 0xf, false));
        }
        const int64_t at = odd ? odd_at : even_at;
        if (at >= 0 && head) {
          const int64_t slot = at % kPage, base = (at - slot + hk) * D;
          *reinterpret_cast<u32x4*>(a.kc + base + (f / 16) * (kPage * 16) + slot * 16) =
              odd ? u32x4{other[0], other[1], mine[0], mine[1]} : u32x4{mine[0], mine[1], other[0], other[1]};
        }
      };
      unit_of(w[0], w[2], where[0], where[2]);
      unit_of(w[1], w[3], where[1], where[3]);
    } else if (whole) {
      const int64_t slot = unit % kPage, base = (unit - slot + hk) * D;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t z[4] = {w[0][i], w[1][i], w[2][i], w[3][i]};
        transpose4x4_b8(z);      // word e: feature f + 4 i + e, tokens 4 g ..
        transpose4x4_groups(z);  // words: tokens 0 .. 15 of feature f + 4 i + g
        if (head)
          *reinterpret_cast<u32x4*>(a.vc + base + (slot / 16) * (D * 16) + (f + 4 * i + g) * 16) = u32x4{z[0], z[1], z[2], z[3]};
      }
    } else if (quad) {
      const int64_t slot = where[0] % kPage, base = (where[0] - slot + hk) * D;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t z[4] = {w[0][i], w[1][i], w[2][i], w[3][i]};
        transpose4x4_b8(z);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (head) *reinterpret_cast<uint32_t*>(a.vc + base + (slot / 16) * (D * 16) + (f + 4 * i + e) * 16 + slot % 16) = z[e];
      }
    } else {
#pragma unroll
      for (int p = 0; p < 4; ++p)
        if (where[p] >= 0 && head) {
          const int64_t slot = where[p] % kPage, base = (where[p] - slot + hk) * D;
          uint8_t* at = a.vc + base + (slot / 16) * (D * 16) + f * 16 + slot % 16;
#pragma unroll
          for (int e = 0; e < 8; ++e) at[16 * e] = static_cast<uint8_t>(w[p][e / 4] >> (8 * (e % 4)));
        }
    }
  }
}

struct ReadArgs {
  const uint8_t *kc, *vc;
  const float *ks, *vs;
  const int32_t *bt, *lens, *start;
  int64_t bt_stride, pages_per_seq, num_pages;
  _Float16 *k, *v;  // [B, Hkv, L, D]
  int L, Hkv, windows;
  uint32_t units;
  FastDiv by_windows, by_heads;
};

// A wavefront: one page of a (sequence, KV head), of K or of V; 16 lanes store a
// run of 256 bytes (half runs in turn, or stores past the caches, 111 us where
// this takes 74).  Row i of the result is token start + i; tokens from lens on are zeros, those of a page
// that the table does not name validly NaN.
template <int KIND, int D>
__global__ __launch_bounds__(kWaves * 64, 6) void read_kernel(ReadArgs a) {
  constexpr int HP = 128 / D;
  const uint32_t u = blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  if (u >= a.units) return;
  const int lane = threadIdx.x % 64;
  const uint32_t r1 = u >> 1, bh = fdiv(r1, a.by_windows), b = fdiv(bh, a.by_heads), h = bh - b * a.Hkv;
  const int win = static_cast<int>(r1 - bh * a.windows);
  const int start = a.start ? max(a.start[b], 0) : 0;
  const int len = a.lens[b];
  const int64_t page_i = start / kPage + win, tok0 = page_i * kPage;
  if (tok0 >= static_cast<int64_t>(start) + a.L) return;
  bool bad = page_i >= a.pages_per_seq;
  int64_t page = 0;
  if (!bad && tok0 < len) {
    page = a.bt[b * a.bt_stride + page_i];
    bad = page < 0 || page >= a.num_pages;
    if (bad) page = 0;
  }
  const bool none = tok0 >= len;  // nothing of the page exists
  const int64_t head = page * a.Hkv + h;
  _Float16* out = ((u & 1) ? a.v : a.k) + static_cast<int64_t>(bh) * a.L * D;
  const float* sc = ((u & 1) ? a.vs : a.ks) + head * kPage;
  auto put = [&](int tok, int f, f16x8 x) {  // features f .. + 7 of the page's token
    const int64_t i = tok0 + tok - start;
    if (i < 0 || i >= a.L) return;
    if (tok0 + tok >= len)
      x = f16x8{};
    else if (bad)
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = static_cast<_Float16>(__builtin_nanf(""));
    *reinterpret_cast<f16x8*>(out + i * D + f) = x;
  };
  auto value = [&](uint32_t w0, uint32_t w1, float s) {
    const f16x8 x = codes_to_f16x8<KIND>(w0, w1);
    f16x8 y;
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = static_cast<_Float16>(static_cast<float>(x[e]) * s);
    return y;
  };
  const bool load = !none && !bad;
  if ((u & 1) == 0) {
    constexpr int LR = D / 8, TS = 64 / LR, N = kPage / TS;  // lanes of a token, 8 features each; tokens of an instruction
    const int f = 8 * (lane % LR), tk = lane / LR;
    const uint8_t* src = a.kc + head * (D * kPage) + f / 16 * (kPage * 16) + f % 16;
    u32x2 x[N];
    float s[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      x[i] = u32x2{0, 0};
      s[i] = 0.f;
      if (load) {
        x[i] = *reinterpret_cast<const u32x2*>(src + (tk + TS * i) * 16);
        s[i] = sc[tk + TS * i];
      }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) put(tk + TS * i, f, value(x[i][0], x[i][1], s[i]));
  } else {
    constexpr int LH = 16 / HP;  // lanes of a 16-token unit's features
    const int rl = lane % 16, g = lane / 16, f = 8 * (rl % LH);
    const uint8_t* src = a.vc + head * (D * kPage);
    u32x4 x[4 / HP][2];
    float s[4 / HP][4];
#pragma unroll
    for (int i = 0; i < 4 / HP; ++i) {
      const int un = i * HP + rl / LH;
      x[i][0] = x[i][1] = u32x4{0, 0, 0, 0};
#pragma unroll
      for (int p = 0; p < 4; ++p) s[i][p] = 0.f;
      if (load) {
        x[i][0] = *reinterpret_cast<const u32x4*>(src + un * (D * 16) + (f + g) * 16);
        x[i][1] = *reinterpret_cast<const u32x4*>(src + un * (D * 16) + (f + 4 + g) * 16);
#pragma unroll
        for (int p = 0; p < 4; ++p) s[i][p] = sc[un * 16 + 4 * g + p];
      }
    }
#pragma unroll
    for (int i = 0; i < 4 / HP; ++i) {
      uint32_t z[2][4];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int w = 0; w < 4; ++w) z[j][w] = x[i][j][w];
        transpose4x4_groups(z[j]);  // word e: feature f + 4 j + e, tokens 4 g ..
        transpose4x4_b8(z[j]);      // word p: token 4 g + p, features f + 4 j ..
      }
#pragma unroll
      for (int p = 0; p < 4; ++p) put((i * HP + rl / LH) * 16 + 4 * g + p, f, value(z[0][p], z[1][p], s[i][p]));
    }
  }
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

template <int KIND, int D>
void launch_append(const AppendArgs& a, bool interleaved, dim3 grid, hipStream_t st) {
  if (a.half == 0)
    append_kernel<KIND, D, false, false><<<grid, kWaves * 64, 0, st>>>(a);
  else if (interleaved)
    append_kernel<KIND, D, true, true><<<grid, kWaves * 64, 0, st>>>(a);
  else
    append_kernel<KIND, D, true, false><<<grid, kWaves * 64, 0, st>>>(a);
}

}  // namespace

extern "C" int spyre_kv_quant_append(const void* q, const int64_t* q_strides, void* q_out, int Hq, const void* k_new,
                                     const int64_t* k_strides, const void* v_new, const int64_t* v_strides,
                                     void* k_cache, void* v_cache, float* k_scale, float* v_scale, int codes,
                                     const int32_t* block_table, int64_t bt_stride, int64_t pages_per_seq,
                                     const int32_t* slots, int64_t slot_sb, int64_t slot_st, const void* positions,
                                     int position_bytes, int64_t pos_sb, int64_t pos_st, const double* frequencies,
                                     int pairs, float amplitude, int interleaved, int B, int T, int Hkv, int D,
                                     int page_size, int64_t num_pages, void* stream) {
  spyre_hip::clear_error();
  SPYRE_REQUIRE(B >= 0 && T >= 0 && Hkv > 0 && Hq >= 0 && num_pages > 0 && bt_stride >= 0 && pages_per_seq >= 0,
                SPYRE_EINVAL, "bad sizes B=%d T=%d Hkv=%d num_pages=%lld", B, T, Hkv, static_cast<long long>(num_pages));
  SPYRE_REQUIRE(D == 64 || D == 128, SPYRE_EUNSUPPORTED, "head_dim %d not in {64, 128}", D);
  SPYRE_REQUIRE(page_size == kPage, SPYRE_EUNSUPPORTED, "page_size %d != %d", page_size, kPage);
  SPYRE_REQUIRE(codes == SPYRE_CODES_E4M3 || codes == SPYRE_CODES_INT8, SPYRE_EINVAL, "unknown codes %d", codes);
  SPYRE_REQUIRE(pairs >= 0 && 2 * pairs <= D, SPYRE_EINVAL, "%d pairs do not fit head_dim %d", pairs, D);
  SPYRE_REQUIRE(pairs % 8 == 0, SPYRE_EUNSUPPORTED, "%d rotated features: whole multiples of 16", 2 * pairs);
  SPYRE_REQUIRE(Hq == 0 || pairs > 0, SPYRE_EINVAL, "q without a rotation");
  if (B == 0 || T == 0) return SPYRE_OK;
  SPYRE_REQUIRE(k_new && k_strides && v_new && v_strides && k_cache && v_cache && k_scale && v_scale && block_table &&
                    slots && (Hq == 0 || (q && q_strides && q_out)) && (pairs == 0 || (positions && frequencies)),
                SPYRE_EINVAL, "null pointer argument");
  SPYRE_REQUIRE(pairs == 0 || position_bytes == 4 || position_bytes == 8, SPYRE_EINVAL, "positions of %d bytes",
                position_bytes);
  SPYRE_REQUIRE(aligned16(k_new) && aligned16(v_new) && aligned16(k_cache) && aligned16(v_cache) &&
                    (Hq == 0 || (aligned16(q) && aligned16(q_out))),
                SPYRE_EINVAL, "q, k_new, v_new and the caches must be 16-byte aligned");
  for (int i = 0; i < 3; ++i)
    SPYRE_REQUIRE(k_strides[i] % 8 == 0 && v_strides[i] % 8 == 0 && (Hq == 0 || q_strides[i] % 8 == 0), SPYRE_EINVAL,
                  "q / k_new / v_new strides must be multiples of 8 elements");
  AppendArgs a{};
  a.q = static_cast<const _Float16*>(q), a.k = static_cast<const _Float16*>(k_new), a.v = static_cast<const _Float16*>(v_new);
  if (Hq) a.q_sb = q_strides[0], a.q_st = q_strides[1], a.q_sh = q_strides[2];
  a.k_sb = k_strides[0], a.k_st = k_strides[1], a.k_sh = k_strides[2];
  a.v_sb = v_strides[0], a.v_st = v_strides[1], a.v_sh = v_strides[2];
  a.q_out = static_cast<_Float16*>(q_out);
  a.kc = static_cast<uint8_t*>(k_cache), a.vc = static_cast<uint8_t*>(v_cache), a.ks = k_scale, a.vs = v_scale;
  a.bt = block_table, a.slots = slots, a.bt_stride = bt_stride, a.pages_per_seq = pages_per_seq;
  a.sl_sb = slot_sb, a.sl_st = slot_st, a.num_pages = num_pages;
  a.rot_pos = positions, a.rp_sb = pos_sb, a.rp_st = pos_st, a.rot_wide = position_bytes == 8;
  a.freq = frequencies, a.amplitude = amplitude, a.half = pairs;
  a.T = T, a.Hq = Hq, a.Hkv = Hkv;
  const int HP = 128 / D;
  a.q_rows = (Hq + HP - 1) / HP, a.kv_rows = (Hkv + HP - 1) / HP;
  a.groups = T == 1 ? 1 : static_cast<int>((static_cast<int64_t>(T) + 2 * kGroup - 2) / kGroup);
  // T == 1: one group, whose token may sit anywhere in it
  const int64_t blocks = static_cast<int64_t>(B) * a.groups;
  SPYRE_REQUIRE(blocks < (int64_t{1} << 31), SPYRE_EUNSUPPORTED, "too many tokens");
  const int rows = a.q_rows + 2 * a.kv_rows;
  // Slices of the rows while the token groups alone leave the device idle.
  int slices = 1;
  while (blocks * slices < 2048 && rows > kWaves * slices) slices *= 2;
  a.rows_per_slice = (rows + slices - 1) / slices;
  a.rows_per_slice = (a.rows_per_slice + kWaves - 1) / kWaves * kWaves;
  slices = (rows + a.rows_per_slice - 1) / a.rows_per_slice;
  a.by_groups = make_fastdiv(static_cast<uint32_t>(a.groups));
  const dim3 grid(static_cast<uint32_t>(blocks), static_cast<uint32_t>(slices));
  hipStream_t st = static_cast<hipStream_t>(stream);
  const bool il = interleaved != 0;
  if (codes == SPYRE_CODES_E4M3)
    D == 128 ? launch_append<SPYRE_CODES_E4M3, 128>(a, il, grid, st) : launch_append<SPYRE_CODES_E4M3, 64>(a, il, grid, st);
  else
    D == 128 ? launch_append<SPYRE_CODES_INT8, 128>(a, il, grid, st) : launch_append<SPYRE_CODES_INT8, 64>(a, il, grid, st);
  const hipError_t e = hipGetLastError();
  SPYRE_REQUIRE(e == hipSuccess, SPYRE_EHIP, "quantised append launch failed: %s", hipGetErrorString(e));
  return SPYRE_OK;
}

extern "C" int spyre_kv_quant_read(const void* k_cache, const void* v_cache, const float* k_scale, const float* v_scale,
                                   int codes, const int32_t* block_table, int64_t bt_stride, int64_t pages_per_seq,
                                   const int32_t* lens, const int32_t* start, void* k, void* v, int B, int Hkv, int L,
                                   int D, int page_size, int64_t num_pages, void* stream) {
  spyre_hip::clear_error();
  SPYRE_REQUIRE(B >= 0 && L >= 0 && Hkv > 0 && num_pages > 0 && bt_stride >= 0 && pages_per_seq >= 0, SPYRE_EINVAL,
                "bad sizes B=%d L=%d Hkv=%d num_pages=%lld", B, L, Hkv, static_cast<long long>(num_pages));
  SPYRE_REQUIRE(D == 64 || D == 128, SPYRE_EUNSUPPORTED, "head_dim %d not in {64, 128}", D);
  SPYRE_REQUIRE(page_size == kPage, SPYRE_EUNSUPPORTED, "page_size %d != %d", page_size, kPage);
  SPYRE_REQUIRE(codes == SPYRE_CODES_E4M3 || codes == SPYRE_CODES_INT8, SPYRE_EINVAL, "unknown codes %d", codes);
  if (B == 0 || L == 0) return SPYRE_OK;
  SPYRE_REQUIRE(k_cache && v_cache && k_scale && v_scale && block_table && lens && k && v, SPYRE_EINVAL,
                "null pointer argument");
  SPYRE_REQUIRE(aligned16(k_cache) && aligned16(v_cache) && aligned16(k) && aligned16(v), SPYRE_EINVAL,
                "the caches, k and v must be 16-byte aligned");
  ReadArgs a{};
  a.kc = static_cast<const uint8_t*>(k_cache), a.vc = static_cast<const uint8_t*>(v_cache), a.ks = k_scale, a.vs = v_scale;
  a.bt = block_table, a.lens = lens, a.start = start, a.bt_stride = bt_stride, a.pages_per_seq = pages_per_seq;
  a.num_pages = num_pages, a.k = static_cast<_Float16*>(k), a.v = static_cast<_Float16*>(v), a.L = L, a.Hkv = Hkv;
  // pages that hold L tokens from anywhere in a page
  const int64_t windows = start ? (static_cast<int64_t>(L) + 2 * kPage - 2) / kPage : (static_cast<int64_t>(L) + kPage - 1) / kPage;
  const int64_t units = static_cast<int64_t>(B) * Hkv * windows * 2;
  SPYRE_REQUIRE(units < (int64_t{1} << 31) - kWaves, SPYRE_EUNSUPPORTED, "too many pages");
  a.windows = static_cast<int>(windows), a.units = static_cast<uint32_t>(units);
  a.by_windows = make_fastdiv(static_cast<uint32_t>(windows)), a.by_heads = make_fastdiv(static_cast<uint32_t>(Hkv));
  const dim3 grid(static_cast<uint32_t>((units + kWaves - 1) / kWaves));
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (codes == SPYRE_CODES_E4M3)
    D == 128 ? read_kernel<SPYRE_CODES_E4M3, 128><<<grid, kWaves * 64, 0, st>>>(a)
             : read_kernel<SPYRE_CODES_E4M3, 64><<<grid, kWaves * 64, 0, st>>>(a);
  else
    D == 128 ? read_kernel<SPYRE_CODES_INT8, 128><<<grid, kWaves * 64, 0, st>>>(a)
             : read_kernel<SPYRE_CODES_INT8, 64><<<grid, kWaves * 64, 0, st>>>(a);
  const hipError_t e = hipGetLastError();
  SPYRE_REQUIRE(e == hipSuccess, SPYRE_EHIP, "quantised read launch failed: %s", hipGetErrorString(e));
  return SPYRE_OK;
}
