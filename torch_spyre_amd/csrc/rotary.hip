// Rotary positions of q and k (spyre_rotary): with theta = position *
// frequency_i, c = amplitude cos theta, s = amplitude sin theta, the pair i of
// every head becomes
//   y1 = x1 c - x2 s      y2 = x2 c + x1 s
// (x1, x2) the features (i, i + R/2) or, interleaved, (2i, 2i + 1); features
// from R on are copied.  The inverse takes s -> -s, which is also the gradient.
//
// Bound by memory: every element is read and written once.  A workgroup takes
// the tokens whose angles its threads can compute one each (the sines cost
// more than the rotation, and all heads of a token share them), leaves cos and
// sin in LDS, then moves (token, head, unit) items of 8 pairs, two 16-byte
// loads and stores of fp16 a lane.  8192 tokens of 64 + 8 heads of 128, fp16:
// 52.4 us, 5.8 TB/s (a large copy 4.88); 32 tokens of 32 + 8 heads 3.9 us, the
// chain of its loads.
#include <hip/hip_runtime.h>

#include <cmath>
#include <type_traits>

#include "fast_div.h"
#include "rotary.h"
#include "spyre_common.h"

namespace {

using spyre_hip::FastDiv;
using spyre_hip::fdiv;

constexpr int kThreads = 256;
constexpr int kMaxPairs = 512;  // R / 2

struct Operand {
  const void* x;
  void* y;
  int64_t xb, xh, xs, yb, yh, ys;  // strides, elements
};

struct RotaryArgs {
  Operand o[2];  // q, k
  int heads[2];
  const void* positions;
  int64_t pb, ps;
  int wide;  // positions are 64-bit
  const double* freq;
  float amplitude;
  int inverse;
  int S, D, half;
  int64_t tokens;            // B S
  int group;                 // tokens of a workgroup
  int head0_per_slice;       // heads a workgroup of a slice takes, of the q heads then the k heads
  FastDiv by_s, by_units, by_heads;  // by_heads: of a full slice
  int units, turn_units;     // units of a head: rotated ones, then copied ones
};

template <typename T, int N>
struct alignas(sizeof(T) * N >= 16 ? 16 : sizeof(T) * N) Vec {
  T v[N];
};

// T: element type; V: pairs of a unit (8, or 1 for any alignment); copied
// units are V elements.
template <typename T, int V, bool INTERLEAVED>
__global__ __launch_bounds__(kThreads) void rotary_kernel(RotaryArgs a) {
  extern __shared__ float s_cs[];  // [group][cos: half, sin: half]
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * a.group;
  const int nt = static_cast<int>(min(static_cast<int64_t>(a.group), a.tokens - t0));
  for (int i = threadIdx.x; i < nt * a.half; i += kThreads) {
    const int t = i / a.half, p = i - t * a.half;
    const uint32_t tok = static_cast<uint32_t>(t0 + t), b = fdiv(tok, a.by_s), s = tok - b * a.S;
    const int64_t at = b * a.pb + s * a.ps;
    const double pos = a.wide ? static_cast<double>(static_cast<const int64_t*>(a.positions)[at])
                              : static_cast<double>(static_cast<const int32_t*>(a.positions)[at]);
    float c, sn;
    spyre_hip::cos_sin_of(pos, a.freq[p], c, sn);
    s_cs[t * 2 * a.half + p] = c * a.amplitude;
    s_cs[t * 2 * a.half + a.half + p] = (a.inverse ? -sn : sn) * a.amplitude;
  }
  __syncthreads();
  const int h0 = blockIdx.y * a.head0_per_slice;
  const int nh = min(a.head0_per_slice, a.heads[0] + a.heads[1] - h0);
  const uint32_t items = static_cast<uint32_t>(nt) * nh * a.units;
  for (uint32_t i = threadIdx.x; i < items; i += kThreads) {
    const uint32_t r = fdiv(i, a.by_units), u = i - r * a.units;
    uint32_t t, hl;
    if (nh == a.head0_per_slice) {
      t = fdiv(r, a.by_heads);
      hl = r - t * nh;
    } else {
      t = r / nh;
      hl = r - t * nh;
    }
    int h = h0 + static_cast<int>(hl);
    const int w = h >= a.heads[0];
    if (w) h -= a.heads[0];
    const Operand& o = a.o[w];
    const uint32_t tok = static_cast<uint32_t>(t0 + t), b = fdiv(tok, a.by_s), s = tok - b * a.S;
    const T* x = static_cast<const T*>(o.x) + b * o.xb + h * o.xh + s * o.xs;
    T* y = static_cast<T*>(o.y) + b * o.yb + h * o.yh + s * o.ys;
    typedef Vec<T, V> VT;
    if (u >= static_cast<uint32_t>(a.turn_units)) {
      const int d = 2 * a.half + (u - a.turn_units) * V;
      *reinterpret_cast<VT*>(y + d) = *reinterpret_cast<const VT*>(x + d);
      continue;
    }
    const int p = u * V;
    const int d1 = INTERLEAVED ? 2 * p : p, d2 = INTERLEAVED ? 2 * p + V : p + a.half;
    const VT x1 = *reinterpret_cast<const VT*>(x + d1), x2 = *reinterpret_cast<const VT*>(x + d2);
    const float* cs = s_cs + t * 2 * a.half + p;
    VT y1, y2;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float c = cs[e], sn = cs[a.half + e];
      const float f = static_cast<float>(INTERLEAVED ? (2 * e < V ? x1.v[2 * e < V ? 2 * e : 0] : x2.v[2 * e >= V ? 2 * e - V : 0]) : x1.v[e]);
      const float g = static_cast<float>(INTERLEAVED ? (2 * e + 1 < V ? x1.v[2 * e + 1 < V ? 2 * e + 1 : 0] : x2.v[2 * e + 1 >= V ? 2 * e + 1 - V : 0]) : x2.v[e]);
      float z1, z2;
      spyre_hip::turn_pair(f, g, c, sn, z1, z2);
      const T r1 = static_cast<T>(z1), r2 = static_cast<T>(z2);
      if constexpr (INTERLEAVED) {
        if (2 * e < V) y1.v[2 * e < V ? 2 * e : 0] = r1; else y2.v[2 * e >= V ? 2 * e - V : 0] = r1;
        if (2 * e + 1 < V) y1.v[2 * e + 1 < V ? 2 * e + 1 : 0] = r2; else y2.v[2 * e + 1 >= V ? 2 * e + 1 - V : 0] = r2;
      } else {
        y1.v[e] = r1;
        y2.v[e] = r2;
      }
    }
    *reinterpret_cast<VT*>(y + d1) = y1;
    *reinterpret_cast<VT*>(y + d2) = y2;
  }
}

template <typename T>
void launch(const RotaryArgs& a, bool vec, bool interleaved, dim3 grid, hipStream_t stream) {
  const size_t lds = static_cast<size_t>(a.group) * 2 * a.half * sizeof(float);
  if (vec) {
    if (interleaved)
      rotary_kernel<T, 8, true><<<grid, kThreads, lds, stream>>>(a);
    else
      rotary_kernel<T, 8, false><<<grid, kThreads, lds, stream>>>(a);
  } else if (interleaved) {
    rotary_kernel<T, 1, true><<<grid, kThreads, lds, stream>>>(a);
  } else {
    rotary_kernel<T, 1, false><<<grid, kThreads, lds, stream>>>(a);
  }
}

}  // namespace

extern "C" int spyre_rotary(const void* q, const int64_t* q_strides, void* q_out, const int64_t* q_out_strides, int Hq,
                            const void* k, const int64_t* k_strides, void* k_out, const int64_t* k_out_strides,
                            int Hkv, int scalar_type, const void* positions, int position_bytes, int64_t pos_sb,
                            int64_t pos_ss, const double* frequencies, int pairs, float amplitude, int interleaved,
                            int inverse, int B, int S, int D, void* stream) {
  spyre_hip::clear_error();
  SPYRE_REQUIRE(B >= 0 && S >= 0 && Hq >= 0 && Hkv >= 0 && D > 0, SPYRE_EINVAL, "bad sizes B=%d S=%d Hq=%d Hkv=%d D=%d",
                B, S, Hq, Hkv, D);
  SPYRE_REQUIRE(pairs > 0 && 2 * static_cast<int64_t>(pairs) <= D, SPYRE_EINVAL,
                "%d pairs do not fit head_dim %d", pairs, D);
  SPYRE_REQUIRE(pairs <= kMaxPairs, SPYRE_EUNSUPPORTED, "more than %d pairs (%d)", kMaxPairs, pairs);
  SPYRE_REQUIRE(scalar_type == SPYRE_DT_FLOAT16 || scalar_type == SPYRE_DT_BFLOAT16 || scalar_type == SPYRE_DT_FLOAT32,
                SPYRE_EUNSUPPORTED, "scalar type %d not float16, bfloat16 or float32", scalar_type);
  SPYRE_REQUIRE(position_bytes == 4 || position_bytes == 8, SPYRE_EINVAL, "positions of %d bytes", position_bytes);
  const int64_t tokens = static_cast<int64_t>(B) * S;
  if (tokens == 0 || Hq + Hkv == 0) return SPYRE_OK;
  SPYRE_REQUIRE(tokens < (int64_t{1} << 31), SPYRE_EUNSUPPORTED, "too many tokens");
  SPYRE_REQUIRE(positions && frequencies && (Hq == 0 || (q && q_out && q_strides && q_out_strides)) &&
                    (Hkv == 0 || (k && k_out && k_strides && k_out_strides)),
                SPYRE_EINVAL, "null pointer argument");
  RotaryArgs a{};
  bool vec = pairs % 8 == 0 && (D - 2 * pairs) % 8 == 0;
  auto operand = [&](int i, const void* x, const int64_t* xs, void* y, const int64_t* ys, int heads) {
    a.heads[i] = heads;
    if (!heads) return;
    a.o[i] = Operand{x, y, xs[0], xs[1], xs[2], ys[0], ys[1], ys[2]};
    for (int j = 0; j < 3; ++j) vec = vec && xs[j] % 8 == 0 && ys[j] % 8 == 0;
    vec = vec && reinterpret_cast<uintptr_t>(x) % 16 == 0 && reinterpret_cast<uintptr_t>(y) % 16 == 0;
  };
  operand(0, q, q_strides, q_out, q_out_strides, Hq);
  operand(1, k, k_strides, k_out, k_out_strides, Hkv);
  a.positions = positions, a.pb = pos_sb, a.ps = pos_ss, a.wide = position_bytes == 8;
  a.freq = frequencies, a.amplitude = amplitude, a.inverse = inverse != 0;
  a.S = S, a.D = D, a.half = pairs, a.tokens = tokens;
  a.turn_units = vec ? pairs / 8 : pairs;
  a.units = a.turn_units + (vec ? (D - 2 * pairs) / 8 : D - 2 * pairs);
  a.group = pairs >= kThreads ? 1 : kThreads / pairs;
  if (a.group > tokens) a.group = static_cast<int>(tokens);
  const int64_t groups = (tokens + a.group - 1) / a.group;
  // Slices of the heads while the groups alone leave compute units idle:
  // at least one item a thread.
  const int heads = Hq + Hkv;
  int slices = 1;
  while (slices < heads && groups * slices < 1024 &&
         static_cast<int64_t>(a.group) * (heads / (2 * slices)) * a.units >= kThreads)
    slices *= 2;
  a.head0_per_slice = (heads + slices - 1) / slices;
  slices = (heads + a.head0_per_slice - 1) / a.head0_per_slice;
  a.by_s = spyre_hip::make_fastdiv(static_cast<uint32_t>(S));
  a.by_units = spyre_hip::make_fastdiv(static_cast<uint32_t>(a.units));
  a.by_heads = spyre_hip::make_fastdiv(static_cast<uint32_t>(a.head0_per_slice));
  SPYRE_REQUIRE(static_cast<int64_t>(a.group) * a.head0_per_slice * a.units < (int64_t{1} << 31) && slices <= 65535,
                SPYRE_EUNSUPPORTED, "too many heads");
  const dim3 grid(static_cast<uint32_t>(groups), static_cast<uint32_t>(slices));
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (scalar_type == SPYRE_DT_FLOAT16)
    launch<_Float16>(a, vec, interleaved != 0, grid, st);
  else if (scalar_type == SPYRE_DT_BFLOAT16)
    launch<__bf16>(a, vec, interleaved != 0, grid, st);
  else
    launch<float>(a, vec, interleaved != 0, grid, st);
  const hipError_t e = hipGetLastError();
  SPYRE_REQUIRE(e == hipSuccess, SPYRE_EHIP, "rotary launch failed: %s", hipGetErrorString(e));
  return SPYRE_OK;
}
