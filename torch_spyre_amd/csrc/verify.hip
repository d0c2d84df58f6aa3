// Drafted tokens checked against the target's probabilities
// (spyre_verify_drafts).
//
// Sequence b has n[b] drafted tokens x_0 .. x_(n-1), the children of one another:
// parent[i] < i is the drafted token that x_i continues, -1 the context's last.
// Row r of the target's probabilities p_r is what it gives behind the context (r =
// 0) or behind x_(r-1).  From the context's end on, the children of the last
// accepted token are tried in their order; x_i, a child of token c, is accepted if
//   u_i q_i(x_i) < p_(c+1)(x_i)      the draft's probabilities q are given (a chain)
//   u_i left    < p_(c+1)(x_i)      else; left = 1 less the p of c's rejected children,
//                                    and a token that c has rejected has probability 0.
// Where no child is accepted one more token is drawn by u_T: the lowest j with
//   w_0 + ... + w_j > u_T (w_0 + ... + w_(V-1)),
// w = max(p - q, 0) behind a rejection by q, else p without the rejected tokens;
// w = p if that has no weight at all.  A probability that is negative, NaN or
// infinite counts as 0.  Tests and sums are in 64 bits: a sum in 32 is off by as much
// as the p of a rare token, and the token drawn next to a border would change.
//
// A workgroup has runs of kRun tokens of one sequence: it walks the drafts (a few loads
// at once, then one a lane), sums its runs and leaves the sums with an arrival flag.
// A workgroup that finds all flags finds the run and then the token where the sums pass
// the limit: one launch, and no row is read twice but for that run.  What bounds it: one
// row of the vocabulary a sequence (two with q), and for few sequences the chain of
// loads.  Measured: 64 x 128000 fp32 tokens with q 22 us (65 MB, 3 TB/s, by loads of 4 bytes a
// lane; wider ones were not tried), 1 x 32000 11 us, trees of 25 over 16 x 100003 bf16 14 us.

#include <hip/hip_runtime.h>

#include <algorithm>

#include "decode_dense.h"
#include "spyre_common.h"

namespace {

using namespace spyre_hip;

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kEach = 8;                // tokens of a thread, its loads in flight at once
constexpr int kRun = kThreads * kEach;  // of a workgroup at a time
constexpr int kMostRuns = 8;            // of a workgroup
constexpr int kMaxDrafts = 1024;        // drafted tokens in LDS

struct VerifyArgs {
  const void* tokens;  // int32 or int64
  int token_bytes;
  int64_t t_sb, t_st;
  const void *target, *draft;
  int64_t p_sb, p_sr, q_sb, q_sr;
  const float* u;
  int64_t u_sb, u_st;
  const int32_t* parents;
  int64_t pa_sb, pa_st;
  const int32_t* lens;
  void* out;  // of the tokens' type
  int32_t *accepted, *path;
  double* sums;     // [B][runs][2]: of w, of p
  uint32_t* flags;  // [B][groups]
  int B, T, V, runs, per, groups;  // per: runs of a workgroup
  uint32_t ticket;
};

template <typename E>
__device__ __forceinline__ auto row_of(const E* p, int n) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<E*>(p), 0, n * static_cast<int>(sizeof(E)), 0x00020000);
}

// Numbered as SPYRE_DT_*.
template <int DT>
struct Elem;
template <>
struct Elem<SPYRE_DT_FLOAT32> {
  typedef float type;
  __device__ static float f32(float x) { return x; }
  __device__ static float load(__amdgpu_buffer_rsrc_t r, int i) {
    return __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(r, 4 * i, 0, 0));
  }
};
template <>
struct Elem<SPYRE_DT_FLOAT16> {
  typedef _Float16 type;
  __device__ static float f32(_Float16 x) { return static_cast<float>(x); }
  __device__ static float load(__amdgpu_buffer_rsrc_t r, int i) {
    return f32(__builtin_bit_cast(_Float16, __builtin_amdgcn_raw_buffer_load_b16(r, 2 * i, 0, 0)));
  }
};
template <>
struct Elem<SPYRE_DT_BFLOAT16> {
  typedef uint16_t type;
  __device__ static float f32(uint16_t x) { return __builtin_bit_cast(float, static_cast<uint32_t>(x) << 16); }
  __device__ static float load(__amdgpu_buffer_rsrc_t r, int i) {
    return f32(static_cast<uint16_t>(__builtin_amdgcn_raw_buffer_load_b16(r, 2 * i, 0, 0)));
  }
};

template <typename T>
__device__ __forceinline__ T weight(T x) { return x > 0 && x < static_cast<T>(INFINITY) ? x : T{0}; }

// Exclusive sums over a wavefront's lanes; total: of all.
__device__ __forceinline__ double scan_lanes(double x, double& total) {
  double y = x;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const double z = __shfl_up(y, d, 64);
    if (static_cast<int>(threadIdx.x % 64) >= d) y += z;
  }
  total = __shfl(y, 63, 64);
  const double z = __shfl_up(y, 1, 64);
  return threadIdx.x % 64 ? z : 0.0;
}

__device__ __forceinline__ double sum_lanes(double x) {
#pragma unroll
  for (int d = 32; d; d /= 2) x += __shfl_xor(x, d, 64);
  return x;
}

// The words of LDS that T drafts take.
constexpr int kArrays = 7;

template <int DT>
__global__ __launch_bounds__(kThreads, 8) void verify_kernel(VerifyArgs a) {
  typedef typename Elem<DT>::type E;
  extern __shared__ int s_drafts[];
  int *s_tok = s_drafts, *s_par = s_tok + a.T, *s_ref = s_par + a.T, *s_path = s_ref + a.T;
  float *s_p = reinterpret_cast<float*>(s_path + a.T), *s_q = s_p + a.T, *s_u = s_q + a.T;
  __shared__ uint32_t s_gone[kMostRuns * kRun / 32];  // of the runs, the tokens that were rejected
  __shared__ int s_last, s_refused, s_accepted, s_all, s_found, s_token;
  __shared__ double s_sum[kMostRuns][2][kWaves], s_limit, s_before;
  const int b = blockIdx.y, group = blockIdx.x, lane = threadIdx.x % 64;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const E* target = static_cast<const E*>(a.target) + b * a.p_sb;
  const E* draft = static_cast<const E*>(a.draft) + b * a.q_sb;
  const int given = a.lens ? a.lens[b] : a.T;
  const float u_last = a.u[b * a.u_sb + a.T * a.u_st];

  for (int i = threadIdx.x; i < a.T; i += kThreads) {
    const int64_t at = b * a.t_sb + i * a.t_st;
    const int64_t x = a.token_bytes == 8 ? static_cast<const int64_t*>(a.tokens)[at] : static_cast<const int32_t*>(a.tokens)[at];
    const int parent = a.parents ? a.parents[b * a.pa_sb + i * a.pa_st] : i - 1;
    const bool known = x >= 0 && x < a.V, child = parent >= -1 && parent < i;
    s_tok[i] = known ? static_cast<int>(x) : -1;
    s_par[i] = child ? parent : -2;
    s_p[i] = known && child ? weight(Elem<DT>::f32(target[(parent + 1) * a.p_sr + x])) : 0.f;
    s_q[i] = known && a.draft ? weight(Elem<DT>::f32(draft[i * a.q_sr + x])) : 0.f;
    s_u[i] = a.u[b * a.u_sb + i * a.u_st];
  }
  for (int k = threadIdx.x; k < kMostRuns * kRun / 32; k += kThreads) s_gone[k] = 0;
  __syncthreads();
  if (wave == 0) {
    // 64 drafts at a time, one a lane; only children of the last accepted one are looked at.
    const int n = min(max(given, 0), a.T);
    int last = -1, refused = 0, accepted = 0;
    int ref = -1;  // lane k: the k-th rejected token (those from 64 on are in LDS only)
    double left = 1.0;
    for (int c = 0; c < n; c += 64) {
      const int i = min(c + lane, n - 1), par = c + lane < n ? s_par[i] : -2, tok = s_tok[i];
      const double p = s_p[i], u = s_u[i], uq = u * static_cast<double>(s_q[i]);
      for (uint64_t children = __ballot(par == last); children != 0;) {
        const int k = __builtin_ctzll(children);
        children &= children - 1;
        const int x = __shfl(tok, k, 64);
        bool again = lane < refused && ref == x;
        for (int r = 64 + lane; r < refused; r += 64) again = again || s_tok[s_ref[r]] == x;
        const double px = __any(again) ? 0.0 : __shfl(p, k, 64);
        if ((a.draft ? __shfl(uq, k, 64) : __shfl(u, k, 64) * left) < px) {
          if (lane == 0) s_path[accepted] = c + k;
          last = c + k, refused = 0, left = 1.0, ++accepted;
          children = __ballot(par == last);  // they come behind it
        } else {
          if (lane == 0) s_ref[refused] = c + k;
          if (lane == refused) ref = x;
          ++refused, left -= px;
        }
      }
    }
    if (lane == 0) s_last = last, s_refused = refused, s_accepted = accepted;
  }
  __syncthreads();
  const int last = __builtin_amdgcn_readfirstlane(s_last), refused = __builtin_amdgcn_readfirstlane(s_refused);
  const E* p_row = target + (last + 1) * a.p_sr;
  const bool minus_q = a.draft && refused;
  const E* q_row = minus_q ? draft + __builtin_amdgcn_readfirstlane(s_ref[0]) * a.q_sr : nullptr;

  // Marks the rejected ones of `tokens` tokens; the workgroup waits for them.
  auto mark = [&](int first, int tokens) {
    if (minus_q || !refused) return;
    for (int k = threadIdx.x; k < refused; k += kThreads) {
      const int x = s_tok[s_ref[k]] - first;
      if (x >= 0 && x < tokens) atomicOr(&s_gone[x / 32], 1u << (x % 32));
    }
    __syncthreads();
  };
  // A thread's tokens of a run: first + from + k step.  Behind the row's end there are zeros.
  auto load = [&](int first, int from, int step, float (&x)[kEach], float (&y)[kEach]) {
    const auto row_p = row_of(p_row + first, min(a.V - first, kRun)), row_q = row_of(q_row + first, min(a.V - first, kRun));
#pragma unroll
    for (int k = 0; k < kEach; ++k) x[k] = Elem<DT>::load(row_p, from + k * step);
#pragma unroll
    for (int k = 0; k < kEach; ++k) y[k] = minus_q ? Elem<DT>::load(row_q, from + k * step) : 0.f;
  };
  auto w_of = [&](int at, double p, float y) {
    const bool gone = (s_gone[at / 32] >> (at % 32)) & 1;
    return gone ? 0.0 : minus_q ? weight(p - static_cast<double>(weight(y))) : p;
  };

  float x[kEach], y[kEach];
  const int run0 = group * a.per, runs = min(a.per, a.runs - run0);
  mark(run0 * kRun, runs * kRun);
  for (int r = 0; r < runs; ++r) {
    load((run0 + r) * kRun, threadIdx.x, kThreads, x, y);
    double sw = 0.0, sp = 0.0;
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      const double p = static_cast<double>(weight(x[k]));
      sw += w_of(r * kRun + k * kThreads + threadIdx.x, p, y[k]), sp += p;
    }
    sw = sum_lanes(sw), sp = sum_lanes(sp);
    if (lane == 0) s_sum[r][0][wave] = sw, s_sum[r][1][wave] = sp;
  }
  __syncthreads();
  double* sums = a.sums + static_cast<int64_t>(b) * a.runs * 2;
  uint32_t* flags = a.flags + static_cast<int64_t>(b) * a.groups;
  // The sums and then the flag go past the caches of this XCD; of two workgroups the
  // one whose flag was stored later sees the other's, so at least one sees them all.
  if (wave == 0) {
    if (lane < 2 * runs) {
      double t = 0.0;
      for (int v = 0; v < kWaves; ++v) t += s_sum[lane / 2][lane % 2][v];
      __hip_atomic_store(sums + run0 * 2 + lane, t, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (lane == 0) __hip_atomic_store(flags + group, a.ticket, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    bool seen = true;
    for (int r = lane; r < a.groups; r += 64)
      seen = seen && __hip_atomic_load(flags + r, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == a.ticket;
    const bool every = __all(seen);
    if (lane == 0) s_all = every ? 1 : 0;
  }
  __syncthreads();
  if (!s_all) return;

  // The run where the sums pass the limit.
  if (wave == 0) {
    auto of = [&](int r, int c) {
      return r < a.runs ? __hip_atomic_load(sums + r * 2 + c, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0.0;
    };
    const double held[2] = {of(lane, 0), of(lane, 1)};  // of the first 64 runs
    double total = 0.0;
    int c = 0;
    for (; c < 2; ++c) {  // 0: of w; 1: of p, where w has none
      total = sum_lanes(c ? held[1] : held[0]);
      for (int r = 64; r < a.runs; r += 64) total += sum_lanes(of(r + lane, c));
      if (total > 0.0) break;
    }
    const double limit = total * fmax(static_cast<double>(u_last), 0.0);
    int found = -1, some = -1;  // the run; the last one with any weight
    double before = 0.0, at = 0.0, some_at = 0.0;
    for (int r = 0; r < a.runs && found < 0 && total > 0.0; r += 64) {
      double t;
      const double z = r ? of(r + lane, c) : c ? held[1] : held[0], e = before + scan_lanes(z, t);
      const uint64_t past = __ballot(z > 0.0 && e + z > limit), any = __ballot(z > 0.0);
      if (past) found = r + __builtin_ctzll(past), at = __shfl(e, __builtin_ctzll(past), 64);
      if (any) some = r + 63 - __builtin_clzll(any), some_at = __shfl(e, 63 - __builtin_clzll(any), 64);
      before += t;
    }
    if (found < 0) found = some, at = some_at;  // a limit at the total
    if (lane == 0) s_found = total > 0.0 ? found * 2 + (c == 1) : -1, s_limit = limit, s_before = at;
  }
  if (threadIdx.x < kRun / 32) s_gone[threadIdx.x] = 0;
  if (threadIdx.x == 0) s_token = -1;
  __syncthreads();
  if (s_found >= 0) {
    // The token in it: a thread has kEach that follow one another.
    const int first = (s_found >> 1) * kRun, from = kEach * threadIdx.x;
    const bool plain = s_found & 1;
    load(first, from, 1, x, y);
    mark(first, kRun);
    double w = 0.0;
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      const double p = static_cast<double>(weight(x[k]));
      w += plain ? p : w_of(from + k, p, y[k]);
    }
    double t;
    double e = scan_lanes(w, t);
    if (lane == 0) s_sum[0][0][wave] = t;
    __syncthreads();
    e += s_before;
    for (int v = 0; v < wave; ++v) e += s_sum[0][0][v];
    const uint64_t past = __ballot(w > 0.0 && e + w > s_limit), any = __ballot(w > 0.0);
    // The first wavefront that passes; the last one with any weight if none does.
    if (lane == 0) s_sum[0][1][wave] = past ? 2.0 : any ? 1.0 : 0.0;
    __syncthreads();
    int of = -1;
    for (int v = kWaves - 1; v >= 0; --v)
      if (s_sum[0][1][v] == 2.0 || (s_sum[0][1][v] == 1.0 && of < 0)) of = v;
    if (wave == of && lane == (past ? __builtin_ctzll(past) : 63 - __builtin_clzll(any))) {
      int some = 0;
      for (int k = 0; k < kEach; ++k) {
        const double p = static_cast<double>(weight(x[k])), one = plain ? p : w_of(from + k, p, y[k]);
        if (!(one > 0.0)) continue;
        some = k, e += one;
        if (e > s_limit) break;
      }
      s_token = first + from + some;
    }
    __syncthreads();
  }
  const int accepted = s_accepted, token = s_token;
  const int64_t row = static_cast<int64_t>(b) * (a.T + 1);
  for (int i = threadIdx.x; i <= a.T; i += kThreads) {
    const int64_t z = i < accepted ? s_tok[s_path[i]] : i == accepted ? token : -1;
    if (a.token_bytes == 8)
      static_cast<int64_t*>(a.out)[row + i] = z;
    else
      static_cast<int32_t*>(a.out)[row + i] = static_cast<int32_t>(z);
    if (i < a.T) a.path[static_cast<int64_t>(b) * a.T + i] = i < accepted ? s_path[i] : -1;
  }
  if (threadIdx.x == 0) a.accepted[b] = accepted;
  // So that a replayed call (the same ticket) starts with none.
  for (int r = threadIdx.x; r < a.groups; r += kThreads) __hip_atomic_store(flags + r, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

constexpr int kEnough = 1024;  // workgroups: 4 to a CU

int runs_of(int V) { return static_cast<int>((static_cast<int64_t>(V) + kRun - 1) / kRun); }

}  // namespace

extern "C" size_t spyre_verify_drafts_workspace_bytes(int B, int V) {
  return B > 0 && V > 0 ? static_cast<size_t>(B) * runs_of(V) * 20 : 0;
}

extern "C" int spyre_verify_drafts(const void* tokens, int token_bytes, int64_t tok_sb, int64_t tok_st, const void* target,
                                   const int64_t* target_strides, const void* draft, const int64_t* draft_strides,
                                   int scalar_type, const float* uniforms, int64_t u_sb, int64_t u_st, const int32_t* parents,
                                   int64_t par_sb, int64_t par_st, const int32_t* draft_lens, void* out_tokens,
                                   int32_t* accepted, int32_t* path, void* workspace, size_t workspace_bytes, int B, int T, int V,
                                   void* stream) {
  spyre_hip::clear_error();
  SPYRE_REQUIRE(B >= 0 && T >= 0 && V > 0, SPYRE_EINVAL, "bad sizes B=%d T=%d V=%d", B, T, V);
  SPYRE_REQUIRE(token_bytes == 4 || token_bytes == 8, SPYRE_EINVAL, "tokens must be int32 or int64");
  SPYRE_REQUIRE(scalar_type == SPYRE_DT_FLOAT32 || scalar_type == SPYRE_DT_FLOAT16 || scalar_type == SPYRE_DT_BFLOAT16,
                SPYRE_EUNSUPPORTED, "probabilities of type %d", scalar_type);
  SPYRE_REQUIRE(!(draft && parents), SPYRE_EUNSUPPORTED, "draft probabilities of a tree");
  SPYRE_REQUIRE(T <= kMaxDrafts, SPYRE_EUNSUPPORTED, "%d drafted tokens, at most %d", T, kMaxDrafts);
  SPYRE_REQUIRE(B < 65536, SPYRE_EUNSUPPORTED, "%d sequences, at most 65535", B);
  SPYRE_REQUIRE(V < (1 << 30), SPYRE_EUNSUPPORTED, "too many tokens in the vocabulary");
  if (B == 0) return SPYRE_OK;
  SPYRE_REQUIRE((tokens || T == 0) && target && target_strides && (!draft || draft_strides) && uniforms && out_tokens && accepted &&
                    (path || T == 0),
                SPYRE_EINVAL, "null pointer argument");
  const size_t need = spyre_verify_drafts_workspace_bytes(B, V);
  SPYRE_REQUIRE(workspace && workspace_bytes >= need && reinterpret_cast<uintptr_t>(workspace) % 16 == 0, SPYRE_ENOSPC,
                "workspace holds %zu bytes, need %zu (16-byte aligned)", workspace ? workspace_bytes : 0, need);
  VerifyArgs a{};
  a.tokens = tokens, a.token_bytes = token_bytes, a.t_sb = tok_sb, a.t_st = tok_st;
  a.target = target, a.p_sb = target_strides[0], a.p_sr = target_strides[1];
  a.draft = draft;
  if (draft) a.q_sb = draft_strides[0], a.q_sr = draft_strides[1];
  a.u = uniforms, a.u_sb = u_sb, a.u_st = u_st;
  a.parents = parents, a.pa_sb = par_sb, a.pa_st = par_st, a.lens = draft_lens;
  a.out = out_tokens, a.accepted = accepted, a.path = path;
  a.B = B, a.T = T, a.V = V, a.runs = runs_of(V);
  // Every workgroup walks the drafts before its first load: 64 x 128000 tokens 32 us with a run
  // to each, 23.5 with 2, 22 with 4.  Few sequences have more workgroups instead.
  a.per = static_cast<int>(std::min<int64_t>((static_cast<int64_t>(B) * a.runs + kEnough - 1) / kEnough, kMostRuns));
  a.groups = (a.runs + a.per - 1) / a.per;
  a.sums = static_cast<double*>(workspace);
  a.flags = reinterpret_cast<uint32_t*>(a.sums + static_cast<int64_t>(B) * a.runs * 2);
  a.ticket = spyre_hip::next_call_ticket();
  const dim3 grid(static_cast<uint32_t>(a.groups), static_cast<uint32_t>(B));
  const size_t lds = static_cast<size_t>(T) * kArrays * 4;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (scalar_type == SPYRE_DT_FLOAT32)
    verify_kernel<SPYRE_DT_FLOAT32><<<grid, kThreads, lds, st>>>(a);
  else if (scalar_type == SPYRE_DT_FLOAT16)
    verify_kernel<SPYRE_DT_FLOAT16><<<grid, kThreads, lds, st>>>(a);
  else
    verify_kernel<SPYRE_DT_BFLOAT16><<<grid, kThreads, lds, st>>>(a);
  const hipError_t e = hipGetLastError();
  SPYRE_REQUIRE(e == hipSuccess, SPYRE_EHIP, "draft verification launch failed: %s", hipGetErrorString(e));
  return SPYRE_OK;
}
