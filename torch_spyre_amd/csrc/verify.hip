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
// A workgroup has one run of kRun tokens of one sequence: it walks the drafts (a few
// loads at once, then a loop in LDS), sums its run and leaves the sum with an arrival
// flag.  A workgroup that finds the flags of all runs finds the run and then the token
// where the sums pass the limit: one launch, and no row is read twice but for that
// run.  What bounds it: one row of the vocabulary a sequence (two with q), or for few
// sequences the chain of loads.

#include <hip/hip_runtime.h>

#include "decode_dense.h"
#include "spyre_common.h"

namespace {

using namespace spyre_hip;

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kEach = 16;               // tokens of a thread
constexpr int kRun = kThreads * kEach;  // of a workgroup
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
  uint32_t* flags;  // [B][runs]
  int B, T, V, runs;
  uint32_t ticket;
};

// Numbered as SPYRE_DT_*.
template <int DT>
struct Elem;
template <>
struct Elem<SPYRE_DT_FLOAT32> {
  typedef float type;
  __device__ static float f32(float x) { return x; }
};
template <>
struct Elem<SPYRE_DT_FLOAT16> {
  typedef _Float16 type;
  __device__ static float f32(_Float16 x) { return static_cast<float>(x); }
};
template <>
struct Elem<SPYRE_DT_BFLOAT16> {
  typedef uint16_t type;
  __device__ static float f32(uint16_t x) { return __builtin_bit_cast(float, static_cast<uint32_t>(x) << 16); }
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

template <int DT>
__global__ __launch_bounds__(kThreads) void verify_kernel(VerifyArgs a) {
  typedef typename Elem<DT>::type E;
  __shared__ int s_tok[kMaxDrafts], s_par[kMaxDrafts], s_ref[kMaxDrafts], s_path[kMaxDrafts];
  __shared__ float s_p[kMaxDrafts], s_q[kMaxDrafts], s_u[kMaxDrafts];
  __shared__ uint32_t s_gone[kRun / 32];  // of the run, the tokens that were rejected
  __shared__ int s_last, s_refused, s_accepted, s_all, s_found;
  __shared__ double s_sum[2][kEach * kWaves], s_limit, s_before;
  const int b = blockIdx.y, run = blockIdx.x, lane = threadIdx.x % 64;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const E* target = static_cast<const E*>(a.target) + b * a.p_sb;
  const E* draft = static_cast<const E*>(a.draft) + b * a.q_sb;
  const int n = a.lens ? min(max(a.lens[b], 0), a.T) : a.T;

  for (int i = threadIdx.x; i < n; i += kThreads) {
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
  if (threadIdx.x < kRun / 32) s_gone[threadIdx.x] = 0;
  __syncthreads();
  if (wave == 0) {
    int last = -1, refused = 0, accepted = 0;
    double left = 1.0;
    for (int i = 0; i < n; ++i) {
      if (s_par[i] != last) continue;
      const int x = s_tok[i];
      bool again = false;
      for (int k = lane; k < refused; k += 64) again = again || s_tok[s_ref[k]] == x;
      const double p = __any(again) ? 0.0 : static_cast<double>(s_p[i]);
      if (static_cast<double>(s_u[i]) * (a.draft ? static_cast<double>(s_q[i]) : left) < p) {
        if (lane == 0) s_path[accepted] = i;
        last = i, refused = 0, left = 1.0, ++accepted;
      } else {
        if (lane == 0) s_ref[refused] = i;
        ++refused, left -= p;
      }
    }
    if (lane == 0) s_last = last, s_refused = refused, s_accepted = accepted;
  }
  __syncthreads();
  const int last = s_last, refused = s_refused;
  const E* p_row = target + (last + 1) * a.p_sr;
  const bool minus_q = a.draft && refused;
  const E* q_row = minus_q ? draft + s_ref[0] * a.q_sr : nullptr;

  // Marks the rejected tokens of a run; the workgroup waits for them.
  auto mark = [&](int first) {
    if (!minus_q)
      for (int k = threadIdx.x; k < refused; k += kThreads) {
        const int x = s_tok[s_ref[k]] - first;
        if (x >= 0 && x < kRun) atomicOr(&s_gone[x / 32], 1u << (x % 32));
      }
    __syncthreads();
  };
  // A thread's tokens of a run: first + 256 k + its number.
  auto weights = [&](int first, double (&w)[kEach], double (&p)[kEach]) {
    float x[kEach], y[kEach];
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      const int j = min(first + k * kThreads + static_cast<int>(threadIdx.x), a.V - 1);
      x[k] = Elem<DT>::f32(p_row[j]);
      y[k] = minus_q ? Elem<DT>::f32(q_row[j]) : 0.f;
    }
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      const int at = k * kThreads + threadIdx.x;
      const bool there = first + at < a.V, gone = (s_gone[at / 32] >> (at % 32)) & 1;
      p[k] = there ? static_cast<double>(weight(x[k])) : 0.0;
      w[k] = gone ? 0.0 : minus_q ? weight(p[k] - static_cast<double>(weight(y[k]))) : p[k];
    }
  };

  double w[kEach], p[kEach];
  mark(run * kRun);
  weights(run * kRun, w, p);
  double sw = 0.0, sp = 0.0;
#pragma unroll
  for (int k = 0; k < kEach; ++k) sw += w[k], sp += p[k];
  sw = sum_lanes(sw), sp = sum_lanes(sp);
  if (lane == 0) s_sum[0][wave] = sw, s_sum[1][wave] = sp;
  __syncthreads();
  double* sums = a.sums + static_cast<int64_t>(b) * a.runs * 2;
  uint32_t* flags = a.flags + static_cast<int64_t>(b) * a.runs;
  // The sums and then the flag go past the caches of this XCD; of two workgroups the
  // one whose flag was stored later sees the other's, so at least one sees them all.
  if (wave == 0) {
    if (lane == 0) {
      double t[2] = {0.0, 0.0};
      for (int v = 0; v < kWaves; ++v) t[0] += s_sum[0][v], t[1] += s_sum[1][v];
      for (int c = 0; c < 2; ++c) __hip_atomic_store(sums + run * 2 + c, t[c], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __hip_atomic_store(flags + run, a.ticket, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    bool seen = true;
    for (int r = lane; r < a.runs; r += 64)
      seen = seen && __hip_atomic_load(flags + r, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == a.ticket;
    const bool all = __all(seen);
    if (lane == 0) s_all = all ? 1 : 0;
  }
  __syncthreads();
  if (!s_all) return;

  // The run where the sums pass the limit.
  if (wave == 0) {
    auto of = [&](int r, int c) {
      return r < a.runs ? __hip_atomic_load(sums + r * 2 + c, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0.0;
    };
    double total = 0.0;
    int c = 0;
    for (; c < 2; ++c) {  // 0: of w; 1: of p, where w has none
      total = 0.0;
      for (int r = 0; r < a.runs; r += 64) {
        double t;
        scan_lanes(of(r + lane, c), t);
        total += t;
      }
      if (total > 0.0) break;
    }
    const double limit = total * fmax(static_cast<double>(a.u[b * a.u_sb + a.T * a.u_st]), 0.0);
    int found = -1, some = -1;  // the run; the last one with any weight
    double before = 0.0, at = 0.0, some_at = 0.0;
    for (int r = 0; r < a.runs && found < 0 && total > 0.0; r += 64) {
      double t;
      const double x = of(r + lane, c), e = before + scan_lanes(x, t);
      const uint64_t past = __ballot(x > 0.0 && e + x > limit), any = __ballot(x > 0.0);
      if (past) found = r + __builtin_ctzll(past), at = __shfl(e, __builtin_ctzll(past), 64);
      if (any) some = r + 63 - __builtin_clzll(any), some_at = __shfl(e, 63 - __builtin_clzll(any), 64);
      before += t;
    }
    if (found < 0) found = some, at = some_at;  // a limit at the total
    if (lane == 0) s_found = found * 2 + (c == 1), s_limit = limit, s_before = at;
    if (total <= 0.0 && lane == 0) s_found = -1;
  }
  if (threadIdx.x < kRun / 32) s_gone[threadIdx.x] = 0;
  __syncthreads();
  int64_t token = -1;
  if (s_found >= 0) {
    // The token in it: sums of 64 tokens, then of one.
    const int first = (s_found >> 1) * kRun;
    const bool plain = s_found & 1;
    mark(first);
    weights(first, w, p);
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      if (plain) w[k] = p[k];
      const double t = sum_lanes(w[k]);
      if (lane == 0) s_sum[0][k * kWaves + wave] = t;
    }
    __syncthreads();
    double t;
    static_assert(kEach * kWaves == 64, "one sum a lane");
    const double x = s_sum[0][lane], e = s_before + scan_lanes(x, t);
    const uint64_t past = __ballot(x > 0.0 && e + x > s_limit), any = __ballot(x > 0.0);
    const int group = past ? __builtin_ctzll(past) : any ? 63 - __builtin_clzll(any) : 0;
    const double base = __shfl(e, group, 64);
    int mine = -1;
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      if (k * kWaves + wave != group) continue;
      const double y = base + scan_lanes(w[k], t) + w[k];
      const uint64_t over = __ballot(w[k] > 0.0 && y > s_limit), some = __ballot(w[k] > 0.0);
      mine = first + group * 64 + (over ? __builtin_ctzll(over) : some ? 63 - __builtin_clzll(some) : 0);
    }
    __syncthreads();
    if (mine >= 0 && lane == 0) s_found = mine;
    __syncthreads();
    token = s_found;
  }
  const int accepted = s_accepted;
  const int64_t row = static_cast<int64_t>(b) * (a.T + 1);
  for (int i = threadIdx.x; i <= a.T; i += kThreads) {
    const int64_t x = i < accepted ? s_tok[s_path[i]] : i == accepted ? token : -1;
    if (a.token_bytes == 8)
      static_cast<int64_t*>(a.out)[row + i] = x;
    else
      static_cast<int32_t*>(a.out)[row + i] = static_cast<int32_t>(x);
    if (i < a.T) a.path[static_cast<int64_t>(b) * a.T + i] = i < accepted ? s_path[i] : -1;
  }
  if (threadIdx.x == 0) a.accepted[b] = accepted;
  // So that a replayed call (the same ticket) starts with none.
  for (int r = threadIdx.x; r < a.runs; r += kThreads) __hip_atomic_store(flags + r, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

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
  a.sums = static_cast<double*>(workspace);
  a.flags = reinterpret_cast<uint32_t*>(a.sums + static_cast<int64_t>(B) * a.runs * 2);
  a.ticket = spyre_hip::next_call_ticket();
  const dim3 grid(static_cast<uint32_t>(a.runs), static_cast<uint32_t>(B));
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (scalar_type == SPYRE_DT_FLOAT32)
    verify_kernel<SPYRE_DT_FLOAT32><<<grid, kThreads, 0, st>>>(a);
  else if (scalar_type == SPYRE_DT_FLOAT16)
    verify_kernel<SPYRE_DT_FLOAT16><<<grid, kThreads, 0, st>>>(a);
  else
    verify_kernel<SPYRE_DT_BFLOAT16><<<grid, kThreads, 0, st>>>(a);
  const hipError_t e = hipGetLastError();
  SPYRE_REQUIRE(e == hipSuccess, SPYRE_EHIP, "draft verification launch failed: %s", hipGetErrorString(e));
  return SPYRE_OK;
}
