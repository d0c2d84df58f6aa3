// Block tables and slot maps from the sequences' lengths (spyre_plan_pages), and
// pages given back (spyre_release_pages).
//
// Sequence b holds the first held[b] pages of its row of the block table.  With
// ctx[b] cached and new[b] further tokens it needs
//   need[b] = max(min(ceil((ctx[b] + new[b]) / 64), pages_per_seq) - held[b], 0)
// more.  Free pages lie in a ring of F entries between two counters that only
// grow, taken and returned; page i of sequence b is
//   ring[(taken + first[b] + i) mod F],   first[b] = need[0] + ... + need[b - 1]
// as long as taken + first[b] + i < returned.  Token t of b goes to position
// p = ctx[b] + t, slot 64 page(b, p / 64) + p mod 64.
// Nothing that a call reads is written by it (fresh entries of the table lie
// behind those that it reads), so a call is one launch: every workgroup sums the
// sequences for itself and takes its share of the tokens and of the pages.
// What bounds it: latency (lengths, sums, a table entry, a store).  Measured: 64 sequences x
// 25 tokens 3.7 us, their pages back 2.9; 256 prompts of 128 to 8192 tokens 10.5 (13 MB, 2.6 at
// a copy's rate): the sums of all lengths, and then for each token the sequence's lengths again before
// its table or ring entry, four rounds of them to a thread.

#include <hip/hip_runtime.h>

#include <algorithm>

#include "fast_div.h"
#include "page_walk.h"
#include "spyre_common.h"

namespace {

using namespace spyre_hip;

constexpr int kThreads = 256;
constexpr int kMaxSeqs = 4096;  // sums of all sequences in LDS: 8 + 4 bytes each

struct PagesArgs {
  int32_t* bt;
  int64_t bt_stride;
  int W;  // pages a sequence
  const int32_t *held, *ctx, *lens;  // lens: new tokens; of a release, tokens kept
  int32_t* ring;
  int64_t F;
  const int64_t* cursor;
  int32_t *held_out, *starts;
  int64_t* cursor_out;
  int32_t* positions;
  int64_t* slots;
  int64_t rows;  // of positions and slots
  int B, length;
  FastDiv by_length;
};

__device__ __forceinline__ int64_t nonneg(int x) { return x > 0 ? x : 0; }

__device__ __forceinline__ int held_of(const PagesArgs& a, int b) { return min(max(a.held[b], 0), a.W); }

// Pages that a row holds for n tokens, if the table were filled.
__device__ __forceinline__ int pages_for(const PagesArgs& a, int64_t n) {
  return static_cast<int>(min((n + kPage - 1) / kPage, static_cast<int64_t>(a.W)));
}

template <typename T>
__device__ __forceinline__ T shuffled_up(T x, int by) { return __shfl_up(x, by, 64); }

// Exclusive sums of x over the workgroup; total: of all.  s_wave: kThreads / 64.
template <typename T>
__device__ __forceinline__ T scan_group(T x, T* s_wave, T& total) {
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  T y = x;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const T z = shuffled_up(y, d);
    y += lane >= d ? z : 0;
  }
  __syncthreads();  // s_wave of the sums before these is read
  if (lane == 63) s_wave[wave] = y;
  __syncthreads();
  T before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) {
    before += w < wave ? s_wave[w] : 0;
    total += s_wave[w];
  }
  return before + y - x;
}

// The last of n ascending sums that is not above x (the first is 0).
template <typename T>
__device__ __forceinline__ int last_not_above(const T* sums, int n, T x) {
  int lo = 0, hi = n;  // sums[lo] <= x, hi == n or sums[hi] > x
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (sums[mid] <= x)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

// first[b] and (starts != null) the tokens before each sequence, of all.
template <bool RELEASE>
__device__ __forceinline__ void sums_of(const PagesArgs& a, int32_t* first, int64_t* starts, int64_t& pages, int64_t& tokens) {
  __shared__ int64_t s_wave[2][kThreads / 64];
  pages = tokens = 0;
  for (int c = 0; c < a.B; c += kThreads) {
    const int b = c + threadIdx.x;
    int64_t need = 0, n = 0;
    if (b < a.B) {
      const int held = held_of(a, b);
      n = nonneg(a.lens[b]);
      need = RELEASE ? held - min(held, pages_for(a, n)) : max(pages_for(a, nonneg(a.ctx[b]) + n) - held, 0);
    }
    int64_t total;
    const int64_t f = scan_group(need, s_wave[0], total);
    if (b < a.B) first[b] = static_cast<int32_t>(pages + f);
    pages += total;
    if (starts) {
      const int64_t s = scan_group(n, s_wave[1], total);
      if (b < a.B) starts[b] = tokens + s;
      tokens += total;
    }
  }
  __syncthreads();
}

template <bool PACKED>
__global__ __launch_bounds__(kThreads) void plan_pages_kernel(PagesArgs a) {
  extern __shared__ int64_t s_mem[];
  int64_t* starts = PACKED ? s_mem : nullptr;
  int32_t* first = reinterpret_cast<int32_t*>(s_mem + (PACKED ? a.B : 0));
  const int64_t taken = a.cursor[0], returned = a.cursor[1];
  int64_t pages, tokens;
  sums_of<false>(a, first, starts, pages, tokens);
  const int64_t left = min(max(returned - taken, int64_t{0}), a.F);
  const int64_t got = min(pages, left);  // of all
  const int64_t base = a.F ? (taken % a.F + a.F) % a.F : 0;
  auto fresh = [&](int64_t k) { return a.ring[base + k < a.F ? base + k : base + k - a.F]; };
  const int64_t id = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x, step = static_cast<int64_t>(gridDim.x) * kThreads;

  for (int64_t k = id; k < got; k += step) {
    const int b = last_not_above(first, a.B, static_cast<int32_t>(k));
    a.bt[b * a.bt_stride + held_of(a, b) + k - first[b]] = fresh(k);
  }
  for (int64_t r = id; r < a.rows; r += step) {
    int b;
    int64_t t;
    bool live;
    if (PACKED) {
      live = r < tokens;
      b = live ? last_not_above(starts, a.B, r) : 0;
      t = live ? r - starts[b] : 0;
    } else {
      b = static_cast<int>(fdiv(static_cast<uint32_t>(r), a.by_length));
      t = r - static_cast<int64_t>(b) * a.length;
      live = t < a.lens[b];
    }
    int64_t p = -1, slot = -1;
    if (live) {
      p = nonneg(a.ctx[b]) + t;
      const int64_t page = p / kPage;
      const int held = held_of(a, b);
      int64_t phys = -1;
      if (page < held)
        phys = a.bt[b * a.bt_stride + page];
      else if (page < a.W && first[b] + page - held < got)
        phys = fresh(first[b] + page - held);
      if (phys >= 0) slot = phys * kPage + p % kPage;
    }
    a.positions[r] = static_cast<int32_t>(p);
    a.slots[r] = slot;
  }
  if (blockIdx.x) return;
  for (int b = threadIdx.x; b < a.B; b += kThreads) {
    const int held = held_of(a, b);
    const int64_t need = max(pages_for(a, nonneg(a.ctx[b]) + nonneg(a.lens[b])) - held, 0);
    a.held_out[b] = held + static_cast<int>(min(need, max(got - first[b], int64_t{0})));
    if (PACKED) a.starts[b] = static_cast<int32_t>(min(starts[b], int64_t{0x7fffffff}));
  }
  if (threadIdx.x == 0) {
    a.cursor_out[0] = taken + got, a.cursor_out[1] = returned;
    if (PACKED) a.starts[a.B] = static_cast<int32_t>(min(tokens, int64_t{0x7fffffff}));
  }
}

__global__ __launch_bounds__(kThreads) void release_pages_kernel(PagesArgs a) {
  extern __shared__ int64_t s_mem[];
  int32_t* first = reinterpret_cast<int32_t*>(s_mem);
  const int64_t taken = a.cursor[0], returned = a.cursor[1];
  int64_t pages, tokens;
  sums_of<true>(a, first, nullptr, pages, tokens);
  // No more than the ring has room for: pages out of it that no row held twice.
  const int64_t back = min(pages, max(a.F - max(returned - taken, int64_t{0}), int64_t{0}));
  const int64_t base = a.F ? (returned % a.F + a.F) % a.F : 0;
  for (int64_t k = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; k < back; k += static_cast<int64_t>(gridDim.x) * kThreads) {
    const int b = last_not_above(first, a.B, static_cast<int32_t>(k));
    const int keep = min(held_of(a, b), pages_for(a, nonneg(a.lens[b])));
    a.ring[base + k < a.F ? base + k : base + k - a.F] = a.bt[b * a.bt_stride + keep + k - first[b]];
  }
  if (blockIdx.x) return;
  for (int b = threadIdx.x; b < a.B; b += kThreads) a.held_out[b] = min(held_of(a, b), pages_for(a, nonneg(a.lens[b])));
  if (threadIdx.x == 0) a.cursor_out[0] = taken, a.cursor_out[1] = returned + back;
}

int check(const void* block_table, int64_t bt_stride, int64_t pages_per_seq, const void* held, const void* lens, const void* ring,
          int64_t ring_size, const void* cursor, const void* held_out, const void* cursor_out, int B) {
  SPYRE_REQUIRE(B >= 0 && pages_per_seq >= 0 && bt_stride >= 0 && ring_size >= 0, SPYRE_EINVAL,
                "bad sizes B=%d pages_per_seq=%lld free_pages=%lld", B, static_cast<long long>(pages_per_seq),
                static_cast<long long>(ring_size));
  SPYRE_REQUIRE(B <= kMaxSeqs, SPYRE_EUNSUPPORTED, "%d sequences, at most %d", B, kMaxSeqs);
  SPYRE_REQUIRE(pages_per_seq * std::max(B, 1) < (int64_t{1} << 31) && ring_size < (int64_t{1} << 31), SPYRE_EUNSUPPORTED,
                "too many pages");
  SPYRE_REQUIRE(cursor && cursor_out && (B == 0 || (held && lens && held_out)) && (ring || ring_size == 0) &&
                    (block_table || B == 0 || pages_per_seq == 0),
                SPYRE_EINVAL, "null pointer argument");
  return SPYRE_OK;
}

}  // namespace

extern "C" int spyre_plan_pages(int32_t* block_table, int64_t bt_stride, int64_t pages_per_seq, const int32_t* held,
                                const int32_t* context_lens, const int32_t* new_lens, const int32_t* free_pages, int64_t num_free,
                                const int64_t* cursor, int length, int64_t tokens, int32_t* positions, int64_t* slots,
                                int32_t* starts, int32_t* held_out, int64_t* cursor_out, int B, void* stream) {
  spyre_hip::clear_error();
  if (int rc = check(block_table, bt_stride, pages_per_seq, held, new_lens, free_pages, num_free, cursor, held_out, cursor_out, B))
    return rc;
  const bool packed = tokens >= 0;
  SPYRE_REQUIRE(packed != (length >= 0), SPYRE_EINVAL, "either length or tokens is given (length %d, tokens %lld)", length,
                static_cast<long long>(tokens));
  const int64_t rows = packed ? tokens : static_cast<int64_t>(B) * length;
  SPYRE_REQUIRE(rows < (int64_t{1} << 31) - kThreads, SPYRE_EUNSUPPORTED, "too many tokens");
  SPYRE_REQUIRE((B == 0 || context_lens) && (rows == 0 || (positions && slots)) && (!packed || starts), SPYRE_EINVAL,
                "null pointer argument");
  PagesArgs a{};
  a.bt = block_table, a.bt_stride = bt_stride, a.W = static_cast<int>(pages_per_seq);
  a.held = held, a.ctx = context_lens, a.lens = new_lens;
  a.ring = const_cast<int32_t*>(free_pages), a.F = num_free, a.cursor = cursor;
  a.held_out = held_out, a.cursor_out = cursor_out, a.starts = starts;
  a.positions = positions, a.slots = slots, a.rows = rows, a.B = B, a.length = std::max(length, 1);
  a.by_length = make_fastdiv(static_cast<uint32_t>(a.length));
  const dim3 grid(static_cast<uint32_t>(std::min<int64_t>(std::max<int64_t>((rows + kThreads - 1) / kThreads, 1), 1024)));
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (packed)
    plan_pages_kernel<true><<<grid, kThreads, static_cast<size_t>(B) * 12, st>>>(a);
  else
    plan_pages_kernel<false><<<grid, kThreads, static_cast<size_t>(B) * 4, st>>>(a);
  const hipError_t e = hipGetLastError();
  SPYRE_REQUIRE(e == hipSuccess, SPYRE_EHIP, "page plan launch failed: %s", hipGetErrorString(e));
  return SPYRE_OK;
}

extern "C" int spyre_release_pages(const int32_t* block_table, int64_t bt_stride, int64_t pages_per_seq, const int32_t* held,
                                   const int32_t* lens, int32_t* free_pages, int64_t num_free, const int64_t* cursor,
                                   int32_t* held_out, int64_t* cursor_out, int B, void* stream) {
  spyre_hip::clear_error();
  if (int rc = check(block_table, bt_stride, pages_per_seq, held, lens, free_pages, num_free, cursor, held_out, cursor_out, B))
    return rc;
  PagesArgs a{};
  a.bt = const_cast<int32_t*>(block_table), a.bt_stride = bt_stride, a.W = static_cast<int>(pages_per_seq);
  a.held = held, a.lens = lens, a.ring = free_pages, a.F = num_free, a.cursor = cursor;
  a.held_out = held_out, a.cursor_out = cursor_out, a.B = B;
  const int64_t most = std::min<int64_t>(pages_per_seq * B, num_free);
  const dim3 grid(static_cast<uint32_t>(std::min<int64_t>(std::max<int64_t>((most + kThreads - 1) / kThreads, 1), 64)));
  release_pages_kernel<<<grid, kThreads, static_cast<size_t>(B) * 4, static_cast<hipStream_t>(stream)>>>(a);
  const hipError_t e = hipGetLastError();
  SPYRE_REQUIRE(e == hipSuccess, SPYRE_EHIP, "page release launch failed: %s", hipGetErrorString(e));
  return SPYRE_OK;
}
