// Writes to and reads from the paged latent cache (spyre_latent_append_f16,
// spyre_latent_read_f16).
//
// A token is one row for all heads: its latent vector (rank features) and its
// rotated key (64).  Pages hold 64 tokens in sticks of 64 features,
// [num_pages, (rank + 64) / 64, 64 tokens, 64]: the layout of an fp16 K page of
// one head of rank + 64 features.
// A wavefront moves one stick of 8 tokens, 16 bytes a lane: 1 KiB that is
// contiguous in the page where the tokens follow each other there, 8 runs of 128
// bytes in the rows.  Bound by memory: 16 x 100-1500 tokens of rank 512 (35 MB each way)
// append 8.5 us, read 8.9, 4.1 TB/s.

#include <hip/hip_runtime.h>

#include "fast_div.h"
#include "page_walk.h"
#include "spyre_common.h"

namespace {

using namespace spyre_hip;

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kRope = 64;
constexpr int kThreads = 256;

struct CacheArgs {
  const _Float16 *latent, *rope;  // append: rows
  int64_t latent_s, rope_s;
  _Float16 *latent_out, *rope_out;  // read
  _Float16* pages;
  const int64_t* slots;
  const int32_t *bt, *lens, *start;
  int64_t bt_stride, pages_per_seq, num_pages;
  uint32_t units, sticks, rows, length;  // units: of 8 rows x 1 stick
  int rank;
  FastDiv by_sticks, by_length;
};

__global__ __launch_bounds__(kThreads) void latent_append_kernel(CacheArgs a) {
  const uint32_t u = blockIdx.x * (kThreads / 64) + threadIdx.x / 64, lane = threadIdx.x % 64;
  if (u >= a.units) return;
  const uint32_t group = fdiv(u, a.by_sticks), stick = u - group * a.sticks, row = group * 8 + lane / 8;
  if (row >= a.rows) return;
  const int64_t slot = a.slots[row];
  if (slot < 0 || slot / kPage >= a.num_pages) return;
  const int f = static_cast<int>(stick * 64 + lane % 8 * 8);
  const _Float16* src = f < a.rank ? a.latent + row * a.latent_s + f : a.rope + row * a.rope_s + f - a.rank;
  const int64_t dst = ((slot / kPage * a.sticks + stick) * kPage + slot % kPage) * 64 + lane % 8 * 8;
  *reinterpret_cast<u32x4*>(a.pages + dst) = *reinterpret_cast<const u32x4*>(src);
}

__global__ __launch_bounds__(kThreads) void latent_read_kernel(CacheArgs a) {
  const uint32_t u = blockIdx.x * (kThreads / 64) + threadIdx.x / 64, lane = threadIdx.x % 64;
  if (u >= a.units) return;
  const uint32_t group = fdiv(u, a.by_sticks), stick = u - group * a.sticks, row = group * 8 + lane / 8;
  if (row >= a.rows) return;
  const uint32_t b = fdiv(row, a.by_length);
  const int64_t t = static_cast<int64_t>(row - b * a.length) + (a.start ? a.start[b] : 0);
  u32x4 x = {0, 0, 0, 0};
  if (t >= 0 && t < a.lens[b]) {
    const int64_t page = t / kPage < a.pages_per_seq ? a.bt[b * a.bt_stride + t / kPage] : -1;
    if (page >= 0 && page < a.num_pages)
      x = *reinterpret_cast<const u32x4*>(a.pages + ((page * a.sticks + stick) * kPage + t % kPage) * 64 + lane % 8 * 8);
    else
      x = u32x4{0x7e007e00u, 0x7e007e00u, 0x7e007e00u, 0x7e007e00u};  // NaN
  }
  const int f = static_cast<int>(stick * 64 + lane % 8 * 8);
  _Float16* dst = f < a.rank ? a.latent_out + static_cast<int64_t>(row) * a.rank + f
                             : a.rope_out + static_cast<int64_t>(row) * kRope + f - a.rank;
  *reinterpret_cast<u32x4*>(dst) = x;
}

bool aligned(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

int check(int rank, int64_t num_pages, int64_t rows) {
  SPYRE_REQUIRE(rank == 256 || rank == 512, SPYRE_EUNSUPPORTED, "rank %d not in {256, 512}", rank);
  SPYRE_REQUIRE(num_pages >= 0, SPYRE_EINVAL, "bad num_pages");
  SPYRE_REQUIRE(rows < (int64_t{1} << 31) && (rows + 7) / 8 * ((rank + kRope) / 64) < (int64_t{1} << 31) - kThreads,
                SPYRE_EUNSUPPORTED, "too many rows");
  return SPYRE_OK;
}

CacheArgs args_of(int rank, int64_t rows) {
  CacheArgs a{};
  a.rank = rank, a.rows = static_cast<uint32_t>(rows), a.sticks = static_cast<uint32_t>((rank + kRope) / 64);
  a.units = static_cast<uint32_t>((rows + 7) / 8) * a.sticks;
  a.by_sticks = make_fastdiv(a.sticks);
  return a;
}

dim3 grid_of(const CacheArgs& a) { return dim3((a.units + kThreads / 64 - 1) / (kThreads / 64)); }

}  // namespace

extern "C" int spyre_latent_append_f16(const void* latent, int64_t latent_stride, const void* k_rope, int64_t k_rope_stride,
                                       void* cache, const int64_t* slots, int64_t rows, int rank, int64_t num_pages,
                                       void* stream) {
  spyre_hip::clear_error();
  SPYRE_REQUIRE(rows >= 0, SPYRE_EINVAL, "bad rows");
  if (int rc = check(rank, num_pages, rows)) return rc;
  if (rows == 0 || num_pages == 0) return SPYRE_OK;  // (every slot is outside of no pages)
  SPYRE_REQUIRE(latent && k_rope && cache && slots, SPYRE_EINVAL, "null pointer argument");
  SPYRE_REQUIRE(aligned(latent) && aligned(k_rope) && aligned(cache) && latent_stride % 8 == 0 && k_rope_stride % 8 == 0,
                SPYRE_EINVAL, "rows and the cache must be 16-byte aligned");
  CacheArgs a = args_of(rank, rows);
  a.latent = static_cast<const _Float16*>(latent), a.latent_s = latent_stride;
  a.rope = static_cast<const _Float16*>(k_rope), a.rope_s = k_rope_stride;
  a.pages = static_cast<_Float16*>(cache), a.slots = slots, a.num_pages = num_pages;
  latent_append_kernel<<<grid_of(a), kThreads, 0, static_cast<hipStream_t>(stream)>>>(a);
  const hipError_t e = hipGetLastError();
  SPYRE_REQUIRE(e == hipSuccess, SPYRE_EHIP, "latent append launch failed: %s", hipGetErrorString(e));
  return SPYRE_OK;
}

extern "C" int spyre_latent_read_f16(const void* cache, const int32_t* block_table, int64_t bt_stride, int64_t pages_per_seq,
                                     const int32_t* lens, const int32_t* start, void* latent, void* k_rope, int B, int length,
                                     int rank, int64_t num_pages, void* stream) {
  spyre_hip::clear_error();
  SPYRE_REQUIRE(B >= 0 && length >= 0 && bt_stride >= 0 && pages_per_seq >= 0, SPYRE_EINVAL, "bad sizes B=%d length=%d", B, length);
  const int64_t rows = static_cast<int64_t>(B) * length;
  if (int rc = check(rank, num_pages, rows)) return rc;
  if (rows == 0) return SPYRE_OK;
  SPYRE_REQUIRE((cache || num_pages == 0) && (block_table || pages_per_seq == 0) && lens && latent && k_rope, SPYRE_EINVAL,
                "null pointer argument");
  SPYRE_REQUIRE(aligned(cache) && aligned(latent) && aligned(k_rope), SPYRE_EINVAL, "the cache and the rows must be 16-byte aligned");
  CacheArgs a = args_of(rank, rows);
  a.pages = const_cast<_Float16*>(static_cast<const _Float16*>(cache)), a.num_pages = num_pages;
  a.bt = block_table, a.bt_stride = bt_stride, a.pages_per_seq = pages_per_seq, a.lens = lens, a.start = start;
  a.latent_out = static_cast<_Float16*>(latent), a.rope_out = static_cast<_Float16*>(k_rope);
  a.length = static_cast<uint32_t>(length), a.by_length = make_fastdiv(a.length);
  latent_read_kernel<<<grid_of(a), kThreads, 0, static_cast<hipStream_t>(stream)>>>(a);
  const hipError_t e = hipGetLastError();
  SPYRE_REQUIRE(e == hipSuccess, SPYRE_EHIP, "latent read launch failed: %s", hipGetErrorString(e));
  return SPYRE_OK;
}
