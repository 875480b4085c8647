// Pages of a cache copied within their pools or into other ones: target page j of every entry and pool gets what source page j
// holds.  A fork of a request needs the page that it ends in, a compaction those that lie behind the holes.
//
// A page of one entry is contiguous (all kv heads), so a CTA moves one page of one entry with accesses of 16 bytes (or of
// 4 or 1, where sizes or addresses allow no more).  The pairs of pages travel in the launch's parameters: no copy to
// the device comes before it.  No page is source and target at once (the host sees to that), so the order does not matter.
#include "common.cuh"

namespace mlr {

constexpr int COPY_POOLS = 8, COPY_PAIRS = 400, COPY_THREADS = 256;

struct PagePool {
  const uint8_t* source;
  uint8_t* target;
  long long source_entry, target_entry;      // bytes from entry to entry
  long long page_bytes;
  int entries;
};
struct PageCopies {
  PagePool pools[COPY_POOLS];
  int first_unit[COPY_POOLS + 1];             // units (entries) of the pools before
  int count, pool_count;
  int2 pairs[COPY_PAIRS];                     // (source, target)
};

// `x` pairs, `y` entries of the pools one behind the other
template <typename PIECE>
__global__ void __launch_bounds__(COPY_THREADS)
copy_pages_kernel(const __grid_constant__ PageCopies copies) {
  pdl_trigger();
  const int unit = blockIdx.y;
  int p = 0;
  while (p + 1 < copies.pool_count && unit >= copies.first_unit[p + 1]) ++p;
  const PagePool& pool = copies.pools[p];
  const int entry = unit - copies.first_unit[p];
  const int2 pair = copies.pairs[blockIdx.x];
  const PIECE* src = reinterpret_cast<const PIECE*>(pool.source + entry * pool.source_entry + pair.x * pool.page_bytes);
  PIECE* dst = reinterpret_cast<PIECE*>(pool.target + entry * pool.target_entry + pair.y * pool.page_bytes);
  const long long pieces = pool.page_bytes / (long long)sizeof(PIECE);
  pdl_wait();
  constexpr int AHEAD = 4;
  for (long long first = threadIdx.x; first < pieces; first += AHEAD * COPY_THREADS) {
    PIECE v[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      if (first + i * COPY_THREADS < pieces) v[i] = src[first + i * COPY_THREADS];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      if (first + i * COPY_THREADS < pieces) dst[first + i * COPY_THREADS] = v[i];
  }
}

}  // namespace mlr

using namespace mlr;

MLR_DEFINE_PDL_SWITCH

// For each of `pools`: where the source's and the target's first page lie, the bytes from entry to entry of each, the bytes of a
// page, the entries (six numbers).  source, target: `count` page numbers each, in host memory.
MLR_EXPORT int mlr_copy_pages(const long long* pools, int pool_count, const int* source, const int* target, int count, cudaStream_t stream) {
  if (count == 0 || pool_count == 0) return MLR_OK;
  if (count < 0 || pool_count < 0 || pool_count > COPY_POOLS) return MLR_BAD_SIZE;
  PageCopies copies;
  int units = 0;
  unsigned long long bits = 0;
  for (int p = 0; p < pool_count; ++p) {
    const long long* f = pools + 6 * p;
    copies.pools[p] = PagePool{(const uint8_t*)(uintptr_t)f[0], (uint8_t*)(uintptr_t)f[1], f[2], f[3], f[4], (int)f[5]};
    if (f[4] <= 0 || f[5] < 0 || f[5] > 65535) return MLR_BAD_SIZE;
    for (int i = 0; i < 5; ++i) bits |= (unsigned long long)f[i];
    copies.first_unit[p] = units;
    units += (int)f[5];
  }
  copies.first_unit[pool_count] = units;
  copies.pool_count = pool_count;
  if (units == 0) return MLR_OK;
  if (units > 65535) return MLR_TOO_LARGE;
  auto kernel = bits % 16 == 0 ? copy_pages_kernel<uint4> : bits % 4 == 0 ? copy_pages_kernel<unsigned int> : copy_pages_kernel<uint8_t>;
  for (int first = 0; first < count; first += COPY_PAIRS) {
    copies.count = count - first < COPY_PAIRS ? count - first : COPY_PAIRS;
    for (int i = 0; i < copies.count; ++i) copies.pairs[i] = make_int2(source[first + i], target[first + i]);
    launch_kernel(kernel, dim3(copies.count, units), dim3(COPY_THREADS), 0, stream, copies);
    const int status = launch_status();
    if (status != MLR_OK) return status;
  }
  return MLR_OK;
}
