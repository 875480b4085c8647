// Attention of decoded tokens whose requests share leading pages: the keys and values of a common prefix are read once for all
// requests of a group, each request's own keys once for itself, and the two are put together.
//
//   o[i,h] = sum_j p_j v_j / sum_j p_j,  p_j = exp(q[i,h] . k_j scale - m)   over j in prefix(i) and own(i)
//
// A part of a row's keys leaves a state (m, l, o): the largest exponent, the sum and the unnormalised output relative to it.
// States of parts add up after scaling by exp(m - max m), in the order of the parts, so the split changes only roundings.
//
// Parts of one (request, head), each with a place of its own in scratch memory:
//   0 .. prefix_parts - 1              `chunk` keys of the prefix each, as many as the request's prefix has
//   prefix_parts .. + own_parts - 1    equal parts of the request's own keys, as many as there are (see own_range)
// Rows of a work item: of a prefix, the query heads of one kv head of up to 128 / heads_per_kv requests; of own keys, those of
// one request.
#include "mma_attention.cuh"

namespace mlr {

constexpr int OWN_LEAST = 256;        // keys of an own part, at least

struct PrefixCall {
  const void* q;                  // [segments, heads * dim]: row of segment i is q_row[i]
  const void *k_pool, *v_pool;    // [pages, kv_heads, page_size, dim]
  const int *q_row, *pos0, *seg_slot, *block_table;
  const int* seg_keys;            // [segments]: shared keys before each segment's own
  const int* members;             // segments of the groups, one behind the other
  const int *tile_first, *tile_count, *tile_keys;      // work items of the prefixes: members, their number, shared keys
  float *acc, *state;             // [parts][segments][heads][dim] and [parts][segments][heads][2]
  void* out;
  int segments, tiles, heads, kv_heads, dim, page_size, pages, table_width;
  int chunk, prefix_parts, own_parts;
  float scale_log2;
};

// A segment's own keys [begin, end) of part `part`; empty if there are fewer parts.  Multiples of 64 keys from the first own key on.
__device__ __forceinline__ void own_range(const PrefixCall& c, int segment, int part, int* begin, int* end) {
  const int first = c.seg_keys[segment], last = __ldcg(c.pos0 + segment) + 1;
  const int own = max(0, last - first);
  const int each = max(OWN_LEAST, ((own + c.own_parts - 1) / c.own_parts + 63) & ~63);
  *begin = min(last, first + part * each);
  *end = min(last, *begin + each);
}

// A cached row's place: null where the request holds no such page.
template <typename T>
__device__ __forceinline__ const T* cached_row(const PrefixCall& c, const void* pool, const int* table, int kv_head, int key) {
  const int logical = key / c.page_size;
  const int page = logical < c.table_width ? __ldcg(table + logical) : -1;
  if (page < 0 || page >= c.pages) return nullptr;
  return (const T*)pool + (((size_t)page * c.kv_heads + kv_head) * c.page_size + (key - logical * c.page_size)) * c.dim;
}

// ------------------------------------------------------------------ any type, any head size up to 256
constexpr int PLAIN_ROWS = 8, PLAIN_KEYS = 32, PLAIN_THREADS = 128;

// CTA = (eight rows of an item, one part of its keys).  PREFIX: y is a tile of the prefixes, else a segment.
template <typename T, bool PREFIX>
__global__ void __launch_bounds__(PLAIN_THREADS)
prefix_parts_plain_kernel(const PrefixCall c) {
  pdl_trigger();
  pdl_wait();
  extern __shared__ float plain_shared[];
  const int dim = c.dim, pitch = dim + 1;
  float* q = plain_shared;                            // [8][dim]
  float* keys = q + PLAIN_ROWS * dim;                 // [32][dim + 1]
  float* values = keys + PLAIN_KEYS * pitch;          // [32][dim]
  __shared__ float p[PLAIN_ROWS][PLAIN_KEYS];
  __shared__ float alpha[PLAIN_ROWS];
  __shared__ int open[PLAIN_KEYS];
  const int per = c.heads / c.kv_heads, kv_head = blockIdx.z;
  const int blocks = PREFIX ? (128 + PLAIN_ROWS - 1) / PLAIN_ROWS : (per + PLAIN_ROWS - 1) / PLAIN_ROWS;
  const int part = blockIdx.x / blocks, row0 = (blockIdx.x - part * blocks) * PLAIN_ROWS;
  int rows, begin, end, owner;
  if (PREFIX) {
    rows = c.tile_count[blockIdx.y] * per - row0;
    begin = part * c.chunk;
    end = min(c.tile_keys[blockIdx.y], begin + c.chunk);
    owner = c.members[c.tile_first[blockIdx.y]];
  } else {
    rows = per - row0;
    owner = blockIdx.y;
    own_range(c, owner, part, &begin, &end);
  }
  rows = min(rows, PLAIN_ROWS);
  if (rows <= 0 || begin >= end) return;
  const int* table = c.block_table + (size_t)__ldcg(c.seg_slot + owner) * c.table_width;
  auto segment_of = [&](int r) { return PREFIX ? c.members[c.tile_first[blockIdx.y] + (row0 + r) / per] : owner; };
  auto head_of = [&](int r) { return kv_head * per + (row0 + r) % per; };
  for (int i = threadIdx.x; i < PLAIN_ROWS * dim; i += PLAIN_THREADS) {
    const int r = i / dim, d = i - r * dim;
    q[i] = r < rows ? to_float(((const T*)c.q)[((size_t)c.q_row[segment_of(r)] * c.heads + head_of(r)) * dim + d]) * c.scale_log2 : 0.f;
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float acc[PLAIN_ROWS][2];                           // columns threadIdx.x and threadIdx.x + 128
#pragma unroll
  for (int r = 0; r < PLAIN_ROWS; ++r) acc[r][0] = acc[r][1] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};      // of rows 2 * warp and 2 * warp + 1, the same in every lane
  for (int key0 = begin; key0 < end; key0 += PLAIN_KEYS) {
    __syncthreads();
    for (int k = warp; k < PLAIN_KEYS; k += PLAIN_THREADS / 32) {
      const T* kr = key0 + k < end ? cached_row<T>(c, c.k_pool, table, kv_head, key0 + k) : nullptr;
      const T* vr = kr != nullptr ? (const T*)c.v_pool + (kr - (const T*)c.k_pool) : nullptr;
      if (lane == 0) open[k] = kr != nullptr;
      for (int d = lane; d < dim; d += 32) {
        keys[k * pitch + d] = kr != nullptr ? to_float(kr[d]) : 0.f;
        values[k * dim + d] = vr != nullptr ? to_float(vr[d]) : 0.f;
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = 2 * warp + i;
      float s = 0.f;
      for (int d = 0; d < dim; ++d) s = fmaf(q[r * dim + d], keys[lane * pitch + d], s);
      if (!open[lane]) s = -INFINITY;
      const float top = fmaxf(m[i], warp_max(s));
      const float base = top == -INFINITY ? 0.f : top;
      const float e = exp2f(s - base), shrink = exp2f(m[i] - base);
      l[i] = l[i] * shrink + warp_sum(e);
      m[i] = top;
      p[r][lane] = e;
      if (lane == 0) alpha[r] = shrink;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < PLAIN_ROWS; ++r) { acc[r][0] *= alpha[r]; acc[r][1] *= alpha[r]; }
    for (int k = 0; k < PLAIN_KEYS; ++k) {
      const float v0 = (int)threadIdx.x < dim ? values[k * dim + threadIdx.x] : 0.f;
      const float v1 = (int)threadIdx.x + 128 < dim ? values[k * dim + threadIdx.x + 128] : 0.f;
#pragma unroll
      for (int r = 0; r < PLAIN_ROWS; ++r) {
        acc[r][0] = fmaf(p[r][k], v0, acc[r][0]);
        acc[r][1] = fmaf(p[r][k], v1, acc[r][1]);
      }
    }
  }
  const int place = PREFIX ? part : c.prefix_parts + part;
#pragma unroll
  for (int r = 0; r < PLAIN_ROWS; ++r) {
    if (r >= rows) break;
    const size_t at = ((size_t)place * c.segments + segment_of(r)) * c.heads + head_of(r);
    if ((int)threadIdx.x < dim) c.acc[at * dim + threadIdx.x] = acc[r][0];
    if ((int)threadIdx.x + 128 < dim) c.acc[at * dim + threadIdx.x + 128] = acc[r][1];
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = 2 * warp + i;
    if (lane == 0 && r < rows) {
      const size_t at = ((size_t)place * c.segments + segment_of(r)) * c.heads + head_of(r);
      c.state[2 * at] = m[i];
      c.state[2 * at + 1] = l[i];
    }
  }
}

// ------------------------------------------------------------------ the parts put together
// One warp per (segment, head); a row that sees no key is zero.
template <typename T>
__global__ void __launch_bounds__(128)
prefix_merge_kernel(const PrefixCall c) {
  pdl_trigger();
  pdl_wait();
  const int row = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (row >= c.segments * c.heads) return;
  const int segment = row / c.heads;
  const int shared = c.seg_keys[segment];
  const int prefix = c.chunk > 0 ? (shared + c.chunk - 1) / c.chunk : 0;
  int own = 0;
  for (int part = 0; part < c.own_parts; ++part) {
    int begin, end;
    own_range(c, segment, part, &begin, &end);
    own += begin < end;
  }
  const int parts = prefix + own;
  const size_t pitch = (size_t)c.segments * c.heads;
  auto place = [&](int part) { return (size_t)(part < prefix ? part : c.prefix_parts + part - prefix) * pitch + row; };
  float top = -INFINITY;
  for (int part = lane; part < parts; part += 32) top = fmaxf(top, __ldcg(c.state + 2 * place(part)));
  top = warp_max(top);
  const float base = top == -INFINITY ? 0.f : top;
  float sum = 0.f;
  float o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int part = 0; part < parts; ++part) {
    const size_t at = place(part);
    const float factor = exp2f(__ldcg(c.state + 2 * at) - base);
    sum = fmaf(__ldcg(c.state + 2 * at + 1), factor, sum);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (lane + 32 * i < c.dim) o[i] = fmaf(__ldcg(c.acc + at * c.dim + lane + 32 * i), factor, o[i]);
  }
  const float inverse = sum == 0.f ? 0.f : 1.f / sum;      // NaN stays
  T* to = (T*)c.out + ((size_t)c.q_row[segment] * c.heads + (row - segment * c.heads)) * c.dim;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (lane + 32 * i < c.dim) to[lane + 32 * i] = from_float<T>(o[i] * inverse);
}

template <typename T>
static int run_plain(const PrefixCall& c, cudaStream_t stream) {
  const size_t shared = (size_t)(PLAIN_ROWS * c.dim + PLAIN_KEYS * (c.dim + 1) + PLAIN_KEYS * c.dim) * 4;
  static OncePerDevice once[2];
  const int most = (PLAIN_ROWS * 256 + PLAIN_KEYS * 257 + PLAIN_KEYS * 256) * 4;
  if (cudaError_t err = once[0]([&] { return cudaFuncSetAttribute(prefix_parts_plain_kernel<T, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, most); }))
    return (int)err;
  if (cudaError_t err = once[1]([&] { return cudaFuncSetAttribute(prefix_parts_plain_kernel<T, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, most); }))
    return (int)err;
  const int per = c.heads / c.kv_heads;
  if (c.tiles > 0)
    launch_kernel(prefix_parts_plain_kernel<T, true>, dim3(c.prefix_parts * (128 / PLAIN_ROWS), c.tiles, c.kv_heads), dim3(PLAIN_THREADS), shared,
                  stream, c);
  launch_kernel(prefix_parts_plain_kernel<T, false>, dim3(c.own_parts * ((per + PLAIN_ROWS - 1) / PLAIN_ROWS), c.segments, c.kv_heads),
                dim3(PLAIN_THREADS), shared, stream, c);
  launch_kernel(prefix_merge_kernel<T>, dim3((c.segments * c.heads + 3) / 4), dim3(128), 0, stream, c);
  return launch_status();
}

}  // namespace mlr

using namespace mlr;

MLR_DEFINE_PDL_SWITCH

// q, out [rows, heads * dim], pools [pages, kv_heads, page_size, dim] of one dtype.  acc, state: float32, (prefix_parts + own_parts) *
// segments * heads * dim and * 2 of them.  chunk: keys of a prefix part (prefix_parts of them reach the longest prefix).
MLR_EXPORT int mlr_attention_prefix(const void* q, const void* k_pool, const void* v_pool, void* out, const int* q_row, const int* pos0,
                                    const int* seg_slot, const int* block_table, const int* seg_keys, const int* members,
                                    const int* tile_first, const int* tile_count, const int* tile_keys, float* acc, float* state,
                                    int segments, int tiles, int heads, int kv_heads, int dim, int page_size, int pages, int table_width,
                                    int chunk, int prefix_parts, int own_parts, float scale, int dtype, cudaStream_t stream) {
  if (segments < 0 || tiles < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 || dim <= 0 || page_size <= 0 || pages <= 0 ||
      table_width <= 0 || own_parts <= 0 || prefix_parts < 0 || (tiles > 0 && (chunk <= 0 || prefix_parts <= 0)))
    return MLR_BAD_SIZE;
  if (segments == 0) return MLR_OK;
  if (dim > 256 || heads / kv_heads > 128 || segments > 65535 || tiles > 65535 || kv_heads > 65535) return MLR_TOO_LARGE;
  const PrefixCall c{q, k_pool, v_pool, q_row, pos0, seg_slot, block_table, seg_keys, members, tile_first, tile_count, tile_keys, acc, state, out,
                     segments, tiles, heads, kv_heads, dim, page_size, pages, table_width, chunk, prefix_parts, own_parts,
                     scale * 1.4426950408889634f};
  if (dtype == MLR_BF16) return run_plain<bf16>(c, stream);
  if (dtype == MLR_F32) return run_plain<float>(c, stream);
  return MLR_BAD_DTYPE;
}
