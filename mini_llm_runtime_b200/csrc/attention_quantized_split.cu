// Decoded tokens over keys and values in 8 bits on the CUDA cores in float32: queries of either type, every head size up to 256, every page
// and block size, any number of query heads per kv head (four or eight at a time).
//
//   out = sum_j e^(q.k_j scale - m) v_j / sum_j e^(q.k_j scale - m),  k_j = kc_j ks, v_j = vc_j vs
// A CTA walks a part of one request's keys for one kv head and up to eight of its query heads, in tiles of 64 keys: every code is read
// once for all of these heads and turned into float32 as it arrives in shared memory (scales stay apart: a score is the codes' dot
// product times ks, a weight is multiplied by vs).  Scores: a thread per key and a quarter of the heads.  Sums: a thread per four
// dimensions and a part of the keys, the weights broadcast from shared memory.  Shared-memory reads bound it: a float of a key or
// value serves two and eight multiply-adds.  Parts are `chunk` keys from absolute positions: 256, or twice as many
// until the parts' states of a large batch fit the host's limit; a second launch merges them in order.  24 requests of up to 2,500 keys, 12 heads of 96
// over 3, float32: 34 us (49 with room for eight heads where four are enough; 1,029 with 16 rows of a prompt's kernel).
// A key that a row does not see gives it nothing, whatever lies there.
#include "common.cuh"

namespace mlr {

constexpr int QS_KEYS = 64, QS_THREADS = 256;
constexpr int QS_MAX_DIM = 256;

// [part][request][head]: top, sum; outputs behind them
template <typename T, int HEADS>
__global__ void __launch_bounds__(QS_THREADS, HEADS == 4 ? 3 : 2)
attention_quantized_split_kernel(const T* q, const int8_t* k_pool, const int8_t* v_pool, const float* k_scales, const float* v_scales,
                                 float2* __restrict__ sums, float* __restrict__ states, const int* __restrict__ decode_seg,
                                 const int* __restrict__ seg_q_start, const int* __restrict__ seg_pos0, const int* __restrict__ block_table,
                                 const int* __restrict__ seg_slot, int table_width, int requests, int heads, int kv_heads, int dim, int page_size,
                                 int block, int pool_pages, int window, float scale, int chunk) {
  pdl_trigger();
  const int request = blockIdx.y / kv_heads, kv_head = blockIdx.y - request * kv_heads, group = heads / kv_heads;
  const int head0 = kv_head * group + blockIdx.z * HEADS, mine = min(HEADS, group - (int)blockIdx.z * HEADS);
  const int segment = decode_seg != nullptr ? decode_seg[request] : request, row = seg_q_start[segment], position = seg_pos0[segment];
  const int lowest = window > 0 ? max(0, position - window + 1) : 0;
  const int first_part = lowest / chunk, part = blockIdx.x;
  // (the last part walks on to the end of a context that is longer than the launch was made for)
  const int begin = max(lowest, (first_part + part) * chunk), end = part == (int)gridDim.x - 1 ? position + 1 : min(position + 1, (first_part + part + 1) * chunk);
  pdl_wait();
  if (begin >= end) return;
  const int* table = block_table + (size_t)(seg_slot != nullptr ? seg_slot[segment] : segment) * table_width;
  extern __shared__ __align__(16) float qs_shared[];
  // rows of `wide` floats: a multiple of four, and of an odd number of them (rows of neighbouring keys start in other banks)
  const int wide = ((dim + 3) / 4 | 1) * 4, quads = (dim + 3) / 4;
  float* queries = qs_shared;                        // [HEADS][wide]
  float* keys = queries + HEADS * wide;           // [QS_KEYS][wide]
  float* values = keys + QS_KEYS * wide;             // [QS_KEYS][wide]
  float* weights = values + QS_KEYS * wide;          // [QS_KEYS][HEADS]
  float* scales = weights + QS_KEYS * HEADS;      // [2][QS_KEYS]
  float* tops = scales + 2 * QS_KEYS;                // [HEADS]: the maximum, the factor of what came before, the sum
  float* factors = tops + HEADS;
  float* totals = factors + HEADS;
  const int thread = threadIdx.x, lane = thread & 31, warp = thread >> 5, per_page = page_size / block;

  for (int i = thread; i < HEADS * wide; i += QS_THREADS) {
    const int h = i / wide, d = i - h * wide;
    queries[i] = h < mine && d < dim ? to_float(q[((size_t)row * heads + head0 + h) * dim + d]) * scale : 0.f;
  }
  if (thread < HEADS) { tops[thread] = -INFINITY; totals[thread] = 0.f; }
  // sums: thread -> four dimensions, of `slices` parts of the keys (no more than there are keys: at the end `slices` rows of `quads` take the
  // place of the QS_KEYS rows of `wide` >= 4 quads floats)
  const int slices = min(QS_THREADS / quads, QS_KEYS), slice = thread / quads, quad = thread - slice * quads;
  float4 out[HEADS];
#pragma unroll
  for (int h = 0; h < HEADS; ++h) out[h] = make_float4(0.f, 0.f, 0.f, 0.f);

  // codes: 16 at a time where rows lie on such boundaries, else one
  const bool wide_rows = dim % 16 == 0 && ((((uintptr_t)k_pool | (uintptr_t)v_pool) & 15) == 0);
  for (int key0 = begin / QS_KEYS * QS_KEYS; key0 < end; key0 += QS_KEYS) {
    __syncthreads();
    auto line_of = [&](int key, int* offset) -> long long {      // -1: no such key
      const int logical = key / page_size;
      const int page = key >= begin && key < end && logical < table_width ? table[logical] : -1;
      *offset = key - logical * page_size;
      return page >= 0 && page < pool_pages ? (long long)page * kv_heads + kv_head : -1;
    };
    if (thread < 2 * QS_KEYS) {
      const bool of_values = thread >= QS_KEYS;
      int offset;
      const long long line = line_of(key0 + (thread & (QS_KEYS - 1)), &offset);
      scales[thread] = line >= 0 ? (of_values ? v_scales : k_scales)[line * per_page + offset / block] : 0.f;
    }
    if (wide_rows) {
      const int pieces = dim / 16;
      for (int i = thread; i < 2 * QS_KEYS * pieces; i += QS_THREADS) {
        const int of_values = i >= QS_KEYS * pieces, at = i - of_values * QS_KEYS * pieces, j = at / pieces, c = at - j * pieces;
        int offset;
        const long long line = line_of(key0 + j, &offset);
        uint4 raw = make_uint4(0u, 0u, 0u, 0u);
        if (line >= 0) raw = __ldcg(reinterpret_cast<const uint4*>((of_values ? v_pool : k_pool) + (line * page_size + offset) * dim) + c);
        const uint32_t words[4] = {raw.x, raw.y, raw.z, raw.w};
        float4* dst = reinterpret_cast<float4*>((of_values ? values : keys) + j * wide + c * 16);
#pragma unroll
        for (int w = 0; w < 4; ++w)
          dst[w] = make_float4((float)(int8_t)words[w], (float)(int8_t)(words[w] >> 8), (float)(int8_t)(words[w] >> 16), (float)(int8_t)(words[w] >> 24));
      }
    } else {
      for (int i = thread; i < 2 * QS_KEYS * wide; i += QS_THREADS) {
        const int of_values = i >= QS_KEYS * wide, at = i - of_values * QS_KEYS * wide, j = at / wide, d = at - j * wide;
        int offset;
        const long long line = line_of(key0 + j, &offset);
        float x = 0.f;
        if (line >= 0 && d < dim) x = (float)(of_values ? v_pool : k_pool)[(line * page_size + offset) * dim + d];
        (of_values ? values : keys)[at] = x;
      }
    }
    __syncthreads();
    // ---- scores: thread -> key, a quarter of the heads
    {
      constexpr int EACH = HEADS / 4;
      const int j = thread & (QS_KEYS - 1), quarter = thread / QS_KEYS;
      const float4* k_row = reinterpret_cast<const float4*>(keys + j * wide);
      const float4* q_row = reinterpret_cast<const float4*>(queries + EACH * quarter * wide);
      float s[EACH] = {};
      if (EACH * quarter < mine) {
#pragma unroll 4
        for (int c = 0; c < quads; ++c) {
          const float4 k = k_row[c];
#pragma unroll
          for (int h = 0; h < EACH; ++h) {
            const float4 a = q_row[h * (wide / 4) + c];
            s[h] = fmaf(k.x, a.x, fmaf(k.y, a.y, fmaf(k.z, a.z, fmaf(k.w, a.w, s[h]))));
          }
        }
      }
      const bool seen = key0 + j >= begin && key0 + j < end;
      const float ks = scales[j];
#pragma unroll
      for (int h = 0; h < EACH; ++h) weights[j * HEADS + EACH * quarter + h] = seen ? s[h] * ks : -INFINITY;
    }
    __syncthreads();
    // ---- maxima and weights: a warp per head
    if (warp < mine) {
      const float a = weights[lane * HEADS + warp], b = weights[(lane + 32) * HEADS + warp];
      const float before = tops[warp], top = fmaxf(before, warp_max(fmaxf(a, b)));      // (NaN is passed over; its weight is NaN)
      const float base = top == -INFINITY ? 0.f : top;
      const float wa = a == -INFINITY ? 0.f : expf(a - base), wb = b == -INFINITY ? 0.f : expf(b - base);
      const float sum = warp_sum(wa + wb), factor = before == -INFINITY ? 0.f : expf(before - base);
      // a key that is not seen has weight zero, and its value's scale counts for nothing; a seen one's counts however small its weight (NaN stays)
      auto seen = [&](int j) { return key0 + j >= begin && key0 + j < end; };
      weights[lane * HEADS + warp] = seen(lane) ? wa * scales[QS_KEYS + lane] : 0.f;
      weights[(lane + 32) * HEADS + warp] = seen(lane + 32) ? wb * scales[QS_KEYS + lane + 32] : 0.f;
      __syncwarp();
      if (lane == 0) {
        tops[warp] = top;
        factors[warp] = factor;
        totals[warp] = (totals[warp] == totals[warp] ? totals[warp] * factor : totals[warp]) + sum;
      }
    }
    __syncthreads();
    // ---- sums
    if (slice < slices) {
#pragma unroll
      for (int h = 0; h < HEADS; ++h)
        if (h < mine) {
          const float f = factors[h];
          out[h] = make_float4(out[h].x * f, out[h].y * f, out[h].z * f, out[h].w * f);
        }
      for (int j = slice; j < QS_KEYS; j += slices) {
        const float4 v = reinterpret_cast<const float4*>(values + j * wide)[quad];
        float w[HEADS];
#pragma unroll
        for (int h = 0; h < HEADS; h += 4) {
          const float4 four = *reinterpret_cast<const float4*>(weights + j * HEADS + h);
          w[h] = four.x, w[h + 1] = four.y, w[h + 2] = four.z, w[h + 3] = four.w;
        }
#pragma unroll
        for (int h = 0; h < HEADS; ++h)
          if (h < mine) {
            out[h].x = fmaf(w[h], v.x, out[h].x);
            out[h].y = fmaf(w[h], v.y, out[h].y);
            out[h].z = fmaf(w[h], v.z, out[h].z);
            out[h].w = fmaf(w[h], v.w, out[h].w);
          }
      }
    }
  }
  // ---- the slices' sums, through the keys' memory; then the part's state
  const size_t state = ((size_t)part * requests + request) * heads + head0;
  for (int h = 0; h < mine; ++h) {
    __syncthreads();
    if (slice < slices) {
      float4 v = out[0];
#pragma unroll
      for (int i = 1; i < HEADS; ++i)
        if (i == h) v = out[i];
      reinterpret_cast<float4*>(keys)[slice * quads + quad] = v;
    }
    __syncthreads();
    for (int d = thread; d < dim; d += QS_THREADS) {
      float sum = 0.f;
      for (int i = 0; i < slices; ++i) sum += keys[i * quads * 4 + d];
      states[(state + h) * dim + d] = sum;
    }
  }
  if (thread < mine) sums[state + thread] = make_float2(tops[thread], totals[thread]);
}

// A CTA per request and head.
template <typename T>
__global__ void __launch_bounds__(128)
merge_quantized_split_kernel(const float2* sums, const float* states, T* __restrict__ out, const int* __restrict__ decode_seg,
                             const int* __restrict__ seg_q_start, const int* __restrict__ seg_pos0, int requests, int heads, int dim, int window,
                             int chunk, int most_parts) {
  pdl_trigger();
  const int request = blockIdx.x / heads, head = blockIdx.x - request * heads;
  const int segment = decode_seg != nullptr ? decode_seg[request] : request, position = seg_pos0[segment];
  const int lowest = window > 0 ? max(0, position - window + 1) : 0, parts = min(most_parts, position / chunk - lowest / chunk + 1);
  T* dst = out + ((size_t)seg_q_start[segment] * heads + head) * dim;
  pdl_wait();
  auto state_of = [&](int part) { return ((size_t)part * requests + request) * heads + head; };
  float top = -INFINITY;
  for (int part = 0; part < parts; ++part) top = fmaxf(top, __ldcg(sums + state_of(part)).x);
  for (int d = threadIdx.x; d < dim; d += 128) {
    float total = 0.f, value = 0.f;
#pragma unroll 4
    for (int part = 0; part < parts; ++part) {
      const float2 state = __ldcg(sums + state_of(part));
      const float weight = state.x == -INFINITY ? 0.f : expf(state.x - top);
      total += state.y == state.y ? state.y * weight : state.y;
      value = fmaf(__ldcg(states + state_of(part) * dim + d), weight, value);
    }
    dst[d] = from_float<T>(value / total);
  }
}

template <typename T, int HEADS>
static int split_launch(const void* q, const void* k_pool, const void* v_pool, const float* k_scales, const float* v_scales, void* out,
                        const int* decode_seg, const int* seg_q_start, const int* seg_pos0, const int* block_table, const int* seg_slot,
                        int table_width, int requests, int heads, int kv_heads, int dim, int page_size, int block, int pool_pages, int window,
                        float scale, int chunk, int parts, uint8_t* scratch, cudaStream_t stream) {
  const int wide = ((dim + 3) / 4 | 1) * 4, group = heads / kv_heads;
  auto bytes = [](int w) { return sizeof(float) * ((size_t)(HEADS + 2 * QS_KEYS) * w + QS_KEYS * HEADS + 2 * QS_KEYS + 3 * HEADS); };
  static OncePerDevice once;
  const cudaError_t err = once([&] {
    return cudaFuncSetAttribute(attention_quantized_split_kernel<T, HEADS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes(QS_MAX_DIM + 4));
  });
  if (err != cudaSuccess) return (int)err;
  const size_t states = (size_t)parts * requests * heads;
  float2* sums = (float2*)scratch;
  float* outputs = (float*)(scratch + states * sizeof(float2));
  launch_kernel(attention_quantized_split_kernel<T, HEADS>, dim3(parts, requests * kv_heads, (group + HEADS - 1) / HEADS), dim3(QS_THREADS), bytes(wide),
                stream, (const T*)q, (const int8_t*)k_pool, (const int8_t*)v_pool, k_scales, v_scales, sums, outputs, decode_seg, seg_q_start, seg_pos0,
                block_table, seg_slot, table_width, requests, heads, kv_heads, dim, page_size, block, pool_pages, window, scale, chunk);
  launch_kernel(merge_quantized_split_kernel<T>, dim3(requests * heads), dim3(128), 0, stream, sums, outputs, (T*)out, decode_seg, seg_q_start, seg_pos0,
                requests, heads, dim, window, chunk, parts);
  return launch_status();
}

}  // namespace mlr

using namespace mlr;

MLR_DEFINE_PDL_SWITCH

// q, out: [rows, heads * dim], of which the rows of `requests` decoded tokens are attended (decode_seg: their segments, or null for segments 0, 1, ..);
// pools [pages, kv_heads, page_size, dim]; scales [pages, kv_heads, page_size / block].  Contexts are walked in parts of `chunk` keys (a multiple of 64),
// `parts` of them at most; scratch: parts * requests * heads * (dim + 2) floats.
MLR_EXPORT int mlr_attention_quantized_split(const void* q, const void* k_pool, const void* v_pool, const float* k_scales, const float* v_scales,
                                             void* out, const int* decode_seg, const int* seg_q_start, const int* seg_pos0, const int* block_table,
                                             const int* seg_slot, int table_width, int requests, int heads, int kv_heads, int dim, int page_size,
                                             int block, int pool_pages, int window, float scale, int chunk, int parts, void* scratch, int dtype,
                                             cudaStream_t stream) {
  if (requests == 0) return MLR_OK;
  if (requests < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || dim <= 0 || page_size <= 0 || block <= 0 || page_size % block ||
      table_width <= 0 || pool_pages <= 0 || chunk <= 0 || chunk % QS_KEYS || parts <= 0)
    return MLR_BAD_SIZE;
  if (dim > QS_MAX_DIM || (long long)requests * kv_heads > 65535 || (long long)requests * heads > 0x7fffffffLL) return MLR_TOO_LARGE;
  if ((uintptr_t)scratch & 15) return MLR_BAD_ALIGNMENT;
#define MLR_SPLIT(T_, HEADS_)                                                                                                                        \
  return split_launch<T_, HEADS_>(q, k_pool, v_pool, k_scales, v_scales, out, decode_seg, seg_q_start, seg_pos0, block_table, seg_slot, table_width, \
                                  requests, heads, kv_heads, dim, page_size, block, pool_pages, window, scale, chunk, parts, (uint8_t*)scratch, stream)
  const bool few = heads / kv_heads <= 4;
  if (dtype == MLR_F32) {
    if (few) MLR_SPLIT(float, 4);
    MLR_SPLIT(float, 8);
  }
  if (dtype == MLR_BF16) {
    if (few) MLR_SPLIT(bf16, 4);
    MLR_SPLIT(bf16, 8);
  }
#undef MLR_SPLIT
  return MLR_BAD_DTYPE;
}
