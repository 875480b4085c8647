// Causal attention of a ragged batch over keys and values in 8 bits with a scale for each block of tokens and kv head, on the
// CUDA cores in float32: every head size up to 256, every page and block size, both types of queries.
//
// k_j = kc_j * ks, v_j = vc_j * vs (ks, vs of j's block); row i of a request sees its keys max(0, p - window + 1) .. p;
// out = sum softmax(q.k * scale) v, by the running maximum and sum of a softmax, keys in tiles of 32 at absolute
// positions: a row's result does not depend on how the prompt was cut nor on the rest of the batch (decoded tokens have kernels of
// their own).  A key that a row does not see gives it nothing, whatever lies there (an infinite or NaN scale included).  Multiply-adds and
// the reads of shared memory beside them bound it; prompts of bfloat16 with head sizes 64 and 128 go to the tensor cores.
#include "common.cuh"

namespace mlr {

constexpr int QA_ROWS = 16;          // query rows per CTA, four per warp
constexpr int QA_KEYS = 32;          // one key per lane
constexpr int QA_MAX_DIM = 256;

template <typename T>
__global__ void __launch_bounds__(128)
attention_quantized_kernel(const T* q, const int8_t* k_pool, const int8_t* v_pool, const float* k_scales, const float* v_scales,
                           T* __restrict__ out, const int* __restrict__ tile_seg, const int* __restrict__ tile_row0,
                           const int* __restrict__ seg_q_start, const int* __restrict__ seg_q_len, const int* __restrict__ seg_pos0,
                           const int* __restrict__ block_table, const int* __restrict__ seg_slot, int table_width, int heads, int kv_heads,
                           int dim, int page_size, int block, int pool_pages, int window, float scale) {
  pdl_trigger();
  pdl_wait();
  extern __shared__ float shared[];
  float* q_rows = shared;                                   // [16][dim]
  float* k_tile = q_rows + QA_ROWS * dim;                   // [32][dim + 1]
  float* v_tile = k_tile + QA_KEYS * (dim + 1);             // [32][dim]
  float* p_tile = v_tile + QA_KEYS * dim;                   // [16][32]

  const int tile = blockIdx.x, head = blockIdx.y;
  const int kv_head = head / (heads / kv_heads);
  const int seg = tile_seg[tile], row0 = tile_row0[tile];
  const int q_start = seg_q_start[seg], q_len = seg_q_len[seg], pos0 = seg_pos0[seg];
  const int rows = min(QA_ROWS, q_len - row0);
  const int* table = block_table + (size_t)(seg_slot != nullptr ? seg_slot[seg] : seg) * table_width;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, per_page = page_size / block;

  for (int idx = threadIdx.x; idx < QA_ROWS * dim; idx += blockDim.x) {
    const int r = idx / dim, d = idx - r * dim;
    q_rows[idx] = r < rows ? to_float(q[((size_t)(q_start + row0 + r) * heads + head) * dim + d]) : 0.f;
  }
  float m[4], l[4], acc[4][QA_MAX_DIM / 32];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int c = 0; c < QA_MAX_DIM / 32; ++c) acc[i][c] = 0.f;
  }
  const int first_pos = pos0 + row0, last_pos = first_pos + rows - 1;
  const int lowest = window > 0 ? max(0, first_pos - window + 1) : 0;
  for (int k0 = lowest / QA_KEYS * QA_KEYS; k0 <= last_pos; k0 += QA_KEYS) {
    __syncthreads();
    for (int idx = threadIdx.x; idx < QA_KEYS * dim; idx += blockDim.x) {
      const int j = idx / dim, d = idx - j * dim, key = k0 + j, logical = key / page_size;
      const int page = key >= lowest && key <= last_pos && logical < table_width ? table[logical] : -1;
      float kv = 0.f, vv = 0.f;
      if (page >= 0 && page < pool_pages) {
        const int offset = key - logical * page_size;
        const size_t line = (size_t)page * kv_heads + kv_head, at = (line * page_size + offset) * dim + d;
        const size_t scale_at = line * per_page + offset / block;
        kv = (float)k_pool[at] * k_scales[scale_at];
        vv = (float)v_pool[at] * v_scales[scale_at];
      }
      k_tile[j * (dim + 1) + d] = kv;
      v_tile[j * dim + d] = vv;
    }
    __syncthreads();
    const int key = k0 + lane;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = warp * 4 + i;
      if (r >= rows) continue;                // uniform per warp
      const int p = first_pos + r;
      const bool visible = key <= p && (window <= 0 || key > p - window);
      float s = 0.f;
      const float* qr = q_rows + r * dim;
      const float* kr = k_tile + lane * (dim + 1);
      for (int d = 0; d < dim; ++d) s = fmaf(qr[d], kr[d], s);
      s = visible ? s * scale : -INFINITY;
      // a score that is no number makes the row none (fmaxf passes over it)
      const float m_new = fmaxf(m[i], warp_max(s));
      const bool any_nan = __any_sync(0xffffffffu, isnan(s));
      if (m_new == -INFINITY && !any_nan) continue;     // nothing visible yet
      const float alpha = m[i] == -INFINITY ? 0.f : expf(m[i] - m_new);
      const float prob = visible ? expf(s - m_new) : 0.f;
      l[i] = l[i] * alpha + warp_sum(prob);
      m[i] = m_new;
      float* pw = p_tile + r * QA_KEYS;
      pw[lane] = prob;
      __syncwarp();
      // the keys of this tile that the row sees
      const int from = window > 0 ? max(0, p - window + 1 - k0) : 0, until = min(QA_KEYS, p - k0 + 1);
#pragma unroll
      for (int c = 0; c < QA_MAX_DIM / 32; ++c) {
        const int d = lane + 32 * c;
        if (d < dim) {
          float a = acc[i][c] * alpha;
          for (int j = from; j < until; ++j) a = fmaf(pw[j], v_tile[j * dim + d], a);
          acc[i][c] = a;
        }
      }
      __syncwarp();
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = warp * 4 + i;
    if (r >= rows) continue;
    const float inv = 1.f / l[i];
    T* dst = out + ((size_t)(q_start + row0 + r) * heads + head) * dim;
#pragma unroll
    for (int c = 0; c < QA_MAX_DIM / 32; ++c) {
      const int d = lane + 32 * c;
      if (d < dim) dst[d] = from_float<T>(acc[i][c] * inv);
    }
  }
}

template <typename T>
static int quantized_launch(const void* q, const void* k_pool, const void* v_pool, const float* k_scales, const float* v_scales, void* out,
                            const int* tile_seg, const int* tile_row0, const int* seg_q_start, const int* seg_q_len, const int* seg_pos0,
                            const int* block_table, const int* seg_slot, int table_width, int tiles, int heads, int kv_heads, int dim,
                            int page_size, int block, int pool_pages, int window, float scale, cudaStream_t stream) {
  const size_t shared = sizeof(float) * ((size_t)QA_ROWS * dim + (size_t)QA_KEYS * (2 * dim + 1) + QA_ROWS * QA_KEYS);
  static OncePerDevice once;
  const size_t most = sizeof(float) * ((size_t)QA_ROWS * QA_MAX_DIM + (size_t)QA_KEYS * (2 * QA_MAX_DIM + 1) + QA_ROWS * QA_KEYS);
  const cudaError_t err = once([&] { return cudaFuncSetAttribute(attention_quantized_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most); });
  if (err != cudaSuccess) return (int)err;
  launch_kernel(attention_quantized_kernel<T>, dim3(tiles, heads), dim3(128), shared, stream, (const T*)q, (const int8_t*)k_pool,
                (const int8_t*)v_pool, k_scales, v_scales, (T*)out, tile_seg, tile_row0, seg_q_start, seg_q_len, seg_pos0, block_table, seg_slot,
                table_width, heads, kv_heads, dim, page_size, block, pool_pages, window, scale);
  return launch_status();
}

}  // namespace mlr

using namespace mlr;

MLR_DEFINE_PDL_SWITCH

// q, out: [rows, heads * dim]; pools [pages, kv_heads, page_size, dim], scales [pages, kv_heads, page_size / block]; tile_seg / tile_row0:
// one entry per CTA tile of up to 16 rows of one segment; window <= 0: every earlier key is visible.
MLR_EXPORT int mlr_attention_quantized(const void* q, const void* k_pool, const void* v_pool, const float* k_scales, const float* v_scales,
                                       void* out, const int* tile_seg, const int* tile_row0, const int* seg_q_start, const int* seg_q_len,
                                       const int* seg_pos0, const int* block_table, const int* seg_slot, int table_width, int tiles, int heads,
                                       int kv_heads, int dim, int page_size, int block, int pool_pages, int window, float scale, int dtype,
                                       cudaStream_t stream) {
  if (tiles == 0) return MLR_OK;
  if (tiles < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || dim <= 0 || page_size <= 0 || block <= 0 || page_size % block ||
      table_width <= 0 || pool_pages <= 0)
    return MLR_BAD_SIZE;
  if (dim > QA_MAX_DIM || heads > 65535) return MLR_TOO_LARGE;
  if (dtype == MLR_F32)
    return quantized_launch<float>(q, k_pool, v_pool, k_scales, v_scales, out, tile_seg, tile_row0, seg_q_start, seg_q_len, seg_pos0, block_table,
                                   seg_slot, table_width, tiles, heads, kv_heads, dim, page_size, block, pool_pages, window, scale, stream);
  if (dtype == MLR_BF16)
    return quantized_launch<bf16>(q, k_pool, v_pool, k_scales, v_scales, out, tile_seg, tile_row0, seg_q_start, seg_q_len, seg_pos0, block_table,
                                  seg_slot, table_width, tiles, heads, kv_heads, dim, page_size, block, pool_pages, window, scale, stream);
  return MLR_BAD_DTYPE;
}
