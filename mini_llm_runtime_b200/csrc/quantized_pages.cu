// Keys and values of a cache in 8 bits: whole numbers between -127 and 127, with a 32-bit scale for each block of `block`
// tokens of a page and kv head; a number stands for code * scale.
//
//   new tokens   s = max(s of the block if it holds tokens already, amax / 127), amax over the block's new tokens; code =
//                x / s rounded to the nearest whole number, ties to even.  Tokens that the block held before are
//                rounded to the new scale where it grew.  Codes behind the block's last token stay as they were.
//   exactness    code is the rounding of the exact quotient, so that the result depends on no order and no instruction:
//                the product with 1 / s is off by less than 2^-16 of a step, and a quotient that lies within 2^-12 of a tie is
//                decided in 64 bits, where the tie itself is exact and nothing else rounds to it.
//   not finite   a block with an infinite or NaN entry gets the scale NaN: whoever attends to it gets NaN, as from the
//                entry itself.
//
// One warp per block, kv head and pool: the warp of the block's first new row takes all its new rows (they follow one
// another in a step), the warps of the other rows end at once.  Bytes bound it: each row is read twice, the
// second time from the L1.
#include "common.cuh"

namespace mlr {

constexpr int QUANT_WARPS = 8;

__device__ __forceinline__ int quantized(float x, float scale, float inverse) {
  const float t = x * inverse;
  const float whole = rintf(t);
  // within 2^-12 of a tie (or no number at all: a scale whose inverse is infinite)
  if (!(fabsf(fabsf(t - whole) - 0.5f) > 0.000244140625f)) {
    if (!(scale > 0.f)) return 0;
    return max(-127, min(127, (int)rint((double)x / (double)scale)));
  }
  return max(-127, min(127, (int)whole));
}
__device__ __forceinline__ int requantized(int code, float older, float newer, float ratio) {
  const float t = (float)code * ratio;
  const float whole = rintf(t);
  if (!(fabsf(fabsf(t - whole) - 0.5f) > 0.000244140625f)) {
    if (!(newer > 0.f)) return 0;
    return (int)rint((double)code * (double)older / (double)newer);
  }
  return (int)whole;
}

// VEC entries at a time: 16 bytes of bfloat16 or float32, or one entry.
template <typename T, int VEC> struct RowPiece { T v[VEC]; };
template <typename T, int VEC>
__device__ __forceinline__ RowPiece<T, VEC> load_piece(const T* p) {
  RowPiece<T, VEC> piece;
  if constexpr (VEC > 1) *reinterpret_cast<uint4*>(&piece) = __ldcg(reinterpret_cast<const uint4*>(p));
  else piece.v[0] = *p;
  return piece;
}
template <int VEC>
__device__ __forceinline__ void store_codes(int8_t* p, const int8_t (&codes)[VEC]) {
  if constexpr (VEC == 8) *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(codes);
  else if constexpr (VEC == 4) *reinterpret_cast<uint32_t*>(p) = *reinterpret_cast<const uint32_t*>(codes);
  else *p = codes[0];
}

template <typename T, int VEC>
__global__ void __launch_bounds__(QUANT_WARPS * 32)
quantize_kv_kernel(const T* key, long long key_stride, const T* value, long long value_stride, const long long* slots, int8_t* k_pool,
                   int8_t* v_pool, float* k_scales, float* v_scales, int rows, int kv_heads, int dim, int page_size, int block,
                   long long total_slots) {
  pdl_trigger();
  const int lane = threadIdx.x & 31;
  const long long unit = (long long)blockIdx.x * QUANT_WARPS + (threadIdx.x >> 5);
  const int row = (int)(unit / (2 * kv_heads)), within = (int)(unit - (long long)row * 2 * kv_heads);
  const int head = within >> 1;
  pdl_wait();
  if (row >= rows) return;
  const long long slot = slots[row];
  if (slot < 0 || slot >= total_slots) return;
  const long long cell = slot / block;
  const int held = (int)(slot - cell * block);                     // tokens of the block before this row
  if (row > 0 && held > 0 && slots[row - 1] == slot - 1) return;      // not the block's first new row
  int count = 1;                                                   // its new rows
  for (int first = 1; first < block - held; first += 32) {
    const int i = first + lane;
    const bool next = i < block - held && row + i < rows && slots[row + i] == slot + i;
    const unsigned run = __ballot_sync(0xffffffffu, next);
    const int more = run == 0xffffffffu ? 32 : __ffs(~run) - 1;
    count += more;
    if (more < 32) break;
  }
  const bool values = within & 1;
  const T* src = (values ? value : key) + (size_t)head * dim;
  const long long stride = values ? value_stride : key_stride;
  const long long page = slot / page_size;
  const int offset = (int)(slot - page * page_size), per_page = page_size / block;
  int8_t* head_codes = (values ? v_pool : k_pool) + ((size_t)page * kv_heads + head) * page_size * dim;
  float* scale_at = (values ? v_scales : k_scales) + ((size_t)page * kv_heads + head) * per_page + offset / block;

  const int pieces = dim / VEC, total = count * pieces;
  unsigned top = 0;                       // largest magnitude as bits: infinities and NaN lie above every number
  for (int i = lane; i < total; i += 32) {
    const int r = i / pieces, c = i - r * pieces;
    const RowPiece<T, VEC> piece = load_piece<T, VEC>(src + (size_t)(row + r) * stride + c * VEC);
#pragma unroll
    for (int e = 0; e < VEC; ++e) top = max(top, __float_as_uint(to_float(piece.v[e])) & 0x7fffffffu);
  }
  top = __reduce_max_sync(0xffffffffu, top);
  const bool finite = top < 0x7f800000u;
  float scale = finite ? __fdiv_rn(__uint_as_float(top), 127.f) : __int_as_float(0x7fffffff);
  const float older = held > 0 ? *scale_at : 0.f;
  if (held > 0) scale = isnan(scale) || isnan(older) ? __int_as_float(0x7fffffff) : fmaxf(scale, older);
  __syncwarp();
  const float inverse = __fdiv_rn(1.f, scale);

  if (held > 0 && !(scale == older)) {      // the tokens before, rounded to the scale that grew
    const float ratio = __fdiv_rn(older, scale);
    int8_t* first = head_codes + (size_t)(offset - held) * dim;
    for (int i = lane; i < held * pieces; i += 32) {
      int8_t codes[VEC];
      if constexpr (VEC == 8) *reinterpret_cast<uint2*>(codes) = *reinterpret_cast<const uint2*>(first + i * VEC);
      else if constexpr (VEC == 4) *reinterpret_cast<uint32_t*>(codes) = *reinterpret_cast<const uint32_t*>(first + i * VEC);
      else codes[0] = first[i];
#pragma unroll
      for (int e = 0; e < VEC; ++e) codes[e] = (int8_t)requantized(codes[e], older, scale, ratio);
      store_codes<VEC>(first + i * VEC, codes);
    }
  }
  for (int i = lane; i < total; i += 32) {
    const int r = i / pieces, c = i - r * pieces;
    const RowPiece<T, VEC> piece = load_piece<T, VEC>(src + (size_t)(row + r) * stride + c * VEC);
    int8_t codes[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) codes[e] = (int8_t)quantized(to_float(piece.v[e]), scale, inverse);
    store_codes<VEC>(head_codes + (size_t)(offset + r) * dim + c * VEC, codes);
  }
  if (lane == 0) *scale_at = scale;
}

// What the codes of pages stand for: out[i] = codes[page i] * scales, a thread per VEC entries.  A page outside the pool gives zeros.
template <typename T, int VEC>
__global__ void __launch_bounds__(256)
dequantize_pages_kernel(const int8_t* k_pool, const int8_t* v_pool, const float* k_scales, const float* v_scales, const int* pages,
                        T* __restrict__ key, T* __restrict__ value, long long total, int kv_heads, int dim, int page_size, int block,
                        int pool_pages) {
  pdl_trigger();
  pdl_wait();
  const long long index = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (index >= total) return;
  const int pieces = dim / VEC;
  const long long token = index / pieces, head = token / page_size, which = head / kv_heads;
  const int c = (int)(index - token * pieces), offset = (int)(token - head * page_size);
  const int page = pages[which];
#pragma unroll
  for (int values = 0; values < 2; ++values) {
    T out[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) out[e] = from_float<T>(0.f);
    if (page >= 0 && page < pool_pages) {
      const size_t line = (size_t)page * kv_heads + (size_t)(head - which * kv_heads);
      const float scale = (values ? v_scales : k_scales)[line * (page_size / block) + offset / block];
      const int8_t* src = (values ? v_pool : k_pool) + (line * page_size + offset) * dim + c * VEC;
      int8_t codes[VEC];
      if constexpr (VEC == 8) *reinterpret_cast<uint2*>(codes) = *reinterpret_cast<const uint2*>(src);
      else if constexpr (VEC == 4) *reinterpret_cast<uint32_t*>(codes) = *reinterpret_cast<const uint32_t*>(src);
      else codes[0] = *src;
#pragma unroll
      for (int e = 0; e < VEC; ++e) out[e] = from_float<T>((float)codes[e] * scale);
    }
    T* dst = (values ? value : key) + index * VEC;
    if constexpr (VEC * sizeof(T) == 16) *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(out);
    else dst[0] = out[0];
  }
}

template <typename T, int WIDE>
static int quantize_launch(bool wide, const void* key, long long key_stride, const void* value, long long value_stride, const long long* slots,
                           void* k_pool, void* v_pool, float* k_scales, float* v_scales, int rows, int kv_heads, int dim, int page_size,
                           int block, long long total_slots, cudaStream_t stream) {
  const long long units = (long long)rows * 2 * kv_heads, blocks = (units + QUANT_WARPS - 1) / QUANT_WARPS;
  if (blocks > 0x7fffffffLL) return MLR_TOO_LARGE;
  auto kernel = wide ? quantize_kv_kernel<T, WIDE> : quantize_kv_kernel<T, 1>;
  launch_kernel(kernel, dim3((unsigned)blocks), dim3(QUANT_WARPS * 32), 0, stream, (const T*)key, key_stride, (const T*)value, value_stride,
                slots, (int8_t*)k_pool, (int8_t*)v_pool, k_scales, v_scales, rows, kv_heads, dim, page_size, block, total_slots);
  return launch_status();
}

template <typename T, int WIDE>
static int dequantize_launch(bool wide, const void* k_pool, const void* v_pool, const float* k_scales, const float* v_scales, const int* pages,
                             void* key, void* value, int count, int kv_heads, int dim, int page_size, int block, int pool_pages,
                             cudaStream_t stream) {
  const long long total = (long long)count * kv_heads * page_size * (dim / (wide ? WIDE : 1)), blocks = (total + 255) / 256;
  if (blocks > 0x7fffffffLL) return MLR_TOO_LARGE;
  auto kernel = wide ? dequantize_pages_kernel<T, WIDE> : dequantize_pages_kernel<T, 1>;
  launch_kernel(kernel, dim3((unsigned)blocks), dim3(256), 0, stream, (const int8_t*)k_pool, (const int8_t*)v_pool, k_scales, v_scales, pages,
                (T*)key, (T*)value, total, kv_heads, dim, page_size, block, pool_pages);
  return launch_status();
}

}  // namespace mlr

using namespace mlr;

MLR_DEFINE_PDL_SWITCH

// key, value: rows of kv_heads * dim entries spaced key_stride / value_stride entries apart; slots: int64 [rows], page * page_size +
// offset (rows with a slot outside the pool are passed over); pools [pages, kv_heads, page_size, dim]; scales [pages, kv_heads, page_size / block].
MLR_EXPORT int mlr_quantize_kv(const void* key, long long key_stride, const void* value, long long value_stride, const long long* slots,
                               void* k_pool, void* v_pool, float* k_scales, float* v_scales, int rows, int kv_heads, int dim, int page_size,
                               int block, int pool_pages, int dtype, cudaStream_t stream) {
  if (rows == 0) return MLR_OK;
  if (rows < 0 || kv_heads <= 0 || dim <= 0 || page_size <= 0 || block <= 0 || page_size % block || pool_pages <= 0) return MLR_BAD_SIZE;
  const int size = dtype == MLR_F32 ? 4 : 2, wide = 16 / size;
  const bool fits = dim % wide == 0 && key_stride % wide == 0 && value_stride % wide == 0 && (((uintptr_t)key | (uintptr_t)value) & 15) == 0 &&
                    (((uintptr_t)k_pool | (uintptr_t)v_pool) & 7) == 0;
  const long long total_slots = (long long)pool_pages * page_size;
  if (dtype == MLR_F32)
    return quantize_launch<float, 4>(fits, key, key_stride, value, value_stride, slots, k_pool, v_pool, k_scales, v_scales, rows, kv_heads, dim,
                                     page_size, block, total_slots, stream);
  if (dtype == MLR_BF16)
    return quantize_launch<bf16, 8>(fits, key, key_stride, value, value_stride, slots, k_pool, v_pool, k_scales, v_scales, rows, kv_heads, dim,
                                    page_size, block, total_slots, stream);
  return MLR_BAD_DTYPE;
}

// key, value: [count, kv_heads, page_size, dim]; pages: int32 [count].
MLR_EXPORT int mlr_dequantize_pages(const void* k_pool, const void* v_pool, const float* k_scales, const float* v_scales, const int* pages,
                                    void* key, void* value, int count, int kv_heads, int dim, int page_size, int block, int pool_pages, int dtype,
                                    cudaStream_t stream) {
  if (count == 0) return MLR_OK;
  if (count < 0 || kv_heads <= 0 || dim <= 0 || page_size <= 0 || block <= 0 || page_size % block || pool_pages <= 0) return MLR_BAD_SIZE;
  const int size = dtype == MLR_F32 ? 4 : 2, wide = 16 / size;
  const bool fits = dim % wide == 0 && (((uintptr_t)key | (uintptr_t)value) & 15) == 0 && (((uintptr_t)k_pool | (uintptr_t)v_pool) & 7) == 0;
  if (dtype == MLR_F32)
    return dequantize_launch<float, 4>(fits, k_pool, v_pool, k_scales, v_scales, pages, key, value, count, kv_heads, dim, page_size, block,
                                       pool_pages, stream);
  if (dtype == MLR_BF16)
    return dequantize_launch<bf16, 8>(fits, k_pool, v_pool, k_scales, v_scales, pages, key, value, count, kv_heads, dim, page_size, block,
                                      pool_pages, stream);
  return MLR_BAD_DTYPE;
}
