// Keys and values of a cache in 8 bits: whole numbers between -127 and 127, with a 32-bit scale for each block of `block`
// tokens of a page and kv head; a number stands for code * scale.
//
//   new tokens   s = max(s of the block if it holds tokens already, amax / 127), amax over the block's new tokens; code =
//                x / s rounded to the nearest whole number, ties to even.  Tokens that the block held before are
//                rounded to the new scale where it grew.  Codes behind the block's last token stay as they were.
//   exactness    code is the rounding of the exact quotient, so that the result depends on no order and no instruction:
//                the product with 1 / s (with s before / s) is off by less than 2^-15 of a step, and a quotient that lies within
//                2^-14 of a tie is decided in 64 bits, where the tie itself is exact and nothing else rounds to it.
//   not finite   a block with an infinite or NaN entry gets the scale NaN: whoever attends to it gets NaN, as from the
//                entry itself.
//
// A CTA of four warps looks at `span` rows (of one kv head and pool) and takes the blocks whose first new row is among them, with all their
// new rows, which follow one another in a step: one or two of them, as of a prompt, with all its warps, more, as of decoded tokens,
// with a warp each.  The span is the least of 1, 4 and 16 that leaves no more CTAs than the device holds at once: few rows get a CTA
// each, and of a prompt few CTAs find nothing.  What is read is held in registers between the search for the largest number and the
// rounding, as far as two pieces per thread go (16 rows of 128 bfloat16); the rest is read twice.  Reads that wait for one another bound
// it, not bytes: 2,056 rows of 4 kv heads of 128 take 20 us with the pages' dequantizing, 64 rows 9.
#include "common.cuh"

namespace mlr {

constexpr int QUANT_WARPS = 4, QUANT_THREADS = QUANT_WARPS * 32;

// x / scale, or code * older / newer, to the nearest whole number in 64 bits; 0 for a scale of zero or NaN.
__device__ __forceinline__ int nearest(double x, float scale) {
  return scale > 0.f ? max(-127, min(127, (int)rint(x / (double)scale))) : 0;
}
// The same of a product t = x * factor in 32 bits, as the low byte of the result; `off` becomes the largest distance from the whole
// number, which tells a quotient next to a tie.
__device__ __forceinline__ unsigned rounded(float x, float factor, float* off) {
  constexpr float RAISE = 12582912.f;      // 1.5 * 2^23: whole numbers from here on, two's complement in the low bits
  const float raised = fmaf(x, factor, RAISE);
  *off = fmaxf(*off, fabsf(fmaf(x, factor, RAISE - raised)));
  return __float_as_uint(raised);
}
// VEC numbers to codes.  `regular`: the factor is an ordinary number and the numbers are at most 127 steps.
template <int VEC, typename Exact>
__device__ __forceinline__ void round_all(const float (&x)[VEC], float factor, bool regular, int8_t (&codes)[VEC], Exact&& exact) {
  float off = regular ? 0.f : 1.f;
  unsigned raised[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) raised[e] = rounded(x[e], factor, &off);
  if (off > 0.49993896484375f) {           // within 2^-14 of a tie: in 64 bits
#pragma unroll 1
    for (int e = 0; e < VEC; ++e) codes[e] = (int8_t)exact(e);
    return;
  }
  if constexpr (VEC >= 4) {
#pragma unroll
    for (int w = 0; w < VEC / 4; ++w)
      reinterpret_cast<uint32_t*>(codes)[w] = __byte_perm(__byte_perm(raised[4 * w], raised[4 * w + 1], 0x0040),
                                                          __byte_perm(raised[4 * w + 2], raised[4 * w + 3], 0x0040), 0x5410);
  } else {
    codes[0] = (int8_t)raised[0];
  }
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
__global__ void __launch_bounds__(QUANT_THREADS)
quantize_kv_kernel(const T* key, long long key_stride, const T* value, long long value_stride, const long long* slots, int8_t* k_pool,
                   int8_t* v_pool, float* k_scales, float* v_scales, int rows, int kv_heads, int dim, int page_size, int block, int span,
                   long long total_slots) {
  pdl_trigger();
  __shared__ unsigned tops[QUANT_WARPS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int row_group = blockIdx.x / (2 * kv_heads), within = blockIdx.x - row_group * 2 * kv_heads;
  const int head = within >> 1, row0 = row_group * span;
  pdl_wait();
  // lane i of each warp: row row0 + i, a block's first new row or not (slots of the pool fit 31 bits)
  const bool here = lane < span && row0 + lane < rows;
  const long long looked_at = here ? slots[row0 + lane] : -1, previous = here && row0 + lane > 0 ? slots[row0 + lane - 1] : -1;
  const bool inside = looked_at >= 0 && looked_at < total_slots;
  const unsigned my_slot = inside ? (unsigned)looked_at : 0u, my_held = my_slot % (unsigned)block;
  unsigned firsts = __ballot_sync(0xffffffffu, inside && (my_held == 0u || previous != looked_at - 1));
  const bool together = __popc(firsts) <= 2;
  const int thread = together ? threadIdx.x : lane, threads = together ? QUANT_THREADS : 32;
  for (int place = 0; firsts != 0u; firsts &= firsts - 1u, ++place) {
    if (!together && place % QUANT_WARPS != warp) continue;
    const int from = __ffs(firsts) - 1, row = row0 + from;
    const int slot = (int)__shfl_sync(0xffffffffu, my_slot, from);
    const int held = (int)__shfl_sync(0xffffffffu, my_held, from);      // tokens of the block before this row
    int count = 1;                                                   // its new rows
    for (int first = 1; first < block - held; first += 32) {
      const int i = first + lane;
      const bool next = i < block - held && row + i < rows && slots[row + i] == (long long)slot + i;
      const unsigned run = __ballot_sync(0xffffffffu, next);
      const int more = run == 0xffffffffu ? 32 : __ffs(~run) - 1;
      count += more;
      if (more < 32) break;
    }
    const bool values = within & 1;
    const T* src = (values ? value : key) + (size_t)head * dim;
    const long long stride = values ? value_stride : key_stride;
    const int page = (unsigned)slot / (unsigned)page_size, offset = slot - page * page_size, per_page = page_size / block;
    int8_t* head_codes = (values ? v_pool : k_pool) + ((size_t)page * kv_heads + head) * page_size * dim;
    float* scale_at = (values ? v_scales : k_scales) + ((size_t)page * kv_heads + head) * per_page + offset / block;

    const int pieces = dim / VEC, total = count * pieces;
    constexpr int KEPT = 2;
    auto at = [&](int i) {
      const int r = i / pieces, c = i - r * pieces;
      return load_piece<T, VEC>(src + (size_t)(row + r) * stride + c * VEC);
    };
    RowPiece<T, VEC> kept[KEPT];
#pragma unroll
    for (int j = 0; j < KEPT; ++j)
      if (thread + threads * j < total) kept[j] = at(thread + threads * j);
    const float older = held > 0 ? *scale_at : 0.f;
    unsigned top = 0;                       // largest magnitude as bits: infinities and NaN lie above every number
    auto look = [&](const RowPiece<T, VEC>& piece) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) top = max(top, __float_as_uint(to_float(piece.v[e])) & 0x7fffffffu);
    };
#pragma unroll
    for (int j = 0; j < KEPT; ++j)
      if (thread + threads * j < total) look(kept[j]);
    for (int i = thread + threads * KEPT; i < total; i += threads) look(at(i));
    top = __reduce_max_sync(0xffffffffu, top);
    __syncwarp();                           // (its scale has been read)
    if (together) {
      __syncthreads();                      // (the block before has been read out of `tops`)
      if (lane == 0) tops[warp] = top;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < QUANT_WARPS; ++w) top = max(top, tops[w]);
    }
    const bool finite = top < 0x7f800000u;
    float scale = finite ? __fdiv_rn(__uint_as_float(top), 127.f) : __int_as_float(0x7fffffff);
    if (held > 0) scale = isnan(scale) || isnan(older) ? __int_as_float(0x7fffffff) : fmaxf(scale, older);
    const float inverse = __fdiv_rn(1.f, scale);
    const bool regular = scale >= 7.888609e-31f && scale < INFINITY;      // 2^-100: the inverse has all its bits

    if (held > 0 && !(scale == older)) {      // the tokens before, rounded to the scale that grew
      const float ratio = __fdiv_rn(older, scale);
      int8_t* first = head_codes + (size_t)(offset - held) * dim;
      for (int i = thread; i < held * pieces; i += threads) {
        alignas(8) int8_t codes[VEC];
        if constexpr (VEC == 8) *reinterpret_cast<uint2*>(codes) = *reinterpret_cast<const uint2*>(first + i * VEC);
        else if constexpr (VEC == 4) *reinterpret_cast<uint32_t*>(codes) = *reinterpret_cast<const uint32_t*>(first + i * VEC);
        else codes[0] = first[i];
        float x[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) x[e] = (float)codes[e];
        int8_t before[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) before[e] = codes[e];
        round_all<VEC>(x, ratio, regular, codes, [&](int e) { return nearest((double)before[e] * (double)older, scale); });
        store_codes<VEC>(first + i * VEC, codes);
      }
    }
    auto round_off = [&](int i, const RowPiece<T, VEC>& piece) {
      alignas(8) int8_t codes[VEC];
      float x[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) x[e] = to_float(piece.v[e]);
      round_all<VEC>(x, inverse, regular, codes, [&](int e) { return nearest((double)to_float(piece.v[e]), scale); });
      store_codes<VEC>(head_codes + (size_t)offset * dim + (size_t)i * VEC, codes);      // rows of a head lie one behind the other
    };
#pragma unroll
    for (int j = 0; j < KEPT; ++j)
      if (thread + threads * j < total) round_off(thread + threads * j, kept[j]);
    for (int i = thread + threads * KEPT; i < total; i += threads) round_off(i, at(i));
    if (thread == 0) *scale_at = scale;
  }
}

// What the codes of pages stand for: codes * scales.  A CTA per page and kv head, its keys by the first half of the threads, its values by
// the second; VEC codes at a time.  A page outside the pool gives zeros.
template <typename T, int VEC>
__global__ void __launch_bounds__(256)
dequantize_pages_kernel(const int8_t* k_pool, const int8_t* v_pool, const float* k_scales, const float* v_scales, const int* pages,
                        T* __restrict__ key, T* __restrict__ value, int kv_heads, int dim, int page_size, int block, int pool_pages) {
  pdl_trigger();
  const int head = blockIdx.x, which = blockIdx.y;
  const bool values = threadIdx.x >= 128;
  pdl_wait();
  const int page = pages[which];
  const bool known = page >= 0 && page < pool_pages;
  const size_t line = known ? (size_t)page * kv_heads + head : 0;
  const int8_t* codes = (values ? v_pool : k_pool) + line * page_size * dim;
  const float* scales = (values ? v_scales : k_scales) + line * (page_size / block);
  T* dst = (values ? value : key) + ((size_t)which * kv_heads + head) * page_size * dim;
  const int total = page_size * dim / VEC, per_block = block * dim / VEC;      // (a piece lies within a row)
  for (int i = threadIdx.x & 127; i < total; i += 128) {
    const float scale = known ? scales[i / per_block] : 0.f;
    alignas(16) int8_t in[VEC];
    if constexpr (VEC == 16) *reinterpret_cast<uint4*>(in) = __ldcg(reinterpret_cast<const uint4*>(codes) + i);
    else in[0] = codes[i];
    alignas(16) T out[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) out[e] = from_float<T>(known ? (float)in[e] * scale : 0.f);
    if constexpr (VEC == 16) {
      constexpr int STORES = VEC * sizeof(T) / 16;
#pragma unroll
      for (int e = 0; e < STORES; ++e) reinterpret_cast<uint4*>(dst)[(size_t)i * STORES + e] = reinterpret_cast<const uint4*>(out)[e];
    } else {
      dst[i] = out[0];
    }
  }
}

template <typename T, int WIDE>
static int quantize_launch(bool wide, const void* key, long long key_stride, const void* value, long long value_stride, const long long* slots,
                           void* k_pool, void* v_pool, float* k_scales, float* v_scales, int rows, int kv_heads, int dim, int page_size,
                           int block, long long total_slots, cudaStream_t stream) {
  int span = 1;
  while (span < 16 && (long long)((rows + span - 1) / span) * 2 * kv_heads > 16ll * sm_count()) span *= 4;
  const long long blocks = (long long)((rows + span - 1) / span) * 2 * kv_heads;
  if (blocks > 0x7fffffffLL) return MLR_TOO_LARGE;
  auto kernel = wide ? quantize_kv_kernel<T, WIDE> : quantize_kv_kernel<T, 1>;
  launch_kernel(kernel, dim3((unsigned)blocks), dim3(QUANT_THREADS), 0, stream, (const T*)key, key_stride, (const T*)value, value_stride,
                slots, (int8_t*)k_pool, (int8_t*)v_pool, k_scales, v_scales, rows, kv_heads, dim, page_size, block, span, total_slots);
  return launch_status();
}

template <typename T>
static int dequantize_launch(bool wide, const void* k_pool, const void* v_pool, const float* k_scales, const float* v_scales, const int* pages,
                             void* key, void* value, int count, int kv_heads, int dim, int page_size, int block, int pool_pages,
                             cudaStream_t stream) {
  auto kernel = wide ? dequantize_pages_kernel<T, 16> : dequantize_pages_kernel<T, 1>;
  constexpr int MOST = 65535;
  for (int first = 0; first < count; first += MOST) {
    const size_t at = (size_t)first * kv_heads * page_size * dim;
    launch_kernel(kernel, dim3(kv_heads, count - first < MOST ? count - first : MOST), dim3(256), 0, stream, (const int8_t*)k_pool,
                  (const int8_t*)v_pool, k_scales, v_scales, pages + first, (T*)key + at, (T*)value + at, kv_heads, dim, page_size, block, pool_pages);
  }
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
  if ((long long)page_size * dim > 0x7fffffffLL) return MLR_TOO_LARGE;
  const bool wide = dim % 16 == 0 && (((uintptr_t)key | (uintptr_t)value | (uintptr_t)k_pool | (uintptr_t)v_pool) & 15) == 0;
  if (dtype == MLR_F32)
    return dequantize_launch<float>(wide, k_pool, v_pool, k_scales, v_scales, pages, key, value, count, kv_heads, dim, page_size, block, pool_pages,
                                    stream);
  if (dtype == MLR_BF16)
    return dequantize_launch<bf16>(wide, k_pool, v_pool, k_scales, v_scales, pages, key, value, count, kv_heads, dim, page_size, block, pool_pages,
                                   stream);
  return MLR_BAD_DTYPE;
}
