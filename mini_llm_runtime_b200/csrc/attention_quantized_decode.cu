// Decoded tokens over keys and values in 8 bits (a scale for each block of tokens and kv head), queries in bfloat16, head sizes 64
// and 128, up to 16 query heads per kv head, pages of a power of two of at least 16 tokens.
//
//   x_j = (q . kc_j) ks_j scale log2 e + log2 vs_j,  M = max x_j,  p_j = 2^(x_j - M),  out = sum p_j vc_j / sum (p_j / vs_j)
// so that the weights that multiply the codes vc_j carry the values' scales and lie near (0, 1] whatever the scales are: they
// fit float16, whose 11 bits round them less than bfloat16 would.  (M follows the largest x in steps of more than 2^8: most tiles
// then need no maximum over their keys, only the look whether one has passed it.)  Codes are exact in float16, and queries are
// there after a power of two per head has brought the largest near one.
//
// Reading 2 * dim bytes per key and kv head is what bounds it.  A warp takes 16 keys (head size 64: 32) at a time and has three such
// tiles on their way.  The heads of a group are the narrow side of the products (n = 8), keys and dimensions the wide one:
//   scores^T [16 keys x 8 heads] = K [16 x dim] Q^T,   out^T [dim x 8 heads] += V^T [dim x 16 keys] P^T
// The order of the dimensions within a product is free, so a thread asks for 16 bytes of a key that are four steps' operands, and
// for 16 (8) dimensions of four keys that are eight (four) tiles' operands: every thread copies asynchronously just the bytes it reads
// itself, conflict-free and without a barrier.  A byte becomes a float16 by a byte permutation: 1024 + 128 + code.  Of the values
// the 1152 is subtracted (exactly); of the keys it is left in, and 1152 times the sum of the query taken off where the scores'
// sums begin (32 bits: 1152 sum |q| 2^-24 beside scores of up to 127 sum |q|).
//
// The keys of all requests and kv heads form one line that the CTAs share evenly, whatever the contexts: a CTA's share may
// end one request's keys and begin another's.  Each beginning counts as QD_BEGIN tiles more, about what it costs.  Pairs of a request and a kv head that more than one CTA walks are merged by the
// CTA that ends last, in the order of the CTAs.
#include <cuda_fp16.h>

#include "common.cuh"

namespace mlr {

constexpr int QD_WARPS = 8, QD_THREADS = QD_WARPS * 32, QD_STAGES = 3;
constexpr int QD_MOST_REQUESTS = 2048;       // whose tiles a CTA counts
constexpr int QD_BEGIN = 24;                 // what the beginning of a pair of a request and a kv head costs a CTA, in tiles
constexpr int QD_LEAST_SHARE = QD_BEGIN + 16;      // of a CTA, at least: two tiles per warp
// The largest exponent follows the maximum in steps of more than this; weights up to 2^8 are far from float16's end.
constexpr float QD_LAZY = 8.f;

template <int D>
struct QdShape {
  static constexpr int SUB = 128 / D;                 // groups of 16 keys in a tile
  static constexpr int KEYS = 16 * SUB;
  static constexpr int DATA = KEYS * D * 2;           // bytes of a tile: 4096
  static constexpr int STAGE = DATA + SUB * 128;      // and the scales of its keys
};

__device__ __forceinline__ void qd_copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void qd_copy8(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void qd_copy4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void qd_mma(float* c, const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t qd_transposed(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
// The larger of two numbers; NaN if one is.
__device__ __forceinline__ float qd_max(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ float qd_log2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float qd_inverse(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float qd_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Codes 0 and 1 (HIGH: 2 and 3) of a word with its sign bits turned round, as float16: with 1152 on them, without.
template <bool HIGH>
__device__ __forceinline__ uint32_t qd_raised(uint32_t turned) { return __byte_perm(turned, 0x64646464u, HIGH ? 0x4342 : 0x4140); }
template <bool HIGH>
__device__ __forceinline__ uint32_t qd_half2(uint32_t turned) {
  const uint32_t raised = qd_raised<HIGH>(turned);
  const uint32_t offset = 0x64806480u;        // 1152
  const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&raised), *reinterpret_cast<const __half2*>(&offset));
  return *reinterpret_cast<const uint32_t*>(&v);
}

// NH: groups of 8 query heads.
template <int D, int NH>
__global__ void __launch_bounds__(QD_THREADS, 2)
attention_quantized_decode_kernel(const bf16* q, const int8_t* k_pool, const int8_t* v_pool, const float* k_scales, const float* v_scales,
                                  bf16* __restrict__ out, const int* __restrict__ decode_seg, const int* __restrict__ seg_q_start,
                                  const int* __restrict__ seg_pos0, const int* __restrict__ block_table, const int* __restrict__ seg_slot,
                                  int table_width, int requests, int heads, int kv_heads, int page_shift, int block_shift, int pool_pages, int window,
                                  float scale_log2, float* __restrict__ scratch, int* __restrict__ counters) {
  using Shape = QdShape<D>;
  constexpr int SUB = Shape::SUB, KEYS = Shape::KEYS, JD = D / 64, VW = D / 32;      // VW: words of a thread's dimensions of a key
  extern __shared__ __align__(128) uint8_t qd_shared[];
  int* before = reinterpret_cast<int*>(qd_shared + QD_WARPS * QD_STAGES * Shape::STAGE);      // [requests + 1] tiles before a request's
  __shared__ int warp_sums[QD_WARPS];
  __shared__ int last_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int group = heads / kv_heads, page_size = 1 << page_shift;
  pdl_trigger();

  auto segment_of = [&](int index) { return decode_seg != nullptr ? decode_seg[index] : index; };
  auto lowest_of = [&](int position) { return window > 0 ? max(0, position - window + 1) : 0; };
  // ---- tiles before each request's (positions are metadata of the step: read before the wait)
  int carried = 0;
  for (int first = 0; first < requests; first += QD_THREADS) {
    const int index = first + threadIdx.x;
    int tiles = 0;
    if (index < requests) {
      const int position = seg_pos0[segment_of(index)];
      tiles = position / KEYS - lowest_of(position) / KEYS + 1;
    }
    int inclusive = tiles;
#pragma unroll
    for (int offset = 1; offset < 32; offset <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, inclusive, offset);
      if (lane >= offset) inclusive += up;
    }
    if (lane == 31) warp_sums[warp] = inclusive;
    __syncthreads();
    int base = carried;
#pragma unroll
    for (int w = 0; w < QD_WARPS; ++w) {
      if (w < warp) base += warp_sums[w];
      carried += warp_sums[w];
    }
    if (index < requests) before[index] = base + inclusive - tiles;
    __syncthreads();
  }
  if (threadIdx.x == 0) before[requests] = carried;
  __syncthreads();
  // the line: request after request, a request's kv heads one behind the other, each QD_BEGIN longer than its tiles
  auto line_of = [&](int index) { return ((long long)before[index] + (long long)index * QD_BEGIN) * kv_heads; };
  const long long units = line_of(requests);
  const long long share = max((long long)QD_LEAST_SHARE, (units + gridDim.x - 1) / gridDim.x);
  long long at = share * blockIdx.x;
  const long long end = min(units, at + share);
  int request = 0;
  if (at < end) {                                   // the last one that begins at or before `at`
    int low = 0, high = requests - 1;
    while (low < high) {
      const int middle = (low + high + 1) >> 1;
      if (line_of(middle) <= at) low = middle;
      else high = middle - 1;
    }
    request = low;
  }
  pdl_wait();

  uint8_t* stages = qd_shared + warp * QD_STAGES * Shape::STAGE;
  const uint32_t stage_at = (uint32_t)__cvta_generic_to_shared(stages);
  while (at < end) {
    const int request_tiles = before[request + 1] - before[request], length = request_tiles + QD_BEGIN;
    const int kv_head = (int)((at - line_of(request)) / length);
    const long long pair_begin = line_of(request) + (long long)kv_head * length, pair_end = pair_begin + length;
    const long long my_end = min(end, pair_end);
    // its tiles, of the pair's
    const int from = max(0, (int)(at - pair_begin) - QD_BEGIN), until = (int)(my_end - pair_begin) - QD_BEGIN;
    const int here = request;
    at = my_end;
    if (kv_head == kv_heads - 1 && my_end == pair_end) ++request;
    if (until <= 0) continue;                       // a share that ends in a pair's beginning has none
    const int segment = segment_of(here), row = seg_q_start[segment], position = seg_pos0[segment];
    const int* table = block_table + (size_t)(seg_slot != nullptr ? seg_slot[segment] : segment) * table_width;
    const int lowest = lowest_of(position);
    const int first_tile = lowest / KEYS + from, tiles = until - from;

    // ---- loads: tile n of this warp is tile first_tile + warp + n * QD_WARPS
    const int my_tiles = tiles > warp ? (tiles - warp + QD_WARPS - 1) / QD_WARPS : 0;
    auto page_of = [&](int n, int sub) -> int {
      const int key0 = (first_tile + warp + n * QD_WARPS) * KEYS + sub * 16, logical = key0 >> page_shift;
      const int page = n < my_tiles && logical < table_width ? table[logical] : 0;
      return page >= 0 && page < pool_pages ? page : 0;
    };
    const int lane_k = g * D + 16 * t, lane_v = 2 * t * D + (D / 8) * g;
    auto issue = [&](int n, int to, const int (&pages)[SUB]) {
      if (n < my_tiles) {
        const uint32_t dst = stage_at + to * Shape::STAGE;
#pragma unroll
        for (int sub = 0; sub < SUB; ++sub) {
          const int key0 = (first_tile + warp + n * QD_WARPS) * KEYS + sub * 16, offset = key0 & (page_size - 1);
          const size_t line = (size_t)pages[sub] * kv_heads + kv_head;
          const size_t token = (line << page_shift) + offset;
          const int8_t* k_src = k_pool + (token * D + lane_k);
          const int8_t* v_src = v_pool + (token * D + lane_v);
          const uint32_t k_dst = dst + sub * (32 * D) + lane * 16;
#pragma unroll
          for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int j = 0; j < JD; ++j) qd_copy16(k_dst + (half * JD + j) * 512, k_src + 8 * half * D + 64 * j);
          const uint32_t v_dst = dst + sub * (32 * D) + 16 * D + lane * (VW * 4);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int8_t* src = v_src + ((i & 1) + 8 * (i >> 1)) * D;
            if constexpr (D == 128) qd_copy16(v_dst + i * 512, src);
            else qd_copy8(v_dst + i * 256, src);
          }
          // lanes 0..15 the keys' scales, 16..31 the values'
          const float* scales = lane < 16 ? k_scales : v_scales;
          qd_copy4(dst + Shape::DATA + sub * 128 + lane * 4, scales + ((token + (lane & 15)) >> block_shift));
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    int pages[SUB];
#pragma unroll
    for (int n = 0; n < QD_STAGES; ++n) {
#pragma unroll
      for (int sub = 0; sub < SUB; ++sub) pages[sub] = page_of(n, sub);
      issue(n, n, pages);
    }
#pragma unroll
    for (int sub = 0; sub < SUB; ++sub) pages[sub] = page_of(QD_STAGES, sub);

    // ---- queries: head 8 h + g, the thread's 16 dimensions of each 64, as float16 times a power of two
    uint32_t qf[NH][JD * 4][2];
    float factor[NH][2];      // of heads 2 t, 2 t + 1: scale, log2 e and the power of two back
    float start[NH][2];       // -1152 times the sum of the query
#pragma unroll
    for (int h = 0; h < NH; ++h) {
      const int head = 8 * h + g;
      uint4 raw[JD][2];
#pragma unroll
      for (int j = 0; j < JD; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          raw[j][i] = head < group ? __ldcg(reinterpret_cast<const uint4*>(q + ((size_t)row * heads + kv_head * group + head) * D + 64 * j + 16 * t + 8 * i))
                                   : make_uint4(0u, 0u, 0u, 0u);
      unsigned top = 0;
#pragma unroll
      for (int j = 0; j < JD; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t words[4] = {raw[j][i].x, raw[j][i].y, raw[j][i].z, raw[j][i].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) top = max(top, max((words[e] << 16) & 0x7fffffffu, words[e] & 0x7fff0000u));
        }
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // 2^-e for a largest of 2^e .. 2^(e+1); none for zeros, tiny ones and what is not finite
      const unsigned exponent = min(top >> 23, 253u);
      const bool scaled = exponent >= 1u && top < 0x7f800000u;
      const float down = scaled ? __uint_as_float((254u - exponent) << 23) : 1.f;
      const float up = scaled ? __uint_as_float(exponent << 23) : 1.f;
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < JD; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t words[4] = {raw[j][i].x, raw[j][i].y, raw[j][i].z, raw[j][i].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const __half2 pair = __floats2half2_rn(__uint_as_float(words[e] << 16) * down, __uint_as_float(words[e] & 0xffff0000u) * down);
            qf[h][j * 4 + 2 * i + (e >> 1)][e & 1] = *reinterpret_cast<const uint32_t*>(&pair);
            const float2 rounded = __half22float2(pair);
            sum += rounded.x + rounded.y;
          }
        }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        factor[h][e] = __shfl_sync(0xffffffffu, up, (2 * t + e) * 4) * scale_log2;
        start[h][e] = -1152.f * __shfl_sync(0xffffffffu, sum, (2 * t + e) * 4);
      }
    }

    // ---- the walk
    float m[NH][2], l[NH][2], o[NH][D / 16][4];
#pragma unroll
    for (int h = 0; h < NH; ++h) {
      m[h][0] = m[h][1] = -INFINITY;
      l[h][0] = l[h][1] = 0.f;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) o[h][i][0] = o[h][i][1] = o[h][i][2] = o[h][i][3] = 0.f;
    }
    int stage_of = 0;
    for (int n = 0; n < my_tiles; ++n) {
      asm volatile("cp.async.wait_group %0;" ::"n"(QD_STAGES - 1) : "memory");
      __syncwarp();
      const uint8_t* stage = stages + stage_of * Shape::STAGE;
      const int key_tile = (first_tile + warp + n * QD_WARPS) * KEYS;
#pragma unroll
      for (int sub = 0; sub < SUB; ++sub) {
        const int key0 = key_tile + sub * 16;
        const uint8_t* k_data = stage + sub * (32 * D) + lane * 16;
        const uint8_t* v_data = stage + sub * (32 * D) + 16 * D + lane * (VW * 4);
        const float* scales = reinterpret_cast<const float*>(stage + Shape::DATA + sub * 128);
        // scores^T: rows keys g, g + 8, columns heads 2 t, 2 t + 1
        float s[NH][4];
#pragma unroll
        for (int h = 0; h < NH; ++h) { s[h][0] = s[h][2] = start[h][0]; s[h][1] = s[h][3] = start[h][1]; }
#pragma unroll
        for (int j = 0; j < JD; ++j) {
          const uint4 low = *reinterpret_cast<const uint4*>(k_data + j * 512), high = *reinterpret_cast<const uint4*>(k_data + (JD + j) * 512);
          const uint32_t a[4] = {low.x, low.y, low.z, low.w}, b[4] = {high.x, high.y, high.z, high.w};
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const uint32_t first = a[w] ^ 0x80808080u, second = b[w] ^ 0x80808080u;
            const uint32_t k[4] = {qd_raised<false>(first), qd_raised<false>(second), qd_raised<true>(first), qd_raised<true>(second)};
#pragma unroll
            for (int h = 0; h < NH; ++h) qd_mma(s[h], k, qf[h][j * 4 + w][0], qf[h][j * 4 + w][1]);
          }
        }
        // scales of the two keys; a value's below 2^-100 counts as 2^-100 (what it stands for is below 2^-93 then)
        float ks[2], lv[2], iv[2];
        const bool ragged = key0 < lowest || key0 + 15 > position;
        bool hidden[2] = {false, false};
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float vs = qd_max(scales[16 + g + 8 * e], 7.888609e-31f);
          ks[e] = scales[g + 8 * e];
          lv[e] = qd_log2(vs);
          iv[e] = qd_inverse(vs);
          if (ragged && (key0 + g + 8 * e < lowest || key0 + g + 8 * e > position)) { hidden[e] = true; iv[e] = 0.f; }
        }
        uint32_t p[NH][2];
#pragma unroll
        for (int h = 0; h < NH; ++h) {
          float x[2][2];
#pragma unroll
          for (int e = 0; e < 2; ++e)      // key
#pragma unroll
            for (int c = 0; c < 2; ++c) {  // head
              x[e][c] = fmaf(s[h][2 * e + c] * ks[e], factor[h][c], lv[e]);
              if (hidden[e]) x[e][c] = -INFINITY;
            }
          float top[2] = {fmaxf(x[0][0], x[1][0]), fmaxf(x[0][1], x[1][1])};
          // (-inf) - (-inf) is NaN and compares false: nothing visible yet
          if (__any_sync(0xffffffffu, top[0] - m[h][0] > QD_LAZY || top[1] - m[h][1] > QD_LAZY)) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              top[c] = fmaxf(top[c], __shfl_xor_sync(0xffffffffu, top[c], 4));
              top[c] = fmaxf(top[c], __shfl_xor_sync(0xffffffffu, top[c], 8));
              top[c] = fmaxf(top[c], __shfl_xor_sync(0xffffffffu, top[c], 16));
              const float higher = fmaxf(m[h][c], top[c]);
              const float alpha = higher == -INFINITY ? 1.f : qd_exp2(m[h][c] - higher);
              m[h][c] = higher;
              l[h][c] *= alpha;
#pragma unroll
              for (int i = 0; i < D / 16; ++i) { o[h][i][c] *= alpha; o[h][i][2 + c] *= alpha; }
            }
          }
#pragma unroll
          for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              x[e][c] = qd_exp2(x[e][c] - (m[h][c] == -INFINITY ? 0.f : m[h][c]));
              l[h][c] = fmaf(x[e][c], iv[e], l[h][c]);
            }
            const __half2 pair = __floats2half2_rn(x[e][0], x[e][1]);
            p[h][e] = qd_transposed(*reinterpret_cast<const uint32_t*>(&pair));
          }
        }
        // out^T: rows dimensions (D / 8) g + 2 i and + 1, columns heads 2 t, 2 t + 1
        uint32_t v[4][VW];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (D == 128) *reinterpret_cast<uint4*>(v[i]) = *reinterpret_cast<const uint4*>(v_data + i * 512);
          else *reinterpret_cast<uint2*>(v[i]) = *reinterpret_cast<const uint2*>(v_data + i * 256);
        }
#pragma unroll
        for (int w = 0; w < VW; ++w) {
#pragma unroll
          for (int upper = 0; upper < 2; ++upper) {
            const int order = upper ? 0x7362 : 0x5140;
            const uint32_t near_keys = __byte_perm(v[0][w], v[1][w], order) ^ 0x80808080u, far_keys = __byte_perm(v[2][w], v[3][w], order) ^ 0x80808080u;
            const uint32_t a[4] = {qd_half2<false>(near_keys), qd_half2<true>(near_keys), qd_half2<false>(far_keys), qd_half2<true>(far_keys)};
#pragma unroll
            for (int h = 0; h < NH; ++h) qd_mma(o[h][2 * w + upper], a, p[h][0], p[h][1]);
          }
        }
      }
      __syncwarp();
      issue(n + QD_STAGES, stage_of, pages);
      stage_of = stage_of + 1 == QD_STAGES ? 0 : stage_of + 1;
#pragma unroll
      for (int sub = 0; sub < SUB; ++sub) pages[sub] = page_of(n + QD_STAGES + 1, sub);
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();

    // ---- the warps' states, then those of the CTAs; the stages' memory is free now
    constexpr int HEADS = 8 * NH;
    float* states = reinterpret_cast<float*>(qd_shared);               // [warp][head][D]
    float* tops = states + QD_WARPS * HEADS * D;                       // [warp][head]
    float* sums = tops + QD_WARPS * HEADS;
#pragma unroll
    for (int h = 0; h < NH; ++h)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float sum = l[h][c];
        sum += __shfl_xor_sync(0xffffffffu, sum, 4);
        sum += __shfl_xor_sync(0xffffffffu, sum, 8);
        sum += __shfl_xor_sync(0xffffffffu, sum, 16);
        const int head = 8 * h + 2 * t + c;
        if (g == 0) { tops[warp * HEADS + head] = m[h][c]; sums[warp * HEADS + head] = sum; }
        if (head < group) {
          float* mine = states + (warp * HEADS + head) * D + (D / 8) * g;
#pragma unroll
          for (int i = 0; i < D / 16; ++i) *reinterpret_cast<float2*>(mine + 2 * i) = make_float2(o[h][i][c], o[h][i][2 + c]);
        }
      }
    __syncthreads();
    const bool whole = from == 0 && my_end == pair_end;
    constexpr int STATE = D + 2;
    // a CTA holds at most two pairs in part: one that began before its share, one that ends behind it
    float* mine = scratch + ((size_t)blockIdx.x * 2 + (from > 0 ? 0 : 1)) * 16 * STATE;
    for (int idx = threadIdx.x; idx < group * D; idx += QD_THREADS) {
      const int head = idx / D, d = idx - head * D;
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < QD_WARPS; ++w) top = fmaxf(top, tops[w * HEADS + head]);
      float sum = 0.f, value = 0.f;
#pragma unroll
      for (int w = 0; w < QD_WARPS; ++w) {
        const float share_of = tops[w * HEADS + head] == -INFINITY ? 0.f : qd_exp2(tops[w * HEADS + head] - top);
        // (a warp without keys has nothing to add; one whose scores are no numbers has a NaN sum and no top)
        sum += sums[w * HEADS + head] * (sums[w * HEADS + head] == sums[w * HEADS + head] ? share_of : 1.f);
        value = fmaf(states[(w * HEADS + head) * D + d], share_of, value);
      }
      if (whole) {
        out[((size_t)row * heads + kv_head * group + head) * D + d] = __float2bfloat16_rn(value / sum);
      } else {
        mine[head * STATE + 2 + d] = value;
        if (d == 0) { mine[head * STATE] = top; mine[head * STATE + 1] = sum; }
      }
    }
    if (!whole) {
      const int pair = here * kv_heads + kv_head;
      const int first_cta = (int)((pair_begin + QD_BEGIN) / share), last_cta = (int)((pair_end - 1) / share);
      __threadfence();
      __syncthreads();
      if (threadIdx.x == 0) last_flag = atomicAdd(&counters[pair], 1) == last_cta - first_cta;
      __syncthreads();
      if (last_flag) {
        __threadfence();
        for (int idx = threadIdx.x; idx < group * D; idx += QD_THREADS) {
          const int head = idx / D, d = idx - head * D;
          float top = -INFINITY, sum = 0.f, value = 0.f;
          for (int c = first_cta; c <= last_cta; ++c) {
            const float* theirs = scratch + ((size_t)c * 2 + (c > first_cta ? 0 : 1)) * 16 * STATE + head * STATE;
            const float their_top = __ldcg(theirs), their_sum = __ldcg(theirs + 1), theirs_value = __ldcg(theirs + 2 + d);
            const float higher = fmaxf(top, their_top);
            const float down = top == -INFINITY ? 0.f : qd_exp2(top - higher), share_of = their_top == -INFINITY ? 0.f : qd_exp2(their_top - higher);
            sum = sum * (sum == sum ? down : 1.f) + their_sum * (their_sum == their_sum ? share_of : 1.f);
            value = fmaf(theirs_value, share_of, value * down);
            top = higher;
          }
          out[((size_t)row * heads + kv_head * group + head) * D + d] = __float2bfloat16_rn(value / sum);
        }
        if (threadIdx.x == 0) counters[pair] = 0;       // ready for the next launch
      }
    }
    __syncthreads();        // the stages are filled again, the flag is written again
  }
}

template <int D, int NH>
static int quantized_decode_launch(const void* q, const void* k_pool, const void* v_pool, const float* k_scales, const float* v_scales, void* out,
                                   const int* decode_seg, const int* seg_q_start, const int* seg_pos0, const int* block_table, const int* seg_slot,
                                   int table_width, int requests, int heads, int kv_heads, int page_shift, int block_shift, int pool_pages, int window,
                                   float scale, long long most_units, float* scratch, int* counters, cudaStream_t stream) {
  auto kernel = attention_quantized_decode_kernel<D, NH>;
  constexpr size_t ring = (size_t)QD_WARPS * QD_STAGES * QdShape<D>::STAGE;
  static_assert((size_t)QD_WARPS * 8 * NH * (D + 2) * sizeof(float) <= ring, "the states lie where the stages were");
  static OncePerDevice once;
  const cudaError_t err = once([&] {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(ring + (QD_MOST_REQUESTS + 1) * sizeof(int)));
  });
  if (err != cudaSuccess) return (int)err;
  const long long shares = (most_units + QD_LEAST_SHARE - 1) / QD_LEAST_SHARE, resident = 2 * sm_count();
  const int ctas = (int)(shares < resident ? shares : resident);
  launch_kernel(kernel, dim3(ctas), dim3(QD_THREADS), ring + (requests + 1) * sizeof(int), stream, (const bf16*)q, (const int8_t*)k_pool,
                (const int8_t*)v_pool, k_scales, v_scales, (bf16*)out, decode_seg, seg_q_start, seg_pos0, block_table, seg_slot, table_width, requests,
                heads, kv_heads, page_shift, block_shift, pool_pages, window, scale * 1.4426950408889634f, scratch, counters);
  return launch_status();
}

static int shift_of(int size) {
  for (int shift = 0; shift < 31; ++shift)
    if ((1 << shift) == size) return shift;
  return -1;
}

}  // namespace mlr

using namespace mlr;

MLR_DEFINE_PDL_SWITCH

// Floats of scratch memory that a launch needs.
MLR_EXPORT int mlr_attention_quantized_decode_scratch(int dim) { return 2 * sm_count() * 2 * 16 * (dim + 2); }

// q, out: [rows, heads * dim] bfloat16, of which the rows of `requests` decoded tokens are attended (decode_seg: their segments, or null for
// segments 0, 1, ..); pools [pages, kv_heads, page_size, dim]; scales [pages, kv_heads, page_size / block]; longest: keys of the longest context;
// counters: requests * kv_heads zeroed ints (left zeroed).
MLR_EXPORT int mlr_attention_quantized_decode(const void* q, const void* k_pool, const void* v_pool, const float* k_scales, const float* v_scales,
                                              void* out, const int* decode_seg, const int* seg_q_start, const int* seg_pos0, const int* block_table,
                                              const int* seg_slot, int table_width, int requests, int heads, int kv_heads, int dim, int page_size,
                                              int block, int pool_pages, int window, float scale, int longest, void* scratch, int* counters,
                                              cudaStream_t stream) {
  if (requests == 0) return MLR_OK;
  if (requests < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || table_width <= 0 || pool_pages <= 0 || longest <= 0) return MLR_BAD_SIZE;
  const int page_shift = shift_of(page_size), block_shift = shift_of(block);
  if ((dim != 64 && dim != 128) || page_shift < 4 || block_shift < 0 || block > page_size) return MLR_BAD_SIZE;
  if (heads / kv_heads > 16 || requests > QD_MOST_REQUESTS) return MLR_TOO_LARGE;
  if (((uintptr_t)q | (uintptr_t)k_pool | (uintptr_t)v_pool) & 15) return MLR_BAD_ALIGNMENT;
  const int keys = window > 0 && window < longest ? window + 16 : longest, tile = 16 * (128 / dim);
  const long long most = (long long)requests * kv_heads * (keys / tile + 2 + QD_BEGIN);
  const bool wide = heads / kv_heads > 8;
#define MLR_DECODE(D_, N_)                                                                                                                       \
  return quantized_decode_launch<D_, N_>(q, k_pool, v_pool, k_scales, v_scales, out, decode_seg, seg_q_start, seg_pos0, block_table, seg_slot,   \
                                         table_width, requests, heads, kv_heads, page_shift, block_shift, pool_pages, window, scale, most,       \
                                         (float*)scratch, counters, stream)
  if (dim == 64) { if (wide) MLR_DECODE(64, 2); MLR_DECODE(64, 1); }
  if (wide) MLR_DECODE(128, 2);
  MLR_DECODE(128, 1);
#undef MLR_DECODE
}
