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
// tiles on their way, by bulk tensor copies of 16 keys into a ring of its own (a copy per 16 bytes and thread into the same ring
// spent seven times the instructions of a tile on them: 64 x 8,192 keys 77 us, so 63).  The heads of a group are the narrow side of the
// products (n = 8), keys and dimensions the wide one:
//   scores^T [16 keys x 8 heads] = K [16 x dim] Q^T,   out^T [dim x 8 heads] += V^T [dim x 16 keys] P^T
// The order of the dimensions within a product is free, so a thread reads 16 bytes of a key that are four steps' operands, and 16
// (8) dimensions of four keys that are eight (four) tiles' operands; the copies' swizzle keeps the reads free of conflicts.  A byte
// becomes a float16 by a byte permutation: 1024 + 128 + code.  Of the values the 1152 is subtracted (exactly); of the keys it
// is left in, and 1152 times the sum of the query taken off where the scores' sums begin (32 bits: 1152 sum |q| 2^-24 beside scores of
// up to 127 sum |q|).
//
// The keys of all requests and kv heads form one line that the warps share evenly, whatever the contexts: a warp's share may
// end one request's keys and begin another's.  Each beginning counts as QD_BEGIN tiles more, about what it costs.  No warp waits for
// another.  Pairs of a request and a kv head that several warps walk are merged by a second launch, in the order of the warps.
// 64 requests of up to 8,192 keys, 28 heads of 128 over 4: 62 us (4.4 TB/s); 100 of up to 16,384, 40 over 8: 332 us (5.2 TB/s), the merge's
// launch included.
#include <cuda_fp16.h>

#include "tma.cuh"

namespace mlr {

constexpr int QD_WARPS = 8, QD_THREADS = QD_WARPS * 32, QD_STAGES = 3;
constexpr int QD_MOST_REQUESTS = 2048;       // whose tiles a CTA counts
constexpr int QD_BEGIN = 1;                  // what the beginning of a pair of a request and a kv head costs a warp, in tiles
constexpr int QD_LEAST_SHARE = QD_BEGIN + 2;       // of a warp, at least
constexpr int QD_MOST_PARTS = 128;           // warps of a pair
// The largest exponent follows the maximum in steps of more than this; weights up to 2^8 are far from float16's end.
constexpr float QD_LAZY = 8.f;

template <int D>
struct QdShape {
  static constexpr int SUB = 128 / D;                 // groups of 16 keys in a tile
  static constexpr int KEYS = 16 * SUB;
  static constexpr int PART = 16 * D;                 // bytes of the keys (the values) of a group
  static constexpr int DATA = 2 * SUB * PART;         // of a tile: 4096
  static constexpr int SCALES = SUB * 128;            // the scales of its keys
  static constexpr int RING = QD_WARPS * QD_STAGES * DATA;
  static constexpr int SHARED = RING + QD_WARPS * QD_STAGES * (SCALES + 8);      // and a barrier per tile
};
// Where 16 bytes of row `row` lie in a group of 16 rows as the copies leave them: 128-byte rows, or 64-byte ones.
template <int D>
__device__ __forceinline__ int qd_place(int row, int chunk) {
  return row * D + ((chunk ^ (D == 128 ? row & 7 : (row >> 1) & 3)) << 4);
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

// The lowest key that a position sees, its tiles, and what a warp takes of a line of `units`, whose longest pair has `most` tiles.
__device__ __forceinline__ int qd_lowest(int position, int window) { return window > 0 ? max(0, position - window + 1) : 0; }
template <int KEYS>
__device__ __forceinline__ int qd_tiles(int position, int window) { return position / KEYS - qd_lowest(position, window) / KEYS + 1; }
__device__ __forceinline__ long long qd_share(long long units, int most, int ctas) {
  const long long walkers = (long long)ctas * QD_WARPS;
  return max((units + walkers - 1) / walkers, (long long)max(QD_LEAST_SHARE, (most + QD_MOST_PARTS - 2) / (QD_MOST_PARTS - 1)));
}

// NH: groups of 8 query heads.
template <int D, int NH>
__global__ void __launch_bounds__(QD_THREADS, 2)
attention_quantized_decode_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, const bf16* q,
                                  const float* k_scales, const float* v_scales, bf16* __restrict__ out, const int* __restrict__ decode_seg, const int* __restrict__ seg_q_start,
                                  const int* __restrict__ seg_pos0, const int* __restrict__ block_table, const int* __restrict__ seg_slot,
                                  int table_width, int requests, int heads, int kv_heads, int page_shift, int block_shift, int pool_pages, int window,
                                  float scale_log2, float* __restrict__ states, float2* __restrict__ sums, int* error_word) {
  using Shape = QdShape<D>;
  constexpr int SUB = Shape::SUB, KEYS = Shape::KEYS, JD = D / 64, VW = D / 32;      // VW: words of a thread's dimensions of a key
  extern __shared__ uint8_t qd_shared_raw[];
  uint8_t* qd_shared = (uint8_t*)(((uintptr_t)qd_shared_raw + 1023) & ~(uintptr_t)1023);      // what swizzled copies need
  int* before = reinterpret_cast<int*>(qd_shared + Shape::SHARED);      // [requests + 1] tiles before a request's
  __shared__ int warp_sums[QD_WARPS], warp_most[QD_WARPS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int group = heads / kv_heads, page_size = 1 << page_shift;
  uint8_t* stages = qd_shared + warp * QD_STAGES * Shape::DATA;
  uint8_t* scale_stages = qd_shared + Shape::RING + warp * QD_STAGES * Shape::SCALES;
  uint64_t* full = reinterpret_cast<uint64_t*>(qd_shared + Shape::RING + QD_WARPS * QD_STAGES * Shape::SCALES) + warp * QD_STAGES;
  if (lane == 0) {
    for (int i = 0; i < QD_STAGES; ++i) mbar_init(full + i, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (threadIdx.x == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&k_map) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&v_map) : "memory");
  }
  pdl_trigger();

  auto segment_of = [&](int index) { return decode_seg != nullptr ? decode_seg[index] : index; };
  auto lowest_of = [&](int position) { return qd_lowest(position, window); };
  // ---- tiles before each request's (positions are metadata of the step: read before the wait)
  int carried = 0, most = 0;
  for (int first = 0; first < requests; first += QD_THREADS) {
    const int index = first + threadIdx.x;
    int tiles = 0;
    if (index < requests) {
      const int position = seg_pos0[segment_of(index)];
      tiles = qd_tiles<KEYS>(position, window);
    }
    const int warp_top = (int)__reduce_max_sync(0xffffffffu, (unsigned)tiles);
    int inclusive = tiles;
#pragma unroll
    for (int offset = 1; offset < 32; offset <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, inclusive, offset);
      if (lane >= offset) inclusive += up;
    }
    if (lane == 31) { warp_sums[warp] = inclusive; warp_most[warp] = warp_top; }
    __syncthreads();
    int base = carried;
#pragma unroll
    for (int w = 0; w < QD_WARPS; ++w) {
      if (w < warp) base += warp_sums[w];
      carried += warp_sums[w];
      most = max(most, warp_most[w]);
    }
    if (index < requests) before[index] = base + inclusive - tiles;
    __syncthreads();
  }
  if (threadIdx.x == 0) before[requests] = carried;
  __syncthreads();
  // the line: request after request, a request's kv heads one behind the other, each QD_BEGIN longer than its tiles
  auto line_of = [&](int index) { return ((long long)before[index] + (long long)index * QD_BEGIN) * kv_heads; };
  const long long units = line_of(requests), share = qd_share(units, most, gridDim.x);
  const long long walker = (long long)blockIdx.x * QD_WARPS + warp;
  long long at = share * walker;
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

  const uint32_t scales_at = smem_u32(scale_stages);
  unsigned tiles_before = 0;        // of this warp's earlier pairs: the ring and its phases run on
  bool gave_up = false;             // a wait ran out: the warp ends, the host raises
  while (at < end && !gave_up) {
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
    const int first_tile = lowest / KEYS + from, my_tiles = until - from;

    // ---- loads
    auto page_of = [&](int n, int sub) -> int {
      const int key0 = (first_tile + n) * KEYS + sub * 16, logical = key0 >> page_shift;
      const int page = n < my_tiles && logical < table_width ? table[logical] : 0;
      return page >= 0 && page < pool_pages ? page : 0;
    };
    auto issue = [&](int n, int to, const int (&pages)[SUB]) {
      if (n < my_tiles) {
        if (lane == 0) mbar_expect_tx(full + to, Shape::DATA);
#pragma unroll
        for (int sub = 0; sub < SUB; ++sub) {
          const int key0 = (first_tile + n) * KEYS + sub * 16;
          const int token = ((pages[sub] * kv_heads + kv_head) << page_shift) + (key0 & (page_size - 1));
          if (lane == 0) {
            uint8_t* dst = stages + to * Shape::DATA + sub * 2 * Shape::PART;
            tma_load_2d(&k_map, full + to, dst, 0, token);
            tma_load_2d(&v_map, full + to, dst + Shape::PART, 0, token);
          }
          // lanes 0..15 the keys' scales, 16..31 the values'
          const float* scales = lane < 16 ? k_scales : v_scales;
          qd_copy4(scales_at + to * Shape::SCALES + sub * 128 + lane * 4, scales + ((token + (lane & 15)) >> block_shift));
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    int stage_of = (int)(tiles_before % QD_STAGES);
    int pages[SUB];
#pragma unroll
    for (int n = 0; n < QD_STAGES; ++n) {
#pragma unroll
      for (int sub = 0; sub < SUB; ++sub) pages[sub] = page_of(n, sub);
      issue(n, (stage_of + n) % QD_STAGES, pages);
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
    for (int n = 0; n < my_tiles; ++n) {
      asm volatile("cp.async.wait_group %0;" ::"n"(QD_STAGES - 1) : "memory");
      gave_up = !mbar_wait(full + stage_of, ((tiles_before + n) / QD_STAGES) & 1u, error_word, 0x91);
      gave_up = __any_sync(0xffffffffu, gave_up);
      if (gave_up) {                  // the copies under way end before the warp does
        for (int later = n; later < my_tiles && later < n + QD_STAGES; ++later)
          mbar_wait(full + (tiles_before + later) % QD_STAGES, ((tiles_before + later) / QD_STAGES) & 1u, error_word, 0x92);
        break;
      }
      __syncwarp();
      const uint8_t* stage = stages + stage_of * Shape::DATA;
      const int key_tile = (first_tile + n) * KEYS;
#pragma unroll
      for (int sub = 0; sub < SUB; ++sub) {
        const int key0 = key_tile + sub * 16;
        const uint8_t* k_data = stage + sub * 2 * Shape::PART;
        const uint8_t* v_data = k_data + Shape::PART;
        const float* scales = reinterpret_cast<const float*>(scale_stages + stage_of * Shape::SCALES + sub * 128);
        // scores^T: rows keys g, g + 8, columns heads 2 t, 2 t + 1
        float s[NH][4];
#pragma unroll
        for (int h = 0; h < NH; ++h) { s[h][0] = s[h][2] = start[h][0]; s[h][1] = s[h][3] = start[h][1]; }
#pragma unroll
        for (int j = 0; j < JD; ++j) {
          const uint4 low = *reinterpret_cast<const uint4*>(k_data + qd_place<D>(g, 4 * j + t));
          const uint4 high = *reinterpret_cast<const uint4*>(k_data + qd_place<D>(g + 8, 4 * j + t));
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
          const int key = 2 * t + (i & 1) + 8 * (i >> 1);
          if constexpr (D == 128) *reinterpret_cast<uint4*>(v[i]) = *reinterpret_cast<const uint4*>(v_data + qd_place<D>(key, g));
          else *reinterpret_cast<uint2*>(v[i]) = *reinterpret_cast<const uint2*>(v_data + qd_place<D>(key, g >> 1) + 8 * (g & 1));
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
    __syncwarp();
    tiles_before += (unsigned)my_tiles;

    // ---- the pair's outputs, or this warp's part of them
    const bool whole = from == 0 && my_end == pair_end;
    // a warp holds at most two pairs in part: one that began before its share, one that ends behind it
    const size_t slot = (size_t)walker * 2 + (from > 0 ? 0 : 1);
#pragma unroll
    for (int h = 0; h < NH; ++h)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float sum = l[h][c];
        sum += __shfl_xor_sync(0xffffffffu, sum, 4);
        sum += __shfl_xor_sync(0xffffffffu, sum, 8);
        sum += __shfl_xor_sync(0xffffffffu, sum, 16);
        const int head = 8 * h + 2 * t + c;
        if (head >= group) continue;
        if (whole) {
          const float inverse = 1.f / sum;
          uint32_t packed[D / 16];
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            const __nv_bfloat162 pair = __floats2bfloat162_rn(o[h][i][c] * inverse, o[h][i][2 + c] * inverse);
            packed[i] = *reinterpret_cast<const uint32_t*>(&pair);
          }
          uint4* dst = reinterpret_cast<uint4*>(out + ((size_t)row * heads + kv_head * group + head) * D + (D / 8) * g);
#pragma unroll
          for (int i = 0; i < D / 64; ++i) dst[i] = make_uint4(packed[4 * i], packed[4 * i + 1], packed[4 * i + 2], packed[4 * i + 3]);
        } else {
          float4* dst = reinterpret_cast<float4*>(states + (slot * 8 * NH + head) * D + (D / 8) * g);
#pragma unroll
          for (int i = 0; i < D / 32; ++i) dst[i] = make_float4(o[h][2 * i][c], o[h][2 * i][2 + c], o[h][2 * i + 1][c], o[h][2 * i + 1][2 + c]);
          if (g == 0) sums[slot * 8 * NH + head] = make_float2(m[h][c], sum);
        }
      }
  }
}

// The parts of pairs that several warps walked.  A CTA per pair, a thread per head and four dimensions.
template <int D, int NH>
__global__ void __launch_bounds__(8 * NH * D / 4)
merge_quantized_decode_kernel(const float* states, const float2* sums, bf16* __restrict__ out, const int* __restrict__ decode_seg,
                              const int* __restrict__ seg_q_start, const int* __restrict__ seg_pos0, int requests, int heads, int kv_heads,
                              int window, int ctas) {
  constexpr int KEYS = QdShape<D>::KEYS, THREADS = 8 * NH * D / 4;
  __shared__ int found[3];       // tiles of the requests before this one, of all, of the longest
  pdl_trigger();
  const int request = blockIdx.x / kv_heads, kv_head = blockIdx.x - request * kv_heads, group = heads / kv_heads;
  const int head = threadIdx.x / (D / 4), d = threadIdx.x % (D / 4), lane = threadIdx.x & 31;
  auto segment_of = [&](int index) { return decode_seg != nullptr ? decode_seg[index] : index; };
  if (threadIdx.x < 3) found[threadIdx.x] = 0;
  __syncthreads();
  unsigned sum = 0, all = 0, most = 0;
  for (int index = threadIdx.x; index < requests; index += THREADS) {
    const unsigned tiles = (unsigned)qd_tiles<KEYS>(seg_pos0[segment_of(index)], window);
    if (index < request) sum += tiles;
    all += tiles;
    most = max(most, tiles);
  }
  sum = __reduce_add_sync(0xffffffffu, sum);
  all = __reduce_add_sync(0xffffffffu, all);
  most = __reduce_max_sync(0xffffffffu, most);
  if (lane == 0) { atomicAdd(&found[0], (int)sum); atomicAdd(&found[1], (int)all); atomicMax(&found[2], (int)most); }
  const int segment = segment_of(request), row = seg_q_start[segment], length = qd_tiles<KEYS>(seg_pos0[segment], window) + QD_BEGIN;
  __syncthreads();
  const int before = found[0];
  const long long share = qd_share(((long long)found[1] + (long long)requests * QD_BEGIN) * kv_heads, found[2], ctas);
  const long long begin = ((long long)before + (long long)request * QD_BEGIN) * kv_heads + (long long)kv_head * length;
  const long long first = (begin + QD_BEGIN) / share, last = (begin + length - 1) / share;
  pdl_wait();                                      // (all: whoever waits for this launch waits for the one before it too)
  if (first == last || head >= group) return;      // one warp wrote the outputs
  const int parts = (int)(last - first) + 1;
  // part i: the first one's pair begins in its share, the others' began before
  auto slot_of = [&](int i) { return (size_t)((first + i) * 2 + (i == 0 ? 1 : 0)) * 8 * NH + head; };
  constexpr int AHEAD = 12;        // parts whose numbers are asked for at once
  float top = -INFINITY, total = 0.f;
  float4 value = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int base = 0; base < parts; base += AHEAD) {
    float2 state[AHEAD];
    float4 v[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      state[i] = base + i < parts ? __ldcg(sums + slot_of(base + i)) : make_float2(-INFINITY, 0.f);
      v[i] = base + i < parts ? __ldcg(reinterpret_cast<const float4*>(states + slot_of(base + i) * D) + d) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    float higher = top;
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) higher = fmaxf(higher, state[i].x);
    const float down = top == -INFINITY ? 0.f : qd_exp2(top - higher);
    top = higher;
    // (a part whose scores are no numbers has no largest one and a NaN sum, which stays)
    total *= total == total ? down : 1.f;
    value = make_float4(value.x * down, value.y * down, value.z * down, value.w * down);
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const float weight = state[i].x == -INFINITY ? 0.f : qd_exp2(state[i].x - top);
      total += state[i].y * (state[i].y == state[i].y ? weight : 1.f);
      value.x = fmaf(v[i].x, weight, value.x);
      value.y = fmaf(v[i].y, weight, value.y);
      value.z = fmaf(v[i].z, weight, value.z);
      value.w = fmaf(v[i].w, weight, value.w);
    }
  }
  const float inverse = 1.f / total;
  const __nv_bfloat162 low = __floats2bfloat162_rn(value.x * inverse, value.y * inverse), high = __floats2bfloat162_rn(value.z * inverse, value.w * inverse);
  reinterpret_cast<uint2*>(out + ((size_t)row * heads + kv_head * group + head) * D)[d] =
      make_uint2(*reinterpret_cast<const uint32_t*>(&low), *reinterpret_cast<const uint32_t*>(&high));
}

// Warps of a launch, and where the parts' memory lies (bytes).
struct QdLayout {
  int ctas;
  long long sums, total;
};
static QdLayout qd_layout(int requests, int kv_heads, int group, int dim, int window, int longest) {
  const int keys = window > 0 && window < longest ? window + 16 : longest, tile = 16 * (128 / dim), per = group > 8 ? 16 : 8;
  const long long units = (long long)requests * kv_heads * (keys / tile + 2 + QD_BEGIN), most = 2 * sm_count();
  const long long ctas = (units + QD_LEAST_SHARE * QD_WARPS - 1) / (QD_LEAST_SHARE * QD_WARPS);
  QdLayout at;
  at.ctas = (int)(ctas < most ? ctas : most);
  const long long slots = (long long)at.ctas * QD_WARPS * 2 * per;
  at.sums = slots * dim * 4;
  at.total = at.sums + slots * 8;
  return at;
}

// rows x dim bytes, row-major, a box of 16 rows; the maps of pools are kept, as in cached_tile_map.
static bool qd_map(CUtensorMap* out, const void* base, long long rows, int dim) {
  constexpr int SLOTS = 1024;
  static TileMapKey keys[SLOTS];
  static CUtensorMap maps[SLOTS];
  const TileMapKey key{base, rows, dim, 16};
  const unsigned long long h = (unsigned long long)(uintptr_t)base * 0x9E3779B97F4A7C15ull + (unsigned long long)rows * 0xBF58476D1CE4E5B9ull + dim;
  const int slot = (int)((h >> 40) % SLOTS);
  if (!(keys[slot] == key) || base == nullptr) {
    auto encode = encode_tiled();
    if (encode == nullptr) return false;
    cuuint64_t dims[2] = {(cuuint64_t)dim, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)dim};
    cuuint32_t box[2] = {(cuuint32_t)dim, 16u};
    cuuint32_t element_strides[2] = {1, 1};
    keys[slot] = TileMapKey{nullptr, 0, 0, 0};
    if (encode(&maps[slot], CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, element_strides,
               CU_TENSOR_MAP_INTERLEAVE_NONE, dim == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return false;
    keys[slot] = key;
  }
  *out = maps[slot];
  return true;
}

template <int D, int NH>
static int quantized_decode_launch(const void* q, const void* k_pool, const void* v_pool, const float* k_scales, const float* v_scales, void* out,
                                   const int* decode_seg, const int* seg_q_start, const int* seg_pos0, const int* block_table, const int* seg_slot,
                                   int table_width, int requests, int heads, int kv_heads, int page_shift, int block_shift, int pool_pages, int window,
                                   float scale, int longest, uint8_t* scratch, int* error_word, cudaStream_t stream) {
  auto kernel = attention_quantized_decode_kernel<D, NH>;
  constexpr size_t shared = 1024 + QdShape<D>::SHARED;
  static_assert(2 * (shared + (QD_MOST_REQUESTS + 1) * sizeof(int) + 1024) <= 228 * 1024, "two CTAs per SM");
  const long long pool_rows = ((long long)pool_pages * kv_heads) << page_shift;
  if (pool_rows >= (1ll << 31)) return MLR_TOO_LARGE;
  CUtensorMap k_map, v_map;
  if (!qd_map(&k_map, k_pool, pool_rows, D) || !qd_map(&v_map, v_pool, pool_rows, D)) return MLR_BAD_SIZE;
  static OncePerDevice once;
  const cudaError_t err = once([&] {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(shared + (QD_MOST_REQUESTS + 1) * sizeof(int)));
  });
  if (err != cudaSuccess) return (int)err;
  const QdLayout at = qd_layout(requests, kv_heads, heads / kv_heads, D, window, longest);
  float* states = (float*)scratch;
  float2* sums = (float2*)(scratch + at.sums);
  launch_kernel(kernel, dim3(at.ctas), dim3(QD_THREADS), shared + (requests + 1) * sizeof(int), stream, k_map, v_map, (const bf16*)q, k_scales,
                v_scales, (bf16*)out, decode_seg, seg_q_start, seg_pos0, block_table, seg_slot, table_width, requests,
                heads, kv_heads, page_shift, block_shift, pool_pages, window, scale * 1.4426950408889634f, states, sums, error_word);
  launch_kernel(merge_quantized_decode_kernel<D, NH>, dim3(requests * kv_heads), dim3(8 * NH * D / 4), 0, stream, states, sums, (bf16*)out, decode_seg,
                seg_q_start, seg_pos0, requests, heads, kv_heads, window, at.ctas);
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

// Bytes of scratch memory (on a 16-byte boundary) that a call needs.
MLR_EXPORT long long mlr_attention_quantized_decode_bytes(int requests, int kv_heads, int group, int dim, int window, int longest) {
  return qd_layout(requests, kv_heads, group, dim, window, longest).total;
}

// q, out: [rows, heads * dim] bfloat16, of which the rows of `requests` decoded tokens are attended (decode_seg: their segments, or null for
// segments 0, 1, ..); pools [pages, kv_heads, page_size, dim]; scales [pages, kv_heads, page_size / block]; longest: keys of the longest context
// (a longer one is attended all the same); scratch: memory of the size above; error_word: host-visible int that
// receives a code if a wait runs out.
MLR_EXPORT int mlr_attention_quantized_decode(const void* q, const void* k_pool, const void* v_pool, const float* k_scales, const float* v_scales,
                                              void* out, const int* decode_seg, const int* seg_q_start, const int* seg_pos0, const int* block_table,
                                              const int* seg_slot, int table_width, int requests, int heads, int kv_heads, int dim, int page_size,
                                              int block, int pool_pages, int window, float scale, int longest, void* scratch,
                                              int* error_word, cudaStream_t stream) {
  if (requests == 0) return MLR_OK;
  if (requests < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || table_width <= 0 || pool_pages <= 0 || longest <= 0 || error_word == nullptr)
    return MLR_BAD_SIZE;
  const int page_shift = shift_of(page_size), block_shift = shift_of(block);
  if ((dim != 64 && dim != 128) || page_shift < 4 || block_shift < 0 || block > page_size) return MLR_BAD_SIZE;
  if (heads / kv_heads > 16 || requests > QD_MOST_REQUESTS) return MLR_TOO_LARGE;
  if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)k_pool | (uintptr_t)v_pool | (uintptr_t)scratch) & 15) return MLR_BAD_ALIGNMENT;
  const bool wide = heads / kv_heads > 8;
#define MLR_DECODE(D_, N_)                                                                                                                       \
  return quantized_decode_launch<D_, N_>(q, k_pool, v_pool, k_scales, v_scales, out, decode_seg, seg_q_start, seg_pos0, block_table, seg_slot,   \
                                         table_width, requests, heads, kv_heads, page_shift, block_shift, pool_pages, window, scale, longest,    \
                                         (uint8_t*)scratch, error_word, stream)
  if (dim == 64) { if (wide) MLR_DECODE(64, 2); MLR_DECODE(64, 1); }
  if (wide) MLR_DECODE(128, 2);
  MLR_DECODE(128, 1);
#undef MLR_DECODE
}
