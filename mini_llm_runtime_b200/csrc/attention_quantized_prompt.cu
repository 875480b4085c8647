// Prompt portions over keys and values in 8 bits on the 5th-generation tensor cores, bfloat16 queries, head sizes 64 and 128.
//
// What bounds a prompt's attention is its products and its softmax, not the bytes of its keys: a key is read by every 128 query rows of
// each head.  So its codes are turned into float16 once, by a kernel of its own, and not by each of them: 8,048 keys of 4
// heads of 128 cost 25 MB of memory traffic beside 206 GFLOP.
//
//   prepare     K' = code * ks / 2^a, V' = code * vs / 2^b in float16, a and b whole numbers for each 64 keys of a kv head (the
//               exponents of their largest scales); Q' = q / 2^c in float16, c for each row and head.  A key whose scale is not finite gets K' =
//               NaN and V' = 0: NaN reaches the rows that see it and no others.  Rounding to float16's 11 bits is half of what
//               the weights' own rounding adds; codes times scales have too many bits for any 16.
//   attend      scores s = Q' K'^T; x = s * 2^(a + c) scale log2 e + b; weights 2^(x - base), which carry V's powers of two, in float16; out = sum
//               weights V' / sum (weights / 2^b): a factor and an exponent for each tile of 64 keys, nothing per key.
//   wide tiles  The largest scale may be that of a key which a row does not see.  Where a tile's value scales lie further apart than 2^6, or
//               a key's scale too far below the largest for K' to have all bits, every key has its own a and b: then a row's weights
//               and sums are those of the keys that it sees, whatever lies beside them.
//
// The attending kernel is the one of the bfloat16 cache in its roles: 128 query rows of one head are a work item; four warps of
// softmax (a thread per row), one that issues the products, one that loads; two CTAs per SM; items drawn heaviest first, long ones
// cut into parts that the last one merges.  The prepared keys of a request and kv head lie one behind the other, so a tile
// is one or two bulk copies and there is no block table to read.  Every wait is bounded; a wait that runs out reports through the
// error word, and the CTA goes on without waiting (its result is invalid, the host raises).  2,048 rows behind 6,000 keys, 28 heads
// of 128 over 4: 283 us (0.73 PFLOP/s), 19 of them to prepare.  The chain from scores to weights to the next product bounds it: one group of
// softmax warps and one buffer of weights a CTA, so that tile j's weights wait for tile j - 1's product (tensor pipe 37 % of cycles, 1.4 instructions of four).
#include <cuda_fp16.h>

#include "tcgen05.cuh"

namespace mlr {

constexpr int QP_ROWS = 128, QP_KEYS = 64, QP_SOFTMAX = 128, QP_THREADS = QP_SOFTMAX + 64;
constexpr uint32_t QP_TMEM_COLS = 256, QP_TMEM_O = 2 * QP_KEYS;     // S0 | S1 | O
constexpr int QP_P_BYTES = QP_ROWS * QP_KEYS * 2;
constexpr int QP_PREPARE = 256;
// The base follows the running max in steps of more than this; weights up to 2^8 are far from float16's end.
constexpr float QP_LAZY = 8.f;

// ------------------------------------------------------------------ what is read, in float16
// Tiles of 64 keys of the segments longer than one row, one segment behind the other, within it one kv head behind the other.
struct QpSegment {
  int base_tile, tiles;      // first tile of 64 keys that a row of the segment sees, and how many
};
__device__ __forceinline__ QpSegment qp_segment(int q_len, int pos0, int window) {
  if (q_len < 2) return QpSegment{0, 0};
  const int base = (window > 0 ? max(0, pos0 - window + 1) : 0) / QP_KEYS;
  return QpSegment{base, (pos0 + q_len - 1) / QP_KEYS - base + 1};
}

__device__ __forceinline__ uint32_t qp_pack(float a, float b) {
  const __half2 pair = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&pair);
}
// 2^e as the largest power of two not above a positive number, from 2^-100 (zero and below too) to 2^126; 2^-e; e
constexpr float QP_LEAST = 7.888609e-31f, QP_MOST = 8.507059e37f;
__device__ __forceinline__ float qp_power(float x) { return __uint_as_float(__float_as_uint(fminf(fmaxf(x, QP_LEAST), QP_MOST)) & 0x7f800000u); }
__device__ __forceinline__ float qp_over(float power) { return __uint_as_float((254u << 23) - __float_as_uint(power)); }
// 2^-e for whole e: with 1.5 * 2^23 on it, 127 - e stands in the low bits
__device__ __forceinline__ float qp_two_to_minus(float e) { return __uint_as_float(__float_as_uint(12583039.f - e) << 23); }
__device__ __forceinline__ float qp_exponent(float power) { return (float)((int)(__float_as_uint(power) >> 23) - 127); }
// Scales of a tile that share their powers of two: of values within 2^6 (weights of a row that sees only the smallest keep 18 of float16's 24
// powers of two below the largest), of keys within 2^14 (codes times them are ordinary float16 numbers; zeros always).  Numbers of
// their own cost a tile two reads of them in the middle of its softmax: 2,048 rows behind 6,000 with all tiles wide 520 us, with none 283.
constexpr float QP_NEAR_VALUES = 1.f / 64.f, QP_NEAR_KEYS = 1.f / 16384.f;

// Units: tiles of a kv head, then groups of 8 (row, head) pairs of q.
template <int D>
__global__ void __launch_bounds__(QP_PREPARE)
quantized_prompt_prepare_kernel(const bf16* q, const int8_t* k_pool, const int8_t* v_pool, const float* k_scales, const float* v_scales,
                                __half* __restrict__ q_out, float* __restrict__ q_factor, __half* __restrict__ k_out, __half* __restrict__ v_out,
                                float2* __restrict__ tile_factor, float2* __restrict__ key_factor, int* __restrict__ seg_tile0, const int* __restrict__ seg_q_len,
                                const int* __restrict__ seg_pos0, const int* __restrict__ block_table, const int* __restrict__ seg_slot, int segments,
                                int table_width, int pairs, int kv_heads, int page_size, int block, int pool_pages, int window, int most_tiles,
                                int* __restrict__ control, int control_len) {
  __shared__ int warp_sums[QP_PREPARE / 32];
  __shared__ int found_segment, found_first;
  __shared__ float scales[2][QP_KEYS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_trigger();
  const int key_units = most_tiles * kv_heads;
  if ((int)blockIdx.x >= key_units) {
    // a warp per row and head of q: power of two, float16
    const long long pair = (long long)(blockIdx.x - key_units) * (QP_PREPARE / 32) + warp;
    pdl_wait();
    if (pair >= pairs) return;
    constexpr int EACH = D / 32;
    float v[EACH];
    unsigned top = 0;
    if constexpr (EACH == 4) {
      const uint2 raw = __ldcg(reinterpret_cast<const uint2*>(q + pair * D) + lane);
      v[0] = __uint_as_float(raw.x << 16); v[1] = __uint_as_float(raw.x & 0xffff0000u);
      v[2] = __uint_as_float(raw.y << 16); v[3] = __uint_as_float(raw.y & 0xffff0000u);
    } else {
      const uint32_t raw = __ldcg(reinterpret_cast<const uint32_t*>(q + pair * D) + lane);
      v[0] = __uint_as_float(raw << 16); v[1] = __uint_as_float(raw & 0xffff0000u);
    }
#pragma unroll
    for (int e = 0; e < EACH; ++e) top = max(top, __float_as_uint(v[e]) & 0x7fffffffu);
    top = __reduce_max_sync(0xffffffffu, top);
    const unsigned exponent = min(top >> 23, 253u);
    const bool scaled = exponent >= 1u && top < 0x7f800000u;
    const float down = scaled ? __uint_as_float((254u - exponent) << 23) : 1.f;
    if constexpr (EACH == 4)
      reinterpret_cast<uint2*>(q_out + pair * D)[lane] = make_uint2(qp_pack(v[0] * down, v[1] * down), qp_pack(v[2] * down, v[3] * down));
    else
      reinterpret_cast<uint32_t*>(q_out + pair * D)[lane] = qp_pack(v[0] * down, v[1] * down);
    if (lane == 0) q_factor[pair] = scaled ? __uint_as_float(exponent << 23) : 1.f;
    return;
  }
  // ---- which segment's tile (the segments' sizes are metadata of the step; the call's own memory is not written before the wait: launches
  // before this one may still use it for a call of their own)
  const int unit = blockIdx.x;
  if (threadIdx.x == 0) found_segment = -1;
  int carried = 0;
  for (int first = 0; first < segments; first += QP_PREPARE) {
    const int index = first + threadIdx.x;
    const int tiles = index < segments ? qp_segment(seg_q_len[index], seg_pos0[index], window).tiles : 0;
    int inclusive = tiles;
#pragma unroll
    for (int offset = 1; offset < 32; offset <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, inclusive, offset);
      if (lane >= offset) inclusive += up;
    }
    __syncthreads();
    if (lane == 31) warp_sums[warp] = inclusive;
    __syncthreads();
    int base = carried;
#pragma unroll
    for (int w = 0; w < QP_PREPARE / 32; ++w) {
      if (w < warp) base += warp_sums[w];
      carried += warp_sums[w];
    }
    const int before = base + inclusive - tiles;
    if (index < segments && unit / kv_heads >= before && unit / kv_heads < before + tiles) { found_segment = index; found_first = before; }
  }
  __syncthreads();
  const int segment = found_segment;
  pdl_wait();                              // (all: whoever waits for this launch waits for the one before it too)
  if (unit == 0)
    for (int i = threadIdx.x; i < control_len; i += QP_PREPARE) control[i] = 0;      // the queue and the counters of the launch that follows
  if (segment < 0) return;                 // a window left fewer tiles than were counted
  if (unit == found_first * kv_heads && threadIdx.x == 0) seg_tile0[segment] = found_first;      // (read of segments that have tiles)
  const int q_len = seg_q_len[segment], pos0 = seg_pos0[segment];
  const QpSegment mine = qp_segment(q_len, pos0, window);
  const int within = unit - found_first * kv_heads, kv_head = within / mine.tiles, key0 = (mine.base_tile + within - kv_head * mine.tiles) * QP_KEYS;
  const int last = pos0 + q_len - 1, lowest = window > 0 ? max(0, pos0 - window + 1) : 0;
  const int* table = block_table + (size_t)(seg_slot != nullptr ? seg_slot[segment] : segment) * table_width;
  auto line_of = [&](int key, int* offset) -> long long {      // -1: no such key
    const int logical = key / page_size;
    const int page = key >= lowest && key <= last && logical < table_width ? table[logical] : -1;
    *offset = key - logical * page_size;
    return page >= 0 && page < pool_pages ? (long long)page * kv_heads + kv_head : -1;
  };
  if (threadIdx.x < 2 * QP_KEYS) {
    const int values = threadIdx.x / QP_KEYS, j = threadIdx.x - values * QP_KEYS;
    int offset;
    const long long line = line_of(key0 + j, &offset);
    scales[values][j] = line >= 0 ? (values ? v_scales : k_scales)[line * (page_size / block) + offset / block] : 0.f;
  }
  __syncthreads();
  float power[2];
  bool near = true;            // of this lane's keys
#pragma unroll
  for (int values = 0; values < 2; ++values) {
    float top = 0.f;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float s = scales[values][lane + 32 * e];
      if (s < INFINITY) top = fmaxf(top, s);
    }
    power[values] = qp_power(warp_max(top));
  }
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int key = key0 + lane + 32 * e;
    const float ks = scales[0][lane + 32 * e], vs = scales[1][lane + 32 * e];
    if (key < lowest || key > last || !(ks < INFINITY && vs < INFINITY)) continue;      // no row sees it, or it gives NaN
    near = near && (ks <= 0.f || qp_power(ks) >= power[0] * QP_NEAR_KEYS) && qp_power(vs) >= power[1] * QP_NEAR_VALUES;
  }
  const bool wide = !__all_sync(0xffffffffu, near);      // the same in every warp
  if (threadIdx.x == 0) tile_factor[unit] = make_float2(wide ? -1.f : power[0], wide ? 0.f : qp_exponent(power[1]));
  if (wide && threadIdx.x < QP_KEYS) {
    const float ks = scales[0][threadIdx.x], vs = scales[1][threadIdx.x];
    key_factor[(size_t)unit * QP_KEYS + threadIdx.x] = make_float2(ks < INFINITY ? qp_power(ks) : 1.f, vs < INFINITY ? qp_exponent(qp_power(vs)) : 0.f);
  }
  const float inverse[2] = {qp_over(power[0]), qp_over(power[1])};
  constexpr int PIECES = D / 16;
#pragma unroll
  for (int idx = threadIdx.x; idx < QP_KEYS * PIECES * 2; idx += QP_PREPARE) {
    const int values = idx / (QP_KEYS * PIECES), at = idx - values * (QP_KEYS * PIECES), j = at / PIECES, c = at - j * PIECES;
    int offset;
    const long long line = line_of(key0 + j, &offset);
    uint4 raw = make_uint4(0u, 0u, 0u, 0u);
    if (line >= 0) raw = __ldcg(reinterpret_cast<const uint4*>((values ? v_pool : k_pool) + (line * page_size + offset) * D) + c);
    const bool finite = scales[0][j] < INFINITY && scales[1][j] < INFINITY;
    const float own = scales[values][j];
    const float factor = finite ? own * (wide ? qp_over(qp_power(own)) : inverse[values]) : values ? 0.f : __int_as_float(0x7fffffff);
    const uint32_t words[4] = {raw.x, raw.y, raw.z, raw.w};
    uint32_t packed[8];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      float v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = (float)(int8_t)(words[w] >> (8 * e)) * factor;
      packed[2 * w] = qp_pack(v[0], v[1]);
      packed[2 * w + 1] = qp_pack(v[2], v[3]);
    }
    uint4* dst = reinterpret_cast<uint4*>((values ? v_out : k_out) + ((size_t)unit * QP_KEYS + j) * D) + 2 * c;
    dst[0] = make_uint4(packed[0], packed[1], packed[2], packed[3]);
    dst[1] = make_uint4(packed[4], packed[5], packed[6], packed[7]);
  }
}

// ------------------------------------------------------------------ attention
template <int D>
struct QpShape {
  static constexpr int HALVES = D / 64, STAGES = D == 64 ? 4 : 2;
  static constexpr int Q_BYTES = QP_ROWS * D * 2, Q_HALF_BYTES = QP_ROWS * 128;
  static constexpr int TILE_BYTES = QP_KEYS * D * 2, STAGE_BYTES = 2 * TILE_BYTES, HALF_BYTES = QP_KEYS * 128;
  static constexpr int DATA_BYTES = Q_BYTES + QP_P_BYTES + STAGES * STAGE_BYTES;
};
struct QpControl {
  uint64_t q_full, k_full[4], v_full[4], qk_done[4], pv_done[4], p_ready;
  uint32_t tmem_holder;
  int item, last;
};
constexpr int QP_CONTROL_BYTES = 256;
static_assert(sizeof(QpControl) <= QP_CONTROL_BYTES, "control block");
// kind::f16 with float16 operands (format 0) and a float32 accumulator
__host__ __device__ constexpr uint32_t qp_idesc(int m, int n, bool b_mn_major) {
  return (1u << 4) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

template <int D>
__global__ void __launch_bounds__(QP_THREADS, 2)
quantized_prompt_attention_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
                                  const __grid_constant__ CUtensorMap v_map, const float* q_factor, const float2* tile_factor, const float2* key_factor,
                                  const int* seg_tile0, bf16* __restrict__ out, const int* __restrict__ tile_seg, const int* __restrict__ tile_row0,
                                  const int* __restrict__ seg_q_start, const int* __restrict__ seg_q_len, const int* __restrict__ seg_pos0,
                                  int num_tiles, int heads, int kv_heads, int window, float scale_log2, int* queue, int* error_word, int max_parts,
                                  int tiles_per_unit, float* __restrict__ scratch, int* __restrict__ counters, int shared_bytes) {
  using Shape = QpShape<D>;
  constexpr int STAGES = Shape::STAGES;
  extern __shared__ uint8_t qp_shared_raw[];
  uint8_t* aligned = (uint8_t*)(((uintptr_t)qp_shared_raw + 1023) & ~(uintptr_t)1023);
  if (aligned + Shape::DATA_BYTES + QP_CONTROL_BYTES > qp_shared_raw + shared_bytes) {
    // the launch gave no room for the 1024-byte alignment the swizzled tiles need
    if (threadIdx.x == 0) atomicCAS(error_word, 0, 0x8f);
    return;
  }
  uint8_t* q_tile = aligned;
  uint8_t* p_tile = aligned + Shape::Q_BYTES;
  uint8_t* ring = p_tile + QP_P_BYTES;
  QpControl& ctl = *reinterpret_cast<QpControl*>(ring + STAGES * Shape::STAGE_BYTES);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(&ctl.q_full, 1);
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&ctl.k_full[s], 1); mbar_init(&ctl.qk_done[s], 1);
      mbar_init(&ctl.v_full[s], 1); mbar_init(&ctl.pv_done[s], 1);
    }
    mbar_init(&ctl.p_ready, 4);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&q_map) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&k_map) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&v_map) : "memory");
  }
  if (warp == 4) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&ctl.tmem_holder)), "r"(QP_TMEM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fa_fence_before();
  pdl_trigger();
  __syncthreads();
  fa_fence_after();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, ctl.tmem_holder, 0);
  pdl_wait();

  const int total_items = num_tiles * heads, total_units = total_items * max_parts;
  unsigned tiles_before = 0, items_before = 0;      // rings and phases run on across items
  unsigned asked[2] = {0, 0};                       // tiles of keys, of values that the loading warp has asked for
  bool gave_up = false;
  for (;;) {
    if (threadIdx.x == 0) ctl.item = atomicAdd(&queue[0], 1);
    __syncthreads();
    const int unit = ctl.item;
    if (unit >= total_units) break;
    const int part = unit / total_items, item = unit - part * total_items;
    const int tile = item / heads, head = item - tile * heads, kv_head = head / (heads / kv_heads);
    const int seg = tile_seg[tile], row0 = tile_row0[tile];
    const int q_start = seg_q_start[seg], q_len = seg_q_len[seg], pos0 = seg_pos0[seg];
    const int rows = min(QP_ROWS, q_len - row0);
    const int first_pos = pos0 + row0, last_pos = first_pos + rows - 1;
    auto lowest_of = [&](int position) { return window > 0 ? max(0, position - window + 1) : 0; };
    const int item_begin = lowest_of(first_pos) / QP_KEYS, item_tiles = last_pos / QP_KEYS - item_begin + 1;
    const int parts = min(max_parts, (item_tiles + tiles_per_unit - 1) / tiles_per_unit);
    if (part >= parts) {
      __syncthreads();              // ctl.item is rewritten by the next draw
      continue;
    }
    const int per_part = (item_tiles + parts - 1) / parts;
    const int tile_begin = item_begin + part * per_part, tiles = min(per_part, item_tiles - part * per_part);
    const QpSegment prepared = qp_segment(q_len, pos0, window);
    // of the prepared tiles: this item's first
    const int prepared0 = __ldcg(seg_tile0 + seg) * kv_heads + kv_head * prepared.tiles + tile_begin - prepared.base_tile;

    if (warp == 5) {
      // ------------------------------------------------------------ loads
      auto load_tile = [&](int j, bool values) {
        const unsigned load = tiles_before + (unsigned)j;
        const int stage = load % STAGES;
        const unsigned use = load / STAGES;
        uint64_t* full = values ? &ctl.v_full[stage] : &ctl.k_full[stage];
        if (use > 0) fa_wait(values ? &ctl.pv_done[stage] : &ctl.qk_done[stage], (use - 1) & 1u, error_word, 0x81, gave_up);
        gave_up = __any_sync(0xffffffffu, gave_up);
        if (gave_up) return;
        if (lane == 0) {
          mbar_expect_tx(full, (uint32_t)Shape::TILE_BYTES);
          uint8_t* dst = ring + (size_t)stage * Shape::STAGE_BYTES + (values ? Shape::TILE_BYTES : 0);
#pragma unroll
          for (int half = 0; half < Shape::HALVES; ++half)
            tma_load_2d(values ? &v_map : &k_map, full, dst + half * Shape::HALF_BYTES, half * 64, (prepared0 + j) * QP_KEYS);
        }
        asked[values] = load + 1;
        __syncwarp();
      };
      if (lane == 0) {
        mbar_expect_tx(&ctl.q_full, Shape::Q_BYTES);
#pragma unroll
        for (int half = 0; half < Shape::HALVES; ++half)
          tma_load_2d(&q_map, &ctl.q_full, q_tile + half * Shape::Q_HALF_BYTES, head * D + half * 64, q_start + row0);
      }
      __syncwarp();
      for (int j = 0; j < STAGES && j < tiles; ++j) { load_tile(j, false); load_tile(j, true); }
      if (STAGES < tiles) load_tile(STAGES, false);       // where tile 0's K was
      for (int j = 1; j < tiles; ++j) {
        // in the order in which the stages come free: V of tile j + STAGES - 1 goes where tile j - 1's was, K of tile j + STAGES where tile j's was
        if (j + STAGES - 1 < tiles) load_tile(j + STAGES - 1, true);
        if (j + STAGES < tiles) load_tile(j + STAGES, false);
      }
    } else if (warp == 4) {
      // ------------------------------------------------------------ products
      constexpr uint32_t idesc_qk = qp_idesc(QP_ROWS, QP_KEYS, false), idesc_pv = qp_idesc(QP_ROWS, D, true);
      const uint64_t q_desc = fa_desc_k_major(smem_u32(q_tile)), k_desc0 = fa_desc_k_major(smem_u32(ring));
      const uint64_t v_desc0 = fa_desc_mn_major(smem_u32(ring) + Shape::TILE_BYTES, Shape::HALF_BYTES), p_desc = fa_desc_k_major(smem_u32(p_tile));
      auto issue_qk = [&](int j) {
        const unsigned t = __shfl_sync(0xffffffffu, tiles_before + (unsigned)j, 0);
        const int stage = t % STAGES, buffer = t & 1;
        fa_wait(&ctl.k_full[stage], (t / STAGES) & 1u, error_word, 0x82, gave_up);
        // (the score buffer is free: the probabilities of tile j - 2 arrived after its scores had been read)
        gave_up = __any_sync(0xffffffffu, gave_up);
        fa_fence_after();
        if (!gave_up && elect_one()) {
          const uint64_t k_desc = k_desc0 + (uint64_t)((stage * Shape::STAGE_BYTES) >> 4);
#pragma unroll
          for (int k = 0; k < D / 16; ++k)
            fa_mma(tmem_base + buffer * QP_KEYS, q_desc + (uint64_t)(((k >> 2) * Shape::Q_HALF_BYTES + (k & 3) * 32) >> 4),
                   k_desc + (uint64_t)(((k >> 2) * Shape::HALF_BYTES + (k & 3) * 32) >> 4), idesc_qk, k > 0 ? 1u : 0u);
          fa_commit(&ctl.qk_done[stage]);
        }
        __syncwarp();
      };
      fa_wait(&ctl.q_full, items_before & 1u, error_word, 0x84, gave_up);
      issue_qk(0);
      if (tiles > 1) issue_qk(1);
      for (int j = 0; j < tiles; ++j) {
        const unsigned t = __shfl_sync(0xffffffffu, tiles_before + (unsigned)j, 0);
        const int stage = t % STAGES;
        fa_wait(&ctl.p_ready, t & 1u, error_word, 0x85, gave_up);
        fa_wait(&ctl.v_full[stage], (t / STAGES) & 1u, error_word, 0x8a, gave_up);
        gave_up = __any_sync(0xffffffffu, gave_up);
        fa_fence_after();
        if (!gave_up && elect_one()) {
          const uint64_t v_desc = v_desc0 + (uint64_t)((stage * Shape::STAGE_BYTES) >> 4);
#pragma unroll
          for (int k = 0; k < QP_KEYS / 16; ++k)       // the output rows accumulate over the unit's tiles
            fa_mma(tmem_base + QP_TMEM_O, p_desc + (uint64_t)((k * 32) >> 4), v_desc + (uint64_t)((k * 2048) >> 4), idesc_pv, (j > 0 || k > 0) ? 1u : 0u);
          fa_commit(&ctl.pv_done[stage]);
        }
        __syncwarp();
        if (j + 2 < tiles) issue_qk(j + 2);
      }
    } else {
      // ------------------------------------------------------------ softmax, one thread per query row
      const int r = threadIdx.x, position = first_pos + r;
      const int limit_hi = r < rows ? position : -1, limit_lo = lowest_of(position);
      const uint32_t lane_base = tmem_base + ((uint32_t)(warp * 32) << 16);
      // every row of this warp sees all of a tile that ends at or before the warp's first position and begins at or after the start of
      // its last row's window
      const bool warp_full = warp * 32 + 31 < rows;
      const int warp_first = first_pos + warp * 32, warp_lo = lowest_of(first_pos + min(rows - 1, warp * 32 + 31));
      const float row_factor = r < rows ? __ldcg(q_factor + (size_t)(q_start + row0 + r) * heads + head) * scale_log2 : 1.f;
      float m_run = -INFINITY;      // running max of x (base-2 exponents)
      float m_base = -INFINITY;     // what sum, weights and output are relative to
      float l = 0.f;
      float2 next = __ldcg(tile_factor + prepared0);
      for (int j = 0; j < tiles; ++j) {
        const unsigned t = tiles_before + (unsigned)j;
        const int buffer = t & 1, stage = t % STAGES, key0 = (tile_begin + j) * QP_KEYS;
        const bool wide = next.x < 0.f;
        // (a product too small for a number would make NaN of what is hidden; scores that small are zero)
        const float factor = wide ? 1.f : fmaxf(next.x * row_factor, 1e-36f), exponent = next.y;
        const float4* key_pairs = reinterpret_cast<const float4*>(key_factor + (size_t)(prepared0 + j) * QP_KEYS);
        if (j + 1 < tiles) next = __ldcg(tile_factor + prepared0 + j + 1);
        fa_wait(&ctl.qk_done[stage], (t / STAGES) & 1u, error_word, 0x86, gave_up);
        fa_fence_after();
        float s[QP_KEYS];
#pragma unroll
        for (int c = 0; c < QP_KEYS; c += 16) fa_tmem_load16(lane_base + buffer * QP_KEYS + c, reinterpret_cast<uint32_t*>(s) + c);
        fa_tmem_wait_ld();
        fa_fence_before();
        if (!(warp_full && key0 + QP_KEYS - 1 <= warp_first && key0 >= warp_lo)) {
#pragma unroll
          for (int c = 0; c < QP_KEYS; ++c) {
            const int key = key0 + c;
            if (!(key >= limit_lo && key <= limit_hi)) s[c] = -INFINITY;
          }
        }
        if (wide) {
#pragma unroll
          for (int c = 0; c < QP_KEYS; c += 2) {
            const float4 pair = __ldcg(key_pairs + c / 2);
            s[c] = fmaf(s[c], fmaxf(pair.x * row_factor, 1e-36f), pair.y);
            s[c + 1] = fmaf(s[c + 1], fmaxf(pair.z * row_factor, 1e-36f), pair.w);
          }
        }
        float part_max[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
        for (int c = 4; c < QP_KEYS - 4; c += 8) {
#pragma unroll
          for (int e = 0; e < 4; ++e) part_max[e] = fa_max3(part_max[e], s[c + 2 * e], s[c + 2 * e + 1]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) part_max[e] = fmaxf(part_max[e], s[QP_KEYS - 4 + e]);
        const float tile_max = fmaxf(fmaxf(part_max[0], part_max[1]), fmaxf(part_max[2], part_max[3]));
        m_run = fmaxf(m_run, fmaf(tile_max, factor, exponent));     // the factor is positive
        // (-inf) - (-inf) is NaN and compares false: nothing visible yet, no step; the first visible key sets the base
        const bool step = m_run - m_base > QP_LAZY;
        const float alpha = step ? fa_exp2(m_base - m_run) : 1.f;
        if (step) m_base = m_run;
        const float base = (m_base == -INFINITY ? 0.f : m_base) - exponent;
        const float2 factor2 = make_float2(factor, factor), minus_base = make_float2(-base, -base);
        float2 part_sum[4] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
        for (int c = 0; c < QP_KEYS; c += 8) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 x = __ffma2_rn(make_float2(s[c + 2 * e], s[c + 2 * e + 1]), factor2, minus_base);
            s[c + 2 * e] = fa_exp2(x.x);
            s[c + 2 * e + 1] = fa_exp2(x.y);
            part_sum[e] = __fadd2_rn(part_sum[e], make_float2(s[c + 2 * e], s[c + 2 * e + 1]));
          }
        }
        const float2 sum2 = __fadd2_rn(__fadd2_rn(part_sum[0], part_sum[1]), __fadd2_rn(part_sum[2], part_sum[3]));
        float tile_sum = (sum2.x + sum2.y) * fa_exp2(-exponent);
        if (wide) {
          tile_sum = 0.f;
#pragma unroll
          for (int c = 0; c < QP_KEYS; c += 2) {
            const float4 pair = __ldcg(key_pairs + c / 2);
            tile_sum += fmaf(s[c], qp_two_to_minus(pair.y), s[c + 1] * qp_two_to_minus(pair.w));
          }
        }
        l = fmaf(l, alpha, tile_sum);

        // The output rows in tensor memory are touched only when a row of this warp moved its base.  The previous tile's product is
        // waited for on every tile all the same: the one buffer of weights must have been read.
        const bool rescale = j > 0 && __any_sync(0xffffffffu, step);
        if (j > 0) {
          fa_wait(&ctl.pv_done[(t - 1) % STAGES], ((t - 1) / STAGES) & 1u, error_word, 0x87, gave_up);
          fa_fence_after();
        }
        if (rescale) {
          const float2 alpha2 = make_float2(alpha, alpha);
#pragma unroll
          for (int c = 0; c < D; c += 32) {
            float o[32];
            fa_tmem_load16(lane_base + QP_TMEM_O + c, reinterpret_cast<uint32_t*>(o));
            fa_tmem_load16(lane_base + QP_TMEM_O + c + 16, reinterpret_cast<uint32_t*>(o) + 16);
            fa_tmem_wait_ld();
#pragma unroll
            for (int d = 0; d < 32; d += 2) {
              const float2 scaled = __fmul2_rn(make_float2(o[d], o[d + 1]), alpha2);
              o[d] = scaled.x;
              o[d + 1] = scaled.y;
            }
            fa_tmem_store16(lane_base + QP_TMEM_O + c, reinterpret_cast<const uint32_t*>(o));
            fa_tmem_store16(lane_base + QP_TMEM_O + c + 16, reinterpret_cast<const uint32_t*>(o) + 16);
          }
          fa_tmem_wait_st();
        }
        {
          uint8_t* p_row = p_tile + r * 128;
#pragma unroll
          for (int chunk = 0; chunk < 8; ++chunk) {
            uint32_t packed[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) packed[e] = qp_pack(s[chunk * 8 + 2 * e], s[chunk * 8 + 2 * e + 1]);
            *reinterpret_cast<uint4*>(p_row + ((chunk ^ (r & 7)) << 4)) = make_uint4(packed[0], packed[1], packed[2], packed[3]);
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        fa_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl.p_ready);
      }
      // the finished output rows, after the last tile's product
      {
        const unsigned t = tiles_before + (unsigned)tiles - 1;
        fa_wait(&ctl.pv_done[t % STAGES], (t / STAGES) & 1u, error_word, 0x89, gave_up);
        fa_fence_after();
        constexpr int STATE = D + 2;
        // a part's state of row r: base, sum, unnormalised output; laid out [value][row]
        float* states = scratch + (size_t)item * max_parts * STATE * QP_ROWS + r;
        float* mine = states + (size_t)part * STATE * QP_ROWS;
        bf16* dst = out + ((size_t)(q_start + row0 + r) * heads + head) * D;
        auto store32 = [&](int c, const float* o, float factor) {
#pragma unroll
          for (int chunk = 0; chunk < 4; ++chunk) {
            uint32_t packed[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const __nv_bfloat162 pair = __floats2bfloat162_rn(o[chunk * 8 + 2 * e] * factor, o[chunk * 8 + 2 * e + 1] * factor);
              packed[e] = *reinterpret_cast<const uint32_t*>(&pair);
            }
            *reinterpret_cast<uint4*>(dst + c + chunk * 8) = make_uint4(packed[0], packed[1], packed[2], packed[3]);
          }
        };
        const float inv = 1.f / l;
#pragma unroll
        for (int c = 0; c < D; c += 32) {
          float o[32];
          fa_tmem_load16(lane_base + QP_TMEM_O + c, reinterpret_cast<uint32_t*>(o));
          fa_tmem_load16(lane_base + QP_TMEM_O + c + 16, reinterpret_cast<uint32_t*>(o) + 16);
          fa_tmem_wait_ld();
          if (parts == 1) {
            if (r < rows) store32(c, o, inv);
          } else {
#pragma unroll
            for (int d = 0; d < 32; ++d) mine[(2 + c + d) * QP_ROWS] = o[d];
          }
        }
        fa_fence_before();
        if (parts > 1) {
          mine[0] = m_base;
          mine[QP_ROWS] = l;
          __threadfence();
          asm volatile("bar.sync 1, 128;" ::: "memory");
          if (threadIdx.x == 0) ctl.last = (atomicAdd(&counters[item], 1) == parts - 1);
          asm volatile("bar.sync 1, 128;" ::: "memory");
          if (ctl.last) {
            __threadfence();
            float m_all = -INFINITY;
            for (int p = 0; p < parts; ++p) m_all = fmaxf(m_all, __ldcg(states + (size_t)p * STATE * QP_ROWS));
            if (r < rows) {
              float share[8];
              float l_all = 0.f;
#pragma unroll
              for (int p = 0; p < 8; ++p) {                 // in the order of the parts
                share[p] = 0.f;
                if (p < parts) {
                  const float* theirs = states + (size_t)p * STATE * QP_ROWS;
                  const float top = __ldcg(theirs);
                  share[p] = top == -INFINITY ? 0.f : fa_exp2(top - m_all);      // a part that saw nothing (or no number: its sum is NaN)
                  l_all = fmaf(__ldcg(theirs + QP_ROWS), share[p], l_all);
                }
              }
              const float inv_all = 1.f / l_all;
#pragma unroll
              for (int c = 0; c < D; c += 32) {
                float o[32];
#pragma unroll
                for (int d = 0; d < 32; ++d) o[d] = 0.f;
#pragma unroll
                for (int p = 0; p < 8; ++p) {
                  if (p < parts) {
                    const float* theirs = states + (size_t)p * STATE * QP_ROWS + (size_t)(2 + c) * QP_ROWS;
#pragma unroll
                    for (int d = 0; d < 32; ++d) o[d] = fmaf(__ldcg(theirs + d * QP_ROWS), share[p], o[d]);
                  }
                }
                store32(c, o, inv_all);
              }
            }
          }
        }
      }
    }
    tiles_before += (unsigned)tiles;
    items_before += 1;
    __syncthreads();                // Q, P and ctl.item are rewritten by the next item
  }

  if (warp == 5 && gave_up) {
    // a wait ran out: the copies under way end before the CTA does
    bool late = false;
    for (int values = 0; values < 2; ++values)
      for (unsigned load = asked[values] > STAGES ? asked[values] - STAGES : 0; load < asked[values]; ++load)
        fa_wait(values ? &ctl.v_full[load % STAGES] : &ctl.k_full[load % STAGES], (load / STAGES) & 1u, error_word, 0x8b, late);
    if (items_before > 0) fa_wait(&ctl.q_full, (items_before - 1) & 1u, error_word, 0x8c, late);
  }
  fa_fence_before();
  __syncthreads();
  if (warp == 4) {
    fa_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(QP_TMEM_COLS) : "memory");
  }
}

// Few items with long key ranges are cut into up to 8 parts, so that every CTA that the device holds gets one.
struct QpParts {
  int parts, per_unit;        // per_unit: tiles of keys
};
static QpParts qp_parts(long long items, int longest, int dim) {
  constexpr long long MOST_STATES = 64ll << 20;
  const int resident = sm_count() * 2, most_tiles = longest / QP_KEYS + 1;
  int target = (int)((resident + items - 1) / items);
  target = target < 1 ? 1 : target > 8 ? 8 : target;
  int per_unit = (most_tiles + target - 1) / target;
  if (per_unit < 4) per_unit = 4;
  int parts = (most_tiles + per_unit - 1) / per_unit;
  if (parts > 8) parts = 8;
  if (parts <= 1 || items * parts * QP_ROWS * (dim + 2) * (long long)sizeof(float) > MOST_STATES) return {1, 1 << 30};
  return {parts, per_unit};
}

// Where the parts of a call's memory lie (bytes), for `key_tiles` tiles of 64 keys of all long segments.  A call shares none of it with another
// one, which may run beside it on another stream: `control` is the attending kernel's queue and a counter per item in parts, zeroed by
// the preparing one.
struct QpLayout {
  long long q, q_factor, k, v, tile_factor, key_factor, seg_tile0, control, states, total;
  int control_len;
};
static QpLayout qp_layout(long long key_tiles, long long q_rows, int heads, int kv_heads, int dim, int segments, int tiles, int longest) {
  auto next = [](long long at) { return (at + 1023) / 1024 * 1024; };
  const long long items = (long long)tiles * heads;
  const int parts = qp_parts(items, longest, dim).parts;
  QpLayout at{};
  at.k = next(at.q + q_rows * heads * dim * 2);
  at.v = next(at.k + key_tiles * kv_heads * QP_KEYS * dim * 2);
  at.q_factor = next(at.v + key_tiles * kv_heads * QP_KEYS * dim * 2);
  at.tile_factor = next(at.q_factor + q_rows * heads * 4);
  at.key_factor = next(at.tile_factor + key_tiles * kv_heads * 8);
  at.seg_tile0 = next(at.key_factor + key_tiles * kv_heads * QP_KEYS * 8);
  at.control = next(at.seg_tile0 + (long long)segments * 4);
  at.control_len = 1 + (parts > 1 ? (int)items : 0);
  at.states = next(at.control + (long long)at.control_len * 4);
  at.total = next(at.states + (parts > 1 ? items * parts * QP_ROWS * (dim + 2) * 4 : 0));
  return at;
}

template <int D>
static int qp_launch(const void* q, const void* k_pool, const void* v_pool, const float* k_scales, const float* v_scales, void* out,
                     const int* tile_seg, const int* tile_row0, const int* seg_q_start, const int* seg_q_len, const int* seg_pos0,
                     const int* block_table, const int* seg_slot, int table_width, int segments, int tiles, int key_tiles, int q_rows, int heads,
                     int kv_heads, int page_size, int block, int pool_pages, int window, float scale, int longest, uint8_t* prepared,
                     int* error_word, cudaStream_t stream) {
  using Shape = QpShape<D>;
  const QpLayout at = qp_layout(key_tiles, q_rows, heads, kv_heads, D, segments, tiles, longest);
  int* control = (int*)(prepared + at.control);
  CUtensorMap q_map, k_map, v_map;
  const long long key_rows = (long long)key_tiles * kv_heads * QP_KEYS;
  if (!cached_tile_map(&q_map, prepared + at.q, q_rows, (long long)heads * D, QP_ROWS) || !cached_tile_map(&k_map, prepared + at.k, key_rows, D, QP_KEYS) ||
      !cached_tile_map(&v_map, prepared + at.v, key_rows, D, QP_KEYS))
    return MLR_BAD_SIZE;
  const int pairs = q_rows * heads, per = QP_PREPARE / 32;
  launch_kernel(quantized_prompt_prepare_kernel<D>, dim3(key_tiles * kv_heads + (pairs + per - 1) / per), dim3(QP_PREPARE), 0, stream, (const bf16*)q,
                (const int8_t*)k_pool, (const int8_t*)v_pool, k_scales, v_scales, (__half*)(prepared + at.q), (float*)(prepared + at.q_factor),
                (__half*)(prepared + at.k), (__half*)(prepared + at.v), (float2*)(prepared + at.tile_factor), (float2*)(prepared + at.key_factor),
                (int*)(prepared + at.seg_tile0), seg_q_len, seg_pos0, block_table, seg_slot, segments, table_width, pairs, kv_heads, page_size, block, pool_pages, window, key_tiles,
                control, at.control_len);
  int status = launch_status();
  if (status != MLR_OK) return status;
  // (with head size 128 two CTAs fit an SM only without a spare kilobyte for aligning the tiles; the kernel checks that it starts aligned)
  const size_t shared = (D < 128 ? 1024 : 0) + (size_t)Shape::DATA_BYTES + QP_CONTROL_BYTES;
  static_assert(2 * ((D < 128 ? 1024 : 0) + Shape::DATA_BYTES + QP_CONTROL_BYTES + 1024) <= 228 * 1024, "two CTAs per SM");
  static OncePerDevice once;
  const cudaError_t err = once([&] { return cudaFuncSetAttribute(quantized_prompt_attention_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)shared); });
  if (err != cudaSuccess) return (int)err;
  const long long items = (long long)tiles * heads;
  const int resident = sm_count() * 2;
  const auto [parts, per_unit] = qp_parts(items, longest, D);
  const long long units = items * parts;
  launch_kernel(quantized_prompt_attention_kernel<D>, dim3((int)(units < resident ? units : resident)), dim3(QP_THREADS), shared, stream, q_map, k_map,
                v_map, (const float*)(prepared + at.q_factor), (const float2*)(prepared + at.tile_factor), (const float2*)(prepared + at.key_factor),
                (const int*)(prepared + at.seg_tile0), (bf16*)out, tile_seg, tile_row0, seg_q_start, seg_q_len, seg_pos0, tiles, heads, kv_heads, window, scale * 1.4426950408889634f, control, error_word,
                parts, per_unit, (float*)(prepared + at.states), control + 1, (int)shared);
  return launch_status();
}

}  // namespace mlr

using namespace mlr;

MLR_DEFINE_PDL_SWITCH

// Bytes of memory (on a 16-byte boundary) that a call needs for itself, by what it gets.
MLR_EXPORT long long mlr_attention_quantized_prompt_bytes(int key_tiles, int q_rows, int heads, int kv_heads, int dim, int segments, int tiles,
                                                          int longest) {
  return qp_layout(key_tiles, q_rows, heads, kv_heads, dim, segments, tiles, longest).total;
}

// The segments longer than one row.  q, out: [q_rows, heads * dim] bfloat16; pools [pages, kv_heads, page_size, dim]; scales [pages, kv_heads,
// page_size / block]; tile_seg / tile_row0: tiles of up to 128 rows of a segment, best ordered by falling key count; key_tiles: sum over the long
// segments of their keys in tiles of 64; longest: keys of the longest context; prepared: memory of the size above; scale > 0.
MLR_EXPORT int mlr_attention_quantized_prompt(const void* q, const void* k_pool, const void* v_pool, const float* k_scales, const float* v_scales,
                                              void* out, const int* tile_seg, const int* tile_row0, const int* seg_q_start, const int* seg_q_len,
                                              const int* seg_pos0, const int* block_table, const int* seg_slot, int table_width, int segments,
                                              int tiles, int key_tiles, int q_rows, int heads, int kv_heads, int dim, int page_size, int block,
                                              int pool_pages, int window, float scale, int longest, void* prepared, int* error_word,
                                              cudaStream_t stream) {
  if (tiles == 0) return MLR_OK;
  if (tiles < 0 || key_tiles <= 0 || q_rows <= 0 || segments <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || page_size <= 0 ||
      block <= 0 || page_size % block || table_width <= 0 || pool_pages <= 0 || longest <= 0 || !(scale > 0.f))
    return MLR_BAD_SIZE;
  if (dim != 64 && dim != 128) return MLR_BAD_SIZE;
  if ((long long)tiles * heads >= (1ll << 27) || (long long)q_rows * heads >= (1ll << 30) || (long long)key_tiles * kv_heads * QP_KEYS >= (1ll << 30))
    return MLR_TOO_LARGE;
  if ((((uintptr_t)q | (uintptr_t)k_pool | (uintptr_t)v_pool) & 15) || ((uintptr_t)prepared & 15)) return MLR_BAD_ALIGNMENT;
#define MLR_PROMPT(D_)                                                                                                                          \
  return qp_launch<D_>(q, k_pool, v_pool, k_scales, v_scales, out, tile_seg, tile_row0, seg_q_start, seg_q_len, seg_pos0, block_table, seg_slot, \
                       table_width, segments, tiles, key_tiles, q_rows, heads, kv_heads, page_size, block, pool_pages, window, scale, longest,   \
                       (uint8_t*)prepared, error_word, stream)
  if (dim == 64) MLR_PROMPT(64);
  MLR_PROMPT(128);
#undef MLR_PROMPT
}
