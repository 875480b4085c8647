// Attention of decoded tokens whose requests share leading pages: the keys and values of a common prefix are read once for all
// requests of a group, each request's own keys once for itself, and the two are put together.
//
//   o[i,h] = sum_j p_j v_j / sum_j p_j,  p_j = exp(q[i,h] . k_j scale - m)   over j in prefix(i) and own(i)
//
// A part of a row's keys leaves a state (m, l, o): the largest exponent, the sum and the unnormalised output relative to it.
// States of parts add up after scaling by exp(m - max m), in the order of the parts, so the split changes only roundings.
// Exponents, sums and outputs are 32-bit; on the tensor cores the weights p are rounded to bfloat16 for their product with V (beside the
// prefix kernel: what that costs), as they are where each request attends by itself.
//
// Parts of one (request, head), each with a place of its own in scratch memory:
//   0 .. prefix_parts - 1              `chunk` keys of the prefix each, as many as the request's prefix has
//   prefix_parts .. + own_parts - 1    equal parts of the request's own keys, as many as there are (see own_range)
// Rows of a work item: of a prefix, the query heads of one kv head of up to 128 / heads_per_kv requests; of own keys, those of
// one request.  A request whose context ends before its group's keys do sees those of its context (pos0 is device memory: what the lists
// were made for is not known to the host of a captured step).
#include "mma_attention.cuh"
#include "tcgen05.cuh"

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

// A segment's own keys [begin, end) of part `part`, and how many parts have any.
__device__ __forceinline__ int own_range(const PrefixCall& c, int segment, int part, int* begin, int* end) {
  const int first = c.seg_keys[segment], last = c.pos0[segment] + 1;
  const int own = max(0, last - first);
  const int each = max(OWN_LEAST, ((own + c.own_parts - 1) / c.own_parts + 63) & ~63);
  *begin = min(last, first + part * each);
  *end = min(last, *begin + each);
  return (own + each - 1) / each;
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

// CTA = (eight rows of an item, one part of its keys).  PREFIX: y is a tile of the prefixes, else a segment.  Bound by the shared-memory reads of
// its multiply-adds (a 32-bit word for each): float32, 8 requests with 14 heads of 64 over 2, 2,048 shared and 500 own keys 166 us, 32 with 28
// heads of 128 over 4, 4,096 shared keys 530 us; each request by itself (the generic kernel of every other step) 1,032 and 7,906 us.
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
  int row_end[2];                                              // the end of their contexts
#pragma unroll
  for (int i = 0; i < 2; ++i) row_end[i] = 2 * warp + i < rows ? min(end, c.pos0[segment_of(2 * warp + i)] + 1) : end;
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
      if (!open[lane] || key0 + lane >= row_end[i]) s = -INFINITY;
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

// ------------------------------------------------------------------ prefixes on tcgen05 (bfloat16, heads of 64 and 128)
// One work item is 128 query rows of one kv head (the query heads of up to 128 / heads_per_kv requests) over one part of the prefix.
// 70, 33 and 25 requests behind 16,384, 9,001 and 4,100 keys, 40 heads of 128 over 8: 54 us, of which a CTA's 36 tiles of 64 keys take 39, at
// 1,830 cycles each and 1.7 GHz (two CTAs on an SM: 710 exponentials and sums, 310 the row's largest score and the other half's, 370
// storing the probabilities, 190 the previous product, 250 the scores and reading them).  Where a part is short the rest is the larger half: 64
// requests behind 8,192 keys, 28 heads of 128 over 4, eight tiles a CTA, 18.7 us, of a CTA's 15: 2.4 until lists are read and tensor memory is
// there, 2.8 to the scores of the second tile, 6.5 the other tiles, 1.4 the last product, 1.9 the output.  Eleven warps: eight of softmax, two
// threads per query row (tensor-memory lane), 32 keys of a tile each, which lend each other their largest score; one that issues S = Q K^T two
// key tiles ahead and O += P V, P in tensor memory where S was; one that loads K and one that loads V, page by page through bulk tensor copies
// into a ring (one warp for both, sixteen copies per tile with pages of 16 keys, was the limit before: 58 us).  Probabilities are rounded to
// bfloat16 for the product with V, as in the other attention kernels on tensor cores: half a step (2^-8) of each weight, not of the sums, which
// add the 32-bit ones (a result's error 0.0023 of its size, where 32-bit weights and the rounding of the result make 0.0017); a second part
// would add half as many products again.  The output stays in tensor memory relative to a base exponent that follows the running max in steps of 2^8.
// The query rows lie in the q of as many requests: the softmax threads gather them.  (One thread per row with P in shared memory: the
// whole call 102 us where two and P in tensor memory took 97.  Q in tensor memory too leaves room for one tile's scores, softmax and products
// in turn: slower.)
constexpr int PT_ROWS = 128, PT_KEYS = 64, PT_SOFTMAX = 256, PT_THREADS = PT_SOFTMAX + 96;
constexpr int PT_MMA_WARP = PT_SOFTMAX / 32, PT_LOAD_WARP = PT_MMA_WARP + 1 /* keys; values one on */, PT_HALF = PT_KEYS / 2;
constexpr uint32_t PT_TMEM_COLS = 256, PT_TMEM_O = 2 * PT_KEYS;      // S0 | S1, which their probabilities replace | O
constexpr float PT_LAZY = 8.f;

template <int D>
struct PrefixShape {
  static constexpr int HALVES = D / 64;
  static constexpr int STAGES = D == 64 ? 4 : 2;
  static constexpr int Q_BYTES = PT_ROWS * D * 2, Q_HALF = PT_ROWS * 128;
  static constexpr int TILE_BYTES = PT_KEYS * D * 2, HALF = PT_KEYS * 128, STAGE_BYTES = 2 * TILE_BYTES;
  static constexpr int DATA_BYTES = Q_BYTES + STAGES * STAGE_BYTES;
};

struct PrefixControl {
  uint64_t q_full, k_full[4], v_full[4], qk_done[4], pv_done[4], p_ready;
  uint32_t tmem_holder;
  float half_max[2][2][PT_ROWS];      // of tiles in turn: the largest score of either half of a row's keys
};

constexpr int PT_CONTROL_BYTES = 2304;
static_assert(sizeof(PrefixControl) <= PT_CONTROL_BYTES, "control block");
template <int D> constexpr int PT_SHARED = PrefixShape<D>::DATA_BYTES + PT_CONTROL_BYTES + 1024;
static_assert(2 * (PT_SHARED<128> + 1024) <= 228 * 1024, "two CTAs per SM");

template <int D>
__global__ void __launch_bounds__(PT_THREADS, 2)
prefix_parts_tcgen05_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, const PrefixCall c,
                            int page_shift, int* error_word) {
  using Shape = PrefixShape<D>;
  constexpr int STAGES = Shape::STAGES;
  extern __shared__ uint8_t prefix_raw[];
  uint8_t* q_tile = (uint8_t*)(((uintptr_t)prefix_raw + 1023) & ~(uintptr_t)1023);      // [halves][128][64]
  if (q_tile + Shape::DATA_BYTES + PT_CONTROL_BYTES > prefix_raw + PT_SHARED<D>) {      // no room for the alignment
    if (threadIdx.x == 0) atomicCAS(error_word, 0, 0x70);
    return;
  }
  uint8_t* ring = q_tile + Shape::Q_BYTES;                                               // stages of (K, V), each [halves][64][64]
  PrefixControl& ctl = *reinterpret_cast<PrefixControl*>(ring + STAGES * Shape::STAGE_BYTES);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  // Which item and part this CTA is: the parts of all items in a row.  Like the segments' slots and the block table these are
  // the step's metadata, complete before any kernel of the step lets the next one in.
  const int kv_head = blockIdx.y;
  int tile = 0, part = blockIdx.x, keys = 0;
  for (int t0 = 0; t0 < c.tiles; t0 += 32) {
    const int mine = t0 + lane < c.tiles ? c.tile_keys[t0 + lane] : 0;
    const int parts = (mine + c.chunk - 1) / c.chunk;
    int upto = parts;      // parts of the items up to and with this lane's
#pragma unroll
    for (int step = 1; step < 32; step <<= 1) {
      const int other = __shfl_up_sync(0xffffffffu, upto, step);
      if (lane >= step) upto += other;
    }
    const unsigned found = __ballot_sync(0xffffffffu, part < upto);
    if (found != 0u) {
      const int at = __ffs(found) - 1;
      tile = t0 + at;
      part -= __shfl_sync(0xffffffffu, upto - parts, at);
      keys = __shfl_sync(0xffffffffu, mine, at);
      break;
    }
    part -= __shfl_sync(0xffffffffu, upto, 31);
  }
  const int begin = part * c.chunk, end = min(keys, begin + c.chunk);
  if (begin >= end) { pdl_wait(); return; }      // no such part: lists that do not belong to the launch
  const int first_member = c.tile_first[tile];
  if (threadIdx.x == 0) {
    mbar_init(&ctl.q_full, PT_SOFTMAX / 32);
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&ctl.k_full[s], 1); mbar_init(&ctl.qk_done[s], 1);
      mbar_init(&ctl.v_full[s], 1); mbar_init(&ctl.pv_done[s], 1);
    }
    mbar_init(&ctl.p_ready, PT_SOFTMAX / 32);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&k_map) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&v_map) : "memory");
  }
  const int boxes = c.page_size >= PT_KEYS ? 1 : PT_KEYS >> page_shift;
  const int box_rows = c.page_size >= PT_KEYS ? PT_KEYS : c.page_size;
  const int tiles = (end - begin + PT_KEYS - 1) / PT_KEYS;
  const int* table = c.block_table + (size_t)c.seg_slot[c.members[first_member]] * c.table_width;
  auto lookup = [&](int j) -> int {                     // the page of this lane's box of key tile j
    if (j >= tiles || lane >= boxes * Shape::HALVES) return 0;
    const int logical = (begin + j * PT_KEYS + (lane % boxes) * box_rows) >> page_shift;
    return logical < c.table_width ? max(0, table[logical]) : 0;
  };
  const int per = c.heads / c.kv_heads;
  const int rows = c.tile_count[tile] * per;
  // softmax threads: the row's segment and head, and where its q stands; warps w and w + 4 share the rows
  const int r = threadIdx.x & (PT_ROWS - 1);
  const bool live = r < rows;
  const int segment = live ? c.members[first_member + r / per] : 0, head = kv_head * per + r % per;
  const int q_at = live ? c.q_row[segment] * c.heads + head : -1;      // in units of a head
  // keys of the row from this thread's first one on: all of the part's, or as far as its context reaches
  int row_keys = (live ? min(end, c.pos0[segment] + 1) : end) - begin - (threadIdx.x >= PT_ROWS ? PT_HALF : 0);
  int first_pages[STAGES + 2];
  if (warp >= PT_LOAD_WARP) {
#pragma unroll
    for (int j = 0; j < STAGES + 2; ++j) first_pages[j] = lookup(j);
  }
  if (warp == PT_MMA_WARP) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&ctl.tmem_holder)), "r"(PT_TMEM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fa_fence_before();
  __syncthreads();
  fa_fence_after();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, ctl.tmem_holder, 0);
  pdl_wait();                       // before the first read of q and cache
  pdl_trigger();                    // after it: see prefix_own_mma_kernel

  bool gave_up = false;

  if (warp >= PT_LOAD_WARP) {
    // ------------------------------------------------------------ loads: keys by one warp, values by another
    const bool values = warp > PT_LOAD_WARP;
    int issued = 0;      // tiles asked for
    auto load = [&](int j, int page) {
      const int stage = j % STAGES;
      // a stage of keys is free once the scores that read it exist, one of values once its product is done
      if (j >= STAGES) fa_wait(values ? &ctl.pv_done[stage] : &ctl.qk_done[stage], (unsigned)(j / STAGES - 1) & 1u, error_word, 0x71, gave_up);
      gave_up = __any_sync(0xffffffffu, gave_up);
      if (gave_up) return;
      uint64_t* full = values ? &ctl.v_full[stage] : &ctl.k_full[stage];
      if (lane == 0) mbar_expect_tx(full, Shape::TILE_BYTES);
      __syncwarp();
      if (lane < boxes * Shape::HALVES) {
        const int box = lane % boxes, half = lane / boxes;
        const int offset = (begin + j * PT_KEYS + box * box_rows) & (c.page_size - 1);
        uint8_t* dst = ring + (size_t)stage * Shape::STAGE_BYTES + (values ? Shape::TILE_BYTES : 0) + half * Shape::HALF + box * box_rows * 128;
        tma_load_2d(values ? &v_map : &k_map, full, dst, half * 64, (page * c.kv_heads + kv_head) * c.page_size + offset);
      }
      issued = j + 1;
    };
#pragma unroll
    for (int j = 0; j < STAGES; ++j)
      if (j < tiles) load(j, first_pages[j]);
    int pages[2] = {first_pages[STAGES], first_pages[STAGES + 1]};      // of tiles j and j + 1
    for (int j = STAGES; j < tiles; ++j) {
      const int after = lookup(j + 2);
      load(j, pages[0]);
      pages[0] = pages[1];
      pages[1] = after;
    }
    // no copy is under way when the CTA ends, should a wait of another warp have run out
    for (int j = max(0, issued - STAGES); j < issued; ++j)
      mbar_wait(values ? &ctl.v_full[j % STAGES] : &ctl.k_full[j % STAGES], (unsigned)(j / STAGES) & 1u, error_word, 0x7c);
  } else if (warp == PT_MMA_WARP) {
    // ------------------------------------------------------------ MMAs
    constexpr uint32_t idesc_qk = fa_idesc(PT_ROWS, PT_KEYS, false);
    constexpr uint32_t idesc_pv = fa_idesc(PT_ROWS, D, true);
    const uint64_t q_desc = fa_desc_k_major(smem_u32(q_tile)), k_desc0 = fa_desc_k_major(smem_u32(ring));
    const uint64_t v_desc0 = fa_desc_mn_major(smem_u32(ring) + Shape::TILE_BYTES, Shape::HALF);
    auto issue_qk = [&](int j) {      // the columns j & 1 are free: the product with tile j - 2's probabilities is in front of this one
      const int stage = j % STAGES;
      fa_wait(&ctl.k_full[stage], (unsigned)(j / STAGES) & 1u, error_word, 0x72, gave_up);
      gave_up = __any_sync(0xffffffffu, gave_up);
      fa_fence_after();
      if (!gave_up && elect_one()) {
        const uint64_t k_desc = k_desc0 + (uint64_t)((stage * Shape::STAGE_BYTES) >> 4);
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          fa_mma(tmem_base + (j & 1) * PT_KEYS, q_desc + (uint64_t)(((k >> 2) * Shape::Q_HALF + (k & 3) * 32) >> 4),
                 k_desc + (uint64_t)(((k >> 2) * Shape::HALF + (k & 3) * 32) >> 4), idesc_qk, k > 0 ? 1u : 0u);
        fa_commit(&ctl.qk_done[stage]);
      }
      __syncwarp();
    };
    fa_wait(&ctl.q_full, 0u, error_word, 0x73, gave_up);
    issue_qk(0);
    if (tiles > 1) issue_qk(1);
    for (int j = 0; j < tiles; ++j) {
      const int stage = j % STAGES;
      fa_wait(&ctl.p_ready, (unsigned)j & 1u, error_word, 0x74, gave_up);
      fa_wait(&ctl.v_full[stage], (unsigned)(j / STAGES) & 1u, error_word, 0x75, gave_up);
      gave_up = __any_sync(0xffffffffu, gave_up);
      fa_fence_after();
      if (!gave_up && elect_one()) {
        const uint64_t v_desc = v_desc0 + (uint64_t)((stage * Shape::STAGE_BYTES) >> 4);
#pragma unroll
        for (int k = 0; k < PT_KEYS / 16; ++k)
          fa_mma_tmem(tmem_base + PT_TMEM_O, tmem_base + (j & 1) * PT_KEYS + k * 8, v_desc + (uint64_t)((k * 2048) >> 4), idesc_pv,
                      (j > 0 || k > 0) ? 1u : 0u);
        fa_commit(&ctl.pv_done[stage]);
      }
      __syncwarp();
      if (j + 2 < tiles) issue_qk(j + 2);
    }
  } else {
    // ------------------------------------------------------------ softmax, two threads per query row: 32 keys of a tile each
    const int quarter = warp & 3, side = warp >> 2;
    {
      // a warp's 16 of 32 rows, whole rows at a time (a row per lane would touch 32 lines with every load: 4.4 us instead of 1.5)
      constexpr int LANES = D / 8, AT_ONCE = 32 / LANES, LOADS = LANES / 2;      // lanes per row, rows per load
      uint4 piece[LOADS];
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int at = __shfl_sync(0xffffffffu, q_at, side * 16 + i * AT_ONCE + lane / LANES);
        piece[i] = at >= 0 ? __ldcg(reinterpret_cast<const uint4*>((const bf16*)c.q + (size_t)at * D) + lane % LANES) : make_uint4(0u, 0u, 0u, 0u);
      }
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int row = quarter * 32 + side * 16 + i * AT_ONCE + lane / LANES, chunk = lane % LANES;
        *reinterpret_cast<uint4*>(q_tile + (chunk >> 3) * Shape::Q_HALF + row * 128 + (((chunk & 7) ^ (row & 7)) << 4)) = piece[i];
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctl.q_full);
    }
    const uint32_t lane_base = tmem_base + ((uint32_t)(quarter * 32) << 16);
    const bool warp_live = quarter * 32 < rows;      // a warp of no rows only keeps the barriers going
    float m_run = -INFINITY, m_base = -INFINITY, l = 0.f;
    const float2 scale2 = make_float2(c.scale_log2, c.scale_log2);
    for (int j = 0; j < tiles; ++j) {
      const int stage = j % STAGES, key0 = begin + j * PT_KEYS;
      const bool ragged = key0 + PT_KEYS > end;
      fa_wait(&ctl.qk_done[stage], (unsigned)(j / STAGES) & 1u, error_word, 0x76, gave_up);
      fa_fence_after();
      const uint32_t scores = lane_base + (j & 1) * PT_KEYS;
      float s[PT_HALF];
      bool step = false;
      float alpha = 1.f;
      if (warp_live) {
#pragma unroll
        for (int i = 0; i < PT_HALF; i += 16)
          fa_tmem_load16(scores + side * PT_HALF + i, reinterpret_cast<uint32_t*>(s) + i);
        fa_tmem_wait_ld();
        fa_fence_before();
        if (row_keys < PT_HALF) {
#pragma unroll
          for (int i = 0; i < PT_HALF; ++i)
            if (i >= row_keys) s[i] = -INFINITY;
        }
        row_keys -= PT_KEYS;
        float part_max[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
        for (int i = 4; i < PT_HALF - 4; i += 8)
#pragma unroll
          for (int e = 0; e < 4; ++e) part_max[e] = fa_max3(part_max[e], s[i + 2 * e], s[i + 2 * e + 1]);
#pragma unroll
        for (int e = 0; e < 4; ++e) part_max[e] = fmaxf(part_max[e], s[PT_HALF - 4 + e]);
        float tile_max = fmaxf(fmaxf(part_max[0], part_max[1]), fmaxf(part_max[2], part_max[3]));
        // the row's, with the other half's (two places in turn: the tile after next comes behind the next one's barrier)
        ctl.half_max[j & 1][side][r] = tile_max;
        asm volatile("bar.sync %0, 64;" ::"r"(1 + quarter) : "memory");
        fa_fence_after();
        tile_max = fmaxf(tile_max, ctl.half_max[j & 1][side ^ 1][r]);
        m_run = fmaxf(m_run, tile_max * c.scale_log2);
        step = m_run - m_base > PT_LAZY;          // nothing seen yet: NaN, no step
        alpha = step ? fa_exp2(m_base - m_run) : 1.f;
        if (step) m_base = m_run;
        const float base = m_base == -INFINITY ? 0.f : m_base;
        const float2 minus_base = make_float2(-base, -base);
        float2 part_sum[4] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
        for (int i = 0; i < PT_HALF; i += 8)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 x = __ffma2_rn(make_float2(s[i + 2 * e], s[i + 2 * e + 1]), scale2, minus_base);
            s[i + 2 * e] = fa_exp2(x.x);
            s[i + 2 * e + 1] = fa_exp2(x.y);
            part_sum[e] = __fadd2_rn(part_sum[e], make_float2(s[i + 2 * e], s[i + 2 * e + 1]));
          }
        const float2 sum2 = __fadd2_rn(__fadd2_rn(part_sum[0], part_sum[1]), __fadd2_rn(part_sum[2], part_sum[3]));
        l = fmaf(l, alpha, sum2.x + sum2.y);      // of this thread's keys
      }
      const bool rescale = j > 0 && __any_sync(0xffffffffu, step);
      if (j > 0) {      // the previous tile's P V: it has read the probabilities, and the output may be touched
        fa_wait(&ctl.pv_done[(j - 1) % STAGES], (unsigned)((j - 1) / STAGES) & 1u, error_word, 0x77, gave_up);
        fa_fence_after();
      }
      if (rescale) {
        const float2 alpha2 = make_float2(alpha, alpha);
#pragma unroll
        for (int d0 = side * (D / 2); d0 < (side + 1) * (D / 2); d0 += 32) {
          float o[32];
          fa_tmem_load16(lane_base + PT_TMEM_O + d0, reinterpret_cast<uint32_t*>(o));
          fa_tmem_load16(lane_base + PT_TMEM_O + d0 + 16, reinterpret_cast<uint32_t*>(o) + 16);
          fa_tmem_wait_ld();
#pragma unroll
          for (int d = 0; d < 32; d += 2) {
            const float2 scaled = __fmul2_rn(make_float2(o[d], o[d + 1]), alpha2);
            o[d] = scaled.x;
            o[d + 1] = scaled.y;
          }
          fa_tmem_store16(lane_base + PT_TMEM_O + d0, reinterpret_cast<const uint32_t*>(o));
          fa_tmem_store16(lane_base + PT_TMEM_O + d0 + 16, reinterpret_cast<const uint32_t*>(o) + 16);
        }
        fa_tmem_wait_st();
      }
      if (ragged) {      // what stands behind the last key becomes zero: a weight of zero times NaN is NaN
        fa_wait(&ctl.v_full[stage], (unsigned)(j / STAGES) & 1u, error_word, 0x78, gave_up);
        uint8_t* v_tile = ring + (size_t)stage * Shape::STAGE_BYTES + Shape::TILE_BYTES;
        for (int i = threadIdx.x; i < PT_KEYS * 8 * Shape::HALVES; i += PT_SOFTMAX) {
          const int half = i / (PT_KEYS * 8), within = i - half * (PT_KEYS * 8);
          if (key0 + (within >> 3) >= end)
            *reinterpret_cast<uint4*>(v_tile + half * Shape::HALF + (within >> 3) * 128 + (within & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
        }
      }
      if (warp_live) {      // where the row's scores were, which both its threads have read; other rows' outputs are not written
        uint32_t packed[PT_HALF / 2];
#pragma unroll
        for (int e = 0; e < PT_HALF / 2; ++e) packed[e] = pack_bf16(s[2 * e], s[2 * e + 1]);
        fa_tmem_store16(scores + side * (PT_HALF / 2), packed);
        fa_tmem_wait_st();
      }
      if (ragged) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");      // the zeros, for the product
      fa_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctl.p_ready);
    }
    fa_wait(&ctl.pv_done[(tiles - 1) % STAGES], (unsigned)((tiles - 1) / STAGES) & 1u, error_word, 0x79, gave_up);
    fa_fence_after();
    // The output rows through shared memory, so that a warp writes 128 bytes of a row together (a row per lane: 3.7 us, so 2).  All
    // products of this CTA are done: the warp takes its share of the ring's space.
    const int at = live ? segment * c.heads + head : -1;
    constexpr int PITCH = 32 + 4;
    static_assert(PT_SOFTMAX * PITCH * 4 <= Shape::DATA_BYTES, "the rows fit");
    float* mine = reinterpret_cast<float*>(ring) + warp * 32 * PITCH;
    if (side == 1) ctl.half_max[tiles & 1][1][r] = l;   // the row's sum: that of both halves
    asm volatile("bar.sync 5, 256;" ::: "memory");      // every warp's last wait is behind it
#pragma unroll
    for (int d0 = side * (D / 2); d0 < (side + 1) * (D / 2); d0 += 32) {
      float o[32];
      fa_tmem_load16(lane_base + PT_TMEM_O + d0, reinterpret_cast<uint32_t*>(o));
      fa_tmem_load16(lane_base + PT_TMEM_O + d0 + 16, reinterpret_cast<uint32_t*>(o) + 16);
      fa_tmem_wait_ld();
#pragma unroll
      for (int e = 0; e < 32; e += 4)
        *reinterpret_cast<float4*>(mine + lane * PITCH + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
      __syncwarp();
      float* acc = c.acc + (size_t)part * c.segments * c.heads * D + d0 + lane % 8 * 4;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int row = i * 4 + lane / 8, to = __shfl_sync(0xffffffffu, at, row);
        if (to >= 0) *reinterpret_cast<float4*>(acc + (size_t)to * D) = *reinterpret_cast<const float4*>(mine + row * PITCH + lane % 8 * 4);
      }
      __syncwarp();
    }
    if (live && side == 0)
      *reinterpret_cast<float2*>(c.state + 2 * ((size_t)part * c.segments * c.heads + at)) = make_float2(m_base, l + ctl.half_max[tiles & 1][1][r]);
    fa_fence_before();
  }
  __syncthreads();
  if (warp == PT_MMA_WARP) {
    fa_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(PT_TMEM_COLS) : "memory");
  }
}

// ------------------------------------------------------------------ own keys on mma.sync (bfloat16, heads of 64 and 128)
// CTA = (request, part of its own keys, kv head): bound by reading them, each once (231 MB in 51 us, 4.5 TB/s).  Keys are the MMA's rows
// and the query heads its eight columns (S^T = K Q^T, O^T = V^T P^T), so that the usual five to eight heads of a kv head fill them: half
// the products and registers of heads as rows, and three CTAs per SM.  Four warps take 16 keys each of a 64-key tile; a fifth loads, page
// by page through bulk tensor copies, as far ahead as the ring is deep (by asynchronous copies of the four warps each table read stood in
// front of its copies: 68 MB of own keys took 72 us from cold caches).  The warps' states meet in shared memory.
// AFTER_PREFIX: launched behind the prefix kernel, which lets the next kernel in after its own wait: everything before both is done then,
// and what this kernel reads is written by neither; it starts beside the prefix kernel and waits for it at its end.
constexpr int OWN_THREADS = 160;
constexpr int FINISH_PARTS = 64;      // parts of a prefix, at most

template <int D>
struct OwnShape {
  static constexpr int HALVES = D / 64;
  static constexpr int STAGES = D == 64 ? 4 : 2;
  static constexpr int TILE_BYTES = 64 * D * 2, HALF = 64 * 128, STAGE_BYTES = 2 * TILE_BYTES;
  static constexpr int DATA_BYTES = STAGES * STAGE_BYTES;
  static constexpr int PITCH = D + 4;
  static_assert(4 * 16 * (PITCH + 2) * 4 <= DATA_BYTES, "the warps' states fit where the tiles were");
};

// An 8 x 8 matrix of 16-bit elements turned over: row g, columns 2t and 2t + 1 of lane 4g + t.
__device__ __forceinline__ uint32_t turned(uint32_t v) {
  uint32_t w;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(w) : "r"(v));
  return w;
}

// FINISH: one own part per request; the CTA then holds everything but the prefix's parts, and puts them together itself (a
// kernel behind that reads all parts again costs its launch and wait, 5 to 10 us).
template <int D, int NT, bool AFTER_PREFIX, bool FINISH>
__global__ void __launch_bounds__(OWN_THREADS)
prefix_own_mma_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, const PrefixCall c,
                      int page_shift, int* error_word) {
  using Shape = OwnShape<D>;
  constexpr int STAGES = Shape::STAGES, HEADS = NT * 8;
  extern __shared__ uint8_t own_raw[];
  uint8_t* ring = (uint8_t*)(((uintptr_t)own_raw + 1023) & ~(uintptr_t)1023);
  __shared__ uint64_t full[4], empty[4];
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 4); }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  const int segment = blockIdx.y, kv_head = blockIdx.z, part = blockIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int begin, end;
  own_range(c, segment, part, &begin, &end);
  const int first = begin & ~63;      // tiles start where pages and copies do; keys before `begin` are masked
  const int tiles = begin < end ? (end - first + 63) / 64 : 0;
  const int boxes = c.page_size >= 64 ? 1 : 64 >> page_shift, box_rows = c.page_size >= 64 ? 64 : c.page_size;
  const int* table = c.block_table + (size_t)c.seg_slot[segment] * c.table_width;
  auto lookup = [&](int j) -> int {
    if (j >= tiles || lane >= boxes * Shape::HALVES) return 0;
    const int logical = (first + j * 64 + (lane % boxes) * box_rows) >> page_shift;
    return logical < c.table_width ? max(0, table[logical]) : 0;
  };
  int pages[STAGES];
  if (warp == 4) {
#pragma unroll
    for (int j = 0; j < STAGES; ++j) pages[j] = lookup(j);
  }
  const int q_row = c.q_row[segment];
  __syncthreads();
  if (!AFTER_PREFIX) pdl_wait();
  pdl_trigger();
  if (tiles > 0) {
    const int per = c.heads / c.kv_heads;
    bool gave_up = false;
    if (warp == 4) {
      int issued = 0;
      for (int j0 = 0; j0 < tiles; j0 += STAGES) {
#pragma unroll
        for (int i = 0; i < STAGES; ++i) {
          const int j = j0 + i;
          if (j < tiles) {
            const int page = pages[i];
            pages[i] = lookup(j + STAGES);
            if (j0 > 0) fa_wait(&empty[i], (unsigned)(j0 / STAGES - 1) & 1u, error_word, 0x7a, gave_up);
            gave_up = __any_sync(0xffffffffu, gave_up);
            if (!gave_up) {
              if (lane == 0) mbar_expect_tx(&full[i], Shape::STAGE_BYTES);
              __syncwarp();
              if (lane < boxes * Shape::HALVES) {
                const int box = lane % boxes, half = lane / boxes;
                const int y = (page * c.kv_heads + kv_head) * c.page_size + ((first + j * 64 + box * box_rows) & (c.page_size - 1));
                uint8_t* dst = ring + i * Shape::STAGE_BYTES + half * Shape::HALF + box * box_rows * 128;
                tma_load_2d(&k_map, &full[i], dst, half * 64, y);
                tma_load_2d(&v_map, &full[i], dst + Shape::TILE_BYTES, half * 64, y);
              }
              issued = j + 1;
            }
          }
        }
      }
      // no copy is under way when the states take the tiles' place, should a wait of another warp have run out
      for (int j = max(0, issued - STAGES); j < issued; ++j)
        mbar_wait(&full[j % STAGES], (unsigned)(j / STAGES) & 1u, error_word, 0x7d);
    }
    // of heads 2t and 2t + 1 (t = lane & 3) of each eight: output rows d = 16 i + g and 8 further (g = lane / 4)
    float o[D / 16][NT][4];
    float m[NT][2], l[NT][2];
    if (warp < 4) {
      uint32_t q_frag[D / 16][NT][2];
      const bf16* q = (const bf16*)c.q + ((size_t)q_row * c.heads + kv_head * per) * D;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int head = n * 8 + (lane >> 2), column = ks * 16 + (lane & 3) * 2 + e * 8;
            q_frag[ks][n][e] = head < per ? __ldcg(reinterpret_cast<const unsigned*>(q + (size_t)head * D + column)) : 0u;
          }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        m[n][0] = m[n][1] = -INFINITY;
        l[n][0] = l[n][1] = 0.f;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) o[i][n][0] = o[i][n][1] = o[i][n][2] = o[i][n][3] = 0.f;
      }
      for (int j = 0; j < tiles; ++j) {
        const int stage = j % STAGES;
        fa_wait(&full[stage], (unsigned)(j / STAGES) & 1u, error_word, 0x7b, gave_up);
        bf16* k_tile = reinterpret_cast<bf16*>(ring + stage * Shape::STAGE_BYTES);
        bf16* v_tile = k_tile + 64 * D;
        const int key0 = first + j * 64 + warp * 16;
        const bool ragged = key0 < begin || key0 + 15 >= end;
        if (key0 < end && key0 + 15 >= begin) {
          if (ragged) {      // what stands in front of and behind the keys becomes zero: a weight of zero times NaN is NaN
            for (int i = lane; i < 16 * D / 8; i += 32) {
              const int row = i / (D / 8), chunk = i - row * (D / 8);
              if (key0 + row < begin || key0 + row >= end)
                *reinterpret_cast<uint4*>(tile_at<D, true>(v_tile, warp * 16 + row, chunk)) = make_uint4(0u, 0u, 0u, 0u);
            }
            __syncwarp();
          }
          float s[NT][4];
#pragma unroll
          for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
          for (int ks = 0; ks < D / 16; ++ks) {
            uint32_t a[4];
            ldmatrix_x4(a, tile_at<D, true>(k_tile, warp * 16 + (lane & 7) + ((lane >> 3) & 1) * 8, ks * 2 + (lane >> 4)));
#pragma unroll
            for (int n = 0; n < NT; ++n) mma_bf16(s[n], a, q_frag[ks][n][0], q_frag[ks][n][1]);
          }
          uint32_t p[NT][2];
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const int low = key0 + (lane >> 2), high = low + 8;
            const bool see_low = !ragged || (low >= begin && low < end), see_high = !ragged || (high >= begin && high < end);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              s[n][e] = see_low ? s[n][e] * c.scale_log2 : -INFINITY;
              s[n][e + 2] = see_high ? s[n][e + 2] * c.scale_log2 : -INFINITY;
              float top = fmaxf(s[n][e], s[n][e + 2]);
#pragma unroll
              for (int step = 4; step < 32; step <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, step));
              const float now = fmaxf(m[n][e], top), base = now == -INFINITY ? 0.f : now;
              const float alpha = exp2f(m[n][e] - base);
              m[n][e] = now;
              s[n][e] = exp2f(s[n][e] - base);
              s[n][e + 2] = exp2f(s[n][e + 2] - base);
              l[n][e] = fmaf(l[n][e], alpha, s[n][e] + s[n][e + 2]);      // of this lane's keys; the lanes' sums meet at the end
#pragma unroll
              for (int i = 0; i < D / 16; ++i) { o[i][n][e] *= alpha; o[i][n][e + 2] *= alpha; }
            }
            p[n][0] = turned(pack_bf16(s[n][0], s[n][1]));
            p[n][1] = turned(pack_bf16(s[n][2], s[n][3]));
          }
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            uint32_t a[4];
            ldmatrix_x4_trans(a, tile_at<D, true>(v_tile, warp * 16 + (lane & 7) + (lane >> 4) * 8, i * 2 + ((lane >> 3) & 1)));
#pragma unroll
            for (int n = 0; n < NT; ++n) mma_bf16(o[i][n], a, p[n][0], p[n][1]);
          }
          // the zeros before the tensor copy that reuses the stage
          if (ragged) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[stage]);
      }
    }
    // the four warps' states, then their sum
    float* states = reinterpret_cast<float*>(ring);                // [4][HEADS][PITCH], then [4][HEADS][2]
    float* sums = states + 4 * HEADS * Shape::PITCH;
    __syncthreads();
    if (warp < 4) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int head = n * 8 + (lane & 3) * 2 + e;
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            states[(warp * HEADS + head) * Shape::PITCH + i * 16 + (lane >> 2)] = o[i][n][e];
            states[(warp * HEADS + head) * Shape::PITCH + i * 16 + (lane >> 2) + 8] = o[i][n][e + 2];
          }
          float sum = l[n][e];
#pragma unroll
          for (int step = 4; step < 32; step <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, step);
          if (lane < 4) {
            sums[2 * (warp * HEADS + head)] = m[n][e];
            sums[2 * (warp * HEADS + head) + 1] = sum;
          }
        }
    }
    __syncthreads();
    if (!FINISH) {
      const size_t at0 = ((size_t)(c.prefix_parts + part) * c.segments + segment) * c.heads + kv_head * per;
      for (int i = threadIdx.x; i < per * D; i += OWN_THREADS) {
        const int row = i / D, d = i - row * D;
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < 4; ++w) top = fmaxf(top, sums[2 * (w * HEADS + row)]);
        const float base = top == -INFINITY ? 0.f : top;
        float sum = 0.f, value = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float factor = exp2f(sums[2 * (w * HEADS + row)] - base);
          sum = fmaf(sums[2 * (w * HEADS + row) + 1], factor, sum);
          value = fmaf(states[(w * HEADS + row) * Shape::PITCH + d], factor, value);
        }
        c.acc[(at0 + row) * D + d] = value;
        if (d == 0) {
          c.state[2 * (at0 + row)] = top;
          c.state[2 * (at0 + row) + 1] = sum;
        }
      }
    }
  }
  if (AFTER_PREFIX) pdl_wait();
  if (FINISH) {
    // parts of a row: the prefix's, then the four warps' states; their factors first, then the sums of whole rows
    constexpr int LANES = D / 4, ROWS_AT_ONCE = 32 / LANES;
    __shared__ float factors[HEADS][FINISH_PARTS + 4], inverses[HEADS];
    const int per = c.heads / c.kv_heads;
    const int parts = c.chunk > 0 ? (c.seg_keys[segment] + c.chunk - 1) / c.chunk : 0;
    const float* states = reinterpret_cast<const float*>(ring);
    const float* sums = states + 4 * HEADS * Shape::PITCH;
    const size_t row0 = (size_t)segment * c.heads + kv_head * per, pitch = (size_t)c.segments * c.heads;
    for (int row = warp; row < per; row += OWN_THREADS / 32) {
      float2 state[3];
#pragma unroll
      for (int i = 0; i < 3; ++i) {
        const int at = lane + 32 * i;
        state[i] = make_float2(-INFINITY, 0.f);
        if (at < parts) state[i] = __ldcg(reinterpret_cast<const float2*>(c.state) + at * pitch + row0 + row);
        else if (at < parts + 4 && tiles > 0) state[i] = *reinterpret_cast<const float2*>(sums + 2 * ((at - parts) * HEADS + row));
      }
      const float top = warp_max(fmaxf(state[0].x, fmaxf(state[1].x, state[2].x))), base = top == -INFINITY ? 0.f : top;
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 3; ++i) {
        const int at = lane + 32 * i;
        const float factor = exp2f(state[i].x - base);
        sum = fmaf(state[i].y, factor, sum);
        if (at < parts + 4) factors[row][at] = factor;
      }
      sum = warp_sum(sum);
      if (lane == 0) inverses[row] = sum == 0.f ? 0.f : 1.f / sum;      // NaN stays
    }
    __syncthreads();
    for (int r0 = warp * ROWS_AT_ONCE; r0 < per; r0 += OWN_THREADS / 32 * ROWS_AT_ONCE) {
      const int row = r0 + lane / LANES, d = lane % LANES * 4;
      if (row >= per) continue;
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
      auto add = [&](const float4& v, float factor) {
        o.x = fmaf(v.x, factor, o.x); o.y = fmaf(v.y, factor, o.y); o.z = fmaf(v.z, factor, o.z); o.w = fmaf(v.w, factor, o.w);
      };
      const float* from = c.acc + (row0 + row) * D + d;
      for (int k0 = 0; k0 < parts; k0 += 8) {
        float4 v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k)
          v[k] = k0 + k < parts ? __ldcg(reinterpret_cast<const float4*>(from + (size_t)(k0 + k) * pitch * D)) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (k0 + k < parts) add(v[k], factors[row][k0 + k]);
      }
      if (tiles > 0)
#pragma unroll
        for (int w = 0; w < 4; ++w)
          add(*reinterpret_cast<const float4*>(states + (w * HEADS + row) * Shape::PITCH + d), factors[row][parts + w]);
      const float inverse = inverses[row];
      *reinterpret_cast<uint2*>((bf16*)c.out + ((size_t)q_row * c.heads + kv_head * per + row) * D + d) =
          make_uint2(pack_bf16(o.x * inverse, o.y * inverse), pack_bf16(o.z * inverse, o.w * inverse));
    }
  }
}

// ------------------------------------------------------------------ the parts put together
// One warp per (segment, head); a row that sees no key is zero.  Bound by the latency of its reads (64 requests, 28 heads of 128, up to 18
// parts: 11 us from cold caches).  W floats per lane and load (4 where rows are whole 16-byte pieces); the states of up to 32 parts come
// with one load, the outputs of eight parts are in flight together.
template <typename T, int W>
__global__ void __launch_bounds__(128)
prefix_merge_kernel(const PrefixCall c) {
  constexpr int PIECES = 8 / W, AHEAD = W == 4 ? 8 : 4;
  pdl_trigger();
  const int row = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (row >= c.segments * c.heads) { pdl_wait(); return; }
  const int segment = row / c.heads;
  int begin, end;
  const int own = own_range(c, segment, 0, &begin, &end);
  const int prefix = c.chunk > 0 ? (c.seg_keys[segment] + c.chunk - 1) / c.chunk : 0;
  const int parts = prefix + own, q_row = c.q_row[segment];
  const size_t pitch = (size_t)c.segments * c.heads;
  auto place = [&](int part) { return (size_t)(part < prefix ? part : c.prefix_parts + part - prefix) * pitch + row; };
  pdl_wait();
  float top = -INFINITY, sum = 0.f;
  float o[PIECES][W];
#pragma unroll
  for (int i = 0; i < PIECES; ++i)
#pragma unroll
    for (int e = 0; e < W; ++e) o[i][e] = 0.f;
  for (int part0 = 0; part0 < parts; part0 += 32) {
    float2 state = make_float2(-INFINITY, 0.f);
    if (part0 + lane < parts) state = __ldcg(reinterpret_cast<const float2*>(c.state) + place(part0 + lane));
    const float now = fmaxf(top, warp_max(state.x)), base = now == -INFINITY ? 0.f : now;
    const float before = exp2f(top - base), mine = exp2f(state.x - base);
    top = now;
    sum = sum * before + warp_sum(mine * state.y);
#pragma unroll
    for (int i = 0; i < PIECES; ++i)
#pragma unroll
      for (int e = 0; e < W; ++e) o[i][e] *= before;
    const int count = min(32, parts - part0);
    for (int k0 = 0; k0 < count; k0 += AHEAD) {
      float v[AHEAD][PIECES][W];
#pragma unroll
      for (int k = 0; k < AHEAD; ++k)
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
          const int d = (i * 32 + lane) * W;
          const bool there = k0 + k < count && d < c.dim;
          const float* from = c.acc + place(part0 + k0 + k) * c.dim + d;
          if (W == 4) {
            const float4 four = there ? __ldcg(reinterpret_cast<const float4*>(from)) : make_float4(0.f, 0.f, 0.f, 0.f);
            v[k][i][0] = four.x; v[k][i][W > 1 ? 1 : 0] = four.y; v[k][i][W > 2 ? 2 : 0] = four.z; v[k][i][W > 3 ? 3 : 0] = four.w;
          } else {
            v[k][i][0] = there ? __ldcg(from) : 0.f;
          }
        }
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        const float factor = __shfl_sync(0xffffffffu, mine, min(31, k0 + k));
#pragma unroll
        for (int i = 0; i < PIECES; ++i)
#pragma unroll
          for (int e = 0; e < W; ++e)
            if (k0 + k < count) o[i][e] = fmaf(v[k][i][e], factor, o[i][e]);
      }
    }
  }
  const float inverse = sum == 0.f ? 0.f : 1.f / sum;      // NaN stays
  T* to = (T*)c.out + ((size_t)q_row * c.heads + (row - segment * c.heads)) * c.dim;
#pragma unroll
  for (int i = 0; i < PIECES; ++i)
#pragma unroll
    for (int e = 0; e < W; ++e) {
      const int d = (i * 32 + lane) * W + e;
      if (d < c.dim) to[d] = from_float<T>(o[i][e] * inverse);
    }
}

template <typename T>
static void launch_merge(const PrefixCall& c, cudaStream_t stream) {
  launch_kernel(c.dim % 4 == 0 ? prefix_merge_kernel<T, 4> : prefix_merge_kernel<T, 1>, dim3((c.segments * c.heads + 3) / 4), dim3(128), 0, stream, c);
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
  launch_merge<T>(c, stream);
  return launch_status();
}

template <int D, int NT>
static int run_fast(const PrefixCall& c, int units, int* error_word, cudaStream_t stream) {
  static OncePerDevice once[5];
  const size_t prefix_shared = PT_SHARED<D>, own_shared = OwnShape<D>::DATA_BYTES + 1024;
  auto allow = [](auto kernel, size_t bytes) { return [=] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes); }; };
  if (cudaError_t err = once[0](allow(prefix_parts_tcgen05_kernel<D>, prefix_shared))) return (int)err;
  if (cudaError_t err = once[1](allow(prefix_own_mma_kernel<D, NT, true, true>, own_shared))) return (int)err;
  if (cudaError_t err = once[2](allow(prefix_own_mma_kernel<D, NT, true, false>, own_shared))) return (int)err;
  if (cudaError_t err = once[3](allow(prefix_own_mma_kernel<D, NT, false, true>, own_shared))) return (int)err;
  if (cudaError_t err = once[4](allow(prefix_own_mma_kernel<D, NT, false, false>, own_shared))) return (int)err;
  int page_shift = 0;
  while (1 << page_shift < c.page_size) ++page_shift;
  CUtensorMap k_map, v_map;
  const long long rows = (long long)c.pages * c.kv_heads * c.page_size;
  const int box = c.page_size < PT_KEYS ? c.page_size : PT_KEYS;
  if (!cached_tile_map(&k_map, c.k_pool, rows, D, box) || !cached_tile_map(&v_map, c.v_pool, rows, D, box)) return MLR_BAD_ALIGNMENT;
  if (units > 0)
    launch_kernel(prefix_parts_tcgen05_kernel<D>, dim3(units, c.kv_heads), dim3(PT_THREADS), prefix_shared, stream, k_map, v_map, c, page_shift,
                  error_word);
  const bool finish = c.own_parts == 1 && c.prefix_parts <= FINISH_PARTS;
  auto own = units > 0 ? (finish ? prefix_own_mma_kernel<D, NT, true, true> : prefix_own_mma_kernel<D, NT, true, false>)
                       : (finish ? prefix_own_mma_kernel<D, NT, false, true> : prefix_own_mma_kernel<D, NT, false, false>);
  launch_kernel(own, dim3(c.own_parts, c.segments, c.kv_heads), dim3(OWN_THREADS), own_shared, stream, k_map, v_map, c, page_shift, error_word);
  if (!finish) launch_merge<bf16>(c, stream);
  return launch_status();
}

}  // namespace mlr

using namespace mlr;

MLR_DEFINE_PDL_SWITCH

// q, out [rows, heads * dim], pools [pages, kv_heads, page_size, dim] of one dtype.  acc, state: float32, (prefix_parts + own_parts) *
// segments * heads * dim and * 2 of them, on boundaries of 16 and 8 bytes.  fast: the tensor cores (bfloat16, dim 64 or 128, at most 16 heads per kv head, pages of a
// power of two from 8 on, a scale above zero); else any type, size and scale.  chunk: keys of a prefix part; prefix_parts of them
// reach the longest prefix, and all items have `units` parts together.
MLR_EXPORT int mlr_attention_prefix(const void* q, const void* k_pool, const void* v_pool, void* out, const int* q_row, const int* pos0,
                                    const int* seg_slot, const int* block_table, const int* seg_keys, const int* members,
                                    const int* tile_first, const int* tile_count, const int* tile_keys, float* acc, float* state,
                                    int segments, int tiles, int heads, int kv_heads, int dim, int page_size, int pages, int table_width,
                                    int chunk, int prefix_parts, int own_parts, int units, float scale, int dtype, int fast, int* error_word, cudaStream_t stream) {
  if (segments < 0 || tiles < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 || dim <= 0 || page_size <= 0 || pages <= 0 ||
      table_width <= 0 || own_parts <= 0 || prefix_parts < 0 || (tiles > 0 && (chunk <= 0 || prefix_parts <= 0 || units < tiles)))
    return MLR_BAD_SIZE;
  if (segments == 0) return MLR_OK;
  if (dim > 256 || heads / kv_heads > 128 || segments > 65535 || tiles > 65535 || kv_heads > 65535) return MLR_TOO_LARGE;
  if (((uintptr_t)acc & 15) != 0 || ((uintptr_t)state & 7) != 0) return MLR_BAD_ALIGNMENT;
  const PrefixCall c{q, k_pool, v_pool, q_row, pos0, seg_slot, block_table, seg_keys, members, tile_first, tile_count, tile_keys, acc, state, out,
                     segments, tiles, heads, kv_heads, dim, page_size, pages, table_width, chunk, prefix_parts, own_parts,
                     scale * 1.4426950408889634f};
  if (fast) {
    const bool boxes = page_size >= 8 && (page_size & (page_size - 1)) == 0;      // a box of a tile is eight rows at least
    const bool rows_fit = (long long)pages * kv_heads * page_size <= 0x7fffffff && chunk % PT_KEYS == 0;
    if (dtype != MLR_BF16 || heads / kv_heads > 16 || !boxes || !rows_fit || !(scale > 0.f)) return MLR_BAD_SIZE;
    if ((((uintptr_t)q | (uintptr_t)k_pool | (uintptr_t)v_pool) & 15) != 0) return MLR_BAD_ALIGNMENT;
    if (dim == 64) return heads / kv_heads <= 8 ? run_fast<64, 1>(c, units, error_word, stream) : run_fast<64, 2>(c, units, error_word, stream);
    if (dim == 128) return heads / kv_heads <= 8 ? run_fast<128, 1>(c, units, error_word, stream) : run_fast<128, 2>(c, units, error_word, stream);
    return MLR_BAD_SIZE;
  }
  if (dtype == MLR_BF16) return run_plain<bf16>(c, stream);
  if (dtype == MLR_F32) return run_plain<float>(c, stream);
  return MLR_BAD_DTYPE;
}
