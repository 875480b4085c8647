// A projection of many rows with low-rank adapters on the 5th-generation tensor cores, in one product (bfloat16):
//
//   y = [x | u_a ..] [W | B_a ..]^T + b        u[m] = scale (x[m] A[a]^T), computed before (adapters.cu)
//
// The adapters extend the sum over K: behind the k blocks of x and W come, for every adapter a that a row of this tile has, blocks of rank
// columns.  Their left operand is u, every row with the sums of its own adapter, the same for all adapters; their right operand is B[a];
// and they accumulate in the rows of a alone: the lanes of the other rows are switched off, so nothing needs zeros, and an adapter that is
// not finite stays with its own rows.  All of it accumulates where the shared product does, in float32 in tensor memory, so the result is
// rounded once and an adapter costs its products and the reading of B, no pass over y.  (A kernel that adds the adapters to a shared
// product in float32 reads and writes 0.5 GB more at 2,048 x 37,888 with K = 3,584 and rank 64: 1,135 us against 500, of which the sums u
// are 20; 1.12 PFLOP/s, the tensor pipe busy for 72 %.)  u comes in bfloat16 parts of eight bits each, as many left operands for one right
// one: two for a bfloat16 result, u to 2^-16, a small part of that result's own rounding (2^-8); three for a float32 result, all of u.
// Every part has u's sign and is zero only where u is: an infinite entry of B gives an infinity with each of them, as it does with u.
//
// One CTA computes 128 or 256 rows (one or two accumulators) x BN columns.  Warp 0 loads (bulk tensor copies into a ring of
// 128-byte-swizzled tiles), warp 1 issues the products, warps 2 to 5 list the tile's adapters while the shared product runs,
// lay out u where the first stages held x, and write the result.  (Left operands of each adapter by itself, with zeros in
// the other rows, built anew for each: 160 rows of 40 adapters, 896 x 1,152, 105 us.)
// Every wait is bounded; one that runs out stores a code into the error word, and the CTA frees its tensor memory and ends.
#include "tcgen05.cuh"

namespace mlr {

constexpr int AT_THREADS = 192;
constexpr int AT_MAX_STAGES = 6;

struct AdapterGemm {
  int M, N, K, adapters, rank, stages;
  int parts, held;            // parts of u, and how many of them lie in shared memory at a time: no more than there are stages
  const bf16* bias;
  const float* u;             // [M, rank]
  const int* row_adapter;     // [M]
  void* out;
  int out_f32;
  int* error_word;
};

// A product of 128 rows that leaves the rows (tensor-memory lanes) whose bits are set as they are.
__device__ __forceinline__ void at_mma_rows(uint32_t tmem_d, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint4 off) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, 1, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%4, %5, %6, %7}, p;\n\t}"
      ::"r"(tmem_d), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(off.x), "r"(off.y), "r"(off.z), "r"(off.w) : "memory");
}
// The first eight bits of the number one step of float32 closer to zero than x: of x's sign and less in magnitude, so that what is left of x
// has its sign too and is not zero.  (Of an infinity the largest bfloat16, which leaves the infinity; NaN leaves NaN.)
__device__ __forceinline__ float at_part(float x) {
  const uint32_t bits = __float_as_uint(x);
  return __uint_as_float((bits - ((bits << 1) != 0u ? 1u : 0u)) & 0xffff0000u);
}
template <int N> struct Parts { static constexpr int value = N; };
// The next bfloat16 part of two numbers, taken off them; last: what is left of them, rounded (of the third part exactly: of u's 24 bits no
// more than eight are left, or the one that follows them).
__device__ __forceinline__ uint32_t at_take_part(float& x0, float& x1, bool last) {
  const float h0 = last ? x0 : at_part(x0), h1 = last ? x1 : at_part(x1);
  x0 -= h0;
  x1 -= h1;
  const __nv_bfloat162 pair = __floats2bfloat162_rn(h0, h1);
  return *reinterpret_cast<const uint32_t*>(&pair);
}
__device__ __forceinline__ void at_wait(uint64_t* bar, uint32_t parity, int* error_word, int code, bool& gave_up) {
  if (!gave_up) gave_up = !mbar_wait(bar, parity, error_word, code);
}

template <int BN, int HALVES>
__global__ void __launch_bounds__(AT_THREADS, HALVES == 1 ? 2 : 1)
adapter_gemm_kernel(const __grid_constant__ CUtensorMap x_map, const __grid_constant__ CUtensorMap w_map,
                    const __grid_constant__ CUtensorMap up_map, const AdapterGemm p) {
  constexpr int BM = 128 * HALVES;
  constexpr uint32_t HALF_BYTES = 128 * 64 * 2, A_BYTES = HALVES * HALF_BYTES, B_BYTES = BN * 64 * 2, STAGE_BYTES = A_BYTES + B_BYTES;
  constexpr uint32_t TMEM_COLS = BN * HALVES;
  extern __shared__ uint8_t at_raw[];
  uint8_t* tiles = (uint8_t*)(((uintptr_t)at_raw + 1023) & ~(uintptr_t)1023);
  __shared__ uint64_t full[AT_MAX_STAGES], empty[AT_MAX_STAGES], listed, base_done, u_ready, u_free, done;
  __shared__ uint32_t tmem_holder;
  __shared__ uint4 rows_off[BM][HALVES];      // of a listed adapter: the rows that are not its own
  __shared__ int ids[BM], list[BM], place[BM], list_count, failed;

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int stages = p.stages;
  const int row0 = blockIdx.x * BM, n0 = blockIdx.y * BN;
  // the extension's rounds: 64 ranks, `held` parts of u
  const int base_blocks = (p.K + 63) / 64, passes = (p.parts + p.held - 1) / p.held, rounds = (p.rank + 63) / 64 * passes;
  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    mbar_init(&listed, 1);
    mbar_init(&base_done, 1);
    mbar_init(&u_ready, 4);
    mbar_init(&u_free, 1);
    mbar_init(&done, 1);
    list_count = 0;
    failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&x_map) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&w_map) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&up_map) : "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_holder)), "r"(TMEM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fa_fence_before();
  __syncthreads();
  fa_fence_after();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, tmem_holder, 0);
  bool gave_up = false;

  if (warp == 0) {
    // ------------------------------------------------------------ loads
    if (lane == 0) {
      auto load_x = [&](int s, int k) {
#pragma unroll
        for (int half = 0; half < HALVES; ++half)
          tma_load_2d(&x_map, &full[s], tiles + (size_t)s * STAGE_BYTES + half * HALF_BYTES, k, row0 + half * 128);
      };
      auto load_w = [&](int s, int k) { tma_load_2d(&w_map, &full[s], tiles + (size_t)s * STAGE_BYTES + A_BYTES, k, n0); };
      const int ahead = min(stages, base_blocks);
      int issued = ahead;      // blocks asked for
      // The kernel before, which makes u, let this one in after its own wait: x was complete then.  The warps that read u wait.
      for (int i = 0; i < ahead; ++i) {
        mbar_expect_tx(&full[i], STAGE_BYTES);
        load_x(i, i * 64);
        load_w(i, i * 64);
      }
      for (int i = ahead; i < base_blocks; ++i) {
        const int s = i % stages;
        at_wait(&empty[s], (unsigned)(i / stages - 1) & 1u, p.error_word, 0x91, gave_up);
        if (gave_up) break;
        mbar_expect_tx(&full[s], STAGE_BYTES);
        load_x(s, i * 64);
        load_w(s, i * 64);
        issued = i + 1;
      }
      at_wait(&listed, 0u, p.error_word, 0x92, gave_up);
      const int blocks = gave_up ? 0 : list_count * rounds;
      for (int e = 0; e < blocks; ++e) {
        const int i = base_blocks + e, s = i % stages;
        if (i >= stages) at_wait(&empty[s], (unsigned)(i / stages - 1) & 1u, p.error_word, 0x93, gave_up);
        if (gave_up) break;
        mbar_expect_tx(&full[s], B_BYTES);
        const int round = e / list_count, adapter = list[e - round * list_count];
        tma_load_2d(&up_map, &full[s], tiles + (size_t)s * STAGE_BYTES + A_BYTES, round / passes * 64, adapter * p.N + n0);
        issued = i + 1;
      }
      // no copy is under way when the CTA ends, should a wait of another warp have run out
      for (int i = max(0, issued - stages); i < issued; ++i) mbar_wait(&full[i % stages], (unsigned)(i / stages) & 1u, p.error_word, 0x9b);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ products
    constexpr uint32_t idesc = fa_idesc(128, BN, false);
    const uint64_t a_desc0 = fa_desc_k_major(smem_u32(tiles)), b_desc0 = fa_desc_k_major(smem_u32(tiles) + A_BYTES);
    for (int i = 0; i < base_blocks && !gave_up; ++i) {
      const int s = i % stages;
      at_wait(&full[s], (unsigned)(i / stages) & 1u, p.error_word, 0x94, gave_up);
      gave_up = __any_sync(0xffffffffu, gave_up);
      if (gave_up) break;
      fa_fence_after();
      if (elect_one()) {
        const uint64_t a = a_desc0 + (uint64_t)((s * STAGE_BYTES) >> 4), b = b_desc0 + (uint64_t)((s * STAGE_BYTES) >> 4);
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int half = 0; half < HALVES; ++half)
            fa_mma(tmem_base + half * BN, a + (uint64_t)((half * HALF_BYTES + k * 32) >> 4), b + (uint64_t)((k * 32) >> 4), idesc,
                   (i > 0 || k > 0) ? 1u : 0u);
        fa_commit(&empty[s]);
      }
      __syncwarp();
    }
    if (elect_one()) fa_commit(&base_done);
    __syncwarp();
    at_wait(&listed, 0u, p.error_word, 0x95, gave_up);
    gave_up = __any_sync(0xffffffffu, gave_up);
    const int count = list_count;
    for (int round = 0; round < rounds && count > 0 && !gave_up; ++round) {
      at_wait(&u_ready, (unsigned)round & 1u, p.error_word, 0x97, gave_up);
      const int steps = min(4, (p.rank - round / passes * 64 + 15) / 16), parts = min(p.held, p.parts - round % passes * p.held);
      for (int l = 0; l < count; ++l) {
        const int i = base_blocks + round * count + l, s = i % stages;
        at_wait(&full[s], (unsigned)(i / stages) & 1u, p.error_word, 0x96, gave_up);
        gave_up = __any_sync(0xffffffffu, gave_up);
        if (gave_up) break;
        fa_fence_after();
        if (elect_one()) {
          const uint64_t b = b_desc0 + (uint64_t)((s * STAGE_BYTES) >> 4);
          for (int half = 0; half < HALVES; ++half) {
            const uint4 off = rows_off[l][half];
            if ((off.x & off.y & off.z & off.w) == 0xffffffffu) continue;      // none of its rows are in this half
            for (int part = 0; part < parts; ++part)
              for (int k = 0; k < steps; ++k)
                at_mma_rows(tmem_base + half * BN, a_desc0 + (uint64_t)((part * STAGE_BYTES + half * HALF_BYTES + k * 32) >> 4),
                            b + (uint64_t)((k * 32) >> 4), idesc, off);
          }
          fa_commit(&empty[s]);
        }
        __syncwarp();
      }
      if (elect_one()) fa_commit(&u_free);
      __syncwarp();
    }
    if (elect_one()) fa_commit(&done);
    __syncwarp();
  } else {
    // ------------------------------------------------------------ the tile's adapters, the extension's left operands, the result
    const int quarter = warp & 3, t = quarter * 32 + lane;      // tensor-memory lane = row within a half
    pdl_wait();
    pdl_trigger();
    // an adapter is listed where its first row stands, in the order of those rows
#pragma unroll
    for (int half = 0; half < HALVES; ++half) {
      const int m = row0 + half * 128 + t;
      const int id = m < p.M ? __ldcg(p.row_adapter + m) : -1;
      ids[half * 128 + t] = id >= 0 && id < p.adapters ? id : -1;
    }
    asm volatile("bar.sync 1, 128;" ::: "memory");
    int leader[HALVES];      // the first row with this row's adapter
#pragma unroll
    for (int half = 0; half < HALVES; ++half) {
      const int at = half * 128 + t, id = ids[at];
      int j = 0;
      if (id >= 0)
        while (ids[j] != id) ++j;
      leader[half] = id >= 0 ? j : -1;
      // this warp's leaders behind those of the warps (and halves) before it
      const bool leads = id >= 0 && j == at;
      const unsigned mine = __ballot_sync(0xffffffffu, leads);
      for (int turn = 0; turn < 4; ++turn) {
        if (turn == quarter) {
          const int to = list_count + __popc(mine & ((1u << lane) - 1u));
          if (leads) {
            list[to] = id;
            place[at] = to;
#pragma unroll
            for (int h = 0; h < HALVES; ++h) rows_off[to][h] = make_uint4(0xffffffffu, 0xffffffffu, 0xffffffffu, 0xffffffffu);
          }
          __syncwarp();
          if (lane == 0) list_count += __popc(mine);
        }
        asm volatile("bar.sync 1, 128;" ::: "memory");
      }
    }
#pragma unroll
    for (int half = 0; half < HALVES; ++half)
      if (leader[half] >= 0) atomicAnd(reinterpret_cast<unsigned*>(&rows_off[place[leader[half]]][half]) + quarter, ~(1u << lane));
    asm volatile("bar.sync 1, 128;" ::: "memory");
    if (t == 0) mbar_arrive(&listed);
    const int count = list_count;
    for (int round = 0; round < rounds && count > 0; ++round) {
      const int chunk = round / passes, part0 = round % passes * p.held, part1 = part0 + p.held;      // parts kept: [part0, part1)
      // the sums are asked for before their place is free
      float v[HALVES][64];
#pragma unroll
      for (int half = 0; half < HALVES; ++half) {
        const float* from = p.u + (size_t)(row0 + half * 128 + t) * p.rank + chunk * 64;
#pragma unroll
        for (int c = 0; c < 64; c += 4) {
          const float4 four = leader[half] >= 0 && chunk * 64 + c < p.rank ? __ldcg(reinterpret_cast<const float4*>(from + c))
                                                                          : make_float4(0.f, 0.f, 0.f, 0.f);
          v[half][c] = four.x; v[half][c + 1] = four.y; v[half][c + 2] = four.z; v[half][c + 3] = four.w;
        }
      }
      if (round == 0) at_wait(&base_done, 0u, p.error_word, 0x9a, gave_up);
      else at_wait(&u_free, (unsigned)(round - 1) & 1u, p.error_word, 0x98, gave_up);
      auto lay_out = [&](auto parts) {
#pragma unroll
        for (int half = 0; half < HALVES; ++half) {
          uint8_t* row = tiles + half * HALF_BYTES + t * 128;      // the first part kept; the next ones a stage on
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            uint8_t* to = row + ((c ^ (t & 7)) << 4);
#pragma unroll
            for (int part = 0; part < parts.value; ++part) {
              uint32_t packed[4];
#pragma unroll
              for (int q = 0; q < 4; ++q)
                packed[q] = at_take_part(v[half][c * 8 + 2 * q], v[half][c * 8 + 2 * q + 1], part == parts.value - 1);
              if (parts.value == 2 || (part >= part0 && part < part1))
                *reinterpret_cast<uint4*>(to + (part - part0) * STAGE_BYTES) = make_uint4(packed[0], packed[1], packed[2], packed[3]);
            }
          }
        }
      };
      if (p.parts == 2) lay_out(Parts<2>());
      else lay_out(Parts<3>());
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&u_ready);
    }
    at_wait(&done, 0u, p.error_word, 0x99, gave_up);
    if (gave_up) atomicOr(&failed, 1);
    asm volatile("bar.sync 1, 128;" ::: "memory");
    const bool ok = failed == 0;
    fa_fence_after();
    const uint32_t lane_base = tmem_base + ((uint32_t)(quarter * 32) << 16);
    if (ok) {
#pragma unroll 1
      for (int cc = 0; cc < HALVES * BN; cc += 64) {
        const int half = cc / BN, c0 = cc - half * BN, m = row0 + half * 128 + t;
        float v[64];
#pragma unroll
        for (int q = 0; q < 64; q += 16) fa_tmem_load16(lane_base + half * BN + c0 + q, reinterpret_cast<uint32_t*>(v) + q);
        fa_tmem_wait_ld();
        if (m >= p.M) continue;
        const int n = n0 + c0;
        if (p.bias != nullptr)
#pragma unroll
          for (int c = 0; c < 64; ++c) v[c] += n + c < p.N ? __bfloat162float(p.bias[n + c]) : 0.f;
        if (p.out_f32) {
          float* to = (float*)p.out + (size_t)m * p.N + n;
#pragma unroll
          for (int c = 0; c < 64; c += 4) {
            if ((p.N & 3) == 0 && n + c + 4 <= p.N) *reinterpret_cast<float4*>(to + c) = make_float4(v[c], v[c + 1], v[c + 2], v[c + 3]);
            else
#pragma unroll
              for (int q = 0; q < 4; ++q)
                if (n + c + q < p.N) to[c + q] = v[c + q];
          }
        } else {
          bf16* to = (bf16*)p.out + (size_t)m * p.N + n;
#pragma unroll
          for (int c = 0; c < 64; c += 8) {
            if ((p.N & 7) == 0 && n + c + 8 <= p.N) {
              uint32_t packed[4];
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                __nv_bfloat162 pair = __floats2bfloat162_rn(v[c + 2 * q], v[c + 2 * q + 1]);
                packed[q] = *reinterpret_cast<uint32_t*>(&pair);
              }
              *reinterpret_cast<uint4*>(to + c) = make_uint4(packed[0], packed[1], packed[2], packed[3]);
            } else {
#pragma unroll
              for (int q = 0; q < 8; ++q)
                if (n + c + q < p.N) to[c + q] = __float2bfloat16_rn(v[c + q]);
            }
          }
        }
      }
      fa_fence_before();
    }
  }
  __syncthreads();
  if (warp == 1) {
    fa_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS) : "memory");
  }
}

template <int BN, int HALVES>
static int launch(const void* x, const void* w, const void* up, AdapterGemm p, int stages, cudaStream_t stream) {
  constexpr size_t STAGE = HALVES * 128 * 128 + BN * 128;
  p.stages = stages;
  p.parts = p.out_f32 ? 3 : 2;
  p.held = p.parts < stages ? p.parts : stages;
  static OncePerDevice once;
  if (cudaError_t err = once([] {
        return cudaFuncSetAttribute(adapter_gemm_kernel<BN, HALVES>, cudaFuncAttributeMaxDynamicSharedMemorySize, 193 * 1024);
      }))
    return (int)err;
  CUtensorMap x_map, w_map, up_map;
  if (!cached_tile_map(&x_map, x, p.M, p.K, 128) || !cached_tile_map(&w_map, w, p.N, p.K, BN) ||
      !cached_tile_map(&up_map, up, (long long)p.adapters * p.N, p.rank, BN))
    return MLR_BAD_ALIGNMENT;
  const dim3 grid((p.M + 128 * HALVES - 1) / (128 * HALVES), (p.N + BN - 1) / BN);
  if (grid.y > 65535) return MLR_TOO_LARGE;
  launch_kernel(adapter_gemm_kernel<BN, HALVES>, grid, dim3(AT_THREADS), stages * STAGE + 1024, stream, x_map, w_map, up_map, p);
  return launch_status();
}

// Which tile and ring: 128 x 128, 128 x 256 or 256 x 256, with rings that leave an SM to two CTAs (three and two stages) where there are
// more CTAs than SMs, else as deep as 192 KB (six, four, three).  A k block costs the largest of its MMAs (0.14 us per 128 x
// 128), its copies' latency spread over the ring and the SM's share of operand bandwidth, a CTA 1.5 us and its epilogue, and
// a launch so many rounds of CTAs.
struct AdapterPlan { int shape, stages; };
static AdapterPlan plan(int M, int N, int K, int sms) {
  const double kb = (K + 63) / 64;
  AdapterPlan best{0, 3};
  double least = 1e30;
  for (int shape = 0; shape < 3; ++shape) {
    const int bn = shape == 0 ? 128 : 256, halves = shape == 2 ? 2 : 1;
    const long long ctas = (long long)((M + 128 * halves - 1) / (128 * halves)) * ((N + bn - 1) / bn);
    const bool alone = ctas <= sms || shape == 2;
    const int stages = shape == 2 ? 3 : alone ? (shape == 0 ? 6 : 4) : (shape == 0 ? 3 : 2), per_sm = alone ? 1 : 2;
    const long long rounds = (ctas + (long long)per_sm * sms - 1) / ((long long)per_sm * sms);
    const double stage_kb = 16.0 * halves + bn / 8.0;
    double each = 0.14 * (bn / 128) * halves * per_sm;
    if ((0.5 + 0.03 * stage_kb) / stages > each) each = (0.5 + 0.03 * stage_kb) / stages;
    if (per_sm * stage_kb / 112.0 > each) each = per_sm * stage_kb / 112.0;
    const double cost = rounds * (1.5 + kb * each + 1.5 * (bn / 128) * halves + (per_sm == 1 && rounds > 1 ? 4.0 : 0.0));
    if (cost < least) { least = cost; best = {shape, stages}; }
  }
  return best;
}

}  // namespace mlr

using namespace mlr;

MLR_DEFINE_PDL_SWITCH

// To be launched right behind mlr_adapter_down, which lets the next kernel in only after its own wait.
// x [M, K], w [N, K], up [adapters, N, rank], bias [N] or null in bfloat16 on 16-byte boundaries, K % 8 == 0 and rank % 8 == 0;
// u float32 [M, rank] (rows without an adapter are not read); out [M, N] bfloat16 or float32.
MLR_EXPORT int mlr_adapter_gemm(const void* x, const void* w, const void* up, const float* u, const int* row_adapter, const void* bias,
                                void* out, int M, int N, int K, int adapters, int rank, int out_f32, int* error_word, cudaStream_t stream) {
  if (M < 0 || N <= 0 || K <= 0 || adapters <= 0 || rank <= 0 || rank > 128) return MLR_BAD_SIZE;
  if (M == 0) return MLR_OK;
  if (K % 8 != 0 || rank % 8 != 0 || (((uintptr_t)x | (uintptr_t)w | (uintptr_t)up | (uintptr_t)u | (uintptr_t)out) & 15) != 0) return MLR_BAD_ALIGNMENT;
  if ((long long)adapters * N > 0x7fffffffll) return MLR_TOO_LARGE;
  AdapterGemm p{M, N, K, adapters, rank, 0, 0, 0, (const bf16*)bias, u, row_adapter, out, out_f32, error_word};
  const AdapterPlan chosen = plan(M, N, K, sm_count());
  if (chosen.shape == 2) return launch<256, 2>(x, w, up, p, chosen.stages, stream);
  if (chosen.shape == 1) return launch<256, 1>(x, w, up, p, chosen.stages, stream);
  return launch<128, 1>(x, w, up, p, chosen.stages, stream);
}
