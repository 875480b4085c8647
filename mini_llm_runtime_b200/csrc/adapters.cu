// Low-rank adapters of many requests beside a shared projection: row m of y = x W^T + b gains
//
//   scale[a] * (x[m] A[a]^T) B[a]^T        a = row_adapter[m], nothing where a is no adapter
//
// with A [adapters, rank, K] and B [adapters, N, rank].  Two kernels around the shared product:
//
//   down   u[m][r] = scale[a] * sum_k x[m][k] A[a][r][k], float32 [rows, rank].
//   up     y[m][n] = base[m][n] + sum_r u[m][r] B[a][n][r], base being x W^T + b in float32, rounded once.
//
// Which adapter a row has is device memory: a captured step finds the adapters of whatever requests its rows belong to.
// The shared product dominates; an adapter costs rank (K + N) elements, read once per step where its rows lie together.
#include "mma_attention.cuh"

namespace mlr {

constexpr int DOWN_RANKS = 16;       // rank rows per CTA of the few-rows kernel
constexpr int DOWN_WARPS = 4;
constexpr int MOST_PARTS = 8;        // of K: CTAs of a cluster
// Rows up to which every row reads its adapter by itself.  (bfloat16, rows of many adapters, captured, us: 16 ranks of 896 columns 64 rows
// 3.4, of 18,944 11.2 (25 MB, 2.2 TB/s); 128 rows as tiles 49; prompts as tiles: one adapter of 64 ranks for 2,048 rows of 3,584 columns 20.)
constexpr int DOWN_ROWS = 128;
constexpr int TILE_DOWN = 32;        // rows per CTA of the many-rows kernel

__device__ __forceinline__ uint32_t rank_in_cluster() {
  uint32_t rank;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  return rank;
}
__device__ __forceinline__ void cluster_meet() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float read_from_cta(const float* mine, uint32_t rank) {
  uint32_t remote;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(shared_address(mine)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(remote) : "memory");
  return v;
}

template <bool FIRST, typename A, typename B> struct Choice { typedef A type; };
template <typename A, typename B> struct Choice<false, A, B> { typedef B type; };
template <int N> struct Count { static constexpr int value = N; };

// 16 bytes of bfloat16 or float32 as floats.
template <typename T> struct Pack { static constexpr int N = 16 / sizeof(T); };
__device__ __forceinline__ void unpack(const uint4& raw, float* v, bf16) {
  const __nv_bfloat162* pair = reinterpret_cast<const __nv_bfloat162*>(&raw);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __bfloat1622float2(pair[i]);
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void unpack(const uint4& raw, float* v, float) {
  v[0] = __uint_as_float(raw.x); v[1] = __uint_as_float(raw.y); v[2] = __uint_as_float(raw.z); v[3] = __uint_as_float(raw.w);
}

// Both down kernels: `early` says that the kernel in front is the shared product of the same x, which lets the next kernel in
// after its own wait: what is read here was complete then, and the sums are taken beside it; this kernel waits for it at its end.
//
// Few rows, each with an adapter of its own as a rule, and 32-bit rows: CTA = (ROWS neighbouring rows, 16 rank rows, part of K), bound by
// reading A.  A warp walks its stretch of K 32 pieces of 16 bytes at a time and holds 16 sums of every row; rows of one adapter (a
// prompt's) share what is read of it, others take turns (float32, 800 rows of 4,864 columns, rank 128: 54 us, each row by itself 157).
// The parts of K meet through the cluster's shared memory, in order.  WIDE: rows are whole 16-byte pieces.
template <typename T, int ROWS, bool WIDE>
__global__ void __launch_bounds__(DOWN_WARPS * 32)
adapter_down_rows_kernel(const T* x, const T* __restrict__ down, const float* __restrict__ scales, const int* row_adapter, float* u,
                         int rows, int adapters, int rank, int K, int parts, int early) {
  constexpr int PIECE = WIDE ? Pack<T>::N : 1;
  __shared__ float sums[DOWN_WARPS][ROWS][DOWN_RANKS];
  __shared__ float total[ROWS][DOWN_RANKS];
  const int part = blockIdx.x % parts, row0 = blockIdx.x / parts * ROWS;
  const int r0 = blockIdx.y * DOWN_RANKS;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (!early) pdl_wait();
  pdl_trigger();      // after the wait: adapter_up_kernel relies on it
  int ids[ROWS];
  bool together = true;
#pragma unroll
  for (int m = 0; m < ROWS; ++m) {
    const int id = row0 + m < rows ? __ldcg(row_adapter + row0 + m) : -1;
    ids[m] = id >= 0 && id < adapters ? id : -1;      // the same in all CTAs of a cluster
    together = together && ids[m] == ids[0];
  }
  const int pieces = K / PIECE;
  const int stretch = (pieces + parts * DOWN_WARPS - 1) / (parts * DOWN_WARPS);
  const int begin = (part * DOWN_WARPS + warp) * stretch, end = min(pieces, begin + stretch);
  const int ranks = min(DOWN_RANKS, rank - r0);
  // the sums of rows m0 .. m0 + COUNT - 1 with one adapter
  auto take = [&](auto count, int m0, int adapter) {
    constexpr int COUNT = decltype(count)::value;
    float acc[COUNT][DOWN_RANKS];
#pragma unroll
    for (int m = 0; m < COUNT; ++m)
#pragma unroll
      for (int r = 0; r < DOWN_RANKS; ++r) acc[m][r] = 0.f;
    const T* xr = x + (size_t)(row0 + m0) * K;
    const T* ar = down + ((size_t)adapter * rank + r0) * K;
    for (int p = begin + lane; p < end; p += 32) {
      if (WIDE) {
        float xv[COUNT][PIECE];
#pragma unroll
        for (int m = 0; m < COUNT; ++m) unpack(__ldcg(reinterpret_cast<const uint4*>(xr + (size_t)m * K) + p), xv[m], T());
        constexpr int BATCH = ROWS == 1 ? DOWN_RANKS : 8;
#pragma unroll
        for (int rb = 0; rb < DOWN_RANKS; rb += BATCH) {
          uint4 raw[BATCH];
#pragma unroll
          for (int r = 0; r < BATCH; ++r)
            raw[r] = __ldg(reinterpret_cast<const uint4*>(ar + (size_t)min(rb + r, ranks - 1) * K) + p);      // past the last: unused sums
#pragma unroll
          for (int r = 0; r < BATCH; ++r) {
            float av[PIECE];
            unpack(raw[r], av, T());
#pragma unroll
            for (int m = 0; m < COUNT; ++m)
#pragma unroll
              for (int e = 0; e < PIECE; ++e) acc[m][rb + r] = fmaf(xv[m][e], av[e], acc[m][rb + r]);
          }
        }
      } else {
#pragma unroll
        for (int m = 0; m < COUNT; ++m) {
          const float xv = to_float(xr[(size_t)m * K + p]);
#pragma unroll
          for (int r = 0; r < DOWN_RANKS; ++r)
            if (r < ranks) acc[m][r] = fmaf(xv, to_float(ar[(size_t)r * K + p]), acc[m][r]);
        }
      }
    }
#pragma unroll
    for (int m = 0; m < COUNT; ++m)
#pragma unroll
      for (int r = 0; r < DOWN_RANKS; ++r) {
        const float sum = warp_sum(acc[m][r]);
        if (lane == 0) sums[warp][m0 + m][r] = sum;
      }
  };
  if (ROWS > 1 && together) {
    if (ids[0] >= 0) take(Count<ROWS>(), 0, ids[0]);
  } else {
    for (int m = 0; m < ROWS; ++m) {
      int id = ids[0];
#pragma unroll
      for (int q = 1; q < ROWS; ++q)
        if (q == m) id = ids[q];
      if (id >= 0) take(Count<1>(), m, id);
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < ROWS * DOWN_RANKS; i += DOWN_WARPS * 32) {
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < DOWN_WARPS; ++w) sum += sums[w][i / DOWN_RANKS][i % DOWN_RANKS];
    total[i / DOWN_RANKS][i % DOWN_RANKS] = sum;      // of rows without an adapter: never looked at
  }
  cluster_meet();
  if (part == 0) {
    for (int i = threadIdx.x; i < ROWS * DOWN_RANKS; i += DOWN_WARPS * 32) {
      const int m = i / DOWN_RANKS, r = i % DOWN_RANKS;
      const int id = row0 + m < rows ? __ldcg(row_adapter + row0 + m) : -1;
      if (id < 0 || id >= adapters || r0 + r >= rank) continue;
      float sum = 0.f;
#pragma unroll
      for (int other = 0; other < MOST_PARTS; ++other) sum += other < parts ? read_from_cta(&total[m][r], other) : 0.f;
      u[(size_t)(row0 + m) * rank + r0 + r] = scales[id] * sum;
    }
  }
  cluster_meet();      // no CTA leaves while another reads its sums
  if (early) pdl_wait();
}

// Many rows, prompts as a rule: a CTA takes 32 rows, a part of K and up to 8 NT rank rows of one adapter after another (those that
// its rows have; TILE_SPLIT CTAs take turns at them), on mma.sync.  Both operands are read straight from global memory, 16
// bytes of a row per lane: the four lanes that share a row hold 32 columns, and since both operands are dealt out alike, which
// of them an MMA calls column 0 does not matter.  The warps' and the parts' sums meet in shared memory, in order.
constexpr int TILE_WARPS = 8, TILE_SPLIT = 8;
template <int NT> constexpr int TILE_SHARED = (TILE_WARPS + 1) * TILE_DOWN * (8 * NT + 4) * 4;

template <int NT>
__global__ void __launch_bounds__(TILE_WARPS * 32)
adapter_down_tile_kernel(const bf16* x, const bf16* __restrict__ down, const float* __restrict__ scales, const int* row_adapter, float* u,
                         int rows, int adapters, int rank, int K, int parts, int early) {
  constexpr int TILE_RANKS = 8 * NT, TILE_PITCH = TILE_RANKS + 4;
  extern __shared__ float tile_shared[];
  float* sums = tile_shared;                                               // [warps][32][pitch]
  float* total = tile_shared + TILE_WARPS * TILE_DOWN * TILE_PITCH;        // [32][pitch]
  __shared__ int ids[TILE_DOWN];
  if (!early) pdl_wait();
  pdl_trigger();
  const int part = blockIdx.x % parts, row0 = blockIdx.x / parts * TILE_DOWN, r0 = blockIdx.y * TILE_RANKS;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  if (threadIdx.x < TILE_DOWN) {
    const int m = row0 + threadIdx.x;
    const int id = m < rows ? __ldcg(row_adapter + m) : -1;
    ids[threadIdx.x] = id >= 0 && id < adapters ? id : -1;
  }
  __syncthreads();
  // the tile's adapters: bit of every row that is its adapter's first
  const int my_id = ids[lane];
  bool leads = my_id >= 0;
  for (int j = 0; j < lane; ++j) leads = leads && ids[j] != my_id;
  unsigned leaders = __ballot_sync(0xffffffffu, leads);      // the same in every warp and every CTA of the cluster
  const int pieces = K / 8;                                  // of 16 bytes
  const int groups = (pieces + 3) / 4;                       // of 32 columns
  const int stretch = (groups + parts * TILE_WARPS - 1) / (parts * TILE_WARPS);
  const int begin = (part * TILE_WARPS + warp) * stretch, end = min(groups, begin + stretch);
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  const int ranks = min(TILE_RANKS, rank - r0);
  const uint4* xr = reinterpret_cast<const uint4*>(x + (size_t)row0 * K);
  for (int turn = 0; leaders != 0u; ++turn) {
    const int adapter = ids[__ffs(leaders) - 1];
    leaders &= leaders - 1u;
    if (turn % TILE_SPLIT != (int)blockIdx.z) continue;
    float acc[2][NT][4];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int n = 0; n < NT; ++n) acc[i][n][0] = acc[i][n][1] = acc[i][n][2] = acc[i][n][3] = 0.f;
    const uint4* ar = reinterpret_cast<const uint4*>(down + ((size_t)adapter * rank + r0) * K);
    for (int k = begin; k < end; ++k) {
      const int piece = k * 4 + t;
      const bool there = piece < pieces;
      uint4 a[4], b[NT];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // rows of another adapter count as zeros (whatever they hold stays out of the sums that are kept anyway)
        const int row = g + i * 8;
        a[i] = there && ids[row] == adapter ? __ldcg(xr + (size_t)row * pieces + piece) : zero;
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) b[n] = there && n * 8 + g < ranks ? __ldg(ar + (size_t)(n * 8 + g) * pieces + piece) : zero;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const uint32_t low[4] = {a[2 * i].x, a[2 * i + 1].x, a[2 * i].y, a[2 * i + 1].y};
          mma_bf16(acc[i][n], low, b[n].x, b[n].y);
          const uint32_t high[4] = {a[2 * i].z, a[2 * i + 1].z, a[2 * i].w, a[2 * i + 1].w};
          mma_bf16(acc[i][n], high, b[n].z, b[n].w);
        }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; e += 2)
          *reinterpret_cast<float2*>(sums + (warp * TILE_DOWN + i * 16 + g + e * 4) * TILE_PITCH + n * 8 + t * 2) =
              make_float2(acc[i][n][e], acc[i][n][e + 1]);
    __syncthreads();
    for (int i = threadIdx.x; i < TILE_DOWN * TILE_RANKS; i += TILE_WARPS * 32) {
      const int at = i / TILE_RANKS * TILE_PITCH + i % TILE_RANKS;
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < TILE_WARPS; ++w) sum += sums[w * TILE_DOWN * TILE_PITCH + at];
      total[at] = sum;
    }
    if (parts > 1) cluster_meet(); else __syncthreads();
    // each CTA of the cluster finishes its share of the rows
    for (int i = threadIdx.x; i < TILE_DOWN * TILE_RANKS; i += TILE_WARPS * 32) {
      const int row = i / TILE_RANKS, r = i - row * TILE_RANKS;
      if (row % parts != part || r >= ranks || ids[row] != adapter) continue;
      const float* at = total + row * TILE_PITCH + r;
      float sum = 0.f;
      if (parts == 1) sum = *at;
      else
#pragma unroll
        for (int other = 0; other < MOST_PARTS; ++other) sum += other < parts ? read_from_cta(at, other) : 0.f;
      u[(size_t)(row0 + row) * rank + r0 + r] = scales[adapter] * sum;
    }
    if (parts > 1) cluster_meet(); else __syncthreads();
  }
  if (early) pdl_wait();
}

// Up: a thread owns one output column and ROWS rows; B's row of the column is read once per run of rows with one adapter, 16 ranks at a
// time, the next ones under way (64 rows of as many adapters, rank 16, N = 3,584: 4 us; rank 64, N = 9,728: 26 us, 80 MB).  The first are
// asked for before the wait: which adapter a row has was complete before the down kernel, in front of this one on the stream, let the
// kernels behind it in.
template <typename T, typename Out, int ROWS, bool WIDE>
__global__ void __launch_bounds__(128)
adapter_up_kernel(const float* u, const T* __restrict__ up, const int* row_adapter, const float* base, Out* out, int rows, int adapters,
                  int rank, int N) {
  constexpr int CHUNK = 16, PIECES = WIDE ? CHUNK / Pack<T>::N : CHUNK;
  typedef typename Choice<WIDE, uint4, T>::type Raw;
  __shared__ float low[ROWS][128];
  const int row0 = blockIdx.y * ROWS;
  const int n = blockIdx.x * 128 + threadIdx.x;
  int ids[ROWS];
  bool same = true;
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const int id = row0 + r < rows ? __ldcg(row_adapter + row0 + r) : -1;
    ids[r] = id >= 0 && id < adapters ? id : -1;
    same = same && (ids[r] == ids[0] || row0 + r >= rows);
  }
  // (no test per piece, so that the loads go out together: past the last rank or column others are read and not used)
  auto load = [&](int id, int k0, Raw* raw) {
    if (id < 0 || k0 >= rank) return;
    const T* from = up + ((size_t)id * N + min(n, N - 1)) * rank;
    constexpr int W = CHUNK / PIECES;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) raw[i] = *reinterpret_cast<const Raw*>(from + min(k0 + i * W, rank - W));
  };
  auto values = [&](const Raw* raw, float* b) {
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      if constexpr (WIDE) unpack(raw[i], b + i * (CHUNK / PIECES), T());
      else b[i] = to_float(raw[i]);
    }
  };
  // of a thread's rows if they are few; of a run of many, what its first row needs
  constexpr int HELD = ROWS <= 2 ? ROWS : 1;
  Raw next[HELD][PIECES];
#pragma unroll
  for (int r = 0; r < HELD; ++r)
    if (r == 0 || ids[r] != ids[0]) load(ids[r], 0, next[r]);
  pdl_wait();
  pdl_trigger();
  for (int i = threadIdx.x; i < ROWS * rank; i += 128) {
    const int r = i / rank, m = row0 + r;
    const int id = m < rows ? __ldcg(row_adapter + m) : -1;
    low[r][i - r * rank] = id >= 0 && id < adapters ? __ldcg(u + (size_t)m * rank + (i - r * rank)) : 0.f;
  }
  float acc[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) acc[r] = n < N && row0 + r < rows ? __ldcg(base + (size_t)(row0 + r) * N + n) : 0.f;
  __syncthreads();
  if (n >= N) return;
  for (int k0 = 0; k0 < rank; k0 += CHUNK) {
    float b[HELD][CHUNK];
#pragma unroll
    for (int r = 0; r < HELD; ++r) {
      if (r > 0 && ids[r] == ids[0]) continue;      // the first row's values
      values(next[r], b[r]);
      load(ids[r], k0 + CHUNK, next[r]);
    }
    auto add = [&](int r, const float* w) {
#pragma unroll
      for (int i = 0; i < CHUNK; ++i)
        if (k0 + i < rank) acc[r] = fmaf(low[r][k0 + i], w[i], acc[r]);
    };
    if (ROWS <= 2) {
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        if (ids[r] < 0) continue;
        if (r > 0 && ids[r] == ids[0]) add(r, b[0]);
        else add(r, b[r < HELD ? r : 0]);
      }
    } else if (same) {
      if (ids[0] >= 0)
#pragma unroll
        for (int r = 0; r < ROWS; ++r) add(r, b[0]);
    } else {
      int held = ids[0];
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        if (ids[r] < 0) continue;
        if (ids[r] != held) {
          held = ids[r];
          Raw raw[PIECES];
          load(held, k0, raw);
          values(raw, b[0]);
        }
        add(r, b[0]);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < ROWS; ++r)
    if (row0 + r < rows) out[(size_t)(row0 + r) * N + n] = from_float<Out>(acc[r]);
}

template <int NT>
static int launch_down_tile(const void* x, const void* down, const float* scales, const int* row_adapter, float* u, int rows, int adapters,
                            int rank, int K, int early, cudaStream_t stream) {
  const int tiles = (rows + TILE_DOWN - 1) / TILE_DOWN, groups = (rank + 8 * NT - 1) / (8 * NT);
  int parts = 1;      // of K: one CTA per SM
  while (parts < MOST_PARTS && 2 * tiles * groups * parts <= sm_count() && K >= 4 * parts * TILE_WARPS * 32) parts *= 2;
  static OncePerDevice once;
  if (cudaError_t err = once([] { return cudaFuncSetAttribute(adapter_down_tile_kernel<NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, TILE_SHARED<NT>); }))
    return (int)err;
  launch_kernel_clustered(adapter_down_tile_kernel<NT>, dim3(tiles * parts, groups, TILE_SPLIT), dim3(TILE_WARPS * 32), TILE_SHARED<NT>, stream,
                          parts, (const bf16*)x, (const bf16*)down, scales, row_adapter, u, rows, adapters, rank, K, parts, early);
  return launch_status();
}

template <typename T, int ROWS>
static int launch_down_rows(const void* x, const void* down, const float* scales, const int* row_adapter, float* u, int rows, int adapters,
                            int rank, int K, int early, cudaStream_t stream) {
  // parts of K: as many CTAs as fill the device four times, at most eight (a cluster), none below 32 pieces per warp
  const bool wide = K % Pack<T>::N == 0;
  const int pieces = wide ? K / Pack<T>::N : K;
  const int groups = (rank + DOWN_RANKS - 1) / DOWN_RANKS, blocks = (rows + ROWS - 1) / ROWS;
  int parts = 1;
  while (parts < MOST_PARTS && (long long)blocks * groups * parts < 4ll * sm_count() && pieces >= 2 * parts * DOWN_WARPS * 32) parts *= 2;
  if ((long long)blocks * parts > 0x7fffffff || groups > 65535) return MLR_TOO_LARGE;
  const dim3 grid(blocks * parts, groups);
  auto kernel = wide ? adapter_down_rows_kernel<T, ROWS, true> : adapter_down_rows_kernel<T, ROWS, false>;
  launch_kernel_clustered(kernel, grid, dim3(DOWN_WARPS * 32), 0, stream, parts, (const T*)x, (const T*)down, scales, row_adapter, u,
                          rows, adapters, rank, K, parts, early);
  return launch_status();
}

template <typename T>
static int launch_down(const void* x, const void* down, const float* scales, const int* row_adapter, float* u, int rows, int adapters,
                       int rank, int K, int early, cudaStream_t stream) {
  return rows <= DOWN_ROWS ? launch_down_rows<T, 1>(x, down, scales, row_adapter, u, rows, adapters, rank, K, early, stream)
                           : launch_down_rows<T, 4>(x, down, scales, row_adapter, u, rows, adapters, rank, K, early, stream);
}

template <typename T, typename Out, int ROWS>
static int launch_up_rows(const float* u, const void* up, const int* row_adapter, const float* base, void* out, int rows, int adapters, int rank,
                          int N, cudaStream_t stream) {
  const bool wide = rank % Pack<T>::N == 0;
  if ((rows + ROWS - 1) / ROWS > 65535) return MLR_TOO_LARGE;
  const dim3 grid((N + 127) / 128, (rows + ROWS - 1) / ROWS);
  auto kernel = wide ? adapter_up_kernel<T, Out, ROWS, true> : adapter_up_kernel<T, Out, ROWS, false>;
  launch_kernel(kernel, grid, dim3(128), 0, stream, u, (const T*)up, row_adapter, base, (Out*)out, rows, adapters, rank, N);
  return launch_status();
}

template <typename T, typename Out>
static int launch_up(const float* u, const void* up, const int* row_adapter, const float* base, void* out, int rows, int adapters, int rank,
                     int N, cudaStream_t stream) {
  return rows <= 256 ? launch_up_rows<T, Out, 2>(u, up, row_adapter, base, out, rows, adapters, rank, N, stream)
                     : launch_up_rows<T, Out, 8>(u, up, row_adapter, base, out, rows, adapters, rank, N, stream);
}

}  // namespace mlr

using namespace mlr;

MLR_DEFINE_PDL_SWITCH

// The entry points of the shared product, of the libraries they live in.
typedef int (*SkinnyProduct)(const void*, const void*, const void*, void*, const void*, int, int, int, int, int, float, cudaStream_t);
typedef int (*TensorProduct)(const void*, const void*, const void*, void*, int, int, int, int, int, float, float, void*, long long, int*, int, int*,
                             cudaStream_t);
typedef int (*SplitProduct)(const float*, const float*, const float*, float*, int, int, int, int, void*, int*, cudaStream_t);

// x [rows, K], down [adapters, rank, K] of one dtype on 16-byte boundaries; u float32 [rows, rank].  Rows without an adapter are
// not written.  early: the kernel in front on the stream is the product of the same x, and lets the next one in after its own wait.
MLR_EXPORT int mlr_adapter_down(const void* x, const void* down, const float* scales, const int* row_adapter, float* u, int rows,
                                int adapters, int rank, int K, int dtype, int early, cudaStream_t stream) {
  if (rows < 0 || adapters <= 0 || rank <= 0 || rank > 128 || K <= 0) return MLR_BAD_SIZE;
  if (rows == 0) return MLR_OK;
  if (((uintptr_t)x & 15) != 0 || ((uintptr_t)down & 15) != 0) return MLR_BAD_ALIGNMENT;
  if (dtype == MLR_BF16 && rows > DOWN_ROWS && K % 8 == 0) {
    if (rank <= 16) return launch_down_tile<2>(x, down, scales, row_adapter, u, rows, adapters, rank, K, early, stream);
    if (rank <= 32) return launch_down_tile<4>(x, down, scales, row_adapter, u, rows, adapters, rank, K, early, stream);
    return launch_down_tile<8>(x, down, scales, row_adapter, u, rows, adapters, rank, K, early, stream);
  }
  if (dtype == MLR_BF16) return launch_down<bf16>(x, down, scales, row_adapter, u, rows, adapters, rank, K, early, stream);
  if (dtype == MLR_F32) return launch_down<float>(x, down, scales, row_adapter, u, rows, adapters, rank, K, early, stream);
  return MLR_BAD_DTYPE;
}

// up [adapters, N, rank], base float32 [rows, N], out [rows, N] in out_dtype (float32: may be base itself).
MLR_EXPORT int mlr_adapter_up(const float* u, const void* up, const int* row_adapter, const float* base, void* out, int rows, int adapters,
                              int rank, int N, int dtype, int out_dtype, cudaStream_t stream) {
  if (rows < 0 || adapters <= 0 || rank <= 0 || rank > 128 || N <= 0) return MLR_BAD_SIZE;
  if (rows == 0) return MLR_OK;
  if (((uintptr_t)up & 15) != 0) return MLR_BAD_ALIGNMENT;
  if (dtype == MLR_BF16 && out_dtype == MLR_BF16)
    return launch_up<bf16, bf16>(u, up, row_adapter, base, out, rows, adapters, rank, N, stream);
  if (dtype == MLR_BF16 && out_dtype == MLR_F32)
    return launch_up<bf16, float>(u, up, row_adapter, base, out, rows, adapters, rank, N, stream);
  if (dtype == MLR_F32 && out_dtype == MLR_F32)
    return launch_up<float, float>(u, up, row_adapter, base, out, rows, adapters, rank, N, stream);
  return MLR_BAD_DTYPE;
}

// The three in one call from the host, whose own steps per launch cost more than few rows' products: small sums, shared product into
// `base` (float32 [rows, N]), adapters' share into `out`.  route: 1 mlr_gemm_skinny, 2 mlr_gemm_tcgen05 (with its scratch and
// counters), 3 mlr_linear_split (with its scratch); `product` is that entry point.  The products that let the next kernel in
// after their own wait (2, and 1 of up to eight rows) come first, with the sums beside them.  A status other than MLR_OK of the
// product is handed on: nothing but it and the sums was launched then.
MLR_EXPORT int mlr_linear_adapters(const void* x, const void* weight, const void* bias, const void* down, const void* up, const float* scales,
                                   const int* row_adapter, float* low, float* base, void* out, int rows, int N, int K, int adapters, int rank,
                                   int dtype, int out_dtype, int route, void* product, void* scratch, long long scratch_bytes, int* counters,
                                   int counters_len, int* error_word, cudaStream_t stream) {
  if (product == nullptr || route < 1 || route > 3) return MLR_BAD_SIZE;
  const bool early = route == 2 || (route == 1 && rows <= 8);
  int status = MLR_OK;
  if (!early) status = mlr_adapter_down(x, down, scales, row_adapter, low, rows, adapters, rank, K, dtype, 0, stream);
  if (status != MLR_OK) return status;
  if (route == 1) status = ((SkinnyProduct)product)(x, weight, bias, base, nullptr, rows, N, K, 1, 0, -1.f, stream);
  else if (route == 2)
    status = ((TensorProduct)product)(x, weight, bias, base, rows, N, K, 1, 0, 0.f, 0.f, scratch, scratch_bytes, counters, counters_len, error_word, stream);
  else
    status = ((SplitProduct)product)((const float*)x, (const float*)weight, (const float*)bias, base, rows, N, K, 0, scratch, error_word, stream);
  if (status != MLR_OK) return status;
  if (early) status = mlr_adapter_down(x, down, scales, row_adapter, low, rows, adapters, rank, K, dtype, 1, stream);
  if (status != MLR_OK) return status;
  return mlr_adapter_up(low, up, row_adapter, base, out, rows, adapters, rank, N, dtype, out_dtype, stream);
}
