// A small projection of one to four rows with low-rank adapters in one launch: y[m] = x[m] W^T + b + scale (x[m] A^T) B^T.
//
// Such a step is all latency: three kernels (the small sums, the shared product, the adapters' share) cost their launches and
// waits, and from the host, whose own work per launch is more than the GPU's, 31 us.  Here every CTA takes the sums u[m][r] =
// scale sum_k x A by itself, a few per warp, from L2 (some KB, hence the bound on rows * rank * K), while its own weights,
// asked for before the kernel before has ended, arrive; then its columns, the adapters' share added to the lanes' sums before
// they meet.  A lane holds 16 bytes of K at a time, everything is summed in float32.  One row of 896 x 1,152 with rank 8: 5.3 us
// in a row of captured calls (three kernels 6.3), 8.2 in a graph of its own, 12 from the host.
#include "common.cuh"

namespace mlr {

constexpr int SMALL_WARPS = 8, SMALL_SUMS = 512;      // sums u a CTA holds

template <typename T> struct Piece { static constexpr int N = 16 / sizeof(T); };
__device__ __forceinline__ void spread(const uint4& raw, float* v, bf16) {
  const __nv_bfloat162* pair = reinterpret_cast<const __nv_bfloat162*>(&raw);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __bfloat1622float2(pair[i]);
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void spread(const uint4& raw, float* v, float) {
  v[0] = __uint_as_float(raw.x); v[1] = __uint_as_float(raw.y); v[2] = __uint_as_float(raw.z); v[3] = __uint_as_float(raw.w);
}

// ROWS: rows of x at most.  A warp owns one output column.
template <typename T, typename Out, int ROWS>
__global__ void __launch_bounds__(SMALL_WARPS * 32)
adapter_small_kernel(const T* x, const T* __restrict__ weight, const T* __restrict__ bias, const T* __restrict__ down,
                     const T* __restrict__ up, const float* __restrict__ scales, const int* row_adapter, Out* out, int rows, int N, int K,
                     int adapters, int rank) {
  constexpr int WIDTH = Piece<T>::N, AHEAD = 4;
  __shared__ float u[SMALL_SUMS];                // [rows][rank]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n = blockIdx.x * SMALL_WARPS + warp;
  const bool column = n < N;
  const int pieces = K / WIDTH;
  // the weights of the first AHEAD rounds
  uint4 w[AHEAD];
  auto load_w = [&](int p) {
    return p < pieces && column ? __ldg(reinterpret_cast<const uint4*>(weight + (size_t)n * K) + p) : make_uint4(0u, 0u, 0u, 0u);
  };
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) w[i] = load_w(lane + 32 * i);
  const float b = bias != nullptr && column ? to_float(bias[n]) : 0.f;
  pdl_wait();
  pdl_trigger();
  const uint4* x4 = reinterpret_cast<const uint4*>(x);
  int ids[ROWS];
  float first_up[ROWS];                          // B of this column and the first 32 ranks, a rank per lane
#pragma unroll
  for (int m = 0; m < ROWS; ++m) {
    const int id = m < rows ? __ldcg(row_adapter + m) : -1;
    ids[m] = id >= 0 && id < adapters ? id : -1;
    first_up[m] = ids[m] >= 0 && column && lane < rank ? to_float(up[((size_t)ids[m] * N + n) * rank + lane]) : 0.f;
  }
  // ---- u, a pair (row, rank) per warp and turn
  for (int pair = warp; pair < rows * rank; pair += SMALL_WARPS) {
    const int m = pair / rank, r = pair - m * rank;
    const int id = __ldcg(row_adapter + m);
    if (id < 0 || id >= adapters) continue;
    const uint4* a4 = reinterpret_cast<const uint4*>(down + ((size_t)id * rank + r) * K);
    float sum = 0.f;
#pragma unroll 4
    for (int p = lane; p < pieces; p += 32) {
      float xv[WIDTH], av[WIDTH];
      spread(__ldcg(x4 + (size_t)m * pieces + p), xv, T());
      spread(__ldg(a4 + p), av, T());
#pragma unroll
      for (int e = 0; e < WIDTH; ++e) sum = fmaf(xv[e], av[e], sum);
    }
    sum = warp_sum(sum) * scales[id];
    if (lane == 0) u[pair] = sum;
  }
  // ---- the shared product of this warp's column
  float acc[ROWS];
#pragma unroll
  for (int m = 0; m < ROWS; ++m) acc[m] = 0.f;
  for (int p0 = lane; p0 < pieces + lane; p0 += 32 * AHEAD) {      // the same rounds in every lane
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int p = p0 + 32 * i;
      float wv[WIDTH];
      spread(w[i], wv, T());
      w[i] = load_w(p + 32 * AHEAD);
      if (p < pieces) {
#pragma unroll
        for (int m = 0; m < ROWS; ++m) {
          if (m < rows) {
            float xv[WIDTH];
            spread(__ldcg(x4 + (size_t)m * pieces + p), xv, T());
#pragma unroll
            for (int e = 0; e < WIDTH; ++e) acc[m] = fmaf(xv[e], wv[e], acc[m]);
          }
        }
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int m = 0; m < ROWS; ++m) {
    if (ids[m] < 0 || !column) continue;
    if (lane < rank) acc[m] = fmaf(u[m * rank + lane], first_up[m], acc[m]);
    for (int r = 32 + lane; r < rank; r += 32) acc[m] = fmaf(u[m * rank + r], to_float(up[((size_t)ids[m] * N + n) * rank + r]), acc[m]);
  }
#pragma unroll
  for (int m = 0; m < ROWS; ++m) {
    if (m < rows) {
      const float sum = warp_sum(acc[m]);
      if (lane == 0 && column) out[(size_t)m * N + n] = from_float<Out>(sum + b);
    }
  }
}

template <typename T, typename Out>
static int run(const void* x, const void* weight, const void* bias, const void* down, const void* up, const float* scales,
               const int* row_adapter, void* out, int rows, int N, int K, int adapters, int rank, cudaStream_t stream) {
  launch_kernel(rows == 1 ? adapter_small_kernel<T, Out, 1> : adapter_small_kernel<T, Out, 4>, dim3((N + SMALL_WARPS - 1) / SMALL_WARPS),
                dim3(SMALL_WARPS * 32), 0, stream, (const T*)x, (const T*)weight, (const T*)bias, (const T*)down, (const T*)up, scales,
                row_adapter, (Out*)out, rows, N, K, adapters, rank);
  return launch_status();
}

}  // namespace mlr

using namespace mlr;

MLR_DEFINE_PDL_SWITCH

// x [rows, K], weight [N, K], bias [N] or null, down [adapters, rank, K], up [adapters, N, rank] of one dtype, x, weight and down on
// 16-byte boundaries with rows of whole 16-byte pieces; rows <= 4; out [rows, N] in out_dtype (that of x, or float32).
MLR_EXPORT int mlr_adapter_small(const void* x, const void* weight, const void* bias, const void* down, const void* up, const float* scales,
                                 const int* row_adapter, void* out, int rows, int N, int K, int adapters, int rank, int dtype, int out_dtype,
                                 cudaStream_t stream) {
  if (rows < 0 || N <= 0 || K <= 0 || adapters <= 0 || rank <= 0 || rank > 128) return MLR_BAD_SIZE;
  if (rows == 0) return MLR_OK;
  if (rows > 4 || rows * rank > SMALL_SUMS) return MLR_TOO_LARGE;
  if ((((uintptr_t)x | (uintptr_t)weight | (uintptr_t)down) & 15) != 0 || K % (dtype == MLR_BF16 ? 8 : 4) != 0) return MLR_BAD_ALIGNMENT;
  if (dtype == MLR_BF16 && out_dtype == MLR_BF16)
    return run<bf16, bf16>(x, weight, bias, down, up, scales, row_adapter, out, rows, N, K, adapters, rank, stream);
  if (dtype == MLR_BF16 && out_dtype == MLR_F32)
    return run<bf16, float>(x, weight, bias, down, up, scales, row_adapter, out, rows, N, K, adapters, rank, stream);
  if (dtype == MLR_F32 && out_dtype == MLR_F32)
    return run<float, float>(x, weight, bias, down, up, scales, row_adapter, out, rows, N, K, adapters, rank, stream);
  return MLR_BAD_DTYPE;
}
