// The next token of each row from given random numbers, under a temperature and limits on what may be drawn: the k most
// probable tokens (top-k), those at least min_p times as probable as the best (min-p), the fewest that hold p of the
// probability that is left (top-p).
//
//   order      tokens by falling logit, equal ones by rising index; each limit keeps a beginning of that order
//   weights    w_i = exp((x_i - max) / T), w of the best is 1
//   kept       the first k; of them those with w >= min_p; of them the shortest beginning whose weights come to at least p of theirs
//   token      the first token, in the order of the vocabulary, whose sum of kept weights up to and with it exceeds u times the
//              sum of all
// T <= 0 (or NaN) takes the best token, the lowest index of a tie.  NaN logits count as -inf; a row of -inf takes token 0.
// Weights, sums and the places of the cuts are held in 64 bits: a sum of 150,000 weights in 32 bits moves the border between
// two tokens by 1e-7 of the whole, as much as a token of a flat row is wide a hundred times over.
//
// A cluster of CTAs takes a row; each CTA keeps its slice of the row in shared memory, so that the logits are read from memory
// once.  Logits are compared as whole numbers of the same order (`order_key`).
//   top-k, min-p   A lower bound of the k-th logit: each thread has met a largest one while it read, and k logits of a slice are as large
//                  as the k-th of these.  Tokens above it (above min-p's border) are few: they go to the first CTA, which sorts them, cuts,
//                  sorts what stays by index and draws.
//   else           The cuts are found together.  All logits are counted in 4,096 bins of T / 128; the CTAs add the bins up through distributed
//                  shared memory, and the bin that holds the cut is known for top-k, and for top-p but for a bin or two (a bin's weights
//                  are within a hundredth of one another).  The weights above it are summed, the tokens around it go to the first CTA, which
//                  sorts them and cuts.  If the cut is not there after all, or more tokens are than one CTA sorts (equal logits, say),
//                  an interval of keys that surely holds it is split eightfold until it is found.  Then the draw: sums by CTA,
//                  by warp, by part of a warp's stretch, and a walk.
// Sums are taken in a fixed order, of sorted numbers or of places (no floating-point atomics): a row's token depends on its row alone.
#include <cooperative_groups.h>

#include "uniform.cuh"

namespace mlr {

namespace cg = cooperative_groups;

constexpr int SL_THREADS = 512, SL_WARPS = SL_THREADS / 32;
constexpr int SL_BINS = 4096, SL_BINS_PER_THREAD = SL_BINS / SL_THREADS;
constexpr int SL_BOUND_BINS = 1024;
constexpr float SL_BINS_PER_T = 128.f;
constexpr int SL_MOST_K = 1200;          // a top-k whose candidates fit a list, it is likely
constexpr int SL_LIST = 2048;            // candidates that one CTA cuts and draws from
constexpr int SL_CUT = 1024;             // keys of an interval that one CTA sorts
constexpr int SL_PARTS = 8;
constexpr int SL_MOST_RANKS = 8;
static_assert(SL_BINS_PER_THREAD == 8, "a thread reads eight bins");

struct LimitSource {
  const float* uniforms;          // by row
  const float* temperatures;      // these four by row, or by slot with row_slot; each may be null
  const int* top_k;
  const float* top_p;
  const float* min_p;
  const int* row_slot;
  SlotState* state;               // with it temperature and random number are those of the slot's record
  int slots, advance;
};

// What a CTA shows the others of its cluster.
struct LimitShared {
  float max, bounds[2];           // the slice's largest logit; lower bounds of its k-th and of its k / ranks-th one
  int argmax;
  int count;                      // candidates in the list
  double sums[2][SL_PARTS];       // of the parts of an interval, two steps by turns
  int counts[2][SL_PARTS];
  unsigned cut_key;               // what the first CTA found
  int cut_index;
  double kept;
  // of this CTA alone
  double warp_double[SL_WARPS], part_double[SL_PARTS][SL_WARPS];
  float warp_float[SL_WARPS], warp_float2[SL_WARPS];
  int warp_int[SL_WARPS], part_int[SL_PARTS][SL_WARPS];
  unsigned found_key;
  float mark_mass[3];
  int found[2], mark_bin[3], mark_tokens[3];
};

// A token in the order of the limits, as a whole number: falling logit, rising index.
typedef unsigned long long Place;
__device__ __forceinline__ Place place_of(unsigned key, int index) { return ((Place)~key << 32) | (unsigned)index; }
__device__ __forceinline__ unsigned key_of(Place place) { return ~(unsigned)(place >> 32); }
__device__ __forceinline__ int index_of(Place place) { return (int)(unsigned)place; }

__device__ __forceinline__ unsigned order_key(float x) {      // larger for larger x
  const unsigned b = __float_as_uint(x);
  return b ^ ((b >> 31) != 0u ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float of_key(unsigned key) { return __uint_as_float((key >> 31) != 0u ? key ^ 0x80000000u : ~key); }
// NaN as -inf, -0 as 0 (they tie)
__device__ __forceinline__ float cleaned(float x) { return x == x ? x + 0.f : -INFINITY; }

// exp((x - top) / T) in 64 bits by Tang's method (table-driven exponentials, 1989): a = (n + 64 m) ln 2 / 64 + r with |r| < ln 2 / 128,
// exp a = 2^m 2^(n / 64) (1 + r + r^2 / 2 ..  r^5 / 120); the polynomial's remainder is below 2^-54.  `table` holds 2^(n / 64).
struct Weights {
  double inverse, top;
  float max;
  const double* table;
  __device__ __forceinline__ double operator()(float x) const {
    if (x == max) return 1.0;
    if (!(x > -INFINITY)) return 0.0;
    const double a = ((double)x - top) * inverse;
    if (!(a > -700.0)) return 0.0;             // (a NaN too: an infinite temperature beside an infinite logit)
    constexpr double RAISE = 6755399441055744.0;      // 1.5 * 2^52
    const double raised = fma(a, 92.33248261689366, RAISE), whole = raised - RAISE;      // 64 / ln 2
    const int n = __double2loint(raised);
    // ln 2 / 64 in two parts, the first of 21 bits: its product with a whole number is exact
    double r = fma(whole, -0x1.62e42p-7, a);
    r = fma(whole, -0x1.fdf473de6af28p-28, r);
    double q = fma(r, 1.0 / 120.0, 1.0 / 24.0);
    q = fma(r, q, 1.0 / 6.0);
    q = fma(r, q, 0.5);
    q = fma(r, q, 1.0);
    const double t = table[n & 63];
    const double value = fma(t, q * r, t);
    return __hiloint2double(__double2hiint(value) + ((n >> 6) << 20), __double2loint(value));
  }
};

__device__ __forceinline__ double warp_sum64(double v) {
#pragma unroll
  for (int offset = 16; offset > 0; offset >>= 1) v += __shfl_xor_sync(0xffffffffu, v, offset);
  return v;
}

// Sum over the block, in every thread; `room` SL_WARPS entries.
template <typename V>
__device__ __forceinline__ V sum_block(V v, V* room) {
#pragma unroll
  for (int offset = 16; offset > 0; offset >>= 1) v += __shfl_xor_sync(0xffffffffu, v, offset);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) room[threadIdx.x >> 5] = v;
  __syncthreads();
  V total = 0;
#pragma unroll
  for (int w = 0; w < SL_WARPS; ++w) total += room[w];
  return total;
}
// What the threads before hold together; `total` of all; `until`: what they hold with this one, the next thread's value to the last bit.
template <typename V>
__device__ __forceinline__ V before_block(V v, V* room, V* total, V* until = nullptr) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  V inclusive = v;
#pragma unroll
  for (int offset = 1; offset < 32; offset <<= 1) {
    const V up = __shfl_up_sync(0xffffffffu, inclusive, offset);
    if (lane >= offset) inclusive += up;
  }
  __syncthreads();
  if (lane == 31) room[warp] = inclusive;
  __syncthreads();
  V base = 0, all = 0;
#pragma unroll
  for (int w = 0; w < SL_WARPS; ++w) {
    if (w == warp) base = all;
    all += room[w];
  }
  *total = all;
  if (until != nullptr) *until = base + inclusive;
  const V previous = __shfl_up_sync(0xffffffffu, inclusive, 1);
  return base + (lane > 0 ? previous : (V)0);
}

// A set of kept tokens: keys above `key`, and of those equal to it the indexes up to `index`.
struct Cut {
  unsigned key;
  int index;
  __device__ __forceinline__ bool keeps(unsigned k, int i) const { return k > key || (k == key && i <= index); }
  __device__ __forceinline__ void tighten(const Cut& other) {
    if (other.key > key || (other.key == key && other.index < index)) *this = other;
  }
};

// How many of equal tokens of weight w stay in the shortest beginning that comes to `target`, `above` being before them.
__device__ __forceinline__ int ties_kept(double above, double w, double target, int ties) {
  if (!(w > 0.0)) return ties;
  const double wanted = ceil((target - above) / w);
  return wanted < 1.0 ? 1 : wanted < (double)ties ? (int)wanted : ties;
}

// Rising order by a bitonic network, EACH neighbouring numbers per thread in registers: pairs of a thread, of a warp by shuffles, of
// further ones through the array itself.  THREADS 32: one warp, which waits for no other.
template <int EACH, int THREADS>
__device__ __forceinline__ void sort_in_registers(Place* a, int n) {
  constexpr int SIZE = EACH * THREADS;
  const int thread = THREADS == 32 ? (int)(threadIdx.x & 31) : (int)threadIdx.x, first = thread * EACH;
  Place v[EACH];
#pragma unroll
  for (int i = 0; i < EACH; ++i) v[i] = first + i < n ? a[first + i] : ~(Place)0;
  auto exchange = [&](Place& low, Place& high, bool rising) {
    if ((low > high) == rising) { const Place x = low; low = high; high = x; }
  };
  for (int run = 2; run <= SIZE; run *= 2) {
    for (int apart = run / 2; apart >= EACH; apart /= 2) {
      if (apart < EACH * 32) {
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
          const Place other = __shfl_xor_sync(0xffffffffu, v[i], apart / EACH);
          const bool smaller = (((first + i) & run) == 0) == (((first + i) & apart) == 0);
          v[i] = (other < v[i]) == smaller ? other : v[i];
        }
      } else {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < EACH; ++i) a[first + i] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
          const Place other = a[(first + i) ^ apart];
          const bool smaller = (((first + i) & run) == 0) == (((first + i) & apart) == 0);
          v[i] = (other < v[i]) == smaller ? other : v[i];
        }
      }
    }
    if constexpr (EACH == 4) {
      if (run >= 4) { exchange(v[0], v[2], (first & run) == 0); exchange(v[1], v[3], (first & run) == 0); }
    }
    if constexpr (EACH >= 2) {
#pragma unroll
      for (int i = 0; i < EACH; i += 2) exchange(v[i], v[i + 1], ((first + i) & run) == 0);
    }
  }
  if (THREADS == 32) __syncwarp();
  else __syncthreads();
#pragma unroll
  for (int i = 0; i < EACH; ++i) a[first + i] = v[i];
}
// The array has room up to the next size that is sorted; behind n lie the largest numbers.
__device__ __noinline__ void sort_places(Place* a, int n) {
  __syncthreads();
  if (n <= 128) {
    if (threadIdx.x < 32) sort_in_registers<4, 32>(a, n);
  } else if (n <= SL_THREADS) {
    sort_in_registers<1, SL_THREADS>(a, n);
  } else if (n <= 2 * SL_THREADS) {
    sort_in_registers<2, SL_THREADS>(a, n);
  } else {
    sort_in_registers<4, SL_THREADS>(a, n);
  }
  __syncthreads();
}

template <bool RESIDENT>
__global__ void __launch_bounds__(SL_THREADS, 2)
sample_limited_kernel(const float* logits, const LimitSource source, int* __restrict__ tokens, int vocab, int slice, int room_bytes) {
  pdl_trigger();
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int row = blockIdx.x / ranks;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  extern __shared__ __align__(16) uint8_t limit_shared[];
  float* held = reinterpret_cast<float*>(limit_shared);                          // the slice
  Place* list = reinterpret_cast<Place*>(limit_shared + room_bytes);             // [SL_LIST] this CTA's candidates
  unsigned* bins = reinterpret_cast<unsigned*>(list + SL_LIST);                  // [SL_BINS]
  Place* all_listed = reinterpret_cast<Place*>(bins);                            // when the bins have been read, the candidates of all CTAs [SL_LIST]
  unsigned* segment = bins + SL_BINS;                                            // [SL_BINS / ranks]
  __shared__ LimitShared s;
  __shared__ double table[64];
  static_assert(SL_LIST * sizeof(Place) <= SL_BINS * sizeof(unsigned), "the candidates lie where the bins were");

  pdl_wait();
  // ---- the slice and its largest logit
  const int begin = min(vocab, rank * slice), size = min(vocab, begin + slice) - begin;
  const float* from = logits + (size_t)row * vocab + begin;
  auto at = [&](int i) -> float {
    if constexpr (RESIDENT) return held[i];
    else return cleaned(__ldcg(from + i));
  };
  float mine = -INFINITY;      // the largest that this thread met
  {
    // 16 bytes at a time where slice and row begin on such boundaries together (a resident slice begins on one)
    const bool wide = ((uintptr_t)from & 15) == 0;
    const int pieces = wide ? size / 4 : 0;
    constexpr int AHEAD = 5;
    for (int i = threadIdx.x; i < pieces; i += AHEAD * SL_THREADS) {
      float4 v[AHEAD];
#pragma unroll
      for (int j = 0; j < AHEAD; ++j)
        if (i + j * SL_THREADS < pieces) v[j] = __ldcg(reinterpret_cast<const float4*>(from) + i + j * SL_THREADS);
#pragma unroll
      for (int j = 0; j < AHEAD; ++j)
        if (i + j * SL_THREADS < pieces) {
          const float4 x = make_float4(cleaned(v[j].x), cleaned(v[j].y), cleaned(v[j].z), cleaned(v[j].w));
          if constexpr (RESIDENT) reinterpret_cast<float4*>(held)[i + j * SL_THREADS] = x;
          mine = fmaxf(mine, fmaxf(fmaxf(x.x, x.y), fmaxf(x.z, x.w)));
        }
    }
    for (int i = 4 * pieces + threadIdx.x; i < size; i += 4 * SL_THREADS) {
      float v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (i + j * SL_THREADS < size) v[j] = __ldcg(from + i + j * SL_THREADS);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (i + j * SL_THREADS < size) {
          const float x = cleaned(v[j]);
          if constexpr (RESIDENT) held[i + j * SL_THREADS] = x;
          mine = fmaxf(mine, x);
        }
    }
  }
  if (threadIdx.x < 64) table[threadIdx.x] = exp2((double)threadIdx.x * (1.0 / 64.0));
  // ---- the row's limits
  const int slot = source.row_slot != nullptr ? source.row_slot[row] : row;
  const bool known = slot >= 0 && slot < source.slots;
  SlotState* record = known && source.state != nullptr ? source.state + slot : nullptr;
  float temperature = 0.f, u = 0.f, p = 1.f, at_least = 0.f;
  int k = 0;
  if (known) {
    temperature = record != nullptr ? record->temperature : source.temperatures[slot];
    if (record != nullptr) u = uniform_from_seed(((unsigned long long)record->seed_high << 32) | record->seed_low, (long long)record->counter);
    else u = source.uniforms[row];
    if (source.top_k != nullptr) k = source.top_k[slot];
    if (source.top_p != nullptr) p = source.top_p[slot];
    if (source.min_p != nullptr) at_least = source.min_p[slot] > 0.f ? fminf(source.min_p[slot], 1.f) : 0.f;      // NaN: none
  }
  const bool greedy = !(temperature > 0.f);
  u = fmaxf(u, 0.f);
  if (p <= 0.f) { k = 1; p = 1.f; }
  const bool by_count = !greedy && k > 0 && k < vocab, by_weight = !greedy && p < 1.f;

  // ---- the slice's largest logit, and two of the threads' largest ones: the k-th, and the k / ranks-th.  All slices together hold k logits that
  // are as large as the least of their k / ranks-th ones, and each holds k as large as its k-th.
  {
    const float high = warp_max(mine), low = -warp_max(mine > -INFINITY ? -mine : -INFINITY);
    if (lane == 0) { s.warp_float[warp] = high; s.warp_float2[warp] = low; }
    const bool bounded = by_count && k <= SL_MOST_K && vocab > SL_LIST;
    if (bounded) for (int b = threadIdx.x; b < SL_BOUND_BINS; b += SL_THREADS) bins[b] = 0u;
    __syncthreads();
    float highest = s.warp_float[0], lowest = s.warp_float2[0];
#pragma unroll
    for (int w = 1; w < SL_WARPS; ++w) { highest = fmaxf(highest, s.warp_float[w]); lowest = fminf(lowest, s.warp_float2[w]); }
    if (threadIdx.x == 0) {
      s.max = highest;
      s.bounds[0] = s.bounds[1] = -INFINITY;
      s.argmax = 0x7fffffff;
    }
    if (bounded) {
      const float scale = highest > lowest && highest < INFINITY ? (float)(SL_BOUND_BINS - 1) / (highest - lowest) : 0.f;
      if (mine > -INFINITY) atomicAdd(&bins[scale > 0.f ? min(SL_BOUND_BINS - 1, (int)((highest - mine) * scale)) : 0], 1u);
      __syncthreads();
      constexpr int EACH = SL_BOUND_BINS / SL_THREADS;
      int counts[EACH], here = 0, total, until;
#pragma unroll
      for (int j = 0; j < EACH; ++j) { counts[j] = (int)bins[threadIdx.x * EACH + j]; here += counts[j]; }
      const int before = before_block(here, s.warp_int, &total, &until);
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const int place = m == 0 ? k : (k + ranks - 1) / ranks;
        if (before < place && until >= place) {      // one thread's (none's where fewer threads met a number)
          int run = before, bin = 0;
#pragma unroll
          for (int j = 0; j < EACH; ++j)
            if (run < place) { run += counts[j]; bin = (int)threadIdx.x * EACH + j; }
          // (a hundredth of a bin is more than the roundings)
          s.bounds[m] = scale > 0.f ? highest - ((float)bin + 1.01f) / scale : lowest;
        }
      }
    }
  }
  cluster.sync();
  float top = -INFINITY, bound = -INFINITY, least = INFINITY;
#pragma unroll
  for (int c = 0; c < SL_MOST_RANKS; ++c)
    if (c < ranks) {
      const LimitShared* theirs = cluster.map_shared_rank(&s, c);
      top = fmaxf(top, theirs->max);
      bound = fmaxf(bound, theirs->bounds[0]);
      least = fminf(least, theirs->bounds[1]);
    }
  bound = fmaxf(bound, least);
  auto finish = [&](int token) {      // by one thread of the cluster
    tokens[row] = token;
    if (record != nullptr) {
      record->last_token = token;
      record->counter += 1;
      if (source.advance) record->length += 1;
    }
  };
  if (greedy || top == -INFINITY) {
    if (top > -INFINITY && s.max == top)      // its first place
      for (int i = threadIdx.x; i < size; i += SL_THREADS)
        if (at(i) == top) atomicMin(&s.argmax, begin + i);
    cluster.sync();
    if (rank == 0 && threadIdx.x == 0) {
      int token = 0x7fffffff;
      for (int c = 0; c < ranks; ++c) token = min(token, cluster.map_shared_rank(&s, c)->argmax);
      finish(token < vocab ? token : 0);
    }
    cluster.sync();            // the first CTA has read the others'
    return;
  }
  Weights weight;
  weight.inverse = 1.0 / (double)temperature;
  weight.top = (double)top;
  weight.max = top;
  weight.table = table;
  const unsigned top_key = order_key(top), no_key = order_key(-INFINITY);

  // ---- min-p: the lowest key whose weight reaches it
  Cut kept{0u, 0x7fffffff};
  if (at_least > 0.f) {
    if (threadIdx.x == 0) {
      const double wanted = (double)at_least;
      float guess = (float)fma((double)temperature, log(wanted), weight.top);
      unsigned key = min(max(order_key(cleaned(guess)), no_key + 1), top_key);
      for (int i = 0; i < 64 && key < top_key && weight(of_key(key)) < wanted; ++i) ++key;
      for (int i = 0; i < 64 && key > no_key + 1 && weight(of_key(key - 1)) >= wanted; ++i) --key;
      s.found_key = key;
    }
    __syncthreads();
    kept.key = s.found_key;
  }

  // counts in bins: those of all CTAs, SL_BINS_PER_THREAD neighbours per thread
  int count[SL_BINS_PER_THREAD];
  const int per = SL_BINS / ranks, first_bin = (int)threadIdx.x * SL_BINS_PER_THREAD;
  auto clear_bins = [&]() {
    for (int b = threadIdx.x; b < SL_BINS; b += SL_THREADS) bins[b] = 0u;
    __syncthreads();
  };
  auto add_up_bins = [&]() {
    cluster.sync();
    for (int b = threadIdx.x; b < per; b += SL_THREADS) {
      unsigned sum = 0u;
#pragma unroll
      for (int c = 0; c < SL_MOST_RANKS; ++c)
        if (c < ranks) sum += cluster.map_shared_rank(bins, c)[rank * per + b];
      segment[b] = sum;
    }
    cluster.sync();
    const int owner = first_bin / per;
    const uint4* theirs = reinterpret_cast<const uint4*>(cluster.map_shared_rank(segment, owner) + (first_bin - owner * per));
    const uint4 low4 = theirs[0], high4 = theirs[1];
    count[0] = (int)low4.x; count[1] = (int)low4.y; count[2] = (int)low4.z; count[3] = (int)low4.w;
    count[4] = (int)high4.x; count[5] = (int)high4.y; count[6] = (int)high4.z; count[7] = (int)high4.w;
  };
  // tokens of [low, high] in `limit` to this CTA's list, in no order
  auto collect = [&](unsigned low, unsigned high, Cut limit) {
    if (threadIdx.x == 0) s.count = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < size; i += SL_THREADS) {
      const unsigned key = order_key(at(i));
      if (key >= low && key <= high && limit.keeps(key, begin + i)) {
        const int to = atomicAdd(&s.count, 1);
        if (to < SL_LIST) list[to] = place_of(key, begin + i);
      }
    }
  };
  auto listed = [&]() {      // by all CTAs, after a barrier of the cluster
    int n = 0;
#pragma unroll
    for (int c = 0; c < SL_MOST_RANKS; ++c)
      if (c < ranks) n += cluster.map_shared_rank(&s, c)->count;
    return n;
  };
  // the lists of all CTAs one behind the other; the first CTA, the others wait
  auto gather = [&](int room) -> int {
    int until[SL_MOST_RANKS], n = 0;
#pragma unroll
    for (int c = 0; c < SL_MOST_RANKS; ++c) until[c] = c < ranks ? cluster.map_shared_rank(&s, c)->count : 0;
#pragma unroll
    for (int c = 0; c < SL_MOST_RANKS; ++c) { n = min(n + until[c], room); until[c] = n; }
    for (int i = threadIdx.x; i < n; i += SL_THREADS) {
      int owner = 0, before = 0;
#pragma unroll
      for (int c = 0; c + 1 < SL_MOST_RANKS; ++c)
        if (i >= until[c]) { owner = c + 1; before = until[c]; }
      all_listed[i] = cluster.map_shared_rank(list, owner)[i - before];
    }
    __syncthreads();
    return n;
  };
  constexpr int SL_EACH = SL_LIST / SL_THREADS;
  // of n sorted tokens the first whose weights, `above` before them, come to `target`
  auto cut_sorted = [&](int n, double above, double target) -> int {
    const int each = (n + SL_THREADS - 1) / SL_THREADS, first = threadIdx.x * each;
    double w[SL_EACH], sum = 0.0, all;
#pragma unroll
    for (int i = 0; i < SL_EACH; ++i) {
      w[i] = i < each && first + i < n ? weight(of_key(key_of(all_listed[first + i]))) : 0.0;
      sum += w[i];
    }
    double run = above + before_block(sum, s.warp_double, &all);
    int passed = 0;          // tokens whose sums stay below the target
#pragma unroll
    for (int i = 0; i < SL_EACH; ++i) {
      run += w[i];
      passed += i < each && first + i < n && run < target;
    }
    return min(n, 1 + sum_block(passed, s.warp_int));
  };

  if ((by_count && k <= SL_MOST_K) || kept.key != 0u || vocab <= SL_LIST) {
    // ---- few candidates, it is likely
    const unsigned lowest = max(order_key(bound), kept.key);
    collect(lowest, 0xffffffffu, kept);
    cluster.sync();
    const int found = listed();
    if (found <= SL_LIST) {
      int n = 0;
      if (rank == 0) n = gather(SL_LIST);
      cluster.sync();
      if (rank != 0) return;
      sort_places(all_listed, n);
      int stay = by_count ? min(n, k) : n;
      if (by_weight) {
        double part = 0.0;
        for (int i = threadIdx.x; i < stay; i += SL_THREADS) part += weight(of_key(key_of(all_listed[i])));
        stay = cut_sorted(stay, 0.0, (double)p * sum_block(part, s.warp_double));
      }
      // what stays, in the order of the vocabulary: index, key
      __syncthreads();
      for (int i = threadIdx.x; i < stay; i += SL_THREADS) {
        const Place place = all_listed[i];
        all_listed[i] = ((Place)(unsigned)index_of(place) << 32) | key_of(place);
      }
      sort_places(all_listed, stay);
      const int each = (stay + SL_THREADS - 1) / SL_THREADS, first = threadIdx.x * each;
      double w[SL_EACH], sum = 0.0, all;
#pragma unroll
      for (int i = 0; i < SL_EACH; ++i) {
        w[i] = i < each && first + i < stay ? weight(of_key((unsigned)all_listed[first + i])) : 0.0;
        sum += w[i];
      }
      double run = before_block(sum, s.warp_double, &all);
      const double target = (double)u * all;
      if (threadIdx.x == 0) { s.found[0] = 0x7fffffff; s.found[1] = 0; }
      __syncthreads();
      int reached = 0x7fffffff, last_kept = -1;
#pragma unroll
      for (int i = 0; i < SL_EACH; ++i) {
        run += w[i];
        if (w[i] > 0.0) {
          last_kept = first + i;
          if (run > target && reached == 0x7fffffff) reached = first + i;
        }
      }
      if (reached != 0x7fffffff) atomicMin(&s.found[0], reached);
      if (last_kept >= 0) atomicMax(&s.found[1], last_kept);
      __syncthreads();
      if (threadIdx.x == 0) finish((int)(all_listed[s.found[0] < stay ? s.found[0] : s.found[1]] >> 32));
      return;
    }
    cluster.sync();            // the counts have been read
  }

  // ---- the cuts are found together
  // a warp's stretch of the slice
  const int stretch = ((size + SL_WARPS - 1) / SL_WARPS + 31) / 32 * 32;
  const int walk_begin = min(size, warp * stretch), walk_end = min(size, walk_begin + stretch);
  int turn = 0;
  // sums and counts of the parts of all CTAs
  auto exchange = [&](double (&sums)[SL_PARTS], int (&counts)[SL_PARTS]) {
#pragma unroll
    for (int j = 0; j < SL_PARTS; ++j) {
      sums[j] = warp_sum64(sums[j]);
      counts[j] = (int)__reduce_add_sync(0xffffffffu, (unsigned)counts[j]);
    }
    if (lane == 0)
#pragma unroll
      for (int j = 0; j < SL_PARTS; ++j) { s.part_double[j][warp] = sums[j]; s.part_int[j][warp] = counts[j]; }
    __syncthreads();
    if (threadIdx.x < SL_PARTS) {
      double sum = 0.0;
      int all = 0;
      for (int w = 0; w < SL_WARPS; ++w) { sum += s.part_double[threadIdx.x][w]; all += s.part_int[threadIdx.x][w]; }
      s.sums[turn][threadIdx.x] = sum;
      s.counts[turn][threadIdx.x] = all;
    }
    cluster.sync();
#pragma unroll
    for (int j = 0; j < SL_PARTS; ++j) {
      sums[j] = 0.0;
      counts[j] = 0;
      for (int c = 0; c < ranks; ++c) {
        const LimitShared* theirs = cluster.map_shared_rank(&s, c);
        sums[j] += theirs->sums[turn][j];
        counts[j] += theirs->counts[turn][j];
      }
    }
    turn ^= 1;
  };
  // The cut in [low, high], which holds `inside` kept keys, `above` before them; `ready`: they are in the lists already.
  auto cut_together = [&](bool weighed, unsigned low, unsigned high, double above, double target, int inside, bool ready) -> Cut {
    while (inside > SL_CUT && low < high) {
      ready = false;
      const unsigned step = (high - low) / SL_PARTS + 1;
      double sums[SL_PARTS];
      int counts[SL_PARTS];
#pragma unroll
      for (int j = 0; j < SL_PARTS; ++j) { sums[j] = 0.0; counts[j] = 0; }
      for (int i = threadIdx.x; i < size; i += SL_THREADS) {
        const float x = at(i);
        const unsigned key = order_key(x);
        if (key >= low && key <= high && kept.keeps(key, begin + i)) {
          const unsigned place = (high - key) / step;
          const double w = weighed ? weight(x) : 1.0;
#pragma unroll
          for (int j = 0; j < SL_PARTS; ++j)
            if (place == (unsigned)j) { sums[j] += w; counts[j] += 1; }
        }
      }
      exchange(sums, counts);
      int chosen = 0;
      bool open = true;
#pragma unroll
      for (int j = 0; j < SL_PARTS; ++j) {
        if (open) {
          const bool last = (unsigned long long)(j + 1) * step > (unsigned long long)(high - low);
          if (above + sums[j] >= target || last) { chosen = j; inside = counts[j]; open = false; }
          else above += sums[j];
        }
      }
      const unsigned long long end = (unsigned long long)high - (unsigned long long)chosen * step;
      low = end >= (unsigned long long)low + step - 1 ? (unsigned)(end - (step - 1)) : low;
      high = (unsigned)end;
    }
    if (inside <= SL_CUT) {
      if (!ready) {
        collect(low, high, kept);
        cluster.sync();
      }
      if (rank == 0) {
        const int n = gather(SL_CUT);
        sort_places(all_listed, n);
        const int stay = weighed ? cut_sorted(n, above, target) : min(n, max(1, (int)(target - above)));
        if (threadIdx.x == 0) {
          s.cut_key = n > 0 ? key_of(all_listed[stay - 1]) : low;
          s.cut_index = n > 0 ? index_of(all_listed[stay - 1]) : 0x7fffffff;
        }
      }
      cluster.sync();
      const LimitShared* first = cluster.map_shared_rank(&s, 0);
      const Cut cut{first->cut_key, first->cut_index};
      cluster.sync();
      return cut;
    }
    // more equal keys than a CTA sorts: the index of the last one that stays, by counting
    const int stay = weighed ? ties_kept(above, weight(of_key(low)), target, inside) : min(inside, max(1, (int)(target - above)));
    int here = 0;
    for (int base = walk_begin; base < walk_end; base += 32) {
      const int i = base + lane;
      here += __popc(__ballot_sync(0xffffffffu, i < walk_end && order_key(at(i)) == low && kept.keeps(low, begin + i)));
    }
    __syncthreads();
    if (lane == 0) s.warp_int[warp] = here;
    __syncthreads();
    if (threadIdx.x == 0) {
      int all = 0;
      for (int w = 0; w < SL_WARPS; ++w) all += s.warp_int[w];
      s.count = all;
      s.cut_index = -1;
    }
    cluster.sync();
    int place = 0;
    for (int c = 0; c < rank; ++c) place += cluster.map_shared_rank(&s, c)->count;
    for (int w = 0; w < warp; ++w) place += s.warp_int[w];
    if (place < stay && stay <= place + here)
      for (int base = walk_begin; base < walk_end; base += 32) {
        const int i = base + lane;
        const bool in = i < walk_end && order_key(at(i)) == low && kept.keeps(low, begin + i);
        const unsigned mask = __ballot_sync(0xffffffffu, in);
        if (in && place + __popc(mask & ((2u << lane) - 1u)) == stay) s.cut_index = begin + i;
        place += __popc(mask);
      }
    cluster.sync();
    Cut cut{low, 0x7fffffff};
    for (int c = 0; c < ranks; ++c) {
      const int found = cluster.map_shared_rank(&s, c)->cut_index;
      if (found >= 0) cut.index = found;
    }
    cluster.sync();
    return cut;
  };

  // ---- bins of T / 128 below the largest logit; the last holds all the rest
  const float bin_scale = SL_BINS_PER_T / temperature;
  if (by_count || by_weight) {
    clear_bins();
    for (int i = threadIdx.x; i < size; i += SL_THREADS)
      atomicAdd(&bins[(int)fminf((top - at(i)) * bin_scale, (float)(SL_BINS - 1))], 1u);      // (infinity times zero: bin 0)
    add_up_bins();
  }
  // keys that surely lie below a bin's beginning (all above: the first bin's)
  auto key_below = [&](float bin) { return bin >= (float)(SL_BINS - 1) ? 0u : order_key(cleaned(top - bin / bin_scale)); };
  double certain = 0.0;            // of this warp's stretch: weights that stay whatever the cut of the weights
  unsigned open_low = 0u, open_high = top_key;      // keys that it lies among
  bool summed = false;
  if (by_count) {
    int here = 0, total, until;
#pragma unroll
    for (int j = 0; j < SL_BINS_PER_THREAD; ++j) here += count[j];
    const int before = before_block(here, s.warp_int, &total, &until);
    if (before < k && until >= k) {
      int run = before, bin = first_bin;
#pragma unroll
      for (int j = 0; j < SL_BINS_PER_THREAD; ++j)
        if (run < k) { run += count[j]; bin = first_bin + j; }
      s.found[0] = bin;
    }
    __syncthreads();
    const int bin = s.found[0];
    const unsigned low = key_below((float)bin + 1.01f), high = bin == 0 ? top_key : key_below((float)bin - 0.01f);
    // every key counts, min-p or not: the smaller of the two beginnings stays
    const Cut before_k = kept;
    kept = Cut{0u, 0x7fffffff};
    double sums[SL_PARTS] = {};
    int counts[SL_PARTS] = {};
    collect(low, high, kept);
    for (int i = threadIdx.x; i < size; i += SL_THREADS) {
      const unsigned key = order_key(at(i));
      counts[0] += key > high;
      counts[1] += key >= low && key <= high;
    }
    exchange(sums, counts);
    const bool holds = counts[0] < k && counts[0] + counts[1] >= k;
    const Cut cut = holds ? cut_together(false, low, high, (double)counts[0], (double)k, counts[1], true)
                          : cut_together(false, 0u, top_key, 0.0, (double)k, vocab, false);
    kept = before_k;
    kept.tighten(cut);
  }
  if (by_weight) {
    // Weights taken in the middle of their bins: the bins where they come to p of theirs, and to a little less and more.  What the
    // estimate is off (single large tokens) shows in the exact sums above an interval; with that known the next one is found.
    float mass[SL_BINS_PER_THREAD], here = 0.f, all, until;
    int tokens_here = 0, tokens_all, tokens_until;
    const int last_bin = kept.key > 0u ? (int)fminf((top - of_key(max(kept.key, no_key))) * bin_scale, (float)(SL_BINS - 1)) : SL_BINS - 1;
#pragma unroll
    for (int j = 0; j < SL_BINS_PER_THREAD; ++j) {
      mass[j] = count[j] > 0 && first_bin + j <= last_bin ? (float)count[j] * expf(-((float)(first_bin + j) + 0.5f) / SL_BINS_PER_T) : 0.f;
      here += mass[j];
      tokens_here += count[j];
    }
    const float before = before_block(here, s.warp_float, &all, &until);
    const int tokens_before = before_block(tokens_here, s.warp_int, &tokens_all, &tokens_until);
    float wanted = p * all;
    Cut cut{0u, 0x7fffffff};
    bool found = false;
    double whole = 0.0;
    for (int attempt = 0; attempt < 3 && !found; ++attempt) {
      __syncthreads();
      if (threadIdx.x < 3) { s.mark_bin[threadIdx.x] = last_bin; s.mark_mass[threadIdx.x] = all; s.mark_tokens[threadIdx.x] = tokens_all; }
      __syncthreads();
#pragma unroll
      for (int m = 0; m < 3; ++m) {
        const float mark = wanted + (float)(m - 1) * 0.003f * all;
        if ((before < mark || threadIdx.x == 0) && until >= mark) {
          float run = before, at_bin = before;
          int bin = first_bin, run_tokens = tokens_before, at_tokens = tokens_before;
#pragma unroll
          for (int j = 0; j < SL_BINS_PER_THREAD; ++j)
            if (run < mark || j == 0) {
              at_bin = run;
              at_tokens = run_tokens;
              run += mass[j];
              run_tokens += count[j];
              bin = first_bin + j;
            }
          s.mark_bin[m] = bin;
          s.mark_mass[m] = at_bin;           // what lies before the bin
          s.mark_tokens[m] = m == 2 ? run_tokens : at_tokens;
        }
      }
      __syncthreads();
      float estimate;                        // of what lies above the interval
      if (s.mark_tokens[2] - s.mark_tokens[0] <= SL_CUT) {
        open_low = key_below((float)s.mark_bin[2] + 1.01f);
        open_high = s.mark_bin[0] == 0 ? top_key : key_below((float)s.mark_bin[0] - 0.01f);
        estimate = s.mark_mass[0];
      } else {
        open_low = key_below((float)s.mark_bin[1] + 1.25f);
        open_high = s.mark_bin[1] == 0 ? top_key : key_below((float)s.mark_bin[1] - 0.25f);
        estimate = s.mark_mass[1];
      }
      collect(open_low, open_high, kept);
      double sums[SL_PARTS] = {};
      int counts[SL_PARTS] = {};
      certain = 0.0;
      for (int i = walk_begin + lane; i < walk_end; i += 32) {
        const float x = at(i);
        const unsigned key = order_key(x);
        if (kept.keeps(key, begin + i)) {
          const double w = weight(x);
          if (key > open_high) certain += w;
          else if (key >= open_low) { sums[1] += w; counts[1] += 1; }
          else sums[2] += w;
        }
      }
      sums[0] = certain;
      certain = warp_sum64(certain);
      exchange(sums, counts);
      whole = sums[0] + sums[1] + sums[2];
      const double target = (double)p * whole;
      found = sums[0] < target && (sums[0] + sums[1] >= target || open_low == 0u);
      if (found) cut = cut_together(true, open_low, open_high, sums[0], target, counts[1], true);
      wanted = (float)(target - sums[0]) + estimate;
    }
    summed = found;
    if (!found) cut = cut_together(true, 0u, top_key, 0.0, (double)p * whole, vocab, false);
    kept.tighten(cut);
  }

  // ---- the draw
  double sum = 0.0;
  for (int i = walk_begin + lane; i < walk_end; i += 32) {
    const float x = at(i);
    const unsigned key = order_key(x);
    if (kept.keeps(key, begin + i) && (!summed || key <= open_high)) sum += weight(x);
  }
  sum = warp_sum64(sum) + (summed ? certain : 0.0);
  __syncthreads();
  if (lane == 0) s.warp_double[warp] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    double all = 0.0;
    for (int w = 0; w < SL_WARPS; ++w) all += s.warp_double[w];
    s.kept = all;
  }
  cluster.sync();
  double all = 0.0, run = 0.0;
  int last_rank = 0;
  for (int c = 0; c < ranks; ++c) {
    const double theirs = cluster.map_shared_rank(&s, c)->kept;
    if (c == rank) run = all;
    all += theirs;
    if (theirs > 0.0) last_rank = c;
  }
  const double target = (double)u * all;
  // the CTA, then the warp's stretch, then its part, whose sums the draw falls into; what rounding leaves behind the last belongs to it
  if (target >= run && s.kept > 0.0 && (target < run + s.kept || rank == last_rank)) {
    auto chosen_of = [&](double& so_far) {
      int last = 0, chosen = -1;
      for (int w = 0; w < SL_WARPS; ++w)
        if (s.warp_double[w] > 0.0) last = w;
      for (int w = 0; w < SL_WARPS && chosen < 0; ++w) {
        if (s.warp_double[w] > 0.0 && (target < so_far + s.warp_double[w] || w == last)) chosen = w;
        else so_far += s.warp_double[w];
      }
      return max(chosen, 0);
    };
    const int stretch_begin = min(size, chosen_of(run) * stretch), stretch_end = min(size, stretch_begin + stretch);
    const int part = ((stretch + SL_WARPS - 1) / SL_WARPS + 31) / 32 * 32;
    const int part_begin = min(stretch_end, stretch_begin + warp * part), part_end = min(stretch_end, part_begin + part);
    double in_part = 0.0;
    for (int i = part_begin + lane; i < part_end; i += 32) {
      const float x = at(i);
      if (kept.keeps(order_key(x), begin + i)) in_part += weight(x);
    }
    in_part = warp_sum64(in_part);
    __syncthreads();
    if (lane == 0) s.warp_double[warp] = in_part;
    __syncthreads();
    if (warp == chosen_of(run)) {
      int found = -1, last_kept = -1;
      for (int base = part_begin; base < part_end && found < 0; base += 32) {
        const int i = base + lane < part_end ? base + lane : -1;
        const float x = i >= 0 ? at(i) : -INFINITY;
        const double w = i >= 0 && kept.keeps(order_key(x), begin + i) ? weight(x) : 0.0;
        double inclusive = w;
#pragma unroll
        for (int offset = 1; offset < 32; offset <<= 1) {
          const double up = __shfl_up_sync(0xffffffffu, inclusive, offset);
          if (lane >= offset) inclusive += up;
        }
        const unsigned some = __ballot_sync(0xffffffffu, w > 0.0);
        const unsigned hit = __ballot_sync(0xffffffffu, w > 0.0 && run + inclusive > target);
        if (some != 0u) last_kept = base + 31 - __clz(some);
        if (hit != 0u) found = base + __ffs(hit) - 1;
        run += __shfl_sync(0xffffffffu, inclusive, 31);
      }
      if (lane == 0) finish(begin + (found >= 0 ? found : max(0, last_kept)));
    }
  }
  cluster.sync();      // the others may still read this CTA's sum
}

}  // namespace mlr

using namespace mlr;

MLR_DEFINE_PDL_SWITCH

// logits float32 [rows, vocab]; uniforms float32 [rows]; temperatures, top_p, min_p float32 and top_k int32, one entry per row or, with
// row_slot int32 [rows], per slot (a row of no slot takes its best token); the last three may be null.  With `state` (SlotState records,
// row_slot given) temperature and random number come from the record, which receives the token.
MLR_EXPORT int mlr_sample_limited(const float* logits, const float* uniforms, const float* temperatures, const int* top_k, const float* top_p,
                                  const float* min_p, const int* row_slot, void* state, int slots, int advance, int* tokens, int rows, int vocab,
                                  cudaStream_t stream) {
  if (rows == 0) return MLR_OK;
  if (rows < 0 || vocab <= 0 || slots < 0) return MLR_BAD_SIZE;
  if (state == nullptr ? uniforms == nullptr || temperatures == nullptr : row_slot == nullptr) return MLR_BAD_SIZE;
  if ((long long)rows * SL_MOST_RANKS > 0x7fffffffLL) return MLR_TOO_LARGE;
  const LimitSource source{uniforms, temperatures, top_k, top_p, min_p, row_slot, (SlotState*)state, slots, advance};
  // CTAs per row: enough that a slice fits twice on an SM, more while the row's CTAs find an SM each
  constexpr int RESIDENT_MOST = 24 * 1024, LEAST = 2048;
  int ranks = 1;
  while (ranks < SL_MOST_RANKS && (vocab > ranks * RESIDENT_MOST || (vocab > ranks * LEAST && rows * ranks * 2 <= sm_count()))) ranks *= 2;
  const int slice = ((vocab + ranks - 1) / ranks + 3) / 4 * 4;
  const bool resident = slice <= RESIDENT_MOST;
  const int most = RESIDENT_MOST * 4;
  const int room = resident ? (slice * 4 + 15) / 16 * 16 : 0;
  const size_t rest = SL_LIST * sizeof(Place) + SL_BINS * sizeof(unsigned) + SL_BINS / ranks * sizeof(unsigned);
  static OncePerDevice once;
  const cudaError_t err = once([&] {
    const int bytes = most + (int)(SL_LIST * sizeof(Place) + 2 * SL_BINS * sizeof(unsigned));
    cudaError_t e = cudaFuncSetAttribute(sample_limited_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    return e == cudaSuccess ? cudaFuncSetAttribute(sample_limited_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) : e;
  });
  if (err != cudaSuccess) return (int)err;
  auto kernel = resident ? sample_limited_kernel<true> : sample_limited_kernel<false>;
  launch_kernel_clustered(kernel, dim3(rows * ranks), dim3(SL_THREADS), room + rest, stream, ranks, logits, source, tokens, vocab, slice, room);
  return launch_status();
}
