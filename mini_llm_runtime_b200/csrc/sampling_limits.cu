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
// once.  Logits are compared as whole numbers of the same order (`order_key`).  While a slice arrives its keys are counted in
// 4,096 bins (sign, exponent, three bits of mantissa), the CTAs add the bins up through distributed shared memory, and every
// CTA finds from them the lowest bin that a cut can lie in: exactly for top-k, by bounds of the bins' weights for top-p.
//   few candidates (<= SL_LIST above that bin)   they go to the first CTA, which sorts them, cuts, sorts what stays by index and draws
//   many                                         the cuts are found together: an eightfold split of the interval of keys that holds
//                                                the cut, weights summed for each part, until few enough keys are in it for one CTA to
//                                                sort; then every CTA sums its kept weights and the one that the draw falls into
//                                                walks there
// Sums are taken in a fixed order, of sorted numbers or of places (no floating-point atomics): a row's token depends on its row alone.
#include <cooperative_groups.h>

#include "uniform.cuh"

namespace mlr {

namespace cg = cooperative_groups;

constexpr int SL_THREADS = 512, SL_WARPS = SL_THREADS / 32;
constexpr int SL_BINS = 4096, SL_BIN_SHIFT = 20, SL_BINS_PER_THREAD = SL_BINS / SL_THREADS;
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
  float max;
  int argmax;
  int count;                      // candidates in the list
  double tail;                    // weights below the candidates
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
  int found[4];
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

struct Weights {
  double inverse, top;
  float max;
  __device__ __forceinline__ double operator()(float x) const {
    if (x == max) return 1.0;
    if (x == -INFINITY) return 0.0;
    const double w = exp(((double)x - top) * inverse);
    return w > 0.0 ? w : 0.0;
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

// Rising order, by one CTA; the array has room up to the next power of two, which is filled with the largest number.  A bitonic
// network: a warp's 32 pairs lie in 64 neighbouring numbers as long as the pairs are at most 32 apart, and wait for no other warp.
__device__ void sort_places(Place* a, int n) {
  int size = 64;
  while (size < n) size *= 2;
  for (int i = n + threadIdx.x; i < size; i += SL_THREADS) a[i] = ~(Place)0;
  __syncthreads();
  for (int run = 2; run <= size; run *= 2) {
    for (int apart = run / 2; apart > 0; apart /= 2) {
      for (int pair = threadIdx.x; pair < size / 2; pair += SL_THREADS) {
        const int low = 2 * pair - (pair & (apart - 1)), high = low + apart;
        const Place x = a[low], y = a[high];
        if ((x > y) == ((low & run) == 0)) { a[low] = y; a[high] = x; }
      }
      if (apart > 32) __syncthreads();
      else __syncwarp();
    }
    __syncthreads();
  }
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
  Place* all_listed = reinterpret_cast<Place*>(bins);                            // later the candidates of all CTAs [SL_LIST]
  unsigned* segment = bins + SL_BINS;                                            // [SL_BINS / ranks]
  __shared__ LimitShared s;
  static_assert(SL_LIST * sizeof(Place) <= SL_BINS * sizeof(unsigned), "the candidates lie where the bins were");

  pdl_wait();
  // ---- the row's limits
  const int slot = source.row_slot != nullptr ? source.row_slot[row] : row;
  const bool known = slot >= 0 && slot < source.slots;
  SlotState* record = known && source.state != nullptr ? source.state + slot : nullptr;
  float temperature = 0.f, u = 0.f, p = 1.f, least = 0.f;
  int k = 0;
  if (known) {
    temperature = record != nullptr ? record->temperature : source.temperatures[slot];
    if (record != nullptr) u = uniform_from_seed(((unsigned long long)record->seed_high << 32) | record->seed_low, (long long)record->counter);
    else u = source.uniforms[row];
    if (source.top_k != nullptr) k = source.top_k[slot];
    if (source.top_p != nullptr) p = source.top_p[slot];
    if (source.min_p != nullptr) least = source.min_p[slot] > 0.f ? fminf(source.min_p[slot], 1.f) : 0.f;      // NaN: none
  }
  const bool greedy = !(temperature > 0.f);
  u = fmaxf(u, 0.f);
  if (p <= 0.f) { k = 1; p = 1.f; }
  const bool by_count = !greedy && k > 0 && k < vocab, by_weight = !greedy && p < 1.f;
  const bool binned = by_count || by_weight;

  // ---- the slice, its best token, its bins
  const int begin = min(vocab, rank * slice), size = min(vocab, begin + slice) - begin;
  const float* from = logits + (size_t)row * vocab + begin;
  auto at = [&](int i) -> float {
    if constexpr (RESIDENT) return held[i];
    else return cleaned(__ldcg(from + i));
  };
  if (binned) {
    for (int b = threadIdx.x; b < SL_BINS; b += SL_THREADS) bins[b] = 0u;
    __syncthreads();
  }
  float best = -INFINITY;
  int best_index = vocab;
  auto take = [&](int i, float x) {
    if constexpr (RESIDENT) held[i] = x;
    if (x > best) { best = x; best_index = begin + i; }
    if (binned) atomicAdd(&bins[order_key(x) >> SL_BIN_SHIFT], 1u);
  };
  const int lead = min(size, (int)((16 - ((uintptr_t)from & 15)) & 15) / 4), pieces = (size - lead) / 4;
  for (int i = threadIdx.x; i < lead; i += SL_THREADS) take(i, cleaned(__ldcg(from + i)));
  const float4* wide = reinterpret_cast<const float4*>(from + lead);
  for (int i = threadIdx.x; i < pieces; i += 4 * SL_THREADS) {
    float4 v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i + j * SL_THREADS < pieces) v[j] = __ldcg(wide + i + j * SL_THREADS);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i + j * SL_THREADS < pieces) {
        const int first = lead + 4 * (i + j * SL_THREADS);
        take(first, cleaned(v[j].x));
        take(first + 1, cleaned(v[j].y));
        take(first + 2, cleaned(v[j].z));
        take(first + 3, cleaned(v[j].w));
      }
  }
  for (int i = lead + 4 * pieces + threadIdx.x; i < size; i += SL_THREADS) take(i, cleaned(__ldcg(from + i)));
#pragma unroll
  for (int offset = 16; offset > 0; offset >>= 1) {
    const float other = __shfl_xor_sync(0xffffffffu, best, offset);
    const int other_index = __shfl_xor_sync(0xffffffffu, best_index, offset);
    if (other > best || (other == best && other_index < best_index)) { best = other; best_index = other_index; }
  }
  if (lane == 0) { s.warp_float[warp] = best; s.warp_int[warp] = best_index; }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < SL_WARPS; ++w)
      if (s.warp_float[w] > best || (s.warp_float[w] == best && s.warp_int[w] < best_index)) { best = s.warp_float[w]; best_index = s.warp_int[w]; }
    s.max = best;
    s.argmax = best_index;
  }
  cluster.sync();
  float top = -INFINITY;
  int top_index = vocab;
  for (int c = 0; c < ranks; ++c) {
    const LimitShared* theirs = cluster.map_shared_rank(&s, c);
    if (theirs->max > top) { top = theirs->max; top_index = theirs->argmax; }      // slices in order: the lowest index of a tie
  }
  auto finish = [&](int token) {      // by one thread of the cluster
    tokens[row] = token;
    if (record != nullptr) {
      record->last_token = token;
      record->counter += 1;
      if (source.advance) record->length += 1;
    }
  };
  if (greedy || top == -INFINITY) {
    if (rank == 0 && threadIdx.x == 0) finish(top_index < vocab ? top_index : 0);
    cluster.sync();            // the others may still read this CTA's best
    return;
  }
  Weights weight;
  weight.inverse = 1.0 / (double)temperature;
  weight.top = (double)top;
  weight.max = top;
  const unsigned top_key = order_key(top), no_key = order_key(-INFINITY);

  // ---- min-p: the lowest key whose weight reaches it
  Cut kept{0u, 0x7fffffff};
  if (least > 0.f) {
    if (threadIdx.x == 0) {
      const double wanted = (double)least;
      float guess = (float)fma((double)temperature, log(wanted), weight.top);
      unsigned key = min(max(order_key(cleaned(guess)), no_key + 1), top_key);
      for (int i = 0; i < 64 && key < top_key && weight(of_key(key)) < wanted; ++i) ++key;
      for (int i = 0; i < 64 && key > no_key + 1 && weight(of_key(key - 1)) >= wanted; ++i) --key;
      s.found_key = key;
    }
    __syncthreads();
    kept.key = s.found_key;
  }

  // ---- from the bins: the lowest key that can be kept, the interval that holds the cut
  unsigned lo = 0u, hi = top_key;
  int candidates = vocab, above_count = 0, interval_count = 0;
  if (binned) {
    const int per = SL_BINS / ranks;
    for (int b = threadIdx.x; b < per; b += SL_THREADS) {
      unsigned sum = 0u;
#pragma unroll
      for (int c = 0; c < SL_MOST_RANKS; ++c)
        if (c < ranks) sum += cluster.map_shared_rank(bins, c)[rank * per + b];
      segment[b] = sum;
    }
    cluster.sync();
    // thread t: SL_BINS_PER_THREAD bins from the top
    int count[SL_BINS_PER_THREAD], mine = 0, total;
    float low_sum = 0.f, high_sum = 0.f;
    const int first_bin = SL_BINS - 1 - (int)threadIdx.x * SL_BINS_PER_THREAD;
    auto edge_weight = [&](unsigned key) {
      const float x = fminf(of_key(key), top);
      return x >= top ? 1.f : x == x ? expf((x - top) / temperature) : 0.f;
    };
    {
      const int lowest_bin = first_bin - (SL_BINS_PER_THREAD - 1), owner = lowest_bin / per;
      const uint4* theirs = reinterpret_cast<const uint4*>(cluster.map_shared_rank(segment, owner) + (lowest_bin - owner * per));
      const uint4 low4 = theirs[0], high4 = theirs[1];
      count[0] = (int)high4.w; count[1] = (int)high4.z; count[2] = (int)high4.y; count[3] = (int)high4.x;
      count[4] = (int)low4.w; count[5] = (int)low4.z; count[6] = (int)low4.y; count[7] = (int)low4.x;
    }
#pragma unroll
    for (int j = 0; j < SL_BINS_PER_THREAD; ++j) mine += count[j];
    const int before = before_block(mine, s.warp_int, &total);
    if (threadIdx.x == 0) { s.found[0] = s.found[1] = 0; }
    __syncthreads();
    if (by_count) {
      int run = before;
#pragma unroll
      for (int j = 0; j < SL_BINS_PER_THREAD; ++j) {
        if (run < k && run + count[j] >= k) { s.found[0] = first_bin - j; s.found[2] = run; s.found[3] = run + count[j]; }
        run += count[j];
      }
      __syncthreads();
      lo = (unsigned)s.found[0] << SL_BIN_SHIFT;
      hi = lo | ((1u << SL_BIN_SHIFT) - 1u);
      above_count = s.found[2];
      interval_count = s.found[3] - above_count;
      candidates = s.found[3];
    } else {
      // bounds of the weights above each bin; a margin of 1e-3 covers the roundings
      float low[SL_BINS_PER_THREAD], high[SL_BINS_PER_THREAD];
#pragma unroll
      for (int j = 0; j < SL_BINS_PER_THREAD; ++j) {
        const unsigned edge = (unsigned)(first_bin - j) << SL_BIN_SHIFT, end = edge | ((1u << SL_BIN_SHIFT) - 1u);
        // a bin that min-p cuts through holds none for sure
        low[j] = count[j] == 0 || edge < kept.key ? 0.f : (float)count[j] * edge_weight(edge);
        high[j] = count[j] == 0 || end < kept.key ? 0.f : (float)count[j] * edge_weight(end);
        low_sum += low[j];
        high_sum += high[j];
      }
      float low_all, high_all, low_end, high_end;
      float low_run = before_block(low_sum, s.warp_float, &low_all, &low_end);
      float high_run = before_block(high_sum, s.warp_float2, &high_all, &high_end);
      low_all = fmaxf(low_all, 1.f);
      const float surely = p * high_all * 1.001f, maybe = p * low_all * 0.999f;
      if (threadIdx.x == 0) { s.found[0] = 0; s.found[1] = SL_BINS - 1; s.found[2] = total; }
      __syncthreads();
      if (low_run < surely && low_end >= surely) {      // one thread's
        int run = before, place = 0;
#pragma unroll
        for (int j = 0; j < SL_BINS_PER_THREAD; ++j)
          if (low_run < surely) { run += count[j]; low_run += low[j]; place = j; }
        s.found[0] = first_bin - place;
        s.found[2] = run;
      }
      if (high_run < maybe && high_end >= maybe) {
        int place = 0;
#pragma unroll
        for (int j = 0; j < SL_BINS_PER_THREAD; ++j)
          if (high_run < maybe) { high_run += high[j]; place = j; }
        s.found[1] = first_bin - place;
      }
      __syncthreads();
      lo = max((unsigned)s.found[0] << SL_BIN_SHIFT, kept.key);
      hi = max(lo, ((unsigned)s.found[1] << SL_BIN_SHIFT) | ((1u << SL_BIN_SHIFT) - 1u));
      candidates = s.found[2];
    }
  }

  // a warp's stretch of the slice, in the order of the vocabulary
  const int stretch = ((size + SL_WARPS - 1) / SL_WARPS + 31) / 32 * 32;
  const int walk_begin = min(size, warp * stretch), walk_end = min(size, walk_begin + stretch);
  auto walk = [&](auto&& visit) {      // every lane of the warp, `i` < 0 behind the end
    for (int base = walk_begin; base < walk_end; base += 32) {
      const int i = base + lane < walk_end ? base + lane : -1;
      visit(i, i >= 0 ? at(i) : -INFINITY);
    }
  };
  // tokens of [low, high] in `limit` to this CTA's list, in no order; counts known to fit
  auto collect = [&](unsigned low, unsigned high, Cut limit, int room) {
    if (threadIdx.x == 0) s.count = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < size; i += SL_THREADS) {
      const unsigned key = order_key(at(i));
      if (key >= low && key <= high && limit.keeps(key, begin + i)) {
        const int to = atomicAdd(&s.count, 1);
        if (to < room) list[to] = place_of(key, begin + i);
      }
    }
  };
  // the lists of all CTAs, sorted; the first CTA, the others wait
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

  if (binned && candidates <= SL_LIST) {
    // ---- few candidates: the first CTA cuts and draws
    const unsigned lowest = max(lo, kept.key);
    collect(lowest, 0xffffffffu, kept, SL_LIST);
    double tail = 0.0;
    if (by_weight && !by_count) {
      for (int i = threadIdx.x; i < size; i += SL_THREADS) {
        const float x = at(i);
        const unsigned key = order_key(x);
        if (key < lowest && key >= kept.key) tail += weight(x);
      }
      tail = sum_block(tail, s.warp_double);
    }
    if (threadIdx.x == 0) s.tail = tail;
    cluster.sync();
    int n = 0;
    if (rank == 0) {
      n = gather(SL_LIST);
      tail = 0.0;
      for (int c = 0; c < ranks; ++c) tail += cluster.map_shared_rank(&s, c)->tail;
    }
    cluster.sync();
    if (rank != 0) return;
    sort_places(all_listed, n);
    // thread t: SL_EACH neighbours
    constexpr int SL_EACH = SL_LIST / SL_THREADS;
    int stay = by_count ? min(n, k) : n;
    const int each = (n + SL_THREADS - 1) / SL_THREADS, first = threadIdx.x * each;
    double w[SL_EACH], all;
    if (by_weight) {
      double mine = 0.0;
#pragma unroll
      for (int i = 0; i < SL_EACH; ++i) {
        w[i] = i < each && first + i < stay ? weight(of_key(key_of(all_listed[first + i]))) : 0.0;
        mine += w[i];
      }
      double run = before_block(mine, s.warp_double, &all);
      const double target = (double)p * (all + tail);
      int passed = 0;          // tokens whose sums stay below the target
#pragma unroll
      for (int i = 0; i < SL_EACH; ++i) {
        run += w[i];
        passed += i < each && first + i < stay && run < target;
      }
      stay = min(stay, 1 + sum_block(passed, s.warp_int));
    }
    // what stays, in the order of the vocabulary: index, key
    __syncthreads();
    for (int i = threadIdx.x; i < stay; i += SL_THREADS) {
      const Place place = all_listed[i];
      all_listed[i] = ((Place)(unsigned)index_of(place) << 32) | key_of(place);
    }
    sort_places(all_listed, stay);
    const int share = (stay + SL_THREADS - 1) / SL_THREADS, from_place = threadIdx.x * share;
    double mine = 0.0;
#pragma unroll
    for (int i = 0; i < SL_EACH; ++i) {
      w[i] = i < share && from_place + i < stay ? weight(of_key((unsigned)all_listed[from_place + i])) : 0.0;
      mine += w[i];
    }
    double run = before_block(mine, s.warp_double, &all);
    const double target = (double)u * all;
    if (threadIdx.x == 0) { s.found[0] = 0x7fffffff; s.found[1] = 0; }
    __syncthreads();
    int reached = 0x7fffffff, last_kept = -1;
#pragma unroll
    for (int i = 0; i < SL_EACH; ++i) {
      run += w[i];
      if (w[i] > 0.0) {
        last_kept = from_place + i;
        if (run > target && reached == 0x7fffffff) reached = from_place + i;
      }
    }
    if (reached != 0x7fffffff) atomicMin(&s.found[0], reached);
    if (last_kept >= 0) atomicMax(&s.found[1], last_kept);
    __syncthreads();
    if (threadIdx.x == 0) finish((int)(all_listed[s.found[0] < stay ? s.found[0] : s.found[1]] >> 32));
    return;
  }

  // ---- many candidates: the cuts are found together
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
      int count = 0;
      for (int w = 0; w < SL_WARPS; ++w) { sum += s.part_double[threadIdx.x][w]; count += s.part_int[threadIdx.x][w]; }
      s.sums[turn][threadIdx.x] = sum;
      s.counts[turn][threadIdx.x] = count;
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
  // the cut in [low, high], which holds `count` kept keys; `above` before them
  auto cut_together = [&](bool weighed, unsigned low, unsigned high, double above, double target, int count) -> Cut {
    while (count > SL_CUT && low < high) {
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
          if (above + sums[j] >= target || last) { chosen = j; count = counts[j]; open = false; }
          else above += sums[j];
        }
      }
      const unsigned long long end = (unsigned long long)high - (unsigned long long)chosen * step;
      low = end >= (unsigned long long)low + step - 1 ? (unsigned)(end - (step - 1)) : low;
      high = (unsigned)end;
    }
    if (count <= SL_CUT) {
      collect(low, high, kept, SL_CUT);
      cluster.sync();
      if (rank == 0) {
        const int n = gather(SL_CUT);
        sort_places(all_listed, n);
        constexpr int EACH = SL_CUT / SL_THREADS;
        const int each = (n + SL_THREADS - 1) / SL_THREADS, first = threadIdx.x * each;
        int stay = min(n, max(1, (int)(target - above)));
        if (weighed) {
          double w[EACH], mine = 0.0, all;
#pragma unroll
          for (int i = 0; i < EACH; ++i) {
            w[i] = i < each && first + i < n ? weight(of_key(key_of(all_listed[first + i]))) : 0.0;
            mine += w[i];
          }
          double run = above + before_block(mine, s.warp_double, &all);
          int passed = 0;
#pragma unroll
          for (int i = 0; i < EACH; ++i) {
            run += w[i];
            passed += i < each && first + i < n && run < target;
          }
          stay = min(n, 1 + sum_block(passed, s.warp_int));
        }
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
    // more equal keys than an interval holds: the index of the last one that stays, by counting
    const int stay = weighed ? ties_kept(above, weight(of_key(low)), target, count) : min(count, max(1, (int)(target - above)));
    int mine = 0;
    walk([&](int i, float x) { mine += __popc(__ballot_sync(0xffffffffu, i >= 0 && order_key(x) == low && kept.keeps(low, begin + i))); });
    __syncthreads();
    if (lane == 0) s.warp_int[warp] = mine;
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
    if (place < stay && stay <= place + mine)
      walk([&](int i, float x) {
        const bool in = i >= 0 && order_key(x) == low && kept.keeps(low, begin + i);
        const unsigned mask = __ballot_sync(0xffffffffu, in);
        if (in && place + __popc(mask & ((2u << lane) - 1u)) == stay) s.cut_index = begin + i;
        place += __popc(mask);
      });
    cluster.sync();
    Cut cut{low, 0x7fffffff};
    for (int c = 0; c < ranks; ++c) {
      const int found = cluster.map_shared_rank(&s, c)->cut_index;
      if (found >= 0) cut.index = found;
    }
    cluster.sync();
    return cut;
  };

  if (by_count) {
    // every key of the interval, min-p or not: the smaller of the two beginnings stays
    const Cut before = kept;
    kept = Cut{0u, 0x7fffffff};
    Cut cut = cut_together(false, lo, hi, (double)above_count, (double)k, interval_count);
    kept = before;
    kept.tighten(cut);
    lo = kept.key;
    hi = top_key;
  }
  if (by_weight) {
    double sums[SL_PARTS];
    int counts[SL_PARTS];
#pragma unroll
    for (int j = 0; j < SL_PARTS; ++j) { sums[j] = 0.0; counts[j] = 0; }
    for (int i = threadIdx.x; i < size; i += SL_THREADS) {
      const float x = at(i);
      const unsigned key = order_key(x);
      if (kept.keeps(key, begin + i)) {
        const double w = weight(x);
        sums[0] += w;
        if (key > hi) sums[1] += w;
        else if (key >= lo) counts[0] += 1;
      }
    }
    exchange(sums, counts);
    kept.tighten(cut_together(true, lo, hi, sums[1], (double)p * sums[0], counts[0]));
  }

  // ---- the draw
  double sum = 0.0;
  walk([&](int i, float x) {
    const unsigned key = order_key(x);
    if (i >= 0 && kept.keeps(key, begin + i)) sum += weight(x);
  });
  sum = warp_sum64(sum);
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
  const double my_end = run + s.kept;
  // the CTA, then the warp, whose sums the draw falls into; what rounding leaves behind the last belongs to it
  if (target >= run && s.kept > 0.0 && (target < my_end || rank == last_rank)) {
    double begin_sum = run;
    int last_warp = 0, chosen = -1;
    for (int w = 0; w < SL_WARPS; ++w)
      if (s.warp_double[w] > 0.0) last_warp = w;
    double so_far = run;
    for (int w = 0; w < SL_WARPS && chosen < 0; ++w) {
      if (s.warp_double[w] > 0.0 && (target < so_far + s.warp_double[w] || w == last_warp)) { chosen = w; begin_sum = so_far; }
      so_far += s.warp_double[w];
    }
    if (warp == chosen) {
      int found = -1, last_kept = -1;
      double running = begin_sum;
      for (int base = walk_begin; base < walk_end && found < 0; base += 32) {
        const int i = base + lane < walk_end ? base + lane : -1;
        const float x = i >= 0 ? at(i) : -INFINITY;
        const double w = i >= 0 && kept.keeps(order_key(x), begin + i) ? weight(x) : 0.0;
        double inclusive = w;
#pragma unroll
        for (int offset = 1; offset < 32; offset <<= 1) {
          const double up = __shfl_up_sync(0xffffffffu, inclusive, offset);
          if (lane >= offset) inclusive += up;
        }
        const unsigned some = __ballot_sync(0xffffffffu, w > 0.0);
        const unsigned hit = __ballot_sync(0xffffffffu, w > 0.0 && running + inclusive > target);
        if (some != 0u) last_kept = base + 31 - __clz(some);
        if (hit != 0u) found = base + __ffs(hit) - 1;
        running += __shfl_sync(0xffffffffu, inclusive, 31);
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
