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
// A cluster of CTAs takes a row, a slice each, which stays in shared memory where it fits and is read again (from the L2 cache, mostly) where
// not.  While it is read the largest logits of blocks of 40 are noted: the k-th of them bounds the k-th logit from below, and
// later passes look only into blocks that reach a bound.
//   few            Logits above such a bound (top-k up to 1,200), above min-p's border, or, for top-p alone, the thousand largest, if a sample of
//                  the rest says that they hold p: the whole is then summed in the pass that finds them.  They go to the first CTA
//                  in the order of the vocabulary; each learns its rank among them, the cut follows, and the draw.
//   else           The cuts are found together.  All logits are counted in 4,096 bins of T / 128; the CTAs add the bins up through distributed
//                  shared memory, and the bin that holds the cut is known for top-k, and for top-p but for a bin or two (a bin's weights
//                  are within a hundredth of one another).  The weights above it are summed, the tokens around it go to the first CTA, which
//                  ranks them and cuts.  If the cut is not there after all, or more tokens are than one CTA ranks (equal logits, say),
//                  an interval of keys that surely holds it is split eightfold until it is found.  Then the draw: sums by CTA,
//                  by warp, by chunk of a warp's stretch, by thread.
// Bound by memory while no more than a few logits of a row need weights, by 64-bit arithmetic where all do (13 instructions each; the pass of
// rows without limits runs at half that pipe's rate), by the steps between CTAs for few rows.  256 rows of 152,064 logits, T 0.8: greedy
// 48 us, top-k 50 76, 1,000 122, top-p 0.9 232, min-p 0.05 63, no limit 125, all kinds mixed 104 to 115; one row: 6, 11, 20, 29, 10 and 13 us.
// Sums are taken in a fixed order, of ranks or of places (no floating-point atomics): a row's token depends on its row alone (and, where the draw lies
// within the last bits of a sum from a border, on how many CTAs a row gets in a batch of this size).
#include <cooperative_groups.h>

#include "uniform.cuh"

namespace mlr {

namespace cg = cooperative_groups;

constexpr int SL_THREADS = 256, SL_WARPS = SL_THREADS / 32;
constexpr int SL_BINS = 4096, SL_BINS_PER_THREAD = SL_BINS / SL_THREADS;
constexpr int SL_BOUND_BINS = 1024;
constexpr float SL_BINS_PER_T = 128.f;
constexpr int SL_MOST_K = 1200;          // a top-k whose candidates fit a list, it is likely
constexpr int SL_NUCLEUS = 1000;         // largest logits among which a top-p is looked for first
constexpr int SL_LIST = 2048;            // candidates that one CTA cuts and draws from
constexpr int SL_CUT = 1024;             // keys of an interval that one CTA orders
constexpr int SL_EACH = SL_LIST / SL_THREADS;
constexpr int SL_AHEAD = 10;             // reads of 16 bytes that a thread has in flight while it looks for the largest logit: a block
constexpr int SL_TOPS = 16;              // largest logits that a thread remembers, of a block each or of some
constexpr int SL_ORDERED = 2048;         // rows that are brought into order
constexpr int SL_BUCKETS = 4096, SL_BUCKET_MOST = 64;
constexpr int SL_PARTS = 8;
constexpr int SL_MOST_RANKS = 8;
static_assert(SL_BINS_PER_THREAD % 4 == 0, "a thread reads bins by fours");

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
  unsigned key_range[2];
  float cut_x;                    // what the first CTA found
  int cut_listed;                 // tokens of the interval that stay, in order in `all_listed`; -1: not there
  int cut_index;
  double kept;
  // of this CTA alone
  double warp_double[SL_WARPS], part_double[SL_PARTS][SL_WARPS];
  float warp_float[SL_WARPS], warp_float2[SL_WARPS];
  int warp_int[SL_WARPS], part_int[SL_PARTS][SL_WARPS];
  float found_x;
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

// exp((x - top) / T) in 64 bits by Tang's method (table-driven exponentials, 1989): (x - top) 16 / (T ln 2) = n + f with n whole and
// |f| <= 1/2; the weight is 2^(n / 16) (1 + g + g^2 / 2 .. g^6 / 720) with g = f ln 2 / 16, |g| < 0.022: the remainder is below 2^-50.
// `table` holds 2^(n / 16), sixteen numbers: they fill the banks of shared memory once, so that a warp reads any of them together.
struct Weights {
  double scale, top;
  float least;                 // weights of logits up to it are below exp(-700), taken as 0
  const double* table;
  __device__ __forceinline__ double operator()(float x) const {
    constexpr double RAISE = 6755399441055744.0;      // 1.5 * 2^52
    constexpr double G = 0.043321698784996581;        // ln 2 / 16
    const double z = ((double)fminf(x, 3.402823466e38f) - top) * scale;
    const double raised = z + RAISE, f = z - (raised - RAISE);
    const int n = __double2loint(raised);
    double q = fma(f, G * G * G * G * G * G / 720.0, G * G * G * G * G / 120.0);
    q = fma(f, q, G * G * G * G / 24.0);
    q = fma(f, q, G * G * G / 6.0);
    q = fma(f, q, G * G / 2.0);
    q = fma(f, q, G);
    const double t = table[n & 15];
    const double value = fma(t, f * q, t);
    const double scaled = __hiloint2double(__double2hiint(value) + ((n >> 4) << 20), __double2loint(value));
    return x > least ? scaled : 0.0;                 // (0 for a NaN too)
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

// A set of kept tokens: logits above `x`, and of those equal to it the indexes up to `index`.  (NaN, which fills up a slice, is never kept.)
struct Cut {
  float x;
  int index;
  __device__ __forceinline__ bool keeps(float other, int i) const { return other > x || (other == x && i <= index); }
  __device__ __forceinline__ void tighten(const Cut& other) {
    if (other.x > x || (other.x == x && other.index < index)) *this = other;
  }
};

// How many of equal tokens of weight w stay in the shortest beginning that comes to `target`, `above` being before them.
__device__ __forceinline__ int ties_kept(double above, double w, double target, int ties) {
  if (!(w > 0.0)) return ties;
  const double wanted = ceil((target - above) / w);
  return wanted < 1.0 ? 1 : wanted < (double)ties ? (int)wanted : ties;
}

// Rising order by a bitonic network, EACH neighbouring numbers per thread in registers: pairs of a thread, of a warp by shuffles, of
// further ones through the array itself.
template <int EACH>
__device__ __forceinline__ void sort_in_registers(Place* a, int n) {
  constexpr int SIZE = EACH * SL_THREADS;
  const int first = (int)threadIdx.x * EACH;
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
#pragma unroll
    for (int apart = EACH / 2; apart > 0; apart /= 2)
      if (apart < run)
#pragma unroll
        for (int i = 0; i < EACH; ++i)
          if ((i & apart) == 0) exchange(v[i], v[i + apart], ((first + i) & run) == 0);
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < EACH; ++i) a[first + i] = v[i];
}
// The array has room up to the next size that is sorted; behind n lie the largest numbers.
__device__ __noinline__ void sort_places(Place* a, int n) {
  __syncthreads();
  if (n <= SL_LIST / 2) sort_in_registers<SL_LIST / 2 / SL_THREADS>(a, n);
  else sort_in_registers<SL_LIST / SL_THREADS>(a, n);
  __syncthreads();
}

// What one thread owns of up to SL_LIST listed tokens: `each` neighbours from `first` on.
struct Owned {
  int each, first;
  __device__ __forceinline__ explicit Owned(int n) : each((n + SL_THREADS - 1) / SL_THREADS), first((int)threadIdx.x * each) {}
  __device__ __forceinline__ bool has(int i, int n) const { return i < each && first + i < n; }
};
// How many of the listed tokens come before each of this thread's own, by the whole CTA.  Up to 256 are compared with one another by several
// threads each (60 tokens: 0.5 us, where a warp sorted them in 2.4).  More fall into buckets of equal width in [low, high],
// and are compared with those of their bucket (1,150 tokens: 5 us, sorted 14).  Where a bucket holds too many, a copy is sorted.
// `buckets` [SL_BUCKETS]; `spare` has room for the next size that is sorted.
__device__ __noinline__ void ranks_of(Place* listed, int n, float low, float high, unsigned* buckets, Place* spare, int* room, int (&ranks)[SL_EACH]) {
  const Owned own(n);
#pragma unroll
  for (int i = 0; i < SL_EACH; ++i) ranks[i] = 0;
  if (n <= 256) {
    int threads = 1;                        // per token
    while (threads < 32 && n * threads * 2 <= SL_THREADS) threads *= 2;
    if (threadIdx.x == 0) listed[n] = ~(Place)0;      // pairs
    __syncthreads();
    const int token = (int)threadIdx.x / threads, sub = (int)threadIdx.x % threads;
    const Place me = token < n ? listed[token] : 0;
    int smaller = 0;
    for (int j = 2 * sub; j < n; j += 2 * threads) {
      const ulonglong2 pair = *reinterpret_cast<const ulonglong2*>(listed + j);
      smaller += (pair.x < me) + (pair.y < me);
    }
    for (int apart = 1; apart < threads; apart *= 2) smaller += __shfl_xor_sync(0xffffffffu, smaller, apart);
    if (sub == 0) buckets[token] = (unsigned)smaller;
    __syncthreads();
    if (own.has(0, n)) ranks[0] = (int)buckets[own.first];
    __syncthreads();
    return;
  }
  const float scale = high > low && low > -INFINITY && high < INFINITY ? (float)SL_BUCKETS / (high - low) : 0.f;
  for (int b = threadIdx.x; b < SL_BUCKETS / 4; b += SL_THREADS) reinterpret_cast<uint4*>(buckets)[b] = make_uint4(0u, 0u, 0u, 0u);
  __syncthreads();
  Place places[SL_EACH];
  int bucket[SL_EACH], order[SL_EACH];
#pragma unroll
  for (int i = 0; i < SL_EACH; ++i) {
    if (!own.has(i, n)) continue;
    places[i] = listed[own.first + i];
    bucket[i] = (int)fminf((high - of_key(key_of(places[i]))) * scale, (float)(SL_BUCKETS - 1));
    order[i] = (int)atomicAdd(&buckets[bucket[i]], 1u);
  }
  __syncthreads();
  constexpr int MINE = SL_BUCKETS / SL_THREADS;
  int counts[MINE], here = 0, most = 0, total;
  int4* my_buckets = reinterpret_cast<int4*>(buckets) + MINE / 4 * threadIdx.x;
#pragma unroll
  for (int j = 0; j < MINE; j += 4) {
    const int4 four = my_buckets[j / 4];
    counts[j] = four.x, counts[j + 1] = four.y, counts[j + 2] = four.z, counts[j + 3] = four.w;
  }
#pragma unroll
  for (int j = 0; j < MINE; ++j) { here += counts[j]; most = max(most, counts[j]); }
  const bool crowded = __syncthreads_or(most > SL_BUCKET_MOST);
  if (crowded) {
#pragma unroll
    for (int i = 0; i < SL_EACH; ++i)
      if (own.has(i, n)) spare[own.first + i] = places[i];
    sort_places(spare, n);
#pragma unroll
    for (int i = 0; i < SL_EACH; ++i) {
      if (!own.has(i, n)) continue;
      int from = 0, until = n;
      while (from < until) {
        const int middle = (from + until) / 2;
        if (spare[middle] < places[i]) from = middle + 1;
        else until = middle;
      }
      ranks[i] = from;
    }
    __syncthreads();
    return;
  }
  int run = before_block(here, room, &total);
#pragma unroll
  for (int j = 0; j < MINE; ++j) { const int count = counts[j]; counts[j] = run; run += count; }
#pragma unroll
  for (int j = 0; j < MINE; j += 4) my_buckets[j / 4] = make_int4(counts[j], counts[j + 1], counts[j + 2], counts[j + 3]);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < SL_EACH; ++i)
    if (own.has(i, n)) spare[buckets[bucket[i]] + order[i]] = places[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < SL_EACH; ++i) {
    if (!own.has(i, n)) continue;
    const int begin = (int)buckets[bucket[i]], end = bucket[i] + 1 < SL_BUCKETS ? (int)buckets[bucket[i] + 1] : n;
    ranks[i] = begin;
    for (int j = begin; j < end; ++j) ranks[i] += spare[j] < places[i];
  }
  __syncthreads();
}

// Quads (four neighbouring logits) of a warp's stretch where a slice has at most so many; the blocks of a thread's `tops`, and how many of them.
__host__ __device__ __forceinline__ int quads_of_warp(int quads) { return (quads + SL_WARPS - 1) / SL_WARPS; }
__host__ __device__ __forceinline__ int blocks_per_top(int quads) {
  const int most = 32 * SL_AHEAD * SL_TOPS, per = (quads_of_warp(quads) + most - 1) / most;
  return per > 1 ? per : 1;
}
__host__ __device__ __forceinline__ int tops_of(int quads) {      // (more quads never make it more than SL_TOPS)
  const int per = blocks_per_top(quads) * 32 * SL_AHEAD;
  return (quads_of_warp(quads) + per - 1) / per;
}

constexpr float NOTHING = __builtin_nanf("");

__device__ __noinline__ float4 edge_quad(const float* from, int size, int i) {
  auto one = [&](int e) { return e >= 0 && e < size ? cleaned(__ldcg(from + e)) : NOTHING; };
  return make_float4(one(i), one(i + 1), one(i + 2), one(i + 3));
}
// A slice of a row by quads: quad q holds the logits 4 q - shift .. 4 q - shift + 3, NaN where these lie outside.
template <bool RESIDENT>
struct Slice {
  const float* from;
  float4* held;               // in shared memory, once they have been read
  int shift, size;
  // from memory: the quads first, first + 32, .. before `end`, NaN from there on; a warp's `first`s are neighbours
  template <int COUNT>
  __device__ __forceinline__ void read(int first, int end, float4 (&x)[COUNT]) const {
    const float4* quads = reinterpret_cast<const float4*>(from - shift);
    const int inner_begin = shift > 0 ? 1 : 0, inner_end = (size + shift) / 4, until = min(end, inner_end);      // these lie inside as a whole
    const int lowest = first - (int)(threadIdx.x & 31);
    if (lowest >= inner_begin && lowest + 32 * COUNT <= until) {
#pragma unroll
      for (int j = 0; j < COUNT; ++j) x[j] = __ldcg(quads + first + 32 * j);
#pragma unroll
      for (int j = 0; j < COUNT; ++j) x[j] = make_float4(cleaned(x[j].x), cleaned(x[j].y), cleaned(x[j].z), cleaned(x[j].w));
      return;
    }
#pragma unroll
    for (int j = 0; j < COUNT; ++j) {
      x[j] = make_float4(NOTHING, NOTHING, NOTHING, NOTHING);
      if (first + 32 * j >= inner_begin && first + 32 * j < until) x[j] = __ldcg(quads + first + 32 * j);
    }
#pragma unroll
    for (int j = 0; j < COUNT; ++j)
      if (first + 32 * j >= inner_begin && first + 32 * j < until)
        x[j] = make_float4(cleaned(x[j].x), cleaned(x[j].y), cleaned(x[j].z), cleaned(x[j].w));
    if (lowest < inner_begin || (end > inner_end && lowest + 32 * COUNT > inner_end)) {      // the slice's first or last quad, in part
#pragma unroll
      for (int j = 0; j < COUNT; ++j) {
        const int q = first + 32 * j;
        if (q < end && (q < inner_begin || q >= inner_end)) x[j] = edge_quad(from, size, 4 * q - shift);
      }
    }
  }
  template <int COUNT>
  __device__ __forceinline__ void get(int first, int end, float4 (&x)[COUNT]) const {
    if constexpr (RESIDENT) {
#pragma unroll
      for (int j = 0; j < COUNT; ++j)
        x[j] = first + 32 * j < end ? held[first + 32 * j] : make_float4(NOTHING, NOTHING, NOTHING, NOTHING);
    } else {
      read(first, end, x);
    }
  }
};

template <bool RESIDENT>
__global__ void __launch_bounds__(SL_THREADS, 2)
sample_limited_kernel(const float* logits, const LimitSource source, int* __restrict__ tokens, int vocab, int slice, int room_bytes, int ordered_rows) {
  pdl_trigger();
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  int row = blockIdx.x / ranks;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  extern __shared__ __align__(16) uint8_t limit_shared[];
  float* held = reinterpret_cast<float*>(limit_shared);                          // the slice
  Place* list = reinterpret_cast<Place*>(limit_shared + room_bytes);             // [SL_LIST] this CTA's candidates
  unsigned* bins = reinterpret_cast<unsigned*>(list + SL_LIST);                  // [SL_BINS]
  Place* all_listed = reinterpret_cast<Place*>(bins);                            // when the bins have been read, the candidates of all CTAs [SL_LIST]
  unsigned* segment = bins + SL_BINS;                                            // [SL_BINS / ranks]
  float* tops = reinterpret_cast<float*>(segment + SL_BINS / ranks);
  double (*chunks)[32] = reinterpret_cast<double (*)[32]>(bins);                 // at last, [SL_WARPS][32] sums of a warp's chunks
  __shared__ LimitShared s;
  __shared__ double table[16];
  static_assert(SL_LIST * sizeof(Place) <= SL_BINS * sizeof(unsigned), "the candidates lie where the bins were");

  if (ordered_rows > 0) {
    // ---- rows whose weights are all needed take longest, and begin first
    pdl_wait();
    constexpr int MOST = SL_ORDERED / SL_THREADS;
    const int each = (ordered_rows + SL_THREADS - 1) / SL_THREADS, first = (int)threadIdx.x * each;
    unsigned heavy = 0u;
#pragma unroll
    for (int j = 0; j < MOST; ++j)
      if (j < each && first + j < ordered_rows) {
        const int slot = source.row_slot != nullptr ? source.row_slot[first + j] : first + j;
        if (slot >= 0 && slot < source.slots) {
          const float temperature = source.state != nullptr ? source.state[slot].temperature : source.temperatures[slot];
          const int k = source.top_k != nullptr ? source.top_k[slot] : 0;
          const float least = source.min_p != nullptr ? source.min_p[slot] : 0.f;
          heavy |= (unsigned)(temperature > 0.f && !(k > 0 && k <= SL_MOST_K) && !(least > 0.f)) << j;
        }
      }
    int all, before = before_block(__popc(heavy), s.warp_int, &all);
    const int place = row;
#pragma unroll
    for (int j = 0; j < MOST; ++j)
      if (j < each && first + j < ordered_rows) {
        const bool one = heavy >> j & 1u;
        if ((one ? before : all + first + j - before) == place) s.found[0] = first + j;
        before += one;
      }
    __syncthreads();
    row = s.found[0];
  }
  // ---- the slice and its largest logits
  const int begin = min(vocab, rank * slice), size = min(vocab, begin + slice) - begin;
  const float* from = logits + (size_t)row * vocab + begin;
  // Four logits at a time, from 16-byte boundaries on: quad q holds the slice's logits 4 q - shift .. 4 q - shift + 3, NaN where these lie outside.
  // A warp looks at neighbouring quads, its stretch, in every pass.
  const int shift = (int)(((uintptr_t)from >> 2) & 3), quads = size > 0 ? (size + shift + 3) / 4 : 0;
  const int per_warp = quads_of_warp(quads), quad_begin = min(quads, warp * per_warp), quad_end = min(quads, quad_begin + per_warp);
  const Slice<RESIDENT> quads_of{from, reinterpret_cast<float4*>(held), shift, size};
  const int per_top = blocks_per_top(quads), num_tops = tops_of(quads);
  float* my_tops = tops + threadIdx.x;                   // [num_tops][SL_THREADS]
  pdl_wait();
  float mine = -INFINITY, least_top = INFINITY;
  for (int t = 0; t < num_tops; ++t) {
    float high = -INFINITY;
    for (int block = t * per_top; block < (t + 1) * per_top; ++block) {
      const int q = quad_begin + block * 32 * SL_AHEAD + lane;
      float4 v[SL_AHEAD];
      quads_of.read(q, quad_end, v);
#pragma unroll
      for (int j = 0; j < SL_AHEAD; ++j) {
        if constexpr (RESIDENT)
          if (q + 32 * j < quad_end) reinterpret_cast<float4*>(held)[q + 32 * j] = v[j];
        high = fmaxf(high, fmaxf(fmaxf(v[j].x, v[j].y), fmaxf(v[j].z, v[j].w)));
      }
    }
    my_tops[t * SL_THREADS] = high;
    mine = fmaxf(mine, high);
    if (high > -INFINITY) least_top = fminf(least_top, high);
  }
  if (threadIdx.x < 16) table[threadIdx.x] = exp2((double)threadIdx.x * (1.0 / 16.0));
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

  // ---- the slice's largest logit, and two of the blocks' largest ones: the k-th, and the k / ranks-th.  All slices together hold k logits that
  // are as large as the least of their k / ranks-th ones, and each holds k as large as its k-th.
  {
    const float high = warp_max(mine), low = -warp_max(-least_top);
    if (lane == 0) { s.warp_float[warp] = high; s.warp_float2[warp] = low; }
    const bool bounded = (by_count ? k <= SL_MOST_K : by_weight) && vocab > SL_LIST;
    const int wanted = by_count ? k : SL_NUCLEUS;
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
      for (int t = 0; t < num_tops; ++t) {
        const float one = my_tops[t * SL_THREADS];
        if (one > -INFINITY) atomicAdd(&bins[scale > 0.f ? min(SL_BOUND_BINS - 1, (int)((highest - one) * scale)) : 0], 1u);
      }
      __syncthreads();
      constexpr int EACH = SL_BOUND_BINS / SL_THREADS;
      int counts[EACH], here = 0, total, until;
#pragma unroll
      for (int j = 0; j < EACH; ++j) { counts[j] = (int)bins[threadIdx.x * EACH + j]; here += counts[j]; }
      const int before = before_block(here, s.warp_int, &total, &until);
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const int place = m == 0 ? wanted : (wanted + ranks - 1) / ranks;
        if (before < place && until >= place) {      // one thread's (none's where fewer blocks hold a number)
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
  // f(quad, its four logits) for the warp's stretch; f(logit, place in the slice) for those as large as `low`, which threads look for only in
  // blocks whose largest one is as large.
  auto for_quads = [&](auto&& f) {
    if constexpr (RESIDENT) {
      for (int base = quad_begin; base < quad_end; base += 32) {
        float4 x[1];
        quads_of.get(base + lane, quad_end, x);
        f(base + lane, x[0]);
      }
    } else {
      constexpr int AHEAD = 4;
      float4 next[AHEAD];
      quads_of.get(quad_begin + lane, quad_end, next);
      for (int base = quad_begin; base < quad_end; base += 32 * AHEAD) {
        float4 x[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) x[j] = next[j];
        quads_of.get(base + 32 * AHEAD + lane, quad_end, next);      // (while these are looked at)
#pragma unroll
        for (int j = 0; j < AHEAD; ++j)
          if (base + 32 * j < quad_end) f(base + 32 * j + lane, x[j]);
      }
    }
  };
  auto for_high = [&](float low, auto&& f) {
    constexpr int AHEAD = 5;
    static_assert(SL_AHEAD % AHEAD == 0, "whole steps of a block");
    for (int t = 0; t < num_tops; ++t) {
      const bool look = my_tops[t * SL_THREADS] >= low;
      if (__ballot_sync(0xffffffffu, look) == 0u) continue;
      const int end = min(quad_end, quad_begin + (t + 1) * per_top * 32 * SL_AHEAD);
      for (int q = quad_begin + t * per_top * 32 * SL_AHEAD + lane; q - lane < end; q += 32 * AHEAD) {
        float4 four[AHEAD];
        quads_of.get(q, look ? end : 0, four);
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
          const float4 x = four[j];
          if (fmaxf(fmaxf(x.x, x.y), fmaxf(x.z, x.w)) >= low) {
            const int i = 4 * (q + 32 * j) - shift;
            if (x.x >= low) f(x.x, i);
            if (x.y >= low) f(x.y, i + 1);
            if (x.z >= low) f(x.z, i + 2);
            if (x.w >= low) f(x.w, i + 3);
          }
        }
      }
    }
  };
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
      for_high(top, [&](float, int i) { atomicMin(&s.argmax, begin + i); });
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
  weight.scale = 23.083120654223414 / (double)temperature;      // 16 / ln 2
  // Logits above the float nearest to top - 700 T are above that number itself; the largest one weighs whatever T is.  An infinite logit
  // counts as the largest number, and no other beside it.
  weight.top = (double)fminf(top, 3.402823466e38f);
  const float next_lower = of_key(order_key(top) - (top == 0.f ? 2u : 1u));      // (-0 is none)
  weight.least = top < INFINITY ? fminf((float)(weight.top - 700.0 * (double)temperature), next_lower) : next_lower;
  weight.table = table;
  const unsigned top_key = order_key(top), no_key = order_key(-INFINITY);

  // ---- min-p: the lowest logit whose weight reaches it
  const Cut everything{-INFINITY, 0x7fffffff};
  Cut kept = everything;
  if (at_least > 0.f) {
    if (threadIdx.x == 0) {
      const double wanted = (double)at_least;
      float guess = (float)fma((double)temperature, log(wanted), weight.top);
      unsigned key = min(max(order_key(cleaned(guess)), no_key + 1), top_key);
      for (int i = 0; i < 64 && key < top_key && weight(of_key(key)) < wanted; ++i) ++key;
      for (int i = 0; i < 64 && key > no_key + 1 && weight(of_key(key - 1)) >= wanted; ++i) --key;
      s.found_x = of_key(key);
    }
    __syncthreads();
    kept.x = s.found_x;
  }

  // counts in bins: those of all CTAs, SL_BINS_PER_THREAD neighbours per thread
  int count[SL_BINS_PER_THREAD];
  const int per = SL_BINS / ranks, first_bin = (int)threadIdx.x * SL_BINS_PER_THREAD;
  auto clear_bins = [&]() {
    for (int b = threadIdx.x; b < SL_BINS / 4; b += SL_THREADS) reinterpret_cast<uint4*>(bins)[b] = make_uint4(0u, 0u, 0u, 0u);
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
    const int4* theirs = reinterpret_cast<const int4*>(cluster.map_shared_rank(segment, owner) + (first_bin - owner * per));
#pragma unroll
    for (int j = 0; j < SL_BINS_PER_THREAD; j += 4) {
      const int4 four = theirs[j / 4];
      count[j] = four.x, count[j + 1] = four.y, count[j + 2] = four.z, count[j + 3] = four.w;
    }
  };
  // to this CTA's list, in no order (its length was set to 0 before a barrier)
  auto append = [&](float x, int i) {
    const int to = atomicAdd(&s.count, 1);
    if (to < SL_LIST) list[to] = place_of(order_key(x), begin + i);
  };
  auto empty_list = [&]() {
    if (threadIdx.x == 0) s.count = 0;
    __syncthreads();
  };
  // a warp's quads, from place i on, in order: the wanted ones to list[to ..), no further than list[room)
  auto put_quad = [&](const float4& x, int i, int& to, int room, auto&& wanted) {
    const bool a = wanted(x.x, i), b = wanted(x.y, i + 1), c = wanted(x.z, i + 2), d = wanted(x.w, i + 3);
    const unsigned before = (1u << lane) - 1u;
    const unsigned as = __ballot_sync(0xffffffffu, a), bs = __ballot_sync(0xffffffffu, b), cs = __ballot_sync(0xffffffffu, c),
                   ds = __ballot_sync(0xffffffffu, d);
    int at_place = to + __popc(as & before) + __popc(bs & before) + __popc(cs & before) + __popc(ds & before);
    auto put = [&](bool in, float one, int place) {
      if (in) {
        if (at_place < room) list[at_place] = place_of(order_key(one), begin + place);
        ++at_place;
      }
    };
    put(a, x.x, i), put(b, x.y, i + 1), put(c, x.z, i + 2), put(d, x.w, i + 3);
    to += __popc(as) + __popc(bs) + __popc(cs) + __popc(ds);
  };
  // Each warp has put `found` tokens into a part of the list of its own: these are moved together.  False: a part is full.
  constexpr int PART = SL_LIST / SL_WARPS;
  auto pack = [&](int found, int& to, int& all) -> bool {
    __syncthreads();
    if (lane == 0) s.warp_int[warp] = found;
    __syncthreads();
    all = 0;
    bool fits = true;
#pragma unroll
    for (int w = 0; w < SL_WARPS; ++w) {
      const int theirs = s.warp_int[w];
      if (w == warp) to = all;
      all += theirs;
      fits = fits && theirs <= PART;
    }
    if (threadIdx.x == 0) s.count = all;
    if (!fits || all > SL_LIST) return false;
    Place moved[PART / 32];
#pragma unroll
    for (int j = 0; j < PART / 32; ++j)
      if (32 * j + lane < found) moved[j] = list[warp * PART + 32 * j + lane];
    __syncthreads();
#pragma unroll
    for (int j = 0; j < PART / 32; ++j)
      if (32 * j + lane < found) list[to + 32 * j + lane] = moved[j];
    return true;
  };
  // the tokens of [low, high] that `limit` keeps to the list, in the order of the vocabulary
  auto collect = [&](float low, float high, Cut limit) {
    auto wanted = [&](float x, int i) { return x >= low && x <= high && limit.keeps(x, begin + i); };
    // the warp's tokens to list[to ..), no further than list[room); returns how many there are
    auto find = [&](int to, int room) {
      const int start = to;
      for (int block = 0; block < num_tops * per_top; ++block) {
        const bool look = my_tops[block / per_top * SL_THREADS] >= low;
        if (__ballot_sync(0xffffffffu, look) == 0u) continue;
        const int first = quad_begin + block * 32 * SL_AHEAD + lane;
        float4 v[SL_AHEAD];
        quads_of.get(first, look ? quad_end : 0, v);
#pragma unroll
        for (int j = 0; j < SL_AHEAD; ++j) {
          const float4 x = v[j];
          if (__ballot_sync(0xffffffffu, fmaxf(fmaxf(x.x, x.y), fmaxf(x.z, x.w)) >= low) == 0u) continue;
          put_quad(x, 4 * (first + 32 * j) - shift, to, room, wanted);
        }
      }
      return to - start;
    };
    int to = 0, all;
    const int found = find(warp * PART, (warp + 1) * PART);
    if (!pack(found, to, all) && all <= SL_LIST) {      // a part is full: all over again, one behind the other
      __syncthreads();
      if (found > 0) find(to, SL_LIST);
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
  // Of n listed tokens the first `stay` in their order have the weights `w`: so many of them, `above` before them, stay until the weights come
  // to `target`, or to `share` of theirs.
  auto cut_by_weight = [&](const double (&w)[SL_EACH], const int (&ranks)[SL_EACH], int n, int stay, double above, double target, double share,
                           double* in_order) -> int {
    const Owned own(n), sorted(stay);
#pragma unroll
    for (int i = 0; i < SL_EACH; ++i)
      if (own.has(i, n) && ranks[i] < stay) in_order[ranks[i]] = w[i];
    __syncthreads();
    double next[SL_EACH], sum = 0.0, all;
#pragma unroll
    for (int i = 0; i < SL_EACH; ++i) {
      next[i] = sorted.has(i, stay) ? in_order[sorted.first + i] : 0.0;
      sum += next[i];
    }
    double run = above + before_block(sum, s.warp_double, &all);
    if (share > 0.0) target = share * all;
    int passed = 0;          // tokens whose sums stay below the target
#pragma unroll
    for (int i = 0; i < SL_EACH; ++i) {
      run += next[i];
      passed += sorted.has(i, stay) && run < target;
    }
    return min(stay, 1 + sum_block(passed, s.warp_int));
  };

  int turn = 0;
  // sums and counts of the parts of all CTAs
  auto exchange = [&](auto& sums, auto& counts) {
    constexpr int PARTS = sizeof(counts) / sizeof(int);
#pragma unroll
    for (int j = 0; j < PARTS; ++j) {
      sums[j] = warp_sum64(sums[j]);
      counts[j] = (int)__reduce_add_sync(0xffffffffu, (unsigned)counts[j]);
    }
    if (lane == 0)
#pragma unroll
      for (int j = 0; j < PARTS; ++j) { s.part_double[j][warp] = sums[j]; s.part_int[j][warp] = counts[j]; }
    __syncthreads();
    if (threadIdx.x < PARTS) {
      double sum = 0.0;
      int all = 0;
      for (int w = 0; w < SL_WARPS; ++w) { sum += s.part_double[threadIdx.x][w]; all += s.part_int[threadIdx.x][w]; }
      s.sums[turn][threadIdx.x] = sum;
      s.counts[turn][threadIdx.x] = all;
    }
    cluster.sync();
#pragma unroll
    for (int j = 0; j < PARTS; ++j) {
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
  bool few = (by_count && k <= SL_MOST_K) || kept.x > -INFINITY || vocab <= SL_LIST;
  const float lowest = by_count || !few ? fmaxf(bound, kept.x) : kept.x;
  double whole = 0.0;              // all weights, where top-p alone is looked for among the largest logits
  if (few) {
    collect(lowest, INFINITY, kept);
    cluster.sync();
  } else if (by_weight && !by_count && lowest > -INFINITY) {
    // Do the largest logits hold p of all weights?  Of them the blocks' largest ones are at hand, of the rest some quads are looked at.
    constexpr int LOOKED_AT = 4;
    float large = 0.f, rest = 0.f;
    for (int t = 0; t < num_tops; ++t) {
      const float one = my_tops[t * SL_THREADS];
      if (one >= lowest) large += expf((one - top) / temperature);
    }
    float4 some[LOOKED_AT];
    const int apart = (per_warp / LOOKED_AT + 31) / 32 * 32, looked_at = min(LOOKED_AT, (per_warp + max(apart, 1) - 1) / max(apart, 1));
#pragma unroll
    for (int j = 0; j < LOOKED_AT; ++j) {
      float4 x[1] = {make_float4(NOTHING, NOTHING, NOTHING, NOTHING)};
      if (j < looked_at) quads_of.get(quad_begin + j * apart + lane, quad_end, x);
      some[j] = x[0];
    }
    auto small = [&](float other) { return other < lowest ? expf((other - top) / temperature) : 0.f; };
#pragma unroll
    for (int j = 0; j < LOOKED_AT; ++j) rest += (small(some[j].x) + small(some[j].y)) + (small(some[j].z) + small(some[j].w));
    rest *= (float)per_warp / (float)max(1, min(per_warp, 32 * looked_at));
    double sums[2] = {(double)large, (double)rest};
    int counts[2] = {};
    exchange(sums, counts);
    if (sums[0] > (double)p * (sums[0] + sums[1])) {
      // all weights are summed, and the largest logits go to the list
      int to = warp * PART, moved_to, all;
      sums[0] = sums[1] = 0.0;
      for_quads([&](int q, const float4& x) {
        sums[0] += (weight(x.x) + weight(x.y)) + (weight(x.z) + weight(x.w));
        if (__ballot_sync(0xffffffffu, fmaxf(fmaxf(x.x, x.y), fmaxf(x.z, x.w)) >= lowest) != 0u)
          put_quad(x, 4 * q - shift, to, (warp + 1) * PART, [&](float one, int) { return one >= lowest; });
      });
      const bool fits = pack(to - warp * PART, moved_to, all);
      counts[0] = fits ? 0 : 1;             // (each lane's)
      __syncthreads();
      if (fits)
        for (int i = threadIdx.x; i < all; i += SL_THREADS) sums[1] += weight(of_key(key_of(list[i])));
      exchange(sums, counts);
      whole = sums[0];
      few = counts[0] == 0 && sums[1] >= (double)p * whole * (1.0 + 1e-12);
    }
  }
  if (few) {
    // ---- few candidates, it is likely
    const int found = listed();
    if (found <= SL_LIST) {
      int n = 0;
      if (rank == 0) n = gather(SL_LIST);
      cluster.sync();
      if (rank != 0) return;
      const Owned own(n);
      int ranks[SL_EACH], stay = by_count ? min(n, k) : n;
      Place* spare = reinterpret_cast<Place*>(held);      // (the slice has served)
      if (by_weight || stay < n) {
        ranks_of(all_listed, n, lowest, top, reinterpret_cast<unsigned*>(list), spare, s.warp_int, ranks);
      } else {
#pragma unroll
        for (int i = 0; i < SL_EACH; ++i) ranks[i] = 0;
      }
      double w[SL_EACH];
#pragma unroll
      for (int i = 0; i < SL_EACH; ++i)
        w[i] = own.has(i, n) && ranks[i] < stay ? weight(of_key(key_of(all_listed[own.first + i]))) : 0.0;
      if (by_weight) stay = cut_by_weight(w, ranks, n, stay, 0.0, (double)p * whole, whole > 0.0 ? 0.0 : (double)p, reinterpret_cast<double*>(spare));
      double sum = 0.0, all;
#pragma unroll
      for (int i = 0; i < SL_EACH; ++i) {
        w[i] = ranks[i] < stay ? w[i] : 0.0;
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
          last_kept = own.first + i;
          if (run > target && reached == 0x7fffffff) reached = own.first + i;
        }
      }
      if (reached != 0x7fffffff) atomicMin(&s.found[0], reached);
      if (last_kept >= 0) atomicMax(&s.found[1], last_kept);
      __syncthreads();
      if (threadIdx.x == 0) finish(index_of(all_listed[s.found[0] < n ? s.found[0] : s.found[1]]));
      return;
    }
    cluster.sync();            // the counts have been read
  }

  // ---- the cuts are found together
  int listed_stay = -1;            // what the last cut keeps of its interval, in the first CTA's list; -1: not there
  // The cut in [low, high], which holds `inside` kept keys, `above` before them; `ready`: they are in the lists already.
  auto cut_together = [&](bool weighed, unsigned low, unsigned high, double above, double target, int inside, bool ready) __attribute__((always_inline)) -> Cut {
    bool whole_interval = true;
    while (inside > SL_CUT && low < high) {
      ready = whole_interval = false;
      // the least and the largest key that it holds: few different ones lie in it where logits were rounded to 16 bits
      unsigned least_key = 0xffffffffu, most_key = 0u;
      auto within = [&](float x, int i, auto&& f) {
        const unsigned key = order_key(x);
        if (x == x && key >= low && key <= high && kept.keeps(x, begin + i)) f(key);
      };
      auto for_each = [&](auto&& f) {
        for_quads([&](int q, const float4& x) {
          const int i = 4 * q - shift;
          f(x.x, i), f(x.y, i + 1), f(x.z, i + 2), f(x.w, i + 3);
        });
      };
      for_each([&](float x, int i) {
        within(x, i, [&](unsigned key) { least_key = min(least_key, key); most_key = max(most_key, key); });
      });
      least_key = __reduce_min_sync(0xffffffffu, least_key);
      most_key = __reduce_max_sync(0xffffffffu, most_key);
      if (threadIdx.x == 0) { s.key_range[0] = 0xffffffffu; s.key_range[1] = 0u; }
      __syncthreads();
      if (lane == 0) { atomicMin(&s.key_range[0], least_key); atomicMax(&s.key_range[1], most_key); }
      cluster.sync();
      for (int c = 0; c < ranks; ++c) {
        const LimitShared* theirs = cluster.map_shared_rank(&s, c);
        least_key = min(least_key, theirs->key_range[0]);
        most_key = max(most_key, theirs->key_range[1]);
      }
      cluster.sync();
      low = max(low, least_key);
      high = min(high, most_key);
      if (low >= high) { low = high; break; }
      const unsigned step = (high - low) / SL_PARTS + 1;
      double sums[SL_PARTS];
      int counts[SL_PARTS];
#pragma unroll
      for (int j = 0; j < SL_PARTS; ++j) { sums[j] = 0.0; counts[j] = 0; }
      for_each([&](float x, int i) {
        within(x, i, [&](unsigned key) {
          const unsigned place = (high - key) / step;
          const double w = weighed ? weight(x) : 1.0;
#pragma unroll
          for (int j = 0; j < SL_PARTS; ++j)
            if (place == (unsigned)j) { sums[j] += w; counts[j] += 1; }
        });
      });
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
        // (-0, which no logit is, would take 0 along)
        collect(of_key(low), of_key(high == 0x7fffffffu ? high - 1u : high), kept);
        cluster.sync();
      }
      if (rank == 0) {
        const int n = gather(SL_CUT);
        const Owned own(n);
        Place* spare = all_listed + SL_CUT;
        int ranks[SL_EACH], stay = min(n, max(1, (int)(target - above)));
        ranks_of(all_listed, n, of_key(low), of_key(high), reinterpret_cast<unsigned*>(list), spare, s.warp_int, ranks);
        if (weighed) {
          double w[SL_EACH];
#pragma unroll
          for (int i = 0; i < SL_EACH; ++i) w[i] = own.has(i, n) ? weight(of_key(key_of(all_listed[own.first + i]))) : 0.0;
          stay = cut_by_weight(w, ranks, n, n, above, target, 0.0, reinterpret_cast<double*>(spare));
        }
        if (threadIdx.x == 0) {
          s.cut_listed = stay;
          if (n == 0) { s.cut_x = of_key(low); s.cut_index = 0x7fffffff; }
        }
        Place places[SL_EACH];
#pragma unroll
        for (int i = 0; i < SL_EACH; ++i)
          if (own.has(i, n)) places[i] = all_listed[own.first + i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < SL_EACH; ++i)
          if (own.has(i, n)) {
            all_listed[ranks[i]] = places[i];
            if (ranks[i] == stay - 1) {
              s.cut_x = of_key(key_of(places[i]));
              s.cut_index = index_of(places[i]);
            }
          }
      }
      cluster.sync();
      const LimitShared* first = cluster.map_shared_rank(&s, 0);
      const Cut cut{first->cut_x, first->cut_index};
      listed_stay = whole_interval ? first->cut_listed : -1;
      cluster.sync();
      return cut;
    }
    listed_stay = -1;
    // more equal keys than a CTA sorts: the index of the last one that stays, by counting
    const float low_x = of_key(low);
    const int stay = weighed ? ties_kept(above, weight(low_x), target, inside) : min(inside, max(1, (int)(target - above)));
    auto tie = [&](float x, int i) { return x == low_x && kept.keeps(x, begin + i); };
    int here = 0;
    for_high(low_x, [&](float x, int i) { here += tie(x, i); });
    here = (int)__reduce_add_sync(0xffffffffu, (unsigned)here);
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
    if (place < stay && stay <= place + here)      // this warp's, which looks again, in the order of the vocabulary
      for (int base = quad_begin; base < quad_end; base += 32 * SL_AHEAD) {
        float4 v[SL_AHEAD];
        quads_of.get(base + lane, quad_end, v);
#pragma unroll
        for (int j = 0; j < SL_AHEAD; ++j) {
          const int i = 4 * (base + 32 * j + lane) - shift;
          const bool in[4] = {tie(v[j].x, i), tie(v[j].y, i + 1), tie(v[j].z, i + 2), tie(v[j].w, i + 3)};
          int before = place;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const unsigned mask = __ballot_sync(0xffffffffu, in[e]);
            before += __popc(mask & ((1u << lane) - 1u));
            place += __popc(mask);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            before += in[e];
            if (in[e] && before == stay) s.cut_index = begin + i + e;
          }
        }
      }
    cluster.sync();
    Cut cut{low_x, 0x7fffffff};
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
    // (with 2^23 added without rounding up, the whole number stands in the low bits; NaN from infinities goes to the last bin)
    auto count_one = [&](float x) {
      const unsigned bin = __float_as_uint(__fadd_rz(fminf((top - x) * bin_scale, (float)(SL_BINS - 1)), 8388608.f)) & (2 * SL_BINS - 1);
      if (x == x) atomicAdd(&bins[bin], 1u);
    };
    for_quads([&](int, const float4& x) { count_one(x.x), count_one(x.y), count_one(x.z), count_one(x.w); });
    add_up_bins();
  }
  // a logit that surely lies below a bin's beginning
  auto below_bin = [&](float bin) { return bin >= (float)(SL_BINS - 1) ? -INFINITY : cleaned(top - bin / bin_scale); };
  double certain = 0.0;            // of this warp's stretch: weights that stay whatever the cut of the weights
  float open_low = -INFINITY, open_high = top;      // logits that it lies among
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
    const float low = below_bin((float)bin + 1.01f), high = bin == 0 ? top : below_bin((float)bin - 0.01f);
    // every logit counts, min-p or not: the smaller of the two beginnings stays
    const Cut before_k = kept;
    kept = everything;
    double sums[2] = {};
    int counts[2] = {};
    empty_list();
    for_high(low, [&](float x, int i) {
      if (x > high) {
        counts[0] += 1;
      } else {
        counts[1] += 1;
        append(x, i);
      }
    });
    exchange(sums, counts);
    const bool holds = counts[0] < k && counts[0] + counts[1] >= k;
    const Cut cut = cut_together(false, holds ? order_key(low) : no_key, holds ? order_key(high) : top_key, holds ? (double)counts[0] : 0.0,
                                 (double)k, holds ? counts[1] : vocab, holds);
    kept = before_k;
    kept.tighten(cut);
  }
  if (by_weight) {
    // Weights taken in the middle of their bins: the bins where they come to p of theirs, and to a little less and more.  What the
    // estimate is off (single large tokens) shows in the exact sums above an interval; with that known the next one is found.
    float mass[SL_BINS_PER_THREAD], here = 0.f, all, until;
    int tokens_here = 0, tokens_all, tokens_until;
    const int last_bin = (int)fminf((top - kept.x) * bin_scale, (float)(SL_BINS - 1));
#pragma unroll
    for (int j = 0; j < SL_BINS_PER_THREAD; ++j) {
      mass[j] = count[j] > 0 && first_bin + j <= last_bin ? (float)count[j] * expf(-((float)(first_bin + j) + 0.5f) / SL_BINS_PER_T) : 0.f;
      here += mass[j];
      tokens_here += count[j];
    }
    const float before = before_block(here, s.warp_float, &all, &until);
    const int tokens_before = before_block(tokens_here, s.warp_int, &tokens_all, &tokens_until);
    float wanted = p * all;
    double above = 0.0;
    int inside = vocab;
    bool found = false;
    whole = 0.0;
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
        open_low = below_bin((float)s.mark_bin[2] + 1.01f);
        open_high = s.mark_bin[0] == 0 ? top : below_bin((float)s.mark_bin[0] - 0.01f);
        estimate = s.mark_mass[0];
      } else {
        open_low = below_bin((float)s.mark_bin[1] + 1.25f);
        open_high = s.mark_bin[1] == 0 ? top : below_bin((float)s.mark_bin[1] - 0.25f);
        estimate = s.mark_mass[1];
      }
      empty_list();
      double sums[3] = {};                   // above the interval, in it, all
      int counts[3] = {};
      const bool limited = kept.x > -INFINITY;
      for_quads([&](int q, float4 x) {
        const int i = 4 * q - shift;
        if (limited) {
          x.x = kept.keeps(x.x, begin + i) ? x.x : NOTHING;
          x.y = kept.keeps(x.y, begin + i + 1) ? x.y : NOTHING;
          x.z = kept.keeps(x.z, begin + i + 2) ? x.z : NOTHING;
          x.w = kept.keeps(x.w, begin + i + 3) ? x.w : NOTHING;
        }
        const double w[4] = {weight(x.x), weight(x.y), weight(x.z), weight(x.w)};
        sums[2] += (w[0] + w[1]) + (w[2] + w[3]);
        sums[0] += ((x.x > open_high ? w[0] : 0.0) + (x.y > open_high ? w[1] : 0.0)) + ((x.z > open_high ? w[2] : 0.0) + (x.w > open_high ? w[3] : 0.0));
        auto in = [&](float one) { return one >= open_low && one <= open_high; };
        if (in(x.x) || in(x.y) || in(x.z) || in(x.w)) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float one = j == 0 ? x.x : j == 1 ? x.y : j == 2 ? x.z : x.w;
            if (in(one)) {
              sums[1] += w[j];
              counts[1] += 1;
              append(one, i + j);
            }
          }
        }
      });
      certain = warp_sum64(sums[0]);
      exchange(sums, counts);
      whole = sums[2];
      const double target = (double)p * whole;
      found = sums[0] < target && (sums[0] + sums[1] >= target || open_low == -INFINITY);
      above = found ? sums[0] : 0.0;
      inside = found ? counts[1] : vocab;
      wanted = (float)(target - sums[0]) + estimate;
    }
    summed = found;
    kept.tighten(cut_together(true, found ? order_key(open_low) : no_key, found ? order_key(open_high) : top_key, above, (double)p * whole, inside,
                              found));
  }

  // ---- the draw
  double sum = 0.0;
  const int chunk = max(128, ((per_warp + 31) / 32 + 31) / 32 * 32);      // quads: a warp sums its stretch by at most 32 chunks
  if (summed && listed_stay >= 0) {
    // the interval's tokens that stay, from the first CTA's list: those of this warp's stretch
    const Place* theirs = cluster.map_shared_rank(all_listed, 0);
    for (int i = threadIdx.x; i < listed_stay; i += SL_THREADS) list[i] = theirs[i];
    __syncthreads();
    const int low = begin + max(0, 4 * quad_begin - shift), high = begin + min(size, max(0, 4 * quad_end - shift));
    for (int i = lane; i < listed_stay; i += 32) {
      const Place place = list[i];
      if (index_of(place) >= low && index_of(place) < high) sum += weight(of_key(key_of(place)));
    }
  } else if (summed) {
    for_high(kept.x, [&](float x, int i) { if (x <= open_high && kept.keeps(x, begin + i)) sum += weight(x); });
  } else {
    double in_chunk = 0.0;
    int rows_left = chunk / 32, at_chunk = 0;
    for_quads([&](int q, const float4& x) {
      const int i = begin + 4 * q - shift;
      double w[4] = {weight(x.x), weight(x.y), weight(x.z), weight(x.w)};
      if (kept.x > -INFINITY) {
        w[0] = kept.keeps(x.x, i) ? w[0] : 0.0;
        w[1] = kept.keeps(x.y, i + 1) ? w[1] : 0.0;
        w[2] = kept.keeps(x.z, i + 2) ? w[2] : 0.0;
        w[3] = kept.keeps(x.w, i + 3) ? w[3] : 0.0;
      }
      in_chunk += (w[0] + w[1]) + (w[2] + w[3]);
      if (--rows_left == 0 || q - lane + 32 >= quad_end) {
        in_chunk = warp_sum64(in_chunk);
        if (lane == 0) { chunks[warp][at_chunk] = in_chunk; sum += in_chunk; }
        in_chunk = 0.0;
        rows_left = chunk / 32;
        ++at_chunk;
      }
    });
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
    auto chosen_of = [&](const double* sums, int count, double& so_far) {
      int last = 0, chosen = -1;
      for (int w = 0; w < count; ++w)
        if (sums[w] > 0.0) last = w;
      for (int w = 0; w < count && chosen < 0; ++w) {
        if (sums[w] > 0.0 && (target < so_far + sums[w] || w == last)) chosen = w;
        else so_far += sums[w];
      }
      return max(chosen, 0);
    };
    const int stretch = chosen_of(s.warp_double, SL_WARPS, run);
    int part_begin = min(quads, stretch * per_warp), part_end = min(quads, part_begin + per_warp);
    if (!summed) {
      part_begin = min(part_end, part_begin + chunk * chosen_of(chunks[stretch], (part_end - part_begin + chunk - 1) / chunk, run));
      part_end = min(part_end, part_begin + chunk);
    }
    auto weights_of = [&](int q, const float4& x, double (&w)[4]) {
      const int i = begin + 4 * q - shift;
      w[0] = kept.keeps(x.x, i) ? weight(x.x) : 0.0;
      w[1] = kept.keeps(x.y, i + 1) ? weight(x.y) : 0.0;
      w[2] = kept.keeps(x.z, i + 2) ? weight(x.z) : 0.0;
      w[3] = kept.keeps(x.w, i + 3) ? weight(x.w) : 0.0;
    };
    constexpr int AHEAD = 4;
    while (part_end - part_begin > 32 * SL_WARPS) {
      const int each = (part_end - part_begin + SL_WARPS - 1) / SL_WARPS;
      const int my_begin = min(part_end, part_begin + warp * each), my_end = min(part_end, my_begin + each);
      double in_part = 0.0;
      float4 ahead[AHEAD];
      quads_of.get(my_begin + lane, my_end, ahead);
#pragma unroll 1
      for (int base = my_begin; base < my_end; base += 32) {
        const float4 x = ahead[0];
        float4 next[1];
#pragma unroll
        for (int j = 0; j + 1 < AHEAD; ++j) ahead[j] = ahead[j + 1];
        quads_of.get(base + 32 * AHEAD + lane, my_end, next);
        ahead[AHEAD - 1] = next[0];
        double w[4];
        weights_of(base + lane, x, w);
        in_part += (w[0] + w[1]) + (w[2] + w[3]);
      }
      in_part = warp_sum64(in_part);
      __syncthreads();
      if (lane == 0) s.warp_double[warp] = in_part;
      __syncthreads();
      part_begin = min(part_end, part_begin + chosen_of(s.warp_double, SL_WARPS, run) * each);
      part_end = min(part_end, part_begin + each);
    }
    // a quad per thread: the warp, then its quad and the logit
    const int q = part_begin + (int)threadIdx.x, i = 4 * q - shift;
    float4 x[1];
    quads_of.get(q, part_end, x);
    double w[4];
    weights_of(q, x[0], w);
    const double until[4] = {w[0], w[0] + w[1], (w[0] + w[1]) + w[2], ((w[0] + w[1]) + w[2]) + w[3]};
    double inclusive = until[3];
#pragma unroll
    for (int offset = 1; offset < 32; offset <<= 1) {
      const double up = __shfl_up_sync(0xffffffffu, inclusive, offset);
      if (lane >= offset) inclusive += up;
    }
    __syncthreads();
    if (lane == 31) s.warp_double[warp] = inclusive;
    __syncthreads();
    if (warp == chosen_of(s.warp_double, SL_WARPS, run)) {
      const double up = __shfl_up_sync(0xffffffffu, inclusive, 1), before = run + (lane > 0 ? up : 0.0);
      int found = -1, last_kept = -1;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (w[e] > 0.0) {
          last_kept = i + e;
          if (found < 0 && before + until[e] > target) found = i + e;
        }
      const unsigned some = __ballot_sync(0xffffffffu, last_kept >= 0), hit = __ballot_sync(0xffffffffu, found >= 0);
      // what rounding leaves behind the last belongs to it
      const int token = hit != 0u ? __shfl_sync(0xffffffffu, found, __ffs(hit) - 1)
                                  : __shfl_sync(0xffffffffu, last_kept, some != 0u ? 31 - __clz(some) : 0);
      if (lane == 0) finish(begin + max(0, token));
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
  if ((long long)rows * SL_MOST_RANKS > 0x7fffffffLL || vocab > 1 << 30) return MLR_TOO_LARGE;
  const LimitSource source{uniforms, temperatures, top_k, top_p, min_p, row_slot, (SlotState*)state, slots, advance};
  // CTAs per row: eight or fewer of at least 2,048 logits while the device holds them at once, two to an SM (a tenth of the SMs lies in no group
  // that holds a cluster of eight); up to four of 4,096 in any case, as a row of top-p alone has work for them.  256 rows of 152,064 logits
  // under various limits: 217 us with one each, 145 with two, 119 with four, 138 with eight, in the order they come in; 256 of 8,000: 42, 45, 67, 91; 33 of
  // 152,064: 84, 54, 34, 30.
  constexpr int LEAST = 2048, USUAL = 4096;
  int ranks = 1;
  while (ranks < SL_MOST_RANKS && ((ranks < 4 && vocab > 2 * ranks * USUAL) || (vocab > ranks * LEAST && (long long)rows * ranks * 2 <= 2LL * sm_count() * 9 / 10)))
    ranks *= 2;
  const int slice = ((vocab + ranks - 1) / ranks + 3) / 4 * 4, quads = slice / 4 + 1;
  const int blocks = (quads_of_warp(quads) + 32 * SL_AHEAD - 1) / (32 * SL_AHEAD), num_tops = blocks < SL_TOPS ? blocks : SL_TOPS;
  const int rest = (int)(SL_LIST * sizeof(Place) + SL_BINS * sizeof(unsigned) + SL_BINS / ranks * sizeof(unsigned)) + num_tops * SL_THREADS * 4;
  // The slice stays in shared memory where two CTAs of an SM, or one on an SM of its own, hold theirs; else it is read again, from the L2 cache
  // as far as that goes.
  constexpr int TWO = 111 * 1024, ONE = 220 * 1024;
  const bool resident = (long long)quads * 16 + rest <= ((long long)rows * ranks <= sm_count() ? ONE : TWO);
  const int room = max(resident ? quads * 16 : 0, (int)(SL_LIST * sizeof(Place)));
  static OncePerDevice once;
  const cudaError_t err = once([&] {
    const cudaError_t e = cudaFuncSetAttribute(sample_limited_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, ONE);
    return e == cudaSuccess ? cudaFuncSetAttribute(sample_limited_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, ONE) : e;
  });
  if (err != cudaSuccess) return (int)err;
  // Rows that take longest first, where not all are taken at once: 256 rows of 152,064 logits under various limits, three drawings, caches flushed,
  // 111, 113 and 127 us, so 131, 135 and 144 without; all rows under the same limits lose by it, as each CTA looks at all rows' limits: greedy 64, so
  // 57, top-k 50 88, so 84, none 138, so 135.  Short slices gain nothing: 256 rows of 32,000 72, so 72.
  constexpr int LONG_SLICE = 16384;
  const bool ordered = (long long)rows * ranks > 2 * sm_count() && rows <= SL_ORDERED && slice >= LONG_SLICE;
  auto kernel = resident ? sample_limited_kernel<true> : sample_limited_kernel<false>;
  launch_kernel_clustered(kernel, dim3(rows * ranks), dim3(SL_THREADS), room + rest, stream, ranks, logits, source, tokens, vocab, slice, room,
                          ordered ? rows : 0);
  return launch_status();
}
