// The rules of a request on its logits, applied before a token is chosen, and the history that they look at.
//
// Of row r, whose request owns slot s, and token t, in this order:
//   known[s][t]          x = x > 0 ? x / repetition[s] : x * repetition[s]
//   n = generated[s][t]  x = x - frequency[s] * n, and x = x - presence[s] if n > 0
//   bias of t in s       x = x + bias (a token listed several times: with the sum)
//   not allowed[s][t]    x = -infinity
// all in float32.  The tables are indexed by slot and stay on the device, like the slot records: a captured step finds
// whatever requests its rows belong to.  A row whose slot is outside the tables passes unchanged.
//
// History.  One word per slot and token: bit 30 says that the token is in the prompt, the bits below it how often it was
// generated.  Beside it a plane of bits, one per word that is not zero.  A row has some thousand known tokens among
// 152,000, so this kernel reads the plane (19 KB) instead of the words (608 KB) and fetches a word where its bit is set.
//
// What it has to move: 8.25 bytes per logit (read, write, two bits) out of place; in place the bits and the few logits that change.  Out of
// place it comes within a quarter of a copy; in place it takes as long (64 x 152,064 18.0 us in a row of captured calls, apart 19.4; 256 x
// 151,936 68.0 and 67.8): the chains of reads and the issue of instructions per piece (2.3 a cycle), not bytes, are its limit.
#include "common.cuh"

namespace mlr {

constexpr int RULE_THREADS = 256;
constexpr int IN_PROMPT = 1 << 30;

struct RuleTables {
  const float* penalties;      // [slots][3]: repetition, presence, frequency; null: none
  const int* counts;           // [slots][vocab], with `penalties`
  const unsigned* seen;        // [slots][words], with `penalties`; bits behind the vocabulary say nothing
  const int* bias_tokens;      // [slots][biases], ascending, the unused end 2^31 - 1; null: none
  const float* bias_values;    // [slots][biases]
  const unsigned* allowed;     // [slots][words]; null: everything
  int biases, slots;
};

// Four bits of a plane from token t0 on: t0 a multiple of four, or any with WHOLE false (bits past the last word are zero).
template <bool WHOLE>
__device__ __forceinline__ unsigned four_bits(const unsigned* plane, int t0, int words) {
  if (WHOLE) return (unsigned)__ldcg(reinterpret_cast<const unsigned char*>(plane) + (t0 >> 3)) >> (t0 & 4) & 15u;
  const int at = t0 >> 5, shift = t0 & 31;
  unsigned bits = __ldcg(plane + at) >> shift;
  if (shift > 28 && at + 1 < words) bits |= __ldcg(plane + at + 1) << (32 - shift);
  return bits & 15u;
}

// Without branches: every second warp has a known token among its 128.  x / repetition is x times the reciprocal, which is rounded
// once per row: up to a second half step of float32 (2^-24).  With a division for each entry 64 x 152,064 takes 24.4 us instead of 23.0, 256 x
// 151,936 74.9 instead of 68.0.
__device__ __forceinline__ float penalised(float x, int word, float repetition, float reciprocal, float presence, float frequency) {
  const int made = word & (IN_PROMPT - 1);
  x *= x > 0.f ? reciprocal : repetition;
  x = fmaf(-frequency, (float)made, x);
  return made > 0 ? x - presence : x;
}

// A CTA takes a stretch of one row, 256 pieces of four logits (a portion) at a time.  What a token may need hangs together (slot, then
// bits, then the words of known tokens), so three portions are under way: the bits of the one after next, the logits and words of the
// next, the arithmetic of the present one.  (A CTA per portion lives through that chain, 4 us, for 16 KB: 64 x 152,064 logits 36 us, 256 x
// 151,936 94 us; as it stands 23 and 68, 4.75 TB/s, where a copy of the same logits takes 18.5 and 55 and the bytes alone 12.6 and 50. Few
// rows are latency: a row of 151,936 2.3 us in a row of captured calls, 8 from the host.)
// Pieces lie on 16-byte boundaries.  WHOLE: the vocabulary is a multiple of four, every piece is one row's, and so are the words of the
// history, which start on such a boundary too; else a row starts inside a piece, its first and last piece go entry by entry, and the words
// of a slot whose row of them starts on another boundary as well.
// IN_PLACE: logits that no rule touches are neither read nor written.
template <bool IN_PLACE, bool WHOLE>
__global__ void __launch_bounds__(RULE_THREADS)
logit_rules_kernel(const float* logits, float* out, const int* row_slot, int vocab, int stretch, const RuleTables tables) {
  constexpr int PORTION = RULE_THREADS * 4;
  pdl_trigger();
  pdl_wait();
  const int row = blockIdx.y;
  const size_t base = (size_t)row * vocab;
  const int lead = WHOLE ? 0 : (int)(base & 3);      // entries of the row's first piece that belong to the row before
  const int words = (vocab + 31) >> 5;
  const float* in = logits + base;
  float* to = out + base;
  const int first = blockIdx.x * stretch - lead;     // first token of this CTA's pieces; may be negative in the first CTA
  const int end = min(vocab, first + stretch);
  int t0 = first + (int)threadIdx.x * 4;             // first token of this thread's present piece

  auto mine = [&](int t) { return (WHOLE || t > -4) && t < end; };
  auto inside = [&](int t) { return WHOLE || (t >= 0 && t + 4 <= vocab); };
  float value[4], ahead[4];
  auto load_values = [&](int t, float* v) {
    if (!mine(t)) return;
    if (inside(t)) {
      const float4 four = *reinterpret_cast<const float4*>(in + t);
      v[0] = four.x; v[1] = four.y; v[2] = four.z; v[3] = four.w;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = t + e >= 0 && t + e < vocab ? in[t + e] : 0.f;
    }
  };
  if (!IN_PLACE) load_values(t0, value);             // needs no slot

  const int slot = __ldcg(row_slot + row);
  const bool ruled = slot >= 0 && slot < tables.slots;
  const unsigned* seen = ruled && tables.penalties != nullptr ? tables.seen + (size_t)slot * words : nullptr;
  const unsigned* allowed = ruled && tables.allowed != nullptr ? tables.allowed + (size_t)slot * words : nullptr;
  const int* counts = seen != nullptr ? tables.counts + (size_t)slot * vocab : nullptr;
  const int biases = ruled && tables.bias_tokens != nullptr ? tables.biases : 0;
  const int* bias_tokens = tables.bias_tokens + (size_t)(biases > 0 ? slot : 0) * tables.biases;

  // bits 0..3: known and allowed; bits 4..7: not allowed
  auto load_bits = [&](int t) {
    if (!mine(t)) return 0u;
    const int shift = !WHOLE && t < 0 ? -t : 0;
    unsigned known = 0u, open = 15u;
    if (seen != nullptr) known = four_bits<WHOLE>(seen, t + shift, words) << shift & 15u;
    if (!WHOLE && t + 4 > vocab) known &= (1u << (vocab - t)) - 1u;      // behind the vocabulary there are no words
    if (allowed != nullptr) open = (four_bits<WHOLE>(allowed, t + shift, words) << shift & 15u) | ((1u << shift) - 1u);
    return (known & open) | (open ^ 15u) << 4;
  };
  const bool aligned = WHOLE || ((uintptr_t)(counts + first) & 15) == 0;      // the slot's words, piece by piece
  int word[4], word_ahead[4];
  auto load_words = [&](int t, unsigned bits, int* w, float* v) {
    if ((bits & 15u) == 0u) return;
    if (WHOLE || (aligned && inside(t))) {
      const int4 four = __ldcg(reinterpret_cast<const int4*>(counts + t));
      w[0] = four.x; w[1] = four.y; w[2] = four.z; w[3] = four.w;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (bits >> e & 1u) w[e] = __ldcg(counts + t + e);
    }
    if (IN_PLACE) load_values(t, v);
  };
  unsigned bits = load_bits(t0), bits_ahead = load_bits(t0 + PORTION);
  const int bias_token = (int)threadIdx.x < biases ? __ldcg(bias_tokens + threadIdx.x) : -1;
  float repetition = 1.f, presence = 0.f, frequency = 0.f;
  if (seen != nullptr) {
    repetition = __ldcg(tables.penalties + 3 * (size_t)slot);
    presence = __ldcg(tables.penalties + 3 * (size_t)slot + 1);
    frequency = __ldcg(tables.penalties + 3 * (size_t)slot + 2);
  }
  load_words(t0, bits, word, value);
  const float reciprocal = 1.f / repetition;

  for (int from = first; from < end; from += PORTION, t0 += PORTION) {
    if (!IN_PLACE) load_values(t0 + PORTION, ahead);
    load_words(t0 + PORTION, bits_ahead, word_ahead, ahead);
    const unsigned bits_after = load_bits(t0 + 2 * PORTION);
    if (mine(t0)) {
      if ((bits & 15u) != 0u) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float y = penalised(value[e], word[e], repetition, reciprocal, presence, frequency);
          value[e] = bits >> e & 1u ? y : value[e];
        }
      }
      if (bits >> 4 != 0u) {
#pragma unroll
        for (int e = 0; e < 4; ++e) value[e] = bits >> (4 + e) & 1u ? -INFINITY : value[e];
      }
      if (!IN_PLACE && inside(t0)) {
        *reinterpret_cast<float4*>(to + t0) = make_float4(value[0], value[1], value[2], value[3]);
      } else {
        const unsigned write = IN_PLACE ? (bits | bits >> 4) & 15u : 15u;
        if (IN_PLACE && write == 15u && inside(t0)) {
          *reinterpret_cast<float4*>(to + t0) = make_float4(value[0], value[1], value[2], value[3]);
        } else if (write != 0u) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if ((write >> e & 1u) != 0u && (WHOLE || (t0 + e >= 0 && t0 + e < vocab))) to[t0 + e] = value[e];
        }
      }
    }
    bits = bits_ahead;
    bits_ahead = bits_after;
#pragma unroll
    for (int e = 0; e < 4; ++e) { value[e] = ahead[e]; word[e] = word_ahead[e]; }
  }

  // Biases of this CTA's tokens, by the thread that holds the first entry of a token: after the stores above.
  if (biases == 0) return;
  __syncthreads();
  const float* values = tables.bias_values + (size_t)slot * biases;
  for (int i = threadIdx.x; i < biases; i += RULE_THREADS) {
    const int t = i < RULE_THREADS ? bias_token : __ldcg(bias_tokens + i);
    if (t < max(0, first) || t >= end || (i > 0 && __ldcg(bias_tokens + i - 1) == t)) continue;
    if (allowed != nullptr && (__ldcg(allowed + (t >> 5)) >> (t & 31) & 1u) == 0u) continue;
    float sum = __ldcg(values + i);
    for (int j = i + 1; j < biases && __ldcg(bias_tokens + j) == t; ++j) sum += __ldcg(values + j);
    to[t] += sum;
  }
}

// One thread per (slot, token) pair; sums of whole numbers: the order of the atomics changes nothing.  Bound by its launch: 64 pairs 0.9 us, 4,000
// 1.2, calls one behind the other.
__global__ void count_tokens_kernel(const int* tokens, const int* slots, int pairs, int* counts, unsigned* seen, int num_slots,
                                    int vocab, int prompt) {
  pdl_trigger();
  pdl_wait();
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= pairs) return;
  const int token = __ldcg(tokens + i), slot = __ldcg(slots + i);
  if (token < 0 || token >= vocab || slot < 0 || slot >= num_slots) return;
  int* word = counts + (size_t)slot * vocab + token;
  if (prompt) atomicOr(word, IN_PROMPT);
  else atomicAdd(word, 1);
  atomicOr(seen + (size_t)slot * ((vocab + 31) >> 5) + (token >> 5), 1u << (token & 31));
}

static void launch_rules(const float* logits, float* out, const int* row_slot, int rows, int vocab, const RuleTables& tables,
                         cudaStream_t stream) {
  // Up to four portions per CTA, as far as every SM still has eight CTAs (64 x 152,064 and 256 x 151,936 logits with one portion
  // each 36 and 94 us, with two 25 and 71, with four 23 and 68, with eight 25 and 70, with sixteen 24 and 72).
  constexpr int PORTION = RULE_THREADS * 4;
  const int portions = (vocab + 3 + PORTION - 1) / PORTION;
  const int each = (int)min(4ll, 1 + (long long)rows * portions / (8 * sm_count()));
  const dim3 grid((portions + each - 1) / each, rows);
  const bool whole = (vocab & 3) == 0 && ((uintptr_t)tables.counts & 15) == 0;
  auto kernel = logits == out ? (whole ? logit_rules_kernel<true, true> : logit_rules_kernel<true, false>)
                              : (whole ? logit_rules_kernel<false, true> : logit_rules_kernel<false, false>);
  launch_kernel(kernel, grid, dim3(RULE_THREADS), 0, stream, logits, out, row_slot, vocab, each * PORTION, tables);
}

}  // namespace mlr

using namespace mlr;

MLR_DEFINE_PDL_SWITCH

// logits, out: float32 [rows, vocab] on 16-byte boundaries, the same memory or apart.  row_slot: int32 [rows].  `tables` is read on
// the host.
MLR_EXPORT int mlr_logit_rules(const float* logits, float* out, const int* row_slot, int rows, int vocab, const RuleTables* tables,
                               cudaStream_t stream) {
  if (tables == nullptr || rows < 0 || vocab <= 0 || vocab > (1 << 30) || tables->slots <= 0 || tables->biases < 0) return MLR_BAD_SIZE;
  if (rows == 0) return MLR_OK;
  if (rows > 65535) return MLR_TOO_LARGE;
  if (((uintptr_t)logits & 15) != 0 || ((uintptr_t)out & 15) != 0) return MLR_BAD_ALIGNMENT;
  RuleTables t = *tables;
  if ((t.penalties != nullptr) != (t.counts != nullptr) || (t.penalties != nullptr) != (t.seen != nullptr)) return MLR_BAD_SIZE;
  if (t.biases == 0) t.bias_tokens = nullptr;
  launch_rules(logits, out, row_slot, rows, vocab, t, stream);
  return launch_status();
}

// tokens, slots: int32 [pairs].  `prompt`: mark them as tokens of the prompt instead of counting them.
MLR_EXPORT int mlr_count_tokens(const int* tokens, const int* slots, int pairs, int* counts, void* seen, int num_slots, int vocab,
                                int prompt, cudaStream_t stream) {
  if (pairs < 0 || vocab <= 0 || num_slots <= 0) return MLR_BAD_SIZE;
  if (pairs == 0) return MLR_OK;
  launch_kernel(count_tokens_kernel, dim3((pairs + 127) / 128), dim3(128), 0, stream, tokens, slots, pairs, counts, (unsigned*)seen,
                num_slots, vocab, prompt);
  return launch_status();
}
