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
// Bound by memory: 8.25 bytes per logit (read, write, two bits) out of place; in place the bits and the few logits
// that change.
#include "common.cuh"

namespace mlr {

constexpr int RULE_THREADS = 256;
constexpr int IN_PROMPT = 1 << 30;

struct RuleTables {
  const float* penalties;      // [slots][3]: repetition, presence, frequency; null: none
  const int* counts;           // [slots][vocab], with `penalties`
  const unsigned* seen;        // [slots][words], with `penalties`
  const int* bias_tokens;      // [slots][biases], ascending, the unused end 2^31 - 1; null: none
  const float* bias_values;    // [slots][biases]
  const unsigned* allowed;     // [slots][words]; null: everything
  int biases, slots;
};

// Four bits of a plane from token t0 >= 0 on (bits past the last word are zero).
__device__ __forceinline__ unsigned four_bits(const unsigned* plane, int t0, int words) {
  const int at = t0 >> 5, shift = t0 & 31;
  unsigned bits = __ldcg(plane + at) >> shift;
  if (shift > 28 && at + 1 < words) bits |= __ldcg(plane + at + 1) << (32 - shift);
  return bits & 15u;
}

__device__ __forceinline__ float penalised(float x, int word, float repetition, float presence, float frequency) {
  x = x > 0.f ? x / repetition : x * repetition;
  const int made = word & (IN_PROMPT - 1);
  if (made > 0) x = __fsub_rn(__fsub_rn(x, __fmul_rn(frequency, (float)made)), presence);
  return x;
}

// A CTA takes PIECES * 256 pieces of four logits of one row.  Pieces lie on 16-byte boundaries (the vocabulary need not be
// a multiple of four: a row then starts inside a piece, and its first and last piece go entry by entry).
// IN_PLACE: logits that no rule touches are neither read nor written.
template <int PIECES, bool IN_PLACE>
__global__ void __launch_bounds__(RULE_THREADS)
logit_rules_kernel(const float* logits, float* out, const int* row_slot, int vocab, const RuleTables tables) {
  pdl_trigger();
  pdl_wait();
  const int row = blockIdx.y;
  const size_t base = (size_t)row * vocab;
  const int lead = (int)(base & 3);                  // entries of the row's first piece that belong to the row before
  const int words = (vocab + 31) >> 5;
  const int slot = __ldcg(row_slot + row);
  const bool ruled = slot >= 0 && slot < tables.slots;
  const float* in = logits + base;
  float* to = out + base;
  const unsigned* seen = ruled && tables.penalties != nullptr ? tables.seen + (size_t)slot * words : nullptr;
  const unsigned* allowed = ruled && tables.allowed != nullptr ? tables.allowed + (size_t)slot * words : nullptr;
  const int* counts = seen != nullptr ? tables.counts + (size_t)slot * vocab : nullptr;
  const int first = blockIdx.x * (PIECES * RULE_THREADS * 4) - lead;      // first token of this CTA's pieces

  float4 value[PIECES];
  unsigned known[PIECES], open[PIECES];
#pragma unroll
  for (int p = 0; p < PIECES; ++p) {
    const int t0 = first + (p * RULE_THREADS + (int)threadIdx.x) * 4;
    known[p] = 0u;
    open[p] = 15u;
    if (t0 <= -4 || t0 >= vocab) continue;
    const bool whole = t0 >= 0 && t0 + 4 <= vocab;
    const int shift = t0 < 0 ? -t0 : 0;
    if (seen != nullptr) known[p] = four_bits(seen, t0 + shift, words) << shift & 15u;
    if (allowed != nullptr) open[p] = (four_bits(allowed, t0 + shift, words) << shift & 15u) | ((1u << shift) - 1u);
    if (!IN_PLACE) {
      if (whole) {
        value[p] = __ldcs(reinterpret_cast<const float4*>(in + t0));
      } else {
        float* v = reinterpret_cast<float*>(&value[p]);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = t0 + e >= 0 && t0 + e < vocab ? in[t0 + e] : 0.f;
      }
    }
  }
  float repetition = 1.f, presence = 0.f, frequency = 0.f;
  if (seen != nullptr) {
    repetition = __ldcg(tables.penalties + 3 * (size_t)slot);
    presence = __ldcg(tables.penalties + 3 * (size_t)slot + 1);
    frequency = __ldcg(tables.penalties + 3 * (size_t)slot + 2);
  }
#pragma unroll
  for (int p = 0; p < PIECES; ++p) {
    const int t0 = first + (p * RULE_THREADS + (int)threadIdx.x) * 4;
    if (t0 <= -4 || t0 >= vocab) continue;
    const bool whole = t0 >= 0 && t0 + 4 <= vocab;
    float* v = reinterpret_cast<float*>(&value[p]);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int t = t0 + e;
      if (t < 0 || t >= vocab) continue;
      const bool touched = (known[p] >> e & 1u) != 0u || (open[p] >> e & 1u) == 0u;
      if (IN_PLACE && !touched) continue;
      if ((open[p] >> e & 1u) == 0u) {
        v[e] = -INFINITY;
      } else {
        if (IN_PLACE) v[e] = in[t];
        if (known[p] >> e & 1u) v[e] = penalised(v[e], __ldcg(counts + t), repetition, presence, frequency);
      }
      if (IN_PLACE || !whole) to[t] = v[e];
    }
    if (!IN_PLACE && whole) *reinterpret_cast<float4*>(to + t0) = value[p];
  }

  // Biases of this CTA's tokens, by the thread that holds the first entry of a token: after the stores above.
  if (!ruled || tables.bias_tokens == nullptr) return;
  __syncthreads();
  const int low = max(0, first), high = min(vocab, first + PIECES * RULE_THREADS * 4);
  const int* tokens = tables.bias_tokens + (size_t)slot * tables.biases;
  const float* values = tables.bias_values + (size_t)slot * tables.biases;
  for (int i = threadIdx.x; i < tables.biases; i += RULE_THREADS) {
    const int t = __ldcg(tokens + i);
    if (t < low || t >= high || (i > 0 && __ldcg(tokens + i - 1) == t)) continue;
    if (allowed != nullptr && (__ldcg(allowed + (t >> 5)) >> (t & 31) & 1u) == 0u) continue;
    float sum = __ldcg(values + i);
    for (int j = i + 1; j < tables.biases && __ldcg(tokens + j) == t; ++j) sum += __ldcg(values + j);
    to[t] += sum;
  }
}

// One thread per (slot, token) pair.  Sums of whole numbers: the order of the atomics changes nothing.
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

template <int PIECES>
static void launch_rules(const float* logits, float* out, const int* row_slot, int rows, int vocab, const RuleTables& tables,
                         cudaStream_t stream) {
  const dim3 grid((vocab + 3 + PIECES * RULE_THREADS * 4 - 1) / (PIECES * RULE_THREADS * 4), rows);
  if (logits == out)
    launch_kernel(logit_rules_kernel<PIECES, true>, grid, dim3(RULE_THREADS), 0, stream, logits, out, row_slot, vocab, tables);
  else
    launch_kernel(logit_rules_kernel<PIECES, false>, grid, dim3(RULE_THREADS), 0, stream, logits, out, row_slot, vocab, tables);
}

}  // namespace mlr

using namespace mlr;

MLR_DEFINE_PDL_SWITCH

// logits, out: float32 [rows, vocab] on 16-byte boundaries, the same memory or apart.  row_slot: int32 [rows].
MLR_EXPORT int mlr_logit_rules(const float* logits, float* out, const int* row_slot, int rows, int vocab, int slots,
                               const float* penalties, const int* counts, const void* seen, const int* bias_tokens,
                               const float* bias_values, int biases, const void* allowed, cudaStream_t stream) {
  if (rows < 0 || vocab <= 0 || vocab > (1 << 30) || slots <= 0 || biases < 0) return MLR_BAD_SIZE;
  if (rows == 0) return MLR_OK;
  if (rows > 65535) return MLR_TOO_LARGE;
  if (((uintptr_t)logits & 15) != 0 || ((uintptr_t)out & 15) != 0) return MLR_BAD_ALIGNMENT;
  if ((penalties != nullptr) != (counts != nullptr) || (penalties != nullptr) != (seen != nullptr)) return MLR_BAD_SIZE;
  RuleTables tables{penalties, counts, (const unsigned*)seen, biases > 0 ? bias_tokens : nullptr, bias_values,
                    (const unsigned*)allowed, biases, slots};
  launch_rules<4>(logits, out, row_slot, rows, vocab, tables, stream);
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
