// What stands between a step's logits and the draw: penalties for tokens that the row's request holds already, biases of single tokens and
// a grammar's mask, in one pass over the row.
//
//   x <- x / rho where x > 0, else x rho       for a token of the prompt or of the answer        (rho: the row's repetition penalty)
//   x <- x - (frequency c + presence [c > 0])  c: how often the token stands in the answer
//   x <- x + the sum of the row's biases for the token, in the order of their list
//   x <- -inf                                  where the row's mask has bit 0 at the token
//
// A CTA has a slice of 4,096 tokens of one row. Which of them the request holds is counted in shared memory (integer atomics, so no order
// shows); biases are added into a second table by one warp in the list's order, lanes that name the same token one after the other.
// Numbers are float; a bfloat16 row is rounded once, at the end.
#include "logit_rows.cuh"

namespace {

constexpr int THREADS = 256;
constexpr int SLICE = 4096;            // places of a CTA's tables
constexpr uint32_t PROMPT = 1u << 31;  // the token stands in the prompt; below it the count in the answer

struct AdjustArgs {
  const void* logits; long long ld;
  void* out; long long out_ld;
  int rows, vocab, n_slices;
  const int32_t* history; long long history_ld; int history_rows, history_cap;
  const int32_t *slots, *lengths, *prompt_lengths;
  const float *repetition, *presence, *frequency;
  const int32_t *bias_start, *bias_ids; const float* bias_values; int n_biases;
  const uint32_t* mask; long long mask_ld; int n_masks;
  const int32_t* mask_rows;
};

template <typename T>
__global__ void __launch_bounds__(THREADS)
adjust_kernel(const AdjustArgs a) {
  constexpr int PER = RowPieces<T>::PER, OWN = SLICE / PER / THREADS;
  __shared__ __align__(16) uint32_t counts[SLICE];
  __shared__ __align__(16) float biases[SLICE];
  pdl_launch_dependents();
  const int row = int(blockIdx.x) / a.n_slices, slice = int(blockIdx.x) % a.n_slices, tid = int(threadIdx.x);
  const RowPieces<T> in(static_cast<const T*>(a.logits) + (long long)row * a.ld, a.vocab);
  T* out = static_cast<T*>(a.out) + (long long)row * a.out_ld;
  const int g0 = slice * (SLICE / PER);
  if (g0 >= in.count) {  // (a slice that only rows of another alignment have)
    pdl_wait();
    return;
  }
#pragma unroll
  for (int i = 0; i < SLICE / 4 / THREADS; ++i) {
    reinterpret_cast<uint4*>(counts)[tid + i * THREADS] = make_uint4(0u, 0u, 0u, 0u);
    reinterpret_cast<float4*>(biases)[tid + i * THREADS] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  pdl_wait();
  __syncthreads();
  const int zero = in.first(g0);   // the token of the tables' first place
  int length = 0, prompt = 0;
  const int32_t* held = nullptr;
  if (a.history != nullptr) {
    const int slot = a.slots != nullptr ? a.slots[row] : row;
    if (slot >= 0 && slot < a.history_rows) {
      length = max(0, min(a.lengths[row], a.history_cap));
      prompt = a.prompt_lengths != nullptr ? a.prompt_lengths[row] : 0;
      held = a.history + (long long)slot * a.history_ld;
    }
  }
  for (int i = tid; i < length; i += THREADS) {
    const int token = held[i], at = token - zero;
    if (token >= 0 && token < a.vocab && at >= 0 && at < SLICE) {
      if (i < prompt) atomicOr(&counts[at], PROMPT);
      else atomicAdd(&counts[at], 1u);
    }
  }
  if (a.bias_start != nullptr && tid < 32) {
    const int begin = max(0, a.bias_start[row]), end = min(a.n_biases, a.bias_start[row + 1]);
    for (int i0 = begin; i0 < end; i0 += 32) {
      const int i = i0 + tid, token = i < end ? a.bias_ids[i] : -1, at = token - zero;
      const bool mine = token >= 0 && token < a.vocab && at >= 0 && at < SLICE;
      const uint32_t some = __ballot_sync(0xffffffffu, mine);
      if (some == 0u) continue;
      const float value = mine ? a.bias_values[i] : 0.f;
      const uint32_t same = __match_any_sync(0xffffffffu, mine ? at : -1 - tid);
      // lanes of one token in lane order: the first adds them all
      if (__any_sync(0xffffffffu, __popc(same) > 1)) {
        float sum = mine ? biases[at] : 0.f;
        for (int l = 0; l < 32; ++l) {
          const float other = __shfl_sync(0xffffffffu, value, l);
          if ((same >> l) & 1u) sum += other;
        }
        if (mine && (__ffs(int(same)) - 1) == tid) biases[at] = sum;
      } else if (mine) {
        biases[at] += value;
      }
      __syncwarp();
    }
  }
  __syncthreads();
  const float rho = a.repetition != nullptr ? a.repetition[row] : 1.f;
  const float presence = a.presence != nullptr ? a.presence[row] : 0.f, frequency = a.frequency != nullptr ? a.frequency[row] : 0.f;
  const int mask_row = a.mask != nullptr ? (a.mask_rows != nullptr ? a.mask_rows[row] : row) : -1;
  const uint32_t* mask = mask_row >= 0 && mask_row < a.n_masks ? a.mask + (long long)mask_row * a.mask_ld : nullptr;
  const bool vectors = ((reinterpret_cast<uintptr_t>(out) ^ reinterpret_cast<uintptr_t>(in.base + in.phase)) & 15) == 0;
#pragma unroll
  for (int o = 0; o < OWN; ++o) {
    const int g = g0 + tid + o * THREADS, at = (tid + o * THREADS) * PER, first = in.first(g);
    if (g >= in.count) continue;
    float x[PER];
    // (a plain load: with the output over the input the row is written in this launch, each piece by the thread that read it)
    unpack(*(reinterpret_cast<const uint4*>(in.base) + g), x, static_cast<const T*>(nullptr));
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const uint32_t c = counts[at + i];
      if (c != 0u) {
        x[i] = x[i] > 0.f ? x[i] / rho : x[i] * rho;
        const uint32_t drawn = c & ~PROMPT;
        if (drawn != 0u) x[i] -= frequency * float(drawn) + presence;
      }
      x[i] += biases[at + i];
      const int token = first + i;
      if (mask != nullptr && token >= 0 && token < a.vocab && !((mask[token >> 5] >> (token & 31)) & 1u)) x[i] = -INFINITY;
    }
    store_piece<T, PER>(out, first, a.vocab, x, vectors);
  }
}

}  // namespace

// logits [rows, vocab] with row stride ld -> out [rows, vocab] with row stride out_ld, both of dtype (out may be logits). Row r's tokens are
// history[slots[r]][0 .. lengths[r]), the first prompt_lengths[r] of them the prompt's; its biases are entries bias_start[r] up to
// bias_start[r + 1]; its mask is mask[mask_rows[r]] (bit token % 32 of word token / 32; a row outside the masks has none).
extern "C" int r2_adjust_logits(int dtype, const void* logits, long long ld, void* out, long long out_ld, int rows, int vocab,
                                const int32_t* history, long long history_ld, int history_rows, int history_cap, const int32_t* slots,
                                const int32_t* lengths, const int32_t* prompt_lengths, const float* repetition, const float* presence,
                                const float* frequency, const int32_t* bias_start, const int32_t* bias_ids, const float* bias_values,
                                int n_biases, const uint32_t* mask, long long mask_ld, int n_masks, const int32_t* mask_rows,
                                cudaStream_t stream) {
  if (dtype != R2_F32 && dtype != R2_BF16) return R2_BAD_DTYPE;
  if (rows < 0 || vocab < 1 || vocab > (1 << 30) || ld < vocab || out_ld < vocab) return R2_BAD_SHAPE;
  if (history != nullptr && (lengths == nullptr || history_cap < 0 || history_rows < 1)) return R2_BAD_SHAPE;
  if (bias_start != nullptr && (n_biases < 0 || (n_biases > 0 && (bias_ids == nullptr || bias_values == nullptr)))) return R2_BAD_SHAPE;
  if (mask != nullptr && mask_ld * 32 < vocab) return R2_BAD_SHAPE;
  if (rows == 0) return R2_OK;
  const int per = dtype == R2_F32 ? 4 : 8;
  const int n_slices = (vocab + per - 1 + SLICE - 1) / SLICE;  // whatever a row's alignment
  if ((long long)rows * n_slices > 0x7fffffffLL) return R2_BAD_SHAPE;
  const AdjustArgs a = {logits, ld, out, out_ld, rows, vocab, n_slices, history, history_ld, history_rows, history_cap, slots, lengths,
                        prompt_lengths, repetition, presence, frequency, bias_start, bias_ids, bias_values, n_biases, mask, mask_ld,
                        n_masks, mask_rows};
  const dim3 grid(unsigned(rows * n_slices));
  if (dtype == R2_F32) r2_launch(adjust_kernel<float>, grid, dim3(THREADS), size_t(0), stream, a);
  else r2_launch(adjust_kernel<bf16>, grid, dim3(THREADS), size_t(0), stream, a);
  return launch_status();
}
