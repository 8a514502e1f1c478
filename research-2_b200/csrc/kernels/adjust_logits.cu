// What stands between a step's logits and the draw: penalties for tokens that the row's request holds already, biases of single tokens and
// a grammar's mask, in one pass over the row.
//
//   x <- x / rho where x > 0, else x rho       for a token of the prompt or of the answer        (rho: the row's repetition penalty)
//   x <- x - (frequency c + presence [c > 0])  c: how often the token stands in the answer
//   x <- x + the sum of the row's biases for the token, in the order of their list
//   x <- -inf                                  where the row's mask has bit 0 at the token
//
// A CTA has a segment of one row's tokens and a place for each of them in shared memory. It reads the whole history and counts in the places
// what falls into its segment (integer atomics, so no order shows); the entry that comes to a token first lists it. The segment then passes
// through registers, 16 bytes at a time, with the mask alone (in place and without a mask there is nothing to pass); pieces of which the mask
// leaves nothing are written without being read. Behind that pass the listed tokens are worked out one by one, a thread a token, and written
// over it, as are the biases' tokens. So a row costs what copying it costs, and a history some twenty instructions an entry and segment:
// segments are as long as shared memory allows where there are CTAs enough without cutting finer. Numbers are float; a bfloat16 row is
// rounded once.
//
// What bounds it. 256 bfloat16 rows of 128,001 with up to 4,000 tokens, 300 biases and a mask: 53 us where their 139 MB take 21. A CTA's 22,000 cycles
// are a chain: the row's numbers (4,000), the history into the places (8,000: an entry is a load, an atomic that answers, a place on the
// list), the segment (4,000), the listed tokens; an SM's schedulers issue in 49 % of the cycles with two such CTAs. 64 rows of 50,257 with
// up to 1,000 tokens: 8.4 us (3.1 TB/s). One row: 2.8 us, a chain of round trips alone. In place, as a step calls it, with a table of 1,024 places a
// request and histories of up to 256: one row 2.5 us, eight 3.1, 64 3.7; with biases and a mask on every other row 4.1, 4.5 and 7.4. The first
// form, which applied all of it inside the pass over the segment (41 instructions a number), took 133 us.
#include "logit_rows.cuh"

namespace {

constexpr int DEPTH = 4, CHUNK = 4;   // pieces, and entries of the history, of a thread on their way
// A place: the token stands in the prompt, it has a bias, how often it stands in the answer. 16 bits where no history is longer than their
// counts, else 32.
template <typename W> struct Place {
  static constexpr uint32_t PROMPT = 1u << (8 * sizeof(W) - 1), BIASED = PROMPT >> 1, DRAWN = BIASED - 1;
  static constexpr int EACH = 4 / int(sizeof(W));   // places of a word
};

struct AdjustArgs {
  const void* logits; long long ld;
  void* out; long long out_ld;
  int rows, vocab, segments, per;   // per: pieces of a segment
  const int32_t* history; long long history_ld; int history_rows, history_cap;
  const int32_t *slots, *lengths, *prompt_lengths;
  const float *repetition, *presence, *frequency;
  const int32_t *bias_start, *bias_ids; const float* bias_values; int n_biases;
  const uint32_t* mask; long long mask_ld; int n_masks;
  const int32_t* mask_rows;
};

template <typename T, typename W, int THREADS>
__global__ void __launch_bounds__(THREADS, THREADS == 512 ? 2 : 4)
adjust_kernel(const AdjustArgs a) {
  constexpr int PER = RowPieces<T>::PER, EACH = Place<W>::EACH;
  constexpr uint32_t PROMPT = Place<W>::PROMPT, BIASED = Place<W>::BIASED, DRAWN = Place<W>::DRAWN, ANY = PROMPT | BIASED | DRAWN;
  extern __shared__ __align__(16) uint32_t places[];
  const int size = a.per * PER;                         // tokens of a segment
  uint32_t* allowed = places + size / EACH;             // the mask's words for the segment
  uint16_t* touched = reinterpret_cast<uint16_t*>(allowed + size / 32 + 3);   // places that the history came to
  __shared__ int n_touched, twice;                      // twice: the row names a token of this segment in more than one bias
  pdl_launch_dependents();
  const int row = int(blockIdx.x) / a.segments, segment = int(blockIdx.x) % a.segments, tid = int(threadIdx.x), lane = tid & 31;
  const T* logits = static_cast<const T*>(a.logits) + (long long)row * a.ld;
  const RowPieces<T> in(logits, a.vocab);
  T* out = static_cast<T*>(a.out) + (long long)row * a.out_ld;
  const int g0 = segment * a.per, n = min(a.per, in.count - g0), zero = in.first(g0);   // zero: the token of the first place
  for (int i = tid; i < size / EACH / 4; i += THREADS) reinterpret_cast<uint4*>(places)[i] = make_uint4(0u, 0u, 0u, 0u);
  if (tid == 0) n_touched = twice = 0;
  pdl_wait();
  if (n <= 0) return;   // (a segment that only rows of another alignment have)

  // everything that one number leads to is asked for before any of it is waited for
  const int mask_row = a.mask == nullptr ? -1 : a.mask_rows != nullptr ? a.mask_rows[row] : row;
  const int slot = a.history == nullptr ? -1 : a.slots != nullptr ? a.slots[row] : row;
  const int length_asked = a.history != nullptr ? a.lengths[row] : 0, prompt = a.prompt_lengths != nullptr ? a.prompt_lengths[row] : 0;
  const int bias_begin = a.bias_start != nullptr ? max(0, a.bias_start[row]) : 0;
  const int bias_end = a.bias_start != nullptr ? min(a.n_biases, a.bias_start[row + 1]) : 0;
  const float repetition = a.repetition != nullptr ? a.repetition[row] : 1.f, presence = a.presence != nullptr ? a.presence[row] : 0.f;
  const float frequency = a.frequency != nullptr ? a.frequency[row] : 0.f;
  const uint32_t* mask = mask_row >= 0 && mask_row < a.n_masks ? a.mask + (long long)mask_row * a.mask_ld : nullptr;
  const int length = slot >= 0 && slot < a.history_rows ? max(0, min(length_asked, a.history_cap)) : 0;
  const int32_t* tokens = a.history + (long long)slot * a.history_ld;
  int ahead[CHUNK];   // entries of the history
  auto load_tokens = [&](int i0) {
#pragma unroll
    for (int i = 0; i < CHUNK; ++i) ahead[i] = i0 + i * THREADS < length ? __ldg(tokens + i0 + i * THREADS) : -1;
  };
  load_tokens(tid);
  int bias_token = -1;
  float bias_value = 0.f;
  if (bias_begin + tid < bias_end) {
    bias_token = a.bias_ids[bias_begin + tid];
    bias_value = a.bias_values[bias_begin + tid];
  }
  // the mask's words from the one before the segment's first on: token t's bit is bit t - bit0 of them
  const int word0 = (max(zero, 0) >> 5) - 1, bit0 = word0 * 32;
  if (mask != nullptr)
    for (int i = tid; i < size / 32 + 3; i += THREADS) allowed[i] = mask[min(max(word0 + i, 0), (a.vocab - 1) >> 5)];
  const bool in_place = static_cast<const void*>(out) == static_cast<const void*>(logits);
  const bool vectors = ((reinterpret_cast<uintptr_t>(out) ^ reinterpret_cast<uintptr_t>(logits)) & 15) == 0, passes = mask != nullptr || !in_place;
  uint4 raw[DEPTH];
  uint32_t left[DEPTH];   // what the mask leaves of a piece
  auto load = [&](int at, uint4& raw, uint32_t& left) {
    if (at >= n) return;
    left = ~0u;
    if (mask != nullptr) {
      const int bit = at * PER + zero - bit0;
      left = __funnelshift_r(allowed[bit >> 5], allowed[(bit >> 5) + 1], bit & 31) & ((1u << PER) - 1u);
    }
    // (not by the read-only path: with the output over the input the row is written in this launch)
    if (left != 0u) raw = load_once(in, g0 + at);
  };
  auto load_first = [&]() {
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) load(tid + d * THREADS, raw[d], left[d]);
  };
  if (mask == nullptr && passes) load_first();
  __syncthreads();
  if (mask != nullptr) load_first();

  // what the request holds of this segment (places before and behind the row may be counted in, and are never written out)
#pragma unroll 1
  for (int i0 = tid; i0 - tid < length; i0 += CHUNK * THREADS) {
    if (i0 != tid) load_tokens(i0);
    uint32_t firsts[CHUNK];   // of the warp's lanes, those whose entry is its token's first
    int all = 0;
#pragma unroll
    for (int c = 0; c < CHUNK; ++c) {
      const int i = i0 + c * THREADS;
      const uint32_t at = uint32_t(ahead[c] - zero), shift = at % EACH * 16;
      bool first = false;
      if (at < uint32_t(size) && i < length) {
        const uint32_t before = i < prompt ? atomicOr(&places[at / EACH], PROMPT << shift) : atomicAdd(&places[at / EACH], 1u << shift);
        first = ((before >> shift) & ANY) == 0u;
      }
      firsts[c] = __ballot_sync(0xffffffffu, first);
      all += __popc(firsts[c]);
    }
    if (all == 0) continue;
    int base = 0;
    if (lane == 0) base = atomicAdd(&n_touched, all);
    base = __shfl_sync(0xffffffffu, base, 0);
#pragma unroll
    for (int c = 0; c < CHUNK; ++c) {
      if ((firsts[c] >> lane) & 1u) touched[base + __popc(firsts[c] & ((1u << lane) - 1u))] = uint16_t(ahead[c] - zero);
      base += __popc(firsts[c]);
    }
  }
  __syncthreads();
  auto mark = [&](int token) {
    const uint32_t at = uint32_t(token - zero), shift = at % EACH * 16;
    if (at < uint32_t(size) && (atomicOr(&places[at / EACH], BIASED << shift) & (BIASED << shift)) != 0u) twice = 1;
  };
  if (bias_begin + tid < bias_end) mark(bias_token);
#pragma unroll 1
  for (int i = bias_begin + tid + THREADS; i < bias_end; i += THREADS) mark(a.bias_ids[i]);

  // the first touched tokens' logits are on their way while the segment passes
  auto logit_at = [&](int i) {
    const int token = zero + (i < n_touched ? int(touched[i]) : -1 - zero);
    return token >= 0 && token < a.vocab ? to_float(logits[token]) : 0.f;
  };
  constexpr int EARLY = 2;
  float early[EARLY];
#pragma unroll
  for (int e = 0; e < EARLY; ++e) early[e] = logit_at(tid + e * THREADS);
  float bias_logit = bias_token >= max(zero, 0) && bias_token < min(zero + size, a.vocab) ? to_float(logits[bias_token]) : 0.f;

  if (passes) {
    // pieces from `low` up to `high` are written whole: the row's ends are not, nor where the output starts at another alignment
    const int last = in.count - 1 - g0, low = !vectors ? n : g0 == 0 && in.phase > 0 ? 1 : 0;
    const int high = last < n && !in.whole(g0 + last) ? last : n;
    uint4* to = reinterpret_cast<uint4*>(out - in.phase) + g0;
#pragma unroll 1
    for (int at0 = tid; at0 < n; at0 += DEPTH * THREADS) {
#pragma unroll
      for (int d = 0; d < DEPTH; ++d) {
        const int at = at0 + d * THREADS;
        if (at >= n) continue;
        if (mask != nullptr) keep_bits<T>(raw[d], left[d]);
        if (at >= low && at < high) to[at] = raw[d];
        else store_elements<T>(out, in.first(g0 + at), a.vocab, raw[d]);
        load(at + DEPTH * THREADS, raw[d], left[d]);
      }
    }
  }
  __syncthreads();   // what follows lies over it

  auto finish = [&](int token, float x, float bias) {
    const uint32_t at = uint32_t(token - zero), place = (places[at / EACH] >> (at % EACH * 16)) & ANY;
    if ((place & ~BIASED) != 0u) {
      x = x > 0.f ? x / repetition : x * repetition;
      if ((place & DRAWN) != 0u) x -= frequency * float(place & DRAWN) + presence;
    }
    if (place & BIASED) x += bias;
    if (mask != nullptr && !((allowed[(token - bit0) >> 5] >> (token & 31)) & 1u)) x = -INFINITY;
    out[token] = from_float<T>(x);
  };
  auto finish_touched = [&](int i, float x) {
    const int at = touched[i], token = zero + at;
    const bool biased = ((places[uint32_t(at) / EACH] >> (uint32_t(at) % EACH * 16)) & BIASED) != 0u;   // (the bias's entry writes it)
    if (!biased && token >= 0 && token < a.vocab) finish(token, x, 0.f);
  };
#pragma unroll
  for (int e = 0; e < EARLY; ++e)
    if (tid + e * THREADS < n_touched) finish_touched(tid + e * THREADS, early[e]);
#pragma unroll 2
  for (int i = tid + EARLY * THREADS; i < n_touched; i += THREADS) finish_touched(i, logit_at(i));
#pragma unroll 1
  for (int i = bias_begin + tid; i < bias_end; i += THREADS) {
    const bool kept = i == bias_begin + tid;
    const int token = kept ? bias_token : a.bias_ids[i];
    if (token < max(zero, 0) || token >= min(zero + size, a.vocab)) continue;
    float bias = kept ? bias_value : a.bias_values[i];
    if (twice) {  // the token's first entry adds them all
      bool earlier = false;
      bias = 0.f;
      for (int j = bias_begin; j < bias_end; ++j) {
        if (a.bias_ids[j] != token) continue;
        earlier |= j < i;
        bias += a.bias_values[j];
      }
      if (earlier) continue;
    }
    finish(token, kept ? bias_logit : to_float(logits[token]), bias);
  }
}

constexpr int MOST_SMEM = 160 * 1024;   // of a CTA

template <typename T, typename W, int THREADS>
int launch(const AdjustArgs& a, size_t smem, cudaStream_t stream) {
  static std::atomic<bool> allowed[64];
  const int status = allow_smem(adjust_kernel<T, W, THREADS>, MOST_SMEM, allowed);
  if (status != R2_OK) return status;
  r2_launch(adjust_kernel<T, W, THREADS>, dim3(unsigned(a.rows * a.segments)), dim3(THREADS), smem, stream, a);
  return launch_status();
}

template <typename T, typename W>
int launch_segments(AdjustArgs a, cudaStream_t stream) {
  constexpr int PER = RowPieces<T>::PER;
  const int pieces = (a.vocab + 2 * PER - 2) / PER;   // of a row at any alignment, at most
  // Tokens of a segment, at most: 64 KB of places for long histories, 32 KB, and so more CTAs an SM, for short ones or none (300 rows of 50,257 bfloat16: up
  // to 6,000 tokens 35 us, with 32 KB 40; up to 1,000 tokens 23.0, 21.7; none 17.8, 17.0, with 16 KB 19.5).
  const int most = (a.history != nullptr && a.history_cap > 2048 ? 64 : 32) * 1024 / int(sizeof(W)) / PER;
  // as many segments as it takes to have three CTAs to an SM (none below 2,048 tokens), more where the places need it: every segment counts the
  // whole history. (256 bfloat16 rows of 128,001: four segments with 64 KB of places 52.9 us, eight with 32 KB 57.6; 64 float32 rows of
  // 50,257: seven segments 8.6, three 9.6, fourteen 11.0; one row: 24 segments 2.9, three 4.3, 49 2.8; eight rows: 24 segments 4.5, three 6.1, 49 4.6.)
  int segments = max(1, min((3 * 148 + a.rows - 1) / a.rows, pieces * PER / 2048));
  segments = max(segments, (pieces + most - 1) / most);
  a.per = ((pieces + segments - 1) / segments * PER + 31) / 32 * 32 / PER;   // whole words of the mask
  a.segments = (pieces + a.per - 1) / a.per;
  if ((long long)a.rows * a.segments > 0x7fffffffLL) return R2_BAD_SHAPE;
  const int size = a.per * PER;   // at most 65,536 places: their numbers have 16 bits
  const size_t smem = size_t(size) * sizeof(W) + size_t(size / 32 + 3) * 4 + (a.history != nullptr ? size_t(min(size, a.history_cap)) * 2 : 0);
  // (the same 256 rows with 256 threads a segment of 32,768: 66 us; the 64 rows with 512 a segment of 7,200: 11.6)
  return size >= 16384 ? launch<T, W, 512>(a, smem, stream) : launch<T, W, 256>(a, smem, stream);
}

template <typename T>
int launch_places(const AdjustArgs& a, cudaStream_t stream) {
  if (a.history != nullptr && a.history_cap > int(Place<uint16_t>::DRAWN)) return launch_segments<T, uint32_t>(a, stream);
  return launch_segments<T, uint16_t>(a, stream);
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
  if (history != nullptr && history_cap > int(Place<uint32_t>::DRAWN)) return R2_UNSUPPORTED;
  if (bias_start != nullptr && (n_biases < 0 || (n_biases > 0 && (bias_ids == nullptr || bias_values == nullptr)))) return R2_BAD_SHAPE;
  if (mask != nullptr && mask_ld * 32 < vocab) return R2_BAD_SHAPE;
  if (rows == 0) return R2_OK;
  const AdjustArgs a = {logits, ld, out, out_ld, rows, vocab, 0, 0, history, history_ld, history_rows, history_cap, slots, lengths,
                        prompt_lengths, repetition, presence, frequency, bias_start, bias_ids, bias_values, n_biases, mask, mask_ld,
                        n_masks, mask_rows};
  return dtype == R2_F32 ? launch_places<float>(a, stream) : launch_places<bf16>(a, stream);
}
