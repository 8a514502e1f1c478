// The k largest logits of every row with their tokens, from the largest down, equal values from the lowest token up, and the logarithm of
// the row's sum of exponentials at a temperature.
//
// A row is read once. While it passes, a thread sums exponentials against its own maximum and keeps the maximum of every group of four
// 16-byte pieces. The k-th largest of these maxima (or a little less) is a value that at least k elements reach, and what reaches it stands
// in the groups whose maximum does: about k groups of 16 or 32 elements, which are read again and give little more than k candidates. Their
// order is found by counting for each how many stand above it. Values are compared as unsigned keys in the floats' order, with
// the token as the lower half.
//
// Rows whose candidates do not fit (thousands of equal values at the edge of the list, or fewer than k numbers that are not NaN) are gone
// over again: the exact k-th value by counts in bins of the keys' range, bin by bin narrower, everything above it, and equal values in the
// order of their tokens until the list is full.
//
// Few rows are cut over the CTAs of a cluster, whose candidates meet in the first one's shared memory.
#include "logit_rows.cuh"

namespace {

constexpr int THREADS = 256, WARPS = THREADS / 32;
constexpr int MOST_K = 256, MOST_RANKS = 8;
constexpr int DEPTH = 4;      // pieces of a group
constexpr int SLOTS = 16;     // groups of a thread
constexpr int CAP = 2304;     // candidates
constexpr int BINS = 512;
constexpr int LEVELS = 4;     // 9 bits of a 32-bit key at each
constexpr int MOST_SORTED = 4096;

struct TopArgs {
  const void* logits; long long ld;
  int vocab, k, ranks, per;
  float tau;
  float* values; int32_t* ids; float* log_sum;
};

struct Shared {
  uint32_t groups[SLOTS][THREADS];        // the groups' maxima, as keys
  unsigned long long found[MOST_SORTED];  // candidates: key, then the token's complement
  uint32_t bins[BINS];
  uint32_t chosen[BINS];                  // groups that are read again: slot * THREADS + thread
  uint32_t warp_numbers[2][WARPS];
  float warp_sums[2][WARPS];
  uint32_t low, high, above, n_found, n_chosen;
  float4 sums[MOST_RANKS];                // of the cluster's CTAs: reference, sum
  uint32_t n_of[MOST_RANKS];
};

__device__ __forceinline__ float value_of(uint32_t key) {
  if (key == 0u) return __uint_as_float(0x7fffffffu);
  return __uint_as_float((key & 0x80000000u) ? (key & 0x7fffffffu) : ~key);
}
__device__ __forceinline__ unsigned long long composite(uint32_t key, int token) {
  return (static_cast<unsigned long long>(key) << 32) | (0xffffffffu - uint32_t(token));
}

// One level: the bins of the keys in [low, high] are counted; from the top, the bin at which the count (with `above`, keys over `high`)
// reaches k becomes the range. True once the bins are single keys.
__device__ __forceinline__ bool narrow(Shared& s, int k, int shift) {
  __syncthreads();
  if (threadIdx.x < 32) {
    const int lane = int(threadIdx.x);
    uint32_t c[BINS / 32], sum = 0u;   // lane l has the bins from BINS - 1 - 16 l down
#pragma unroll
    for (int j = 0; j < BINS / 32; ++j) {
      c[j] = s.bins[BINS - 1 - lane * (BINS / 32) - j];
      sum += c[j];
    }
    uint32_t upto = sum;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint32_t other = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += other;
    }
    const uint32_t low = s.low, high = s.high, before = s.above;
    __syncwarp();
    uint32_t above = before + upto - sum;
    if (above < uint32_t(k) && uint32_t(k) <= before + upto) {
#pragma unroll
      for (int j = 0; j < BINS / 32; ++j) {
        if (above < uint32_t(k) && uint32_t(k) <= above + c[j]) {
          const uint32_t bin = uint32_t(BINS - 1 - lane * (BINS / 32) - j);
          s.low = low + (bin << shift);
          s.high = min(high, s.low + ((1u << shift) - 1u));
          s.above = above;
          s.n_chosen = above + c[j];   // how many reach the new `low`
        }
        above += c[j];
      }
    }
  }
  __syncthreads();
  return shift == 0;
}
__device__ __forceinline__ int shift_of(uint32_t low, uint32_t high) {   // (high - low) >> shift < BINS
  const int bits = 32 - __clz(int(high - low));
  return bits > 9 ? bits - 9 : 0;
}

template <typename T>
struct Row {
  RowPieces<T> x;
  int g0, n;   // this CTA's pieces
  __device__ __forceinline__ uint4 load(int at) const {   // a piece of the share, -inf where it is not the row's
    uint4 raw = load_once(x, g0 + at);
    if (g0 + at == 0 || g0 + at == x.count - 1) blank_outside(raw, x, g0 + at);
    return raw;
  }
  __device__ __forceinline__ bool inside(int token) const { return token >= 0 && token < x.vocab; }
};

// The row again, from its exact k-th value: at least k of the share's elements reach `reached`, or it is 0.
template <typename T>
__device__ __noinline__ void go_over(Shared& s, const Row<T>& row, int k, uint32_t reached) {
  constexpr int PER = RowPieces<T>::PER;
  const int tid = int(threadIdx.x), lane = tid & 31, warp = tid >> 5;
  auto over = [&](auto&& f) {   // every element of the share: (key, token)
    for (int at = tid; at < row.n; at += THREADS) {
      float v[PER];
      unpack(row.load(at), v, static_cast<const T*>(nullptr));
#pragma unroll
      for (int e = 0; e < PER; ++e) {
        const int token = row.x.first(row.g0 + at) + e;
        if (row.inside(token)) f(logit_key(v[e]), token);
      }
    }
  };
  __syncthreads();
  if (tid == 0) {
    s.low = reached;
    s.high = 0xffffffffu;
    s.above = 0u;
    s.n_found = 0u;
  }
  __syncthreads();
  // whether fewer than k lie above `reached`: then it is the k-th value
  uint32_t more = 0u;
  over([&](uint32_t key, int) { more += key > reached ? 1u : 0u; });
  more = __reduce_add_sync(0xffffffffu, more);
  if (lane == 0) atomicAdd(&s.n_found, more);
  __syncthreads();
  const bool is_kth = s.n_found < uint32_t(k);
  __syncthreads();
  if (is_kth) {
    if (tid == 0) s.high = s.low;
  } else {
    for (int level = 0; level < LEVELS; ++level) {
      for (int b = tid; b < BINS; b += THREADS) s.bins[b] = 0u;
      __syncthreads();
      const uint32_t low = s.low, high = s.high;
      const int shift = shift_of(low, high);
      over([&](uint32_t key, int) {
        if (key >= low && key <= high) atomicAdd(&s.bins[(key - low) >> shift], 1u);
      });
      if (narrow(s, k, shift)) break;
    }
  }
  if (tid == 0) s.n_found = 0u;
  __syncthreads();
  const uint32_t kth = s.low;
  over([&](uint32_t key, int token) {
    if (key > kth) s.found[atomicAdd(&s.n_found, 1u)] = composite(key, token);   // (fewer than k)
  });
  __syncthreads();
  // equal values in the tokens' order
  int wanted = k - int(s.n_found), have = int(s.n_found);
  for (int base = 0; base < row.n && wanted > 0; base += THREADS) {
    const int at = base + tid;
    uint32_t equal = 0u;
    if (at < row.n) {
      float v[PER];
      unpack(row.load(at), v, static_cast<const T*>(nullptr));
#pragma unroll
      for (int e = 0; e < PER; ++e)
        if (row.inside(row.x.first(row.g0 + at) + e) && logit_key(v[e]) == kth) equal |= 1u << e;
    }
    const uint32_t mine = uint32_t(__popc(equal));
    uint32_t upto = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint32_t other = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += other;
    }
    __syncthreads();
    if (lane == 31) s.warp_numbers[0][warp] = upto;
    __syncthreads();
    uint32_t before = upto - mine, all = 0u;
    for (int i = 0; i < WARPS; ++i) {
      before += i < warp ? s.warp_numbers[0][i] : 0u;
      all += s.warp_numbers[0][i];
    }
    for (int e = 0; e < PER; ++e) {
      if (!((equal >> e) & 1u)) continue;
      if (int(before) < wanted) s.found[have + int(before)] = composite(kth, row.x.first(row.g0 + at) + e);
      ++before;
    }
    const int taken = min(wanted, int(all));
    wanted -= taken;
    have += taken;
  }
  __syncthreads();
  if (tid == 0) s.n_found = uint32_t(have);
  __syncthreads();
}

template <typename T>
__global__ void __launch_bounds__(THREADS, 4)
top_kernel(const TopArgs a) {
  constexpr int PER = RowPieces<T>::PER, PAIRS = PER / 2;
  extern __shared__ __align__(16) uint8_t top_smem[];
  Shared& s = *reinterpret_cast<Shared*>(top_smem);
  pdl_launch_dependents();
  const int ranks = a.ranks, row_index = int(blockIdx.x) / ranks, rank = int(blockIdx.x) % ranks, tid = int(threadIdx.x), lane = tid & 31, warp = tid >> 5;
  if (tid == 0) s.n_found = s.n_chosen = s.above = 0u;
  for (int b = tid; b < BINS; b += THREADS) s.bins[b] = 0u;
  pdl_wait();
  Row<T> row = {RowPieces<T>(static_cast<const T*>(a.logits) + (long long)row_index * a.ld, a.vocab), rank * a.per, 0};
  row.n = max(0, min(a.per, row.x.count - row.g0));
  const float c = 1.44269504f / a.tau;
  const uint64_t cc = two_of(c, c);
  const int rounds = (row.n + THREADS * DEPTH - 1) / (THREADS * DEPTH), together = (rounds + SLOTS - 1) / SLOTS;   // of a group

  // one pass: sums, and every group's maximum
  float reference = -INFINITY, sum = 0.f;
  uint32_t thread_max = 0u, slot_max = 0u;
  uint4 raw[DEPTH];
  auto load = [&](int round) {
    const int at = round * THREADS * DEPTH + tid;
#pragma unroll
    for (int i = 0; i < DEPTH; ++i) {
      const uint32_t nothing = sizeof(T) == 4 ? 0xff800000u : 0xff80ff80u;
      raw[i] = make_uint4(nothing, nothing, nothing, nothing);
      if (at + i * THREADS < row.n) raw[i] = load_once(row.x, row.g0 + at + i * THREADS);
    }
  };
  load(0);
#pragma unroll 1
  for (int round = 0; round < rounds; ++round) {
    const int at = round * THREADS * DEPTH + tid;
    uint4 now[DEPTH];
#pragma unroll
    for (int i = 0; i < DEPTH; ++i) now[i] = raw[i];
    if (round + 1 < rounds) load(round + 1);
    float most = -INFINITY;
#pragma unroll
    for (int i = 0; i < DEPTH; ++i) {
      if (row.g0 + at + i * THREADS == 0 || row.g0 + at + i * THREADS == row.x.count - 1) blank_outside(now[i], row.x, row.g0 + at + i * THREADS);
      float v[PER];
      unpack(now[i], v, static_cast<const T*>(nullptr));
#pragma unroll
      for (int e = 0; e < PER; ++e) most = fmaxf(most, v[e]);
    }
    const float up = fminf(most * c, 3e38f);   // (an infinity sums to infinity against any number)
    if (up > reference) {
      sum *= rebase(reference, up);
      reference = up;
    }
    const float shift = -no_less(reference);
    const uint64_t ss = two_of(shift, shift);
    uint64_t acc[DEPTH];
#pragma unroll
    for (int i = 0; i < DEPTH; ++i) {
      uint64_t p[PAIRS];
      unpack_pairs(now[i], p, static_cast<const T*>(nullptr));
      acc[i] = exp2_two(fma_two(p[0], cc, ss));
#pragma unroll
      for (int j = 1; j < PAIRS; ++j) acc[i] = add_two(acc[i], exp2_two(fma_two(p[j], cc, ss)));
    }
#pragma unroll
    for (int i = 1; i < DEPTH; ++i) acc[0] = add_two(acc[0], acc[i]);
    const float2 both = halves(acc[0]);
    sum += both.x + both.y;
    slot_max = max(slot_max, logit_key(most));
    if ((round + 1) % together == 0 || round + 1 == rounds) {
      s.groups[round / together][tid] = slot_max;
      thread_max = max(thread_max, slot_max);
      slot_max = 0u;
    }
  }
  const int slots = (rounds + together - 1) / max(together, 1);
  {
    const float common = warp_max(reference);
    sum = warp_sum(sum * rebase(reference, common));
    const uint32_t most = __reduce_max_sync(0xffffffffu, thread_max), least = __reduce_min_sync(0xffffffffu, thread_max);
    if (lane == 0) {
      s.warp_sums[0][warp] = common;
      s.warp_sums[1][warp] = sum;
      s.warp_numbers[0][warp] = most;
      s.warp_numbers[1][warp] = least;
    }
  }
  __syncthreads();
  uint32_t low = 0xffffffffu, high = 0u;   // every thread has a group that reaches `low`: 256 of them or more
  for (int i = 0; i < WARPS; ++i) {
    high = max(high, s.warp_numbers[0][i]);
    low = min(low, s.warp_numbers[1][i]);
  }
  float total = 0.f, common = -INFINITY;
  for (int i = 0; i < WARPS; ++i) common = fmaxf(common, s.warp_sums[0][i]);
  for (int i = 0; i < WARPS; ++i) total += s.warp_sums[1][i] * rebase(s.warp_sums[0][i], common);

  // what the k-th largest maximum reaches
  const int first_token = max(0, row.x.first(row.g0)), end_token = min(a.vocab, row.x.first(row.g0) + row.n * PER);
  const int k = min(a.k, end_token - first_token);   // of this share
  const int limit = k + max(32, k / 4);
  uint32_t reached = 0u;
  bool fits = true;
  if (row.n >= THREADS) {   // a group for every thread
    if (tid == 0) {
      s.low = low;
      s.high = high;
    }
    __syncthreads();
    for (int level = 0; level < LEVELS; ++level) {
      const uint32_t from = s.low, to = s.high;
      const int shift = shift_of(from, to);
      for (int g = 0; g < slots; ++g) {
        const uint32_t key = s.groups[g][tid];
        if (key >= from && key <= to) atomicAdd(&s.bins[(key - from) >> shift], 1u);
      }
      const bool last = narrow(s, k, shift);
      if (last || s.n_chosen <= uint32_t(limit)) break;
      for (int b = tid; b < BINS; b += THREADS) s.bins[b] = 0u;
      __syncthreads();
    }
    reached = s.low;
    fits = s.n_chosen <= uint32_t(BINS);
    __syncthreads();
    if (tid == 0) s.n_chosen = 0u;
    __syncthreads();
    if (fits) {
      for (int g = 0; g < slots; ++g)
        if (s.groups[g][tid] >= reached) s.chosen[atomicAdd(&s.n_chosen, 1u)] = uint32_t(g * THREADS + tid);
      __syncthreads();
      // a group's pieces again, a piece a thread
      const int pieces = int(s.n_chosen) * together * DEPTH;
      for (int p = tid; p < pieces; p += THREADS) {
        const uint32_t group = s.chosen[p / (together * DEPTH)];
        const int at = (int(group / THREADS) * together * DEPTH + p % (together * DEPTH)) * THREADS + int(group % THREADS);
        if (at >= row.n) continue;
        float v[PER];
        unpack(row.load(at), v, static_cast<const T*>(nullptr));
#pragma unroll
        for (int e = 0; e < PER; ++e) {
          const uint32_t key = logit_key(v[e]);
          const int token = row.x.first(row.g0 + at) + e;
          if (key >= reached && row.inside(token)) {
            const uint32_t place = atomicAdd(&s.n_found, 1u);
            if (place < uint32_t(CAP)) s.found[place] = composite(key, token);
          }
        }
      }
    }
  } else {   // a short share: everything is a candidate
    if (tid == 0) s.n_found = uint32_t(end_token - first_token);
    for (int at = tid; at < row.n; at += THREADS) {
      float v[PER];
      unpack(row.load(at), v, static_cast<const T*>(nullptr));
#pragma unroll
      for (int e = 0; e < PER; ++e) {
        const int token = row.x.first(row.g0 + at) + e;
        if (row.inside(token)) s.found[token - first_token] = composite(logit_key(v[e]), token);
      }
    }
  }
  __syncthreads();
  if (!fits || s.n_found > uint32_t(CAP)) go_over(s, row, k, reached);
  else if (s.n_found < uint32_t(k)) go_over(s, row, k, 0u);

  // the cluster's candidates into its first CTA
  int n = int(s.n_found);
  if (ranks > 1) {
    if (n > MOST_SORTED / MOST_RANKS) {   // (more than the first CTA has places for from each: the exact k)
      go_over(s, row, k, reached);
      n = k;
    }
    cluster_arrive();   // the first CTA has what it found itself in the first of its places, the others are free
    cluster_wait();
    const uint32_t found = cluster_address(s.found, 0), counts = cluster_address(s.n_of, 0), sums = cluster_address(s.sums, 0);
    if (rank > 0)
      for (int i = tid; i < n; i += THREADS)
        asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(found + uint32_t(rank * (MOST_SORTED / MOST_RANKS) + i) * 8u), "l"(s.found[i]) : "memory");
    if (tid == 0) {
      asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(counts + uint32_t(rank) * 4u), "r"(uint32_t(n)) : "memory");
      cluster_store(sums + uint32_t(rank) * 16u, make_float4(common, total, 0.f, 0.f));
    }
    cluster_arrive();
    cluster_wait();
    if (rank > 0) return;
    common = -INFINITY;
    total = 0.f;
    for (int r = 0; r < ranks; ++r) common = fmaxf(common, s.sums[r].x);
    for (int r = 0; r < ranks; ++r) total += s.sums[r].y * rebase(s.sums[r].x, common);
    int all = n;   // close the gaps
    for (int r = 1; r < ranks; ++r) {
      const int count = int(s.n_of[r]), from = r * (MOST_SORTED / MOST_RANKS);
      const unsigned long long one = tid < count ? s.found[from + tid] : 0ull, two = tid + THREADS < count ? s.found[from + tid + THREADS] : 0ull;
      __syncthreads();
      if (tid < count) s.found[all + tid] = one;
      if (tid + THREADS < count) s.found[all + tid + THREADS] = two;
      all += count;
      __syncthreads();
    }
    n = all;
  }
  if (tid == 0) a.log_sum[row_index] = (no_less(common) + log2f(total)) * 0.693147181f;

  float* values = a.values + (long long)row_index * a.k;
  int32_t* ids = a.ids + (long long)row_index * a.k;
  if (n <= 2 * THREADS) {
    // a candidate's place: how many stand above it
    for (int i = tid; i < n; i += THREADS) {
      const unsigned long long mine = s.found[i];
      int place = 0;
#pragma unroll 4
      for (int j = 0; j < n; ++j) place += s.found[j] > mine ? 1 : 0;
      if (place < a.k) {
        values[place] = value_of(uint32_t(mine >> 32));
        ids[place] = int32_t(0xffffffffu - uint32_t(mine & 0xffffffffull));
      }
    }
    return;
  }
  // many candidates: sorted in place (bitonic, from the largest down)
  int size = 2 * THREADS;
  while (size < n) size *= 2;
  for (int i = n + tid; i < size; i += THREADS) s.found[i] = 0ull;
  __syncthreads();
  for (int run = 2; run <= size; run *= 2) {
    for (int apart = run / 2; apart > 0; apart /= 2) {
      for (int i = tid; i < size / 2; i += THREADS) {
        const int lo = 2 * i - (i & (apart - 1)), hi = lo + apart;
        const unsigned long long x = s.found[lo], y = s.found[hi];
        if ((x < y) == ((lo & run) == 0)) {
          s.found[lo] = y;
          s.found[hi] = x;
        }
      }
      __syncthreads();
    }
  }
  for (int i = tid; i < a.k; i += THREADS) {
    values[i] = value_of(uint32_t(s.found[i] >> 32));
    ids[i] = int32_t(0xffffffffu - uint32_t(s.found[i] & 0xffffffffull));
  }
}

template <typename T>
int launch(TopArgs a, int rows, cudaStream_t stream) {
  const int pieces = (a.vocab + 2 * RowPieces<T>::PER - 2) / RowPieces<T>::PER;   // of a row at any alignment, at most
  a.ranks = 1;
  while (a.ranks < MOST_RANKS && (long long)rows * a.ranks * 2 <= 296 && pieces / (2 * a.ranks) >= THREADS * DEPTH) a.ranks *= 2;
  a.per = (pieces + a.ranks - 1) / a.ranks;
  if ((long long)rows * a.ranks > 0x7fffffffLL) return R2_BAD_SHAPE;
  static std::atomic<bool> allowed[64];
  const int status = allow_smem(top_kernel<T>, sizeof(Shared), allowed);
  if (status != R2_OK) return status;
  r2_launch_clusters(top_kernel<T>, a.ranks, dim3(unsigned(rows) * unsigned(a.ranks)), dim3(THREADS), sizeof(Shared), stream, a);
  return launch_status();
}

}  // namespace

// logits [rows, vocab] of dtype with row stride ld -> values [rows, k] float, ids [rows, k], log_sum [rows].
extern "C" int r2_top_logits(int dtype, const void* logits, long long ld, int rows, int vocab, int k, float temperature, float* values,
                             int32_t* ids, float* log_sum, cudaStream_t stream) {
  if (dtype != R2_F32 && dtype != R2_BF16) return R2_BAD_DTYPE;
  if (rows < 0 || vocab < 1 || vocab > (1 << 30) || ld < vocab || k < 1 || k > vocab) return R2_BAD_SHAPE;
  if (k > MOST_K || !(temperature > 0.f)) return R2_UNSUPPORTED;
  if (rows == 0) return R2_OK;
  const TopArgs a = {logits, ld, vocab, k, 1, 0, temperature, values, ids, log_sum};
  return dtype == R2_F32 ? launch<float>(a, rows, stream) : launch<bf16>(a, rows, stream);
}
