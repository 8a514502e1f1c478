// The k largest logits of every row with their tokens, from the largest down, equal values from the lowest token up, and the logarithm of
// the row's sum of exponentials at a temperature.
//
// A row is read once. While it passes, a thread sums exponentials against its own maximum and keeps the maximum of every group of four
// 16-byte pieces. The k-th largest of the maxima of 384 pairs of threads (or a little less) is a value that at least k elements reach, and
// what reaches it stands in the groups whose maximum does: little more than k groups of 16 or 32 elements, which are read again and give
// little more than k candidates. Their order is found by counting for each how many stand above it. Values are compared as unsigned keys in the
// floats' order, with the token as the lower half.
//
// Rows whose candidates do not fit (thousands of equal values at the edge of the list, or fewer than k numbers that are not NaN) are gone
// over again: the exact k-th value by counts in bins of the keys' range, bin by bin narrower, everything above it, and equal values in the
// order of their tokens until the list is full.
//
// An SM has one CTA: 24 warps read, row after row, and two teams of four choose, in turn: the candidates of two rows are looked for while the
// next one passes. Few rows are cut over the CTAs of a cluster, whose candidates meet in the first one's shared memory.
#include "logit_rows.cuh"

namespace {

constexpr int READERS = 768, PAIRS_OF_READERS = READERS / 2, READING_WARPS = READERS / 32;
constexpr int CHOOSERS = 128, CHOOSING_WARPS = CHOOSERS / 32, TEAMS = 2;   // of a team
// Rows that are between reading and choosing. A place is always the same team's: with a place that changed teams, one that is ahead of the
// other would take the readers' word for the other's row as its own.
constexpr int PLACES = 2 * TEAMS;
constexpr int MOST_K = 256, MOST_RANKS = 8;
constexpr int DEPTH = 4;      // pieces of a group
constexpr int SLOTS = 6;      // groups of a thread (of several rounds each in long rows)
constexpr int CAP = 2304;     // candidates
constexpr int BINS = 512;
constexpr int LEVELS = 4;     // 9 bits of a 32-bit key at each
constexpr int MOST_SORTED = 4096;

struct TopArgs {
  const void* logits; long long ld;
  int rows, vocab, k, ranks, per;
  float tau;
  float* values; int32_t* ids; float* log_sum;
};

// From those who read to those who choose.
struct __align__(16) Place {
  uint32_t groups[SLOTS][READERS];        // the groups' maxima, as keys
  uint32_t most[PAIRS_OF_READERS];        // the maxima of pairs of threads
  float2 sums[READING_WARPS];             // the warps' references and sums
};
// A team's own.
struct __align__(16) Shared {
  unsigned long long found[MOST_SORTED];  // candidates: key, then the token's complement
  uint32_t bins[BINS];
  uint32_t chosen[BINS];                  // groups that are read again: slot * READERS + thread
  uint32_t warp_numbers[CHOOSING_WARPS];
  uint32_t low, high, above, n_found, n_chosen;
  float2 rank_sums[MOST_RANKS];           // of the cluster's CTAs
  uint32_t n_of[MOST_RANKS];
  int team;
};
struct TopShared {
  Place places[PLACES];
  Shared teams[TEAMS];
};

template <int ID, int COUNT> __device__ __forceinline__ void bar_sync() { asm volatile("bar.sync %0, %1;" ::"n"(ID), "n"(COUNT) : "memory"); }
template <int ID, int COUNT> __device__ __forceinline__ void bar_arrive() { asm volatile("bar.arrive %0, %1;" ::"n"(ID), "n"(COUNT) : "memory"); }
__device__ __forceinline__ void choosers_meet(int team) {
  if (team) bar_sync<2, CHOOSERS>();
  else bar_sync<1, CHOOSERS>();
}
// Between the readers and the team whose turn it is, for each place: it is full, it may be filled again.
constexpr int BOTH = READERS + CHOOSERS;
static_assert(PLACES == 4, "a case for each place");
__device__ __forceinline__ void wait_full(int p) {
  switch (p) {
    case 0: return bar_sync<3, BOTH>();
    case 1: return bar_sync<4, BOTH>();
    case 2: return bar_sync<5, BOTH>();
    default: return bar_sync<6, BOTH>();
  }
}
__device__ __forceinline__ void say_full(int p) {
  switch (p) {
    case 0: return bar_arrive<3, BOTH>();
    case 1: return bar_arrive<4, BOTH>();
    case 2: return bar_arrive<5, BOTH>();
    default: return bar_arrive<6, BOTH>();
  }
}
__device__ __forceinline__ void wait_empty(int p) {
  switch (p) {
    case 0: return bar_sync<7, BOTH>();
    case 1: return bar_sync<8, BOTH>();
    case 2: return bar_sync<9, BOTH>();
    default: return bar_sync<10, BOTH>();
  }
}
__device__ __forceinline__ void say_empty(int p) {
  switch (p) {
    case 0: return bar_arrive<7, BOTH>();
    case 1: return bar_arrive<8, BOTH>();
    case 2: return bar_arrive<9, BOTH>();
    default: return bar_arrive<10, BOTH>();
  }
}

__device__ __forceinline__ float value_of(uint32_t key) {
  if (key == 0u) return __uint_as_float(0x7fffffffu);
  return __uint_as_float((key & 0x80000000u) ? (key & 0x7fffffffu) : ~key);
}
__device__ __forceinline__ unsigned long long composite(uint32_t key, int token) {
  return (static_cast<unsigned long long>(key) << 32) | (0xffffffffu - uint32_t(token));
}

// One level: the bins of the keys in [low, high] are counted; from the top, the bin at which the count (with `above`, keys over `high`)
// reaches k becomes the range. True once the bins are single keys.
__device__ __forceinline__ bool narrow(Shared& s, int k, int shift, int tid) {
  choosers_meet(s.team);
  if (tid < 32) {
    const int lane = tid;
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
  choosers_meet(s.team);
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

template <typename T, int N>
__device__ __forceinline__ float largest(const uint4 (&raw)[N]) {
  if (sizeof(T) == 4) {
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < N; ++i)
      m = fmaxf(m, fmaxf(fmaxf(__uint_as_float(raw[i].x), __uint_as_float(raw[i].y)), fmaxf(__uint_as_float(raw[i].z), __uint_as_float(raw[i].w))));
    return m;
  }
  __nv_bfloat162 m;   // two at a time; a NaN gives way to a number
  *reinterpret_cast<uint32_t*>(&m) = 0xff80ff80u;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) m = __hmax2(m, *reinterpret_cast<const __nv_bfloat162*>(&w[j]));
  }
  return fmaxf(__low2float(m), __high2float(m));
}

// The row again, from its exact k-th value: at least k of the share's elements reach `reached`, or it is 0.
template <typename T>
__device__ __noinline__ void go_over(Shared& s, const Row<T>& row, int k, uint32_t reached, int tid) {
  constexpr int PER = RowPieces<T>::PER;
  const int lane = tid & 31, warp = tid >> 5;
  auto over = [&](auto&& f) {   // every element of the share: (key, token)
    for (int at = tid; at < row.n; at += CHOOSERS) {
      float v[PER];
      unpack(row.load(at), v, static_cast<const T*>(nullptr));
#pragma unroll
      for (int e = 0; e < PER; ++e) {
        const int token = row.x.first(row.g0 + at) + e;
        if (row.inside(token)) f(logit_key(v[e]), token);
      }
    }
  };
  choosers_meet(s.team);
  if (tid == 0) {
    s.low = reached;
    s.high = 0xffffffffu;
    s.above = 0u;
    s.n_found = 0u;
  }
  choosers_meet(s.team);
  // whether fewer than k lie above `reached`: then it is the k-th value
  uint32_t more = 0u;
  over([&](uint32_t key, int) { more += key > reached ? 1u : 0u; });
  more = __reduce_add_sync(0xffffffffu, more);
  if (lane == 0) atomicAdd(&s.n_found, more);
  choosers_meet(s.team);
  const bool is_kth = s.n_found < uint32_t(k);
  choosers_meet(s.team);
  if (is_kth) {
    if (tid == 0) s.high = s.low;
  } else {
    for (int level = 0; level < LEVELS; ++level) {
      for (int b = tid; b < BINS; b += CHOOSERS) s.bins[b] = 0u;
      choosers_meet(s.team);
      const uint32_t low = s.low, high = s.high;
      const int shift = shift_of(low, high);
      over([&](uint32_t key, int) {
        if (key >= low && key <= high) atomicAdd(&s.bins[(key - low) >> shift], 1u);
      });
      if (narrow(s, k, shift, tid)) break;
    }
  }
  if (tid == 0) s.n_found = 0u;
  choosers_meet(s.team);
  const uint32_t kth = s.low;
  over([&](uint32_t key, int token) {
    if (key > kth) s.found[atomicAdd(&s.n_found, 1u)] = composite(key, token);   // (fewer than k)
  });
  choosers_meet(s.team);
  // equal values in the tokens' order
  int wanted = k - int(s.n_found), have = int(s.n_found);
  for (int base = 0; base < row.n && wanted > 0; base += CHOOSERS) {
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
    choosers_meet(s.team);
    if (lane == 31) s.warp_numbers[warp] = upto;
    choosers_meet(s.team);
    uint32_t before = upto - mine, all = 0u;
    for (int i = 0; i < CHOOSING_WARPS; ++i) {
      before += i < warp ? s.warp_numbers[i] : 0u;
      all += s.warp_numbers[i];
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
  choosers_meet(s.team);
  if (tid == 0) s.n_found = uint32_t(have);
  choosers_meet(s.team);
}

// What a CTA's readers do: shares of rows, round after round, the pieces of the two rounds behind the one in hand on their way, over the rows'
// ends too. Of every share its groups' and pairs' maxima and its warps' sums.
template <typename T, typename ShareOf>
__device__ __forceinline__ void read_shares(TopShared& shared, const ShareOf& share_of, int first_row, int rows, int step, int shift, float c, int tid) {
  constexpr int PAIRS = RowPieces<T>::PER / 2, ROUND = READERS * DEPTH;
  const int together = 1 << shift;
  const uint64_t cc = two_of(c, c);
  // the round that is asked for next
  int next_row = first_row, next_round = 0, next_n = 0;
  const uint4* from = nullptr;
  auto open = [&]() {
    if (next_row >= rows) return;
    const Row<T> row = share_of(next_row);
    next_n = row.n;
    from = reinterpret_cast<const uint4*>(row.x.base) + row.g0 + tid;
  };
  open();
  auto ask = [&](uint4 (&raw)[DEPTH]) {
    if (next_row >= rows) return;
    if ((next_round + 1) * ROUND <= next_n) {
#pragma unroll
      for (int i = 0; i < DEPTH; ++i) raw[i] = load_16(from + i * READERS);
    } else {
#pragma unroll
      for (int i = 0; i < DEPTH; ++i) {
        const uint32_t nothing = sizeof(T) == 4 ? 0xff800000u : 0xff80ff80u;
        raw[i] = make_uint4(nothing, nothing, nothing, nothing);
        if (next_round * ROUND + i * READERS + tid < next_n) raw[i] = load_16(from + i * READERS);
      }
    }
    from += ROUND;
    if (++next_round * ROUND >= next_n) {
      next_row += step;
      next_round = 0;
      open();
    }
  };
  // the round in hand
  int r = first_row, round = 0, rounds = 0, turn = 0, slot = 0, until = together;   // until: rounds that the slot still takes
  float reference = -INFINITY, sum = 0.f;
  uint32_t pair_max = 0u, slot_max = 0u;
  auto take = [&](uint4 (&raw)[DEPTH]) {
    Place& place = shared.places[turn % PLACES];
    if (round == 0) {
      rounds = (share_of(r).n + ROUND - 1) / ROUND;
      if (turn >= PLACES) wait_empty(turn % PLACES);
    }
    const bool last = round + 1 == rounds;
    if (round == 0 || last) {   // the ends of the row
      const Row<T> row = share_of(r);
      if (row.g0 == 0 && round == 0 && tid == 0) blank_outside(raw[0], row.x, 0);
      const int end = row.x.count - 1 - row.g0 - round * ROUND;
#pragma unroll
      for (int i = 0; i < DEPTH; ++i)
        if (end == i * READERS + tid && end + round * ROUND < row.n) blank_outside(raw[i], row.x, row.x.count - 1);
    }
    const float most = largest<T, DEPTH>(raw), up = fminf(most * c, 3e38f);   // (an infinity sums to infinity against any number)
    if (up > reference) {
      sum *= rebase(reference, up);
      reference = up;
    }
    const float minus = -no_less(reference);
    const uint64_t ss = two_of(minus, minus);
    uint64_t acc[DEPTH];
#pragma unroll
    for (int i = 0; i < DEPTH; ++i) {
      uint64_t p[PAIRS];
      unpack_pairs(raw[i], p, static_cast<const T*>(nullptr));
      acc[i] = exp2_two(fma_two(p[0], cc, ss));
#pragma unroll
      for (int j = 1; j < PAIRS; ++j) acc[i] = add_two(acc[i], exp2_two(fma_two(p[j], cc, ss)));
    }
#pragma unroll
    for (int i = 1; i < DEPTH; ++i) acc[0] = add_two(acc[0], acc[i]);
    const float2 both = halves(acc[0]);
    sum += both.x + both.y;
    slot_max = max(slot_max, logit_key(most));
    if (--until == 0 || last) {
      place.groups[slot][tid] = slot_max;
      pair_max = max(pair_max, slot_max);
      slot_max = 0u;
      ++slot;
      until = together;
    }
    ++round;
    if (!last) return;
    pair_max = max(pair_max, __shfl_xor_sync(0xffffffffu, pair_max, 1));
    if ((tid & 1) == 0) place.most[tid >> 1] = pair_max;
    const float common = warp_max(reference);
    sum = warp_sum(sum * rebase(reference, common));
    if ((tid & 31) == 0) place.sums[tid >> 5] = make_float2(common, sum);
    say_full(turn % PLACES);
    reference = -INFINITY;
    sum = 0.f;
    pair_max = 0u;
    round = slot = 0;
    r += step;
    ++turn;
  };
  uint4 one[DEPTH], two[DEPTH];
  ask(one);
  ask(two);
#pragma unroll 1
  while (r < rows) {
    take(one);
    ask(one);
    if (r >= rows) break;
    take(two);
    ask(two);
  }
}

template <typename T>
__global__ void __launch_bounds__(READERS + TEAMS * CHOOSERS, 1)
top_kernel(const TopArgs a) {
  constexpr int PER = RowPieces<T>::PER;
  extern __shared__ __align__(16) uint8_t top_smem[];
  TopShared& shared = *reinterpret_cast<TopShared*>(top_smem);
  pdl_launch_dependents();
  const int ranks = a.ranks, step = int(gridDim.x) / ranks, rank = int(blockIdx.x) % ranks, first_row = int(blockIdx.x) / ranks;
  const float c = 1.44269504f / a.tau;
  auto share_of = [&](int r) {
    Row<T> row = {RowPieces<T>(static_cast<const T*>(a.logits) + (long long)r * a.ld, a.vocab), rank * a.per, 0};
    row.n = max(0, min(a.per, row.x.count - row.g0));
    return row;
  };
  const int most_rounds = (a.per + READERS * DEPTH - 1) / (READERS * DEPTH);
  int shift = 0;   // a group is 2^shift rounds
  while ((SLOTS << shift) < most_rounds) ++shift;
  pdl_wait();

  if (threadIdx.x < READERS) {
    const int tid = int(threadIdx.x);
    read_shares<T>(shared, share_of, first_row, a.rows, step, shift, c, tid);
    if (ranks > 1) {  // (one row to a cluster: the choosers' two barriers)
      cluster_arrive();
      cluster_wait();
      cluster_arrive();
      cluster_wait();
    }
    return;
  }

  const int team = (int(threadIdx.x) - READERS) / CHOOSERS, tid = (int(threadIdx.x) - READERS) % CHOOSERS, lane = tid & 31;
  Shared& s = shared.teams[team];
  if (tid == 0) s.team = team;
  if (team > 0 && ranks > 1) {  // (one row to a cluster, the first team's)
    cluster_arrive();
    cluster_wait();
    cluster_arrive();
    cluster_wait();
    return;
  }
  for (int r = first_row + team * step, turn = team; r < a.rows; r += TEAMS * step, turn += TEAMS) {
    const Row<T> row = share_of(r);
    const int p = turn % PLACES, rounds = (row.n + READERS * DEPTH - 1) / (READERS * DEPTH), slots = (rounds + (1 << shift) - 1) >> shift;
    Place& place = shared.places[p];
    const int first_token = max(0, row.x.first(row.g0)), end_token = min(a.vocab, row.x.first(row.g0) + row.n * PER);
    const int k = min(a.k, end_token - first_token);   // of this share
    choosers_meet(team);   // (the row before has been written out)
    if (tid == 0) s.n_found = s.n_chosen = s.above = 0u;
    wait_full(p);
    float2 part = lane < READING_WARPS ? place.sums[lane] : make_float2(-INFINITY, 0.f);
    float common = warp_max(part.x), total = warp_sum(part.y * rebase(part.x, common));
    uint32_t reached = 0u;
    bool fits = true;
    if (row.n >= READERS) {   // a group for every reader
      // what k pairs' maxima or a few more reach, by halving, in every warp for itself
      constexpr int OWN = PAIRS_OF_READERS / 32;
      uint32_t most[OWN], low = 0xffffffffu, high = 0u;
#pragma unroll
      for (int i = 0; i < OWN; ++i) {
        most[i] = place.most[lane + i * 32];
        low = min(low, most[i]);
        high = max(high, most[i]);
      }
      low = __reduce_min_sync(0xffffffffu, low);
      high = __reduce_max_sync(0xffffffffu, high);
      const int enough = k + max(8, k / 8);
      while (low < high) {
        const uint32_t middle = low + (high - low) / 2 + 1;
        int reach = 0;
#pragma unroll
        for (int i = 0; i < OWN; ++i) reach += most[i] >= middle ? 1 : 0;
        reach = __reduce_add_sync(0xffffffffu, reach);
        if (reach >= k) low = middle;
        else high = middle - 1;
        if (reach >= k && reach <= enough) break;
      }
      reached = low;
      // the groups that reach it
#pragma unroll
      for (int i = 0; i < PAIRS_OF_READERS / CHOOSERS; ++i) {
        const int pair = tid + i * CHOOSERS;
        if (place.most[pair] < reached) continue;
        uint2 both[SLOTS];
#pragma unroll
        for (int g = 0; g < SLOTS; ++g) both[g] = g < slots ? *reinterpret_cast<const uint2*>(&place.groups[g][2 * pair]) : make_uint2(0u, 0u);
#pragma unroll
        for (int g = 0; g < SLOTS; ++g) {
          if (g < slots && both[g].x >= reached) {
            const uint32_t at = atomicAdd(&s.n_chosen, 1u);
            if (at < uint32_t(BINS)) s.chosen[at] = uint32_t(g * READERS + 2 * pair);
          }
          if (g < slots && both[g].y >= reached) {
            const uint32_t at = atomicAdd(&s.n_chosen, 1u);
            if (at < uint32_t(BINS)) s.chosen[at] = uint32_t(g * READERS + 2 * pair + 1);
          }
        }
      }
      choosers_meet(s.team);
      if (r + PLACES * step < a.rows) say_empty(p);
      fits = s.n_chosen <= uint32_t(BINS);
      if (fits) {
        // their pieces again, a piece a thread, several on their way
        const int pieces = int(s.n_chosen) << (shift + 2);
        constexpr int WAY = 4;
        const float reached_value = value_of(reached);
#pragma unroll 1
        for (int p0 = tid; p0 < pieces; p0 += WAY * CHOOSERS) {
          uint4 raw[WAY];
          int at[WAY];
#pragma unroll
          for (int i = 0; i < WAY; ++i) {
            const int piece = p0 + i * CHOOSERS;
            at[i] = row.n;
            if (piece < pieces) {
              const uint32_t group = s.chosen[piece >> (shift + 2)];
              at[i] = ((int(group / READERS) << (shift + 2)) + (piece & ((DEPTH << shift) - 1))) * READERS + int(group % READERS);
            }
            if (at[i] < row.n) raw[i] = row.load(at[i]);
          }
#pragma unroll
          for (int i = 0; i < WAY; ++i) {
            if (at[i] >= row.n) continue;
            float v[PER];
            unpack(raw[i], v, static_cast<const T*>(nullptr));
#pragma unroll
            for (int e = 0; e < PER; ++e) {
              if (!(v[e] >= reached_value)) continue;
              const int token = row.x.first(row.g0 + at[i]) + e;
              if (!row.inside(token)) continue;
              const uint32_t place = atomicAdd(&s.n_found, 1u);
              if (place < uint32_t(CAP)) s.found[place] = composite(logit_key(v[e]), token);
            }
          }
        }
      }
    } else {   // a short share: everything is a candidate, or too many for the list
      choosers_meet(s.team);
      if (r + PLACES * step < a.rows) say_empty(p);
      if (tid == 0) s.n_found = uint32_t(end_token - first_token);
      if (end_token - first_token <= CAP) {
        for (int at = tid; at < row.n; at += CHOOSERS) {
          float v[PER];
          unpack(row.load(at), v, static_cast<const T*>(nullptr));
#pragma unroll
          for (int e = 0; e < PER; ++e) {
            const int token = row.x.first(row.g0 + at) + e;
            if (row.inside(token)) s.found[token - first_token] = composite(logit_key(v[e]), token);
          }
        }
      }
    }
    choosers_meet(s.team);
    if (!fits || s.n_found > uint32_t(CAP)) go_over(s, row, k, reached, tid);
    if (s.n_found < uint32_t(k)) go_over(s, row, k, 0u, tid);   // (fewer than k numbers that are not NaN)

    // the cluster's candidates into its first CTA
    int n = int(s.n_found);
    if (ranks > 1) {
      if (n > MOST_SORTED / MOST_RANKS) {   // (more than the first CTA has places for from each: the exact k)
        go_over(s, row, k, reached, tid);
        n = k;
      }
      cluster_arrive();   // the first CTA has what it found itself in the first of its places, the others are free
      cluster_wait();
      const uint32_t found = cluster_address(s.found, 0), counts = cluster_address(s.n_of, 0), sums = cluster_address(s.rank_sums, 0);
      if (rank > 0)
        for (int i = tid; i < n; i += CHOOSERS)
          asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(found + uint32_t(rank * (MOST_SORTED / MOST_RANKS) + i) * 8u), "l"(s.found[i]) : "memory");
      if (tid == 0) {
        asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(counts + uint32_t(rank) * 4u), "r"(uint32_t(n)) : "memory");
        asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(sums + uint32_t(rank) * 8u), "f"(common), "f"(total) : "memory");
      }
      cluster_arrive();
      cluster_wait();
      if (rank > 0) return;
      part = lane < ranks ? s.rank_sums[lane] : make_float2(-INFINITY, 0.f);
      common = warp_max(part.x);
      total = warp_sum(part.y * rebase(part.x, common));
      int all = n;   // close the gaps
      for (int q = 1; q < ranks; ++q) {
        const int count = int(s.n_of[q]), from = q * (MOST_SORTED / MOST_RANKS);
        constexpr int EACH = MOST_SORTED / MOST_RANKS / CHOOSERS;
        unsigned long long keep[EACH];
#pragma unroll
        for (int i = 0; i < EACH; ++i) keep[i] = tid + i * CHOOSERS < count ? s.found[from + tid + i * CHOOSERS] : 0ull;
        choosers_meet(s.team);
#pragma unroll
        for (int i = 0; i < EACH; ++i)
          if (tid + i * CHOOSERS < count) s.found[all + tid + i * CHOOSERS] = keep[i];
        all += count;
      }
      choosers_meet(s.team);
      n = all;
    }
    if (tid == 0) a.log_sum[r] = (no_less(common) + log2f(total)) * 0.693147181f;

    float* values = a.values + (long long)r * a.k;
    int32_t* ids = a.ids + (long long)r * a.k;
    if (n <= 4 * CHOOSERS) {
      // a candidate's place: how many stand above it
      if ((n & 1) && tid == 0) s.found[n] = 0ull;
      choosers_meet(s.team);
      for (int i = tid; i < n; i += CHOOSERS) {
        const unsigned long long mine = s.found[i];
        int above = 0, also = 0;
#pragma unroll 4
        for (int j = 0; j < n; j += 2) {
          const ulonglong2 two = *reinterpret_cast<const ulonglong2*>(s.found + j);   // (behind the last one stands a 0)
          above += two.x > mine ? 1 : 0;
          also += two.y > mine ? 1 : 0;
        }
        above += also;
        if (above < a.k) {
          values[above] = value_of(uint32_t(mine >> 32));
          ids[above] = int32_t(0xffffffffu - uint32_t(mine & 0xffffffffull));
        }
      }
      continue;
    }
    // many candidates: sorted in place (bitonic, from the largest down)
    int size = 4 * CHOOSERS;
    while (size < n) size *= 2;
    for (int i = n + tid; i < size; i += CHOOSERS) s.found[i] = 0ull;
    choosers_meet(s.team);
    for (int run = 2; run <= size; run *= 2) {
      for (int apart = run / 2; apart > 0; apart /= 2) {
        for (int i = tid; i < size / 2; i += CHOOSERS) {
          const int lo = 2 * i - (i & (apart - 1)), hi = lo + apart;
          const unsigned long long x = s.found[lo], y = s.found[hi];
          if ((x < y) == ((lo & run) == 0)) {
            s.found[lo] = y;
            s.found[hi] = x;
          }
        }
        choosers_meet(s.team);
      }
    }
    for (int i = tid; i < a.k; i += CHOOSERS) {
      values[i] = value_of(uint32_t(s.found[i] >> 32));
      ids[i] = int32_t(0xffffffffu - uint32_t(s.found[i] & 0xffffffffull));
    }
  }
}

template <typename T>
int launch(TopArgs a, int rows, cudaStream_t stream) {
  const int pieces = (a.vocab + 2 * RowPieces<T>::PER - 2) / RowPieces<T>::PER;   // of a row at any alignment, at most
  a.ranks = 1;
  while (a.ranks < MOST_RANKS && (long long)rows * a.ranks * 2 <= 148 && pieces / (2 * a.ranks) >= 1024) a.ranks *= 2;
  a.per = (pieces + a.ranks - 1) / a.ranks;
  if ((long long)rows * a.ranks > 0x7fffffffLL) return R2_BAD_SHAPE;
  static std::atomic<bool> allowed[64];
  const int status = allow_smem(top_kernel<T>, sizeof(TopShared), allowed);
  if (status != R2_OK) return status;
  const int walking = a.ranks > 1 ? rows : min(rows, 148);   // as many as run at a time
  r2_launch_clusters(top_kernel<T>, a.ranks, dim3(unsigned(walking) * unsigned(a.ranks)), dim3(READERS + TEAMS * CHOOSERS), sizeof(TopShared), stream, a);
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
  const TopArgs a = {logits, ld, rows, vocab, k, 1, 0, temperature, values, ids, log_sum};
  return dtype == R2_F32 ? launch<float>(a, rows, stream) : launch<bf16>(a, rows, stream);
}
