// The k largest logits of every row with their tokens, from the largest down, equal values from the lowest token up, and the logarithm of
// the row's sum of exponentials at a temperature.
//
// A row is read once. While it passes, a thread sums exponentials against its own maximum and keeps the maximum of every group of four
// 16-byte pieces, rounded down to bfloat16. What k of the 512 threads' maxima (or a few more) reach is a value that at least k elements reach,
// and what reaches it stands in the groups whose maximum does: little more than k groups of 16 or 32 elements, which are read again and give
// little more than k candidates. Warps sort 32 of them at a time, and a candidate's place is how many stand above it in all of these runs.
// Candidates are compared as unsigned keys in the floats' order, with the token as the lower half.
//
// Rows whose candidates do not fit (thousands of equal values at the edge of the list, or fewer than k numbers that are not NaN) are gone
// over again: the exact k-th value by counts in bins of the keys' range, bin by bin narrower, everything above it, and equal values in the
// order of their tokens until the list is full.
//
// An SM has one CTA. One thread brings: it has rounds of 32 KB copied into three stages, over the rows' ends too, so that memory never waits
// for a row's end. 16 warps read them, and two teams of five choose, in turn: the candidates of two rows are looked for while the next one
// passes. Behind a CTA's last row nothing passes any more, and its readers choose it themselves. Few rows are cut over the CTAs of a cluster,
// whose candidates meet in the first one's shared memory: while twice as many CTAs still have an SM each and 1,024 pieces a share. Short rows
// have a kernel of their own, whose threads hold them: seven rows an SM, or 28 of a warp each.
//
// What bounds it. Bytes: the readers alone take 2,048 float32 rows of 50,257 at 6.6 TB/s, as fast as a copy. With the teams beside them (k 64)
// a pass is 75.7 us (5.45 TB/s): choosing a row is a chain of some 16,000 cycles for a team, as long as two rows take to pass, and the last
// row's 8,000 have nothing beside them. 1,000 bfloat16 rows of 128,001 (k 128): 63.8 us (4.03 TB/s), of which the readers alone take 50 (a copy
// 39): schedulers issue in 56 % of the cycles and the special-function units are busy in 52 %, so neither is full; a round's exponentials wait
// for that round's maximum. A single row of 50,257 (k 5): 6.7 us, 2.6 of them until it is read, the rest the chain: a value by halving, groups, pieces, runs,
// the cluster's hand-over.
// Measured and not taken: readers' loads into their registers (85.2 and 67.1 us: what is on its way is bound by registers and by what shared
// memory leaves of L1), two stages (83.0, 63.7), three teams of three warps (75.6, 64.3) or four (81.2, 62.3), 20 reading warps (79.0, 63.5).
#include "logit_rows.cuh"
#include "sm100_ptx.cuh"

#define R2_ERR_TIMEOUT_ROUND 9

namespace {

constexpr int READERS = 512, READING_WARPS = READERS / 32;
constexpr int CHOOSERS = 160, TEAMS = 2;   // of a team
// Rows that are between reading and choosing. A place is always the same team's: with a place that changed teams, one that is ahead of the
// other would take the readers' word for the other's row as its own.
constexpr int PLACES = 2 * TEAMS;
constexpr int MOST_K = 256, MOST_RANKS = 8;
constexpr int DEPTH = 4;      // pieces of a group
constexpr int STAGES = 3;     // rounds on their way
constexpr int SLOTS = 8;      // groups of a thread (of several rounds each in long rows)
constexpr int CAP = 1536;     // candidates
constexpr int MOST_CHOSEN = 1024, BINS = 512;
constexpr int SHORT_THREADS = 128, SHORT_PIECES = 8;   // of a short row: its threads where a warp does not do, and what each holds
constexpr int LEVELS = 4;     // 9 bits of a 32-bit key at each
struct TopArgs {
  const void* logits; long long ld;
  int rows, vocab, k, ranks, per;
  float tau;
  float* values; int32_t* ids; float* log_sum;
  int* error;
};

// From those who read to those who choose.
struct __align__(16) Place {
  uint16_t groups[SLOTS][READERS];        // the groups' maxima, rounded down to bfloat16
  uint16_t most[READERS];                 // the threads'
  float2 sums[READING_WARPS];             // the warps' references and sums
};
// Of those who choose a row.
template <int N>
struct __align__(16) Lists {
  unsigned long long found[N];            // candidates: key, then the token's complement
  union {
    uint16_t chosen[MOST_CHOSEN];         // groups that are read again: slot * READERS + thread
    uint32_t bins[BINS];
  };
  uint32_t warp_numbers[READING_WARPS];
  uint32_t low, high, above, n_found, n_chosen;
  float2 rank_sums[MOST_RANKS];           // of the cluster's CTAs
  uint32_t n_of[MOST_RANKS];
  int team;
};
using Shared = Lists<CAP>;
struct TopShared {
  uint4 rounds[STAGES][READERS * DEPTH];   // a share's pieces, copied
  Place places[PLACES];
  Shared teams[TEAMS + 1];   // the last one: the readers'
  uint64_t full[STAGES], empty[STAGES];
};
// Clusters have one row, the readers': what they send each other stands in the other places, what the first CTA puts together in the teams'.
static_assert((MOST_RANKS - 1) * MOST_K * sizeof(unsigned long long) <= (PLACES - 1) * sizeof(Place), "");
static_assert(MOST_RANKS * MOST_K * sizeof(unsigned long long) <= TEAMS * sizeof(Shared), "");
static_assert(CHOOSERS != SHORT_THREADS && READERS != SHORT_THREADS, "each has its own barrier");
static_assert(SLOTS * READERS <= 65536 && READERS >= MOST_K && READERS < 1024 && 2 * SLOTS <= 16, "");

template <int ID, int COUNT> __device__ __forceinline__ void bar_sync() { asm volatile("bar.sync %0, %1;" ::"n"(ID), "n"(COUNT) : "memory"); }
template <int ID, int COUNT> __device__ __forceinline__ void bar_arrive() { asm volatile("bar.arrive %0, %1;" ::"n"(ID), "n"(COUNT) : "memory"); }
// those who choose a row: a team, the readers, or all of a short row's
template <int THREADS>
__device__ __forceinline__ void choosers_meet(int team) {
  if (THREADS == 32) __syncwarp();
  else if (THREADS == SHORT_THREADS) __syncthreads();
  else if (THREADS == READERS) bar_sync<11, READERS>();
  else if (team) bar_sync<2, CHOOSERS>();
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

// The logarithm of `total` against `common`; of a row that is nothing against it (FAR_REFERENCE), the largest term's, beside which the others' number
// does not show.
__device__ __forceinline__ float log_sum_of(float common, float total) { return (total != 0.f ? common + log2f(total) : common) * 0.693147181f; }

__device__ __forceinline__ uint32_t floor_bits(float v) { return uint32_t(__bfloat16_as_ushort(__float2bfloat16_rd(v))); }
// bfloat16 bits as 16-bit keys in the numbers' order, and back
__device__ __forceinline__ uint32_t short_key(uint32_t bits) { return (bits & 0x8000u) ? ~bits & 0xffffu : bits | 0x8000u; }
__device__ __forceinline__ __nv_bfloat162 both_of(uint32_t key) {
  const uint32_t bits = (key & 0x8000u) ? key & 0x7fffu : ~key & 0xffffu;
  return __bfloat162bfloat162(__ushort_as_bfloat16(static_cast<unsigned short>(bits)));
}
__device__ __forceinline__ __nv_bfloat162 as_two(uint32_t word) { return *reinterpret_cast<const __nv_bfloat162*>(&word); }
// A piece's elements that are not less than `least`, as bits.
__device__ __forceinline__ uint32_t reaching(const uint4& raw, __nv_bfloat162 both, const float*) {
  const float least = __low2float(both);
  return (__uint_as_float(raw.x) >= least ? 1u : 0u) | (__uint_as_float(raw.y) >= least ? 2u : 0u) | (__uint_as_float(raw.z) >= least ? 4u : 0u) |
         (__uint_as_float(raw.w) >= least ? 8u : 0u);
}
__device__ __forceinline__ uint32_t reaching(const uint4& raw, __nv_bfloat162 both, const bf16*) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  uint32_t bits = 0u;
#pragma unroll
  for (int j = 0; j < 4; ++j) bits |= __hge2_mask(as_two(w[j]), both) & (0x00020001u << (2 * j));
  return (bits | bits >> 16) & 0xffu;
}

// One level: the bins of the keys in [low, high] are counted; from the top, the bin at which the count (with `above`, keys over `high`)
// reaches k becomes the range. True once the bins are single keys.
template <int THREADS, typename L>
__device__ __forceinline__ bool narrow(L& s, int k, int shift, int tid) {
  choosers_meet<THREADS>(s.team);
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
  choosers_meet<THREADS>(s.team);
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
template <typename T, int THREADS, typename L>
__device__ __noinline__ void go_over(L& s, const Row<T>& row, int k, uint32_t reached, int tid) {
  constexpr int PER = RowPieces<T>::PER;
  const int lane = tid & 31, warp = tid >> 5;
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
  choosers_meet<THREADS>(s.team);
  if (tid == 0) {
    s.low = reached;
    s.high = 0xffffffffu;
    s.above = 0u;
    s.n_found = 0u;
  }
  choosers_meet<THREADS>(s.team);
  // whether fewer than k lie above `reached`: then it is the k-th value
  uint32_t more = 0u;
  over([&](uint32_t key, int) { more += key > reached ? 1u : 0u; });
  more = __reduce_add_sync(0xffffffffu, more);
  if (lane == 0) atomicAdd(&s.n_found, more);
  choosers_meet<THREADS>(s.team);
  const bool is_kth = s.n_found < uint32_t(k);
  choosers_meet<THREADS>(s.team);
  if (is_kth) {
    if (tid == 0) s.high = s.low;
  } else {
    for (int level = 0; level < LEVELS; ++level) {
      for (int b = tid; b < BINS; b += THREADS) s.bins[b] = 0u;
      choosers_meet<THREADS>(s.team);
      const uint32_t low = s.low, high = s.high;
      const int shift = shift_of(low, high);
      over([&](uint32_t key, int) {
        if (key >= low && key <= high) atomicAdd(&s.bins[(key - low) >> shift], 1u);
      });
      if (narrow<THREADS>(s, k, shift, tid)) break;
    }
  }
  if (tid == 0) s.n_found = 0u;
  choosers_meet<THREADS>(s.team);
  const uint32_t kth = s.low;
  over([&](uint32_t key, int token) {
    if (key > kth) s.found[atomicAdd(&s.n_found, 1u)] = composite(key, token);   // (fewer than k)
  });
  choosers_meet<THREADS>(s.team);
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
    choosers_meet<THREADS>(s.team);
    if (lane == 31) s.warp_numbers[warp] = upto;
    choosers_meet<THREADS>(s.team);
    uint32_t before = upto - mine, all = 0u;
    for (int i = 0; i < THREADS / 32; ++i) {
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
  choosers_meet<THREADS>(s.team);
  if (tid == 0) s.n_found = uint32_t(have);
  choosers_meet<THREADS>(s.team);
}

// What a CTA's bringing thread does: shares of rows, round after round, over the rows' ends too, into the stages that have been read.
template <typename T, typename ShareOf>
__device__ __forceinline__ void bring_shares(TopShared& shared, const ShareOf& share_of, int first_row, int rows, int step, int* error) {
  constexpr int ROUND = READERS * DEPTH;
  int n = 0;
  for (int r = first_row; r < rows; r += step) {
    const Row<T> row = share_of(r);
    const uint4* from = reinterpret_cast<const uint4*>(row.x.base) + row.g0;
    for (int left = row.n; left > 0; left -= ROUND, from += ROUND, ++n) {
      const int stage = n % STAGES;
      if (n >= STAGES && !r2ptx::mbar_wait(r2ptx::smem_u32(&shared.empty[stage]), uint32_t(n / STAGES - 1) & 1u)) {
        atomicMax(error, R2_ERR_TIMEOUT_ROUND);
        return;
      }
      const uint32_t bytes = uint32_t(min(left, ROUND)) * 16u, barrier = r2ptx::smem_u32(&shared.full[stage]);
      r2ptx::mbar_expect_tx(barrier, bytes);
      asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                       r2ptx::smem_u32(shared.rounds[stage])), "l"(from), "r"(bytes), "r"(barrier)
                   : "memory");
    }
  }
}

// (Out of the loop's way. The place's next copy comes by another path than what is written here.)
template <typename T>
__device__ __noinline__ void blank_in(uint4& place, const RowPieces<T>& x, int g) {
  uint4 piece = place;
  blank_outside(piece, x, g);
  place = piece;
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// What its readers do. Of every share its groups' and threads' maxima and its warps' sums. -> the turn of the last one.
template <typename T, typename ShareOf>
__device__ __forceinline__ int read_shares(TopShared& shared, const ShareOf& share_of, int first_row, int rows, int step, int shift, float c, int tid,
                                           int* error) {
  constexpr int PAIRS = RowPieces<T>::PER / 2, ROUND = READERS * DEPTH;
  const int together = 1 << shift;
  const uint64_t cc = two_of(c, c);
  uint32_t stage = 0u, phase = 0u;
  bool lost = false;
  // the round in hand
  int r = first_row, left = 0, turn = 0, slot = 0, until = together;   // left: pieces from its first one on; until: rounds that the slot still takes
  float reference = -INFINITY, sum = 0.f;
  float row_max = -INFINITY, slot_max = -INFINITY;
#pragma unroll 1
  while (r < rows) {
    Place& place = shared.places[turn % PLACES];
    bool begins = false;
    if (left == 0) {
      const Row<T> row = share_of(r);
      left = row.n;
      begins = row.g0 == 0;
      if (turn >= PLACES) wait_empty(turn % PLACES);
    }
    const bool last = left <= ROUND;
    const int end = left - 1 - tid;   // the share's last piece is this thread's i-th where i * READERS == end
    if (!lost && !r2ptx::mbar_wait(r2ptx::smem_u32(&shared.full[stage]), phase)) {
      lost = true;
      atomicMax(error, R2_ERR_TIMEOUT_ROUND);
    }
    if (begins && tid == 0) blank_in(shared.rounds[stage][0], share_of(r).x, 0);   // the ends of the row
    if (last && end >= 0 && end % READERS == 0) {
      const Row<T> row = share_of(r);
      if (row.g0 + row.n == row.x.count) blank_in(shared.rounds[stage][left - 1], row.x, row.x.count - 1);
    }
    uint4 raw[DEPTH];
    if (!last) {
#pragma unroll
      for (int i = 0; i < DEPTH; ++i) raw[i] = shared.rounds[stage][i * READERS + tid];
    } else {
      const uint32_t nothing = sizeof(T) == 4 ? 0xff800000u : 0xff80ff80u;
#pragma unroll
      for (int i = 0; i < DEPTH; ++i) {
        raw[i] = make_uint4(nothing, nothing, nothing, nothing);
        if (i * READERS <= end) raw[i] = shared.rounds[stage][i * READERS + tid];
      }
    }
    __syncwarp();
    if ((tid & 31) == 0) r2ptx::mbar_arrive(r2ptx::smem_u32(&shared.empty[stage]));
    if (++stage == STAGES) {
      stage = 0u;
      phase ^= 1u;
    }
    const float most = largest<T, DEPTH>(raw), up = fminf(most * c, 3e38f);   // (an infinity sums to infinity against any number)
    if (up > reference) {
      sum *= rebase(reference, up);
      reference = up;
    }
    const float minus = shift_to(reference);
    const uint64_t ss = two_of(minus, minus);
    auto sum_of = [&](const uint4& piece) {
      uint64_t p[PAIRS];
      unpack_pairs(piece, p, static_cast<const T*>(nullptr));
      uint64_t acc = exp2_two(fma_two(p[0], cc, ss));
#pragma unroll
      for (int j = 1; j < PAIRS; ++j) acc = add_two(acc, exp2_two(fma_two(p[j], cc, ss)));
      return acc;
    };
    uint64_t acc = 0ull;
    if (!last) {
      uint64_t of[DEPTH];
#pragma unroll
      for (int i = 0; i < DEPTH; ++i) of[i] = sum_of(raw[i]);
      acc = add_two(add_two(of[0], of[1]), add_two(of[2], of[3]));
    } else {
#pragma unroll
      for (int i = 0; i < DEPTH; ++i)
        if (i * READERS <= end) acc = add_two(acc, sum_of(raw[i]));
    }
    const float2 both = halves(acc);
    sum += both.x + both.y;
    slot_max = fmaxf(slot_max, most);
    if (--until == 0 || last) {
      place.groups[slot][tid] = uint16_t(floor_bits(slot_max));
      row_max = fmaxf(row_max, slot_max);
      slot_max = -INFINITY;
      ++slot;
      until = together;
    }
    left -= ROUND;
    if (!last) continue;
    place.most[tid] = uint16_t(floor_bits(row_max));
    const float common = warp_max(reference);
    sum = warp_sum(sum * rebase(reference, common));
    if ((tid & 31) == 0) place.sums[tid >> 5] = make_float2(common, sum);
    r += step;
    if (r < rows) say_full(turn % PLACES);   // (the last one is the readers' own)
    reference = -INFINITY;
    sum = 0.f;
    row_max = -INFINITY;
    left = slot = 0;
    ++turn;
  }
  if (lost) {  // (copies still under way get as long again: one of a barrier's two phases is always over)
    for (int i = 0; i < STAGES; ++i)
      for (uint32_t of = 0u; of < 2u; ++of) r2ptx::mbar_wait(r2ptx::smem_u32(&shared.full[i]), of);
  }
  return turn - 1;
}

// A warp's values from the largest down.
__device__ __forceinline__ unsigned long long sorted(unsigned long long v, int lane) {
#pragma unroll
  for (int run = 2; run <= 32; run *= 2) {
#pragma unroll
    for (int apart = run / 2; apart > 0; apart /= 2) {
      const unsigned long long other = __shfl_xor_sync(0xffffffffu, v, apart);
      const bool larger = ((lane & run) == 0) == ((lane & apart) == 0);   // this lane keeps the larger one
      if (larger == (other > v)) v = other;
    }
  }
  return v;
}
// How many of a run of 32 stand above `mine`.
__device__ __forceinline__ int above_in(const unsigned long long* run, unsigned long long mine) {
  int at = 0;
#pragma unroll
  for (int step = 16; step > 0; step /= 2) at += run[at + step - 1] > mine ? step : 0;
  return at + (run[at] > mine ? 1 : 0);
}
// What stands at place `above` of a list's runs: f(above, candidate), for the first k.
template <int THREADS, typename F>
__device__ __forceinline__ void in_order(const unsigned long long* list, int n, int k, int tid, F&& f) {
  for (int i = tid; i < n; i += THREADS) {
    const unsigned long long mine = list[i];
    int above = 0;
#pragma unroll 4
    for (int run = 0; run < n; run += 32) above += above_in(list + run, mine);
    if (mine != 0ull && above < k) f(above, mine);
  }
}
template <int THREADS>
__device__ __forceinline__ void write_list(const TopArgs& a, int r, const unsigned long long* list, int n, int tid) {
  float* values = a.values + (long long)r * a.k;
  int32_t* ids = a.ids + (long long)r * a.k;
  in_order<THREADS>(list, n, a.k, tid, [&](int at, unsigned long long entry) {
    values[at] = value_of(uint32_t(entry >> 32));
    ids[at] = int32_t(0xffffffffu - uint32_t(entry & 0xffffffffull));
  });
}
// Places on a list for every thread's `mine` entries, one atomic a warp. -> the first one's.
__device__ __forceinline__ uint32_t places_for(uint32_t mine, uint32_t* count, int lane) {
  uint32_t upto = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint32_t other = __shfl_up_sync(0xffffffffu, upto, d);
    if (lane >= d) upto += other;
  }
  uint32_t base = 0u;
  if (lane == 31) base = atomicAdd(count, upto);
  return __shfl_sync(0xffffffffu, base, 31) + upto - mine;
}

// A row's k, from its share's maxima and sums; `released` once the place is no longer read. (A cluster's shares are chosen by readers.)
template <typename T, int THREADS, typename Released>
__device__ __forceinline__ void choose(const TopArgs& a, TopShared& shared, Shared& s, const Place& place, const Row<T>& row, int r, int shift, int rank,
                                       int tid, const Released& released) {
  constexpr int PER = RowPieces<T>::PER;
  const int lane = tid & 31, warp = tid >> 5, slots = ((row.n + READERS * DEPTH - 1) / (READERS * DEPTH) + (1 << shift) - 1) >> shift;
  const int first_token = max(0, row.x.first(row.g0)), end_token = min(a.vocab, row.x.first(row.g0) + row.n * PER);
  const int k = min(a.k, end_token - first_token);   // of this share
  float common = 0.f, total = 0.f;   // (the second warp's)
  auto write_sum = [&]() {
    if (lane == 0) a.log_sum[r] = log_sum_of(common, total);
  };
  if (warp == 1) {
    const float2 part = lane < READING_WARPS ? place.sums[lane] : make_float2(-INFINITY, 0.f);
    common = warp_max(part.x);
    total = warp_sum(part.y * rebase(part.x, common));
    if (a.ranks == 1) write_sum();
  }
  // what k threads' maxima or a few more reach, three values tried at a time (their counts in ten bits each)
  const uint32_t* most = reinterpret_cast<const uint32_t*>(place.most);
  if (warp == 0) {
    constexpr int OWN = READERS / 64;   // pairs
    __nv_bfloat162 own[OWN], least, largest;
#pragma unroll
    for (int i = 0; i < OWN; ++i) {
      own[i] = as_two(most[lane + i * 32]);
      least = i == 0 ? own[i] : __hmin2(least, own[i]);
      largest = i == 0 ? own[i] : __hmax2(largest, own[i]);
    }
    least = __halves2bfloat162(__hmin(__low2bfloat16(least), __high2bfloat16(least)), __hmax(__low2bfloat16(largest), __high2bfloat16(largest)));
    uint32_t low = __reduce_min_sync(0xffffffffu, short_key(__bfloat16_as_ushort(__low2bfloat16(least))));
    uint32_t high = __reduce_max_sync(0xffffffffu, short_key(__bfloat16_as_ushort(__high2bfloat16(least))));
    const int enough = k + max(8, k / 8);
    while (low < high) {
      const uint32_t half = (high - low) / 2, one = low + half / 2 + 1, two = low + half + 1, three = two + half / 2;   // all in (low, high]
      const __nv_bfloat162 of_key[3] = {both_of(one), both_of(two), both_of(three)};
      uint32_t reach = 0u;
#pragma unroll
      for (int t = 0; t < 3; ++t) {
        __nv_bfloat162 count = __hge2(own[0], of_key[t]);
#pragma unroll
        for (int i = 1; i < OWN; ++i) count = __hadd2(count, __hge2(own[i], of_key[t]));
        reach += uint32_t(__low2float(count) + __high2float(count)) << (10 * t);
      }
      reach = __reduce_add_sync(0xffffffffu, reach);
      const int of_one = int(reach & 1023u), of_two = int((reach >> 10) & 1023u), of_three = int(reach >> 20);
      int of_low = 0;
      if (of_three >= k) {
        low = three;
        of_low = of_three;
      } else if (of_two >= k) {
        low = two;
        high = three - 1;
        of_low = of_two;
      } else if (of_one >= k) {
        low = one;
        high = two - 1;
        of_low = of_one;
      } else {
        high = one - 1;
      }
      if (of_low >= k && of_low <= enough) break;
    }
    if (lane == 0) s.low = low;
  }
  choosers_meet<THREADS>(s.team);
  const __nv_bfloat162 least = both_of(s.low);
  const uint32_t reached = logit_key(__low2float(least));
  // the groups that reach it
  constexpr int EACH = (READERS / 2 + THREADS - 1) / THREADS;
  uint32_t hits[EACH], mine = 0u;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int pair = tid + i * THREADS;
    hits[i] = 0u;
    if (pair < READERS / 2 && __hge2_mask(as_two(most[pair]), least) != 0u) {
#pragma unroll
      for (int g = 0; g < SLOTS; ++g)
        if (g < slots) hits[i] |= __hge2_mask(as_two(reinterpret_cast<const uint32_t*>(place.groups[g])[pair]), least) & (0x00020001u << (2 * g));
      hits[i] = (hits[i] | hits[i] >> 16) & 0xffffu;
    }
    mine += uint32_t(__popc(hits[i]));
  }
  if (__any_sync(0xffffffffu, mine != 0u)) {
    uint32_t at = places_for(mine, &s.n_chosen, lane);
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      for (uint32_t left = hits[i]; left != 0u; left &= left - 1u, ++at) {
        const int bit = __ffs(int(left)) - 1;
        if (at < uint32_t(MOST_CHOSEN)) s.chosen[at] = uint16_t((bit >> 1) * READERS + 2 * (tid + i * THREADS) + (bit & 1));
      }
    }
  }
  choosers_meet<THREADS>(s.team);
  released();
  const bool fits = s.n_chosen <= uint32_t(MOST_CHOSEN);
  if (fits) {
    // their pieces again, a piece a thread, several on their way
    const int pieces = int(s.n_chosen) << (shift + 2);
    constexpr int WAY = 2;
#pragma unroll 1
    for (int p0 = 0; p0 < pieces; p0 += WAY * THREADS) {
      uint4 raw[WAY];
      int at[WAY];
      uint32_t found = 0u;   // elements that reach it
#pragma unroll
      for (int i = 0; i < WAY; ++i) {
        const int piece = p0 + tid + i * THREADS;
        at[i] = row.n;
        if (piece < pieces) {
          const uint32_t group = s.chosen[piece >> (shift + 2)];
          at[i] = ((int(group / READERS) << (shift + 2)) + (piece & ((DEPTH << shift) - 1))) * READERS + int(group % READERS);
        }
        if (at[i] < row.n) raw[i] = load_once(row.x, row.g0 + at[i]);
      }
#pragma unroll
      for (int i = 0; i < WAY; ++i) {
        if (at[i] >= row.n) continue;
        const int first = row.x.first(row.g0 + at[i]);
        uint32_t bits = reaching(raw[i], least, static_cast<const T*>(nullptr));
        if (first < 0) bits &= ~0u << -first;
        if (first + PER > a.vocab) bits &= (1u << (a.vocab - first)) - 1u;
        found |= bits << (i * PER);
      }
      if (!__any_sync(0xffffffffu, found != 0u)) continue;
      uint32_t to = places_for(uint32_t(__popc(found)), &s.n_found, lane);
#pragma unroll 1
      for (; found != 0u; found &= found - 1u, ++to) {   // (few of a thread: their words are picked out of its registers)
        const int bit = __ffs(int(found)) - 1, i = bit / PER, e = bit % PER, w = e * 4 / PER;
        uint4 piece = raw[0];
        int from = at[0];
#pragma unroll
        for (int o = 1; o < WAY; ++o) {
          if (o == i) {
            piece = raw[o];
            from = at[o];
          }
        }
        const uint32_t word = (w & 2) ? ((w & 1) ? piece.w : piece.z) : ((w & 1) ? piece.y : piece.x);
        const float v = __uint_as_float(PER == 4 ? word : (e & 1) ? word & 0xffff0000u : word << 16);
        if (to < uint32_t(CAP)) s.found[to] = composite(logit_key(v), row.x.first(row.g0 + from) + e);
      }
    }
  }
  choosers_meet<THREADS>(s.team);
  if (!fits || s.n_found > uint32_t(CAP)) go_over<T, THREADS>(s, row, k, reached, tid);
  if (s.n_found < uint32_t(k)) go_over<T, THREADS>(s, row, k, 0u, tid);   // (fewer than k numbers that are not NaN)

  // runs of 32 from the largest down, filled up with 0
  unsigned long long* list = s.found;
  int n = (int(s.n_found) + 31) / 32 * 32;
  for (int i = tid; i < n; i += THREADS) list[i] = sorted(i < int(s.n_found) ? list[i] : 0ull, lane);
  choosers_meet<THREADS>(s.team);
  if (THREADS == READERS && a.ranks > 1) {
    unsigned long long* sent = reinterpret_cast<unsigned long long*>(&shared.places[1]);   // by the other CTAs, MOST_K places each
    cluster_wait();   // (the first CTA runs)
    const uint32_t to = cluster_address(sent, 0) + uint32_t(max(0, rank - 1) * MOST_K) * 8u;
    auto send = [&](int at, unsigned long long v) {
      if (rank > 0) asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(to + uint32_t(at) * 8u), "l"(v) : "memory");
      else reinterpret_cast<unsigned long long*>(&shared.teams[0])[at] = v;
    };
    if (n <= MOST_K) {
      for (int i = tid; i < n; i += THREADS) send(i, list[i]);
    } else {   // the first k of them, in order
      in_order<THREADS>(list, n, a.k, tid, send);
      n = (k + 31) / 32 * 32;
      if (tid < n - k) send(k + tid, 0ull);
    }
    if (tid == 32) {
      asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cluster_address(s.n_of, 0) + uint32_t(rank) * 4u), "r"(uint32_t(n)) : "memory");
      asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(cluster_address(s.rank_sums, 0) + uint32_t(rank) * 8u), "f"(common), "f"(total) : "memory");
    }
    cluster_arrive();
    cluster_wait();
    if (rank > 0) return;
    if (warp == 1) {
      const float2 part = lane < a.ranks ? s.rank_sums[lane] : make_float2(-INFINITY, 0.f);
      common = warp_max(part.x);
      total = warp_sum(part.y * rebase(part.x, common));
      write_sum();
    }
    list = reinterpret_cast<unsigned long long*>(&shared.teams[0]);
    static_assert(READERS >= MOST_K, "one of a CTA's candidates a thread");
#pragma unroll 1
    for (int q = 1; q < a.ranks; ++q) {
      const int count = int(s.n_of[q]);
      if (tid < count) list[n + tid] = sent[(q - 1) * MOST_K + tid];
      n += count;
    }
    choosers_meet<THREADS>(s.team);
  }
  write_list<THREADS>(a, r, list, n, tid);
}

template <typename T>
__global__ void __launch_bounds__(READERS + TEAMS * CHOOSERS + 32, 1)
top_kernel(const TopArgs a) {
  extern __shared__ __align__(16) uint8_t top_smem[];
  TopShared& shared = *reinterpret_cast<TopShared*>(top_smem);
  pdl_launch_dependents();
  if (a.ranks > 1) cluster_arrive();   // (waited for before anything is sent)
  const int ranks = a.ranks, step = int(gridDim.x) / ranks, rank = int(blockIdx.x) % ranks, first_row = int(blockIdx.x) / ranks;
  auto share_of = [&](int r) {
    Row<T> row = {RowPieces<T>(static_cast<const T*>(a.logits) + (long long)r * a.ld, a.vocab), rank * a.per, 0};
    row.n = max(0, min(a.per, row.x.count - row.g0));
    return row;
  };
  const int most_rounds = (a.per + READERS * DEPTH - 1) / (READERS * DEPTH);
  int shift = 0;   // a group is 2^shift rounds
  while ((SLOTS << shift) < most_rounds) ++shift;

  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      r2ptx::mbar_init(r2ptx::smem_u32(&shared.full[i]), 1u);
      r2ptx::mbar_init(r2ptx::smem_u32(&shared.empty[i]), uint32_t(READING_WARPS));
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();

  if (threadIdx.x >= TEAMS * CHOOSERS + 32) {
    const int tid = int(threadIdx.x) - TEAMS * CHOOSERS - 32;
    Shared& s = shared.teams[TEAMS];
    if (tid == 0) {
      s.team = TEAMS;
      s.n_found = s.n_chosen = s.above = 0u;
    }
    pdl_wait();
    const int turn = read_shares<T>(shared, share_of, first_row, a.rows, step, shift, 1.44269504f / a.tau, tid, a.error), r = first_row + turn * step;
    choosers_meet<READERS>(TEAMS);
    choose<T, READERS>(a, shared, s, shared.places[turn % PLACES], share_of(r), r, shift, rank, tid, [] {});
    return;
  }

  const int team = int(threadIdx.x) / CHOOSERS, tid = int(threadIdx.x) % CHOOSERS;   // TEAMS: who brings
  if (team < TEAMS && tid == 0 && ranks == 1) shared.teams[team].team = team;
  pdl_wait();
  if (team == TEAMS) {
    if (tid == 0) bring_shares<T>(shared, share_of, first_row, a.rows, step, a.error);
    __syncwarp();
  }
  for (int r = team < TEAMS ? first_row + team * step : a.rows, turn = team; r + step < a.rows; r += TEAMS * step, turn += TEAMS) {
    Shared& s = shared.teams[team];
    const int p = turn % PLACES;
    choosers_meet<CHOOSERS>(team);   // (the row before has been written out)
    if (tid == 0) s.n_found = s.n_chosen = s.above = 0u;
    wait_full(p);
    choose<T, CHOOSERS>(a, shared, s, shared.places[p], share_of(r), r, shift, rank, tid, [&] {
      if (r + PLACES * step < a.rows) say_empty(p);
    });
  }
  if (ranks > 1) {  // (one row to a cluster: its readers' barriers)
    cluster_wait();
    cluster_arrive();
    cluster_wait();
  }
}

template <typename T>
__device__ __noinline__ uint4 blanked(uint4 raw, RowPieces<T> x, int g) {   // (out of the way)
  blank_outside(raw, x, g);
  return raw;
}

// A short row, which its threads hold: a warp, or four. Nothing is read again, and an SM has as many rows in hand as registers allow.
template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS, THREADS == 32 ? 28 : 7)
top_short_kernel(const TopArgs a) {
  constexpr int PER = RowPieces<T>::PER, PAIRS = PER / 2, WARPS = THREADS / 32, HOLDS = SHORT_PIECES;
  constexpr int MOST = THREADS == 32 ? 512 : 1024;
  __shared__ Lists<MOST> s;
  __shared__ float2 sums[WARPS];
  pdl_launch_dependents();
  const int tid = int(threadIdx.x), lane = tid & 31, warp = tid >> 5, r = int(blockIdx.x);
  if (tid == 0) {
    s.team = 0;
    s.n_found = s.above = 0u;
  }
  choosers_meet<THREADS>(0);
  pdl_wait();
  Row<T> row = {RowPieces<T>(static_cast<const T*>(a.logits) + (long long)r * a.ld, a.vocab), 0, 0};
  row.n = row.x.count;
  const int n = row.n, k = a.k;
  const uint32_t nothing = sizeof(T) == 4 ? 0xff800000u : 0xff80ff80u;
  uint4 raw[HOLDS];
#pragma unroll
  for (int i = 0; i < HOLDS; ++i) {
    raw[i] = make_uint4(nothing, nothing, nothing, nothing);
    load_16_if(raw[i], reinterpret_cast<const uint4*>(row.x.base) + i * THREADS + tid, i * THREADS + tid < n);
  }
#pragma unroll
  for (int i = 0; i < HOLDS; ++i)
    if (i * THREADS + tid == n - 1 || (i == 0 && tid == 0)) raw[i] = blanked(raw[i], row.x, i * THREADS + tid);

  // sums, and the maxima of the pieces
  const float c = 1.44269504f / a.tau;
  float most[HOLDS], row_most = -INFINITY;
#pragma unroll
  for (int i = 0; i < HOLDS; ++i) {
    const uint4 one[1] = {raw[i]};
    most[i] = largest<T, 1>(one);
    row_most = fmaxf(row_most, most[i]);
  }
  const float reference = warp_max(fminf(row_most * c, 3e38f)), minus = shift_to(reference);
  const uint64_t cc = two_of(c, c), ss = two_of(minus, minus);
  uint64_t acc = 0ull;
#pragma unroll
  for (int i = 0; i < HOLDS; ++i) {
    if (i * THREADS + warp * 32 >= n) continue;
    uint64_t p[PAIRS];
    unpack_pairs(raw[i], p, static_cast<const T*>(nullptr));
#pragma unroll
    for (int j = 0; j < PAIRS; ++j) acc = add_two(acc, exp2_two(fma_two(p[j], cc, ss)));
  }
  const float2 both = halves(acc);
  float common = reference, total = warp_sum(both.x + both.y);
  if (WARPS > 1) {
    if (lane == 0) sums[warp] = make_float2(common, total);
    __syncthreads();
    const float2 part = lane < WARPS ? sums[lane] : make_float2(-INFINITY, 0.f);
    common = warp_max(part.x);
    total = warp_sum(part.y * rebase(part.x, common));
  }
  if (tid == 0) a.log_sum[r] = log_sum_of(common, total);

  // what k pieces' maxima reach, or k numbers where there are not twice as many pieces: two values tried at a time (counts in 16 bits each)
  const bool fine = n < 2 * k;
  uint32_t low = 0x7fu, high = 0xff80u;   // -inf, inf
  const int enough = k + max(8, k / 8);
  for (int turn = 0; low < high; turn ^= 1) {
    const uint32_t third = (high - low) / 3, one = low + third + 1, two = high - third;   // in (low, high], one <= two
    const __nv_bfloat162 of_one = both_of(one), of_two = both_of(two);
    const float least_one = __low2float(of_one), least_two = __low2float(of_two);
    uint32_t reach = 0u;
    if (fine) {
#pragma unroll
      for (int i = 0; i < HOLDS; ++i) {
        if (i * THREADS + warp * 32 >= n) continue;
        reach += uint32_t(__popc(reaching(raw[i], of_one, static_cast<const T*>(nullptr)))) +
                 (uint32_t(__popc(reaching(raw[i], of_two, static_cast<const T*>(nullptr)))) << 16);
      }
    } else {
#pragma unroll
      for (int i = 0; i < HOLDS; ++i) reach += (most[i] >= least_one ? 1u : 0u) + (most[i] >= least_two ? 1u << 16 : 0u);
    }
    reach = __reduce_add_sync(0xffffffffu, reach);
    if (WARPS > 1) {
      if (lane == 0) s.bins[turn * WARPS + warp] = reach;
      __syncthreads();
      reach = 0u;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) reach += s.bins[turn * WARPS + w];
    }
    const int reach_one = int(reach & 0xffffu), reach_two = int(reach >> 16);
    int of_low = 0;
    if (reach_two >= k) {
      low = two;
      of_low = reach_two;
    } else if (reach_one >= k) {
      low = one;
      high = two - 1;
      of_low = reach_one;
    } else {
      high = one - 1;
    }
    if (of_low >= k && of_low <= enough) break;
  }
  const __nv_bfloat162 least = both_of(low);
  uint32_t bits[HOLDS], mine = 0u;
#pragma unroll
  for (int i = 0; i < HOLDS; ++i) {
    const int at = i * THREADS + tid, first = row.x.first(at);
    bits[i] = at < n ? reaching(raw[i], least, static_cast<const T*>(nullptr)) : 0u;
    if (first < 0) bits[i] &= ~0u << -first;
    if (first < a.vocab && first + PER > a.vocab) bits[i] &= (1u << (a.vocab - first)) - 1u;
    mine += uint32_t(__popc(bits[i]));
  }
  uint32_t to = places_for(mine, &s.n_found, lane);
#pragma unroll
  for (int i = 0; i < HOLDS; ++i) {
#pragma unroll 1
    for (uint32_t left = bits[i]; left != 0u; left &= left - 1u, ++to) {
      const int e = __ffs(int(left)) - 1, w = e * 4 / PER;
      const uint32_t word = (w & 2) ? ((w & 1) ? raw[i].w : raw[i].z) : ((w & 1) ? raw[i].y : raw[i].x);
      const float v = __uint_as_float(PER == 4 ? word : (e & 1) ? word & 0xffff0000u : word << 16);
      if (to < uint32_t(MOST)) s.found[to] = composite(logit_key(v), row.x.first(i * THREADS + tid) + e);
    }
  }
  choosers_meet<THREADS>(0);
  const uint32_t reached = logit_key(__low2float(least));
  if (s.n_found > uint32_t(MOST)) go_over<T, THREADS>(s, row, k, reached, tid);
  if (s.n_found < uint32_t(k)) go_over<T, THREADS>(s, row, k, 0u, tid);   // (fewer than k numbers that are not NaN)
  const int filled = (int(s.n_found) + 31) / 32 * 32;
  for (int i = tid; i < filled; i += THREADS) s.found[i] = sorted(i < int(s.n_found) ? s.found[i] : 0ull, lane);
  choosers_meet<THREADS>(0);
  write_list<THREADS>(a, r, s.found, filled, tid);
}

template <typename T>
int launch(TopArgs a, int rows, cudaStream_t stream) {
  const int pieces = (a.vocab + 2 * RowPieces<T>::PER - 2) / RowPieces<T>::PER;   // of a row at any alignment, at most
  // Rows that 128 threads hold in their registers (4,096 rows of 4,000 float32 numbers, k 64: 37.3 us, the other kernel 69.7; 16 rows 6.0, 5.9). One
  // warp where that does, there is a row for every scheduler and k is not large (4,096 rows of 300, k 10: 8.2 us, 128 threads 19.5; but 300 rows
  // of 1,000, k 100: 9.8, 9.0; 2,000 of them, k 128: 25.8, 24.6, k 256: 37.5, 31.4).
  if (pieces <= SHORT_PIECES * SHORT_THREADS) {
    if (pieces <= SHORT_PIECES * 32 && rows >= 4 * 148 && a.k <= 128) r2_launch(top_short_kernel<T, 32>, dim3(unsigned(rows)), dim3(32), size_t(0), stream, a);
    else r2_launch(top_short_kernel<T, SHORT_THREADS>, dim3(unsigned(rows)), dim3(SHORT_THREADS), size_t(0), stream, a);
    return launch_status();
  }
  a.ranks = 1;
  while (a.ranks < MOST_RANKS && (long long)rows * a.ranks * 2 <= 148 && pieces / (2 * a.ranks) >= 1024) a.ranks *= 2;
  a.per = (pieces + a.ranks - 1) / a.ranks;
  if ((long long)rows * a.ranks > 0x7fffffffLL) return R2_BAD_SHAPE;
  static std::atomic<bool> allowed[64];
  const int status = allow_smem(top_kernel<T>, sizeof(TopShared), allowed);
  if (status != R2_OK) return status;
  const int walking = a.ranks > 1 ? rows : min(rows, 148);   // as many as run at a time
  r2_launch_clusters(top_kernel<T>, a.ranks, dim3(unsigned(walking) * unsigned(a.ranks)), dim3(READERS + TEAMS * CHOOSERS + 32), sizeof(TopShared), stream, a);
  return launch_status();
}

}  // namespace

// logits [rows, vocab] of dtype with row stride ld -> values [rows, k] float, ids [rows, k], log_sum [rows].
extern "C" int r2_top_logits(int dtype, const void* logits, long long ld, int rows, int vocab, int k, float temperature, float* values,
                             int32_t* ids, float* log_sum, int* error, cudaStream_t stream) {
  if (dtype != R2_F32 && dtype != R2_BF16) return R2_BAD_DTYPE;
  if (rows < 0 || vocab < 1 || vocab > (1 << 30) || ld < vocab || k < 1 || k > vocab) return R2_BAD_SHAPE;
  if (k > MOST_K || !(temperature > 0.f)) return R2_UNSUPPORTED;
  if (rows == 0) return R2_OK;
  const TopArgs a = {logits, ld, rows, vocab, k, 1, 0, temperature, values, ids, log_sum, error};
  return dtype == R2_F32 ? launch<float>(a, rows, stream) : launch<bf16>(a, rows, stream);
}
