// Rows of a token table, and the gradient of the table whose rows were looked up:
//
//   out_t = scale * W[i_t]  (zeros where i_t is no token),   dW_v = scale * sum over t with i_t = v of above_t, in one order
//
// The gradient in two launches:
//
//   deal_kernel  sorts the places by token, stable. The table's rows are dealt out to CTAs by the remainder of their number (tokens that stand often lie side
//                by side in a vocabulary). A CTA goes through all tokens, a share a warp, and lists its own with their rank among the share's of their row, beside a
//                count of those of lower deals, so that it knows where in the sorted list its part begins without a word between CTAs. (Places wait until there are 32 of
//                them to look at: the CTA of a token that stands everywhere is the last to be done. 32,768 tokens, one in ten the same: 26.5 to 16.0 us.) Running sums of the shares' and rows'
//                counts then say where each place goes. Meanwhile zeros go to the table's first part in bulk copies from shared memory, without a look at which rows
//                need them: they are most of what a small batch costs, and hide the sorting; the rows that are written twice are fewer than the places.
//   sum_kernel   a CTA takes the sorted places of eight windows, a warp each, and up to 256 columns: a token that stands everywhere and tokens that stand once
//                take the same time. A row whose places lie in several windows is joined in shared memory; one that goes on in other CTAs leaves float sums in
//                memory, and the last of those CTAs adds them, in the order of the places whoever that is. Beside them, the other rows' zeros.
//
// Bound by the bytes of the rows from above and of the table where these are many: 1,024 float32 rows of 768 into 50,257 take 27.2 us (157 MB, 0.87 of a copy's rate). 32,768 bfloat16 rows of
// 1,600 take 66.7 us (266 MB, 0.61): sorting 16 beside two thirds of the zeros, then the sums (45 alone, issue slots half full) beside the rest.
#include "common.cuh"

namespace {

constexpr int THREADS = 256, WARPS = 8;
constexpr int SLICE = 256;             // columns of a warp at most
constexpr int DEAL_WARPS = 31, DEAL_THREADS = DEAL_WARPS * 32;   // of a dealing CTA, beside a warp that writes zeros
constexpr int MOST_ROWS = 1200;        // of a deal
constexpr int DEAL_BYTES = 200 * 1024; // of shared memory: rows' counts, and the rest for what dealing warps list (where one has more places, all go through the tokens again)
constexpr int ZEROS = 16384;           // bytes of a bulk copy

// Zeros that are written beside the sorting, as many as it takes time for (1,024 tokens, 154 MB: with 24, 32 and 44 MB 28.2, 27.2 and 26.7 us, with all 34.2; 32,768 tokens, 161 MB: with 1,024,
// 2,304 and 3,200 bytes a token 71.5, 66.7 and 67.5, with all 69.6). The others go beside the sums, to rows that no token came for, if rows are long enough to be runs of bulk copies.
constexpr long long EARLY_BYTES = 32 << 20, EARLY_BYTES_A_TOKEN = 2304, LONG_ROW = 512;
constexpr int UNIT = 8;   // rows of a warp's step, a CTA an SM: what an SM can write bounds it, so all of them have to have the same

struct Work {
  const int32_t* ids;
  const void* above;
  long long ld;
  void* out;
  long long ld_o;
  int tokens, width, vocab;
  float scale;
  int add;
  int deals;                        // rows v with v mod deals = the CTA's
  int listed;                       // logarithm of the places that a dealing warp lists
  unsigned inverse, shift;          // v / deals = v * inverse >> 32 + shift
  int32_t *row, *place;             // [tokens]: the sorted list: by deal, row and place
  int* held;                        // how many places hold a token
  int zero_ctas;                    // of the sums' launch, its first ones
  int zero_from;                    // rows from this one on get zeros beside the sums, and only where no token came; those before it beside the sorting
  uint32_t* has;                    // [deal][62]: bits of a deal's rows that a token came for, 32 even ones, 32 odd ones in turn
  int slices, slice, window;        // of the columns, columns of one, sorted places of a warp
  int* arrived;                     // [CTA of places][slice]: CTAs that have left their share of the row that goes on from this one
  float* shares;                    // [CTA of places][2][width_up]: sums of a row that an earlier CTA began; of one that the next goes on with
  int width_up, groups;             // (groups: CTAs of places)
  int out_size;                     // bytes of a number of the table
};

// A lane's columns of a slice: pieces of 16 bytes, or every 32nd number.
template <typename T, bool WIDE> struct Lane {
  static constexpr int PIECE = WIDE ? 16 / int(sizeof(T)) : 1, PIECES = SLICE / (32 * PIECE);
  float v[SLICE / 32];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < SLICE / 32; ++i) v[i] = 0.f;
  }
  __device__ __forceinline__ static int column(int piece, int lane) { return (piece * 32 + lane) * PIECE; }
};

template <typename T, bool WIDE> struct Raw {
  using L = Lane<T, WIDE>;
  uint4 wide[WIDE ? L::PIECES : 1];
  T one[WIDE ? 1 : L::PIECES];
  __device__ __forceinline__ void load(const T* row, int width, int lane) {
#pragma unroll
    for (int p = 0; p < L::PIECES; ++p) {
      const int c = L::column(p, lane);
      if constexpr (WIDE) wide[p] = c < width ? __ldg(reinterpret_cast<const uint4*>(row + c)) : make_uint4(0, 0, 0, 0);
      else one[p] = c < width ? row[c] : from_float<T>(0.f);
    }
  }
  __device__ __forceinline__ void add_to(L& sum) const {
#pragma unroll
    for (int p = 0; p < L::PIECES; ++p) {
      if constexpr (WIDE) {
        const uint32_t w[4] = {wide[p].x, wide[p].y, wide[p].z, wide[p].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if constexpr (sizeof(T) == 2) {
            sum.v[p * 8 + 2 * j] += __uint_as_float(w[j] << 16);
            sum.v[p * 8 + 2 * j + 1] += __uint_as_float(w[j] & 0xffff0000u);
          } else {
            sum.v[p * 4 + j] += __uint_as_float(w[j]);
          }
        }
      } else {
        sum.v[p] += to_float(one[p]);
      }
    }
  }
};

template <bool ADD, typename T, typename O, bool WIDE>
__device__ __forceinline__ void put_row(O* row, const Lane<T, WIDE>& sum, int width, float scale, int lane) {
  using L = Lane<T, WIDE>;
#pragma unroll
  for (int p = 0; p < L::PIECES; ++p) {
    const int c = L::column(p, lane);
    if (c >= width) continue;
    float old[L::PIECE];
#pragma unroll
    for (int j = 0; j < L::PIECE; ++j) old[j] = 0.f;
    if (ADD) {
#pragma unroll
      for (int j = 0; j < L::PIECE; ++j) old[j] = to_float(row[c + j]);
    }
    alignas(16) O out[L::PIECE];
#pragma unroll
    for (int j = 0; j < L::PIECE; ++j) out[j] = from_float<O>(fmaf(sum.v[p * L::PIECE + j], scale, old[j]));
    if constexpr (WIDE) {
      if constexpr (sizeof(out) == 32) {
        reinterpret_cast<uint4*>(row + c)[0] = reinterpret_cast<const uint4*>(out)[0];
        reinterpret_cast<uint4*>(row + c)[1] = reinterpret_cast<const uint4*>(out)[1];
      } else if constexpr (sizeof(out) == 16) {
        *reinterpret_cast<uint4*>(row + c) = *reinterpret_cast<const uint4*>(out);
      } else {
        *reinterpret_cast<uint2*>(row + c) = *reinterpret_cast<const uint2*>(out);
      }
    } else {
      row[c] = out[0];
    }
  }
}

__device__ __forceinline__ unsigned quotient_of(unsigned v, const Work& w) { return __umulhi(v, w.inverse) >> w.shift; }

__device__ __forceinline__ long long row_bytes(const Work& w) { return static_cast<long long>(w.width) * w.out_size; }

// Zeros for the rows from zero_from on that no token came for: runs of empty ones at once, in bulk copies between what is left of 16 bytes at a run's ends.
__device__ __forceinline__ void write_zeros(const Work& w, uint4* zeros, int block, int blocks) {
  const int lane = threadIdx.x & 31;
  for (int j = threadIdx.x; j < ZEROS / 16; j += THREADS) zeros[j] = make_uint4(0, 0, 0, 0);
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncthreads();
  const long long size = row_bytes(w);
  for (long long first = w.zero_from + (block + (threadIdx.x >> 5) * blocks) * static_cast<long long>(UNIT); first < w.vocab; first += blocks * WARPS * static_cast<long long>(UNIT)) {
    const bool there = lane < UNIT && first + lane < w.vocab;
    const unsigned v = unsigned(there ? first + lane : first), row = quotient_of(v, w), deal = v - row * w.deals;
    unsigned empty = __ballot_sync(0xffffffffu, there && (w.has[(deal * DEAL_WARPS + row / 64) * 2 + row % 2] >> (row / 2 % 32) & 1u) == 0);
    while (empty != 0) {
      const int begin = __ffs(int(empty)) - 1, rows = __ffs(int(~(empty >> begin) | (begin > 0 ? 1u << (32 - begin) : 0u))) - 1, n = rows < 0 ? 32 : rows;
      empty &= n == 32 ? 0u : ~(((1u << n) - 1u) << begin);
      char* at = static_cast<char*>(w.out) + (first + begin) * size;
      const long long bytes = n * size, short_of_16 = -reinterpret_cast<intptr_t>(at) & 15, head = short_of_16 < bytes ? short_of_16 : bytes, whole = (bytes - head) / 16 * 16;
      if (lane < head) at[lane] = 0;
      for (long long o = lane * ZEROS; o < whole; o += 32 * ZEROS) {
        const unsigned piece = unsigned(whole - o < ZEROS ? whole - o : ZEROS);
        asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(at + head + o), "r"(uint32_t(__cvta_generic_to_shared(zeros))), "r"(piece) : "memory");
      }
      if (head + whole + lane < bytes) at[head + whole + lane] = 0;
    }
  }
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
  asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
}

__global__ void __launch_bounds__(DEAL_THREADS + 32, 1) deal_kernel(const Work w) {
  extern __shared__ int32_t shared[];
  __shared__ int mine[DEAL_WARPS], lower[DEAL_WARPS], running[DEAL_WARPS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, deal = blockIdx.x;
  const int rows = int((static_cast<long long>(w.vocab) - deal + w.deals - 1) / w.deals);
  int32_t* counts = shared;                          // [warp][rows]: a row's places in the warp's share, then where the first of them goes
  int32_t* list_place = counts + DEAL_WARPS * rows;  // [warp][listed]
  uint32_t* list_row = reinterpret_cast<uint32_t*>(list_place + (DEAL_WARPS << w.listed));   // row << listed, rank
  __shared__ alignas(16) uint4 zeros[ZEROS / 16];
  auto sync = [] { asm volatile("bar.sync 1, %0;" ::"n"(DEAL_THREADS) : "memory"); };
  if (w.zero_ctas == 0) pdl_launch_dependents();   // (CTAs that write zeros have to lie evenly on the SMs: started in what shared memory the sorting leaves, they took twice the time)
  if (warp == DEAL_WARPS) {
    // ---- zeros: the CTAs' pieces side by side, so that all of them write in one part of the table; a lane a piece
    if (w.add) return;
    for (int j = lane; j < ZEROS / 16; j += 32) zeros[j] = make_uint4(0, 0, 0, 0);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    pdl_wait();
    char* out = static_cast<char*>(w.out);
    const long long bytes = w.zero_from * row_bytes(w), whole = bytes / 16 * 16;
    for (long long at = (deal + static_cast<long long>(lane) * w.deals) * ZEROS; at < whole; at += 32ll * w.deals * ZEROS) {
      const unsigned n = unsigned(whole - at < ZEROS ? whole - at : ZEROS);
      asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(out + at), "r"(uint32_t(__cvta_generic_to_shared(zeros))), "r"(n) : "memory");
    }
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    if (deal == 0 && whole + lane < bytes) out[whole + lane] = 0;
    asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    return;
  }
  for (int j = threadIdx.x; j < DEAL_WARPS * rows; j += DEAL_THREADS) counts[j] = 0;
  sync();
  pdl_wait();
  for (long long i = deal * DEAL_THREADS + threadIdx.x; i < static_cast<long long>(w.groups) * w.slices; i += w.deals * DEAL_THREADS) w.arrived[i] = 0;

  // ---- a warp's share of the places, in order: each(row, place, rank behind what counts says at the start, how many of the share came before)
  constexpr int LOADS = 16;
  const int share = ((w.tokens + DEAL_WARPS - 1) / DEAL_WARPS + 31) / 32 * 32;
  const int first = int(min(static_cast<long long>(warp) * share, static_cast<long long>(w.tokens))), last = int(min(static_cast<long long>(first) + share, static_cast<long long>(w.tokens)));
  int32_t* own_counts = counts + warp * rows;
  int n_mine = 0, n_lower = 0;
  __shared__ int waiting[DEAL_WARPS][64];   // places that a warp has come across, a ring: they are looked at 32 at a time
  const unsigned before = (1u << lane) - 1u;
  auto walk = [&](auto&& each) {
    n_mine = n_lower = 0;
    int pending = 0;
    auto look = [&](int n) {
      if (lane < n) {
        const unsigned all = n == 32 ? 0xffffffffu : (1u << n) - 1u;
        const int place = waiting[warp][(n_mine + lane) & 63], row = int(quotient_of(unsigned(w.ids[place]), w));
        const unsigned peers = __match_any_sync(all, row);
        const int count = own_counts[row];
        __syncwarp(all);
        if ((peers >> lane) == 1u) own_counts[row] = count + __popc(peers);   // (the last of them)
        each(row, place, count + __popc(peers & before), n_mine + lane);
      }
      __syncwarp();
      n_mine += n;
      pending -= n;
    };
    for (int t0 = first; t0 < last; t0 += 32 * LOADS) {
      unsigned id[LOADS];
#pragma unroll
      for (int j = 0; j < LOADS; ++j) id[j] = t0 + 32 * j + lane < last ? unsigned(w.ids[t0 + 32 * j + lane]) : 0xffffffffu;
      // few of 32 tokens are the CTA's: which of the pieces hold one, first
      unsigned pieces = 0;
#pragma unroll
      for (int j = 0; j < LOADS; ++j) {
        const unsigned at = id[j] < unsigned(w.vocab) ? id[j] - quotient_of(id[j], w) * unsigned(w.deals) : 0xffffffffu;
        n_lower += at < unsigned(deal) ? 1 : 0;
        pieces |= at == unsigned(deal) ? 1u << j : 0u;
      }
      const unsigned own_pieces = pieces;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) pieces |= __shfl_xor_sync(0xffffffffu, pieces, o);
#pragma unroll 1
      for (; pieces != 0; pieces &= pieces - 1u) {
        const int j = __ffs(int(pieces)) - 1;
        const bool own = own_pieces >> j & 1u;
        const unsigned owners = __ballot_sync(0xffffffffu, own);
        if (own) waiting[warp][(n_mine + pending + __popc(owners & before)) & 63] = t0 + 32 * j + lane;
        __syncwarp();
        pending += __popc(owners);
        if (pending >= 32) look(32);
      }
    }
    if (pending > 0) look(pending);
  };
  walk([&](int row, int place, int rank, int at) {
    if (at < 1 << w.listed) {
      list_row[(warp << w.listed) + at] = (unsigned(row) << w.listed) + unsigned(rank);
      list_place[(warp << w.listed) + at] = place;
    }
  });
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) n_lower += __shfl_xor_sync(0xffffffffu, n_lower, o);
  if (lane == 0) {
    mine[warp] = n_mine;
    lower[warp] = n_lower;
  }
  sync();
  int total = lane < DEAL_WARPS ? mine[lane] : 0, offset = lane < DEAL_WARPS ? lower[lane] : 0, most = total;   // (a lane a warp)
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    total += __shfl_xor_sync(0xffffffffu, total, o);
    offset += __shfl_xor_sync(0xffffffffu, offset, o);
    most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
  }
  if (deal == w.deals - 1 && threadIdx.x == 0) *w.held = offset + total;

  // ---- running sums: of a row over the shares, of the rows (up to two a thread, side by side) over the threads
  constexpr int PER = (MOST_ROWS + DEAL_THREADS - 1) / DEAL_THREADS;
  int of_row[PER], own = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int j = int(threadIdx.x) * PER + i;
    of_row[i] = 0;
    if (j < rows) {
      for (int part = 0; part < DEAL_WARPS; ++part) of_row[i] += counts[part * rows + j];
    }
    static_assert(PER == 2);
    const unsigned bits = __ballot_sync(0xffffffffu, of_row[i] > 0);
    if (lane == 0 && warp * 64 < rows && w.zero_from < w.vocab) w.has[(deal * DEAL_WARPS + warp) * 2 + i] = bits;
    own += of_row[i];
  }
  int up = own;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, up, o);
    up += lane >= o ? x : 0;
  }
  if (lane == 31) running[warp] = up;
  sync();
  int begin = lane < warp ? running[lane] : 0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) begin += __shfl_xor_sync(0xffffffffu, begin, o);
  begin += offset + up - own;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int j = int(threadIdx.x) * PER + i;
    if (j >= rows) continue;
    for (int part = 0; part < DEAL_WARPS; ++part) {
      const int n = counts[part * rows + j];
      counts[part * rows + j] = begin;
      begin += n;
    }
  }
  sync();

  // ---- where each place goes
  if (most <= 1 << w.listed) {
    for (int i = lane; i < n_mine; i += 32) {
      const unsigned entry = list_row[(warp << w.listed) + i];
      const int row = int(entry >> w.listed), at = own_counts[row] + int(entry & ((1u << w.listed) - 1u));
      w.row[at] = row * w.deals + deal;
      w.place[at] = list_place[(warp << w.listed) + i];
    }
  } else {
    walk([&](int row, int place, int at, int) {
      w.row[at] = row * w.deals + deal;
      w.place[at] = place;
    });
  }
}

template <typename T, typename O, bool WIDE, bool ADD>
__global__ void __launch_bounds__(THREADS, 3) sum_kernel(const Work w) {
  __shared__ alignas(16) float ends[2][WARPS][SLICE];
  auto &heads = ends[0], &tails = ends[1];                     // of a window: the sum of the row that an earlier one began; of the row that the next goes on with
  __shared__ int head_row[WARPS], tail_row[WARPS];             // -1: none
  __shared__ int last_of_chain;
  pdl_launch_dependents();
  pdl_wait();
  if constexpr (!ADD) {
    if (int(blockIdx.x) < w.zero_ctas) {
      static_assert(sizeof(ends) == ZEROS);
      write_zeros(w, reinterpret_cast<uint4*>(ends), int(blockIdx.x), w.zero_ctas);
      return;
    }
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int held = *w.held;
  const int block = int(blockIdx.x) - w.zero_ctas, group = block / w.slices, slice = block % w.slices, span = WARPS * w.window;
  const int col = slice * w.slice, width = min(w.slice, w.width - col);
  const int group_from = group * span;
  if (group_from >= held) return;
  const T* above = static_cast<const T*>(w.above) + col;
  O* out = static_cast<O*>(w.out) + col;

  // ---- a warp's window
  const int from = group_from + warp * w.window, n = min(w.window, held - from);
  int head = -1, tail = -1;
  if (n > 0) {
    const int place = lane < n ? w.place[from + lane] : 0, number = lane < n ? w.row[from + lane] : -1;
    const int before = from > 0 ? w.row[from - 1] : -1, after = from + n < held ? w.row[from + n] : -1;
    const long long from_place = place * w.ld, to_number = number * w.ld_o;   // (a lane's, once; the warp asks the lane)
    constexpr int BATCH = WIDE && sizeof(T) == 2 ? 4 : 2;   // rows asked for together; two batches are on their way (what the registers of three CTAs an SM hold)
    Raw<T, WIDE> raw[2][BATCH];
    auto load = [&](Raw<T, WIDE> (&r)[BATCH], int i0) {
#pragma unroll
      for (int j = 0; j < BATCH; ++j) {
        const long long t = __shfl_sync(0xffffffffu, from_place, (i0 + j) & 31);
        if (i0 + j < n) r[j].load(above + t, width, lane);
      }
    };
    Lane<T, WIDE> sum;
    sum.clear();
    int row = __shfl_sync(0xffffffffu, number, 0);
    bool began_here = before != row;
    auto keep = [&](float* to) {
#pragma unroll
      for (int k = 0; k < SLICE / 32; ++k) to[Lane<T, WIDE>::column(k / Lane<T, WIDE>::PIECE, lane) + k % Lane<T, WIDE>::PIECE] = sum.v[k];
    };
    auto take = [&](const Raw<T, WIDE> (&r)[BATCH], int i0) {
#pragma unroll
      for (int j = 0; j < BATCH; ++j) {
        const int i = i0 + j;
        if (i < n) {
          r[j].add_to(sum);
          const int other = __shfl_sync(0xffffffffu, number, (i + 1) & 31), next = i + 1 < n ? other : after;
          if (next != row) {
            const long long to_row = __shfl_sync(0xffffffffu, to_number, i);
            if (began_here) {
              put_row<ADD>(out + to_row, sum, width, w.scale, lane);
            } else {
              head = row;
              keep(heads[warp]);
            }
            began_here = true;
            sum.clear();
            row = next;
          } else if (i + 1 == n) {   // the next window goes on with it (it may have gone through this one whole)
            tail = row;
            keep(tails[warp]);
          }
        }
      }
    };
    load(raw[0], 0);
#pragma unroll 1
    for (int i = 0; i < n; i += 2 * BATCH) {
      load(raw[1], i + BATCH);
      take(raw[0], i);
      load(raw[0], i + 2 * BATCH);
      take(raw[1], i + BATCH);
    }
  }
  if (lane == 0) {
    head_row[warp] = head;
    tail_row[warp] = tail;
  }
  __syncthreads();

  // ---- rows of several windows, a thread a column
  const int c = threadIdx.x;
  bool began_before = group_from > 0 && w.row[group_from - 1] == w.row[group_from];   // (the first row; it ends in a head, or goes on as a tail)
  float* shares = w.shares + static_cast<long long>(group) * 2 * w.width_up + col;
  auto put = [&](int row, float sum) {
    O* to = out + row * w.ld_o + c;
    *to = from_float<O>(fmaf(sum, w.scale, ADD ? to_float(*to) : 0.f));
  };
  int ended = -1, open = -1;   // rows of other CTAs, too: the one that ends here, the one that goes on
  float sum = 0.f;
  for (int i = 0; i < WARPS; ++i) {
    if (head_row[i] >= 0) {
      if (c < width) {
        sum += heads[i][c];
        if (began_before) shares[c] = sum;
        else put(head_row[i], sum);
      }
      if (began_before) ended = head_row[i];
      began_before = false;
      sum = 0.f;
    }
    open = tail_row[i];
    if (open >= 0 && c < width) sum += tails[i][c];
  }
  if (open >= 0 && c < width) shares[w.width_up + c] = sum;

  // ---- rows of several CTAs: whoever comes last adds their shares
  auto chain = [&](int row, int first, int last) {   // CTAs first .. last of places hold it
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) {
      last_of_chain = atomicAdd(w.arrived + static_cast<long long>(first) * w.slices + slice, 1) == last - first;
      __threadfence();
    }
    __syncthreads();
    if (last_of_chain && c < width) {
      const float* from_here = w.shares + static_cast<long long>(first) * 2 * w.width_up + col + c;
      float all = 0.f;
#pragma unroll 8
      for (int i = 0; i < last - first; ++i) all += __ldcg(from_here + (2ll * i + 1) * w.width_up);
      all += __ldcg(from_here + 2ll * (last - first) * w.width_up);
      put(row, all);
    }
    __syncthreads();
  };
  auto first_of = [&](int row) {   // of the CTAs of a row that began before this one, 32 at a look
    int g = group - 1;
    while (true) {
      const int at = g - lane;
      const bool through = at > 0 && w.row[at > 0 ? at * span : 0] == row && w.row[at > 0 ? at * span - 1 : 0] == row;
      const unsigned stops = ~__ballot_sync(0xffffffffu, through);
      if (stops != 0) return g - (__ffs(int(stops)) - 1);
      g -= 32;
    }
  };
  const bool open_before = began_before;   // (nothing has ended since the CTA's first place)
  if (ended >= 0) chain(ended, first_of(ended), group);
  if (open >= 0) {
    const int first = open_before ? first_of(open) : group;
    int g = group + 1;
    while (true) {
      const long long next = (g + 1ll + lane) * span;
      const unsigned stops = ~__ballot_sync(0xffffffffu, next < held && w.row[next < held ? next : 0] == open);
      if (stops != 0) {
        g += __ffs(int(stops)) - 1;
        break;
      }
      g += 32;
    }
    chain(open, first, g);
  }
}

// A warp a row.
template <typename T, typename O, bool WIDE>
__global__ void __launch_bounds__(THREADS) token_rows_kernel(const int32_t* ids, const T* table, long long ld, O* out, long long ld_o, int tokens, int width, int vocab,
                                                             float scale) {
  using L = Lane<T, WIDE>;
  const int lane = threadIdx.x & 31;
  for (long long t = blockIdx.x * static_cast<long long>(WARPS) + (threadIdx.x >> 5); t < tokens; t += gridDim.x * static_cast<long long>(WARPS)) {
    const int id = ids[t];
    const bool held = id >= 0 && id < vocab;
    for (int c = 0; c < width; c += SLICE) {
      Lane<T, WIDE> row;
      row.clear();
      if (held) {
        Raw<T, WIDE> raw;
        raw.load(table + id * ld + c, width - c, lane);
        raw.add_to(row);
      }
      put_row<false>(out + t * ld_o + c, row, width - c, held ? scale : 0.f, lane);
    }
  }
}

int n_sms() {
  static std::atomic<int> cached[64];
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 148;
  if (dev < 64 && (n = cached[dev].load()) > 0) return n;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n < 1) {
    cudaGetLastError();
    n = 148;
  }
  if (dev < 64) cached[dev].store(n);
  return n;
}

// As many deals as SMs, of no more rows than a CTA counts.
int deals_of(int vocab) {
  int deals = n_sms();
  if (deals > vocab) deals = vocab;
  if (deals < (vocab - 1) / MOST_ROWS + 1) deals = (vocab - 1) / MOST_ROWS + 1;
  return deals < 2 ? 2 : deals;
}

int launch_deal(const Work& w, cudaStream_t stream) {
  static std::atomic<bool> done[64];
  const int status = allow_smem(deal_kernel, DEAL_BYTES, done);
  if (status != R2_OK) return status;
  r2_launch(deal_kernel, dim3(w.deals), dim3(DEAL_THREADS + 32), size_t(DEAL_WARPS) * (((w.vocab - 1) / w.deals + 1) * 4 + (8 << w.listed)), stream, w);
  return launch_status();
}

template <typename T, typename O, bool WIDE>
int launch_sums(const Work& w, cudaStream_t stream) {
  r2_launch(w.add ? sum_kernel<T, O, WIDE, true> : sum_kernel<T, O, WIDE, false>, dim3(unsigned(w.groups) * unsigned(w.slices) + unsigned(w.zero_ctas)), dim3(THREADS), size_t(0), stream, w);
  return launch_status();
}

// Slices of the columns; windows of 32 places, or of fewer where that would leave SMs without a CTA.
void share_out(Work& w) {
  w.slices = (w.width + SLICE - 1) / SLICE;
  w.slice = ((w.width + w.slices - 1) / w.slices + 63) / 64 * 64;   // (whole lines of 128 bytes)
  w.slices = (w.width + w.slice - 1) / w.slice;
  w.window = 32;
  while (w.window > 4 && static_cast<long long>(w.tokens) * w.slices < 2ll * n_sms() * WARPS * w.window) w.window /= 2;
  w.groups = (w.tokens + WARPS * w.window - 1) / (WARPS * w.window);
  w.width_up = (w.width + 7) / 8 * 8;
  w.deals = deals_of(w.vocab);
  // v / deals for v < 2^30: with 2^(s - 1) < deals <= 2^s the inverse of 2^(31 + s), rounded up, is below 2^32, and v times its excess below 2^30 deals < 2^(31 + s)
  int s = 1;
  while (1ll << s < w.deals) ++s;
  w.inverse = unsigned(((1ull << (31 + s)) + unsigned(w.deals) - 1) / unsigned(w.deals));
  w.shift = unsigned(s - 1);
  const int rows = (w.vocab - 1) / w.deals + 1;
  w.listed = 7;   // (MOST_ROWS leave room for 128)
  while (w.listed < 10 && DEAL_WARPS * (rows * 4 + (16 << w.listed)) <= DEAL_BYTES) ++w.listed;
}

bool at_16(const void* p, long long ld, int size) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * size % 16 == 0; }

constexpr int MOST = 1 << 30;

}  // namespace

extern "C" int r2_token_rows(int dtype, int out_dtype, const int32_t* ids, const void* table, long long ld, void* out, long long ld_o, int tokens, int width, int vocab,
                             float scale, cudaStream_t stream) {
  if (tokens < 1 || width < 1) return R2_BAD_SHAPE;
  const int size = dtype == R2_F32 ? 4 : 2, out_size = out_dtype == R2_F32 ? 4 : 2;
  const bool wide = at_16(table, ld, size) && at_16(out, ld_o, out_size) && width * size % 16 == 0;
  const int grid = tokens < 8 * WARPS * n_sms() ? (tokens + WARPS - 1) / WARPS : 8 * n_sms();
#define R2_CASE(T, O)                                                                                                                                        \
  (wide ? token_rows_kernel<T, O, true><<<grid, THREADS, 0, stream>>>(ids, (const T*)table, ld, (O*)out, ld_o, tokens, width, vocab, scale)                 \
        : token_rows_kernel<T, O, false><<<grid, THREADS, 0, stream>>>(ids, (const T*)table, ld, (O*)out, ld_o, tokens, width, vocab, scale))
  if (dtype == R2_F32 && out_dtype == R2_F32) R2_CASE(float, float);
  else if (dtype == R2_F32 && out_dtype == R2_BF16) R2_CASE(float, bf16);
  else if (dtype == R2_BF16 && out_dtype == R2_F32) R2_CASE(bf16, float);
  else if (dtype == R2_BF16 && out_dtype == R2_BF16) R2_CASE(bf16, bf16);
  else return R2_BAD_DTYPE;
#undef R2_CASE
  return launch_status();
}

// Bytes of scratch for a gradient: two lists of the places, their number, what CTAs of places leave of rows that lie in several.
extern "C" long long r2_token_rows_space(int tokens, int width, int vocab) {
  Work w = {};
  w.tokens = tokens;
  w.width = width;
  w.vocab = vocab;
  share_out(w);
  return 8ll * tokens + 16 + static_cast<long long>(w.groups) * (2ll * w.width_up + w.slices) * 4 + w.deals * (DEAL_WARPS * 8ll);
}

extern "C" int r2_token_rows_gradient(int dtype, int out_dtype, const int32_t* ids, const void* above, long long ld, void* out, long long ld_o, int tokens, int width,
                                      int vocab, float scale, int add, void* space, cudaStream_t stream) {
  if (tokens < 1 || width < 1 || vocab < 1) return R2_BAD_SHAPE;
  if (tokens > MOST || width > MOST || vocab > MOST) return R2_UNSUPPORTED;
  if (!add && (ld_o != width || reinterpret_cast<uintptr_t>(out) % 16 != 0)) return R2_BAD_ALIGN;   // (a new table is one piece)
  const int size = dtype == R2_F32 ? 4 : 2, out_size = out_dtype == R2_F32 ? 4 : 2;
  const bool wide = at_16(above, ld, size) && at_16(out, ld_o, out_size) && width * size % 16 == 0 && width * out_size % 16 == 0;
  Work w = {ids, above, ld, out, ld_o, tokens, width, vocab, scale, add};
  share_out(w);
  if (static_cast<long long>(w.groups) * w.slices >= 1ll << 31) return R2_UNSUPPORTED;
  w.row = static_cast<int32_t*>(space);
  w.place = w.row + tokens;
  w.held = w.place + tokens;
  w.shares = reinterpret_cast<float*>(w.held + 4);
  w.arrived = reinterpret_cast<int*>(w.shares + static_cast<long long>(w.groups) * 2 * w.width_up);
  w.has = reinterpret_cast<uint32_t*>(w.arrived + static_cast<long long>(w.groups) * w.slices);
  w.out_size = out_size;
  const long long row = static_cast<long long>(width) * out_size, early = (EARLY_BYTES + EARLY_BYTES_A_TOKEN * tokens) / row;
  w.zero_from = add || row < LONG_ROW || early > vocab ? vocab : int(early);
  const int rest = (vocab - w.zero_from + UNIT - 1) / UNIT;
  w.zero_ctas = rest < n_sms() ? rest : n_sms();
  if (dtype < R2_F32 || dtype > R2_BF16 || out_dtype < R2_F32 || out_dtype > R2_BF16) return R2_BAD_DTYPE;
  const int status = launch_deal(w, stream);
  if (status != R2_OK) return status;
#define R2_CASE(T, O) (wide ? launch_sums<T, O, true>(w, stream) : launch_sums<T, O, false>(w, stream))
  if (dtype == R2_F32 && out_dtype == R2_F32) return R2_CASE(float, float);
  if (dtype == R2_F32) return R2_CASE(float, bf16);
  if (dtype == R2_BF16 && out_dtype == R2_F32) return R2_CASE(bf16, float);
  return R2_CASE(bf16, bf16);
#undef R2_CASE
}
