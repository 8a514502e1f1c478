// Rows of a token table, and the gradient of the table whose rows were looked up:
//
//   out_t = scale * W[i_t]  (zeros where i_t is no token),   dW_v = scale * sum over t with i_t = v of above_t, in one order
//
// The gradient is one launch and needs nothing between CTAs. The table's rows are dealt out by the remainder of their number (tokens that stand often
// lie side by side in a vocabulary), its columns in slices, and a CTA owns a deal and a slice: it goes through all tokens, lists the places of its own in
// their order, sorts the list by token (a count, a running sum, a stable placing), writes zeros to the rows without one and adds up the others. Its eight warps
// share the sorted places evenly, eight rows from above on their way to each at any time, so that a token that stands everywhere and tokens that stand once take the
// same time; a token whose places lie in several warps' shares is joined behind them, in their order. Going through the tokens costs each CTA 4 bytes
// a token twice, read from L2; the rows from above, which are hundreds of times as much, are read once.
//
// Bound by the bytes of the rows from above and of the table.
#include "common.cuh"

namespace {

constexpr int THREADS = 256, WARPS = 8;
constexpr int SLICE = 256;          // columns of a CTA at most
constexpr int LISTED = 6144;        // places that shared memory holds (beyond them: the scratch)
constexpr int LISTED_BYTES = LISTED * 12;
constexpr int MOST_ROWS = 8192;     // of a CTA (16 bits hold one)

struct Work {
  const int32_t* ids;
  const void* above;
  long long ld;
  void* out;
  long long ld_o;
  int tokens, width, vocab;
  float scale;
  int add;
  int deals, slice;                 // rows v with v mod deals = the CTA's; columns of a slice
  unsigned long long inverse;       // v / deals = v * inverse >> 64
  int32_t* spill;                   // [slice]: places [2][tokens], rows as 16 bits [2][tokens]
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

template <typename T, typename O, bool WIDE>
__device__ __forceinline__ void put_row(O* row, const Lane<T, WIDE>& sum, int width, float scale, bool add, int lane) {
  using L = Lane<T, WIDE>;
#pragma unroll
  for (int p = 0; p < L::PIECES; ++p) {
    const int c = L::column(p, lane);
    if (c >= width) continue;
    alignas(16) O out[L::PIECE];
#pragma unroll
    for (int j = 0; j < L::PIECE; ++j) out[j] = from_float<O>(sum.v[p * L::PIECE + j] * scale + (add ? to_float(row[c + j]) : 0.f));
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

template <typename T, typename O, bool WIDE>
__global__ void __launch_bounds__(THREADS, 2) gradient_kernel(const Work w) {
  extern __shared__ int32_t shared[];
  __shared__ int mine[WARPS], lower[WARPS], running[WARPS];
  __shared__ int head_row[WARPS], tail_row[WARPS];   // whose sums are in `heads` and `tails`, -1: none
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int deal = blockIdx.x % w.deals, slice = blockIdx.x / w.deals;
  const int rows = int((static_cast<long long>(w.vocab) - deal + w.deals - 1) / w.deals);   // that this CTA owns
  int32_t* ends = shared;   // [rows]: counts, then where a row's places begin, then where they end
  const unsigned inverse_high = unsigned(w.inverse >> 32), inverse_low = unsigned(w.inverse);
  auto quotient = [&](int id) {
    const unsigned long long v = unsigned(id);
    return int((v * inverse_high + (v * inverse_low >> 32)) >> 32);
  };

  for (int j = threadIdx.x; j < rows; j += THREADS) ends[j] = 0;
  __syncthreads();

  // ---- a warp's share of the places: how many are this CTA's, how many of a lower deal
  const int share = ((w.tokens + WARPS - 1) / WARPS + 255) / 256 * 256;
  const int first = int(min(static_cast<long long>(warp) * share, static_cast<long long>(w.tokens))), last = int(min(static_cast<long long>(first) + share, static_cast<long long>(w.tokens)));
  int n_mine = 0, n_lower = 0;
  for (int t0 = first; t0 < last; t0 += 256) {
    int id[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) id[j] = t0 + 32 * j + lane < last ? __ldg(w.ids + t0 + 32 * j + lane) : -1;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (id[j] < 0 || id[j] >= w.vocab) continue;
      const int row = quotient(id[j]), at = id[j] - row * w.deals;
      if (at == deal) {
        atomicAdd(&ends[row], 1);
        ++n_mine;
      }
      n_lower += at < deal ? 1 : 0;
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    n_mine += __shfl_xor_sync(0xffffffffu, n_mine, o);
    n_lower += __shfl_xor_sync(0xffffffffu, n_lower, o);
  }
  if (lane == 0) {
    mine[warp] = n_mine;
    lower[warp] = n_lower;
  }
  __syncthreads();
  int total = 0, before = 0, offset = 0;
#pragma unroll
  for (int i = 0; i < WARPS; ++i) {
    before += i < warp ? mine[i] : 0;
    total += mine[i];
    offset += lower[i];
  }

  // ---- rows without a place
  const int col = slice * w.slice, width = min(w.slice, w.width - col);
  const T* above = static_cast<const T*>(w.above) + col;
  O* out = static_cast<O*>(w.out) + col;
  Lane<T, WIDE> sum;
  sum.clear();
  if (!w.add) {
    for (int j = warp; j < rows; j += WARPS)
      if (ends[j] == 0) put_row<T, O, WIDE>(out + (static_cast<long long>(j) * w.deals + deal) * w.ld_o, sum, width, 1.f, false, lane);
  }
  if (total == 0) return;
  __syncthreads();   // (the counts become places)

  // ---- the list (token and place) and the sorted one: in shared memory, or in this deal's part of the slice's scratch
  int32_t* places = shared + rows;
  long long apart = LISTED;
  uint16_t* numbers = reinterpret_cast<uint16_t*>(places + 2 * LISTED);
  if (total > LISTED) {
    places = w.spill + static_cast<long long>(slice) * 3 * w.tokens + offset;
    numbers = reinterpret_cast<uint16_t*>(w.spill + static_cast<long long>(slice) * 3 * w.tokens + 2 * static_cast<long long>(w.tokens)) + offset;
    apart = w.tokens;
  }
  int32_t *list_place = places, *sorted_place = places + apart;
  uint16_t *list_row = numbers, *sorted_row = numbers + apart;
  if (n_mine > 0) {
    for (int t0 = first; t0 < last; t0 += 256) {
      int id[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) id[j] = t0 + 32 * j + lane < last ? __ldg(w.ids + t0 + 32 * j + lane) : -1;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int row = quotient(id[j] < 0 ? 0 : id[j]);
        const bool own = id[j] >= 0 && id[j] < w.vocab && id[j] - row * w.deals == deal;
        const unsigned mask = __ballot_sync(0xffffffffu, own);
        if (own) {
          const int at = before + __popc(mask & ((1u << lane) - 1u));
          list_row[at] = uint16_t(row);
          list_place[at] = t0 + 32 * j + lane;
        }
        before += __popc(mask);
      }
    }
  }
  // where each row's places begin: a thread's share of the rows, then the threads'
  {
    const int per = (rows + THREADS - 1) / THREADS, from = min(rows, int(threadIdx.x) * per), to = min(rows, from + per);
    int own = 0;
    for (int j = from; j < to; ++j) own += ends[j];
    int up = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, up, o);
      up += lane >= o ? x : 0;
    }
    if (lane == 31) running[warp] = up;
    __syncthreads();
    int begin = up - own;
#pragma unroll
    for (int i = 0; i < WARPS; ++i) begin += i < warp ? running[i] : 0;
    for (int j = from; j < to; ++j) {
      const int n = ends[j];
      ends[j] = begin;
      begin += n;
    }
    __syncthreads();
  }
  // a stable placing: a warp takes the rows of its number mod 8 from the list, in the list's order
  int next_row = lane < total ? list_row[lane] : -1, next_place = lane < total ? list_place[lane] : 0;
  for (int i0 = 0; i0 < total; i0 += 32) {
    const int row = next_row, place = next_place;
    if (i0 + 32 < total) {   // (asked for ahead: the list may lie in memory)
      next_row = i0 + 32 + lane < total ? list_row[i0 + 32 + lane] : -1;
      next_place = i0 + 32 + lane < total ? list_place[i0 + 32 + lane] : 0;
    }
    const bool own = row >= 0 && (row & (WARPS - 1)) == warp;
    const unsigned owners = __ballot_sync(0xffffffffu, own);
    if (owners == 0) continue;
    int at = 0;
    unsigned peers = 0;
    if (own) {
      peers = __match_any_sync(owners, row);
      at = ends[row] + __popc(peers & ((1u << lane) - 1u));
      sorted_row[at] = uint16_t(row);
      sorted_place[at] = place;
    }
    __syncwarp();
    if (own && (peers >> lane) == 1u) ends[row] = at + 1;   // (the last of them)
    __syncwarp();
  }
  __syncthreads();

  // ---- sums: an even share of the sorted places a warp, in order. A lane holds one of 32 places and rows, of this window and of the next.
  constexpr int AHEAD = WIDE && sizeof(T) == 2 ? 16 : 8;   // rows from above on their way to a warp (what registers hold)
  float (*heads)[SLICE] = reinterpret_cast<float (*)[SLICE]>(shared);   // (the counts and the list, which are done with)
  float (*tails)[SLICE] = heads + WARPS;
  const int part = max(((total + WARPS - 1) / WARPS + 7) / 8 * 8, 8);
  const int from = min(total, warp * part), to = min(total, from + part);
  const int before_row = from > 0 && from < to ? sorted_row[from - 1] : -1, after_row = to < total && from < to ? sorted_row[to] : -1;
  int head = -1, tail = -1;
  auto at_place = [&](int i) { return i < to ? sorted_place[i] : -1; };
  auto at_row = [&](int i) { return i < to ? int(sorted_row[i]) : after_row; };
  int place[2] = {at_place(from + lane), at_place(from + 32 + lane)}, number[2] = {at_row(from + lane), at_row(from + 32 + lane)};
  __syncthreads();   // (behind it the sums of warps take the place of the counts and of the list; the sorted places stay)
  if (from < to) {
    Raw<T, WIDE> raw[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const int t = __shfl_sync(0xffffffffu, place[0], j);
      if (t >= 0) raw[j].load(above + t * w.ld, width, lane);
    }
    int row = __shfl_sync(0xffffffffu, number[0], 0);
    bool began_here = before_row != row;
    for (int i0 = from; i0 < to; i0 += 32) {
      const int place2 = at_place(i0 + 64 + lane), number2 = at_row(i0 + 64 + lane);
#pragma unroll 1
      for (int g = 0; g < 32; g += AHEAD) {
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
          const int i = g + j;   // of the window
          if (i0 + i >= to) break;
          raw[j].add_to(sum);
          const int t = __shfl_sync(0xffffffffu, i + AHEAD < 32 ? place[0] : place[1], (i + AHEAD) & 31);
          if (t >= 0) raw[j].load(above + t * w.ld, width, lane);
          const int next = __shfl_sync(0xffffffffu, i + 1 < 32 ? number[0] : number[1], (i + 1) & 31);
          if (next != row) {
            if (began_here) {
              put_row<T, O, WIDE>(out + (static_cast<long long>(row) * w.deals + deal) * w.ld_o, sum, width, w.scale, w.add != 0, lane);
            } else {
              head = row;
#pragma unroll
              for (int k = 0; k < SLICE / 32; ++k) heads[warp][k * 32 + lane] = sum.v[k];
            }
            began_here = true;
            sum.clear();
            row = next;
          } else if (i0 + i + 1 == to) {   // the next share goes on with it (it may have gone through this one whole)
            tail = row;
#pragma unroll
            for (int k = 0; k < SLICE / 32; ++k) tails[warp][k * 32 + lane] = sum.v[k];
          }
        }
      }
      place[0] = place[1];
      number[0] = number[1];
      place[1] = place2;
      number[1] = number2;
    }
  }
  if (lane == 0) {
    head_row[warp] = head;
    tail_row[warp] = tail;
  }
  __syncthreads();
  if (warp == 0) {
    sum.clear();
    for (int i = 0; i < WARPS; ++i) {
      if (head_row[i] >= 0) {   // the end of the row that is open
#pragma unroll
        for (int k = 0; k < SLICE / 32; ++k) sum.v[k] += heads[i][k * 32 + lane];
        put_row<T, O, WIDE>(out + (static_cast<long long>(head_row[i]) * w.deals + deal) * w.ld_o, sum, width, w.scale, w.add != 0, lane);
        sum.clear();
      }
      if (tail_row[i] >= 0) {
#pragma unroll
        for (int k = 0; k < SLICE / 32; ++k) sum.v[k] += tails[i][k * 32 + lane];
      }
    }
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
      put_row<T, O, WIDE>(out + t * ld_o + c, row, width - c, held ? scale : 0.f, false, lane);
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

struct Deal {
  int slices, slice, deals;
  unsigned long long inverse;
};

// Slices of the columns, and as many deals of the rows as give every SM two CTAs; no CTA more rows than its shared memory counts. The quotient
// v / deals is v * inverse >> 64 with the inverse of 2^64 rounded up (two deals at least, so that it is below 2^64): exact, since the excess
// of v * inverse is below v * deals < 2^64 parts of 1 / deals.
Deal deal_of(int width, int vocab) {
  Deal d;
  d.slices = (width + SLICE - 1) / SLICE;
  d.slice = ((width + d.slices - 1) / d.slices + 7) / 8 * 8;
  d.slices = (width + d.slice - 1) / d.slice;
  int deals = 2 * n_sms() / d.slices;
  if (deals > vocab) deals = vocab;
  if (deals < (vocab - 1) / MOST_ROWS + 1) deals = (vocab - 1) / MOST_ROWS + 1;
  d.deals = deals < 2 ? 2 : deals;
  d.inverse = ~0ull / unsigned(d.deals) + 1;
  return d;
}

template <typename T, typename O, bool WIDE>
int launch_gradient(const Work& w, const Deal& d, cudaStream_t stream) {
  auto kernel = gradient_kernel<T, O, WIDE>;
  static std::atomic<bool> done[64];
  const int status = allow_smem(kernel, MOST_ROWS * 4 + LISTED_BYTES, done);
  if (status != R2_OK) return status;
  const int rows = (w.vocab - 1) / d.deals + 1;
  kernel<<<unsigned(d.slices) * d.deals, THREADS, size_t(rows) * 4 + LISTED_BYTES, stream>>>(w);
  return launch_status();
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

// Bytes of scratch for a gradient.
extern "C" long long r2_token_rows_space(int tokens, int width, int vocab) { return static_cast<long long>(deal_of(width, vocab).slices) * 3 * tokens * 4; }

extern "C" int r2_token_rows_gradient(int dtype, int out_dtype, const int32_t* ids, const void* above, long long ld, void* out, long long ld_o, int tokens, int width,
                                      int vocab, float scale, int add, void* space, cudaStream_t stream) {
  if (tokens < 1 || width < 1 || vocab < 1) return R2_BAD_SHAPE;
  if (tokens > MOST || width > MOST) return R2_UNSUPPORTED;
  const int size = dtype == R2_F32 ? 4 : 2, out_size = out_dtype == R2_F32 ? 4 : 2;
  const Deal d = deal_of(width, vocab);
  const Work w = {ids, above, ld, out, ld_o, tokens, width, vocab, scale, add, d.deals, d.slice, d.inverse, static_cast<int32_t*>(space)};
  const bool wide = at_16(above, ld, size) && at_16(out, ld_o, out_size) && width * size % 16 == 0;
#define R2_CASE(T, O) (wide ? launch_gradient<T, O, true>(w, d, stream) : launch_gradient<T, O, false>(w, d, stream))
  if (dtype == R2_F32 && out_dtype == R2_F32) return R2_CASE(float, float);
  if (dtype == R2_F32 && out_dtype == R2_BF16) return R2_CASE(float, bf16);
  if (dtype == R2_BF16 && out_dtype == R2_F32) return R2_CASE(bf16, float);
  if (dtype == R2_BF16 && out_dtype == R2_BF16) return R2_CASE(bf16, bf16);
#undef R2_CASE
  return R2_BAD_DTYPE;
}
