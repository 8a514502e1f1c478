// Rows of a token table, and the gradient of the table whose rows were looked up:
//
//   out_t = scale * W[i_t]  (zeros where i_t is no token),   dW_v = scale * sum over t with i_t = v of above_t, in one order
//
// The gradient is one launch and needs nothing between CTAs. The table's rows are dealt out by the low bits of their number (tokens that stand often
// lie side by side in a vocabulary), its columns in slices, and a CTA owns a deal and a slice: it goes through all tokens, lists the places of its own in
// their order, sorts the list by token (a count, a running sum, a stable placing) and writes every row that it owns: zeros, or the sum. Going through
// the tokens costs each CTA 4 bytes a token, read from L2; the rows from above, which are hundreds of times as much, are read once. A row of more than 64 places is
// added by the CTA's eight warps, a share of the places each, and the shares in order.
//
// Bound by the bytes of the rows from above and of the table.
#include "common.cuh"

namespace {

constexpr int THREADS = 256, WARPS = 8;
constexpr int SLICE = 256;          // columns of a CTA at most
constexpr int LISTED = 4096;        // places that shared memory holds (beyond them: the scratch)
constexpr int MOST_ROWS = 8192;     // of a CTA
constexpr int ALONE = 64;           // the most places that a warp adds by itself

struct Work {
  const int32_t* ids;
  const void* above;
  long long ld;
  void* out;
  long long ld_o;
  int tokens, width, vocab;
  float scale;
  int add;
  int deal_bits, slice;             // rows v with v mod 2^deal_bits = the CTA's; columns of a slice
  int32_t* spill;                   // [slice][3][tokens]
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

// The rows at places [begin, end) of the sorted list, in order, eight on their way at a time.
template <typename T, bool WIDE>
__device__ __forceinline__ void add_rows(Lane<T, WIDE>& sum, const int32_t* sorted, int begin, int end, const T* above, long long ld, int width, int lane) {
  constexpr int AHEAD = 8;
  int i = begin;
  for (; i + AHEAD <= end; i += AHEAD) {
    Raw<T, WIDE> raw[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) raw[j].load(above + sorted[i + j] * ld, width, lane);
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) raw[j].add_to(sum);
  }
  if (i < end) {
    Raw<T, WIDE> raw[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
      if (i + j < end) raw[j].load(above + sorted[i + j] * ld, width, lane);
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
      if (i + j < end) raw[j].add_to(sum);
  }
}

template <typename T, typename O, bool WIDE>
__global__ void __launch_bounds__(THREADS, 2) gradient_kernel(const Work w) {
  extern __shared__ int32_t shared[];
  __shared__ int mine[WARPS], lower[WARPS], running[WARPS];
  __shared__ float shares[WARPS][SLICE];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int deals = 1 << w.deal_bits, deal = blockIdx.x & (deals - 1), slice = blockIdx.x >> w.deal_bits;
  const int rows = int((static_cast<long long>(w.vocab) - deal + deals - 1) >> w.deal_bits);   // that this CTA owns; 0 for a deal beyond the vocabulary
  int32_t* ends = shared;                                         // [rows]: counts, then where a row's places begin, then where they end

  for (int j = threadIdx.x; j < rows; j += THREADS) ends[j] = 0;
  __syncthreads();

  // ---- a warp's share of the places: how many are this CTA's, how many of a lower deal
  const int share = ((w.tokens + WARPS - 1) / WARPS + 127) / 128 * 128;
  const int first = min(static_cast<long long>(warp) * share, static_cast<long long>(w.tokens)), last = min(static_cast<long long>(first) + share, static_cast<long long>(w.tokens));
  int n_mine = 0, n_lower = 0;
  for (int t0 = first; t0 < last; t0 += 128) {
    int id[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) id[j] = t0 + 32 * j + lane < last ? __ldg(w.ids + t0 + 32 * j + lane) : -1;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool token = id[j] >= 0 && id[j] < w.vocab;
      const int at = id[j] & (deals - 1);
      if (token && at == deal) {
        atomicAdd(&ends[id[j] >> w.deal_bits], 1);
        ++n_mine;
      }
      n_lower += token && at < deal ? 1 : 0;
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
  // the list (token and place) and the sorted places: in shared memory, or in this deal's part of the slice's scratch
  int32_t *list_row, *list_place, *sorted;
  if (total <= LISTED) {
    list_row = shared + rows;
    list_place = list_row + LISTED;
    sorted = list_place + LISTED;
  } else {
    list_row = w.spill + static_cast<long long>(slice) * 3 * w.tokens + offset;
    list_place = list_row + w.tokens;
    sorted = list_place + w.tokens;
  }
  if (total > 0) {
    if (n_mine > 0) {
      for (int t0 = first; t0 < last; t0 += 128) {
        int id[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) id[j] = t0 + 32 * j + lane < last ? __ldg(w.ids + t0 + 32 * j + lane) : -1;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const bool own = id[j] >= 0 && id[j] < w.vocab && (id[j] & (deals - 1)) == deal;
          const unsigned mask = __ballot_sync(0xffffffffu, own);
          if (own) {
            const int at = before + __popc(mask & ((1u << lane) - 1u));
            list_row[at] = id[j] >> w.deal_bits;
            list_place[at] = t0 + 32 * j + lane;
          }
          before += __popc(mask);
        }
      }
    }
    // where each row's places begin: a thread's share of the rows, then the threads'
    const int per = (rows + THREADS - 1) / THREADS, from = min(rows, int(threadIdx.x) * per), to = min(rows, from + per);
    int sum = 0;
    for (int j = from; j < to; ++j) sum += ends[j];
    int up = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, up, o);
      up += lane >= o ? x : 0;
    }
    if (lane == 31) running[warp] = up;
    __syncthreads();
    int begin = up - sum;
#pragma unroll
    for (int i = 0; i < WARPS; ++i) begin += i < warp ? running[i] : 0;
    for (int j = from; j < to; ++j) {
      const int n = ends[j];
      ends[j] = begin;
      begin += n;
    }
    __syncthreads();
    // a stable placing: a warp takes the rows of its number mod 8 from the list, in the list's order
    for (int i0 = 0; i0 < total; i0 += 32) {
      const int row = i0 + lane < total ? list_row[i0 + lane] : -1;
      const bool own = row >= 0 && (row & (WARPS - 1)) == warp;
      const unsigned owners = __ballot_sync(0xffffffffu, own);
      if (owners == 0) continue;
      int at = 0;
      unsigned peers = 0;
      if (own) {
        peers = __match_any_sync(owners, row);
        at = ends[row] + __popc(peers & ((1u << lane) - 1u));
        sorted[at] = list_place[i0 + lane];
      }
      __syncwarp();
      if (own && (peers >> lane) == 1u) ends[row] = at + 1;   // (the last of them)
      __syncwarp();
    }
    __syncthreads();
  }

  // ---- the rows: a warp one, where it has few places
  const int col = slice * w.slice, width = min(w.slice, w.width - col);
  const T* above = static_cast<const T*>(w.above) + col;
  O* out = static_cast<O*>(w.out) + col;
  for (int j = warp; j < rows; j += WARPS) {
    const int begin = j > 0 ? ends[j - 1] : 0, end = ends[j];   // (all zeros where the CTA has no place at all)
    if (end - begin > ALONE || (end == begin && w.add)) continue;
    Lane<T, WIDE> sum;
    sum.clear();
    add_rows<T, WIDE>(sum, sorted, begin, end, above, w.ld, width, lane);
    put_row<T, O, WIDE>(out + ((static_cast<long long>(j) << w.deal_bits) + deal) * w.ld_o, sum, width, w.scale, w.add != 0, lane);
  }
  if (total <= ALONE) return;
  // ---- and all warps one, where it has many
  for (int j0 = 0; j0 < rows; j0 += 32) {
    const int j = j0 + lane;
    unsigned many = __ballot_sync(0xffffffffu, j < rows && ends[j] - (j > 0 ? ends[j - 1] : 0) > ALONE);
    while (many != 0) {
      const int row = j0 + __ffs(int(many)) - 1;
      many &= many - 1;
      const int begin = row > 0 ? ends[row - 1] : 0, n = ends[row] - begin, part = (n + WARPS - 1) / WARPS;
      Lane<T, WIDE> sum;
      sum.clear();
      add_rows<T, WIDE>(sum, sorted, begin + min(n, warp * part), begin + min(n, (warp + 1) * part), above, w.ld, width, lane);
#pragma unroll
      for (int i = 0; i < SLICE / 32; ++i) shares[warp][i * 32 + lane] = sum.v[i];
      __syncthreads();
      if (warp == 0) {
        for (int other = 1; other < WARPS; ++other)
#pragma unroll
          for (int i = 0; i < SLICE / 32; ++i) sum.v[i] += shares[other][i * 32 + lane];
        put_row<T, O, WIDE>(out + ((static_cast<long long>(row) << w.deal_bits) + deal) * w.ld_o, sum, width, w.scale, w.add != 0, lane);
      }
      __syncthreads();
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
  int slices, slice, bits;
};

// Slices of the columns, and as many deals of the rows as give every SM two CTAs; no CTA more rows than its shared memory counts.
Deal deal_of(int width, int vocab) {
  Deal d;
  d.slices = (width + SLICE - 1) / SLICE;
  d.slice = ((width + d.slices - 1) / d.slices + 7) / 8 * 8;
  d.slices = (width + d.slice - 1) / d.slice;
  d.bits = 0;
  while (d.bits < 30 && (((1ll << d.bits) * d.slices < 2 * n_sms() && (1 << d.bits) < vocab) || ((vocab - 1) >> d.bits) >= MOST_ROWS)) ++d.bits;
  return d;
}

template <typename T, typename O, bool WIDE>
int launch_gradient(const Work& w, const Deal& d, cudaStream_t stream) {
  auto kernel = gradient_kernel<T, O, WIDE>;
  static std::atomic<bool> done[64];
  const int status = allow_smem(kernel, (MOST_ROWS + 3 * LISTED) * 4, done);
  if (status != R2_OK) return status;
  const int rows = ((w.vocab - 1) >> d.bits) + 1;
  kernel<<<unsigned(d.slices) << d.bits, THREADS, (rows + 3 * LISTED) * 4, stream>>>(w);
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
  const Work w = {ids, above, ld, out, ld_o, tokens, width, vocab, scale, add, d.bits, d.slice, static_cast<int32_t*>(space)};
  const bool wide = at_16(above, ld, size) && at_16(out, ld_o, out_size) && width * size % 16 == 0;
#define R2_CASE(T, O) (wide ? launch_gradient<T, O, true>(w, d, stream) : launch_gradient<T, O, false>(w, d, stream))
  if (dtype == R2_F32 && out_dtype == R2_F32) return R2_CASE(float, float);
  if (dtype == R2_F32 && out_dtype == R2_BF16) return R2_CASE(float, bf16);
  if (dtype == R2_BF16 && out_dtype == R2_F32) return R2_CASE(bf16, float);
  if (dtype == R2_BF16 && out_dtype == R2_BF16) return R2_CASE(bf16, bf16);
#undef R2_CASE
  return R2_BAD_DTYPE;
}
