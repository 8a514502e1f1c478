// The loss of given tokens from hidden rows and a token table, and its gradients, without the logits in memory. With hidden rows x [N, D], table
// W [V, D], tokens y [N] and weights a [N]:
//
//   u = x W^T,  z = u  or  c tanh(u / c),  s_r = log(sum_v exp z_rv),  loss_r = a_r (s_r - z_r,y)
//   dz = a_r (exp(z_rv - s_r) - [v = y_r]) (1 - (z_rv / c)^2),  dx = dz W,  dW = dz^T x
//
// Plain tiles on the CUDA cores: 64 x 64 results a CTA, 4 x 4 a thread.
#include <math.h>

#include "common.cuh"

namespace {

constexpr int TILE = 64, DEPTH = 16;

enum Mode { LOGITS, DZ, STORE, ADD };

struct Operand {
  const void* p;
  long long outer, inner;   // strides of (row of the result or column of it, k)
};

struct Work {
  Operand a, b;
  int m, n, k;
  float softcap;
  const int32_t* targets;
  const float* weight;
  const float* log_sum;
  int first, vocab;          // of the tile's columns: tokens
  float2* part;              // LOGITS: [column tile][row] the largest logit and the sum against it
  float* at_target;          // LOGITS: [row]
  void* out;                 // DZ: float [m, ld]; STORE, ADD: T or float [m, ld]
  long long ld;
};

template <typename TA, typename TB, typename TO, int MODE>
__global__ void __launch_bounds__(256) tile_kernel(const Work w) {
  __shared__ float as[DEPTH][TILE + 4], bs[DEPTH][TILE + 4];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int m0 = blockIdx.y * TILE, n0 = blockIdx.x * TILE;
  const TA* a = static_cast<const TA*>(w.a.p);
  const TB* b = static_cast<const TB*>(w.b.p);
  float acc[4][4] = {};
  for (int k0 = 0; k0 < w.k; k0 += DEPTH) {
    for (int i = threadIdx.x; i < TILE * DEPTH; i += 256) {
      const int r = w.a.inner == 1 ? i / DEPTH : i % TILE, k = w.a.inner == 1 ? i % DEPTH : i / TILE;
      as[k][r] = (m0 + r < w.m && k0 + k < w.k) ? to_float(a[(m0 + r) * w.a.outer + (k0 + k) * w.a.inner]) : 0.f;
    }
    for (int i = threadIdx.x; i < TILE * DEPTH; i += 256) {
      const int r = w.b.inner == 1 ? i / DEPTH : i % TILE, k = w.b.inner == 1 ? i % DEPTH : i / TILE;
      bs[k][r] = (n0 + r < w.n && k0 + k < w.k) ? to_float(b[(n0 + r) * w.b.outer + (k0 + k) * w.b.inner]) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < DEPTH; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float f = as[k][ty * 4 + i];
          // (a row without a target has no part in the table's gradient, whatever it holds)
          if (MODE != STORE || f != 0.f) acc[i][j] = fmaf(f, bs[k][tx * 4 + j], acc[i][j]);
        }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = m0 + ty * 4 + i;
    if (r >= w.m) continue;   // (the sixteen threads of a row go together)
    if constexpr (MODE == LOGITS) {
      float top = -INFINITY, sum = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (w.softcap > 0.f) acc[i][j] = w.softcap * tanhf(acc[i][j] / w.softcap);
        const int v = n0 + tx * 4 + j;
        if (v >= w.n) acc[i][j] = -INFINITY;
        else if (w.targets[r] == w.first + v) w.at_target[r] = acc[i][j];
        top = fmaxf(top, acc[i][j]);
      }
      const unsigned half = 0xffffu << (threadIdx.x & 16);
      for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(half, top, o));
      const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
      for (int j = 0; j < 4; ++j) sum += expf(acc[i][j] - ref);
      for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(half, sum, o);
      if (tx == 0) w.part[size_t(blockIdx.x) * w.m + r] = make_float2(top, sum);
    } else {
      TO* out = static_cast<TO*>(w.out) + r * w.ld;
      const int y = MODE == DZ ? w.targets[r] : 0;
      const float factor = MODE == DZ ? (y >= 0 && y < w.vocab ? (w.weight ? w.weight[r] : 1.f) : 0.f) : 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int v = n0 + tx * 4 + j;
        if (v >= w.n) continue;
        float g = acc[i][j];
        if constexpr (MODE == DZ) {
          float z = g, slope = 1.f;
          if (w.softcap > 0.f) {
            const float t = tanhf(z / w.softcap);
            z = w.softcap * t;
            slope = 1.f - t * t;
          }
          g = factor == 0.f ? 0.f : factor * (expf(z - w.log_sum[r]) - (w.first + v == y ? 1.f : 0.f)) * slope;
        }
        if constexpr (MODE == ADD) g += to_float(out[v]);
        out[v] = from_float<TO>(g);
      }
    }
  }
}

__global__ void finish_kernel(const float2* part, int tiles, const float* at_target, const int32_t* targets, const float* weight, int rows, int vocab,
                              float* loss, float* log_sum) {
  const int r = blockIdx.x * blockDim.x + threadIdx.x;
  if (r >= rows) return;
  float top = -INFINITY, sum = 0.f;
  for (int t = 0; t < tiles; ++t) top = fmaxf(top, part[size_t(t) * rows + r].x);
  const float ref = top == -INFINITY ? 0.f : top;
  for (int t = 0; t < tiles; ++t) {
    const float2 p = part[size_t(t) * rows + r];
    sum += p.x == -INFINITY ? p.y : p.y * expf(p.x - ref);
  }
  const float s = ref + logf(sum);
  log_sum[r] = s;
  const int y = targets[r];
  const float factor = weight ? weight[r] : 1.f;
  loss[r] = (y >= 0 && y < vocab && factor != 0.f) ? factor * (s - at_target[r]) : 0.f;
}

template <typename TA, typename TB, typename TO, int MODE>
void tiles(const Work& w, cudaStream_t stream) {
  tile_kernel<TA, TB, TO, MODE><<<dim3((w.n + TILE - 1) / TILE, (w.m + TILE - 1) / TILE), 256, 0, stream>>>(w);
}

constexpr int PIECE = 8192;   // tokens whose logits' gradients are in memory at a time

template <typename T>
int loss_of(const void* hidden, long long ld_h, const void* table, long long ld_t, int rows, int width, int vocab, const int32_t* targets, const float* weight,
            float softcap, float* loss, float* log_sum, char* space, cudaStream_t stream) {
  Work w = {};
  w.a = {hidden, ld_h, 1};
  w.b = {table, ld_t, 1};
  w.m = rows;
  w.n = vocab;
  w.k = width;
  w.softcap = softcap;
  w.targets = targets;
  w.vocab = vocab;
  w.at_target = reinterpret_cast<float*>(space);
  w.part = reinterpret_cast<float2*>(space + (size_t(rows) * 4 + 15) / 16 * 16);
  tiles<T, T, T, LOGITS>(w, stream);
  finish_kernel<<<(rows + 127) / 128, 128, 0, stream>>>(w.part, (vocab + TILE - 1) / TILE, w.at_target, targets, weight, rows, vocab, loss, log_sum);
  return launch_status();
}

template <typename T>
int gradient_of(const void* hidden, long long ld_h, const void* table, long long ld_t, int rows, int width, int vocab, const int32_t* targets, const float* weight,
                const float* log_sum, float softcap, void* d_hidden, long long ld_dh, void* d_table, long long ld_dt, char* space, cudaStream_t stream) {
  float* dz = reinterpret_cast<float*>(space);
  const int piece = vocab < PIECE ? vocab : PIECE;
  float* sums = dz + size_t(rows) * piece;
  cudaMemsetAsync(sums, 0, size_t(rows) * width * 4, stream);
  for (int first = 0; first < vocab; first += piece) {
    const int n = vocab - first < piece ? vocab - first : piece;
    const T* part = static_cast<const T*>(table) + size_t(first) * ld_t;
    Work w = {};
    w.a = {hidden, ld_h, 1};
    w.b = {part, ld_t, 1};
    w.m = rows;
    w.n = n;
    w.k = width;
    w.softcap = softcap;
    w.targets = targets;
    w.weight = weight;
    w.log_sum = log_sum;
    w.first = first;
    w.vocab = vocab;
    w.out = dz;
    w.ld = piece;
    tiles<T, T, float, DZ>(w, stream);
    if (d_hidden) {
      Work d = {};
      d.a = {dz, piece, 1};
      d.b = {part, 1, ld_t};
      d.m = rows;
      d.n = width;
      d.k = n;
      d.out = sums;
      d.ld = width;
      tiles<float, T, float, ADD>(d, stream);
    }
    if (d_table) {
      Work d = {};
      d.a = {dz, 1, piece};
      d.b = {hidden, 1, ld_h};
      d.m = n;
      d.n = width;
      d.k = rows;
      d.out = static_cast<T*>(d_table) + size_t(first) * ld_dt;
      d.ld = ld_dt;
      tiles<float, T, T, STORE>(d, stream);
    }
  }
  return launch_status();
}

template <typename T>
__global__ void round_kernel(const float* from, T* to, long long ld, int rows, int width) {
  for (size_t i = size_t(blockIdx.x) * blockDim.x + threadIdx.x; i < size_t(rows) * width; i += size_t(gridDim.x) * blockDim.x)
    to[i / width * ld + i % width] = from_float<T>(from[i]);
}

}  // namespace

extern "C" long long r2_token_loss_space(int dtype, int rows, int width, int vocab, int gradient) {
  if (!gradient) return (size_t(rows) * 4 + 15) / 16 * 16 + size_t((vocab + TILE - 1) / TILE) * rows * 8;
  return (size_t(rows) * (vocab < PIECE ? vocab : PIECE) + size_t(rows) * width) * 4;
}

extern "C" int r2_token_loss(int dtype, const void* hidden, long long ld_h, const void* table, long long ld_t, int rows, int width, int vocab,
                             const int32_t* targets, const float* weight, float softcap, float* loss, float* log_sum, void* space, int* error, cudaStream_t stream) {
  if (dtype == R2_F32) return loss_of<float>(hidden, ld_h, table, ld_t, rows, width, vocab, targets, weight, softcap, loss, log_sum, (char*)space, stream);
  if (dtype == R2_BF16) return loss_of<bf16>(hidden, ld_h, table, ld_t, rows, width, vocab, targets, weight, softcap, loss, log_sum, (char*)space, stream);
  return R2_BAD_DTYPE;
}

extern "C" int r2_token_loss_gradient(int dtype, const void* hidden, long long ld_h, const void* table, long long ld_t, int rows, int width, int vocab,
                                      const int32_t* targets, const float* weight, const float* log_sum, float softcap, void* d_hidden, long long ld_dh,
                                      void* d_table, long long ld_dt, void* space, int* error, cudaStream_t stream) {
  const float* sums = (const float*)space + size_t(rows) * (vocab < PIECE ? vocab : PIECE);
  const int grid = int((size_t(rows) * width + 255) / 256 < 4096 ? (size_t(rows) * width + 255) / 256 : 4096);
  int status;
  if (dtype == R2_F32) {
    status = gradient_of<float>(hidden, ld_h, table, ld_t, rows, width, vocab, targets, weight, log_sum, softcap, d_hidden, ld_dh, d_table, ld_dt, (char*)space, stream);
    if (status == R2_OK && d_hidden) round_kernel<float><<<grid, 256, 0, stream>>>(sums, (float*)d_hidden, ld_dh, rows, width);
  } else if (dtype == R2_BF16) {
    status = gradient_of<bf16>(hidden, ld_h, table, ld_t, rows, width, vocab, targets, weight, log_sum, softcap, d_hidden, ld_dh, d_table, ld_dt, (char*)space, stream);
    if (status == R2_OK && d_hidden) round_kernel<bf16><<<grid, 256, 0, stream>>>(sums, (bf16*)d_hidden, ld_dh, rows, width);
  } else {
    return R2_BAD_DTYPE;
  }
  return status == R2_OK ? launch_status() : status;
}
