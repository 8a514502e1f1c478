// The k largest logits of every row with their tokens, from the largest down, equal values from the lowest token up, and the logarithm of
// the row's sum of exponentials at a temperature.
#include "logit_rows.cuh"

namespace {

constexpr int THREADS = 512;
constexpr int MOST_K = 256;

__device__ __forceinline__ unsigned long long warp_max_u64(unsigned long long v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long other = __shfl_xor_sync(0xffffffffu, v, o);
    v = other > v ? other : v;
  }
  return v;
}

template <typename T>
__global__ void __launch_bounds__(THREADS)
top_kernel(const T* logits, long long ld, int vocab, int k, float inv_temperature, float* values, int32_t* ids, float* log_sum) {
  __shared__ unsigned long long best_s[THREADS / 32];
  __shared__ float scratch[33];
  pdl_launch_dependents();
  pdl_wait();
  const int row = int(blockIdx.x), tid = int(threadIdx.x);
  const T* x = logits + (long long)row * ld;
  unsigned long long below = ~0ull;
  for (int n = 0; n < k; ++n) {
    unsigned long long mine = 0ull;
    for (int i = tid; i < vocab; i += THREADS) {
      const unsigned long long c = (static_cast<unsigned long long>(logit_key(to_float(x[i]))) << 32) | (0xffffffffu - unsigned(i));
      if (c < below && c > mine) mine = c;
    }
    mine = warp_max_u64(mine);
    __syncthreads();
    if ((tid & 31) == 0) best_s[tid >> 5] = mine;
    __syncthreads();
    unsigned long long best = best_s[0];
    for (int w = 1; w < THREADS / 32; ++w) best = best_s[w] > best ? best_s[w] : best;
    below = best;
    if (tid == 0) {
      const int id = int(0xffffffffu - unsigned(best & 0xffffffffu));
      values[(long long)row * k + n] = to_float(x[id]);
      ids[(long long)row * k + n] = id;
    }
  }
  if (log_sum == nullptr) return;
  float m = -INFINITY;
  for (int i = tid; i < vocab; i += THREADS) m = fmaxf(m, to_float(x[i]));
  m = warp_max(m);
  __syncthreads();
  if ((tid & 31) == 0) scratch[tid >> 5] = m;
  __syncthreads();
  for (int w = 0; w < THREADS / 32; ++w) m = fmaxf(m, scratch[w]);
  const float shift = fabsf(m) == INFINITY ? 0.f : m;
  float sum = 0.f;
  for (int i = tid; i < vocab; i += THREADS) sum += expf((to_float(x[i]) - shift) * inv_temperature);
  sum = block_sum(sum, scratch);
  if (tid == 0) log_sum[row] = shift * inv_temperature + logf(sum);
}

}  // namespace

// logits [rows, vocab] of dtype with row stride ld -> values [rows, k] float and ids [rows, k]; log_sum [rows] may be null.
extern "C" int r2_top_logits(int dtype, const void* logits, long long ld, int rows, int vocab, int k, float temperature, float* values,
                             int32_t* ids, float* log_sum, cudaStream_t stream) {
  if (dtype != R2_F32 && dtype != R2_BF16) return R2_BAD_DTYPE;
  if (rows < 0 || vocab < 1 || vocab > (1 << 30) || ld < vocab || k < 1 || k > vocab) return R2_BAD_SHAPE;
  if (k > MOST_K || !(temperature > 0.f)) return R2_UNSUPPORTED;
  if (rows == 0) return R2_OK;
  if (dtype == R2_F32)
    r2_launch(top_kernel<float>, dim3(unsigned(rows)), dim3(THREADS), size_t(0), stream, static_cast<const float*>(logits), ld, vocab, k,
              1.f / temperature, values, ids, log_sum);
  else
    r2_launch(top_kernel<bf16>, dim3(unsigned(rows)), dim3(THREADS), size_t(0), stream, static_cast<const bf16*>(logits), ld, vocab, k,
              1.f / temperature, values, ids, log_sum);
  return launch_status();
}
