// A student's loss against a teacher's top logits, and its gradient with respect to the student's logits.
//
//   q = softmax(x / tau) over the whole row; p_k = exp(t_k / tau - log_sum) for the listed tokens, and one more outcome, "another token",
//   with what is left of the teacher's mass and of q; without log_sum p = softmax(t / tau) over the listed tokens and no such outcome.
//   loss = w tau^2 KL(p || q)
//   d loss / d x_j = w tau (q_j P - p_j)                               j listed, P the mass of all outcomes (1 with "another token")
//                    w tau q_j (sum p - sum q over the listed) / rest  j not listed, rest = q's mass outside the list
//                    w tau q_j sum p                                   j not listed, without "another token"
//
// With "another token" both sides are whole distributions and the loss is summed as p log(p / q) - p + q, terms that are never negative: a
// teacher and a student that nearly agree lose no digits to cancellation, and for the same reason the mass outside the list is summed from its own
// tokens, not taken from 1. A row whose weight is 0 is not read: its loss and gradient are 0 whatever stands there.
#include "logit_rows.cuh"

namespace {

constexpr int THREADS = 512;
constexpr int MOST_K = 256;

struct DistillArgs {
  const void* logits; long long ld;
  int vocab, k;
  const int32_t* ids; const float* teacher; const float* log_sum; const float* weight;
  float tau;
  float* loss;
  void* grad; long long grad_ld;
};

template <typename T>
__global__ void __launch_bounds__(THREADS)
distill_kernel(const DistillArgs a) {
  __shared__ float scratch[33];
  __shared__ int32_t ids[MOST_K];
  __shared__ float p[MOST_K], xk[MOST_K];
  __shared__ unsigned char once[MOST_K];   // the entry is the first that names its token
  pdl_launch_dependents();
  pdl_wait();
  const int row = int(blockIdx.x), tid = int(threadIdx.x), k = a.k;
  const T* x = static_cast<const T*>(a.logits) + (long long)row * a.ld;
  T* grad = a.grad != nullptr ? static_cast<T*>(a.grad) + (long long)row * a.grad_ld : nullptr;
  const float w = a.weight != nullptr ? a.weight[row] : 1.f;
  if (w == 0.f) {
    if (grad != nullptr)
      for (int i = tid; i < a.vocab; i += THREADS) grad[i] = from_float<T>(0.f);
    if (tid == 0) a.loss[row] = 0.f;
    return;
  }
  const float inv = 1.f / a.tau;
  float t = -INFINITY;
  if (tid < k) {
    const int id = a.ids[(long long)row * k + tid];
    const bool held = id >= 0 && id < a.vocab;
    ids[tid] = held ? id : -1;
    xk[tid] = held ? to_float(x[id]) : 0.f;
    if (held) t = a.teacher[(long long)row * k + tid] * inv;
  }
  float m = -INFINITY;
  for (int i = tid; i < a.vocab; i += THREADS) m = fmaxf(m, to_float(x[i]));
  float t_max = warp_max(t);
  m = warp_max(m);
  if ((tid & 31) == 0) scratch[tid >> 5] = m;
  __syncthreads();
  for (int i = 0; i < THREADS / 32; ++i) m = fmaxf(m, scratch[i]);
  __syncthreads();
  if ((tid & 31) == 0) scratch[tid >> 5] = t_max;
  __syncthreads();
  for (int i = 0; i < THREADS / 32; ++i) t_max = fmaxf(t_max, scratch[i]);
  const bool tail = a.log_sum != nullptr;
  float log_p = -INFINITY;
  if (tail) {
    log_p = t - a.log_sum[row];
  } else {
    const float total_t = block_sum(t == -INFINITY ? 0.f : expf(t - t_max), scratch);
    if (t != -INFINITY) log_p = t - t_max - logf(total_t);
  }
  const float pk = log_p == -INFINITY ? 0.f : expf(log_p);
  if (tid < k) {
    p[tid] = pk;
    bool first = ids[tid] >= 0;
    for (int j = 0; j < tid && first; ++j) first = ids[j] != ids[tid];
    once[tid] = first;
  }
  __syncthreads();
  const float mass = block_sum(pk, scratch);
  float sum = 0.f, rest = 0.f;
  for (int i = tid; i < a.vocab; i += THREADS) {
    const float e = expf((to_float(x[i]) - m) * inv);
    sum += e;
    bool listed = false;
    if (tail)
      for (int j = 0; j < k && !listed; ++j) listed = ids[j] == i;
    if (!listed) rest += e;
  }
  const float total = block_sum(sum, scratch);
  rest = block_sum(rest, scratch) / total;
  const float log_total = logf(total);
  const float log_q = tid < k && ids[tid] >= 0 ? (xk[tid] - m) * inv - log_total : 0.f;
  const float qk = tid < k && once[tid] ? expf(log_q) : 0.f;
  const float d = log_p - log_q;
  const float rest_p = tail && rest > 0.f ? fmaxf(1.f - mass, 0.f) : 0.f;
  float term = 0.f, outside = mass, whole = mass;
  if (tid < k && ids[tid] >= 0) term = tail ? (pk > 0.f ? pk * d - pk : 0.f) + qk : (pk > 0.f ? pk * d : 0.f);
  if (tail && pk > 0.f && tid < k && once[tid]) term = pk * (d + expm1f(-d));
  float kl = block_sum(term, scratch);
  const float mass_q = block_sum(qk, scratch);
  if (tail) {
    if (rest_p > 0.f) {
      const float rest_d = logf(rest_p) - logf(rest);
      kl += rest_p * (rest_d + expm1f(-rest_d));
      outside = (mass - mass_q) / rest;
      whole = 1.f;
    } else {
      kl += rest > 0.f ? rest : mass - 1.f;
    }
  }
  if (tid == 0) a.loss[row] = w * a.tau * a.tau * kl;
  if (grad == nullptr) return;
  const float scale = w * a.tau, by = scale * outside / total;
  __syncthreads();
  for (int i = tid; i < a.vocab; i += THREADS) grad[i] = from_float<T>(by * expf((to_float(x[i]) - m) * inv));
  __syncthreads();
  if (tid < k && once[tid]) {
    float listed_p = 0.f;
    for (int j = 0; j < k; ++j) listed_p += ids[j] == ids[tid] ? p[j] : 0.f;
    grad[ids[tid]] = from_float<T>(scale * (qk * whole - listed_p));
  }
}

}  // namespace

// logits [rows, vocab] of dtype with row stride ld, ids and teacher [rows, k] (an id outside the vocabulary: no entry), log_sum and weight
// [rows] or null -> loss [rows] float; grad [rows, vocab] of dtype with row stride grad_ld, null, or the logits themselves.
extern "C" int r2_distill(int dtype, const void* logits, long long ld, int rows, int vocab, const int32_t* ids, const float* teacher, int k,
                          const float* log_sum, const float* weight, float temperature, float* loss, void* grad, long long grad_ld,
                          cudaStream_t stream) {
  if (dtype != R2_F32 && dtype != R2_BF16) return R2_BAD_DTYPE;
  if (rows < 0 || vocab < 1 || vocab > (1 << 30) || ld < vocab || (grad != nullptr && grad_ld < vocab) || k < 1) return R2_BAD_SHAPE;
  if (k > MOST_K || !(temperature > 0.f)) return R2_UNSUPPORTED;
  if (rows == 0) return R2_OK;
  const DistillArgs a = {logits, ld, vocab, k, ids, teacher, log_sum, weight, temperature, loss, grad, grad_ld};
  if (dtype == R2_F32) r2_launch(distill_kernel<float>, dim3(unsigned(rows)), dim3(THREADS), size_t(0), stream, a);
  else r2_launch(distill_kernel<bf16>, dim3(unsigned(rows)), dim3(THREADS), size_t(0), stream, a);
  return launch_status();
}
