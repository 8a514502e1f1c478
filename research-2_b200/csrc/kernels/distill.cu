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
//
// A row is read once and its gradient written once: the CTAs of a cluster hold a row's 16-byte pieces in registers between the two. A
// thread sums exponentials against its own maximum, warps and CTAs join these with their maxima, and one cluster barrier stands between
// the sums and the gradient; float32 rows keep the exponentials in the logits' place, so that each is computed once. Rows beyond what
// eight CTAs hold are read a second time.
#include "logit_rows.cuh"

namespace {

constexpr int MOST_K = 256;
constexpr int MOST_RANKS = 8;
constexpr int PIECES = 8;   // of a thread, in registers

struct DistillArgs {
  const void* logits; long long ld;
  int vocab, k, ranks;
  const int32_t* ids; const float* teacher; const float* log_sum; const float* weight;
  float tau;
  float* loss;
  void* grad; long long grad_ld;
};

__device__ __forceinline__ float no_less(float reference) { return reference == -INFINITY ? 0.f : reference; }
// what sums against `reference` are in sums against `common`, the largest of several references
__device__ __forceinline__ float rebase(float reference, float common) { return reference == -INFINITY ? 0.f : exp2_approx(reference - common); }

// One (reference, sum over listed, sum over others) per lane into one per warp.
__device__ __forceinline__ float3 warp_join(float3 v) {
  const float common = warp_max(v.x), f = rebase(v.x, common);
  return make_float3(common, warp_sum(v.y * f), warp_sum(v.z * f));
}

// ONE: a CTA's share of a row fits its registers. TAIL: there is a log_sum.
template <typename T, int THREADS, bool ONE, bool TAIL>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS)
distill_kernel(const DistillArgs a) {
  constexpr int PER = RowPieces<T>::PER, CHUNK = THREADS * PIECES, WORDS = CHUNK * PER / 32;
  constexpr bool KEEP = ONE && sizeof(T) == 4;   // exponentials stand in the logits' place
  __shared__ uint32_t listed[WORDS];
  __shared__ float parts[THREADS / 32][4];
  __shared__ __align__(16) float4 shares[MOST_RANKS];
  __shared__ int32_t ids[MOST_K];
  __shared__ float teacher[MOST_K], xk[MOST_K];
  __shared__ int twice;
  pdl_launch_dependents();
  const int ranks = a.ranks, row = int(blockIdx.x) / ranks, rank = int(blockIdx.x) % ranks, tid = int(threadIdx.x), lane = tid & 31, k = a.k;
  if (tid == 0) twice = 0;
  pdl_wait();
  const RowPieces<T> x(static_cast<const T*>(a.logits) + (long long)row * a.ld, a.vocab);
  T* grad = a.grad != nullptr ? static_cast<T*>(a.grad) + (long long)row * a.grad_ld : nullptr;
  const bool vectors = ((reinterpret_cast<uintptr_t>(grad) ^ reinterpret_cast<uintptr_t>(x.base + x.phase)) & 15) == 0;
  const int per = (x.count + ranks - 1) / ranks, g0 = rank * per, n = max(0, min(per, x.count - g0));
  const float w = a.weight != nullptr ? a.weight[row] : 1.f;
  if (w == 0.f) {  // (every CTA of the cluster)
    if (grad != nullptr) {
      const float zeros[PER] = {};
      for (int i = tid; i < n; i += THREADS) store_piece<T, PER>(grad, x.first(g0 + i), a.vocab, zeros, vectors);
    }
    if (rank == 0 && tid == 0) a.loss[row] = 0.f;
    return;
  }
  if (ranks > 1) cluster_arrive();   // this CTA runs: the others may write into its shared memory once all have arrived

  uint4 raw[PIECES];
  auto load = [&](int c0) {
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int at = c0 + tid + i * THREADS;
      if (at < n) raw[i] = load_once(x, g0 + at);
    }
  };
  load(0);
  const float inv = 1.f / a.tau, c = 1.44269504f / a.tau;
  for (int j = tid; j < k; j += THREADS) {
    const int id = a.ids[(long long)row * k + j];
    const bool held = id >= 0 && id < a.vocab;
    ids[j] = held ? id : -1;
    teacher[j] = held ? a.teacher[(long long)row * k + j] * inv : -INFINITY;
    xk[j] = held ? to_float(x.base[x.phase + id]) : 0.f;
  }

  float3 sums = make_float3(-INFINITY, 0.f, 0.f);   // this thread's reference (an exponent of two), over listed tokens, over the others
  for (int c0 = 0; ONE ? c0 == 0 : c0 < n; c0 += CHUNK) {
    if (!ONE && c0 > 0) {
      __syncthreads();
      load(c0);
    }
    if (TAIL || c0 == 0) {
      const int zero = x.first(g0 + c0);   // the token of the first bit
      for (int i = tid; i < WORDS; i += THREADS) listed[i] = 0u;
      __syncthreads();
      for (int j = tid; j < k; j += THREADS) {
        const int at = ids[j] - zero;
        if (ids[j] >= 0 && at >= 0 && at < CHUNK * PER) {
          const uint32_t bit = 1u << (at & 31);
          if (atomicOr(&listed[at >> 5], bit) & bit) twice = 1;
        }
      }
      __syncthreads();
    }
    float most = -INFINITY;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int at = c0 + tid + i * THREADS;
      if (at >= n) continue;
      blank_outside(raw[i], x, g0 + at);
      float v[PER];
      unpack(raw[i], v, static_cast<const T*>(nullptr));
#pragma unroll
      for (int e = 0; e < PER; ++e) most = fmaxf(most, v[e]);
    }
    const float reference = fmaxf(sums.x, most * c), shift = no_less(reference);
    if (!ONE) {
      const float f = rebase(sums.x, shift);
      sums.y *= f;
      sums.z *= f;
    }
    sums.x = reference;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int at = tid + i * THREADS;
      if (c0 + at >= n) continue;
      float v[PER];
      unpack(raw[i], v, static_cast<const T*>(nullptr));
#pragma unroll
      for (int e = 0; e < PER; ++e) v[e] = exp2_approx(fmaf(v[e], c, -shift));
      float all = 0.f;
#pragma unroll
      for (int e = 0; e < PER; ++e) all += v[e];
      uint32_t bits = 0u;
      if (TAIL) bits = (listed[at * PER / 32] >> (at * PER % 32)) & ((1u << PER) - 1u);
      if (bits == 0u) {
        sums.z += all;
      } else {
#pragma unroll
        for (int e = 0; e < PER; ++e) {
          if ((bits >> e) & 1u) sums.y += v[e];
          else sums.z += v[e];
        }
      }
      if (KEEP) raw[i] = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    }
  }

  // the teacher's side, in every warp for itself: no barrier
  float t_sum = 0.f, mass = 0.f;
  if (TAIL) {
    t_sum = a.log_sum[row];
  } else {
    float t_max = -INFINITY;
    for (int j = lane; j < k; j += 32) t_max = fmaxf(t_max, teacher[j]);
    t_max = no_less(warp_max(t_max));
    for (int j = lane; j < k; j += 32) t_sum += teacher[j] == -INFINITY ? 0.f : expf(teacher[j] - t_max);
    t_sum = t_max + logf(warp_sum(t_sum));
  }
  auto log_p = [&](int j) { return teacher[j] == -INFINITY ? -INFINITY : teacher[j] - t_sum; };
  for (int j = lane; j < k; j += 32) mass += expf(log_p(j));
  mass = warp_sum(mass);

  const float own_reference = sums.x;
  sums = warp_join(sums);
  if (lane == 0) {
    parts[tid >> 5][0] = sums.x;
    parts[tid >> 5][1] = sums.y;
    parts[tid >> 5][2] = sums.z;
  }
  __syncthreads();
  if (tid < 32) {
    const bool some = tid < THREADS / 32;
    const float3 v = warp_join(make_float3(some ? parts[tid % (THREADS / 32)][0] : -INFINITY, some ? parts[tid % (THREADS / 32)][1] : 0.f,
                                           some ? parts[tid % (THREADS / 32)][2] : 0.f));
    if (ranks > 1) {
      cluster_wait();
      if (tid < ranks) cluster_store(cluster_address(&shares[rank], tid), make_float4(v.x, v.y, v.z, 0.f));
    } else if (tid == 0) {
      shares[0] = make_float4(v.x, v.y, v.z, 0.f);
    }
  } else if (ranks > 1) {
    cluster_wait();
  }
  if (ranks > 1) {
    cluster_arrive();
    cluster_wait();
  } else {
    __syncthreads();
  }
  float common = -INFINITY, in_list = 0.f, rest = 0.f;
  for (int r = 0; r < ranks; ++r) common = fmaxf(common, shares[r].x);
  for (int r = 0; r < ranks; ++r) {
    const float f = rebase(shares[r].x, common);
    in_list += shares[r].y * f;
    rest += shares[r].z * f;
  }
  const float total = in_list + rest;   // (without TAIL everything stands in `rest`)
  float outside = mass, whole = mass, rest_p = 0.f;
  rest /= total;
  if (TAIL) {
    rest_p = rest > 0.f ? fmaxf(1.f - mass, 0.f) : 0.f;
    if (rest_p > 0.f) {
      outside = (mass - in_list / total) / rest;
      whole = 1.f;
    }
  }
  const float log2_total = log2f(total), log2_e = 0.693147181f;
  if (rank == 0 && tid < 32) {
    float kl = 0.f;
    for (int j = lane; j < k; j += 32) {
      if (ids[j] < 0) continue;
      const float lq = (fmaf(xk[j], c, -common) - log2_total) * log2_e, lp = log_p(j), p = expf(lp), d = lp - lq;
      if (TAIL) kl += p > 0.f ? p * (d + expm1f(-d)) : expf(lq);
      else if (p > 0.f) kl += p * d;
    }
    kl = warp_sum(kl);
    if (TAIL) {
      const float d = logf(rest_p) - logf(rest);
      kl += rest_p > 0.f ? rest_p * (d + expm1f(-d)) : rest > 0.f ? rest : mass - 1.f;
    }
    if (lane == 0) a.loss[row] = w * a.tau * a.tau * kl;
  }
  if (grad == nullptr) return;

  const float scale = w * a.tau, by = scale * outside / total, f = rebase(own_reference, common) * by;
  for (int c0 = 0; ONE ? c0 == 0 : c0 < n; c0 += CHUNK) {
    if (!ONE) load(c0);
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int at = c0 + tid + i * THREADS;
      if (at >= n) continue;
      float v[PER];
      unpack(raw[i], v, static_cast<const T*>(nullptr));
#pragma unroll
      for (int e = 0; e < PER; ++e) v[e] = KEEP ? v[e] * f : exp2_approx(fmaf(v[e], c, -common)) * by;
      store_piece<T, PER>(grad, x.first(g0 + at), a.vocab, v, vectors);
    }
  }
  __syncthreads();   // what follows lies over it
  const int from = x.first(g0), to = from + n * PER;
  for (int j = tid; j < k; j += THREADS) {
    const int id = ids[j];
    if (id < 0 || id < from || id >= to) continue;
    float p = expf(log_p(j));
    if (twice) {  // a list that names a token more than once: its first entry writes for all
      bool earlier = false;
      p = 0.f;
      for (int o = 0; o < k; ++o) {
        if (ids[o] != id) continue;
        earlier |= o < j;
        p += expf(log_p(o));
      }
      if (earlier) continue;
    }
    grad[id] = from_float<T>(scale * (exp2_approx(fmaf(xk[j], c, -common)) / total * whole - p));
  }
}

template <typename T, int THREADS, bool ONE>
void launch_tail(const DistillArgs& a, int rows, cudaStream_t stream) {
  const dim3 grid(unsigned(rows) * unsigned(a.ranks));
  if (a.log_sum != nullptr) r2_launch_clusters(distill_kernel<T, THREADS, ONE, true>, a.ranks, grid, dim3(THREADS), size_t(0), stream, a);
  else r2_launch_clusters(distill_kernel<T, THREADS, ONE, false>, a.ranks, grid, dim3(THREADS), size_t(0), stream, a);
}

template <typename T>
int launch(DistillArgs a, int rows, cudaStream_t stream) {
  const int pieces = (a.vocab + 2 * RowPieces<T>::PER - 2) / RowPieces<T>::PER;   // of a row at any alignment, at most
  if (pieces <= 128 * PIECES) {
    a.ranks = 1;
    launch_tail<T, 128, true>(a, rows, stream);
    return launch_status();
  }
  a.ranks = min(MOST_RANKS, (pieces + 512 * PIECES - 1) / (512 * PIECES));
  if ((long long)rows * a.ranks > 0x7fffffffLL) return R2_BAD_SHAPE;
  if ((pieces + a.ranks - 1) / a.ranks <= 512 * PIECES) launch_tail<T, 512, true>(a, rows, stream);
  else launch_tail<T, 512, false>(a, rows, stream);
  return launch_status();
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
  const DistillArgs a = {logits, ld, vocab, k, 1, ids, teacher, log_sum, weight, temperature, loss, grad, grad_ld};
  return dtype == R2_F32 ? launch<float>(a, rows, stream) : launch<bf16>(a, rows, stream);
}
