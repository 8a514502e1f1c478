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
// tokens, not taken from 1. It is summed against a reference of its own: against the row's largest logit it would be nothing in 32 bits where the
// list stands 87 temperatures above all others, and the outcome whose loss is largest would be lost. So its logarithm is at hand however little it
// is, and the others' gradients, shares of what is pulled outside the list, are taken against that reference as well. "Another token" is left out
// only where the student leaves it nothing at all. A row whose weight is 0 is not read: its loss and gradient are 0 whatever stands there.
//
// A row is read once and its gradient written once. The CTAs of a cluster hold a row's 16-byte pieces in shared memory between the two; a
// thread sums exponentials against its own maxima, and every warp sends what it has to all CTAs of the cluster, whose barriers count the
// bytes. Clusters walk over the rows: while one is worked on, the next one's pieces are on their way. The listed tokens are taken out of a
// row (their places become -inf) before it is summed, so that what is left is summed without looking at the list. Losses alone, and rows that
// no cluster holds, take a second kernel that streams.
//
// What bounds it. 1,024 float32 rows of 50,257 (64 listed): 75.7 us for 399 MB, 5.3 TB/s, 0.81 of a copy (with the list alone as outcomes the
// same); nothing runs beside the first share's arrival and the last one's gradient, 8 us. 4,096 bfloat16 rows (32 listed): 155 us, 5.0 TB/s (165 with
// "another token"): the special-function units are busy 57 % of the time, with two exponentials a number. Losses of 2,047 float32 rows of
// 128,001: 155 us, 6.3 TB/s, 0.97 of a copy; of bfloat16 rows 98 us, 5.4 TB/s. 16 rows of 1,031: 5.0 us, a row's chain.
#include "logit_rows.cuh"
#include "sm100_ptx.cuh"

namespace {

constexpr int MOST_K = 256;
constexpr int MOST_RANKS = 8;
constexpr int MOST_WARPS = 12;     // of a block, that work on pieces
constexpr uint32_t LANDING = 4096; // polls, some 16 ms, for 16 bytes that another CTA has sent already
#define R2_ERR_TIMEOUT_SHARES 8
#ifndef R2_SHARE_POLLS
#define R2_SHARE_POLLS r2ptx::SPIN_LIMIT   // of a wait for a row's share or for the cluster's sums (a test lets them run out)
#endif

struct DistillArgs {
  const void* logits; long long ld;
  int rows, vocab, k, ranks, per;   // per: pieces of a row that a CTA has, whatever the row's alignment (the last one has what is left)
  const int32_t* ids; const float* teacher; const float* log_sum; const float* weight;
  float tau;
  float* loss;
  void* grad; long long grad_ld;
  int* error;
};

// (reference, sum) over the listed tokens and over the others: one of every lane into one of the warp.
__device__ __forceinline__ float4 warp_join(float4 v) {
  const float listed = warp_max(v.x), others = warp_max(v.z);
  return make_float4(listed, warp_sum(v.y * rebase(v.x, listed)), others, warp_sum(v.w * rebase(v.z, others)));
}

// What a row's list says, from shared memory, by every warp for itself: the logarithm that the teacher's exponentials are taken against, and
// their sum's mass.
__device__ __forceinline__ float2 teacher_mass(const float* teacher, int k, int lane, bool tail, float log_sum) {
  float against = log_sum, mass = 0.f;
  if (!tail) {
    float most = -INFINITY, sum = 0.f;
    for (int j = lane; j < k; j += 32) most = fmaxf(most, teacher[j]);
    most = no_less(warp_max(most));
    for (int j = lane; j < k; j += 32) sum += expf(teacher[j] - most);
    against = most + logf(warp_sum(sum));
    if (against == -INFINITY) against = 0.f;   // no entries
  }
  for (int j = lane; j < k; j += 32) mass += expf(teacher[j] - against);
  return make_float2(against, warp_sum(mass));
}

// p log(p / q) - p + q of one outcome. Where q is larger by far, e^(log q - log p) is beyond 32 bits before p times it is, and nothing cancels.
__device__ __forceinline__ float outcome(float p, float log_p, float log_q) {
  const float d = log_p - log_q;
  if (!(p > 0.f)) return expf(log_q);
  return d < -1.f ? p * d + (expf(log_q) - p) : p * (d + expm1f(-d));
}

// The student's side of a row, joined over its warps.
struct Student {
  float common, total, inv_total, whole;   // whole: the mass that its tokens' gradients share
  float rest, log_rest, rest_p;            // the mass outside the list, its logarithm (-inf: none at all), the teacher's where the student has some
  float from, by;                          // an unlisted token's gradient: by 2^(x c - from)

  Student() = default;
  // From (reference, sum) over the listed and over the others of every warp, by any warp for itself.
  __device__ __forceinline__ Student(const float4* shares, int n, int lane, bool tail, float mass) {
    float4 v = make_float4(-INFINITY, 0.f, -INFINITY, 0.f);
    for (int i = lane; i < n; i += 32) {
      const float4 s = shares[i];
      const float listed = fmaxf(v.x, s.x), others = fmaxf(v.z, s.z);
      v = make_float4(listed, v.y * rebase(v.x, listed) + s.y * rebase(s.x, listed), others, v.w * rebase(v.z, others) + s.w * rebase(s.z, others));
    }
    v = warp_join(v);
    common = fmaxf(v.x, v.z);
    const float listed = v.y * rebase(v.x, common), others = v.w * rebase(v.z, common);   // (may be nothing in 32 bits)
    total = listed + others;
    inv_total = __frcp_rn(total);
    rest = others * inv_total;
    log_rest = -INFINITY;
    rest_p = 0.f;
    whole = mass;
    from = common;
    by = mass * inv_total;
    if (tail && v.w != 0.f) {
      log_rest = rest > 1e-30f ? logf(rest) : (v.z - common + (log2f(v.w) - log2f(total))) * 0.693147181f;
      rest_p = fmaxf(1.f - mass, 0.f);
      if (rest_p > 0.f) {
        whole = 1.f;
        from = v.z;
        by = __fdividef(mass - listed * inv_total, v.w);
      }
    }
  }

  // The row's divergence, by one warp.
  __device__ __forceinline__ float divergence(const int32_t* ids, const float* teacher, const float* xk, int k, int lane, bool tail, float c,
                                              float against, float mass) const {
    const float log2_total = log2f(total);
    float kl = 0.f;
    for (int j = lane; j < k; j += 32) {
      if (ids[j] < 0) continue;
      const float lq = (fmaf(xk[j], c, -common) - log2_total) * 0.693147181f, lp = teacher[j] - against, p = expf(lp);
      if (tail) kl += outcome(p, lp, lq);
      else if (p > 0.f) kl += p * (lp - lq);
    }
    kl = warp_sum(kl);
    if (!(total > 0.f) && (tail || mass > 0.f)) return NAN;   // a row of nothing (without outcomes there is nothing to compare)
    if (tail) kl += rest_p > 0.f ? outcome(rest_p, logf(rest_p), log_rest) : (log_rest > -INFINITY ? rest : 0.f) + (mass - 1.f);
    return kl;
  }
};

// Entry j's gradient, over what stands there. A list that names a token more than once (`twice`): its first entry writes for all.
template <typename T>
__device__ __forceinline__ void write_listed(T* grad, const int32_t* ids, const float* teacher, const float* logits, int k, int j, bool twice,
                                             float c, float against, float scale, const Student& q) {
  float p = expf(teacher[j] - against), x = logits[j];
  if (twice) {
    p = 0.f;
    for (int o = 0; o < k; ++o) {
      if (ids[o] != ids[j]) continue;
      if (o < j) return;
      p += expf(teacher[o] - against);
      x = fmaxf(x, logits[o]);   // (one entry took the logit out of the row, the others found -inf)
    }
  }
  grad[ids[j]] = from_float<T>(scale * (exp2_approx(fmaf(x, c, -q.common)) * q.inv_total * q.whole - p));
}

// Sets the bits of the listed tokens among `bits` tokens from `zero` on; whether one was set already.
__device__ __forceinline__ bool mark_listed(uint32_t* listed, const int32_t* ids, int k, int zero, int bits, int tid, int threads) {
  bool again = false;
  for (int j = tid; j < k; j += threads) {
    const int at = ids[j] - zero;
    if (ids[j] < 0 || at < 0 || at >= bits) continue;
    const uint32_t bit = 1u << (at & 31);
    again |= (atomicOr(&listed[at >> 5], bit) & bit) != 0u;
  }
  return again;
}

// Takes an element of the staged row out of it: what stood there; -inf stays.
__device__ __forceinline__ float take_out(float* at) { return __uint_as_float(atomicExch(reinterpret_cast<unsigned int*>(at), 0xff800000u)); }
__device__ __forceinline__ float take_out(bf16* at) {
  unsigned short* bits = reinterpret_cast<unsigned short*>(at);
  unsigned short old = *bits, seen;
  while ((seen = atomicCAS(bits, old, static_cast<unsigned short>(0xff80))) != old) old = seen;
  return __uint_as_float(static_cast<uint32_t>(old) << 16);
}

// 16 bytes into another CTA's shared memory, counted by that CTA's barrier; both places by their address there.
__device__ __forceinline__ void send(uint32_t to, uint32_t barrier, float4 v) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(to), "f"(v.x), "f"(v.y),
               "f"(v.z), "f"(v.w), "r"(barrier)
               : "memory");
}
__device__ __forceinline__ bool arrived(uint32_t barrier, uint32_t parity, uint32_t polls = R2_SHARE_POLLS) {   // false: gave up
  for (uint32_t spin = 0; spin < polls; ++spin) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(barrier), "r"(parity)
        : "memory");
    if (done) return true;
    if (spin > 1024) __nanosleep(64);
  }
  return false;
}

// Sums of exponentials against a reference that the thread chooses as it goes.
template <typename T>
struct Sums {
  float reference = -INFINITY, sum = 0.f;   // an exponent of two; what is summed is 2^(x c - reference)

  __device__ __forceinline__ void raise(float to) {
    if (!(to > reference && to > -FAR_REFERENCE)) return;   // (what is lower leaves it as it is: nothing summed)
    sum *= rebase(reference, to);
    reference = to;
  }
  __device__ __forceinline__ void add(float x, float c) {
    raise(x * c);
    sum += exp2_approx(fmaf(x, c, shift_to(reference)));
  }
  // N pieces. The reference is raised where a sum leaves the middle of the range; a maximum of every piece is not looked for.
  template <int N>
  __device__ __forceinline__ void add(const uint4 (&raw)[N], float c) {
    constexpr int PAIRS = RowPieces<T>::PER / 2;
    const uint64_t cc = two_of(c, c);
    float more;
    auto exponentials = [&]() {
      const float shift = shift_to(reference);
      const uint64_t ss = two_of(shift, shift);
      uint64_t acc[N];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        uint64_t p[PAIRS];
        unpack_pairs(raw[i], p, static_cast<const T*>(nullptr));
        acc[i] = exp2_two(fma_two(p[0], cc, ss));
#pragma unroll
        for (int j = 1; j < PAIRS; ++j) acc[i] = add_two(acc[i], exp2_two(fma_two(p[j], cc, ss)));
      }
#pragma unroll
      for (int i = 1; i < N; ++i) acc[0] = add_two(acc[0], acc[i]);
      const float2 v = halves(acc[0]);
      more = v.x + v.y;
    };
    exponentials();
    if (reference == -INFINITY || !(more > 1e-18f && more < 1e18f)) {
      const float before = reference;
      raise(most(raw) * c);
      if (reference != before) exponentials();
    }
    sum += more;
  }
  template <int N>
  static __device__ __forceinline__ float most(const uint4 (&raw)[N]) {
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float v[RowPieces<T>::PER];
      unpack(raw[i], v, static_cast<const T*>(nullptr));
#pragma unroll
      for (int e = 0; e < RowPieces<T>::PER; ++e) m = fmaxf(m, v[e]);
    }
    return m;
  }
};

// What a CTA has in shared memory beside its pieces and the sums.
struct __align__(16) HeldShared {
  uint64_t landed, shared_in[2];     // barriers: a row's share is there; every warp of the cluster has sent its sums
  int32_t ids[2][MOST_K];
  float teacher[2][MOST_K], xk[2][MOST_K], taken[MOST_K];
  float2 of_teacher[2];              // what the teacher's exponentials are taken against, and their sum
  Student students[2];
  int twice[2];
};
constexpr int sums_bytes(int ranks, int warps) { return 2 * ranks * warps * int(sizeof(float4)); }   // (reference, sum) twice of every warp

// A block is twelve warps (fewer for short rows) that work on pieces and one more that brings: it has the next row's share copied, brings
// its list and takes its mass, and finishes the loss of the row before, all beside the others, which meet it once a row. Rows that weigh
// nothing are not brought; `slot` counts the others, two at a time.
//
// A wait that ran out ends the CTA's walk: at the row's next barrier its threads learn of it, the rows from that one on become NaN (the loss in
// the first CTA, each CTA's share of the gradient), and nothing more is copied or sent. The cluster's other CTAs then miss its sums and end
// likewise. A CTA that gave up stays until the others have sent what they send, what they sent has had its time (LANDING), and its own copy has landed
// or had as long again as a wait takes.
template <typename T>
__global__ void __launch_bounds__(32 * (MOST_WARPS + 1), 2)
distill_held_kernel(const DistillArgs a) {
  constexpr int PER = RowPieces<T>::PER, AHEAD = 16 / PER;   // pieces that a thread takes at a time
  extern __shared__ __align__(16) uint4 pieces[];            // of this CTA's share; behind them the sums of two rows
  __shared__ HeldShared shared;
  uint64_t &landed = shared.landed, (&shared_in)[2] = shared.shared_in;
  int32_t (&ids)[2][MOST_K] = shared.ids;
  float (&teacher)[2][MOST_K] = shared.teacher, (&xk)[2][MOST_K] = shared.xk, (&taken)[MOST_K] = shared.taken;
  float2 (&of_teacher)[2] = shared.of_teacher;
  Student (&students)[2] = shared.students;
  int (&twice)[2] = shared.twice;
  pdl_launch_dependents();
  const int threads = int(blockDim.x) - 32, warps = threads >> 5;   // that work on pieces
  const int ranks = a.ranks, step = int(gridDim.x) / ranks, rank = int(blockIdx.x) % ranks, tid = int(threadIdx.x), lane = tid & 31, warp = tid >> 5;
  const int g0 = rank * a.per, k = a.k;
  const bool tail = a.log_sum != nullptr;
  const float c = 1.44269504f / a.tau;
  int row = int(blockIdx.x) / ranks;
  uint32_t slot = 0;   // rows brought so far, less this one: its places are slot % 2, its barriers' phase slot / 2
  auto weight = [&](int r) { return r >= a.rows ? 0.f : a.weight != nullptr ? a.weight[r] : 1.f; };
  uint32_t copies = 0;   // of one thread, begun
  // The end of a CTA that gave up (all of its threads). The cluster's barrier counts CTAs that have ended as arrived. Which sums still come is not
  // known: both phases of both barriers are waited for, one of which is over.
  auto settle = [&]() {
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    if (tid != 0) return;
    if (copies > 0) arrived(r2ptx::smem_u32(&landed), (copies - 1) & 1, r2ptx::SPIN_LIMIT);
    for (uint32_t of = 0u; of < 4u; ++of) arrived(r2ptx::smem_u32(&shared_in[of >> 1]), of & 1, LANDING);
  };

  if (warp == warps) {
    if (lane == 0) {
      r2ptx::mbar_init(r2ptx::smem_u32(&landed), 1u);
      for (int i = 0; i < 2; ++i) r2ptx::mbar_init(r2ptx::smem_u32(&shared_in[i]), 1u);
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    cluster_arrive();
    pdl_wait();
    const float inv = 1.f / a.tau;
    auto bring = [&](int r, int b) {
      const float log_sum = tail ? a.log_sum[r] : 0.f;
#pragma unroll 4
      for (int j = lane; j < k; j += 32) {
        const int id = a.ids[(long long)r * k + j];
        const float t = a.teacher[(long long)r * k + j];
        const bool held = id >= 0 && id < a.vocab;
        ids[b][j] = held ? id : -1;
        teacher[b][j] = held ? t * inv : -INFINITY;
      }
      __syncwarp();
      if (rank == 0) {
#pragma unroll 4
        for (int j = lane; j < k; j += 32) xk[b][j] = ids[b][j] >= 0 ? to_float(static_cast<const T*>(a.logits)[(long long)r * a.ld + ids[b][j]]) : 0.f;
      }
      const float2 m = teacher_mass(teacher[b], k, lane, tail, log_sum);
      if (lane == 0) {
        of_teacher[b] = m;
        twice[b] = 0;
      }
      __syncwarp();
    };
    float w = weight(row), w_next = weight(row + step), w_before = 0.f;
    if (w != 0.f) bring(row, 0);
    cluster_wait();
    for (int before = -1;; row += step) {
      const bool gave_up = __syncthreads_or(0) != 0;
      if (before >= 0 && rank == 0) {   // the loss of the row before
        float loss = w_before != 0.f ? NAN : 0.f;
        if (w_before != 0.f && !gave_up) {
          const int b = (slot - 1) & 1;
          const float2 t = of_teacher[b];
          loss = w_before * a.tau * a.tau * students[b].divergence(ids[b], teacher[b], xk[b], k, lane, tail, c, t.x, t.y);
        }
        if (lane == 0) a.loss[before] = loss;
      }
      if (gave_up) {
        if (rank == 0 && lane == 0)
          for (; row < a.rows; row += step) a.loss[row] = weight(row) != 0.f ? NAN : 0.f;
        settle();
        return;
      }
      if (row >= a.rows) return;
      const float w_after = weight(row + 2 * step);
      if (w != 0.f) ++slot;
      if (w_next != 0.f) bring(row + step, slot & 1);
      before = row;
      w_before = w;
      w = w_next;
      w_next = w_after;
    }
  }

  cluster_arrive();
  pdl_wait();
  auto meet = [&]() { asm volatile("bar.sync 1, %0;" ::"r"(threads) : "memory"); };
  auto copy = [&](int r) {   // one thread's: a row's share into its place
    const RowPieces<T> x(static_cast<const T*>(a.logits) + (long long)r * a.ld, a.vocab);
    const uint32_t bytes = uint32_t(min(a.per, x.count - g0)) * 16u, barrier = r2ptx::smem_u32(&landed);
    ++copies;
    r2ptx::mbar_expect_tx(barrier, bytes);
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(r2ptx::smem_u32(pieces)),
                 "l"(reinterpret_cast<const uint4*>(x.base) + g0), "r"(bytes), "r"(barrier)
                 : "memory");
  };
  float w = weight(row), w_next = weight(row + step);
  cluster_wait();
  if (tid == 0 && w != 0.f) copy(row);
  bool lost = false, gave_up = false;   // a wait of this thread ran out; of any of the CTA's
  for (; row < a.rows; row += step) {
    const RowPieces<T> x(static_cast<const T*>(a.logits) + (long long)row * a.ld, a.vocab);
    const int n = max(0, min(a.per, x.count - g0)), last = x.count - 1 - g0, zero = x.first(g0);
    T* grad = static_cast<T*>(a.grad) + (long long)row * a.grad_ld;
    uint4* out = reinterpret_cast<uint4*>(grad - x.phase) + g0;
    const bool vectors = (reinterpret_cast<uintptr_t>(out) & 15) == 0;   // the gradient's row starts at the logits' alignment
    const float w_after = weight(row + 2 * step);
    // pieces from `low` up to `high` lie in the row as a whole; the ends of the row may not
    const int low = g0 == 0 && x.phase > 0 ? 1 : 0, high = last >= 0 && last < n && !x.whole(g0 + last) ? min(n, last) : n;
    const int b = slot & 1;
    T* tokens = reinterpret_cast<T*>(pieces);
    gave_up = __syncthreads_or(lost) != 0;   // the row's list is there; the row before has done with its own
    if (gave_up) break;
    // this lane's token at the row's ends (the first warp's: in a first piece, in a last piece)
    int end = -1;
    if (warp == 0 && lane < 2 * PER) {
      const int at = lane < PER ? lane : last * PER + lane - PER;
      if (lane < PER ? low == 1 && (last > 0 || high == n) : high < n) end = at;
    }
    if (w == 0.f) {
      const float zeros[PER] = {};
      if (tid == 0 && w_next != 0.f) copy(row + step);
#pragma unroll 1
      for (int at = low + tid; at < high; at += threads) store_piece<T, PER>(grad, x.first(g0 + at), a.vocab, zeros, vectors);
      if (end >= 0 && zero + end >= 0 && zero + end < a.vocab) grad[zero + end] = from_float<T>(0.f);
    } else {
      const uint32_t barrier = r2ptx::smem_u32(&shared_in[b]), phase = (slot >> 1) & 1;
      ++slot;
      lost = !arrived(r2ptx::smem_u32(&landed), (slot - 1) & 1);
      if (end >= 0 && (zero + end < 0 || zero + end >= a.vocab)) {
        tokens[end] = from_float<T>(-INFINITY);
        end = -1;
      }
      if (tid == 0) r2ptx::mbar_expect_tx(barrier, uint32_t(ranks * warps) * 16u);
      Sums<T> listed, sums;
#pragma unroll 1
      for (int j = tid; j < k; j += threads) {
        const int at = ids[b][j] - zero;
        if (ids[b][j] < 0 || at < 0 || at >= n * PER) continue;
        const float v = take_out(tokens + at);
        if (v == -INFINITY) twice[b] = 1;
        taken[j] = v;   // (read again behind a barrier)
        listed.add(v, c);
      }
      meet();
      int at = tid;
      if (at < n) {
        const uint4 first[1] = {pieces[at]};
        sums.raise(Sums<T>::most(first) * c);
      }
#pragma unroll 1
      for (; at + (AHEAD - 1) * threads < n; at += AHEAD * threads) {
        uint4 raw[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) raw[i] = pieces[at + i * threads];
        sums.add(raw, c);
      }
#pragma unroll 1
      for (; at < n; at += threads) {
        const uint4 raw[1] = {pieces[at]};
        sums.add(raw, c);
      }
      if (lost) sums.sum = NAN;   // (no sums of a share that is not there)
      float4* of_warps = reinterpret_cast<float4*>(pieces + a.per) + b * ranks * warps;
      const float4 joined = warp_join(make_float4(listed.reference, listed.sum, sums.reference, sums.sum));
      if (lane < ranks)
        send(cluster_address(of_warps + rank * warps + warp, lane), cluster_address(&shared_in[b], lane), joined);
      lost |= !arrived(barrier, phase);
      const float2 t = of_teacher[b];
      const Student q(of_warps, ranks * warps, lane, tail, t.y);
      if (tid == 0) students[b] = q;
      const float scale = w * a.tau, by = scale * q.by;
      if (vectors) {
        const uint64_t cc = two_of(c, c), ss = two_of(-q.from, -q.from), bb = two_of(by, by);
        auto gradient = [&](const uint4& raw) {
          uint64_t p[PER / 2];
          unpack_pairs(raw, p, static_cast<const T*>(nullptr));
#pragma unroll
          for (int i = 0; i < PER / 2; ++i) p[i] = mul_two(exp2_two(fma_two(p[i], cc, ss)), bb);
          return pack_pairs(p, static_cast<const T*>(nullptr));
        };
        at = low + tid;
#pragma unroll 1
        for (; at + (AHEAD - 1) * threads < high; at += AHEAD * threads) {
          uint4 raw[AHEAD];
#pragma unroll
          for (int i = 0; i < AHEAD; ++i) raw[i] = pieces[at + i * threads];
#pragma unroll
          for (int i = 0; i < AHEAD; ++i) out[at + i * threads] = gradient(raw[i]);
        }
#pragma unroll 1
        for (; at < high; at += threads) out[at] = gradient(pieces[at]);
      } else {
#pragma unroll 1
        for (at = low * PER + tid; at < high * PER; at += threads) grad[zero + at] = from_float<T>(exp2_approx(fmaf(to_float(tokens[at]), c, -q.from)) * by);
      }
      if (end >= 0) grad[zero + end] = from_float<T>(exp2_approx(fmaf(to_float(tokens[end]), c, -q.from)) * by);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // (the next copy comes by another path than what was written here)
      meet();   // the listed tokens' gradients lie over what stands there
      if (tid == 0 && w_next != 0.f && !lost) copy(row + step);
#pragma unroll 1
      for (int j = tid; j < k; j += threads) {
        const int at = ids[b][j] - zero;
        if (ids[b][j] >= 0 && at >= 0 && at < n * PER) write_listed(grad, ids[b], teacher[b], taken, k, j, twice[b] != 0, c, t.x, scale, q);
      }
    }
    w = w_next;
    w_next = w_after;
  }
  if (!gave_up) gave_up = __syncthreads_or(lost) != 0;
  if (!gave_up) return;
  if (tid == 0) atomicMax(a.error, R2_ERR_TIMEOUT_SHARES);
  for (int r = row - step; r < a.rows; r += step) {
    const RowPieces<T> x(static_cast<const T*>(a.logits) + (long long)r * a.ld, a.vocab);
    T* grad = static_cast<T*>(a.grad) + (long long)r * a.grad_ld;
    const int end = min(a.vocab, x.first(g0 + a.per));
    const T value = from_float<T>(weight(r) != 0.f ? NAN : 0.f);
    for (int token = max(0, x.first(g0)) + tid; token < end; token += threads) grad[token] = value;
  }
  settle();
}

// Losses alone (one pass over the row), and gradients of rows that no cluster holds (two).
template <typename T, bool TAIL, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS)
distill_streamed_kernel(const DistillArgs a) {
  constexpr int PER = RowPieces<T>::PER, DEPTH = 4;
  extern __shared__ __align__(16) uint32_t bits_s[];   // a bit for each token of this CTA's share
  __shared__ __align__(16) float4 shares[MOST_RANKS * (THREADS / 32)];
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
  const int g0 = rank * a.per, n = max(0, min(a.per, x.count - g0));
  const float w = a.weight != nullptr ? a.weight[row] : 1.f;
  if (w == 0.f) {  // (every CTA of the cluster)
    if (grad != nullptr) {
      const float zeros[PER] = {};
      for (int i = tid; i < n; i += THREADS) store_piece<T, PER>(grad, x.first(g0 + i), a.vocab, zeros, vectors);
    }
    if (rank == 0 && tid == 0) a.loss[row] = 0.f;
    return;
  }
  if (ranks > 1) cluster_arrive();
  const float inv = 1.f / a.tau, c = 1.44269504f / a.tau;
  for (int j = tid; j < k; j += THREADS) {
    const int id = a.ids[(long long)row * k + j];
    const bool held = id >= 0 && id < a.vocab;
    ids[j] = held ? id : -1;
    teacher[j] = held ? a.teacher[(long long)row * k + j] * inv : -INFINITY;
    xk[j] = held ? to_float(x.base[x.phase + id]) : 0.f;
  }
  if (TAIL || grad != nullptr)
    for (int i = tid; i < (n * PER + 31) / 32; i += THREADS) bits_s[i] = 0u;
  __syncthreads();
  if (TAIL || grad != nullptr)
    if (mark_listed(bits_s, ids, k, x.first(g0), n * PER, tid, THREADS)) twice = 1;
  __syncthreads();
  Sums<T> own;
  // listed tokens and places that are not the row's are -inf in what is summed
  auto clear = [&](uint4& raw, int at) {
    if (TAIL) {
      const uint32_t bits = (bits_s[at * PER / 32] >> (at * PER % 32)) & ((1u << PER) - 1u);
      if (bits != 0u) keep_bits<T>(raw, ~bits);
    }
    if (g0 + at == 0 || g0 + at == x.count - 1) blank_outside(raw, x, g0 + at);
  };
  uint4 raw[DEPTH];
  auto load = [&](int at) {
#pragma unroll
    for (int i = 0; i < DEPTH; ++i) raw[i] = load_once(x, g0 + at + i * THREADS);
  };
  int at = tid;
  if (at + (DEPTH - 1) * THREADS < n) {
    load(at);
    uint4 first[DEPTH];
#pragma unroll
    for (int i = 0; i < DEPTH; ++i) {
      first[i] = raw[i];
      clear(first[i], at + i * THREADS);
    }
    own.raise(Sums<T>::most(first) * c);
  }
#pragma unroll 1
  for (; at + (DEPTH - 1) * THREADS < n; at += DEPTH * THREADS) {
    uint4 now[DEPTH];
#pragma unroll
    for (int i = 0; i < DEPTH; ++i) now[i] = raw[i];
    if (at + (2 * DEPTH - 1) * THREADS < n) load(at + DEPTH * THREADS);
#pragma unroll
    for (int i = 0; i < DEPTH; ++i) clear(now[i], at + i * THREADS);
    own.add(now, c);
  }
#pragma unroll 1
  for (; at < n; at += THREADS) {
    uint4 one[1] = {load_once(x, g0 + at)};
    clear(one[0], at);
    own.add(one, c);
  }
  Sums<T> listed;   // (here, not before the row: its registers are the row's)
  if (TAIL) {
    for (int j = tid; j < k; j += THREADS) {
      const int at = ids[j] - x.first(g0);
      if (ids[j] < 0 || at < 0 || at >= n * PER) continue;
      // (of a token that the list names more than once, one entry counts)
      bool first = true;
      if (twice)
        for (int o = 0; o < j; ++o) first &= ids[o] != ids[j];
      if (!first) continue;
      listed.add(xk[j], c);
    }
  }
  const float4 sums = warp_join(make_float4(listed.reference, listed.sum, own.reference, own.sum));
  if (ranks > 1) {
    cluster_wait();
    if (lane < ranks) cluster_store(cluster_address(&shares[rank * (THREADS / 32) + (tid >> 5)], lane), sums);
    cluster_arrive();
    cluster_wait();
  } else {
    if (lane == 0) shares[tid >> 5] = sums;
    __syncthreads();
  }
  if (grad == nullptr && (rank > 0 || tid >= 32)) return;
  const float2 t = teacher_mass(teacher, k, lane, TAIL, TAIL ? a.log_sum[row] : 0.f);
  const Student q(shares, ranks * (THREADS / 32), lane, TAIL, t.y);
  if (rank == 0 && tid < 32) {
    const float kl = q.divergence(ids, teacher, xk, k, lane, TAIL, c, t.x, t.y);
    if (lane == 0) a.loss[row] = w * a.tau * a.tau * kl;
  }
  if (grad == nullptr) return;
  const float scale = w * a.tau, by = scale * q.by;
  for (int c0 = tid; c0 < n; c0 += DEPTH * THREADS) {
    uint4 raw[DEPTH];
#pragma unroll
    for (int i = 0; i < DEPTH; ++i)
      if (c0 + i * THREADS < n) raw[i] = load_once(x, g0 + c0 + i * THREADS);
#pragma unroll
    for (int i = 0; i < DEPTH; ++i) {
      if (c0 + i * THREADS >= n) continue;
      float v[PER];
      unpack(raw[i], v, static_cast<const T*>(nullptr));
#pragma unroll
      for (int e = 0; e < PER; ++e) v[e] = exp2_approx(fmaf(v[e], c, -q.from)) * by;
      store_piece<T, PER>(grad, x.first(g0 + c0 + i * THREADS), a.vocab, v, vectors);
    }
  }
  __syncthreads();
  for (int j = tid; j < k; j += THREADS) {
    const int at = ids[j] - x.first(g0);
    if (ids[j] >= 0 && at >= 0 && at < n * PER) write_listed(grad, ids, teacher, xk, k, j, twice != 0, c, t.x, scale, q);
  }
}

constexpr int MOST_STREAMED_BITS = 1 << 20;   // tokens of a CTA's share (128 KB of bits)

// Pieces of a CTA's share where two CTAs, or one, fit an SM. A row takes as few CTAs as hold it with two to an SM, so that one's sum runs beside
// the other's copies (1,024 rows of 50,257: two CTAs of 100 KB a row 75 us, one of 200 KB with an SM to itself 77, shares for three or
// four CTAs an SM 100 to 117); eight CTAs of a whole SM each hold the longest rows.
constexpr int HELD_TWO = 6600, HELD_ONE = 13600;
constexpr int SM_BYTES = 228 * 1024, CTA_BYTES = 227 * 1024, RESERVED = 1024;   // shared memory; RESERVED: the system's of every CTA's
// (eight CTAs' sums are 0.3 KB too many: rows of eight shares of more than 6,584 pieces have the SMs to themselves)
static_assert(2 * (HELD_TWO * 16 + sums_bytes(MOST_RANKS - 1, MOST_WARPS) + int(sizeof(HeldShared)) + RESERVED) <= SM_BYTES, "two CTAs an SM");
static_assert(HELD_ONE * 16 + sums_bytes(MOST_RANKS, MOST_WARPS) + int(sizeof(HeldShared)) <= CTA_BYTES, "one CTA an SM");

template <typename T>
int launch_held(const DistillArgs& a, cudaStream_t stream) {
  // Short rows get few warps, so that more of them are in hand: two pieces a thread at least, and beyond three warps sixteen (4,096 rows of 4,000
  // float32 numbers: twelve warps 62.6 us, three 30.0, one 38.5; 2,000 of 12,000: twelve 47.3, five 42.0, one 56.5; 100 of 4,000: twelve 6.0, three 6.3,
  // one 8.1). By the row alone: its sums are then added in the same order in every call.
  const int warps = max(1, min(min(MOST_WARPS, a.per / 64), max(3, a.per / 512)));
  const size_t smem = size_t(a.per) * 16 + size_t(sums_bytes(a.ranks, warps));
  static std::atomic<bool> allowed[64];
  const int status = allow_smem(distill_held_kernel<T>, size_t(HELD_ONE) * 16 + sums_bytes(MOST_RANKS, MOST_WARPS), allowed);
  if (status != R2_OK) return status;
  // how many clusters run at a time, asked once for each device and shape (a table that forgets)
  struct Resident {
    std::atomic<unsigned long long> shape_and_clusters;
  };
  static Resident resident[64];
  int device = 0, clusters = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return int(e);
  const unsigned long long shape = (static_cast<unsigned long long>(device) << 56) | (static_cast<unsigned long long>(a.ranks) << 48) |
                                   (static_cast<unsigned long long>(a.per * 16 + warps) << 24);
  Resident& place = resident[(a.per * 8 + a.ranks + device) % 64];
  const unsigned long long known = place.shape_and_clusters.load(std::memory_order_relaxed);
  if ((known >> 24) == (shape >> 24) && known != 0) {
    clusters = int(known & 0xffffff);
  } else {
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(unsigned(a.ranks) * 4096u);
    config.blockDim = dim3(unsigned(32 * (warps + 1)));
    config.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = unsigned(a.ranks);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    config.attrs = attr;
    config.numAttrs = 1;
    e = cudaOccupancyMaxActiveClusters(&clusters, distill_held_kernel<T>, &config);
    if (e != cudaSuccess) return int(e);
    if (clusters < 1) return R2_UNSUPPORTED;
    place.shape_and_clusters.store(shape | static_cast<unsigned long long>(clusters), std::memory_order_relaxed);
  }
  r2_launch_clusters(distill_held_kernel<T>, a.ranks, dim3(unsigned(min(a.rows, clusters) * a.ranks)), dim3(unsigned(32 * (warps + 1))), smem, stream, a);
  return launch_status();
}

template <typename T, bool TAIL, int THREADS>
int launch_streamed(const DistillArgs& a, cudaStream_t stream) {
  static std::atomic<bool> allowed[64];
  const int status = allow_smem(distill_streamed_kernel<T, TAIL, THREADS>, MOST_STREAMED_BITS / 8, allowed);
  if (status != R2_OK) return status;
  r2_launch_clusters(distill_streamed_kernel<T, TAIL, THREADS>, a.ranks, dim3(unsigned(a.rows) * unsigned(a.ranks)), dim3(THREADS),
                     size_t(a.per * RowPieces<T>::PER + 31) / 32 * 4, stream, a);
  return launch_status();
}
template <typename T, bool TAIL>
int launch_streamed(DistillArgs a, int pieces, cudaStream_t stream) {
  // a row to a CTA where there are CTAs enough for the SMs, else cut over several
  a.ranks = 1;
  while (a.ranks < MOST_RANKS && ((long long)a.rows * a.ranks < 592 || (pieces / a.ranks + 1) * RowPieces<T>::PER > MOST_STREAMED_BITS)
         && pieces / a.ranks > 1024) a.ranks *= 2;
  a.per = (pieces + a.ranks - 1) / a.ranks;
  if (a.per * RowPieces<T>::PER > MOST_STREAMED_BITS) return R2_UNSUPPORTED;
  if ((long long)a.rows * a.ranks > 0x7fffffffLL) return R2_BAD_SHAPE;
  // Half the threads where the rows are more than four CTAs an SM (2,047 rows of 128,001, 100 listed: 163 us with 256 threads, 155 with 128;
  // 4,096 of 4,000, 64 listed: 54.1, 33.4; but 592 of 50,257: 21.8, 26.1).
  if ((long long)a.rows * a.ranks > 592) return launch_streamed<T, TAIL, 128>(a, stream);
  return launch_streamed<T, TAIL, 256>(a, stream);
}

template <typename T, bool TAIL>
int launch(DistillArgs a, cudaStream_t stream) {
  const int pieces = (a.vocab + 2 * RowPieces<T>::PER - 2) / RowPieces<T>::PER;   // of a row at any alignment, at most
  if (a.grad == nullptr || pieces > MOST_RANKS * HELD_ONE) return launch_streamed<T, TAIL>(a, pieces, stream);
  a.ranks = min(MOST_RANKS, (pieces + HELD_TWO - 1) / HELD_TWO);
  a.per = (pieces + a.ranks - 1) / a.ranks;
  return launch_held<T>(a, stream);
}

// Rows times a factor each. In place a row whose factor is 1 is not touched.
// A CTA has 2,048 pieces, eight a thread, one under way each. 1,024 float32 rows of 50,257: 70 us into new rows (floor 63), 84 in place, 8 where
// all factors are 1; bfloat16 38, 44 and 5.
template <typename T>
__global__ void __launch_bounds__(256)
scale_rows_kernel(const T* x, long long ld, T* out, long long out_ld, int vocab, int slices, const float* factors, int factor_step) {
  pdl_launch_dependents();
  pdl_wait();
  const int row = int(blockIdx.x) / slices, slice = int(blockIdx.x) % slices;
  const float f = factors[(long long)row * factor_step];
  const T* at = x + (long long)row * ld;
  T* to = out + (long long)row * out_ld;
  if (f == 1.f && at == to) return;
  const bool vectors = ((reinterpret_cast<uintptr_t>(at) ^ reinterpret_cast<uintptr_t>(to)) & 15) == 0;
  const RowPieces<T> pieces(at, vocab);
  for (int g = slice * 2048 + int(threadIdx.x); g < min(pieces.count, (slice + 1) * 2048); g += 256) {
    float v[RowPieces<T>::PER];
    unpack(load_once(pieces, g), v, static_cast<const T*>(nullptr));
#pragma unroll
    for (int e = 0; e < RowPieces<T>::PER; ++e) v[e] *= f;
    store_piece<T, RowPieces<T>::PER>(to, pieces.first(g), vocab, v, vectors);
  }
}

}  // namespace

// x [rows, vocab] of dtype with row stride ld, times factors[row * factor_step] -> out of dtype with row stride out_ld (x itself, or apart from it).
extern "C" int r2_scale_rows(int dtype, const void* x, long long ld, void* out, long long out_ld, int rows, int vocab, const float* factors,
                             int factor_step, cudaStream_t stream) {
  if (dtype != R2_F32 && dtype != R2_BF16) return R2_BAD_DTYPE;
  if (rows < 0 || vocab < 1 || vocab > (1 << 30) || ld < vocab || out_ld < vocab || factor_step < 0 || factor_step > 1) return R2_BAD_SHAPE;
  if (rows == 0) return R2_OK;
  const int per = dtype == R2_F32 ? 4 : 8, slices = ((vocab + 2 * per - 2) / per + 2047) / 2048;
  if ((long long)rows * slices > 0x7fffffffLL) return R2_BAD_SHAPE;
  const dim3 grid(unsigned(rows) * unsigned(slices));
  if (dtype == R2_F32)
    r2_launch(scale_rows_kernel<float>, grid, dim3(256), size_t(0), stream, static_cast<const float*>(x), ld, static_cast<float*>(out), out_ld, vocab, slices, factors, factor_step);
  else
    r2_launch(scale_rows_kernel<bf16>, grid, dim3(256), size_t(0), stream, static_cast<const bf16*>(x), ld, static_cast<bf16*>(out), out_ld, vocab, slices, factors, factor_step);
  return launch_status();
}

// logits [rows, vocab] of dtype with row stride ld, ids and teacher [rows, k] (an id outside the vocabulary: no entry), log_sum and weight
// [rows] or null -> loss [rows] float; grad [rows, vocab] of dtype with row stride grad_ld, null, or the logits themselves.
extern "C" int r2_distill(int dtype, const void* logits, long long ld, int rows, int vocab, const int32_t* ids, const float* teacher, int k,
                          const float* log_sum, const float* weight, float temperature, float* loss, void* grad, long long grad_ld,
                          int* error, cudaStream_t stream) {
  if (dtype != R2_F32 && dtype != R2_BF16) return R2_BAD_DTYPE;
  if (rows < 0 || vocab < 1 || vocab > (1 << 30) || ld < vocab || (grad != nullptr && grad_ld < vocab) || k < 1) return R2_BAD_SHAPE;
  if (k > MOST_K || !(temperature > 0.f)) return R2_UNSUPPORTED;
  if (rows == 0) return R2_OK;
  const DistillArgs a = {logits, ld, rows, vocab, k, 1, 0, ids, teacher, log_sum, weight, temperature, loss, grad, grad_ld, error};
  if (log_sum != nullptr) return dtype == R2_F32 ? launch<float, true>(a, stream) : launch<bf16, true>(a, stream);
  return dtype == R2_F32 ? launch<float, false>(a, stream) : launch<bf16, false>(a, stream);
}
