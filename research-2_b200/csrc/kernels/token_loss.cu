// The loss of given tokens from hidden rows and a token table, and its gradients, without keeping logits. With hidden rows x [N, D], table
// W [V, D], tokens y [N] and weights a [N]:
//
//   u = x W^T,  z = u  or  c tanh(u / c),  s_r = log(sum_v exp z_rv),  loss_r = a_r (s_r - z_r,y)
//   dz = a_r (exp(z_rv - s_r) - [v = y_r]) (1 - (z_rv / c)^2),  dx = dz W,  dW = dz^T x
//
// All four products run on one kernel (`product_kernel`): CTA pairs (cta_group::2) with 256 x 256 tiles, operands by TMA, two accumulators in tensor memory, so
// that eight warps work on one tile's results while the next one's products run. What differs is what those warps do with a tile:
//
//   LOGSUM   a tile of z, reduced to each row's largest number and the sum of exponentials against it, by halves of a tile; `finish_kernel` joins them
//   FACTORS  a tile of z made again, turned into dz and rounded to bfloat16, a piece of the vocabulary at a time
//   ROWS     dx: dz times the piece of the table, K split over the pairs where tiles are few; shares are float and added in one order (`join_kernel`)
//   TABLE    dW: dz^T times the hidden rows, whole for each piece of the vocabulary and rounded once
//
// dz is rounded to bfloat16, the type of the gradients that it makes, so that both products run on the tensor cores at full rate. Its largest number by far is often the token's
// own, a_r (p - 1): what the rounding leaves of that one (`rest`) is kept in float and goes into dx where its shares are joined, and into dW with a tile's results. (Without it either
// gradient's error was that of two roundings, 1.44 times that of its own.)
//
// float32 operands are three bfloat16 planes each: x = x0 + x1 + x2 to the last bit (8 bits each), and a product is the six products x_i w_j
// with i + j <= 2; what is left out is below 2^-24 of it. dz is kept in three planes then, too. The tensor cores add to an accumulator without rounding to nearest: each
// addition of 16 products takes up to a unit of 2^-24 off, always towards zero (4e-6 off a sum of 768 products, when all six went into it for each k). So
// only 256 of k (or 128) are added there, the small products first, while the accumulator is small; the sums of these pieces are added in registers, rounded to nearest,
// while the next piece's products run.
//
// Rows without a token or of weight 0 have no part in the gradients: `gather_kernel` puts the others side by side, so that no product reads them
// (whatever they hold) or spends time on them; the rest of the last 256 rows is zeros.
//
// Bound by the tensor cores from some 200 rows on, by the pass over the table below. At a table of 50,257 x 768, bfloat16, 1,965 MHz: LOGSUM of 4,096 rows 189 us (1.68 PFLOP/s, tensor cores
// active 96 % of an SM's time), FACTORS of 3,840 that count 206 us (1.44; 190 without the stores of dz, which the operands' loads share the L2 with), ROWS 196 (1.51) and TABLE
// 184 to 200 (1.61; operands whose rows lie along K are read at 0.9 of the rate). Tiles of 256 x 256 on pairs read 64 KB for each 64 of k and pair where 128 x 128 read twice that for the work,
// which shared memory does not keep up with.
#include <math.h>

#include <type_traits>

#include "common.cuh"
#include "sm100_ptx.cuh"
#include "tensor_maps.cuh"

namespace {

using namespace r2ptx;

constexpr int BM = 128;          // rows of a tile in one CTA
constexpr int BN = 256;          // columns of a tile, half of their operand in each CTA
constexpr int HALF = BN / 2;
constexpr int BK = 64;           // one 128-byte swizzle span of bfloat16
constexpr int UMMA_K = 16;
constexpr int THREADS = 320;     // warp 0: TMA, warp 1: products + tensor memory, warps 2-9: results
constexpr int WARPS = 8;
constexpr int STAGES = 5;
constexpr uint32_t A_BYTES = BM * BK * 2, B_BYTES = HALF * BK * 2;
constexpr uint32_t SLAB = 32 * 128;   // 32 rows of 128 bytes on their way out; a warp has two
constexpr size_t SMEM = 1024 + STAGES * size_t(A_BYTES + B_BYTES) + 2 * WARPS * SLAB + (2 * STAGES + 4) * 8 + 16;

// Rows that go through the other kernel below, at most. At GPT-2's table with cold caches, loss and gradients of 16, 64 and 128 rows: float32 53 and 245, 57 and 249, 70 and 288 us (by the
// tiles of 256 rows 161 and 282, 153 and 284, 153 and 302), bfloat16 25 and 69, 27 and 73, 29 and 87 (106 where a tenth of the rows has one token, whose rests a lane adds; by rests_kernel 80, 84, 99 and 98).
constexpr int FEW = 128;

constexpr int WINDOW = 512;   // sorted rows whose sums by token are made together

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

constexpr int ERR_FULL = 1, ERR_EMPTY = 2, ERR_ACC = 3;   // codes of waits that ran out, as of the other products

// A wait that ran out leaves NaN: a sum that is not whole is not handed over, so that the wait for it runs out, too; warps that have given up a wait hand nothing back, which others would take for
// a word of those that still read, and make NaN of their tile and the later ones, in dz as in the results. (A test builds this file with warps that give up: of results, 1, or of products, 2.)
#ifndef R2_LOSS_GIVES_UP
#define R2_LOSS_GIVES_UP 0
#endif

enum Mode { LOGSUM, FACTORS, ROWS, TABLE, TABLE_FEW };   // (TABLE_FEW: bfloat16 rows that a tile's warps find by themselves)

constexpr bool is_table(int mode) { return mode == TABLE || mode == TABLE_FEW; }

struct Work {
  int m, n, k;               // rows and columns of the result, and what is summed over
  const int* count;          // FACTORS, ROWS: m, TABLE: k, on the device (the gathered rows)
  int splits, per_split;     // ROWS: shares of k, in steps of BK
  int add;                   // ROWS: to what earlier pieces left
  float cap, cap_out;        // c > 0: 1 / c and c log2 e, so that z log2 e = cap_out tanh(cap u); else 0
  const int32_t* targets;    // FACTORS: of the gathered rows, with their factors and sums
  const float* factor;
  const float* log_sum;
  int first;                 // FACTORS, TABLE: the piece's first token
  float* rest;               // bfloat16: what rounding left of dz at each row's token; FACTORS writes it, TABLE_FEW adds it
  const bf16* x;             // TABLE_FEW: the gathered rows
  long long ld_x;
  const int2* runs;          // bfloat16 TABLE: of each of the piece's tokens, in each segment of the sorted rows, its first row and the one behind its last
  const float* sums;         // and what rounding left at its own rows, summed by WINDOW of them (rests_kernel)
  long long ld_sums;
  int segments, run_tokens;
  float2* part;              // LOGSUM: [row][parts]: of a half tile the largest z log2 e and the sum of 2^(z log2 e - it)
  int parts;
  void* out;                 // TABLE, where tensor copies cannot write it
  long long ld;
  int* error_flag;
};

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void load_pair(uint32_t dst, const CUtensorMap* map, int x, int y, int plane, uint32_t leader_bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(dst), "l"(map), "r"(leader_bar), "r"(x), "r"(y), "r"(plane)
      : "memory");
}
__device__ __forceinline__ void umma_pair(uint32_t tmem_d, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(tmem_d), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void commit_pair(uint32_t bar) {   // arrives on both CTAs' barrier at this offset
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
               ::"r"(bar), "h"(uint16_t(3)) : "memory");
}
// Hands over tensor memory that this warp has read (ordered by tcgen05.wait::ld and the fence before it).
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// The whole warp's wait: its lanes go on together, also when it ran out (after some 17 seconds; 65 ms where a test has warps give up).
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity) {
  bool done = false;
  if constexpr (R2_LOSS_GIVES_UP == 0) done = mbar_wait(bar, parity);
  else
    for (int i = 0; i < 1 << 14 && !done; ++i) done = mbar_try_wait(bar, parity) != 0;
  return __all_sync(0xffffffffu, done);
}
// 32 rows of 128 bytes from shared memory into a box of the map (what lies outside is left out), or added to float numbers there.
__device__ __forceinline__ void store_box(const CUtensorMap* map, int x, int y, int plane, uint32_t from) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(map), "r"(from), "r"(x), "r"(y), "r"(plane) : "memory");
}
__device__ __forceinline__ void add_box(const CUtensorMap* map, int x, int y, int plane, uint32_t from) {
  asm volatile("cp.reduce.async.bulk.tensor.3d.global.shared::cta.add.bulk_group [%0, {%2, %3, %4}], [%1];"
               ::"l"(map), "r"(from), "r"(x), "r"(y), "r"(plane) : "memory");
}
__device__ __forceinline__ void st_shared16(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
// Behind a wait that ran out: the copies that this warp has asked for land (or that wait runs out, too) before its CTA ends. Stages below `stage` were filled
// in this round of the ring, the others in the one before.
__device__ __forceinline__ void settle(uint32_t full, int stages, int stage, uint32_t parity) {
  for (int s = 0; s < stages; ++s) warp_wait(full + s * 8, s < stage ? parity : parity ^ 1u);
}
__device__ __forceinline__ float fast_rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The planes of the k-th of the six products of float32 operands, smallest products first.
__device__ __forceinline__ int plane_a(int terms, int t) { return terms == 1 ? 0 : (0x001102 >> (4 * t)) & 3; }   // 2 0 1 1 0 0
__device__ __forceinline__ int plane_b(int terms, int t) { return terms == 1 ? 0 : (0x010120 >> (4 * t)) & 3; }   // 0 2 1 0 1 0

// x = p[0] + p[1] + p[2] for a finite x; infinities become the largest bfloat16 numbers, NaN stays in p[0].
__device__ __forceinline__ void split3(float x, bf16 (&p)[3]) {
  const float most = 3.3895313892515355e38f;
  if (fabsf(x) > most) x = copysignf(most, x);    // (false for NaN)
  p[0] = __float2bfloat16_rn(x);
  float rest = x - __bfloat162float(p[0]);
  p[1] = __float2bfloat16_rn(rest);
  rest -= __bfloat162float(p[1]);
  p[2] = __float2bfloat16_rn(rest);
}

// tanh(x) and 1 - tanh(x)^2: with h = 1 / (e^(2 |x|) + 1), which is half at most, 1 - 2 h with x's sign, and 4 h (1 - h); near 0, where the difference would cancel, the odd
// series up to x^7 (its next term is below 6e-8 of it). The tanh is off by less than 1e-6 of itself, so that a cap far above the logits leaves them as they are; the slope, on either side of 0, by
// half a millionth and what rounding the exponent makes of it, 1.2e-7 |x|.
__device__ __forceinline__ float cap_tanh(float x, float& slope) {
  const float h = fast_rcp(fast_exp2(fabsf(x) * (2.f * LOG2E)) + 1.f), q = x * x;
  const float series = fmaf(x * q, fmaf(q, fmaf(q, -17.f / 315.f, 2.f / 15.f), -1.f / 3.f), x);
  const bool near = q < 0.04f;
  slope = near ? fmaf(-series, series, 1.f) : 4.f * h * (1.f - h);
  return near ? series : copysignf(fmaf(-2.f, h, 1.f), x);
}

// z log2 e of an accumulator.
template <bool CAPPED> __device__ __forceinline__ float log2_units(float u, const Work& w) {
  if constexpr (!CAPPED) return u * LOG2E;
  float slope;
  return w.cap_out * cap_tanh(u * w.cap, slope);
}

struct Unit {   // one tile, or one share of its k
  int row, col, split, kb_begin, kb_end;
};

template <int MODE> __device__ __forceinline__ Unit unit_of(const Work& w, long long i, int row_tiles, int col_tiles, int n_kb) {
  Unit u;
  u.split = 0;
  u.kb_begin = 0;
  u.kb_end = n_kb;
  if constexpr (MODE == LOGSUM || MODE == FACTORS) {   // all rows of a column tile follow one another: the table is read once
    u.col = int(i / row_tiles);
    u.row = int(i % row_tiles);
  } else {
    const long long tile = i % (static_cast<long long>(row_tiles) * col_tiles);
    u.row = int(tile / col_tiles);
    u.col = int(tile % col_tiles);
    if constexpr (MODE == ROWS) {
      u.split = int(i / (static_cast<long long>(row_tiles) * col_tiles));
      u.kb_begin = u.split * w.per_split;
      u.kb_end = min(n_kb, u.kb_begin + w.per_split);
    }
  }
  return u;
}

// Steps of k that are added in tensor memory before their sum goes into registers (0: all): 256 of k with the products of planes; 512 where logits are
// made of more than 768 bfloat16 products (1,024 of them: off by up to 1.2e-6 of the loss otherwise; 1,600: by 2.4e-7 in place of 7.7e-7, and 5 % slower); 1,024 for the
// factors' logits, whose tiles take longer to finish than two accumulators of 512 hold products for (2,047 rows of 1,600: 728 us, of 1,024 615, all in one 572); 32,768 in gradients, whose sums are then off by 2^-13 at most, a 32th of half a step of bfloat16.
constexpr int PLANES_CHUNK = 4, LONG_CHUNK = 8, LONG_STEPS = 12, FACTORS_CHUNK = 16, GRADIENT_CHUNK = 512;

// How many times a unit's products go through an accumulator.
template <int CHUNKED> __device__ __forceinline__ int sums_of(const Unit& u) {
  if constexpr (CHUNKED > 0) return max(0, (u.kb_end - u.kb_begin + CHUNKED - 1) / CHUNKED);
  return 1;
}

// A warp's way out: rows of 128 bytes (the lane's row), two slabs in turn, each stored once it is whole.
struct Slabs {
  uint32_t base;   // of the warp's two
  int lane, turn;
  __device__ __forceinline__ uint32_t begin() {   // a slab that the copies have read
    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
    __syncwarp();
    return base + (turn++ & 1) * SLAB;
  }
  __device__ __forceinline__ void put16(uint32_t slab, int piece, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {   // swizzled, as the map has it
    st_shared16(slab + lane * 128 + ((piece ^ (lane & 7)) << 4), a, b, c, d);
  }
  __device__ __forceinline__ void end(const CUtensorMap* map, int x, int y, int plane, uint32_t slab, bool add) {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (lane == 0) {
      if (add) add_box(map, x, y, plane, slab);
      else store_box(map, x, y, plane, slab);
      asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    }
  }
};

// 64 columns of the thread's tensor-memory lane.
__device__ __forceinline__ void tmem_row64(uint32_t taddr, float (&v)[64]) {
  uint32_t a[32], b[32];
  tmem_load32(taddr, a);
  tmem_load32(taddr + 32, b);
  tmem_load_wait(a);
  tmem_tie(b);
#pragma unroll
  for (int j = 0; j < 32; ++j) {
    v[j] = __uint_as_float(a[j]);
    v[32 + j] = __uint_as_float(b[j]);
  }
}

// The work of pair `pair` of `n_pairs`.
template <int MODE, bool CAPPED, typename T, bool PLANES, int CHUNKED>
__device__ __forceinline__ void product(const CUtensorMap& map_a, const CUtensorMap& map_b, const CUtensorMap& map_out, const Work& w, const int pair, const int n_pairs) {
  constexpr bool A_MN = is_table(MODE), B_MN = MODE == ROWS || is_table(MODE);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t a_base = smem_u32(smem), b_base = a_base + STAGES * A_BYTES;
  const uint32_t slabs = b_base + STAGES * B_BYTES, full = slabs + 2 * WARPS * SLAB, empty = full + STAGES * 8, acc_full = empty + STAGES * 8, acc_empty = acc_full + 16;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + STAGES * size_t(A_BYTES + B_BYTES) + 2 * WARPS * SLAB + (2 * STAGES + 4) * 8);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t rank;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full + s * 8, 1);
      mbar_init(empty + s * 8, 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(acc_full + b * 8, 1);
      mbar_init(acc_empty + b * 8, 2 * WARPS);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_a) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_b) : "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(uint32_t(2 * BN)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  cluster_sync();   // both CTAs' barriers exist before either's loads, commits or arrivals signal them
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = *tmem_slot;
  pdl_wait();
  uint32_t leader_full, leader_acc_empty;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(leader_full) : "r"(full), "r"(0u));
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(leader_acc_empty) : "r"(acc_empty), "r"(0u));

  const int m = (MODE == FACTORS || MODE == ROWS) ? *w.count : w.m;
  const int k = is_table(MODE) ? *w.count : w.k;
  constexpr int TERMS = PLANES ? 6 : 1;
  const int n_kb = (k + BK - 1) / BK, row_tiles = (m + 2 * BM - 1) / (2 * BM), col_tiles = (w.n + BN - 1) / BN;
  const long long n_units = static_cast<long long>(row_tiles) * col_tiles * (MODE == ROWS ? w.splits : 1);

  if (warp == 0) {
    // ---- operands: the warp runs the loop, one elected lane issues. A stage is waited for with the opposite of the ring's parity, which a
    // fresh barrier passes at once.
    int stage = 0;
    uint32_t parity = 0;
    bool ok = true;
    for (long long i = pair; i < n_units && ok; i += n_pairs) {
      const Unit u = unit_of<MODE>(w, i, row_tiles, col_tiles, n_kb);
      const int a0 = (u.row * 2 + int(rank)) * BM, b0 = u.col * BN + int(rank) * HALF;
      for (int lo = u.kb_begin; lo < u.kb_end && ok; lo += CHUNKED > 0 ? CHUNKED : u.kb_end - u.kb_begin) {
        const int hi = CHUNKED > 0 ? min(lo + CHUNKED, u.kb_end) : u.kb_end;
        for (int t = 0; t < TERMS && ok; ++t) {   // (the smallest products first)
          for (int kb = lo; kb < hi; ++kb) {
            if (!warp_wait(empty + stage * 8, parity ^ 1u)) {
              if (lane == 0) atomicMax(w.error_flag, ERR_EMPTY);
              ok = false;
              break;
            }
            if (elect_one()) {
              const uint32_t bar = leader_full + stage * 8;
              const int k0 = kb * BK, pa = plane_a(TERMS, t), pb = plane_b(TERMS, t);
              if (rank == 0) mbar_expect_tx(full + stage * 8, 2 * (A_BYTES + B_BYTES));
              const uint32_t a = a_base + stage * A_BYTES, b = b_base + stage * B_BYTES;
              if constexpr (A_MN) {
                load_pair(a, &map_a, a0, k0, pa, bar);
                load_pair(a + BK * 128, &map_a, a0 + 64, k0, pa, bar);
              } else {
                load_pair(a, &map_a, k0, a0, pa, bar);
              }
              if constexpr (B_MN) {
                load_pair(b, &map_b, b0, k0, pb, bar);
                load_pair(b + BK * 128, &map_b, b0 + 64, k0, pb, bar);
              } else {
                load_pair(b, &map_b, k0, b0, pb, bar);
              }
            }
            __syncwarp();
            if (++stage == STAGES) {
              stage = 0;
              parity ^= 1u;
            }
          }
        }
      }
    }
    if (!ok && rank == 0) settle(full, STAGES, stage, parity);
  } else if (warp == 1 && rank == 0) {
    // ---- products of the pair (256 rows over the two CTAs)
    constexpr uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | (uint32_t(A_MN) << 15) | (uint32_t(B_MN) << 16) | (uint32_t(BN >> 3) << 17) |
                               (uint32_t((2 * BM) >> 4) << 24);
    const uint64_t a_desc = A_MN ? smem_desc(0, BK * 128, 1024) : smem_desc(0, 16, 1024);
    const uint64_t b_desc = B_MN ? smem_desc(0, BK * 128, 1024) : smem_desc(0, 16, 1024);
    constexpr uint32_t a_step = (A_MN ? UMMA_K * 128 : 32) >> 4, b_step = (B_MN ? UMMA_K * 128 : 32) >> 4;
    int stage = 0;
    uint32_t parity = 0, local = 0;   // this pair's count of sums: accumulator local & 1
    bool ok = true;
    for (long long i = pair; i < n_units && ok; i += n_pairs) {
      const Unit u = unit_of<MODE>(w, i, row_tiles, col_tiles, n_kb);
      const int sums = sums_of<CHUNKED>(u);
      for (int s = 0; s < sums && ok; ++s, ++local) {
        const uint32_t buf = local & 1u;
        if (!warp_wait(acc_empty + buf * 8, ((local >> 1) & 1u) ^ 1u)) {
          if (lane == 0) atomicMax(w.error_flag, ERR_ACC);
          ok = false;
          break;
        }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t acc = tmem + buf * BN;
        const int steps = CHUNKED > 0 ? min(CHUNKED, u.kb_end - u.kb_begin - s * CHUNKED) * TERMS : u.kb_end - u.kb_begin;
        for (int it = 0; it < steps; ++it) {
          if (!warp_wait(full + stage * 8, parity)) {
            if (lane == 0) atomicMax(w.error_flag, ERR_FULL);
            ok = false;
            break;
          }
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          if (elect_one()) {
            const uint32_t a = (a_base + stage * A_BYTES) >> 4, b = (b_base + stage * B_BYTES) >> 4;
#pragma unroll
            for (int kk = 0; kk < BK / UMMA_K; ++kk)
              umma_pair(acc, a_desc + (a & 0x3FFF) + kk * a_step, b_desc + (b & 0x3FFF) + kk * b_step, idesc, (it > 0 || kk > 0) ? 1u : 0u);
            commit_pair(empty + stage * 8);
          }
          __syncwarp();
          if (++stage == STAGES) {
            stage = 0;
            parity ^= 1u;
          }
        }
        if (R2_LOSS_GIVES_UP == 2) {
          if (lane == 0) atomicMax(w.error_flag, ERR_FULL);
          ok = false;
        }
        if (ok && elect_one()) commit_pair(acc_full + buf * 8);
        __syncwarp();
      }
    }
  } else if (warp >= 2) {
    // ---- results: each CTA its own 128 rows; a warp 32 of them (the lanes of tensor memory that it may read) and half of the columns
    const int q = warp & 3, side = (warp - 2) >> 2;
    Slabs out = {slabs + (warp - 2) * 2 * SLAB, lane, 0};
    uint32_t local = 0;
    bool ok = true;
    constexpr bool RESTS = MODE == TABLE && sizeof(T) == 2;
    auto run_of = [&](long long i, const Unit& u) {   // of the lane's token of a unit
      const int row = (u.row * 2 + int(rank)) * BM + q * 32 + lane;
      return i < n_units && row < m && w.segments > 0 ? __ldg(w.runs + row) : make_int2(0, 0);
    };
    [[maybe_unused]] Unit u_ahead = {};
    [[maybe_unused]] int2 run_ahead = make_int2(0, 0);
    if constexpr (RESTS) {
      u_ahead = unit_of<MODE>(w, pair, row_tiles, col_tiles, n_kb);
      run_ahead = run_of(pair, u_ahead);
    }
    for (long long i = pair; i < n_units; i += n_pairs) {
      const Unit u = RESTS ? u_ahead : unit_of<MODE>(w, i, row_tiles, col_tiles, n_kb);
      const int row = (u.row * 2 + int(rank)) * BM + q * 32 + lane;
      const int col0 = u.col * BN;
      int target = -1;
      float factor = 0.f, less2 = 0.f;   // |factor| exp(z - log_sum) is 2^(z log2 e - less2)
      if constexpr (MODE == FACTORS) {
        if (row < m) {
          target = w.targets[row] - w.first - col0;   // (no overflow: both lie in [0, vocab))
          factor = w.factor[row];
          less2 = w.log_sum[row] * LOG2E - log2f(fabsf(factor));
        }
      }
      const int row0 = (u.row * 2 + int(rank)) * BM + q * 32;
      float top = -3.4028234663852886e38f, sum = 0.f;
      // TABLE_FEW: what rounding left of dz at the tokens of the warp's 32 rows, in the order of the gathered rows (FEW of them at most; their tokens are asked for
      // before the accumulator is waited for)
      int token[FEW / 32];
      if constexpr (MODE == TABLE_FEW) {
#pragma unroll
        for (int i = 0; i < FEW / 32; ++i) token[i] = 32 * i + lane < k ? w.targets[32 * i + lane] - w.first - row0 : -1;
      }
      auto add_rest = [&](int c, float (&v)[64]) {
        if constexpr (MODE == TABLE_FEW) {
#pragma unroll
          for (int i = 0; i < FEW / 32; ++i) {
#pragma unroll 1
            for (unsigned mask = __ballot_sync(0xffffffffu, token[i] >= 0 && token[i] < 32); mask != 0; mask &= mask - 1u) {
              const int from = __ffs(int(mask)) - 1, to = __shfl_sync(0xffffffffu, token[i], from);
              if (lane == to) {
                const float rest = w.rest[32 * i + from];
                const bf16* x = w.x + (32 * i + from) * w.ld_x + col0 + c;
#pragma unroll
                for (int p = 0; p < 8; ++p) {
                  if (col0 + c + 8 * p < w.n) {   // (rows of whole eights)
                    const uint4 q8 = *reinterpret_cast<const uint4*>(x + 8 * p);
                    const uint32_t q2[4] = {q8.x, q8.y, q8.z, q8.w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                      v[8 * p + 2 * j] = fmaf(rest, __uint_as_float(q2[j] << 16), v[8 * p + 2 * j]);
                      v[8 * p + 2 * j + 1] = fmaf(rest, __uint_as_float(q2[j] & 0xffff0000u), v[8 * p + 2 * j + 1]);
                    }
                  }
                }
              }
            }
          }
        }
      };
      // bfloat16 TABLE: their sums by rests_kernel, of a few of the warp's 32 tokens (asked for a tile ahead)
      const int2 run = run_ahead;
      if constexpr (RESTS) {
        u_ahead = unit_of<MODE>(w, i + n_pairs, row_tiles, col_tiles, n_kb);
        run_ahead = run_of(i + n_pairs, u_ahead);
      }
      auto add_rests = [&](int c, float (&v)[64]) {
        if constexpr (RESTS) {
          for (int segment = 0; segment < w.segments; ++segment) {
            const int2 of = segment == 0 ? run : row < m ? __ldg(w.runs + static_cast<long long>(segment) * w.run_tokens + row) : make_int2(0, 0);
#pragma unroll 1
            for (int at = of.x; at < of.y; at = (at / WINDOW + 1) * WINDOW) {
              const float4* sum = reinterpret_cast<const float4*>(w.sums + at * w.ld_sums + col0 + c);
              const int last = (w.n - col0 - c - 1) / 4;   // (what is added behind it is not stored)
              float4 q[16];
#pragma unroll
              for (int p = 0; p < 16; ++p) q[p] = __ldg(sum + min(p, last));
#pragma unroll
              for (int p = 0; p < 16; ++p) v[4 * p] += q[p].x, v[4 * p + 1] += q[p].y, v[4 * p + 2] += q[p].z, v[4 * p + 3] += q[p].w;
            }
          }
        }
      };
      // 64 finished numbers of a row, from column c of the tile on
      auto finish = [&](int c, float (&v)[64]) {
        if constexpr (MODE == TABLE_FEW) add_rest(c, v);
        if constexpr (RESTS) add_rests(c, v);
        if constexpr (MODE == LOGSUM) {
#pragma unroll
          for (int j = 0; j < 64; ++j) v[j] = log2_units<CAPPED>(v[j], w);
          if (col0 + c + 64 > w.n) {
#pragma unroll
            for (int j = 0; j < 64; ++j) v[j] = col0 + c + j < w.n ? v[j] : -INFINITY;
          }
          float most = top;
#pragma unroll
          for (int j = 0; j < 64; j += 2) most = max3(most, v[j], v[j + 1]);
          float s0 = sum * fast_exp2(top - most), s1 = 0.f;
#pragma unroll
          for (int j = 0; j < 64; j += 2) {
            s0 += fast_exp2(v[j] - most);
            s1 += fast_exp2(v[j + 1] - most);
          }
          sum = s0 + s1;
          top = most;
        } else if constexpr (MODE == FACTORS) {
          const float size = fabsf(factor);
          // of a pair, once it is rounded: the factor's sign; zeros in rows behind the last one, which the table's gradient adds to its sums
          const uint32_t sign = factor < 0.f ? 0x80008000u : 0u, held = row < m ? 0xffffffffu : 0u;
          const bool learns = __any_sync(0xffffffffu, target >= c && target < c + 64);
          if constexpr (CAPPED) {
#pragma unroll
            for (int j = 0; j < 64; ++j) {
              float slope;
              v[j] = fast_exp2(fmaf(w.cap_out, cap_tanh(v[j] * w.cap, slope), -less2));
              if (learns) v[j] -= target == c + j ? size : 0.f;
              v[j] *= slope;
            }
          } else {
#pragma unroll
            for (int j = 0; j < 64; ++j) v[j] = fast_exp2(fmaf(v[j], LOG2E, -less2));
            if (learns) {
#pragma unroll
              for (int j = 0; j < 64; ++j) v[j] -= target == c + j ? size : 0.f;
            }
          }
          if constexpr (!PLANES) {
            if (learns && target >= c && target < c + 64) {
              float rest = 0.f;
#pragma unroll
              for (int j = 0; j < 64; ++j) rest = target == c + j ? v[j] - __bfloat162float(__float2bfloat16_rn(v[j])) : rest;
              w.rest[row] = factor < 0.f ? -rest : rest;
            }
          }
          for (int plane = 0; plane < (PLANES ? 3 : 1); ++plane) {
            const uint32_t slab = out.begin();
#pragma unroll
            for (int p = 0; p < 8; ++p) {
              uint32_t r[4];
#pragma unroll
              for (int j = 0; j < 4; ++j) r[j] = pack_bf16(v[8 * p + 2 * j], v[8 * p + 2 * j + 1]);
              out.put16(slab, p, (r[0] & held) ^ sign, (r[1] & held) ^ sign, (r[2] & held) ^ sign, (r[3] & held) ^ sign);
              if constexpr (PLANES) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  v[8 * p + 2 * j] -= __uint_as_float(r[j] << 16);
                  v[8 * p + 2 * j + 1] -= __uint_as_float(r[j] & 0xffff0000u);
                }
              }
            }
            out.end(&map_out, col0 + c, row0, plane, slab, false);
          }
        } else if (is_table(MODE) && w.out != nullptr) {
          T* to = static_cast<T*>(w.out) + row * w.ld + col0 + c;
#pragma unroll
          for (int j = 0; j < 64; ++j)
            if (row < m && col0 + c + j < w.n) to[j] = from_float<T>(v[j]);
        } else if constexpr (is_table(MODE) && sizeof(T) == 2) {
          const uint32_t slab = out.begin();
#pragma unroll
          for (int p = 0; p < 8; ++p)
            out.put16(slab, p, pack_bf16(v[8 * p], v[8 * p + 1]), pack_bf16(v[8 * p + 2], v[8 * p + 3]), pack_bf16(v[8 * p + 4], v[8 * p + 5]),
                      pack_bf16(v[8 * p + 6], v[8 * p + 7]));
          out.end(&map_out, col0 + c, row0, 0, slab, false);
        } else {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const uint32_t slab = out.begin();
#pragma unroll
            for (int p = 0; p < 8; ++p)
              out.put16(slab, p, __float_as_uint(v[32 * half + 4 * p]), __float_as_uint(v[32 * half + 4 * p + 1]), __float_as_uint(v[32 * half + 4 * p + 2]),
                        __float_as_uint(v[32 * half + 4 * p + 3]));
            out.end(&map_out, col0 + c + 32 * half, row0, u.split, slab, MODE == ROWS && w.add);
          }
        }
      };
      auto left = [&](int c) { return col0 + c < w.n && (MODE == LOGSUM || MODE == FACTORS || row0 < m); };
      auto give_up = [&] {   // NaN in place of the warp's part of the tile (for LOGSUM below)
        if constexpr (MODE != LOGSUM) {
          constexpr bool NARROW = MODE == FACTORS || sizeof(T) == 2;   // two numbers to four bytes
          constexpr int COLUMNS = NARROW ? 64 : 32;
          const uint32_t nan = MODE == FACTORS && row >= m ? 0u : NARROW ? 0x7fff7fffu : 0x7fffffffu;
          if constexpr (MODE == FACTORS && !PLANES) {
            if (target >= side * HALF && target < (side + 1) * HALF) w.rest[row] = NAN;
          }
#pragma unroll 1
          for (int c = side * HALF; c < (side + 1) * HALF && left(c); c += COLUMNS) {
            if (is_table(MODE) && w.out != nullptr) {
#pragma unroll 1
              for (int j = 0; j < COLUMNS; ++j)
                if (row < m && col0 + c + j < w.n) static_cast<T*>(w.out)[row * w.ld + col0 + c + j] = from_float<T>(NAN);
              continue;
            }
#pragma unroll 1
            for (int plane = 0; plane < (PLANES && MODE == FACTORS ? 3 : 1); ++plane) {
              const uint32_t slab = out.begin();
#pragma unroll 1
              for (int p = 0; p < 8; ++p) out.put16(slab, p, nan, nan, nan, nan);
              out.end(&map_out, col0 + c, row0, MODE == ROWS ? u.split : plane, slab, MODE == ROWS && w.add);
            }
          }
        }
      };
      const uint32_t lanes = uint32_t(q * 32) << 16;
      auto wait_sum = [&](uint32_t buf) {
        if (ok && (!warp_wait(acc_full + buf * 8, (local >> 1) & 1u) || R2_LOSS_GIVES_UP == 1)) {
          if (lane == 0) atomicMax(w.error_flag, ERR_ACC);
          ok = false;
        }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      };
      auto hand_back = [&](uint32_t buf) {
        if (!ok) return;
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) arrive_cluster(leader_acc_empty + buf * 8);
        ++local;
      };
      if constexpr (CHUNKED > 0) {
        float lo[64], hi[64];
#pragma unroll
        for (int j = 0; j < 64; ++j) lo[j] = hi[j] = 0.f;
        const int sums = sums_of<CHUNKED>(u);   // (none: zeros)
#pragma unroll 1
        for (int s = 0; s < sums; ++s) {
          const uint32_t buf = local & 1u;
          wait_sum(buf);
          if (ok && left(side * HALF)) {
            uint32_t r[32];
#pragma unroll
            for (int part = 0; part < 4; ++part) {
              tmem_load32(tmem + buf * BN + uint32_t(side * HALF + part * 32) + lanes, r);
              tmem_load_wait(r);
#pragma unroll
              for (int j = 0; j < 32; ++j) (part < 2 ? lo : hi)[part % 2 * 32 + j] += __uint_as_float(r[j]);
            }
          }
          hand_back(buf);
        }
        if (!ok) give_up();
        if (ok && left(side * HALF)) finish(side * HALF, lo);
        if (ok && left(side * HALF + 64)) finish(side * HALF + 64, hi);
      } else {
        const uint32_t buf = local & 1u;
        wait_sum(buf);
        const bool none = u.kb_end <= u.kb_begin;   // nothing to sum over: zeros
#pragma unroll 1
        for (int c = side * HALF; c < (side + 1) * HALF && ok && left(c); c += 64) {
          float v[64];
          tmem_row64(tmem + buf * BN + uint32_t(c) + lanes, v);
          if constexpr (MODE == ROWS || is_table(MODE)) {
#pragma unroll
            for (int j = 0; j < 64; ++j) v[j] = none ? 0.f : v[j];
          }
          finish(c, v);
        }
        if (!ok) give_up();
        hand_back(buf);
      }
      if constexpr (MODE == LOGSUM) {
        if (row < m) w.part[size_t(row) * w.parts + u.col * 2 + side] = ok ? make_float2(top, sum) : make_float2(NAN, NAN);
      }
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }

  // (The next kernel's CTAs start when this one's have ended: let in at this point they cost a product of 105 us 4 to 6 us, let in at the start 12.)
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  cluster_sync();   // neither CTA frees tensor memory or leaves while the other may still use it
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(uint32_t(2 * BN)) : "memory");
  }
}

template <int MODE, bool CAPPED, typename T, bool PLANES, int CHUNKED>
__global__ void __launch_bounds__(THREADS, 1) product_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                                                              const __grid_constant__ CUtensorMap map_out, const Work w) {
  product<MODE, CAPPED, T, PLANES, CHUNKED>(map_a, map_b, map_out, w, int(blockIdx.x >> 1), int(gridDim.x >> 1));   // the cluster lies along x
}

// Both products with dz side by side, where their tiles do not fill the GPU together: a launch less, and neither waits for the other (16 float32 rows of 100, 1,031 tokens: loss and gradients 55 to 47 us with the copies of rows and table in one launch).
struct Both {
  CUtensorMap rows_a, rows_b, rows_out, table_a, table_b, table_out;
  Work rows, table;
  int rows_pairs;
};

template <int TABLE_MODE, typename T, bool PLANES, int CHUNKED> __global__ void __launch_bounds__(THREADS, 1) both_kernel(const __grid_constant__ Both b) {
  const int pair = int(blockIdx.x >> 1), n_pairs = int(gridDim.x >> 1);
  if (pair < b.rows_pairs) product<ROWS, false, float, PLANES, CHUNKED>(b.rows_a, b.rows_b, b.rows_out, b.rows, pair, b.rows_pairs);
  else product<TABLE_MODE, false, T, PLANES, CHUNKED>(b.table_a, b.table_b, b.table_out, b.table, pair - b.rows_pairs, n_pairs - b.rows_pairs);
}

// ---- few rows: LOGSUM and FACTORS of up to 128 ----------------------------------------------
//
// The pass over the table is what such a call costs, so the operands change sides: a tile is 128 tokens of the vocabulary by all rows (up to 128 columns of the
// accumulator), one CTA to an SM, and float32 tables are read as they are: eight warps turn each 128 x 32 numbers into the three planes in shared memory, where
// the others' planes would have been written to memory and read again (six bytes a number, twice). A tile's results go through shared memory, 32
// rows of the batch at a time, so that a thread has 32 tokens of one row: sums over them need no exchange, and dz leaves in pieces of 64 bytes.
//
// LOGSUM keeps a row's largest logit and sum for each of a CTA's four parts of 32 tokens over all its tiles.

constexpr int FEW_STAGES = 8;       // of operands, at most
constexpr int TURNED = 132;         // floats of a row of the turned tile (128 tokens and four of padding)
constexpr int FEW_CHUNK = 256;      // of k are added in tensor memory before their sum is rounded (three bfloat16 rows of 768: loss off by 1.4e-6 without, 8e-7 with; same time)

// Groups of four warps that split float32 numbers, and stages of planes. At GPT-2's table, a call with cold caches: 96 rows with two groups 66.6 us, three 68.6; 16 rows with three,
// four and five stages 56 to 58. (Without five of the six products 52 and 58, without the splitting 54 and 63: no part of a step bounds it alone.)
constexpr int GROUPS = 2, F32_STAGES = 3;
constexpr int few_threads(bool f32) { return 192 + (f32 ? GROUPS * 128 : 0); }

struct FewWork {
  int rows, columns;                // of the batch; a multiple of 16: columns of the accumulator
  int n, k;                         // tokens (of the table, or of a piece); width
  int stages, loads;                // of operands; float32: of operands in planes, of the table's numbers
  Work w;                           // count, cap, cap_out, targets, factor, log_sum, first, part, error_flag as above
  bf16* dz;
  long long dz_plane, ld;
};

__device__ __forceinline__ uint64_t smem_desc_64(uint32_t addr) {   // K-major rows of 64 bytes, 64-byte swizzle
  uint64_t d = 0;
  d |= uint64_t((addr >> 4) & 0x3FFF);
  d |= uint64_t(1) << 16;
  d |= uint64_t(512 >> 4) << 32;
  d |= uint64_t(1) << 46;
  d |= uint64_t(4) << 61;
  return d;
}
__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap* map, int x, int y, int plane, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
               ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(plane) : "memory");
}

// Whether any of the 128 threads of barrier 1 says so, which meet there.
__device__ __forceinline__ bool any_of_128(bool mine) {
  uint32_t any;
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, 1, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(any) : "r"(uint32_t(mine)) : "memory");
  return any != 0;
}

// Shared memory from its 1,024-byte aligned start. bfloat16: stages of 16 KB of the table and columns * 128 bytes of rows. float32: `loads` of 16 KB of the
// table's numbers, stages of three planes of 8 KB and columns * 64 bytes each. Then the turned tile and the barriers.
template <bool F32> __host__ __device__ constexpr uint32_t few_stage_bytes(int columns) {
  return F32 ? 3u * (8192u + uint32_t(columns) * 64u) : 16384u + uint32_t(columns) * 128u;
}
constexpr uint32_t TURNED_BYTES = 32 * TURNED * 4;
template <bool F32> __host__ __device__ constexpr uint32_t few_smem(int columns, int stages, int loads) {
  return 1024u + uint32_t(stages) * few_stage_bytes<F32>(columns) + (F32 ? uint32_t(loads) * 16384u : 0u) + TURNED_BYTES + (4 * FEW_STAGES + 4) * 8 + 16;
}

template <int MODE, bool CAPPED, bool F32, bool SUMS>
__global__ void __launch_bounds__(few_threads(F32), 1) few_kernel(const __grid_constant__ CUtensorMap map_t, const __grid_constant__ CUtensorMap map_x, const FewWork f) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t stage_bytes = few_stage_bytes<F32>(f.columns);
  const uint32_t loads_at = smem_u32(smem), stages_at = loads_at + (F32 ? uint32_t(f.loads) * 16384u : 0u);
  float* turned = reinterpret_cast<float*>(smem + (stages_at - loads_at) + size_t(f.stages) * stage_bytes);
  const uint32_t full = smem_u32(turned) + TURNED_BYTES, empty = full + FEW_STAGES * 8, loaded = empty + FEW_STAGES * 8, taken = loaded + FEW_STAGES * 8,
                 acc_full = taken + FEW_STAGES * 8, acc_empty = acc_full + 16;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(reinterpret_cast<uint8_t*>(turned) + TURNED_BYTES + (4 * FEW_STAGES + 4) * 8);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // Two accumulators, in float32 of two parts each: the products of the first planes, and the small ones, which would be cut off against them; behind them the
  // sums of a tile's pieces. (More than 96 float32 rows have one: tensor memory has no columns for another.)
  const uint32_t apart = uint32_t(f.columns + 31) / 32 * 32, both = F32 ? 2 * apart : apart;
  const uint32_t bufs = 2 * both + (SUMS ? apart : 0) <= 512 ? 2 : 1, sums_at = bufs * both;
  uint32_t tmem_cols = 32;
  while (tmem_cols < sums_at + (SUMS ? apart : 0)) tmem_cols <<= 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < FEW_STAGES; ++s) {
      mbar_init(full + s * 8, F32 ? 5 : 1);   // the copies, and four warps' planes
      mbar_init(empty + s * 8, 1);
      mbar_init(loaded + s * 8, 1);
      mbar_init(taken + s * 8, 4);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(acc_full + b * 8, 1);
      mbar_init(acc_empty + b * 8, 4);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_t) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_x) : "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(tmem_cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = *tmem_slot;
  pdl_wait();

  const int tiles = (f.n + 127) / 128;
  constexpr int STEP = F32 ? 32 : 64;   // of k
  const int n_kb = (f.k + STEP - 1) / STEP;
  const int per_sum = SUMS ? FEW_CHUNK / STEP : n_kb;
  const uint32_t x_bytes = uint32_t(f.columns) * STEP * 2;

  if (warp == 0) {
    // ---- copies
    int stage = 0;
    uint32_t parity = 0;
    bool ok = true;
    for (int tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x) {
      for (int kb = 0; kb < n_kb; ++kb) {
        // (float32: the table's numbers; the rows' planes come with the table's, below)
        const uint32_t slot = F32 ? taken : empty;
        if (!warp_wait(slot + stage * 8, parity ^ 1u)) {
          if (lane == 0) atomicMax(f.w.error_flag, ERR_EMPTY);
          ok = false;
          break;
        }
        if (elect_one()) {
          if constexpr (F32) {
            mbar_expect_tx(loaded + stage * 8, 16384);
            load_box(loads_at + stage * 16384, &map_t, kb * STEP, tile * 128, 0, loaded + stage * 8);
          } else {
            const uint32_t at = stages_at + stage * stage_bytes, bar = full + stage * 8;
            mbar_expect_tx(bar, 16384 + x_bytes);
            load_box(at, &map_t, kb * STEP, tile * 128, 0, bar);
            load_box(at + 16384, &map_x, kb * STEP, 0, 0, bar);
          }
        }
        __syncwarp();
        if (++stage == (F32 ? f.loads : f.stages)) {
          stage = 0;
          parity ^= 1u;
        }
      }
    }
    if (!ok) settle(F32 ? loaded : full, F32 ? f.loads : f.stages, stage, parity);
  } else if (warp == 1) {
    // ---- products
    const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | (uint32_t(f.columns >> 3) << 17) | (uint32_t(128 >> 4) << 24);
    int stage = 0;
    uint32_t parity = 0, local = 0;
    bool ok = true;
    for (int tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x) {
      for (int lo = 0; lo < n_kb && ok; lo += per_sum, ++local) {
        const uint32_t buf = local & (bufs - 1);
        if (!warp_wait(acc_empty + buf * 8, ((local >> (bufs - 1)) & 1u) ^ 1u)) {
          if (lane == 0) atomicMax(f.w.error_flag, ERR_ACC);
          ok = false;
          break;
        }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t acc = tmem + buf * both;
        for (int kb = lo; kb < min(n_kb, lo + per_sum); ++kb) {
          if (!warp_wait(full + stage * 8, parity)) {
            if (lane == 0) atomicMax(f.w.error_flag, ERR_FULL);
            ok = false;
            break;
          }
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          if (elect_one()) {
            const uint32_t at = stages_at + stage * stage_bytes;
            if constexpr (F32) {
#pragma unroll
              for (int t = 0; t < 6; ++t) {
                const uint64_t a = smem_desc_64(at + plane_a(6, t) * 8192), b = smem_desc_64(at + 3 * 8192 + plane_b(6, t) * x_bytes);
#pragma unroll
                for (int kk = 0; kk < 2; ++kk)
                  umma_bf16(t < 5 ? acc + apart : acc, a + kk * 2, b + kk * 2, idesc, (kb > lo || (t > 0 && t < 5) || kk > 0) ? 1u : 0u);
              }
            } else {
              const uint64_t a = smem_desc(at, 16, 1024), b = smem_desc(at + 16384, 16, 1024);
#pragma unroll
              for (int kk = 0; kk < 4; ++kk) umma_bf16(acc, a + kk * 2, b + kk * 2, idesc, (kb > lo || kk > 0) ? 1u : 0u);
            }
            umma_commit(empty + stage * 8);
          }
          __syncwarp();
          if (++stage == f.stages) {
            stage = 0;
            parity ^= 1u;
          }
        }
        if (R2_LOSS_GIVES_UP == 2) {
          if (lane == 0) atomicMax(f.w.error_flag, ERR_FULL);
          ok = false;
        }
        if (ok && elect_one()) umma_commit(acc_full + buf * 8);
        __syncwarp();
      }
    }
  } else if (warp < 6) {
    // ---- results
    const int q = warp & 3, part = warp - 2;   // tensor-memory lanes q * 32 ..; behind the turn: 32 tokens (part) of row `lane` of 32
    const int m = MODE == FACTORS ? *f.w.count : f.rows;
    const int groups = MODE == FACTORS ? (f.rows + 63) / 64 * 2 : (f.rows + 31) / 32;   // of 32 rows; dz has zeros up to a multiple of 64 rows
    float top[FEW / 32], sum[FEW / 32];
#pragma unroll
    for (int g = 0; g < FEW / 32; ++g) {
      top[g] = -3.4028234663852886e38f;
      sum[g] = 0.f;
    }
    uint32_t local = 0;
    bool ok = true;
    for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
      const int left = f.n - tile * 128 - part * 32;   // tokens of the thread's 32 that there are
      uint32_t buf = 0;
      for (int lo = 0; lo < n_kb; lo += per_sum) {
        buf = local & (bufs - 1);
        if (ok && (!warp_wait(acc_full + buf * 8, (local >> (bufs - 1)) & 1u) || R2_LOSS_GIVES_UP == 1)) {
          if (lane == 0) atomicMax(f.w.error_flag, ERR_ACC);
          ok = false;
        }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if constexpr (SUMS) {   // the sum of the pieces of k so far
#pragma unroll 1
          for (uint32_t c = uint32_t(q * 32) << 16; (c & 0xffffu) < apart; c += 32) {
            uint32_t r[32], more[32];
            tmem_load32(tmem + buf * both + c, r);
            if constexpr (F32) {
              tmem_load32(tmem + buf * both + apart + c, more);
              tmem_load_wait(r);
              tmem_tie(more);
#pragma unroll
              for (int j = 0; j < 32; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) + __uint_as_float(more[j]));
            }
            if (lo > 0) {
              tmem_load32(tmem + sums_at + c, more);
              tmem_load_wait(r);
              tmem_tie(more);
#pragma unroll
              for (int j = 0; j < 32; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) + __uint_as_float(more[j]));
            } else {
              tmem_load_wait(r);
            }
            tmem_store32(tmem + sums_at + c, r);
          }
          tmem_store_wait();
          asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
          __syncwarp();
          if (lane == 0 && ok) mbar_arrive(acc_empty + buf * 8);
          ++local;
        }
      }
#pragma unroll
      for (int g = 0; g < FEW / 32; ++g) {
        if (g >= groups) break;
        if (uint32_t(g * 32) < apart) {
          uint32_t r[32];
          tmem_load32(tmem + (SUMS ? sums_at : buf * both) + uint32_t(g * 32) + (uint32_t(q * 32) << 16), r);
          tmem_load_wait(r);
#pragma unroll
          for (int j = 0; j < 32; ++j) turned[j * TURNED + q * 32 + lane] = __uint_as_float(r[j]);
        }
        ok = !any_of_128(!ok);   // (what a warp turns is of all four warps' lanes)
        if (!ok) {
#pragma unroll 1
          for (int j = 0; j < 32; ++j) turned[lane * TURNED + part * 32 + j] = NAN;   // (what this thread reads)
        }
        const int row = g * 32 + lane;
        float v[32];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float4 x = *reinterpret_cast<const float4*>(turned + lane * TURNED + part * 32 + 4 * i);   // (given up: NaN, below)
          v[4 * i] = x.x, v[4 * i + 1] = x.y, v[4 * i + 2] = x.z, v[4 * i + 3] = x.w;
        }
        if constexpr (MODE == LOGSUM) {
          float most = top[g];
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = log2_units<CAPPED>(v[j], f.w);
          if (left < 32) {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = j < left ? v[j] : -INFINITY;
          }
#pragma unroll
          for (int j = 0; j < 32; j += 2) most = max3(most, v[j], v[j + 1]);
          float s0 = sum[g] * fast_exp2(top[g] - most), s1 = 0.f;
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            s0 += fast_exp2(v[j] - most);
            s1 += fast_exp2(v[j + 1] - most);
          }
          sum[g] = s0 + s1;
          top[g] = most;
        } else {
          int target = -1;
          float factor = 0.f, size = 0.f, less2 = 0.f;
          const int token0 = tile * 128 + part * 32;
          if (row < m) {
            target = f.w.targets[row] - f.w.first - token0;
            factor = f.w.factor[row];
            size = fabsf(factor);
            less2 = f.w.log_sum[row] * LOG2E - log2f(size);
          }
          const bool learns = target >= 0 && target < 32;
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            if constexpr (CAPPED) {
              float slope;
              v[j] = fast_exp2(fmaf(f.w.cap_out, cap_tanh(v[j] * f.w.cap, slope), -less2));
              if (learns) v[j] -= target == j ? size : 0.f;
              v[j] *= slope;
            } else {
              v[j] = fast_exp2(fmaf(v[j], LOG2E, -less2));
              if (learns) v[j] -= target == j ? size : 0.f;
            }
          }
          if constexpr (!F32) {
            if (learns) {
              float rest = 0.f;
#pragma unroll
              for (int j = 0; j < 32; ++j) rest = target == j ? v[j] - __bfloat162float(__float2bfloat16_rn(v[j])) : rest;
              f.w.rest[row] = factor < 0.f ? -rest : rest;
            }
          }
          const uint32_t sign = factor < 0.f ? 0x80008000u : 0u, held = row < m ? 0xffffffffu : 0u;
          if (left > 0) {
            bf16* to = f.dz + row * f.ld + token0;
            for (int plane = 0; plane < (F32 ? 3 : 1); ++plane) {
#pragma unroll
              for (int p = 0; p < 4; ++p) {
                uint32_t r[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) r[j] = pack_bf16(v[8 * p + 2 * j], v[8 * p + 2 * j + 1]);
                *reinterpret_cast<uint4*>(to + plane * f.dz_plane + 8 * p) =
                    make_uint4((r[0] & held) ^ sign, (r[1] & held) ^ sign, (r[2] & held) ^ sign, (r[3] & held) ^ sign);
                if constexpr (F32) {
#pragma unroll
                  for (int j = 0; j < 4; ++j) {
                    v[8 * p + 2 * j] -= __uint_as_float(r[j] << 16);
                    v[8 * p + 2 * j + 1] -= __uint_as_float(r[j] & 0xffff0000u);
                  }
                }
              }
            }
          }
        }
        asm volatile("bar.sync 1, 128;" ::: "memory");   // (the turned tile is read)
      }
      if constexpr (!SUMS) {
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0 && ok) mbar_arrive(acc_empty + buf * 8);
        ++local;
      }
    }
    if constexpr (MODE == LOGSUM) {
#pragma unroll
      for (int g = 0; g < FEW / 32; ++g) {
        const int row = g * 32 + lane;
        if (row < m) f.w.part[size_t(row) * f.w.parts + blockIdx.x * 4 + part] = ok ? make_float2(top[g], sum[g]) : make_float2(NAN, NAN);
      }
    }
  } else if constexpr (F32) {
    // ---- planes: a thread a token's 32 numbers; groups of four warps take the steps in turn
    const int group = (warp - 6) / 4, row = (warp - 6) % 4 * 32 + lane;
    const int steps = (tiles - int(blockIdx.x) + int(gridDim.x) - 1) / int(gridDim.x) * n_kb;   // of all this CTA's tiles
    int stage = 0, load = 0, kb = 0;
    uint32_t parity = 0, load_parity = 0;
    auto forward = [&](int n) {
      kb = (kb + n) % n_kb;
      for (stage += n; stage >= f.stages; stage -= f.stages) parity ^= 1u;
      for (load += n; load >= f.loads; load -= f.loads) load_parity ^= 1u;
    };
    forward(group);
    bool ok = true;
    for (int i = group; i < steps; i += GROUPS, forward(GROUPS)) {
      if (!warp_wait(loaded + load * 8, load_parity)) {
        if (lane == 0) atomicMax(f.w.error_flag, ERR_FULL);
        ok = false;
        break;
      }
      const uint8_t* from = smem + load * 16384 + row * 128;
      float v[32];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float4 x = *reinterpret_cast<const float4*>(from + ((j ^ (row & 7)) << 4));
        v[4 * j] = x.x, v[4 * j + 1] = x.y, v[4 * j + 2] = x.z, v[4 * j + 3] = x.w;
      }
      if (!warp_wait(empty + stage * 8, parity ^ 1u)) {
        if (lane == 0) atomicMax(f.w.error_flag, ERR_EMPTY);
        ok = false;
        break;
      }
      if (warp == 6 + 4 * group && elect_one()) {
        mbar_expect_tx(full + stage * 8, 3 * x_bytes);
        for (int p = 0; p < 3; ++p) load_box(stages_at + stage * stage_bytes + 3 * 8192 + p * x_bytes, &map_x, kb * STEP, 0, p, full + stage * 8);
      }
      __syncwarp();
      const uint32_t to = stages_at + stage * stage_bytes + row * 64;
      const float most = 3.3895313892515355e38f;
#pragma unroll
      for (int j = 0; j < 32; ++j) asm("min.NaN.f32 %0, %0, %1;\n\tmax.NaN.f32 %0, %0, %2;" : "+f"(v[j]) : "f"(most), "f"(-most));   // (as split3)
#pragma unroll
      for (int p = 0; p < 3; ++p) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t r[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            r[j] = pack_bf16(v[8 * c + 2 * j], v[8 * c + 2 * j + 1]);
            if (p < 2) {
              v[8 * c + 2 * j] -= __uint_as_float(r[j] << 16);
              v[8 * c + 2 * j + 1] -= __uint_as_float(r[j] & 0xffff0000u);
            }
          }
          st_shared16(to + p * 8192 + ((c ^ ((row >> 1) & 3)) << 4), r[0], r[1], r[2], r[3]);
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(full + stage * 8);
        mbar_arrive(taken + load * 8);   // (here, where the numbers have been used: handed back right behind the loads, the next copy has overtaken them)
      }
    }
    if (!ok && warp == 6 + 4 * group) settle(full, f.stages, stage, parity);
  }

  pdl_launch_dependents();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(tmem_cols) : "memory");
  }
}

// Eight numbers of a row from column c on (zeros behind the last); `wide`: rows start at 16 bytes and hold whole eights.
template <typename T> __device__ __forceinline__ void load8(const T* row, int c, int width, bool wide, float (&v)[8]) {
  if (wide) {
    if constexpr (sizeof(T) == 2) {
      const uint4 x = __ldg(reinterpret_cast<const uint4*>(row + c));
      const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[2 * j] = __uint_as_float(w[j] << 16);
        v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
      }
    } else {
      const float4 x = __ldg(reinterpret_cast<const float4*>(row + c)), y = __ldg(reinterpret_cast<const float4*>(row + c + 4));
      v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w, v[4] = y.x, v[5] = y.y, v[6] = y.z, v[7] = y.w;
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = c + j < width ? to_float(row[c + j]) : 0.f;
}

// The same numbers in one plane or in three, at places of 16 bytes.
template <typename T> __device__ __forceinline__ void put_planes8(bf16* to, long long plane, const float (&v)[8]) {
  uint4 out[sizeof(T) == 2 ? 1 : 3];
  bf16(*p)[8] = reinterpret_cast<bf16(*)[8]>(out);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if constexpr (sizeof(T) == 2) {
      p[0][j] = __float2bfloat16_rn(v[j]);
    } else {
      bf16 s[3];
      split3(v[j], s);
#pragma unroll
      for (int i = 0; i < 3; ++i) p[i][j] = s[i];
    }
  }
#pragma unroll
  for (int i = 0; i < int(sizeof(T) == 2 ? 1 : 3); ++i) *reinterpret_cast<uint4*>(to + i * plane) = out[i];
}

template <typename T> __device__ __forceinline__ bool rows_wide(const T* at, long long ld, int width) {
  return reinterpret_cast<uintptr_t>(at) % 16 == 0 && ld * sizeof(T) % 16 == 0 && width % 8 == 0;
}

// A warp a row: its parts joined, and the target's logit as a sum of float products.
template <typename T>
__global__ void __launch_bounds__(256) finish_kernel(const float2* part, int parts, const T* hidden, long long ld_h, const T* table, long long ld_t, const int32_t* targets,
                                                     const float* weight, int rows, int width, int vocab, float softcap, float* loss, float* log_sum) {
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, r = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (r >= rows) return;
  const int y = targets[r];
  const float factor = weight ? weight[r] : 1.f;
  const bool counts = y >= 0 && y < vocab && factor != 0.f;
  const T* x = hidden + size_t(r) * ld_h;
  const T* t = table + size_t(counts ? y : 0) * ld_t;
  const bool wide = rows_wide(hidden, ld_h, width) && rows_wide(table, ld_t, width);
  float dot = 0.f;
  bool fine = true;   // (float32's planes hold no infinities: a row with one, or with NaN, has no sum)
  if (counts || sizeof(T) == 4) {
    constexpr int AHEAD = sizeof(T) == 2 ? 2 : 4;   // pieces of a lane asked for together (bfloat16 with four: registers for fewer warps, 4,096 rows 7.9 to 12 us)
    for (int c0 = lane * 8; c0 < width; c0 += 256 * AHEAD) {
      float a[AHEAD][8], b[AHEAD][8];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        const bool there = c0 + 256 * i < width;   // (else the row's first numbers, which count for nothing)
        load8(x, there ? c0 + 256 * i : 0, width, wide, a[i]);
        load8(t, there ? c0 + 256 * i : 0, width, wide, b[i]);
      }
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        if (c0 + 256 * i >= width) break;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (sizeof(T) == 4) fine = fine && fabsf(a[i][j]) < INFINITY;
          dot = fmaf(a[i][j], b[i][j], dot);
        }
      }
    }
  }
  pdl_wait();   // (the sums' kernel lets this one in behind its own wait: what was there before that call is there)
  float top = -3.4028234663852886e38f, sum = 0.f;
  for (int i0 = lane; i0 < parts; i0 += 32 * 16) {
    float2 p[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) p[j] = i0 + 32 * j < parts ? part[size_t(r) * parts + i0 + 32 * j] : make_float2(-3.4028234663852886e38f, 0.f);
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const float most = fmaxf(top, p[j].x);
      sum = sum * fast_exp2(top - most) + p[j].y * fast_exp2(p[j].x - most);
      top = most;
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float other = __shfl_xor_sync(0xffffffffu, top, o), more = __shfl_xor_sync(0xffffffffu, sum, o), most = fmaxf(top, other);
    sum = sum * fast_exp2(top - most) + more * fast_exp2(other - most);
    top = most;
  }
  dot = warp_sum(dot);
  fine = __all_sync(0xffffffffu, fine);
  if (lane == 0) {
    const float s = fine ? fmaf(top, LN2, logf(sum)) : NAN;
    log_sum[r] = s;
    const float z = softcap > 0.f ? softcap * tanhf(dot / softcap) : dot;
    const float gap = s - z;   // (never negative but by rounding)
    loss[r] = counts ? factor * (gap < 0.f ? 0.f : gap) : 0.f;
  }
}

// A matrix in planes of bfloat16 whose rows start at 16 bytes: float32 in three, bfloat16 that tensor copies cannot read in one.
template <typename T> struct Planes {
  const T* from;
  long long ld;
  int rows, width, blocks;
  bf16* to;
  long long ld_to, plane;
};

template <typename T> __device__ __forceinline__ void split_rows(const Planes<T>& p, int block) {
  const int lane = threadIdx.x & 31;
  const bool wide = rows_wide(p.from, p.ld, p.width);
  for (long long r = block * 8LL + (threadIdx.x >> 5); r < p.rows; r += p.blocks * 8LL) {
#pragma unroll 2
    for (int c = lane * 8; c < p.width; c += 256) {
      float v[8];
      load8(p.from + r * p.ld, c, p.width, wide, v);
      put_planes8<T>(p.to + r * p.ld_to + c, p.plane, v);
    }
  }
}

template <typename T> __global__ void __launch_bounds__(256) planes_kernel(const Planes<T> p) {
  pdl_launch_dependents();
  pdl_wait();
  split_rows(p, int(blockIdx.x));
}

// The rows that count (a token of the vocabulary, a weight that is not 0) side by side, their numbers in one plane or three, zeros behind them up to a
// multiple of 256 rows; `place[r]` is where row r went, -1 for none. SORTED (bfloat16, more than FEW): by their tokens (rows of one token in their order), SEGMENT of the call's rows at a time, `starts` says
// where a segment's begin: what the table's gradient adds in float for a token then stands side by side. A block looks at all rows' tokens and takes its own; a sorted row's place is the number
// of those of its segment that go before it, a comparison each (4,096 rows 1 us; segments keep it below the products' time however many rows there are). Behind these blocks: the table's planes.
constexpr int SEGMENT = 8192;
constexpr int OWN = 128;   // rows of a block at most; a segment's are whole blocks

template <typename T, bool SORTED>
__global__ void __launch_bounds__(256) gather_kernel(const T* hidden, long long ld, int rows, int width, int vocab, int own, const int32_t* targets, const float* weight,
                                                     const float* log_sum, bf16* x, long long ld_x, long long plane, int32_t* y_out, float* f_out, float* s_out,
                                                     int32_t* place, int* count, int* starts, const Planes<T> table) {
  constexpr int NONE = 0x7ffffffe, PASS = 8, AHEAD = 8;   // (PASS: rows whose places are found in one look at the segment)
  __shared__ int totals[2][8], before_of[OWN], key_of[OWN], ranks[PASS][8], keys[SORTED ? SEGMENT : 1];
  pdl_launch_dependents();
  pdl_wait();
  const int blocks = int(gridDim.x) - table.blocks;
  if (int(blockIdx.x) >= blocks) {
    split_rows(table, int(blockIdx.x) - blocks);
    return;
  }
  const int first = blockIdx.x * own, last = min(rows, first + own);
  const int begin = SORTED ? first / SEGMENT * SEGMENT : first, end = SORTED ? min(rows, begin + SEGMENT) : first;   // of the block's segment
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto key = [&](int r) {
    const int y = __ldg(targets + r);
    const float a = weight ? __ldg(weight + r) : 1.f;   // (not asked for behind the token: both are on their way together)
    return (unsigned(y) < unsigned(vocab)) & (a != 0.f) ? y : NONE;
  };
  auto scan = [&](long long from, long long to, auto&& keep) {   // how many rows count
    int counted = 0;
    for (long long r0 = from + threadIdx.x; r0 < to; r0 += 256 * AHEAD) {
      int k[AHEAD];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) k[i] = key(int(min(r0 + 256 * i, to - 1)));
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        if (r0 + 256 * i < to) {
          counted += k[i] != NONE ? 1 : 0;
          keep(int(r0 + 256 * i), k[i]);
        }
      }
    }
    return counted;
  };
  auto forget = [](int, int) {};
  if (threadIdx.x < OWN) key_of[threadIdx.x] = first + int(threadIdx.x) < last ? key(first + threadIdx.x) : NONE;
  int before = scan(0, begin, forget);
  int all = before + scan(end, rows, forget);
  if constexpr (SORTED) all += scan(begin, end, [&](int r, int k) { keys[r - begin] = k; });
  before = __reduce_add_sync(0xffffffffu, before);
  all = __reduce_add_sync(0xffffffffu, all);
  if (lane == 0) {
    totals[0][warp] = before;
    totals[1][warp] = all;
  }
  __syncthreads();
  before = all = 0;
  for (int i = 0; i < 8; ++i) {
    before += totals[0][i];
    all += totals[1][i];
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) *count = all;
  if constexpr (SORTED) {
    if (first == begin && threadIdx.x == 0) starts[first / SEGMENT] = before;
    if (int(threadIdx.x) < last - first) {   // equal ones of the block
      int equal = 0;
      for (int i = 0; i < int(threadIdx.x); ++i) equal += key_of[i] == key_of[threadIdx.x] ? 1 : 0;
      before_of[threadIdx.x] = before + equal;
    }
    for (int p = 0; p < last - first; p += PASS) {
      int mine[PASS], n[PASS];
#pragma unroll
      for (int j = 0; j < PASS; ++j) {
        mine[j] = key_of[p + j];
        n[j] = 0;
      }
#pragma unroll 4
      for (int r = threadIdx.x; r < end - begin; r += 256) {
        const int with = keys[r] + (begin + r >= first ? 1 : 0);   // (of the block's own, equal ones are counted above)
#pragma unroll
        for (int j = 0; j < PASS; ++j) n[j] += with <= mine[j] ? 1 : 0;
      }
#pragma unroll
      for (int j = 0; j < PASS; ++j) {
        n[j] = __reduce_add_sync(0xffffffffu, n[j]);
        if (lane == 0) ranks[j][warp] = n[j];
      }
      __syncthreads();
      if (int(threadIdx.x) < min(PASS, last - first - p)) {
        int rank = 0;
        for (int i = 0; i < 8; ++i) rank += ranks[threadIdx.x][i];
        before_of[p + threadIdx.x] += rank;
      }
      __syncthreads();
    }
  } else {
    if (int(threadIdx.x) < last - first) {
      int counted = before;
      for (int i = 0; i < int(threadIdx.x); ++i) counted += key_of[i] != NONE ? 1 : 0;
      before_of[threadIdx.x] = counted;
    }
    __syncthreads();
  }
  const bool wide = rows_wide(hidden, ld, width);
  auto copy = [&](int to, const T* from) {   // (null: zeros)
    for (int c = lane * 8; c < width; c += 256) {
      float v[8] = {};
      if (from) load8(from, c, width, wide, v);
      put_planes8<T>(x + size_t(to) * ld_x + c, plane, v);
    }
  };
  if (int(threadIdx.x) < last - first) {
    const int r = first + threadIdx.x, at = before_of[threadIdx.x];
    const bool c = key_of[threadIdx.x] != NONE;
    place[r] = c ? at : -1;
    if (c) {
      y_out[at] = targets[r];
      f_out[at] = weight ? weight[r] : 1.f;
      s_out[at] = log_sum[r];
    }
  }
  for (int i = warp; i < last - first; i += 8)
    if (key_of[i] != NONE) copy(before_of[i], hidden + size_t(first + i) * ld);
  const int filled = (all + 255) / 256 * 256;
  for (int at = all + blockIdx.x + warp * blocks; at < filled; at += 8 * blocks) copy(at, static_cast<const T*>(nullptr));
}

// bfloat16, more than FEW rows: what rounding left of dz at the tokens' own rows, times the hidden rows, summed in float by token, for the piece's tokens. A CTA takes WINDOW of the sorted rows and 128
// columns, a warp 32 of the rows, and leaves a token's sum at the place of the first of its rows in the window; one that lies in several warps' is joined in shared memory. A token that stands
// everywhere is many CTAs' work, and TABLE adds its sums, in order. Other CTAs look up where each token's rows begin and end, a warp 32 tokens. (4,096 rows, a tenth of them one token: 11 us; TABLE
// adding the rows themselves took 100 us longer, a CTA for 128 tokens 40. Sums of 64 rows: TABLE, where a lane adds a token's, 470 in place of 344 for 65,536 rows of 64.)
struct Rests {
  const bf16* x;
  long long ld_x;
  const int32_t* targets;
  const float* rest;
  const int *count, *starts;
  int first, n, width, slices, segments;   // of the piece: its first token, tokens; of the columns
  long long blocks;                        // of sums; those that look up stand behind them
  float* sums;
  long long ld_sums;
  int2* runs;
  int run_tokens;
};

constexpr int REST_WARPS = WINDOW / 32;

__global__ void __launch_bounds__(REST_WARPS * 32) rests_kernel(const Rests w) {
  constexpr int SLICE = 128;
  __shared__ int head[REST_WARPS], tail[REST_WARPS], tail_at[REST_WARPS];   // a sum that an earlier warp began ends here; one goes on from here; its place, -1: an earlier warp's
  __shared__ alignas(16) float heads[REST_WARPS][SLICE], tails[REST_WARPS][SLICE];
  pdl_launch_dependents();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, k = *w.count;
  if (blockIdx.x >= w.blocks) {
    // ---- where the rows of 32 tokens begin: the warp looks for the first and the last, and counts between them
    const long long groups = w.run_tokens / 32, job = (blockIdx.x - w.blocks) * REST_WARPS + warp;
    const int segment = int(job / groups), first = w.first + int(job % groups) * 32;
    if (segment >= w.segments) return;
    int from = __ldg(w.starts + segment), end = segment + 1 < w.segments ? __ldg(w.starts + segment + 1) : k, to = from, to_end = end;
    auto narrow = [&](int& a, int& b, int token) {   // a .. b holds the first place whose token is `token` or a later one
      const int step = (b - a + 31) / 32, at = a + lane * step;
      const int n = __popc(__ballot_sync(0xffffffffu, at < b && __ldg(w.targets + at) < token));
      b = n == 0 ? a : min(b, a + n * step);
      a += n == 0 ? 0 : (n - 1) * step + 1;
    };
    while (from < end || to < to_end) {
      narrow(from, end, first);
      narrow(to, to_end, first + 32);
    }
    int begin = from;   // of the lane's token
    if (to - from <= 32) {
      const int token = from + lane < to ? __ldg(w.targets + from + lane) - first : 32;
      for (int j = 0; j < to - from; ++j) begin += __shfl_sync(0xffffffffu, token, j) < lane ? 1 : 0;
    } else {
      for (int last = to; begin < last;) {
        const int middle = begin + (last - begin) / 2;
        if (__ldg(w.targets + middle) < first + lane) begin = middle + 1;
        else last = middle;
      }
    }
    int next = __shfl_down_sync(0xffffffffu, begin, 1);
    if (lane == 31) next = to;
    w.runs[static_cast<long long>(segment) * w.run_tokens + (first - w.first) + lane] = make_int2(begin, next);
    return;
  }
  const int window = int(blockIdx.x / w.slices) * WINDOW, slice = int(blockIdx.x % w.slices) * SLICE, col = slice + lane * 4;
  const int from = window + warp * 32, to = min(k, from + 32), window_end = min(k, window + WINDOW);
  const bool there = from + lane < to;
  const int token = there ? __ldg(w.targets + from + lane) : -1;
  const int in_front = from < to && warp > 0 ? __ldg(w.targets + from - 1) : -1, behind = to < window_end ? __ldg(w.targets + to) : -1;
  unsigned begins = 0;       // bits of the rows that a segment begins with, then of those that a sum begins with
  bool behind_begins = false;
  for (int s = 0; s < w.segments; s += 32) {
    const int start = s + lane < w.segments ? __ldg(w.starts + s + lane) : -1;
    begins |= __reduce_or_sync(0xffffffffu, start >= from && start < to ? 1u << (start - from) : 0u);
    behind_begins |= __any_sync(0xffffffffu, start == to) != 0;
  }
  if (!__syncthreads_or(there && token >= w.first && token - w.first < w.n)) return;   // (tokens of other pieces: nobody reads their sums now)
  const bool wide = col < w.width;   // (rows of whole eights)
  float sum[4] = {};
  int at = -1;          // the place of what is summed, -1: an earlier warp's
  bool ended = false;   // that one ends in this warp
  auto keep = [&] {
    if (at < 0) {
      ended = true;
      *reinterpret_cast<float4*>(&heads[warp][lane * 4]) = make_float4(sum[0], sum[1], sum[2], sum[3]);
    } else if (wide) {
      *reinterpret_cast<float4*>(w.sums + at * w.ld_sums + col) = make_float4(sum[0], sum[1], sum[2], sum[3]);
    }
    sum[0] = sum[1] = sum[2] = sum[3] = 0.f;
  };
  bool goes_on = false;
  if (from < to) {
    const float rest = there ? __ldg(w.rest + from + lane) : 0.f;
    uint2 x[32];
#pragma unroll
    for (int j = 0; j < 32; ++j) x[j] = wide && from + j < to ? __ldg(reinterpret_cast<const uint2*>(w.x + (from + j) * w.ld_x + col)) : make_uint2(0, 0);
    const int shifted = __shfl_up_sync(0xffffffffu, token, 1), last = __shfl_sync(0xffffffffu, token, 31);
    begins |= __ballot_sync(0xffffffffu, there && token != (lane == 0 ? in_front : shifted));
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      const float by = __shfl_sync(0xffffffffu, rest, j);
      if (begins >> j & 1u) {
        if (j > 0) keep();
        at = from + j;
      }
      sum[0] = fmaf(by, __uint_as_float(x[j].x << 16), sum[0]);
      sum[1] = fmaf(by, __uint_as_float(x[j].x & 0xffff0000u), sum[1]);
      sum[2] = fmaf(by, __uint_as_float(x[j].y << 16), sum[2]);
      sum[3] = fmaf(by, __uint_as_float(x[j].y & 0xffff0000u), sum[3]);
    }
    goes_on = to < window_end && !behind_begins && behind == last;
    if (goes_on) *reinterpret_cast<float4*>(&tails[warp][lane * 4]) = make_float4(sum[0], sum[1], sum[2], sum[3]);
    else keep();
  }
  if (lane == 0) {
    head[warp] = ended;
    tail[warp] = goes_on;
    tail_at[warp] = at;
  }
  __syncthreads();
  const int c = threadIdx.x;   // a thread a column
  if (c >= SLICE || slice + c >= w.width) return;
  float all = 0.f;
  int place = -1;
  for (int i = 0; i < REST_WARPS; ++i) {
    if (head[i]) w.sums[place * w.ld_sums + slice + c] = all + heads[i][c];
    if (tail[i]) {
      all = tail_at[i] >= 0 ? tails[i][c] : all + tails[i][c];
      place = tail_at[i] >= 0 ? tail_at[i] : place;
    }
  }
}

// The hidden rows' gradient: shares of a gathered row added in one order, and what rounding left of dz at its token (`rest`, null in float32) times the token's row of the
// table; zeros for the rows that were left out.
template <typename T>
__global__ void __launch_bounds__(256) join_kernel(const float* shares, int splits, long long plane, long long ld, const int32_t* place, const float* rest, const int32_t* targets,
                                                   const T* table, long long ld_t, T* out, long long ld_o, int rows, int width) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, pieces = (width + 127) / 128;   // a warp a row's 128 numbers: the shares of a few rows are one chain of loads otherwise
  const bool wide = rows_wide(out, ld_o, width);
  for (long long i = blockIdx.x * 8LL + (threadIdx.x >> 5); i < static_cast<long long>(rows) * pieces; i += gridDim.x * 8LL) {
    const long long r = i / pieces;
    const int c = int(i % pieces) * 128 + lane * 4, at = place[r];
    if (c >= width) continue;
    T* o = out + r * ld_o;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    if (at >= 0) {
      const float* s = shares + at * ld + c;   // (rows of whole eights)
#pragma unroll 8
      for (int j = 0; j < splits; ++j) {
        const float4 v = __ldg(reinterpret_cast<const float4*>(s + j * plane));
        sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
      }
      if (sizeof(T) == 2) {
        const T* t = table + targets[at] * ld_t + c;
        const float left = rest[at];
        sum.x = fmaf(left, to_float(t[0]), sum.x);
        if (c + 1 < width) sum.y = fmaf(left, to_float(t[1]), sum.y);
        if (c + 2 < width) sum.z = fmaf(left, to_float(t[2]), sum.z);
        if (c + 3 < width) sum.w = fmaf(left, to_float(t[3]), sum.w);
      }
    }
    if (wide) {
      if constexpr (sizeof(T) == 2) *reinterpret_cast<uint2*>(o + c) = make_uint2(pack_bf16(sum.x, sum.y), pack_bf16(sum.z, sum.w));
      else *reinterpret_cast<float4*>(o + c) = sum;
    } else {
      const float v[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (c + j < width) o[c + j] = from_float<T>(v[j]);
    }
  }
}

// ---- host side ------------------------------------------------------------------------------

inline long long up(long long x, long long to) { return (x + to - 1) / to * to; }

// A matrix [rows, width] as tensor copies read it.
struct Operand {
  const void* at;
  long long ld, plane;
  int planes;
};

bool encode(CUtensorMap* map, CUtensorMapDataType type, int size, const void* at, long long inner, long long outer, long long planes, long long ld, long long plane, int box_inner,
            int box_outer, CUtensorMapSwizzle swizzle = CU_TENSOR_MAP_SWIZZLE_128B) {
  const r2::EncodeTiledFn fn = r2::encode_fn();
  cuuint64_t dims[3] = {cuuint64_t(inner), cuuint64_t(outer), cuuint64_t(planes)};
  cuuint64_t strides[2] = {cuuint64_t(ld) * size, cuuint64_t(planes > 1 ? plane : ld) * size};
  cuuint32_t box[3] = {cuuint32_t(box_inner), cuuint32_t(box_outer), 1}, steps[3] = {1, 1, 1};
  return fn != nullptr && fn(map, type, 3, const_cast<void*>(at), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Boxes of 64 numbers and box_outer rows, as the products load them.
bool make_map(CUtensorMap* map, const Operand& o, long long inner, long long outer, int box_outer) {
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, o.at, inner, outer, o.planes, o.ld, o.plane, BK, box_outer);
}

// Boxes of 128 bytes and 32 rows, as results are stored.
template <typename T> bool make_out_map(CUtensorMap* map, const void* at, long long inner, long long outer, long long planes, long long ld, long long plane) {
  return encode(map, sizeof(T) == 2 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, int(sizeof(T)), at, inner, outer, planes, ld, plane,
                128 / int(sizeof(T)), 32);
}

// How many CTA pairs the current device holds at once.
int resident_pairs() {
  static std::atomic<int> cached[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 1;
  if (dev < 64 && cached[dev].load() > 0) return cached[dev].load();
  auto kernel = product_kernel<LOGSUM, false, bf16, false, 0>;
  cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(SMEM));
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(2, 1, 1);
  config.blockDim = dim3(THREADS);
  config.dynamicSmemBytes = SMEM;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  config.attrs = attr;
  config.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, kernel, &config) != cudaSuccess || n < 1) {
    cudaGetLastError();
    n = 64;
  }
  if (dev < 64) cached[dev].store(n);
  return n;
}

template <typename... P, typename... Args> int launch_pairs(void (*kernel)(P...), std::atomic<bool> (&done)[64], long long pairs, cudaStream_t stream, const Args&... args) {
  const int status = allow_smem(kernel, SMEM, done);
  if (status != R2_OK) return status;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(2 * unsigned(pairs), 1, 1);
  config.blockDim = dim3(THREADS);
  config.dynamicSmemBytes = SMEM;
  config.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attr;
  config.numAttrs = g_r2_pdl ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&config, kernel, args...);
  return e != cudaSuccess ? int(e) : launch_status();
}

template <int MODE, bool CAPPED, typename T, bool PLANES, int CHUNKED>
int launch(const CUtensorMap& ma, const CUtensorMap& mb, const CUtensorMap& mo, const Work& w, long long units, cudaStream_t stream) {
  static std::atomic<bool> done[64];
  const int pairs = resident_pairs();
  return launch_pairs(product_kernel<MODE, CAPPED, T, PLANES, CHUNKED>, done, units < pairs ? units : pairs, stream, ma, mb, mo, w);
}

template <int MODE, typename T, bool PLANES, int CHUNKED = PLANES ? PLANES_CHUNK : 0>
int launch(const CUtensorMap& ma, const CUtensorMap& mb, const CUtensorMap& mo, const Work& w, long long units, bool capped, cudaStream_t stream) {
  if constexpr (MODE == LOGSUM || MODE == FACTORS) {
    if (capped) return launch<MODE, true, T, PLANES, CHUNKED>(ma, mb, mo, w, units, stream);
  }
  return launch<MODE, false, T, PLANES, CHUNKED>(ma, mb, mo, w, units, stream);
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

int few_ctas(long long vocab) {
  const long long tiles = (vocab + 127) / 128;
  return int(tiles < n_sms() ? tiles : n_sms());
}

template <int MODE, bool CAPPED, bool F32, bool SUMS>
int launch_few(const CUtensorMap& mt, const CUtensorMap& mx, FewWork f, cudaStream_t stream) {
  constexpr uint32_t most = 227 * 1024;
  auto kernel = few_kernel<MODE, CAPPED, F32, SUMS>;
  static std::atomic<bool> done[64];
  const int status = allow_smem(kernel, most, done);
  if (status != R2_OK) return status;
  // float32: as many stages of planes as there are groups at least, and loads that go evenly into the groups, so that a group comes back to the barriers it has waited
  // for (one that others have waited for could be two phases behind, which a wait by parity takes for done).
  constexpr int LEAST = F32 ? GROUPS : 2;
  static_assert(F32_STAGES >= GROUPS && F32_STAGES <= FEW_STAGES && few_smem<F32>(FEW, LEAST, F32 ? GROUPS : 0) <= most);   // (the loops below leave so many, whatever the rows)
  f.stages = F32 ? F32_STAGES : FEW_STAGES;
  f.loads = F32 ? GROUPS : 0;
  while (f.stages > LEAST && few_smem<F32>(f.columns, f.stages, f.loads) > most) --f.stages;
  while (F32 && f.loads + GROUPS <= FEW_STAGES && few_smem<F32>(f.columns, f.stages, f.loads + GROUPS) <= most) f.loads += GROUPS;
  r2_launch(kernel, dim3(few_ctas(f.n)), dim3(few_threads(F32)), size_t(few_smem<F32>(f.columns, f.stages, f.loads)), stream, mt, mx, f);
  return launch_status();
}

template <int MODE, bool F32> int launch_few(const CUtensorMap& mt, const CUtensorMap& mx, const FewWork& f, bool capped, cudaStream_t stream) {
  if constexpr (!F32) {
    if (f.k > FEW_CHUNK) return capped ? launch_few<MODE, true, F32, true>(mt, mx, f, stream) : launch_few<MODE, false, F32, true>(mt, mx, f, stream);
  }
  return capped ? launch_few<MODE, true, F32, F32>(mt, mx, f, stream) : launch_few<MODE, false, F32, F32>(mt, mx, f, stream);
}

// Both operands' maps for few rows: the table [vocab, width] as it lies, the rows in planes.
template <typename T> bool make_few_maps(CUtensorMap* mt, CUtensorMap* mx, const void* table, long long ld_t, long long vocab, const Operand& x, long long width, long long rows,
                                         int columns) {
  constexpr bool F32 = sizeof(T) == 4;
  return encode(mt, F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, int(sizeof(T)), table, width, vocab, 1, ld_t, 0, 128 / int(sizeof(T)), 128) &&
         encode(mx, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, x.at, width, rows, x.planes, x.ld, x.plane, F32 ? 32 : 64, columns,
                F32 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B);
}

int row_blocks(long long rows) { return int(rows < 8 * 4736 ? (rows + 7) / 8 : 4736); }

// What a call's scratch holds, in bytes from its start.
// Of dz at a time: pieces bound what a call takes, and a call whose dz is smaller has one. (4,096 rows at GPT-2's table with 128, 256, 512 MB and 1 GB: 931, 855, 833 and 833 us; 2,047 at a table of 128,001 x 1,600 2,487, 2,441, 2,418 and 2,418. Pieces that L2
// would hold make for more launches and rounds that are not full.)
constexpr long long FACTOR_BYTES = 512ll << 20;

struct Layout {
  int planes;                       // bfloat16 planes of an operand
  bool copied;                      // the table's planes are in the scratch; else it is read where it lies
  long long rows_up, width_up;      // rows to a multiple of 256, numbers to one of 8
  int pieces, splits;
  long long piece;                  // tokens at a time, a multiple of 256
  long long parts;
  long long table, hidden, part, factors, shares, targets, factor, sums, rest, rests, runs, place, starts, count, total;
};

bool copies_read(const void* at, long long ld, long long rows, long long width, int size = 2) {
  return reinterpret_cast<uintptr_t>(at) % 16 == 0 && (rows <= 1 || (ld * size % 16 == 0 && ld >= width));
}

// Up to FEW rows read a table as it lies, in either type, where tensor copies can. (The hidden rows' gradient reads float32's planes all the same.)
bool few_rows(int dtype, const void* table, long long ld_t, long long rows, long long width, long long vocab) {
  return rows <= FEW && (dtype == R2_BF16 || copies_read(table, ld_t, vocab, width, 4));
}

Layout layout(int dtype, const void* table, long long ld_t, long long rows, long long width, long long vocab, bool few, bool gradient, bool d_hidden) {
  Layout l = {};
  l.planes = dtype == R2_F32 ? 3 : 1;
  l.rows_up = up(rows, 256);
  l.width_up = up(width, 8);
  long long at = 0;
  auto take = [&](long long bytes) {
    const long long begin = at;
    at += up(bytes, 256);
    return begin;
  };
  l.copied = dtype == R2_BF16 ? !copies_read(table, ld_t, vocab, width) : !few || d_hidden;
  l.table = take(l.copied ? l.planes * vocab * l.width_up * 2 : 0);
  l.hidden = take(l.planes * l.rows_up * l.width_up * 2);
  if (!gradient) {
    l.parts = few ? few_ctas(vocab) * 4 : up(vocab, BN) / BN * 2;
    l.part = take(l.parts * rows * 8);
  } else {
    const int pairs = resident_pairs(), terms = l.planes * (l.planes + 1) / 2;
    const long long row_tiles = l.rows_up / 256, width_tiles = up(width, BN) / BN, tiles = row_tiles * width_tiles, all = up(vocab, BN) / BN;
    // tokens at a time: as few rounds of the pairs as can be in all pieces' FACTORS and TABLE (a piece of as many tiles as there are pairs leaves none of them idle)
    long long most = FACTOR_BYTES / (l.rows_up * 2 * l.planes) / BN, piece = 1;
    most = most < 1 ? 1 : most > all ? all : most;
    auto rounds = [&](long long n) {   // of a piece of n tiles, in steps of k; and its launches
      return double((n * row_tiles + pairs - 1) / pairs) * (up(width, BK) / BK * terms + 2) + double((n * width_tiles + pairs - 1) / pairs) * (l.rows_up / BK * terms + 2) + 40;
    };
    double least = -1;
    for (long long p = most; p >= 1 && p >= most / 2; --p) {
      const double cost = double(all / p) * rounds(p) + (all % p ? rounds(all % p) : 0);
      if (least < 0 || cost < least) {
        least = cost;
        piece = p;
      }
    }
    l.piece = piece * BN;
    l.pieces = int((all + piece - 1) / piece);
    const int n_kb = int((l.piece + BK - 1) / BK);
    // shares of k, of no fewer than eight steps: more of them fill the last round of pairs, and each is written for every piece and read once more (a tile's
    // 256 KB take a seventh of a step's time, a step of 64 being 0.29 us on a pair)
    double best = -1;
    for (int s = 1; s <= 64 && (s == 1 || n_kb * terms / s >= 8); ++s) {
      const int per = (n_kb + s - 1) / s;
      const double steps = per * terms + 8;
      const double cost = l.pieces * double((tiles * s + pairs - 1) / pairs) * steps + double(s) * tiles * 0.14 * (l.pieces + 1);
      if (best < 0 || cost < best) {
        best = cost;
        l.splits = (n_kb + per - 1) / per;
      }
    }
    l.factors = take(l.planes * l.rows_up * l.piece * 2);
    l.shares = take(d_hidden ? l.splits * l.rows_up * l.width_up * 4 : 0);
    l.targets = take(l.rows_up * 4);
    l.factor = take(l.rows_up * 4);
    l.sums = take(l.rows_up * 4);
    l.rest = take(l.rows_up * 4);
    const long long segments = up(rows, SEGMENT) / SEGMENT;
    l.rests = take(dtype == R2_BF16 && !few ? l.rows_up * l.width_up * 4 : 0);
    l.runs = take(dtype == R2_BF16 && !few ? segments * l.piece * 8 : 0);
    l.place = take(rows * 4);
    l.starts = take(dtype == R2_BF16 && !few ? segments * 4 : 0);
    l.count = take(4);
  }
  l.total = at;
  return l;
}

// The matrix itself where tensor copies can read it, else where its planes will be: `p` says how they are made.
template <typename T> Operand operand(const void* at, long long ld, long long rows, long long width, const Layout& l, char* space, Planes<T>& p) {
  if (sizeof(T) == 2 && copies_read(at, ld, rows, width)) return {at, rows <= 1 ? l.width_up : ld, 0, 1};
  p = {static_cast<const T*>(at), ld, int(rows), int(width), row_blocks(rows), reinterpret_cast<bf16*>(space), l.width_up, rows * l.width_up};
  return {space, l.width_up, rows * l.width_up, l.planes};
}
template <typename T> Operand operand(const void* at, long long ld, long long rows, long long width, const Layout& l, char* space, cudaStream_t stream) {
  Planes<T> p = {};
  const Operand o = operand<T>(at, ld, rows, width, l, space, p);
  if (p.blocks > 0) r2_launch(planes_kernel<T>, dim3(p.blocks), dim3(256), size_t(0), stream, p);
  return o;
}

void set_cap(Work& w, float softcap) {
  if (softcap > 0.f) {
    w.cap = 1.f / softcap;
    w.cap_out = softcap * LOG2E;
  }
}

template <typename T>
int loss_of(const void* hidden, long long ld_h, const void* table, long long ld_t, int rows, int width, int vocab, const int32_t* targets, const float* weight,
            float softcap, bool alike, float* loss, float* log_sum, char* space, int* error, cudaStream_t stream) {
  constexpr int dtype = sizeof(T) == 4 ? R2_F32 : R2_BF16;
  const bool few = !alike && few_rows(dtype, table, ld_t, rows, width, vocab);
  const Layout l = layout(dtype, table, ld_t, rows, width, vocab, few, false, false);
  const Operand x = operand<T>(hidden, ld_h, rows, width, l, space + l.hidden, stream);
  Work w = {};
  w.part = reinterpret_cast<float2*>(space + l.part);
  w.parts = int(l.parts);
  w.error_flag = error;
  set_cap(w, softcap);
  CUtensorMap ma, mb;
  int status;
  if (few) {
    const void* at = table;
    long long ld = vocab > 1 ? ld_t : l.width_up;
    if (sizeof(T) == 2) {
      const Operand t = operand<T>(table, ld_t, vocab, width, l, space + l.table, stream);
      at = t.at;
      ld = t.ld;
    }
    FewWork f = {};
    f.rows = rows;
    f.columns = (rows + 15) / 16 * 16;
    f.n = vocab;
    f.k = width;
    f.w = w;
    if (!make_few_maps<T>(&mb, &ma, at, ld, vocab, x, width, rows, f.columns)) return R2_BAD_ALIGN;
    status = launch_few<LOGSUM, sizeof(T) == 4>(mb, ma, f, softcap > 0.f, stream);
  } else {
    const Operand t = operand<T>(table, ld_t, vocab, width, l, space + l.table, stream);
    if (!make_map(&ma, x, width, rows, BM) || !make_map(&mb, t, width, vocab, HALF)) return R2_BAD_ALIGN;
    w.m = rows;
    w.n = vocab;
    w.k = width;
    const long long tiles = (l.rows_up / 256) * (up(vocab, BN) / BN);
    if (sizeof(T) == 2 && width > LONG_STEPS * BK) status = launch<LOGSUM, bf16, false, LONG_CHUNK>(ma, mb, ma, w, tiles, softcap > 0.f, stream);
    else status = launch<LOGSUM, bf16, sizeof(T) == 4>(ma, mb, ma, w, tiles, softcap > 0.f, stream);
  }
  if (status != R2_OK) return status;
  const T *h = static_cast<const T*>(hidden), *tab = static_cast<const T*>(table);
  r2_launch(finish_kernel<T>, dim3((rows + 7) / 8), dim3(256), size_t(0), stream, static_cast<const float2*>(w.part), int(l.parts), h, ld_h, tab, ld_t, targets, weight, rows, width, vocab, softcap, loss, log_sum);
  return launch_status();
}

template <typename T>
int gradient_of(const void* hidden, long long ld_h, const void* table, long long ld_t, int rows, int width, int vocab, const int32_t* targets, const float* weight,
                const float* log_sum, float softcap, void* d_hidden, long long ld_dh, void* d_table, long long ld_dt, char* space, int* error, cudaStream_t stream) {
  constexpr int dtype = sizeof(T) == 4 ? R2_F32 : R2_BF16;
  const bool few = few_rows(dtype, table, ld_t, rows, width, vocab);
  const Layout l = layout(dtype, table, ld_t, rows, width, vocab, few, true, d_hidden != nullptr);
  Operand t = {};   // (few float32 rows read the table as it is for their factors)
  Planes<T> planes = {};
  if (sizeof(T) == 2 || l.copied) t = operand<T>(table, ld_t, vocab, width, l, space + l.table, planes);
  bf16* gathered = reinterpret_cast<bf16*>(space + l.hidden);
  const Operand x = {gathered, l.width_up, l.rows_up * l.width_up, l.planes};
  int* count = reinterpret_cast<int*>(space + l.count);
  int32_t* place = reinterpret_cast<int32_t*>(space + l.place);
  int* starts = reinterpret_cast<int*>(space + l.starts);
  int own = (rows + 591) / 592;
  if (sizeof(T) == 4 || few || rows <= SEGMENT) {
    own = own > 32 ? 32 : own;
  } else {
    own = own > OWN ? OWN : own;
    while (SEGMENT % own != 0) ++own;
  }
  constexpr bool BF16 = sizeof(T) == 2;
  r2_launch(BF16 && !few ? gather_kernel<T, BF16> : gather_kernel<T, false>, dim3((rows + own - 1) / own + planes.blocks), dim3(256), size_t(0), stream,
      static_cast<const T*>(hidden), ld_h, rows, width, vocab, own, targets, weight, log_sum, gathered, x.ld, x.plane, reinterpret_cast<int32_t*>(space + l.targets),
      reinterpret_cast<float*>(space + l.factor), reinterpret_cast<float*>(space + l.sums), place, count, starts, planes);
  Work w = {};
  w.m = rows;
  w.count = count;
  w.targets = reinterpret_cast<int32_t*>(space + l.targets);
  w.factor = reinterpret_cast<float*>(space + l.factor);
  w.log_sum = reinterpret_cast<float*>(space + l.sums);
  w.rest = reinterpret_cast<float*>(space + l.rest);
  w.error_flag = error;
  set_cap(w, softcap);
  const Operand dz = {space + l.factors, l.piece, l.rows_up * l.piece, l.planes};
  float* shares = reinterpret_cast<float*>(space + l.shares);
  const long long share_plane = l.rows_up * l.width_up;
  CUtensorMap ma, mb, mo;   // of the factors
  int status = launch_status();
  const long long row_tiles = l.rows_up / 256, width_tiles = up(width, BN) / BN;
  for (long long first = 0; first < vocab && status == R2_OK; first += l.piece) {
    const int n = int(vocab - first < l.piece ? vocab - first : l.piece);
    const Operand part = {static_cast<const bf16*>(t.at) + first * t.ld, t.ld, t.plane, t.planes};
    w.first = int(first);
    w.n = n;
    w.k = width;
    if (few) {
      FewWork f = {};
      f.rows = rows;
      f.columns = (rows + 15) / 16 * 16;
      f.n = n;
      f.k = width;
      f.w = w;
      f.dz = reinterpret_cast<bf16*>(space + l.factors);
      f.dz_plane = dz.plane;
      f.ld = l.piece;
      const void* at = sizeof(T) == 2 ? part.at : static_cast<const T*>(table) + first * ld_t;
      const long long ld = sizeof(T) == 2 ? part.ld : n > 1 ? ld_t : l.width_up;
      if (!make_few_maps<T>(&mb, &ma, at, ld, n, x, width, l.rows_up, f.columns)) return R2_BAD_ALIGN;
      status = launch_few<FACTORS, sizeof(T) == 4>(mb, ma, f, softcap > 0.f, stream);
    } else {
      if (!make_map(&ma, x, width, l.rows_up, BM) || !make_map(&mb, part, width, n, HALF) ||
          !make_out_map<bf16>(&mo, dz.at, l.piece, l.rows_up, l.planes, l.piece, dz.plane))
        return R2_BAD_ALIGN;
      const long long tiles = row_tiles * (up(n, BN) / BN);
      if (BF16 && width > FACTORS_CHUNK * BK) status = launch<FACTORS, bf16, false, FACTORS_CHUNK>(ma, mb, mo, w, tiles, softcap > 0.f, stream);
      else status = launch<FACTORS, bf16, sizeof(T) == 4>(ma, mb, mo, w, tiles, softcap > 0.f, stream);
    }
    if (status != R2_OK) break;
    Both b = {};
    long long rows_units = 0, table_units = 0;
    if (d_hidden) {
      Work& d = b.rows = w;
      d.n = width;
      d.k = n;
      d.per_split = ((n + BK - 1) / BK + l.splits - 1) / l.splits;   // (the last piece is shorter)
      d.splits = l.splits;
      d.add = first > 0;
      if (!make_map(&b.rows_a, dz, n, l.rows_up, BM) || !make_map(&b.rows_b, part, width, n, BK) ||
          !make_out_map<float>(&b.rows_out, shares, width, l.rows_up, l.splits, l.width_up, share_plane))
        return R2_BAD_ALIGN;
      rows_units = row_tiles * width_tiles * d.splits;
    }
    if (d_table) {
      Work& d = b.table = w;
      d.x = gathered;
      d.ld_x = x.ld;
      if (BF16 && !few) {
        const int segments = int(up(rows, SEGMENT) / SEGMENT);
        const long long slices = up(width, 128) / 128, sums = up(rows, WINDOW) / WINDOW * slices;
        const Rests rests = {gathered, x.ld, w.targets, w.rest, count, starts, int(first), n, width, int(slices), segments, sums, reinterpret_cast<float*>(space + l.rests), l.width_up,
                             reinterpret_cast<int2*>(space + l.runs), int(up(n, 32))};
        const long long blocks = sums + (segments * (rests.run_tokens / 32ll) + REST_WARPS - 1) / REST_WARPS;
        if (blocks >= 1ll << 31) return R2_UNSUPPORTED;
        r2_launch(rests_kernel, dim3(unsigned(blocks)), dim3(REST_WARPS * 32), size_t(0), stream, rests);
        d.runs = rests.runs;
        d.sums = rests.sums;
        d.ld_sums = rests.ld_sums;
        d.segments = segments;
        d.run_tokens = rests.run_tokens;
      }
      d.m = n;
      d.n = width;
      T* out = static_cast<T*>(d_table) + first * ld_dt;
      if (!make_map(&b.table_a, dz, n, l.rows_up, BK) || !make_map(&b.table_b, x, width, l.rows_up, BK)) return R2_BAD_ALIGN;
      if (reinterpret_cast<uintptr_t>(out) % 16 == 0 && ld_dt * sizeof(T) % 16 == 0 && width * sizeof(T) % 16 == 0) {   // (a copy writes whole 16 bytes, beyond a row's end, too)
        if (!make_out_map<T>(&b.table_out, out, width, n, 1, ld_dt, 0)) return R2_BAD_ALIGN;
      } else {
        b.table_out = b.table_a;
        d.out = out;
        d.ld = ld_dt;
      }
      table_units = up(n, 256) / 256 * width_tiles;
    }
    constexpr bool F32 = sizeof(T) == 4;
    if (rows_units > 0 && table_units > 0 && rows_units + table_units <= resident_pairs()) {
      static std::atomic<bool> done[64], done_few[64];
      constexpr int CHUNKED = F32 ? PLANES_CHUNK : 0;
      b.rows_pairs = int(rows_units);
      status = few && !F32 ? launch_pairs(both_kernel<F32 ? TABLE : TABLE_FEW, T, F32, CHUNKED>, done_few, rows_units + table_units, stream, b)
                           : launch_pairs(both_kernel<TABLE, T, F32, CHUNKED>, done, rows_units + table_units, stream, b);
      continue;
    }
    if constexpr (F32) {
      if (rows_units > 0) status = launch<ROWS, float, true>(b.rows_a, b.rows_b, b.rows_out, b.rows, rows_units, false, stream);
      if (status == R2_OK && table_units > 0) status = launch<TABLE, T, true>(b.table_a, b.table_b, b.table_out, b.table, table_units, false, stream);
    } else {
      if (rows_units > 0)
        status = b.rows.per_split > GRADIENT_CHUNK ? launch<ROWS, float, false, GRADIENT_CHUNK>(b.rows_a, b.rows_b, b.rows_out, b.rows, rows_units, false, stream)
                                                   : launch<ROWS, float, false>(b.rows_a, b.rows_b, b.rows_out, b.rows, rows_units, false, stream);
      if (status == R2_OK && table_units > 0)
        status = few                         ? launch<TABLE_FEW, T, false>(b.table_a, b.table_b, b.table_out, b.table, table_units, false, stream)
                 : rows > GRADIENT_CHUNK * BK ? launch<TABLE, T, false, GRADIENT_CHUNK>(b.table_a, b.table_b, b.table_out, b.table, table_units, false, stream)
                                             : launch<TABLE, T, false>(b.table_a, b.table_b, b.table_out, b.table, table_units, false, stream);
    }
  }
  if (status == R2_OK && d_hidden) {
    r2_launch(join_kernel<T>, dim3(row_blocks(static_cast<long long>(rows) * ((width + 127) / 128))), dim3(256), size_t(0), stream, static_cast<const float*>(shares), l.splits, share_plane, l.width_up,
              static_cast<const int32_t*>(place), static_cast<const float*>(w.rest), w.targets, static_cast<const T*>(table), ld_t, static_cast<T*>(d_hidden), ld_dh, rows, width);
    status = launch_status();
  }
  return status;
}

constexpr int MOST = 1 << 30;   // rows, numbers of a row, tokens: indexes of tiles stay in 32 bits

}  // namespace

// Bytes of scratch for a call: of a loss (`choice`: `alike`), or (`gradient`) of gradients, of the hidden rows' too (`choice`) or of the table's alone.
extern "C" long long r2_token_loss_space(int dtype, const void* table, long long ld_t, int rows, int width, int vocab, int gradient, int choice) {
  const bool few = (gradient || !choice) && few_rows(dtype, table, ld_t, rows, width, vocab);
  return layout(dtype, table, ld_t, rows, width, vocab, few, gradient != 0, gradient && choice).total;
}

// `space`: 256-byte aligned, r2_token_loss_space bytes. `alike`: a row's results do not depend on how many rows there are (few ones go through the many's kernel).
extern "C" int r2_token_loss(int dtype, const void* hidden, long long ld_h, const void* table, long long ld_t, int rows, int width, int vocab,
                             const int32_t* targets, const float* weight, float softcap, int alike, float* loss, float* log_sum, void* space, int* error, cudaStream_t stream) {
  if (rows < 1 || width < 1 || vocab < 1) return R2_BAD_SHAPE;
  if (rows > MOST || width > MOST || vocab > MOST) return R2_UNSUPPORTED;
  if (dtype == R2_F32) return loss_of<float>(hidden, ld_h, table, ld_t, rows, width, vocab, targets, weight, softcap, alike != 0, loss, log_sum, (char*)space, error, stream);
  if (dtype == R2_BF16) return loss_of<bf16>(hidden, ld_h, table, ld_t, rows, width, vocab, targets, weight, softcap, alike != 0, loss, log_sum, (char*)space, error, stream);
  return R2_BAD_DTYPE;
}

extern "C" int r2_token_loss_gradient(int dtype, const void* hidden, long long ld_h, const void* table, long long ld_t, int rows, int width, int vocab,
                                      const int32_t* targets, const float* weight, const float* log_sum, float softcap, void* d_hidden, long long ld_dh,
                                      void* d_table, long long ld_dt, void* space, int* error, cudaStream_t stream) {
  if (rows < 1 || width < 1 || vocab < 1) return R2_BAD_SHAPE;
  if (rows > MOST || width > MOST || vocab > MOST) return R2_UNSUPPORTED;
  if (dtype == R2_F32)
    return gradient_of<float>(hidden, ld_h, table, ld_t, rows, width, vocab, targets, weight, log_sum, softcap, d_hidden, ld_dh, d_table, ld_dt, (char*)space, error, stream);
  if (dtype == R2_BF16)
    return gradient_of<bf16>(hidden, ld_h, table, ld_t, rows, width, vocab, targets, weight, log_sum, softcap, d_hidden, ld_dh, d_table, ld_dt, (char*)space, error, stream);
  return R2_BAD_DTYPE;
}
