// Rows of logits as 16-byte pieces, whatever a row's alignment: a vocabulary of odd size puts most rows off a 16-byte boundary.
//
// Piece g of a row is the aligned 16 bytes that hold its elements g * PER - phase and up, phase the number of elements by which the row
// starts behind a boundary. A piece that holds at least one element of the row may be read whole: its other bytes lie in the same aligned
// 16 bytes as that element and so in the same allocation.
#pragma once

#include "common.cuh"

template <typename T>
struct RowPieces {
  static constexpr int PER = 16 / int(sizeof(T));
  const T* base;    // of piece 0: the row's start less the phase
  int phase, count; // count: pieces that hold elements of the row
  int vocab;

  __device__ RowPieces(const T* row, int vocab_) : vocab(vocab_) {
    phase = int((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    base = row - phase;
    count = (phase + vocab + PER - 1) / PER;
  }
  // the row's element that stands first in piece g (negative in a first piece that starts before the row)
  __device__ int first(int g) const { return g * PER - phase; }
  // whether every element of piece g belongs to the row
  __device__ bool whole(int g) const { return first(g) >= 0 && first(g) + PER <= vocab; }
  __device__ uint4 load(int g) const { return __ldg(reinterpret_cast<const uint4*>(base) + g); }
};

__device__ __forceinline__ void unpack(const uint4& raw, float (&x)[4], const float*) {
  x[0] = __uint_as_float(raw.x);
  x[1] = __uint_as_float(raw.y);
  x[2] = __uint_as_float(raw.z);
  x[3] = __uint_as_float(raw.w);
}
__device__ __forceinline__ void unpack(const uint4& raw, float (&x)[8], const bf16*) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ uint4 pack(const float (&x)[4], const float*) {
  return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
}
__device__ __forceinline__ uint4 pack(const float (&x)[8], const bf16*) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 two = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&two);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Piece g of an output row whose alignment is the input's (`vectors`) or another: whole pieces as one store, others element by element.
template <typename T, int PER>
__device__ __forceinline__ void store_piece(T* row, int first, int vocab, const float (&x)[PER], bool vectors) {
  if (vectors && first >= 0 && first + PER <= vocab) {
    *reinterpret_cast<uint4*>(row + first) = pack(x, static_cast<const T*>(nullptr));
    return;
  }
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (first + i >= 0 && first + i < vocab) row[first + i] = from_float<T>(x[i]);
}

// Floats as unsigned keys in the floats' order; equal values have equal keys (-0 is +0), and a NaN stands below everything.
__device__ __forceinline__ uint32_t logit_key(float v) {
  if (v != v) return 0u;
  const uint32_t b = __float_as_uint(v + 0.f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

// A piece of the row for a reader that may also be its writer in the same launch (no read-only path), not kept in L1. Elements beyond the row
// are -inf.
__device__ __forceinline__ uint4 load_16(const uint4* from) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(from));
  return v;
}
__device__ __forceinline__ void load_16_if(uint4& v, const uint4* from, bool asked) {   // (else what was there stays)
  asm volatile("{\n .reg .pred p;\n setp.ne.u32 p, %5, 0;\n @p ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];\n}"
               : "+r"(v.x), "+r"(v.y), "+r"(v.z), "+r"(v.w) : "l"(from), "r"(uint32_t(asked)));
}
template <typename T>
__device__ __forceinline__ uint4 load_once(const RowPieces<T>& row, int g) { return load_16(reinterpret_cast<const uint4*>(row.base) + g); }

// Elements of a piece to -inf where their bits are 0. A bit becomes a byte's highest (the product puts bit i at 8 i + 7 and nothing else
// there), and a byte's highest bit becomes whole bytes (prmt's sign mode).
__device__ __forceinline__ uint32_t spread(uint32_t four_bits) { return (four_bits * 0x10204080u) & 0x80808080u; }
__device__ __forceinline__ uint32_t signs(uint32_t bytes, uint32_t selector) {
  uint32_t d;
  asm("prmt.b32 %0, %1, %1, %2;" : "=r"(d) : "r"(bytes), "r"(selector));
  return d;
}
template <typename T>
__device__ __forceinline__ void keep_bits(uint4& raw, uint32_t bits) {
  uint32_t m[4];
  const uint32_t low = spread(bits & 15u);
  if (sizeof(T) == 4) {
    m[0] = signs(low, 0x8888u);
    m[1] = signs(low, 0x9999u);
    m[2] = signs(low, 0xaaaau);
    m[3] = signs(low, 0xbbbbu);
  } else {
    const uint32_t high = spread((bits >> 4) & 15u);
    m[0] = signs(low, 0x9988u);
    m[1] = signs(low, 0xbbaau);
    m[2] = signs(high, 0x9988u);
    m[3] = signs(high, 0xbbaau);
  }
  constexpr uint32_t NOTHING = sizeof(T) == 4 ? 0xff800000u : 0xff80ff80u;
  raw = make_uint4((raw.x & m[0]) | (NOTHING & ~m[0]), (raw.y & m[1]) | (NOTHING & ~m[1]), (raw.z & m[2]) | (NOTHING & ~m[2]),
                   (raw.w & m[3]) | (NOTHING & ~m[3]));
}
template <typename T>
__device__ __forceinline__ void blank_outside(uint4& raw, const RowPieces<T>& row, int g) {
  if (row.whole(g)) return;
  const int first = row.first(g);
  uint32_t bits = first < 0 ? (1u << -first) - 1u : 0u;
  if (first + RowPieces<T>::PER > row.vocab) bits |= ~0u << (row.vocab - first);
  keep_bits<T>(raw, ~bits);
}
// A piece's elements that belong to the row, one by one.
template <typename T>
__device__ __noinline__ void store_elements(T* row, int first, int vocab, uint4 raw) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < RowPieces<T>::PER; ++i) {
    if (first + i < 0 || first + i >= vocab) continue;
    if (sizeof(T) == 4) reinterpret_cast<uint32_t*>(row)[first + i] = w[i & 3];
    else reinterpret_cast<uint16_t*>(row)[first + i] = uint16_t(w[(i >> 1) & 3] >> (i % 2 * 16));
  }
}

__device__ __forceinline__ float exp2_approx(float x) {  // 2^x within 2^-22; 0 below the normal range
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Sums of exponentials are kept against a reference, an exponent of two; -inf where nothing has been summed. A reference is a rounded product, and
// 2^x is taken of exact products less it: off by up to 64 for references below 2^31, which the sums bear, and by ever more beyond. What is
// summed against a reference beyond counts as nothing, a mask's low number as well as one above any logit; infinity against it is infinity.
constexpr float FAR_REFERENCE = 2147483648.f, LARGEST_FLOAT = 3.40282347e38f;
__device__ __forceinline__ float shift_to(float reference) {
  return fabsf(reference) < FAR_REFERENCE ? -reference : reference > 0.f ? -LARGEST_FLOAT : 0.f;
}
__device__ __forceinline__ float no_less(float reference) { return reference == -INFINITY ? 0.f : reference; }
// what sums against `reference` are in sums against `common`, the largest of several references
__device__ __forceinline__ float rebase(float reference, float common) { return reference == -INFINITY ? 0.f : exp2_approx(reference - common); }

// The CTAs of a cluster along x share a row.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t cluster_address(const void* own, uint32_t rank) {  // of `own` in the shared memory of CTA `rank`
  uint32_t there;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(uint32_t(__cvta_generic_to_shared(own))), "r"(rank));
  return there;
}
__device__ __forceinline__ void cluster_store(uint32_t address, float4 v) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(address), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}

template <typename... KArgs, typename... Args>
static inline void r2_launch_clusters(void (*kernel)(KArgs...), int cluster, dim3 grid, dim3 block, size_t smem, cudaStream_t stream,
                                      Args&&... args) {
  cudaLaunchConfig_t config = {};
  config.gridDim = grid;
  config.blockDim = block;
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = unsigned(cluster);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attr;
  config.numAttrs = (g_r2_pdl && !t_r2_plain_order) ? 2 : 1;
  cudaLaunchKernelEx(&config, kernel, static_cast<Args&&>(args)...);  // a failure shows in launch_status()
}

// Two floats side by side: one instruction for both, each rounded as the single one rounds.
__device__ __forceinline__ uint64_t two_of(float lo, float hi) {
  uint64_t p;
  asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(lo), "f"(hi));
  return p;
}
__device__ __forceinline__ float2 halves(uint64_t p) {
  float2 v;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(p));
  return v;
}
__device__ __forceinline__ uint64_t fma_two(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t mul_two(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t add_two(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t exp2_two(uint64_t p) {
  const float2 v = halves(p);
  return two_of(exp2_approx(v.x), exp2_approx(v.y));
}
// A piece as pairs.
__device__ __forceinline__ void unpack_pairs(const uint4& raw, uint64_t (&p)[2], const float*) {
  p[0] = two_of(__uint_as_float(raw.x), __uint_as_float(raw.y));
  p[1] = two_of(__uint_as_float(raw.z), __uint_as_float(raw.w));
}
__device__ __forceinline__ void unpack_pairs(const uint4& raw, uint64_t (&p)[4], const bf16*) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) p[i] = two_of(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
}
__device__ __forceinline__ uint4 pack_pairs(const uint64_t (&p)[2], const float*) {
  const float2 a = halves(p[0]), b = halves(p[1]);
  return make_uint4(__float_as_uint(a.x), __float_as_uint(a.y), __float_as_uint(b.x), __float_as_uint(b.y));
}
__device__ __forceinline__ uint4 pack_pairs(const uint64_t (&p)[4], const bf16*) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = halves(p[i]);
    const __nv_bfloat162 two = __floats2bfloat162_rn(v.x, v.y);
    w[i] = *reinterpret_cast<const uint32_t*>(&two);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
