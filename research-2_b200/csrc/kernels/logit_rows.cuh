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
