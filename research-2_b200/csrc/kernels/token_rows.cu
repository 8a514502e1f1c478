// Rows of a token table, and the gradient of the table whose rows were looked up:
//
//   out_t = scale * W[i_t]  (zeros where i_t is no token),   dW_v = scale * sum over t with i_t = v of above_t, in the order of t
#include "common.cuh"

namespace {

template <typename T, typename O>
__global__ void token_rows_kernel(const int32_t* ids, const T* table, long long ld, O* out, long long ld_o, int width, int vocab, float scale) {
  const int t = blockIdx.x, id = ids[t];
  const bool held = id >= 0 && id < vocab;
  const T* row = table + size_t(held ? id : 0) * ld;
  O* o = out + size_t(t) * ld_o;
  for (int d = threadIdx.x; d < width; d += blockDim.x) o[d] = from_float<O>(held ? to_float(row[d]) * scale : 0.f);
}

template <typename T, typename O>
__global__ void gradient_kernel(const int32_t* ids, const T* above, long long ld, O* out, long long ld_o, int tokens, int width, float scale, int add) {
  const int v = blockIdx.x;
  O* o = out + size_t(v) * ld_o;
  bool any = false;
  for (int d = threadIdx.x; d < width; d += blockDim.x) {
    float sum = 0.f;
    for (int t = 0; t < tokens; ++t) {
      if (ids[t] == v) {
        sum += to_float(above[size_t(t) * ld + d]);
        any = true;
      }
    }
    if (any || !add) o[d] = from_float<O>(sum * scale + (add ? to_float(o[d]) : 0.f));
  }
}

}  // namespace

extern "C" int r2_token_rows(int dtype, int out_dtype, const int32_t* ids, const void* table, long long ld, void* out, long long ld_o, int tokens, int width, int vocab,
                             float scale, cudaStream_t stream) {
#define R2_CASE(T, O) token_rows_kernel<T, O><<<tokens, 128, 0, stream>>>(ids, (const T*)table, ld, (O*)out, ld_o, width, vocab, scale)
  if (dtype == R2_F32 && out_dtype == R2_F32) R2_CASE(float, float);
  else if (dtype == R2_F32) R2_CASE(float, bf16);
  else if (out_dtype == R2_F32) R2_CASE(bf16, float);
  else R2_CASE(bf16, bf16);
#undef R2_CASE
  return launch_status();
}

extern "C" long long r2_token_rows_space(int tokens, int width, int vocab) { return 16; }

extern "C" int r2_token_rows_gradient(int dtype, int out_dtype, const int32_t* ids, const void* above, long long ld, void* out, long long ld_o, int tokens, int width,
                                      int vocab, float scale, int add, void* space, cudaStream_t stream) {
#define R2_CASE(T, O) gradient_kernel<T, O><<<vocab, 128, 0, stream>>>(ids, (const T*)above, ld, (O*)out, ld_o, tokens, width, scale, add)
  if (dtype == R2_F32 && out_dtype == R2_F32) R2_CASE(float, float);
  else if (dtype == R2_F32) R2_CASE(float, bf16);
  else if (out_dtype == R2_F32) R2_CASE(bf16, float);
  else R2_CASE(bf16, bf16);
#undef R2_CASE
  return launch_status();
}
