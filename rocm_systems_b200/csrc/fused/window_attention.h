// Arguments of the windowed attention's launchers.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace b200 {
namespace wattn {

// A bf16 tensor [batch, heads, seq, D] with a dense last dimension; strides in elements.
struct Tensor {
  const __nv_bfloat16* p;
  long long b, h, s;
  __host__ __device__ __nv_bfloat16* at(int batch, int head, long long pos) const { return const_cast<__nv_bfloat16*>(p) + batch * b + head * h + pos * s; }
};

struct Args {
  Tensor q, k, v, out, dout, dq, dk, dv;
  Tensor rest;         // what rounding took from out (bf16), kept for the backward pass, or nullptr
  float* lse;          // [batch, heads, padded()]: minus log2 of the sum of exp over a row's visible scores, minus infinity behind the sequence's end
  __nv_bfloat16* stat; // [batch, heads, padded(), 8]: of a row -lse / c and -delta, the sum of dout * out, as three values each (backward)
  const int* lengths;  // [batch] or nullptr
  int B, H, KV, S, D;
  int window, sinks;   // window >= 1 (S or more: everything)
  float scale;

  __host__ __device__ int group() const { return H / KV; }
  __host__ __device__ int padded() const { return (S + 127) / 128 * 128; }  // rows' statistics of a head, in whole tiles
};

__device__ __forceinline__ int lengthOf(const Args& a, int batch) {
  const int n = a.lengths ? a.lengths[batch] : a.S;
  return n < 0 ? 0 : n > a.S ? a.S : n;
}
}  // namespace wattn
}  // namespace b200
