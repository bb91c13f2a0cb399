// Causal attention in which a query sees the last `window` keys (itself among them) and the first `sinks` keys of its sequence:
//   s_ij = scale q_i k_j for j <= i and (i - j < window or j < sinks);  P = softmax over j;  O = P V
//   dV = P^T dO, dP = dO V^T, delta_i = sum_d dO_id O_id, dS = P (dP - delta), dQ = scale dS K, dK = scale dS^T Q
// Query heads share key heads in groups; a sequence may be shorter than the batch (lengths): the rows behind its end answer zeros, and
// nothing that lies there is used.
#include "../core/cudrv.h"
#include "gemm_host.h"
#include "window_attention_sm100.cuh"

namespace b200 {
namespace wattn {

constexpr int kThreads = 256;

// One warp per row, four elements of the head per lane.
__device__ __forceinline__ void load4(const __nv_bfloat16* row, int D, float (&f)[4]) {
  const int lane = threadIdx.x & 31;
  f[0] = f[1] = f[2] = f[3] = 0.f;
  if (4 * lane < D) unpack4(*reinterpret_cast<const uint2*>(row + 4 * lane), f);
}
__device__ __forceinline__ void store4(__nv_bfloat16* row, int D, const float (&f)[4]) {
  const int lane = threadIdx.x & 31;
  if (4 * lane < D) *reinterpret_cast<uint2*>(row + 4 * lane) = pack4(f);
}
__device__ __forceinline__ float dot4(const float (&x)[4], const float (&y)[4]) { return laneSum<32>(x[0] * y[0] + x[1] * y[1] + x[2] * y[2] + x[3] * y[3]); }

// Next visible key from j on: the sinks, then the window.
__device__ __forceinline__ int nextKey(const Args& a, int i, int j) { return visible(a, i, j) || j > i ? j : max(j, i - a.window + 1); }

__global__ void __launch_bounds__(kThreads) queryGradRows(const Args a) {
  const long long row = (long long)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  if (row >= (long long)a.B * a.H * a.S) return;
  const int i = (int)(row % a.S), h = (int)(row / a.S % a.H), b = (int)(row / a.S / a.H), kh = h / a.group();
  float acc[4] = {}, q[4], g[4], o[4];
  if (i < lengthOf(a, b)) {
    load4(a.q.at(b, h, i), a.D, q);
    load4(a.dout.at(b, h, i), a.D, g);
    load4(a.out.at(b, h, i), a.D, o);
    float rest[4];
    load4(a.rest.at(b, h, i), a.D, rest);
    const float delta = dot4(g, o) + dot4(g, rest), lse = a.lse[row], c = a.scale * kLog2e;
    if ((threadIdx.x & 31) == 0) a.delta[row] = delta;
    for (int j = nextKey(a, i, 0); j <= i; j = nextKey(a, i, j + 1)) {
      float k[4], v[4];
      load4(a.k.at(b, kh, j), a.D, k);
      load4(a.v.at(b, kh, j), a.D, v);
      const float ds = exp2Fast(dot4(q, k) * c - lse) * (dot4(g, v) - delta) * a.scale;
#pragma unroll
      for (int e = 0; e < 4; e++) acc[e] += ds * k[e];
    }
  }
  store4(a.dq.at(b, h, i), a.D, acc);
}

__global__ void __launch_bounds__(kThreads) keyGradRows(const Args a) {
  const long long row = (long long)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  if (row >= (long long)a.B * a.KV * a.S) return;
  const int j = (int)(row % a.S), kh = (int)(row / a.S % a.KV), b = (int)(row / a.S / a.KV), L = lengthOf(a, b);
  float dk[4] = {}, dv[4] = {}, k[4], v[4];
  if (j < L) {
    load4(a.k.at(b, kh, j), a.D, k);
    load4(a.v.at(b, kh, j), a.D, v);
    const float c = a.scale * kLog2e;
    const int last = j < a.sinks || a.window > L - j ? L : j + a.window;
    for (int h = kh * a.group(); h < (kh + 1) * a.group(); h++)
      for (int i = j; i < last; i++) {
        float q[4], g[4];
        load4(a.q.at(b, h, i), a.D, q);
        load4(a.dout.at(b, h, i), a.D, g);
        const size_t r = ((size_t)b * a.H + h) * a.S + i;
        const float p = exp2Fast(dot4(q, k) * c - a.lse[r]), ds = p * (dot4(g, v) - a.delta[r]) * a.scale;
#pragma unroll
        for (int e = 0; e < 4; e++) {
          dk[e] += ds * q[e];
          dv[e] += p * g[e];
        }
      }
  }
  store4(a.dk.at(b, kh, j), a.D, dk);
  store4(a.dv.at(b, kh, j), a.D, dv);
}

static bool good(const Args& a) {
  return a.B > 0 && a.H > 0 && a.KV > 0 && a.H % a.KV == 0 && a.S > 0 && a.D >= 8 && a.D <= 128 && a.D % 8 == 0 && a.window > 0 && a.sinks >= 0 && a.scale >= 0.f &&
         (long long)a.B * a.H * a.S <= 0x3fffffffffLL;
}
static Tensor packed(const void* p, const Args& a) { return {(const __nv_bfloat16*)p, (long long)a.S * a.H * a.D, a.D, (long long)a.H * a.D}; }
static bool aligned(const Tensor& t) { return t.p && ((uintptr_t)t.p & 15) == 0 && t.b % 8 == 0 && t.h % 8 == 0 && t.s % 8 == 0; }

// Boxes of 128 positions x 64 elements of one head, 128-byte swizzle; what lies outside the tensor reads as zeros.
static bool headMap(CUtensorMap* map, const Tensor& t, int B, int heads, int S, int D) {
  const CuDrv& d = CuDrv::get();
  if (!d.cuTensorMapEncodeTiled) return false;
  const auto stride = [&](long long st, int n) { return (cuuint64_t)(n > 1 ? st : D) * 2; };  // of a dimension of one it does not matter
  const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)S, (cuuint64_t)heads, (cuuint64_t)B};
  const cuuint64_t strides[3] = {stride(t.s, S), stride(t.h, heads), stride(t.b, B)};
  const cuuint32_t box[4] = {64, kTile, 1, 1}, ones[4] = {1, 1, 1, 1};
  return d.cuTensorMapEncodeTiled(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<__nv_bfloat16*>(t.p), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Lets a kernel use `bytes` of dynamic shared memory on the current device; remembered per device.
template <typename K> static cudaError_t allowSmem(K kernel, size_t bytes, bool (&done)[64]) {
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && done[dev]) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e == cudaSuccess && dev >= 0 && dev < 64) done[dev] = true;
  return e;
}

template <int HD> static cudaError_t forward(const Args& a, cudaStream_t s) {
  static bool done[64] = {};
  FwdParams p{};
  p.a = a;
  p.c = fmaxf(a.scale * kLog2e, 1e-30f);  // times the scores' minus infinities it has to stay one
  p.tiles = (a.S + 2 * kTile - 1) / (2 * kTile);
  p.err = gemm::errWord();
  if (!p.err) return cudaErrorMemoryAllocation;
  const long long ctas = (long long)p.tiles * a.B * a.H;
  if (ctas > 0x7fffffffLL || !headMap(&p.q, a.q, a.B, a.H, a.S, a.D) || !headMap(&p.k, a.k, a.B, a.KV, a.S, a.D) || !headMap(&p.v, a.v, a.B, a.KV, a.S, a.D))
    return cudaErrorInvalidValue;
  const cudaError_t e = allowSmem(forwardKernel<HD>, FwdCfg<HD>::kSmem, done);
  if (e != cudaSuccess) return e;
  forwardKernel<HD><<<(unsigned)ctas, FwdCfg<HD>::kThreads, FwdCfg<HD>::kSmem, s>>>(p);
  return cudaGetLastError();
}

static unsigned rowCtas(long long rows) { return (unsigned)((rows + kThreads / 32 - 1) / (kThreads / 32)); }

}  // namespace wattn
}  // namespace b200

using namespace b200::wattn;

extern "C" {

// q, out [B, H, S, D], k, v [B, KV, S, D] bf16, 16-byte aligned, with strides (batch, head, position) of q, k, v, out in turn (elements,
// multiples of 8). lse (fp32 [B, H, S]) and rest (bf16 [B, S, H, D], what rounding took from out) are for the backward call, or nullptr. lengths: int32 [B] on the device, or nullptr. window 0: no window.
int b200ops_window_attention_fwd(const void* q, const void* k, const void* v, void* out, float* lse, void* rest, const int* lengths, const long long* strides, int B, int H, int KV,
                                 int S, int D, int window, int sinks, float scale, cudaStream_t s) {
  const auto tensor = [&](const void* p, int i) { return Tensor{(const __nv_bfloat16*)p, strides[3 * i], strides[3 * i + 1], strides[3 * i + 2]}; };
  Args a{};
  a.q = tensor(q, 0);
  a.k = tensor(k, 1);
  a.v = tensor(v, 2);
  a.out = tensor(out, 3);
  a.lse = lse;
  a.lengths = lengths;
  a.B = B, a.H = H, a.KV = KV, a.S = S, a.D = D;
  a.window = window == 0 ? S : window;
  a.sinks = sinks;
  a.scale = scale;
  a.rest = packed(rest, a);
  if (!good(a) || !aligned(a.q) || !aligned(a.k) || !aligned(a.v) || !aligned(a.out) || ((uintptr_t)rest & 15)) return (int)cudaErrorInvalidValue;
  return (int)(D <= 64 ? forward<64>(a, s) : forward<128>(a, s));
}

// strides: of q, k, v, out, dout, dq, dk, dv in turn. lse and rest as the forward call left them; delta: fp32 [B, H, S] scratch.
int b200ops_window_attention_bwd(const void* q, const void* k, const void* v, const void* out, const void* rest, const void* dout, const float* lse, float* delta, void* dq, void* dk,
                                 void* dv, const int* lengths, const long long* strides, int B, int H, int KV, int S, int D, int window, int sinks, float scale,
                                 cudaStream_t s) {
  const auto tensor = [&](const void* p, int i) { return Tensor{(const __nv_bfloat16*)p, strides[3 * i], strides[3 * i + 1], strides[3 * i + 2]}; };
  Args a{};
  a.q = tensor(q, 0);
  a.k = tensor(k, 1);
  a.v = tensor(v, 2);
  a.out = tensor(out, 3);
  a.dout = tensor(dout, 4);
  a.dq = tensor(dq, 5);
  a.dk = tensor(dk, 6);
  a.dv = tensor(dv, 7);
  a.lse = const_cast<float*>(lse);
  a.delta = delta;
  a.lengths = lengths;
  a.B = B, a.H = H, a.KV = KV, a.S = S, a.D = D;
  a.window = window == 0 ? S : window;
  a.sinks = sinks;
  a.scale = scale;
  a.rest = packed(rest, a);
  if (!good(a) || !lse || !delta || !rest || ((uintptr_t)rest & 15)) return (int)cudaErrorInvalidValue;
  for (const Tensor* t : {&a.q, &a.k, &a.v, &a.out, &a.dout, &a.dq, &a.dk, &a.dv})
    if (!aligned(*t)) return (int)cudaErrorInvalidValue;
  queryGradRows<<<rowCtas((long long)B * H * S), kThreads, 0, s>>>(a);
  keyGradRows<<<rowCtas((long long)B * KV * S), kThreads, 0, s>>>(a);
  return (int)cudaGetLastError();
}

}  // extern "C"
