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

static bool good(const Args& a) {
  return a.B > 0 && a.H > 0 && a.KV > 0 && a.H % a.KV == 0 && a.S > 0 && a.D >= 8 && a.D <= 128 && a.D % 8 == 0 && a.window > 0 && a.sinks >= 0 && a.scale >= 0.f &&
         (long long)a.B * a.H * a.S <= 0x3fffffffffLL;
}
static bool wide(const Tensor& t) { return ((uintptr_t)t.p & 31) == 0 && t.b % 16 == 0 && t.h % 16 == 0 && t.s % 16 == 0; }
static Tensor packed(const void* p, const Args& a) { return {(const __nv_bfloat16*)p, (long long)a.S * a.H * a.D, a.D, (long long)a.H * a.D}; }
static bool aligned(const Tensor& t) { return t.p && ((uintptr_t)t.p & 15) == 0 && t.b % 8 == 0 && t.h % 8 == 0 && t.s % 8 == 0; }

static Args sizes(int B, int H, int KV, int S, int D, int window, int sinks) {
  Args a{};
  a.B = B, a.H = H, a.KV = KV, a.S = S, a.D = D;
  a.window = window == 0 || sinks >= S ? S : window;  // S or more: every earlier key
  a.sinks = sinks < S ? sinks : S;
  return a;
}

// The device's context made current on this thread: encoding a tensor map asks for one, and a backward pass may be the first that its
// thread does.
static void bindContext() {
  static thread_local int bound = -1;
  int dev = 0;
  if (cudaGetDevice(&dev) == cudaSuccess && dev != bound && cudaSetDevice(dev) == cudaSuccess) bound = dev;
}

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

template <int HD, bool FINE> static cudaError_t forward(const Args& a, cudaStream_t s) {
  static bool done[64] = {};
  bindContext();
  FwdParams p{};
  p.a = a;
  p.c = fmaxf(a.scale * kLog2e, 1e-30f);  // times the scores' minus infinities it has to stay one
  p.tiles = (a.S + 2 * kTile - 1) / (2 * kTile);
  p.err = gemm::errWord();
  if (!p.err) return cudaErrorMemoryAllocation;
  const long long items = (long long)p.tiles * a.B * a.H;
  p.items = (uint32_t)items;
  p.wide = wide(a.out) && (!a.rest.p || wide(a.rest)) && a.D % 16 == 0;
  const int ctas = (int)(items < gemm::smCount() ? items : gemm::smCount());  // one per SM
  if (items > 0x3fffffffLL || !headMap(&p.q, a.q, a.B, a.H, a.S, a.D) || !headMap(&p.k, a.k, a.B, a.KV, a.S, a.D) || !headMap(&p.v, a.v, a.B, a.KV, a.S, a.D))
    return cudaErrorInvalidValue;
  const cudaError_t e = allowSmem(forwardKernel<HD, FINE>, FwdCfg<HD>::kSmem, done);
  if (e != cudaSuccess) return e;
  forwardKernel<HD, FINE><<<ctas, FwdCfg<HD>::kThreads, FwdCfg<HD>::kSmem, s>>>(p);
  return cudaGetLastError();
}

// Whether the weights and their gradients of all rows are held as two bf16 values.
static bool fine(const Args& a) { return a.S <= kFineSeq || a.window <= kFineKeys - a.sinks; }

// How the sinks' far queries are split: every key tile that holds sinks and is not through with its window's queries. With kMostSplits such
// tiles there is work for all SMs without, and the partial sums stay below 2 kMostSplits blocks (268 MB at D = 128).
constexpr int kMostSplits = 1024;
static void splitSinks(const Args& a, BwdParams& p) {
  p.tiles = (a.S + kTile - 1) / kTile;
  if (a.sinks == 0 || a.window >= a.S) return;
  const int near = (kTile + a.window - 2) / kTile + 1;  // query tiles that see a key tile through the window
  const int far = p.tiles - near;                       // of the first tile; the others have fewer
  if (far <= 0) return;
  const long long sinkTiles = (a.sinks + kTile - 1) / kTile, splits = kMostSplits / (sinkTiles * a.B * a.KV);
  if (splits == 0) return;
  p.sinkTiles = (int)sinkTiles;
  p.farChunk = (int)((far + splits - 1) / splits);
  if (p.farChunk < near) p.farChunk = near;
  if (p.farChunk < 4) p.farChunk = 4;
  p.farCount = (far + p.farChunk - 1) / p.farChunk;
}
static long long partialWords(const Args& a, const BwdParams& p) {
  return (long long)a.B * a.KV * p.sinkTiles * (1 + p.farCount) * 2 * (a.sinks < kTile ? a.sinks : kTile) * a.D;
}

template <int HD, bool FINE> static cudaError_t backward(const Args& a, float* partials, cudaStream_t s) {
  static bool doneQ[64] = {}, doneK[64] = {};
  using Q = BwdCfg<HD, kQueries>;
  using K = BwdCfg<HD, kKeys>;
  bindContext();
  BwdParams p{};
  p.a = a;
  p.c = fmaxf(a.scale * kLog2e, 1e-30f);
  p.err = gemm::errWord();
  if (!p.err) return cudaErrorMemoryAllocation;
  splitSinks(a, p);
  p.partials = partials;
  p.wide = a.D % 16 == 0 && wide(a.dq) && wide(a.dk) && wide(a.dv);
  BwdParams k = p;
  const long long itemsQ = (long long)p.tiles * a.B * a.H, itemsK = (long long)(p.tiles + p.sinkTiles * p.farCount) * a.B * a.KV;
  p.items = (uint32_t)itemsQ;
  k.items = (uint32_t)itemsK;
  if (itemsQ > 0x3fffffffLL || itemsK > 0x3fffffffLL || a.B * (long long)a.KV > 65535 || !headMap(&p.x1, a.q, a.B, a.H, a.S, a.D) ||
      !headMap(&p.x2, a.dout, a.B, a.H, a.S, a.D) || !headMap(&p.y1, a.k, a.B, a.KV, a.S, a.D) || !headMap(&p.y2, a.v, a.B, a.KV, a.S, a.D) ||
      !headMap(&p.out, a.out, a.B, a.H, a.S, a.D) || !headMap(&p.rest, a.rest, a.B, a.H, a.S, a.D))
    return cudaErrorInvalidValue;
  k.x1 = p.y1, k.x2 = p.y2, k.y1 = p.x1, k.y2 = p.x2;
  cudaError_t e = allowSmem(backwardKernel<HD, kQueries, FINE>, Q::kSmem, doneQ);
  if (e == cudaSuccess) e = allowSmem(backwardKernel<HD, kKeys, FINE>, K::kSmem, doneK);
  if (e != cudaSuccess) return e;
  const auto ctas = [](long long items) { return (unsigned)(items < gemm::smCount() ? items : gemm::smCount()); };  // one per SM
  backwardKernel<HD, kQueries, FINE><<<ctas(itemsQ), Q::kThreads, Q::kSmem, s>>>(p);
  backwardKernel<HD, kKeys, FINE><<<ctas(itemsK), K::kThreads, K::kSmem, s>>>(k);
  if (p.sinkTiles) joinSinks<<<dim3(a.sinks, a.B * a.KV), 128, 0, s>>>(k);
  return cudaGetLastError();
}

}  // namespace wattn
}  // namespace b200

using namespace b200::wattn;

extern "C" {

// q, out [B, H, S, D], k, v [B, KV, S, D] bf16, 16-byte aligned, with strides (batch, head, position) of q, k, v, out in turn (elements,
// multiples of 8). lse (fp32 [B, H, S rounded up to 128]) and rest (bf16 [B, S, H, D], what rounding took from out) are for the backward call,
// or nullptr. lengths: int32 [B] on the device, or nullptr. window 0: no window.
int b200ops_window_attention_fwd(const void* q, const void* k, const void* v, void* out, float* lse, void* rest, const int* lengths, const long long* strides, int B, int H, int KV,
                                 int S, int D, int window, int sinks, float scale, cudaStream_t s) {
  const auto tensor = [&](const void* p, int i) { return Tensor{(const __nv_bfloat16*)p, strides[3 * i], strides[3 * i + 1], strides[3 * i + 2]}; };
  Args a = sizes(B, H, KV, S, D, window, sinks);
  a.q = tensor(q, 0);
  a.k = tensor(k, 1);
  a.v = tensor(v, 2);
  a.out = tensor(out, 3);
  a.lse = lse;
  a.lengths = lengths;
  a.scale = scale;
  a.rest = packed(rest, a);
  if (!good(a) || !aligned(a.q) || !aligned(a.k) || !aligned(a.v) || !aligned(a.out) || ((uintptr_t)rest & 15)) return (int)cudaErrorInvalidValue;
  if (fine(a)) return (int)(D <= 64 ? forward<64, true>(a, s) : forward<128, true>(a, s));
  return (int)(D <= 64 ? forward<64, false>(a, s) : forward<128, false>(a, s));
}

// strides: of q, k, v, out, dout, dq, dk, dv in turn. lse and rest as the forward call left them; scratch: as many fp32
// words as b200ops_window_attention_bwd_scratch says.
int b200ops_window_attention_bwd(const void* q, const void* k, const void* v, const void* out, const void* rest, const void* dout, const float* lse, float* scratch, void* dq, void* dk,
                                 void* dv, const int* lengths, const long long* strides, int B, int H, int KV, int S, int D, int window, int sinks, float scale,
                                 cudaStream_t s) {
  const auto tensor = [&](const void* p, int i) { return Tensor{(const __nv_bfloat16*)p, strides[3 * i], strides[3 * i + 1], strides[3 * i + 2]}; };
  Args a = sizes(B, H, KV, S, D, window, sinks);
  a.q = tensor(q, 0);
  a.k = tensor(k, 1);
  a.v = tensor(v, 2);
  a.out = tensor(out, 3);
  a.dout = tensor(dout, 4);
  a.dq = tensor(dq, 5);
  a.dk = tensor(dk, 6);
  a.dv = tensor(dv, 7);
  a.lse = const_cast<float*>(lse);
  a.stat = reinterpret_cast<__nv_bfloat16*>(scratch);
  a.lengths = lengths;
  a.scale = scale;
  a.rest = packed(rest, a);
  if (!good(a) || !lse || !scratch || !rest || (((uintptr_t)rest | (uintptr_t)lse | (uintptr_t)scratch) & 15)) return (int)cudaErrorInvalidValue;
  for (const Tensor* t : {&a.q, &a.k, &a.v, &a.out, &a.dout, &a.dq, &a.dk, &a.dv})
    if (!aligned(*t)) return (int)cudaErrorInvalidValue;
  float* partials = scratch + (size_t)B * H * a.padded() * 4;
  if (fine(a)) return (int)(D <= 64 ? backward<64, true>(a, partials, s) : backward<128, true>(a, partials, s));
  return (int)(D <= 64 ? backward<64, false>(a, partials, s) : backward<128, false>(a, partials, s));
}

long long b200ops_window_attention_bwd_scratch(int B, int H, int KV, int S, int D, int window, int sinks) {
  const Args a = sizes(B, H, KV, S, D, window, sinks);
  if (!good(a)) return -1;
  BwdParams p{};
  splitSinks(a, p);
  return (long long)B * H * a.padded() * 4 + partialWords(a, p);
}

// Kernels that the backward call launches: for the queries, for the keys and, where the sinks' queries are split, for their sums.
int b200ops_window_attention_bwd_launches(int B, int H, int KV, int S, int D, int window, int sinks) {
  const Args a = sizes(B, H, KV, S, D, window, sinks);
  if (!good(a)) return -1;
  BwdParams p{};
  splitSinks(a, p);
  return p.sinkTiles ? 3 : 2;
}

}  // extern "C"
