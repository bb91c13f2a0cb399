// Distillation from a teacher's top logits, mixed with cross-entropy: per row of student logits z [V] the loss and its gradient.
//   c = softmax(z), q = softmax(z / tau), p = softmax(teacher values / tau) over the row's K stored entries
//   loss = (1 - a) (lse(z) - z_t) + a tau^2 sum_k p_k (log p_k - log q_{id k})
//   dz   = [(1 - a) (c - onehot_t) + a tau (q - sum_{k: id k = v} p_k)] * gradScale
// An entry whose id lies outside [0, V) does not exist; a row without entries has no distillation term. A row whose target lies outside
// [0, V) counts nothing: zero loss, zero gradient.
#include "rows.cuh"

namespace b200 {
namespace distill {

using namespace rows;

constexpr int kThreads = 512;
constexpr int kMaxEntries = 1024;

struct Args {
  const __nv_bfloat16* z;
  __nv_bfloat16* grad;   // may be z
  const long long* targets;
  const void* ids;       // [T, K] int64 or int32
  const void* values;    // [T, K] fp32 or bf16
  float* loss;
  long long zStride, gradStride;
  int V, K;
  float a, tau, gradScale;
};

template <int NT> __device__ __forceinline__ float blockReduce(float v, float* sh, bool maximum) {
  v = maximum ? laneMax<32>(v) : laneSum<32>(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  v = (threadIdx.x & 31) < NT / 32 ? sh[threadIdx.x & 31] : maximum ? -INFINITY : 0.f;
  return maximum ? laneMax<32>(v) : laneSum<32>(v);
}

// One CTA per row, three passes over it: maximum, sums, gradient.
template <typename I, typename W>
__global__ void __launch_bounds__(kThreads) distillKernel(const Args p) {
  __shared__ float sh[32];
  __shared__ int id[kMaxEntries];
  __shared__ float prob[kMaxEntries], logProb[kMaxEntries], zAt[kMaxEntries];
  const size_t row = blockIdx.x;
  const __nv_bfloat16* z = p.z + row * p.zStride;
  __nv_bfloat16* grad = p.grad + row * p.gradStride;
  const long long target = p.targets[row];
  if (target < 0 || target >= p.V) {
    if (threadIdx.x == 0) p.loss[row] = 0.f;
    for (int v = threadIdx.x; v < p.V; v += kThreads) grad[v] = __float2bfloat16(0.f);
    return;
  }
  float m = -INFINITY;
  for (int v = threadIdx.x; v < p.V; v += kThreads) m = fmaxf(m, __bfloat162float(z[v]));
  m = blockReduce<kThreads>(m, sh, true);
  const float one = kLog2e, soft = kLog2e / p.tau;
  float sumOne = 0.f, sumSoft = 0.f;
  for (int v = threadIdx.x; v < p.V; v += kThreads) {
    const float d = __bfloat162float(z[v]) - m;
    sumOne += exp2Fast(d * one);
    sumSoft += exp2Fast(d * soft);
  }
  sumOne = blockReduce<kThreads>(sumOne, sh, false);
  sumSoft = blockReduce<kThreads>(sumSoft, sh, false);

  // the teacher's entries
  float best = -INFINITY;
  for (int k = threadIdx.x; k < p.K; k += kThreads) {
    const long long i = (long long)reinterpret_cast<const I*>(p.ids)[row * p.K + k];
    const bool exists = i >= 0 && i < p.V;
    const float y = exists ? toFloat(reinterpret_cast<const W*>(p.values)[row * p.K + k]) / p.tau : -INFINITY;
    id[k] = exists ? (int)i : -1;
    logProb[k] = y;
    zAt[k] = exists ? __bfloat162float(z[i]) : 0.f;
    best = fmaxf(best, y);
  }
  best = blockReduce<kThreads>(best, sh, true);
  float norm = 0.f;
  if (best > -INFINITY)
    for (int k = threadIdx.x; k < p.K; k += kThreads)
      if (id[k] >= 0) norm += exp2Fast((logProb[k] - best) * kLog2e);
  norm = blockReduce<kThreads>(norm, sh, false);
  const float a = norm == 0.f ? 0.f : p.a;
  const float logNorm = logf(norm), logSoft = logf(sumSoft);
  float kl = 0.f;
  for (int k = threadIdx.x; k < p.K; k += kThreads) {
    const float lp = logProb[k] - best - logNorm;
    const float pk = id[k] >= 0 && norm != 0.f ? exp2Fast(lp * kLog2e) : 0.f;
    prob[k] = pk;
    if (pk != 0.f) kl += pk * (lp - ((zAt[k] - m) / p.tau - logSoft));
  }
  kl = blockReduce<kThreads>(kl, sh, false);
  const float zt = __bfloat162float(z[target]);
  if (threadIdx.x == 0) p.loss[row] = (1.f - p.a) * (m + logf(sumOne) - zt) + a * p.tau * p.tau * kl;
  __syncthreads();

  const float fOne = (1.f - p.a) / sumOne * p.gradScale, fSoft = a * p.tau / sumSoft * p.gradScale;
  const auto dense = [&](float x) { return fOne * exp2Fast((x - m) * one) + fSoft * exp2Fast((x - m) * soft); };
  for (int v = threadIdx.x; v < p.V; v += kThreads) grad[v] = __float2bfloat16(dense(__bfloat162float(z[v])));
  __syncthreads();
  // The teacher's entries and the target once more, from their logits in 32 bits. An id's first entry writes for all of them.
  for (int k = threadIdx.x; k <= p.K; k += kThreads) {
    const int v = k < p.K ? id[k] : (int)target;
    if (v < 0) continue;
    float mass = 0.f;
    bool first = true;
    for (int o = 0; o < p.K; o++)
      if (id[o] == v) {
        mass += prob[o];
        first = first && o >= k;
      }
    if (!first) continue;
    const float x = k < p.K ? zAt[k] : zt;
    grad[v] = __float2bfloat16(dense(x) - p.gradScale * (a * p.tau * mass + (v == target ? 1.f - p.a : 0.f)));
  }
}

}  // namespace distill
}  // namespace b200

extern "C" {

// Rows of logits [T, V] bf16 (row stride in elements) and of grad (the same buffer and stride, or another); targets int64 [T];
// ids [T, K] int64 (idBytes 8) or int32 (4); values [T, K] fp32 (valueBytes 4) or bf16 (2); loss fp32 [T].
int b200ops_distill_loss(const void* logits, void* grad, const long long* targets, const void* ids, int idBytes, const void* values, int valueBytes, float* loss,
                         long long T, int V, int K, long long stride, long long gradStride, float a, float tau, float gradScale, cudaStream_t s) {
  using namespace b200::distill;
  if (T < 0 || T > 0x7fffffffLL || V <= 0 || K <= 0 || K > kMaxEntries || !(tau > 0.f) || stride < V || gradStride < V || (idBytes != 4 && idBytes != 8) ||
      (valueBytes != 2 && valueBytes != 4))
    return (int)cudaErrorInvalidValue;
  if (T == 0) return 0;
  const Args p{(const __nv_bfloat16*)logits, (__nv_bfloat16*)grad, targets, ids, values, loss, stride, gradStride, V, K, a, tau, gradScale};
  const auto go = [&](auto kernel) { kernel<<<(unsigned)T, kThreads, 0, s>>>(p); };
  if (idBytes == 8) go(valueBytes == 4 ? distillKernel<long long, float> : distillKernel<long long, __nv_bfloat16>);
  else go(valueBytes == 4 ? distillKernel<int, float> : distillKernel<int, __nv_bfloat16>);
  return (int)cudaGetLastError();
}

}  // extern "C"
