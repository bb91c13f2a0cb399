// Distillation from a teacher's top logits, mixed with cross-entropy: per row of student logits z [V] the loss and its gradient.
//   c = softmax(z), q = softmax(z / tau), p = softmax(teacher values / tau) over the row's K stored entries
//   loss = (1 - a) (lse(z) - z_t) + a tau^2 sum_k p_k (log p_k - log q_{id k})
//   dz   = [(1 - a) (c - onehot_t) + a tau (q - sum_{k: id k = v} p_k)] * gradScale
// An entry whose id lies outside [0, V) does not exist; a row without entries has no distillation term. A row whose target lies outside
// [0, V) counts nothing: zero loss, zero gradient.
//
// A row is read once and its gradient written once: a cluster of 1 to 8 CTAs holds it in shared memory, a slice each (32 KB if that is
// enough, so that six CTAs of 128 threads share an SM and one row's loads and stores run beside another's arithmetic). Maximum and sums meet
// through the cluster's shared memory, the gradient takes the logits' place there and leaves by a bulk store. Each pass then costs one power
// of two per element where one exponent serves both softmaxes, or where the temperature is 2, 3 or 4 and c is a power of q by multiplication
// (kPower2 to kPower4); two otherwise.
//
// 1024 rows of 128256 with 64 entries (525 MB, 80 us at the copy's rate), cold: 135 us with one exponent, 141, 148 and 145 with its square, third and
// fourth power, 184 with two. Two exponents keep the pipe for powers of two busy for 78% of the time. The others wait in turn on
// instructions (half of all slots) and on memory. 4096 rows at temperature 2: 484 us for 2.1 GB, 4.4 TB/s. Entries are compared with all
// others for equal ids: with 1024 of them 1024 rows take 3.2 ms.
#include "gemm_host.h"
#include "sm100.cuh"
#include "rows.cuh"

namespace b200 {
namespace distill {

using namespace rows;

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxEntries = 1024;
constexpr int kMaxCluster = 8;
constexpr int kSlice = 16384;      // elements of a slice, as long as a cluster of eight can hold the row
constexpr int kMaxSlice = 104 * 1024;
// Scores are scaled by 1 / tau before their maximum is taken off, in fp32: below kMinTau the rounding of that maximum shows (logits of 100: 1e-3
// of a probability). The divergence is of the size of 1 / tau^2 and multiplied by tau^2: above kMaxTau little is left of it.
constexpr float kMinTau = 0.01f, kMaxTau = 100.f;
constexpr int kErrLoad = 31, kErrMeet = 32;

struct Args {
  const __nv_bfloat16* z;
  __nv_bfloat16* grad;   // may be z
  const long long* targets;
  const void* ids;       // [T, K] int64 or int32
  const void* values;    // [T, K] fp32 or bf16
  float* loss;
  long long zStride, gradStride;
  int V, K, idBytes, valueBytes, slice;
  bool zBulk, gradBulk;  // rows start on 16-byte boundaries
  float a, tau, gradScale;
  int* err;
};

// One: a single exponent (temperature one, or one of the two losses alone). Power: c = q^2, q^3 or q^4, by the compiler's knowledge: with the
// power looked up in the loops, 4096 rows of 128256 at temperature 2 took 542 us where they then took 479. Two: both.
enum Mode { kOne, kTwo, kPower2, kPower3, kPower4 };

// Over the block; `sh` (a float per warp) is used once in a kernel.
__device__ __forceinline__ float blockMax(float v, float* sh) {
  v = laneMax<32>(v);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  return laneMax<32>(sh[(threadIdx.x & 31) % kWarps]);
}
__device__ __forceinline__ float2 blockSum(float2 v, float2* sh) {
  v.x = laneSum<32>(v.x);
  v.y = laneSum<32>(v.y);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  v = (threadIdx.x & 31) < kWarps ? sh[threadIdx.x & 31] : make_float2(0.f, 0.f);
  return make_float2(laneSum<32>(v.x), laneSum<32>(v.y));
}

__device__ __forceinline__ float teacherValue(const Args& p, size_t row, int k) {
  return (p.valueBytes == 4 ? reinterpret_cast<const float*>(p.values)[row * p.K + k] : toFloat(reinterpret_cast<const __nv_bfloat16*>(p.values)[row * p.K + k])) / p.tau;
}

template <Mode MODE>
__global__ void __launch_bounds__(kThreads, 6) distillKernel(const Args p, int ctas) {
  using namespace sm100;
  extern __shared__ __align__(128) uint8_t smem[];
  __nv_bfloat16* x = reinterpret_cast<__nv_bfloat16*>(smem);
  int* id = reinterpret_cast<int*>(smem + (size_t)p.slice * 2);
  float* prob = reinterpret_cast<float*>(id + p.K);
  float* zAt = prob + p.K;
  __shared__ float tops[kWarps];
  __shared__ float2 sums[kWarps];
  __shared__ float4 meet[kMaxCluster];            // of the cluster's CTAs: maximum, sums relative to it
  __shared__ float teacher[4];                    // largest value, logarithm of the sum, 1 if there are entries; the target's logit
  __shared__ uint64_t bar, met;

  const size_t row = blockIdx.x / ctas;
  const int rank = blockIdx.x % ctas, lane = threadIdx.x & 31;
  const int first = rank * p.slice, n = max(0, min(p.slice, p.V - first)), nvec = n >> 3;
  const __nv_bfloat16* z = p.z + row * p.zStride;
  __nv_bfloat16* grad = p.grad + row * p.gradStride;
  const bool bulk = p.zBulk && nvec > 0;
  if (threadIdx.x == 0) {
    mbarInit(&bar, 1);
    mbarInit(&met, 1);
    fenceBarrierInit();
    mbarArriveExpectTx(&met, ctas * sizeof(float4));
    if (bulk) {
      mbarArriveExpectTx(&bar, nvec * 16);
      bulkLoad(x, z + first, nvec * 16, &bar);
    }
  }
  __syncthreads();
  clusterArriveRelaxed();  // waited for before the first store into another CTA
  const long long target = p.targets[row];
  const bool counts = target >= 0 && target < p.V;  // for all CTAs of the cluster alike
  for (int j = (p.zBulk ? nvec * 8 : 0) + threadIdx.x; j < n; j += kThreads) x[j] = z[first + j];

  // What the teacher says, in every CTA, while the slice is on its way.
  if (counts) {
    for (int k = threadIdx.x; k < p.K; k += kThreads) {
      const long long i = p.idBytes == 8 ? reinterpret_cast<const long long*>(p.ids)[row * p.K + k] : (long long)reinterpret_cast<const int*>(p.ids)[row * p.K + k];
      const bool exists = i >= 0 && i < p.V && p.a > 0.f;
      id[k] = exists ? (int)i : -1;
      prob[k] = exists ? teacherValue(p, row, k) : -INFINITY;
      zAt[k] = exists ? __bfloat162float(z[i]) : 0.f;
    }
    if (threadIdx.x == kThreads - 1) teacher[3] = __bfloat162float(z[target]);
  }
  if (bulk) mbarWait(&bar, 0, p.err, kErrLoad);  // given up or not, the CTA stays: its cluster writes into it
  if (!counts) {
    if (rank == 0 && threadIdx.x == 0) p.loss[row] = 0.f;
    if (p.gradBulk)
      for (int j = threadIdx.x; j < nvec; j += kThreads) reinterpret_cast<uint4*>(grad + first)[j] = make_uint4(0, 0, 0, 0);
    for (int j = (p.gradBulk ? nvec * 8 : 0) + threadIdx.x; j < n; j += kThreads) grad[first + j] = __float2bfloat16(0.f);
    clusterWait();
    return;
  }
  __syncthreads();  // plainly loaded elements and the teacher's entries are in shared memory

  // ---- the slice's maximum
  uint4* xv = reinterpret_cast<uint4*>(x);
  __nv_bfloat162 top2 = __float2bfloat162_rn(-INFINITY);
  for (int j = threadIdx.x; j < nvec; j += kThreads) {
    const uint4 raw = xv[j];
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&raw);
    top2 = __hmax2(top2, __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
  }
  float m = fmaxf(__low2float(top2), __high2float(top2));
  for (int j = nvec * 8 + threadIdx.x; j < n; j += kThreads) m = fmaxf(m, __bfloat162float(x[j]));
  m = blockMax(m, tops);

  if (threadIdx.x < 32) {  // the teacher's softmax, by one warp from shared memory
    float best = -INFINITY, norm = 0.f;
    for (int k = lane; k < p.K; k += 32) best = fmaxf(best, prob[k]);
    best = laneMax<32>(best);
    // Entries of minus infinity have no weight, also where nothing is larger; a value that is not a number (the maximum passes over it) shows.
    for (int k = lane; k < p.K; k += 32)
      if (id[k] >= 0 && prob[k] != -INFINITY) norm += exp2Fast((prob[k] - best) * kLog2e);
    norm = laneSum<32>(norm);
    const float logNorm = logf(norm);
    for (int k = lane; k < p.K; k += 32) prob[k] = id[k] >= 0 && prob[k] != -INFINITY ? exp2Fast((prob[k] - best - logNorm) * kLog2e) : 0.f;
    if (lane == 0) teacher[0] = best, teacher[1] = logNorm, teacher[2] = norm == 0.f ? 0.f : 1.f;
  }

  // ---- the slice's sums, relative to its own maximum: one exchange with the cluster is enough
  const float soft = MODE == kOne && p.a == 0.f ? kLog2e : kLog2e / p.tau, one = kLog2e;
  const F2 soft2 = makeF2(soft, soft), one2 = makeF2(one, one);
  // Exponents are v soft + off with off = -(top soft) rounded, so that each is (v - top) soft and, for all of a slice alike, what that rounding took.
  // It is taken out of the sums again: of 100 / 0.01 in powers of two it is up to 2^-11.
  F2 offSoft, offOne;
  float tookSoft, tookOne;
  constexpr float kPower = MODE == kPower2 ? 2.f : MODE == kPower3 ? 3.f : 4.f;
  const auto relativeTo = [&](float top) {
    offSoft = makeF2(-top * soft, -top * soft);
    offOne = makeF2(-top * one, -top * one);
    tookSoft = fmaf(top, soft, -top * soft);
    tookOne = MODE >= kPower2 ? kPower * tookSoft : MODE == kTwo ? fmaf(top, one, -top * one) : tookSoft;
  };
  const auto powers = [&](F2 v, F2& q, F2& c) {
    q = exp2F2(fmaF2(v, soft2, offSoft));
    if constexpr (MODE >= kPower2) {
      c = mulF2(q, q);
      if constexpr (MODE == kPower3) c = mulF2(c, q);
      if constexpr (MODE == kPower4) c = mulF2(c, c);
    } else if constexpr (MODE == kTwo) {
      c = exp2F2(fmaF2(v, one2, offOne));
    } else {
      c = q;
    }
  };
  relativeTo(m == -INFINITY ? 0.f : m);  // nothing but minus infinity in this slice: sums of zero
  F2 partSoft = makeF2(0.f, 0.f), partOne = partSoft;
  for (int j = threadIdx.x; j < nvec; j += kThreads) {
    const uint4 raw = xv[j];
    F2 q[4], c[4];
    powers(unpackF2(raw.x), q[0], c[0]);
    powers(unpackF2(raw.y), q[1], c[1]);
    powers(unpackF2(raw.z), q[2], c[2]);
    powers(unpackF2(raw.w), q[3], c[3]);
    partSoft = addF2(partSoft, addF2(addF2(q[0], q[1]), addF2(q[2], q[3])));
    if (MODE != kOne) partOne = addF2(partOne, addF2(addF2(c[0], c[1]), addF2(c[2], c[3])));
  }
  for (int j = nvec * 8 + threadIdx.x; j < n; j += kThreads) {
    F2 q, c;
    powers(makeF2(__bfloat162float(x[j]), -INFINITY), q, c);
    partSoft = addF2(partSoft, q);
    partOne = addF2(partOne, c);
  }
  float sumSoft, sumOne, upper, upperOne;
  splitF2(partSoft, sumSoft, upper);
  splitF2(partOne, sumOne, upperOne);
  float2 both = blockSum(make_float2(sumSoft + upper, sumOne + upperOne), sums);
  both.x *= exp2f(-tookSoft);
  both.y *= exp2f(-tookOne);
  // Each CTA tells all of them, and goes on when all have told it: then they have also read the logits that they look up, which the gradient
  // may be about to take the place of.
  clusterWait();
  if (threadIdx.x < ctas) storeAsync4(mapToCta(smemAddr(&meet[rank]), threadIdx.x), m, both.x, both.y, 0.f, mapToCta(smemAddr(&met), threadIdx.x));
  mbarWait(&met, 0, p.err, kErrMeet);
  m = -INFINITY;
  for (int r = 0; r < ctas; r++) m = fmaxf(m, meet[r].x);
  sumSoft = sumOne = 0.f;
  for (int r = 0; r < ctas; r++) {
    const float d = meet[r].x - m;
    if (meet[r].y == 0.f) continue;  // nothing but minus infinity in this slice
    sumSoft += meet[r].y * exp2Fast(d * soft);
    sumOne += meet[r].z * exp2Fast(d * one);
  }
  if (MODE == kOne) sumOne = sumSoft;
  relativeTo(m);
  // The gradient's powers have the row's own rounding in them, so its factors have the sums with it.
  const float gradSoft = sumSoft * exp2f(tookSoft), gradOne = sumOne * exp2f(tookOne);
  const float a = teacher[2] == 0.f ? 0.f : p.a;

  // ---- the gradient, in the logits' place
  const float fOne = p.a < 1.f ? (1.f - p.a) / gradOne * p.gradScale : 0.f, fSoft = a == 0.f ? 0.f : a * p.tau / gradSoft * p.gradScale;
  const F2 fOne2 = makeF2(fOne, fOne), fSoft2 = MODE == kOne ? makeF2(fOne + fSoft, fOne + fSoft) : makeF2(fSoft, fSoft);
  const auto dense = [&](F2 v) {
    F2 q, c;
    powers(v, q, c);
    if constexpr (MODE == kOne) return mulF2(fSoft2, q);
    if constexpr (MODE == kPower2) return mulF2(q, fmaF2(fOne2, q, fSoft2));
    return fmaF2(fOne2, c, mulF2(fSoft2, q));
  };
  for (int j = threadIdx.x; j < nvec; j += kThreads) {
    const uint4 raw = xv[j];
    xv[j] = make_uint4(pack2(dense(unpackF2(raw.x))), pack2(dense(unpackF2(raw.y))), pack2(dense(unpackF2(raw.z))), pack2(dense(unpackF2(raw.w))));
  }
  const auto denseOne = [&](float v) {
    float lo, hi;
    splitF2(dense(makeF2(v, v)), lo, hi);
    return lo;
  };
  for (int j = nvec * 8 + threadIdx.x; j < n; j += kThreads) x[j] = __float2bfloat16(denseOne(__bfloat162float(x[j])));
  __syncthreads();
  // The teacher's entries and the target once more, from their logits in 32 bits. An id's first entry writes for all of them.
  for (int k = threadIdx.x; k <= p.K; k += kThreads) {
    const int v = k < p.K ? id[k] : (int)target;
    if (v < first || v >= first + n) continue;
    float mass = 0.f;
    bool again = false;
    for (int o = 0; o < p.K; o++)
      if (id[o] == v) {
        mass += prob[o];
        again = again || o < k;
      }
    const float at = k < p.K ? zAt[k] : teacher[3];
    if (!again) x[v - first] = __float2bfloat16(denseOne(at) - p.gradScale * (a * p.tau * mass + (v == target ? 1.f - p.a : 0.f)));
  }
  fenceProxyAsync();
  __syncthreads();
  if (p.gradBulk) {
    for (int j = nvec * 8 + threadIdx.x; j < n; j += kThreads) grad[first + j] = x[j];
    if (threadIdx.x == 0 && nvec > 0) {
      bulkStore(grad + first, x, nvec * 16);
      tmaStoreCommit();
    }
  } else {
    for (int j = threadIdx.x; j < n; j += kThreads) grad[first + j] = x[j];
  }

  // ---- the loss, while the gradient leaves
  if (rank == 0 && threadIdx.x < 32) {
    const float logSoft = logf(sumSoft);
    float kl = 0.f;
    for (int k = lane; k < p.K; k += 32)
      if (prob[k] != 0.f) kl += prob[k] * ((teacherValue(p, row, k) - teacher[0] - teacher[1]) - ((zAt[k] - m) / p.tau - logSoft));
    kl = laneSum<32>(kl);
    if (lane == 0) {
      float loss = a == 0.f ? 0.f : a * p.tau * p.tau * kl;
      if (p.a < 1.f) loss += (1.f - p.a) * ((m - teacher[3]) + logf(sumOne));
      p.loss[row] = loss;
    }
  }
  if (threadIdx.x == 0) tmaStoreWaitRead0();
}

template <Mode MODE> cudaError_t launch(const Args& p, long long T, int ctas, size_t smem, cudaStream_t s) {
  static bool done[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !done[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(distillKernel<MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, 2 * kMaxSlice + 12 * kMaxEntries);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) done[dev] = true;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(T * ctas));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute cluster{};
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = ctas;
  cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
  cfg.attrs = &cluster;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, distillKernel<MODE>, p, ctas);
}

}  // namespace distill
}  // namespace b200

extern "C" {

// Rows of logits [T, V] bf16 (row stride in elements) and of grad (the same buffer and stride, or another); targets int64 [T];
// ids [T, K] int64 (idBytes 8) or int32 (4); values [T, K] fp32 (valueBytes 4) or bf16 (2); loss fp32 [T]. V up to 851,968, K up to 1024.
int b200ops_distill_loss(const void* logits, void* grad, const long long* targets, const void* ids, int idBytes, const void* values, int valueBytes, float* loss,
                         long long T, int V, int K, long long stride, long long gradStride, float a, float tau, float gradScale, cudaStream_t s) {
  using namespace b200::distill;
  if (T < 0 || V <= 0 || V > kMaxCluster * kMaxSlice || K <= 0 || K > kMaxEntries || !(tau >= kMinTau && tau <= kMaxTau) || !(a >= 0.f && a <= 1.f) || stride < V || gradStride < V ||
      (idBytes != 4 && idBytes != 8) || (valueBytes != 2 && valueBytes != 4) || (((uintptr_t)logits | (uintptr_t)grad) & 1))
    return (int)cudaErrorInvalidValue;
  if (T == 0) return 0;
  int ctas = 1;
  while (ctas < kMaxCluster && (long long)ctas * kSlice < V) ctas *= 2;
  if (T * ctas > 0x7fffffffLL) return (int)cudaErrorInvalidValue;
  Args p{};
  p.z = (const __nv_bfloat16*)logits;
  p.grad = (__nv_bfloat16*)grad;
  p.targets = targets;
  p.ids = ids;
  p.values = values;
  p.loss = loss;
  p.zStride = stride;
  p.gradStride = gradStride;
  p.V = V, p.K = K, p.idBytes = idBytes, p.valueBytes = valueBytes;
  p.slice = ((V + ctas - 1) / ctas + 63) / 64 * 64;
  p.zBulk = ((uintptr_t)logits & 15) == 0 && (stride % 8 == 0 || T == 1);
  p.gradBulk = ((uintptr_t)grad & 15) == 0 && (gradStride % 8 == 0 || T == 1);
  p.a = a, p.tau = tau, p.gradScale = gradScale;
  p.err = b200::gemm::errWord();
  if (!p.err) return (int)cudaErrorMemoryAllocation;
  const size_t smem = (size_t)p.slice * 2 + (size_t)K * 12;
  if (tau == 1.f || a == 0.f || a == 1.f) return (int)launch<kOne>(p, T, ctas, smem, s);
  if (tau == 2.f) return (int)launch<kPower2>(p, T, ctas, smem, s);
  if (tau == 3.f) return (int)launch<kPower3>(p, T, ctas, smem, s);
  if (tau == 4.f) return (int)launch<kPower4>(p, T, ctas, smem, s);
  return (int)launch<kTwo>(p, T, ctas, smem, s);
}

}  // extern "C"
