// Per-head RMSNorm of queries and keys and the rotation to their positions (rotate-half convention), one pass each way over the packed
// projection [tokens, heads + 2 kvHeads, D]:
//   forward   n = x r w with r = 1 / sqrt(mean(x^2) + eps) over a head's D elements; (y_a, y_b) = (n_a c - n_b s, n_b c + n_a s) for the pairs
//             (j, j + D / 2) and the table's (c, s) of the token's position. Value heads are left where they are.
//   backward  g = the inverse rotation of dy; dx = r (g w - x r^2 mean(g w x)), dw = sum over rows of g x r. r is formed again from x, which
//             has to be read anyway. The values' gradient is copied beside them, so that one launch writes the whole packed gradient.
//
// A head's row belongs to 8, 16 or 32 lanes; lane j holds elements [4j, 4j + 4) and their partners at + D / 2, so the rotation needs no
// exchange and the sums take three to five shuffles. A warp stays with one token, whose cosines and sines it keeps in registers, and walks a
// share of its heads.
// Both directions are bound by memory traffic.
#include "rows.cuh"

namespace b200 {
namespace qkn {

using namespace rows;

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kUnroll = 4, kUnrollBack = 2;  // rows of a lane whose loads are under way together
constexpr int kCtasPerSm = 2;                // backward

struct Shape {
  long long tokens;  // batch * seq
  int seq, heads, kv, D;
  int split;         // warps that share a token's heads
  float eps;
};
// Element strides of a gradient [batch, heads, seq, D] whose last dimension is dense.
struct Grad {
  const __nv_bfloat16* p;
  long long b, h, s;
  __device__ const __nv_bfloat16* at(long long batch, int head, int pos) const { return p + batch * b + head * h + pos * s; }
};

template <int LANES, typename W>
__global__ void __launch_bounds__(kThreads) forwardKernel(const __nv_bfloat16* __restrict__ x, const W* __restrict__ wq, const W* __restrict__ wk,
                                                          const float2* __restrict__ table, __nv_bfloat16* __restrict__ q, __nv_bfloat16* __restrict__ k, Shape sh) {
  constexpr int kGroups = 32 / LANES;
  const int lane = threadIdx.x & 31, j = lane % LANES, group = lane / LANES;
  const int half = sh.D >> 1, rot = sh.heads + sh.kv, all = rot + sh.kv;
  const bool in = 8 * j < sh.D;
  const uint32_t item = blockIdx.x * kWarps + (threadIdx.x >> 5), t = item / (uint32_t)sh.split;
  if (t >= sh.tokens) return;
  const int part = item - t * sh.split;
  float w[2][8];
  float2 cs[4] = {};
  if (in) {
#pragma unroll
    for (int e = 0; e < 4; e++) {
      w[0][e] = toFloat(wq[4 * j + e]);
      w[0][4 + e] = toFloat(wq[half + 4 * j + e]);
      w[1][e] = toFloat(wk[4 * j + e]);
      w[1][4 + e] = toFloat(wk[half + 4 * j + e]);
      cs[e] = table[(size_t)(t % (uint32_t)sh.seq) * half + 4 * j + e];
    }
  }
  const int step = sh.split * kGroups;
  for (int h0 = part * kGroups + group; h0 - group < rot; h0 += kUnroll * step) {
    uint2 raw[kUnroll][2];
#pragma unroll
    for (int u = 0; u < kUnroll; u++) {
      const int h = h0 + u * step;
      raw[u][0] = raw[u][1] = make_uint2(0, 0);
      if (in && h < rot) {
        const __nv_bfloat16* row = x + ((size_t)t * all + h) * sh.D + 4 * j;
        raw[u][0] = *reinterpret_cast<const uint2*>(row);
        raw[u][1] = *reinterpret_cast<const uint2*>(row + half);
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; u++) {
      const int h = h0 + u * step;
      float a[4], b[4];
      unpack4(raw[u][0], a);
      unpack4(raw[u][1], b);
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 4; e++) ss += a[e] * a[e] + b[e] * b[e];
      const float r = rsqrtf(laneSum<LANES>(ss) / (float)sh.D + sh.eps);
      if (in && h < rot) {
        const int which = h >= sh.heads;
        float ya[4], yb[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const float na = a[e] * r * (which ? w[1][e] : w[0][e]), nb = b[e] * r * (which ? w[1][4 + e] : w[0][4 + e]);
          ya[e] = na * cs[e].x - nb * cs[e].y;
          yb[e] = nb * cs[e].x + na * cs[e].y;
        }
        __nv_bfloat16* out = (which ? k + ((size_t)t * sh.kv + h - sh.heads) * sh.D : q + ((size_t)t * sh.heads + h) * sh.D) + 4 * j;
        *reinterpret_cast<uint2*>(out) = pack4(ya);
        *reinterpret_cast<uint2*>(out + half) = pack4(yb);
      }
    }
  }
}

// partials [CTAs][2][D]: every CTA's share of the weights' gradients, summed by weightSum in a fixed order.
template <int LANES, typename W>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) backwardKernel(Grad dq, Grad dk, Grad dv, const __nv_bfloat16* __restrict__ x, const W* __restrict__ wq,
                                                           const W* __restrict__ wk, const float2* __restrict__ table, __nv_bfloat16* __restrict__ dx,
                                                           float* __restrict__ partials, Shape sh) {
  constexpr int kGroups = 32 / LANES;
  __shared__ float part[kWarps][2][8 * LANES];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, j = lane % LANES, group = lane / LANES;
  const int half = sh.D >> 1, rot = sh.heads + sh.kv, all = rot + sh.kv;
  const bool in = 8 * j < sh.D;
  float w[2][8] = {}, dw[2][8] = {};
  if (in) {
#pragma unroll
    for (int e = 0; e < 4; e++) {
      w[0][e] = toFloat(wq[4 * j + e]);
      w[0][4 + e] = toFloat(wq[half + 4 * j + e]);
      w[1][e] = toFloat(wk[4 * j + e]);
      w[1][4 + e] = toFloat(wk[half + 4 * j + e]);
    }
  }
  const uint32_t items = (uint32_t)sh.tokens * sh.split;
  for (uint32_t item = blockIdx.x * kWarps + warp; item < items; item += gridDim.x * kWarps) {
    const uint32_t t = item / (uint32_t)sh.split, batch = t / (uint32_t)sh.seq;
    const int pos = t - batch * sh.seq;
    float2 cs[4] = {};
    if (in)
#pragma unroll
      for (int e = 0; e < 4; e++) cs[e] = table[(size_t)pos * half + 4 * j + e];
    const int step = sh.split * kGroups;
    for (int h0 = (item - t * sh.split) * kGroups + group; h0 - group < all; h0 += kUnrollBack * step) {
      uint2 grad[kUnrollBack][2], row[kUnrollBack][2];
#pragma unroll
      for (int u = 0; u < kUnrollBack; u++) {
        const int h = h0 + u * step;
        grad[u][0] = grad[u][1] = row[u][0] = row[u][1] = make_uint2(0, 0);
        if (in && h < all) {
          const __nv_bfloat16* g = (h < sh.heads ? dq.at(batch, h, pos) : h < rot ? dk.at(batch, h - sh.heads, pos) : dv.at(batch, h - rot, pos)) + 4 * j;
          grad[u][0] = *reinterpret_cast<const uint2*>(g);
          grad[u][1] = *reinterpret_cast<const uint2*>(g + half);
          if (h < rot) {
            const __nv_bfloat16* p = x + ((size_t)t * all + h) * sh.D + 4 * j;
            row[u][0] = *reinterpret_cast<const uint2*>(p);
            row[u][1] = *reinterpret_cast<const uint2*>(p + half);
          }
        }
      }
#pragma unroll
      for (int u = 0; u < kUnrollBack; u++) {
        const int h = h0 + u * step;
        const bool key = h >= sh.heads, rotated = h < rot;  // (values: all sums below are zeros)
        float a[4], b[4], ya[4], yb[4], ga[4], gb[4], wa[4], wb[4];
        unpack4(row[u][0], a);
        unpack4(row[u][1], b);
        unpack4(grad[u][0], ya);
        unpack4(grad[u][1], yb);
        float ss = 0.f, dot = 0.f;
#pragma unroll
        for (int e = 0; e < 4; e++) {
          ga[e] = ya[e] * cs[e].x + yb[e] * cs[e].y;
          gb[e] = yb[e] * cs[e].x - ya[e] * cs[e].y;
          wa[e] = key ? w[1][e] : w[0][e];
          wb[e] = key ? w[1][4 + e] : w[0][4 + e];
          ss += a[e] * a[e] + b[e] * b[e];
          dot += ga[e] * wa[e] * a[e] + gb[e] * wb[e] * b[e];
        }
        const float r = rsqrtf(laneSum<LANES>(ss) / (float)sh.D + sh.eps);
        const float c = laneSum<LANES>(dot) * r * r / (float)sh.D;
        if (in && h < all) {
          if (rotated) {
            float oa[4], ob[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
              oa[e] = r * (ga[e] * wa[e] - a[e] * c);
              ob[e] = r * (gb[e] * wb[e] - b[e] * c);
              const float da = ga[e] * a[e] * r, db = gb[e] * b[e] * r;
              dw[0][e] += key ? 0.f : da;
              dw[0][4 + e] += key ? 0.f : db;
              dw[1][e] += key ? da : 0.f;
              dw[1][4 + e] += key ? db : 0.f;
            }
            grad[u][0] = pack4(oa);
            grad[u][1] = pack4(ob);
          }
          __nv_bfloat16* out = dx + ((size_t)t * all + h) * sh.D + 4 * j;
          *reinterpret_cast<uint2*>(out) = grad[u][0];
          *reinterpret_cast<uint2*>(out + half) = grad[u][1];
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 2; i++)
#pragma unroll
    for (int e = 0; e < 8; e++) {
      float v = dw[i][e];
#pragma unroll
      for (int o = LANES; o < 32; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
      if (group == 0) part[warp][i][8 * j + e] = v;
    }
  __syncthreads();
  for (int c = threadIdx.x; c < 2 * sh.D; c += kThreads) {
    const int i = c / sh.D, d = c % sh.D;
    const int hi = d >= half, dd = hi ? d - half : d;
    const int slot = 8 * (dd >> 2) + 4 * hi + (dd & 3);
    float v = 0.f;
#pragma unroll
    for (int wp = 0; wp < kWarps; wp++) v += part[wp][i][slot];
    partials[(size_t)blockIdx.x * 2 * sh.D + c] = v;
  }
}

// The weights' gradients [2][D] from the CTAs' shares: 32 columns per CTA, 32 row groups that meet in shared memory.
template <typename W>
__global__ void __launch_bounds__(1024) weightSum(const float* __restrict__ partials, W* __restrict__ dwq, W* __restrict__ dwk, int rows, int D) {
  __shared__ float sh[32][33];
  const int cx = threadIdx.x & 31, g = threadIdx.x >> 5, c = blockIdx.x * 32 + cx;
  float acc = 0.f;
  if (c < 2 * D)
#pragma unroll 4
    for (int r = g; r < rows; r += 32) acc += partials[(size_t)r * 2 * D + c];
  sh[g][cx] = acc;
  __syncthreads();
  if (g == 0 && c < 2 * D) {
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < 32; i++) v += sh[i][cx];
    if (c < D) store(dwq + c, v);
    else store(dwk + c - D, v);
  }
}

int smCount() {
  static int n[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return 148;
  if (!n[dev]) cudaDeviceGetAttribute(&n[dev], cudaDevAttrMultiProcessorCount, dev);
  return n[dev] ? n[dev] : 148;
}

// Warps that share a token's heads: one, unless there are too few tokens to give every SM 32 warps.
int splitFor(long long tokens, int heads, int groups) {
  const long long want = 32LL * smCount(), most = (heads + groups - 1) / groups;
  long long s = (want + tokens - 1) / tokens;
  return (int)(s < 1 ? 1 : s > most ? most : s);
}

template <int LANES, typename W>
cudaError_t forward(const void* x, const void* wq, const void* wk, const float* table, void* q, void* k, Shape sh, cudaStream_t s) {
  sh.split = splitFor(sh.tokens, sh.heads + sh.kv, 32 / LANES);
  const long long ctas = (sh.tokens * sh.split + kWarps - 1) / kWarps;
  if (ctas * kWarps > 0x7fffffffLL) return cudaErrorInvalidValue;
  forwardKernel<LANES, W><<<(unsigned)ctas, kThreads, 0, s>>>((const __nv_bfloat16*)x, (const W*)wq, (const W*)wk, (const float2*)table, (__nv_bfloat16*)q,
                                                             (__nv_bfloat16*)k, sh);
  return cudaGetLastError();
}

template <int LANES, typename W>
cudaError_t backward(Grad dq, Grad dk, Grad dv, const void* x, const void* wq, const void* wk, const float* table, void* dx, float* partials, void* dwq, void* dwk,
                     Shape sh, cudaStream_t s) {
  sh.split = splitFor(sh.tokens, sh.heads + 2 * sh.kv, 32 / LANES);
  const long long need = (sh.tokens * sh.split + kWarps - 1) / kWarps;
  if (need * kWarps > 0x3fffffffLL) return cudaErrorInvalidValue;
  const int ctas = (int)(need < kCtasPerSm * smCount() ? need : kCtasPerSm * smCount());
  backwardKernel<LANES, W><<<ctas, kThreads, 0, s>>>(dq, dk, dv, (const __nv_bfloat16*)x, (const W*)wq, (const W*)wk, (const float2*)table, (__nv_bfloat16*)dx, partials, sh);
  weightSum<W><<<(2 * sh.D + 31) / 32, 1024, 0, s>>>(partials, (W*)dwq, (W*)dwk, ctas, sh.D);
  return cudaGetLastError();
}

bool good(const Shape& sh) { return sh.tokens >= 0 && sh.seq > 0 && sh.heads > 0 && sh.kv > 0 && sh.D >= 8 && sh.D <= 256 && sh.D % 8 == 0; }

}  // namespace qkn
}  // namespace b200

using namespace b200::qkn;

extern "C" {

// x [batch * seq, heads + 2 kv, D] bf16; q [batch * seq, heads, D], k [batch * seq, kv, D]; weights [D] fp32 or bf16 (wBf16); table
// [>= seq, D / 2] (cos, sin).
int b200ops_qk_norm_rope_fwd(const void* x, const void* wq, const void* wk, int wBf16, const float* table, void* q, void* k, long long tokens, int seq, int heads,
                             int kv, int D, float eps, cudaStream_t s) {
  const Shape sh{tokens, seq, heads, kv, D, 1, eps};
  if (!good(sh)) return (int)cudaErrorInvalidValue;
  if (tokens == 0) return 0;
  const auto go = [&](auto lanes) {
    constexpr int L = decltype(lanes)::value;
    return (int)(wBf16 ? forward<L, __nv_bfloat16>(x, wq, wk, table, q, k, sh, s) : forward<L, float>(x, wq, wk, table, q, k, sh, s));
  };
  return D <= 64 ? go(std::integral_constant<int, 8>{}) : D <= 128 ? go(std::integral_constant<int, 16>{}) : go(std::integral_constant<int, 32>{});
}

// fp32 words of scratch for the backward call.
long long b200ops_qk_norm_rope_bwd_scratch(int D) { return (long long)kCtasPerSm * smCount() * 2 * D; }

// strides: batch, head and position strides (elements, multiples of 4) of dq, dk, dv in turn. dx like x; dwq, dwk [D] of the weights' type.
int b200ops_qk_norm_rope_bwd(const void* dq, const void* dk, const void* dv, const long long* strides, const void* x, const void* wq, const void* wk, int wBf16,
                             const float* table, void* dx, float* scratch, void* dwq, void* dwk, long long tokens, int seq, int heads, int kv, int D, float eps,
                             cudaStream_t s) {
  const Shape sh{tokens, seq, heads, kv, D, 1, eps};
  if (!good(sh) || tokens == 0) return (int)cudaErrorInvalidValue;
  const auto grad = [&](const void* p, int i) { return Grad{(const __nv_bfloat16*)p, strides[3 * i], strides[3 * i + 1], strides[3 * i + 2]}; };
  const auto go = [&](auto lanes) {
    constexpr int L = decltype(lanes)::value;
    return (int)(wBf16 ? backward<L, __nv_bfloat16>(grad(dq, 0), grad(dk, 1), grad(dv, 2), x, wq, wk, table, dx, scratch, dwq, dwk, sh, s)
                       : backward<L, float>(grad(dq, 0), grad(dk, 1), grad(dv, 2), x, wq, wk, table, dx, scratch, dwq, dwk, sh, s));
  };
  return D <= 64 ? go(std::integral_constant<int, 8>{}) : D <= 128 ? go(std::integral_constant<int, 16>{}) : go(std::integral_constant<int, 32>{});
}

}  // extern "C"
