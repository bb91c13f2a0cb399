// Per-head RMSNorm of queries and keys and the rotation to their positions (rotate-half convention), one pass each way over the packed
// projection [tokens, heads + 2 kvHeads, D]:
//   forward   n = x r w with r = 1 / sqrt(mean(x^2) + eps) over a head's D elements; (y_a, y_b) = (n_a c - n_b s, n_b c + n_a s) for the pairs
//             (j, j + D / 2) and the table's (c, s) of the token's position. Value heads are left where they are.
//   backward  g = the inverse rotation of dy; dx = r (g w - x r^2 mean(g w x)), dw = sum over rows of g x r. r is formed again from x, which
//             has to be read anyway. The values' gradient is copied beside them, so that one launch writes the whole packed gradient.
//
// A head's row belongs to 8, 16 or 32 lanes; lane j holds elements [4j, 4j + 4) and their partners at + D / 2, so the rotation needs no
// exchange and the sums take three to five shuffles. A warp stays with a few heads of one kind, whose weights (and the sums of their
// gradients) it keeps in registers, and goes from token to token. Forward, the rows of four heads per lane group are loaded together;
// backward, where a row needs twice the registers, rows travel through shared memory, six tokens deep (a row at a time: 59 us).
//
// 4096 tokens, 32 + 8 + 8 heads of 128: forward 20 us for 84 MB (4.2 TB/s), backward 47 us for 142 MB (3.0 TB/s) and 3 for the weights' sums; with
// fp32 weights 23, 47 and 3. The backward pass fills neither memory nor the issue slots (half each; about 290 instructions per pair of rows):
// with a quarter of an SM's warps, each waits for its token's row of the table.
#include "rows.cuh"

#include <type_traits>

namespace b200 {
namespace qkn {

using namespace rows;

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kUnrollFwd = 4, kUnrollBwd = 2;  // rows of a lane that are dealt with together
constexpr int kStages = 6;                     // backward: tokens whose rows are on their way or in shared memory
constexpr int kCtasFwd = 3, kCtasBwd = 2;  // per SM

struct Shape {
  uint32_t tokens, seq;  // tokens = batch * seq
  int heads, kv, D;
  float eps;
};
// Element strides of a gradient [batch, heads, seq, D] whose last dimension is dense.
struct Grad {
  const __nv_bfloat16* p;
  long long b, h, s;
  __device__ const __nv_bfloat16* at(long long batch, int head, int pos) const { return p + batch * b + head * h + pos * s; }
};

// The heads that a warp stays with, and its tokens: kind 0 queries, 1 keys, 2 values.
template <int LANES, int kUnroll> struct Share {
  static constexpr int kHeads = 32 / LANES * kUnroll;
  int kind, first, end, before;  // heads [first, end) of the kind; heads of a token before the kind's
  uint32_t token, step;
  __host__ __device__ static int count(int heads, int kv, bool values) { return (heads + kHeads - 1) / kHeads + (values ? 2 : 1) * ((kv + kHeads - 1) / kHeads); }
  __device__ Share(const Shape& sh, bool values) {
    const uint32_t n = count(sh.heads, sh.kv, values), warp = blockIdx.x * kWarps + (threadIdx.x >> 5);
    const int nq = (sh.heads + kHeads - 1) / kHeads, nk = (sh.kv + kHeads - 1) / kHeads;
    step = gridDim.x * kWarps / n;
    token = warp / n;
    int c = warp - token * n;
    if (token >= step) token = sh.tokens;  // a warp that is left over
    kind = c < nq ? 0 : c < nq + nk ? 1 : 2;
    c -= kind == 0 ? 0 : kind == 1 ? nq : nq + nk;
    first = c * kHeads;
    end = min(first + kHeads, kind == 0 ? sh.heads : sh.kv);
    before = kind == 0 ? 0 : kind == 1 ? sh.heads : sh.heads + sh.kv;
  }
};

template <int LANES, typename W>
__global__ void __launch_bounds__(kThreads, kCtasFwd) forwardKernel(const __nv_bfloat16* __restrict__ x, const W* __restrict__ wq, const W* __restrict__ wk,
                                                                    const float2* __restrict__ table, __nv_bfloat16* __restrict__ q,
                                                                    __nv_bfloat16* __restrict__ k, Shape sh) {
  constexpr int kGroups = 32 / LANES;
  const int lane = threadIdx.x & 31, j = lane % LANES, group = lane / LANES, half = sh.D >> 1, all = sh.heads + 2 * sh.kv;
  const bool in = 8 * j < sh.D;
  const Share<LANES, kUnrollFwd> mine(sh, false);
  const W* w = mine.kind ? wk : wq;
  float wa[4] = {}, wb[4] = {};
  if (in)
#pragma unroll
    for (int e = 0; e < 4; e++) {
      wa[e] = toFloat(w[4 * j + e]);
      wb[e] = toFloat(w[half + 4 * j + e]);
    }
  __nv_bfloat16* const to = mine.kind ? k : q;
  const int toHeads = mine.kind ? sh.kv : sh.heads;
  for (uint32_t t = mine.token; t < sh.tokens; t += mine.step) {
    uint2 raw[kUnrollFwd][2];
#pragma unroll
    for (int u = 0; u < kUnrollFwd; u++) {
      const int h = mine.first + u * kGroups + group;
      raw[u][0] = raw[u][1] = make_uint2(0, 0);
      if (in && h < mine.end) {
        const __nv_bfloat16* row = x + ((size_t)t * all + mine.before + h) * sh.D + 4 * j;
        raw[u][0] = *reinterpret_cast<const uint2*>(row);
        raw[u][1] = *reinterpret_cast<const uint2*>(row + half);
      }
    }
    float2 cs[4] = {};
    if (in)
#pragma unroll
      for (int e = 0; e < 4; e++) cs[e] = table[(size_t)(t % sh.seq) * half + 4 * j + e];
#pragma unroll
    for (int u = 0; u < kUnrollFwd; u++) {
      const int h = mine.first + u * kGroups + group;
      float a[4], b[4];
      unpack4(raw[u][0], a);
      unpack4(raw[u][1], b);
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 4; e++) ss += a[e] * a[e] + b[e] * b[e];
      const float r = rsqrtf(laneSum<LANES>(ss) / (float)sh.D + sh.eps);
      if (in && h < mine.end) {
        float ya[4], yb[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const float na = a[e] * r * wa[e], nb = b[e] * r * wb[e];
          ya[e] = na * cs[e].x - nb * cs[e].y;
          yb[e] = nb * cs[e].x + na * cs[e].y;
        }
        __nv_bfloat16* out = to + ((size_t)t * toHeads + h) * sh.D + 4 * j;
        *reinterpret_cast<uint2*>(out) = pack4(ya);
        *reinterpret_cast<uint2*>(out + half) = pack4(yb);
      }
    }
  }
}

__device__ __forceinline__ void copyAsync16(void* smem, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(smem)), "l"(src) : "memory");
}

// partials [CTAs][2][D]: every CTA's share of the weights' gradients, summed by weightSum in a fixed order.
template <int LANES, typename W>
__global__ void __launch_bounds__(kThreads, kCtasBwd) backwardKernel(Grad dq, Grad dk, Grad dv, const __nv_bfloat16* __restrict__ x, const W* __restrict__ wq,
                                                                       const W* __restrict__ wk, const float2* __restrict__ table, __nv_bfloat16* __restrict__ dx,
                                                                       float* __restrict__ partials, Shape sh) {
  constexpr int kGroups = 32 / LANES;
  __shared__ float part[kWarps][8 * LANES];
  __shared__ int kinds[kWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, j = lane % LANES, group = lane / LANES, half = sh.D >> 1, all = sh.heads + 2 * sh.kv;
  const bool in = 8 * j < sh.D;
  const Share<LANES, kUnrollBwd> mine(sh, true);
  const W* w = mine.kind ? wk : wq;
  const Grad from = mine.kind == 0 ? dq : mine.kind == 1 ? dk : dv;
  float wa[4] = {}, wb[4] = {}, dwa[4] = {}, dwb[4] = {};
  if (in && mine.kind < 2)
#pragma unroll
    for (int e = 0; e < 4; e++) {
      wa[e] = toFloat(w[4 * j + e]);
      wb[e] = toFloat(w[half + 4 * j + e]);
    }
  // The rows of the next tokens are on their way into shared memory meanwhile: [stage][row][gradient, x] of this lane's group.
  extern __shared__ __align__(16) uint8_t ring[];
  constexpr uint32_t kRow = 16 * LANES, kStage = kUnrollBwd * 2 * kGroups * kRow;
  uint8_t* const rows = ring + warp * kStages * kStage + group * kRow;
  const __nv_bfloat16* const fromHead = from.p + (mine.first + group) * from.h + 8 * j;
  const __nv_bfloat16* const xHead = x + (size_t)(mine.before + mine.first + group) * sh.D + 8 * j;
  const auto fetch = [&](uint32_t t, int stage) {
    if (t < sh.tokens && in) {
      const uint32_t batch = t / sh.seq, pos = t - batch * sh.seq;
      const __nv_bfloat16* g = fromHead + batch * from.b + pos * from.s;
      const __nv_bfloat16* p = xHead + (size_t)t * all * sh.D;
#pragma unroll
      for (int u = 0; u < kUnrollBwd; u++)
        if (mine.first + u * kGroups + group < mine.end) {
          uint8_t* to = rows + stage * kStage + u * 2 * kGroups * kRow + 16 * j;
          copyAsync16(to, g + u * kGroups * from.h);
          if (mine.kind < 2) copyAsync16(to + kGroups * kRow, p + u * kGroups * sh.D);
        }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int n = 0; n < kStages - 1; n++) fetch(mine.token + n * mine.step, n);
  int stage = 0;
  for (uint32_t t = mine.token; t < sh.tokens; t += mine.step) {
    fetch(t + (kStages - 1) * mine.step, stage == 0 ? kStages - 1 : stage - 1);
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
    __syncwarp();
    float2 cs[4] = {};
    if (in && mine.kind < 2)
#pragma unroll
      for (int e = 0; e < 4; e++) cs[e] = table[(size_t)(t % sh.seq) * half + 4 * j + e];
#pragma unroll
    for (int u = 0; u < kUnrollBwd; u++) {
      const int h = mine.first + u * kGroups + group;
      const bool live = in && h < mine.end;
      const uint8_t* at = rows + stage * kStage + u * 2 * kGroups * kRow + 8 * j;
      uint2 ra = make_uint2(0, 0), rb = ra, xa = ra, xb = ra;
      if (live) {
        ra = *reinterpret_cast<const uint2*>(at);
        rb = *reinterpret_cast<const uint2*>(at + sh.D);
        if (mine.kind < 2) {
          xa = *reinterpret_cast<const uint2*>(at + kGroups * kRow);
          xb = *reinterpret_cast<const uint2*>(at + kGroups * kRow + sh.D);
        }
      }
      if (mine.kind < 2) {
        float a[4], b[4], ya[4], yb[4], ga[4], gb[4];
        unpack4(xa, a);
        unpack4(xb, b);
        unpack4(ra, ya);
        unpack4(rb, yb);
        float ss = 0.f, dot = 0.f;
#pragma unroll
        for (int e = 0; e < 4; e++) {
          ga[e] = ya[e] * cs[e].x + yb[e] * cs[e].y;
          gb[e] = yb[e] * cs[e].x - ya[e] * cs[e].y;
          ss += a[e] * a[e] + b[e] * b[e];
          dot += ga[e] * wa[e] * a[e] + gb[e] * wb[e] * b[e];
        }
        const float r = rsqrtf(laneSum<LANES>(ss) / (float)sh.D + sh.eps);
        const float c = laneSum<LANES>(dot) * r * r / (float)sh.D;
#pragma unroll
        for (int e = 0; e < 4; e++) {  // of a head that does not exist zeros
          dwa[e] += ga[e] * a[e] * r;
          dwb[e] += gb[e] * b[e] * r;
          ga[e] = r * (ga[e] * wa[e] - a[e] * c);
          gb[e] = r * (gb[e] * wb[e] - b[e] * c);
        }
        ra = pack4(ga);
        rb = pack4(gb);
      }
      if (live) {
        __nv_bfloat16* out = dx + ((size_t)t * all + mine.before + h) * sh.D + 4 * j;
        *reinterpret_cast<uint2*>(out) = ra;
        *reinterpret_cast<uint2*>(out + half) = rb;
      }
    }
    __syncwarp();  // the stage is read before it is filled again
    if (++stage == kStages) stage = 0;
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll
  for (int e = 0; e < 4; e++) {
#pragma unroll
    for (int o = LANES; o < 32; o <<= 1) {
      dwa[e] += __shfl_xor_sync(0xffffffffu, dwa[e], o);
      dwb[e] += __shfl_xor_sync(0xffffffffu, dwb[e], o);
    }
    if (group == 0) {
      part[warp][8 * j + e] = dwa[e];
      part[warp][8 * j + 4 + e] = dwb[e];
    }
  }
  if (lane == 0) kinds[warp] = mine.kind;
  __syncthreads();
  for (int c = threadIdx.x; c < 2 * sh.D; c += kThreads) {
    const int i = c / sh.D, d = c % sh.D;
    const int hi = d >= half, dd = hi ? d - half : d;
    const int slot = 8 * (dd >> 2) + 4 * hi + (dd & 3);
    float v = 0.f;
#pragma unroll
    for (int wp = 0; wp < kWarps; wp++) v += kinds[wp] == i ? part[wp][slot] : 0.f;
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

// A warp per token and share of its heads, as long as every SM takes them all at once.
template <typename S> unsigned ctasFor(const Shape& sh, bool values) {
  const long long need = ((long long)sh.tokens * S::count(sh.heads, sh.kv, values) + kWarps - 1) / kWarps, most = (long long)(values ? kCtasBwd : kCtasFwd) * smCount();
  const long long least = (S::count(sh.heads, sh.kv, values) + kWarps - 1) / kWarps;  // every share has a warp
  return (unsigned)(need < most ? need : most > least ? most : least);
}

template <int LANES, typename W>
cudaError_t forward(const void* x, const void* wq, const void* wk, const float* table, void* q, void* k, const Shape& sh, cudaStream_t s) {
  forwardKernel<LANES, W><<<ctasFor<Share<LANES, kUnrollFwd>>(sh, false), kThreads, 0, s>>>((const __nv_bfloat16*)x, (const W*)wq, (const W*)wk, (const float2*)table, (__nv_bfloat16*)q,
                                                                        (__nv_bfloat16*)k, sh);
  return cudaGetLastError();
}

template <int LANES, typename W>
cudaError_t backward(Grad dq, Grad dk, Grad dv, const void* x, const void* wq, const void* wk, const float* table, void* dx, float* partials, void* dwq, void* dwk,
                     const Shape& sh, cudaStream_t s) {
  const unsigned ctas = ctasFor<Share<LANES, kUnrollBwd>>(sh, true);
  constexpr int kSmem = kWarps * kStages * kUnrollBwd * 2 * (32 / LANES) * 16 * LANES;  // 64 KB
  static bool done[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !done[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(backwardKernel<LANES, W>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) done[dev] = true;
  }
  backwardKernel<LANES, W><<<ctas, kThreads, kSmem, s>>>(dq, dk, dv, (const __nv_bfloat16*)x, (const W*)wq, (const W*)wk, (const float2*)table, (__nv_bfloat16*)dx, partials, sh);
  weightSum<W><<<(2 * sh.D + 31) / 32, 1024, 0, s>>>(partials, (W*)dwq, (W*)dwk, (int)ctas, sh.D);
  return cudaGetLastError();
}

bool good(long long tokens, int seq, const Shape& sh) {
  return tokens >= 0 && tokens < (1LL << 30) && seq > 0 && sh.heads > 0 && sh.kv > 0 && sh.D >= 8 && sh.D <= 256 && sh.D % 8 == 0 && (long long)sh.heads + 2LL * sh.kv < (1 << 14);
}

}  // namespace qkn
}  // namespace b200

using namespace b200::qkn;

extern "C" {

// x [batch * seq, heads + 2 kv, D] bf16; q [batch * seq, heads, D], k [batch * seq, kv, D]; weights [D] fp32 or bf16 (wBf16); table
// [>= seq, D / 2] (cos, sin).
int b200ops_qk_norm_rope_fwd(const void* x, const void* wq, const void* wk, int wBf16, const float* table, void* q, void* k, long long tokens, int seq, int heads,
                             int kv, int D, float eps, cudaStream_t s) {
  const Shape sh{(uint32_t)tokens, (uint32_t)seq, heads, kv, D, eps};
  if (!good(tokens, seq, sh)) return (int)cudaErrorInvalidValue;
  if (tokens == 0) return 0;
  const auto go = [&](auto lanes) {
    constexpr int L = decltype(lanes)::value;
    return (int)(wBf16 ? forward<L, __nv_bfloat16>(x, wq, wk, table, q, k, sh, s) : forward<L, float>(x, wq, wk, table, q, k, sh, s));
  };
  return D <= 64 ? go(std::integral_constant<int, 8>{}) : D <= 128 ? go(std::integral_constant<int, 16>{}) : go(std::integral_constant<int, 32>{});
}

// fp32 words of scratch for the backward call.
long long b200ops_qk_norm_rope_bwd_scratch(int D, int heads, int kv) {
  const long long most = (long long)kCtasBwd * smCount(), least = ((long long)heads + 2LL * kv + kWarps - 1) / kWarps;
  return (most > least ? most : least) * 2 * D;
}

// strides: batch, head and position strides (elements, multiples of 4) of dq, dk, dv in turn. dx like x; dwq, dwk [D] of the weights' type.
int b200ops_qk_norm_rope_bwd(const void* dq, const void* dk, const void* dv, const long long* strides, const void* x, const void* wq, const void* wk, int wBf16,
                             const float* table, void* dx, float* scratch, void* dwq, void* dwk, long long tokens, int seq, int heads, int kv, int D, float eps,
                             cudaStream_t s) {
  const Shape sh{(uint32_t)tokens, (uint32_t)seq, heads, kv, D, eps};
  if (!good(tokens, seq, sh) || tokens == 0) return (int)cudaErrorInvalidValue;
  const auto grad = [&](const void* p, int i) { return Grad{(const __nv_bfloat16*)p, strides[3 * i], strides[3 * i + 1], strides[3 * i + 2]}; };
  const auto go = [&](auto lanes) {
    constexpr int L = decltype(lanes)::value;
    return (int)(wBf16 ? backward<L, __nv_bfloat16>(grad(dq, 0), grad(dk, 1), grad(dv, 2), x, wq, wk, table, dx, scratch, dwq, dwk, sh, s)
                       : backward<L, float>(grad(dq, 0), grad(dk, 1), grad(dv, 2), x, wq, wk, table, dx, scratch, dwq, dwk, sh, s));
  };
  return D <= 64 ? go(std::integral_constant<int, 8>{}) : D <= 128 ? go(std::integral_constant<int, 16>{}) : go(std::integral_constant<int, 32>{});
}

}  // extern "C"
