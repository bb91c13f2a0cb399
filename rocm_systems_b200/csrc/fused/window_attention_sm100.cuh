// Windowed attention on the 5th-generation tensor cores: the forward pass.
//
// A CTA owns two tiles of 128 queries of one head and walks the 128-key tiles that either of them sees (the sinks', then the window's). Warp
// 8 feeds queries once and keys and values through a ring of TMA tiles; one thread of warp 9 issues S = Q K^T into tensor memory and, once
// the softmax is through with it, O += P V with P read from tensor memory as well; warps 0-3 and 4-7 are the two tiles' softmax, one
// thread per row, so that row maxima and sums need no exchange. P (bf16) takes the place of the scores it was made of. While one tile's
// softmax runs, the tensor cores work for the other.
//
// The running maximum is moved, and O in tensor memory scaled down, only when a row's maximum has grown by more than 2^kSlack: weights stay
// below 2^kSlack, which costs no precision in bf16 and fp32, and O is hardly ever touched in between.
#pragma once

#include "gemm_sm100.cuh"
#include "rows.cuh"
#include "window_attention.h"

namespace b200 {
namespace wattn {

using namespace rows;

constexpr int kTile = 128;  // queries and keys of a tile
constexpr uint32_t kBox = kTile * 128;  // bytes of a TMA box: 128 rows of 64 elements
constexpr float kSlack = 8.f;

enum ErrCode : int { ERR_FWD_LOAD = 21, ERR_FWD_MMA, ERR_FWD_SOFTMAX, ERR_BWD_LOAD, ERR_BWD_MMA, ERR_BWD_MATH };

struct FwdParams {
  CUtensorMap q, k, v;  // [B][H or KV][S][D], boxes of 128 positions x 64 elements
  Args a;
  float c;              // scores' factor in powers of two, never zero
  int tiles;            // pairs of query tiles
  int* err;
};

// The keys that queries [r0, rLast] see, as tiles: [0, sinkTiles) and [first, last].
struct KeyRange {
  int sinkTiles, first, last;
  __device__ KeyRange(const Args& a, int r0, int rLast) {
    first = max(0, r0 - a.window + 1) / kTile;
    last = rLast / kTile;
    sinkTiles = (a.sinks + kTile - 1) / kTile;
  }
  __device__ bool has(int tile) const { return tile <= last && (tile >= first || tile < sinkTiles); }
};

// Bits of the keys [j, j + 32) that query i sees.
__device__ __forceinline__ uint32_t maskBits(const Args& a, int i, int j) {
  const auto below = [](int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; };
  return below(i - j + 1) & (~below(i - j + 1 - a.window) | below(a.sinks - j));
}
// Whether queries [r0, rLast] see all keys [j0, j0 + kTile).
__device__ __forceinline__ bool seesAll(const Args& a, int r0, int rLast, int j0) {
  return j0 + kTile - 1 <= r0 && (rLast - j0 < a.window || j0 + kTile <= a.sinks);
}

template <int HD> struct FwdCfg {
  static constexpr int kThreads = 384;                   // launched with 168 registers each, split as 2 x 128 x 216 and 128 x 64
  static constexpr int kMathRegs = 216, kOtherRegs = 64;
  static constexpr int kSlots = 4;                       // key and value tiles in turn
  static constexpr int kBoxes = HD / 64;
  static constexpr uint32_t kTileBytes = kBoxes * kBox;
  static constexpr uint32_t kQBytes = 4 * 32 * 256;      // a query tile, later the staging buffers of its four warps
  static constexpr size_t kSmem = 1024 + 2 * kQBytes + kSlots * kTileBytes + 256;
  static constexpr uint32_t kTmemS = 0, kTmemO = 256;    // columns: S0, S1 (128 each), O0, O1 (HD each)
  static constexpr uint32_t kTmemCols = 512;
};

// Zeroes rows [from, kTile) of a tile in shared memory; all lanes of a warp. Then the tensor cores may read it.
template <int BOXES> __device__ __forceinline__ void zeroRows(uint8_t* tile, int from, int lane) {
  for (int n = from * 8 + lane; n < kTile * 8; n += 32)
#pragma unroll
    for (int x = 0; x < BOXES; x++) *reinterpret_cast<uint4*>(tile + x * kBox + n * 16) = make_uint4(0, 0, 0, 0);
  sm100::fenceProxyAsync();
  __syncwarp();
}

// Rows [row0, row0 + 128) of a head to zeros, from warps 0-3 or 4-7.
__device__ __forceinline__ void zeroOut(const Tensor& t, int b, int h, int row0, int S, int D, int tid) {
  for (int n = tid; n < kTile * (D / 8); n += 128) {
    const int r = row0 + n / (D / 8);
    if (r < S) reinterpret_cast<uint4*>(t.at(b, h, r))[n % (D / 8)] = make_uint4(0, 0, 0, 0);
  }
}

template <int HD>
__global__ void __launch_bounds__(FwdCfg<HD>::kThreads, 1) forwardKernel(const __grid_constant__ FwdParams p) {
  using C = FwdCfg<HD>;
  using namespace sm100;
  extern __shared__ uint8_t smemRaw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smemRaw) + 1023) & ~(uintptr_t)1023);
  uint8_t* smemQ = smem;
  uint8_t* ring = smem + 2 * C::kQBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(ring + C::kSlots * C::kTileBytes);
  uint64_t* qFull = bars;                 // [2]
  uint64_t* full = bars + 2;              // [kSlots]
  uint64_t* empty = full + C::kSlots;     // [kSlots]
  uint64_t* sFull = empty + C::kSlots;    // [2] scores in tensor memory
  uint64_t* pReady = sFull + 2;           // [2] weights in their place, O scaled
  uint64_t* oDone = pReady + 2;           // [2] O complete
  uint32_t* tmemSlot = reinterpret_cast<uint32_t*>(oDone + 2);

  const Args& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* err = p.err;
  const int heads = a.B * a.H, bh = blockIdx.x % heads, h = bh % a.H, b = bh / a.H, kh = h / a.group();
  const int r0 = (p.tiles - 1 - (int)(blockIdx.x / heads)) * 2 * kTile;  // the longest rows first
  const int L = lengthOf(a, b);
  if (r0 >= L) {
    if (warp < 8) zeroOut(a.out, b, h, r0 + (warp >> 2) * kTile, a.S, a.D, threadIdx.x & 127);
    if (warp < 8 && a.rest.p) zeroOut(a.rest, b, h, r0 + (warp >> 2) * kTile, a.S, a.D, threadIdx.x & 127);
    return;
  }
  const bool two = r0 + kTile < L;
  const KeyRange own[2] = {KeyRange(a, r0, min(r0 + kTile, L) - 1), KeyRange(a, two ? r0 + kTile : r0, min(r0 + 2 * kTile, L) - 1)};
  const int nSinks = min(own[0].sinkTiles, own[0].first), count = nSinks + own[1].last - own[0].first + 1;
  const auto tileOf = [&](int n) { return n < nSinks ? n : own[0].first + n - nSinks; };
  const auto active = [&](int t, int n) { return (t == 0 || two) && own[t].has(tileOf(n)); };

  if (threadIdx.x == 0) {
    prefetchTensorMap(&p.q);
    prefetchTensorMap(&p.k);
    prefetchTensorMap(&p.v);
    for (int t = 0; t < 2; t++) {
      mbarInit(&qFull[t], 1);
      mbarInit(&sFull[t], 1);
      mbarInit(&pReady[t], 4);
      mbarInit(&oDone[t], 1);
    }
    for (int s = 0; s < C::kSlots; s++) {
      mbarInit(&full[s], 1);
      mbarInit(&empty[s], 1);
    }
    fenceBarrierInit();
  }
  if (warp == 9) {
    tmemAlloc(tmemSlot, C::kTmemCols);
    tmemRelinquish();
  }
  tcFenceBefore();
  __syncthreads();
  tcFenceAfter();
  const uint32_t tmem = *tmemSlot;

  if (warp == 8) {
    setMaxRegsDown<C::kOtherRegs>();
    if (lane == 0) {
      for (int t = 0; t < 1 + two; t++) {
        mbarArriveExpectTx(&qFull[t], C::kTileBytes);
        for (int x = 0; x < C::kBoxes; x++) tmaLoad4d(smemQ + t * C::kQBytes + x * kBox, &p.q, x * 64, r0 + t * kTile, h, b, &qFull[t]);
      }
      bool ok = true;
      for (int n = 0; n < 2 * count && ok; n++) {
        const int s = n % C::kSlots;
        ok = mbarWait(&empty[s], ((n / C::kSlots) & 1) ^ 1, err, ERR_FWD_LOAD);
        if (!ok) break;
        mbarArriveExpectTx(&full[s], C::kTileBytes);
        for (int x = 0; x < C::kBoxes; x++) tmaLoad4d(ring + s * C::kTileBytes + x * kBox, n & 1 ? &p.v : &p.k, x * 64, tileOf(n >> 1) * kTile, kh, b, &full[s]);
      }
      if (!ok) {  // let loads in flight land
        for (int t = 0; t < 1 + two; t++) mbarWait(&qFull[t], 0, err, 0, 2000u);
        for (int s = 0; s < C::kSlots; s++) mbarWait(&full[s], 0, err, 0, 2000u);
      }
    }
  } else if (warp == 9) {
    setMaxRegsDown<C::kOtherRegs>();
    constexpr uint32_t idescS = instrDesc(kTile, kTile, 1 /*bf16*/), idescO = instrDescMajor(kTile, HD, 1, 0, 1);
    const auto slot = [&](int n) { return n % C::kSlots; };
    const auto wait = [&](int n) { return mbarWait(&full[slot(n)], (n / C::kSlots) & 1, err, ERR_FWD_MMA); };
    const auto scores = [&](int t, int n) {
      if (lane == 0) {
        const uint32_t q = smemAddr(smemQ + t * C::kQBytes), k = smemAddr(ring + slot(2 * n) * C::kTileBytes);
#pragma unroll
        for (int kk = 0; kk < HD / 16; kk++) {
          const uint32_t o = (kk / 4) * kBox + (kk % 4) * 32;
          mmaF16(tmem + C::kTmemS + t * kTile, smemDescSw128(q + o), smemDescSw128(k + o), idescS, kk != 0);
        }
        mmaCommit(&sFull[t]);
      }
    };
    bool ok = true, started[2] = {false, false};
    uint32_t phase[2] = {0, 0};
    for (int t = 0; t < 1 + two && ok; t++) ok = mbarWait(&qFull[t], 0, err, ERR_FWD_MMA);
    ok = ok && wait(0);
    if (ok) {
      for (int t = 0; t < 2; t++)
        if (active(t, 0)) scores(t, 0);
      if (lane == 0) mmaCommit(&empty[slot(0)]);
    }
    for (int n = 0; n < count && ok; n++) {
      if (!(ok = wait(2 * n + 1))) break;
      uint8_t* vTile = ring + slot(2 * n + 1) * C::kTileBytes;
      const int beyond = L - tileOf(n) * kTile;
      if (beyond < kTile) zeroRows<C::kBoxes>(vTile, beyond, lane);  // a weight of zero does not silence what lies behind the sequence's end
      for (int t = 0; t < 2 && ok; t++) {
        if (active(t, n)) {
          if (!(ok = mbarWait(&pReady[t], phase[t], err, ERR_FWD_MMA))) break;
          phase[t] ^= 1;
          tcFenceAfter();
          if (lane == 0) {
            const uint32_t v = smemAddr(vTile);
#pragma unroll
            for (int kk = 0; kk < kTile / 16; kk++)
              mmaF16FromTmem(tmem + C::kTmemO + t * HD, tmem + C::kTmemS + t * kTile + kk * 8, smemDescSw128Mn(v + kk * 2048, kBox), idescO, started[t] || kk != 0);
            if (tileOf(n) == own[t].last) mmaCommit(&oDone[t]);
          }
          started[t] = true;
        }
        if (n + 1 < count && active(t, n + 1)) {
          if (!(ok = wait(2 * n + 2))) break;
          scores(t, n + 1);
        }
      }
      if (!ok) break;
      if (lane == 0) {
        mmaCommit(&empty[slot(2 * n + 1)]);
        if (n + 1 < count) mmaCommit(&empty[slot(2 * n + 2)]);
      }
      __syncwarp();
    }
  } else if (warp >= 10) {
    setMaxRegsDown<C::kOtherRegs>();
  } else {
    setMaxRegsUp<C::kMathRegs>();
    const int t = warp >> 2, q4 = warp & 3;
    const int row = r0 + t * kTile + q4 * 32 + lane;
    const int rLast = min(r0 + (t + 1) * kTile, L) - 1;
    const uint32_t laneBase = (uint32_t)(q4 * 32) << 16;
    const uint32_t tS = tmem + laneBase + C::kTmemS + t * kTile, tO = tmem + laneBase + C::kTmemO + t * HD;
    float m = -INFINITY, l = 0.f;
    uint32_t phase = 0;
    bool ok = t == 0 || two, any = false;
    for (int n = 0; n < count && ok; n++) {
      if (!active(t, n)) continue;
      if (!(ok = mbarWait(&sFull[t], phase, err, ERR_FWD_SOFTMAX))) break;
      phase ^= 1;
      tcFenceAfter();
      const int j0 = tileOf(n) * kTile;
      uint32_t s[4][32];
#pragma unroll
      for (int x = 0; x < 4; x++) tmemLoad32(tS + x * 32, s[x]);
      tmemLoadWait();
      if (!seesAll(a, r0 + t * kTile, rLast, j0)) {
#pragma unroll
        for (int x = 0; x < 4; x++) {
          const uint32_t bits = maskBits(a, row, j0 + x * 32);
#pragma unroll
          for (int e = 0; e < 32; e++)
            if (!((bits >> e) & 1)) s[x][e] = 0xff800000u;  // -inf
        }
      }
      float top = -INFINITY;
#pragma unroll
      for (int x = 0; x < 4; x++)
#pragma unroll
        for (int e = 0; e < 32; e++) top = fmaxf(top, __uint_as_float(s[x][e]));
      const bool move = top > -INFINITY && (m == -INFINITY || (top - m) * p.c > kSlack);
      const float f = move ? exp2Fast((m - top) * p.c) : 1.f;
      if (move) {
        m = top;
        l *= f;
      }
      if (any && __any_sync(0xffffffffu, move)) {
#pragma unroll 1
        for (int x = 0; x < HD / 16; x++) {
          uint32_t o[16];
          tmemLoad16(tO + x * 16, o);
          tmemLoadWait();
#pragma unroll
          for (int e = 0; e < 16; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
          tmemStore16(tO + x * 16, o);
        }
      }
      any = true;
      const float off = m == -INFINITY ? 0.f : m * p.c;
#pragma unroll
      for (int x = 0; x < 4; x++) {
        uint32_t w[16];
#pragma unroll
        for (int e = 0; e < 16; e++) {
          const float p0 = exp2Fast(fmaf(__uint_as_float(s[x][2 * e]), p.c, -off)), p1 = exp2Fast(fmaf(__uint_as_float(s[x][2 * e + 1]), p.c, -off));
          l += p0 + p1;
          w[e] = pack2(p0, p1);
        }
        tmemStore16(tS + x * 16, w);
      }
      tmemStoreWait();
      tcFenceBefore();
      __syncwarp();
      if (lane == 0) mbarArrive(&pReady[t]);
    }
    ok = ok && any && mbarWait(&oDone[t], 0, err, ERR_FWD_SOFTMAX);
    if (ok) {
      tcFenceAfter();
      const bool live = row < L;
      if (a.lse && live) a.lse[(size_t)bh * a.S + row] = m * p.c + log2f(l);
      const float inv = 1.f / l;
      uint8_t* stage = smemQ + t * C::kQBytes + q4 * 32 * 256;
      const auto rowsOf = [&](const Tensor& dst) {
        return [&](int r) -> __nv_bfloat16* { return row - lane + r < a.S ? dst.at(b, h, row - lane + r) : nullptr; };
      };
      const auto load = [&](int x, uint32_t(&acc)[32]) {
        tmemLoad32(tO + x * 32, acc);
        tmemLoadWait();
#pragma unroll
        for (int e = 0; e < 32; e++) acc[e] = live ? __float_as_uint(__uint_as_float(acc[e]) * inv) : 0u;
      };
      gemm::drainStaged(stage, lane, HD, a.D, load, rowsOf(a.out));
      if (a.rest.p)
        gemm::drainStaged(
            stage, lane, HD, a.D,
            [&](int x, uint32_t(&acc)[32]) {
              load(x, acc);
#pragma unroll
              for (int e = 0; e < 32; e++) {
                const float v = __uint_as_float(acc[e]);
                acc[e] = __float_as_uint(v - __bfloat162float(__float2bfloat16(v)));
              }
            },
            rowsOf(a.rest));
    } else if (t == 1 && !two) {
      zeroOut(a.out, b, h, r0 + kTile, a.S, a.D, threadIdx.x & 127);
      if (a.rest.p) zeroOut(a.rest, b, h, r0 + kTile, a.S, a.D, threadIdx.x & 127);
    }
  }
  tcFenceBefore();
  __syncthreads();
  if (warp == 9) tmemDealloc(tmem, C::kTmemCols);
}

}  // namespace wattn
}  // namespace b200
