// Windowed attention on the 5th-generation tensor cores.
//
// Forward: a persistent CTA takes pairs of 128-query tiles of a head and walks the 128-key tiles that either of them sees (the sinks', then
// the window's). One warp feeds queries, and keys and values through a ring of TMA tiles; one issues S = Q K^T into tensor memory and, once
// the softmax is through with it, O += P V with P read from tensor memory as well; eight warps for each of the two tiles are its softmax, two
// threads per row. P (bf16) takes the place of the scores it was made of. While one tile's softmax runs, the tensor cores work for the other;
// while a pair's answer is written, the next pair's first scores are made.
//
// The running maximum is moved, and O in tensor memory scaled down, only when a row's maximum has grown by more than 2^kSlack: weights stay
// below 2^kSlack, which costs no precision in bf16 and fp32, and O is hardly ever touched in between.
//
// 4096 tokens, 32 query and 8 key heads of 128: 122 us for all earlier keys (137 GFLOP, 1.13 PFLOP/s), 85 for a window of 1024 with 4 sinks. No
// unit is full: the tensor cores are busy for 47 to 57% of the time, the special-function pipe for 40, and instructions are issued in half of
// the cycles. The softmax of a tile is the longest link; what is left over is waiting for one another, 100 to 200 cycles for each barrier
// that is already satisfied.
#pragma once

#include <type_traits>

#include "gemm_sm100.cuh"
#include "rows.cuh"
#include "window_attention.h"

namespace b200 {
namespace wattn {

using namespace rows;

constexpr int kTile = 128;  // queries and keys of a tile
constexpr uint32_t kBox = kTile * 128;  // bytes of a TMA box: 128 rows of 64 elements
constexpr float kSlack = 8.f;
// Of a row's pairs of powers of two, one in so many is a polynomial (4096 tokens, 32 heads of 128, no window: 124 us; none and every other 127, every fourth 124).
constexpr int kPoly = 3;

enum ErrCode : int { ERR_FWD_LOAD = 21, ERR_FWD_MMA, ERR_FWD_SOFTMAX, ERR_BWD_LOAD, ERR_BWD_MMA, ERR_BWD_MATH };

struct FwdParams {
  CUtensorMap q, k, v;  // [B][H or KV][S][D], boxes of 128 positions x 64 elements
  Args a;
  float c;              // scores' factor in powers of two, never zero
  int tiles;            // pairs of query tiles
  uint32_t items;       // pairs of all heads
  bool wide;            // rows of out and rest start on 32-byte boundaries and are whole 32-byte pieces
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

// Weights and their gradients (P and dS) go to the tensor cores in bf16, each off by 2^-9 of itself. Over many keys that averages out. Where rows
// see a few keys the gradient is a small difference of such numbers (3 tokens: 0.0039 to 0.0052 of its norm). So in sequences of at most
// kFineSeq tokens, for the first kTile queries of longer ones, and where no row sees more than kFineKeys keys, they are handed over as the sum
// of two bf16 values, which leaves the result's own rounding. The rule looks at a sequence's own length and a query's position: what a sequence
// answers does not hang on the batch that it is padded in.
//
// Kernels for calls of such rows only (FINE) multiply by both values in one step. In the others the first tiles are streamed a second time, for
// what rounding took: the same products in the same order, so the same bits, and the issuing warp need not know. (A question in each of its
// steps made the windowed passes 5 to 7% slower, whatever the answer was.)
// The second time takes 339 instead of 329 us of a window of 1024 with 4 sinks over 4096 tokens both ways, and 552 instead of 548 of all earlier keys.
// A window of 128 keys throughout as two values would take 55 instead of 47 us forward and 239 instead of 159 backward.
constexpr int kFineSeq = 2 * kTile, kFineKeys = 64;
// So many of a sequence's first query tiles come a second time, where not all do in one step.
template <bool FINE> __device__ __forceinline__ int secondTiles(int length) { return FINE ? 0 : length <= kFineSeq ? kFineSeq / kTile : 1; }

template <int HD> struct FwdCfg {
  static constexpr int kMath = 16;                       // warps 0-7 and 8-15 are the two tiles' softmax
  static constexpr int kThreads = 32 * (kMath + 4);      // launched with 96 registers each, split as 4 x 128 x 104 and 128 x 64
  static constexpr int kMathRegs = 104, kOtherRegs = 64;
  static constexpr int kSlots = HD == 128 ? 4 : 8;       // key and value tiles in turn
  static constexpr int kBoxes = HD / 64;
  static constexpr uint32_t kTileBytes = kBoxes * kBox;
  static constexpr uint32_t kMeet = 2 * 2 * kTile * 4;   // what a row's two threads tell each other
  static constexpr size_t kSmem = 1024 + (2 + kSlots) * kTileBytes + kMeet + 256;
  static constexpr uint32_t kTmemS = 0, kTmemO = 256;    // columns: S0, S1 (128 each), O0, O1 (HD each)
  static constexpr uint32_t kTmemCols = 512;
};

// What a persistent CTA does in its turn `k`: items are sorted by falling cost, so every other turn goes through the CTAs backwards.
__device__ __forceinline__ uint32_t itemOf(uint32_t k) { return k * gridDim.x + (k & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x); }

// Zeroes rows [from, ROWS) of a tile of BOXES boxes of ROWS rows x 128 bytes, by a whole warp: a weight of zero does not silence what may lie
// behind a sequence's end, so it must not be there where the tensor cores sum over a tile's rows.
template <int BOXES, int ROWS> __device__ __forceinline__ void zeroRows(uint8_t* tile, int from, int lane) {
  for (int n = from * 8 + lane; n < ROWS * 8; n += 32)
#pragma unroll
    for (int x = 0; x < BOXES; x++) *reinterpret_cast<uint4*>(tile + x * ROWS * 128 + n * 16) = make_uint4(0, 0, 0, 0);
  sm100::fenceProxyAsync();
}

// Rows [row0, row0 + 128) of a head to zeros, by 128 threads.
__device__ __forceinline__ void zeroOut(const Tensor& t, int b, int h, int row0, int S, int D, int tid) {
  if (!t.p) return;
  for (int n = tid; n < kTile * (D / 8); n += 128) {
    const int r = row0 + n / (D / 8);
    if (r < S) reinterpret_cast<uint4*>(t.at(b, h, r))[n % (D / 8)] = make_uint4(0, 0, 0, 0);
  }
}

// What rounding to two bf16 values (`packed`) took from `v`.
__device__ __forceinline__ F2 remainder(F2 v, uint32_t packed) { return fmaF2(unpackF2(packed), makeF2(-1.f, -1.f), v); }

// FINE: all weights as the sum of two bf16 values.
template <int HD, bool FINE>
__global__ void __launch_bounds__(FwdCfg<HD>::kThreads, 1) forwardKernel(const __grid_constant__ FwdParams p) {
  using C = FwdCfg<HD>;
  using namespace sm100;
  extern __shared__ uint8_t smemRaw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smemRaw) + 1023) & ~(uintptr_t)1023);
  uint8_t* smemQ = smem;
  uint8_t* ring = smem + 2 * C::kTileBytes;
  float* meet = reinterpret_cast<float*>(ring + C::kSlots * C::kTileBytes);  // [tile][half][128]
  uint64_t* bars = reinterpret_cast<uint64_t*>(meet + 4 * kTile);
  uint64_t *qFull = bars, *qEmpty = bars + 1;
  uint64_t* full = bars + 2;              // [kSlots]
  uint64_t* empty = full + C::kSlots;     // [kSlots]
  uint64_t* sFull = empty + C::kSlots;    // [2] scores in tensor memory
  uint64_t* pReady = sFull + 2;           // [2] weights in their place, O scaled; this step's values and the next one's keys have landed
  uint64_t* oDone = pReady + 2;           // [2] O complete
  uint64_t* oFree = oDone + 2;            // [2] O read
  uint32_t* tmemSlot = reinterpret_cast<uint32_t*>(oFree + 2);

  const Args& a = p.a;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;  // (the compiler is to know that it is a warp's)
  volatile int* err = p.err;

  if (threadIdx.x == 0) {
    prefetchTensorMap(&p.q);
    prefetchTensorMap(&p.k);
    prefetchTensorMap(&p.v);
    mbarInit(qFull, 2);
    mbarInit(qEmpty, 1);
    for (int t = 0; t < 2; t++) {
      mbarInit(&sFull[t], 1);
      mbarInit(&pReady[t], 9);
      mbarInit(&oDone[t], 1);
      mbarInit(&oFree[t], 8);
    }
    for (int s = 0; s < C::kSlots; s++) {
      mbarInit(&full[s], 1);
      mbarInit(&empty[s], 1);
    }
    fenceBarrierInit();
  }
  if (warp == C::kMath + 1) {
    tmemAlloc(tmemSlot, C::kTmemCols);
    tmemRelinquish();
  }
  tcFenceBefore();
  __syncthreads();
  tcFenceAfter();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmemSlot, 0);

  // A pair of query tiles of one head and its key tiles.
  struct Item {
    int h, b, kh, r0, L, count, nSinks, twice;  // twice: so many key tiles come twice, behind one another
    bool two, one;                              // one: a second time for the first query tile only
    KeyRange own0, own1;
    __device__ Item(const FwdParams& p, uint32_t item) : own0(p.a, 0, 0), own1(p.a, 0, 0) {
      const Args& a = p.a;
      const uint32_t heads = a.B * a.H, bh = item % heads;
      h = bh % (uint32_t)a.H;
      b = bh / (uint32_t)a.H;
      kh = h / a.group();
      r0 = (p.tiles - 1 - (int)(item / heads)) * 2 * kTile;  // the longest rows first
      L = lengthOf(a, b);
      count = nSinks = twice = 0;
      two = r0 + kTile < L;
      one = secondTiles<FINE>(L) == 1;
      if (r0 >= L) return;
      own0 = KeyRange(a, r0, min(r0 + kTile, L) - 1);
      own1 = KeyRange(a, two ? r0 + kTile : r0, min(r0 + 2 * kTile, L) - 1);
      nSinks = min(own0.sinkTiles, own0.first);
      twice = FINE || r0 ? 0 : one ? 1 : own1.last + 1;
      count = nSinks + own1.last - own0.first + 1 + twice;
    }
    __device__ int tileOf(int n) const {
      if constexpr (!FINE) n = n < 2 * twice ? n >> 1 : n - twice;
      return n < nSinks ? n : own0.first + n - nSinks;
    }
    __device__ bool fine(int t) const { return FINE || (twice && !(t && one)); }
    __device__ bool again(int n) const { return !FINE && n < 2 * twice && (n & 1); }
    __device__ bool active(int t, int n) const { return t == 0 ? own0.has(tileOf(n)) : two && own1.has(tileOf(n)) && !(again(n) && one); }
    __device__ bool last(int t, int n) const { return tileOf(n) == (t ? own1.last : own0.last) && (FINE || n >= 2 * twice || (n & 1) || (t && one)); }
    __device__ bool straddles(int n) const { return L - tileOf(n) * kTile < kTile; }
  };

  if (warp == C::kMath) {
    setMaxRegsDown<C::kOtherRegs>();
    if (lane == 0) {
      bool ok = true;
      int slot = 0;
      uint32_t turn = 1, qTurn = 1;
      for (int k = 0; ok && itemOf(k) < p.items; k++) {
        const Item it(p, itemOf(k));
        if (it.count == 0) continue;
        if (!(ok = mbarWait(qEmpty, qTurn, err, ERR_FWD_LOAD))) break;
        qTurn ^= 1;
        mbarArriveExpectTx(qFull, (1 + it.two) * C::kTileBytes);
        for (int t = 0; t < 1 + it.two; t++)
          for (int x = 0; x < C::kBoxes; x++) tmaLoad4d(smemQ + t * C::kTileBytes + x * kBox, &p.q, x * 64, it.r0 + t * kTile, it.h, it.b, qFull);
        for (int n = 0; n < 2 * it.count; n++) {
          if (!(ok = mbarWait(&empty[slot], turn, err, ERR_FWD_LOAD))) break;
          mbarArriveExpectTx(&full[slot], C::kTileBytes);
          for (int x = 0; x < C::kBoxes; x++)
            tmaLoad4d(ring + slot * C::kTileBytes + x * kBox, n & 1 ? &p.v : &p.k, x * 64, it.tileOf(n >> 1) * kTile, it.kh, it.b, &full[slot]);
          if (++slot == C::kSlots) slot = 0, turn ^= 1;
        }
      }
      if (!ok) {  // let loads in flight land
        mbarWait(qFull, 0, err, 0, 2000u);
        for (int s = 0; s < C::kSlots; s++) mbarWait(&full[s], 0, err, 0, 2000u);
      }
    }
  } else if (warp == C::kMath + 1) {
    setMaxRegsDown<C::kOtherRegs>();
    constexpr uint32_t idescS = instrDesc(kTile, kTile, 1 /*bf16*/), idescO = instrDescMajor(kTile, HD, 1, 0, 1);
    // The whole warp walks along and one elected lane issues: what the instructions take from uniform registers is then formed there. (With
    // `lane == 0` in the place of the election each cost 100 cycles to issue, and runs 64.)
    const uint64_t descQ = smemDescSw128(smemAddr(smemQ)), descK = smemDescSw128(smemAddr(ring)), descV = smemDescSw128Mn(smemAddr(ring), kBox);
    bool ok = true, all = true;  // of this lane's waits; of the warp's, looked at once per tile and off the products' way: waits behind one that was given up are short
    const auto wait = [&](uint64_t* bar, uint32_t parity) { ok = mbarWait(bar, parity, err, ERR_FWD_MMA) && ok; };
    uint32_t qPhase = 0, pPhase[2] = {0, 0}, oTurn[2] = {1, 1};
    int slotK = 0;
    const auto after = [](int s) { return s + 1 == C::kSlots ? 0 : s + 1; };
    const auto scores = [&](int t, int slot) {  // by the elected lane
#pragma unroll
      for (int kk = 0; kk < HD / 16; kk++) {
        const uint32_t o = (kk / 4) * kBox + (kk % 4) * 32;
        mmaF16(tmem + C::kTmemS + t * kTile, descQ + ((t * C::kTileBytes + o) >> 4), descK + ((slot * C::kTileBytes + o) >> 4), idescS, kk != 0);
      }
      mmaCommit(&sFull[t]);
    };
    for (int k = 0; all && itemOf(k) < p.items; k++) {
      const Item it(p, itemOf(k));
      if (it.count == 0) continue;
      wait(qFull, qPhase);  // and the first keys, see the next warp
      qPhase ^= 1;
      if (electOne()) {
        scores(0, slotK);
        if (it.active(1, 0)) scores(1, slotK);
        mmaCommit(&empty[slotK]);
        if (it.count == 1) mmaCommit(qEmpty);
      }
      __syncwarp();
      bool started[2] = {false, false};
      for (int n = 0; n < it.count && all; n++) {
        const bool more = n + 1 < it.count;
        const int slotV = after(slotK), slotNext = after(slotV);
#pragma unroll
        for (int t = 0; t < 2; t++) {
          const bool now = it.active(t, n), next = more && it.active(t, n + 1), last = it.last(t, n);
          if (now) {
            if (!started[t]) {
              wait(&oFree[t], oTurn[t]);
              oTurn[t] ^= 1;
            }
            wait(&pReady[t], pPhase[t]);
            pPhase[t] ^= 1;
            tcFenceAfter();
          }
          if (electOne()) {
            if (now) {
#pragma unroll
              for (int kk = 0; kk < kTile / 16; kk++)
                mmaF16FromTmem(tmem + C::kTmemO + t * HD, tmem + C::kTmemS + t * kTile + (kk / 4) * 64 + (kk % 4) * 8, descV + ((slotV * C::kTileBytes + kk * 2048) >> 4), idescO,
                               started[t] || kk != 0);
              if constexpr (FINE)
#pragma unroll
                for (int kk = 0; kk < kTile / 16; kk++)
                  mmaF16FromTmem(tmem + C::kTmemO + t * HD, tmem + C::kTmemS + t * kTile + (kk / 4) * 64 + 32 + (kk % 4) * 8,
                                 descV + ((slotV * C::kTileBytes + kk * 2048) >> 4), idescO, 1);
              if (last) mmaCommit(&oDone[t]);
            }
            if (t == 1) mmaCommit(&empty[slotV]);
            if (next) scores(t, slotNext);
            if (t == 1 && more) {
              mmaCommit(&empty[slotNext]);
              if (n + 2 == it.count) mmaCommit(qEmpty);
            }
          }
          __syncwarp();
          started[t] = started[t] || now;
        }
        if (more) slotK = slotNext;
        all = __all_sync(0xffffffffu, ok);
      }
      slotK = after(after(slotK));
    }
  } else if (warp == C::kMath + 2) {
    // Looks after the landed tiles, so that the issuing warp has one barrier to wait for per step (each wait is 100 to 200 cycles of its time,
    // which the tensor cores stand still): takes part in the barriers that it waits for when the tiles of the step are there.
    setMaxRegsDown<C::kOtherRegs>();
    int slot = 0;
    uint32_t phase = 0, pPhase[2] = {0, 0};
    bool ok = true;
    const auto landed = [&]() {
      const int s = slot;
      ok = ok && mbarWait(&full[s], phase, err, ERR_FWD_MMA);
      if (++slot == C::kSlots) slot = 0, phase ^= 1;
      return s;
    };
    for (int k = 0; ok && itemOf(k) < p.items; k++) {
      const Item it(p, itemOf(k));
      if (it.count == 0) continue;
      landed();
      __syncwarp();
      if (lane == 0) mbarArrive(qFull);
      for (int n = 0; n < it.count && ok; n++) {
        const int v = landed();
        if (n + 1 < it.count) landed();
        if (it.straddles(n)) zeroRows<C::kBoxes, kTile>(ring + v * C::kTileBytes, it.L - it.tileOf(n) * kTile, lane);
        __syncwarp();
#pragma unroll
        for (int t = 0; t < 2; t++)
          if (lane == 0 && it.active(t, n)) mbarArrive(&pReady[t]);
#pragma unroll
        for (int t = 0; t < 2; t++)
          if (it.active(t, n)) {  // not ahead of them
            ok = ok && mbarWait(&pReady[t], pPhase[t], err, ERR_FWD_MMA);
            pPhase[t] ^= 1;
          }
      }
    }
  } else if (warp == C::kMath + 3) {
    setMaxRegsDown<C::kOtherRegs>();
  } else {
    setMaxRegsUp<C::kMathRegs>();
    constexpr int kCols = kTile / 2;  // of a row's scores, this thread's
    const int t = warp >> 3, side = warp >> 2 & 1, q4 = warp & 3, r = q4 * 32 + lane;
    const uint32_t laneBase = (uint32_t)(q4 * 32) << 16;
    const uint32_t tS = tmem + laneBase + C::kTmemS + t * kTile + side * kCols, tO = tmem + laneBase + C::kTmemO + t * HD + side * (HD / 2);
    const float slack = kSlack / p.c;
    float *mine = meet + (2 * t + side) * kTile + r, *other = meet + (2 * t + 1 - side) * kTile + r;
    // Both halves of a row's warps; what is told is read before the next S, or the next item, is there.
    const auto meeting = [&]() { asm volatile("bar.sync %0, 64;" ::"r"(1 + t * 4 + q4) : "memory"); };
    uint32_t sPhase = 0, oPhase = 0;
    bool ok = true;
    for (int k = 0; ok && itemOf(k) < p.items; k++) {
      const Item it(p, itemOf(k));
      const int rFirst = it.r0 + t * kTile, row = rFirst + r, rLast = min(rFirst + kTile, it.L) - 1;
      if (rFirst >= it.L) {
        zeroOut(side ? a.rest : a.out, it.b, it.h, rFirst, a.S, a.D, threadIdx.x & 127);
        continue;
      }
      const KeyRange own = t ? it.own1 : it.own0;
      float m = -INFINITY, limit = -INFINITY, l = 0.f;
      bool any = false;
      for (int n = 0; n < it.count; n++) {
        const int tile = it.tileOf(n);
        if (!own.has(tile) || (t && it.again(n) && it.one)) continue;
        const int j0 = tile * kTile;
        const bool every = seesAll(a, rFirst, rLast, j0);
        if (!(ok = mbarWait(&sFull[t], sPhase, err, ERR_FWD_SOFTMAX))) break;
        sPhase ^= 1;
        tcFenceAfter();
        uint32_t s[2][32];
#pragma unroll
        for (int x = 0; x < 2; x++) tmemLoad32(tS + x * 32, s[x]);
        tmemLoadWait();
        if (!every) {
#pragma unroll
          for (int x = 0; x < 2; x++) {
            const uint32_t bits = maskBits(a, row, j0 + side * kCols + x * 32);
#pragma unroll
            for (int e = 0; e < 32; e++)
              if (!((bits >> e) & 1)) s[x][e] = 0xff800000u;  // -inf
          }
        }
        float best[4];
#pragma unroll
        for (int x = 0; x < 4; x++) {
          best[x] = __uint_as_float(s[x / 2][x % 2 * 16]);
#pragma unroll
          for (int e = 1; e < 15; e += 2)
            best[x] = fmaxf(fmaxf(best[x], __uint_as_float(s[x / 2][x % 2 * 16 + e])), __uint_as_float(s[x / 2][x % 2 * 16 + e + 1]));
          best[x] = fmaxf(best[x], __uint_as_float(s[x / 2][x % 2 * 16 + 15]));
        }
        float top = fmaxf(fmaxf(best[0], best[1]), fmaxf(best[2], best[3]));
        *mine = top;
        meeting();
        top = fmaxf(top, *other);
        const bool move = top > limit;
        if (__any_sync(0xffffffffu, move)) {
          const float f = move ? exp2Fast((m - top) * p.c) : 1.f;
          if (move) {
            m = top;
            limit = top + slack;
            l *= f;
          }
          if (any) {  // this thread's half of the row's answer
#pragma unroll 1
            for (int x = 0; x < HD / 32; x++) {
              uint32_t o[16];
              tmemLoad16(tO + x * 16, o);
              tmemLoadWait();
#pragma unroll
              for (int e = 0; e < 16; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              tmemStore16(tO + x * 16, o);
            }
          }
        }
        any = true;
        const float off = m == -INFINITY ? 0.f : m * p.c;
        const F2 c2 = makeF2(p.c, p.c), off2 = makeF2(-off, -off);
        F2 sum[2] = {makeF2(l, 0.f), makeF2(0.f, 0.f)};
        const auto weights = [&](auto poly, auto rest) {
#pragma unroll
          for (int x = 0; x < (FINE ? 4 : 2); x++) {  // FINE: once more for what rounding took (formed again, registers are short)
            uint32_t w[16];
#pragma unroll
            for (int e = 0; e < 16; e++) {
              const F2 v = fmaF2(makeF2(__uint_as_float(s[x & 1][2 * e]), __uint_as_float(s[x & 1][2 * e + 1])), c2, off2);
              const F2 pr = decltype(poly)::value && e % kPoly == kPoly - 1 ? exp2Poly(v) : exp2F2(v);
              w[e] = pack2(pr);
              if (x >= 2 || decltype(rest)::value) w[e] = pack2(remainder(pr, w[e]));
              else sum[e & 1] = addF2(sum[e & 1], pr);
            }
            tmemStore16(tS + x * 16, w);
          }
        };
        // Masked scores have to become zeros, which the polynomial does not give.
        if (!it.fine(t) && every) weights(std::true_type{}, std::false_type{});
        else if (!it.again(n)) weights(std::false_type{}, std::false_type{});
        else weights(std::false_type{}, std::true_type{});
        tmemStoreWait();
        tcFenceBefore();
        __syncwarp();
        if (lane == 0) mbarArrive(&pReady[t]);
        float upper;
        splitF2(addF2(sum[0], sum[1]), l, upper);
        l += upper;
      }
      if (!ok || !(ok = mbarWait(&oDone[t], oPhase, err, ERR_FWD_SOFTMAX))) break;
      oPhase ^= 1;
      tcFenceAfter();
      *mine = l;  // the other's maximum was read before the last weights were handed over
      meeting();
      l += *other;
      const bool live = row < it.L;
      if (a.lse && side == 0) a.lse[((size_t)it.b * a.H + it.h) * a.padded() + row] = live ? -(m * p.c + log2f(l)) : -INFINITY;
      // (A row whose every score is minus infinity has no softmax; what the polynomial gave for such scores is no answer.)
      const float inv = !live ? 0.f : m == -INFINITY ? NAN : 1.f / l;
#pragma unroll
      for (int x = 0; x < HD / 64; x++) {
        uint32_t o[32], w[16];
        tmemLoad32(tO + x * 32, o);
        tmemLoadWait();
        if (x == HD / 64 - 1) {
          tcFenceBefore();
          __syncwarp();
          if (lane == 0) mbarArrive(&oFree[t]);
        }
        const int col = side * (HD / 2) + x * 32, words = (a.D - col) / 2;
#pragma unroll
        for (int e = 0; e < 32; e++) o[e] = live ? __float_as_uint(__uint_as_float(o[e]) * inv) : 0u;
#pragma unroll
        for (int e = 0; e < 16; e++) w[e] = pack2(__uint_as_float(o[2 * e]), __uint_as_float(o[2 * e + 1]));
        if (row < a.S) storeRow16(a.out.at(it.b, it.h, row) + col, w, words, p.wide);
        if (a.rest.p) {
#pragma unroll
          for (int e = 0; e < 16; e++)
            w[e] = pack2(__uint_as_float(o[2 * e]) - __uint_as_float(w[e] << 16), __uint_as_float(o[2 * e + 1]) - __uint_as_float(w[e] & 0xffff0000u));
          if (row < a.S) storeRow16(a.rest.at(it.b, it.h, row) + col, w, words, p.wide);
        }
      }
      meeting();  // the sums are read before the next item's maxima are written
    }
  }
  tcFenceBefore();
  __syncthreads();
  if (warp == C::kMath + 1) tmemDealloc(tmem, C::kTmemCols);
}

// ---- backward ---------------------------------------------------------------------------------------------------
// Two kernels of one shape, which both form the weights again instead of sharing them through memory, so that no gradient is summed by
// atomics: a persistent CTA takes 128 rows of two operands (X1, X2) after one another, streams 128-row tiles of two others (Y1, Y2) and has in
// tensor memory
//   S = X1 Y1^T   and   dP = X2 Y2^T   (or their transposes),
// from which 256 threads, two per row, make P = 2^(S c - lse) and dS = P (dP - delta) in bf16, both in dP's place, as the tensor-memory
// operands of the products that follow, while the next tile's S, whose place is free once it has been read, is already there:
//   queries: X = Q, dO;  Y = K, V;   dQ += dS Y1. X is copied into tensor memory, so that every product reads one operand only from shared memory,
//            which hands out 128 bytes a cycle: just what a product of 128 x 128 x 16 with both operands there takes (64 cycles, and 85 while
//            the tiles are written as well). delta is formed here.
//   keys:    X = K, V;   Y = Q, dO;  dV += P^T Y2, dK += dS^T Y1, over all query heads of the key head. With two accumulators tensor memory has no
//            room for X.
//
// In the keys' kernel lse and delta belong to the columns. Read from shared memory by every thread they took half of its bandwidth. So
// they enter by one more step of the products instead: each row of Y gets six more elements, -lse / c and -delta as the sums of three
// bf16 values each (`stat`, left by the queries' kernel), each row of X1 ones at the first three and of X2 at the others. Then
// P = 2^(S c) and dS = P dP.
//
// While an item's gradients are written, the next one's first products run.
//
// Keys that every later query sees (sinks) would keep their CTAs far longer than the others: the queries behind the window are split over
// further items, whose fp32 sums joinSinks adds up in a fixed order.
//
// 4096 tokens, 32 query and 8 key heads of 128: 390 us for all earlier keys (344 GFLOP, and 137 more as both make S and dP), 256 for a window of 1024
// with 4 sinks (queries 116, keys 134, partial sums 3). Tensor cores are busy for 60 and 77% (48 and 68%) of that time; the rest is the chain of
// a tile (scores, weights, gradients of scores, products), which only one tile of look-ahead covers.
enum Side { kQueries, kKeys };

struct BwdParams {
  CUtensorMap x1, x2, y1, y2;
  CUtensorMap out, rest;   // queries
  Args a;
  float c;
  int tiles;      // 128-row tiles of a sequence
  int sinkTiles;  // key tiles whose far queries are split off; 0: none
  int farChunk, farCount;  // query tiles per split, splits per sink tile
  uint32_t items;
  bool wide;               // rows of the gradients start on 32-byte boundaries and are whole 32-byte pieces
  float* partials;         // [B * KV][sinkTiles][1 + farCount][dK, dV][min(sinks, 128)][D]
  int* err;
};

template <int HD, Side SIDE> struct BwdCfg {
  static constexpr int kThreads = 384;                // split as in the forward kernel
  static constexpr int kMathRegs = 216, kOtherRegs = 64;
  static constexpr int kBoxes = HD / 64;
  static constexpr int kSlots = 4;
  static constexpr uint32_t kTileBytes = kBoxes * kBox;
  static constexpr uint32_t kStat = kTile * 16;       // eight more elements of a tile's rows
  static constexpr uint32_t kExtra = SIDE == kQueries ? 2 * kTile * 4 : 5 * kStat;
  static constexpr size_t kSmem = 1024 + (2 + kSlots) * kTileBytes + kExtra + 256;
  static constexpr uint32_t kTmemCols = 512;
  // columns: queries: X1, X2 (64 each), S, dP, dQ; keys: S, dP, dV, dK
  static constexpr uint32_t kX1 = 0, kX2 = 64, kS = SIDE == kQueries ? 128 : 0, kDp = kS + 128, kAcc1 = SIDE == kQueries ? 384 : 256, kAcc2 = 384;
};

// FINE: P and dS of all rows as the sum of two bf16 values. What rounding took goes where the queries' kernel has P's columns free and where the keys'
// kernel has had S, which then is not made a tile ahead.
template <int HD, Side SIDE, bool FINE>
__global__ void __launch_bounds__(BwdCfg<HD, SIDE>::kThreads, 1) backwardKernel(const __grid_constant__ BwdParams p) {
  using C = BwdCfg<HD, SIDE>;
  using namespace sm100;
  extern __shared__ uint8_t smemRaw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smemRaw) + 1023) & ~(uintptr_t)1023);
  uint8_t* smemX = smem;                              // X1, X2
  uint8_t* ring = smem + 2 * C::kTileBytes;
  uint8_t* extra = ring + C::kSlots * C::kTileBytes;  // keys: X1's and X2's further elements, Y's of two tiles, zeros
  float* half = reinterpret_cast<float*>(extra);      // queries: [2][128] halves of delta
  uint64_t* bars = reinterpret_cast<uint64_t*>(extra + C::kExtra);
  uint64_t *xFull = bars, *xEmpty = bars + 19, *xReady = bars + 1, *sFull = bars + 2, *sTaken = bars + 3, *dpFull = bars + 4,
           *dsReady = bars + 5, *statFull = bars + 6 /*[2]*/, *statEmpty = bars + 8 /*[2]*/, *done = bars + 10, *full = bars + 11,
           *empty = full + C::kSlots;
  uint32_t* tmemSlot = reinterpret_cast<uint32_t*>(bars + 20);

  const Args& a = p.a;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  volatile int* err = p.err;

  // Rows [x0, x0 + 128) of head xh against `yTiles` streamed tiles (queries: the sinks' first) of `group` heads from yh on.
  struct Item {
    int b, xh, bh, L, xTile, x0, far, yFirst, yTiles, sinkTiles, yh, count, partRows;
    __device__ Item(const BwdParams& p, uint32_t item) {
      const Args& a = p.a;
      const uint32_t xHeads = SIDE == kQueries ? a.H : a.KV, all = a.B * xHeads;
      const int turn = item / all;
      bh = item % all;
      xh = (uint32_t)bh % xHeads;
      b = (uint32_t)bh / xHeads;
      L = lengthOf(a, b);
      far = -1;
      sinkTiles = partRows = 0;
      if constexpr (SIDE == kQueries) {
        xTile = p.tiles - 1 - turn;  // the longest rows first
        x0 = xTile * kTile;
        const KeyRange r(a, x0, min(x0 + kTile, L) - 1);
        yFirst = r.first;
        sinkTiles = min(r.sinkTiles, r.first);
        yTiles = sinkTiles + r.last - r.first + 1;
        yh = xh / a.group();
        count = x0 < L ? (xTile < secondTiles<FINE>(L) ? 2 * yTiles : yTiles) : 0;
      } else {
        xTile = turn < p.tiles ? turn : (turn - p.tiles) / p.farCount;
        if (turn >= p.tiles) far = (turn - p.tiles) % p.farCount;
        x0 = xTile * kTile;
        const int lastTile = (L - 1) / kTile;                                   // of the sequence
        const int reach = a.window > a.S - x0 ? a.S : x0 + kTile + a.window - 1;  // first query that sees none of the tile's keys through the window
        const int nearLast = x0 < a.sinks && p.sinkTiles == 0 ? lastTile : min(lastTile, (reach - 1) / kTile);
        if (far < 0) {
          yFirst = x0 / kTile;
          yTiles = nearLast - yFirst + 1;
        } else {
          yFirst = (reach - 1) / kTile + 1 + far * p.farChunk;
          yTiles = min(p.farChunk, lastTile - yFirst + 1);
        }
        if (x0 >= L || yTiles < 0) yTiles = 0;
        yh = xh * a.group();
        count = (yTiles + max(0, min(secondTiles<FINE>(L), yFirst + yTiles) - yFirst)) * a.group();
        if (xTile < p.sinkTiles) partRows = min(kTile, a.sinks - x0);
      }
    }
    // The streamed tiles in their order; `again`: the second time, for what rounding took.
    __device__ int firstTile() const { return SIDE == kQueries && sinkTiles ? 0 : yFirst; }
    __device__ void next(int& tile, bool& again) const {
      if (!FINE && !again && (SIDE == kQueries ? xTile : tile) < secondTiles<FINE>(L)) {
        again = true;
        return;
      }
      again = false;
      const int end = SIDE == kQueries ? sinkTiles : yFirst + yTiles;  // queries: from the sinks to the window; keys: to the next head's first
      tile = tile + 1 == end ? yFirst : tile + 1;
    }
    __device__ bool straddles(int tile) const { return L - tile * kTile < kTile; }
    // Where the sums of this item's sinks go: dK's rows, then dV's.
    __device__ float* part(const BwdParams& p, bool dv) const {
      const int pitch = min(p.a.sinks, kTile);
      return p.partials + (((size_t)(bh * p.sinkTiles + xTile) * (1 + p.farCount) + 1 + far) * 2 + dv) * pitch * p.a.D;
    }
  };
  // The streamed tiles are counted through all items. Y1 of a tile takes the slot of Y2 of the tile but one before it, which is through first, and
  // the other way round.
  const auto slot1 = [](uint32_t g) { return 2 * (g & 1) + (g >> 1 & 1); };
  const auto slot2 = [](uint32_t g) { return 2 * (g & 1) + 1 - (g >> 1 & 1); };
  const auto ringPhase = [](uint32_t g) { return g >> 1 & 1; };

  if (threadIdx.x == 0) {
    prefetchTensorMap(&p.x1);
    prefetchTensorMap(&p.x2);
    prefetchTensorMap(&p.y1);
    prefetchTensorMap(&p.y2);
    if (SIDE == kQueries) {
      prefetchTensorMap(&p.out);
      prefetchTensorMap(&p.rest);
    }
    mbarInit(xFull, 1);
    mbarInit(xEmpty, SIDE == kQueries ? 8 : 1);
    mbarInit(xReady, SIDE == kQueries ? 9 : 1);
    mbarInit(sFull, 1);
    mbarInit(sTaken, 9);
    mbarInit(dpFull, 1);
    mbarInit(dsReady, 9);
    mbarInit(done, 1);
    for (int s = 0; s < 2; s++) {
      mbarInit(&statFull[s], 1);
      mbarInit(&statEmpty[s], 1);
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
  if (SIDE == kKeys && warp < 4) {
    const uint32_t two = 0x3f803f80u, low = 0x3f80u, high = 0x3f800000u;  // bf16 ones
    uint4* rows = reinterpret_cast<uint4*>(extra) + threadIdx.x;  // X1's, X2's, of two streamed tiles, zeros
    rows[0] = make_uint4(two, low, 0, 0);
    rows[kTile] = make_uint4(0, high, two, 0);
    rows[4 * kTile] = make_uint4(0, 0, 0, 0);
    fenceProxyAsync();
  }
  tcFenceBefore();
  __syncthreads();
  tcFenceAfter();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmemSlot, 0);

  if (warp == 8) {
    setMaxRegsDown<C::kOtherRegs>();
    if (lane == 0) {
      uint32_t g = 0, turn = 1;  // tiles and items so far
      bool ok = true;
      for (int k = 0; ok && itemOf(k) < p.items; k++) {
        const Item it(p, itemOf(k));
        if (it.count == 0) continue;
        if (!(ok = mbarWait(xEmpty, turn, err, ERR_BWD_LOAD))) break;
        turn ^= 1;
        mbarArriveExpectTx(xFull, 2 * C::kTileBytes);
        for (int x = 0; x < C::kBoxes; x++) {
          tmaLoad4d(smemX + x * kBox, &p.x1, x * 64, it.x0, it.xh, it.b, xFull);
          tmaLoad4d(smemX + C::kTileBytes + x * kBox, &p.x2, x * 64, it.x0, it.xh, it.b, xFull);
        }
        int tile = it.firstTile(), h = it.yh;
        bool again = false;
        // Queries: the answer and what rounding took from it take the place of X when that is in tensor memory, delta is made of them; behind as many
        // streamed tiles as the ring takes meanwhile.
        const auto answer = [&]() {
          if (!(ok = mbarWait(xEmpty, turn, err, ERR_BWD_LOAD))) return;
          turn ^= 1;
          mbarArriveExpectTx(xFull, 2 * C::kTileBytes);
          for (int x = 0; x < C::kBoxes; x++) {
            tmaLoad4d(smemX + x * kBox, &p.out, x * 64, it.x0, it.xh, it.b, xFull);
            tmaLoad4d(smemX + C::kTileBytes + x * kBox, &p.rest, x * 64, it.x0, it.xh, it.b, xFull);
          }
        };
        for (int n = 0; n < it.count && ok; n++, g++) {
          const int y0 = tile * kTile;
          if constexpr (SIDE == kKeys) {  // first, as its place is free long before the tiles'
            if (!(ok = mbarWait(&statEmpty[g & 1], (g >> 1 & 1) ^ 1, err, ERR_BWD_LOAD))) break;
            mbarArriveExpectTx(&statFull[g & 1], C::kStat);
            bulkLoad(extra + (2 + (g & 1)) * C::kStat, a.stat + (((size_t)it.b * a.H + h) * a.padded() + y0) * 8, C::kStat, &statFull[g & 1]);
          }
          for (int w = 0; w < 2 && ok; w++) {
            const int s = w ? slot2(g) : slot1(g);
            if (!(ok = mbarWait(&empty[s], ringPhase(g) ^ 1, err, ERR_BWD_LOAD))) break;
            mbarArriveExpectTx(&full[s], C::kTileBytes);
            for (int x = 0; x < C::kBoxes; x++) tmaLoad4d(ring + s * C::kTileBytes + x * kBox, w ? &p.y2 : &p.y1, x * 64, y0, h, it.b, &full[s]);
          }
          it.next(tile, again);
          if (SIDE == kKeys && tile == it.yFirst && !again) h++;
          if (SIDE == kQueries && ok && n == min(1, it.count - 1)) answer();
        }
      }
      if (!ok) {  // let loads in flight land
        mbarWait(xFull, 0, err, 0, 2000u);
        for (int s = 0; s < C::kSlots; s++) mbarWait(&full[s], 0, err, 0, 2000u);
      }
    }
  } else if (warp == 9) {
    setMaxRegsDown<C::kOtherRegs>();
    constexpr uint32_t idescS = instrDesc(kTile, kTile, 1 /*bf16*/), idescAcc = instrDescMajor(kTile, HD, 1, 0, 1);
    // As in the forward kernel the whole warp walks along and one elected lane issues.
    const uint64_t descX = smemDescSw128(smemAddr(smemX)), descY = smemDescSw128(smemAddr(ring)), descSum = smemDescSw128Mn(smemAddr(ring), kBox);
    const auto product = [&](uint32_t d, int x, int s) {  // d = X Y^T
#pragma unroll
      for (int kk = 0; kk < HD / 16; kk++) {
        const uint32_t o = (kk / 4) * kBox + (kk % 4) * 32;
        const uint64_t y = descY + ((s * C::kTileBytes + o) >> 4);
        if (SIDE == kQueries) mmaF16FromTmem(tmem + d, tmem + (x ? C::kX2 : C::kX1) + kk * 8, y, idescS, kk != 0);
        else mmaF16(tmem + d, descX + ((x * C::kTileBytes + o) >> 4), y, idescS, kk != 0);
      }
    };
    // acc += W Y, W: two halves of the tile's columns, each packed into half of its own; FINE: and what rounding took from W
    const auto gather = [&](uint32_t acc, uint32_t w, uint32_t rest, int s, bool first) {
      constexpr int kSteps = kTile / 32;
#pragma unroll 1
      for (int part = 0; part < (FINE ? 2 : 1); part++, w = rest)
#pragma unroll
        for (int kk = 0; kk < kTile / 16; kk++)
          mmaF16FromTmem(tmem + acc, tmem + w + (kk / kSteps) * (kTile / 2) + (kk % kSteps) * 8, descSum + ((s * C::kTileBytes + kk * 2048) >> 4), idescAcc,
                         !first || part != 0 || kk != 0);
    };
    const auto further = [&](uint32_t d, int x, uint32_t g) {  // keys: the step of lse or delta
      const uint32_t at = smemAddr(extra);
      const int y = 2 + (g & 1);
      mmaF16(tmem + d, smemDescPlain(at + x * C::kStat, (4 - x) * C::kStat, 128), smemDescPlain(at + y * C::kStat, (4 - y) * C::kStat, 128), idescS, 1);
    };
    uint32_t g = 0, xPhase = 0;
    bool ok = true, all = true;  // of this lane's waits; of the warp's, looked at once per tile and off the products' way: waits behind one that was given up are short
    const auto wait = [&](uint64_t* bar, uint32_t parity) { ok = mbarWait(bar, parity, err, ERR_BWD_MMA) && ok; };
    for (int k = 0; all && itemOf(k) < p.items; k++) {
      const Item it(p, itemOf(k));
      if (it.count == 0) continue;
      const auto scores = [&](uint32_t g) {  // by the elected lane, as grads
        product(C::kS, 0, slot1(g));
        if (SIDE == kKeys) further(C::kS, 0, g);
        mmaCommit(sFull);
      };
      const auto grads = [&](uint32_t g) {
        product(C::kDp, 1, slot2(g));
        if (SIDE == kKeys) further(C::kDp, 1, g);
        mmaCommit(dpFull);
        mmaCommit(SIDE == kQueries ? &empty[slot2(g)] : &statEmpty[g & 1]);
      };
      wait(xReady, xPhase);  // the first tiles have landed too, see warp 10
      xPhase ^= 1;
      tcFenceAfter();
      if (electOne()) {
        scores(g);
        grads(g);
      }
      __syncwarp();
      for (int n = 0; n < it.count && all; n++, g++) {
        const bool more = n + 1 < it.count;
        constexpr bool kAhead = !(FINE && SIDE == kKeys);  // the next tile's scores may be made while this one's place is in use
        if (more && kAhead) {
          wait(sTaken, g & 1);
          tcFenceAfter();
          if (electOne()) scores(g + 1);
          __syncwarp();
        }
        wait(dsReady, g & 1);
        if (more && !kAhead) wait(sTaken, g & 1);
        tcFenceAfter();
        if (electOne()) {
          if constexpr (SIDE == kKeys) {
            gather(C::kAcc1, C::kDp, C::kS, slot2(g), n == 0);
            mmaCommit(&empty[slot2(g)]);
          }
          if constexpr (SIDE == kQueries) gather(C::kAcc1, C::kDp, C::kDp + 32, slot1(g), n == 0);
          else gather(C::kAcc2, C::kDp + 32, C::kS + 32, slot1(g), n == 0);
          mmaCommit(&empty[slot1(g)]);
          if (more && !kAhead) scores(g + 1);
          if (more) grads(g + 1);
          else {
            mmaCommit(done);
            if (SIDE == kKeys) mmaCommit(xEmpty);
          }
        }
        __syncwarp();
        all = __all_sync(0xffffffffu, ok);
      }
    }
  } else if (warp == 10) {
    // As in the forward kernel: looks after the landed tiles and takes part in the barriers that the issuing warp waits for.
    setMaxRegsDown<C::kOtherRegs>();
    uint32_t g = 0, xPhase = 0;
    bool ok = true;
    const auto landed = [&](const Item& it, int tile, uint32_t g, int which) {
      const int s = which ? slot2(g) : slot1(g);
      ok = ok && mbarWait(&full[s], ringPhase(g), err, ERR_BWD_MMA);
      if (SIDE == kKeys && which == 0) ok = ok && mbarWait(&statFull[g & 1], g >> 1 & 1, err, ERR_BWD_MMA);
      if ((SIDE == kKeys || which == 0) && it.straddles(tile)) zeroRows<C::kBoxes, kTile>(ring + s * C::kTileBytes, it.L - tile * kTile, lane);
      __syncwarp();
    };
    for (int k = 0; ok && itemOf(k) < p.items; k++) {
      const Item it(p, itemOf(k));
      if (it.count == 0) continue;
      int tile = it.firstTile();
      bool again = false;
      if (SIDE == kKeys) {
        ok = ok && mbarWait(xFull, xPhase, err, ERR_BWD_MMA);
        xPhase ^= 1;
      }
      landed(it, tile, g, 0);
      landed(it, tile, g, 1);
      if (lane == 0) mbarArrive(xReady);
      for (int n = 0; n < it.count && ok; n++, g++) {
        it.next(tile, again);
        if (n + 1 < it.count) landed(it, tile, g + 1, 0);
        if (lane == 0) mbarArrive(sTaken);
        if (n + 1 < it.count) landed(it, tile, g + 1, 1);
        if (lane == 0) mbarArrive(dsReady);
        ok = ok && mbarWait(sTaken, g & 1, err, ERR_BWD_MMA) && mbarWait(dsReady, g & 1, err, ERR_BWD_MMA);  // not ahead of them
      }
    }
  } else if (warp == 11) {
    setMaxRegsDown<C::kOtherRegs>();
  } else {
    setMaxRegsUp<C::kMathRegs>();
    constexpr int kCols = kTile / 2, kPairs = kCols / 2;   // of a tile's columns, this thread's
    constexpr int kWords = HD / 4;                         // of X's rows, this thread's
    const int q4 = warp & 3, side = warp >> 2, r = q4 * 32 + lane;
    const uint32_t base = tmem + ((uint32_t)(q4 * 32) << 16), cols = side * kCols;
    uint32_t g = 0, xPhase = 0, donePhase = 0;
    bool ok = true;
    uint32_t mine[kWords];  // queries: half a row of dO
    // The next item that has anything to do; what the others have to write is zeros.
    const auto advance = [&](int k) {
      for (; itemOf(k) < p.items; k++) {
        const Item it(p, itemOf(k));
        if (it.count) break;
        const int tid = threadIdx.x & 127;
        if constexpr (SIDE == kQueries) {
          if (side == 0) zeroOut(a.dq, it.b, it.xh, it.x0, a.S, a.D, tid);
        } else {
          if (it.far < 0) zeroOut(side ? a.dk : a.dv, it.b, it.xh, it.x0, a.S, a.D, tid);
          if (it.partRows)
            for (int n = tid; n < it.partRows * a.D; n += 128) it.part(p, side == 0)[n] = 0.f;
        }
      }
      return k;
    };
    // Words [4 i, 4 i + 4) of this thread's half of its row of X1 or X2 in shared memory.
    const auto rowWords = [&](int x, int i) {
      const uint8_t* row = smemX + x * C::kTileBytes + (HD == 128 ? side * kBox : 0) + r * 128;
      return *reinterpret_cast<const uint4*>(row + ((((HD == 128 ? 0 : side * 4) + i) ^ (r & 7)) << 4));
    };
    const auto copyX = [&]() {  // this thread's halves of X1's and X2's row to tensor memory
      if (!mbarWait(xFull, xPhase, err, ERR_BWD_MATH)) return false;
      xPhase ^= 1;
#pragma unroll
      for (int x = 0; x < 2; x++) {
#pragma unroll
        for (int i = 0; i < kWords; i += 4) {
          const uint4 v = rowWords(x, i / 4);
          mine[i] = v.x, mine[i + 1] = v.y, mine[i + 2] = v.z, mine[i + 3] = v.w;
        }
#pragma unroll
        for (int i = 0; i < kWords; i += 16) {
          uint32_t w[16];
#pragma unroll
          for (int e = 0; e < 16; e++) w[e] = mine[i + e];
          tmemStore16(base + (x ? C::kX2 : C::kX1) + side * kWords + i, w);
        }
      }
      tmemStoreWait();
      tcFenceBefore();
      __syncwarp();
      if (lane == 0) {
        mbarArrive(xReady);
        mbarArrive(xEmpty);
      }
      return true;
    };
    int k = advance(0);
    if (SIDE == kQueries && itemOf(k) < p.items) ok = copyX();
    while (ok && itemOf(k) < p.items) {
      const Item it(p, itemOf(k));
      const int row = it.x0 + r;
      const bool live = row < it.L;
      float lse = 0.f, delta = 0.f;
      if constexpr (SIDE == kQueries) {
        const size_t at = (size_t)it.bh * a.padded() + row;
        if (live) lse = a.lse[at];
        if (!(ok = mbarWait(xFull, xPhase, err, ERR_BWD_MATH))) break;
        xPhase ^= 1;
#pragma unroll
        for (int n = 0; n < kWords / 4; n++) {
          float x[8], y[8], z[8];
          unpack8(rowWords(0, n), x);
          unpack8(rowWords(1, n), y);
          unpack8(make_uint4(mine[4 * n], mine[4 * n + 1], mine[4 * n + 2], mine[4 * n + 3]), z);
#pragma unroll
          for (int i = 0; i < 8; i++) delta += (x[i] + y[i]) * z[i];
        }
        __syncwarp();
        if (lane == 0) mbarArrive(xEmpty);
        half[side * kTile + r] = delta;
        asm volatile("bar.sync 1, 256;" ::: "memory");
        delta = half[r] + half[kTile + r];
        asm volatile("bar.sync 1, 256;" ::: "memory");  // read by all before the next item's is written
        if (side == 0) {
          uint32_t w[3];
          __nv_bfloat16 part[6];
          const float of[2] = {live ? lse / p.c : 0.f, live ? -delta : 0.f};
#pragma unroll
          for (int i = 0; i < 2; i++) {
            part[3 * i] = __float2bfloat16(of[i]);
            const float rest = of[i] - __bfloat162float(part[3 * i]);
            part[3 * i + 1] = __float2bfloat16(rest);
            part[3 * i + 2] = __float2bfloat16(rest - __bfloat162float(part[3 * i + 1]));
          }
#pragma unroll
          for (int i = 0; i < 3; i++) w[i] = (uint32_t)__bfloat16_as_ushort(part[2 * i]) | (uint32_t)__bfloat16_as_ushort(part[2 * i + 1]) << 16;
          reinterpret_cast<uint4*>(a.stat)[at] = make_uint4(w[0], w[1], w[2], 0);
        }
      }
      const F2 c2 = makeF2(p.c, p.c), rowLse = makeF2(lse, lse), rowDelta = makeF2(-delta, -delta);
      const auto step = [&](int y0, auto rest) {  // rest: what rounding took
        const bool again = rest;
        const bool every = !again && (SIDE == kQueries ? it.x0 + kTile <= it.L && seesAll(a, it.x0, it.x0 + kTile - 1, y0)
                                                       : y0 + kTile <= it.L && seesAll(a, y0, y0 + kTile - 1, it.x0));
        uint32_t bits[kCols / 32];
        if (!every) {
#pragma unroll
          for (int x = 0; x < kCols / 32; x++) {
            const int y = y0 + cols + x * 32;
            if constexpr (SIDE == kQueries) {
              bits[x] = live ? maskBits(a, row, y) : 0u;
            } else {  // queries [row, end) see key `row`
              const auto below = [](int b) { return b <= 0 ? 0u : b >= 32 ? 0xffffffffu : (1u << b) - 1u; };
              const int end = row < a.sinks || a.window > it.L - row ? it.L : row + a.window;
              bits[x] = below(end - y) & ~below(row - y);
            }
          }
        }
        const auto masked = [&](F2 v, int e) {  // pair e of this thread's
          float lo, hi;
          splitF2(v, lo, hi);
          const uint32_t b = bits[e / 16] >> (2 * e % 32);
          return makeF2(b & 1 ? lo : 0.f, b & 2 ? hi : 0.f);
        };
        if (!mbarWait(sFull, g & 1, err, ERR_BWD_MATH)) return false;
        tcFenceAfter();
        F2 w[kPairs];  // the weights
        {
          uint32_t s[kCols / 32][32];
#pragma unroll
          for (int x = 0; x < kCols / 32; x++) tmemLoad32(base + C::kS + cols + x * 32, s[x]);
          tmemLoadWait();
          tcFenceBefore();
          __syncwarp();
          if (lane == 0) mbarArrive(sTaken);
          const auto weights = [&](auto all) {
#pragma unroll
            for (int e = 0; e < kPairs; e++) {
              const F2 score = makeF2(__uint_as_float(s[e / 16][2 * e % 32]), __uint_as_float(s[e / 16][2 * e % 32 + 1]));
              const F2 v = SIDE == kQueries ? fmaF2(score, c2, rowLse) : mulF2(score, c2);
              w[e] = decltype(all)::value ? exp2F2(v) : masked(exp2F2(v), e);
            }
          };
          if (every) weights(std::true_type{});
          else weights(std::false_type{});
        }
        if constexpr (FINE && SIDE == kKeys) {
#pragma unroll
          for (int x = 0; x < kCols / 32; x++) {
            uint32_t o[16];
#pragma unroll
            for (int e = 0; e < 16; e++) o[e] = pack2(remainder(w[x * 16 + e], pack2(w[x * 16 + e])));
            tmemStore16(base + C::kS + cols + x * 16, o);
          }
        }
        if (!mbarWait(dpFull, g & 1, err, ERR_BWD_MATH)) return false;
        tcFenceAfter();
        {
          uint32_t d[kCols / 32][32];
#pragma unroll
          for (int x = 0; x < kCols / 32; x++) tmemLoad32(base + C::kDp + cols + x * 32, d[x]);
          tmemLoadWait();
          if constexpr (SIDE == kKeys) {
#pragma unroll
            for (int x = 0; x < kCols / 32; x++) {
              uint32_t o[16];
#pragma unroll
              for (int e = 0; e < 16; e++) o[e] = pack2(w[x * 16 + e]);
              if (again)
#pragma unroll
                for (int e = 0; e < 16; e++) o[e] = pack2(remainder(w[x * 16 + e], o[e]));
              tmemStore16(base + C::kDp + cols + x * 16, o);
            }
          }
          const auto gradients = [&](auto all, auto rest) {
#pragma unroll
            for (int x = 0; x < kCols / 32; x++) {
              uint32_t o[16];
#pragma unroll
              for (int e = 0; e < 16; e++) {
                const F2 dp = makeF2(__uint_as_float(d[x][2 * e]), __uint_as_float(d[x][2 * e + 1]));
                F2 of = SIDE == kQueries ? addF2(dp, rowDelta) : dp;
                if (!decltype(all)::value) of = masked(of, x * 16 + e);  // what is masked may be anything
                const F2 v = mulF2(w[x * 16 + e], of);
                o[e] = pack2(v);
                if constexpr (FINE) d[x][e] = pack2(remainder(v, o[e]));
                if constexpr (decltype(rest)::value) o[e] = pack2(remainder(v, o[e]));
              }
              tmemStore16(base + C::kDp + cols + (SIDE == kKeys ? 32 : 0) + x * 16, o);
              if constexpr (FINE) {
#pragma unroll
                for (int e = 0; e < 16; e++) o[e] = d[x][e];
                tmemStore16(base + (SIDE == kKeys ? C::kS : C::kDp) + 32 + cols + x * 16, o);
              }
            }
          };
          if (!every) {  // rows that see one key alone (a sequence's first; all with a window of one): its weight is one whatever the score is
            const bool alone = a.window == 1 && a.sinks == 0;
#pragma unroll
            for (int x = 0; x < kCols / 32; x++) {
              if (alone || (SIDE == kQueries && row == 0)) bits[x] = 0;
              if (SIDE == kKeys && y0 + cols + x * 32 == 0) bits[x] &= ~1u;
            }
          }
          if (every) gradients(std::true_type{}, std::false_type{});
          else if (!again) gradients(std::false_type{}, std::false_type{});
          else gradients(std::false_type{}, std::bool_constant<!FINE>{});
        }
        tmemStoreWait();
        tcFenceBefore();
        __syncwarp();
        if (lane == 0) mbarArrive(dsReady);
        return true;
      };
      int tile = it.firstTile();
      bool again = false;
      for (int n = 0; n < it.count && ok; n++, g++) {
        const int y0 = tile * kTile;
        if constexpr (FINE) ok = step(y0, std::false_type{});
        else if constexpr (SIDE == kQueries) ok = step(y0, again);
        else ok = again ? step(y0, std::true_type{}) : step(y0, std::false_type{});
        it.next(tile, again);
      }
      if (!ok || !(ok = mbarWait(done, donePhase, err, ERR_BWD_MATH))) break;
      donePhase ^= 1;
      tcFenceAfter();
      k = advance(k + 1);
      if (SIDE == kQueries && itemOf(k) < p.items && !(ok = copyX())) break;

      // ---- the gradients: queries: each of a row's two threads has half of dQ's columns; keys: one has dV, the other dK
      const float f = SIDE == kKeys && side == 0 ? 1.f : a.scale;
      const uint32_t acc = base + (SIDE == kQueries ? C::kAcc1 + side * (HD / 2) : side ? C::kAcc2 : C::kAcc1);
      constexpr int kWidth = SIDE == kQueries ? HD / 2 : HD;
      const int col0 = SIDE == kQueries ? side * (HD / 2) : 0;
      const Tensor& dst = SIDE == kQueries ? a.dq : side ? a.dk : a.dv;
      const bool summed = r < it.partRows, written = it.far < 0 && !summed && row < a.S;
#pragma unroll 1
      for (int x = 0; x < kWidth / 32; x++) {
        uint32_t v[32];
        tmemLoad32(acc + x * 32, v);
        tmemLoadWait();
        const int col = col0 + x * 32;
        if (summed) {
          float* to = it.part(p, side == 0) + (size_t)r * a.D + col;
#pragma unroll
          for (int e = 0; e < 32; e += 4)
            if (col + e < a.D)
              *reinterpret_cast<float4*>(to + e) = live ? make_float4(__uint_as_float(v[e]), __uint_as_float(v[e + 1]), __uint_as_float(v[e + 2]), __uint_as_float(v[e + 3]))
                                                        : make_float4(0.f, 0.f, 0.f, 0.f);
        } else if (written) {
          uint32_t w[16];
#pragma unroll
          for (int e = 0; e < 16; e++) w[e] = live ? pack2(__uint_as_float(v[2 * e]) * f, __uint_as_float(v[2 * e + 1]) * f) : 0u;
          storeRow16(dst.at(it.b, it.xh, row) + col, w, (a.D - col) / 2, p.wide);
        }
      }
    }
  }
  tcFenceBefore();
  __syncthreads();
  if (warp == 9) tmemDealloc(tmem, C::kTmemCols);
}

// dK and dV of the sinks from the sums of their CTAs.
__global__ void __launch_bounds__(128) joinSinks(const __grid_constant__ BwdParams p) {
  const Args& a = p.a;
  const int j = blockIdx.x, bh = blockIdx.y, h = bh % a.KV, b = bh / a.KV, tile = j / kTile, pitch = min(a.sinks, kTile);
  const float* from = p.partials + (size_t)(bh * p.sinkTiles + tile) * (1 + p.farCount) * 2 * pitch * a.D + (size_t)(j % kTile) * a.D;
  for (int n = threadIdx.x; n < 2 * a.D; n += blockDim.x) {
    const int d = n % a.D, which = n / a.D;
    float v = 0.f;
    for (int x = 0; x <= p.farCount; x++) v += from[((size_t)2 * x + which) * pitch * a.D + d];
    (which ? a.dv : a.dk).at(b, h, j)[d] = __float2bfloat16(which ? v : v * a.scale);
  }
}

}  // namespace wattn
}  // namespace b200
