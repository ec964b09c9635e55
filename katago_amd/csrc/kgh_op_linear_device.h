// What the matrix products on the caller's tensors share: the loop of aligned tiles
// and the epilogue in registers.
#ifndef KGH_OP_LINEAR_DEVICE_H
#define KGH_OP_LINEAR_DEVICE_H

#include "kgh_conv_device.h"
#include "kgh_ops_device.h"

#include <algorithm>

namespace {

// Row strides (elements) from which a tile's offsets would pass 32 bits.
constexpr int64_t LIN_DMA_STRIDE = 1 << 22;

struct LinearArgs {
  const void* x;
  const void* w;
  const float* bias;
  const void* residual;
  void* out;
  int64_t ldx, ldw, ldr, ldo;
  int M, N, K;
  // K split over gridDim.y workgroups of `chunk` k each, their sums to
  // part[split][M][N] (linearJoinKernel adds them); null without a split.
  float* part;
  int chunk;
};

// What becomes of a sum, and the bits of a residual that is not there.
template<typename T, int ACT>
struct LinearFinish {
  static constexpr unsigned NO_RESIDUAL = 0;
  static __device__ __forceinline__ float activated(float sum, float bias) { return activate<T, ACT>(sum + bias); }
  static __device__ __forceinline__ float added(float y, float residual) { return y + residual; }
};

// Two groups of four columns, bias and activation, and the residual's 16 bytes of
// this lane's columns, to the 16 bytes of the same columns.
template<typename T, typename Finish>
__device__ __forceinline__ uint4 finishGroup(floatx4 v0, floatx4 v1, floatx4 b0, floatx4 b1, uint4 res) {
  const uint2 r01 = swapHalves(res.x, res.z), r23 = swapHalves(res.y, res.w);
  union Four {
    uint2 v;
    T e[4];
  } ra[2], oa[2];
  ra[0].v = make_uint2(r01.x, r23.x);
  ra[1].v = make_uint2(r01.y, r23.y);
#pragma unroll
  for(int e = 0; e < 4; e++) {
    oa[0].e[e] = (T)Finish::added(Finish::activated(v0[e], b0[e]), (float)ra[0].e[e]);
    oa[1].e[e] = (T)Finish::added(Finish::activated(v1[e], b1[e]), (float)ra[1].e[e]);
  }
  const uint2 o01 = swapHalves(oa[0].v.x, oa[1].v.x), o23 = swapHalves(oa[0].v.y, oa[1].v.y);
  return make_uint4(o01.x, o23.x, o01.y, o23.y);
}

// The epilogue of a wave's RB x CB blocks at row mBase, column nBase. The weights
// are the products' row operand, so a lane has four consecutive columns of row
// laneRow, and its partner lane ^ 32 the four behind them; in 16 bits two such
// groups of both swap halves into 16 consecutive bytes a lane.
template<typename T, int RB, int CB, typename Finish>
__device__ __forceinline__ void storeTile(const LinearArgs& a, const floatx16 (&acc)[RB][CB], int mBase, int nBase) {
  const int lane = threadIdx.x & 63, laneRow = lane & 31, half = lane >> 5;
  constexpr unsigned NONE = Finish::NO_RESIDUAL;
  const T* res = (const T*)a.residual;
  T* out = (T*)a.out;
  if constexpr(sizeof(T) == 2) {
    // A block that lies inside the result: all of the residual is under way before
    // the first of it is used.
    if(mBase + 32 * RB <= a.M && nBase + 32 * CB <= a.N && a.part == nullptr) {
      u32x4_t rv[RB][CB][2];
#pragma unroll
      for(int i = 0; i < RB; i++)
#pragma unroll
        for(int j = 0; j < CB; j++)
#pragma unroll
          for(int p = 0; p < 2; p++) {
            rv[i][j][p] = u32x4_t{NONE, NONE, NONE, NONE};
            if(res != nullptr)
              __builtin_memcpy(&rv[i][j][p], res + (int64_t)(mBase + i * 32 + laneRow) * a.ldr + nBase + j * 32 + (2 * p + half) * 8, 16);
          }
#pragma unroll
      for(int j = 0; j < CB; j++) {
        const int nj = nBase + j * 32;
        floatx4 bias[4];
#pragma unroll
        for(int q = 0; q < 4; q++) {
          bias[q] = (floatx4)0.0f;
          if(a.bias != nullptr) __builtin_memcpy(&bias[q], a.bias + nj + q * 8 + half * 4, 16);
        }
#pragma unroll
        for(int i = 0; i < RB; i++)
#pragma unroll
          for(int p = 0; p < 2; p++) {
            const u32x4_t r = rv[i][j][p];
            const floatx4 v0 = {acc[i][j][8 * p], acc[i][j][8 * p + 1], acc[i][j][8 * p + 2], acc[i][j][8 * p + 3]};
            const floatx4 v1 = {acc[i][j][8 * p + 4], acc[i][j][8 * p + 5], acc[i][j][8 * p + 6], acc[i][j][8 * p + 7]};
            const uint4 o = finishGroup<T, Finish>(v0, v1, bias[2 * p], bias[2 * p + 1], make_uint4(r.x, r.y, r.z, r.w));
            __builtin_memcpy(out + (int64_t)(mBase + i * 32 + laneRow) * a.ldo + nj + (2 * p + half) * 8, &o, 16);
          }
      }
      return;
    }
  }
#pragma unroll
  for(int j = 0; j < CB; j++) {
    const int nj = nBase + j * 32;
    floatx4 bias[4];
#pragma unroll
    for(int q = 0; q < 4; q++) {
      const int n = nj + q * 8 + half * 4;
      bias[q] = (floatx4)0.0f;
      if(a.bias != nullptr && n < a.N) {
        const uint4 u = loadGroupSmall(a.bias + n, a.N - n);
        bias[q] = *(const floatx4*)&u;
      }
    }
#pragma unroll
    for(int i = 0; i < RB; i++) {
      const int m = mBase + i * 32 + laneRow;
      if(sizeof(T) == 4 || a.part != nullptr) {
#pragma unroll
        for(int q = 0; q < 4; q++) {
          const int n = nj + q * 8 + half * 4;
          if(m >= a.M || n >= a.N) continue;
          floatx4 v = {acc[i][j][q * 4], acc[i][j][q * 4 + 1], acc[i][j][q * 4 + 2], acc[i][j][q * 4 + 3]};
          if(a.part != nullptr) {
            storeGroup(a.part + ((int64_t)blockIdx.y * a.M + m) * a.N + n, *(const uint4*)&v, a.N - n);
            continue;
          }
#pragma unroll
          for(int e = 0; e < 4; e++) v[e] = Finish::activated(v[e], bias[q][e]);
          if(res != nullptr) {
            const uint4 r = loadGroupSmall((const float*)a.residual + (int64_t)m * a.ldr + n, a.N - n);
            v += *(const floatx4*)&r;
          }
          storeGroup((float*)a.out + (int64_t)m * a.ldo + n, *(const uint4*)&v, a.N - n);
        }
      }
      else if constexpr(sizeof(T) == 2) {
        uint4 rv[2];
#pragma unroll
        for(int p = 0; p < 2; p++) {
          const int n = nj + (2 * p + half) * 8;
          rv[p] = make_uint4(NONE, NONE, NONE, NONE);
          if(res != nullptr && m < a.M && n < a.N) rv[p] = loadGroupSmall(res + (int64_t)m * a.ldr + n, a.N - n);
        }
#pragma unroll
        for(int p = 0; p < 2; p++) {
          const floatx4 v0 = {acc[i][j][8 * p], acc[i][j][8 * p + 1], acc[i][j][8 * p + 2], acc[i][j][8 * p + 3]};
          const floatx4 v1 = {acc[i][j][8 * p + 4], acc[i][j][8 * p + 5], acc[i][j][8 * p + 6], acc[i][j][8 * p + 7]};
          const uint4 o = finishGroup<T, Finish>(v0, v1, bias[2 * p], bias[2 * p + 1], rv[p]);
          const int n = nj + (2 * p + half) * 8;
          if(m < a.M && n < a.N) storeGroup(out + (int64_t)m * a.ldo + n, o, a.N - n);
        }
      }
    }
  }
}

// Rows that are 16-byte aligned (K whole groups of 16 bytes): tiles of WM x WN
// waves of 32 RB rows x 32 CB columns (KW = 2: twice as many, which share each
// step's K), steps of 128 bytes of K, whose rows L2 serves in one request. (Of 64
// bytes, in steps of half the K: 13 GB in 208 million requests for 8192 cubed, 0.8
// of what L2 takes, and 53% of the cycles with products; 0.6 times the rate.)
// A step's rows go from memory to LDS without registers, into the buffer that the
// last step has left; fragments are read one 32-byte part ahead of their products,
// over the step's border too: the barrier stands before a step's last part, whose
// fragments every wave then holds. The buffers are arrays of their own, so that the
// compiler does not make a fragment read wait for a load in flight to another one.
// early(column tile's first column, this wave's row and column) is called while the
// first steps' loads are under way; a barrier follows before the loop.
// Returns whether this wave has a block of the result, at row m and column n.
struct NothingEarly {
  __device__ __forceinline__ void operator()(int, int, int) const {}
};
template<typename T, int WM, int WN, int KW, int RB, int CB, typename Acc, typename Early = NothingEarly>
__device__ __forceinline__ bool dmaTile(const LinearArgs& a, int rowTiles, int colTiles, Acc (&acc)[RB][CB], int& m, int& n, Early early = Early()) {
  typedef typename Vec16<T>::V V;
  constexpr int SIZE = (int)sizeof(T), VEC = 16 / SIZE, STEP = 128 / SIZE;
  constexpr int WAVES = WM * WN * KW, PARTS = 4 / KW;  // a wave's 32-byte parts of a step
  constexpr int BM = 32 * RB * WM, BN = 32 * CB * WN;
  constexpr int A_PER = BM / 8 / WAVES, B_PER = BN / 8 / WAVES;  // loads of 8 rows a wave
  static_assert(A_PER * 8 * WAVES == BM && B_PER * 8 * WAVES == BN, "rows split evenly over the waves");
  __shared__ __attribute__((aligned(1024))) unsigned char a0s[BM * 128];
  __shared__ __attribute__((aligned(1024))) unsigned char a1s[BM * 128];
  __shared__ __attribute__((aligned(1024))) unsigned char b0s[BN * 128];
  __shared__ __attribute__((aligned(1024))) unsigned char b1s[BN * 128];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int laneRow = lane & 31, half = lane >> 5;
  int rowTile, colTile;
  blockedTile(rowTiles, colTiles, rowTile, colTile);
  const int m0 = rowTile * BM, n0 = colTile * BN;

  // A load's lane l writes slot l & 7 of row l >> 3 of eight, which holds the
  // row's group dGroup; load i of a wave is of the eight rows i * WAVES + wave, so
  // that the group is the same for all of them. Byte offsets of this lane's rows from the tile's first,
  // and how far the last step's group lies behind K.
  const int dRow = lane >> 3, dGroup = (lane & 7) ^ ((dRow >> 1) | ((wave & 1) << 2));
  static_assert(WAVES % 2 == 0, "a wave's rows of eight are all even or all odd");
  unsigned aOff[A_PER], bOff[B_PER];
#pragma unroll
  for(int i = 0; i < A_PER; i++) aOff[i] = (unsigned)(min(8 * (i * WAVES + wave) + dRow, a.M - 1 - m0) * a.ldx * SIZE) + dGroup * 16;
#pragma unroll
  for(int i = 0; i < B_PER; i++) bOff[i] = (unsigned)(min(8 * (i * WAVES + wave) + dRow, a.N - 1 - n0) * a.ldw * SIZE) + dGroup * 16;
  const int k0 = blockIdx.y * a.chunk;
  const int kEnd = min(k0 + a.chunk, a.K);
  const int last = (kEnd - k0 - 1) / STEP;
  const int groups = (kEnd - k0 - last * STEP) / VEC;  // of the last step
  const unsigned past = max(0, dGroup + 1 - groups) * 16;
  const char* xTile = (const char*)a.x + ((int64_t)m0 * a.ldx + k0) * SIZE;
  const char* wTile = (const char*)a.w + ((int64_t)n0 * a.ldw + k0) * SIZE;

  auto aBuf = [&](int i) -> unsigned char* { return i == 0 ? a0s : a1s; };
  auto bBuf = [&](int i) -> unsigned char* { return i == 0 ? b0s : b1s; };
  // Groups behind K read the row's last group; the last step's fragments have
  // zeros in their place.
  // Steps past the end read the last one again, into a buffer that nobody reads
  // any more (loads under a condition would have the compiler wait for them all).
  auto load = [&](auto buf, int st) {
    const int64_t at = (int64_t)min(st, last) * 128;
    const unsigned back = st >= last ? past : 0;
#pragma unroll
    for(int i = 0; i < A_PER; i++)
      __builtin_amdgcn_global_load_lds((const void*)(xTile + at + (aOff[i] - back)), (lds_void_t*)(aBuf(buf.value) + (i * WAVES + wave) * 1024), 16, 0, 0);
#pragma unroll
    for(int i = 0; i < B_PER; i++)
      __builtin_amdgcn_global_load_lds((const void*)(wTile + at + (bOff[i] - back)), (lds_void_t*)(bBuf(buf.value) + (i * WAVES + wave) * 1024), 16, 0, 0);
  };

#pragma unroll
  for(int i = 0; i < RB; i++)
#pragma unroll
    for(int j = 0; j < CB; j++)
#pragma unroll
      for(int r = 0; r < 16; r++) acc[i][j][r] = 0;
  const int kw = wave / (WM * WN);
  const int wm = wave % (WM * WN) / WN * 32 * RB, wn = wave % WN * 32 * CB;
  struct Frags {
    V a[RB], b[CB];
  };
  // 32 rows further the swizzle is the same: one offset per part and operand.
  int aAt[PARTS], bAt[PARTS];
#pragma unroll
  for(int s = 0; s < PARTS; s++) {
    aAt[s] = swizzled128(wm + laneRow, 2 * (kw * PARTS + s) + half);
    bAt[s] = swizzled128(wn + laneRow, 2 * (kw * PARTS + s) + half);
  }
  auto read = [&](const unsigned char* ab, const unsigned char* bb, int s, Frags& f) {
#pragma unroll
    for(int i = 0; i < RB; i++) f.a[i] = *(const V*)(ab + aAt[s] + i * 4096);
#pragma unroll
    for(int j = 0; j < CB; j++) f.b[j] = *(const V*)(bb + bAt[s] + j * 4096);
  };
  auto products = [&](const Frags& f) {
#pragma unroll
    for(int i = 0; i < RB; i++)
#pragma unroll
      for(int j = 0; j < CB; j++) acc[i][j] = mma32(f.b[j], f.a[i], acc[i][j]);
  };

  typedef std::integral_constant<int, 0> B0;
  typedef std::integral_constant<int, 1> B1;
  Frags f, g;  // f holds part 0 at a step's start
  // The reads stand behind the first product, whose wait for its own fragments
  // (the compiler waits for every read under way) then has nothing else to wait for.
  auto part = [&](const unsigned char* ab, const unsigned char* bb, int s, const Frags& now, Frags& ahead) {
    acc[0][0] = mma32(now.b[0], now.a[0], acc[0][0]);
    __builtin_amdgcn_sched_barrier(0);
    read(ab, bb, s, ahead);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for(int t = 1; t < RB * CB; t++) acc[t / CB][t % CB] = mma32(now.b[t % CB], now.a[t / CB], acc[t / CB][t % CB]);
    __builtin_amdgcn_sched_barrier(0);
  };
  auto step = [&](auto cur, auto next, int st) {
    part(aBuf(cur.value), bBuf(cur.value), 1, f, g);
    if constexpr(PARTS == 4) {
      part(aBuf(cur.value), bBuf(cur.value), 2, g, f);
      part(aBuf(cur.value), bBuf(cur.value), 3, f, g);
    }
    __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
    barrierNoFence();
    load(cur, st + 2);
    part(aBuf(next.value), bBuf(next.value), 0, g, f);
  };
  load(B0(), 0);
  load(B1(), 1);
  early(n0, m0 + wm, n0 + wn);
  __builtin_amdgcn_s_waitcnt(0x0070);
  barrierNoFence();
  read(a0s, b0s, 0, f);
  // Whole pairs in the loop: a way round it that left one out would have the
  // compiler wait for every load at its head.
  int st = 0;
  for(; st + 2 <= last; st += 2) {
    step(B0(), B1(), st);
    step(B1(), B0(), st + 1);
  }
  if(st < last) step(B0(), B1(), st);
#pragma unroll
  for(int s = 0; s < PARTS; s++) {
    const int group = 2 * (kw * PARTS + s);
    if(group >= groups) break;
    read(aBuf(last & 1), bBuf(last & 1), s, f);
    if(group + half >= groups) {
#pragma unroll
      for(int i = 0; i < RB; i++) f.a[i] = V{};
#pragma unroll
      for(int j = 0; j < CB; j++) f.b[j] = V{};
    }
    products(f);
  }

  // The loads past the end arrive before the LDS is used otherwise, here or by the
  // workgroup that has it next.
  waitVmcnt<0>();
  if constexpr(KW == 2) {
    // The two halves of K, added in order.
    static_assert(RB == 1 && CB == 1, "a wave's sums fit in its part of a buffer");
    auto* sums = (decltype(acc[0][0][0] + acc[0][0][0])*)a0s + (wave % (WM * WN)) * 1024 + lane;
    __syncthreads();
    if(kw == 1) {
#pragma unroll
      for(int r = 0; r < 16; r++) sums[r * 64] = acc[0][0][r];
    }
    __syncthreads();
    if(kw == 1) return false;
#pragma unroll
    for(int r = 0; r < 16; r++) acc[0][0][r] += sums[r * 64];
  }
  m = m0 + wm;
  n = n0 + wn;
  return true;
}

}  // namespace

#endif
