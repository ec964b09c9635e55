// Matrix product with bias, activation and residual in its epilogue
// (kgh_linear).
#include "kgh_conv_device.h"
#include "kgh_ops_device.h"

#include <algorithm>

namespace {

// Rows and channels are counted in 32 bits, with room for a tile past them; a
// launch counts its threads in 32 bits, 512 for 16 output channels.
constexpr int64_t LINEAR_MAX = 1 << 30, LINEAR_MAX_OUT = 1 << 26;
// Row strides from which a tile's offsets would pass 32 bits.
constexpr int64_t LIN_DMA_STRIDE = 1 << 22;
constexpr int LIN_ACTS[] = {KGH_ACT_IDENTITY, KGH_ACT_RELU, KGH_ACT_MISH, KGH_ACT_SILU, KGH_ACTIVATION_GELU};

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

// The activations: a result is rounded to its type once, so what a value left of 0
// keeps of itself (e^v or erfc) has to be right relative to itself, down to the type's
// smallest normal numbers.
constexpr float LIN_LOG2E = 1.44269504088896341f;

// For results in 16 bits, to within 2^-15 of the result. The exponential's
// instruction gives 0 below fp32's normal numbers, where v times it is not yet: it is
// taken 2^64 times as large or small, which the denominator or the polynomial's
// coefficients undo (a product may be below the normal numbers).
//   silu(v) = v / (1 + e^-v);
//   mish(v) = v n / (n + 2), n = e^v (e^v + 2); from 20 on v;
//   gelu(v) = v (1 - q), or v q left of 0, q = erfc(|v| / sqrt(2)) / 2 =
//             e^(-v^2 / 2) t P(t), t = 1 / (1 + p |v| / sqrt(2)): P and p fitted to
//             the smallest largest relative error, 4.2e-6 for all |v| < 14.1 (the
//             result is below every type's numbers behind).
// fp16 46208 x 384 x 1024, us: identity 62, SiLU 67, mish 71, GELU 77.
template<int ACT>
__device__ __forceinline__ float linActivateFast(float v) {
  if constexpr(ACT == KGH_ACT_SILU) return v * (__builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(fmaf(v, -LIN_LOG2E, -64.0f)) + 0x1p-64f) * 0x1p-64f);
  else if constexpr(ACT == KGH_ACT_MISH) {
    const float big = __builtin_amdgcn_exp2f(fmaf(fminf(v, 20.0f), LIN_LOG2E, 64.0f));
    const float n = big * fmaf(big, 0x1p-64f, 2.0f);
    return v * (n * __builtin_amdgcn_rcpf(n + 0x1p65f));
  }
  else {
    constexpr float S = 0x1p-65f;
    const float t = __builtin_amdgcn_rcpf(fmaf(0.435f * 0.70710678118654752f, fabsf(v), 1.0f));
    float poly = fmaf(t, S * -0.15086693f, S * 0.38131212f);
    poly = fmaf(t, poly, S * 0.01284851f);
    poly = fmaf(t, poly, S * 0.27344433f);
    poly = fmaf(t, poly, S * 0.23733569f);
    poly = fmaf(t, poly, S * 0.24592536f);
    const float q = t * poly * __builtin_amdgcn_exp2f(fmaf(v * v, -0.5f * LIN_LOG2E, 64.0f));
    return v * (v < 0.0f ? q : 1.0f - q);
  }
}

// For results in fp32, to within 2^-18 of the result: the same forms by the accurate functions.
template<int ACT>
__device__ __forceinline__ float linActivateFp32(float v) {
  if constexpr(ACT == KGH_ACTIVATION_GELU) {
    // erfc falls by 2 z times its argument's error, so what the argument's rounding
    // leaves is put right.
    constexpr float C = 0.70710678118654752f, REST = (float)(0.70710678118654752440 - (double)C);
    const float z = v * -C;
    const float rest = fmaf(v, -C, -z) - v * REST;
    float q = erfcf(z);
    if(z > 1.0f) q = fmaf(q * -2.0f * z, rest, q);
    return 0.5f * v * q;
  }
  else if(v < -20.0f) {
    // Both are v e^v to within 2^-28, by the exponential's root.
    const float root = expf(0.5f * v);
    return v * root * root;
  }
  else {
    const float e = expf(-fabsf(v)), twice = e + e;
    if constexpr(ACT == KGH_ACT_SILU) return v * ((v < 0.0f ? e : 1.0f) / (1.0f + e));
    else if(v < 0.0f) return v * (fmaf(e, e, twice) / (fmaf(e, e, twice) + 2.0f));
    else return v * ((1.0f + twice) / fmaf(twice, e, 1.0f + twice));
  }
}

template<typename T, int ACT>
__device__ __forceinline__ float linActivate(float v) {
  if constexpr(ACT == KGH_ACT_IDENTITY) return v;
  else if constexpr(ACT == KGH_ACT_RELU) return v < 0.0f ? 0.0f : v;  // NaN stays NaN
  else if constexpr(sizeof(T) == 4) return linActivateFp32<ACT>(v);
  else return linActivateFast<ACT>(v);
}

// Tiles of a launch in runs of 8 row tiles by 1 column tile, column after column,
// a contiguous part of them to each XCD: what the XCD's CUs work on at a time is
// about square, so its L2 serves each row of x and of the weights to several tiles.
__device__ __forceinline__ void blockedTile(int rowTiles, int colTiles, int& rowTile, int& colTile) {
  const int id = xcdContiguousTile();
  const int per = 8 * colTiles;
  const int run = id / per, at = id - run * per;
  const int height = min(8, rowTiles - run * 8);
  colTile = at / height;
  rowTile = run * 8 + (at - colTile * height);
}

// XOR swizzle of a row's eight 16-byte groups: the sixteen consecutive rows of a
// ds_read_b128 phase, the same group of each, fall in distinct banks (by row & 7 in
// place of (row >> 1) & 7, two rows would meet in each).
__device__ __forceinline__ int swizzled128(int row, int group) { return row * 128 + ((group ^ ((row >> 1) & 7)) << 4); }

// Two groups of four columns, bias and activation, and the residual's 16 bytes of
// this lane's columns, to the 16 bytes of the same columns.
template<typename T, int ACT>
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
    oa[0].e[e] = (T)(linActivate<T, ACT>(v0[e] + b0[e]) + (float)ra[0].e[e]);
    oa[1].e[e] = (T)(linActivate<T, ACT>(v1[e] + b1[e]) + (float)ra[1].e[e]);
  }
  const uint2 o01 = swapHalves(oa[0].v.x, oa[1].v.x), o23 = swapHalves(oa[0].v.y, oa[1].v.y);
  return make_uint4(o01.x, o23.x, o01.y, o23.y);
}

// The epilogue of a wave's RB x CB blocks at row mBase, column nBase. The weights
// are the products' row operand, so a lane has four consecutive columns of row
// laneRow, and its partner lane ^ 32 the four behind them; in 16 bits two such
// groups of both swap halves into 16 consecutive bytes a lane.
template<typename T, int RB, int CB, int ACT>
__device__ __forceinline__ void storeTile(const LinearArgs& a, const floatx16 (&acc)[RB][CB], int mBase, int nBase) {
  const int lane = threadIdx.x & 63, laneRow = lane & 31, half = lane >> 5;
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
            rv[i][j][p] = u32x4_t{0, 0, 0, 0};
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
            const uint4 o = finishGroup<T, ACT>(v0, v1, bias[2 * p], bias[2 * p + 1], make_uint4(r.x, r.y, r.z, r.w));
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
          for(int e = 0; e < 4; e++) v[e] = linActivate<T, ACT>(v[e] + bias[q][e]);
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
          rv[p] = make_uint4(0, 0, 0, 0);
          if(res != nullptr && m < a.M && n < a.N) rv[p] = loadGroupSmall(res + (int64_t)m * a.ldr + n, a.N - n);
        }
#pragma unroll
        for(int p = 0; p < 2; p++) {
          const floatx4 v0 = {acc[i][j][8 * p], acc[i][j][8 * p + 1], acc[i][j][8 * p + 2], acc[i][j][8 * p + 3]};
          const floatx4 v1 = {acc[i][j][8 * p + 4], acc[i][j][8 * p + 5], acc[i][j][8 * p + 6], acc[i][j][8 * p + 7]};
          const uint4 o = finishGroup<T, ACT>(v0, v1, bias[2 * p], bias[2 * p + 1], rv[p]);
          const int n = nj + (2 * p + half) * 8;
          if(m < a.M && n < a.N) storeGroup(out + (int64_t)m * a.ldo + n, o, a.N - n);
        }
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Any sizes, strides and alignment: tiles of 2 x 2 waves of 32 RB x 32 CB, steps of
// 128 bytes of K, loaded into registers two steps ahead, put into one LDS buffer
// while the other one's products run (fp32: one step ahead, one buffer, and two
// workgroups a CU that overlap). What is left of K behind the whole steps is a step
// of its own. Bound by the loads, which straddle cache lines where rows are not
// aligned: bf16 8192 x 4096 x 8192 830 to 858 us by the card (499 to 514 aligned).
//
// fp32 runs on the bf16 matrix cores: a number is three bf16 numbers to within
// 2^-27 of itself, a product the six bf16 products above 2^-27 of it, 6 x 32 cycles
// for 16 k of a 32 x 32 block where the fp32 instructions take 8 x 64. The pieces
// are put into LDS as three 64-byte runs and a gap a row (an odd number of 16-byte
// groups: the rows of a ds_read_b128 phase fall in distinct banks). 4096 cubed 744
// us (185 TFLOP/s; fp32 instructions 975, the library 895): with 128 x 128 tiles the
// splitting, about 200 vector instructions a step and wave, takes about as long as the
// products, and with 64 x 64 LDS is 0.9 busy. Small sizes run fp32 instructions.
// Pieces hold no number that rounds to a bf16 infinity, and of one below 2^-96 the
// third may lie below bf16's normal numbers. A tile that has met a small one, or whose
// sums are not all finite, is computed once more by the fp32 instructions (2.3 times
// its time in all). Only the first pieces are looked at, two a register, so numbers
// whose first piece is 0, below 2^-133, count as 0. (A look at every step that sends
// it to the fp32 instructions costs every product 8% more: 4096 cubed 805 us.)
typedef __bf16 bf16x4_t __attribute__((ext_vector_type(4)));
typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));
constexpr unsigned LIN_PIECES_FROM = 0x0f80;  // bits of 2^-96

// The smallest of the pieces but 0, by their bits twice and less one: 0 is the largest.
__device__ __forceinline__ u16x2_t smallestPiece(u16x2_t least, bf16x4_t piece) {
  u16x2_t u[2];
  __builtin_memcpy(u, &piece, 8);
#pragma unroll
  for(int i = 0; i < 2; i++) {
    u16x2_t twice;
    asm("v_pk_mad_u16 %0, %1, %2, %3" : "=v"(twice) : "v"(u[i]), "v"(0x00020002), "v"(0xffffffff));
    least = __builtin_elementwise_min(least, twice);
  }
  return least;
}
__device__ __forceinline__ void splitGroup(u32x4_t v, bf16x4_t (&piece)[3]) {
  float rest[4] = {__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), __uint_as_float(v.w)};
#pragma unroll
  for(int q = 0; q < 3; q++)
#pragma unroll
    for(int j = 0; j < 4; j++) {
      const __bf16 b = (__bf16)rest[j];
      piece[q][j] = b;
      rest[j] -= (float)b;
    }
}

template<typename T, int RB, int CB, int ACT>
__global__ __launch_bounds__(256, sizeof(T) == 4 ? (RB == 2 ? 2 : 4) : 1) void linearTileKernel(LinearArgs a, int rowTiles, int colTiles) {
  constexpr bool SPLIT = sizeof(T) == 4;
  constexpr int VEC = 16 / (int)sizeof(T), STEP = 8 * VEC;
  constexpr int BM = 64 * RB, BN = 64 * CB, LD = SPLIT ? 208 : 128, LOADS = 2 * (RB + CB);
  __shared__ __attribute__((aligned(16))) unsigned char lds0[(BM + BN) * LD];
  __shared__ __attribute__((aligned(16))) unsigned char lds1[SPLIT ? 16 : (BM + BN) * LD];
  __shared__ int again;  // whether a tile is computed once more
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int laneRow = lane & 31, half = lane >> 5;
  int rowTile, colTile;
  blockedTile(rowTiles, colTiles, rowTile, colTile);
  const int m0 = rowTile * BM, n0 = colTile * BN;
  const int kBegin = blockIdx.y * a.chunk, kEnd = min(kBegin + a.chunk, a.K);
  const int whole = (kEnd - kBegin) / STEP;

  // Thread t loads group t & 7 of rows t >> 3, + 32, ...
  const int lr = tid >> 3, lg = tid & 7;
  const T* src[LOADS];
#pragma unroll
  for(int i = 0; i < 2 * RB; i++) src[i] = (const T*)a.x + (int64_t)min(m0 + lr + 32 * i, a.M - 1) * a.ldx + kBegin + lg * VEC;
#pragma unroll
  for(int i = 0; i < 2 * CB; i++) src[2 * RB + i] = (const T*)a.w + (int64_t)min(n0 + lr + 32 * i, a.N - 1) * a.ldw + kBegin + lg * VEC;
  struct Rows {
    u32x4_t v[LOADS];
  };
  // Steps past the last whole one read that one again (into a buffer that nobody
  // reads): a condition here would keep the loads from staying in flight.
  auto fetch = [&](int step, Rows& r) {
    const int k = min(step, whole - 1) * STEP;
#pragma unroll
    for(int i = 0; i < LOADS; i++) __builtin_memcpy(&r.v[i], src[i] + k, 16);
  };
  u16x2_t least = {0xffff, 0xffff};
  auto stage = [&](unsigned char* lds, const Rows& r, auto pieces) {
#pragma unroll
    for(int i = 0; i < LOADS; i++) {
      if constexpr(decltype(pieces)::value) {
        bf16x4_t piece[3];
        splitGroup(r.v[i], piece);
        least = smallestPiece(least, piece[0]);
#pragma unroll
        for(int q = 0; q < 3; q++) *(bf16x4_t*)(lds + (lr + 32 * i) * LD + q * 64 + lg * 8) = piece[q];
      }
      else if constexpr(SPLIT) *(u32x4_t*)(lds + (lr + 32 * i) * LD + lg * 16) = r.v[i];
      else *(u32x4_t*)(lds + swizzled128(lr + 32 * i, lg)) = r.v[i];
    }
  };
  floatx16 acc[RB][CB];
  auto clear = [&] {
#pragma unroll
    for(int i = 0; i < RB; i++)
#pragma unroll
      for(int j = 0; j < CB; j++)
#pragma unroll
        for(int r = 0; r < 16; r++) acc[i][j][r] = 0.0f;
  };
  clear();
  const int wm = (wave >> 1) * 32 * RB, wn = (wave & 1) * 32 * CB;
  auto products = [&](const unsigned char* lds) {
    if constexpr(SPLIT) {
#pragma unroll
      for(int s = 0; s < 2; s++) {
        bf16x8_t af[RB][3], bf[CB][3];
#pragma unroll
        for(int q = 0; q < 3; q++) {
#pragma unroll
          for(int i = 0; i < RB; i++) af[i][q] = *(const bf16x8_t*)(lds + (wm + i * 32 + laneRow) * LD + q * 64 + s * 32 + half * 16);
#pragma unroll
          for(int j = 0; j < CB; j++) bf[j][q] = *(const bf16x8_t*)(lds + (BM + wn + j * 32 + laneRow) * LD + q * 64 + s * 32 + half * 16);
        }
        // The small products first.
        constexpr int PA[6] = {2, 0, 1, 1, 0, 0}, PB[6] = {0, 2, 1, 0, 1, 0};
#pragma unroll
        for(int p = 0; p < 6; p++)
#pragma unroll
          for(int i = 0; i < RB; i++)
#pragma unroll
            for(int j = 0; j < CB; j++) acc[i][j] = mma32(bf[j][PB[p]], af[i][PA[p]], acc[i][j]);
      }
    }
    else {
      typedef typename Vec16<T>::V V;
      V af[4][RB], bf[4][CB];
#pragma unroll
      for(int s = 0; s < 4; s++) {
#pragma unroll
        for(int i = 0; i < RB; i++) af[s][i] = *(const V*)(lds + swizzled128(wm + i * 32 + laneRow, 2 * s + half));
#pragma unroll
        for(int j = 0; j < CB; j++) bf[s][j] = *(const V*)(lds + swizzled128(BM + wn + j * 32 + laneRow, 2 * s + half));
      }
#pragma unroll
      for(int s = 0; s < 4; s++)
#pragma unroll
        for(int i = 0; i < RB; i++)
#pragma unroll
          for(int j = 0; j < CB; j++) acc[i][j] = mma32(bf[s][j], af[s][i], acc[i][j]);
    }
  };
  // fp32 numbers as they are.
  auto products32 = [&](const unsigned char* lds) {
    if constexpr(SPLIT) {
#pragma unroll
      for(int s = 0; s < 4; s++)
#pragma unroll
        for(int i = 0; i < RB; i++)
#pragma unroll
          for(int j = 0; j < CB; j++)
            acc[i][j] = mma32(*(const floatx4*)(lds + (BM + wn + j * 32 + laneRow) * LD + (2 * s + half) * 16),
                              *(const floatx4*)(lds + (wm + i * 32 + laneRow) * LD + (2 * s + half) * 16), acc[i][j]);
    }
  };
  auto put = [&](const Rows& r) {
    stage(lds0, r, std::integral_constant<bool, SPLIT>());
    barrierLds();
  };
  auto rest = [&](Rows& r) {
#pragma unroll
    for(int i = 0; i < LOADS; i++) {
      const uint4 u = loadGroupSmall(src[i] + whole * STEP, kEnd - kBegin - whole * STEP - lg * VEC);
      r.v[i] = u32x4_t{u.x, u.y, u.z, u.w};
    }
  };
  if constexpr(SPLIT) {
    if(tid == 0) again = 0;
    Rows r;
    if(whole > 0) fetch(0, r);
    for(int at = 0; at < whole; at++) {
      put(r);
      fetch(at + 1, r);
      __builtin_amdgcn_sched_barrier(0);
      products(lds0);
      barrierLds();
    }
  }
  else if(whole > 0) {
    auto step = [&](const unsigned char* now, unsigned char* then, Rows& use, Rows& load, int at) {
      fetch(at + 2, load);
      __builtin_amdgcn_sched_barrier(0);
      products(now);
      stage(then, use, std::false_type());
      barrierLds();
    };
    Rows r0, r1;
    fetch(0, r0);
    fetch(1, r1);
    put(r0);
    int at = 0;
    for(; at + 2 <= whole; at += 2) {
      step(lds0, lds1, r1, r0, at);
      step(lds1, lds0, r0, r1, at + 1);
    }
    if(at < whole) step(lds0, lds1, r1, r0, at);
  }
  if(kBegin + whole * STEP < kEnd) {
    Rows r;
    rest(r);
    put(r);
    products(lds0);
  }
  if constexpr(SPLIT) {
    // (0 times a sum that is infinite or NaN is NaN)
    float sum = 0.0f;
#pragma unroll
    for(int i = 0; i < RB; i++)
#pragma unroll
      for(int j = 0; j < CB; j++)
#pragma unroll
        for(int r = 0; r < 16; r++) sum = fmaf(0.0f, acc[i][j][r], sum);
    if(min(least[0], least[1]) < 2 * LIN_PIECES_FROM - 1 || sum != 0.0f) again = 1;
    __syncthreads();
    if(again != 0) {
      clear();
      Rows r;
      for(int at = 0; at <= whole; at++) {
        if(at < whole) fetch(at, r);
        else rest(r);
        __syncthreads();
        stage(lds0, r, std::false_type());
        __syncthreads();
        products32(lds0);
      }
    }
  }
  storeTile<T, RB, CB, ACT>(a, acc, m0 + wm, n0 + wn);
}

// ---------------------------------------------------------------------------
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
// bf16, us: 8192 x 8192 x 8192 847 (1298 TFLOP/s; the library 781), 8192 x 4096 x
// 8192 458, with bias, GELU and residual 505 (1089): of a 256 x 256 tile's 117,
// about 20 are its first loads and its stores, 10 more the residual and GELU. The
// power limit holds the clock at about 2 GHz.
template<typename T, int WM, int WN, int KW, int RB, int CB, int PER_CU, int ACT>
__global__ __launch_bounds__(64 * WM * WN * KW, PER_CU * WM * WN * KW / 4) void linearDmaKernel(LinearArgs a, int rowTiles, int colTiles) {
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

  floatx16 acc[RB][CB];
#pragma unroll
  for(int i = 0; i < RB; i++)
#pragma unroll
    for(int j = 0; j < CB; j++)
#pragma unroll
      for(int r = 0; r < 16; r++) acc[i][j][r] = 0.0f;
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
      for(int i = 0; i < RB; i++) f.a[i] = (V)(T)0.0f;
#pragma unroll
      for(int j = 0; j < CB; j++) f.b[j] = (V)(T)0.0f;
    }
    products(f);
  }

  // The loads past the end arrive before the LDS is used otherwise, here or by the
  // workgroup that has it next.
  waitVmcnt<0>();
  if constexpr(KW == 2) {
    // The two halves of K, added in order.
    static_assert(RB == 1 && CB == 1, "a wave's sums fit in its part of a buffer");
    float* sums = (float*)a0s + (wave % (WM * WN)) * 1024 + lane;
    __syncthreads();
    if(kw == 1) {
#pragma unroll
      for(int r = 0; r < 16; r++) sums[r * 64] = acc[0][0][r];
    }
    __syncthreads();
    if(kw == 1) return;
#pragma unroll
    for(int r = 0; r < 16; r++) acc[0][0][r] += sums[r * 64];
  }
  storeTile<T, RB, CB, ACT>(a, acc, m0 + wm, n0 + wn);
}

template<typename T, int WM, int WN, int KW, int RB, int CB, int PER_CU, int ACT>
void launchDma(const LinearArgs& a, int splits, hipStream_t stream) {
  constexpr int BM = 32 * RB * WM, BN = 32 * CB * WN;
  const int rowTiles = (a.M + BM - 1) / BM, colTiles = (a.N + BN - 1) / BN;
  linearDmaKernel<T, WM, WN, KW, RB, CB, PER_CU, ACT><<<dim3((unsigned)(rowTiles * colTiles), (unsigned)splits), 64 * WM * WN * KW, 0, stream>>>(a, rowTiles, colTiles);
}

// ---------------------------------------------------------------------------
// Few rows (at most 16 MT), any strides and alignment: the weights are read once,
// and what counts is how many of their bytes are under way. A workgroup has 16 NT
// output channels; its waves take units of 128 bytes of K in turn (every wave's
// loads of UNROLL units are issued before the first product), and their sums are
// added in wave order in LDS. bf16 8 x 4096 x 8192: 14.6 us, 4.6 TB/s; rows that are
// not aligned 32, each line read twice.
template<typename T, int MT, int NT, int WAVES, int UNROLL, int ACT>
__global__ __launch_bounds__(64 * WAVES) void linearSkinnyKernel(LinearArgs a) {
  typedef typename Vec16<T>::V V;
  constexpr int VEC = 16 / (int)sizeof(T);
  constexpr int UNIT = 8 * VEC;  // k of a unit: two products of 4 VEC
  __shared__ float sums[WAVES][MT * NT][4][64];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, quad = lane >> 4;
  const int n0 = blockIdx.x * 16 * NT;
  const T* wRow[NT];
  const T* xRow[MT];
#pragma unroll
  for(int j = 0; j < NT; j++) wRow[j] = (const T*)a.w + (int64_t)min(n0 + j * 16 + l16, a.N - 1) * a.ldw + quad * VEC;
#pragma unroll
  for(int i = 0; i < MT; i++) xRow[i] = (const T*)a.x + (int64_t)min(i * 16 + l16, a.M - 1) * a.ldx + quad * VEC;
  floatx4 acc[MT][NT];
#pragma unroll
  for(int i = 0; i < MT; i++)
#pragma unroll
    for(int j = 0; j < NT; j++) acc[i][j] = (floatx4)0.0f;

  auto run = [&](int k0, auto units, auto whole) {
    constexpr int U = decltype(units)::value;
    uint4 wv[U][2][NT], xv[U][2][MT];
#pragma unroll
    for(int u = 0; u < U; u++)
#pragma unroll
      for(int s = 0; s < 2; s++) {
        const int k = k0 + (u * WAVES * 2 + s) * 4 * VEC;
#pragma unroll
        for(int j = 0; j < NT; j++) {
          if constexpr(decltype(whole)::value) __builtin_memcpy(&wv[u][s][j], wRow[j] + k, 16);
          else wv[u][s][j] = loadGroup(wRow[j] + k, a.K - quad * VEC - k);
        }
#pragma unroll
        for(int i = 0; i < MT; i++) {
          if constexpr(decltype(whole)::value) __builtin_memcpy(&xv[u][s][i], xRow[i] + k, 16);
          else xv[u][s][i] = loadGroup(xRow[i] + k, a.K - quad * VEC - k);
        }
      }
#pragma unroll
    for(int u = 0; u < U; u++)
#pragma unroll
      for(int s = 0; s < 2; s++)
#pragma unroll
        for(int i = 0; i < MT; i++)
#pragma unroll
          for(int j = 0; j < NT; j++) acc[i][j] = mma16(*(const V*)&wv[u][s][j], *(const V*)&xv[u][s][i], acc[i][j]);
  };
  const int kEnd = min((int)(blockIdx.y + 1) * a.chunk, a.K);
  int k = blockIdx.y * a.chunk + wave * UNIT;
  for(; k + (UNROLL - 1) * WAVES * UNIT + UNIT <= kEnd; k += UNROLL * WAVES * UNIT) run(k, std::integral_constant<int, UNROLL>(), std::true_type());
  for(; k + UNIT <= kEnd; k += WAVES * UNIT) run(k, std::integral_constant<int, 1>(), std::true_type());
  if(k < kEnd) run(k, std::integral_constant<int, 1>(), std::false_type());

#pragma unroll
  for(int i = 0; i < MT; i++)
#pragma unroll
    for(int j = 0; j < NT; j++)
#pragma unroll
      for(int r = 0; r < 4; r++) sums[wave][i * NT + j][r][lane] = acc[i][j][r];
  __syncthreads();
  const T* res = (const T*)a.residual;
  for(int o = tid; o < 256 * MT * NT; o += 64 * WAVES) {
    const int c = o % (16 * NT), m = o / (16 * NT);
    const int n = n0 + c;
    if(n >= a.N || m >= a.M) continue;
    float v = 0.0f;
#pragma unroll
    for(int w = 0; w < WAVES; w++) v += sums[w][(m >> 4) * NT + (c >> 4)][c & 3][((c & 15) >> 2) * 16 + (m & 15)];
    if(a.part != nullptr) {
      a.part[((int64_t)blockIdx.y * a.M + m) * a.N + n] = v;
      continue;
    }
    v = linActivate<T, ACT>(v + (a.bias != nullptr ? a.bias[n] : 0.0f));
    if(res != nullptr) v += (float)res[(int64_t)m * a.ldr + n];
    ((T*)a.out)[(int64_t)m * a.ldo + n] = (T)v;
  }
}

template<typename T, int RB, int CB, int ACT>
void launchTile(const LinearArgs& a, int splits, hipStream_t stream) {
  const int rowTiles = (a.M + 64 * RB - 1) / (64 * RB), colTiles = (a.N + 64 * CB - 1) / (64 * CB);
  linearTileKernel<T, RB, CB, ACT><<<dim3((unsigned)(rowTiles * colTiles), (unsigned)splits), 256, 0, stream>>>(a, rowTiles, colTiles);
}

// The sums of K's splits added in their order, and the epilogue; a thread takes
// four columns.
template<typename T, int ACT>
__global__ __launch_bounds__(256) void linearJoinKernel(LinearArgs a, int splits) {
  const int cols = (a.N + 3) / 4;
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int m = (int)(id / cols), n = (int)(id - (int64_t)m * cols) * 4;
  if(m >= a.M) return;
  const int count = min(4, a.N - n);
  float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  const float* p = a.part + (int64_t)m * a.N + n;
#pragma unroll 4
  for(int s = 0; s < splits; s++) {
    const uint4 u = loadGroup(p + (int64_t)s * a.M * a.N, count);
    v[0] += __uint_as_float(u.x);
    v[1] += __uint_as_float(u.y);
    v[2] += __uint_as_float(u.z);
    v[3] += __uint_as_float(u.w);
  }
#pragma unroll
  for(int j = 0; j < 4; j++) {
    if(j >= count) break;
    float y = linActivate<T, ACT>(v[j] + (a.bias != nullptr ? a.bias[n + j] : 0.0f));
    if(a.residual != nullptr) y += (float)((const T*)a.residual)[(int64_t)m * a.ldr + n + j];
    ((T*)a.out)[(int64_t)m * a.ldo + n + j] = (T)y;
  }
}

template<typename T, int MT, int NT, int WAVES, int UNROLL, int ACT>
void launchSkinny(const LinearArgs& a, int splits, hipStream_t stream) {
  const dim3 grid((unsigned)((a.N + 16 * NT - 1) / (16 * NT)), (unsigned)splits);
  linearSkinnyKernel<T, MT, NT, WAVES, UNROLL, ACT><<<grid, 64 * WAVES, 0, stream>>>(a);
}

template<typename F>
void withLinearAct(int act, F&& f) {
  switch(act) {
    case KGH_ACTIVATION_RELU: f(std::integral_constant<int, KGH_ACT_RELU>()); break;
    case KGH_ACTIVATION_MISH: f(std::integral_constant<int, KGH_ACT_MISH>()); break;
    case KGH_ACTIVATION_SILU: f(std::integral_constant<int, KGH_ACT_SILU>()); break;
    case KGH_ACTIVATION_GELU: f(std::integral_constant<int, KGH_ACTIVATION_GELU>()); break;
    default: f(std::integral_constant<int, KGH_ACT_IDENTITY>()); break;
  }
}

}  // namespace

namespace kgh {

void checkLinear(const kgh_linear_params& p, bool pointers) {
  const char* op = "kgh_linear";
  opCheckDtype(op, p.dtype);
  if(std::find(std::begin(LIN_ACTS), std::end(LIN_ACTS), p.activation) == std::end(LIN_ACTS))
    opInvalid(op, "activation " + std::to_string(p.activation) + " is none of KGH_ACTIVATION_*");
  if(p.rows < 0 || p.rows > LINEAR_MAX) opInvalid(op, "rows " + std::to_string(p.rows) + " outside 0.." + std::to_string(LINEAR_MAX));
  if(p.in_channels < 1 || p.in_channels > LINEAR_MAX) opInvalid(op, "in_channels must be in 1.." + std::to_string(LINEAR_MAX));
  if(p.out_channels < 1 || p.out_channels > LINEAR_MAX_OUT) opInvalid(op, "out_channels must be in 1.." + std::to_string(LINEAR_MAX_OUT));
  // 64 x 64 tiles of 256 threads, counted in 32 bits by the launch.
  if((p.rows + 63) / 64 * ((p.out_channels + 63) / 64) >= (1 << 24)) opInvalid(op, "rows times out_channels is too large for one call");
  if(p.x_stride < 0 || p.weights_stride < 0 || p.residual_stride < 0) opInvalid(op, "negative stride");
  if(p.rows > 1 && p.out_stride < p.out_channels) opInvalid(op, "out_stride " + std::to_string(p.out_stride) + " is less than out_channels");
  if(!pointers || p.rows == 0) return;
  const size_t e = opElemBytes(p.dtype);
  opCheckPointer(op, "x", p.x, e);
  opCheckPointer(op, "weights", p.weights, e);
  opCheckPointer(op, "out", p.out, e);
  if(p.residual != nullptr) opCheckPointer(op, "residual", p.residual, e);
  if(p.bias != nullptr) opCheckPointer(op, "bias", p.bias, 4);
  if(p.workspace != nullptr) opCheckPointer(op, "workspace", p.workspace, 16);
  opCheckApart(op, "x", p.x, p.out);
  opCheckApart(op, "weights", p.weights, p.out);
  if(p.residual == p.out && p.rows > 1 && p.residual_stride != p.out_stride) opInvalid(op, "in place, residual_stride must be out_stride");
}

namespace {

enum LinearKernel { LIN_SKINNY, LIN_DMA_256, LIN_DMA_128, LIN_DMA_64, LIN_TILE_128, LIN_TILE_64 };
struct LinearPlan {
  LinearKernel kernel;
  int splits;  // of K
  int chunk;   // k of a split
};

// Which kernel runs, and in how many splits of K with `bytes` of workspace.
// Times are us a call on bf16 unless said otherwise, replayed from graphs, both
// sides of a rule measured together (later steps may have made both shorter).
LinearPlan planLinear(const kgh_linear_params& p, bool aligned, uint64_t bytes) {
  const auto tiles = [&](int64_t side) { return (p.rows + side - 1) / side * ((p.out_channels + side - 1) / side); };
  const int64_t size = (int64_t)opElemBytes(p.dtype), kBytes = p.in_channels * size;
  const int64_t big = tiles(256);
  LinearPlan plan;
  int64_t most = 1;  // splits worth their sums' way through memory and a second launch (about 3 us)
  if(p.rows <= 64) {
    // Against 64-row tiles: 8 x 4096 x 8192 14.6 (35.8), 64 x 4096 x 8192 30
    // (37.5), 48 x 8192 x 1024 33 (49). Split where few workgroups would each
    // have long rows: 16 x 8192 x 1024 in four 9.8 (16.7 whole), but 16 x 2048 x
    // 512 in two 7.9 (6.2).
    plan.kernel = LIN_SKINNY;
    if(kBytes >= 12288) most = std::min<int64_t>(256 / ((p.out_channels + 15) / 16), kBytes / 4096);
  }
  else if(p.dtype != KGH_DTYPE_FP32 && aligned && p.in_channels >= 1024 && big * 10 >= (big + 255) / 256 * 256 * 7) {
    // A tile a CU, where they fill at least 0.7 of their rounds and K is long
    // enough for a tile's start and end: 8192 x 4096 x 8192 505 (595 on 128 x
    // 128 tiles), 2888 x 4096 x 4096 102 (112); 46208 x 384 x 1152 83 (74).
    plan.kernel = LIN_DMA_256;
  }
  else if(tiles(128) >= 224 && (p.dtype == KGH_DTYPE_FP32 || !aligned)) {
    // fp32 5776 x 1024 x 1024 93 (106 on 64 x 64 tiles), 2888 x 384 x 1152 (207
    // tiles) 38 (33); unaligned 8192 x 4096 x 8192 830 (1358).
    plan.kernel = LIN_TILE_128;
  }
  else if(tiles(128) >= 224) {
    // 1000 x 4096 x 4096 (256 tiles) 53 (60 on 64 x 64 tiles), 5776 x 200 x 2000
    // 18.6 (20); 5776 x 384 x 384 (138) 9.6 (7.9).
    plan.kernel = LIN_DMA_128;
  }
  else {
    // Split as the skinny kernel: 128 x 4096 x 1024 in eight 12.1 (29.5 whole),
    // fp32 361 x 1024 x 384 in four 12.8 (18.2); 361 x 1024 x 384 in two 9.6 (6.8).
    plan.kernel = aligned ? LIN_DMA_64 : LIN_TILE_64;
    if(kBytes >= 4096) most = std::min<int64_t>(512 / tiles(64), kBytes / 1024);
  }
  const int64_t unit = 128 / size;  // k that a split is a multiple of
  const uint64_t one = (uint64_t)p.rows * p.out_channels * 4;
  const int64_t splits = std::max<int64_t>(1, std::min<int64_t>(most, (int64_t)std::min<uint64_t>(bytes / one, 1024)));
  plan.chunk = (int)((p.in_channels + splits * unit - 1) / (splits * unit) * unit);
  plan.splits = (p.in_channels + plan.chunk - 1) / plan.chunk;
  return plan;
}

template<typename T, int ACT>
void runLinear(const LinearPlan& plan, const LinearArgs& a, hipStream_t stream) {
  const int s = plan.splits;
  if(plan.kernel == LIN_SKINNY) {
    const bool wide = a.N >= 8192;  // 32 columns a workgroup still give every CU one: 32 x 4096 x 8192 20.8 us (24.9)
    if(a.M <= 16) launchSkinny<T, 1, 1, 8, 4, ACT>(a, s, stream);
    else if(a.M <= 32 && wide) launchSkinny<T, 2, 2, 8, 4, ACT>(a, s, stream);
    else if(a.M <= 32) launchSkinny<T, 2, 1, 8, 4, ACT>(a, s, stream);
    else if(wide) launchSkinny<T, 4, 2, 8, 2, ACT>(a, s, stream);
    else launchSkinny<T, 4, 1, 8, 2, ACT>(a, s, stream);
  }
  else if(plan.kernel == LIN_TILE_128) launchTile<T, 2, 2, ACT>(a, s, stream);
  else if(plan.kernel == LIN_TILE_64) launchTile<T, 1, 1, ACT>(a, s, stream);
  // fp32's products take long, so that what counts is an even share of them: 64 x
  // 32 tiles with K over two waves, 2888 x 1024 x 384 33.6 us (39.5 on 64 x 64; now 29.5).
  else if constexpr(sizeof(T) == 4) launchDma<T, 2, 1, 2, 1, 1, 4, ACT>(a, s, stream);
  else if(plan.kernel == LIN_DMA_256) launchDma<T, 2, 4, 1, 4, 2, 1, ACT>(a, s, stream);
  else if(plan.kernel == LIN_DMA_128) launchDma<T, 2, 2, 1, 2, 2, 2, ACT>(a, s, stream);
  else launchDma<T, 2, 2, 1, 1, 1, 4, ACT>(a, s, stream);
  KGH_CHECK_LAUNCH();
  if(s > 1) {
    const int64_t threads = (int64_t)a.M * ((a.N + 3) / 4);
    linearJoinKernel<T, ACT><<<dim3((unsigned)((threads + 255) / 256)), 256, 0, stream>>>(a, s);
    KGH_CHECK_LAUNCH();
  }
}

bool linearAligned(const kgh_linear_params& p) {
  const int vec = 16 / (int)opElemBytes(p.dtype);
  return (((uintptr_t)p.x | (uintptr_t)p.weights) & 15) == 0 && p.in_channels % vec == 0 && p.x_stride % vec == 0 && p.weights_stride % vec == 0 &&
         p.x_stride < LIN_DMA_STRIDE && p.weights_stride < LIN_DMA_STRIDE;
}

}  // namespace

// By the sizes alone: as if the rows were aligned.
uint64_t linearWorkspace(const kgh_linear_params& p) {
  if(p.rows == 0) return 0;
  const LinearPlan plan = planLinear(p, true, UINT64_MAX);
  return plan.splits > 1 ? (uint64_t)plan.splits * p.rows * p.out_channels * 4 : 0;
}

void launchLinear(const kgh_linear_params& p, hipStream_t stream) {
  if(p.rows == 0) return;
  const LinearPlan plan = planLinear(p, linearAligned(p), p.workspace != nullptr ? p.workspace_bytes : 0);
  const LinearArgs a{p.x, p.weights, p.bias, p.residual, p.out, p.x_stride, p.weights_stride, p.residual_stride, p.out_stride,
                     (int)p.rows, p.out_channels, p.in_channels, plan.splits > 1 ? (float*)p.workspace : nullptr, plan.chunk};
  withDtype(p.dtype, [&](auto t) { withLinearAct(p.activation, [&](auto act) { runLinear<decltype(t), decltype(act)::value>(plan, a, stream); }); });
}

}  // namespace kgh
