// Matrix product of 8-bit integers with scales for rows and channels
// (kgh_linear_int8).
#include "kgh_op_linear_device.h"

namespace {

// Rows and channels are counted in 32 bits, with room for a tile past them; a
// launch counts its threads in 32 bits.
constexpr int64_t LIN8_MAX = 1 << 30, LIN8_MAX_OUT = 1 << 26;

struct Scales {
  const float* x;
  const float* w;
};

// Bytes [k, end) of a row, up to 16 of them, zeros behind them: 16 bytes that lie in the
// row wherever it ends, moved to their places.
__device__ __forceinline__ u32x4_t loadBytes(const int8_t* row, int k, int end) {
  u32x4_t v = {0, 0, 0, 0};
  if(end >= 16) {
    const int at = min(k, end - 16), excess = min(k - at, 16);
    __builtin_memcpy(&v, row + at, 16);
    if(excess & 8) v = u32x4_t{v[2], v[3], 0, 0};
    if(excess & 4) v = u32x4_t{v[1], v[2], v[3], 0};
    const unsigned n = excess & 3;
    v = u32x4_t{__builtin_amdgcn_alignbyte(v[1], v[0], n), __builtin_amdgcn_alignbyte(v[2], v[1], n), __builtin_amdgcn_alignbyte(v[3], v[2], n), v[3] >> (8 * n)};
    return excess >= 16 ? u32x4_t{0, 0, 0, 0} : v;
  }
#pragma unroll 1
  for(int j = 0; j < 16; j++) {  // byte j enters at the top and moves down to its place
    v[0] = __builtin_amdgcn_alignbit(v[1], v[0], 8);
    v[1] = __builtin_amdgcn_alignbit(v[2], v[1], 8);
    v[2] = __builtin_amdgcn_alignbit(v[3], v[2], 8);
    v[3] = v[3] >> 8 | (k + j < end ? (unsigned)(uint8_t)row[k + j] << 24 : 0);
  }
  return v;
}

// A result's steps, each rounded by itself and to 32 bits in every kernel, so that a
// call's bits depend on neither kernel nor workspace: the compiler would else take the
// activation's last product and the residual into one operation, or into the conversion
// to 16 bits, in some kernels and not in others.
__device__ __forceinline__ float rounded(float v) {
  asm("" : "+v"(v));
  return v;
}
// A sum's value with its bias: the sum's conversion, a product, and a product and sum
// rounded once.
__device__ __forceinline__ float scaled(int sum, float x, float w, float bias) { return rounded(fmaf((float)sum * x, w, bias)); }
// (a residual that is not there is -0: it leaves every number as it is, -0 too)
template<typename T, int ACT>
struct Int8Finish {
  static constexpr unsigned NO_RESIDUAL = 0x80008000u;
  static __device__ __forceinline__ float activated(float scaled, float) { return rounded(activate<T, ACT>(scaled)); }
  static __device__ __forceinline__ float added(float y, float residual) { return rounded(y + residual); }
};

// storeTile of sums: by their scales, or as they are where K is split.
template<typename T, int RB, int CB, int ACT>
__device__ __forceinline__ void storeSums(LinearArgs a, const Scales& s, const intx16 (&sums)[RB][CB], int m, int n) {
  const int lane = threadIdx.x & 63, laneRow = lane & 31, half = lane >> 5;
  floatx16 acc[RB][CB];
  if(a.part != nullptr) {
#pragma unroll
    for(int i = 0; i < RB; i++)
#pragma unroll
      for(int j = 0; j < CB; j++) acc[i][j] = __builtin_bit_cast(floatx16, sums[i][j]);
  }
  else {
    float x[RB];
#pragma unroll
    for(int i = 0; i < RB; i++) x[i] = s.x[min(m + i * 32 + laneRow, a.M - 1)];
#pragma unroll
    for(int j = 0; j < CB; j++)
#pragma unroll
      for(int q = 0; q < 4; q++) {
        const int c = n + j * 32 + q * 8 + half * 4, at = min(c, a.N - 1), count = c < a.N ? a.N - c : 1;
        const uint4 u = loadGroupSmall(s.w + at, count);
        const uint4 v = a.bias != nullptr ? loadGroupSmall(a.bias + at, count) : make_uint4(0, 0, 0, 0);
        const floatx4 w = *(const floatx4*)&u, b = *(const floatx4*)&v;
#pragma unroll
        for(int i = 0; i < RB; i++)
#pragma unroll
          for(int e = 0; e < 4; e++) acc[i][j][4 * q + e] = scaled(sums[i][j][4 * q + e], x[i], w[e], b[e]);
      }
    a.bias = nullptr;
  }
  storeTile<T, RB, CB, Int8Finish<T, ACT>>(a, acc, m, n);
}

// What a wave's block of the result needs beside the sums, for blocks that lie inside it
// (in 16 bits): loaded while the first steps are under way, the columns' scales and biases
// into LDS.
template<typename T, int RB, int CB>
struct EarlyLoads {
  float x[RB];
  u32x4_t residual[RB][CB][2];
};

// Two groups of four columns to the 16 bytes of the same columns, as finishGroup.
template<typename T, int ACT, bool RES>
__device__ __forceinline__ uint4 finishSums(const int (&s0)[4], const int (&s1)[4], float x, floatx4 w0, floatx4 w1, floatx4 b0, floatx4 b1, u32x4_t res) {
  typedef Int8Finish<T, ACT> Finish;
  union Four {
    uint2 v;
    T e[4];
  } ra[2], oa[2];
  if constexpr(RES) {
    const uint2 r01 = swapHalves(res.x, res.z), r23 = swapHalves(res.y, res.w);
    ra[0].v = make_uint2(r01.x, r23.x);
    ra[1].v = make_uint2(r01.y, r23.y);
  }
#pragma unroll
  for(int e = 0; e < 4; e++) {
    const float v0 = Finish::activated(scaled(s0[e], x, w0[e], b0[e]), 0.0f), v1 = Finish::activated(scaled(s1[e], x, w1[e], b1[e]), 0.0f);
    oa[0].e[e] = (T)(RES ? Finish::added(v0, (float)ra[0].e[e]) : v0);
    oa[1].e[e] = (T)(RES ? Finish::added(v1, (float)ra[1].e[e]) : v1);
  }
  const uint2 o01 = swapHalves(oa[0].v.x, oa[1].v.x), o23 = swapHalves(oa[0].v.y, oa[1].v.y);
  return make_uint4(o01.x, o23.x, o01.y, o23.y);
}

// columns: scales of this wave's columns, their biases BN behind them.
template<typename T, int RB, int CB, int ACT, bool RES, int BN>
__device__ __forceinline__ void storeInside(const LinearArgs& a, const intx16 (&sums)[RB][CB], const EarlyLoads<T, RB, CB>& early, const float* columns, int m, int n) {
  const int lane = threadIdx.x & 63, laneRow = lane & 31, half = lane >> 5;
  T* out = (T*)a.out + (int64_t)(m + laneRow) * a.ldo + n;
#pragma unroll
  for(int j = 0; j < CB; j++)
#pragma unroll
    for(int p = 0; p < 2; p++) {
      const float* c = columns + j * 32 + p * 16 + half * 4;
      const floatx4 w0 = *(const floatx4*)c, w1 = *(const floatx4*)(c + 8), b0 = *(const floatx4*)(c + BN), b1 = *(const floatx4*)(c + BN + 8);
#pragma unroll
      for(int i = 0; i < RB; i++) {
        const intx16& t = sums[i][j];
        const int s0[4] = {t[8 * p], t[8 * p + 1], t[8 * p + 2], t[8 * p + 3]}, s1[4] = {t[8 * p + 4], t[8 * p + 5], t[8 * p + 6], t[8 * p + 7]};
        const uint4 o = finishSums<T, ACT, RES>(s0, s1, early.x[i], w0, w1, b0, b1, RES ? early.residual[i][j][p] : u32x4_t{0, 0, 0, 0});
        __builtin_memcpy(out + (int64_t)i * 32 * a.ldo + j * 32 + (2 * p + half) * 8, &o, 16);
      }
    }
}

// ---------------------------------------------------------------------------
// Rows that are 16-byte aligned: dmaTile's loop, 128 k a step. 8192 x 4096 x 8192 bf16 on
// 256 x 256 tiles: 287 us, 1915 TOP/s (the library's product, without scales, 267), at
// the clock that the power limit leaves (1.66 GHz); GELU and a residual add 46, a tile's
// end which nothing covers on one workgroup a CU. 46208 x 1024 x 384 fp16 with a residual
// on 128 x 128: 42 us, 2.8 TB/s, a tile's first loads and stores around eight steps; with
// the epilogue's own loads behind the steps 54.
template<typename T, int WM, int WN, int RB, int CB, int PER_CU, int ACT>
__global__ __launch_bounds__(64 * WM * WN, PER_CU * WM * WN / 4) void linear8DmaKernel(LinearArgs a, Scales s, int rowTiles, int colTiles) {
  intx16 acc[RB][CB];
  int m, n;
  // (blocks of more registers leave no room for what is loaded early)
  if constexpr(sizeof(T) == 2 && RB * CB <= 4) {
    constexpr int BN = 32 * CB * WN;
    __shared__ __attribute__((aligned(16))) float columns[2 * BN];  // scales, biases
    const int lane = threadIdx.x & 63, laneRow = lane & 31, half = lane >> 5;
    EarlyLoads<T, RB, CB> early;
    int column = 0;
    bool inside = false;
    dmaTile<int8_t, WM, WN, 1, RB, CB>(a, rowTiles, colTiles, acc, m, n, [&](int n0, int row, int col) {
      inside = a.part == nullptr && row + 32 * RB <= a.M && col + 32 * CB <= a.N;
      column = col - n0;
#pragma unroll
      for(int i = 0; i < RB; i++) early.x[i] = s.x[min(row + i * 32 + laneRow, a.M - 1)];
      if(inside && a.residual != nullptr) {
        const T* res = (const T*)a.residual + (int64_t)(row + laneRow) * a.ldr + col;
#pragma unroll
        for(int i = 0; i < RB; i++)
#pragma unroll
          for(int j = 0; j < CB; j++)
#pragma unroll
            for(int p = 0; p < 2; p++) __builtin_memcpy(&early.residual[i][j][p], res + (int64_t)i * 32 * a.ldr + j * 32 + (2 * p + half) * 8, 16);
      }
      for(int c = threadIdx.x; c < BN; c += 64 * WM * WN) {
        const int at = min(n0 + c, a.N - 1);
        columns[c] = s.w[at];
        columns[BN + c] = a.bias != nullptr ? a.bias[at] : 0.0f;
      }
    });
    if(inside) {
      if(a.residual != nullptr) storeInside<T, RB, CB, ACT, true, BN>(a, acc, early, columns + column, m, n);
      else storeInside<T, RB, CB, ACT, false, BN>(a, acc, early, columns + column, m, n);
    }
    else storeSums<T, RB, CB, ACT>(a, s, acc, m, n);
  }
  else {
    dmaTile<int8_t, WM, WN, 1, RB, CB>(a, rowTiles, colTiles, acc, m, n);
    storeSums<T, RB, CB, ACT>(a, s, acc, m, n);
  }
}

// ---------------------------------------------------------------------------
// Any strides and alignment: tiles of 2 x 2 waves of 32 RB x 32 CB, steps of 128 bytes
// of K, loaded into registers two steps ahead, put into one LDS buffer while the other
// one's products run. 8192 x 4096 x 8192 bf16, rows 7 bytes apart, 612 us, 46208 x 1000 x
// 384 bf16 66. In 16 bits 128 x 128 tiles take 257 to 272 registers a lane, so that a SIMD
// has one wave, and nothing covers a step's wait; whether that bounds it or loads that
// straddle cache lines do is not measured.
template<typename T, int RB, int CB, int ACT>
__global__ __launch_bounds__(256) void linear8TileKernel(LinearArgs a, Scales s, int rowTiles, int colTiles) {
  constexpr int STEP = 128, BM = 64 * RB, BN = 64 * CB, LOADS = 2 * (RB + CB);
  __shared__ __attribute__((aligned(16))) unsigned char lds0[(BM + BN) * 128];
  __shared__ __attribute__((aligned(16))) unsigned char lds1[(BM + BN) * 128];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int laneRow = lane & 31, half = lane >> 5;
  int rowTile, colTile;
  blockedTile(rowTiles, colTiles, rowTile, colTile);
  const int m0 = rowTile * BM, n0 = colTile * BN;
  const int kBegin = blockIdx.y * a.chunk, kEnd = min(kBegin + a.chunk, a.K);
  const int whole = (kEnd - kBegin) / STEP;
  // Thread t loads group t & 7 of rows t >> 3, + 32, ...
  const int lr = tid >> 3, lg = tid & 7;
  const int8_t* src[LOADS];  // the rows' first bytes of this part of K
#pragma unroll
  for(int i = 0; i < 2 * RB; i++) src[i] = (const int8_t*)a.x + (int64_t)min(m0 + lr + 32 * i, a.M - 1) * a.ldx + kBegin;
#pragma unroll
  for(int i = 0; i < 2 * CB; i++) src[2 * RB + i] = (const int8_t*)a.w + (int64_t)min(n0 + lr + 32 * i, a.N - 1) * a.ldw + kBegin;
  struct Rows {
    u32x4_t v[LOADS];
  };
  // Steps past the last whole one read that one again, into a buffer that nobody reads.
  auto fetch = [&](int step, Rows& r) {
    const int k = min(step, whole - 1) * STEP + lg * 16;
#pragma unroll
    for(int i = 0; i < LOADS; i++) __builtin_memcpy(&r.v[i], src[i] + k, 16);
  };
  auto stage = [&](unsigned char* lds, const Rows& r) {
#pragma unroll
    for(int i = 0; i < LOADS; i++) *(u32x4_t*)(lds + swizzled128(lr + 32 * i, lg)) = r.v[i];
  };
  intx16 acc[RB][CB];
#pragma unroll
  for(int i = 0; i < RB; i++)
#pragma unroll
    for(int j = 0; j < CB; j++)
#pragma unroll
      for(int r = 0; r < 16; r++) acc[i][j][r] = 0;
  const int wm = (wave >> 1) * 32 * RB, wn = (wave & 1) * 32 * CB;
  auto products = [&](const unsigned char* lds) {
    intx4 af[4][RB], bf[4][CB];
#pragma unroll
    for(int p = 0; p < 4; p++) {
#pragma unroll
      for(int i = 0; i < RB; i++) af[p][i] = *(const intx4*)(lds + swizzled128(wm + i * 32 + laneRow, 2 * p + half));
#pragma unroll
      for(int j = 0; j < CB; j++) bf[p][j] = *(const intx4*)(lds + swizzled128(BM + wn + j * 32 + laneRow, 2 * p + half));
    }
#pragma unroll
    for(int p = 0; p < 4; p++)
#pragma unroll
      for(int i = 0; i < RB; i++)
#pragma unroll
        for(int j = 0; j < CB; j++) acc[i][j] = mma32(bf[p][j], af[p][i], acc[i][j]);
  };
  if(whole > 0) {
    auto step = [&](const unsigned char* now, unsigned char* then, Rows& use, Rows& load, int at) {
      fetch(at + 2, load);
      __builtin_amdgcn_sched_barrier(0);
      products(now);
      stage(then, use);
      barrierLds();
    };
    Rows r0, r1;
    fetch(0, r0);
    fetch(1, r1);
    stage(lds0, r0);
    barrierLds();
    int at = 0;
    for(; at + 2 <= whole; at += 2) {
      step(lds0, lds1, r1, r0, at);
      step(lds1, lds0, r0, r1, at + 1);
    }
    if(at < whole) step(lds0, lds1, r1, r0, at);
  }
  if(kBegin + whole * STEP < kEnd) {
    Rows r;
#pragma unroll
    for(int i = 0; i < LOADS; i++) r.v[i] = loadBytes(src[i], whole * STEP + lg * 16, kEnd - kBegin);
    stage(lds0, r);
    barrierLds();
    products(lds0);
  }
  storeSums<T, RB, CB, ACT>(a, s, acc, m0 + wm, n0 + wn);
}

// ---------------------------------------------------------------------------
// Few rows (at most 16 MT), any strides and alignment: the weights are read once. A
// workgroup has 16 NT output channels; its waves take units of 128 bytes of K in turn
// (every wave's loads of UNROLL units are issued before the first product: 32 x 4096 x
// 8192 12.1 us, 15.4 where the compiler spreads them), and their sums meet in LDS. 1 x
// 4096 x 8192 bf16: 8.4 us, 4.0 TB/s; x, which every workgroup loads, costs the more the
// more rows it has: 8 rows 9.4, 16 10.6.
template<typename T, int MT, int NT, int WAVES, int UNROLL, int ACT>
__global__ __launch_bounds__(64 * WAVES) void linear8SkinnyKernel(LinearArgs a, Scales s) {
  constexpr int UNIT = 128;
  __shared__ int sums[WAVES][MT * NT][4][64];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, quad = lane >> 4;
  const int n0 = blockIdx.x * 16 * NT;
  const int8_t* wRow[NT];
  const int8_t* xRow[MT];
#pragma unroll
  for(int j = 0; j < NT; j++) wRow[j] = (const int8_t*)a.w + (int64_t)min(n0 + j * 16 + l16, a.N - 1) * a.ldw;
#pragma unroll
  for(int i = 0; i < MT; i++) xRow[i] = (const int8_t*)a.x + (int64_t)min(i * 16 + l16, a.M - 1) * a.ldx;
  intx4 acc[MT][NT];
#pragma unroll
  for(int i = 0; i < MT; i++)
#pragma unroll
    for(int j = 0; j < NT; j++) acc[i][j] = intx4{0, 0, 0, 0};
  const int kEnd = min((int)(blockIdx.y + 1) * a.chunk, a.K);
  auto run = [&](int k0, auto units, auto whole) {
    constexpr int U = decltype(units)::value;
    u32x4_t wv[U][2][NT], xv[U][2][MT];
#pragma unroll
    for(int u = 0; u < U; u++)
#pragma unroll
      for(int p = 0; p < 2; p++) {
        const int k = k0 + (u * WAVES * 2 + p) * 64 + quad * 16;
#pragma unroll
        for(int j = 0; j < NT; j++) {
          if constexpr(decltype(whole)::value) __builtin_memcpy(&wv[u][p][j], wRow[j] + k, 16);
          else wv[u][p][j] = loadBytes(wRow[j], k, kEnd);
        }
#pragma unroll
        for(int i = 0; i < MT; i++) {
          if constexpr(decltype(whole)::value) __builtin_memcpy(&xv[u][p][i], xRow[i] + k, 16);
          else xv[u][p][i] = loadBytes(xRow[i], k, kEnd);
        }
      }
    __builtin_amdgcn_sched_barrier(0);  // every load before the first product
#pragma unroll
    for(int u = 0; u < U; u++)
#pragma unroll
      for(int p = 0; p < 2; p++)
#pragma unroll
        for(int i = 0; i < MT; i++)
#pragma unroll
          for(int j = 0; j < NT; j++) acc[i][j] = mma16(*(const intx4*)&wv[u][p][j], *(const intx4*)&xv[u][p][i], acc[i][j]);
  };
  int k = blockIdx.y * a.chunk + wave * UNIT;
  // (a second loop of one unit each would be the same sums)
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
  for(int o = tid; o < 256 * MT * NT; o += 64 * WAVES) {
    const int c = o % (16 * NT), m = o / (16 * NT);
    const int n = n0 + c;
    if(n >= a.N || m >= a.M) continue;
    int sum = 0;
#pragma unroll
    for(int w = 0; w < WAVES; w++) sum += sums[w][(m >> 4) * NT + (c >> 4)][c & 3][((c & 15) >> 2) * 16 + (m & 15)];
    if(a.part != nullptr) {
      ((int*)a.part)[((int64_t)blockIdx.y * a.M + m) * a.N + n] = sum;
      continue;
    }
    float v = Int8Finish<T, ACT>::activated(scaled(sum, s.x[m], s.w[n], a.bias != nullptr ? a.bias[n] : 0.0f), 0.0f);
    if(a.residual != nullptr) v = Int8Finish<T, ACT>::added(v, (float)((const T*)a.residual)[(int64_t)m * a.ldr + n]);
    ((T*)a.out)[(int64_t)m * a.ldo + n] = (T)v;
  }
}

// The sums of K's splits, and the epilogue; a thread takes four columns.
template<typename T, int ACT>
__global__ __launch_bounds__(256) void linear8JoinKernel(LinearArgs a, Scales s, int splits) {
  const int cols = (a.N + 3) / 4;
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int m = (int)(id / cols), n = (int)(id - (int64_t)m * cols) * 4;
  if(m >= a.M) return;
  const int count = min(4, a.N - n);
  int v[4] = {0, 0, 0, 0};
  const int* p = (const int*)a.part + (int64_t)m * a.N + n;
#pragma unroll 4
  for(int i = 0; i < splits; i++) {
    const uint4 u = loadGroup((const float*)(p + (int64_t)i * a.M * a.N), count);
    v[0] += (int)u.x;
    v[1] += (int)u.y;
    v[2] += (int)u.z;
    v[3] += (int)u.w;
  }
  const float x = s.x[m];
#pragma unroll
  for(int j = 0; j < 4; j++) {
    if(j >= count) break;
    float y = Int8Finish<T, ACT>::activated(scaled(v[j], x, s.w[n + j], a.bias != nullptr ? a.bias[n + j] : 0.0f), 0.0f);
    if(a.residual != nullptr) y = Int8Finish<T, ACT>::added(y, (float)((const T*)a.residual)[(int64_t)m * a.ldr + n + j]);
    ((T*)a.out)[(int64_t)m * a.ldo + n + j] = (T)y;
  }
}

template<typename T, int WM, int WN, int RB, int CB, int PER_CU, int ACT>
void launchDma(const LinearArgs& a, const Scales& s, int splits, hipStream_t stream) {
  constexpr int BM = 32 * RB * WM, BN = 32 * CB * WN;
  const int rowTiles = (a.M + BM - 1) / BM, colTiles = (a.N + BN - 1) / BN;
  linear8DmaKernel<T, WM, WN, RB, CB, PER_CU, ACT><<<dim3((unsigned)(rowTiles * colTiles), (unsigned)splits), 64 * WM * WN, 0, stream>>>(a, s, rowTiles, colTiles);
}

template<typename T, int RB, int CB, int ACT>
void launchTile(const LinearArgs& a, const Scales& s, int splits, hipStream_t stream) {
  const int rowTiles = (a.M + 64 * RB - 1) / (64 * RB), colTiles = (a.N + 64 * CB - 1) / (64 * CB);
  linear8TileKernel<T, RB, CB, ACT><<<dim3((unsigned)(rowTiles * colTiles), (unsigned)splits), 256, 0, stream>>>(a, s, rowTiles, colTiles);
}

template<typename T, int MT, int NT, int WAVES, int UNROLL, int ACT>
void launchSkinny(const LinearArgs& a, const Scales& s, int splits, hipStream_t stream) {
  const dim3 grid((unsigned)((a.N + 16 * NT - 1) / (16 * NT)), (unsigned)splits);
  linear8SkinnyKernel<T, MT, NT, WAVES, UNROLL, ACT><<<grid, 64 * WAVES, 0, stream>>>(a, s);
}

enum Linear8Kernel { LIN8_SKINNY, LIN8_DMA_256, LIN8_DMA_128, LIN8_DMA_64, LIN8_TILE_128, LIN8_TILE_64 };
struct Linear8Plan {
  Linear8Kernel kernel;
  int splits;  // of K
  int chunk;   // k of a split
};

// Which kernel runs, and in how many splits of K with `bytes` of workspace.
Linear8Plan planLinear8(const kgh_linear_int8_params& p, bool aligned, uint64_t bytes) {
  const auto tiles = [&](int64_t side) { return (p.rows + side - 1) / side * ((p.out_channels + side - 1) / side); };
  const int64_t K = p.in_channels, big = tiles(256);
  Linear8Plan plan;
  int64_t most = 1;  // splits worth their sums' way through memory and a second launch
  const uint64_t one = (uint64_t)p.rows * p.out_channels * 4;
  // Each workgroup of the kernel for few rows loads all of x: from 17 rows on that costs
  // more than the weights do, and from some K on more than 64 x 64 tiles in splits with
  // their join, if there is the workspace for them. us without and with: 64x16384x4096
  // 39 and 21, 64x8192x1024 21 and 12, 32x8192x1024 13.7 and 11.2, 64x4096x8192 17.7 and
  // 15.9, 64x8192x30000 112 and 73, but 32x4096x8192 12.1 and 14.2, 17x384x1024 3.5 and 5.1.
  const int64_t parts = std::min<int64_t>(512 / tiles(64), K / 1024);
  const bool tiled = aligned && p.rows > 16 && K >= (p.rows > 32 ? 4096 : 8192) && (parts <= 1 || bytes / one >= (uint64_t)(parts + 1) / 2);
  if(p.rows <= 64 && !tiled) {
    plan.kernel = LIN8_SKINNY;
    if(K >= 12288) most = std::min<int64_t>(256 / ((p.out_channels + 15) / 16), K / 4096);
  }
  // 256 x 256 tiles move half the bytes into LDS, one workgroup a CU; 128 x 128 tiles, two a
  // CU, cover each other's starts and ends, which weigh more the fewer steps there are. us on
  // 256 and 128: 8192x4096x8192 with GELU and residual 327 and 355, 2888x4096x4096 55 and 61,
  // 5776x1024x4096 44 and 39, 46208x1024x384 59 and 44. (0.7: their rounds of 256 CUs full.)
  else if(aligned && K >= 2048 && big * 10 >= (big + 255) / 256 * 256 * 7) plan.kernel = LIN8_DMA_256;
  // us on 128 x 128 and on 64 x 64: 2888x1024x1024 (184 tiles of 128) 11.7 and 9.8,
  // 2888x384x384 8.0 and 5.7, 128x4096x1024 14.5 and 11; 1000x4096x4096 (256) 28 on 128.
  else if(tiles(128) >= 224) plan.kernel = aligned ? LIN8_DMA_128 : LIN8_TILE_128;
  else {
    plan.kernel = aligned ? LIN8_DMA_64 : LIN8_TILE_64;
    if(K >= 4096) most = parts;
  }
  const int64_t splits = std::max<int64_t>(1, std::min<int64_t>(most, (int64_t)std::min<uint64_t>(bytes / one, 1024)));
  plan.chunk = (int)((K + splits * 128 - 1) / (splits * 128) * 128);
  plan.splits = (int)((K + plan.chunk - 1) / plan.chunk);
  return plan;
}

template<typename T, int ACT>
void runLinear8(const Linear8Plan& plan, const LinearArgs& a, const Scales& scales, hipStream_t stream) {
  const int s = plan.splits;
  if(plan.kernel == LIN8_SKINNY) {
    const bool wide = a.N >= 8192;
    if(a.M <= 16) launchSkinny<T, 1, 1, 8, 4, ACT>(a, scales, s, stream);
    else if(a.M <= 32 && wide) launchSkinny<T, 2, 2, 8, 4, ACT>(a, scales, s, stream);
    else if(a.M <= 32) launchSkinny<T, 2, 1, 8, 4, ACT>(a, scales, s, stream);
    else if(wide) launchSkinny<T, 4, 2, 8, 2, ACT>(a, scales, s, stream);
    else launchSkinny<T, 4, 1, 8, 2, ACT>(a, scales, s, stream);
  }
  else if(plan.kernel == LIN8_TILE_128) launchTile<T, 2, 2, ACT>(a, scales, s, stream);
  else if(plan.kernel == LIN8_TILE_64) launchTile<T, 1, 1, ACT>(a, scales, s, stream);
  else if(plan.kernel == LIN8_DMA_256) launchDma<T, 2, 4, 4, 2, 1, ACT>(a, scales, s, stream);
  else if(plan.kernel == LIN8_DMA_128) launchDma<T, 2, 2, 2, 2, 2, ACT>(a, scales, s, stream);
  else launchDma<T, 2, 2, 1, 1, 4, ACT>(a, scales, s, stream);
  KGH_CHECK_LAUNCH();
  if(s > 1) {
    const int64_t threads = (int64_t)a.M * ((a.N + 3) / 4);
    linear8JoinKernel<T, ACT><<<dim3((unsigned)((threads + 255) / 256)), 256, 0, stream>>>(a, scales, s);
    KGH_CHECK_LAUNCH();
  }
}

bool linear8Aligned(const kgh_linear_int8_params& p) {
  return (((uintptr_t)p.x | (uintptr_t)p.weights) & 15) == 0 && p.in_channels % 16 == 0 && p.x_stride % 16 == 0 && p.weights_stride % 16 == 0 &&
         p.x_stride < LIN_DMA_STRIDE && p.weights_stride < LIN_DMA_STRIDE;
}

}  // namespace

namespace kgh {

void checkLinearInt8(const kgh_linear_int8_params& p, bool pointers) {
  const char* op = "kgh_linear_int8";
  opCheckDtype(op, p.dtype);
  opCheckActivation(op, p.activation);
  if(p.rows < 0 || p.rows > LIN8_MAX) opInvalid(op, "rows " + std::to_string(p.rows) + " outside 0.." + std::to_string(LIN8_MAX));
  if(p.in_channels < 1 || p.in_channels > KGH_LINEAR_INT8_MAX_IN)
    opInvalid(op, "in_channels must be in 1.." + std::to_string(KGH_LINEAR_INT8_MAX_IN) + ", so that sums fit 32 bits");
  if(p.out_channels < 1 || p.out_channels > LIN8_MAX_OUT) opInvalid(op, "out_channels must be in 1.." + std::to_string(LIN8_MAX_OUT));
  // 64 x 64 tiles of 256 threads, counted in 32 bits by the launch.
  if((p.rows + 63) / 64 * ((p.out_channels + 63) / 64) >= (1 << 24)) opInvalid(op, "rows times out_channels is too large for one call");
  if(p.x_stride < 0 || p.weights_stride < 0 || p.residual_stride < 0) opInvalid(op, "negative stride");
  if(p.rows > 1 && p.out_stride < p.out_channels) opInvalid(op, "out_stride " + std::to_string(p.out_stride) + " is less than out_channels");
  if(!pointers || p.rows == 0) return;
  const size_t e = opElemBytes(p.dtype);
  opCheckPointer(op, "x", p.x, 1);
  opCheckPointer(op, "x_scales", p.x_scales, 4);
  opCheckPointer(op, "weights", p.weights, 1);
  opCheckPointer(op, "weight_scales", p.weight_scales, 4);
  opCheckPointer(op, "out", p.out, e);
  if(p.residual != nullptr) opCheckPointer(op, "residual", p.residual, e);
  if(p.bias != nullptr) opCheckPointer(op, "bias", p.bias, 4);
  opCheckWorkspace(op, p.workspace, p.workspace_bytes, 0);
  opCheckApart(op, "x", p.x, p.out);
  opCheckApart(op, "x_scales", p.x_scales, p.out);
  opCheckApart(op, "weights", p.weights, p.out);
  opCheckApart(op, "weight_scales", p.weight_scales, p.out);
  if(p.bias != nullptr) opCheckApart(op, "bias", p.bias, p.out);
  if(p.residual == p.out && p.rows > 1 && p.residual_stride != p.out_stride) opInvalid(op, "in place, residual_stride must be out_stride");
}

// By the sizes alone: as if the rows were aligned.
uint64_t linearInt8Workspace(const kgh_linear_int8_params& p) {
  if(p.rows == 0) return 0;
  const Linear8Plan plan = planLinear8(p, true, UINT64_MAX);
  return plan.splits > 1 ? (uint64_t)plan.splits * p.rows * p.out_channels * 4 : 0;
}

void launchLinearInt8(const kgh_linear_int8_params& p, hipStream_t stream) {
  if(p.rows == 0) return;
  const Linear8Plan plan = planLinear8(p, linear8Aligned(p), p.workspace != nullptr ? p.workspace_bytes : 0);
  const LinearArgs a{p.x, p.weights, p.bias, p.residual, p.out, p.x_stride, p.weights_stride, p.residual_stride, p.out_stride,
                     (int)p.rows, p.out_channels, p.in_channels, plan.splits > 1 ? (float*)p.workspace : nullptr, plan.chunk};
  const Scales s{p.x_scales, p.weight_scales};
  withDtype(p.dtype, [&](auto t) {
    withActivation(p.activation, [&](auto act) { runLinear8<decltype(t), decltype(act)::value>(plan, a, s, stream); });
  });
}

}  // namespace kgh
