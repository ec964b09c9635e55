// Matrix product with bias, activation and residual in its epilogue
// (kgh_linear).
#include "kgh_op_linear_device.h"

#include <algorithm>

namespace {

// Rows and channels are counted in 32 bits, with room for a tile past them; a
// launch counts its threads in 32 bits, 512 for 16 output channels.
constexpr int64_t LINEAR_MAX = 1 << 30, LINEAR_MAX_OUT = 1 << 26;

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
  storeTile<T, RB, CB, LinearFinish<T, ACT>>(a, acc, m0 + wm, n0 + wn);
}

// ---------------------------------------------------------------------------
// Rows that are 16-byte aligned (K whole groups of 16 bytes), dmaTile's loop.
// bf16, us: 8192 x 8192 x 8192 847 (1298 TFLOP/s; the library 781), 8192 x 4096 x
// 8192 458, with bias, GELU and residual 505 (1089): of a 256 x 256 tile's 117,
// about 20 are its first loads and its stores, 10 more the residual and GELU. The
// power limit holds the clock at about 2 GHz.
template<typename T, int WM, int WN, int KW, int RB, int CB, int PER_CU, int ACT>
__global__ __launch_bounds__(64 * WM * WN * KW, PER_CU * WM * WN * KW / 4) void linearDmaKernel(LinearArgs a, int rowTiles, int colTiles) {
  floatx16 acc[RB][CB];
  int m, n;
  if(dmaTile<T, WM, WN, KW, RB, CB>(a, rowTiles, colTiles, acc, m, n)) storeTile<T, RB, CB, LinearFinish<T, ACT>>(a, acc, m, n);
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
    v = activate<T, ACT>(v + (a.bias != nullptr ? a.bias[n] : 0.0f));
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
    float y = activate<T, ACT>(v[j] + (a.bias != nullptr ? a.bias[n + j] : 0.0f));
    if(a.residual != nullptr) y += (float)((const T*)a.residual)[(int64_t)m * a.ldr + n + j];
    ((T*)a.out)[(int64_t)m * a.ldo + n + j] = (T)y;
  }
}

template<typename T, int MT, int NT, int WAVES, int UNROLL, int ACT>
void launchSkinny(const LinearArgs& a, int splits, hipStream_t stream) {
  const dim3 grid((unsigned)((a.N + 16 * NT - 1) / (16 * NT)), (unsigned)splits);
  linearSkinnyKernel<T, MT, NT, WAVES, UNROLL, ACT><<<grid, 64 * WAVES, 0, stream>>>(a);
}

}  // namespace

namespace kgh {

void checkLinear(const kgh_linear_params& p, bool pointers) {
  const char* op = "kgh_linear";
  opCheckDtype(op, p.dtype);
  opCheckActivation(op, p.activation);
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
  withDtype(p.dtype, [&](auto t) { withActivation(p.activation, [&](auto act) { runLinear<decltype(t), decltype(act)::value>(plan, a, stream); }); });
}

}  // namespace kgh
