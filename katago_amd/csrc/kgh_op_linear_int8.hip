// Matrix product of 8-bit integers with scales for rows and channels
// (kgh_linear_int8).
#include "kgh_conv_device.h"
#include "kgh_ops_device.h"

#include <algorithm>

namespace {

// Rows and channels are counted in 32 bits, with room for a tile past them; a
// launch counts its threads in 32 bits.
constexpr int64_t LIN8_MAX = 1 << 30, LIN8_MAX_OUT = 1 << 26;

typedef int intx4 __attribute__((ext_vector_type(4)));
typedef int intx16 __attribute__((ext_vector_type(16)));

struct Linear8Args {
  const int8_t* x;
  const int8_t* w;
  const float* xScales;
  const float* wScales;
  const float* bias;
  const void* residual;
  void* out;
  int64_t ldx, ldw, ldr, ldo;
  int M, N, K;
};

// 16 bytes of k per lane half times the other operand's: 32 x 32 results, laid out
// as mma32's.
__device__ __forceinline__ intx16 mma32(intx4 a, intx4 b, intx16 c) { return __builtin_amdgcn_mfma_i32_32x32x32_i8(a, b, c, 0, 0, 0); }

// Elements [0, n) of the 16 bytes at p, zeros behind them.
__device__ __forceinline__ u32x4_t loadBytes(const int8_t* p, int n) {
  u32x4_t v = {0, 0, 0, 0};
  if(n >= 16) __builtin_memcpy(&v, p, 16);
  else
    for(int j = 0; j < n; j++) v[j >> 2] |= (unsigned)(uint8_t)p[j] << (8 * (j & 3));
  return v;
}

template<typename T, int ACT>
__device__ __forceinline__ T finish(const Linear8Args& a, int sum, int m, int n) {
  float v = (float)sum * a.xScales[m] * a.wScales[n];
  v = activate<T, ACT>(v + (a.bias != nullptr ? a.bias[n] : 0.0f));
  if(a.residual != nullptr) v += (float)((const T*)a.residual)[(int64_t)m * a.ldr + n];
  return (T)v;
}

// Any sizes, strides and alignment: 64 x 64 tiles of four waves, steps of 128 bytes
// of K through LDS.
template<typename T, int ACT>
__global__ __launch_bounds__(256) void linear8TileKernel(Linear8Args a, int rowTiles, int colTiles) {
  __shared__ __attribute__((aligned(16))) unsigned char lds[128 * 128];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int laneRow = lane & 31, half = lane >> 5;
  int rowTile, colTile;
  blockedTile(rowTiles, colTiles, rowTile, colTile);
  const int m0 = rowTile * 64, n0 = colTile * 64;
  const int lr = tid >> 3, lg = tid & 7;
  const int wm = (wave >> 1) * 32, wn = (wave & 1) * 32;
  intx16 acc;
#pragma unroll
  for(int r = 0; r < 16; r++) acc[r] = 0;
  for(int k = 0; k < a.K; k += 128) {
    __syncthreads();
#pragma unroll
    for(int i = 0; i < 4; i++) {
      const int row = lr + 32 * i;
      const int8_t* src = row < 64 ? a.x + (int64_t)min(m0 + row, a.M - 1) * a.ldx : a.w + (int64_t)min(n0 + row - 64, a.N - 1) * a.ldw;
      *(u32x4_t*)(lds + swizzled128(row, lg)) = loadBytes(src + k + lg * 16, a.K - k - lg * 16);
    }
    __syncthreads();
#pragma unroll
    for(int s = 0; s < 4; s++)
      acc = mma32(*(const intx4*)(lds + swizzled128(64 + wn + laneRow, 2 * s + half)), *(const intx4*)(lds + swizzled128(wm + laneRow, 2 * s + half)), acc);
  }
  const int m = m0 + wm + laneRow;
  if(m >= a.M) return;
#pragma unroll
  for(int r = 0; r < 16; r++) {
    const int n = n0 + wn + (r >> 2) * 8 + half * 4 + (r & 3);
    if(n < a.N) ((T*)a.out)[(int64_t)m * a.ldo + n] = finish<T, ACT>(a, acc[r], m, n);
  }
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

uint64_t linearInt8Workspace(const kgh_linear_int8_params&) { return 0; }

void launchLinearInt8(const kgh_linear_int8_params& p, hipStream_t stream) {
  if(p.rows == 0) return;
  const Linear8Args a{p.x, p.weights, p.x_scales, p.weight_scales, p.bias, p.residual, p.out, p.x_stride, p.weights_stride, p.residual_stride,
                      p.out_stride, (int)p.rows, p.out_channels, p.in_channels};
  const int rowTiles = (a.M + 63) / 64, colTiles = (a.N + 63) / 64;
  withDtype(p.dtype, [&](auto t) {
    withActivation(p.activation, [&](auto act) {
      linear8TileKernel<decltype(t), decltype(act)::value><<<dim3((unsigned)(rowTiles * colTiles)), 256, 0, stream>>>(a, rowTiles, colTiles);
    });
  });
  KGH_CHECK_LAUNCH();
}

}  // namespace kgh
