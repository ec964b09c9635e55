// Matrix product with bias, activation and residual in its epilogue
// (kgh_linear).
#include "kgh_conv_device.h"
#include "kgh_ops_device.h"

#include <algorithm>

namespace {

// Rows and channels are counted in 32 bits, with room for a tile past them.
constexpr int64_t LINEAR_MAX = 1 << 30;
constexpr int LIN_ACTS[] = {KGH_ACT_IDENTITY, KGH_ACT_RELU, KGH_ACT_MISH, KGH_ACT_SILU, KGH_ACTIVATION_GELU};

struct LinearArgs {
  const void* x;
  const void* w;
  const float* bias;
  const void* residual;
  void* out;
  int64_t ldx, ldw, ldr, ldo;
  int M, N, K;
};

// Phi(x) to 1e-7 by the rational approximation of erfc in Abramowitz and Stegun,
// 7.1.26: 1 - erf(z) = (a1 t + ... + a5 t^5) e^(-z^2), t = 1 / (1 + p z), z >= 0.
__device__ __forceinline__ float normalCdfFast(float x) {
  const float z = fabsf(x) * 0.70710678118654752f;
  const float t = __builtin_amdgcn_rcpf(fmaf(0.3275911f, z, 1.0f));
  const float poly = t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, 1.061405429f, -1.453152027f), 1.421413741f), -0.284496736f), 0.254829592f);
  const float tail = 0.5f * poly * __expf(-z * z);
  return x < 0.0f ? tail : 1.0f - tail;
}

// The epilogue's activation: accurate forms for fp32 outputs, the fast ones
// (error of about 1e-6) where the result is rounded to 16 bits.
template<typename T, int ACT>
__device__ __forceinline__ float linActivate(float v) {
  if constexpr(ACT == KGH_ACTIVATION_GELU) return sizeof(T) == 4 ? 0.5f * v * erfcf(v * -0.70710678118654752f) : v * normalCdfFast(v);
  else if constexpr(sizeof(T) == 4) return kgh_activate(v, ACT);
  else return kgh_activate_fast(v, ACT);
}

// ---------------------------------------------------------------------------
// Any sizes, strides and alignment: BM x BN tiles of 2 x 2 waves, K in steps of
// a 64-byte row, loaded through registers one step ahead of its use.
template<typename T, int RB, int CB, int ACT>
__global__ __launch_bounds__(256) void linearTileKernel(LinearArgs a, int colTiles) {
  typedef typename Vec16<T>::V V;
  constexpr int VEC = 16 / (int)sizeof(T);
  constexpr int BK = 4 * VEC, BM = 64 * RB, BN = 64 * CB;
  __shared__ __attribute__((aligned(16))) unsigned char lds[2][(BM + BN) * 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int laneRow = lane & 31, half = lane >> 5;
  int rowTile, colTile;
  rowColTile(colTiles, rowTile, colTile);
  const int m0 = rowTile * BM, n0 = colTile * BN;
  const T* x = (const T*)a.x;
  const T* w = (const T*)a.w;

  // Thread t loads 16-byte group t & 3 of rows t >> 2, + 64, ...: RB of x, CB of w.
  const int lr = tid >> 2, lg = tid & 3;
  const T* src[RB + CB];
#pragma unroll
  for(int i = 0; i < RB; i++) src[i] = x + (int64_t)min(m0 + lr + 64 * i, a.M - 1) * a.ldx;
#pragma unroll
  for(int i = 0; i < CB; i++) src[RB + i] = w + (int64_t)min(n0 + lr + 64 * i, a.N - 1) * a.ldw;
  uint4 next[RB + CB];
  auto fetch = [&](int k0) {
    const int k = k0 + lg * VEC;
#pragma unroll
    for(int i = 0; i < RB + CB; i++) next[i] = loadGroup(src[i] + k, a.K - k);
  };
  auto stage = [&](unsigned char* buf) {
#pragma unroll
    for(int i = 0; i < RB + CB; i++) *(uint4*)(buf + (i < RB ? 0 : BM * 64) + swizzled(lr + 64 * (i < RB ? i : i - RB), lg)) = next[i];
  };

  floatx16 acc[RB][CB];
#pragma unroll
  for(int i = 0; i < RB; i++)
#pragma unroll
    for(int j = 0; j < CB; j++)
#pragma unroll
      for(int r = 0; r < 16; r++) acc[i][j][r] = 0.0f;
  const int wm = (wave >> 1) * 32 * RB, wn = (wave & 1) * 32 * CB;
  fetch(0);
  stage(lds[0]);
  __syncthreads();
  int cur = 0;
  for(int k0 = 0; k0 < a.K; k0 += BK) {
    const bool more = k0 + BK < a.K;
    if(more) fetch(k0 + BK);
    const unsigned char* buf = lds[cur];
#pragma unroll
    for(int s = 0; s < 2; s++) {
      V af[RB], bf[CB];
#pragma unroll
      for(int i = 0; i < RB; i++) af[i] = *(const V*)(buf + swizzled(wm + i * 32 + laneRow, 2 * s + half));
#pragma unroll
      for(int j = 0; j < CB; j++) bf[j] = *(const V*)(buf + BM * 64 + swizzled(wn + j * 32 + laneRow, 2 * s + half));
#pragma unroll
      for(int i = 0; i < RB; i++)
#pragma unroll
        for(int j = 0; j < CB; j++) acc[i][j] = mma32(af[i], bf[j], acc[i][j]);
    }
    if(more) stage(lds[cur ^ 1]);
    __syncthreads();
    cur ^= 1;
  }

  const T* res = (const T*)a.residual;
  T* out = (T*)a.out;
#pragma unroll
  for(int j = 0; j < CB; j++) {
    const int n = n0 + wn + j * 32 + laneRow;
    if(n >= a.N) continue;
    const float b = a.bias != nullptr ? a.bias[n] : 0.0f;
#pragma unroll
    for(int i = 0; i < RB; i++)
#pragma unroll
      for(int r = 0; r < 16; r++) {
        const int m = m0 + wm + i * 32 + (r >> 2) * 8 + half * 4 + (r & 3);
        if(m >= a.M) continue;
        float v = linActivate<T, ACT>(acc[i][j][r] + b);
        if(res != nullptr) v += (float)res[(int64_t)m * a.ldr + n];
        out[(int64_t)m * a.ldo + n] = (T)v;
      }
  }
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
  if(p.in_channels < 1 || p.out_channels < 1 || p.in_channels > LINEAR_MAX || p.out_channels > LINEAR_MAX)
    opInvalid(op, "in_channels and out_channels must be in 1.." + std::to_string(LINEAR_MAX));
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
}

uint64_t linearWorkspace(const kgh_linear_params&) { return 0; }

void launchLinear(const kgh_linear_params& p, hipStream_t stream) {
  if(p.rows == 0) return;
  LinearArgs a{p.x, p.weights, p.bias, p.residual, p.out, p.x_stride, p.weights_stride, p.residual_stride, p.out_stride,
               (int)p.rows, p.out_channels, p.in_channels};
  withDtype(p.dtype, [&](auto t) {
    typedef decltype(t) T;
    withLinearAct(p.activation, [&](auto act) {
      const int64_t rows = (p.rows + 63) / 64, cols = (p.out_channels + 63) / 64;
      linearTileKernel<T, 1, 1, decltype(act)::value><<<dim3((unsigned)(rows * cols)), 256, 0, stream>>>(a, (int)cols);
      KGH_CHECK_LAUNCH();
    });
  });
}

}  // namespace kgh
