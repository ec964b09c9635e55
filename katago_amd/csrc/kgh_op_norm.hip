// Group norm with an activation, channels last, and its gradient (kgh_group_norm,
// kgh_group_norm_backward).
#include "kgh_op_quantize_device.h"

#include <algorithm>
#include <cfloat>

namespace {

constexpr int NORM_MAX_LEN = 1 << 30, NORM_MAX_CHANNELS = 1 << 20;

// What both directions read. Strides count elements.
struct NormArgs {
  const void* x;
  const float* weight;
  const float* bias;
  const int32_t* lengths;
  const uint8_t* mask;
  int64_t xB, xP, maskB;
  int batch, positions, channels, groups, per;  // per: channels of a group
  float eps;
};

__device__ __forceinline__ int validLength(const NormArgs& a, int b) {
  return a.lengths == nullptr ? a.positions : min(max(a.lengths[b], 0), a.positions);
}
__device__ __forceinline__ bool takesPart(const NormArgs& a, int b, int p, int len) { return p < len && (a.mask == nullptr || a.mask[b * a.maskB + p] != 0); }

// The sum over a workgroup of 256, for all of its threads.
__device__ __forceinline__ double sumAll(double v, double* lds) {
#pragma unroll
  for(int w = 32; w > 0; w >>= 1) v += __shfl_xor(v, w);
  __syncthreads();
  if((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  return (lds[0] + lds[1]) + (lds[2] + lds[3]);
}

// Mean and 1 / sqrt(variance + eps) of a group of an item.
template<typename T>
__global__ __launch_bounds__(256) void normStatsKernel(NormArgs a, float* stats) {
  __shared__ double lds[4];
  for(int64_t i = blockIdx.x; i < (int64_t)a.batch * a.groups; i += gridDim.x) {
  const int b = (int)(i / a.groups), g = (int)(i - (int64_t)b * a.groups);
  const T* x = (const T*)a.x + b * a.xB + g * a.per;
  const int len = validLength(a, b);
  double sum = 0.0, count = 0.0;
  for(int64_t e = threadIdx.x; e < (int64_t)len * a.per; e += 256) {
    const int p = (int)(e / a.per);
    if(!takesPart(a, b, p, len)) continue;
    sum += (double)(float)x[p * a.xP + (e - (int64_t)p * a.per)];
    count += 1.0;
  }
  count = sumAll(count, lds);
  const double mean = sumAll(sum, lds) / fmax(count, 1.0);
  double squares = 0.0;
  for(int64_t e = threadIdx.x; e < (int64_t)len * a.per; e += 256) {
    const int p = (int)(e / a.per);
    if(!takesPart(a, b, p, len)) continue;
    const double d = (double)(float)x[p * a.xP + (e - (int64_t)p * a.per)] - mean;
    squares += d * d;
  }
  const double var = sumAll(squares, lds) / fmax(count, 1.0);
  if(threadIdx.x == 0) {
    float* s = stats + ((int64_t)b * a.groups + g) * 2;
    s[0] = count == 0.0 ? 0.0f : (float)mean;
    s[1] = count == 0.0 ? 0.0f : (float)(1.0 / sqrt(var + (double)a.eps));
  }
  }
}

// A row (item, position).
template<typename T, int ACT>
__global__ __launch_bounds__(256) void normApplyKernel(NormArgs a, const float* stats, void* out, int64_t oB, int64_t oP, float* scales) {
  __shared__ unsigned tops[4];
  for(int i = blockIdx.x; i < a.batch * a.positions; i += gridDim.x) {
  const int p = i % a.positions, b = i / a.positions;
  const T* x = (const T*)a.x + b * a.xB + p * a.xP;
  const bool on = takesPart(a, b, p, validLength(a, b));
  const int64_t at = b * oB + p * oP;
  auto value = [&](int c) {
    if(!on) return 0.0f;
    const float* s = stats + ((int64_t)b * a.groups + c / a.per) * 2;
    const float h = ((float)x[c] - s[0]) * s[1];
    return activate<T, ACT>(fmaf(h, a.weight != nullptr ? a.weight[c] : 1.0f, a.bias != nullptr ? a.bias[c] : 0.0f));
  };
  if(scales == nullptr) {
    for(int c = threadIdx.x; c < a.channels; c += 256) ((T*)out)[at + c] = (T)value(c);
    continue;
  }
  unsigned top = 0;
  for(int c = threadIdx.x; c < a.channels; c += 256) top = max(top, magnitudeBits(value(c)));
#pragma unroll
  for(int w = 32; w > 0; w >>= 1) top = max(top, (unsigned)__shfl_xor((int)top, w));
  if((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
  __syncthreads();
  const RowScale s(max(max(tops[0], tops[1]), max(tops[2], tops[3])));
  for(int c = threadIdx.x; c < a.channels; c += 256) ((int8_t*)out)[at + c] = (int8_t)s.quantized(value(c));
  if(threadIdx.x == 0) scales[(int64_t)b * a.positions + p] = s.scale;
  __syncthreads();
  }
}

// The activations' derivatives, by the accurate functions.
template<int ACT>
__device__ __forceinline__ float slope(float v) {
  if constexpr(ACT == KGH_ACT_IDENTITY) return 1.0f;
  else if constexpr(ACT == KGH_ACT_RELU) return v > 0.0f ? 1.0f : v != v ? v : 0.0f;
  else if constexpr(ACT == KGH_ACT_SILU) {
    const float s = 1.0f / (1.0f + expf(-v));
    return s * fmaf(v, 1.0f - s, 1.0f);
  }
  else if constexpr(ACT == KGH_ACT_MISH) {
    const float e = expf(fminf(v, 20.0f)), n = e * (e + 2.0f), w = 1.0f / (n + 2.0f);
    return v > 20.0f ? 1.0f : w * fmaf(4.0f * v * e * (1.0f + e), w, n);
  }
  else return fmaf(0.5f, erfcf(-0.70710678118654752f * v), v * expf(-0.5f * v * v) * 0.39894228040143268f);
}

struct NormBackArgs {
  const void* grad;
  int64_t gB, gP;
  const float* stats;
  void* out;
  int64_t oB, oP;
  float* gradWeight;
  float* gradBias;
  float* sums;  // [batch][channels][2]: of u and u h over an item's positions
};

template<typename T, int ACT>
__device__ __forceinline__ void backValues(const NormArgs& a, const NormBackArgs& k, int b, int p, int c, float& u, float& h, float& rstd) {
  const float* s = k.stats + ((int64_t)b * a.groups + c / a.per) * 2;
  rstd = s[1];
  h = ((float)((const T*)a.x)[b * a.xB + p * a.xP + c] - s[0]) * rstd;
  const float z = fmaf(h, a.weight != nullptr ? a.weight[c] : 1.0f, a.bias != nullptr ? a.bias[c] : 0.0f);
  u = (float)((const T*)k.grad)[b * k.gB + p * k.gP + c] * slope<ACT>(z);
}

template<typename T, int ACT>
__global__ __launch_bounds__(256) void normBackSumsKernel(NormArgs a, NormBackArgs k) {
  __shared__ double lds[4];
  for(int64_t i = blockIdx.x; i < (int64_t)a.batch * a.channels; i += gridDim.x) {
  const int b = (int)(i / a.channels), c = (int)(i - (int64_t)b * a.channels);
  const int len = validLength(a, b);
  double s0 = 0.0, s1 = 0.0;
  for(int p = threadIdx.x; p < len; p += 256) {
    if(!takesPart(a, b, p, len)) continue;
    float u, h, rstd;
    backValues<T, ACT>(a, k, b, p, c, u, h, rstd);
    s0 += u;
    s1 += (double)u * h;
  }
  s0 = sumAll(s0, lds);
  s1 = sumAll(s1, lds);
  if(threadIdx.x == 0) {
    k.sums[((int64_t)b * a.channels + c) * 2] = (float)s0;
    k.sums[((int64_t)b * a.channels + c) * 2 + 1] = (float)s1;
  }
  }
}

template<typename T, int ACT>
__global__ __launch_bounds__(256) void normBackApplyKernel(NormArgs a, NormBackArgs k) {
  __shared__ double lds[4];
  for(int64_t i = blockIdx.x; i < (int64_t)a.batch * a.groups; i += gridDim.x) {
  const int b = (int)(i / a.groups), g = (int)(i - (int64_t)b * a.groups);
  const int len = validLength(a, b);
  double count = 0.0, m1 = 0.0, m2 = 0.0;
  for(int p = threadIdx.x; p < len; p += 256) count += takesPart(a, b, p, len) ? 1.0 : 0.0;
  for(int c = threadIdx.x; c < a.per; c += 256) {
    const float* s = k.sums + ((int64_t)b * a.channels + g * a.per + c) * 2;
    const double w = a.weight != nullptr ? a.weight[g * a.per + c] : 1.0;
    m1 += s[0] * w;
    m2 += s[1] * w;
  }
  count = fmax(sumAll(count, lds) * a.per, 1.0);
  const float a1 = (float)(sumAll(m1, lds) / count), a2 = (float)(sumAll(m2, lds) / count);
  for(int64_t e = threadIdx.x; e < (int64_t)a.positions * a.per; e += 256) {
    const int p = (int)(e / a.per), c = g * a.per + (int)(e - (int64_t)p * a.per);
    float y = 0.0f;
    if(takesPart(a, b, p, len)) {
      float u, h, rstd;
      backValues<T, ACT>(a, k, b, p, c, u, h, rstd);
      y = rstd * (u * (a.weight != nullptr ? a.weight[c] : 1.0f) - a1 - h * a2);
    }
    ((T*)k.out)[b * k.oB + p * k.oP + c] = (T)y;
  }
  }
}

__global__ __launch_bounds__(256) void normBackJoinKernel(NormArgs a, NormBackArgs k) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if(c >= a.channels) return;
  double s0 = 0.0, s1 = 0.0;
  for(int b = 0; b < a.batch; b++) {
    s0 += k.sums[((int64_t)b * a.channels + c) * 2];
    s1 += k.sums[((int64_t)b * a.channels + c) * 2 + 1];
  }
  if(k.gradBias != nullptr) k.gradBias[c] = (float)s0;
  if(k.gradWeight != nullptr) k.gradWeight[c] = (float)s1;
}

// Rows (item, position) of a tensor that is written lie apart.
void checkApartRows(const char* op, const char* name, int64_t batchStride, int64_t positionStride, int batch, int positions, int channels) {
  const bool positionsInside = (positions == 1 || positionStride >= channels) && (batch == 1 || batchStride >= (positions - 1) * positionStride + channels);
  const bool itemsInside = (batch == 1 || batchStride >= channels) && (positions == 1 || positionStride >= (batch - 1) * batchStride + channels);
  if(!positionsInside && !itemsInside) kgh::opInvalid(op, std::string("the strides of ") + name + " make its rows overlap");
}

template<typename P>
void checkNormSizes(const char* op, const P& p) {
  kgh::opCheckDtype(op, p.dtype);
  kgh::opCheckActivation(op, p.activation);
  if(p.batch < 0 || p.positions < 0 || (int64_t)p.batch * p.positions > NORM_MAX_LEN)
    kgh::opInvalid(op, "batch and positions must be 0 or more, their product at most " + std::to_string(NORM_MAX_LEN));
  if(p.channels < 1 || p.channels > NORM_MAX_CHANNELS) kgh::opInvalid(op, "channels must be in 1.." + std::to_string(NORM_MAX_CHANNELS));
  if(p.groups < 1 || p.channels % p.groups != 0) kgh::opInvalid(op, "groups must divide channels");
}

template<typename P>
NormArgs normArgs(const P& p, float eps) {
  return NormArgs{p.x, p.weight, p.bias, p.lengths, p.mask, p.x_batch_stride, p.x_position_stride, p.mask_stride,
                  p.batch, p.positions, p.channels, p.groups, p.channels / p.groups, eps};
}

}  // namespace

namespace kgh {

void checkGroupNorm(const kgh_group_norm_params& p, bool pointers) {
  const char* op = "kgh_group_norm";
  checkNormSizes(op, p);
  if(!pointers) return;
  if(!(p.eps >= FLT_MIN) || p.eps > FLT_MAX) opInvalid(op, "eps must be a number of at least 2^-126");
  for(int64_t s : {p.x_batch_stride, p.x_position_stride, p.mask_stride, p.out_batch_stride, p.out_position_stride})
    if(s < 0) opInvalid(op, "negative stride");
  if(p.batch == 0 || p.positions == 0) return;
  checkApartRows(op, "out", p.out_batch_stride, p.out_position_stride, p.batch, p.positions, p.channels);
  const size_t e = opElemBytes(p.dtype);
  opCheckPointer(op, "x", p.x, e);
  opCheckPointer(op, "out", p.out, p.out_scales != nullptr ? 1 : e);
  if(p.weight != nullptr) opCheckPointer(op, "weight", p.weight, 4);
  if(p.bias != nullptr) opCheckPointer(op, "bias", p.bias, 4);
  if(p.lengths != nullptr) opCheckPointer(op, "lengths", p.lengths, 4);
  if(p.out_scales != nullptr) opCheckPointer(op, "out_scales", p.out_scales, 4);
  if(p.statistics != nullptr) opCheckPointer(op, "statistics", p.statistics, 4);
  if(p.x == p.out) {
    if(p.out_scales != nullptr) opInvalid(op, "out is x itself, in another type");
    if((p.batch > 1 && p.x_batch_stride != p.out_batch_stride) || (p.positions > 1 && p.x_position_stride != p.out_position_stride))
      opInvalid(op, "in place, the strides must be the same");
  }
  opCheckWorkspace(op, p.workspace, p.workspace_bytes, groupNormWorkspace(p));
}

uint64_t groupNormWorkspace(const kgh_group_norm_params& p) { return (uint64_t)p.batch * p.groups * 8; }

void launchGroupNorm(const kgh_group_norm_params& p, hipStream_t stream) {
  if(p.batch == 0 || p.positions == 0) return;
  const NormArgs a = normArgs(p, p.eps);
  float* stats = p.statistics != nullptr ? p.statistics : (float*)p.workspace;
  withDtype(p.dtype, [&](auto t) {
    typedef decltype(t) T;
    normStatsKernel<T><<<dim3((unsigned)std::min<int64_t>((int64_t)p.groups * p.batch, 1 << 20)), 256, 0, stream>>>(a, stats);
    KGH_CHECK_LAUNCH();
    withActivation(p.activation, [&](auto act) {
      normApplyKernel<T, decltype(act)::value><<<dim3((unsigned)std::min<int64_t>(p.batch * p.positions, 1 << 20)), 256, 0, stream>>>(a, stats, p.out, p.out_batch_stride,
                                                                                                             p.out_position_stride, p.out_scales);
    });
    KGH_CHECK_LAUNCH();
  });
}

void checkGroupNormBackward(const kgh_group_norm_backward_params& p, bool pointers) {
  const char* op = "kgh_group_norm_backward";
  checkNormSizes(op, p);
  if(!pointers) return;
  for(int64_t s : {p.x_batch_stride, p.x_position_stride, p.mask_stride, p.grad_out_batch_stride, p.grad_out_position_stride, p.grad_x_batch_stride,
                   p.grad_x_position_stride})
    if(s < 0) opInvalid(op, "negative stride");
  if(p.grad_weight != nullptr) opCheckPointer(op, "grad_weight", p.grad_weight, 4);
  if(p.grad_bias != nullptr) opCheckPointer(op, "grad_bias", p.grad_bias, 4);
  if(p.grad_weight != nullptr && p.grad_weight == p.grad_bias) opInvalid(op, "grad_weight is grad_bias itself");
  if(p.batch == 0 || p.positions == 0) return;
  checkApartRows(op, "grad_x", p.grad_x_batch_stride, p.grad_x_position_stride, p.batch, p.positions, p.channels);
  const size_t e = opElemBytes(p.dtype);
  opCheckPointer(op, "x", p.x, e);
  opCheckPointer(op, "grad_out", p.grad_out, e);
  opCheckPointer(op, "grad_x", p.grad_x, e);
  opCheckPointer(op, "statistics", p.statistics, 4);
  if(p.weight != nullptr) opCheckPointer(op, "weight", p.weight, 4);
  if(p.bias != nullptr) opCheckPointer(op, "bias", p.bias, 4);
  if(p.lengths != nullptr) opCheckPointer(op, "lengths", p.lengths, 4);
  if(p.x == p.grad_x) opInvalid(op, "grad_x is x itself");
  if(p.grad_out == p.grad_x) opInvalid(op, "grad_x is grad_out itself");
  opCheckWorkspace(op, p.workspace, p.workspace_bytes, groupNormBackwardWorkspace(p));
}

uint64_t groupNormBackwardWorkspace(const kgh_group_norm_backward_params& p) { return (uint64_t)p.batch * p.channels * 8; }

void launchGroupNormBackward(const kgh_group_norm_backward_params& p, hipStream_t stream) {
  NormArgs a = normArgs(p, 0.0f);
  if(p.positions == 0) a.batch = 0;
  const NormBackArgs k{p.grad_out, p.grad_out_batch_stride, p.grad_out_position_stride, p.statistics, p.grad_x, p.grad_x_batch_stride,
                       p.grad_x_position_stride, p.grad_weight, p.grad_bias, (float*)p.workspace};
  if(p.batch > 0 && p.positions > 0)
    withDtype(p.dtype, [&](auto t) {
      typedef decltype(t) T;
      withActivation(p.activation, [&](auto act) {
        normBackSumsKernel<T, decltype(act)::value><<<dim3((unsigned)std::min<int64_t>((int64_t)p.channels * p.batch, 1 << 20)), 256, 0, stream>>>(a, k);
        KGH_CHECK_LAUNCH();
        normBackApplyKernel<T, decltype(act)::value><<<dim3((unsigned)std::min<int64_t>((int64_t)p.groups * p.batch, 1 << 20)), 256, 0, stream>>>(a, k);
        KGH_CHECK_LAUNCH();
      });
    });
  if(p.grad_weight == nullptr && p.grad_bias == nullptr) return;
  normBackJoinKernel<<<dim3((unsigned)((p.channels + 255) / 256)), 256, 0, stream>>>(a, k);
  KGH_CHECK_LAUNCH();
}

}  // namespace kgh
