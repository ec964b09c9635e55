// What the kernels that make 8-bit rows share: a row's scale and its whole numbers.
#ifndef KGH_OP_QUANTIZE_DEVICE_H
#define KGH_OP_QUANTIZE_DEVICE_H

#include "kgh_ops_device.h"

namespace {

// A number's bits without its sign: ordered as magnitudes, infinity above every
// number and NaN above infinity.
__device__ __forceinline__ unsigned magnitudeBits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

constexpr unsigned QUANT_LEAST_BITS = (127u - 120u) << 23;  // of 2^-120: 127 over it is a float
constexpr unsigned QUANT_INFINITE_BITS = 0x7f800000u;

// A row's scale and factor by the largest magnitude in it. Both are divisions
// rounded once, so that a plain fp32 form of the definition has the same bits.
struct RowScale {
  float scale, factor;
  __device__ __forceinline__ explicit RowScale(unsigned top) {
    const float t = __uint_as_float(top);
    const bool none = top < QUANT_LEAST_BITS || top >= QUANT_INFINITE_BITS;
    factor = none ? 0.0f : __fdiv_rn(127.0f, t);
    scale = top >= QUANT_INFINITE_BITS ? __builtin_nanf("") : none ? 0.0f : __fdiv_rn(t, 127.0f);
  }
  // 0 where the factor is: also of infinities and NaN.
  __device__ __forceinline__ int quantized(float v) const { return factor == 0.0f ? 0 : (int)rintf(v * factor); }
};

}  // namespace

#endif
