// What the kernels that make 8-bit rows share: a row's scale and its whole numbers.
#ifndef KGH_OP_QUANTIZE_DEVICE_H
#define KGH_OP_QUANTIZE_DEVICE_H

#include "kgh_ops_device.h"

namespace {

// Elements of a 16-byte group as floats.
template<typename T>
struct Values {
  static constexpr int VEC = 16 / (int)sizeof(T);
  float f[VEC];
  __device__ __forceinline__ explicit Values(u32x4_t v) {
    if constexpr(__is_same(T, bf16_t)) {
#pragma unroll
      for(int i = 0; i < 4; i++) {
        f[2 * i] = __uint_as_float(v[i] << 16);
        f[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
      }
    }
    else {
      T e[VEC];
      __builtin_memcpy(e, &v, 16);
#pragma unroll
      for(int j = 0; j < VEC; j++) f[j] = (float)e[j];
    }
  }
};

// A number's bits without its sign: ordered as magnitudes, infinity above every
// number and NaN above infinity.
__device__ __forceinline__ unsigned magnitudeBits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

constexpr unsigned QUANT_LEAST_BITS = (127u - 120u) << 23;  // of 2^-120: 127 over it is a float
constexpr unsigned QUANT_INFINITE_BITS = 0x7f800000u;

// A row's scale and factor by the largest magnitude in it. Both are divisions
// rounded once, so that a plain fp32 form of the definition has the same bits.
struct RowScale {
  float scale, factor;
  unsigned keep;  // of the whole numbers' bytes: none where the row's are zeros
  __device__ __forceinline__ explicit RowScale(unsigned top) {
    const float t = __uint_as_float(top);
    const bool none = top < QUANT_LEAST_BITS || top >= QUANT_INFINITE_BITS;
    factor = none ? 0.0f : __fdiv_rn(127.0f, t);
    keep = none ? 0u : ~0u;
    scale = top >= QUANT_INFINITE_BITS ? __builtin_nanf("") : none ? 0.0f : __fdiv_rn(t, 127.0f);
  }
  // The whole number nearest to v's product with the factor, in the lowest byte: of that
  // number and 1.5 * 2^23, whose steps are 1. Of a NaN that byte is any (arithmetic hands
  // on a NaN's own lower bits): what is stored goes through `keep`.
  __device__ __forceinline__ unsigned quantized(float v) const {
    float p = v * factor;
    asm("" : "+v"(p));  // rounded by itself
    return __float_as_uint(p + 12582912.0f);
  }
};

// The largest of a row that `lanes` threads side by side have (a power of two up to 64,
// or a workgroup of 256, whose waves meet in lds).
__device__ __forceinline__ unsigned rowTop(unsigned top, int lanes, unsigned* lds) {
  if(lanes >= 16) {  // within sixteen threads by rotations
    top = max(top, (unsigned)__builtin_amdgcn_update_dpp(0, (int)top, 0x128, 0xf, 0xf, true));
    top = max(top, (unsigned)__builtin_amdgcn_update_dpp(0, (int)top, 0x124, 0xf, 0xf, true));
    top = max(top, (unsigned)__builtin_amdgcn_update_dpp(0, (int)top, 0x122, 0xf, 0xf, true));
    top = max(top, (unsigned)__builtin_amdgcn_update_dpp(0, (int)top, 0x121, 0xf, 0xf, true));
    if(lanes >= 32) top = max(top, (unsigned)__shfl_xor((int)top, 16));
    if(lanes >= 64) top = max(top, (unsigned)__shfl_xor((int)top, 32));
  }
  else
    for(int w = lanes >> 1; w > 0; w >>= 1) top = max(top, (unsigned)__shfl_xor((int)top, w));
  if(lanes <= 64) return top;
  if((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = top;
  __syncthreads();
  return max(max(lds[0], lds[1]), max(lds[2], lds[3]));
}

// How threads share a row of `groups` 16-byte groups, at most `most` each: by the fewest
// a thread that a wave manages with, in the power of two that leaves the fewest threads
// idle; by a workgroup of 256 above; lanes is 0 where the row is longer.
struct RowLanes {
  int lanes, each;
};
inline RowLanes rowLanes(int groups, int most) {
  for(int each = 1; each <= most; each *= 2)
    for(int lanes : {8, 16, 32, 64})
      if(lanes * each >= groups) return RowLanes{lanes, each};
  for(int each = 1; each <= most; each *= 2)
    if(256 * each >= groups) return RowLanes{256, each};
  return RowLanes{0, 0};
}

// Bytes [from, to) of VEC (4 or 8), to p + from and on.
template<int VEC>
__device__ __forceinline__ void storeBytes(int8_t* p, uint2 v, int from, int to) {
  if(from == 0 && to >= VEC) __builtin_memcpy(p, &v, VEC);
  else {
#pragma unroll 1
    for(int j = 0; j < VEC; j++) {
      if(j >= from && j < to) p[j] = (int8_t)(v.x & 0xff);
      v.x = __builtin_amdgcn_alignbit(v.y, v.x, 8);
      v.y >>= 8;
    }
  }
}

// VEC values in 8 bits.
template<int VEC>
__device__ __forceinline__ uint2 quantized(const float (&y)[VEC], const RowScale& s) {
  unsigned w[2] = {0, 0};
#pragma unroll
  for(int j = 0; j < VEC; j += 4) {
    const unsigned low = __builtin_amdgcn_perm(s.quantized(y[j + 1]), s.quantized(y[j]), 0x0c0c0400);
    const unsigned high = __builtin_amdgcn_perm(s.quantized(y[j + 3]), s.quantized(y[j + 2]), 0x04000c0c);
    w[j >> 2] = low | high;
  }
  return make_uint2(w[0] & s.keep, w[1] & s.keep);
}

}  // namespace

#endif
