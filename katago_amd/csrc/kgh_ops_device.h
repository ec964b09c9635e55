// Device code shared by the operators on the caller's tensors.
#ifndef KGH_OPS_DEVICE_H
#define KGH_OPS_DEVICE_H

#include "kgh_conv_device.h"
#include "kgh_ops.h"

namespace {

// 16 bytes as a vector value (HIP's uint4 is a struct, whose copies can end in memory).
typedef unsigned u32x4_t __attribute__((ext_vector_type(4)));

// A 16-byte group of T, as loaded and as the matrix cores take it.
template<typename T> struct Vec16;
template<> struct Vec16<half_t> { typedef half8_t V; };
template<> struct Vec16<bf16_t> { typedef bf16x8_t V; };
template<> struct Vec16<float> { typedef floatx4 V; };
typedef int intx4 __attribute__((ext_vector_type(4)));
typedef int intx16 __attribute__((ext_vector_type(16)));
template<> struct Vec16<int8_t> { typedef intx4 V; };

// Elements [0, n) of the 16-byte group at p, zeros behind them; p need not be
// aligned to more than an element (the memory takes any alignment).
template<typename T>
__device__ __forceinline__ uint4 loadGroup(const T* __restrict__ p, int n) {
  constexpr int VEC = 16 / (int)sizeof(T);
  union {
    uint4 v;
    T e[VEC];
  } u;
  if(n >= VEC) __builtin_memcpy(&u.v, p, 16);
  else {
    u.v = make_uint4(0, 0, 0, 0);
#pragma unroll
    for(int j = 0; j < VEC - 1; j++)
      if(j < n) u.e[j] = p[j];
  }
  return u.v;
}

// A group's elements one place down or up, for the loops over part of a group
// (a few instructions, where the cases written out would be the bulk of a kernel).
template<typename T>
__device__ __forceinline__ uint4 shiftDown(uint4 v) {
  if constexpr(sizeof(T) == 4) return make_uint4(v.y, v.z, v.w, 0);
  else return make_uint4(__builtin_amdgcn_alignbit(v.y, v.x, 16), __builtin_amdgcn_alignbit(v.z, v.y, 16), __builtin_amdgcn_alignbit(v.w, v.z, 16), v.w >> 16);
}

// The first n elements of a 16-byte group to p, which is aligned to an element.
template<typename T>
__device__ __forceinline__ void storeGroup(T* p, uint4 v, int n) {
  constexpr int VEC = 16 / (int)sizeof(T);
  if(n >= VEC) __builtin_memcpy(p, &v, 16);
  else {
#pragma unroll 1
    for(int j = 0; j < n; j++) {
      T e;
      __builtin_memcpy(&e, &v.x, sizeof(T));
      p[j] = e;
      v = shiftDown<T>(v);
    }
  }
}

// loadGroup in few instructions, for the tails of epilogues.
template<typename T>
__device__ __forceinline__ uint4 loadGroupSmall(const T* __restrict__ p, int n) {
  constexpr int VEC = 16 / (int)sizeof(T);
  uint4 v = make_uint4(0, 0, 0, 0);
  if(n >= VEC) __builtin_memcpy(&v, p, 16);
  else {
#pragma unroll 1
    for(int j = 0; j < VEC; j++) {  // element j enters at the top and moves down to its place
      unsigned e = 0;
      if(j < n) __builtin_memcpy(&e, p + j, sizeof(T));
      v = shiftDown<T>(v);
      v.w |= sizeof(T) == 4 ? e : e << 16;
    }
  }
  return v;
}

// Groups of rows of `dims` elements, group `g` a lane, in two steps, so that loads
// stay in flight (a load under a lane's own condition makes the compiler wait
// where its register is cleared first): load() reads 16 bytes that lie in the row
// wherever the group ends, place() puts the group's elements in their places and
// zeros behind the row's end.
// FULL: the rows are as long as the groups of all lanes.
template<typename T, bool FULL>
struct RowGroup {
  static constexpr int VEC = 16 / (int)sizeof(T);
  int at;      // first element read
  int excess;  // elements to drop: VEC where the whole group lies behind the row
  int dims;
  __device__ __forceinline__ RowGroup(int g, int d) {
    dims = d;
    at = max(0, min(g * VEC, d - VEC));
    excess = min(VEC, g * VEC - at);
  }
  __device__ __forceinline__ u32x4_t load(const T* __restrict__ row) const {
    u32x4_t v;
    if(FULL || dims >= VEC) __builtin_memcpy(&v, row + at, 16);
    else {
      const uint4 u = loadGroupSmall(row, dims);
      v = u32x4_t{u.x, u.y, u.z, u.w};
    }
    return v;
  }
  __device__ __forceinline__ u32x4_t place(u32x4_t v) const {
    if constexpr(!FULL) {
      if(dims % VEC != 0 && excess < VEC) {
        uint4 u = make_uint4(v.x, v.y, v.z, v.w);
#pragma unroll 1
        for(int i = 0; i < excess; i++) u = shiftDown<T>(u);
        v = u32x4_t{u.x, u.y, u.z, u.w};
      }
      const u32x4_t zero = {0, 0, 0, 0};
      v = excess >= VEC ? zero : v;
    }
    return v;
  }
};

// x and y with y's lower 32 lanes and x's upper ones exchanged.
__device__ __forceinline__ uint2 swapHalves(unsigned x, unsigned y) {
  const auto r = __builtin_amdgcn_permlane32_swap(x, y, false, false);
  return make_uint2(r[0], r[1]);
}

// A workgroup barrier for LDS alone: __syncthreads() would wait for the loads that
// are to arrive during the next step too.
__device__ __forceinline__ void barrierLds() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  barrierNoFence();
}

// One 16-byte group of k per lane half times the other operand's: 32 x 32
// results, lane l, register r at row (r/4)*8 + (l/32)*4 + r%4, column l % 32.
// In 16 bits a half's group is 8 consecutive k of v_mfma_f32_32x32x16; in fp32
// its four k go to four v_mfma_f32_32x32x2_f32 (exact products, fp32 sums).
__device__ __forceinline__ floatx16 mma32(half8_t a, half8_t b, floatx16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ floatx16 mma32(bf16x8_t a, bf16x8_t b, floatx16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ floatx16 mma32(floatx4 a, floatx4 b, floatx16 c) {
#pragma unroll
  for(int j = 0; j < 4; j++) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
  return c;
}
// The same for 16 x 16 results and four lane groups: lane l, register r at row
// (l/16)*4 + r, column l % 16.
__device__ __forceinline__ floatx4 mma16(half8_t a, half8_t b, floatx4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ floatx4 mma16(bf16x8_t a, bf16x8_t b, floatx4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ floatx4 mma16(floatx4 a, floatx4 b, floatx4 c) {
#pragma unroll
  for(int j = 0; j < 4; j++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
  return c;
}

// The same of 8-bit integers, 16 consecutive k a lane half (quarter): exact sums.
__device__ __forceinline__ intx16 mma32(intx4 a, intx4 b, intx16 c) { return __builtin_amdgcn_mfma_i32_32x32x32_i8(a, b, c, 0, 0, 0); }
__device__ __forceinline__ intx4 mma16(intx4 a, intx4 b, intx4 c) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0); }

// The activations: a result is rounded to its type once, so what a value left of 0
// keeps of itself (e^v or erfc) has to be right relative to itself, down to the type's
// smallest normal numbers.
constexpr float ACT_LOG2E = 1.44269504088896341f;

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
__device__ __forceinline__ float activateFast(float v) {
  if constexpr(ACT == KGH_ACT_SILU) return v * (__builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(fmaf(v, -ACT_LOG2E, -64.0f)) + 0x1p-64f) * 0x1p-64f);
  else if constexpr(ACT == KGH_ACT_MISH) {
    const float big = __builtin_amdgcn_exp2f(fmaf(fminf(v, 20.0f), ACT_LOG2E, 64.0f));
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
    const float q = t * poly * __builtin_amdgcn_exp2f(fmaf(v * v, -0.5f * ACT_LOG2E, 64.0f));
    return v * (v < 0.0f ? q : 1.0f - q);
  }
}

// For results in fp32, to within 2^-18 of the result: the same forms by the accurate functions.
template<int ACT>
__device__ __forceinline__ float activateFp32(float v) {
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
__device__ __forceinline__ float activate(float v) {
  if constexpr(ACT == KGH_ACT_IDENTITY) return v;
  else if constexpr(ACT == KGH_ACT_RELU) return v < 0.0f ? 0.0f : v;  // NaN stays NaN
  else if constexpr(sizeof(T) == 4) return activateFp32<ACT>(v);
  else return activateFast<ACT>(v);
}

template<typename F>
void withActivation(int act, F&& f) {
  switch(act) {
    case KGH_ACTIVATION_RELU: f(std::integral_constant<int, KGH_ACT_RELU>()); break;
    case KGH_ACTIVATION_MISH: f(std::integral_constant<int, KGH_ACT_MISH>()); break;
    case KGH_ACTIVATION_SILU: f(std::integral_constant<int, KGH_ACT_SILU>()); break;
    case KGH_ACTIVATION_GELU: f(std::integral_constant<int, KGH_ACTIVATION_GELU>()); break;
    default: f(std::integral_constant<int, KGH_ACT_IDENTITY>()); break;
  }
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

}  // namespace

#endif
