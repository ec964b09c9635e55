// Attention to an encoder's states (kgh_cross_attention).
#include "kgh_conv_device.h"
#include "kgh_ops_device.h"

#include <algorithm>
#include <cmath>
#include <utility>

namespace {

constexpr int ATT_MAX_LEN = 1 << 30;  // positions are counted in 32 bits, with room for a tile past them

struct AttnArgs {
  const void* q;
  const void* k;
  const void* v;
  void* out;
  int64_t qB, qT, qH, kB, kT, kH, vB, vT, vH, oB, oT, oH;
  const int32_t* lengths;
  const uint8_t* mask;
  int64_t maskB;
  int lq, lk, heads, kvHeads, dq, dv;
  float scaleLog2;  // scale * log2(e): differences of scores, times this, are exponents to base 2
};

// Where a split's sums go: [split][row][v dim] in fp32, then [split][row] pairs of
// reference point and sum. Rows are counted over batch, kv head and (query, head
// of the group).
struct AttnSplit {
  int splits;
  float* out;   // null without a split
  float* state;
};

__device__ __forceinline__ int validLength(const AttnArgs& a, int b) {
  return a.lengths == nullptr ? a.lk : min(max(a.lengths[b], 0), a.lk);
}

// ---------------------------------------------------------------------------
// LDS layouts of key rows of D elements. K rows are read 16 bytes a lane, 16
// consecutive rows a phase, the same group: the groups are permuted so that they
// fall in distinct banks. V rows in 16 bits are read transposed, 8 bytes a lane,
// four consecutive rows of 64 bytes a phase: 64-byte granules are permuted. V
// rows in fp32 are read a float a lane, from rows 4 apart in the two lane halves.
template<typename T, int D>
__device__ __forceinline__ int kAt(int key, int group) {  // bytes
  constexpr int GROUPS = D * (int)sizeof(T) / 16;
  const int term = GROUPS >= 16 ? key : GROUPS == 8 ? key >> 1 : key >> 2;
  return (key * GROUPS + (group ^ (term & (GROUPS - 1) & 15))) * 16;
}
template<typename T, int D>
__device__ __forceinline__ int vAt(int key, int group) {
  constexpr int GROUPS = D * (int)sizeof(T) / 16;
  int term;
  if constexpr(sizeof(T) == 4) term = D >= 64 ? ((key >> 2) & 1) * 8 : 0;
  else term = GROUPS >= 16 ? (key & 3) * 4 : GROUPS == 8 ? ((key >> 1) & 1) * 4 : 0;
  return (key * GROUPS + (group ^ term)) * 16;
}

// Where a lane reads its V^T operands: of keys base .. base + VEC / 4 * 8 - 1 (base
// a multiple of 8, in the accumulator's row order: a lane half has keys half * 4 +
// {0..3}, + 8, ...) and dims 32 db + laneRow. One offset for each db; what is added
// for base is a constant.
template<typename T, int D>
struct ValueReads {
  int at[D / 32];
  __device__ __forceinline__ ValueReads() {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for(int db = 0; db < D / 32; db++) {
      if constexpr(sizeof(T) == 4) {
        const int d = db * 32 + (lane & 31);
        at[db] = vAt<T, D>((lane >> 5) * 4, d >> 2) + (d & 3) * 4;
      }
      else {
        // Sixteen lanes read four rows of 16 dims and get a column each.
        const int d = db * 32 + (lane & 16) + (lane & 3) * 4;
        at[db] = vAt<T, D>((lane >> 5) * 4 + ((lane & 15) >> 2), d >> 3) + (d & 7) * 2;
      }
    }
  }
  __device__ __forceinline__ typename Vec16<T>::V read(const unsigned char* vs, int base, int db) const {
    constexpr int ROW = D * (int)sizeof(T);
    typename Vec16<T>::V v;
    if constexpr(sizeof(T) == 4) {
#pragma unroll
      for(int j = 0; j < 4; j++) v[j] = *(const float*)(vs + at[db] + (base + j) * ROW);
    }
    else {
      typedef short short4v __attribute__((ext_vector_type(4)));
      typedef __attribute__((address_space(3))) short4v* Ptr;
      union {
        short4v h[2];
        typename Vec16<T>::V v;
      } u;
#pragma unroll
      for(int h = 0; h < 2; h++) u.h[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Ptr)(vs + at[db] + (base + h * 8) * ROW));
      v = u.v;
    }
    return v;
  }
};

// One row's running softmax: p = 2^((s - ref) c + shift), with a reference point
// that only moves when a tile's maximum passes it by more than 8 / c (the
// normalisation by the fp32 sum of the same p makes the choice cancel).
// The reference is a score, taken off before the product: s c - ref c would have
// the rounding of ref c, half a step of a number that may be any size, for the
// largest key's exponent in place of 0.
// The shift makes p at most 1 where its type has fp32's exponents, so that sums of
// p v are no larger than sums of v; fp16's p is at most 2^15, its largest as large
// as the type allows, so that many keys of little weight each are not lost below
// its smallest numbers, and its values are far from fp32's end.
template<typename T>
constexpr float P_SHIFT = sizeof(T) == 2 && !__is_same(T, bf16_t) ? 7.0f : -8.0f;
struct RowState {
  float ref = -INFINITY, sum = 0.0f;
};

// Scores of keys that take no part become minus infinity. valid: bit per key.
template<int BLOCKS>
__device__ __forceinline__ void maskTile(floatx16 (&s)[BLOCKS], unsigned long long valid) {
  const int half = (threadIdx.x & 63) >> 5;
  if(valid != (BLOCKS == 2 ? ~0ull : 0xffffffffull)) {
#pragma unroll
    for(int kb = 0; kb < BLOCKS; kb++) {
      const unsigned bits = (unsigned)(valid >> (kb * 32)) >> (half * 4);
#pragma unroll
      for(int i = 0; i < 16; i++)
        if(!((bits >> ((i >> 2) * 8 + (i & 3))) & 1)) s[kb][i] = -INFINITY;
    }
  }
}

// The scores of BLOCKS * 32 keys become p; returns what the accumulators before
// them are to be multiplied by.
template<typename T, int BLOCKS>
__device__ __forceinline__ float softmaxTile(floatx16 (&s)[BLOCKS], float scaleLog2, RowState& row) {
  float top = -INFINITY;
#pragma unroll
  for(int kb = 0; kb < BLOCKS; kb++)
#pragma unroll
    for(int i = 0; i < 16; i += 2) top = fmaxf(fmaxf(top, s[kb][i]), s[kb][i + 1]);
  const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
  top = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
  // (of two infinities alike this is NaN, and the reference stays)
  const float ref = (top - row.ref) * scaleLog2 > 8.0f ? top : row.ref;
  const float corr = ref == row.ref ? 1.0f : __builtin_amdgcn_exp2f((row.ref - ref) * scaleLog2);
  row.ref = ref;
  // While a row has met no score above -inf its base is 0: every p is 0.
  const float base = ref == -INFINITY ? 0.0f : ref;
  float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for(int kb = 0; kb < BLOCKS; kb++)
#pragma unroll
    for(int i = 0; i < 16; i++) {
      s[kb][i] = __builtin_amdgcn_exp2f(fmaf(s[kb][i] - base, scaleLog2, P_SHIFT<T>));
      part[i & 3] += s[kb][i];
    }
  row.sum = row.sum * corr + ((part[0] + part[1]) + (part[2] + part[3]));  // of this lane half's keys; joined at the end
  return corr;
}

// The largest magnitude of a lane's values in 16 bits, as far as to tell whether
// one is infinite or NaN: bits without the sign, two numbers a register.
typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));
template<typename T>
constexpr unsigned short INFINITE_BITS = __is_same(T, bf16_t) ? 0x7f80 : 0x7c00;
template<typename T>
struct Magnitude {
  u16x2_t most = {0, 0};
  __device__ __forceinline__ void take(u32x4_t v) {
    if constexpr(sizeof(T) == 2) {
#pragma unroll
      for(int i = 0; i < 4; i++) most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2_t, v[i] & 0x7fff7fffu));
    }
  }
  __device__ __forceinline__ bool infinite() const { return max(most[0], most[1]) >= INFINITE_BITS<T>; }
};
// Zeros in the place of a group's infinities and NaN.
template<typename T>
__device__ __forceinline__ typename Vec16<T>::V finiteOnly(typename Vec16<T>::V v) {
  u16x2_t u[4];
  __builtin_memcpy(u, &v, 16);
#pragma unroll
  for(int i = 0; i < 4; i++)
#pragma unroll
    for(int j = 0; j < 2; j++) u[i][j] = (u[i][j] & 0x7fff) >= INFINITE_BITS<T> ? 0 : u[i][j];
  __builtin_memcpy(&v, u, 16);
  return v;
}

// The two lane halves' sums.
__device__ __forceinline__ float joinHalves(float v) { return v + __shfl_xor(v, 32); }

// ---------------------------------------------------------------------------
// At most 32 rows a kv head: (query, head of the group) pairs, so that grouped
// heads share the keys that are read. Bound by the keys' and values' bytes: each
// of four waves goes through 32-key tiles of its own, the next tile's loads under
// way while it computes, and nothing but the end makes waves wait for each other;
// the keys are split over workgroups too where there are few. S^T = K Q^T (lane =
// row, 16 of 32 keys), so that P^T is the second product's operand as it stands.
// Here the matrix cores have time: P goes through them in two pieces, so that the
// result is not off by P's rounding (an infinite value meets one of them only: times
// the second one, of any sign or 0, it would be NaN). bf16, 32 streams, 32/8 heads of 128, up to 4096
// keys each: 69 us, 4.9 TB/s of keys and values (a copy reaches 5.2); one stream of
// 16384 keys 20 us, where a wave's four tiles take a round trip to memory each.
template<typename T, int D, bool FULL>
__global__ __launch_bounds__(256, sizeof(T) == 2 ? 2 : 1) void attentionFewKernel(AttnArgs a, AttnSplit split) {
  typedef typename Vec16<T>::V V;
  constexpr int VEC = 16 / (int)sizeof(T), GROUPS = D / VEC, LOADS = 32 * GROUPS / 64;
  constexpr int ROWS_BYTES = 32 * D * (int)sizeof(T);
  constexpr int OLD = 33;  // floats between dims of a wave's sums [dim][row]
  constexpr int WAVE_BYTES = 2 * ROWS_BYTES > D * OLD * 4 ? 2 * ROWS_BYTES : D * OLD * 4;
  __shared__ __attribute__((aligned(16))) unsigned char lds[4][WAVE_BYTES];
  __shared__ float refs[4][32], totals[4][32];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int laneRow = lane & 31, half = lane >> 5;
  const int kvh = blockIdx.y, b = blockIdx.z;
  const int group = a.heads / a.kvHeads;
  const int rows = a.lq * group;
  const int rc = min(laneRow, rows - 1);
  const T* qRow = (const T*)a.q + b * a.qB + (int64_t)(rc / group) * a.qT + (int64_t)(kvh * group + rc % group) * a.qH;
  const T* kBase = (const T*)a.k + b * a.kB + kvh * a.kH;
  const T* vBase = (const T*)a.v + b * a.vB + kvh * a.vH;
  const int len = validLength(a, b);
  const int tiles = (len + 31) / 32;
  const int first = (int)((int64_t)tiles * blockIdx.x / split.splits) + wave;
  const int end = (int)((int64_t)tiles * (blockIdx.x + 1) / split.splits);

  V qf[D / VEC / 2];
#pragma unroll
  for(int i = 0; i < D / VEC / 2; i++) {
    const RowGroup<T, FULL> g(2 * i + half, a.dq);
    const u32x4_t u = g.place(g.load(qRow));
    qf[i] = *(const V*)&u;
  }
  floatx16 o[D / 32];
#pragma unroll
  for(int db = 0; db < D / 32; db++)
#pragma unroll
    for(int i = 0; i < 16; i++) o[db][i] = 0.0f;
  RowState row;

  // A tile's rows in registers: lane's group lane % GROUPS of keys lane / GROUPS + ...
  const int lg = lane % GROUPS, lk = lane / GROUPS;
  const RowGroup<T, FULL> kGroup(lg, a.dq), vGroup(lg, a.dv);
  struct Rows {
    u32x4_t k[LOADS], v[LOADS];
    unsigned long long mask;
  };
  auto load = [&](int tile, Rows& r) {
    const int k0 = min(tile, end - 1) * 32;
    const int key = k0 + laneRow;
    r.mask = a.mask != nullptr && key < len ? a.mask[b * a.maskB + key] : 1;
#pragma unroll
    for(int i = 0; i < LOADS; i++) {
      const int64_t at = min(k0 + lk + i * (64 / GROUPS), len - 1);
      r.k[i] = kGroup.load(kBase + at * a.kT);
      r.v[i] = vGroup.load(vBase + at * a.vT);
    }
  };
  const ValueReads<T, D> reads;
  unsigned char* ks = lds[wave];
  unsigned char* vs = lds[wave] + ROWS_BYTES;
  Rows r;
  if(first < end) load(first, r);
  for(int t = first; t < end; t += 4) {
    const unsigned valid = (unsigned)__ballot(r.mask != 0 && t * 32 + laneRow < len);
    asm volatile("" ::: "memory");  // a wave's LDS accesses run in order
    Magnitude<T> largest;
#pragma unroll
    for(int i = 0; i < LOADS; i++) {
      const int key = lk + i * (64 / GROUPS);
      const u32x4_t zero = {0, 0, 0, 0};
      *(u32x4_t*)(ks + kAt<T, D>(key, lg)) = kGroup.place(r.k[i]);
      const u32x4_t v = (valid >> key) & 1 ? vGroup.place(r.v[i]) : zero;
      largest.take(v);
      *(u32x4_t*)(vs + vAt<T, D>(key, lg)) = v;
    }
    const bool infinite = __any(largest.infinite());
    asm volatile("" ::: "memory");
    load(t + 4, r);
    floatx16 s[1];
#pragma unroll
    for(int i = 0; i < 16; i++) s[0][i] = 0.0f;
#pragma unroll
    for(int i = 0; i < D / VEC / 2; i++) s[0] = mma32(*(const V*)(ks + kAt<T, D>(laneRow, 2 * i + half)), qf[i], s[0]);
    maskTile<1>(s, valid);
    const float corr = softmaxTile<T, 1>(s, a.scaleLog2, row);
    if(__any(corr != 1.0f)) {
#pragma unroll
      for(int db = 0; db < D / 32; db++)
#pragma unroll
        for(int i = 0; i < 16; i++) o[db][i] *= corr;
    }
#pragma unroll
    for(int g = 0; g < 16 / VEC; g++) {
      V hi, lo;
#pragma unroll
      for(int i = 0; i < VEC; i++) {
        hi[i] = (T)s[0][g * VEC + i];
        lo[i] = (T)(s[0][g * VEC + i] - (float)hi[i]);
      }
#pragma unroll
      for(int db = 0; db < D / 32; db++) {
        const V vf = reads.read(vs, g * VEC / 4 * 8, db);
        o[db] = mma32(vf, hi, o[db]);
        if constexpr(sizeof(T) == 2) o[db] = mma32(infinite ? finiteOnly<T>(vf) : vf, lo, o[db]);
      }
    }
  }

  // The waves' sums, on one reference point.
  row.sum = joinHalves(row.sum);
  if(half == 0) {
    refs[wave][laneRow] = row.ref;
    totals[wave][laneRow] = row.sum;
  }
  __syncthreads();
  float ref = -INFINITY;
#pragma unroll
  for(int w = 0; w < 4; w++) ref = fmaxf(ref, refs[w][laneRow]);
  const float mine = row.ref == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((row.ref - ref) * a.scaleLog2);
  float* sums = (float*)lds[wave];
#pragma unroll
  for(int db = 0; db < D / 32; db++)
#pragma unroll
    for(int i = 0; i < 16; i++) sums[(db * 32 + (i >> 2) * 8 + half * 4 + (i & 3)) * OLD + laneRow] = o[db][i] * mine;
  __syncthreads();
  for(int e = tid; e < rows * a.dv; e += 256) {
    const int m = e / a.dv, d = e - m * a.dv;
    float top = -INFINITY, total = 0.0f, v = 0.0f;
#pragma unroll
    for(int w = 0; w < 4; w++) top = fmaxf(top, refs[w][m]);
#pragma unroll
    for(int w = 0; w < 4; w++) {
      total += refs[w][m] == -INFINITY ? totals[w][m] : totals[w][m] * __builtin_amdgcn_exp2f((refs[w][m] - top) * a.scaleLog2);
      v += ((const float*)lds[w])[d * OLD + m];
    }
    if(split.out != nullptr) {
      const int64_t at = ((int64_t)blockIdx.x * gridDim.z + b) * a.kvHeads * rows + (int64_t)kvh * rows + m;
      split.out[at * a.dv + d] = v;
      if(d == 0) {
        split.state[at * 2] = top;
        split.state[at * 2 + 1] = total;
      }
    }
    else {
      T* out = (T*)a.out + b * a.oB + (int64_t)(m / group) * a.oT + (int64_t)(kvh * group + m % group) * a.oH;
      out[d] = (T)(total == 0.0f ? 0.0f : v / total);
    }
  }
}

// ---------------------------------------------------------------------------
// Many rows: a workgroup of WAVES waves has 32 rows a wave of one kv head, and
// goes through tiles of 64 keys (or 32) that all of them read from LDS. Of tile t + 1 the
// scores are computed before tile t's softmax, so that the matrix cores have them
// to do while the vector units work; a tile's rows are loaded into registers two
// barriers before they are read. Bound by what a wave does between barriers: the
// softmax's vector work (16 cycles for an exponential, about 32 a score in all)
// and the products take as long as both one after the other, two waves a SIMD.
// bf16, 4096 queries to 5000 keys, 32/8 heads: of 128 762 us (881 TFLOP/s), of 64
// 480 (699); 64 boards of 361 queries to boards of three sizes, fp16, heads of 64,
// 37 us, where two thirds are a workgroup's start and end.
// In 16 bits p is rounded to the tensors' type for its product with v (its sum is
// not): the result is off by a third more than its own rounding (bf16, 5000 keys:
// 0.0022 of its norm, 0.0017 with p exact). PRECISE, the caller's choice, has p in two
// pieces: 0.0017, and 1012 us for 762, 655 for 480, 43 for 37.
constexpr int64_t ATT_NEAR = 1 << 23;  // token strides below it: 64 of them are less than 2^31 bytes
constexpr int ATT_LIST = 256;  // key tiles whose masks are looked at at a time

// 32-key blocks of a tile: one where two would not leave registers for the reads
// ahead (16 bits, 4096 queries to 5000 keys, heads of 128: 822 us, two 1064); and
// in fp32, heads up to 64, where one lets a CU hold two workgroups (`pairs`).
template<typename T, int D>
constexpr int attBlocks(bool pairs) { return pairs || (sizeof(T) == 2 && D == 128) ? 1 : 2; }
__device__ __forceinline__ constexpr unsigned long long attWhole(int blocks) { return blocks == 2 ? ~0ull : 0xffffffffull; }

template<typename T, int D, int WAVES, bool FULL, bool PAIRS = sizeof(T) == 2, bool PRECISE = false>
__global__ __launch_bounds__(64 * WAVES, PAIRS ? 2 : 1) void attentionManyKernel(AttnArgs a, AttnSplit split) {
  typedef typename Vec16<T>::V V;
  constexpr int THREADS = 64 * WAVES;
  constexpr int VEC = 16 / (int)sizeof(T), GROUPS = D / VEC, BLOCKS = attBlocks<T, D>(sizeof(T) == 4 && PAIRS), KEYS = 32 * BLOCKS, LOADS = KEYS * GROUPS / THREADS;
  static_assert(LOADS * THREADS == KEYS * GROUPS && THREADS % GROUPS == 0, "whole loads");
  constexpr int TILE = KEYS * D * (int)sizeof(T);
  __shared__ __attribute__((aligned(16))) unsigned char k0s[TILE];
  __shared__ __attribute__((aligned(16))) unsigned char k1s[TILE];
  __shared__ __attribute__((aligned(16))) unsigned char v0s[TILE];
  __shared__ __attribute__((aligned(16))) unsigned char v1s[TILE];
  // Tiles with a key that takes part, and which keys (bits), in order.
  __shared__ unsigned long long listBits[ATT_LIST + 1];
  __shared__ int listTile[ATT_LIST];
  __shared__ int listCount;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int laneRow = lane & 31, half = lane >> 5;
  const int kvh = blockIdx.y, b = blockIdx.z;
  const int group = a.heads / a.kvHeads;
  const int rows = a.lq * group;
  const int rowBlock = blockIdx.x / split.splits, part = blockIdx.x - rowBlock * split.splits;
  const int r = (rowBlock * WAVES + wave) * 32 + laneRow;
  const int rc = min(r, rows - 1);
  const int qi = rc / group, h = kvh * group + (rc - qi * group);
  const T* qRow = (const T*)a.q + b * a.qB + qi * a.qT + h * a.qH;
  const T* kBase = (const T*)a.k + b * a.kB + kvh * a.kH;
  const T* vBase = (const T*)a.v + b * a.vB + kvh * a.vH;
  const int len = validLength(a, b);
  const int allTiles = (len + KEYS - 1) / KEYS;
  const int begin = (int)((int64_t)allTiles * part / split.splits), end = (int)((int64_t)allTiles * (part + 1) / split.splits);

  V qf[D / VEC / 2];
#pragma unroll
  for(int i = 0; i < D / VEC / 2; i++) {
    const RowGroup<T, FULL> g(2 * i + half, a.dq);
    const u32x4_t u = g.place(g.load(qRow));
    qf[i] = *(const V*)&u;
  }
  floatx16 o[D / 32];
#pragma unroll
  for(int db = 0; db < D / 32; db++)
#pragma unroll
    for(int i = 0; i < 16; i++) o[db][i] = 0.0f;
  RowState row;

  const int lg = tid % GROUPS, lk = tid / GROUPS;
  const RowGroup<T, FULL> kGroup(lg, a.dq), vGroup(lg, a.dv);
  struct Rows {
    u32x4_t v[LOADS];
  };
  int count = 0, from = begin;  // tiles of this round, and its first
  // What item i of the round is: a tile, and which of its keys take part.
  auto tileOf = [&](int i) { return a.mask == nullptr ? from + i : __builtin_amdgcn_readfirstlane(listTile[i]); };
  auto bitsOf = [&](int i) -> unsigned long long {
    if(a.mask != nullptr) {
      const unsigned long long v = listBits[i];
      return ((unsigned long long)(unsigned)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32) | (unsigned)__builtin_amdgcn_readfirstlane((int)v);
    }
    const int n = len - (from + i) * KEYS;
    return n >= KEYS ? attWhole(BLOCKS) : (1ull << max(n, 0)) - 1;
  };
  // A lane's offset in a tile, where it fits 32 bits (ATT_NEAR): a whole tile's
  // addresses are then a scalar and this.
  const unsigned kNear = (unsigned)(lk * a.kT + kGroup.at) * (unsigned)sizeof(T), vNear = (unsigned)(lk * a.vT + vGroup.at) * (unsigned)sizeof(T);
  auto load = [&](const T* base, int64_t stride, unsigned near, const RowGroup<T, FULL>& g, int i, Rows& x) {
    const int k0 = tileOf(min(i, count - 1)) * KEYS;
    if(FULL && k0 + KEYS <= len && stride < ATT_NEAR) {
#pragma unroll
      for(int j = 0; j < LOADS; j++) __builtin_memcpy(&x.v[j], (const char*)(base + (int64_t)(k0 + j * (THREADS / GROUPS)) * stride) + near, 16);
    }
    else {
#pragma unroll
      for(int j = 0; j < LOADS; j++) {
        const int64_t at = min(k0 + lk + j * (THREADS / GROUPS), len - 1);
        x.v[j] = g.load(base + at * stride);
      }
    }
  };
  auto loadK = [&](int i, Rows& x) { load(kBase, a.kT, kNear, kGroup, i, x); };
  auto loadV = [&](int i, Rows& x) { load(vBase, a.vT, vNear, vGroup, i, x); };
  auto stageK = [&](unsigned char* ks, const Rows& x) {
#pragma unroll
    for(int j = 0; j < LOADS; j++) *(u32x4_t*)(ks + kAt<T, D>(lk + j * (THREADS / GROUPS), lg)) = kGroup.place(x.v[j]);
  };
  // What V holds at keys that take no part must not meet their p of 0.
  auto stageV = [&](unsigned char* vs, const Rows& x, unsigned long long bits) {
#pragma unroll
    for(int j = 0; j < LOADS; j++) {
      const int key = lk + j * (THREADS / GROUPS);
      const u32x4_t zero = {0, 0, 0, 0};
      *(u32x4_t*)(vs + vAt<T, D>(key, lg)) = (bits >> key) & 1 ? vGroup.place(x.v[j]) : zero;
    }
  };
  auto scores = [&](const unsigned char* ks, floatx16 (&s)[BLOCKS]) {
#pragma unroll
    for(int kb = 0; kb < BLOCKS; kb++)
#pragma unroll
      for(int i = 0; i < 16; i++) s[kb][i] = 0.0f;
#pragma unroll
    for(int i = 0; i < D / VEC / 2; i++)
#pragma unroll
      for(int kb = 0; kb < BLOCKS; kb++) s[kb] = mma32(*(const V*)(ks + kAt<T, D>(kb * 32 + laneRow, 2 * i + half)), qf[i], s[kb]);
  };
  const ValueReads<T, D> reads;
  constexpr int GROUPS_P = KEYS / 2 / VEC;  // 16-byte groups of a lane's p
  struct Values {
    V v[D / 32];
  };
  auto readValues = [&](const unsigned char* vs, int g, Values& x) {
#pragma unroll
    for(int db = 0; db < D / 32; db++) x.v[db] = reads.read(vs, g * VEC / 4 * 8, db);
  };
  // x: the operands of the first group. The next group's are read behind a group's
  // first product, whose wait for its own operands then waits for nothing else.
  // PRECISE: p's second piece pl follows (finite values only, see attentionFewKernel).
  auto values = [&](const unsigned char* vs, const V (&p)[GROUPS_P], const V (&pl)[GROUPS_P], Values& x) {
    Values y;
#pragma unroll
    for(int g = 0; g < GROUPS_P; g++) {
      const Values& now = g % 2 == 0 ? x : y;
      o[0] = mma32(now.v[0], p[g], o[0]);
      __builtin_amdgcn_sched_barrier(0);
      if(g + 1 < GROUPS_P) readValues(vs, g + 1, g % 2 == 0 ? y : x);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for(int db = 1; db < D / 32; db++) o[db] = mma32(now.v[db], p[g], o[db]);
      if constexpr(PRECISE) {
        Magnitude<T> largest;
#pragma unroll
        for(int db = 0; db < D / 32; db++) largest.take(__builtin_bit_cast(u32x4_t, now.v[db]));
        const bool infinite = __any(largest.infinite());
#pragma unroll
        for(int db = 0; db < D / 32; db++) o[db] = mma32(infinite ? finiteOnly<T>(now.v[db]) : now.v[db], pl[g], o[db]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  Rows kr, vr;
  // Item i: its scores are in s; K of i + 1 and V of i are in LDS, K of i + 2 and V
  // of i + 1 in registers.
  auto step = [&](int i, floatx16 (&s)[BLOCKS], floatx16 (&sNext)[BLOCKS], unsigned char* kNow, const unsigned char* kNext, const unsigned char* vNow,
                  unsigned char* vNext) {
    const unsigned long long bits = bitsOf(i), bitsNext = bitsOf(min(i + 1, count - 1));
    maskTile<BLOCKS>(s, bits);
    __builtin_amdgcn_sched_barrier(0);
    scores(kNext, sNext);
    const float corr = softmaxTile<T, BLOCKS>(s, a.scaleLog2, row);
    V p[GROUPS_P], pl[GROUPS_P];
#pragma unroll
    for(int g = 0; g < GROUPS_P; g++) {
#pragma unroll
      for(int j = 0; j < VEC; j++) p[g][j] = (T)s[g * VEC / 16][g * VEC % 16 + j];
      // Here, not where it is used: beside the scores' products.
      asm volatile("" : "+v"(p[g]));
      if constexpr(PRECISE) {
#pragma unroll
        for(int j = 0; j < VEC; j++) pl[g][j] = (T)(s[g * VEC / 16][g * VEC % 16 + j] - (float)p[g][j]);
        asm volatile("" : "+v"(pl[g]));
      }
    }
    if constexpr(sizeof(T) == 2) {
      // A product, then vector work in its shadow.
      __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
      for(int j = 0; j < D / 16 * BLOCKS; j++) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x402, D == 128 ? 12 : 22, 0);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    Values x;
    readValues(vNow, 0, x);
    __builtin_amdgcn_sched_barrier(0);
    if(__any(corr != 1.0f)) {
#pragma unroll
      for(int db = 0; db < D / 32; db++)
#pragma unroll
        for(int j = 0; j < 16; j++) o[db][j] *= corr;
    }
    values(vNow, p, pl, x);
    stageK(kNow, kr);
    stageV(vNext, vr, bitsNext);
    loadK(i + 3, kr);
    loadV(i + 2, vr);
    barrierLds();
  };

  for(; from < end; from += ATT_LIST) {
    count = min(ATT_LIST, end - from);
    if(a.mask != nullptr) {
      __syncthreads();
      for(int t = wave; t < count; t += WAVES) {
        const int j = (from + t) * KEYS + lane % KEYS;
        const unsigned long long bits = __ballot(j < len && a.mask[b * a.maskB + j] != 0) & attWhole(BLOCKS);
        if(lane == 0) listBits[t] = bits;
      }
      __syncthreads();
      if(wave == 0) {
        int n = 0;
        for(int t0 = 0; t0 < count; t0 += 64) {
          const unsigned long long bits = t0 + lane < count ? listBits[t0 + lane] : 0;
          const unsigned long long on = __ballot(bits != 0);
          const int at = n + __popcll(on & ((1ull << lane) - 1));
          // Entries move down only, and the 64 of a round are read before any is written.
          if(bits != 0) {
            listBits[at] = bits;
            listTile[at] = from + t0 + lane;
          }
          n += __popcll(on);
        }
        if(lane == 0) listCount = n;
      }
      __syncthreads();
      count = listCount;
      if(count == 0) continue;
    }
    {
      Rows kFirst;
      loadK(0, kFirst);
      loadK(1, kr);
      loadV(0, vr);
      if(from > begin) __syncthreads();  // the buffers' readers of the round before
      stageK(k0s, kFirst);
      stageK(k1s, kr);
      stageV(v0s, vr, bitsOf(0));
    }
    loadK(2, kr);
    loadV(1, vr);
    barrierLds();
    floatx16 sA[BLOCKS], sB[BLOCKS];
    scores(k0s, sA);
    // A wave that is ahead puts item 2's keys where others still read item 0's.
    barrierLds();
    int i = 0;
    for(; i + 2 <= count; i += 2) {
      step(i, sA, sB, k0s, k1s, v0s, v1s);
      step(i + 1, sB, sA, k1s, k0s, v1s, v0s);
    }
    if(i < count) step(i, sA, sB, k0s, k1s, v0s, v1s);
  }

  row.sum = joinHalves(row.sum);
  const bool on = r < rows;
  if(split.out != nullptr) {
    if(!on) return;
    const int64_t at = ((int64_t)part * gridDim.z + b) * a.kvHeads * rows + (int64_t)kvh * rows + r;
    if(half == 0) {
      split.state[at * 2] = row.ref;
      split.state[at * 2 + 1] = row.sum;
    }
#pragma unroll
    for(int db = 0; db < D / 32; db++)
#pragma unroll
      for(int q = 0; q < 4; q++) {
        const int d = db * 32 + q * 8 + half * 4;
        const floatx4 v = {o[db][q * 4], o[db][q * 4 + 1], o[db][q * 4 + 2], o[db][q * 4 + 3]};
        if(d < a.dv) storeGroup(split.out + at * a.dv + d, *(const uint4*)&v, a.dv - d);
      }
    return;
  }
  const float inv = row.sum == 0.0f ? 0.0f : 1.0f / row.sum;
  // Without a key the sums may be NaN, of a p of 0 and an infinite value.
  if(row.sum == 0.0f) {
#pragma unroll
    for(int db = 0; db < D / 32; db++)
#pragma unroll
      for(int i = 0; i < 16; i++) o[db][i] = 0.0f;
  }
  T* oRow = (T*)a.out + b * a.oB + qi * a.oT + h * a.oH;
#pragma unroll
  for(int db = 0; db < D / 32; db++) {
    if constexpr(sizeof(T) == 4) {
#pragma unroll
      for(int q = 0; q < 4; q++) {
        const int d = db * 32 + q * 8 + half * 4;
        const floatx4 v = {o[db][q * 4] * inv, o[db][q * 4 + 1] * inv, o[db][q * 4 + 2] * inv, o[db][q * 4 + 3] * inv};
        if(on && d < a.dv) storeGroup((float*)oRow + d, *(const uint4*)&v, a.dv - d);
      }
    }
    else {
      // A lane has four of eight consecutive dims, its partner lane ^ 32 the others;
      // two such groups of both swap halves into 16 bytes a lane.
#pragma unroll
      for(int p = 0; p < 2; p++) {
        union Four {
          uint2 v;
          T e[4];
        } f[2];
#pragma unroll
        for(int q = 0; q < 2; q++)
#pragma unroll
          for(int i = 0; i < 4; i++) f[q].e[i] = (T)(o[db][(2 * p + q) * 4 + i] * inv);
        const uint2 x = swapHalves(f[0].v.x, f[1].v.x), y = swapHalves(f[0].v.y, f[1].v.y);
        const int d = db * 32 + (2 * p + half) * 8;
        if(on && d < a.dv) storeGroup(oRow + d, make_uint4(x.x, y.x, x.y, y.y), a.dv - d);
      }
    }
  }
}

// The splits' sums on one reference point: a workgroup takes a row, a thread four
// dims of every eighth split (their loads are what takes time, one round trip
// instead of one for each split), added in order in LDS.
template<typename T>
__global__ __launch_bounds__(256) void attentionJoinKernel(AttnArgs a, AttnSplit split, int64_t rowsAll) {
  __shared__ float sums[8][128];
  __shared__ float totals[8];
  const int64_t r = blockIdx.x;
  const int quad = threadIdx.x & 31, slice = threadIdx.x >> 5;
  const int d = quad * 4, n = min(4, a.dv - d);
  float ref = -INFINITY;
  for(int s = quad; s < split.splits; s += 32) ref = fmaxf(ref, split.state[(s * rowsAll + r) * 2]);
#pragma unroll
  for(int w = 16; w > 0; w >>= 1) ref = fmaxf(ref, __shfl_xor(ref, w));
  float total = 0.0f, v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
  for(int s = slice; s < split.splits; s += 8) {
    const float* st = split.state + (s * rowsAll + r) * 2;
    const uint4 u = n > 0 ? loadGroup(split.out + (s * rowsAll + r) * a.dv + d, n) : make_uint4(0, 0, 0, 0);
    const float f = st[0] == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((st[0] - ref) * a.scaleLog2);
    total = fmaf(st[1], f, total);
    v[0] = fmaf(__uint_as_float(u.x), f, v[0]);
    v[1] = fmaf(__uint_as_float(u.y), f, v[1]);
    v[2] = fmaf(__uint_as_float(u.z), f, v[2]);
    v[3] = fmaf(__uint_as_float(u.w), f, v[3]);
  }
  *(float4*)&sums[slice][d] = make_float4(v[0], v[1], v[2], v[3]);
  if(quad == 0) totals[slice] = total;
  __syncthreads();
  const int e = threadIdx.x;
  if(e >= a.dv) return;
  float all = 0.0f, y = 0.0f;
#pragma unroll
  for(int i = 0; i < 8; i++) {
    all += totals[i];
    y += sums[i][e];
  }
  // r counts batch, kv head, query, head of the group.
  const int group = a.heads / a.kvHeads;
  const int64_t rows = (int64_t)a.lq * group, outer = r / rows;
  const int at = (int)(r - outer * rows);
  const int64_t b = outer / a.kvHeads;
  const int h = (int)(outer - b * a.kvHeads) * group + at % group;
  ((T*)a.out)[b * a.oB + (int64_t)(at / group) * a.oT + h * a.oH + e] = (T)(all == 0.0f ? 0.0f : y / all);
}

}  // namespace

namespace kgh {

void checkAttention(const kgh_attention_params& p, bool pointers) {
  const char* op = "kgh_cross_attention";
  opCheckDtype(op, p.dtype);
  if(p.batch < 0 || p.q_len < 0 || p.k_len < 0 || p.q_len > ATT_MAX_LEN || p.k_len > ATT_MAX_LEN)
    opInvalid(op, "batch and lengths must be 0 or more (lengths at most " + std::to_string(ATT_MAX_LEN) + ")");
  if(p.kv_heads < 1 || p.heads < 1 || p.heads % p.kv_heads != 0) opInvalid(op, "kv_heads must divide heads");
  for(int d : {p.q_head_dim, p.v_head_dim})
    if(d < 1 || d > KGH_ATTENTION_MAX_HEAD_DIM) opInvalid(op, "head dim " + std::to_string(d) + " outside 1.." + std::to_string(KGH_ATTENTION_MAX_HEAD_DIM));
  if(p.precise != 0 && p.precise != 1) opInvalid(op, "precise must be 0 or 1");
  if(!(p.scale > 0.0f) || p.scale > KGH_ATTENTION_MAX_SCALE) opInvalid(op, "scale must be positive and at most 1e30");
  for(int64_t s : {p.q_batch_stride, p.q_token_stride, p.q_head_stride, p.k_batch_stride, p.k_token_stride, p.k_head_stride, p.v_batch_stride,
                   p.v_token_stride, p.v_head_stride, p.out_batch_stride, p.out_token_stride, p.out_head_stride, p.key_mask_stride})
    if(s < 0) opInvalid(op, "negative stride");
  const int64_t group = p.heads / p.kv_heads;
  if((int64_t)p.q_len * group > ATT_MAX_LEN) opInvalid(op, "too many queries for one call");
  if(p.batch > 65535 || p.kv_heads > 65535) opInvalid(op, "batch and kv_heads must be at most 65535");
  if(!pointers || p.batch == 0 || p.q_len == 0) return;
  // The output's rows lie apart: sorted by stride, each axis steps over the ones inside it.
  std::pair<int64_t, int64_t> axes[3] = {{p.out_batch_stride, p.batch}, {p.out_token_stride, p.q_len}, {p.out_head_stride, p.heads}};
  std::sort(axes, axes + 3);
  int64_t inside = p.v_head_dim;
  for(const auto& [stride, size] : axes) {
    if(size == 1) continue;
    if(stride < inside) opInvalid(op, "the output's strides make its rows overlap");
    inside += stride * (size - 1);
  }
  const size_t e = opElemBytes(p.dtype);
  opCheckPointer(op, "q", p.q, e);
  opCheckPointer(op, "out", p.out, e);
  if(p.k_len > 0) {
    opCheckPointer(op, "k", p.k, e);
    opCheckPointer(op, "v", p.v, e);
  }
  if(p.key_lengths != nullptr) opCheckPointer(op, "key_lengths", p.key_lengths, 4);
  if(p.workspace != nullptr) opCheckPointer(op, "workspace", p.workspace, 16);
  opCheckApart(op, "q", p.q, p.out);
  opCheckApart(op, "k", p.k, p.out);
  opCheckApart(op, "v", p.v, p.out);
}

namespace {

struct AttentionPlan {
  bool few;   // at most 32 rows a kv head
  int waves;  // of the kernel for more
  bool pairs; // fp32: of its variant with two workgroups a CU
  bool precise;  // 16 bits: of its variant with p in two pieces
  int splits; // of the keys
  int64_t rows;
};

// Which kernel runs, and in how many splits of the keys with `bytes` of workspace.
AttentionPlan planAttention(const kgh_attention_params& p, uint64_t bytes) {
  AttentionPlan plan;
  const int64_t rows = (int64_t)p.q_len * (p.heads / p.kv_heads);
  plan.rows = rows * p.batch * p.kv_heads;
  plan.few = rows <= 32;
  // 256-row workgroups where they are at most an eighth empty: 512 rows, heads of
  // 128, 85 us (90 with 128 rows), 16384 rows 795 (962); 361 rows 112 (94).
  const bool wide = rows >= 512 && rows * 8 >= (rows + 255) / 256 * 256 * 7;
  // (p in two pieces leaves heads above 64 no registers with four waves)
  const int dim = std::max(p.q_head_dim, p.v_head_dim);
  plan.precise = p.precise != 0 && p.dtype != KGH_DTYPE_FP32 && !plan.few;
  plan.waves = p.dtype != KGH_DTYPE_FP32 && ((wide && dim > 32) || (plan.precise && dim > 64)) ? 8 : 4;
  const int64_t groups = plan.few ? (int64_t)p.batch * p.kv_heads : (rows + plan.waves * 32 - 1) / (plan.waves * 32) * p.batch * p.kv_heads;
  // Where there are more workgroups than CUs: 16 boards of 361 queries and keys, 6
  // heads of 64, 63 us (73 with one a CU and 64 keys a tile), of 32 36.6 (37.3).
  plan.pairs = p.dtype == KGH_DTYPE_FP32 && groups > 256 && dim <= 64;
  // Workgroups that the CUs hold at a time: two a CU of the kernel for few rows in
  // 16 bits, one of the others; and at least 128 keys a split. One query of 8 kv
  // heads to 16384 keys, us: whole 306, 8 splits 47, 32 21.6, 64 22.1; of 32
  // streams and 8 kv heads: whole 92, two 76, four 80; 361 queries of 6 heads to
  // 4096 keys: whole 98, 16 21.6, 32 28.
  const int64_t wanted = plan.few && p.dtype != KGH_DTYPE_FP32 ? 512 : 256;
  int64_t splits = std::min<int64_t>({wanted / groups, p.k_len / 128, 64});
  // Many rows in fp32, whose products take longer: 6 heads of 64, 361 queries and keys,
  // whole 35, in two 24; 84 workgroups, heads of 74, 484 keys 113 and 62 in three.
  const bool slow = p.dtype == KGH_DTYPE_FP32 && !plan.few;
  if(p.k_len < (slow ? 256 : 512)) splits = 1;  // 6 heads of 16 bits, 361 keys: whole 7.9, in two 9.3
  // Many rows' sums are many bytes: 96 workgroups, 361 keys, whole 20, in two 29;
  // fp32 300 keys 29 and 32, but 500 keys 45 and 38.
  if(!plan.few && groups > (slow && p.k_len >= 384 ? 128 : 64)) splits = 1;
  const uint64_t one = (uint64_t)plan.rows * (p.v_head_dim + 2) * 4;
  splits = std::min<int64_t>(splits, (int64_t)std::min<uint64_t>(bytes / one, 64));
  plan.splits = (int)std::max<int64_t>(1, splits);
  return plan;
}

template<typename T, int D, bool FULL>
void runAttention(const AttentionPlan& plan, const AttnArgs& a, const AttnSplit& split, int batch, hipStream_t stream) {
  const int64_t rows = (int64_t)a.lq * (a.heads / a.kvHeads), block = plan.waves * 32;
  const dim3 grid((unsigned)((plan.few ? 1 : (rows + block - 1) / block) * plan.splits), (unsigned)a.kvHeads, (unsigned)batch);
  if(plan.few) attentionFewKernel<T, D, FULL><<<grid, 256, 0, stream>>>(a, split);
  else if(sizeof(T) == 4 && D <= 64 && plan.pairs) attentionManyKernel<T, D, 4, FULL, sizeof(T) == 2 || D <= 64><<<grid, 256, 0, stream>>>(a, split);
  else if(plan.precise) {
    if constexpr(sizeof(T) == 2) {
      if(plan.waves == 4) {
        if constexpr(D <= 64) attentionManyKernel<T, D, 4, FULL, true, true><<<grid, 256, 0, stream>>>(a, split);
      }
      else if constexpr(D >= 64) attentionManyKernel<T, D, 8, FULL, true, true><<<grid, 512, 0, stream>>>(a, split);
    }
  }
  else if(plan.waves == 4) attentionManyKernel<T, D, 4, FULL><<<grid, 256, 0, stream>>>(a, split);
  else if constexpr(sizeof(T) == 2 && D >= 64) attentionManyKernel<T, D, 8, FULL><<<grid, 512, 0, stream>>>(a, split);
  KGH_CHECK_LAUNCH();
  if(plan.splits > 1) {
    attentionJoinKernel<T><<<dim3((unsigned)plan.rows), 256, 0, stream>>>(a, split, plan.rows);
    KGH_CHECK_LAUNCH();
  }
}

}  // namespace

uint64_t attentionWorkspace(const kgh_attention_params& p) {
  if(p.batch == 0 || p.q_len == 0) return 0;
  const AttentionPlan plan = planAttention(p, UINT64_MAX);
  return plan.splits > 1 ? (uint64_t)plan.splits * plan.rows * (p.v_head_dim + 2) * 4 : 0;
}

void launchAttention(const kgh_attention_params& p, hipStream_t stream) {
  if(p.batch == 0 || p.q_len == 0) return;
  AttnArgs a{};
  a.q = p.q;
  a.k = p.k;
  a.v = p.v;
  a.out = p.out;
  a.qB = p.q_batch_stride, a.qT = p.q_token_stride, a.qH = p.q_head_stride;
  a.kB = p.k_batch_stride, a.kT = p.k_token_stride, a.kH = p.k_head_stride;
  a.vB = p.v_batch_stride, a.vT = p.v_token_stride, a.vH = p.v_head_stride;
  a.oB = p.out_batch_stride, a.oT = p.out_token_stride, a.oH = p.out_head_stride;
  a.lengths = p.key_lengths;
  a.mask = p.key_mask;
  a.maskB = p.key_mask_stride;
  a.lq = p.q_len;
  a.lk = p.k_len;
  a.heads = p.heads;
  a.kvHeads = p.kv_heads;
  a.dq = p.q_head_dim;
  a.dv = p.v_head_dim;
  a.scaleLog2 = p.scale * 1.44269504088896341f;
  const AttentionPlan plan = planAttention(p, p.workspace != nullptr ? p.workspace_bytes : 0);
  AttnSplit split{plan.splits, nullptr, nullptr};
  if(plan.splits > 1) {
    split.out = (float*)p.workspace;
    split.state = split.out + (size_t)plan.splits * plan.rows * p.v_head_dim;
  }
  const int d = std::max(p.q_head_dim, p.v_head_dim);
  withDtype(p.dtype, [&](auto t) {
    typedef decltype(t) T;
    const auto run = [&](auto dim) {
      constexpr int D = decltype(dim)::value;
      if(p.q_head_dim == D && p.v_head_dim == D) runAttention<T, D, true>(plan, a, split, p.batch, stream);
      else runAttention<T, D, false>(plan, a, split, p.batch, stream);
    };
    if(d <= 32) run(std::integral_constant<int, 32>());
    else if(d <= 64) run(std::integral_constant<int, 64>());
    else run(std::integral_constant<int, 128>());
  });
}

}  // namespace kgh
