// What group norm and its gradient share: arguments, layouts of threads, sums.
#ifndef KGH_OP_NORM_DEVICE_H
#define KGH_OP_NORM_DEVICE_H

#include "kgh_op_quantize_device.h"

#include <algorithm>
#include <initializer_list>
#include <utility>

namespace {

constexpr int NORM_MAX_LEN = 1 << 30, NORM_MAX_CHANNELS = 1 << 20;
constexpr int NORM_MAX_GRID = 1 << 20;  // workgroups of a launch

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

// A unit's threads: an item's run of `run` channels (whole groups), `cols` 16-byte
// columns of it side by side in `rowLanes` rows of threads; a thread has places row,
// row + rowLanes, ..., `nv` of them, in the list of the item's positions that begins
// with those that take part. `units` units share a workgroup.
// Sums go through LDS as pairs: `pv` a column (one where a group is whole columns, else
// one a channel), `entries` = cols pv a row; a group's are added by 2^lanesLog threads,
// whose steps are stepRows rows and stepEntries entries; where channels' sums are wanted,
// `segments` threads add up the rows of an entry before that.
struct NormSlab {
  int threads, units, run, runs, cols, rowLanes, nv, pv, entries, segments, groupEntries, lanesLog, stepRows, stepEntries;
  int ldsPairs;  // a unit's LDS, in pairs of floats: sums, then groups' state
  int listAt;    // its list of positions (16 bits each) behind the pairs of all units, in bytes; only where there is a mask
  int firstItem, launched;   // of this launch: its first item and its number of units
};

// 16 bytes that the compiler is to take for new ones: it would otherwise keep the floats
// of a unit's registers from one use to the next, twice as many registers.
__device__ __forceinline__ void renew(u32x4_t& v) { asm volatile("" : "+v"(v)); }

// The same of a number that all threads have: products of it are not kept from one loop
// to the next.
__device__ __forceinline__ int fresh(int n) {
  asm volatile("" : "+s"(n));
  return n;
}

template<typename T>
__device__ __forceinline__ uint4 packed(const float (&y)[16 / sizeof(T)]) {
  T e[16 / sizeof(T)];
#pragma unroll
  for(int j = 0; j < 16 / (int)sizeof(T); j++) e[j] = (T)y[j];
  uint4 u;
  __builtin_memcpy(&u, e, 16);
  return u;
}

// A thread's 16 bytes of a row of `channels` (at least VEC): those of channels c0..
// where they end in the row, else the row's last ones, the first `skip` of which are
// another thread's.
template<int VEC>
struct Window {
  int at, skip;
  __device__ __forceinline__ Window(int c0, int channels) {
    at = max(0, min(c0, channels - VEC));
    skip = min(c0 - at, VEC);
  }
};
// The window's own elements to p, the address of its first one.
template<typename T>
__device__ __forceinline__ void storeWindow(T* p, uint4 v, int skip) {
  if(skip == 0) __builtin_memcpy(p, &v, 16);
  else {
#pragma unroll 1
    for(int j = 0; j < 16 / (int)sizeof(T); j++) {
      T e;
      __builtin_memcpy(&e, &v.x, sizeof(T));
      if(j >= skip) p[j] = e;
      v = shiftDown<T>(v);
    }
  }
}

// n of the VEC floats from p on, `other` where p is null or behind them.
template<int VEC>
__device__ __forceinline__ void loadFloats(float (&f)[VEC], const float* p, int n, float other) {
  if(p != nullptr && n >= VEC) __builtin_memcpy(f, p, sizeof(f));
  else {
#pragma unroll
    for(int j = 0; j < VEC; j++) f[j] = p != nullptr && j < n ? p[j] : other;
  }
}

// What a thread of a unit is.
template<int VEC>
struct SlabThread {
  int unit, tt, row, col;
  int b, r, c1, groups;  // its item, run, first channel and groups
  int channel;           // its own first channel in the run
  int at, skip;          // see Window
  bool live, on;         // (units of the last workgroup that have no work go along)
  __device__ __forceinline__ SlabThread(const NormArgs& a, const NormSlab& s) {
    unit = s.units == 1 ? 0 : threadIdx.x >> 6;
    tt = threadIdx.x - unit * s.threads;
    row = tt / s.cols;
    col = tt - row * s.cols;
    const unsigned id = xcdContiguousTile() * s.units + unit;
    live = id < (unsigned)s.launched;
    const unsigned mine = live ? id : s.launched - 1;
    const unsigned item = mine / (unsigned)s.runs;
    b = s.firstItem + (int)item;
    r = (int)(mine - item * s.runs);
    c1 = r * s.run;
    groups = min(s.run / a.per, a.groups - c1 / a.per);
    channel = col * VEC;
    on = row < s.rowLanes && channel < min(s.run, a.channels - c1);
    const Window<VEC> win(c1 + channel, a.channels);
    at = win.at;
    skip = win.skip;
  }
  // f(j, q) for its channels j and their groups q in the run.
  template<typename F>
  __device__ __forceinline__ void eachGroup(const NormArgs& a, F&& f) const {
    int q = channel / a.per, rest = channel - q * a.per;
#pragma unroll
    for(int j = 0; j < VEC; j++) {
      f(j, min(q, groups - 1));
      rest += j >= skip ? 1 : 0;
      if(rest >= a.per) {
        rest = 0;
        q++;
      }
    }
  }
};

// The positions that take part, in order, then the others: list[0..positions). Returns
// how many take part. Every wave of a unit writes the whole list by itself, the same
// numbers in the same places, so that it need not wait for another one to read it.
__device__ __forceinline__ int listPositions(const NormArgs& a, int b, int len, unsigned short* list) {
  constexpr int AHEAD = 8;
  const uint8_t* mask = a.mask + b * a.maskB;
  const int lane = threadIdx.x & 63;
  int count = 0;
  for(int from = 0; from < a.positions; from += 64 * AHEAD) {
    uint8_t m[AHEAD];
#pragma unroll
    for(int i = 0; i < AHEAD; i++) m[i] = mask[min(from + i * 64 + lane, a.positions - 1)];
#pragma unroll
    for(int i = 0; i < AHEAD; i++) {
      const int p = from + i * 64 + lane;
      if(from + i * 64 >= a.positions) break;
      const bool on = p < len && m[i] != 0;
      const unsigned long long bits = __ballot(on);
      const int at = count + __popcll(bits & ((1ull << lane) - 1));
      if(p < a.positions) list[on ? at : a.positions - 1 - (p - at)] = (unsigned short)p;
      count += __popcll(bits);
    }
  }
  asm volatile("" ::: "memory");  // a wave's LDS accesses run in order
  return count;
}

// The sum of v over the 2^log threads side by side that share it, for all of them: within
// sixteen by rotations, without LDS.
__device__ __forceinline__ float rotated(float v, std::integral_constant<int, 8>) { return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x128, 0xf, 0xf, true)); }
__device__ __forceinline__ float rotated(float v, std::integral_constant<int, 4>) { return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x124, 0xf, 0xf, true)); }
__device__ __forceinline__ float rotated(float v, std::integral_constant<int, 2>) { return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x122, 0xf, 0xf, true)); }
__device__ __forceinline__ float rotated(float v, std::integral_constant<int, 1>) { return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x121, 0xf, 0xf, true)); }
__device__ __forceinline__ float2 addLanes(float2 v, int log) {
  if(log >= 4) {
    const auto add = [&](auto n) {
      v.x += rotated(v.x, n);
      v.y += rotated(v.y, n);
    };
    add(std::integral_constant<int, 8>());
    add(std::integral_constant<int, 4>());
    add(std::integral_constant<int, 2>());
    add(std::integral_constant<int, 1>());
  }
  else
    for(int k = (1 << log) >> 1; k > 0; k >>= 1) {
      v.x += __shfl_xor(v.x, k);
      v.y += __shfl_xor(v.y, k);
    }
  if(log >= 5) {
    v.x += __shfl_xor(v.x, 16);
    v.y += __shfl_xor(v.y, 16);
  }
  if(log >= 6) {
    v.x += __shfl_xor(v.x, 32);
    v.y += __shfl_xor(v.y, 32);
  }
  return v;
}

// f(pair, entry of the run) of this thread's part of group q: of pairs of sums
// [rows][entries].
template<typename F>
__device__ __forceinline__ void eachEntry(const float2* part, const NormSlab& s, int rows, int q, int tt, F&& f) {
  int row = 0, e = tt & ((1 << s.lanesLog) - 1);
  if(e >= s.groupEntries) {
    row = e / s.groupEntries;
    e -= row * s.groupEntries;
  }
#pragma unroll 4
  while(row < rows) {
    const int at = q * s.groupEntries + e;
    f(part[row * s.entries + at], at);
    row += s.stepRows;
    e += s.stepEntries;
    if(e >= s.groupEntries) {
      e -= s.groupEntries;
      row++;
    }
  }
}

// Rows (item, position) of a tensor that is written lie apart.
inline void checkApartRows(const char* op, const char* name, int64_t batchStride, int64_t positionStride, int batch, int positions, int channels) {
  const bool positionsInside = (positions == 1 || positionStride >= channels) && (batch == 1 || batchStride >= (positions - 1) * positionStride + channels);
  const bool itemsInside = (batch == 1 || batchStride >= channels) && (positions == 1 || positionStride >= (batch - 1) * batchStride + channels);
  if(!positionsInside && !itemsInside) kgh::opInvalid(op, std::string("the strides of ") + name + " make its rows overlap");
}

// An output that is no other one of the call's tensors.
inline void checkApartFrom(const char* op, const char* name, const void* out, std::initializer_list<std::pair<const char*, const void*>> others) {
  for(const auto& o : others)
    if(out != nullptr && out == o.second) kgh::opInvalid(op, std::string(name) + " is " + o.first + " itself");
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

__host__ __device__ __forceinline__ int listBytes(int positions) { return (positions * 2 + 15) / 16 * 16; }
inline unsigned normGrid(int64_t blocks) { return (unsigned)std::min<int64_t>(blocks, NORM_MAX_GRID); }

// Launches f(slab, grid, threads, bytes of LDS) for all units.
template<typename F>
void forUnits(const NormArgs& a, NormSlab s, F&& f) {
  const int64_t items = std::max<int64_t>(1, (int64_t)NORM_MAX_GRID * s.units / s.runs);
  for(int64_t item = 0; item < a.batch; item += items) {
    s.firstItem = (int)item;
    s.launched = (int)(std::min(items, a.batch - item) * s.runs);
    s.listAt = s.ldsPairs * 8 * s.units;
    f(s, (unsigned)((s.launched + s.units - 1) / s.units), (unsigned)(s.threads * s.units),
      (size_t)s.listAt + (a.mask != nullptr ? (size_t)listBytes(a.positions) * s.units : 0));
  }
}

// The layout of a unit's threads for items of these sizes: at most `most` positions a
// thread and `wide` threads; threads is 0 where there is none. Runs of at least `bytes` a
// row, or (wholeRows) of all channels. perChannel: sums of each channel are wanted. What a
// group has in LDS beside the sums: `state` pairs.
inline NormSlab planSlab(int positions, int channels, int groups, int size, int bytes, bool perChannel, int most, int wide, bool wholeRows,
                         int state) {
  const int vec = 16 / size, per = channels / groups;
  NormSlab none{};
  if(channels < vec || positions > 65536) return none;
  int64_t base = per;
  while(base % vec != 0) base += per;
  int64_t run = wholeRows ? channels : (bytes + base * size - 1) / (base * size) * base;
  if(run > channels) run = channels;
  // (whole rounds of the four SIMDs: waves that one of them has more of hold the others up)
  for(int threads : {64, 128, 256, 512, 768, 1024}) {
    NormSlab s{};
    if(threads > wide) break;
    s.run = (int)run;
    s.runs = (int)((channels + run - 1) / run);
    s.cols = (int)((run + vec - 1) / vec);
    s.threads = threads;
    s.units = threads == 64 ? 4 : 1;
    if(s.cols > threads) continue;
    s.rowLanes = std::min(threads / s.cols, positions);
    s.nv = (positions + s.rowLanes - 1) / s.rowLanes;
    if(s.nv > most) continue;
    s.pv = !perChannel && per % vec == 0 ? 1 : vec;
    s.entries = s.cols * s.pv;
    s.groupEntries = s.pv == 1 ? per / vec : per;
    s.segments = std::min(std::max(threads / s.entries, 1), s.rowLanes);
    s.ldsPairs = (s.rowLanes + (perChannel ? s.segments : 0)) * s.entries;
    const int inRun = s.run / per;
    s.lanesLog = 6;
    while(s.lanesLog > 0 && (inRun << s.lanesLog) > threads) s.lanesLog--;
    s.stepRows = (1 << s.lanesLog) / s.groupEntries;
    s.stepEntries = (1 << s.lanesLog) - s.stepRows * s.groupEntries;
    s.ldsPairs += state * inRun;
    if(((int64_t)s.ldsPairs * 8 + listBytes(positions)) * s.units > 60000) continue;
    return s;
  }
  return none;
}

}  // namespace

#endif
