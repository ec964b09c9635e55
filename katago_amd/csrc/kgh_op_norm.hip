// Group norm with an activation, channels last (kgh_group_norm).
#include "kgh_op_norm_device.h"

#include <cfloat>

namespace {

struct NormOut {
  void* out;
  int64_t oB, oP;
  float* scales;  // of rows in 8 bits, or null
  float* stats;   // [batch][groups][2]: mean and 1 / sqrt(variance + eps), or null
};

// ---------------------------------------------------------------------------
// Sums of a group's values are of differences from a reference point, 0 at first: n,
// sum d and sum d^2 give mean and variance, and rounding costs them little where the
// reference lies within two deviations of the mean. Where it does not, they are taken
// once more from the mean found so far; where they pass the largest float, once more of
// values 2^-80 times as large. A group is done after three turns at most, almost every
// one after the first.
constexpr int NORM_TURNS = 3;
constexpr float NORM_SMALL = 0x1p-80f;

struct GroupTurn {
  float ref, factor;
};
struct GroupSums {
  float mean, var;  // var in units of the factor's square
  GroupTurn next;
  bool again;
};

// What a turn's sums over n values say.
__device__ __forceinline__ GroupSums groupSums(float n, float sum, float squares, GroupTurn turn, int turns) {
  GroupSums r;
  r.next = turn;
  r.again = false;
  const float share = 1.0f / n, m = sum * share;
  r.mean = fmaf(m, turn.factor == 1.0f ? 1.0f : 1.0f / NORM_SMALL, turn.ref);
  r.var = fmaf(-m, m, squares * share);
  if(!(fabsf(sum) <= FLT_MAX && squares <= FLT_MAX)) {
    r.var = __builtin_nanf("");
    r.again = turn.factor == 1.0f;
    r.next = GroupTurn{0.0f, NORM_SMALL};
  }
  else {
    r.var = fmaxf(r.var, 0.0f);
    r.again = turn.ref == 0.0f && m * m > 4.0f * r.var;
    r.next.ref = r.mean;
  }
  if(turns + 1 >= NORM_TURNS || n == 0.0f) r.again = false;
  if(!r.again) r.next = turn;
  return r;
}

__device__ __forceinline__ float reciprocalDeviation(const GroupSums& r, float eps) {
  if(r.next.factor == 1.0f) return 1.0f / sqrtf(r.var + eps);
  return (float)(1.0 / sqrt((double)r.var * 0x1p160 + (double)eps));
}

// (x - mean) / deviation, weight, bias and activation of VEC channels. (With the mean in
// the bias, one operation less, a group of equal values would not be its bias exactly; it
// was no faster.)
template<typename T, int ACT, int VEC>
__device__ __forceinline__ void normalise(float (&y)[VEC], const Values<T>& x, const float (&mean)[VEC], const float (&scale)[VEC], const float (&bias)[VEC]) {
#pragma unroll
  for(int j = 0; j < VEC; j++) y[j] = activate<T, ACT>(fmaf(x.f[j] - mean[j], scale[j], bias[j]));
}

// ---------------------------------------------------------------------------
// An item's run of channels lies in a unit's registers from its one way in to its way
// out: sums over a thread's positions for each of its channels, over the unit's threads
// in LDS, then norm and activation of the same registers. Positions that take no part are
// neither read nor computed: threads have places in a list of those that do. QUANT: rows
// in 8 bits, a unit being an item with all of its channels.
// 256 x 361 x 384 fp16, 32 groups, mish: 50 us of 142 MB (2.9 TB/s), with 54% of the
// positions 42; vector instructions are 0.65 of the cycles, and a CU's four workgroups
// come in two rounds that overlap in part. Registers decide: with 12 vectors a thread
// four workgroups of 256 threads a CU, where the floats of x beside them, or another
// turn from registers, left three or spilled. (Instances hold 2, 4, 12 and 16 vectors, by 76,
// 80, 116 and 128 registers in 16 bits; ones between 4 and 12 were not tried.)
template<typename T, int ACT, int NV, bool QUANT>
__global__ __launch_bounds__(NV == 2 ? 1024 : 512, NV == 16 ? 3 : 4) void normSlabKernel(NormArgs a, NormOut o, NormSlab s) {
  constexpr int VEC = 16 / (int)sizeof(T);
  extern __shared__ float2 lds[];
  __shared__ int again;  // the last turn that a group needs
  if(threadIdx.x == 0) again = 0;
  const SlabThread<VEC> th(a, s);
  const int inRun = s.run / a.per;
  float2* part = lds + th.unit * s.ldsPairs;
  float2* state = part + s.ldsPairs - 2 * inRun;  // a group's reference and factor
  float2* result = state + inRun;                 // its mean and reciprocal deviation
  unsigned short* list = (unsigned short*)((char*)lds + s.listAt) + th.unit * (listBytes(a.positions) / 2);
  const T* x = (const T*)a.x + th.b * a.xB + th.at;
  int count = validLength(a, th.b);  // places that take part
  if(a.mask != nullptr) count = listPositions(a, th.b, count, list);
  count = __builtin_amdgcn_readfirstlane(count);
  auto position = [&](int place) -> unsigned { return a.mask != nullptr ? list[place] : place; };
  u32x4_t v[NV];
#pragma unroll
  for(int i = 0, from = 0; i < NV; i++, from += s.rowLanes)
    if(from < count) __builtin_memcpy(&v[i], x + (uint64_t)position(min(th.row + from, a.positions - 1)) * a.xP, 16);

  {
    const int rowLanes = fresh(s.rowLanes);
    float s1[VEC], s2[VEC];
#pragma unroll
    for(int j = 0; j < VEC; j++) s1[j] = s2[j] = 0.0f;
#pragma unroll
    for(int i = 0, from = 0; i < NV; i++, from += rowLanes)
      if(from < count) {
        if(from + rowLanes > count) {  // the last places that take part
          const u32x4_t zero = {0, 0, 0, 0};
          v[i] = th.row + from < count ? v[i] : zero;
        }
        const Values<T> d(v[i]);
#pragma unroll
        for(int j = 0; j < VEC; j++) {
          s1[j] += d.f[j];
          s2[j] = fmaf(d.f[j], d.f[j], s2[j]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    if(th.on) {
      float2* p = part + th.row * s.entries + th.col * s.pv;
      if(s.pv == 1) {
#pragma unroll
        for(int j = 1; j < VEC; j++) s1[0] += s1[j], s2[0] += s2[j];
        *p = make_float2(s1[0], s2[0]);
      }
      else {
#pragma unroll
        for(int j = 0; j < VEC; j++)
          if(j >= th.skip) p[j - th.skip] = make_float2(s1[j], s2[j]);
      }
    }
    __syncthreads();
  }
  // The groups' mean and deviation by a turn's sums; whether one needs another turn.
  auto finish = [&](int turn) {
    const float n = (float)count * (float)a.per;
    for(int q = th.tt >> s.lanesLog; q < th.groups; q += s.threads >> s.lanesLog) {
      float2 sums = make_float2(0.0f, 0.0f);
      eachEntry(part, s, s.rowLanes, q, th.tt, [&](float2 u, int) {
        sums.x += u.x;
        sums.y += u.y;
      });
      sums = addLanes(sums, s.lanesLog);
      const GroupSums t = groupSums(n, sums.x, sums.y, turn == 0 ? GroupTurn{0.0f, 1.0f} : GroupTurn{state[q].x, state[q].y}, turn);
      if((th.tt & ((1 << s.lanesLog) - 1)) == 0) {
        const float rd = reciprocalDeviation(t, a.eps);
        state[q] = make_float2(t.next.ref, t.next.factor);
        result[q] = n == 0.0f ? make_float2(0.0f, 0.0f) : make_float2(t.mean, rd);
        if(t.again) again = turn + 1;
      }
    }
    __syncthreads();
    return again == turn + 1;
  };
  if(finish(0)) {
    // Other turns read x again, from a cache: in the registers' copy they would cost
    // every unit a quarter of its workgroups a CU.
#pragma unroll 1
    for(int turn = 1;; turn++) {
      // (four channels at a time, for the same reason)
      float2 all = make_float2(0.0f, 0.0f);
#pragma unroll 1
      for(int j0 = 0; j0 < VEC; j0 += 4) {
        float s1[4], s2[4], ref[4], factor[4];
#pragma unroll
        for(int j = 0; j < 4; j++) {
          const float2 t = state[min((th.channel + max(j0 + j - th.skip, 0)) / a.per, th.groups - 1)];
          s1[j] = s2[j] = 0.0f;
          ref[j] = t.x * t.y;
          factor[j] = t.y;
        }
#pragma unroll 1
        for(int place = th.row; place < count; place += s.rowLanes) {
          T e[4];
          __builtin_memcpy(e, x + j0 + (uint64_t)position(place) * a.xP, sizeof(e));
#pragma unroll
          for(int j = 0; j < 4; j++) {
            const float d = fmaf((float)e[j], factor[j], -ref[j]);
            s1[j] += d;
            s2[j] = fmaf(d, d, s2[j]);
          }
        }
#pragma unroll
        for(int j = 0; j < 4; j++) {
          all.x += s1[j];
          all.y += s2[j];
          if(s.pv > 1 && th.on && j0 + j >= th.skip) part[th.row * s.entries + th.channel + j0 + j - th.skip] = make_float2(s1[j], s2[j]);
        }
      }
      if(s.pv == 1 && th.on) part[th.row * s.entries + th.col] = all;
      __syncthreads();
      if(!finish(turn)) break;
    }
  }

  if(o.stats != nullptr && th.live)
    for(int q = th.tt; q < th.groups; q += s.threads) *(float2*)(o.stats + 2 * ((int64_t)th.b * a.groups + th.c1 / a.per + q)) = result[q];
  float scale[VEC], bias[VEC], mean[VEC];
  loadFloats(scale, a.weight == nullptr ? nullptr : a.weight + th.at, VEC, 1.0f);
  loadFloats(bias, a.bias == nullptr ? nullptr : a.bias + th.at, VEC, 0.0f);
  th.eachGroup(a, [&](int j, int q) {
    const float2 t = result[q];
    mean[j] = t.x;
    scale[j] *= t.y;
  });
  const bool stores = th.on && th.live;
  if constexpr(!QUANT) {
    if(!stores) return;
    T* out = (T*)o.out + th.b * o.oB + th.at;
    const int rowLanes = fresh(s.rowLanes);
#pragma unroll
    for(int i = 0, from = 0; i < NV; i++, from += rowLanes)
      if(from < a.positions) {
        const int place = th.row + from;
        uint4 u = make_uint4(0, 0, 0, 0);
        if(from < count) {
          float y[VEC];
          renew(v[i]);
          normalise<T, ACT>(y, Values<T>(v[i]), mean, scale, bias);
          u = packed<T>(y);
          if(from + rowLanes > count && place >= count) u = make_uint4(0, 0, 0, 0);
        }
        if(place < a.positions) {
          T* p = out + (uint64_t)position(place) * o.oP;
          if(a.channels % VEC == 0) __builtin_memcpy(p, &u, 16);
          else storeWindow(p, u, th.skip);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
  }
  else {
    unsigned* tops = (unsigned*)part;  // of places
    for(int p = th.tt; p < a.positions; p += s.threads) tops[p] = 0;
    __syncthreads();
    float y[NV][VEC];
#pragma unroll
    for(int i = 0; i < NV; i++)
      if(i * s.rowLanes < count) {
        const int place = th.row + i * s.rowLanes;
        renew(v[i]);
        normalise<T, ACT>(y[i], Values<T>(v[i]), mean, scale, bias);
        unsigned top = 0;
#pragma unroll
        for(int j = 0; j < VEC; j++) top = max(top, j >= th.skip ? magnitudeBits(y[i][j]) : 0);
        if(th.on && place < count) atomicMax(&tops[place], top);
      }
    __syncthreads();
    int8_t* out = (int8_t*)o.out + th.b * o.oB + th.at;
#pragma unroll
    for(int i = 0; i < NV; i++) {
      const int place = th.row + i * s.rowLanes;
      if(stores && place < a.positions) {
        const unsigned p = position(place);
        const RowScale rs(tops[place]);
        const uint2 q = quantized(y[i], rs);
        storeBytes<VEC>(out + (uint64_t)p * o.oP, place < count ? q : make_uint2(0, 0), th.skip, VEC);
        if(th.col == 0) o.scales[(int64_t)th.b * a.positions + p] = rs.scale;
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Items that no workgroup's registers hold: their positions in `chunks`, their columns in
// `blocks` of `cols`, each a workgroup. A part's groups have their
// number of values, mean, sum of squares about it and that sum's factor in
// parts[item][chunk][block][slot], slot 0 being the block's first group. A chunk's rows
// are every chunks-th `rowLanes` rows, so that the card reads one stretch at a time; with
// eight rows of a thread under way 4 x 16384 x 512 bf16 takes 22 us (3.0 TB/s of reads;
// reading alone reaches 4.0), 24 for the results behind it and 4 for the join.
struct NormParts {
  float4* parts;
  int chunks, chunkRows, blocks, cols, rowLanes, slots, lanes, pv;  // lanes: threads that add up a group; pv: see NormSlab
};

constexpr int PARTS_AHEAD = 8, APPLY_AHEAD = 8;  // rows of a thread under way

template<typename T>
__global__ __launch_bounds__(256) void normPartsKernel(NormArgs a, NormParts k) {
  constexpr int VEC = 16 / (int)sizeof(T);
  __shared__ float2 part[256 * VEC];
  __shared__ float2 state[256 * VEC];
  __shared__ int counted;
  const int row = threadIdx.x / k.cols, col = threadIdx.x - row * k.cols;
  const int64_t all = (int64_t)a.batch * k.chunks * k.blocks;
  for(int64_t id = blockIdx.x; id < all; id += gridDim.x) {
    const int64_t itemChunk = id / k.blocks;
    const int block = (int)(id - itemChunk * k.blocks);
    const int b = (int)(itemChunk / k.chunks), chunk = (int)(itemChunk - (int64_t)b * k.chunks);
    const int from = block * k.cols * VEC, to = min(from + k.cols * VEC, a.channels);
    const int c0 = from + col * VEC, nc = min(to - c0, VEC);
    const bool on = row < k.rowLanes && nc > 0;
    const int firstGroup = from / a.per, groups = (to - 1) / a.per - firstGroup + 1;
    const int len = validLength(a, b);
    const int step = k.chunks * k.rowLanes;
    const RowGroup<T, false> g((on ? c0 : 0) / VEC, a.channels);
    const T* x = (const T*)a.x + b * a.xB;
    const uint8_t* mask = a.mask == nullptr ? nullptr : a.mask + b * a.maskB;
    if(threadIdx.x == 0) counted = 0;
    __syncthreads();
    auto groupOf = [&](int j) { return (c0 + max(min(j, nc - 1), 0)) / a.per - firstGroup; };
    int rows = 0;
    for(int turns = 0;; turns++) {
      float s1[VEC], s2[VEC], ref[VEC], factor[VEC];
#pragma unroll
      for(int j = 0; j < VEC; j++) {
        s1[j] = s2[j] = ref[j] = 0.0f;
        factor[j] = 1.0f;
        if(turns > 0 && on) {
          const float2 t = state[groupOf(j)];
          factor[j] = t.y;
          ref[j] = t.x * t.y;
        }
      }
      rows = 0;
      if(on) {
        for(int p = chunk * k.rowLanes + row; p < len; p += PARTS_AHEAD * step) {
          u32x4_t v[PARTS_AHEAD];
          bool take[PARTS_AHEAD];
#pragma unroll
          for(int i = 0; i < PARTS_AHEAD; i++) {
            const int q = p + i * step;
            take[i] = q < len && (mask == nullptr || mask[q] != 0);
          }
#pragma unroll
          for(int i = 0; i < PARTS_AHEAD; i++) v[i] = g.load(x + (uint64_t)(unsigned)(take[i] ? p + i * step : p) * a.xP);
#pragma unroll
          for(int i = 0; i < PARTS_AHEAD; i++) {
            rows += take[i] ? 1 : 0;
            const u32x4_t zero = {0, 0, 0, 0};
            const Values<T> u(take[i] ? g.place(v[i]) : zero);
#pragma unroll
            for(int j = 0; j < VEC; j++) {
              const float d = turns == 0 ? u.f[j] : take[i] && j < nc ? fmaf(u.f[j], factor[j], -ref[j]) : 0.0f;
              s1[j] += d;
              s2[j] = fmaf(d, d, s2[j]);
            }
          }
        }
      }
      if(turns == 0 && on && col == 0 && rows > 0) atomicAdd(&counted, rows);
      if(row < k.rowLanes) {
        if(k.pv == 1) {
#pragma unroll
          for(int j = 1; j < VEC; j++) s1[0] += s1[j], s2[0] += s2[j];
          part[row * k.cols + col] = make_float2(s1[0], s2[0]);
        }
        else {
#pragma unroll
          for(int j = 0; j < VEC; j++) part[(row * k.cols + col) * VEC + j] = make_float2(s1[j], s2[j]);
        }
      }
      __syncthreads();
      // A group's entries in this block, over the rows, by `lanes` threads.
      const int sub = threadIdx.x & (k.lanes - 1);
      bool again = false;
      for(int q = threadIdx.x / k.lanes; q < groups; q += 256 / k.lanes) {
        const int c0 = max((firstGroup + q) * a.per - from, 0), c1 = min((firstGroup + q + 1) * a.per, to) - from;
        const int e0 = k.pv == 1 ? c0 / VEC : c0, e1 = k.pv == 1 ? c1 / VEC : c1;
        float sum = 0.0f, squares = 0.0f;
#pragma unroll 4
        for(int i = sub; i < (e1 - e0) * k.rowLanes; i += k.lanes) {
          const int r = i / (e1 - e0);
          const float2 u = part[r * k.cols * k.pv + e0 + (i - r * (e1 - e0))];
          sum += u.x;
          squares += u.y;
        }
        for(int w = k.lanes >> 1; w > 0; w >>= 1) {
          sum += __shfl_xor(sum, w);
          squares += __shfl_xor(squares, w);
        }
        const float n = (float)counted * (float)(c1 - c0);
        const GroupSums t = groupSums(n, sum, squares, turns == 0 ? GroupTurn{0.0f, 1.0f} : GroupTurn{state[q].x, state[q].y}, turns);
        again |= t.again;
        if(sub == 0) {
          state[q] = make_float2(t.next.ref, t.next.factor);
          k.parts[id * k.slots + q] = n == 0.0f ? make_float4(0.0f, 0.0f, 0.0f, 1.0f) : make_float4(n, t.mean, t.var, t.next.factor);
        }
      }
      if(!__syncthreads_or(again)) break;
    }
  }
}

// The parts of a group in one: mean, then the squares about it, in 64 bits (numbers are
// few, and may be any fp32's square). A wave a group of an item; up to 64 JOIN_AHEAD
// parts are all under way at a time and stay in registers between the two.
constexpr int JOIN_AHEAD = 8;

__global__ __launch_bounds__(256) void normJoinKernel(NormArgs a, NormParts k, float* stats, int vec) {
  const int lane = threadIdx.x & 63;
  for(int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); i < (int64_t)a.batch * a.groups; i += (int64_t)gridDim.x * 4) {
    const int b = (int)(i / a.groups), g = (int)(i - (int64_t)b * a.groups);
    const int width = k.cols * vec;
    const int block0 = g * a.per / width, blocks = ((g + 1) * a.per - 1) / width - block0 + 1;
    const int64_t parts = (int64_t)k.chunks * blocks, first = (int64_t)b * k.chunks;
    auto part = [&](int64_t e) {
      const int64_t chunk = blocks == 1 ? e : e / blocks;
      const int block = block0 + (int)(e - chunk * blocks);
      return k.parts[((first + chunk) * k.blocks + block) * k.slots + g - block * width / a.per];
    };
    float4 v[JOIN_AHEAD];
#pragma unroll
    for(int q = 0; q < JOIN_AHEAD; q++) v[q] = lane + 64 * q < parts ? part(lane + 64 * q) : make_float4(0.0f, 0.0f, 0.0f, 1.0f);
    double n = 0.0, sum = 0.0, squares = 0.0;
    const auto add = [&](float4 t) {
      n += t.x;
      sum += (double)t.x * t.y;
    };
#pragma unroll
    for(int q = 0; q < JOIN_AHEAD; q++) add(v[q]);
    for(int64_t e = lane + 64 * JOIN_AHEAD; e < parts; e += 64) add(part(e));
#pragma unroll
    for(int w = 32; w > 0; w >>= 1) {
      n += __shfl_xor(n, w);
      sum += __shfl_xor(sum, w);
    }
    const double mean = n == 0.0 ? 0.0 : sum / n;
    const auto square = [&](float4 t) {
      const double d = t.y - mean;
      squares += t.x == 0.0f ? 0.0 : t.x * ((t.w == 1.0f ? (double)t.z : t.z * 0x1p160) + d * d);
    };
#pragma unroll
    for(int q = 0; q < JOIN_AHEAD; q++) square(v[q]);
    for(int64_t e = lane + 64 * JOIN_AHEAD; e < parts; e += 64) square(part(e));
#pragma unroll
    for(int w = 32; w > 0; w >>= 1) squares += __shfl_xor(squares, w);
    if(lane == 0) {
      stats[i * 2] = (float)mean;
      stats[i * 2 + 1] = n == 0.0 ? 0.0f : (float)(1.0 / sqrt(squares / n + (double)a.eps));
    }
  }
}

// Norm and activation of what normJoinKernel has the statistics of: the same chunks and
// blocks, a thread with a column's constants in registers.
template<typename T, int ACT>
__global__ __launch_bounds__(256) void normApplyKernel(NormArgs a, NormOut o, NormParts k) {
  constexpr int VEC = 16 / (int)sizeof(T);
  const int row = threadIdx.x / k.cols, col = threadIdx.x - row * k.cols;
  const int64_t all = (int64_t)a.batch * k.chunks * k.blocks;
  if(row >= k.rowLanes) return;
  for(int64_t id = blockIdx.x; id < all; id += gridDim.x) {
    const int64_t itemChunk = id / k.blocks;
    const int block = (int)(id - itemChunk * k.blocks);
    const int b = (int)(itemChunk / k.chunks), chunk = (int)(itemChunk - (int64_t)b * k.chunks);
    const int c0 = (block * k.cols + col) * VEC, nc = min(a.channels - c0, VEC);
    if(nc <= 0) continue;
    const int len = validLength(a, b);
    const int p0 = chunk * k.chunkRows, p1 = min(p0 + k.chunkRows, a.positions);
    const RowGroup<T, false> g(c0 / VEC, a.channels);
    const T* x = (const T*)a.x + b * a.xB;
    T* out = (T*)o.out + b * o.oB + c0;
    const uint8_t* mask = a.mask == nullptr ? nullptr : a.mask + b * a.maskB;
    float mean[VEC], scale[VEC], bias[VEC];
    loadFloats(scale, a.weight == nullptr ? nullptr : a.weight + c0, nc, 1.0f);
    loadFloats(bias, a.bias == nullptr ? nullptr : a.bias + c0, nc, 0.0f);
#pragma unroll
    for(int j = 0; j < VEC; j++) {
      const float* t = o.stats + 2 * ((int64_t)b * a.groups + (c0 + min(j, nc - 1)) / a.per);
      mean[j] = t[0];
      scale[j] *= t[1];
    }
    for(int p = p0 + row; p < p1; p += APPLY_AHEAD * k.rowLanes) {
      u32x4_t v[APPLY_AHEAD];
      bool take[APPLY_AHEAD];
#pragma unroll
      for(int i = 0; i < APPLY_AHEAD; i++) {
        const int q = min(p + i * k.rowLanes, p1 - 1);
        take[i] = q < len && (mask == nullptr || mask[q] != 0);
      }
#pragma unroll
      for(int i = 0; i < APPLY_AHEAD; i++) v[i] = g.load(x + (take[i] ? min(p + i * k.rowLanes, p1 - 1) : 0) * a.xP);
#pragma unroll
      for(int i = 0; i < APPLY_AHEAD; i++) {
        const int q = p + i * k.rowLanes;
        float y[VEC];
        normalise<T, ACT>(y, Values<T>(g.place(v[i])), mean, scale, bias);
        const uint4 u = packed<T>(y), zero = make_uint4(0, 0, 0, 0);
        if(q < p1) storeGroup(out + q * o.oP, take[i] ? u : zero, nc);
      }
    }
  }
}

// The same in 8 bits: a row's columns by `lanes` threads, K each, and R rows at a time.
// 46208 x 384 bf16, SiLU: 27 us (2.0 TB/s); vector instructions bound it. In 16 bits four
// groups a thread (4097 to 8192 channels) take 256 registers, one wave a SIMD: 4096 x 8192
// bf16 60 us (1.7 TB/s).
template<typename T, int ACT, int K, int R>
__global__ __launch_bounds__(256) void normQuantKernel(NormArgs a, NormOut o, int lanes, int chunks, int chunkRows) {
  constexpr int VEC = 16 / (int)sizeof(T);
  __shared__ unsigned tops[2][R][4];
  const int sub = threadIdx.x & (lanes - 1), row = threadIdx.x / lanes, rows = 256 / lanes;
  const int groups = (a.channels + VEC - 1) / VEC;
  const bool whole = a.channels % VEC == 0;  // no thread has part of a group
  for(int64_t id = blockIdx.x; id < (int64_t)a.batch * chunks; id += gridDim.x) {
    const int b = (int)(id / chunks), chunk = (int)(id - (int64_t)b * chunks);
    const int len = validLength(a, b);
    const int p0 = chunk * chunkRows, p1 = min(p0 + chunkRows, a.positions);
    const T* x = (const T*)a.x + b * a.xB;
    int8_t* out = (int8_t*)o.out + b * o.oB;
    const uint8_t* mask = a.mask == nullptr ? nullptr : a.mask + b * a.maskB;
    float mean[K][VEC], scale[K][VEC], bias[K][VEC];
#pragma unroll
    for(int i = 0; i < K; i++) {
      const int c0 = (sub + i * lanes) * VEC, nc = a.channels - c0;
      loadFloats(scale[i], a.weight == nullptr ? nullptr : a.weight + c0, nc, 1.0f);
      loadFloats(bias[i], a.bias == nullptr ? nullptr : a.bias + c0, nc, 0.0f);
      int q = c0 / a.per, rest = c0 - q * a.per;
#pragma unroll
      for(int j = 0; j < VEC; j++) {
        const float2 t = *(const float2*)(o.stats + 2 * ((int64_t)b * a.groups + min(q, a.groups - 1)));
        mean[i][j] = t.x;
        scale[i][j] *= t.y;
        if(++rest == a.per) {
          rest = 0;
          q++;
        }
      }
    }
    int turn = 0;
    for(int from = p0; from < p1; from += R * rows, turn ^= 1) {
      u32x4_t v[R][K];
      bool take[R];
#pragma unroll
      for(int r = 0; r < R; r++) {
        const int p = from + r * rows + row;
        take[r] = p < min(p1, len) && (mask == nullptr || mask[p] != 0);
      }
#pragma unroll
      for(int r = 0; r < R; r++)
#pragma unroll
        for(int i = 0; i < K; i++)
          v[r][i] = RowGroup<T, false>(min(sub + i * lanes, groups - 1), a.channels).load(x + (uint64_t)(unsigned)(take[r] ? from + r * rows + row : 0) * a.xP);
#pragma unroll
      for(int r = 0; r < R; r++) {
        const int p = from + r * rows + row;
        float y[K][VEC];
        unsigned top = 0;
#pragma unroll
        for(int i = 0; i < K; i++) {
          const int nc = a.channels - (sub + i * lanes) * VEC;
          const unsigned before = top;
          normalise<T, ACT>(y[i], Values<T>(RowGroup<T, false>(min(sub + i * lanes, groups - 1), a.channels).place(v[r][i])), mean[i], scale[i], bias[i]);
#pragma unroll
          for(int j = 0; j < VEC; j++) top = max(top, whole || j < nc ? magnitudeBits(y[i][j]) : 0);
          if(whole && nc <= 0) top = before;
        }
        top = rowTop(take[r] ? top : 0, lanes, tops[turn][r]);
        const RowScale rs(top);
        if(p < p1) {
#pragma unroll
          for(int i = 0; i < K; i++) {
            const int c0 = (sub + i * lanes) * VEC, nc = a.channels - c0;
            if(nc > 0) storeBytes<VEC>(out + (uint64_t)(unsigned)p * o.oP + c0, take[r] ? quantized(y[i], rs) : make_uint2(0, 0), 0, nc);
          }
          if(sub == 0) o.scales[(int64_t)b * a.positions + p] = rs.scale;
        }
      }
    }
    __syncthreads();
  }
}

// Rows of any length in 8 bits: each value computed twice.
template<typename T, int ACT>
__global__ __launch_bounds__(256) void normQuantLongKernel(NormArgs a, NormOut o) {
  __shared__ unsigned tops[4];
  for(int i = blockIdx.x; i < a.batch * a.positions; i += gridDim.x) {
    const int b = i / a.positions, p = i - b * a.positions;
    const T* x = (const T*)a.x + b * a.xB + p * a.xP;
    int8_t* out = (int8_t*)o.out + b * o.oB + p * o.oP;
    const bool take = p < validLength(a, b) && (a.mask == nullptr || a.mask[b * a.maskB + p] != 0);
    auto value = [&](int c) {
      const float* t = o.stats + 2 * ((int64_t)b * a.groups + c / a.per);
      const float scale = (a.weight != nullptr ? a.weight[c] : 1.0f) * t[1];
      return activate<T, ACT>(fmaf((float)x[c] - t[0], scale, a.bias != nullptr ? a.bias[c] : 0.0f));
    };
    unsigned top = 0;
    if(take)
      for(int c = threadIdx.x; c < a.channels; c += 256) top = max(top, magnitudeBits(value(c)));
    const RowScale rs(rowTop(top, 256, tops));
    for(int c = threadIdx.x; c < a.channels; c += 256) out[c] = (int8_t)(take ? rs.quantized(value(c)) & rs.keep & 0xff : 0);
    if(threadIdx.x == 0) o.scales[i] = rs.scale;
    __syncthreads();
  }
}

// The statistics of items without positions, where there is nothing else.
__global__ __launch_bounds__(256) void normNothingKernel(float* stats, int64_t n) {
  for(int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) stats[i] = 0.0f;
}

constexpr int NORM_QUANT_EACH = 4;  // 16-byte groups of a thread
constexpr int NORM_RUN_BYTES = 96;  // of a unit's rows at least; see planNorm

struct NormPlan {
  NormSlab slab;    // threads 0: parts
  NormParts parts;
  uint64_t partsBytes, statsBytes;
};

NormPlan planNorm(const kgh_group_norm_params& p) {
  const int size = (int)kgh::opElemBytes(p.dtype), vec = 16 / size;
  const bool quant = p.out_scales != nullptr;
  NormPlan plan{};
  // In registers where they hold an item's run, else in parts: us of 256 x 361 x 384 fp16
  // in 32 groups 50 and 73, of 16 x 361 x 384 9.8 and 18.5, of 24 x 1531 x 190 fp32 in 19
  // 29 and 39, of 8192 x 1 x 4096 bf16 in 8 bits 63 and 161. Longer runs' rows are fewer
  // pieces of lines of memory, shorter ones' units more: 48, 96 and 192 bytes take the same
  // time within 5%.
  const auto slab = [&](int bytes, int most, int wide) {
    if(plan.slab.threads == 0) plan.slab = planSlab(p.positions, p.channels, p.groups, size, bytes, false, most, wide, quant, 2);
  };
  if(quant) slab(NORM_RUN_BYTES, 2, 1024);
  else {
    slab(NORM_RUN_BYTES, 12, 512);
    slab(NORM_RUN_BYTES, 16, 512);
    slab(32, 16, 512);
    slab(32, 2, 1024);
  }
  if(plan.slab.threads != 0) return plan;
  NormParts& k = plan.parts;
  const int cols = (p.channels + vec - 1) / vec, per = p.channels / p.groups;
  k.cols = std::min(cols, 256);
  k.blocks = (cols + k.cols - 1) / k.cols;
  k.rowLanes = std::min(256 / k.cols, p.positions);
  // A thread's rows are added one after the other: at most 128; where they are fewer, four
  // workgroups a CU (4 x 16384 x 512 bf16: 512, 1024 and 2048 workgroups 52, 50 and 53 us).
  const int64_t rows = std::max<int64_t>(1, std::min<int64_t>(128, (int64_t)p.batch * p.positions * k.blocks / k.rowLanes / 1024));
  k.chunkRows = (int)std::min<int64_t>(p.positions, (rows + PARTS_AHEAD - 1) / PARTS_AHEAD * PARTS_AHEAD * k.rowLanes);
  k.chunks = (p.positions + k.chunkRows - 1) / k.chunkRows;
  k.slots = (k.cols * vec + per - 2) / per + 1;
  k.pv = per % vec == 0 ? 1 : vec;
  k.lanes = 64;
  while(k.lanes > 1 && k.lanes * k.slots > 256) k.lanes /= 2;
  plan.partsBytes = (uint64_t)p.batch * k.chunks * k.blocks * k.slots * sizeof(float4);
  plan.statsBytes = (uint64_t)p.batch * p.groups * 8;
  return plan;
}

template<typename T, int ACT>
void launchNorm(const NormPlan& plan, const NormArgs& a, NormOut o, void* workspace, hipStream_t stream) {
  const bool quant = o.scales != nullptr;
  if(plan.slab.threads != 0) {
    forUnits(a, plan.slab, [&](const NormSlab& s, unsigned grid, unsigned threads, size_t bytes) {
      if(quant) normSlabKernel<T, ACT, 2, true><<<grid, threads, bytes, stream>>>(a, o, s);
      else if(s.nv <= 2) normSlabKernel<T, ACT, 2, false><<<grid, threads, bytes, stream>>>(a, o, s);
      else if(s.nv <= 4) normSlabKernel<T, ACT, 4, false><<<grid, threads, bytes, stream>>>(a, o, s);
      else if(s.nv <= 12) normSlabKernel<T, ACT, 12, false><<<grid, threads, bytes, stream>>>(a, o, s);
      else normSlabKernel<T, ACT, 16, false><<<grid, threads, bytes, stream>>>(a, o, s);
      KGH_CHECK_LAUNCH();
    });
    return;
  }
  NormParts k = plan.parts;
  k.parts = (float4*)workspace;
  if(o.stats == nullptr) o.stats = (float*)((char*)workspace + plan.partsBytes);
  const unsigned grid = normGrid((int64_t)a.batch * k.chunks * k.blocks);
  normPartsKernel<T><<<grid, 256, 0, stream>>>(a, k);
  KGH_CHECK_LAUNCH();
  normJoinKernel<<<normGrid(((int64_t)a.batch * a.groups + 3) / 4), 256, 0, stream>>>(a, k, o.stats, 16 / (int)sizeof(T));
  KGH_CHECK_LAUNCH();
  if(!quant) normApplyKernel<T, ACT><<<grid, 256, 0, stream>>>(a, o, k);
  else {
    constexpr int VEC = 16 / (int)sizeof(T);
    const RowLanes r = rowLanes((a.channels + VEC - 1) / VEC, NORM_QUANT_EACH);
    if(r.lanes == 0) normQuantLongKernel<T, ACT><<<normGrid((int64_t)a.batch * a.positions), 256, 0, stream>>>(a, o);
    else {
      // Chunks of five workgroups a CU: a chunk begins with its columns' constants (128 x 361
      // x 384: 640, 1280 and 2560 workgroups 45.9, 43.0 and 43.8 us).
      const int rows = 256 / r.lanes * (r.each == 1 ? 2 : 1);
      const int chunkRows = (int)std::min<int64_t>((int64_t)a.positions, std::max<int64_t>(1, (int64_t)a.batch * a.positions / rows / 1280) * rows);
      const int chunks = (a.positions + chunkRows - 1) / chunkRows;
      const unsigned g = normGrid((int64_t)a.batch * chunks);
      if(r.each == 1) normQuantKernel<T, ACT, 1, 2><<<g, 256, 0, stream>>>(a, o, r.lanes, chunks, chunkRows);
      else if(r.each == 2) normQuantKernel<T, ACT, 2, 1><<<g, 256, 0, stream>>>(a, o, r.lanes, chunks, chunkRows);
      else normQuantKernel<T, ACT, 4, 1><<<g, 256, 0, stream>>>(a, o, r.lanes, chunks, chunkRows);
    }
  }
  KGH_CHECK_LAUNCH();
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
  if(p.batch > 0 && p.statistics != nullptr) opCheckPointer(op, "statistics", p.statistics, 4);
  if(p.batch == 0 || p.positions == 0) return;
  checkApartRows(op, "out", p.out_batch_stride, p.out_position_stride, p.batch, p.positions, p.channels);
  const size_t e = opElemBytes(p.dtype);
  opCheckPointer(op, "x", p.x, e);
  opCheckPointer(op, "out", p.out, p.out_scales != nullptr ? 1 : e);
  if(p.weight != nullptr) opCheckPointer(op, "weight", p.weight, 4);
  if(p.bias != nullptr) opCheckPointer(op, "bias", p.bias, 4);
  if(p.lengths != nullptr) opCheckPointer(op, "lengths", p.lengths, 4);
  if(p.out_scales != nullptr) opCheckPointer(op, "out_scales", p.out_scales, 4);
  if(p.x == p.out) {
    if(p.out_scales != nullptr) opInvalid(op, "out is x itself, in another type");
    if((p.batch > 1 && p.x_batch_stride != p.out_batch_stride) || (p.positions > 1 && p.x_position_stride != p.out_position_stride))
      opInvalid(op, "in place, the strides must be the same");
  }
  checkApartFrom(op, "out", p.out, {{"weight", p.weight}, {"bias", p.bias}, {"lengths", p.lengths}, {"mask", p.mask}, {"out_scales", p.out_scales}, {"statistics", p.statistics}});
  checkApartFrom(op, "out_scales", p.out_scales, {{"x", p.x}, {"weight", p.weight}, {"bias", p.bias}, {"lengths", p.lengths}, {"mask", p.mask}, {"statistics", p.statistics}});
  checkApartFrom(op, "statistics", p.statistics, {{"x", p.x}, {"weight", p.weight}, {"bias", p.bias}, {"lengths", p.lengths}, {"mask", p.mask}});
  opCheckWorkspace(op, p.workspace, p.workspace_bytes, groupNormWorkspace(p));
}

uint64_t groupNormWorkspace(const kgh_group_norm_params& p) {
  if(p.batch == 0 || p.positions == 0) return 0;
  const NormPlan plan = planNorm(p);
  return plan.partsBytes + plan.statsBytes;
}

void launchGroupNorm(const kgh_group_norm_params& p, hipStream_t stream) {
  if(p.batch > 0 && p.positions == 0 && p.statistics != nullptr) {
    const int64_t n = (int64_t)p.batch * p.groups * 2;
    normNothingKernel<<<normGrid((n + 255) / 256), 256, 0, stream>>>(p.statistics, n);
    KGH_CHECK_LAUNCH();
  }
  if(p.batch == 0 || p.positions == 0) return;
  const NormPlan plan = planNorm(p);
  const NormArgs a = normArgs(p, p.eps);
  const NormOut o{p.out, p.out_batch_stride, p.out_position_stride, p.out_scales, p.statistics};
  withDtype(p.dtype, [&](auto t) {
    withActivation(p.activation, [&](auto act) { launchNorm<decltype(t), decltype(act)::value>(plan, a, o, p.workspace, stream); });
  });
}

}  // namespace kgh
