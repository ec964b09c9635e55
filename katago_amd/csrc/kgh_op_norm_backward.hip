// The gradient of group norm with an activation (kgh_group_norm_backward).
#include "kgh_op_norm_device.h"

namespace {

// The activations' slopes. In 16 bits by the hardware's exponential and reciprocal, to
// within 2^-18 of 1; in fp32 by the accurate functions, to within 2^-20.
//   silu: s (1 + v (1 - s)), s = 1 / (1 + e^-v);
//   mish: with n = e^v (e^v + 2): n w + 4 v e^v (1 + e^v) w^2, w = 1 / (n + 2) (v e^v
//         before anything else: it is 0 where 4 v would pass the largest float);
//   gelu: Phi(v) + v phi(v).
template<typename T, int ACT>
__device__ __forceinline__ float slope(float v) {
  if constexpr(ACT == KGH_ACT_IDENTITY) return 1.0f;
  else if constexpr(ACT == KGH_ACT_RELU) return v > 0.0f ? 1.0f : v != v ? v : 0.0f;
  else if constexpr(ACT == KGH_ACT_SILU) {
    if constexpr(sizeof(T) == 4) {
      // (1 - s of an s next to 1 would have lost the bits that v multiplies)
      const float e = expf(-fabsf(v)), most = 1.0f / (1.0f + e), least = e * most;
      return (v < 0.0f ? least : most) * fmaf(v, v < 0.0f ? most : least, 1.0f);
    }
    else {
      const float s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(v * -ACT_LOG2E));
      return s * fmaf(v, 1.0f - s, 1.0f);
    }
  }
  else if constexpr(ACT == KGH_ACT_MISH) {
    const float c = v > 20.0f ? 20.0f : v;  // NaN stays NaN
    float e, w;
    if constexpr(sizeof(T) == 4) e = expf(c);
    else e = __builtin_amdgcn_exp2f(c * ACT_LOG2E);
    const float n = fmaf(e, e, 2.0f * e);
    if constexpr(sizeof(T) == 4) w = 1.0f / (n + 2.0f);
    else w = __builtin_amdgcn_rcpf(n + 2.0f);
    return w * fmaf(c * e * fmaf(e, 4.0f, 4.0f), w, n);
  }
  else if constexpr(sizeof(T) == 4) return fmaf(0.5f, erfcf(-0.70710678118654752f * v), v * expf(-0.5f * v * v) * 0.39894228040143268f);
  else {
    // erfc(|v| / sqrt(2)) / 2 = t poly(t) e^(-v^2 / 2), t = 1 / (1 + 0.4 |v| / sqrt(2)), right
    // to 1.6e-7 of it, and to 6e-7 (1.1e-7 rms) with its roundings: the gradients of weight
    // and bias are fp32, so activateFast's 4.2e-6, which has the same sign in many values,
    // would be seen in their sums.
    const float t = __builtin_amdgcn_rcpf(fmaf(0.282842712f, fabsf(v), 1.0f));
    float poly = fmaf(t, 0.025129477f, -0.0914449404f);
    poly = fmaf(t, poly, 0.0845342149f);
    poly = fmaf(t, poly, -0.00279735801f);
    poly = fmaf(t, poly, 0.0707130809f);
    poly = fmaf(t, poly, 0.084271567f);
    poly = fmaf(t, poly, 0.103921288f);
    poly = fmaf(t, poly, 0.112834802f);
    poly = fmaf(t, poly, 0.112837931f);
    const float e = __builtin_amdgcn_exp2f(v * v * (-0.5f * ACT_LOG2E));
    const float q = t * poly * e;
    return fmaf(v, e * 0.39894228040143268f, v < 0.0f ? q : 1.0f - q);
  }
}

struct NormBackArgs {
  const void* grad;
  int64_t gB, gP;
  const float* stats;
  void* out;
  int64_t oB, oP;
  float* gradWeight;
  float* gradBias;
  float2* sums;  // [item or slice][channels]: of u and u h
};

// u (the gradient behind the activation) and h (the normalised input) of VEC channels.
template<typename T, int ACT, int VEC>
__device__ __forceinline__ void backward(float (&u)[VEC], float (&h)[VEC], const Values<T>& x, const Values<T>& grad, const float (&mean)[VEC],
                                         const float (&rstd)[VEC], const float (&weight)[VEC], const float (&bias)[VEC]) {
#pragma unroll
  for(int j = 0; j < VEC; j++) {
    h[j] = (x.f[j] - mean[j]) * rstd[j];
    u[j] = grad.f[j] * slope<T, ACT>(fmaf(h[j], weight[j], bias[j]));
  }
}

// The gradient by the group's means a.x of u weight and a.y of u weight h.
__device__ __forceinline__ float backwardX(float u, float h, float weight, float rstd, float2 a) { return rstd * (fmaf(u, weight, -a.x) - h * a.y); }

// A thread's channels' constants.
template<int VEC>
struct BackChannels {
  float weight[VEC], bias[VEC], mean[VEC], rstd[VEC];
  __device__ __forceinline__ BackChannels(const NormArgs& a, const float* stats, int b, int c0, int nc) {
    loadFloats(weight, a.weight == nullptr ? nullptr : a.weight + c0, nc, 1.0f);
    loadFloats(bias, a.bias == nullptr ? nullptr : a.bias + c0, nc, 0.0f);
#pragma unroll
    for(int j = 0; j < VEC; j++) {
      const float* t = stats + 2 * ((int64_t)b * a.groups + min(c0 + j, a.channels - 1) / a.per);
      mean[j] = t[0];
      rstd[j] = t[1];
    }
  }
};

// ---------------------------------------------------------------------------
// An item's run of channels in a unit's registers, as in the forward pass: x as it came
// and u in fp32 (its slope is most of the work, and is computed once). sums has a row for
// each item. 128 x 361 x 384 bf16, mish: 40 us of 107 MB (2.7 TB/s), with 54% of the
// positions 34; vector instructions are 0.58 of the cycles.
template<typename T, int ACT, int NV>
__global__ __launch_bounds__(512, NV == 2 ? 4 : 3) void normBackSlabKernel(NormArgs a, NormBackArgs k, NormSlab s) {
  constexpr int VEC = 16 / (int)sizeof(T);
  extern __shared__ float2 lds[];
  const SlabThread<VEC> th(a, s);
  const int inRun = s.run / a.per;
  float2* part = lds + th.unit * s.ldsPairs;
  float2* means = part + s.ldsPairs - inRun;
  unsigned short* list = (unsigned short*)((char*)lds + s.listAt) + th.unit * (listBytes(a.positions) / 2);
  const T* x = (const T*)a.x + th.b * a.xB + th.at;
  const T* grad = (const T*)k.grad + th.b * k.gB + th.at;
  int count = validLength(a, th.b);
  if(a.mask != nullptr) count = listPositions(a, th.b, count, list);
  count = __builtin_amdgcn_readfirstlane(count);
  auto position = [&](int place) -> unsigned { return a.mask != nullptr ? list[place] : place; };
  u32x4_t v[NV], d[NV];
#pragma unroll
  for(int i = 0, from = 0; i < NV; i++, from += s.rowLanes)
    if(from < count) {
      const uint64_t p = position(min(th.row + from, a.positions - 1));
      __builtin_memcpy(&v[i], x + p * a.xP, 16);
      __builtin_memcpy(&d[i], grad + p * k.gP, 16);
    }
  float weight[VEC], bias[VEC], mean[VEC], rstd[VEC];
  loadFloats(weight, a.weight == nullptr ? nullptr : a.weight + th.at, VEC, 1.0f);
  loadFloats(bias, a.bias == nullptr ? nullptr : a.bias + th.at, VEC, 0.0f);
  const float* stats = k.stats + 2 * ((int64_t)th.b * a.groups + th.c1 / a.per);
  th.eachGroup(a, [&](int j, int q) {
    mean[j] = stats[2 * q];
    rstd[j] = stats[2 * q + 1];
  });
  float u[NV][VEC], s0[VEC], s1[VEC];
#pragma unroll
  for(int j = 0; j < VEC; j++) s0[j] = s1[j] = 0.0f;
#pragma unroll
  for(int i = 0; i < NV; i++)
    if(i * s.rowLanes < count) {
      float h[VEC];
      backward<T, ACT>(u[i], h, Values<T>(v[i]), Values<T>(d[i]), mean, rstd, weight, bias);
      if(th.row + i * s.rowLanes < count) {
#pragma unroll
        for(int j = 0; j < VEC; j++) {
          s0[j] += u[i][j];
          s1[j] = fmaf(u[i][j], h[j], s1[j]);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  if(th.on) {
    float2* p = part + th.row * s.entries + th.channel;
#pragma unroll
    for(int j = 0; j < VEC; j++)
      if(j >= th.skip) p[j - th.skip] = make_float2(s0[j], s1[j]);
  }
  __syncthreads();
  // The rows' sums in `segments` parts, which are kept for the weight's and bias's gradients.
  float2* red = part + s.rowLanes * s.entries;
  for(int i = th.tt; i < s.segments * s.entries; i += s.threads) {
    const int seg = i / s.entries, e = i - seg * s.entries;
    float2 t = make_float2(0.0f, 0.0f);
#pragma unroll 4
    for(int r = seg; r < s.rowLanes; r += s.segments) {
      const float2 w = part[r * s.entries + e];
      t.x += w.x;
      t.y += w.y;
    }
    red[i] = t;
  }
  __syncthreads();
  const float n = (float)count * (float)a.per;
  for(int q = th.tt >> s.lanesLog; q < th.groups; q += s.threads >> s.lanesLog) {
    float2 m = make_float2(0.0f, 0.0f);
    eachEntry(red, s, s.segments, q, th.tt, [&](float2 t, int e) {
      const float w = a.weight == nullptr ? 1.0f : a.weight[th.c1 + e];
      m.x = fmaf(t.x, w, m.x);
      m.y = fmaf(t.y, w, m.y);
    });
    m = addLanes(m, s.lanesLog);
    if((th.tt & ((1 << s.lanesLog) - 1)) == 0) means[q] = make_float2(m.x / n, m.y / n);
  }
  __syncthreads();
  float2 mean2[VEC];
  th.eachGroup(a, [&](int j, int q) { mean2[j] = means[q]; });
  T* out = (T*)k.out + th.b * k.oB + th.at;
  const bool stores = th.on && th.live;
  const int rowLanes = fresh(s.rowLanes);
#pragma unroll
  for(int i = 0, from = 0; i < NV; i++, from += rowLanes)
    if(from < a.positions) {
      const int place = th.row + from;
      uint4 w = make_uint4(0, 0, 0, 0);
      if(from < count) {
        renew(v[i]);
        const Values<T> xv(v[i]);
        float y[VEC];
#pragma unroll
        for(int j = 0; j < VEC; j++) y[j] = backwardX(u[i][j], (xv.f[j] - mean[j]) * rstd[j], weight[j], rstd[j], mean2[j]);
        w = packed<T>(y);
        if(from + rowLanes > count && place >= count) w = make_uint4(0, 0, 0, 0);
      }
      if(stores && place < a.positions) {
        T* p = out + (uint64_t)position(place) * k.oP;
        if(a.channels % VEC == 0) __builtin_memcpy(p, &w, 16);
        else storeWindow(p, w, th.skip);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  if(th.live)
    for(int e = th.tt; e < min(s.run, a.channels - th.c1); e += s.threads) {
      float2 t = red[e];
      for(int r = 1; r < s.segments; r++) {
        t.x += red[r * s.entries + e].x;
        t.y += red[r * s.entries + e].y;
      }
      k.sums[(int64_t)th.b * a.channels + th.c1 + e] = t;
    }
}

// ---------------------------------------------------------------------------
// Items that do not fit: chunks of positions and blocks of columns, each a workgroup.
// parts[item][chunk][channel]: sums of u and u h. counts[item][chunk]: positions that
// take part.
struct BackParts {
  float2* parts;
  int* counts;
  float2* means;  // [item][group]
  int chunks, chunkRows, blocks, cols, rowLanes, segments;
};

constexpr int BACK_AHEAD = 2;  // rows of a thread under way

// Items that no workgroup's registers hold: first the sums of chunks of positions, then,
// behind their join, the results of the same chunks, u computed in both (kept, it would be
// as many bytes again as x in fp32, twice as many in 16 bits). 8 x 4096 x 320 fp32, SiLU:
// 26 us (3.2 TB/s) and 25 (5.0), the joins 9 and 5.
template<typename T, int ACT, bool APPLY>
__global__ __launch_bounds__(256) void normBackPartsKernel(NormArgs a, NormBackArgs k, BackParts s) {
  constexpr int VEC = 16 / (int)sizeof(T);
  __shared__ float2 part[APPLY ? 1 : 256 * VEC];
  __shared__ int counted;
  const int row = threadIdx.x / s.cols, col = threadIdx.x - row * s.cols;
  const int64_t all = (int64_t)a.batch * s.chunks * s.blocks;
  for(int64_t id = blockIdx.x; id < all; id += gridDim.x) {
    const int64_t itemChunk = id / s.blocks;
    const int block = (int)(id - itemChunk * s.blocks);
    const int b = (int)(itemChunk / s.chunks), chunk = (int)(itemChunk - (int64_t)b * s.chunks);
    const int from = block * s.cols * VEC;
    const int c0 = from + col * VEC, nc = min(a.channels - c0, VEC);
    const bool on = row < s.rowLanes && nc > 0;
    const int len = validLength(a, b);
    const int p0 = chunk * s.chunkRows, p1 = min(p0 + s.chunkRows, a.positions);
    const RowGroup<T, false> g((on ? c0 : 0) / VEC, a.channels);
    const T* x = (const T*)a.x + b * a.xB;
    const T* grad = (const T*)k.grad + b * k.gB;
    const uint8_t* mask = a.mask == nullptr ? nullptr : a.mask + b * a.maskB;
    const BackChannels<VEC> ch(a, k.stats, b, min(c0, a.channels - 1), nc);
    float s0[VEC], s1[VEC];
    float2 mean2[VEC];
#pragma unroll
    for(int j = 0; j < VEC; j++) {
      s0[j] = s1[j] = 0.0f;
      mean2[j] = APPLY ? s.means[(int64_t)b * a.groups + min(c0 + j, a.channels - 1) / a.per] : make_float2(0.0f, 0.0f);
    }
    if(!APPLY) {
      if(threadIdx.x == 0) counted = 0;
      __syncthreads();
    }
    int rows = 0;
    if(on) {
      for(int p = p0 + row; p < p1; p += BACK_AHEAD * s.rowLanes) {
        u32x4_t v[BACK_AHEAD], d[BACK_AHEAD];
        bool take[BACK_AHEAD];
#pragma unroll
        for(int i = 0; i < BACK_AHEAD; i++) {
          const int q = p + i * s.rowLanes;
          take[i] = q < p1 && q < len && (mask == nullptr || mask[q] != 0);
        }
#pragma unroll
        for(int i = 0; i < BACK_AHEAD; i++) {
          const int64_t q = take[i] ? p + i * s.rowLanes : 0;
          v[i] = g.load(x + q * a.xP);
          d[i] = g.load(grad + q * k.gP);
        }
#pragma unroll
        for(int i = 0; i < BACK_AHEAD; i++) {
          float u[VEC], h[VEC];
          backward<T, ACT>(u, h, Values<T>(g.place(v[i])), Values<T>(g.place(d[i])), ch.mean, ch.rstd, ch.weight, ch.bias);
          if constexpr(APPLY) {
            const int q = p + i * s.rowLanes;
            float y[VEC];
#pragma unroll
            for(int j = 0; j < VEC; j++) y[j] = backwardX(u[j], h[j], ch.weight[j], ch.rstd[j], mean2[j]);
            const uint4 o = packed<T>(y), zero = make_uint4(0, 0, 0, 0);
            if(q < p1) storeGroup((T*)k.out + b * k.oB + q * k.oP + c0, take[i] ? o : zero, nc);
          }
          else if(take[i]) {
            rows++;
#pragma unroll
            for(int j = 0; j < VEC; j++) {
              s0[j] += u[j];
              s1[j] = fmaf(u[j], h[j], s1[j]);
            }
          }
        }
      }
    }
    if constexpr(!APPLY) {
      if(col == 0 && rows > 0) atomicAdd(&counted, rows);
      if(row < s.rowLanes) {
#pragma unroll
        for(int j = 0; j < VEC; j++) part[(row * s.cols + col) * VEC + j] = make_float2(s0[j], s1[j]);
      }
      __syncthreads();
      const int width = s.cols * VEC;
      for(int e = threadIdx.x; e < min(width, a.channels - from); e += 256) {
        double2 t = make_double2(0.0, 0.0);  // rows of threads may be 256
        for(int q = 0; q < s.rowLanes; q++) {
          t.x += part[q * width + e].x;
          t.y += part[q * width + e].y;
        }
        s.parts[itemChunk * a.channels + from + e] = make_float2((float)t.x, (float)t.y);
      }
      if(threadIdx.x == 0 && block == 0) s.counts[itemChunk] = counted;
      __syncthreads();
    }
  }
}

// Many items of few positions, a thread one: a workgroup has a run of channels of every
// `slices`-th item, and its channels' sums in registers all the while; sums has a row for
// each slice (a row for each item would be more bytes than the tensors). 8192 x 4096 bf16:
// 71 us (2.8 TB/s); an item's way through three barriers bounds it, beside that of the
// CU's other workgroup: 128 registers a thread leave room for two of 512 threads.
template<typename T, int ACT>
__global__ __launch_bounds__(1024) void normBackItemsKernel(NormArgs a, NormBackArgs k, NormSlab s, int slices) {
  constexpr int VEC = 16 / (int)sizeof(T);
  extern __shared__ float2 lds[];
  const int run = blockIdx.x % s.runs, slice = blockIdx.x / s.runs;
  const int row = threadIdx.x / s.cols, col = threadIdx.x - row * s.cols;
  const int c1 = run * s.run, channel = col * VEC;
  const int groups = min(s.run / a.per, a.groups - c1 / a.per);
  const bool on = row < s.rowLanes && channel < min(s.run, a.channels - c1);
  const Window<VEC> win(c1 + channel, a.channels);
  float2* part = lds;
  float2* means = part + s.ldsPairs - s.run / a.per;
  float weight[VEC], bias[VEC], all0[VEC], all1[VEC];
  unsigned pair[VEC / 2];  // channels' groups, 16 bits each: registers are what a second workgroup a CU wants
  loadFloats(weight, a.weight == nullptr ? nullptr : a.weight + win.at, VEC, 1.0f);
  loadFloats(bias, a.bias == nullptr ? nullptr : a.bias + win.at, VEC, 0.0f);
#pragma unroll
  for(int j = 0; j < VEC; j++) {
    all0[j] = all1[j] = 0.0f;
    const unsigned q = min((channel + max(j - win.skip, 0)) / a.per, groups - 1);
    pair[j / 2] = j & 1 ? pair[j / 2] | q << 16 : q;
  }
  const auto group = [&](int j) { return j & 1 ? pair[j / 2] >> 16 : pair[j / 2] & 0xffff; };
  for(int b = slice; b < a.batch; b += slices) {
#pragma unroll
    for(int i = 0; i < VEC / 2; i++) asm volatile("" : "+v"(pair[i]));  // (else they are taken apart before the loop)
    const int len = validLength(a, b);
    const T* x = (const T*)a.x + b * a.xB + win.at;
    const T* grad = (const T*)k.grad + b * k.gB + win.at;
    int count = len;
    if(a.mask != nullptr) {
      count = 0;
      for(int p = 0; p < len; p++) count += a.mask[b * a.maskB + p] != 0 ? 1 : 0;
    }
    const int p = min(row, a.positions - 1);
    const bool take = row < len && (a.mask == nullptr || a.mask[b * a.maskB + p] != 0);
    u32x4_t v, d;
    __builtin_memcpy(&v, x + (uint64_t)(unsigned)p * a.xP, 16);
    __builtin_memcpy(&d, grad + (uint64_t)(unsigned)p * k.gP, 16);
    const float* stats = k.stats + 2 * ((int64_t)b * a.groups + c1 / a.per);
    float mean[VEC], rstd[VEC], u[VEC], h[VEC];
#pragma unroll
    for(int j = 0; j < VEC; j++) {
      const float2 t = ((const float2*)stats)[group(j)];
      mean[j] = t.x;
      rstd[j] = t.y;
    }
    backward<T, ACT>(u, h, Values<T>(v), Values<T>(d), mean, rstd, weight, bias);
    __builtin_amdgcn_sched_barrier(0);
    __syncthreads();  // the item before has read its means
    float2 m = make_float2(0.0f, 0.0f);
#pragma unroll
    for(int j = 0; j < VEC; j++) {
      const float s0 = take ? u[j] : 0.0f, s1 = take ? u[j] * h[j] : 0.0f;
      all0[j] += s0;
      all1[j] += s1;
      if(s.pv == 1) {
        m.x = fmaf(s0, weight[j], m.x);
        m.y = fmaf(s1, weight[j], m.y);
      }
      else if(on && j >= win.skip) part[row * s.entries + channel + j - win.skip] = make_float2(s0 * weight[j], s1 * weight[j]);
    }
    if(s.pv == 1 && on) part[row * s.entries + col] = m;
    __syncthreads();
    const float n = (float)count * (float)a.per;
    const int lanes = 1 << s.lanesLog, sub = threadIdx.x & (lanes - 1);
    for(int q = threadIdx.x >> s.lanesLog; q < groups; q += s.threads >> s.lanesLog) {
      float2 t = make_float2(0.0f, 0.0f);
      eachEntry(part, s, s.rowLanes, q, threadIdx.x, [&](float2 w, int) {
        t.x += w.x;
        t.y += w.y;
      });
      t = addLanes(t, s.lanesLog);
      if(sub == 0) means[q] = make_float2(t.x / n, t.y / n);
    }
    __syncthreads();
    T* out = (T*)k.out + b * k.oB + win.at;
    float y[VEC];
#pragma unroll
    for(int j = 0; j < VEC; j++) y[j] = take ? backwardX(u[j], h[j], weight[j], rstd[j], means[group(j)]) : 0.0f;
    if(on && row < a.positions) storeWindow(out + (uint64_t)(unsigned)row * k.oP, packed<T>(y), win.skip);
  }
  // The channels' sums over the rows of threads.
  for(int turn = 0; turn < s.rowLanes; turn++) {
    __syncthreads();
    if(row == turn && on) {
#pragma unroll
      for(int j = 0; j < VEC; j++)
        if(j >= win.skip) {
          float2& t = k.sums[(int64_t)slice * a.channels + c1 + channel + j - win.skip];
          if(turn == 0) t = make_float2(all0[j], all1[j]);
          else {
            t.x += all0[j];
            t.y += all1[j];
          }
        }
    }
  }
}

// The chunks' sums of an item's group: its channels' sums and its means, in 64 bits
// (chunks may be thousands, and roundings of terms of one sign add up: 262144 positions of
// 1024 channels that are all the same were 7e-6 off in fp32). Threads are (chunk slice,
// channel); channels of long groups in turns.
__global__ __launch_bounds__(256) void normBackJoinKernel(NormArgs a, NormBackArgs k, BackParts s) {
  __shared__ double2 part[256];
  __shared__ double2 total[4];
  __shared__ int counted;
  const int width = min(a.per, 64), slices = 256 / width;
  const int slice = threadIdx.x / width, c = threadIdx.x - slice * width;
  for(int64_t i = blockIdx.x; i < (int64_t)a.batch * a.groups; i += gridDim.x) {
    const int b = (int)(i / a.groups), g = (int)(i - (int64_t)b * a.groups);
    if(threadIdx.x == 0) counted = 0;
    __syncthreads();
    int rows = 0;
    for(int q = threadIdx.x; q < s.chunks; q += 256) rows += s.counts[(int64_t)b * s.chunks + q];
    if(rows > 0) atomicAdd(&counted, rows);
    double m1 = 0.0, m2 = 0.0;
    for(int from = 0; from < a.per; from += width) {
      const bool on = slice < slices && from + c < a.per;
      const int ch = g * a.per + from + c;
      double2 t = make_double2(0.0, 0.0);
      if(on)
#pragma unroll 8
        for(int q = slice; q < s.chunks; q += slices) {
          const float2 v = s.parts[((int64_t)b * s.chunks + q) * a.channels + ch];
          t.x += v.x;
          t.y += v.y;
        }
      part[threadIdx.x] = t;
      __syncthreads();
      if(slice == 0 && on) {
        for(int q = 1; q < slices; q++) {
          t.x += part[q * width + c].x;
          t.y += part[q * width + c].y;
        }
        k.sums[(int64_t)b * a.channels + ch] = make_float2((float)t.x, (float)t.y);
        const double w = a.weight == nullptr ? 1.0 : a.weight[ch];
        m1 = fma(t.x, w, m1);
        m2 = fma(t.y, w, m2);
      }
      __syncthreads();
    }
#pragma unroll
    for(int w = 32; w > 0; w >>= 1) {
      m1 += __shfl_xor(m1, w);
      m2 += __shfl_xor(m2, w);
    }
    if((threadIdx.x & 63) == 0) total[threadIdx.x >> 6] = make_double2(m1, m2);
    __syncthreads();
    if(threadIdx.x == 0) {
      const double n = (double)counted * a.per;
      s.means[i] = make_float2((float)(((total[0].x + total[1].x) + (total[2].x + total[3].x)) / n), (float)(((total[0].y + total[1].y) + (total[2].y + total[3].y)) / n));
    }
    __syncthreads();
  }
}

// The items' (or slices') sums: the gradients of weight and bias. 32 channels a workgroup;
// rows may be many, so in 64 bits.
__global__ __launch_bounds__(1024) void normBackWeightsKernel(NormBackArgs k, int channels, int rows) {
  __shared__ double2 part[1024];
  const int c = blockIdx.x * 32 + (threadIdx.x & 31), slice = threadIdx.x >> 5;
  double2 t = make_double2(0.0, 0.0);
  if(c < channels)
#pragma unroll 8
    for(int b = slice; b < rows; b += 32) {
      const float2 v = k.sums[(int64_t)b * channels + c];
      t.x += v.x;
      t.y += v.y;
    }
  part[threadIdx.x] = t;
  __syncthreads();
  if(slice != 0 || c >= channels) return;
#pragma unroll 8
  for(int q = 1; q < 32; q++) {
    t.x += part[q * 32 + threadIdx.x].x;
    t.y += part[q * 32 + threadIdx.x].y;
  }
  if(k.gradBias != nullptr) k.gradBias[c] = (float)t.x;
  if(k.gradWeight != nullptr) k.gradWeight[c] = (float)t.y;
}

struct NormBackPlan {
  NormSlab slab;  // threads 0: parts
  int slices;     // 0: a row of sums for each item
  BackParts parts;
  uint64_t sumsBytes, partsBytes, countsBytes, meansBytes;
};

NormBackPlan planBackward(const kgh_group_norm_backward_params& p) {
  const int size = (int)kgh::opElemBytes(p.dtype), vec = 16 / size;
  const auto round16 = [](uint64_t n) { return (n + 15) / 16 * 16; };
  NormBackPlan plan{};
  // Few positions an item: us with a row of sums for each item and with one for a slice
  // (bf16) 8192 x 1 x 4096 600 and 75, 64 x 1 x 4096 54 and 12, 1024 x 1 x 384 15 and 12,
  // 1 x 1 x 384 9.2 and 7.2, 4096 x 2 x 256 70 and 21, 1024 x 4 x 384 29 and 20; but
  // 256 x 4 x 1024 14 and 19, 1024 x 8 x 384 29 and 64.
  if(p.positions == 1 || (p.positions <= 4 && p.batch >= 1024)) {
    plan.slab = planSlab(p.positions, p.channels, p.groups, size, 1024, false, 1, 1024, false, 1);
    if(plan.slab.threads != 0) {
      // Slices that fill the card: of 512 threads two a CU (8192 x 1 x 4096 SiLU: 256 slices
      // 114 us, one workgroup a CU; 512 82), of few threads more (8192 x 1 x 384: 512 38 us,
      // 1024 27). Of two items at least where there are many (512 x 1 x 4096: 27 us with one,
      // 20 with two; 64 x 1 x 4096: 12 and 13.5), of at most 64, sums' terms one after the
      // other (the launch's threads are counted in 32 bits: room for more bytes of items
      // than the card holds).
      const int64_t room = std::min(1024, 262144 / plan.slab.threads) / plan.slab.runs;
      const int64_t most = std::max<int64_t>(1, ((int64_t)1 << 31) / ((int64_t)plan.slab.threads * plan.slab.runs));
      plan.slices = (int)std::min(most, std::max<int64_t>({1, std::min<int64_t>(room, p.batch <= 256 ? p.batch : p.batch / 2), ((int64_t)p.batch + 63) / 64}));
      plan.sumsBytes = round16((uint64_t)plan.slices * p.channels * 8);
      return plan;
    }
  }
  plan.sumsBytes = round16((uint64_t)p.batch * p.channels * 8);
  const auto slab = [&](int bytes, int most, int wide) {
    if(plan.slab.threads == 0) plan.slab = planSlab(p.positions, p.channels, p.groups, size, bytes, true, most, wide, false, 1);
  };
  // us of 128 x 361 x 384 bf16 in 32 groups: runs of 48 bytes 45, of 96 53, in parts 61.
  slab(48, 6, 256);
  slab(48, 6, 512);
  slab(16, 6, 512);
  if(plan.slab.threads != 0) return plan;
  BackParts& s = plan.parts;
  const int cols = (p.channels + vec - 1) / vec;
  s.cols = std::min(cols, 256);
  s.blocks = (cols + s.cols - 1) / s.cols;
  s.rowLanes = std::min(256 / s.cols, p.positions);
  const int64_t rows = std::max<int64_t>(1, std::min<int64_t>(64, (int64_t)p.batch * p.positions * s.blocks / s.rowLanes / 1024));
  s.chunkRows = (int)std::min<int64_t>(p.positions, (rows + BACK_AHEAD - 1) / BACK_AHEAD * BACK_AHEAD * s.rowLanes);
  s.chunks = (p.positions + s.chunkRows - 1) / s.chunkRows;
  plan.partsBytes = round16((uint64_t)p.batch * s.chunks * p.channels * 8);
  plan.countsBytes = round16((uint64_t)p.batch * s.chunks * 4);
  plan.meansBytes = round16((uint64_t)p.batch * p.groups * 8);
  return plan;
}

template<typename T, int ACT>
void launchBackward(const NormBackPlan& plan, const NormArgs& a, const NormBackArgs& k, hipStream_t stream) {
  if(plan.slices > 0) {
    const NormSlab& s = plan.slab;
    normBackItemsKernel<T, ACT><<<(unsigned)(plan.slices * s.runs), (unsigned)s.threads, (size_t)s.ldsPairs * 8, stream>>>(a, k, s, plan.slices);
    KGH_CHECK_LAUNCH();
    return;
  }
  if(plan.slab.threads != 0) {
    forUnits(a, plan.slab, [&](const NormSlab& s, unsigned grid, unsigned threads, size_t bytes) {
      if(s.nv <= 2) normBackSlabKernel<T, ACT, 2><<<grid, threads, bytes, stream>>>(a, k, s);
      else if(s.nv <= 4) normBackSlabKernel<T, ACT, 4><<<grid, threads, bytes, stream>>>(a, k, s);
      else normBackSlabKernel<T, ACT, 6><<<grid, threads, bytes, stream>>>(a, k, s);
      KGH_CHECK_LAUNCH();
    });
    return;
  }
  BackParts parts = plan.parts;
  char* at = (char*)k.sums + plan.sumsBytes;
  parts.parts = (float2*)at;
  parts.counts = (int*)(at + plan.partsBytes);
  parts.means = (float2*)(at + plan.partsBytes + plan.countsBytes);
  const unsigned grid = normGrid((int64_t)a.batch * parts.chunks * parts.blocks);
  normBackPartsKernel<T, ACT, false><<<grid, 256, 0, stream>>>(a, k, parts);
  KGH_CHECK_LAUNCH();
  normBackJoinKernel<<<normGrid((int64_t)a.batch * a.groups), 256, 0, stream>>>(a, k, parts);
  KGH_CHECK_LAUNCH();
  normBackPartsKernel<T, ACT, true><<<grid, 256, 0, stream>>>(a, k, parts);
  KGH_CHECK_LAUNCH();
}

}  // namespace

namespace kgh {

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
  checkApartFrom(op, "grad_x", p.grad_x, {{"statistics", p.statistics}, {"weight", p.weight}, {"bias", p.bias}, {"lengths", p.lengths}, {"mask", p.mask}});
  for(const auto& out : {std::make_pair("grad_weight", p.grad_weight), std::make_pair("grad_bias", p.grad_bias)})
    checkApartFrom(op, out.first, out.second, {{"x", p.x}, {"grad_out", p.grad_out}, {"grad_x", p.grad_x}, {"statistics", p.statistics}, {"weight", p.weight}, {"bias", p.bias},
                                               {"lengths", p.lengths}, {"mask", p.mask}});
  opCheckWorkspace(op, p.workspace, p.workspace_bytes, groupNormBackwardWorkspace(p));
}

uint64_t groupNormBackwardWorkspace(const kgh_group_norm_backward_params& p) {
  if(p.batch == 0 || p.positions == 0) return 0;
  const NormBackPlan plan = planBackward(p);
  return plan.sumsBytes + plan.partsBytes + plan.countsBytes + plan.meansBytes;
}

void launchGroupNormBackward(const kgh_group_norm_backward_params& p, hipStream_t stream) {
  const NormArgs a = normArgs(p, 0.0f);
  const NormBackArgs k{p.grad_out, p.grad_out_batch_stride, p.grad_out_position_stride, p.statistics, p.grad_x, p.grad_x_batch_stride,
                       p.grad_x_position_stride, p.grad_weight, p.grad_bias, (float2*)p.workspace};
  int rows = 0;  // of sums; without any the gradients of weight and bias are zeros
  if(p.batch > 0 && p.positions > 0) {
    const NormBackPlan plan = planBackward(p);
    rows = plan.slices > 0 ? plan.slices : p.batch;
    withDtype(p.dtype, [&](auto t) {
      withActivation(p.activation, [&](auto act) { launchBackward<decltype(t), decltype(act)::value>(plan, a, k, stream); });
    });
  }
  if(p.grad_weight == nullptr && p.grad_bias == nullptr) return;
  normBackWeightsKernel<<<dim3((unsigned)((p.channels + 31) / 32)), 1024, 0, stream>>>(k, p.channels, rows);
  KGH_CHECK_LAUNCH();
}

}  // namespace kgh
