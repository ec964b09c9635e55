// Rotary positions with several axes (kgh_rope_axes).
#include "kgh_ops_device.h"

#include <algorithm>

namespace {

constexpr int64_t ROPE_MAX_TOKENS = (int64_t)1 << 32;

struct RopeArgs {
  const void* x;
  void* out;
  const int32_t* positions;
  const float* freqs;
  int64_t xToken, xHead, outToken, outHead, ldPos;
  int64_t items;  // tokens x head runs x groups
  int heads, dim, pairs, axes, tables, headRun, headRuns, groups, pairGroups;
  float sign;
};

// Sine and cosine of an angle given in turns, |turns| <= 1/2. The hardware's own
// functions take turns; their error of about 1e-6 is below 16 bits' rounding.
template<typename T>
__device__ __forceinline__ void sinCosTurns(float turns, float& s, float& c) {
  if constexpr(sizeof(T) == 4) sincospif(2.0f * turns, &s, &c);
  else {
    s = __builtin_amdgcn_sinf(turns);
    c = __builtin_amdgcn_cosf(turns);
  }
}

// A thread takes VEC pairs (two 16-byte groups) of a token, or as many of the
// channels behind the pairs, and a run of heads that share a table: the angles
// are computed once for the run, whose rows are loaded ROPE_AHEAD heads at a time.
// Bound by the tensor's way in and out of memory where a run has four heads and
// more, else by the angles (about 130 cycles for 64 pairs).
constexpr int ROPE_AHEAD = 4;

template<typename T, bool HALVES, int AXES>
__global__ __launch_bounds__(256) void ropeAxesKernel(RopeArgs a) {
  constexpr int VEC = 16 / (int)sizeof(T);
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if(id >= a.items) return;
  const int64_t rest = id / a.groups;
  const int group = (int)(id - rest * a.groups);
  const int64_t token = rest / a.headRuns;
  const int h0 = (int)(rest - token * a.headRuns) * a.headRun;
  const bool turns = group < a.pairGroups;
  // The two groups' first channels, and their lengths.
  int c0, c1, n0, n1;
  float cs[VEC], sn[VEC];
  if(turns) {
    const int p0 = group * VEC;
    const int np = min(VEC, a.pairs - p0);
    if(HALVES) {
      c0 = p0;
      c1 = a.pairs + p0;
      n0 = n1 = np;
    }
    else {
      c0 = 2 * p0;
      c1 = c0 + VEC;
      n0 = min(VEC, 2 * np);
      n1 = 2 * np - n0;
    }
    const int table = h0 / (a.heads / a.tables);
    const float* src = a.freqs + ((int64_t)table * a.pairs + p0) * AXES;
    float f[VEC * AXES];
    if(np == VEC) __builtin_memcpy(f, src, sizeof(f));
    else {
#pragma unroll
      for(int j = 0; j < VEC * AXES; j++) f[j] = j < np * AXES ? src[j] : 0.0f;
    }
    double pos[AXES];
#pragma unroll
    for(int x = 0; x < AXES; x++) pos[x] = (double)a.positions[token * a.ldPos + x];
#pragma unroll
    for(int j = 0; j < VEC; j++) {
      double angle = 0.0;
#pragma unroll
      for(int x = 0; x < AXES; x++) angle = fma(pos[x], (double)f[j * AXES + x], angle);
      // Far positions turn many times: whole turns are taken off in 64 bits.
      const double t = angle * 0.15915494309189533577;
      sinCosTurns<T>((float)(t - rint(t)), sn[j], cs[j]);
      sn[j] *= a.sign;
    }
  }
  else {
    c0 = 2 * a.pairs + (group - a.pairGroups) * 2 * VEC;
    c1 = c0 + VEC;
    n0 = min(VEC, a.dim - c0);
    n1 = min(VEC, max(0, a.dim - c1));
  }
  const T* src = (const T*)a.x + token * a.xToken;
  T* dst = (T*)a.out + token * a.outToken;
  union Group {
    u32x4_t v;
    T e[VEC];
  };
  auto turn = [&](Group& u0, Group& u1) {
#pragma unroll
    for(int j = 0; j < VEC; j++) {
      T& e0 = HALVES ? u0.e[j] : (2 * j < VEC ? u0.e[(2 * j) % VEC] : u1.e[(2 * j) % VEC]);
      T& e1 = HALVES ? u1.e[j] : (2 * j < VEC ? u0.e[(2 * j + 1) % VEC] : u1.e[(2 * j + 1) % VEC]);
      float y0, y1;
      kgh_rope_pair((float)e0, (float)e1, cs[j], sn[j], y0, y1);
      e0 = (T)y0;
      e1 = (T)y1;
    }
  };
  const int h1 = min(h0 + a.headRun, a.heads);
  if(n0 == VEC && n1 == VEC) {
    for(int h = h0; h < h1; h += ROPE_AHEAD) {
      Group u[ROPE_AHEAD][2];
#pragma unroll
      for(int i = 0; i < ROPE_AHEAD; i++) {
        const T* row = src + min(h + i, h1 - 1) * a.xHead;
        __builtin_memcpy(&u[i][0].v, row + c0, 16);
        __builtin_memcpy(&u[i][1].v, row + c1, 16);
      }
#pragma unroll
      for(int i = 0; i < ROPE_AHEAD; i++) {
        if(h + i >= h1) break;
        T* row = dst + (h + i) * a.outHead;
        if(turns) turn(u[i][0], u[i][1]);
        __builtin_memcpy(row + c0, &u[i][0].v, 16);
        __builtin_memcpy(row + c1, &u[i][1].v, 16);
      }
    }
    return;
  }
  for(int h = h0; h < h1; h++) {
    Group u0, u1;
    const uint4 v0 = loadGroupSmall(src + h * a.xHead + c0, n0), v1 = loadGroupSmall(src + h * a.xHead + c1, n1);
    u0.v = u32x4_t{v0.x, v0.y, v0.z, v0.w};
    u1.v = u32x4_t{v1.x, v1.y, v1.z, v1.w};
    if(turns) turn(u0, u1);
    storeGroup(dst + h * a.outHead + c0, make_uint4(u0.v.x, u0.v.y, u0.v.z, u0.v.w), n0);
    storeGroup(dst + h * a.outHead + c1, make_uint4(u1.v.x, u1.v.y, u1.v.z, u1.v.w), n1);
  }
}

template<typename T, bool HALVES>
void launchAxes(const RopeArgs& a, int64_t blocks, hipStream_t stream) {
  const dim3 grid((unsigned)blocks);
  if(a.axes == 1) ropeAxesKernel<T, HALVES, 1><<<grid, 256, 0, stream>>>(a);
  else if(a.axes == 2) ropeAxesKernel<T, HALVES, 2><<<grid, 256, 0, stream>>>(a);
  else if(a.axes == 3) ropeAxesKernel<T, HALVES, 3><<<grid, 256, 0, stream>>>(a);
  else ropeAxesKernel<T, HALVES, 4><<<grid, 256, 0, stream>>>(a);
}

}  // namespace

namespace kgh {

void checkRope(const kgh_rope_params& p) {
  const char* op = "kgh_rope_axes";
  opCheckDtype(op, p.dtype);
  if(p.layout != KGH_ROPE_INTERLEAVED && p.layout != KGH_ROPE_HALVES) opInvalid(op, "layout " + std::to_string(p.layout) + " is none of KGH_ROPE_*");
  if(p.axes < 1 || p.axes > KGH_ROPE_MAX_AXES) opInvalid(op, "axes " + std::to_string(p.axes) + " outside 1.." + std::to_string(KGH_ROPE_MAX_AXES));
  if(p.tokens < 0 || p.tokens > ROPE_MAX_TOKENS) opInvalid(op, "tokens " + std::to_string(p.tokens) + " outside 0.." + std::to_string(ROPE_MAX_TOKENS));
  if(p.heads < 1 || p.head_dim < 1 || p.pairs < 1 || p.head_dim > (1 << 20)) opInvalid(op, "heads, head_dim and pairs must be positive (head_dim at most 2^20)");
  if(2 * (int64_t)p.pairs > p.head_dim) opInvalid(op, "a head of " + std::to_string(p.head_dim) + " channels has no " + std::to_string(p.pairs) + " pairs");
  // A launch takes 2^32 groups of channels; so many are no tensor either.
  if((double)p.tokens * p.heads * p.head_dim > 1099511627776.0) opInvalid(op, "too many tokens for one call");
  if(p.tables < 1 || p.heads % p.tables != 0) opInvalid(op, "tables must divide heads");
  if(p.x_token_stride < 0 || p.x_head_stride < 0 || p.positions_stride < 0) opInvalid(op, "negative stride");
  if(p.tokens == 0) return;
  // Rows of the output lie apart: heads inside a token or tokens inside a head.
  const int64_t ht = p.out_head_stride, tt = p.out_token_stride;
  const bool headsInside = (p.heads == 1 || ht >= p.head_dim) && (p.tokens == 1 || tt >= (p.heads - 1) * ht + p.head_dim);
  const bool tokensInside = (p.tokens == 1 || tt >= p.head_dim) && (p.heads == 1 || ht >= (p.tokens - 1) * tt + p.head_dim);
  if(ht < 0 || tt < 0 || (!headsInside && !tokensInside)) opInvalid(op, "the output's strides make its rows overlap");
  const size_t e = opElemBytes(p.dtype);
  opCheckPointer(op, "x", p.x, e);
  opCheckPointer(op, "out", p.out, e);
  opCheckPointer(op, "positions", p.positions, 4);
  opCheckPointer(op, "freqs", p.freqs, 4);
  if(p.x == p.out && p.tokens > 1 && p.x_token_stride != tt) opInvalid(op, "in place, the strides must be the same");
  if(p.x == p.out && p.heads > 1 && p.x_head_stride != ht) opInvalid(op, "in place, the strides must be the same");
}

void launchRope(const kgh_rope_params& p, hipStream_t stream) {
  if(p.tokens == 0) return;
  const int vec = 16 / (int)opElemBytes(p.dtype);
  RopeArgs a{};
  a.x = p.x;
  a.out = p.out;
  a.positions = p.positions;
  a.freqs = p.freqs;
  a.xToken = p.x_token_stride;
  a.xHead = p.x_head_stride;
  a.outToken = p.out_token_stride;
  a.outHead = p.out_head_stride;
  a.ldPos = p.positions_stride;
  a.heads = p.heads;
  a.dim = p.head_dim;
  a.pairs = p.pairs;
  a.axes = p.axes;
  a.tables = p.tables;
  a.sign = p.inverse ? -1.0f : 1.0f;
  a.pairGroups = (p.pairs + vec - 1) / vec;
  a.groups = a.pairGroups + (p.head_dim - 2 * p.pairs + 2 * vec - 1) / (2 * vec);
  // Runs of up to 4 heads of a table, as long as the threads still fill the CUs:
  // 20011 tokens of 32 x 128 bf16, three axes: 72 us with runs of one head, 57 of
  // two, 58 of four, 66 of sixteen; 46208 x 12 x 64 fp16 with a table for two heads
  // 31 and 26 (5.5 TB/s).
  const int shared = p.heads / p.tables;
  a.headRun = 1;
  while(a.headRun < 4 && shared % (2 * a.headRun) == 0 && p.tokens * (p.heads / (2 * a.headRun)) * a.groups >= (1 << 18)) a.headRun *= 2;
  a.headRuns = p.heads / a.headRun;
  a.items = p.tokens * a.headRuns * a.groups;
  const int64_t blocks = (a.items + 255) / 256;
  // The launch counts threads in 32 bits.
  if(blocks >= (1 << 24)) opInvalid("kgh_rope_axes", "too many tokens for one call");
  withDtype(p.dtype, [&](auto t) {
    typedef decltype(t) T;
    if(p.layout == KGH_ROPE_HALVES) launchAxes<T, true>(a, blocks, stream);
    else launchAxes<T, false>(a, blocks, stream);
  });
  KGH_CHECK_LAUNCH();
}

}  // namespace kgh
