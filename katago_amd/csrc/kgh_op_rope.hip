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
  int64_t tokens, items;  // items: token runs x head runs x groups
  int heads, dim, pairs, axes, tables, tokenRun, headRun, headRuns, groups, pairGroups;
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

// The first n elements of v (n may be none), in as few stores as they have bits.
template<typename T>
__device__ __forceinline__ void storeParts(T* p, u32x4_t v, int n) {
  constexpr int VEC = 16 / (int)sizeof(T);
  if(n >= VEC) {
    __builtin_memcpy(p, &v, 16);
    return;
  }
  if(n >= VEC / 2) {
    const uint2 u = make_uint2(v.x, v.y);
    __builtin_memcpy(p, &u, 8);
    p += VEC / 2;
    n -= VEC / 2;
    v.x = v.z;
    v.y = v.w;
  }
  if(n >= VEC / 4) {
    const unsigned u = v.x;
    __builtin_memcpy(p, &u, 4);
    p += VEC / 4;
    n -= VEC / 4;
    v.x = v.y;
  }
  if(sizeof(T) == 2 && n > 0) {
    const unsigned short u = (unsigned short)v.x;
    __builtin_memcpy(p, &u, 2);
  }
}

// A thread takes VEC pairs (two 16-byte groups) of a token, or as many of the
// channels behind the pairs, and a run of heads that share a table: the angles
// are computed once for the run, whose rows are loaded ROPE_AHEAD heads at a time.
// Or (TOKENS) it takes them of a run of up to ROPE_AHEAD tokens of one head, for
// which the frequencies are loaded once.
// Bound by the tensor's way in and out of memory where a run has four heads and
// more, else by the angles (about 130 cycles for 64 pairs).
constexpr int ROPE_AHEAD = 4;

template<typename T, bool HALVES, int AXES, bool TOKENS>
__global__ __launch_bounds__(256) void ropeAxesKernel(RopeArgs a) {
  constexpr int VEC = 16 / (int)sizeof(T);
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if(id >= a.items) return;
  const int64_t rest = id / a.groups;
  const int group = (int)(id - rest * a.groups);
  const int64_t tokens = rest / a.headRuns, token = TOKENS ? tokens * a.tokenRun : tokens;
  const int h0 = (int)(rest - tokens * a.headRuns) * a.headRun;
  const bool turns = group < a.pairGroups;
  // The two groups' first channels, and their lengths.
  int c0, c1, n0, n1;
  float f[VEC * AXES], cs[VEC], sn[VEC];
  struct Position {
    int at[AXES];
  };
  auto position = [&](int64_t t, Position& p) {
#pragma unroll
    for(int x = 0; x < AXES; x++) p.at[x] = a.positions[t * a.ldPos + x];
  };
  auto angles = [&](const Position& p) {
    double pos[AXES];
#pragma unroll
    for(int x = 0; x < AXES; x++) pos[x] = (double)p.at[x];
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
  };
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
    if(np == VEC) __builtin_memcpy(f, src, sizeof(f));
    else {
#pragma unroll
      for(int j = 0; j < VEC * AXES; j++) f[j] = j < np * AXES ? src[j] : 0.0f;
    }
    if(!TOKENS) {
      Position p;
      position(token, p);
      angles(p);
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
  // The run's rows: heads h0.. of the token, or tokens of head h0.
  const int64_t xStep = TOKENS ? a.xToken : a.xHead, outStep = TOKENS ? a.outToken : a.outHead;
  const int rows = TOKENS ? (int)min((int64_t)a.tokenRun, a.tokens - token) : min(a.headRun, a.heads - h0);
  src += h0 * a.xHead;
  dst += h0 * a.outHead;
  if(a.dim >= VEC) {
    // 16 bytes that lie in the row wherever a group ends, moved to their places
    // (what other threads write beside them is not used).
    const int at0 = min(c0, a.dim - VEC), at1 = min(c1, a.dim - VEC);
    const int drop0 = c0 - at0, drop1 = n1 > 0 ? c1 - at1 : 0;
    auto drop = [](Group& g, int n) {
#pragma unroll 1
      for(int i = 0; i < n; i++) {
        const uint4 w = shiftDown<T>(make_uint4(g.v.x, g.v.y, g.v.z, g.v.w));
        g.v = u32x4_t{w.x, w.y, w.z, w.w};
      }
    };
    for(int r = 0; r < rows; r += ROPE_AHEAD) {
      Group u[ROPE_AHEAD][2];
      Position p[ROPE_AHEAD];
#pragma unroll
      for(int i = 0; i < ROPE_AHEAD; i++) {
        if(TOKENS) position(token + min(r + i, rows - 1), p[i]);
        const T* row = src + min(r + i, rows - 1) * xStep;
        __builtin_memcpy(&u[i][0].v, row + at0, 16);
        __builtin_memcpy(&u[i][1].v, row + at1, 16);
      }
#pragma unroll
      for(int i = 0; i < ROPE_AHEAD; i++) {
        if(r + i >= rows) break;
        T* row = dst + (r + i) * outStep;
        if(TOKENS && turns) angles(p[i]);
        drop(u[i][0], drop0);
        drop(u[i][1], drop1);
        if(turns) turn(u[i][0], u[i][1]);
        storeParts(row + c0, u[i][0].v, n0);
        storeParts(row + c1, u[i][1].v, n1);
      }
    }
    return;
  }
  for(int r = 0; r < rows; r++) {
    Group u0, u1;
    const uint4 v0 = loadGroupSmall(src + r * xStep + c0, n0), v1 = loadGroupSmall(src + r * xStep + c1, n1);
    u0.v = u32x4_t{v0.x, v0.y, v0.z, v0.w};
    u1.v = u32x4_t{v1.x, v1.y, v1.z, v1.w};
    if(TOKENS && turns) {
      Position p;
      position(token + r, p);
      angles(p);
    }
    if(turns) turn(u0, u1);
    storeGroup(dst + r * outStep + c0, make_uint4(u0.v.x, u0.v.y, u0.v.z, u0.v.w), n0);
    storeGroup(dst + r * outStep + c1, make_uint4(u1.v.x, u1.v.y, u1.v.z, u1.v.w), n1);
  }
}

template<typename T, bool HALVES, int AXES>
void launchRuns(const RopeArgs& a, int64_t blocks, hipStream_t stream) {
  const dim3 grid((unsigned)blocks);
  if(a.tokenRun > 1) ropeAxesKernel<T, HALVES, AXES, true><<<grid, 256, 0, stream>>>(a);
  else ropeAxesKernel<T, HALVES, AXES, false><<<grid, 256, 0, stream>>>(a);
}

template<typename T, bool HALVES>
void launchAxes(const RopeArgs& a, int64_t blocks, hipStream_t stream) {
  if(a.axes == 1) launchRuns<T, HALVES, 1>(a, blocks, stream);
  else if(a.axes == 2) launchRuns<T, HALVES, 2>(a, blocks, stream);
  else if(a.axes == 3) launchRuns<T, HALVES, 3>(a, blocks, stream);
  else launchRuns<T, HALVES, 4>(a, blocks, stream);
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
  // Heads with tables of their own: runs of up to 4 tokens, in the same way. 20011
  // tokens of 32 x 128 bf16, three axes: 82 us with runs of one, 61 of four; 19377 x
  // 17 x 120 fp16, four axes, 76 and 37 (there with wide loads for a head's last
  // pairs too); 46208 x 6 x 64 fp32 28 and 25.
  a.tokenRun = 1;
  while(a.headRun == 1 && a.tokenRun < ROPE_AHEAD && (p.tokens + 2 * a.tokenRun - 1) / (2 * a.tokenRun) * p.heads * a.groups >= (1 << 18)) a.tokenRun *= 2;
  a.tokens = p.tokens;
  a.items = (p.tokens + a.tokenRun - 1) / a.tokenRun * a.headRuns * a.groups;
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
