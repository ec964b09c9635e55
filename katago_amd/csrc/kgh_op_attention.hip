// Attention to an encoder's states (kgh_cross_attention).
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
  float scaleLog2;  // scale * log2(e): exponents are taken to base 2
};

// Keys 64 tile .. + 63 that take part, lane l's key in bit l; wave-uniform.
__device__ __forceinline__ unsigned long long validKeys(const AttnArgs& a, int b, int len, int k0) {
  const int j = k0 + (int)(threadIdx.x & 63);
  const bool on = j < len && (a.mask == nullptr || a.mask[b * a.maskB + j] != 0);
  return __ballot(on);
}

__device__ __forceinline__ int validLength(const AttnArgs& a, int b) {
  return a.lengths == nullptr ? a.lk : min(max(a.lengths[b], 0), a.lk);
}

// One row's running softmax: p = 2^(s c - ref), with a reference point that only
// moves when a tile's maximum passes it by more than 8 (p is at most 256, summed
// in fp32; the normalisation by the sum of the same p makes the choice cancel).
struct RowState {
  float ref = -INFINITY, sum = 0.0f;
};

// ---------------------------------------------------------------------------
// Any sizes, strides and alignment. The rows of a kv head are (query, head of
// the group) pairs, so that grouped heads share the keys that are staged. A wave
// owns 32 rows and computes S^T = K Q^T (lane = row, 16 of 32 keys per lane), so
// a row's softmax is in one lane and its partner lane ^ 32, and P^T is the
// second product's operand as it stands: the key order inside that product's k
// is the accumulator's row order, and V^T is read in the same order.
template<typename T, int D>
__global__ __launch_bounds__(256) void attentionTileKernel(AttnArgs a) {
  typedef typename Vec16<T>::V V;
  constexpr int VEC = 16 / (int)sizeof(T);
  constexpr int KLD = D + VEC;                    // elements of a K row (16-byte gap)
  constexpr int VLD = 64 + 8 / (int)sizeof(T);    // of a V^T row (8-byte gap)
  constexpr int GROUPS = D / VEC;                 // 16-byte groups of a row
  constexpr int LOADS = 64 * GROUPS / 256;
  __shared__ __attribute__((aligned(16))) T Ks[64 * KLD];
  __shared__ __attribute__((aligned(16))) T Vt[D * VLD];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int laneRow = lane & 31, half = lane >> 5;
  const int kvh = blockIdx.y, b = blockIdx.z;
  const int group = a.heads / a.kvHeads;
  const int rows = a.lq * group;
  const int r = ((int)blockIdx.x * 4 + wave) * 32 + laneRow;
  const int rc = min(r, rows - 1);
  const int qi = rc / group, h = kvh * group + (rc - qi * group);
  const T* qRow = (const T*)a.q + b * a.qB + qi * a.qT + h * a.qH;
  const T* kBase = (const T*)a.k + b * a.kB + kvh * a.kH;
  const T* vBase = (const T*)a.v + b * a.vB + kvh * a.vH;

  V qf[D / VEC / 2];
#pragma unroll
  for(int i = 0; i < D / VEC / 2; i++) {
    const int c = (2 * i + half) * VEC;
    const uint4 u = loadGroup(qRow + c, a.dq - c);
    qf[i] = *(const V*)&u;
  }
  floatx16 o[D / 32];
#pragma unroll
  for(int db = 0; db < D / 32; db++)
#pragma unroll
    for(int i = 0; i < 16; i++) o[db][i] = 0.0f;
  RowState row;

  const int len = validLength(a, b);
  for(int k0 = 0; k0 < len; k0 += 64) {
    const unsigned long long valid = validKeys(a, b, len, k0);
    if(valid == 0) continue;  // the same for every wave
    uint4 kr[LOADS], vr[LOADS];
#pragma unroll
    for(int i = 0; i < LOADS; i++) {
      const int key = (tid + i * 256) / GROUPS, c = (tid + i * 256) % GROUPS * VEC;
      const bool on = (valid >> key) & 1;
      kr[i] = loadGroup(kBase + (k0 + key) * a.kT + c, on ? a.dq - c : 0);
      vr[i] = loadGroup(vBase + (k0 + key) * a.vT + c, on ? a.dv - c : 0);
    }
    __syncthreads();
#pragma unroll
    for(int i = 0; i < LOADS; i++) {
      const int key = (tid + i * 256) / GROUPS, c = (tid + i * 256) % GROUPS * VEC;
      *(uint4*)&Ks[key * KLD + c] = kr[i];
      const T* e = (const T*)&vr[i];
#pragma unroll
      for(int j = 0; j < VEC; j++) Vt[(c + j) * VLD + key] = e[j];
    }
    __syncthreads();

    floatx16 s[2];
#pragma unroll
    for(int kb = 0; kb < 2; kb++) {
#pragma unroll
      for(int i = 0; i < 16; i++) s[kb][i] = 0.0f;
#pragma unroll
      for(int i = 0; i < D / VEC / 2; i++) {
        const V kf = *(const V*)&Ks[(kb * 32 + laneRow) * KLD + (2 * i + half) * VEC];
        s[kb] = mma32(kf, qf[i], s[kb]);
      }
      if(valid != ~0ull) {
#pragma unroll
        for(int i = 0; i < 16; i++)
          if(!((valid >> (kb * 32 + (i >> 2) * 8 + half * 4 + (i & 3))) & 1)) s[kb][i] = -INFINITY;
      }
    }
    float top = -INFINITY;
#pragma unroll
    for(int kb = 0; kb < 2; kb++)
#pragma unroll
      for(int i = 0; i < 16; i++) top = fmaxf(top, s[kb][i]);
    top = fmaxf(top, __shfl_xor(top, 32)) * a.scaleLog2;
    float corr = 1.0f;
    if(top > row.ref + 8.0f) {
      corr = __builtin_amdgcn_exp2f(row.ref - top);
      row.ref = top;
    }
    // While a row has met no score above -inf its offset is 0: every p is 0.
    const float off = row.ref == -INFINITY ? 0.0f : -row.ref;
    float sum = 0.0f;
#pragma unroll
    for(int kb = 0; kb < 2; kb++)
#pragma unroll
      for(int i = 0; i < 16; i++) {
        s[kb][i] = __builtin_amdgcn_exp2f(fmaf(s[kb][i], a.scaleLog2, off));
        sum += s[kb][i];
      }
    sum += __shfl_xor(sum, 32);
    row.sum = row.sum * corr + sum;
    if(__any(corr != 1.0f)) {
#pragma unroll
      for(int db = 0; db < D / 32; db++)
#pragma unroll
        for(int i = 0; i < 16; i++) o[db][i] *= corr;
    }
    // VEC accumulator rows per 16-byte group of keys.
#pragma unroll
    for(int kb = 0; kb < 2; kb++)
#pragma unroll
      for(int g = 0; g < 16 / VEC; g++) {
        V pf;
#pragma unroll
        for(int i = 0; i < VEC; i++) pf[i] = (T)s[kb][g * VEC + i];
#pragma unroll
        for(int db = 0; db < D / 32; db++) {
          V vf;
          const T* vRow = &Vt[(db * 32 + laneRow) * VLD + kb * 32 + half * 4];
#pragma unroll
          for(int q = 0; q < VEC / 4; q++)
#pragma unroll
            for(int i = 0; i < 4; i++) vf[q * 4 + i] = vRow[(g * VEC / 4 + q) * 8 + i];
          o[db] = mma32(vf, pf, o[db]);
        }
      }
  }

  if(r >= rows) return;
  const float inv = row.sum == 0.0f ? 0.0f : 1.0f / row.sum;
  T* oRow = (T*)a.out + b * a.oB + qi * a.oT + h * a.oH;
#pragma unroll
  for(int db = 0; db < D / 32; db++)
#pragma unroll
    for(int i = 0; i < 16; i++) {
      const int d = db * 32 + (i >> 2) * 8 + half * 4 + (i & 3);
      if(d < a.dv) oRow[d] = (T)(o[db][i] * inv);
    }
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
  if(!(p.scale > 0.0f) || !std::isfinite(p.scale)) opInvalid(op, "scale must be positive and finite");
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
}

uint64_t attentionWorkspace(const kgh_attention_params&) { return 0; }

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
  const int64_t rows = (int64_t)p.q_len * (p.heads / p.kv_heads);
  const dim3 grid((unsigned)((rows + 127) / 128), (unsigned)p.kv_heads, (unsigned)p.batch);
  const int d = std::max(p.q_head_dim, p.v_head_dim);
  withDtype(p.dtype, [&](auto t) {
    typedef decltype(t) T;
    if(d <= 32) attentionTileKernel<T, 32><<<grid, 256, 0, stream>>>(a);
    else if(d <= 64) attentionTileKernel<T, 64><<<grid, 256, 0, stream>>>(a);
    else attentionTileKernel<T, 128><<<grid, 256, 0, stream>>>(a);
  });
  KGH_CHECK_LAUNCH();
}

}  // namespace kgh
