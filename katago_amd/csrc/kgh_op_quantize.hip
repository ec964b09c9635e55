// Rows in 8 bits with a scale each (kgh_quantize_rows).
#include "kgh_op_quantize_device.h"

#include <algorithm>

namespace {

constexpr int64_t QUANT_MAX_ROWS = 1 << 30;
constexpr int QUANT_MAX_CHANNELS = 1 << 30;

struct QuantArgs {
  const void* x;
  int8_t* out;
  float* scales;
  int64_t ldx, ldo, rows;
  int channels;
};

// A row by `lanes` threads side by side, K 16-byte groups each, which stay in registers
// between the largest value and the whole numbers: bound by the row's way in and out,
// 8192 x 8192 bf16 41.8 us (4.8 TB/s; a copy reaches 5.1).
template<typename T, int K>
__global__ __launch_bounds__(256) void quantizeRowsKernel(QuantArgs a, int lanes) {
  constexpr int VEC = 16 / (int)sizeof(T);
  __shared__ unsigned tops[2][4];
  const int sub = threadIdx.x & (lanes - 1), perBlock = 256 / lanes;
  const int64_t row0 = threadIdx.x / lanes;
  int turn = 0;
  for(int64_t base = (int64_t)blockIdx.x * perBlock; base < a.rows; base += (int64_t)gridDim.x * perBlock, turn ^= 1) {
    const int64_t row = min(base + row0, a.rows - 1);
    const T* x = (const T*)a.x + row * a.ldx;
    u32x4_t v[K];
#pragma unroll
    for(int i = 0; i < K; i++) v[i] = RowGroup<T, false>(min(sub + i * lanes, (a.channels - 1) / VEC), a.channels).load(x);
    unsigned top = 0;
#pragma unroll
    for(int i = 0; i < K; i++) {
      v[i] = RowGroup<T, false>(min(sub + i * lanes, (a.channels - 1) / VEC), a.channels).place(v[i]);
      const Values<T> f(v[i]);
#pragma unroll
      for(int j = 0; j < VEC; j++) top = max(top, magnitudeBits(f.f[j]));
    }
    const RowScale s(rowTop(top, lanes, tops[turn]));
    if(base + row0 >= a.rows) continue;
    int8_t* out = a.out + row * a.ldo;
#pragma unroll
    for(int i = 0; i < K; i++) {
      const int c = (sub + i * lanes) * VEC;
      if(c < a.channels) storeBytes<VEC>(out + c, quantized(Values<T>(v[i]).f, s), 0, a.channels - c);
    }
    if(sub == 0) a.scales[row] = s.scale;
  }
}

// How threads share a row of `groups` 16-byte groups, at most `most` each: the power of
// two in a wave, or the workgroup, that leaves the fewest idle (46208 x 384 fp16: three
// each of 16 threads 12.1 us, one each of 48 of 64 18.1); lanes is 0 where the row is
// longer.
inline RowLanes rowLanesFull(int groups, int most) {
  RowLanes best{0, 0};
  for(int lanes : {64, 32, 16, 8, 256}) {
    const int each = (groups + lanes - 1) / lanes;
    if(each <= most && (best.lanes == 0 || lanes * each < best.lanes * best.each)) best = RowLanes{lanes, each};
  }
  return best;
}

// Rows of any length, read twice.
template<typename T>
__global__ __launch_bounds__(256) void quantizeRowsLongKernel(QuantArgs a) {
  constexpr int VEC = 16 / (int)sizeof(T);
  __shared__ unsigned tops[2][4];
  int turn = 0;
  for(int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1) {
    const T* x = (const T*)a.x + row * a.ldx;
    int8_t* out = a.out + row * a.ldo;
    const int groups = (a.channels + VEC - 1) / VEC;
    unsigned top = 0;
#pragma unroll 4
    for(int g = threadIdx.x; g < groups; g += 256) {
      const RowGroup<T, false> r(g, a.channels);
      const Values<T> f(r.place(r.load(x)));
#pragma unroll
      for(int j = 0; j < VEC; j++) top = max(top, magnitudeBits(f.f[j]));
    }
    const RowScale s(rowTop(top, 256, tops[turn]));
#pragma unroll 4
    for(int g = threadIdx.x; g < groups; g += 256) {
      const RowGroup<T, false> r(g, a.channels);
      storeBytes<VEC>(out + g * VEC, quantized(Values<T>(r.place(r.load(x))).f, s), 0, a.channels - g * VEC);
    }
    if(threadIdx.x == 0) a.scales[row] = s.scale;
  }
}

}  // namespace

namespace kgh {

void checkQuantize(const kgh_quantize_params& p) {
  const char* op = "kgh_quantize_rows";
  opCheckDtype(op, p.dtype);
  if(p.rows < 0 || p.rows > QUANT_MAX_ROWS) opInvalid(op, "rows " + std::to_string(p.rows) + " outside 0.." + std::to_string(QUANT_MAX_ROWS));
  if(p.channels < 1 || p.channels > QUANT_MAX_CHANNELS) opInvalid(op, "channels must be in 1.." + std::to_string(QUANT_MAX_CHANNELS));
  if(p.x_stride < 0) opInvalid(op, "negative stride");
  if(p.rows > 1 && p.out_stride < p.channels) opInvalid(op, "out_stride " + std::to_string(p.out_stride) + " is less than channels");
  if(p.rows == 0) return;
  opCheckPointer(op, "x", p.x, opElemBytes(p.dtype));
  opCheckPointer(op, "out", p.out, 1);
  opCheckPointer(op, "scales", p.scales, 4);
  opCheckApart(op, "x", p.x, p.out);
  opCheckApart(op, "scales", p.scales, p.out);
  if(p.x == p.scales) opInvalid(op, "scales is x itself");
}

void launchQuantize(const kgh_quantize_params& p, hipStream_t stream) {
  if(p.rows == 0) return;
  const QuantArgs a{p.x, p.out, p.scales, p.x_stride, p.out_stride, p.rows, p.channels};
  withDtype(p.dtype, [&](auto t) {
    typedef decltype(t) T;
    constexpr int VEC = 16 / (int)sizeof(T);
    const RowLanes r = rowLanesFull((p.channels + VEC - 1) / VEC, 8);
    const int64_t perBlock = r.lanes == 0 ? 1 : 256 / r.lanes;
    const dim3 grid((unsigned)std::min<int64_t>((p.rows + perBlock - 1) / perBlock, 1 << 20));
    if(r.lanes == 0) quantizeRowsLongKernel<T><<<grid, 256, 0, stream>>>(a);
    else if(r.each <= 1) quantizeRowsKernel<T, 1><<<grid, 256, 0, stream>>>(a, r.lanes);
    else if(r.each <= 2) quantizeRowsKernel<T, 2><<<grid, 256, 0, stream>>>(a, r.lanes);
    else if(r.each <= 3) quantizeRowsKernel<T, 3><<<grid, 256, 0, stream>>>(a, r.lanes);
    else if(r.each <= 4) quantizeRowsKernel<T, 4><<<grid, 256, 0, stream>>>(a, r.lanes);
    else quantizeRowsKernel<T, 8><<<grid, 256, 0, stream>>>(a, r.lanes);
  });
  KGH_CHECK_LAUNCH();
}

}  // namespace kgh
