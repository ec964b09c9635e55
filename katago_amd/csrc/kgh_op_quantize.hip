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

template<typename T>
__global__ __launch_bounds__(256) void quantizeRowsKernel(QuantArgs a) {
  __shared__ unsigned tops[4];
  for(int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
  const T* x = (const T*)a.x + row * a.ldx;
  int8_t* out = a.out + row * a.ldo;
  unsigned top = 0;
  for(int c = threadIdx.x; c < a.channels; c += 256) top = max(top, magnitudeBits((float)x[c]));
#pragma unroll
  for(int w = 32; w > 0; w >>= 1) top = max(top, (unsigned)__shfl_xor((int)top, w));
  if((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
  __syncthreads();
  top = max(max(tops[0], tops[1]), max(tops[2], tops[3]));
  const RowScale s(top);
  for(int c = threadIdx.x; c < a.channels; c += 256) out[c] = (int8_t)s.quantized((float)x[c]);
  if(threadIdx.x == 0) a.scales[row] = s.scale;
  __syncthreads();
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
  withDtype(p.dtype, [&](auto t) { quantizeRowsKernel<decltype(t)><<<dim3((unsigned)std::min<int64_t>(p.rows, 1 << 20)), 256, 0, stream>>>(a); });
  KGH_CHECK_LAUNCH();
}

}  // namespace kgh
