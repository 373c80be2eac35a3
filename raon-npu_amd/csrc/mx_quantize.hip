// Rows to microscaled 4-bit codes and scales (mx.h), and if asked to the values these stand for in the rows' own
// type (a forward pass in training computes with those; its gradient passes unchanged).
//
// Bound by HBM: each value is read once, 17/32 of a byte and the value itself written.  A lane takes eight
// columns (16 bytes of bf16), a quad of lanes a block: its largest magnitude meets in two exchanges between
// lanes, and one conversion instruction rounds two values.  Where the rows are whole blocks the matrix is one run of them
// and no lane divides by the row's length.  24,064 rows of 2,560 fp32 values, to codes and what they stand for, 525 MB:
// 90 us, 5.8 TB/s; 53,600 rows of 2,048 in bf16 to codes alone, 278 MB: 46 us, 6.0 TB/s (a large copy: 4.9).  One row
// of 2,048 takes 2.4 us, a launch and a trip to memory.
#include <algorithm>

#include "mx.h"

namespace rmoe {
namespace {

struct QuantArgs {
  const void* x;
  uint8_t *codes, *scales;
  void* values;
  size_t T;
  int K, P;  // width, and rounded up to 32
};

// kWide: K a multiple of 32, x and values aligned to 16 bytes.
template <int DT, bool kWide, bool kValues>
__global__ __launch_bounds__(256) void mx_quantize_kernel(QuantArgs a, size_t first) {
  typedef typename RowElem<DT>::T E;
  const size_t u = first + (size_t)blockIdx.x * 256 + threadIdx.x, per = (size_t)a.P / 8;
  if (u >= a.T * per) return;  // a quad leaves as one: P / 8 is a multiple of 4
  size_t row = 0;
  int c = 0;
  if constexpr (!kWide) {
    row = u / per;
    c = (int)(u - row * per) * 8;
  }
  const E* xr = static_cast<const E*>(a.x) + (kWide ? u * 8 : row * a.K);
  const Chunk<DT> in = load_chunk<DT, kWide>(xr, c, a.K);
  float x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = RowElem<DT>::get(in.v[i]);
  uint32_t scale;
  const uint32_t q = mx_quantize8(x, scale);
  reinterpret_cast<uint32_t*>(a.codes)[u] = q;
  if ((u & 3) == 0) a.scales[u >> 2] = (uint8_t)scale;
  if constexpr (kValues) {
    Chunk<DT> out;
#pragma unroll
    for (int i = 0; i < 8; ++i) out.v[i] = RowElem<DT>::put(mx_value(q, i, scale));
    store_chunk<DT, kWide>(static_cast<E*>(a.values) + (kWide ? u * 8 : row * a.K), c, a.K, out);
  }
}

template <int DT>
hipError_t quantize_with(const QuantArgs& a, hipStream_t st) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.values);
  const bool wide = a.K == a.P && at % 16 == 0;
  auto* kernel = a.values ? (wide ? mx_quantize_kernel<DT, true, true> : mx_quantize_kernel<DT, false, true>)
                          : (wide ? mx_quantize_kernel<DT, true, false> : mx_quantize_kernel<DT, false, false>);
  const size_t units = a.T * ((size_t)a.P / 8), step = (((size_t)1 << 32) / 256 - 1) * 256;  // threads of a launch
  for (size_t u = 0; u < units; u += step) {
    const size_t n = std::min(step, units - u);
    hipLaunchKernelGGL(kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, a, u);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace

hipError_t launch_mx_quantize(const void* x, int dtype, int T, int K, uint8_t* codes, uint8_t* scales, void* values,
                              hipStream_t st) {
  const QuantArgs a{x, codes, scales, values, (size_t)T, K, (K + kMxBlock - 1) / kMxBlock * kMxBlock};
  if (dtype == RMOE_DT_BF16) return quantize_with<RMOE_DT_BF16>(a, st);
  if (dtype == RMOE_DT_F16) return quantize_with<RMOE_DT_F16>(a, st);
  return quantize_with<RMOE_DT_F32>(a, st);
}

}  // namespace rmoe
