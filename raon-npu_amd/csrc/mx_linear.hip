// y[n, M'] = RTNE(act(x[n, K] @ W^T + bias) + residual) of microscaled 4-bit rows and weights (mx.h), of one
// matrix or of each row's expert, on the scaled MFMA: codes and scale bytes go into the matrix pipes as they are
// held, products are exact, sums fp32.
#include <algorithm>

#include "linear_act.h"
#include "mx.h"

namespace rmoe {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kFp4 = 4;         // the instruction's number of the e2m1 format, for both operands
constexpr int kScaleOne = 127;  // a scale byte of 2^0

// Codes as the instruction's operand: its upper half belongs to the wider formats.
__device__ __forceinline__ i32x8 operand(const i32x4& v) { return i32x8{v.x, v.y, v.z, v.w, 0, 0, 0, 0}; }

// Four consecutive outputs of row t from the sums z (and u of the up half).
struct Epilogue {
  const float* bias;  // of this matrix, or null
  const uint16_t* residual;
  uint16_t* y;
  int width, up, act;
  float gb, vb;
  bool wide;
  __device__ __forceinline__ Epilogue(const MxLin& a, int e, bool gated)
      : bias(a.bias ? a.bias + (size_t)e * a.M : nullptr), residual(a.residual), y(a.y), width(gated ? a.M / 2 : a.M),
        up(a.M / 2), act(a.act), gb(a.gb), vb(a.vb),
        wide(width % 4 == 0 && ((reinterpret_cast<uintptr_t>(a.y) | reinterpret_cast<uintptr_t>(a.residual)) & 7) == 0) {}
  template <bool kGated>
  __device__ __forceinline__ void put(size_t t, int col, float (&z)[4], float (&u)[4]) const {
    if (col >= width) return;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int c = min(col + k, width - 1);
      if (bias) z[k] += bias[c];
      if constexpr (kGated) {
        if (bias) u[k] += bias[up + c];
        z[k] = act_pair(act, z[k], u[k], gb, vb);
      } else {
        z[k] = act_single(act, z[k]);
      }
    }
    const size_t at = t * width + col;
    if (wide) {
      if (residual) {
        const uint2 r = *reinterpret_cast<const uint2*>(residual + at);
        z[0] += __uint_as_float(r.x << 16);
        z[1] += __uint_as_float(r.x & 0xffff0000u);
        z[2] += __uint_as_float(r.y << 16);
        z[3] += __uint_as_float(r.y & 0xffff0000u);
      }
      *reinterpret_cast<uint2*>(y + at) =
          make_uint2(f32_to_bf16(z[0]) | (f32_to_bf16(z[1]) << 16), f32_to_bf16(z[2]) | (f32_to_bf16(z[3]) << 16));
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (col + k < width)
          y[at + k] = (uint16_t)f32_to_bf16(residual ? z[k] + bf16_to_f32(residual[at + k]) : z[k]);
    }
  }
};

// ------------------------------------------------------------------ few rows --
// Tiles of 16 rows of x.  A wave takes NA fragments of 16 weight rows; the workgroup's four waves are WR
// stripes of them by WK = 4 / WR parts of K, whose sums meet in LDS and are added in their order.
// A gated stripe holds 8 NA gate rows, then the up rows of the same outputs.
template <int NA, int WR, bool kGated, bool kTail>
__global__ __launch_bounds__(256) void mx_few_kernel(MxLin a, int n_nt) {
  constexpr int WK = 4 / WR, kRows = 16 * NA, kOut = kGated ? kRows / 2 : kRows, kStride = kRows + 4;
  __shared__ __attribute__((aligned(16))) float sums[4][16 * kStride];
  RowTiles<16> rt;
  const int n_mt = a.offsets ? rt.total(a.offsets, a.n_experts, a.n) : (a.n + 15) / 16;
  // XCD x takes a contiguous eighth of the tiles, the row tiles of one weight tile (by expert: the weight
  // tiles of one row tile) back to back.
  const long total = (long)n_mt * n_nt, per = (total + 7) / 8, slot = blockIdx.x / 8;
  const long id = (long)(blockIdx.x % 8) * per + slot;
  if (slot >= per || id >= total) return;
  int nt, e = 0, row0, nrow;
  if (a.offsets) {
    nt = (int)(id % n_nt);
    rt.find((int)(id / n_nt), e, row0, nrow);
  } else {
    nt = (int)(id / n_mt);
    row0 = (int)(id % n_mt) * 16;
    nrow = min(16, a.n - row0);
  }
  const int tid = threadIdx.x, lane = tid & 63, wave = wave_id(), l16 = lane & 15, lq = lane >> 4;
  const int wr = wave % WR, wk = wave / WR;
  const int kb = a.K / kMxBlock, steps = (kb + 3) / 4, s0 = wk * steps / WK, s1 = (wk + 1) * steps / WK;
  const int width = kGated ? a.M / 2 : a.M, out0 = (nt * WR + wr) * kOut;
  // Rows past the tile repeat the last one; their results are not stored.
  const size_t xrow = (size_t)row0 + min(l16, nrow - 1);
  const uint8_t* xp = a.x + xrow * (a.K / 2);
  const uint8_t* xsp = a.xs + xrow * kb;
  const uint8_t *wp[NA], *wsp[NA];
#pragma unroll
  for (int f = 0; f < NA; ++f) {
    const int r = 16 * f + l16;
    const size_t row = (size_t)e * a.M + (kGated ? (r >= kOut ? a.M / 2 : 0) + min(out0 + r % kOut, width - 1)
                                                 : min(out0 + r, width - 1));
    wp[f] = a.w + row * (a.K / 2);
    wsp[f] = a.ws + row * kb;
  }
  f32x4 acc[NA];
#pragma unroll
  for (int f = 0; f < NA; ++f) acc[f] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int s = s0; s < s1; ++s) {
    const int b = 4 * s + lq, at = kTail ? min(b, kb - 1) : b;
    const bool in = !kTail || b < kb;
    i32x4 x = *reinterpret_cast<const i32x4*>(xp + (size_t)at * 16);
    const int xsc = in ? xsp[at] : kScaleOne;
    if (!in) x = i32x4{0, 0, 0, 0};
#pragma unroll
    for (int f = 0; f < NA; ++f) {
      const i32x4 w = *reinterpret_cast<const i32x4*>(wp[f] + (size_t)at * 16);
      const int wsc = in ? wsp[f][at] : kScaleOne;
      acc[f] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(operand(w), operand(x), acc[f], kFp4, kFp4, 0, wsc, 0, xsc);
    }
  }
  // acc[f][i]: weight row 16 f + 4 lq + i, row of x l16.
#pragma unroll
  for (int f = 0; f < NA; ++f) *reinterpret_cast<f32x4*>(&sums[wave][l16 * kStride + 16 * f + 4 * lq]) = acc[f];
  __syncthreads();
  const Epilogue ep(a, e, kGated);
  auto sum = [&](int stripe, int t, int r, float (&z)[4]) {
    f32x4 v = *reinterpret_cast<const f32x4*>(&sums[stripe][t * kStride + r]);
#pragma unroll
    for (int k = 1; k < WK; ++k) v += *reinterpret_cast<const f32x4*>(&sums[stripe + k * WR][t * kStride + r]);
#pragma unroll
    for (int i = 0; i < 4; ++i) z[i] = v[i];
  };
  constexpr int kQuads = WR * kOut / 4;
  for (int i = tid; i < nrow * kQuads; i += 256) {
    const int t = i / kQuads, q = i % kQuads, stripe = q / (kOut / 4), c = 4 * (q % (kOut / 4));
    float z[4], u[4] = {0.f, 0.f, 0.f, 0.f};
    sum(stripe, t, c, z);
    if constexpr (kGated) sum(stripe, t, kOut + c, u);
    ep.template put<kGated>((size_t)row0 + t, (nt * WR + stripe) * kOut + c, z, u);
  }
}

template <int NA, int WR>
hipError_t launch_few(const MxLin& a, hipStream_t st) {
  const bool gated = act_gated(a.act), tail = a.K % (4 * kMxBlock) != 0;
  const int width = gated ? a.M / 2 : a.M, out = 16 * NA * WR / (gated ? 2 : 1), n_nt = (width + out - 1) / out;
  const size_t mt = a.offsets ? std::min<size_t>(a.n, (size_t)a.n / 16 + a.n_experts) : ((size_t)a.n + 15) / 16;
  const size_t grid = 8 * ((mt * n_nt + 7) / 8);
  if (grid * 256 >= (size_t)1 << 32) return hipErrorInvalidValue;
  auto* kernel = gated ? (tail ? mx_few_kernel<NA, WR, true, true> : mx_few_kernel<NA, WR, true, false>)
                       : (tail ? mx_few_kernel<NA, WR, false, true> : mx_few_kernel<NA, WR, false, false>);
  hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(256), 0, st, a, n_nt);
  return hipGetLastError();
}

}  // namespace

hipError_t mx_linear_setup() { return hipSuccess; }

hipError_t launch_mx_linear(const MxLin& a, hipStream_t st) {
  const size_t mt = a.offsets ? std::min<size_t>(a.n, (size_t)a.n / 16 + a.n_experts) : ((size_t)a.n + 15) / 16;
  if (mt * a.M >= (size_t)512 * 256) return launch_few<4, 4>(a, st);
  if (mt * a.M >= (size_t)512 * 32) return launch_few<2, 1>(a, st);
  return launch_few<1, 1>(a, st);
}

}  // namespace rmoe
