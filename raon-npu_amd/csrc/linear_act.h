// What the kernels of y = act(x W^T + bias) + residual share: the epilogue's arithmetic and
// the row tiles of a product by expert.
#pragma once

#include "../../include/raon_moe.h"
#include "rmoe_internal.h"

namespace rmoe {

__host__ __device__ constexpr bool act_gated(int act) { return act == RMOE_ACT_SITU || act == RMOE_ACT_SWIGLU; }

// Activations of one value.  Each is z times a probability formed without cancellation: the
// sigmoid from exp(-|z|), the normal distribution's from erfc, so that small results keep
// their relative accuracy.  exp2 and the reciprocal are the hardware's (1 ulp each); with the
// exponent's own rounding exp(z) is off by (2 + |z|) 2^-23 of it, far below a bf16 rounding.
// They are kept short: a product with 4,096 x 1,088 SiTU outputs took 83 us with IEEE
// divisions, Newton steps and clamps, and 77 without.  The calls over whole MoE layers keep
// act_situ() and act_swiglu() (rmoe_internal.h), which follow the CPU path's operations and whose
// gate and up are rounded to bf16 first; both are within a few steps of fp32 of the formula.
__device__ __forceinline__ float recip(float d) { return __builtin_amdgcn_rcpf(d); }
__device__ __forceinline__ float exp_of(float z) {
  const float t = 1.44269504088896341f * z;
  const int s = t < -100.f ? 40 : 0;  // the instruction gives 0 for a subnormal result
  return __builtin_amdgcn_ldexpf(__builtin_amdgcn_exp2f(t + (float)s), -s);
}
__device__ __forceinline__ float sigmoid_of(float z) {
  const float e = exp_of(-fabsf(z)), r = recip(1.0f + e);
  return z >= 0.f ? r : e * r;
}
// tanh: 1 - 2 / (1 + exp(2 |z|)), which an infinite exp makes 1, and below 0.3, where that
// cancels, its power series to z^9 (the next term is (1382 / 155925) z^10 = 5.3e-8 of z there).
__device__ __forceinline__ float tanh_of(float z) {
  const float a = fabsf(z), q = z * z;
  const float big = fmaf(-2.0f, recip(1.0f + __builtin_amdgcn_exp2f(2.88539008177792681f * a)), 1.0f);
  const float s = fmaf(q, fmaf(q, fmaf(q, fmaf(q, 62.f / 2835.f, -17.f / 315.f), 2.f / 15.f), -1.f / 3.f), 1.0f);
  return a < 0.3f ? z * s : copysignf(big, z);
}
__device__ __forceinline__ float act_pair(int act, float g, float u, float gb, float vb) {
  if (act == RMOE_ACT_SWIGLU) return g * sigmoid_of(g) * u;
  return gb * tanh_of(g * (1.0f / gb)) * sigmoid_of(g) * (vb * tanh_of(u * (1.0f / vb)));
}
__device__ __forceinline__ float act_single(int act, float z) {
  if (act == RMOE_ACT_SILU) return z * sigmoid_of(z);
  if (act == RMOE_ACT_GELU) return z * (0.5f * erfcf(-0.70710678118654752f * z));
  // 0.5 (1 + tanh(u)) = sigmoid(2 u), u = sqrt(2 / pi) (z + 0.044715 z^3)
  if (act == RMOE_ACT_GELU_TANH) return z * sigmoid_of(1.5957691216057308f * fmaf(0.044715f * z * z, z, z));
  return z;
}

// The tiles of BM rows over the experts' sorted rows, listed by expert; the calling wave's
// lane l holds experts 4l..4l+3 (at most 256).  Offsets are clamped to [0, n] so that no
// value of theirs leaves the rows.
template <int BM>
struct RowTiles {
  int b[5], excl, sum;
  __device__ __forceinline__ int total(const int32_t* __restrict__ offsets, int E, int n) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < 5; ++i) b[i] = min(max(offsets[min(4 * lane + i, E)], 0), n);
    sum = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) sum += tiles(i);
    int incl = sum;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int y = __shfl_up(incl, d, 64);
      if (lane >= d) incl += y;
    }
    excl = incl - sum;
    return __builtin_amdgcn_readlane(incl, 63);
  }
  __device__ __forceinline__ int tiles(int i) const { return b[i + 1] > b[i] ? (b[i + 1] - b[i] + BM - 1) / BM : 0; }
  // Tile mt (below total): its expert, first row and rows, the same in every lane.
  __device__ __forceinline__ void find(int mt, int& e, int& row0, int& rows) const {
    const int lane = threadIdx.x & 63;
    int le = 0, lrow = 0, lrows = 0, t = mt - excl;
    const bool mine = t >= 0 && t < sum;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = tiles(i);
      if (t >= 0 && t < c) {
        le = 4 * lane + i;
        lrow = b[i] + t * BM;
        lrows = min(BM, b[i + 1] - lrow);
      }
      t -= c;
    }
    const int src = __ffsll((unsigned long long)__ballot(mine)) - 1;
    e = __builtin_amdgcn_readlane(le, src);
    row0 = __builtin_amdgcn_readlane(lrow, src);
    rows = __builtin_amdgcn_readlane(lrows, src);
  }
};

}  // namespace rmoe
