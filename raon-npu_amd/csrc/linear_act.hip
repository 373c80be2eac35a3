// y[n, M'] = RTNE(act(x[n, K] @ W^T + bias) + residual), q4nx or bfp16 weights, of one matrix
// or of each row's expert, on bf16 MFMA (wave_gemm.h): exact products, fp32 sums, one
// rounding at the end.  Gated activations pair weight row i (gate) with row M/2 + i.
//
// One workgroup takes 16 MF rows x 16 NF weight rows (half of them gate, half up when the
// activation is gated), its W waves a W-th of K each; the waves' sums meet in LDS and are
// added in wave order, where bias, activation and residual cost nothing but their own bytes.
// One row of q4nx [2048, 768] takes 4.4 us, the 8 experts of a token's gate/up (15.7 MB) 8.5; 445
// rows of [1536, 2048] with SwiGLU 12.8 us (220 TFLOP/s), bound by the vector instructions around
// the MFMAs (one FMA per group and output, the unpacking), which grow with the rows.  Eight
// waves a tile 17.1, 32 x 64 tiles 14.3 (336 of them).
// By expert, a workgroup finds its rows from the experts' offsets itself (a wave scan over at
// most 256 experts), so that the offsets stay on the device.
#include <algorithm>

#include "linear_act.h"
#include "wave_gemm.h"

namespace rmoe {
namespace {

constexpr int kPad = 4;  // floats of padding per row of the partial sums

// Gated tiles hold NF / 2 fragments of gate rows, then the up rows of the same units.
// kTail: the rows end inside a K tile.
template <int kFmt, int MF, int NF, int XI, bool kGated, bool kTail>
__global__ __launch_bounds__(512) void linear_act_kernel(LinAct a, int n_nt) {
  extern __shared__ __attribute__((aligned(16))) float la_lds[];
  constexpr int kTB = kFmt == RMOE_FMT_BFP16 ? kB16TileBytes : kTileBytes;
  constexpr int kCols = 16 * NF, kStride = kCols + kPad, kOut = kGated ? kCols / 2 : kCols;
  constexpr int BM = XI == 1 ? 4 : 16 * MF;  // rows of a tile
  RowTiles<BM> rt;
  const int n_mt = a.offsets ? rt.total(a.offsets, a.n_experts, a.n) : (a.n + BM - 1) / BM;
  // XCD x takes a contiguous eighth of the tiles, the row tiles of one weight tile (by
  // expert: the weight tiles of one row tile) back to back.
  const int total = n_mt * n_nt, per = (total + 7) / 8, slot = (int)blockIdx.x / 8;
  const int id = ((int)blockIdx.x % 8) * per + slot;
  if (slot >= per || id >= total) return;
  int nt, e = 0, row0, nrow;
  if (a.offsets) {
    nt = id % n_nt;
    rt.find(id / n_nt, e, row0, nrow);
  } else {
    nt = id / n_mt;
    row0 = (id % n_mt) * BM;
    nrow = min(BM, a.n - row0);
  }
  const int tid = threadIdx.x, lane = tid & 63, wave = wave_id(), W = blockDim.x >> 6;
  const int l16 = lane & 15, lq = lane >> 4;
  const int nkt = a.K / kTileCols, nkt_in = (a.K_in + kTileCols - 1) / kTileCols;
  const uint8_t* tiles = a.tiles + (size_t)e * a.wstride;
  WaveOperands<MF, NF, XI, kTail> o;
#pragma unroll
  for (int f = 0; f < NF; ++f) {
    const int row = kGated ? nt * kOut + 16 * (f % (NF / 2 > 0 ? NF / 2 : 1)) + (f >= NF / 2 ? a.M / 2 : 0)
                           : nt * kCols + 16 * f;
    o.w[f] = tiles + (size_t)(row / kTileRows) * nkt * kTB + (row % kTileRows) * 16;
  }
  // Rows past the tile repeat its last one; their results are not stored.
  o.x = reinterpret_cast<const uint8_t*>(a.x + (size_t)row0 * a.ldx);
#pragma unroll
  for (int m = 0; m < MF; ++m)
#pragma unroll
    for (int i = 0; i < XI; ++i)
      o.xoff[m][i] = (uint32_t)min(16 * m + 4 * i + lq, nrow - 1) * (uint32_t)(2 * a.ldx) + 16u * (uint32_t)l16;
  o.xchunks = (uint32_t)a.K_in / 8u;
  o.lds = reinterpret_cast<uint8_t*>(la_lds) + (size_t)wave * 4096 * MF;
  wg_f32x4 acc[MF][NF];
#pragma unroll
  for (int m = 0; m < MF; ++m)
#pragma unroll
    for (int f = 0; f < NF; ++f) acc[m][f] = wg_f32x4{0.f, 0.f, 0.f, 0.f};
  wave_gemm<kFmt, MF, NF, XI>(o, wave * nkt_in / W, (wave + 1) * nkt_in / W, acc);
  __syncthreads();  // the partial sums reuse the waves' activation regions
  float* mine = la_lds + (size_t)wave * 16 * MF * kStride;
#pragma unroll
  for (int m = 0; m < MF; ++m)
#pragma unroll
    for (int f = 0; f < NF; ++f)
#pragma unroll
      for (int i = 0; i < 4; ++i) mine[(16 * m + 4 * lq + i) * kStride + 16 * f + l16] = acc[m][f][i];
  __syncthreads();
  constexpr float kUnit = kFmt == RMOE_FMT_BFP16 ? 4.f : 1.f;  // see wave_gemm.h
  auto sum = [&](int t, int c) {
    const float* q = la_lds + t * kStride + c;
    float4 v = *reinterpret_cast<const float4*>(q);
    for (int w = 1; w < W; ++w) {
      const float4 u = *reinterpret_cast<const float4*>(q + (size_t)w * 16 * MF * kStride);
      v.x += u.x;
      v.y += u.y;
      v.z += u.z;
      v.w += u.w;
    }
    return v;
  };
  const int width = kGated ? a.M / 2 : a.M;
  const float* bias = a.bias ? a.bias + (size_t)e * a.M : nullptr;
  const bool wide = ((reinterpret_cast<uintptr_t>(a.y) | reinterpret_cast<uintptr_t>(a.residual)) & 7) == 0;
  // Four columns a thread.
  for (int i = tid; i < nrow * (kOut / 4); i += blockDim.x) {
    const int t = i / (kOut / 4), c = 4 * (i % (kOut / 4)), col = nt * kOut + c;
    float z[4], u[4];
    *reinterpret_cast<float4*>(z) = sum(t, c);
    if constexpr (kGated) *reinterpret_cast<float4*>(u) = sum(t, kOut + c);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      z[k] *= kUnit;
      if (bias) z[k] += bias[col + k];
      if constexpr (kGated) {
        u[k] *= kUnit;
        if (bias) u[k] += bias[a.M / 2 + col + k];
        z[k] = act_pair(a.act, z[k], u[k], a.gb, a.vb);
      } else {
        z[k] = act_single(a.act, z[k]);
      }
    }
    const size_t at = (size_t)(row0 + t) * width + col;
    if (wide) {
      if (a.residual) {
        const uint2 r = *reinterpret_cast<const uint2*>(a.residual + at);
        z[0] += __uint_as_float(r.x << 16);
        z[1] += __uint_as_float(r.x & 0xffff0000u);
        z[2] += __uint_as_float(r.y << 16);
        z[3] += __uint_as_float(r.y & 0xffff0000u);
      }
      *reinterpret_cast<uint2*>(a.y + at) =
          make_uint2(f32_to_bf16(z[0]) | (f32_to_bf16(z[1]) << 16), f32_to_bf16(z[2]) | (f32_to_bf16(z[3]) << 16));
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        a.y[at + k] = (uint16_t)f32_to_bf16(a.residual ? z[k] + bf16_to_f32(a.residual[at + k]) : z[k]);
    }
  }
}

// Dynamic LDS of W waves: their activation regions, then in the same place their partial sums.
constexpr size_t act_lds(int MF, int NF, int W) {
  const size_t sums = (size_t)16 * MF * (16 * NF + kPad) * 4, rows = (size_t)4096 * MF;
  return W * (sums > rows ? sums : rows);
}

template <int kFmt, int MF, int NF, int XI>
hipError_t launch(const LinAct& a, hipStream_t st) {
  const int nkt = (a.K_in + kTileCols - 1) / kTileCols, W = std::min(nkt, nkt >= 64 ? 8 : 4);
  constexpr int BM = XI == 1 ? 4 : 16 * MF;
  const size_t mt = a.offsets ? std::min<size_t>(a.n, (size_t)a.n / BM + a.n_experts) : ((size_t)a.n + BM - 1) / BM;
  const size_t total = mt * (a.M / (16 * NF)), grid = 8 * ((total + 7) / 8);
  if (grid * 64 * W >= (size_t)1 << 32 || total >= (size_t)1 << 31) return hipErrorInvalidValue;
  constexpr bool kPair = NF > 1;
  auto* kernel = a.K_in % kTileCols ? (act_gated(a.act) ? linear_act_kernel<kFmt, MF, NF, XI, kPair, true>
                                                        : linear_act_kernel<kFmt, MF, NF, XI, false, true>)
                                    : (act_gated(a.act) ? linear_act_kernel<kFmt, MF, NF, XI, kPair, false>
                                                        : linear_act_kernel<kFmt, MF, NF, XI, false, false>);
  hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(64 * W), act_lds(MF, NF, W), st, a, a.M / (16 * NF));
  return hipGetLastError();
}

// The largest tile that still gives the chip's 256 CUs kFillTiles workgroups, as for the
// product without an epilogue (linear_mfma.hip); a gated tile needs a gate and an up fragment.
// By expert, fewer rows than experts mostly come one to an expert: tiles of four rows then.
constexpr int kFillTiles = 448;

template <int kFmt>
hipError_t pick(const LinAct& a, hipStream_t st) {
  const bool gated = act_gated(a.act), sparse = a.offsets && a.n < a.n_experts;
  auto fills = [&](int rows, int nf) {
    const size_t mt = sparse ? (size_t)a.n : ((size_t)a.n + rows - 1) / rows;
    return mt * (size_t)(a.M / (16 * nf)) >= kFillTiles;
  };
  if (a.n <= 4 || sparse) {  // only the first row quartet of the fragment is loaded
    if (fills(4, 4)) return launch<kFmt, 1, 4, 1>(a, st);
    if (gated || fills(4, 2)) return launch<kFmt, 1, 2, 1>(a, st);
    return launch<kFmt, 1, 1, 1>(a, st);
  }
  if (a.n > 16) {
    if (fills(32, 4)) return launch<kFmt, 2, 4, 4>(a, st);
    if (fills(32, 2)) return launch<kFmt, 2, 2, 4>(a, st);
  } else if (fills(16, 4)) {
    return launch<kFmt, 1, 4, 4>(a, st);
  }
  if (gated || fills(16, 2)) return launch<kFmt, 1, 2, 4>(a, st);
  return launch<kFmt, 1, 1, 4>(a, st);
}

}  // namespace

template <int kFmt>
static hipError_t setup() {
  const void* fns[4] = {(const void*)linear_act_kernel<kFmt, 2, 4, 4, true, true>,
                        (const void*)linear_act_kernel<kFmt, 2, 4, 4, true, false>,
                        (const void*)linear_act_kernel<kFmt, 2, 4, 4, false, true>,
                        (const void*)linear_act_kernel<kFmt, 2, 4, 4, false, false>};
  for (const void* f : fns) {
    const hipError_t e = hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, (int)act_lds(2, 4, 8));
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}
// Allow the 32 x 64 tiles of eight waves their 68 KB of dynamic LDS (the others stay under 64).
hipError_t linear_act_setup() {
  const hipError_t e = setup<RMOE_FMT_Q4NX>();
  return e == hipSuccess ? setup<RMOE_FMT_BFP16>() : e;
}

hipError_t launch_linear_act(const LinAct& a, uint8_t* scratch, size_t bytes, hipStream_t st) {
  if (act_tiles_serve(a.fmt, a.M, a.K, a.offsets ? a.n_experts : 1, a.n)) return launch_act_tiles(a, scratch, bytes, st);
  return a.fmt == RMOE_FMT_BFP16 ? pick<RMOE_FMT_BFP16>(a, st) : pick<RMOE_FMT_Q4NX>(a, st);
}

}  // namespace rmoe
