// The norms before and after a block with its gate and residual scale, and their gradients.
//
//   n = (mean_j b_j^2 + eps)^-1/2,   u = n b wpost      (u = b without a norm after)
//   y = R(c r + g u)                                    (g: none, by column, by row or by element)
//   m = (mean_j y_j^2 + eps)^-1/2,   h = R(m y wpre)
//
// in fp32, R one rounding to the rows' type; h is the norm of y as it is stored, so that a norm of the stored
// rows gives the same bits.  Without a block y is an input and only h is computed.  h may also go (or only go)
// into microscaled 4-bit codes (mx.h), from its rounded values: a product reads them without another pass.
//
// The gradient from dy (of y where it goes on as the residual) and dh, with a = dh wpre:
//   D  = dy + m a - y m^3 (sum_j a_j y_j) / H,          dwpre  = sum_t dh y m
//   dr = c D,   du = g D,   v = du wpost
//   db = n v - b n^3 (sum_j v_j b_j) / H,               dwpost = sum_t du b n
//   dg = D u, summed over what g is shared by.
// n and m are formed again from b and y, which have to be read in any case.
//
// Bound by HBM.  A row is held in the registers of W waves (eight columns a thread and V of these), which meet in
// LDS once for each sum: every element is read and written once.
#include <algorithm>

#include "mx.h"

namespace rmoe {
namespace {

constexpr int kMaxWaves = 8;  // of a row: 256 registers a thread

// Sums of N values over the W waves of a row: a slot per wave, `slots` alternating between calls so that one
// barrier a call is enough.
template <int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float (*slots)[N], int wave, int W) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = wave_sum(v[i]);
  if (W == 1) return;
  if ((threadIdx.x & 63) == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) slots[wave][i] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = slots[0][i];
  for (int w = 1; w < W; ++w) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += slots[w][i];
  }
}

template <int DT>
__device__ __forceinline__ void to_float(const Chunk<DT>& c, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = RowElem<DT>::get(c.v[i]);
}

// Columns c..c+7 of an fp32 vector of H, zeros past it.
__device__ __forceinline__ void load_vector(const float* p, int c, int H, float (&f)[8]) {
  if (c + 8 <= H && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
    *reinterpret_cast<float4*>(f) = *reinterpret_cast<const float4*>(p + c);
    *reinterpret_cast<float4*>(f + 4) = *reinterpret_cast<const float4*>(p + c + 4);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = c + i < H ? p[c + i] : 0.f;
  }
}

__device__ __forceinline__ float inv_rms(float squares, int H, float eps) {
  return 1.0f / sqrtf(squares / (float)H + eps);
}

// The gate of columns c..c+7 of row t as fp32.
template <int DT, bool kWide>
__device__ __forceinline__ void load_gate(const NormArgs& a, size_t t, int c, float (&g)[8]) {
  if (a.gate_kind == RMOE_GATE_COLUMN) {
    load_vector(static_cast<const float*>(a.gate), c, a.H, g);
  } else if (a.gate_kind == RMOE_GATE_FULL) {
    to_float<DT>(load_chunk<DT, kWide>(static_cast<const typename RowElem<DT>::T*>(a.gate) + t * a.H, c, a.H), g);
  } else {
    const float v = a.gate_kind == RMOE_GATE_ROW ? static_cast<const float*>(a.gate)[t] : 1.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) g[i] = v;
  }
}

template <int DT, int V, bool kWide>
__global__ __launch_bounds__(64 * kMaxWaves) void norm_kernel(NormArgs a, size_t first) {
  typedef typename RowElem<DT>::T E;
  __shared__ float slots[2][kMaxWaves][1];
  const size_t t = first + blockIdx.x;
  const int W = blockDim.x >> 6, wave = wave_id(), H = a.H;
  auto column = [&](int v) { return 8 * ((int)threadIdx.x + v * (int)blockDim.x); };
  auto row = [&](const void* p) { return static_cast<const E*>(p) + t * H; };
  float y[V][8];
  if (a.block) {
    Chunk<DT> r[V];
    float u[V][8], g[V][8];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = column(v);
      if (c < H) {
        to_float<DT>(load_chunk<DT, kWide>(row(a.block), c, H), u[v]);
        r[v] = load_chunk<DT, kWide>(row(a.residual), c, H);
        load_gate<DT, kWide>(a, t, c, g[v]);
      } else {
        r[v] = Chunk<DT>{};
#pragma unroll
        for (int i = 0; i < 8; ++i) u[v][i] = g[v][i] = 0.f;
      }
    }
    if (a.post) {
      float s[1] = {0.f};
#pragma unroll
      for (int v = 0; v < V; ++v)
#pragma unroll
        for (int i = 0; i < 8; ++i) s[0] = fmaf(u[v][i], u[v][i], s[0]);
      row_sum<1>(s, slots[0], wave, W);
      const float n = inv_rms(s[0], H, a.eps);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float w[8];
        load_vector(a.post, column(v), H, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) u[v][i] = u[v][i] * n * w[i];
      }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = column(v);
      Chunk<DT> o;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        o.v[i] = RowElem<DT>::put(fmaf(g[v][i], u[v][i], a.scale * RowElem<DT>::get(r[v].v[i])));
        y[v][i] = c + i < H ? RowElem<DT>::get(o.v[i]) : 0.f;
      }
      if (c < H) store_chunk<DT, kWide>(static_cast<E*>(a.y) + t * H, c, H, o);
    }
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if (column(v) < H) to_float<DT>(load_chunk<DT, kWide>(row(a.residual), column(v), H), y[v]);
      else
#pragma unroll
        for (int i = 0; i < 8; ++i) y[v][i] = 0.f;
    }
  }
  if (!a.h && !a.codes) return;
  float s[1] = {0.f};
#pragma unroll
  for (int v = 0; v < V; ++v)
#pragma unroll
    for (int i = 0; i < 8; ++i) s[0] = fmaf(y[v][i], y[v][i], s[0]);
  row_sum<1>(s, slots[1], wave, W);
  const float m = inv_rms(s[0], H, a.eps);
  const int P = (H + kMxBlock - 1) / kMxBlock * kMxBlock;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int c = column(v);
    float w[8], x[8];
    load_vector(a.pre, c, H, w);
    Chunk<DT> o;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      o.v[i] = RowElem<DT>::put(y[v][i] * m * w[i]);
      x[i] = c + i < H ? RowElem<DT>::get(o.v[i]) : 0.f;
    }
    if (a.h && c < H) store_chunk<DT, kWide>(static_cast<E*>(a.h) + t * H, c, H, o);
    if (a.codes) {
      uint32_t scale;
      const uint32_t q = mx_quantize8(x, scale);
      if (c < P) {
        *reinterpret_cast<uint32_t*>(a.codes + t * (P / 2) + c / 2) = q;
        if (c % kMxBlock == 0) a.scales[t * (P / kMxBlock) + c / kMxBlock] = (uint8_t)scale;
      }
    }
  }
}

// A workgroup takes the rows t = blockIdx.x, + gridDim.x, ...; each thread keeps its columns' shares of the
// weights' and the column gate's gradients and leaves them at work[which][blockIdx.x][H].
template <int DT, int V, bool kWide>
__global__ __launch_bounds__(64 * kMaxWaves) void norm_backward_kernel(NormGradArgs a) {
  typedef typename RowElem<DT>::T E;
  __shared__ float first_sums[2][kMaxWaves][3], second_sums[2][kMaxWaves][2];
  const int W = blockDim.x >> 6, wave = wave_id(), H = a.f.H;
  auto column = [&](int v) { return 8 * ((int)threadIdx.x + v * (int)blockDim.x); };
  float dpre[V][8], dpost[V][8], dgate[V][8];
#pragma unroll
  for (int v = 0; v < V; ++v)
#pragma unroll
    for (int i = 0; i < 8; ++i) dpre[v][i] = dpost[v][i] = dgate[v][i] = 0.f;
  const float inv_H = 1.0f / (float)H;
  int turn = 0;
  for (size_t t = blockIdx.x; t < (size_t)a.f.T; t += gridDim.x, turn ^= 1) {
    auto row = [&](const void* p) { return static_cast<const E*>(p) + t * H; };
    float b[V][8], y[V][8], d[V][8], dh[V][8];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = column(v);
      auto load = [&](const void* p, float (&f)[8]) {
        if (p && c < H) to_float<DT>(load_chunk<DT, kWide>(row(p), c, H), f);
        else
#pragma unroll
          for (int i = 0; i < 8; ++i) f[i] = 0.f;
      };
      load(a.f.block, b[v]);
      load(a.f.y, y[v]);
      load(a.dy, d[v]);
      load(a.dh, dh[v]);
    }
    float s[3] = {0.f, 0.f, 0.f};  // of b^2, y^2, a y
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float w[8];
      if (a.dh) load_vector(a.f.pre, column(v), H, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        s[0] = fmaf(b[v][i], b[v][i], s[0]);
        s[1] = fmaf(y[v][i], y[v][i], s[1]);
        if (a.dh) s[2] = fmaf(dh[v][i] * w[i], y[v][i], s[2]);
      }
    }
    row_sum<3>(s, first_sums[turn], wave, W);
    const float n = a.f.post ? inv_rms(s[0], H, a.f.eps) : 1.f;
    if (a.dh) {
      const float m = inv_rms(s[1], H, a.f.eps), k = s[2] * inv_H * m * m * m;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float w[8];
        load_vector(a.f.pre, column(v), H, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          d[v][i] += fmaf(dh[v][i] * w[i], m, -(y[v][i] * k));
          dpre[v][i] = fmaf(dh[v][i] * y[v][i], m, dpre[v][i]);
        }
      }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      Chunk<DT> o;
#pragma unroll
      for (int i = 0; i < 8; ++i) o.v[i] = RowElem<DT>::put(a.f.scale * d[v][i]);
      if (column(v) < H) store_chunk<DT, kWide>(static_cast<E*>(a.dresidual) + t * H, column(v), H, o);
    }
    if (!a.f.block) continue;
    float q[2] = {0.f, 0.f};  // of v b, and D u
    float w[V][8];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = column(v);
      float g[8];
      if (c < H) load_gate<DT, kWide>(a.f, t, c, g);
      else
#pragma unroll
        for (int i = 0; i < 8; ++i) g[i] = 0.f;
      if (a.f.post) load_vector(a.f.post, c, H, w[v]);
      else
#pragma unroll
        for (int i = 0; i < 8; ++i) w[v][i] = 1.f;
      Chunk<DT> o;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float bn = b[v][i] * n, dg = d[v][i] * (bn * w[v][i]);
        q[1] += dg;
        dgate[v][i] += dg;
        o.v[i] = RowElem<DT>::put(dg);
        d[v][i] *= g[i];  // du
        dpost[v][i] = fmaf(d[v][i], bn, dpost[v][i]);
        q[0] = fmaf(d[v][i] * w[v][i], b[v][i], q[0]);
      }
      if (a.f.gate_kind == RMOE_GATE_FULL && a.dgate && c < H)
        store_chunk<DT, kWide>(static_cast<E*>(a.dgate) + t * H, c, H, o);
    }
    if (a.f.post || a.f.gate_kind == RMOE_GATE_ROW) row_sum<2>(q, second_sums[turn], wave, W);
    if (a.f.gate_kind == RMOE_GATE_ROW && a.dgate && threadIdx.x == 0) static_cast<float*>(a.dgate)[t] = q[1];
    const float k = a.f.post ? q[0] * inv_H * n * n * n : 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      Chunk<DT> o;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        o.v[i] = RowElem<DT>::put(a.f.post ? fmaf(d[v][i] * w[v][i], n, -(b[v][i] * k)) : d[v][i]);
      if (column(v) < H) store_chunk<DT, kWide>(static_cast<E*>(a.dblock) + t * H, column(v), H, o);
    }
  }
  auto leave = [&](int which, float (&f)[V][8]) {
    float* p = a.work + ((size_t)which * gridDim.x + blockIdx.x) * H;
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (column(v) + i < H) p[column(v) + i] = f[v][i];
  };
  if (a.dpre) leave(0, dpre);
  if (a.dpost) leave(1, dpost);
  if (a.f.gate_kind == RMOE_GATE_COLUMN && a.dgate) leave(2, dgate);
}

// The columns' sums over the workgroups' shares, in their order: 64 columns a workgroup, a wave for each 16th.
__global__ __launch_bounds__(1024) void norm_columns_kernel(const float* __restrict__ work, int groups, int H,
                                                            float* dpre, float* dpost, float* dgate) {
  __shared__ float part[16][64];
  const int lane = threadIdx.x & 63, wave = wave_id(), c = (int)blockIdx.x * 64 + lane;
  float* out = blockIdx.y == 0 ? dpre : blockIdx.y == 1 ? dpost : dgate;
  if (!out) return;
  const float* p = work + (size_t)blockIdx.y * groups * H;
  float s = 0.f;
  if (c < H)
    for (int g = wave * groups / 16; g < (wave + 1) * groups / 16; ++g) s += p[(size_t)g * H + c];
  part[wave][lane] = s;
  __syncthreads();
  if (wave == 0 && c < H) {
    for (int w = 1; w < 16; ++w) s += part[w][lane];
    out[c] = s;
  }
}

bool wide_rows(int dtype, int H, std::initializer_list<const void*> ps) {
  uintptr_t at = 0;
  for (const void* p : ps) at |= reinterpret_cast<uintptr_t>(p);
  return at % 16 == 0 && H % 8 == 0 && (dtype == RMOE_DT_F32 || H * 2 % 16 == 0);
}

// Waves of a row of eight columns a thread, or of 16 where that takes more than kMaxWaves.
bool two_chunks(int H) { return H > 512 * kMaxWaves; }
int waves_for(int H) { return two_chunks(H) ? (H + 1023) / 1024 : (H + 511) / 512; }

template <int DT>
hipError_t norm_with(const NormArgs& a, hipStream_t st) {
  const bool wide = wide_rows(DT, a.H, {a.block, a.residual, a.y, a.h, a.gate_kind == RMOE_GATE_FULL ? a.gate : nullptr});
  const int W = waves_for(a.H);
  auto* kernel = two_chunks(a.H) ? (wide ? norm_kernel<DT, 2, true> : norm_kernel<DT, 2, false>)
                                 : (wide ? norm_kernel<DT, 1, true> : norm_kernel<DT, 1, false>);
  const size_t step = ((size_t)1 << 32) / (64 * W) - 1;
  for (size_t t = 0; t < (size_t)a.T; t += step) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)std::min(step, (size_t)a.T - t)), dim3(64 * W), 0, st, a, t);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

template <int DT>
hipError_t grad_with(const NormGradArgs& a, hipStream_t st) {
  const NormArgs& f = a.f;
  const bool full = f.gate_kind == RMOE_GATE_FULL;
  const bool wide = wide_rows(DT, f.H, {f.block, f.y, a.dy, a.dh, a.dblock, a.dresidual, full ? f.gate : nullptr,
                                        full ? a.dgate : nullptr});
  const int W = waves_for(f.H), groups = norm_groups(f.T);
  auto* kernel = two_chunks(f.H) ? (wide ? norm_backward_kernel<DT, 2, true> : norm_backward_kernel<DT, 2, false>)
                                 : (wide ? norm_backward_kernel<DT, 1, true> : norm_backward_kernel<DT, 1, false>);
  hipLaunchKernelGGL(kernel, dim3(groups), dim3(64 * W), 0, st, a);
  hipError_t e = hipGetLastError();
  float* column_gate = f.gate_kind == RMOE_GATE_COLUMN ? static_cast<float*>(a.dgate) : nullptr;
  if (e == hipSuccess && (a.dpre || a.dpost || column_gate)) {
    hipLaunchKernelGGL(norm_columns_kernel, dim3((f.H + 63) / 64, 3), dim3(1024), 0, st, a.work, groups, f.H, a.dpre,
                       a.dpost, column_gate);
    e = hipGetLastError();
  }
  return e;
}

}  // namespace

hipError_t launch_norm(const NormArgs& a, int dtype, hipStream_t st) {
  if (dtype == RMOE_DT_BF16) return norm_with<RMOE_DT_BF16>(a, st);
  if (dtype == RMOE_DT_F16) return norm_with<RMOE_DT_F16>(a, st);
  return norm_with<RMOE_DT_F32>(a, st);
}

hipError_t launch_norm_backward(const NormGradArgs& a, int dtype, hipStream_t st) {
  if (dtype == RMOE_DT_BF16) return grad_with<RMOE_DT_BF16>(a, st);
  if (dtype == RMOE_DT_F16) return grad_with<RMOE_DT_F16>(a, st);
  return grad_with<RMOE_DT_F32>(a, st);
}

}  // namespace rmoe
