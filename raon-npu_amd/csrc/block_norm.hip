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
// n and m are formed again from b and y, which have to be read in any case.  m a - y m^3 S / H, S = sum a y, is formed as
// m (a - (y m) (m S / H)), and db likewise: y m is at most sqrt(H) and m S / H at most max |a|, where m^3 leaves fp32 for
// rows past 2^42 and, with an eps as small, for those below 2^-42.
//
// Bound by HBM.  A row is held in the registers of W waves (eight columns a thread and V of these), which meet in
// LDS once for each sum: every element is read and written once.  6,700 rows of 2,560 in bf16 through both norms and a
// gate, 137 MB: 30 us, 4.6 TB/s, two copies of as many bytes 29.4; one row 3 us, a launch and a trip to memory.
// Their gradients: 4,099 rows of 2,048 in bf16, 101 MB, 28 us and 4 for the weights' sums over the workgroups; 4,099
// of 2,560 in fp32, 252 MB, 67 us together; 445 of 2,560 in fp32 13 and 4, where two rows a workgroup, one behind the
// other, are the time.
#include <algorithm>
#include <type_traits>

#include "mx.h"

namespace rmoe {
namespace {

constexpr int kMaxWaves = 8;  // of a workgroup: up to 256 registers a thread

// The sum over the wave's lanes, in every lane: exchanges within the vector unit up to 16 lanes, then the four
// sixteens' by scalar reads (six exchanges through LDS hardware take 0.3 us, these 0.1).
__device__ __forceinline__ float lanes_sum(float v) {
  auto moved = [](float x, auto control) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), decltype(control)::value, 0xF, 0xF, false));
  };
  v += moved(v, std::integral_constant<int, 0xB1>());   // lane ^ 1
  v += moved(v, std::integral_constant<int, 0x4E>());   // lane ^ 2
  v += moved(v, std::integral_constant<int, 0x141>());  // eight lanes mirrored
  v += moved(v, std::integral_constant<int, 0x140>());  // sixteen mirrored
  const int i = __float_as_int(v);
  return (__int_as_float(__builtin_amdgcn_readlane(i, 0)) + __int_as_float(__builtin_amdgcn_readlane(i, 16))) +
         (__int_as_float(__builtin_amdgcn_readlane(i, 32)) + __int_as_float(__builtin_amdgcn_readlane(i, 48)));
}

// Sums of N values over the W waves of a row, the first of which is wave `first` of the workgroup: a slot per wave;
// calls in turn use different slots, so that one barrier a call is enough (all the workgroup's waves make it).
template <int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float (*slots)[N], int wave, int first, int W) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = lanes_sum(v[i]);
  if (W == 1) return;
  if ((threadIdx.x & 63) == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) slots[wave][i] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = slots[first][i];
  for (int w = 1; w < W; ++w) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += slots[first + w][i];
  }
}

// The sum over a row of its chunks' of 512 columns, a wave's s[v] that of chunk v W + wave: each over the lanes, then in
// the chunks' order, so that no result depends on how many waves a row has.
template <int V>
__device__ __forceinline__ float chunks_sum(float (&s)[V], float* slots, int wave, int W) {
#pragma unroll
  for (int v = 0; v < V; ++v) s[v] = lanes_sum(s[v]);
  float sum;
  if (W == 1) {
    sum = s[0];
#pragma unroll
    for (int v = 1; v < V; ++v) sum += s[v];
  } else {
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int v = 0; v < V; ++v) slots[v * W + wave] = s[v];
    }
    __syncthreads();
    sum = slots[0];
    for (int i = 1; i < V * W; ++i) sum += slots[i];
  }
  return sum;
}

template <int DT>
__device__ __forceinline__ void to_float(const Chunk<DT>& c, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = RowElem<DT>::get(c.v[i]);
}

__device__ __forceinline__ float inv_rms(float squares, int H, float eps) {
  return 1.0f / sqrtf(squares / (float)H + eps);
}

// Where a thread's chunks of a row are.  Of aligned rows (kWide) the threads past the row's end repeat its last chunk,
// so that loads and stores are free of branches: they compute (and store) what its owner does, and take no part in sums.
template <int V, bool kWide>
struct Columns {
  int first, step, H;
  __device__ __forceinline__ Columns(int thread, int W, int H) : first(8 * thread), step(512 * W), H(H) {}
  __device__ __forceinline__ int raw(int v) const { return first + v * step; }
  __device__ __forceinline__ int at(int v) const { return kWide ? min(raw(v), H - 8) : raw(v); }
  __device__ __forceinline__ bool counts(int v, int i) const { return kWide ? raw(v) < H : raw(v) + i < H; }
};

template <int DT, bool kOnce = false, int V, bool kWide>
__device__ __forceinline__ void load_row(const void* rows, size_t t, const Columns<V, kWide>& c, Chunk<DT> (&o)[V]) {
  const auto* p = static_cast<const typename RowElem<DT>::T*>(rows) + t * c.H;
#pragma unroll
  for (int v = 0; v < V; ++v) o[v] = load_chunk<DT, kWide, kOnce>(p, c.at(v), c.H);
}
// With one chunk a thread the repeating threads are in their owner's wave, whose loads and stores of an address keep
// their order; with two they may be in another, which would read a row that is written in place too late: they do not
// store.
template <int DT, int V, bool kWide>
__device__ __forceinline__ void store_row(void* rows, size_t t, const Columns<V, kWide>& c, int v, const Chunk<DT>& o) {
  if constexpr (V > 1)
    if (!c.counts(v, 0)) return;
  store_chunk<DT, kWide>(static_cast<typename RowElem<DT>::T*>(rows) + t * c.H, c.at(v), c.H, o);
}
// A thread's columns of an fp32 vector of H, or ones where there is none.  Of aligned rows without a branch: the
// vector is a buffer of 4 H bytes, or of none, past whose end the hardware reads zeros.  (With a branch the values are
// waited for where it ends, before anything behind it is requested: 6,700 rows of 2,560 took 50 us and not 35.)
template <int V, bool kWide>
__device__ __forceinline__ void load_columns(const float* p, const Columns<V, kWide>& c, float (&f)[V][8]) {
  if constexpr (kWide) {
    const auto buffer = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(p), 0, p ? 4 * c.H : 0, 0x00027000);
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int i = 0; i < 8; i += 4) {
        const u32x4_t q = __builtin_amdgcn_raw_buffer_load_b128(buffer, 4 * (c.at(v) + i), 0, 0);
#pragma unroll
        for (int k = 0; k < 4; ++k) f[v][i + k] = __uint_as_float(p ? q[k] : 0x3f800000u);
      }
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int i = 0; i < 8; ++i) f[v][i] = p && c.raw(v) + i < c.H ? p[c.raw(v) + i] : 1.f;
  }
}

// A workgroup is blockDim / (64 W) rows; more than one only of one wave each.
template <int DT, int V, bool kWide, bool kBlock, bool kFull, bool kOnce>
__global__ __launch_bounds__(64 * kMaxWaves) void norm_kernel(NormArgs a, int W, size_t first) {
  __shared__ float slots[2][kNormMaxWidth / 512 + kMaxWaves];  // the last chunks may be none
  const int wave = wave_id(), H = a.H, group = wave / W;
  const size_t t = first + (size_t)blockIdx.x * ((blockDim.x >> 6) / W) + group;
  if (t >= (size_t)a.T) return;
  const Columns<V, kWide> col((int)threadIdx.x - 64 * W * group, W, H);
  Chunk<DT> b[V], r[V], fg[V];
  if constexpr (kBlock) load_row<DT, kOnce>(a.block, t, col, b);
  load_row<DT, kOnce>(a.residual, t, col, r);
  if constexpr (kFull) load_row<DT>(a.gate, t, col, fg);
  float g[V][8], post[V][8], pre[V][8], y[V][8];
  load_columns(a.post, col, post);
  load_columns(a.gate_kind == RMOE_GATE_COLUMN ? static_cast<const float*>(a.gate) : nullptr, col, g);
  load_columns(a.pre, col, pre);
  if constexpr (kBlock) {
    float u[V][8];
#pragma unroll
    for (int v = 0; v < V; ++v) to_float<DT>(b[v], u[v]);
    const float one = a.gate_kind == RMOE_GATE_ROW ? static_cast<const float*>(a.gate)[t] : 1.f;
    if (a.post) {
      float s[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        s[v] = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (col.counts(v, i)) s[v] = fmaf(u[v][i], u[v][i], s[v]);
      }
      const float n = inv_rms(chunks_sum<V>(s, slots[0], wave, W), H, a.eps);
#pragma unroll
      for (int v = 0; v < V; ++v)
#pragma unroll
        for (int i = 0; i < 8; ++i) u[v][i] = u[v][i] * n * post[v][i];
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if constexpr (kFull) to_float<DT>(fg[v], g[v]);
      Chunk<DT> o;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        o.v[i] = RowElem<DT>::put(fmaf(g[v][i] * one, u[v][i], a.scale * RowElem<DT>::get(r[v].v[i])));
        y[v][i] = RowElem<DT>::get(o.v[i]);
      }
      store_row<DT>(a.y, t, col, v, o);
    }
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) to_float<DT>(r[v], y[v]);
  }
  if (!a.pre) return;
  float s[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    s[v] = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (col.counts(v, i)) s[v] = fmaf(y[v][i], y[v][i], s[v]);
  }
  const float m = inv_rms(chunks_sum<V>(s, slots[1], wave, W), H, a.eps);
  const int P = (H + kMxBlock - 1) / kMxBlock * kMxBlock;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    float x[8];
    Chunk<DT> o;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      o.v[i] = RowElem<DT>::put(y[v][i] * m * pre[v][i]);
      x[i] = col.counts(v, i) ? RowElem<DT>::get(o.v[i]) : 0.f;
    }
    if (a.h) store_row<DT>(a.h, t, col, v, o);
    if (a.codes) {
      const int c = col.raw(v);
      uint32_t scale;
      const uint32_t q = mx_quantize8(x, scale);
      if (c < P) {
        *reinterpret_cast<uint32_t*>(a.codes + t * (P / 2) + c / 2) = q;
        if (c % kMxBlock == 0) a.scales[t * (P / kMxBlock) + c / kMxBlock] = (uint8_t)scale;
      }
    }
  }
}

// A workgroup's waves are blockDim / (64 W) rows at a time, the first ones at blockIdx.x times as many, then
// gridDim.x times as many further, ...; each thread keeps its columns' shares of the weights' and the column gate's
// gradients, which the workgroup adds up in LDS at the end and leaves at work[which][blockIdx.x][H].  The next row is
// under way while one is worked on (one chunk a thread; with two there are no registers for it): its loads come before
// the row's stores and nothing else is loaded, for a wait for loads is one for every load and store before them.
template <int DT, int V, bool kWide, bool kBlock, bool kFull>
__global__ __launch_bounds__(64 * kMaxWaves, 2) void norm_backward_kernel(NormGradArgs a, int W) {
  __shared__ float first_sums[2][kMaxWaves][3], second_sums[2][kMaxWaves][2];
  __shared__ __attribute__((aligned(16))) float shares[kMaxWaves][512];
  const int wave = wave_id(), H = a.f.H, groups = (int)(blockDim.x >> 6) / W, group = wave / W, own = W * group;
  const Columns<V, kWide> col((int)threadIdx.x - 64 * own, W, H);
  const bool by_row = kBlock && a.f.gate_kind == RMOE_GATE_ROW;
  float pre[V][8], post[V][8], gate[V][8], dpre[V][8], dpost[V][8], dgate[V][8];
  load_columns(a.f.pre, col, pre);
  load_columns(kBlock ? a.f.post : nullptr, col, post);
  load_columns(kBlock && a.f.gate_kind == RMOE_GATE_COLUMN ? static_cast<const float*>(a.f.gate) : nullptr, col, gate);
#pragma unroll
  for (int v = 0; v < V; ++v)
#pragma unroll
    for (int i = 0; i < 8; ++i) dpre[v][i] = dpost[v][i] = dgate[v][i] = 0.f;
  const float inv_H = 1.0f / (float)H;

  struct Row {
    Chunk<DT> b[V], y[V], d[V], h[V], g[V];
    float one;
  };
  // Operands that are not given read y, and count for nothing.
  const void *pd = a.dy ? a.dy : a.f.y, *ph = a.dh ? a.dh : a.f.y;
  const float* prow = by_row ? static_cast<const float*>(a.f.gate) : nullptr;
  auto load = [&](Row& q, size_t t) {
    t = min(t, (size_t)a.f.T - 1);
    if constexpr (kBlock) load_row<DT>(a.f.block, t, col, q.b);
    load_row<DT>(a.f.y, t, col, q.y);
    load_row<DT>(pd, t, col, q.d);
    load_row<DT>(ph, t, col, q.h);
    if constexpr (kFull) load_row<DT>(a.f.gate, t, col, q.g);
    if constexpr (kBlock) q.one = prow ? prow[t] : 1.f;
  };
  auto work = [&](const Row& now, size_t t, bool live, int turn) {
    float b[V][8], y[V][8], d[V][8], dh[V][8];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if constexpr (kBlock) to_float<DT>(now.b[v], b[v]);
      to_float<DT>(now.y[v], y[v]);
      to_float<DT>(now.d[v], d[v]);
      to_float<DT>(now.h[v], dh[v]);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (!a.dy) d[v][i] = 0.f;
        if (!a.dh) dh[v][i] = 0.f;
      }
    }
    float s[3] = {0.f, 0.f, 0.f};  // of b^2, y^2, a y
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (col.counts(v, i)) {
          if constexpr (kBlock) s[0] = fmaf(b[v][i], b[v][i], s[0]);
          s[1] = fmaf(y[v][i], y[v][i], s[1]);
          s[2] = fmaf(dh[v][i] * pre[v][i], y[v][i], s[2]);
        }
    row_sum<3>(s, first_sums[turn], wave, own, W);
    const float n = kBlock && a.f.post ? inv_rms(s[0], H, a.f.eps) : 1.f;
    if (a.dh) {
      const float m = inv_rms(s[1], H, a.f.eps), k = s[2] * inv_H * m;
#pragma unroll
      for (int v = 0; v < V; ++v)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float ym = y[v][i] * m;
          d[v][i] = fmaf(fmaf(-ym, k, dh[v][i] * pre[v][i]), m, d[v][i]);
          const float p = fmaf(dh[v][i], ym, dpre[v][i]);
          dpre[v][i] = live ? p : dpre[v][i];
        }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      Chunk<DT> o;
#pragma unroll
      for (int i = 0; i < 8; ++i) o.v[i] = RowElem<DT>::put(a.f.scale * d[v][i]);
      if (live) store_row<DT>(a.dresidual, t, col, v, o);
    }
    if constexpr (kBlock) {
      float q[2] = {0.f, 0.f};  // of v b, and D u
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float g[8];
        if constexpr (kFull) to_float<DT>(now.g[v], g);
        Chunk<DT> o;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float bn = b[v][i] * n, dg = d[v][i] * (bn * post[v][i]);
          o.v[i] = RowElem<DT>::put(dg);
          d[v][i] *= kFull ? g[i] : gate[v][i] * now.one;  // du
          if (col.counts(v, i)) {
            q[0] = fmaf(d[v][i] * post[v][i], b[v][i], q[0]);
            q[1] += dg;
          }
          const float p = fmaf(d[v][i], bn, dpost[v][i]), c = dgate[v][i] + dg;
          dpost[v][i] = live ? p : dpost[v][i];
          dgate[v][i] = live ? c : dgate[v][i];
        }
        if constexpr (kFull)
          if (a.dgate && live) store_row<DT>(a.dgate, t, col, v, o);
      }
      if (a.f.post || by_row) row_sum<2>(q, second_sums[turn], wave, own, W);
      if (by_row && a.dgate && col.first == 0 && live) static_cast<float*>(a.dgate)[t] = q[1];
      const float k = q[0] * inv_H * n;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        Chunk<DT> o;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          o.v[i] = RowElem<DT>::put(a.f.post ? fmaf(-(b[v][i] * n), k, d[v][i] * post[v][i]) * n : d[v][i]);
        if (live) store_row<DT>(a.dblock, t, col, v, o);
      }
    }
  };

  const size_t T = (size_t)a.f.T, step = (size_t)gridDim.x * groups;
  size_t t = (size_t)blockIdx.x * groups;
  int turn = 0;
  Row now;
  if constexpr (V == 1) {
    Row ahead;
    load(now, t + group);
    for (; t + groups <= T; t += step, turn ^= 1) {
      load(ahead, t + step + group);
      work(now, t + group, true, turn);
      now = ahead;
    }
    if (t < T) work(now, t + group, t + group < T, turn);
  } else {
    for (; t < T; t += step, turn ^= 1) {
      load(now, t + group);
      work(now, t + group, t + group < T, turn);
    }
  }

  auto leave = [&](int which, float (&f)[V][8]) {
    float* p = a.work + ((size_t)which * gridDim.x + blockIdx.x) * H;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      __syncthreads();
      *reinterpret_cast<float4*>(&shares[wave][8 * (threadIdx.x & 63)]) = *reinterpret_cast<float4*>(f[v]);
      *reinterpret_cast<float4*>(&shares[wave][8 * (threadIdx.x & 63) + 4]) = *reinterpret_cast<float4*>(f[v] + 4);
      __syncthreads();
      for (int i = threadIdx.x; i < 512 * W; i += blockDim.x) {
        const int c = 512 * W * v + i;
        float s = shares[i / 512][i % 512];
        for (int g = 1; g < groups; ++g) s += shares[g * W + i / 512][i % 512];
        if (c < H) p[c] = s;
      }
    }
  };
  if (a.dpre) leave(0, dpre);
  if constexpr (kBlock) {
    if (a.dpost) leave(1, dpost);
    if (a.f.gate_kind == RMOE_GATE_COLUMN && a.dgate) leave(2, dgate);
  }
}

// The columns' sums over the workgroups' shares, in their order: 64 columns a workgroup, a wave for each 16th of the
// shares, of which kLoads are under way at once.
__global__ __launch_bounds__(1024) void norm_columns_kernel(const float* __restrict__ work, int groups, int H,
                                                            float* dpre, float* dpost, float* dgate) {
  __shared__ float part[16][64];
  constexpr int kLoads = 16;
  const int lane = threadIdx.x & 63, wave = wave_id(), c = (int)blockIdx.x * 64 + lane;
  float* out = blockIdx.y == 0 ? dpre : blockIdx.y == 1 ? dpost : dgate;
  if (!out) return;
  const float* p = work + (size_t)blockIdx.y * groups * H + min(c, H - 1);
  const int end = (wave + 1) * groups / 16;
  float s = 0.f;
  for (int g = wave * groups / 16; g < end; g += kLoads) {
    float v[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) v[i] = g + i < end ? p[(size_t)(g + i) * H] : 0.f;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) s += v[i];
  }
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

template <int DT>
hipError_t norm_with(const NormArgs& a, hipStream_t st) {
  const bool wide = wide_rows(DT, a.H, {a.block, a.residual, a.y, a.h, a.gate_kind == RMOE_GATE_FULL ? a.gate : nullptr});
  // Block and residual of 6,700 rows of 2,560 (69 MB): 34.7 us, read past the caches' order 32.2; of 2,000 rows, which
  // are in the caches from the call before, 11.4 and 12.2.
  const bool once = wide && (size_t)a.T * a.H * sizeof(typename RowElem<DT>::T) * (a.block ? 2 : 1) >= kOnceBytes;
  // A row to as many waves as it has chunks for, or of many rows to one wave, or two or four, of up to kManyChunks a
  // thread: more bytes under way on each CU, fewer waves that meet.  6,700 rows in bf16 through both norms and a gate: of
  // 2,048 25.6 us and 26.8 in as many waves, of 2,560 30.1 and 32, of 4,096 48 and 49.7; in fp32 of 2,560 58.4 and 63.4; a
  // norm alone into codes of 2,560 12.3 and 15, of 2,048 10.5 and 11.3.  1,500 rows of 2,560 9.4 and 8.9, a norm alone 5.0
  // and 5.3; 1,000 rows alone 3.9 and 4.0, one row 3.0 and 2.4.  Without a norm after the block 6,700 rows of 2,560 take
  // 27.7 and 25, with a gate by element 34.8 and 34.1.
  constexpr int kManyRows = 3000, kManyAlone = 1500, kManyChunks = 5;
  const bool many = wide && (a.block ? a.post && a.gate_kind != RMOE_GATE_FULL && a.T >= kManyRows : a.T >= kManyAlone);
  int V = a.H > 512 * kMaxWaves ? 2 : 1, W = (a.H + 512 * V - 1) / (512 * V);
  if (many) {
    for (W = 1; a.H > 512 * kManyChunks * W;) W *= 2;
    V = (a.H + 512 * W - 1) / (512 * W);
  }
  const int rows = W == 1 && !many ? 4 : 1;
  auto at = [&](auto block, auto full, auto chunks) {
    constexpr bool B = decltype(block)::value, F = decltype(full)::value;
    constexpr int N = decltype(chunks)::value;
    if constexpr (N <= 2)
      if (!wide) return norm_kernel<DT, N, false, B, F, false>;
    return once ? norm_kernel<DT, N, true, B, F, true> : norm_kernel<DT, N, true, B, F, false>;
  };
  auto pick = [&](auto block, auto full) {
    const std::integral_constant<int, 1> one;
    const std::integral_constant<int, 2> two;
    if constexpr (!decltype(full)::value) {
      if (V == 3) return at(block, full, std::integral_constant<int, 3>());
      if (V == 4) return at(block, full, std::integral_constant<int, 4>());
      if (V == 5) return at(block, full, std::integral_constant<int, 5>());
    }
    return V == 1 ? at(block, full, one) : at(block, full, two);
  };
  auto* kernel = a.gate_kind == RMOE_GATE_FULL ? pick(std::true_type(), std::true_type())
                 : a.block                     ? pick(std::true_type(), std::false_type())
                                               : pick(std::false_type(), std::false_type());
  const size_t step = (((size_t)1 << 32) / (64 * W * rows) - 1) * rows;
  for (size_t t = 0; t < (size_t)a.T; t += step) {
    const size_t n = std::min(step, (size_t)a.T - t);
    hipLaunchKernelGGL(kernel, dim3((unsigned)((n + rows - 1) / rows)), dim3(64 * W * rows), 0, st, a, W, t);
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
  const int V = f.H > 512 * kMaxWaves ? 2 : 1;
  const int W = (f.H + 512 * V - 1) / (512 * V), rows = kMaxWaves / W;
  const int groups = std::min((f.T + rows - 1) / rows, norm_groups(f.T));
  auto pick = [&](auto block, auto full) {
    constexpr bool B = decltype(block)::value, F = decltype(full)::value;
    return V == 1 ? (wide ? norm_backward_kernel<DT, 1, true, B, F> : norm_backward_kernel<DT, 1, false, B, F>)
                  : (wide ? norm_backward_kernel<DT, 2, true, B, F> : norm_backward_kernel<DT, 2, false, B, F>);
  };
  auto* kernel = full      ? pick(std::true_type(), std::true_type())
                 : f.block ? pick(std::true_type(), std::false_type())
                           : pick(std::false_type(), std::false_type());
  hipLaunchKernelGGL(kernel, dim3(groups), dim3(64 * W * rows), 0, st, a, W);
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
