// y[n, M'] = RTNE(act(x[n, K] @ W^T + bias) + residual) of microscaled 4-bit rows and weights (mx.h), of one
// matrix or of each row's expert, on the scaled MFMA: codes and scale bytes go into the matrix pipes as they are
// held, products are exact, sums fp32.
//
// Few rows are bound by the weights' bytes: 4 rows of [260096, 2560] read 354 MB in 66.7 us, 5.3 TB/s (a large copy
// reaches 4.9, a large write 6.8); the smallest calls by the way from a launch to the first weights and back, 4.3 us
// for one row of [1536, 2048].  Many rows are bound by the matrix pipes and what feeds them: 6,700 gated rows of
// [24064, 2560] take 243 to 250 us (medians on several cards; single runs from 232), 3.3 to 3.4 PFLOP/s, 8,192^3 takes
// 269 to 275, 4.0 to 4.1 (the instruction alone, from registers, reaches 6.1 at the power that the card allows; the
// library's bf16 product 1.2).
#include <algorithm>
#include <type_traits>

#include "linear_act.h"
#include "mx.h"

namespace rmoe {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kFp4 = 4;         // the instruction's number of the e2m1 format, for both operands
constexpr int kScaleOne = 127;  // a scale byte of 2^0

// Codes as the instruction's operand: its upper half belongs to the wider formats.
__device__ __forceinline__ i32x8 operand(const i32x4& v) { return i32x8{v.x, v.y, v.z, v.w, 0, 0, 0, 0}; }

// g sigmoid(g) u with q = exp(g): q / (1 + q) takes an exponential and a reciprocal, few others.  The exponential of half
// the argument is squared, so that results down to fp32's subnormal ones are formed (the instruction itself gives 0 for
// those); past exp(87) the quotient is 1.  exp(g) is off by (4 + |g|) 2^-23 of it.
__device__ __forceinline__ float swiglu(float g, float u) {
  const float p = __builtin_amdgcn_exp2f(fminf(g * 0.72134752044448170f, 63.f)), q = p * p;
  return g * (q * recip(1.0f + q)) * u;
}

// bf16 bits of v (RTNE), by the conversion instruction.
__device__ __forceinline__ uint32_t bf16_bits(float v) { return __builtin_bit_cast(uint16_t, (__bf16)v); }

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
        z[k] = act == RMOE_ACT_SWIGLU ? swiglu(z[k], u[k]) : act_pair(RMOE_ACT_SITU, z[k], u[k], gb, vb);
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

// Scale bytes at .. at + 15 of a row of kb; those past its end are anything.
__device__ __forceinline__ uint4 load_scales(const uint8_t* row, int at, int kb) {
  uint4 v = make_uint4(0u, 0u, 0u, 0u);
  if (at + 16 <= kb) {
    __builtin_memcpy(&v, row + at, 16);
    return v;
  }
  uint32_t d[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int b = at + 4 * i;
    if (b + 4 <= kb) {
      __builtin_memcpy(&d[i], row + b, 4);
    } else if (b < kb) {
#pragma unroll
      for (int k = 0; k < 3; ++k) d[i] |= (uint32_t)row[min(b + k, kb - 1)] << (8 * k);
    }
  }
  return make_uint4(d[0], d[1], d[2], d[3]);
}

// ------------------------------------------------------------------ few rows --
// Tiles of 16 rows of x.  A wave takes NA fragments of 16 weight rows; the workgroup's four waves are WR
// stripes of them by WK = 4 / WR parts of K, whose sums meet in LDS and are added in their order: with one row the card
// has few workgroups, and shares of K are what keeps enough bytes under way.  Codes go from memory into the operands'
// registers, 16 bytes a lane, for no wave reads another's weights (of large matrices from three rows on LDS tiles are
// the faster ones all the same: more bytes under way for their registers).  Windows of four steps, the next one
// requested ahead: 32 rows of 128 experts' gated [1536, 2048] take 12.1 us, step by step 16.8; one row of [260096, 2560]
// takes 64 to 66.  A gated stripe holds 8 NA gate rows, then the up rows of the same outputs.
template <int NA, int WR, bool kGated>
__global__ __launch_bounds__(256) void mx_few_kernel(MxLin a, int n_nt) {
  constexpr int WK = 4 / WR, kRows = 16 * NA, kOut = kGated ? kRows / 2 : kRows, kStride = kRows + 4;
  __shared__ __attribute__((aligned(16))) float sums[4][16 * kStride];
  RowTiles<16> rt;
  const int n_mt = a.offsets ? rt.total(a.offsets, a.n_experts, a.n) : (a.n + 15) / 16;
  // XCD x takes a contiguous eighth of the tiles, the row tiles of one weight tile (by expert: the weight
  // tiles of one row tile) back to back.
  const uint32_t total = (uint32_t)n_mt * n_nt, per = (total + 7) / 8, slot = blockIdx.x / 8;  // a launch's fit 24 bits
  const uint32_t id = blockIdx.x % 8 * per + slot;
  if (slot >= per || id >= total) return;
  int nt, e = 0, row0, nrow;
  if (a.offsets) {
    rt.find((int)(id / (uint32_t)n_nt), e, row0, nrow);
    nt = (int)(id % (uint32_t)n_nt);
  } else {
    nt = (int)(id / (uint32_t)n_mt);
    row0 = (int)(id % (uint32_t)n_mt) * 16;
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
  // Four steps (512 columns) at once, the next four requested before these are used.  Steps past the wave's part
  // repeat its last one and are not used; blocks past the row's end repeat its last one as zeros.
  struct Window {
    i32x4 w[NA][4], x[4];
    uint4 ws[NA], xs;
  };
  auto load = [&](Window& q, int s) {
    size_t at[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) at[i] = (size_t)min(4 * min(s + i, s1 - 1) + lq, kb - 1) * 16;
#pragma unroll
    for (int f = 0; f < NA; ++f) {
#pragma unroll
      for (int i = 0; i < 4; ++i) q.w[f][i] = *reinterpret_cast<const i32x4*>(wp[f] + at[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) q.x[i] = *reinterpret_cast<const i32x4*>(xp + at[i]);
#pragma unroll
    for (int f = 0; f < NA; ++f) q.ws[f] = load_scales(wsp[f], 4 * s, kb);
    q.xs = load_scales(xsp, 4 * s, kb);
  };
  auto work = [&](Window& q, int s) {
    const uint32_t xs[4] = {q.xs.x, q.xs.y, q.xs.z, q.xs.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (s + i >= s1) break;
      const bool in = 4 * (s + i) + lq < kb;
      const int xsc = in ? (int)(xs[i] >> (8 * lq)) : kScaleOne;
      if (!in) q.x[i] = i32x4{0, 0, 0, 0};
#pragma unroll
      for (int f = 0; f < NA; ++f) {
        const uint32_t ws[4] = {q.ws[f].x, q.ws[f].y, q.ws[f].z, q.ws[f].w};
        const int wsc = in ? (int)(ws[i] >> (8 * lq)) : kScaleOne;
        acc[f] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(operand(q.w[f][i]), operand(q.x[i]), acc[f], kFp4, kFp4, 0,
                                                                  wsc, 0, xsc);
      }
    }
  };
  if (s0 < s1) {
    Window now, ahead;
    load(now, s0);
    int s = s0;
    for (; s + 4 < s1; s += 4) {
      load(ahead, s + 4);
      work(now, s);
      now = ahead;
    }
    work(now, s);
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

// The launch that serves a call: `fits` says whether its threads are within the 2^32 that a launch takes.
struct Plan {
  void (*kernel)(MxLin, int);
  size_t grid;
  unsigned threads;
  size_t lds;
  int n_nt;
  bool fits;
};

template <int NA, int WR>
Plan plan_few(const MxLin& a) {
  const bool gated = act_gated(a.act);
  const int width = gated ? a.M / 2 : a.M, out = 16 * NA * WR / (gated ? 2 : 1), n_nt = (width + out - 1) / out;
  const size_t mt = a.offsets ? std::min<size_t>(a.n, (size_t)a.n / 16 + a.n_experts) : ((size_t)a.n + 15) / 16;
  const size_t grid = 8 * ((mt * n_nt + 7) / 8);
  auto* kernel = gated ? mx_few_kernel<NA, WR, true> : mx_few_kernel<NA, WR, false>;
  return Plan{kernel, grid, 256, 0, n_nt, grid * 256 < (size_t)1 << 32};
}

// ----------------------------------------------------------------- many rows --
// Tiles of 32 MA WA weight rows by 32 NB WB rows of x; a wave takes 32 MA by 32 NB of them as 32 x 32 MFMAs
// of 64 columns.  Codes are copied to LDS past the registers, ahead of their use.  Where K is whole windows of 512
// columns (kWhole), in two stages of 256 columns, 128 bytes a row, and the scale bytes of a window likewise, 16 a row;
// else in three of 128 columns, and scale bytes are fetched by the registers and put beside a stage's codes, a dword a
// row (pieces of 128 bytes a row are the cheaper ones: in stages of 128 columns 8,192^3 took 345 us, now 270; 40,200
// rows of 128 experts' [2560, 1088] take 197 us, of K = 1024 144).  A
// lane's row of a fragment is lane % 32, and of the four blocks of 128 columns it holds 2 h and 2 h + 1, h = lane / 32,
// for two MFMA steps.  A gated wave's rows are 16 MA gate rows and the up rows of the same outputs.
//
// kStays: a workgroup takes tile after tile and requests the next one's first stage before it finishes one, as many
// workgroups as CUs.  In turn: 6,700 gated rows of [24064, 2560] 249 us, with a workgroup a tile 257; 53,600 rows of 128
// experts' gated [1536, 2048] 145 and 152; 8,192^3 275 and 278.  What is left between tiles is their activation and
// stores, some fifth of the time: all the waves are at them at once, for the sums of a second tile have no registers.
// SiTU's divisions and exponentials make it more: the 6,700 rows take 309 us with it, the 53,600 184.

template <int MA, int NB, int WA, int WB, bool kWhole, bool kStays>
struct TileShape {
  static_assert(kWhole || !kStays, "whole windows are two stages or more of an even number");
  static constexpr int KT = kWhole ? 2 : 1;
  static constexpr int kWaves = WA * WB, kThreads = 64 * kWaves, BW = 32 * MA * WA, BT = 32 * NB * WB, R = BW + BT;
  static constexpr int kStages = kWhole ? 2 : 3, kRow = 64 * KT;
  // A stage's codes, behind them a dword of scales a row, or behind the first stage's alone a window of scales.
  static constexpr int kCodes = R * kRow, kStage = kCodes + R * (kWhole ? 16 : 4);
  static constexpr int kCopyRows = 16 / KT;                            // rows of a copy
  static constexpr int kCopies = R / kCopyRows / kWaves;               // a wave's copies of a stage
  static constexpr int kScaleCopies = (R / 64 + kWaves - 1) / kWaves;  // and of a window of scales, 64 rows each
  static constexpr int kScales = (R + kThreads - 1) / kThreads;
  static_assert(KT == 1 || kCopies % 2 == 0, "the parity of a copy's rows is its number's");
  static_assert(R % 64 == 0 && R % (kCopyRows * kWaves) == 0, "whole copies");
  // Outputs of a wave, how many of them are in LDS at once (32 rows of them), and where.
  static constexpr int outputs(bool gated) { return (gated ? 16 : 32) * MA; }
  static constexpr int part(bool gated) { return kStays && outputs(gated) > 64 ? 64 : outputs(gated); }
  static constexpr int kOutputs = kStays ? kStage : 0;
  static constexpr int kTiles = kOutputs + kWaves * 32 * 68 * 4;  // the experts' table of row tiles (kStays)
  static constexpr size_t lds(bool gated) {
    const size_t out = kOutputs + (size_t)kWaves * 32 * (part(gated) + 4) * 4 + (kStays ? 64 * sizeof(RowTiles<BT>) : 0);
    const size_t in = (size_t)(kStages - 1) * kStage + kCodes + (kWhole ? 0 : R * 4);
    return out > in ? out : in;
  }
};

// 16 bytes a lane from base + offset to LDS at `lds` + 16 lane.
__device__ __forceinline__ void copy16(const void* base, uint32_t offset, uint32_t lds) {
  uint32_t saved;
  asm volatile(
      "s_mov_b32 %0, m0\n\t"
      "s_mov_b32 m0, %3\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %1, %2\n\t"
      "s_mov_b32 m0, %0"
      : "=&s"(saved)
      : "v"(offset), "s"(base), "s"(__builtin_amdgcn_readfirstlane(lds))
      : "memory");
}
// All but this wave's last kPending copies have landed, then the workgroup meets.
template <int kPending>
__device__ __forceinline__ void copies_landed() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kPending) : "memory");
  __syncthreads();
}

template <int MA, int NB, int WA, int WB, bool kWhole, bool kStays, bool kGated>
__global__ __launch_bounds__(64 * WA * WB, 2) void mx_tiles_kernel(MxLin a, int n_nt) {
  typedef TileShape<MA, NB, WA, WB, kWhole, kStays> S;
  constexpr int KT = S::KT;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  constexpr int kOut = S::outputs(kGated), kPart = S::part(kGated);
  RowTiles<S::BT> rt;
  const int n_mt = a.offsets ? rt.total(a.offsets, a.n_experts, a.n) : (a.n + S::BT - 1) / S::BT;
  // XCD x takes a contiguous eighth of the tiles: by expert the weight tiles of a row tile back to back, else
  // blocks of up to eight row tiles for each weight tile, so that both operands' tiles meet again in its L2.
  const uint32_t total = (uint32_t)n_mt * n_nt, per = (total + 7) / 8;  // a launch's fit 24 bits
  struct Tile {
    int nt, e, row0, nrow;
  };
  auto tile_at = [&](uint32_t slot, Tile& q) {  // false: there are no more
    const uint32_t id = blockIdx.x % 8 * per + slot;
    if (slot >= per || id >= total) return false;
    q.e = 0;
    if (a.offsets) {
      rt.find((int)(id / (uint32_t)n_nt), q.e, q.row0, q.nrow);
      q.nt = (int)(id % (uint32_t)n_nt);
    } else {
      constexpr uint32_t kBlock = 8;
      const uint32_t group = id / (kBlock * n_nt), m0 = group * kBlock, nm = min(kBlock, n_mt - m0);
      const uint32_t in = id - group * kBlock * n_nt;
      q.nt = (int)(in / nm);
      q.row0 = (int)(m0 + in % nm) * S::BT;
      q.nrow = min(S::BT, a.n - q.row0);
    }
    return true;
  };
  uint32_t slot = blockIdx.x / 8;
  Tile tile;
  if (!tile_at(slot, tile)) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = wave_id(), l32 = lane & 31, h = lane >> 5;
  const int wa = wave % WA, wb = wave / WA;
  const int kb = a.K / kMxBlock, tiles = (kb + 3) / 4, stages = tiles / KT, rem = kb % 4;
  uint32_t ldb = (uint32_t)a.K / 2;
  const int width = kGated ? a.M / 2 : a.M;
  // Row of an LDS row slot: of the weights (e's matrix) or of x; rows past the ends repeat the last one.
  auto weight_row = [&](const Tile& q, int r) {
    const int w = r / (32 * MA), rr = r % (32 * MA), o = (q.nt * WA + w) * kOut + rr % kOut;
    return (kGated && rr >= kOut ? width : 0) + min(o, width - 1);
  };
  auto token_row = [&](const Tile& q, int r) { return min(r - S::BW, q.nrow - 1); };

  // A copy's first row, and how many rows behind it there are: those past them repeat the last one.
  const uint8_t* cbase[S::kCopies];
  int cmore[S::kCopies];
  auto aim_copies = [&](const Tile& q) {
#pragma unroll
    for (int j = 0; j < S::kCopies; ++j) {
      const int r0 = S::kCopyRows * (wave * S::kCopies + j);
      if (r0 < S::BW) {
        const int o = (q.nt * WA + r0 / (32 * MA)) * kOut + r0 % (32 * MA) % kOut;
        cbase[j] = a.w + ((size_t)q.e * a.M + weight_row(q, r0)) * ldb;
        cmore[j] = max(width - 1 - o, 0);
      } else {
        cbase[j] = a.x + ((size_t)q.row0 + token_row(q, r0)) * ldb;
        cmore[j] = max(q.nrow - 1 - (r0 - S::BW), 0);
      }
    }
  };
  // Chunk c of a row's 4 KT stands at c ^ place(row), so that sixteen rows' chunks of one number are in different banks.
  auto place = [](int row) { return KT == 1 ? (row >> 2) & 3 : (row >> 1) & 7; };
  const int cchunk = KT == 1 ? (lane & 3) ^ (lane >> 4) : (lane & 7) ^ (lane >> 4);  // of the rows from an even copy's on
  auto chunk_of = [&](int t) { return (uint32_t)(kWhole ? 4 * KT * t + cchunk : min(4 * t + cchunk, kb - 1)) * 16u; };
  auto copy = [&](int j, uint32_t chunk, int stage) {
    // Both factors fit 24 bits: K is at most 2^20.
    const uint32_t row = __umul24((uint32_t)min(lane / (4 * KT), cmore[j]), ldb);
    copy16(cbase[j], row + (KT == 2 && j % 2 ? chunk ^ 64u : chunk),
           (uint32_t)(stage * S::kStage + S::kCopyRows * (wave * S::kCopies + j) * S::kRow));
  };
  auto copies = [&](int t, int stage) {
    const uint32_t k = chunk_of(t);
#pragma unroll
    for (int j = 0; j < S::kCopies; ++j) copy(j, k, stage);
  };
  // Scales of whole windows (K a multiple of 512): copied as the codes are, 16 bytes a row, into the one window there is
  // once every wave has the one before in its registers.
  uint32_t soff[S::kScaleCopies];
  const uint8_t* wbase[S::kScaleCopies];
  uint32_t wslot[S::kScaleCopies];
  auto window_copies = [&](int w) {
#pragma unroll
    for (int j = 0; j < S::kScaleCopies; ++j) copy16(wbase[j], soff[j] + 16 * w, S::kCodes + wslot[j]);
  };
  auto aim_windows = [&](const Tile& q) {
    int l = lane;
    asm volatile("" : "+v"(l));
#pragma unroll
    for (int j = 0; j < S::kScaleCopies; ++j) {
      const int r0 = 64 * ((wave + j * S::kWaves) % (S::R / 64)), r = r0 + l;  // a wave without a copy repeats another's
      wslot[j] = 16 * r0;
      if (r0 < S::BW) {
        const int first = weight_row(q, r0);  // the least: a group of 64 begins with gate rows or holds up rows alone
        wbase[j] = a.ws + ((size_t)q.e * a.M + first) * kb;
        soff[j] = (uint32_t)(weight_row(q, r) - first) * (uint32_t)kb;
      } else {
        const int first = token_row(q, r0);
        wbase[j] = a.xs + ((size_t)q.row0 + first) * kb;
        soff[j] = (uint32_t)(token_row(q, r) - first) * (uint32_t)kb;
      }
    }
  };
  // Other scales: fetched 16 a row by the registers and put beside a stage's codes, a dword a row.
  const uint8_t* sbase[S::kScales];
  uint4 q[S::kScales], qn[S::kScales];
  if constexpr (!kWhole) {
#pragma unroll
    for (int j = 0; j < S::kScales; ++j) {
      const int r = min(tid + j * S::kThreads, S::R - 1);
      sbase[j] = r < S::BW ? a.ws + ((size_t)tile.e * a.M + weight_row(tile, r)) * kb
                           : a.xs + ((size_t)tile.row0 + token_row(tile, r)) * kb;
    }
  }
  auto put_scales = [&](int t, int stage) {  // called for t = 0, 1, 2, ...
    if ((t & 3) == 0) {
#pragma unroll
      for (int j = 0; j < S::kScales; ++j) {
        q[j] = t == 0 ? load_scales(sbase[j], 0, kb) : qn[j];
        if (t + 4 < tiles) qn[j] = load_scales(sbase[j], 16 * (t / 4 + 1), kb);
      }
    }
#pragma unroll
    for (int j = 0; j < S::kScales; ++j) {
      uint32_t v = q[j].x;
      q[j] = make_uint4(q[j].y, q[j].z, q[j].w, 0u);
      if (rem && t == tiles - 1) v = (v & ~(~0u << (8 * rem))) | 0x7f7f7f7fu << (8 * rem);  // blocks past the end: 2^0
      const int r = tid + j * S::kThreads;
      if (S::R % S::kThreads == 0 || r < S::R) *reinterpret_cast<uint32_t*>(lds + stage * S::kStage + S::kCodes + 4 * r) = v;
    }
  };

  f32x16 acc[MA][NB];
  struct Frags {
    i32x4 a[MA], b[NB];
  } f[2];
  uint32_t sa[MA], sb[NB];
  const int arow = wa * 32 * MA + l32, brow = S::BW + wb * 32 * NB + l32;  // multiples of 32 away: l32's place
  // A lane's chunk of step 0; that of step s is (4 (s / 2) + s % 2) * 16 away, by exclusive or.
  uint32_t aat = arow * S::kRow + (2 * h ^ place(l32 & 15)) * 16u, bat = brow * S::kRow + (2 * h ^ place(l32 & 15)) * 16u;
  // What addresses are formed from is made new in each turn of the loop: kept, they would take a quarter of the
  // registers.
  auto fresh = [&] { asm volatile("" : "+v"(aat), "+v"(bat), "+s"(ldb)); };
  // Piece p of a step's fragments, in the order in which the products need them: b0, a0, the other b, the other a.
  constexpr int kPieces = MA + NB, kProducts = MA * NB;
  auto read = [&](Frags& g, int stage, int s, int p) {
    const uint8_t* from = lds + stage * S::kStage;
    const uint32_t step = (4 * (s / 2) + s % 2) * 16;
    const int n = p == 0 ? 0 : p <= NB ? p - 1 : -1, m = p == 1 ? 0 : p - NB;
    if (p == 0 || (p > 1 && p <= NB)) g.b[n] = *reinterpret_cast<const i32x4*>(from + (bat ^ step) + 32 * n * S::kRow);
    else g.a[m] = *reinterpret_cast<const i32x4*>(from + (aat ^ step) + 32 * m * S::kRow);
  };
  auto read_all = [&](Frags& g, int stage, int s) {
#pragma unroll
    for (int p = 0; p < kPieces; ++p) read(g, stage, s, p);
  };
  // The dwords of a tile's scales (kWhole: of a window's four tiles, the next one's first); the lane's two bytes are
  // brought down where they are used, for a shift here would wait for every read before it.
  constexpr int kD = kWhole ? 4 : 1;
  uint32_t da[MA][kD], db[NB][kD];
  auto read_scales = [&](int stage) {
    const uint8_t* p = lds + (kWhole ? 0 : stage * S::kStage) + S::kCodes;
    auto get = [&](uint32_t (&d)[kD], int r) {
      if constexpr (kWhole) *reinterpret_cast<uint4*>(d) = *reinterpret_cast<const uint4*>(p + r * 16);
      else d[0] = *reinterpret_cast<const uint32_t*>(p + r * 4);
    };
#pragma unroll
    for (int m = 0; m < MA; ++m) get(da[m], arow + 32 * m);
#pragma unroll
    for (int n = 0; n < NB; ++n) get(db[n], brow + 32 * n);
  };
  auto take_scales = [&] {
    auto take = [&](uint32_t (&d)[kD]) {
      const uint32_t v = d[0] >> (16 * h);
#pragma unroll
      for (int i = 1; i < kD; ++i) d[i - 1] = d[i];
      return v;
    };
#pragma unroll
    for (int m = 0; m < MA; ++m) sa[m] = take(da[m]);
#pragma unroll
    for (int n = 0; n < NB; ++n) sb[n] = take(db[n]);
    __builtin_amdgcn_sched_barrier(0);
  };
  // The products of a step, `between(i)` behind the i-th: the reads and copies that go on meanwhile are dealt out
  // among them, since a wave issues in order and a row of reads would keep the products behind it waiting.  The
  // scheduling barriers keep the compiler from gathering them.
  auto multiply = [&](const Frags& g, auto step, auto between) {
    constexpr int s = decltype(step)::value;
#pragma unroll
    for (int i = 0; i < kProducts; ++i) {
      const int m = i / NB, n = i % NB;
      acc[m][n] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(operand(g.a[m]), operand(g.b[n]), acc[m][n], kFp4, kFp4, s,
                                                                  (int)sa[m], s, (int)sb[n]);
      between(i);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // Those of 0..n-1 that are behind the i-th product.
  auto deal = [&](int i, int n, auto what) {
#pragma unroll
    for (int p = 0; p < n; ++p)
      if (min(p, kProducts - 1) == i) what(p);
  };
  const std::integral_constant<int, 0> first;
  const std::integral_constant<int, 1> second;
  auto reading = [&](Frags& g, int stage, int s) {
    return [&, stage, s](int i) { deal(i, kPieces, [&](int p) { read(g, stage, s, p); }); };
  };
  const auto nothing = [](int) {};
  // Products written before this are not moved behind the branches after it.
  auto pin = [&] {
#pragma unroll
    for (int m = 0; m < MA; ++m)
#pragma unroll
      for (int n = 0; n < NB; ++n) asm volatile("" : "+v"(acc[m][n]));
  };

  // A step's fragments are read while the step before is multiplied.  A stage is met by the workgroup before its
  // last step: every wave has read it (and the window, where that is new), the next stage's copies have landed.
  auto most_steps = [&](int stage) {
    take_scales();
    multiply(f[0], first, reading(f[1], stage, 1));
    if constexpr (KT == 2) {
      multiply(f[1], second, reading(f[0], stage, 2));
      take_scales();
      multiply(f[0], first, reading(f[1], stage, 3));
    }
  };
  int stage;
  // Stage t, and the first fragments of the next.  kMore: with the copies of the stage that takes its place; kNext: of
  // the next tile's first, which the copies are already aimed at.
  auto turn = [&](int t, auto more, auto then) {
    constexpr bool kNext = decltype(then)::value, kMore = decltype(more)::value || kNext;
    const int next = stage == S::kStages - 1 ? 0 : stage + 1;
    fresh();
    most_steps(stage);
    pin();
    if (S::kStages > 2 && t + S::kStages - 1 < stages) copies_landed<(S::kStages - 2) * S::kCopies>();
    else copies_landed<0>();
    if constexpr (kWhole) {
      if constexpr (kNext) window_copies(0);
      else if (KT * t % 4 == 0 && KT * t + 4 < tiles) window_copies(KT * t / 4 + 1);
    } else if constexpr (kMore) {
      put_scales(t + S::kStages, stage);
    }
    if (!kWhole || KT * (t + 1) % 4 == 0) read_scales(next);
    const uint32_t chunk = kNext ? chunk_of(0) : kMore ? chunk_of(t + S::kStages) : 0u;
    __builtin_amdgcn_sched_barrier(0);
    multiply(f[1], second, [&](int i) {
      deal(i, kPieces, [&](int p) { read(f[0], next, 0, p); });
      if constexpr (kMore) deal(i, S::kCopies, [&](int j) { copy(j, chunk, stage); });
    });
    stage = next;
  };
  aim_copies(tile);
  if constexpr (kWhole) {
    aim_windows(tile);
    window_copies(0);
  }
#pragma unroll
  for (int t = 0; t < S::kStages; ++t)
    if (t < stages) {
      if constexpr (!kWhole) put_scales(t, t);
      copies(t, t);
    }
  if (stages >= S::kStages) copies_landed<(S::kStages - 1) * S::kCopies>();
  else copies_landed<0>();
  if constexpr (kStays)
    if (a.offsets) reinterpret_cast<RowTiles<S::BT>*>(lds + S::kTiles)[lane] = rt;  // the same by every wave

  for (;;) {
#pragma unroll
    for (int m = 0; m < MA; ++m)
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[m][n][i] = 0.f;
    Tile ahead = tile;
    bool goes_on = false;
    if constexpr (kStays) {
      if (a.offsets) rt = reinterpret_cast<const RowTiles<S::BT>*>(lds + S::kTiles)[lane];
      slot += gridDim.x / 8;
      goes_on = tile_at(slot, ahead);
    }
    stage = 0;
    read_all(f[0], 0, 0);
    read_scales(0);
    const std::true_type yes;
    const std::false_type no;
    int t = 0;
    for (; t < stages - S::kStages; ++t) turn(t, yes, no);
    if constexpr (kStays) {
      // There are two stages or more, of which the last is in the second place: the first is free for the next tile.
      // Without one this tile's is copied again: copies in a branch cost as much as these, each launch once.
      aim_copies(ahead);
      aim_windows(ahead);
      turn(t, no, yes);
    } else {
      for (; t < stages - 1; ++t) turn(t, no, no);
    }
    if constexpr (kWhole) {
      most_steps(stage);
    } else {
      take_scales();
      read_all(f[1], stage, 1);
#pragma unroll
      for (int s = 0; s < 2; ++s)
        if (rem && 2 * h + s >= rem) {  // blocks past the end: weights of zero
#pragma unroll
          for (int m = 0; m < MA; ++m) f[s].a[m] = i32x4{0, 0, 0, 0};
        }
      multiply(f[0], first, nothing);
    }
    multiply(f[1], second, nothing);
    pin();
    // The outputs are where the last stage was.  The next tile's first stage has landed: waited for here, not behind
    // the outputs' stores, which the wait would be one for too.
    copies_landed<0>();

    // acc[m][n][i]: weight row 32 m + 8 (i / 4) + 4 h + i % 4, row of x 32 n + l32.  Outputs go through LDS, 32 rows
    // of x at a time, so that a row's stand together: gated ones with their activation, others as sums.
    constexpr int kStride = kPart + 4;
    int at = lane;
    asm volatile("" : "+v"(at));  // what follows is formed for each tile again
    float* mine = reinterpret_cast<float*>(lds + S::kOutputs) + wave * 32 * kStride;
    const int col0 = (tile.nt * WA + wa) * kOut;
    const float* bias = a.bias ? a.bias + (size_t)tile.e * a.M : nullptr;
    const bool wide =
        width % 8 == 0 && ((reinterpret_cast<uintptr_t>(a.y) | reinterpret_cast<uintptr_t>(a.residual)) & 15) == 0;
    if constexpr (kGated) {
      if (bias) {
#pragma unroll
        for (int m = 0; m < MA; ++m)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const int r = 32 * m + 8 * g;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int c = min(col0 + r % kOut + 4 * (at >> 5) + i, width - 1);
              const float v = bias[(uint32_t)((r >= kOut ? width : 0) + c)];
#pragma unroll
              for (int n = 0; n < NB; ++n) acc[m][n][4 * g + i] += v;
            }
            __builtin_amdgcn_sched_barrier(0);  // no more than these at once: registers
          }
      }
    }
    auto put = [&](int n, int part, auto pair) {
#pragma unroll
      for (int k = 0; k < (kGated && MA == 1 ? 2 : kPart / 8); ++k) {
        const int m = part * (kPart / 32) + k / 4, g = k % 4;
        f32x4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (kGated) {
            const float u = MA == 1 ? acc[m][n][4 * (g + 2) % 16 + i] : acc[(m + MA / 2) % MA][n][4 * g + i];
            v[i] = pair(acc[m][n][4 * g + i], u);
          } else {
            v[i] = acc[m][n][4 * g + i];
          }
        }
        *reinterpret_cast<f32x4*>(mine + (at & 31) * kStride + 8 * k + 4 * (at >> 5)) = v;
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    constexpr int kLanes = kPart / 8;  // of a row, eight outputs each
    auto take = [&](int t0, int r, int part, bool plain) {
      const int t = r + at / kLanes, o = 8 * (at % kLanes), col = col0 + part * kPart + o;
      if (t0 + t >= tile.nrow || col >= width) return;
      float v[8];
      *reinterpret_cast<f32x4*>(v) = *reinterpret_cast<const f32x4*>(mine + t * kStride + o);
      *reinterpret_cast<f32x4*>(v + 4) = *reinterpret_cast<const f32x4*>(mine + t * kStride + o + 4);
      if constexpr (!kGated) {
        if (bias) {
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] += bias[min(col + i, width - 1)];
        }
        if (!plain) {
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = act_single(a.act, v[i]);
        }
      }
      const size_t to = ((size_t)tile.row0 + t0 + t) * width + col;
      if (wide) {
        if (a.residual) {
          const uint4 r4 = *reinterpret_cast<const uint4*>(a.residual + to);
          const uint32_t rw[4] = {r4.x, r4.y, r4.z, r4.w};
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] += __uint_as_float(i % 2 ? rw[i / 2] & 0xffff0000u : rw[i / 2] << 16);
        }
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = bf16_bits(v[2 * i]) | bf16_bits(v[2 * i + 1]) << 16;
        *reinterpret_cast<uint4*>(a.y + to) = make_uint4(w[0], w[1], w[2], w[3]);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (col + i < width)
            a.y[to + i] = (uint16_t)bf16_bits(a.residual ? v[i] + bf16_to_f32(a.residual[to + i]) : v[i]);
      }
    };
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int part = 0; part < kOut / kPart; ++part) {
        if (kGated && a.act != RMOE_ACT_SWIGLU)
          put(n, part, [&](float g, float u) { return act_pair(RMOE_ACT_SITU, g, u, a.gb, a.vb); });
        else
          put(n, part, [](float g, float u) { return swiglu(g, u); });
        const int t0 = wb * 32 * NB + 32 * n;
        if (kGated || a.act == RMOE_ACT_NONE) {
#pragma unroll
          for (int r = 0; r < 32; r += 64 / kLanes) take(t0, r, part, true);
        } else {
#pragma unroll 1
          for (int r = 0; r < 32; r += 64 / kLanes) take(t0, r, part, false);
        }
      }
    if (!kStays || !goes_on) return;
    __syncthreads();  // the outputs' place is the second stage's again
    tile = ahead;
    copies(1, 1);
  }
}

// Workgroups that take tile after tile: one a CU, which their LDS fills.  Calls of no more tiles than that do not take
// them so: the copies for a tile that does not come made 445 rows of [24064, 2560] 27.2 us and not 26.
constexpr size_t kStaying = 256;

template <int MA, int NB, int WA, int WB, bool kWhole, bool kStays>
Plan plan_tiles(const MxLin& a) {
  typedef TileShape<MA, NB, WA, WB, kWhole, kStays> S;
  const bool gated = act_gated(a.act);
  const int width = gated ? a.M / 2 : a.M, out = S::BW / (gated ? 2 : 1), n_nt = (width + out - 1) / out;
  const size_t mt = a.offsets ? std::min<size_t>(a.n, (size_t)a.n / S::BT + a.n_experts) : ((size_t)a.n + S::BT - 1) / S::BT;
  const size_t all = 8 * ((mt * n_nt + 7) / 8), grid = kStays ? std::min(all, kStaying) : all;
  auto* kernel = gated ? mx_tiles_kernel<MA, NB, WA, WB, kWhole, kStays, true>
                       : mx_tiles_kernel<MA, NB, WA, WB, kWhole, kStays, false>;
  // Of workgroups that stay the tiles count too: their numbers are kept to 24 bits.
  return Plan{kernel, grid, S::kThreads, S::lds(gated), n_nt, all * S::kThreads < (size_t)1 << 32};
}
// stays: more tiles than kStaying are taken by as many workgroups.
template <int MA, int NB, int WA, int WB, bool kStays = false>
Plan pick_tiles(const MxLin& a) {
  const bool whole = a.K % 512 == 0 && ((reinterpret_cast<uintptr_t>(a.xs) | reinterpret_cast<uintptr_t>(a.ws)) & 15) == 0;
  return whole ? plan_tiles<MA, NB, WA, WB, true, kStays>(a) : plan_tiles<MA, NB, WA, WB, false, false>(a);
}
template <int MA, int NB, int WA, int WB, bool kWhole, bool kStays>
hipError_t setup_tiles() {
  typedef TileShape<MA, NB, WA, WB, kWhole, kStays> S;
  hipError_t e = hipFuncSetAttribute((const void*)mx_tiles_kernel<MA, NB, WA, WB, kWhole, kStays, true>,
                                     hipFuncAttributeMaxDynamicSharedMemorySize, (int)S::lds(true));
  if (e == hipSuccess)
    e = hipFuncSetAttribute((const void*)mx_tiles_kernel<MA, NB, WA, WB, kWhole, kStays, false>,
                            hipFuncAttributeMaxDynamicSharedMemorySize, (int)S::lds(false));
  return e;
}

// Which kernel serves a call; times in us at 2,560 columns or those given.
//   Weight rows over all tiles of 16 rows of x, at most kFewRows: the kernel of few rows, for its waves share K.  32
//   rows of [4096, 4096] 7.1 and 11.0 with the smallest tiles, 64 rows (16,384) 10.7 and 11.3, 96 rows 14.2 and 11.5.
//   Fragments a wave: up to kOneFragment weight rows one (four rows of [4096, 4096] 5.3, two 6.2), above two (64 rows
//   of [1536, 2048] 5.1 and 5.6).  One or two rows of x have it without shared parts of K where there are kFillSmall
//   tiles of 64 weight rows (one row of [260096] 64.3 and 66.5 in tiles of 128 x 64, four 67.2 and 65.7; one row of
//   [24064] 10.3 and 9.4 in 64 x 64).
//   Up to kFlat rows of x the flattest tiles: 128 x 64 where there are kFillSmall of 64 x 64 (32 rows of [260096] 77, in
//   64 x 64 80, in 256 x 256 102; 65 rows 101, 110 and 111; 128 rows 116, 137 and 116), else 64 x 64 (16 rows of [24064]
//   9.4 and without LDS 11.8, 32 rows 9.8 and 18).
//   By expert few rows each (under kFewEach) leave the tiles empty: two parts of K, 32 rows of 128 experts' [1536, 2048]
//   12.1 and 14.8 without, 256 rows 36.7 and 38.4 in tiles of 128 x 64; 512 rows 41.6 and 41.3.
//   Tiles of 256 x 256 where there are kFillLarge of them (445 rows of [24064] 26.2, in tiles of 128 x 128 27.1; 256 rows
//   24.2 and 17.9) and, by expert, kFillEach rows each (128 experts' gated [1536, 2048]: 24,000 rows 79 and in 128 x 64
//   98, 16,000 rows 73 and 76, 12,000 rows 72 and 68).  Else by expert 128 x 64; dense 64 x 64 up to kFillSmall of them
//   (1,024 rows of [4096, 4096] 22.8 and 20.2 in 128 x 128, 2,048 of [1536, 2048] 11.1 and 12.2), above 128 x 128.
constexpr size_t kOneFragment = 4096, kFewRows = 16384, kFlat = 96, kFillSmall = 1000, kFillLarge = 180;
constexpr int kFewEach = 4, kFillEach = 120;

Plan plan_mx_linear(const MxLin& a) {
  const size_t n = a.n, M = a.M, groups = a.offsets ? a.n_experts : 1;
  auto tiles = [&](size_t weights, size_t rows) { return (n + rows - 1) / rows * ((M + weights - 1) / weights); };
  const size_t rows = M * (a.offsets ? std::min(n, n / 16 + groups) : (n + 15) / 16);
  if (rows <= kOneFragment) return plan_few<1, 1>(a);
  if (rows <= kFewRows) return plan_few<2, 1>(a);
  // The tiles' offsets within a matrix's scales and 16 rows' codes take 32 bits.
  const bool wide = a.K > 1 << 20 || M * (a.K / kMxBlock) >= (size_t)1 << 32;
  auto large = [&] {
    return tiles(256, 256) > kStaying ? pick_tiles<4, 2, 2, 4, true>(a) : pick_tiles<4, 2, 2, 4, false>(a);
  };
  if (a.offsets) {
    if (wide || n < kFewEach * groups) return plan_few<2, 2>(a);
    if (n >= kFillEach * groups && tiles(256, 256) >= kFillLarge) return large();
    return pick_tiles<2, 1, 2, 2>(a);
  }
  const bool fill = tiles(64, 64) >= kFillSmall;
  if (wide || (n <= 2 && fill)) return plan_few<2, 4>(a);
  if (n <= kFlat) return fill ? pick_tiles<2, 1, 2, 2>(a) : pick_tiles<1, 1, 2, 2>(a);
  if (tiles(256, 256) >= kFillLarge) return large();
  return fill ? pick_tiles<2, 2, 2, 2>(a) : pick_tiles<1, 1, 2, 2>(a);
}

}  // namespace

// Allow the tiles of more than 64 KB of dynamic LDS theirs (up to 142).
hipError_t mx_linear_setup() {
  for (const hipError_t e : {setup_tiles<4, 2, 2, 4, true, true>(), setup_tiles<4, 2, 2, 4, true, false>(),
                             setup_tiles<4, 2, 2, 4, false, false>(), setup_tiles<2, 2, 2, 2, true, false>()})
    if (e != hipSuccess) return e;
  return hipSuccess;
}

bool mx_linear_fits(const MxLin& a) { return plan_mx_linear(a).fits; }

hipError_t launch_mx_linear(const MxLin& a, hipStream_t st) {
  const Plan p = plan_mx_linear(a);
  hipLaunchKernelGGL(p.kernel, dim3((unsigned)p.grid), dim3(p.threads), p.lds, st, a, p.n_nt);
  return hipGetLastError();
}

}  // namespace rmoe
