// y[n, M'] = RTNE(act(x[n, K] @ W^T + bias) + residual) for many rows, of one matrix or of
// each row's expert, on fp16 MFMA.
//
// Operands.  A row of x becomes fp16 times a power of two that brings its largest value into
// [2^14, 2^15): bf16's 8 significant bits fit, values down to 2^-31 of the largest are exact.
// A weight is formed in fp16 as its row's power of two brings the row's largest into
// [2^10, 2^11): bfp16's m * 2^(e-133) exactly, q4nx's m + s * n by one fused multiply-add,
// rounded once to fp16's 11 bits.  That rounding, at most 2^-11 of a weight (and 2^-35 of the
// row's largest), adds to a sum what is an eighth of its bf16 rounding in the mean (rel-L2
// against 64 bits 1.65e-3 with and without it); keeping s * (n - 8) exact instead costs a
// second product over the group sums of x (one MFMA in five) and their preparation.  Sums
// are fp32; the powers of two are taken back exactly.
#include <algorithm>

#include "linear_act.h"

namespace rmoe {
namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// --------------------------------------------------------------- preparation --
// Workgroups 0..n_x-1: four rows of x each, to fp16 (zero past K_in) and their exponents; the
// rest: the exponents of 256 weight rows each.
struct PrepArgs {
  LinAct a;
  uint16_t* xh;
  int32_t *xe, *we;
  int n_x;
};

// The power of two e with v * 2^-e in [2^top, 2^(top+1)); 0 for zero and non-finite v.
__device__ __forceinline__ int exponent_for(float v, int top) {
  const int be = (int)(__float_as_uint(v) >> 23) & 0xff;
  if (v == 0.f || be == 0xff) return 0;
  return max(be, 1) - 127 - top;
}
__device__ __forceinline__ uint32_t half_pair(float lo, float hi) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(lo, hi));
}
__device__ __forceinline__ uint32_t bf16_pair_to_half(uint32_t v, int e) {
  return half_pair(__builtin_amdgcn_ldexpf(__uint_as_float(v << 16), -e),
                   __builtin_amdgcn_ldexpf(__uint_as_float(v & 0xffff0000u), -e));
}

__global__ __launch_bounds__(256) void act_prep_kernel(PrepArgs p) {
  const LinAct& a = p.a;
  const int lane = threadIdx.x & 63, wave = wave_id();
  if ((int)blockIdx.x < p.n_x) {
    const size_t t = (size_t)blockIdx.x * 4 + wave;
    if (t >= (size_t)a.n) return;
    const uint4* src = reinterpret_cast<const uint4*>(a.x + t * a.K_in);
    uint4* dst = reinterpret_cast<uint4*>(p.xh + t * a.K);
    const int nch = a.K_in / 8, nout = a.K / 8;
    float mx = 0.f;
    for (int c = lane; c < nch; c += 64) {
      const uint4 v = src[c];
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 4; ++i)
        mx = fmaxf(mx, fmaxf(fabsf(__uint_as_float(w[i] << 16)), fabsf(__uint_as_float(w[i] & 0xffff0000u))));
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor(mx, off, 64));
    const int e = exponent_for(mx, 14);
    for (int c = lane; c < nout; c += 64) {
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if (c < nch) {
        const uint4 s = src[c];
        v = make_uint4(bf16_pair_to_half(s.x, e), bf16_pair_to_half(s.y, e), bf16_pair_to_half(s.z, e),
                       bf16_pair_to_half(s.w, e));
      }
      dst[c] = v;
    }
    if (lane == 0) p.xe[t] = e;
    return;
  }
  const size_t r = ((size_t)blockIdx.x - p.n_x) * 256 + threadIdx.x;  // row r % M of matrix r / M
  const size_t rows = (size_t)a.M * (a.offsets ? a.n_experts : 1);
  if (r >= rows) return;
  const int row = (int)(r % a.M), nkt = a.K / kTileCols;
  const bool b16 = a.fmt == RMOE_FMT_BFP16;
  const int tb = b16 ? kB16TileBytes : kTileBytes, at = b16 ? kB16MantBytes : kCodeBytes;
  const uint8_t* q = a.tiles + (r / a.M) * a.wstride + (size_t)(row / kTileRows) * nkt * tb + at + (row % kTileRows) * 16;
  float mx = 0.f;
  uint32_t emax = 7u;
#pragma unroll 4
  for (int kt = 0; kt < nkt; ++kt) {
    const uint4 v = *reinterpret_cast<const uint4*>(q + (size_t)kt * tb);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (b16) {
#pragma unroll
        for (int b = 0; b < 4; ++b) emax = max(emax, (w[i] >> (8 * b)) & 0xffu);
      } else {
        const float s = __uint_as_float(w[i] << 16), m = __uint_as_float(w[i] & 0xffff0000u);
        mx = fmaxf(mx, fmaxf(fabsf(m), fabsf(fmaf(15.f, s, m))));
      }
    }
  }
  // |m| <= 2^7 in bfp16
  p.we[r] = b16 ? (int)emax - 133 + 7 - 10 : exponent_for(mx, 10);
}

// ---------------------------------------------------------------------- tiles --
struct TileArgs {
  LinAct a;
  const uint16_t* xh;
  const int32_t *xe, *we;
  int n_nt;
};

constexpr int kActBM = 128;
constexpr int kStage = kActBM * 128;  // bytes of 128 rows x 64 columns of fp16
constexpr int kEpilogueLds = 65536;

// A wave's weights in LDS, as its tiles hold them: its 64 weight rows' sub-blocks of half a K
// tile (64 columns: two of codes, four of mantissas; 1 KB each, two stages), then the 1 KB of
// scale | min words or exponents of a whole K tile (two, by the tile's parity).
template <int kFmt>
constexpr int kHalfBlocks = kFmt == RMOE_FMT_BFP16 ? 4 : 2;
template <int kFmt>
constexpr int kWaveWeights = 2 * 1024 * kHalfBlocks<kFmt> + 2 * 1024;

__device__ __forceinline__ f16x2 as_f16x2(uint32_t v) { return __builtin_bit_cast(f16x2, v); }
__device__ __forceinline__ uint32_t as_u32(f16x2 v) { return __builtin_bit_cast(uint32_t, v); }

__device__ __forceinline__ f16x2 low2(f16x2 v) { return __builtin_shufflevector(v, v, 0, 0); }
__device__ __forceinline__ f16x2 high2(f16x2 v) { return __builtin_shufflevector(v, v, 1, 1); }

// Masks of the code unpacking in registers: (x & m) | o is one instruction then, which takes
// no literal and one scalar register.
struct CodeMasks {
  uint32_t lo, hi, magic;  // 0x000f000f, 0x00f000f0 (scalar), 0x64006400 (vector)
};
__device__ __forceinline__ CodeMasks code_masks() {
  CodeMasks k;
  asm volatile("s_mov_b32 %0, 0xf000f\n\ts_mov_b32 %1, 0xf000f0\n\tv_mov_b32 %2, 0x64006400"
               : "=&s"(k.lo), "=&s"(k.hi), "=&v"(k.magic));
  return k;
}
// Four codes times s plus m (sm: s low, m high), in the low 16 bits' nibble order: one nibble
// pair of the dword sits where the bits 0x6400 make it 1024 + n, one where they make it
// 1024 + 16 n, which meets s / 16.
__device__ __forceinline__ uint2 q4_operand(uint32_t c, f16x2 sm, const CodeMasks& k) {
  const f16x2 k1024 = {(_Float16)1024.f, (_Float16)1024.f}, sixteenth = {(_Float16)0.0625f, (_Float16)0.0625f};
  const f16x2 s = low2(sm), s16 = s * sixteenth, m = high2(sm);
  const f16x2 n0 = as_f16x2((c & k.lo) | k.magic) - k1024, n1 = as_f16x2((c & k.hi) | k.magic) - k1024;
  return make_uint2(as_u32(__builtin_elementwise_fma(n0, s, m)), as_u32(__builtin_elementwise_fma(n1, s16, m)));
}
// Four int8 mantissas times s, a power of two: a byte u = m + 128 below 0x64 is 1024 + u, and
// (1024 + u) s - 1152 s = m s without a rounding.
__device__ __forceinline__ uint2 b16_operand_half(uint32_t v, f16x2 s) {
  const f16x2 k = {(_Float16)-1152.f, (_Float16)-1152.f}, t = s * k;
  const uint32_t u = v ^ 0x80808080u, h = 0x64646464u;
  return make_uint2(as_u32(__builtin_elementwise_fma(as_f16x2(__builtin_amdgcn_perm(h, u, 0x04010400u)), s, t)),
                    as_u32(__builtin_elementwise_fma(as_f16x2(__builtin_amdgcn_perm(h, u, 0x04030402u)), s, t)));
}

__device__ __forceinline__ void swap32(uint32_t& a, uint32_t& b) {
  const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
  a = r[0];
  b = r[1];
}
__device__ __forceinline__ void swap16(uint32_t& a, uint32_t& b) {
  const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
  a = r[0];
  b = r[1];
}

// q4nx: the scale | min words of a K tile in the wave's LDS, brought to the row's power of two
// and to fp16 once for all that read them (lane = weight row; four words).
__device__ __forceinline__ void convert_words(uint8_t* wp, int we) {
  uint4* p = reinterpret_cast<uint4*>(wp) + (threadIdx.x & 63u);
  uint4 v = *p;
  auto half = [&](uint32_t w) {
    return half_pair(__builtin_amdgcn_ldexpf(__uint_as_float(w << 16), -we),
                     __builtin_amdgcn_ldexpf(__uint_as_float(w & 0xffff0000u), -we));
  };
  *p = make_uint4(half(v.x), half(v.y), half(v.z), half(v.w));
}

// What a wave keeps of a stage's weights while it forms MFMA operands from them: 64 columns
// of its NF fragments of 16 rows, two operands (steps of 32 columns) each.
template <int kFmt, int NF>
struct StageWeights;
template <int NF>
struct StageWeights<RMOE_FMT_Q4NX, NF> {
  uint32_t c[NF / 2][4];
  uint2 sm[NF];
  // wl: the wave's sub-blocks, wp: its words of the tile, j: the half of the tile
  __device__ __forceinline__ void read(const uint8_t* wl, const uint8_t* wp, int j) {
    const uint32_t lane = threadIdx.x & 63u, l16 = lane & 15u, lq = lane >> 4;
#pragma unroll
    for (int p = 0; p < NF / 2; ++p) {
      // lane quarter lq: group lq % 2 of fragment lq / 2 of the pair
      const uint4 v = *reinterpret_cast<const uint4*>(wl + 1024u * (lq & 1u) + 256u * (lq >> 1) + 16u * l16 + 512 * p);
      c[p][0] = v.x;
      c[p][1] = v.y;
      c[p][2] = v.z;
      c[p][3] = v.w;
    }
#pragma unroll
    for (int f = 0; f < NF; ++f) sm[f] = *reinterpret_cast<const uint2*>(wp + 256 * f + 16u * l16 + 8 * j);
  }
  // A 4 x 4 transpose over the lane quarters gives each dword lq of a pair's four (fragment,
  // group)s.
  __device__ __forceinline__ void arrange() {
#pragma unroll
    for (int p = 0; p < NF / 2; ++p) {
      swap32(c[p][0], c[p][2]);
      swap32(c[p][1], c[p][3]);
      swap16(c[p][0], c[p][1]);
      swap16(c[p][2], c[p][3]);
    }
  }
  // Half `part` of fragment f's operand of step g.
  __device__ __forceinline__ void form(int g, int f, int part, const int (&)[NF], const CodeMasks& k, uint4& b) const {
    const uint32_t v = c[f / 2][2 * (f % 2) + g];
    const uint2 r = q4_operand(part ? v >> 8 : v, as_f16x2(g ? sm[f].y : sm[f].x), k);
    if (part) b.z = r.x, b.w = r.y;
    else b.x = r.x, b.y = r.y;
  }
  // The rows' chunk (8 columns) that lane quarter lq multiplies in step g.
  static __device__ __forceinline__ uint32_t chunk(int g) { return 4u * g + ((threadIdx.x & 63u) >> 4); }
};
template <int NF>
struct StageWeights<RMOE_FMT_BFP16, NF> {
  uint4 v[NF];      // 16 mantissas: blocks 2 lq and 2 lq + 1 of the half
  uint32_t ex[NF];  // the exponents of blocks 4 (lq / 2)..+3
  __device__ __forceinline__ void read(const uint8_t* wl, const uint8_t* wp, int j) {
    const uint32_t lane = threadIdx.x & 63u, l16 = lane & 15u, lq = lane >> 4;
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      v[f] = *reinterpret_cast<const uint4*>(wl + 1024u * lq + 256 * f + 16u * l16);
      ex[f] = *reinterpret_cast<const uint32_t*>(wp + 256 * f + 16u * l16 + 8 * j + 4u * (lq >> 1));
    }
  }
  __device__ __forceinline__ void arrange() {}
  __device__ __forceinline__ void form(int g, int f, int part, const int (&we)[NF], const CodeMasks&, uint4& b) const {
    const uint32_t lq = (threadIdx.x & 63u) >> 4;
    const int e = (int)max((ex[f] >> (16u * (lq & 1u) + 8u * g)) & 0xffu, 7u) - 133 - we[f];
    const float s = __builtin_amdgcn_ldexpf(1.f, e);
    const uint32_t w = g ? (part ? v[f].w : v[f].z) : (part ? v[f].y : v[f].x);
    const uint2 r = b16_operand_half(w, as_f16x2(half_pair(s, s)));
    if (part) b.z = r.x, b.w = r.y;
    else b.x = r.x, b.y = r.y;
  }
  static __device__ __forceinline__ uint32_t chunk(int g) { return 2u * ((threadIdx.x & 63u) >> 4) + g; }
};

// One step of 32 columns: MF x NF products with the operands b, and under them the 2 NF
// halves of the next step's operands n (from `from`, its step g), spread evenly: an MFMA takes
// 16 cycles and its issue 4, so a wave's vector instructions fit between its own.  Chunk c
// (16 bytes) of row r of a stage sits at chunk c ^ (r / 2 % 8): the 16 rows of a fragment then
// cover all 64 banks.
template <int kFmt, int MF, int NF>
__device__ __forceinline__ void mfma_step(const uint8_t* stage, uint32_t chunk, const uint4 (&b)[NF],
                                          const StageWeights<kFmt, NF>& from, int g, const int (&we)[NF],
                                          const CodeMasks& masks, uint4 (&n)[NF], f32x4 (&acc)[8][NF]) {
  const uint32_t l16 = threadIdx.x & 15u;
  const uint8_t* p = stage + 128u * l16 + 16u * (chunk ^ (l16 >> 1));
  uint4 x[MF];
#pragma unroll
  for (int m = 0; m < 2; ++m) x[m] = *reinterpret_cast<const uint4*>(p + 2048 * m);
#pragma unroll
  for (int m = 0; m < MF; ++m) {
    if (m + 2 < MF) x[m + 2] = *reinterpret_cast<const uint4*>(p + 2048 * (m + 2));
#pragma unroll
    for (int f = 0; f < NF; ++f)
      acc[m][f] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, x[m]), __builtin_bit_cast(f16x8, b[f]),
                                                         acc[m][f], 0, 0, 0);
#pragma unroll
    for (int q = 2 * NF * m / MF; q < 2 * NF * (m + 1) / MF; ++q) from.form(g, q / 2, q % 2, we, masks, n[q / 2]);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// 16 bytes per lane from global memory straight into LDS, lane L to lds + 16 L: no registers
// and no LDS store instruction.  Inline assembly, because the compiler makes every LDS read
// after its own form wait for all copies in flight; copies_landed() orders them instead.  An
// LDS copy needs one wait state after a write of M0, which is restored.
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
// Every copy of this wave has landed, then the workgroup meets.
__device__ __forceinline__ void copies_landed() {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
}

// One tile of up to 16 MF rows x 64 NF weight rows; wave w takes all rows and 16 NF = 64
// weight rows of its own (w: the matrix; wo: byte offset of weight row `lane` of the 64).
// Stages of 64 columns, two in LDS: a stage's rows are copied under the one before, its
// weights, which no other wave reads, under the one before that, so that their operands are
// formed under products throughout.  One barrier a stage.
template <int kFmt, int MF, int NF>
__device__ __forceinline__ void tile_product(const TileArgs& t, const uint8_t* w, uint32_t wo, int we_lane,
                                             const int (&we)[NF], int row0, uint8_t* lds, f32x4 (&acc)[8][NF]) {
  static_assert(NF == 4, "64 weight rows a wave");
  constexpr int kTB = kFmt == RMOE_FMT_BFP16 ? kB16TileBytes : kTileBytes, kBlocks = kHalfBlocks<kFmt>;
  const int lane = threadIdx.x & 63, wave = wave_id(), nkt = t.a.K / kTileCols;
  const uint32_t lds0 = (uint32_t)(uintptr_t)lds;
  const int wbase = 2 * kStage + wave * kWaveWeights<kFmt>, pbase = wbase + 2 * 1024 * kBlocks;
  // Copy q = wave + 4i fills LDS rows 8q..8q+7 (1 KB): lane L brings row 8q + L / 8 the chunk
  // that sits at position L % 8.  Rows past the tile are the next tiles' or, behind the last
  // row, the kActBM spare rows of the scratch; their results are not stored.
  const uint8_t* xb = reinterpret_cast<const uint8_t*>(t.xh + (size_t)row0 * t.a.K);
  const uint32_t ld = 2u * (uint32_t)t.a.K;
  const uint32_t xo = (uint32_t)(8 * wave + lane / 8) * ld + 16u * (uint32_t)((lane % 8) ^ ((4 * wave + lane / 16) % 8));
  uint32_t rows0 = lds0 + 1024u * (uint32_t)wave;
  asm volatile("" : "+s"(rows0));  // kept in a scalar register
  auto load_rows = [&](const uint8_t* x, int slot) {
#pragma unroll
    for (int i = 0; i < MF / 2; ++i) copy16(x + (size_t)(32 * i) * ld, xo, rows0 + (uint32_t)(slot * kStage + 4096 * i));
  };
  auto load_weights = [&](const uint8_t* tile, int j) {
#pragma unroll
    for (int i = 0; i < kBlocks; ++i)
      copy16(tile + 1024 * (kBlocks * j + i), wo, lds0 + (uint32_t)(wbase + 1024 * (kBlocks * j + i)));
  };
  auto load_words = [&](const uint8_t* tile, int par) {
    copy16(tile + 2048 * kBlocks, wo, lds0 + (uint32_t)(pbase + 1024 * par));
  };
  const CodeMasks masks = code_masks();
  load_rows(xb, 0);
  load_weights(w, 0);
  load_weights(w, 1);
  load_words(w, 0);
  copies_landed();
  if constexpr (kFmt == RMOE_FMT_Q4NX) convert_words(lds + pbase, we_lane);
  StageWeights<kFmt, NF> cur, next;
  uint4 b0[NF], b1[NF];
  cur.read(lds + wbase, lds + pbase, 0);
  cur.arrange();
#pragma unroll
  for (int q = 0; q < 2 * NF; ++q) cur.form(0, q / 2, q % 2, we, masks, b0[q / 2]);
#pragma unroll 1
  for (int kt = 0; kt < nkt; ++kt) {
    const uint8_t* wp = lds + pbase + 1024 * (kt & 1);
    const uint8_t* wp_next = lds + pbase + 1024 * ((kt + 1) & 1);
    const bool more = kt + 1 < nkt;
    // First half of the tile.  Its weights are in registers; their place in LDS takes the
    // next tile's.
    load_rows(xb + 128, 1);
    if (more) {
      load_weights(w + kTB, 0);
      load_words(w + kTB, (kt + 1) & 1);
    }
    mfma_step<kFmt, MF, NF>(lds, StageWeights<kFmt, NF>::chunk(0), b0, cur, 1, we, masks, b1, acc);
    next.read(lds + wbase + 1024 * kBlocks, wp, 1);
    next.arrange();
    mfma_step<kFmt, MF, NF>(lds, StageWeights<kFmt, NF>::chunk(1), b1, next, 0, we, masks, b0, acc);
    copies_landed();
    // Second half; past the last tile the operands formed are of old weights and not used.
    if (more) {
      xb += 256;
      w += kTB;
      load_rows(xb, 0);
      load_weights(w, 1);
      if constexpr (kFmt == RMOE_FMT_Q4NX) convert_words(lds + pbase + 1024 * ((kt + 1) & 1), we_lane);
    }
    mfma_step<kFmt, MF, NF>(lds + kStage, StageWeights<kFmt, NF>::chunk(0), b0, next, 1, we, masks, b1, acc);
    cur.read(lds + wbase, wp_next, 0);
    cur.arrange();
    mfma_step<kFmt, MF, NF>(lds + kStage, StageWeights<kFmt, NF>::chunk(1), b1, cur, 0, we, masks, b0, acc);
    copies_landed();
  }
}

template <int kFmt, int NF, bool kGated>
__global__ __launch_bounds__(256, 2) void act_tile_kernel(TileArgs t) {
  constexpr int kLds = 2 * kStage + 4 * kWaveWeights<kFmt>;
  __shared__ __attribute__((aligned(16))) uint8_t lds[kLds > kEpilogueLds ? kLds : kEpilogueLds];
  constexpr int kCols = 64 * NF, kOut = kGated ? kCols / 2 : kCols;
  constexpr int kTB = kFmt == RMOE_FMT_BFP16 ? kB16TileBytes : kTileBytes;
  const LinAct& a = t.a;
  RowTiles<kActBM> rt;
  const int n_mt = a.offsets ? rt.total(a.offsets, a.n_experts, a.n) : (a.n + kActBM - 1) / kActBM;
  const int total = n_mt * t.n_nt, per = (total + 7) / 8, slot = (int)blockIdx.x / 8;
  const int id = ((int)blockIdx.x % 8) * per + slot;
  if (slot >= per || id >= total) return;
  const int nt = id % t.n_nt;
  int e = 0, row0 = id / t.n_nt * kActBM, nrow = min(kActBM, a.n - row0);
  if (a.offsets) rt.find(id / t.n_nt, e, row0, nrow);
  const int wave = wave_id(), nkt = a.K / kTileCols, width = kGated ? a.M / 2 : a.M;
  const uint8_t* tiles = a.tiles + (size_t)e * a.wstride;
  // The wave's weight rows: 64 consecutive ones, or 32 gate rows and their up rows.  Columns
  // past the matrix (its width is a multiple of 64) repeat its first rows.
  const int c0 = nt * kOut + wave * (kOut / 4), base = c0 < width ? c0 : 0;
  auto row_of = [&](int r) { return kGated && r >= 32 ? width + base + r - 32 : base + r; };
  const int wr = row_of(threadIdx.x & 63);
  const uint32_t wo = (uint32_t)(wr / kTileRows) * (uint32_t)(nkt * kTB) + (uint32_t)(wr % kTileRows) * 16u;
  const int32_t* wes = t.we + (size_t)e * a.M;
  int we[NF];
#pragma unroll
  for (int f = 0; f < NF; ++f) we[f] = wes[row_of(16 * f + (threadIdx.x & 15))];
  f32x4 acc[8][NF];
#pragma unroll
  for (int m = 0; m < 8; ++m)
#pragma unroll
    for (int f = 0; f < NF; ++f) acc[m][f] = f32x4{0.f, 0.f, 0.f, 0.f};
  // A short tile multiplies only the fragments that hold rows.
  if (nrow > 64) tile_product<kFmt, 8, NF>(t, tiles, wo, wes[wr], we, row0, lds, acc);
  else if (nrow > 32) tile_product<kFmt, 4, NF>(t, tiles, wo, wes[wr], we, row0, lds, acc);
  else tile_product<kFmt, 2, NF>(t, tiles, wo, wes[wr], we, row0, lds, acc);

  // Epilogue: sums and bias through LDS as fp32, kRows rows at a time, so that the activation
  // has its operands at hand and residual and y move 16 bytes a thread.  Columns of
  // different lq go to different banks: column c of row r sits at c ^ 16 (r / 4 % 4).
  constexpr int kRows = kEpilogueLds / 4 / kCols;
  int tid = threadIdx.x;
  asm volatile("" : "+v"(tid));  // what follows from it is computed here, not kept across the products
  const int l16 = tid & 15, lq = (tid & 63) >> 4;
  float* out = reinterpret_cast<float*>(lds);
  float bias[NF];
#pragma unroll
  for (int f = 0; f < NF; ++f) we[f] = wes[row_of(16 * f + l16)];
#pragma unroll
  for (int f = 0; f < NF; ++f) bias[f] = a.bias ? a.bias[(size_t)e * a.M + row_of(16 * f + l16)] : 0.f;
  const bool wide = ((reinterpret_cast<uintptr_t>(a.y) | reinterpret_cast<uintptr_t>(a.residual)) & 15) == 0;
#pragma unroll
  for (int r0 = 0; r0 < kActBM; r0 += kRows) {
    if (r0 >= nrow) break;
    if (r0) __syncthreads();
#pragma unroll
    for (int m = r0 / 16; m < (r0 + kRows) / 16; ++m)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = 16 * m + 4 * lq + i;
        const int xe = t.xe[row0 + min(r, nrow - 1)];
        float* o = out + (r - r0) * kCols;
#pragma unroll
        for (int f = 0; f < NF; ++f) {
          const int c = kGated ? wave * (kOut / 4) + 16 * (f % (NF / 2)) + (f >= NF / 2 ? kOut : 0) : wave * (kOut / 4) + 16 * f;
          o[(c + l16) ^ (16 * lq)] = __builtin_amdgcn_ldexpf(acc[m][f][i], xe + we[f]) + bias[f];
        }
      }
    __syncthreads();
    const int rows = min(kRows, nrow - r0), cols = min(kOut, width - nt * kOut);
#pragma unroll 1
    for (int i = tid; i < rows * (kOut / 8); i += 256) {
      const int r = i / (kOut / 8), c = 8 * (i % (kOut / 8));
      if (c >= cols) continue;
      const float* o = out + r * kCols + (c ^ (16 * ((r >> 2) & 3)));
      float v[8];
      *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(o);
      *reinterpret_cast<float4*>(v + 4) = *reinterpret_cast<const float4*>(o + 4);
      if constexpr (kGated) {
        float u[8];
        *reinterpret_cast<float4*>(u) = *reinterpret_cast<const float4*>(o + kOut);
        *reinterpret_cast<float4*>(u + 4) = *reinterpret_cast<const float4*>(o + kOut + 4);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = act_pair(a.act, v[k], u[k], a.gb, a.vb);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = act_single(a.act, v[k]);
      }
      const size_t at = (size_t)(row0 + r0 + r) * width + nt * kOut + c;
      if (wide) {
        if (a.residual) {
          const uint4 q = *reinterpret_cast<const uint4*>(a.residual + at);
          const uint32_t qw[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            v[2 * k] += __uint_as_float(qw[k] << 16);
            v[2 * k + 1] += __uint_as_float(qw[k] & 0xffff0000u);
          }
        }
        uint32_t y[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) y[k] = f32_to_bf16(v[2 * k]) | (f32_to_bf16(v[2 * k + 1]) << 16);
        *reinterpret_cast<uint4*>(a.y + at) = make_uint4(y[0], y[1], y[2], y[3]);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          a.y[at + k] = (uint16_t)f32_to_bf16(a.residual ? v[k] + bf16_to_f32(a.residual[at + k]) : v[k]);
      }
    }
  }
}

template <int kFmt, int NF>
hipError_t launch_tiles(const TileArgs& t0, hipStream_t st) {
  TileArgs t = t0;
  const LinAct& a = t.a;
  t.n_nt = (a.M + 64 * NF - 1) / (64 * NF);
  const size_t mt = a.offsets ? std::min<size_t>(a.n, (size_t)a.n / kActBM + a.n_experts) : ((size_t)a.n + kActBM - 1) / kActBM;
  const size_t grid = 8 * ((mt * t.n_nt + 7) / 8);
  if (grid * 256 >= (size_t)1 << 32) return hipErrorInvalidValue;
  auto* kernel = act_gated(a.act) ? act_tile_kernel<kFmt, NF, true> : act_tile_kernel<kFmt, NF, false>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(256), 0, st, t);
  return hipGetLastError();
}

size_t round256(size_t n) { return (n + 255) / 256 * 256; }

}  // namespace

// The rule, and the scratch of n rows with it (0: the kernel of few rows, which needs none).
bool act_tiles_serve(int fmt, int M, int K, int groups, size_t n) {
  const size_t bytes = fmt == RMOE_FMT_BFP16 ? matrix_bytes_bfp16(M, K) : matrix_bytes(M, K);
  if (bytes >= (size_t)1 << 32) return false;  // 32-bit byte offsets into a matrix
  return n >= (groups == 1 ? 128 : (size_t)16 * groups);
}
size_t act_tiles_scratch(int fmt, int M, int K, int groups, size_t n) {
  if (!act_tiles_serve(fmt, M, K, groups, n)) return 0;
  return round256((n + kActBM) * K * 2) + round256(n * 4) + round256((size_t)groups * M * 4);
}

hipError_t launch_act_tiles(const LinAct& a, uint8_t* scratch, size_t bytes, hipStream_t st) {
  const int groups = a.offsets ? a.n_experts : 1;
  if (act_tiles_scratch(a.fmt, a.M, a.K, groups, a.n) > bytes) return hipErrorOutOfMemory;
  uint16_t* xh = reinterpret_cast<uint16_t*>(scratch);
  int32_t* xe = reinterpret_cast<int32_t*>(scratch + round256(((size_t)a.n + kActBM) * a.K * 2));
  int32_t* we = reinterpret_cast<int32_t*>(reinterpret_cast<uint8_t*>(xe) + round256((size_t)a.n * 4));
  const size_t n_x = ((size_t)a.n + 3) / 4, n_w = ((size_t)groups * a.M + 255) / 256;
  if ((n_x + n_w) * 256 >= (size_t)1 << 32) return hipErrorInvalidValue;
  hipLaunchKernelGGL(act_prep_kernel, dim3((unsigned)(n_x + n_w)), dim3(256), 0, st, PrepArgs{a, xh, xe, we, (int)n_x});
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const TileArgs t{a, xh, xe, we, 0};
  return a.fmt == RMOE_FMT_BFP16 ? launch_tiles<RMOE_FMT_BFP16, 4>(t, st) : launch_tiles<RMOE_FMT_Q4NX, 4>(t, st);
}

}  // namespace rmoe
