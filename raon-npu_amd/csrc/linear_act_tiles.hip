// y[n, M'] = RTNE(act(x[n, K] @ W^T + bias) + residual) for many rows, of one matrix or of
// each row's expert, on fp16 MFMA.
//
// Operands.  A row of x becomes fp16 times a power of two that brings its largest value into
// [2^kXTop, 2^(kXTop + 1)): bf16's 8 significant bits fit, values down to 2^-30 of the largest are exact
// (those below are cut by at most 2^-37 of it).  A weight row is brought to a power of two as well:
// bfp16's m * 2^(e-133) into [2^10, 2^11), exactly in blocks whose largest is no less than 2^-27 of the
// row's.  q4nx's m + s * n is s * (n - 8) + (m + 8 s): the first has 8 bits times 4, which fp16 holds
// exactly in groups whose scale is no less than 2^-27 of the row's largest (below, a weight is off by
// up to 2^-35 of it), and the second meets the sum of x over the group of 32 columns, of which the
// preparation keeps 22 bits: a product of its own whose 32 steps are eight groups' 8 s and m, each
// with both halves of the sum, one MFMA in nine.  Sums are fp32; the powers of two are taken back exactly.
// (With the weight rounded to fp16's 11 bits, 53,600 rows of gate/up take 425 us and not 467, but
// results depend on which kernel a number of rows selects: 3.3e-4 off in rel-L2, now 6e-5, which the
// order of the sums leaves.)
//
// Bound by the matrix pipes and the vector instructions between them, which form the weights.
// 53,600 rows of 128 experts' q4nx [1536, 2048], SwiGLU: 395 to 423 us (337 GFLOP, 800 to 850
// TFLOP/s without the group sums' MFMAs, an eighth more; torch's bf16 8192^3 reaches 1,210) behind 66
// for the rows of x; 8,192 rows of [8192, 4096] 533 us in all (1,030 TFLOP/s); 128 experts' bfp16
// [2560, 1088] of 21 rows each 97 to 101 us, in which 425 MB of weights stream at 4.2 to 4.4 TB/s.
#include <algorithm>

#include "linear_act.h"

namespace rmoe {
namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// --------------------------------------------------------------- preparation --
// A row of x is brought to [2^kXTop, 2^(kXTop + 1)).  q4nx's sums of 32 of its values then reach 2^19, 16
// times too much for fp16: they are divided by that, and so are the scales that meet the values
// themselves; the result is 2^kShift times the accumulated sums.
template <int kFmt>
constexpr int kXTop = kFmt == RMOE_FMT_BFP16 ? 14 : 13;
template <int kFmt>
constexpr int kShift = kFmt == RMOE_FMT_BFP16 ? 0 : 4;

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

// Rows of x to fp16 (zero past K_in to the end of its pair of K tiles) and their exponents, one wave
// a row; clears the counters of split tiles (256 at `arrived`, if any).  A copy's work: 53,600 rows
// of 2,048 (440 MB) take 64 us where half of them are in the caches, 90 where not, 2 more with the sums.
// kSums: also, per group of 32 columns, the sum of its fp16 values times 2^-4 as two fp16 values (22
// bits), at xs [n][K / 128 tiles][first, second][4 groups], zero like the columns past K_in.
template <bool kSums>
__global__ __launch_bounds__(256) void act_prep_kernel(LinAct a, uint16_t* __restrict__ xh, int32_t* __restrict__ xe,
                                                       uint16_t* __restrict__ xs, int* __restrict__ arrived) {
  if (arrived && blockIdx.x == 0) arrived[threadIdx.x] = 0;
  const int lane = threadIdx.x & 63, wave = wave_id();
  const size_t t = (size_t)blockIdx.x * 4 + wave;
  if (t >= (size_t)a.n) return;
  const uint4* src = reinterpret_cast<const uint4*>(a.x + t * a.ldx);
  uint4* dst = reinterpret_cast<uint4*>(xh + t * a.K);
  const int nch = a.K_in / 8, nout = (a.K_in + 2 * kTileCols - 1) / (2 * kTileCols) * (2 * kTileCols / 8);
  constexpr int kKeep = 5;  // 16-byte chunks a lane keeps between the two passes (2,560 columns)
  uint4 v[kKeep];
  float mx = 0.f;
  auto largest = [&](const uint4& q) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      mx = fmaxf(mx, fmaxf(fabsf(__uint_as_float(w[i] << 16)), fabsf(__uint_as_float(w[i] & 0xffff0000u))));
  };
#pragma unroll
  for (int i = 0; i < kKeep; ++i) {
    v[i] = lane + 64 * i < nch ? src[lane + 64 * i] : make_uint4(0u, 0u, 0u, 0u);
    largest(v[i]);
  }
  for (int c = lane + 64 * kKeep; c < nch; c += 64) largest(src[c]);
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor(mx, off, 64));
  const int e = exponent_for(mx, kXTop<kSums ? RMOE_FMT_Q4NX : RMOE_FMT_BFP16>);
  auto half = [&](const uint4& q) {
    return make_uint4(bf16_pair_to_half(q.x, e), bf16_pair_to_half(q.y, e), bf16_pair_to_half(q.z, e),
                      bf16_pair_to_half(q.w, e));
  };
  // Chunk c's eight columns; nout is a multiple of 32, so that all four lanes of a group are here.
  auto put = [&](int c, const uint4& h) {
    dst[c] = h;
    if constexpr (kSums) {
      const uint32_t w[4] = {h.x, h.y, h.z, h.w};
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f16x2 p = __builtin_bit_cast(f16x2, w[i]);
        s += (float)p[0] + (float)p[1];
      }
      s += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(s), 0xB1, 0xF, 0xF, false));  // lane ^ 1
      s += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(s), 0x4E, 0xF, 0xF, false));  // lane ^ 2
      s *= 0x1p-4f;
      const _Float16 hi = (_Float16)s, lo = (_Float16)(s - (float)hi);
      const int part = c & 3;  // the group's first lane writes the first value, its second the other
      if (part < 2)
        xs[(t * (a.K / kTileCols) + c / 16) * 8 + 4 * part + (c / 4) % 4] = __builtin_bit_cast(uint16_t, part ? lo : hi);
    }
  };
#pragma unroll
  for (int i = 0; i < kKeep; ++i)
    if (lane + 64 * i < nout) put(lane + 64 * i, half(v[i]));
  for (int c = lane + 64 * kKeep; c < nout; c += 64) put(c, c < nch ? half(src[c]) : make_uint4(0u, 0u, 0u, 0u));
  if (lane == 0) xe[t] = e;
}

// The exponent of each weight row, from the scale | min words or block exponents of its first
// K_live columns: those behind do not count (a down's padding, whose bytes may be anything).  64 rows a
// workgroup, every fourth K tile a wave: the words of 128 experts of [1536, 2048], 50 MB, at once.
__global__ __launch_bounds__(256) void row_exponents_kernel(const uint8_t* __restrict__ tiles, int fmt, int M, int K,
                                                            int K_live, int16_t* __restrict__ out) {
  __shared__ uint32_t part[4][64];
  const int lane = threadIdx.x & 63, wave = wave_id(), nkt = K / kTileCols;
  const size_t row = (size_t)blockIdx.x * kTileRows + lane;  // M % 64 == 0
  const bool b16 = fmt == RMOE_FMT_BFP16;
  const int tb = b16 ? kB16TileBytes : kTileBytes, at = b16 ? kB16MantBytes : kCodeBytes;
  const int per = b16 ? 16 : 4, unit = b16 ? 8 : 32, nlive = (K_live + unit - 1) / unit;  // a tile's blocks or groups
  const int nkt_live = (K_live + kTileCols - 1) / kTileCols;
  const uint8_t* q = tiles + (size_t)blockIdx.x * nkt * tb + at + lane * 16;
  float mx = 0.f;
  uint32_t emax = 7u;
#pragma unroll 4
  for (int kt = wave; kt < nkt_live; kt += 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(q + (size_t)kt * tb);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (b16) {
#pragma unroll
        for (int b = 0; b < 4; ++b)
          if (per * kt + 4 * i + b < nlive) emax = max(emax, (w[i] >> (8 * b)) & 0xffu);
      } else if (per * kt + i < nlive) {
        const float s = __uint_as_float(w[i] << 16), m = __uint_as_float(w[i] & 0xffff0000u);
        // m + 15 s may pass fp32's range where the codes that are taken do not.
        mx = fmaxf(mx, fmaxf(fabsf(m), fminf(fabsf(fmaf(15.f, s, m)), 0x1.fffffep127f)));
      }
    }
  }
  // The bits of positive floats are ordered as they are.
  part[wave][lane] = b16 ? emax : __float_as_uint(mx);
  __syncthreads();
  if (wave) return;
  const uint32_t m = max(max(part[0][lane], part[1][lane]), max(part[2][lane], part[3][lane]));
  emax = m;
  mx = __uint_as_float(m);
  // |m| <= 2^7 in bfp16
  out[row] = (int16_t)(b16 ? (int)emax - 133 + 7 - 10 : exponent_for(mx, 14));
}

// ---------------------------------------------------------------------- tiles --
struct TileArgs {
  LinAct a;
  const uint16_t* xh;
  const int32_t* xe;
  const uint16_t* xs;  // q4nx: see act_prep_kernel
  int n_nt;
  // One matrix's last tiles, `slices` parts of K each (kSplit; see split_tail()).
  int n_whole, slices;
  uint64_t* part;
  int* arrived;
};

constexpr int kActBM = 128;  // rows of the largest tile
// A kernel's tiles have up to 16 BF rows (BF = 2, 4, 8 fragments); a stage in LDS holds 64
// columns of them in fp16.
template <int BF>
constexpr int kStage = 16 * BF * 128;

// A wave's weights in LDS, as its tiles hold them: its 64 weight rows' sub-blocks of half a K
// tile (64 columns: two of codes, four of mantissas; 1 KB each) in a ring, then the 1 KB of
// scale | min words or exponents of a whole K tile (two, by the tile's parity).
template <int kFmt>
constexpr int kHalfBlocks = kFmt == RMOE_FMT_BFP16 ? 4 : 2;
// Stages in LDS, of rows and of weights.  Three (where two workgroups a CU still fit) gained
// nothing: 53,600 x gate/up 529 us with two, 537 with three.
constexpr int kRing = 2;
// q4nx: the group sums of a pair of K tiles, 32 bytes a row.
template <int kFmt, int BF>
constexpr int kSumBytes = kFmt == RMOE_FMT_BFP16 ? 0 : 16 * BF * 32;
template <int kFmt>
constexpr int kWaveWeights = 1024 * kHalfBlocks<kFmt> * kRing + 2 * 1024;

__device__ __forceinline__ f16x2 as_f16x2(uint32_t v) { return __builtin_bit_cast(f16x2, v); }
__device__ __forceinline__ uint32_t as_u32(f16x2 v) { return __builtin_bit_cast(uint32_t, v); }

__device__ __forceinline__ f16x2 low2(f16x2 v) { return __builtin_shufflevector(v, v, 0, 0); }

// Masks of the code unpacking in registers: (x & m) | o is one instruction then, which takes
// no literal and one scalar register.
struct CodeMasks {
  uint32_t lo, hi, magic_lo, magic_hi;  // 0x000f000f, 0x00f000f0 (scalar), 0x48004800, 0x38003800 (vector)
};
__device__ __forceinline__ CodeMasks code_masks() {
  CodeMasks k;
  asm volatile("s_mov_b32 %0, 0xf000f\n\ts_mov_b32 %1, 0xf000f0\n\tv_mov_b32 %2, 0x48004800\n\tv_mov_b32 %3, 0x38003800"
               : "=&s"(k.lo), "=&s"(k.hi), "=&v"(k.magic_lo), "=&v"(k.magic_hi));
  return k;
}
// Four codes less 8, times s 2^-4 (sm: 8 s low), in the low 16 bits' nibble order: the exponents 0x4800
// and 0x3800 make the nibble pairs of the dword 8 + n / 128 and 0.5 + n / 128, from which (n - 8) / 128
// is left exactly.  It has 4 bits and s bf16's 8: fp16 holds their product.
__device__ __forceinline__ uint2 q4_operand(uint32_t c, f16x2 sm, const CodeMasks& k) {
  const f16x2 k0 = {(_Float16)8.0625f, (_Float16)8.0625f}, k1 = {(_Float16)0.5625f, (_Float16)0.5625f};
  const f16x2 s = low2(sm);
  return make_uint2(as_u32((as_f16x2((c & k.lo) | k.magic_lo) - k0) * s), as_u32((as_f16x2((c & k.hi) | k.magic_hi) - k1) * s));
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
// and to fp16, as 8 s and m, once for all that read them (lane = weight row; four words, the first `live` of
// them: the words behind x's columns meet zeros, and are taken as zero, since they may be anything).
__device__ __forceinline__ void convert_words(uint8_t* wp, int we, int live) {
  uint4* p = reinterpret_cast<uint4*>(wp) + (threadIdx.x & 63u);
  uint4 v = *p;
  auto half = [&](uint32_t w, int i) {
    const uint32_t h = half_pair(__builtin_amdgcn_ldexpf(__uint_as_float(w << 16), 3 - we),
                                 __builtin_amdgcn_ldexpf(__uint_as_float(w & 0xffff0000u), -we));
    return i < live ? h : 0u;
  };
  *p = make_uint4(half(v.x, 0), half(v.y, 1), half(v.z, 2), half(v.w, 3));
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
    // No more than the row's own shift, 10 - 7: blocks behind x's columns may hold any exponent, and
    // their weights, which meet zeros, stay finite.
    const int e = min((int)max((ex[f] >> (16u * (lq & 1u) + 8u * g)) & 0xffu, 7u) - 133 - we[f], 3);
    const float s = __builtin_amdgcn_ldexpf(1.f, e);
    const uint32_t w = g ? (part ? v[f].w : v[f].z) : (part ? v[f].y : v[f].x);
    const uint2 r = b16_operand_half(w, as_f16x2(half_pair(s, s)));
    if (part) b.z = r.x, b.w = r.y;
    else b.x = r.x, b.y = r.y;
  }
  static __device__ __forceinline__ uint32_t chunk(int g) { return 2u * ((threadIdx.x & 63u) >> 4) + g; }
};

// One stage: two steps of 32 columns, each MF x NF products, the first with the operands b0.
// Under the first step the second's operands b1 are formed from cur, under the second the next
// stage's b0 from next, whose words are read halfway through the first; the forming is spread
// evenly: an MFMA takes 16 cycles and its issue 4, so a wave's vector instructions fit between
// its own.  Rows are read two fragments ahead.  Chunk c (16 bytes) of row r of a stage sits at
// chunk c ^ (r / 2 % 8): the 16 rows of a fragment then cover all 64 banks.
template <int kFmt, int BF, int MF, int NF, typename Copy, typename Read>
__device__ __forceinline__ void mfma_stage(const uint8_t* stage, uint4 (&b0)[NF], const StageWeights<kFmt, NF>& cur,
                                           StageWeights<kFmt, NF>& next, const int (&we)[NF], const CodeMasks& masks,
                                           f32x4 (&acc)[BF][NF], Copy copy, Read read) {
  const uint32_t l16 = threadIdx.x & 15u;
  const uint8_t* p[2];
#pragma unroll
  for (int g = 0; g < 2; ++g) p[g] = stage + 128u * l16 + 16u * (StageWeights<kFmt, NF>::chunk(g) ^ (l16 >> 1));
  auto row = [&](int i) { return *reinterpret_cast<const uint4*>(p[i / MF] + 2048 * (i % MF)); };
  uint4 x[2 * MF], b1[NF];
  x[0] = row(0);
  x[1] = row(1);
#pragma unroll
  for (int i = 0; i < 2 * MF; ++i) {
    const int m = i % MF;
    if (i + 2 < 2 * MF) x[i + 2] = row(i + 2);
    if (i == MF / 2) read();
    if (i == MF) {
      next.arrange();
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // read()'s place may be copied to from here on
    }
    copy(i);
#pragma unroll
    for (int f = 0; f < NF; ++f)
      acc[m][f] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, x[i]),
                                                         __builtin_bit_cast(f16x8, i < MF ? b0[f] : b1[f]), acc[m][f], 0, 0, 0);
#pragma unroll
    for (int q = 2 * NF * m / MF; q < 2 * NF * (m + 1) / MF; ++q) {
      if (i < MF) cur.form(1, q / 2, q % 2, we, masks, b1[q / 2]);
      else next.form(0, q / 2, q % 2, we, masks, b0[q / 2]);
    }
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
// All but the last kPending copies of this wave have landed, then the workgroup meets.
template <int kPending>
__device__ __forceinline__ void copies_landed() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kPending) : "memory");
  __syncthreads();
}

// One tile of up to 16 MF rows x 64 NW weight rows over the K tiles [kt0, kt0 + nkt); each of
// its NW waves takes all rows and 16 NF = 64 weight rows of its own (w: the matrix; wo: byte
// offset of weight row `lane` of the 64).
// Stages s of 64 columns.  Rows are copied R - 1 stages ahead into a ring of R = kRing, and
// weights, which no other wave reads, R + 1 ahead into the place that stage s + 1's left when
// their words went to registers, so that operands are formed under products throughout.  A
// wave waits in the order of its copies: at a stage's end for those issued by the end of the
// stage R - 1 before.  One barrier a stage.  Copies past the end repeat the last stage's.
template <int kFmt, int BF, int MF, int NF, int NW>
__device__ __forceinline__ void tile_product(const TileArgs& t, const uint8_t* w, uint32_t wo, int we_lane,
                                             const int (&we)[NF], int row0, int kt0, int nkt, uint8_t* lds,
                                             f32x4 (&acc)[BF][NF]) {
  static_assert(NF == 4, "64 weight rows a wave");
  constexpr int kTB = kFmt == RMOE_FMT_BFP16 ? kB16TileBytes : kTileBytes, kBlocks = kHalfBlocks<kFmt>;
  constexpr int R = kRing, kAhead = R - 1;
  const int lane = threadIdx.x & 63, wave = wave_id() % NW, ns = 2 * nkt;
  w += (size_t)kt0 * kTB;
  const uint32_t lds0 = (uint32_t)(uintptr_t)lds;
  const int wbase = R * kStage<BF> + wave * kWaveWeights<kFmt>, pbase = wbase + R * 1024 * kBlocks;
  // Copy q = wave + NW i fills LDS rows 8q..8q+7 (1 KB): lane L brings row 8q + L / 8 the chunk
  // that sits at position L % 8.  Rows past the tile are the next tiles' or, behind the last
  // row, the kActBM spare rows of the scratch; their results are not stored.
  constexpr int kRowCopies = 2 * MF / NW;
  const uint8_t* xb = reinterpret_cast<const uint8_t*>(t.xh + (size_t)row0 * t.a.K) + (size_t)kt0 * 256;
  const uint32_t ld = 2u * (uint32_t)t.a.K;
  const uint32_t xo = (uint32_t)(8 * wave + lane / 8) * ld + 16u * (uint32_t)((lane % 8) ^ ((4 * wave + lane / 16) % 8));
  uint32_t rows0 = lds0 + 1024u * (uint32_t)wave;
  asm volatile("" : "+s"(rows0));  // kept in a scalar register
  auto row_copy = [&](int i, int s, uint32_t slot) {
    copy16(xb + 128 * min(s, ns - 1) + (size_t)(8 * NW * i) * ld, xo, rows0 + slot + (uint32_t)(1024 * NW * i));
  };
  // Stage q's weights, q of the parity j, at byte `at` of the wave's ring: kBlocks + 1 - j copies.
  auto weight_copy = [&](int i, int q, uint32_t at) {
    const int j = q & 1;
    const uint8_t* tile = w + (size_t)min(q >> 1, nkt - 1) * kTB;
    if (i < kBlocks) copy16(tile + 1024 * (kBlocks * j + i), wo, lds0 + (uint32_t)wbase + at + (uint32_t)(1024 * i));
    else copy16(tile + 2048 * kBlocks, wo, lds0 + (uint32_t)(pbase + 1024 * ((q >> 1) & 1)));
  };
  auto load_weights = [&](int q, uint32_t at) {
#pragma unroll
    for (int i = 0; i < kBlocks; ++i) weight_copy(i, q, at);
    if ((q & 1) == 0) weight_copy(kBlocks, q, at);
  };
  // A stage's copies, spread over its 2 MF turns (a wave stands still at a copy until the
  // copies before it are taken up): rows under the first step, weights under the second.
  auto copies = [&](int i, int s, int q, int nw, uint32_t there, uint32_t at) {
#pragma unroll
    for (int c = 0; c < kRowCopies; ++c)
      if (i == (2 * c + 1) * MF / (2 * kRowCopies)) row_copy(c, s, there);
#pragma unroll
    for (int c = 0; c < nw; ++c)
      if (i == MF + (c + 1) * (MF - 1) / nw) weight_copy(c, q, at);
  };
  // q4nx: sum over the groups of (m + 8 s) X, X the group's sum of x, by products whose 32 steps are the words
  // (8 s, m) of two K tiles' groups, met by X's first part (lane quarters 0, 1: tile 0, 1) and its
  // second (2, 3).  Tile kt's sums and the next one's (past the last tile its own again, met by zeros).
  const uint8_t* sb = reinterpret_cast<const uint8_t*>(t.xs) + (size_t)row0 * (t.a.K / kTileCols) * 16;
  const int sbase = R * kStage<BF> + NW * kWaveWeights<kFmt>;
  // The lane, as a value that the compiler does not know: the addresses below are formed where they are
  // used, not kept in registers across the products.
  auto lane_here = [&]() {
    uint32_t l = threadIdx.x & 63u;
    asm volatile("" : "+v"(l));
    return l;
  };
  auto sums_copy = [&](int kt) {
    const uint32_t l = lane_here(), n = (uint32_t)t.a.K / kTileCols;
    const int part = wave % (MF / 2);  // 32 rows
    copy16(sb, ((32u * (uint32_t)part + l / 2) * n + (uint32_t)kt0 + min((uint32_t)kt + l % 2, (uint32_t)nkt - 1u)) * 16u,
           lds0 + (uint32_t)(sbase + 1024 * part));
  };
  auto add_mins = [&](int kt) {
    const uint32_t l = lane_here(), l16 = l & 15u, lq = l >> 4;
    const bool in = (lq & 1u) == 0u || kt + 1 < nkt;
    const uint8_t* wp = lds + pbase + 1024 * ((kt + (lq & 1u)) & 1) + 16u * l16;
    const uint8_t* sp = lds + sbase + 32u * l16 + 16u * (lq & 1u) + 8u * (lq >> 1);
    uint4 b[NF];
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      b[f] = *reinterpret_cast<const uint4*>(wp + 256 * f);
      if (!in) b[f] = make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int m = 0; m < MF; ++m) {
      const uint2 v = *reinterpret_cast<const uint2*>(sp + 512 * m);
      const uint4 x = make_uint4(__builtin_amdgcn_perm(v.x, v.x, 0x01000100u), __builtin_amdgcn_perm(v.x, v.x, 0x03020302u),
                                 __builtin_amdgcn_perm(v.y, v.y, 0x01000100u), __builtin_amdgcn_perm(v.y, v.y, 0x03020302u));
#pragma unroll
      for (int f = 0; f < NF; ++f)
        acc[m][f] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, x), __builtin_bit_cast(f16x8, b[f]),
                                                           acc[m][f], 0, 0, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  const CodeMasks masks = code_masks();
#pragma unroll
  for (int s = 0; s < kAhead; ++s)
#pragma unroll
    for (int i = 0; i < kRowCopies; ++i) row_copy(i, s, (uint32_t)(s * kStage<BF>));
#pragma unroll
  for (int s = 0; s < R; ++s) load_weights(s, (uint32_t)(s * 1024 * kBlocks));
  copies_landed<0>();
  const int groups = (t.a.K_in + 31) / 32 - 4 * kt0;  // that x's columns reach, from this slice's first on
  if constexpr (kFmt == RMOE_FMT_Q4NX) convert_words(lds + pbase, we_lane, groups);
  StageWeights<kFmt, NF> cur, next;
  uint4 b0[NF];
  cur.read(lds + wbase, lds + pbase, 0);
  cur.arrange();
#pragma unroll
  for (int q = 0; q < 2 * NF; ++q) cur.form(0, q / 2, q % 2, we, masks, b0[q / 2]);
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  load_weights(R, 0u);
  // Ring offsets: stage s's rows, stage s + kAhead's rows, stage s + 1's weights.
  uint32_t here = 0u, there = (uint32_t)(kAhead * kStage<BF>), ws = (uint32_t)(1024 * kBlocks);
  auto turn = [&]() {
    here = here == (uint32_t)((R - 1) * kStage<BF>) ? 0u : here + (uint32_t)kStage<BF>;
    there = there == (uint32_t)((R - 1) * kStage<BF>) ? 0u : there + (uint32_t)kStage<BF>;
    ws = ws == (uint32_t)((R - 1) * 1024 * kBlocks) ? 0u : ws + (uint32_t)(1024 * kBlocks);
  };
  // Copies that may be in flight at the end of a stage: the last, of its weights, with words
  // every second stage.
  static_assert(R == 2, "counts of the copies in flight");
  constexpr int kEvenEnd = kBlocks, kOddEnd = kBlocks + 1;
#pragma unroll 1
  for (int kt = 0; kt < nkt; ++kt) {
    const uint8_t* wp = lds + pbase + 1024 * (kt & 1);
    const uint8_t* wp_next = lds + pbase + 1024 * ((kt + 1) & 1);
    const int s = 2 * kt;
    mfma_stage<kFmt, BF, MF, NF>(
        lds + here, b0, cur, next, we, masks, acc,
        [&](int i) {
          // The last pair's sums have been read, a barrier ago at least.
          if (kFmt == RMOE_FMT_Q4NX && i == 0 && kt % 2 == 0) sums_copy(kt);
          copies(i, s + kAhead, s + 1 + R, kBlocks + R % 2, there, ws);
        },
        [&] { next.read(lds + wbase + ws, wp, 1); });
    copies_landed<kEvenEnd>();
    turn();
    if constexpr (kFmt == RMOE_FMT_Q4NX) {
      // The next tile's words have landed (past the last tile the operands are not used); those of kt
      // stay until the coming stage's last copies.
      convert_words(lds + pbase + 1024 * ((kt + 1) & 1), we_lane, groups - 4 * (kt + 1));
      if (kt % 2 == 0) add_mins(kt);
    }
    mfma_stage<kFmt, BF, MF, NF>(
        lds + here, b0, next, cur, we, masks, acc,
        [&](int i) {
          copies(i, s + 1 + kAhead, s + 2 + R, kBlocks + 1 - R % 2, there, ws);
        },
        [&] { cur.read(lds + wbase + ws, wp_next, 0); });
    copies_landed<kOddEnd>();
    turn();
  }
  copies_landed<0>();  // the epilogue reuses the memory
}

// Tiles of 16 BF rows x 64 NW weight rows by KS groups of NW waves, which take a KS-th of K each.
// kSplit: the workgroups behind those of n_whole tiles take a slice of K each of the last
// tiles, and the last of a tile to arrive adds their sums in the order of the slices.
template <int kFmt, int NF, bool kGated, int BF, int NW, int KS, bool kSplit>
__global__ __launch_bounds__(64 * NW * KS, BF == 8 ? 2 : BF == 4 ? 3 : 4) void act_tile_kernel(TileArgs t) {
  constexpr int kLds = kRing * kStage<BF> + NW * kWaveWeights<kFmt> + kSumBytes<kFmt, BF>, kTile = 16 * BF;
  static_assert(kLds <= 80 * 1024, "two groups a CU");
  __shared__ __attribute__((aligned(16))) uint8_t lds[KS * kLds];
  constexpr int kCols = 16 * NF * NW, kOut = kGated ? kCols / 2 : kCols;
  constexpr int kTB = kFmt == RMOE_FMT_BFP16 ? kB16TileBytes : kTileBytes;
  const LinAct& a = t.a;
  RowTiles<kTile> rt;
  const int n_mt = a.offsets ? rt.total(a.offsets, a.n_experts, a.n) : (a.n + kTile - 1) / kTile;
  const int total = kSplit ? t.n_whole : n_mt * t.n_nt, per = (total + 7) / 8, slot = (int)blockIdx.x / 8;
  int id = ((int)blockIdx.x % 8) * per + slot, slice = 0, slices = 1;
  if (kSplit && (int)blockIdx.x >= 8 * per) {
    const int p = (int)blockIdx.x - 8 * per;
    slices = t.slices;
    id = total + p / slices;
    slice = p % slices;
    if (id >= n_mt * t.n_nt) return;
  } else if (slot >= per || id >= total) {
    return;
  }
  const int nt = id % t.n_nt;
  int e = 0, row0 = id / t.n_nt * kTile, nrow = min(kTile, a.n - row0);
  if (a.offsets) rt.find(id / t.n_nt, e, row0, nrow);
  const int wave = wave_id() % NW, group = wave_id() / NW, nkt = a.K / kTileCols, width = kGated ? a.M / 2 : a.M;
  const uint8_t* tiles = a.tiles + (size_t)e * a.wstride;
  // The wave's weight rows: 64 consecutive ones, or 32 gate rows and their up rows.  Columns
  // past the matrix (its width is a multiple of 64) repeat its first rows.
  const int c0 = nt * kOut + wave * (kOut / NW), base = c0 < width ? c0 : 0;
  auto row_of = [&](int r) { return kGated && r >= 32 ? width + base + r - 32 : base + r; };
  const int wr = row_of(threadIdx.x & 63);
  const uint32_t wo = (uint32_t)(wr / kTileRows) * (uint32_t)(nkt * kTB) + (uint32_t)(wr % kTileRows) * 16u;
  const int16_t* wes = a.exps + (size_t)e * a.M;
  int we[NF];
#pragma unroll
  for (int f = 0; f < NF; ++f) we[f] = wes[row_of(16 * f + (threadIdx.x & 15))];
  f32x4 acc[BF][NF];
#pragma unroll
  for (int m = 0; m < BF; ++m)
#pragma unroll
    for (int f = 0; f < NF; ++f) acc[m][f] = f32x4{0.f, 0.f, 0.f, 0.f};
  // A short tile multiplies only the fragments that hold rows.
  static_assert(!kSplit || KS == 1, "one way to split K");
  const int nkt_in = (a.K_in + kTileCols - 1) / kTileCols, half = (nkt_in + KS - 1) / KS;  // K % 256 == 0
  const int kt0 = kSplit ? slice * nkt_in / slices : group * half;
  const int nk = kSplit ? (slice + 1) * nkt_in / slices - kt0 : half;
  uint8_t* mine = lds + group * kLds;
  if (BF == 8 && nrow > 64) tile_product<kFmt, BF, BF, NF, NW>(t, tiles, wo, wes[wr], we, row0, kt0, nk, mine, acc);
  else if (BF >= 4 && nrow > 32)
    tile_product<kFmt, BF, BF < 4 ? BF : 4, NF, NW>(t, tiles, wo, wes[wr], we, row0, kt0, nk, mine, acc);
  else tile_product<kFmt, BF, 2, NF, NW>(t, tiles, wo, wes[wr], we, row0, kt0, nk, mine, acc);

  if constexpr (kSplit) {
    if (slices > 1) {
      // Stores of device scope go past the XCD's L2: no fence has to write it back (all of it, for
      // every slice: 25 us more).  The few that read invalidate theirs.
      constexpr int kPairs = 2 * BF * NF;
      uint64_t* p = t.part + (size_t)(id - total) * slices * (kPairs * 256) + threadIdx.x;
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        const f32x4 v = acc[i / 2 / NF][i / 2 % NF];
        const uint64_t q = (uint64_t)__float_as_uint(v[2 * (i % 2) + 1]) << 32 | __float_as_uint(v[2 * (i % 2)]);
        __hip_atomic_store(p + ((size_t)slice * kPairs + i) * 256, q, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      int* last = reinterpret_cast<int*>(lds);
      if (threadIdx.x == 0) *last = atomicAdd(t.arrived + (id - total), 1) == slices - 1;
      __syncthreads();
      if (!*last) return;
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
#pragma unroll
      for (int i = 0; i < BF * NF; ++i) acc[i / NF][i % NF] = f32x4{0.f, 0.f, 0.f, 0.f};
      constexpr int kBatch = 32;  // loads in flight
#pragma unroll 1
      for (int s = 0; s < slices; ++s) {
#pragma unroll
        for (int i0 = 0; i0 < kPairs; i0 += kBatch) {
          uint64_t q[kBatch];
#pragma unroll
          for (int i = 0; i < kBatch; ++i) q[i] = p[(size_t)(i0 + i) * 256];
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int i = 0; i < kBatch; ++i) {
            f32x4& v = acc[(i0 + i) / 2 / NF][(i0 + i) / 2 % NF];
            v[2 * (i % 2)] += __uint_as_float((uint32_t)q[i]);
            v[2 * (i % 2) + 1] += __uint_as_float((uint32_t)(q[i] >> 32));
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        p += (size_t)kPairs * 256;
      }
      __syncthreads();  // the epilogue reuses the memory
    }
  }

  // Epilogue: sums and bias through LDS as fp32, kRows rows at a time, so that the activation
  // has its operands at hand and residual and y move 16 bytes a thread.  Columns of
  // different lq go to different banks: column c of row r sits at c ^ 16 (r / 4 % 4).
  constexpr int kAll = KS * kLds;
  constexpr int kRows = kAll >= kTile * kCols * 4 ? kTile : kAll >= kTile / 2 * kCols * 4 ? kTile / 2 : kTile / 4;
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
  for (int r0 = 0; r0 < kTile; r0 += kRows) {
    if (r0 >= nrow) break;
    if (r0) __syncthreads();
    auto at_column = [&](int f) {
      return wave * (kOut / NW) + l16 + (kGated ? 16 * (f % (NF / 2)) + (f >= NF / 2 ? kOut : 0) : 16 * f);
    };
    if constexpr (KS > 1) {  // the second group's sums first
      if (group == 1) {
#pragma unroll
        for (int m = r0 / 16; m < (r0 + kRows) / 16; ++m)
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int f = 0; f < NF; ++f)
              out[(16 * m + 4 * lq + i - r0) * kCols + (at_column(f) ^ (16 * lq))] = acc[m][f][i];
      }
      __syncthreads();
    }
    if (group == 0) {
#pragma unroll
      for (int m = r0 / 16; m < (r0 + kRows) / 16; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = 16 * m + 4 * lq + i;
          const int xe = t.xe[row0 + min(r, nrow - 1)];
          float* o = out + (r - r0) * kCols;
#pragma unroll
          for (int f = 0; f < NF; ++f) {
            float& v = o[at_column(f) ^ (16 * lq)];
            v = __builtin_amdgcn_ldexpf(KS > 1 ? acc[m][f][i] + v : acc[m][f][i], xe + we[f] + kShift<kFmt>) + bias[f];
          }
        }
    }
    __syncthreads();
    const int rows = min(kRows, nrow - r0), cols = min(kOut, width - nt * kOut);
#pragma unroll 1
    for (int i = tid; i < rows * (kOut / 8); i += 64 * NW * KS) {
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

template <int kFmt, int BF, int NW = 4, int KS = 1, bool kSplit = false>
hipError_t launch_tiles(const TileArgs& t0, hipStream_t st) {
  constexpr int NF = 4, kTile = 16 * BF;
  TileArgs t = t0;
  const LinAct& a = t.a;
  t.n_nt = (a.M + 16 * NF * NW - 1) / (16 * NF * NW);
  const size_t mt = a.offsets ? std::min<size_t>(a.n, (size_t)a.n / kTile + a.n_experts) : ((size_t)a.n + kTile - 1) / kTile;
  size_t grid = 8 * ((mt * t.n_nt + 7) / 8);
  if (kSplit) grid = 8 * (((size_t)t.n_whole + 7) / 8) + (mt * t.n_nt - t.n_whole) * t.slices;
  constexpr int kThreads = 64 * NW * KS;
  if (grid * kThreads >= (size_t)1 << 32) return hipErrorInvalidValue;
  auto* kernel = act_gated(a.act) ? act_tile_kernel<kFmt, NF, true, BF, NW, KS, kSplit>
                                  : act_tile_kernel<kFmt, NF, false, BF, NW, KS, kSplit>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(kThreads), 0, st, t);
  return hipGetLastError();
}
// Tiles of 128 x 256 and of 64 x 128 weight rows over one matrix of M rows.
size_t large_tiles(int M, size_t n) { return (n + 127) / 128 * ((M + 255) / 256); }
size_t small_tiles(int M, size_t n) { return (n + 63) / 64 * (M / 128); }
constexpr size_t kFillLarge = 200;
// Fewer 64 x 128 tiles than this are left to linear_act_kernel (see act_tiles_serve()).
constexpr size_t fill_small(int fmt) { return fmt == RMOE_FMT_BFP16 ? 256 : 320; }

// Large tiles past a multiple of 256: a CU takes 50 us for one of [2176, 2560] alone and 72 for
// two, so a few of them beyond are cut along K into three or four slices, of two K tiles at
// least, and as many as there are CUs.  q4nx, 4,096 rows of [2176, 2560] (32 beyond) 87 us
// whole, in 2, 3 and 4 slices 77, 71 and 70; 6,000 of [1536, 2048] (26) 75, and 68, 64 and 62; 5,060
// of [2176, 2560] (104) 90, in 2 slices 90.  (Six and eight slices of the 32 were slower than four by
// 5 and 13 %.)  Returns the slices (1: none are cut).
constexpr size_t kCus = 256, kMinSlices = 3, kMaxSlices = 4;
size_t split_tail(size_t tiles, int K_in) {
  const size_t over = tiles % kCus;
  if (tiles < kCus || over == 0) return 1;
  const size_t slices = std::min<size_t>({kCus / over, kMaxSlices, (size_t)K_in / (2 * kTileCols)});
  return slices < kMinSlices ? 1 : slices;
}
constexpr size_t kTailBytes = kCus * kActBM * 256 * 4;  // the sums of at most kCus slices

// By expert: by the rows an expert has in the mean (128 experts, q4nx gate/up [1536, 2048], tiles
// of 32, 64 and 128 rows: 16 rows 59, 59 and 67 us, 28 rows 74, 72 and 83, 44 rows 110, 86 and 100,
// 62 rows 132, 113 and 123, 94 rows 180, 147 and 138; bfp16 down [2560, 1088]: 12 rows 100, 108 and 108, 47 rows 147,
// 138 and 137, 70 rows 180, 164 and 158).
// One matrix: 128 x 256 from kFillLarge tiles of it on, below that 64 x 128 by two groups of K,
// which make 3.75 times the workgroups (q4nx [2176, 2560], SwiGLU, 64 x 128 / 128 x 256: 1,024
// rows 37 / 57 us, 2,048 (144 large tiles) 58 / 61, 3,000 (216) 70 / 62, 4,096 85 / 87).
template <int kFmt>
hipError_t pick_tiles(const TileArgs& t, hipStream_t st) {
  const LinAct& a = t.a;
  if (t.slices > 1) return launch_tiles<kFmt, 8, 4, 1, true>(t, st);
  if (!a.offsets || a.n_experts == 1)
    return large_tiles(a.M, a.n) >= kFillLarge ? launch_tiles<kFmt, 8>(t, st) : launch_tiles<kFmt, 4, 2, 2>(t, st);
  const size_t rows = (size_t)a.n / a.n_experts;
  if (rows <= 24) return launch_tiles<kFmt, 2>(t, st);
  if (rows <= 64) return launch_tiles<kFmt, 4>(t, st);
  return launch_tiles<kFmt, 8>(t, st);
}

size_t round256(size_t n) { return (n + 255) / 256 * 256; }
// q4nx's group sums of n rows and the spare ones.
size_t sum_bytes(int K, size_t n) { return round256((n + kActBM) * (K / kTileCols) * 16); }

}  // namespace

hipError_t launch_row_exponents(const uint8_t* tiles, int fmt, int M, int K, int K_live, int16_t* exps, hipStream_t st) {
  hipLaunchKernelGGL(row_exponents_kernel, dim3(M / kTileRows), dim3(256), 0, st, tiles, fmt, M, K, K_live, exps);
  return hipGetLastError();
}

// Which rows this kernel serves, against linear_act_kernel (whose cost grows with every 32 rows).
// One matrix: from fill_small() tiles of 64 x 128 on (this kernel / that one, with SwiGLU.  q4nx:
// [2176, 2560], 1,100 rows (306 tiles) 39 / 38 us, 1,250 rows (340) 39 / 45; [1536, 2048], 1,500 rows
// (288) 34 / 31, 1,700 rows (324) 35 / 37; [512, 2048], 4,500 rows (284) 40 / 33, 5,500 rows (344) 39 / 39,
// 6,500 rows (408) 39 / 44.  bfp16: [2176, 2560], 1,024 rows (272) 34 / 40; [1536, 2048], 1,024 rows (192)
// 24 / 22, 1,360 rows (264) 31 / 34; [512, 2048], 4,096 rows (256) 31 / 30, 5,500 rows (344) 35 / 41).  By
// expert: from one row an expert on (128 experts, q4nx gate/up [1536, 2048]: 128 rows 43 / 42 us, 700
// rows 55 / 69, 8,000 rows 115 / 185; down [2048, 768]: 128 rows 27 / 32).
bool act_tiles_serve(int fmt, int M, int K, int groups, size_t n) {
  const size_t bytes = fmt == RMOE_FMT_BFP16 ? matrix_bytes_bfp16(M, K) : matrix_bytes(M, K);
  if (bytes >= (size_t)1 << 32) return false;  // 32-bit byte offsets into a matrix
  return groups > 1 ? n >= (size_t)groups : small_tiles(M, n) >= fill_small(fmt);
}
size_t act_tiles_scratch(int fmt, int M, int K, int groups, size_t n) {
  if (!act_tiles_serve(fmt, M, K, groups, n)) return 0;
  const bool tail = groups == 1 && large_tiles(M, n) >= kCus;
  return round256((n + kActBM) * K * 2) + round256(n * 4) + (size_t)groups * M * sizeof(int16_t) +
         (fmt == RMOE_FMT_Q4NX ? sum_bytes(K, n) : 0) + (tail ? kTailBytes + kCus * 4 : 0);
}

hipError_t launch_act_tiles(const LinAct& a, uint8_t* scratch, size_t bytes, hipStream_t st) {
  if (act_tiles_scratch(a.fmt, a.M, a.K, a.offsets ? a.n_experts : 1, a.n) > bytes) return hipErrorOutOfMemory;
  const size_t groups = ((size_t)a.n + 3) / 4;
  if (groups * 256 >= (size_t)1 << 32) return hipErrorInvalidValue;
  uint16_t* xh = reinterpret_cast<uint16_t*>(scratch);
  int32_t* xe = reinterpret_cast<int32_t*>(scratch + round256(((size_t)a.n + kActBM) * a.K * 2));
  TileArgs t{a, xh, xe, nullptr, 0, 0, 1, nullptr, nullptr};
  uint8_t* next = reinterpret_cast<uint8_t*>(xe) + round256((size_t)a.n * 4);
  // Narrower x: the kept exponents count weights that take no part, which may be of any size.  Those
  // of the columns that do are taken for this call.
  const int unit = a.fmt == RMOE_FMT_BFP16 ? 8 : 32, rows = (a.offsets ? a.n_experts : 1) * a.M;
  if ((a.K_in + unit - 1) / unit != (a.live + unit - 1) / unit) {
    int16_t* exps = reinterpret_cast<int16_t*>(next);
    t.a.exps = exps;
    const hipError_t e = launch_row_exponents(a.tiles, a.fmt, rows, a.K, a.K_in, exps, st);
    if (e != hipSuccess) return e;
  }
  next += (size_t)rows * sizeof(int16_t);  // M is a multiple of 128
  const bool q4 = a.fmt == RMOE_FMT_Q4NX;
  uint16_t* xs = reinterpret_cast<uint16_t*>(next);
  if (q4) {
    t.xs = xs;
    next += sum_bytes(a.K, a.n);
  }
  const size_t tiles = large_tiles(a.M, a.n);
  if (!a.offsets && (t.slices = (int)split_tail(tiles, a.K_in)) > 1) {
    t.n_whole = (int)(tiles / kCus * kCus);
    t.part = reinterpret_cast<uint64_t*>(next);
    t.arrived = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(t.part) + kTailBytes);
  }
  hipLaunchKernelGGL(q4 ? act_prep_kernel<true> : act_prep_kernel<false>, dim3((unsigned)groups), dim3(256), 0, st, a, xh, xe,
                     xs, t.arrived);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  return q4 ? pick_tiles<RMOE_FMT_Q4NX>(t, st) : pick_tiles<RMOE_FMT_BFP16>(t, st);
}

}  // namespace rmoe
