// Tokens to expert-sorted rows and back, with their gradients.
//
//   sort:       pos(a) = #{b : 0 <= e_b < e_a} + #{b < a : e_b = e_a} for the assignments
//               a = t k + r with expert e_a = ids[t][r] (negative: the route has no row);
//               rows[pos(a)] = x[t], order[pos(a)] = a, inv[a] = pos(a) or -1,
//               offsets[e] = #{b : 0 <= e_b < e}.
//   its gradient:  dx[t] = sum_r drows[inv[t][r]].
//   combine:       out[t] = sum_r w[t][r] rows[inv[t][r]], products and sums in fp32 in the
//               order of the sorted positions, which is ascending expert id as in the
//               grouped prefill's combine, one rounding at the end.
//   its gradient:  drows[inv[t][r]] = w[t][r] dout[t];  dw[t][r] = <dout[t], rows[inv[t][r]]>.
//
// Every one of them moves k rows per token and is bound by HBM; small calls are bound by
// their chain of dependent loads (routes, then rows) and the launch (4 us for four tokens).
// Each element is read and written once.  The sort and the combine's gradient take a workgroup a
// token, which keeps the k positions (the dot products' shares) in LDS; the sums take a wave for
// one token and 1 KB of its columns, which finds the k positions in its own lanes, without LDS or
// barriers.  6,700 tokens of 8 rows of 4 KB (240 MB), buffers not in the caches: the sort 58 us
// (10 of them for the positions), the combine 49 (4.9 TB/s); 4,099 tokens: the combine's
// gradient 60 (286 MB, 4.8 TB/s; a copy reaches 4.8).
#include <algorithm>

#include "../../include/raon_moe.h"
#include "rmoe_internal.h"

namespace rmoe {
namespace {

constexpr int kMaxRoutes = 16;
constexpr int kErrExpert = 4, kErrPosition = 16;

// Assignments up to which every token's workgroup finds its own positions by k comparisons
// with each of them, in one launch with the rows; up to which every chunk's workgroup counts
// all of them, in two launches; beyond, four.  H 256, k 8, by events / replayed in a graph: 1,024
// assignments in one 7.4 / 6.6 us, in two 9.6 / 7.0; 2,048 9.6 / 9.7 and 9.8 / 7.2; 4,096 in two
// 9.7 / 7.5, in four 14.9 / 11.4; 32,768 12.9 and 16.3; 53,600 16.8 and 18.8; 72,000 20.0 and 19.7;
// 128,000 31 and 27.
constexpr int kOneLaunch = 1024, kTwoLaunches = 65536;

// One element of a type as fp32, and fp32 rounded to it (RTNE).
template <int DT>
struct Elem;
template <>
struct Elem<RMOE_DT_BF16> {
  typedef uint16_t T;
  static __device__ __forceinline__ float get(T v) { return bf16_to_f32(v); }
  static __device__ __forceinline__ T put(float v) { return (T)f32_to_bf16(v); }
};
template <>
struct Elem<RMOE_DT_F16> {
  typedef uint16_t T;
  static __device__ __forceinline__ float get(T v) { return (float)__builtin_bit_cast(_Float16, v); }
  static __device__ __forceinline__ T put(float v) { return __builtin_bit_cast(uint16_t, (_Float16)v); }
};
template <>
struct Elem<RMOE_DT_F32> {
  typedef float T;
  static __device__ __forceinline__ float get(T v) { return v; }
  static __device__ __forceinline__ T put(float v) { return v; }
};

// N elements in one load: 16 bytes, or (N = 1) one element where rows are not 16-byte aligned.
template <int DT, int N>
struct Pack {
  typename Elem<DT>::T v[N];
};
template <int DT, int N, bool kOnce = false>
__device__ __forceinline__ Pack<DT, N> load_pack(const typename Elem<DT>::T* p) {
  if constexpr (N == 1) {
    Pack<DT, N> r;
    r.v[0] = *p;
    return r;
  } else {
    static_assert(sizeof(Pack<DT, N>) == 16, "16-byte packs");
    if constexpr (kOnce)
      return __builtin_bit_cast(Pack<DT, N>, __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(p)));
    else
      return __builtin_bit_cast(Pack<DT, N>, *reinterpret_cast<const u32x4_t*>(p));
  }
}
template <int DT, int N>
__device__ __forceinline__ void store_pack(typename Elem<DT>::T* p, const Pack<DT, N>& r) {
  if constexpr (N == 1) *p = r.v[0];
  else *reinterpret_cast<u32x4_t*>(p) = __builtin_bit_cast(u32x4_t, r);
}

// ------------------------------------------------------------------- positions --
// The expert of an assignment, -1 where it has none; an id past the experts is flagged.
__device__ __forceinline__ int route_expert(int id, int E, int* err) {
  if (id >= E) atomicOr(err, kErrExpert);
  return id < 0 || id >= E ? -1 : id;
}

// Up to kOneLaunch assignments: workgroup t counts its own token's positions over all ids (4 KB
// at most, read from L2), workgroup T the offsets; no workspace.
struct SortArgs {
  const int32_t* ids;
  int T, k, E, n;
  int32_t *order, *inv, *offsets;
  int* err;
};
__device__ void small_offsets(const SortArgs& a, int* hist) {
  const int tid = threadIdx.x;
  hist[tid] = 0;
  __syncthreads();
  for (int j0 = tid; j0 < a.n; j0 += 8 * 256) {  // eight loads in flight
    int id[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) id[u] = j0 + 256 * u < a.n ? a.ids[j0 + 256 * u] : -1;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int e = route_expert(id[u], a.E, a.err);
      if (e >= 0) atomicAdd(&hist[e], 1);
    }
  }
  __syncthreads();
  if (tid < 64) {
    int run = 0;
    for (int e0 = 0; e0 < a.E; e0 += 64) {
      const int e = e0 + tid, own = e < a.E ? hist[e] : 0;
      int incl = own;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int y = __shfl_up(incl, d, 64);
        if (tid >= d) incl += y;
      }
      if (e < a.E) a.offsets[e] = run + incl - own;
      run += __shfl(incl, 63, 64);
    }
    if (tid == 0) a.offsets[a.E] = run;
  }
}

// The row copy of one wave: bytes [16 lane ...] of token t's row to its k rows.
template <typename U>
__device__ __forceinline__ void scatter_row(const uint8_t* __restrict__ src, uint8_t* __restrict__ rows, size_t rb,
                                            const int* pos, int k, int first, int step) {
  const int n = (int)(rb / sizeof(U));
  for (int c = first; c < n; c += step) {
    const U v = reinterpret_cast<const U*>(src)[c];
    for (int r = 0; r < k; ++r)
      if (pos[r] >= 0) reinterpret_cast<U*>(rows + (size_t)pos[r] * rb)[c] = v;
  }
}

template <typename U>
__global__ __launch_bounds__(256) void sort_small_kernel(SortArgs a, const uint8_t* __restrict__ x,
                                                         uint8_t* __restrict__ rows, size_t rb) {
  __shared__ int hist[256];
  __shared__ int part[4][kMaxRoutes], pos[kMaxRoutes];
  const int t = blockIdx.x, tid = threadIdx.x, wave = wave_id(), lane = tid & 63;
  if (t == a.T) {
    small_offsets(a, hist);
    return;
  }
  int e[kMaxRoutes], cnt[kMaxRoutes];
#pragma unroll
  for (int r = 0; r < kMaxRoutes; ++r) {
    const int id = r < a.k ? a.ids[t * a.k + r] : -1;
    e[r] = id >= a.E ? -1 : id;
    cnt[r] = 0;
  }
  for (int j0 = 64 * wave; j0 < a.n; j0 += 4 * 256) {
    int ej[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) ej[u] = j0 + 256 * u + lane < a.n ? a.ids[j0 + 256 * u + lane] : -1;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (j0 + 256 * u >= a.n) break;
      const int j = j0 + 256 * u + lane;
#pragma unroll
      for (int r = 0; r < kMaxRoutes; ++r)
        if (r < a.k) cnt[r] += __popcll(__ballot(ej[u] >= 0 && (ej[u] < e[r] || (ej[u] == e[r] && j < t * a.k + r))));
    }
  }
  if (lane == 0)
#pragma unroll
    for (int r = 0; r < kMaxRoutes; ++r) part[wave][r] = cnt[r];
  __syncthreads();
  if (tid < a.k) {
    const int id = a.ids[t * a.k + tid], a0 = t * a.k + tid;
    const int p = id < 0 || id >= a.E ? -1 : part[0][tid] + part[1][tid] + part[2][tid] + part[3][tid];
    pos[tid] = p;
    a.inv[a0] = p;
    if (p >= 0) a.order[p] = a0;
  }
  __syncthreads();
  scatter_row<U>(x + (size_t)t * rb, rows, rb, pos, a.k, tid, 256);
}

// Up to kTwoLaunches: one places them, one moves the rows.  Workgroup c takes chunk c and counts
// the assignments before and behind it itself (n reads from L2 a workgroup, no workspace).  Its
// 16 waves take 64 assignments each and rank the lanes of equal expert by ballots on the id's
// bits (stable, no order of atomics in the result).
__global__ __launch_bounds__(1024) void sort_place_all_kernel(SortArgs a) {
  // Counts in kCopies copies, 16 banks apart: lanes of one wave that count the same expert (a
  // popular one, of eight tokens) wait for each other (53,600 assignments 11.2 -> 10.4 us; more
  // loads in flight gain nothing).
  constexpr int kCopies = 4, kCopy = 256 + 16;
  __shared__ int before[kCopies * kCopy], total[kCopies * kCopy], slot[16][256];
  const int c = blockIdx.x, tid = threadIdx.x, wave = wave_id(), lane = tid & 63, copy = (lane >> 3) % kCopies * kCopy;
  for (int q = tid; q < kCopies * kCopy; q += 1024) before[q] = total[q] = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) slot[w * 4 + tid / 256][tid % 256] = 0;
  const int i = c * kDispatchChunk + tid, ev = i < a.n ? route_expert(a.ids[i], a.E, a.err) : -1;
  __syncthreads();
  constexpr int kAhead = 8;  // loads in flight
  for (int c0 = 0; c0 * kDispatchChunk < a.n; c0 += kAhead) {
    int id[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int j = (c0 + u) * kDispatchChunk + tid;
      id[u] = j < a.n ? a.ids[j] : -1;
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (id[u] >= 0 && id[u] < a.E) atomicAdd((c0 + u < c ? before : total) + copy + id[u], 1);
  }
  unsigned long long same = __ballot(ev >= 0);
#pragma unroll
  for (int b = 0; b < 8; ++b) {
    const unsigned long long bb = __ballot((ev >> b) & 1);
    same &= ((ev >> b) & 1) ? bb : ~bb;
  }
  if (ev < 0) same = 0ull;
  if (same && (same >> lane) == 1ull) slot[wave][ev] = __popcll(same);  // one writer per expert
  __syncthreads();
  if (tid < 64) {  // offsets: exclusive sums over the experts
    int run = 0;
#pragma unroll
    for (int e0 = 0; e0 < 256; e0 += 64) {
      const int e = e0 + tid;
      int ahead = 0, own = 0;
#pragma unroll
      for (int q = 0; q < kCopies; ++q) {
        ahead += before[q * kCopy + e];
        own += total[q * kCopy + e];
      }
      own += ahead;
      int incl = own;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int y = __shfl_up(incl, d, 64);
        if (tid >= d) incl += y;
      }
      const int first = run + incl - own;
      before[e] = ahead + first;  // the chunk's first position
      if (c == 0 && e < a.E) a.offsets[e] = first;
      run += __shfl(incl, 63, 64);
    }
    if (c == 0 && tid == 0) a.offsets[a.E] = run;
  }
  __syncthreads();
  if (tid < 256) {
    int run = before[tid];
#pragma unroll
    for (int w = 0; w < 16; ++w) {
      const int v = slot[w][tid];
      slot[w][tid] = run;
      run += v;
    }
  }
  __syncthreads();
  int pos = -1;
  if (same) pos = slot[wave][ev] + __popcll(same & ((1ull << lane) - 1ull));
  if (i < a.n) a.inv[i] = pos;
  if (pos >= 0) a.order[pos] = i;
}

// More assignments: chunks of kDispatchChunk are counted, the counts summed over the chunks
// before, and each chunk placed.  Chunk c's counts, then its sums, stay in its own part of
// inv (E <= 256 words of its 1,024), which only its workgroup overwrites, after reading
// them: calls share no memory but their own.  The last chunk, whose part may be shorter,
// keeps none: its base is what is left below the next expert's offset.
__global__ __launch_bounds__(256) void sort_count_kernel(SortArgs a) {
  __shared__ int hist[256];
  const int c = blockIdx.x, tid = threadIdx.x;
  hist[tid] = 0;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kDispatchChunk / 256; ++j) {
    const int i = c * kDispatchChunk + 256 * j + tid;
    const int e = i < a.n ? route_expert(a.ids[i], a.E, a.err) : -1;
    if (e >= 0) atomicAdd(&hist[e], 1);
  }
  __syncthreads();
  if (tid < a.E) a.inv[(size_t)c * kDispatchChunk + tid] = hist[tid];
}

// One workgroup: thread (s, e) sums expert e's counts over the s-th quarter of the chunks.
__global__ __launch_bounds__(1024) void sort_scan_kernel(SortArgs a, int nchunks) {
  __shared__ int quarter[4][256], last[256], base[256];
  const int tid = threadIdx.x, e = tid & 255, s = tid >> 8;
  const int full = nchunks - 1, c0 = full * s / 4, c1 = full * (s + 1) / 4;
  if (tid < 256) last[tid] = 0;
  __syncthreads();
  {
    const int i = full * kDispatchChunk + tid;
    const int ei = i < a.n ? route_expert(a.ids[i], a.E, a.err) : -1;
    if (ei >= 0) atomicAdd(&last[ei], 1);
  }
  int sum = 0;
  if (e < a.E) {
#pragma unroll 8
    for (int c = c0; c < c1; ++c) sum += a.inv[(size_t)c * kDispatchChunk + e];
  }
  quarter[s][e] = sum;
  __syncthreads();
  if (tid < 64) {  // offsets: exclusive sums over the experts
    int run = 0;
    for (int e0 = 0; e0 < 256; e0 += 64) {
      const int q = e0 + tid;
      const int own = quarter[0][q] + quarter[1][q] + quarter[2][q] + quarter[3][q] + last[q];
      int incl = own;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int y = __shfl_up(incl, d, 64);
        if (tid >= d) incl += y;
      }
      base[q] = run + incl - own;
      if (q < a.E) a.offsets[q] = base[q];
      run += __shfl(incl, 63, 64);
    }
    if (tid == 0) a.offsets[a.E] = run;
  }
  __syncthreads();
  if (e < a.E) {
    int run = base[e];
    for (int q = 0; q < s; ++q) run += quarter[q][e];
#pragma unroll 8
    for (int c = c0; c < c1; ++c) {
      int32_t* p = a.inv + (size_t)c * kDispatchChunk + e;
      const int v = *p;
      *p = run;
      run += v;
    }
  }
}

// Places chunk c: its four waves take 256 assignments each, 64 at a time in order, and rank
// the lanes of equal expert by ballots on the id's bits (stable, no atomics).
__global__ __launch_bounds__(256) void sort_place_kernel(SortArgs a, int nchunks) {
  __shared__ int slot[4][256];
  const int c = blockIdx.x, tid = threadIdx.x, wave = wave_id(), lane = tid & 63;
#pragma unroll
  for (int w = 0; w < 4; ++w) slot[w][tid] = 0;
  const int begin = c * kDispatchChunk + 256 * wave;
  int ev[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int i = begin + 64 * j + lane, id = i < a.n ? a.ids[i] : -1;
    ev[j] = id >= a.E ? -1 : id;
  }
  const bool is_last = c == nchunks - 1;
  int first = 0;
  if (tid < a.E) first = is_last ? a.offsets[tid + 1] : a.inv[(size_t)c * kDispatchChunk + tid];
  __syncthreads();
  unsigned long long same[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const bool ok = ev[j] >= 0;
    unsigned long long m = __ballot(ok);
#pragma unroll
    for (int b = 0; b < 8; ++b) {
      const unsigned long long bb = __ballot((ev[j] >> b) & 1);
      m &= ((ev[j] >> b) & 1) ? bb : ~bb;
    }
    same[j] = ok ? m : 0ull;
    if (ok && (m >> lane) == 1ull) slot[wave][ev[j]] += __popcll(m);  // one writer per expert and round
  }
  __syncthreads();
  if (tid < a.E) {
    int run = first;
    if (is_last)
#pragma unroll
      for (int w = 0; w < 4; ++w) run -= slot[w][tid];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const int v = slot[w][tid];
      slot[w][tid] = run;
      run += v;
    }
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int i = begin + 64 * j + lane;
    int pos = -1;
    if (same[j]) pos = slot[wave][ev[j]] + __popcll(same[j] & ((1ull << lane) - 1ull));
    if (i < a.n) a.inv[i] = pos;
    if (pos >= 0) a.order[pos] = i;
    __builtin_amdgcn_wave_barrier();  // every lane has read its slot before the last of its expert moves it
    if (same[j] && (same[j] >> lane) == 1ull) slot[wave][ev[j]] += __popcll(same[j]);
    __builtin_amdgcn_wave_barrier();
  }
}

template <typename U>
__global__ __launch_bounds__(256) void sort_rows_kernel(const int32_t* __restrict__ inv, int t0, int k,
                                                        const uint8_t* __restrict__ x, uint8_t* __restrict__ rows,
                                                        size_t rb) {
  __shared__ int pos[kMaxRoutes];
  const size_t t = (size_t)t0 + blockIdx.x;
  if ((int)threadIdx.x < k) pos[threadIdx.x] = inv[t * k + threadIdx.x];
  __syncthreads();
  scatter_row<U>(x + t * rb, rows, rb, pos, k, threadIdx.x, blockDim.x);
}

// ------------------------------------------------------------ sums over routes --
// Lane r of a wave holds token t's route r: its sorted row (-1: none) and weight, and the
// rank of that row among the token's.
struct Routes {
  int pos;
  float w;
  int rank, live;
};
__device__ __forceinline__ Routes load_routes(const int32_t* __restrict__ inv, const float* __restrict__ wts, size_t t,
                                              int k, int n, int* err) {
  const int lane = threadIdx.x & 63;
  Routes q{-1, 1.f, 0, 0};
  if (lane < k) {
    q.pos = inv[t * k + lane];
    if (wts) q.w = wts[t * k + lane];
    if (q.pos >= n) {
      atomicOr(err, kErrPosition);
      q.pos = -1;
    }
  }
  for (int r = 0; r < k; ++r) {
    const int p = __builtin_amdgcn_readlane(q.pos, r);
    if (p >= 0) {
      ++q.live;
      q.rank += (p < q.pos) || (p == q.pos && r < lane);
    }
  }
  if (q.pos < 0) q.rank = -1;
  return q;
}

struct SumArgs {
  const void* rows;
  const int32_t* inv;
  const float* wts;  // null: ones
  void* out;
  int t0, T, H, k, n, nslab;
  int* err;
};

// out[t] = sum over the token's rows in ascending position; one wave per (token, slab of 64 N
// columns), up to kMaxRoutes / 2 row loads in flight.
template <int DT, int N, bool kWeighted, bool kOnce>
__global__ __launch_bounds__(256) void sum_rows_kernel(SumArgs a) {
  typedef typename Elem<DT>::T E;
  const size_t id = (size_t)blockIdx.x * 4 + wave_id();
  const size_t tl = id / a.nslab;
  if (tl >= (size_t)a.T) return;
  const size_t t = (size_t)a.t0 + tl;
  const int c = ((int)(id % a.nslab) * 64 + (int)(threadIdx.x & 63)) * N;
  const Routes q = load_routes(a.inv, a.wts, t, a.k, a.n, a.err);
  const bool in = c < a.H;
  float acc[N];
#pragma unroll
  for (int i = 0; i < N; ++i) acc[i] = 0.f;
  constexpr int kBatch = kMaxRoutes / 2;
  for (int s0 = 0; s0 < q.live; s0 += kBatch) {
    Pack<DT, N> v[kBatch];
    float w[kBatch];
#pragma unroll
    for (int s = 0; s < kBatch; ++s) {
      if (s0 + s < q.live) {
        const int r = __ffsll((unsigned long long)__ballot(q.rank == s0 + s)) - 1;
        const int p = __builtin_amdgcn_readlane(q.pos, r);
        w[s] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(q.w), r));
        if (in) v[s] = load_pack<DT, N, kOnce>(static_cast<const E*>(a.rows) + (size_t)p * a.H + c);
      }
    }
#pragma unroll
    for (int s = 0; s < kBatch; ++s) {
      if (s0 + s < q.live && in) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float f = Elem<DT>::get(v[s].v[i]);
          acc[i] = __fadd_rn(acc[i], kWeighted ? __fmul_rn(f, w[s]) : f);
        }
      }
    }
  }
  if (in) {
    Pack<DT, N> o;
#pragma unroll
    for (int i = 0; i < N; ++i) o.v[i] = Elem<DT>::put(acc[i]);
    store_pack<DT, N>(static_cast<E*>(a.out) + t * a.H + c, o);
  }
}

// ----------------------------------------------------------- combine's gradient --
struct CombineGradArgs {
  const void *dout, *rows;
  const int32_t* inv;
  const float* wts;
  void* drows;
  float* dwts;
  int t0, H, k, n;
  int* err;
};

// One workgroup per token: every thread keeps a column piece of dout, writes the k products
// and adds its share of the k dot products, which meet in LDS in wave order.
template <int DT, int N>
__global__ __launch_bounds__(256) void combine_grad_kernel(CombineGradArgs a) {
  typedef typename Elem<DT>::T E;
  __shared__ float part[4][kMaxRoutes];
  const size_t t = (size_t)a.t0 + blockIdx.x;
  const int lane = threadIdx.x & 63, wave = wave_id(), nw = blockDim.x >> 6;
  int pos = -1;
  float wt = 0.f;
  if (lane < a.k) {
    pos = a.inv[t * a.k + lane];
    wt = a.wts[t * a.k + lane];
    if (pos >= a.n) {
      atomicOr(a.err, kErrPosition);
      pos = -1;
    }
  }
  float dot[kMaxRoutes];
#pragma unroll
  for (int r = 0; r < kMaxRoutes; ++r) dot[r] = 0.f;
  for (int c = (int)threadIdx.x * N; c < a.H; c += (int)blockDim.x * N) {
    const Pack<DT, N> d = load_pack<DT, N>(static_cast<const E*>(a.dout) + t * a.H + c);
    float df[N];
#pragma unroll
    for (int i = 0; i < N; ++i) df[i] = Elem<DT>::get(d.v[i]);
#pragma unroll
    for (int r = 0; r < kMaxRoutes; ++r) {
      const int p = __builtin_amdgcn_readlane(pos, r);
      if (r >= a.k || p < 0) continue;
      const float w = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(wt), r));
      const Pack<DT, N> v = load_pack<DT, N>(static_cast<const E*>(a.rows) + (size_t)p * a.H + c);
      Pack<DT, N> o;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        float p = __fmul_rn(w, df[i]);
        // The product is rounded to fp32 first, at every address and column: the compiler makes one
        // instruction with a single rounding of some products with their conversion to fp16.
        if constexpr (DT == RMOE_DT_F16) asm("" : "+v"(p));
        o.v[i] = Elem<DT>::put(p);
        dot[r] = fmaf(df[i], Elem<DT>::get(v.v[i]), dot[r]);
      }
      store_pack<DT, N>(static_cast<E*>(a.drows) + (size_t)p * a.H + c, o);
    }
  }
#pragma unroll
  for (int r = 0; r < kMaxRoutes; ++r) {
    if (r >= a.k) break;
    const float s = wave_sum(dot[r]);
    if (lane == 0) part[wave][r] = s;
  }
  __syncthreads();
  if ((int)threadIdx.x < a.k) {
    float s = part[0][threadIdx.x];
    for (int w = 1; w < nw; ++w) s += part[w][threadIdx.x];
    a.dwts[t * a.k + threadIdx.x] = pos >= 0 ? s : 0.f;
  }
}

bool aligned(size_t to, std::initializer_list<const void*> ps, size_t row_bytes) {
  for (const void* p : ps)
    if (reinterpret_cast<uintptr_t>(p) % to) return false;
  return row_bytes % to == 0;
}

size_t dtype_bytes(int dt) { return dt == RMOE_DT_F32 ? 4 : 2; }

// Fewer than 2^32 threads in a launch.
constexpr size_t kMaxGroups = ((size_t)1 << 32) / 256 - 1;

template <typename U>
hipError_t sort_with(const SortArgs& a, const void* x, void* rows, size_t rb, hipStream_t st) {
  if (a.n <= kOneLaunch) {
    hipLaunchKernelGGL(sort_small_kernel<U>, dim3(a.T + 1), dim3(256), 0, st, a, (const uint8_t*)x, (uint8_t*)rows, rb);
    return hipGetLastError();
  }
  const int nchunks = (int)(((size_t)a.n + kDispatchChunk - 1) / kDispatchChunk);
  if (a.n <= kTwoLaunches) {
    hipLaunchKernelGGL(sort_place_all_kernel, dim3(nchunks), dim3(1024), 0, st, a);
  } else {
    hipLaunchKernelGGL(sort_count_kernel, dim3(nchunks - 1), dim3(256), 0, st, a);
    hipLaunchKernelGGL(sort_scan_kernel, dim3(1), dim3(1024), 0, st, a, nchunks);
    hipLaunchKernelGGL(sort_place_kernel, dim3(nchunks), dim3(256), 0, st, a, nchunks);
  }
  hipError_t e = hipGetLastError();
  const int threads = (int)std::min<size_t>(256, (rb / sizeof(U) + 63) / 64 * 64);
  for (size_t t0 = 0; e == hipSuccess && t0 < (size_t)a.T; t0 += kMaxGroups) {
    hipLaunchKernelGGL(sort_rows_kernel<U>, dim3((unsigned)std::min(kMaxGroups, (size_t)a.T - t0)), dim3(threads), 0, st,
                       a.inv, (int)t0, a.k, (const uint8_t*)x, (uint8_t*)rows, rb);
    e = hipGetLastError();
  }
  return e;
}

template <int DT, int N>
hipError_t sum_with(SumArgs a, hipStream_t st) {
  a.nslab = (a.H + 64 * N - 1) / (64 * N);
  const int total = a.T;
  // Sorted rows of kOnceBytes and more are summed with non-temporal loads: they are read once
  // and do not fit the caches anyway (6,700 tokens alone, other buffers each time: 58 -> 49 us; the
  // combine's gradient gains nothing).  H 2,048, k 8, sort and combine in turn (the same buffers /
  // others each time): 220 MB of rows 92 / 100 us without the hint, 89 / 93 with it; 67 MB 35 / 36 and
  // 36 / 33; 34 MB 20 / 22 and 23 / 22.  (Storing them so makes the sort alone 60 -> 54 us and the two
  // 100 -> 113: what comes next finds less of them in the cache.)
  const bool once = (size_t)a.n * a.H * dtype_bytes(DT) >= kOnceBytes;
  const size_t step = std::max<size_t>(1, kMaxGroups * 4 / a.nslab);
  for (size_t t0 = 0; t0 < (size_t)total; t0 += step) {
    a.t0 = (int)t0;
    a.T = (int)std::min(step, (size_t)total - t0);
    const dim3 grid((unsigned)(((size_t)a.T * a.nslab + 3) / 4)), block(256);
    auto* kernel = once ? (a.wts ? sum_rows_kernel<DT, N, true, N != 1> : sum_rows_kernel<DT, N, false, N != 1>)
                        : (a.wts ? sum_rows_kernel<DT, N, true, false> : sum_rows_kernel<DT, N, false, false>);
    hipLaunchKernelGGL(kernel, grid, block, 0, st, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

template <int DT, int N>
hipError_t grad_with(CombineGradArgs a, int T, hipStream_t st) {
  const int threads = std::min(256, ((a.H + N - 1) / N + 63) / 64 * 64);
  for (size_t t0 = 0; t0 < (size_t)T; t0 += kMaxGroups) {
    a.t0 = (int)t0;
    hipLaunchKernelGGL((combine_grad_kernel<DT, N>), dim3((unsigned)std::min(kMaxGroups, (size_t)T - t0)), dim3(threads),
                       0, st, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace

hipError_t launch_sort_tokens(const void* x, int dtype, int T, int H, const int32_t* ids, int k, int n_experts,
                              void* rows, int32_t* order, int32_t* inv, int32_t* offsets, int* err, hipStream_t st) {
  const SortArgs a{ids, T, k, n_experts, T * k, order, inv, offsets, err};
  const size_t rb = (size_t)H * dtype_bytes(dtype);
  if (aligned(16, {x, rows}, rb)) return sort_with<uint4>(a, x, rows, rb, st);
  if (aligned(4, {x, rows}, rb)) return sort_with<uint32_t>(a, x, rows, rb, st);
  return sort_with<uint16_t>(a, x, rows, rb, st);
}

hipError_t launch_sum_rows(const void* rows, int dtype, int T, int H, const int32_t* inv, const float* wts, int k,
                           void* out, int* err, hipStream_t st) {
  const SumArgs a{rows, inv, wts, out, 0, T, H, k, T * k, 0, err};
  const bool wide = aligned(16, {rows, out}, (size_t)H * dtype_bytes(dtype));
  if (dtype == RMOE_DT_BF16) return wide ? sum_with<RMOE_DT_BF16, 8>(a, st) : sum_with<RMOE_DT_BF16, 1>(a, st);
  if (dtype == RMOE_DT_F16) return wide ? sum_with<RMOE_DT_F16, 8>(a, st) : sum_with<RMOE_DT_F16, 1>(a, st);
  return wide ? sum_with<RMOE_DT_F32, 4>(a, st) : sum_with<RMOE_DT_F32, 1>(a, st);
}

hipError_t launch_combine_grad(const void* dout, const void* rows, int dtype, int T, int H, const int32_t* inv,
                               const float* wts, int k, void* drows, float* dwts, int* err, hipStream_t st) {
  const CombineGradArgs a{dout, rows, inv, wts, drows, dwts, 0, H, k, T * k, err};
  const bool wide = aligned(16, {dout, rows, drows}, (size_t)H * dtype_bytes(dtype));
  if (dtype == RMOE_DT_BF16) return wide ? grad_with<RMOE_DT_BF16, 8>(a, T, st) : grad_with<RMOE_DT_BF16, 1>(a, T, st);
  if (dtype == RMOE_DT_F16) return wide ? grad_with<RMOE_DT_F16, 8>(a, T, st) : grad_with<RMOE_DT_F16, 1>(a, T, st);
  return wide ? grad_with<RMOE_DT_F32, 4>(a, T, st) : grad_with<RMOE_DT_F32, 1>(a, T, st);
}

}  // namespace rmoe
