// The next token from a row of logits: temperature, top-k, top-p, min-p, and a draw with a given random number.
//
//   w = 2^((l - m) c), m the largest logit, c = log2(e) / temperature; 1 where l == m;   then (w + 2^-12) - 2^-12 in fp32
//
// The last step makes every weight a multiple of 2^-35 (w is at most 1), so sums of up to 2^18 of them are exact in fp64: they
// come out the same in any order and over any split of the row, and so do the token and every cut through the distribution;
// atomics may add them up.  Weights below 2^-36 become zero; such tokens are never drawn.
//
// Tokens are ranked by falling logit, the lower index first among equals.  Every filter but min-p keeps a beginning of that order,
// which its last token (logit, index) describes; min-p is a bound on the weight itself.  The draw walks the kept tokens by index,
// which needs no sort of the row: a sum per cell of the row (16 vectors of 16 bytes), then the cell that the drawn weight falls into.
//
// Up to four launches, the two in the middle only where a row may need them, the last one alone for rows of up to 1024 logits:
//   sample_cells_kernel  the row split over workgroups: the largest logit of each cell.  It reads everything, once, and is bound by HBM.
//   sample_mass_kernel   rows without top-k: the weight of each cell (no filter at all), or of each of 2048 stretches of the logit's
//                        range (top-p): the row again, from the caches unless the batch is larger than they are.
//   sample_walk_kernel   top-p without top-k: the stretch that the cut lies in is known now; the weight of what ranks before it, cell by
//                        cell, and a list of its tokens.
//   sample_pick_kernel   a workgroup per row.  A short list of tokens decides: with top-k, those not below the k-th largest of the
//                        cells' largest logits (at least k tokens are not), found in the few cells that hold any; with top-p, the list
//                        above; with min-p, those that have the weight.  It is ranked, cut, and drawn from.  Where it would not fit
//                        (more than 1024 tokens in a stretch, top-k above 960), the cut is found digit by digit over an order-preserving
//                        integer key of the logits, in six or more passes of one workgroup over its row: 0.3 to 0.9 ms.
//
// Measured, rows of 128256 fp32 logits: one row with top-k 50 and top-p 0.95 11.9 us (3.1 + 8.9, the second a chain of some forty
// dependent LDS and memory accesses), with top-p alone 27 us (3.0 + 5.9 + 7.2 + 11.3); 256 rows with top-k 37 us (25 us of it the
// first launch, 5.3 TB/s), with top-p alone 114 us (the histogram's LDS atomics 40, the walk 36), with settings of their own 76 us.  One row and
// 256, us: greedy 6.8, 32; min-p 0.05 alone 9.5, 34; no filter 15, 59; by digits: top-k 1000 or 5000 301, 362, with top-p behind it 426, 520,
// top-p over equal logits 895, 1138.
#pragma once
#include <float.h>

#include <algorithm>

#include "common.hpp"

namespace tp {

constexpr float SAMPLE_LOG2E = 1.4426950408889634f;
constexpr int SAMPLE_THREADS = 1024, SAMPLE_WAVES = SAMPLE_THREADS / WAVE;
constexpr int SAMPLE_MOST = 1 << 18;  // logits per row
constexpr int SAMPLE_CELL = 16;       // vectors of 16 bytes, one per lane of a group of 16
constexpr int SAMPLE_CELLS = SAMPLE_MOST / 4 / SAMPLE_CELL + 3;
constexpr int SAMPLE_SPLIT = 256;     // threads of a workgroup that takes a part of a row
constexpr int SAMPLE_FIRST = 2;       // vectors per thread of the first launch
constexpr int SAMPLE_PARTS = SAMPLE_CELLS * SAMPLE_CELL / (SAMPLE_SPLIT * SAMPLE_FIRST) + 1;
constexpr int SAMPLE_LIST = 1024;     // tokens that are sorted at most
constexpr int SAMPLE_COUNTED = 128;   // tokens that are compared with each other at most; more are sorted
constexpr int SAMPLE_TOP_K = 960;     // the largest top-k that goes by the list
constexpr int SAMPLE_BINS = 2048;     // over weights from 1 down to 2^-36
constexpr float SAMPLE_BIN = SAMPLE_BINS / 36.5f;

struct SampleArgs {
  const void* logits;
  const float *uniform, *temperatures, *top_ps, *min_ps;
  const int32_t* top_ks;
  float temperature, top_p, min_p;
  int top_k;
  int64_t* tokens;
  float* logprobs;
  char* ws;
  int64_t row_stride;
  int V;
  int cells;  // of any row, at most
  // per row: what sample_walk_kernel found, its list, the bins, the cells' weights, the largest logits of the first launch's workgroups
  // and of the cells
  struct Walk {
    double before, goal;
    int count;
  };
  static constexpr int64_t ws_row(int cells) { return (sizeof(Walk) + SAMPLE_LIST * 8 + SAMPLE_BINS * 8 + SAMPLE_PARTS * 4 + (int64_t)cells * 12 + 15) / 16 * 16; }
  __device__ __forceinline__ Walk* walk(int r) const { return reinterpret_cast<Walk*>(ws + r * ws_row(cells)); }
  __device__ __forceinline__ uint64_t* list(int r) const { return reinterpret_cast<uint64_t*>(walk(r) + 1); }
  __device__ __forceinline__ double* bins(int r) const { return reinterpret_cast<double*>(list(r) + SAMPLE_LIST); }
  __device__ __forceinline__ double* masses(int r) const { return bins(r) + SAMPLE_BINS; }
  __device__ __forceinline__ float* parts(int r) const { return reinterpret_cast<float*>(masses(r) + cells); }
  __device__ __forceinline__ float* maxima(int r) const { return parts(r) + SAMPLE_PARTS; }
};
inline int sample_cells(int V) { return (V / 4 + SAMPLE_CELL - 1) / SAMPLE_CELL + 2; }  // at most, for any type and address

// larger logit, larger key; -0 and +0 have the same
__device__ __forceinline__ unsigned sample_key(float l) {
  const unsigned u = __float_as_uint(l + 0.f);
  return u ^ ((unsigned)((int)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float sample_logit(unsigned key) {
  return __uint_as_float(key ^ (key & 0x80000000u ? 0x80000000u : 0xffffffffu));
}

// what a row's weights depend on
struct Weights {
  float m, c;
  __device__ __forceinline__ Weights(float largest, float temperature) : m(largest), c(fmaxf(SAMPLE_LOG2E / temperature, FLT_MIN)) {}  // (c = 0 would not keep -inf out)
  __device__ __forceinline__ float power(float l) const { return l == m ? 0.f : (l - m) * c; }
  __device__ __forceinline__ float of_power(float x) const { return (__builtin_amdgcn_exp2f(x) + 0x1p-12f) - 0x1p-12f; }
  __device__ __forceinline__ float operator()(float l) const { return of_power(power(l)); }
  // falls as the logit rises; beyond the last bin nothing has a weight
  __device__ __forceinline__ static int bin(float x) { return (int)fminf(-x * SAMPLE_BIN, (float)SAMPLE_BINS); }
};

enum SampleKind { GREEDY, LIST, TOP_K, TOP_P, MIN_P, ALL, DIGITS };
struct Settings {
  float temperature, top_p, min_p;
  int top_k;  // 0: all
  SampleKind kind;
  __device__ __forceinline__ Settings(const SampleArgs& a, int row) {
    temperature = a.temperatures ? a.temperatures[row] : a.temperature;
    top_k = a.top_ks ? a.top_ks[row] : a.top_k;
    top_p = fminf(fmaxf(a.top_ps ? a.top_ps[row] : a.top_p, 0.f), 1.f);
    min_p = fminf(fmaxf(a.min_ps ? a.min_ps[row] : a.min_p, 0.f), 1.f);
    if (top_k <= 0 || top_k >= a.V) top_k = 0;
    if (!(temperature > 0.f) || top_k == 1 || top_p <= 0.f) kind = GREEDY;
    else if (a.V <= SAMPLE_LIST) kind = LIST;
    else if (top_k) kind = top_k <= SAMPLE_TOP_K ? TOP_K : DIGITS;
    else if (top_p < 1.f) kind = TOP_P;
    else kind = min_p > 0.f ? MIN_P : ALL;
  }
};

// The logits of a row in vectors of 16 bytes at 16-byte addresses, and one cell each for the few elements before the first and
// behind the last of them, one element a vector.  What is not there, and NaN, is -inf.
template <typename T>
struct Row {
  static constexpr int E = 16 / sizeof(T);
  const T* p;
  int head, full, padded;  // elements before the vectors; vectors; vectors up to a whole cell
  int V;
  __device__ __forceinline__ Row(const SampleArgs& a, int row) : p(reinterpret_cast<const T*>(a.logits) + row * a.row_stride), V(a.V) {
    head = min(V, (int)((16 - ((size_t)p & 15)) % 16 / sizeof(T)));
    full = (V - head) / E;
    padded = (full + SAMPLE_CELL - 1) / SAMPLE_CELL * SAMPLE_CELL;
  }
  __device__ __forceinline__ int vectors() const { return padded + 2 * SAMPLE_CELL; }
  __device__ __forceinline__ int cells() const { return padded / SAMPLE_CELL + 2; }
  // of an element that is there
  __device__ __forceinline__ int index(int vec, int e) const {
    const int v = vec - SAMPLE_CELL;
    return v < 0 ? vec : v < padded ? head + v * E + e : head + full * E + (v - padded);
  }
  __device__ __forceinline__ int cell_of(int i) const {
    return i < head ? 0 : i < head + full * E ? 1 + (i - head) / (E * SAMPLE_CELL) : 1 + padded / SAMPLE_CELL;
  }
  __device__ __forceinline__ void load(int vec, float (&x)[E]) const {
    const int v = vec - SAMPLE_CELL;
    if ((unsigned)v < (unsigned)full) {
      load_f<T, E>(p + head + (int64_t)v * E, x);
#pragma unroll
      for (int e = 0; e < E; e++) x[e] = x[e] == x[e] ? x[e] : -INFINITY;
    } else {
      const int i = index(vec, 0);
      const bool there = v < 0 ? vec < head : v >= padded && i < V;
#pragma unroll
      for (int e = 1; e < E; e++) x[e] = -INFINITY;
      const float y = there ? Elem<T>::to_f(p[i]) : -INFINITY;
      x[0] = y == y ? y : -INFINITY;
    }
  }
};

__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
// over the 16 lanes of a cell, in the vector units (an exchange through LDS for every vector took as long as its arithmetic)
template <int N> __device__ __forceinline__ int rotate16(int v) { return __builtin_amdgcn_update_dpp(0, v, 0x120 + N, 0xf, 0xf, false); }
template <int N> __device__ __forceinline__ double rotated_sum(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint64_t r = (uint64_t)(unsigned)rotate16<N>((int)(u >> 32)) << 32 | (unsigned)rotate16<N>((int)u);
  return v + __builtin_bit_cast(double, r);
}
template <int N> __device__ __forceinline__ float rotated_max(float v) { return fmaxf(v, __int_as_float(rotate16<N>(__float_as_int(v)))); }
__device__ __forceinline__ double cell_sum(double v) { return rotated_sum<1>(rotated_sum<2>(rotated_sum<4>(rotated_sum<8>(v)))); }
__device__ __forceinline__ float cell_max(float v) { return rotated_max<1>(rotated_max<2>(rotated_max<4>(rotated_max<8>(v)))); }

// ------------------------------------------------------------------------------------------------
constexpr int SAMPLE_SHARES = 2048;  // workgroups of the second and third launch
template <typename T>
__global__ __launch_bounds__(SAMPLE_SPLIT) void sample_cells_kernel(SampleArgs a) {
  constexpr int E = Row<T>::E, U = SAMPLE_FIRST;
  __shared__ float wm[SAMPLE_SPLIT / WAVE];
  const int row = blockIdx.y;
  const Row<T> x(a, row);
  const int nv = x.vectors(), v0 = blockIdx.x * (SAMPLE_SPLIT * U) + threadIdx.x;
  float l[U][E];
#pragma unroll
  for (int u = 0; u < U; u++)
    if (v0 + u * SAMPLE_SPLIT < nv) x.load(v0 + u * SAMPLE_SPLIT, l[u]);
  float* out = a.maxima(row);
  float all = -INFINITY;
#pragma unroll
  for (int u = 0; u < U; u++) {
    const int v = v0 + u * SAMPLE_SPLIT;
    float m = -INFINITY;
    if (v < nv) {
#pragma unroll
      for (int e = 0; e < E; e++) m = fmaxf(m, l[u][e]);
    }
    m = cell_max(m);
    if (threadIdx.x % SAMPLE_CELL == 0 && v < nv) out[v / SAMPLE_CELL] = m;
    all = fmaxf(all, m);
  }
  all = wave_max(all);
  if (threadIdx.x % WAVE == 0) wm[threadIdx.x / WAVE] = all;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < SAMPLE_SPLIT / WAVE; i++) all = fmaxf(all, wm[i]);
    a.parts(row)[blockIdx.x] = all;
  }
  // cleared for the next kernel to add to
  for (int i = blockIdx.x * SAMPLE_SPLIT + threadIdx.x; i < SAMPLE_BINS; i += gridDim.x * SAMPLE_SPLIT) a.bins(row)[i] = 0;
  if (blockIdx.x == 0 && threadIdx.x == 0) a.walk(row)->count = 0;
}

// f(vector, its logits) of every SAMPLE_SPLIT-th vector from v on, the loads four at a time
template <typename T, typename F>
__device__ __forceinline__ void each_vector(const Row<T>& x, int v, int end, F&& f) {
  constexpr int E = Row<T>::E, U = 4;
  for (; v < end; v += U * SAMPLE_SPLIT) {
    float l[U][E];
#pragma unroll
    for (int u = 0; u < U; u++)
      if (v + u * SAMPLE_SPLIT < end) x.load(v + u * SAMPLE_SPLIT, l[u]);
#pragma unroll
    for (int u = 0; u < U; u++)
      if (v + u * SAMPLE_SPLIT < end) f(v + u * SAMPLE_SPLIT, l[u]);
  }
}

// the row's largest logit, by every wave
__device__ __forceinline__ float row_max(const SampleArgs& a, int row, int parts) {
  const float* p = a.parts(row);
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < SAMPLE_PARTS; i += WAVE) m = fmaxf(m, i + (int)(threadIdx.x % WAVE) < parts ? p[i + threadIdx.x % WAVE] : -INFINITY);
  return wave_max(m);
}

template <typename T>
__global__ __launch_bounds__(SAMPLE_SPLIT) void sample_mass_kernel(SampleArgs a, int share, int parts) {
  constexpr int E = Row<T>::E;
  __shared__ double bins[SAMPLE_BINS];
  const int row = blockIdx.y, tid = threadIdx.x;
  const Row<T> x(a, row);
  const int v0 = blockIdx.x * share, v1 = min(v0 + share, x.vectors());
  const Settings s(a, row);
  if (s.kind != TOP_P && s.kind != ALL) return;
  if (s.kind == TOP_P)
    for (int i = tid; i < SAMPLE_BINS; i += SAMPLE_SPLIT) bins[i] = 0.;
  const Weights weight(row_max(a, row, parts), s.temperature);
  __syncthreads();
  each_vector(x, v0 + tid, v1, [&](int v, const float (&l)[E]) {  // (whole cells: shares and vectors() are multiples of 16)
    double sum = 0.;
#pragma unroll
    for (int e = 0; e < E; e++) {
      const float p = weight.power(l[e]), w = weight.of_power(p);
      if (s.kind == ALL) sum += (double)w;
      else if (w > 0.f) atomicAdd(&bins[Weights::bin(p)], (double)w);
    }
    if (s.kind == ALL) {
      sum = cell_sum(sum);
      if (tid % SAMPLE_CELL == 0) a.masses(row)[v / SAMPLE_CELL] = sum;
    }
  });
  if (s.kind == ALL) return;
  __syncthreads();
  double* out = a.bins(row);
  for (int i = tid; i < SAMPLE_BINS; i += SAMPLE_SPLIT)
    if (bins[i] > 0.) __hip_atomic_fetch_add(&out[i], bins[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// larger logits, and lower indices among equals, first
__device__ __forceinline__ uint64_t sample_rank(float l, int i) { return (uint64_t)~sample_key(l) << 32 | (unsigned)i; }

template <typename T>
__global__ __launch_bounds__(SAMPLE_SPLIT) void sample_walk_kernel(SampleArgs a, int share, int parts) {
  constexpr int E = Row<T>::E, WAVES = SAMPLE_SPLIT / WAVE, PER = SAMPLE_BINS / SAMPLE_SPLIT;
  __shared__ double wd[WAVES], found;
  __shared__ uint64_t list[SAMPLE_LIST];
  __shared__ int found_bin, count, begin_at;
  const int row = blockIdx.y, tid = threadIdx.x, lane = tid % WAVE, wave = tid / WAVE;
  const Row<T> x(a, row);
  const int v0 = blockIdx.x * share, v1 = min(v0 + share, x.vectors());
  const Settings s(a, row);
  if (s.kind != TOP_P) return;
  const Weights weight(row_max(a, row, parts), s.temperature);
  // the stretch of weights that the cut lies in
  double w[PER], sum = 0.;
#pragma unroll
  for (int i = 0; i < PER; i++) sum += w[i] = a.bins(row)[tid * PER + i];
  double upto = sum;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double y = __shfl_up(upto, o, 64);
    if (lane >= o) upto += y;
  }
  if (tid == 0) count = 0;
  if (lane == WAVE - 1) wd[wave] = upto;
  __syncthreads();
  double all = 0.;
  for (int i = 0; i < WAVES; i++) {
    upto += i < wave ? wd[i] : 0.;
    all += wd[i];
  }
  const double goal = (double)s.top_p * all;
  if (upto >= goal && upto - sum < goal) {  // (one thread: the sums are exact, and goal is above 0)
    double begin = upto - sum;
    int b = tid * PER;
#pragma unroll
    for (int i = 0; i < PER - 1; i++)
      if (b == tid * PER + i && begin + w[i] < goal) {
        begin += w[i];
        b++;
      }
    found_bin = b;
    found = begin;
  }
  __syncthreads();
  const int b = found_bin;
  SampleArgs::Walk* out = a.walk(row);
  if (blockIdx.x == 0 && tid == 0) {
    out->before = found;
    out->goal = goal;
  }
  each_vector(x, v0 + tid, v1, [&](int v, const float (&l)[E]) {
    double cell = 0.;
#pragma unroll
    for (int e = 0; e < E; e++) {
      const float p = weight.power(l[e]);
      const int bin = Weights::bin(p);
      if (bin > b) continue;
      const float y = weight.of_power(p);
      if (bin < b) {
        cell += y >= s.min_p ? (double)y : 0.;
      } else if (y > 0.f) {
        const int at = atomicAdd(&count, 1);
        if (at < SAMPLE_LIST) list[at] = sample_rank(l[e], x.index(v, e));
      }
    }
    cell = cell_sum(cell);
    if (tid % SAMPLE_CELL == 0) a.masses(row)[v / SAMPLE_CELL] = cell;
  });
  // the workgroups' lists one behind the other, in the order that they come (the row's list is sorted later); beyond the list's end
  // only the count goes on
  __syncthreads();
  if (tid == 0 && count) begin_at = __hip_atomic_fetch_add(&out->count, count, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  for (int i = tid; i < min(count, SAMPLE_LIST); i += SAMPLE_SPLIT)
    if (begin_at + i < SAMPLE_LIST) a.list(row)[begin_at + i] = list[i];
}

// ------------------------------------------------------------------------------------------------
struct PickLds {
  double mass[SAMPLE_CELLS];
  float maxima[SAMPLE_CELLS];
  unsigned short chosen[SAMPLE_CELLS];
  uint64_t list[SAMPLE_LIST];
  double weight[SAMPLE_COUNTED], sums[2][SAMPLE_COUNTED];
  int ranks[SAMPLE_COUNTED];
  double wd[SAMPLE_WAVES];
  float most[SAMPLE_WAVES], least[SAMPLE_WAVES];
  int wi[SAMPLE_WAVES];
  int count, cells, at;
  double begin;
  uint64_t last;
};

// the sum of v over the threads before this one and itself; `all` over all.  For the whole workgroup.
__device__ __forceinline__ double group_scan(double v, PickLds& s, double& all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double y = __shfl_up(v, o, 64);
    if (lane >= o) v += y;
  }
  if (lane == 63) s.wd[wave] = v;
  __syncthreads();
  double before = 0.;
  all = 0.;
#pragma unroll
  for (int i = 0; i < SAMPLE_WAVES; i++) {
    before += i < wave ? s.wd[i] : 0.;
    all += s.wd[i];
  }
  __syncthreads();
  return before + v;
}

// the value of lane ^ J
template <int J> __device__ __forceinline__ uint64_t lane_xor(uint64_t v) {
  constexpr int CTRL = J == 1 ? 0xb1 : J == 2 ? 0x4e : J == 8 ? 0x128 : -1;  // quads' permutations, a row's half rotation
  if constexpr (CTRL >= 0)
    return (uint64_t)(unsigned)__builtin_amdgcn_update_dpp(0, (int)(v >> 32), CTRL, 0xf, 0xf, false) << 32 |
           (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, false);
  else
    return __shfl_xor((unsigned long long)v, J, 64);
}
template <int J> __device__ __forceinline__ void sort_within(uint64_t& x, int tid, int k) {
  if constexpr (J > 0) {
    const uint64_t y = lane_xor<J>(x);
    x = (((tid & J) == 0) == ((tid & k) == 0)) == (x < y) ? x : y;
    sort_within<J / 2>(x, tid, k);
  }
}
template <int K> __device__ __forceinline__ void sort_wave(uint64_t& x, int tid) {
  if constexpr (K > 1) {
    sort_wave<K / 2>(x, tid);
    sort_within<K / 2>(x, tid, K);
  }
}
// list[0, n) in rising order, bitonic, an element a thread; only distances from a wave up go through LDS
__device__ __forceinline__ void sort_list(PickLds& s, int n) {
  const int tid = threadIdx.x;
  int size = WAVE;
  while (size < n) size *= 2;
  uint64_t x = tid < n ? s.list[tid] : ~0ull;
  if (tid < size) sort_wave<WAVE>(x, tid);
  for (int k = 2 * WAVE; k <= size; k *= 2) {
    for (int j = k / 2; j >= WAVE; j /= 2) {
      __syncthreads();
      if (tid < size) s.list[tid] = x;
      __syncthreads();
      if (tid < size) {
        const uint64_t y = s.list[tid ^ j];
        x = (((tid & j) == 0) == ((tid & k) == 0)) == (x < y) ? x : y;
      }
    }
    if (tid < size) sort_within<WAVE / 2>(x, tid, k);
  }
  __syncthreads();
  if (tid < size) s.list[tid] = x;
  __syncthreads();
}

template <typename T>
struct Picker {
  static constexpr int E = Row<T>::E;
  const SampleArgs& a;
  PickLds& s;
  const int row, tid, lane, wave;
  const Row<T> x;
  const int nv, cells;
  const Settings set;
  float m, least, scale;  // of the cells' maxima, the largest and the smallest that is not -inf

  __device__ __forceinline__ Picker(const SampleArgs& args, PickLds& lds)
      : a(args), s(lds), row(blockIdx.x), tid(threadIdx.x), lane(tid & 63), wave(tid >> 6), x(args, blockIdx.x), nv(x.vectors()), cells(x.cells()),
        set(args, blockIdx.x) {
    m = -INFINITY;
    least = INFINITY;
    // a row that fits the list has had no first launch
    const float* maxima = a.maxima(row);
    const bool small = a.V <= SAMPLE_LIST;
    if (small) {
      visit([&](int c, int, const float (&l)[E]) {
        float t = l[0];
#pragma unroll
        for (int e = 1; e < E; e++) t = fmaxf(t, l[e]);
        t = cell_max(t);
        if (tid % SAMPLE_CELL == 0) s.maxima[c] = t;
      });
      __syncthreads();
    }
    for (int i = tid; i < cells; i += SAMPLE_THREADS) {
      const float c = small ? s.maxima[i] : maxima[i];
      s.maxima[i] = c;
      m = fmaxf(m, c);
      least = fminf(least, c > -INFINITY ? c : INFINITY);
    }
    m = wave_max(m);
    least = -wave_max(-least);
    if (lane == 0) {
      s.most[wave] = m;
      s.least[wave] = least;
    }
    if (tid == 0) {
      s.count = s.cells = 0;
      s.begin = 0.;
      s.at = 0x7fffffff;
    }
    reinterpret_cast<int*>(s.mass)[tid] = 0;  // (the counts of pivot)
    __syncthreads();
    for (int i = 0; i < SAMPLE_WAVES; i++) {
      m = fmaxf(m, s.most[i]);
      least = fminf(least, s.least[i]);
    }
    scale = 1023.f / (m - least);
  }

  __device__ __forceinline__ void answer(int token, double chosen, double all) const {
    a.tokens[row] = token;
    a.logprobs[row] = (float)log(chosen / all);
  }

  // f(cell, vector, its logits), every lane of a cell's 16 together, the loads four at a time: of all cells, or of the `n` chosen ones
  template <typename F>
  __device__ __forceinline__ void visit(F&& f, int n = -1) const {
    constexpr int U = 4, STEP = SAMPLE_THREADS / SAMPLE_CELL;
    const int end = n < 0 ? cells : n;
    for (int i = tid / SAMPLE_CELL; i < end; i += U * STEP) {
      float l[U][E];
      int c[U];
#pragma unroll
      for (int u = 0; u < U; u++)
        if (i + u * STEP < end) {
          c[u] = n < 0 ? i + u * STEP : s.chosen[i + u * STEP];
          x.load(c[u] * SAMPLE_CELL + tid % SAMPLE_CELL, l[u]);
        }
#pragma unroll
      for (int u = 0; u < U; u++)
        if (i + u * STEP < end) f(c[u], c[u] * SAMPLE_CELL + tid % SAMPLE_CELL, l[u]);
    }
  }

  // the cells that `wants`, in any order, and how many
  template <typename W>
  __device__ __forceinline__ int choose(W&& wants) const {
    for (int c = tid; c < cells; c += SAMPLE_THREADS)
      if (wants(s.maxima[c])) s.chosen[atomicAdd(&s.cells, 1)] = (unsigned short)c;
    __syncthreads();
    return s.cells;
  }

  // the first index of the largest logit
  __device__ __forceinline__ void greedy() const {
    const int n = choose([&](float l) { return l == m; });
    visit([&](int, int v, const float (&l)[E]) {
#pragma unroll
      for (int e = 0; e < E; e++)
        if (l[e] == m) atomicMin(&s.at, x.index(v, e));
    }, n);
    __syncthreads();
    if (tid == 0) answer(s.at, 1., 1.);
  }

  // Tokens for the list, ranked: the inverted key above the index
  __device__ __forceinline__ void push(float l, int i) const {
    const int at = atomicAdd(&s.count, 1);
    if (at < SAMPLE_LIST) s.list[at] = sample_rank(l, i);
  }
  __device__ __forceinline__ float listed(int at) const { return sample_logit(~(unsigned)(s.list[at] >> 32)); }

  // A bound that at least k tokens reach: the k-th largest of the cells' maxima, rounded down to 1/1023 of their range.  About
  // C log(1 / (1 - k / C)) tokens of C cells reach it; where k is more than half the cells, the k-th largest of all logits in
  // that range is taken instead, in a walk over the row.  A logit reaches the bound where !(scaled(l) < bound); that is monotone in l,
  // and true for the largest whatever the range is.
  __device__ __forceinline__ float scaled(float l) const { return (l - least) * scale; }
  __device__ __forceinline__ float pivot(int k) const {
    static_assert(SAMPLE_THREADS == 1024, "a thread per step");
    int* counts = reinterpret_cast<int*>(s.mass);
    const auto count = [&](float l) {
      // (the range may be beyond fp32, or all infinities: NaN is step 0, which every logit from `least` up reaches)
      if (l >= least) atomicAdd(&counts[1023 - (int)fminf(fmaxf(scaled(l), 0.f), 1023.f)], 1);
    };
    if (2 * k <= cells) {
      for (int i = tid; i < cells; i += SAMPLE_THREADS) count(s.maxima[i]);
    } else {
      visit([&](int, int, const float (&l)[E]) {
#pragma unroll
        for (int e = 0; e < E; e++) count(l[e]);
      });
    }
    __syncthreads();
    const int n = counts[tid];
    int upto = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_up(upto, o, 64);
      if (lane >= o) upto += y;
    }
    if (lane == 63) s.wi[wave] = upto;
    __syncthreads();
    for (int i = 0; i < wave; i++) upto += s.wi[i];
    if (upto >= k && upto - n < k) s.at = 1023 - tid;
    __syncthreads();
    // (fewer than k may have been counted: then all tokens are taken, and the list may come out too long)
    return s.at > 1023 ? -INFINITY : (float)s.at;
  }

  // Of the sorted list, behind tokens of weight `before`: the last token kept by top-k and top-p (goal < 0: of the list's own weight)
  __device__ __forceinline__ uint64_t cut(const Weights& weight, int n, int k, double before, double goal) const {
    const int most = k ? min(k, n) : n;
    const double w = tid < most ? (double)weight(listed(tid)) : 0.;
    double all;
    const double upto = before + group_scan(w, s, all);
    if (goal < 0.) goal = set.top_p < 1.f ? (double)set.top_p * all : INFINITY;
    // kept: what has less than the goal before it (weights that are zero stay out of the draw by themselves)
    const bool kept = tid < most && (tid == 0 || upto - w < goal);
    const bool next = tid + 1 < most && upto < goal;
    if (kept && !next) s.last = s.list[tid];
    __syncthreads();
    return s.last;
  }

  // The same for a list in any order, of up to SAMPLE_COUNTED tokens, by comparing all with all: a thread adds up what a share of the
  // list puts before its token, and the shares of a token meet in LDS (sums are exact).  That has fewer steps that wait for each
  // other than a sort, but reads LDS n^2 / 64 times: one row with top-k 50, of which 52 tokens are listed, 14.6 us sorted and 11.8
  // counted; 256 rows with top-k 200 (230 tokens) 42.8 and 47.2.
  __device__ __forceinline__ int mine(int n, int& part, int& parts) const {
    int size = WAVE;
    while (size < n) size *= 2;
    part = tid / size;
    parts = SAMPLE_THREADS / size;
    return tid & (size - 1);
  }
  __device__ __forceinline__ void count_ranks(const Weights& weight, int n) const {
    if (tid < n) {
      s.weight[tid] = (double)weight(listed(tid));
      s.sums[0][tid] = s.sums[1][tid] = 0.;
      s.ranks[tid] = 0;
    }
    __syncthreads();
    int part, parts;
    const int i = mine(n, part, parts);
    if (i < n) {
      const uint64_t token = s.list[i];
      int rank = 0;
      double before = 0.;
      for (int j = part; j < n; j += parts) {
        const bool first = s.list[j] < token;
        rank += first;
        before += first ? s.weight[j] : 0.;
      }
      atomicAdd(&s.ranks[i], rank);
      atomicAdd(&s.sums[0][i], before);
    }
    __syncthreads();
  }
  __device__ __forceinline__ uint64_t cut_counted(const Weights& weight, int n, double before, double goal) const {
    count_ranks(weight, n);
    const bool kept = tid < n && (s.ranks[tid] == 0 || before + s.sums[0][tid] < goal);
    // the last one kept is the one that as many are kept before as its rank says
    const int many = __syncthreads_count(kept);
    if (kept && s.ranks[tid] == many - 1) s.last = s.list[tid];
    __syncthreads();
    return s.last;
  }
  // Draws from list[0, n), n up to SAMPLE_COUNTED, in any order: weight[i] is a token's weight, 0 where it is not kept; sums[1] is zero
  __device__ __forceinline__ void draw_by_index(int n) const {
    __syncthreads();
    int part, parts;
    const int i = mine(n, part, parts);
    double mass = 0.;
    if (i < n) {
      const unsigned index = (unsigned)s.list[i];
      double before = 0.;
      for (int j = part; j < n; j += parts) {
        before += (unsigned)s.list[j] < index ? s.weight[j] : 0.;
        mass += s.weight[j];
      }
      atomicAdd(&s.sums[1][i], before);
      if (i == 0) atomicAdd(&s.begin, mass);
    }
    __syncthreads();
    mass = s.begin;
    const double drawn = (double)fminf(fmaxf(a.uniform[row], 0.f), 0x1.fffffep-1f) * mass;
    if (tid < n && s.weight[tid] > 0. && s.sums[1][tid] <= drawn && s.sums[1][tid] + s.weight[tid] > drawn)
      answer((int)(unsigned)s.list[tid], s.weight[tid], mass);
  }
  __device__ __forceinline__ void draw_counted(const Weights& weight, int n, int k) const {
    count_ranks(weight, n);
    const double w = tid < n ? s.weight[tid] : 0.;
    const bool in = tid < n && (k == 0 || s.ranks[tid] < k);
    double goal = INFINITY;
    if (set.top_p < 1.f) {
      double all;
      group_scan(in ? w : 0., s, all);
      goal = (double)set.top_p * all;
    }
    const double kept = in && (s.ranks[tid] == 0 || s.sums[0][tid] < goal) && (float)w >= set.min_p ? w : 0.;
    if (tid < n) s.weight[tid] = kept;
    draw_by_index(n);
  }

  // Draws from the list (`n` sorted by rank, those up to `last` kept)
  __device__ __forceinline__ void draw_listed(const Weights& weight, int n, uint64_t last) const {
    const int many = __syncthreads_count(tid < n && s.list[tid] <= last);
    if (many <= SAMPLE_COUNTED) {  // (the first ones)
      if (tid < many) {
        const float w = weight(listed(tid));
        s.weight[tid] = w >= set.min_p ? (double)w : 0.;
        s.sums[1][tid] = 0.;
      }
      return draw_by_index(many);
    }
    // by index: the kept ones only
    uint64_t mine = ~0ull;
    if (tid < n && s.list[tid] <= last && weight(listed(tid)) >= set.min_p) mine = (s.list[tid] << 32) | (s.list[tid] >> 32);
    const int kept = __syncthreads_count(mine != ~0ull);
    // (with min-p or without, they are a beginning of the list, but for weights that the hardware's exponential does not order)
    if (tid == 0) s.count = 0;
    __syncthreads();
    if (mine != ~0ull) s.list[atomicAdd(&s.count, 1)] = mine;
    __syncthreads();
    sort_list(s, kept);
    const double w = tid < kept ? (double)weight(sample_logit(~(unsigned)s.list[tid])) : 0.;
    double all;
    const double upto = group_scan(w, s, all);
    const double goal = (double)fminf(fmaxf(a.uniform[row], 0.f), 0x1.fffffep-1f) * all;
    if (w > 0. && upto > goal && upto - w <= goal) answer((int)(s.list[tid] >> 32), w, all);
  }

  // The weight in the draw of a token of the row, of which those that rank up to `last` are kept
  __device__ __forceinline__ double kept(const Weights& weight, float l, int i, uint64_t last) const {
    const float w = weight(l);
    return sample_rank(l, i) <= last && w >= set.min_p ? (double)w : 0.;
  }
  // Draws from the whole row, the cells' weights in s.mass
  __device__ __forceinline__ void draw_cells(const Weights& weight, uint64_t last) const {
    constexpr int PER = (SAMPLE_CELLS + SAMPLE_THREADS - 1) / SAMPLE_THREADS;
    double w[PER], sum = 0., all;
#pragma unroll
    for (int i = 0; i < PER; i++) {
      w[i] = tid * PER + i < cells ? s.mass[tid * PER + i] : 0.;
      sum += w[i];
    }
    const double upto = group_scan(sum, s, all);
    const double goal = (double)fminf(fmaxf(a.uniform[row], 0.f), 0x1.fffffep-1f) * all;
    if (upto > goal && upto - sum <= goal) {  // (one thread: sums are exact)
      double begin = upto - sum;
      int c = tid * PER;
#pragma unroll
      for (int i = 0; i < PER - 1; i++)
        if (c == tid * PER + i && begin + w[i] <= goal) {
          begin += w[i];
          c++;
        }
      s.at = c;
      s.begin = begin;
    }
    __syncthreads();
    if (tid >= SAMPLE_CELL) return;
    const int v = s.at * SAMPLE_CELL + tid;
    const double begin = s.begin;
    float l[E];
    double token[E];
    sum = 0.;
    x.load(v, l);
#pragma unroll
    for (int e = 0; e < E; e++) sum += token[e] = l[e] > -INFINITY ? kept(weight, l[e], x.index(v, e), last) : 0.;
    double here = sum;
#pragma unroll
    for (int o = 1; o < SAMPLE_CELL; o <<= 1) {
      const double y = __shfl_up(here, o, SAMPLE_CELL);
      if (tid >= o) here += y;
    }
    double left = begin + (here - sum);
    if (!(left + sum > goal && left <= goal)) return;
#pragma unroll
    for (int e = 0; e < E; e++) {
      if (left <= goal && left + token[e] > goal) answer(x.index(v, e), token[e], all);
      left += token[e];
    }
  }

  // ---- the cut by digits, over the whole row ----
  struct Digits {
    unsigned key;
    int ties;  // tokens of that key, the first by index
  };
  // the cut that keeps the first `goal_n` tokens, or the first tokens with a weight of goal_w
  __device__ __forceinline__ Digits find(const Weights& weight, bool by_count, int goal_n, double goal_w) const {
    double* mass = s.mass;
    int* count = reinterpret_cast<int*>(s.mass + 256);
    unsigned prefix = 0;
    double before = 0.;
    const double goal = by_count ? (double)goal_n : goal_w;
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = tid; i < 256; i += SAMPLE_THREADS) {
        mass[i] = 0.;
        count[i] = 0;
      }
      __syncthreads();
      for (int v = tid; v < nv; v += SAMPLE_THREADS) {
        float l[E];
        x.load(v, l);
#pragma unroll
        for (int e = 0; e < E; e++) {
          const unsigned key = sample_key(l[e]);
          if (shift < 24 && (key >> (shift + 8)) != (prefix >> (shift + 8))) continue;
          const unsigned digit = key >> shift & 255u;
          if (by_count) atomicAdd(&count[digit], 1);
          else if (const float w = weight(l[e]); w > 0.f) atomicAdd(&mass[digit], (double)w);
        }
      }
      __syncthreads();
      if (wave == 0) {
        // four digits a lane, the largest first
        double w[4], sum = 0.;
        for (int i = 0; i < 4; i++) sum += w[i] = by_count ? (double)count[255 - 4 * lane - i] : mass[255 - 4 * lane - i];
        double upto = sum;
        for (int o = 1; o < 64; o <<= 1) {
          const double y = __shfl_up(upto, o, 64);
          if (lane >= o) upto += y;
        }
        double begin = before + (upto - sum);
        const uint64_t reached = __ballot(before + upto >= goal);
        const int first = reached ? __ffsll((unsigned long long)reached) - 1 : 63;
        if (lane == first) {
          int i = 0;
          for (; i < 3 && begin + w[i] < goal; i++) begin += w[i];
          s.at = (int)(prefix | (unsigned)(255 - 4 * lane - i) << shift);
          s.begin = begin;
        }
      }
      __syncthreads();
      prefix = (unsigned)s.at;
      before = s.begin;
      __syncthreads();
    }
    if (by_count) return {prefix, prefix == sample_key(-INFINITY) ? 0 : goal_n - (int)before};  // (what is -inf has no weight)
    // equals have one weight: the j-th (from 0) is kept where what stands before it is below the goal
    const double w = (double)weight(sample_logit(prefix));
    double n = w > 0. ? ceil((goal_w - before) / w) : 1.;
    while (n > 1. && !(before + (n - 1.) * w < goal_w)) n -= 1.;
    while (w > 0. && before + n * w < goal_w) n += 1.;
    return {prefix, n < 1. ? 1 : n > 1e9 ? 1000000000 : (int)n};
  }
  // the weight of such a beginning, the same in every thread
  __device__ __forceinline__ double weigh(const Weights& weight, const Digits& d) const {
    double sum = 0.;
    for (int v = tid; v < nv; v += SAMPLE_THREADS) {
      float l[E];
      x.load(v, l);
#pragma unroll
      for (int e = 0; e < E; e++)
        if (sample_key(l[e]) > d.key) sum += (double)weight(l[e]);
    }
    double all;
    group_scan(sum, s, all);
    return d.ties ? all + (double)d.ties * (double)weight(sample_logit(d.key)) : all;
  }
  // where the cut goes through equals: the index of the first one left out
  __device__ __forceinline__ int end_of(const Digits& d) const {
    if (!d.ties) return 0;
    int* here = reinterpret_cast<int*>(s.mass);
    visit([&](int c, int v, const float (&l)[E]) {
            int n = 0;
#pragma unroll
            for (int e = 0; e < E; e++) n += sample_key(l[e]) == d.key;
#pragma unroll
            for (int o = SAMPLE_CELL / 2; o > 0; o >>= 1) n += __shfl_xor(n, o, 64);
            if (tid % SAMPLE_CELL == 0) here[c] = n;
          });
    if (tid == 0) s.at = 0x7fffffff;
    __syncthreads();
    if (tid == 0) {
      int left = d.ties;
      for (int c = 0; c < cells; c++) {
        if (here[c] > left) {
          for (int i = x.index(c * SAMPLE_CELL, 0); i < a.V; i++)
            if (sample_key(Elem<T>::to_f(x.p[i])) == d.key && left-- == 0) {
              s.at = i;
              break;
            }
          break;
        }
        left -= here[c];
      }
    }
    __syncthreads();
    const int end = s.at;
    __syncthreads();
    return end;
  }
  // the last token kept; weighs the cells
  __device__ __forceinline__ uint64_t by_digits(const Weights& weight) const {
    Digits d{sample_key(-INFINITY), 0};  // all tokens above -inf
    for (int by = 0; by < 2; by++) {
      if (by == 0 ? set.top_k == 0 : !(set.top_p < 1.f)) continue;
      const double goal = by == 0 ? 0. : (double)set.top_p * weigh(weight, d);
      d = find(weight, by == 0, set.top_k, goal);
    }
    const uint64_t last = ((uint64_t)~d.key << 32) + (int64_t)end_of(d) - 1;
    visit([&](int c, int v, const float (&l)[E]) {
            double sum = 0.;
#pragma unroll
            for (int e = 0; e < E; e++) sum += l[e] > -INFINITY ? kept(weight, l[e], x.index(v, e), last) : 0.;
            sum = cell_sum(sum);
            if (tid % SAMPLE_CELL == 0) s.mass[c] = sum;
          });
    __syncthreads();
    return last;
  }
};

template <typename T>
__global__ __launch_bounds__(SAMPLE_THREADS) void sample_pick_kernel(SampleArgs a) {
  __shared__ PickLds lds;
  const Picker<T> p(a, lds);
  const Settings& set = p.set;
  constexpr int E = Picker<T>::E;
  if (p.m == -INFINITY) {
    if (p.tid == 0) {
      a.tokens[p.row] = -1;
      a.logprobs[p.row] = -INFINITY;
    }
    return;
  }
  if (set.kind == GREEDY) return p.greedy();
  const Weights weight(p.m, set.temperature);
  uint64_t last = ~0ull;
  bool digits = set.kind == DIGITS;
  if (set.kind == LIST || set.kind == TOP_K || set.kind == MIN_P) {
    // all that may be kept is listed (a cell is looked into unless its largest weight is below min-p by more than the exponential's
    // own error)
    const float bound = set.kind == TOP_K ? p.pivot(set.top_k) : -INFINITY, floor = set.kind == MIN_P ? set.min_p : 0.f;
    const int cells = p.choose([&](float l) { return l > -INFINITY && !(p.scaled(l) < bound) && (floor == 0.f || weight(l) >= floor * 0.9999f); });
    p.visit([&](int, int v, const float (&l)[E]) {
#pragma unroll
      for (int e = 0; e < E; e++)
        if (l[e] > -INFINITY && !(p.scaled(l[e]) < bound) && (floor == 0.f || weight(l[e]) >= floor)) p.push(l[e], p.x.index(v, e));
    }, cells);
    __syncthreads();
    const int n = lds.count;
    if (n <= SAMPLE_COUNTED) return p.draw_counted(weight, n, set.top_k);
    if (n <= SAMPLE_LIST) {
      sort_list(lds, n);
      return p.draw_listed(weight, n, p.cut(weight, n, set.top_k, 0., -1.));
    }
    digits = true;
  }
  if (set.kind == TOP_P) {
    // what ranks before the cut's stretch has been weighed, what lies in it is on the list
    const SampleArgs::Walk& walk = *a.walk(p.row);
    const int n = walk.count;
    digits = n > SAMPLE_LIST;
    if (!digits) {
      for (int c = p.tid; c < p.cells; c += SAMPLE_THREADS) lds.mass[c] = a.masses(p.row)[c];
      if (p.tid < n) lds.list[p.tid] = a.list(p.row)[p.tid];
      __syncthreads();
      if (n <= SAMPLE_COUNTED) {
        last = p.cut_counted(weight, n, walk.before, walk.goal);
      } else {
        sort_list(lds, n);
        last = p.cut(weight, n, 0, walk.before, walk.goal);
      }
      if (p.tid < n && lds.list[p.tid] <= last) {
        const float y = weight(p.listed(p.tid));
        if (y >= set.min_p) atomicAdd(&lds.mass[p.x.cell_of((int)(unsigned)lds.list[p.tid])], (double)y);
      }
    }
  }
  if (set.kind == ALL)
    for (int c = p.tid; c < p.cells; c += SAMPLE_THREADS) lds.mass[c] = a.masses(p.row)[c];
  __syncthreads();
  if (digits) last = p.by_digits(weight);
  p.draw_cells(weight, last);
}

inline bool sample_needs_mass(const SampleArgs& a) {  // whether any row may, from what the host knows
  const bool greedy = !a.temperatures && !(a.temperature > 0.f), top_k = !a.top_ks && a.top_k > 0 && a.top_k < a.V;
  const bool min_p = !a.min_ps && a.min_p > 0.f && !a.top_ps && a.top_p >= 1.f;
  return a.V > SAMPLE_LIST && !greedy && !top_k && !min_p;
}

template <typename T>
void sample_launch(const SampleArgs& a, int B, hipStream_t st) {
  // vectors a thread of the first launch; us, one row of 128256 fp32, 256 rows: 2 14.3, 38.4; 4 15.1, 39.9; 8 16.6, 41.7
  const int vectors = a.V / Row<T>::E + 3 * SAMPLE_CELL, first = (vectors + SAMPLE_SPLIT * SAMPLE_FIRST - 1) / (SAMPLE_SPLIT * SAMPLE_FIRST);
  if (a.V > SAMPLE_LIST) sample_cells_kernel<T><<<dim3(first, B), SAMPLE_SPLIT, 0, st>>>(a);
  if (sample_needs_mass(a)) {
    // a share's fixed work - the cells' maxima, the bins - is that of some thousand logits, so no more shares than fill the CUs; twice as
    // many where the settings are the rows' own, since only some rows need this then.  256 rows, 2048 : 4096, us: all with top-p 119 : 135,
    // settings of their own 90 : 84
    const int shares = SAMPLE_SHARES * (a.top_ks || a.top_ps || a.temperatures ? 2 : 1);
    const int parts = std::max(1, std::min((vectors + 4 * SAMPLE_SPLIT - 1) / (4 * SAMPLE_SPLIT), shares / B)), share = ((vectors + parts - 1) / parts + SAMPLE_CELL - 1) / SAMPLE_CELL * SAMPLE_CELL;
    sample_mass_kernel<T><<<dim3(parts, B), SAMPLE_SPLIT, 0, st>>>(a, share, first);
    if (a.top_ps || a.top_p < 1.f) sample_walk_kernel<T><<<dim3(parts, B), SAMPLE_SPLIT, 0, st>>>(a, share, first);
  }
  sample_pick_kernel<T><<<B, SAMPLE_THREADS, 0, st>>>(a);
}

}  // namespace tp

extern "C" size_t tp_sample_workspace_bytes(int B, int V) {
  using namespace tp;
  if (B < 1 || V < 1 || V > SAMPLE_MOST) return 0;
  return V <= SAMPLE_LIST ? 16 : B * (size_t)SampleArgs::ws_row(sample_cells(V));  // (a row that fits the list stays in its workgroup)
}

extern "C" int tp_sample(const void* logits, const float* uniform, const float* temperatures, const int32_t* top_ks, const float* top_ps,
                         const float* min_ps, float temperature, int top_k, float top_p, float min_p, int64_t* tokens, float* logprobs, void* ws,
                         int B, int V, int64_t row_stride, int dtype, void* stream) {
  using namespace tp;
  TP_REQUIRE(logits && uniform && tokens && logprobs, TP_ERR_BAD_ARG, "tp_sample: null pointer");
  TP_REQUIRE(B >= 1 && V >= 1 && row_stride >= V, TP_ERR_BAD_ARG, "tp_sample: sizes must be positive and rows must not overlap");
  TP_REQUIRE(V <= SAMPLE_MOST && B < (1 << 16), TP_ERR_UNSUPPORTED, "tp_sample: V=%d (at most 2^18), B=%d (below 2^16)", V, B);
  TP_REQUIRE(dtype >= TP_BF16 && dtype <= TP_F32, TP_ERR_UNSUPPORTED, "tp_sample: unsupported dtype code %d", dtype);
  TP_REQUIRE(((uintptr_t)logits & (dtype == TP_F32 ? 3 : 1)) == 0 && aligned16(ws), TP_ERR_BAD_ARG, "tp_sample: misaligned logits or workspace");
  TP_REQUIRE(ws, TP_ERR_BAD_ARG, "tp_sample: no workspace");
  const SampleArgs a{logits, uniform, temperatures, top_ps, min_ps, top_ks, temperature, top_p, min_p, top_k, tokens, logprobs, (char*)ws, row_stride, V,
                     sample_cells(V)};
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == TP_F32) sample_launch<float>(a, B, st);
  else if (dtype == TP_BF16) sample_launch<bf16_t>(a, B, st);
  else sample_launch<f16_t>(a, B, st);
  return check_launch("tp_sample");
}
