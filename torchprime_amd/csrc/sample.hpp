// The next token from a row of logits: temperature, top-k, top-p, min-p, and a draw with a given random number.
//
//   w = 2^((l - m) c), m the largest logit, c = log2(e) / temperature; 1 where l == m;   then (w + 2^-12) - 2^-12 in fp32
//
// The last step makes every weight a multiple of 2^-35 (w is at most 1), so sums of up to 2^18 of them are exact in fp64: they
// come out the same in any order and over any split of the row, and so do the token and every cut through the distribution.
// Weights below 2^-36 become zero; such tokens are never drawn.
//
// Tokens are ranked by falling logit, the lower index first among equals.  Every filter keeps a beginning of that order, which a
// logit and a number of its equals describe (Cut); the cut of top-k (by count) and of top-p (by weight) is found digit by
// digit over the 32 bits of an order-preserving integer key of the logit.  The draw walks the kept tokens by index, which needs no
// sort: a sum per stretch of the row, then the stretch that the drawn weight falls into.
#pragma once
#include <float.h>

#include "common.hpp"

namespace tp {

constexpr float SAMPLE_LOG2E = 1.4426950408889634f;
constexpr int SAMPLE_THREADS = 1024, SAMPLE_WAVES = SAMPLE_THREADS / WAVE;
constexpr int SAMPLE_MOST = 1 << 18;  // logits per row

struct SampleArgs {
  const void* logits;
  const float *uniform, *temperatures, *top_ps, *min_ps;
  const int32_t* top_ks;
  float temperature, top_p, min_p;
  int top_k;
  int64_t* tokens;
  float* logprobs;
  int64_t row_stride;
  int V;
};

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
  __device__ __forceinline__ float operator()(float l) const {
    const float w = l == m ? 1.f : __builtin_amdgcn_exp2f((l - m) * c);
    return (w + 0x1p-12f) - 0x1p-12f;
  }
};

// A beginning of the ranking: every key above `key`, and the first `ties` tokens (by index) that have it.
struct Cut {
  unsigned key;
  int ties;
};

// The logits of a row, 16 bytes at a time from 16-byte addresses; elements outside the row are -inf.
template <typename T>
struct Row {
  static constexpr int E = 16 / sizeof(T);
  const T* base;  // 16-byte aligned, `lead` elements before the row's first
  int lead, V;
  __device__ __forceinline__ Row(const T* p, int v) : lead((int)(((size_t)p & 15) / sizeof(T))), V(v) { base = p - lead; }
  __device__ __forceinline__ int vectors() const { return (V + lead + E - 1) / E; }
  __device__ __forceinline__ void load(int vec, float (&x)[E]) const {
    const int i0 = vec * E - lead;
    if (i0 >= 0 && i0 + E <= V) {
      load_f<T, E>(base + (int64_t)vec * E, x);
    } else {
#pragma unroll
      for (int e = 0; e < E; e++) x[e] = i0 + e >= 0 && i0 + e < V ? Elem<T>::to_f(base[(int64_t)vec * E + e]) : -INFINITY;
    }
#pragma unroll
    for (int e = 0; e < E; e++) x[e] = x[e] == x[e] ? x[e] : -INFINITY;
  }
};

__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

template <typename T>
__global__ __launch_bounds__(SAMPLE_THREADS) void sample_rows_kernel(SampleArgs a) {
  constexpr int E = Row<T>::E;
  __shared__ double mass[256];
  __shared__ int count[256];
  __shared__ double stretch[SAMPLE_MOST / WAVE / E + 2];
  __shared__ float wm[SAMPLE_WAVES];
  __shared__ int wi[SAMPLE_WAVES];
  __shared__ double wd[SAMPLE_WAVES];
  __shared__ unsigned found_key;
  __shared__ int found_at;
  __shared__ double found_before;
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const Row<T> x(reinterpret_cast<const T*>(a.logits) + row * a.row_stride, a.V);
  const int nv = x.vectors(), stretches = (nv + WAVE - 1) / WAVE;

  // the largest logit, its first index
  float m = -INFINITY;
  int at = 0x7fffffff;
  for (int v = tid; v < nv; v += SAMPLE_THREADS) {
    float l[E];
    x.load(v, l);
#pragma unroll
    for (int e = 0; e < E; e++)
      if (l[e] > m) {
        m = l[e];
        at = v * E + e - x.lead;
      }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const float m2 = __shfl_xor(m, o, 64);
    const int at2 = __shfl_xor(at, o, 64);
    if (m2 > m || (m2 == m && at2 < at)) {
      m = m2;
      at = at2;
    }
  }
  if (lane == 0) {
    wm[wave] = m;
    wi[wave] = at;
  }
  __syncthreads();
  for (int i = 0; i < SAMPLE_WAVES; i++)
    if (wm[i] > m || (wm[i] == m && wi[i] < at)) {
      m = wm[i];
      at = wi[i];
    }
  const float temperature = a.temperatures ? a.temperatures[row] : a.temperature;
  if (m == -INFINITY || !(temperature > 0.f)) {  // (the same for the whole workgroup)
    if (tid == 0) {
      a.tokens[row] = m == -INFINITY ? -1 : at;
      a.logprobs[row] = m == -INFINITY ? -INFINITY : 0.f;
    }
    return;
  }
  const Weights weight{m, fmaxf(SAMPLE_LOG2E / temperature, FLT_MIN)};  // (not 0: an infinite temperature keeps -inf out)

  // the cut that keeps the first `goal_n` tokens, or the first tokens with a weight of goal_w
  const auto find = [&](bool by_count, int goal_n, double goal_w) {
    unsigned prefix = 0;
    double w_before = 0.;
    int n_before = 0;
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
          else atomicAdd(&mass[digit], (double)weight(l[e]));
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
        const double goal = by_count ? (double)goal_n : goal_w, before = by_count ? (double)n_before : w_before;
        double begin = before + (upto - sum);
        const uint64_t reached = __ballot(before + upto >= goal);
        const int first = reached ? __ffsll((unsigned long long)reached) - 1 : 63;
        if (lane == first) {
          int i = 0;
          for (; i < 3 && begin + w[i] < goal; i++) begin += w[i];
          found_key = prefix | (unsigned)(255 - 4 * lane - i) << shift;
          found_before = begin;
        }
      }
      __syncthreads();
      prefix = found_key;
      if (by_count) n_before = (int)found_before;
      else w_before = found_before;
      __syncthreads();
    }
    Cut cut{prefix, 0};
    if (by_count) {
      cut.ties = prefix == sample_key(-INFINITY) ? 0 : goal_n - n_before;  // (what is -inf has no weight)
    } else {
      // equals have one weight: the j-th (from 0) is kept where what stands before it is below the goal
      const double w = (double)weight(sample_logit(prefix));
      double n = w > 0. ? ceil((goal_w - w_before) / w) : 1.;
      while (n > 1. && !(w_before + (n - 1.) * w < goal_w)) n -= 1.;
      while (w > 0. && w_before + n * w < goal_w) n += 1.;
      cut.ties = n < 1. ? 1 : n > 1e9 ? 1000000000 : (int)n;
    }
    return cut;
  };
  // the weight of a beginning, the same in every thread; equals beyond the cut are told apart by number, not by index
  const auto weigh = [&](const Cut& cut) {
    double sum = 0.;
    for (int v = tid; v < nv; v += SAMPLE_THREADS) {
      float l[E];
      x.load(v, l);
#pragma unroll
      for (int e = 0; e < E; e++)
        if (sample_key(l[e]) > cut.key) sum += (double)weight(l[e]);
    }
    sum = wave_sum_f64(sum);
    if (lane == 0) wd[wave] = sum;
    __syncthreads();
    sum = 0.;
    for (int i = 0; i < SAMPLE_WAVES; i++) sum += wd[i];
    __syncthreads();
    return cut.ties ? sum + (double)cut.ties * (double)weight(sample_logit(cut.key)) : sum;
  };

  Cut cut{sample_key(-INFINITY), 0};  // all tokens above -inf
  const int top_k = a.top_ks ? a.top_ks[row] : a.top_k;
  const float top_p = fminf(fmaxf(a.top_ps ? a.top_ps[row] : a.top_p, 0.f), 1.f);
  if (top_k > 0 && top_k < a.V) cut = find(true, top_k, 0.);
  if (top_p < 1.f) {
    const double goal = (double)top_p * weigh(cut);
    if (goal > 0.) cut = find(false, 0, goal);
    else cut = Cut{sample_key(m), 1};
  }
  // where the cut goes through equals: the index of the first one left out
  int end = 0x7fffffff;
  if (cut.ties) {
    int* here = reinterpret_cast<int*>(stretch);
    for (int s = wave; s < stretches; s += SAMPLE_WAVES) {
      const int v = s * WAVE + lane;
      int n = 0;
      if (v < nv) {
        float l[E];
        x.load(v, l);
#pragma unroll
        for (int e = 0; e < E; e++) n += sample_key(l[e]) == cut.key;
      }
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o, 64);
      if (lane == 0) here[s] = n;
    }
    if (tid == 0) found_at = 0x7fffffff;
    __syncthreads();
    if (tid == 0) {
      int left = cut.ties;
      for (int s = 0; s < stretches; s++) {
        if (here[s] > left) {
          for (int i = max(0, s * WAVE * E - x.lead); i < a.V; i++) {
            const float l = Elem<T>::to_f(x.base[i + x.lead]);
            if (sample_key(l) == cut.key && left-- == 0) {
              found_at = i;
              break;
            }
          }
          break;
        }
        left -= here[s];
      }
    }
    __syncthreads();
    end = found_at;
    __syncthreads();
  }
  const float min_p = fminf(fmaxf(a.min_ps ? a.min_ps[row] : a.min_p, 0.f), 1.f);
  // weight of token i with logit l in the draw: zero where it is not kept
  const auto kept = [&](float l, int i) {
    const unsigned key = sample_key(l);
    const float w = weight(l);
    return (key > cut.key || (key == cut.key && i < end && cut.ties)) && w >= min_p ? (double)w : 0.;
  };
  for (int s = wave; s < stretches; s += SAMPLE_WAVES) {
    const int v = s * WAVE + lane;
    double sum = 0.;
    if (v < nv) {
      float l[E];
      x.load(v, l);
#pragma unroll
      for (int e = 0; e < E; e++) sum += kept(l[e], v * E + e - x.lead);
    }
    sum = wave_sum_f64(sum);
    if (lane == 0) stretch[s] = sum;
  }
  __syncthreads();
  if (wave == 0) {
    const int per = (stretches + 63) / 64;
    double sum = 0.;
    for (int i = 0; i < per && lane * per + i < stretches; i++) sum += stretch[lane * per + i];
    double upto = sum;
    for (int o = 1; o < 64; o <<= 1) {
      const double y = __shfl_up(upto, o, 64);
      if (lane >= o) upto += y;
    }
    const double all = __shfl(upto, 63, 64);
    const float u = fminf(fmaxf(a.uniform[row], 0.f), 0x1.fffffep-1f);
    const double goal = (double)u * all;
    int l0 = __ffsll((unsigned long long)__ballot(upto > goal)) - 1;  // (all > goal)
    double before = __shfl(upto - sum, l0, 64);
    int s = l0 * per;
    while (before + stretch[s] <= goal) before += stretch[s++];
    // inside the stretch
    const int v = s * WAVE + lane;
    double w[E];
    sum = 0.;
    float l[E];
    if (v < nv) x.load(v, l);
#pragma unroll
    for (int e = 0; e < E; e++) sum += w[e] = v < nv ? kept(l[e], v * E + e - x.lead) : 0.;
    upto = sum;
    for (int o = 1; o < 64; o <<= 1) {
      const double y = __shfl_up(upto, o, 64);
      if (lane >= o) upto += y;
    }
    l0 = __ffsll((unsigned long long)__ballot(before + upto > goal)) - 1;
    if (lane == l0) {
      before += upto - sum;
      int e = 0;
#pragma unroll
      for (int i = 0; i < E - 1; i++)
        if (e == i && before + w[i] <= goal) {
          before += w[i];
          e = i + 1;
        }
      double chosen = w[0];
#pragma unroll
      for (int i = 1; i < E; i++) chosen = e == i ? w[i] : chosen;
      a.tokens[row] = v * E + e - x.lead;
      a.logprobs[row] = (float)log(chosen / all);
    }
  }
}

}  // namespace tp

extern "C" size_t tp_sample_workspace_bytes(int B, int V) { return 0; }

extern "C" int tp_sample(const void* logits, const float* uniform, const float* temperatures, const int32_t* top_ks, const float* top_ps,
                         const float* min_ps, float temperature, int top_k, float top_p, float min_p, int64_t* tokens, float* logprobs, void* ws,
                         int B, int V, int64_t row_stride, int dtype, void* stream) {
  using namespace tp;
  TP_REQUIRE(logits && uniform && tokens && logprobs, TP_ERR_BAD_ARG, "tp_sample: null pointer");
  TP_REQUIRE(B >= 1 && V >= 1 && row_stride >= V, TP_ERR_BAD_ARG, "tp_sample: sizes must be positive and rows must not overlap");
  TP_REQUIRE(V <= SAMPLE_MOST && B < (1 << 22), TP_ERR_UNSUPPORTED, "tp_sample: V=%d (at most 2^18), B=%d (below 2^22)", V, B);
  TP_REQUIRE(dtype >= TP_BF16 && dtype <= TP_F32, TP_ERR_UNSUPPORTED, "tp_sample: unsupported dtype code %d", dtype);
  TP_REQUIRE(((uintptr_t)logits & (dtype == TP_F32 ? 3 : 1)) == 0, TP_ERR_BAD_ARG, "tp_sample: misaligned logits");
  const SampleArgs a{logits, uniform, temperatures, top_ps, min_ps, top_ks, temperature, top_p, min_p, top_k, tokens, logprobs, row_stride, V};
  if (dtype == TP_F32) sample_rows_kernel<float><<<B, SAMPLE_THREADS, 0, (hipStream_t)stream>>>(a);
  else if (dtype == TP_BF16) sample_rows_kernel<bf16_t><<<B, SAMPLE_THREADS, 0, (hipStream_t)stream>>>(a);
  else sample_rows_kernel<f16_t><<<B, SAMPLE_THREADS, 0, (hipStream_t)stream>>>(a);
  return check_launch("tp_sample");
}
