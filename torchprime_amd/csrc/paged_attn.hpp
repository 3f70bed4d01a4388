// Attention of one new token per sequence over the paged cache (kv_cache.hpp):
//
//   s_j = cap(scale * q . k_j),   out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),   m = max_j s_j
//
// in one pass over the keys, with a running maximum, sum and weighted sum of values (Milakov and Gimelshein, "Online normalizer
// calculation for softmax", 2018).  A key and its value are used by the g = Hq / Hkv query heads that share them: 2 g flops for
// each element read, so it is the reading of the cache that bounds long calls, and the chain of dependent loads short ones.
//
// paged_attn_kernel: the g heads are the 16 columns of 16x16x32 matrix products (fp32: 16x16x4; more than 16 heads: blocks of 16, the
// unused columns zero), which costs a few percent of the time that the bytes take, whatever g is.  Layouts (lane: r = lane
// % 16, g = lane / 16): A and B hold row / column r, k = 8 g + 0..7; C holds column r, rows 4 g + 0..3.  A wave takes 32 keys at a
// time, straight from memory into the operands, without LDS and without an exchange between lanes:
//   * scores are S^T = K Q^T, two products of 16 keys.  Row i of product t is key 8 (i / 4) + 4 t + i % 4, so that the scores of a
//     lane, rows 4 g + 0..3 of both, are those of keys 8 g + 0..7, which is its share of the B operand of O^T += V^T P^T.
//   * for V^T a lane needs 8 keys of one column, memory holds columns side by side: a lane loads the same DV / 16 columns of its 8
//     keys, pairs the keys' halves with one v_perm per two elements, and product t takes column DV / 16 * r + t.  A row of values is
//     read in one instruction by the 16 lanes of a group, and a lane ends with DV / 4 neighbouring columns of its head.
//
// Measured (8 kv heads of 128, 32 query heads, bfloat16 unless said): one sequence of 131072 keys 92 us = 5.8 TB/s, in 8 bits 59 us =
// 4.7 TB/s, heads of 64 60 us = 4.4 TB/s (8 bits 44 us = 3.3 TB/s: loads of 8 and 4 bytes a lane for the values); 128 sequences of 512
// to 8192 265 us = 6.1 TB/s, in 8 bits 157 us = 5.3 TB/s; 128 heads of (192, 128), float16, up to 1537 keys 68 us = 4.6 TB/s, in 8 bits 52 us =
// 3.1 TB/s; fp32, 16384 keys 34 us = 3.9 TB/s; one sequence of 461 keys 9.0 us.  In the long ones the workgroups of a round keep 26 MB on their way and a tile takes 4 us, which is the
// memory's rate; around that stand the launch and the chain lengths -> table -> keys of the first tile (about 2 us), and the join (4 to
// 5 us with its launch).  The short ones are that chain, and what one CU can load.  Loading a wave's next tile into registers while it
// works on one was slower everywhere (118 against 92 us at 131072 keys: 256 registers and spills; 9.4 against 8.8 at 461).
#pragma once
#include "attn_common.hpp"
#include "kv_cache.hpp"

namespace tp {

struct PagedAttnArgs {
  PageRows k, v;
  PageTable table;
  const void* q;
  const int32_t* lengths;
  void* out;
  float* lse;
  float* ws;
  int64_t q_b, q_h, o_b, o_h;
  int B, Hq, heads;  // heads: of keys and values
  int blocks;        // of 16 query heads that share a kv head
  int rows;          // query heads per block, at most 16
  float scale;       // log2(e) * sm_scale; without log2(e) where soft_cap is set
  float cap;         // soft_cap, 0: none
  int window;        // keys before the newest that are seen, negative: all
};

// ------------------------------------------------------------------------------------------------
// fp32 heads of (192, 128), whose operands do not fit a wave's registers: one workgroup per (sequence, query head); a thread takes a
// key of every 256, then a few columns of the values.  Not split over the keys: 512 heads of up to 1537 keys 171 us = 3.7 TB/s, but one
// sequence of 16384 with 32 heads, which are 32 workgroups, 1184 us = 0.6 TB/s
// ------------------------------------------------------------------------------------------------
constexpr int PA_KEYS = 256;
__global__ __launch_bounds__(PA_KEYS) void paged_attn_rows_kernel(PagedAttnArgs a) {
  __shared__ float q[512], p[PA_KEYS], part[4], acc_lds[PA_KEYS * 8];
  __shared__ int64_t at_v[PA_KEYS];
  const int b = blockIdx.x / a.Hq, h = blockIdx.x - b * a.Hq, kv = h / (a.Hq / a.heads), tid = threadIdx.x;
  const float* qp = reinterpret_cast<const float*>(a.q) + b * a.q_b + h * a.q_h;
  for (int i = tid; i < a.k.dim; i += PA_KEYS) q[i] = qp[i];
  const int n = min(a.lengths[b], a.table.width << a.table.page_shift);
  const int first = a.window >= 0 ? max(0, n - 1 - a.window) : 0;
  const int lane = tid & (a.v.group - 1), sub = tid / a.v.group, subs = PA_KEYS / a.v.group;
  float m = -INFINITY, l = 0.f, acc[8] = {};
  __syncthreads();
  for (int j0 = first; j0 < n; j0 += PA_KEYS) {
    const int j = j0 + tid, page = j < n ? a.table.page_of(b, j) : -1, slot = j & ((1 << a.table.page_shift) - 1);
    float s = -INFINITY;
    if (page >= 0) {
      const int64_t at = page * a.k.page + kv * a.k.head + slot * a.k.slot;
      s = 0.f;
      for (int d = 0; d < a.k.dim; d += 8) {
        float x[8];
        load_f<float, 8>(reinterpret_cast<const float*>(a.k.base) + at + d, x);
#pragma unroll
        for (int e = 0; e < 8; e++) s += x[e] * q[d + e];
      }
      s *= a.scale;
      if (a.cap > 0.f) s = a.cap * LOG2E * tanhf(s / a.cap);
    }
    float mx = wave_max(s);
    if ((tid & 63) == 0) part[tid >> 6] = mx;
    __syncthreads();
    mx = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
    const float m_new = fmaxf(m, mx), base = m_new == -INFINITY ? 0.f : m_new;
    const float shrink = exp2f(m - base);
    const float w = page >= 0 ? exp2f(s - base) : 0.f;
    l = l * shrink + w;  // this thread's keys
    p[tid] = w;
    at_v[tid] = page >= 0 ? page * a.v.page + kv * a.v.head + slot * a.v.slot : -1;
    m = m_new;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 8; e++) acc[e] *= shrink;
    if (lane * 8 < a.v.dim) {
      for (int i = sub; i < PA_KEYS && j0 + i < n; i += subs) {
        if (at_v[i] < 0) continue;  // (not loaded: what lies there takes no part, whatever it is)
        float x[8];
        load_f<float, 8>(reinterpret_cast<const float*>(a.v.base) + at_v[i] + lane * 8, x);
#pragma unroll
        for (int e = 0; e < 8; e++) acc[e] += p[i] * x[e];
      }
    }
    __syncthreads();
  }
  l = wave_sum(l);
  if ((tid & 63) == 0) part[tid >> 6] = l;
#pragma unroll
  for (int e = 0; e < 8; e++) acc_lds[tid * 8 + e] = acc[e];
  __syncthreads();
  l = part[0] + part[1] + part[2] + part[3];
  for (int d = tid; d < a.v.dim; d += PA_KEYS) {
    float o = 0.f;
    for (int i = 0; i < subs; i++) o += acc_lds[(i * a.v.group + d / 8) * 8 + d % 8];
    reinterpret_cast<float*>(a.out)[b * a.o_b + h * a.o_h + d] = l != 0.f ? o / l : 0.f;
  }
  if (tid == 0 && a.lse) a.lse[(int64_t)b * a.Hq + h] = l != 0.f ? (m + log2f(l)) * LN2 : -INFINITY;
}

// ------------------------------------------------------------------------------------------------
// how the work is shared out
// ------------------------------------------------------------------------------------------------
// A segment is a (sequence, kv head, block of query heads); a unit is what a workgroup takes of it in one step, 32 keys a wave.
// Segments in order are one line of units, of which every workgroup takes the same number: a long sequence among short ones is
// shared by many workgroups, and short ones go several to a workgroup.  Nothing of that needs the host to know the lengths.  A
// segment that lies in one workgroup leaves as the result; one that is cut leaves its pieces (maximum, sum, weighted sum) in the
// workspace: piece 2 w of workgroup w if it begins there with the workgroup, else 2 w + 1; paged_attn_join_kernel adds them up in
// their order, so that a call gives the same bits every time.
constexpr int PA_TILE = 32;

struct Keys {  // of one sequence: [first, end), and `base`, the multiple of 32 at or below first, where units begin
  int first, end, base;
  __device__ __forceinline__ Keys(const PagedAttnArgs& a, int length) {
    end = max(0, min(length, a.table.width << a.table.page_shift));
    first = a.window >= 0 ? max(0, end - 1 - a.window) : 0;
    base = first & ~(PA_TILE - 1);
  }
  // (an empty sequence has its unit, too: its zeros have to be written)
  __device__ __forceinline__ int units(int unit) const { return max(1, (end - base + unit - 1) / unit); }
};

struct Share {
  int per, total;  // units per workgroup, and in all
  int b, at;       // the sequence that the share's first unit belongs to, and the number of units before that sequence
  int length;      // that sequence's
};
__device__ __forceinline__ int wave_scan(int v, int lane) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(v, o, 64);
    if (lane >= o) v += y;
  }
  return v;
}
// Every wave works this out by itself; a lane counts ceil(B / 64) sequences.
template <int UNIT>
__device__ __forceinline__ Share share_of(const PagedAttnArgs& a, int groups, int w) {
  const int lane = threadIdx.x & 63, each = (a.B + 63) / 64, segs = a.heads * a.blocks;
  const int b0 = min(lane * each, a.B), b1 = min(b0 + each, a.B);
  int n = 0, length = 0;
  for (int b = b0; b < b1; b++) {
    length = a.lengths[b];
    n += Keys(a, length).units(UNIT);
  }
  const int upto = wave_scan(n, lane);
  Share s;
  s.total = __shfl(upto, 63, 64) * segs;
  s.per = (s.total + groups - 1) / groups;
  const int u = w * s.per;
  s.b = s.at = s.length = 0;
  if (u >= s.total) return s;
  const int l0 = __ffsll((unsigned long long)__ballot(upto * segs > u)) - 1;
  s.b = min(l0 * each, a.B - 1);
  s.at = __shfl(upto - n, l0, 64) * segs;
  s.length = __shfl(length, l0, 64);
  if (each > 1) {
    for (;;) {  // (ends within the lane's sequences: their units reach beyond u)
      s.length = a.lengths[s.b];
      const int here = Keys(a, s.length).units(UNIT) * segs;
      if (s.at + here > u) break;
      s.at += here;
      s.b++;
    }
  }
  return s;
}

// What a workgroup whose first unit lies inside a segment says about it, where this is the segment's first cut (else rows = 0)
struct SegmentCut {
  int rows, b, h0, first, last, lead;  // its workgroups; 1 where the first one's piece is not its first
  int none[2];
};
constexpr int pa_piece_floats(int dv) { return 2 * 16 + 16 * dv; }  // maxima, sums, weighted sums
__device__ __forceinline__ float* pa_piece(const PagedAttnArgs& a, int groups, int i, int dv) {  // behind the cuts
  return a.ws + (int64_t)groups * (int)(sizeof(SegmentCut) / 4) + (int64_t)i * pa_piece_floats(dv);
}

template <typename T> struct MM;
template <> struct MM<float> {
  static __device__ __forceinline__ f32x4 dot(float a, float b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }
};
template <> struct MM<bf16_t> {
  static __device__ __forceinline__ f32x4 dot(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ unsigned from_fp8(unsigned w, bool hi) {
    return __builtin_bit_cast(unsigned, hi ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, true) : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, false));
  }
};
template <> struct MM<f16_t> {
  static __device__ __forceinline__ f32x4 dot(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ unsigned from_fp8(unsigned w, bool hi) {
    return __builtin_bit_cast(unsigned, hi ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, true) : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, false));
  }
};

// over the four lane groups that hold one head
__device__ __forceinline__ float groups_max(float v) {
  v = half_max(v);
  return fmaxf(v, __shfl_xor(v, 16, 64));
}
__device__ __forceinline__ float groups_sum(float v) {
  v = half_sum(v);
  return v + __shfl_xor(v, 16, 64);
}

// What a wave has of a segment.  The maximum m is lazy: it moves only when a score exceeds it by more than 8 (log2 units), so that the
// sums are rarely rescaled.  Weights (at most 2^8; float16: 2^15) go into the product as two numbers of type T, the rounded weight and the rest,
// which are off by 2^-18 of the weight together in bfloat16 and 2^-24 in float16 (or half its smallest step), where the result's rounding is
// off by 2^-9 and 2^-12; the second product costs less than the bytes leave room for.  In an 8-bit cache
// they carry the value's scale, and for float16, whose range is short, relative to 2^c, c the largest exponent of a scale so far.
template <int DV> struct Partial {
  float m, l;  // of this lane's head; l over this lane's keys
  int c;
  f32x4 o[DV / 16];
  __device__ __forceinline__ void clear() {
    m = -INFINITY;
    l = 0.f;
    c = -150;
#pragma unroll
    for (int t = 0; t < DV / 16; t++) o[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
};

template <typename T>
__device__ __forceinline__ void store4(T* p, f32x4 x) {
  if constexpr (std::is_same<T, float>::value) *reinterpret_cast<f32x4*>(p) = x;
  else *reinterpret_cast<u32x2*>(p) = pack4<T>(x[0], x[1], x[2], x[3]);
}

template <typename T, bool QUANT, int DQK, int DV>
struct PagedTile {
  static constexpr bool F32 = std::is_same<T, float>::value;
  typedef T v8 __attribute__((ext_vector_type(F32 ? 4 : 8)));  // 16 bytes
  static constexpr int B = QUANT ? 1 : sizeof(T);     // bytes of a cached element
  static constexpr int KL = DQK * B / 64;             // 16-byte loads of a key per lane
  static constexpr int KS = DQK / (F32 ? 16 : 32);    // 16-byte pieces of a query per lane
  static constexpr int C = DV / 16;                   // columns of V per lane
  static constexpr int VB = C * B;                    // their bytes
  static constexpr bool F16 = std::is_same<T, f16_t>::value, RANGE = QUANT && F16;
  static constexpr bool REST = !F32 && !QUANT;  // values may be infinite (e4m3 has no infinity), and a weight's rest 0
  // float16: weights from 2^7 (2^15 where the maximum lags) down to its smallest step, 2^-31 of the largest, so that thousands of keys far
  // below the maximum add up as they should
  static constexpr float UP = F16 ? 7.f : 0.f;

  static __device__ __forceinline__ void load_q(const PagedAttnArgs& a, const T* q, bool mine, v8 (&f)[KS]) {
    const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int i = 0; i < KS; i++) {
      // (8-bit keys: 16 bytes of a key, two products' shares, lie side by side)
      const int d = QUANT ? 64 * (i / 2) + 16 * g + 8 * (i % 2) : 64 / B * i + 16 / B * g;
      f[i] = mine ? *reinterpret_cast<const v8*>(q + d) : v8{};
    }
  }

  // One tile of keys key0 .. key0 + 31 on its way: where it lies, then what was loaded.
  struct Where {
    int pk, pv;  // pages of this lane's rows of keys and of values, -1: none
  };
  struct Data {
    u32x4 k[2][KL];
    unsigned v[8][VB / 4];
    float ks[QUANT ? 8 : 1], vs[QUANT ? 8 : 1];
    int tv;     // the first of this lane's eight keys
    bool page;  // they lie in a page
  };
  static __device__ __forceinline__ Where find(const PagedAttnArgs& a, int b, int key0) {
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int tk = key0 + 8 * (r >> 2), tv = key0 + 8 * g;  // eight keys from a multiple of 8 lie in one page
    return {a.table.page_of(b, tk), a.table.page_of(b, tv)};
  }
  // (Rows without a page are read from page 0, which is there, and dropped later.)
  static __device__ __forceinline__ void load(const PagedAttnArgs& a, const Where& at, int kv, int key0, Data& x) {
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4, mask = (1 << a.table.page_shift) - 1;
    const int tk = key0 + 8 * (r >> 2), tv = key0 + 8 * g;
    const char* kp = a.k.base + B * (max(at.pk, 0) * a.k.page + kv * a.k.head + ((tk & mask) + (r & 3)) * a.k.slot) + 16 * g;
    const char* vp = a.v.base + B * (max(at.pv, 0) * a.v.page + kv * a.v.head + (tv & mask) * a.v.slot) + VB * r;
    if constexpr (QUANT) {
      const int64_t row = (((int64_t)max(at.pv, 0) * a.heads + kv) << a.table.page_shift) + (tv & mask);
      load_f<float, 8>(a.k.scale + row, x.ks);
      load_f<float, 8>(a.v.scale + row, x.vs);
    }
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int i = 0; i < KL; i++) x.k[t][i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(kp + B * 4 * t * a.k.slot + 64 * i));
#pragma unroll
    for (int e = 0; e < 8; e++) {
      constexpr int W = VB > 16 ? 16 : VB;  // bytes of a load
      typedef unsigned row_t __attribute__((ext_vector_type(W / 4)));
#pragma unroll
      for (int j = 0; j < VB / W; j++) {
        const char* from = vp + B * e * a.v.slot + W * j;
        if constexpr (W == 4) {
          x.v[e][0] = __builtin_nontemporal_load(reinterpret_cast<const unsigned*>(from));
        } else {
          const row_t w = __builtin_nontemporal_load(reinterpret_cast<const row_t*>(from));
#pragma unroll
          for (int i = 0; i < W / 4; i++) x.v[e][W / 4 * j + i] = w[i];
        }
      }
    }
    x.tv = tv;
    x.page = at.pv >= 0;
  }

  // takes the keys of a tile that are in [first, end) into the sums; `halves`: see add_values
  static __device__ __forceinline__ void add(const PagedAttnArgs& a, const v8 (&q)[KS], Data& x, int first, int end, bool halves, Partial<DV>& p) {
    const int tv = x.tv;
    // scores
    float s[8];
#pragma unroll
    for (int t = 0; t < 2; t++) {
      f32x4 acc{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < KS; i++) {
        if constexpr (F32) {
          const v8 f = __builtin_bit_cast(v8, x.k[t][i]);
#pragma unroll
          for (int e = 0; e < 4; e++) acc = MM<T>::dot(f[e], q[i][e], acc);
        } else if constexpr (QUANT) {
          u32x4 f;
#pragma unroll
          for (int w = 0; w < 4; w++) f[w] = MM<T>::from_fp8(x.k[t][i / 2][2 * (i % 2) + w / 2], w % 2);
          acc = MM<T>::dot(__builtin_bit_cast(v8, f), q[i], acc);
        } else {
          acc = MM<T>::dot(__builtin_bit_cast(v8, x.k[t][i]), q[i], acc);
        }
      }
#pragma unroll
      for (int e = 0; e < 4; e++) s[4 * t + e] = acc[e];
    }
#pragma unroll
    for (int e = 0; e < 8; e++) {
      if constexpr (QUANT) s[e] *= x.ks[e];
      s[e] *= a.scale;
    }
    if (a.cap > 0.f) {
      // (fast_tanh is off by 2^-23 of 1, which the cap multiplies: too much for fp32 where logits are small beside it)
#pragma unroll
      for (int e = 0; e < 8; e++) s[e] = a.cap * LOG2E * (F32 ? tanhf(s[e] / a.cap) : fast_tanh(s[e] / a.cap));
    }
    const bool whole = x.page && tv >= first && tv + 8 <= end;
    if (!__all(whole)) {
      // what lies in slots without a key takes no part, whatever it is: no score, and zeros for the products
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const bool in = x.page && tv + e >= first && tv + e < end;
        s[e] = in ? s[e] : -INFINITY;
#pragma unroll
        for (int i = 0; i < VB / 4; i++) x.v[e][i] = in ? x.v[e][i] : 0u;
        if constexpr (QUANT) x.vs[e] = in ? x.vs[e] : 0.f;
      }
    }
    float mx = s[0];
#pragma unroll
    for (int e = 1; e < 8; e++) mx = fmaxf(mx, s[e]);
    mx = groups_max(mx);
    int cx = p.c;
    if constexpr (RANGE) {
      float top = x.vs[0];
#pragma unroll
      for (int e = 1; e < 8; e++) top = fmaxf(top, x.vs[e]);
      top = groups_max(top);  // (the same in every lane)
      if (top > 0.f) cx = max(cx, __builtin_amdgcn_frexp_expf(top));
    }
    if (__any(mx > p.m + 8.f || (mx > -INFINITY && p.m == -INFINITY)) || (RANGE && cx > p.c)) {
      const float m = fmaxf(p.m, mx), shrink = m == -INFINITY ? 1.f : fast_exp2(p.m - m);
      const float so = RANGE ? __builtin_amdgcn_ldexpf(shrink, p.c - cx) : shrink;
      p.l *= shrink;
#pragma unroll
      for (int t = 0; t < C; t++) p.o[t] *= so;
      p.m = m;
      p.c = cx;
    }
    const float m = (p.m == -INFINITY ? 0.f : p.m) - UP;
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
      y[e] = fast_exp2(s[e] - m);
      p.l += y[e];
      if constexpr (RANGE) y[e] *= __builtin_amdgcn_ldexpf(x.vs[e], -p.c);
      else if constexpr (QUANT) y[e] *= x.vs[e];
    }
    if constexpr (F32) {
#pragma unroll
      for (int e = 0; e < 8; e++)
#pragma unroll
        for (int t = 0; t < C; t++) p.o[t] = MM<T>::dot(__uint_as_float(x.v[e][t]), y[e], p.o[t]);
    } else {
      add_values(x, y, halves, p);
    }
  }

  // A positive weight times an infinity is one, a rest of 0 times it is NaN: a wave whose sums are not finite takes its keys again with each
  // weight as two positive halves, for the columns where they are not (floored in float16, where a half might be 0).  To look for that
  // costs a call 0.1 to 0.25 us; sums of the rests by themselves, which need no second pass, cost 0.4 to 0.6 in another 32 registers.
  static __device__ __forceinline__ void add_values(const Data& x, const float (&y)[8], bool halves, Partial<DV>& p) {
    v8 w, rest;
    if (REST && halves) {
#pragma unroll
      for (int e = 0; e < 8; e++) w[e] = rest[e] = (T)(0.5f * (F16 && y[e] > 0.f ? fmaxf(y[e], 0x1p-20f) : y[e]));
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++) {
        w[e] = (T)y[e];
        rest[e] = (T)(y[e] - (float)w[e]);
      }
    }
    // values: column C r + t of the eight keys, paired from the rows as they came
    unsigned cols[8][C / 2];
#pragma unroll
    for (int e = 0; e < 8; e++)
#pragma unroll
      for (int i = 0; i < C / 2; i++) {
        if constexpr (QUANT) cols[e][i] = MM<T>::from_fp8(x.v[e][i / 2], i % 2);
        else cols[e][i] = x.v[e][i];
      }
#pragma unroll
    for (int t = 0; t < C; t++) {
      u32x4 f;
#pragma unroll
      for (int i = 0; i < 4; i++) f[i] = __builtin_amdgcn_perm(cols[2 * i + 1][t / 2], cols[2 * i][t / 2], t % 2 ? 0x07060302u : 0x05040100u);
      p.o[t] = MM<T>::dot(__builtin_bit_cast(v8, f), w, p.o[t]);
      p.o[t] = MM<T>::dot(__builtin_bit_cast(v8, f), rest, p.o[t]);
    }
  }
};

// One segment's sums over the waves that hold a part of it.  `n` parts: m, l at parts[i * stride + row], [.. + 16 + row],
// weighted sums at [.. + 32 + row * ROW + d].  Threads take four columns each.
template <typename T, int DV, int ROW>
__device__ __forceinline__ void join_parts(const PagedAttnArgs& a, int b, int h0, int rows, const float* parts, int64_t stride, int n, int threads, bool result,
                                           float* piece) {
  for (int i = threadIdx.x; i < rows * (DV / 4); i += threads) {
    const int row = i / (DV / 4), d = (i - row * (DV / 4)) * 4;
    float m = -INFINITY;
    for (int k = 0; k < n; k++) m = fmaxf(m, parts[k * stride + row]);
    const float base = m == -INFINITY ? 0.f : m;
    float l = 0.f;
    f32x4 o{0.f, 0.f, 0.f, 0.f};
    for (int k = 0; k < n; k++) {
      const float* p = parts + k * stride;
      const float f = fast_exp2(p[row] - base);
      l += f * p[16 + row];
      o += f * *reinterpret_cast<const f32x4*>(p + 32 + row * ROW + d);
    }
    if (result) {
      const float inv = l != 0.f ? 1.f / l : 0.f;
      store4(reinterpret_cast<T*>(a.out) + b * a.o_b + (h0 + row) * a.o_h + d, o * inv);
      if (d == 0 && a.lse) a.lse[(int64_t)b * a.Hq + h0 + row] = l != 0.f ? (m + log2f(l)) * LN2 : -INFINITY;
    } else {
      *reinterpret_cast<f32x4*>(piece + 32 + row * DV + d) = o;
      if (d == 0) {
        piece[row] = m;
        piece[16 + row] = l;
      }
    }
  }
}

// WHOLE: a workgroup per segment (few keys at most); otherwise equal shares of all units
template <typename T, bool QUANT, int DQK, int DV, int WAVES, int OCC, bool WHOLE>
__global__ __launch_bounds__(64 * WAVES, OCC) void paged_attn_kernel(PagedAttnArgs a) {
  typedef PagedTile<T, QUANT, DQK, DV> Tile;
  constexpr int ROW = DV + 4;  // (heads 4 banks apart)
  constexpr int UNIT = WAVES * PA_TILE;
  extern __shared__ float lds[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int segs = a.heads * a.blocks, rep = a.Hq / a.heads;
  int u, u1, b, at, per = 0, length;
  if constexpr (WHOLE) {
    b = blockIdx.x / segs;
    at = 0;  // (units are counted from the sequence's first)
    length = a.lengths[b];
  } else {
    const Share s = share_of<UNIT>(a, gridDim.x, blockIdx.x);
    per = s.per;
    u = blockIdx.x * per;
    u1 = min(u + per, s.total);
    b = s.b;
    at = s.at;
    length = s.length;
  }
  Keys keys(a, length);
  int units = keys.units(UNIT);
  if constexpr (WHOLE) {
    u = (blockIdx.x - b * segs) * units;
    u1 = u + units;
  } else {
    const int seg = (u - at) / units, begin = at + seg * units, kv = seg / a.blocks, block = seg - kv * a.blocks;
    if (threadIdx.x == 0) {
      const bool cut = u < u1 && begin < u && begin >= u - per;
      const int first = begin / per;
      reinterpret_cast<SegmentCut*>(a.ws)[blockIdx.x] = {cut ? min(16, rep - 16 * block) : 0, b, kv * rep + 16 * block, first, (begin + units - 1) / per, first * per < begin, {0, 0}};
    }
  }
  const int stride = 32 + a.rows * ROW;
  float* mine = lds + wave * stride;
  int piece = 2 * blockIdx.x;
  while (u < u1) {
    const int seg = (u - at) / units, step0 = u - at - seg * units, step1 = min(units, step0 + u1 - u);
    const int kv = seg / a.blocks, block = seg - kv * a.blocks, h0 = kv * rep + 16 * block, rows = min(16, rep - 16 * block);
    typename Tile::v8 q[Tile::KS];
    Tile::load_q(a, reinterpret_cast<const T*>(a.q) + b * a.q_b + (h0 + r) * a.q_h, r < rows, q);
    Partial<DV> p;
    const int stop = step1 == units ? keys.end : keys.base + step1 * UNIT;
    for (bool again = false;; again = true) {
      p.clear();
      int key0 = keys.base + (step0 * WAVES + wave) * PA_TILE;
      typename Tile::Where at_keys = Tile::find(a, b, key0);
      for (; key0 < stop; key0 += UNIT) {
        const typename Tile::Where now = at_keys;
        at_keys = Tile::find(a, b, key0 + UNIT);  // (on its way before the loads of this tile)
        typename Tile::Data x;
        Tile::load(a, now, kv, key0, x);
        Tile::add(a, q, x, keys.first, keys.end, again, p);
      }
      p.l = groups_sum(p.l);
      float finite = 0.f;  // not, where one of this lane's sums is not
      if (r < rows) {
        if (g == 0) {
          mine[r] = p.m - Tile::UP;  // (what the weights are relative to)
          mine[16 + r] = p.l;
        }
        float* o = mine + 32 + r * ROW + (DV / 4) * g;
        const float up = Tile::RANGE ? __builtin_amdgcn_ldexpf(1.f, p.c) : 1.f;
        constexpr int C = DV / 16;
#pragma unroll
        for (int e = 0; e < 4; e++)
#pragma unroll
          for (int t = 0; t < C; t += 4) {
            f32x4* out = reinterpret_cast<f32x4*>(o + e * C + t);
            f32x4 x{p.o[t][e], p.o[t + 1][e], p.o[t + 2][e], p.o[t + 3][e]};
            x *= up;
            if (again) {
              const f32x4 before = *out;
#pragma unroll
              for (int i = 0; i < 4; i++) x[i] = __builtin_isfinite(before[i]) ? before[i] : x[i];
            }
            *out = x;
            finite += x[0] + x[1] + (x[2] + x[3]);
          }
      }
      if (!Tile::REST || again || __all(__builtin_isfinite(finite))) break;
    }
    __syncthreads();
    const bool result = step0 == 0 && step1 == units;
    join_parts<T, DV, ROW>(a, b, h0, rows, lds, stride, WAVES, 64 * WAVES, result, pa_piece(a, gridDim.x, piece, DV));
    piece = 2 * blockIdx.x + 1;
    u += step1 - step0;
    if (u < u1) {
      __syncthreads();
      if (u - at == units * segs) {
        at = u;
        keys = Keys(a, a.lengths[++b]);
        units = keys.units(UNIT);
      }
    }
  }
}

// Workgroup (w, y) adds up rows of the cut that workgroup w + 1 named: DV / 4 lanes for every SETS-th piece of a row, then the sets
// through LDS.
constexpr int PA_JOIN = 256;
template <typename T, int DV, int SETS>
__global__ __launch_bounds__(PA_JOIN) void paged_attn_join_kernel(PagedAttnArgs a, int groups) {
  constexpr int LANES = DV / 4, ROWS = PA_JOIN / (LANES * SETS);
  __shared__ float lm[ROWS][SETS], ll[ROWS][SETS];
  __shared__ f32x4 lo[ROWS][SETS][LANES];
  const SegmentCut s = reinterpret_cast<const SegmentCut*>(a.ws)[blockIdx.x + 1];
  const int lane = threadIdx.x % LANES, set = threadIdx.x / LANES % SETS, at = threadIdx.x / (LANES * SETS), row = blockIdx.y * ROWS + at;
  if (blockIdx.y * ROWS >= (unsigned)s.rows) return;
  const bool mine = row < s.rows;
  float m = -INFINITY, l = 0.f;
  f32x4 o{0.f, 0.f, 0.f, 0.f};
  for (int k = s.first + set; k <= s.last && mine; k += SETS) {
    const float* p = pa_piece(a, groups, 2 * k + (k == s.first ? s.lead : 0), DV);
    const float pm = p[row], pl = p[16 + row];
    const f32x4 po = *reinterpret_cast<const f32x4*>(p + 32 + row * DV + 4 * lane);
    const float top = fmaxf(m, pm), base = top == -INFINITY ? 0.f : top, f = fast_exp2(m - base), g = fast_exp2(pm - base);
    l = l * f + pl * g;
    o = o * f + po * g;
    m = top;
  }
  if constexpr (SETS > 1) {
    if (lane == 0) {
      lm[at][set] = m;
      ll[at][set] = l;
    }
    lo[at][set][lane] = o;
    __syncthreads();
    if (set) return;
    for (int k = 1; k < SETS; k++) m = fmaxf(m, lm[at][k]);
    const float base = m == -INFINITY ? 0.f : m;
    l = 0.f;
    o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < SETS; k++) {
      const float f = fast_exp2(lm[at][k] - base);
      l += f * ll[at][k];
      o += f * lo[at][k][lane];
    }
  }
  if (!mine) return;
  const int h = s.h0 + row;
  const float inv = l != 0.f ? 1.f / l : 0.f;
  store4(reinterpret_cast<T*>(a.out) + s.b * a.o_b + h * a.o_h + 4 * lane, o * inv);
  if (lane == 0 && a.lse) a.lse[(int64_t)s.b * a.Hq + h] = l != 0.f ? (m + log2f(l)) * LN2 : -INFINITY;
}

// ---- host --------------------------------------------------------------------------------------
// Workgroups of a call, and their waves.  Where the table has room for no more than PA_WHOLE keys a sequence, a
// workgroup (of more waves) takes a whole segment, no piece is left over and no second launch follows.
//   us, one CU's waves 4 : 8, up to 512 keys: one sequence of 461 keys and 8 kv heads 8.95 : 8.83, 16 of 20 to 300 9.8 : 9.0,
//   64 of 20 to 300 13.1 : 15.2: eight waves where the segments do not fill the CUs, four where they do.
inline bool paged_tiles(const tp_kv_cache* c) { return c->dtype != TP_F32 || c->k_dim == c->v_dim; }
// Shares: workgroups of four waves, as many as are resident.  us, waves a workgroup x workgroups, at 131072 keys, 128 long sequences in
// bfloat16, in 8 bits: 8 x 256 90.6, 268, 186; 8 x 512 96.9, 275, 191; 4 x 512 93.5, 263, 177; 4 x 768 (three waves per SIMD) 96.5, 261,
// 157; 2 x 1024 97.5, 263, 175; 4 x 1024 128, 349, 214 (128 registers).
struct PagedPlan {
  bool whole;
  int waves, groups;
};
constexpr int PA_WAVES = 4, PA_WHOLE_FEW = 8, PA_CUS = 256, PA_GROUPS = 512, PA_GROUPS_8BIT = 768, PA_WHOLE = 512;
inline PagedPlan paged_plan(const tp_kv_cache* c, int B, int Hq) {
  const int64_t segs = (int64_t)B * c->heads * ((Hq / c->heads + 15) / 16), keys = (int64_t)c->table_width * c->page_size;
  if (keys <= PA_WHOLE) return {true, segs <= PA_CUS ? PA_WHOLE_FEW : PA_WAVES, (int)segs};
  const int64_t units = (keys + PA_TILE) / (PA_WAVES * PA_TILE) + 1, most = c->dtype == TP_FP8 ? PA_GROUPS_8BIT : PA_GROUPS;
  return {false, PA_WAVES, (int)std::min(most, segs * units)};
}

template <typename T, bool QUANT, int DQK, int DV>
int paged_launch(const PagedAttnArgs& a, const PagedPlan& plan, hipStream_t st) {
  // waves per SIMD; 8-bit keys of 192 spill a dozen registers at three, which costs less than a third wave gives (54.2 : 51.8 us)
  constexpr int OCC = QUANT ? 3 : 2;
  const int lds = plan.waves * (32 + a.rows * (DV + 4)) * 4;
  const auto kern = !plan.whole                  ? paged_attn_kernel<T, QUANT, DQK, DV, PA_WAVES, OCC, false>
                    : plan.waves == PA_WHOLE_FEW ? paged_attn_kernel<T, QUANT, DQK, DV, PA_WHOLE_FEW, 2, true>
                                                 : paged_attn_kernel<T, QUANT, DQK, DV, PA_WAVES, OCC, true>;
  if (lds > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
    TP_REQUIRE(e == hipSuccess, TP_ERR_LAUNCH, "tp_paged_attn: hipFuncSetAttribute failed: %s", hipGetErrorString(e));
  }
  kern<<<plan.groups, 64 * plan.waves, lds, st>>>(a);
  if (!plan.whole && plan.groups > 1) {
    const int per_row = PA_JOIN / (DV / 4);
    // many workgroups to a segment: eight threads share out the pieces of four columns
    if (plan.groups > 4 * a.B * a.heads * a.blocks)
      paged_attn_join_kernel<T, DV, 8><<<dim3(plan.groups - 1, (a.rows * 8 + per_row - 1) / per_row), PA_JOIN, 0, st>>>(a, plan.groups);
    else
      paged_attn_join_kernel<T, DV, 1><<<dim3(plan.groups - 1, (a.rows + per_row - 1) / per_row), PA_JOIN, 0, st>>>(a, plan.groups);
  }
  return check_launch("tp_paged_attn");
}

}  // namespace tp

extern "C" size_t tp_paged_attn_workspace_bytes(const tp_kv_cache* c, int B, int Hq, int dtype) {
  using namespace tp;
  if (check_cache(c, dtype, B, "tp_paged_attn_workspace_bytes") != TP_OK || Hq < 1 || Hq % c->heads || !paged_tiles(c)) return 0;
  const PagedPlan plan = paged_plan(c, B, Hq);
  return plan.whole ? 0 : plan.groups * (sizeof(SegmentCut) + sizeof(float) * 2 * pa_piece_floats(c->v_dim));
}

extern "C" int tp_paged_attn(const tp_kv_cache* c, const void* q, const int32_t* lengths, void* out, float* lse, void* ws, int B, int Hq,
                             const int64_t* q_strides, const int64_t* o_strides, float sm_scale, int window_left, float soft_cap, int dtype,
                             void* stream) {
  using namespace tp;
  if (int rc = check_cache(c, dtype, B, "tp_paged_attn")) return rc;
  TP_REQUIRE(q && lengths && out && q_strides && o_strides, TP_ERR_BAD_ARG, "tp_paged_attn: null pointer");
  TP_REQUIRE(Hq >= 1 && Hq % c->heads == 0, TP_ERR_BAD_ARG, "tp_paged_attn: %d query heads are not a multiple of %d kv heads", Hq, c->heads);
  TP_REQUIRE(sm_scale > 0.f && soft_cap >= 0.f, TP_ERR_BAD_ARG, "tp_paged_attn: sm_scale must be positive, soft_cap not negative");
  TP_REQUIRE((c->k_dim == c->v_dim && (c->k_dim == 64 || c->k_dim == 128)) || (c->k_dim == 192 && c->v_dim == 128), TP_ERR_UNSUPPORTED,
             "tp_paged_attn: head dims (qk=%d, v=%d) not built; supported: (64, 64), (128, 128), (192, 128)", c->k_dim, c->v_dim);
  const int e = elem_size(dtype);
  TP_REQUIRE(aligned16(q) && aligned16(out), TP_ERR_BAD_ARG, "tp_paged_attn: q and out must start at 16-byte addresses");
  for (int i = 0; i < 2; i++)
    TP_REQUIRE(q_strides[i] * e % 16 == 0 && o_strides[i] * e % 16 == 0, TP_ERR_BAD_ARG, "tp_paged_attn: strides must keep rows 16-byte aligned");
  TP_REQUIRE((int64_t)B * Hq < (1ll << 24), TP_ERR_UNSUPPORTED, "tp_paged_attn: too many rows");
  TP_REQUIRE((int64_t)B * c->heads * ((Hq / c->heads + 15) / 16) * (((int64_t)c->table_width * c->page_size) / (PA_WAVES * PA_TILE) + 2) < (1ll << 30),
             TP_ERR_UNSUPPORTED, "tp_paged_attn: the table covers too many keys");
  const int rep = Hq / c->heads;
  const PagedAttnArgs a{rows_of(c, false), rows_of(c, true), table_of(c), q, lengths, out, lse, (float*)ws, q_strides[0], q_strides[1], o_strides[0],
                        o_strides[1], B, Hq, c->heads, (rep + 15) / 16, std::min(rep, 16), soft_cap > 0.f ? sm_scale : sm_scale * LOG2E, soft_cap,
                        window_left};
  const hipStream_t st = (hipStream_t)stream;
  if (!paged_tiles(c)) {
    paged_attn_rows_kernel<<<B * Hq, PA_KEYS, 0, st>>>(a);
    return check_launch("tp_paged_attn");
  }
  const PagedPlan plan = paged_plan(c, B, Hq);
  TP_REQUIRE(plan.whole || (ws && aligned16(ws)), TP_ERR_BAD_ARG, "tp_paged_attn: the workspace must be there and start at a 16-byte address");
  int rc = TP_OK;
  kv_dispatch(dtype, c->dtype == TP_FP8, [&](auto t, auto quant) {
    typedef decltype(t) T;
    constexpr bool Q = quant.value;
    if (c->k_dim == 64) rc = paged_launch<T, Q, 64, 64>(a, plan, st);
    else if (c->k_dim == 128) rc = paged_launch<T, Q, 128, 128>(a, plan, st);
    else if constexpr (!std::is_same<T, float>::value) rc = paged_launch<T, Q, 192, 128>(a, plan, st);
  });
  return rc;
}
