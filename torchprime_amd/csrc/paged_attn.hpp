// Attention of one new token per sequence over the paged cache (kv_cache.hpp):
//
//   s_j = cap(scale * q . k_j),   out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),   m = max_j s_j
//
// in one pass over the keys, with a running maximum, sum and weighted sum of values (Milakov and Gimelshein, "Online normalizer
// calculation for softmax", 2018).
#pragma once
#include "kv_cache.hpp"

namespace tp {

constexpr float ATT_LOG2E = 1.4426950408889634f, ATT_LN2 = 0.6931471805599453f;

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
  float scale;       // log2(e) * sm_scale; without log2(e) where soft_cap is set
  float cap;         // soft_cap, 0: none
  int window;        // keys before the newest that are seen, negative: all
};

// ------------------------------------------------------------------------------------------------
// one workgroup per (sequence, query head): a thread takes a key of every 256, then a few columns of the values
// ------------------------------------------------------------------------------------------------
constexpr int PA_KEYS = 256;
template <typename T, bool QUANT>
__global__ __launch_bounds__(PA_KEYS) void paged_attn_rows_kernel(PagedAttnArgs a) {
  __shared__ float q[512], p[PA_KEYS], part[4], acc_lds[PA_KEYS * 8];
  __shared__ int64_t at_v[PA_KEYS];
  const int b = blockIdx.x / a.Hq, h = blockIdx.x - b * a.Hq, kv = h / (a.Hq / a.heads), tid = threadIdx.x;
  const T* qp = reinterpret_cast<const T*>(a.q) + b * a.q_b + h * a.q_h;
  for (int i = tid; i < a.k.dim; i += PA_KEYS) q[i] = Elem<T>::to_f(qp[i]);
  const int n = min(a.lengths[b], a.table.width << a.table.page_shift);
  const int first = a.window >= 0 ? max(0, n - 1 - a.window) : 0;
  const int lane = tid & (a.v.group - 1), sub = tid / a.v.group, subs = PA_KEYS / a.v.group;
  float m = -INFINITY, l = 0.f, acc[8] = {};
  __syncthreads();
  for (int j0 = first; j0 < n; j0 += PA_KEYS) {
    const int j = j0 + tid, page = j < n ? a.table.page_of(b, j) : -1, slot = j & ((1 << a.table.page_shift) - 1);
    float s = -INFINITY, vs = 1.f;
    if (page >= 0) {
      const int64_t at = page * a.k.page + kv * a.k.head + slot * a.k.slot;
      s = 0.f;
      for (int d = 0; d < a.k.dim; d += 8) {
        float x[8];
        if constexpr (QUANT) unpack_fp8(*reinterpret_cast<const u32x2*>(a.k.base + at + d), x);
        else load_f<T, 8>(reinterpret_cast<const T*>(a.k.base) + at + d, x);
#pragma unroll
        for (int e = 0; e < 8; e++) s += x[e] * q[d + e];
      }
      if constexpr (QUANT) {
        const int64_t row = (((int64_t)page * a.heads + kv) << a.table.page_shift) + slot;
        s *= a.k.scale[row];
        vs = a.v.scale[row];
      }
      s *= a.scale;
      if (a.cap > 0.f) s = a.cap * ATT_LOG2E * tanhf(s / a.cap);
    }
    float mx = wave_max(s);
    if ((tid & 63) == 0) part[tid >> 6] = mx;
    __syncthreads();
    mx = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
    const float m_new = fmaxf(m, mx), base = m_new == -INFINITY ? 0.f : m_new;
    const float shrink = exp2f(m - base);
    const float w = page >= 0 ? exp2f(s - base) : 0.f;
    l = l * shrink + w;  // this thread's keys
    p[tid] = w * vs;
    at_v[tid] = page >= 0 ? page * a.v.page + kv * a.v.head + slot * a.v.slot : -1;
    m = m_new;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 8; e++) acc[e] *= shrink;
    if (lane * 8 < a.v.dim) {
      for (int i = sub; i < PA_KEYS && j0 + i < n; i += subs) {
        if (at_v[i] < 0) continue;  // (not loaded: what lies there takes no part, whatever it is)
        float x[8];
        if constexpr (QUANT) unpack_fp8(*reinterpret_cast<const u32x2*>(a.v.base + at_v[i] + lane * 8), x);
        else load_f<T, 8>(reinterpret_cast<const T*>(a.v.base) + at_v[i] + lane * 8, x);
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
    reinterpret_cast<T*>(a.out)[b * a.o_b + h * a.o_h + d] = Elem<T>::from_f(l != 0.f ? o / l : 0.f);
  }
  if (tid == 0 && a.lse) a.lse[(int64_t)b * a.Hq + h] = l != 0.f ? (m + log2f(l)) * ATT_LN2 : -INFINITY;
}

}  // namespace tp

extern "C" size_t tp_paged_attn_workspace_bytes(const tp_kv_cache* c, int B, int Hq, int dtype) { return 0; }

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
  PagedAttnArgs a{rows_of(c, false), rows_of(c, true), table_of(c), q, lengths, out, lse, (float*)ws, q_strides[0], q_strides[1], o_strides[0],
                  o_strides[1], B, Hq, c->heads, soft_cap > 0.f ? sm_scale : sm_scale * ATT_LOG2E, soft_cap, window_left};
  kv_dispatch(dtype, c->dtype == TP_FP8, [&](auto t, auto quant) {
    paged_attn_rows_kernel<decltype(t), quant.value><<<B * Hq, PA_KEYS, 0, (hipStream_t)stream>>>(a);
  });
  return check_launch("tp_paged_attn");
}
