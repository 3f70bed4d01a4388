// The paged key-value cache: where a cached token lies, and the two kernels that move whole rows (one head of one token)
// into the pages and out of them again.
//
//   position t of sequence b  ->  page table[b][t / page_size], slot t % page_size
//
// An 8-bit cache (float8_e4m3fn) has one fp32 scale per row:  a = max |x|,  scale = a / 448,  stored = e4m3(x * (448 / a)),
// each operation rounded once in fp32, so that the stored values can be reproduced bit for bit.  Rows whose a is below 2^-100
// (448 / a would leave fp32's range at 2^-119) are stored as zeros of scale 0; a row with an infinity or a NaN gets the scale NaN
// and reads back as NaN, whole, and no other row does.
//
// Both kernels stream: each byte is touched once and nothing is kept, so what bounds them is HBM (large calls) or the launch and
// three dependent loads: position, table entry, row (small ones).  A lane moves 8 elements, or stores 16 of
// an 8-bit cache where the head dims allow (4 prompts of 8192 tokens, 8 heads of 128: 51 : 43 us; reading back is better with 8, whose
// stores lie side by side, 43 : 51); a row is a group of 4 to 64 lanes of one wave, where the row's maximum is taken with lane exchanges.
// Measured, 8 heads of 128, bfloat16: 4 prompts of 8192 stored 46 us = 5.9 TB/s, read back 5.9 TB/s; in 8 bits 44 us (4.7 TB/s) and
// 43 us (4.7 TB/s: pieces of 8 bytes on the 8-bit side); 4 of 4096 in fp32 51 us (5.3 TB/s) and 53 us (5.1 TB/s); the tokens of one step of
// 64 sequences 2.5 us, which is what an empty launch takes.
#pragma once
#include "common.hpp"

namespace tp {

// One 16-bit, 32-bit or 8-bit tensor of the cache: (page, head, slot) strides in elements, dim contiguous
struct PageRows {
  char* base;
  float* scale;  // (page, head, slot), contiguous; null where the values are stored as they are
  int64_t page, head, slot;
  int dim, group, shift;  // lanes per row, a power of two, and its logarithm
};
struct PageTable {
  const int32_t* ids;
  int64_t stride;
  int width, pages, page_shift;
  // the page that holds position t of sequence b, or -1 where t is outside the table or the entry names no page
  __device__ __forceinline__ int page_of(int b, int t) const {
    const unsigned i = (unsigned)t >> page_shift;
    if (t < 0 || i >= (unsigned)width) return -1;
    const int id = ids[b * stride + i];
    return (unsigned)id < (unsigned)pages ? id : -1;
  }
};

template <int N> using bytes_t = unsigned __attribute__((ext_vector_type(N / 4)));  // N bytes
template <int N>
__device__ __forceinline__ bytes_t<N> pack_fp8(const float (&x)[N]) {
  bytes_t<N> r;
#pragma unroll
  for (int i = 0; i < N / 4; i++) {
    const int w = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i], x[4 * i + 1], 0, false);
    r[i] = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i + 2], x[4 * i + 3], w, true);
  }
  return r;
}
template <int N>
__device__ __forceinline__ void unpack_fp8(const bytes_t<N> w, float (&x)[N]) {
#pragma unroll
  for (int i = 0; i < N / 4; i++) {
    const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], true);
    x[4 * i] = lo[0];
    x[4 * i + 1] = lo[1];
    x[4 * i + 2] = hi[0];
    x[4 * i + 3] = hi[1];
  }
}

constexpr int KV_THREADS = 256;
constexpr float FP8_MAX = 448.f, FP8_TINY = 0x1p-100f;

struct KvRowsIn {  // the new tokens: (batch, head, token) strides
  const char* base;
  int64_t b, h, s;
};

// Row r of a launch is (b, s, h) with the head fastest: the order of the memory that the projections write.  A workgroup takes
// ROWS times as many rows as its lanes hold; all its loads are on their way before a page is known.
template <typename T, bool QUANT, int N, int ROWS>
__device__ __forceinline__ void kv_write_rows(const PageRows& c, const KvRowsIn& in, const PageTable& tab, const int32_t* positions,
                                              const int32_t* counts, unsigned block, unsigned rows, unsigned S, unsigned H) {
  const int lane = threadIdx.x & (c.group - 1), per = KV_THREADS >> c.shift;
  const unsigned r0 = block * (per * ROWS) + (threadIdx.x >> c.shift);
  const bool mine = lane * N < c.dim;
  Raw<T, N> raw[ROWS];
  int b[ROWS], h[ROWS], t[ROWS], page[ROWS];
#pragma unroll
  for (int u = 0; u < ROWS; u++) {
    const unsigned r = r0 + u * per, bs = r / H, s = bs % S;
    b[u] = bs / S;
    h[u] = r - bs * H;
    t[u] = -1;
    if (r < rows) {
      if (mine) raw[u] = load_raw_nt<T, N>(reinterpret_cast<const T*>(in.base) + b[u] * in.b + h[u] * in.h + s * in.s + lane * N);
      const int64_t at = (int64_t)positions[b[u]] + s;
      if (at < 0x7fffffff && !(counts && (int)s >= counts[b[u]])) t[u] = (int)at;
    }
  }
#pragma unroll
  for (int u = 0; u < ROWS; u++) page[u] = tab.page_of(b[u], t[u]);
#pragma unroll
  for (int u = 0; u < ROWS; u++) {
    if (page[u] < 0) continue;  // (a row's lanes together)
    const int slot = t[u] & ((1 << tab.page_shift) - 1);
    const int64_t dst = page[u] * c.page + h[u] * c.head + slot * c.slot + lane * N;
    if constexpr (!QUANT) {
      if (mine) {
        u32x4* d = reinterpret_cast<u32x4*>(reinterpret_cast<T*>(c.base) + dst);
#pragma unroll
        for (int i = 0; i < (int)(N * sizeof(T) / 16); i++) __builtin_nontemporal_store(raw[u].q[i], d + i);
      }
    } else {
      float x[N] = {};
      if (mine) unpack_f<T, N>(raw[u], x);
      // the largest magnitude by its bits: a NaN is above an infinity, and that above every number
      unsigned top = 0;
#pragma unroll
      for (int e = 0; e < N; e++) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
      for (int o = c.group / 2; o > 0; o >>= 1) top = max(top, (unsigned)__shfl_xor((int)top, o, 64));
      const float a = __uint_as_float(top);
      const bool finite = top < 0x7f800000u, some = finite && a >= FP8_TINY;
      const float back = some ? FP8_MAX / a : 0.f;
#pragma unroll
      for (int e = 0; e < N; e++) x[e] = finite ? x[e] * back : 0.f;
      if (mine) {
        __builtin_nontemporal_store(pack_fp8(x), reinterpret_cast<bytes_t<N>*>(c.base + dst));
        if (lane == 0)
          c.scale[(((int64_t)page[u] * H + h[u]) << tab.page_shift) + slot] = !finite ? __uint_as_float(0x7fc00000u) : some ? a / FP8_MAX : 0.f;
      }
    }
  }
}

// blocks [0, k_blocks) take the keys, the others the values
template <typename T, bool QUANT, int N, int ROWS>
__global__ __launch_bounds__(KV_THREADS) void kv_write_kernel(PageRows ck, PageRows cv, KvRowsIn k, KvRowsIn v, PageTable tab,
                                                              const int32_t* __restrict__ positions, const int32_t* __restrict__ counts,
                                                              unsigned rows, unsigned S, unsigned H, unsigned k_blocks) {
  if (blockIdx.x < k_blocks) kv_write_rows<T, QUANT, N, ROWS>(ck, k, tab, positions, counts, blockIdx.x, rows, S, H);
  else kv_write_rows<T, QUANT, N, ROWS>(cv, v, tab, positions, counts, blockIdx.x - k_blocks, rows, S, H);
}

// Row r of a launch is (b, h, t) with the position fastest: whole pages are read and whole stretches written.
template <typename T, bool QUANT, int N, int ROWS>
__device__ __forceinline__ void kv_read_rows(const PageRows& c, const KvRowsIn& out, const PageTable& tab, const int32_t* lengths,
                                             unsigned block, unsigned rows, unsigned L, unsigned H) {
  const int lane = threadIdx.x & (c.group - 1), per = KV_THREADS >> c.shift;
  const unsigned r0 = block * (per * ROWS) + (threadIdx.x >> c.shift);
  if (lane * N >= c.dim) return;
  T* dst[ROWS];
  int b[ROWS], h[ROWS], t[ROWS], page[ROWS];
#pragma unroll
  for (int u = 0; u < ROWS; u++) {
    const unsigned r = r0 + u * per, bh = r / L;
    t[u] = r - bh * L;
    b[u] = bh / H;
    h[u] = bh - b[u] * H;
    page[u] = -1;
    dst[u] = reinterpret_cast<T*>(const_cast<char*>(out.base)) + b[u] * out.b + h[u] * out.h + t[u] * out.s + lane * N;
    if (r < rows) {
      const int length = lengths[b[u]];
      page[u] = tab.page_of(b[u], t[u]);  // (not behind the length: the two loads run side by side)
      if (t[u] >= length) page[u] = -1;
    }
  }
  Raw<T, N> raw[ROWS];
  bytes_t<N> bytes[ROWS];
  float scale[ROWS];
#pragma unroll
  for (int u = 0; u < ROWS; u++) {
    raw[u] = {};
    bytes[u] = {};
    scale[u] = 0.f;
    if (page[u] < 0) continue;
    const int slot = t[u] & ((1 << tab.page_shift) - 1);
    const int64_t src = page[u] * c.page + h[u] * c.head + slot * c.slot + lane * N;
    if constexpr (QUANT) {
      bytes[u] = __builtin_nontemporal_load(reinterpret_cast<const bytes_t<N>*>(c.base + src));
      scale[u] = c.scale[(((int64_t)page[u] * H + h[u]) << tab.page_shift) + slot];
    } else {
      raw[u] = load_raw_nt<T, N>(reinterpret_cast<const T*>(c.base) + src);
    }
  }
#pragma unroll
  for (int u = 0; u < ROWS; u++) {
    if (r0 + u * per >= rows) break;
    if constexpr (QUANT) {
      float x[N];
      unpack_fp8<N>(bytes[u], x);
#pragma unroll
      for (int e = 0; e < N; e++) {
        x[e] = page[u] >= 0 ? x[e] * scale[u] : 0.f;
        asm("" : "+v"(x[e]));  // rounded here: float16's mixed product would round the exact one
      }
      store_f_nt<T, N>(dst[u], x);
    } else {
      u32x4* d = reinterpret_cast<u32x4*>(dst[u]);
#pragma unroll
      for (int i = 0; i < (int)(N * sizeof(T) / 16); i++) __builtin_nontemporal_store(raw[u].q[i], d + i);
    }
  }
}

template <typename T, bool QUANT, int N, int ROWS>
__global__ __launch_bounds__(KV_THREADS) void kv_read_kernel(PageRows ck, PageRows cv, KvRowsIn k, KvRowsIn v, PageTable tab,
                                                             const int32_t* __restrict__ lengths, unsigned rows, unsigned L, unsigned H,
                                                             unsigned k_blocks) {
  if (blockIdx.x < k_blocks) kv_read_rows<T, QUANT, N, ROWS>(ck, k, tab, lengths, blockIdx.x, rows, L, H);
  else kv_read_rows<T, QUANT, N, ROWS>(cv, v, tab, lengths, blockIdx.x - k_blocks, rows, L, H);
}

// ---- host --------------------------------------------------------------------------------------
inline int elem_size(int dtype) { return dtype == TP_F32 ? 4 : dtype == TP_FP8 ? 1 : 2; }

// 16 bytes of an 8-bit row per lane
inline bool wide_lanes(const tp_kv_cache* c) { return c->dtype == TP_FP8 && c->k_dim % 16 == 0 && c->v_dim % 16 == 0; }

// what every entry point asks of a cache; `dtype` is the type of the tensors that go in or come out
inline int check_cache(const tp_kv_cache* c, int dtype, int B, const char* who) {
  TP_REQUIRE(c && c->k && c->v && c->table, TP_ERR_BAD_ARG, "%s: null pointer", who);
  TP_REQUIRE(dtype >= TP_BF16 && dtype <= TP_F32, TP_ERR_UNSUPPORTED, "%s: unsupported dtype code %d", who, dtype);
  TP_REQUIRE(c->dtype == dtype || (c->dtype == TP_FP8 && dtype != TP_F32), TP_ERR_UNSUPPORTED,
             "%s: a cache of dtype code %d does not go with tensors of code %d", who, c->dtype, dtype);
  TP_REQUIRE(B >= 1 && c->pages >= 1 && c->heads >= 1 && c->table_width >= 1 && c->table_stride >= 0, TP_ERR_BAD_ARG, "%s: sizes must be positive", who);
  TP_REQUIRE(c->page_size >= 8 && (c->page_size & (c->page_size - 1)) == 0, TP_ERR_UNSUPPORTED, "%s: page_size %d is not a power of two from 8 up", who, c->page_size);
  TP_REQUIRE((int64_t)c->table_width * c->page_size <= 1 << 30, TP_ERR_UNSUPPORTED, "%s: the table covers more than 2^30 positions", who);
  for (int d : {c->k_dim, c->v_dim})
    TP_REQUIRE(d >= 8 && d <= 512 && d % 8 == 0, TP_ERR_UNSUPPORTED, "%s: head dim %d is not a multiple of 8 up to 512", who, d);
  const int e = elem_size(c->dtype), step = c->dtype == TP_FP8 && !wide_lanes(c) ? 8 : 16;
  TP_REQUIRE((((uintptr_t)c->k | (uintptr_t)c->v) & 15) == 0, TP_ERR_BAD_ARG, "%s: the cache must start at 16-byte addresses", who);
  for (int i = 0; i < 3; i++)
    TP_REQUIRE(c->k_strides[i] >= 0 && c->v_strides[i] >= 0 && c->k_strides[i] * e % step == 0 && c->v_strides[i] * e % step == 0, TP_ERR_BAD_ARG,
               "%s: strides of the cache must keep rows %d-byte aligned", who, step);
  TP_REQUIRE((((uintptr_t)c->k_scale | (uintptr_t)c->v_scale) & 15) == 0, TP_ERR_BAD_ARG, "%s: the scales must start at 16-byte addresses", who);
  TP_REQUIRE((c->dtype == TP_FP8) == (c->k_scale != nullptr) && (c->dtype == TP_FP8) == (c->v_scale != nullptr), TP_ERR_BAD_ARG,
             "%s: an 8-bit cache needs k_scale and v_scale, another cache has none", who);
  return TP_OK;
}
inline int log2_of(int n) { int s = 0; while ((1 << s) < n) s++; return s; }
inline PageTable table_of(const tp_kv_cache* c) { return {c->table, c->table_stride, c->table_width, c->pages, log2_of(c->page_size)}; }
// (n: elements of a lane)
inline PageRows rows_of(const tp_kv_cache* c, bool values, int n = 8) {
  const int64_t* s = values ? c->v_strides : c->k_strides;
  const int dim = values ? c->v_dim : c->k_dim;
  int group = 4, shift = 2;
  for (; group * n < dim; group *= 2) shift++;
  return {(char*)(values ? c->v : c->k), values ? c->v_scale : c->k_scale, s[0], s[1], s[2], dim, group, shift};
}
inline int check_rows(const void* k, const void* v, const int64_t* ks, const int64_t* vs, int dtype, const char* who) {
  TP_REQUIRE(k && v && ks && vs, TP_ERR_BAD_ARG, "%s: null pointer", who);
  TP_REQUIRE(aligned16(k) && aligned16(v), TP_ERR_BAD_ARG, "%s: k and v must start at 16-byte addresses", who);
  for (int i = 0; i < 3; i++)
    TP_REQUIRE(ks[i] * elem_size(dtype) % 16 == 0 && vs[i] * elem_size(dtype) % 16 == 0, TP_ERR_BAD_ARG, "%s: strides must keep rows 16-byte aligned", who);
  return TP_OK;
}

// f(T{}, std::bool_constant<QUANT>{}) for the types of a call that check_cache has passed
template <typename F>
void kv_dispatch(int dtype, bool quant, F&& f) {
  if (dtype == TP_F32) f(float{}, std::false_type{});
  else if (dtype == TP_BF16) { if (quant) f(bf16_t{}, std::true_type{}); else f(bf16_t{}, std::false_type{}); }
  else { if (quant) f(f16_t{}, std::true_type{}); else f(f16_t{}, std::false_type{}); }
}

// rows a lane: one where they are few, two for more bytes on their way.  64 rows of 8 heads 2.5 : 2.9 us, 4 x 8192 49.1 : 46.2
inline int kv_rows(int64_t rows) { return rows <= 16384 ? 1 : 2; }

// workgroups of a launch over `rows` rows of both tensors: those of the keys, and all of them (fewer than 2^24: a launch has at most
// 2^32 lanes)
inline bool kv_blocks(const PageRows& ck, const PageRows& cv, int64_t rows, int per_lane, unsigned& k_blocks, unsigned& all) {
  const auto blocks = [&](const PageRows& c) { const int64_t per = (KV_THREADS >> c.shift) * per_lane; return (rows + per - 1) / per; };
  k_blocks = (unsigned)blocks(ck);
  all = (unsigned)(blocks(ck) + blocks(cv));
  return rows < (1ll << 31) && blocks(ck) + blocks(cv) < (1ll << 32) / KV_THREADS;
}

}  // namespace tp

extern "C" int tp_kv_cache_write(const tp_kv_cache* c, const void* k, const void* v, const int32_t* positions, const int32_t* counts, int B, int S,
                                 const int64_t* k_strides, const int64_t* v_strides, int dtype, void* stream) {
  using namespace tp;
  if (int rc = check_cache(c, dtype, B, "tp_kv_cache_write")) return rc;
  if (int rc = check_rows(k, v, k_strides, v_strides, dtype, "tp_kv_cache_write")) return rc;
  TP_REQUIRE(positions && S >= 1, TP_ERR_BAD_ARG, "tp_kv_cache_write: null positions or no tokens");
  const int n = wide_lanes(c) ? 16 : 8;
  const PageRows ck = rows_of(c, false, n), cv = rows_of(c, true, n);
  const int64_t rows = (int64_t)B * S * c->heads;
  unsigned k_blocks, blocks;
  const int per_lane = kv_rows(rows);
  TP_REQUIRE(kv_blocks(ck, cv, rows, per_lane, k_blocks, blocks), TP_ERR_UNSUPPORTED, "tp_kv_cache_write: too many rows");
  const KvRowsIn ki{(const char*)k, k_strides[0], k_strides[1], k_strides[2]}, vi{(const char*)v, v_strides[0], v_strides[1], v_strides[2]};
  kv_dispatch(dtype, c->dtype == TP_FP8, [&](auto t, auto quant) {
    typedef decltype(t) T;
    constexpr int WIDE = quant.value ? 16 : 8;
    const auto kern = n == 8 ? (per_lane == 1 ? kv_write_kernel<T, quant.value, 8, 1> : kv_write_kernel<T, quant.value, 8, 2>)
                             : (per_lane == 1 ? kv_write_kernel<T, quant.value, WIDE, 1> : kv_write_kernel<T, quant.value, WIDE, 2>);
    kern<<<blocks, KV_THREADS, 0, (hipStream_t)stream>>>(ck, cv, ki, vi, table_of(c), positions, counts, (unsigned)rows, S, c->heads, k_blocks);
  });
  return check_launch("tp_kv_cache_write");
}

extern "C" int tp_kv_cache_read(const tp_kv_cache* c, const int32_t* lengths, void* k, void* v, int B, int L, const int64_t* k_strides,
                                const int64_t* v_strides, int dtype, void* stream) {
  using namespace tp;
  if (int rc = check_cache(c, dtype, B, "tp_kv_cache_read")) return rc;
  if (int rc = check_rows(k, v, k_strides, v_strides, dtype, "tp_kv_cache_read")) return rc;
  TP_REQUIRE(lengths && L >= 1, TP_ERR_BAD_ARG, "tp_kv_cache_read: null lengths or no positions");
  const PageRows ck = rows_of(c, false), cv = rows_of(c, true);
  const int64_t rows = (int64_t)B * L * c->heads;
  unsigned k_blocks, blocks;
  const int per_lane = kv_rows(rows);
  TP_REQUIRE(kv_blocks(ck, cv, rows, per_lane, k_blocks, blocks), TP_ERR_UNSUPPORTED, "tp_kv_cache_read: too many rows");
  const KvRowsIn ko{(const char*)k, k_strides[0], k_strides[1], k_strides[2]}, vo{(const char*)v, v_strides[0], v_strides[1], v_strides[2]};
  kv_dispatch(dtype, c->dtype == TP_FP8, [&](auto t, auto quant) {
    const auto kern = per_lane == 1 ? kv_read_kernel<decltype(t), quant.value, 8, 1> : kv_read_kernel<decltype(t), quant.value, 8, 2>;
    kern<<<blocks, KV_THREADS, 0, (hipStream_t)stream>>>(ck, cv, ko, vo, table_of(c), lengths, (unsigned)rows, L, c->heads, k_blocks);
  });
  return check_launch("tp_kv_cache_read");
}
