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
// three dependent loads: position, table entry, row (small ones).  A lane moves 8 elements; a row is D / 8 lanes of a group of
// 8, 16, 32 or 64, the group of one row inside one wave, where the row's maximum is taken with lane exchanges.
#pragma once
#include "common.hpp"

namespace tp {

typedef unsigned char fp8_t;  // a float8_e4m3fn, moved as its bits

// One 16-bit, 32-bit or 8-bit tensor of the cache: (page, head, slot) strides in elements, dim contiguous
struct PageRows {
  char* base;
  float* scale;  // (page, head, slot), contiguous; null where the values are stored as they are
  int64_t page, head, slot;
  int dim, group;  // lanes per row: the power of two from dim / 8 up, at least 8
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

__device__ __forceinline__ u32x2 pack_fp8(const float (&x)[8]) {
  u32x2 r;
#pragma unroll
  for (int i = 0; i < 2; i++) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i], x[4 * i + 1], 0, false);
    r[i] = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i + 2], x[4 * i + 3], w, true);
  }
  return r;
}
__device__ __forceinline__ void unpack_fp8(const u32x2 w, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 2; i++) {
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

// Row r of a launch is (b, s, h) with the head fastest: the order of the memory that the projections write.
template <typename T, bool QUANT>
__device__ __forceinline__ void kv_write_rows(const PageRows& c, const KvRowsIn& in, const PageTable& tab, const int32_t* positions,
                                              const int32_t* counts, int64_t first, int64_t rows, int S, int H) {
  const int64_t at = first * KV_THREADS + threadIdx.x;
  const int64_t r = at / c.group;
  const int lane = (int)(at & (c.group - 1));
  if (r >= rows) return;  // (whole groups leave together)
  const int64_t bs = r / H;
  const int h = (int)(r - bs * H), b = (int)(bs / S), s = (int)(bs - (int64_t)b * S);
  if (counts && s >= counts[b]) return;
  const int64_t t = (int64_t)positions[b] + s;
  const int page = t < 0x7fffffff ? tab.page_of(b, (int)t) : -1;
  if (page < 0) return;
  const int slot = (int)t & ((1 << tab.page_shift) - 1);
  const bool mine = lane * 8 < c.dim;
  const T* src = reinterpret_cast<const T*>(in.base) + b * in.b + h * in.h + s * in.s + lane * 8;
  const int64_t dst = page * c.page + h * c.head + slot * c.slot + lane * 8;
  if constexpr (!QUANT) {
    if (mine) {
      const Raw<T, 8> x = load_raw_nt<T, 8>(src);
      u32x4* d = reinterpret_cast<u32x4*>(reinterpret_cast<T*>(c.base) + dst);
#pragma unroll
      for (int i = 0; i < (int)(sizeof(T) / 2); i++) __builtin_nontemporal_store(x.q[i], d + i);
    }
  } else {
    float x[8] = {};
    if (mine) load_f_nt<T, 8>(src, x);
    // the largest magnitude by its bits: a NaN is above an infinity, and that above every number
    unsigned top = 0;
#pragma unroll
    for (int e = 0; e < 8; e++) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
    for (int o = c.group / 2; o > 0; o >>= 1) top = max(top, (unsigned)__shfl_xor((int)top, o, 64));
    const float a = __uint_as_float(top);
    const bool finite = top < 0x7f800000u, some = finite && a >= FP8_TINY;
    const float back = some ? FP8_MAX / a : 0.f;
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] = finite ? x[e] * back : 0.f;
    if (mine) {
      __builtin_nontemporal_store(pack_fp8(x), reinterpret_cast<u32x2*>(c.base + dst));
      if (lane == 0)
        c.scale[(((int64_t)page * H + h) << tab.page_shift) + slot] = !finite ? __uint_as_float(0x7fc00000u) : some ? a / FP8_MAX : 0.f;
    }
  }
}

// blocks [0, k_blocks) take the keys, the others the values
template <typename T, bool QUANT>
__global__ __launch_bounds__(KV_THREADS) void kv_write_kernel(PageRows ck, PageRows cv, KvRowsIn k, KvRowsIn v, PageTable tab,
                                                              const int32_t* __restrict__ positions, const int32_t* __restrict__ counts,
                                                              int64_t rows, int S, int H, unsigned k_blocks) {
  if (blockIdx.x < k_blocks) kv_write_rows<T, QUANT>(ck, k, tab, positions, counts, blockIdx.x, rows, S, H);
  else kv_write_rows<T, QUANT>(cv, v, tab, positions, counts, blockIdx.x - k_blocks, rows, S, H);
}

// Row r of a launch is (b, h, t) with the position fastest: whole pages are read and whole stretches written.
template <typename T, bool QUANT>
__device__ __forceinline__ void kv_read_rows(const PageRows& c, const KvRowsIn& out, const PageTable& tab, const int32_t* lengths,
                                             int64_t first, int64_t rows, int L, int H) {
  const int64_t at = first * KV_THREADS + threadIdx.x;
  const int64_t r = at / c.group;
  const int lane = (int)(at & (c.group - 1));
  if (r >= rows || lane * 8 >= c.dim) return;
  const int64_t bh = r / L;
  const int t = (int)(r - bh * L), b = (int)(bh / H), h = (int)(bh - (int64_t)b * H);
  const int page = t < lengths[b] ? tab.page_of(b, t) : -1;
  const int slot = t & ((1 << tab.page_shift) - 1);
  T* dst = reinterpret_cast<T*>(const_cast<char*>(out.base)) + b * out.b + h * out.h + t * out.s + lane * 8;
  const int64_t src = page * c.page + h * c.head + slot * c.slot + lane * 8;
  if constexpr (!QUANT) {
    Raw<T, 8> x{};
    if (page >= 0) x = load_raw_nt<T, 8>(reinterpret_cast<const T*>(c.base) + src);
    u32x4* d = reinterpret_cast<u32x4*>(dst);
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) / 2); i++) __builtin_nontemporal_store(x.q[i], d + i);
  } else {
    float x[8] = {};
    if (page >= 0) {
      unpack_fp8(__builtin_nontemporal_load(reinterpret_cast<const u32x2*>(c.base + src)), x);
      const float scale = c.scale[(((int64_t)page * H + h) << tab.page_shift) + slot];
#pragma unroll
      for (int e = 0; e < 8; e++) x[e] *= scale;
    }
    store_f_nt<T, 8>(dst, x);
  }
}

template <typename T, bool QUANT>
__global__ __launch_bounds__(KV_THREADS) void kv_read_kernel(PageRows ck, PageRows cv, KvRowsIn k, KvRowsIn v, PageTable tab,
                                                             const int32_t* __restrict__ lengths, int64_t rows, int L, int H,
                                                             unsigned k_blocks) {
  if (blockIdx.x < k_blocks) kv_read_rows<T, QUANT>(ck, k, tab, lengths, blockIdx.x, rows, L, H);
  else kv_read_rows<T, QUANT>(cv, v, tab, lengths, blockIdx.x - k_blocks, rows, L, H);
}

// ---- host --------------------------------------------------------------------------------------
inline int elem_size(int dtype) { return dtype == TP_F32 ? 4 : dtype == TP_FP8 ? 1 : 2; }

// what every entry point asks of a cache; `dtype` is the type of the tensors that go in or come out
inline int check_cache(const tp_kv_cache* c, int dtype, int B, const char* who) {
  TP_REQUIRE(c && c->k && c->v && c->table, TP_ERR_BAD_ARG, "%s: null pointer", who);
  TP_REQUIRE(dtype >= TP_BF16 && dtype <= TP_F32, TP_ERR_UNSUPPORTED, "%s: unsupported dtype code %d", who, dtype);
  TP_REQUIRE(c->dtype == dtype || (c->dtype == TP_FP8 && dtype != TP_F32), TP_ERR_UNSUPPORTED,
             "%s: a cache of dtype code %d does not go with tensors of code %d", who, c->dtype, dtype);
  TP_REQUIRE(B >= 1 && c->pages >= 1 && c->heads >= 1 && c->table_width >= 1 && c->table_stride >= 0, TP_ERR_BAD_ARG, "%s: sizes must be positive", who);
  TP_REQUIRE(c->page_size >= 8 && (c->page_size & (c->page_size - 1)) == 0, TP_ERR_UNSUPPORTED, "%s: page_size %d is not a power of two from 8 up", who, c->page_size);
  TP_REQUIRE((int64_t)c->table_width * c->page_size <= 0x7fffffff, TP_ERR_UNSUPPORTED, "%s: the table covers more than 2^31 positions", who);
  for (int d : {c->k_dim, c->v_dim})
    TP_REQUIRE(d >= 8 && d <= 512 && d % 8 == 0, TP_ERR_UNSUPPORTED, "%s: head dim %d is not a multiple of 8 up to 512", who, d);
  const int e = elem_size(c->dtype), step = c->dtype == TP_FP8 ? 8 : 16;
  TP_REQUIRE((((uintptr_t)c->k | (uintptr_t)c->v) & 15) == 0, TP_ERR_BAD_ARG, "%s: the cache must start at 16-byte addresses", who);
  for (int i = 0; i < 3; i++)
    TP_REQUIRE(c->k_strides[i] >= 0 && c->v_strides[i] >= 0 && c->k_strides[i] * e % step == 0 && c->v_strides[i] * e % step == 0, TP_ERR_BAD_ARG,
               "%s: strides of the cache must keep rows %d-byte aligned", who, step);
  TP_REQUIRE((c->dtype == TP_FP8) == (c->k_scale != nullptr) && (c->dtype == TP_FP8) == (c->v_scale != nullptr), TP_ERR_BAD_ARG,
             "%s: an 8-bit cache needs k_scale and v_scale, another cache has none", who);
  return TP_OK;
}
inline int log2_of(int n) { int s = 0; while ((1 << s) < n) s++; return s; }
inline PageTable table_of(const tp_kv_cache* c) { return {c->table, c->table_stride, c->table_width, c->pages, log2_of(c->page_size)}; }
inline PageRows rows_of(const tp_kv_cache* c, bool values) {
  const int64_t* s = values ? c->v_strides : c->k_strides;
  const int dim = values ? c->v_dim : c->k_dim;
  int group = 8;
  while (group * 8 < dim) group *= 2;
  return {(char*)(values ? c->v : c->k), values ? c->v_scale : c->k_scale, s[0], s[1], s[2], dim, group};
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

// blocks of a launch over `rows` rows of both tensors: (those of the keys, all of them)
inline bool kv_blocks(const PageRows& ck, const PageRows& cv, int64_t rows, unsigned& k_blocks, unsigned& all) {
  const int64_t kb = (rows * ck.group + KV_THREADS - 1) / KV_THREADS, vb = (rows * cv.group + KV_THREADS - 1) / KV_THREADS;
  k_blocks = (unsigned)kb;
  all = (unsigned)(kb + vb);
  return kb + vb < (1ll << 32) / KV_THREADS;  // (a launch has fewer than 2^32 lanes)
}

}  // namespace tp

extern "C" int tp_kv_cache_write(const tp_kv_cache* c, const void* k, const void* v, const int32_t* positions, const int32_t* counts, int B, int S,
                                 const int64_t* k_strides, const int64_t* v_strides, int dtype, void* stream) {
  using namespace tp;
  if (int rc = check_cache(c, dtype, B, "tp_kv_cache_write")) return rc;
  if (int rc = check_rows(k, v, k_strides, v_strides, dtype, "tp_kv_cache_write")) return rc;
  TP_REQUIRE(positions && S >= 1, TP_ERR_BAD_ARG, "tp_kv_cache_write: null positions or no tokens");
  const PageRows ck = rows_of(c, false), cv = rows_of(c, true);
  const int64_t rows = (int64_t)B * S * c->heads;
  unsigned k_blocks, blocks;
  TP_REQUIRE(kv_blocks(ck, cv, rows, k_blocks, blocks), TP_ERR_UNSUPPORTED, "tp_kv_cache_write: too many rows");
  const KvRowsIn ki{(const char*)k, k_strides[0], k_strides[1], k_strides[2]}, vi{(const char*)v, v_strides[0], v_strides[1], v_strides[2]};
  kv_dispatch(dtype, c->dtype == TP_FP8, [&](auto t, auto quant) {
    kv_write_kernel<decltype(t), quant.value><<<blocks, KV_THREADS, 0, (hipStream_t)stream>>>(ck, cv, ki, vi, table_of(c), positions, counts, rows, S, c->heads, k_blocks);
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
  TP_REQUIRE(kv_blocks(ck, cv, rows, k_blocks, blocks), TP_ERR_UNSUPPORTED, "tp_kv_cache_read: too many rows");
  const KvRowsIn ko{(const char*)k, k_strides[0], k_strides[1], k_strides[2]}, vo{(const char*)v, v_strides[0], v_strides[1], v_strides[2]};
  kv_dispatch(dtype, c->dtype == TP_FP8, [&](auto t, auto quant) {
    kv_read_kernel<decltype(t), quant.value><<<blocks, KV_THREADS, 0, (hipStream_t)stream>>>(ck, cv, ko, vo, table_of(c), lengths, rows, L, c->heads, k_blocks);
  });
  return check_launch("tp_kv_cache_read");
}
