// paged.cuh -- the layout of a paged key/value pool (paged.cu, paged_attention.cu).
#pragma once
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "ggml_blocks.cuh"

namespace pyr {

// Page sizes: powers of two, so a token's page is a shift and a page's keys of
// one head fill whole 16-key tiles.
__host__ __device__ inline bool page_size_ok(int ps) { return ps >= 16 && ps <= 256 && (ps & (ps - 1)) == 0; }
__host__ __device__ inline int log2_of(int ps) {
  int l = 0;
  while ((1 << l) < ps) ++l;
  return l;
}
// A slot index and a (page, head) tile index fit 32 bits; element offsets are 64-bit.
inline bool pool_ok(int n_pages, int page_size, int n_kv_heads) {
  return n_pages > 0 && page_size_ok(page_size) && (long long)n_pages * page_size <= 0x7fffffffLL &&
         n_kv_heads <= 1024 && (long long)n_pages * n_kv_heads <= 0x7fffffffLL;
}
inline bool kv_type_ok(int t) { return t == F32 || t == F16 || t == BF16; }

// One rounding from fp64 (or fp32) to the cache type: through fp32 first, a
// 16-bit result could be rounded twice.
__device__ __forceinline__ float2 cvt2(double x, double y, float*) { return make_float2((float)x, (float)y); }
__device__ __forceinline__ __half2 cvt2(double x, double y, __half*) {
  return __halves2half2(__double2half(x), __double2half(y));
}
__device__ __forceinline__ __nv_bfloat162 cvt2(double x, double y, __nv_bfloat16*) {
  return __halves2bfloat162(__double2bfloat16(x), __double2bfloat16(y));
}
__device__ __forceinline__ float2 cvt2(float x, float y, float*) { return make_float2(x, y); }
__device__ __forceinline__ __half2 cvt2(float x, float y, __half*) { return __floats2half2_rn(x, y); }
__device__ __forceinline__ __nv_bfloat162 cvt2(float x, float y, __nv_bfloat16*) { return __floats2bfloat162_rn(x, y); }

template <typename T> struct Pair;
template <> struct Pair<float> { using type = float2; };
template <> struct Pair<__half> { using type = __half2; };
template <> struct Pair<__nv_bfloat16> { using type = __nv_bfloat162; };

template <typename T> struct PagePool {
  T* k;
  T* v;
  int n_pages;
  int ps_log2;
  // Values 2 lane, 2 lane + 1, 64 + 2 lane, 65 + 2 lane of one head at a slot.
  template <typename V>
  __device__ __forceinline__ void store2(T* base, int slot, int head, int nkv, int lane, V a, V b, V c, V d) const {
    const int ps = 1 << ps_log2;
    const size_t row = ((size_t)(slot >> ps_log2) * nkv + head) * ps + (slot & (ps - 1));
    auto* p = reinterpret_cast<typename Pair<T>::type*>(base + row * 128);
    p[lane] = cvt2(a, b, (T*)nullptr);
    p[lane + 32] = cvt2(c, d, (T*)nullptr);
  }
};

// ---- attention over the pool (paged_attention.cu, paged_attention_tc.cu) ------------------
constexpr int kPart = 128 + 4;    // floats of a part: m, l, 2 unused, o[128]
constexpr float kLazy = 8.f;      // the running maximum (base 2) moves when it would grow by more
constexpr float kUp = 7.f;        // weights are held times 2^kUp: at most 2^15, inside fp16

// The work of one attention launch: `rows` lists of keys (the rows' own ones, or
// the one prefix), `items` items each (KV head x tile of `tile` query rows).
struct AttnWork {
  const float* q;
  long long ldq;
  const int* pages;        // the rows' page lists, table_stride apart
  long long table_stride;
  const int* lens;         // own: tokens of each row (device), at most max_len; prefix: NULL
  int max_len, fixed_len;  // prefix: its length
  int rows, items, tile;
  int count, nq, nkv;
  bool behind_prefix;      // own keys, launched behind the prefix's
  float* parts;
  float qscale;
  int* status;
};

// A power of two that brings a row's largest value to the upper end of fp16, [2^kHigh, 2^(kHigh + 1))
// (fp16 planes; bf16 has fp32's range and takes 1): down multiplies q, `back` the scores.  Two planes then leave out
// less than 2^-24 of a value, or 2^-38 of the row's largest where that is more, so a few channels far above the
// others (to 2^14 times) cost these nothing.  Any finite row fits: with fp32's last exponent, whose reciprocal is no
// normal number, the largest becomes less than 2^(kHigh + 2).
constexpr int kHigh = 13;
template <typename T> __device__ __forceinline__ float row_scale(float largest, float& back);
template <> __device__ __forceinline__ float row_scale<__half>(float largest, float& back) {
  // exponent of the largest value, while both powers are normal numbers
  const int x = min(max((int)(__float_as_uint(largest) >> 23) - 127, kHigh - 126), 126);
  const int e = (largest > 0.f && largest < INFINITY ? x : 0) - kHigh;
  back = __uint_as_float((uint32_t)(127 + e) << 23);
  return __uint_as_float((uint32_t)(127 - e) << 23);
}
template <> __device__ __forceinline__ float row_scale<__nv_bfloat16>(float, float& back) { return back = 1.f; }

// The two values rounded to T, packed; what is left of them stays in x and y.
template <typename T> __device__ __forceinline__ uint32_t plane2(float& x, float& y);
template <> __device__ __forceinline__ uint32_t plane2<__half>(float& x, float& y) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  x -= f.x;
  y -= f.y;
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t plane2<__nv_bfloat16>(float& x, float& y) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
  const uint32_t b = *reinterpret_cast<const uint32_t*>(&h);
  x -= __uint_as_float(b << 16);
  y -= __uint_as_float(b & 0xffff0000u);
  return b;
}

// 2^x by the special function unit: 2 units in the last place, results below the
// normal range are 0.
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Parts per (KV head, 128 query rows) when the prefix of these sizes goes to
// prefix_tc_kernel, 0 when to the row kernels.
int prefix_tc_split(int query_rows, int n_kv_heads, int prefix_len, int kv_type);
int launch_prefix_tc(const AttnWork& w, void* k, void* v, int kv_type, int n_pages, int page_size, int split,
                     cudaStream_t stream);

}  // namespace pyr
