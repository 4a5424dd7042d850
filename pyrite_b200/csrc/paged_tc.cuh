// paged_tc.cuh -- what the tcgen05 attention kernels over a paged pool share
// (paged_attention_tc.cu, paged_chunks_tc.cu): descriptors, tensor memory access, the
// planes of the weights, and the pools as tensor maps.
#pragma once
#include <atomic>
#include <cuda.h>

#include "paged.cuh"
#include "ptx.cuh"

namespace pyr {
namespace tc {

constexpr uint32_t kHalf = 128 * 128;  // bytes of 128 rows of 64 16-bit values
constexpr uint32_t kTileBytes = 2 * kHalf;

template <typename T> struct Planes;
template <> struct Planes<__half> { static constexpr int n = 2, format = 0; };
template <> struct Planes<__nv_bfloat16> { static constexpr int n = 3, format = 1; };

// kind::f16 with fp32 accumulation; b_mn: B is stored along N.
__host__ __device__ constexpr uint32_t idesc(int format, int m, int n, bool b_mn) {
  return (1u << 4) | ((uint32_t)format << 7) | ((uint32_t)format << 10) | ((b_mn ? 1u : 0u) << 16) |
         ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
// V as B, stored along N (the head dimension): 64-value halves kHalf apart, 8-key
// groups 1024 bytes apart, 128-byte swizzle.
__device__ __forceinline__ uint64_t desc_v(uint32_t saddr) {
  uint64_t d = (uint64_t)((saddr >> 4) & 0x3FFFu);
  d |= (uint64_t)(kHalf >> 4) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t acc) {
  ptx::tc_mma_bf16(d, a, b, id, acc);
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a_tmem, uint64_t b, uint32_t id, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
      "r"(a_tmem), "l"(b), "r"(id), "r"(acc)
      : "memory");
}
// 32 columns of this warp's 32 TMEM lanes; the values are there after tmem_wait_ld32.
__device__ __forceinline__ void tmem_ld32(uint32_t a, float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(a));
}
// The values pass through the wait, so nothing that uses them can move before it.
__device__ __forceinline__ void tmem_wait_ld32(float* v) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]), "+f"(v[8]),
                 "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]), "+f"(v[16]),
                 "+f"(v[17]), "+f"(v[18]), "+f"(v[19]), "+f"(v[20]), "+f"(v[21]), "+f"(v[22]), "+f"(v[23]), "+f"(v[24]),
                 "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]), "+f"(v[29]), "+f"(v[30]), "+f"(v[31])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t a, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(a),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t a, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(a), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tma_box(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::
          "r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}

// Two fp32 values a register pair, two operations an instruction.
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pair(float a, float b) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpair(f32x2 v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// One plane of a pair of weights; what is left of them stays in x and y.  bf16: cut
// off instead of rounded (8 bits a plane: three hold fp32's 24), which needs no conversion.
template <typename T> __device__ __forceinline__ uint32_t weight_plane(float& x, float& y, bool rest);
template <> __device__ __forceinline__ uint32_t weight_plane<__half>(float& x, float& y, bool rest) {
  const __half2 h = __floats2half2_rn(x, y);
  if (rest) {
    const float2 f = __half22float2(h);
    unpair(fma2(pair(f.x, f.y), pair(-1.f, -1.f), pair(x, y)), x, y);
  }
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t weight_plane<__nv_bfloat16>(float& x, float& y, bool rest) {
  const uint32_t a = __float_as_uint(x), b = __float_as_uint(y);
  if (rest) {
    const f32x2 cut = pair(__uint_as_float(a & 0xffff0000u), __uint_as_float(b & 0xffff0000u));
    unpair(fma2(cut, pair(-1.f, -1.f), pair(x, y)), x, y);
  }
  return __byte_perm(a, b, 0x7632);
}

typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                             const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                             CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeFn encode_fn() {
  static std::atomic<void*> fn;  // idempotent: concurrent first calls look up the same entry
  void* f = fn.load(std::memory_order_acquire);
  if (!f) {
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess)
      return nullptr;
    fn.store(f, std::memory_order_release);
  }
  return reinterpret_cast<EncodeFn>(f);
}

// A pool as [page][head and token][128]: a box is `tokens_of_box` tokens (at most a page) of
// one head, half of their values, in the 128-byte swizzle.
inline bool encode_pool(CUtensorMap* map, void* pool, int format, int n_kv_heads, int ps_log2, int n_pages,
                        int tokens_of_box) {
  EncodeFn encode = encode_fn();
  if (!encode) return false;
  const cuuint64_t tokens = (cuuint64_t)n_kv_heads << ps_log2;
  const cuuint64_t dims[3] = {128, tokens, (cuuint64_t)n_pages}, strides[2] = {256, tokens * 256};
  const cuuint32_t box[3] = {64, (cuuint32_t)tokens_of_box, 1}, ones[3] = {1, 1, 1};
  return encode(map, format ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, pool, dims, strides,
                box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace tc
}  // namespace pyr
