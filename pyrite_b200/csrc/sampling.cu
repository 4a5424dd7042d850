// sampling.cu -- the next token of each row of logits by temperature, top-k,
// top-p and min-p, from given random numbers.
//
// In the order of falling logits (ties: the lower id first) with weights
// w_i = e^((l_i - max) / T), every filter keeps a beginning of that order:
//   top-k  the first k;
//   top-p  the tokens whose preceding weight is below top_p * (weight of the first k);
//   min-p  the tokens with w_i >= min_p;
// and the token is the first whose cumulative weight exceeds u * (kept weight).
// So everything is three searches "where does the cumulative count or weight
// pass a target".  Weights are held as 64-bit integers w_i * 2^S: their sums do
// not depend on the order of the additions, so any split of a row gives the same
// token, and S = 62 - ceil(log2 n) keeps at least 44 bits for 2^18 tokens below the largest
// weight, far below the 2^-24 spacing of 32-bit random numbers.
#include <cfloat>

#include "kernels.cuh"
#include "../../include/pyrite_b200.h"

namespace pyr {
namespace {

typedef unsigned long long u64;

// Orders as the floats do (NaN with -inf, last; -0 with +0).
__device__ __forceinline__ uint32_t sort_key(float x) {
  if (!(x > -INFINITY)) return 0u;
  const uint32_t b = __float_as_uint(x == 0.f ? 0.f : x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return k == 0u ? -INFINITY : __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

struct SampleArgs {
  const float* logits;
  long long ld;
  int n;
  const float* u;
  const float* temperature;
  const int* top_k;
  const float* top_p;
  const float* min_p;
  int* ids;
  float* probs;
  int scale_log2;  // S
};

// e^((value - max) / T): 1 at the maximum even where that is infinite.
__device__ __forceinline__ double weight(uint32_t key, uint32_t top, double inv_t) {
  if (key == top) return 1.0;
  if (key == 0u) return 0.0;
  return exp(((double)key_value(key) - (double)key_value(top)) * inv_t);
}

__device__ __forceinline__ u64 block_add(u64 v, u64* sh) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  u64 t = (threadIdx.x & 31) < (blockDim.x >> 5) ? sh[threadIdx.x & 31] : 0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
  return t;
}

// One CTA per row; a search decides one bit of the key a pass.
__global__ void __launch_bounds__(1024) sample_rows_kernel(SampleArgs a) {
  __shared__ u64 sh[32];
  __shared__ int found;
  pdl_wait();
  const float* row = a.logits + (long long)blockIdx.x * a.ld;
  const int tid = threadIdx.x, n = a.n;
  const double unit = (double)(1ull << a.scale_log2);
  u64 best = 0;
  for (int i = tid; i < n; i += 1024) {
    const u64 c = ((u64)sort_key(row[i]) << 32) | (uint32_t)~i;
    best = c > best ? c : best;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const u64 c = __shfl_xor_sync(0xffffffffu, best, o);
    best = c > best ? c : best;
  }
  if ((tid & 31) == 0) sh[tid >> 5] = best;
  __syncthreads();
  best = sh[tid & 31];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const u64 c = __shfl_xor_sync(0xffffffffu, best, o);
    best = c > best ? c : best;
  }
  const uint32_t top = (uint32_t)(best >> 32);
  const float temp = a.temperature[blockIdx.x];
  int id = top ? (int)~(uint32_t)best : -1;
  double prob = top ? 1.0 : 0.0;
  if (top && temp > 0.f) {
    const double inv_t = 1.0 / (double)temp;
    auto fixed = [&](uint32_t key) { return (u64)__double2ull_rn(weight(key, top, inv_t) * unit); };
    // the largest key whose count (or weight) of keys >= it reaches the target
    auto search = [&](bool count, u64 target) {
      uint32_t key = 0;
      for (int bit = 31; bit >= 0; --bit) {
        const uint32_t c = key | (1u << bit);
        u64 s = 0;
        for (int i = tid; i < n; i += 1024) {
          const uint32_t k = sort_key(row[i]);
          if (k >= c) s += count ? 1ull : fixed(k);
        }
        if (block_add(s, sh) >= target) key = c;
      }
      return key;
    };
    auto above = [&](bool count, uint32_t key) {
      u64 s = 0;
      for (int i = tid; i < n; i += 1024) {
        const uint32_t k = sort_key(row[i]);
        if (k > key) s += count ? 1ull : fixed(k);
      }
      return block_add(s, sh);
    };
    u64 mass;
    const int k = a.top_k ? a.top_k[blockIdx.x] : 0;
    if (k > 0 && k < n) {
      const uint32_t key = search(true, (u64)k);
      mass = above(false, key) + ((u64)k - above(true, key)) * fixed(key);
    } else {
      u64 s = 0;
      for (int i = tid; i < n; i += 1024) s += fixed(sort_key(row[i]));
      mass = block_add(s, sh);
    }
    u64 kept = mass;
    const float p = a.top_p ? a.top_p[blockIdx.x] : 1.f;
    if (p < 1.f) {
      u64 target = (u64)ceil(fmax((double)p, 0.0) * (double)mass);
      target = target < 1 ? 1 : target;
      const uint32_t key = search(false, target);
      const u64 over = above(false, key), w = fixed(key);
      const u64 m = over + (target - over + w - 1) / w * w;
      kept = m < kept ? m : kept;
    }
    const float mp = a.min_p ? a.min_p[blockIdx.x] : 0.f;
    if (mp > 0.f) {
      const double lim = fmin((double)mp, 1.0);
      u64 s = 0;
      for (int i = tid; i < n; i += 1024) {
        const uint32_t key = sort_key(row[i]);
        if (weight(key, top, inv_t) >= lim) s += fixed(key);
      }
      s = block_add(s, sh);
      kept = s < kept ? s : kept;
    }
    const float uf = a.u[blockIdx.x];
    u64 x = uf > 0.f ? (u64)((double)uf * (double)kept) : 0;
    x = x < kept ? x : kept - 1;
    const uint32_t key = search(false, x + 1);
    const u64 w = fixed(key);
    u64 rank = (x - above(false, key)) / w;
    // the rank-th token with this key, in id order
    if (tid == 0) found = 0;
    for (int base = 0; base < n; base += 1024) {
      const int i = base + tid;
      const bool hit = i < n && sort_key(row[i]) == key;
      const unsigned vote = __ballot_sync(0xffffffffu, hit);
      __syncthreads();
      if ((tid & 31) == 0) sh[tid >> 5] = __popc(vote);
      __syncthreads();
      u64 before = 0, all = 0;
      for (int q = 0; q < 32; ++q) {
        if (q < (tid >> 5)) before += sh[q];
        all += sh[q];
      }
      if (hit && before + __popc(vote & ((1u << (tid & 31)) - 1u)) == rank) found = i;
      if (rank < all) break;
      rank -= all;
    }
    __syncthreads();
    id = found;
    prob = (double)w / (double)kept;
  }
  if (tid == 0) {
    a.ids[blockIdx.x] = id;
    if (a.probs) a.probs[blockIdx.x] = (float)prob;
  }
  pdl_launch_dependents();
}

int rc(int e) { return e > 0 ? PYRITE_E_CUDA : e; }

}  // namespace
}  // namespace pyr

using namespace pyr;

extern "C" {

int pyrite_cuda_sample_rows(const float* logits, long long ld, size_t n, size_t count, const float* uniforms,
                            const float* temperature, const int* top_k, const float* top_p, const float* min_p,
                            int* ids, float* probs, void* stream) {
  if (!logits || !uniforms || !temperature || !ids) return PYRITE_E_BUFFER;
  if (n == 0 || n > (1u << 20) || count == 0 || count > 65535 || ld < (long long)n) return PYRITE_E_SHAPE;
  int bits = 0;
  while ((1u << bits) < n) ++bits;
  const SampleArgs a{logits, ld, (int)n, uniforms, temperature, top_k, top_p, min_p, ids, probs, 62 - bits};
  return rc(launch_pdl(sample_rows_kernel, dim3((unsigned)count), dim3(1024), 0, static_cast<cudaStream_t>(stream), a));
}

}  // extern "C"
