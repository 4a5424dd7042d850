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
// token.  S is 44, or 62 - log2 n for rows wider than 2^18, so that the sums fit.  A
// weight is good to 2^-(S + 1) of the largest and a sum of n of them to n 2^-(S + 1) at
// worst, about its root where the roundings point either way: 2^-27 for 151936 tokens,
// 2^-23 for the widest rows (2^20), beside the 2^-24 spacing of 32-bit random numbers.
#include <atomic>
#include <cfloat>

#include "kernels.cuh"
#include "ptx.cuh"
#include "../../include/pyrite_b200.h"

namespace pyr {
namespace {

typedef unsigned long long u64;

// A row belongs to a cluster of C CTAs (one CTA where there are many rows), each
// with a slice of it; what the searches need crosses the cluster through
// distributed shared memory.
//   1. The row's maximum (first index).  A slice that fits stays in shared
//      memory; a whole row is read again from L2 in the later passes.
//   2. The weights' histogram over bins of (max - l) / T, 1/128 wide: 64-bit sums
//      as two 32-bit words, the carry passed on (shared memory adds 32-bit
//      integers natively; one such pass over 128 rows of 151936 took 23 us, with
//      64-bit atomic additions 76 us).  The CTAs exchange sums of kFine bins; a search
//      finds its place among those and then asks for the bins of that one.
//   3. The tokens of the bins where the searches end go to CTA 0, which orders (by
//      counting what precedes each) and scans them.  Bins of more than kList tokens (ties, coarse logits) are
//      divided again by the bits of their keys until they are short or one value,
//      whose tokens count in id order.
// With a short top-k (the usual case) step 2 counts only, step 3 gathers all
// first k at once and CTA 0 finishes alone: no weight is computed for the rest
// of the vocabulary.
//
// A row of 151936 alone, on eight CTAs, takes 18 us, a chain of short phases: maxima of
// the slices 1.9, of the cluster 2.6, counts 1.7, search 3.7, gather 1.4, to CTA 0 1.2, order
// and pick 3.4; four cluster barriers among them.  128 rows of 151936 under top-p take 94
// us from HBM (the bytes alone 12 us), 87 with the logits partly in L2, of which: 10 to
// find the maxima, 42 to weigh (fp64 weights, shared-memory additions; half of the issue
// slots are taken), 16 to gather, the rest searches and lists.
constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 4096;
constexpr float kBinsPerNat = 128.f;
constexpr int kList = 2048;
constexpr int kPer = kList / kThreads;  // list entries a thread
constexpr int kShort = 128;             // lists up to this length are one warp's work
constexpr int kExpBits = 9;             // table of 2^(j / 512)
constexpr int kMaxCluster = 8;
constexpr int kFine = 64, kCoarse = kBins / kFine;
constexpr int kTargets = 2;             // searches at a time

__device__ __forceinline__ float clean(float x) { return x > -INFINITY ? x + 0.f : -INFINITY; }  // NaN: -inf; -0: 0
__device__ __forceinline__ uint32_t sort_key(float x) {  // orders as the floats do
  const uint32_t b = __float_as_uint(clean(x));
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

struct SampleArgs {
  const float* logits;
  long long ld;
  int n;
  int slice;     // tokens of a CTA
  int resident;  // slices are kept in shared memory
  const float* u;
  const float* temperature;
  const int* top_k;
  const float* top_p;
  const float* min_p;
  int* ids;
  float* probs;
  int scale_log2;  // S, at most 44
};

// ---- distributed shared memory ------------------------------------------------------------
__device__ __forceinline__ uint32_t remote(const void* p, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(ptx::smem_addr(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ void st_remote64(uint32_t a, u64 v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(a), "l"(v) : "memory");
}
__device__ __forceinline__ uint32_t add_remote32(uint32_t a, uint32_t v) {
  uint32_t o;
  asm volatile("atom.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(o) : "r"(a), "r"(v) : "memory");
  return o;
}

struct Found {  // a bin, the sum before it and its own
  int bin;
  u64 before, in;
};

struct alignas(16) Fixed {  // shared memory of one CTA, before the slice
  double exp_table[1 << kExpBits];
  uint32_t lo[kBins], hi[kBins];  // this CTA's histogram
  u64 stage[2][kList];            // this CTA's tokens on their way to CTA 0
  u64 list[2][kList];             // CTA 0: gathered tokens (key, ~id)
  u64 coarse[kMaxCluster][kCoarse];           // every CTA's sums of kFine bins
  u64 before[kCoarse + 1];                    // over the cluster: the sums before them
  u64 fine[2][kTargets][kMaxCluster][kFine];  // every CTA's bins where a search ends
  Found found[kTargets];
  u64 part[2][kMaxCluster];  // reduction operands
  u64 answer[2];             // CTA 0 to all
  u64 warp_sum[kWarps];
  u64 hit[2];  // the mass up to the picked token, its units
  uint32_t list_len[2], stage_len[2], stage_at;
  int picked;
};

extern __shared__ __align__(16) uint8_t smem[];
__device__ __forceinline__ Fixed& shared() { return *reinterpret_cast<Fixed*>(smem); }

// A token's bin and weight, given the row's maximum and temperature (held in
// registers in the passes over a slice).
struct Scale {
  float top, bin_scale;
  double to_table;  // 512 log2(e) / T
  int log2;         // S

  // Bins fall with the logit; every rounding keeps the order.
  __device__ __forceinline__ int bin(float x) const {
    const float t = fminf((top - x) * bin_scale, (float)(kBins - 1));
    return __float_as_int(__fadd_rd(t, 8388608.f)) & (kBins - 1);  // floor: 2^23 + t
  }
  // e^((x - max) / T) = 2^(k / 512) e^r by a table and a cubic (Tang's
  // table-driven method); 0 <= r < ln2 / 512, so the first term left out is below
  // 1.5e-13 relative.  x must be finite; the weight is 2^(k >> 9) times the result,
  // which lies in [1, 2).
  __device__ __forceinline__ double mantissa(float x, int& k) const {
    const double magic = 6755399441055744.0;  // 1.5 * 2^52: the sum's low word is the integer part
    const double t = ((double)x - (double)top) * to_table;  // the difference first: exact, however far from zero
    const double s = __dadd_rd(t, magic);
    k = __double2loint(s);
    const double g = t - (s - magic);
    constexpr double c1 = 0.0013538030870311431, c2 = c1 * c1 / 2, c3 = c1 * c1 * c1 / 6;  // ln2 / 512
    const double q = g * fma(g, fma(g, c3, c2), c1), e = shared().exp_table[k & ((1 << kExpBits) - 1)];
    return fma(e, q, e);
  }
  // Past the bins (32 / T below the maximum) a weight is below 2^-46: nothing.
  __device__ __forceinline__ double weight(float x) const {
    if (x == top) return 1.0;
    if (bin(x) == kBins - 1) return 0.0;
    int k;
    const double m = mantissa(x, k);
    return __hiloint2double(__double2hiint(m) + ((k >> kExpBits) << 20), __double2loint(m));
  }
  // The weight in units of 2^-S, rounded to nearest: added to 1.5 * 2^52 it
  // stands in the low bits.
  __device__ __forceinline__ u64 units(float x, int b) const {
    int k;
    const double m = mantissa(x, k), magic = 6755399441055744.0;
    const double w = __hiloint2double(__double2hiint(m) + (((k >> kExpBits) + log2) << 20), __double2loint(m));
    const u64 r = (u64)__double_as_longlong(w + magic) & 0x7ffffffffffffull;
    return b < kBins - 1 ? r : 0;
  }
  __device__ __forceinline__ u64 units(float x) const { return units(x, bin(x)); }
};

struct Row {
  const SampleArgs& a;
  Scale z;
  float* slice;       // resident slice, or NULL
  const float* src;   // the slice in global memory
  uint32_t rank, C;
  int len, base, head;  // tokens of this slice, its first id, tokens before a 16-byte boundary
  bool infinite;        // the largest logit is +inf: it reads as 0, all else as -inf
  int parity_fine = 0, parity_part = 0, parity_answer = 0;

  // Logits as they are read: NaN and -0 too (bin and sort_key put them in their places).
  __device__ __forceinline__ float seen(float x) const { return infinite ? (x == INFINITY ? 0.f : -INFINITY) : x; }
  __device__ __forceinline__ float get(int i) const { return slice ? slice[i] : seen(__ldg(src + i)); }
  // fn(value, index) for every token of the slice.
  template <typename Fn> __device__ __forceinline__ void each(Fn fn) const {
    const int head = this->head, n4 = (len - head) >> 2, tail = head + 4 * n4;
    if (const float* slice = this->slice) {
      for (int v = threadIdx.x; v < n4; v += kThreads) {
        const int i = head + 4 * v;
        const float4 x = *reinterpret_cast<const float4*>(slice + i);
        fn(x.x, i);
        fn(x.y, i + 1);
        fn(x.z, i + 2);
        fn(x.w, i + 3);
      }
    } else {
      const float* src = this->src;
      const bool infinite = this->infinite;
      auto seen = [=](float x) { return infinite ? (x == INFINITY ? 0.f : -INFINITY) : x; };
#pragma unroll 4
      for (int v = threadIdx.x; v < n4; v += kThreads) {
        const int i = head + 4 * v;
        const float4 x = __ldg(reinterpret_cast<const float4*>(src + i));
        fn(seen(x.x), i);
        fn(seen(x.y), i + 1);
        fn(seen(x.z), i + 2);
        fn(seen(x.w), i + 3);
      }
    }
    // at most 3 tokens before and 3 behind the 16-byte groups
    const int t = threadIdx.x, i = t < head ? t : tail + t - head;
    if (t < head + len - tail) fn(get(i), i);
  }

  __device__ __forceinline__ void sync() const {
    if (C > 1) ptx::cluster_sync();
    else __syncthreads();
  }

  __device__ __forceinline__ void clear_bins() const {
    for (int i = threadIdx.x; i < kBins; i += kThreads) shared().lo[i] = shared().hi[i] = 0;
    __syncthreads();
  }
  __device__ __forceinline__ void add_mass(int b, u64 w) const {
    const uint32_t l = (uint32_t)w;
    uint32_t h = (uint32_t)(w >> 32);
    h += atomicAdd(&shared().lo[b], l) > ~l ? 1u : 0u;
    if (h) atomicAdd(&shared().hi[b], h);
  }

  // Exclusive scan over the CTA; the total to every thread.
  __device__ __noinline__ u64 scan(u64 x, u64& total) const {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    u64 ix = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 p = __shfl_up_sync(0xffffffffu, ix, o);
      if (lane >= o) ix += p;
    }
    __syncthreads();
    if (lane == 31) shared().warp_sum[warp] = ix;
    __syncthreads();
    u64 w = shared().warp_sum[lane & (kWarps - 1)];  // every warp scans the warps' totals
#pragma unroll
    for (int o = 1; o < kWarps; o <<= 1) {
      const u64 p = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += p;
    }
    total = __shfl_sync(0xffffffffu, w, kWarps - 1);
    const u64 b = __shfl_sync(0xffffffffu, w, (warp + 31) & 31);
    return (warp ? b : 0) + ix - x;
  }

  // The sum of all histograms; afterwards searches can run.  Each CTA adds up
  // kFine bins at a time and sends those sums to all.
  __device__ __noinline__ u64 merge() {
    Fixed& f = shared();
    const int t = threadIdx.x;
    __syncthreads();
    u64 s = 0;
#pragma unroll
    for (int e = 0; e < kBins / kThreads; ++e) {
      const int b = t * (kBins / kThreads) + e;
      s += f.lo[b] | ((u64)f.hi[b] << 32);
    }
    constexpr int G = kFine * kThreads / kBins;  // threads of a coarse sum
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    for (uint32_t r = t % G; r < C; r += G) st_remote64(remote(&f.coarse[rank][t / G], r), s);
    sync();
    if (t < 32) {
      u64 v[kCoarse / 32], sum = 0;
#pragma unroll
      for (int e = 0; e < kCoarse / 32; ++e) {
        v[e] = 0;
#pragma unroll
        for (uint32_t r = 0; r < kMaxCluster; ++r) v[e] += r < C ? f.coarse[r][t * (kCoarse / 32) + e] : 0;
        sum += v[e];
      }
      u64 in = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const u64 q = __shfl_up_sync(0xffffffffu, in, o);
        if (t >= o) in += q;
      }
      u64 at = in - sum;
#pragma unroll
      for (int e = 0; e < kCoarse / 32; ++e) {
        f.before[t * (kCoarse / 32) + e] = at;
        at += v[e];
      }
      if (t == 31) f.before[kCoarse] = at;
    }
    __syncthreads();
    return f.before[kCoarse];
  }

  // The bins in which the cumulative sum reaches the targets (1 .. all).
  __device__ __noinline__ void search(u64 t0, u64 t1) {
    Fixed& f = shared();
    const int t = threadIdx.x, lane = t & 31, w = t >> 5;
    __syncthreads();  // the last search's results have been read
    if (t < kTargets * kFine) {  // a CTA's bins of the coarse sum where target t / kFine ends, to all
      const int which = t / kFine, e = t % kFine;
      const u64 target = which ? t1 : t0;
      const unsigned lo = __ballot_sync(0xffffffffu, f.before[lane + 1] < target);
      const unsigned hi = __ballot_sync(0xffffffffu, f.before[lane + 33] < target);
      const int b = (__popc(lo) + __popc(hi)) * kFine + e;
      const u64 v = f.lo[b] | ((u64)f.hi[b] << 32);
#pragma unroll
      for (uint32_t r = 0; r < kMaxCluster; ++r)
        if (r < C) st_remote64(remote(&f.fine[parity_fine][which][rank][e], r), v);
      if (e == 0) f.found[which].bin = b;
    }
    sync();
    if (w < kTargets) {
      const u64 target = w ? t1 : t0;
      const int c = f.found[w].bin;
      u64 v0 = 0, v1 = 0;
#pragma unroll
      for (uint32_t r = 0; r < kMaxCluster; ++r) {
        v0 += r < C ? f.fine[parity_fine][w][r][2 * lane] : 0;
        v1 += r < C ? f.fine[parity_fine][w][r][2 * lane + 1] : 0;
      }
      u64 in = v0 + v1;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const u64 q = __shfl_up_sync(0xffffffffu, in, o);
        if (lane >= o) in += q;
      }
      const u64 at = f.before[c / kFine] + in - v0 - v1;
      __syncwarp();
      if (at < target && target <= at + v0) f.found[w] = Found{c + 2 * lane, at, v0};
      else if (at + v0 < target && target <= at + v0 + v1) f.found[w] = Found{c + 2 * lane + 1, at + v0, v1};
    }
    __syncthreads();
    parity_fine ^= 1;
  }
  __device__ __forceinline__ Found search(u64 target) {
    search(target, target);
    const Found r = shared().found[0];
    return r;
  }

  // This CTA's members -> its stage (counted past kList, stored up to it).
  __device__ __forceinline__ void stage_one(int l, float x, int i) const {
    const uint32_t at = atomicAdd(&shared().stage_len[l], 1u);
    if (at < kList) shared().stage[l][at] = ((u64)sort_key(x) << 32) | (uint32_t)~(base + i);
  }
  // The stages of all CTAs -> CTA 0's list.
  __device__ __noinline__ void collect(int l) {
    __syncthreads();
    const uint32_t n = shared().stage_len[l];
    if (threadIdx.x == 0) shared().stage_at = n ? add_remote32(remote(&shared().list_len[l], 0), n) : 0;
    __syncthreads();
    const uint32_t at = shared().stage_at, lst = remote(shared().list[l], 0);
    for (uint32_t i = threadIdx.x; i < n && i < kList; i += kThreads)
      if (at + i < kList) st_remote64(lst + 8 * (at + i), shared().stage[l][i]);
    if (threadIdx.x == 0) shared().stage_len[l] = 0;
    __syncthreads();
  }

  // CTA 0: list l in falling order (key, then the lower id); returns its length.
  __device__ __noinline__ int sort_list(int l) const {
    Fixed& f = shared();
    u64* list = f.list[l];
    const int m = (int)min(f.list_len[l], (uint32_t)kList), t = threadIdx.x;
    if (m <= kShort) {
      // 8 threads count what precedes a token: its place
      const u64 x = t / 8 < m ? list[t / 8] : 0;
      int n = 0;
      for (int i = t % 8; i < m; i += 8) n += list[i] > x ? 1 : 0;
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
      __syncthreads();
      if (t % 8 == 0 && t / 8 < m) list[n] = x;
      __syncthreads();
      return m;
    }
    // buckets of the keys' range; within a bucket (a few tokens) each counts what
    // precedes it
    u64 x[kPer];
    uint32_t hi = 0, lo = 0xffffffffu;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      x[e] = t + e * kThreads < m ? list[t + e * kThreads] : 0;
      if (t + e * kThreads < m) hi = max(hi, (uint32_t)(x[e] >> 32)), lo = min(lo, (uint32_t)(x[e] >> 32));
    }
    hi = __reduce_max_sync(0xffffffffu, hi);
    lo = __reduce_min_sync(0xffffffffu, lo);
    __syncthreads();
    if ((t & 31) == 0) f.warp_sum[t >> 5] = ((u64)hi << 32) | lo;
    for (int i = t; i < kBins; i += kThreads) f.lo[i] = 0;
    __syncthreads();
    const u64 w = f.warp_sum[t & (kWarps - 1)];
    hi = __reduce_max_sync(0xffffffffu, (uint32_t)(w >> 32));
    lo = __reduce_min_sync(0xffffffffu, (uint32_t)w);
    int shift = 0;
    while (((hi - lo) >> shift) >= kBins) ++shift;
    int b[kPer], at[kPer];
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      b[e] = (int)((hi - (uint32_t)(x[e] >> 32)) >> shift);
      if (t + e * kThreads < m) at[e] = (int)atomicAdd(&f.lo[b[e]], 1u);
    }
    __syncthreads();
    constexpr int B = kBins / kThreads;
    u64 n = 0, total;
    uint32_t most = 0;
#pragma unroll
    for (int e = 0; e < B; ++e) n += f.lo[B * t + e], most = max(most, f.lo[B * t + e]);
    n = scan(n, total);
#pragma unroll
    for (int e = 0; e < B; ++e) {
      f.hi[B * t + e] = (uint32_t)n;
      n += f.lo[B * t + e];
    }
    if (__syncthreads_or(most > 64)) {
      bitonic(list, m);  // many equal keys
      return m;
    }
    u64* tmp = f.stage[l];
#pragma unroll
    for (int e = 0; e < kPer; ++e)
      if (t + e * kThreads < m) tmp[f.hi[b[e]] + at[e]] = x[e];
    __syncthreads();
#pragma unroll
    for (int e = 0; e < kPer; ++e)
      if (t + e * kThreads < m) {
        const uint32_t first = f.hi[b[e]], last = first + f.lo[b[e]];
        uint32_t r = first;
        for (uint32_t i = first; i < last; ++i) r += tmp[i] > x[e] ? 1 : 0;
        list[r] = x[e];
      }
    __syncthreads();
    return m;
  }
  __device__ __noinline__ static void bitonic(u64* list, int m) {
    const int t = threadIdx.x;
    int p = 2;
    while (p < m) p <<= 1;
    for (int i = m + t; i < p; i += kThreads) list[i] = 0;
    for (int k = 2; k <= p; k <<= 1)
      for (int j = k >> 1; j > 0; j >>= 1) {
        __syncthreads();
        if (t < p / 2) {  // kList / 2 = kThreads
          const int i = 2 * t - (t & (j - 1)), q = i + j;
          const u64 x = list[i], y = list[q];
          if ((x < y) == ((i & k) == 0)) list[i] = y, list[q] = x;
        }
      }
    __syncthreads();
  }
  // The rest of the list's work runs in one warp where the list is short (no
  // barriers of the whole CTA), else in all: N threads.
  template <int N> __device__ __forceinline__ u64 scan_n(u64 x, u64& total) const {
    if (N > 32) return scan(x, total);
    const int lane = threadIdx.x & 31;
    u64 in = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 q = __shfl_up_sync(0xffffffffu, in, o);
      if (lane >= o) in += q;
    }
    total = __shfl_sync(0xffffffffu, in, 31);
    return in - x;
  }
  __device__ __forceinline__ float list_value(int l, int i) const { return key_value((uint32_t)(shared().list[l][i] >> 32)); }
  __device__ __forceinline__ int list_id(int l, int i) const { return (int)~(uint32_t)shared().list[l][i]; }

  // Sum (or maximum) of a value over the cluster; the result to every thread.
  template <bool MAX> __device__ __noinline__ u64 reduce(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const u64 w = __shfl_xor_sync(0xffffffffu, v, o);
      v = MAX ? (w > v ? w : v) : v + w;
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) shared().warp_sum[threadIdx.x >> 5] = v;
    __syncthreads();
    v = shared().warp_sum[threadIdx.x & (kWarps - 1)];
#pragma unroll
    for (int o = kWarps / 2; o > 0; o >>= 1) {
      const u64 w = __shfl_xor_sync(0xffffffffu, v, o);
      v = MAX ? (w > v ? w : v) : v + w;
    }
    return across<MAX>(v);
  }
  // The same of a value per CTA.
  template <bool MAX> __device__ __forceinline__ u64 across(u64 v) {
    if (C == 1) return v;
    if (threadIdx.x < C) st_remote64(remote(&shared().part[parity_part][rank], threadIdx.x), v);
    sync();
    u64 t = 0;
#pragma unroll
    for (uint32_t r = 0; r < kMaxCluster; ++r) {
      const u64 w = r < C ? shared().part[parity_part][r] : 0;
      t = MAX ? (w > t ? w : t) : t + w;
    }
    parity_part ^= 1;  // the next write to this half comes after another barrier
    return t;
  }
  // The largest (key, ~id) over the cluster, the first index of the largest key; key 0: none.
  __device__ __noinline__ u64 best_of(uint32_t key, uint32_t not_id) {
    uint32_t k = __reduce_max_sync(0xffffffffu, key), i = __reduce_max_sync(0xffffffffu, key == k ? not_id : 0u);
    if ((threadIdx.x & 31) == 0) shared().warp_sum[threadIdx.x >> 5] = ((u64)k << 32) | i;
    __syncthreads();
    const u64 v = shared().warp_sum[threadIdx.x & (kWarps - 1)];
    k = __reduce_max_sync(0xffffffffu, (uint32_t)(v >> 32));
    i = __reduce_max_sync(0xffffffffu, (uint32_t)(v >> 32) == k ? (uint32_t)v : 0u);
    return across<true>(k ? ((u64)k << 32) | i : 0);
  }

  // Where a search ends: the mass up to and with the token that reaches the
  // target, that token's units and id (-1 in the CTAs that do not hold it).
  struct Place {
    u64 mass, w;
    int id;
  };

  // CTA 0: the place in list l, before which there is `before`.  by_count: the
  // target is the number of tokens, else the mass.
  __device__ __noinline__ Place in_list(int l, u64 before, bool by_count, u64 target) {
    Fixed& f = shared();
    const int m = sort_list(l);
    if (m > kShort) in_list_n<kThreads>(l, m, before, by_count, target);
    else if (threadIdx.x < 32) in_list_n<32>(l, m, before, by_count, target);
    __syncthreads();
    const Place r{f.hit[0], f.hit[1], list_id(l, f.picked)};
    if (threadIdx.x == 0) f.list_len[l] = 0;
    __syncthreads();
    return r;
  }
  template <int N>
  __device__ __forceinline__ void in_list_n(int l, int m, u64 before, bool by_count, u64 target) const {
    Fixed& f = shared();
    const Scale z = this->z;
    constexpr int E = N == 32 ? kShort / 32 : kPer;
    u64 w[E], s = 0, t;
    const int per = (m + N - 1) / N, first = (int)threadIdx.x * per;
#pragma unroll
    for (int j = 0; j < E; ++j) {
      w[j] = j < per && first + j < m ? z.units(list_value(l, first + j)) : 0;
      s += w[j];
    }
    s = scan_n<N>(s, t) + before;
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const bool here = by_count ? (u64)(first + j + 1) == target : s < target && target <= s + w[j];
      s += w[j];
      if (here && j < per && first + j < m) {
        f.picked = first + j;
        f.hit[0] = s;
        f.hit[1] = w[j];
      }
    }
  }
  __device__ __forceinline__ u64 tell(u64 v) {  // CTA 0's value to all
    if (C == 1) return v;
    if (rank == 0 && threadIdx.x < C) st_remote64(remote(&shared().answer[parity_answer], threadIdx.x), v);
    sync();
    v = shared().answer[parity_answer];
    parity_answer ^= 1;
    return v;
  }

  // The place among the tokens with keys in [klo, khi], `count` of them, however
  // many; the target counts them (by_count) or is a mass with `before` ahead of
  // them.  The histogram is used up.
  __device__ __noinline__ Place descend(uint32_t klo, uint32_t khi, u64 count, u64 before, bool by_count, u64 target) {
    const Scale z = this->z;
    bool one = false;
    while (count > kList) {
      // the tight range of the keys, then bins of that range
      key_range([&](float x) { return sort_key(x) >= klo && sort_key(x) <= khi; }, klo, khi);
      one = klo == khi;
      if (one) break;
      int shift = 0;
      while (((khi - klo) >> shift) >= kBins) ++shift;
      __syncthreads();
      clear_bins();
      each([&](float x, int) {
        const uint32_t k = sort_key(x);
        if (k >= klo && k <= khi) add_mass((int)((khi - k) >> shift), by_count ? 1ull : z.units(x));
      });
      merge();
      const Found b = search(by_count ? target : target - before);
      if (by_count) target -= b.before;
      else before += b.before;
      const uint32_t top_key = khi - (uint32_t)(b.bin << shift);
      const u64 low = (u64)top_key + 1 > (1ull << shift) ? (u64)top_key + 1 - (1ull << shift) : 0ull;
      klo = klo > low ? klo : (uint32_t)low;
      khi = top_key;
      u64 c = 0;
      each([&](float x, int) { c += sort_key(x) >= klo && sort_key(x) <= khi ? 1 : 0; });
      count = reduce<false>(c);
    }
    if (by_count) {
      u64 s = 0;
      each([&](float x, int) {
        if (sort_key(x) > khi) s += z.units(x);
      });
      before = reduce<false>(s);
    }
    if (one) return ties(klo, before, by_count, target);
    each([&](float x, int i) {
      if (sort_key(x) >= klo && sort_key(x) <= khi) stage_one(0, x, i);
    });
    collect(0);
    sync();
    Place r{0, 0, -1};
    if (rank == 0) r = in_list(0, before, by_count, target);
    r.mass = tell(r.mass);
    return r;
  }
  template <typename Member> __device__ __forceinline__ void key_range(Member member, uint32_t& klo, uint32_t& khi) {
    u64 mx = 0, mn = 0;
    each([&](float x, int) {
      if (member(x)) {
        const u64 k = sort_key(x);
        mx = k > mx ? k : mx;
        mn = 0xffffffffu - k > mn ? 0xffffffffu - k : mn;
      }
    });
    khi = (uint32_t)reduce<true>(mx);
    klo = 0xffffffffu - (uint32_t)reduce<true>(mn);
  }
  // The weights' histogram, merged; the sum of all.
  __device__ __noinline__ u64 weigh() {
    const Scale z = this->z;
    each([&](float x, int) {
      const int b = z.bin(x);
      add_mass(b, z.units(x, b));
    });
    return merge();
  }
  // The place in bin b (`before` ahead of it) of more than kList tokens; b < 0: it
  // has to be searched again.
  __device__ __noinline__ Place bin_place(int b, u64 before, u64 target) {
    const Scale z = this->z;
    if (b < 0) {
      __syncthreads();
      clear_bins();
      weigh();
      const Found at = search(target);
      b = (int)at.bin;
      before = at.before;
    }
    u64 c = 0;
    each([&](float x, int) { c += z.bin(x) == b ? 1 : 0; });
    const u64 count = reduce<false>(c);
    uint32_t klo, khi;
    key_range([&](float x) { return z.bin(x) == b; }, klo, khi);
    return descend(klo, khi, count, before, false, target);
  }
  // One value: its tokens count in id order.
  __device__ __noinline__ Place ties(uint32_t key, u64 before, bool by_count, u64 target) {
    const u64 w = z.units(key_value(key));
    const u64 nth = by_count ? target : (target - before + w - 1) / w;  // 1 ..: how many of them reach the target
    Place r{before + nth * w, w, -1};
    u64 mine = 0;
    for (int i = threadIdx.x; i < len; i += kThreads) mine += sort_key(get(i)) == key ? 1 : 0;
    u64 all, got;
    scan(mine, all);
    if (threadIdx.x < C) st_remote64(remote(&shared().part[parity_part][rank], threadIdx.x), all);
    sync();
    u64 ahead = 0;
    for (uint32_t q = 0; q < rank; ++q) ahead += shared().part[parity_part][q];
    parity_part ^= 1;
    if (nth > ahead && nth <= ahead + all) {  // in this slice
      u64 want = nth - ahead;
      for (int i0 = 0; i0 < len && want; i0 += kThreads) {
        const int i = i0 + (int)threadIdx.x;
        const u64 hit = i < len && sort_key(get(i)) == key ? 1 : 0;
        const u64 h = scan(hit, got);
        if (want <= got) {
          if (hit && h + 1 == want) shared().picked = base + i;
          want = 0;
        } else {
          want -= got;
        }
      }
      __syncthreads();
      r.id = shared().picked;
    }
    sync();
    return r;
  }

  // With the first k tokens in CTA 0's list: all filters and the pick.
  __device__ __noinline__ void finish_short(int row, int k, float p, float mp, float uf) const {
    const int m = sort_list(0);
    if (m > kShort) finish_n<kThreads>(row, m, k, p, mp, uf);
    else if (threadIdx.x < 32) finish_n<32>(row, m, k, p, mp, uf);
  }
  template <int N> __device__ __forceinline__ void finish_n(int row, int m, int k, float p, float mp, float uf) const {
    const Scale z = this->z;
    m = min(m, k);
    constexpr int E = N == 32 ? kShort / 32 : kPer;
    const int per = (m + N - 1) / N, first = (int)threadIdx.x * per;
    const double lim = mp > 0.f ? fmin((double)mp, 1.0) : 0.0;
    u64 w[E], s = 0, t;
    bool in[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const bool on = e < per && first + e < m;
      const float x = on ? list_value(0, first + e) : -INFINITY;
      w[e] = on ? z.units(x) : 0;
      in[e] = on && (lim == 0.0 || z.weight(x) >= lim);
      s += w[e];
    }
    s = scan_n<N>(s, t);
    const u64 limit = p < 1.f ? target_of(p, t) : t;  // tokens whose preceding mass is below it are kept
    u64 kept = 0, before = s;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (in[e] && before < limit) kept += w[e];
      before += w[e];
    }
    u64 total;
    scan_n<N>(kept, total);
    const u64 x = pick_of(uf, total);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (s < x && x <= s + w[e]) put(row, list_id(0, first + e), w[e], total);
      s += w[e];
    }
  }
  // The mass that top-p asks for, and the one that the token has to reach: above u times the kept.
  __device__ __forceinline__ static u64 target_of(float p, u64 mass) {
    const double want = ceil(fmax((double)p, 0.0) * (double)mass);
    return want < 1.0 ? 1 : (u64)want < mass ? (u64)want : mass;
  }
  __device__ __forceinline__ static u64 pick_of(float u, u64 kept) {
    const u64 x = u > 0.f ? (u64)((double)u * (double)kept) : 0;
    return (x < kept ? x : kept - 1) + 1;
  }
  __device__ __forceinline__ void put(int row, int id, u64 w, u64 kept) const {
    a.ids[row] = id;
    if (a.probs) a.probs[row] = (float)((double)w / (double)kept);
  }
};

__global__ void __launch_bounds__(kThreads, 1) sample_rows_kernel(SampleArgs a) {
  Fixed& f = shared();
  const uint32_t C = ptx::cluster_nctarank(), rank = ptx::cluster_ctarank();
  const int tid = threadIdx.x, j = (int)(blockIdx.x / C);
  Row r{a};
  r.rank = rank;
  r.C = C;
  r.base = (int)rank * a.slice;
  r.len = max(0, min(a.slice, a.n - r.base));
  r.src = a.logits + (long long)j * a.ld + r.base;
  r.head = min((int)((16 - ((uintptr_t)r.src & 15)) & 15) >> 2, r.len);
  // the resident copy keeps the global one's place within 16 bytes
  r.slice = a.resident ? reinterpret_cast<float*>(smem + sizeof(Fixed)) + (((uintptr_t)r.src & 15) >> 2) : nullptr;
  r.infinite = false;
  for (int i = tid; i < (1 << kExpBits); i += kThreads) f.exp_table[i] = exp2((double)i / (1 << kExpBits));
  for (int i = tid; i < kBins; i += kThreads) f.lo[i] = f.hi[i] = 0;
  if (tid < 2) f.list_len[tid] = f.stage_len[tid] = 0;
  if (tid == 0) f.picked = 0;
  // every CTA of the cluster runs before another writes to its shared memory
  asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");
  pdl_wait();
  const float temp = a.temperature[j];
  const int k = a.top_k ? a.top_k[j] : 0;
  const float p = a.top_p ? a.top_p[j] : 1.f, mp = a.min_p ? a.min_p[j] : 0.f, uf = a.u[j];

  // 1. the row's maximum, and the slice
  float best = -INFINITY;
  int at = 0;
  {
    const int n4 = (r.len - r.head) >> 2, tail = r.head + 4 * n4;
    const int i1 = tid < r.head ? tid : tail + tid - r.head;
    if (tid < r.head + r.len - tail) {
      const float x = clean(__ldg(r.src + i1));
      if (r.slice) r.slice[i1] = x;
      if (x > best) best = x, at = i1;
    }
#pragma unroll 4
    for (int v = tid; v < n4; v += kThreads) {
      const int i = r.head + 4 * v;
      float4 x = __ldg(reinterpret_cast<const float4*>(r.src + i));
      x.x = clean(x.x); x.y = clean(x.y); x.z = clean(x.z); x.w = clean(x.w);
      if (r.slice) *reinterpret_cast<float4*>(r.slice + i) = x;
      const float m = fmaxf(fmaxf(x.x, x.y), fmaxf(x.z, x.w));
      // the first index of this thread's maximum; its odd token may lie on either side
      if (m > best || (m == best && i < at)) {
        best = m;
        at = i + (x.x == m ? 0 : x.y == m ? 1 : x.z == m ? 2 : 3);
      }
    }
  }
  asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
  const u64 whole = r.best_of(best > -INFINITY ? sort_key(best) : 0u, (uint32_t)~(r.base + at));
  if (whole == 0 || !(temp > 0.f)) {  // nothing to take, or greedy
    if (rank == 0 && tid == 0) {
      a.ids[j] = whole ? (int)~(uint32_t)whole : -1;
      if (a.probs) a.probs[j] = whole ? 1.f : 0.f;
    }
    pdl_launch_dependents();
    return;
  }
  r.z.top = key_value((uint32_t)(whole >> 32));
  if (r.z.top == INFINITY) {  // the infinite ones share everything
    r.infinite = true;
    r.z.top = 0.f;
    if (r.slice)
      for (int i = tid; i < r.len; i += kThreads) r.slice[i] = r.slice[i] == INFINITY ? 0.f : -INFINITY;
  }
  r.z.bin_scale = fminf(kBinsPerNat / temp, FLT_MAX);
  r.z.to_table = (double)(1 << kExpBits) * 1.4426950408889634 / (double)temp;
  r.z.log2 = a.scale_log2;
  const Scale z = r.z;
  __syncthreads();

  const bool some = k > 0 && k < a.n;
  u64 mass_k = 0;
  if (some) {
    r.each([&](float x, int) { atomicAdd(&f.lo[z.bin(x)], 1u); });
    r.merge();
    const Found b = r.search((u64)k);
    const int last = b.bin;
    if (b.before + b.in <= kList) {
      r.each([=](float x, int i) {
        if (z.bin(x) <= last) r.stage_one(0, x, i);
      });
      r.collect(0);
      r.sync();
      if (rank == 0) r.finish_short(j, k, p, mp, uf);
      pdl_launch_dependents();
      return;
    }
    // a long top-k: the place of the k-th token in its bin, and the mass up to it
    uint32_t klo, khi;
    r.key_range([&](float x) { return z.bin(x) == last; }, klo, khi);
    mass_k = r.descend(klo, khi, b.in, 0, true, (u64)k - b.before).mass;
    __syncthreads();
    r.clear_bins();
  }
  // 2. the weights' histogram
  const u64 all = r.weigh();
  const u64 mass = some ? mass_k : all;
  u64 kept = mass;
  if (mp > 0.f) {
    const double lim = fmin((double)mp, 1.0);
    // beyond this bin every weight is below lim (a bin more for its rounding)
    const int last = (int)fmin(-log(lim) * kBinsPerNat + 2.0, (double)kBins);
    u64 s = 0;
    r.each([&](float x, int) {
      const int b = z.bin(x);
      if (b <= last && z.weight(x) >= lim) s += z.units(x, b);
    });
    s = r.reduce<false>(s);
    kept = s < kept ? s : kept;
  }
  // 3. the bins of top-p's border and of the token, whose mass lies between the
  // picks from the least and the most that can be kept
  const bool cut = p < 1.f && Row::target_of(p, mass) <= kept;
  const u64 target = cut ? Row::target_of(p, mass) : kept;
  const Found b = r.search(target);
  const u64 most = cut ? (kept < b.before + b.in ? kept : b.before + b.in) : kept;
  r.search(Row::pick_of(uf, target), Row::pick_of(uf, most));
  const u64 u_before = f.found[0].before;
  const int cut_bin = cut ? b.bin : -1, u_lo = f.found[0].bin, u_hi = f.found[1].bin;
  r.each([=](float x, int i) {
    const int d = z.bin(x);
    if (d == cut_bin) r.stage_one(0, x, i);
    if (d >= u_lo && d <= u_hi) r.stage_one(1, x, i);
  });
  __syncthreads();
  const u64 staged = r.reduce<false>(tid == 0 ? f.stage_len[0] + ((u64)f.stage_len[1] << 32) : 0);
  if ((uint32_t)staged <= kList && (staged >> 32) <= kList) {
    if (cut) r.collect(0);
    r.collect(1);
    r.sync();
    if (rank == 0) {
      if (cut) {
        const u64 m = r.in_list(0, b.before, false, target).mass;
        kept = m < kept ? m : kept;
      }
      const Row::Place got = r.in_list(1, u_before, false, Row::pick_of(uf, kept));
      if (tid == 0) r.put(j, got.id, got.w, kept);
    }
    pdl_launch_dependents();
    return;
  }
  __syncthreads();
  if (tid < 2) f.stage_len[tid] = 0;
  if (cut) {
    const u64 m = r.bin_place(b.bin, b.before, target).mass;
    kept = m < kept ? m : kept;
  }
  const u64 x = Row::pick_of(uf, kept);
  const Row::Place got = r.bin_place(-1, 0, x);
  if (got.id >= 0 && tid == 0) r.put(j, got.id, got.w, kept);
  pdl_launch_dependents();
}

constexpr size_t kSliceMax = 104 * 1024;  // bytes of a resident slice: 117 KB of tables beside it, up to 227 KB

}  // namespace
}  // namespace pyr

using namespace pyr;

extern "C" {

int pyrite_cuda_sample_rows(const float* logits, long long ld, size_t n, size_t count, const float* uniforms,
                            const float* temperature, const int* top_k, const float* top_p, const float* min_p,
                            int* ids, float* probs, void* stream) {
  if (!logits || !uniforms || !temperature || !ids) return PYRITE_E_BUFFER;
  if (n == 0 || n > (1u << 20) || count == 0 || count > 65535 || ld < (long long)n || ((uintptr_t)logits & 3))
    return PYRITE_E_SHAPE;
  int bits = 0;
  while ((1u << bits) < n) ++bits;
  // CTAs a row: as many as find an SM each, of at least 1024 tokens
  int cluster = 1;
  while (cluster < kMaxCluster && count * cluster * 2 <= 144 && n > 1024u * cluster) cluster *= 2;
  const size_t slice = ((n + cluster - 1) / cluster + 3) & ~(size_t)3;
  const bool resident = slice * sizeof(float) <= kSliceMax;
  const size_t smem = sizeof(Fixed) + (resident ? slice * sizeof(float) + 16 : 0);
  static_assert(8 * kShort <= kThreads && kList <= 2 * kThreads, "threads of the sorts");
  static_assert(sizeof(Fixed) + kSliceMax + 16 <= 227 * 1024, "tables and slice fit one CTA's shared memory");
  static std::atomic<bool> smem_set[64];  // idempotent: concurrent first calls only repeat it
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return PYRITE_E_CUDA;
  if (!smem_set[dev].load(std::memory_order_acquire)) {
    if (launch_code(cudaFuncSetAttribute(sample_rows_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024)))
      return PYRITE_E_CUDA;
    smem_set[dev].store(true, std::memory_order_release);
  }
  const SampleArgs a{logits, ld,    (int)n, (int)slice, resident ? 1 : 0, uniforms, temperature,
                     top_k,  top_p, min_p,  ids,        probs,            bits <= 18 ? 44 : 62 - bits};
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(count * cluster));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return launch_code(cudaLaunchKernelEx(&cfg, sample_rows_kernel, a)) ? PYRITE_E_CUDA : 0;
}

}  // extern "C"
