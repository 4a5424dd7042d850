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
#include <atomic>
#include <cfloat>

#include "kernels.cuh"
#include "ptx.cuh"
#include "../../include/pyrite_b200.h"

namespace pyr {
namespace {

typedef unsigned long long u64;

// A row belongs to a cluster of C CTAs, each holding a slice of it in shared
// memory (read from HBM once); what the searches need crosses the cluster
// through distributed shared memory.
//   1. slice -> shared memory, the row's maximum (first index) over the cluster.
//   2. Histogram over bins of (max - l) / T, 1/64 wide: counts, and where the
//      search is by weight the weights' integers too (two 32-bit words with the
//      carry passed on: shared memory adds 32-bit integers natively).  Each CTA
//      merges and scans a share of the bins, so a search is one comparison a bin.
//   3. The bin where the target is passed: its tokens are gathered into CTA 0,
//      sorted and scanned.  A bin of more than kList tokens (ties, coarse logits)
//      is divided again by the bits of its keys until it is short or one value,
//      whose tokens count in id order.
// With a short top-k (the usual case) step 2 counts only, step 3 gathers all
// first k at once and CTA 0 finishes alone: no weight is computed for the rest
// of the vocabulary.
constexpr int kThreads = 512;
constexpr int kBins = 2048;
constexpr float kBinsPerNat = 64.f;
constexpr int kList = 2048;
constexpr int kExpBits = 8;  // table of 2^(j / 256)

__device__ __forceinline__ uint32_t sort_key(float x) {  // orders as the floats do (no NaN, no -0)
  const uint32_t b = __float_as_uint(x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ float clean(float x) { return x > -INFINITY ? x + 0.f : -INFINITY; }  // NaN: -inf; -0: 0

struct SampleArgs {
  const float* logits;
  long long ld;
  int n;
  int slice;     // tokens of a CTA (multiple of 4)
  int resident;  // slices are kept in shared memory; else each pass reads them from L2
  const float* u;
  const float* temperature;
  const int* top_k;
  const float* top_p;
  const float* min_p;
  int* ids;
  float* probs;
  int scale_log2;  // S
};

// ---- distributed shared memory ------------------------------------------------------------
__device__ __forceinline__ uint32_t remote(const void* p, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(ptx::smem_addr(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ uint32_t ld_remote32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void st_remote64(uint32_t a, u64 v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(a), "l"(v) : "memory");
}
__device__ __forceinline__ uint32_t add_remote32(uint32_t a, uint32_t v) {
  uint32_t o;
  asm volatile("atom.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(o) : "r"(a), "r"(v) : "memory");
  return o;
}

struct Found {  // the bin of a search: what precedes it, what it holds
  u64 bin, count, before_count, before_mass;
};

// Shared memory of one CTA.  The merged share's size depends on the cluster.
struct alignas(16) Fixed {
  double exp_table[1 << kExpBits];
  uint32_t cnt[kBins], lo[kBins], hi[kBins];  // this CTA's histogram
  u64 list[kList];                            // CTA 0: gathered tokens (key, ~id)
  Found found[2];                             // written by the CTA that owns the bin
  u64 tot_count[8], tot_mass[8];              // each CTA's share of the bins
  u64 best[8];                                // each CTA's largest (key, ~id), or reduction operand
  u64 answer[2];                              // CTA 0 to all
  u64 warp_a[kThreads / 32], warp_b[kThreads / 32];
  uint32_t list_len;
  int picked;
};

struct Row {
  const SampleArgs& a;
  Fixed& f;
  u64* e_count;  // [share + 1] counts before each bin of this CTA's share, [..] masses
  u64* e_mass;
  const float* slice;
  const float* src;  // the slice in global memory
  uint32_t rank, C;
  int len, base;     // tokens of this slice, its first id
  float top;
  float bin_scale;
  double to_table;   // 256 log2(e) / T
  int parity = 0;

  __device__ __forceinline__ float get(int i) const { return slice ? slice[i] : clean(__ldg(src + i)); }

  // Bins fall with the logit; rounding keeps the order (each step is monotonic).
  __device__ __forceinline__ int bin(float x) const {
    if (x == top) return 0;
    const float t = (top - x) * bin_scale;
    return t < (float)(kBins - 1) ? (int)t : kBins - 1;
  }
  // e^((x - max) / T) by a table of 2^(j/256) and a cubic for the rest (Tang's
  // table-driven method): |rest| <= ln2 / 512, so the first term left out is
  // below 1.5e-13 relative.
  __device__ __forceinline__ double weight(float x) const {
    if (x == top) return 1.0;
    const double t = ((double)x - (double)top) * to_table;
    if (!(t > -256.0 * 64.0)) return 0.0;  // below 2^-64, far less than half a unit
    const double magic = 6755399441055744.0;  // 1.5 * 2^52: the sum's low word is the rounded integer
    const double s = t + magic;
    const int k = __double2loint(s);
    const double g = t - (s - magic);
    constexpr double c1 = 0.0027076061740622863, c2 = c1 * c1 / 2, c3 = c1 * c1 * c1 / 6;  // ln2 / 256
    const double q = g * fma(g, fma(g, c3, c2), c1);
    const double w = fma(f.exp_table[k & 255], q, f.exp_table[k & 255]);
    return __hiloint2double(__double2hiint(w) + ((k >> kExpBits) << 20), __double2loint(w));
  }
  __device__ __forceinline__ u64 units(float x) const {
    return (u64)__double2ull_rn(weight(x) * (double)(1ull << a.scale_log2));
  }
  __device__ __forceinline__ void sync() const { ptx::cluster_sync(); }

  __device__ __forceinline__ void clear_bins() const {
    for (int i = threadIdx.x; i < kBins; i += kThreads) f.cnt[i] = f.lo[i] = f.hi[i] = 0;
    __syncthreads();
  }
  __device__ __forceinline__ void add_bin(int b, bool with_mass, float x) const {
    atomicAdd(&f.cnt[b], 1u);
    if (with_mass) {
      const u64 w = units(x);
      const uint32_t l = (uint32_t)w;
      uint32_t h = (uint32_t)(w >> 32);
      if (l) h += atomicAdd(&f.lo[b], l) > ~l ? 1u : 0u;
      if (h) atomicAdd(&f.hi[b], h);
    }
  }

  // Exclusive scan of two values a thread over the CTA; totals to every thread.
  __device__ __forceinline__ void scan2(u64& x, u64& y, u64& tx, u64& ty) const {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    u64 ix = x, iy = y;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 px = __shfl_up_sync(0xffffffffu, ix, o), py = __shfl_up_sync(0xffffffffu, iy, o);
      if (lane >= o) ix += px, iy += py;
    }
    __syncthreads();
    if (lane == 31) f.warp_a[warp] = ix, f.warp_b[warp] = iy;
    __syncthreads();
    u64 bx = 0, by = 0;
    tx = ty = 0;
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w == warp) bx = tx, by = ty;
      tx += f.warp_a[w];
      ty += f.warp_b[w];
    }
    x = bx + ix - x;
    y = by + iy - y;
  }

  // Histograms of all CTAs -> scanned shares; totals.  The histograms are free afterwards.
  __device__ void merge(u64& total_count, u64& total_mass) {
    const int share = kBins / (int)C, per = share > kThreads ? share / kThreads : 1;
    const int b0 = (int)rank * share;
    sync();
    u64 c[kBins / kThreads], m[kBins / kThreads], sc = 0, sm = 0;
#pragma unroll
    for (int j = 0; j < kBins / kThreads; ++j) {
      c[j] = m[j] = 0;
      const int i = (int)threadIdx.x * per + j;
      if (j < per && i < share)
        for (uint32_t r = 0; r < C; ++r) {
          c[j] += ld_remote32(remote(&f.cnt[b0 + i], r));
          m[j] += ld_remote32(remote(&f.lo[b0 + i], r)) + ((u64)ld_remote32(remote(&f.hi[b0 + i], r)) << 32);
        }
      sc += c[j];
      sm += m[j];
    }
    u64 tc, tm;
    scan2(sc, sm, tc, tm);
    if (threadIdx.x < C) {
      st_remote64(remote(&f.tot_count[rank], threadIdx.x), tc);
      st_remote64(remote(&f.tot_mass[rank], threadIdx.x), tm);
    }
    sync();
    u64 bc = 0, bm = 0;
    total_count = total_mass = 0;
    for (uint32_t r = 0; r < C; ++r) {
      if (r == rank) bc = total_count, bm = total_mass;
      total_count += f.tot_count[r];
      total_mass += f.tot_mass[r];
    }
    sc += bc;
    sm += bm;
#pragma unroll
    for (int j = 0; j < kBins / kThreads; ++j) {
      const int i = (int)threadIdx.x * per + j;
      if (j < per && i < share) {
        e_count[i] = sc;
        e_mass[i] = sm;
        sc += c[j];
        sm += m[j];
        if (i == share - 1) e_count[share] = sc, e_mass[share] = sm;
      }
    }
    __syncthreads();
  }

  // The bin in which the cumulative count (or mass) reaches target (1 .. total).
  __device__ Found search(const u64* ec, const u64* em, bool by_count, u64 target) {
    const int share = kBins / (int)C;
    const u64* e = by_count ? ec : em;
    for (int i = threadIdx.x; i < share; i += kThreads)
      if (e[i] < target && target <= e[i + 1]) {
        for (uint32_t r = 0; r < C; ++r) {
          const uint32_t d = remote(&f.found[parity], r);
          st_remote64(d, (u64)((int)rank * share + i));
          st_remote64(d + 8, ec[i + 1] - ec[i]);
          st_remote64(d + 16, ec[i]);
          st_remote64(d + 24, em[i]);
        }
      }
    sync();
    const Found r = f.found[parity];
    parity ^= 1;
    return r;
  }

  // Tokens whose bin (or key) lies in [lo, hi] -> CTA 0's list.
  template <typename Member> __device__ void gather(Member member) {
    const uint32_t lst = remote(f.list, 0), len_at = remote(&f.list_len, 0);
    const int lane = threadIdx.x & 31;
    for (int i0 = (int)(threadIdx.x & ~31u); i0 < len; i0 += kThreads) {
      const int i = i0 + lane;
      const float x = i < len ? get(i) : 0.f;
      const bool in = i < len && member(x);
      const unsigned vote = __ballot_sync(0xffffffffu, in);
      if (!vote) continue;
      uint32_t at = 0;
      if (lane == 0) at = add_remote32(len_at, (uint32_t)__popc(vote));
      at = __shfl_sync(0xffffffffu, at, 0) + (uint32_t)__popc(vote & ((1u << lane) - 1u));
      if (in && at < kList) st_remote64(lst + 8 * at, ((u64)sort_key(x) << 32) | (uint32_t)~(base + i));
    }
    sync();
  }

  // CTA 0: the list in falling order (key, then the lower id).
  __device__ int sort_list() const {
    const int m = (int)min(f.list_len, (uint32_t)kList);
    int p = 2;
    while (p < m) p <<= 1;
    for (int i = m + (int)threadIdx.x; i < p; i += kThreads) f.list[i] = 0;
    for (int k = 2; k <= p; k <<= 1)
      for (int j = k >> 1; j > 0; j >>= 1) {
        __syncthreads();
        for (int t = threadIdx.x; t < p / 2; t += kThreads) {
          const int i = 2 * t - (t & (j - 1)), l = i + j;
          const u64 x = f.list[i], y = f.list[l];
          if ((x < y) == ((i & k) == 0)) f.list[i] = y, f.list[l] = x;
        }
      }
    __syncthreads();
    return m;
  }
  __device__ __forceinline__ float list_value(int i) const { return key_value((uint32_t)(f.list[i] >> 32)); }
  __device__ __forceinline__ int list_id(int i) const { return (int)~(uint32_t)f.list[i]; }

  // Sum (or maximum) of a value over the cluster; the result to every thread.
  template <bool MAX> __device__ u64 reduce(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const u64 w = __shfl_xor_sync(0xffffffffu, v, o);
      v = MAX ? (w > v ? w : v) : v + w;
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) f.warp_a[threadIdx.x >> 5] = v;
    __syncthreads();
    v = f.warp_a[threadIdx.x & (kThreads / 32 - 1)];
#pragma unroll
    for (int o = kThreads / 64; o > 0; o >>= 1) {
      const u64 w = __shfl_xor_sync(0xffffffffu, v, o);
      v = MAX ? (w > v ? w : v) : v + w;
    }
    if (C == 1) return v;
    if (threadIdx.x < C) st_remote64(remote(&f.best[rank], threadIdx.x), v);
    sync();
    u64 t = 0;
    for (uint32_t r = 0; r < C; ++r) {
      const u64 w = f.best[r];
      t = MAX ? (w > t ? w : t) : t + w;
    }
    sync();  // best is free again
    return t;
  }

  // The position `in_bin` tokens (by_count) or `target` units of mass into a bin:
  // by_count: the mass of everything up to there; else the mass up to and with
  // the token that reaches target; that token to id / units (pick only).
  struct Place {
    u64 mass, w;
    int id;
  };
  __device__ Place resolve(Found b, bool by_count, u64 target, bool pick) {
    uint32_t klo = 0, khi = 0xffffffffu;
    const int level0 = (int)b.bin;
    bool by_key = false;
    auto member = [&](float x) {
      if (!by_key) return bin(x) == level0;
      const uint32_t k = sort_key(x);
      return k >= klo && k <= khi;
    };
    while (b.count > kList) {
      // a long bin: the range of its keys, then bins of that range
      u64 mx = 0, mn = 0;
      for (int i = threadIdx.x; i < len; i += kThreads) {
        const float x = get(i);
        if (member(x)) {
          const u64 k = sort_key(x);
          mx = k > mx ? k : mx;
          mn = 0xffffffffu - k > mn ? 0xffffffffu - k : mn;
        }
      }
      khi = (uint32_t)reduce<true>(mx);
      klo = 0xffffffffu - (uint32_t)reduce<true>(mn);
      by_key = true;
      if (klo == khi) return ties(b, klo, by_count, target, pick);
      int shift = 0;
      while (((khi - klo) >> shift) >= kBins) ++shift;
      clear_bins();
      for (int i = threadIdx.x; i < len; i += kThreads) {
        const float x = get(i);
        if (member(x)) add_bin((int)((khi - sort_key(x)) >> shift), true, x);
      }
      const u64 bc = b.before_count, bm = b.before_mass;
      u64 *keep_c = e_count, *keep_m = e_mass, tc, tm;
      e_count += kBins / C + 1;  // the second pair of shares: the first stays for later searches
      e_mass += kBins / C + 1;
      merge(tc, tm);
      b = search(e_count, e_mass, by_count, by_count ? target - bc : target - bm);
      e_count = keep_c;
      e_mass = keep_m;
      b.before_count += bc;
      b.before_mass += bm;
      const uint32_t top_key = khi - (uint32_t)(b.bin << shift);
      klo = max((u64)klo, (u64)top_key + 1 > (1ull << shift) ? (u64)top_key + 1 - (1ull << shift) : 0ull);
      khi = top_key;
    }
    gather(member);
    Place r{0, 0, -1};
    if (rank == 0) {
      const int m = sort_list();
      u64 w[kList / kThreads], s = 0, zero = 0, t, tz;
#pragma unroll
      for (int j = 0; j < kList / kThreads; ++j) {
        const int i = (int)threadIdx.x * (kList / kThreads) + j;
        w[j] = i < m ? units(list_value(i)) : 0;
        s += w[j];
      }
      scan2(s, zero, t, tz);
      s += b.before_mass;
#pragma unroll
      for (int j = 0; j < kList / kThreads; ++j) {
        const int i = (int)threadIdx.x * (kList / kThreads) + j;
        const bool here = by_count ? b.before_count + i + 1 == target : s < target && target <= s + w[j];
        s += w[j];
        if (here && i < m) {
          f.picked = i;
          f.answer[0] = s;
          f.answer[1] = w[j];
        }
      }
      __syncthreads();
      if (pick) {
        r = Place{f.answer[0], f.answer[1], list_id(f.picked)};
        return r;
      }
      if (threadIdx.x == 0) {
        f.list_len = 0;
        for (uint32_t q = 1; q < C; ++q) st_remote64(remote(&f.answer[0], q), f.answer[0]);
      }
    }
    if (pick) return r;
    sync();
    r.mass = f.answer[0];
    sync();  // answer is free again
    return r;
  }
  // All of a bin has one value: its tokens count in id order.
  __device__ Place ties(const Found& b, uint32_t key, bool by_count, u64 target, bool pick) {
    const u64 w = units(key_value(key));
    Place r{0, w, -1};
    if (by_count) {
      r.mass = b.before_mass + (target - b.before_count) * w;
      return r;
    }
    u64 nth = (target - b.before_mass + w - 1) / w;  // 1 ..: how many of them reach target
    r.mass = b.before_mass + nth * w;
    if (!pick) return r;
    u64 mine = 0;
    for (int i = threadIdx.x; i < len; i += kThreads) mine += sort_key(get(i)) == key ? 1 : 0;
    u64 z = 0, all, tz;
    scan2(mine, z, all, tz);
    if (threadIdx.x < C) st_remote64(remote(&f.best[rank], threadIdx.x), all);
    if (threadIdx.x == 0) f.picked = -1;
    sync();
    u64 before = 0;
    for (uint32_t q = 0; q < rank; ++q) before += f.best[q];
    if (nth > before && nth <= before + all) {  // in this slice
      u64 want = nth - before;
      for (int i0 = 0; i0 < len && want; i0 += kThreads) {
        const int i = i0 + (int)threadIdx.x;
        u64 hit = i < len && sort_key(get(i)) == key ? 1 : 0, h = hit, got;
        z = 0;
        scan2(h, z, got, tz);
        if (want <= got) {
          if (hit && h + 1 == want) f.picked = base + i;
          want = 0;
        } else {
          want -= got;
        }
      }
      __syncthreads();
      r.id = f.picked;
    }
    return r;  // id on the CTA that holds it
  }
};

__global__ void __launch_bounds__(kThreads, 2) sample_rows_kernel(SampleArgs a) {
  extern __shared__ __align__(16) uint8_t smem[];
  Fixed& f = *reinterpret_cast<Fixed*>(smem);
  const uint32_t C = ptx::cluster_nctarank(), rank = ptx::cluster_ctarank();
  u64* shares = reinterpret_cast<u64*>(smem + sizeof(Fixed));
  const int per = kBins / (int)C + 1;
  const int tid = threadIdx.x, j = (int)(blockIdx.x / C);
  Row r{a, f};
  r.e_count = shares;             // [2][per]: level 0, refinement
  r.e_mass = shares + 2 * per;    // [2][per]
  float* sl = reinterpret_cast<float*>(shares + 4 * per);
  r.rank = rank;
  r.C = C;
  r.base = (int)rank * a.slice;
  r.len = max(0, min(a.slice, a.n - r.base));
  r.src = a.logits + (long long)j * a.ld + r.base;
  r.slice = nullptr;
  if (tid == 0) f.list_len = 0;
  for (int i = tid; i < (1 << kExpBits); i += kThreads) f.exp_table[i] = exp2((double)i / (1 << kExpBits));
  for (int i = tid; i < kBins; i += kThreads) f.cnt[i] = f.lo[i] = f.hi[i] = 0;
  // every CTA of the cluster runs before another writes to its shared memory
  asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");
  pdl_wait();
  const float temp = a.temperature[j];
  const int k = a.top_k ? a.top_k[j] : 0;
  const float p = a.top_p ? a.top_p[j] : 1.f, mp = a.min_p ? a.min_p[j] : 0.f, uf = a.u[j];

  // 1. the slice and the row's maximum
  float best = -INFINITY;
  int at = 0;
  const bool vec = a.resident && ((uintptr_t)r.src & 15) == 0;
  if (vec) {
    const int n4 = r.len >> 2;
    const float4* s4 = reinterpret_cast<const float4*>(r.src);
#pragma unroll 4
    for (int i = tid; i < n4; i += kThreads) {
      float4 x = __ldcs(s4 + i);
      x.x = clean(x.x); x.y = clean(x.y); x.z = clean(x.z); x.w = clean(x.w);
      reinterpret_cast<float4*>(sl)[i] = x;
      if (x.x > best) best = x.x, at = 4 * i;
      if (x.y > best) best = x.y, at = 4 * i + 1;
      if (x.z > best) best = x.z, at = 4 * i + 2;
      if (x.w > best) best = x.w, at = 4 * i + 3;
    }
  }
#pragma unroll 4
  for (int i = (vec ? r.len & ~3 : 0) + tid; i < r.len; i += kThreads) {
    const float x = clean(__ldg(r.src + i));
    if (a.resident) sl[i] = x;
    if (x > best) best = x, at = i;
  }
  if (a.resident) r.slice = sl;
  asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
  // the largest (key, ~id) over the cluster: the first index of the maximum
  const u64 whole = r.reduce<true>(best > -INFINITY ? ((u64)sort_key(best) << 32) | (uint32_t)~(r.base + at) : 0);
  if (whole == 0 || !(temp > 0.f)) {  // nothing to take, or greedy
    if (rank == 0 && tid == 0) {
      a.ids[j] = whole ? (int)~(uint32_t)whole : -1;
      if (a.probs) a.probs[j] = whole ? 1.f : 0.f;
    }
    pdl_launch_dependents();
    return;
  }
  r.top = key_value((uint32_t)(whole >> 32));
  r.bin_scale = fminf(kBinsPerNat / temp, FLT_MAX);
  r.to_table = 256.0 * 1.4426950408889634 / (double)temp;
  __syncthreads();

  // the kept mass, then the token at u of it; CTA 0 has the list of the first k tokens when it is short
  if (k > 0 && k < a.n && k <= kList / 2) {
    for (int i = tid; i < r.len; i += kThreads) r.add_bin(r.bin(r.get(i)), false, 0.f);
    u64 tc, tm;
    r.merge(tc, tm);
    const Found b = r.search(r.e_count, r.e_mass, true, (u64)k);
    if (b.before_count + b.count <= kList) {
      const int last = (int)b.bin;
      r.gather([&](float x) { return r.bin(x) <= last; });
      if (rank == 0) {
        const int m = min(r.sort_list(), k);
        constexpr int E = kList / kThreads;
        u64 w[E], s = 0, in_p = 0, t, tz;
        double wd[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const int i = tid * E + e;
          wd[e] = i < m ? r.weight(r.list_value(i)) : 0.0;
          w[e] = i < m ? r.units(r.list_value(i)) : 0;
          s += w[e];
        }
        r.scan2(s, in_p, t, tz);
        // top-p: tokens whose preceding mass is below the target; min-p: by weight
        u64 limit = t;
        if (p < 1.f) {
          const double want = ceil(fmax((double)p, 0.0) * (double)t);
          limit = want < 1.0 ? 1 : (u64)want;
        }
        const double lim = mp > 0.f ? fmin((double)mp, 1.0) : 0.0;
        u64 kept = 0, before = s, none = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          if (tid * E + e < m && (before < limit || p >= 1.f || !(p == p)) && wd[e] >= lim) kept += w[e];
          before += w[e];
        }
        u64 total, tn;
        u64 kk = kept;
        r.scan2(kk, none, total, tn);
        u64 x = uf > 0.f ? (u64)((double)uf * (double)total) : 0;
        x = x < total ? x : total - 1;
        before = s;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          if (before <= x && x < before + w[e]) {
            a.ids[j] = r.list_id(tid * E + e);
            if (a.probs) a.probs[j] = (float)((double)w[e] / (double)total);
          }
          before += w[e];
        }
      }
      pdl_launch_dependents();
      return;
    }
    r.clear_bins();
  }
  for (int i = tid; i < r.len; i += kThreads) {
    const float x = r.get(i);
    r.add_bin(r.bin(x), true, x);
  }
  u64 count, mass;
  r.merge(count, mass);
  if (k > 0 && k < a.n) mass = r.resolve(r.search(r.e_count, r.e_mass, true, (u64)k), true, (u64)k, false).mass;
  u64 kept = mass;
  if (p < 1.f) {
    const double want = ceil(fmax((double)p, 0.0) * (double)mass);
    const u64 target = want < 1.0 ? 1 : (u64)want < mass ? (u64)want : mass;
    const u64 m = r.resolve(r.search(r.e_count, r.e_mass, false, target), false, target, false).mass;
    kept = m < kept ? m : kept;
  }
  if (mp > 0.f) {
    const double lim = fmin((double)mp, 1.0);
    // beyond this bin every weight is below lim (a bin more for its rounding)
    const int last = (int)fmin(-log(lim) * kBinsPerNat + 2.0, (double)kBins);
    u64 s = 0;
    for (int i = tid; i < r.len; i += kThreads) {
      const float x = r.get(i);
      if (r.bin(x) <= last && r.weight(x) >= lim) s += r.units(x);
    }
    s = r.reduce<false>(s);
    kept = s < kept ? s : kept;
  }
  u64 x = uf > 0.f ? (u64)((double)uf * (double)kept) : 0;
  x = x < kept ? x : kept - 1;
  const Row::Place got = r.resolve(r.search(r.e_count, r.e_mass, false, x + 1), false, x + 1, true);
  if (got.id >= 0 && tid == 0) {
    a.ids[j] = got.id;
    if (a.probs) a.probs[j] = (float)((double)got.w / (double)kept);
  }
  pdl_launch_dependents();
}

constexpr size_t kSliceMax = 128 * 1024;  // bytes of a resident slice: 44 KB of tables beside it, up to 227 KB

size_t sample_smem(int cluster, size_t slice_bytes) {
  return sizeof(Fixed) + 4 * (size_t)(kBins / cluster + 1) * sizeof(u64) + slice_bytes;
}

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
  // CTAs a row: few rows take more of them (a slice of at least 1024 tokens
  // each), many rows as few as hold the row
  int cluster = 1;
  while (cluster < 8 && (n + cluster - 1) / cluster > (count <= 37 ? 1024u : 20480u)) cluster *= 2;
  const size_t slice = ((n + cluster - 1) / cluster + 3) & ~(size_t)3;
  const bool resident = slice * sizeof(float) <= kSliceMax;
  const size_t smem = sample_smem(cluster, resident ? slice * sizeof(float) : 0);
  static std::atomic<bool> smem_set[64];  // idempotent: concurrent first calls only repeat it
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return PYRITE_E_CUDA;
  if (!smem_set[dev].load(std::memory_order_acquire)) {
    if (cudaFuncSetAttribute(sample_rows_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024) !=
        cudaSuccess)
      return PYRITE_E_CUDA;
    smem_set[dev].store(true, std::memory_order_release);
  }
  const SampleArgs a{logits, ld,    (int)n, (int)slice, resident ? 1 : 0, uniforms, temperature,
                     top_k,  top_p, min_p,  ids,        probs,            62 - bits};
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
  return cudaLaunchKernelEx(&cfg, sample_rows_kernel, a) == cudaSuccess ? 0 : PYRITE_E_CUDA;
}

}  // extern "C"
