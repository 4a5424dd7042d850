// paged_attention.cu -- attention of a batch whose requests share a prefix, over
// a paged key/value pool (paged.cuh).
//
// Row b's query heads attend to the P tokens of the shared prefix and then to
// the row's own kv_lens[b] tokens:
//   o = sum_t e^(s_t - m) v_t / sum_t e^(s_t - m),  s_t = q . k_t / sqrt(128).
// The sums split over any partition of the keys: a part that has seen some keys
// is (m, l, o) = (max s, sum e^(s - m), sum e^(s - m) v), and two parts join as
// m = max(m1, m2), l = l1 e^(m1 - m) + l2 e^(m2 - m), o likewise.  So the prefix
// is computed for tiles of query rows of all requests (every key read once per
// tile, not once per row), the own keys per request, both split over CTAs, and a
// last kernel joins the parts.  A row without a key gives zeros.  Scores and
// statistics are fp32, in base 2 (q is scaled by log2(e) / sqrt(128)).
//
// The keys of all work items (an item: up to 16 query rows that share their keys)
// are cut into blocks of 64, and the blocks, in order, into as many equal runs
// as there are CTAs: lengths may differ by any factor and every SM still gets the
// same work.  An item counts kItemCost units besides its blocks: a piece takes about
// 4 us to begin and to end, a block 1.3 us at full bandwidth (64 requests of 100 to
// 1000 keys: 31 us without, 26 us with them).  A CTA works through the items of its
// run; the piece of item i in CTA c is part i + c (both only grow along the order, so
// no two pieces meet).
//
// Four kernels compute parts:
//   attn_simt_kernel   fp32 caches, up to 8 query rows an item; fp32 arithmetic.  Bound by
//                      its bytes where keys are many (24 rows of up to 16000 keys, 8 KV
//                      heads: 297 us, the bytes alone 284 us), else by its loads in
//                      flight (16 rows of up to 512 keys: 8 us of a call's 26, whose
//                      bytes alone take 6.4).
//   attn_f32_kernel    fp32 caches, 16 query rows an item; tf32 matrix instructions, operands
//                      straight from global memory.  Bound by the matrix unit.
//   attn_mma_kernel    16-bit caches; matrix instructions over 16 query rows, a
//                      warp per 16 keys.  Bound by the cache's bytes (24 rows of up to
//                      16000 keys, fp16: 141 us, the bytes alone 130 us; bf16, a plane
//                      more: 157 us where fp16 takes 149).
//   prefix_tc_kernel   (paged_attention_tc.cu) 16-bit caches, prefixes with many query
//                      rows: tcgen05 tiles of 128 rows x 128 keys.
// In 16-bit products q and the weights are split into sums of 16-bit values
// (planes): a cache value is exact, so the products lose only what the planes
// leave out, 2^-22 (fp16: two planes) or 2^-24 (bf16: three).  With fp32 caches every
// operand is split into two tf32 values; the product of the small ones, 2^-22 of the
// whole, is left out.
#include <atomic>
#include <cfloat>

#include "kernels.cuh"
#include "paged.cuh"
#include "ptx.cuh"
#include "../../include/pyrite_b200.h"

namespace pyr {
namespace {

constexpr int HD = 128;
constexpr float kNegInf = -INFINITY;
constexpr int kBlock = 64;       // keys of a work unit
constexpr int kMaxRows = 4096;   // rows of one call

// A launch of own keys behind one of prefix keys depends on nothing of it: the
// prefix launch lets it start once everything before has ended (its own wait has
// returned in every CTA), and it ends only after the prefix launch has (its wait
// is its last step), so the join behind it waits for both.  The join starts beside
// the own keys in the same way: what it reads before its wait, the lengths, was there
// before either launch.
__device__ __forceinline__ void begin_part(const AttnWork& w) {
  if (!w.behind_prefix) pdl_wait();
  pdl_launch_dependents();
}
__device__ __forceinline__ void end_part(const AttnWork& w) {
  if (w.behind_prefix) pdl_wait();
}

__device__ __forceinline__ float4 load4(const float* p) { return *reinterpret_cast<const float4*>(p); }

// ---- the runs ------------------------------------------------------------------------------
constexpr int kItemCost = 3;
__device__ __forceinline__ int units_of(int blocks) { return blocks ? blocks + kItemCost : 0; }
// starts[b] = units of an item of each row before b (a prefix counts as one row).
__device__ __forceinline__ int blocks_of(const AttnWork& w, int len) {
  return (min(max(len, 0), w.max_len) + kBlock - 1) / kBlock;
}
__device__ __forceinline__ int row_blocks(const AttnWork& w, int b) {
  return w.lens ? blocks_of(w, w.lens[b]) : (w.fixed_len + kBlock - 1) / kBlock;
}
// All threads: starts[0 .. rows] in shared memory.
__device__ void scan_rows(const AttnWork& w, int* starts) {
  const int lane = threadIdx.x & 31;
  if (threadIdx.x < 32) {
    int base = 0;
    for (int b0 = 0; b0 < w.rows; b0 += 32) {
      int n = b0 + lane < w.rows ? units_of(row_blocks(w, b0 + lane)) : 0, s = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += t;
      }
      if (b0 + lane < w.rows) starts[b0 + lane] = base + s - n;
      base += __shfl_sync(0xffffffffu, s, 31);
    }
    if (lane == 0) starts[w.rows] = base;
  }
  __syncthreads();
}
// Up to kSms units, a CTA takes one each; beyond, at least four on average: a run costs
// some microseconds to begin, its part has to be joined, and beside a prefix launch only
// some SMs are free (16 rows behind 4096 keys: 18 us with four, 24 us with two).  The
// first CTAs take them, so no run between an item's first and last piece is empty.
constexpr int kSms = 148;
__device__ __forceinline__ int run_count(long long total, int grid) {
  const long long few = min(total, (long long)kSms), most = (total + 3) / 4;
  return (int)min((long long)grid, max(few, most));
}
__device__ __forceinline__ long long run_start(long long total, int c, int grid) {
  const int g = run_count(total, grid);
  if (c >= g) return total;
  return total <= 0x7fffff ? (long long)((unsigned)total * (unsigned)c / (unsigned)g) : total * c / g;
}
// The CTA whose run holds unit u.
__device__ __forceinline__ int run_of(long long total, long long u, int grid) {
  const int g = run_count(total, grid);
  if (total <= 0x7fffff) return (int)((((unsigned)u + 1) * (unsigned)g - 1) / (unsigned)total);
  return (int)(((u + 1) * g - 1) / total);
}

struct Piece {
  int b, item;  // row, item of the row (KV head x tile)
  int k0, k1;   // keys
};
// The piece of the run at unit u; u moves past it.  An item's first kItemCost units
// are no blocks: a run that ends within them leaves a piece without keys.
__device__ __forceinline__ Piece next_piece(const AttnWork& w, const int* starts, long long& u, long long end) {
  const int x = u <= 0x7fffffff ? (int)((unsigned)u / (unsigned)w.items) : (int)(u / w.items);
  int lo = 0, hi = w.rows;
  while (hi - lo > 1) {  // the last row that starts at or before x: the one that holds it
    const int mid = (lo + hi) >> 1;
    if (starts[mid] <= x) lo = mid;
    else hi = mid;
  }
  const int nu = starts[lo + 1] - starts[lo];
  const long long rem = u - (long long)starts[lo] * w.items;
  Piece p;
  p.b = lo;
  p.item = rem <= 0x7fffffff ? (int)((unsigned)rem / (unsigned)nu) : (int)(rem / nu);
  const int at = (int)(rem - (long long)p.item * nu), n = (int)min((long long)(nu - at), end - u);
  u += n;
  const int len = w.lens ? min(max(w.lens[lo], 0), w.max_len) : w.fixed_len;
  p.k0 = max(at - kItemCost, 0) * kBlock;
  p.k1 = min(max(at + n - kItemCost, 0) * kBlock, len);
  return p;
}
// Query row i of a tile: its row and head.
__device__ __forceinline__ void query_of(const AttnWork& w, const Piece& p, int i, int& row, int& head, bool& on) {
  const int group = w.nq / w.nkv, tiles = w.items / w.nkv, kvh = p.item / tiles, r = (p.item % tiles) * w.tile + i;
  on = i < w.tile && r < (w.lens ? group : w.count * group);
  row = w.lens ? p.b : r / group;
  head = kvh * group + (w.lens ? r : r % group);
}

// The warps' sums of 16 rows in shared memory, mem [warp][16][kPart] (l and o) and stat
// [warp][16] (maxima), to one part per row; each warp's factor of each row is made
// once.  All threads; mem and stat are free afterwards.
template <int WARPS> __device__ __forceinline__ void join_warps(const AttnWork& w, const float* mem, float* stat, float* part) {
  const int tid = threadIdx.x;
  __syncthreads();
  float fac = 0.f;
  if (tid < WARPS * 16) {
    const int i = tid & 15;
    float M = kNegInf;
#pragma unroll
    for (int v = 0; v < WARPS; ++v) M = fmaxf(M, stat[v * 16 + i]);
    const float mine = stat[tid];
    fac = mine == kNegInf ? 0.f : ex2(mine - M);
    if (tid < w.tile) part[i * kPart] = M == kNegInf ? M : M - kUp;
  }
  __syncthreads();
  if (tid < WARPS * 16) stat[tid] = fac;
  __syncthreads();
  for (int e = tid; e < w.tile * 33; e += 32 * WARPS) {  // 33: the row's m and l, then o
    const int i = e / 33;
    float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int v = 0; v < WARPS; ++v) {
      const float f = stat[v * 16 + i];
      const float4 y = load4(mem + v * 16 * kPart + 4 * e);
      if (f != 0.f) O.x += y.x * f, O.y += y.y * f, O.z += y.z * f, O.w += y.w * f;
    }
    if (e % 33 == 0) {
      part[4 * e + 1] = O.y;
      if (O.y != O.y) part[4 * e] = O.y;
    } else {
      *reinterpret_cast<float4*>(part + 4 * e) = O;
    }
  }
  __syncthreads();
}

// ---- fp32 caches -----------------------------------------------------------------------------
// Sum 32 values over the 32 lanes, value i's sum left in lane i: each step
// halves the values a lane holds, so 31 shuffles serve all 32 sums.
__device__ __forceinline__ float transpose_sum(float (&v)[32], int lane) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const bool up = lane & o;
#pragma unroll
    for (int i = 0; i < o; ++i) {
      const float keep = up ? v[i + o] : v[i], give = up ? v[i] : v[i + o];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
    }
  }
  return v[0];
}

// Few query rows: tiles of QT, 8 warps taking every 8th group of 32 / QT keys.  A lane
// holds 4 of the 128 dimensions of every query and accumulator; a group's 32
// (query, key) scores are summed by transpose_sum, one left to each lane.
template <int QT> __global__ void __launch_bounds__(256) attn_simt_kernel(AttnWork w, PagePool<float> pool) {
  constexpr int KG = 32 / QT;  // keys of a group: at most 16, so a group lies in one page
  extern __shared__ int starts[];
  __shared__ float sm_p[8][32];
  __shared__ float sm_m[8][QT], sm_l[8][QT];
  __shared__ __align__(16) float sm_o[8][QT][HD];
  begin_part(w);
  scan_rows(w, starts);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int ps_log2 = pool.ps_log2, ps = 1 << ps_log2;
  const long long total = (long long)starts[w.rows] * w.items;
  const long long end = run_start(total, blockIdx.x + 1, gridDim.x);
  for (long long u = run_start(total, blockIdx.x, gridDim.x); u < end;) {
    const Piece pc = next_piece(w, starts, u, end);
    if (pc.k0 >= pc.k1) continue;
    const int kvh = pc.item / (w.items / w.nkv);
    const int* list = w.pages + (long long)pc.b * w.table_stride;
    float4 q[QT], o[QT];
#pragma unroll
    for (int i = 0; i < QT; ++i) {
      int row, head;
      bool on;
      query_of(w, pc, i, row, head, on);
      o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      q[i] = o[i];
      if (on) q[i] = load4(w.q + (long long)row * w.ldq + (size_t)head * HD + 4 * lane);
      q[i].x *= w.qscale; q[i].y *= w.qscale; q[i].z *= w.qscale; q[i].w *= w.qscale;
    }
    const int qi = lane / KG, kj = lane % KG;  // this lane's score
    float m = kNegInf, l = 0.f;                // of query qi, l over this lane's keys
    for (int t0 = pc.k0 + warp * KG; t0 < pc.k1; t0 += 8 * KG) {
      const int page = list[t0 >> ps_log2];
      const bool ok = page >= 0 && page < pool.n_pages;
      if (!ok) {  // a page outside the pool: its keys are left out, the status word says so
        if (lane == 0) atomicOr(w.status, (int)kStatusBadPage);
        continue;
      }
      const size_t at = (((size_t)page * w.nkv + kvh) * ps + (t0 & (ps - 1))) * HD + 4 * lane;
      const int n = min(KG, pc.k1 - t0);
      float4 kk[KG], vv[KG];
#pragma unroll
      for (int j = 0; j < KG; ++j) {
        kk[j] = vv[j] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (j < n) {
          kk[j] = load4(pool.k + at + (size_t)j * HD);
          vv[j] = load4(pool.v + at + (size_t)j * HD);
        }
      }
      float s[32];
#pragma unroll
      for (int i = 0; i < QT; ++i)
#pragma unroll
        for (int j = 0; j < KG; ++j)
          s[i * KG + j] = fmaf(q[i].x, kk[j].x, fmaf(q[i].y, kk[j].y, fmaf(q[i].z, kk[j].z, q[i].w * kk[j].w)));
      float sc = transpose_sum(s, lane);
      if (kj >= n) sc = kNegInf;
      float mn = sc;
#pragma unroll
      for (int off = KG / 2; off > 0; off >>= 1) mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, off));
      mn = fmaxf(mn, m);
      const float p = sc == kNegInf ? 0.f : ex2(sc - mn);
      const float alpha = m == kNegInf ? 0.f : ex2(m - mn);
      const bool rescale = __any_sync(0xffffffffu, mn != m);
      m = mn;
      l = l * alpha + p;
      __syncwarp();
      sm_p[warp][lane] = p;
      __syncwarp();
#pragma unroll
      for (int i = 0; i < QT; ++i) {
        if (rescale) {
          const float al = __shfl_sync(0xffffffffu, alpha, i * KG);
          o[i].x *= al; o[i].y *= al; o[i].z *= al; o[i].w *= al;
        }
#pragma unroll
        for (int j = 0; j < KG; ++j) {
          const float pj = sm_p[warp][i * KG + j];
          o[i].x = fmaf(pj, vv[j].x, o[i].x);
          o[i].y = fmaf(pj, vv[j].y, o[i].y);
          o[i].z = fmaf(pj, vv[j].z, o[i].z);
          o[i].w = fmaf(pj, vv[j].w, o[i].w);
        }
      }
    }
#pragma unroll
    for (int off = KG / 2; off > 0; off >>= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
    if (kj == 0) {
      sm_m[warp][qi] = l != l ? l : m;  // a NaN score counts however it compares
      sm_l[warp][qi] = l;
    }
#pragma unroll
    for (int i = 0; i < QT; ++i) *reinterpret_cast<float4*>(&sm_o[warp][i][4 * lane]) = o[i];
    __syncthreads();
    // join the warps; one part per query row
    float* part = w.parts + ((size_t)(pc.b * w.items + pc.item) + blockIdx.x) * w.tile * kPart;
    for (int e = tid; e < w.tile * HD; e += 256) {
      const int i = e / HD, d = e % HD;
      float M = kNegInf, L = 0.f, O = 0.f;
      for (int v = 0; v < 8; ++v) M = fmaxf(M, sm_m[v][i]);
      for (int v = 0; v < 8; ++v) {
        const float f = sm_m[v][i] == kNegInf ? 0.f : ex2(sm_m[v][i] - M);
        L += sm_l[v][i] * f;
        O += sm_o[v][i][d] * f;
      }
      part[i * kPart + 4 + d] = O;
      if (d == 0) {
        part[i * kPart] = L != L ? L : M;
        part[i * kPart + 1] = L;
      }
    }
    __syncthreads();
  }
  end_part(w);
}

// A value's tf32 part (rounded to 11 bits) and what that leaves, of which the matrix
// unit reads 11 bits more.
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
  hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
  lo = __float_as_uint(x - __uint_as_float(hi));
}
__device__ __forceinline__ void mma_tf32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float part4(const float4& v, int c) { return c == 0 ? v.x : c == 1 ? v.y : c == 2 ? v.z : v.w; }

// 16 query rows, 8 warps taking every 8th group of 16 keys.  Keys and values go
// from global memory straight into the registers of the matrix operands, 16 bytes a
// load: in a score the order of the dimensions is free, and in weights x V that of the
// keys and of the output's columns, so a thread takes as "k" and "n" what its loads
// hold.  K of the next group is on its way during the weights, V during the scores.
// Every operand is two tf32 values and the product of the small ones is left out.
constexpr int kF32Warps = 8;
constexpr uint32_t kF32Frags = 2 * 16 * 32 * 16;  // q's planes as A fragments
constexpr uint32_t kF32Fixed = kF32Frags + kF32Warps * 16 * kPart * 4 + kF32Warps * 16 * 4;
__global__ void __launch_bounds__(32 * kF32Warps, 1) attn_f32_kernel(AttnWork w, PagePool<float> pool) {
  extern __shared__ __align__(128) uint8_t ring[];
  uint4* frag = reinterpret_cast<uint4*>(ring);                // [plane][step][lane]
  float* mem = reinterpret_cast<float*>(ring + kF32Frags);     // [warp][16][kPart]
  float* stat = mem + kF32Warps * 16 * kPart;                  // [warp][16]
  int* starts = reinterpret_cast<int*>(ring + kF32Fixed);
  begin_part(w);
  scan_rows(w, starts);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, t4 = lane & 3, g8 = lane >> 2;
  const int ps_log2 = pool.ps_log2, ps = 1 << ps_log2;
  const long long total = (long long)starts[w.rows] * w.items;
  const long long end = run_start(total, blockIdx.x + 1, gridDim.x);
  for (long long u = run_start(total, blockIdx.x, gridDim.x); u < end;) {
    const Piece pc = next_piece(w, starts, u, end);
    if (pc.k0 >= pc.k1) continue;
    const int kvh = pc.item / (w.items / w.nkv);
    const int* list = w.pages + (long long)pc.b * w.table_stride;
    const int groups = (pc.k1 - pc.k0 + 15) / 16;
    const int mine = groups > warp ? (groups - warp + kF32Warps - 1) / kF32Warps : 0;
    // q: of the 16 steps, two a warp; step s has dimensions 16 (s / 2) + 4 t4 + 2 (s % 2), + 1
    {
      uint32_t b[2][2][4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        int row, head;
        bool on;
        query_of(w, pc, g8 + 8 * h, row, head, on);
        const float4 x = on ? load4(w.q + (long long)row * w.ldq + (size_t)head * HD + 16 * warp + 4 * t4)
                            : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int up = 0; up < 2; ++up)
            split_tf32(part4(x, 2 * k + up) * w.qscale, b[k][0][h + 2 * up], b[k][1][h + 2 * up]);
      }
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int p = 0; p < 2; ++p)
          frag[(p * 16 + 2 * warp + k) * 32 + lane] = make_uint4(b[k][p][0], b[k][p][1], b[k][p][2], b[k][p][3]);
    }
    int ids = 0;  // lane: the page of group g0 + lane, g0 the multiple of 32 at or below the current one
    // the first key's place of group g in the pool and its number of keys (0: none, or a
    // page outside the pool: left out, the status word says so)
    auto find = [&](int g, size_t& at) {
      if (g >= mine) return 0;
      if ((g & 31) == 0 && g + lane < mine) ids = list[(pc.k0 + (warp + (g + lane) * kF32Warps) * 16) >> ps_log2];
      const int page = __shfl_sync(0xffffffffu, ids, g & 31), t0 = pc.k0 + (warp + g * kF32Warps) * 16;
      const bool ok = page >= 0 && page < pool.n_pages;
      if (!ok && lane == 0) atomicOr(w.status, (int)kStatusBadPage);
      at = (((size_t)(ok ? page : 0) * w.nkv + kvh) * ps + (t0 & (ps - 1))) * HD;
      return ok ? min(16, pc.k1 - t0) : 0;
    };
    float4 kr[2][8], vr[2][2][4];  // keys g8, g8 + 8: dimensions 16 i + 4 t4 ..; keys 8 t + 2 t4 + e: 32 i + 4 g8 ..
    const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
    auto load_k = [&](size_t at, int n) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          kr[t][i] = g8 + 8 * t < n ? load4(pool.k + at + (size_t)(g8 + 8 * t) * HD + 16 * i + 4 * t4) : zero;
    };
    auto load_v = [&](size_t at, int n) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = 8 * t + 2 * t4 + e;
            vr[t][e][i] = r < n ? load4(pool.v + at + (size_t)r * HD + 32 * i + 4 * g8) : zero;
          }
    };
    size_t at = 0;
    int n = find(0, at);
    load_k(at, n);
    load_v(at, n);
    __syncthreads();  // q's fragments
    float o[16][4], m[2] = {kNegInf, kNegInf}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 16; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    for (int g = 0; g < mine; ++g) {
      // the even and odd steps' leading products and the small ones are summed apart: the
      // matrix unit's additions round toward zero
      float s[2][4] = {}, s1[2][4] = {}, s2[2][4] = {};
#pragma unroll
      for (int ks = 0; ks < 16; ++ks) {
        alignas(16) uint32_t q0[4], q1[4];
        *reinterpret_cast<uint4*>(q0) = frag[ks * 32 + lane];
        *reinterpret_cast<uint4*>(q1) = frag[(16 + ks) * 32 + lane];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          uint32_t hi[2], lo[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) split_tf32(part4(kr[t][ks >> 1], 2 * (ks & 1) + e), hi[e], lo[e]);
          mma_tf32(ks & 1 ? s1[t] : s[t], q0, hi[0], hi[1]);
          mma_tf32(s2[t], q0, lo[0], lo[1]);
          mma_tf32(s2[t], q1, hi[0], hi[1]);
        }
      }
      const int n_now = n;
      size_t next = 0;
      n = find(g + 1, next);
      load_k(next, n);
      float mx[2] = {kNegInf, kNegInf};
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = 8 * t + 2 * t4 + (e & 1);
          s[t][e] = key < n_now ? s[t][e] + s1[t][e] + s2[t][e] : kNegInf;
          mx[e >> 1] = fmaxf(mx[e >> 1], s[t][e]);
        }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
        mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
      }
      if (__any_sync(0xffffffffu, mx[0] > m[0] + kLazy || mx[1] > m[1] + kLazy)) {
        float f[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float mn = fmaxf(m[h], mx[h]);
          f[h] = m[h] == kNegInf ? 0.f : ex2(m[h] - mn);
          l[h] *= f[h];
          m[h] = mn;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          o[i][0] *= f[0]; o[i][1] *= f[0]; o[i][2] *= f[1]; o[i][3] *= f[1];
        }
      }
      // a score's registers are a weight fragment's, with keys 2 t4 and 2 t4 + 1 as k and k + 4
      uint32_t ph[2][4], pl[2][4];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float p = s[t][e] == kNegInf ? 0.f : ex2(s[t][e] - m[e >> 1] + kUp);
          l[e >> 1] += p;
          split_tf32(p, ph[t][(e >> 1) + 2 * (e & 1)], pl[t][(e >> 1) + 2 * (e & 1)]);
        }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) {  // columns n: dimensions 32 i + 4 n + c
          float t0[4] = {}, t1[4] = {};
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            uint32_t hi[2], lo[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) split_tf32(part4(vr[t][e][i], c), hi[e], lo[e]);
            mma_tf32(t0, ph[t], hi[0], hi[1]);
            mma_tf32(t1, ph[t], lo[0], lo[1]);
            mma_tf32(t1, pl[t], hi[0], hi[1]);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) o[4 * i + c][e] += t0[e] + t1[e];
        }
      load_v(next, n);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float* row = mem + (warp * 16 + g8 + 8 * h) * kPart;
      float sum = l[h];
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      if (t4 == 0) {
        stat[warp * 16 + g8 + 8 * h] = sum != sum ? sum : m[h];  // a NaN score counts however it compares
        row[1] = sum;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int v = 0; v < 2; ++v)
          *reinterpret_cast<float4*>(row + 4 + 32 * i + 8 * t4 + 4 * v) =
              make_float4(o[4 * i][2 * h + v], o[4 * i + 1][2 * h + v], o[4 * i + 2][2 * h + v], o[4 * i + 3][2 * h + v]);
    }
    join_warps<kF32Warps>(w, mem, stat, w.parts + ((size_t)(pc.b * w.items + pc.item) + blockIdx.x) * w.tile * kPart);
  }
  end_part(w);
}

// ---- 16-bit caches -----------------------------------------------------------------------------
template <typename T> struct Mma;
template <> struct Mma<__half> {
  static constexpr int kPlanes = 2;
  static constexpr bool kScaled = true;  // q rows have scales (row_scale)
  __device__ __forceinline__ static void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};
template <> struct Mma<__nv_bfloat16> {
  static constexpr int kPlanes = 3;
  static constexpr bool kScaled = false;
  __device__ __forceinline__ static void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a));
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a));
}
// 16 bytes, or zeros where on is false.
__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}

constexpr int kMmaWarps = 4, kStages = 3;
constexpr uint32_t kTile16 = 16 * HD * 2;              // bytes of 16 keys (or values)
constexpr uint32_t kWarpSmem = kStages * 2 * kTile16;  // a warp's ring
constexpr uint32_t kFragBytes = 3 * 8 * 32 * 16 + kMmaWarps * 16 * 4;  // q's planes as fragments, rows' maxima

// One warp takes every 4th group of 16 keys of the piece, through a ring of its
// own (no barrier in the loop): scores = q K^T (16 x 16), weights in place as the
// A operand of weights x V (16 x 128).  The 16 rows are the query heads that
// share the KV head; a group of 4 fills a quarter of them and still costs less
// time than its bytes.  The running maximum moves only when it grows by 2^8, so
// the accumulators are rescaled a few times per piece.
template <typename T> __global__ void __launch_bounds__(32 * kMmaWarps, 2) attn_mma_kernel(AttnWork w, PagePool<T> pool) {
  constexpr int NP = Mma<T>::kPlanes;
  extern __shared__ __align__(128) uint8_t ring[];
  int* starts = reinterpret_cast<int*>(ring + kMmaWarps * kWarpSmem + kFragBytes);
  begin_part(w);
  scan_rows(w, starts);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int ps_log2 = pool.ps_log2, ps = 1 << ps_log2;
  const uint32_t base = ptx::smem_addr(ring) + warp * kWarpSmem;
  const long long total = (long long)starts[w.rows] * w.items;
  const long long end = run_start(total, blockIdx.x + 1, gridDim.x);
  for (long long u = run_start(total, blockIdx.x, gridDim.x); u < end;) {
    const Piece pc = next_piece(w, starts, u, end);
    if (pc.k0 >= pc.k1) continue;
    const int kvh = pc.item / (w.items / w.nkv);
    const int* list = w.pages + (long long)pc.b * w.table_stride;
    const int groups = (pc.k1 - pc.k0 + 15) / 16;
    const int mine = groups > warp ? (groups - warp + kMmaWarps - 1) / kMmaWarps : 0;
    // a quarter of q, on its way while the ring fills: the two k steps ks = 2 warp + e / 4
    // of the A fragments, e % 4: rows lane / 4 and + 8, k and k + 8
    float2 x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      int row, head;
      bool on;
      query_of(w, pc, (lane >> 2) + 8 * (e & 1), row, head, on);
      const int d = 16 * (2 * warp + (e >> 2)) + 8 * ((e >> 1) & 1) + 2 * (lane & 3);
      x[e] = on ? *reinterpret_cast<const float2*>(w.q + (long long)row * w.ldq + (size_t)head * HD + d)
                : make_float2(0.f, 0.f);
    }
    int ids = 0;        // lane: the page of group g0 + lane, g0 the multiple of 32 at or below the last issued
    unsigned skip = 0;  // of the groups in the ring: bit g % 32 set: the page is outside the pool
    // group g of this warp -> ring slot g % kStages
    auto issue = [&](int g) {
      if (g < mine) {
        if ((g & 31) == 0 && g + lane < mine) ids = list[(pc.k0 + (warp + (g + lane) * kMmaWarps) * 16) >> ps_log2];
        const int t0 = pc.k0 + (warp + g * kMmaWarps) * 16;
        const int page = __shfl_sync(0xffffffffu, ids, g & 31);
        const bool ok = page >= 0 && page < pool.n_pages;
        if (ok) skip &= ~(1u << (g & 31));
        else skip |= 1u << (g & 31);
        if (!ok && lane == 0) atomicOr(w.status, (int)kStatusBadPage);
        const int n = ok ? min(16, pc.k1 - t0) : 0;
        const size_t at = (((size_t)(ok ? page : 0) * w.nkv + kvh) * ps + (t0 & (ps - 1))) * HD;
        const int c = lane & 15;
        const uint32_t dst = base + (uint32_t)(g % kStages) * 2 * kTile16;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int r = 2 * i + (lane >> 4);
          const uint32_t off = (uint32_t)r * 256 + (uint32_t)((c ^ (r & 7)) << 4);
          const size_t src = at + (size_t)r * HD + 8 * c;
          cp_async16_or_zero(dst + off, pool.k + src, r < n);
          cp_async16_or_zero(dst + kTile16 + off, pool.v + src, r < n);
        }
      }
      ptx::cp_async_commit();
    };
#pragma unroll
    for (int g = 0; g < kStages - 1; ++g) issue(g);
    // q as A fragments, a power of two taken out of each row (row_scale); each warp makes its quarter for all
    alignas(16) uint32_t qa[NP][8][4];
    float qmul[2] = {1.f, 1.f};
    {
      uint4* frag = reinterpret_cast<uint4*>(ring + kMmaWarps * kWarpSmem);  // [plane][ks][lane]
      float* row_top = reinterpret_cast<float*>(frag + NP * 8 * 32);         // [warp][16]
      float top[2] = {0.f, 0.f};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e].x *= w.qscale;
        x[e].y *= w.qscale;
        top[e & 1] = fmaxf(top[e & 1], fmaxf(fabsf(x[e].x), fabsf(x[e].y)));
      }
      float down[2] = {1.f, 1.f};
      if (Mma<T>::kScaled) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
          top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
          if ((lane & 3) == 0) row_top[warp * 16 + (lane >> 2) + 8 * h] = top[h];
        }
        __syncthreads();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int v = 0; v < kMmaWarps; ++v) top[h] = fmaxf(top[h], row_top[v * 16 + (lane >> 2) + 8 * h]);
          down[h] = row_scale<T>(top[h], qmul[h]);
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e].x *= down[e & 1], x[e].y *= down[e & 1];
#pragma unroll
      for (int p = 0; p < NP; ++p)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          uint4 b;
          b.x = plane2<T>(x[4 * k].x, x[4 * k].y);
          b.y = plane2<T>(x[4 * k + 1].x, x[4 * k + 1].y);
          b.z = plane2<T>(x[4 * k + 2].x, x[4 * k + 2].y);
          b.w = plane2<T>(x[4 * k + 3].x, x[4 * k + 3].y);
          frag[(p * 8 + 2 * warp + k) * 32 + lane] = b;
        }
      __syncthreads();
#pragma unroll
      for (int p = 0; p < NP; ++p)
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) *reinterpret_cast<uint4*>(qa[p][ks]) = frag[(p * 8 + ks) * 32 + lane];
    }
    float o[16][4], m[2] = {kNegInf, kNegInf}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 16; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    for (int g = 0; g < mine; ++g) {
      __syncwarp();  // every lane is done with the slot that is filled next
      issue(g + kStages - 1);
      ptx::cp_async_wait<kStages - 1>();
      __syncwarp();  // group g has landed for every lane
      const uint32_t kt = base + (uint32_t)(g % kStages) * 2 * kTile16, vt = kt + kTile16;
      // The matrix unit's additions round toward zero, so long chains drift: the
      // even and odd steps' leading planes and the small planes are summed apart.
      float s[2][4] = {}, s1[2][4] = {}, s2[2][4] = {};
#pragma unroll
      for (int ks = 0; ks < 8; ++ks) {
        // matrices: keys 0-7 | 8-15, dimensions 0-7 | 8-15 of this step
        const int r = (lane & 7) + ((lane >> 4) << 3), c = 2 * ks + ((lane >> 3) & 1);
        uint32_t kb[4];
        ldsm4(kb, kt + (uint32_t)r * 256 + (uint32_t)((c ^ (r & 7)) << 4));
        Mma<T>::mma(ks & 1 ? s1[0] : s[0], qa[0][ks], kb[0], kb[1]);
        Mma<T>::mma(ks & 1 ? s1[1] : s[1], qa[0][ks], kb[2], kb[3]);
#pragma unroll
        for (int p = 1; p < NP; ++p) {
          Mma<T>::mma(s2[0], qa[p][ks], kb[0], kb[1]);
          Mma<T>::mma(s2[1], qa[p][ks], kb[2], kb[3]);
        }
      }
      const int n = (skip >> (g & 31)) & 1 ? 0 : min(16, pc.k1 - pc.k0 - (warp + g * kMmaWarps) * 16);
      float mx[2] = {kNegInf, kNegInf};
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = 8 * t + 2 * (lane & 3) + (e & 1);
          s[t][e] = key < n ? (s[t][e] + s1[t][e] + s2[t][e]) * qmul[e >> 1] : kNegInf;
          mx[e >> 1] = fmaxf(mx[e >> 1], s[t][e]);
        }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
        mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
      }
      if (__any_sync(0xffffffffu, mx[0] > m[0] + kLazy || mx[1] > m[1] + kLazy)) {
        float f[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float mn = fmaxf(m[h], mx[h]);
          f[h] = m[h] == kNegInf ? 0.f : ex2(m[h] - mn);
          l[h] *= f[h];
          m[h] = mn;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          o[i][0] *= f[0]; o[i][1] *= f[0]; o[i][2] *= f[1]; o[i][3] *= f[1];
        }
      }
      uint32_t pa[NP][4];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          // 2^kUp keeps fp16's lower plane out of its subnormals
          float p0 = s[t][2 * h] == kNegInf ? 0.f : ex2(s[t][2 * h] - m[h] + kUp);
          float p1 = s[t][2 * h + 1] == kNegInf ? 0.f : ex2(s[t][2 * h + 1] - m[h] + kUp);
          l[h] += p0 + p1;
#pragma unroll
          for (int p = 0; p < NP; ++p) pa[p][2 * t + h] = plane2<T>(p0, p1);
        }
#pragma unroll
      for (int ds = 0; ds < 8; ++ds) {
        const int r = (lane & 7) + (((lane >> 3) & 1) << 3), c = 2 * ds + (lane >> 4);
        uint32_t vb[4];
        ldsm4_t(vb, vt + (uint32_t)r * 256 + (uint32_t)((c ^ (r & 7)) << 4));
        float t0[4] = {}, t1[4] = {};  // joined by rounded additions: the chain over the keys is long
#pragma unroll
        for (int p = NP - 1; p >= 0; --p) {
          Mma<T>::mma(t0, pa[p], vb[0], vb[1]);
          Mma<T>::mma(t1, pa[p], vb[2], vb[3]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          o[2 * ds][e] += t0[e];
          o[2 * ds + 1][e] += t1[e];
        }
      }
    }
    ptx::cp_async_wait<0>();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    }
    // the warps' sums meet in the ring; each warp's factor of each row is made once
    float* mem = reinterpret_cast<float*>(ring);  // [warp][16][kPart]
    float* stat = mem + kMmaWarps * 16 * kPart;    // [warp][16]: maxima, then factors
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float* row = mem + (warp * 16 + (lane >> 2) + 8 * h) * kPart;
      if ((lane & 3) == 0) {
        stat[warp * 16 + (lane >> 2) + 8 * h] = l[h] != l[h] ? l[h] : m[h];  // a NaN score counts however it compares
        row[1] = l[h];
      }
#pragma unroll
      for (int i = 0; i < 16; ++i)
        *reinterpret_cast<float2*>(row + 4 + 8 * i + 2 * (lane & 3)) = make_float2(o[i][2 * h], o[i][2 * h + 1]);
    }
    join_warps<kMmaWarps>(w, mem, stat, w.parts + ((size_t)(pc.b * w.items + pc.item) + blockIdx.x) * w.tile * kPart);
  }
  end_part(w);
}

// ---- joining -----------------------------------------------------------------------------------
struct JoinArgs {
  AttnWork pre, own;  // pre.rows = 0: no prefix
  int pre_grid, own_grid;
  int share;          // warps a head
  int tc_split;       // > 0: the prefix came from prefix_tc_kernel: this many parts per (KV head, 128 rows)
  float* out;
  long long ldo;
};

struct Sum {
  float m = kNegInf, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  __device__ __forceinline__ void add(float m2, float l2, float4 o2) {
    if (m2 == kNegInf) return;
    const float mn = fmaxf(m, m2);
    const float f = m == kNegInf ? 0.f : ex2(m - mn), g = ex2(m2 - mn);
    l = l * f + l2 * g;
    o.x = o.x * f + o2.x * g; o.y = o.y * f + o2.y * g; o.z = o.z * f + o2.z * g; o.w = o.w * f + o2.w * g;
    m = m2 != m2 ? m2 : mn;
  }
};

// n parts, `stride` floats apart.
struct Parts {
  const float* first = nullptr;
  size_t stride = 0;
  int n = 0;
};
struct Four {  // up to four parts of every `share`, their loads in flight together
  float m[4], l[4];
  float4 o[4];
  __device__ __forceinline__ void load(const Parts& p, int c, int share, int lane) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      m[e] = kNegInf;
      l[e] = 0.f;
      o[e] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (c + e * share < p.n) {
        const float* at = p.first + (size_t)(c + e * share) * p.stride;
        const float2 ml = *reinterpret_cast<const float2*>(at);
        m[e] = ml.x;
        l[e] = ml.y;
        o[e] = load4(at + 4 + 4 * lane);
      }
    }
  }
  __device__ __forceinline__ void add_to(Sum& s) const {
#pragma unroll
    for (int e = 0; e < 4; ++e) s.add(m[e], l[e], o[e]);
  }
};

// A CTA per row and 8 / share query heads of a KV head: `share` warps a head take its
// parts in turn, a lane holds 4 dimensions.  Which parts there are follows from the
// lengths, before the wait; behind it the first parts of the prefix and of the own keys
// are on their way together.
constexpr int kJoinWarps = 8;
__global__ void __launch_bounds__(32 * kJoinWarps) attn_join_kernel(JoinArgs a) {
  __shared__ __align__(16) float sm[kJoinWarps][kPart];
  __shared__ int sums[2][kJoinWarps];
  const AttnWork& w = a.own;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int group = w.nq / w.nkv, share = a.share, heads = kJoinWarps / share, chunks = (group + heads - 1) / heads;
  const int row = blockIdx.x / (w.nkv * chunks), kvh = blockIdx.x / chunks % w.nkv;
  const int mine = warp % share, g = blockIdx.x % chunks * heads + warp / share;
  auto pieces = [&](const AttnWork& k, int grid, int r, int item, long long first, int nb, long long total) {
    Parts p;
    if (nb == 0) return p;
    const int c0 = run_of(total, first + kItemCost, grid), c1 = run_of(total, first + kItemCost + nb - 1, grid);
    p.first = k.parts + ((size_t)(item + c0) * k.tile + r) * kPart;
    p.stride = (size_t)k.tile * kPart;
    p.n = c1 - c0 + 1;
    return p;
  };
  // units of the rows before this one, and of all
  int before = 0, all = 0;
  for (int b = threadIdx.x; b < w.rows; b += 32 * kJoinWarps) {
    const int n = units_of(row_blocks(w, b));
    all += n;
    if (b < row) before += n;
  }
  const int nb = row_blocks(w, row);
  Parts pre, own;
  if (g < group && a.pre.rows) {
    const AttnWork& p = a.pre;
    const int r = row * group + g;
    if (a.tc_split) {
      const int qt = (w.count * group + 127) / 128;
      pre.first = p.parts + ((size_t)(kvh * qt + r / 128) * a.tc_split * 128 + r % 128) * kPart;
      pre.stride = (size_t)128 * kPart;
      pre.n = a.tc_split;
    } else {
      const int pt = p.items / p.nkv, pi = kvh * pt + r / p.tile, pb = row_blocks(p, 0);
      pre = pieces(p, a.pre_grid, r % p.tile, pi, (long long)pi * units_of(pb), pb, (long long)units_of(pb) * p.items);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    before += __shfl_xor_sync(0xffffffffu, before, o);
    all += __shfl_xor_sync(0xffffffffu, all, o);
  }
  if (lane == 0) sums[0][warp] = before, sums[1][warp] = all;
  __syncthreads();
  before = all = 0;
#pragma unroll
  for (int v = 0; v < kJoinWarps; ++v) before += sums[0][v], all += sums[1][v];
  if (g < group) {
    const int tiles = w.items / w.nkv, it = kvh * tiles + g / w.tile;
    own = pieces(w, a.own_grid, g % w.tile, row * w.items + it,
                 (long long)before * w.items + (long long)it * units_of(nb), nb, (long long)all * w.items);
  }
  pdl_wait();
  Sum s;
  {
    Four x, y;
    x.load(pre, mine, share, lane);
    y.load(own, mine, share, lane);
    x.add_to(s);
    for (int c = mine + 4 * share; c < pre.n; c += 4 * share) {
      x.load(pre, c, share, lane);
      x.add_to(s);
    }
    y.add_to(s);
    for (int c = mine + 4 * share; c < own.n; c += 4 * share) {
      y.load(own, c, share, lane);
      y.add_to(s);
    }
  }
  if (share > 1) {
    if (lane == 0) sm[warp][0] = s.m, sm[warp][1] = s.l;
    *reinterpret_cast<float4*>(&sm[warp][4 + 4 * lane]) = s.o;
    __syncthreads();
    if (mine == 0)
      for (int v = 1; v < share; ++v) s.add(sm[warp + v][0], sm[warp + v][1], load4(&sm[warp + v][4 + 4 * lane]));
  }
  if (g < group && mine == 0) {
    const float inv = s.m == kNegInf ? 0.f : 1.0f / s.l;  // no key: zeros
    *reinterpret_cast<float4*>(a.out + (long long)row * a.ldo + (size_t)(kvh * group + g) * HD + 4 * lane) =
        make_float4(s.o.x * inv, s.o.y * inv, s.o.z * inv, s.o.w * inv);
  }
  pdl_launch_dependents();
}

int rc(int e) { return e > 0 ? PYRITE_E_CUDA : e; }

// ---- the plan of a call (sizes only, so the workspace can be asked for beforehand) ----
struct Plan {
  int own_tile, own_items, own_grid;  // query rows of an item, items of a row, CTAs
  int pre_tile, pre_items, pre_grid;  // the prefix by the row kernels
  int tc_split;                       // ... or by tcgen05 tiles
  size_t own_floats, pre_floats;
};
constexpr int kSimtRows = 8;
// Query rows of an item.  fp32: at least 2 (a group of 32 / QT keys then lies inside one
// 16-token page); beyond kSimtRows the matrix instructions of attn_f32_kernel: with 10 to 16
// query heads a KV head, 24 requests of up to 16000 keys take 188 us, in two tiles of 8 rows
// 450 us; with 8 the tiles of 8 are bound by the bytes already.
int tile_rows(int rows, int kv_type) {
  if (kv_type != F32) return rows < 16 ? rows : 16;
  return rows > kSimtRows ? 16 : rows > 4 ? 8 : rows > 2 ? 4 : 2;
}
Plan make_plan(int count, int nq, int nkv, int prefix_len, int kv_type) {
  Plan p{};
  const int group = nq / nkv;
  p.own_tile = tile_rows(group, kv_type);
  p.own_items = nkv * ((group + p.own_tile - 1) / p.own_tile);
  // as many as run at once (of the 16-bit kernel one an SM beyond 1200 rows, whose starts
  // take the room of the second: 1024 rows of 100 keys 221 us, 2048 rows 652 us)
  p.own_grid = kv_type == F32 ? kSms : 2 * kSms;
  p.own_floats = ((size_t)count * p.own_items + p.own_grid) * p.own_tile * kPart;
  if (prefix_len > 0) {
    const int rows = count * group;
    p.tc_split = prefix_tc_split(rows, nkv, prefix_len, kv_type);
    if (p.tc_split) {
      p.pre_floats = (size_t)nkv * ((rows + 127) / 128) * p.tc_split * 128 * kPart;
    } else {
      p.pre_tile = tile_rows(rows, kv_type);
      p.pre_items = nkv * ((rows + p.pre_tile - 1) / p.pre_tile);
      p.pre_grid = p.own_grid;
      p.pre_floats = ((size_t)p.pre_items + p.pre_grid) * p.pre_tile * kPart;
    }
  }
  return p;
}

// The dynamic shared memory limit of a kernel, once per device.
template <typename K> int allow_smem(K kernel, size_t bytes, std::atomic<bool> (&set)[64]) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -4;
  if (!set[dev].load(std::memory_order_acquire)) {  // idempotent: concurrent first calls only repeat it
    if (const int e = launch_code(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes)))
      return e;
    set[dev].store(true, std::memory_order_release);
  }
  return 0;
}
// Tiles of 8 keep 34 KB of sums: with the starts of more than 3711 rows that passes the
// 48 KB that need no asking.
template <int QT> int launch_simt(const AttnWork& w, int grid, const PagePool<float>& pool, cudaStream_t s) {
  static std::atomic<bool> set[64];
  if (int e = allow_smem(attn_simt_kernel<QT>, (kMaxRows + 1) * sizeof(int), set)) return e;
  return launch_pdl(attn_simt_kernel<QT>, dim3(grid), dim3(256), (w.rows + 1) * sizeof(int), s, w, pool);
}
int launch_parts(const AttnWork& w, int grid, const PagePool<float>& pool, cudaStream_t s) {
  switch (w.tile) {
    case 2: return launch_simt<2>(w, grid, pool, s);
    case 4: return launch_simt<4>(w, grid, pool, s);
    case 8: return launch_simt<8>(w, grid, pool, s);
    default: break;
  }
  static std::atomic<bool> set[64];
  if (int e = allow_smem(attn_f32_kernel, kF32Fixed + (kMaxRows + 1) * sizeof(int), set)) return e;
  return launch_pdl(attn_f32_kernel, dim3(grid), dim3(32 * kF32Warps), kF32Fixed + (w.rows + 1) * sizeof(int), s, w, pool);
}
template <typename T> int launch_parts(const AttnWork& w, int grid, const PagePool<T>& pool, cudaStream_t s) {
  static std::atomic<bool> set[64];
  if (int e = allow_smem(attn_mma_kernel<T>, kMmaWarps * kWarpSmem + kFragBytes + (kMaxRows + 1) * sizeof(int), set))
    return e;
  return launch_pdl(attn_mma_kernel<T>, dim3(grid), dim3(32 * kMmaWarps),
                    kMmaWarps * kWarpSmem + kFragBytes + (w.rows + 1) * sizeof(int), s, w, pool);
}

template <typename T>
int launch_attention(AttnWork w, const int* prefix_pages, int prefix_len, const int* table, long long table_stride,
                     const int* lens, int table_width, void* k, void* v, int kv_type, int n_pages, int ps, float* out,
                     long long ldo, float* ws, cudaStream_t s) {
  const PagePool<T> pool{static_cast<T*>(k), static_cast<T*>(v), n_pages, log2_of(ps)};
  const Plan p = make_plan(w.count, w.nq, w.nkv, prefix_len, kv_type);
  JoinArgs j{};
  j.out = out;
  j.ldo = ldo;
  j.pre_grid = p.pre_grid;
  j.own_grid = p.own_grid;
  j.tc_split = p.tc_split;
  if (prefix_len > 0) {
    j.pre = w;
    j.pre.pages = prefix_pages;
    j.pre.fixed_len = prefix_len;
    j.pre.rows = 1;
    j.pre.items = p.pre_items;
    j.pre.tile = p.pre_tile;
    j.pre.parts = ws + p.own_floats;
    const int e = p.tc_split ? launch_prefix_tc(j.pre, k, v, kv_type, n_pages, ps, p.tc_split, s)
                             : launch_parts(j.pre, p.pre_grid, pool, s);
    if (e) return rc(e);
  }
  j.own = w;
  j.own.pages = table;
  j.own.table_stride = table_stride;
  j.own.lens = lens;
  j.own.max_len = table_width * ps;
  j.own.rows = w.count;
  j.own.items = p.own_items;
  j.own.tile = p.own_tile;
  j.own.parts = ws;
  j.own.behind_prefix = prefix_len > 0;
  if (int e = launch_parts(j.own, p.own_grid, pool, s)) return rc(e);
  // about four parts a warp, and no idle warps where heads are few
  const int group = w.nq / w.nkv;
  const int parts = p.tc_split + p.own_grid / (w.count * p.own_items) + 2 + (p.pre_items ? p.pre_grid / p.pre_items + 2 : 0);
  j.share = 1;
  while (j.share < kJoinWarps && (parts > 8 * j.share || group * j.share * 2 <= kJoinWarps)) j.share *= 2;
  const int heads = kJoinWarps / j.share;
  return rc(launch_pdl(attn_join_kernel, dim3((unsigned)(w.count * w.nkv * ((group + heads - 1) / heads))),
                       dim3(32 * kJoinWarps), 0, s, j));
}

}  // namespace
}  // namespace pyr

using namespace pyr;

extern "C" {

size_t pyrite_cuda_attention_paged_workspace_size(int count, int n_heads, int n_kv_heads, int prefix_len,
                                                  int kv_type) {
  if (count <= 0 || count > kMaxRows || n_heads <= 0 || n_heads > 1024 || n_kv_heads <= 0 || n_heads % n_kv_heads ||
      prefix_len < 0 || !kv_type_ok(kv_type))
    return 0;
  const Plan p = make_plan(count, n_heads, n_kv_heads, prefix_len, kv_type);
  return (p.own_floats + p.pre_floats) * sizeof(float);
}

int pyrite_cuda_attention_paged(const float* q, long long ldq, const void* k_pool, const void* v_pool, int kv_type,
                                int n_pages, int page_size, const int* prefix_pages, int prefix_len,
                                const int* block_table, long long table_stride, int table_width, const int* kv_lens,
                                int count, int n_heads, int n_kv_heads, int head_dim, float* out, long long ldo,
                                void* workspace, size_t workspace_len, void* stream) {
  if (!kv_type_ok(kv_type)) return PYRITE_E_TYPE;
  if (!q || !k_pool || !v_pool || !block_table || !kv_lens || !out || (prefix_len > 0 && !prefix_pages))
    return PYRITE_E_BUFFER;
  if (head_dim != HD || count <= 0 || count > kMaxRows || n_heads <= 0 || n_heads > 1024 || n_kv_heads <= 0 ||
      n_heads % n_kv_heads || prefix_len < 0 || !pool_ok(n_pages, page_size, n_kv_heads) || table_width <= 0 ||
      table_stride < 0 || (count > 1 && table_stride != 0 && table_stride < table_width) ||
      (long long)table_width * page_size > 0x7fffff00LL ||
      (long long)count * ((long long)table_width * page_size / kBlock + 1 + kItemCost) > 0x7fffffffLL ||
      prefix_len > 0x7fffff00 || ldq < (long long)n_heads * HD || ldo < (long long)n_heads * HD || (ldq & 3) || (ldo & 3) ||
      (((uintptr_t)q | (uintptr_t)out | (uintptr_t)k_pool | (uintptr_t)v_pool) & 15))
    return PYRITE_E_SHAPE;
  const size_t need = pyrite_cuda_attention_paged_workspace_size(count, n_heads, n_kv_heads, prefix_len, kv_type);
  if (!workspace || workspace_len < need || ((uintptr_t)workspace & 15)) return PYRITE_E_BUFFER;
  int* status = device_status_word();
  if (!status) return PYRITE_E_CUDA;
  AttnWork w{};
  w.q = q;
  w.ldq = ldq;
  w.count = count;
  w.nq = n_heads;
  w.nkv = n_kv_heads;
  w.qscale = (float)(1.4426950408889634 / 11.313708498984761);  // log2(e) / sqrt(128)
  w.status = status;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  void *k = const_cast<void*>(k_pool), *v = const_cast<void*>(v_pool);
  float* ws = static_cast<float*>(workspace);
  switch (kv_type) {
    case F32:
      return launch_attention<float>(w, prefix_pages, prefix_len, block_table, table_stride, kv_lens, table_width, k, v,
                                     kv_type, n_pages, page_size, out, ldo, ws, s);
    case F16:
      return launch_attention<__half>(w, prefix_pages, prefix_len, block_table, table_stride, kv_lens, table_width, k, v,
                                      kv_type, n_pages, page_size, out, ldo, ws, s);
    default:
      return launch_attention<__nv_bfloat16>(w, prefix_pages, prefix_len, block_table, table_stride, kv_lens,
                                             table_width, k, v, kv_type, n_pages, page_size, out, ldo, ws, s);
  }
}

}  // extern "C"
