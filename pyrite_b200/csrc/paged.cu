// paged.cu -- the key/value cache in pages, for requests of different lengths:
// block tables and slot maps from the requests' lengths, QK norm + RoPE + the
// append into page slots, and the copy of finished cache rows into slots.
// (The attention that reads the pages is in paged_attention.cu.)
//
// A pool holds n_pages pages of page_size tokens, each page one contiguous
// block [n_kv_heads][page_size][128] of the cache type (fp32, fp16 or bf16), so
// the keys of one KV head in one page are one contiguous tile.  Slot s is
// token s % page_size of page s / page_size.
#include "kernels.cuh"
#include "paged.cuh"
#include "../../include/pyrite_b200.h"

namespace pyr {
namespace {

// ---- block tables and slot maps ---------------------------------------------------------
// Request i holds lens[i] tokens in ceil(lens[i] / ps) pages and gets n_i =
// new_tokens[i] more.  Its fresh pages are free_pages[used + first_i ...],
// first_i the exclusive sum of the requests' fresh page counts in request order,
// so the result does not depend on how the work is split.  Every CTA scans all
// requests (at most kTabRequests: a few KB from L2) into shared memory and then
// takes its share of the fresh table entries and of the tokens; a token finds
// its request by a binary search over the starts.  Bound by launch latency for a
// decode step and by its stores for an admission (8 bytes a token).
constexpr int kTabThreads = 512;
constexpr int kTabRequests = 4080;

struct TabArgs {
  const int* lens;
  const int* fresh_tokens;
  int n;
  int ps_log2;
  const int* free_pages;
  int n_free;
  const int* used;
  int* used_out;
  int* table;
  long long table_stride;
  int width;
  int row_stride;  // > 0: request i's tokens at i * row_stride; 0: packed
  int* slots;
  int* positions;
  int capacity;
  int* starts;
  int* kv_lens;
  unsigned* ticket;
  int* status;
};

// Largest i < n with a[i] <= x (a ascending, a[0] <= x).
__device__ __forceinline__ int last_le(const int* a, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(kTabThreads) page_tables_kernel(TabArgs a) {
  extern __shared__ int tab_sh[];
  int* s_start = tab_sh;                     // [n + 1] first token of each request (packed order)
  int* s_first = tab_sh + a.n + 1;           // [n + 1] first fresh page of each request
  int* s_len = tab_sh + 2 * (a.n + 1);       // [n] held tokens; -1: not served
  __shared__ int w_tok[kTabThreads / 32], w_pg[kTabThreads / 32];
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int ps = 1 << a.ps_log2;
  const int used = *a.used;
  const int avail = used >= 0 ? a.n_free - used : 0;
  // each thread scans a run of `per` consecutive requests
  const int per = (a.n + kTabThreads - 1) / kTabThreads;
  const int lo = min(tid * per, a.n), hi = min(lo + per, a.n);
  int tok = 0, pg = 0;
  bool bad = used < 0;
  for (int i = lo; i < hi; ++i) {
    const int len = a.lens[i], nt = a.fresh_tokens[i];
    // a request outside its table row (or of negative size) is not served
    bool ok = len >= 0 && nt >= 0 && (long long)len + nt <= ((long long)a.width << a.ps_log2) &&
              (a.row_stride == 0 || nt <= a.row_stride);
    // in the packed order a request takes its tokens' places; places end at capacity
    const int t = nt > 0 && (ok || a.row_stride == 0) ? min(nt, a.capacity + 1) : 0;
    const int need = ok ? ((len + nt + ps - 1) >> a.ps_log2) - ((len + ps - 1) >> a.ps_log2) : 0;
    bad |= !ok;
    s_len[i] = ok ? len : -1;
    s_start[i] = tok;  // relative to this thread's run for now
    s_first[i] = pg;
    tok = min(tok + t, a.capacity + 1);  // saturates just past capacity: no overflow
    pg = min(pg + need, a.n_free + 1);
  }
  int tx = tok, px = pg;  // inclusive scans over the warp, then over the warps
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t2 = __shfl_up_sync(0xffffffffu, tx, o), p2 = __shfl_up_sync(0xffffffffu, px, o);
    if (lane >= o) {
      tx = min(tx + t2, a.capacity + 1);
      px = min(px + p2, a.n_free + 1);
    }
  }
  if (lane == 31) { w_tok[warp] = tx; w_pg[warp] = px; }
  __syncthreads();
  int tb = 0, pb = 0;
  for (int w = 0; w < warp; ++w) {
    tb = min(tb + w_tok[w], a.capacity + 1);
    pb = min(pb + w_pg[w], a.n_free + 1);
  }
  int tprev = __shfl_up_sync(0xffffffffu, tx, 1), pprev = __shfl_up_sync(0xffffffffu, px, 1);
  if (lane == 0) tprev = pprev = 0;
  tb = min(tb + tprev, a.capacity + 1);
  pb = min(pb + pprev, a.n_free + 1);
  for (int i = lo; i < hi; ++i) {
    s_start[i] = min(s_start[i] + tb, a.capacity + 1);
    s_first[i] = min(s_first[i] + pb, a.n_free + 1);
  }
  if (tid == kTabThreads - 1) {
    s_start[a.n] = min(tb + tok, a.capacity + 1);
    s_first[a.n] = min(pb + pg, a.n_free + 1);
  }
  __syncthreads();
  // requests whose fresh pages end past the free list, or whose places end past
  // capacity, are not served (and no later one that needs a page is: the sums only grow)
  for (int i = tid; i < a.n; i += kTabThreads) {
    const int len = a.lens[i], nt = a.fresh_tokens[i];
    // (the sums saturate, so whether it needs a page is asked of its own lengths)
    const bool served = s_len[i] >= 0 &&
                        (s_first[i + 1] <= avail ||
                         (len + nt + ps - 1) >> a.ps_log2 == (len + ps - 1) >> a.ps_log2) &&
                        (a.row_stride > 0 || nt == 0 || s_start[i + 1] <= a.capacity);
    if (!served) bad = true;
    if (blockIdx.x == 0) {
      a.kv_lens[i] = served ? len + nt : max(len, 0);
      if (a.starts) a.starts[i] = min(s_start[i], a.capacity);
    }
    if (!served) s_len[i] = -1;
  }
  if (blockIdx.x == 0 && tid == 0 && a.starts) a.starts[a.n] = min(s_start[a.n], a.capacity);
  const bool full = s_first[a.n] > avail || (s_start[a.n] > a.capacity && a.row_stride == 0);
  __syncthreads();
  if (blockIdx.x == 0) {
    if (bad) atomicOr(a.status, (int)kStatusBadPage);
  }
  // used_out may be `used` itself: the CTA that takes the last ticket writes it, when
  // every CTA has read the old value (it has been used above)
  if (tid == 0 && (gridDim.x == 1 || atomicAdd(a.ticket, 1u) == gridDim.x - 1)) {
    // end of the last served request's pages; served ends ascend, so when the list
    // or the places run out the last served request with pages decides
    int served_pg = full ? 0 : s_first[a.n];
    for (int i = a.n - 1; i >= 0 && full; --i)
      if (s_len[i] >= 0 && s_first[i + 1] > s_first[i]) {
        served_pg = s_first[i + 1];
        break;
      }
    *a.used_out = used + served_pg;
    if (gridDim.x > 1) *a.ticket = 0u;
  }
  const int total_pg = min(s_first[a.n], max(avail, 0));
  const int gtid = blockIdx.x * kTabThreads + tid, gsz = gridDim.x * kTabThreads;
  // fresh table entries
  for (int p = gtid; p < total_pg; p += gsz) {
    const int i = last_le(s_first, a.n, p);
    const int len = s_len[i];
    if (len < 0) continue;
    const int has = (len + ps - 1) >> a.ps_log2;
    a.table[(long long)i * a.table_stride + has + (p - s_first[i])] = a.free_pages[used + p];
  }
  // tokens: slots and positions, four in a row a thread; a page id whose slots pass 31
  // bits, or a negative one, belongs to no pool
  const int last_page = 0x7fffffff >> a.ps_log2;
  bool no_page = false;
  const bool wide = (((uintptr_t)a.slots | (uintptr_t)a.positions) & 15) == 0;
  for (int g0 = 4 * gtid; g0 < a.capacity; g0 += 4 * gsz) {
    int i = a.row_stride > 0 ? min(g0 / a.row_stride, a.n - 1) : last_le(s_start, a.n, g0);
    int slot[4], pos[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int g = g0 + e;
      int t;
      if (a.row_stride > 0) {
        while (i + 1 < a.n && g >= (i + 1) * a.row_stride) ++i;
        t = g - i * a.row_stride;
      } else {
        while (i + 1 < a.n && g >= s_start[i + 1]) ++i;
        t = g - s_start[i];
      }
      slot[e] = pos[e] = -1;
      const int len = s_len[i];
      if (t < s_start[i + 1] - s_start[i] && len >= 0) {
        const int has = (len + ps - 1) >> a.ps_log2;
        pos[e] = len + t;
        const int pi = pos[e] >> a.ps_log2;
        const int page = pi < has ? a.table[(long long)i * a.table_stride + pi]
                                  : a.free_pages[used + s_first[i] + pi - has];
        if (page >= 0 && page <= last_page) slot[e] = (page << a.ps_log2) + (pos[e] & (ps - 1));
        else no_page = true;
      }
    }
    if (wide && g0 + 3 < a.capacity) {
      *reinterpret_cast<int4*>(a.slots + g0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
      *reinterpret_cast<int4*>(a.positions + g0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (g0 + e < a.capacity) a.slots[g0 + e] = slot[e], a.positions[g0 + e] = pos[e];
    }
  }
  if (no_page) atomicOr(a.status, (int)kStatusBadPage);
  pdl_launch_dependents();
}

// 1 / sqrt(v): the fp32 root is good to 2^-22, one Newton step squares that.  Outside
// fp32's comfortable range (and for 0, infinities and NaN) the root itself.
__device__ __forceinline__ double inverse_root(double v) {
  if (!(v > 1e-30 && v < 1e30)) return 1.0 / sqrt(v);
  const double y = rsqrtf((float)v);
  return y * fma(-0.5 * v * y, y, 1.5);
}

// ---- QK norm, RoPE and the append into page slots ------------------------------------------
// qk_rope_kv_rows_kernel's arithmetic (fp64 sums and rotation, one
// rounding to fp32 for q and one to the cache type for k and v) for rows at
// positions of their own; only the inverse root is made from fp32's, good to 2^-43,
// far below the 2^-24 of the rounding behind it.  One warp per (row, head): lane l holds the pairs
// (2l, 2l + 64) and (2l + 1, 2l + 65), so a rotated pair is in one lane and every
// access of the warp is 256 bytes (128 in 16-bit caches).  1537 rows of 40 heads take
// 18.3 us from HBM (the bytes alone 9.4 us) and 12.6 to 13.4 us from L2, where a step's qkv is
// (13.8 us with a root and a division in fp64): more rows in flight would help, but the
// fp64 values take 48 registers, and loading ahead (64 to 76 registers) gained 0.9 us from
// HBM and lost 1 from L2.
template <typename T>
__global__ void __launch_bounds__(256) append_paged_kernel(const float* __restrict__ qkv, long long ldqkv,
                                                           const float* __restrict__ qnw,
                                                           const float* __restrict__ knw, int nq, int nkv, double eps,
                                                           int first, const int* __restrict__ positions,
                                                           const int* __restrict__ slots, int count,
                                                           const double2* __restrict__ rope, int max_ctx,
                                                           float* __restrict__ qout, long long ldq, PagePool<T> pool,
                                                           int* status) {
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int j = blockIdx.x, heads = nq + 2 * nkv;
  const int own = positions[j], slot = slots[j];
  const long long pos = (long long)first + own;
  const bool at = own >= 0 && pos < max_ctx;
  const long long total_slots = (long long)pool.n_pages << pool.ps_log2;
  const bool store = slot >= 0 && slot < total_slots;
  if (threadIdx.x == 0 && (slot >= total_slots || slot < -1 || (!at && slot >= 0))) atomicOr(status, (int)kStatusBadPage);
  if (at) {
    const double2* rr = rope + (size_t)pos * 64;
    const double2 c0 = rr[2 * lane], c1 = rr[2 * lane + 1];
    for (int h = blockIdx.y * 8 + warp; h < heads; h += gridDim.y * 8) {
      if (h >= nq && !store) continue;
      const float2* src = reinterpret_cast<const float2*>(qkv + (size_t)j * ldqkv + (size_t)h * 128);
      const float2 a = src[lane], b = src[lane + 32];
      if (h >= nq + nkv) {  // v: stored as it is
        pool.store2(pool.v, slot, h - nq - nkv, nkv, lane, a.x, a.y, b.x, b.y);
        continue;
      }
      double x0 = a.x, x1 = a.y, y0 = b.x, y1 = b.y;
      const float* nw = h < nq ? qnw : knw;
      if (nw) {
        double ss = x0 * x0 + x1 * x1 + y0 * y0 + y1 * y1;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const double inv = inverse_root(fma(ss, 1.0 / 128.0, eps));
        const float2 w0 = reinterpret_cast<const float2*>(nw)[lane], w1 = reinterpret_cast<const float2*>(nw)[lane + 32];
        x0 *= inv * w0.x; x1 *= inv * w0.y; y0 *= inv * w1.x; y1 *= inv * w1.y;
      }
      const double u0 = x0 * c0.x - y0 * c0.y, v0 = x0 * c0.y + y0 * c0.x;
      const double u1 = x1 * c1.x - y1 * c1.y, v1 = x1 * c1.y + y1 * c1.x;
      if (h < nq) {
        float2* dst = reinterpret_cast<float2*>(qout + (size_t)j * ldq + (size_t)h * 128);
        dst[lane] = make_float2((float)u0, (float)u1);
        dst[lane + 32] = make_float2((float)v0, (float)v1);
      } else {
        pool.store2(pool.k, slot, h - nq, nkv, lane, u0, u1, v0, v1);
      }
    }
  }
  pdl_launch_dependents();
}

// Rows of one-sequence fp32 caches (ld floats apart) into slots: a copy with one rounding
// (1537 rows of 4 heads to fp16 4.2 us, the bytes alone 1.5; 64 rows 2.9: launches).
template <typename T>
__global__ void __launch_bounds__(256) store_paged_kernel(const float* __restrict__ k, const float* __restrict__ v,
                                                          long long ld, const int* __restrict__ slots, int nkv,
                                                          PagePool<T> pool, int* status) {
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, j = blockIdx.x;
  const int slot = slots[j];
  const long long total_slots = (long long)pool.n_pages << pool.ps_log2;
  if ((slot >= total_slots || slot < -1) && threadIdx.x == 0) atomicOr(status, (int)kStatusBadPage);
  if (slot >= 0 && slot < total_slots) {
    for (int h = warp; h < 2 * nkv; h += 8) {
      const int kh = h < nkv ? h : h - nkv;
      const float2* src = reinterpret_cast<const float2*>((h < nkv ? k : v) + (size_t)j * ld + (size_t)kh * 128);
      const float2 a = src[lane], b = src[lane + 32];
      pool.store2(h < nkv ? pool.k : pool.v, slot, kh, nkv, lane, a.x, a.y, b.x, b.y);
    }
  }
  pdl_launch_dependents();
}

// The end of a step for requests at positions of their own: request j (live
// while fresh[j] == 1) has run position pos[j].  Its next position p = pos[j] + 1
// holds the prompt's token or takes the sampled ids[j]; current[j] is the token
// the next step runs.  A request stops (fresh[j] = 0) when the token at its last
// position, limits[j] - 1, is known, or when no token could be sampled (-1).
__global__ void __launch_bounds__(128) commit_tokens_kernel(const int* __restrict__ ids, int count,
                                                            int* __restrict__ tokens, long long stride,
                                                            int* __restrict__ pos, int* __restrict__ fresh,
                                                            int* __restrict__ current,
                                                            const int* __restrict__ prompt_lens,
                                                            const int* __restrict__ limits) {
  pdl_wait();
  const int j = blockIdx.x * blockDim.x + threadIdx.x;
  if (j < count && fresh[j] == 1) {
    const int p = pos[j] + 1, lim = (int)min((long long)limits[j], stride);
    pos[j] = p;
    int next = -1;
    if (p >= 0 && p < lim) {
      int* t = tokens + (size_t)j * stride + p;
      if (p >= prompt_lens[j]) *t = ids[j];
      next = *t;
      current[j] = next;
    }
    if (p + 1 >= lim || next < 0) fresh[j] = 0;
  }
  pdl_launch_dependents();
}

int rc(int e) { return e > 0 ? PYRITE_E_CUDA : e; }

template <typename T>
int launch_append(const float* qkv, long long ldqkv, const float* qn, const float* kn, int nq, int nkv, double eps,
                  int first, const int* positions, const int* slots, int count, const void* rope, int max_ctx,
                  float* q_out, long long ldq, void* k, void* v, int n_pages, int ps, cudaStream_t s) {
  const PagePool<T> pool{static_cast<T*>(k), static_cast<T*>(v), n_pages, log2_of(ps)};
  const int heads = nq + 2 * nkv;
  // few rows: a warp per head for the shortest chain; many rows: a warp takes
  // several heads of its row and reads the rope row once
  const int gy = count >= 296 ? (heads + 31) / 32 : (heads + 7) / 8;
  return rc(launch_pdl(append_paged_kernel<T>, dim3((unsigned)count, (unsigned)gy), dim3(256), 0, s, qkv, ldqkv, qn, kn,
                       nq, nkv, eps, first, positions, slots, count, static_cast<const double2*>(rope), max_ctx, q_out,
                       ldq, pool, device_status_word()));
}

template <typename T>
int launch_store(const float* k, const float* v, long long ld, const int* slots, int count, int nkv, void* kp, void* vp,
                 int n_pages, int ps, cudaStream_t s) {
  const PagePool<T> pool{static_cast<T*>(kp), static_cast<T*>(vp), n_pages, log2_of(ps)};
  return rc(launch_pdl(store_paged_kernel<T>, dim3((unsigned)count), dim3(256), 0, s, k, v, ld, slots, nkv, pool,
                       device_status_word()));
}

}  // namespace
}  // namespace pyr

using namespace pyr;

extern "C" {

int pyrite_cuda_page_tables(const int* lens, const int* new_tokens, int requests, int page_size, const int* free_pages,
                            int n_free, const int* used, int* used_out, int* table, long long table_stride,
                            int table_width, int row_stride, int* slots, int* positions, int capacity, int* starts,
                            int* kv_lens, unsigned* ticket, void* stream) {
  if (!lens || !new_tokens || !free_pages || !used || !used_out || !table || !slots || !positions || !kv_lens ||
      !ticket || (row_stride == 0 && !starts))
    return PYRITE_E_BUFFER;
  if (requests <= 0 || requests > kTabRequests || !page_size_ok(page_size) || n_free <= 0 || n_free > (1 << 30) ||
      (long long)n_free * page_size > 0x7fffffffLL || table_width <= 0 || table_stride < table_width ||
      (long long)table_width * page_size > 0x7fffffffLL || row_stride < 0 || capacity <= 0 || capacity >= (1 << 30) - 1 ||
      (row_stride > 0 && (long long)requests * row_stride != capacity))
    return PYRITE_E_SHAPE;
  int* status = device_status_word();
  if (!status) return PYRITE_E_CUDA;
  const TabArgs a{lens,  new_tokens, requests,  log2_of(page_size), free_pages, n_free, used,   used_out, table,  table_stride,
                  table_width, row_stride, slots, positions,         capacity,   starts, kv_lens, ticket,  status};
  const int grid = (capacity + 4 * kTabThreads - 1) / (4 * kTabThreads);
  const size_t smem = (size_t)(3 * requests + 2) * sizeof(int);
  static_assert((3 * kTabRequests + 2) * sizeof(int) <= 49152 - 160, "request arrays fit the default shared memory");
  return rc(launch_pdl(page_tables_kernel, dim3(grid < 148 ? grid : 148), dim3(kTabThreads), smem,
                       static_cast<cudaStream_t>(stream), a));
}

int pyrite_cuda_qk_rope_kv_paged(const float* qkv, long long ldqkv, const float* q_norm, const float* k_norm,
                                 int n_heads, int n_kv_heads, int head_dim, double eps, int first,
                                 const int* positions, const int* slots, int count, const void* rope_table,
                                 int max_ctx, float* q_out, long long ldq, void* k_pool, void* v_pool, int kv_type,
                                 int n_pages, int page_size, void* stream) {
  if (!kv_type_ok(kv_type)) return PYRITE_E_TYPE;
  if (!qkv || !positions || !slots || !rope_table || !q_out || !k_pool || !v_pool) return PYRITE_E_BUFFER;
  if (head_dim != 128 || n_heads <= 0 || n_kv_heads <= 0 || n_heads % n_kv_heads || n_heads > 1024 || count <= 0 ||
      count > (1 << 24) || first < 0 || max_ctx <= 0 || !pool_ok(n_pages, page_size, n_kv_heads) ||
      ldqkv < (long long)(n_heads + 2 * n_kv_heads) * 128 || ldq < (long long)n_heads * 128 || (ldqkv & 1) ||
      (ldq & 1) || (((uintptr_t)qkv | (uintptr_t)q_out | (uintptr_t)q_norm | (uintptr_t)k_norm) & 7) ||
      (((uintptr_t)k_pool | (uintptr_t)v_pool | (uintptr_t)rope_table) & 15))
    return PYRITE_E_SHAPE;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (kv_type) {
    case F32:
      return launch_append<float>(qkv, ldqkv, q_norm, k_norm, n_heads, n_kv_heads, eps, first, positions, slots, count,
                                  rope_table, max_ctx, q_out, ldq, k_pool, v_pool, n_pages, page_size, s);
    case F16:
      return launch_append<__half>(qkv, ldqkv, q_norm, k_norm, n_heads, n_kv_heads, eps, first, positions, slots, count,
                                   rope_table, max_ctx, q_out, ldq, k_pool, v_pool, n_pages, page_size, s);
    default:
      return launch_append<__nv_bfloat16>(qkv, ldqkv, q_norm, k_norm, n_heads, n_kv_heads, eps, first, positions, slots,
                                          count, rope_table, max_ctx, q_out, ldq, k_pool, v_pool, n_pages, page_size,
                                          s);
  }
}

int pyrite_cuda_kv_store_paged(const float* k, const float* v, long long ld, const int* slots, int count,
                               int n_kv_heads, int head_dim, void* k_pool, void* v_pool, int kv_type, int n_pages,
                               int page_size, void* stream) {
  if (!kv_type_ok(kv_type)) return PYRITE_E_TYPE;
  if (!k || !v || !slots || !k_pool || !v_pool) return PYRITE_E_BUFFER;
  if (head_dim != 128 || n_kv_heads <= 0 || count <= 0 || count > (1 << 24) ||
      !pool_ok(n_pages, page_size, n_kv_heads) || ld < (long long)n_kv_heads * 128 || (ld & 1) ||
      (((uintptr_t)k | (uintptr_t)v) & 7) || (((uintptr_t)k_pool | (uintptr_t)v_pool) & 15))
    return PYRITE_E_SHAPE;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (kv_type) {
    case F32: return launch_store<float>(k, v, ld, slots, count, n_kv_heads, k_pool, v_pool, n_pages, page_size, s);
    case F16: return launch_store<__half>(k, v, ld, slots, count, n_kv_heads, k_pool, v_pool, n_pages, page_size, s);
    default:
      return launch_store<__nv_bfloat16>(k, v, ld, slots, count, n_kv_heads, k_pool, v_pool, n_pages, page_size, s);
  }
}

int pyrite_cuda_commit_tokens(const int* ids, int count, int* tokens, long long tok_stride, int* pos, int* fresh,
                              int* current, const int* prompt_lens, const int* limits, void* stream) {
  if (!ids || !tokens || !pos || !fresh || !current || !prompt_lens || !limits) return PYRITE_E_BUFFER;
  if (count <= 0 || count > (1 << 24) || tok_stride <= 0) return PYRITE_E_SHAPE;
  return rc(launch_pdl(commit_tokens_kernel, dim3((unsigned)((count + 127) / 128)), dim3(128), 0,
                       static_cast<cudaStream_t>(stream), ids, count, tokens, tok_stride, pos, fresh, current,
                       prompt_lens, limits));
}

}  // extern "C"
