// paged_attention.cu -- attention of a batch whose requests share a prefix, over
// a paged key/value pool (paged.cuh).
//
// Row b's query heads attend to the P tokens of the shared prefix and then to
// the row's own kv_lens[b] tokens:
//   o = sum_t e^(s_t - m) v_t / sum_t e^(s_t - m),  s_t = q . k_t / sqrt(128).
// The sums split over any partition of the keys: a part that has seen some keys
// is (m, l, o) = (max s, sum e^(s - m), sum e^(s - m) v), and two parts join as
// m = max(m1, m2), l = l1 e^(m1 - m) + l2 e^(m2 - m), o likewise.  So the prefix
// is computed for all rows at once (every key read once per tile of query
// rows, not once per row), the own keys per row, both split over CTAs, and a
// last kernel joins the parts.  A row without a key gives zeros.  Scores and
// statistics are fp32, in base 2 (q is scaled by log2(e) / sqrt(128)).
#include <cfloat>

#include "kernels.cuh"
#include "paged.cuh"
#include "../../include/pyrite_b200.h"

namespace pyr {
namespace {

constexpr int HD = 128;
constexpr int kPart = HD + 4;  // floats of a part: m, l, 2 pad, o[128]
constexpr float kNegInf = -INFINITY;

struct AttnArgs {
  const float* q;
  long long ldq;
  const int* pages;        // prefix: its page list; own: the block table
  long long table_stride;
  const int* lens;         // own: tokens of each row (device); prefix: NULL
  int fixed_len;           // prefix: its length
  int max_pages;           // entries of a page list
  int count, nq, nkv;
  int split0, nsplit;      // this launch writes splits split0 ..; nsplit in all
  float* parts;            // [(row, head)][split][kPart]
  float* out;
  long long ldo;
  float qscale;
  int* status;
};

__device__ __forceinline__ float4 load4(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ float4 load4(const __half* p) {
  const uint2 r = *reinterpret_cast<const uint2*>(p);
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&r.x));
  const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&r.y));
  return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ float4 load4(const __nv_bfloat16* p) {
  const uint2 r = *reinterpret_cast<const uint2*>(p);
  return make_float4(__uint_as_float(r.x << 16), __uint_as_float(r.x & 0xffff0000u), __uint_as_float(r.y << 16),
                     __uint_as_float(r.y & 0xffff0000u));
}

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

// One CTA: a tile of QT query rows that share a key range, 8 warps taking every
// 8th group of 32 / QT keys.  A lane holds 4 of the 128 dimensions of every
// query and accumulator; a group's 32 (query, key) scores are summed by
// transpose_sum, one left to each lane.
template <typename T, int QT>
__global__ void __launch_bounds__(256) attn_simt_kernel(AttnArgs a, PagePool<T> pool) {
  constexpr int KG = 32 / QT;  // keys of a group
  __shared__ float sm_p[8][32];
  __shared__ float sm_m[8][QT], sm_l[8][QT];
  __shared__ __align__(16) float sm_o[8][QT][HD];
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int group = a.nq / a.nkv, ps_log2 = pool.ps_log2, ps = 1 << ps_log2;
  const bool own = a.lens != nullptr;
  // the tile's query rows: own: up to QT heads of one KV head of row b;
  // prefix: QT of the count * group (row, head) pairs of a KV head
  const int tiles = own ? (group + QT - 1) / QT : (a.count * group + QT - 1) / QT;
  const int kvh = (blockIdx.x / tiles) % a.nkv, tile = blockIdx.x % tiles;
  const int b = own ? blockIdx.x / (tiles * a.nkv) : 0;
  const int nrow = own ? group : a.count * group;
  const int* list = a.pages + (own ? (long long)b * a.table_stride : 0);
  const int len = own ? min(max(a.lens[b], 0), a.max_pages << ps_log2) : a.fixed_len;
  const int nsplit = gridDim.y;
  // this CTA's keys: a share of whole pages' 16-key groups
  const int chunk = ((len + nsplit - 1) / nsplit + 15) & ~15;
  const int k0 = min((int)blockIdx.y * chunk, len), k1 = min(k0 + chunk, len);

  float4 q[QT], o[QT];
#pragma unroll
  for (int i = 0; i < QT; ++i) {
    const int r = tile * QT + i;
    o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    q[i] = o[i];
    if (r < nrow) {
      const int row = own ? b : r / group, g = own ? r : r % group;
      q[i] = load4(a.q + (long long)row * a.ldq + (size_t)(kvh * group + g) * HD + 4 * lane);
      q[i].x *= a.qscale; q[i].y *= a.qscale; q[i].z *= a.qscale; q[i].w *= a.qscale;
    }
  }
  const int qi = lane / KG, kj = lane % KG;  // this lane's score
  float m = kNegInf, l = 0.f;                // of query qi, l over this lane's keys
  for (int t0 = k0 + warp * KG; t0 < k1; t0 += 8 * KG) {
    const int page = list[t0 >> ps_log2];
    const bool ok = page >= 0 && page < pool.n_pages;
    if (!ok) {  // a page outside the pool: its keys are left out, the status word says so
      if (lane == 0) atomicOr(a.status, (int)kStatusBadPage);
      continue;
    }
    const size_t at = (((size_t)page * a.nkv + kvh) * ps + (t0 & (ps - 1))) * HD + 4 * lane;
    const int n = min(KG, k1 - t0);
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
    const float p = sc == kNegInf ? 0.f : exp2f(sc - mn);
    const float alpha = m == kNegInf ? 0.f : exp2f(m - mn);
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
    sm_m[warp][qi] = m;
    sm_l[warp][qi] = l;
  }
#pragma unroll
  for (int i = 0; i < QT; ++i) *reinterpret_cast<float4*>(&sm_o[warp][i][4 * lane]) = o[i];
  __syncthreads();
  // join the warps; one part per query row
  for (int e = tid; e < QT * HD; e += 256) {
    const int i = e / HD, d = e % HD, r = tile * QT + i;
    if (r >= nrow) continue;
    float M = kNegInf, L = 0.f, O = 0.f;
    for (int w = 0; w < 8; ++w) M = fmaxf(M, sm_m[w][i]);
    for (int w = 0; w < 8; ++w) {
      const float f = sm_m[w][i] == kNegInf ? 0.f : exp2f(sm_m[w][i] - M);
      L += sm_l[w][i] * f;
      O += sm_o[w][i][d] * f;
    }
    const int row = own ? b : r / group, h = kvh * group + (own ? r : r % group);
    float* part = a.parts + (((size_t)row * a.nq + h) * a.nsplit + a.split0 + blockIdx.y) * kPart;
    part[4 + d] = O;
    if (d == 0) {
      part[0] = M;
      part[1] = L;
    }
  }
  pdl_launch_dependents();
}

// Join the parts of one (row, head): 32 threads, 4 dimensions each.
__global__ void __launch_bounds__(128) attn_join_kernel(AttnArgs a) {
  pdl_wait();
  const int rh = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (rh < a.count * a.nq) {
    const float* p = a.parts + (size_t)rh * a.nsplit * kPart;
    float M = kNegInf, L = 0.f;
    float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s = 0; s < a.nsplit; ++s) M = fmaxf(M, p[(size_t)s * kPart]);
    for (int s = 0; s < a.nsplit; ++s) {
      const float* ps = p + (size_t)s * kPart;
      const float ms = ps[0];
      if (ms == kNegInf) continue;
      const float f = exp2f(ms - M);
      const float4 o = load4(ps + 4 + 4 * lane);
      L += ps[1] * f;
      O.x += o.x * f; O.y += o.y * f; O.z += o.z * f; O.w += o.w * f;
    }
    const float inv = L > 0.f ? 1.0f / L : (M == kNegInf ? 0.f : L / 0.f);  // no key: zeros; NaN stays NaN
    const int row = rh / a.nq, h = rh % a.nq;
    *reinterpret_cast<float4*>(a.out + (long long)row * a.ldo + (size_t)h * HD + 4 * lane) =
        make_float4(O.x * inv, O.y * inv, O.z * inv, O.w * inv);
  }
  pdl_launch_dependents();
}

int rc(int e) { return e > 0 ? PYRITE_E_CUDA : e; }

// at least 2: a group of 32 / QT keys then lies inside one 16-token page
int tile_rows(int rows) { return rows >= 5 ? 8 : rows >= 3 ? 4 : 2; }

struct Plan {
  int pre_qt = 0, pre_items = 0, pre_split = 0;
  int own_qt = 0, own_items = 0, own_split = 0;
  int splits() const { return pre_split + own_split; }
};
// Splits: enough CTAs for two per SM, each with at least 64 keys of the prefix.
Plan make_plan(int count, int nq, int nkv, int prefix_len) {
  Plan p;
  const int group = nq / nkv;
  if (prefix_len > 0) {
    p.pre_qt = tile_rows(count * group < 8 ? count * group : 8);
    p.pre_items = nkv * ((count * group + p.pre_qt - 1) / p.pre_qt);
    const int most = (prefix_len + 63) / 64;
    p.pre_split = (2 * 148 + p.pre_items - 1) / p.pre_items;
    if (p.pre_split > most) p.pre_split = most;
  }
  p.own_qt = tile_rows(group);
  p.own_items = count * nkv * ((group + p.own_qt - 1) / p.own_qt);
  p.own_split = (4 * 148 + p.own_items - 1) / p.own_items;
  return p;
}

template <typename T>
int launch_simt(int qt, int items, int split, const AttnArgs& a, const PagePool<T>& pool, cudaStream_t s) {
  const dim3 grid((unsigned)items, (unsigned)split), block(256);
  switch (qt) {
    case 2: return launch_pdl(attn_simt_kernel<T, 2>, grid, block, 0, s, a, pool);
    case 4: return launch_pdl(attn_simt_kernel<T, 4>, grid, block, 0, s, a, pool);
    default: return launch_pdl(attn_simt_kernel<T, 8>, grid, block, 0, s, a, pool);
  }
}

template <typename T>
int launch_attention(AttnArgs a, const int* prefix_pages, int prefix_len, const int* table, const int* lens,
                     int table_width, void* k, void* v, int n_pages, int ps, cudaStream_t s) {
  const PagePool<T> pool{static_cast<T*>(k), static_cast<T*>(v), n_pages, log2_of(ps)};
  const Plan p = make_plan(a.count, a.nq, a.nkv, prefix_len);
  a.nsplit = p.splits();
  if (p.pre_split) {
    AttnArgs pa = a;
    pa.pages = prefix_pages;
    pa.lens = nullptr;
    pa.fixed_len = prefix_len;
    pa.max_pages = (prefix_len + ps - 1) / ps;
    pa.split0 = 0;
    if (int e = launch_simt(p.pre_qt, p.pre_items, p.pre_split, pa, pool, s)) return rc(e);
  }
  a.pages = table;
  a.lens = lens;
  a.max_pages = table_width;
  a.split0 = p.pre_split;
  if (int e = launch_simt(p.own_qt, p.own_items, p.own_split, a, pool, s)) return rc(e);
  return rc(launch_pdl(attn_join_kernel, dim3((unsigned)((a.count * a.nq + 3) / 4)), dim3(128), 0, s, a));
}

}  // namespace
}  // namespace pyr

using namespace pyr;

extern "C" {

size_t pyrite_cuda_attention_paged_workspace_size(int count, int n_heads, int n_kv_heads, int prefix_len,
                                                  int kv_type) {
  if (count <= 0 || count > 4096 || n_heads <= 0 || n_heads > 1024 || n_kv_heads <= 0 || n_heads % n_kv_heads ||
      prefix_len < 0 || !kv_type_ok(kv_type))
    return 0;
  return (size_t)count * n_heads * make_plan(count, n_heads, n_kv_heads, prefix_len).splits() * kPart * sizeof(float);
}

int pyrite_cuda_attention_paged(const float* q, long long ldq, const void* k_pool, const void* v_pool, int kv_type,
                                int n_pages, int page_size, const int* prefix_pages, int prefix_len,
                                const int* block_table, long long table_stride, int table_width, const int* kv_lens,
                                int count, int n_heads, int n_kv_heads, int head_dim, float* out, long long ldo,
                                void* workspace, size_t workspace_len, void* stream) {
  if (!kv_type_ok(kv_type)) return PYRITE_E_TYPE;
  if (!q || !k_pool || !v_pool || !block_table || !kv_lens || !out || (prefix_len > 0 && !prefix_pages))
    return PYRITE_E_BUFFER;
  if (head_dim != HD || count <= 0 || count > 4096 || n_heads <= 0 || n_heads > 1024 || n_kv_heads <= 0 ||
      n_heads % n_kv_heads || prefix_len < 0 || !pool_ok(n_pages, page_size, n_kv_heads) || table_width <= 0 ||
      table_stride < 0 || (count > 1 && table_stride != 0 && table_stride < table_width) ||
      (long long)table_width * page_size > 0x7fffff00LL || prefix_len > 0x7fffff00 || ldq < (long long)n_heads * HD ||
      ldo < (long long)n_heads * HD || (ldq & 3) || (ldo & 3) ||
      (((uintptr_t)q | (uintptr_t)out | (uintptr_t)k_pool | (uintptr_t)v_pool) & 15))
    return PYRITE_E_SHAPE;
  const size_t need = pyrite_cuda_attention_paged_workspace_size(count, n_heads, n_kv_heads, prefix_len, kv_type);
  if (!workspace || workspace_len < need || ((uintptr_t)workspace & 15)) return PYRITE_E_BUFFER;
  int* status = device_status_word();
  if (!status) return PYRITE_E_CUDA;
  AttnArgs a{};
  a.q = q;
  a.ldq = ldq;
  a.table_stride = table_stride;
  a.count = count;
  a.nq = n_heads;
  a.nkv = n_kv_heads;
  a.parts = static_cast<float*>(workspace);
  a.out = out;
  a.ldo = ldo;
  a.qscale = (float)(1.4426950408889634 / 11.313708498984761);  // log2(e) / sqrt(128)
  a.status = status;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  void *k = const_cast<void*>(k_pool), *v = const_cast<void*>(v_pool);
  switch (kv_type) {
    case F32:
      return launch_attention<float>(a, prefix_pages, prefix_len, block_table, kv_lens, table_width, k, v, n_pages,
                                     page_size, s);
    case F16:
      return launch_attention<__half>(a, prefix_pages, prefix_len, block_table, kv_lens, table_width, k, v, n_pages,
                                      page_size, s);
    default:
      return launch_attention<__nv_bfloat16>(a, prefix_pages, prefix_len, block_table, kv_lens, table_width, k, v,
                                             n_pages, page_size, s);
  }
}

}  // extern "C"
