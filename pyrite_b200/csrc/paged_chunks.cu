// paged_chunks.cu -- attention of several new tokens of every request (a chunk of a
// prompt, drafted tokens) over a paged key/value pool (paged.cuh).
//
// Request i's n_i new tokens are the rows starts[i] .. starts[i + 1] - 1 of q, the last of
// its kv_lens[i] tokens.  Row t of them attends to the prefix that all requests share
// and to the request's own tokens 0 .. kv_lens[i] - n_i + t:
//   o = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),  s_j = q . k_j / sqrt(128).
// A row without a key gives zeros; rows of no request are left as they were.
//
// The sums split over any partition of the keys: a part that has seen some keys is (m, l,
// o) = (max s, sum e^(s - m), sum e^(s - m) v), and parts join by adding l and o, each times
// e^(its m - the largest m).  Scores and statistics are fp32, in base 2 (q is scaled by log2(e) /
// sqrt(128)).
#include "paged_chunks.cuh"
#include "../../include/pyrite_b200.h"

namespace pyr {
namespace {

using namespace chunks;

// ---- joining -----------------------------------------------------------------------------------
// The items that more than one CTA works on: the one that CTA c begins last and others go
// on with.  A warp a row, its parts in the order of the CTAs.  Bound by latency (records, then
// parts: 3 to 5 us), so four CTAs share a run's rows.
constexpr int kJoinBlocks = 4, kJoinWarps = 8;
__global__ void __launch_bounds__(32 * kJoinWarps) chunks_join_kernel(ChunkArgs a) {
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x / kJoinBlocks;
  const int4 rec = a.records[c];
  if (rec.x & kBegins) {
    Piece pc;
    pc.r = request_of(a, rec.y);
    pc.request = rec.y;
    pc.sub = rec.z;
    pc.tile = rec.w;
    const Tile t = tile_of(a, pc);
    int last = c;  // the CTA with the item's last part
    for (int base = c + 1; base < kGrid; base += 32) {
      const unsigned end = __ballot_sync(0xffffffffu, base + lane < kGrid && (a.records[base + lane].x & kEnds));
      if (end) {
        last = base + __ffs(end) - 1;
        break;
      }
    }
    for (int row = (int)(blockIdx.x % kJoinBlocks) * kJoinWarps + warp; row < kRows; row += kJoinBlocks * kJoinWarps) {
      const Query q = query_of(a, pc, t, row);
      if (!q.on) continue;
      float m = -INFINITY, l = 0.f;
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
      constexpr int N = 4;  // parts whose loads are in flight together
      for (int k = c; k <= last; k += N) {
        float2 ml[N];
        float4 x[N];
#pragma unroll
        for (int e = 0; e < N; ++e) {
          ml[e] = make_float2(-INFINITY, 0.f);
          x[e] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (k + e <= last) {
            const float* at = a.parts + ((size_t)(2 * (k + e) + (k + e == c ? 1 : 0)) * kRows + row) * kPart;
            ml[e] = *reinterpret_cast<const float2*>(at);
            x[e] = *reinterpret_cast<const float4*>(at + 4 + 4 * lane);
          }
        }
#pragma unroll
        for (int e = 0; e < N; ++e) {
          if (ml[e].x == -INFINITY) continue;
          const float mn = fmaxf(m, ml[e].x), f = m == -INFINITY ? 0.f : ex2(m - mn), g = ex2(ml[e].x - mn);
          l = l * f + ml[e].y * g;
          o.x = o.x * f + x[e].x * g;
          o.y = o.y * f + x[e].y * g;
          o.z = o.z * f + x[e].z * g;
          o.w = o.w * f + x[e].w * g;
          m = ml[e].x != ml[e].x ? ml[e].x : mn;
        }
      }
      const float inv = m == -INFINITY ? 0.f : 1.f / l;  // no key: zeros
      *reinterpret_cast<float4*>(a.out + (long long)(pc.r.first + q.token) * a.ldo + (size_t)q.head * HD + 4 * lane) =
          make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
    }
  }
  pdl_launch_dependents();
}

int rc(int e) { return e > 0 ? PYRITE_E_CUDA : e; }

bool sizes_ok(int rows, int requests, int n_heads, int n_kv_heads) {
  return rows > 0 && rows <= kMaxRows && requests > 0 && requests <= kMaxRequests && n_heads > 0 && n_heads <= 1024 &&
         n_kv_heads > 0 && n_heads % n_kv_heads == 0;
}

}  // namespace
}  // namespace pyr

using namespace pyr;

extern "C" {

size_t pyrite_cuda_attention_chunks_workspace_size(int rows, int requests, int n_heads, int n_kv_heads, int kv_type) {
  if (!sizes_ok(rows, requests, n_heads, n_kv_heads) || !kv_type_ok(kv_type)) return 0;
  return kGrid * sizeof(int4) + (size_t)2 * kGrid * kRows * kPart * sizeof(float);
}

int pyrite_cuda_attention_chunks(const float* q, long long ldq, const void* k_pool, const void* v_pool, int kv_type,
                                 int n_pages, int page_size, const int* prefix_pages, int prefix_len,
                                 const int* block_table, long long table_stride, int table_width, const int* starts,
                                 const int* kv_lens, int rows, int requests, int n_heads, int n_kv_heads, int head_dim,
                                 float* out, long long ldo, void* workspace, size_t workspace_len, void* stream) {
  if (!kv_type_ok(kv_type)) return PYRITE_E_TYPE;
  if (!q || !k_pool || !v_pool || !block_table || !starts || !kv_lens || !out || (prefix_len > 0 && !prefix_pages))
    return PYRITE_E_BUFFER;
  if (!sizes_ok(rows, requests, n_heads, n_kv_heads) || head_dim != HD || prefix_len < 0 || prefix_len > 0x3fffff00 ||
      !pool_ok(n_pages, page_size, n_kv_heads) || table_width <= 0 || table_stride < 0 ||
      (requests > 1 && table_stride != 0 && table_stride < table_width) ||
      (long long)table_width * page_size > 0x3fffff00LL || ldq < (long long)n_heads * HD ||
      ldo < (long long)n_heads * HD || (ldq & 3) || (ldo & 3) ||
      (((uintptr_t)q | (uintptr_t)out | (uintptr_t)k_pool | (uintptr_t)v_pool) & 15))
    return PYRITE_E_SHAPE;
  // in place: an item's output goes where its own queries were; otherwise it would go over others' that wait
  if (!(out == q && (ldo == ldq || rows == 1)) && rows_overlap(q, ldq, out, ldo, rows, (long long)n_heads * HD))
    return PYRITE_E_BUFFER;
  const size_t need = pyrite_cuda_attention_chunks_workspace_size(rows, requests, n_heads, n_kv_heads, kv_type);
  if (!workspace || workspace_len < need || ((uintptr_t)workspace & 15)) return PYRITE_E_BUFFER;
  int* status = device_status_word();
  if (!status) return PYRITE_E_CUDA;
  ChunkArgs a{};
  a.q = q;
  a.ldq = ldq;
  a.prefix_pages = prefix_pages;
  a.prefix = prefix_len;
  a.table = block_table;
  a.table_stride = table_stride;
  a.width = table_width;
  a.starts = starts;
  a.lens = kv_lens;
  a.rows = rows;
  a.requests = requests;
  a.nq = n_heads;
  a.nkv = n_kv_heads;
  const int group = n_heads / n_kv_heads;
  a.subs = (group + chunks::kRows - 1) / chunks::kRows;
  a.heads = (group + a.subs - 1) / a.subs;
  a.tokens = chunks::kRows / a.heads;
  a.heads_log2 = a.heads & (a.heads - 1) ? -1 : log2_of(a.heads);
  a.ps_log2 = log2_of(page_size);
  a.n_pages = n_pages;
  a.box_log2 = a.ps_log2 < 7 ? a.ps_log2 : 7;
  a.out = out;
  a.ldo = ldo;
  a.qscale = (float)(1.4426950408889634 / 11.313708498984761);  // log2(e) / sqrt(128)
  a.status = status;
  a.records = static_cast<int4*>(workspace);
  a.parts = reinterpret_cast<float*>(a.records + kGrid);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  void *k = const_cast<void*>(k_pool), *v = const_cast<void*>(v_pool);
  if (const int e = launch_chunks_tc(a, k, v, kv_type, s)) return rc(e);
  return rc(launch_pdl(chunks_join_kernel, dim3(kGrid * kJoinBlocks), dim3(32 * kJoinWarps), 0, s, a));
}

}  // extern "C"
