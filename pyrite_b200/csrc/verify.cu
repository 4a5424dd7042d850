// verify.cu -- drafted tokens against the target's probabilities, from given random
// numbers.
//
// Request i has the rows starts[i] .. starts[i + 1] - 1 of target probabilities p: the
// distribution of the token that follows 0, 1, ... of its drafted tokens, the last row
// the one behind all of them.  Draft x of row r is accepted while u[r] q_r(x) < p_r(x),
// q the distribution that it was drawn from (none given: q(x) = 1).  At the first
// refusal the token comes from max(p - q, 0), behind the last draft from p: then every
// token has the probabilities p, whatever q is.  A token from weights w is the first, in id
// order, whose cumulative weight exceeds pick[i] times their sum.
//
// p and q are fp32: u q(x) is exact in fp64, and p - q too but for q far below p (rounded
// to 2^-53), so a decision is the definition's; sums are fp64, in an order that does not
// depend on the launch's timing.
#include "kernels.cuh"
#include "ptx.cuh"
#include "../../include/pyrite_b200.h"

namespace pyr {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kWide = 4 * 32;  // tokens of a warp's step

struct VerifyArgs {
  const float* p;
  long long ldp;
  const float* q;  // NULL: drafts without a distribution
  long long ldq;
  int n, rows;
  const int* drafts;
  const int* starts;
  const float* accept;
  const float* pick;
  int* out;
  int* counts;
  int slice, segment;  // tokens of a CTA, of a warp: multiples of kWide
  int* status;
};

__device__ __forceinline__ float positive(float x) { return x > 0.f ? x : 0.f; }  // NaN and negative: 0

// The two weights of a token: from p, and from what p has beyond q.
struct Row {
  const float* p;
  const float* q;  // NULL: one draft, `draft` (or -1: no draft)
  int n, draft;
  __device__ __forceinline__ double rest(float p, float q, int i) const {
    if (this->q) return fmax((double)p - (double)q, 0.0);
    return i == draft ? 0.0 : (double)p;
  }
  // four tokens from i on; past the end: 0.  wide: both rows begin on 16 bytes
  __device__ __forceinline__ void load(int i, bool wide, float (&a)[4], float (&b)[4]) const {
    if (wide && i + 4 <= n) {
      const float4 x = __ldg(reinterpret_cast<const float4*>(p + i));
      a[0] = x.x, a[1] = x.y, a[2] = x.z, a[3] = x.w;
      float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
      if (q) y = __ldg(reinterpret_cast<const float4*>(q + i));
      b[0] = y.x, b[1] = y.y, b[2] = y.z, b[3] = y.w;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        a[e] = i + e < n ? __ldg(p + i + e) : 0.f;
        b[e] = q && i + e < n ? __ldg(q + i + e) : 0.f;
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) a[e] = positive(a[e]), b[e] = positive(b[e]);
  }
};

// A cluster per request: each CTA has a slice of the row, each warp a segment of it.  Bound by
// the chain of starts, drafts, sums, cluster barrier and segment: 1 request of 7 drafts over 151936
// tokens 8.7 us, 16 requests of 4 drafts over 128256 with the drafts' distributions 10.5 (2.5 for
// the bytes).  40 of them 17 (6.3 for the bytes) and 128 of them 44 (20): three CTAs run on an SM, so their 320 and
// 1024 CTAs are 0.7 and 2.3 waves of that chain, and both sums are formed for every token, though one is used.
// First the segments' sums, which cross the cluster; then the CTA in which the target lies
// finds the token in the segment that holds it.
__global__ void __launch_bounds__(kThreads) verify_drafts_kernel(VerifyArgs a) {
  __shared__ double seg[2][kWarps];
  __shared__ double total[2][kMaxCluster];  // of every CTA
  __shared__ double step_sum[kWarps];
  __shared__ int step_last[kWarps], hit_at;
  const uint32_t C = ptx::cluster_nctarank(), rank = ptx::cluster_ctarank();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, j = (int)(blockIdx.x / C);
  // every CTA of the cluster runs before another writes to its shared memory
  asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");
  pdl_wait();
  const int first = min(max(a.starts[j], 0), a.rows), end = min(max(a.starts[j + 1], first), a.rows);
  const int drafts = end - first - 1;
  if (rank == 0 && threadIdx.x == 0 && a.starts[j + 1] < a.starts[j]) atomicOr(a.status, (int)kStatusBadPage);  // rows of several requests
  asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
  if (drafts < 0) {  // a request without a row
    if (rank == 0 && threadIdx.x == 0) a.counts[j] = 0;
    pdl_launch_dependents();
    return;
  }
  // the first draft that is refused: 32 at a time, every warp for itself
  int taken = drafts;
  for (int t0 = 0; t0 < drafts; t0 += 32) {
    bool good = true;
    if (t0 + lane < drafts) {
      const int r = first + t0 + lane, x = a.drafts[r];
      good = false;
      if (x >= 0 && x < a.n) {
        const double q = a.q ? (double)positive(a.q[(long long)r * a.ldq + x]) : 1.0;
        good = (double)a.accept[r] * q < (double)a.p[(long long)r * a.ldp + x];
      }
    }
    const unsigned no = __ballot_sync(0xffffffffu, !good);
    if (no) {
      taken = t0 + __ffs(no) - 1;
      break;
    }
  }
  const int r = first + taken;
  const int x = taken < drafts ? a.drafts[r] : -1;
  const bool draft = x >= 0 && x < a.n;  // refused; otherwise the token comes from p itself
  const Row row{a.p + (long long)r * a.ldp, draft && a.q ? a.q + (long long)r * a.ldq : nullptr, a.n, draft ? x : -1};
  const bool wide = (((uintptr_t)row.p | (uintptr_t)row.q) & 15) == 0;
  const int lo = (int)rank * a.slice + warp * a.segment;
  double s0 = 0, s1 = 0;  // of p, of the rest
#pragma unroll 4
  for (int i = lo + 4 * lane; i < lo + a.segment; i += kWide) {
    float pv[4], qv[4];
    row.load(i, wide, pv, qv);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      s0 += (double)pv[e];
      s1 += row.rest(pv[e], qv[e], i + e);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    s0 += __shfl_xor_sync(0xffffffffu, s0, o);
    s1 += __shfl_xor_sync(0xffffffffu, s1, o);
  }
  if (lane == 0) seg[0][warp] = s0, seg[1][warp] = s1;
  __syncthreads();
  if (threadIdx.x < 2 * C) {
    const int w = threadIdx.x & 1;
    double s = 0;
    for (int i = 0; i < kWarps; ++i) s += seg[w][i];
    uint32_t to;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(ptx::smem_addr(&total[w][rank])), "r"(threadIdx.x >> 1));
    asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(to), "d"(s) : "memory");
  }
  ptx::cluster_sync();
  // the weights are those of the rest, or of p where nothing is left
  double base[2] = {0, 0}, all[2] = {0, 0};
  for (uint32_t c = 0; c < C; ++c)
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      if (c == rank) base[w] = all[w];
      all[w] += total[w][c];
    }
  const int w = all[1] > 0.0 ? 1 : 0;
  const float u = a.pick[j];
  const double target = (u > 0.f ? (double)fminf(u, 0.99999994f) : 0.0) * all[w];
  const bool any = all[w] > 0.0 && all[w] < __longlong_as_double(0x7ff0000000000000LL);
  if (rank == 0) {
    for (int t = threadIdx.x; t <= drafts; t += kThreads)
      if (t != taken) a.out[first + t] = t < taken ? a.drafts[first + t] : -1;
    if (threadIdx.x == 0) {
      a.counts[j] = any ? taken + 1 : taken;
      if (!any) a.out[r] = -1;
    }
  }
  if (any && base[w] <= target && target < base[w] + total[w][rank]) {
    // this CTA's warp whose segment the target falls in
    double at = base[w];
    int mine = -1, last = 0;
    double from = 0;
    for (int i = 0; i < kWarps; ++i) {
      if (seg[w][i] > 0.0) {
        last = i;
        if (mine < 0 && target < at + seg[w][i]) mine = i, from = at;
      }
      at += seg[w][i];
    }
    if (mine < 0) {  // the sums' roundings: the last segment with a weight, its last token
      mine = last;
      from = -1.0;
    }
    // all warps on that segment, 4 kThreads tokens at a time
    double cum = from < 0.0 ? 0.0 : from;
    const double want = from < 0.0 ? __longlong_as_double(0x7ff0000000000000LL) : target;
    const int start = (int)rank * a.slice + mine * a.segment;
    int behind = -1;
    for (int i0 = start; i0 < start + a.segment; i0 += 4 * kThreads) {
      const int i = i0 + 4 * (int)threadIdx.x;
      float pv[4] = {0.f, 0.f, 0.f, 0.f}, qv[4] = {0.f, 0.f, 0.f, 0.f};
      if (i < start + a.segment) row.load(i, wide, pv, qv);
      double v[4], sum = 0;
      int heavy = -1;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[e] = w ? row.rest(pv[e], qv[e], i + e) : (double)pv[e];
        if (v[e] > 0.0) heavy = i + e;
        sum += v[e];
      }
      double in = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double d = __shfl_up_sync(0xffffffffu, in, o);
        if (lane >= o) in += d;
      }
      if (lane == 31) step_sum[warp] = in;
      heavy = __reduce_max_sync(0xffffffffu, heavy);
      if (lane == 0) step_last[warp] = heavy;
      if (threadIdx.x == 0) hit_at = 0x7fffffff;
      __syncthreads();
      double c = cum + (in - sum);
      for (int k = 0; k < kWarps; ++k) {
        if (k < warp) c += step_sum[k];
        cum += step_sum[k];
        behind = max(behind, step_last[k]);
      }
      int hit = -1;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        c += v[e];
        if (hit < 0 && v[e] > 0.0 && c > want) hit = i + e;
      }
      if (hit >= 0) atomicMin(&hit_at, hit);
      __syncthreads();
      const int found = hit_at;
      __syncthreads();
      if (found != 0x7fffffff) {
        behind = found;
        break;
      }
    }
    if (threadIdx.x == 0) a.out[r] = behind;
  }
  pdl_launch_dependents();
}

}  // namespace
}  // namespace pyr

using namespace pyr;

extern "C" {

int pyrite_cuda_verify_drafts(const float* probs, long long ldp, size_t n, size_t rows, const float* draft_probs,
                              long long ldq, const int* draft_tokens, const int* starts, int requests,
                              const float* accept, const float* pick, int* out, int* counts, void* stream) {
  if (!probs || !draft_tokens || !starts || !accept || !pick || !out || !counts) return PYRITE_E_BUFFER;
  if (n == 0 || n > (1u << 20) || rows == 0 || rows > (1u << 24) || requests <= 0 || requests > 65535 ||
      ldp < (long long)n || (draft_probs && ldq < (long long)n) || (((uintptr_t)probs | (uintptr_t)draft_probs) & 3))
    return PYRITE_E_SHAPE;
  // in place: a request's entries are read before they are written; another's would not be
  if (out != draft_tokens && rows_overlap(reinterpret_cast<const float*>(draft_tokens), (long long)rows,
                                          reinterpret_cast<const float*>(out), (long long)rows, 1, (long long)rows))
    return PYRITE_E_BUFFER;
  // CTAs a request: while every one finds an SM, of more than 1024 tokens; beyond that, up to eight for an SM
  // (three run at a time), of more than 8192.  In us, one CTA a request against this rule: 16 requests of
  // 128256 tokens 57 and 18, 40 of them 59 and 22, 128 of them 65 and 51; eight CTAs where there are many
  // or rows are short: 400 of 128256 91 -> 125, 128 of 4000 14 -> 27.
  int cluster = 1;
  while (cluster < kMaxCluster && ((requests * cluster * 2 <= 148 && n > (size_t)kThreads * 4 * cluster) ||
                                   (requests * cluster * 2 <= 8 * 148 && n > (size_t)kThreads * 32 * cluster)))
    cluster *= 2;
  const int segment = (int)((n + (size_t)cluster * kWarps * kWide - 1) / ((size_t)cluster * kWarps * kWide)) * kWide;
  int* status = device_status_word();
  if (!status) return PYRITE_E_CUDA;
  const VerifyArgs a{probs, ldp,    draft_probs, ldq, (int)n, (int)rows, draft_tokens,     starts,
                     accept, pick, out,         counts, segment * kWarps, segment,         status};
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(requests * cluster));
  cfg.blockDim = dim3(kThreads);
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
  return launch_code(cudaLaunchKernelEx(&cfg, verify_drafts_kernel, a)) ? PYRITE_E_CUDA : 0;
}

}  // extern "C"
