// paged_attention_tc.cu -- the shared prefix on the 5th-generation tensor cores.
//
// All rows of a batch that share a KV head ask the same prefix keys: with R rows
// of G query heads each there are R G query rows against every key, a matrix
// product.  A CTA takes a tile of 128 query rows and a range of 128-key tiles:
//   S = Q K^T        tcgen05.mma, Q and K in shared memory, S (128 x 128) in TMEM
//   P = 2^(S - m)    two threads a query row, read from and written back to TMEM
//   O = P V          tcgen05.mma, P from TMEM, V in shared memory, O in TMEM
// Two groups of 128 threads share a tile, 64 keys each (a row's two threads agree on
// its maximum through shared memory), and S is there twice, so that products and
// exponentials run beside each other:
//   tensor:   QK0 QK1 | PV0 QK2 | PV1 QK3 | PV2 ...
//   threads:      P0  |   P1    |   P2    | ...
// A tile's O is added to fp32 registers one tile later (the matrix unit's additions
// round toward zero: over thousands of keys in TMEM they would drift), 64 columns a
// thread.  Keys and values come by TMA straight from the pool's pages, 16 keys a
// box, in the 128-byte swizzle that the descriptors name; a box of a page outside
// the pool, or past the prefix, is read out of range and so zero.
//
// Planes (see paged_attention.cu): Q is split into 2 (fp16) or 3 (bf16) 16-bit
// values, P likewise; P's planes overwrite the S they came from, 16 keys at a
// time (the third one has columns of its own), so one MMA step's operand is one
// or two runs of 8 columns.
//
// Bound by the matrix unit and the threads that feed it: 4 (fp16) or 6 (bf16) MMA
// passes over every pair.  1024 query rows for each of 4 KV heads against 8191
// bf16 keys take 48 us, 31 us of products at the library's matrix rate (the matrix pipe
// is busy 62% of the cycles): 32 tiles in 4 parts leave 20 of the 148 SMs without work,
// and a tile's softmax takes about as long as its products.
#include <atomic>
#include <cuda.h>

#include "kernels.cuh"
#include "paged.cuh"
#include "ptx.cuh"
#include "../../include/pyrite_b200.h"

namespace pyr {
namespace {

using namespace ptx;

constexpr int kRows = 128, kKeys = 128;           // query rows and keys of a tile
constexpr int kTcThreads = 320;                   // 2 x 128 softmax, a warp to issue MMAs, a warp to load
constexpr int kMmaWarp = 8, kLoadWarp = 9;
constexpr uint32_t kHalf = 128 * 128;             // bytes of 128 rows of 64 16-bit values
constexpr uint32_t kTileBytes = 2 * kHalf;
// TMEM columns
constexpr uint32_t kS = 0, kO = 256, kX = 384;    // S0, S1 (128 each); O; third planes (64 each)

template <typename T> struct Planes;
template <> struct Planes<__half> { static constexpr int n = 2, format = 0; };
template <> struct Planes<__nv_bfloat16> { static constexpr int n = 3, format = 1; };

struct TcArgs {
  AttnWork w;
  int split;    // CTAs a (KV head, query tile)
  int tiles;    // query tiles of a KV head
  int ps_log2;
  int n_pages;
};

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
  tc_mma_bf16(d, a, b, id, acc);
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
// off instead of rounded (8 bits a plane: three leave out less than 2^-23), which
// needs no conversion.
template <typename T> __device__ __forceinline__ uint32_t weight_plane(float& x, float& y, bool rest);
template <> __device__ __forceinline__ uint32_t weight_plane<__half>(float& x, float& y, bool) {
  return plane2<__half>(x, y);
}
template <> __device__ __forceinline__ uint32_t weight_plane<__nv_bfloat16>(float& x, float& y, bool rest) {
  const uint32_t a = __float_as_uint(x), b = __float_as_uint(y);
  if (rest) {
    const f32x2 cut = pair(__uint_as_float(a & 0xffff0000u), __uint_as_float(b & 0xffff0000u));
    unpair(fma2(cut, pair(-1.f, -1.f), pair(x, y)), x, y);
  }
  return __byte_perm(a, b, 0x7632);
}

template <typename T>
__global__ void __launch_bounds__(kTcThreads, 1)
    prefix_tc_kernel(TcArgs a, const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map) {
  constexpr int NP = Planes<T>::n;
  constexpr uint32_t kIdQK = idesc(Planes<T>::format, kRows, kKeys, false);
  constexpr uint32_t kIdPV = idesc(Planes<T>::format, kRows, 128, true);
  extern __shared__ __align__(128) uint8_t raw[];
  const uint32_t raw0 = smem_addr(raw), sq = (raw0 + 1023u) & ~1023u;
  const uint32_t sk = sq + NP * kTileBytes, sv = sk + 2 * kTileBytes, bars = sv + 2 * kTileBytes;
  uint8_t* mem = raw + (sq - raw0);
  const uint32_t qfull = bars, ofree = bars + 8;
  auto kfull = [&](int s) { return bars + 16 + 8 * s; };
  auto vfull = [&](int s) { return bars + 32 + 8 * s; };
  auto vempty = [&](int s) { return bars + 48 + 8 * s; };
  auto sfull = [&](int s) { return bars + 64 + 8 * s; };
  auto pready = [&](int s) { return bars + 80 + 8 * s; };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(mem + (bars - sq) + 96);
  volatile int* gave_up = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const AttnWork& w = a.w;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int item = blockIdx.x / a.split, part_no = blockIdx.x % a.split;
  const int kvh = item / a.tiles, tile = item % a.tiles;
  const int all = (w.fixed_len + kKeys - 1) / kKeys;
  const int first = (int)((long long)all * part_no / a.split), n = (int)((long long)all * (part_no + 1) / a.split) - first;

  if (tid == 0) {
    mbar_init(qfull, 256);
    mbar_init(ofree, 256);
    for (int s = 0; s < 2; ++s) {
      mbar_init(kfull(s), 1);
      mbar_init(vfull(s), 1);
      mbar_init(vempty(s), 1);
      mbar_init(sfull(s), 1);
      mbar_init(pready(s), 256);
    }
    fence_mbar_init();
    *gave_up = 0;
  }
  if (warp == kMmaWarp) {
    tmem_alloc(smem_addr(tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();
  pdl_launch_dependents();  // the own keys' launch (see begin_part)

  // a bounded wait that gives up at once after any earlier time-out
  auto wait = [&](uint32_t bar, int parity) {
    if (*gave_up) return;
    if (!mbar_wait_bounded(bar, (uint32_t)parity & 1u)) {
      *gave_up = 1;
      atomicOr(w.status, (int)kStatusWaitTimeout);
    }
  };

  if (warp == kLoadWarp) {
    // ---------------- keys and values, 16 at a time ----------------
    if (lane == 0) {
      const int ps = 1 << a.ps_log2;
      for (int i = 0; i < n; ++i) {
        const int t0 = (first + i) * kKeys, s = i & 1;
        int page[8];
#pragma unroll
        for (int g = 0; g < 8; ++g) {
          const int t = t0 + 16 * g;
          page[g] = t < w.fixed_len ? w.pages[t >> a.ps_log2] : -1;
          if (page[g] < 0 || page[g] >= a.n_pages) page[g] = a.n_pages;  // out of range: zeros
        }
        for (int kv = 0; kv < 2; ++kv) {
          const uint32_t bar = kv ? vfull(s) : kfull(s), dst = (kv ? sv : sk) + s * kTileBytes;
          if (i >= 2) wait(kv ? vempty(s) : sfull(s), (i >> 1) - 1);  // S ready: its keys have been read
          if (*gave_up) break;
          mbar_expect_tx(bar, kTileBytes);
#pragma unroll
          for (int g = 0; g < 8; ++g) {
            const int y = kvh * ps + ((t0 + 16 * g) & (ps - 1));
            tma_box(dst + g * 2048, kv ? &v_map : &k_map, 0, y, page[g], bar);
            tma_box(dst + kHalf + g * 2048, kv ? &v_map : &k_map, 64, y, page[g], bar);
          }
        }
        if (*gave_up) break;
      }
    }
  } else if (warp == kMmaWarp) {
    // ---------------- matrix products ----------------
    wait(qfull, 0);
    auto qk = [&](int i) {
      const int s = i & 1;
      wait(kfull(s), i >> 1);
      tc_fence_after();
      if (elect_one()) {
        // small planes first: the chain of truncated additions starts near zero
#pragma unroll
        for (int p = NP - 1; p >= 0; --p)
#pragma unroll
          for (int ks = 0; ks < 8; ++ks) {
            const uint32_t off = (uint32_t)(ks >> 2) * kHalf + (uint32_t)(ks & 3) * 32;
            mma_ss(tmem + kS + 128 * s, desc_sw128(sq + p * kTileBytes + off), desc_sw128(sk + s * kTileBytes + off),
                   kIdQK, p != NP - 1 || ks != 0 ? 1u : 0u);
          }
        tc_commit(sfull(s));
      }
      __syncwarp();
    };
    if (n > 0) qk(0);
    if (n > 1) qk(1);
    for (int j = 0; j < n; ++j) {
      const int s = j & 1;
      wait(pready(s), j >> 1);
      wait(vfull(s), j >> 1);
      if (j > 0) wait(ofree, j - 1);
      tc_fence_after();
      if (elect_one()) {
#pragma unroll
        for (int p = NP - 1; p >= 0; --p)
#pragma unroll
          for (int ks = 0; ks < 8; ++ks) {
            const uint32_t at = p == 2 ? kX + 64 * s + 8 * ks : kS + 128 * s + 16 * ks + 8 * p;
            mma_ts(tmem + kO, tmem + at, desc_v(sv + s * kTileBytes + ks * 2048), kIdPV,
                   p != NP - 1 || ks != 0 ? 1u : 0u);
          }
        tc_commit(vempty(s));
      }
      __syncwarp();
      if (j + 2 < n) {
        wait(vempty(s), j >> 1);  // P of this tile has been read: its columns take the next S
        qk(j + 2);
      }
    }
  } else if (warp < kMmaWarp) {
    // ---------------- softmax: a query row is two threads, one a group, 64 keys of a tile each ----------------
    const int wg = warp >> 2, row = tid & 127;
    const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
    const int group = w.nq / w.nkv;
    // the planes of Q: a warp takes 16 rows, a lane 4 of a row's values
    // the maxima of both groups' keys, [tile % 2][group][row]; before the second tile
    // its half holds the rows' scales, at the end the first half one group's sums
    float* row_max = reinterpret_cast<float*>(mem + (bars - sq) + 128);
    float* row_mul = row_max + 2 * kRows;
    {
      float4 v[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int r = tile * kRows + 16 * warp + i;
        v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (r < w.count * group)
          v[i] = *reinterpret_cast<const float4*>(w.q + (long long)(r / group) * w.ldq +
                                                  (size_t)(kvh * group + r % group) * 128 + 4 * lane);
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int qr = 16 * warp + i;
        float4& x = v[i];
        x.x *= w.qscale; x.y *= w.qscale; x.z *= w.qscale; x.w *= w.qscale;
        float back = 1.f;
        if (sizeof(T) == 2 && Planes<T>::format == 0) {
          float mx = fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w)));
#pragma unroll
          for (int off = 16; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
          const float down = row_scale<T>(mx, back);
          x.x *= down; x.y *= down; x.z *= down; x.w *= down;
        }
        if (lane == 0) row_mul[qr] = back;
        const int c = (lane & 15) >> 1;  // 16-byte chunk of the row's half
        const uint32_t at = sq + (lane >> 4) * kHalf + qr * 128 + ((c ^ (qr & 7)) << 4) + (lane & 1) * 8;
#pragma unroll
        for (int p = 0; p < NP; ++p) {
          const uint32_t b0 = plane2<T>(x.x, x.y), b1 = plane2<T>(x.z, x.w);
          asm volatile("st.shared.v2.u32 [%0], {%1,%2};" ::"r"(at + p * kTileBytes), "r"(b0), "r"(b1) : "memory");
        }
      }
    }
    fence_proxy_async();
    mbar_arrive(qfull);
    named_bar_sync(1, 256);  // row_mul
    const float qmul = row_mul[row];
    f32x2 o[32];  // columns 64 wg .. of the row's output
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int d = 0; d < 32; ++d) o[d] = 0;
    const uint32_t to = tmem + lanes + kO + 64 * wg;
    // O of tile j: a scaled sum, once its products are done
    auto add_o = [&](int j, float f) {
      wait(vempty(j & 1), j >> 1);
      tc_fence_after();
      const f32x2 f2 = pair(f, f);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float s[32];
        tmem_ld32(to + 32 * c, s);
        tmem_wait_ld32(s);
#pragma unroll
        for (int e = 0; e < 16; ++e) o[16 * c + e] = fma2(pair(s[2 * e], s[2 * e + 1]), f2, o[16 * c + e]);
      }
      tc_fence_before();
      mbar_arrive(ofree);
    };
    // the page of this lane's 16-key group of tile j, read a tile ahead
    auto page_of = [&](int j) {
      const int t = (first + j) * kKeys + 16 * lane;
      return j < n && lane < 8 && t < w.fixed_len ? w.pages[t >> a.ps_log2] : 0;
    };
    int page = page_of(0);
    for (int j = 0; j < n; ++j) {
      const int st = j & 1, valid = min(kKeys, w.fixed_len - (first + j) * kKeys);
      const uint32_t ts = tmem + lanes + kS + 128 * st + 64 * wg, tx = tmem + lanes + kX + 64 * st + 32 * wg;
      // which groups lie outside the pool
      const unsigned bad = __ballot_sync(0xffffffffu, page < 0 || page >= a.n_pages);
      if (bad && warp == 0 && lane == 0) atomicOr(w.status, (int)kStatusBadPage);
      page = page_of(j + 1);
      wait(sfull(st), j >> 1);
      tc_fence_after();
      float s[64], mx = -INFINITY;
      tmem_ld32(ts, s);
      tmem_ld32(ts + 32, s + 32);
      tmem_wait_ld32(s);
      tmem_wait_ld32(s + 32);
      if (valid < kKeys || bad) {  // keys past the prefix, or without a page
#pragma unroll
        for (int e = 0; e < 64; ++e) {
          const int key = 64 * wg + e;
          if (key >= valid || ((bad >> (key >> 4)) & 1)) s[e] = -INFINITY;
        }
      }
#pragma unroll
      for (int e = 0; e < 64; e += 2) mx = fmaxf(mx, fmaxf(s[e], s[e + 1]));
      mx *= qmul;
      row_max[(st * 2 + wg) * kRows + row] = mx;
      named_bar_sync(1, 256);
      mx = fmaxf(mx, row_max[(st * 2 + (wg ^ 1)) * kRows + row]);
      float f = 1.f;
      if (mx > m + kLazy) {
        f = m == -INFINITY ? 0.f : ex2(m - mx);
        m = mx;
        l *= f;
#pragma unroll
        for (int d = 0; d < 32; ++d) o[d] = fma2(o[d], pair(f, f), 0);
      }
      const float shift = m == -INFINITY ? 0.f : kUp - m;
      const f32x2 mul2 = pair(qmul, qmul), shift2 = pair(shift, shift);
      f32x2 l2 = 0;
#pragma unroll
      for (int h = 0; h < 4; ++h) {  // 16 keys: one step of the product
        float* p = s + 16 * h;
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
          float x, y;
          unpair(fma2(pair(p[e], p[e + 1]), mul2, shift2), x, y);
          p[e] = ex2(x);
          p[e + 1] = ex2(y);
          l2 = add2(l2, pair(p[e], p[e + 1]));
        }
        uint32_t b[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) b[e] = weight_plane<T>(p[2 * (e & 7)], p[2 * (e & 7) + 1], e < 8 || NP == 3);
        tmem_st16(ts + 16 * h, b);
        if (NP == 3) {
#pragma unroll
          for (int e = 0; e < 8; ++e) b[e] = weight_plane<T>(p[2 * e], p[2 * e + 1], false);
          tmem_st8(tx + 8 * h, b);
        }
      }
      float l0, l1;
      unpair(l2, l0, l1);
      l += l0 + l1;
      if (valid & 15) {
        // the prefix's last page goes on past it: those values may be anything, also NaN
        wait(vfull(st), j >> 1);
        for (int e = tid; e < (16 - (valid & 15)) * 16; e += 256)
          sts128(sv + st * kTileBytes + ((e >> 3) & 1) * kHalf + (valid + (e >> 4)) * 128 + (e & 7) * 16, 0, 0, 0, 0);
        fence_proxy_async();
      }
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(pready(st));
      if (j > 0) add_o(j - 1, f);
    }
    add_o(n - 1, 1.f);
    // m, l and o in rows in shared memory, over the tiles (every product is done once
    // both groups have passed the barrier), then out in whole lines
    float* row_l = row_max;
    if (wg == 1) row_l[row] = l;
    named_bar_sync(1, 256);
    float* buf = reinterpret_cast<float*>(mem) + (size_t)row * kPart;
    if (wg == 0) {
      l += row_l[row];
      buf[0] = l != l ? l : m == -INFINITY ? m : m - kUp;  // a NaN score counts however it compares
      buf[1] = l;
    }
#pragma unroll
    for (int d = 0; d < 32; d += 2) {
      float4 v;
      unpair(o[d], v.x, v.y);
      unpair(o[d + 1], v.z, v.w);
      *reinterpret_cast<float4*>(buf + 4 + 64 * wg + 2 * d) = v;
    }
    named_bar_sync(1, 256);
    float* part = w.parts + (size_t)blockIdx.x * kRows * kPart;
    const int rows = min(kRows, w.count * group - tile * kRows);  // rows past the last: left as they are
    for (int e = tid; e < rows * (kPart / 4); e += 256)
      reinterpret_cast<float4*>(part)[e] = reinterpret_cast<const float4*>(mem)[e];
  }
  __syncwarp();
  // after a time-out: copies and products in flight end before the memory is given back
  tc_fence_before();
  __syncthreads();
  if (*gave_up && tid == 0) {
    for (int s = 0; s < 2; ++s) {
      const int last = n - 1 - ((n - 1 - s) & 1);  // the last tile of this stage
      if (last >= 0) {
        (void)mbar_wait_bounded(kfull(s), (uint32_t)(last >> 1) & 1u);
        (void)mbar_wait_bounded(vfull(s), (uint32_t)(last >> 1) & 1u);
        (void)mbar_wait_bounded(vempty(s), (uint32_t)(last >> 1) & 1u);
      }
    }
  }
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                             const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                             CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn encode_fn() {
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

template <typename T> int launch_tc(const TcArgs& a, void* k, void* v, cudaStream_t stream) {
  static std::atomic<bool> smem_set[64];  // idempotent: concurrent first calls only repeat it
  constexpr size_t smem = 896 /* to a 1024-byte boundary */ + (Planes<T>::n + 4) * (size_t)kTileBytes + 128 /* barriers */ + 2048;
  static_assert(smem <= 227 * 1024, "tiles fit one CTA's shared memory");
  static_assert(kRows * kPart * 4 <= (Planes<T>::n + 4) * kTileBytes, "the rows fit over the tiles");
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -4;
  if (!smem_set[dev].load(std::memory_order_acquire)) {
    if (const int e =
            launch_code(cudaFuncSetAttribute(prefix_tc_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem)))
      return e;
    smem_set[dev].store(true, std::memory_order_release);
  }
  EncodeFn encode = encode_fn();
  if (!encode) return -4;
  // the pool as [page][head and token][128]: a box is 16 tokens of one head, half of their values
  const cuuint64_t tokens = (cuuint64_t)a.w.nkv << a.ps_log2;
  const cuuint64_t dims[3] = {128, tokens, (cuuint64_t)a.n_pages}, strides[2] = {256, tokens * 256};
  const cuuint32_t box[3] = {64, 16, 1}, ones[3] = {1, 1, 1};
  CUtensorMap maps[2];
  for (int i = 0; i < 2; ++i)
    if (encode(&maps[i], Planes<T>::format ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
               i ? v : k, dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return -4;
  return launch_pdl(prefix_tc_kernel<T>, dim3((unsigned)(a.w.nkv * a.tiles * a.split)), dim3(kTcThreads), smem, stream, a,
                    maps[0], maps[1]);
}

}  // namespace

// The tiles pay once there is work for them: with 64 query rows a KV head and 4 KV heads
// they break even with the row kernel at 2048 keys (16 us either way; 8000 keys: 21 and
// 24 us), with 128 rows between 512 (16.5 and 14.9 us) and 2048 keys (17.6 and 22 us); with
// 16 or 32 rows, a tile mostly empty, never (8000 keys: 20 and 19 us).
int prefix_tc_split(int query_rows, int n_kv_heads, int prefix_len, int kv_type) {
  if (kv_type == F32 || query_rows < 48 || (long long)query_rows * n_kv_heads * prefix_len < (1 << 19)) return 0;
  const int items = n_kv_heads * ((query_rows + kRows - 1) / kRows), all = (prefix_len + kKeys - 1) / kKeys;
  // One CTA an SM; at least two tiles each: a part is as large as a tile's keys.  Where
  // half the SMs do with at most four tiles each, the other half is left to the own keys,
  // which run beside (16 rows of 8 heads a KV head, 4 KV heads: 6000 keys 23.5 -> 20.2 us,
  // 8000 keys 26.6 -> 22.0 us; with few and long parts it costs: 64 rows of 16 heads behind
  // 800 keys 39 -> 43 us, so parts stay at nine or more).
  const int full = items >= 148 ? 1 : 148 / items, half = 74 / items, most = (all + 1) / 2;
  const int split = half >= 9 && all <= 4 * half ? half : full;
  return split < most ? split : most;
}

int launch_prefix_tc(const AttnWork& w, void* k, void* v, int kv_type, int n_pages, int page_size, int split,
                     cudaStream_t stream) {
  TcArgs a{w, split, (w.count * (w.nq / w.nkv) + kRows - 1) / kRows, log2_of(page_size), n_pages};
  return kv_type == F16 ? launch_tc<__half>(a, k, v, stream) : launch_tc<__nv_bfloat16>(a, k, v, stream);
}

}  // namespace pyr
