// paged_chunks_tc.cu -- attention of chunks on the 5th-generation tensor cores.
//
// A piece (paged_chunks.cuh) is 128 query rows against a run of 128-key tiles:
//   S = Q K^T        tcgen05.mma, Q and K in shared memory, S (128 x 128) in TMEM
//   P = 2^(S - m)    a thread a query row, read from and written back to TMEM
//   O = P V          tcgen05.mma, P from TMEM, V in shared memory, O in TMEM
// and a tile's O is added to fp32 registers (the matrix unit's additions round toward zero:
// over thousands of keys in TMEM they would drift).
//
// Planes: an fp32 operand is split into 16-bit values whose sum it is.  16-bit caches: Q and P
// into 2 (fp16) or 3 (bf16), K and V are exact.  fp32 caches: Q and K into two fp16 values, P and V into three
// bf16 values, whose range needs no scale; the products of two small planes are left out: below 2^-24 of a term of
// Q K^T, with either sign; below 2^-21 of a term of P V, about 2^-24 on average and always toward zero (bf16 planes are
// cut off, not rounded, so a second one reaches 2^-7 and a third 2^-15 of the first).  A row that goes into fp16 planes takes a power of two that brings its largest value
// to the upper end of fp16 (kHigh): what is left out of a value is below 2^-24 of it, or 2^-38 of the row's largest
// where that is more.  So rows with a few channels far above the others (to 2^14 times) are as good as in
// fp32; with the largest near 1, 2^-25 of it was left out of every value, and a channel at 2000 times the others made the
// rms error of the output 5.0e-5 of it instead of 4.9e-7, in fp32 caches and, for such q, in fp16 ones.
//
// What bounds it: long chunks the tensor pipe (fp16: 4 products of 128 x 128 x 128 a tile, 2048 cycles
// at the nominal rate, of about 3200 that a tile takes; 2048 tokens of 32 heads behind 13001 in 655 us at full clocks, 0.87 of the
// rate that the library's product reaches in a burst, 720 to 820 under the power cap that calls one after the other
// reach).  Short ones bytes and beginnings: 16 requests of 5 drafts behind 3000 tokens
// 48 us (18 for the bytes), of which about 9 from the launch to the first weights (the run 2, its piece and
// the way to the warps 0.5, the first queries 3, mostly instructions that come from L2) and 4 the join; some 17 are
// not accounted for: 20 of a tile's 128 rows are live, and one warp of a group's four makes their weights.  fp32: the making of
// planes, 11 000 of about 12 000 cycles a tile (5000 the keys, 3000 the values, the rest pages and what has
// no register), made again for every query tile of a KV head; 2048 tokens behind 13001 2.6 to 2.9 ms.
// Tried: 16 warps for the weights (no gain: the products wait for O as before), O read 64 columns at a time
// (spills), L2 prefetches by the loading warps of 16-bit caches (slower), runs whose ends move to the ends of
// items nearby (2 us less for tiles of few keys, 2 to 20 us more elsewhere).
#include <atomic>

#include "paged_chunks.cuh"
#include "paged_tc.cuh"
#include "../../include/pyrite_b200.h"

namespace pyr {
namespace {

using namespace ptx;
using namespace tc;
using namespace chunks;

template <typename T> struct Cache {  // 16-bit
  using Q = T;  // operands of Q K^T, of P V
  using P = T;
  static constexpr bool kSplit = false;  // keys and values are operands as they are
  static constexpr int kKeyPlanes = 1, kValuePlanes = 1, kStages = 2;
};
template <> struct Cache<float> {
  using Q = __half;
  using P = __nv_bfloat16;
  static constexpr bool kSplit = true;
  static constexpr int kKeyPlanes = 2, kValuePlanes = 3, kStages = 1;
};
// Groups of four warps make the weights, a thread a query row, each group every G-th tile:
// S stands in TMEM G times.  fp16 takes three (S and O fill the tensor memory), the others, whose
// third planes need the room, two.  From S to its weights a group takes about 3000 cycles, a tile's
// products of two planes each (fp16) 2048, of three (bf16) half as much again, of fp32's three and six 4608.  Behind them four warps that add up O; two that issue
// the two products (a wait that has nothing to wait for costs a warp about 100 cycles, in which the
// other's products run); one that finds the pieces and loads keys, one that loads values (a box takes
// a warp about 60 cycles to issue: one warp for both took longer than a tile's bytes do).  fp32: eight
// more that make the planes of the keys and values.
template <typename T> struct Layout : Cache<T> {
  using C = Cache<T>;
  static constexpr int G = Planes<typename C::P>::n == 2 ? 3 : 2;
  static constexpr int kGroups = G + 2 + (C::kSplit ? 2 : 0), kThreads = 128 * kGroups;
  static constexpr int kSumWarp = 4 * G, kScoreWarp = kSumWarp + 4, kKeyWarp = kScoreWarp + 2, kMakeWarp = kScoreWarp + 4;
  // registers a thread: at the launch, then of each role
  static constexpr int kRegs = C::kSplit ? 80 : G == 3 ? 96 : 128, kSoftRegs = C::kSplit ? 80 : G == 3 ? 88 : 144,
                       kSumRegs = G == 3 || C::kSplit ? 168 : 176, kIssueRegs = C::kSplit ? 40 : 48, kMakeRegs = 56;
  static_assert(G * kSoftRegs + kSumRegs + kIssueRegs + (C::kSplit ? 2 * kMakeRegs : 0) <= kGroups * kRegs,
                "a split of the launch's registers");
  // TMEM columns: S of G tiles, O, third planes (64 each)
  static constexpr uint32_t kO = 128 * G, kX = kO + 128;
  static constexpr int kRing = C::kSplit ? 2 : 4;  // pieces found ahead
  static constexpr uint32_t kQBytes = Planes<typename C::Q>::n * kTileBytes,
                            kKBytes = C::kStages * C::kKeyPlanes * kTileBytes,
                            kVBytes = C::kStages * C::kValuePlanes * kTileBytes;
  static constexpr bool kScaled = Planes<typename C::Q>::format == 0;  // fp16: rows of Q (and of split keys) have scales
  static constexpr uint32_t kSmem = kQBytes + kKBytes + kVBytes + 336 + kRing * 64 + (C::kSplit ? 1 : 2) * G * kRows * 4 +
                                    (kScaled ? (G + 1) * kRows * 2 : 0) + (C::kSplit ? 3 * kRows * 2 : 0);
  static_assert(kSmem <= 227 * 1024, "tiles fit one CTA's shared memory");
};
constexpr uint32_t kBarBytes = 336;
struct Shown {  // a piece as the walking warp shows it to all
  Piece p;
  Tile t;
  int none;  // there are no more pieces
  int last;  // none behind this one
};
static_assert(sizeof(Shown) == 64, "the ring of pieces");
// Four values that pass by (L1 keeps what a thread has no register for).
__device__ __forceinline__ void load4(const float* p, float* v) {
  asm volatile("ld.global.L1::no_allocate.v4.f32 {%0,%1,%2,%3}, [%4];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3])
               : "l"(p));
}
__device__ __align__(16) const float no_key[HD] = {};
__device__ __forceinline__ void mbar_arrive_n(uint32_t bar, int count) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
template <int FROM, int TO> __device__ __forceinline__ void set_regs() {
  if (TO == FROM) return;
  if (TO > FROM) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(TO));
  else asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(TO));
}

// Two packed values as floats, and the bits from which on a value is not finite.
template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t b);
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t b) {
  return __half22float2(*reinterpret_cast<const __half2*>(&b));
}
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t b) {
  return make_float2(__uint_as_float(b << 16), __uint_as_float(b & 0xffff0000u));
}
template <typename T> constexpr uint32_t kInfinity = Planes<T>::format ? 0x7f80u : 0x7c00u;

__device__ __forceinline__ uint32_t tmem_ld1(uint32_t a) {
  uint32_t r;
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(r) : "r"(a));
  asm volatile("tcgen05.wait::ld.sync.aligned;" : "+r"(r) : : "memory");
  return r;
}
// O += P V of one tile by the threads themselves: a key that a row does not see has weight
// zero and is left out, whatever its value is, while in a matrix product zero times an
// infinity or a NaN would be NaN.  `p` is the row's weights in TMEM as the product would read
// them, `v` the tile's values (NV planes); o 128 columns, times f.
template <typename T, int NV>
__device__ __noinline__ void add_tile(f32x2* o, uint32_t p, uint32_t third, uint32_t v, float mul) {
#pragma unroll 1  // (seldom run: small rather than fast)
  for (int h = 0; h < 64; ++h) {  // two keys
    float2 w = make_float2(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < Planes<T>::n; ++k) {
      const float2 y = unpack2<T>(tmem_ld1(k == 2 ? third + h : p + 16 * (h >> 3) + 8 * k + (h & 7)));
      w.x += y.x;
      w.y += y.y;
    }
#pragma unroll 1
    for (int e = 0; e < 2; ++e) {
      const float f = (e ? w.y : w.x) * mul;
      const int key = 2 * h + e;
      if (f != 0.f)
#pragma unroll 4
        for (int i = 0; i < 16 * NV; ++i) {
          const uint4 q = lds128(v + (i >> 3) * kHalf + key * 128 + (((i & 7) ^ (key & 7)) << 4));  // (two halves a plane)
          const uint32_t r[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
          for (int d = 0; d < 4; ++d) {
            const float2 z = unpack2<T>(r[d]);
            o[4 * (i & 15) + d] = fma2(pair(z.x, z.y), pair(f, f), o[4 * (i & 15) + d]);
          }
        }
    }
  }
}

// As mbar_try_wait, asleep for up to about `ns` (warps that look again and again take issue slots).
__device__ __forceinline__ bool mbar_try_wait_for(uint32_t bar, uint32_t parity, uint32_t ns) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(ok)
      : "r"(bar), "r"(parity), "r"(ns)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ float largest(const float (&s)[32]) {
  float a = -INFINITY, b = -INFINITY;
#pragma unroll
  for (int k = 0; k < 32; k += 4) {
    a = fmaxf(a, fmaxf(s[k], s[k + 1]));
    b = fmaxf(b, fmaxf(s[k + 2], s[k + 3]));
  }
  return fmaxf(a, b);
}
// The weights of the first `chunks` times 32 keys of a tile, in all planes, times a power of two.
template <typename T> __device__ __noinline__ void scale_weights(uint32_t p, uint32_t third, int chunks, float f) {
  auto times = [&](float (&v)[8], uint32_t* b) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float2 w = unpack2<T>(__float_as_uint(v[k]));
      const auto r = cvt2(w.x * f, w.y * f, (T*)nullptr);
      b[k] = *reinterpret_cast<const uint32_t*>(&r);
    }
  };
  for (int h = 0; h < 2 * chunks; ++h) {
    float v[8];
    uint32_t b[8];
    for (int k = 0; k < 16; k += 8) {
      tmem_ld8(p + 16 * h + k, v);
      times(v, b);
      tmem_st8(p + 16 * h + k, b);
    }
    if (Planes<T>::n == 3) {
      tmem_ld8(third + 8 * h, v);
      times(v, b);
      tmem_st8(third + 8 * h, b);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(Layout<T>::kThreads, 1)
    chunks_tc_kernel(const __grid_constant__ ChunkArgs a, const __grid_constant__ CUtensorMap k_map,
                     const __grid_constant__ CUtensorMap v_map) {
  using L = Layout<T>;
  using TQ = typename L::Q;
  using TP = typename L::P;
  constexpr int NQ = Planes<TQ>::n, NP = Planes<TP>::n, G = L::G, kRing = L::kRing;
  constexpr bool kSplit = L::kSplit, kScaled = L::kScaled;
  constexpr uint32_t kIdQK = idesc(Planes<TQ>::format, kRows, kKeys, false);
  constexpr uint32_t kIdPV = idesc(Planes<TP>::format, kRows, 128, true);
  extern __shared__ __align__(1024) uint8_t mem[];
  const uint32_t sq = smem_addr(mem);
  const uint32_t sk = sq + L::kQBytes, sv = sk + L::kKBytes, bars = sv + L::kVBytes;
  uint8_t* small = mem + (bars - sq);
  // a tile's stage in shared memory, and how often it was used before
  auto stage = [](int e) { return kSplit ? 0 : e & 1; };
  auto used = [](int e) { return kSplit ? e : e >> 1; };
  // per piece
  const uint32_t qfull = bars, lready = bars + 8, pdone = bars + 16;
  auto shown = [&](int k) { return bars + 24 + 8 * (k & (kRing - 1)); };  // piece k is in its place of the ring
  auto seen = [&](int k) { return bars + 56 + 8 * (k & (kRing - 1)); };   // it has been used
  // per tile, by its stage in shared memory
  auto kfull = [&](int s) { return bars + 88 + 8 * s; };
  auto vfull = [&](int s) { return bars + 104 + 8 * s; };
  // per tile, by its place in TMEM (tile % G)
  auto sfull = [&](int g) { return bars + 120 + 8 * g; };   // S is there, K has been read
  auto mready = [&](int g) { return bars + 144 + 8 * g; };  // the rows' references of the weights are there
  auto pready = [&](int g) { return bars + 168 + 8 * g; };  // the weights are there, V is fit for them, O is free
  auto vempty = [&](int g) { return bars + 192 + 8 * g; };  // O is there, weights and V have been read
  auto ofree = [&](int g) { return bars + 216 + 8 * g; };   // O has been read
  const uint32_t together = bars + 256;  // the warps that add up O
  volatile uint8_t* say = reinterpret_cast<volatile uint8_t*>(small + 264);  // ... what each says, twice
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(small + 240);
  volatile int* gave_up = reinterpret_cast<volatile int*>(small + 244);
  volatile unsigned* bad_boxes = reinterpret_cast<volatile unsigned*>(small + 272);  // of tiles i, by i & 7
  volatile unsigned* bad_keys = bad_boxes;                                             // fp32: [i % 3][32 keys]
  volatile uint8_t* odd_values = reinterpret_cast<volatile uint8_t*>(small + 320);   // fp32: of 16 keys
  volatile int* scored = reinterpret_cast<volatile int*>(small + 252);                // fp32: tiles whose scores are under way
  Shown* ring = reinterpret_cast<Shown*>(small + kBarBytes);
  float* reference = reinterpret_cast<float*>(ring + kRing);  // [place][row]: weights are 2^(score - reference + kUp)
  float* row_sum = kSplit ? reference : reference + G * kRows;  // [group][row], at a piece's end
  // powers of two as bf16: of the rows of Q [piece % (G + 1)][row], of split keys [i % 3][key]
  __nv_bfloat16* row_scale_of = reinterpret_cast<__nv_bfloat16*>(row_sum + G * kRows);
  __nv_bfloat16* key_scale_of = row_scale_of + (G + 1) * kRows;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    mbar_init(qfull, 4 * G);
    mbar_init(lready, 4 * G);
    mbar_init(pdone, 4);
    mbar_init(together, 4);
    for (int s = 0; s < 2; ++s) {
      mbar_init(kfull(s), kSplit ? 8 : 1);
      mbar_init(vfull(s), kSplit ? 8 : 1);
    }
    for (int g = 0; g < G; ++g) {
      mbar_init(sfull(g), 1);
      mbar_init(mready(g), 4);
      mbar_init(pready(g), 8);
      mbar_init(vempty(g), 1);
      mbar_init(ofree(g), 4);
    }
    for (int k = 0; k < kRing; ++k) {
      mbar_init(shown(k), 1);
      mbar_init(seen(k), L::kThreads / 32 - 1);  // all but the one that finds them
    }
    fence_mbar_init();
    *gave_up = 0;
    *scored = 0;
  }
  if (warp == L::kScoreWarp) {
    tmem_alloc(smem_addr(tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();
  pdl_launch_dependents();
  const int ps = 1 << a.ps_log2, prefix_tiles = tiles_of(a.prefix);

  // A bounded wait; after any time-out every wait that would go on gives up too.
  auto wait = [&](uint32_t bar, int parity) {
    if (mbar_try_wait(bar, (uint32_t)parity & 1u)) return;
    const uint64_t t0 = globaltimer_ns();
    while (!*gave_up && !mbar_try_wait_for(bar, (uint32_t)parity & 1u, 20000)) {
      if (globaltimer_ns() - t0 > 2000000000ull) {
        *gave_up = 1;
        atomicOr(a.status, (int)kStatusWaitTimeout);
        return;
      }
    }
  };
  // One arrival a warp, behind all of its lanes' work.
  auto arrive = [&](uint32_t bar) {
    __syncwarp();
    if (lane == 0) mbar_arrive(bar);
  };
  int i = 0;      // key tiles so far; tile i takes stage i & 1
  int piece = 0;  // pieces so far
  // The next piece, or none.  A warp that is done with it says so (done).
  auto next = [&]() -> const Shown* {
    if (*gave_up) return nullptr;
    wait(shown(piece), piece / kRing);
    const Shown* s = ring + (piece & (kRing - 1));
    return *gave_up || s->none ? nullptr : s;
  };
  auto done = [&]() { arrive(seen(piece++)); };

  if (warp < L::kSumWarp) {
    // ---------------- weights: a thread a query row, a group every G-th tile ----------------
    set_regs<L::kRegs, L::kSoftRegs>();
    const int g = warp >> 2, row = tid & 127;
    const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
    const uint32_t ts = tmem + lanes + 128 * g, tx = tmem + lanes + L::kX + 64 * g;
    int pieces = 0, e = g, turn = 0;  // this group's next tile of all, how many it has had
    while (const Shown* sh = next()) {
      const Piece& pc = sh->p;
      const Tile& t = sh->t;
      const int n = pc.j1 - pc.j0;
      const Query me = query_of(a, pc, t, row);
      if (n == 0) {  // rows without a key
        if (me.on && g < 2) {
          float* out = a.out + (long long)(pc.r.first + me.token) * a.ldo + (size_t)me.head * HD + 64 * g;
          for (int d = 0; d < 64; d += 4) *reinterpret_cast<float4*>(out + d) = make_float4(0.f, 0.f, 0.f, 0.f);
        }
        done();
        continue;
      }
      // The planes of Q, by the group that has the piece's first tile: it is the first to be done with the
      // last piece, so this runs beside that one's last tiles.  The first piece's, for which all wait, by all.
      // (A row's scale has been read once G further tiles have their scores: the places of G + 1 pieces are
      // enough.)
      if (g == i % G || i == 0) {
        // a warp takes 32 rows, half of it one row at a time, a lane 8 of its values; lane r knows where row r is
        const Query mine = query_of(a, pc, t, row);
        const long long at = mine.on ? (long long)(pc.r.first + mine.token) * a.ldq + (long long)mine.head * HD : -1ll;
        const int h = lane >> 4, c = lane & 15;  // half of the warp, 16-byte chunk of the row's planes
        constexpr int N = G == 3 ? 2 : 4;          // pairs of rows on their way (twice as many: drafts 4 us longer, no register for them)
        float4 v[N][2];
        auto load = [&](int e, int pair) {
          const long long from = __shfl_sync(0xffffffffu, at, 2 * pair + h);
          v[e][0] = v[e][1] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (from >= 0) {
            v[e][0] = *reinterpret_cast<const float4*>(a.q + from + 8 * c);
            v[e][1] = *reinterpret_cast<const float4*>(a.q + from + 8 * c + 4);
          }
        };
        const int from = i == 0 ? N * g : 0, step = i == 0 ? N * G : N;
#pragma unroll
        for (int e = 0; e < N; ++e) load(e, from + e);
        if (i > 0) wait(sfull((i + G - 1) % G), (i - 1) / G);  // the last piece's products of Q are done
#pragma unroll 1
        for (int e0 = from; e0 < 16; e0 += step) {
#pragma unroll
          for (int e = 0; e < N; ++e) {
            const int qr = 32 * (warp & 3) + 2 * (e0 + e) + h;
            float x[8] = {v[e][0].x, v[e][0].y, v[e][0].z, v[e][0].w, v[e][1].x, v[e][1].y, v[e][1].z, v[e][1].w};
            float mul = a.qscale;
            if (kScaled) {
              float most = fmaxf(fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3]))),
                                 fmaxf(fmaxf(fabsf(x[4]), fabsf(x[5])), fmaxf(fabsf(x[6]), fabsf(x[7])))) * mul;
#pragma unroll
              for (int off = 8; off > 0; off >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, off));
              float back;
              mul *= row_scale<TQ>(most, back);
              if (c == 0) row_scale_of[pieces % (G + 1) * kRows + qr] = __float2bfloat16(back);
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) x[k] *= mul;
            if (e0 + step < 16) load(e, e0 + step + e);
            const uint32_t to = sq + (c >> 3) * kHalf + qr * 128 + (((c & 7) ^ (qr & 7)) << 4);
#pragma unroll
            for (int p = 0; p < NQ; ++p) {
              uint32_t b[4];
#pragma unroll
              for (int k = 0; k < 4; ++k) b[k] = weight_plane<TQ>(x[2 * k], x[2 * k + 1], p < NQ - 1);
              sts128(to + p * kTileBytes, b[0], b[1], b[2], b[3]);
            }
          }
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive_n(qfull, i == 0 ? 1 : G);
      }
      float qmul = 1.f;
      // own keys that the row sees (all, where there is no row)
      const int reach = me.on ? max(pc.r.base + me.token + 1, 0) : 0x7fffffff;
      const bool idle = !__any_sync(0xffffffffu, me.on);
      float m = -INFINITY, l = 0.f;
      // the place of this group's references is free: that of its tile before has been read
      bool first = true;
      auto free_reference = [&]() {
        if (kSplit && first && pieces > 0) wait(pdone, pieces - 1);  // (there the sums stand in their place)
        first = false;
        if (turn > 0) wait(ofree(g), turn - 1);
      };
      for (; e < i + n; e += G, ++turn) {
        const int j = pc.j0 + e - i;
        const bool pre = j < prefix_tiles;
        const int t0 = (pre ? j : j - prefix_tiles) * kKeys;
        const int valid = min(kKeys, (pre ? a.prefix : t.most) - t0);  // keys of the tile that some row sees
        const int mine = pre ? valid : min(reach - t0, kKeys);          // that this row sees, the first ones
        wait(sfull(g), turn);
        if (kScaled) qmul = __bfloat162float(row_scale_of[pieces % (G + 1) * kRows + row]);
        // split keys have scales too: a small one of q comes first, a large one last, so what lies between
        // leaves fp32's range only where the score does
        const float qfirst = kSplit ? fminf(qmul, 1.f) : 1.f;
        if (kSplit) qmul = fmaxf(qmul, 1.f);
        unsigned bad;  // boxes (split keys: whether some keys) lie outside the pool
        if (kSplit) bad = bad_keys[e % 3 * 4] | bad_keys[e % 3 * 4 + 1] | bad_keys[e % 3 * 4 + 2] | bad_keys[e % 3 * 4 + 3];
        else bad = bad_boxes[e & 7];
        const bool masked = bad || __any_sync(0xffffffffu, mine < kKeys);
        tc_fence_after();
        auto mask = [&](float* s, int first) {  // 32 keys
          const int n = mine - first;
          unsigned hidden = n >= 32 ? 0u : n > 0 ? ~0u << n : ~0u;
          if (kSplit && bad) hidden |= bad_keys[e % 3 * 4 + first / 32];
          if (!kSplit && bad) {
            if ((bad >> (first >> a.box_log2)) & 1) hidden |= 0xffffu;
            if ((bad >> ((first + 16) >> a.box_log2)) & 1) hidden |= 0xffff0000u;
          }
#pragma unroll
          for (int k = 0; k < 32; ++k)
            if ((hidden >> k) & 1) s[k] = -INFINITY;
        };
        if (!idle) {
          float shift = m == -INFINITY ? 0.f : kUp - m;
          const f32x2 mul2 = pair(qmul, qmul);
          f32x2 l2 = 0;
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            float s[32];
            tmem_ld32(ts + 32 * c, s);
            tmem_wait_ld32(s);
            if (kSplit) {  // the keys' scales
              const uint32_t at = smem_addr(key_scale_of + e % 3 * kRows + 32 * c);
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const uint4 x = lds128(at + 16 * k);
                const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                  const float2 f = unpack2<__nv_bfloat16>(w[d]);
                  s[8 * k + 2 * d] *= f.x * qfirst;
                  s[8 * k + 2 * d + 1] *= f.y * qfirst;
                }
              }
            }
            if (masked) mask(s, 32 * c);
            const float mx = largest(s) * qmul;
            if (__any_sync(0xffffffffu, mx > m + kLazy)) {
              // Seldom: a row's first scores, whose largest is its reference, or one far above the reference, which
              // then moves up by whole powers of two; the weights that the tile has already move down.
              float f = 1.f;
              if (m == -INFINITY) {
                m = mx;
              } else if (mx > m + kLazy) {
                const float old = m;
                m += ceilf(mx - m);
                if (fabsf(m - mx) > 1.f) m = mx;  // scores past 2^24, where the sum is rounded: nothing else counts
                f = ex2(old - m);
                l *= f;
                l2 = fma2(l2, pair(f, f), 0);
              }
              shift = m == -INFINITY ? 0.f : kUp - m;
              if (c > 0 && __any_sync(0xffffffffu, f != 1.f)) {
                tmem_wait_st();
                scale_weights<TP>(ts, tx, c, f);
              }
            }
            const f32x2 shift2 = pair(shift, shift);
#pragma unroll
            for (int h = 0; h < 2; ++h) {  // 16 keys: one step of the product
              float* p = s + 16 * h;
#pragma unroll
              for (int k = 0; k < 16; k += 2) {
                float x, y;
                unpair(fma2(pair(p[k], p[k + 1]), mul2, shift2), x, y);
                p[k] = ex2(x);
                p[k + 1] = ex2(y);
                l2 = add2(l2, pair(p[k], p[k + 1]));
              }
              uint32_t b[16];
#pragma unroll
              for (int k = 0; k < 16; ++k) b[k] = weight_plane<TP>(p[2 * (k & 7)], p[2 * (k & 7) + 1], k < 8 || NP == 3);
              tmem_st16(ts + 32 * c + 16 * h, b);
              if (NP == 3) {
#pragma unroll
                for (int k = 0; k < 8; ++k) b[k] = weight_plane<TP>(p[2 * k], p[2 * k + 1], false);
                tmem_st8(tx + 16 * c + 8 * h, b);
              }
            }
          }
          float l0, l1;
          unpair(l2, l0, l1);
          l += l0 + l1;
        }
        tmem_wait_st();
        tc_fence_before();
        arrive(pready(g));
        free_reference();
        reference[g * kRows + row] = m;
        arrive(mready(g));
      }
      i += n;
      if (kSplit) free_reference();
      else if (pieces > 0) wait(pdone, pieces - 1);  // the last piece's sums have been read
      ++pieces;
      row_sum[g * kRows + row] = l;
      arrive(lready);
      done();
    }
  } else if (warp < L::kScoreWarp) {
    // ---------------- O: a tile's sum, times its weights' reference, to the row's ----------------
    set_regs<L::kRegs, L::kSumRegs>();
    const int row = tid & 127;
    const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
    int meetings = 0;
    // True in all four warps when it holds for a lane of one of them; behind all of their work before.  (A
    // wait like the others: a named barrier has no end if a warp gives up.)
    auto any_of_us = [&](bool x) {
      const int at = (meetings & 1) * 4;
      x = __any_sync(0xffffffffu, x);
      if (lane == 0) say[at + (warp & 3)] = x;
      arrive(together);
      wait(together, meetings++);
      return *reinterpret_cast<volatile uint32_t*>(small + 264 + at) != 0;
    };
    int pieces = 0, flags = 0, g = 0, turn = 0;  // the next tile's place, and how often it has been used
    int4 begun = make_int4(0, 0, 0, 0);
    while (const Shown* sh = next()) {
      const Piece& pc = sh->p;
      const Tile& t = sh->t;
      const int n = pc.j1 - pc.j0;
      if (n == 0) {
        done();
        continue;
      }
      const Query me = query_of(a, pc, t, row);
      const bool idle = !__any_sync(0xffffffffu, me.on);
      f32x2 o[64];
      float M = -INFINITY, of_group[G];
#pragma unroll
      for (int k = 0; k < G; ++k) of_group[k] = -INFINITY;
#pragma unroll
      for (int d = 0; d < 64; ++d) o[d] = 0;
      const int least = max(pc.r.base + t.token0 + 1, 0);  // own keys that every row sees
      // Tile e's values: those behind its keys become zeros (a page goes on past them and may hold
      // anything, also NaN).  True: some row does not see some key, and not all values are finite.
      auto look_at = [&](int e) {
        const int j = pc.j0 + e - i;
        const bool pre = j < prefix_tiles;
        const int t0 = (pre ? j : j - prefix_tiles) * kKeys, valid = min(kKeys, (pre ? a.prefix : t.most) - t0);
        const int over = -valid & ((1 << a.box_log2) - 1);
        const bool hidden = !pre && t0 + valid > least;
        if (!over && !hidden) return false;
        if (kSplit) {  // (those who made the planes know; the tile before has its O, so this is the barrier's phase)
          if (!hidden) return false;
          wait(vfull(0), e);
          return *reinterpret_cast<volatile unsigned long long*>(small + 320) != 0;
        }
        const uint32_t vt = sv + stage(e) * kTileBytes;
        wait(vfull(stage(e)), used(e));
        for (int k = row; k < over * 16; k += 128)
          sts128(vt + ((k >> 3) & 1) * kHalf + (valid + (k >> 4)) * 128 + (k & 7) * 16, 0, 0, 0, 0);
        if (over) fence_proxy_async();
        if (!hidden) return false;
        uint32_t most = 0;
#pragma unroll 4
        for (int k = row; k < (int)kTileBytes / 16; k += 128) {
          if (((k >> 3) & 127) >= valid) continue;
          const uint4 x = lds128(vt + k * 16);
          most = __vmaxu2(__vmaxu2(most, x.x & 0x7fff7fffu), __vmaxu2(x.y & 0x7fff7fffu, x.z & 0x7fff7fffu));
          most = __vmaxu2(most, x.w & 0x7fff7fffu);
        }
        return any_of_us((most >> 16) >= kInfinity<TP> || (most & 0xffffu) >= kInfinity<TP>);
      };
      bool odd = look_at(i);
      if (!odd) arrive(pready(g));
      for (int e = i; e < i + n; ++e) {
        wait(mready(g), turn);
        const float m = reference[g * kRows + row];
#pragma unroll
        for (int k = 0; k < G; ++k) of_group[k] = g == k ? m : of_group[k];
        if (m > M + kLazy) {  // seldom: M then is the largest reference so far
          const float f = M == -INFINITY ? 0.f : ex2(M - m);
          M = m;
#pragma unroll
          for (int d = 0; d < 64; ++d) o[d] = fma2(o[d], pair(f, f), 0);
        }
        const float f = m == -INFINITY ? 0.f : ex2(m - M);
        if (odd) {
          const uint32_t vt = sv + stage(e) * kTileBytes;
          tc_fence_after();
          if (!idle) {
            f32x2 sum[64];  // (o itself stays in registers)
#pragma unroll
            for (int d = 0; d < 64; ++d) sum[d] = o[d];
            add_tile<TP, L::kValuePlanes>(sum, tmem + lanes + 128 * g, tmem + lanes + L::kX + 64 * g, vt, f);
#pragma unroll
            for (int d = 0; d < 64; ++d) o[d] = sum[d];
          }
          any_of_us(false);  // then the product adds nothing
          for (int k = row; k < (int)(L::kValuePlanes * kTileBytes) / 16; k += 128) sts128(vt + k * 16, 0, 0, 0, 0);
          fence_proxy_async();
          tc_fence_before();
          arrive(pready(g));
        }
        const bool more = e + 1 < i + n;
        // fp32: the next tile is looked at when this one's O is there, and its product waits for that
        const bool later = kSplit && more && pc.j0 + e + 1 - i >= prefix_tiles &&
                           min((pc.j0 + e + 2 - i - prefix_tiles) * kKeys, t.most) > least;
        if (!kSplit) odd = more && look_at(e + 1);
        else odd = false;
        wait(vempty(g), turn);
        auto taken = [&]() {  // O is free
          tc_fence_before();
          arrive(ofree(g));
          if (more && !odd && !later && lane == 0) mbar_arrive(pready(g + 1 == G ? 0 : g + 1));
        };
        if (!idle) {
          tc_fence_after();
          const f32x2 f2 = pair(f, f);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            float s[32];
            tmem_ld32(tmem + lanes + L::kO + 32 * c, s);
            tmem_wait_ld32(s);
            if (c == 3) taken();
#pragma unroll
            for (int d = 0; d < 16; ++d) o[16 * c + d] = fma2(pair(s[2 * d], s[2 * d + 1]), f2, o[16 * c + d]);
          }
        } else {
          taken();
        }
        if (later) {
          odd = look_at(e + 1);
          if (!odd) arrive(pready(g + 1 == G ? 0 : g + 1));
        }
        if (++g == G) g = 0, ++turn;
      }
      i += n;
      wait(lready, pieces++);
      float l = 0.f;
#pragma unroll
      for (int k = 0; k < G; ++k) {
        const float x = row_sum[k * kRows + row];
        if (x != 0.f) l += of_group[k] == -INFINITY ? x : x * ex2(of_group[k] - M);  // (a NaN score has no reference)
      }
      arrive(pdone);
      const bool whole = pc.j0 == 0 && pc.j1 == pc.T;
      float mul = 1.f, *out;
      if (whole) {
        mul = l == 0.f ? 0.f : 1.f / l;  // no key: zeros
        out = a.out + (long long)(pc.r.first + me.token) * a.ldo + (size_t)me.head * HD;
      } else {
        const int slot = 2 * (int)blockIdx.x + (pc.j0 == 0 ? 1 : 0);
        out = a.parts + ((size_t)slot * kRows + row) * kPart;
        if (me.on) *reinterpret_cast<float2*>(out) = make_float2(l != l ? l : M, l);  // a NaN score counts however it compares
        out += 4;
        if (pc.j0 == 0) {
          flags |= kBegins;
          begun = make_int4(0, pc.request, pc.sub, pc.tile);
        } else {
          flags |= pc.j1 == pc.T ? kGoesOn | kEnds : kGoesOn;
        }
      }
      const f32x2 mul2 = pair(mul, mul);
#pragma unroll
      for (int d = 0; d < 64; ++d) o[d] = fma2(o[d], mul2, 0);
      if (sh->last) {
        // nothing runs beside: in whole rows by way of the place of Q and the keys (a thread's own row touches
        // 32 lines a warp's store: 6000 cycles; between pieces they run beside the next one's first tile)
        const uint32_t mine = sq + row * 512;
#pragma unroll
        for (int d = 0; d < 64; d += 2) {
          float4 v;
          unpair(o[d], v.x, v.y);
          unpair(o[d + 1], v.z, v.w);
          sts128(mine + (((d >> 1) ^ (row & 31)) << 4), __float_as_uint(v.x), __float_as_uint(v.y), __float_as_uint(v.z),
                 __float_as_uint(v.w));
        }
        __syncwarp();
        const unsigned on = __ballot_sync(0xffffffffu, me.on);
#pragma unroll 4
        for (int r = 0; r < 32; ++r) {
          float* to = reinterpret_cast<float*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(out), r));
          const uint4 x = lds128(sq + (32 * (warp & 3) + r) * 512 + ((lane ^ r) << 4));
          if ((on >> r) & 1) *reinterpret_cast<uint4*>(to + 4 * lane) = x;
        }
      } else if (me.on) {
#pragma unroll
        for (int d = 0; d < 64; d += 2) {
          float4 v;
          unpair(o[d], v.x, v.y);
          unpair(o[d + 1], v.z, v.w);
          *reinterpret_cast<float4*>(out + 2 * d) = v;
        }
      }
      done();
    }
    if (row == 0) a.records[blockIdx.x] = make_int4(flags, begun.y, begun.z, begun.w);
  } else if (warp < L::kMakeWarp) {
    set_regs<L::kRegs, L::kIssueRegs>();
    if (warp == L::kKeyWarp || warp == L::kKeyWarp + 1) {
      // ---------------- keys, or values, a box of a page at a time ----------------
      // lane g has the page of box g, read a tile ahead (of one piece)
      const bool values = warp != L::kKeyWarp;
      const CUtensorMap* map = values ? &v_map : &k_map;
      const int boxes = kKeys >> a.box_log2;
      const uint32_t box_bytes = 128u << a.box_log2;
      Walk walk(a, values ? Place{0, 0, 0, 0, 0} : find_run(a, (int)blockIdx.x, (int)gridDim.x));
      // the next piece: found by the keys' warp, which shows it to all and asks for its rows of q
      auto find = [&]() -> const Shown* {
        if (values) return next();
        Shown* sh = ring + (piece & (kRing - 1));
        Piece pc;
        const bool more = walk.step(pc) && !*gave_up;
        if (piece >= kRing) wait(seen(piece), piece / kRing - 1);
        Tile t{};
        if (more) t = tile_of(a, pc);
        if (lane == 0) {
          sh->p = pc;
          sh->t = t;
          sh->none = !more;
          sh->last = walk.p.left <= 0;
        }
        arrive(shown(piece++));
        if (!more) return nullptr;
        for (int r = lane; r < 4 * kRows; r += 32) {  // 128 bytes each
          const Query w = query_of(a, pc, t, r >> 2);
          if (w.on)
            asm volatile("prefetch.global.L2 [%0];" ::"l"(a.q + (long long)(pc.r.first + w.token) * a.ldq +
                                                          (size_t)w.head * HD + 32 * (r & 3)));
        }
        return sh;
      };
      if (kSplit) {
        if (values) {  // asks for the keys and values of the tiles ahead
          while (const Shown* sh = next()) {
            const Piece& pc = sh->p;
            const Tile& t = sh->t;
            const int* own = a.table + (long long)pc.request * a.table_stride;
            for (int j = pc.j0; j < pc.j1; ++j, ++i) {
              const bool pre = j < prefix_tiles;
              // (three tiles ahead at most; nothing depends on it, so it does not wait for good)
              for (int k = 0; k < 1 << 16 && *scored + 3 < i && !*gave_up; ++k) __nanosleep(200);
              for (int r = lane; r < kKeys; r += 32) {
                const int k = (pre ? j : j - prefix_tiles) * kKeys + r;
                const int page = k < (pre ? a.prefix : t.most) ? (pre ? a.prefix_pages : own)[k >> a.ps_log2] : -1;
                if (page < 0 || page >= a.n_pages) continue;
                const size_t at = (((size_t)page * a.nkv + t.kvh) * ps + (k & (ps - 1))) * HD;
                for (int x = 0; x < HD; x += 32) {
                  asm volatile("prefetch.global.L2 [%0];" ::"l"(a.k32 + at + x));
                  asm volatile("prefetch.global.L2 [%0];" ::"l"(a.v32 + at + x));
                }
              }
            }
            done();
          }
        } else {
          while (find()) {
          }
        }
      }
      while (const Shown* sh = kSplit ? nullptr : find()) {
        const Piece& pc = sh->p;
        const Tile& t = sh->t;
        const int* own = a.table + (long long)pc.request * a.table_stride;
        const int j1 = pc.j1, most = t.most, head = t.kvh << a.ps_log2;
        auto page_of = [&](int j) {
          const bool pre = j < prefix_tiles;
          const int k = (pre ? j : j - prefix_tiles) * kKeys + (lane << a.box_log2);
          return j < j1 && lane < boxes && k < (pre ? a.prefix : most) ? (pre ? a.prefix_pages : own)[k >> a.ps_log2] : -2;
        };
        int ahead = page_of(pc.j0);
        for (int j = pc.j0; j < j1; ++j, ++i) {
          const int t0 = (j < prefix_tiles ? j : j - prefix_tiles) * kKeys, s = i & 1;
          int page = ahead;
          ahead = page_of(j + 1);
          const bool ok = page >= 0 && page < a.n_pages;
          const unsigned bad = __ballot_sync(0xffffffffu, !ok && page != -2);  // boxes of keys that lie outside the pool
          if (!ok) page = a.n_pages;  // out of range: zeros
          const uint32_t bar = values ? vfull(s) : kfull(s), dst = (values ? sv : sk) + s * kTileBytes;
          // the tile before in this stage: S ready, its keys have been read; O, its values
          if (i >= 2) wait(values ? vempty((i - 2) % G) : sfull((i - 2) % G), (i - 2) / G);
          if (*gave_up) break;
          if (lane == 0) {
            if (!values) {
              bad_boxes[i & 7] = bad;  // (that of tile i - 8 has been read: S of tile i - 2 is there)
              if (bad) atomicOr(a.status, (int)kStatusBadPage);
            }
            mbar_expect_tx(bar, kTileBytes);
          }
#pragma unroll 4
          for (int g = 0; g < boxes; ++g) {
            const int p = __shfl_sync(0xffffffffu, page, g), y = head + ((t0 + (g << a.box_log2)) & (ps - 1));
            if (lane == 0) {
              tma_box(dst + g * box_bytes, map, 0, y, p, bar);
              tma_box(dst + kHalf + g * box_bytes, map, 64, y, p, bar);
            }
          }
        }
        if (values) done();
      }
      if (!kSplit && *gave_up && lane == 0)  // what may be in flight lands before the memory is given back
        for (int s = 0; s < 2; ++s)
          for (int e = 0; e < 2; ++e) (void)mbar_wait_bounded(values ? vfull(s) : kfull(s), (uint32_t)e);
    } else {
      // ---------------- the two products, a warp each ----------------
      const bool scores = warp == L::kScoreWarp;
      const uint64_t q_desc = desc_sw128(sq), k_desc = desc_sw128(sk), v_desc = desc_v(sv);  // (addresses in 16 bytes)
      int pieces = 0, g = 0, turn = 0;  // the next tile's place in TMEM, how often it has been used
      while (const Shown* sh = next()) {
        const int n = sh->p.j1 - sh->p.j0;
        done();
        if (n == 0) continue;
        if (scores) wait(qfull, pieces++);
        for (int e = i; e < i + n; ++e) {
          const int s = stage(e);
          if (scores) {
            wait(kfull(s), used(e));
            if (turn > 0) wait(vempty(g), turn - 1);  // the weights that stood there have been read
            tc_fence_after();
            if (elect_one()) {
              // small planes first: the chain of truncated additions starts near zero
              constexpr int kProducts = kSplit ? 3 : NQ;
              constexpr int kOfQ[3] = {kSplit ? 1 : NQ - 1, kSplit ? 0 : NQ - 2, 0}, kOfK[3] = {0, kSplit ? 1 : 0, 0};
#pragma unroll
              for (int p = 0; p < kProducts; ++p)
#pragma unroll
                for (int ks = 0; ks < 8; ++ks) {
                  const uint32_t off = ((uint32_t)(ks >> 2) * kHalf + (uint32_t)(ks & 3) * 32) >> 4;
                  mma_ss(tmem + 128 * g, q_desc + (off + kOfQ[p] * (kTileBytes >> 4)),
                         k_desc + (off + (kOfK[p] + s) * (kTileBytes >> 4)), kIdQK, p != 0 || ks != 0 ? 1u : 0u);
                }
              tc_commit(sfull(g));
              if (kSplit) *scored = e;
            }
          } else {
            wait(vfull(s), used(e));
            wait(pready(g), turn);
            tc_fence_after();
            if (elect_one()) {
              constexpr int kProducts = kSplit ? 6 : NP;
              constexpr int kOfP[6] = {kSplit ? 2 : NP - 1, kSplit ? 0 : NP - 2, kSplit ? 1 : 0, 1, 0, 0};
              constexpr int kOfV[6] = {0, kSplit ? 2 : 0, kSplit ? 1 : 0, 0, 1, 0};
#pragma unroll
              for (int p = 0; p < kProducts; ++p)
#pragma unroll
                for (int ks = 0; ks < 8; ++ks) {
                  const uint32_t at = kOfP[p] == 2 ? L::kX + 64 * g + 8 * ks : 128 * g + 16 * ks + 8 * kOfP[p];
                  mma_ts(tmem + L::kO, tmem + at, v_desc + ((kOfV[p] + s) * (kTileBytes >> 4) + ks * (2048 >> 4)), kIdPV,
                         p != 0 || ks != 0 ? 1u : 0u);
                }
              tc_commit(vempty(g));
            }
          }
          __syncwarp();
          if (++g == G) g = 0, ++turn;
        }
        i += n;
      }
      if (*gave_up && lane == 0)  // products in flight end too
        for (int k = 0; k < G; ++k)
          for (int e = 0; e < 2; ++e) (void)mbar_wait_bounded(scores ? sfull(k) : vempty(k), (uint32_t)e);
    }
  } else if (kSplit) {
    // ---------------- the planes of fp32 keys and values: a warp 16 of a tile's ----------------
    // First the keys, whose scores take a while to become weights, then the values: all eight warps at both,
    // since a tile's keys wait for the last one's scores, and its values for the last one's O.  (Registers are
    // what there is least of: a value that a pass keeps outside of them comes back from L2, shared memory
    // leaves little of L1.)
    set_regs<L::kRegs, L::kMakeRegs>();
    const int w = warp - L::kMakeWarp;
    while (const Shown* sh = next()) {
      auto page_of = [&](int j) {  // of this lane's key of tile j
        const bool pre = j < prefix_tiles;
        const int k = (pre ? j : j - prefix_tiles) * kKeys + 16 * w + (lane & 15);
        if (j >= sh->p.j1 || k >= (pre ? a.prefix : sh->t.most)) return -2;
        return (pre ? a.prefix_pages : a.table + (long long)sh->p.request * a.table_stride)[k >> a.ps_log2];
      };
      int ahead = page_of(sh->p.j0);
      for (int j = sh->p.j0; j < sh->p.j1; ++j, ++i) {
        const bool ok = ahead >= 0 && ahead < a.n_pages;
        const unsigned bad = __ballot_sync(0xffffffffu, !ok && ahead != -2);
        // the key's row of the pool (2^32 of them would be 2 TB)
        const unsigned at = ok ? ((((unsigned)ahead * a.nkv + sh->t.kvh) << a.ps_log2) |
                                  (((j < prefix_tiles ? j : j - prefix_tiles) * kKeys + 16 * w + (lane & 15)) & (ps - 1)))
                               : ~0u;
        ahead = page_of(j + 1);
        if (i == 0 && ok)  // (later tiles have been asked for)
          for (int x = 0; x < HD; x += 32)
            asm volatile("prefetch.global.L2 [%0];" ::"l"((lane < 16 ? a.k32 : a.v32) + (size_t)at * HD + x));
        // half of the warp one row, a lane 8 of its values; N pairs of rows on their way, M at a time
        constexpr int N = 4, M = 2;
        const int h = lane >> 4, c = lane & 15;
        float v[N][8];
        auto load = [&](const float* pool, int e, int pair) {
          const unsigned from = __shfl_sync(0xffffffffu, at, 2 * pair + h);
          const float* row = (from == ~0u ? no_key : pool + (size_t)from * HD) + 8 * c;
          load4(row, v[e]);
          load4(row + 4, v[e] + 4);
        };
        const uint32_t swizzle = ((c & 7) ^ h) << 4;
        uint32_t to = sk + (c >> 3) * kHalf + (16 * w + h) * 128;
#pragma unroll
        for (int e = 0; e < N; ++e) load(a.k32, e, e);
        if (i > 0) wait(sfull((i - 1) % G), (i - 1) / G);  // the last tile's scores are there, its keys have been read
#pragma unroll 1
        for (int e0 = 0; e0 < 8; e0 += N, to += 2 * N * 128)
#pragma unroll
          for (int d = 0; d < N; d += M) {
            float most[M];
#pragma unroll
            for (int e = 0; e < M; ++e) {
              const float* x = v[d + e];
              most[e] = fmaxf(fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3]))),
                              fmaxf(fmaxf(fabsf(x[4]), fabsf(x[5])), fmaxf(fabsf(x[6]), fabsf(x[7]))));
            }
#pragma unroll
            for (int off = 8; off > 0; off >>= 1)
#pragma unroll
              for (int e = 0; e < M; ++e) most[e] = fmaxf(most[e], __shfl_xor_sync(0xffffffffu, most[e], off));
#pragma unroll
            for (int e = 0; e < M; ++e) {
              float back;
              const float mul = row_scale<TQ>(most[e], back);
#pragma unroll
              for (int x = 0; x < 8; ++x) v[d + e][x] *= mul;
              if (c == 0) key_scale_of[i % 3 * kRows + 16 * w + 2 * (e0 + d + e) + h] = __float2bfloat16(back);
            }
#pragma unroll
            for (int p = 0; p < 2; ++p)
#pragma unroll
              for (int e = d; e < d + M; ++e) {
                uint32_t b[4];
#pragma unroll
                for (int x = 0; x < 4; ++x) b[x] = weight_plane<TQ>(v[e][2 * x], v[e][2 * x + 1], p < 1);
                sts128(to + p * kTileBytes + e * 256 + (swizzle ^ (e * 32)), b[0], b[1], b[2], b[3]);
              }
            if (e0 + N < 8)
#pragma unroll
              for (int e = d; e < d + M; ++e) load(a.k32, e, e0 + N + e);
          }
        if (lane == 0) {
          // (what stood there of tile i - 3 has been read: the scores of tile i - 1 are there)
          reinterpret_cast<volatile uint16_t*>(bad_keys)[i % 3 * 8 + w] = (uint16_t)bad;
          if (bad) atomicOr(a.status, (int)kStatusBadPage);
        }
        fence_proxy_async();
        arrive(kfull(0));
#pragma unroll
        for (int e = 0; e < N; ++e) load(a.v32, e, e);
        if (i > 0) wait(vempty((i - 1) % G), (i - 1) / G);  // the last tile's O is there, its values have been read
        f32x2 none = 0;  // 0, or NaN: some value is not finite
        to += (sv - sk) - 16 * 128;
#pragma unroll 1
        for (int e0 = 0; e0 < 8; e0 += N, to += 2 * N * 128)
#pragma unroll
          for (int e = 0; e < N; ++e) {
#pragma unroll
            for (int x = 0; x < 8; x += 2) none = fma2(pair(v[e][x], v[e][x + 1]), 0, none);
#pragma unroll
            for (int p = 0; p < 3; ++p) {
              uint32_t b[4];
#pragma unroll
              for (int x = 0; x < 4; ++x) b[x] = weight_plane<TP>(v[e][2 * x], v[e][2 * x + 1], p < 2);
              sts128(to + p * kTileBytes + e * 256 + (swizzle ^ (e * 32)), b[0], b[1], b[2], b[3]);
            }
            if (e0 + N < 8) load(a.v32, e, e0 + N + e);
          }
        float n0, n1;
        unpair(none, n0, n1);
        const bool odd = __any_sync(0xffffffffu, !(n0 + n1 == 0.f));
        if (lane == 0) odd_values[w] = odd;
        fence_proxy_async();
        arrive(vfull(0));
      }
      done();
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == L::kScoreWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <typename T> int launch_tc(ChunkArgs a, void* k, void* v, cudaStream_t stream) {
  using L = Layout<T>;
  static std::atomic<bool> smem_set[64];  // idempotent: concurrent first calls only repeat it
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -4;
  if (!smem_set[dev].load(std::memory_order_acquire)) {
    if (const int e =
            launch_code(cudaFuncSetAttribute(chunks_tc_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)L::kSmem)))
      return e;
    smem_set[dev].store(true, std::memory_order_release);
  }
  CUtensorMap maps[2] = {};
  if (L::kSplit) {
    a.k32 = static_cast<const float*>(k);
    a.v32 = static_cast<const float*>(v);
  } else {
    for (int i = 0; i < 2; ++i)
      if (!encode_pool(&maps[i], i ? v : k, Planes<typename L::P>::format, a.nkv, a.ps_log2, a.n_pages, 1 << a.box_log2)) return -4;
  }
  return launch_pdl(chunks_tc_kernel<T>, dim3(kGrid), dim3(L::kThreads), L::kSmem, stream, a, maps[0], maps[1]);
}

}  // namespace

namespace chunks {

int launch_chunks_tc(const ChunkArgs& a, void* k, void* v, int kv_type, cudaStream_t stream) {
  if (kv_type == F32) return launch_tc<float>(a, k, v, stream);
  return kv_type == F16 ? launch_tc<__half>(a, k, v, stream) : launch_tc<__nv_bfloat16>(a, k, v, stream);
}

}  // namespace chunks
}  // namespace pyr
