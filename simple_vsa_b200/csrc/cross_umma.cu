// Cross attention on the Blackwell tensor path: bf16 and fp16, head dims that are multiples of 8 up to 128 (tiles of 64 or 128 dims, the
// rest of a box lies outside the tensor and is zero-filled), any lengths, strides of multiples of 16 bytes read in place by TMA.
//
// Unlike the sparse kernels a query tile meets few key tiles (an encoder's states: four tiles of 128 at 512 keys), so set-up, first
// loads and epilogue must not be paid per tile: the CTAs are persistent, and every role runs ahead of the others from one piece of
// work to the next.
#include <cuda.h>

#include <atomic>

#include "common.cuh"
#include "kernels.h"
#include "umma.cuh"

namespace vsa {
namespace {

using namespace umma;

constexpr int kRows = 128;                 // rows of a tile: queries or keys
constexpr int kHalf = kRows * 128;         // 64 head dims of a tile: 128 rows x 128 bytes
constexpr uint32_t kTmemCols = 512;

template <typename T> constexpr uint32_t kFmt = 1u;
template <> constexpr uint32_t kFmt<__half> = 0u;

// Whole-warp wait, bounded by the SM's clock.  Short on purpose: a role's loop with a dozen inlined waits that each look at a global
// timer and the status word as well is more code than the instruction caches keep beside the softmax (a wait for a barrier that
// had long flipped took 340 cycles).
constexpr uint32_t kWaitCycles = 500u * 1000u * 1000u;      // a quarter of a second
__device__ __forceinline__ uint32_t sm_clock() {
  uint32_t t;
  asm volatile("mov.u32 %0, %%clock;" : "=r"(t));
  return t;
}
__device__ __forceinline__ bool wait_for(uint32_t bar, uint32_t parity) {
  if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
  const uint32_t t0 = sm_clock();
#pragma unroll 1
  for (;;) {
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    if (__any_sync(0xffffffffu, sm_clock() - t0 > kWaitCycles)) return false;
  }
}
#define CROSS_WAIT(bar_, parity_) wait_for((bar_), (parity_))

// The end of every role: a __syncthreads, and where a wait of any thread has run out, time for copies and products that are still in flight
// to land (a millisecond; they take microseconds) before the CTA gives its shared and tensor memory back.
constexpr uint32_t kSettleCycles = 2u * 1000u * 1000u;
__device__ __forceinline__ void settle(bool ok) {
  if (__syncthreads_or(!ok)) {
    const uint32_t t0 = sm_clock();
#pragma unroll 1
    while (sm_clock() - t0 < kSettleCycles) {
    }
  }
}

// Division of n < 2^31 by a number known on the host: (n + umulhi(n, mul)) >> shift.
struct Divisor {
  uint32_t by, mul, shift;
  explicit Divisor(uint32_t d) : by(d), shift(0) {
    while ((1ull << shift) < d) ++shift;
    mul = (uint32_t)(((1ull << 32) * ((1ull << shift) - d)) / d + 1);
  }
  __device__ __forceinline__ int operator()(int n) const { return (int)(((uint32_t)n + __umulhi((uint32_t)n, mul)) >> shift); }
};

// D[128 x N] = A[128 x HD] B[N x HD]^T, both K-major; halves of 64 head dims kHalf / B_HALF bytes apart.
template <typename T, int HD, int N, int B_HALF>
__device__ __forceinline__ void issue_scores(uint32_t d_tmem, uint32_t a_tile, uint32_t b_tile) {
  constexpr uint32_t idesc = instr_desc(128, N, 0, 0, kFmt<T>);
  constexpr uint32_t hi = desc_hi(1024);
  const uint32_t a0 = desc_lo(a_tile, 16), b0 = desc_lo(b_tile, 16);
#pragma unroll
  for (int ks = 0; ks < HD / 16; ++ks)
    mma_ss(d_tmem, desc_pack(a0 + (uint32_t)(((ks >> 2) * kHalf + (ks & 3) * 32) >> 4), hi),
           desc_pack(b0 + (uint32_t)(((ks >> 2) * B_HALF + (ks & 3) * 32) >> 4), hi), idesc, ks > 0 ? 1u : 0u);
}
// D[128 x HD] (+)= A[128 x ROWS] (tensor memory, 16-bit) B[ROWS x HD] (dims contiguous, TILE rows a half).  The A columns were written
// by groups of GROUP scores each, every group packing its half-width result at the start of its own columns.
template <typename T, int HD, int ROWS, int GROUP, int TILE>
__device__ __forceinline__ void issue_product(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_tile, bool accumulate) {
  constexpr uint32_t idesc = instr_desc(128, HD, 0, 1, kFmt<T>);
  constexpr uint32_t hi = desc_hi(1024);
  const uint32_t b0 = desc_lo(b_tile, TILE * 128);
  const uint32_t acc0 = accumulate ? 1u : 0u;
#pragma unroll
  for (int ks = 0; ks < ROWS / 16; ++ks)
    mma_ts(d_tmem, a_tmem + (uint32_t)((ks * 16 / GROUP) * GROUP + (ks * 16 % GROUP) / 2), desc_pack(b0 + (uint32_t)(ks * 128), hi), idesc,
           ks > 0 ? 1u : acc0);
}
template <typename T>
__device__ __forceinline__ uint4 pack8(const uint32_t* r) {
  return make_uint4(Elem<T>::pack(__uint_as_float(r[0]), __uint_as_float(r[1])), Elem<T>::pack(__uint_as_float(r[2]), __uint_as_float(r[3])),
                    Elem<T>::pack(__uint_as_float(r[4]), __uint_as_float(r[5])), Elem<T>::pack(__uint_as_float(r[6]), __uint_as_float(r[7])));
}
// HD/64 boxes of rows x 64 dims of one (batch, head) slice on one barrier, whose bytes the caller has announced
template <int HD>
__device__ __forceinline__ void load_rows(uint32_t dst, const CUtensorMap* map, int row, int head, int batch, uint32_t half_bytes, uint32_t bar) {
#pragma unroll
  for (int h = 0; h < HD / 64; ++h) tma_load_4d(dst + h * half_bytes, map, h * 64, row, head, batch, bar);
}

__device__ __forceinline__ float max3(float x, uint32_t y, uint32_t z) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(__uint_as_float(y)), "f"(__uint_as_float(z)));
  return r;
}

// 2^x of two values on the FMA pipe, for a share of the exponentials (the MUFU makes 16 a clock and SM, one for every 64 multiply-adds
// of the tensor cores at head dim 128): x = n + f with n the nearest integer, a polynomial in f on [-1/2, 1/2] (minimax of the relative
// error: degree 3, 7.5e-5, a twentieth of bf16's half step; degree 4, 2.6e-6, for fp16), times 2^n.  Below 2^-126: 2^-126.  NaN stays NaN.
template <typename T>
__device__ __forceinline__ float2 poly_exp2(float2 x) {
  asm("max.NaN.f32 %0, %0, 0fC2FC0000;" : "+f"(x.x));       // -126
  asm("max.NaN.f32 %0, %0, 0fC2FC0000;" : "+f"(x.y));
  const float2 magic = make_float2(12582912.f, 12582912.f);           // 1.5 * 2^23: the integer lands in the low bits
  const float2 t = add2(x, magic), n = add2(t, make_float2(-12582912.f, -12582912.f));
  const float2 f = fma2(n, make_float2(-1.f, -1.f), x);
  float2 p;
  if (sizeof(T) == 2 && kFmt<T> == 1u) {
    p = fma2(make_float2(0.0551716685f, 0.0551716685f), f, make_float2(0.242611125f, 0.242611125f));
    p = fma2(p, f, make_float2(0.693260968f, 0.693260968f));
    p = fma2(p, f, make_float2(0.999928057f, 0.999928057f));
  } else {
    p = fma2(make_float2(0.00957010221f, 0.00957010221f), f, make_float2(0.0559178591f, 0.0559178591f));
    p = fma2(p, f, make_float2(0.240247443f, 0.240247443f));
    p = fma2(p, f, make_float2(0.693121791f, 0.693121791f));
    p = fma2(p, f, make_float2(0.999999285f, 0.999999285f));
  }
  return mul2(p, make_float2(__uint_as_float((__float_as_uint(t.x) << 23) + 0x3f800000u), __uint_as_float((__float_as_uint(t.y) << 23) + 0x3f800000u)));
}
template <typename T>
__device__ __forceinline__ float2 exp2_pair(float2 x, bool poly) {
  return poly ? poly_exp2<T>(x) : make_float2(fast_exp2(x.x), fast_exp2(x.y));
}

// fp16 holds numbers from 2^16 down to 2^-14 in full, and small gradients against many keys are below that long before the result is: the
// backward's 16-bit operands are therefore kept in the middle of the range by powers of two that the way out takes back (bf16 has the range
// of fp32).  P, at most 1, is held as P 2^14.  dS = P (dP - delta): with dP_ij = do_i.v_j and delta the mean of dP_i under P_i,
// |dS_ij| = P_ij |sum_k P_ik (dP_ij - dP_ik)| <= P (1 - P) 2 |do_i| max|v| <= |do_i| max|v| / 2, so that the largest 2^e with
// 2^e |do_i| max|v| <= 2^15 keeps it within 2^14 whatever the operands hold.  The factor of four to the type's end is for the roundings of
// delta and of exponents of many thousands.  dQ takes an e for each row; dK and dV add rows up, and take one for all rows of a key head.
template <typename T> constexpr bool kRanged = kFmt<T> == 0u;
constexpr int kPShift = 14;
// e from the product of the squared norms (0: nothing to hold; infinite or NaN: nothing to save)
__device__ __forceinline__ int range_exponent(float squares) {
  const int log2 = (int)(__float_as_uint(squares) >> 23) - 127;      // floor; squares >= 0
  return max(-30, min(60, 14 - (log2 >> 1)));
}
// P and dS of the backward, to 16 bits.  In fp16 never to infinity: where the scores are so large that the last place of their fp32 statistic is
// several units (from 2^25 on), the weights formed with it may come out above four.
template <typename T>
__device__ __forceinline__ uint32_t pack_weights(float lo, float hi) {
  if constexpr (!kRanged<T>) {
    return Elem<T>::pack(lo, hi);
  } else {
    uint32_t w;
    asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(hi), "f"(lo));
    return w;
  }
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// ------------------------------------------------------------------------------------------------------
// forward
// ------------------------------------------------------------------------------------------------------
// A piece of work is 256 query rows of one head (two tiles of 128, which are the M dimension) against the key tiles of one split.  Both
// tiles take every K and V tile from the same buffers; four softmax warps own a tile, a thread a row.  The keys are walked 64 at a
// time and a tile has two score accumulators, so that the next scores are there when a softmax group has finished (with one accumulator
// of 128 keys the groups idled 42 % of the time behind S).  P goes over the scores it came from in tensor memory; the MMAs have an
// issuer warp for each product of each tile.
// The softmax keeps a running maximum, but moves the accumulated row only when the maximum has grown by more than 2^8: P stays below
// 2^8 (fp16 holds 2^16, the sums are fp32), and moving O through registers is rare.
//
// [1, 40, 92160, 128] x 512 keys, bf16: 867 us, 1115 TFLOP/s (959 in a long loop, power limit); [2, 12 + 4, 8190, 64] x 801 of 1001: 80 us.
// Counters at [1, 8, 92160, 128]: 1705 cycles per 256 x 64 scores, set-up and ends included; tensor pipe active for 60 % of them, its operand
// reads 54 % of what shared memory gives (128 KB, and 32 KB more arrive by TMA), exponentials 45 % with a quarter of them on the FMA pipe,
// instruction issue 53 %.  No pipe is full: what bounds it is a softmax group's chain (scores from tensor memory, maximum, exponentials, P
// back), which two groups overlap, and MMAs of 64 keys, which take 48 cycles of the 32 that their size asks for.
// More warps were slower: eight a tile sharing its rows, and four groups on alternating steps with the maximum handed on (982 for
// 860 us).  A piece's end (O out, the next piece's set-up) is some 3000 of 16000 cycles at 512 keys, but the other tile's group works
// under it: four warps that write O while both groups go on brought nothing (880 -> 891 us, at eight heads 181 -> 188).
constexpr int kFwdThreads = 256 + 256;     // loads and four issuers of MMAs (eight warps), two softmax groups
constexpr int kKeys = 64;                  // keys of a step
constexpr int kFwdPoly = 2;                // of eight pairs of exponentials, on the FMA pipe
template <int HD>
struct FwdSmem {
  static constexpr uint32_t tile = HD * 256;                      // 128 rows
  static constexpr int stages = HD == 128 ? 4 : 8;                // K and V tiles in turn
  static constexpr uint32_t q = 0;                                // two tiles
  static constexpr uint32_t kv = q + 2 * tile;
  static constexpr uint32_t stage = kv + stages * tile;           // 32 rows x 128 bytes a softmax warp
  static constexpr uint32_t bars = stage + 8 * 4096;
  static constexpr uint32_t misc = bars + 34 * 8;
  static constexpr uint32_t total = misc + 16;
};
static_assert(FwdSmem<128>::total <= 232448 && FwdSmem<64>::total <= 232448, "shared memory of the cross attention forward");
// the score accumulators of a tile: index 2 * tile + (step & 1)
enum FwdBar { F_Q_FULL = 0, F_Q_EMPTY = 2, F_O_FULL = 4, F_S_FULL = 6, F_S_EMPTY = 10, F_P_FULL = 14, F_KV_FULL = 18, F_KV_EMPTY = 26 };

struct FwdWork {
  Divisor splits, pairs, heads, group;          // splits of the keys; pairs of query tiles per head; query heads, and per key head
  int items;                                    // all pieces
  float *part_out, *part_lse;
};
struct FwdItem {
  int b, h, row0, tiles, len, j0, j1, split;    // tiles: 1 or 2 live query tiles; key tiles j0 .. j1
  __device__ __forceinline__ FwdItem(const VsaCross& a, const FwdWork& w, int item) {
    const int rest = w.splits(item), bh = w.pairs(rest);
    split = item - rest * (int)w.splits.by;
    b = w.heads(bh);
    h = bh - b * (int)w.heads.by;
    row0 = (rest - bh * (int)w.pairs.by) * 2 * kRows;
    tiles = row0 + kRows < (int)a.Lq ? 2 : 1;
    len = cross_length(a, b);
    const int n = (len + kRows - 1) / kRows, per = w.splits(n + (int)w.splits.by - 1);
    j0 = split * per;
    j1 = min(n, j0 + per);
  }
  // steps of 64 keys: the last tile may need only one
  __device__ __forceinline__ int halves() const { return j1 <= j0 ? 0 : min(2 * (j1 - j0), (len + kKeys - 1) / kKeys - 2 * j0); }
};

template <typename T, int HD>
__global__ void __launch_bounds__(kFwdThreads, 1)
cross_fwd_umma_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                      const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_out,
                      const __grid_constant__ VsaCross a, const FwdWork w, int* status) {
  using Sm = FwdSmem<HD>;
  extern __shared__ __align__(1024) uint8_t cross_smem[];
  if (*(volatile int*)status != 0) return;
  uint8_t* sm = cross_smem;
  const uint32_t base = smem_u32(sm);
  if (base & 1023u) {                              // the operand layouts need it
    if (threadIdx.x == 0) atomicCAS(status, 0, 70);
    return;
  }
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  volatile uint32_t* misc = reinterpret_cast<volatile uint32_t*>(sm + Sm::misc);
  auto bar = [&](int i) -> uint32_t { return base + Sm::bars + 8u * i; };
  if (tid == 0) {
    for (int t = 0; t < 2; ++t) {
      mbar_init(bar(F_Q_FULL + t), 1);
      mbar_init(bar(F_Q_EMPTY + t), 1);
      mbar_init(bar(F_O_FULL + t), 1);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(bar(F_S_FULL + i), 1);
      mbar_init(bar(F_S_EMPTY + i), 1);
      mbar_init(bar(F_P_FULL + i), 4);
    }
    for (int i = 0; i < Sm::stages; ++i) {
      mbar_init(bar(F_KV_FULL + i), 1);
      mbar_init(bar(F_KV_EMPTY + i), 2);           // one issuer for each query tile
    }
    fence_barrier_init();
    tma_prefetch_desc(&map_q);
    tma_prefetch_desc(&map_k);
    tma_prefetch_desc(&map_v);
  }
  if (warp == 5) {
    tmem_alloc(base + Sm::misc, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = misc[0];
  const uint32_t tmem_o = tmem + 256;              // two score accumulators of each tile, then O of the two tiles
  bool ok = true;

  if (warp >= 8) {                                 // 256 x 184 + 256 x 72 registers are the block's 512 x 128 at launch
    registers_inc<184>();
    const int quarter = warp & 3, t = (warp - 8) >> 2, row = quarter * 32 + lane;
    const uint32_t lane_addr = (uint32_t)(quarter * 32) << 16;
    const uint32_t o_addr = tmem_o + HD * t + lane_addr;
    const float c = a.scale * kLog2e;          // > 0
    uint32_t u = 0, pieces = 0, tiles = 0;         // steps and pieces of this tile so far; K/V tiles
    for (int item = blockIdx.x; item < w.items && ok; item += gridDim.x) {
      const FwdItem it(a, w, item);
      const int halves = it.halves();
      if (t >= it.tiles) {
        tiles += (halves + 1) >> 1;
        continue;
      }
      float m = -INFINITY;
      float2 lsum = make_float2(0.f, 0.f);
      for (int i = 0; i < halves; ++i, ++u) {
        const int key0 = it.j0 * kRows + i * kKeys;
        const int live = it.len - key0;                            // keys of this step that take part, or more
        const bool full = live >= kKeys;
        const int acc = 2 * t + (u & 1);
        const uint32_t s_addr = tmem + 64 * acc + lane_addr;
        ok = CROSS_WAIT(bar(F_S_FULL + acc), (u >> 1) & 1);
        if (!ok) break;
        tc_fence_after();
        uint32_t sv[2][32];
        tmem_ld(s_addr, sv[0]);
        tmem_ld(s_addr + 32, sv[1]);
        tmem_ld_wait();
        if (!full) {                               // what stands in a key that takes no part may be anything: P = 2^-inf
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            if (e >= live) sv[0][e] = 0xff800000u;
            if (32 + e >= live) sv[1][e] = 0xff800000u;
          }
        }
        float x[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int e = 0; e < 32; e += 4)
#pragma unroll
          for (int q = 0; q < 4; ++q) x[q] = max3(x[q], sv[q & 1][e + (q & 2)], sv[q & 1][e + (q & 2) + 1]);
        const float top = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])) * c;
        if (i == 0) {
          m = top;
        } else {
          const bool up = top > m + 8.f;
          if (__any_sync(0xffffffffu, up)) {       // all products before this step's must be in O; only this group lets the next start
            ok = CROSS_WAIT(bar(F_S_EMPTY + (acc ^ 1)), ((u - 1) >> 1) & 1);
            if (!ok) break;
            tc_fence_after();
            const float keep = up ? fast_exp2(m - top) : 1.f;
            if (up) m = top;
            lsum = mul2(lsum, make_float2(keep, keep));
#pragma unroll 1
            for (int d = 0; d < HD; d += 16) {
              uint32_t ov[16];
              tmem_ld(o_addr + d, ov);
              tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 16; ++e) ov[e] = __float_as_uint(__uint_as_float(ov[e]) * keep);
              tmem_st(o_addr + d, ov);
            }
          }
        }
        if (!full) {                               // rows of V that no key takes part with meet P = 0: they must be finite.  Both tiles'
                                                   // groups clear them, each before the product that it starts.
          const uint32_t r = 2 * (tiles + (i >> 1)) + 1, s = r % Sm::stages;
          ok = CROSS_WAIT(bar(F_KV_FULL + s), (r / Sm::stages) & 1);
          if (!ok) break;
          const int vr = (i & 1) * kKeys + (row & 63);             // two threads a row
          if ((row & 63) >= live) {
            uint8_t* vrow = sm + Sm::kv + s * Sm::tile + vr * 128;
#pragma unroll
            for (int e = 0; e < HD / 16; ++e) {
              const int ch = (row >> 6) * (HD / 16) + e;
              *reinterpret_cast<uint4*>(vrow + (ch >> 3) * kHalf + ((ch ^ vr) & 7) * 16) = make_uint4(0, 0, 0, 0);
            }
          }
          fence_proxy_async_smem();
        }
        const float shift = m == -INFINITY ? 0.f : m;
        const float2 c2 = make_float2(c, c), m2 = make_float2(-shift, -shift);
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          uint32_t pk[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float2 p = exp2_pair<T>(fma2(word_pair(sv[q] + 2 * e), c2, m2), kFwdPoly > 0 && e % 8 < kFwdPoly);
            lsum = add2(lsum, p);
            pk[e] = Elem<T>::pack(p.x, p.y);
          }
          tmem_st(s_addr + 16 * q, pk);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(F_P_FULL + acc));
      }
      if (!ok) break;
      tiles += (halves + 1) >> 1;
      const float sum = lsum.x + lsum.y, l = sum < 1e-6f ? 0.f : sum, inv = l == 0.f ? 0.f : 1.f / l;      // a live key is worth 2^-8 at least
      const bool any = halves > 0;
      if (any) {
        ok = CROSS_WAIT(bar(F_O_FULL + t), pieces & 1);
        if (!ok) break;
        ++pieces;
        tc_fence_after();
      }
      const int row_w = it.row0 + t * kRows + quarter * 32;         // first row of this warp
      const long long bh = (long long)it.b * a.H + it.h;
      if (w.splits.by == 1) {
        a.lse2[bh * cross_rows(a.Lq) + row_w + lane] = l == 0.f || row_w + lane >= a.Lq ? INFINITY : m + log2f(l);
        // 64 dims at a time through 32 rows x 128 bytes of shared memory and out by TMA, which leaves what lies outside the tensor
        uint8_t* stage = sm + Sm::stage + (warp - 8) * 4096;
#pragma unroll 1
        for (int d0 = 0; d0 < HD; d0 += 64) {
          uint32_t ov[2][32];
          tmem_ld(o_addr + d0, ov[0]);
          tmem_ld(o_addr + d0 + 32, ov[1]);
          if (lane == 0) bulk_wait_read();         // the boxes before have left the buffer
          __syncwarp();
          tmem_ld_wait();
#pragma unroll
          for (int q = 0; q < 2; ++q) {
#pragma unroll
            for (int e = 0; e < 32; ++e) ov[q][e] = any ? __float_as_uint(__uint_as_float(ov[q][e]) * inv) : 0u;
#pragma unroll
            for (int e = 0; e < 4; ++e)
              *reinterpret_cast<uint4*>(stage + lane * 128 + (((4 * q + e) ^ (lane & 7)) << 4)) = pack8<T>(ov[q] + 8 * e);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            if (row_w < a.Lq) tma_store_4d(&map_out, smem_u32(stage), d0, row_w, it.h, it.b);
            bulk_commit();
          }
        }
      } else {
        const long long at = (it.split * (long long)a.B * a.H + bh) * a.Lq + row_w + lane;
        const bool there = row_w + lane < a.Lq;
        if (there) w.part_lse[at] = l == 0.f ? -INFINITY : m + log2f(l);
#pragma unroll 1
        for (int d = 0; d < HD; d += 16) {
          uint32_t ov[16];
          tmem_ld(o_addr + d, ov);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 16; e += 4)
            if (there && d + e < a.D)
              *reinterpret_cast<float4*>(w.part_out + at * a.D + d + e) =
                  any ? make_float4(__uint_as_float(ov[e]) * inv, __uint_as_float(ov[e + 1]) * inv, __uint_as_float(ov[e + 2]) * inv,
                                    __uint_as_float(ov[e + 3]) * inv)
                      : make_float4(0.f, 0.f, 0.f, 0.f);
        }
      }
    }
    if (lane == 0) bulk_wait();
    if (!ok && lane == 0) atomicCAS(status, 0, 71);
  } else {
    registers_dec<72>();
    if (warp == 0) {
      uint32_t q_phase = 3, r = 0;                 // a bit per tile
      auto load_q = [&](const FwdItem& it, int t) {
        ok = CROSS_WAIT(bar(F_Q_EMPTY + t), q_phase >> t & 1);
        if (!ok) return;
        q_phase ^= 1u << t;
        if (elect_one()) {
          mbar_arrive_expect_tx(bar(F_Q_FULL + t), Sm::tile);
          load_rows<HD>(base + Sm::q + t * Sm::tile, &map_q, it.row0 + t * kRows, it.h, it.b, kHalf, bar(F_Q_FULL + t));
        }
        __syncwarp();
      };
      auto load_kv = [&](const FwdItem& it, const CUtensorMap* map, int j, int hk) {
        const uint32_t s = r % Sm::stages;
        ok = CROSS_WAIT(bar(F_KV_EMPTY + s), ((r / Sm::stages) & 1) ^ 1);
        if (!ok) return;
        ++r;
        if (elect_one()) {
          mbar_arrive_expect_tx(bar(F_KV_FULL + s), Sm::tile);
          load_rows<HD>(base + Sm::kv + s * Sm::tile, map, j * kRows, hk, it.b, kHalf, bar(F_KV_FULL + s));
        }
        __syncwarp();
      };
      for (int item = blockIdx.x; item < w.items && ok; item += gridDim.x) {
        const FwdItem it(a, w, item);
        if (it.halves() == 0) continue;
        const int hk = w.group(it.h);
        load_q(it, 0);
        for (int j = it.j0; j < it.j1 && ok; ++j) {
          load_kv(it, &map_k, j, hk);
          if (j == it.j0 && it.tiles == 2 && ok) load_q(it, 1);
          if (ok) load_kv(it, &map_v, j, hk);
        }
      }
      if (!ok && lane == 0) atomicCAS(status, 0, 72);
    } else if (warp <= 2) {
      // S = Q K^T of query tile t: K tile n is in buffer 2n of the ring.  A warp issues an MMA in 40 cycles and a commit in 70 to 100; one
      // warp for both products of both tiles took 3500 cycles per step and was what bounded the kernel.
      const int t = warp - 1;
      uint32_t u = 0, pieces = 0, r = 0;
      for (int item = blockIdx.x; item < w.items && ok; item += gridDim.x) {
        const FwdItem it(a, w, item);
        const int halves = it.halves();
        if (t < it.tiles && halves > 0) {
          ok = CROSS_WAIT(bar(F_Q_FULL + t), pieces & 1);
          ++pieces;
          for (int i = 0; i < halves && ok; ++i, ++u) {
            const uint32_t rk = r + (i & ~1), s = rk % Sm::stages;
            const int acc = 2 * t + (u & 1);
            ok = CROSS_WAIT(bar(F_KV_FULL + s), (rk / Sm::stages) & 1) && CROSS_WAIT(bar(F_S_EMPTY + acc), ((u >> 1) & 1) ^ 1);
            if (!ok) break;
            tc_fence_after();
            if (elect_one()) {
              issue_scores<T, HD, kKeys, kHalf>(tmem + 64 * acc, base + Sm::q + t * Sm::tile, base + Sm::kv + s * Sm::tile + (i & 1) * kKeys * 128);
              mma_commit(bar(F_S_FULL + acc));
              if (i == halves - 1) mma_commit(bar(F_Q_EMPTY + t));
              if ((i & 1) || i == halves - 1) mma_commit(bar(F_KV_EMPTY + s));
            }
            __syncwarp();
          }
        } else if (t == 1) {                       // a piece of one query tile: its K tiles are free when the other has read them
          for (int i = 0; i < halves; i += 2) {
            const uint32_t s = (r + i) % Sm::stages;
            ok = ok && CROSS_WAIT(bar(F_KV_FULL + s), ((r + i) / Sm::stages) & 1);
            if (ok && lane == 0) mbar_arrive(bar(F_KV_EMPTY + s));
          }
        }
        r += (halves + 1) & ~1;
      }
      if (!ok && lane == 0) atomicCAS(status, 0, 73);
    } else if (warp <= 4) {
      // O += P V of query tile t: V tile n is in buffer 2n + 1
      const int t = warp - 3;
      uint32_t u = 0, r = 0;
      for (int item = blockIdx.x; item < w.items && ok; item += gridDim.x) {
        const FwdItem it(a, w, item);
        const int halves = it.halves();
        if (t < it.tiles) {
          for (int i = 0; i < halves && ok; ++i, ++u) {
            const uint32_t rv = r + (i & ~1) + 1, s = rv % Sm::stages;
            const int acc = 2 * t + (u & 1);
            ok = CROSS_WAIT(bar(F_KV_FULL + s), (rv / Sm::stages) & 1) && CROSS_WAIT(bar(F_P_FULL + acc), (u >> 1) & 1);
            if (!ok) break;
            tc_fence_after();
            if (elect_one()) {
              issue_product<T, HD, kKeys, kKeys, kRows>(tmem_o + HD * t, tmem + 64 * acc, base + Sm::kv + s * Sm::tile + (i & 1) * kKeys * 128, i > 0);
              mma_commit(bar(F_S_EMPTY + acc));
              if (i == halves - 1) mma_commit(bar(F_O_FULL + t));
              if ((i & 1) || i == halves - 1) mma_commit(bar(F_KV_EMPTY + s));
            }
            __syncwarp();
          }
        } else {
          for (int i = 0; i < halves; i += 2) {
            const uint32_t rv = r + i + 1, s = rv % Sm::stages;
            ok = ok && CROSS_WAIT(bar(F_KV_FULL + s), (rv / Sm::stages) & 1);
            if (ok && lane == 0) mbar_arrive(bar(F_KV_EMPTY + s));
          }
        }
        r += (halves + 1) & ~1;
      }
      if (!ok && lane == 0) atomicCAS(status, 0, 74);
    }
  }
  tc_fence_before();
  settle(ok);
  if (warp == 5) tmem_dealloc(tmem, kTmemCols);
}

// ------------------------------------------------------------------------------------------------------
// dQ (and delta)
// ------------------------------------------------------------------------------------------------------
// A piece of work is 128 query rows of one head: S = Q K^T, dP = dO V^T, dQ += dS K per key tile.  Sixteen elementwise warps share a
// tile, 32 score columns a thread; S (later dS) in two accumulators, dP in one that is free again as soon as it has been read.  Four warps
// form delta = rowsum(out * dout) and the statistics of the next piece's rows from memory, into two buffers, and ask L2 for the rows
// of the piece after it; four more write a finished dQ while the elementwise warps are at the next piece.
//
// [1, 8, 92160, 128] x 512 keys: 265 us, 1094 TFLOP/s.  9770 cycles a piece of four key tiles, set-up and ends included; tensor pipe active for
// 63 % of them, issue 55 %, operand reads 49 %.  By clock readings in the roles a tile takes 1700 to 1800 (1536 of MMAs, 1024 of exponentials
// before three of eight moved to the FMA pipe), and a piece's elementwise warps wait 500 to 800 more for the delta warps, which are at loads
// of 64 KB all the time.  With delta and dQ done by the elementwise warps it took an eighth longer (268 us for 236, on a faster board).
// Loads of two delta rows in flight, and Q and dO on barriers of their own, changed nothing.
constexpr int kDqCols = 32;
constexpr int kDqGroups = kRows / kDqCols;
constexpr int kDqPoly = 3;                 // of eight pairs of exponentials, on the FMA pipe
constexpr int kDqThreads = 384 + 128 * kDqGroups;      // loads and issuers of MMAs, dQ out, delta, elementwise warps
template <int HD>
struct DqSmem {
  static constexpr uint32_t tile = HD * 256;
  static constexpr int k_stages = 3, v_stages = HD == 128 ? 1 : 2;
  static constexpr uint32_t q = 0;
  static constexpr uint32_t d_o = q + tile;
  static constexpr uint32_t k = d_o + tile;
  static constexpr uint32_t v = k + k_stages * tile;
  static constexpr uint32_t stage = v + v_stages * tile;          // 32 rows x 64 bytes x HD / 32 a helper warp
  static constexpr uint32_t stats = stage + 4 * (HD / 32) * 2048; // float2 [2][128]: delta and the statistic of a row
  static constexpr uint32_t exps = stats + 2048;                  // int8 [2][128]: kRanged's e of a row
  static constexpr uint32_t bars = exps + 256;
  static constexpr uint32_t misc = bars + 32 * 8;
  static constexpr uint32_t total = misc + 16;
};
static_assert(DqSmem<128>::total <= 232448, "shared memory of the cross attention dQ pass");
enum DqBar { Q_QDO_FULL = 0, Q_QDO_EMPTY = 1, Q_K_FULL = 2, Q_K_EMPTY = 5, Q_V_FULL = 8, Q_V_EMPTY = 10, Q_S_FULL = 12, Q_S_EMPTY = 14,
             Q_DP_FULL = 16, Q_DP_EMPTY = 17, Q_DS_FULL = 18, Q_ACC_FULL = 20, Q_ACC_EMPTY = 21, Q_STATS_FULL = 22, Q_STATS_EMPTY = 24 };

struct DqItem {
  int b, h, row0, len, n;                       // n key tiles
  __device__ __forceinline__ DqItem(const VsaCross& a, const Divisor& qtiles, const Divisor& heads, int item) {
    const int bh = qtiles(item);
    row0 = (item - bh * (int)qtiles.by) * kRows;
    b = heads(bh);
    h = bh - b * (int)heads.by;
    len = cross_length(a, b);
    n = (len + kRows - 1) / kRows;
  }
};

template <typename T, int HD>
__global__ void __launch_bounds__(kDqThreads, 1)
cross_dq_umma_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_do,
                     const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                     const __grid_constant__ CUtensorMap map_dq, const __grid_constant__ VsaCross a, const Divisor qtiles, const Divisor heads,
                     const Divisor group_heads, int items, int* status) {
  using Sm = DqSmem<HD>;
  extern __shared__ __align__(1024) uint8_t cross_smem[];
  if (*(volatile int*)status != 0) return;
  uint8_t* sm = cross_smem;
  const uint32_t base = smem_u32(sm);
  if (base & 1023u) {
    if (threadIdx.x == 0) atomicCAS(status, 0, 80);
    return;
  }
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  volatile uint32_t* misc = reinterpret_cast<volatile uint32_t*>(sm + Sm::misc);
  auto bar = [&](int i) -> uint32_t { return base + Sm::bars + 8u * i; };
  if (tid == 0) {
    mbar_init(bar(Q_QDO_FULL), 1);
    mbar_init(bar(Q_QDO_EMPTY), 2);              // the last products that read them
    for (int i = 0; i < Sm::k_stages; ++i) {
      mbar_init(bar(Q_K_FULL + i), 1);
      mbar_init(bar(Q_K_EMPTY + i), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar(Q_V_FULL + i), 1);
      mbar_init(bar(Q_V_EMPTY + i), 1);
      mbar_init(bar(Q_S_FULL + i), 1);
      mbar_init(bar(Q_S_EMPTY + i), 1);
      mbar_init(bar(Q_DS_FULL + i), 4 * kDqGroups);
      mbar_init(bar(Q_STATS_FULL + i), 4);
      mbar_init(bar(Q_STATS_EMPTY + i), 4 * kDqGroups + (kRanged<T> ? 4 : 0));
    }
    mbar_init(bar(Q_ACC_EMPTY), 4);
    mbar_init(bar(Q_DP_FULL), 1);
    mbar_init(bar(Q_DP_EMPTY), 4 * kDqGroups);
    mbar_init(bar(Q_ACC_FULL), 1);
    fence_barrier_init();
    tma_prefetch_desc(&map_q);
    tma_prefetch_desc(&map_do);
    tma_prefetch_desc(&map_k);
    tma_prefetch_desc(&map_v);
  }
  if (warp == 1) {
    tmem_alloc(base + Sm::misc, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = misc[0];
  const uint32_t tmem_dp = tmem + 256, tmem_acc = tmem + 384;
  bool ok = true;
  uint32_t n = 0, live_items = 0;                // key tiles and pieces (with a key tile) so far

  if (warp == 0) {
    for (int item = blockIdx.x; item < items && ok; item += gridDim.x) {
      const DqItem it(a, qtiles, heads, item);
      if (it.n == 0) continue;
      ok = CROSS_WAIT(bar(Q_QDO_EMPTY), (live_items & 1) ^ 1);
      if (!ok) break;
      ++live_items;
      if (elect_one()) {
        mbar_arrive_expect_tx(bar(Q_QDO_FULL), 2 * Sm::tile);
        load_rows<HD>(base + Sm::q, &map_q, it.row0, it.h, it.b, kHalf, bar(Q_QDO_FULL));
        load_rows<HD>(base + Sm::d_o, &map_do, it.row0, it.h, it.b, kHalf, bar(Q_QDO_FULL));
      }
      __syncwarp();
      const int hk = group_heads(it.h);
      for (int j = 0; j < it.n; ++j, ++n) {
        const uint32_t sk = n % Sm::k_stages, sv = n % Sm::v_stages;
        ok = CROSS_WAIT(bar(Q_K_EMPTY + sk), ((n / Sm::k_stages) & 1) ^ 1);
        if (!ok) break;
        if (elect_one()) {
          mbar_arrive_expect_tx(bar(Q_K_FULL + sk), Sm::tile);
          load_rows<HD>(base + Sm::k + sk * Sm::tile, &map_k, j * kRows, hk, it.b, kHalf, bar(Q_K_FULL + sk));
        }
        __syncwarp();
        ok = CROSS_WAIT(bar(Q_V_EMPTY + sv), ((n / Sm::v_stages) & 1) ^ 1);
        if (!ok) break;
        if (elect_one()) {
          mbar_arrive_expect_tx(bar(Q_V_FULL + sv), Sm::tile);
          load_rows<HD>(base + Sm::v + sv * Sm::tile, &map_v, j * kRows, hk, it.b, kHalf, bar(Q_V_FULL + sv));
        }
        __syncwarp();
      }
    }
    if (!ok && lane == 0) atomicCAS(status, 0, 81);
  } else if (warp == 2) {
    // S = Q K^T
    for (int item = blockIdx.x; item < items && ok; item += gridDim.x) {
      const DqItem it(a, qtiles, heads, item);
      if (it.n == 0) continue;
      ok = CROSS_WAIT(bar(Q_QDO_FULL), live_items & 1);
      ++live_items;
      for (int j = 0; j < it.n && ok; ++j, ++n) {
        const uint32_t s = n % Sm::k_stages, b = n & 1;
        ok = CROSS_WAIT(bar(Q_K_FULL + s), (n / Sm::k_stages) & 1) && CROSS_WAIT(bar(Q_S_EMPTY + b), ((n >> 1) & 1) ^ 1);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          issue_scores<T, HD, 128, kHalf>(tmem + b * 128, base + Sm::q, base + Sm::k + s * Sm::tile);
          mma_commit(bar(Q_S_FULL + b));
          if (j == it.n - 1) mma_commit(bar(Q_QDO_EMPTY));
        }
        __syncwarp();
      }
    }
    if (!ok && lane == 0) atomicCAS(status, 0, 82);
  } else if (warp == 1) {
    // dP = dO V^T
    for (int item = blockIdx.x; item < items && ok; item += gridDim.x) {
      const DqItem it(a, qtiles, heads, item);
      if (it.n == 0) continue;
      ok = CROSS_WAIT(bar(Q_QDO_FULL), live_items & 1);
      ++live_items;
      for (int j = 0; j < it.n && ok; ++j, ++n) {
        const uint32_t s = n % Sm::v_stages;
        ok = CROSS_WAIT(bar(Q_V_FULL + s), (n / Sm::v_stages) & 1) && CROSS_WAIT(bar(Q_DP_EMPTY), (n & 1) ^ 1);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          issue_scores<T, HD, 128, kHalf>(tmem_dp, base + Sm::d_o, base + Sm::v + s * Sm::tile);
          mma_commit(bar(Q_V_EMPTY + s));
          mma_commit(bar(Q_DP_FULL));
          if (j == it.n - 1) mma_commit(bar(Q_QDO_EMPTY));
        }
        __syncwarp();
      }
    }
    if (!ok && lane == 0) atomicCAS(status, 0, 83);
  } else if (warp == 3) {
    // dQ += dS K
    for (int item = blockIdx.x; item < items && ok; item += gridDim.x) {
      const DqItem it(a, qtiles, heads, item);
      for (int j = 0; j < it.n && ok; ++j, ++n) {
        const uint32_t s = n % Sm::k_stages, b = n & 1;
        ok = CROSS_WAIT(bar(Q_K_FULL + s), (n / Sm::k_stages) & 1) && CROSS_WAIT(bar(Q_DS_FULL + b), (n >> 1) & 1);
        if (ok && j == 0) ok = CROSS_WAIT(bar(Q_ACC_EMPTY), (live_items++ & 1) ^ 1);      // dQ of the piece before has been read
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          issue_product<T, HD, 128, kDqCols, 128>(tmem_acc, tmem + b * 128, base + Sm::k + s * Sm::tile, j > 0);
          mma_commit(bar(Q_K_EMPTY + s));
          mma_commit(bar(Q_S_EMPTY + b));
          if (j == it.n - 1) mma_commit(bar(Q_ACC_FULL));
        }
        __syncwarp();
      }
    }
    if (!ok && lane == 0) atomicCAS(status, 0, 84);
  } else if (warp < 8) {
    // dQ of a piece on its way out while the elementwise warps are at the next one.
    const int quarter = warp & 3, st = tid - 128;
    const uint32_t lane_addr = (uint32_t)(quarter * 32) << 16;
    uint8_t* stage = sm + Sm::stage + quarter * (HD / 32) * 2048;
    for (int item = blockIdx.x; item < items && ok; item += gridDim.x) {
      const DqItem it(a, qtiles, heads, item);
      if (it.n == 0) {                           // no key: zeros
        const long long stat = ((long long)it.b * a.H + it.h) * cross_rows(a.Lq) + it.row0;
        T* dq = (T*)a.dq + it.b * a.dq_stride[0] + it.h * a.dq_stride[1] + (long long)it.row0 * a.dq_stride[2];
        a.delta[stat + st] = 0.f;
        for (int i = st; i < kRows * (HD / 8); i += 128) {
          const int r = i / (HD / 8), d = i % (HD / 8) * 8;
          if (it.row0 + r < a.Lq && d < a.D) *reinterpret_cast<uint4*>(dq + r * a.dq_stride[2] + d) = make_uint4(0, 0, 0, 0);
        }
        continue;
      }
      float mul = 1.f;                           // bf16: the scale is in dS
      if (kRanged<T>) {
        ok = CROSS_WAIT(bar(Q_STATS_FULL + (live_items & 1)), (live_items >> 1) & 1);
        if (!ok) break;
        mul = a.scale * power_of_two(-reinterpret_cast<const int8_t*>(sm + Sm::exps)[(live_items & 1) * kRows + quarter * 32 + lane]);
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(Q_STATS_EMPTY + (live_items & 1)));
      }
      ok = CROSS_WAIT(bar(Q_ACC_FULL), live_items & 1);
      if (!ok) break;
      ++live_items;
      tc_fence_after();
      if (lane == 0) bulk_wait_read();           // the boxes before have left the buffer
      __syncwarp();
#pragma unroll 1
      for (int c = 0; c < HD / 32; ++c) {
        uint32_t av[32];
        tmem_ld(tmem_acc + lane_addr + 32 * c, av);
        tmem_ld_wait();
        if (c == HD / 32 - 1) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(Q_ACC_EMPTY));
        }
        if (kRanged<T>)
#pragma unroll
          for (int i = 0; i < 32; ++i) av[i] = __float_as_uint(__uint_as_float(av[i]) * mul);
        // TMA's 64-byte swizzle (pieces xor row / 2); what lies outside the tensor is not written
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *reinterpret_cast<uint4*>(stage + c * 2048 + lane * 64 + ((q ^ (lane >> 1 & 3)) << 4)) = pack8<T>(av + 8 * q);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        for (int c = 0; c < HD / 32; ++c)
          if (it.row0 + quarter * 32 < a.Lq && 32 * c < a.D)
            tma_store_4d(&map_dq, smem_u32(stage) + c * 2048, 32 * c, it.row0 + quarter * 32, it.h, it.b);
        bulk_commit();
      }
    }
    if (lane == 0) bulk_wait();
    if (!ok && lane == 0) atomicCAS(status, 0, 86);
  } else if (warp < 12) {
    // delta and the statistics of the next piece's rows while this one is worked on
    const int st = tid - 256;
    const float log_scale = kRanged<T> ? 0.f : log2f(a.scale);      // > 0
    const long long lp = cross_rows(a.Lq);
    // The rows of the next piece into L2: its loads come when there is room for them, too late to wait for memory.
    auto ask = [&](const void* p, const int64_t(&stride)[3], const DqItem& it) {
      const T* row = (const T*)p + it.b * stride[0] + it.h * stride[1] + (long long)min(it.row0 + st, (int)a.Lq - 1) * stride[2];
#pragma unroll
      for (int d = 0; d < HD; d += 64) asm volatile("prefetch.global.L2 [%0];" ::"l"(row + min(d, a.D - 1)));
    };
    for (int item = blockIdx.x; item < items && ok; item += gridDim.x) {
      const DqItem it(a, qtiles, heads, item);
      const long long bhk = (long long)it.b * a.Hkv + group_heads(it.h);
      const float v_part = kRanged<T> ? a.bounds[bhk * VSA_CROSS_BOUNDS + lane] : 0.f;
      if (item + (int)gridDim.x < items) {
        const DqItem next(a, qtiles, heads, item + gridDim.x);
        ask(a.out, a.out_stride, next);
        ask(a.q, a.q_stride, next);
        ask(a.dout, a.dout_stride, next);
      }
      if (it.n == 0) continue;
      ok = CROSS_WAIT(bar(Q_STATS_EMPTY + (live_items & 1)), ((live_items >> 1) & 1) ^ 1);
      if (!ok) break;
      float2* to = reinterpret_cast<float2*>(sm + Sm::stats) + (live_items & 1) * kRows;
      int8_t* to_exp = reinterpret_cast<int8_t*>(sm + Sm::exps) + (live_items & 1) * kRows;
      const float v_bound = kRanged<T> ? warp_max(v_part) : 0.f;
      float g_bound = 0.f;                       // max |do|^2 of this thread's rows
      const long long stat = ((long long)it.b * a.H + it.h) * lp + it.row0;
      const T* o = (const T*)a.out + it.b * a.out_stride[0] + it.h * a.out_stride[1] + (long long)it.row0 * a.out_stride[2];
      const T* g = (const T*)a.dout + it.b * a.dout_stride[0] + it.h * a.dout_stride[1] + (long long)it.row0 * a.dout_stride[2];
      // four neighbouring threads a row, 16-byte pieces in turn
#pragma unroll 1
      for (int r = st >> 2; r < kRows; r += 32) {
        uint4 x[HD / 32], y[HD / 32];
        const int rr = min(it.row0 + r, (int)a.Lq - 1) - it.row0;
#pragma unroll
        for (int i = 0; i < HD / 32; ++i) {
          const int d = min((4 * i + (st & 3)) * 8, a.D - 8);
          x[i] = *reinterpret_cast<const uint4*>(o + rr * a.out_stride[2] + d);
          y[i] = *reinterpret_cast<const uint4*>(g + rr * a.dout_stride[2] + d);
        }
        const float lse = a.lse2[stat + r];
        float sum = 0.f, norm = 0.f;
#pragma unroll
        for (int i = 0; i < HD / 32; ++i) {
          if ((4 * i + (st & 3)) * 8 >= a.D) continue;
          const uint32_t *p = &x[i].x, *q = &y[i].x;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 u = Elem<T>::unpack(p[e]), w = Elem<T>::unpack(q[e]);
            sum = fmaf(u.x, w.x, fmaf(u.y, w.y, sum));
            if (kRanged<T>) norm = fmaf(w.x, w.x, fmaf(w.y, w.y, norm));
          }
        }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        int e = 0;
        if (kRanged<T>) {
          norm += __shfl_xor_sync(0xffffffffu, norm, 1);
          norm += __shfl_xor_sync(0xffffffffu, norm, 2);
          g_bound = __uint_as_float(max(__float_as_uint(g_bound), __float_as_uint(norm)));      // NaN stays
          e = range_exponent(norm * v_bound);
        }
        if ((st & 3) == 0) {
          if (it.row0 + r >= a.Lq) sum = 0.f;
          a.delta[stat + r] = sum;
          // bf16: 2^(s c - lse) * scale in one exponential; fp16: delta of the dP 2^e that the elementwise warps form
          to[r] = make_float2(kRanged<T> ? sum * power_of_two(e) : sum, log_scale - lse);
          if (kRanged<T>) to_exp[r] = (int8_t)e;
        }
      }
      if (kRanged<T>) {                          // for the dK/dV pass; the order of the rows changes nothing
        const unsigned top = __reduce_max_sync(0xffffffffu, __float_as_uint(g_bound));
        if (lane == 0) atomicMax(reinterpret_cast<unsigned*>(a.bounds) + bhk * VSA_CROSS_BOUNDS + VSA_CROSS_BOUNDS - 1, top);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(Q_STATS_FULL + (live_items & 1)));
      ++live_items;
    }
    if (!ok && lane == 0) atomicCAS(status, 0, 87);
  } else {
    const int quarter = warp & 3, cg = (warp - 12) >> 2, row = quarter * 32 + lane, c0 = cg * kDqCols;
    const uint32_t lane_addr = (uint32_t)(quarter * 32) << 16;
    const float c = a.scale * kLog2e;
    const float2 c2 = make_float2(c, c);
    const float2* stats = reinterpret_cast<const float2*>(sm + Sm::stats) + row;
    for (int item = blockIdx.x; item < items && ok; item += gridDim.x) {
      const DqItem it(a, qtiles, heads, item);
      if (it.n == 0) continue;
      ok = CROSS_WAIT(bar(Q_STATS_FULL + (live_items & 1)), (live_items >> 1) & 1);
      if (!ok) break;
      const float2 row_stats = stats[(live_items & 1) * kRows];
      float2 f2 = make_float2(1.f, 1.f);
      if (kRanged<T>) f2.x = f2.y = power_of_two(reinterpret_cast<const int8_t*>(sm + Sm::exps)[(live_items & 1) * kRows + row]);
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(Q_STATS_EMPTY + (live_items & 1)));
      ++live_items;
      const float2 l2 = make_float2(row_stats.y, row_stats.y), d2 = make_float2(-row_stats.x, -row_stats.x);
      for (int j = 0; j < it.n; ++j, ++n) {
        const uint32_t b = n & 1;
        const int live = it.len - j * kRows;     // keys of this tile that take part, or more
        ok = CROSS_WAIT(bar(Q_S_FULL + b), (n >> 1) & 1);
        if (!ok) break;
        tc_fence_after();
        const uint32_t s_addr = tmem + b * 128 + lane_addr + c0;
        if (live < kRows && cg == 0) {           // rows of K that no key takes part with meet dS = 0: they must be finite (S is done)
          if (row >= live) {
            uint8_t* krow = sm + Sm::k + (n % Sm::k_stages) * Sm::tile + row * 128;
#pragma unroll 1
            for (int ch = 0; ch < HD / 8; ++ch)
              *reinterpret_cast<uint4*>(krow + (ch >> 3) * kHalf + ((ch ^ row) & 7) * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
        }
        float2 pf[kDqCols / 2];
        uint32_t pk[kDqCols / 2];
#pragma unroll
        for (int h = 0; h < kDqCols; h += 16) {
          uint32_t sv[16];
          tmem_ld(s_addr + h, sv);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 8; ++i) pf[h / 2 + i] = exp2_pair<T>(fma2(word_pair(sv + 2 * i), c2, l2), kDqPoly > 0 && i < kDqPoly);
        }
        ok = CROSS_WAIT(bar(Q_DP_FULL), n & 1);
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int h = 0; h < kDqCols; h += 16) {
          uint32_t dv[16];
          tmem_ld(tmem_dp + lane_addr + c0 + h, dv);
          tmem_ld_wait();
          if (h + 16 == kDqCols) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(Q_DP_EMPTY));
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float2 y = mul2(pf[h / 2 + i], kRanged<T> ? fma2(word_pair(dv + 2 * i), f2, d2) : add2(word_pair(dv + 2 * i), d2));
            pk[h / 2 + i] = pack_weights<T>(y.x, y.y);
          }
        }
        if (c0 + kDqCols > live) {               // what stands in a key that takes no part may be anything
#pragma unroll
          for (int i = 0; i < kDqCols / 2; ++i) {
            if (c0 + 2 * i >= live) pk[i] = 0u;
            else if (c0 + 2 * i + 1 >= live) pk[i] &= 0xffffu;
          }
        }
        tmem_st(s_addr, pk);                     // over this thread's own scores
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(Q_DS_FULL + b));
      }
    }
    if (!ok && lane == 0) atomicCAS(status, 0, 85);
  }
  tc_fence_before();
  settle(ok);
  if (warp == 1) tmem_dealloc(tmem, kTmemCols);
}

// ------------------------------------------------------------------------------------------------------
// dK / dV: lanes = 128 key rows, columns = 64 query rows of a streamed tile
// ------------------------------------------------------------------------------------------------------
// A CTA owns 128 keys of one key head and walks a range of the query tiles of all heads that share it; K and V stay in shared memory,
// dK and dV in tensor memory.  S^T = K Q^T, dP^T = V dO^T, dV += P^T dO, dK += dS^T Q: 2560 cycles of MMAs per 128 x 128 scores, of 2700, which
// is what bounds it at D = 128: [1, 8, 92160, 128] x 512 keys 287 us, 1350 TFLOP/s (tensor pipe active for 76 %, operand reads 71 %).  At
// D = 64 a step's chain does (159 us at [2, 12 + 4, 8190, 64] x 801 of 1001 keys, fp16, 153 before its operands were kept in range; tensor
// pipe 38 %, issue 43 %; with two buffers and all exponentials on the MUFU a tenth longer).  The range is cut so that the CTAs
// fill whole waves of SMs; parts are added by a kernel of their own, in the order of the cuts.
constexpr int kQTile = 64;
constexpr int kSlab = kQTile * 128;
constexpr int kDkCols = 32;
constexpr int kDkGroups = kQTile / kDkCols;
constexpr int kDkEwThreads = 128 * kDkGroups;
constexpr int kDkThreads = 128 + kDkEwThreads;
template <int HD> constexpr int kDkPoly = HD == 64 ? 2 : 0;      // of eight pairs of exponentials, on the FMA pipe
template <int HD>
struct DkSmem {
  static constexpr uint32_t tile = HD * 256;          // 128 resident rows
  static constexpr uint32_t part = HD * 128;          // 64 streamed rows
  static constexpr int q_stages = 5, do_stages = 5;
  // buffers of (S^T, dP^T): at head dim 64 the gradients leave room for a third, and a step's chain is longer than its products
  static constexpr int bufs = HD == 64 ? 3 : 2;
  static constexpr uint32_t k = 0;
  static constexpr uint32_t v = k + tile;
  static constexpr uint32_t q = v + tile;
  static constexpr uint32_t d_o = q + q_stages * part;
  static constexpr uint32_t stats = d_o + do_stages * part;       // per Q stage: lse [64], delta [64]
  static constexpr uint32_t bars = stats + q_stages * 512;
  static constexpr uint32_t misc = bars + 40 * 8;
  static constexpr uint32_t total = misc + 16;
};
static_assert(DkSmem<128>::total <= 232448, "shared memory of the cross attention dK/dV pass");
enum DkBar { K_KV_FULL = 0, K_Q_FULL = 1, K_Q_EMPTY = 6, K_DO_FULL = 11, K_DO_EMPTY = 16, K_S_FULL = 21, K_S_EMPTY = 24,
             K_DP_FULL = 27, K_DP_EMPTY = 30, K_P_FULL = 33, K_DS_FULL = 36, K_ACC_FULL = 39 };

template <typename T, int HD>
__global__ void __launch_bounds__(kDkThreads, 1)
cross_dkdv_umma_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_do,
                       const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ VsaCross a,
                       int ktiles, int splits, float* part, int* status) {
  using Sm = DkSmem<HD>;
  extern __shared__ __align__(1024) uint8_t cross_smem[];
  if (*(volatile int*)status != 0) return;
  uint8_t* sm = cross_smem;
  const uint32_t base = smem_u32(sm);
  if (base & 1023u) {
    if (threadIdx.x == 0) atomicCAS(status, 0, 90);
    return;
  }
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  // the parts of a key head's tiles lie next to each other in launch order: they stream the same query tiles
  const int unit = blockIdx.x;
  const int ktile = unit % ktiles, rest = unit / ktiles, split = rest % splits, bhk = rest / splits;
  const int b = bhk / (int)a.Hkv, hk = bhk - b * (int)a.Hkv, group_heads = (int)(a.H / a.Hkv);
  const int krow0 = ktile * kRows;
  const int live_keys = cross_length(a, b) - krow0;      // keys of this tile that take part, or more
  const int qtiles = (int)((a.Lq + kQTile - 1) / kQTile);
  const long long total = (long long)qtiles * group_heads, per = (total + splits - 1) / splits;
  const long long first = split * per, last = first + per < total ? first + per : total;
  const int n_tiles = live_keys > 0 && last > first ? (int)(last - first) : 0;
  const float c = a.scale * kLog2e;
  const long long lp = cross_rows(a.Lq);
  const long long one = (long long)a.B * a.Hkv * a.Lkv * a.D;      // values of a partial dK
  const long long part_row = ((long long)bhk * a.Lkv + krow0) * a.D;

  if (n_tiles == 0) {                             // no query, or no key that takes part: zeros
    for (int i = tid; i < kRows * HD / 8; i += kDkThreads) {
      const int r = i / (HD / 8), d = i % (HD / 8) * 8;
      if (krow0 + r >= a.Lkv || d >= a.D) continue;
      if (part == nullptr) {
        *reinterpret_cast<uint4*>((T*)a.dk + b * a.dk_stride[0] + hk * a.dk_stride[1] + (krow0 + r) * a.dk_stride[2] + d) = make_uint4(0, 0, 0, 0);
        *reinterpret_cast<uint4*>((T*)a.dv + b * a.dv_stride[0] + hk * a.dv_stride[1] + (krow0 + r) * a.dv_stride[2] + d) = make_uint4(0, 0, 0, 0);
      } else {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          float* p = part + (2 * split + x) * one + part_row + (long long)r * a.D + d;
          reinterpret_cast<float4*>(p)[0] = reinterpret_cast<float4*>(p)[1] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
      }
    }
    return;
  }
  volatile uint32_t* misc = reinterpret_cast<volatile uint32_t*>(sm + Sm::misc);
  auto bar = [&](int i) -> uint32_t { return base + Sm::bars + 8u * i; };
  if (tid == 0) {
    mbar_init(bar(K_KV_FULL), 1);
    for (int i = 0; i < Sm::q_stages; ++i) {
      mbar_init(bar(K_Q_FULL + i), 33);       // the TMA boxes' lane and 32 lanes' copies of the statistics
      mbar_init(bar(K_Q_EMPTY + i), 1);
    }
    for (int i = 0; i < Sm::do_stages; ++i) {
      mbar_init(bar(K_DO_FULL + i), 1);
      mbar_init(bar(K_DO_EMPTY + i), 2);      // read by the dP products of one issuer and the dV products of the other
    }
    for (int i = 0; i < Sm::bufs; ++i) {
      mbar_init(bar(K_S_FULL + i), 1);
      mbar_init(bar(K_S_EMPTY + i), 1);
      mbar_init(bar(K_DP_FULL + i), 1);
      mbar_init(bar(K_DP_EMPTY + i), 1);
      mbar_init(bar(K_P_FULL + i), 4 * kDkGroups);
      mbar_init(bar(K_DS_FULL + i), 4 * kDkGroups);
    }
    mbar_init(bar(K_ACC_FULL), 1);
    fence_barrier_init();
    tma_prefetch_desc(&map_q);
    tma_prefetch_desc(&map_do);
    mbar_arrive_expect_tx(bar(K_KV_FULL), 2 * Sm::tile);
    load_rows<HD>(base + Sm::k, &map_k, krow0, hk, b, kHalf, bar(K_KV_FULL));
    load_rows<HD>(base + Sm::v, &map_v, krow0, hk, b, kHalf, bar(K_KV_FULL));
  }
  if (warp == 1) {
    tmem_alloc(base + Sm::misc, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = misc[0];
  // buffers of (S^T 64 columns, dP^T 64 columns), P^T and dS^T packed over them; then dK and dV
  const uint32_t tmem_dk = tmem + 128 * Sm::bufs, tmem_dv = tmem_dk + HD;
  static_assert(128 * Sm::bufs + 2 * HD <= (int)kTmemCols, "tensor memory of the dK/dV pass");
  bool ok = true;
  int e = 0;                                      // kRanged: dS is held as dS 2^e, P as P 2^kPShift
  if (kRanged<T> && (warp == 0 || warp >= 4)) {
    const float* bounds = a.bounds + (long long)bhk * VSA_CROSS_BOUNDS;      // 32 parts of max |v|^2, then max |do|^2
    e = range_exponent(warp_max(bounds[lane]) * bounds[VSA_CROSS_BOUNDS - 1]);
  }
  const float range = kRanged<T> ? power_of_two(e - kPShift) : 1.f;      // dP and delta take what P has not

  if (warp == 0) {       // dO tiles; Q tiles and the statistics of their rows
    int g = (int)(first / qtiles), qt = (int)(first - (long long)g * qtiles);
    float stats[4];                               // kRanged: of the tile to come, on their way through registers
    auto fetch = [&]() {
      const long long stat = ((long long)b * a.H + hk * group_heads + g) * lp + qt * kQTile + lane;
      stats[0] = a.lse2[stat];
      stats[1] = a.lse2[stat + 32];
      stats[2] = a.delta[stat];
      stats[3] = a.delta[stat + 32];
    };
    if (kRanged<T>) fetch();
    for (int p = 0; p < n_tiles; ++p) {
      const int sq = p % Sm::q_stages, sd = p % Sm::do_stages;
      const int h = hk * group_heads + g, row0 = qt * kQTile;
      ok = CROSS_WAIT(bar(K_Q_EMPTY + sq), ((p / Sm::q_stages) & 1) ^ 1) && CROSS_WAIT(bar(K_DO_EMPTY + sd), ((p / Sm::do_stages) & 1) ^ 1);
      if (!ok) break;
      if (kRanged<T>) {
        float* st = reinterpret_cast<float*>(sm + Sm::stats + sq * 512) + lane;
        st[0] = stats[0] - kPShift;
        st[32] = stats[1] - kPShift;
        st[64] = stats[2] * range;
        st[96] = stats[3] * range;
        mbar_arrive(bar(K_Q_FULL + sq));
      } else {
        const uint32_t st = base + Sm::stats + sq * 512 + lane * 4;
        const long long stat = ((long long)b * a.H + h) * lp + row0 + lane;
        cp_async4(st, a.lse2 + stat);
        cp_async4(st + 128, a.lse2 + stat + 32);
        cp_async4(st + 256, a.delta + stat);
        cp_async4(st + 384, a.delta + stat + 32);
        cp_async_arrive_noinc(bar(K_Q_FULL + sq));
      }
      if (lane == 0) {
        mbar_arrive_expect_tx(bar(K_Q_FULL + sq), Sm::part);
        load_rows<HD>(base + Sm::q + sq * Sm::part, &map_q, row0, h, b, kSlab, bar(K_Q_FULL + sq));
        mbar_arrive_expect_tx(bar(K_DO_FULL + sd), Sm::part);
        load_rows<HD>(base + Sm::d_o + sd * Sm::part, &map_do, row0, h, b, kSlab, bar(K_DO_FULL + sd));
      }
      if (++qt == qtiles) qt = 0, ++g;
      if (kRanged<T> && p + 1 < n_tiles) fetch();
    }
    if (!ok && lane == 0) atomicCAS(status, 0, 91);
  } else if (warp == 2) {
    // S^T = K Q^T
    ok = CROSS_WAIT(bar(K_KV_FULL), 0);
    for (int p = 0; p < n_tiles && ok; ++p) {
      const int s = p % Sm::q_stages, bf = p % Sm::bufs;
      ok = CROSS_WAIT(bar(K_Q_FULL + s), (p / Sm::q_stages) & 1) && CROSS_WAIT(bar(K_S_EMPTY + bf), ((p / Sm::bufs) & 1) ^ 1);
      if (!ok) break;
      tc_fence_after();
      if (elect_one()) {
        issue_scores<T, HD, 64, kSlab>(tmem + bf * 128, base + Sm::k, base + Sm::q + s * Sm::part);
        mma_commit(bar(K_S_FULL + bf));
      }
      __syncwarp();
    }
    if (!ok && lane == 0) atomicCAS(status, 0, 92);
  } else if (warp == 1) {
    // dP^T = V dO^T
    ok = CROSS_WAIT(bar(K_KV_FULL), 0);
    for (int p = 0; p < n_tiles && ok; ++p) {
      const int s = p % Sm::do_stages, bf = p % Sm::bufs;
      ok = CROSS_WAIT(bar(K_DO_FULL + s), (p / Sm::do_stages) & 1) && CROSS_WAIT(bar(K_DP_EMPTY + bf), ((p / Sm::bufs) & 1) ^ 1);
      if (!ok) break;
      tc_fence_after();
      if (elect_one()) {
        issue_scores<T, HD, 64, kSlab>(tmem + bf * 128 + 64, base + Sm::v, base + Sm::d_o + s * Sm::part);
        mma_commit(bar(K_DO_EMPTY + s));
        mma_commit(bar(K_DP_FULL + bf));
      }
      __syncwarp();
    }
    if (!ok && lane == 0) atomicCAS(status, 0, 93);
  } else if (warp == 3) {
    // dV += P^T dO, dK += dS^T Q
    for (int p = 0; p < n_tiles && ok; ++p) {
      const int sq = p % Sm::q_stages, sd = p % Sm::do_stages, bf = p % Sm::bufs;
      const uint32_t ph = (p / Sm::bufs) & 1;
      ok = CROSS_WAIT(bar(K_DO_FULL + sd), (p / Sm::do_stages) & 1) && CROSS_WAIT(bar(K_P_FULL + bf), ph);
      if (!ok) break;
      tc_fence_after();
      if (elect_one()) {
        issue_product<T, HD, 64, kDkCols, 64>(tmem_dv, tmem + bf * 128, base + Sm::d_o + sd * Sm::part, p > 0);
        mma_commit(bar(K_DO_EMPTY + sd));
        mma_commit(bar(K_S_EMPTY + bf));
      }
      __syncwarp();
      ok = CROSS_WAIT(bar(K_DS_FULL + bf), ph);
      if (!ok) break;
      tc_fence_after();
      if (elect_one()) {
        issue_product<T, HD, 64, kDkCols, 64>(tmem_dk, tmem + bf * 128 + 64, base + Sm::q + sq * Sm::part, p > 0);
        mma_commit(bar(K_Q_EMPTY + sq));
        mma_commit(bar(K_DP_EMPTY + bf));
      }
      __syncwarp();
    }
    if (ok && elect_one()) mma_commit(bar(K_ACC_FULL));
    __syncwarp();
    if (!ok && lane == 0) atomicCAS(status, 0, 94);
  } else {
    const int quarter = warp & 3, cg = (warp - 4) >> 2;
    const int row = quarter * 32 + lane, c0 = cg * kDkCols, st = tid - 128;
    const uint32_t lane_addr = (uint32_t)(quarter * 32) << 16;
    const bool live = row < live_keys;
    const float2 c2 = make_float2(-c, -c), m1 = make_float2(-1.f, -1.f), mf = make_float2(-range, -range);
    for (int p = 0; p < n_tiles && ok; ++p) {
      const int bf = p % Sm::bufs, sq = p % Sm::q_stages;
      const uint32_t ph = (p / Sm::bufs) & 1;
      ok = CROSS_WAIT(bar(K_S_FULL + bf), ph) && CROSS_WAIT(bar(K_Q_FULL + sq), (p / Sm::q_stages) & 1);
      if (!ok) break;
      tc_fence_after();
      const float4* s_lse = reinterpret_cast<const float4*>(sm + Sm::stats + sq * 512 + c0 * 4);
      const uint32_t s_addr = tmem + bf * 128 + lane_addr + c0;
      uint32_t sv[kDkCols];
      tmem_ld(s_addr, sv);
      tmem_ld_wait();
      float2 pf[kDkCols / 2];
      uint32_t pk[kDkCols / 2];
#pragma unroll
      for (int i = 0; i < kDkCols / 4; ++i) {
        const float4 l4 = s_lse[i];
        // lse - S c, negated in the exponential: the packed operations have no sign of their own to spend on the statistics
        const float2 x = fma2(word_pair(sv + 4 * i), c2, make_float2(l4.x, l4.y));
        const float2 y = fma2(word_pair(sv + 4 * i + 2), c2, make_float2(l4.z, l4.w));
        pf[2 * i] = kDkPoly<HD> > 2 * i % 8 ? poly_exp2<T>(mul2(x, m1)) : make_float2(fast_exp2(-x.x), fast_exp2(-x.y));
        pf[2 * i + 1] = kDkPoly<HD> > (2 * i + 1) % 8 ? poly_exp2<T>(mul2(y, m1)) : make_float2(fast_exp2(-y.x), fast_exp2(-y.y));
        // a key that takes no part: its scores come from whatever sits in K there
        pk[2 * i] = live ? pack_weights<T>(pf[2 * i].x, pf[2 * i].y) : 0u;
        pk[2 * i + 1] = live ? pack_weights<T>(pf[2 * i + 1].x, pf[2 * i + 1].y) : 0u;
      }
      tmem_st(s_addr, pk);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(K_P_FULL + bf));
      ok = CROSS_WAIT(bar(K_DP_FULL + bf), ph);
      if (!ok) break;
      tc_fence_after();
      uint32_t dvv[kDkCols];
      tmem_ld(s_addr + 64, dvv);
      tmem_ld_wait();
#pragma unroll
      for (int i = 0; i < kDkCols / 4; ++i) {
        const float4 d4 = s_lse[16 + i];       // delta: 64 floats behind the statistics
        const float2 x = mul2(pf[2 * i], fma2(word_pair(dvv + 4 * i), mf, make_float2(d4.x, d4.y)));      // -dS
        const float2 y = mul2(pf[2 * i + 1], fma2(word_pair(dvv + 4 * i + 2), mf, make_float2(d4.z, d4.w)));
        pk[2 * i] = live ? pack_weights<T>(x.x, x.y) : 0u;
        pk[2 * i + 1] = live ? pack_weights<T>(y.x, y.y) : 0u;
      }
      tmem_st(s_addr + 64, pk);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(K_DS_FULL + bf));
    }
    if (!ok && lane == 0) atomicCAS(status, 0, 95);
    if (ok) ok = CROSS_WAIT(bar(K_ACC_FULL), 0);
    uint8_t* stage_k = sm + Sm::k;            // every MMA is done: dK over K, dV over V
    uint8_t* stage_v = sm + Sm::v;
    if (ok) {
      tc_fence_after();
      for (int j = cg; j < 2 * (HD / 32); j += kDkGroups) {
        const bool is_k = j < HD / 32;
        const int jj = is_k ? j : j - HD / 32;
        uint32_t av[32];
        tmem_ld((is_k ? tmem_dk : tmem_dv) + lane_addr + 32 * jj, av);
        tmem_ld_wait();
        // the products summed -dS
        const float mul = is_k ? -a.scale * (kRanged<T> ? power_of_two(-e) : 1.f) : kRanged<T> ? power_of_two(-kPShift) : 1.f;
#pragma unroll
        for (int i = 0; i < 32; ++i) av[i] = live ? __float_as_uint(__uint_as_float(av[i]) * mul) : 0u;
        if (part == nullptr) {
#pragma unroll
          for (int q4 = 0; q4 < 4; ++q4)
            *reinterpret_cast<uint4*>((is_k ? stage_k : stage_v) + row * (HD * 2) + (((4 * jj + q4) ^ (row & 7)) << 4)) = pack8<T>(av + 8 * q4);
        } else if (krow0 + row < a.Lkv) {
          float* dst = part + (2 * split + !is_k) * one + part_row + (long long)row * a.D + 32 * jj;
#pragma unroll
          for (int i = 0; i < 32; i += 4)
            if (32 * jj + i < a.D) *reinterpret_cast<uint4*>(dst + i) = make_uint4(av[i], av[i + 1], av[i + 2], av[i + 3]);
        }
      }
    }
    if (part == nullptr) {
      named_barrier(1, kDkEwThreads);          // of every warp: one whose wait ran out must not leave the others in it
      for (int i = st; i < kRows * HD / 8 && ok; i += kDkEwThreads) {
        const int r = i / (HD / 8), ch = i % (HD / 8);
        if (krow0 + r >= a.Lkv || ch * 8 >= a.D) continue;
        const uint32_t off = r * (HD * 2) + ((ch ^ (r & 7)) << 4);
        *reinterpret_cast<uint4*>((T*)a.dk + b * a.dk_stride[0] + hk * a.dk_stride[1] + (krow0 + r) * a.dk_stride[2] + ch * 8) =
            *reinterpret_cast<const uint4*>(stage_k + off);
        *reinterpret_cast<uint4*>((T*)a.dv + b * a.dv_stride[0] + hk * a.dv_stride[1] + (krow0 + r) * a.dv_stride[2] + ch * 8) =
            *reinterpret_cast<const uint4*>(stage_v + off);
      }
    }
  }
  tc_fence_before();
  settle(ok);
  if (warp == 1) tmem_dealloc(tmem, kTmemCols);
}

// max |v|^2 of a key head's live keys in 32 parts, and a zero where dQ will put max |do|^2.  A row is D / 8 lanes of 16 bytes.
template <typename T, int LANES>
__global__ void __launch_bounds__(256) cross_bounds_kernel(const __grid_constant__ VsaCross a) {
  __shared__ unsigned top[8];
  constexpr int kParts = VSA_CROSS_BOUNDS - 1;
  const int piece = blockIdx.x, tid = threadIdx.x, lane = tid % LANES;
  for (long long bhk = blockIdx.y; bhk < a.B * a.Hkv; bhk += gridDim.y) {
    const int b = (int)(bhk / a.Hkv), hk = (int)(bhk - b * a.Hkv), len = cross_length(a, b);
    const int per = (len + kParts - 1) / kParts, r1 = (int)min((long long)len, (long long)per * (piece + 1));
    const T* v = (const T*)a.v + b * a.v_stride[0] + hk * a.v_stride[1] + lane * 8;
    unsigned most = 0;
    for (int r0 = piece * per; r0 < r1; r0 += 256 / LANES) {
      const int r = r0 + tid / LANES;
      float x = 0.f;
      if (r < r1 && lane * 8 < a.D) {
        const uint4 p = *reinterpret_cast<const uint4*>(v + r * a.v_stride[2]);
        const uint32_t* w = &p.x;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 f = Elem<T>::unpack(w[i]);
          x = fmaf(f.x, f.x, fmaf(f.y, f.y, x));
        }
      }
#pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
      most = max(most, __float_as_uint(x));        // non-negative numbers, NaN above them all
    }
    most = __reduce_max_sync(0xffffffffu, most);
    if ((tid & 31) == 0) top[tid >> 5] = most;
    __syncthreads();
    if (tid == 0) {
      for (int i = 1; i < 8; ++i) most = max(most, top[i]);
      float* to = a.bounds + bhk * VSA_CROSS_BOUNDS;
      to[piece] = __uint_as_float(most);
      if (piece == 0) to[kParts] = 0.f;
    }
    __syncthreads();
  }
}

// ---- host ------------------------------------------------------------------------------------------------------
// The kernels' shared memory, once per device: `ready` has a bit for each.
template <typename Kern>
int reserve(Kern kern, int bytes, const char* what, std::atomic<uint64_t>& ready) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  const uint64_t bit = 1ull << (dev & 63);
  if (e == cudaSuccess && dev < 64 && (ready.load(std::memory_order_relaxed) & bit)) return VSA_OK;
  if (e == cudaSuccess) e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return fail(VSA_ERR_LAUNCH, "%s: shared memory: %s", what, cudaGetErrorString(e));
  if (dev < 64) ready.fetch_or(bit, std::memory_order_relaxed);
  return VSA_OK;
}

int map_of(CUtensorMap* map, const VsaCross& a, const void* p, const int64_t (&stride)[3], int64_t heads, int64_t rows, int box, const char* what,
           int box_dims = 64) {
  return make_map_rows(map, a.dtype == VSA_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, p, a.D, rows, heads, a.B,
                       stride[2], stride[1], stride[0], box, what, box_dims);
}

template <typename T, int HD>
int launch_fwd(const VsaCross& a, int splits, float* part_out, float* part_lse, cudaStream_t st) {
  CUtensorMap mq, mk, mv, mo;
  int rc, *status;
  if ((rc = device_status_word(&status))) return rc;      // first: it binds the device's context to the thread
  if ((rc = map_of(&mq, a, a.q, a.q_stride, a.H, a.Lq, kRows, "cross attention forward (q)"))) return rc;
  if ((rc = map_of(&mk, a, a.k, a.k_stride, a.Hkv, a.Lkv, kRows, "cross attention forward (k)"))) return rc;
  if ((rc = map_of(&mv, a, a.v, a.v_stride, a.Hkv, a.Lkv, kRows, "cross attention forward (v)"))) return rc;
  if ((rc = map_of(&mo, a, a.out, a.out_stride, a.H, a.Lq, 32, "cross attention forward (out)"))) return rc;
  static std::atomic<uint64_t> ready{0};
  if ((rc = reserve(cross_fwd_umma_kernel<T, HD>, FwdSmem<HD>::total, "cross attention forward", ready))) return rc;
  const int64_t pairs = (a.Lq + 2 * kRows - 1) / (2 * kRows), items = a.B * a.H * pairs * splits;
  if (items > 0x3fffffff) return fail(VSA_ERR_UNSUPPORTED, "cross attention forward: too many query rows");
  const FwdWork w{Divisor((uint32_t)splits), Divisor((uint32_t)pairs), Divisor((uint32_t)a.H), Divisor((uint32_t)(a.H / a.Hkv)), (int)items, part_out, part_lse};
  const int64_t sms = device_sms();
  cross_fwd_umma_kernel<T, HD><<<(unsigned)(items < sms ? items : sms), kFwdThreads, FwdSmem<HD>::total, st>>>(mq, mk, mv, mo, a, w, status);
  return check_launch("cross_fwd_umma_kernel");
}

template <typename T, int HD>
int launch_bwd(const VsaCross& a, int splits, bool parts, float* part, cudaStream_t st) {
  CUtensorMap mq, mdo, mk, mv, mq64, mdo64, mdq;
  int rc, *status;
  if ((rc = device_status_word(&status))) return rc;      // first: it binds the device's context to the thread
  if ((rc = map_of(&mq, a, a.q, a.q_stride, a.H, a.Lq, kRows, "cross attention backward (q)"))) return rc;
  if ((rc = map_of(&mdo, a, a.dout, a.dout_stride, a.H, a.Lq, kRows, "cross attention backward (dout)"))) return rc;
  if ((rc = map_of(&mq64, a, a.q, a.q_stride, a.H, a.Lq, kQTile, "cross attention backward (q)"))) return rc;
  if ((rc = map_of(&mdo64, a, a.dout, a.dout_stride, a.H, a.Lq, kQTile, "cross attention backward (dout)"))) return rc;
  if ((rc = map_of(&mk, a, a.k, a.k_stride, a.Hkv, a.Lkv, kRows, "cross attention backward (k)"))) return rc;
  if ((rc = map_of(&mv, a, a.v, a.v_stride, a.Hkv, a.Lkv, kRows, "cross attention backward (v)"))) return rc;
  if ((rc = map_of(&mdq, a, a.dq, a.dq_stride, a.H, a.Lq, 32, "cross attention backward (dq)", 32))) return rc;
  static std::atomic<uint64_t> dq_ready{0}, dkdv_ready{0};
  if ((rc = reserve(cross_dq_umma_kernel<T, HD>, DqSmem<HD>::total, "cross attention dQ", dq_ready))) return rc;
  if ((rc = reserve(cross_dkdv_umma_kernel<T, HD>, DkSmem<HD>::total, "cross attention dK/dV", dkdv_ready))) return rc;
  const int64_t qtiles = (a.Lq + kRows - 1) / kRows, items = a.B * a.H * qtiles, ktiles = (a.Lkv + kRows - 1) / kRows;
  const int64_t units = a.B * a.Hkv * ktiles * splits;
  if (items > 0x3fffffff || units > 0x3fffffff) return fail(VSA_ERR_UNSUPPORTED, "cross attention backward: too many rows");
  if constexpr (kRanged<T>) {
    const int64_t heads = a.B * a.Hkv;
    cross_bounds_kernel<T, HD / 8><<<dim3(VSA_CROSS_BOUNDS - 1, (unsigned)(heads < 65535 ? heads : 65535)), 256, 0, st>>>(a);
    if ((rc = check_launch("cross_bounds_kernel"))) return rc;
  }
  const int64_t sms = device_sms();
  cross_dq_umma_kernel<T, HD><<<(unsigned)(items < sms ? items : sms), kDqThreads, DqSmem<HD>::total, st>>>(
      mq, mdo, mk, mv, mdq, a, Divisor((uint32_t)qtiles), Divisor((uint32_t)a.H), Divisor((uint32_t)(a.H / a.Hkv)), (int)items, status);
  if ((rc = check_launch("cross_dq_umma_kernel")) || a.dk == nullptr) return rc;
  cross_dkdv_umma_kernel<T, HD><<<(unsigned)units, kDkThreads, DkSmem<HD>::total, st>>>(mq64, mdo64, mk, mv, a, (int)ktiles, splits, parts ? part : nullptr, status);
  return check_launch("cross_dkdv_umma_kernel");
}

bool aligned(const void* p, const int64_t (&s)[3], int64_t heads, int64_t rows, int64_t batch) {
  const int64_t n[3] = {batch, heads, rows};
  if (reinterpret_cast<uintptr_t>(p) % 16) return false;
  for (int i = 0; i < 3; ++i)
    if (n[i] > 1 && (s[i] <= 0 || s[i] % 8 || s[i] >= (1LL << 38))) return false;
  return true;
}

}  // namespace

bool cross_umma_shape(int D, int dtype) { return (dtype == VSA_BF16 || dtype == VSA_F16) && D % 8 == 0 && D >= 8 && D <= 128; }

bool cross_umma_eligible(const VsaCross& a, bool backward) {
  return a.scale > 0.f && !(backward && a.Lkv > cross_umma_sum(a.dtype)) && cross_aligned(a, backward);
}

bool cross_aligned(const VsaCross& a, bool backward) {
  if (!cross_umma_shape(a.D, a.dtype) || a.Lkv < 1 || a.Lq < 1) return false;
  if (!aligned(a.q, a.q_stride, a.H, a.Lq, a.B) || !aligned(a.k, a.k_stride, a.Hkv, a.Lkv, a.B) || !aligned(a.v, a.v_stride, a.Hkv, a.Lkv, a.B) ||
      !aligned(a.out, a.out_stride, a.H, a.Lq, a.B))
    return false;
  return !backward || (aligned(a.dout, a.dout_stride, a.H, a.Lq, a.B) && aligned(a.dq, a.dq_stride, a.H, a.Lq, a.B) &&
                       (a.dk == nullptr || (aligned(a.dk, a.dk_stride, a.Hkv, a.Lkv, a.B) && aligned(a.dv, a.dv_stride, a.Hkv, a.Lkv, a.B))));
}

int cross_fwd_umma(const VsaCross& a, int splits, float* part_out, float* part_lse, cudaStream_t st) {
  if (a.dtype == VSA_F16)
    return a.D <= 64 ? launch_fwd<__half, 64>(a, splits, part_out, part_lse, st) : launch_fwd<__half, 128>(a, splits, part_out, part_lse, st);
  return a.D <= 64 ? launch_fwd<__nv_bfloat16, 64>(a, splits, part_out, part_lse, st)
                   : launch_fwd<__nv_bfloat16, 128>(a, splits, part_out, part_lse, st);
}

int cross_bwd_umma(const VsaCross& a, int splits, bool parts, float* part, cudaStream_t st) {
  if (a.dtype == VSA_F16) return a.D <= 64 ? launch_bwd<__half, 64>(a, splits, parts, part, st) : launch_bwd<__half, 128>(a, splits, parts, part, st);
  return a.D <= 64 ? launch_bwd<__nv_bfloat16, 64>(a, splits, parts, part, st) : launch_bwd<__nv_bfloat16, 128>(a, splits, parts, part, st);
}

}  // namespace vsa
