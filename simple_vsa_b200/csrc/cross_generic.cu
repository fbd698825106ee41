// Cross attention on CUDA cores: fp32, head dims up to 256 of any alignment, any strides.  Also the small kernels that both families of
// cross attention share: the packed key mask, the join of a forward split over the keys, the sum of partial dK and dV.
//
// out_i = sum_j p_ij v_j with p_i the softmax of scale q_i.k_j over the live keys j of the sample; a row without one gets zeros.
// Tiles of 128 query rows x 64 keys, 64 x 64 where there are few (64 x 64 and 32 x 32 above head dim 128; dK/dV up to 128 keys x 64 query
// rows), 256 threads, a patch of 8 x 4 scores each, everything in fp32 and one rounding at the end.  Bound by the FP32 pipe and the
// shared-memory reads that feed it (12 of 16 bytes for 128 multiply-adds in the scores, 16 for 256 in the products): at
// [1, 12, 4096, 128] x 2048 the forward takes 1433 us (36 of 72 TFLOP/s; pipe 62 % busy, reads 47 %), the backward 4475 (its seven products at
// 40; 65 and 67 %, 51 and 61 %).  8 x 8 scores a thread spill (4 % slower); chains without pairs are 11 % slower in the backward, two CTAs
// an SM at head dim 64 spill too (5 %).  With few query rows a pass is cut over the keys, with few keys dK/dV is over the query rows.
#include <atomic>

#include "common.cuh"
#include "kernels.h"

namespace vsa {
namespace {

constexpr int kThreads = 256;

template <typename T> __device__ __forceinline__ float to_f(T x) { return Elem<T>::to(x); }
template <> __device__ __forceinline__ float to_f<float>(float x) { return x; }
template <typename T> __device__ __forceinline__ T from_f(float x) { return Elem<T>::from(x); }
template <> __device__ __forceinline__ float from_f<float>(float x) { return x; }

// DP: head dim rounded up; RT, CT: rows and columns of a tile of scores, PI x PJ of them a thread; OVER: the scores go over a tile of
// operands that has been read
template <int DP_, int RT_, int CT_ = RT_, bool OVER_ = false>
struct Tile {
  static constexpr int DP = DP_, RT = RT_, CT = CT_, PI = RT / 16, PJ = CT / 16, PITCH = DP_ + 4, SPITCH = CT + 4;
  static constexpr int row_floats = RT * PITCH, col_floats = CT * PITCH, score_floats = RT * SPITCH;
  static constexpr bool OVER = OVER_;
};

// 16 bytes global -> shared past the registers, zeros where `there` is false (src is then not read)
__device__ __forceinline__ void copy16(float* dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((unsigned)__cvta_generic_to_shared(dst)), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }

// ROWS rows of one (batch, head) slice, converted, as one group of copies; rows that `live` says no to and dims from D on are zeros.
template <typename T, typename TL, int ROWS, typename LIVE>
__device__ __forceinline__ void load_tile(float* sm, const T* __restrict__ g, long long stride, int D, bool vec, LIVE live) {
  constexpr int C = TL::DP / 4, N = ROWS * C / kThreads;
  static_assert(ROWS * C % kThreads == 0, "whole pieces a thread");
  if (sizeof(T) == 4 && vec) {
#pragma unroll 4
    for (int i = 0; i < N; ++i) {
      const int e = threadIdx.x + i * kThreads, r = e / C, c = (e % C) * 4;
      const bool there = live(r) && c < D;
      copy16(sm + r * TL::PITCH + c, there ? g + r * stride + c : g, there);
    }
  } else {
    constexpr int U = N % 4 == 0 ? 4 : 2;        // pieces whose loads fly together
    static_assert(N % U == 0, "whole batches of pieces");
#pragma unroll 1
    for (int i = 0; i < N; i += U) {
      float4 x[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int e = threadIdx.x + (i + u) * kThreads, r = e / C, c = (e % C) * 4;
        x[u] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (live(r) && c < D) {
          const T* p = g + r * stride + c;
          x[u].x = to_f<T>(p[0]);
          if (c + 1 < D) x[u].y = to_f<T>(p[1]);
          if (c + 2 < D) x[u].z = to_f<T>(p[2]);
          if (c + 3 < D) x[u].w = to_f<T>(p[3]);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int e = threadIdx.x + (i + u) * kThreads;
        *reinterpret_cast<float4*>(sm + e / C * TL::PITCH + (e % C) * 4) = x[u];
      }
    }
  }
  copies_commit();
}

// s[i][j] = a[PI ty + i] . b[tx + 16 j], even and odd dims in two chains that one instruction advances
template <typename TL>
__device__ __forceinline__ void scores(float (&s)[TL::PI][TL::PJ], const float* a, const float* b, int tx, int ty) {
  float2 t[TL::PI][TL::PJ];
#pragma unroll
  for (int i = 0; i < TL::PI; ++i)
#pragma unroll
    for (int j = 0; j < TL::PJ; ++j) t[i][j] = make_float2(0.f, 0.f);
#pragma unroll 2
  for (int d = 0; d < TL::DP; d += 4) {
    float4 y[TL::PJ];
#pragma unroll
    for (int j = 0; j < TL::PJ; ++j) y[j] = *reinterpret_cast<const float4*>(b + (tx + 16 * j) * TL::PITCH + d);
#pragma unroll
    for (int i = 0; i < TL::PI; ++i) {
      const float4 x = *reinterpret_cast<const float4*>(a + (TL::PI * ty + i) * TL::PITCH + d);
#pragma unroll
      for (int j = 0; j < TL::PJ; ++j)
        t[i][j] = fma2(make_float2(x.z, x.w), make_float2(y[j].z, y[j].w), fma2(make_float2(x.x, x.y), make_float2(y[j].x, y[j].y), t[i][j]));
    }
  }
#pragma unroll
  for (int i = 0; i < TL::PI; ++i)
#pragma unroll
    for (int j = 0; j < TL::PJ; ++j) s[i][j] = t[i][j].x + t[i][j].y;
}

// acc[i][2 h + f] += sum_n p[PI ty + i][n] * b[n][64 h + 4 tx + 2 f ..]
template <typename TL>
__device__ __forceinline__ void product(float2 (&acc)[TL::PI][TL::DP / 32], const float* p, const float* b, int tx, int ty) {
#pragma unroll 1
  for (int n = 0; n < TL::CT; n += 4) {
    float4 w[TL::PI];
#pragma unroll
    for (int i = 0; i < TL::PI; ++i) w[i] = *reinterpret_cast<const float4*>(p + (TL::PI * ty + i) * TL::SPITCH + n);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float4 x[TL::DP / 64];
#pragma unroll
      for (int h = 0; h < TL::DP / 64; ++h) x[h] = *reinterpret_cast<const float4*>(b + (n + e) * TL::PITCH + 64 * h + 4 * tx);
#pragma unroll
      for (int i = 0; i < TL::PI; ++i) {
        const float f = e == 0 ? w[i].x : e == 1 ? w[i].y : e == 2 ? w[i].z : w[i].w;
        const float2 f2 = make_float2(f, f);
#pragma unroll
        for (int h = 0; h < TL::DP / 64; ++h) {
          acc[i][2 * h] = fma2(f2, make_float2(x[h].x, x[h].y), acc[i][2 * h]);
          acc[i][2 * h + 1] = fma2(f2, make_float2(x[h].z, x[h].w), acc[i][2 * h + 1]);
        }
      }
    }
  }
}

template <typename T, typename TL>
__device__ __forceinline__ void store_rows(T* __restrict__ g, long long stride, int D, int rows, const float2 (&acc)[TL::PI][TL::DP / 32],
                                           const float (&mul)[TL::PI], int tx, int ty) {
#pragma unroll
  for (int i = 0; i < TL::PI; ++i) {
    const int r = TL::PI * ty + i;
    if (r >= rows) continue;
#pragma unroll
    for (int h = 0; h < TL::DP / 64; ++h)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = 64 * h + 4 * tx + e;
        const float2 x = acc[i][2 * h + e / 2];
        if (d < D) g[r * stride + d] = from_f<T>(mul[i] == 0.f ? 0.f : (e & 1 ? x.y : x.x) * mul[i]);
      }
  }
}

__device__ __forceinline__ float lanes16_max(float x) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
  return x;
}
__device__ __forceinline__ float lanes16_sum(float x) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

struct Ctx {                   // what a CTA knows about its sample's keys
  int len;
  const uint32_t* bits;
  __device__ __forceinline__ bool live(int key) const { return key < len && (bits == nullptr || (bits[key >> 5] >> (key & 31) & 1u)); }
};
__device__ __forceinline__ Ctx keys_of(const VsaCross& a, int b) {
  Ctx c;
  c.len = cross_length(a, b);
  c.bits = a.key_bits == nullptr ? nullptr : a.key_bits + (long long)b * cross_words(a.Lkv);
  return c;
}

template <typename T> __device__ __forceinline__ const T* slice(const void* p, const int64_t (&st)[3], int b, int h) {
  return (const T*)p + b * st[0] + h * st[1];
}
template <typename T> __device__ __forceinline__ T* slice(void* p, const int64_t (&st)[3], int b, int h) {
  return (T*)p + b * st[0] + h * st[1];
}

// ---- forward: one tile of query rows, one range of key tiles ----------------------------------------------------
template <typename T, typename TL>
__global__ void __launch_bounds__(kThreads) cross_fwd_generic_kernel(const __grid_constant__ VsaCross a, int splits, float* part_out, float* part_lse,
                                                                     bool vec) {
  extern __shared__ __align__(16) float sm[];
  float *sq = sm, *sk = sq + TL::row_floats, *sv = sk + TL::col_floats, *ss = sv + TL::col_floats;
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const int split = blockIdx.x % splits, qt = blockIdx.x / splits, h = blockIdx.y, b = blockIdx.z, hk = h / (int)(a.H / a.Hkv);
  const int row0 = qt * TL::RT, rows = (int)min((long long)TL::RT, (long long)a.Lq - row0);
  const Ctx keys = keys_of(a, b);
  const int tiles = (keys.len + TL::CT - 1) / TL::CT, per = (tiles + splits - 1) / splits;
  const int t0 = split * per, t1 = min(tiles, t0 + per);
  const float c = a.scale * kLog2e;
  load_tile<T, TL, TL::RT>(sq, slice<T>(a.q, a.q_stride, b, h) + row0 * a.q_stride[2], a.q_stride[2], a.D, vec, [&](int r) { return r < rows; });
  float m[TL::PI], l[TL::PI];
  float2 acc[TL::PI][TL::DP / 32];
#pragma unroll
  for (int i = 0; i < TL::PI; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int d = 0; d < TL::DP / 32; ++d) acc[i][d] = make_float2(0.f, 0.f);
  }
  for (int t = t0; t < t1; ++t) {
    const int k0 = t * TL::CT;
    __syncthreads();
    auto live = [&](int r) { return keys.live(k0 + r); };
    load_tile<T, TL, TL::CT>(sk, slice<T>(a.k, a.k_stride, b, hk) + k0 * a.k_stride[2], a.k_stride[2], a.D, vec, live);
    load_tile<T, TL, TL::CT>(sv, slice<T>(a.v, a.v_stride, b, hk) + k0 * a.v_stride[2], a.v_stride[2], a.D, vec, live);
    copies_wait<1>();                              // Q and K; V may be on its way
    __syncthreads();
    float s[TL::PI][TL::PJ];
    scores<TL>(s, sq, sk, tx, ty);
    bool on[TL::PJ];
#pragma unroll
    for (int j = 0; j < TL::PJ; ++j) on[j] = live(tx + 16 * j);
#pragma unroll
    for (int i = 0; i < TL::PI; ++i) {
      float top = -INFINITY;
#pragma unroll
      for (int j = 0; j < TL::PJ; ++j)
        if (on[j]) top = fmaxf(top, s[i][j] * c);
      const float mn = fmaxf(m[i], lanes16_max(top)), shift = mn == -INFINITY ? 0.f : mn;
      const float keep = exp2f(m[i] - shift);
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < TL::PJ; ++j) {
        const float p = on[j] ? exp2f(fmaf(s[i][j], c, -shift)) : 0.f;
        sum += p;
        ss[(TL::PI * ty + i) * TL::SPITCH + tx + 16 * j] = p;
      }
      l[i] = l[i] * keep + lanes16_sum(sum);
      m[i] = mn;
#pragma unroll
      for (int d = 0; d < TL::DP / 32; ++d) acc[i][d] = mul2(acc[i][d], make_float2(keep, keep));
    }
    copies_wait<0>();
    __syncthreads();
    product<TL>(acc, ss, sv, tx, ty);
  }
  copies_wait<0>();
  float mul[TL::PI];
#pragma unroll
  for (int i = 0; i < TL::PI; ++i) mul[i] = l[i] == 0.f ? 0.f : 1.f / l[i];
  const long long bh = (long long)b * a.H + h, lp = cross_rows(a.Lq);
  if (splits == 1) {
    store_rows<T, TL>(slice<T>(a.out, a.out_stride, b, h) + row0 * a.out_stride[2], a.out_stride[2], a.D, rows, acc, mul, tx, ty);
  } else {
    const long long at = (split * (long long)a.B * a.H + bh) * a.Lq + row0;
    store_rows<float, TL>(part_out + at * a.D, a.D, a.D, rows, acc, mul, tx, ty);
  }
  if (tx == 0) {
#pragma unroll
    for (int i = 0; i < TL::PI; ++i) {
      const int r = TL::PI * ty + i;
      const float lse = l[i] == 0.f ? (splits == 1 ? INFINITY : -INFINITY) : m[i] + log2f(l[i]);
      if (splits > 1) {
        if (r < rows) part_lse[(split * (long long)a.B * a.H + bh) * a.Lq + row0 + r] = lse;
      } else if (row0 + r < lp) {
        a.lse2[bh * lp + row0 + r] = r < rows ? lse : INFINITY;
      }
    }
  }
  if (splits == 1 && row0 + TL::RT >= a.Lq)
    for (long long r = row0 + TL::RT + tid; r < lp; r += kThreads) a.lse2[bh * lp + r] = INFINITY;
}

// ---- backward: dQ (and delta) of one tile of query rows, one range of key tiles -----------------------------------------------------------
template <typename T, typename TL>
__global__ void __launch_bounds__(kThreads) cross_dq_generic_kernel(const __grid_constant__ VsaCross a, int splits, float* part, bool vec) {
  extern __shared__ __align__(16) float sm[];
  float *sq = sm, *sdo = sq + TL::row_floats, *sk = sdo + TL::row_floats, *sv = sk + TL::col_floats, *ss = TL::OVER ? sv : sv + TL::col_floats;
  static_assert(TL::RT <= 2 * TL::CT, "the rows of out pass through the tiles of K and V");
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const int split = blockIdx.x % splits, qt = blockIdx.x / splits, h = blockIdx.y, b = blockIdx.z, hk = h / (int)(a.H / a.Hkv);
  const int row0 = qt * TL::RT, rows = (int)min((long long)TL::RT, (long long)a.Lq - row0);
  const Ctx keys = keys_of(a, b);
  const int tiles = (keys.len + TL::CT - 1) / TL::CT, per = (tiles + splits - 1) / splits, t1 = min(tiles, (split + 1) * per);
  const float c = a.scale * kLog2e;
  const long long bh = (long long)b * a.H + h, lp = cross_rows(a.Lq);
  auto there = [&](int r) { return r < rows; };
  load_tile<T, TL, TL::RT>(sk, slice<T>((const void*)a.out, a.out_stride, b, h) + row0 * a.out_stride[2], a.out_stride[2], a.D, vec, there);
  load_tile<T, TL, TL::RT>(sq, slice<T>(a.q, a.q_stride, b, h) + row0 * a.q_stride[2], a.q_stride[2], a.D, vec, there);
  load_tile<T, TL, TL::RT>(sdo, slice<T>(a.dout, a.dout_stride, b, h) + row0 * a.dout_stride[2], a.dout_stride[2], a.D, vec, there);
  copies_wait<0>();
  __syncthreads();
  float lse[TL::PI], delta[TL::PI], mul[TL::PI];
  float2 acc[TL::PI][TL::DP / 32];
#pragma unroll
  for (int i = 0; i < TL::PI; ++i) {
    const int r = TL::PI * ty + i;
    float d = 0.f;
    for (int e = tx; e < TL::DP; e += 16) d = fmaf(sk[r * TL::PITCH + e], sdo[r * TL::PITCH + e], d);
    delta[i] = lanes16_sum(d);
    lse[i] = row0 + r < lp ? a.lse2[bh * lp + row0 + r] : INFINITY;
    if (tx == 0 && split == 0 && row0 + r < lp) a.delta[bh * lp + row0 + r] = r < rows ? delta[i] : 0.f;
    mul[i] = a.scale;
#pragma unroll
    for (int e = 0; e < TL::DP / 32; ++e) acc[i][e] = make_float2(0.f, 0.f);
  }
  for (int t = split * per; t < t1; ++t) {
    const int k0 = t * TL::CT;
    __syncthreads();
    auto live = [&](int r) { return keys.live(k0 + r); };
    load_tile<T, TL, TL::CT>(sk, slice<T>(a.k, a.k_stride, b, hk) + k0 * a.k_stride[2], a.k_stride[2], a.D, vec, live);
    load_tile<T, TL, TL::CT>(sv, slice<T>(a.v, a.v_stride, b, hk) + k0 * a.v_stride[2], a.v_stride[2], a.D, vec, live);
    copies_wait<1>();                              // K; V may be on its way
    __syncthreads();
    float s[TL::PI][TL::PJ], dp[TL::PI][TL::PJ];
    scores<TL>(s, sq, sk, tx, ty);
    copies_wait<0>();
    __syncthreads();
    scores<TL>(dp, sdo, sv, tx, ty);
    if (TL::OVER) __syncthreads();
#pragma unroll
    for (int j = 0; j < TL::PJ; ++j) {
      const bool on = live(tx + 16 * j);
#pragma unroll
      for (int i = 0; i < TL::PI; ++i)
        ss[(TL::PI * ty + i) * TL::SPITCH + tx + 16 * j] = on ? exp2f(fmaf(s[i][j], c, -lse[i])) * (dp[i][j] - delta[i]) : 0.f;
    }
    __syncthreads();
    product<TL>(acc, ss, sk, tx, ty);
  }
  if (split == 0 && row0 + TL::RT >= a.Lq)
    for (long long r = row0 + TL::RT + tid; r < lp; r += kThreads) a.delta[bh * lp + r] = 0.f;
  if (splits > 1) {
    store_rows<float, TL>(part + ((split * (long long)a.B * a.H + bh) * a.Lq + row0) * a.D, a.D, a.D, rows, acc, mul, tx, ty);
    return;
  }
  store_rows<T, TL>(slice<T>(a.dq, a.dq_stride, b, h) + row0 * a.dq_stride[2], a.dq_stride[2], a.D, rows, acc, mul, tx, ty);
}

// The parts of dQ, added in the order of the splits.
template <typename T>
__global__ void __launch_bounds__(256) cross_dq_sum_kernel(const __grid_constant__ VsaCross a, int splits, const float* __restrict__ part) {
  const long long one = (long long)a.B * a.H * a.Lq * a.D, at = (long long)blockIdx.x * 256 + threadIdx.x;
  if (at >= one) return;
  const long long row = at / a.D, bh = row / a.Lq, b = bh / a.H;
  float x = 0.f;
#pragma unroll 4
  for (int s = 0; s < splits; ++s) x += part[s * one + at];
  ((T*)a.dq)[b * a.dq_stride[0] + (bh - b * a.H) * a.dq_stride[1] + (row - bh * a.Lq) * a.dq_stride[2] + (at - row * a.D)] = from_f<T>(x);
}

// ---- backward: dK, dV of one tile of keys, one range of the query tiles of all heads that share them ------------------
template <typename T, typename TL>
__global__ void __launch_bounds__(kThreads) cross_dkdv_generic_kernel(const __grid_constant__ VsaCross a, int splits, float* part, bool vec) {
  extern __shared__ __align__(16) float sm[];
  float *sk = sm, *sv = sk + TL::row_floats, *sq = sv + TL::row_floats, *sdo = sq + TL::col_floats, *sp = sdo + TL::col_floats;
  float* sds = TL::OVER ? sp : sp + TL::score_floats;      // dS after P, or beside it
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const int split = blockIdx.x % splits, kt = blockIdx.x / splits, hk = blockIdx.y, b = blockIdx.z, group = (int)(a.H / a.Hkv);
  const int k0 = kt * TL::RT, krows = (int)min((long long)TL::RT, (long long)a.Lkv - k0);
  const Ctx keys = keys_of(a, b);
  const float c = a.scale * kLog2e;
  auto live = [&](int r) { return keys.live(k0 + r); };
  load_tile<T, TL, TL::RT>(sk, slice<T>(a.k, a.k_stride, b, hk) + k0 * a.k_stride[2], a.k_stride[2], a.D, vec, live);
  load_tile<T, TL, TL::RT>(sv, slice<T>(a.v, a.v_stride, b, hk) + k0 * a.v_stride[2], a.v_stride[2], a.D, vec, live);
  float2 dk[TL::PI][TL::DP / 32], dv[TL::PI][TL::DP / 32];
  float mul_k[TL::PI], mul_v[TL::PI];
#pragma unroll
  for (int i = 0; i < TL::PI; ++i) {
    const bool on = live(TL::PI * ty + i);
    mul_k[i] = on ? a.scale : 0.f;
    mul_v[i] = on ? 1.f : 0.f;
#pragma unroll
    for (int e = 0; e < TL::DP / 32; ++e) dk[i][e] = dv[i][e] = make_float2(0.f, 0.f);
  }
  const int qtiles = (int)((a.Lq + TL::CT - 1) / TL::CT);
  const long long total = (long long)qtiles * group, per = (total + splits - 1) / splits;
  const long long t1 = k0 < keys.len ? min(total, (split + 1) * per) : 0, lp = cross_rows(a.Lq);
  for (long long t = split * per; t < t1; ++t) {
    const int h = hk * group + (int)(t / qtiles), row0 = (int)(t % qtiles) * TL::CT;
    const int rows = (int)min((long long)TL::CT, (long long)a.Lq - row0);
    const long long stat = ((long long)b * a.H + h) * lp + row0;
    auto there = [&](int r) { return r < rows; };
    __syncthreads();
    load_tile<T, TL, TL::CT>(sq, slice<T>(a.q, a.q_stride, b, h) + row0 * a.q_stride[2], a.q_stride[2], a.D, vec, there);
    load_tile<T, TL, TL::CT>(sdo, slice<T>(a.dout, a.dout_stride, b, h) + row0 * a.dout_stride[2], a.dout_stride[2], a.D, vec, there);
    float lse[TL::PJ], delta[TL::PJ];
#pragma unroll
    for (int j = 0; j < TL::PJ; ++j) {
      const int r = tx + 16 * j;
      lse[j] = there(r) ? a.lse2[stat + r] : INFINITY;
      delta[j] = there(r) ? a.delta[stat + r] : 0.f;
    }
    copies_wait<1>();                              // K, V and Q; dO may be on its way
    __syncthreads();
    float s[TL::PI][TL::PJ], dp[TL::PI][TL::PJ];
    scores<TL>(s, sk, sq, tx, ty);
    copies_wait<0>();
    __syncthreads();
    scores<TL>(dp, sv, sdo, tx, ty);
#pragma unroll
    for (int j = 0; j < TL::PJ; ++j)
#pragma unroll
      for (int i = 0; i < TL::PI; ++i) {
        const int at = (TL::PI * ty + i) * TL::SPITCH + tx + 16 * j;
        const float p = exp2f(fmaf(s[i][j], c, -lse[j]));
        sp[at] = p;
        s[i][j] = p * (dp[i][j] - delta[j]);
        if (!TL::OVER) sds[at] = s[i][j];
      }
    __syncthreads();
    product<TL>(dv, sp, sdo, tx, ty);
    if (TL::OVER) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < TL::PJ; ++j)
#pragma unroll
        for (int i = 0; i < TL::PI; ++i) sds[(TL::PI * ty + i) * TL::SPITCH + tx + 16 * j] = s[i][j];
      __syncthreads();
    }
    product<TL>(dk, sds, sq, tx, ty);
  }
  copies_wait<0>();
  if (splits == 1) {
    store_rows<T, TL>(slice<T>(a.dk, a.dk_stride, b, hk) + k0 * a.dk_stride[2], a.dk_stride[2], a.D, krows, dk, mul_k, tx, ty);
    store_rows<T, TL>(slice<T>(a.dv, a.dv_stride, b, hk) + k0 * a.dv_stride[2], a.dv_stride[2], a.D, krows, dv, mul_v, tx, ty);
  } else {
    const long long one = (long long)a.B * a.Hkv * a.Lkv * a.D, at = (((long long)b * a.Hkv + hk) * a.Lkv + k0) * a.D;
    store_rows<float, TL>(part + (2 * split) * one + at, a.D, a.D, krows, dk, mul_k, tx, ty);
    store_rows<float, TL>(part + (2 * split + 1) * one + at, a.D, a.D, krows, dv, mul_v, tx, ty);
  }
}

// ---- shared: joins and the key mask ------------------------------------------------------------------------------------
// One warp per query row: the parts' weights are 2^(lse - max), their outputs already normalised.
template <typename T>
__global__ void __launch_bounds__(256) cross_join_kernel(const __grid_constant__ VsaCross a, int splits, const float* __restrict__ part_out,
                                                         const float* __restrict__ part_lse) {
  const long long rows = (long long)a.B * a.H * a.Lq, row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5), lp = cross_rows(a.Lq);
  const int lane = threadIdx.x & 31;
  if (row < rows) {
    const long long bh = row / a.Lq, l = row - bh * a.Lq;
    float top = -INFINITY;
    for (int s = lane; s < splits; s += 32) top = fmaxf(top, part_lse[s * rows + row]);
    top = warp_max(top);
    float sum = 0.f;
    for (int s = lane; s < splits; s += 32) sum += top == -INFINITY ? 0.f : exp2f(part_lse[s * rows + row] - top);
    sum = warp_sum(sum);
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    T* out = (T*)a.out + (bh / a.H) * a.out_stride[0] + (bh % a.H) * a.out_stride[1] + l * a.out_stride[2];
    for (int d = lane; d < a.D; d += 32) {
      float x = 0.f;
      for (int s = 0; s < splits; ++s) {
        const float ls = part_lse[s * rows + row];
        // a part without a live key holds zeros; its weight is zero too
        x = fmaf(top == -INFINITY ? 0.f : exp2f(ls - top), part_out[(s * rows + row) * a.D + d], x);
      }
      out[d] = from_f<T>(x * inv);
    }
    if (lane == 0) a.lse2[bh * lp + l] = top == -INFINITY ? INFINITY : top + log2f(sum);
  }
  // the padding behind each slice's rows, which the backward reads
  const long long pad = lp - a.Lq, pads = (long long)a.B * a.H * pad, at = (long long)blockIdx.x * 256 + threadIdx.x;
  const long long step = (long long)gridDim.x * 256;
  for (long long i = at; i < pads; i += step) a.lse2[(i / pad) * lp + a.Lq + i % pad] = INFINITY;
}

__global__ void __launch_bounds__(256) cross_bits_kernel(const uint8_t* __restrict__ mask, long long stride, const int32_t* __restrict__ lengths,
                                                         uint32_t* __restrict__ bits, long long Lkv, long long words) {
  const int b = blockIdx.y;
  const long long w = (long long)blockIdx.x * 8 + (threadIdx.x >> 5), key = w * 32 + (threadIdx.x & 31);
  if (w >= words) return;
  long long len = Lkv;
  if (lengths != nullptr) len = min(len, (long long)max(0, lengths[b]));
  const unsigned word = __ballot_sync(0xffffffffu, key < len && mask[b * stride + key] != 0);
  if ((threadIdx.x & 31) == 0) bits[b * words + w] = word;
}

// ---- compacted keys ---------------------------------------------------------------------------------------------------------
// The tensor path knows lengths only: with a mask, the rows of K and V that take part are gathered into dense tensors first (a few MB,
// once per call, against a select per score and the clearing of rows of V in every tile: forward 135 us at [2, 12 + 4, 8190, 64] x
// 1001 keys, 78 with them compacted), in their order; their gradients go back the same way when the parts are added.
// prefix [B][words]: live keys of the sample before each word; counts [B].
__global__ void __launch_bounds__(1024) cross_rank_kernel(const uint32_t* __restrict__ bits, int words, int32_t* __restrict__ prefix,
                                                          int32_t* __restrict__ counts) {
  __shared__ int warp_sums[32];
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int before = 0;
  for (int w0 = 0; w0 < words; w0 += 1024) {
    const int n = w0 + tid < words ? __popc(bits[(long long)b * words + w0 + tid]) : 0;
    int x = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) warp_sums[warp] = x;
    __syncthreads();
    if (warp == 0) {
      int s = warp_sums[lane];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += y;
      }
      warp_sums[lane] = s;
    }
    __syncthreads();
    if (w0 + tid < words) prefix[(long long)b * words + w0 + tid] = before + x - n + (warp ? warp_sums[warp - 1] : 0);
    before += warp_sums[31];
    __syncthreads();
  }
  if (tid == 0) counts[b] = before;
}

// The place of key l among the live ones of its sample, or -1.
__device__ __forceinline__ int rank_of(const uint32_t* bits, const int32_t* prefix, long long b, int words, int l) {
  const long long w = b * words + (l >> 5);
  const uint32_t word = bits[w], bit = 1u << (l & 31);
  return word & bit ? prefix[w] + __popc(word & (bit - 1u)) : -1;
}

// One 16-byte piece of a row a thread: K and V rows to their places, zeros behind the last one.
__global__ void __launch_bounds__(256) cross_compact_kernel(const __grid_constant__ VsaCross a, const int32_t* __restrict__ prefix,
                                                            const int32_t* __restrict__ counts, uint4* __restrict__ k_out, uint4* __restrict__ v_out) {
  const unsigned per_row = (unsigned)(a.D / 8), rows = (unsigned)(a.B * a.Hkv * a.Lkv);
  const unsigned row = blockIdx.x * blockDim.y + threadIdx.y;
  if (row >= rows) return;
  const unsigned bh = row / (unsigned)a.Lkv, b = bh / (unsigned)a.Hkv, h = bh - b * (unsigned)a.Hkv;
  const int l = (int)(row - bh * (unsigned)a.Lkv), words = (int)cross_words(a.Lkv);
  const int to = rank_of(a.key_bits, prefix, b, words, l);
  const bool behind = l >= counts[b];
  const __half* k = (const __half*)a.k + b * a.k_stride[0] + h * a.k_stride[1] + l * a.k_stride[2];      // any 16-bit type
  const __half* v = (const __half*)a.v + b * a.v_stride[0] + h * a.v_stride[1] + l * a.v_stride[2];
  for (unsigned c = threadIdx.x; c < per_row; c += blockDim.x) {
    const size_t at = (size_t)bh * a.Lkv;
    if (to >= 0) {
      k_out[(at + to) * per_row + c] = reinterpret_cast<const uint4*>(k)[c];
      v_out[(at + to) * per_row + c] = reinterpret_cast<const uint4*>(v)[c];
    }
    if (behind) k_out[(at + l) * per_row + c] = v_out[(at + l) * per_row + c] = make_uint4(0, 0, 0, 0);
  }
}

// dK and dV: the parts are added in the order of the splits, whatever ran first.  A thread owns W neighbouring dims of a key row; the
// loads of eight parts fly together (bound by their latency: a few MB).  With `prefix` the parts' rows are those of the compacted keys.
template <typename T, int W>
__global__ void __launch_bounds__(256) cross_sum_kernel(const __grid_constant__ VsaCross a, int splits, const float* __restrict__ part,
                                                        const int32_t* __restrict__ prefix) {
  struct alignas(4 * W) Floats { float v[W]; };
  struct alignas(W * sizeof(T)) Values { T v[W]; };
  const long long one = (long long)a.B * a.Hkv * a.Lkv * a.D;
  const unsigned per_row = (unsigned)(a.D / W), rows = (unsigned)(a.B * a.Hkv * a.Lkv);
  const unsigned row = blockIdx.x * blockDim.y + threadIdx.y, is_v = blockIdx.y;
  if (row >= rows) return;
  const unsigned bh = row / (unsigned)a.Lkv, l = row - bh * (unsigned)a.Lkv, b = bh / (unsigned)a.Hkv;
  const int64_t(&st)[3] = is_v ? a.dv_stride : a.dk_stride;
  const int from = prefix == nullptr ? (int)l : rank_of(a.key_bits, prefix, b, (int)cross_words(a.Lkv), (int)l);
  if (from < 0) splits = 0;            // a key that takes no part
  T* out = (T*)(is_v ? a.dv : a.dk) + b * st[0] + (bh - b * (unsigned)a.Hkv) * st[1] + l * st[2];
  for (unsigned c = threadIdx.x; c < per_row; c += blockDim.x) {
    const float* p = part + is_v * one + ((long long)bh * a.Lkv + from) * a.D + c * W;
    float sum[W] = {};
    for (int s = 0; s < splits; s += 8) {
      Floats x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (s + i < splits) x[i] = *reinterpret_cast<const Floats*>(p + 2 * (s + i) * one);
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < W; ++j)
          if (s + i < splits) sum[j] += x[i].v[j];
    }
    Values y;
#pragma unroll
    for (int j = 0; j < W; ++j) y.v[j] = from_f<T>(sum[j]);
    *reinterpret_cast<Values*>(out + c * W) = y;
  }
}

bool vec4(const VsaCross& a, bool backward) {      // 16-byte reads of fp32 rows
  if (a.dtype != VSA_F32 || a.D % 4) return false;
  auto fine = [](const void* p, const int64_t (&s)[3]) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && s[0] % 4 == 0 && s[1] % 4 == 0 && s[2] % 4 == 0;
  };
  return fine(a.q, a.q_stride) && fine(a.k, a.k_stride) && fine(a.v, a.v_stride) &&
         (!backward || (fine(a.out, a.out_stride) && fine(a.dout, a.dout_stride)));
}

// The kernel's shared memory, once per device: `ready` has a bit for each.
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

template <typename T, typename TL>
int fwd(const VsaCross& a, int splits, float* part_out, float* part_lse, cudaStream_t st) {
  const int bytes = (TL::row_floats + 2 * TL::col_floats + TL::score_floats) * 4;
  static std::atomic<uint64_t> ready{0};
  int rc = reserve(cross_fwd_generic_kernel<T, TL>, bytes, "cross attention forward", ready);
  if (rc) return rc;
  const int64_t tiles = (a.Lq + TL::RT - 1) / TL::RT;
  cross_fwd_generic_kernel<T, TL><<<dim3((unsigned)(tiles * splits), (unsigned)a.H, (unsigned)a.B), kThreads, bytes, st>>>(
      a, splits, part_out, part_lse, vec4(a, false));
  return check_launch("cross_fwd_generic_kernel");
}
template <typename T, typename TL>
int dq_pass(const VsaCross& a, int splits, float* part, cudaStream_t st) {
  constexpr int last = TL::OVER ? (TL::score_floats > TL::col_floats ? TL::score_floats : TL::col_floats) : TL::col_floats + TL::score_floats;
  const int bytes = (2 * TL::row_floats + TL::col_floats + last) * 4;
  static std::atomic<uint64_t> ready{0};
  int rc = reserve(cross_dq_generic_kernel<T, TL>, bytes, "cross attention dQ", ready);
  if (rc) return rc;
  cross_dq_generic_kernel<T, TL><<<dim3((unsigned)((a.Lq + TL::RT - 1) / TL::RT * splits), (unsigned)a.H, (unsigned)a.B), kThreads, bytes, st>>>(
      a, splits, part, vec4(a, true));
  if ((rc = check_launch("cross_dq_generic_kernel")) || splits == 1) return rc;
  cross_dq_sum_kernel<T><<<(unsigned)((a.B * a.H * a.Lq * a.D + 255) / 256), 256, 0, st>>>(a, splits, part);
  return check_launch("cross_dq_sum_kernel");
}
template <typename T, typename TL>
int dkdv_pass(const VsaCross& a, int splits, float* part, cudaStream_t st) {
  const int bytes = (2 * TL::row_floats + 2 * TL::col_floats + (TL::OVER ? 1 : 2) * TL::score_floats) * 4;
  static std::atomic<uint64_t> ready{0};
  const int rc = reserve(cross_dkdv_generic_kernel<T, TL>, bytes, "cross attention dK/dV", ready);
  if (rc) return rc;
  cross_dkdv_generic_kernel<T, TL><<<dim3((unsigned)((a.Lkv + TL::RT - 1) / TL::RT * splits), (unsigned)a.Hkv, (unsigned)a.B), kThreads, bytes,
                                     st>>>(a, splits, part, vec4(a, true));
  return check_launch("cross_dkdv_generic_kernel");
}

template <typename T>
int fwd_by_dim(const VsaCross& a, int splits, float* part_out, float* part_lse, cudaStream_t st) {
  const bool large = cross_generic_fwd_tile(a.B, a.H, a.Lq, a.Lkv, a.D).large;
  if (a.D <= 64) return large ? fwd<T, Tile<64, 128, 64>>(a, splits, part_out, part_lse, st) : fwd<T, Tile<64, 64>>(a, splits, part_out, part_lse, st);
  if (a.D <= 128)
    return large ? fwd<T, Tile<128, 128, 64>>(a, splits, part_out, part_lse, st) : fwd<T, Tile<128, 64>>(a, splits, part_out, part_lse, st);
  return large ? fwd<T, Tile<256, 64>>(a, splits, part_out, part_lse, st) : fwd<T, Tile<256, 32>>(a, splits, part_out, part_lse, st);
}
template <typename T>
int bwd_by_dim(const VsaCross& a, int splits, int dq_splits, float* part, cudaStream_t st) {
  const bool most = cross_generic_dq_tile(a.B, a.H, a.Lq, a.D).large;
  int rc;
  if (a.D <= 64) rc = most ? dq_pass<T, Tile<64, 128, 64>>(a, dq_splits, part, st) : dq_pass<T, Tile<64, 64>>(a, dq_splits, part, st);
  else if (a.D <= 128) rc = most ? dq_pass<T, Tile<128, 128, 64, true>>(a, dq_splits, part, st) : dq_pass<T, Tile<128, 64>>(a, dq_splits, part, st);
  else rc = most ? dq_pass<T, Tile<256, 64, 32>>(a, dq_splits, part, st) : dq_pass<T, Tile<256, 32>>(a, dq_splits, part, st);
  if (rc || a.Lkv == 0 || a.dk == nullptr) return rc;
  const bool large = cross_generic_bwd_tile(a.B, a.H, a.Hkv, a.Lq, a.Lkv, a.D).large;
  if (a.D <= 64) return large ? dkdv_pass<T, Tile<64, 128, 64, true>>(a, splits, part, st) : dkdv_pass<T, Tile<64, 64>>(a, splits, part, st);
  if (a.D <= 128) return large ? dkdv_pass<T, Tile<128, 96, 64, true>>(a, splits, part, st) : dkdv_pass<T, Tile<128, 64>>(a, splits, part, st);
  return large ? dkdv_pass<T, Tile<256, 64, 32, true>>(a, splits, part, st) : dkdv_pass<T, Tile<256, 32>>(a, splits, part, st);
}

}  // namespace

// Rows of `large` edge where tiles of them do not compute a quarter more than those of `small` would, and there are enough tiles of scores
// to fill the SMs: us of the large and the small ones, forward [1, 8, 1600, 128] x 150 (312 tiles) 49 / 59, [1, 1, 1500, 128] x 1500 (288)
// 53 / 46; dK/dV [1, 1, 1500, 128] x 1500 (384) 69 / 72, [1, 2, 1500, 128] x 300 (192) 49 / 40.
static bool large_tiles(int64_t rows, int64_t large, int64_t small, int64_t others, int64_t enough) {
  const int64_t n = (rows + large - 1) / large;
  return n * large * 4 <= (rows + small - 1) / small * small * 5 && n * others >= enough;
}
CrossTile cross_generic_fwd_tile(int64_t B, int64_t H, int64_t Lq, int64_t Lkv, int D) {
  if (D > 128) return large_tiles(Lq, 64, 32, B * H * ((Lkv + 63) / 64), 300) ? CrossTile{64, 64, true} : CrossTile{32, 32, false};
  return large_tiles(Lq, 128, 64, B * H * ((Lkv + 63) / 64), 300) ? CrossTile{128, 64, true} : CrossTile{64, 64, false};
}
CrossTile cross_generic_dq_tile(int64_t B, int64_t H, int64_t Lq, int D) {
  if (D > 128) return large_tiles(Lq, 64, 32, B * H, 74) ? CrossTile{64, 32, true} : CrossTile{32, 32, false};
  return large_tiles(Lq, 128, 64, B * H, 74) ? CrossTile{128, 64, true} : CrossTile{64, 64, false};
}
CrossTile cross_generic_bwd_tile(int64_t B, int64_t H, int64_t Hkv, int64_t Lq, int64_t Lkv, int D) {
  if (D > 128) return large_tiles(Lkv, 64, 32, B * H * ((Lq + 31) / 32), 300) ? CrossTile{64, 32, true} : CrossTile{32, 32, false};
  const int rows = D <= 64 ? 128 : 96;
  return large_tiles(Lkv, rows, 64, B * H * ((Lq + 63) / 64), 300) ? CrossTile{rows, 64, true} : CrossTile{64, 64, false};
}

int cross_fwd_generic(const VsaCross& a, int splits, float* part_out, float* part_lse, cudaStream_t st) {
  if (a.dtype == VSA_F32) return fwd_by_dim<float>(a, splits, part_out, part_lse, st);
  return a.dtype == VSA_F16 ? fwd_by_dim<__half>(a, splits, part_out, part_lse, st) : fwd_by_dim<__nv_bfloat16>(a, splits, part_out, part_lse, st);
}
int cross_bwd_generic(const VsaCross& a, int splits, int dq_splits, float* part, cudaStream_t st) {
  if (a.dtype == VSA_F32) return bwd_by_dim<float>(a, splits, dq_splits, part, st);
  return a.dtype == VSA_F16 ? bwd_by_dim<__half>(a, splits, dq_splits, part, st) : bwd_by_dim<__nv_bfloat16>(a, splits, dq_splits, part, st);
}

int cross_join(const VsaCross& a, int splits, const float* part_out, const float* part_lse, cudaStream_t st) {
  const unsigned blocks = (unsigned)((a.B * a.H * a.Lq + 7) / 8);
  if (a.dtype == VSA_F32) cross_join_kernel<float><<<blocks, 256, 0, st>>>(a, splits, part_out, part_lse);
  else if (a.dtype == VSA_F16) cross_join_kernel<__half><<<blocks, 256, 0, st>>>(a, splits, part_out, part_lse);
  else cross_join_kernel<__nv_bfloat16><<<blocks, 256, 0, st>>>(a, splits, part_out, part_lse);
  return check_launch("cross_join_kernel");
}
template <typename T>
static int sum_of(const VsaCross& a, int splits, const float* part, const int32_t* prefix, cudaStream_t st) {
  // four dims a thread where rows and their places allow it
  bool wide = a.D % 4 == 0;
  for (int i = 0; i < 3; ++i) wide = wide && a.dk_stride[i] % 4 == 0 && a.dv_stride[i] % 4 == 0;
  wide = wide && reinterpret_cast<uintptr_t>(a.dk) % 16 == 0 && reinterpret_cast<uintptr_t>(a.dv) % 16 == 0;
  const int64_t rows = a.B * a.Hkv * a.Lkv;
  if (rows > 0x7fffffffLL) return fail(VSA_ERR_UNSUPPORTED, "cross attention backward: too many key rows");
  const int cols = a.D / (wide ? 4 : 1), x = cols <= 16 ? 16 : cols <= 32 ? 32 : 64, y = 256 / x;
  const dim3 grid((unsigned)((rows + y - 1) / y), 2), block((unsigned)x, (unsigned)y);
  if (wide) cross_sum_kernel<T, 4><<<grid, block, 0, st>>>(a, splits, part, prefix);
  else cross_sum_kernel<T, 1><<<grid, block, 0, st>>>(a, splits, part, prefix);
  return check_launch("cross_sum_kernel");
}
int cross_sum(const VsaCross& a, int splits, const float* part, cudaStream_t st, const int32_t* prefix) {
  if (a.dtype == VSA_F32) return sum_of<float>(a, splits, part, prefix, st);
  return a.dtype == VSA_F16 ? sum_of<__half>(a, splits, part, prefix, st) : sum_of<__nv_bfloat16>(a, splits, part, prefix, st);
}
int cross_compact(const VsaCross& a, int32_t* prefix, int32_t* counts, void* k, void* v, cudaStream_t st) {
  const int64_t rows = a.B * a.Hkv * a.Lkv;
  if (rows > 0x7fffffffLL) return fail(VSA_ERR_UNSUPPORTED, "cross attention: too many key rows for a mask");
  cross_rank_kernel<<<(unsigned)a.B, 1024, 0, st>>>(a.key_bits, (int)cross_words(a.Lkv), prefix, counts);
  const int rc = check_launch("cross_rank_kernel");
  if (rc) return rc;
  const int x = a.D <= 64 ? 8 : 16, y = 256 / x;
  cross_compact_kernel<<<(unsigned)((rows + y - 1) / y), dim3((unsigned)x, (unsigned)y), 0, st>>>(a, prefix, counts, (uint4*)k, (uint4*)v);
  return check_launch("cross_compact_kernel");
}
int cross_key_bits(const uint8_t* mask, int64_t stride, const int32_t* lengths, uint32_t* bits, int64_t B, int64_t Lkv, cudaStream_t st) {
  const int64_t words = cross_words(Lkv);
  if (B == 0 || words == 0) return VSA_OK;
  cross_bits_kernel<<<dim3((unsigned)((words + 7) / 8), (unsigned)B), 256, 0, st>>>(mask, stride, lengths, bits, Lkv, words);
  return check_launch("cross_bits_kernel");
}

}  // namespace vsa
