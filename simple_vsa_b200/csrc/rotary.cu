// Rotary positions of q and k in one launch, optionally on the way between raster and tile order.
//
// A pair (a, b) of a head's first R dims turns by the angle of its token: (a cos - b sin, b cos + a sin); the gradient is the turn
// by the opposite angle.  Pairs are neighbours (2i, 2i+1) or halves (i, i + R/2).  Bound by HBM: 3 flops per value against 4 bytes
// moved (16-bit), so a value is read and written once and the table once per token, not once per head: a thread owns 16 bytes of
// a token's head dim, keeps their cosines and sines in registers and walks the heads of q and k.  Halves: the partners of a
// thread's 16 bytes are another thread's, and come through L1 (no shuffles, any R; both halves of a row are in flight anyway).
#include "common.cuh"
#include "kernels.h"

namespace vsa {
namespace {

constexpr int kThreads = 256;

struct RotaryArgs {
  VsaRotary a;
  int chunks;                            // 16-byte pieces (or elements) of a head
  int rows_per_block;
  int heads_per_block;
  uint32_t total_rows;
  bool wide_table;                       // rows of the table in 16-byte pieces
};

// N consecutive elements of T, moved as one word
template <typename T, int N> struct alignas(N * sizeof(T)) Pack { T e[N]; };

// How the partners of a thread's elements are read (halves): whole pieces, two elements at a time, one at a time.
enum Partner { kNeighbour, kPieces, kTwos, kOnes };

// U heads a batch; the next batch's loads are in flight while one is turned and stored.  Neighbours, us for U = 2 (five blocks an SM)
// and U = 4 (three): [1, 12 + 12, 16384, 128] 48 / 53; tiling [1, 81000, 8, 128] 83 / 100; raster [2, 92160, 40 + 40, 128] 1337 / 1264: the
// short form unless a block walks many heads.  (U = 4 with four blocks: 74 / 125 / 1976, U = 2 with four: 72 / 85 / 1311.)
constexpr int kManyHeads = 48;
template <Partner PARTNER, int U> constexpr int kBlocks = PARTNER == kNeighbour && U == 2 ? 5 : 3;

template <typename T> __device__ __forceinline__ float to_f(T x) { return Elem<T>::to(x); }
template <> __device__ __forceinline__ float to_f<float>(float x) { return x; }
template <typename T> __device__ __forceinline__ T from_f(float x) { return Elem<T>::from(x); }
template <> __device__ __forceinline__ float from_f<float>(float x) { return x; }

template <typename T, int VEC, Partner PARTNER, int U>
__global__ void __launch_bounds__(kThreads, kBlocks<PARTNER, U>) rotary_kernel(const __grid_constant__ RotaryArgs args) {
  const VsaRotary& a = args.a;
  const int r_in = threadIdx.x / args.chunks, chunk = threadIdx.x - r_in * args.chunks;
  const uint32_t row = blockIdx.x * (uint32_t)args.rows_per_block + r_in;
  if (r_in >= args.rows_per_block || row >= args.total_rows) return;
  const uint32_t b32 = row / (uint32_t)a.rows, l32 = row - b32 * (uint32_t)a.rows;
  const long long b = b32, l = l32;
  long long s = l;
  if (a.src_map != nullptr) {
    s = a.src_map[l32];
    if (s >= a.src_rows) s = -1;
  }
  const bool absent = s < 0;             // a padding row: zeros
  long long pos = l;
  if (a.positions != nullptr) pos = a.positions[b * a.positions_stride + l];
  const bool turned = !absent && pos >= 0 && pos < a.table_rows;
  const int half = a.rotary_dim >> 1, e0 = chunk * VEC;

  // Angles of this thread's elements.  Neighbours: one per pair, in the even places.  Halves: one per element, the sine with the
  // sign that the element's partner gets.  `live` has a bit per element that turns: the others are copied, not multiplied by
  // one and zero, so that an infinite neighbour stays where it is.
  float c[VEC], n[VEC];
  unsigned live = 0;
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    c[i] = 1.f;
    n[i] = 0.f;
  }
  if (turned && e0 < a.rotary_dim) {
    const float *cos_row = a.cos_table + pos * half, *sin_row = a.sin_table + pos * half;
    constexpr int N = PARTNER == kNeighbour ? VEC / 2 : VEC;      // angles of a thread
    // With one head a block this prologue was most of the kernel (scalar loads and 64-bit divisions: 130 us instead of 51 at
    // [1, 12 + 12, 16384, 128]).
    if (args.wide_table && N >= 4 && e0 + VEC <= a.rotary_dim && (PARTNER == kNeighbour || PARTNER == kPieces)) {
      const bool second = PARTNER == kPieces && e0 >= half;
      const int p = PARTNER == kNeighbour ? e0 >> 1 : (second ? e0 - half : e0);
      const bool plus = second != (a.inverse != 0);
      constexpr int W = N / 4 > 0 ? N / 4 : 1;
      float4 cv[W], sv[W];
#pragma unroll
      for (int i = 0; i < W; ++i) {
        cv[i] = reinterpret_cast<const float4*>(cos_row + p)[i];
        sv[i] = reinterpret_cast<const float4*>(sin_row + p)[i];
      }
      const float *cf = &cv[0].x, *sf = &sv[0].x;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int e = PARTNER == kNeighbour ? 2 * i : i;
        c[e % VEC] = cf[i % (4 * W)];
        n[e % VEC] = plus ? sf[i % (4 * W)] : -sf[i % (4 * W)];
      }
      live = (1u << VEC) - 1u;
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const int e = e0 + i;
        if (e >= a.rotary_dim) continue;
        const bool second = PARTNER == kNeighbour ? (e & 1) : e >= half;
        const int p = PARTNER == kNeighbour ? e >> 1 : (second ? e - half : e);
        if (PARTNER != kNeighbour || VEC == 1 || (i & 1) == 0) {
          c[i] = cos_row[p];
          const float sine = sin_row[p];
          n[i] = second != (a.inverse != 0) ? sine : -sine;
        }
        live |= 1u << i;
      }
    }
  }

  using P = Pack<T, VEC>;
  const int total = a.heads[0] + a.heads[1];
  const int h_begin = blockIdx.y * args.heads_per_block;
  const int h_end = min(total, h_begin + args.heads_per_block);
  // where the token's heads begin in q and in k; head h of the two together
  const T* src0 = (const T*)a.x[0] + b * a.x_stride[0][0] + s * a.x_stride[0][2];
  const T* src1 = (const T*)a.x[1] + b * a.x_stride[1][0] + s * a.x_stride[1][2] - a.heads[0] * a.x_stride[1][1];
  T* dst0 = (T*)a.y[0] + b * a.y_stride[0][0] + l * a.y_stride[0][2] + e0;
  T* dst1 = (T*)a.y[1] + b * a.y_stride[1][0] + l * a.y_stride[1][2] - a.heads[0] * a.y_stride[1][1] + e0;
  auto load = [&](int h0, P(&own)[U], P(&other)[U]) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = h0 + u;
      if (h >= h_end || absent) continue;
      const T* src = h < a.heads[0] ? src0 + h * a.x_stride[0][1] : src1 + h * a.x_stride[1][1];
      own[u] = *reinterpret_cast<const P*>(src + e0);
      if (PARTNER == kNeighbour) {
        if (VEC == 1 && live) other[u].e[0] = src[e0 ^ 1];
      } else if (PARTNER == kPieces) {
        if (live) other[u] = *reinterpret_cast<const P*>(src + (e0 < half ? e0 + half : e0 - half));
      } else {
        constexpr int W = PARTNER == kTwos && VEC >= 2 ? 2 : 1;
#pragma unroll
        for (int i = 0; i < VEC; i += W)
          if (live >> i & 1u) {
            const int e = e0 + i;
            const Pack<T, W> w = *reinterpret_cast<const Pack<T, W>*>(src + (e < half ? e + half : e - half));
#pragma unroll
            for (int j = 0; j < W; ++j) other[u].e[i + j] = w.e[j];
          }
      }
    }
  };
  P own[U], other[U];
  load(h_begin, own, other);
  for (int h0 = h_begin; h0 < h_end; h0 += U) {
    P own_next[U], other_next[U];
    if (h0 + U < h_end) load(h0 + U, own_next, other_next);      // in flight under this batch's arithmetic and stores
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = h0 + u;
      if (h >= h_end) continue;
      P res;
      if (absent) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) res.e[i] = from_f<T>(0.f);
      } else if (PARTNER == kNeighbour && VEC > 1) {
#pragma unroll
        for (int i = 0; i < VEC; i += 2) {
          const float x = to_f<T>(own[u].e[i]), y = to_f<T>(own[u].e[(i + 1) % VEC]);
          // n is minus the sine for the first of the pair
          const bool on = live >> i & 1u;
          res.e[i] = on ? from_f<T>(fmaf(y, n[i], x * c[i])) : own[u].e[i];
          res.e[(i + 1) % VEC] = on ? from_f<T>(fmaf(-x, n[i], y * c[i])) : own[u].e[(i + 1) % VEC];
        }
      } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i)
          res.e[i] = live >> i & 1u ? from_f<T>(fmaf(to_f<T>(other[u].e[i]), n[i], to_f<T>(own[u].e[i]) * c[i])) : own[u].e[i];
      }
      *reinterpret_cast<P*>(h < a.heads[0] ? dst0 + h * a.y_stride[0][1] : dst1 + h * a.y_stride[1][1]) = res;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) own[u] = own_next[u], other[u] = other_next[u];
  }
}

template <typename T, int VEC, Partner PARTNER, int U>
int launch_of(const VsaRotary& a, cudaStream_t st) {
  const bool wide = a.rotary_dim % 8 == 0 && reinterpret_cast<uintptr_t>(a.cos_table) % 16 == 0 && reinterpret_cast<uintptr_t>(a.sin_table) % 16 == 0;
  RotaryArgs args{a, a.D / VEC, 0, 0, (uint32_t)(a.B * a.rows), wide};
  if (args.chunks > kThreads) return fail(VSA_ERR_UNSUPPORTED, "rotary: head dim %d is above 256", a.D);
  args.rows_per_block = kThreads / args.chunks;
  const long long rows = a.B * a.rows, blocks = (rows + args.rows_per_block - 1) / args.rows_per_block;
  if (rows > 0x7fffffffLL) return fail(VSA_ERR_UNSUPPORTED, "rotary: 2^31 tokens at most");
  // All heads of a token in one block where that fills the GPU sixteen times over (the table is then read once); fewer heads a
  // block, down to one, where there are few tokens.
  const int total = a.heads[0] + a.heads[1];
  const long long want = 148LL * 16;
  long long hpb = blocks >= want ? total : (total * blocks + want - 1) / want;
  if (hpb > U) hpb = (hpb + U - 1) / U * U;
  if ((total + hpb - 1) / hpb > 65535) hpb = (total + 65534) / 65535;
  args.heads_per_block = (int)(hpb < 1 ? 1 : hpb);
  const dim3 grid((unsigned)blocks, (unsigned)((total + args.heads_per_block - 1) / args.heads_per_block));
  rotary_kernel<T, VEC, PARTNER, U><<<grid, kThreads, 0, st>>>(args);
  return check_launch("rotary_kernel");
}

template <typename T, int VEC, Partner PARTNER>
int launch(const VsaRotary& a, cudaStream_t st) {
  if (PARTNER == kNeighbour && VEC > 1 && a.heads[0] + a.heads[1] >= kManyHeads) return launch_of<T, VEC, PARTNER, 4>(a, st);
  return launch_of<T, VEC, PARTNER, 2>(a, st);
}

template <typename T>
int by_alignment(const VsaRotary& a, cudaStream_t st) {
  constexpr int VEC = 16 / (int)sizeof(T);
  bool whole = a.D % VEC == 0;
  for (int t = 0; t < 2; ++t) {
    if (a.heads[t] == 0) continue;
    whole = whole && reinterpret_cast<uintptr_t>(a.x[t]) % 16 == 0 && reinterpret_cast<uintptr_t>(a.y[t]) % 16 == 0;
    for (int i = 0; i < 3; ++i) whole = whole && a.x_stride[t][i] % VEC == 0 && a.y_stride[t][i] % VEC == 0;
  }
  const int half = a.rotary_dim / 2;
  if (a.interleaved) return whole ? launch<T, VEC, kNeighbour>(a, st) : launch<T, 1, kNeighbour>(a, st);
  if (!whole) return launch<T, 1, kOnes>(a, st);
  return half % VEC == 0 ? launch<T, VEC, kPieces>(a, st) : half % 2 == 0 ? launch<T, VEC, kTwos>(a, st) : launch<T, VEC, kOnes>(a, st);
}

}  // namespace

int rotary(const VsaRotary& a, cudaStream_t st) {
  if (a.D > 256) return fail(VSA_ERR_UNSUPPORTED, "rotary: head dim %d is above 256", a.D);
  if (a.B == 0 || a.rows == 0 || a.D == 0 || a.heads[0] + a.heads[1] == 0) return VSA_OK;
  if (a.dtype == VSA_F32) return by_alignment<float>(a, st);
  return a.dtype == VSA_F16 ? by_alignment<__half>(a, st) : by_alignment<__nv_bfloat16>(a, st);
}

}  // namespace vsa
