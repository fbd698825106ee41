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
constexpr int kUnroll = 4;               // heads whose loads are in flight together

struct RotaryArgs {
  VsaRotary a;
  int chunks;                            // 16-byte pieces (or elements) of a head
  int rows_per_block;
  int heads_per_block;
};

// N consecutive elements of T, moved as one word
template <typename T, int N> struct alignas(N * sizeof(T)) Pack { T e[N]; };

// How the partners of a thread's elements are read (halves): whole pieces, two elements at a time, one at a time.
enum Partner { kNeighbour, kPieces, kTwos, kOnes };

template <typename T> __device__ __forceinline__ float to_f(T x) { return Elem<T>::to(x); }
template <> __device__ __forceinline__ float to_f<float>(float x) { return x; }
template <typename T> __device__ __forceinline__ T from_f(float x) { return Elem<T>::from(x); }
template <> __device__ __forceinline__ float from_f<float>(float x) { return x; }

template <typename T, int VEC, Partner PARTNER>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const __grid_constant__ RotaryArgs args) {
  const VsaRotary& a = args.a;
  const int r_in = threadIdx.x / args.chunks, chunk = threadIdx.x - r_in * args.chunks;
  const long long row = (long long)blockIdx.x * args.rows_per_block + r_in;
  if (r_in >= args.rows_per_block || row >= a.B * a.rows) return;
  const long long b = row / a.rows, l = row - b * a.rows;
  long long s = l;
  if (a.src_map != nullptr) {
    s = a.src_map[l];
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
    const int e = e0 + i;
    c[i] = 1.f;
    n[i] = 0.f;
    if (turned && e < a.rotary_dim) {
      const bool second = PARTNER == kNeighbour ? (e & 1) : e >= half;
      const int p = PARTNER == kNeighbour ? e >> 1 : (second ? e - half : e);
      if (PARTNER != kNeighbour || VEC == 1 || (i & 1) == 0) {
        c[i] = a.cos_table[pos * half + p];
        const float sine = a.sin_table[pos * half + p];
        n[i] = second != (a.inverse != 0) ? sine : -sine;
      }
      live |= 1u << i;
    }
  }

  using P = Pack<T, VEC>;
  const int total = a.heads[0] + a.heads[1];
  const int h_begin = blockIdx.y * args.heads_per_block;
  const int h_end = min(total, h_begin + args.heads_per_block);
  for (int h0 = h_begin; h0 < h_end; h0 += kUnroll) {
    P own[kUnroll], other[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int h = h0 + u;
      if (h >= h_end || absent) continue;
      const int t = h >= a.heads[0] ? 1 : 0, hh = t ? h - a.heads[0] : h;
      const T* src = (const T*)a.x[t] + b * a.x_stride[t][0] + hh * a.x_stride[t][1] + s * a.x_stride[t][2];
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
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int h = h0 + u;
      if (h >= h_end) continue;
      const int t = h >= a.heads[0] ? 1 : 0, hh = t ? h - a.heads[0] : h;
      T* dst = (T*)a.y[t] + b * a.y_stride[t][0] + hh * a.y_stride[t][1] + l * a.y_stride[t][2];
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
      *reinterpret_cast<P*>(dst + e0) = res;
    }
  }
}

template <typename T, int VEC, Partner PARTNER>
int launch(const VsaRotary& a, cudaStream_t st) {
  RotaryArgs args{a, a.D / VEC, 0, 0};
  if (args.chunks > kThreads) return fail(VSA_ERR_UNSUPPORTED, "rotary: head dim %d is above 256", a.D);
  args.rows_per_block = kThreads / args.chunks;
  const long long rows = a.B * a.rows, blocks = (rows + args.rows_per_block - 1) / args.rows_per_block;
  if (blocks > 0x7fffffffLL) return fail(VSA_ERR_UNSUPPORTED, "rotary: too many tokens");
  // All heads of a token in one block where that fills the GPU sixteen times over (the table is then read once); fewer heads a
  // block, down to one, where there are few tokens.
  const int total = a.heads[0] + a.heads[1];
  const long long want = 148LL * 16;
  long long hpb = blocks >= want ? total : (total * blocks + want - 1) / want;
  if (hpb > kUnroll) hpb = (hpb + kUnroll - 1) / kUnroll * kUnroll;
  if ((total + hpb - 1) / hpb > 65535) hpb = (total + 65534) / 65535;
  args.heads_per_block = (int)(hpb < 1 ? 1 : hpb);
  const dim3 grid((unsigned)blocks, (unsigned)((total + args.heads_per_block - 1) / args.heads_per_block));
  rotary_kernel<T, VEC, PARTNER><<<grid, kThreads, 0, st>>>(args);
  return check_launch("rotary_kernel");
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
