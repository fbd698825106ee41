// Rotary positions of q and k in one launch, optionally on the way between raster and tile order.
//
// A pair (a, b) of a head's first R dims turns by the angle of its token: (a cos - b sin, b cos + a sin); the gradient is the turn
// by the opposite angle.  Pairs are neighbours (2i, 2i+1) or halves (i, i + R/2).  Bound by HBM: 3 flops per value against 4 bytes
// moved (16-bit), so a value is read and written once and the table once per token, not once per head: a thread owns 16 bytes of
// a token's head dim (halves: 16 of each), keeps their cosines and sines in registers and walks the heads of q and k.  Halves that
// do not begin on a 16-byte piece: the partners of a thread's elements are other threads', and come through L1.
// [2, 92160, 40 + 40, 128], 7.6 GB: 1.18 ms, 6.45 TB/s of 6.54 that a copy reaches.
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
  bool wide_table, twos_table;           // rows of the table in pieces of 16 and of 8 bytes
};

// N consecutive elements of T, moved as one word
template <typename T, int N> struct alignas(N * sizeof(T)) Pack { T e[N]; };

// How the partners of a thread's elements come to it: in the same piece; as a second piece that the thread turns too (halves of whole
// pieces); read beside its own two elements or one at a time, another thread turning them.
enum Partner { kNeighbour, kPieces, kTwos, kOnes };

// Heads whose loads are in flight together, and blocks an SM.  More in flight is slower, not only fewer: us at [1, 12 + 12, 16384, 128],
// tiling [1, 81000, 8, 128] and raster [2, 92160, 40 + 40, 128] for neighbours with four heads and four blocks 41 / 69 / 1177 (the copy
// rate), four and six 77 / 125 / 2163, two and eight 76 / 124 / 2148; halves of whole pieces with one and four 41 / 72 / 1235, two and
// four 47 / 83 / 1424, one and six 77 / 123 / 2275.  Halves of 54 (two elements at a time): 81,000 tokens, one and five 91, two and four 135.
template <Partner PARTNER> constexpr int kHeads = PARTNER == kNeighbour ? 4 : 1;
template <Partner PARTNER> constexpr int kBlocks = PARTNER == kNeighbour || PARTNER == kPieces ? 4 : 5;

template <typename T> __device__ __forceinline__ float to_f(T x) { return Elem<T>::to(x); }
template <> __device__ __forceinline__ float to_f<float>(float x) { return x; }
template <typename T> __device__ __forceinline__ T from_f(float x) { return Elem<T>::from(x); }
template <> __device__ __forceinline__ float from_f<float>(float x) { return x; }

template <typename T, int VEC, Partner PARTNER>
__global__ void __launch_bounds__(kThreads, kBlocks<PARTNER>) rotary_kernel(const __grid_constant__ RotaryArgs args) {
  constexpr int U = kHeads<PARTNER>;
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
  const int half = a.rotary_dim >> 1;
  // this thread's elements, and with kPieces its second piece (the pair's other half, or the next piece of those that are copied)
  const int turns = half / VEC;
  const int e0 = PARTNER != kPieces || chunk < turns ? chunk * VEC : a.rotary_dim + 2 * (chunk - turns) * VEC;
  const int e1 = chunk < turns ? e0 + half : e0 + VEC;
  const bool two = PARTNER == kPieces && e1 < a.D;

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
  if (turned && e0 < a.rotary_dim) {               // (kPieces: in the first half)
    const float *cos_row = a.cos_table + pos * half, *sin_row = a.sin_table + pos * half;
    constexpr int N = PARTNER == kNeighbour ? VEC / 2 : VEC;      // angles of a thread
    // With one head a block this prologue was most of the kernel (scalar loads and 64-bit divisions: 130 us instead of 51 at
    // [1, 12 + 12, 16384, 128]).
    if (args.wide_table && N >= 4 && e0 + VEC <= a.rotary_dim && (PARTNER == kNeighbour || PARTNER == kPieces)) {
      const int p = PARTNER == kNeighbour ? e0 >> 1 : e0;
      const bool plus = a.inverse != 0;
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
    } else if (args.twos_table && PARTNER == kTwos && VEC >= 2) {
      constexpr int Q = VEC / 2 > 0 ? VEC / 2 : 1;
#pragma unroll
      for (int i = 0; i < Q; ++i) {
        const int e = e0 + 2 * i;
        if (e >= a.rotary_dim) continue;
        const bool second = e >= half, plus = second != (a.inverse != 0);
        const int p = second ? e - half : e;
        const float2 cv = *reinterpret_cast<const float2*>(cos_row + p), sv = *reinterpret_cast<const float2*>(sin_row + p);
        c[2 * i % VEC] = cv.x;
        c[(2 * i + 1) % VEC] = cv.y;
        n[2 * i % VEC] = plus ? sv.x : -sv.x;
        n[(2 * i + 1) % VEC] = plus ? sv.y : -sv.y;
        live |= 3u << (2 * i);
      }
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
  const int h_begin = blockIdx.y * args.heads_per_block, h_end = h_begin + args.heads_per_block;
#pragma unroll 1
  for (int t = 0; t < 2; ++t) {            // this block's heads of q, then of k
    const int before = t ? a.heads[0] : 0;
    int h = max(h_begin - before, 0);
    const int last = min(h_end - before, a.heads[t]);
    if (h >= last) continue;
    const long long s_step = a.x_stride[t][1], d_step = a.y_stride[t][1];
    const T* src = (const T*)a.x[t] + b * a.x_stride[t][0] + s * a.x_stride[t][2] + h * s_step;
    T* dst = (T*)a.y[t] + b * a.y_stride[t][0] + l * a.y_stride[t][2] + h * d_step + e0;
    if (absent) {
      P zero;
#pragma unroll
      for (int i = 0; i < VEC; ++i) zero.e[i] = from_f<T>(0.f);
      for (; h < last; ++h, dst += d_step) {
        *reinterpret_cast<P*>(dst) = zero;
        if (two) *reinterpret_cast<P*>(dst + (e1 - e0)) = zero;
      }
      continue;
    }
#pragma unroll 1
    for (; h < last; h += U, src += U * s_step, dst += U * d_step) {
      P own[U], other[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (h + u >= last) continue;
        const T* row_u = src + u * s_step;
        own[u] = *reinterpret_cast<const P*>(row_u + e0);
        if (PARTNER == kNeighbour) {
          if (VEC == 1 && live) other[u].e[0] = row_u[e0 ^ 1];
        } else if (PARTNER == kPieces) {
          if (two) other[u] = *reinterpret_cast<const P*>(row_u + e1);
        } else {
          constexpr int W = PARTNER == kTwos && VEC >= 2 ? 2 : 1;
#pragma unroll
          for (int i = 0; i < VEC; i += W)
            if (live >> i & 1u) {
              const int e = e0 + i;
              const Pack<T, W> w = *reinterpret_cast<const Pack<T, W>*>(row_u + (e < half ? e + half : e - half));
#pragma unroll
              for (int j = 0; j < W; ++j) other[u].e[i + j] = w.e[j];
            }
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (h + u >= last) continue;
        P res;
        if (PARTNER == kNeighbour && VEC > 1) {
#pragma unroll
          for (int i = 0; i < VEC; i += 2) {
            const float x = to_f<T>(own[u].e[i]), y = to_f<T>(own[u].e[(i + 1) % VEC]);
            // n is minus the sine for the first of the pair
            const bool on = live >> i & 1u;
            res.e[i] = on ? from_f<T>(fmaf(y, n[i], x * c[i])) : own[u].e[i];
            res.e[(i + 1) % VEC] = on ? from_f<T>(fmaf(-x, n[i], y * c[i])) : own[u].e[(i + 1) % VEC];
          }
        } else if (PARTNER == kPieces) {
          P res1 = other[u];
          res = own[u];
          if (live) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
              const float x = to_f<T>(own[u].e[i]), y = to_f<T>(other[u].e[i]);
              res.e[i] = from_f<T>(fmaf(y, n[i], x * c[i]));
              res1.e[i] = from_f<T>(fmaf(-x, n[i], y * c[i]));
            }
          }
          if (two) *reinterpret_cast<P*>(dst + u * d_step + (e1 - e0)) = res1;
        } else {
#pragma unroll
          for (int i = 0; i < VEC; ++i)
            res.e[i] = live >> i & 1u ? from_f<T>(fmaf(to_f<T>(other[u].e[i]), n[i], to_f<T>(own[u].e[i]) * c[i])) : own[u].e[i];
        }
        *reinterpret_cast<P*>(dst + u * d_step) = res;
      }
    }
  }
}

template <typename T, int VEC, Partner PARTNER>
int launch(const VsaRotary& a, cudaStream_t st) {
  const bool wide = a.rotary_dim % 8 == 0 && reinterpret_cast<uintptr_t>(a.cos_table) % 16 == 0 && reinterpret_cast<uintptr_t>(a.sin_table) % 16 == 0;
  const bool twos = a.rotary_dim % 4 == 0 && reinterpret_cast<uintptr_t>(a.cos_table) % 8 == 0 && reinterpret_cast<uintptr_t>(a.sin_table) % 8 == 0;
  const int pieces = a.D / VEC, turned = a.rotary_dim / VEC;
  RotaryArgs args{a, PARTNER == kPieces ? turned / 2 + (pieces - turned + 1) / 2 : pieces, 0, 0, (uint32_t)(a.B * a.rows), wide, twos};
  if (args.chunks > kThreads) return fail(VSA_ERR_UNSUPPORTED, "rotary: head dim %d is above 256", a.D);
  args.rows_per_block = kThreads / args.chunks;
  const long long rows = a.B * a.rows, blocks = (rows + args.rows_per_block - 1) / args.rows_per_block;
  if (rows > 0x7fffffffLL) return fail(VSA_ERR_UNSUPPORTED, "rotary: 2^31 tokens at most");
  // All heads of a token in one block where that fills the GPU sixteen times over (the table is then read once); fewer heads a
  // block, down to one, where there are few tokens.
  const int total = a.heads[0] + a.heads[1];
  const long long want = 148LL * 16;
  long long hpb = blocks >= want ? total : (total * blocks + want - 1) / want;
  constexpr int U = kHeads<PARTNER>;
  if (hpb > U) hpb = (hpb + U - 1) / U * U;
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
