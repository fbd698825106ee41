// Cross attention for up to four query rows (the tokens of all query heads of a key head together): bf16 and fp16, the decoding form.
// Bound by HBM: every key and value is read once for two flops per byte and row, so there is nothing for the tensor cores to do, and a
// tile of 128 rows spends its time on rows that do not exist.
//
// A key is D / 8 neighbouring lanes with 16 bytes of it each; a group of lanes walks keys of its own with its own running maximum, sum
// and output, four keys (K and V) in flight, and the groups of a CTA are joined through shared memory.  fp32 throughout, one
// rounding of the result.  [8, 40, 1, 128] against 512 keys (ragged, 57 MB): 17 us against 23 on the 128-row tiles.
#include "common.cuh"
#include "kernels.h"

namespace vsa {
namespace {

constexpr int kThreads = 256;
constexpr int kBatch = 4;                  // keys of a group whose loads are in flight together

template <typename T, int ROWS, int LANES>
__global__ void __launch_bounds__(kThreads, ROWS <= 2 ? 3 : 1) cross_rows_kernel(const __grid_constant__ VsaCross a, int splits, float* part_out, float* part_lse) {
  constexpr int kGroups = kThreads / LANES;
  __shared__ float s_max[kGroups][ROWS], s_sum[kGroups][ROWS];
  __shared__ float s_out[kGroups / (32 / LANES)][ROWS][LANES * 8];       // a warp's groups are joined by shuffles first
  const int split = blockIdx.x, hk = blockIdx.y, b = blockIdx.z, heads = (int)(a.H / a.Hkv), rows = heads * (int)a.Lq;
  const int tid = threadIdx.x, lane = tid % LANES, group = tid / LANES, d = lane * 8;
  const bool mine = d < a.D;
  const int len = cross_length(a, b);
  const uint32_t* bits = a.key_bits == nullptr ? nullptr : a.key_bits + (long long)b * cross_words(a.Lkv);
  const int per = ((len + splits - 1) / splits + kGroups - 1) / kGroups * kGroups, k0 = split * per, k1 = min(len, k0 + per);
  const float c = a.scale * kLog2e;

  float q[ROWS][8], acc[ROWS][8], m[ROWS], l[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
    uint4 x = make_uint4(0, 0, 0, 0);
    if (r < rows && mine) {
      const int h = hk * heads + r / (int)a.Lq, t = r % (int)a.Lq;
      x = *reinterpret_cast<const uint4*>((const T*)a.q + b * a.q_stride[0] + h * a.q_stride[1] + t * a.q_stride[2] + d);
    }
    const uint32_t* w = &x.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = Elem<T>::unpack(w[i]);
      q[r][2 * i] = f.x * c;
      q[r][2 * i + 1] = f.y * c;
      acc[r][2 * i] = acc[r][2 * i + 1] = 0.f;
    }
  }
  const T* kp = (const T*)a.k + b * a.k_stride[0] + hk * a.k_stride[1] + d;
  const T* vp = (const T*)a.v + b * a.v_stride[0] + hk * a.v_stride[1] + d;
  for (int at = k0 + group; __any_sync(0xffffffffu, at < k1); at += kBatch * kGroups) {
    uint4 k[kBatch], v[kBatch];
    unsigned live = 0;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int key = at + i * kGroups;
      const bool on = key < k1 && (bits == nullptr || (bits[key >> 5] >> (key & 31) & 1u));
      live |= (unsigned)on << i;
      k[i] = v[i] = make_uint4(0, 0, 0, 0);
      if (on && mine) {
        k[i] = *reinterpret_cast<const uint4*>(kp + key * a.k_stride[2]);
        v[i] = *reinterpret_cast<const uint4*>(vp + key * a.v_stride[2]);
      }
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      float s[kBatch], top = m[r];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const uint32_t* w = &k[i].x;
        float x = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 f = Elem<T>::unpack(w[e]);
          x = fmaf(f.x, q[r][2 * e], fmaf(f.y, q[r][2 * e + 1], x));
        }
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
        s[i] = live >> i & 1u ? x : -INFINITY;
        top = fmaxf(top, s[i]);
      }
      const float shift = top == -INFINITY ? 0.f : top, keep = exp2f(m[r] - shift);
      m[r] = top;
      l[r] *= keep;
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[r][e] *= keep;
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const float p = exp2f(s[i] - shift);
        l[r] += p;
        const uint32_t* w = &v[i].x;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 f = Elem<T>::unpack(w[e]);
          acc[r][2 * e] = fmaf(p, f.x, acc[r][2 * e]);
          acc[r][2 * e + 1] = fmaf(p, f.y, acc[r][2 * e + 1]);
        }
      }
    }
  }

  // join: every group scales its sums to the CTA's maximum
  if (lane == 0)
#pragma unroll
    for (int r = 0; r < ROWS; ++r) s_max[group][r] = m[r];
  __syncthreads();
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    float top = s_max[0][r];
    for (int g = 1; g < kGroups; ++g) top = fmaxf(top, s_max[g][r]);
    const float f = top == -INFINITY ? 0.f : exp2f(m[r] - top);
    m[r] = top;
    if (lane == 0) s_sum[group][r] = l[r] * f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float x = acc[r][e] * f;
#pragma unroll
      for (int o = LANES; o < 32; o <<= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
      if ((tid & 31) < LANES) s_out[tid >> 5][r][d + e] = x;
    }
  }
  __syncthreads();
  const long long lp = cross_rows(a.Lq);
  for (int e = tid; e < rows * a.D; e += kThreads) {
    const int r = e / a.D, dd = e - r * a.D, h = hk * heads + r / (int)a.Lq, t = r % (int)a.Lq;
    float sum = 0.f, x = 0.f;
    for (int g = 0; g < kGroups; ++g) sum += s_sum[g][r];
#pragma unroll
    for (int g = 0; g < kThreads / 32; ++g) x += s_out[g][r][dd];
    x = sum == 0.f ? 0.f : x / sum;
    const long long bh = (long long)b * a.H + h;
    float top = -INFINITY;
    if (dd == 0)
      for (int g = 0; g < kGroups; ++g) top = fmaxf(top, s_max[g][r]);
    if (splits == 1) {
      ((T*)a.out)[b * a.out_stride[0] + h * a.out_stride[1] + t * a.out_stride[2] + dd] = Elem<T>::from(x);
      if (dd == 0) a.lse2[bh * lp + t] = sum == 0.f ? INFINITY : top + log2f(sum);
    } else {
      const long long at = (split * (long long)a.B * a.H + bh) * a.Lq + t;
      part_out[at * a.D + dd] = x;
      if (dd == 0) part_lse[at] = sum == 0.f ? -INFINITY : top + log2f(sum);
    }
  }
  if (splits == 1)                          // the padding behind the rows, which a backward reads
    for (int e = tid; e < heads * (int)(lp - a.Lq); e += kThreads) {
      const int pad = (int)(lp - a.Lq), h = e / pad;
      a.lse2[((long long)b * a.H + hk * heads + h) * lp + a.Lq + (e - h * pad)] = INFINITY;
    }
}

template <typename T, int LANES>
int by_rows(const VsaCross& a, int splits, float* part_out, float* part_lse, cudaStream_t st) {
  const dim3 grid((unsigned)splits, (unsigned)a.Hkv, (unsigned)a.B);
  const int64_t rows = a.H / a.Hkv * a.Lq;
  if (rows <= 1) cross_rows_kernel<T, 1, LANES><<<grid, kThreads, 0, st>>>(a, splits, part_out, part_lse);
  else if (rows <= 2) cross_rows_kernel<T, 2, LANES><<<grid, kThreads, 0, st>>>(a, splits, part_out, part_lse);
  else cross_rows_kernel<T, 4, LANES><<<grid, kThreads, 0, st>>>(a, splits, part_out, part_lse);
  return check_launch("cross_rows_kernel");
}

}  // namespace

int cross_fwd_rows(const VsaCross& a, int splits, float* part_out, float* part_lse, cudaStream_t st) {
  if (a.dtype == VSA_F16)
    return a.D <= 64 ? by_rows<__half, 8>(a, splits, part_out, part_lse, st) : by_rows<__half, 16>(a, splits, part_out, part_lse, st);
  return a.D <= 64 ? by_rows<__nv_bfloat16, 8>(a, splits, part_out, part_lse, st) : by_rows<__nv_bfloat16, 16>(a, splits, part_out, part_lse, st);
}

}  // namespace vsa
