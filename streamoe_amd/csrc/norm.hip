// norm.hip — the residual's addition with the RMSNorm in front of a block,
// for any number of rows, with an 8-bit copy of the normalised rows.
//
//   r = x + residual,  inv = 1 / sqrt(sum r^2 / hidden + eps),  y = r inv w
//   8 bits: over each group (or the row) top = max |y|, scale = top / 127,
//   code = rint(y / scale)
//
// The sum and its root are f64 (an f32 r^2 leaves the range from 2^64 on),
// 1 / sqrt and both quotients round to f32; only the outputs round further
// (bf16 and int8 to nearest even).
#include "common.h"
#include "kernels.h"

namespace smoe {

typedef __bf16 nbf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x8 __attribute__((ext_vector_type(8)));

constexpr uint32_t kNormThreads = 256;

// One block per row, the row in registers between its two uses, so it is read
// once: thread t holds the eights t, t + 256, ... (VEC), or the elements t,
// t + 256, ... where rows are no whole number of eights. Memory bounds many
// rows (1000 of 4096, bf16 in and out, codes in groups of 64, 53 MB: 13.2 us,
// 4.0 TB/s, of the 5.0 of a large copy), one round trip a single one (2048: 2.0
// us). The weight's loads go out with the row's. Rows of less than 2048 leave
// threads without values (65536 rows of 256: 3.4 TB/s, of 128: 1.7).
// 1 / sqrt(m) by one Newton step on the hardware's estimate (good to 2^-23):
// to 2^-45; 0 for an infinity.
__device__ __forceinline__ float norm_rsqrt(double m) {
  const double y = __builtin_amdgcn_rsq(m), e = __builtin_fma(-m * y, y, 1.0);
  return m == (double)INFINITY ? 0.f : (float)__builtin_fma(0.5 * y, e, y);
}

template <bool XBF16, int V, bool VEC>
__global__ __launch_bounds__(kNormThreads) void k_rmsnorm(NormArgs a) {
  __shared__ double sums[kNormThreads / 64];
  __shared__ float tops[kNormThreads / 64];
  const uint32_t t = threadIdx.x, H = a.hidden;
  const uint64_t row = (uint64_t)blockIdx.x * H;
  auto at = [&](int i, int j) { return VEC ? (i * kNormThreads + t) * 8 + j : t + kNormThreads * (i * 8 + j); };
  float r[V][8], w[V][8];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    if constexpr (VEC) {
      f32x8 v = {0, 0, 0, 0, 0, 0, 0, 0}, wv = v;
      if (at(i, 0) < H) {
        const uint64_t e = row + at(i, 0);
        if constexpr (XBF16)
          v = __builtin_convertvector(*reinterpret_cast<const nbf16x8*>((const uint16_t*)a.x + e), f32x8);
        else
          v = *reinterpret_cast<const f32x8*>((const float*)a.x + e);
        if (a.residual) v += *reinterpret_cast<const f32x8*>(a.residual + e);
        if (a.w) wv = __builtin_convertvector(*reinterpret_cast<const nbf16x8*>(a.w + at(i, 0)), f32x8);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) r[i][j] = v[j], w[i][j] = a.w ? wv[j] : 1.f;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t c = at(i, j);
        float v = 0.f, wv = 1.f;
        if (c < H) {
          v = XBF16 ? bf16f(((const uint16_t*)a.x)[row + c]) : ((const float*)a.x)[row + c];
          if (a.residual) v += a.residual[row + c];
          if (a.w) wv = bf16f(a.w[c]);
        }
        r[i][j] = v;
        w[i][j] = wv;
      }
    }
  }
  double ss = 0.0;
#pragma unroll
  for (int i = 0; i < V; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) ss = __builtin_fma((double)r[i][j], (double)r[i][j], ss);
  ss = wave_sum_f64(ss);
  if ((t & 63) == 0) sums[t >> 6] = ss;
  __syncthreads();
  const float inv = norm_rsqrt(((sums[0] + sums[1]) + (sums[2] + sums[3])) * a.inv_hidden + (double)a.eps);
  if (a.sum) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if constexpr (VEC) {
        if (at(i, 0) < H) {
          f32x8 v;
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = r[i][j];
          *reinterpret_cast<f32x8*>(a.sum + row + at(i, 0)) = v;
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (at(i, j) < H) a.sum[row + at(i, j)] = r[i][j];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) r[i][j] = r[i][j] * inv * w[i][j];
  if (a.out) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if constexpr (VEC) {
        if (at(i, 0) < H) {
          f32x8 v;
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = r[i][j];
          if (a.out_bf16)
            *reinterpret_cast<nbf16x8*>((uint16_t*)a.out + row + at(i, 0)) = __builtin_convertvector(v, nbf16x8);
          else
            *reinterpret_cast<f32x8*>((float*)a.out + row + at(i, 0)) = v;
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (at(i, j) < H) {
            if (a.out_bf16)
              reinterpret_cast<__bf16*>(a.out)[row + at(i, j)] = (__bf16)r[i][j];
            else
              ((float*)a.out)[row + at(i, j)] = r[i][j];
          }
      }
    }
  }
  if (!a.q) return;
  // Largest magnitude of the thread's values; `fin` is 0 while all are finite,
  // else NaN. Values past the row are zeros.
  float top[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    float m = 0.f, fin = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const bool in = VEC || at(i, j) < H;
      m = fmaxf(m, in ? fabsf(r[i][j]) : 0.f);
      fin = __builtin_fmaf(in ? r[i][j] : 0.f, 0.f, fin);
    }
    top[i] = fin == 0.f ? m : INFINITY;
  }
  const uint32_t G = a.group ? a.group : H;
  if (a.group == 0) {  // the whole row
    float m = top[0];
#pragma unroll
    for (int i = 1; i < V; ++i) m = fmaxf(m, top[i]);
    m = wave_max(m);
    if ((t & 63) == 0) tops[t >> 6] = m;
    __syncthreads();
    m = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
#pragma unroll
    for (int i = 0; i < V; ++i) top[i] = m;
  } else {  // 4, 8 or 16 neighbouring threads hold a group
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float m = top[i];
      m = fmaxf(m, __shfl_xor(m, 1, kWave));
      m = fmaxf(m, __shfl_xor(m, 2, kWave));
      if (a.group >= 64) m = fmaxf(m, __shfl_xor(m, 4, kWave));
      if (a.group == 128) m = fmaxf(m, __shfl_xor(m, 8, kWave));
      top[i] = m;
    }
  }
  const uint32_t ng = H / G;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    // An infinity or NaN in the group: scale NaN, codes 0.
    const bool ok = top[i] >= kQuantFloor && top[i] < INFINITY;
    const float s = top[i] < INFINITY ? (ok ? top[i] / 127.f : 0.f) : __builtin_nanf("");
    // y / s rounded to an integer, by way of y (127 / top): the two quotients
    // differ by less than 4 2^-24 of at most 127.5, so only a product within
    // 2^-14 of a tie needs the division itself (one thread in a thousand; with
    // all values divided the 1000 rows above take 0.4 us more).
    const float f = ok ? 127.f / top[i] : 0.f;
    float k[8], off = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float v = ok ? r[i][j] * f : 0.f;
      k[j] = __builtin_rintf(v);
      off = fmaxf(off, fabsf(v - k[j]));
    }
    if (off > 0.5f - 0x1p-14f) {
#pragma unroll
      for (int j = 0; j < 8; ++j) k[j] = __builtin_rintf(r[i][j] / s);
    }
    int32_t c[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) c[j] = (int32_t)k[j];
    if constexpr (VEC) {
      const uint32_t e = at(i, 0);
      if (e < H) {
        uint2 v;
        v.x = pack_bytes(c[0], c[1], c[2], c[3]);
        v.y = pack_bytes(c[4], c[5], c[6], c[7]);
        *reinterpret_cast<uint2*>(a.q + row + e) = v;
        if (e % G == 0) a.scales[(uint64_t)blockIdx.x * ng + e / G] = s;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (at(i, j) < H) a.q[row + at(i, j)] = (int8_t)c[j];
      if (i == 0 && t == 0) a.scales[blockIdx.x] = s;
    }
  }
}

template <bool XBF16, bool VEC>
static hipError_t norm_go(const NormArgs& a, uint32_t n, hipStream_t st) {
  const uint32_t eights = (a.hidden + 7) / 8, v = (eights + kNormThreads - 1) / kNormThreads;
  auto go = [&](auto fn) {
    hipLaunchKernelGGL(fn, dim3(n), dim3(kNormThreads), 0, st, a);
    return hipGetLastError();
  };
  if (v <= 1) return go(k_rmsnorm<XBF16, 1, VEC>);
  if (v <= 2) return go(k_rmsnorm<XBF16, 2, VEC>);
  if (v <= 4) return go(k_rmsnorm<XBF16, 4, VEC>);
  return go(k_rmsnorm<XBF16, 8, VEC>);
}

hipError_t launch_rmsnorm(const NormArgs& a, bool x_bf16, uint32_t n, hipStream_t st) {
  if (a.hidden % 8 == 0) return x_bf16 ? norm_go<true, true>(a, n, st) : norm_go<false, true>(a, n, st);
  return x_bf16 ? norm_go<true, false>(a, n, st) : norm_go<false, false>(a, n, st);
}

}  // namespace smoe
