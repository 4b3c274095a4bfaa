// Products of a few rows with 4-bit weights:
//   out[m, n] = act( sum_g s[n, g] * sum_{k in g} (q[n, k] - z[n, g]) * x[m, k] + bias[n] )
// with codes q in 0..15 packed two to a byte (the even column in the low half), a scale s and,
// where given, a zero point z for each group of 32, 64 or 128 columns of a row (z = 8 otherwise).
#pragma once
#include "common.cuh"

namespace s1c {

struct NibbleArgs {
  const void* x;
  const uint8_t* codes;
  const void* scales;
  const void* zeros;  // nullable: 8
  void* out;
  const float* bias;  // nullable
  int64_t x_stride, pitch, scale_stride, out_stride;
  int M, N, K, group, act, out_f32;
};

S1C_DEV float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
S1C_DEV float to_f32(__half v) { return __half2float(v); }
S1C_DEV float to_f32(float v) { return v; }
template <typename T>
S1C_DEV T from_f32(float v);
template <>
S1C_DEV __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
S1C_DEV __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
S1C_DEV float from_f32<float>(float v) { return v; }

// The epilogue of one output: bias, activation (0 none, 1 ReLU, 2 GELU with erf), one rounding.
template <typename T>
S1C_DEV void nibble_store(const NibbleArgs& a, int m, int n, float v) {
  if (a.bias) v += a.bias[n];
  if (a.act == 1) v = v < 0.f ? 0.f : v;  // keeps NaN
  if (a.act == 2) v = 0.5f * v * (1.f + erff(v * 0.70710678118654752f));
  const int64_t at = m * a.out_stride + n;
  if (a.out_f32)
    static_cast<float*>(a.out)[at] = v;
  else
    static_cast<T*>(a.out)[at] = from_f32<T>(v);
}

// One warp for each row of the weights, eight rows of x at a time; a lane takes every 32nd word of
// eight codes, so no word straddles a group.
template <typename T>
__global__ void __launch_bounds__(256) nibble_kernel(const NibbleArgs a) {
  const int n = blockIdx.x * 8 + threadIdx.x / 32, lane = threadIdx.x % 32;
  if (n >= a.N) return;
  const T* x = static_cast<const T*>(a.x);
  const T* scales = static_cast<const T*>(a.scales) + n * a.scale_stride;
  const T* zeros = a.zeros ? static_cast<const T*>(a.zeros) + n * a.scale_stride : nullptr;
  const uint32_t* codes = reinterpret_cast<const uint32_t*>(a.codes + n * a.pitch);
  for (int m0 = 0; m0 < a.M; m0 += 8) {
    float acc[8] = {};
    for (int w = lane; 8 * w < a.K; w += 32) {
      const uint32_t word = codes[w];
      const int g = 8 * w / a.group;
      const float s = to_f32(scales[g]), z = zeros ? to_f32(zeros[g]) : 8.f;
      for (int j = 0; j < 8 && 8 * w + j < a.K; ++j) {
        const float v = s * ((float)((word >> (4 * j)) & 15u) - z);
#pragma unroll
        for (int m = 0; m < 8; ++m)
          if (m0 + m < a.M) acc[m] += v * to_f32(x[(m0 + m) * a.x_stride + 8 * w + j]);
      }
    }
#pragma unroll
    for (int m = 0; m < 8; ++m) {
      for (int o = 16; o; o >>= 1) acc[m] += __shfl_xor_sync(0xffffffffu, acc[m], o);
      if (lane == m && m0 + m < a.M) nibble_store<T>(a, m0 + m, n, acc[m]);
    }
  }
}

}  // namespace s1c
