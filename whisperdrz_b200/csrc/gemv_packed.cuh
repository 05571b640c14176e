// The decoder's linear layer with 4-bit weights: y[M, N] = x[M, K] . W[N, K]^T (+ bias) (+ residual),
//   W[n, k] = (u - 8) * scale[n, k / group],  u = 4 bits.
// Storage: K is padded to a multiple of 128 (padding u = 8); of every 128 weights of a row, 32-bit word 4 t + i holds
// elements 32 i + 8 t .. + 7, element 2 j in bits 4 j and element 2 j + 1 in bits 4 (j + 4).
#pragma once
#include "common.cuh"

namespace wdz {

struct GemvPackedParams {
  const void* x; int64_t ldx;
  const uint32_t* W;       // [N][Kp / 8]
  const bf16* scale;       // [N][Kp / group]
  const void* bias;        // x's type, or nullptr
  const float* residual;   // f32 [M, N], or nullptr; may be y
  float* y;
  int M, N, K, Kp, group;
};

// A warp per output feature.
template <typename T>
__global__ void __launch_bounds__(128) gemv_packed_kernel(GemvPackedParams p) {
  pdl_trigger();
  pdl_wait();
  const int n = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (n >= p.N) return;
  const T* x = reinterpret_cast<const T*>(p.x);
  for (int m = 0; m < p.M; ++m) {
    float acc = 0.0f;
    for (int wi = lane; wi < p.Kp / 8; wi += 32) {
      const uint32_t w = p.W[(int64_t)n * (p.Kp / 8) + wi];
      const int k0 = (wi >> 4) * 128 + 32 * (wi & 3) + 8 * ((wi & 15) >> 2);
      const float s = to_f(p.scale[(int64_t)n * (p.Kp / p.group) + k0 / p.group]);
      float part = 0.0f;
      for (int j = 0; j < 8; ++j) {
        const int k = k0 + 2 * (j & 3) + (j >> 2);
        if (k < p.K) part = fmaf((float)((int)((w >> (4 * j)) & 15) - 8), to_f(x[(int64_t)m * p.ldx + k]), part);
      }
      acc = fmaf(part, s, acc);
    }
    acc = warp_sum(acc);
    if (lane == 0) {
      if (p.bias) acc += to_f(reinterpret_cast<const T*>(p.bias)[n]);
      if (p.residual) acc += p.residual[(int64_t)m * p.N + n];
      p.y[(int64_t)m * p.N + n] = acc;
    }
  }
}

}  // namespace wdz
