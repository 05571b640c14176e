// The decoder's linear layer with 4-bit weights: y[M, N] = x[M, K] . W[N, K]^T (+ bias) (+ residual),
//   W[n, k] = (u - 8) * scale[n, k / group],  u = 4 bits.
// Storage: K is padded to a multiple of 128 (padding u = 8); of every 128 weights of a row, 32-bit word 4 t + i holds
// elements 32 i + 8 t .. + 7, element 2 j in bits 4 j and element 2 j + 1 in bits 4 (j + 4).
//
// A few rows: bound by the weights' bytes, and, since half a byte is a weight, nearly as much by the instructions that
// take them apart.  A warp owns 16 features and reads 128 weights of each at a time as 16-byte pieces, straight into
// registers: lane (g, t) = (lane / 4, lane % 4) has words 4 t .. 4 t + 3 of features g and g + 8, which is what the A
// operand of mma.m16n8k16 wants from it for four groups of 32 weights.  A word becomes four pairs of bf16 with a shift,
// a mask and one fused add each: bits u placed under the exponent of 128 are 128 + u, minus 136 is the weight, exactly.
// x is the B operand, eight rows a tile: bf16 rows as they lie, f32 rows cut into three bf16 pieces (8 + 8 + 8 bits) that
// add up to the value.  Products are exact and their sums fp32; a group's sum is multiplied by its scale in fp32.
// K is split over the warps of a CTA when there are too few features to fill the SMs; the partial sums meet in shared
// memory in a fixed order.
#pragma once
#include "common.cuh"
#include "gemv_mma.cuh"

namespace wdz {

struct GemvPackedParams {
  const void* x; int64_t ldx;
  const uint32_t* W;       // [N][Kp / 8]
  const bf16* scale;       // [N][Kp / group]
  const void* bias;        // x's type, or nullptr
  const float* residual;   // f32 [M, N], or nullptr; may be y
  float* y;
  int M, N, K, Kp, group;
  int split;               // warps that share a tile of 16 features
  bool vec;                // rows of x can be read in pieces of eight
};

constexpr int GP_WARPS = 8;
constexpr int GP_AHEAD = 4;   // segments of 128 weights that a warp has under way

// One 32-bit word of weights -> pairs (element 2 j, element 2 j + 1), j = 0..3, as bf16.
__device__ __forceinline__ void gp_unpack(uint32_t w, uint32_t (&r)[4]) {
  const __nv_bfloat162 off = __halves2bfloat162(__float2bfloat16_rn(-136.0f), __float2bfloat16_rn(-136.0f));
  const __nv_bfloat162 one = __halves2bfloat162(__float2bfloat16_rn(1.0f), __float2bfloat16_rn(1.0f));
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t u = ((w >> (4 * j)) & 0x000f000fu) | 0x43004300u;
    const __nv_bfloat162 v = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&u), one, off);
    r[j] = *reinterpret_cast<const uint32_t*>(&v);
  }
}

// Eight neighbouring values of a row of x from k0 on, zeros behind its end, as pairs of bf16 (PIECES of them a value).
template <typename T, int PIECES>
__device__ __forceinline__ void gp_row(const T* row, int k0, int K, bool vec, uint32_t (&b)[PIECES][4]);
template <>
__device__ __forceinline__ void gp_row<bf16, 1>(const bf16* row, int k0, int K, bool vec, uint32_t (&b)[1][4]) {
  if (vec) {
    uint4 v = make_uint4(0, 0, 0, 0);
    if (k0 < K) v = __ldg(reinterpret_cast<const uint4*>(row + k0));
    b[0][0] = v.x; b[0][1] = v.y; b[0][2] = v.z; b[0][3] = v.w;
  } else {
    const uint16_t* r = reinterpret_cast<const uint16_t*>(row);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t lo = k0 + 2 * j < K ? r[k0 + 2 * j] : 0, hi = k0 + 2 * j + 1 < K ? r[k0 + 2 * j + 1] : 0;
      b[0][j] = lo | hi << 16;
    }
  }
}
template <>
__device__ __forceinline__ void gp_row<float, 3>(const float* row, int k0, int K, bool vec, uint32_t (&b)[3][4]) {
  float v[8];
  if (vec) {
    float4 lo = make_float4(0, 0, 0, 0), hi = lo;
    if (k0 < K) { lo = __ldg(reinterpret_cast<const float4*>(row + k0)); hi = __ldg(reinterpret_cast<const float4*>(row + k0 + 4)); }
    v[0] = lo.x; v[1] = lo.y; v[2] = lo.z; v[3] = lo.w; v[4] = hi.x; v[5] = hi.y; v[6] = hi.z; v[7] = hi.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = k0 + i < K ? row[k0 + i] : 0.0f;
  }
#pragma unroll
  for (int piece = 0; piece < 3; ++piece) {   // the upper 16 bits of what is left, cut off, not rounded: nothing overflows
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t x0 = __float_as_uint(v[2 * j]), x1 = __float_as_uint(v[2 * j + 1]);
      b[piece][j] = __byte_perm(x0, x1, 0x7632);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float top = __uint_as_float(__float_as_uint(v[i]) & 0xffff0000u);
      v[i] = fabsf(v[i]) == INFINITY ? 0.0f : v[i] - top;
    }
  }
}

// Block = 8 warps; grid = (tiles of 16 features x split / 8, rows / (8 NT)).  GS: scales of a segment of 128 weights.
template <typename T, int NT, int GS>
__global__ void __launch_bounds__(GP_WARPS * 32) gemv_packed_kernel(GemvPackedParams p) {
  constexpr int PIECES = sizeof(T) == 2 ? 1 : 3;
  __shared__ float red[GP_WARPS][8 * NT][17];
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int part = warp % p.split, tile = blockIdx.x * (GP_WARPS / p.split) + warp / p.split;
  const int m0 = blockIdx.y * 8 * NT, segs = p.Kp >> 7;
  const int na = min(tile * 16 + g, p.N - 1), nb = min(tile * 16 + g + 8, p.N - 1);
  const uint4* wa = reinterpret_cast<const uint4*>(p.W + (int64_t)na * (p.Kp >> 3)) + t;   // a segment is four uint4
  const uint4* wb = reinterpret_cast<const uint4*>(p.W + (int64_t)nb * (p.Kp >> 3)) + t;
  const bf16* sa = p.scale + (int64_t)na * segs * GS;
  const bf16* sb = p.scale + (int64_t)nb * segs * GS;
  pdl_wait();

  float acc[NT][4];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = 0.0f;

  for (int base = part; base < segs; base += GP_AHEAD * p.split) {
    uint4 a[GP_AHEAD], b[GP_AHEAD];
    float fa[GP_AHEAD][GS], fb[GP_AHEAD][GS];
#pragma unroll
    for (int u = 0; u < GP_AHEAD; ++u) {
      const int sg = min(base + u * p.split, segs - 1);   // the last ones are read again and left out below
      a[u] = __ldg(wa + 4 * sg);
      b[u] = __ldg(wb + 4 * sg);
#pragma unroll
      for (int i = 0; i < GS; ++i) { fa[u][i] = to_f(sa[sg * GS + i]); fb[u][i] = to_f(sb[sg * GS + i]); }
    }
#pragma unroll
    for (int u = 0; u < GP_AHEAD; ++u) {
      const int sg = base + u * p.split;
      if (sg < segs) {
        const uint32_t* aw = reinterpret_cast<const uint32_t*>(&a[u]);
        const uint32_t* bw = reinterpret_cast<const uint32_t*>(&b[u]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t ra[4], rb[4];
          gp_unpack(aw[i], ra);
          gp_unpack(bw[i], rb);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const int m = m0 + 8 * nt + g;
            uint32_t xb[PIECES][4] = {};
            if (m < p.M) gp_row<T, PIECES>(reinterpret_cast<const T*>(p.x) + (int64_t)m * p.ldx, sg * 128 + 32 * i + 8 * t, p.K, p.vec, xb);
            float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int q = PIECES - 1; q >= 0; --q) {
              mma_bf16_16816(c, ra[0], rb[0], ra[1], rb[1], xb[q][0], xb[q][1]);
              mma_bf16_16816(c, ra[2], rb[2], ra[3], rb[3], xb[q][2], xb[q][3]);
            }
            acc[nt][0] = fmaf(fa[u][i * GS / 4], c[0], acc[nt][0]);
            acc[nt][1] = fmaf(fa[u][i * GS / 4], c[1], acc[nt][1]);
            acc[nt][2] = fmaf(fb[u][i * GS / 4], c[2], acc[nt][2]);
            acc[nt][3] = fmaf(fb[u][i * GS / 4], c[3], acc[nt][3]);
          }
        }
      }
    }
  }
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    red[warp][8 * nt + 2 * t][g] = acc[nt][0];
    red[warp][8 * nt + 2 * t + 1][g] = acc[nt][1];
    red[warp][8 * nt + 2 * t][g + 8] = acc[nt][2];
    red[warp][8 * nt + 2 * t + 1][g + 8] = acc[nt][3];
  }
  __syncthreads();
  const int rows = min(8 * NT, p.M - m0), cols = 16 * (GP_WARPS / p.split), n_first = blockIdx.x * cols;
  for (int i = threadIdx.x; i < rows * cols; i += GP_WARPS * 32) {
    const int row = i / cols, col = i % cols, n = n_first + col;
    if (n >= p.N) continue;
    float v = 0.0f;
    for (int w = 0; w < p.split; ++w) v += red[(col >> 4) * p.split + w][row][col & 15];
    if (p.bias) v += to_f(reinterpret_cast<const T*>(p.bias)[n]);
    const int64_t at = (int64_t)(m0 + row) * p.N + n;
    if (p.residual) v += p.residual[at];
    p.y[at] = v;
  }
}

}  // namespace wdz
