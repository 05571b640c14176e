// The decoder's linear layer with 4-bit weights: y[M, N] = x[M, K] . W[N, K]^T (+ bias) (+ residual),
//   W[n, k] = (u - 8) * scale[n, k / group],  u = 4 bits.
// Storage: K is padded to a multiple of 128 (padding u = 8); of every 128 weights of a row, 32-bit word 4 t + i holds
// elements 32 i + 8 t .. + 7, element 2 j in bits 4 j and element 2 j + 1 in bits 4 (j + 4).
//
// A few rows: bound by the weights' bytes, and, since half a byte is a weight, nearly as much by the instructions that
// take them apart.  A warp owns 16 features and reads 128 weights of each at a time as 16-byte pieces, straight into
// registers: lane (g, t) = (lane / 4, lane % 4) has words 4 t .. 4 t + 3 of features g and g + 8, which is what the A
// operand of a matrix instruction wants from it for four groups of 32 weights.  K is split over the warps of a CTA when
// there are too few features to fill the SMs; the partial sums meet in shared memory in a fixed order.
//
//   gemv_packed_s8_kernel    bf16 rows, up to two.  m16n8k32 on bytes: a word becomes two operands with three
//       instructions (a nibble in a byte's upper half is 16 times a signed weight).  x is written as a whole number of
//       48 bits times a power of two of its row, six signed bytes that take six columns: exact for values down to 2^-38 of
//       the row's largest, off by at most 2^-46 of that below.  Sums of products of bytes are exact.
//   gemv_packed_mma_kernel   all others.  m16n8k16 on bf16.  A word becomes four pairs of bf16 with a shift, a mask and one
//       fused add each: bits u placed under the exponent of 128 are 128 + u, minus 136 is the weight, exactly.  A bf16 row
//       is one column, as it is; an f32 row is cut into three bf16 pieces (8 + 8 + 8 bits) that add up to it, as far down as
//       bf16 goes (2^-133), and take three.
// Either way a group's sum is multiplied by its scale in fp32.
//
// Measured (B200, device time): one bf16 row, 1280 x 1280 3.0 us (a launch's latency; the weights' bytes alone 0.13); one row
// over 51866 x 1280 9.1 us, 3.8 TB/s, and 11.7 us for three on bf16 operands (88 instructions against 24 to take 64 weights
// apart); 16 rows, 5120 -> 1280 6.0 us; five f32 rows, 1237 -> 5003 7.2 us.
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
  int split, split_log;    // warps that share a tile of 16 features: 1, 2, 4 or 8
  bool vec;                // rows of x can be read in pieces of eight
  int chunk;               // segments of x that one pass of gemv_packed_mma_kernel keeps in shared memory
};

constexpr int GP_WARPS = 8;
constexpr int GP_AHEAD = 2;   // segments of 128 weights that a warp of the byte kernel has under way (3: 0.7 us slower at 51866 features, fewer warps)

__device__ __forceinline__ void mma_s8_16832(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The same with an accumulator of zeros.
__device__ __forceinline__ void mma_s8_16832_first(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
               : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(0));
}

// bf16 product whose accumulator starts from zeros.
__device__ __forceinline__ void mma_bf16_16816_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
               : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}

// One 32-bit word of weights -> pairs (element 2 j, element 2 j + 1), j = 0..3, as bf16.  low = 0x000f000f, base = 128 twice:
// both in registers, so that mask and exponent are one instruction.
__device__ __forceinline__ void gp_unpack(uint32_t w, uint32_t low, uint32_t base, uint32_t (&r)[4]) {
  const __nv_bfloat162 off = __halves2bfloat162(__float2bfloat16_rn(-136.0f), __float2bfloat16_rn(-136.0f));
  const __nv_bfloat162 one = __halves2bfloat162(__float2bfloat16_rn(1.0f), __float2bfloat16_rn(1.0f));
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t u;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(u) : "r"(w >> (4 * j)), "r"(low), "r"(base));   // (w & low) | base
    const __nv_bfloat162 v = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&u), one, off);
    r[j] = *reinterpret_cast<const uint32_t*>(&v);
  }
}

// Eight neighbouring values of a row of x from k0 on, zeros behind its end.
__device__ __forceinline__ uint4 gp_row(const bf16* row, int k0, int K, bool vec) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (vec) {
    if (k0 < K) v = *reinterpret_cast<const uint4*>(row + k0);   // plain loads: the kernel before may have written x
    return v;
  }
  // rows at any two bytes: the words that hold the values, shifted by half a word where they start in the middle of one.
  // A word is only read where a value of the row lies in it, so it lies in the row's allocation.
  const uint32_t half = (uint32_t)((uintptr_t)(row + k0) & 2) >> 1;
  const uint32_t* w = reinterpret_cast<const uint32_t*>((uintptr_t)(row + k0) & ~(uintptr_t)3);
  uint32_t in[5], out[4];
#pragma unroll
  for (int j = 0; j < 5; ++j) in[j] = k0 + 2 * j - (int)half < K && (j < 4 || half) && k0 < K ? w[j] : 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    out[j] = half ? __funnelshift_r(in[j], in[j + 1], 16) : in[j];
    if (k0 + 2 * j + 1 >= K) out[j] = k0 + 2 * j < K ? out[j] & 0xffffu : 0;
  }
  return make_uint4(out[0], out[1], out[2], out[3]);
}
__device__ __forceinline__ void gp_row8(const bf16* row, int k0, int K, bool vec, float (&v)[8]) {
  const uint4 u = gp_row(row, k0, K, vec);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
}
__device__ __forceinline__ void gp_row8(const float* row, int k0, int K, bool vec, float (&v)[8]) {
  if (vec) {
    float4 lo = make_float4(0, 0, 0, 0), hi = lo;
    if (k0 < K) { lo = *reinterpret_cast<const float4*>(row + k0); hi = *reinterpret_cast<const float4*>(row + k0 + 4); }
    v[0] = lo.x; v[1] = lo.y; v[2] = lo.z; v[3] = lo.w; v[4] = hi.x; v[5] = hi.y; v[6] = hi.z; v[7] = hi.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = k0 + i < K ? row[k0 + i] : 0.0f;
  }
}

// The scales of one segment of a feature, GS of them.
template <int GS> struct GpScale;
template <> struct GpScale<1> {
  uint32_t v;
  __device__ void load(const bf16* p) { v = *reinterpret_cast<const uint16_t*>(p); }
  __device__ float get(int) const { return __uint_as_float(v << 16); }
};
template <> struct GpScale<2> {
  uint32_t v;
  __device__ void load(const bf16* p) { v = __ldg(reinterpret_cast<const uint32_t*>(p)); }
  __device__ float get(int i) const { return __uint_as_float(i & 1 ? v & 0xffff0000u : v << 16); }
};
template <> struct GpScale<4> {
  uint2 v;
  __device__ void load(const bf16* p) { v = __ldg(reinterpret_cast<const uint2*>(p)); }
  __device__ float get(int i) const { const uint32_t w = i & 2 ? v.y : v.x; return __uint_as_float(i & 1 ? w & 0xffff0000u : w << 16); }
};

// The 16 features' sums of `split` warps, plus bias and residual, for rows m0 .. m0 + rows.
template <typename T, int ROWS>
__device__ __forceinline__ void gp_finish(const GemvPackedParams& p, const float (&red)[GP_WARPS][ROWS][17], int m0) {
  const int rows = min(ROWS, p.M - m0), shift = 7 - p.split_log, cols = 1 << shift, n_first = blockIdx.x << shift;
  for (int i0 = threadIdx.x; i0 < rows << shift; i0 += 4 * GP_WARPS * 32) {   // four loads of bias and residual at a time
    float v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = i0 + k * GP_WARPS * 32, n = n_first + (i & (cols - 1));
      v[k] = 0.0f;
      if (i < rows << shift && n < p.N) {
        if (p.residual) v[k] = p.residual[(int64_t)(m0 + (i >> shift)) * p.N + n];
        if (p.bias) v[k] += to_f(reinterpret_cast<const T*>(p.bias)[n]);
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = i0 + k * GP_WARPS * 32, row = i >> shift, col = i & (cols - 1), n = n_first + col;
      if (i >= rows << shift || n >= p.N) continue;
      float sum = 0.0f;
      for (int w = 0; w < p.split; ++w) sum += red[((col >> 4) << p.split_log) + w][row][col & 15];
      p.y[(int64_t)(m0 + row) * p.N + n] = v[k] + sum;
    }
  }
}

// The byte kernel: segments of x that one pass keeps in shared memory (64 KB).
template <int ROWS> constexpr int GP_S8_CHUNK = ROWS == 1 ? 64 : 32;

// The upper nibbles u of four bytes as 16 (u - 8): one instruction with both masks in registers.
__device__ __forceinline__ uint32_t gp_signed16(uint32_t w, uint32_t flip, uint32_t keep) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0x28;" : "=r"(r) : "r"(w), "r"(flip), "r"(keep));   // (w ^ flip) & keep
  return r;
}

// What whole numbers cannot give, value by value in 64 bits: the lane's share for its two features.
//   odd   rows with infinities or NaN, which have no whole number.  Such a row is infinite or NaN in every feature, whatever its
//         other values are: only these are multiplied.
//   !odd  rows whose sum is not finite: a group's whole number, up to 2^29, times its scale leaves fp32 where the scale is large
//         and x so small that the result need not (x of 1e-20 under scales of 1e33).
// A function of its own, which works out its place anew: as a loop in the kernel the first kind costs rows without any 0.2 to
// 0.4 us of 9.1 (51866 features), and a power of two ahead of the scale instead of the second 0.1 us, of two rows up to 1.2 of 10.9.
template <int GS>
__device__ __noinline__ float2 gp_by_value(const GemvPackedParams& p, int m, bool odd) {
  const int warp = threadIdx.x >> 5, g = (threadIdx.x & 31) >> 2, t = threadIdx.x & 3;
  const int tile = blockIdx.x * (GP_WARPS >> p.split_log) + (warp >> p.split_log), segs = p.Kp >> 7;
  const int64_t na = min(tile * 16 + g, p.N - 1), nb = min(tile * 16 + g + 8, p.N - 1);
  const bf16* x = reinterpret_cast<const bf16*>(p.x) + m * p.ldx;
  double sum[2] = {0.0, 0.0};
  for (int sg = warp & (p.split - 1); sg < segs; sg += p.split)
#pragma unroll 1
    for (int i = 0; i < 32; ++i) {
      const int k = sg * 128 + 32 * (i >> 3) + 8 * t + (i & 7), bit = 4 * ((i & 7) >> 1) + 16 * (i & 1);
      if (k >= p.K) break;   // the rest of these eight, and of the segment, lies behind the row too
      const float v = to_f(x[k]);
      if (odd && fabsf(v) <= 3.402823466e38f) continue;
      const int word = 16 * sg + 4 * t + (i >> 3), f = sg * GS + i / (32 / GS);
      const int ua = p.W[na * (p.Kp >> 3) + word] >> bit & 15, ub = p.W[nb * (p.Kp >> 3) + word] >> bit & 15;
      sum[0] += (double)v * ((ua - 8) * (double)to_f(p.scale[na * segs * GS + f]));
      sum[1] += (double)v * ((ub - 8) * (double)to_f(p.scale[nb * segs * GS + f]));
    }
  return make_float2((float)sum[0], (float)sum[1]);
}

// Block = 8 warps; grid = tiles of 16 features x split / 8.  ROWS = M, 1 or 2.  GS: scales of a segment of 128 weights.
template <int ROWS, int GS>
__global__ void __launch_bounds__(GP_WARPS * 32, 3) gemv_packed_s8_kernel(const __grid_constant__ GemvPackedParams p) {
  extern __shared__ __align__(16) uint2 xs[];   // [segment][row][i][lane]: a lane's two operand words
  __shared__ float red[GP_WARPS][ROWS][17];
  __shared__ float tops[GP_WARPS][ROWS];
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int part = warp & (p.split - 1), tile = blockIdx.x * (GP_WARPS >> p.split_log) + (warp >> p.split_log);
  const int segs = p.Kp >> 7;
  const int na = min(tile * 16 + g, p.N - 1), nb = min(tile * 16 + g + 8, p.N - 1);
  const uint4* wa = reinterpret_cast<const uint4*>(p.W + (int64_t)na * (p.Kp >> 3)) + t;   // a segment is four uint4
  const uint4* wb = reinterpret_cast<const uint4*>(p.W + (int64_t)nb * (p.Kp >> 3)) + t;
  const bf16* sa = p.scale + (int64_t)na * segs * GS;
  const bf16* sb = p.scale + (int64_t)nb * segs * GS;
  const bf16* x = reinterpret_cast<const bf16*>(p.x);
  pdl_wait();

  float sum[ROWS][2];
#pragma unroll
  for (int m = 0; m < ROWS; ++m) sum[m][0] = sum[m][1] = 0.0f;
  uint32_t odd = 0;   // bit m: row m holds infinities or NaN
  // columns 6 and 7 take the operands of 4 and 5 once more; what they give is left out below
  const uint32_t xs_mine = (uint32_t)__cvta_generic_to_shared(xs) + 8 * ((g < 6 ? g : g - 2) * 4 + t);
  constexpr int CHUNK = GP_S8_CHUNK<ROWS>;
  for (int first = 0; first < segs; first += CHUNK) {
    const int here = min(CHUNK, segs - first);
    const int n = part < here ? (here - part + p.split - 1) >> p.split_log : 0;   // segments of this warp
    uint4 a[GP_AHEAD], b[GP_AHEAD];
    GpScale<GS> fa[GP_AHEAD], fb[GP_AHEAD];
    auto fetch = [&](int u, int j) {
      const int sg = first + part + (j << p.split_log);
      a[u] = __ldg(wa + 4 * sg);
      b[u] = __ldg(wb + 4 * sg);
      fa[u].load(sa + sg * GS);
      fb[u].load(sb + sg * GS);
    };
#pragma unroll
    for (int u = 0; u < GP_AHEAD; ++u) if (u < n) fetch(u, u);   // under way while x is taken apart

    // largest value of each row, 8 values a thread and step
    const int units = here * 16;
    float top[ROWS];
#pragma unroll
    for (int m = 0; m < ROWS; ++m) {
      top[m] = 0.0f;
      for (int i = threadIdx.x; i < units; i += GP_WARPS * 32) {
        float v[8];
        gp_row8(x + m * p.ldx, first * 128 + 8 * i, p.K, p.vec, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) top[m] = fabsf(v[j]) <= 3.402823466e38f ? fmaxf(top[m], fabsf(v[j])) : INFINITY;
      }
    }
    __syncthreads();   // the pass before has read xs and tops
#pragma unroll
    for (int m = 0; m < ROWS; ++m) {
      top[m] = warp_max(top[m]);
      if (lane == 0) tops[warp][m] = top[m];
    }
    __syncthreads();
#pragma unroll
    for (int m = 0; m < ROWS; ++m) {
#pragma unroll
      for (int w = 0; w < GP_WARPS; ++w) top[m] = fmaxf(top[m], tops[w][m]);
      // x in units of 2^(e - 45), e the exponent of the largest: whole numbers below 2^46, exact down to 2^(e - 38)
      const int e = max((int)(__float_as_uint(top[m]) >> 23), 1) - 127;
      const double unit = top[m] < INFINITY ? __hiloint2double((1023 + 45 - e) << 20, 0) : 0.0;
      for (int i = threadIdx.x; i < units; i += GP_WARPS * 32) {
        float v[8];
        gp_row8(x + m * p.ldx, first * 128 + 8 * i, p.K, p.vec, v);
        // i = word of lane tt of a segment; the bytes' lower nibbles are elements 0 4 1 5, the upper 2 6 3 7
        const int sg = i >> 4, wi = i & 15, at = wi >> 2, tt = wi & 3;
        uint32_t lo[8], hi[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint64_t w = unit > 0.0 ? (uint64_t)__double2ll_rn((double)v[j] * unit) + 0x808080808080ull : 0x808080808080ull;   // bytes + 128
          lo[j] = (uint32_t)w; hi[j] = (uint32_t)(w >> 32);
        }
        uint2 d[6];   // columns d1, d0, d3, d2, d5, d4
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int e0 = 2 * h, e1 = 2 * h + 4, e2 = 2 * h + 1, e3 = 2 * h + 5;
          const uint32_t x01 = __byte_perm(lo[e0], lo[e1], 0x5140), x23 = __byte_perm(lo[e2], lo[e3], 0x5140);
          const uint32_t y01 = __byte_perm(lo[e0], lo[e1], 0x7362), y23 = __byte_perm(lo[e2], lo[e3], 0x7362);
          const uint32_t z01 = __byte_perm(hi[e0], hi[e1], 0x5140), z23 = __byte_perm(hi[e2], hi[e3], 0x5140);
          (h ? d[0].y : d[0].x) = __byte_perm(x01, x23, 0x7632) ^ 0x80808080u;
          (h ? d[1].y : d[1].x) = __byte_perm(x01, x23, 0x5410) ^ 0x80808080u;
          (h ? d[2].y : d[2].x) = __byte_perm(y01, y23, 0x7632) ^ 0x80808080u;
          (h ? d[3].y : d[3].x) = __byte_perm(y01, y23, 0x5410) ^ 0x80808080u;
          (h ? d[4].y : d[4].x) = __byte_perm(z01, z23, 0x7632) ^ 0x80808080u;
          (h ? d[5].y : d[5].x) = __byte_perm(z01, z23, 0x5410) ^ 0x80808080u;
        }
#pragma unroll
        for (int q = 0; q < 6; ++q) xs[((sg * ROWS + m) * 4 + at) * 32 + q * 4 + tt] = d[q];
      }
    }
    __syncthreads();

    float acc[ROWS][2];
#pragma unroll
    for (int m = 0; m < ROWS; ++m) acc[m][0] = acc[m][1] = 0.0f;
    uint32_t flip = 0x80808080u, keep = 0xf0f0f0f0u;
    asm volatile("" : "+r"(flip), "+r"(keep));   // known to nobody: they stay in registers
    uint32_t xq = xs_mine + part * (ROWS * 1024);
    for (int j = 0; j < n; j += GP_AHEAD) {
#pragma unroll
      for (int u = 0; u < GP_AHEAD; ++u) {
        if (j + u >= n) break;
        uint32_t op[4][4];
        const uint32_t aw[4] = {a[u].x, a[u].y, a[u].z, a[u].w}, bw[4] = {b[u].x, b[u].y, b[u].z, b[u].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          op[i][0] = gp_signed16(aw[i] << 4, flip, keep);
          op[i][1] = gp_signed16(bw[i] << 4, flip, keep);
          op[i][2] = gp_signed16(aw[i], flip, keep);
          op[i][3] = gp_signed16(bw[i], flip, keep);
        }
        float sa_g[GS], sb_g[GS];
#pragma unroll
        for (int i = 0; i < GS; ++i) { sa_g[i] = fa[u].get(i); sb_g[i] = fb[u].get(i); }
        if (j + u + GP_AHEAD < n) fetch(u, j + u + GP_AHEAD);
#pragma unroll
        for (int m = 0; m < ROWS; ++m) {
          int c[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint2 xb;
            asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(xb.x), "=r"(xb.y) : "r"(xq + 1024 * m + 256 * i) : "memory");
            if (i % (4 / GS) == 0) mma_s8_16832_first(c, op[i][0], op[i][1], op[i][2], op[i][3], xb.x, xb.y);
            else mma_s8_16832(c, op[i][0], op[i][1], op[i][2], op[i][3], xb.x, xb.y);
            if ((i + 1) % (4 / GS) == 0) {   // the end of a group: columns (d1, d0), (d3, d2) or (d5, d4) fold into one number
              acc[m][0] = fmaf((float)(c[0] * 256 + c[1]), sa_g[i / (4 / GS)], acc[m][0]);
              acc[m][1] = fmaf((float)(c[2] * 256 + c[3]), sb_g[i / (4 / GS)], acc[m][1]);
            }
          }
        }
        xq += (ROWS * 1024) << p.split_log;
      }
    }
    // times 2^-45 of the unit, 2^-4 of the shifted nibble and the column's 2^16 t; the row's own size last, so that nothing
    // underflows before the result does.
    const float column = t == 0 ? 1.7763568394002505e-15f : t == 1 ? 1.1641532182693481e-10f : t == 2 ? 7.62939453125e-6f : 0.0f;
#pragma unroll
    for (int m = 0; m < ROWS; ++m) {
      const float size = top[m] < INFINITY ? ldexpf(1.0f, max((int)(__float_as_uint(top[m]) >> 23), 1) - 127) : 0.0f;
      sum[m][0] = fmaf(acc[m][0] * column, size, sum[m][0]);
      sum[m][1] = fmaf(acc[m][1] * column, size, sum[m][1]);
      odd |= top[m] == INFINITY ? 1u << m : 0u;
    }
  }
#pragma unroll
  for (int m = 0; m < ROWS; ++m)
    if (__any_sync(0xffffffffu, odd >> m & 1 || !(fabsf(sum[m][0]) + fabsf(sum[m][1]) <= 3.402823466e38f))) {
      const float2 v = gp_by_value<GS>(p, m, odd >> m & 1);
      sum[m][0] = v.x;
      sum[m][1] = v.y;
    }
#pragma unroll
  for (int m = 0; m < ROWS; ++m)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float v = sum[m][h] + __shfl_xor_sync(0xffffffffu, sum[m][h], 1);
      v += __shfl_xor_sync(0xffffffffu, v, 2);
      if (t == 0) red[warp][m][g + 8 * h] = v;
    }
  __syncthreads();
  gp_finish<bf16>(p, red, 0);
}

// Rows as bf16 operands.  A tile is the eight columns of an operand: eight bf16 rows, or two f32 rows of three pieces each (the
// fourth column is never written and never read).  x is brought into shared memory once a CTA, in the operand's order, so that
// rows of any alignment cost the loop nothing (value by value from global memory: 37 us instead of 9 for 7 rows, 1275 ->
// 47372).  FIT: CTAs that share an SM.  Three where that makes one wave of what would be two (7 rows over 47372 features: 13 us
// against 16), else two, whose registers save a third of the instructions (3 rows over 36319: 10 us against 13.5).
// Block = 8 warps; grid = (tiles of 16 features x split / 8, rows / rows of TILES tiles).
template <typename T> constexpr int GP_TILE_ROWS = sizeof(T) == 2 ? 8 : 2;

template <typename T, int TILES, int GS, int FIT>
__global__ void __launch_bounds__(GP_WARPS * 32, FIT) gemv_packed_mma_kernel(GemvPackedParams p) {
  constexpr int TILE_ROWS = GP_TILE_ROWS<T>, ROWS = TILES * TILE_ROWS;
  extern __shared__ __align__(16) uint4 xf[];   // [segment][tile][i][lane]: eight values of a lane's column
  __shared__ float red[GP_WARPS][ROWS][17];
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int part = warp & (p.split - 1), tile = blockIdx.x * (GP_WARPS >> p.split_log) + (warp >> p.split_log);
  const int m0 = blockIdx.y * ROWS, segs = p.Kp >> 7, rows = min(ROWS, p.M - m0);
  const int na = min(tile * 16 + g, p.N - 1), nb = min(tile * 16 + g + 8, p.N - 1);
  const uint4* wa = reinterpret_cast<const uint4*>(p.W + (int64_t)na * (p.Kp >> 3)) + t;   // a segment is four uint4
  const uint4* wb = reinterpret_cast<const uint4*>(p.W + (int64_t)nb * (p.Kp >> 3)) + t;
  const bf16* sa = p.scale + (int64_t)na * segs * GS;
  const bf16* sb = p.scale + (int64_t)nb * segs * GS;
  const T* x = reinterpret_cast<const T*>(p.x) + (int64_t)m0 * p.ldx;
  const uint32_t xf_mine = (uint32_t)__cvta_generic_to_shared(xf) + 16 * lane;
  pdl_wait();

  float acc[TILES][4];
#pragma unroll
  for (int q = 0; q < TILES; ++q)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[q][j] = 0.0f;
  for (int first = 0; first < segs; first += p.chunk) {
    const int here = min(p.chunk, segs - first);
    const int n = part < here ? (here - part + p.split - 1) >> p.split_log : 0;   // segments of this warp
    uint4 a[2], b[2];
    GpScale<GS> fa[2], fb[2];
    auto fetch = [&](int u, int j) {
      const int sg = first + part + (j << p.split_log);
      a[u] = __ldg(wa + 4 * sg);
      b[u] = __ldg(wb + 4 * sg);
      fa[u].load(sa + sg * GS);
      fb[u].load(sb + sg * GS);
    };
    if (n > 0) fetch(0, 0);
    if (n > 1) fetch(1, 1);
    __syncthreads();   // the pass before has read xf
    for (int unit = threadIdx.x; unit < here * 16; unit += GP_WARPS * 32) {   // of eight values, in every row
      uint4* to = xf + (((unit >> 4) * TILES * 4 + ((unit & 15) >> 2)) * 32 + (unit & 3));
      const int k0 = first * 128 + 8 * unit;
      if (sizeof(T) == 2 && p.vec) {   // as it lies: asynchronous copies, all under way at once
        for (int m = 0; m < rows; ++m)
          asm volatile("cp.async.ca.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(to + (m >> 3) * 128 + (m & 7) * 4)),
                       "l"(k0 < p.K ? x + (int64_t)m * p.ldx + k0 : x), "r"(k0 < p.K ? 16 : 0) : "memory");
      } else if constexpr (sizeof(T) == 2) {
#pragma unroll 4
        for (int m = 0; m < rows; ++m) to[(m >> 3) * 128 + (m & 7) * 4] = gp_row(x + (int64_t)m * p.ldx, k0, p.K, false);
      } else {
#pragma unroll 1
        for (int pair = 0; 2 * pair < rows; ++pair, to += 128) {
          float v[2][8];
#pragma unroll
          for (int k = 0; k < 2; ++k)
            if (2 * pair + k < rows) gp_row8(x + (int64_t)(2 * pair + k) * p.ldx, k0, p.K, p.vec, v[k]);
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            if (2 * pair + k >= rows) break;
#pragma unroll
            for (int q = 0; q < 3; ++q) {   // the upper 16 bits of what is left, cut off, not rounded: nothing overflows
              uint32_t w[4];
#pragma unroll
              for (int j = 0; j < 4; ++j) w[j] = __byte_perm(__float_as_uint(v[k][2 * j]), __float_as_uint(v[k][2 * j + 1]), 0x7632);
              to[16 * k + 4 * q] = make_uint4(w[0], w[1], w[2], w[3]);
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                const float cut = __uint_as_float(__float_as_uint(v[k][j]) & 0xffff0000u);
                v[k][j] = fabsf(v[k][j]) == INFINITY ? 0.0f : v[k][j] - cut;
              }
            }
          }
        }
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
    uint32_t low = 0x000f000fu, base = 0x43004300u;
    asm volatile("" : "+r"(low), "+r"(base));   // known to nobody: they stay in registers
    uint32_t xq = xf_mine + part * (TILES * 2048);
    for (int j = 0; j < n; j += 2) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (j + u >= n) break;
        const uint32_t aw[4] = {a[u].x, a[u].y, a[u].z, a[u].w}, bw[4] = {b[u].x, b[u].y, b[u].z, b[u].w};
        float c[TILES][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t ra[4], rb[4];
          gp_unpack(aw[i], low, base, ra);
          gp_unpack(bw[i], low, base, rb);
#pragma unroll
          for (int q = 0; q < TILES; ++q) {
            uint4 xb;
            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(xb.x), "=r"(xb.y), "=r"(xb.z), "=r"(xb.w) : "r"(xq + 2048 * q + 512 * i) : "memory");
            if (i % (4 / GS) == 0) mma_bf16_16816_first(c[q], ra[0], rb[0], ra[1], rb[1], xb.x, xb.y);
            else mma_bf16_16816(c[q], ra[0], rb[0], ra[1], rb[1], xb.x, xb.y);
            mma_bf16_16816(c[q], ra[2], rb[2], ra[3], rb[3], xb.z, xb.w);
            if ((i + 1) % (4 / GS) == 0) {   // the end of a group
              const float sa_g = fa[u].get(i / (4 / GS)), sb_g = fb[u].get(i / (4 / GS));
              acc[q][0] = fmaf(sa_g, c[q][0], acc[q][0]);
              acc[q][1] = fmaf(sa_g, c[q][1], acc[q][1]);
              acc[q][2] = fmaf(sb_g, c[q][2], acc[q][2]);
              acc[q][3] = fmaf(sb_g, c[q][3], acc[q][3]);
            }
          }
        }
        xq += (TILES * 2048) << p.split_log;
        if (j + u + 2 < n) fetch(u, j + u + 2);   // into the registers just used; the other segment's work covers its way
      }
    }
  }
#pragma unroll
  for (int q = 0; q < TILES; ++q)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if constexpr (sizeof(T) == 2) {
        red[warp][8 * q + 2 * t][g + 8 * h] = acc[q][2 * h];
        red[warp][8 * q + 2 * t + 1][g + 8 * h] = acc[q][2 * h + 1];
      } else {   // the pieces' columns: two in a lane, the third in the next
        const float mine = t & 1 ? acc[q][2 * h] : acc[q][2 * h] + acc[q][2 * h + 1];
        const float v = mine + __shfl_xor_sync(0xffffffffu, mine, 1);
        if (!(t & 1)) red[warp][2 * q + (t >> 1)][g + 8 * h] = v;
      }
    }
  __syncthreads();
  gp_finish<T>(p, red, m0);
}

}  // namespace wdz
